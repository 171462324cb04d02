// Wide affine layers: y = act(x W^T + bias) + residual and its gradients as matrix products on the MFMA units.
//
// One kernel does the three products, D[m][n] = sum_k A[m][k] B[n][k]:
//   forward   m = position, n = output, k = input     A = x (k contiguous)    B = W (n contiguous)
//   grad_x    m = position, n = input,  k = output    A = gz (k contiguous)   B = W (k contiguous)
//   dW        m = input,    n = output, k = position  A = x (m contiguous)    B = gz (n contiguous)
// A k-contiguous operand is staged in LDS as rows of 128 bytes of k and read 16 bytes a lane; one that is contiguous the
// other way is staged as it lies and read transposed (ds_read_b64_tr_b16 for 16-bit types, single words for f32), so no
// operand is ever transposed in memory. f32 goes through v_mfma_f32_16x16x4_f32: exact products, 32-bit sums.
//
// Times in this file: of a long run of calls, over operands that the caches do not hold where they are large. The first calls
// after the card has idled take more, 264 us instead of 218 of the largest product; comparisons of two variants are of one run.
#include <type_traits>

#include "common.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

template <typename T>
struct Elem {
    static constexpr int V = 16 / sizeof(T);          // elements of a 16-byte chunk
    static constexpr int BK = 128 / sizeof(T);        // k per tile: 128 bytes
    typedef T frag __attribute__((ext_vector_type(16 / sizeof(T))));
};

// acc += a b^T over the k of one fragment: lane l holds row l % 16 and, of 16-bit types, k = 8 (l / 16) .. + 7 of 32 (one
// MFMA), of f32 k = 4 (l / 16) .. + 3 of 16 (four of them, each taking one k from every 16 lanes)
__device__ __forceinline__ void mma(v4f &acc, const Elem<__bf16>::frag &a, const Elem<__bf16>::frag &b, int) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(v4f &acc, const Elem<_Float16>::frag &a, const Elem<_Float16>::frag &b, int) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(v4f &acc, const Elem<float>::frag &a, const Elem<float>::frag &b, int j) {
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], acc, 0, 0, 0);
}
// products of one fragment of m with the wave's fragments of n
template <typename T, int FM, int FN>
__device__ __forceinline__ void mma_col(v4f (&acc)[FN][FM], int j, const typename Elem<T>::frag (&b)[FN], const typename Elem<T>::frag &a) {
#pragma unroll
    for (int q = 0; q < (sizeof(T) == 4 ? 4 : 1); q++)  // (f32: four in turn on each block of sums, others in between)
#pragma unroll
        for (int i = 0; i < FN; i++) mma(acc[i][j], b[i], a, q);
}

// One operand's tile. KC: rows of m (or n), contiguous in k; otherwise rows of k, contiguous in m (or n). Slot s of the tile
// is its s-th 16 bytes in LDS; which chunk of the matrix it holds is permuted inside each row so that the lanes that are
// served together hit different banks:
//   KC        16 lanes read one chunk column of 16 rows 128 bytes apart: chunk ^ (row & 7)
//   16-bit    a transposed read takes 32 bytes of each of 4 consecutive rows, rows r and r + 8 next to each other in time
//   f32       words of 16 lanes are 64 bytes of a row; the four groups of lanes read rows 4 apart
template <typename T, bool KC, int SPAN>  // SPAN: tile extent in m or n
struct Tile {
    static constexpr int V = Elem<T>::V, BK = Elem<T>::BK;
    static constexpr int ROWS = KC ? SPAN : BK;
    static constexpr int CPR = KC ? 8 : SPAN / V;  // chunks per row
    static constexpr int SLOTS = ROWS * CPR, BYTES = SLOTS * 16;
    static __device__ __forceinline__ int swizzle(int row, int c) {
        if (KC) return c ^ (row & 7);
        if (sizeof(T) == 4) return c ^ ((((row >> 2) & 3) << 2) & (CPR - 1));
        return c ^ ((((row & 3) | ((row >> 3) & 1) << 2) << 1) & (CPR - 1));
    }
    // Where lane l's part of fragment f0 (16 of SPAN; a multiple of the wave's number of fragments, a power of two) lies at
    // k-step 0, and its fragment f0 + f at k-step s from there: the swizzle leaves the rest to a flipped bit or two and
    // constant distances. LDS addresses; tiles start on 1024 bytes.
    static __device__ __forceinline__ uint32_t origin(int f0, int lane) {
        const int g = lane >> 4, i = lane & 15;
        if (KC) return (f0 * 16 + i) * 128 + (g ^ (i & 7)) * 16;
        if (sizeof(T) == 4) {
            const int row = g * 4;
            return (row * CPR + swizzle(row, f0 * 4 + (i >> 2))) * 16 + (i & 3) * 4;
        }
        // 16 lanes give the addresses of 4 rows of 16 elements and get 4 rows of one column each
        const int row = g * 8 + (i >> 2);
        return (row * CPR + swizzle(row, f0 * 2 + ((i >> 1) & 1))) * 16 + (i & 1) * 8;
    }
    static __device__ __forceinline__ typename Elem<T>::frag read(uint32_t at, int f, int s) {
        typedef typename Elem<T>::frag frag;
        if constexpr (KC) {
            return *(const __attribute__((address_space(3))) frag *)(uintptr_t)((at ^ (s * 64)) + f * 2048);
        } else if constexpr (sizeof(T) == 4) {
            frag r;
#pragma unroll
            for (int j = 0; j < 4; j++)
                r[j] = *(const __attribute__((address_space(3))) float *)(uintptr_t)((at ^ (f * 64)) + (s * 16 + j) * CPR * 16);
            return r;
        } else {
            typedef short s4 __attribute__((ext_vector_type(4)));
            s4 h[2];
#pragma unroll
            for (int q = 0; q < 2; q++)
                h[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s4 *)(uintptr_t)((at ^ (f * 32)) + (s * 32 + q * 4) * CPR * 16));
            return __builtin_bit_cast(frag, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// An operand in memory: `rows` rows of `len` contiguous elements, `ld` apart.
struct Operand {
    const void *p0, *p1, *p2;  // the summands that a 16-bit gradient may be kept as, or the same matrix three times
    long long ld;
    int rows, len;
    int aligned;  // every chunk of every row starts on 16 bytes
    // the pointers in registers of their own: a choice between them must not become a choice of where to load one from
    // (that puts the kernel's arguments into scratch memory)
    __device__ __forceinline__ Operand pinned() const {
        Operand o = *this;
        asm("" : "+s"(o.p0), "+s"(o.p1), "+s"(o.p2));
        return o;
    }
    __device__ __forceinline__ const void *summand(int i) const { return i == 0 ? p0 : i == 1 ? p1 : p2; }
};

// chunk (row, element e) of the matrix, zeros outside it
template <typename T>
__device__ __forceinline__ v4u load_chunk(const T *base, const Operand &o, int row, long long e) {
    constexpr int V = Elem<T>::V;
    typedef typename Elem<T>::frag frag __attribute__((aligned(sizeof(T))));
    typename Elem<T>::frag r = {};
    if (row < o.rows && e < o.len) {
        const auto *p = (const __attribute__((address_space(1))) T *)base + ((size_t)row * o.ld + e);
        if (o.len - e >= V) {
            r = *(const __attribute__((address_space(1))) frag *)p;
        } else {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (j < o.len - e) r[j] = p[j];
        }
    }
    return __builtin_bit_cast(v4u, r);
}

enum { OUT_LAYER = 0, OUT_TYPE = 1, OUT_F32 = 2, OUT_PART = 3 };
struct Epilogue {
    const float *bias;
    const void *residual;
    void *out, *saved;
    long long ld;
    int act;
    float alpha;
    int past;  // outputs are stored past the caches (see past_caches)
};

// W neighbouring columns of one row, n of them inside the matrix
template <typename T, int W>
struct Cols {
    typedef float sums __attribute__((ext_vector_type(W)));
    typedef T vec __attribute__((ext_vector_type(W)));
    static __device__ __forceinline__ vec load(const T *p, int n) {
        vec v = {};
        if (n >= W) {
            __builtin_memcpy(&v, p, sizeof(v));
        } else {
#pragma unroll
            for (int j = 0; j < W; j++)
                if (j < n) v[j] = p[j];
        }
        return v;
    }
    static __device__ __forceinline__ void store(T *p, sums v, int n, bool past) {
        typedef T any __attribute__((ext_vector_type(W), aligned(sizeof(T))));
        vec q;
#pragma unroll
        for (int j = 0; j < W; j++) q[j] = (T)v[j];
        if (n >= W && past) {
            __builtin_nontemporal_store((any)q, (any *)p);
        } else if (n >= W) {
            __builtin_memcpy(p, &q, sizeof(q));
        } else {
#pragma unroll
            for (int j = 0; j < W; j++)
                if (j < n) p[j] = q[j];
        }
    }
};
template <typename T, int OUT, int W>
__device__ __forceinline__ typename Cols<T, W>::vec residual_at(const Epilogue &e, int row, int c, int n) {
    if (OUT != OUT_LAYER || !e.residual) return typename Cols<T, W>::vec{};
    return Cols<T, W>::load((const T *)e.residual + ((size_t)row * e.ld + c), n);
}
template <int OUT, int W>
__device__ __forceinline__ typename Cols<float, W>::sums bias_at(const Epilogue &e, int c, int n) {
    if (OUT != OUT_LAYER || !e.bias || n <= 0) return typename Cols<float, W>::sums{};
    return Cols<float, W>::load(e.bias + c, n);
}
// what becomes of W sums of one row, columns from c on
template <typename T, int OUT, int W>
__device__ __forceinline__ void finish_at(const Epilogue &e, int row, int c, int n, typename Cols<T, W>::sums v,
                                          typename Cols<T, W>::sums bias, typename Cols<T, W>::vec residual) {
    const size_t at = (size_t)row * e.ld + c;
    if constexpr (OUT == OUT_F32) {
        Cols<float, W>::store((float *)e.out + at, v * e.alpha, n, e.past);
    } else if constexpr (OUT == OUT_TYPE) {
        Cols<T, W>::store((T *)e.out + at, v * e.alpha, n, e.past);
    } else {
        v += bias;
        // bt_act_fwd without its branches, but for NaN: this is unrolled over a whole tile
        const float top = e.act == BT_ACT_CRELU || e.act == BT_ACT_SCRELU ? 1.0f : __builtin_huge_valf();
        const bool clamp = e.act != BT_ACT_IDENTITY, square = e.act == BT_ACT_SCRELU || e.act == BT_ACT_SQRRELU;
#pragma unroll
        for (int j = 0; j < W; j++) {
            const float a = fminf(fmaxf(v[j], 0.0f), top), b = square ? a * a : a;
            v[j] = clamp && v[j] == v[j] ? b : v[j];  // (NaN stays: a layer that has diverged shows)
        }
        if (e.saved) Cols<T, W>::store((T *)e.saved + at, v, n, e.past);
        if (e.residual) {
#pragma unroll
            for (int j = 0; j < W; j++) v[j] += (float)residual[j];
        }
        Cols<T, W>::store((T *)e.out + at, v, n, e.past);
    }
}

constexpr float F16_LIFT = 2048.0f;  // between the two summands of an f16 gradient (affine_gz)

// a launch holds less than 2^32 threads a dimension: many workgroups fold into the grid's second one (the last of its rows may
// hold some that have no work)
__device__ __forceinline__ long long folded_block() { return (long long)blockIdx.y * gridDim.x + blockIdx.x; }
dim3 folded(long long blocks) {
    constexpr long long W = 1 << 21;
    return dim3((unsigned)(blocks < W ? blocks : W), (unsigned)((blocks + W - 1) / W));
}

// dbias from the row ranges' sums that affine_prepare leaves, by workgroups of their own behind a product's
struct BiasSum {
    const float *part;  // [parts][n]
    float *out;
    int parts, n, blocks;
    float alpha;
};
constexpr int BIAS_COLS = 32;
template <int NT>
__device__ __forceinline__ void bias_sum(const BiasSum b, int block, float *lds) {  // lds: NT floats
    if (block >= b.blocks) return;
    const int c = threadIdx.x % BIAS_COLS, r = threadIdx.x / BIAS_COLS, col = block * BIAS_COLS + c;
    float s = 0.0f;
    if (col < b.n)
#pragma unroll 8
        for (int p = r; p < b.parts; p += NT / BIAS_COLS) s += b.part[(size_t)p * b.n + col];
    lds[threadIdx.x] = s;
    __syncthreads();
    if (r || col >= b.n) return;
    for (int q = 1; q < NT / BIAS_COLS; q++) s += lds[q * BIAS_COLS + c];
    b.out[col] = s * b.alpha;
}
__global__ __launch_bounds__(256) void affine_dbias(BiasSum b) {
    __shared__ float lds[256];
    bias_sum<256>(b, (int)folded_block(), lds);
}

struct Product {
    Operand a, b;
    int m, n, k;
    int passes;          // summands of the operands, taken one after the other
    int lift;            // the first of two summands is F16_LIFT times too large: one half of the splits takes it, the other
                         // half the second one, and affine_join puts it right
    int tiles_m, tiles_n;
    int splits;          // workgroups that share one tile's k, each leaving its sums in `part`
    float *part;         // [splits][m][part_ld]
    long long part_ld;
    Epilogue e;
    BiasSum bias;
    int wgs;             // workgroups of the product; bias.blocks more follow them in its launch
};
// A chunk straight from memory into LDS, 16 bytes a lane: lane l's lands 16 l bytes behind `lds` (the same in all lanes).
// Written out, since the compiler lets every LDS read wait for all such loads of its own; wait_loads() is the wait (for all but
// the N youngest loads), in front of the barrier behind which the chunk is read. The s_nop is the wait state between m0 and
// its use.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (that m0 is a reserved register: it is, and this is where it changes)
__device__ __forceinline__ void to_lds(const char *base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %2" : : "v"(offset), "s"(lds), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N = 0>
__device__ __forceinline__ void wait_loads() {
    static_assert(N < 64, "what the counter holds");
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const char *p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)p;
}

// between a wave's writes to LDS and its own lanes' reads of them, which the hardware takes in order
__device__ __forceinline__ void lds_turn() {
    asm volatile("" : : : "memory");
    __builtin_amdgcn_wave_barrier();
}

// One operand's tiles on their way into LDS, for a workgroup of NT threads.
template <typename T, bool KC, int SPAN, int NT>
struct Stage {
    typedef Tile<T, KC, SPAN> L;
    static constexpr int V = Elem<T>::V, BK = Elem<T>::BK, N = L::SLOTS / NT;
    // chunk of slot s of the tile at (s0, k0), zeros where the matrix has nothing
    static __device__ __forceinline__ v4u chunk(const Operand &o, int pass, int s0, int k0, int s) {
        const int row = s / L::CPR, c = L::swizzle(row, s % L::CPR);
        return load_chunk<T>((const T *)o.summand(pass), o, (KC ? s0 : k0) + row, (long long)(KC ? k0 : s0) + c * V);
    }
    static __device__ __forceinline__ void get(const Operand &o, int pass, int s0, int k0, int tid, v4u (&r)[N]) {
#pragma unroll
        for (int q = 0; q < N; q++) r[q] = chunk(o, pass, s0, k0, q * NT + tid);
    }
    static __device__ __forceinline__ void put(const v4u (&r)[N], int tid, char *lds) {
#pragma unroll
        for (int q = 0; q < N; q++) *(v4u *)(lds + (q * NT + tid) * 16) = r[q];
    }
    // Direct loads: byte offsets of this thread's chunks from the tile's first element, the same for every tile. Rows (or
    // chunks) of m or n beyond the end are taken from the last one: their sums are not stored. Where that chunk is ragged,
    // the elements behind it are whatever lies there up to the next row; there is no next row behind the last one.
    static __device__ __forceinline__ bool ragged(const Operand &o, int s0) { return !KC && o.len - s0 < SPAN && o.len % V; }
    static __device__ __forceinline__ void offsets(const Operand &o, int s0, int tid, uint32_t (&off)[N]) {
        const int left = (KC ? o.rows : o.len) - s0;  // > 0
#pragma unroll
        for (int q = 0; q < N; q++) {
            const int s = q * NT + tid;
            int row = s / L::CPR, c = L::swizzle(row, s % L::CPR);
            if (KC) row = min(row, left - 1);
            if (!KC) c = min(c, (left - 1) / V);
            off[q] = (uint32_t)row * (uint32_t)(o.ld * sizeof(T)) + c * 16;
        }
    }
    // a tile that the matrix does not fill: its whole chunks directly, the others through registers with zeros for what is
    // not there
    static __device__ __forceinline__ void careful(const Operand &o, int pass, int s0, int k0, int tid, char *lds) {
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds_address(lds) + (tid & ~63) * 16);
        const char *base = first(o, pass, s0, k0);
#pragma unroll 1
        for (int q = 0; q < N; q++) {
            const int s = q * NT + tid, row = s / L::CPR, c = L::swizzle(row, s % L::CPR);
            const int r = (KC ? s0 : k0) + row, e = (KC ? k0 : s0) + c * V;
            if (r < o.rows && o.len - e >= V)
                to_lds(base, (uint32_t)row * (uint32_t)(o.ld * sizeof(T)) + c * 16, to + q * NT * 16);
            else
                *(v4u *)(lds + s * 16) = chunk(o, pass, s0, k0, s);
        }
    }
    static __device__ __forceinline__ const char *first(const Operand &o, int pass, int s0, int k0) {
        return (const char *)o.summand(pass) + ((KC ? s0 : k0) * (size_t)o.ld + (KC ? k0 : s0)) * sizeof(T);
    }
    static __device__ __forceinline__ size_t step(const Operand &o) { return KC ? 128 : (size_t)o.ld * sizeof(T) * BK; }
};

// Workgroups go to the 8 XCDs in turn, each with an L2 of its own: what number makes every XCD's share contiguous
__device__ __forceinline__ int xcd_share(int wg, int wgs) {
    const int per = wgs / 8, rest = wgs % 8, xcd = wg % 8;
    return xcd * per + min(xcd, rest) + wg / 8;
}
// Which tile a workgroup takes: an XCD walks its share in bands of 8 tiles of m, so that what it holds of both operands is
// reused.
__device__ __forceinline__ void tile_of(int wg, int wgs, int tiles_m, int tiles_n, int &split, int &tm, int &tn) {
    wg = xcd_share(wg, wgs);
    // (a division costs more than a tile's worth of products of a short sum: none where the answer is known)
    const unsigned tiles = tiles_m * tiles_n;
    split = wgs == (int)tiles ? 0 : (unsigned)wg / tiles;
    const unsigned t = wg - split * tiles, per_band = 8 * tiles_n, band = t / per_band, in = t - band * per_band;
    const unsigned high = min(8, tiles_m - (int)band * 8);
    tn = high == 8 ? in / 8 : in / high;
    tm = band * 8 + (in - tn * high);
}

// What the kernels below share: a BM x BN tile by WM x WN waves, each with FM x FN blocks of 16 x 16 sums.
template <typename T, int BM, int BN, int WM, int WN, bool AK, bool BKC, int OUT>
struct Mm {
    static constexpr int NT = 64 * WM * WN, BK = Elem<T>::BK, FM = BM / WM / 16, FN = BN / WN / 16;
    typedef Tile<T, AK, BM> TA;
    typedef Tile<T, BKC, BN> TB;
    typedef Stage<T, AK, BM, NT> SA;
    typedef Stage<T, BKC, BN, NT> SB;
    static constexpr int BYTES = TA::BYTES + TB::BYTES;  // of one buffer
    typedef typename Elem<T>::frag frag;
    const Product &P;
    const Operand a, b;
    char *lds;
    int tid, lane, wm, wn, split, m0, n0;
    uint32_t at_a, at_b;  // where this lane reads a tile of the first buffer
    v4f acc[FN][FM];

    // workgroup `wg` of the product's
    __device__ __forceinline__ Mm(const Product &P_, char *lds_, int wg)
        : P(P_), a(P_.a.pinned()), b(P_.b.pinned()), lds(lds_) {
        tid = threadIdx.x, lane = tid & 63;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        wm = wave / WN, wn = wave % WN;
        int tm, tn;
        tile_of(wg, P.wgs, P.tiles_m, P.tiles_n, split, tm, tn);
        m0 = tm * BM, n0 = tn * BN;
        at_a = lds_address(lds) + TA::origin(wm * FM, lane), at_b = lds_address(lds) + TA::BYTES + TB::origin(wn * FN, lane);
#pragma unroll
        for (int i = 0; i < FN; i++)
#pragma unroll
            for (int j = 0; j < FM; j++) acc[i][j] = v4f{0, 0, 0, 0};
    }
    // This workgroup's share of `ktiles` tiles of k a summand: the summands [p0, p1), the tiles [t0, t1) of theirs put one
    // behind the other, and whether that is the last share of them.
    __device__ __forceinline__ bool share(int ktiles, int &p0, int &p1, int &t0, int &t1) const {
        const int half = P.lift ? P.splits / 2 : 0;  // splits of the first summand, where each takes one of the two
        const bool second = P.lift && split >= half;
        const int subs = P.lift ? half : P.splits, sub = second ? split - half : split;
        p0 = second, p1 = P.lift ? p0 + 1 : P.passes;
        const unsigned all = (unsigned)ktiles * (p1 - p0);
        if (subs == 1) {
            t0 = 0, t1 = all;
        } else {  // the first all % subs shares are one longer
            const unsigned each = all / subs, rest = all - each * subs;
            t0 = sub * each + min((unsigned)sub, rest), t1 = t0 + each + ((unsigned)sub < rest);
        }
        return sub == subs - 1;
    }
    __device__ __forceinline__ frag read_a(int buf, int j, int s) const { return TA::read(at_a + buf * BYTES, j, s); }
    __device__ __forceinline__ frag read_b(int buf, int i, int s) const { return TB::read(at_b + buf * BYTES, i, s); }
    __device__ __forceinline__ void multiply(int buf) {
#pragma unroll
        for (int s = 0; s < 2; s++) {
            frag fa[FM], fb[FN];
#pragma unroll
            for (int j = 0; j < FM; j++) fa[j] = read_a(buf, j, s);
#pragma unroll
            for (int i = 0; i < FN; i++) fb[i] = read_b(buf, i, s);
#pragma unroll
            for (int j = 0; j < FM; j++) mma_col<T, FM, FN>(acc, j, fb, fa[j]);
        }
    }
    // Lane l holds, of each 16 x 16 block, row m = l % 16 and columns n = 4 (l / 16) .. + 3. Every wave turns 16 rows at a
    // time in its own piece of LDS, so that neighbouring lanes finish (and load and store) 16 bytes each of one row's
    // consecutive columns. (8 bytes each take twice as long: 67 MB of bf16 in 21 us, as long as 134 MB of f32.)
    __device__ __forceinline__ void finish() {
        constexpr int W = OUT <= OUT_TYPE ? Elem<T>::V : 4;
        constexpr int COLS = FN * 16, STRIDE = COLS + 4, LANES = COLS / W, ROWS = 64 / LANES;
        static_assert(WM * WN * 16 * STRIDE * 4 <= 2 * BYTES, "the waves' strips fit the tiles' LDS");
        typedef Cols<T, W> Row;
        float *strip = (float *)lds + (wm * WN + wn) * 16 * STRIDE;
        const int n = n0 + wn * COLS + (lane % LANES) * W;
        // the residual's loads go ahead of everything, as far as registers allow: in turn with the stores (which may go to
        // the same buffer) each would wait for memory
        constexpr int PASSES = 16 / ROWS, AHEAD = FM <= 4 ? FM : 1;
        typename Row::vec res[AHEAD][PASSES];
        const auto ahead = [&](int j) {
#pragma unroll
            for (int i = 0; i < PASSES; i++) {
                const int m = m0 + (wm * FM + j) * 16 + i * ROWS + lane / LANES;
                if (m < P.m && n < P.n) res[j % AHEAD][i] = residual_at<T, OUT, W>(P.e, m, n, P.n - n);
            }
        };
        if (AHEAD > 1)
#pragma unroll
            for (int j = 0; j < AHEAD; j++) ahead(j);
        const typename Row::sums bias = bias_at<OUT, W>(P.e, n, P.n - n);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < FM; j++) {
            if (AHEAD == 1) ahead(j);
#pragma unroll
            for (int i = 0; i < FN; i++) *(v4f *)(strip + (lane & 15) * STRIDE + i * 16 + (lane >> 4) * 4) = acc[i][j];
            lds_turn();
#pragma unroll
            for (int i = 0; i < PASSES; i++) {
                const int r = i * ROWS + lane / LANES, m = m0 + (wm * FM + j) * 16 + r;
                typename Row::sums v;
#pragma unroll
                for (int q = 0; q < W; q += 4) {
                    const v4f x = *(const v4f *)(strip + r * STRIDE + (lane % LANES) * W + q);
#pragma unroll
                    for (int c = 0; c < 4; c++) v[q + c] = x[c];
                }
                if (m >= P.m || n >= P.n) continue;
                if constexpr (OUT == OUT_PART)
                    *(v4f *)(P.part + ((size_t)split * P.m + m) * P.part_ld + n) = v;  // (part_ld: a multiple of 4)
                else
                    finish_at<T, OUT, W>(P.e, m, n, P.n - n, v, bias, res[j % AHEAD][i]);
            }
            lds_turn();
        }
    }
};

// Operands of any alignment: the next tile is loaded into registers while this one is multiplied.
template <typename T, int BM, int BN, int WM, int WN, bool AK, bool BKC, int OUT>
__global__ __launch_bounds__(64 * WM * WN) void affine_mm_any(Product P) {
    typedef Mm<T, BM, BN, WM, WN, AK, BKC, OUT> M;
    extern __shared__ __align__(1024) char lds[];
    const int wg = (int)folded_block();
    if (wg >= P.wgs) return bias_sum<M::NT>(P.bias, wg - P.wgs, (float *)lds);
    M mm(P, lds, wg);
    const int ktiles = (P.k + M::BK - 1) / M::BK;
    int p0, p1, t0, t1;
    mm.share(ktiles, p0, p1, t0, t1);
    v4u ra[M::SA::N], rb[M::SB::N];
    auto get = [&](int kt) {
        const int pass = kt / ktiles, k0 = (kt - pass * ktiles) * M::BK;
        M::SA::get(mm.a, p0 + pass, mm.m0, k0, mm.tid, ra);
        M::SB::get(mm.b, p0 + pass, mm.n0, k0, mm.tid, rb);
    };
    if (t0 < t1) get(t0);
    for (int kt = t0; kt < t1; kt++) {
        char *buf = lds + ((kt - t0) & 1) * M::BYTES;
        M::SA::put(ra, mm.tid, buf);
        M::SB::put(rb, mm.tid, buf + M::TA::BYTES);
        __syncthreads();  // this tile is here, and every wave is done with the other buffer
        if (kt + 1 < t1) get(kt + 1);
        mm.multiply((kt - t0) & 1);
    }
    mm.finish();
}

// Operands whose chunks start on 16 bytes: tiles go straight into LDS, and three things are under way at any time. While
// the first half of a tile's k is multiplied the second half's fragments are read; behind the barrier that says that the
// next tile has arrived its first fragments are read, and another tile is sent for into the buffer just left, while the
// second half is multiplied. Each fragment's products carry their share of those reads and loads.
// The tiles that k fills come first; the others, one of each summand (the rest of k; the last full one, where its last row
// must not be read to the end of a chunk), take the same way with a check of every chunk.
//
// Bound by the MFMA units and, close behind, by the LDS bytes that feed them, which is why the largest tile that still fills
// the chip is taken: for one product of 16 x 16 x 32 a 256 x 256 tile reads 384 bytes of LDS, a 128 x 128 one 512 and a
// 64 x 64 one 1024. 16384 x 2048 -> 4096 bf16 takes 218 us, 1.26 PFLOP/s (the MFMA units are busy 58 % of the clocks, bank
// conflicts are few); dW of 16384 x 2048 -> 2048 with 4 workgroups to a tile 108 us and grad_x 105, 1.27 and 1.32 PFLOP/s;
// 4096 x 1024 -> 1024 f32 with 64 x 64 tiles, residual and kept activation 71 us, 121 TFLOP/s, 79 % of a large library product's.
template <typename T, int BM, int BN, int WM, int WN, bool AK, bool BKC, int OUT, int BUFS>
__device__ __forceinline__ void mm_direct(const Product &P, int wg, char *lds) {
    typedef Mm<T, BM, BN, WM, WN, AK, BKC, OUT> M;
    typedef typename M::frag frag;
    constexpr int FM = M::FM, FN = M::FN, NA = M::SA::N, NB = M::SB::N;
    if (wg >= P.wgs) return bias_sum<M::NT>(P.bias, wg - P.wgs, (float *)lds);
    M mm(P, lds, wg);
    const bool ragged = M::SA::ragged(mm.a, mm.m0) || M::SB::ragged(mm.b, mm.n0);
    const int full = (P.k - ragged) / M::BK;
    int p0, p1, t0, t1;
    const bool last = mm.share(full, p0, p1, t0, t1);
    const int quick = t1 - t0, tiles = quick + (last && full * M::BK < P.k ? p1 - p0 : 0);

    uint32_t oa[NA], ob[NB];
    M::SA::offsets(mm.a, mm.m0, mm.tid, oa);
    M::SB::offsets(mm.b, mm.n0, mm.tid, ob);
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_address(lds) + (mm.tid & ~63) * 16);
    // the filled tile to be sent for next: its summand, its number in there, its first elements
    int pass = p0, at = 0;
    if (t0) pass += t0 / full, at = t0 % full;  // (t0 > 0: so is full)
    const char *pa = M::SA::first(mm.a, pass, mm.m0, at * M::BK), *pb = M::SB::first(mm.b, pass, mm.n0, at * M::BK);
    const size_t step_a = M::SA::step(P.a), step_b = M::SB::step(P.b);
    const auto send = [&](int q, int buf) {  // chunk q of both operands' NA + NB
        if (q < NA)
            to_lds(pa, oa[q < NA ? q : 0], to + buf * M::BYTES + q * M::NT * 16);
        else
            to_lds(pb, ob[q < NA ? 0 : q - NA], to + buf * M::BYTES + M::TA::BYTES + (q - NA) * M::NT * 16);
    };
    const auto advance = [&]() {
        pa += step_a, pb += step_b;
        if (++at == full) {
            at = 0, pass = min(pass + 1, p1 - 1);
            pa = M::SA::first(mm.a, pass, mm.m0, 0), pb = M::SB::first(mm.b, pass, mm.n0, 0);
        }
    };
    const auto careful = [&](int tile, int buf) {
        M::SA::careful(mm.a, p0 + tile - quick, mm.m0, full * M::BK, mm.tid, lds + buf * M::BYTES);
        M::SB::careful(mm.b, p0 + tile - quick, mm.n0, full * M::BK, mm.tid, lds + buf * M::BYTES + M::TA::BYTES);
    };
    frag fa[FM], fb[2][FN];
    // The products of half 1 - s, and beside them: fragments of half s of the tile in buffer `buf` (of m: into the registers
    // just used; of n: into a second set), and with SEND the next tile's chunks into buffer `to_buf`.
    const auto half = [&](auto s_, auto send_, int buf, int to_buf) {
        constexpr int s = decltype(s_)::value;
        constexpr bool SEND = decltype(send_)::value;
#pragma unroll
        for (int j = 0; j < FM; j++) {
            if (SEND) {
#pragma unroll
                for (int q = (NA + NB) * j / FM; q < (NA + NB) * (j + 1) / FM; q++) send(q, to_buf);
            }
#pragma unroll
            for (int i = FN * j / FM; i < FN * (j + 1) / FM; i++) fb[s][i] = mm.read_b(buf, i, s);
            mma_col<T, FM, FN>(mm.acc, j, fb[1 - s], fa[j]);
            fa[j] = mm.read_a(buf, j, s);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    const std::integral_constant<int, 0> zero;
    const std::integral_constant<int, 1> one;
    if (tiles > 0) {
#pragma unroll 1
        for (int t = 0; t < BUFS && t < tiles; t++) {
            if (t < quick) {
#pragma unroll
                for (int q = 0; q < NA + NB; q++) send(q, t);
                advance();
            } else {
                careful(t, t);
            }
        }
        if (quick >= BUFS)
            wait_loads<(BUFS - 1) * (NA + NB)>();
        else
            wait_loads();
        __syncthreads();
#pragma unroll
        for (int j = 0; j < FM; j++) fa[j] = mm.read_a(0, j, 0);
#pragma unroll
        for (int i = 0; i < FN; i++) fb[0][i] = mm.read_b(0, i, 0);
    }
    int t = 0, cur = 0;
    const auto next = [&]() { return BUFS == 2 ? cur ^ 1 : cur == BUFS - 1 ? 0 : cur + 1; };
    for (; t + BUFS < quick; t++, cur = next()) {
        half(one, std::false_type(), cur, 0);
        wait_loads<(BUFS - 2) * (NA + NB)>();
        __syncthreads();  // the next tile is here, and every wave has read this one
        half(zero, std::true_type(), next(), cur);
        advance();
    }
#pragma unroll 1
    for (; t < tiles; t++, cur = next()) {
        half(one, std::false_type(), cur, 0);
        wait_loads();
        __syncthreads();
        if (t + BUFS < tiles) careful(t + BUFS, cur);
        half(zero, std::false_type(), next(), 0);  // (behind the last tile: fragments that nothing uses)
    }
    mm.finish();
}

template <typename T, int BM, int BN, int WM, int WN, bool AK, bool BKC, int OUT, int BUFS>
__global__ __launch_bounds__(64 * WM * WN, 2) void affine_mm_direct(Product P) {
    extern __shared__ __align__(1024) char lds[];
    mm_direct<T, BM, BN, WM, WN, AK, BKC, OUT, BUFS>(P, (int)folded_block(), lds);
}
// dW and grad_x of a small layer in one launch: neither has tiles enough to fill the chip, or to hide its own latency
// (200 x 512 -> 333 f32: 7.2 us, 288 workgroups of 32 x 32 that each walk their whole k; 76 of 64 x 64: 11)
template <typename T, int B, int OUT_W, int OUT_X, int BUFS>
__global__ __launch_bounds__(256, 2) void affine_mm_both(Product W, Product X) {
    extern __shared__ __align__(1024) char lds[];
    const int wg = (int)folded_block(), first = W.wgs + W.bias.blocks;
    if (wg < first)
        mm_direct<T, B, B, 2, 2, false, false, OUT_W, BUFS>(W, wg, lds);
    else
        mm_direct<T, B, B, 2, 2, true, true, OUT_X, BUFS>(X, wg - first, lds);
}

// The splits' sums added in order, then the epilogue. Memory bound: 4 splits of 2048 x 2048 (67 MB of sums, 17 MB out) 13 us,
// 6.5 TB/s, some of the sums still in the caches.
template <typename T, int OUT>
__global__ __launch_bounds__(256) void affine_join(Product P) {
    const long long q = folded_block() * 256 + threadIdx.x, cols = P.part_ld / 4;
    if (q >= cols * P.m) return;
    const int m = (int)(q / cols), n = (int)(q % cols) * 4;
    v4f v = {0, 0, 0, 0};
    const float *part = P.part + (size_t)m * P.part_ld + n;
    const size_t step = (size_t)P.m * P.part_ld;
    const auto add = [&](int s0, int s1) {
#pragma unroll 8
        for (int s = s0; s < s1; s++) v += *(const v4f *)(part + s * step);
    };
    const int lifted = P.lift ? P.splits / 2 : 0;
    add(0, lifted);
    if (P.lift) v *= 1.0f / F16_LIFT;
    add(lifted, P.splits);
    finish_at<T, OUT, 4>(P.e, m, n, P.n - n, v, bias_at<OUT, 4>(P.e, n, P.n - n), residual_at<T, OUT, 4>(P.e, m, n, P.n - n));
}

// What a product needs made before it, in one launch: copies of matrices, and gz.
//
// A copy has rows on 128 bytes (so that a tile's row of k is one line of memory), of the layer's type (f32 weights are
// rounded), with zeros up to a whole chunk. One chunk a thread. Both the copies and gz are bound by memory: gz of 16384 x 2048
// bf16 (two reads, one write, 201 MB) 38 us, 5.3 TB/s.
template <typename T>
struct Copy {
    const void *from;
    T *to;
    long long from_ld, to_ld;
    int rows, len, f32, blocks;
};
template <typename From, typename T>
__device__ __forceinline__ void copy_chunk(const From *p, int left, T *to) {
    constexpr int V = Elem<T>::V;
    typedef From vec __attribute__((ext_vector_type(V)));
    vec v = {};
    if (left >= V) {
        __builtin_memcpy(&v, p, sizeof(v));
    } else {
#pragma unroll
        for (int j = 0; j < V; j++)
            if (j < left) v[j] = p[j];
    }
    typename Elem<T>::frag r;
#pragma unroll
    for (int j = 0; j < V; j++) r[j] = (T)(float)v[j];
    *(typename Elem<T>::frag *)to = r;
}
template <typename T>
__device__ __forceinline__ void copy_block(const Copy<T> &c, long long block) {
    constexpr int V = Elem<T>::V;
    const long long q = block * 256 + threadIdx.x, cols = (c.len + V - 1) / V;
    if (q >= cols * c.rows) return;
    const long long row = q / cols;
    const int e = (int)(q % cols) * V;
    T *to = c.to + row * c.to_ld + e;
    if (c.f32)
        copy_chunk<float, T>((const float *)c.from + row * c.from_ld + e, c.len - e, to);
    else
        copy_chunk<T, T>((const T *)c.from + row * c.from_ld + e, c.len - e, to);
}

// gz = grad_y act'(out) (half of it where act' carries a factor 2: the products' alpha gives it back, exactly), as one
// number of the layer's type or, NP > 1, as a sum: each further summand takes what the rounding of those before left over
// (two of f16: 22 bits, the second one times 2^11 so that it stays clear of the subnormals; three of bf16: 24 bits, two
// where the product is rounded to bf16 anyway). And the column sums of gz over this workgroup's rows.
// Thread (c, r) takes column chunk c and every 8th row from r on.
constexpr int GZ_COLS = 32, GZ_ROWS = 8;
template <typename T>
struct Gz {
    const T *gy, *out;  // out: null = no derivative
    T *p[3];            // summands, largest first; null = sums only
    float *sums;        // [ranges][n], or null
    long long ld, gz_ld;
    int batch, n, act, range, col_blocks, blocks;
};
template <typename T, int NP>
__device__ __forceinline__ void gz_block(const Gz<T> &G, int block) {
    constexpr int V = Elem<T>::V;
    constexpr float LIFT = std::is_same<T, _Float16>::value ? F16_LIFT : 1.0f;
    typedef typename Elem<T>::frag frag;
    __shared__ float red[GZ_ROWS][GZ_COLS * V];
    const int bx = block % G.col_blocks, by = block / G.col_blocks;
    const int c = threadIdx.x % GZ_COLS, r = threadIdx.x / GZ_COLS;
    const long long e = ((long long)bx * GZ_COLS + c) * V;
    const long long b0 = (long long)by * G.range, b1 = b0 + G.range < G.batch ? b0 + G.range : G.batch;
    const int left = e < G.n ? (int)(G.n - e < V ? G.n - e : V) : 0;
    const bool root = G.act == BT_ACT_SCRELU || G.act == BT_ACT_SQRRELU;
    const bool clipped = G.act == BT_ACT_CRELU || G.act == BT_ACT_SCRELU;
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; j++) sum[j] = 0.0f;
    if (left)
        for (long long b = b0 + r; b < b1; b += GZ_ROWS) {
            frag g = {}, o = {}, part[NP];
            const T *pg = G.gy + b * G.ld + e, *po = G.out ? G.out + b * G.ld + e : nullptr;
            if (left == V) {
                __builtin_memcpy(&g, pg, 16);
                if (po) __builtin_memcpy(&o, po, 16);
            } else {
                for (int j = 0; j < V; j++)
                    if (j < left) {
                        g[j] = pg[j];
                        if (po) o[j] = po[j];
                    }
            }
#pragma unroll
            for (int j = 0; j < V; j++) {
                // bt_act_deriv, halved where it has a factor 2, without its branches (for every output an activation has; one that
                // was too large for the type, infinity, has ReLU's slope 1 and squared ReLU's infinity)
                const float a = (float)o[j];
                float slope = a > 0.0f && (!clipped || a < 1.0f) ? 1.0f : 0.0f;
                if (root) slope *= __builtin_amdgcn_sqrtf(a);
                const float v = po ? (float)g[j] * slope : (float)g[j];
                sum[j] += v;
                float rest = v;
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    part[p][j] = (T)rest;
                    rest = (rest - (float)part[p][j]) * LIFT;
                    if (!(fabsf(rest) < __builtin_huge_valf())) rest = 0.0f;  // (an infinite gradient stays one)
                }
            }
            if (G.p[0]) {
#pragma unroll
                for (int p = 0; p < NP; p++)  // (gz_ld is a multiple of V: a last chunk is whole)
                    __builtin_memcpy(G.p[p] + b * G.gz_ld + e, &part[p], 16);
            }
        }
    if (!G.sums) return;
#pragma unroll
    for (int j = 0; j < V; j++) red[r][c * V + j] = sum[j];
    __syncthreads();
    for (int i = threadIdx.x; i < GZ_COLS * V; i += 256) {
        const long long col = (long long)bx * GZ_COLS * V + i;
        if (col >= G.n) continue;
        float s = 0.0f;
        for (int q = 0; q < GZ_ROWS; q++) s += red[q][i];
        G.sums[(size_t)by * G.n + col] = s;
    }
}

template <typename T>
struct Prepare {
    Copy<T> w, x;
    Gz<T> gz;
};
template <typename T, int NP>  // NP = 0: copies only
__global__ __launch_bounds__(256) void affine_prepare(Prepare<T> p) {
    long long block = folded_block();
    if constexpr (NP > 0) {
        if (block < p.gz.blocks) return gz_block<T, NP>(p.gz, (int)block);
        block -= p.gz.blocks;
    }
    if (block < p.w.blocks) return copy_block<T>(p.w, block);
    if (block - p.w.blocks < p.x.blocks) copy_block<T>(p.x, block - p.w.blocks);
}

// Forward of at most R rows (one position, or a few): the weights are all there is to read, and each is used R times, so
// there is nothing for the matrix cores. A workgroup takes 4 chunks of outputs (64 bytes of every weight column; f32
// weights of a 16-bit layer: 128) for all inputs: its groups of 4 lanes walk the inputs V at a time with V weight loads in
// flight each, and their sums meet in DPP, shuffles and LDS, in a fixed order. 1024 threads, or 512 where the sums and
// loads of more than 2 rows need the registers. 1 x 2048 -> 4096 bf16: 7.8 us with the weights (16.8 MB) in memory, which a copy
// would read in 3.3: 128 workgroups leave half of the CUs idle, and launch, the first load's latency and the reduction have nothing
// to hide behind. (Long sums into few outputs are one workgroup's: nothing shares k here.)
constexpr int few_threads(int rows) { return rows > 2 ? 512 : 1024; }
template <typename T, typename TW, int R>
__global__ __launch_bounds__(few_threads(R)) void affine_few(const TW *__restrict__ w, long long w_ld, const T *__restrict__ x, long long x_ld,
                                                   int batch, int in, int out, Epilogue e) {
    constexpr int V = Elem<T>::V, COLS = 4 * V, NT = few_threads(R);
    typedef TW wvec __attribute__((ext_vector_type(V)));
    typedef typename Elem<T>::frag xvec;
    __shared__ __align__(16) float red[NT / 64][R][COLS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = threadIdx.x >> 2;
    const int all = (out + COLS - 1) / COLS;
    if (folded_block() >= all) return;
    const int chunk = xcd_share((int)folded_block(), all);  // (neighbours read halves of the same lines)
    const int c = chunk * COLS + (threadIdx.x & 3) * V;
    float acc[R][V];
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < V; j++) acc[r][j] = 0.0f;
    for (long long k = (long long)group * V; k < in; k += NT / 4 * V) {
        const int nk = in - k < V ? (int)(in - k) : V;
        wvec wv[V];
        xvec xv[R];
#pragma unroll
        for (int i = 0; i < V; i++) {
            wv[i] = wvec{};
            if (i < nk) {
                const TW *p = w + (k + i) * w_ld + c;
                if (out - c >= V) {
                    __builtin_memcpy(&wv[i], p, sizeof(wvec));
                } else {
#pragma unroll
                    for (int j = 0; j < V; j++)
                        if (j < out - c) wv[i][j] = p[j];
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            const T *p = x + (long long)min(r, batch - 1) * x_ld + k;
            xv[r] = xvec{};
            if (nk == V) {
                __builtin_memcpy(&xv[r], p, 16);
            } else {
#pragma unroll
                for (int i = 0; i < V; i++)
                    if (i < nk) xv[r][i] = p[i];
            }
        }
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < nk)
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float f = (float)(T)wv[i][j];
#pragma unroll
                    for (int r = 0; r < R; r++) acc[r][j] = fmaf((float)xv[r][i], f, acc[r][j]);
                }
    }
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < V; j++) {
            float v = acc[r][j];  // the 16 lanes of a wave with the same columns
            v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xf, 0xf, false));  // 4 lanes on
            v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, false));  // 8 lanes on
            v += __shfl_xor(v, 16, 64);
            v += __shfl_xor(v, 32, 64);
            if (lane < 4) red[wave][r][lane * V + j] = v;
        }
    __syncthreads();
    if (threadIdx.x >= R * V) return;  // one thread for 4 outputs of a row
    const int r = threadIdx.x / V, q = (threadIdx.x % V) * 4, col = chunk * COLS + q;
    if (r >= batch || col >= out) return;
    v4f v = {0, 0, 0, 0};
    for (int i = 0; i < NT / 64; i++) v += *(const v4f *)&red[i][r][q];
    finish_at<T, OUT_LAYER, 4>(e, r, col, out - col, v, bias_at<OUT_LAYER, 4>(e, col, out - col),
                               residual_at<T, OUT_LAYER, 4>(e, r, col, out - col));
}

// ---- host side
size_t type_size(int type) { return type == BT_TYPE_F32 ? 4 : 2; }
bool elem_aligned(const void *p, size_t es) { return (reinterpret_cast<uintptr_t>(p) & (es - 1)) == 0; }

int validate(const bt_affine_desc *d, const char *fn) {
    BT_REQUIRE(d, "%s: null pointer", fn);
    BT_REQUIRE(d->batch > 0 && d->in > 0 && d->out > 0, "%s: Mismatched sizes! (%d x %d -> %d)", fn, d->batch, d->in, d->out);
    BT_REQUIRE(d->type == BT_TYPE_F32 || d->type == BT_TYPE_BF16 || d->type == BT_TYPE_F16, "%s: unknown element type %d", fn,
               d->type);
    BT_REQUIRE(d->w_type == d->type || d->w_type == BT_TYPE_F32, "%s: weights of type %d in a layer of type %d", fn, d->w_type,
               d->type);
    BT_REQUIRE(d->act >= BT_ACT_IDENTITY && d->act <= BT_ACT_SQRRELU, "%s: unknown activation %d", fn, d->act);
    BT_REQUIRE(d->w_ld >= d->out && d->x_ld >= d->in && d->y_ld >= d->out,
               "%s: Mismatched sizes! (a leading dimension is less than its row: w %d / %d, x %d / %d, y %d / %d)", fn, d->w_ld,
               d->out, d->x_ld, d->in, d->y_ld, d->out);
    // (each matrix is less than 2^36 elements, so that numbers of tiles, chunks and rows of partial sums fit 32 bits)
    const long long b = d->batch, i = d->in, o = d->out, most = 1ll << 36;
    BT_REQUIRE(b <= (1 << 30) && i <= (1 << 30) && o <= (1 << 30) && b * i <= most && b * o <= most && i * o <= most,
               "%s: Mismatched sizes! (too large)", fn);
    return BT_OK;
}

struct Shape {
    int bm, tiles_m, tiles_n, splits;
    double us;  // the estimate
    size_t part_bytes(int m, int n) const { return splits > 1 ? bt_align((size_t)splits * m * ((n + 3) / 4 * 4) * 4) : 0; }
};
// Tile size and number of workgroups that share a tile's k: the pair whose estimate is lowest. Measured, in us for one
// tile and 128 bytes of k: alone on its CU, and per workgroup where a CU has several (256 x 256: never more than one).
//            256        128           64            32
//   16-bit   1.75       0.58, 0.48    0.22, 0.18    (waits for memory, not for the matrix cores: nothing to gain)
//   f32                 2.30, 2.10    0.52, 0.50    0.20, 0.17    (128: never better than four of 64, so not built)
// and for sharing k a launch and the partial sums' way through memory (7 TB/s). What this decides, measured both ways, in us
// with all launches: bf16 dW of 16384 x 2048 -> 2048 113 as 256 / 4, 123 as 128 / 2, 151 as 128 / 1; bf16 forward 2048 x 2048 ->
// 2048 21.7 as 128 / 1, 27.3 as 64 / 1, 1024 x 1024 -> 1024 7.4 as 64 / 1, 12.9 as 128 / 4; f32 forward 512 x 512 -> 512 7.1 as
// 32 / 1, 10.9 as 64 / 2, 4096 x 1024 -> 1024 66 as 64 / 1, 78 as 32 / 1.
constexpr double LAUNCH_US = 4.0;
Shape shape_of(int m, int n, int k, int passes, size_t es, bool lift = false, int only = 0) {
    struct Cost {
        int b;
        double alone, busy;
    };
    static const Cost of_2[] = {{256, 1.75, 1.75}, {128, 0.58, 0.48}, {64, 0.22, 0.18}};
    static const Cost of_4[] = {{64, 0.52, 0.50}, {32, 0.20, 0.17}};
    const long long ktiles = (long long)bt_div_up(k, (int)(128 / es)) * passes;
    Shape best = {};
    for (int i = 0; i < (es == 2 ? 3 : 2); i++) {
        const Cost &t = es == 2 ? of_2[i] : of_4[i];
        if (only && t.b != only) continue;
        const long long count = (long long)bt_div_up(m, t.b) * bt_div_up(n, t.b);
        for (int splits = lift ? 2 : 1; splits <= 32; splits += lift || splits >= 4 ? 2 : 1) {
            if (splits > 1 && !lift && ktiles / splits < 2) break;
            const double each = (double)((ktiles + splits - 1) / splits), per_cu = (double)((count * splits + 255) / 256);
            double us = each * (per_cu * t.busy > t.alone ? per_cu * t.busy : t.alone);
            if (splits > 1) us += LAUNCH_US + splits * (double)m * n * 8.0 / 7.0e6;
            if (best.bm == 0 || us < best.us)
                best = Shape{t.b, bt_div_up(m, t.b), bt_div_up(n, t.b), splits, us};
        }
    }
    return best;
}

// Buffers for direct loads. A third one keeps two tiles on their way at any time, which a workgroup that is alone on its CU
// needs: the products of a 64 x 64 tile take a third of a load's latency. Where more workgroups share a CU they hide it from
// each other, and need the LDS. (bf16 dW of 2048 x 1024 -> 1024, 256 workgroups: 21.5 us with two, 15.7 with three; f32 4096 x
// 1024 -> 1024, 1024 workgroups: 67 with two, 80 with three.)
constexpr int three_up_to(int b) { return b == 256 ? 0 : b == 128 ? 256 : 512; }  // workgroups up to which there are three

// the tile sizes shape_of chooses from, with or without direct loads
template <typename T, int BM, int BN, int WM, int WN, bool AK, bool BKC, int OUT, int BUFS>
int direct_launch(hipStream_t st, const Product &P, dim3 grid) {
    const size_t lds = BUFS * Mm<T, BM, BN, WM, WN, AK, BKC, OUT>::BYTES;
    const auto kernel = affine_mm_direct<T, BM, BN, WM, WN, AK, BKC, OUT, BUFS>;
    if (int rc = bt_set_max_lds(reinterpret_cast<const void *>(kernel), lds)) return rc;
    BT_LAUNCH(BTK_AFFINE, st, (affine_mm_direct<T, BM, BN, WM, WN, AK, BKC, OUT, BUFS>), grid, dim3(64 * WM * WN), lds, P);
    BT_LAUNCH_CHECK();
    return BT_OK;
}
template <typename T, int BM, int BN, int WM, int WN, bool AK, bool BKC, int OUT>
int mm_launch(hipStream_t st, const Product &P, bool direct) {
    const dim3 grid = folded((long long)P.wgs + P.bias.blocks);
    if constexpr (BM <= 128) {
        if (!direct) {
            const size_t lds = 2 * Mm<T, BM, BN, WM, WN, AK, BKC, OUT>::BYTES;
            const auto kernel = affine_mm_any<T, BM, BN, WM, WN, AK, BKC, OUT>;
            if (int rc = bt_set_max_lds(reinterpret_cast<const void *>(kernel), lds)) return rc;
            BT_LAUNCH(BTK_AFFINE, st, (affine_mm_any<T, BM, BN, WM, WN, AK, BKC, OUT>), grid, dim3(64 * WM * WN), lds, P);
            BT_LAUNCH_CHECK();
            return BT_OK;
        }
        if (P.wgs <= three_up_to(BM)) return direct_launch<T, BM, BN, WM, WN, AK, BKC, OUT, 3>(st, P, grid);
    }
    return direct_launch<T, BM, BN, WM, WN, AK, BKC, OUT, 2>(st, P, grid);
}
template <typename T, bool AK, bool BKC, int OUT>
int tile_launch(hipStream_t st, const Product &P, const Shape &s, bool direct) {
    if constexpr (sizeof(T) == 2) {
        if (s.bm == 256) return mm_launch<T, 256, 256, 2, 4, AK, BKC, OUT>(st, P, direct);
        if (s.bm == 128) return mm_launch<T, 128, 128, 2, 2, AK, BKC, OUT>(st, P, direct);
    } else {
        if (s.bm == 32) return mm_launch<T, 32, 32, 2, 2, AK, BKC, OUT>(st, P, direct);
    }
    return mm_launch<T, 64, 64, 2, 2, AK, BKC, OUT>(st, P, direct);
}
void set_shape(Product &P, const Shape &s) {
    // (of at most 2^36 outputs and 2^30 rows there are at most 2^26 tiles of any size; k is shared only where they are few)
    P.tiles_m = s.tiles_m, P.tiles_n = s.tiles_n, P.splits = s.splits, P.wgs = s.tiles_m * s.tiles_n * s.splits;
    P.part_ld = (P.n + 3) / 4 * 4;
}
template <typename T, int OUT>
int join_launch(hipStream_t st, const Product &P) {
    BT_LAUNCH(BTK_AFFINE, st, (affine_join<T, OUT>), folded(bt_div_up(P.part_ld / 4 * P.m, 256)), dim3(256), 0, P);
    BT_LAUNCH_CHECK();
    return BT_OK;
}
// (256 x 256 tiles have no registers to spare for operands on their way into LDS)
Shape fitted(Shape s, int m, int n, bool direct) {
    if (s.bm == 256 && !direct) s.bm = 128, s.tiles_m = bt_div_up(m, 128), s.tiles_n = bt_div_up(n, 128);
    return s;
}
template <typename T, bool AK, bool BKC, int OUT>
int product_launch(hipStream_t st, Product &P, const Shape &shape) {
    const bool dma = P.a.aligned && P.b.aligned;
    const Shape s = fitted(shape, P.m, P.n, dma);
    set_shape(P, s);
    if (s.splits == 1) return tile_launch<T, AK, BKC, OUT>(st, P, s, dma);
    if (int rc = tile_launch<T, AK, BKC, OUT_PART>(st, P, s, dma)) return rc;
    return join_launch<T, OUT>(st, P);
}
// both products of a backward pass, each with its sums in a place of its own
template <typename T, int B, int OUT_W, int OUT_X>
int both_launch(hipStream_t st, const Product &W, const Product &X) {
    const long long all = (long long)W.wgs + W.bias.blocks + X.wgs;
    typedef Mm<T, B, B, 2, 2, false, false, OUT_W> MW;
    typedef Mm<T, B, B, 2, 2, true, true, OUT_X> MX;
    static_assert(MW::BYTES == MX::BYTES && 3 * MW::BYTES <= 65536, "tiles of one size, within what needs no attribute");
    const dim3 grid = folded(all), block(256);
    if (all <= three_up_to(B))
        BT_LAUNCH(BTK_AFFINE, st, (affine_mm_both<T, B, OUT_W, OUT_X, 3>), grid, block, 3 * MW::BYTES, W, X);
    else
        BT_LAUNCH(BTK_AFFINE, st, (affine_mm_both<T, B, OUT_W, OUT_X, 2>), grid, block, 2 * MW::BYTES, W, X);
    BT_LAUNCH_CHECK();
    return BT_OK;
}
template <typename T, int B>
int both_of(hipStream_t st, const Product &W, const Product &X) {
    const bool pw = W.splits > 1, px = X.splits > 1;
    if (int rc = pw ? (px ? both_launch<T, B, OUT_PART, OUT_PART>(st, W, X) : both_launch<T, B, OUT_PART, OUT_TYPE>(st, W, X))
                    : (px ? both_launch<T, B, OUT_F32, OUT_PART>(st, W, X) : both_launch<T, B, OUT_F32, OUT_TYPE>(st, W, X)))
        return rc;
    if (pw)
        if (int rc = join_launch<T, OUT_F32>(st, W)) return rc;
    return px ? join_launch<T, OUT_TYPE>(st, X) : BT_OK;
}
template <typename T>
int both_products(hipStream_t st, Product &W, const Shape &sw, Product &X, const Shape &sx) {
    set_shape(W, sw), set_shape(X, sx);
    if constexpr (sizeof(T) == 4)
        if (sw.bm == 32) return both_of<T, 32>(st, W, X);
    return both_of<T, 64>(st, W, X);
}

long long padded(int n, size_t es) { return (n + (128 / es) - 1) / (128 / es) * (128 / es); }  // rows on 128 bytes
int whole_chunks(int n, size_t es) { return (int)((n + (16 / es) - 1) / (16 / es) * (16 / es)); }
// direct loads need rows on 16 bytes, and reach those of one tile through 32-bit offsets
bool direct_ld(long long ld, size_t es) { return ld * es % 16 == 0 && ld < (1 << 21); }
Operand matrix(const void *p, long long ld, int rows, int len, size_t es) {
    return Operand{p, p, p, ld, rows, len, (reinterpret_cast<uintptr_t>(p) & 15) == 0 && direct_ld(ld, es)};
}
// one of the workspace's: the zeros behind a row are part of it
Operand own_matrix(const void *p, int rows, int len, size_t es) { return matrix(p, padded(len, es), rows, whole_chunks(len, es), es); }

// Outputs whose rows start on 16 bytes are stored past the caches, where they would only push out the operands (16384 x 2048 ->
// 4096 bf16 218 us, 229 through them; backward of 2048 -> 2048 263 and 271). Pieces of other rows share lines, which the caches put
// together (1537 x 1027 -> 1881 f16, rows 3 apart: 21.6 us through them, 22.7 past them).
bool past_caches(const void *out, const void *saved, long long ld, size_t es) {
    return ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(saved)) & 15) == 0 && ld * es % 16 == 0;
}

// Matrices that are copied into the workspace first: those whose rows do not start on 16 bytes (read through registers
// instead, both operands of 4096 x 1024 -> 1024 make the forward product 38 us of bf16 and 102 of f32; the copies take 8 and
// 13 us and leave 18 and 73), and f32 weights of a 16-bit layer. One whose first element alone is off is read through registers.
size_t copy_bytes(bool copy, int rows, int len, size_t es) { return copy ? bt_align((size_t)rows * padded(len, es) * es) : 0; }
bool copy_w(const bt_affine_desc *d) { return d->w_type != d->type || !direct_ld(d->w_ld, type_size(d->type)); }
bool copy_x(const bt_affine_desc *d) { return !direct_ld(d->x_ld, type_size(d->type)); }

template <typename T>
Copy<T> copy_of(const void *from, long long ld, bool f32, void *to, int rows, int len) {
    Copy<T> c{from, (T *)to, ld, padded(len, sizeof(T)), rows, len, f32, 0};
    c.blocks = bt_div_up((long long)whole_chunks(len, sizeof(T)) / Elem<T>::V * rows, 256);
    return c;
}
// w / x as the products take them; adds the copy, if there is one, to `p`
template <typename T>
Operand weights(const bt_affine_desc *d, const void *w, void *ws, Prepare<T> &p) {
    if (!copy_w(d)) return matrix(w, d->w_ld, d->in, d->out, sizeof(T));
    p.w = copy_of<T>(w, d->w_ld, d->w_type != d->type, ws, d->in, d->out);
    return own_matrix(ws, d->in, d->out, sizeof(T));
}
template <typename T>
Operand inputs(const bt_affine_desc *d, const void *x, void *ws, Prepare<T> &p) {
    if (!copy_x(d)) return matrix(x, d->x_ld, d->batch, d->in, sizeof(T));
    p.x = copy_of<T>(x, d->x_ld, false, ws, d->batch, d->in);
    return own_matrix(ws, d->batch, d->in, sizeof(T));
}
template <typename T>
int prepare_launch(hipStream_t st, const Prepare<T> &p, int np) {
    const long long blocks = (long long)p.w.blocks + p.x.blocks + p.gz.blocks;
    if (blocks == 0) return BT_OK;
    const dim3 grid = folded(blocks), block(256);
    if (p.gz.blocks == 0)
        BT_LAUNCH(BTK_AFFINE, st, (affine_prepare<T, 0>), grid, block, 0, p);
    else if (np == 1)
        BT_LAUNCH(BTK_AFFINE, st, (affine_prepare<T, 1>), grid, block, 0, p);
    else if constexpr (sizeof(T) == 2) {
        if (np == 2)
            BT_LAUNCH(BTK_AFFINE, st, (affine_prepare<T, 2>), grid, block, 0, p);
        else if constexpr (std::is_same<T, __bf16>::value)
            BT_LAUNCH(BTK_AFFINE, st, (affine_prepare<T, 3>), grid, block, 0, p);
    }
    BT_LAUNCH_CHECK();
    return BT_OK;
}

// Rows that affine_few takes: 8, but 4 where both weights and rows have 16 bits (2048 -> 4096 bf16: 4 rows 9.0 us against 10.4 on
// the matrix cores, 8 rows 13.3 against 9.9; f32: 8 rows 11.1 against 12.6; f32 weights that would have to be rounded into a
// copy first: 8 rows 16 against 20)
int few_rows(const bt_affine_desc *d) { return d->w_type == BT_TYPE_F32 ? 8 : 4; }
template <typename T, typename TW>
int few_launch(hipStream_t st, const bt_affine_desc *d, const void *w, const void *x, const Epilogue &e) {
    const dim3 grid = folded(bt_div_up(d->out, 4 * Elem<T>::V));
#define FEW_CASE(R)                                                                                                         \
    BT_LAUNCH(BTK_AFFINE, st, (affine_few<T, TW, R>), grid, dim3(few_threads(R)), 0, (const TW *)w, (long long)d->w_ld,     \
              (const T *)x, (long long)d->x_ld, d->batch, d->in, d->out, e)
    if (d->batch == 1)
        FEW_CASE(1);
    else if (d->batch == 2)
        FEW_CASE(2);
    else if (d->batch <= 4)
        FEW_CASE(4);
    else if constexpr (sizeof(TW) == 4)
        FEW_CASE(8);
#undef FEW_CASE
    BT_LAUNCH_CHECK();
    return BT_OK;
}

struct ForwardPlan {
    Shape s;
    size_t w_bytes, x_bytes, total;
};
ForwardPlan forward_plan(const bt_affine_desc *d) {
    ForwardPlan p = {};
    if (d->batch <= few_rows(d)) return p;
    const size_t es = type_size(d->type);
    p.s = shape_of(d->batch, d->out, d->in, 1, es);
    p.w_bytes = copy_bytes(copy_w(d), d->in, d->out, es), p.x_bytes = copy_bytes(copy_x(d), d->batch, d->in, es);
    p.total = p.w_bytes + p.x_bytes + p.s.part_bytes(d->batch, d->out);
    return p;
}
template <typename T>
int forward(hipStream_t st, const bt_affine_desc *d, const void *w, const float *bias, const void *x, const void *residual, void *y,
            void *saved, char *ws) {
    const Epilogue e{bias, residual, y, saved, d->y_ld, d->act, 1.0f, past_caches(y, saved, d->y_ld, sizeof(T))};
    if (d->batch <= few_rows(d))
        return d->w_type == d->type ? few_launch<T, T>(st, d, w, x, e) : few_launch<T, float>(st, d, w, x, e);
    const ForwardPlan p = forward_plan(d);
    Product P = {};
    Prepare<T> prep = {};
    P.b = weights<T>(d, w, ws, prep);
    P.a = inputs<T>(d, x, ws + p.w_bytes, prep);
    if (int rc = prepare_launch<T>(st, prep, 0)) return rc;
    P.m = d->batch, P.n = d->out, P.k = d->in, P.passes = 1;
    P.part = (float *)(ws + p.w_bytes + p.x_bytes);
    P.e = e;
    return product_launch<T, true, false, OUT_LAYER>(st, P, p.s);
}

struct BackwardPlan {
    bool gz;             // gz is kept, with rows on 16 bytes (else grad_y is gz)
    int np_dw, np_dx;    // summands it is kept as for dW (whose outputs are f32), and how many of them grad_x takes
    float alpha;
    int lift;
    int range, ranges, col_blocks;
    Shape dw, dx;
    bool both;  // dW and grad_x in one launch; grad_x's partial sums then lie behind dW's
    size_t w_bytes, x_bytes, gz_bytes, sum_bytes, part_dx, part_bytes, total;
};
BackwardPlan backward_plan(const bt_affine_desc *d) {
    BackwardPlan p;
    const size_t es = type_size(d->type);
    const bool root = d->act == BT_ACT_SCRELU || d->act == BT_ACT_SQRRELU;
    p.gz = d->act != BT_ACT_IDENTITY || !direct_ld(d->y_ld, es);
    p.np_dw = !root || es == 4 ? 1 : d->type == BT_TYPE_BF16 ? 3 : 2;
    p.np_dx = p.np_dw > 2 ? 2 : p.np_dw;
    p.alpha = root ? 2.0f : 1.0f;
    p.lift = d->type == BT_TYPE_F16 && root;
    // row ranges of affine_prepare: as many workgroups as fill the chip, at least the rows that one takes at once, and no
    // more ranges than bias_sum adds up in a few us (8192 x 288 -> 6 f16: 1024 ranges 66 us in all, 256 50 us)
    p.col_blocks = bt_div_up(d->out, GZ_COLS * (int)(16 / es));
    const int fill = bt_div_up((long long)d->batch * p.col_blocks, 1024 * GZ_ROWS), few = bt_div_up(d->batch, 256 * GZ_ROWS);
    p.range = GZ_ROWS * (fill > few ? fill : few);
    p.ranges = bt_div_up(d->batch, p.range);
    p.dw = shape_of(d->in, d->out, d->batch, p.np_dw, es, p.lift);
    p.dx = shape_of(d->batch, d->in, d->out, p.np_dx, es, p.lift);
    // One launch does both where their tiles are of one size, at most 64 x 64; the size that suits each best, or that. (bf16
    // 4096 x 1024 -> 1024 37 us in one, 40 in two; 2048 x 2048 -> 2048 57 and 50; f32 200 x 512 -> 333 with 64 x 64 tiles 14 and 23.)
    double us = p.dw.us + p.dx.us + LAUNCH_US;
    p.both = false;
    for (int b = 64; b >= (es == 4 ? 32 : 64); b /= 2) {
        const Shape w = shape_of(d->in, d->out, d->batch, p.np_dw, es, p.lift, b);
        const Shape x = shape_of(d->batch, d->in, d->out, p.np_dx, es, p.lift, b);
        if (w.us + x.us <= us) p.dw = w, p.dx = x, p.both = true, us = w.us + x.us;
    }
    p.w_bytes = copy_bytes(copy_w(d), d->in, d->out, es), p.x_bytes = copy_bytes(copy_x(d), d->batch, d->in, es);
    p.gz_bytes = p.gz ? bt_align((size_t)d->batch * padded(d->out, es) * es) : 0;
    p.sum_bytes = bt_align((size_t)p.ranges * d->out * 4);
    const size_t a = p.dw.part_bytes(d->in, d->out), b = p.dx.part_bytes(d->batch, d->in);
    p.part_dx = p.both ? a : 0;
    p.part_bytes = p.both ? a + b : a > b ? a : b;
    p.total = p.w_bytes + p.x_bytes + p.gz_bytes * p.np_dw + p.sum_bytes + p.part_bytes;
    return p;
}

template <typename T>
int backward(hipStream_t st, const bt_affine_desc *d, const void *w, const void *x, const void *out, const void *gy, float *dw,
             float *dbias, void *gx, char *ws) {
    const BackwardPlan p = backward_plan(d);
    char *own_w = ws, *own_x = own_w + p.w_bytes, *kept = own_x + p.x_bytes, *sums = kept + p.gz_bytes * p.np_dw, *part = sums + p.sum_bytes;
    const bool keep = p.gz && (dw || gx);
    const int np = dw ? p.np_dw : p.np_dx;
    Prepare<T> prep = {};
    const Operand ow = gx ? weights<T>(d, w, own_w, prep) : Operand{}, ox = dw ? inputs<T>(d, x, own_x, prep) : Operand{};
    if (keep || dbias) {
        Gz<T> &g = prep.gz;
        g.gy = (const T *)gy, g.out = d->act != BT_ACT_IDENTITY ? (const T *)out : nullptr;
        for (int i = 0; i < np && keep; i++) g.p[i] = (T *)(kept + i * p.gz_bytes);
        g.sums = dbias ? (float *)sums : nullptr;
        g.ld = d->y_ld, g.gz_ld = padded(d->out, sizeof(T));
        g.batch = d->batch, g.n = d->out, g.act = d->act, g.range = p.range, g.col_blocks = p.col_blocks;
        g.blocks = p.col_blocks * p.ranges;
    }
    if (int rc = prepare_launch<T>(st, prep, keep ? np : 1)) return rc;
    BiasSum bias = {};
    if (dbias) bias = BiasSum{(const float *)sums, dbias, p.ranges, d->out, bt_div_up(d->out, BIAS_COLS), p.alpha};
    if (dbias && !dw && !gx) {
        BT_LAUNCH(BTK_AFFINE, st, affine_dbias, folded(bias.blocks), dim3(256), 0, bias);
        BT_LAUNCH_CHECK();
    }
    const auto gz_operand = [&](int n) {  // its n largest summands, the smallest of them first
        if (!p.gz) return matrix(gy, d->y_ld, d->batch, d->out, sizeof(T));
        Operand o = own_matrix(kept, d->batch, d->out, sizeof(T));
        o.p0 = kept + (n - 1) * p.gz_bytes, o.p1 = n > 1 ? kept + (n - 2) * p.gz_bytes : kept, o.p2 = kept;
        return o;
    };
    Product W = {}, X = {};
    if (dw) {
        W.a = ox, W.b = gz_operand(p.np_dw);
        W.m = d->in, W.n = d->out, W.k = d->batch, W.passes = p.np_dw, W.lift = p.lift;
        W.part = (float *)part;
        W.e.out = dw, W.e.ld = d->w_ld, W.e.alpha = p.alpha, W.e.past = past_caches(dw, nullptr, d->w_ld, sizeof(float));
    }
    if (gx) {
        X.a = gz_operand(p.np_dx), X.b = ow;
        X.m = d->batch, X.n = d->in, X.k = d->out, X.passes = p.np_dx, X.lift = p.lift;
        X.part = (float *)(part + p.part_dx);
        X.e.out = gx, X.e.ld = d->x_ld, X.e.alpha = p.alpha, X.e.past = past_caches(gx, nullptr, d->x_ld, sizeof(T));
    }
    (dw ? W : X).bias = bias;
    if (dw && gx && p.both && W.a.aligned && W.b.aligned && X.a.aligned && X.b.aligned)
        return both_products<T>(st, W, p.dw, X, p.dx);
    if (dw)
        if (int rc = product_launch<T, false, false, OUT_F32>(st, W, p.dw)) return rc;
    if (gx) return product_launch<T, true, true, OUT_TYPE>(st, X, p.dx);
    return BT_OK;
}

}  // namespace

extern "C" {

size_t bt_affine_forward_workspace_bytes(const bt_affine_desc *d) {
    if (validate(d, "bt_affine_forward_workspace_bytes")) return 0;
    return forward_plan(d).total;
}

int bt_affine_forward(void *stream, const bt_affine_desc *d, const void *w, const float *bias, const void *x,
                      const void *residual, void *y, void *saved, void *workspace, size_t workspace_bytes) {
    if (int rc = validate(d, "bt_affine_forward")) return rc;
    BT_REQUIRE(w && x && y, "bt_affine_forward: null pointer");
    const size_t es = type_size(d->type), need = bt_affine_forward_workspace_bytes(d);
    BT_REQUIRE(workspace_bytes >= need && (workspace || !need), "bt_affine_forward: workspace too small (%zu < %zu)",
               workspace_bytes, need);
    BT_REQUIRE(!need || elem_aligned(workspace, 16), "bt_affine_forward: workspace is not aligned to 16 bytes");
    BT_REQUIRE(elem_aligned(x, es) && elem_aligned(y, es) && elem_aligned(residual, es) && elem_aligned(saved, es) &&
                   elem_aligned(w, type_size(d->w_type)) && elem_aligned(bias, 4),
               "bt_affine_forward: a buffer is not aligned to its element type");
    BT_REQUIRE(saved != y && (!saved || saved != residual) && x != y && x != saved,
               "bt_affine_forward: outputs overlap each other or the input");
    hipStream_t s = bt_stream(stream);
    char *ws = static_cast<char *>(workspace);
    if (d->type == BT_TYPE_F32) return forward<float>(s, d, w, bias, x, residual, y, saved, ws);
    if (d->type == BT_TYPE_BF16) return forward<__bf16>(s, d, w, bias, x, residual, y, saved, ws);
    return forward<_Float16>(s, d, w, bias, x, residual, y, saved, ws);
}

size_t bt_affine_backward_workspace_bytes(const bt_affine_desc *d) {
    if (validate(d, "bt_affine_backward_workspace_bytes")) return 0;
    return backward_plan(d).total;
}

int bt_affine_backward(void *stream, const bt_affine_desc *d, const void *w, const void *x, const void *out,
                       const void *grad_y, float *dw, float *dbias, void *grad_x, void *workspace, size_t workspace_bytes) {
    if (int rc = validate(d, "bt_affine_backward")) return rc;
    BT_REQUIRE(grad_y && (dw || dbias || grad_x), "bt_affine_backward: null pointer");
    BT_REQUIRE((x || !dw) && (w || !grad_x) && (out || d->act == BT_ACT_IDENTITY), "bt_affine_backward: null pointer");
    BT_REQUIRE(!(d->type == BT_TYPE_F16 && d->act == BT_ACT_SQRRELU),
               "bt_affine_backward: the squared ReLU's gradient can leave the range of f16");
    const size_t es = type_size(d->type), need = bt_affine_backward_workspace_bytes(d);
    BT_REQUIRE(workspace && workspace_bytes >= need, "bt_affine_backward: workspace too small (%zu < %zu)", workspace_bytes, need);
    BT_REQUIRE(elem_aligned(workspace, 16), "bt_affine_backward: workspace is not aligned to 16 bytes");
    BT_REQUIRE(elem_aligned(x, es) && elem_aligned(out, es) && elem_aligned(grad_y, es) && elem_aligned(grad_x, es) &&
                   elem_aligned(w, type_size(d->w_type)) && elem_aligned(dw, 4) && elem_aligned(dbias, 4),
               "bt_affine_backward: a buffer is not aligned to its element type");
    BT_REQUIRE((!grad_x || (grad_x != x && grad_x != grad_y && grad_x != out && grad_x != w)) &&
                   (!dw || (const void *)dw != w),
               "bt_affine_backward: an output overlaps an input");
    hipStream_t s = bt_stream(stream);
    char *ws = static_cast<char *>(workspace);
    if (d->type == BT_TYPE_F32) return backward<float>(s, d, w, x, out, grad_y, dw, dbias, grad_x, ws);
    if (d->type == BT_TYPE_BF16) return backward<__bf16>(s, d, w, x, out, grad_y, dw, dbias, grad_x, ws);
    return backward<_Float16>(s, d, w, x, out, grad_y, dw, dbias, grad_x, ws);
}

// Tests ask which variant a call takes: the tile, the workgroups that share one, and whether both gradients take one launch
// (product 0: forward, 1: dw, 2: grad_x; direct: whether the operands' first elements are on 16 bytes). Tile 0: affine_few.
int bt_internal_affine_variant(const bt_affine_desc *d, int product, int direct, int *tile, int *splits, int *both) {
    if (int rc = validate(d, "bt_internal_affine_variant")) return rc;
    BT_REQUIRE(product >= 0 && product <= 2 && tile && splits && both, "bt_internal_affine_variant: no such product");
    Shape s = {};
    *both = 0;
    if (product == 0) {
        s = fitted(forward_plan(d).s, d->batch, d->out, direct);
    } else {
        const BackwardPlan p = backward_plan(d);
        *both = p.both && direct;
        s = product == 1 ? fitted(p.dw, d->in, d->out, direct) : fitted(p.dx, d->batch, d->in, direct);
    }
    *tile = s.bm, *splits = s.splits;
    return BT_OK;
}

}  // extern "C"
