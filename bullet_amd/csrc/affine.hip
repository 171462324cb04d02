// Wide affine layers: y = act(x W^T + bias) + residual and its gradients as matrix products on the MFMA units.
//
// One kernel does the three products, D[m][n] = sum_k A[m][k] B[n][k]:
//   forward   m = position, n = output, k = input     A = x (k contiguous)    B = W (n contiguous)
//   grad_x    m = position, n = input,  k = output    A = gz (k contiguous)   B = W (k contiguous)
//   dW        m = input,    n = output, k = position  A = x (m contiguous)    B = gz (n contiguous)
// A k-contiguous operand is staged in LDS as rows of 128 bytes of k and read 16 bytes a lane; one that is contiguous the
// other way is staged as it lies and read transposed (ds_read_b64_tr_b16 for 16-bit types, single words for f32), so no
// operand is ever transposed in memory. f32 goes through v_mfma_f32_16x16x4_f32: exact products, 32-bit sums.
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
    typedef T quad __attribute__((ext_vector_type(4)));
};

// acc += a b^T over the k of one fragment: lane l holds row l % 16 and, of 16-bit types, k = 8 (l / 16) .. + 7 of 32 (one
// MFMA), of f32 k = 4 (l / 16) .. + 3 of 16 (four of them, each taking one k from every 16 lanes)
__device__ __forceinline__ void mma(v4f &acc, const Elem<__bf16>::frag &a, const Elem<__bf16>::frag &b) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(v4f &acc, const Elem<_Float16>::frag &a, const Elem<_Float16>::frag &b) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(v4f &acc, const Elem<float>::frag &a, const Elem<float>::frag &b) {
#pragma unroll
    for (int j = 0; j < 4; j++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], acc, 0, 0, 0);
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
    // fragment `f` (16 of SPAN) at k-step s
    static __device__ __forceinline__ typename Elem<T>::frag read(const char *lds, int f, int s, int lane) {
        typedef typename Elem<T>::frag frag;
        const int g = lane >> 4, i = lane & 15;
        if constexpr (KC) {
            const int row = f * 16 + i;
            return *(const frag *)(lds + row * 128 + swizzle(row, s * 4 + g) * 16);
        } else if constexpr (sizeof(T) == 4) {
            frag r;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int row = s * 16 + g * 4 + j, c = f * 4 + (i >> 2);
                r[j] = *(const float *)(lds + (row * CPR + swizzle(row, c)) * 16 + (i & 3) * 4);
            }
            return r;
        } else {
            typedef short s4 __attribute__((ext_vector_type(4)));
            s4 h[2];
#pragma unroll
            for (int q = 0; q < 2; q++) {
                // 16 lanes give the addresses of 4 rows of 16 elements and get 4 rows of one column each
                const int row = s * 32 + g * 8 + q * 4 + (i >> 2), c = f * 2 + ((i >> 1) & 1);
                const char *p = lds + (row * CPR + swizzle(row, c)) * 16 + (i & 1) * 8;
                h[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)p);
            }
            return __builtin_bit_cast(frag, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// An operand in memory: `rows` rows of `len` contiguous elements, `ld` apart.
struct Operand {
    const void *p[2];  // two summands of one product (the pair a 16-bit gradient may be kept in), or the same twice
    long long ld;
    int rows, len;
    int aligned;  // every chunk of every row starts on 16 bytes
};

// chunk (row, element e) of the matrix, zeros outside it
template <typename T>
__device__ __forceinline__ v4u load_chunk(const T *base, const Operand &o, int row, long long e) {
    constexpr int V = Elem<T>::V;
    v4u r = {0, 0, 0, 0};
    if (row >= o.rows || e >= o.len) return r;
    const T *p = base + (size_t)row * o.ld + e;
    if (o.len - e >= V) {
        __builtin_memcpy(&r, p, 16);
    } else {
        typename Elem<T>::frag t = {};
#pragma unroll
        for (int j = 0; j < V; j++)
            if (j < o.len - e) t[j] = p[j];
        r = __builtin_bit_cast(v4u, t);
    }
    return r;
}

enum { OUT_LAYER = 0, OUT_TYPE = 1, OUT_F32 = 2, OUT_PART = 3 };
struct Epilogue {
    const float *bias;
    const void *residual;
    void *out, *saved;
    long long ld;
    int act;
    float alpha;
};

template <typename T>
__device__ __forceinline__ void store4(T *p, v4f v, int n) {  // the first n of 4
    typedef T quad __attribute__((ext_vector_type(4)));
    quad q;
#pragma unroll
    for (int j = 0; j < 4; j++) q[j] = (T)v[j];
    if (n >= 4) {
        __builtin_memcpy(p, &q, sizeof(q));
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (j < n) p[j] = q[j];
    }
}
// what becomes of 4 sums of one row, columns c .. c + 3 (n of them inside the matrix)
template <typename T, int OUT>
__device__ __forceinline__ void finish4(const Epilogue &e, int row, int c, int n, v4f v) {
    const size_t at = (size_t)row * e.ld + c;
    if constexpr (OUT == OUT_F32) {
        store4<float>((float *)e.out + at, v * e.alpha, n);
    } else if constexpr (OUT == OUT_TYPE) {
        store4<T>((T *)e.out + at, v * e.alpha, n);
    } else {
        if (e.bias) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (j < n) v[j] += e.bias[c + j];
        }
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = bt_act_fwd(e.act, v[j]);
        if (e.saved) store4<T>((T *)e.saved + at, v, n);
        if (e.residual) {
            const T *r = (const T *)e.residual + at;
            if (n >= 4) {
                typename Elem<T>::quad q;
                __builtin_memcpy(&q, r, sizeof(q));
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] += (float)q[j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (j < n) v[j] += (float)r[j];
            }
        }
        store4<T>((T *)e.out + at, v, n);
    }
}

struct Product {
    Operand a, b;
    int m, n, k;
    int passes;          // 1, or 2: both summands of the operands, one after the other
    int tiles_m, tiles_n;
    int splits;          // workgroups that share one tile's k, each leaving its sums in `part`
    float *part;         // [splits][m][part_ld]
    long long part_ld;
    Epilogue e;
};

// BM x BN tile by 4 waves of BM/2 x BN/2. Double-buffered LDS: the next tile is on its way while this one is multiplied.
template <typename T, int BM, int BN, bool AK, bool BKC, int OUT>
__global__ __launch_bounds__(256) void affine_mm(Product P) {
    typedef Tile<T, AK, BM> TA;
    typedef Tile<T, BKC, BN> TB;
    constexpr int BK = Elem<T>::BK, V = Elem<T>::V;
    constexpr int FM = BM / 32, FN = BN / 32;
    constexpr int NA = TA::SLOTS / 256, NB = TB::SLOTS / 256;
    __shared__ __align__(16) char lds[2][TA::BYTES + TB::BYTES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave >> 1, wn = wave & 1;
    const int tiles = P.tiles_m * P.tiles_n;
    const int split = blockIdx.x / tiles;
    int t = blockIdx.x % tiles;
    const int tm = t / P.tiles_n, tn = t % P.tiles_n;
    const int m0 = tm * BM, n0 = tn * BN;
    const int ktiles = (P.k + BK - 1) / BK, all = ktiles * P.passes;
    const int t0 = (int)((long long)all * split / P.splits), t1 = (int)((long long)all * (split + 1) / P.splits);

    v4f acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
        for (int j = 0; j < FM; j++) acc[i][j] = v4f{0, 0, 0, 0};

    v4u ra[NA], rb[NB];
    auto load = [&](int kt) {
        const int pass = kt >= ktiles, k0 = (kt - pass * ktiles) * BK;
#pragma unroll
        for (int q = 0; q < NA; q++) {
            const int s = q * 256 + tid, row = s / TA::CPR, c = TA::swizzle(row, s % TA::CPR);
            ra[q] = load_chunk<T>((const T *)P.a.p[pass], P.a, (AK ? m0 : k0) + row, (long long)(AK ? k0 : m0) + c * V);
        }
#pragma unroll
        for (int q = 0; q < NB; q++) {
            const int s = q * 256 + tid, row = s / TB::CPR, c = TB::swizzle(row, s % TB::CPR);
            rb[q] = load_chunk<T>((const T *)P.b.p[pass], P.b, (BKC ? n0 : k0) + row, (long long)(BKC ? k0 : n0) + c * V);
        }
    };
    if (t0 < t1) load(t0);
    for (int kt = t0; kt < t1; kt++) {
        char *buf = lds[(kt - t0) & 1];
#pragma unroll
        for (int q = 0; q < NA; q++) *(v4u *)(buf + (q * 256 + tid) * 16) = ra[q];
#pragma unroll
        for (int q = 0; q < NB; q++) *(v4u *)(buf + TA::BYTES + (q * 256 + tid) * 16) = rb[q];
        __syncthreads();  // (the other buffer's readers passed the barrier of this iteration, too, before it is written again)
        if (kt + 1 < t1) load(kt + 1);
#pragma unroll
        for (int s = 0; s < 2; s++) {
            typename Elem<T>::frag fa[FM], fb[FN];
#pragma unroll
            for (int j = 0; j < FM; j++) fa[j] = TA::read(buf, wm * FM + j, s, lane);
#pragma unroll
            for (int i = 0; i < FN; i++) fb[i] = TB::read(buf + TA::BYTES, wn * FN + i, s, lane);
#pragma unroll
            for (int i = 0; i < FN; i++)
#pragma unroll
                for (int j = 0; j < FM; j++) mma(acc[i][j], fb[i], fa[j]);
        }
    }
    // lane l holds, of each 16 x 16 block, row m = l % 16 and columns n = 4 (l / 16) .. + 3
#pragma unroll
    for (int j = 0; j < FM; j++) {
        const int m = m0 + (wm * FM + j) * 16 + (lane & 15);
        if (m >= P.m) continue;
#pragma unroll
        for (int i = 0; i < FN; i++) {
            const int n = n0 + (wn * FN + i) * 16 + (lane >> 4) * 4;
            if (n >= P.n) continue;
            if constexpr (OUT == OUT_PART)
                *(v4f *)(P.part + ((size_t)split * P.m + m) * P.part_ld + n) = acc[i][j];  // (part_ld: a multiple of 4)
            else
                finish4<T, OUT>(P.e, m, n, P.n - n, acc[i][j]);
        }
    }
}

// the splits' sums added in order, then the epilogue
template <typename T, int OUT>
__global__ __launch_bounds__(256) void affine_join(Product P) {
    const long long q = (long long)blockIdx.x * 256 + threadIdx.x, cols = P.part_ld / 4;
    if (q >= cols * P.m) return;
    const int m = (int)(q / cols), n = (int)(q % cols) * 4;
    v4f v = {0, 0, 0, 0};
    for (int s = 0; s < P.splits; s++) v += *(const v4f *)(P.part + ((size_t)s * P.m + m) * P.part_ld + n);
    finish4<T, OUT>(P.e, m, n, P.n - n, v);
}

// f32 weights rounded to the layer's type, rows `to_ld` apart
template <typename T>
__global__ __launch_bounds__(256) void affine_round_w(const float *__restrict__ from, long long from_ld, T *__restrict__ to,
                                                      long long to_ld, int rows, int len) {
    const long long q = (long long)blockIdx.x * 256 + threadIdx.x, cols = (len + 3) / 4;
    if (q >= cols * rows) return;
    const long long row = q / cols;
    const int c = (int)(q % cols) * 4;
    v4f v = {0, 0, 0, 0};
    const float *p = from + row * from_ld + c;
    if (len - c >= 4) {
        __builtin_memcpy(&v, p, 16);
    } else {
        for (int j = 0; j < len - c; j++) v[j] = p[j];
    }
    store4<T>(to + row * to_ld + c, v, len - c);
}

// gz = grad_y act'(out) (half of it where act' carries a factor 2: the products' alpha gives it back, exactly), as one
// number of the layer's type or as the sum of two, and the column sums of gz over this workgroup's rows.
// Thread (c, r) takes column chunk c and every 8th row from r on.
constexpr int GZ_COLS = 32, GZ_ROWS = 8;
template <typename T, bool PAIR>
__global__ __launch_bounds__(256) void affine_gz(const T *__restrict__ gy, const T *__restrict__ out, long long ld, T *__restrict__ hi,
                                                 T *__restrict__ lo, long long gz_ld, float *__restrict__ part, int batch, int n,
                                                 int act, int range) {
    constexpr int V = Elem<T>::V;
    typedef typename Elem<T>::frag frag;
    __shared__ float red[GZ_ROWS][GZ_COLS * V];
    const int c = threadIdx.x % GZ_COLS, r = threadIdx.x / GZ_COLS;
    const long long e = ((long long)blockIdx.x * GZ_COLS + c) * V;
    const long long b0 = (long long)blockIdx.y * range, b1 = b0 + range < batch ? b0 + range : batch;
    const int left = e < n ? (int)(n - e < V ? n - e : V) : 0;
    const float half = act == BT_ACT_SCRELU || act == BT_ACT_SQRRELU ? 0.5f : 1.0f;
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; j++) sum[j] = 0.0f;
    if (left)
        for (long long b = b0 + r; b < b1; b += GZ_ROWS) {
            frag g = {}, o = {}, h, l;
            const T *pg = gy + b * ld + e, *po = out ? out + b * ld + e : nullptr;
            if (left == V) {
                __builtin_memcpy(&g, pg, 16);
                if (out) __builtin_memcpy(&o, po, 16);
            } else {
                for (int j = 0; j < V; j++)
                    if (j < left) {
                        g[j] = pg[j];
                        if (out) o[j] = po[j];
                    }
            }
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float v = out ? (float)g[j] * (bt_act_deriv(act, (float)o[j]) * half) : (float)g[j];
                sum[j] += v;
                h[j] = (T)v;
                if (PAIR) l[j] = (T)(v - (float)h[j]);
            }
            if (hi) __builtin_memcpy(hi + b * gz_ld + e, &h, 16);  // (gz_ld is a multiple of V: a last chunk is whole)
            if (PAIR) __builtin_memcpy(lo + b * gz_ld + e, &l, 16);
        }
    if (!part) return;
#pragma unroll
    for (int j = 0; j < V; j++) red[r][c * V + j] = sum[j];
    __syncthreads();
    for (int i = threadIdx.x; i < GZ_COLS * V; i += 256) {
        const long long col = (long long)blockIdx.x * GZ_COLS * V + i;
        if (col >= n) continue;
        float s = 0.0f;
        for (int q = 0; q < GZ_ROWS; q++) s += red[q][i];
        part[(size_t)blockIdx.y * n + col] = s;
    }
}

// dbias: the row ranges' sums, 16 threads a column, in a fixed order
__global__ __launch_bounds__(1024) void affine_dbias(const float *__restrict__ part, int parts, int n, float alpha,
                                                     float *__restrict__ dbias) {
    __shared__ float red[16][64];
    const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
    const long long col = (long long)blockIdx.x * 64 + c;
    float s = 0.0f;
    if (col < n)
        for (int p = r; p < parts; p += 16) s += part[(size_t)p * n + col];
    red[r][c] = s;
    __syncthreads();
    if (r || col >= n) return;
    for (int q = 1; q < 16; q++) s += red[q][c];
    dbias[col] = s * alpha;
}

// ---- host side
size_t type_size(int type) { return type == BT_TYPE_F32 ? 4 : 2; }
bool chunk_aligned(const void *p, long long ld, size_t es) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * es) % 16 == 0;
}
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
    BT_REQUIRE(d->batch <= (1 << 30) && d->in <= (1 << 30) && d->out <= (1 << 30), "%s: Mismatched sizes! (too large)", fn);
    return BT_OK;
}

struct Shape {
    int bm, bn, tiles_m, tiles_n, splits;
    size_t part_bytes(int m, int n) const { return splits > 1 ? bt_align((size_t)splits * m * ((n + 3) / 4 * 4) * 4) : 0; }
};
// Tile and split: 128 x 128 tiles where they give every CU one; smaller tiles, then several workgroups on one tile's k,
// where they do not.
Shape shape_of(int m, int n, int k, int passes, size_t es) {
    Shape s;
    const auto count = [&](int b) { return (long long)bt_div_up(m, b) * bt_div_up(n, b); };
    s.bm = s.bn = count(128) >= 256 ? 128 : 64;
    s.tiles_m = bt_div_up(m, s.bm), s.tiles_n = bt_div_up(n, s.bn);
    const long long tiles = count(s.bm), ktiles = (long long)bt_div_up(k, (int)(128 / es)) * passes;
    long long splits = 512 / tiles;
    if (splits > ktiles / 4) splits = ktiles / 4;
    s.splits = splits < 1 ? 1 : splits > 32 ? 32 : (int)splits;
    return s;
}

template <typename T, bool AK, bool BKC, int OUT>
int product_launch(hipStream_t st, Product &P, const Shape &s) {
    P.tiles_m = s.tiles_m, P.tiles_n = s.tiles_n, P.splits = s.splits;
    P.part_ld = (P.n + 3) / 4 * 4;
    const long long blocks = (long long)s.tiles_m * s.tiles_n * s.splits;
    BT_REQUIRE(blocks < (1 << 24), "bt_affine: Mismatched sizes! (%lld tiles)", blocks);
    const dim3 grid((unsigned)blocks), block(256);
    if (s.splits > 1) {
        if (s.bm == 128)
            BT_LAUNCH(BTK_AFFINE, st, (affine_mm<T, 128, 128, AK, BKC, OUT_PART>), grid, block, 0, P);
        else
            BT_LAUNCH(BTK_AFFINE, st, (affine_mm<T, 64, 64, AK, BKC, OUT_PART>), grid, block, 0, P);
        BT_LAUNCH_CHECK();
        BT_LAUNCH(BTK_AFFINE, st, (affine_join<T, OUT>), dim3(bt_div_up(P.part_ld / 4 * P.m, 256)), block, 0, P);
    } else if (s.bm == 128) {
        BT_LAUNCH(BTK_AFFINE, st, (affine_mm<T, 128, 128, AK, BKC, OUT>), grid, block, 0, P);
    } else {
        BT_LAUNCH(BTK_AFFINE, st, (affine_mm<T, 64, 64, AK, BKC, OUT>), grid, block, 0, P);
    }
    BT_LAUNCH_CHECK();
    return BT_OK;
}

long long padded(int n, size_t es) { return (n + (16 / es) - 1) / (16 / es) * (16 / es); }
bool round_w(const bt_affine_desc *d) { return d->w_type != d->type; }
size_t round_w_bytes(const bt_affine_desc *d) {
    return round_w(d) ? bt_align((size_t)d->in * padded(d->out, 2) * 2) : 0;
}

template <typename T>
int make_w(hipStream_t st, const bt_affine_desc *d, const void *w, void *ws, Operand &o) {
    o.rows = d->in, o.len = d->out;
    if (round_w(d)) {
        const long long ld = padded(d->out, 2), quads = (long long)bt_div_up(d->out, 4) * d->in;
        BT_LAUNCH(BTK_AFFINE, st, affine_round_w<T>, dim3(bt_div_up(quads, 256)), dim3(256), 0, (const float *)w, (long long)d->w_ld,
                  (T *)ws, ld, d->in, d->out);
        BT_LAUNCH_CHECK();
        o.p[0] = o.p[1] = ws, o.ld = ld;
    } else {
        o.p[0] = o.p[1] = w, o.ld = d->w_ld;
    }
    o.aligned = chunk_aligned(o.p[0], o.ld, sizeof(T));
    return BT_OK;
}
Operand matrix(const void *p, long long ld, int rows, int len, size_t es) {
    return Operand{{p, p}, ld, rows, len, chunk_aligned(p, ld, es)};
}

template <typename T>
int forward(hipStream_t st, const bt_affine_desc *d, const void *w, const float *bias, const void *x, const void *residual, void *y,
            void *saved, char *ws) {
    const Shape s = shape_of(d->batch, d->out, d->in, 1, sizeof(T));
    Product P = {};
    if (int rc = make_w<T>(st, d, w, ws, P.b)) return rc;
    P.a = matrix(x, d->x_ld, d->batch, d->in, sizeof(T));
    P.m = d->batch, P.n = d->out, P.k = d->in, P.passes = 1;
    P.part = (float *)(ws + round_w_bytes(d));
    P.e = Epilogue{bias, residual, y, saved, d->y_ld, d->act, 1.0f};
    return product_launch<T, true, false, OUT_LAYER>(st, P, s);
}

struct BackwardPlan {
    bool pair, gz;   // gz kept as two numbers; kept at all (else grad_y is gz)
    float alpha;
    int range, ranges;
    Shape dw, dx;
    size_t w_bytes, gz_bytes, sum_bytes, part_bytes, total;
};
BackwardPlan backward_plan(const bt_affine_desc *d) {
    BackwardPlan p;
    const size_t es = type_size(d->type);
    const bool root = d->act == BT_ACT_SCRELU || d->act == BT_ACT_SQRRELU;
    p.gz = d->act != BT_ACT_IDENTITY;
    p.pair = root && es == 2;
    p.alpha = root ? 2.0f : 1.0f;
    p.range = 128;
    while (bt_div_up(d->batch, p.range) > 1024) p.range *= 2;
    p.ranges = bt_div_up(d->batch, p.range);
    p.dw = shape_of(d->in, d->out, d->batch, p.pair ? 2 : 1, es);
    p.dx = shape_of(d->batch, d->in, d->out, p.pair ? 2 : 1, es);
    p.w_bytes = round_w_bytes(d);
    p.gz_bytes = p.gz ? bt_align((size_t)d->batch * padded(d->out, es) * es) : 0;
    p.sum_bytes = bt_align((size_t)p.ranges * d->out * 4);
    const size_t a = p.dw.part_bytes(d->in, d->out), b = p.dx.part_bytes(d->batch, d->in);
    p.part_bytes = a > b ? a : b;
    p.total = p.w_bytes + p.gz_bytes * (p.pair ? 2 : 1) + p.sum_bytes + p.part_bytes;
    return p;
}

template <typename T>
int backward(hipStream_t st, const bt_affine_desc *d, const void *w, const void *x, const void *out, const void *gy, float *dw,
             float *dbias, void *gx, char *ws) {
    const BackwardPlan p = backward_plan(d);
    char *w16 = ws, *hi = w16 + p.w_bytes, *lo = hi + p.gz_bytes, *sums = hi + p.gz_bytes * (p.pair ? 2 : 1),
         *part = sums + p.sum_bytes;
    const bool keep = p.gz && (dw || gx);
    if (keep || dbias) {
        const dim3 grid(bt_div_up(d->out, GZ_COLS * Elem<T>::V), p.ranges);
        T *h = keep ? (T *)hi : nullptr;
        float *sum = dbias ? (float *)sums : nullptr;
        const T *o = p.gz ? (const T *)out : nullptr;
        if (keep && p.pair)
            BT_LAUNCH(BTK_AFFINE, st, (affine_gz<T, true>), grid, dim3(256), 0, (const T *)gy, o, (long long)d->y_ld, h, (T *)lo,
                      padded(d->out, sizeof(T)), sum, d->batch, d->out, d->act, p.range);
        else
            BT_LAUNCH(BTK_AFFINE, st, (affine_gz<T, false>), grid, dim3(256), 0, (const T *)gy, o, (long long)d->y_ld, h,
                      (T *)nullptr, padded(d->out, sizeof(T)), sum, d->batch, d->out, d->act, p.range);
        BT_LAUNCH_CHECK();
    }
    if (dbias) {
        BT_LAUNCH(BTK_AFFINE, st, affine_dbias, dim3(bt_div_up(d->out, 64)), dim3(1024), 0, (const float *)sums, p.ranges, d->out,
                  p.alpha, dbias);
        BT_LAUNCH_CHECK();
    }
    Operand gz = p.gz ? matrix(hi, padded(d->out, sizeof(T)), d->batch, d->out, sizeof(T))
                      : matrix(gy, d->y_ld, d->batch, d->out, sizeof(T));
    if (p.pair) gz.p[1] = lo;
    if (dw) {
        Product P = {};
        P.a = matrix(x, d->x_ld, d->batch, d->in, sizeof(T));
        P.b = gz;
        P.m = d->in, P.n = d->out, P.k = d->batch, P.passes = p.pair ? 2 : 1;
        P.part = (float *)part;
        P.e.out = dw, P.e.ld = d->w_ld, P.e.alpha = p.alpha;
        if (int rc = product_launch<T, false, false, OUT_F32>(st, P, p.dw)) return rc;
    }
    if (gx) {
        Product P = {};
        if (int rc = make_w<T>(st, d, w, w16, P.b)) return rc;
        P.a = gz;
        P.m = d->batch, P.n = d->in, P.k = d->out, P.passes = p.pair ? 2 : 1;
        P.part = (float *)part;
        P.e.out = gx, P.e.ld = d->x_ld, P.e.alpha = p.alpha;
        if (int rc = product_launch<T, true, true, OUT_TYPE>(st, P, p.dx)) return rc;
    }
    return BT_OK;
}

}  // namespace

extern "C" {

size_t bt_affine_forward_workspace_bytes(const bt_affine_desc *d) {
    if (validate(d, "bt_affine_forward_workspace_bytes")) return 0;
    return round_w_bytes(d) + shape_of(d->batch, d->out, d->in, 1, type_size(d->type)).part_bytes(d->batch, d->out);
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

}  // extern "C"
