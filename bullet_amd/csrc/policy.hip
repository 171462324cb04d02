// Losses of a policy head over masked moves, each with its gradient: the clipped policy loss with a KL term and the
// preference loss over pairs of lines of moves.
//
// Both are bound by the bytes of the logits: one group of lanes owns a row, keeps it in registers between the softmax
// statistics and the gradient, and so reads every logit once and writes every gradient once. Per-row scalars (log-sum,
// log-probability, ratio, losses) are computed in 64 bits from the row's 32-bit sum: they cost one evaluation a row and
// keep the rounding of values near 7 out of differences that may be near 0.
//
// Times in this file: of the last of some thousand launches in a row, over inputs that the caches do not hold.
#include <type_traits>

#include "common.h"

namespace {

constexpr float NEG_INF = -__builtin_huge_valf();

template <typename T>
struct Row {
    static constexpr int V = 16 / sizeof(T);  // elements of a 16-byte chunk
    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
    typedef typename std::conditional<sizeof(T) == 4, uint32_t, uint64_t>::type bytes;  // one mask byte per element
};

// exp(x) for x <= 0 in 32 bits, to 2^-22 of itself: 2^t of the rounded t = x log2(e), and what the rounding left over, x - t ln 2
// (ln 2 as two numbers), multiplied in; without it the entries of a gradient lose 2^-24 |x|. Below -150 it is 0 in 32 bits; the
// maximum keeps -infinity out of the differences and lets NaN pass.
__device__ __forceinline__ float exp_neg(float x) {
    const float c = __builtin_elementwise_maximum(x, -150.0f), t = c * 1.44269502f;
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, fmaf(t, 1.90465421e-9f, fmaf(t, -0.693147182f, c)), e);
}

// The scalars of a row in 64 bits, each computed by all its lanes, so shorter than the library's functions: their arguments
// are finite sums and differences of logits, and 1e-13 is plenty.
// (e^r - 1 - r) / r^2 for |r| <= ln 2 / 2, by the Taylor series to r^11 / 11! (remainder below 1e-13)
__device__ __forceinline__ double exp_rest(double r) {
    double p = 1.0 / 39916800.0;
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    return fma(p, r, 0.5);
}
// e^x = 2^n e^r, n = round(x log2 e)
__device__ __forceinline__ double exp64(double x) {
    const double n = rint(x * 1.4426950408889634074);
    // (x - n ln 2 after Cody and Waite: of ln 2 first its 40 leading bits, whose product with n is exact, then the rest)
    double r = fma(n, -0x1.62e42fefa2p-1, x);
    r = fma(n, -0x1.9ef35793c7673p-41, r);
    const double p = fma(fma(exp_rest(r), r, 1.0), r, 1.0);
    const double m = fmin(fmax(n, -1100.0), 1100.0);
    const double v = ldexp(p, (int)m);
    // (beyond the range of r's reduction, and infinities: the limits; NaN goes through)
    return x > 709.0 ? __builtin_huge_val() : x < -745.0 ? 0.0 : v;
}
// The estimate exp(x) - 1 - x of a KL and its derivative exp(x) - 1. Near 0 their own series: the difference would leave the
// rounding of the 1, which is more than x^2 / 2 below |x| = 1e-8 and can be less than 0, what the estimate never is.
__device__ __forceinline__ double kl_estimate(double x, double &em1) {
    if (fabs(x) < 0.3) {
        const double rest = x * x * exp_rest(x);
        em1 = x + rest;
        return rest;
    }
    em1 = exp64(x) - 1.0;
    return em1 < __builtin_huge_val() ? em1 - x : em1;  // (a move at -infinity, x = infinity: not infinity - infinity)
}
// 1 / d: the hardware's estimate, squared twice in its error by Newton's steps
__device__ __forceinline__ double inverse64(double d) {
    double i = __builtin_amdgcn_rcp(d);
    i = i * fma(-d, i, 2.0);
    return i * fma(-d, i, 2.0);
}
// log s for a normal s > 0: s = 2^n m, m in [sqrt 1/2, sqrt 2), log m = 2 atanh t, t = (m - 1) / (m + 1), |t| <= 0.172, by its
// series to t^15 / 15 (remainder below 1e-14)
__device__ __forceinline__ double log64(double s) {
    int n;
    double m = frexp(s, &n);  // [1/2, 1)
    if (m < 0.70710678118654752440) m *= 2.0, n -= 1;
    const double t = (m - 1.0) * inverse64(m + 1.0), u = t * t;
    double p = 2.0 / 15.0;
    p = fma(p, u, 2.0 / 13.0);
    p = fma(p, u, 2.0 / 11.0);
    p = fma(p, u, 2.0 / 9.0);
    p = fma(p, u, 2.0 / 7.0);
    p = fma(p, u, 2.0 / 5.0);
    p = fma(p, u, 2.0 / 3.0);
    p = fma(p, u, 2.0);
    return fma((double)n, 0.69314718055994530942, t * p);
}

// a launch holds less than 2^32 threads a dimension: many rows fold into the grid's second one
__device__ __forceinline__ long long row_block() { return (long long)blockIdx.y * gridDim.x + blockIdx.x; }
dim3 row_grid(long long blocks) {
    constexpr long long W = 1 << 22;
    return blocks <= W ? dim3((unsigned)blocks) : dim3((unsigned)W, (unsigned)((blocks + W - 1) / W));
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float lane_value(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

// Reductions over the G lanes that own a row: 8 lanes (short rows, eight rows a wave), a wave, or a workgroup of 256.
// The order is fixed. Lane exchanges inside 16 lanes are DPP moves, no LDS.
template <int G>
struct Group {
    template <typename F>
    static __device__ __forceinline__ float reduce(float v, F f, float *red) {
        v = f(v, dpp<0xB1>(v));   // lane ^ 1
        v = f(v, dpp<0x4E>(v));   // lane ^ 2
        v = f(v, dpp<0x141>(v));  // mirrored within 8
        if (G == 8) return v;
        v = f(v, dpp<0x140>(v));  // mirrored within 16
        v = f(f(lane_value(v, 0), lane_value(v, 16)), f(lane_value(v, 32), lane_value(v, 48)));
        if (G == 64) return v;
        __syncthreads();  // the previous reduction's values have been read
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        return f(f(red[0], red[1]), f(red[2], red[3]));
    }
    static __device__ __forceinline__ float max(float v, float *red) {
        return reduce(v, [](float a, float b) { return fmaxf(a, b); }, red);
    }
    static __device__ __forceinline__ float sum(float v, float *red) {
        return reduce(v, [](float a, float b) { return a + b; }, red);
    }
    static __device__ double sum64(double v, double *red) {
        for (int o = 1; o < (G < 64 ? G : 64); o <<= 1) v += __shfl_xor(v, o, 64);
        if (G <= 64) return v;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        return (red[0] + red[1]) + (red[2] + red[3]);
    }
};

// one mask byte per element of the chunk that starts at element e0: 0 where there is no element or no legal move
template <typename T>
__device__ __forceinline__ typename Row<T>::bytes legal_bytes(const uint8_t *mask, int e0, int width) {
    typedef typename Row<T>::bytes B;
    constexpr int V = Row<T>::V;
    const int n = width - e0;
    if (n <= 0) return 0;
    if (!mask) return n >= V ? (B)0x0101010101010101ull : (B)0x0101010101010101ull & (((B)1 << (8 * n)) - 1);
    B b = 0;
    if (n >= V) {
        __builtin_memcpy(&b, mask + e0, V);
    } else {
        for (int j = 0; j < n; j++) b |= (B)mask[e0 + j] << (8 * j);
    }
    return b;
}
template <typename B>
__device__ __forceinline__ bool legal_at(B b, int j) {
    return (b >> (8 * j)) & 0xff;
}
// the chunk that starts at element e0. (Not under the mask's control, although few moves are legal: waiting for the mask's
// bytes costs more than the skipped chunks save, 112 us instead of 83 for 16384 x 1880 f32 with 35 legal moves a row.)
template <typename T>
__device__ __forceinline__ void load_chunk(const T *row, int e0, int width, typename Row<T>::vec &v) {
    constexpr int V = Row<T>::V;
    if (e0 < width) {
        if (width - e0 >= V) {
            __builtin_memcpy(&v, row + e0, 16);
        } else {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (j < width - e0) v[j] = row[e0 + j];
        }
    }
}
// (without a mask only a row's last chunk can have anything to leave out; chunks beyond it count as such)
template <typename T>
__device__ __forceinline__ void keep_legal(const uint8_t *mask, int e0, int width, typename Row<T>::bytes b, typename Row<T>::vec &v) {
    if (mask || width - e0 < Row<T>::V) {
#pragma unroll
        for (int j = 0; j < Row<T>::V; j++) v[j] = legal_at(b, j) ? v[j] : (T)NEG_INF;
    }
}
// (Past the caches: nothing here reads it again, and the logits stay where the gradient would push them out. Whole calls: 8192 x
// 4096 bf16 37 us, with ordinary stores 40; 256 pairs of lines, whose logits are read twice, 54 and 60; 16384 x 1880 f32 83 and 85.
// Loads past the caches are slower, 112 us instead of 83 for the last.)
template <typename T>
__device__ __forceinline__ void store_chunk(T *row, int e0, int width, typename Row<T>::vec v) {
    constexpr int V = Row<T>::V;
    typedef T any __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    if (width - e0 >= V) {
        __builtin_nontemporal_store((any)v, (any *)(row + e0));
    } else {
#pragma unroll
        for (int j = 0; j < V; j++)
            if (j < width - e0) row[e0 + j] = v[j];
    }
}

// Softmax statistics of one row, and what the KL over the whole policy needs beside them.
template <typename S>  // (32 bits where rows fill registers: 64 would cost one of three waves a SIMD, 87 us instead of 83)
struct RowStats {
    float top, ref_top;  // largest legal logit
    S sum, ref_sum;      // sum of exp(z - top)
    S cross;             // sum of exp(z - top) (z - q)
};

// What a row's element needs for its gradient: with e = exp(z - top), g = ce e (+ a share of its own for the action taken),
// and for the full KL + ck e (z - q - shift). Masked (and vanishing) places, e = 0, get 0 whatever the row's scalars are.
struct RowGrad {
    float top, ce, ck, shift;
    bool plain;  // ce is finite: ce e is 0 by itself where e is
};
template <typename T, bool FULL>
__device__ __forceinline__ typename Row<T>::vec grad_chunk(const float (&e)[Row<T>::V], const typename Row<T>::vec &z,
                                                           const typename Row<T>::vec &q, const RowGrad &r) {
    typename Row<T>::vec out;
    if (FULL || !r.plain) {
#pragma unroll
        for (int j = 0; j < Row<T>::V; j++) {
            float g = r.ce * e[j];
            if (FULL && r.ck != 0.0f) g = fmaf(r.ck * e[j], ((float)z[j] - (float)q[j]) - r.shift, g);
            out[j] = (T)(e[j] == 0.0f ? 0.0f : g);
        }
    } else {
#pragma unroll
        for (int j = 0; j < Row<T>::V; j++) out[j] = (T)(r.ce * e[j]);
    }
    return out;
}

struct PolicyArgs {
    const void *z, *ref;
    const uint8_t *mask;
    const int32_t *actions;
    const float *old_logp, *advantages, *weights;
    void *grad;
    float *row_loss, *row_logp, *row_kl;
    bt_policy_desc d;
};

// The whole of one row once its statistics are known: losses, row outputs and the coefficients of its gradient.
// `near` is set when the ratio stands so close to a clipping border that the row's 32-bit sum cannot say on which side:
// the caller then sums again in 64 bits and asks once more (sum64 > 0).
struct PolicyRow {
    float za, qa;    // logit (and reference logit) of the action taken
    bool counted;
};
template <typename S>
__device__ __forceinline__ bool policy_scalars(const PolicyArgs &a, int row, const PolicyRow &pr, const RowStats<S> &st,
                                               double sum64, bool full, RowGrad &g, double &logp, double &kl, float &loss, float &grad_taken) {
    const bt_policy_desc &d = a.d;
    const double logsum = log64(sum64 > 0.0 ? sum64 : (double)st.sum);
    logp = ((double)pr.za - (double)st.top) - logsum;
    const double adv = a.advantages[row], w = a.weights ? (double)a.weights[row] : 1.0;
    const double r = exp64(logp - (double)a.old_logp[row]);
    const double lo = 1.0 - (double)d.clip_low, hi = 1.0 + (double)d.clip_high;
    // (sum: 74 roundings of 2^-24 at most, 64 of a lane's own and 10 of the lanes', or 7 where chunks are added in 64 bits;
    // with its terms' own errors less than 1e-5 of it)
    const bool near = fabs(r - lo) < 1e-5 * lo || fabs(r - hi) < 1e-5 * hi;
    const double free_gain = r * adv, held_gain = fmin(fmax(r, lo), hi) * adv;
    double slope = free_gain <= held_gain || free_gain != free_gain ? -free_gain : 0.0;
    kl = 0.0;
    double ck = 0.0;
    g.shift = 0.0f;
    if (d.kl == BT_KL_TAKEN) {
        const double x = (double)((const float *)a.ref)[row] - logp;
        double em1;
        kl = kl_estimate(x, em1);
        if (d.kl_weight != 0.0f) slope -= (double)d.kl_weight * em1;
    } else if (full) {
        const double dl = ((double)st.top + logsum) - ((double)st.ref_top + log64((double)st.ref_sum));
        kl = (double)st.cross / (double)st.sum - dl;
        ck = w * (double)d.kl_weight;
        g.shift = (float)(dl + kl);
    }
    // (no weight: a KL that is infinite is none either; NaN stays)
    const double held_kl = d.kl_weight != 0.0f || kl != kl ? (double)d.kl_weight * kl : 0.0;
    loss = (float)(w * (held_kl - (free_gain != free_gain ? free_gain : fmin(free_gain, held_gain))));
    g.top = st.top == NEG_INF ? 0.0f : st.top;  // (nothing but NaN)
    const double inv = inverse64((double)st.sum);
    g.ce = -(float)(w * slope * inv);
    g.ck = (float)(ck * inv);
    g.plain = fabsf(g.ce) < __builtin_huge_valf();
    const double pa = exp64(logp);
    grad_taken = (float)(w * slope * (1.0 - pa));
    if (full && pa > 0.0 && ck != 0.0) grad_taken += (float)(ck * pa * (((double)pr.za - (double)pr.qa) - (double)g.shift));
    return near;
}

template <typename T>
__device__ __forceinline__ PolicyRow policy_row_begin(const PolicyArgs &a, const T *z, const T *q, const uint8_t *mask, int row,
                                                      bool full) {
    PolicyRow pr{0.0f, 0.0f, false};
    const int act = a.actions[row];
    pr.counted = act >= 0 && act < a.d.width && (!mask || mask[act]);
    if (pr.counted) {
        pr.za = (float)z[act];
        if (full) pr.qa = (float)q[act];
    }
    return pr;
}
// The gradient may lie where the logits are: the move's logit has to be here in every wave of a row before the barrier behind
// which another one of them may write there.
__device__ __forceinline__ void taken_is_here(const PolicyRow &pr) { asm volatile("" : : "v"(pr.za) : "memory"); }
__device__ __forceinline__ void policy_row_out(const PolicyArgs &a, int row, bool counted, float loss, double logp, double kl) {
    a.row_loss[row] = counted ? loss : 0.0f;
    if (a.row_logp) a.row_logp[row] = counted ? (float)logp : 0.0f;
    if (a.row_kl) a.row_kl[row] = counted ? (float)kl : 0.0f;
}

// this lane's share of the row's sum, from memory and in 64 bits (rare: see policy_scalars)
template <typename T, int G>
__device__ __noinline__ double sum_again(const T *z, const uint8_t *mask, int width, int lane, float top) {
    double s = 0.0;
    for (long long e = lane; e < width; e += G)
        if (!mask || mask[e]) s += exp((double)(float)z[e] - (double)top);
    return s;
}

// One group of G lanes per row, at most K chunks a lane, all in registers.
// Bound by memory where there are many rows: 16384 x 1880 f32 with the full KL (two rows of logits and the mask in, gradient
// out, 401 MB) 80 us, 5.0 TB/s, what a copy reaches; 8192 x 4096 bf16 (134 MB) 33 us, 4.0 TB/s. Few rows: 6.7 us for 64 of
// 1880, the time of a launch and of four loads in turn (mask and logits, the action, its logit, its row's scalars).
template <typename T, int G, int K, bool FULL>
__global__ __launch_bounds__(256) void policy_rows(PolicyArgs a) {
    constexpr int V = Row<T>::V;
    typedef typename Row<T>::vec vec;
    typedef typename Row<T>::bytes bytes;
    __shared__ float red[4];
    __shared__ double red64[4];
    const int lane = threadIdx.x % G;
    const long long row64 = row_block() * (256 / G) + threadIdx.x / G;
    if (row64 >= a.d.batch) return;  // (whole groups)
    const int row = (int)row64;
    const int width = a.d.width;
    const T *z = (const T *)a.z + (size_t)row * a.d.ld;
    const T *q = FULL ? (const T *)a.ref + (size_t)row * a.d.ld : nullptr;
    const uint8_t *mask = a.mask ? a.mask + (size_t)row * a.d.mask_ld : nullptr;
    bytes b[K];
    vec zc[K], qc[FULL ? K : 1];
#pragma unroll
    for (int k = 0; k < K; k++) b[k] = legal_bytes<T>(mask, (lane + k * G) * V, width);
#pragma unroll
    for (int k = 0; k < K; k++) {
        load_chunk<T>(z, (lane + k * G) * V, width, zc[k]);
        if (FULL) load_chunk<T>(q, (lane + k * G) * V, width, qc[FULL ? k : 0]);
    }
    const PolicyRow pr = policy_row_begin(a, z, q, mask, row, FULL);  // (its three loads in turn: behind those of the row)
    float top = NEG_INF, ref_top = NEG_INF;
#pragma unroll
    for (int k = 0; k < K; k++) {
        keep_legal<T>(mask, (lane + k * G) * V, width, b[k], zc[k]);
#pragma unroll
        for (int j = 0; j < V; j++) top = fmaxf(top, (float)zc[k][j]);
        if (FULL) {
            keep_legal<T>(mask, (lane + k * G) * V, width, b[k], qc[FULL ? k : 0]);
#pragma unroll
            for (int j = 0; j < V; j++) ref_top = fmaxf(ref_top, (float)qc[FULL ? k : 0][j]);
        }
    }
    RowStats<float> st;
    st.top = Group<G>::max(top, red);
    st.ref_top = FULL ? Group<G>::max(ref_top, red) : 0.0f;
    const float base = st.top == NEG_INF ? 0.0f : st.top;  // (nothing left: every term is exp(-infinity) = 0)
    float e[K][V], s = 0.0f, sq = 0.0f, cross = 0.0f;
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float zv = (float)zc[k][j];
            e[k][j] = exp_neg(zv - base);
            s += e[k][j];
            if (FULL) {
                const float qv = (float)qc[FULL ? k : 0][j];
                sq += exp_neg(qv - st.ref_top);
                cross += e[k][j] == 0.0f ? 0.0f : e[k][j] * (zv - qv);
            }
        }
    if (G > 64) taken_is_here(pr);
    st.sum = Group<G>::sum(s, red);
    st.ref_sum = FULL ? Group<G>::sum(sq, red) : 1.0f;
    st.cross = FULL ? Group<G>::sum(cross, red) : 0.0f;
    const bool counted = pr.counted && st.sum != 0.0f;  // (0: nothing above -infinity; NaN counts)

    T *grad = a.grad ? (T *)a.grad + (size_t)row * a.d.ld : nullptr;
    if (!counted) {
        if (lane == 0) policy_row_out(a, row, false, 0.0f, 0.0, 0.0);
        if (grad) {
            vec zero = {};
#pragma unroll
            for (int k = 0; k < K; k++) store_chunk<T>(grad, (lane + k * G) * V, width, zero);
        }
        return;
    }
    RowGrad g;
    double logp, kl;
    float loss, grad_taken;
    if (policy_scalars(a, row, pr, st, 0.0, FULL, g, logp, kl, loss, grad_taken)) {
        const double s64 = Group<G>::sum64(sum_again<T, G>(z, mask, width, lane, st.top), red64);
        policy_scalars(a, row, pr, st, s64, FULL, g, logp, kl, loss, grad_taken);
    }
    if (lane == 0) policy_row_out(a, row, true, loss, logp, kl);
    if (!grad) return;
#pragma unroll
    for (int k = 0; k < K; k++) {
        store_chunk<T>(grad, (lane + k * G) * V, width, grad_chunk<T, FULL>(e[k], zc[k], qc[FULL ? k : 0], g));
    }
    // the action taken: written again by the lane that wrote its chunk
    const int act = a.actions[row];
    if (lane == (act / V) % G) grad[act] = (T)grad_taken;
}

// A lane's running maximum and sum of exponentials, for rows too wide for registers. A chunk's terms are added in 32 bits, the
// chunks in 64: thousands of equal terms (16-bit logits repeat) round the same way every time, and what 32 bits would lose,
// 6e-5 of the sum of 2^20 of them, is more than a ratio next to a clipping border can bear.
struct Running {
    float top = NEG_INF;
    double sum = 0.0;
    __device__ __forceinline__ float base() const { return top == NEG_INF ? 0.0f : top; }
    // what the sums so far are multiplied by
    __device__ __forceinline__ double raise(float m) {
        const double f = exp64((double)top - (double)m);
        sum *= f, top = m;
        return f;
    }
    // this lane's share of the sum beside the row's maximum (without a finite maximum: 0 or NaN)
    __device__ __forceinline__ double scale(float row_top) const { return top == NEG_INF ? 1.0 : exp64((double)top - (double)row_top); }
};

// Rows too wide for the registers of a workgroup: running maximum and sums in one pass, the gradient in a second one.
template <typename T, bool FULL>
__global__ __launch_bounds__(256) void policy_rows_long(PolicyArgs a) {
    constexpr int V = Row<T>::V;
    typedef typename Row<T>::vec vec;
    typedef typename Row<T>::bytes bytes;
    __shared__ float red[4];
    __shared__ double red64[4];
    const long long row64 = row_block();
    if (row64 >= a.d.batch) return;
    const int row = (int)row64, lane = threadIdx.x, width = a.d.width;
    const T *z = (const T *)a.z + (size_t)row * a.d.ld;
    const T *q = FULL ? (const T *)a.ref + (size_t)row * a.d.ld : nullptr;
    const uint8_t *mask = a.mask ? a.mask + (size_t)row * a.d.mask_ld : nullptr;
    const PolicyRow pr = policy_row_begin(a, z, q, mask, row, FULL);
    Running z_run, q_run;
    double cross = 0.0;
    for (long long e0 = (long long)lane * V; e0 < width; e0 += 256 * V) {
        const bytes b = legal_bytes<T>(mask, (int)e0, width);
        vec zc, qc;
        load_chunk<T>(z, (int)e0, width, zc);
        keep_legal<T>(mask, (int)e0, width, b, zc);
        if (FULL) {
            load_chunk<T>(q, (int)e0, width, qc);
            keep_legal<T>(mask, (int)e0, width, b, qc);
        }
        float m = z_run.top, mq = q_run.top;
        for (int j = 0; j < V; j++) {
            m = fmaxf(m, (float)zc[j]);
            if (FULL) mq = fmaxf(mq, (float)qc[j]);
        }
        if (m > z_run.top) cross *= z_run.raise(m);
        if (FULL && mq > q_run.top) q_run.raise(mq);
        float s = 0.0f, sq = 0.0f, sc = 0.0f;  // of this chunk
        for (int j = 0; j < V; j++) {
            const float zv = (float)zc[j], e = exp_neg(zv - z_run.base());
            s += e;
            if (FULL) {
                const float qv = (float)qc[j];
                sq += exp_neg(qv - q_run.base());
                sc += e == 0.0f ? 0.0f : e * (zv - qv);
            }
        }
        z_run.sum += s, q_run.sum += sq, cross += sc;
    }
    RowStats<double> st;
    st.top = Group<256>::max(z_run.top, red);
    taken_is_here(pr);
    const double f = z_run.scale(st.top);
    st.sum = Group<256>::sum64(z_run.sum * f, red64);
    st.ref_top = FULL ? Group<256>::max(q_run.top, red) : 0.0f;
    st.ref_sum = FULL ? Group<256>::sum64(q_run.sum * q_run.scale(st.ref_top), red64) : 1.0;
    st.cross = FULL ? Group<256>::sum64(cross * f, red64) : 0.0;
    const bool counted = pr.counted && st.sum != 0.0;  // (0: nothing above -infinity; NaN counts)
    T *grad = a.grad ? (T *)a.grad + (size_t)row * a.d.ld : nullptr;
    RowGrad g;
    double logp = 0.0, kl = 0.0;
    float loss = 0.0f, grad_taken = 0.0f;
    if (counted && policy_scalars(a, row, pr, st, 0.0, FULL, g, logp, kl, loss, grad_taken)) {
        const double s64 = Group<256>::sum64(sum_again<T, 256>(z, mask, width, lane, st.top), red64);
        policy_scalars(a, row, pr, st, s64, FULL, g, logp, kl, loss, grad_taken);
    }
    if (lane == 0) policy_row_out(a, row, counted, loss, logp, kl);
    if (!grad) return;
    for (long long e0 = (long long)lane * V; e0 < width; e0 += 256 * V) {
        vec out = {};
        if (counted) {
            const bytes b = legal_bytes<T>(mask, (int)e0, width);
            vec zc = {}, qc = {};
            load_chunk<T>(z, (int)e0, width, zc);
            keep_legal<T>(mask, (int)e0, width, b, zc);
            if (FULL) {
                load_chunk<T>(q, (int)e0, width, qc);
                keep_legal<T>(mask, (int)e0, width, b, qc);
            }
            float e[V];
            for (int j = 0; j < V; j++) e[j] = exp_neg((float)zc[j] - g.top);
            out = grad_chunk<T, FULL>(e, zc, qc, g);
        }
        store_chunk<T>(grad, (int)e0, width, out);
    }
    const int act = a.actions[row];
    if (counted && lane == (act / V) % 256) grad[act] = (T)grad_taken;
}

// loss_sum = sum of n losses, in 64 bits and a fixed order, by THREADS threads: 1.7 us for 64 losses, 4.6 for 16384. (A launch of
// its own, since the last row kernel's workgroup to finish could only add them up behind an atomic counter, which a captured
// and an eager call of the same buffers would have to share.)
template <int THREADS>
__device__ __forceinline__ void loss_sum(const float *rows, int n, float *out) {
    __shared__ double red[THREADS / 64];
    double s = 0.0;
    const int tid = threadIdx.x;
    long long i = tid;
    for (; i + 7 * THREADS < n; i += 8 * THREADS) {  // eight loads in flight
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = rows[i + j * THREADS];
#pragma unroll
        for (int j = 0; j < 8; j++) s += (double)v[j];
    }
    for (; i < n; i += THREADS) s += (double)rows[i];
    for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
    if ((tid & 63) == 0) red[tid >> 6] = s;
    __syncthreads();
    if (tid == 0) {
        for (int j = 1; j < THREADS / 64; j++) s += red[j];
        out[0] = (float)s;
    }
}
__global__ __launch_bounds__(1024) void loss_sum_kernel(const float *__restrict__ rows, int n, float *__restrict__ out) {
    loss_sum<1024>(rows, n, out);
}

// ---- preference loss: row statistics -> pairs -> gradient rows
struct PrefArgs {
    const void *z;
    const uint8_t *mask;
    const int32_t *actions, *offsets;
    const float *ref, *weights;
    void *grad;
    float *pair_loss, *line_logp, *loss_sum;
    // per row: logit of the action taken, the largest legal one, the sum of exp(z - top) (0: the row is not
    // counted), and what the pair kernel adds: the gradient's factor on p and the taken action's own gradient
    float *za, *top, *sum, *ce, *taken;
    bt_preference_desc d;
};
__device__ __forceinline__ int pref_offset(const PrefArgs &a, int k) { return min(max(a.offsets[k], 0), a.d.rows); }

// Statistics of one row, as in policy_rows. The rows are read again for the gradient, since a pair's factor needs all
// rows of both its lines first: 16740 x 1880 bf16 (logits and mask 94 MB) 22 us, 4.3 TB/s.
template <typename T, int G, int K>
__global__ __launch_bounds__(256) void pref_rows(PrefArgs a) {
    constexpr int V = Row<T>::V;
    __shared__ float red[4];
    __shared__ double red64[4];
    const int lane = threadIdx.x % G;
    const long long row64 = row_block() * (256 / G) + threadIdx.x / G;
    if (row64 < pref_offset(a, 0) || row64 >= pref_offset(a, 2 * a.d.pairs)) return;
    const int row = (int)row64;
    const int width = a.d.width;
    const T *z = (const T *)a.z + (size_t)row * a.d.ld;
    const uint8_t *mask = a.mask ? a.mask + (size_t)row * a.d.mask_ld : nullptr;
    const int act = a.actions[row];
    const bool can = act >= 0 && act < width && (!mask || mask[act]);
    const float za = can ? (float)z[act] : 0.0f;
    float top = NEG_INF, s = 0.0f;
    if constexpr (K > 0) {
        typename Row<T>::bytes b[K];
        typename Row<T>::vec zc[K];
#pragma unroll
        for (int k = 0; k < K; k++) b[k] = legal_bytes<T>(mask, (lane + k * G) * V, width);
#pragma unroll
        for (int k = 0; k < K; k++) load_chunk<T>(z, (lane + k * G) * V, width, zc[k]);
#pragma unroll
        for (int k = 0; k < K; k++) {
            keep_legal<T>(mask, (lane + k * G) * V, width, b[k], zc[k]);
#pragma unroll
            for (int j = 0; j < V; j++) top = fmaxf(top, (float)zc[k][j]);
        }
        top = Group<G>::max(top, red);
        const float base = top == NEG_INF ? 0.0f : top;
#pragma unroll
        for (int k = 0; k < K; k++)
#pragma unroll
            for (int j = 0; j < V; j++) s += exp_neg((float)zc[k][j] - base);
        s = Group<G>::sum(s, red);
    } else {  // any width
        Running run;
        for (long long e0 = (long long)lane * V; e0 < width; e0 += G * V) {
            const typename Row<T>::bytes b = legal_bytes<T>(mask, (int)e0, width);
            typename Row<T>::vec zc;
            load_chunk<T>(z, (int)e0, width, zc);
            keep_legal<T>(mask, (int)e0, width, b, zc);
            float m = run.top;
            for (int j = 0; j < V; j++) m = fmaxf(m, (float)zc[j]);
            if (m > run.top) run.raise(m);
            float c = 0.0f;
            for (int j = 0; j < V; j++) c += exp_neg((float)zc[j] - run.base());
            run.sum += c;
        }
        top = Group<G>::max(run.top, red);
        s = (float)Group<G>::sum64(run.sum * run.scale(top), red64);
    }
    if (lane == 0) {
        a.za[row] = za;
        a.top[row] = top == NEG_INF ? 0.0f : top;  // (nothing, or nothing but NaN)
        a.sum[row] = can ? s : 0.0f;
    }
}

// One wave per pair, one row a lane: the lines' sums and the pair's loss, then what its rows' gradients need. Loads in turn
// bound it (the offsets, the rows' numbers, then 64-bit arithmetic on them): 4.4 us for 4 pairs, 5.9 for 256.
__global__ __launch_bounds__(256) void pref_pairs(PrefArgs a) {
    const long long p64 = row_block() * 4 + (threadIdx.x >> 6);
    const int p = (int)p64, lane = threadIdx.x & 63;
    if (p64 >= a.d.pairs) return;
    // a lane's first row of each line stays in registers (lines are seldom longer than a wave)
    struct Entry {
        float sum;
        double logp;
    };
    const auto entry = [&](long long r) {
        Entry e{a.sum[r], 0.0};
        const double rel = (double)a.za[r] - (double)a.top[r];
        if (e.sum != 0.0f) e.logp = rel - log64((double)e.sum);
        return e;
    };
    int r0[2], r1[2];
    Entry first[2];
#pragma unroll
    for (int h = 0; h < 2; h++) r0[h] = pref_offset(a, 2 * p + h) + lane, r1[h] = pref_offset(a, 2 * p + h + 1);
#pragma unroll
    for (int h = 0; h < 2; h++) first[h] = r0[h] < r1[h] ? entry(r0[h]) : Entry{0.0f, 0.0};
    double s[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        double v = first[h].logp;
        for (long long r = r0[h] + 64ll; r < r1[h]; r += 64) v += entry(r).logp;
        for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
        s[h] = v;
    }
    const double beta = a.d.beta, eps = a.d.smoothing, w = a.weights ? (double)a.weights[p] : 1.0;
    const double x = beta * ((s[0] - (double)a.ref[2 * p]) - (s[1] - (double)a.ref[2 * p + 1]));
    // sigmoid(x) - (1 - eps), written so that nothing cancels for large x
    const double slope = w * beta * (eps - 1.0 / (1.0 + exp64(x)));
    if (lane == 0) {
        const double soft = log1p(exp64(-fabs(x)));  // -log sigmoid(x) = soft - min(x, 0)
        const double other = eps > 0.0 || x != x ? eps * (soft + fmax(x, 0.0)) : 0.0;  // (an infinite one that has no share is none)
        a.pair_loss[p] = (float)(w * ((1.0 - eps) * (soft - fmin(x, 0.0)) + other));
        if (a.line_logp) a.line_logp[2 * p] = (float)s[0], a.line_logp[2 * p + 1] = (float)s[1];
    }
    if (!a.grad) return;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const double c = h ? -slope : slope;
        const auto put = [&](long long r, const Entry &e) {
            const bool counted = e.sum != 0.0f;
            a.ce[r] = counted ? -(float)(c * inverse64((double)e.sum)) : 0.0f;
            a.taken[r] = counted ? (float)(c * (1.0 - exp64(e.logp))) : 0.0f;
        };
        if (r0[h] < r1[h]) put(r0[h], first[h]);
        for (long long r = r0[h] + 64ll; r < r1[h]; r += 64) put(r, entry(r));
    }
}

// The gradient of one row: its logits once more, the numbers its pair left for it, one write. 16740 x 1880 bf16: 26 us for
// logits, mask and gradient, 157 MB at 6.0 TB/s, some of it still in the caches. (The first workgroup adds the pairs'
// losses up, the others follow with the rows.)
template <typename T, int G, int K>
__global__ __launch_bounds__(256) void pref_grad(PrefArgs a) {
    constexpr int V = Row<T>::V;
    const long long block = row_block();
    if (block == 0) {
        loss_sum<256>(a.pair_loss, a.d.pairs, a.loss_sum);
        return;
    }
    const int lane = threadIdx.x % G;
    const long long row64 = (block - 1) * (256 / G) + threadIdx.x / G;
    if (row64 < pref_offset(a, 0) || row64 >= pref_offset(a, 2 * a.d.pairs)) return;
    const int row = (int)row64;
    const int width = a.d.width, act = a.actions[row];
    const T *z = (const T *)a.z + (size_t)row * a.d.ld;
    const uint8_t *mask = a.mask ? a.mask + (size_t)row * a.d.mask_ld : nullptr;
    T *grad = (T *)a.grad + (size_t)row * a.d.ld;
    RowGrad g{a.top[row], a.ce[row], 0.0f, 0.0f, false};
    g.plain = fabsf(g.ce) < __builtin_huge_valf();
    const bool counted = a.sum[row] != 0.0f;
    const float taken = a.taken[row];
    const auto gradient = [&](int e0, typename Row<T>::bytes b, typename Row<T>::vec &zc) {
        keep_legal<T>(mask, e0, width, b, zc);
        float e[V];
#pragma unroll
        for (int j = 0; j < V; j++) e[j] = exp_neg((float)zc[j] - g.top);
        store_chunk<T>(grad, e0, width, grad_chunk<T, false>(e, zc, zc, g));
    };
    const typename Row<T>::vec none = {};
    if constexpr (K > 0) {
        typename Row<T>::bytes b[K];
        typename Row<T>::vec zc[K];
#pragma unroll
        for (int k = 0; k < K; k++) b[k] = legal_bytes<T>(mask, (lane + k * G) * V, width);
#pragma unroll
        for (int k = 0; k < K; k++) load_chunk<T>(z, (lane + k * G) * V, width, zc[k]);
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (counted)
                gradient((lane + k * G) * V, b[k], zc[k]);
            else
                store_chunk<T>(grad, (lane + k * G) * V, width, none);
        }
    } else {
        for (long long e0 = (long long)lane * V; e0 < width; e0 += G * V) {
            if (counted) {
                const typename Row<T>::bytes b = legal_bytes<T>(mask, (int)e0, width);
                typename Row<T>::vec zc;
                load_chunk<T>(z, (int)e0, width, zc);
                gradient((int)e0, b, zc);
            } else {
                store_chunk<T>(grad, (int)e0, width, none);
            }
        }
    }
    if (counted && lane == (act / V) % G) grad[act] = (T)taken;
}

// ---- host side
int type_size(int type) { return type == BT_TYPE_F32 ? 4 : 2; }
bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

int matrix_validate(const char *fn, int type, int width, int ld, int mask_ld, bool mask) {
    BT_REQUIRE(type == BT_TYPE_F32 || type == BT_TYPE_BF16 || type == BT_TYPE_F16, "%s: unknown element type %d", fn, type);
    BT_REQUIRE(width > 0, "%s: Mismatched sizes! (width <= 0)", fn);
    BT_REQUIRE(ld >= width, "%s: Mismatched sizes! (leading dimension %d < width %d)", fn, ld, width);
    BT_REQUIRE(!mask || mask_ld >= width, "%s: Mismatched sizes! (mask leading dimension %d < width %d)", fn, mask_ld, width);
    return BT_OK;
}

// Lanes per row and chunks per lane. A row stays in one wave's registers up to 8 chunks a lane (2048 f32 or 4096 16-bit
// elements), in a workgroup's up to 4 times that; rows of at most 8 chunks share a wave.
#define ROW_SHAPES(X)                       \
    if (chunks <= 8) X(8, 1)                \
    else if (chunks <= 64) X(64, 1)         \
    else if (chunks <= 128) X(64, 2)        \
    else if (chunks <= 256) X(64, 4)        \
    else if (chunks <= 512) X(64, 8)        \
    else if (chunks <= 1024) X(256, 4)      \
    else if (chunks <= 2048) X(256, 8)

template <typename T, bool FULL>
int policy_launch(hipStream_t s, const PolicyArgs &a) {
    const int chunks = bt_div_up(a.d.width, Row<T>::V);
#define POLICY_CASE(G, K) \
    BT_LAUNCH(BTK_POLICY, s, (policy_rows<T, G, K, FULL>), row_grid(bt_div_up(a.d.batch, 256 / G)), dim3(256), 0, a);
    ROW_SHAPES(POLICY_CASE)
    else BT_LAUNCH(BTK_POLICY, s, (policy_rows_long<T, FULL>), row_grid(a.d.batch), dim3(256), 0, a);
#undef POLICY_CASE
    BT_LAUNCH_CHECK();
    return BT_OK;
}
template <typename T>
int policy_launch(hipStream_t s, const PolicyArgs &a) {
    return a.d.kl == BT_KL_FULL ? policy_launch<T, true>(s, a) : policy_launch<T, false>(s, a);
}

template <typename T>
int pref_launch(hipStream_t s, const PrefArgs &a) {
    const int chunks = bt_div_up(a.d.width, Row<T>::V);
    if (a.d.rows > 0) {
#define PREF_CASE(G, K) BT_LAUNCH(BTK_POLICY, s, (pref_rows<T, G, K>), row_grid(bt_div_up(a.d.rows, 256 / G)), dim3(256), 0, a);
        ROW_SHAPES(PREF_CASE)
        else BT_LAUNCH(BTK_POLICY, s, (pref_rows<T, 256, 0>), row_grid(a.d.rows), dim3(256), 0, a);
#undef PREF_CASE
        BT_LAUNCH_CHECK();
    }
    BT_LAUNCH(BTK_POLICY, s, pref_pairs, row_grid(bt_div_up(a.d.pairs, 4)), dim3(256), 0, a);
    BT_LAUNCH_CHECK();
    if (a.grad && a.d.rows > 0) {
#define GRAD_CASE(G, K) BT_LAUNCH(BTK_POLICY, s, (pref_grad<T, G, K>), row_grid(1 + (long long)bt_div_up(a.d.rows, 256 / G)), dim3(256), 0, a);
        ROW_SHAPES(GRAD_CASE)
        else BT_LAUNCH(BTK_POLICY, s, (pref_grad<T, 256, 0>), row_grid(1 + (long long)a.d.rows), dim3(256), 0, a);
#undef GRAD_CASE
    } else {
        BT_LAUNCH(BTK_POLICY, s, loss_sum_kernel, dim3(1), dim3(1024), 0, a.pair_loss, a.d.pairs, a.loss_sum);
    }
    BT_LAUNCH_CHECK();
    return BT_OK;
}

int pref_validate(const bt_preference_desc *d, const char *fn, bool mask) {
    BT_REQUIRE(d, "%s: null pointer", fn);
    BT_REQUIRE(d->pairs > 0 && d->pairs <= (1 << 29), "%s: Mismatched sizes! (pairs = %d)", fn, d->pairs);
    BT_REQUIRE(d->rows >= 0, "%s: Mismatched sizes! (rows < 0)", fn);
    if (int rc = matrix_validate(fn, d->type, d->width, d->ld, d->mask_ld, mask)) return rc;
    BT_REQUIRE(d->beta >= 0.0f && d->beta <= 3.0e38f, "%s: beta = %g must not be negative", fn, d->beta);
    BT_REQUIRE(d->smoothing >= 0.0f && d->smoothing < 0.5f, "%s: smoothing = %g is outside [0, 0.5)", fn, d->smoothing);
    return BT_OK;
}

}  // namespace

extern "C" {

int bt_policy_loss(void *stream, const bt_policy_desc *d, const void *logits, const uint8_t *mask, const int32_t *actions,
                   const float *old_logp, const float *advantages, const void *ref, const float *row_weights,
                   float *loss_sum, void *grad, float *row_loss, float *row_logp, float *row_kl) {
    BT_REQUIRE(d, "bt_policy_loss: null pointer");
    BT_REQUIRE(d->batch > 0, "bt_policy_loss: Mismatched sizes! (batch <= 0)");
    if (int rc = matrix_validate("bt_policy_loss", d->type, d->width, d->ld, d->mask_ld, mask)) return rc;
    BT_REQUIRE(d->kl == BT_KL_NONE || d->kl == BT_KL_TAKEN || d->kl == BT_KL_FULL, "bt_policy_loss: unknown KL kind %d", d->kl);
    BT_REQUIRE(d->clip_low >= 0.0f && d->clip_low <= 1.0f && d->clip_high >= 0.0f && d->clip_high <= 3.0e38f,
               "bt_policy_loss: clipping range (%g, %g) is not one", d->clip_low, d->clip_high);
    BT_REQUIRE(d->kl_weight >= 0.0f && d->kl_weight <= 3.0e38f, "bt_policy_loss: kl_weight = %g must not be negative",
               d->kl_weight);
    BT_REQUIRE(logits && actions && old_logp && advantages && loss_sum && row_loss, "bt_policy_loss: null pointer");
    BT_REQUIRE(d->kl == BT_KL_NONE || ref, "bt_policy_loss: this KL term needs the reference policy");
    const size_t es = type_size(d->type);
    BT_REQUIRE(aligned(logits, es) && aligned(grad, es) && (d->kl == BT_KL_NONE || aligned(ref, d->kl == BT_KL_FULL ? es : 4)),
               "bt_policy_loss: a buffer is not aligned to its element type");
    BT_REQUIRE(d->kl != BT_KL_FULL || ref != grad || !grad, "bt_policy_loss: grad must not be the reference logits");
    PolicyArgs a{logits, ref, mask, actions, old_logp, advantages, row_weights, grad, row_loss, row_logp, row_kl, *d};
    hipStream_t s = bt_stream(stream);
    if (int rc = d->type == BT_TYPE_F32    ? policy_launch<float>(s, a)
                 : d->type == BT_TYPE_BF16 ? policy_launch<__bf16>(s, a)
                                           : policy_launch<_Float16>(s, a))
        return rc;
    BT_LAUNCH(BTK_POLICY, s, loss_sum_kernel, dim3(1), dim3(1024), 0, row_loss, d->batch, loss_sum);
    BT_LAUNCH_CHECK();
    return BT_OK;
}

size_t bt_preference_loss_workspace_bytes(const bt_preference_desc *d) {
    if (pref_validate(d, "bt_preference_loss_workspace_bytes", false)) return 0;
    return 5 * bt_align((size_t)d->rows * 4) + 256;
}

int bt_preference_loss(void *stream, const bt_preference_desc *d, const void *logits, const uint8_t *mask,
                       const int32_t *actions, const int32_t *offsets, const float *ref_logp, const float *pair_weights,
                       float *loss_sum, void *grad, float *pair_loss, float *line_logp, void *workspace,
                       size_t workspace_bytes) {
    if (int rc = pref_validate(d, "bt_preference_loss", mask)) return rc;
    BT_REQUIRE(offsets && ref_logp && loss_sum && pair_loss && workspace, "bt_preference_loss: null pointer");
    BT_REQUIRE(d->rows == 0 || (logits && actions), "bt_preference_loss: null pointer");
    BT_REQUIRE(workspace_bytes >= bt_preference_loss_workspace_bytes(d), "bt_preference_loss: workspace too small");
    BT_REQUIRE(aligned(workspace, 4), "bt_preference_loss: workspace is not aligned to 4 bytes");
    const size_t es = type_size(d->type);
    BT_REQUIRE(aligned(logits, es) && aligned(grad, es), "bt_preference_loss: a buffer is not aligned to its element type");
    const size_t per_row = bt_align((size_t)d->rows * 4) / sizeof(float);
    float *ws = static_cast<float *>(workspace);
    PrefArgs a{logits, mask, actions, offsets, ref_logp, pair_weights, grad, pair_loss, line_logp, loss_sum, ws, ws + per_row,
               ws + 2 * per_row, ws + 3 * per_row, ws + 4 * per_row, *d};
    hipStream_t s = bt_stream(stream);
    if (int rc = d->type == BT_TYPE_F32    ? pref_launch<float>(s, a)
                 : d->type == BT_TYPE_BF16 ? pref_launch<__bf16>(s, a)
                                           : pref_launch<_Float16>(s, a))
        return rc;
    return BT_OK;
}

}  // extern "C"
