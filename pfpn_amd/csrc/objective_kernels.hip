// Objectives of a policy beside its clipped loss: the loss over preferred pairs of segments (paired log ratios) and the
// balance loss over the choices of categorical weights with their counts.  Forward and backward.
#include "objective_common.h"

#include <cstddef>

namespace pfpn {

// =====================================================================================================================
// Preference loss.  Segment s = rows [offsets[s], offsets[s + 1]) of the [T] log-probs; pair p compares segment 2p (preferred)
// with 2p + 1:  S_s = sum_t w_t (logp_t - logp_ref_t),  delta = S_2p - S_2p+1,  margin = beta delta,
//   logistic:  -(1 - e) log sigma(margin) - e log sigma(-margin)      squared:  (delta - 1 / (2 beta))^2
// mean over the pairs;  dlogp_t = +-(d loss / d delta) w_t.  Segment sums in 64 bits: thousands of terms, and their difference.
// =====================================================================================================================
struct PrefArgs {
    const float* logp;
    const float* logp_ref;      // optional
    const float* weight;        // optional
    const long long* offsets;   // [2P + 1]
    int P;
    long long T;
    double beta, smoothing;
    int kind;                   // 0 logistic, 1 squared
    float* dlogp;
    float* margin;
    double* sums;               // [2P][splits]
    double* terms;              // [P][3] = loss, margin > 0, margin
    int splits;
};

__device__ __forceinline__ void segment_of(const PrefArgs& p, int s, long long& lo, long long& hi) {
    lo = p.offsets[s];
    hi = p.offsets[s + 1];
    lo = lo < 0 ? 0 : (lo > p.T ? p.T : lo);
    hi = hi < lo ? lo : (hi > p.T ? p.T : hi);
}
__device__ __forceinline__ void slice_of(const PrefArgs& p, int s, int part, long long& lo, long long& hi) {
    long long a, b;
    segment_of(p, s, a, b);
    const long long width = (b - a + p.splits - 1) / p.splits;
    lo = a + part * width < b ? a + part * width : b;
    hi = lo + width < b ? lo + width : b;
}
// a step of weight 0 is not read any further: what stands there does not matter
__device__ __forceinline__ double step_gap(const PrefArgs& p, long long t) {
    const float w = p.weight ? p.weight[t] : 1.f;
    if (w == 0.f) return 0.0;
    const double d = (double)p.logp[t] - (p.logp_ref ? (double)p.logp_ref[t] : 0.0);
    return p.weight ? d * (double)w : d;
}

// loss of one pair -> d loss / d delta (of the mean); fills terms and margin when `write`
__device__ __forceinline__ double pair_head(const PrefArgs& p, int pair, double delta, bool write) {
    const double m = p.beta * delta;
    double loss, slope;
    if (p.kind == 0) {
        // log sigma(m) = -softplus(-m); both halves from ONE exponential of -|m|
        const double z = exp(-fabs(m)), l = log1p(z);
        const double good = m >= 0 ? 1.0 / (1.0 + z) : z / (1.0 + z), bad = m >= 0 ? z / (1.0 + z) : 1.0 / (1.0 + z);
        const double sp_neg = l + (m < 0 ? -m : 0.0), sp_pos = l + (m > 0 ? m : 0.0);
        loss = (1.0 - p.smoothing) * sp_neg + p.smoothing * sp_pos;
        slope = p.beta * (p.smoothing * good - (1.0 - p.smoothing) * bad);
    } else {
        const double u = delta - 0.5 / p.beta;
        loss = u * u;
        slope = 2.0 * u;
    }
    if (write) {
        p.margin[pair] = (float)m;
        p.terms[(size_t)pair * 3] = loss;
        p.terms[(size_t)pair * 3 + 1] = m > 0 ? 1.0 : 0.0;
        p.terms[(size_t)pair * 3 + 2] = m;
    }
    return slope / (double)p.P;
}

__global__ __launch_bounds__(256) void k_pref_sums(PrefArgs p) {
    __shared__ double red[4];
    const int s = blockIdx.x / p.splits, part = blockIdx.x % p.splits;
    long long lo, hi;
    slice_of(p, s, part, lo, hi);
    double v = 0.0;
    for (long long t = lo + threadIdx.x; t < hi; t += 256) v += step_gap(p, t);
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) p.sums[blockIdx.x] = ((red[0] + red[1]) + red[2]) + red[3];
}

__global__ __launch_bounds__(256) void k_pref_grad(PrefArgs p) {
    const long long blocks = 2ll * p.P * p.splits;
    if (blockIdx.x >= blocks) {
        // rows outside every segment have no gradient
        const long long first = p.offsets[0] < 0 ? 0 : p.offsets[0], last = p.offsets[2 * (size_t)p.P];
        const long long at = (blockIdx.x - blocks) * 256 + threadIdx.x, step = (gridDim.x - blocks) * 256;
        for (long long t = at; t < first && t < p.T; t += step) p.dlogp[t] = 0.f;
        for (long long t = (last < 0 ? 0 : last) + at; t < p.T; t += step) p.dlogp[t] = 0.f;
        return;
    }
    const int s = blockIdx.x / p.splits, part = blockIdx.x % p.splits, pair = s >> 1;
    const double* sums = p.sums + (size_t)pair * 2 * p.splits;
    double a = 0.0, b = 0.0;
    for (int i = 0; i < p.splits; ++i) { a += sums[i]; b += sums[p.splits + i]; }
    double g = pair_head(p, pair, a - b, threadIdx.x == 0 && part == 0 && (s & 1) == 0);
    if (s & 1) g = -g;
    long long lo, hi;
    slice_of(p, s, part, lo, hi);
    const float gf = (float)g;
    for (long long t = lo + threadIdx.x; t < hi; t += 256) {
        const float w = p.weight ? p.weight[t] : 1.f;
        p.dlogp[t] = p.weight ? (w == 0.f ? 0.f : (float)(g * (double)w)) : gf;
    }
}

__global__ __launch_bounds__(1024) void k_pref_finish(const double* __restrict__ terms, int P, float* __restrict__ loss3) {
    __shared__ double red[3 * 16];
    __shared__ double out[3];
    HeadTerms t = {0.0, 0.0, 0.0};
    for (int i = threadIdx.x; i < P; i += 1024) {
        t.policy += terms[(size_t)i * 3];
        t.kl += terms[(size_t)i * 3 + 1];
        t.clipped += terms[(size_t)i * 3 + 2];
    }
    block_terms(t, red, out);
    __syncthreads();
    if (threadIdx.x < 3) loss3[threadIdx.x] = (float)(out[threadIdx.x] / (double)P);
}

// =====================================================================================================================
// Balance loss.  p = softmax(l[b, a, :]); a row counts for its K largest logits (equal ones: the lowest index first; a
// closed choice, logit -inf, never).  Over the V rows the mask leaves:
//   counts[a, n],  f = counts / (K V),  P = sum_b p / V,  loss = coef N / A sum_a sum_n f P,
//   d l[b, a, n] = coef N / (A V) p_n (f_n - sum_m f_m p_m)         (f is a count: no gradient through it)
// k_bal_stats leaves sums and counts of every chunk of rows as slabs, k_bal_reduce adds the slabs (64 bits, in order), k_bal_grad
// writes the gradient.  A group of G lanes keeps ONE choice a while it walks rows: its sums, and f, stay in registers.
// =====================================================================================================================
struct BalArgs {
    const void* logits;
    long long ld;
    const unsigned char* mask;      // optional [R]
    int R, A, N, K;
    double scale;                   // coef N / A
    int accumulate;
    float* loss;
    int* counts;
    float* mean_prob;
    void* dlogits;
    long long ldd;
    int AT, RR, tiles, chunks;      // choices and rows side by side in a block; blocks = tiles * chunks
    float* slab_p;                  // [chunks][A N]
    uint32_t* slab_n;               // [chunks][A N]
    uint32_t* slab_v;               // [chunks] valid rows
    float* f;                       // [A N] coef N / (A V) f
    double* terms;                  // [blocks of k_bal_reduce]
};
constexpr int BAL_NT = 512;

template <typename T, int G, int E>
__device__ __forceinline__ void load_segment(const BalArgs& p, bool on, size_t b, int a, int j, float (&x)[E]) {
    const T* l = static_cast<const T*>(p.logits) + b * p.ld + (size_t)a * p.N;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int n = j + G * e;
        x[e] = (on && n < p.N) ? to_f32(l[n]) : -INFINITY;
    }
}

template <typename T, int G, int E>
__global__ __launch_bounds__(BAL_NT) void k_bal_stats(BalArgs p) {
    extern __shared__ char lds_raw[];
    const int tile = blockIdx.x % p.tiles, chunk = blockIdx.x / p.tiles;
    const int j = threadIdx.x % G, gid = threadIdx.x / G;
    const int a0 = tile * p.AT, al = gid % p.AT, rr = gid / p.AT, a = a0 + al;
    const bool mine = rr < p.RR && a < p.A;
    const int per = (p.R + p.chunks - 1) / p.chunks;
    const long long r0 = (long long)chunk * per;
    const long long r1 = r0 + per < p.R ? r0 + per : p.R;
    float* sums = reinterpret_cast<float*>(lds_raw);                            // [RR][AT N]
    uint32_t* cnts = reinterpret_cast<uint32_t*>(sums + (size_t)p.RR * p.AT * p.N);    // [AT N]
    for (int i = threadIdx.x; i < p.AT * p.N; i += blockDim.x) cnts[i] = 0;
    float acc[E];
    uint32_t cnt[E];
#pragma unroll
    for (int e = 0; e < E; ++e) { acc[e] = 0.f; cnt[e] = 0; }
    uint32_t valid = 0;
    for (long long rb = r0; rb < r1; rb += p.RR) {
        const long long b = rb + rr;
        const bool row = mine && b < r1 && (!p.mask || p.mask[b]);
        float x[E];
        load_segment<T, G, E>(p, row, (size_t)b, a, j, x);
        valid += row;
        float m = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) m = fmaxf(m, x[e]);
        m = group_max<G>(m);
        const float ms = m == -INFINITY ? 0.f : m;
        float ex[E], s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) { ex[e] = exp_below(x[e], ms); s += ex[e]; }
        s = group_sum<G>(s);
        const float inv = s == 0.f ? 0.f : 1.f / s;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += ex[e] * inv;
        for (int k = 0; k < p.K; ++k) {
            if (k) {
                m = -INFINITY;
#pragma unroll
                for (int e = 0; e < E; ++e) m = fmaxf(m, x[e]);
                m = group_max<G>(m);
            }
            uint32_t at = 0xffffffffu;
#pragma unroll
            for (int e = E - 1; e >= 0; --e)
                if (x[e] == m) at = j + G * e;
            at = group_min<G>(at);
            if (m > -INFINITY) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (at == (uint32_t)(j + G * e)) { cnt[e] += 1; x[e] = -INFINITY; }
            }
        }
    }
    __syncthreads();
    if (mine) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int n = j + G * e;
            if (n < p.N) {
                sums[((size_t)rr * p.AT + al) * p.N + n] = acc[e];
                if (cnt[e]) atomicAdd(&cnts[al * p.N + n], cnt[e]);
            }
        }
    }
    __syncthreads();
    const size_t AN = (size_t)p.A * p.N;
    const int cols = (p.A - a0 < p.AT ? p.A - a0 : p.AT) * p.N;
    for (int i = threadIdx.x; i < cols; i += blockDim.x) {
        float s = 0.f;
        for (int q = 0; q < p.RR; ++q) s += sums[(size_t)q * p.AT * p.N + i];
        p.slab_p[(size_t)chunk * AN + (size_t)a0 * p.N + i] = s;
        p.slab_n[(size_t)chunk * AN + (size_t)a0 * p.N + i] = cnts[i];
    }
    if (tile == 0) {
        __syncthreads();
        if (threadIdx.x == 0) cnts[0] = 0;
        __syncthreads();
        if (al == 0 && j == 0 && valid) atomicAdd(&cnts[0], valid);
        __syncthreads();
        if (threadIdx.x == 0) p.slab_v[chunk] = cnts[0];
    }
}

// 64 columns x 16 lanes over the slabs
__global__ __launch_bounds__(1024) void k_bal_reduce(BalArgs p) {
    __shared__ double rs[16][64];
    __shared__ uint32_t rn[16][64];
    __shared__ uint32_t v_all;
    const size_t AN = (size_t)p.A * p.N;
    const int cl = threadIdx.x & 63, kl = threadIdx.x >> 6;
    const size_t col = (size_t)blockIdx.x * 64 + cl;
    if (threadIdx.x == 0) v_all = 0;
    __syncthreads();
    uint32_t v = 0;
    for (int k = threadIdx.x; k < p.chunks; k += 1024) v += p.slab_v[k];
    if (v) atomicAdd(&v_all, v);
    double s = 0.0;
    uint32_t n = 0;
    if (col < AN)
        for (int k = kl; k < p.chunks; k += 16) {
            s += (double)p.slab_p[(size_t)k * AN + col];
            n += p.slab_n[(size_t)k * AN + col];
        }
    rs[kl][cl] = s;
    rn[kl][cl] = n;
    __syncthreads();
    if (kl == 0) {
        for (int i = 1; i < 16; ++i) { s += rs[i][cl]; n += rn[i][cl]; }
        const double inv_v = v_all ? 1.0 / (double)v_all : 0.0;
        const double mean = s * inv_v, share = (double)n * inv_v / p.K;
        double term = 0.0;
        if (col < AN) {
            p.mean_prob[col] = (float)mean;
            p.counts[col] = (int)n;
            p.f[col] = (float)(p.scale * inv_v * share);
            term = share * mean;
        }
        term = wave_sum(term);
        if (cl == 0) p.terms[blockIdx.x] = term;
    }
}

template <typename T, int G, int E>
__global__ __launch_bounds__(BAL_NT) void k_bal_grad(BalArgs p) {
    const int tile = blockIdx.x % p.tiles, chunk = blockIdx.x / p.tiles;
    const int j = threadIdx.x % G, gid = threadIdx.x / G;
    const int al = gid % p.AT, rr = gid / p.AT, a = tile * p.AT + al;
    const bool mine = rr < p.RR && a < p.A;
    const int per = (p.R + p.chunks - 1) / p.chunks;
    const long long r0 = (long long)chunk * per;
    const long long r1 = r0 + per < p.R ? r0 + per : p.R;
    float f[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int n = j + G * e;
        f[e] = (mine && n < p.N) ? p.f[(size_t)a * p.N + n] : 0.f;
    }
    for (long long rb = r0; rb < r1; rb += p.RR) {
        const long long b = rb + rr;
        const bool have = mine && b < r1;
        const bool row = have && (!p.mask || p.mask[b]);
        float x[E];
        load_segment<T, G, E>(p, row, (size_t)b, a, j, x);
        float m = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) m = fmaxf(m, x[e]);
        m = group_max<G>(m);
        if (m == -INFINITY) m = 0.f;
        float s = 0.f, d = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) { x[e] = exp_below(x[e], m); s += x[e]; d += x[e] * f[e]; }
        s = group_sum<G>(s);
        d = group_sum<G>(d);
        const float inv = s == 0.f ? 0.f : 1.f / s;
        d *= inv;
        if (have) {
            T* o = static_cast<T*>(p.dlogits) + (size_t)b * p.ldd + (size_t)a * p.N;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int n = j + G * e;
                if (n < p.N) {
                    float v = row ? x[e] * inv * (f[e] - d) : 0.f;
                    if (p.accumulate) v += to_f32(o[n]);
                    if (row || !p.accumulate) o[n] = from_f32<T>(v);
                }
            }
        }
    }
    if (blockIdx.x == 0) {
        __shared__ double red[BAL_NT / 64];
        const size_t parts = ((size_t)p.A * p.N + 63) / 64;
        double t = 0.0;
        for (size_t i = threadIdx.x; i < parts; i += blockDim.x) t += p.terms[i];
        t = wave_sum(t);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = t;
        __syncthreads();
        if (threadIdx.x == 0) {
            t = 0.0;
            for (unsigned i = 0; i < (blockDim.x + 63) / 64; ++i) t += red[i];
            p.loss[0] = (float)(p.scale * t);
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
constexpr int BAL_MAX_N = 1024, BAL_MAX_K = 64, BAL_MAX_A = 4096;

static int group_width(int N) { return N <= 40 ? 8 : N <= 96 ? 16 : N <= 192 ? 32 : 64; }

static void bal_shape(BalArgs& p) {
    const int G = group_width(p.N), groups = BAL_NT / G;
    p.AT = p.A < groups ? p.A : groups;
    while (p.AT > 1 && p.AT * p.N > 4096) p.AT = (p.AT + 1) / 2;
    p.RR = groups / p.AT;
    p.tiles = (p.A + p.AT - 1) / p.AT;
    int c = (1024 + p.tiles - 1) / p.tiles;
    const int most = (p.R + p.RR - 1) / p.RR;       // a row or more for every group
    if (c > most) c = most;
    if (c < 1) c = 1;
    p.chunks = c;
}
static size_t bal_bytes(const BalArgs& p) {
    const size_t AN = (size_t)p.A * p.N;
    return ((AN + 63) / 64) * sizeof(double) + (size_t)p.chunks * AN * 8 + (size_t)p.chunks * 4 + AN * 4;
}

template <typename T, int G, int E>
static void launch_bal(const BalArgs& p, hipStream_t st) {
    const int threads = (p.AT * p.RR * G + 63) / 64 * 64;
    const size_t lds = ((size_t)p.RR + 1) * p.AT * p.N * 4;
    const size_t AN = (size_t)p.A * p.N;
    hipLaunchKernelGGL((k_bal_stats<T, G, E>), dim3(p.tiles * p.chunks), dim3(threads), lds, st, p);
    hipLaunchKernelGGL(k_bal_reduce, dim3((unsigned)((AN + 63) / 64)), dim3(1024), 0, st, p);
    hipLaunchKernelGGL((k_bal_grad<T, G, E>), dim3(p.tiles * p.chunks), dim3(threads), 0, st, p);
}
template <typename T>
static void pick_bal(const BalArgs& p, hipStream_t st) {
    const int N = p.N;
    if (N <= 8) launch_bal<T, 8, 1>(p, st);
    else if (N <= 16) launch_bal<T, 8, 2>(p, st);
    else if (N <= 24) launch_bal<T, 8, 3>(p, st);
    else if (N <= 32) launch_bal<T, 8, 4>(p, st);
    else if (N <= 40) launch_bal<T, 8, 5>(p, st);
    else if (N <= 64) launch_bal<T, 16, 4>(p, st);
    else if (N <= 96) launch_bal<T, 16, 6>(p, st);
    else if (N <= 128) launch_bal<T, 32, 4>(p, st);
    else if (N <= 192) launch_bal<T, 32, 6>(p, st);
    else if (N <= 256) launch_bal<T, 64, 4>(p, st);
    else if (N <= 512) launch_bal<T, 64, 8>(p, st);
    else launch_bal<T, 64, 16>(p, st);
}

static void pref_shape(PrefArgs& p) {
    // pieces of a segment: about 4096 steps of the average one, and no more blocks than fill the chip a few times
    const long long avg = p.T / (2ll * p.P);
    long long s = (avg + 4095) / 4096;
    const long long most = (8192 + 2ll * p.P - 1) / (2ll * p.P);
    if (s > most) s = most;
    p.splits = (int)(s < 1 ? 1 : s);
}

}  // namespace pfpn

using namespace pfpn;

extern "C" {

size_t pfpn_preference_workspace_bytes(int P, long long T) {
    if (P < 1 || T < 0) return 0;
    PrefArgs p = {};
    p.P = P; p.T = T;
    pref_shape(p);
    return ((size_t)P * 3 + 2 * (size_t)P * p.splits) * sizeof(double);
}

int pfpn_preference_loss(const float* logp, const float* logp_ref, const float* weight, const int64_t* offsets, int P,
                         long long T, double beta, double label_smoothing, int kind, float* dlogp, float* margin,
                         float* loss3, void* workspace, size_t workspace_bytes, void* stream) {
    PFPN_BEGIN();
    if (!offsets || !margin || !loss3 || P < 1 || P > (1 << 22) || T < 0 || (T > 0 && (!logp || !dlogp)) || !(beta > 0.0) ||
        !(label_smoothing >= 0.0 && label_smoothing <= 0.5) || kind < 0 || kind > 1)
        return PFPN_ERR_ARG;
    if (!workspace || workspace_bytes < pfpn_preference_workspace_bytes(P, T)) return PFPN_ERR_WORKSPACE;
    PrefArgs p = {};
    p.logp = logp; p.logp_ref = logp_ref; p.weight = weight; p.offsets = reinterpret_cast<const long long*>(offsets);
    p.P = P; p.T = T; p.beta = beta; p.smoothing = label_smoothing; p.kind = kind; p.dlogp = dlogp; p.margin = margin;
    pref_shape(p);
    p.terms = static_cast<double*>(workspace);
    p.sums = p.terms + (size_t)P * 3;
    hipStream_t st = (hipStream_t)stream;
    const unsigned blocks = 2u * (unsigned)P * (unsigned)p.splits;
    const unsigned outside = (unsigned)(T / 4096 + 1 < 64 ? T / 4096 + 1 : 64);
    hipLaunchKernelGGL(k_pref_sums, dim3(blocks), dim3(256), 0, st, p);
    hipLaunchKernelGGL(k_pref_grad, dim3(blocks + outside), dim3(256), 0, st, p);
    hipLaunchKernelGGL(k_pref_finish, dim3(1), dim3(1024), 0, st, (const double*)p.terms, P, loss3);
    PFPN_CHECK_LAUNCH();
    return PFPN_OK;
}

size_t pfpn_balance_workspace_bytes(int R, int A, int N) {
    if (R < 1 || A < 1 || N < 1 || N > BAL_MAX_N || A > BAL_MAX_A) return 0;
    BalArgs p = {};
    p.R = R; p.A = A; p.N = N;
    bal_shape(p);
    return bal_bytes(p);
}

int pfpn_balance_loss(const void* logits, int dtype, long long row_stride, const uint8_t* mask, int R, int A, int N, int topk,
                      double coef, int accumulate, float* loss, int32_t* counts, float* mean_prob, void* dlogits,
                      long long grad_stride, void* workspace, size_t workspace_bytes, void* stream) {
    PFPN_BEGIN();
    if (!logits || dtype < DT_F32 || dtype > DT_F16 || R < 1 || R > (1 << 30) || A < 1 || N < 1 || N > BAL_MAX_N || A > BAL_MAX_A || topk < 1 ||
        topk > N || topk > BAL_MAX_K || row_stride < (long long)A * N || grad_stride < (long long)A * N || !loss || !counts ||
        !mean_prob || !dlogits)
        return PFPN_ERR_ARG;
    BalArgs p = {};
    p.logits = logits; p.ld = row_stride; p.mask = mask; p.R = R; p.A = A; p.N = N; p.K = topk;
    p.scale = coef * (double)N / (double)A;
    p.accumulate = accumulate; p.loss = loss; p.counts = counts; p.mean_prob = mean_prob;
    p.dlogits = dlogits; p.ldd = grad_stride;
    bal_shape(p);
    if (!workspace || workspace_bytes < bal_bytes(p)) return PFPN_ERR_WORKSPACE;
    const size_t AN = (size_t)A * N;
    p.terms = static_cast<double*>(workspace);
    p.slab_p = reinterpret_cast<float*>(p.terms + (AN + 63) / 64);
    p.slab_n = reinterpret_cast<uint32_t*>(p.slab_p + (size_t)p.chunks * AN);
    p.slab_v = p.slab_n + (size_t)p.chunks * AN;
    p.f = reinterpret_cast<float*>(p.slab_v + p.chunks);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == DT_F32) pick_bal<float>(p, st);
    else if (dtype == DT_BF16) pick_bal<bf16_t>(p, st);
    else pick_bal<f16_t>(p, st);
    PFPN_CHECK_LAUNCH();
    return PFPN_OK;
}

}  // extern "C"
