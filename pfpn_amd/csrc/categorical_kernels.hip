// Log-probabilities of chosen categories and the clipped policy loss with a KL term, straight from categorical logits
// [B, A, N] (A choices of N categories make one joint action; A = 1: a token row), forward and backward.
//
//   logp[b]       = sum_a (l[b,a,k] - m[b,a] - log s[b,a]),   m = max_n l, s = sum_n exp(l - m)
//   d logits      = dlogp[b] (1[n = k] - exp(l - m) / s)
//
// (the particle index a policy drew: reference networks/utils.py:187-194; the clipped surrogate: networks/actor_critic/ppo.py:44-54)
#include "objective_common.h"

#include <cstddef>

namespace pfpn {

enum { CAT_FWD = 0, CAT_BWD = 1, CAT_PPO = 2 };

struct CatArgs {
    const void* logits;
    long long ld;               // elements from one row of logits to the next
    const void* index;
    int index64;
    int B, A, N;
    const float* dlogp;         // CAT_BWD
    HeadArgs head;              // CAT_PPO
    float* logp;
    void* dlogits;
    long long ldd;
    int accumulate;             // CAT_BWD: dlogits += instead of =
    int rows_per_block;
    uint32_t magic_A;           // ceil(2^32 / A) (A > 1)
    double* part;               // CAT_PPO: three sums per block
};

__device__ __forceinline__ long long chosen(const CatArgs& p, size_t i) {
    return p.index64 ? static_cast<const long long*>(p.index)[i] : (long long)static_cast<const int*>(p.index)[i];
}
__device__ __forceinline__ int div_A(const CatArgs& p, int q) {
    return p.A == 1 ? q : (int)__umulhi((uint32_t)q, p.magic_A);
}
__device__ __forceinline__ double row_weight(const CatArgs& p, size_t b) {
    return p.head.weight ? (double)p.head.weight[b] : p.head.inv_B;
}

// ---------------------------------------------------------------------------------------------------------------------
// Short axes (N <= 1024): a group of G lanes owns a segment (row, choice), a lane E of its logits.  A block owns
// rows_per_block whole rows, so the joint log-prob of a row and with it the upstream gradient are known inside the block:
// the loss needs ONE launch.  Phase 1: {l_k, m, s} of every segment into LDS; phase 2: the rows' log-probs and loss heads
// (64 bits); phase 3: the gradients, from the logits again (they are in the caches).
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int MODE, int G, int E>
__global__ __launch_bounds__(512) void k_cat_rows(CatArgs p) {
    constexpr int NT = 512, NG = NT / G;
    extern __shared__ char lds_raw[];
    const int tid = threadIdx.x, j = tid % G, gid = tid / G;
    const int RB = p.rows_per_block;
    const size_t row0 = (size_t)blockIdx.x * RB;
    const int rows = (int)((size_t)p.B - row0 < (size_t)RB ? (size_t)p.B - row0 : (size_t)RB);
    const int nseg = rows * p.A;
    float* seg = reinterpret_cast<float*>(lds_raw + 48 * sizeof(double));      // [RB * A][3] = l_k, m, s
    float* row_g = seg + (size_t)RB * p.A * 3;                                  // [RB]
    const T* logits = static_cast<const T*>(p.logits);
    T* dlogits = static_cast<T*>(p.dlogits);

    if (MODE != CAT_BWD) {
        for (int q0 = 0; q0 < nseg; q0 += NG) {
            const int q = q0 + gid;
            float x[E];
            const int r = q < nseg ? div_A(p, q) : 0, a = q < nseg ? q - r * p.A : 0;
            const size_t b = row0 + r;
            bool on = q < nseg;
            if (MODE == CAT_PPO && on && row_weight(p, b) == 0.0) on = false;
            const T* l = logits + b * p.ld + (size_t)a * p.N;
            float m = -INFINITY;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int n = j + G * e;
                x[e] = (on && n < p.N) ? to_f32(l[n]) : -INFINITY;
                m = fmaxf(m, x[e]);
            }
            m = group_max<G>(m);
            if (m == -INFINITY) m = 0.f;
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) s += exp_below(x[e], m);
            s = group_sum<G>(s);
            if (on && j == 0) {
                const long long k = chosen(p, b * p.A + a);
                const bool in = k >= 0 && k < p.N;          // (another index: this choice does not enter the row)
                seg[q * 3] = in ? to_f32(l[k]) : 0.f;
                seg[q * 3 + 1] = in ? m : 0.f;
                seg[q * 3 + 2] = in ? s : 1.f;
            }
        }
        __syncthreads();
        HeadTerms t = {0.0, 0.0, 0.0};
        // a wave per row, lanes over its choices
        const int lane = tid & 63;
        for (int r = tid >> 6; r < rows; r += NT / 64) {
            const size_t b = row0 + r;
            const double w = MODE == CAT_PPO ? row_weight(p, b) : 1.0;
            double lp = 0.0;
            if (w != 0.0) {
                for (int a = lane; a < p.A; a += 64) {
                    const float* v = seg + (size_t)(r * p.A + a) * 3;
                    lp += v[2] == 0.f ? (double)-INFINITY : (double)v[0] - (double)v[1] - log((double)v[2]);
                }
            }
            lp = wave_sum(lp);
            if (lane == 0) {
                p.logp[b] = (float)lp;
                if (MODE == CAT_PPO) row_g[r] = w != 0.0 ? (float)policy_head(lp, b, w, p.head, t) : 0.f;
            }
        }
        if (MODE == CAT_FWD) return;
        block_terms(t, reinterpret_cast<double*>(lds_raw), p.part + (size_t)blockIdx.x * 3);
        __syncthreads();
    }
    for (int q0 = 0; q0 < nseg; q0 += NG) {
        const int q = q0 + gid;
        float x[E];
        const int r = q < nseg ? div_A(p, q) : 0, a = q < nseg ? q - r * p.A : 0;
        const size_t b = row0 + r;
        const bool have = q < nseg;
        const float g = !have ? 0.f : (MODE == CAT_PPO ? row_g[r] : p.dlogp[b]);
        const bool on = have && (MODE == CAT_PPO ? row_weight(p, b) != 0.0 : g != 0.f);
        const T* l = logits + b * p.ld + (size_t)a * p.N;
        float m, s;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int n = j + G * e;
            x[e] = (on && n < p.N) ? to_f32(l[n]) : -INFINITY;
        }
        const long long k = have ? chosen(p, b * p.A + a) : -1;
        const bool in = k >= 0 && k < p.N;
        if (MODE == CAT_PPO) {
            m = on ? seg[q * 3 + 1] : 0.f;
            s = on ? seg[q * 3 + 2] : 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = exp_below(x[e], m);
        } else {
            m = -INFINITY;
#pragma unroll
            for (int e = 0; e < E; ++e) m = fmaxf(m, x[e]);
            m = group_max<G>(m);
            if (m == -INFINITY) m = 0.f;
            s = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) { x[e] = exp_below(x[e], m); s += x[e]; }
            s = group_sum<G>(s);
        }
        // a segment with no open choice (s = 0), an index outside the axis and a row without weight get zeros
        const bool live = on && in && s != 0.f;
        const float inv = live ? 1.f / s : 0.f;
        if (have) {
            T* d = dlogits + b * p.ldd + (size_t)a * p.N;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int n = j + G * e;
                if (n < p.N) {
                    float v = live ? g * ((n == (int)k ? 1.f : 0.f) - x[e] * inv) : 0.f;
                    if (MODE == CAT_BWD && p.accumulate) v += to_f32(d[n]);
                    d[n] = from_f32<T>(v);
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Long axes (N > 1024): a block owns one of `splits` pieces of a segment.  k_cat_long_stats leaves {m, s} of every piece,
// k_cat_long_logp joins them to log-probs, k_cat_long_grad joins them (every block its own row's, in the same order: the
// same bits) and writes its piece of the gradient.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int LONG_NT = 256;

__device__ __forceinline__ void piece_of(const CatArgs& p, int splits, int piece, int V, int& lo, int& hi) {
    const int width = ((p.N + splits - 1) / splits + V - 1) / V * V;
    const long long at = (long long)piece * width;
    lo = at < p.N ? (int)at : p.N;
    hi = p.N - lo > width ? lo + width : p.N;
}

template <typename T>
__global__ __launch_bounds__(LONG_NT) void k_cat_long_stats(CatArgs p, int splits, int mode, float* stats) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float red[2 * (LONG_NT / 64)];
    const size_t s_id = blockIdx.x / splits;
    const int piece = blockIdx.x % splits;
    const size_t b = s_id / p.A;
    const int a = (int)(s_id % p.A);
    const bool on = mode == CAT_PPO ? row_weight(p, b) != 0.0 : (mode == CAT_BWD ? p.dlogp[b] != 0.f : true);
    int lo, hi;
    piece_of(p, splits, piece, V, lo, hi);
    const T* l = static_cast<const T*>(p.logits) + b * p.ld + (size_t)a * p.N;
    float m = -INFINITY, s = 0.f;
    if (on) {
        const int full = lo + (hi - lo) / V * V;
        for (int n = lo + (int)threadIdx.x * V; n < full; n += LONG_NT * V) {
            T t[V];
            load_pack<T, V>(l + n, t);
            float mv = to_f32(t[0]);
#pragma unroll
            for (int i = 1; i < V; ++i) mv = fmaxf(mv, to_f32(t[i]));
            if (mv > m) {
                s *= exp_below(m, mv);
                m = mv;
            }
            const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int i = 0; i < V; ++i) s += exp_below(to_f32(t[i]), ms);
        }
        const int n = full + (int)threadIdx.x;
        if (n < hi) {
            const float x = to_f32(l[n]);
            const float mv = fmaxf(m, x);
            const float ms = mv == -INFINITY ? 0.f : mv;
            s = s * exp_below(m, ms) + exp_below(x, ms);
            m = mv;
        }
    }
    const float mw = group_max<64>(m);
    const float ms = mw == -INFINITY ? 0.f : mw;
    const float sw = group_sum<64>(s * exp_below(m, ms));
    const int wid = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) { red[wid * 2] = mw; red[wid * 2 + 1] = sw; }
    __syncthreads();
    if (threadIdx.x == 0) {
        float mb = red[0], sb = red[1];
        for (int i = 1; i < LONG_NT / 64; ++i) join_softmax(mb, sb, red[i * 2], red[i * 2 + 1]);
        stats[(size_t)blockIdx.x * 2] = mb;
        stats[(size_t)blockIdx.x * 2 + 1] = sb;
    }
}

// {m, s} of one segment joined over its pieces by ONE thread, in order
__device__ __forceinline__ void join_pieces(const float* st, int splits, float& m, float& s) {
    m = st[0];
    s = st[1];
    for (int i = 1; i < splits; ++i) join_softmax(m, s, st[i * 2], st[i * 2 + 1]);
    if (m == -INFINITY) m = 0.f;
}

template <typename T>
__device__ __forceinline__ double segment_logp(const CatArgs& p, size_t b, int a, float m, float s) {
    const long long k = chosen(p, b * p.A + a);
    if (k < 0 || k >= p.N) return 0.0;
    if (s == 0.f) return (double)-INFINITY;
    const float x = to_f32(static_cast<const T*>(p.logits)[b * p.ld + (size_t)a * p.N + k]);
    return (double)x - (double)m - log((double)s);
}

template <typename T>
__global__ __launch_bounds__(64) void k_cat_long_logp(CatArgs p, int splits, const float* stats) {
    const size_t b = blockIdx.x;
    double lp = 0.0;
    for (int a = threadIdx.x; a < p.A; a += 64) {
        float m, s;
        join_pieces(stats + (b * p.A + a) * splits * 2, splits, m, s);
        lp += segment_logp<T>(p, b, a, m, s);
    }
    lp = wave_sum(lp);
    if (threadIdx.x == 0) p.logp[b] = (float)lp;
}

template <typename T, int MODE>
__global__ __launch_bounds__(LONG_NT) void k_cat_long_grad(CatArgs p, int splits, const float* stats) {
    constexpr int V = 16 / sizeof(T);
    __shared__ double red[LONG_NT / 64];
    __shared__ float own[3];                 // m, s of this segment, upstream gradient
    const size_t s_id = blockIdx.x / splits;
    const int piece = blockIdx.x % splits;
    const size_t b = s_id / p.A;
    const int a = (int)(s_id % p.A);
    const double w = MODE == CAT_PPO ? row_weight(p, b) : (double)p.dlogp[b];
    const bool first = MODE == CAT_PPO && piece == 0 && a == 0;
    if (w != 0.0) {
        double lp = 0.0;
        if (MODE == CAT_PPO) {
            for (int c = threadIdx.x; c < p.A; c += LONG_NT) {
                float m, s;
                join_pieces(stats + (b * p.A + c) * splits * 2, splits, m, s);
                if (c == a) { own[0] = m; own[1] = s; }
                lp += segment_logp<T>(p, b, c, m, s);
            }
            lp = wave_sum(lp);
            if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = lp;
            __syncthreads();
        }
        if (threadIdx.x == 0) {
            if (MODE == CAT_PPO) {
                lp = 0.0;
                for (int i = 0; i < LONG_NT / 64; ++i) lp += red[i];
                HeadTerms t = {0.0, 0.0, 0.0};
                own[2] = (float)policy_head(lp, b, w, p.head, t);
                if (first) {
                    p.logp[b] = (float)lp;
                    p.part[b * 3] = t.policy; p.part[b * 3 + 1] = t.kl; p.part[b * 3 + 2] = t.clipped;
                }
            } else {
                join_pieces(stats + s_id * splits * 2, splits, own[0], own[1]);
                own[2] = (float)w;
            }
        }
    } else if (first && threadIdx.x == 0) {
        p.logp[b] = 0.f;
        p.part[b * 3] = p.part[b * 3 + 1] = p.part[b * 3 + 2] = 0.0;
    }
    __syncthreads();
    int lo, hi;
    piece_of(p, splits, piece, V, lo, hi);
    const T* l = static_cast<const T*>(p.logits) + b * p.ld + (size_t)a * p.N;
    T* d = static_cast<T*>(p.dlogits) + b * p.ldd + (size_t)a * p.N;
    const long long k = chosen(p, b * p.A + a);
    const bool live = w != 0.0 && k >= 0 && k < p.N && own[1] != 0.f;
    const float m = live ? own[0] : 0.f, g = live ? own[2] : 0.f;
    const float inv = live ? 1.f / own[1] : 0.f;
    const bool acc = MODE == CAT_BWD && p.accumulate;
    if (!live && acc) return;
    const int full = lo + (hi - lo) / V * V;
    for (int n = lo + (int)threadIdx.x * V; n < full; n += LONG_NT * V) {
        T t[V], o[V];
        float v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = 0.f;
        if (live) {
            load_pack<T, V>(l + n, t);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = g * ((n + i == (int)k ? 1.f : 0.f) - exp_below(to_f32(t[i]), m) * inv);
        }
        if (acc) {
            load_pack<T, V>(d + n, o);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] += to_f32(o[i]);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = from_f32<T>(v[i]);
        store_pack<T, V>(d + n, o);
    }
    const int n = full + (int)threadIdx.x;
    if (n < hi) {
        float v = live ? g * ((n == (int)k ? 1.f : 0.f) - exp_below(to_f32(l[n]), m) * inv) : 0.f;
        if (acc) v += to_f32(d[n]);
        d[n] = from_f32<T>(v);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// The same loss on log-probs that come from elsewhere (the particle mixture's own density): one pass over [n] vectors.
// ---------------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_policy_rows(const float* __restrict__ logp, HeadArgs h, size_t n,
                                                     float* __restrict__ dlogp, double* __restrict__ part) {
    __shared__ double red[3 * 16];
    HeadTerms t = {0.0, 0.0, 0.0};
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const double w = h.weight ? (double)h.weight[i] : h.inv_B;
        dlogp[i] = w != 0.0 ? (float)policy_head((double)logp[i], i, w, h, t) : 0.f;
    }
    block_terms(t, red, part + (size_t)blockIdx.x * 3);
}

// loss4 = {policy + c kl, policy, kl, clipped}: the blocks' sums in a fixed order
__global__ __launch_bounds__(1024) void k_policy_finish(const double* __restrict__ part, size_t nparts, double kl_coef,
                                                        float* __restrict__ loss4) {
    __shared__ double red[3 * 16];
    __shared__ double out[3];
    HeadTerms t = {0.0, 0.0, 0.0};
    for (size_t i = threadIdx.x; i < nparts; i += 1024) {
        t.policy += part[i * 3];
        t.kl += part[i * 3 + 1];
        t.clipped += part[i * 3 + 2];
    }
    block_terms(t, red, out);
    __syncthreads();
    if (threadIdx.x == 0) {
        loss4[0] = (float)(out[0] + kl_coef * out[1]);
        loss4[1] = (float)out[0];
        loss4[2] = (float)out[1];
        loss4[3] = (float)out[2];
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------
constexpr int CAT_MAX_A = 4096, CAT_MAX_N = 1 << 30, CAT_SHORT_N = 1024;
constexpr size_t MAX_BLOCKS = 1u << 22;         // blocks * threads of one launch stay under 2^32

static int splits_for(const CatArgs& p) {
    // pieces of a long axis: enough blocks for the chip (two waves of it), pieces of at least 4096 logits
    const long long segs = (long long)p.B * p.A;
    long long s = (2048 + segs - 1) / segs;
    const long long most = (p.N + 4095) / 4096;
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s);
}
static int rows_per_block(int B, int A, int G) {
    const int groups = 512 / G;
    int rb = (4 * groups + A - 1) / A;              // about four rounds of segments
    const int by_chip = (B + 511) / 512;            // but fill the chip first
    if (rb > by_chip) rb = by_chip;
    if (rb < 1) rb = 1;
    while (rb > 1 && (size_t)rb * A > 4096) --rb;
    return rb;
}

template <typename T, int MODE, int G, int E>
static void launch_rows(CatArgs p, hipStream_t st, int& blocks) {
    p.rows_per_block = rows_per_block(p.B, p.A, G);
    blocks = (int)(((long long)p.B + p.rows_per_block - 1) / p.rows_per_block);
    if ((size_t)blocks > MAX_BLOCKS) { blocks = -1; return; }
    const size_t lds = 48 * sizeof(double) + ((size_t)p.rows_per_block * p.A * 3 + p.rows_per_block) * sizeof(float);
    hipLaunchKernelGGL((k_cat_rows<T, MODE, G, E>), dim3(blocks), dim3(512), lds, st, p);
}

// groups of lanes by the axis: the fewest idle slots among the widths (35 particles: 8 lanes x 5, 40 slots)
template <typename T, int MODE>
static void pick_rows(const CatArgs& p, hipStream_t st, int& blocks) {
    const int N = p.N;
    if (N <= 8) launch_rows<T, MODE, 8, 1>(p, st, blocks);
    else if (N <= 16) launch_rows<T, MODE, 8, 2>(p, st, blocks);
    else if (N <= 24) launch_rows<T, MODE, 8, 3>(p, st, blocks);
    else if (N <= 32) launch_rows<T, MODE, 8, 4>(p, st, blocks);
    else if (N <= 40) launch_rows<T, MODE, 8, 5>(p, st, blocks);
    else if (N <= 64) launch_rows<T, MODE, 16, 4>(p, st, blocks);
    else if (N <= 96) launch_rows<T, MODE, 16, 6>(p, st, blocks);
    else if (N <= 128) launch_rows<T, MODE, 32, 4>(p, st, blocks);
    else if (N <= 192) launch_rows<T, MODE, 32, 6>(p, st, blocks);
    else if (N <= 256) launch_rows<T, MODE, 64, 4>(p, st, blocks);
    else if (N <= 512) launch_rows<T, MODE, 64, 8>(p, st, blocks);
    else launch_rows<T, MODE, 64, 16>(p, st, blocks);
}

template <typename T, int MODE>
static int run_cat(CatArgs p, void* ws, size_t ws_bytes, float* loss4, hipStream_t st) {
    p.magic_A = p.A > 1 ? (uint32_t)((0x100000000ull + p.A - 1) / p.A) : 0;
    size_t nparts = 0;
    if (p.N <= CAT_SHORT_N) {
        const size_t need = MODE == CAT_PPO ? (size_t)p.B * 3 * sizeof(double) : 0;
        if (need && (!ws || ws_bytes < need)) return PFPN_ERR_WORKSPACE;
        p.part = static_cast<double*>(ws);
        int blocks = 0;
        pick_rows<T, MODE>(p, st, blocks);
        if (blocks < 0) return PFPN_ERR_ARG;
        nparts = blocks;
    } else {
        const int S = splits_for(p);
        const size_t pieces = (size_t)p.B * p.A * S;
        const size_t parts = MODE == CAT_PPO ? (size_t)p.B * 3 * sizeof(double) : 0;
        if (pieces > MAX_BLOCKS) return PFPN_ERR_ARG;
        if (!ws || ws_bytes < parts + pieces * 2 * sizeof(float)) return PFPN_ERR_WORKSPACE;
        p.part = static_cast<double*>(ws);
        float* stats = reinterpret_cast<float*>(static_cast<char*>(ws) + parts);
        hipLaunchKernelGGL((k_cat_long_stats<T>), dim3((unsigned)pieces), dim3(LONG_NT), 0, st, p, S, MODE, stats);
        if (MODE == CAT_FWD)
            hipLaunchKernelGGL((k_cat_long_logp<T>), dim3(p.B), dim3(64), 0, st, p, S, (const float*)stats);
        else
            hipLaunchKernelGGL((k_cat_long_grad<T, MODE>), dim3((unsigned)pieces), dim3(LONG_NT), 0, st, p, S, (const float*)stats);
        nparts = p.B;
    }
    if (MODE == CAT_PPO)
        hipLaunchKernelGGL(k_policy_finish, dim3(1), dim3(1024), 0, st, (const double*)p.part, nparts, p.head.kl_coef, loss4);
    PFPN_CHECK_LAUNCH();
    return PFPN_OK;
}

template <int MODE>
static int run_typed(const CatArgs& p, int dtype, void* ws, size_t ws_bytes, float* loss4, void* stream) {
    hipStream_t st = (hipStream_t)stream;
    if (dtype == DT_F32) return run_cat<float, MODE>(p, ws, ws_bytes, loss4, st);
    if (dtype == DT_BF16) return run_cat<bf16_t, MODE>(p, ws, ws_bytes, loss4, st);
    return run_cat<f16_t, MODE>(p, ws, ws_bytes, loss4, st);
}

static bool bad_shape(const void* logits, int dtype, long long ld, const void* index, int B, int A, int N) {
    return !logits || !index || dtype < DT_F32 || dtype > DT_F16 || B < 1 || A < 1 || N < 1 || A > CAT_MAX_A ||
           N > CAT_MAX_N || ld < (long long)A * N;
}
static bool bad_head(const HeadArgs& h) {
    return !h.logp_old || !h.adv || !(h.clip_lo <= 1.0) || !(h.clip_hi >= 1.0) || (h.kl_coef != 0.0 && !h.logp_ref);
}
static int policy_row_blocks(long long n) { return (int)(n / 1024 + 1 < 1024 ? n / 1024 + 1 : 1024); }

}  // namespace pfpn

using namespace pfpn;

extern "C" {

size_t pfpn_categorical_workspace_bytes(int B, int A, int N) {
    if (B < 1 || A < 1 || N < 1) return 0;
    CatArgs p = {};
    p.B = B; p.A = A; p.N = N;
    const size_t parts = (size_t)B * 3 * sizeof(double);
    return N <= CAT_SHORT_N ? parts : parts + (size_t)B * A * splits_for(p) * 2 * sizeof(float);
}

int pfpn_categorical_logprob_fwd(const void* logits, int dtype, long long row_stride, const void* index, int index64,
                                 int B, int A, int N, float* logp, void* workspace, size_t workspace_bytes, void* stream) {
    PFPN_BEGIN();
    if (bad_shape(logits, dtype, row_stride, index, B, A, N) || !logp) return PFPN_ERR_ARG;
    CatArgs p = {};
    p.logits = logits; p.ld = row_stride; p.index = index; p.index64 = index64;
    p.B = B; p.A = A; p.N = N; p.logp = logp;
    return run_typed<CAT_FWD>(p, dtype, workspace, workspace_bytes, nullptr, stream);
}

int pfpn_categorical_logprob_bwd(const void* logits, int dtype, long long row_stride, const void* index, int index64,
                                 const float* dlogp, int B, int A, int N, int accumulate, void* dlogits,
                                 long long grad_stride, void* workspace, size_t workspace_bytes, void* stream) {
    PFPN_BEGIN();
    if (bad_shape(logits, dtype, row_stride, index, B, A, N) || !dlogp || !dlogits || grad_stride < (long long)A * N)
        return PFPN_ERR_ARG;
    CatArgs p = {};
    p.logits = logits; p.ld = row_stride; p.index = index; p.index64 = index64;
    p.B = B; p.A = A; p.N = N; p.dlogp = dlogp; p.dlogits = dlogits; p.ldd = grad_stride; p.accumulate = accumulate;
    return run_typed<CAT_BWD>(p, dtype, workspace, workspace_bytes, nullptr, stream);
}

int pfpn_categorical_ppo_fwd_bwd(const void* logits, int dtype, long long row_stride, const void* index, int index64,
                                 const float* logp_old, const float* adv, const float* logp_ref, const float* weight,
                                 const float* adv_stats, int B, int A, int N, double clip_eps_low, double clip_eps_high,
                                 double kl_coef, float* logp, void* dlogits, long long grad_stride, float* loss4,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    PFPN_BEGIN();
    CatArgs p = {};
    p.head = {logp_old, adv, logp_ref, weight, adv_stats, 1.0 - clip_eps_low, 1.0 + clip_eps_high, kl_coef,
              B > 0 ? 1.0 / B : 0.0};
    if (bad_shape(logits, dtype, row_stride, index, B, A, N) || bad_head(p.head) || !logp || !dlogits || !loss4 ||
        grad_stride < (long long)A * N)
        return PFPN_ERR_ARG;
    p.logits = logits; p.ld = row_stride; p.index = index; p.index64 = index64;
    p.B = B; p.A = A; p.N = N; p.logp = logp; p.dlogits = dlogits; p.ldd = grad_stride;
    return run_typed<CAT_PPO>(p, dtype, workspace, workspace_bytes, loss4, stream);
}

size_t pfpn_policy_kl_workspace_bytes(long long n) {
    return n < 1 ? 0 : (size_t)policy_row_blocks(n) * 3 * sizeof(double);
}

int pfpn_policy_kl_loss(const float* logp, const float* logp_old, const float* adv, const float* logp_ref,
                        const float* weight, const float* adv_stats, long long n, double clip_eps_low, double clip_eps_high,
                        double kl_coef, float* dlogp, float* loss4, void* workspace, size_t workspace_bytes, void* stream) {
    PFPN_BEGIN();
    const HeadArgs h = {logp_old, adv, logp_ref, weight, adv_stats, 1.0 - clip_eps_low, 1.0 + clip_eps_high, kl_coef,
                        n > 0 ? 1.0 / (double)n : 0.0};
    if (!logp || bad_head(h) || !dlogp || !loss4 || n < 1) return PFPN_ERR_ARG;
    if (!workspace || workspace_bytes < pfpn_policy_kl_workspace_bytes(n)) return PFPN_ERR_WORKSPACE;
    const int blocks = policy_row_blocks(n);
    double* part = static_cast<double*>(workspace);
    hipLaunchKernelGGL(k_policy_rows, dim3(blocks), dim3(256), 0, (hipStream_t)stream, logp, h, (size_t)n, dlogp, part);
    hipLaunchKernelGGL(k_policy_finish, dim3(1), dim3(1024), 0, (hipStream_t)stream, (const double*)part, (size_t)blocks,
                       kl_coef, loss4);
    PFPN_CHECK_LAUNCH();
    return PFPN_OK;
}

}  // extern "C"
