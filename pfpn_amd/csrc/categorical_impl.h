// Kernels of categorical_kernels.hip for one element type of the logits (instantiated by categorical_f32 / _bf16 / _f16.hip).
#pragma once
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
    int rows_per_block, lanes_per_row;
    int stream;                 // the gradient is larger than the infinity cache: stores past it
    uint32_t magic_A;           // ceil(2^32 / A) (A > 1)
    double* part;               // CAT_PPO: three sums per block
    float* loss4;               // ... or, where one block takes the whole batch, the loss itself
};

__device__ __forceinline__ void write_loss4(const double* sums, double kl_coef, float* loss4) {
    loss4[0] = (float)(kl_coef != 0.0 ? sums[0] + kl_coef * sums[1] : sums[0]);
    loss4[1] = (float)sums[0];
    loss4[2] = (float)sums[1];
    loss4[3] = (float)sums[2];
}

constexpr int CAT_MAX_A = 4096, CAT_MAX_N = 1 << 30, CAT_SHORT_N = 1024;
constexpr int CAT_MAX_SPLITS = 64;              // pieces of a long axis: one wave joins them
constexpr size_t MAX_BLOCKS = (1u << 22) - 1;   // blocks * threads of one launch stay under 2^32

// one call for logits of type T; *nparts: the blocks that left loss terms (CAT_PPO)
template <typename T, int MODE>
int run_cat(CatArgs p, void* ws, size_t ws_bytes, size_t* nparts, hipStream_t st);

int cat_splits(int B, int A, int N);

#ifdef PFPN_CATEGORICAL_TYPE

// the chosen category, -1 where it is outside the axis (that choice does not enter the row); no branch on the index type
__device__ __forceinline__ int chosen_in(const CatArgs& p, size_t i) {
    const int* at = static_cast<const int*>(p.index) + (i << p.index64);
    const int lo = at[0], second = at[p.index64], hi = p.index64 ? second : lo >> 31;
    return hi == 0 && lo >= 0 && lo < p.N ? lo : -1;
}
__device__ __forceinline__ int div_A(const CatArgs& p, int q) {
    return p.A == 1 ? q : (int)__umulhi((uint32_t)q, p.magic_A);
}
__device__ __forceinline__ double row_weight(const CatArgs& p, size_t b) {
    return p.head.weight ? (double)p.head.weight[b] : p.head.inv_B;
}

// ---------------------------------------------------------------------------------------------------------------------
// Short axes (N <= 1024): a group of G lanes owns a segment (row, choice), a lane E consecutive logits of it.  A block owns whole
// rows, so the joint log-prob of a row and with it the upstream gradient are known inside the block: the loss takes ONE pass.
// Phase 1: {l_k, m, s} of every segment into LDS; phase 2: the rows' log-probs and loss heads (64 bits), lanes_per_row lanes a
// row; phase 3: the gradients from the exponentials that phase 1 left in registers (IT segments a group; IT = 0, rows too wide
// for that: from the logits again, out of the caches).
// Bound: HBM, one read of the logits and one write of the gradient.  8192 x 128 x 256 float32: 380 us = 5.7 TB/s (a 1-GiB copy on
// the same card: 425 us); 4096 x 36 x 35: 13.0 us = 3.2 TB/s, one wave of blocks: instructions issue for 5.4 us of
// it, waves wait for half of their time.
// What it measured on the way, 8192 x 128 x 256: reading the logits twice 933 us; holding 64 exponentials a thread, spilled around
// the 64-bit head, 555 us; loads behind bounds branches (hipcc waits for each one) 511 us; clamped loads without a branch and half
// of the exponentials parked in LDS 395 us.  Eight lanes x 5 for 35 particles, not 4 x 9: fewer waves, 14.1 against 16.2 us.
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int MODE, int G, int E, int IT, int NT>
__global__ __launch_bounds__(NT, E * IT > 32 ? 4 : 8) void k_cat_rows(CatArgs p) {
    constexpr int NG = NT / G, HOLD = IT > 0 ? IT : 1;
    struct Segment { float xk, m, s; int k; };
    extern __shared__ char lds_raw[];
    const int tid = threadIdx.x, gid = tid / G;
    const Axis<T, G, E> ln(tid % G, p.N);
    const int RB = p.rows_per_block;
    const size_t row0 = (size_t)blockIdx.x * RB;
    const int rows = (int)((size_t)p.B - row0 < (size_t)RB ? (size_t)p.B - row0 : (size_t)RB);
    const int nseg = rows * p.A;
    Segment* seg = reinterpret_cast<Segment*>(lds_raw);                         // [RB * A]
    double* terms = reinterpret_cast<double*>(seg + (size_t)RB * p.A);          // [RB][3]
    float* row_g = reinterpret_cast<float*>(terms + RB * 3);                    // [RB] upstream gradient
    float* row_in = row_g + RB;                                                 // [RB][3] = logp_old, adv, logp_ref
    // (a block's rows span less than 2^31 bytes: 32-bit offsets from its first)
    const T* logits = static_cast<const T*>(p.logits) + row0 * p.ld;
    T* dlogits = static_cast<T*>(p.dlogits) + row0 * p.ldd;
    const int ld = (int)p.ld, ldd = (int)p.ldd;
    // half of the exponentials wait in LDS while the heads run: their 64-bit arithmetic needs the registers
    float* parked = row_in + RB * 3;                                            // [IT / 2 * E][NT]
    const bool weighted = MODE == CAT_PPO && p.head.weight;

    // where segment q of this block lies (past the last one: the last one again); a row without weight: the block's first row, which
    // costs no traffic of its own -- what is read there is not used
    auto weight_of = [&](int q) { return weighted ? p.head.weight[row0 + div_A(p, q < nseg ? q : nseg - 1)] : 1.f; };
    auto segment_at = [&](int q, float w) {
        q = q < nseg ? q : nseg - 1;
        const int r = div_A(p, q), a = q - r * p.A;
        return logits + (unsigned)((w == 0.f ? 0 : r) * ld + a * p.N);
    };
    const bool whole = p.N % ln.V == 0;          // packs belong to their lane entirely or not at all
    // one segment: exponentials, m, s
    auto softmax_of = [&](const T (&raw)[E], float (&x)[E], float& m, float& s) {
        m = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = to_f32(raw[e]);
            m = fmaxf(m, x[e]);
        }
        m = group_max<G>(m);
        if (m == -INFINITY) m = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = exp_below_exact(x[e], m);
        s = 0.f;
        if (whole) {
#pragma unroll
            for (int u = 0; u < ln.U; ++u) {
                float t = x[u * ln.V];
#pragma unroll
                for (int v = 1; v < ln.V; ++v) t += x[u * ln.V + v];
                s += ln.has(u) ? t : 0.f;
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) s += ln.own(e) ? x[e] : 0.f;
        }
        s = group_sum<G>(s);
    };
    // a segment with no open choice (s = 0), an index outside the axis and a row without upstream gradient get zeros
    auto put_gradient = [&](int q, const float (&x)[E], int k, float g, float s) {
        const int r = div_A(p, q), a = q - r * p.A;
        const bool live = k >= 0 && s != 0.f && g != 0.f;
        const float gi = g * (1.f / s);
        T* d = dlogits + (unsigned)(r * ldd + a * p.N);
        T o[E];
        if (MODE == CAT_BWD && p.accumulate) {
            if (!live) return;
            ln.load(d, o);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float v = live ? (ln.at(e) == k ? g : 0.f) - x[e] * gi : 0.f;
            if (MODE == CAT_BWD && p.accumulate) v += to_f32(o[e]);
            o[e] = from_f32<T>(v);
        }
        ln.store(d, o, p.stream);
    };

    if (MODE == CAT_BWD) {
        for (int q0 = 0; q0 < nseg; q0 += NG) {
            const int q = q0 + gid;
            T raw[E];
            float x[E], m, s;
            ln.load(segment_at(q, 1.f), raw);
            const int k = q < nseg ? chosen_in(p, row0 * p.A + q) : -1;
            const float g = q < nseg ? p.dlogp[row0 + div_A(p, q)] : 0.f;
            softmax_of(raw, x, m, s);
            if (q < nseg) put_gradient(q, x, k, g, s);
        }
        return;
    }

    // on the way while the logits are read: the loss inputs of the rows, and the chosen logits
    HeadRow hr = {0.f, 0.f, 0.f, 0.0};
    if (MODE == CAT_PPO && tid < rows) hr = head_row(p.head, row0 + tid);
    int k0 = -1;
    if (tid < nseg) k0 = chosen_in(p, row0 * p.A + tid);
    float x[HOLD][E];
    T raw[HOLD][E];
    if (IT > 0) {
        float w[HOLD];
#pragma unroll
        for (int it = 0; it < HOLD; ++it) w[it] = weight_of(it * NG + gid);
#pragma unroll
        for (int it = 0; it < HOLD; ++it) ln.load(segment_at(it * NG + gid, w[it]), raw[it]);
    }
    if (MODE == CAT_PPO && tid < rows) {
        row_in[tid * 3] = hr.logp_old;
        row_in[tid * 3 + 1] = hr.a;
        row_in[tid * 3 + 2] = hr.logp_ref;
    }
    for (int q = tid; q < nseg; q += NT) {
        const int k = q == tid ? k0 : chosen_in(p, row0 * p.A + q);
        seg[q].k = k;
        seg[q].xk = k >= 0 ? to_f32(segment_at(q, 1.f)[k]) : 0.f;
    }
    if (IT > 0) {
#pragma unroll
        for (int it = 0; it < HOLD; ++it) {
            const int q = it * NG + gid;
            float m, s;
            softmax_of(raw[it], x[it], m, s);
            if (ln.j == 0 && q < nseg) { seg[q].m = m; seg[q].s = s; }
            if (it >= IT / 2) {
#pragma unroll
                for (int e = 0; e < E; ++e) parked[((it - IT / 2) * E + e) * NT + tid] = x[it][e];
            }
        }
    } else {
        for (int q0 = 0; q0 < nseg; q0 += NG) {
            const int q = q0 + gid;
            float m, s;
            ln.load(segment_at(q, weight_of(q)), raw[0]);
            softmax_of(raw[0], x[0], m, s);
            if (ln.j == 0 && q < nseg) { seg[q].m = m; seg[q].s = s; }
        }
    }
    __syncthreads();
    // (waves without a row go past: the 64-bit head needs registers that their exponentials occupy)
    const int LP = p.lanes_per_row, my_row = tid / LP;
    if (__builtin_amdgcn_readfirstlane(my_row) < rows) {
        double lp = 0.0;
        const double w = MODE == CAT_PPO && my_row < rows ? row_weight(p, row0 + my_row) : 1.0;
        if (my_row < rows && w != 0.0) {
            // one logarithm a lane: of the product of its sums (at most 64 of them, each 0 or within [1, 1024]; 1048 x 4000 x 8: 63 of
            // them a lane, 129 -> 95 us)
            double prod = 1.0;
            for (int a = tid % LP; a < p.A; a += LP) {
                const Segment v = seg[my_row * p.A + a];
                if (v.k >= 0) {
                    lp += (double)v.xk - (double)v.m;
                    prod *= (double)v.s;
                }
            }
            lp = prod == 0.0 ? (double)-INFINITY : lp - log(prod);
        }
        lp = LP == 1 ? lp : LP == 4 ? group_sum<4>(lp) : LP == 16 ? group_sum<16>(lp) : group_sum<64>(lp);
        if (tid % LP == 0 && my_row < rows) {
            p.logp[row0 + my_row] = (float)lp;
            if (MODE == CAT_PPO) {
                HeadTerms t = {0.0, 0.0, 0.0};
                const HeadRow row = {row_in[my_row * 3], row_in[my_row * 3 + 1], row_in[my_row * 3 + 2], w};
                row_g[my_row] = w != 0.0 ? (float)policy_head(lp, row, p.head, t) : 0.f;
                terms[my_row * 3] = t.policy;
                terms[my_row * 3 + 1] = t.kl;
                terms[my_row * 3 + 2] = t.clipped;
            }
        }
    }
    if (MODE == CAT_FWD) return;
    __syncthreads();
    if (IT > 0) {
#pragma unroll
        for (int it = 0; it < HOLD; ++it) {
            const int q = it * NG + gid;
            if (it >= IT / 2) {
#pragma unroll
                for (int e = 0; e < E; ++e) x[it][e] = parked[((it - IT / 2) * E + e) * NT + tid];
            }
            if (q < nseg) put_gradient(q, x[it], seg[q].k, row_g[div_A(p, q)], seg[q].s);
        }
    } else {
        for (int q = gid; q < nseg; q += NG) {
            ln.load(segment_at(q, weight_of(q)), raw[0]);
            const float m = seg[q].m;
#pragma unroll
            for (int e = 0; e < E; ++e) x[0][e] = exp_below_exact(to_f32(raw[0][e]), m);
            put_gradient(q, x[0], seg[q].k, row_g[div_A(p, q)], seg[q].s);
        }
    }
    // the block's loss terms, in row order (a wave per term), while the stores drain
    const int wid = tid >> 6, lane = tid & 63;
    if (wid < 3) {
        double t = 0.0;
        for (int r = lane; r < rows; r += 64) t += terms[r * 3 + wid];
        t = group_sum<64>(t);
        if (lane == 0 && !p.loss4) p.part[(size_t)blockIdx.x * 3 + wid] = t;
        if (lane == 0 && p.loss4) terms[(rows - 1) * 3 + wid] = t;      // (the last row's terms have been added)
    }
    if (p.loss4) {
        __syncthreads();
        if (tid == 0) write_loss4(terms + (rows - 1) * 3, p.head.kl_coef, p.loss4);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Long axes (N > 1024), rows that one block can hold (few very long ones: in pieces, below): a block owns a segment and keeps ALL of
// it in registers (H wide loads a thread, raw), so the logits are read once whatever their length: one pass finds {m, s}, the gradient
// is formed from the registers.  For A = 1 (a token row) the loss head sits in between, run by one wave (of eight packs three wait in
// LDS meanwhile: its 64-bit arithmetic would spill them).  64 to 1024 threads of four packs, 1024 of eight (two blocks a CU: one reads
// while the other writes) or sixteen (one block a CU), the fewest that hold the row.
// Bound: HBM.  6001 x 50021 bfloat16, a fifth of the rows without weight: 241 us = 4.5 TB/s (two kernels that read the logits twice:
// 337 us); gradient of 2047 x 32001 float16: 55 us = 4.8 TB/s (86 us).  One fma an exponent, packed maxima and
// the join of the waves a lane each: 60 -> 55 us, 253 -> 241 us (13 vector instructions an element now, 25 us of issue in the 55).
// ---------------------------------------------------------------------------------------------------------------------
template <int NW>
__device__ __forceinline__ void block_softmax(float m, float s, float* red, float& M, float& S) {
    // (m, s) of a wave, wave-uniform -> of the block: a lane a wave
    if ((threadIdx.x & 63) == 0) {
        red[(threadIdx.x >> 6) * 2] = m;
        red[(threadIdx.x >> 6) * 2 + 1] = s;
    }
    __syncthreads();
    const int i = threadIdx.x & (NW - 1);
    const float mi = red[i * 2], si = red[i * 2 + 1];
    M = group_max<NW>(mi);
    if (M == -INFINITY) M = 0.f;
    S = group_sum<NW>(si * exp_below(mi, M));
}

// exp(x - m) as v_exp_f32 of ONE fma, x log2(e) - c: what rounding c = m log2(e) does is common to all terms, `left` (in powers of two).
// Within |m| <= 256: beyond, and where m is infinite, the difference is formed first.
constexpr float EXP_NEAR = 256.f;
struct NearExp {
    float c, left;
    __device__ __forceinline__ explicit NearExp(float m) : c(-m * PFPN_LOG2E), left(__builtin_fmaf(m, PFPN_LOG2E, c)) {}
    __device__ __forceinline__ float operator()(float x) const {
        return __builtin_amdgcn_exp2f(__builtin_fmaf(x, PFPN_LOG2E, c));
    }
};

// |g| p of one logit of a 16-bit gradient: log2 |g / s| joins the exponent too (rounded at 2^-24 of some hundreds, far under
// the output's half step)
struct NearProb {
    float c;
    __device__ __forceinline__ NearProb(float m, float log_scale) : c(__builtin_fmaf(-m, PFPN_LOG2E, log_scale)) {}
    __device__ __forceinline__ float operator()(float x) const {
        return __builtin_amdgcn_exp2f(__builtin_fmaf(x, PFPN_LOG2E, c));
    }
};
// -g p of one logit, any type, any m
template <typename T>
struct NegProb {
    float m, scale, log_scale;
    __device__ __forceinline__ NegProb(float m_, float g, float inv) : m(m_), scale(-g * inv), log_scale(__log2f(fabsf(g * inv))) {}
    __device__ __forceinline__ float operator()(float x) const {
        if (sizeof(T) == 4) return exp_below_exact(x, m) * scale;
        const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(x - m, PFPN_LOG2E, log_scale));
        return __builtin_copysignf(v, scale);
    }
};

// 32 bits of -inf logits
template <typename T> __device__ __forceinline__ uint32_t closed_logits();
template <> __device__ __forceinline__ uint32_t closed_logits<float>() { return 0xff800000u; }
template <> __device__ __forceinline__ uint32_t closed_logits<bf16_t>() { return 0xff80ff80u; }
template <> __device__ __forceinline__ uint32_t closed_logits<f16_t>() { return 0xfc00fc00u; }

__device__ __forceinline__ double token_logp(int k, float xk, float m, float s) {
    return k < 0 ? 0.0 : (s == 0.f ? (double)-INFINITY : (double)xk - (double)m - log((double)s));
}

template <typename T, int MODE, int H, int NT>
__global__ __launch_bounds__(NT, H > 8 ? 4 : 8) void k_cat_long_held(CatArgs p) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float red[2 * (NT / 64)];
    const size_t s_id = blockIdx.x;
    const size_t b = p.A == 1 ? s_id : s_id / p.A;
    const int a = p.A == 1 ? 0 : (int)(s_id % p.A), N = p.N, tid = threadIdx.x;
    const T* l = static_cast<const T*>(p.logits) + b * p.ld + (size_t)a * N;
    T* d = MODE == CAT_FWD ? nullptr : static_cast<T*>(p.dlogits) + b * p.ldd + (size_t)a * N;
    const int k = chosen_in(p, s_id);
    float g = 1.f;
    if (MODE == CAT_BWD) g = p.dlogp[b];
    const bool on = MODE == CAT_PPO ? row_weight(p, b) != 0.0 : g != 0.f;
    const int full = N / V * V, last = full + tid;
    if (!on || (MODE == CAT_BWD && k < 0)) {
        if (MODE == CAT_PPO && tid == 0) {
            p.logp[b] = 0.f;
            p.part[b * 3] = p.part[b * 3 + 1] = p.part[b * 3 + 2] = 0.0;
        }
        if (MODE == CAT_BWD && p.accumulate) return;
        const T zero[V] = {};
        for (int n = tid * V; n < full; n += NT * V) store_pack<T, V>(d + n, zero);
        if (last < N) d[last] = zero[0];
        return;
    }
    // slots past the axis hold closed categories: the sums need no bounds
    Held<T, V> raw[H];
    float tail = -INFINITY;
#pragma unroll
    for (int h = 0; h < H; ++h) {
        // (no branch: all of a thread's loads are in flight together; past the end the last pack again)
        const int n = (h * NT + tid) * V;
        raw[h].load(l + (n < full ? n : full - V));
    }
#pragma unroll
    for (int h = 0; h < H; ++h)
        if ((h * NT + tid) * V >= full) raw[h].fill(closed_logits<T>());
    if (last < N) tail = to_f32(l[last]);
    const float xk = k >= 0 ? to_f32(l[k]) : 0.f;
    HeldMax<T> top;
#pragma unroll
    for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int i = 0; i < raw[h].W; ++i) top.take(raw[h].w[i]);
        raw[h].forget();
    }
    const float m = group_max<64>(fmaxf(tail, top.value()));
    const float mw = m == -INFINITY ? 0.f : m;
    const bool near = fabsf(mw) <= EXP_NEAR;        // (the same in the whole wave; false for a NaN)
    const NearExp ne(mw);
    float s = 0.f;
    if (near) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if (h * NT * V < full) {
                float t = ne(raw[h][0]);
#pragma unroll
                for (int i = 1; i < V; ++i) t += ne(raw[h][i]);
                s += t;
            }
            raw[h].forget();
        }
        s = (s + ne(tail)) * __builtin_amdgcn_exp2f(-ne.left);
    } else {
#pragma unroll
        for (int h = 0; h < H; ++h) {
#pragma unroll
            for (int i = 0; i < V; ++i) s += exp_below(raw[h][i], mw);
            raw[h].forget();
        }
        s += exp_below(tail, mw);
    }
    s = group_sum<64>(s);
    float M, S;
    block_softmax<NT / 64>(m, s, red, M, S);
    if (MODE == CAT_FWD) {
        if (tid == 0) p.logp[b] = (float)token_logp(k, xk, M, S);
        return;
    }
    if (MODE == CAT_PPO) {
        // one wave: the 64-bit head needs registers that the others' logits occupy
        __shared__ float up;
        constexpr int PARK = H == 8 ? 3 : 0;            // (packs of eight that wait in LDS meanwhile)
        __shared__ uint32_t parked[PARK ? PARK * 4 * NT : 1];
#pragma unroll
        for (int i = 0; i < PARK * 4; ++i) parked[i * NT + tid] = raw[H - PARK + i / 4].w[i % 4];
        if (tid < 64) {
            const double lp = token_logp(k, xk, M, S);
            const HeadRow hr = head_row(p.head, b);
            HeadTerms t;
            const float gw = (float)policy_head(lp, hr, p.head, t);
            if (tid == 0) {
                up = gw;
                p.logp[b] = (float)lp;
                p.part[b * 3] = t.policy;
                p.part[b * 3 + 1] = t.kl;
                p.part[b * 3 + 2] = t.clipped;
            }
        }
        __syncthreads();
        g = up;
#pragma unroll
        for (int i = 0; i < PARK * 4; ++i) raw[H - PARK + i / 4].w[i % 4] = parked[i * NT + tid];
    }
    const bool live = k >= 0 && S != 0.f && g != 0.f, acc = MODE == CAT_BWD && p.accumulate;
    const float inv = live ? 1.f / S : 0.f;
    const NegProb<T> np(live ? M : 0.f, live ? g : 0.f, inv);
    const float gk = live ? g - exp_below_exact(xk, M) * (g * inv) : 0.f;
    if (sizeof(T) == 2 && live && !acc && fabsf(M) <= EXP_NEAR) {
        // the usual case of a 16-bit gradient: two instructions, a conversion of two and the sign of two an element
        const NearProb pr(M, np.log_scale);
        const uint32_t sign = np.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const int n = (h * NT + tid) * V;
            if (n < full) {
                T o[V];
#pragma unroll
                for (int i = 0; i < V; i += 2) {
                    const T a0 = from_f32<T>(pr(raw[h][i])), a1 = from_f32<T>(pr(raw[h][i + 1]));
                    const uint32_t w = ((uint32_t)__builtin_bit_cast(typename Bits<T>::type, a0) |
                                        (uint32_t)__builtin_bit_cast(typename Bits<T>::type, a1) << 16) | sign;
                    o[i] = __builtin_bit_cast(T, (typename Bits<T>::type)w);
                    o[i + 1] = __builtin_bit_cast(T, (typename Bits<T>::type)(w >> 16));
                }
                if ((unsigned)(k - n) < (unsigned)V) {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (n + i == k) o[i] = from_f32<T>(gk);
                }
                store_pack<T, V>(d + n, o, p.stream);
            }
        }
    } else {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const int n = (h * NT + tid) * V;
            if (n < full) {
                float v[V];
                T o[V];
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = live ? np(raw[h][i]) : 0.f;
                if ((unsigned)(k - n) < (unsigned)V) {
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] = n + i == k ? gk : v[i];
                }
                if (acc) {
                    load_pack<T, V>(d + n, o);
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] += to_f32(o[i]);
                }
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = from_f32<T>(v[i]);
                store_pack<T, V>(d + n, o, p.stream);
            }
        }
    }
    if (last < N) {
        float v = !live ? 0.f : last == k ? gk : np(tail);
        if (acc) v += to_f32(d[last]);
        d[last] = from_f32<T>(v);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Long axes, few rows, several long choices in a row, or an axis beyond the registers: a block owns one of `splits` pieces of a
// segment.  k_cat_long_stats leaves {m, s} of every piece, k_cat_long_rows joins them to log-probs, k_cat_long_grad joins them
// (every block its own row's, in the same order: the same bits) and writes its piece of the gradient.
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
    float M, S;
    block_softmax<LONG_NT / 64>(mw, sw, red, M, S);
    if (threadIdx.x == 0) {
        stats[(size_t)blockIdx.x * 2] = S == 0.f ? -INFINITY : M;
        stats[(size_t)blockIdx.x * 2 + 1] = S;
    }
}

// {m, s} of one segment joined over its pieces by a wave (a lane a piece)
__device__ __forceinline__ void join_pieces(const float* st, int splits, float& m, float& s) {
    const int lane = threadIdx.x & 63;
    const float mi = lane < splits ? st[lane * 2] : -INFINITY, si = lane < splits ? st[lane * 2 + 1] : 0.f;
    m = group_max<64>(mi);
    if (m == -INFINITY) m = 0.f;
    s = group_sum<64>(si * exp_below(mi, m));
}

template <typename T>
__device__ __forceinline__ double segment_logp(const CatArgs& p, size_t b, int a, float m, float s) {
    const int k = chosen_in(p, b * p.A + a);
    if (k < 0) return 0.0;
    if (s == 0.f) return (double)-INFINITY;
    const float x = to_f32(static_cast<const T*>(p.logits)[b * p.ld + (size_t)a * p.N + k]);
    return (double)x - (double)m - log((double)s);
}

// a block a row: its joint log-prob (a wave per choice, in turn) and, CAT_PPO, its upstream gradient and loss terms
template <typename T, int MODE>
__global__ __launch_bounds__(LONG_NT) void k_cat_long_rows(CatArgs p, int splits, const float* stats, float* row_g) {
    __shared__ double red[LONG_NT / 64];
    const size_t b = blockIdx.x;
    const int wid = threadIdx.x >> 6, nw = blockDim.x >> 6;
    const bool on = MODE != CAT_PPO || row_weight(p, b) != 0.0;
    double lp = 0.0;
    for (int c = wid; on && c < p.A; c += nw) {
        float m, s;
        join_pieces(stats + (b * p.A + c) * splits * 2, splits, m, s);
        lp += segment_logp<T>(p, b, c, m, s);
    }
    if ((threadIdx.x & 63) == 0) red[wid] = lp;
    __syncthreads();
    if (threadIdx.x == 0) {
        lp = 0.0;
        for (int i = 0; i < nw; ++i) lp += red[i];
        p.logp[b] = (float)lp;
        if (MODE == CAT_PPO) {
            HeadTerms t = {0.0, 0.0, 0.0};
            row_g[b] = on ? (float)policy_head(lp, head_row(p.head, b), p.head, t) : 0.f;
            p.part[b * 3] = t.policy;
            p.part[b * 3 + 1] = t.kl;
            p.part[b * 3 + 2] = t.clipped;
        }
    }
}

// MODE CAT_PPO: one choice a row, every wave joins and runs its head; CAT_BWD: the upstream gradient of the row is p.dlogp's
template <typename T, int MODE>
__global__ __launch_bounds__(LONG_NT) void k_cat_long_grad(CatArgs p, int splits, const float* stats) {
    constexpr int V = 16 / sizeof(T);
    const size_t s_id = blockIdx.x / splits;
    const int piece = blockIdx.x % splits;
    const size_t b = s_id / p.A;
    const int a = (int)(s_id % p.A);
    const int k = chosen_in(p, s_id);
    float m = 0.f, s = 0.f, g = MODE == CAT_BWD ? p.dlogp[b] : 0.f;
    const bool on = MODE == CAT_PPO ? row_weight(p, b) != 0.0 : g != 0.f;
    if (on) join_pieces(stats + s_id * splits * 2, splits, m, s);
    if (MODE == CAT_PPO) {
        HeadTerms t = {0.0, 0.0, 0.0};
        double lp = 0.0;
        if (on) {
            lp = segment_logp<T>(p, b, 0, m, s);
            g = (float)policy_head(lp, head_row(p.head, b), p.head, t);
        }
        if (piece == 0 && threadIdx.x == 0) {
            p.logp[b] = (float)lp;
            p.part[b * 3] = t.policy;
            p.part[b * 3 + 1] = t.kl;
            p.part[b * 3 + 2] = t.clipped;
        }
    }
    int lo, hi;
    piece_of(p, splits, piece, V, lo, hi);
    const T* l = static_cast<const T*>(p.logits) + b * p.ld + (size_t)a * p.N;
    T* d = static_cast<T*>(p.dlogits) + b * p.ldd + (size_t)a * p.N;
    const bool live = on && k >= 0 && s != 0.f && g != 0.f;
    const NegProb<T> np(m, g, live ? 1.f / s : 0.f);
    const float gi = live ? g * (1.f / s) : 0.f;
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
            for (int i = 0; i < V; ++i) v[i] = np(to_f32(t[i]));
            if (k >= n && k < n + V) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (n + i == k) v[i] = g - exp_below_exact(to_f32(t[i]), m) * gi;
            }
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
        const float x = live ? to_f32(l[n]) : 0.f;
        float v = !live ? 0.f : n == k ? g - exp_below_exact(x, m) * gi : np(x);
        if (acc) v += to_f32(d[n]);
        d[n] = from_f32<T>(v);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------
static int lanes_per_row(int A) { return A <= 2 ? 1 : A <= 8 ? 4 : A <= 64 ? 16 : 64; }

template <typename T, int MODE, int G, int E, int IT, int NT>
static int launch_rows(CatArgs p, int rb, hipStream_t st) {
    const long long widest = p.ld > p.ldd ? p.ld : p.ldd;
    while (!p.loss4 && rb > 1 && (long long)rb * widest * (long long)sizeof(T) >= (1ll << 31)) rb = (rb + 1) / 2;
    const long long blocks = ((long long)p.B + rb - 1) / rb;
    if (blocks > (long long)MAX_BLOCKS) return -1;
    p.rows_per_block = rb;
    p.lanes_per_row = lanes_per_row(p.A);
    const size_t lds = MODE == CAT_BWD ? 0 : (size_t)rb * p.A * 16 + (size_t)rb * (3 * sizeof(double) + 4 * sizeof(float)) +
                                              (size_t)(IT / 2) * E * NT * sizeof(float);
    if (lds > (64u << 10) && hipFuncSetAttribute(reinterpret_cast<const void*>(&k_cat_rows<T, MODE, G, E, IT, NT>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
        return -1;
    hipLaunchKernelGGL((k_cat_rows<T, MODE, G, E, IT, NT>), dim3((unsigned)blocks), dim3(NT), lds, st, p);
    return (int)blocks;
}

// whole rows a block takes: `segments` of them at most (one row always), fewer while the chip is not full (four blocks a CU)
static int rows_of(const CatArgs& p, int segments, int nt, bool head) {
    int rb = segments / p.A;
    if (head && rb > nt / lanes_per_row(p.A)) rb = nt / lanes_per_row(p.A);
    const int by_chip = (int)(((long long)p.B + 1023) / 1024);
    if (rb > by_chip) rb = by_chip;
    return rb < 1 ? 1 : rb;
}

template <typename T, int MODE, int G, int E>
static int launch_axis(CatArgs& p, hipStream_t st) {
    constexpr int NG = 256 / G;
    if constexpr (MODE != CAT_PPO) {
        return launch_rows<T, MODE, G, E, 0, 256>(p, rows_of(p, 4 * NG, 256, MODE == CAT_FWD), st);
    } else {
        // a small batch: one block, which finishes the loss itself.  (Only while the block holds its exponentials: 32 x 36 x 35, two
        // readings by one block, took 14.8 us against 6.2 + 3.2 us on five blocks and the finishing launch.)
        if (p.loss4 && p.B <= 1024 / lanes_per_row(p.A) && p.B * p.A <= 4 * (1024 / G) &&
            (long long)p.B * (p.ld > p.ldd ? p.ld : p.ldd) * (long long)sizeof(T) < (1ll << 31))
            return launch_rows<T, MODE, G, E, 4, 1024>(p, p.B, st);
        p.loss4 = nullptr;
        // the exponentials of four segments a group stay in registers: rows of up to 4 * 32 (1024 threads: 128) of its segments
        if (p.A <= 4 * NG) return launch_rows<T, MODE, G, E, 4, 256>(p, rows_of(p, 4 * NG, 256, true), st);
        if (p.A <= 16 * NG) return launch_rows<T, MODE, G, E, 4, 1024>(p, 1, st);
        return launch_rows<T, MODE, G, E, 0, 256>(p, 1, st);
    }
}

// groups of lanes by the axis: few idle slots (35 particles: 8 lanes x 5 = 40), 16 bytes or more a lane where that can be
template <typename T, int MODE>
static int pick_rows(CatArgs& p, hipStream_t st) {
    const int N = p.N;
    if (N <= 4) return launch_axis<T, MODE, 4, 1>(p, st);
    if (N <= 8) return launch_axis<T, MODE, 2, 4>(p, st);
    if (N <= 16) return launch_axis<T, MODE, 4, 4>(p, st);
    if (N <= 24) return launch_axis<T, MODE, 4, 6>(p, st);
    if (N <= 32) return launch_axis<T, MODE, 8, 4>(p, st);
    if (N <= 40) return launch_axis<T, MODE, 8, 5>(p, st);
    if (N <= 64) return launch_axis<T, MODE, 8, 8>(p, st);
    if (N <= 96) return launch_axis<T, MODE, 16, 6>(p, st);
    if (N <= 128) return launch_axis<T, MODE, 16, 8>(p, st);
    if (N <= 192) return launch_axis<T, MODE, 32, 6>(p, st);
    if (N <= 256) return launch_axis<T, MODE, 32, 8>(p, st);
    if (N <= 384) return launch_axis<T, MODE, 64, 6>(p, st);
    if (N <= 512) return launch_axis<T, MODE, 64, 8>(p, st);
    return launch_axis<T, MODE, 64, 16>(p, st);
}

template <typename T, int MODE, int H, int NT>
static void launch_held(const CatArgs& p, hipStream_t st) {
    hipLaunchKernelGGL((k_cat_long_held<T, MODE, H, NT>), dim3((unsigned)((size_t)p.B * p.A)), dim3(NT), 0, st, p);
}

template <typename T, int MODE>
int run_cat(CatArgs p, void* ws, size_t ws_bytes, size_t* nparts, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    p.magic_A = p.A > 1 ? (uint32_t)((0x100000000ull + p.A - 1) / p.A) : 0;
    const size_t parts = MODE == CAT_PPO ? (size_t)p.B * 3 * sizeof(double) : 0;
    if (parts && (!ws || ws_bytes < parts)) return PFPN_ERR_WORKSPACE;
    p.part = static_cast<double*>(ws);
    p.stream = (size_t)p.B * p.A * p.N * sizeof(T) > (256u << 20);
    if (p.N <= CAT_SHORT_N) {
        const int blocks = pick_rows<T, MODE>(p, st);
        if (blocks < 0) return PFPN_ERR_ARG;
        *nparts = p.loss4 ? 0 : blocks;         // (0: nothing is left to add up)
        PFPN_CHECK_LAUNCH();
        return PFPN_OK;
    }
    *nparts = p.B;
    const size_t segs = (size_t)p.B * p.A;
    const int S = cat_splits(p.B, p.A, p.N);
    if (segs * S > MAX_BLOCKS) return PFPN_ERR_ARG;
    const size_t pieces = segs * S;
    if (!ws || ws_bytes < parts + pieces * 2 * sizeof(float) + (MODE == CAT_PPO ? (size_t)p.B * sizeof(float) : 0))
        return PFPN_ERR_WORKSPACE;
    // A row held whole by one block takes one launch, pieces two or three.  One row of 8192 logits, float32, log-prob / gradient:
    // 2.6 / 3.3 us held, 4.7 / 6.3 us in pieces; of 32768: 3.5 / 5.7 against 4.7 / 6.5; of 65536: 4.8 / 8.9 against 4.8 / 6.7, and
    // 128 rows of 65536: 5.9 / 15.3 against 9.8 / 20.7 us.
    if ((p.A == 1 || MODE == CAT_BWD) && p.N <= 1024 * 16 * V && (S == 1 || p.N <= 32768 || segs >= 128)) {
        // (fewest idle slots: 32736 x 1025 bfloat16 by 256 threads, most of whose slots are idle: log-prob 63 us, gradient 71 us; by 64 threads 23 and 31 us)
        if (p.N <= 64 * 4 * V) launch_held<T, MODE, 4, 64>(p, st);
        else if (p.N <= 128 * 4 * V) launch_held<T, MODE, 4, 128>(p, st);
        else if (p.N <= 256 * 4 * V) launch_held<T, MODE, 4, 256>(p, st);
        else if (p.N <= 512 * 4 * V) launch_held<T, MODE, 4, 512>(p, st);
        else if (p.N <= 1024 * 4 * V) launch_held<T, MODE, 4, 1024>(p, st);
        else if (p.N <= 1024 * 8 * V) launch_held<T, MODE, 8, 1024>(p, st);
        else launch_held<T, MODE, 16, 1024>(p, st);
        PFPN_CHECK_LAUNCH();
        return PFPN_OK;
    }
    float* stats = reinterpret_cast<float*>(static_cast<char*>(ws) + parts);
    hipLaunchKernelGGL((k_cat_long_stats<T>), dim3((unsigned)pieces), dim3(LONG_NT), 0, st, p, S, MODE, stats);
    constexpr int ROWS = MODE == CAT_PPO ? CAT_PPO : CAT_FWD;
    if (MODE == CAT_FWD || (MODE == CAT_PPO && p.A > 1)) {
        float* row_g = stats + pieces * 2;
        hipLaunchKernelGGL((k_cat_long_rows<T, ROWS>), dim3(p.B), dim3(p.A < 4 ? 64 : LONG_NT), 0, st, p, S, (const float*)stats, row_g);
        p.dlogp = row_g;
    }
    if (MODE == CAT_PPO && p.A == 1)
        hipLaunchKernelGGL((k_cat_long_grad<T, CAT_PPO>), dim3((unsigned)pieces), dim3(LONG_NT), 0, st, p, S, (const float*)stats);
    else if (MODE != CAT_FWD)
        hipLaunchKernelGGL((k_cat_long_grad<T, CAT_BWD>), dim3((unsigned)pieces), dim3(LONG_NT), 0, st, p, S, (const float*)stats);
    PFPN_CHECK_LAUNCH();
    return PFPN_OK;
}

template int run_cat<PFPN_CATEGORICAL_TYPE, CAT_FWD>(CatArgs, void*, size_t, size_t*, hipStream_t);
template int run_cat<PFPN_CATEGORICAL_TYPE, CAT_BWD>(CatArgs, void*, size_t, size_t*, hipStream_t);
template int run_cat<PFPN_CATEGORICAL_TYPE, CAT_PPO>(CatArgs, void*, size_t, size_t*, hipStream_t);

#endif  // PFPN_CATEGORICAL_TYPE

}  // namespace pfpn
