// Shared device pieces of the policy-objective kernels (categorical log-probs, clipped loss with a KL term, balance loss):
// logit types, unaligned wide loads, reductions over groups of lanes, the loss head of one row.
#pragma once
#include "pfpn_common.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace pfpn {

// dtype codes of the C ABI
enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };

struct bf16_t { uint16_t u; };
struct f16_t { uint16_t u; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return __uint_as_float((uint32_t)v.u << 16); }
__device__ __forceinline__ float to_f32(f16_t v) { return (float)__builtin_bit_cast(_Float16, v.u); }
// one rounding, to nearest even: the only one between a gradient's 32-bit value and its 16-bit tensor
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float v) {
    return bf16_t{__builtin_bit_cast(uint16_t, (__bf16)v)};
}
template <> __device__ __forceinline__ f16_t from_f32<f16_t>(float v) {
    return f16_t{__builtin_bit_cast(uint16_t, (_Float16)v)};
}

template <typename T> struct Bits { typedef uint16_t type; };
template <> struct Bits<float> { typedef uint32_t type; };

// V elements loaded / stored at once from an address that is only element-aligned (rows of an odd length start anywhere;
// gfx950 global accesses take any alignment, and hipcc emits the wide form for a packed struct)
template <typename T, int V>
struct __attribute__((packed, aligned(alignof(T)))) Pack { T v[V]; };

template <typename T, int V>
__device__ __forceinline__ void load_pack(const T* p, T (&out)[V]) {
    const Pack<T, V> t = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = t.v[i];
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const T (&in)[V]) {
    Pack<T, V> t;
#pragma unroll
    for (int i = 0; i < V; ++i) t.v[i] = in[i];
    *reinterpret_cast<Pack<T, V>*>(p) = t;
}
// ... past the caches (gradients larger than the infinity cache: nobody finds them there)
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const T (&in)[V], bool stream) {
    if (stream && (V * sizeof(T)) % 16 == 0) {
        typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
        Pack<T, V> t;
#pragma unroll
        for (int i = 0; i < V; ++i) t.v[i] = in[i];
        const Words* w = reinterpret_cast<const Words*>(&t);
#pragma unroll
        for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i) __builtin_nontemporal_store(w[i], reinterpret_cast<Words*>(p) + i);
    } else {
        store_pack<T, V>(p, in);
    }
}

// Wide loads kept in registers as they came, for several passes: `forget` makes the compiler convert them anew in the next
// pass (it would keep the 32-bit values of 16-bit logits alive, twice the registers).
template <typename T, int V>
struct Held {
    static constexpr int W = V * sizeof(T) / 4;
    uint32_t w[W];
    __device__ __forceinline__ void load(const T* p) {
        struct __attribute__((packed, aligned(alignof(T)))) Words { uint32_t w[W]; };
        const Words t = *reinterpret_cast<const Words*>(p);
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = t.w[i];
    }
    __device__ __forceinline__ void fill(uint32_t v) {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = v;
    }
    __device__ __forceinline__ void forget() {
#pragma unroll
        for (int i = 0; i < W; ++i) asm("" : "+v"(w[i]));
    }
    __device__ __forceinline__ float operator[](int i) const {
        if (sizeof(T) == 4) return __uint_as_float(w[i]);
        const uint32_t h = (i & 1) ? w[i / 2] >> 16 : w[i / 2] & 0xffffu;
        return to_f32(__builtin_bit_cast(T, (typename Bits<T>::type)h));
    }
};

// Running maximum of held logits: two 16-bit ones an instruction (bfloat16 as integers in the same order; a NaN may be passed
// over here, it reaches the sum)
template <typename T> struct HeldMax;
template <> struct HeldMax<float> {
    float m = -INFINITY;
    __device__ __forceinline__ void take(uint32_t w) { m = fmaxf(m, __uint_as_float(w)); }
    __device__ __forceinline__ float value() const { return m; }
};
template <> struct HeldMax<f16_t> {
    typedef _Float16 Pair __attribute__((ext_vector_type(2)));
    Pair m = {(_Float16)-INFINITY, (_Float16)-INFINITY};
    __device__ __forceinline__ void take(uint32_t w) { m = __builtin_elementwise_max(m, __builtin_bit_cast(Pair, w)); }
    __device__ __forceinline__ float value() const { return fmaxf((float)m[0], (float)m[1]); }
};
template <> struct HeldMax<bf16_t> {
    typedef short Pair __attribute__((ext_vector_type(2)));
    Pair m = {(short)0x8000, (short)0x8000};
    static __device__ __forceinline__ Pair ordered(Pair v) { return v ^ ((v >> 15) & (short)0x7fff); }
    __device__ __forceinline__ void take(uint32_t w) { m = __builtin_elementwise_max(m, ordered(__builtin_bit_cast(Pair, w))); }
    __device__ __forceinline__ float value() const {
        const Pair v = ordered(m);
        return fmaxf(to_f32(bf16_t{(uint16_t)v[0]}), to_f32(bf16_t{(uint16_t)v[1]}));
    }
};

// Reductions over aligned groups of G lanes (2 .. 64), every lane gets the result, no LDS round trip: quad_perm xor 1, xor 2,
// row_half_mirror (quads of a half row), row_mirror (half rows), then gfx950's row / half-wave swaps.
template <int CTRL>
__device__ __forceinline__ uint32_t lane_move(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int G, typename F>
__device__ __forceinline__ uint32_t group_reduce(uint32_t v, F op) {
    if (G > 1) v = op(v, lane_move<0xB1>(v));
    if (G > 2) v = op(v, lane_move<0x4E>(v));
    if (G > 4) v = op(v, lane_move<0x141>(v));
    if (G > 8) v = op(v, lane_move<0x140>(v));
    if (G > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = op(r[0], r[1]);
    }
    if (G > 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = op(r[0], r[1]);
    }
    return v;
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
    return __uint_as_float(group_reduce<G>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
    return __uint_as_float(group_reduce<G>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
// (64 bits: both halves move, where a shuffle through LDS takes six round trips)
__device__ __forceinline__ double halves(uint32_t lo, uint32_t hi) {
    return __longlong_as_double((long long)((unsigned long long)hi << 32 | lo));
}
template <int CTRL>
__device__ __forceinline__ double add_moved(double v) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(v);
    const uint32_t lo = lane_move<CTRL>((uint32_t)b), hi = lane_move<CTRL>((uint32_t)(b >> 32));
    return v + halves(lo, hi);
}
template <int G>
__device__ __forceinline__ double group_sum(double v) {
    if (G > 1) v = add_moved<0xB1>(v);
    if (G > 2) v = add_moved<0x4E>(v);
    if (G > 4) v = add_moved<0x141>(v);
    if (G > 8) v = add_moved<0x140>(v);
    if (G > 16) {
        const unsigned long long b = (unsigned long long)__double_as_longlong(v);
        const auto l = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false);
        const auto h = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
        v = halves(l[0], h[0]) + halves(l[1], h[1]);
    }
    if (G > 32) {
        const unsigned long long b = (unsigned long long)__double_as_longlong(v);
        const auto l = __builtin_amdgcn_permlane32_swap((uint32_t)b, (uint32_t)b, false, false);
        const auto h = __builtin_amdgcn_permlane32_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
        v = halves(l[0], h[0]) + halves(l[1], h[1]);
    }
    return v;
}
template <int G>
__device__ __forceinline__ uint32_t group_min(uint32_t v) {
    return group_reduce<G>(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}

// Sum over the lanes of a wave that stand at the same place of their groups of G (every lane gets it): rotations inside the rows of
// 16, then the row and half-wave swaps.
template <int G, typename F>
__device__ __forceinline__ uint32_t across_groups(uint32_t v, F op) {
    if (G < 16) v = op(v, lane_move<0x128>(v));
    if (G < 8) v = op(v, lane_move<0x124>(v));
    if (G < 4) v = op(v, lane_move<0x122>(v));
    if (G < 2) v = op(v, lane_move<0x121>(v));
    if (G < 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = op(r[0], r[1]);
    }
    if (G < 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = op(r[0], r[1]);
    }
    return v;
}

// exp(x - m): the difference first (exact where it matters: near the maximum), then ONE v_exp_f32
__device__ __forceinline__ float exp_below(float x, float m) {
    return __builtin_amdgcn_exp2f((x - m) * PFPN_LOG2E);
}
// the same with log2(e) in two parts (float32's own is off by 1.3e-8, always to the same side: 128 choices add that up)
__device__ __forceinline__ float exp_below_exact(float x, float m) {
    const float d = x - m;
    return __builtin_amdgcn_exp2f(__builtin_fmaf(d, PFPN_LOG2E, d * 1.92596299e-8f));
}

// ---- a short axis (N <= 1024) over a group of G lanes: U packs of V consecutive categories a lane -------------------------------
// Pack u of lane j is the segment's pack u G + j: a pack is one wide access from any alignment, the lanes' packs lie side by side.
// The segment's last pack is moved down to end at N, so that every access is whole and inside the segment (V <= N): its first
// categories then belong to the pack before, `own` says which count.
template <typename T, int G, int E>
struct Axis {
    static constexpr int V = E * sizeof(T) <= 24 ? E : 16 / (int)sizeof(T), U = E / V;
    static_assert(U * V == E, "whole packs");
    int j, N;
    __device__ __forceinline__ Axis(int j_, int N_) : j(j_), N(N_) {}
    __device__ __forceinline__ int lo(int u) const { return (u * G + j) * V; }
    __device__ __forceinline__ bool has(int u) const { return lo(u) < N; }
    __device__ __forceinline__ int start(int u) const { return lo(u) < N - V ? lo(u) : N - V; }
    __device__ __forceinline__ int at(int e) const { return start(e / V) + e % V; }                     // category of element e
    __device__ __forceinline__ bool own(int e) const { return has(e / V) && at(e) >= lo(e / V); }
    // (packs past the axis read its last one again: no branch, so that all loads of a thread are in flight together)
    __device__ __forceinline__ void load(const T* segment, T (&raw)[E]) const {
#pragma unroll
        for (int u = 0; u < U; ++u) load_pack<T, V>(segment + start(u), reinterpret_cast<T (&)[V]>(raw[u * V]));
    }
    __device__ __forceinline__ void store(T* segment, const T (&o)[E], bool stream) const {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (has(u)) store_pack<T, V>(segment + start(u), reinterpret_cast<const T (&)[V]>(o[u * V]), stream);
    }
};

// ---- the loss head of one row ---------------------------------------------------------------------------------------
// a = clip((adv - mean) * rstd), r = exp(logp - logp_old), d = logp_ref - logp,
// loss_row = w (-min(r a, clip(r) a) + c (exp(d) - 1 - d)),   d loss / d logp = w ([not clipped] (-a r) - c (exp(d) - 1)).
// The log-probs of a choice under two policies may lie hundreds apart (a joint log-prob of many dimensions is some hundreds):
// differences, exponentials and products are 64-bit, so that a ratio beyond float32 under a small weight, or an advantage of zero,
// gives the loss and gradient it has.  exp(d) - 1 - d = d^2 / 2 + ... by its series where it would cancel.
struct HeadArgs {
    const float* logp_old;
    const float* adv;
    const float* logp_ref;      // optional
    const float* weight;        // optional: 1 / B each
    const float* stats;         // optional: {mean, rstd, clip_lo, clip_hi}
    double clip_lo, clip_hi;    // bounds of the ratio
    double kl_coef;
    double inv_B;
};
struct HeadRow {
    float logp_old, a, logp_ref;
    double w;
};
struct HeadTerms {
    double policy, kl, clipped;
};

__device__ __forceinline__ HeadRow head_row(const HeadArgs& h, size_t b) {
    HeadRow r;
    r.logp_old = h.logp_old[b];
    r.a = h.adv[b];
    r.logp_ref = h.logp_ref ? h.logp_ref[b] : 0.f;
    r.w = h.weight ? (double)h.weight[b] : h.inv_B;
    if (h.stats) r.a = clip_adv((r.a - h.stats[0]) * h.stats[1], h.stats[2], h.stats[3]);
    return r;
}

// exp(d) - 1 - d; em1 = exp(d) - 1.  |d| < 1: d^2 sum_k d^k / (k + 2)!, the sum in 32 bits (a few 2^-24 of itself), the first term left
// out under 2^-28 of it
__device__ __forceinline__ double kl_sample(double d, double& em1) {
    if (fabs(d) < 1.0) {
        const float x = (float)d;
        float q = 1.f / 6227020800.f;
        q = __builtin_fmaf(q, x, 1.f / 479001600.f);
        q = __builtin_fmaf(q, x, 1.f / 39916800.f);
        q = __builtin_fmaf(q, x, 1.f / 3628800.f);
        q = __builtin_fmaf(q, x, 1.f / 362880.f);
        q = __builtin_fmaf(q, x, 1.f / 40320.f);
        q = __builtin_fmaf(q, x, 1.f / 5040.f);
        q = __builtin_fmaf(q, x, 1.f / 720.f);
        q = __builtin_fmaf(q, x, 1.f / 120.f);
        q = __builtin_fmaf(q, x, 1.f / 24.f);
        q = __builtin_fmaf(q, x, 1.f / 6.f);
        q = __builtin_fmaf(q, x, 0.5f);
        const double kl = (double)q * d * d;
        em1 = d + kl;
        return kl;
    }
    em1 = exp(d) - 1.0;
    return em1 == INFINITY ? em1 : em1 - d;         // (an impossible choice: infinite, not inf - inf)
}

// -> d loss / d logp of a row of weight != 0; its terms
__device__ __forceinline__ double policy_head(double logp, const HeadRow& row, const HeadArgs& h, HeadTerms& t) {
    const double r = exp(logp - (double)row.logp_old), a = (double)row.a;
    const double held_r = r < h.clip_lo ? h.clip_lo : (r > h.clip_hi ? h.clip_hi : r);
    const double sur = a == 0.0 && r > 1.0 ? 0.0 : r * a;              // (no advantage, no surrogate: not inf * 0)
    const double held = held_r * a;
    const bool clipped = held < sur;
    double g = clipped ? 0.0 : -sur;
    double kl = 0.0;
    if (h.logp_ref) {
        double em1;
        kl = kl_sample((double)row.logp_ref - logp, em1);
        if (h.kl_coef != 0.0) g -= h.kl_coef * em1;                // (a term that is only reported may be infinite)
    }
    t.policy = row.w * (clipped ? -held : -sur);
    t.kl = row.w * kl;
    t.clipped = clipped ? row.w : 0.0;
    return row.w * g;
}

// per-block sums {policy, kl, clipped} -> part[3]; `red` needs 3 * 16 doubles of LDS.  Fixed order.
__device__ __forceinline__ void block_terms(const HeadTerms& t, double* red, double* part) {
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, nw = (blockDim.x + 63) >> 6;
    const double a = group_sum<64>(t.policy), b = group_sum<64>(t.kl), c = group_sum<64>(t.clipped);
    __syncthreads();
    if (lane == 0) { red[wid * 3] = a; red[wid * 3 + 1] = b; red[wid * 3 + 2] = c; }
    __syncthreads();
    if (threadIdx.x < 3) {
        double s = 0.0;
        for (int i = 0; i < nw; ++i) s += red[i * 3 + threadIdx.x];
        part[threadIdx.x] = s;
    }
}

// n triples of terms, `step` triples apart, added by one block of 15 waves, five a term, sixteen loads of a lane in flight; out[3] in
// LDS, fixed order.  One CU reads 8190 triples in 5.6 us, 32736 in 19 us, 200000 in 143 us: past FOLD_FROM of them `fold_terms`
// first adds every FOLD into the first of them (a launch that fills the chip); returns the distance of what is left, n its number.
constexpr size_t FOLD = 512, FOLD_FROM = 8192;
int fold_terms(double* part, size_t& n, hipStream_t st);
constexpr int FINISH_NT = 960;
__device__ __forceinline__ void sum_terms(const double* __restrict__ part, size_t n, int step, double* out) {
    constexpr int LANES = FINISH_NT / 3, DEEP = 16;
    __shared__ double red[15];
    const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63, term = wid % 3;
    double s = 0.0;
    for (size_t i = (size_t)(wid / 3) * 64 + lane; i < n; i += LANES * DEEP) {
        double t[DEEP];
#pragma unroll
        for (int k = 0; k < DEEP; ++k) {
            const size_t j = i + LANES * k;
            t[k] = part[(j < n ? j : i) * step * 3 + term];
        }
#pragma unroll
        for (int k = 0; k < DEEP; ++k) s += i + LANES * k < n ? t[k] : 0.0;
    }
    s = group_sum<64>(s);
    if (lane == 0) red[wid] = s;
    __syncthreads();
    if (threadIdx.x < 3) {
        s = red[threadIdx.x];
        for (int k = 1; k < 5; ++k) s += red[3 * k + threadIdx.x];
        out[threadIdx.x] = s;
    }
    __syncthreads();
}

}  // namespace pfpn
