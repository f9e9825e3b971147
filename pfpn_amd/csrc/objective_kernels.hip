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
// Bound: HBM / cache (12-16 bytes a step) for long segments; 1500 pairs of 3000017 steps: 15.0 us + 3.8 us for the sum of the pairs =
// 3.2 TB/s, held back by what a block does once (bounds, 64-bit sums across lanes, the head: its instructions issue for 4.2 us of the 15,
// waves wait for half of their time): 128 threads a pair 18.5 us, 512 15.0 us, 256 15.3 us with half the waves.  Two kernels, sums and
// gradients, took 38 us.  24 pairs: 4.9 us, one block, one launch (was 9 us).
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
    double* sums;               // [P][splits]
    double* terms;              // [P][3] = loss, margin > 0, margin
    int splits;
};

// A pair's two segments lie side by side: rows [lo, mid) count for it, [mid, hi) against it.  Bounds are clamped to the vectors
// and to ascend within the pair, so that nothing outside is touched whatever they hold (bounds that descend from one pair to the
// next make pairs share rows, whose gradient is then one of theirs).
struct PairRows {
    long long lo, mid, hi;
};
__device__ __forceinline__ long long clamped(long long v, long long lo, long long hi) { return v < lo ? lo : (v > hi ? hi : v); }
__device__ __forceinline__ PairRows rows_of_pair(const PrefArgs& p, int pair) {
    const long long* o = p.offsets + 2 * (size_t)pair;
    PairRows r;
    const long long a = o[0], b = o[1], c = o[2];
    r.lo = clamped(a, 0, p.T);
    r.mid = clamped(b, r.lo, p.T);
    r.hi = clamped(c, r.mid, p.T);
    return r;
}
// piece `part` of `splits` of rows [lo, hi)
__device__ __forceinline__ void piece_of_pair(const PrefArgs& p, const PairRows& r, int part, long long& lo, long long& hi) {
    const long long width = (r.hi - r.lo + p.splits - 1) / p.splits;
    lo = r.lo + part * width < r.hi ? r.lo + part * width : r.hi;
    hi = lo + width < r.hi ? lo + width : r.hi;
}
// +- w (logp - logp_ref) of one step; a step of weight 0: 0, whatever stands there
__device__ __forceinline__ double step_gap(float lp, float ref, float w, bool against) {
    const double d = w == 0.f ? 0.0 : ((double)lp - (double)ref) * (double)w;
    return against ? -d : d;
}
// a thread's share of rows [lo, hi): four steps a load (from any alignment), `id` of `n` threads
__device__ __forceinline__ double span_sum(const PrefArgs& p, long long lo, long long hi, long long mid, int id, int n) {
    double v = 0.0;
    const long long full = lo + (hi - lo) / 4 * 4;
    for (long long t = lo + 4ll * id; t < full; t += 4ll * n) {
        float a[4], r[4] = {0.f, 0.f, 0.f, 0.f}, w[4] = {1.f, 1.f, 1.f, 1.f};
        load_pack<float, 4>(p.logp + t, a);
        if (p.logp_ref) load_pack<float, 4>(p.logp_ref + t, r);
        if (p.weight) load_pack<float, 4>(p.weight + t, w);
        v += (step_gap(a[0], r[0], w[0], t >= mid) + step_gap(a[1], r[1], w[1], t + 1 >= mid)) +
             (step_gap(a[2], r[2], w[2], t + 2 >= mid) + step_gap(a[3], r[3], w[3], t + 3 >= mid));
    }
    const long long t = full + id;
    if (t < hi) v += step_gap(p.logp[t], p.logp_ref ? p.logp_ref[t] : 0.f, p.weight ? p.weight[t] : 1.f, t >= mid);
    return v;
}
// ... and its share of their gradients
__device__ __forceinline__ float step_grad(double g, float w) { return w == 0.f ? 0.f : (float)(g * (double)w); }
__device__ __forceinline__ void span_grad(const PrefArgs& p, long long lo, long long hi, long long mid, int id, int n, double g) {
    const long long full = lo + (hi - lo) / 4 * 4;
    for (long long t = lo + 4ll * id; t < full; t += 4ll * n) {
        float d[4], w[4] = {1.f, 1.f, 1.f, 1.f};
        if (p.weight) load_pack<float, 4>(p.weight + t, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = step_grad(t + i >= mid ? -g : g, w[i]);
        store_pack<float, 4>(p.dlogp + t, d);
    }
    const long long t = full + id;
    if (t < hi) p.dlogp[t] = step_grad(t >= mid ? -g : g, p.weight ? p.weight[t] : 1.f);
}
// rows outside every segment, before the first pair's and behind the last pair's, have no gradient
__device__ __forceinline__ void outside_zero(const PrefArgs& p, long long id, long long n) {
    const long long first = rows_of_pair(p, 0).lo, last = rows_of_pair(p, p.P - 1).hi;
    for (long long t = id; t < first; t += n) p.dlogp[t] = 0.f;
    for (long long t = last + id; t < p.T; t += n) p.dlogp[t] = 0.f;
}

// A pair's head, in 64 bits: e sigma(m) - (1 - e) sigma(-m) cancels near its zero, and an exponential in 32 is off by |m| 2^-24 of
// itself.  Both halves of it from ONE exponential of -|m|; log sigma(m) = -softplus(-m).
// d loss / d delta, of the mean over the pairs; z = e^-|margin|
__device__ __forceinline__ double pair_slope(const PrefArgs& p, double delta, double& z) {
    z = 0.0;
    if (p.kind) return 2.0 * (delta - 0.5 / p.beta) / (double)p.P;
    const double m = p.beta * delta, e = p.smoothing;
    z = exp(-fabs(m));
    const double near = 1.0 / (1.0 + z), far = z * near;
    return p.beta * (m >= 0 ? e * near - (1.0 - e) * far : e * far - (1.0 - e) * near) / (double)p.P;
}
// log(1 + z), z in [0, 1]: 2 artanh(z / (2 + z)), whose argument is 1/3 at most: the first term left out is under 2^-40 of the sum
__device__ __forceinline__ double log_one_plus(double z) {
    const double s = z / (2.0 + z), q = s * s;
    double t = 1.0 / 23.0;
#pragma unroll
    for (int k = 21; k > 0; k -= 2) t = __builtin_fma(t, q, 1.0 / k);
    return 2.0 * s * t;
}
// {loss, margin > 0, margin}, and the pair's margin
__device__ __forceinline__ void pair_terms(const PrefArgs& p, int pair, double delta, double z, double* terms) {
    const double m = p.beta * delta;
    double loss;
    if (p.kind == 0) {
        const double e = p.smoothing, am = fabs(m), l = log_one_plus(z);
        loss = (1.0 - e) * (l + (m < 0 ? am : 0.0)) + (e > 0 ? e * (l + (m > 0 ? am : 0.0)) : 0.0);     // (infinite margin: 0, not 0 * inf)
    } else {
        const double u = delta - 0.5 / p.beta;
        loss = u * u;
    }
    p.margin[pair] = (float)m;
    terms[0] = loss;
    terms[1] = m > 0 ? 1.0 : 0.0;
    terms[2] = m;
}

// Few steps: ONE block, a wave per pair in turn.  It saves a launch, 2 us of a call's 14 on the host, as long as its own time stays under
// the call's (us by one block / by the general forms, in a graph): 24 pairs of 100 steps 4.6 / 4.6, 16 of 1000 6.6 / 4.7, 64 of 256
// 9.0 / 4.7, all in calls of 12 / 14; 1 of 2000 6.1 / 4.6.  Beyond, it costs more: 128 of 64 15.8 / 5.1, 1 of 16384 32 / 12.
constexpr int PREF_SMALL_P = 64, PREF_SMALL_T = 16384, PREF_SMALL_MEAN = 2048;
// PREF_SHORT: up to so many steps a pair, many pairs go by lanes (16 up to 128 steps, else 64), not by blocks, with the blocks' terms
// summed: from three times as many pairs as steps on there are lanes enough to fill the chip.  By lanes / by blocks: 20000 pairs of 20
// 11.5 / 35, of 100 13.1 / 38, of 300 31 / 42; 3000 of 300 10.6 / 12.5, of 1000 14.4 / 15.2; 600 of 300 8.6 / 8.8, of 600 9.1 / 9.1;
// fewer: 600 of 1000 9.6 / 9.2, 1500 of 1000 11.4 / 10.9, 200 of 1000 9.0 / 8.0.
constexpr int PREF_SHORT = 1024;
__global__ __launch_bounds__(1024) void k_pref_small(PrefArgs p, float* __restrict__ loss3) {
    __shared__ double terms[PREF_SMALL_P * 3], gap[PREF_SMALL_P];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    for (int pair = wid; pair < p.P; pair += 16) {
        const PairRows r = rows_of_pair(p, pair);
        const double delta = group_sum<64>(span_sum(p, r.lo, r.hi, r.mid, lane, 64));
        if (lane == 0) gap[pair] = delta;
    }
    outside_zero(p, threadIdx.x, 1024);
    __syncthreads();
    // (a thread a pair: a wave that runs its pairs' heads in turn takes 1 us for each)
    double delta = 0.0, z = 0.0;
    if ((int)threadIdx.x < p.P) {
        delta = gap[threadIdx.x];
        gap[threadIdx.x] = pair_slope(p, delta, z);
    }
    __syncthreads();
    for (int pair = wid; pair < p.P; pair += 16) {
        const PairRows r = rows_of_pair(p, pair);
        span_grad(p, r.lo, r.hi, r.mid, lane, 64, gap[pair]);
    }
    if ((int)threadIdx.x < p.P) pair_terms(p, threadIdx.x, delta, z, terms + threadIdx.x * 3);
    __syncthreads();
    if (wid < 3) {
        double t = 0.0;
        for (int i = lane; i < p.P; i += 64) t += terms[i * 3 + wid];
        t = group_sum<64>(t);
        if (lane == 0) loss3[wid] = (float)(t / (double)p.P);
    }
}

// Pairs that fill a block: a block per pair, sums and gradients in one launch.
__global__ __launch_bounds__(256) void k_pref_pairs(PrefArgs p) {
    __shared__ double red[4];
    if (blockIdx.x >= (unsigned)p.P) {
        outside_zero(p, (long long)(blockIdx.x - p.P) * 256 + threadIdx.x, (long long)(gridDim.x - p.P) * 256);
        return;
    }
    const PairRows r = rows_of_pair(p, blockIdx.x);
    constexpr int H = 4;
    if (r.hi - r.lo >= 4 * 256 && r.hi - r.lo < 4 * 256 * H) {
        // all of the pair's steps in flight at once (packs past the end: the last one again), the weights held for the gradients:
        // 3000 pairs of 4095 steps 41 -> 33 us; pairs of 1000, which would read the last pack three times, 9.5 -> 11.1 us
        const int steps = (int)(r.hi - r.lo), mid = (int)(r.mid - r.lo), packs = steps / 4, tail = packs * 4 + (int)threadIdx.x;
        const float *lp = p.logp + r.lo, *ref = p.logp_ref + r.lo, *wt = p.weight + r.lo;
        float a[H][4], q[H][4] = {}, w[H][4], at = 0.f, qt = 0.f, wl = 1.f;
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) w[h][i] = 1.f;
        int where[H];
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const int i = h * 256 + (int)threadIdx.x;
            where[h] = 4 * (i < packs ? i : packs - 1);
        }
#pragma unroll
        for (int h = 0; h < H; ++h) load_pack<float, 4>(lp + where[h], a[h]);
        if (p.logp_ref) {
#pragma unroll
            for (int h = 0; h < H; ++h) load_pack<float, 4>(ref + where[h], q[h]);
        }
        if (p.weight) {
#pragma unroll
            for (int h = 0; h < H; ++h) load_pack<float, 4>(wt + where[h], w[h]);
        }
        if (tail < steps) {
            at = lp[tail];
            if (p.logp_ref) qt = ref[tail];
            if (p.weight) wl = wt[tail];
        }
        double v = 0.0;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const int t = where[h];
            const double part = (step_gap(a[h][0], q[h][0], w[h][0], t >= mid) + step_gap(a[h][1], q[h][1], w[h][1], t + 1 >= mid)) +
                                (step_gap(a[h][2], q[h][2], w[h][2], t + 2 >= mid) + step_gap(a[h][3], q[h][3], w[h][3], t + 3 >= mid));
            v += h * 256 + (int)threadIdx.x < packs ? part : 0.0;
        }
        if (tail < steps) v += step_gap(at, qt, wl, tail >= mid);
        v = group_sum<64>(v);
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        const double delta = ((red[0] + red[1]) + red[2]) + red[3];
        double z;
        const double g = pair_slope(p, delta, z);
        float* d = p.dlogp + r.lo;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if (h * 256 + (int)threadIdx.x < packs) {
                float o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = step_grad(where[h] + i >= mid ? -g : g, w[h][i]);
                store_pack<float, 4>(d + where[h], o);
            }
        }
        if (tail < steps) d[tail] = step_grad(tail >= mid ? -g : g, wl);
        if (threadIdx.x == 0) pair_terms(p, blockIdx.x, delta, z, p.terms + (size_t)blockIdx.x * 3);
        return;
    }
    const double v = group_sum<64>(span_sum(p, r.lo, r.hi, r.mid, threadIdx.x, 256));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    const double delta = ((red[0] + red[1]) + red[2]) + red[3];
    double z;
    span_grad(p, r.lo, r.hi, r.mid, threadIdx.x, 256, pair_slope(p, delta, z));
    if (threadIdx.x == 0) pair_terms(p, blockIdx.x, delta, z, p.terms + (size_t)blockIdx.x * 3);
}

// Many short pairs: G lanes a pair, no barrier between sums and gradients; a block leaves the sum of its pairs' terms (fixed order).
template <int G>
__global__ __launch_bounds__(256) void k_pref_groups(PrefArgs p, int blocks) {
    constexpr int PER = 256 / G;
    __shared__ double red[3 * PER];
    if (blockIdx.x >= (unsigned)blocks) {
        outside_zero(p, (long long)(blockIdx.x - blocks) * 256 + threadIdx.x, (long long)(gridDim.x - blocks) * 256);
        return;
    }
    const int lane = threadIdx.x % G;
    double t[3] = {0.0, 0.0, 0.0};
    for (int first = blockIdx.x * PER; first < p.P; first += blocks * PER) {
        const int pair = first + (int)threadIdx.x / G;
        const bool on = pair < p.P;
        const PairRows r = rows_of_pair(p, on ? pair : p.P - 1);
        double delta = on ? span_sum(p, r.lo, r.hi, r.mid, lane, G) : 0.0;
        delta = group_sum<G>(delta);
        if (on) {
            double z;
            span_grad(p, r.lo, r.hi, r.mid, lane, G, pair_slope(p, delta, z));
            if (lane == 0) {
                double own[3];
                pair_terms(p, pair, delta, z, own);
                t[0] += own[0];
                t[1] += own[1];
                t[2] += own[2];
            }
        }
    }
    if (lane == 0) {
        double* mine = red + threadIdx.x / G * 3;
        mine[0] = t[0];
        mine[1] = t[1];
        mine[2] = t[2];
    }
    __syncthreads();
    if (threadIdx.x < 3) {
        double sum = red[threadIdx.x];
        for (int i = 1; i < PER; ++i) sum += red[i * 3 + threadIdx.x];
        p.terms[(size_t)blockIdx.x * 3 + threadIdx.x] = sum;
    }
}

// Few, long pairs: a block per piece of one; its sum, then (every block joining its pair's pieces, in order) its gradients.
__global__ __launch_bounds__(256) void k_pref_sums(PrefArgs p) {
    __shared__ double red[4];
    const PairRows r = rows_of_pair(p, blockIdx.x / p.splits);
    long long lo, hi;
    piece_of_pair(p, r, blockIdx.x % p.splits, lo, hi);
    const double v = group_sum<64>(span_sum(p, lo, hi, r.mid, threadIdx.x, 256));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) p.sums[blockIdx.x] = ((red[0] + red[1]) + red[2]) + red[3];
}

__global__ __launch_bounds__(256) void k_pref_grad(PrefArgs p) {
    const unsigned blocks = (unsigned)p.P * p.splits;
    if (blockIdx.x >= blocks) {
        outside_zero(p, (long long)(blockIdx.x - blocks) * 256 + threadIdx.x, (long long)(gridDim.x - blocks) * 256);
        return;
    }
    const int pair = blockIdx.x / p.splits, part = blockIdx.x % p.splits, lane = threadIdx.x & 63;
    const double* sums = p.sums + (size_t)pair * p.splits;
    double d = 0.0;
    for (int i = lane; i < p.splits; i += 64) d += sums[i];
    const double delta = group_sum<64>(d);
    const PairRows r = rows_of_pair(p, pair);
    long long lo, hi;
    piece_of_pair(p, r, part, lo, hi);
    double z;
    span_grad(p, lo, hi, r.mid, threadIdx.x, 256, pair_slope(p, delta, z));
    if (threadIdx.x == 0 && part == 0) pair_terms(p, pair, delta, z, p.terms + (size_t)pair * 3);
}

__global__ __launch_bounds__(FINISH_NT) void k_pref_finish(const double* __restrict__ terms, size_t n, int step, int P, float* __restrict__ loss3) {
    __shared__ double out[3];
    sum_terms(terms, n, step, out);
    if (threadIdx.x < 3) loss3[threadIdx.x] = (float)(out[threadIdx.x] / (double)P);
}

// =====================================================================================================================
// Balance loss.  p = softmax(l[b, a, :]); a row counts for its K largest logits (equal ones: the lowest index first; a
// closed choice, logit -inf, never).  Over the V rows the mask leaves:
//   counts[a, n],  f = counts / (K V),  P = sum_b p / V,  loss = coef N / A sum_a sum_n f P,
//   d l[b, a, n] = coef N / (A V) p_n (f_n - sum_m f_m p_m)         (f is a count: no gradient through it)
// k_bal_stats leaves sums and counts of every chunk of rows as slabs, k_bal_reduce adds the slabs (64 bits, in order), k_bal_grad
// writes the gradient.  A group of G lanes keeps ONE choice a while it walks rows: its sums, and f, stay in registers.
// Bound: k_bal_stats instructions (the K-th largest: issue 31 of its 44 us), k_bal_grad HBM, k_bal_reduce latency.  262147 x 128 bfloat16,
// top 8, masked: 44 + 5 + 29 us (two readings and a writing of 67 MB: 40 us); 4096 x 36 x 35 float32, top 1: 10.8 + 5.2 + 9.8 us (20 MB:
// 6.4 us; three launches, each of them issue for half of its time and waiting for the other).
// Top 8 of 128 on the way: eight rounds of the group's maximum 117 us, rounds on sorted lists 74 us, joined lists of eight 66 us, keys that
// hold the index (no ranking of equal logits afterwards) 57 us, 256 instead of 512 chunks of rows 49 us, eight waves a block for nine 44 us.
// =====================================================================================================================
struct BalArgs {
    const void* logits;
    long long ld;
    const unsigned char* mask;      // optional [R]
    int R, A, N, K;
    double scale;                   // coef N / A
    int accumulate, stream;
    float* loss;
    int* counts;
    float* mean_prob;
    void* dlogits;
    long long ldd;
    int AT, RR, tiles;              // choices and rows side by side in a block
    int chunks, grad_chunks;        // of rows; blocks = tiles * chunks
    float* slab_p;                  // [chunks][A N]
    uint32_t* slab_n;               // [chunks][A N]
    uint32_t* slab_v;               // [chunks] valid rows
    double* unit;                   // coef N / (A V) of one row's choice: coef N / (A K V^2)
    double* terms;                  // [blocks of k_bal_reduce]
};
constexpr int BAL_NT = 576, BAL_COLS = 32;

// Where a group works: its choice, and its row beside the block's other rows
template <int G>
struct BalPlace {
    int tile, chunk, j, al, rr, a;
    bool mine;
    long long r0, r1;
    __device__ __forceinline__ BalPlace(const BalArgs& p, int chunks) {
        tile = blockIdx.x % p.tiles;
        chunk = blockIdx.x / p.tiles;
        j = threadIdx.x % G;
        const int gid = threadIdx.x / G;
        al = gid % p.AT;
        rr = gid / p.AT;
        a = tile * p.AT + al;
        mine = rr < p.RR && a < p.A;
        const long long per = ((long long)p.R + chunks - 1) / chunks;
        r0 = chunk * per;
        r1 = r0 + per < p.R ? r0 + per : p.R;
    }
};

// A group's segment, row after row; past the chunk's end it stays where it is
template <typename T>
struct RowWalk {
    const T* at;
    long long row;
    __device__ __forceinline__ RowWalk(const BalArgs& p, long long r0, long long r1, int rr, size_t off) {
        row = r0 + rr < r1 ? r0 + rr : (r1 > 0 ? r1 - 1 : 0);
        at = static_cast<const T*>(p.logits) + row * p.ld + off;
    }
    __device__ __forceinline__ bool counts(const BalArgs& p) const { return !p.mask || p.mask[row]; }
    __device__ __forceinline__ void step(const BalArgs& p, long long r1) {
        const bool on = row + p.RR < r1;
        row += on ? p.RR : 0;
        at += on ? p.RR * p.ld : 0;
    }
};

// The K-th largest of a group's values, K > 1: every lane sorts its E values once; then up to K rounds of the group's largest head,
// which all lanes that hold it pop (a group that has popped K is done).  Keys are the float bits ordered as integers.
__device__ __forceinline__ int order_key(float x) {
    const int b = __float_as_int(x);            // (-0 below +0: the K-th VALUE is the same either way)
    return b ^ ((b >> 31) & 0x7fffffff);
}
template <int G>
__device__ __forceinline__ int group_max_key(int v) {
    return (int)group_reduce<G>((uint32_t)v, [](uint32_t a, uint32_t b) { return (uint32_t)((int)a > (int)b ? (int)a : (int)b); });
}
template <int G>
__device__ __forceinline__ uint32_t group_add(uint32_t v) {
    return group_reduce<G>(v, [](uint32_t a, uint32_t b) { return a + b; });
}
template <int G, int E>
__device__ __forceinline__ int kth_largest(const int (&keys)[E], int K) {
    int s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = keys[e];
    // odd-even transposition, descending
#pragma unroll
    for (int r = 0; r < E; ++r)
#pragma unroll
        for (int e = r & 1; e + 1 < E; e += 2) {
            const int hi = s[e] > s[e + 1] ? s[e] : s[e + 1], lo = s[e] > s[e + 1] ? s[e + 1] : s[e];
            s[e] = hi;
            s[e + 1] = lo;
        }
    const int lane = threadIdx.x & 63;
    const unsigned long long group = (G == 64 ? ~0ull : ((1ull << (G & 63)) - 1)) << (lane / G * G & 63);
    int left = K, kth = s[0];
    for (int k = 0; k < K; ++k) {
        const int top = group_max_key<G>(s[0]);
        const unsigned long long held = __builtin_amdgcn_ballot_w64(s[0] == top) & group;
        if (left > 0) kth = top;
        const int pop = left > 0 && s[0] == top ? -1 : 0;       // (a mask: hipcc makes an indexed load of a selection)
        left -= (int)__popcll(held);
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] ^= (s[e] ^ (e + 1 < E ? s[e + 1] : (int)0x80000000)) & pop;
        if (__builtin_amdgcn_ballot_w64(left > 0) == 0) break;
    }
    return kth;
}

// ... and for K <= 8, three times cheaper than the rounds (8 of 128: 160 instructions for 16 lanes' lists): every lane's eight
// largest in order, then the lists of two lanes, of two pairs, ... joined: the eight largest of both are max(a[i], b[7 - i]), a bitonic
// sequence, which three stages of exchanges put in order.
__device__ __forceinline__ void exchange(int& a, int& b) {
    const int hi = a > b ? a : b, lo = a > b ? b : a;
    a = hi;
    b = lo;
}
__device__ __forceinline__ void bitonic8(int (&s)[8]) {
#pragma unroll
    for (int d = 4; d; d >>= 1)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (!(i & d)) exchange(s[i], s[i + d]);
}
__device__ __forceinline__ void sort8(int (&s)[8]) {          // odd-even merge sort, descending
#pragma unroll
    for (int p = 1; p < 8; p <<= 1)
#pragma unroll
        for (int k = p; k; k >>= 1)
#pragma unroll
            for (int j = k % p; j + k < 8; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < 8 && (i + j) / (2 * p) == (i + j + k) / (2 * p)) exchange(s[i + j], s[i + j + k]);
}
__device__ __forceinline__ void join8(int (&s)[8], const int (&o)[8]) {
    int t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = s[i] > o[7 - i] ? s[i] : o[7 - i];
    bitonic8(t);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = t[i];
}
template <int CTRL>
__device__ __forceinline__ void join8_lanes(int (&s)[8]) {
    int o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (int)lane_move<CTRL>((uint32_t)s[i]);
    join8(s, o);
}
template <int G, int E>
__device__ __forceinline__ int kth_of_eight(const int (&keys)[E], int K) {
    int s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = i < E ? keys[i < E ? i : 0] : (int)0x80000000;
    sort8(s);
    if (E > 8) {
        int t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = 8 + i < E ? keys[8 + i < E ? 8 + i : 0] : (int)0x80000000;
        sort8(t);
        join8(s, t);
    }
    static_assert(E <= 16, "two lists of eight");
    if (G > 1) join8_lanes<0xB1>(s);
    if (G > 2) join8_lanes<0x4E>(s);
    if (G > 4) join8_lanes<0x141>(s);
    if (G > 8) join8_lanes<0x140>(s);
    if (G > 16) {
        int a[8], b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const auto r = __builtin_amdgcn_permlane16_swap((uint32_t)s[i], (uint32_t)s[i], false, false);
            a[i] = (int)r[0];
            b[i] = (int)r[1];
        }
        join8(a, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = a[i];
    }
    if (G > 32) {
        int a[8], b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const auto r = __builtin_amdgcn_permlane32_swap((uint32_t)s[i], (uint32_t)s[i], false, false);
            a[i] = (int)r[0];
            b[i] = (int)r[1];
        }
        join8(a, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = a[i];
    }
    int kth = s[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) kth = K == i + 1 ? s[i] : kth;
    return kth;
}

template <typename T, int G, int E, bool FULL>
__global__ __launch_bounds__(BAL_NT) void k_bal_stats(BalArgs p) {
    extern __shared__ char lds_raw[];
    const BalPlace<G> at(p, p.chunks);
    const Axis<T, G, E> ln(at.j, p.N);
    float* sums = reinterpret_cast<float*>(lds_raw);                            // [RR][AT N]
    uint32_t* cnts = reinterpret_cast<uint32_t*>(sums + (size_t)p.RR * p.AT * p.N);    // [AT N]
    for (int i = threadIdx.x; i < p.AT * p.N; i += blockDim.x) cnts[i] = 0;
    float acc[E];
    uint32_t cnt[E];
#pragma unroll
    for (int e = 0; e < E; ++e) { acc[e] = 0.f; cnt[e] = 0; }
    uint32_t valid = 0;
    RowWalk<T> walk(p, at.r0, at.r1, at.rr, (size_t)(at.a < p.A ? at.a : p.A - 1) * p.N);
    T next[E];
    bool next_on = false;
    if (at.r0 < at.r1) {
        ln.load(walk.at, next);
        next_on = walk.counts(p);
    }
    for (long long rb = at.r0; rb < at.r1; rb += p.RR) {
        const bool row = at.mine && rb + at.rr < at.r1 && next_on;
        float x[E], m = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = row && (FULL || ln.own(e)) ? to_f32(next[e]) : -INFINITY;
            m = fmaxf(m, x[e]);
        }
        if (rb + p.RR < at.r1) {                // the next row is on its way meanwhile
            walk.step(p, at.r1);
            ln.load(walk.at, next);
            next_on = walk.counts(p);
        }
        valid += row;
        m = group_max<G>(m);
        const float ms = m == -INFINITY ? 0.f : m;
        float ex[E], s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            ex[e] = sizeof(T) == 4 ? exp_below_exact(x[e], ms) : exp_below(x[e], ms);
            s += ex[e];
        }
        s = group_sum<G>(s);
        const float inv = s == 0.f ? 0.f : 1.f / s;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = __builtin_fmaf(ex[e], inv, acc[e]);
        // the chosen: at or above the K-th largest (a closed choice never), of equal ones the first
        if constexpr (sizeof(T) == 2) {
            // 16-bit logits leave 13 bits of their 32-bit form free: with the index there no two keys are equal (equal logits are
            // common at 8 bits of mantissa: ranking them afterwards took as long as all the rest)
            int keys[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int b = __float_as_int(x[e] + 0.f);           // (-0 -> +0: equal values)
                keys[e] = (b ^ ((b >> 31) & 0x7fffe000)) + (0x1fff - ln.at(e));
            }
            int kth;
            if (p.K == 1) {
                kth = keys[0];
#pragma unroll
                for (int e = 1; e < E; ++e) kth = keys[e] > kth ? keys[e] : kth;
                kth = group_max_key<G>(kth);
            } else {
                kth = p.K <= 8 ? kth_of_eight<G, E>(keys, p.K) : kth_largest<G, E>(keys, p.K);
            }
            constexpr int open = (int)0x80800000;                   // above every key of -inf, below those of finite logits
            kth = kth > open ? kth : open;
#pragma unroll
            for (int e = 0; e < E; ++e) cnt[e] += keys[e] >= kth;
            continue;
        }
        float kth = m;
        if (p.K > 1) {
            int keys[E];
#pragma unroll
            for (int e = 0; e < E; ++e) keys[e] = order_key(x[e]);
            const int key = p.K <= 8 ? kth_of_eight<G, E>(keys, p.K) : kth_largest<G, E>(keys, p.K);
            kth = __int_as_float(key ^ ((key >> 31) & 0x7fffffff));
        }
        // (counted over the wave by the scalar unit: with K open choices or more in every row, more than K a row means equal ones)
        int taken = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) taken += __popcll(__builtin_amdgcn_ballot_w64(x[e] >= kth && row));
        const unsigned long long few = __builtin_amdgcn_ballot_w64(row && kth == -INFINITY);
        if (kth == -INFINITY) kth = -3.402823466e38f;
        if (few == 0 && taken * G <= p.K * __popcll(__builtin_amdgcn_ballot_w64(row))) {
#pragma unroll
            for (int e = 0; e < E; ++e) cnt[e] += x[e] >= kth;
        } else {
            // more equal values than room: rank them by index, pack by pack (a pack row is in lane order)
            uint32_t above = 0, before = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) above += x[e] > kth;
            const int room = p.K - (int)group_add<G>(above);
#pragma unroll
            for (int u = 0; u < ln.U; ++u) {
                uint32_t mine = 0;
#pragma unroll
                for (int v = 0; v < ln.V; ++v) mine += x[u * ln.V + v] == kth;
                uint32_t lower = mine;                          // inclusive prefix over the group's lanes
                for (int o = 1; o < G; o <<= 1) {
                    const uint32_t t = (uint32_t)__shfl_up((int)lower, o, G);
                    if (at.j >= o) lower += t;
                }
                uint32_t rank = before + lower - mine;
#pragma unroll
                for (int v = 0; v < ln.V; ++v) {
                    const int e = u * ln.V + v;
                    const bool eq = x[e] == kth;
                    cnt[e] += x[e] > kth || (eq && (int)rank < room);
                    rank += eq;
                }
                before += (uint32_t)__shfl((int)lower, G - 1, G);
            }
        }
    }
    // one choice in the block: its groups in a wave add up first, a row of the merge is a wave (a block of 72 rows spent more time
    // in the merge than a sixth of its work)
    const bool single = p.AT == 1;
    int merge = p.RR, my = at.rr;
    bool writes = at.mine;
    if (single) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            acc[e] = __uint_as_float(across_groups<G>(__float_as_uint(acc[e]), [](uint32_t a, uint32_t b) {
                return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
            }));
            cnt[e] = across_groups<G>(cnt[e], [](uint32_t a, uint32_t b) { return a + b; });
        }
        merge = blockDim.x / 64;
        my = threadIdx.x >> 6;
        writes = (threadIdx.x & 63) < G;
    }
    __syncthreads();
    if (writes) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (ln.own(e)) {
                sums[((size_t)my * p.AT + at.al) * p.N + ln.at(e)] = acc[e];
                if (cnt[e]) atomicAdd(&cnts[at.al * p.N + ln.at(e)], cnt[e]);
            }
        }
    }
    __syncthreads();
    const size_t AN = (size_t)p.A * p.N;
    const int a0 = at.tile * p.AT, cols = (p.A - a0 < p.AT ? p.A - a0 : p.AT) * p.N;
    for (int i = threadIdx.x; i < cols; i += blockDim.x) {
        float s = 0.f;
        for (int q = 0; q < merge; ++q) s += sums[(size_t)q * p.AT * p.N + i];
        p.slab_p[(size_t)at.chunk * AN + (size_t)a0 * p.N + i] = s;
        p.slab_n[(size_t)at.chunk * AN + (size_t)a0 * p.N + i] = cnts[i];
    }
    if (at.tile == 0) {
        __syncthreads();
        if (threadIdx.x == 0) cnts[0] = 0;
        __syncthreads();
        if (at.al == 0 && at.j == 0 && valid) atomicAdd(&cnts[0], valid);
        __syncthreads();
        if (threadIdx.x == 0) p.slab_v[at.chunk] = cnts[0];
    }
}

// 32 columns x 32 lanes over the slabs, sixteen of them in flight a lane; then 32 lanes a column
__global__ __launch_bounds__(1024) void k_bal_reduce(BalArgs p) {
    constexpr int DEEP = 16;
    __shared__ double rs[32][BAL_COLS + 1];
    __shared__ uint32_t rn[32][BAL_COLS + 1], rv[16];
    __shared__ double rt[16];
    const size_t AN = (size_t)p.A * p.N;
    const int cl = threadIdx.x % BAL_COLS, kl = threadIdx.x / BAL_COLS, lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const size_t mine = (size_t)blockIdx.x * BAL_COLS + cl, col = mine < AN ? mine : AN - 1;
    uint32_t v = 0;
    for (int k = threadIdx.x; k < p.chunks; k += 1024) v += p.slab_v[k];
    double s = 0.0;
    uint32_t n = 0;
    for (int k0 = kl; k0 < p.chunks; k0 += 32 * DEEP) {
        float fp[DEEP];
        uint32_t fn[DEEP];
#pragma unroll
        for (int i = 0; i < DEEP; ++i) {
            const int k = k0 + 32 * i < p.chunks ? k0 + 32 * i : kl;
            fp[i] = p.slab_p[(size_t)k * AN + col];
            fn[i] = p.slab_n[(size_t)k * AN + col];
        }
#pragma unroll
        for (int i = 0; i < DEEP; ++i) {
            const bool on = k0 + 32 * i < p.chunks;
            s += on ? (double)fp[i] : 0.0;
            n += on ? fn[i] : 0u;
        }
    }
    rs[kl][cl] = s;
    rn[kl][cl] = n;
    v = group_add<64>(v);
    if (lane == 0) rv[wid] = v;
    __syncthreads();
    const int c2 = threadIdx.x / 32, k2 = threadIdx.x % 32;         // (a column by half a wave)
    const size_t out = (size_t)blockIdx.x * BAL_COLS + c2;
    s = rs[k2][c2];
    n = group_add<32>(rn[k2][c2]);
    s = group_sum<32>(s);
    const uint32_t rows = group_add<16>(rv[threadIdx.x & 15]);
    const double inv_v = rows ? 1.0 / (double)rows : 0.0;
    const double mean = s * inv_v, share = (double)n * inv_v / p.K;
    if (k2 == 0 && out < AN) {
        p.mean_prob[out] = (float)mean;
        p.counts[out] = (int)n;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.unit = p.scale * inv_v * inv_v / p.K;
    double term = out < AN ? share * mean : 0.0;                    // (the same in a column's lanes)
    term += __shfl_xor(term, 32, 64);
    if (lane == 0) rt[wid] = term;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < 16; ++i) t += rt[i];
        p.terms[blockIdx.x] = t;
    }
}

template <typename T, int G, int E, bool FULL>
__global__ __launch_bounds__(BAL_NT) void k_bal_grad(BalArgs p) {
    const BalPlace<G> at(p, p.grad_chunks);
    const Axis<T, G, E> ln(at.j, p.N);
    const size_t off = (size_t)(at.a < p.A ? at.a : p.A - 1) * p.N;
    RowWalk<T> walk(p, at.r0, at.r1, at.rr, off);
    // f less its least entry: f_n - sum f p stays the same, and the difference is one of counts, exact (shares rounded to 32 bits agree
    // in their leading digits where the loss does its work: 262147 rows, top 8 of 128, bfloat16, left 0.3 % of the entries a step off)
    uint32_t count[E], least = 0xffffffffu;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        count[e] = (uint32_t)p.counts[off + ln.at(e)];
        least = count[e] < least ? count[e] : least;
    }
    least = group_min<G>(least);
    const double unit = *p.unit;
    float f[E];
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = (float)(unit * (double)(count[e] - least));
    T next[E];
    bool next_on = false;
    if (at.r0 < at.r1) {
        ln.load(walk.at, next);
        next_on = walk.counts(p);
    }
    for (long long rb = at.r0; rb < at.r1; rb += p.RR) {
        const long long b = rb + at.rr;
        const bool have = at.mine && b < at.r1, row = next_on;
        float x[E], m = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = to_f32(next[e]);
            m = fmaxf(m, x[e]);
        }
        if (rb + p.RR < at.r1) {                // the next row is on its way meanwhile
            walk.step(p, at.r1);
            ln.load(walk.at, next);
            next_on = walk.counts(p);
        }
        m = group_max<G>(m);
        if (m == -INFINITY) m = 0.f;
        float s = 0.f, d = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = sizeof(T) == 4 ? exp_below_exact(x[e], m) : exp_below(x[e], m);
            const float own = FULL || ln.own(e) ? x[e] : 0.f;
            s += own;
            d = __builtin_fmaf(own, f[e], d);
        }
        s = group_sum<G>(s);
        d = group_sum<G>(d);
        const float inv = s == 0.f ? 0.f : 1.f / s, dot = d * inv, di = -dot * inv;
        if (have && (row || !p.accumulate)) {               // (a masked row's gradient: zeros, or left alone)
            T* to = static_cast<T*>(p.dlogits) + b * p.ldd + off;
            T o[E];
            if (p.accumulate) ln.load(to, o);
            // p_n (f_n - sum f p) with p = x / s, sum f p = d / s; 32-bit gradients form the difference, which cancels, first
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float v = sizeof(T) == 4 ? (x[e] * inv) * (f[e] - dot) : x[e] * __builtin_fmaf(f[e], inv, di);
                if (p.accumulate) v += to_f32(o[e]);
                o[e] = from_f32<T>(row ? v : 0.f);
            }
            ln.store(to, o, p.stream);
        }
    }
    if (blockIdx.x == 0) {
        __shared__ double red[BAL_NT / 64];
        const size_t parts = ((size_t)p.A * p.N + BAL_COLS - 1) / BAL_COLS;
        double t = 0.0;
        for (size_t i = threadIdx.x; i < parts; i += blockDim.x) t += p.terms[i];
        t = group_sum<64>(t);
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

static int group_width(int N) {
    return N <= 4 ? 4 : N <= 8 ? 2 : N <= 24 ? 4 : N <= 64 ? 8 : N <= 96 ? 16 : N <= 128 ? 8 : N <= 256 ? 32 : 64;
}

// choices and rows side by side in a block of up to `threads`; -> its time for a row of all choices: the tiles of choices over the rows
// that a block takes at once, by the waves of its fullest SIMD (k_bal_stats is bound by issue, one block a CU)
static double bal_block(BalArgs& p, int threads) {
    const int G = group_width(p.N), groups = threads / G;
    p.AT = p.A < groups ? p.A : groups;
    while (p.AT > 1 && p.AT * p.N > 4096) p.AT = (p.AT + 1) / 2;
    p.RR = groups / p.AT;
    p.tiles = (p.A + p.AT - 1) / p.AT;
    return (double)p.tiles / p.RR * ((p.AT * p.RR * G + 255) / 256);
}
static void bal_shape(BalArgs& p) {
    // Eight waves, two a SIMD, or nine where they take another row of choices or a tile less, by that time.  Loss, eight / nine waves
    // (us): 262147 x 128 bfloat16 top 8 67 / 78, 8192 x 128 x 256 656 / 901, 200000 x 300 274 / 315, 20000 x 17 x 24 28.7 / 30.0;
    // 4096 x 36 x 35 27.9 / 24.7, 3000 x 130 x 40 53.8 / 48.6, 9000 x 3 x 1000 78 / 75.
    const double eight = bal_block(p, 512);
    if (bal_block(p, BAL_NT) > eight) bal_block(p, 512);
    // chunks of rows: a block a CU; four rows or more for a group of k_bal_stats (a chunk costs 8 A N bytes of slabs), and 256 at most:
    // a lane's 32-bit sum of as many equal weights, as a fresh policy has, is off by under 60 steps of 2^-24, of 3640 by 600 (the
    // chunks are added in 64 bits)
    const long long most = ((long long)p.R + p.RR - 1) / p.RR, fill = (256 + p.tiles - 1) / p.tiles;
    const long long short_sums = (most + 255) / 256, wanted = fill > short_sums ? fill : short_sums;
    p.chunks = (int)((most + 3) / 4 < wanted ? (most + 3) / 4 : wanted);
    p.grad_chunks = (int)(most < 4 * fill ? most : 4 * fill);
}
static size_t bal_terms(const BalArgs& p) { return ((size_t)p.A * p.N + BAL_COLS - 1) / BAL_COLS; }
static size_t bal_bytes(const BalArgs& p) {
    const size_t AN = (size_t)p.A * p.N;
    return (bal_terms(p) + 1) * sizeof(double) + (size_t)p.chunks * AN * 8 + (size_t)p.chunks * 4;
}

template <typename T, int G, int E, bool FULL>
static void launch_bal_as(const BalArgs& p, hipStream_t st) {
    const int threads = (p.AT * p.RR * G + 63) / 64 * 64;
    const size_t lds = ((size_t)p.RR + 1) * p.AT * p.N * 4;         // (RR AT N <= 576 E, AT N <= 4096: 52 KB at most)
    hipLaunchKernelGGL((k_bal_stats<T, G, E, FULL>), dim3(p.tiles * p.chunks), dim3(threads), lds, st, p);
    hipLaunchKernelGGL(k_bal_reduce, dim3((unsigned)bal_terms(p)), dim3(1024), 0, st, p);
    hipLaunchKernelGGL((k_bal_grad<T, G, E, FULL>), dim3(p.tiles * p.grad_chunks), dim3(threads), 0, st, p);
}
template <typename T, int G, int E>
static void launch_bal(const BalArgs& p, hipStream_t st) {
    if (p.N == G * E) launch_bal_as<T, G, E, true>(p, st);      // (no lane without a category: nothing to mask)
    else launch_bal_as<T, G, E, false>(p, st);
}
template <typename T>
static void pick_bal(const BalArgs& p, hipStream_t st) {
    const int N = p.N;
    if (N <= 4) launch_bal<T, 4, 1>(p, st);
    else if (N <= 8) launch_bal<T, 2, 4>(p, st);
    else if (N <= 16) launch_bal<T, 4, 4>(p, st);
    else if (N <= 24) launch_bal<T, 4, 6>(p, st);
    else if (N <= 32) launch_bal<T, 8, 4>(p, st);
    else if (N <= 40) launch_bal<T, 8, 5>(p, st);
    else if (N <= 64) launch_bal<T, 8, 8>(p, st);
    else if (N <= 96) launch_bal<T, 16, 6>(p, st);
    else if (N <= 128) launch_bal<T, 8, 16>(p, st);
    else if (N <= 192) launch_bal<T, 32, 6>(p, st);
    else if (N <= 256) launch_bal<T, 32, 8>(p, st);
    else if (N <= 384) launch_bal<T, 64, 6>(p, st);
    else if (N <= 512) launch_bal<T, 64, 8>(p, st);
    else launch_bal<T, 64, 16>(p, st);
}

static void pref_shape(PrefArgs& p) {
    // pieces of a pair: about 8192 steps of the average one, and no more blocks than fill the chip a few times
    long long s = (p.T / p.P + 8191) / 8192;
    const long long most = (4096ll + p.P - 1) / p.P;
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
    return ((size_t)P * 3 + (size_t)P * p.splits) * sizeof(double);
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
    const unsigned blocks = (unsigned)P * (unsigned)p.splits;
    const unsigned outside = (unsigned)(T / 4096 + 1 < 64 ? T / 4096 + 1 : 64);
    if (P <= PREF_SMALL_P && T <= PREF_SMALL_T && T / P <= PREF_SMALL_MEAN) {
        hipLaunchKernelGGL(k_pref_small, dim3(1), dim3(1024), 0, st, p, loss3);
        PFPN_CHECK_LAUNCH();
        return PFPN_OK;
    }
    size_t left = P;                                       // triples of terms that are left to add up
    if (p.splits == 1 && T / P <= PREF_SHORT && 3 * (T / P) <= P) {
        const bool few = T / P <= 128;
        const int need = few ? (P + 15) / 16 : (P + 3) / 4;
        const int blocks = need < 2048 ? need : 2048;
        left = blocks;
        if (few) hipLaunchKernelGGL((k_pref_groups<16>), dim3((unsigned)blocks + outside), dim3(256), 0, st, p, blocks);
        else hipLaunchKernelGGL((k_pref_groups<64>), dim3((unsigned)blocks + outside), dim3(256), 0, st, p, blocks);
    } else if (p.splits == 1) {
        hipLaunchKernelGGL(k_pref_pairs, dim3((unsigned)P + outside), dim3(256), 0, st, p);
    } else {
        hipLaunchKernelGGL(k_pref_sums, dim3(blocks), dim3(256), 0, st, p);
        hipLaunchKernelGGL(k_pref_grad, dim3(blocks + outside), dim3(256), 0, st, p);
    }
    const int step = fold_terms(p.terms, left, st);
    hipLaunchKernelGGL(k_pref_finish, dim3(1), dim3(FINISH_NT), 0, st, (const double*)p.terms, left, step, P, loss3);
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
    p.stream = (size_t)R * A * N * (dtype == DT_F32 ? 4 : 2) > (256u << 20);
    bal_shape(p);
    if (!workspace || workspace_bytes < bal_bytes(p)) return PFPN_ERR_WORKSPACE;
    const size_t AN = (size_t)A * N;
    p.terms = static_cast<double*>(workspace);
    p.unit = p.terms + bal_terms(p);
    p.slab_p = reinterpret_cast<float*>(p.unit + 1);
    p.slab_n = reinterpret_cast<uint32_t*>(p.slab_p + (size_t)p.chunks * AN);
    p.slab_v = p.slab_n + (size_t)p.chunks * AN;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == DT_F32) pick_bal<float>(p, st);
    else if (dtype == DT_BF16) pick_bal<bf16_t>(p, st);
    else pick_bal<f16_t>(p, st);
    PFPN_CHECK_LAUNCH();
    return PFPN_OK;
}

}  // extern "C"
