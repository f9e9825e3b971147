// Log-probabilities of chosen categories and the clipped policy loss with a KL term, straight from categorical logits
// [B, A, N] (A choices of N categories make one joint action; A = 1: a token row), forward and backward.
//
//   logp[b]       = sum_a (l[b,a,k] - m[b,a] - log s[b,a]),   m = max_n l, s = sum_n exp(l - m)
//   d logits      = dlogp[b] (1[n = k] - exp(l - m) / s)
//
// (the particle index a policy drew: reference networks/utils.py:187-194; the clipped surrogate: networks/actor_critic/ppo.py:44-54)
#include "categorical_impl.h"

namespace pfpn {

// ---------------------------------------------------------------------------------------------------------------------
// The same loss on log-probs that come from elsewhere (the particle mixture's own density): one pass over [n] vectors.
// 1000003 rows, weighted: 8.3 us + 2.3 us for the sum of the blocks (24 MB: 3.7 us at the cache's rate): latency, two waves a SIMD that
// wait for half of their time; their instructions, the 64-bit exponential among them, issue for 3.2 us.
// ---------------------------------------------------------------------------------------------------------------------
// Four rows a load, from any alignment.  One block (n <= 4096) finishes the sums itself.
constexpr long long ROWS_SMALL = 4096;

template <int NT>
__global__ __launch_bounds__(NT) void k_policy_rows(const float* __restrict__ logp, HeadArgs h, size_t n,
                                                    float* __restrict__ dlogp, double* __restrict__ part, float* __restrict__ loss4) {
    __shared__ double red[3 * 16], sums[3];
    HeadTerms t = {0.0, 0.0, 0.0};
    float mean = 0.f, rstd = 1.f, lo = -INFINITY, hi = INFINITY;
    if (h.stats) { mean = h.stats[0]; rstd = h.stats[1]; lo = h.stats[2]; hi = h.stats[3]; }
    auto one = [&](float lp, float old, float adv, float ref, float w) -> float {
        const double wd = h.weight ? (double)w : h.inv_B;
        if (wd == 0.0) return 0.f;
        const HeadRow row = {old, h.stats ? clip_adv((adv - mean) * rstd, lo, hi) : adv, ref, wd};
        HeadTerms q;
        const float g = (float)policy_head((double)lp, row, h, q);
        t.policy += q.policy;
        t.kl += q.kl;
        t.clipped += q.clipped;
        return g;
    };
    const size_t full = n / 4 * 4;
    for (size_t i = ((size_t)blockIdx.x * NT + threadIdx.x) * 4; i < full; i += (size_t)gridDim.x * NT * 4) {
        float lp[4], old[4], adv[4], ref[4] = {}, w[4] = {}, d[4];
        load_pack<float, 4>(logp + i, lp);
        load_pack<float, 4>(h.logp_old + i, old);
        load_pack<float, 4>(h.adv + i, adv);
        if (h.logp_ref) load_pack<float, 4>(h.logp_ref + i, ref);
        if (h.weight) load_pack<float, 4>(h.weight + i, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = one(lp[e], old[e], adv[e], ref[e], w[e]);
        store_pack<float, 4>(dlogp + i, d);
    }
    const size_t i = full + threadIdx.x;
    if (blockIdx.x == 0 && i < n)
        dlogp[i] = one(logp[i], h.logp_old[i], h.adv[i], h.logp_ref ? h.logp_ref[i] : 0.f, h.weight ? h.weight[i] : 0.f);
    double* out = loss4 ? sums : part + (size_t)blockIdx.x * 3;
    block_terms(t, red, out);
    if (loss4) {
        __syncthreads();
        if (threadIdx.x == 0) write_loss4(sums, h.kl_coef, loss4);
    }
}

// a wave a term: it reads and writes nothing but its term of the block's FOLD triples
__global__ __launch_bounds__(192) void k_fold_terms(double* part, size_t n) {
    const size_t first = (size_t)blockIdx.x * FOLD;
    const int term = threadIdx.x >> 6, lane = threadIdx.x & 63;
    double t[FOLD / 64], s = 0.0;
#pragma unroll
    for (int k = 0; k < (int)FOLD / 64; ++k) {
        const size_t j = first + lane + 64 * k;
        t[k] = part[(j < n ? j : first) * 3 + term];
    }
#pragma unroll
    for (int k = 0; k < (int)FOLD / 64; ++k) s += first + lane + 64 * k < n ? t[k] : 0.0;
    s = group_sum<64>(s);
    if (lane == 0) part[first * 3 + term] = s;
}
int fold_terms(double* part, size_t& n, hipStream_t st) {
    if (n <= FOLD_FROM) return 1;
    const size_t left = (n + FOLD - 1) / FOLD;
    hipLaunchKernelGGL(k_fold_terms, dim3((unsigned)left), dim3(192), 0, st, part, n);
    n = left;
    return (int)FOLD;
}

// loss4 = {policy + c kl, policy, kl, clipped}: the blocks' sums in a fixed order
__global__ __launch_bounds__(FINISH_NT) void k_policy_finish(const double* __restrict__ part, size_t nparts, int step, double kl_coef,
                                                             float* __restrict__ loss4) {
    __shared__ double out[3];
    sum_terms(part, nparts, step, out);
    if (threadIdx.x == 0) write_loss4(out, kl_coef, loss4);
}

// ---------------------------------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------------------------------
int cat_splits(int B, int A, int N) {
    // pieces of a long axis: two blocks a CU, pieces of at least 4096 logits; one piece from 512 segments on
    const long long segs = (long long)B * A;
    long long s = (512 + segs - 1) / segs;
    const long long most = ((long long)N + 4095) / 4096;
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s > CAT_MAX_SPLITS ? CAT_MAX_SPLITS : s);
}

// One launch takes MAX_BLOCKS blocks: more rows go in turns.  Their loss terms line up in the workspace; what else a turn keeps there
// lies behind its own terms, and is done with before the next turn's are written.
static size_t rows_of_a_launch(const CatArgs& p, size_t size) {
    if (p.N > CAT_SHORT_N) return MAX_BLOCKS / p.A;                 // a block a segment (many rows: one piece each)
    // (a block of a large batch takes sixteen segments in whole rows, or more, where they span less than 2^31 bytes)
    const size_t widest = (size_t)(p.ld > p.ldd ? p.ld : p.ldd) * size;
    return p.A < 16 && widest < (1ull << 31) / 16 ? MAX_BLOCKS * (16 / p.A) : MAX_BLOCKS;
}

template <int MODE>
static int run_typed(CatArgs p, int dtype, void* ws, size_t ws_bytes, float* loss4, void* stream) {
    hipStream_t st = (hipStream_t)stream;
    const size_t size = dtype == DT_F32 ? 4 : 2, rows = p.B, most = rows_of_a_launch(p, size);
    size_t total = 0;
    for (size_t r = 0; r < rows; r += most) {
        CatArgs q = p;
        q.B = (int)(rows - r < most ? rows - r : most);
        q.logits = static_cast<const char*>(p.logits) + r * p.ld * size;
        q.index = static_cast<const int*>(p.index) + (r * p.A << p.index64);
        if (p.logp) q.logp += r;
        if (p.dlogp) q.dlogp += r;
        if (p.dlogits) q.dlogits = static_cast<char*>(p.dlogits) + r * p.ldd * size;
        if (MODE == CAT_PPO) {
            q.head.logp_old += r;
            q.head.adv += r;
            if (p.head.logp_ref) q.head.logp_ref += r;
            if (p.head.weight) q.head.weight += r;
        }
        q.loss4 = rows <= most ? loss4 : nullptr;
        const size_t used = total * 3 * sizeof(double);
        void* at = ws ? static_cast<char*>(ws) + used : nullptr;
        const size_t left = ws_bytes > used ? ws_bytes - used : 0;
        size_t nparts = 0;
        const int rc = dtype == DT_F32 ? run_cat<float, MODE>(q, at, left, &nparts, st)
                     : dtype == DT_BF16 ? run_cat<bf16_t, MODE>(q, at, left, &nparts, st)
                                        : run_cat<f16_t, MODE>(q, at, left, &nparts, st);
        if (rc != PFPN_OK) return rc;
        if (MODE == CAT_PPO) total += nparts;
    }
    if (MODE != CAT_PPO || total == 0) return PFPN_OK;
    double* part = static_cast<double*>(ws);
    const int step = fold_terms(part, total, st);
    hipLaunchKernelGGL(k_policy_finish, dim3(1), dim3(FINISH_NT), 0, st, (const double*)part, total, step, p.head.kl_coef, loss4);
    PFPN_CHECK_LAUNCH();
    return PFPN_OK;
}

static bool bad_shape(const void* logits, int dtype, long long ld, const void* index, int B, int A, int N) {
    return !logits || !index || dtype < DT_F32 || dtype > DT_F16 || B < 1 || A < 1 || N < 1 || A > CAT_MAX_A ||
           N > CAT_MAX_N || ld < (long long)A * N;
}
static bool bad_head(const HeadArgs& h) {
    return !h.logp_old || !h.adv || !(h.clip_lo <= 1.0) || !(h.clip_hi >= 1.0) || (h.kl_coef != 0.0 && !h.logp_ref);
}
static int policy_row_blocks(long long n) { return (int)(n / 2048 + 1 < 2048 ? n / 2048 + 1 : 2048); }

}  // namespace pfpn

using namespace pfpn;

extern "C" {

size_t pfpn_categorical_workspace_bytes(int B, int A, int N) {
    if (B < 1 || A < 1 || N < 1) return 0;
    const size_t parts = (size_t)B * 3 * sizeof(double);
    return N <= CAT_SHORT_N ? parts : parts + (size_t)B * A * cat_splits(B, A, N) * 2 * sizeof(float) + (size_t)B * sizeof(float);
}

int pfpn_categorical_logprob_fwd(const void* logits, int dtype, long long row_stride, const void* index, int index64,
                                 int B, int A, int N, float* logp, void* workspace, size_t workspace_bytes, void* stream) {
    PFPN_BEGIN();
    if (bad_shape(logits, dtype, row_stride, index, B, A, N) || !logp) return PFPN_ERR_ARG;
    CatArgs p = {};
    p.logits = logits; p.ld = row_stride; p.index = index; p.index64 = index64 != 0;
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
    p.logits = logits; p.ld = row_stride; p.index = index; p.index64 = index64 != 0;
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
    p.logits = logits; p.ld = row_stride; p.index = index; p.index64 = index64 != 0;
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
    double* part = static_cast<double*>(workspace);
    hipStream_t st = (hipStream_t)stream;
    if (n <= ROWS_SMALL) {
        hipLaunchKernelGGL((k_policy_rows<1024>), dim3(1), dim3(1024), 0, st, logp, h, (size_t)n, dlogp, part, loss4);
    } else {
        const int blocks = policy_row_blocks(n);
        hipLaunchKernelGGL((k_policy_rows<256>), dim3(blocks), dim3(256), 0, st, logp, h, (size_t)n, dlogp, part, (float*)nullptr);
        hipLaunchKernelGGL(k_policy_finish, dim3(1), dim3(FINISH_NT), 0, st, (const double*)part, (size_t)blocks, 1, kl_coef, loss4);
    }
    PFPN_CHECK_LAUNCH();
    return PFPN_OK;
}

}  // extern "C"
