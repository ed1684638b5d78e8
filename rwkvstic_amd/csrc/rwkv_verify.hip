// Drafted tokens held against the target's logits (rwkv_verify_drafts).  All arithmetic is float64: with 50277 tokens a running
// sum in float32 would put one draw in a hundred on another token than the definition does.
#include "rwkv_types.h"

namespace rwkv {

namespace {

constexpr int kVT = 256;             // threads
constexpr int kMaxDrafts = 64;

struct RowStat { double max, sum; int64_t first; };      // of a row: the largest logit, the sum of the weights, the first maximum (-1: none)

struct VerifyArgs {
    int64_t B, K, V;
    const void *logits; int64_t seq, row;
    const void *draft; int64_t draft_seq, draft_row;
    const int64_t *drafts;
    const int32_t *lengths;
    const float *u;
    double inv_temp;
    int greedy;
    int64_t *tokens, *accepted;
    RowStat *stat;                   // [B][K+1], then [B][K] of the drafts' logits
};

// A logit's weight beside the row's largest; NaN and -infinity have none, and where the largest is +infinity the others have none.
__device__ __forceinline__ double weight(double x, double max, double inv_temp) {
    if (!(x > -INFINITY)) return 0.0;
    return x == max ? 1.0 : exp((x - max) * inv_temp);
}

__device__ __forceinline__ void better(double &x, int64_t &i, double y, int64_t j) {
    if (j >= 0 && (i < 0 || y > x || (y == x && j < i))) { x = y; i = j; }
}

// A workgroup per row.
template <typename Real>
__global__ void __launch_bounds__(kVT) verify_rows_kernel(VerifyArgs a) {
    __shared__ double s_max[kWaves], red[kWaves];
    __shared__ int64_t s_first[kWaves];
    const int64_t targets = a.B * (a.K + 1), at = blockIdx.x, of = at < targets ? a.K + 1 : a.K, row = at < targets ? at : at - targets;
    const Real *x = at < targets ? (const Real *)a.logits + row / of * a.seq + row % of * a.row
                                 : (const Real *)a.draft + row / of * a.draft_seq + row % of * a.draft_row;
    double m = -INFINITY;
    int64_t first = -1;
    for (int64_t j = threadIdx.x; j < a.V; j += kVT) { const double y = x[j]; if (y > m) { m = y; first = j; } }
    for (int off = 32; off >= 1; off >>= 1) better(m, first, __shfl_xor(m, off, 64), __shfl_xor((long long)first, off, 64));
    if ((threadIdx.x & 63) == 0) { s_max[threadIdx.x >> 6] = m; s_first[threadIdx.x >> 6] = first; }
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) better(m, first, s_max[w], s_first[w]);
    double s[1] = {0.0};
    if (!a.greedy)
        for (int64_t j = threadIdx.x; j < a.V; j += kVT) s[0] += weight(x[j], m, a.inv_temp);
    block_sum(s, red);
    if (threadIdx.x == 0) a.stat[at] = {m, s[0], first};
}

// A workgroup per sequence.
template <typename Real>
__global__ void __launch_bounds__(kVT) verify_pick_kernel(VerifyArgs a) {
    __shared__ double sums[kVT], s_total;
    __shared__ int s_n, s_count, s_any, s_pick;
    const int64_t b = blockIdx.x;
    const int tid = threadIdx.x;
    const Real *logits = (const Real *)a.logits + b * a.seq, *draft = a.draft ? (const Real *)a.draft + b * a.draft_seq : nullptr;
    const RowStat *ps = a.stat + b * (a.K + 1), *qs = a.stat + a.B * (a.K + 1) + b * a.K;
    if (tid == 0) {
        const int count = a.lengths ? max(0, min((int)a.K, a.lengths[b])) : (int)a.K;
        int n = 0;
        for (; n < count; ++n) {
            const int64_t d = a.drafts[b * a.K + n];
            if (d < 0 || d >= a.V) break;
            if (a.greedy) { if (ps[n].first != d) break; continue; }
            const double p = ps[n].sum > 0 ? weight(logits[n * a.row + d], ps[n].max, a.inv_temp) / ps[n].sum : 0.0;
            const double q = !draft ? 1.0 : qs[n].sum > 0 ? weight(draft[n * a.draft_row + d], qs[n].max, a.inv_temp) / qs[n].sum : 0.0;
            if (!((double)a.u[b * (a.K + 1) + n] * q < p)) break;
        }
        s_n = n; s_count = count; s_pick = -1;
    }
    __syncthreads();
    const int n = s_n;
    int64_t pick = -1;
    if (a.greedy) pick = ps[n].first;
    else if (ps[n].sum > 0) {
        const Real *x = logits + n * a.row, *y = draft ? draft + n * a.draft_row : nullptr;
        const int64_t gone = n < s_count ? a.drafts[b * a.K + n] : -1;
        bool left = n < s_count;                      // what is left of p once q is taken off, or p itself
        const int64_t per = ceil_div(a.V, kVT), j0 = min(a.V, per * tid), j1 = min(a.V, j0 + per);
        auto value = [&](int64_t j) {
            const double p = weight(x[j], ps[n].max, a.inv_temp) / ps[n].sum;
            if (!left) return p;
            const double q = !y ? (j == gone ? 1.0 : 0.0) : qs[n].sum > 0 ? weight(y[j], qs[n].max, a.inv_temp) / qs[n].sum : 0.0;
            return fmax(p - q, 0.0);
        };
        for (;;) {
            double s = 0.0;
            for (int64_t j = j0; j < j1; ++j) s += value(j);
            __syncthreads();
            sums[tid] = s;
            if (tid == 0) s_any = 0;
            __syncthreads();
            if (tid == 0) {
                double run = 0.0;
                for (int i = 0; i < kVT; ++i) { const double v = sums[i]; sums[i] = run; run += v; }
                s_total = run;
            }
            __syncthreads();
            if (s_total > 0.0 || !left) break;
            left = false;
        }
        // the lowest index whose running weight is over the aim; rounding can leave none: then the last one that has weight
        const double aim = (double)a.u[b * (a.K + 1) + a.K] * s_total;
        double run = sums[tid];
        int last = -1, hit = -1;
        for (int64_t j = j0; j < j1 && hit < 0; ++j) {
            const double w = value(j);
            run += w;
            if (w > 0.0) { last = (int)j; if (run > aim) hit = (int)j; }
        }
        __shared__ int s_hit;
        if (tid == 0) s_hit = 0x7fffffff;
        __syncthreads();
        if (hit >= 0) atomicMin(&s_hit, hit);
        if (last >= 0) atomicMax(&s_pick, last);
        __syncthreads();
        pick = s_hit != 0x7fffffff ? s_hit : s_pick;
    }
    for (int64_t i = tid; i <= a.K; i += kVT) a.tokens[b * (a.K + 1) + i] = i < n ? a.drafts[b * a.K + i] : i == n ? pick : -1;
    if (tid == 0) a.accepted[b] = n;
}

}  // namespace

}  // namespace rwkv

using namespace rwkv;

extern "C" {

size_t rwkv_verify_drafts_workspace_bytes(int64_t B, int64_t K, int64_t V) {
    if (B <= 0 || K < 0 || V <= 0) return 0;
    return (size_t)(B * (2 * K + 1)) * sizeof(RowStat);
}

int rwkv_verify_drafts(rwkv_stream_t stream, int64_t B, int64_t K, int64_t V, int real, const void *logits, int64_t logits_seq_stride,
                       int64_t logits_row_stride, const void *draft_logits, int64_t draft_seq_stride, int64_t draft_row_stride,
                       const int64_t *drafts, const int32_t *lengths, const float *u, double temp, int greedy, int64_t *tokens,
                       int64_t *accepted, void *workspace, size_t workspace_bytes) {
    RWKV_CHECK_ARG(logits && tokens && accepted && (drafts || K == 0) && (u || greedy), "rwkv_verify_drafts: null pointer");
    RWKV_CHECK_ARG(B > 0 && K >= 0 && V > 0, "rwkv_verify_drafts: bad sizes");
    RWKV_CHECK_ARG(real == RWKV_F32 || real == RWKV_F64, "rwkv_verify_drafts: logits are float32 or float64");
    RWKV_CHECK_ARG(greedy || temp > 0.0, "rwkv_verify_drafts: temp must be positive");
    RWKV_CHECK_ARG(logits_seq_stride >= 0 && logits_row_stride >= 0 && draft_seq_stride >= 0 && draft_row_stride >= 0, "rwkv_verify_drafts: negative stride");
    if (K > kMaxDrafts || V >= (1ll << 31) || B >= (1ll << 24)) return set_error(RWKV_ERR_SIZE, "rwkv_verify_drafts: at most %d drafts", kMaxDrafts);
    RWKV_CHECK_ALIGN(workspace, 16);
    if (!workspace || workspace_bytes < rwkv_verify_drafts_workspace_bytes(B, K, V))
        return set_error(RWKV_ERR_WORKSPACE, "rwkv_verify_drafts: workspace too small");
    const bool of_drafts = draft_logits && !greedy && K > 0;
    const VerifyArgs a{B, K, V, logits, logits_seq_stride, logits_row_stride, of_drafts ? draft_logits : nullptr, draft_seq_stride, draft_row_stride,
                       drafts, lengths, u, 1.0 / temp, greedy != 0, tokens, accepted, (RowStat *)workspace};
    with_real(real, [&](auto re) {
        using Real = typename decltype(re)::type;
        hipLaunchKernelGGL(verify_rows_kernel<Real>, dim3((unsigned)(B * (K + 1) + (of_drafts ? B * K : 0))), dim3(kVT), 0, (hipStream_t)stream, a);
        hipLaunchKernelGGL(verify_pick_kernel<Real>, dim3((unsigned)B), dim3(kVT), 0, (hipStream_t)stream, a);
    });
    RWKV_CHECK_LAUNCH("verify_pick_kernel");
    return RWKV_OK;
}

}  // extern "C"
