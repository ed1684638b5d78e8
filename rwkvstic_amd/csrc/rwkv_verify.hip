// Drafted tokens held against the target's logits (rwkv_verify_drafts).  All arithmetic is float64: with 50277 tokens a running
// sum in float32 would put one draw in a hundred on another token than the definition does.
//
// Each row of logits is cut into segments, at most kSegments of at least kChunk tokens:
//   verify_rows_kernel  largest logit, and sum of the weights beside it (or first maximum), of every segment of every row
//   verify_left_kernel  which drafts are accepted, and the sums of what the next token is drawn from, piece by piece
//   verify_pick_kernel  the piece that the drawn token is in, and the token
// Of the logits the first kernel reads everything once; the others read one row of each a sequence (from cache).  64 sequences of
// 8 drafts, 65536 tokens, float32, with the drafts' logits: 64 us (4.5 TB/s) + 21 + 7; one of 4, 50277 tokens, float64: 5 + 6 + 6, latency.
#include "rwkv_types.h"

#include <algorithm>

namespace rwkv {

namespace {

constexpr int kVT = kThreads;        // threads of verify_rows_kernel
constexpr int kPer = 16;             // tokens of a thread
constexpr int kChunk = kVT * kPer;   // tokens of a workgroup at a time
// The kernels that draw are short and run once a sequence: what they wait for is their own code, so a thread has four tokens.
constexpr int kDT = 1024, kFew = kChunk / kDT, kDWaves = kDT / 64, kLT = 512;
constexpr int kSegments = 64;
constexpr int kMaxDrafts = 64;

struct RowStat { double max, sum; int first, pad; };     // of a segment: largest logit, sum of the weights beside it, first maximum (-1: none)

struct Verdict {                     // of a sequence
    double p_max, p_sum, q_max, q_sum;               // row n of both: the largest logit and the sum of the weights
    int n, left;                                     // drafts accepted; whether q is taken off p
};

struct VerifyArgs {
    int64_t B, K, V;
    const void *logits; int64_t seq, row;
    const void *draft; int64_t draft_seq, draft_row;
    const int64_t *drafts;
    const int32_t *lengths;
    const float *u;
    double inv_temp;
    int64_t *tokens, *accepted;
    int segments;
    int64_t segment;                 // tokens of one, a multiple of kChunk
    RowStat *stat;                   // [B][K+1][segments], then [B][K][segments] of the drafts' logits
    int64_t piece;                   // a part of a segment: tokens whose weights verify_left_kernel adds up; kSegments at most
    double *sums;                    // [B][kSegments]
    Verdict *verdict;                // [B]
};

// e^(d / temp) for d <= 0 (0 for anything that is not a number), to 2^-51 or so of it: the exponent in 32nds of log2 e from a table, the
// rest by its series (P. T. P. Tang, ACM TOMS 15, 1989) to the sixth power (the seventh is below 2^-57).  Half the instructions of exp(),
// which takes longer than the logits take to come.
struct Exp {
    const double *table;                             // LDS: 2^(i/32)
    double inv_temp;
    __device__ __forceinline__ double operator()(double d) const {
        constexpr double kMagic = 6755399441055744.0;                        // 3 * 2^51: adding it rounds to a whole number
        constexpr double k32 = 46.16624130844683;                            // 32 log2 e, to 2^-56 of it
        const double y = fmax(d * inv_temp, -800.0);                         // (2^-1154 is 0; what is no number gives way to it)
        const double z = fma(y, k32, kMagic), f = fma(y, k32, -(z - kMagic));
        const int n = (int)__double_as_longlong(z);
        double p = fma(f, 1.4345655584131934e-13, 3.9737099845494161e-11);          // (ln 2 / 32)^k / k!
        p = fma(f, p, 9.1725627018246432e-09);
        p = fma(f, p, 1.6938509724371820e-06);
        p = fma(f, p, 2.3459619820224679e-04);
        p = fma(f, p, 2.1660849392498291e-02);
        p = fma(f, p, 1.0);
        return ldexp(table[n & 31] * p, n >> 5);
    }
};
__constant__ const double kTable[32] = {               // 2^(i/32)
    1.0000000000000000000, 1.0218971486541166782, 1.0442737824274138403, 1.0671404006768236182,
    1.0905077326652576592, 1.1143867425958925363, 1.1387886347566916537, 1.1637248587775775138,
    1.1892071150027210667, 1.2152473599804688781, 1.2418578120734840486, 1.2690509571917332226,
    1.2968395546510096659, 1.3252366431597412946, 1.3542555469368927283, 1.3839098819638319549,
    1.4142135623730950488, 1.4451808069770466200, 1.4768261459394993114, 1.5091644275934227398,
    1.5422108254079408236, 1.5759808451078864865, 1.6104903319492543082, 1.6457554781539648445,
    1.6817928305074290861, 1.7186192981224779156, 1.7562521603732994831, 1.7947090750031071864,
    1.8340080864093424635, 1.8741676341102999013, 1.9152065613971472939, 1.9571441241754002690};
__device__ __forceinline__ Exp exp_table(double (&table)[32], double inv_temp) {              // (before a barrier)
    if (threadIdx.x < 32) table[threadIdx.x] = kTable[threadIdx.x];
    return {table, inv_temp};
}

// A logit's weight beside the largest; NaN and -infinity have none, and where the largest is +infinity the others have none.
__device__ __forceinline__ double weight(Exp e, double x, double max) { return max == INFINITY ? (x == max ? 1.0 : 0.0) : e(x - max); }

__device__ __forceinline__ void better(double &x, int &i, double y, int j) {
    if (j >= 0 && (i < 0 || y > x || (y == x && j < i))) { x = y; i = j; }
}

template <typename Real> struct Wide;                // 16 bytes of logits, wherever a row starts
template <> struct Wide<double> { typedef double type __attribute__((ext_vector_type(2), aligned(8))); };
template <> struct Wide<float> { typedef float type __attribute__((ext_vector_type(4), aligned(4))); };

// A chunk of a row, 16 bytes a load: thread t has tokens j + (256 k + t) E + e as its element k E + e; -infinity behind the end.
template <typename Real>
__device__ __forceinline__ void load_chunk(Real (&to)[kPer], const Real *x, int64_t j, int64_t end) {
    using Vec = typename Wide<Real>::type;
    constexpr int E = 16 / sizeof(Real);
#pragma unroll
    for (int k = 0; k < kPer / E; ++k) {
        const int64_t i = j + (k * kVT + (int)threadIdx.x) * E;
        Vec v;
        if (i + E <= end) v = *reinterpret_cast<const Vec *>(x + i);
        else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = i + e < end ? x[i + e] : (Real)-INFINITY;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) to[k * E + e] = v[e];
    }
}
template <typename Real> __device__ __forceinline__ int in_chunk(int k) {              // which of the chunk's tokens element k is
    constexpr int E = 16 / sizeof(Real);
    return (k / E * kVT + (int)threadIdx.x) * E + k % E;
}
// The four tokens i .. i + 3.
template <typename Real>
__device__ __forceinline__ void load_few(Real (&to)[kFew], const Real *x, int64_t i, int64_t end) {
    using Vec = typename Wide<Real>::type;
    constexpr int E = 16 / sizeof(Real);
    if (i + kFew <= end) {
#pragma unroll
        for (int k = 0; k < kFew; k += E) {
            const Vec v = *reinterpret_cast<const Vec *>(x + i + k);
#pragma unroll
            for (int e = 0; e < E; ++e) to[k + e] = v[e];
        }
    } else {
#pragma unroll
        for (int k = 0; k < kFew; ++k) to[k] = i + k < end ? x[i + k] : (Real)-INFINITY;
    }
}

// A workgroup per row and segment.
template <typename Real, bool GREEDY>
__global__ void __launch_bounds__(kVT) verify_rows_kernel(VerifyArgs a) {
    __shared__ double s_max[kWaves], red[kWaves], s_exp[32];
    __shared__ int s_first[kWaves];
    const Exp e = exp_table(s_exp, a.inv_temp);
    const int64_t targets = a.B * (a.K + 1), at = blockIdx.x, of = at < targets ? a.K + 1 : a.K, row = at < targets ? at : at - targets;
    const Real *x = at < targets ? (const Real *)a.logits + row / of * a.seq + row % of * a.row
                                 : (const Real *)a.draft + row / of * a.draft_seq + row % of * a.draft_row;
    const int64_t j0 = blockIdx.y * a.segment, j1 = min(a.V, j0 + a.segment);
    double m = -INFINITY, s = 0.0;
    int first = -1;
    Real next[kPer];
    load_chunk(next, x, j0, j1);
    __syncthreads();
    for (int64_t j = j0; j < j1; j += kChunk) {
        Real v[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) v[k] = next[k];
        if (j + kChunk < j1) load_chunk(next, x, j + kChunk, j1);
        if (GREEDY) {
#pragma unroll
            for (int k = 0; k < kPer; ++k) if ((double)v[k] > m) { m = v[k]; first = (int)j + in_chunk<Real>(k); }
        } else {
            Real top = (Real)m;                       // (m is a logit, or -infinity)
#pragma unroll
            for (int k = 0; k < kPer; ++k) top = top < v[k] ? v[k] : top;
            s *= weight(e, m, top);
            m = top;
            if (m == INFINITY) {
#pragma unroll
                for (int k = 0; k < kPer; ++k) s += v[k] == INFINITY ? 1.0 : 0.0;
            } else {
                double part[2] = {0.0, 0.0};
#pragma unroll
                for (int k = 0; k < kPer; ++k) part[k & 1] += e((double)v[k] - m);
                s += part[0] + part[1];
            }
        }
    }
    RowStat *to = a.stat + at * a.segments + blockIdx.y;
    const double own = m;
    if (GREEDY) {
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) better(m, first, __shfl_xor(m, off, 64), __shfl_xor(first, off, 64));
        if ((threadIdx.x & 63) == 0) { s_max[threadIdx.x >> 6] = m; s_first[threadIdx.x >> 6] = first; }
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) better(m, first, s_max[w], s_first[w]);
        if (threadIdx.x == 0) *to = {m, 0.0, first, 0};
    } else {
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) m = fmax(m, __shfl_xor(m, off, 64));
        if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = m;
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) m = fmax(m, s_max[w]);
        double sum[1] = {s * weight(e, own, m)};
        block_sum(sum, red);
        if (threadIdx.x == 0) *to = {m, sum[0], 0, 0};
    }
}

__device__ __forceinline__ int drafts_of(const VerifyArgs &a, int64_t b) { return a.lengths ? max(0, min((int)a.K, a.lengths[b])) : (int)a.K; }

// What is left of p once q is taken off (or p itself) at tokens of one sequence's row n.
template <typename Real>
struct Left {
    const Real *x, *y;
    int64_t gone;                    // drafts without a distribution: the one that was refused
    Verdict v;
    double per_p, per_q;
    Exp e;
    __device__ Left(const VerifyArgs &a, int64_t b, const Verdict &v_, Exp e_) : v(v_), e(e_) {
        x = (const Real *)a.logits + b * a.seq + v.n * a.row;
        y = a.draft && v.left ? (const Real *)a.draft + b * a.draft_seq + v.n * a.draft_row : nullptr;
        gone = v.left ? a.drafts[b * a.K + v.n] : -1;
        per_p = 1.0 / v.p_sum;
        per_q = v.q_sum > 0 ? 1.0 / v.q_sum : 0.0;
    }
    // (px, qx: the logits at j)
    __device__ __forceinline__ double of(double px, double qx, int64_t j) const {
        const double p = weight(e, px, v.p_max) * per_p;
        if (!v.left) return p;
        return fmax(p - (y ? weight(e, qx, v.q_max) * per_q : j == gone ? 1.0 : 0.0), 0.0);
    }
};

// A workgroup per sequence and segment; each finds out for itself how many drafts are accepted: rows' segments put together by
// 16 lanes (64 where there are more), then a thread to a draft.  Then the weights of what the token is drawn from, piece by piece.
template <typename Real>
__global__ void __launch_bounds__(kLT) verify_left_kernel(VerifyArgs a) {
    __shared__ double red[kLT / 64], s_exp[32], s_max[2 * kMaxDrafts + 1], s_sum[2 * kMaxDrafts + 1];
    __shared__ Verdict s_v;
    const int64_t b = blockIdx.x;
    const int tid = threadIdx.x, count = drafts_of(a, b), K = (int)a.K;
    const Exp e = exp_table(s_exp, a.inv_temp);
    const RowStat *ps = a.stat + b * (K + 1) * a.segments, *qs = a.stat + (a.B * (K + 1) + b * K) * a.segments;
    // the drafts' own logits, on the way meanwhile
    int64_t d = -1;
    double px = -INFINITY, qx = -INFINITY, u = 0.0;
    if (tid < count) {
        d = a.drafts[b * K + tid];
        u = a.u[b * (K + 1) + tid];
        if (d >= 0 && d < a.V) {
            px = ((const Real *)a.logits)[b * a.seq + tid * a.row + d];
            if (a.draft) qx = ((const Real *)a.draft)[b * a.draft_seq + tid * a.draft_row + d];
        } else d = -1;
    }
    __syncthreads();
    const int lanes = a.segments <= 16 ? 16 : 64, rows = K + 1 + (a.draft ? K : 0);
    for (int row = tid / lanes; row < (int)round_up(rows, kLT / lanes); row += kLT / lanes) {
        const int i = tid % lanes;
        const bool in = row < rows && i < a.segments;
        const RowStat *s = (row <= K ? ps + row * a.segments : qs + (row - K - 1) * a.segments) + i;
        const double own = in ? s->max : -INFINITY;
        double max = own, sum = in ? s->sum : 0.0;
        for (int off = lanes / 2; off >= 1; off >>= 1) max = fmax(max, __shfl_xor(max, off, 64));
        sum *= weight(e, own, max);
        for (int off = lanes / 2; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
        if (in && i == 0) { s_max[row] = max; s_sum[row] = sum; }
    }
    __syncthreads();
    if (tid < 64) {
        bool taken = tid >= count;                    // (beyond the drafts nothing refuses)
        if (d >= 0 && s_sum[tid] > 0) {
            const double p = weight(e, px, s_max[tid]) / s_sum[tid];
            const double q = !a.draft ? 1.0 : s_sum[K + 1 + tid] > 0 ? weight(e, qx, s_max[K + 1 + tid]) / s_sum[K + 1 + tid] : 0.0;
            taken = u * q < p;
        }
        const unsigned long long refused = __ballot(!taken);
        if (tid == 0) {
            const int n = refused ? min(__ffsll(refused) - 1, count) : count;
            const bool left = n < count, of_drafts = left && a.draft;
            s_v = {s_max[n], s_sum[n], of_drafts ? s_max[K + 1 + n] : -INFINITY, of_drafts ? s_sum[K + 1 + n] : 0.0, n, left};
            if (blockIdx.y == 0) a.verdict[b] = s_v;
        }
    }
    __syncthreads();
    const Verdict v = s_v;
    if (!(v.p_sum > 0)) return;
    const Left<Real> left(a, b, v, e);
    const int64_t j0 = blockIdx.y * a.segment, j1 = min(a.V, j0 + a.segment);
    for (int64_t p0 = j0; p0 < j1; p0 += a.piece) {
        const int64_t p1 = min(j1, p0 + a.piece);
        double s = 0.0;
#pragma unroll 2
        for (int64_t j = p0 + tid * kFew; j < p1; j += kLT * kFew) {
            Real x[kFew], y[kFew];
            load_few(x, left.x, j, p1);
            if (left.y) load_few(y, left.y, j, p1);
#pragma unroll
            for (int k = 0; k < kFew; ++k) s += left.of(x[k], y[k], j + k);
        }
        s = wave_sum(s);
        __syncthreads();
        if ((tid & 63) == 0) red[tid >> 6] = s;
        __syncthreads();
        if (tid == 0) {
#pragma unroll
            for (int w = 1; w < kLT / 64; ++w) s += red[w];
            a.sums[b * kSegments + p0 / a.piece] = s;
        }
    }
}

// Accepted drafts, the token drawn, -1.
__device__ __forceinline__ void answer(const VerifyArgs &a, int64_t b, int n, int64_t drawn) {
    if (threadIdx.x <= a.K) a.tokens[b * (a.K + 1) + threadIdx.x] = threadIdx.x < n ? a.drafts[b * a.K + threadIdx.x] : threadIdx.x == n ? drawn : -1;
    if (threadIdx.x == 0) a.accepted[b] = n;
}

__device__ __forceinline__ double upto(double v, int lane) {                 // the lanes' values up to this one's
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) { const double o = __shfl_up(v, off, 64); if (lane >= off) v += o; }
    return v;
}

// A workgroup per sequence.
template <typename Real>
__global__ void __launch_bounds__(kDT) verify_pick_kernel(VerifyArgs a) {
    __shared__ double s_wave[kDWaves], s_aim, s_before, s_exp[32];
    __shared__ int s_piece, s_hit[kDWaves], s_last[kDWaves];
    const int64_t b = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Exp e = exp_table(s_exp, a.inv_temp);
    Verdict v = a.verdict[b];
    const int pieces = (int)ceil_div(a.V, a.piece);
    const double own = tid < pieces ? a.sums[b * kSegments + tid] : 0.0, u = a.u[b * (a.K + 1) + a.K];
    __syncthreads();
    if (!(v.p_sum > 0)) { answer(a, b, v.n, -1); return; }
    if (tid < 64) {
        // the piece that passes the aim first, or the last that has anything; where nothing is left, all of p, which adds up to 1
        const double run = upto(own, lane), aim = u * __shfl(run, 63, 64);
        const unsigned long long any = __ballot(own > 0.0), over = __ballot(own > 0.0 && run > aim);
        const int at = over ? __ffsll(over) - 1 : any ? 63 - __clzll(any) : 0;
        if (lane == at) { s_piece = any ? at : -1; s_before = any ? run - own : 0.0; s_aim = any ? aim : u; }
    }
    __syncthreads();
    if (s_piece < 0) v.left = 0;
    const Left<Real> left(a, b, v, e);
    const int64_t j0 = max(s_piece, 0) * a.piece, j1 = s_piece < 0 ? a.V : min(a.V, j0 + a.piece);
    const double aim = s_aim;
    double before = s_before;
    int pick = -1, nearly = -1;                       // rounding can leave no token over the aim: then the segment's last that has weight
    for (int64_t j = j0; j < j1; j += kChunk) {                         // (one chunk, unless the vocabulary is over kSegments of them or nothing was left)
        const int64_t i0 = j + tid * kFew;
        double w[kFew], own = 0.0;
        Real x[kFew], y[kFew];
        load_few(x, left.x, i0, j1);
        if (left.y) load_few(y, left.y, i0, j1);
#pragma unroll
        for (int k = 0; k < kFew; ++k) { w[k] = left.of(x[k], y[k], i0 + k); own += w[k]; }
        double run = upto(own, lane);
        if (lane == 63) s_wave[wave] = run;
        __syncthreads();
        double after = before;
        run += before - own;
#pragma unroll
        for (int q = 0; q < kDWaves; ++q) { run += q < wave ? s_wave[q] : 0.0; after += s_wave[q]; }
        int hit = 0x7fffffff, last = -1;
#pragma unroll
        for (int k = 0; k < kFew; ++k) {
            run += w[k];
            if (w[k] > 0.0) { last = (int)(i0 + k); if (run > aim && hit == 0x7fffffff) hit = last; }
        }
        // (the first of the wavefront's hits and the last of its tokens with weight; an LDS atomic of 1024 lanes takes 3 us)
        const unsigned long long hits = __ballot(hit != 0x7fffffff), some = __ballot(last >= 0);
        if (hits ? lane == __ffsll(hits) - 1 : lane == 0) s_hit[wave] = hit;
        if (some ? lane == 63 - __clzll(some) : lane == 0) s_last[wave] = last;
        __syncthreads();
#pragma unroll
        for (int q = kDWaves - 1; q >= 0; --q) if (s_hit[q] != 0x7fffffff) pick = s_hit[q];
        if (pick >= 0) break;
#pragma unroll
        for (int q = 0; q < kDWaves; ++q) if (s_last[q] >= 0) nearly = s_last[q];
        before = after;
    }
    answer(a, b, v.n, pick >= 0 ? pick : nearly);
}

// A workgroup per sequence, 16 lanes to a row.
__global__ void __launch_bounds__(kVT) verify_greedy_kernel(VerifyArgs a) {
    __shared__ int best[kMaxDrafts + 1];
    const int64_t b = blockIdx.x;
    const int tid = threadIdx.x, count = drafts_of(a, b), K = (int)a.K;
    const int64_t d = tid < count ? a.drafts[b * K + tid] : -1;
    for (int row = tid / 16; row < (int)round_up(K + 1, kVT / 16); row += kVT / 16) {
        const RowStat *s = a.stat + (b * (K + 1) + min(row, K)) * a.segments;
        double m = -INFINITY;
        int first = -1;
        for (int i = tid % 16; i < a.segments; i += 16) better(m, first, s[i].max, s[i].first);
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) better(m, first, __shfl_xor(m, off, 64), __shfl_xor(first, off, 64));
        if (tid % 16 == 0 && row <= K) best[row] = first;
    }
    __syncthreads();
    __shared__ int s_n;
    if (tid < 64) {
        const unsigned long long refused = __ballot(tid < count && !(best[min(tid, K)] >= 0 && best[min(tid, K)] == d));
        if (tid == 0) s_n = refused ? min(__ffsll(refused) - 1, count) : count;
    }
    __syncthreads();
    answer(a, b, s_n, best[s_n]);
}

struct VerifyPlan {
    int segments;
    int64_t segment, piece;
    size_t stat_bytes, sum_bytes, verdict_bytes;
    VerifyPlan(int64_t B, int64_t K, int64_t V) {
        // no more workgroups than fill the device a few times: each costs as much as 2000 tokens
        int64_t wanted = ceil_div(4096, B * (2 * K + 1));
        if (wanted > kSegments) wanted = kSegments;
        piece = round_up(ceil_div(V, kSegments), kChunk);
        segment = round_up(ceil_div(V, wanted), piece);
        segments = (int)ceil_div(V, segment);
        stat_bytes = (size_t)(B * (2 * K + 1) * segments) * sizeof(RowStat);
        sum_bytes = (size_t)(B * kSegments) * 8;
        verdict_bytes = (size_t)B * sizeof(Verdict);
    }
    size_t bytes() const { return stat_bytes + sum_bytes + verdict_bytes; }
};

}  // namespace

}  // namespace rwkv

using namespace rwkv;

extern "C" {

size_t rwkv_verify_drafts_workspace_bytes(int64_t B, int64_t K, int64_t V) {
    if (B <= 0 || K < 0 || V <= 0) return 0;
    return VerifyPlan(B, K, V).bytes();
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
    if (K > kMaxDrafts || V >= (1ll << 31)) return set_error(RWKV_ERR_SIZE, "rwkv_verify_drafts: at most %d drafts", kMaxDrafts);
    if (B >= (1ll << 24) || !launchable(B * (2 * K + 1), kVT) || !launchable(B, kDT)) return set_error(RWKV_ERR_SIZE, "rwkv_verify_drafts: too many sequences");
    RWKV_CHECK_ALIGN(workspace, 16);
    const VerifyPlan pl(B, K, V);
    if (!workspace || workspace_bytes < pl.bytes()) return set_error(RWKV_ERR_WORKSPACE, "rwkv_verify_drafts: workspace too small");
    const bool of_drafts = draft_logits && !greedy && K > 0;
    const int64_t e = (int64_t)type_bytes(real), token_bytes = B * (K + 1) * 8;
    auto apart = [&](const void *from, int64_t bytes) {
        return !from || bytes <= 0 || (!rows_share(1, tokens, 0, token_bytes, from, 0, bytes) && !rows_share(1, accepted, 0, B * 8, from, 0, bytes));
    };
    RWKV_CHECK_ARG(apart(logits, ((B - 1) * logits_seq_stride + K * logits_row_stride + V) * e) &&
                       apart(of_drafts ? draft_logits : nullptr, ((B - 1) * draft_seq_stride + (K - 1) * draft_row_stride + V) * e) && apart(drafts, B * K * 8) &&
                       apart(lengths, B * 4) && apart(greedy ? nullptr : u, B * (K + 1) * 4) && !rows_share(1, tokens, 0, token_bytes, accepted, 0, B * 8),
                   "rwkv_verify_drafts: tokens or accepted share memory with another argument");
    uint8_t *ws = (uint8_t *)workspace;
    const VerifyArgs a{B, K, V, logits, logits_seq_stride, logits_row_stride, of_drafts ? draft_logits : nullptr, draft_seq_stride, draft_row_stride,
                       drafts, lengths, u, 1.0 / std::max(temp, 1e-300), tokens, accepted, pl.segments, pl.segment, (RowStat *)ws, pl.piece, (double *)(ws + pl.stat_bytes),
                       (Verdict *)(ws + pl.stat_bytes + pl.sum_bytes)};
    const hipStream_t st = (hipStream_t)stream;
    const dim3 rows((unsigned)(B * (K + 1) + (of_drafts ? B * K : 0)), (unsigned)pl.segments), left((unsigned)B, (unsigned)pl.segments);
    with_real(real, [&](auto re) {
        using Real = typename decltype(re)::type;
        if (greedy) {
            hipLaunchKernelGGL((verify_rows_kernel<Real, true>), rows, dim3(kVT), 0, st, a);
            hipLaunchKernelGGL(verify_greedy_kernel, dim3((unsigned)B), dim3(kVT), 0, st, a);
        } else {
            hipLaunchKernelGGL((verify_rows_kernel<Real, false>), rows, dim3(kVT), 0, st, a);
            hipLaunchKernelGGL(verify_left_kernel<Real>, left, dim3(kLT), 0, st, a);
            hipLaunchKernelGGL(verify_pick_kernel<Real>, dim3((unsigned)B), dim3(kDT), 0, st, a);
        }
    });
    RWKV_CHECK_LAUNCH("verify_pick_kernel");
    return RWKV_OK;
}

}  // extern "C"
