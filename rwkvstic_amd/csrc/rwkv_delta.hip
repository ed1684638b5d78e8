// The gated delta rule over packed sequences (rwkv_delta_rule), per value head with a state S [dk, dv]:
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = scale S^T q.
//
// Few rows a sequence: step by step (delta_steps_kernel), a wavefront to 16 columns of the state; the state is read and written once.
// Many: in chunks of 64 rows.  With G_i = g_1 + .. + g_i within the chunk and K, Q, V its rows,
//   U = T (V - e^G K S),  T = (1 + A)^-1 diag(beta),  A_ij = beta_i e^(G_i - G_j) k_i.k_j below the diagonal,
//   O = scale e^G Q S + P U,  P_ij = scale e^(G_i - G_j) q_i.k_j up to the diagonal,  S <- e^G_64 S + K^T (e^(G_64 - G) U).
//   delta_within_kernel   T and P of every chunk, all at once
//   delta_chunks_kernel   chunk after chunk, a wavefront to 16 columns of the state
// Where that leaves most of the device idle (few sequences and heads), a sequence is cut into segments: what a segment makes of the
// state before it, S -> M S + N, is computed for all of them side by side (the chunks from 0, and from the identity without values), then
//   delta_join_kernel     puts the segments together, for the state in front of each,
// and the segments are gone through once more from there, for their outputs.
// Both on the matrix cores with float32 sums; G and its differences are float64, as a decay is the exponential of a difference of sums.
// A float32 operand goes into the bfloat16 matrix instructions as the sum of three bfloat16 values, its 24 bits cut in three
// (planes); of the products of planes those whose numbers (0, 1, 2) add up to three or more are left out, 2^-24.5 of a product
// on average, 2^-21 at most (and planes under 2^-126, which the instructions take for 0: up to 2^-125 of a value under 2^-103): three products with bfloat16 keys (nothing left out), six of two float32 operands, against 16 times the
// time of one for float32 instructions.  (Two planes for what only reaches a bfloat16 output are not enough: with keys that repeat,
// Q S and P U cancel.)
#include "rwkv_types.h"

#include <type_traits>

namespace rwkv {

namespace {

struct DeltaArgs {
    int64_t T, B, each;                   // each: rows of a sequence where there are no starts
    int share, Hv, dk, dv;                // share: value heads to a key head
    const void *q, *k, *v; int64_t q_stride, k_stride, v_stride;
    const float *g, *beta;
    float scale;
    const int32_t *starts;
    float *state;
    void *o;
    int segments;                         // of a sequence, as many as its chunks allow
    float *ends, *fronts;                 // with segments: [B][Hv][segments][dk][across] N and M; [B][Hv][segments][dk][dv] states in front
    int values, across;                   // columns of N, dv filled up to 64s, and of N and M, with dk filled up to the kernel's tiles
};

// First row and number of rows of sequence b, cut to the rows there are.
__device__ __forceinline__ void rows_of(const DeltaArgs &a, int64_t b, int64_t &first, int64_t &n) {
    if (!a.starts) { n = a.each; first = b * n; return; }
    const int64_t lo = a.starts[b], hi = a.starts[b + 1];
    first = min(max(lo, (int64_t)0), a.T);
    n = max(min(hi, a.T) - first, (int64_t)0);
}

// The sequence at a place of the order in which they are begun: the longest first, so that none of them is begun when the others are
// nearly done; as they come where there are more than a wavefront's lanes.  (8192 rows of seven ragged sequences, 32 heads of
// 128 x 128, bfloat16: 248 us against 270)
__device__ __forceinline__ int64_t begun(const DeltaArgs &a, int64_t at) {
    if (!a.starts || a.B > 64) return at;
    const int lane = threadIdx.x & 63;
    int64_t first, n = -1;
    if (lane < a.B) rows_of(a, lane, first, n);
    int before = 0;
    for (int other = 0; other < a.B; ++other) {
        const int m = __builtin_amdgcn_readlane((int)n, other);
        before += m > (int)n || (m == (int)n && other < lane);
    }
    return __ffsll((long long)__ballot(before == (int)at)) - 1;
}

// A segment of a sequence of n rows: its first chunk, and how many; none where the sequence has fewer.
__device__ __forceinline__ int64_t segment_of(const DeltaArgs &a, int64_t n, int segment, int64_t &begin) {
    const int64_t chunks = (n + 63) / 64, each = (chunks + a.segments - 1) / a.segments;
    begin = segment * each;
    return max(min(each, chunks - begin), (int64_t)0);
}

// Sum over the 16 lanes of a DPP row, in every one of them.
template <int CTRL>
__device__ __forceinline__ float turned(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false)); }
__device__ __forceinline__ float row_sum(float v) {
    v += turned<0x128>(v);                            // row_ror:8, 4, 2, 1
    v += turned<0x124>(v);
    v += turned<0x122>(v);
    return v + turned<0x121>(v);
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <typename T, int N> struct Some { typedef T type __attribute__((ext_vector_type(N))); };

// N neighbouring elements of a row of n from k on, zeros behind its end; WIDE: aligned to their size, up to 16 bytes, and n a multiple of N.
template <int N, bool WIDE, typename T>
__device__ __forceinline__ typename Some<T, N>::type take(const T *row, int k, int n) {
    typename Some<T, N>::type to;
    if constexpr (WIDE) {
        if (k >= n) return (T)0.f;
        if constexpr (N * sizeof(T) <= 16) return *reinterpret_cast<const typename Some<T, N>::type *>(row + k);
        constexpr int E = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < N; i += E) {
            const auto v = *reinterpret_cast<const typename Some<T, E>::type *>(row + k + i);
#pragma unroll
            for (int e = 0; e < E; ++e) to[i + e] = v[e];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = k + i < n ? row[k + i] : (T)0.f;
    }
    return to;
}

// Lane (c, r) = (lane / 16, lane % 16) holds rows NR r .. NR r + NR - 1 of columns 4 c .. 4 c + 3, so that the sums over a
// column's rows stay in a DPP row and no wavefront waits for another.  Both products are taken with the state before the step, so
// that their sums are made side by side: S'^T q = e^g S^T q + (k.q) u.  The next row is under way meanwhile.
// Memory bounds it at a row each (32 sequences, 40 heads of 64 x 64, float32: 10.5 us for 42 MB, 4.0 TB/s), from a few rows on the
// instructions of a step (16 ragged sequences of 80 rows, 32 heads of 128 x 128: 27 us, 14.6 of it for the state).
template <typename T, int NR, bool WIDE>
__global__ void __launch_bounds__(256) delta_steps_kernel(DeltaArgs a, int tiles) {
    const int64_t job = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (job >= a.B * a.Hv * tiles) return;
    const int lane = threadIdx.x & 63, r = lane & 15, col = (int)(job % tiles) * 16 + (lane >> 4) * 4;
    const int h = (int)(job / tiles % a.Hv), hk = h / a.share;
    const int64_t b = job / tiles / a.Hv;
    int64_t first, n;
    rows_of(a, b, first, n);
    if (n <= 0) return;
    const T *q = (const T *)a.q + first * a.q_stride + (int64_t)hk * a.dk, *k = (const T *)a.k + first * a.k_stride + (int64_t)hk * a.dk;
    const T *v = (const T *)a.v + first * a.v_stride + (int64_t)h * a.dv;
    T *o = (T *)a.o + (first * a.Hv + h) * a.dv;
    const float *g = a.g + first * a.Hv + h, *beta = a.beta + first * a.Hv + h;
    float *state = a.state + (b * a.Hv + h) * a.dk * a.dv;
    struct Row { typename Some<T, NR>::type k, q; typename Some<T, 4>::type v; float g, beta; };
    auto load = [&](Row &to, int64_t t) {
        to.k = take<NR, WIDE>(k + t * a.k_stride, r * NR, a.dk);
        to.q = take<NR, WIDE>(q + t * a.q_stride, r * NR, a.dk);
        to.v = take<4, WIDE>(v + t * a.v_stride, col, a.dv);
        to.g = g[t * a.Hv]; to.beta = beta[t * a.Hv];
    };
    Row next;
    load(next, 0);
    f32x4 S[NR];                                      // (rows and columns there are not: others, and zeros in their place)
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const float *row = state + (int64_t)min(r * NR + i, a.dk - 1) * a.dv;
        if (WIDE) S[i] = *reinterpret_cast<const f32x4 *>(row + (col < a.dv ? col : 0));
        else {
#pragma unroll
            for (int c = 0; c < 4; ++c) S[i][c] = row[min(col + c, a.dv - 1)];
        }
    }
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) S[i][c] = r * NR + i < a.dk ? S[i][c] : 0.f;
    // (a row's output is stored a step later, in front of the next loads: behind them, they would be waited for together)
    float out = 0.f;
    auto store = [&](int64_t t) { if (r < 4 && col + r < a.dv) o[t * a.Hv * a.dv + col + r] = (T)out; };
#pragma unroll 1
    for (int64_t t = 0; t < n; ++t) {
        const Row now = next;
        if (t) store(t - 1);
        if (t + 1 < n) load(next, t + 1);
        const float e = expf(now.g);
        float kq = 0.f;
        f32x4 kS = {0, 0, 0, 0}, qS = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const float kk = now.k[i], qq = now.q[i];
            kq = fmaf(kk, qq, kq);
#pragma unroll
            for (int c = 0; c < 4; ++c) { kS[c] = fmaf(kk, S[i][c], kS[c]); qS[c] = fmaf(qq, S[i][c], qS[c]); }
        }
        kq = row_sum(kq);
        float u[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            u[c] = now.beta * ((float)now.v[c] - e * row_sum(kS[c]));
            const float y = a.scale * (e * row_sum(qS[c]) + kq * u[c]);
            out = r == c ? y : out;
        }
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) S[i][c] = fmaf(e, S[i][c], (float)now.k[i] * u[c]);
    }
    store(n - 1);
    if (col >= a.dv) return;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        if (r * NR + i >= a.dk) break;
        float *row = state + (int64_t)(r * NR + i) * a.dv + col;
        if (WIDE) *reinterpret_cast<f32x4 *>(row) = S[i];
        else {
#pragma unroll
            for (int c = 0; c < 4; ++c) if (col + c < a.dv) row[c] = S[i][c];
        }
    }
}

// ---- chunks -----------------------------------------------------------------------------------------------------------
constexpr int kChunk = 64;
constexpr int kBlocks = 10;                          // 16 x 16 blocks up to the diagonal
// What delta_within_kernel leaves of a chunk and head, in units of 4 floats: T block by block, a unit to lane (i, g) with terms
// 4 g .. 4 g + 3 of row i; P; e^G; e^(G_64 - G).
constexpr int kUnitP = kBlocks * 64, kUnitG = 2 * kUnitP, kUnits = kUnitG + 2 * kChunk / 4;
constexpr float kForgotten = -1e5f;                  // a decay's logarithm below which nothing is left; -infinity would have no differences

// Lane (j, g) = (lane % 16, lane / 16) holds rows 4 g + v, v < 4, of column j of a 16 x 16 product.  As a right operand it is to
// hold one term k of column j at a time; the order of the terms being free, what a product leaves in the registers is the next
// one's right operand, term 4 g + v in the v-th of four instructions, if lane (i, g) has terms 4 g .. 4 g + 3 of row i of the left one.
__device__ __forceinline__ void add_product(f32x4 &acc, const f32x4 &left, const f32x4 &right) {
#pragma unroll
    for (int v = 0; v < 4; ++v) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(left[v], right[v], acc, 0, 0, 0);
}

// Chunks of sequence b have the places first / 64 + b and on: no two the same, none past T / 64 + B.
__device__ __forceinline__ int64_t place_of(int64_t first, int64_t b) { return first / kChunk + b; }

constexpr __host__ __device__ int block_of(int row, int column) { return row * (row + 1) / 2 + column; }
constexpr __host__ __device__ int row_of(int block) { return block < 1 ? 0 : block < 3 ? 1 : block < 6 ? 2 : 3; }
constexpr int kPairs = 6;                            // blocks two by two, as the matrix instructions take them: (row, columns 32 p .. 32 p + 31)
constexpr __host__ __device__ int pair_of(int row, int p) { return row < 2 ? row : 2 * (row - 1) + p; }

// Planes: bfloat16 values, most significant first, that add up to a float32 (or are its first 8 or 16 bits).
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
template <int N> struct Planes { u32x4 p[N]; };                 // of eight values
__device__ __forceinline__ float rest(float v) { return v - __uint_as_float(__float_as_uint(v) & 0xffff0000u); }
__device__ __forceinline__ uint32_t upper(float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u); }
template <int N> __device__ __forceinline__ Planes<N> planes(f32x4 a, f32x4 b) {
    Planes<N> to;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        to.p[n] = u32x4{upper(a[0], a[1]), upper(a[2], a[3]), upper(b[0], b[1]), upper(b[2], b[3])};
        if (n + 1 < N)
#pragma unroll
            for (int c = 0; c < 4; ++c) { a[c] = rest(a[c]); b[c] = rest(b[c]); }
    }
    return to;
}
// acc[m] += left[m] x right, of the planes' products those whose numbers add up to less than 3, the small ones first; products of
// different sums one after the other, as the next one of the same sum has to wait for it.  SWAPPED: the transposed product, of the same
// registers: lane (j, g) gets columns 4 g + v of row j.
template <bool SWAPPED = false, int M, int A, int B> __device__ __forceinline__ void add_planes(f32x4 (&acc)[M], const Planes<A> (&left)[M], const Planes<B> &right) {
#pragma unroll
    for (int sum = 2; sum >= 0; --sum)
#pragma unroll
        for (int n = 0; n <= sum; ++n)
            if (n < A && sum - n < B)
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    const bf16x8 l = __builtin_bit_cast(bf16x8, left[m].p[n]), r = __builtin_bit_cast(bf16x8, right.p[sum - n]);
                    acc[m] = SWAPPED ? __builtin_amdgcn_mfma_f32_16x16x32_bf16(r, l, acc[m], 0, 0, 0) : __builtin_amdgcn_mfma_f32_16x16x32_bf16(l, r, acc[m], 0, 0, 0);
                }
}

// Planes of a value of type T (float16: 8 and 3 bits).
template <typename T> constexpr int kPlanes = sizeof(T) == 4 ? 3 : std::is_same_v<T, __bf16> ? 1 : 2;
__device__ __forceinline__ Planes<1> planes_of(bf16x8 v) { return {{__builtin_bit_cast(u32x4, v)}}; }
template <typename V> __device__ __forceinline__ auto planes_of(V v) {
    return planes<kPlanes<std::decay_t<decltype(v[0])>>>(f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]}, f32x4{(float)v[4], (float)v[5], (float)v[6], (float)v[7]});
}


// Products of 16 rows with 16 rows, lane (i, g) giving the i-th of each: the operands' own type where the matrix cores have it
// (the products are exact), else float32.  The rows come from memory straight into the registers that the instruction reads.
__device__ __forceinline__ f32x4 dot_step(Some<float, 4>::type l, Some<float, 4>::type r, f32x4 acc) { add_product(acc, l, r); return acc; }
__device__ __forceinline__ f32x4 dot_step(Some<__bf16, 8>::type l, Some<__bf16, 8>::type r, f32x4 acc) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(l, r, acc, 0, 0, 0); }
__device__ __forceinline__ f32x4 dot_step(Some<_Float16, 8>::type l, Some<_Float16, 8>::type r, f32x4 acc) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(l, r, acc, 0, 0, 0); }

// T and P of one chunk and value head; (1 + A)^-1 by blocks of 16.  A chain of short dependent parts bounds it (640 workgroups of 64
// channels, float32: 18.5 us; 4096 of 128, bfloat16: 68 us).  Blocks go to the wavefronts by rows: dealt out evenly they need twice the
// loads (23 and 87 us).
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) delta_within_kernel(DeltaArgs a, f32x4 *slots) {
    __shared__ double s_G[kChunk];
    __shared__ float s_beta[kChunk];
    __shared__ __align__(16) float s_A[kChunk][kChunk + 4], s_X[4][16][20];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, g = lane >> 4;
    const int h = blockIdx.y, hk = h / a.share;
    const int64_t place = blockIdx.x;
    // the last sequence whose places begin here or before
    int64_t b = -1;
    for (int64_t b0 = 0; b0 < a.B; b0 += 64) {
        int64_t first = 0, n = 0;
        if (b0 + lane < a.B) rows_of(a, b0 + lane, first, n);
        const unsigned long long upto = __ballot(b0 + lane < a.B && place_of(first, b0 + lane) <= place);
        if (upto) b = b0 + 63 - __clzll(upto);
    }
    if (b < 0) return;
    int64_t first, n;
    rows_of(a, b, first, n);
    const int64_t done = (place - place_of(first, b)) * kChunk;
    if (done >= n) return;
    first += done;
    const int live = (int)min((int64_t)kChunk, n - done);
    // (rows behind the last: the last again; beta is 0 there, and what comes of them is not used)
    const T *keys = (const T *)a.k + first * a.k_stride + (int64_t)hk * a.dk, *queries = (const T *)a.q + first * a.q_stride + (int64_t)hk * a.dk;
    f32x4 *slot = slots + (place * a.Hv + h) * kUnits;
    if (wave == 0) {
        float decay = lane < live ? a.g[(first + lane) * a.Hv + h] : 0.f;
        if (decay < kForgotten) decay = kForgotten;
        double G = decay;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) { const double before = __shfl_up(G, off, 64); if (lane >= off) G += before; }
        s_G[lane] = G;
        s_beta[lane] = lane < live ? a.beta[(first + lane) * a.Hv + h] : 0.f;
        float *decays = reinterpret_cast<float *>(slot + kUnitG);
        decays[lane] = expf((float)G);
        decays[kChunk + lane] = expf((float)(__shfl(G, 63, 64) - G));
    }
    // transposed products, so that a lane has four neighbours of a row: of the wavefront's row of blocks, whose keys are an operand of all
    constexpr int E = sizeof(T) == 4 ? 4 : 8;
    f32x4 kk[4], qk[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) kk[c] = qk[c] = f32x4{0, 0, 0, 0};
    auto products = [&](auto count) {
        constexpr int N = decltype(count)::value;            // blocks of the row
        const T *kr[N], *qr = queries + min(16 * (N - 1) + i, live - 1) * a.q_stride;
#pragma unroll
        for (int c = 0; c < N; ++c) kr[c] = keys + min(16 * c + i, live - 1) * a.k_stride;
        auto terms = [&](int k, auto whole) {                 // (whole: none of the block's 4 E terms is behind the last)
            auto some = [&](const T *row) {
                if constexpr (decltype(whole)::value && WIDE) return *reinterpret_cast<const typename Some<T, E>::type *>(row + k);
                else return take<E, WIDE>(row, k, a.dk);
            };
            typename Some<T, E>::type l[N], q = some(qr);
#pragma unroll
            for (int c = 0; c < N; ++c) l[c] = some(kr[c]);
#pragma unroll
            for (int c = 0; c < N; ++c) { kk[c] = dot_step(l[c], l[N - 1], kk[c]); qk[c] = dot_step(l[c], q, qk[c]); }
        };
        int k = 0;
#pragma unroll 4
        for (; k + 4 * E <= a.dk; k += 4 * E) terms(k + E * g, std::true_type{});
        if (k < a.dk) terms(k + E * g, std::false_type{});
    };
    if (wave == 0) products(std::integral_constant<int, 1>{});
    else if (wave == 1) products(std::integral_constant<int, 2>{});
    else if (wave == 2) products(std::integral_constant<int, 3>{});
    else products(std::integral_constant<int, 4>{});
    __syncthreads();
    // A into LDS, P out
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (c > wave) break;
        const int block = block_of(wave, c), row = 16 * wave + i;
        f32x4 A, P;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int column = 16 * c + 4 * g + v;
            const float decay = expf((float)(s_G[row] - s_G[column]));
            A[v] = column < row ? s_beta[row] * decay * kk[c][v] : 0.f;
            P[v] = column <= row ? a.scale * decay * qk[c][v] : 0.f;
        }
        *reinterpret_cast<f32x4 *>(&s_A[row][16 * c + 4 * g]) = A;
        slot[kUnitP + block * 64 + lane] = P;
    }
    __syncthreads();
    // (1 + A)^-1: the blocks on the diagonal by substitution, a lane to a column ...
    if (lane < 16) {
        float x[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float s = r == lane ? 1.f : 0.f;
#pragma unroll
            for (int l = 0; l < r; ++l) s = fmaf(-s_A[16 * wave + r][16 * wave + l], x[l], s);
            x[r] = s;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s_X[wave][r][lane] = x[r];
    }
    __syncthreads();
    // ... the others below them, a wavefront to a column of blocks: X_mc = -X_mm sum_l A_ml X_lc; 0 above the diagonal.  Chosen without
    // branches: with "if (m > wave)" around the products, wave being scalar, what clang 22 builds goes from a product through two jumps
    // to the read of its registers, 3 instructions where 10 are needed, and T came out wrong.  (With a wave that differs from lane to lane
    // it waits, and so it does where the branches of products() above meet.)
    f32x4 X[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        f32x4 Y = {0, 0, 0, 0}, below = {0, 0, 0, 0};
#pragma unroll
        for (int l = 0; l < m; ++l) add_product(Y, *reinterpret_cast<const f32x4 *>(&s_A[16 * m + i][16 * l + 4 * g]), X[l]);
        if (m) add_product(below, *reinterpret_cast<const f32x4 *>(&s_X[m][i][4 * g]), -Y);
#pragma unroll
        for (int v = 0; v < 4; ++v) X[m][v] = m == wave ? s_X[m][4 * g + v][i] : m > wave ? below[v] : 0.f;
    }
    __syncthreads();
    // by rows again, through LDS: a wavefront writes and reads its own columns only
    const float beta = s_beta[16 * wave + i];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int v = 0; v < 4; ++v) if (m >= wave) s_A[16 * m + 4 * g + v][16 * wave + i] = X[m][v] * beta;
    __syncthreads();
#pragma unroll
    for (int m = 0; m < 4; ++m)
        if (m >= wave) slot[block_of(m, wave) * 64 + lane] = *reinterpret_cast<const f32x4 *>(&s_A[16 * m + i][16 * wave + 4 * g]);
}

// What a workgroup of the chunks goes through: a segment of a sequence, for 64 columns of a value head's state.
// SUMMARY: a segment's N (the columns of the values, from 0 or, the first segment, from the state) and M (columns behind them, from the
// identity, of no values); no outputs.
struct Work {
    int segment, h, hk, col0, col;
    bool identity, at_end, in;
    int64_t b, bh, begin, first, n;       // begin: chunks of the sequence in front of it; its rows
    const f32x4 *slot;
};
template <bool SUMMARY> __device__ __forceinline__ bool work_of(const DeltaArgs &a, const f32x4 *slots, int groups, Work &w) {
    const int places = SUMMARY ? a.across / 64 : groups, place = (int)(blockIdx.x % places);
    const uint32_t unit = blockIdx.x / places, heads = (uint32_t)(a.B * a.Hv);          // (segments last: each compute unit gets some of all)
    w.segment = (int)(unit / heads); w.h = (int)(unit % a.Hv); w.hk = w.h / a.share;
    w.b = begun(a, unit % heads / a.Hv); w.bh = w.b * a.Hv + w.h;
    w.identity = SUMMARY && place >= groups;
    w.col0 = (place - (w.identity ? groups : 0)) * 64;
    w.col = w.col0 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 16 + (threadIdx.x & 15);
    w.in = w.col < a.dv;
    rows_of(a, w.b, w.first, w.n);
    if (w.n <= 0) return false;
    const int64_t chunks = segment_of(a, w.n, w.segment, w.begin);
    w.at_end = (w.begin + chunks) * kChunk >= w.n;
    if (chunks <= 0 || (SUMMARY && (w.at_end || (w.identity && w.segment == 0)))) return false;
    w.slot = slots + ((place_of(w.first, w.b) + w.begin) * a.Hv + w.h) * kUnits;
    w.first += w.begin * kChunk;
    w.n = min(w.n - w.begin * kChunk, chunks * kChunk);
    return true;
}
template <bool SUMMARY, int NK> __device__ __forceinline__ void begin_with(const DeltaArgs &a, const Work &w, f32x4 (&S)[NK]) {
    float *const state = a.state + w.bh * a.dk * a.dv, *const front = a.fronts + (w.bh * a.segments + w.segment) * a.dk * a.dv;
    const float *const from = SUMMARY || (w.segment == 0 && w.at_end) ? state : front;          // (a sequence of one segment has no summary)
    const int g = threadIdx.x >> 4 & 3;
#pragma unroll
    for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int row = 16 * k + 4 * g + v;
            if (SUMMARY && (w.identity || w.segment)) S[k][v] = w.identity && row == w.col && row < a.dk ? 1.f : 0.f;
            else {
                S[k][v] = row < a.dk ? from[(int64_t)row * a.dv + (w.in ? w.col : 0)] : 0.f;
                if (SUMMARY && w.in && row < a.dk) front[(int64_t)row * a.dv + w.col] = S[k][v];          // (the last segment writes the state while the first reads it)
            }
        }
}
template <bool SUMMARY, int NK> __device__ __forceinline__ void end_with(const DeltaArgs &a, const Work &w, int groups, const f32x4 (&S)[NK]) {
    float *const state = a.state + w.bh * a.dk * a.dv, *const ends = a.ends + (w.bh * a.segments + w.segment) * a.dk * a.across + (w.identity ? groups * 64 : 0);
    const int g = threadIdx.x >> 4 & 3;
#pragma unroll
    for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int row = 16 * k + 4 * g + v;
            if (row >= a.dk) continue;
            if (SUMMARY) { if (!w.identity || w.col < NK * 16) ends[(int64_t)row * a.across + w.col] = S[k][v]; }
            else if (w.at_end && w.in) state[(int64_t)row * a.dv + w.col] = S[k][v];
        }
}

// NK tiles of 16 key channels; four wavefronts of 16 columns of the state each.  S, and what is multiplied with it and comes of it,
// stay in the wavefront's registers; the left operands lie in LDS, where a lane's eight terms are 16 bytes:
//   K, Q   [plane][row][block of 32 channels][unit g ^ (row / 16)], unit g: channels 4 g .. + 3 and 16 + 4 g .. + 3 of the block
//   K^T    [plane][channel][block of 32 rows][unit g], the same of rows; channels 144 bytes apart
//   T, P   [pair][plane][lane]; then e^G and e^(G_64 - G)
//   V^T    [column][row], columns 64 rows and 16 bytes apart
// A wavefront has its SIMD to itself, so what fetches the next chunk and puts it into LDS stands between the products of this one,
// each part as soon as its place is free: K, Q and V by pieces of a few rows of eight channels to a thread, T and P by blocks.
// What bounds it is the instructions that one wavefront issues, some 4.5 us a chunk of 128 bfloat16 channels (float32, 64: 5.6).
template <typename T, int NK> struct Chunks {
    static constexpr int kIn = kPlanes<T>, kRowBytes = NK * 32 + 16, kPlane = kChunk * kRowBytes, kTransposed = NK * 16 * 144;
    static constexpr int kQ = kIn * kPlane, kT = 2 * kQ, kPairsAt = kT + kIn * kTransposed, kDecays = kPairsAt + 2 * kPairs * 3 * 1024, kV = kDecays + 2 * kChunk * 4;
    static constexpr int kColumn = kChunk * sizeof(T) + 16, kBytes = kV + 64 * kColumn;
    static constexpr int kRows = NK >= 8 ? 4 : 2, kPieces = NK * 2 * (kChunk / kRows) / kThreads;          // rows of a piece of K or Q, pieces of a thread
};

template <typename T, int NK, bool WIDE, bool SUMMARY>
__global__ void __launch_bounds__(kThreads, NK <= 4 ? 2 : 1) delta_chunks_kernel(DeltaArgs a, const f32x4 *slots, int groups) {
    using C = Chunks<T, NK>;
    using V8 = typename Some<T, 8>::type;
    using V4 = typename Some<T, 4>::type;
    constexpr int kIn = C::kIn, kRows = C::kRows, kPieces = C::kPieces, kAcross = kChunk / kRows;
    extern __shared__ __align__(16) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, g = lane >> 4;
    Work w;
    if (!work_of<SUMMARY>(a, slots, groups, w)) return;
    const int h = w.h, hk = w.hk, col0 = w.col0;
    const bool identity = w.identity;
    const int64_t first = w.first, n = w.n;
    const f32x4 *slot = w.slot;
    const int64_t end = (n - 1) / kChunk * kChunk;       // the last chunk
    // Offsets within a chunk fit 32 bits (the host has looked).  Rows behind the last are the last again, columns the first: T's
    // columns are 0 there, and what comes of them is not written.  Behind the last chunk it is fetched again.
    auto piece = [&](V8 *to, const T *from, int64_t stride, int64_t done, int count, int r, int c, int channels) {
        const int last = (int)min((int64_t)kChunk, n - done) - 1;
        const T *chunk = from + (first + done) * stride;
#pragma unroll
        for (int x = 0; x < count; ++x) {
            const uint32_t row = min(count * r + x, last) * (uint32_t)stride;
            if constexpr (WIDE) to[x] = take<8, true>(chunk + (row + (8 * c < channels ? 8 * c : 0)), 0, 8);
            else to[x] = take<8, false>(chunk + row, 8 * c, channels);
        }
    };
    V8 keys_next[kPieces][kRows], queries_next[kPieces][kRows], keys_now[kPieces][kRows], values_next[2];
    f32x4 blocks_next[kBlocks / 2];
    float decay_next;
    // (four neighbouring lanes to a row: the memory pipeline takes four 16-byte loads of one line at a time)
    const int r = (tid >> 2) % kAcross, c0 = (tid & 3) + tid / (4 * kAcross) * 4, r_values = tid >> 2 & 31, c_values = (tid & 3) + (tid >> 7) * 4;
    auto fetch_rows = [&](int64_t done) {
#pragma unroll
        for (int m = 0; m < kPieces; ++m) {
            piece(keys_next[m], (const T *)a.k + (int64_t)hk * a.dk, a.k_stride, done, kRows, r, c0 + m * (kThreads / kAcross), a.dk);
            if (!SUMMARY) piece(queries_next[m], (const T *)a.q + (int64_t)hk * a.dk, a.q_stride, done, kRows, r, c0 + m * (kThreads / kAcross), a.dk);
        }
    };
    auto fetch_rest = [&](int64_t done) {
        const f32x4 *units = slot + done / kChunk * a.Hv * kUnits;
#pragma unroll
        for (int m = 0; m < kBlocks / 2; ++m) blocks_next[m] = units[m * kThreads + tid];
        decay_next = reinterpret_cast<const float *>(units + kUnitG)[tid % (2 * kChunk)];
        if (identity) values_next[0] = values_next[1] = V8((T)0.f);
        else piece(values_next, (const T *)a.v + (int64_t)h * a.dv + col0, a.v_stride, done, 2, r_values, c_values, a.dv - col0);
    };
    auto cut = [&](const V8 &x, int c) { return planes_of(WIDE && 8 * c >= a.dk ? V8((T)0.f) : x); };
    auto put_rows = [&](const V8 (&x)[kPieces][kRows], int of) {
#pragma unroll
        for (int m = 0; m < kPieces; ++m) {
            const int c = c0 + m * (kThreads / kAcross), unit = (c >> 2) * 4 + (c & 1) * 2, half = (c >> 1 & 1) * 8, swap = kRows * r >> 4;
            unsigned char *const to = lds + of * C::kQ + kRows * r * C::kRowBytes + half, *const low = to + (unit ^ swap) * 16, *const high = to + ((unit + 1) ^ swap) * 16;
#pragma unroll
            for (int y = 0; y < kRows; ++y) {
                const Planes<kIn> p = cut(x[m][y], c);
#pragma unroll
                for (int plane = 0; plane < kIn; ++plane) {
                    *reinterpret_cast<uint2 *>(low + plane * C::kPlane + y * C::kRowBytes) = make_uint2(p.p[plane][0], p.p[plane][1]);
                    *reinterpret_cast<uint2 *>(high + plane * C::kPlane + y * C::kRowBytes) = make_uint2(p.p[plane][2], p.p[plane][3]);
                }
            }
        }
    };
    auto put_transposed = [&](const V8 (&x)[kPieces][kRows]) {
#pragma unroll
        for (int m = 0; m < kPieces; ++m) {
            const int c = c0 + m * (kThreads / kAcross), four = kRows * r >> 2;          // (group of four rows)
            unsigned char *const to = lds + C::kT + 8 * c * 144 + ((four >> 3) * 4 + (four & 3)) * 16 + (four >> 2 & 1) * 8 + (kRows * r & 3) * 2;
            Planes<kIn> p[kRows];
#pragma unroll
            for (int y = 0; y < kRows; ++y) p[y] = cut(x[m][y], c);
#pragma unroll
            for (int plane = 0; plane < kIn; ++plane)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    uint32_t w[kRows / 2];
#pragma unroll
                    for (int y = 0; y < kRows; y += 2) w[y / 2] = __builtin_amdgcn_perm(p[y + 1].p[plane][e / 2], p[y].p[plane][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
                    unsigned char *const at = to + plane * C::kTransposed + e * 144;
                    if constexpr (kRows == 4) *reinterpret_cast<uint2 *>(at) = make_uint2(w[0], w[1]);
                    else *reinterpret_cast<uint32_t *>(at) = w[0];
                }
        }
    };
    auto put_rest = [&] {
#pragma unroll
        for (int m = 0; m < kBlocks / 2; ++m) {
            const int at = m * 4 + wave, of = at / kBlocks, block = at % kBlocks, row = row_of(block), c = block - block_of(row, 0);
            unsigned char *to = lds + C::kPairsAt + ((of * kPairs + pair_of(row, c >> 1)) * 3 * 64 + lane) * 16 + (c & 1) * 8;
            f32x4 x = blocks_next[m];
#pragma unroll
            for (int plane = 0; plane < 3; ++plane) {
                *reinterpret_cast<uint2 *>(to + plane * 1024) = make_uint2(upper(x[0], x[1]), upper(x[2], x[3]));
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = rest(x[e]);
            }
        }
        reinterpret_cast<float *>(lds + C::kDecays)[tid % (2 * kChunk)] = decay_next;
        typedef T Two __attribute__((ext_vector_type(2)));
        unsigned char *const to = lds + C::kV + c_values * 8 * C::kColumn + r_values * sizeof(Two);
#pragma unroll
        for (int e = 0; e < 8; ++e) *reinterpret_cast<Two *>(to + e * C::kColumn) = Two{values_next[0][e], values_next[1][e]};
    };
    auto rows = [&](int of, int m, int k) {              // K or Q, rows 16 m .., channels 32 k ..
        Planes<kIn> p;
#pragma unroll
        for (int plane = 0; plane < kIn; ++plane)
            p.p[plane] = *reinterpret_cast<const u32x4 *>(lds + of * C::kQ + plane * C::kPlane + (16 * m + i) * C::kRowBytes + k * 64 + (g ^ m) * 16);
        return p;
    };
    auto transposed = [&](int k, int m) {                // channels 16 k .., rows 32 m ..
        Planes<kIn> p;
#pragma unroll
        for (int plane = 0; plane < kIn; ++plane)
            p.p[plane] = *reinterpret_cast<const u32x4 *>(lds + C::kT + plane * C::kTransposed + (16 * k + i) * 144 + (m * 4 + g) * 16);
        return p;
    };
    auto pair = [&](int of, int m, int p) {              // T or P
        Planes<3> to;
#pragma unroll
        for (int plane = 0; plane < 3; ++plane) to.p[plane] = *reinterpret_cast<const u32x4 *>(lds + C::kPairsAt + (((of * kPairs + pair_of(m, p)) * 3 + plane) * 64 + lane) * 16);
        return to;
    };
    const float *decays = reinterpret_cast<const float *>(lds + C::kDecays);

    fetch_rows(0);
    fetch_rest(0);
    for (int at = tid; at < 2 * kPairs * 3 * 64; at += kThreads) reinterpret_cast<u32x4 *>(lds + C::kPairsAt)[at] = u32x4{0, 0, 0, 0};      // (pairs' blocks above the diagonal)
    f32x4 S[NK];
    begin_with<SUMMARY>(a, w, S);
    __syncthreads();
    auto keep = [&] {
#pragma unroll
        for (int m = 0; m < kPieces; ++m)
#pragma unroll
            for (int y = 0; y < kRows; ++y) keys_now[m][y] = keys_next[m][y];
    };
    put_rows(keys_next, 0);
    if (!SUMMARY) put_rows(queries_next, 1);
    put_rest();
    keep();
    fetch_rows(min((int64_t)kChunk, end));
    __syncthreads();
#pragma unroll 1
    for (int64_t done = 0; done < n; done += kChunk) {
        const int64_t next = min(done + kChunk, end);
        // K S and Q S; K^T of this chunk into LDS
        fetch_rest(next);
        put_transposed(keys_now);
        f32x4 kS[4], O[4], U[4], R[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) { kS[m] = O[m] = f32x4{0, 0, 0, 0}; }
#pragma unroll
        for (int k = 0; k < NK / 2; ++k) {
            const Planes<3> s = planes<3>(S[2 * k], S[2 * k + 1]);
            const Planes<kIn> keys[4] = {rows(0, 0, k), rows(0, 1, k), rows(0, 2, k), rows(0, 3, k)};
            add_planes(kS, keys, s);
            if constexpr (!SUMMARY) {
                const Planes<kIn> queries[4] = {rows(1, 0, k), rows(1, 1, k), rows(1, 2, k), rows(1, 3, k)};
                add_planes<true>(O, queries, s);
            }
        }
        __syncthreads();
        // U and O; K and Q of the next chunk into LDS
        put_rows(keys_next, 0);
        if (!SUMMARY) put_rows(queries_next, 1);
        keep();
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const V4 v = *reinterpret_cast<const V4 *>(lds + C::kV + (wave * 16 + i) * C::kColumn + (16 * m + 4 * g) * sizeof(T));
            const f32x4 eG = *reinterpret_cast<const f32x4 *>(decays + 16 * m + 4 * g);
#pragma unroll
            for (int c = 0; c < 4; ++c) R[m][c] = (float)v[c] - eG[c] * kS[m][c];
            O[m] *= decays[16 * m + i] * a.scale;
            U[m] = f32x4{0, 0, 0, 0};
        }
        auto below = [&](auto swapped, f32x4 (&acc)[4], int of, const f32x4 (&x)[4]) {         // acc += T x, or (P x)^T
            const Planes<3> left[4] = {pair(of, 0, 0), pair(of, 1, 0), pair(of, 2, 0), pair(of, 3, 0)};
            add_planes<decltype(swapped)::value>(acc, left, planes<3>(x[0], x[1]));
            const Planes<3> lower[2] = {pair(of, 2, 1), pair(of, 3, 1)};
            f32x4 two[2] = {acc[2], acc[3]};
            add_planes<decltype(swapped)::value>(two, lower, planes<3>(x[2], x[3]));
            acc[2] = two[0]; acc[3] = two[1];
        };
        below(std::false_type{}, U, 0, R);
        if constexpr (!SUMMARY) below(std::true_type{}, O, 1, U);
        const float last = decays[kChunk - 1];
#pragma unroll
        for (int m = 0; m < 4; ++m) U[m] *= *reinterpret_cast<const f32x4 *>(decays + kChunk + 16 * m + 4 * g);
        __syncthreads();
        // S; T, P and V of the next chunk into LDS, K and Q of the one after that on the way (behind the stores, which are waited for with them)
        put_rest();
        T *const o = (T *)a.o + ((first + done) * a.Hv + h) * a.dv;
        const int live = SUMMARY ? 0 : (int)min((int64_t)kChunk, n - done), from = col0 + wave * 16 + 4 * g;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            if (16 * m + i >= live) break;
            T *const to = o + ((16 * m + i) * (uint32_t)(a.Hv * a.dv) + from);
            if (WIDE) { if (from < a.dv) *reinterpret_cast<V4 *>(to) = __builtin_convertvector(O[m], V4); }
            else {
#pragma unroll
                for (int c = 0; c < 4; ++c) if (from + c < a.dv) to[c] = (T)O[m][c];
            }
        }
        fetch_rows(min(next + kChunk, end));
        const Planes<3> u[2] = {planes<3>(U[0], U[1]), planes<3>(U[2], U[3])};
#pragma unroll
        for (int k = 0; k < NK; k += 2) {
            f32x4 two[2] = {S[k] * last, S[k + 1] * last};
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const Planes<kIn> left[2] = {transposed(k, m), transposed(k + 1, m)};
                add_planes(two, left, u[m]);
            }
            S[k] = two[0]; S[k + 1] = two[1];
        }
        __syncthreads();
    }
    end_with<SUMMARY>(a, w, groups, S);
}

// The state in front of each segment but the first: X_1 = N_0, X_(s+1) = N_s + M_s X_s, with float32 instructions.  A workgroup to 16
// columns, a wavefront to NK / 4 tiles of 16 rows; X goes round through LDS as the accumulators hold it, which is how the products
// take it: lane (i, g) has rows 4 g .. + 3 of column i.  Each piece of the next M is asked for as soon as this one's is used.
template <int NK>
__global__ void __launch_bounds__(kThreads) delta_join_kernel(DeltaArgs a, int columns) {
    constexpr int kTiles = NK / 4;
    __shared__ f32x4 s_X[2][NK * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int64_t bh = blockIdx.x / columns;
    const int col = (int)(blockIdx.x % columns) * 16 + i;
    int64_t first, n;
    rows_of(a, bh / a.Hv, first, n);
    const int64_t chunks = (n + kChunk - 1) / kChunk, each = max((chunks + a.segments - 1) / a.segments, (int64_t)1);
    const int last = (int)((chunks + each - 1) / each) - 1;            // (its state in front is the last one)
    f32x4 M[kTiles][NK], N[kTiles];
    auto left = [&](int segment, int t, int k) {
        const float *row = a.ends + ((bh * a.segments + segment) * a.dk + min(16 * (wave * kTiles + t) + i, a.dk - 1)) * a.across + a.values;
        return *reinterpret_cast<const f32x4 *>(row + 16 * k + 4 * g);
    };
    auto added = [&](int segment, int t) {
        f32x4 to;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int row = 16 * (wave * kTiles + t) + 4 * g + v;
            to[v] = row < a.dk ? a.ends[((bh * a.segments + segment) * a.dk + row) * a.across + col] : 0.f;
        }
        return to;
    };
    if (last < 1) return;
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
        N[t] = added(0, t);
        if (last > 1) {
#pragma unroll
            for (int k = 0; k < NK; ++k) M[t][k] = left(1, t, k);
        }
    }
    for (int segment = 0; segment < last; ++segment) {
        const int next = min(segment + 1, last - 1);
        const f32x4 *X = s_X[segment & 1];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            f32x4 sum[2] = {N[t], f32x4{0, 0, 0, 0}};
            N[t] = added(next, t);
            if (segment) {
#pragma unroll
                for (int k = 0; k < NK; ++k) {
                    const f32x4 x = X[k * 64 + lane], m = M[t][k];
#pragma unroll
                    for (int v = 0; v < 4; ++v) sum[k & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(m[v], x[v], sum[k & 1], 0, 0, 0);
                    M[t][k] = left(next, t, k);
                }
            }
            sum[0] += sum[1];
            const int row = 16 * (wave * kTiles + t) + 4 * g;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                if (row + v >= a.dk) sum[0][v] = 0.f;          // (its row of M is the last one's)
                else if (col < a.dv) a.fronts[((bh * a.segments + segment + 1) * a.dk + row + v) * a.dv + col] = sum[0][v];
            }
            s_X[~segment & 1][(wave * kTiles + t) * 64 + lane] = sum[0];
        }
        __syncthreads();
    }
}

// The same with float32 operands and instructions, where K, Q and K^T in planes are more than LDS holds.  The instructions bound it
// (some 6 of the 11 us of a chunk at 128 channels: 2048 rows, 32 heads of 128 x 128, float32, in three segments 92 + 10 + 138 us).
template <typename T, int NK, bool WIDE, bool SUMMARY>
__global__ void __launch_bounds__(kThreads) delta_chunks_f32_kernel(DeltaArgs a, const f32x4 *slots, int groups) {
    constexpr int kRow = NK * 16 + 4, E = 16 / sizeof(T), kAcross = NK * 16 / E, kPieces = kChunk * kAcross / kThreads;          // (pieces of 16 bytes)
    extern __shared__ __align__(16) unsigned char smem[];
    float *ks = reinterpret_cast<float *>(smem), *qs = ks + kChunk * kRow;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    Work w;
    if (!work_of<SUMMARY>(a, slots, groups, w)) return;
    const int h = w.h, hk = w.hk, col = w.col;
    const bool in = w.in;
    const int64_t first = w.first, n = w.n;
    const f32x4 *slot = w.slot;
    f32x4 S[NK];
    begin_with<SUMMARY>(a, w, S);
    // Keys, queries and values of the next chunk are on the way during this one, T during the products with S, P as T is used.  (rows behind the
    // last: the last again, as above)
    typename Some<T, E>::type keys[kPieces], queries[kPieces];
    T values[4][4];
    auto fetch = [&](int64_t done) {
        const int end = (int)min((int64_t)kChunk, n - done) - 1;
#pragma unroll
        for (int m = 0; m < kPieces; ++m) {
            const int at = m * kThreads + threadIdx.x;
            const int64_t row = first + done + min(at / kAcross, end);
            keys[m] = take<E, WIDE>((const T *)a.k + row * a.k_stride + (int64_t)hk * a.dk, at % kAcross * E, a.dk);
            if (!SUMMARY) queries[m] = take<E, WIDE>((const T *)a.q + row * a.q_stride + (int64_t)hk * a.dk, at % kAcross * E, a.dk);
        }
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int v = 0; v < 4; ++v) values[m][v] = w.identity ? (T)0.f : ((const T *)a.v)[(first + done + min(16 * m + 4 * g + v, end)) * a.v_stride + (int64_t)h * a.dv + (in ? col : 0)];
    };
    fetch(0);
    const int64_t end = (n - 1) / kChunk * kChunk;
    for (int64_t done = 0; done < n; done += kChunk, slot += (int64_t)a.Hv * kUnits) {
        const float *decays = reinterpret_cast<const float *>(slot + kUnitG);
        const int live = (int)min((int64_t)kChunk, n - done);
        f32x4 R[4], eG[4], eL[4], blocks[kBlocks];
        __syncthreads();
#pragma unroll
        for (int m = 0; m < kPieces; ++m) {
            const int at = m * kThreads + threadIdx.x;
            float *to = ks + at / kAcross * kRow + at % kAcross * E, *other = qs + at / kAcross * kRow + at % kAcross * E;
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                *reinterpret_cast<f32x4 *>(to + e) = f32x4{(float)keys[m][e], (float)keys[m][e + 1], (float)keys[m][e + 2], (float)keys[m][e + 3]};
                if (!SUMMARY) *reinterpret_cast<f32x4 *>(other + e) = f32x4{(float)queries[m][e], (float)queries[m][e + 1], (float)queries[m][e + 2], (float)queries[m][e + 3]};
            }
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
#pragma unroll
            for (int v = 0; v < 4; ++v) R[m][v] = (float)values[m][v];
            eG[m] = *reinterpret_cast<const f32x4 *>(decays + 16 * m + 4 * g);
            eL[m] = *reinterpret_cast<const f32x4 *>(decays + kChunk + 16 * m + 4 * g);
        }
#pragma unroll
        for (int at = 0; at < kBlocks; ++at) blocks[at] = slot[at * 64 + lane];
        const float last = decays[kChunk - 1];
        __syncthreads();
        fetch(min(done + kChunk, end));
        f32x4 kS[4], O[4], U[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) { kS[m] = O[m] = U[m] = f32x4{0, 0, 0, 0}; }
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                add_product(kS[m], *reinterpret_cast<const f32x4 *>(ks + (16 * m + i) * kRow + 16 * k + 4 * g), S[k]);
                if (!SUMMARY) add_product(O[m], *reinterpret_cast<const f32x4 *>(qs + (16 * m + i) * kRow + 16 * k + 4 * g), S[k]);
            }
#pragma unroll
        for (int m = 0; m < 4; ++m) { R[m] -= eG[m] * kS[m]; O[m] *= eG[m] * a.scale; }
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int c = 0; c <= m; ++c) {
                f32x4 &block = blocks[block_of(m, c)];
                add_product(U[m], block, R[c]);
                if (!SUMMARY) block = slot[kUnitP + block_of(m, c) * 64 + lane];
            }
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int c = 0; c <= m; ++c) if (!SUMMARY) add_product(O[m], blocks[block_of(m, c)], U[c]);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int row = 16 * m + 4 * g + v;
                if (!SUMMARY && in && row < live) ((T *)a.o)[((first + done + row) * a.Hv + h) * a.dv + col] = (T)O[m][v];
            }
            U[m] *= eL[m];
        }
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            S[k] *= last;
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    S[k] = __builtin_amdgcn_mfma_f32_16x16x4f32(ks[(16 * m + 4 * g + v) * kRow + 16 * k + i], U[m][v], S[k], 0, 0, 0);
        }
    }
    end_with<SUMMARY>(a, w, groups, S);
}

// Chunks from this many rows a sequence on.  (32 heads of 128 x 128, bfloat16, 16 sequences of 32 rows: 86 us in chunks, 72 in steps; of
// 48: 93 and 95; of 64: 101 and 125.  64 sequences: 310 and 227, 366 and 325, 451 and 429; one: 24 and 28, 25 and 39, 26 and 51.)
// It is the average that counts, as the host does not know the lengths: a long sequence among many short ones, fewer rows than this on
// average, goes step by step too (2000 rows among 63 single ones: 1490 us, where alone they take 152 in chunks).
constexpr int kManyRows = 48;
bool in_chunks(int64_t T, int64_t B) { return T >= kManyRows * B; }

// How the chunks are gone through; the same for a call's workspace and its launches.
struct DeltaPlan {
    bool chunks;
    int tiles, groups, across, segments;             // tiles of 16 key channels, groups of 64 value channels
    size_t slot_bytes, end_bytes, front_bytes;
    DeltaPlan(int64_t T, int64_t B, int64_t Hv, int64_t dk, int64_t dv) {
        chunks = in_chunks(T, B);
        tiles = dk <= 64 ? 4 : dk <= 128 ? 8 : 16;
        groups = (int)ceil_div(dv, 64);
        across = 64 * groups + 16 * tiles;
        // As many segments as leave a compute unit to every workgroup and four chunks to a segment; of two nothing would be gained.
        // One sequence of 1024 rows, 40 heads of 64 x 64, float32: 88 us in one piece, 28 (N and M) + 6 (joined) + 29 (outputs) in
        // four; of 2048 rows, 32 heads of 128 x 128, bfloat16: 148 in one, 56 + 10 + 64 in three (float16: 209, 69 + 10 + 87).
        const int64_t each = B * Hv, all = across / 64;
        int64_t s = T / B / (4 * kChunk);
        while (s > 2 && (each * (groups + (s - 2) * all) > 256 || each * groups * s > 256)) --s;
        segments = (int)(s > 2 ? s < 16 ? s : 16 : 1);
        slot_bytes = (size_t)((T / kChunk + B) * Hv) * kUnits * 16;
        end_bytes = segments > 1 ? (size_t)(each * segments * dk * across) * 4 : 0;
        front_bytes = segments > 1 ? (size_t)(each * segments * dk * dv) * 4 : 0;
    }
    size_t bytes() const { return chunks ? slot_bytes + end_bytes + front_bytes : 0; }
};

template <typename F> int by_channels(int dk, F &&fn) {
    return dk <= 32 ? fn(std::integral_constant<int, 2>{}) : dk <= 64 ? fn(std::integral_constant<int, 4>{}) : dk <= 128 ? fn(std::integral_constant<int, 8>{}) : fn(std::integral_constant<int, 16>{});
}

template <typename T, bool WIDE>
int launch(hipStream_t st, const DeltaArgs &a, const DeltaPlan &pl, f32x4 *slots) {
    if (!pl.chunks) {
        const int tiles = (int)ceil_div(a.dv, 16);
        return by_channels(a.dk, [&](auto nr) {
            hipLaunchKernelGGL((delta_steps_kernel<T, decltype(nr)::value, WIDE>), dim3((unsigned)ceil_div(a.B * a.Hv * tiles, 4)), dim3(256), 0, st, a, tiles);
            RWKV_CHECK_LAUNCH("delta_steps_kernel");
            return (int)RWKV_OK;
        });
    }
    hipLaunchKernelGGL((delta_within_kernel<T, WIDE>), dim3((unsigned)(a.T / kChunk + a.B), (unsigned)a.Hv), dim3(256), 0, st, a, slots);
    RWKV_CHECK_LAUNCH("delta_within_kernel");
    return by_channels(a.dk, [&](auto nk) {
        constexpr int NK = decltype(nk)::value < 4 ? 4 : decltype(nk)::value;
        auto go = [&](auto summary) {
            constexpr bool SUMMARY = decltype(summary)::value, PLANES = Chunks<T, NK>::kBytes <= 160 * 1024;
            constexpr size_t bytes = PLANES ? Chunks<T, NK>::kBytes : 2 * kChunk * (NK * 16 + 4) * 4;
            const dim3 grid((unsigned)(a.B * a.Hv * a.segments * (SUMMARY ? a.across / 64 : pl.groups)));
            if constexpr (PLANES) {
                if (const int rc = allow_lds<&delta_chunks_kernel<T, NK, WIDE, SUMMARY>>(bytes)) return rc;
                hipLaunchKernelGGL((delta_chunks_kernel<T, NK, WIDE, SUMMARY>), grid, dim3(kThreads), bytes, st, a, slots, pl.groups);
            } else {
                if (const int rc = allow_lds<&delta_chunks_f32_kernel<T, NK, WIDE, SUMMARY>>(bytes)) return rc;
                hipLaunchKernelGGL((delta_chunks_f32_kernel<T, NK, WIDE, SUMMARY>), grid, dim3(kThreads), bytes, st, a, slots, pl.groups);
            }
            RWKV_CHECK_LAUNCH("delta_chunks_kernel");
            return (int)RWKV_OK;
        };
        if (a.segments > 1) {
            if (const int rc = go(std::true_type{})) return rc;
            const int columns = (int)ceil_div(a.dv, 16);
            hipLaunchKernelGGL(delta_join_kernel<NK>, dim3((unsigned)(a.B * a.Hv * columns)), dim3(kThreads), 0, st, a, columns);
            RWKV_CHECK_LAUNCH("delta_join_kernel");
        }
        return go(std::false_type{});
    });
}

}  // namespace

}  // namespace rwkv

using namespace rwkv;

extern "C" {

size_t rwkv_delta_rule_workspace_bytes(int64_t T, int64_t B, int64_t Hk, int64_t Hv, int64_t dk, int64_t dv) {
    if (T <= 0 || B <= 0 || Hk <= 0 || Hv <= 0 || dk <= 0 || dv <= 0) return 0;
    return DeltaPlan(T, B, Hv, dk, dv).bytes();
}

int rwkv_delta_rule(rwkv_stream_t stream, int64_t T, int64_t B, int64_t Hk, int64_t Hv, int64_t dk, int64_t dv, int type, const void *q,
                    int64_t q_stride, const void *k, int64_t k_stride, const void *v, int64_t v_stride, const float *g, const float *beta,
                    float scale, const int32_t *starts, float *state, void *o, void *workspace, size_t workspace_bytes) {
    RWKV_CHECK_ARG(q && k && v && g && beta && state && o, "rwkv_delta_rule: null pointer");
    RWKV_CHECK_ARG(T > 0 && B > 0 && Hk > 0 && Hv > 0 && dk > 0 && dv > 0, "rwkv_delta_rule: sizes must be positive");
    RWKV_CHECK_ARG(Hv % Hk == 0, "rwkv_delta_rule: value heads must be a multiple of key heads");
    RWKV_CHECK_ARG(starts || T % B == 0, "rwkv_delta_rule: rows must be a multiple of the sequences where there are no starts");
    RWKV_CHECK_ARG(type == RWKV_F32 || type == RWKV_BF16 || type == RWKV_F16, "rwkv_delta_rule: rows are float32, bfloat16 or float16");
    RWKV_CHECK_ARG(q_stride >= 0 && k_stride >= 0 && v_stride >= 0, "rwkv_delta_rule: negative row stride");
    if (dk > 256 || dv > 65536 || Hv > 65535 || T >= (1ll << 31) || B * Hv * ceil_div(dv, 16) >= (1ll << 27) || (T / 64 + B) * Hv >= (1ll << 30))
        return set_error(RWKV_ERR_SIZE, "rwkv_delta_rule: keys of at most 256 channels");
    const int64_t e = (int64_t)type_bytes(type);
    const int64_t o_bytes = T * Hv * dv * e, state_bytes = B * Hv * dk * dv * 4;
    auto apart = [&](const void *from, int64_t bytes) { return !rows_share(1, o, 0, o_bytes, from, 0, bytes) && !rows_share(1, state, 0, state_bytes, from, 0, bytes); };
    RWKV_CHECK_ARG(apart(q, ((T - 1) * q_stride + Hk * dk) * e) && apart(k, ((T - 1) * k_stride + Hk * dk) * e) && apart(v, ((T - 1) * v_stride + Hv * dv) * e) &&
                       apart(g, T * Hv * 4) && apart(beta, T * Hv * 4) && (!starts || apart(starts, (B + 1) * 4)) && !rows_share(1, o, 0, o_bytes, state, 0, state_bytes),
                   "rwkv_delta_rule: o or state shares memory with another argument");
    const DeltaPlan pl(T, B, Hv, dk, dv);
    if (pl.chunks ? !launchable(T / kChunk + B, 256) || !launchable(B * Hv * pl.segments * ceil_div(pl.across, 64), kThreads) : !launchable(ceil_div(B * Hv * ceil_div(dv, 16), 4), 256))
        return set_error(RWKV_ERR_SIZE, "rwkv_delta_rule: too many sequences and heads");
    if (pl.chunks) {
        if (q_stride >= (1 << 24) || k_stride >= (1 << 24) || v_stride >= (1 << 24) || Hv * dv >= (1 << 24))
            return set_error(RWKV_ERR_SIZE, "rwkv_delta_rule: rows of 2^24 elements or more");
        RWKV_CHECK_ALIGN(workspace, 16);
        if (!workspace || workspace_bytes < pl.bytes())
            return set_error(RWKV_ERR_WORKSPACE, "rwkv_delta_rule: workspace too small");
    }
    const DeltaArgs a{T, B, T / B, (int)(Hv / Hk), (int)Hv, (int)dk, (int)dv, q, k, v, q_stride, k_stride, v_stride, g, beta, scale, starts, state, o,
                      pl.segments, (float *)((uint8_t *)workspace + pl.slot_bytes), (float *)((uint8_t *)workspace + pl.slot_bytes + pl.end_bytes), 64 * pl.groups, pl.across};
    const size_t size = type_bytes(type);
    auto fits = [&](const void *at, int64_t stride, int64_t channels) { return ((uintptr_t)at | (uintptr_t)(stride * size) | (uintptr_t)(channels * size)) % 16 == 0; };
    // (heads of whole 16 bytes, which are also what a lane of delta_steps_kernel takes at a time, or multiples of it)
    const bool wide = fits(q, q_stride, dk) && fits(k, k_stride, dk) && fits(v, v_stride, dv) && (uintptr_t)state % 16 == 0 && (uintptr_t)o % 16 == 0 && dk % 16 == 0 && dv % 8 == 0;
    return with_low(type, [&](auto ty) {
        using E = typename decltype(ty)::type;
        return wide ? launch<E, true>((hipStream_t)stream, a, pl, (f32x4 *)workspace) : launch<E, false>((hipStream_t)stream, a, pl, (f32x4 *)workspace);
    });
}

}  // extern "C"
