// The gated delta rule over packed sequences (rwkv_delta_rule), per value head with a state S [dk, dv]:
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = scale S^T q.
//
// Few rows a sequence: step by step (delta_steps_kernel), a wavefront to 16 columns of the state; the state is read and written once.
// Many: in chunks of 64 rows.  With G_i = g_1 + .. + g_i within the chunk and K, Q, V its rows,
//   U = T (V - e^G K S),  T = (1 + A)^-1 diag(beta),  A_ij = beta_i e^(G_i - G_j) k_i.k_j below the diagonal,
//   O = scale e^G Q S + P U,  P_ij = scale e^(G_i - G_j) q_i.k_j up to the diagonal,  S <- e^G_64 S + K^T (e^(G_64 - G) U).
//   delta_within_kernel   T and P of every chunk, all at once
//   delta_chunks_kernel   chunk after chunk, a wavefront to 16 columns of the state
// Both on the matrix cores with float32 sums; G and its differences are float64, as a decay is the exponential of a difference of sums.
#include "rwkv_types.h"

#include <type_traits>

namespace rwkv {

namespace {

struct DeltaArgs {
    int64_t T, B;
    int Hk, Hv, dk, dv;
    const void *q, *k, *v; int64_t q_stride, k_stride, v_stride;
    const float *g, *beta;
    float scale;
    const int32_t *starts;
    float *state;
    void *o;
};

// First row and number of rows of sequence b, cut to the rows there are.
__device__ __forceinline__ void rows_of(const DeltaArgs &a, int64_t b, int64_t &first, int64_t &n) {
    if (!a.starts) { n = a.T / a.B; first = b * n; return; }
    const int64_t lo = a.starts[b], hi = a.starts[b + 1];
    first = min(max(lo, (int64_t)0), a.T);
    n = max(min(hi, a.T) - first, (int64_t)0);
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

// N neighbouring elements of a row of n from k on; WIDE: aligned to their size, up to 16 bytes, and n a multiple of N.
template <int N, bool WIDE, typename T>
__device__ __forceinline__ void take(T (&to)[N], const T *row, int k, int n) {
    if constexpr (WIDE) {
        constexpr int E = N * sizeof(T) < 16 ? N : 16 / sizeof(T);
        typedef T Some __attribute__((ext_vector_type(E)));
        Some v[N / E];
#pragma unroll
        for (int i = 0; i < N / E; ++i) v[i] = k < n ? *reinterpret_cast<const Some *>(row + k + i * E) : Some((T)0.f);
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = v[i / E][i % E];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = k + i < n ? row[k + i] : (T)0.f;
    }
}

// Lane (c, r) = (lane / 16, lane % 16) holds rows NR r .. NR r + NR - 1 of columns 4 c .. 4 c + 3, so that the sums over a
// column's rows stay in a DPP row and no wavefront waits for another.  Both products are taken with the state before the step, so
// that their sums are made side by side: S'^T q = e^g S^T q + (k.q) u.  The next row is under way meanwhile.
template <typename T, int NR, bool WIDE>
__global__ void __launch_bounds__(256) delta_steps_kernel(DeltaArgs a, int tiles) {
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    const int64_t job = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (job >= a.B * a.Hv * tiles) return;
    const int lane = threadIdx.x & 63, r = lane & 15, col = (int)(job % tiles) * 16 + (lane >> 4) * 4;
    const int h = (int)(job / tiles % a.Hv), hk = h / (a.Hv / a.Hk);
    const int64_t b = job / tiles / a.Hv;
    int64_t first, n;
    rows_of(a, b, first, n);
    if (n <= 0) return;
    const T *q = (const T *)a.q + first * a.q_stride + (int64_t)hk * a.dk, *k = (const T *)a.k + first * a.k_stride + (int64_t)hk * a.dk;
    const T *v = (const T *)a.v + first * a.v_stride + (int64_t)h * a.dv;
    T *o = (T *)a.o + (first * a.Hv + h) * a.dv;
    const float *g = a.g + first * a.Hv + h, *beta = a.beta + first * a.Hv + h;
    float *state = a.state + (b * a.Hv + h) * a.dk * a.dv + (int64_t)r * NR * a.dv + col;
    struct Row { T k[NR], q[NR], v[4]; float g, beta; };
    auto load = [&](Row &to, int64_t t) {
        take<NR, WIDE>(to.k, k + t * a.k_stride, r * NR, a.dk);
        take<NR, WIDE>(to.q, q + t * a.q_stride, r * NR, a.dk);
        take<4, WIDE>(to.v, v + t * a.v_stride, col, a.dv);
        to.g = g[t * a.Hv]; to.beta = beta[t * a.Hv];
    };
    Row next;
    load(next, 0);
    f32x4 S[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        S[i] = f32x4{0, 0, 0, 0};
        if (r * NR + i >= a.dk) continue;
        if (WIDE) { if (col < a.dv) S[i] = *reinterpret_cast<const f32x4 *>(state + (int64_t)i * a.dv); }
        else {
#pragma unroll
            for (int c = 0; c < 4; ++c) if (col + c < a.dv) S[i][c] = state[(int64_t)i * a.dv + c];
        }
    }
#pragma unroll 1
    for (int64_t t = 0; t < n; ++t) {
        const Row now = next;
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
        float out = 0.f, u[4];
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
        if (r < 4 && col + r < a.dv) o[t * a.Hv * a.dv + col + r] = (T)out;
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        if (r * NR + i >= a.dk) continue;
        if (WIDE) { if (col < a.dv) *reinterpret_cast<f32x4 *>(state + (int64_t)i * a.dv) = S[i]; }
        else {
#pragma unroll
            for (int c = 0; c < 4; ++c) if (col + c < a.dv) state[(int64_t)i * a.dv + c] = S[i][c];
        }
    }
}

// ---- chunks -----------------------------------------------------------------------------------------------------------
constexpr int kChunk = 64;
constexpr int kBlocks = 10;                          // 16 x 16 blocks up to the diagonal
constexpr int kSlot = 2 * kBlocks * 256 + 2 * kChunk;        // floats of a chunk and head: T, P, e^G, e^(G_64 - G)
constexpr float kForgotten = -1e5f;                  // a decay's logarithm below which nothing is left; -infinity would have no differences

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Lane (j, g) = (lane % 16, lane / 16) holds rows 4 g + v, v < 4, of column j of a 16 x 16 product.  As a right operand it is to
// hold one term k of column j at a time; the order of the terms being free, what a product leaves in the registers is the next
// one's right operand, term 4 g + v in the v-th of four instructions, if lane (i, g) has terms 4 g .. 4 g + 3 of row i of the left one.
__device__ __forceinline__ void add_product(f32x4 &acc, const f32x4 &left, const f32x4 &right) {
#pragma unroll
    for (int v = 0; v < 4; ++v) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(left[v], right[v], acc, 0, 0, 0);
}

// Chunks of sequence b have the places first / 64 + b and on: no two the same, none past T / 64 + B.
__device__ __forceinline__ int64_t place_of(int64_t first, int64_t b) { return first / kChunk + b; }

__device__ __forceinline__ int block_of(int row, int column) { return row * (row + 1) / 2 + column; }

// 64 rows (zeros behind the n-th) of dk channels into LDS, as To, rows `stride` apart; WIDE: 16-byte aligned rows that fill whole 16 bytes.
template <bool WIDE, typename To, typename T>
__device__ __forceinline__ void stage(To *lds, int stride, int filled, const T *from, int64_t from_stride, int n, int dk) {
    constexpr int E = WIDE ? 16 / sizeof(T) : 1;
    const int per = filled / E;
    for (int at = threadIdx.x; at < kChunk * per; at += blockDim.x) {
        const int row = at / per, k = at % per * E;
        T v[E];
        take<E, WIDE>(v, from + row * from_stride, k, row < n ? dk : 0);
#pragma unroll
        for (int e = 0; e < E; ++e) lds[row * stride + k + e] = (To)v[e];
    }
}

// Products of rows of keys and queries: the operands' own type where the matrix cores have it (the products are exact), else float32.
template <typename T> struct Dot;
template <> struct Dot<float> {
    static constexpr int kPad = 4;
    static __device__ __forceinline__ f32x4 of(const float *left, const float *right, int n, int g) {
        f32x4 acc = {0, 0, 0, 0};
        for (int k = 4 * g; k < n; k += 16) add_product(acc, *reinterpret_cast<const f32x4 *>(left + k), *reinterpret_cast<const f32x4 *>(right + k));
        return acc;
    }
};
template <> struct Dot<__bf16> {
    static constexpr int kPad = 8;
    typedef __bf16 Eight __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 of(const __bf16 *left, const __bf16 *right, int n, int g) {
        f32x4 acc = {0, 0, 0, 0};
        for (int k = 8 * g; k < n; k += 32)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const Eight *>(left + k), *reinterpret_cast<const Eight *>(right + k), acc, 0, 0, 0);
        return acc;
    }
};
template <> struct Dot<_Float16> {
    static constexpr int kPad = 8;
    typedef _Float16 Eight __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x4 of(const _Float16 *left, const _Float16 *right, int n, int g) {
        f32x4 acc = {0, 0, 0, 0};
        for (int k = 8 * g; k < n; k += 32)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const Eight *>(left + k), *reinterpret_cast<const Eight *>(right + k), acc, 0, 0, 0);
        return acc;
    }
};

// T and P of one chunk and value head, block by block as lane (i, g) of delta_chunks_kernel wants them: row i, terms 4 g .. 4 g + 3.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) delta_within_kernel(DeltaArgs a, float *slots, int filled) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ double s_G[kChunk];
    __shared__ float s_beta[kChunk];
    __shared__ __align__(16) float s_A[kChunk][kChunk + 4], s_X[4][16][20];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 15, g = lane >> 4;
    const int h = blockIdx.y, hk = h / (a.Hv / a.Hk);
    // the last sequence whose places begin here or before
    const int64_t place = blockIdx.x;
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
    const int live = (int)min((int64_t)kChunk, n - done), stride = filled + Dot<T>::kPad;
    T *ks = reinterpret_cast<T *>(smem), *qs = ks + kChunk * stride;
    stage<WIDE>(ks, stride, filled, (const T *)a.k + first * a.k_stride + (int64_t)hk * a.dk, a.k_stride, live, a.dk);
    stage<WIDE>(qs, stride, filled, (const T *)a.q + first * a.q_stride + (int64_t)hk * a.dk, a.q_stride, live, a.dk);
    float *slot = slots + (place * a.Hv + h) * kSlot;
    if (wave == 0) {
        float decay = lane < live ? a.g[(first + lane) * a.Hv + h] : 0.f;
        if (decay < kForgotten) decay = kForgotten;
        double G = decay;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) { const double before = __shfl_up(G, off, 64); if (lane >= off) G += before; }
        s_G[lane] = G;
        s_beta[lane] = lane < live ? a.beta[(first + lane) * a.Hv + h] : 0.f;
        slot[2 * kBlocks * 256 + lane] = expf((float)G);
        slot[2 * kBlocks * 256 + kChunk + lane] = expf((float)(__shfl(G, 63, 64) - G));
    }
    __syncthreads();
    // A into LDS, P out; transposed products, so that a lane has four neighbours of a row
    for (int block = wave; block < kBlocks; block += 4) {
        const int m = block < 1 ? 0 : block < 3 ? 1 : block < 6 ? 2 : 3, c = block - m * (m + 1) / 2;
        const T *columns = ks + (16 * c + i) * stride;
        const f32x4 kk = Dot<T>::of(columns, ks + (16 * m + i) * stride, filled, g), qk = Dot<T>::of(columns, qs + (16 * m + i) * stride, filled, g);
        const int row = 16 * m + i;
        f32x4 A, P;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const int column = 16 * c + 4 * g + v;
            const float decay = expf((float)(s_G[row] - s_G[column]));
            A[v] = column < row ? s_beta[row] * decay * kk[v] : 0.f;
            P[v] = column <= row ? a.scale * decay * qk[v] : 0.f;
        }
        *reinterpret_cast<f32x4 *>(&s_A[row][16 * c + 4 * g]) = A;
        *reinterpret_cast<f32x4 *>(slot + (kBlocks + block) * 256 + lane * 4) = P;
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
    // ... the others below them, a wavefront to a column of blocks: X_mc = -X_mm sum_l A_ml X_lc
    f32x4 X[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        if (m < wave) continue;
        if (m == wave) {
#pragma unroll
            for (int v = 0; v < 4; ++v) X[m][v] = s_X[m][4 * g + v][i];
        } else {
            f32x4 Y = {0, 0, 0, 0}, Z = {0, 0, 0, 0};
#pragma unroll
            for (int l = 0; l < m; ++l)
                if (l >= wave) add_product(Y, *reinterpret_cast<const f32x4 *>(&s_A[16 * m + i][16 * l + 4 * g]), X[l]);
            add_product(Z, *reinterpret_cast<const f32x4 *>(&s_X[m][i][4 * g]), Y);
            X[m] = -Z;
        }
        // lane (j, g) has rows 4 g + v of column j
        const float beta = s_beta[16 * wave + i];
#pragma unroll
        for (int v = 0; v < 4; ++v) slot[block_of(m, wave) * 256 + (4 * g + v + 16 * (i >> 2)) * 4 + (i & 3)] = X[m][v] * beta;
    }
}

// NK tiles of 16 key channels.  S, and what is multiplied with it and comes of it, stay in the wavefront's registers.
template <typename T, int NK, bool WIDE>
__global__ void __launch_bounds__(256) delta_chunks_kernel(DeltaArgs a, const float *slots, int groups) {
    constexpr int kRow = NK * 16 + 4;
    extern __shared__ __align__(16) unsigned char smem[];
    float *ks = reinterpret_cast<float *>(smem), *qs = ks + kChunk * kRow;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int h = (int)(blockIdx.x / groups % a.Hv), hk = h / (a.Hv / a.Hk);
    const int64_t b = blockIdx.x / groups / a.Hv;
    const int col = (int)(blockIdx.x % groups) * (int)(blockDim.x >> 2) + wave * 16 + i;
    const bool in = col < a.dv;
    int64_t first, n;
    rows_of(a, b, first, n);
    if (n <= 0) return;
    float *state = a.state + (b * a.Hv + h) * a.dk * a.dv + col;
    f32x4 S[NK];
#pragma unroll
    for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int v = 0; v < 4; ++v) { const int row = 16 * k + 4 * g + v; S[k][v] = in && row < a.dk ? state[(int64_t)row * a.dv] : 0.f; }
    const float *slot = slots + (place_of(first, b) * a.Hv + h) * kSlot;
    for (int64_t done = 0; done < n; done += kChunk, first += kChunk, slot += (int64_t)a.Hv * kSlot) {
        const int live = (int)min((int64_t)kChunk, n - done);
        f32x4 R[4], eG[4], eL[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int row = 16 * m + 4 * g + v;
                R[m][v] = in && row < live ? (float)((const T *)a.v)[(first + row) * a.v_stride + (int64_t)h * a.dv + col] : 0.f;
            }
            eG[m] = *reinterpret_cast<const f32x4 *>(slot + 2 * kBlocks * 256 + 16 * m + 4 * g);
            eL[m] = *reinterpret_cast<const f32x4 *>(slot + 2 * kBlocks * 256 + kChunk + 16 * m + 4 * g);
        }
        const float last = slot[2 * kBlocks * 256 + kChunk - 1];
        __syncthreads();
        stage<WIDE>(ks, kRow, NK * 16, (const T *)a.k + first * a.k_stride + (int64_t)hk * a.dk, a.k_stride, live, a.dk);
        stage<WIDE>(qs, kRow, NK * 16, (const T *)a.q + first * a.q_stride + (int64_t)hk * a.dk, a.q_stride, live, a.dk);
        __syncthreads();
        f32x4 kS[4], O[4], U[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) { kS[m] = O[m] = U[m] = f32x4{0, 0, 0, 0}; }
#pragma unroll
        for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                add_product(kS[m], *reinterpret_cast<const f32x4 *>(ks + (16 * m + i) * kRow + 16 * k + 4 * g), S[k]);
                add_product(O[m], *reinterpret_cast<const f32x4 *>(qs + (16 * m + i) * kRow + 16 * k + 4 * g), S[k]);
            }
#pragma unroll
        for (int m = 0; m < 4; ++m) { R[m] -= eG[m] * kS[m]; O[m] *= eG[m] * a.scale; }
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int c = 0; c <= m; ++c) add_product(U[m], *reinterpret_cast<const f32x4 *>(slot + block_of(m, c) * 256 + lane * 4), R[c]);
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int c = 0; c <= m; ++c) add_product(O[m], *reinterpret_cast<const f32x4 *>(slot + (kBlocks + block_of(m, c)) * 256 + lane * 4), U[c]);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int row = 16 * m + 4 * g + v;
                if (in && row < live) ((T *)a.o)[((first + row) * a.Hv + h) * a.dv + col] = (T)O[m][v];
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
#pragma unroll
    for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int v = 0; v < 4; ++v) { const int row = 16 * k + 4 * g + v; if (in && row < a.dk) state[(int64_t)row * a.dv] = S[k][v]; }
}

// Chunks from this many rows a sequence on.
constexpr int kManyRows = 48;
bool in_chunks(int64_t T, int64_t B) { return T >= kManyRows * B; }

template <typename F> int by_channels(int dk, F &&fn) {
    return dk <= 32 ? fn(std::integral_constant<int, 2>{}) : dk <= 64 ? fn(std::integral_constant<int, 4>{}) : dk <= 128 ? fn(std::integral_constant<int, 8>{}) : fn(std::integral_constant<int, 16>{});
}

template <typename T, bool WIDE>
int launch(hipStream_t st, const DeltaArgs &a, float *slots) {
    if (!in_chunks(a.T, a.B)) {
        const int tiles = (int)ceil_div(a.dv, 16);
        return by_channels(a.dk, [&](auto nr) {
            hipLaunchKernelGGL((delta_steps_kernel<T, decltype(nr)::value, WIDE>), dim3((unsigned)ceil_div(a.B * a.Hv * tiles, 4)), dim3(256), 0, st, a, tiles);
            RWKV_CHECK_LAUNCH("delta_steps_kernel");
            return (int)RWKV_OK;
        });
    }
    const int filled = (int)round_up(a.dk, 32);
    const size_t lds = (size_t)2 * kChunk * (filled + Dot<T>::kPad) * sizeof(T);
    if (const int rc = allow_lds<&delta_within_kernel<T, WIDE>>(lds)) return rc;
    hipLaunchKernelGGL((delta_within_kernel<T, WIDE>), dim3((unsigned)(a.T / kChunk + a.B), (unsigned)a.Hv), dim3(256), lds, st, a, slots, filled);
    RWKV_CHECK_LAUNCH("delta_within_kernel");
    return by_channels(a.dk, [&](auto nk) {
        constexpr int NK = decltype(nk)::value;
        constexpr size_t lds = (size_t)2 * kChunk * (NK * 16 + 4) * 4;
        if (const int rc = allow_lds<&delta_chunks_kernel<T, NK, WIDE>>(lds)) return rc;
        const int waves = a.dv <= 16 ? 1 : a.dv <= 32 ? 2 : 4, groups = (int)ceil_div(a.dv, 16 * waves);
        hipLaunchKernelGGL((delta_chunks_kernel<T, NK, WIDE>), dim3((unsigned)(a.B * a.Hv * groups)), dim3(64 * waves), lds, st, a, slots, groups);
        RWKV_CHECK_LAUNCH("delta_chunks_kernel");
        return (int)RWKV_OK;
    });
}

}  // namespace

}  // namespace rwkv

using namespace rwkv;

extern "C" {

size_t rwkv_delta_rule_workspace_bytes(int64_t T, int64_t B, int64_t Hk, int64_t Hv, int64_t dk, int64_t dv) {
    if (T <= 0 || B <= 0 || Hv <= 0 || !in_chunks(T, B)) return 0;
    return (size_t)((T / kChunk + B) * Hv) * kSlot * sizeof(float);
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
    if (dk > 256 || dv > 65536 || Hv > 65535 || T >= (1ll << 31) || B * Hv * ceil_div(dv, 16) >= (1ll << 31))
        return set_error(RWKV_ERR_SIZE, "rwkv_delta_rule: keys of at most 256 channels");
    if (in_chunks(T, B)) {
        RWKV_CHECK_ALIGN(workspace, 16);
        if (!workspace || workspace_bytes < rwkv_delta_rule_workspace_bytes(T, B, Hk, Hv, dk, dv))
            return set_error(RWKV_ERR_WORKSPACE, "rwkv_delta_rule: workspace too small");
    }
    const DeltaArgs a{T, B, (int)Hk, (int)Hv, (int)dk, (int)dv, q, k, v, q_stride, k_stride, v_stride, g, beta, scale, starts, state, o};
    const size_t size = type_bytes(type);
    auto fits = [&](const void *at, int64_t stride, int64_t channels) { return ((uintptr_t)at | (uintptr_t)(stride * size) | (uintptr_t)(channels * size)) % 16 == 0; };
    // (heads of whole 16 bytes, which are also what a lane of delta_steps_kernel takes at a time, or multiples of it)
    const bool wide = fits(q, q_stride, dk) && fits(k, k_stride, dk) && fits(v, v_stride, dv) && (uintptr_t)state % 16 == 0 && dk % 16 == 0 && dv % 4 == 0;
    return with_low(type, [&](auto ty) {
        using E = typename decltype(ty)::type;
        return wide ? launch<E, true>((hipStream_t)stream, a, (float *)workspace) : launch<E, false>((hipStream_t)stream, a, (float *)workspace);
    });
}

}  // extern "C"
