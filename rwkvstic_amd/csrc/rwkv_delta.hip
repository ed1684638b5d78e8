// The gated delta rule over packed sequences (rwkv_delta_rule), per value head with a state S [dk, dv]:
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = scale S^T q.
#include "rwkv_types.h"

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

// Step by step, a wavefront to 16 columns of the state: lane (c, r) = (lane / 16, lane % 16) holds rows r + 16 i, i < NR, of
// columns 4 c .. 4 c + 3, so that the sums over a column's rows stay in a DPP row and no wavefront waits for another.  Both
// products are taken with the state before the step, so that their sums are made side by side:
//   S'^T q = e^g S^T q + (k.q) u.
template <typename T, int NR>
__global__ void __launch_bounds__(256) delta_steps_kernel(DeltaArgs a, int tiles) {
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
    float *state = a.state + (b * a.Hv + h) * a.dk * a.dv;
    float S[NR][4];
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) S[i][c] = r + 16 * i < a.dk && col + c < a.dv ? state[(int64_t)(r + 16 * i) * a.dv + col + c] : 0.f;
    for (int64_t t = 0; t < n; ++t) {
        float kk[NR], kq = 0.f, kS[4] = {0.f, 0.f, 0.f, 0.f}, qS[4] = {0.f, 0.f, 0.f, 0.f};
        const float e = expf(g[t * a.Hv]), be = beta[t * a.Hv];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const bool in = r + 16 * i < a.dk;
            kk[i] = in ? (float)k[t * a.k_stride + r + 16 * i] : 0.f;
            const float qq = in ? (float)q[t * a.q_stride + r + 16 * i] : 0.f;
            kq = fmaf(kk[i], qq, kq);
#pragma unroll
            for (int c = 0; c < 4; ++c) { kS[c] = fmaf(kk[i], S[i][c], kS[c]); qS[c] = fmaf(qq, S[i][c], qS[c]); }
        }
        kq = row_sum(kq);
        float out = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float x = col + c < a.dv ? (float)v[t * a.v_stride + col + c] : 0.f;
            const float u = be * (x - e * row_sum(kS[c]));
            const float y = a.scale * (e * row_sum(qS[c]) + kq * u);
            out = r == c ? y : out;
#pragma unroll
            for (int i = 0; i < NR; ++i) S[i][c] = fmaf(e, S[i][c], kk[i] * u);
        }
        if (r < 4 && col + r < a.dv) o[t * a.Hv * a.dv + col + r] = (T)out;
    }
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (r + 16 * i < a.dk && col + c < a.dv) state[(int64_t)(r + 16 * i) * a.dv + col + c] = S[i][c];
}

template <typename T>
void launch_steps(hipStream_t st, const DeltaArgs &a) {
    const int tiles = (int)ceil_div(a.dv, 16);
    const dim3 grid((unsigned)ceil_div(a.B * a.Hv * tiles, 4));
    if (a.dk <= 32) hipLaunchKernelGGL((delta_steps_kernel<T, 2>), grid, dim3(256), 0, st, a, tiles);
    else if (a.dk <= 64) hipLaunchKernelGGL((delta_steps_kernel<T, 4>), grid, dim3(256), 0, st, a, tiles);
    else if (a.dk <= 128) hipLaunchKernelGGL((delta_steps_kernel<T, 8>), grid, dim3(256), 0, st, a, tiles);
    else hipLaunchKernelGGL((delta_steps_kernel<T, 16>), grid, dim3(256), 0, st, a, tiles);
}

}  // namespace

}  // namespace rwkv

using namespace rwkv;

extern "C" {

size_t rwkv_delta_rule_workspace_bytes(int64_t T, int64_t B, int64_t Hk, int64_t Hv, int64_t dk, int64_t dv) { return 0; }

int rwkv_delta_rule(rwkv_stream_t stream, int64_t T, int64_t B, int64_t Hk, int64_t Hv, int64_t dk, int64_t dv, int type, const void *q,
                    int64_t q_stride, const void *k, int64_t k_stride, const void *v, int64_t v_stride, const float *g, const float *beta,
                    float scale, const int32_t *starts, float *state, void *o, void *workspace, size_t workspace_bytes) {
    RWKV_CHECK_ARG(q && k && v && g && beta && state && o, "rwkv_delta_rule: null pointer");
    RWKV_CHECK_ARG(T > 0 && B > 0 && Hk > 0 && Hv > 0 && dk > 0 && dv > 0, "rwkv_delta_rule: sizes must be positive");
    RWKV_CHECK_ARG(Hv % Hk == 0, "rwkv_delta_rule: value heads must be a multiple of key heads");
    RWKV_CHECK_ARG(starts || T % B == 0, "rwkv_delta_rule: rows must be a multiple of the sequences where there are no starts");
    RWKV_CHECK_ARG(type == RWKV_F32 || type == RWKV_BF16 || type == RWKV_F16, "rwkv_delta_rule: rows are float32, bfloat16 or float16");
    RWKV_CHECK_ARG(q_stride >= 0 && k_stride >= 0 && v_stride >= 0, "rwkv_delta_rule: negative row stride");
    if (dk > 256 || dv > 65536 || Hv > 65536 || T >= (1ll << 31) || B * Hv * ceil_div(dv, 16) >= (1ll << 31))
        return set_error(RWKV_ERR_SIZE, "rwkv_delta_rule: keys of at most 256 channels");
    const DeltaArgs a{T, B, (int)Hk, (int)Hv, (int)dk, (int)dv, q, k, v, q_stride, k_stride, v_stride, g, beta, scale, starts, state, o};
    with_low(type, [&](auto ty) { launch_steps<typename decltype(ty)::type>((hipStream_t)stream, a); });
    RWKV_CHECK_LAUNCH("delta_steps_kernel");
    return RWKV_OK;
}

}  // extern "C"
