// Low-rank adapters of many requests beside a shared projection (rwkv_lora_rows):
//   h[t] = scale[i] (a[i] x[t]),  out[t] = base[t] + b[i] h[t],  i = adapter[t].
#include "rwkv_types.h"

namespace rwkv {

namespace {

struct LoraArgs {
    int64_t T, n_in, n_out, N, R;
    const void *x; int64_t x_stride;
    const void *a, *b;
    const int32_t *adapter;
    const float *scale;
    const void *base; int64_t base_stride;
    void *out; int64_t out_stride;
    void *h;                              // [T, R]
};

// A wavefront per row and rank.
template <typename Real, typename Low>
__global__ void __launch_bounds__(256) lora_down_kernel(LoraArgs p) {
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), t = at / p.R, r = at % p.R;
    if (t >= p.T) return;
    const int32_t i = p.adapter[t];
    if (i < 0 || i >= p.N) return;
    const Real *x = (const Real *)p.x + t * p.x_stride;
    const Low *a = (const Low *)p.a + (i * p.R + r) * p.n_in;
    Real s = 0;
    for (int64_t j = threadIdx.x & 63; j < p.n_in; j += 64) s += x[j] * (Real)a[j];
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) ((Real *)p.h)[at] = p.scale ? s * (Real)p.scale[i] : s;
}

// A thread per row and output.
template <typename Real, typename Low>
__global__ void __launch_bounds__(256) lora_up_kernel(LoraArgs p) {
    const int64_t blocks = ceil_div(p.n_out, 256), t = blockIdx.x / blocks, n = blockIdx.x % blocks * 256 + threadIdx.x;
    if (n >= p.n_out) return;
    const int32_t i = p.adapter[t];
    Real s = 0;
    if (i >= 0 && i < p.N) {
        const Real *h = (const Real *)p.h + t * p.R;
        const Low *b = (const Low *)p.b + (i * p.n_out + n) * p.R;
        for (int64_t r = 0; r < p.R; ++r) s += h[r] * (Real)b[r];
    }
    ((Real *)p.out)[t * p.out_stride + n] = p.base ? ((const Real *)p.base)[t * p.base_stride + n] + s : s;
}

}  // namespace

}  // namespace rwkv

using namespace rwkv;

extern "C" {

size_t rwkv_lora_rows_workspace_bytes(int64_t T, int64_t n_in, int64_t n_out, int64_t N, int64_t R, int real) {
    if (T <= 0 || n_in <= 0 || n_out <= 0 || N <= 0 || R <= 0) return 0;
    return (size_t)(T * R) * type_bytes(real);
}

int rwkv_lora_rows(rwkv_stream_t stream, int64_t T, int64_t n_in, int64_t n_out, int64_t N, int64_t R, int real, const void *x,
                   int64_t x_stride, int low, const void *a, const void *b, const int32_t *adapter, const float *scale, const void *base,
                   int64_t base_stride, void *out, int64_t out_stride, void *workspace, size_t workspace_bytes) {
    RWKV_CHECK_ARG(x && a && b && adapter && out, "rwkv_lora_rows: null pointer");
    RWKV_CHECK_ARG(T > 0 && n_in > 0 && n_out > 0 && N > 0 && R > 0, "rwkv_lora_rows: sizes must be positive");
    RWKV_CHECK_ARG(real == RWKV_F32 || real == RWKV_F64, "rwkv_lora_rows: rows are float32 or float64");
    RWKV_CHECK_ARG(low == RWKV_F32 || low == RWKV_BF16 || low == RWKV_F16, "rwkv_lora_rows: adapters are float32, bfloat16 or float16");
    RWKV_CHECK_ARG(x_stride >= 0 && out_stride >= (T > 1 ? n_out : 0) && (!base || base_stride >= 0), "rwkv_lora_rows: row stride too small");
    if (R > 256 || T * R >= (1ll << 31) || T * ceil_div(n_out, 256) >= (1ll << 31) || n_in >= (1ll << 31) || N >= (1ll << 31))
        return set_error(RWKV_ERR_SIZE, "rwkv_lora_rows: too many rows, or a rank over 256");
    RWKV_CHECK_ALIGN(workspace, 16);
    if (!workspace || workspace_bytes < rwkv_lora_rows_workspace_bytes(T, n_in, n_out, N, R, real))
        return set_error(RWKV_ERR_WORKSPACE, "rwkv_lora_rows: workspace too small");
    const LoraArgs p{T, n_in, n_out, N, R, x, x_stride, a, b, adapter, scale, base, base_stride, out, out_stride, workspace};
    with_real(real, [&](auto re) {
        with_low(low, [&](auto lo) {
            using Real = typename decltype(re)::type; using Low = typename decltype(lo)::type;
            hipLaunchKernelGGL((lora_down_kernel<Real, Low>), dim3((unsigned)ceil_div(T * R, 4)), dim3(256), 0, (hipStream_t)stream, p);
            hipLaunchKernelGGL((lora_up_kernel<Real, Low>), dim3((unsigned)(T * ceil_div(n_out, 256))), dim3(256), 0, (hipStream_t)stream, p);
        });
    });
    RWKV_CHECK_LAUNCH("lora_up_kernel");
    return RWKV_OK;
}

}  // extern "C"
