// Low-rank adapters of many requests beside a shared projection (rwkv_lora_rows):
//   h[t] = scale[i] (a[i] x[t]),  out[t] = base[t] + b[i] h[t],  i = adapter[t].
//
// Rows of one adapter are put together in tiles, and both products run on the matrix cores in the rows' own type
// (v_mfma_f32_16x16x4f32, v_mfma_f64_16x16x4f64; the adapters are exact in either): the left operand is 16 rows of a or b, the right
// one 16 rows of x or h, and as the order of a sum's terms is free, each group of 16 lanes takes 8 neighbouring ones, so that
// operands come from memory in 16-byte loads, straight into the registers that the matrix instruction reads.
//   lora_plan_kernel   (over kDirect rows) sorts the rows of each window by adapter and cuts the runs into tiles
//   lora_down_kernel   a wavefront per 16 rows, up to 128 ranks and slice of n_in: parts of h
//   lora_up_kernel     a workgroup per tile and range of n_out: the parts added up into LDS, then b h on top of base
#include "rwkv_types.h"

namespace rwkv {

namespace {

constexpr int kDirect = 256;          // most rows whose tiles the wavefronts find for themselves
constexpr int kWindow = 1024;         // rows sorted together by lora_plan_kernel: a thread each
constexpr int kSlices = 8;            // most slices of n_in
constexpr int kStep = 32;             // outputs a wavefront of lora_up_kernel makes at once

struct Tile { int first, n, adapter; };          // rows order[first .. first + n - 1]

struct LoraArgs {
    int64_t T, n_in, n_out, N, R;
    const void *x; int64_t x_stride;
    const void *a, *b;
    const int32_t *adapter;
    const float *scale;
    const void *base; int64_t base_stride;
    void *out; int64_t out_stride;
    int slices, steps, range;             // slices of n_in, blocks of 32 in a quarter of each; outputs of a workgroup
    int ranks;                            // R filled up to what the kernels' tiles hold
    void *h;                              // [slices][T][ranks]
    int32_t *order;                       // rows by window and adapter, or null: tiles are found directly
    Tile *tiles;                          // [windows][slots]
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef double f64x4 __attribute__((ext_vector_type(4)));

template <typename Real> struct Four;
template <> struct Four<float> { using type = f32x4; };
template <> struct Four<double> { using type = f64x4; };

__device__ __forceinline__ f32x4 mfma(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f64x4 mfma(double a, double b, f64x4 c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }

// Lane (j, g) = (lane % 16, lane / 16) holds the rows 4 g + v, v < 4, of column j of a float32 product, and 4 v + g of a float64
// one: with its left rows in this order, it is 4 g + v there too.
template <typename Real> __device__ __forceinline__ int left_row(int i) { return sizeof(Real) == 4 ? i : 4 * (i & 3) + (i >> 2); }

// Eight neighbouring elements k .. k + 7 of a row of n; WIDE: the row is 16-byte aligned and n fills whole 16 bytes.
template <typename T> union Eight { u32x4 part[sizeof(T) / 2]; T e[8]; };
template <bool WIDE, typename T>
__device__ __forceinline__ void load8(Eight<T> &to, const T *row, int64_t k, int64_t n) {
    if constexpr (WIDE) {
        constexpr int E = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 8 / E; ++i) to.part[i] = k + i * E < n ? *reinterpret_cast<const u32x4 *>(row + k + i * E) : u32x4{0, 0, 0, 0};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) to.e[i] = k + i < n ? row[k + i] : (T)0.f;
    }
}

// The tile of a workgroup: its rows in `rows` (LDS, 64 at most).  false: this workgroup has none.  Directly: slot t has a tile if the
// rows before t hold a multiple of 16 with t's adapter; it is t and the next 15 of them.
__device__ __forceinline__ bool find_tile(const LoraArgs &p, int64_t slot, Tile &tile, int *rows) {
    if (p.order) {
        tile = p.tiles[slot];
        if (tile.n == 0) return false;
        if (threadIdx.x < tile.n) rows[threadIdx.x] = p.order[tile.first + threadIdx.x];
    } else {
        const int lane = threadIdx.x & 63, t = (int)slot;
        const int32_t own = p.adapter[t];
        const bool none = own < 0 || own >= p.N;
        unsigned long long same[kDirect / 64];
        int before = 0;
#pragma unroll
        for (int w = 0; w < kDirect / 64; ++w) {
            const int s = 64 * w + lane;
            const int32_t i = s < p.T ? p.adapter[s] : 0;
            same[w] = __ballot(s < p.T && (i == own || (none && (i < 0 || i >= p.N))));
            before += __popcll(64 * w + 63 < t ? same[w] : 64 * w > t ? 0ull : same[w] & ((1ull << (t & 63)) - 1));
        }
        if (before & 15) return false;
        int at = -before, n = 0;
#pragma unroll
        for (int w = 0; w < kDirect / 64; ++w) {
            const int rank = at + __popcll(same[w] & ((1ull << lane) - 1));
            if ((same[w] >> lane & 1) && rank >= 0 && rank < 16 && threadIdx.x < 64) rows[rank] = 64 * w + lane;
            at += __popcll(same[w]);
        }
        n = min(at, 16);
        tile = {0, n, none ? -1 : own};
    }
    __syncthreads();
    return true;
}

__global__ void __launch_bounds__(kWindow) lora_plan_kernel(LoraArgs p, int slots, int bits) {
    __shared__ int s_key[kWindow], s_row[kWindow], s_count[kWindow / 64], s_first[kWindow / 64], s_next[kWindow / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t begin = (int64_t)blockIdx.x * kWindow;
    const int live = (int)min((int64_t)kWindow, p.T - begin);
    const unsigned long long below = (1ull << lane) - 1;
    // a stable sort by adapter, bit by bit; rows without one last, and behind them the places of the last window that are no rows
    int key = 0x7fffffff, row = tid;
    if (tid < live) { const int32_t i = p.adapter[begin + tid]; key = i < 0 || i >= p.N ? (int)p.N : i; }
    for (int bit = 0; bit < bits; ++bit) {
        const bool one = key >> bit & 1;
        const unsigned long long zeros = __ballot(!one);
        if (lane == 0) s_count[wave] = __popcll(zeros);
        __syncthreads();
        int all = 0, before = 0;
#pragma unroll
        for (int w = 0; w < kWindow / 64; ++w) { before += w < wave ? s_count[w] : 0; all += s_count[w]; }
        before += __popcll(zeros & below);
        const int to = one ? all + tid - before : before;
        s_key[to] = key; s_row[to] = row;
        __syncthreads();
        key = s_key[tid]; row = s_row[tid];
    }
    if (tid < live) p.order[begin + tid] = (int)(begin + row);
    s_key[tid] = key;
    __syncthreads();
    // runs of one adapter, tiles of 64 of them
    const bool starts = tid == 0 || s_key[tid - 1] != key;
    const unsigned long long runs = __ballot(starts);
    if (lane == 0) { s_first[wave] = runs ? 64 * wave + 63 - __clzll(runs) : -1; s_next[wave] = runs ? 64 * wave + __ffsll(runs) - 1 : -1; }
    __syncthreads();
    const unsigned long long upto = runs & (below | 1ull << lane), after = runs & ~(below | 1ull << lane);
    int first = upto ? 64 * wave + 63 - __clzll(upto) : -1, next = after ? 64 * wave + __ffsll(after) - 1 : -1;
    for (int w = wave - 1; w >= 0 && first < 0; --w) first = s_first[w];
    for (int w = wave + 1; w < kWindow / 64 && next < 0; ++w) next = s_next[w];
    const bool heads = tid < live && (tid - first) % 64 == 0;
    const unsigned long long tiles = __ballot(heads);
    if (lane == 0) s_count[wave] = __popcll(tiles);
    __syncthreads();
    int at = __popcll(tiles & below), all = 0;
    for (int w = 0; w < kWindow / 64; ++w) { at += w < wave ? s_count[w] : 0; all += s_count[w]; }
    Tile *to = p.tiles + (int64_t)blockIdx.x * slots;
    if (heads) to[at] = {(int)begin + tid, min(64, min(next < 0 ? live : next, live) - tid), key == (int)p.N ? -1 : key};
    for (int i = all + tid; i < slots; i += kWindow) to[i] = {0, 0, -1};
}

// A workgroup to 16 rows, RT tiles of 16 ranks and a slice of n_in, of which each wavefront takes a quarter.
template <typename Real, typename Low, int RT, bool WIDE>
__global__ void __launch_bounds__(256) lora_down_kernel(LoraArgs p) {
    using Vec = typename Four<Real>::type;
    __shared__ int rows[64];
    __shared__ Vec sums[3][RT][64];
    const int parts = p.order ? 4 : 1, part = blockIdx.x % parts, rank0 = blockIdx.z * RT * 16;
    Tile tile;
    if (!find_tile(p, blockIdx.x / parts, tile, rows) || tile.adapter < 0 || part * 16 >= tile.n) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int64_t t = rows[min(part * 16 + i, tile.n - 1)];
    const Real *x = (const Real *)p.x + t * p.x_stride;
    const Low *a[RT];
#pragma unroll
    for (int q = 0; q < RT; ++q)              // (ranks past the last: the last again, what comes of it is dropped)
        a[q] = (const Low *)p.a + ((int64_t)tile.adapter * p.R + min(rank0 + q * 16 + left_row<Real>(i), (int)p.R - 1)) * p.n_in;
    Vec acc[RT];
#pragma unroll
    for (int q = 0; q < RT; ++q) acc[q] = Vec{0, 0, 0, 0};
    const int64_t k0 = ((int64_t)blockIdx.y * 4 + wave) * p.steps * 32, k1 = min(p.n_in, k0 + (int64_t)p.steps * 32);
    Eight<Real> xv;
    Eight<Low> av[RT];
    auto load = [&](int64_t k) {
        load8<WIDE>(xv, x, k, k1);
#pragma unroll
        for (int q = 0; q < RT; ++q) load8<WIDE>(av[q], a[q], k, k1);
    };
    if (k0 < k1) load(k0 + 8 * g);
    for (int64_t k = k0; k < k1; k += 32) {
        const Eight<Real> xn = xv;
        Eight<Low> an[RT];
#pragma unroll
        for (int q = 0; q < RT; ++q) an[q] = av[q];
        if (k + 32 < k1) load(k + 32 + 8 * g);
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int q = 0; q < RT; ++q) acc[q] = mfma((Real)an[q].e[e], xn.e[e], acc[q]);
    }
    if (wave)
#pragma unroll
        for (int q = 0; q < RT; ++q) sums[wave - 1][q][lane] = acc[q];
    __syncthreads();
    if (wave || part * 16 + i >= tile.n) return;
    const Real scale = p.scale ? (Real)p.scale[tile.adapter] : (Real)1;
    Real *h = (Real *)p.h + ((int64_t)blockIdx.y * p.T + t) * p.ranks + rank0 + 4 * g;
#pragma unroll
    for (int q = 0; q < RT; ++q) {
        const Vec s = ((acc[q] + sums[0][q][lane]) + sums[1][q][lane]) + sums[2][q][lane];
        Vec v;
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = rank0 + q * 16 + 4 * g + c < p.R ? s[c] * scale : (Real)0;
        *reinterpret_cast<Vec *>(h + q * 16) = v;
    }
}

// RB blocks of 32 ranks, NT times 16 rows of the tile: as many as 64 KiB of LDS hold.
template <typename Real, typename Low, int RB, int NT, bool WIDE>
__global__ void __launch_bounds__(256) lora_up_kernel(LoraArgs p) {
    using Vec = typename Four<Real>::type;
    constexpr int kPad = 16 / sizeof(Real), kRow = RB * 32 + kPad;              // rows 16 bytes apart in the banks
    extern __shared__ __align__(16) unsigned char smem[];
    Real *hs = reinterpret_cast<Real *>(smem);                                  // [NT * 16][kRow]
    __shared__ int rows[64];
    Tile tile;
    const int row0 = blockIdx.z * NT * 16;
    if (!find_tile(p, blockIdx.x, tile, rows) || row0 >= tile.n) return;
    const int n_rows = min(NT * 16, tile.n - row0);
    const int64_t n0 = (int64_t)blockIdx.y * p.range, n1 = min(p.n_out, n0 + p.range);
    const Real *base = (const Real *)p.base;
    Real *out = (Real *)p.out;
    if (tile.adapter < 0) {                           // rows without an adapter
        if (out == base && p.out_stride == p.base_stride) return;
        for (int r = row0; r < row0 + n_rows; ++r)
            for (int64_t n = n0 + threadIdx.x; n < n1; n += 256)
                out[(int64_t)rows[r] * p.out_stride + n] = base ? base[(int64_t)rows[r] * p.base_stride + n] : (Real)0;
        return;
    }
    for (int i = threadIdx.x; i < n_rows * RB * 8; i += 256) {
        const int r = i / (RB * 8), c = i % (RB * 8) * 4;
        const Real *h = (const Real *)p.h + (int64_t)rows[row0 + r] * p.ranks + c;
        Vec s = *reinterpret_cast<const Vec *>(h);
#pragma unroll 4
        for (int k = 1; k < p.slices; ++k) s += *reinterpret_cast<const Vec *>(h + k * p.T * p.ranks);
        *reinterpret_cast<Vec *>(hs + r * kRow + c) = s;
    }
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const Low *b = (const Low *)p.b + (int64_t)tile.adapter * p.n_out * p.R;
    for (int64_t n = n0 + wave * kStep; n < n1; n += 4 * kStep) {
        // two tiles of outputs, in an order that leaves each lane with the eight n + 8 g .. n + 8 g + 7
        Eight<Low> bv[2][RB];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int l = left_row<Real>(i);
            const Low *row = b + min(n + 8 * (l >> 2) + 4 * q + (l & 3), n1 - 1) * p.R;
#pragma unroll
            for (int k = 0; k < RB; ++k) load8<WIDE>(bv[q][k], row, k * 32 + 8 * g, p.R);
        }
#pragma unroll
        for (int s = 0; s < NT; ++s) {
            if (s * 16 >= n_rows) break;
            const bool in = s * 16 + i < n_rows;
            const int64_t t = rows[row0 + min(s * 16 + i, n_rows - 1)];
            Vec acc[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int64_t at = n + 8 * g + 4 * q;
                acc[q] = Vec{0, 0, 0, 0};
                if (base && in) {
                    const Real *from = base + t * p.base_stride + at;
                    if (WIDE) { if (at < n1) acc[q] = *reinterpret_cast<const Vec *>(from); }
                    else {
#pragma unroll
                        for (int c = 0; c < 4; ++c) if (at + c < n1) acc[q][c] = from[c];
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < RB; ++k) {
                Eight<Real> hv;
                load8<true>(hv, hs + (s * 16 + i) * kRow, k * 32 + 8 * g, RB * 32);
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int q = 0; q < 2; ++q) acc[q] = mfma((Real)bv[q][k].e[e], hv.e[e], acc[q]);
            }
            if (!in) continue;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int64_t at = n + 8 * g + 4 * q;
                Real *to = out + t * p.out_stride + at;
                if (WIDE) { if (at < n1) *reinterpret_cast<Vec *>(to) = acc[q]; }
                else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) if (at + c < n1) to[c] = acc[q][c];
                }
            }
        }
    }
}

// How a call is cut up; the same for its workspace and its launches.
struct LoraPlan {
    bool direct;
    int windows, slots;                   // tiles are looked for in windows * slots places
    int group, groups, ranks;             // tiles of 16 ranks to a wavefront of lora_down_kernel, and wavefronts
    int slices, steps, range;
    size_t h_bytes, order_bytes, tile_bytes;
    LoraPlan(int64_t T, int64_t n_in, int64_t n_out, int64_t N, int64_t R, int real) {
        direct = T <= kDirect;
        windows = direct ? 1 : (int)ceil_div(T, kWindow);
        slots = (int)(direct ? T : kWindow / 64 + (N + 1 < kWindow ? N + 1 : kWindow));
        group = R <= 32 ? 2 : R <= 64 ? 4 : 8;
        groups = (int)ceil_div(R, group * 16);
        ranks = group * groups * 16;
        const int64_t blocks = ceil_div(n_in, 32), tiles = direct ? T : ceil_div(T, 16);
        int64_t s = ceil_div(512, tiles);
        s = s < 1 ? 1 : s > kSlices ? kSlices : s;
        steps = (int)ceil_div(blocks, 4 * s);
        slices = (int)ceil_div(blocks, 4 * steps);
        const int64_t chunks = ceil_div(direct ? 1024 : 2048, direct ? T : ceil_div(T, 64));
        range = (int)round_up(ceil_div(n_out, chunks), 4 * kStep);
        h_bytes = round_up((size_t)slices * T * ranks * type_bytes(real), 256);
        order_bytes = direct ? 0 : round_up((size_t)T * 4, 256);
        tile_bytes = direct ? 0 : (size_t)windows * slots * sizeof(Tile);
    }
    size_t bytes() const { return h_bytes + order_bytes + tile_bytes; }
};

template <typename Real, typename Low, bool WIDE>
void launch(hipStream_t st, const LoraPlan &pl, const LoraArgs &p) {
    const int places = pl.windows * pl.slots;
    const dim3 down((unsigned)(places * (pl.direct ? 1 : 4)), (unsigned)pl.slices, (unsigned)pl.groups);
    auto go_down = [&](auto k) { hipLaunchKernelGGL(k, down, dim3(256), 0, st, p); };
    if (pl.group == 2) go_down(lora_down_kernel<Real, Low, 2, WIDE>);
    else if (pl.group == 4) go_down(lora_down_kernel<Real, Low, 4, WIDE>);
    else go_down(lora_down_kernel<Real, Low, 8, WIDE>);
    auto go_up = [&](auto one, auto many, int nt) {
        const int rows = 16 * (pl.direct ? 1 : nt);
        const dim3 up((unsigned)places, (unsigned)ceil_div(p.n_out, pl.range), (unsigned)(pl.direct ? 1 : 4 / nt));
        hipLaunchKernelGGL(pl.direct ? one : many, up, dim3(256), (size_t)rows * (pl.ranks * sizeof(Real) + 16), st, p);
    };
    constexpr int k128 = sizeof(Real) == 4 ? 4 : 2, k256 = k128 / 2;
    if (pl.ranks == 32) go_up(lora_up_kernel<Real, Low, 1, 1, WIDE>, lora_up_kernel<Real, Low, 1, 4, WIDE>, 4);
    else if (pl.ranks == 64) go_up(lora_up_kernel<Real, Low, 2, 1, WIDE>, lora_up_kernel<Real, Low, 2, 4, WIDE>, 4);
    else if (pl.ranks == 128) go_up(lora_up_kernel<Real, Low, 4, 1, WIDE>, lora_up_kernel<Real, Low, 4, k128, WIDE>, k128);
    else go_up(lora_up_kernel<Real, Low, 8, 1, WIDE>, lora_up_kernel<Real, Low, 8, k256, WIDE>, k256);
}

}  // namespace

}  // namespace rwkv

using namespace rwkv;

extern "C" {

size_t rwkv_lora_rows_workspace_bytes(int64_t T, int64_t n_in, int64_t n_out, int64_t N, int64_t R, int real) {
    if (T <= 0 || n_in <= 0 || n_out <= 0 || N <= 0 || R <= 0) return 0;
    return LoraPlan(T, n_in, n_out, N, R, real).bytes();
}

int rwkv_lora_rows(rwkv_stream_t stream, int64_t T, int64_t n_in, int64_t n_out, int64_t N, int64_t R, int real, const void *x,
                   int64_t x_stride, int low, const void *a, const void *b, const int32_t *adapter, const float *scale, const void *base,
                   int64_t base_stride, void *out, int64_t out_stride, void *workspace, size_t workspace_bytes) {
    RWKV_CHECK_ARG(x && a && b && adapter && out, "rwkv_lora_rows: null pointer");
    RWKV_CHECK_ARG(T > 0 && n_in > 0 && n_out > 0 && N > 0 && R > 0, "rwkv_lora_rows: sizes must be positive");
    RWKV_CHECK_ARG(real == RWKV_F32 || real == RWKV_F64, "rwkv_lora_rows: rows are float32 or float64");
    RWKV_CHECK_ARG(low == RWKV_F32 || low == RWKV_BF16 || low == RWKV_F16, "rwkv_lora_rows: adapters are float32, bfloat16 or float16");
    RWKV_CHECK_ARG(x_stride >= 0 && out_stride >= (T > 1 ? n_out : 0) && (!base || base_stride >= 0), "rwkv_lora_rows: row stride too small");
    if (R > 256 || T > (1 << 24) || n_in >= (1ll << 30) || n_out >= (1ll << 30) || N >= (1ll << 30))
        return set_error(RWKV_ERR_SIZE, "rwkv_lora_rows: too many rows, or a rank over 256");
    RWKV_CHECK_ALIGN(workspace, 16);
    const LoraPlan pl(T, n_in, n_out, N, R, real);
    if (!workspace || workspace_bytes < pl.bytes()) return set_error(RWKV_ERR_WORKSPACE, "rwkv_lora_rows: workspace too small");
    uint8_t *ws = (uint8_t *)workspace;
    const LoraArgs p{T, n_in, n_out, N, R, x, x_stride, a, b, adapter, scale, base, base_stride, out, out_stride, pl.slices, pl.steps, pl.range, pl.ranks,
                     ws, pl.direct ? nullptr : (int32_t *)(ws + pl.h_bytes), (Tile *)(ws + pl.h_bytes + pl.order_bytes)};
    const size_t er = type_bytes(real), el = type_bytes(low);
    auto fits = [](const void *at, int64_t elements, size_t size) { return ((uintptr_t)at | (uintptr_t)(elements * size)) % 16 == 0; };
    // (a row of four outputs may be 32 bytes, which 16-byte alignment serves)
    const bool wide = fits(x, x_stride, er) && fits(a, n_in, el) && fits(x, n_in, er) && fits(b, R, el) && fits(out, out_stride, er) && n_out % 4 == 0 &&
                      (!base || fits(base, base_stride, er));
    if (!pl.direct) {
        int bits = 1;
        while (N >> bits) ++bits;
        hipLaunchKernelGGL(lora_plan_kernel, dim3((unsigned)pl.windows), dim3(kWindow), 0, (hipStream_t)stream, p, pl.slots, bits);
        RWKV_CHECK_LAUNCH("lora_plan_kernel");
    }
    with_real(real, [&](auto re) {
        with_low(low, [&](auto lo) {
            using Real = typename decltype(re)::type; using Low = typename decltype(lo)::type;
            if (wide) launch<Real, Low, true>((hipStream_t)stream, pl, p);
            else launch<Real, Low, false>((hipStream_t)stream, pl, p);
        });
    });
    RWKV_CHECK_LAUNCH("lora_up_kernel");
    return RWKV_OK;
}

}  // extern "C"
