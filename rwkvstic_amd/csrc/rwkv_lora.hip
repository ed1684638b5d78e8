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
// Memory bounds them where rows or adapters are many: 2048 rows, 5120 to 20480, 8 bfloat16 adapters of rank 128, float32 rows: 6 + 39 +
// 118 us, the last one at 3.2 TB/s.  Float64 rows, 1024 of 2560 to 2560, 5 adapters of rank 32: 5 + 13 + 15 us (5 of them
// matrix instructions; the rest is few workgroups that wait twice for their own loads, and 21 MB each way).  One row: 4 + 4 us, each the time from an empty kernel's start to its first loads and back.
#include "rwkv_types.h"

namespace rwkv {

namespace {

// Most rows whose tiles the wavefronts find for themselves.  (2560 to 2560 of rank 32, 8 adapters: 96 rows 10.3 us directly and 15.7
// sorted in float32, 15.8 and 18.2 in float64; 192 rows 16.6 and 16.2, 25.7 and 18.7; 8 adapters or 32, the same within 2 us)
constexpr int kDirect = 128;
constexpr int kWindow = 1024;         // rows sorted together by lora_plan_kernel: a thread each
constexpr int kSlices = 8;            // most slices of n_in
constexpr int kFew = 4;               // rows of a tile that are multiplied without the matrix cores, where tiles are found directly
constexpr int kDownWaves = 8;         // wavefronts of lora_down_kernel: parts of a slice

struct Tile { int first, n, adapter; };          // rows order[first .. first + n - 1]

struct LoraArgs {
    int64_t T, n_in, n_out, N, R;
    const void *x; int64_t x_stride;
    const void *a, *b;
    const int32_t *adapter;
    const float *scale;
    const void *base; int64_t base_stride;
    void *out; int64_t out_stride;
    int slices, steps, range;             // slices of n_in, blocks of 32 in a wavefront's part of each; outputs of a workgroup
    int chunks;                           // ranges, filled up to whole rounds of the XCDs
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

template <typename Real, typename Low>
__device__ __forceinline__ void add_whole(typename Four<Real>::type &acc, const Eight<Low> &l, const Eight<Real> &r) {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = mfma((Real)l.e[e], r.e[e], acc);
}
// Whether one of four values is no number, and those of them that are none from another four.
__device__ __forceinline__ bool no_number(f32x4 v) { return __builtin_isunordered(v[0], v[1]) || __builtin_isunordered(v[2], v[3]); }
__device__ __forceinline__ void numbers(f32x4 &v, f32x4 others) {
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = v[c] == v[c] ? v[c] : others[c];
}

// What the matrix instructions make of eight terms (32 with the other lanes'): left operand from an adapter, right one from x or h.
// In LDS the right operands of a row of n lie in planes [rows][n + pad]; the pad leaves rows an odd number of 16 bytes apart.
template <typename Real, typename Low> struct Product {
    using Vec = typename Four<Real>::type;
    using Right = Eight<Real>;
    static constexpr bool kParts = false;
    static constexpr int kPad = 16 / sizeof(Real);
    static constexpr int row_bytes(int n) { return (n + kPad) * sizeof(Real); }
    static __device__ __forceinline__ Right right(const Eight<Real> &v) { return v; }
    static __device__ __forceinline__ void put(unsigned char *lds, int rows, int n, int row, int k, const Vec &v) {
        *reinterpret_cast<Vec *>(reinterpret_cast<Real *>(lds) + row * (n + kPad) + k) = v;
    }
    static __device__ __forceinline__ Right get(const unsigned char *lds, int rows, int n, int row, int k) {
        Right r;
        load8<true>(r, reinterpret_cast<const Real *>(lds) + row * (n + kPad), k, n);
        return r;
    }
    static __device__ __forceinline__ void add(Vec &acc, const Eight<Low> &l, const Right &r) { add_whole(acc, l, r); }
};

// float32 rows and bfloat16 adapters: a float32 value is the sum of three bfloat16 ones, its 24 bits cut in three, so that three
// bfloat16 products with float32 sums lose nothing, in a fifth of the matrix cores' time for float32 operands.  But for parts under
// 2^-126, which the instructions take for 0: of a value under 2^-103 up to 2^-125 can be lost (float32 instructions lose
// none), which does not show beside terms of ordinary size.  And but for infinities:
// one has no rest, and a part that is 0 must not meet one.  A sum with an infinite term comes out as no number, or right; the sums that
// are none are taken again of whole operands (kParts), so that they are what the other types' are.
template <> struct Product<float, __bf16> {
    typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
    using Vec = f32x4;
    struct Right { u32x4 part[3]; };
    static constexpr bool kParts = true;
    static constexpr int kPad = 8;
    static constexpr int row_bytes(int n) { return 3 * (n + kPad) * 2; }
    static __device__ __forceinline__ float rest(float v) { return v - __uint_as_float(__float_as_uint(v) & 0xffff0000u); }
    static __device__ __forceinline__ uint32_t upper(float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u); }
    static __device__ __forceinline__ Right right(const Eight<float> &v) {
        Right r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = v.e[2 * i], b = v.e[2 * i + 1], a1 = rest(a), b1 = rest(b);
            r.part[0][i] = upper(a, b); r.part[1][i] = upper(a1, b1); r.part[2][i] = upper(rest(a1), rest(b1));
        }
        return r;
    }
    static __device__ __forceinline__ void put(unsigned char *lds, int rows, int n, int row, int k, const Vec &v) {
        float f[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int part = 0; part < 3; ++part) {
            *reinterpret_cast<uint2 *>(lds + ((part * rows + row) * (n + kPad) + k) * 2) = make_uint2(upper(f[0], f[1]), upper(f[2], f[3]));
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = fabsf(f[i]) == INFINITY ? 0.f : rest(f[i]);          // (so that the parts add up to the value)
        }
    }
    static __device__ __forceinline__ float whole(const unsigned char *lds, int rows, int n, int row, int k) {
        float v = 0.f;
#pragma unroll
        for (int part = 2; part >= 0; --part) v += (float)*reinterpret_cast<const __bf16 *>(lds + ((part * rows + row) * (n + kPad) + k) * 2);
        return v;
    }
    static __device__ __forceinline__ Right get(const unsigned char *lds, int rows, int n, int row, int k) {
        Right r;
#pragma unroll
        for (int part = 0; part < 3; ++part) r.part[part] = *reinterpret_cast<const u32x4 *>(lds + ((part * rows + row) * (n + kPad) + k) * 2);
        return r;
    }
    static __device__ __forceinline__ void add(Vec &acc, const Eight<__bf16> &l, const Right &r) {
#pragma unroll
        for (int part = 2; part >= 0; --part)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, l.part[0]), __builtin_bit_cast(bf16x8, r.part[part]), acc, 0, 0, 0);
    }
};

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

// A workgroup to NT times 16 rows, RT tiles of 16 ranks and a slice of n_in, of which each wavefront takes a part, with the
// loads of the next 32 terms under way.  Neighbouring workgroups (on different XCDs) have different slices, so that an XCD's L2
// holds its slices of a.
template <typename Real, typename Low, int RT, int NT, bool WIDE>
__global__ void __launch_bounds__(64 * kDownWaves) lora_down_kernel(LoraArgs p) {
    using Op = Product<Real, Low>;
    using Vec = typename Op::Vec;
    __shared__ int rows[64];
    extern __shared__ __align__(16) unsigned char smem[];
    Vec *sums = reinterpret_cast<Vec *>(smem);        // [kDownWaves / 2][NT * RT][64]
    constexpr int kParts = 4 / NT;
    const int slice = blockIdx.x % p.slices, place = blockIdx.x / p.slices, parts = p.order ? kParts : 1;
    const int row0 = place % parts * NT * 16, rank0 = blockIdx.z * RT * 16;
    Tile tile;
    if (!find_tile(p, place / parts, tile, rows) || tile.adapter < 0 || row0 >= tile.n) return;
    // (wave the same for all lanes: the loop's bounds are scalar then, and its matrix instructions, which do not look at EXEC, stand behind no mask)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const Real *x[NT];
#pragma unroll
    for (int s = 0; s < NT; ++s) x[s] = (const Real *)p.x + (int64_t)rows[min(row0 + s * 16 + i, tile.n - 1)] * p.x_stride;
    const Low *a[RT];
#pragma unroll
    for (int q = 0; q < RT; ++q)              // (ranks past the last: the last again, what comes of it is dropped)
        a[q] = (const Low *)p.a + ((int64_t)tile.adapter * p.R + min(rank0 + q * 16 + left_row<Real>(i), (int)p.R - 1)) * p.n_in;
    Vec acc[NT][RT];
#pragma unroll
    for (int s = 0; s < NT; ++s)
#pragma unroll
        for (int q = 0; q < RT; ++q) acc[s][q] = Vec{0, 0, 0, 0};
    const int64_t k0 = ((int64_t)slice * kDownWaves + wave) * p.steps * 32, k1 = min(p.n_in, k0 + (int64_t)p.steps * 32);
    struct Terms { Eight<Real> x[NT]; Eight<Low> a[RT]; };
    auto load = [&](Terms &v, int64_t k) {
        if (k >= k1) return;
#pragma unroll
        for (int s = 0; s < NT; ++s) load8<WIDE>(v.x[s], x[s], k + 8 * g, k1);
#pragma unroll
        for (int q = 0; q < RT; ++q) load8<WIDE>(v.a[q], a[q], k + 8 * g, k1);
    };
    auto multiply = [&](const Terms &v) {
#pragma unroll
        for (int s = 0; s < NT; ++s) {
            const typename Op::Right r = Op::right(v.x[s]);
#pragma unroll
            for (int q = 0; q < RT; ++q) Op::add(acc[s][q], v.a[q], r);
        }
    };
    Terms even, odd;
    load(even, k0);
    for (int64_t k = k0; k < k1; k += 64) {
        load(odd, k + 32);
        multiply(even);
        load(even, k + 64);
        if (k + 32 < k1) multiply(odd);
    }
    if constexpr (Op::kParts) {
        bool again = false;
#pragma unroll
        for (int c = 0; c < NT * RT; ++c) again |= no_number(acc[c / RT][c % RT]);
        if (__any(again)) {
            Vec whole[NT][RT] = {};
#pragma unroll 1
            for (int64_t k = k0; k < k1; k += 32) {
                load(even, k);
#pragma unroll
                for (int c = 0; c < NT * RT; ++c) add_whole(whole[c / RT][c % RT], even.a[c % RT], even.x[c / RT]);
            }
#pragma unroll
            for (int c = 0; c < NT * RT; ++c) numbers(acc[c / RT][c % RT], whole[c / RT][c % RT]);
        }
    }
#pragma unroll
    for (int half = kDownWaves / 2; half >= 1; half /= 2) {
        if (half < kDownWaves / 2) __syncthreads();
#pragma unroll
        for (int c = 0; c < NT * RT; ++c)
            if (wave >= half && wave < 2 * half) sums[((wave - half) * NT * RT + c) * 64 + lane] = acc[c / RT][c % RT];
        __syncthreads();
#pragma unroll
        for (int c = 0; c < NT * RT; ++c)
            if (wave < half) acc[c / RT][c % RT] += sums[(wave * NT * RT + c) * 64 + lane];
    }
    if (wave) return;
    const Real scale = p.scale ? (Real)p.scale[tile.adapter] : (Real)1;
#pragma unroll
    for (int s = 0; s < NT; ++s) {
        if (row0 + s * 16 + i >= tile.n) break;
        Real *h = (Real *)p.h + ((int64_t)slice * p.T + rows[row0 + s * 16 + i]) * p.ranks + rank0 + 4 * g;
#pragma unroll
        for (int q = 0; q < RT; ++q) {
            Vec v = acc[s][q];
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = rank0 + q * 16 + 4 * g + c < p.R ? v[c] * scale : (Real)0;
            *reinterpret_cast<Vec *>(h + q * 16) = v;
        }
    }
}

// Few rows of an adapter, float64: on the matrix cores 16 rows would be multiplied all the same, at 64 clocks an instruction.  A thread
// to an output, whose row of b it reads by itself.  (32 rows of 24 adapters, 2560 to 10240 outputs of rank 64: 17.4 / 13.0 us; float32, whose
// instructions take 16 clocks: 8.9 / 12.5.)
template <typename Real, typename Low, bool WIDE>
__device__ __forceinline__ void up_few(const LoraArgs &p, const Tile &tile, const int *rows, Real *h, int64_t n0, int64_t n1) {
    for (int at = threadIdx.x; at < tile.n * p.ranks; at += 256) {          // (ranks past the last are 0 in h)
        const Real *from = (const Real *)p.h + (int64_t)rows[at / p.ranks] * p.ranks + at % p.ranks;
        Real sum = *from;
#pragma unroll 4
        for (int k = 1; k < p.slices; ++k) sum += from[k * p.T * p.ranks];
        h[at] = sum;
    }
    __syncthreads();
    for (int64_t n = n0 + threadIdx.x; n < n1; n += 256) {
        const Low *b = (const Low *)p.b + ((int64_t)tile.adapter * p.n_out + n) * p.R;
        Real base[kFew], acc[kFew] = {};
#pragma unroll
        for (int s = 0; s < kFew; ++s) base[s] = p.base && s < tile.n ? ((const Real *)p.base)[(int64_t)rows[s] * p.base_stride + n] : (Real)0;
#pragma unroll 4
        for (int k = 0; k < p.R; k += 8) {
            Eight<Low> bv;
            load8<WIDE>(bv, b, k, p.R);
#pragma unroll
            for (int s = 0; s < kFew; ++s) {
                if (s >= tile.n) break;
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[s] = fma((Real)bv.e[e], h[s * p.ranks + k + e], acc[s]);
            }
        }
#pragma unroll
        for (int s = 0; s < kFew; ++s) if (s < tile.n) ((Real *)p.out)[(int64_t)rows[s] * p.out_stride + n] = base[s] + acc[s];
    }
}

// RB blocks of 32 ranks, NT times 16 rows of the tile: as many as 64 KiB of LDS hold.  An XCD takes the same ranges of outputs
// for all tiles, and so reads these rows of b once.  Two wavefronts to a SIMD for operands in parts: where sums are taken
// again the compiler would use the registers of one (2048 rows of 5120 to 5120, rank 256: 74 us, and 109 with one).
template <typename Real, typename Low, int RB, int NT, int QT, bool WIDE>
__global__ void __launch_bounds__(256, (Product<Real, Low>::kParts && WIDE && NT > 1 ? 2 : 1)) lora_up_kernel(LoraArgs p) {
    using Op = Product<Real, Low>;
    using Vec = typename Op::Vec;
    extern __shared__ __align__(16) unsigned char hs[];                        // right operands of the tile's rows
    __shared__ int rows[64];
    Tile tile;
    const int row0 = blockIdx.z * NT * 16;
    const int64_t n0 = (int64_t)(blockIdx.x % p.chunks) * p.range, n1 = min(p.n_out, n0 + p.range);
    if (n0 >= n1 || !find_tile(p, blockIdx.x / p.chunks, tile, rows) || row0 >= tile.n) return;
    const int n_rows = min(NT * 16, tile.n - row0);
    const Real *base = (const Real *)p.base;
    Real *out = (Real *)p.out;
    if (tile.adapter < 0) {                           // rows without an adapter
        if (out == base && p.out_stride == p.base_stride) return;
        constexpr int E = WIDE ? 16 / sizeof(Real) : 1;
        typedef Real Some __attribute__((ext_vector_type(E)));
        const int wide = (int)((n1 - n0) / E);
#pragma unroll 4
        for (int at = threadIdx.x; at < n_rows * wide; at += 256) {
            const int64_t t = rows[row0 + at / wide], n = n0 + at % wide * E;
            *reinterpret_cast<Some *>(out + t * p.out_stride + n) = base ? *reinterpret_cast<const Some *>(base + t * p.base_stride + n) : Some(0);
        }
        return;
    }
    if (NT == 1 && sizeof(Real) == 8 && !p.order && tile.n <= kFew) { up_few<Real, Low, WIDE>(p, tile, rows, reinterpret_cast<Real *>(hs), n0, n1); return; }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const Low *b = (const Low *)p.b + (int64_t)tile.adapter * p.n_out * p.R;
    // QT tiles of outputs: lane (j, g) comes out with n + 16 q + 4 g .. + 3 of row j, 64 bytes of a row (128 of float64) to a store
    struct Rows { Eight<Low> v[QT][RB]; };
    auto row_of = [&](int64_t n, int q) { return b + min(n + 16 * q + left_row<Real>(i), p.n_out - 1) * p.R; };
    auto load = [&](Rows &to, int64_t n) {
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            const Low *row = row_of(n, q);
#pragma unroll
            for (int k = 0; k < RB; ++k) load8<WIDE>(to.v[q][k], row, k * 32 + 8 * g, p.R);
        }
    };
    struct Onto { Vec v[QT]; };
    auto load_base = [&](Onto &to, int s, int64_t n) {
#pragma unroll
        for (int q = 0; q < QT; ++q) to.v[q] = Vec{0, 0, 0, 0};
        if (!base || s * 16 + i >= n_rows) return;
        const Real *from = base + (int64_t)rows[row0 + s * 16 + i] * p.base_stride + n + 4 * g;
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            if (WIDE) { if (n + 4 * g + 16 * q < n1) to.v[q] = *reinterpret_cast<const Vec *>(from + 16 * q); }
            else {
#pragma unroll
                for (int c = 0; c < 4; ++c) if (n + 4 * g + 16 * q + c < n1) to.v[q][c] = from[16 * q + c];
            }
        }
    };
    constexpr int kAll = 4 * 16 * QT;
    // (everything of the next outputs is on the way while these are multiplied)
    Rows next;
    Onto ahead[NT];
    int64_t n = n0 + wave * 16 * QT;
    load(next, n);
#pragma unroll
    for (int s = 0; s < NT; ++s) load_base(ahead[s], s, n);
    for (int at = threadIdx.x; at < n_rows * RB * 8; at += 256) {
        const int r = at / (RB * 8), c = at % (RB * 8) * 4;
        const Real *h = (const Real *)p.h + (int64_t)rows[row0 + r] * p.ranks + c;
        Vec s = *reinterpret_cast<const Vec *>(h);
#pragma unroll 4
        for (int k = 1; k < p.slices; ++k) s += *reinterpret_cast<const Vec *>(h + k * p.T * p.ranks);
        Op::put(hs, NT * 16, RB * 32, r, c, s);
    }
    __syncthreads();
    for (; n < n1; n += kAll) {
        const Rows now = next;
        Onto onto[NT];
#pragma unroll
        for (int s = 0; s < NT; ++s) onto[s] = ahead[s];
        if (n + kAll < n1) {
            load(next, n + kAll);
#pragma unroll
            for (int s = 0; s < NT; ++s) load_base(ahead[s], s, n + kAll);
        }
#pragma unroll
        for (int s = 0; s < NT; ++s) {
            if (s * 16 >= n_rows) break;
            Vec acc[QT];
#pragma unroll
            for (int q = 0; q < QT; ++q) acc[q] = Vec{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < RB; ++k) {
                const typename Op::Right r = Op::get(hs, NT * 16, RB * 32, s * 16 + i, k * 32 + 8 * g);
#pragma unroll
                for (int q = 0; q < QT; ++q) Op::add(acc[q], now.v[q][k], r);
            }
            if constexpr (Op::kParts) {
                bool again = false;
#pragma unroll
                for (int q = 0; q < QT; ++q) again |= no_number(acc[q]);
                if (__any(again && s * 16 + i < n_rows)) {
#pragma unroll
                    for (int q = 0; q < QT; ++q) {
                        Vec whole = {0, 0, 0, 0};
#pragma unroll 1
                        for (int term = 0; term < RB * 8; ++term) {          // (one at a time, for what that takes of registers)
                            const int k = term / 8 * 32 + 8 * g + term % 8;
                            whole = mfma(k < p.R ? (float)row_of(n, q)[k] : 0.f, Op::whole(hs, NT * 16, RB * 32, s * 16 + i, k), whole);
                        }
                        numbers(acc[q], whole);
                    }
                }
            }
            if (s * 16 + i >= n_rows) continue;
            Real *to = out + (int64_t)rows[row0 + s * 16 + i] * p.out_stride + n + 4 * g;
#pragma unroll
            for (int q = 0; q < QT; ++q) {
                acc[q] += onto[s].v[q];
                if (WIDE) { if (n + 4 * g + 16 * q < n1) *reinterpret_cast<Vec *>(to + 16 * q) = acc[q]; }
                else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) if (n + 4 * g + 16 * q + c < n1) to[16 * q + c] = acc[q][c];
                }
            }
        }
    }
}

// Tiles of 16 rows to a wavefront of lora_down_kernel where rows are sorted: two read the same of a, where their sums stay in registers.
constexpr int many_rows(int real) { return real == RWKV_F32 ? 2 : 1; }

// How a call is cut up; the same for its workspace and its launches.
struct LoraPlan {
    bool direct;
    int windows, slots;                   // tiles are looked for in windows * slots places
    int group, groups, ranks;             // tiles of 16 ranks to a wavefront of lora_down_kernel, and wavefronts; ranks: 32, 64, 128 or 256
    int slices, steps, range, chunks;
    size_t h_bytes, order, tile_bytes;
    LoraPlan(int64_t T, int64_t n_in, int64_t n_out, int64_t N, int64_t R, int real) {
        direct = T <= kDirect;
        windows = direct ? 1 : (int)ceil_div(T, kWindow);
        slots = (int)(direct ? T : kWindow / 64 + (N + 1 < kWindow ? N + 1 : kWindow));
        R = R < 1 ? 1 : R;                                  // (without adapters there may be no rank)
        group = R <= 32 ? 2 : R <= 64 ? 4 : 8;
        groups = (int)ceil_div(R, group * 16);
        ranks = group * groups * 16;
        // workgroups for the whole device, while a wavefront has terms left to do (float64, 2560 to 2560, 8 adapters of rank 16, 100 rows:
        // slices up to 256 workgroups 20 us, 512 15.6, 1024 14.1; 2048 rows: 512 47.0, 1024 44.7, 2048 44.8)
        const int64_t blocks = ceil_div(n_in, 32), tiles = direct ? T : ceil_div(T, 16);
        int64_t s = 1;
        while (s < kSlices && s * tiles < (direct ? 512 : 1024) && blocks > s * kDownWaves) s *= 2;
        steps = (int)ceil_div(blocks, kDownWaves * s);
        slices = (int)ceil_div(blocks, kDownWaves * steps);
        // (2560 to 10240, 24 adapters of rank 64, 32 rows: up to 1024 workgroups 16.4 us in float32 and 26.8 in float64, 2048 13.7 and
        // 21.9, 4096 14.7 and 22.1; 2048 rows of 5120 to 5120 in float32: 512 91.4, 1024 91.5, 2048 98.5)
        const int64_t wanted = ceil_div(direct || real == RWKV_F64 ? 2048 : 1024, direct ? T : ceil_div(T, 64));
        range = (int)round_up(ceil_div(n_out, wanted), direct ? 256 : 128);
        chunks = (int)ceil_div(n_out, range);
        if (chunks > 8) chunks = (int)round_up(chunks, 8);
        h_bytes = round_up((size_t)slices * T * ranks * type_bytes(real), 256);
        order = direct ? 0 : round_up((size_t)T * 4, 256);
        tile_bytes = direct ? 0 : (size_t)windows * slots * sizeof(Tile);
    }
    size_t bytes() const { return h_bytes + order + tile_bytes; }
};

template <typename Real, typename Low, bool WIDE>
void launch(hipStream_t st, const LoraPlan &pl, const LoraArgs &p) {
    using Op = Product<Real, Low>;
    const int places = pl.windows * pl.slots;
    constexpr int kMany = many_rows(sizeof(Real) == 4 ? RWKV_F32 : RWKV_F64);
    auto go_down = [&](auto one, auto many, int group) {
        if (p.N == 0) return;                 // (every row gets base)
        const int nt = pl.direct ? 1 : kMany;
        const dim3 down((unsigned)(places * (pl.direct ? 1 : 4 / nt) * pl.slices), 1, (unsigned)pl.groups);
        hipLaunchKernelGGL(pl.direct ? one : many, down, dim3(64 * kDownWaves), (size_t)kDownWaves / 2 * nt * group * 64 * 4 * sizeof(Real), st, p);
    };
    if (pl.group == 2) go_down(lora_down_kernel<Real, Low, 2, 1, WIDE>, lora_down_kernel<Real, Low, 2, kMany, WIDE>, 2);
    else if (pl.group == 4) go_down(lora_down_kernel<Real, Low, 4, 1, WIDE>, lora_down_kernel<Real, Low, 4, kMany, WIDE>, 4);
    else go_down(lora_down_kernel<Real, Low, 8, 1, WIDE>, lora_down_kernel<Real, Low, 8, kMany, WIDE>, 8);
    auto go_up = [&](auto one, auto many, int nt) {
        const int rows = 16 * (pl.direct ? 1 : nt);
        const dim3 up((unsigned)(places * pl.chunks), 1, (unsigned)(pl.direct ? 1 : 4 / nt));
        hipLaunchKernelGGL(pl.direct ? one : many, up, dim3(256), (size_t)rows * Op::row_bytes(pl.ranks), st, p);
    };
    constexpr int k128 = sizeof(Real) == 4 ? 4 : 2, k256 = k128 / 2;            // rows in LDS, by ranks
    constexpr int kWide = sizeof(Real) == 4 ? 2 : 1;                            // tiles of outputs to a wavefront: 128 bytes of a row
    if (pl.ranks == 32) go_up(lora_up_kernel<Real, Low, 1, 1, kWide, WIDE>, lora_up_kernel<Real, Low, 1, 4, kWide, WIDE>, 4);
    else if (pl.ranks == 64) go_up(lora_up_kernel<Real, Low, 2, 1, kWide, WIDE>, lora_up_kernel<Real, Low, 2, 4, kWide, WIDE>, 4);
    else if (pl.ranks == 128) go_up(lora_up_kernel<Real, Low, 4, 1, kWide, WIDE>, lora_up_kernel<Real, Low, 4, k128, kWide, WIDE>, k128);
    else go_up(lora_up_kernel<Real, Low, 8, 1, kWide, WIDE>, lora_up_kernel<Real, Low, 8, k256, kWide, WIDE>, k256);
}

}  // namespace

}  // namespace rwkv

using namespace rwkv;

extern "C" {

size_t rwkv_lora_rows_workspace_bytes(int64_t T, int64_t n_in, int64_t n_out, int64_t N, int64_t R, int real) {
    if (T <= 0 || n_in <= 0 || n_out <= 0 || N < 0 || (R <= 0 && N > 0)) return 0;
    return LoraPlan(T, n_in, n_out, N, R, real).bytes();
}

int rwkv_lora_rows(rwkv_stream_t stream, int64_t T, int64_t n_in, int64_t n_out, int64_t N, int64_t R, int real, const void *x,
                   int64_t x_stride, int low, const void *a, const void *b, const int32_t *adapter, const float *scale, const void *base,
                   int64_t base_stride, void *out, int64_t out_stride, void *workspace, size_t workspace_bytes) {
    RWKV_CHECK_ARG(x && adapter && out && ((a && b) || N == 0), "rwkv_lora_rows: null pointer");
    RWKV_CHECK_ARG(T > 0 && n_in > 0 && n_out > 0 && N >= 0 && (R > 0 || N == 0), "rwkv_lora_rows: sizes must be positive");
    RWKV_CHECK_ARG(real == RWKV_F32 || real == RWKV_F64, "rwkv_lora_rows: rows are float32 or float64");
    RWKV_CHECK_ARG(low == RWKV_F32 || low == RWKV_BF16 || low == RWKV_F16, "rwkv_lora_rows: adapters are float32, bfloat16 or float16");
    RWKV_CHECK_ARG(x_stride >= 0 && out_stride >= (T > 1 ? n_out : 0) && (!base || base_stride >= 0), "rwkv_lora_rows: row stride too small");
    if (R > 256 || T > (1 << 24) || n_in >= (1ll << 30) || n_out >= (1ll << 30) || N >= (1ll << 30))
        return set_error(RWKV_ERR_SIZE, "rwkv_lora_rows: too many rows, or a rank over 256");
    if (base && (base != out || base_stride != out_stride)) {
        const int64_t e = (int64_t)type_bytes(real);
        RWKV_CHECK_ARG(!rows_share(T, base, base_stride * e, n_out * e, out, out_stride * e, n_out * e), "rwkv_lora_rows: out shares memory with base and is not base");
    }
    RWKV_CHECK_ALIGN(workspace, 16);
    const LoraPlan pl(T, n_in, n_out, N, R, real);
    if (!launchable((int64_t)pl.windows * pl.slots * (pl.direct ? 1 : 4 / many_rows(real)) * pl.slices, 64 * kDownWaves) ||
        !launchable((int64_t)pl.windows * pl.slots * pl.chunks, 256))
        return set_error(RWKV_ERR_SIZE, "rwkv_lora_rows: too many rows for so many adapters");
    if (!workspace || workspace_bytes < pl.bytes()) return set_error(RWKV_ERR_WORKSPACE, "rwkv_lora_rows: workspace too small");
    // (x aside: it has been read when the first output is written)
    const int64_t er = (int64_t)type_bytes(real), el = (int64_t)type_bytes(low);
    auto apart = [&](const void *from, int64_t bytes) { return !from || !rows_share(T, out, out_stride * er, n_out * er, from, 0, bytes); };
    RWKV_CHECK_ARG(apart(a, N * R * n_in * el) && apart(b, N * n_out * R * el) && apart(adapter, T * 4) && apart(scale, N * 4),
                   "rwkv_lora_rows: out shares memory with an argument");
    uint8_t *ws = (uint8_t *)workspace;
    const LoraArgs p{T, n_in, n_out, N, R, x, x_stride, a, b, adapter, scale, base, base_stride, out, out_stride, pl.slices, pl.steps, pl.range, pl.chunks, pl.ranks,
                     ws, pl.direct ? nullptr : (int32_t *)(ws + pl.h_bytes), (Tile *)(ws + pl.h_bytes + pl.order)};
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
