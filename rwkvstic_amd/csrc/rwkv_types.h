// Element types of the serving operators: rwkv_type to C++ types, and a call made for one of them.
#pragma once

#include "rwkv_common.h"

#include <atomic>

namespace rwkv {

template <typename T> struct Elem { using type = T; };

inline size_t type_bytes(int t) { return t == RWKV_F64 ? 8 : t == RWKV_F32 ? 4 : 2; }

// fn(Elem<T>{}) for the element type T of the number t
template <typename F> auto with_low(int t, F &&fn) { return t == RWKV_F32 ? fn(Elem<float>{}) : t == RWKV_BF16 ? fn(Elem<__bf16>{}) : fn(Elem<_Float16>{}); }
template <typename F> auto with_real(int t, F &&fn) { return t == RWKV_F64 ? fn(Elem<double>{}) : fn(Elem<float>{}); }

// Whether T rows of n bytes at a, and of m bytes at b, share memory; rows as many bytes apart as is said.  Rows equally far apart may lie
// between each other.
inline bool rows_share(int64_t T, const void *a, int64_t a_apart, int64_t n, const void *b, int64_t b_apart, int64_t m) {
    const int64_t at = (int64_t)((uintptr_t)b - (uintptr_t)a);
    if (at >= (T - 1) * a_apart + n || -at >= (T - 1) * b_apart + m) return false;
    if (a_apart != b_apart || a_apart <= 0 || T == 1) return true;
    const int64_t off = (at % a_apart + a_apart) % a_apart;
    return off < n || off + m > a_apart;
}

// Whether a launch of this many workgroups has fewer than 2^32 threads, which is what a dispatch counts in 32 bits.
inline bool launchable(int64_t groups, int64_t threads) { return groups * threads < (1ll << 32); }

// Lets a kernel have this much dynamic LDS where that is over the default limit; asked of the runtime once a device.
template <auto Kernel> int allow_lds(size_t bytes) {
    if (bytes <= 65536) return RWKV_OK;
    static std::atomic<size_t> allowed[64];
    int dev = 0;
    RWKV_CHECK_HIP(hipGetDevice(&dev));
    if (dev < 0 || dev >= 64 || allowed[dev].load() < bytes) {
        RWKV_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
        if (dev >= 0 && dev < 64) allowed[dev].store(bytes);
    }
    return RWKV_OK;
}

}  // namespace rwkv
