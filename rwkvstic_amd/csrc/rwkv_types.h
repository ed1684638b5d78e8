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
