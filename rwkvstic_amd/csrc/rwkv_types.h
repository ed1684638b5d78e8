// Element types of the serving operators: rwkv_type to C++ types, and a call made for one of them.
#pragma once

#include "rwkv_common.h"

namespace rwkv {

template <typename T> struct Elem { using type = T; };

inline size_t type_bytes(int t) { return t == RWKV_F64 ? 8 : t == RWKV_F32 ? 4 : 2; }

// fn(Elem<T>{}) for the element type T of the number t
template <typename F> auto with_low(int t, F &&fn) { return t == RWKV_F32 ? fn(Elem<float>{}) : t == RWKV_BF16 ? fn(Elem<__bf16>{}) : fn(Elem<_Float16>{}); }
template <typename F> auto with_real(int t, F &&fn) { return t == RWKV_F64 ? fn(Elem<double>{}) : fn(Elem<float>{}); }

}  // namespace rwkv
