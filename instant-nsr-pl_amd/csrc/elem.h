// Elements of the three storage types that the training operators take (fp32, fp16, bf16): loads widen to fp32, stores round
// to nearest even.  The codes are those of the C ABI.
#pragma once
#include "nsr_common.h"

enum : uint32_t { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2 };

template <int DT> struct Elem;
template <> struct Elem<DT_F32> { using T = float; };
template <> struct Elem<DT_F16> { using T = _Float16; };
template <> struct Elem<DT_BF16> { using T = __bf16; };

template <class T, int N> struct alignas(N * sizeof(T)) Vec { T e[N]; };

static inline uint32_t dtype_size(uint32_t dt) { return dt == DT_F32 ? 4 : 2; }
