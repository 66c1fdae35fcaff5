// Element types of the operators that work on fp32, bf16 or fp16 tensors: storage, conversion to and from fp32 (round to nearest
// even; overflow to infinity, as a torch cast does) and 16-byte vectors of them.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace adx {

enum Dtype : int { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// N elements moved as one load or store (16, 8, 4 or 2 bytes)
template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

inline int dtype_bytes(int dt) { return dt == DT_F32 ? 4 : 2; }
inline bool dtype_ok(int dt) { return dt == DT_F32 || dt == DT_BF16 || dt == DT_F16; }

// Calls f(T{}) with the element type that `dt` names.
template <typename F> inline void with_dtype(int dt, F&& f) {
    if (dt == DT_BF16) f(__bf16{});
    else if (dt == DT_F16) f(_Float16{});
    else f(float{});
}

}  // namespace adx
