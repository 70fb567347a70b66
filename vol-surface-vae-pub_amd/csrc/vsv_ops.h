// What the sequence-memory and optimizer kernels share: element types, the activations and the launchers' checks.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

#include "../../include/vsv_hip.h"

namespace vsv {

void set_error(const char* fmt, ...);

inline int op_launch_check(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) { set_error("%s: %s", what, hipGetErrorString(e)); return (int)e; }
    return 0;
}

constexpr float kLog2e = 1.44269504088896340736f;

template <typename T> __device__ inline float to_f(T v) { return (float)v; }
template <typename T> __device__ inline T from_f(float v) { return (T)v; }    // to nearest, ties to even

// VEC neighbouring elements of one row, moved as one access of VEC * sizeof(T) bytes (the caller checks the alignment)
template <typename T, int VEC> struct alignas(VEC * sizeof(T)) Pack { T v[VEC]; };

template <typename T, int VEC> __device__ inline void load_vec(const T* p, float (&out)[VEC]) {
    const Pack<T, VEC> r = *reinterpret_cast<const Pack<T, VEC>*>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) out[i] = to_f(r.v[i]);
}
template <typename T, int VEC> __device__ inline void store_vec(T* p, const float (&in)[VEC]) {
    Pack<T, VEC> r;
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.v[i] = from_f<T>(in[i]);
    *reinterpret_cast<Pack<T, VEC>*>(p) = r;
}

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }       // 1 ulp; below 2^-126: 0
__device__ inline float sigmoid_f(float x) { return __builtin_amdgcn_rcpf(1.0f + exp2_fast(-x * kLog2e)); }

// log(1 + e^x) = max(x, 0) + log1p(e^-|x|).  log1p(u) = 2 atanh(s), s = u / (2 + u) <= 1/3, as s P(s^2): an interpolation
// of 2 atanh(s) / s at the Chebyshev nodes of s^2 in [0, 1/9], 4e-9 relative.  (log(1 + u) itself would lose the small
// time steps: softplus(-7) = 9e-4 needs all 24 bits of u, of which 1 + u keeps 14.)  u has the rounding of its own argument,
// relative to it 4.4e-7 at |x| = 7 and 1.9e-6 at 40.
__device__ inline float softplus_f(float x) {
    const float u = exp2_fast(-__builtin_fabsf(x) * kLog2e);
    const float s = u * __builtin_amdgcn_rcpf(2.0f + u), z = s * s;
    float p = 0x1.2055eep-2f;
    p = __builtin_fmaf(p, z, 0x1.1e5cfcp-2f);
    p = __builtin_fmaf(p, z, 0x1.99da14p-2f);
    p = __builtin_fmaf(p, z, 0x1.5554e2p-1f);
    p = __builtin_fmaf(p, z, 2.0f);
    return __builtin_fmaf(s, p, __builtin_fmaxf(x, 0.0f));                 // (of a NaN, s is one)
}

template <typename F> int by_dtype(int dtype, const char* what, F&& f) {
    switch (dtype) {
        case VSV_F32: return f(float{});
        case VSV_BF16: return f(__bf16{});
        case VSV_F16: return f(_Float16{});
    }
    set_error("%s: dtype must be VSV_F32, VSV_BF16 or VSV_F16", what);
    return -1;
}

}  // namespace vsv
