// What the operators of a user's right-hand side share (group norm: tode_norm.hip, cross attention: tode_attention*.hip): their
// element types and the vectors that they are loaded and stored in.
#pragma once
#include <hip/hip_runtime.h>

#include "tode_internal.h"

namespace tode {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// sums, statistics and everything between load and store: float32, for float64 data float64
template <typename T> struct Wide { typedef float type; };
template <> struct Wide<double> { typedef double type; };

// 16 bytes of T as they lie in memory.  The copy through __builtin_memcpy asks for no alignment beyond the element's own (rows of odd
// length): one global_load_dwordx4 either way.
template <typename T> struct alignas(16) Raw {
    static constexpr int N = 16 / sizeof(T);
    unsigned w[4];
    __device__ __forceinline__ void load(const T *p) { __builtin_memcpy(w, p, 16); }
    __device__ __forceinline__ void store(T *p) const { __builtin_memcpy(p, w, 16); }
    __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0; }
};

__device__ __forceinline__ void unpack(const Raw<float> &r, float *v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r.w[i]);
}
__device__ __forceinline__ void unpack(const Raw<double> &r, double *v) {
#pragma unroll
    for (int i = 0; i < 2; ++i) v[i] = __hiloint2double((int)r.w[2 * i + 1], (int)r.w[2 * i]);
}
__device__ __forceinline__ void unpack(const Raw<bf16> &r, float *v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(r.w[i] << 16), v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
}
__device__ __forceinline__ void unpack(const Raw<f16> &r, float *v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f16x2 h = __builtin_bit_cast(f16x2, r.w[i]);
        v[2 * i] = (float)h.x, v[2 * i + 1] = (float)h.y;
    }
}
__device__ __forceinline__ void pack(Raw<float> &r, const float *v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = __float_as_uint(v[i]);
}
__device__ __forceinline__ void pack(Raw<double> &r, const double *v) {
#pragma unroll
    for (int i = 0; i < 2; ++i) r.w[2 * i] = (unsigned)__double2loint(v[i]), r.w[2 * i + 1] = (unsigned)__double2hiint(v[i]);
}
__device__ __forceinline__ void pack(Raw<bf16> &r, const float *v) {  // (to the nearest, ties to even)
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{v[2 * i], v[2 * i + 1]}, bf16x2));
}
__device__ __forceinline__ void pack(Raw<f16> &r, const float *v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{v[2 * i], v[2 * i + 1]}, f16x2));
}

// A grid of n workgroups in a row, wrapped where it would pass 2^32 threads (the last line has workgroups beyond the n-th).
constexpr long long GRID_LINE = 1ll << 22;
inline dim3 grid_line(long long n) { return n <= GRID_LINE ? dim3((unsigned)n) : dim3((unsigned)GRID_LINE, (unsigned)((n + GRID_LINE - 1) / GRID_LINE)); }
__device__ __forceinline__ unsigned block_number() { return blockIdx.x + (unsigned)GRID_LINE * blockIdx.y; }

inline int bytes_of(int dtype) { return dtype == TODE_F64 ? 8 : dtype == TODE_F32 ? 4 : 2; }
inline bool known_field_dtype(int dtype) { return dtype == TODE_F32 || dtype == TODE_F64 || dtype == TODE_BF16 || dtype == TODE_F16; }

}  // namespace tode
