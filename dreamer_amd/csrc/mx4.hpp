// Microscaled 4-bit matrices: rows of blocks of 32 elements.  A block is 16 bytes of e2m1 codes (element 2i in the low, 2i + 1 in
// the high half of byte i) and one scale byte s standing for 2^(s - 127); s = 255 makes the block NaN.  A matrix (rows, K) is
// codes (rows, nb, 16) and scales (rows, nb), nb = ceil(K / 32), both dense; codes behind column K are zero.
#pragma once
#include "elem.hpp"

namespace drm {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct Mx4 {
    const uint8_t* codes; const uint8_t* scales;
    int rows, nb;
};

// scale byte as the scale operand of the conversion instructions: they read its exponent field, 0 as 2^-127 and 255 as NaN
__device__ __forceinline__ float mx4_scale(uint32_t s) { return __builtin_bit_cast(float, s << 23); }

// eight codes of a block to bf16 (exact: at most two significant bits; below 2^-126 subnormal)
__device__ __forceinline__ bf16x8 mx4_bf16x8(uint32_t codes, float scale) {
    bf16x8 r;
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1),
                 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
    r[0] = a[0]; r[1] = a[1]; r[2] = b[0]; r[3] = b[1]; r[4] = c[0]; r[5] = c[1]; r[6] = d[0]; r[7] = d[1];
    return r;
}

// Eight elements of a float row as a sum of bf16 parts that is exact: bf16 one part, fp16 (11 bits) two, fp32 (24 bits) three.
// The parts are cut, not rounded, so that no part overflows; an infinity stays in the first part.
template <typename T> struct Parts;
template <> struct Parts<__bf16> { static constexpr int N = 1; };
template <> struct Parts<_Float16> { static constexpr int N = 2; };
template <> struct Parts<float> { static constexpr int N = 3; };

// eight elements as they lie in memory; 0 behind the row
template <typename T>
struct Eight { T v[8]; };
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Packed8 { Eight<T> e; };
template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T* __restrict__ row, int64_t at, int64_t len) {
    if (at + 8 <= len) return reinterpret_cast<const Packed8<T>*>(row + at)->e;
    Eight<T> r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = at + i < len ? row[at + i] : (T)0.f;
    return r;
}
template <typename T>
__device__ __forceinline__ void split_eight(const Eight<T>& e, bf16x8 (&p)[Parts<T>::N]) {
    if constexpr (Parts<T>::N == 1) {
        p[0] = __builtin_bit_cast(bf16x8, e);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float x = (float)e.v[i];
#pragma unroll
            for (int q = 0; q < Parts<T>::N; ++q) {
                const uint32_t u = __builtin_bit_cast(uint32_t, x);
                const float cut = __builtin_bit_cast(float, u & 0xffff0000u);
                p[q][i] = __builtin_bit_cast(__bf16, (uint16_t)(u >> 16));
                x = fabsf(x) == INFINITY ? 0.f : x - cut;
            }
        }
    }
}
template <typename T>
__device__ __forceinline__ void load_parts(const T* __restrict__ row, int64_t at, int64_t len, bf16x8 (&p)[Parts<T>::N]) {
    split_eight<T>(load_eight(row, at, len), p);
}

}  // namespace drm
