// Element types of the operators that take fp32, bf16 and fp16 tensors: 16-byte loads and stores that need only the
// element's own alignment (rows of odd length and views start anywhere), conversion to and from fp32.
#pragma once
#include "common.hpp"

namespace drm {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Elem;
template <> struct Elem<float> { static constexpr int VEC = 4; static constexpr int ID = DRM_F32; };
template <> struct Elem<__bf16> { static constexpr int VEC = 8; static constexpr int ID = DRM_BF16; };
template <> struct Elem<_Float16> { static constexpr int VEC = 8; static constexpr int ID = DRM_F16; };

static inline size_t elem_bytes(int dtype) { return dtype == DRM_F32 ? 4 : 2; }
static inline bool elem_ok(int dtype) { return dtype == DRM_F32 || dtype == DRM_BF16 || dtype == DRM_F16; }

// A launch takes fewer than 2^32 threads along an axis: the most workgroups of `threads` that one can have.  Kernels with a workgroup
// per row or tile are launched more than once beyond that (a second grid axis in the kernels costs them 3 to 5%).
static inline int64_t launch_limit(int threads) { return ((int64_t)1 << 32) / threads - 1; }

// one 16-byte slot of VEC elements, aligned like a single element (global memory takes dword accesses at any byte address)
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Slot { T v[Elem<T>::VEC]; };

// elements [at, at + VEC) of a row of `len` elements; what lies beyond the row reads as `fill` and is not touched
template <typename T>
__device__ __forceinline__ void load_slot(const T* __restrict__ row, int64_t at, int64_t len, float fill, float (&out)[Elem<T>::VEC]) {
    constexpr int VEC = Elem<T>::VEC;
    if (at + VEC <= len) {
        const Slot<T> s = *reinterpret_cast<const Slot<T>*>(row + at);
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = (float)s.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = at + i < len ? (float)row[at + i] : fill;
    }
}

template <typename T>
__device__ __forceinline__ void store_slot(T* __restrict__ row, int64_t at, int64_t len, const float (&v)[Elem<T>::VEC]) {
    constexpr int VEC = Elem<T>::VEC;
    if (at + VEC <= len) {
        Slot<T> s;
#pragma unroll
        for (int i = 0; i < VEC; ++i) s.v[i] = (T)v[i];   // nearest even
        *reinterpret_cast<Slot<T>*>(row + at) = s;
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (at + i < len) row[at + i] = (T)v[i];
    }
}

// Slot `at` of a row of `len` >= VEC elements without a branch: the slot is moved back into the row where it would leave it, so that
// every lane's load can be issued before the first one is waited for.  The elements of such a slot that belong to an earlier
// one (or all of them, behind the row) are not its own: owned(at, len, i) tells.
template <typename T>
__device__ __forceinline__ int64_t slot_at(int64_t at, int64_t len) { return at + Elem<T>::VEC <= len ? at : len - Elem<T>::VEC; }
template <typename T>
__device__ __forceinline__ bool owned(int64_t at, int64_t len, int i) { return slot_at<T>(at, len) + i >= at; }
template <typename T>
__device__ __forceinline__ Slot<T> raw_slot(const T* __restrict__ row, int64_t at, int64_t len) {
    return *reinterpret_cast<const Slot<T>*>(row + slot_at<T>(at, len));
}

// a vector of another type held beside the rows (weights, biases): element by runtime type
__device__ __forceinline__ float load_elem(const void* p, int dtype, int64_t i) {
    if (dtype == DRM_F32) return reinterpret_cast<const float*>(p)[i];
    if (dtype == DRM_BF16) return (float)reinterpret_cast<const __bf16*>(p)[i];
    return (float)reinterpret_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void store_elem(void* p, int dtype, int64_t i, float v) {
    if (dtype == DRM_F32) reinterpret_cast<float*>(p)[i] = v;
    else if (dtype == DRM_BF16) reinterpret_cast<__bf16*>(p)[i] = (__bf16)v;
    else reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
}

// f(T{}) for the element type `dtype` names (checked by the caller)
template <typename F>
static inline int with_elem(int dtype, F&& f) {
    if (dtype == DRM_F32) return f((float)0);
    if (dtype == DRM_BF16) return f((__bf16)0.f);
    return f((_Float16)0.f);
}

}  // namespace drm
