// Rows held in fp32, bf16 or fp16 and computed on in fp32: 16-byte pieces per lane, whatever the row's length and alignment.
#pragma once
#include "common.h"

namespace marius {

// A lane owns pieces of VEC consecutive elements: 16 bytes of the 16-bit types, 16 bytes of fp32.  A piece that ends behind the row is moved element by
// element (one lane of a row at most); a whole piece is one load of 16 bytes, which the hardware takes at any address of the element's alignment.
template <typename T, int VEC>
__device__ __forceinline__ void piece_load(const T* __restrict__ row, int c, int d, float (&v)[VEC]) {
    if (c + VEC <= d) {
        T t[VEC];
        __builtin_memcpy(t, row + c, sizeof(t));
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = (float)t[e];
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = c + e < d ? (float)row[c + e] : 0.f;
    }
}
// (rounds to nearest even: one rounding, at the store)
template <typename T, int VEC>
__device__ __forceinline__ void piece_store(T* __restrict__ row, int c, int d, const float (&v)[VEC]) {
    if (c + VEC <= d) {
        T t[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) t[e] = (T)v[e];
        __builtin_memcpy(row + c, t, sizeof(t));
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (c + e < d) row[c + e] = (T)v[e];
    }
}
// the same from a base whose type is known at run time only (parameters: read once per workgroup)
template <int VEC>
__device__ __forceinline__ void piece_load_any(const void* row, int type, int c, int d, float (&v)[VEC]) {
    if (type == MARIUS_F32) piece_load<float, VEC>((const float*)row, c, d, v);
    else if (type == MARIUS_BF16) piece_load<__bf16, VEC>((const __bf16*)row, c, d, v);
    else piece_load<_Float16, VEC>((const _Float16*)row, c, d, v);
}
__device__ __forceinline__ float element_any(const void* p, int type, int64_t i) {
    return type == MARIUS_F32 ? ((const float*)p)[i] : type == MARIUS_BF16 ? (float)((const __bf16*)p)[i] : (float)((const _Float16*)p)[i];
}
__device__ __forceinline__ void element_store_any(void* p, int type, int64_t i, float v) {
    if (type == MARIUS_F32) ((float*)p)[i] = v;
    else if (type == MARIUS_BF16) ((__bf16*)p)[i] = (__bf16)v;
    else ((_Float16*)p)[i] = (_Float16)v;
}

inline bool float_type_ok(int t) { return t == MARIUS_F32 || t == MARIUS_BF16 || t == MARIUS_F16; }

}  // namespace marius
