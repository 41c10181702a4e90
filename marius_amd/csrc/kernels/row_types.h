// Rows held in fp32, bf16 or fp16 and computed on in fp32, whatever their length and alignment: pieces of a row per lane, sums over a row's lanes.
#pragma once
#include "common.h"

namespace marius {

// A lane's piece of a row: VEC consecutive elements, moved whole (the hardware takes such a load at any address of the element's alignment).
template <typename T, int VEC>
struct Piece {
    T t[VEC];
    __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(t, p, sizeof(t)); }
    __device__ __forceinline__ void get(float (&v)[VEC]) const {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = (float)t[e];
    }
};
// (rounds to nearest even: one rounding, at the store)
template <typename T, int VEC>
__device__ __forceinline__ void put(T* p, const float (&v)[VEC]) {
    T t[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) t[e] = (T)v[e];
    __builtin_memcpy(p, t, sizeof(t));
}
// Where piece number `unit` of a row of `d` elements lies (d >= VEC).  A row that is no multiple of VEC ends with a piece that ends with the row and overlaps
// its neighbour's; lanes behind the row repeat the last piece.  `first` is the first element that is the piece's own (VEC: none).
template <int VEC>
struct Place {
    int at, first;
    __device__ __forceinline__ Place(int unit, int d) : at(unit * VEC < d - VEC ? unit * VEC : d - VEC) {
        first = unit * VEC - at;
        first = first > VEC ? VEC : first;
    }
};

// Sums over groups of lanes, the same bits on all of them: neighbours within a row of 16 lanes by data-parallel moves, rows of 16 and halves of the
// wave by lane swaps: nothing goes through LDS.
__device__ __forceinline__ int bits_of(float v) {
    int w;
    __builtin_memcpy(&w, &v, 4);
    return w;
}
__device__ __forceinline__ float float_of(int w) {
    float v;
    __builtin_memcpy(&v, &w, 4);
    return v;
}
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) { return v + float_of(__builtin_amdgcn_update_dpp(0, bits_of(v), CTRL, 0xf, 0xf, true)); }
template <int LANES>  // adds the other half of a group of LANES lanes, whose halves hold one value each
__device__ __forceinline__ float add_half(float v) {
    if (LANES == 2) return dpp_add<0xB1>(v);    // lane ^ 1
    if (LANES == 4) return dpp_add<0x4E>(v);    // lane ^ 2
    if (LANES == 8) return dpp_add<0x141>(v);   // mirrored in 8
    if (LANES == 16) return dpp_add<0x140>(v);  // mirrored in 16
    const auto r = LANES == 32 ? __builtin_amdgcn_permlane16_swap(bits_of(v), bits_of(v), false, false) : __builtin_amdgcn_permlane32_swap(bits_of(v), bits_of(v), false, false);
    return float_of(r[0]) + float_of(r[1]);
}
template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
    if (LANES >= 2) v = add_half<2>(v);
    if (LANES >= 4) v = add_half<4>(v);
    if (LANES >= 8) v = add_half<8>(v);
    if (LANES >= 16) v = add_half<16>(v);
    if (LANES >= 32) v = add_half<32>(v);
    if (LANES >= 64) v = add_half<64>(v);
    return v;
}

// a piece of a row whose type is known at run time only (parameters: read once per workgroup)
template <int VEC>
__device__ __forceinline__ void piece_any(const void* row, int type, int at, float (&v)[VEC]) {
    if (type == MARIUS_F32) {
        Piece<float, VEC> p;
        p.load((const float*)row + at);
        p.get(v);
    } else if (type == MARIUS_BF16) {
        Piece<__bf16, VEC> p;
        p.load((const __bf16*)row + at);
        p.get(v);
    } else {
        Piece<_Float16, VEC> p;
        p.load((const _Float16*)row + at);
        p.get(v);
    }
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
