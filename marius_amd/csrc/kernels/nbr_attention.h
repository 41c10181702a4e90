// What the sweeps of the neighbour attention share (nbr_attention.hip says what they compute): a lane's part of a head, work items, joins of long lists, launches.
#pragma once
#include <type_traits>

#include "row_types.h"

namespace marius {

constexpr float NA_INF = __builtin_inff();
constexpr int NA_JOIN = 2;   // waves that join the parts of a long list, for one head (hubs back: all heads of a list in one workgroup of 8 waves 778 us, one head in 2 waves 759, 4 761, 8 787)
constexpr int NA_WAVES = 1;  // (waves of a workgroup: items differ in length, and a workgroup holds its registers until its longest wave ends: 4 waves 951 us, 2 852, 1 840 for the hubs of a power-law graph back)

struct NaArgs {
    const char *q, *k, *v, *go;
    int64_t q_hd, k_hd, v_hd, go_hd;                            // head strides, bytes
    uint32_t q_ld, k_ld, v_ld, go_ld;                           // row strides, bytes (an address is one multiply-add of 32 bits by 32 on 64)
    const float* bias;                                          // [T, H] or NULL
    float *out_bias, *stats, *lse, *part;                       // lse: [n, H] or NULL (m + log l of a list, for the caller; the sweeps use `stats`)
    float2* part2;                                              // a part's (m, sum), or its delta
    float4* rowstats;                                           // [n, H]: m, log l, delta of a target's list, for the sweep over the rows' lists
    void *out, *dk, *dv;                                        // contiguous [n, H, D], [rows, Hkv, D]
    const int32_t *index, *owner, *entry;                       // forward lists: index; reverse lists: owner, entry (position in the forward lists)
    const int4 *items, *splits;
    int n_items, n_splits, H, Hkv, D, hp;                       // hp: heads per slot
    bool dense;                                                 // items of more than two entries on average
    bool spread;                                                // sweep over the rows' lists: a lane group for each query head, not for each key head
    float scale;
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// A lane's part of a head's row, and what of it is the lane's own.  Elements that are a neighbour's are cleared where the row does not fill its lanes (`tail`, the
// same for a whole launch), in every row that is loaded: they add nothing to sums over the row and nothing is stored for them.
template <typename T, int VEC, int LPH>
struct Part {
    int at, first;
    bool tail;
    uint32_t mask[(sizeof(T) * VEC + 3) / 4];
    __device__ __forceinline__ Part(int l, int D) : tail(D != LPH * VEC) {
        const Place<VEC> p(l, D);
        at = p.at;
        first = p.first;
        constexpr int PER = sizeof(T) >= 4 ? 1 : 4 / (int)sizeof(T);  // elements of a word
#pragma unroll
        for (int i = 0; i < (int)(sizeof(mask) / 4); ++i) {
            mask[i] = 0;
#pragma unroll
            for (int e = 0; e < PER && i * PER + e < VEC; ++e) mask[i] |= i * PER + e >= first ? (PER == 1 ? ~0u : 0xffffu << (16 * e)) : 0u;
        }
    }
    __device__ __forceinline__ void leave_own(Piece<T, VEC>& p) const {
        if (!tail) return;
        uint32_t w[sizeof(mask) / 4] = {};
        __builtin_memcpy(w, p.t, sizeof(p.t));
#pragma unroll
        for (int i = 0; i < (int)(sizeof(mask) / 4); ++i) w[i] &= mask[i];
        __builtin_memcpy(p.t, w, sizeof(p.t));
    }
    template <typename O>
    __device__ __forceinline__ void store(O* p, const float (&v)[VEC]) const {
        if (!tail || first == 0) {
            put<O, VEC>(p + at, v);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (e >= first) p[at + e] = (O)v[e];
        }
    }
};
// a row that stays in registers for products with many others: bf16 as it is (a product of pairs is one instruction; products are exact, sums fp32), the others as fp32
template <typename T, int VEC>
struct Fixed {
    static constexpr bool PAIRS = std::is_same<T, __bf16>::value && VEC % 2 == 0;
    Piece<T, VEC> raw;
    float f[PAIRS ? 1 : VEC];
    __device__ __forceinline__ void set(const Piece<T, VEC>& p) {
        raw = p;
        if constexpr (!PAIRS) p.get(f);
    }
    __device__ __forceinline__ float dot(const Piece<T, VEC>& o) const {
        float s = 0.f;
        if constexpr (PAIRS) {
            bf16x2 a[VEC / 2], b[VEC / 2];
            __builtin_memcpy(a, raw.t, sizeof(a));
            __builtin_memcpy(b, o.t, sizeof(b));
#pragma unroll
            for (int e = 0; e < VEC / 2; ++e) s = __builtin_amdgcn_fdot2_f32_bf16(a[e], b[e], s, false);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) s += f[e] * (float)o.t[e];
        }
        return s;
    }
};
// weight of a running sum that goes from maximum m to `ref`; a maximum of -inf has weight zero
__device__ __forceinline__ float weight_to(float m, float ref) { return m == -NA_INF ? 0.f : __expf(m - ref); }
__device__ __forceinline__ float finite_ref(float m) { return m == -NA_INF ? 0.f : m; }
__device__ __forceinline__ const char* row_at(const char* base, int row, uint32_t ld) { return base + (uint64_t)(uint32_t)row * ld; }

// a launch's workgroups along x and z (a dimension holds less than 2^32 lanes)
inline dim3 na_grid(int64_t groups, int64_t y) {
    const int64_t x = groups < (1 << 22) ? groups : 1 << 22;
    return dim3((unsigned)x, (unsigned)y, (unsigned)cdiv(groups, x));
}
__device__ __forceinline__ uint32_t na_block() { return blockIdx.z * gridDim.x + blockIdx.x; }

// which item, head and piece a lane works on
template <int LPH>
struct Lane {
    int l, h;
    uint32_t slot;
    bool work;
    __device__ __forceinline__ Lane(const NaArgs& A, int heads) {
        const int lane = threadIdx.x & 63, g = lane / LPH, slots = 64 / (LPH * A.hp);
        l = lane & (LPH - 1);
        h = blockIdx.y * A.hp + (g & (A.hp - 1));
        slot = (na_block() * NA_WAVES + (threadIdx.x >> 6)) * slots + g / A.hp;
        work = h < heads && slot < (uint32_t)A.n_items;
    }
};
template <int UN>
__device__ __forceinline__ void load_numbers(const int32_t* p, int (&v)[UN]) { __builtin_memcpy(v, p, sizeof(v)); }  // (lists end with four spare entries)
// biases of UN entries from t on, for one head; behind the list -inf
template <int UN>
__device__ __forceinline__ void load_biases(const NaArgs& A, int t, int end, int h, float (&b)[UN]) {
#pragma unroll
    for (int u = 0; u < UN; ++u) b[u] = t + u < end ? A.bias[(uint64_t)(uint32_t)(t + u) * (uint32_t)A.H + h] : -NA_INF;
}

// a list's statistics, from its largest score and its sum
__device__ __forceinline__ void store_stats(const NaArgs& A, int64_t o, float m, float sum) {
    const float logl = sum == 0.f ? 0.f : logf(sum);
    A.stats[o * 2] = m;
    A.stats[o * 2 + 1] = logl;
    if (A.lse) A.lse[o] = m + logl;
}

// p from a score and its list's (m, log l); a list without a live entry has m = -inf.  (The hardware's exponential: two steps of fp32 and, from its rounded argument, |x| more;
// results are about 5 % further from 64 bits than with a correctly rounded one, and are rounded to the output's type anyhow.)
__device__ __forceinline__ float probability(float s, float m, float logl) { return __expf((s - finite_ref(m)) - logl); }

// The parts of a long list, one head a workgroup: lane group g of G takes parts g, g + G, ... in order, then the groups' results are added in a fixed order.
template <int LPH>
struct JoinLane {
    static constexpr int G = 64 * NA_JOIN / LPH;
    int l, g, wave, h;
    __device__ __forceinline__ JoinLane() : l(threadIdx.x & (LPH - 1)), g(threadIdx.x / LPH), wave(threadIdx.x >> 6), h(blockIdx.y) {}
};
// This for sums: two rows of D, and (`more`) a number of their own; true for the lanes that hold the result.
template <int VEC, int LPH>
__device__ __forceinline__ bool join_sums(const NaArgs& A, const JoinLane<LPH>& w, int heads, bool more, int at, float (&a)[VEC], float (&b)[VEC], float& first) {
    __shared__ float red[NA_JOIN][2 * VEC + 1][LPH];
    if (na_block() >= (uint32_t)A.n_splits) return false;
    const int4 sp = A.splits[na_block()];
    first = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) a[e] = b[e] = 0.f;
#pragma unroll 4
    for (int s = w.g; s < sp.z; s += w.G) {
        const int64_t o = (int64_t)(sp.y + s) * heads + w.h;
        float x[VEC], y[VEC];
        __builtin_memcpy(x, A.part + o * 2 * A.D + at, sizeof(x));
        __builtin_memcpy(y, A.part + o * 2 * A.D + A.D + at, sizeof(y));
        if (more) first += A.part2[o].x;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            a[e] += x[e];
            b[e] += y[e];
        }
    }
#pragma unroll
    for (int o = LPH; o < 64; o <<= 1) {
        first += __shfl_xor(first, o, 64);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            a[e] += __shfl_xor(a[e], o, 64);
            b[e] += __shfl_xor(b[e], o, 64);
        }
    }
    if ((threadIdx.x & 63) < LPH) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            red[w.wave][e][w.l] = a[e];
            red[w.wave][VEC + e][w.l] = b[e];
        }
        red[w.wave][2 * VEC][w.l] = first;
    }
    __syncthreads();
    if (w.g != 0) return false;
    for (int s = 1; s < NA_JOIN; ++s) {
        first += red[s][2 * VEC][w.l];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            a[e] += red[s][e][w.l];
            b[e] += red[s][VEC + e][w.l];
        }
    }
    return true;
}

// ---------------------------------------------------------------------------------------------------------------- launches
// One sweep is Pass::launch<T, VEC, LPH>(args, grid, block, stream).  Lanes per head: the power of two that covers its pieces of 16 bytes (heads shorter than
// one piece: an element per lane).
template <typename Pass, typename T, int VEC, int LPH>
static void na_launch(NaArgs A, int heads, hipStream_t st) {
    const int groups = 64 / LPH;
    // key heads that a power of two of query heads share: their lane groups work side by side where a slot holds them all, and are added at the end (a whole pass over
    // 1.5 M entries with 8 query and 4 key heads of 64: 957 us, one group after the other 990; over 300,000 with 8 and 4 of 32: 101 and 120; over 100,000 with 8 and 2 of 64: 92 and 89)
    const int share = A.H / A.Hkv;
    A.spread = Pass::ROWS && share > 1 && (share & (share - 1)) == 0 && share <= groups;
    const int lanes_heads = A.spread ? A.H : heads;
    A.hp = 1;
    while (A.hp < groups && A.hp < lanes_heads) A.hp <<= 1;
    Pass::template launch<T, VEC, LPH>(A, na_grid(cdiv(A.n_items, NA_WAVES * (groups / A.hp)), cdiv(lanes_heads, A.hp)), dim3(64 * NA_WAVES), st);
    if (A.n_splits > 0) Pass::template join<T, VEC, LPH>(A, na_grid(A.n_splits, heads), dim3(64 * NA_JOIN), st);
}
template <typename Pass, typename T>
static void na_launch_width(const NaArgs& A, int heads, hipStream_t st) {
    constexpr int VEC = 16 / (int)sizeof(T);
    const int pieces = (int)cdiv(A.D, VEC);
    if (A.D < VEC) na_launch<Pass, T, 1, VEC>(A, heads, st);
    else if (pieces <= 1) na_launch<Pass, T, VEC, 1>(A, heads, st);
    else if (pieces <= 2) na_launch<Pass, T, VEC, 2>(A, heads, st);
    else if (pieces <= 4) na_launch<Pass, T, VEC, 4>(A, heads, st);
    else if (pieces <= 8) na_launch<Pass, T, VEC, 8>(A, heads, st);
    else if (pieces <= 16) na_launch<Pass, T, VEC, 16>(A, heads, st);
    else if (pieces <= 32) na_launch<Pass, T, VEC, 32>(A, heads, st);
    else na_launch<Pass, T, VEC, VEC == 4 ? 64 : 32>(A, heads, st);  // (256 elements of 16 bits are 32 pieces)
}
template <typename Pass>
static void na_launch_typed(const NaArgs& A, int type, hipStream_t st) {
    if (A.n_items == 0) return;
    const int heads = Pass::ROWS ? A.Hkv : A.H;
    if (type == MARIUS_F32) na_launch_width<Pass, float>(A, heads, st);
    else if (type == MARIUS_BF16) na_launch_width<Pass, __bf16>(A, heads, st);
    else na_launch_width<Pass, _Float16>(A, heads, st);
}
// the sweeps of the backward pass, each in a file of its own
void nbr_attention_dq(const NaArgs& A, int type, hipStream_t st);
void nbr_attention_dkv(const NaArgs& A, int type, hipStream_t st);

}  // namespace marius
