// Attention of target nodes over their neighbour lists (marius_neighbor_plan), forward and backward.
//
//     s_e = scale q_i . k_j + b_e          entry e = (target i <- row j), per query head; query head h reads key head h / (H / Hkv)
//     p_e = exp(s_e - m_i - log l_i)       m_i: largest score of i's list, l_i: sum of exp(s_e - m_i)
//     o_i = sum_e p_e v_j                  an entry whose bias is -inf is masked: neither its key nor its value enters; an empty list gives o = 0, m = -inf
//
// Backward, probabilities recomputed from (m, log l):
//     d_e = do_i . v_j,  delta_i = sum_e p_e d_e,  g_e = p_e (d_e - delta_i)
//     dq_i = scale (sum_e p_e d_e k_j - delta_i sum_e p_e k_j)      one sweep over the list gives both sums and delta: o is neither kept nor read
//     dk_j = scale sum g_e q_i,  dv_j = sum p_e do_i,  db_e = g_e    over j's reverse list and the query heads that share j's key: no atomics, fixed order
//
// (m, log l) are kept apart because their sum can lose log l: a list whose entries all carry the type's lowest value as bias has m = -3.4e38.
//
// A work item is a list, or a part of a long one.  A head's row is spread over LPH lanes, 16 bytes each; hp heads (the power of two that covers them, or
// what a wave holds) make a slot, and every slot of a wave walks an item of its own: most lists have a handful of entries, and what bounds
// them is how many dependent loads (item -> row number -> row) are in flight.  UN entries are loaded at a time, the next ones' numbers while these are
// computed.  Parts of a long list are written as partial results and joined by a second launch in order.
// Bound by the gather of rows: 2 rows per entry in each of the three sweeps.
#include <type_traits>

#include "row_types.h"

namespace marius {

constexpr float NA_INF = __builtin_inff();
constexpr int NA_WAVES = 1;  // (waves of a workgroup: items differ in length, and a workgroup holds its registers until its longest wave ends: 4 waves 951 us, 2 852, 1 840 for the hubs of a power-law graph back)

struct NaArgs {
    const char *q, *k, *v, *go;
    int64_t q_hd, k_hd, v_hd, go_hd;                            // head strides, bytes
    uint32_t q_ld, k_ld, v_ld, go_ld;                           // row strides, bytes (an address is one multiply-add of 32 bits by 32 on 64)
    const float* bias;                                          // [T, H] or NULL
    float *out_bias, *stats, *part;
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

// which item, head and piece a lane works on
template <int LPH>
struct Lane {
    int l, h, slot;
    bool head;
    __device__ __forceinline__ Lane(const NaArgs& A, int heads) {
        const int lane = threadIdx.x & 63, g = lane / LPH, slots = 64 / (LPH * A.hp);
        l = lane & (LPH - 1);
        h = blockIdx.y * A.hp + (g & (A.hp - 1));
        head = h < heads;
        h = head ? h : heads - 1;
        slot = (blockIdx.x * NA_WAVES + (threadIdx.x >> 6)) * slots + g / A.hp;
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

// ---------------------------------------------------------------------------------------------------------------- forward
template <typename T, int VEC, int LPH, bool BIAS>
__global__ __launch_bounds__(64 * NA_WAVES) void nbr_attention_kernel(NaArgs A) {
    constexpr int UN = 4;
    const Lane<LPH> w(A, A.H);
    if (w.slot >= A.n_items || !w.head) return;
    const int4 it = A.items[w.slot];
    const Part<T, VEC, LPH> part(w.l, A.D);
    const int kv = w.h / (A.H / A.Hkv);
    float acc[VEC], m = -NA_INF, sum = 0.f, bias[UN];
    Piece<T, VEC> raw;
    Fixed<T, VEC> q;
    raw.load((const T*)(row_at(A.q, it.x, A.q_ld) + w.h * A.q_hd) + part.at);
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    const char *kp = A.k + kv * A.k_hd + part.at * sizeof(T), *vp = A.v + kv * A.v_hd + part.at * sizeof(T);
    int next[UN];
    load_numbers<UN>(A.index + it.y, next);
    if (BIAS) load_biases<UN>(A, it.y, it.z, w.h, bias);
    part.leave_own(raw);
    q.set(raw);
    for (int t = it.y; t < it.z; t += UN) {
        Piece<T, VEC> kk[UN], vv[UN];
        float s[UN];
        bool ok[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            ok[u] = t + u < it.z;
            const int j = ok[u] ? next[u] : next[0];  // (behind the list: its last rows once more, computed on by nobody)
            kk[u].load((const T*)row_at(kp, j, A.k_ld));
            vv[u].load((const T*)row_at(vp, j, A.v_ld));
            s[u] = 0.f;
            if (BIAS) {
                s[u] = bias[u];
                ok[u] = bias[u] != -NA_INF;
            }
        }
        if (t + UN < it.z) {
            load_numbers<UN>(A.index + t + UN, next);
            if (BIAS) load_biases<UN>(A, t + UN, it.z, w.h, bias);
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            part.leave_own(kk[u]);
            const float d = group_sum<LPH>(q.dot(kk[u])) * A.scale;
            s[u] = ok[u] ? d + s[u] : -NA_INF;
            top = fmaxf(top, s[u]);
        }
        const float ref = finite_ref(top), scale = weight_to(m, ref);
        m = top;
        sum *= scale;
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] *= scale;
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            if (!ok[u]) continue;
            const float p = __expf(s[u] - ref);
            sum += p;
            part.leave_own(vv[u]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += p * (float)vv[u].t[e];
        }
    }
    if (it.w >= 0) {
        const int64_t o = (int64_t)it.w * A.H + w.h;
        part.store(A.part + o * A.D, acc);
        if (w.l == 0) A.part2[o] = make_float2(m, sum);
    } else {
        const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;  // (NaN stays)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] *= inv;
        const int64_t o = (int64_t)it.x * A.H + w.h;
        part.store((T*)A.out + o * A.D, acc);
        if (w.l == 0) {
            A.stats[o * 2] = m;
            A.stats[o * 2 + 1] = sum == 0.f ? 0.f : logf(sum);
        }
    }
}

// The parts of a long list: wave w takes parts w, w + NA_JOIN, ... in order, then the waves' results are joined in order.
constexpr int NA_JOIN = 8;
template <typename T, int VEC, int LPH>
__global__ __launch_bounds__(64 * NA_JOIN) void nbr_attention_join_kernel(NaArgs A) {
    __shared__ float red[NA_JOIN][VEC + 2][64];
    const int4 sp = A.splits[blockIdx.x];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = blockIdx.y * (64 / LPH) + lane / LPH, hc = h < A.H ? h : A.H - 1;
    const Part<T, VEC, LPH> part(lane & (LPH - 1), A.D);
    float acc[VEC], m = -NA_INF, sum = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    auto join = [&](float om, float os, const float(&v)[VEC]) {
        const float top = fmaxf(m, om), ref = finite_ref(top), w = weight_to(m, ref), ow = weight_to(om, ref);
        sum = sum * w + os * ow;
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] = acc[e] * w + v[e] * ow;
        m = top;
    };
#pragma unroll 4
    for (int s = wave; s < sp.z; s += NA_JOIN) {
        const int64_t o = (int64_t)(sp.y + s) * A.H + hc;
        float v[VEC];
        __builtin_memcpy(v, A.part + o * A.D + part.at, sizeof(v));
        const float2 ms = A.part2[o];
        join(ms.x, ms.y, v);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) red[wave][e][lane] = acc[e];
    red[wave][VEC][lane] = m;
    red[wave][VEC + 1][lane] = sum;
    __syncthreads();
    if (wave != 0 || h >= A.H) return;
    for (int s = 1; s < NA_JOIN; ++s) {
        float v[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = red[s][e][lane];
        join(red[s][VEC][lane], red[s][VEC + 1][lane], v);
    }
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] *= inv;
    const int64_t o = (int64_t)sp.x * A.H + h;
    part.store((T*)A.out + o * A.D, acc);
    if ((lane & (LPH - 1)) == 0) {
        A.stats[o * 2] = m;
        A.stats[o * 2 + 1] = sum == 0.f ? 0.f : logf(sum);
    }
}
// the same for sums: two rows of D, and (`more`) a number of their own; true for the lanes that hold the result
template <int VEC>
__device__ __forceinline__ bool join_sums(const NaArgs& A, int heads, bool more, int at, int h, float (&a)[VEC], float (&b)[VEC], float& first) {
    __shared__ float red[NA_JOIN][2 * VEC + 1][64];
    const int4 sp = A.splits[blockIdx.x];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hc = h < heads ? h : heads - 1;
    first = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) a[e] = b[e] = 0.f;
#pragma unroll 4
    for (int s = wave; s < sp.z; s += NA_JOIN) {
        const int64_t o = (int64_t)(sp.y + s) * heads + hc;
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
    for (int e = 0; e < VEC; ++e) {
        red[wave][e][lane] = a[e];
        red[wave][VEC + e][lane] = b[e];
    }
    red[wave][2 * VEC][lane] = first;
    __syncthreads();
    if (wave != 0 || h >= heads) return false;
    for (int s = 1; s < NA_JOIN; ++s) {
        first += red[s][2 * VEC][lane];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            a[e] += red[s][e][lane];
            b[e] += red[s][VEC + e][lane];
        }
    }
    return true;
}

// p from a score and its list's (m, log l); a list without a live entry has m = -inf
__device__ __forceinline__ float probability(float s, float m, float logl) { return __expf((s - finite_ref(m)) - logl); }

// dq = scale (sum p d k - delta sum p k): two roundings, not a fused one, so that a list of one entry gives exactly zero
template <int VEC>
__device__ __forceinline__ void dq_of(float (&pdk)[VEC], const float (&pk)[VEC], float delta, float scale) {
#pragma clang fp contract(off)
#pragma unroll
    for (int e = 0; e < VEC; ++e) pdk[e] = scale * (pdk[e] - delta * pk[e]);
}

// ---------------------------------------------------------------------------------------------------------------- backward over the targets' lists: dq, delta
template <typename T, int VEC, int LPH, bool BIAS>
__global__ __launch_bounds__(64 * NA_WAVES) void nbr_attention_dq_kernel(NaArgs A) {
    constexpr int UN = 4;
    const Lane<LPH> w(A, A.H);
    if (w.slot >= A.n_items || !w.head) return;
    const int4 it = A.items[w.slot];
    const Part<T, VEC, LPH> part(w.l, A.D);
    const int kv = w.h / (A.H / A.Hkv);
    const int64_t o = (int64_t)it.x * A.H + w.h;
    float pdk[VEC], pk[VEC], delta = 0.f, bias[UN];
    Piece<T, VEC> raw, raw2;
    Fixed<T, VEC> q, go;
    raw.load((const T*)(row_at(A.q, it.x, A.q_ld) + w.h * A.q_hd) + part.at);
    raw2.load((const T*)(row_at(A.go, it.x, A.go_ld) + w.h * A.go_hd) + part.at);
    const float m = A.stats[o * 2], logl = A.stats[o * 2 + 1];
#pragma unroll
    for (int e = 0; e < VEC; ++e) pdk[e] = pk[e] = 0.f;
    const char *kp = A.k + kv * A.k_hd + part.at * sizeof(T), *vp = A.v + kv * A.v_hd + part.at * sizeof(T);
    int next[UN];
    load_numbers<UN>(A.index + it.y, next);
    if (BIAS) load_biases<UN>(A, it.y, it.z, w.h, bias);
    part.leave_own(raw);
    part.leave_own(raw2);
    q.set(raw);
    go.set(raw2);
    for (int t = it.y; t < it.z; t += UN) {
        Piece<T, VEC> kk[UN], vv[UN];
        float b[UN];
        bool ok[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            ok[u] = t + u < it.z;
            const int j = ok[u] ? next[u] : next[0];
            kk[u].load((const T*)row_at(kp, j, A.k_ld));
            vv[u].load((const T*)row_at(vp, j, A.v_ld));
            b[u] = 0.f;
            if (BIAS) {
                b[u] = bias[u];
                ok[u] = bias[u] != -NA_INF;
            }
        }
        if (t + UN < it.z) {
            load_numbers<UN>(A.index + t + UN, next);
            if (BIAS) load_biases<UN>(A, t + UN, it.z, w.h, bias);
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            if (!ok[u]) continue;
            part.leave_own(kk[u]);
            part.leave_own(vv[u]);
            const float s = group_sum<LPH>(q.dot(kk[u])) * A.scale + b[u], d = group_sum<LPH>(go.dot(vv[u]));
            const float p = probability(s, m, logl), pd = p * d;
            delta += pd;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float k = (float)kk[u].t[e];
                pdk[e] += pd * k;
                pk[e] += p * k;
            }
        }
    }
    if (it.w >= 0) {
        const int64_t p = (int64_t)it.w * A.H + w.h;
        part.store(A.part + p * 2 * A.D, pdk);
        part.store(A.part + p * 2 * A.D + A.D, pk);
        if (w.l == 0) A.part2[p] = make_float2(delta, 0.f);
    } else {
        dq_of<VEC>(pdk, pk, delta, A.scale);
        part.store((T*)A.out + o * A.D, pdk);
        if (w.l == 0) A.rowstats[o] = make_float4(m, logl, delta, 0.f);
    }
}
template <typename T, int VEC, int LPH>
__global__ __launch_bounds__(64 * NA_JOIN) void nbr_attention_dq_join_kernel(NaArgs A) {
    const int lane = threadIdx.x & 63, h = blockIdx.y * (64 / LPH) + lane / LPH;
    const Part<T, VEC, LPH> part(lane & (LPH - 1), A.D);
    float pdk[VEC], pk[VEC], delta;
    if (!join_sums<VEC>(A, A.H, true, part.at, h, pdk, pk, delta)) return;
    dq_of<VEC>(pdk, pk, delta, A.scale);
    const int64_t o = (int64_t)A.splits[blockIdx.x].x * A.H + h;
    part.store((T*)A.out + o * A.D, pdk);
    if ((lane & (LPH - 1)) == 0) A.rowstats[o] = make_float4(A.stats[o * 2], A.stats[o * 2 + 1], delta, 0.f);
}

// ---------------------------------------------------------------------------------------------------------------- backward over the rows' lists: dk, dv, db
// UN entries at a time: four where items are long enough to fill them, two where most rows are in a list or two
template <typename T, int VEC, int LPH, bool BIAS, int UN>
__global__ __launch_bounds__(64 * NA_WAVES) void nbr_attention_dkv_kernel(NaArgs A) {
    const Lane<LPH> w(A, A.spread ? A.H : A.Hkv);
    if (w.slot >= A.n_items || !w.head) return;
    const int4 it = A.items[w.slot];
    const Part<T, VEC, LPH> part(w.l, A.D);
    const int share = A.H / A.Hkv, R = A.spread ? 1 : share, kv = A.spread ? w.h / share : w.h;
    float dk[VEC], dv[VEC];
    Piece<T, VEC> raw, raw2;
    Fixed<T, VEC> k, v;
    raw.load((const T*)(row_at(A.k, it.x, A.k_ld) + kv * A.k_hd) + part.at);
    raw2.load((const T*)(row_at(A.v, it.x, A.v_ld) + kv * A.v_hd) + part.at);
    int next[UN], next_e[UN];
    load_numbers<UN>(A.owner + it.y, next);
    if (BIAS) load_numbers<UN>(A.entry + it.y, next_e);
    part.leave_own(raw);
    part.leave_own(raw2);
    k.set(raw);
    v.set(raw2);
#pragma unroll
    for (int e = 0; e < VEC; ++e) dk[e] = dv[e] = 0.f;
    for (int t = it.y; t < it.z; t += UN) {
        int i[UN], e_at[UN];
        bool in[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            in[u] = t + u < it.z;
            i[u] = in[u] ? next[u] : next[0];
            e_at[u] = BIAS ? (in[u] ? next_e[u] : next_e[0]) : 0;
        }
        if (t + UN < it.z) {
            load_numbers<UN>(A.owner + t + UN, next);
            if (BIAS) load_numbers<UN>(A.entry + t + UN, next_e);
        }
        for (int r = 0; r < R; ++r) {
            const int h = w.h * R + r;
            const char *qp = A.q + h * A.q_hd + part.at * sizeof(T), *gp = A.go + h * A.go_hd + part.at * sizeof(T);
            Piece<T, VEC> qq[UN], gg[UN];
            float4 st[UN];
            float bias[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                st[u] = *(const float4*)row_at((const char*)(A.rowstats + h), i[u], (uint32_t)A.H * sizeof(float4));
                bias[u] = BIAS ? *(const float*)row_at((const char*)(A.bias + h), e_at[u], (uint32_t)A.H * sizeof(float)) : 0.f;
                qq[u].load((const T*)row_at(qp, i[u], A.q_ld));
                gg[u].load((const T*)row_at(gp, i[u], A.go_ld));
            }
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                if (!in[u]) continue;
                part.leave_own(qq[u]);
                part.leave_own(gg[u]);
                const bool live = !BIAS || bias[u] != -NA_INF;
                const float s = group_sum<LPH>(k.dot(qq[u])) * A.scale + bias[u], d = group_sum<LPH>(v.dot(gg[u]));
                const float p = live ? probability(s, st[u].x, st[u].y) : 0.f, ds = live ? p * (d - st[u].z) : 0.f;
                if (BIAS && A.out_bias && w.l == 0) *(float*)row_at((const char*)(A.out_bias + h), e_at[u], (uint32_t)A.H * sizeof(float)) = ds;
                if (!live) continue;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    dk[e] += ds * (float)qq[u].t[e];
                    dv[e] += p * (float)gg[u].t[e];
                }
            }
        }
    }
    if (A.spread) {  // the lanes of the query heads that share this key head
        for (int o = LPH; o < LPH * share; o <<= 1)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                dk[e] += __shfl_xor(dk[e], o, 64);
                dv[e] += __shfl_xor(dv[e], o, 64);
            }
        if (w.h & (share - 1)) return;
    }
    if (it.w >= 0) {
        const int64_t p = (int64_t)it.w * A.Hkv + kv;
        part.store(A.part + p * 2 * A.D, dk);
        part.store(A.part + p * 2 * A.D + A.D, dv);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) dk[e] *= A.scale;
        const int64_t o = ((int64_t)it.x * A.Hkv + kv) * A.D;
        part.store((T*)A.dk + o, dk);
        part.store((T*)A.dv + o, dv);
    }
}
template <typename T, int VEC, int LPH>
__global__ __launch_bounds__(64 * NA_JOIN) void nbr_attention_dkv_join_kernel(NaArgs A) {
    const int lane = threadIdx.x & 63, h = blockIdx.y * (64 / LPH) + lane / LPH;
    const Part<T, VEC, LPH> part(lane & (LPH - 1), A.D);
    float dk[VEC], dv[VEC], none;
    if (!join_sums<VEC>(A, A.Hkv, false, part.at, h, dk, dv, none)) return;
#pragma unroll
    for (int e = 0; e < VEC; ++e) dk[e] *= A.scale;
    const int64_t o = ((int64_t)A.splits[blockIdx.x].x * A.Hkv + h) * A.D;
    part.store((T*)A.dk + o, dk);
    part.store((T*)A.dv + o, dv);
}

// ---------------------------------------------------------------------------------------------------------------- launches
enum NaPass { NA_FWD = 0, NA_DQ, NA_DKV };

template <typename T, int VEC, int LPH>
static void na_launch(NaArgs A, NaPass pass, hipStream_t st) {
    const int groups = 64 / LPH, share = A.H / A.Hkv;
    // key heads that a power of two of query heads share: their lane groups work side by side where a slot holds them all, and are added at the end
    A.spread = pass == NA_DKV && share > 1 && (share & (share - 1)) == 0 && share <= groups;
    const int heads = pass == NA_DKV && !A.spread ? A.Hkv : A.H;
    A.hp = 1;
    while (A.hp < groups && A.hp < heads) A.hp <<= 1;
    const dim3 grid((unsigned)cdiv(A.n_items, NA_WAVES * (groups / A.hp)), (unsigned)cdiv(heads, A.hp)), jgrid((unsigned)A.n_splits, (unsigned)cdiv(pass == NA_DKV ? A.Hkv : A.H, groups));
    const dim3 block(64 * NA_WAVES);
    if (pass == NA_FWD) {
        if (A.bias) nbr_attention_kernel<T, VEC, LPH, true><<<grid, block, 0, st>>>(A);
        else nbr_attention_kernel<T, VEC, LPH, false><<<grid, block, 0, st>>>(A);
        if (A.n_splits > 0) nbr_attention_join_kernel<T, VEC, LPH><<<jgrid, dim3(64 * NA_JOIN), 0, st>>>(A);
    } else if (pass == NA_DQ) {
        if (A.bias) nbr_attention_dq_kernel<T, VEC, LPH, true><<<grid, block, 0, st>>>(A);
        else nbr_attention_dq_kernel<T, VEC, LPH, false><<<grid, block, 0, st>>>(A);
        if (A.n_splits > 0) nbr_attention_dq_join_kernel<T, VEC, LPH><<<jgrid, dim3(64 * NA_JOIN), 0, st>>>(A);
    } else {
        if (A.bias && A.dense) nbr_attention_dkv_kernel<T, VEC, LPH, true, 4><<<grid, block, 0, st>>>(A);
        else if (A.bias) nbr_attention_dkv_kernel<T, VEC, LPH, true, 2><<<grid, block, 0, st>>>(A);
        else if (A.dense) nbr_attention_dkv_kernel<T, VEC, LPH, false, 4><<<grid, block, 0, st>>>(A);
        else nbr_attention_dkv_kernel<T, VEC, LPH, false, 2><<<grid, block, 0, st>>>(A);
        if (A.n_splits > 0) nbr_attention_dkv_join_kernel<T, VEC, LPH><<<jgrid, dim3(64 * NA_JOIN), 0, st>>>(A);
    }
}
// lanes per head: the power of two that covers its pieces of 16 bytes (heads shorter than one piece: an element per lane)
template <typename T>
static void na_launch_width(const NaArgs& A, NaPass pass, hipStream_t st) {
    constexpr int VEC = 16 / (int)sizeof(T);
    const int pieces = (int)cdiv(A.D, VEC);
    if (A.D < VEC) na_launch<T, 1, VEC>(A, pass, st);
    else if (pieces <= 1) na_launch<T, VEC, 1>(A, pass, st);
    else if (pieces <= 2) na_launch<T, VEC, 2>(A, pass, st);
    else if (pieces <= 4) na_launch<T, VEC, 4>(A, pass, st);
    else if (pieces <= 8) na_launch<T, VEC, 8>(A, pass, st);
    else if (pieces <= 16) na_launch<T, VEC, 16>(A, pass, st);
    else if (pieces <= 32) na_launch<T, VEC, 32>(A, pass, st);
    else na_launch<T, VEC, VEC == 4 ? 64 : 32>(A, pass, st);  // (256 elements of 16 bits are 32 pieces)
}
static void na_launch_typed(const NaArgs& A, int type, NaPass pass, hipStream_t st) {
    if (A.n_items == 0) return;
    if (type == MARIUS_F32) na_launch_width<float>(A, pass, st);
    else if (type == MARIUS_BF16) na_launch_width<__bf16>(A, pass, st);
    else na_launch_width<_Float16>(A, pass, st);
}

// the workspace: (backward: row statistics,) the parts' small numbers, the parts' rows, each at a multiple of 16 bytes
static size_t na_small_bytes(const marius_neighbor_plan* P, int heads) { return ((size_t)P->n_slots * heads * sizeof(float2) + 15) & ~(size_t)15; }

static int na_args(const marius_neighbor_plan* P, const marius_neighbor_attention* m, const char* what, NaArgs& A) {
    MARIUS_REQUIRE(P && m, "%s: null descriptor", what);
    MARIUS_REQUIRE(P->n >= 0 && P->rows >= 0 && P->T >= 0 && P->n_items >= 0 && P->n_splits >= 0 && P->r_n_items >= 0 && P->r_n_splits >= 0, "%s: bad plan", what);
    MARIUS_REQUIRE(float_type_ok(m->type), "%s: types are MARIUS_F32 / BF16 / F16", what);
    MARIUS_REQUIRE(m->heads > 0 && m->kv_heads > 0 && m->heads % m->kv_heads == 0 && m->heads <= 1024, "%s: query heads (up to 1024) are a multiple of the key heads", what);
    MARIUS_REQUIRE(m->dim > 0 && m->dim <= 256, "%s: heads of 1 to 256 elements", what);
    MARIUS_REQUIRE(P->n == 0 || (m->q && P->items), "%s: null pointer", what);
    MARIUS_REQUIRE(P->T == 0 || (m->k && m->v && P->index), "%s: null pointer", what);
    const int64_t size = m->type == MARIUS_F32 ? 4 : 2;
    for (int64_t row : {m->q_row, m->k_row, m->v_row})
        MARIUS_REQUIRE(row >= 0 && row * size < (1ll << 32), "%s: rows are at most 4 GiB apart", what);
    A = NaArgs{};
    A.q = (const char*)m->q;
    A.k = (const char*)m->k;
    A.v = (const char*)m->v;
    A.q_ld = (uint32_t)(m->q_row * size);
    A.q_hd = m->q_head * size;
    A.k_ld = (uint32_t)(m->k_row * size);
    A.k_hd = m->k_head * size;
    A.v_ld = (uint32_t)(m->v_row * size);
    A.v_hd = m->v_head * size;
    A.bias = m->bias;
    A.stats = m->stats;
    A.H = m->heads;
    A.Hkv = m->kv_heads;
    A.D = m->dim;
    A.scale = m->scale;
    A.index = P->index;
    A.items = (const int4*)P->items;
    A.splits = (const int4*)P->splits;
    A.n_items = P->n_items;
    A.n_splits = P->n_splits;
    return MARIUS_OK;
}

}  // namespace marius

using namespace marius;

extern "C" size_t marius_neighbor_attention_workspace_bytes(const marius_neighbor_plan* P, int32_t heads, int32_t kv_heads, int32_t dim, int32_t backward) {
    if (!P || heads <= 0 || kv_heads <= 0 || dim <= 0) return 0;
    const size_t small = na_small_bytes(P, heads);
    if (!backward) return small + (size_t)P->n_slots * heads * dim * sizeof(float);
    const size_t dq = (size_t)P->n_slots * heads * 2 * dim, dkv = (size_t)P->r_n_slots * kv_heads * 2 * dim;
    return (size_t)P->n * heads * sizeof(float4) + small + (dq > dkv ? dq : dkv) * sizeof(float);
}

extern "C" int marius_neighbor_attention_forward(const marius_neighbor_plan* P, const marius_neighbor_attention* m, void* out, void* workspace, size_t workspace_bytes,
                                                 marius_stream_t stream) {
    NaArgs A;
    const int rc = na_args(P, m, "neighbor_attention_forward", A);
    if (rc) return rc;
    if (P->n == 0) return MARIUS_OK;
    MARIUS_REQUIRE(out && m->stats, "neighbor_attention_forward: null output");
    MARIUS_REQUIRE(P->n_slots == 0 || (workspace && P->splits && workspace_bytes >= marius_neighbor_attention_workspace_bytes(P, m->heads, m->kv_heads, m->dim, 0)),
                   "neighbor_attention_forward: workspace too small");
    A.out = out;
    A.part2 = (float2*)workspace;
    A.part = (float*)((char*)workspace + na_small_bytes(P, A.H));
    na_launch_typed(A, m->type, NA_FWD, as_stream(stream));
    return check_launch("neighbor_attention_forward");
}

extern "C" int marius_neighbor_attention_backward(const marius_neighbor_plan* P, const marius_neighbor_attention* m, const void* grad_out, int64_t grad_row, int64_t grad_head,
                                                  void* dq, void* dk, void* dv, float* dbias, void* workspace, size_t workspace_bytes, marius_stream_t stream) {
    NaArgs A;
    const int rc = na_args(P, m, "neighbor_attention_backward", A);
    if (rc) return rc;
    MARIUS_REQUIRE(P->n == 0 || (grad_out && dq && m->stats), "neighbor_attention_backward: null pointer");
    MARIUS_REQUIRE(P->rows == 0 || (m->k && m->v && dk && dv && P->r_items), "neighbor_attention_backward: null pointer");
    MARIUS_REQUIRE(P->T == 0 || (P->r_owner && P->r_entry), "neighbor_attention_backward: null pointer");
    MARIUS_REQUIRE(!dbias || m->bias, "neighbor_attention_backward: the gradient of a bias that is not there");
    const size_t need = marius_neighbor_attention_workspace_bytes(P, m->heads, m->kv_heads, m->dim, 1);
    MARIUS_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "neighbor_attention_backward: workspace too small");
    hipStream_t st = as_stream(stream);
    const int64_t size = m->type == MARIUS_F32 ? 4 : 2;
    MARIUS_REQUIRE(grad_row >= 0 && grad_row * size < (1ll << 32), "neighbor_attention_backward: rows are at most 4 GiB apart");
    A.go = (const char*)grad_out;
    A.go_ld = (uint32_t)(grad_row * size);
    A.go_hd = grad_head * size;
    A.rowstats = (float4*)workspace;
    A.part2 = (float2*)(A.rowstats + (size_t)P->n * A.H);
    A.part = (float*)((char*)A.part2 + na_small_bytes(P, A.H));
    A.out = dq;
    na_launch_typed(A, m->type, NA_DQ, st);
    A.dk = dk;
    A.dv = dv;
    A.out_bias = dbias;
    A.owner = P->r_owner;
    A.entry = P->r_entry;
    A.items = (const int4*)P->r_items;
    A.splits = (const int4*)P->r_splits;
    A.n_items = P->r_n_items;
    A.dense = P->T > 2 * (int64_t)P->r_n_items;
    A.n_splits = P->r_n_splits;
    na_launch_typed(A, m->type, NA_DKV, st);
    return check_launch("neighbor_attention_backward");
}
