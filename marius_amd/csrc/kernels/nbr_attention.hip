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
#include "row_types.h"

namespace marius {

constexpr float NA_INF = __builtin_inff();
constexpr int NA_WAVES = 4;

struct NaArgs {
    const void *q, *k, *v, *go;
    int64_t q_ld, q_hd, k_ld, k_hd, v_ld, v_hd, go_ld, go_hd;   // row and head strides, elements
    const float* bias;                                          // [T, H] or NULL
    float *out_bias, *stats, *part;
    float2* part2;                                              // a part's (m, sum), or its delta
    float4* rowstats;                                           // [n, H]: m, log l, delta of a target's list, for the sweep over the rows' lists
    void *out, *dk, *dv;                                        // contiguous [n, H, D], [rows, Hkv, D]
    const int32_t *index, *owner, *entry;                       // forward lists: index; reverse lists: owner, entry (position in the forward lists)
    const int4 *items, *splits;
    int n_items, n_splits, H, Hkv, D, hp;                       // hp: heads per slot
    bool dense;                                                 // items of more than two entries on average
    float scale;
};

// weight of a running sum that goes from maximum m to `ref`; a maximum of -inf has weight zero
__device__ __forceinline__ float weight_to(float m, float ref) { return m == -NA_INF ? 0.f : __expf(m - ref); }
__device__ __forceinline__ float finite_ref(float m) { return m == -NA_INF ? 0.f : m; }

// which item, head and piece a lane works on
template <int VEC, int LPH>
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
__device__ __forceinline__ void load_numbers(const int32_t* p, int (&v)[UN]) { __builtin_memcpy(v, p, sizeof(v)); }  // (lists end with UN spare entries)

// ---------------------------------------------------------------------------------------------------------------- forward
template <typename T, int VEC, int LPH, bool BIAS>
__global__ __launch_bounds__(64 * NA_WAVES) void nbr_attention_kernel(NaArgs A) {
    constexpr int UN = 4;
    const Lane<VEC, LPH> w(A, A.H);
    if (w.slot >= A.n_items || !w.head) return;
    const int4 it = A.items[w.slot];
    const Place<VEC> at(w.l, A.D, A.D != LPH * VEC);
    const int kv = w.h / (A.H / A.Hkv);
    float q[VEC], acc[VEC], m = -NA_INF, sum = 0.f, bias[UN];
    Piece<T, VEC> raw;
    raw.load((const T*)A.q + (int64_t)it.x * A.q_ld + w.h * A.q_hd + at.at);
    raw.get(q);
    at.leave_own(q);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        q[e] *= A.scale;
        acc[e] = 0.f;
    }
    const T *kp = (const T*)A.k + kv * A.k_hd + at.at, *vp = (const T*)A.v + kv * A.v_hd + at.at;
    int next[UN];
    load_numbers<UN>(A.index + it.y, next);
    if (BIAS)
#pragma unroll
        for (int u = 0; u < UN; ++u) bias[u] = it.y + u < it.z ? A.bias[(int64_t)(it.y + u) * A.H + w.h] : -NA_INF;
    for (int t = it.y; t < it.z; t += UN) {
        Piece<T, VEC> kk[UN], vv[UN];
        float s[UN];
        bool ok[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            ok[u] = t + u < it.z;
            const int64_t j = ok[u] ? next[u] : next[0];  // (behind the list: its last rows once more, computed on by nobody)
            kk[u].load(kp + j * A.k_ld);
            vv[u].load(vp + j * A.v_ld);
            s[u] = 0.f;
            if (BIAS) {
                s[u] = bias[u];
                ok[u] = bias[u] != -NA_INF;
            }
        }
        if (t + UN < it.z) {
            load_numbers<UN>(A.index + t + UN, next);
            if (BIAS)
#pragma unroll
                for (int u = 0; u < UN; ++u) bias[u] = t + UN + u < it.z ? A.bias[(int64_t)(t + UN + u) * A.H + w.h] : -NA_INF;
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            float k[VEC], d = 0.f;
            kk[u].get(k);
            at.leave_own(k);
#pragma unroll
            for (int e = 0; e < VEC; ++e) d += q[e] * k[e];
            d = group_sum<LPH>(d);
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
            float v[VEC];
            vv[u].get(v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += p * v[e];
        }
    }
    if (it.w >= 0) {
        const int64_t o = (int64_t)it.w * A.H + w.h;
        put<float, VEC>(A.part + o * A.D + at.at, acc);
        if (w.l == 0) A.part2[o] = make_float2(m, sum);
    } else {
        const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;  // (NaN stays)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] *= inv;
        const int64_t o = (int64_t)it.x * A.H + w.h;
        put<T, VEC>((T*)A.out + o * A.D + at.at, acc);
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
    const Place<VEC> at(lane & (LPH - 1), A.D, A.D != LPH * VEC);
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
        __builtin_memcpy(v, A.part + o * A.D + at.at, sizeof(v));
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
    put<T, VEC>((T*)A.out + o * A.D + at.at, acc);
    if ((lane & (LPH - 1)) == 0) {
        A.stats[o * 2] = m;
        A.stats[o * 2 + 1] = sum == 0.f ? 0.f : logf(sum);
    }
}
// the same for sums: two rows of D, and (`more`) a number of their own; true for the lanes that hold the result
template <int VEC, int LPH>
__device__ __forceinline__ bool join_sums(const NaArgs& A, int heads, bool more, const Place<VEC>& at, int h, float (&a)[VEC], float (&b)[VEC], float& first) {
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
        __builtin_memcpy(x, A.part + o * 2 * A.D + at.at, sizeof(x));
        __builtin_memcpy(y, A.part + o * 2 * A.D + A.D + at.at, sizeof(y));
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
    const Lane<VEC, LPH> w(A, A.H);
    if (w.slot >= A.n_items || !w.head) return;
    const int4 it = A.items[w.slot];
    const Place<VEC> at(w.l, A.D, A.D != LPH * VEC);
    const int kv = w.h / (A.H / A.Hkv);
    const int64_t o = (int64_t)it.x * A.H + w.h;
    float q[VEC], go[VEC], pdk[VEC], pk[VEC], delta = 0.f, bias[UN];
    Piece<T, VEC> raw, raw2;
    raw.load((const T*)A.q + (int64_t)it.x * A.q_ld + w.h * A.q_hd + at.at);
    raw2.load((const T*)A.go + (int64_t)it.x * A.go_ld + w.h * A.go_hd + at.at);
    const float m = A.stats[o * 2], logl = A.stats[o * 2 + 1];
    raw.get(q);
    raw2.get(go);
    at.leave_own(q);
    at.leave_own(go);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        q[e] *= A.scale;
        pdk[e] = pk[e] = 0.f;
    }
    const T *kp = (const T*)A.k + kv * A.k_hd + at.at, *vp = (const T*)A.v + kv * A.v_hd + at.at;
    int next[UN];
    load_numbers<UN>(A.index + it.y, next);
    if (BIAS)
#pragma unroll
        for (int u = 0; u < UN; ++u) bias[u] = it.y + u < it.z ? A.bias[(int64_t)(it.y + u) * A.H + w.h] : -NA_INF;
    for (int t = it.y; t < it.z; t += UN) {
        Piece<T, VEC> kk[UN], vv[UN];
        float b[UN];
        bool ok[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            ok[u] = t + u < it.z;
            const int64_t j = ok[u] ? next[u] : next[0];
            kk[u].load(kp + j * A.k_ld);
            vv[u].load(vp + j * A.v_ld);
            b[u] = 0.f;
            if (BIAS) {
                b[u] = bias[u];
                ok[u] = bias[u] != -NA_INF;
            }
        }
        if (t + UN < it.z) {
            load_numbers<UN>(A.index + t + UN, next);
            if (BIAS)
#pragma unroll
                for (int u = 0; u < UN; ++u) bias[u] = t + UN + u < it.z ? A.bias[(int64_t)(t + UN + u) * A.H + w.h] : -NA_INF;
        }
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            if (!ok[u]) continue;
            float k[VEC], own[VEC], v[VEC], s = 0.f, d = 0.f;
            kk[u].get(k);
            vv[u].get(v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) own[e] = k[e];
            at.leave_own(own);
            at.leave_own(v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                s += q[e] * own[e];
                d += go[e] * v[e];
            }
            s = group_sum<LPH>(s) + b[u];
            d = group_sum<LPH>(d);
            const float p = probability(s, m, logl), pd = p * d;
            delta += pd;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                pdk[e] += pd * k[e];
                pk[e] += p * k[e];
            }
        }
    }
    if (it.w >= 0) {
        const int64_t p = (int64_t)it.w * A.H + w.h;
        put<float, VEC>(A.part + p * 2 * A.D + at.at, pdk);
        put<float, VEC>(A.part + p * 2 * A.D + A.D + at.at, pk);
        if (w.l == 0) A.part2[p] = make_float2(delta, 0.f);
    } else {
        dq_of<VEC>(pdk, pk, delta, A.scale);
        put<T, VEC>((T*)A.out + o * A.D + at.at, pdk);
        if (w.l == 0) A.rowstats[o] = make_float4(m, logl, delta, 0.f);
    }
}
template <typename T, int VEC, int LPH>
__global__ __launch_bounds__(64 * NA_JOIN) void nbr_attention_dq_join_kernel(NaArgs A) {
    const int lane = threadIdx.x & 63, h = blockIdx.y * (64 / LPH) + lane / LPH;
    const Place<VEC> at(lane & (LPH - 1), A.D, A.D != LPH * VEC);
    float pdk[VEC], pk[VEC], delta;
    if (!join_sums<VEC, LPH>(A, A.H, true, at, h, pdk, pk, delta)) return;
    dq_of<VEC>(pdk, pk, delta, A.scale);
    const int64_t o = (int64_t)A.splits[blockIdx.x].x * A.H + h;
    put<T, VEC>((T*)A.out + o * A.D + at.at, pdk);
    if ((lane & (LPH - 1)) == 0) A.rowstats[o] = make_float4(A.stats[o * 2], A.stats[o * 2 + 1], delta, 0.f);
}

// ---------------------------------------------------------------------------------------------------------------- backward over the rows' lists: dk, dv, db
template <typename T, int VEC, int LPH, bool BIAS, int UN>
__global__ __launch_bounds__(64 * NA_WAVES) void nbr_attention_dkv_kernel(NaArgs A) {
    const Lane<VEC, LPH> w(A, A.Hkv);
    if (w.slot >= A.n_items || !w.head) return;
    const int4 it = A.items[w.slot];
    const Place<VEC> at(w.l, A.D, A.D != LPH * VEC);
    const int R = A.H / A.Hkv;
    float k[VEC], v[VEC], dk[VEC], dv[VEC];
    Piece<T, VEC> raw, raw2;
    raw.load((const T*)A.k + (int64_t)it.x * A.k_ld + w.h * A.k_hd + at.at);
    raw2.load((const T*)A.v + (int64_t)it.x * A.v_ld + w.h * A.v_hd + at.at);
    int next[UN], next_e[UN];
    load_numbers<UN>(A.owner + it.y, next);
    if (BIAS) load_numbers<UN>(A.entry + it.y, next_e);
    raw.get(k);
    raw2.get(v);
    at.leave_own(k);
    at.leave_own(v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        k[e] *= A.scale;
        dk[e] = dv[e] = 0.f;
    }
    for (int t = it.y; t < it.z; t += UN) {
        int64_t i[UN], e_at[UN];
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
            Piece<T, VEC> qq[UN], gg[UN];
            float4 st[UN];
            float bias[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                st[u] = A.rowstats[i[u] * A.H + h];
                bias[u] = BIAS ? A.bias[e_at[u] * A.H + h] : 0.f;
                qq[u].load((const T*)A.q + i[u] * A.q_ld + h * A.q_hd + at.at);
                gg[u].load((const T*)A.go + i[u] * A.go_ld + h * A.go_hd + at.at);
            }
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                if (!in[u]) continue;
                float q[VEC], g[VEC], oq[VEC], og[VEC], s = 0.f, d = 0.f;
                qq[u].get(q);
                gg[u].get(g);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    oq[e] = q[e];
                    og[e] = g[e];
                }
                at.leave_own(oq);
                at.leave_own(og);
                const bool live = !BIAS || bias[u] != -NA_INF;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    s += oq[e] * k[e];
                    d += og[e] * v[e];
                }
                s = group_sum<LPH>(s) + bias[u];
                d = group_sum<LPH>(d);
                const float p = live ? probability(s, st[u].x, st[u].y) : 0.f, ds = live ? p * (d - st[u].z) : 0.f;
                if (BIAS && A.out_bias && w.l == 0) A.out_bias[e_at[u] * A.H + h] = ds;
                if (!live) continue;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    dk[e] += ds * q[e];
                    dv[e] += p * g[e];
                }
            }
        }
    }
    if (it.w >= 0) {
        float* part = A.part + ((int64_t)it.w * A.Hkv + w.h) * 2 * A.D;
        put<float, VEC>(part + at.at, dk);
        put<float, VEC>(part + A.D + at.at, dv);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) dk[e] *= A.scale;
        const int64_t o = ((int64_t)it.x * A.Hkv + w.h) * A.D + at.at;
        put<T, VEC>((T*)A.dk + o, dk);
        put<T, VEC>((T*)A.dv + o, dv);
    }
}
template <typename T, int VEC, int LPH>
__global__ __launch_bounds__(64 * NA_JOIN) void nbr_attention_dkv_join_kernel(NaArgs A) {
    const int lane = threadIdx.x & 63, h = blockIdx.y * (64 / LPH) + lane / LPH;
    const Place<VEC> at(lane & (LPH - 1), A.D, A.D != LPH * VEC);
    float dk[VEC], dv[VEC], none;
    if (!join_sums<VEC, LPH>(A, A.Hkv, false, at, h, dk, dv, none)) return;
#pragma unroll
    for (int e = 0; e < VEC; ++e) dk[e] *= A.scale;
    const int64_t o = ((int64_t)A.splits[blockIdx.x].x * A.Hkv + h) * A.D + at.at;
    put<T, VEC>((T*)A.dk + o, dk);
    put<T, VEC>((T*)A.dv + o, dv);
}

// ---------------------------------------------------------------------------------------------------------------- launches
enum NaPass { NA_FWD = 0, NA_DQ, NA_DKV };

template <typename T, int VEC, int LPH>
static void na_launch(NaArgs A, NaPass pass, hipStream_t st) {
    const int heads = pass == NA_DKV ? A.Hkv : A.H, groups = 64 / LPH;
    A.hp = 1;
    while (A.hp < groups && A.hp < heads) A.hp <<= 1;
    const dim3 grid((unsigned)cdiv(A.n_items, NA_WAVES * (groups / A.hp)), (unsigned)cdiv(heads, A.hp)), jgrid((unsigned)A.n_splits, (unsigned)cdiv(heads, groups));
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
    A = NaArgs{};
    A.q = m->q;
    A.k = m->k;
    A.v = m->v;
    A.q_ld = m->q_row;
    A.q_hd = m->q_head;
    A.k_ld = m->k_row;
    A.k_hd = m->k_head;
    A.v_ld = m->v_row;
    A.v_hd = m->v_head;
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
    A.go = grad_out;
    A.go_ld = grad_row;
    A.go_hd = grad_head;
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
