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
// One wave per work item (a list, or 256 entries of a long one).  A head's row is spread over LPH lanes, 16 bytes each; the wave's 64 / LPH lane groups
// are hp heads (the power of two that covers them) times as many entries in flight side by side as are left, each lane group with its own running maximum, sum
// and accumulator, joined by shuffles at the end.  Parts of a long list are written as partial results and joined by a second launch in order.
// Bound by the gather of rows: 2 rows per entry in each of the three sweeps.
#include "row_types.h"

namespace marius {

constexpr float LOG2E = 1.4426950408889634f, NA_INF = __builtin_inff();
constexpr int NA_WAVES = 4;

struct NaArgs {
    const void *q, *k, *v, *go;
    int64_t q_ld, q_hd, k_ld, k_hd, v_ld, v_hd, go_ld, go_hd;   // row and head strides, elements
    const float* bias;                                          // [T, H] or NULL
    float *out_bias, *stats, *delta, *part;
    void *out, *dk, *dv;                                        // contiguous [n, H, D], [rows, Hkv, D]
    const int32_t *index, *owner, *entry;                       // forward lists: index; reverse lists: owner, entry (position in the forward lists)
    const int4 *items, *splits;
    int n_items, n_splits, H, Hkv, D, hp;                       // hp: heads per wave
    float scale;
};

template <int LPH>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = LPH >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// `cur` and `other`: running (maximum, sum) pairs and their weights to a common maximum; a maximum of -inf has weight zero
__device__ __forceinline__ float weight_to(float m, float top) { return m == -NA_INF ? 0.f : __expf(m - top); }

// ---------------------------------------------------------------------------------------------------------------- forward
template <typename T, int LPH, bool BIAS>
__global__ __launch_bounds__(64 * NA_WAVES) void nbr_attention_kernel(NaArgs A) {
    constexpr int VEC = 16 / sizeof(T), UN = 4;
    const int lane = threadIdx.x & 63, item = blockIdx.x * NA_WAVES + (threadIdx.x >> 6);
    if (item >= A.n_items) return;
    const int4 it = A.items[item];
    const int l = lane & (LPH - 1), g = lane / LPH, hp = A.hp, ES = 64 / (LPH * hp), es = g / hp, h = blockIdx.y * hp + (g & (hp - 1));
    const bool head = h < A.H;
    const int hc = head ? h : A.H - 1, kv = hc / (A.H / A.Hkv), c = l * VEC;
    float q[VEC], acc[VEC], m = -NA_INF, sum = 0.f;
    piece_load<T, VEC>((const T*)A.q + (int64_t)it.x * A.q_ld + hc * A.q_hd, c, A.D, q);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        q[e] *= A.scale;
        acc[e] = 0.f;
    }
    const T *kp = (const T*)A.k + kv * A.k_hd, *vp = (const T*)A.v + kv * A.v_hd;
    for (int b = it.y; b < it.z; b += 64) {
        const int mine = b + lane < it.z ? A.index[b + lane] : 0;
        const int end = it.z - b < 64 ? it.z - b : 64;
        for (int t = 0; t < end; t += ES * UN) {
            float kk[UN][VEC], vv[UN][VEC], s[UN];
            bool ok[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const int at = t + u * ES + es;
                const int64_t j = __shfl(mine, at & 63, 64);
                ok[u] = at < end;
                float bias = 0.f;
                if (BIAS && ok[u]) bias = A.bias[(int64_t)(b + at) * A.H + hc];
                if (BIAS && bias == -NA_INF) ok[u] = false;
                s[u] = bias;
#pragma unroll
                for (int e = 0; e < VEC; ++e) kk[u][e] = vv[u][e] = 0.f;
                if (ok[u]) {
                    piece_load<T, VEC>(kp + j * A.k_ld, c, A.D, kk[u]);
                    piece_load<T, VEC>(vp + j * A.v_ld, c, A.D, vv[u]);
                }
            }
            float top = m;
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                float d = 0.f;
#pragma unroll
                for (int e = 0; e < VEC; ++e) d += q[e] * kk[u][e];
                d = group_sum<LPH>(d);
                s[u] = ok[u] ? d + s[u] : -NA_INF;
                top = fmaxf(top, s[u]);
            }
            const float ref = top == -NA_INF ? 0.f : top, w = weight_to(m, ref);
            m = top;
            sum *= w;
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] *= w;
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const float p = __expf(s[u] - ref);
                sum += p;
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] += p * vv[u][e];
            }
        }
    }
    for (int o = LPH * hp; o < 64; o <<= 1) {  // the entries side by side
        const float om = __shfl_xor(m, o, 64), os = __shfl_xor(sum, o, 64), top = fmaxf(m, om), ref = top == -NA_INF ? 0.f : top;
        const float w = weight_to(m, ref), ow = weight_to(om, ref);
        sum = sum * w + os * ow;
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] = acc[e] * w + __shfl_xor(acc[e], o, 64) * ow;
        m = top;
    }
    if (es != 0 || !head) return;
    if (it.w >= 0) {
        float* part = A.part + (int64_t)it.w * A.H * (A.D + 2) + (int64_t)h * (A.D + 2);
        piece_store<float, VEC>(part + 2, c, A.D, acc);
        if (l == 0) {
            part[0] = m;
            part[1] = sum;
        }
    } else {
        const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;  // (NaN stays)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] *= inv;
        piece_store<T, VEC>((T*)A.out + ((int64_t)it.x * A.H + h) * A.D, c, A.D, acc);
        if (l == 0) {
            A.stats[((int64_t)it.x * A.H + h) * 2] = m;
            A.stats[((int64_t)it.x * A.H + h) * 2 + 1] = sum == 0.f ? 0.f : logf(sum);
        }
    }
}

// the parts of a long list, in order
template <typename T, int LPH>
__global__ __launch_bounds__(64) void nbr_attention_join_kernel(NaArgs A) {
    constexpr int VEC = 16 / sizeof(T);
    const int4 sp = A.splits[blockIdx.x];
    const int l = threadIdx.x & (LPH - 1), h = blockIdx.y * (64 / LPH) + threadIdx.x / LPH, c = l * VEC;
    if (h >= A.H) return;
    float acc[VEC], m = -NA_INF, sum = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    for (int s = 0; s < sp.z; ++s) {
        const float* part = A.part + (int64_t)(sp.y + s) * A.H * (A.D + 2) + (int64_t)h * (A.D + 2);
        float v[VEC];
        const float om = part[0], os = part[1], top = fmaxf(m, om), ref = top == -NA_INF ? 0.f : top;
        const float w = weight_to(m, ref), ow = weight_to(om, ref);
        piece_load<float, VEC>(part + 2, c, A.D, v);
        sum = sum * w + os * ow;
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] = acc[e] * w + v[e] * ow;
        m = top;
    }
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] *= inv;
    piece_store<T, VEC>((T*)A.out + ((int64_t)sp.x * A.H + h) * A.D, c, A.D, acc);
    if (l == 0) {
        A.stats[((int64_t)sp.x * A.H + h) * 2] = m;
        A.stats[((int64_t)sp.x * A.H + h) * 2 + 1] = sum == 0.f ? 0.f : logf(sum);
    }
}

// p from a score and its list's (m, log l); a list without a live entry has m = -inf
__device__ __forceinline__ float probability(float s, float m, float logl) { return __expf((s - (m == -NA_INF ? 0.f : m)) - logl); }

// ---------------------------------------------------------------------------------------------------------------- backward over the targets' lists: dq, delta
template <typename T, int LPH, bool BIAS>
__global__ __launch_bounds__(64 * NA_WAVES) void nbr_attention_dq_kernel(NaArgs A) {
    constexpr int VEC = 16 / sizeof(T), UN = 4;
    const int lane = threadIdx.x & 63, item = blockIdx.x * NA_WAVES + (threadIdx.x >> 6);
    if (item >= A.n_items) return;
    const int4 it = A.items[item];
    const int l = lane & (LPH - 1), g = lane / LPH, hp = A.hp, ES = 64 / (LPH * hp), es = g / hp, h = blockIdx.y * hp + (g & (hp - 1));
    const bool head = h < A.H;
    const int hc = head ? h : A.H - 1, kv = hc / (A.H / A.Hkv), c = l * VEC;
    float q[VEC], go[VEC], pdk[VEC], pk[VEC], delta = 0.f;
    piece_load<T, VEC>((const T*)A.q + (int64_t)it.x * A.q_ld + hc * A.q_hd, c, A.D, q);
    piece_load<T, VEC>((const T*)A.go + (int64_t)it.x * A.go_ld + hc * A.go_hd, c, A.D, go);
    const float m = A.stats[((int64_t)it.x * A.H + hc) * 2], logl = A.stats[((int64_t)it.x * A.H + hc) * 2 + 1];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        q[e] *= A.scale;
        pdk[e] = pk[e] = 0.f;
    }
    const T *kp = (const T*)A.k + kv * A.k_hd, *vp = (const T*)A.v + kv * A.v_hd;
    for (int b = it.y; b < it.z; b += 64) {
        const int mine = b + lane < it.z ? A.index[b + lane] : 0;
        const int end = it.z - b < 64 ? it.z - b : 64;
        for (int t = 0; t < end; t += ES * UN) {
            float kk[UN][VEC], vv[UN][VEC], bias[UN];
            bool ok[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const int at = t + u * ES + es;
                const int64_t j = __shfl(mine, at & 63, 64);
                ok[u] = at < end;
                bias[u] = 0.f;
                if (BIAS && ok[u]) bias[u] = A.bias[(int64_t)(b + at) * A.H + hc];
                if (BIAS && bias[u] == -NA_INF) ok[u] = false;
#pragma unroll
                for (int e = 0; e < VEC; ++e) kk[u][e] = vv[u][e] = 0.f;
                if (ok[u]) {
                    piece_load<T, VEC>(kp + j * A.k_ld, c, A.D, kk[u]);
                    piece_load<T, VEC>(vp + j * A.v_ld, c, A.D, vv[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                float s = 0.f, d = 0.f;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    s += q[e] * kk[u][e];
                    d += go[e] * vv[u][e];
                }
                s = group_sum<LPH>(s) + bias[u];
                d = group_sum<LPH>(d);
                const float p = ok[u] ? probability(s, m, logl) : 0.f, pd = ok[u] ? p * d : 0.f;
                delta += pd;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    pdk[e] += pd * kk[u][e];
                    pk[e] += p * kk[u][e];
                }
            }
        }
    }
    for (int o = LPH * hp; o < 64; o <<= 1) {
        delta += __shfl_xor(delta, o, 64);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            pdk[e] += __shfl_xor(pdk[e], o, 64);
            pk[e] += __shfl_xor(pk[e], o, 64);
        }
    }
    if (es != 0 || !head) return;
    if (it.w >= 0) {
        float* part = A.part + ((int64_t)it.w * A.H + h) * (2 * A.D + 1);
        piece_store<float, VEC>(part + 1, c, A.D, pdk);
        piece_store<float, VEC>(part + 1 + A.D, c, A.D, pk);
        if (l == 0) part[0] = delta;
    } else {
        // (two roundings, not a fused one: a list of one entry then gives exactly zero)
        {
#pragma clang fp contract(off)
#pragma unroll
            for (int e = 0; e < VEC; ++e) pdk[e] = A.scale * (pdk[e] - delta * pk[e]);
        }
        piece_store<T, VEC>((T*)A.out + ((int64_t)it.x * A.H + h) * A.D, c, A.D, pdk);
        if (l == 0) A.delta[(int64_t)it.x * A.H + h] = delta;
    }
}
template <typename T, int LPH>
__global__ __launch_bounds__(64) void nbr_attention_dq_join_kernel(NaArgs A) {
    constexpr int VEC = 16 / sizeof(T);
    const int4 sp = A.splits[blockIdx.x];
    const int l = threadIdx.x & (LPH - 1), h = blockIdx.y * (64 / LPH) + threadIdx.x / LPH, c = l * VEC;
    if (h >= A.H) return;
    float pdk[VEC], pk[VEC], delta = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) pdk[e] = pk[e] = 0.f;
    for (int s = 0; s < sp.z; ++s) {
        const float* part = A.part + ((int64_t)(sp.y + s) * A.H + h) * (2 * A.D + 1);
        float a[VEC], b[VEC];
        piece_load<float, VEC>(part + 1, c, A.D, a);
        piece_load<float, VEC>(part + 1 + A.D, c, A.D, b);
        delta += part[0];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            pdk[e] += a[e];
            pk[e] += b[e];
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) pdk[e] = A.scale * (pdk[e] - delta * pk[e]);
    piece_store<T, VEC>((T*)A.out + ((int64_t)sp.x * A.H + h) * A.D, c, A.D, pdk);
    if (l == 0) A.delta[(int64_t)sp.x * A.H + h] = delta;
}

// ---------------------------------------------------------------------------------------------------------------- backward over the rows' lists: dk, dv, db
template <typename T, int LPH, bool BIAS>
__global__ __launch_bounds__(64 * NA_WAVES) void nbr_attention_dkv_kernel(NaArgs A) {
    constexpr int VEC = 16 / sizeof(T), UN = 4;
    const int lane = threadIdx.x & 63, item = blockIdx.x * NA_WAVES + (threadIdx.x >> 6);
    if (item >= A.n_items) return;
    const int4 it = A.items[item];
    const int l = lane & (LPH - 1), g = lane / LPH, hp = A.hp, ES = 64 / (LPH * hp), es = g / hp, kv = blockIdx.y * hp + (g & (hp - 1)), R = A.H / A.Hkv;
    const bool head = kv < A.Hkv;
    const int kc = head ? kv : A.Hkv - 1, c = l * VEC;
    float k[VEC], v[VEC], dk[VEC], dv[VEC];
    piece_load<T, VEC>((const T*)A.k + (int64_t)it.x * A.k_ld + kc * A.k_hd, c, A.D, k);
    piece_load<T, VEC>((const T*)A.v + (int64_t)it.x * A.v_ld + kc * A.v_hd, c, A.D, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        k[e] *= A.scale;
        dk[e] = dv[e] = 0.f;
    }
    for (int b = it.y; b < it.z; b += 64) {
        const int mine = b + lane < it.z ? A.owner[b + lane] : 0, mine_e = BIAS && b + lane < it.z ? A.entry[b + lane] : 0;
        const int end = it.z - b < 64 ? it.z - b : 64;
        for (int t = 0; t < end; t += ES * UN) {
            for (int r = 0; r < R; ++r) {
                const int h = kc * R + r;
                float qq[UN][VEC], go[UN][VEC], m[UN], logl[UN], delta[UN], bias[UN];
                bool ok[UN];
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    const int at = t + u * ES + es;
                    const int64_t i = __shfl(mine, at & 63, 64), e_at = BIAS ? __shfl(mine_e, at & 63, 64) : 0;
                    ok[u] = at < end;
                    bias[u] = 0.f;
                    if (BIAS && ok[u]) bias[u] = A.bias[e_at * A.H + h];
                    if (BIAS && bias[u] == -NA_INF) ok[u] = false;
                    m[u] = logl[u] = delta[u] = 0.f;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) qq[u][e] = go[u][e] = 0.f;
                    if (ok[u]) {
                        piece_load<T, VEC>((const T*)A.q + i * A.q_ld + h * A.q_hd, c, A.D, qq[u]);
                        piece_load<T, VEC>((const T*)A.go + i * A.go_ld + h * A.go_hd, c, A.D, go[u]);
                        m[u] = A.stats[(i * A.H + h) * 2];
                        logl[u] = A.stats[(i * A.H + h) * 2 + 1];
                        delta[u] = A.delta[i * A.H + h];
                    }
                }
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    float s = 0.f, d = 0.f;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        s += qq[u][e] * k[e];
                        d += go[u][e] * v[e];
                    }
                    s = group_sum<LPH>(s) + bias[u];
                    d = group_sum<LPH>(d);
                    const float p = ok[u] ? probability(s, m[u], logl[u]) : 0.f, ds = ok[u] ? p * (d - delta[u]) : 0.f;
                    if (BIAS) {
                        const int at = t + u * ES + es;
                        const int64_t e_at = __shfl(mine_e, at & 63, 64);
                        if (A.out_bias && l == 0 && head && at < end) A.out_bias[e_at * A.H + h] = ds;
                    }
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        dk[e] += ds * qq[u][e];
                        dv[e] += p * go[u][e];
                    }
                }
            }
        }
    }
    for (int o = LPH * hp; o < 64; o <<= 1)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            dk[e] += __shfl_xor(dk[e], o, 64);
            dv[e] += __shfl_xor(dv[e], o, 64);
        }
    if (es != 0 || !head) return;
    if (it.w >= 0) {
        float* part = A.part + ((int64_t)it.w * A.Hkv + kv) * 2 * A.D;
        piece_store<float, VEC>(part, c, A.D, dk);
        piece_store<float, VEC>(part + A.D, c, A.D, dv);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) dk[e] *= A.scale;
        piece_store<T, VEC>((T*)A.dk + ((int64_t)it.x * A.Hkv + kv) * A.D, c, A.D, dk);
        piece_store<T, VEC>((T*)A.dv + ((int64_t)it.x * A.Hkv + kv) * A.D, c, A.D, dv);
    }
}
template <typename T, int LPH>
__global__ __launch_bounds__(64) void nbr_attention_dkv_join_kernel(NaArgs A) {
    constexpr int VEC = 16 / sizeof(T);
    const int4 sp = A.splits[blockIdx.x];
    const int l = threadIdx.x & (LPH - 1), h = blockIdx.y * (64 / LPH) + threadIdx.x / LPH, c = l * VEC;
    if (h >= A.Hkv) return;
    float dk[VEC], dv[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) dk[e] = dv[e] = 0.f;
    for (int s = 0; s < sp.z; ++s) {
        const float* part = A.part + ((int64_t)(sp.y + s) * A.Hkv + h) * 2 * A.D;
        float a[VEC], b[VEC];
        piece_load<float, VEC>(part, c, A.D, a);
        piece_load<float, VEC>(part + A.D, c, A.D, b);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            dk[e] += a[e];
            dv[e] += b[e];
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) dk[e] *= A.scale;
    piece_store<T, VEC>((T*)A.dk + ((int64_t)sp.x * A.Hkv + h) * A.D, c, A.D, dk);
    piece_store<T, VEC>((T*)A.dv + ((int64_t)sp.x * A.Hkv + h) * A.D, c, A.D, dv);
}

// ---------------------------------------------------------------------------------------------------------------- launches
enum NaPass { NA_FWD = 0, NA_DQ, NA_DKV };

template <typename T, int LPH>
static void na_launch(NaArgs A, NaPass pass, hipStream_t st) {
    const int heads = pass == NA_DKV ? A.Hkv : A.H, groups = 64 / LPH;
    A.hp = 1;
    while (A.hp < groups && A.hp < heads) A.hp <<= 1;
    const dim3 grid((unsigned)cdiv(A.n_items, NA_WAVES), (unsigned)cdiv(heads, A.hp)), jgrid((unsigned)A.n_splits, (unsigned)cdiv(heads, groups));
    if (pass == NA_FWD) {
        if (A.bias) nbr_attention_kernel<T, LPH, true><<<grid, dim3(64 * NA_WAVES), 0, st>>>(A);
        else nbr_attention_kernel<T, LPH, false><<<grid, dim3(64 * NA_WAVES), 0, st>>>(A);
        if (A.n_splits > 0) nbr_attention_join_kernel<T, LPH><<<jgrid, dim3(64), 0, st>>>(A);
    } else if (pass == NA_DQ) {
        if (A.bias) nbr_attention_dq_kernel<T, LPH, true><<<grid, dim3(64 * NA_WAVES), 0, st>>>(A);
        else nbr_attention_dq_kernel<T, LPH, false><<<grid, dim3(64 * NA_WAVES), 0, st>>>(A);
        if (A.n_splits > 0) nbr_attention_dq_join_kernel<T, LPH><<<jgrid, dim3(64), 0, st>>>(A);
    } else {
        if (A.bias) nbr_attention_dkv_kernel<T, LPH, true><<<grid, dim3(64 * NA_WAVES), 0, st>>>(A);
        else nbr_attention_dkv_kernel<T, LPH, false><<<grid, dim3(64 * NA_WAVES), 0, st>>>(A);
        if (A.n_splits > 0) nbr_attention_dkv_join_kernel<T, LPH><<<jgrid, dim3(64), 0, st>>>(A);
    }
}
template <typename T>
static void na_launch_width(const NaArgs& A, NaPass pass, hipStream_t st) {
    const int pieces = (int)cdiv(A.D, 16 / (int)sizeof(T));
    if (pieces <= 1) na_launch<T, 1>(A, pass, st);
    else if (pieces <= 2) na_launch<T, 2>(A, pass, st);
    else if (pieces <= 4) na_launch<T, 4>(A, pass, st);
    else if (pieces <= 8) na_launch<T, 8>(A, pass, st);
    else if (pieces <= 16) na_launch<T, 16>(A, pass, st);
    else if (pieces <= 32) na_launch<T, 32>(A, pass, st);
    else na_launch<T, 64>(A, pass, st);
}
static void na_launch_typed(const NaArgs& A, int type, NaPass pass, hipStream_t st) {
    if (A.n_items == 0) return;
    if (type == MARIUS_F32) na_launch_width<float>(A, pass, st);
    else if (type == MARIUS_BF16) na_launch_width<__bf16>(A, pass, st);
    else na_launch_width<_Float16>(A, pass, st);
}

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
    if (!backward) return (size_t)P->n_slots * heads * (dim + 2) * sizeof(float);
    const size_t dq = (size_t)P->n_slots * heads * (2 * dim + 1), dkv = (size_t)P->r_n_slots * kv_heads * 2 * dim;
    return ((size_t)P->n * heads + (dq > dkv ? dq : dkv)) * sizeof(float);
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
    A.part = (float*)workspace;
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
    A.delta = (float*)workspace;
    A.part = A.delta + (size_t)P->n * A.H;
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
    A.n_splits = P->r_n_splits;
    na_launch_typed(A, m->type, NA_DKV, st);
    return check_launch("neighbor_attention_backward");
}
