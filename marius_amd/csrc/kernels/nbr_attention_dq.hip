// Neighbour attention, backward over the targets' lists: dq, and delta for the sweep over the rows' lists (nbr_attention.hip has the formulas).
#include "nbr_attention.h"

namespace marius {

// dq = scale (sum p d k - delta sum p k): two roundings, not a fused one, so that a list of one entry gives exactly zero
template <int VEC>
__device__ __forceinline__ void dq_of(float (&pdk)[VEC], const float (&pk)[VEC], float delta, float scale) {
#pragma clang fp contract(off)
#pragma unroll
    for (int e = 0; e < VEC; ++e) pdk[e] = scale * (pdk[e] - delta * pk[e]);
}

template <typename T, int VEC, int LPH, bool BIAS>
__global__ __launch_bounds__(64 * NA_WAVES) void nbr_attention_dq_kernel(NaArgs A) {
    constexpr int UN = 4;
    const Lane<LPH> w(A, A.H);
    if (!w.work) return;
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
    const JoinLane<LPH> w;
    const Part<T, VEC, LPH> part(w.l, A.D);
    float pdk[VEC], pk[VEC], delta;
    if (!join_sums<VEC, LPH>(A, w, A.H, true, part.at, pdk, pk, delta)) return;
    dq_of<VEC>(pdk, pk, delta, A.scale);
    const int64_t o = (int64_t)A.splits[na_block()].x * A.H + w.h;
    part.store((T*)A.out + o * A.D, pdk);
    if (w.l == 0) A.rowstats[o] = make_float4(A.stats[o * 2], A.stats[o * 2 + 1], delta, 0.f);
}

struct DqPass {
    static constexpr bool ROWS = false;
    template <typename T, int VEC, int LPH>
    static void launch(const NaArgs& A, dim3 grid, dim3 block, hipStream_t st) {
        if (A.bias) nbr_attention_dq_kernel<T, VEC, LPH, true><<<grid, block, 0, st>>>(A);
        else nbr_attention_dq_kernel<T, VEC, LPH, false><<<grid, block, 0, st>>>(A);
    }
    template <typename T, int VEC, int LPH>
    static void join(const NaArgs& A, dim3 grid, dim3 block, hipStream_t st) {
        nbr_attention_dq_join_kernel<T, VEC, LPH><<<grid, block, 0, st>>>(A);
    }
};
void nbr_attention_dq(const NaArgs& A, int type, hipStream_t st) { na_launch_typed<DqPass>(A, type, st); }

}  // namespace marius
