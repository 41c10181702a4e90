// Neighbour attention, backward over the rows' lists: dk, dv and the biases' gradients (nbr_attention.hip has the formulas).
#include "nbr_attention.h"

namespace marius {

// UN entries at a time: four where items are long enough to fill them, two where most rows are in a list or two (a whole pass over 200,003 entries of 30,011 rows: four
// 86 us, two 91; over 900,000 entries of 800,000 rows: four 825, two 788; over 1.5 M of a power-law graph: 957 and 944)
template <typename T, int VEC, int LPH, bool BIAS, int UN>
__global__ __launch_bounds__(64 * NA_WAVES) void nbr_attention_dkv_kernel(NaArgs A) {
    const Lane<LPH> w(A, A.spread ? A.H : A.Hkv);
    if (!w.work) return;
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
    const JoinLane<LPH> w;
    const Part<T, VEC, LPH> part(w.l, A.D);
    float dk[VEC], dv[VEC], none;
    if (!join_sums<VEC, LPH>(A, w, A.Hkv, false, part.at, dk, dv, none)) return;
#pragma unroll
    for (int e = 0; e < VEC; ++e) dk[e] *= A.scale;
    const int64_t o = ((int64_t)A.splits[na_block()].x * A.Hkv + w.h) * A.D;
    part.store((T*)A.dk + o, dk);
    part.store((T*)A.dv + o, dv);
}

struct DkvPass {
    static constexpr bool ROWS = true;
    template <typename T, int VEC, int LPH>
    static void launch(const NaArgs& A, dim3 grid, dim3 block, hipStream_t st) {
        if (A.bias && A.dense) nbr_attention_dkv_kernel<T, VEC, LPH, true, 4><<<grid, block, 0, st>>>(A);
        else if (A.bias) nbr_attention_dkv_kernel<T, VEC, LPH, true, 2><<<grid, block, 0, st>>>(A);
        else if (A.dense) nbr_attention_dkv_kernel<T, VEC, LPH, false, 4><<<grid, block, 0, st>>>(A);
        else nbr_attention_dkv_kernel<T, VEC, LPH, false, 2><<<grid, block, 0, st>>>(A);
    }
    template <typename T, int VEC, int LPH>
    static void join(const NaArgs& A, dim3 grid, dim3 block, hipStream_t st) {
        nbr_attention_dkv_join_kernel<T, VEC, LPH><<<grid, block, 0, st>>>(A);
    }
};
void nbr_attention_dkv(const NaArgs& A, int type, hipStream_t st) { na_launch_typed<DkvPass>(A, type, st); }

}  // namespace marius
