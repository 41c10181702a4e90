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
// Bound by the gather of rows, 2 per entry in each of the three sweeps.  Measured: 900,000 entries of 4 x 32 fp32 over 800,000 rows 200 us forward, 184 (targets) and
// 410 (rows: 1.8 GB at 4.4 TB/s, half of it written) back; 1.5 M entries of a power-law graph, 8 query and 4 key heads of 64 bf16, 226, 255 and 506 us: 7 TB/s
// of requests that no L2 holds in each sweep; 64 targets of 15 entries 5 us.
#include "nbr_attention.h"

namespace marius {

// ---------------------------------------------------------------------------------------------------------------- forward
template <typename T, int VEC, int LPH, bool BIAS>
__global__ __launch_bounds__(64 * NA_WAVES) void nbr_attention_kernel(NaArgs A) {
    constexpr int UN = 4;
    const Lane<LPH> w(A, A.H);
    if (!w.work) return;
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
        if (w.l == 0) store_stats(A, o, m, sum);
    }
}

// the parts of a long list
template <typename T, int VEC, int LPH>
__global__ __launch_bounds__(64 * NA_JOIN) void nbr_attention_join_kernel(NaArgs A) {
    __shared__ float red[NA_JOIN][VEC + 2][LPH];
    if (na_block() >= (uint32_t)A.n_splits) return;
    const int4 sp = A.splits[na_block()];
    const JoinLane<LPH> w;
    const Part<T, VEC, LPH> part(w.l, A.D);
    float acc[VEC], m = -NA_INF, sum = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    auto join = [&](float om, float os, const float(&v)[VEC]) {
        const float top = fmaxf(m, om), ref = finite_ref(top), mine = weight_to(m, ref), other = weight_to(om, ref);
        sum = sum * mine + os * other;
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] = acc[e] * mine + v[e] * other;
        m = top;
    };
#pragma unroll 4
    for (int s = w.g; s < sp.z; s += w.G) {
        const int64_t o = (int64_t)(sp.y + s) * A.H + w.h;
        float v[VEC];
        __builtin_memcpy(v, A.part + o * A.D + part.at, sizeof(v));
        const float2 ms = A.part2[o];
        join(ms.x, ms.y, v);
    }
#pragma unroll
    for (int o = LPH; o < 64; o <<= 1) {
        float v[VEC];
        const float om = __shfl_xor(m, o, 64), os = __shfl_xor(sum, o, 64);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = __shfl_xor(acc[e], o, 64);
        join(om, os, v);
    }
    if ((threadIdx.x & 63) < LPH) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) red[w.wave][e][w.l] = acc[e];
        red[w.wave][VEC][w.l] = m;
        red[w.wave][VEC + 1][w.l] = sum;
    }
    __syncthreads();
    if (w.g != 0) return;
    for (int s = 1; s < NA_JOIN; ++s) {
        float v[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = red[s][e][w.l];
        join(red[s][VEC][w.l], red[s][VEC + 1][w.l], v);
    }
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] *= inv;
    const int64_t o = (int64_t)sp.x * A.H + w.h;
    part.store((T*)A.out + o * A.D, acc);
    if (w.l == 0) store_stats(A, o, m, sum);
}
struct ForwardPass {
    static constexpr bool ROWS = false;
    template <typename T, int VEC, int LPH>
    static void launch(const NaArgs& A, dim3 grid, dim3 block, hipStream_t st) {
        if (A.bias) nbr_attention_kernel<T, VEC, LPH, true><<<grid, block, 0, st>>>(A);
        else nbr_attention_kernel<T, VEC, LPH, false><<<grid, block, 0, st>>>(A);
    }
    template <typename T, int VEC, int LPH>
    static void join(const NaArgs& A, dim3 grid, dim3 block, hipStream_t st) {
        nbr_attention_join_kernel<T, VEC, LPH><<<grid, block, 0, st>>>(A);
    }
};

// the workspace: (backward: row statistics,) the parts' small numbers, the parts' rows, each at a multiple of 16 bytes
static size_t na_small_bytes(const marius_neighbor_plan* P, int heads) { return ((size_t)P->n_slots * heads * sizeof(float2) + 15) & ~(size_t)15; }

static int na_args(const marius_neighbor_plan* P, const marius_neighbor_attention* m, const char* what, NaArgs& A) {
    MARIUS_REQUIRE(P && m, "%s: null descriptor", what);
    MARIUS_REQUIRE(P->n >= 0 && P->rows >= 0 && P->T >= 0 && P->n_items >= P->n && P->n_splits >= 0 && P->n_slots >= 0 && P->r_n_items >= 0 && P->r_n_splits >= 0 && P->r_n_slots >= 0,
                   "%s: bad plan", what);  // (a list without a work item would not be written)
    MARIUS_REQUIRE(float_type_ok(m->type), "%s: types are MARIUS_F32 / BF16 / F16", what);
    MARIUS_REQUIRE(m->heads > 0 && m->kv_heads > 0 && m->heads % m->kv_heads == 0 && m->heads <= 1024, "%s: query heads (up to 1024) are a multiple of the key heads", what);
    MARIUS_REQUIRE(m->dim > 0 && m->dim <= 256, "%s: heads of 1 to 256 elements", what);
    MARIUS_REQUIRE(P->n == 0 || m->q, "%s: null pointer", what);
    MARIUS_REQUIRE(P->T == 0 || (m->k && m->v), "%s: null pointer", what);
    MARIUS_REQUIRE(P->n_items == 0 || (P->items && P->index), "%s: null pointer", what);  // (an item of no entries reads numbers ahead as well)
    MARIUS_REQUIRE(P->n_splits == 0 || P->splits, "%s: null pointer", what);
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
    MARIUS_REQUIRE(P->n_slots == 0 || (workspace && workspace_bytes >= marius_neighbor_attention_workspace_bytes(P, m->heads, m->kv_heads, m->dim, 0)),
                   "neighbor_attention_forward: workspace too small");
    A.out = out;
    A.lse = m->lse;
    A.part2 = (float2*)workspace;
    A.part = (float*)((char*)workspace + na_small_bytes(P, A.H));
    na_launch_typed<ForwardPass>(A, m->type, as_stream(stream));
    return check_launch("neighbor_attention_forward");
}

extern "C" int marius_neighbor_attention_backward(const marius_neighbor_plan* P, const marius_neighbor_attention* m, const void* grad_out, int64_t grad_row, int64_t grad_head,
                                                  void* dq, void* dk, void* dv, float* dbias, void* workspace, size_t workspace_bytes, marius_stream_t stream) {
    NaArgs A;
    const int rc = na_args(P, m, "neighbor_attention_backward", A);
    if (rc) return rc;
    MARIUS_REQUIRE(P->n == 0 || (grad_out && dq && m->stats), "neighbor_attention_backward: null pointer");
    MARIUS_REQUIRE(P->rows == 0 || (m->k && m->v && dk && dv), "neighbor_attention_backward: null pointer");
    MARIUS_REQUIRE(P->r_n_items >= P->rows, "neighbor_attention_backward: bad plan");
    MARIUS_REQUIRE(P->r_n_items == 0 || (P->r_items && P->r_owner && (P->r_entry || !m->bias)), "neighbor_attention_backward: null pointer");
    MARIUS_REQUIRE(P->r_n_splits == 0 || P->r_splits, "neighbor_attention_backward: null pointer");
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
    nbr_attention_dq(A, m->type, st);
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
    nbr_attention_dkv(A, m->type, st);
    return check_launch("neighbor_attention_backward");
}
