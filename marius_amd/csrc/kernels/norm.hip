// The norms before and after a block of an encoder, fused with the block's gate and the scaled residual:
//
//     u = norm_post(z)              z [n, d]: the block's output (absent post norm: u = z)
//     y = s x + act(g) u            x [n, d]: the residual stream, s: a number, g: absent, [d] or [n, d]
//     h = norm_pre(y)               the next block's input (absent pre norm: no h)
//
//     norm(v) = (v - mean v) r w + b,   r = 1 / sqrt(mean (v - mean v)^2 + eps)         LAYER
//     norm(v) = v r w + b,              r = 1 / sqrt(mean v^2 + eps)                    RMS
//
// and its backward from the gradients of y and h, the stored y and the stored z (the statistics are taken again: the row is in registers anyhow, so
// nothing but y and z has to be kept between the passes):
//
//     dt = dy + r (a - [mean a] - yn mean(a yn)),  a = dh w_pre, yn = (y - [mean y]) r       (bracketed terms: LAYER only)
//     dx = s dt,   dg = dt u act'(g),   du = act(g) dt,   dz = the same norm gradient of du w_post at z
//     dw = sum over rows of (gradient of the norm's output) times (normalised row),   db = sum over rows of that gradient
//
// Bound by HBM: every element is read once and written once, about ten operations each.  A row lives in the registers of 2 to 64 lanes of one wave (several
// rows per wave where they are short) or of a whole workgroup (long rows), so the two statistics cost shuffles, not passes over memory.  Sums over rows are
// deterministic: a workgroup adds its rows in order in registers, its lanes in a fixed order in LDS, and a second launch adds the workgroups' partials in
// order.  Statistics, sums and the residual are fp32; y and h are rounded once each, at their stores (h comes from the unrounded y).
#include "row_types.h"

namespace marius {

constexpr int NORM_T = 256, NORM_MAX_D = 8192, NORM_MAX_WG = 1024;

struct NormArgs {
    const void *x, *z, *gate, *post_w, *post_b, *pre_w, *pre_b, *dy, *dh;  // forward: x; backward: x = the stored y
    void *y, *h, *dx, *dz, *dgate;                                         // dgate: [n, d] gates only
    int64_t x_ld, z_ld, gate_ld, y_ld, h_ld, dy_ld, dh_ld, dx_ld, dz_ld, dgate_ld, n;
    int d, tpr, gate_mode /* 0 none, 1 [d], 2 [n, d] */, param_type, act, layer, post, pre;
    float eps, scale;
    float* partial;    // backward: [workgroup][5][d] sums of post_w, post_b, pre_w, pre_b, gate
    int want;          // bit k: sum k is wanted
};
enum { SUM_POST_W = 0, SUM_POST_B, SUM_PRE_W, SUM_PRE_B, SUM_GATE, SUMS };

__device__ __forceinline__ float gate_act(float v, int act) {
    if (act == MARIUS_ACT_RELU) return v > 0.f ? v : 0.f;
    if (act == MARIUS_ACT_SIGMOID) return 1.f / (1.f + expf(-v));
    return v;
}
// act' from the gate g and a = act(g)
__device__ __forceinline__ float gate_slope(float g, float a, int act) {
    if (act == MARIUS_ACT_RELU) return g > 0.f ? 1.f : 0.f;
    if (act == MARIUS_ACT_SIGMOID) return a * (1.f - a);
    return 1.f;
}

// sums over a row's lanes, the same bits on all of them
template <int N, bool BLK>
__device__ __forceinline__ void row_sums(float (&v)[N], int tpr, float* red) {
    for (int o = BLK ? 32 : tpr >> 1; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o, 64);
    if (BLK) {
        const int nw = blockDim.x >> 6, w = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) red[w * N + i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = 0.f;
            for (int k = 0; k < nw; ++k) v[i] += red[k * N + i];
        }
    }
}

// mean (LAYER) and 1 / sqrt(mean square deviation + eps) of a row in registers; elements behind the row are zero on entry
template <int NCH, int VEC, bool BLK>
__device__ __forceinline__ void row_stats(const float (&v)[NCH][VEC], const NormArgs& A, int lane, float* red, float& mean, float& r) {
    const float inv = 1.f / (float)A.d;
    mean = 0.f;
    if (A.layer) {
        float s[1] = {0.f};
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) s[0] += v[j][e];
        row_sums<1, BLK>(s, A.tpr, red);
        mean = s[0] * inv;
    }
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float t = (j * A.tpr + lane) * VEC + e < A.d ? v[j][e] - mean : 0.f;
            s[0] += t * t;
        }
    row_sums<1, BLK>(s, A.tpr, red);
    r = 1.f / sqrtf(s[0] * inv + A.eps);
}

template <int NCH, int VEC>
__device__ __forceinline__ void load_param(const void* p, int type, int tpr, int lane, int d, float missing, float (&v)[NCH][VEC]) {
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
        if (p) piece_load_any<VEC>(p, type, (j * tpr + lane) * VEC, d, v[j]);
        else
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[j][e] = missing;
    }
}

template <typename S, typename T, int NCH, bool BLK>
__global__ __launch_bounds__(BLK ? 512 : NORM_T) void residual_norm_kernel(NormArgs A) {
    constexpr int VEC = 16 / sizeof(T);
    __shared__ float red[8];
    const int tpr = BLK ? (int)blockDim.x : A.tpr, lane = BLK ? (int)threadIdx.x : (int)threadIdx.x & (tpr - 1);
    const int rpw = BLK ? 1 : NORM_T / tpr, mine = BLK ? 0 : (int)threadIdx.x / tpr;
    float w2[NCH][VEC], b2[NCH][VEC], w1[NCH][VEC], b1[NCH][VEC], gc[NCH][VEC];
    load_param<NCH, VEC>(A.post ? A.post_w : nullptr, A.param_type, tpr, lane, A.d, 1.f, w1);
    load_param<NCH, VEC>(A.post ? A.post_b : nullptr, A.param_type, tpr, lane, A.d, 0.f, b1);
    load_param<NCH, VEC>(A.pre ? A.pre_w : nullptr, A.param_type, tpr, lane, A.d, 1.f, w2);
    load_param<NCH, VEC>(A.pre ? A.pre_b : nullptr, A.param_type, tpr, lane, A.d, 0.f, b2);
    load_param<NCH, VEC>(A.gate_mode == 1 ? A.gate : nullptr, A.param_type, tpr, lane, A.d, 1.f, gc);
    if (A.gate_mode == 1)
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) gc[j][e] = gate_act(gc[j][e], A.act);
    for (int64_t base = (int64_t)blockIdx.x * rpw; base < A.n; base += (int64_t)gridDim.x * rpw) {
        const bool live = base + mine < A.n;
        const int64_t row = live ? base + mine : A.n - 1;  // (lanes behind the last row take part in the shuffles with its values and store nothing)
        float y[NCH][VEC];
#pragma unroll
        for (int j = 0; j < NCH; ++j) piece_load<S, VEC>((const S*)A.x + row * A.x_ld, (j * tpr + lane) * VEC, A.d, y[j]);
        if (A.z) {
            float z[NCH][VEC], g[NCH][VEC];
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                piece_load<T, VEC>((const T*)A.z + row * A.z_ld, (j * tpr + lane) * VEC, A.d, z[j]);
                if (A.gate_mode == 2) piece_load<T, VEC>((const T*)A.gate + row * A.gate_ld, (j * tpr + lane) * VEC, A.d, g[j]);
            }
            float mean = 0.f, r = 1.f;
            if (A.post) row_stats<NCH, VEC, BLK>(z, A, lane, red, mean, r);
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float u = A.post ? (z[j][e] - mean) * r * w1[j][e] + b1[j][e] : z[j][e];
                    const float open = A.gate_mode == 2 ? gate_act(g[j][e], A.act) : gc[j][e];
                    y[j][e] = A.scale * y[j][e] + open * u;
                }
            if (live)
#pragma unroll
                for (int j = 0; j < NCH; ++j) piece_store<S, VEC>((S*)A.y + row * A.y_ld, (j * tpr + lane) * VEC, A.d, y[j]);
        }
        if (A.pre) {
            float mean, r;
            // (elements behind the row: gate, weights and z are zero or one there, so y may not be zero: clear it for the statistics)
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if ((j * tpr + lane) * VEC + e >= A.d) y[j][e] = 0.f;
            row_stats<NCH, VEC, BLK>(y, A, lane, red, mean, r);
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e) y[j][e] = (y[j][e] - mean) * r * w2[j][e] + b2[j][e];
            if (live)
#pragma unroll
                for (int j = 0; j < NCH; ++j) piece_store<T, VEC>((T*)A.h + row * A.h_ld, (j * tpr + lane) * VEC, A.d, y[j]);
        }
    }
}

// gradient of the norm's input from a = (gradient of its output) times w, at v: r (a - [mean a] - vn mean(a vn)).  v becomes the normalised row.
template <int NCH, int VEC, bool BLK>
__device__ __forceinline__ void norm_gradient(float (&v)[NCH][VEC], float (&a)[NCH][VEC], const NormArgs& A, float mean, float r, float* red) {
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            s[0] += a[j][e] * v[j][e];
            s[1] += a[j][e];
        }
    row_sums<2, BLK>(s, A.tpr, red);
    const float inv = 1.f / (float)A.d, ma = A.layer ? s[1] * inv : 0.f, mv = s[0] * inv;
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) a[j][e] = r * (a[j][e] - ma - v[j][e] * mv);
}

template <typename S, typename T, int NCH, bool BLK>
__global__ __launch_bounds__(BLK ? 512 : NORM_T) void residual_norm_backward_kernel(NormArgs A) {
    constexpr int VEC = 16 / sizeof(T);
    __shared__ float red[16];
    __shared__ float fold[BLK ? 1 : NORM_T * VEC];
    const int tpr = BLK ? (int)blockDim.x : A.tpr, lane = BLK ? (int)threadIdx.x : (int)threadIdx.x & (tpr - 1);
    const int rpw = BLK ? 1 : NORM_T / tpr, mine = BLK ? 0 : (int)threadIdx.x / tpr;
    float w2[NCH][VEC], w1[NCH][VEC], b1[NCH][VEC], gc[NCH][VEC], acc[SUMS][NCH][VEC];
    load_param<NCH, VEC>(A.post ? A.post_w : nullptr, A.param_type, tpr, lane, A.d, 1.f, w1);
    load_param<NCH, VEC>(A.post ? A.post_b : nullptr, A.param_type, tpr, lane, A.d, 0.f, b1);
    load_param<NCH, VEC>(A.pre ? A.pre_w : nullptr, A.param_type, tpr, lane, A.d, 1.f, w2);
    load_param<NCH, VEC>(A.gate_mode == 1 ? A.gate : nullptr, A.param_type, tpr, lane, A.d, 1.f, gc);
    if (A.gate_mode == 1)
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) gc[j][e] = gate_act(gc[j][e], A.act);
#pragma unroll
    for (int k = 0; k < SUMS; ++k)
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[k][j][e] = 0.f;
    for (int64_t base = (int64_t)blockIdx.x * rpw; base < A.n; base += (int64_t)gridDim.x * rpw) {
        const bool live = base + mine < A.n;
        const int64_t row = live ? base + mine : A.n - 1;
        float dt[NCH][VEC];
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            if (A.dy) piece_load<S, VEC>((const S*)A.dy + row * A.dy_ld, (j * tpr + lane) * VEC, A.d, dt[j]);
            else
#pragma unroll
                for (int e = 0; e < VEC; ++e) dt[j][e] = 0.f;
        }
        if (A.pre && A.dh) {
            float y[NCH][VEC], a[NCH][VEC], mean, r;
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                piece_load<S, VEC>((const S*)A.x + row * A.x_ld, (j * tpr + lane) * VEC, A.d, y[j]);
                piece_load<T, VEC>((const T*)A.dh + row * A.dh_ld, (j * tpr + lane) * VEC, A.d, a[j]);
            }
            row_stats<NCH, VEC, BLK>(y, A, lane, red, mean, r);
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    y[j][e] = (y[j][e] - mean) * r;
                    if (live) {
                        acc[SUM_PRE_W][j][e] += a[j][e] * y[j][e];
                        acc[SUM_PRE_B][j][e] += a[j][e];
                    }
                    a[j][e] *= w2[j][e];
                }
            norm_gradient<NCH, VEC, BLK>(y, a, A, mean, r, red);
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e) dt[j][e] += a[j][e];
        }
        if (A.dx && live) {
            float o[VEC];
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) o[e] = A.scale * dt[j][e];
                piece_store<S, VEC>((S*)A.dx + row * A.dx_ld, (j * tpr + lane) * VEC, A.d, o);
            }
        }
        if (!A.z) continue;
        float z[NCH][VEC], g[NCH][VEC], mean = 0.f, r = 1.f;
        if (A.post || A.gate_mode) {
#pragma unroll
            for (int j = 0; j < NCH; ++j) piece_load<T, VEC>((const T*)A.z + row * A.z_ld, (j * tpr + lane) * VEC, A.d, z[j]);
            if (A.post) {
                row_stats<NCH, VEC, BLK>(z, A, lane, red, mean, r);
#pragma unroll
                for (int j = 0; j < NCH; ++j)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) z[j][e] = (z[j][e] - mean) * r;
            }
        }
        if (A.gate_mode == 2)
#pragma unroll
            for (int j = 0; j < NCH; ++j) piece_load<T, VEC>((const T*)A.gate + row * A.gate_ld, (j * tpr + lane) * VEC, A.d, g[j]);
        if (A.gate_mode) {
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                float o[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float u = A.post ? z[j][e] * w1[j][e] + b1[j][e] : z[j][e];
                    const float du = dt[j][e] * u;
                    if (A.gate_mode == 2) {
                        const float open = gate_act(g[j][e], A.act);
                        o[e] = du * gate_slope(g[j][e], open, A.act);
                        dt[j][e] *= open;
                    } else {
                        if (live) acc[SUM_GATE][j][e] += du;
                        dt[j][e] *= gc[j][e];
                    }
                }
                if (A.gate_mode == 2 && live) piece_store<T, VEC>((T*)A.dgate + row * A.dgate_ld, (j * tpr + lane) * VEC, A.d, o);
            }
        }
        if (A.post) {
#pragma unroll
            for (int j = 0; j < NCH; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const bool in = (j * tpr + lane) * VEC + e < A.d;  // (behind the row z is -mean r: keep it out of the sums)
                    if (!in) z[j][e] = 0.f;
                    if (live) {
                        acc[SUM_POST_W][j][e] += dt[j][e] * z[j][e];
                        acc[SUM_POST_B][j][e] += dt[j][e];
                    }
                    dt[j][e] = in ? dt[j][e] * w1[j][e] : 0.f;
                }
            norm_gradient<NCH, VEC, BLK>(z, dt, A, mean, r, red);
        }
        if (live)
#pragma unroll
            for (int j = 0; j < NCH; ++j) piece_store<T, VEC>((T*)A.dz + row * A.dz_ld, (j * tpr + lane) * VEC, A.d, dt[j]);
    }
    // this workgroup's sums: lanes that own the same columns are added in a fixed order
#pragma unroll
    for (int k = 0; k < SUMS; ++k) {
        if (!(A.want >> k & 1)) continue;  // (uniform)
        float* out = A.partial + ((int64_t)blockIdx.x * SUMS + k) * A.d;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            const int c = (j * tpr + lane) * VEC;
            if (BLK) {
                piece_store<float, VEC>(out, c, A.d, acc[k][j]);
            } else {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < VEC; ++e) fold[threadIdx.x * VEC + e] = acc[k][j][e];
                __syncthreads();
                if (mine == 0) {
                    float s[VEC];
#pragma unroll
                    for (int e = 0; e < VEC; ++e) s[e] = 0.f;
                    for (int q = 0; q < rpw; ++q)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) s[e] += fold[(q * tpr + lane) * VEC + e];
                    piece_store<float, VEC>(out, c, A.d, s);
                }
            }
        }
    }
}

struct NormSumArgs {
    const float* partial;
    int nwg, d, want, type, act;
    const void* gate;      // channel gate: its sum is multiplied by act'
    void* out[SUMS];
};
// 32 columns x 8 slices of the workgroups: a slice adds its workgroups in order, the slices are added in order
__global__ __launch_bounds__(256) void residual_norm_sums_kernel(NormSumArgs A) {
    __shared__ float red[256];
    const int k = blockIdx.y, c = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
    if (!(A.want >> k & 1)) return;  // (uniform)
    float s = 0.f;
    if (c < A.d)
        for (int w = slice; w < A.nwg; w += 8) s += A.partial[((int64_t)w * SUMS + k) * A.d + c];
    red[threadIdx.x] = s;
    __syncthreads();
    if (slice == 0 && c < A.d) {
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) t += red[q * 32 + threadIdx.x];
        if (k == SUM_GATE) {
            const float g = element_any(A.gate, A.type, c);
            t *= gate_slope(g, gate_act(g, A.act), A.act);
        }
        element_store_any(A.out[k], A.type, c, t);
    }
}

// lanes per row and pieces per lane: a row of up to 128 pieces stays in one wave (two pieces a lane at most), a longer one takes a workgroup
struct NormShape {
    int tpr, nch;
    bool blk;
};
static NormShape norm_shape(int d, int vec) {
    const int units = (int)cdiv(d, vec);
    NormShape s{1, 1, units > 128};
    if (!s.blk) {
        while (s.tpr < 64 && s.tpr < units) s.tpr <<= 1;
        s.nch = units > 64 ? 2 : 1;
    } else {
        s.tpr = units > 1024 ? 512 : 256;
        s.nch = (int)cdiv(units, s.tpr) <= 1 ? 1 : cdiv(units, s.tpr) <= 2 ? 2 : 4;
    }
    return s;
}

template <typename S, typename T>
static void launch_norm(const NormArgs& A, const NormShape& s, bool backward, unsigned grid, hipStream_t st) {
    const dim3 g(grid), b(s.blk ? s.tpr : NORM_T);
    if (backward) {
        if (!s.blk && s.nch == 1) residual_norm_backward_kernel<S, T, 1, false><<<g, b, 0, st>>>(A);
        else if (!s.blk) residual_norm_backward_kernel<S, T, 2, false><<<g, b, 0, st>>>(A);
        else if (s.nch == 1) residual_norm_backward_kernel<S, T, 1, true><<<g, b, 0, st>>>(A);
        else if (s.nch == 2) residual_norm_backward_kernel<S, T, 2, true><<<g, b, 0, st>>>(A);
        else residual_norm_backward_kernel<S, T, 4, true><<<g, b, 0, st>>>(A);
    } else {
        if (!s.blk && s.nch == 1) residual_norm_kernel<S, T, 1, false><<<g, b, 0, st>>>(A);
        else if (!s.blk) residual_norm_kernel<S, T, 2, false><<<g, b, 0, st>>>(A);
        else if (s.nch == 1) residual_norm_kernel<S, T, 1, true><<<g, b, 0, st>>>(A);
        else if (s.nch == 2) residual_norm_kernel<S, T, 2, true><<<g, b, 0, st>>>(A);
        else residual_norm_kernel<S, T, 4, true><<<g, b, 0, st>>>(A);
    }
}
static void launch_norm_typed(const NormArgs& A, const NormShape& s, int stream_type, int type, bool backward, unsigned grid, hipStream_t st) {
    if (type == MARIUS_F32) launch_norm<float, float>(A, s, backward, grid, st);
    else if (type == MARIUS_BF16 && stream_type == MARIUS_F32) launch_norm<float, __bf16>(A, s, backward, grid, st);
    else if (type == MARIUS_BF16) launch_norm<__bf16, __bf16>(A, s, backward, grid, st);
    else if (stream_type == MARIUS_F32) launch_norm<float, _Float16>(A, s, backward, grid, st);
    else launch_norm<_Float16, _Float16>(A, s, backward, grid, st);
}

// what both directions ask of a descriptor; fills the shared arguments
static int norm_args(const marius_residual_norm* m, const char* what, NormArgs& A) {
    MARIUS_REQUIRE(m, "%s: null descriptor", what);
    MARIUS_REQUIRE(m->n >= 0 && m->d > 0 && m->d <= NORM_MAX_D, "%s: rows of 1 to %d elements (n = %lld, d = %d)", what, NORM_MAX_D, (long long)m->n, m->d);
    MARIUS_REQUIRE(float_type_ok(m->type) && float_type_ok(m->param_type) && (m->stream_type == m->type || m->stream_type == MARIUS_F32),
                   "%s: the stream is fp32 or of the block's type, types are MARIUS_F32 / BF16 / F16", what);
    MARIUS_REQUIRE(m->kind == MARIUS_NORM_RMS || m->kind == MARIUS_NORM_LAYER, "%s: unknown norm", what);
    MARIUS_REQUIRE(m->gate_mode >= MARIUS_GATE_NONE && m->gate_mode <= MARIUS_GATE_ELEMENT, "%s: unknown gate mode", what);
    MARIUS_REQUIRE(m->gate_activation == MARIUS_ACT_NONE || m->gate_activation == MARIUS_ACT_RELU || m->gate_activation == MARIUS_ACT_SIGMOID, "Unsupported activation function");
    MARIUS_REQUIRE(m->eps >= 0.f, "%s: eps must not be negative", what);
    MARIUS_REQUIRE(m->pre_norm || m->has_block, "%s: neither a block nor a norm: nothing to compute", what);
    MARIUS_REQUIRE(m->has_block || (!m->post_norm && m->gate_mode == MARIUS_GATE_NONE), "%s: a post norm and a gate need a block", what);
    MARIUS_REQUIRE(m->gate_mode == MARIUS_GATE_NONE || m->gate || (m->gate_mode == MARIUS_GATE_ELEMENT && m->n == 0), "%s: null gate", what);
    MARIUS_REQUIRE(m->gate_mode != MARIUS_GATE_ELEMENT || m->gate_ld >= m->d, "%s: gate rows overlap", what);
    A = NormArgs{};
    A.gate = m->gate;
    A.gate_ld = m->gate_ld;
    A.gate_mode = m->gate_mode;
    A.post_w = m->post_weight;
    A.post_b = m->post_bias;
    A.pre_w = m->pre_weight;
    A.pre_b = m->pre_bias;
    A.n = m->n;
    A.d = m->d;
    A.param_type = m->param_type;
    A.act = m->gate_activation;
    A.layer = m->kind == MARIUS_NORM_LAYER;
    A.post = m->post_norm != 0;
    A.pre = m->pre_norm != 0;
    A.eps = m->eps;
    A.scale = m->has_block ? m->residual_scale : 1.f;
    return MARIUS_OK;
}

}  // namespace marius

using namespace marius;

extern "C" int marius_residual_norm_forward(const marius_residual_norm* m, const void* x, int64_t x_ld, const void* block, int64_t block_ld, void* y, int64_t y_ld,
                                            void* h, int64_t h_ld, marius_stream_t stream) {
    NormArgs A;
    const int rc = norm_args(m, "residual_norm_forward", A);
    if (rc) return rc;
    if (A.n == 0) return MARIUS_OK;
    MARIUS_REQUIRE(x && x_ld >= A.d && (!m->has_block || (block && block_ld >= A.d && y && y_ld >= A.d)) && (!A.pre || (h && h_ld >= A.d)),
                   "residual_norm_forward: null pointer or overlapping rows");
    A.x = x;
    A.x_ld = x_ld;
    A.z = m->has_block ? block : nullptr;
    A.z_ld = block_ld;
    A.y = y;
    A.y_ld = y_ld;
    A.h = h;
    A.h_ld = h_ld;
    const NormShape s = norm_shape(A.d, m->type == MARIUS_F32 ? 4 : 8);
    A.tpr = s.tpr;
    const int64_t groups = cdiv(A.n, s.blk ? 1 : NORM_T / s.tpr);
    launch_norm_typed(A, s, m->stream_type, m->type, false, (unsigned)(groups < 2048 ? groups : 2048), as_stream(stream));
    return check_launch("residual_norm_forward");
}

extern "C" size_t marius_residual_norm_workspace_bytes(int64_t n, int32_t d) {
    return n > 0 && d > 0 ? (size_t)NORM_MAX_WG * SUMS * (size_t)d * sizeof(float) : 0;
}

extern "C" int marius_residual_norm_backward(const marius_residual_norm* m, const marius_residual_norm_grads* g, const void* y, int64_t y_ld, const void* block,
                                             int64_t block_ld, void* workspace, size_t workspace_bytes, marius_stream_t stream) {
    NormArgs A;
    const int rc = norm_args(m, "residual_norm_backward", A);
    if (rc) return rc;
    MARIUS_REQUIRE(g, "residual_norm_backward: null descriptor");
    MARIUS_REQUIRE((!g->dpost_weight && !g->dpost_bias) || A.post, "residual_norm_backward: gradients of a post norm that is not there");
    MARIUS_REQUIRE((!g->dpre_weight && !g->dpre_bias) || A.pre, "residual_norm_backward: gradients of a pre norm that is not there");
    void* sums[SUMS] = {g->dpost_weight, g->dpost_bias, g->dpre_weight, g->dpre_bias, A.gate_mode == MARIUS_GATE_CHANNEL ? g->dgate : nullptr};
    for (int k = 0; k < SUMS; ++k) A.want |= (sums[k] ? 1 : 0) << k;
    hipStream_t st = as_stream(stream);
    int nwg = 0;
    if (A.n > 0) {
        MARIUS_REQUIRE(g->grad_y || (A.pre && g->grad_h), "residual_norm_backward: no gradient to go back from");
        MARIUS_REQUIRE((!g->grad_y || g->grad_y_ld >= A.d) && (!g->grad_h || g->grad_h_ld >= A.d) && (!g->dx || g->dx_ld >= A.d), "residual_norm_backward: overlapping rows");
        MARIUS_REQUIRE(!(A.pre && g->grad_h) || (y && y_ld >= A.d), "residual_norm_backward: the norm's gradient needs the stored stream");
        MARIUS_REQUIRE(!m->has_block || (g->dblock && g->dblock_ld >= A.d), "residual_norm_backward: null or overlapping block gradient");
        MARIUS_REQUIRE(!(A.post || A.gate_mode) || (block && block_ld >= A.d), "residual_norm_backward: null or overlapping block");
        MARIUS_REQUIRE(A.gate_mode != MARIUS_GATE_ELEMENT || (g->dgate && g->dgate_ld >= A.d), "residual_norm_backward: null or overlapping gate gradient");
        MARIUS_REQUIRE(!A.want || (workspace && workspace_bytes >= marius_residual_norm_workspace_bytes(A.n, A.d)), "residual_norm_backward: workspace too small");
        A.x = y;
        A.x_ld = y_ld;
        A.z = m->has_block ? (block ? block : g->dblock) : nullptr;  // (no post norm and no gate: the block itself is not read)
        A.z_ld = block_ld;
        A.dy = g->grad_y;
        A.dy_ld = g->grad_y_ld;
        A.dh = A.pre ? g->grad_h : nullptr;
        A.dh_ld = g->grad_h_ld;
        A.dx = g->dx;
        A.dx_ld = g->dx_ld;
        A.dz = g->dblock;
        A.dz_ld = g->dblock_ld;
        A.dgate = A.gate_mode == MARIUS_GATE_ELEMENT ? g->dgate : nullptr;
        A.dgate_ld = g->dgate_ld;
        A.partial = (float*)workspace;
        const NormShape s = norm_shape(A.d, m->type == MARIUS_F32 ? 4 : 8);
        A.tpr = s.tpr;
        const int64_t groups = cdiv(A.n, s.blk ? 1 : NORM_T / s.tpr);
        nwg = (int)(groups < NORM_MAX_WG ? groups : NORM_MAX_WG);
        launch_norm_typed(A, s, m->stream_type, m->type, true, (unsigned)nwg, st);
    }
    if (A.want) {  // (no rows: the sums are zero)
        NormSumArgs S{};
        S.partial = (const float*)workspace;
        S.nwg = nwg;
        S.d = A.d;
        S.want = A.want;
        S.type = A.param_type;
        S.act = A.act;
        S.gate = A.gate;
        for (int k = 0; k < SUMS; ++k) S.out[k] = sums[k];
        residual_norm_sums_kernel<<<dim3((unsigned)cdiv(A.d, 32), SUMS), dim3(256), 0, st>>>(S);
    }
    return check_launch("residual_norm_backward");
}
