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
// Bound by HBM: every element is read once and written once, about ten operations each (forward, 100,000 rows of 512, fp32 stream and bf16 block: 124 us, 4.9 TB/s;
// back, 160,000 rows of 100 in fp32: 82 us, 4.7 TB/s).  A row lives in registers up to 4096 elements, four elements a lane: in 1 to 64 lanes of one wave
// (several rows per wave where they are short) or, longer than 256 elements, in a workgroup, so the statistics cost lane moves (and a barrier), not passes over memory.
// Four elements, not eight, for the 16-bit types too: the backward pass holds five rows and five sums a lane, and with eight elements one wave per SIMD was
// left (50,000 rows of 1024 in bf16: 579 us, against 190 us now).  Rows of 4097 to 8192 elements hold 16 a lane: forward 50,000 rows of 8192 in bf16 639 us (5.1 TB/s), but back
// some registers go to scratch, most of them with a channel gate: 969 us (5.1 TB/s) without a gate, 1245 (5.3) with one for each element, 1519 (3.2) with one for each channel.
// A row whose squares leave fp32 (elements above 1.8e19) is normalised to zeros.
// Sums over rows are deterministic: a workgroup adds its rows in order in registers, its lanes in a fixed order in LDS, and a second launch adds the
// workgroups' partials in order.  Statistics, sums and the residual are fp32; y and h are rounded once each, at their stores (h comes from the unrounded y).
#include "row_types.h"

namespace marius {

constexpr int NORM_T = 256, NORM_MAX_T = 1024, NORM_MAX_D = 8192, NORM_MAX_WG = 1024;

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

// (sigmoid: the hardware's exponential and reciprocal: a step of fp32 or two, and |v| more from the exponential's rounded argument where it counts)
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + __expf(-v)); }
// sigmoid(v) -> v, its slope: t / (1 + t)^2 of t = exp(-|v|), because a (1 - a) of a rounded a cancels where the gate is almost open (0.9 % off at v = 12, zero from 17 on)
__device__ __forceinline__ float sigmoid_slope(float& v) {
    const float t = __expf(-fabsf(v)), r = __builtin_amdgcn_rcpf(1.f + t);
    v = v >= 0.f ? r : t * r;
    return t * r * r;
}
// act'(g)
__device__ __forceinline__ float gate_slope(float g, int act) {
    if (act == MARIUS_ACT_RELU) return g <= 0.f ? 0.f : 1.f;
    return act == MARIUS_ACT_SIGMOID ? sigmoid_slope(g) : 1.f;
}

// 1 / sqrt(v) within a step of fp32 (a rounded root and quotient would cost more than they give: a gradient's fp32 error is 2.2e-7 against 2.0e-7); the instruction takes no subnormal numbers, which an eps of zero and rows below 1e-19 leave
__device__ __forceinline__ float inverse_root(float v) {
    const bool tiny = v < 0x1p-96f;
    return __builtin_amdgcn_rsqf(tiny ? v * 0x1p96f : v) * (tiny ? 0x1p48f : 1.f);
}

// What is done to every element of a lane's pieces; the conditions that hold for a whole launch stand outside of it (in front of every element they cost more than
// the arithmetic: 250 vector operations an element, 50,000 rows of 1024 in bf16 back in 334 us).
#define EACH(NCH, VEC)                  \
    _Pragma("unroll") for (int j = 0; j < NCH; ++j) _Pragma("unroll") for (int e = 0; e < VEC; ++e)

// A row's lanes: tpr lanes of a wave (a power of two), or, BLK, the workgroup.  Every lane holds NCH pieces of VEC elements.
template <int VEC, int NCH, bool BLK>
struct Row {
    typedef float Values[NCH][VEC];
    int tpr, lane, rows, mine;  // lanes of a row, this one's number, rows a workgroup holds, this one's
    int at[NCH], first[NCH];
    bool tail;                  // (uniform: the row does not fill its lanes' pieces)
    float inv_d, *red;          // red: LDS of two reductions, used in turn
    int turn;
    __device__ __forceinline__ Row(const NormArgs& A, float* red_) : red(red_), turn(0) {
        tpr = BLK ? (int)blockDim.x : A.tpr;
        lane = BLK ? (int)threadIdx.x : (int)threadIdx.x & (tpr - 1);
        rows = BLK ? 1 : NORM_T / tpr;
        mine = BLK ? 0 : (int)threadIdx.x / tpr;
        tail = A.d != tpr * NCH * VEC;
        inv_d = 1.f / (float)A.d;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            const Place<VEC> p(j * tpr + lane, A.d);
            at[j] = p.at;
            first[j] = p.first;
        }
    }
    template <typename T>
    __device__ __forceinline__ void load(Piece<T, VEC> (&p)[NCH], const void* base, int64_t row, int64_t ld) const {
#pragma unroll
        for (int j = 0; j < NCH; ++j) p[j].load((const T*)base + row * ld + at[j]);
    }
    template <typename T>
    __device__ __forceinline__ void store(void* base, int64_t row, int64_t ld, const Values& v) const {
#pragma unroll
        for (int j = 0; j < NCH; ++j) put<T, VEC>((T*)base + row * ld + at[j], v[j]);
    }
    template <typename T>
    __device__ __forceinline__ void get(const Piece<T, VEC> (&p)[NCH], Values& v) const {
#pragma unroll
        for (int j = 0; j < NCH; ++j) p[j].get(v[j]);
    }
    // elements that are a neighbour's (or behind the row): zero, for a sum
    __device__ __forceinline__ void leave_own(Values& v) const {
        if (tail) EACH(NCH, VEC) v[j][e] = e >= first[j] ? v[j][e] : 0.f;
    }
    // sums over the row of N values a lane
    template <int N>
    __device__ __forceinline__ void sums(float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (BLK) {
                v[i] = group_sum<64>(v[i]);
            } else {
                if (tpr >= 2) v[i] = add_half<2>(v[i]);
                if (tpr >= 4) v[i] = add_half<4>(v[i]);
                if (tpr >= 8) v[i] = add_half<8>(v[i]);
                if (tpr >= 16) v[i] = add_half<16>(v[i]);
                if (tpr >= 32) v[i] = add_half<32>(v[i]);
                if (tpr >= 64) v[i] = add_half<64>(v[i]);
            }
        }
        if (BLK) {
            // (one barrier: what the next reduction writes is the other half, and the one after that is behind the next barrier)
            const int nw = (int)blockDim.x >> 6, w = (int)threadIdx.x >> 6, q = (int)threadIdx.x & 15;
            float* r = red + turn * (NORM_MAX_T / 64) * 2;
            turn ^= 1;
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int i = 0; i < N; ++i) r[w * 2 + i] = v[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = group_sum<16>(q < nw ? r[q * 2 + i] : 0.f);
        }
    }
    // v -> the normalised row (v - mean) r; r = 1 / sqrt(mean square deviation + eps)
    __device__ __forceinline__ float normalise(Values& v, const NormArgs& A) {
        Values t;
        if (A.layer) {
            float s[1] = {0.f};
            EACH(NCH, VEC) t[j][e] = v[j][e];
            leave_own(t);
            EACH(NCH, VEC) s[0] += t[j][e];
            sums<1>(s);
            const float mean = s[0] * inv_d;
            EACH(NCH, VEC) v[j][e] -= mean;
        }
        float s[1] = {0.f};
        EACH(NCH, VEC) t[j][e] = v[j][e];
        leave_own(t);
        EACH(NCH, VEC) s[0] += t[j][e] * t[j][e];
        sums<1>(s);
        const float r = inverse_root(s[0] * inv_d + A.eps);
        EACH(NCH, VEC) v[j][e] *= r;
        return r;
    }
    // a: gradient of the normalised row vn -> of what was normalised: r (a - [mean a] - vn mean(a vn))
    __device__ __forceinline__ void gradient(Values& a, const Values& vn, const NormArgs& A, float r) {
        Values t;
        float s[2] = {0.f, 0.f};
        EACH(NCH, VEC) t[j][e] = a[j][e];
        leave_own(t);
        EACH(NCH, VEC) {
            s[0] += t[j][e] * vn[j][e];
            s[1] += t[j][e];
        }
        sums<2>(s);
        const float ma = A.layer ? s[1] * inv_d : 0.f, mv = s[0] * inv_d;
        EACH(NCH, VEC) a[j][e] = r * (a[j][e] - ma - vn[j][e] * mv);
    }
    __device__ __forceinline__ void param(const void* p, int type, float missing, Values& v) const {
        if (p) {
#pragma unroll
            for (int j = 0; j < NCH; ++j) piece_any<VEC>(p, type, at[j], v[j]);
        } else {
            EACH(NCH, VEC) v[j][e] = missing;
        }
    }
    // g -> act(g)
    __device__ __forceinline__ void open(Values& g, int act) const {
        if (act == MARIUS_ACT_SIGMOID) EACH(NCH, VEC) g[j][e] = sigmoid(g[j][e]);
        else if (act == MARIUS_ACT_RELU) EACH(NCH, VEC) g[j][e] = g[j][e] < 0.f ? 0.f : g[j][e];  // (NaN stays)
    }
};

template <typename S, typename T, int VEC, int NCH, bool BLK, int GATE>
__global__ __launch_bounds__(!BLK ? NORM_T : NCH > 1 ? NORM_MAX_T / 2 : NORM_MAX_T) void residual_norm_kernel(NormArgs A) {
    __shared__ float red[BLK ? 4 * NORM_MAX_T / 64 : 1];
    Row<VEC, NCH, BLK> R(A, red);
    float w2[NCH][VEC], b2[NCH][VEC], w1[NCH][VEC], b1[NCH][VEC], gc[NCH][VEC];
    R.param(A.post ? A.post_w : nullptr, A.param_type, 1.f, w1);
    R.param(A.post ? A.post_b : nullptr, A.param_type, 0.f, b1);
    R.param(A.pre ? A.pre_w : nullptr, A.param_type, 1.f, w2);
    R.param(A.pre ? A.pre_b : nullptr, A.param_type, 0.f, b2);
    if (GATE == 1) {
        R.param(A.gate, A.param_type, 1.f, gc);
        R.open(gc, A.act);
    }
    const int64_t stride = (int64_t)gridDim.x * R.rows;
    for (int64_t base = (int64_t)blockIdx.x * R.rows; base < A.n; base += stride) {
        const bool live = BLK || base + R.mine < A.n;
        const int64_t row = live ? base + R.mine : A.n - 1;  // (lanes behind the last row take part in the sums with its values and store nothing)
        Piece<S, VEC> xp[NCH];
        Piece<T, VEC> zp[NCH], gp[NCH];
        float y[NCH][VEC];
        R.load(xp, A.x, row, A.x_ld);
        if (A.z) R.load(zp, A.z, row, A.z_ld);
        if (GATE == 2) R.load(gp, A.gate, row, A.gate_ld);
        R.get(xp, y);
        if (A.z) {
            float u[NCH][VEC];
            R.get(zp, u);
            if (A.post) {
                R.normalise(u, A);
                EACH(NCH, VEC) u[j][e] = u[j][e] * w1[j][e] + b1[j][e];
            }
            if (GATE == 2) {
                R.get(gp, gc);
                R.open(gc, A.act);
            }
            if (GATE) EACH(NCH, VEC) u[j][e] *= gc[j][e];
            EACH(NCH, VEC) y[j][e] = A.scale * y[j][e] + u[j][e];
            if (live) R.template store<S>(A.y, row, A.y_ld, y);
        }
        if (A.pre) {
            R.normalise(y, A);
            EACH(NCH, VEC) y[j][e] = y[j][e] * w2[j][e] + b2[j][e];
            if (live) R.template store<T>(A.h, row, A.h_ld, y);
        }
    }
}

template <typename S, typename T, int VEC, int NCH, bool BLK, int GATE>
__global__ __launch_bounds__(!BLK ? NORM_T : NCH > 1 ? NORM_MAX_T / 2 : NORM_MAX_T) void residual_norm_backward_kernel(NormArgs A) {
    __shared__ float red[BLK ? 4 * NORM_MAX_T / 64 : 1];
    __shared__ float fold[BLK ? 1 : NORM_T * VEC];
    Row<VEC, NCH, BLK> R(A, red);
    float w2[NCH][VEC], w1[NCH][VEC], b1[NCH][VEC], gc[NCH][VEC], acc[SUMS][NCH][VEC];
    R.param(A.post ? A.post_w : nullptr, A.param_type, 1.f, w1);
    R.param(A.post ? A.post_b : nullptr, A.param_type, 0.f, b1);
    R.param(A.pre ? A.pre_w : nullptr, A.param_type, 1.f, w2);
    if (GATE == 1) {
        R.param(A.gate, A.param_type, 1.f, gc);
        R.open(gc, A.act);
    }
#pragma unroll
    for (int k = 0; k < SUMS; ++k) EACH(NCH, VEC) acc[k][j][e] = 0.f;
    const bool pre = A.pre && A.dh, reads_z = A.post || GATE;
    const int64_t stride = (int64_t)gridDim.x * R.rows;
    for (int64_t base = (int64_t)blockIdx.x * R.rows; base < A.n; base += stride) {
        const bool live = BLK || base + R.mine < A.n;
        const int64_t row = live ? base + R.mine : A.n - 1;
        Piece<S, VEC> dyp[NCH], yp[NCH];
        Piece<T, VEC> dhp[NCH], zp[NCH], gp[NCH];
        float dt[NCH][VEC];
        if (pre) {
            R.load(yp, A.x, row, A.x_ld);
            R.load(dhp, A.dh, row, A.dh_ld);
        }
        if (A.dy) R.load(dyp, A.dy, row, A.dy_ld);
        if (reads_z) R.load(zp, A.z, row, A.z_ld);
        if (GATE == 2) R.load(gp, A.gate, row, A.gate_ld);
        if (pre) {
            float y[NCH][VEC];
            R.get(yp, y);
            R.get(dhp, dt);
            const float r = R.normalise(y, A);
            if (live) EACH(NCH, VEC) {
                acc[SUM_PRE_W][j][e] += dt[j][e] * y[j][e];
                acc[SUM_PRE_B][j][e] += dt[j][e];
            }
            EACH(NCH, VEC) dt[j][e] *= w2[j][e];
            R.gradient(dt, y, A, r);
            if (A.dy) {
                float dy[NCH][VEC];
                R.get(dyp, dy);
                EACH(NCH, VEC) dt[j][e] += dy[j][e];
            }
        } else {
            R.get(dyp, dt);  // (one of the two gradients is there)
        }
        if (A.dx && live) {
            float dx[NCH][VEC];
            EACH(NCH, VEC) dx[j][e] = A.scale * dt[j][e];
            R.template store<S>(A.dx, row, A.dx_ld, dx);
        }
        if (!A.z) continue;
        float z[NCH][VEC], r = 1.f;
        if (reads_z) R.get(zp, z);
        if (A.post) r = R.normalise(z, A);
        if (GATE) {
            float u[NCH][VEC];
            if (A.post) EACH(NCH, VEC) u[j][e] = z[j][e] * w1[j][e] + b1[j][e];
            else EACH(NCH, VEC) u[j][e] = z[j][e];
            EACH(NCH, VEC) u[j][e] *= dt[j][e];  // gradient of act(g)
            if (GATE == 1) {
                if (live) EACH(NCH, VEC) acc[SUM_GATE][j][e] += u[j][e];
            } else {
                R.get(gp, gc);
                if (A.act == MARIUS_ACT_SIGMOID) {
                    EACH(NCH, VEC) u[j][e] *= sigmoid_slope(gc[j][e]);
                } else if (A.act == MARIUS_ACT_RELU) {
                    EACH(NCH, VEC) u[j][e] = gc[j][e] <= 0.f ? 0.f : u[j][e];
                    R.open(gc, A.act);
                }
                if (live) R.template store<T>(A.dgate, row, A.dgate_ld, u);
            }
            EACH(NCH, VEC) dt[j][e] *= gc[j][e];
        }
        if (A.post) {
            if (live) EACH(NCH, VEC) {
                acc[SUM_POST_W][j][e] += dt[j][e] * z[j][e];
                acc[SUM_POST_B][j][e] += dt[j][e];
            }
            EACH(NCH, VEC) dt[j][e] *= w1[j][e];
            R.gradient(dt, z, A, r);
        }
        if (live) R.template store<T>(A.dz, row, A.dz_ld, dt);
    }
    // this workgroup's sums: lanes that own the same columns are added in a fixed order
#pragma unroll
    for (int k = 0; k < SUMS; ++k) {
        if (!(A.want >> k & 1)) continue;  // (uniform)
        float* out = A.partial + ((int64_t)blockIdx.x * SUMS + k) * A.d;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            if (BLK) {
                put<float, VEC>(out + R.at[j], acc[k][j]);
            } else {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < VEC; ++e) fold[threadIdx.x * VEC + e] = acc[k][j][e];
                __syncthreads();
                if (R.mine == 0) {
                    float s[VEC];
#pragma unroll
                    for (int e = 0; e < VEC; ++e) s[e] = 0.f;
                    for (int q = 0; q < R.rows; ++q)
#pragma unroll
                        for (int e = 0; e < VEC; ++e) s[e] += fold[(q * R.tpr + R.lane) * VEC + e];
                    put<float, VEC>(out + R.at[j], s);
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
// 32 columns x 32 slices of the workgroups: a slice adds its workgroups in order, the slices are added in order
__global__ __launch_bounds__(1024) void residual_norm_sums_kernel(NormSumArgs A) {
    __shared__ float red[1024];
    const int k = blockIdx.y, c = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
    if (!(A.want >> k & 1)) return;  // (uniform)
    float s = 0.f;
    if (c < A.d)
#pragma unroll 8
        for (int w = slice; w < A.nwg; w += 32) s += A.partial[((int64_t)w * SUMS + k) * A.d + c];
    red[threadIdx.x] = s;
    __syncthreads();
    if (slice == 0 && c < A.d) {
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < 32; ++q) t += red[q * 32 + threadIdx.x];
        if (k == SUM_GATE) {
            t *= gate_slope(element_any(A.gate, A.type, c), A.act);
        }
        element_store_any(A.out[k], A.type, c, t);
    }
}

// A row of up to 64 pieces of four elements stays in one wave, several of them side by side where they are short (160,000 rows of 100 back: 82 us, a workgroup for each 268); a
// longer one takes a workgroup of as many waves as hold it, and beyond 4096 elements four pieces a lane.  (Two pieces in twice the lanes: 50,000 rows of 8192 in bf16 back
// 1040 us against 969, with a channel gate 1429 against 1519; 40,000 of 5000 forward 319 against 385, back 696 against 664.)
struct NormShape {
    int vec, tpr, nch, threads;
    bool blk;
};
static NormShape norm_shape(int d) {
    NormShape s{d < 4 ? 1 : 4, 1, 1, NORM_T, false};
    const int units = (int)cdiv(d, s.vec);
    s.blk = units > 64;
    if (s.blk) {
        s.nch = units > NORM_MAX_T ? 4 : 1;
        s.threads = s.tpr = (int)cdiv(cdiv(units, s.nch), 64) * 64;
    } else {
        while (s.tpr < units) s.tpr <<= 1;
    }
    return s;
}
static unsigned norm_groups(const NormShape& s, int64_t n, int most) {
    const int64_t groups = cdiv(n, s.blk ? 1 : NORM_T / s.tpr);
    return (unsigned)(groups < most ? groups : most);
}

template <typename S, typename T, int GATE>
static void launch_norm_gated(const NormArgs& A, const NormShape& s, bool backward, unsigned grid, hipStream_t st) {
    const dim3 g(grid), b(s.threads);
    if (backward) {
        if (s.vec == 1) residual_norm_backward_kernel<S, T, 1, 1, false, GATE><<<g, b, 0, st>>>(A);
        else if (!s.blk) residual_norm_backward_kernel<S, T, 4, 1, false, GATE><<<g, b, 0, st>>>(A);
        else if (s.nch == 1) residual_norm_backward_kernel<S, T, 4, 1, true, GATE><<<g, b, 0, st>>>(A);
        else residual_norm_backward_kernel<S, T, 4, 4, true, GATE><<<g, b, 0, st>>>(A);
    } else {
        if (s.vec == 1) residual_norm_kernel<S, T, 1, 1, false, GATE><<<g, b, 0, st>>>(A);
        else if (!s.blk) residual_norm_kernel<S, T, 4, 1, false, GATE><<<g, b, 0, st>>>(A);
        else if (s.nch == 1) residual_norm_kernel<S, T, 4, 1, true, GATE><<<g, b, 0, st>>>(A);
        else residual_norm_kernel<S, T, 4, 4, true, GATE><<<g, b, 0, st>>>(A);
    }
}
template <typename S, typename T>
static void launch_norm(const NormArgs& A, const NormShape& s, bool backward, unsigned grid, hipStream_t st) {
    if (A.gate_mode == 0) launch_norm_gated<S, T, 0>(A, s, backward, grid, st);
    else if (A.gate_mode == 1) launch_norm_gated<S, T, 1>(A, s, backward, grid, st);
    else launch_norm_gated<S, T, 2>(A, s, backward, grid, st);
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
    const NormShape s = norm_shape(A.d);
    A.tpr = s.tpr;
    launch_norm_typed(A, s, m->stream_type, m->type, false, norm_groups(s, A.n, 2048), as_stream(stream));
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
        const NormShape s = norm_shape(A.d);
        A.tpr = s.tpr;
        nwg = (int)norm_groups(s, A.n, NORM_MAX_WG);
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
        residual_norm_sums_kernel<<<dim3((unsigned)cdiv(A.d, 32), SUMS), dim3(1024), 0, st>>>(S);
    }
    return check_launch("residual_norm_backward");
}
