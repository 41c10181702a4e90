// AdamW over many tensors in one launch, its two moments in fp32 or in 8 bits.
//
//     g = gradient (* *grad_scale)            m = beta1 m + (1 - beta1) g            v = beta2 v + (1 - beta2) g g
//     p = p (1 - lr wd) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// 8-bit states: blocks of 256 elements with one fp32 scale each.  m is held as e4m3 times its block's scale; of v the ROOT is held (what the step divides
// by), e4m3 times its scale: e4m3 reaches 2^18 down from a block's largest value, which for the root is 2^36 of v.  A root above zero never becomes zero (it
// stays at the type's smallest value): a weight whose gradients are tiny beside its block's would otherwise be divided by eps alone.  scale = largest / 448,
// the type's largest value; a block whose largest magnitude is below 2^-100 is zero (its reciprocal would leave fp32).  The step itself uses the new
// moments before they are rounded.  All of it is single fp32 operations in the order written (no contraction): moments, codes and scales have the
// bits of any other program that does them in this order; the parameter's quotient is a product with a reciprocal within a step of fp32.
//
// Bound by HBM: 28 bytes an element with fp32 states, 16.1 with 8-bit ones (fp32 parameters and gradients).  A workgroup takes tiles of 2048 elements, eight
// per lane (16-byte loads of every stream; the 32 lanes of a block share its scale by shuffles), and finds its tensor by binary search: up to 64 tensors in
// the launch's own arguments, more in a table that short launches copy from theirs into the workspace of this call (300 tensors, 20 M elements in 8 bits: 56 us
// against 86 with a launch for every 64 tensors, each of which fills and drains the card anew; 200 M elements in fp32: 1072 us, 5.2 TB/s).
// With the step's number on the device one lane of a workgroup takes the two factors behind the loads: the times are those of a number on the host (in every lane, the 300
// tensors in 8 bits took 7 us more).
#include "row_types.h"

namespace marius {

constexpr int AW_T = 256, AW_EPT = 8, AW_TILE = AW_T * AW_EPT, AW_TENSORS = 64, AW_BLOCK = 256;

struct AwTensor {
    void* p;
    const void* g;
    void *m, *v;
    float *ms, *vs;
    int64_t n;
};
struct AwTable {
    AwTensor t[AW_TENSORS];
    int first[AW_TENSORS];        // first tile of every tensor
    uint16_t number[AW_TENSORS];  // its number in the caller's list, behind the part's first
};
struct AwStep {
    int count, steps;           // steps: 0, one number for all tensors on the device; 1, one for each
    float decay, rate, beta1, omb1, beta2, omb2, inv_root, eps;
    const float* grad_scale;
    const int64_t* step_dev;    // the steps' numbers on the device: rate and inv_root are taken from them
    double lr, beta1_d, beta2_d;
};
static_assert(sizeof(AwTable) + sizeof(AwStep) <= 4096, "kernel arguments");

// a part of the table, from the launch's arguments to memory: tensors [at, at + count)
__global__ __launch_bounds__(64) void adamw_table_kernel(AwTable P, int count, int at, int base, AwTensor* __restrict__ t, int* __restrict__ first, int* __restrict__ number) {
    const int i = threadIdx.x;
    if (i >= count) return;
    t[at + i] = P.t[i];
    first[at + i] = P.first[i];
    number[at + i] = base + P.number[i];
}

template <typename X>
__device__ __forceinline__ void aw_load(const X* p, int64_t i, int left, float (&v)[AW_EPT]) {
    if (left >= AW_EPT) {
        X t[AW_EPT];
        __builtin_memcpy(t, p + i, sizeof(t));
#pragma unroll
        for (int e = 0; e < AW_EPT; ++e) v[e] = (float)t[e];
    } else {
#pragma unroll
        for (int e = 0; e < AW_EPT; ++e) v[e] = e < left ? (float)p[i + e] : 0.f;
    }
}
template <typename X>
__device__ __forceinline__ void aw_store(X* p, int64_t i, int left, const float (&v)[AW_EPT]) {
    if (left >= AW_EPT) {
        X t[AW_EPT];
#pragma unroll
        for (int e = 0; e < AW_EPT; ++e) t[e] = (X)v[e];
        __builtin_memcpy(p + i, t, sizeof(t));
    } else {
#pragma unroll
        for (int e = 0; e < AW_EPT; ++e)
            if (e < left) p[i + e] = (X)v[e];
    }
}
// eight e4m3 codes <-> floats (the conversions round to nearest even)
__device__ __forceinline__ void aw_load8(const uint8_t* p, int64_t i, int left, float (&v)[AW_EPT]) {
    uint8_t c[AW_EPT] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (left >= AW_EPT) __builtin_memcpy(c, p + i, sizeof(c));
    else
#pragma unroll
        for (int e = 0; e < AW_EPT; ++e)
            if (e < left) c[e] = p[i + e];
    int w[2];
    __builtin_memcpy(w, c, sizeof(w));
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w[q], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w[q], true);
        v[4 * q] = a[0];
        v[4 * q + 1] = a[1];
        v[4 * q + 2] = b[0];
        v[4 * q + 3] = b[1];
    }
}
__device__ __forceinline__ void aw_store8(uint8_t* p, int64_t i, int left, const float (&v)[AW_EPT]) {
    int w[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        w[q] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * q], v[4 * q + 1], 0, false);
        w[q] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * q + 2], v[4 * q + 3], w[q], true);
    }
    uint8_t c[AW_EPT];
    __builtin_memcpy(c, w, sizeof(c));
    if (left >= AW_EPT) __builtin_memcpy(p + i, c, sizeof(c));
    else
#pragma unroll
        for (int e = 0; e < AW_EPT; ++e)
            if (e < left) p[i + e] = c[e];
}
// a block's 32 lanes: largest |x| -> the scale to keep and the factor that takes x to e4m3's range
__device__ __forceinline__ void aw_scale(const float (&x)[AW_EPT], float& scale, float& inv) {
#pragma clang fp contract(off)
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < AW_EPT; ++e) top = fmaxf(top, fabsf(x[e]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if (top < 0x1p-100f) top = 0.f;
    scale = top * (1.f / 448.f);
    inv = top > 0.f ? (1.f / top) * 448.f : 0.f;
}

__device__ __forceinline__ int aw_find(const int* first, int count, int tile) {
    int lo = 0, hi = count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= tile) lo = mid;
        else hi = mid;
    }
    return lo;
}
template <typename P, typename G, bool BITS8>
__device__ __forceinline__ void adamw_tile(const AwStep& A, const AwTensor& t, int tile, int number) {
#pragma clang fp contract(off)
    const int64_t i = (int64_t)tile * AW_TILE + (int)threadIdx.x * AW_EPT;
    const int left = t.n - i >= AW_EPT ? AW_EPT : t.n > i ? (int)(t.n - i) : 0;
    float rate = A.rate, inv_root = A.inv_root;
    const float gs = A.grad_scale ? *A.grad_scale : 1.f;
    float p[AW_EPT], g[AW_EPT], m[AW_EPT], v[AW_EPT], r[AW_EPT];
    aw_load<P>((const P*)t.p, i, left, p);
    aw_load<G>((const G*)t.g, i, left, g);
    if (BITS8) {
        aw_load8((const uint8_t*)t.m, i, left, m);
        aw_load8((const uint8_t*)t.v, i, left, v);
        const float sm = left > 0 ? t.ms[i / AW_BLOCK] : 0.f, sv = left > 0 ? t.vs[i / AW_BLOCK] : 0.f;
#pragma unroll
        for (int e = 0; e < AW_EPT; ++e) {
            m[e] = m[e] * sm;
            v[e] = v[e] * sv;
            v[e] = v[e] * v[e];
        }
    } else {
        aw_load<float>((const float*)t.m, i, left, m);
        aw_load<float>((const float*)t.v, i, left, v);
    }
    if (A.step_dev) {  // (uniform) one lane takes the powers of 64 bits while the loads are under way
        __shared__ float factors[2];
        if (threadIdx.x == 0) {
            const double step = (double)A.step_dev[A.steps ? number : 0];
            factors[0] = (float)(A.lr / (1.0 - pow(A.beta1_d, step)));
            factors[1] = (float)(1.0 / sqrt(1.0 - pow(A.beta2_d, step)));
        }
        __syncthreads();
        rate = factors[0];
        inv_root = factors[1];
    }
#pragma unroll
    for (int e = 0; e < AW_EPT; ++e) {
        if (A.grad_scale) g[e] = g[e] * gs;
        m[e] = m[e] * A.beta1 + g[e] * A.omb1;
        v[e] = v[e] * A.beta2 + (g[e] * A.omb2) * g[e];
        r[e] = sqrtf(v[e]);
        p[e] = p[e] * A.decay - rate * (m[e] * __builtin_amdgcn_rcpf(r[e] * inv_root + A.eps));  // (a reciprocal within a step of fp32)
    }
    aw_store<P>((P*)t.p, i, left, p);
    if (BITS8) {
        float scale, inv;
        aw_scale(m, scale, inv);  // (every lane takes part: elements behind the tensor are zero)
        float rscale, rinv;
        aw_scale(r, rscale, rinv);
        if (left > 0 && (threadIdx.x & 31) == 0) {
            t.ms[i / AW_BLOCK] = scale;
            t.vs[i / AW_BLOCK] = rscale;
        }
#pragma unroll
        for (int e = 0; e < AW_EPT; ++e) {
            m[e] = m[e] * inv;
            r[e] = r[e] * rinv;
            if (r[e] > 0.f && r[e] < 0x1p-9f) r[e] = 0x1p-9f;
        }
        aw_store8((uint8_t*)t.m, i, left, m);
        aw_store8((uint8_t*)t.v, i, left, r);
    } else {
        aw_store<float>((float*)t.m, i, left, m);
        aw_store<float>((float*)t.v, i, left, v);
    }
}

template <typename P, typename G, bool BITS8>
__global__ __launch_bounds__(AW_T) void adamw_kernel(AwTable P_, AwStep A) {
    const int k = aw_find(P_.first, A.count, (int)blockIdx.x);
    adamw_tile<P, G, BITS8>(A, P_.t[k], (int)blockIdx.x - P_.first[k], P_.number[k]);
}
template <typename P, typename G, bool BITS8>
__global__ __launch_bounds__(AW_T) void adamw_many_kernel(const AwTensor* __restrict__ t, const int* __restrict__ first, const int* __restrict__ number, AwStep A) {
    const int k = aw_find(first, A.count, (int)blockIdx.x);
    adamw_tile<P, G, BITS8>(A, t[k], (int)blockIdx.x - first[k], number[k]);
}

// one launch over the tensors of `table` (up to 64), or over those of the table in memory: t, then first, then number
template <typename P, typename G, bool BITS8>
static void launch_adamw(const AwTable* table, const AwTensor* t, const int* first, const AwStep& A, unsigned tiles, hipStream_t st) {
    if (table) adamw_kernel<P, G, BITS8><<<dim3(tiles), dim3(AW_T), 0, st>>>(*table, A);
    else adamw_many_kernel<P, G, BITS8><<<dim3(tiles), dim3(AW_T), 0, st>>>(t, first, first + A.count, A);
}
template <typename P, typename G>
static void launch_adamw_bits(bool bits8, const AwTable* table, const AwTensor* t, const int* first, const AwStep& A, unsigned tiles, hipStream_t st) {
    if (bits8) launch_adamw<P, G, true>(table, t, first, A, tiles, st);
    else launch_adamw<P, G, false>(table, t, first, A, tiles, st);
}
template <typename P>
static void launch_adamw_grad(int grad_type, bool bits8, const AwTable* table, const AwTensor* t, const int* first, const AwStep& A, unsigned tiles, hipStream_t st) {
    if (grad_type == MARIUS_F32) launch_adamw_bits<P, float>(bits8, table, t, first, A, tiles, st);
    else if (grad_type == MARIUS_BF16) launch_adamw_bits<P, __bf16>(bits8, table, t, first, A, tiles, st);
    else launch_adamw_bits<P, _Float16>(bits8, table, t, first, A, tiles, st);
}
static void launch_adamw_typed(int param_type, int grad_type, bool bits8, const AwTable* table, const AwTensor* t, const int* first, const AwStep& A, unsigned tiles, hipStream_t st) {
    if (param_type == MARIUS_F32) launch_adamw_grad<float>(grad_type, bits8, table, t, first, A, tiles, st);
    else if (param_type == MARIUS_BF16) launch_adamw_grad<__bf16>(grad_type, bits8, table, t, first, A, tiles, st);
    else launch_adamw_grad<_Float16>(grad_type, bits8, table, t, first, A, tiles, st);
}

}  // namespace marius

using namespace marius;

extern "C" size_t marius_adamw_workspace_bytes(int32_t count) { return count > AW_TENSORS ? (size_t)count * (sizeof(AwTensor) + 2 * sizeof(int)) : 0; }

extern "C" int marius_adamw_check(const marius_adamw_tensor* tensors, int32_t count, int32_t param_type, int32_t grad_type, int32_t state_bits, int64_t step,
                                  const int64_t* step_dev, int32_t step_count, double lr, double beta1, double beta2, double eps, double weight_decay) {
    MARIUS_REQUIRE(count >= 0 && (count == 0 || tensors), "adamw_step: bad tensor list");
    MARIUS_REQUIRE(float_type_ok(param_type) && float_type_ok(grad_type), "adamw_step: types are MARIUS_F32 / BF16 / F16");
    MARIUS_REQUIRE(state_bits == 32 || state_bits == 8, "adamw_step: states are held in 32 or in 8 bits");
    MARIUS_REQUIRE(step_dev || step >= 1, "adamw_step: steps are counted from 1");
    MARIUS_REQUIRE(!step_dev || step_count == 1 || step_count == count, "adamw_step: one step on the device, or one for each tensor");
    MARIUS_REQUIRE(lr >= 0 && beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && weight_decay >= 0, "adamw_step: lr, eps, weight_decay >= 0, betas in [0, 1)");
    int64_t tiles = 0;
    for (int k = 0; k < count; ++k) {
        const marius_adamw_tensor& s = tensors[k];
        MARIUS_REQUIRE(s.n >= 0, "adamw_step: bad size of tensor %d", k);
        if (s.n == 0) continue;
        MARIUS_REQUIRE(s.param && s.grad && s.exp_avg && s.exp_avg_sq && (state_bits == 32 || (s.exp_avg_scale && s.exp_avg_sq_scale)), "adamw_step: null pointer in tensor %d", k);
        const int64_t more = cdiv(s.n, AW_TILE);
        MARIUS_REQUIRE(tiles + more < (1ll << 24), "adamw_step: over 2^35 elements in one call");  // (a launch holds less than 2^32 lanes)
        tiles += more;
    }
    return MARIUS_OK;
}

extern "C" int marius_adamw_step(const marius_adamw_tensor* tensors, int32_t count, int32_t param_type, int32_t grad_type, int32_t state_bits, int64_t step,
                                 const int64_t* step_dev, int32_t step_count, double lr, double beta1, double beta2, double eps, double weight_decay, const float* grad_scale,
                                 void* workspace, size_t workspace_bytes, marius_stream_t stream) {
    // before anything is launched: a refused list leaves every tensor as it was
    const int rc = marius_adamw_check(tensors, count, param_type, grad_type, state_bits, step, step_dev, step_count, lr, beta1, beta2, eps, weight_decay);
    if (rc) return rc;
    int live = 0, last = 0;
    for (int k = 0; k < count; ++k)
        if (tensors[k].n > 0) {
            ++live;
            last = k;
        }
    if (live == 0) return MARIUS_OK;
    const bool many = live > AW_TENSORS || last > UINT16_MAX;
    MARIUS_REQUIRE(!many || (workspace && workspace_bytes >= marius_adamw_workspace_bytes(count)), "adamw_step: workspace too small");
    hipStream_t st = as_stream(stream);
    AwTensor* t_dev = (AwTensor*)workspace;
    int* first_dev = many ? (int*)(t_dev + live) : nullptr;
    AwStep A;
    A.decay = (float)(1.0 - lr * weight_decay);
    A.rate = step_dev ? 0.f : (float)(lr / (1.0 - std::pow(beta1, (double)step)));
    A.inv_root = step_dev ? 0.f : (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
    A.beta1 = (float)beta1;
    A.omb1 = (float)(1.0 - beta1);
    A.beta2 = (float)beta2;
    A.omb2 = (float)(1.0 - beta2);
    A.eps = (float)eps;
    A.grad_scale = grad_scale;
    A.step_dev = step_dev;
    A.steps = step_count > 1;
    A.lr = lr;
    A.beta1_d = beta1;
    A.beta2_d = beta2;
    A.count = live;
    AwTable T{};
    int filled = 0, at = 0, base = 0;
    int64_t tiles = 0;
    auto send = [&] {
        adamw_table_kernel<<<dim3(1), dim3(64), 0, st>>>(T, filled, at, base, t_dev, first_dev, first_dev + live);
        at += filled;
        filled = 0;
    };
    for (int k = 0; k < count; ++k) {
        const marius_adamw_tensor& s = tensors[k];
        if (s.n == 0) continue;
        if (many && filled > 0 && (filled == AW_TENSORS || k - base > UINT16_MAX)) send();
        if (many && filled == 0) base = k;
        T.number[filled] = (uint16_t)(k - base);
        T.t[filled] = AwTensor{s.param, s.grad, s.exp_avg, s.exp_avg_sq, s.exp_avg_scale, s.exp_avg_sq_scale, s.n};
        T.first[filled++] = (int)tiles;
        tiles += cdiv(s.n, AW_TILE);
    }
    if (many) send();
    launch_adamw_typed(param_type, grad_type, state_bits == 8, many ? nullptr : &T, t_dev, first_dev, A, (unsigned)tiles, st);
    return check_launch("adamw_step");
}
