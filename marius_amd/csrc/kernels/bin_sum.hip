// Sums of rows by a small number of bins: out[b, h] = sum of g[e, h] over the entries e with bin[e] = b.  The gradient of a table of biases (a row for each
// relation) that many entries of an attention share.
//
// Every lane has its own sums of all bins, a column of LDS: no atomics, no sort, and the same bits on every run (a lane's entries in order, then the lanes of a
// workgroup in order, then the workgroups by a second launch).  A workgroup is one wave: 64 / H entries of H heads side by side, so a load is 64 neighbouring elements.
// Measured: 1.5 M entries of 8 heads over 6 bins 27 us (2.2 TB/s), over 200 bins 55 us, 900,000 of 16 over 41 34 us, up to 200,000 entries 17 us (two launches).
// That is below the 4.76 TB/s of a large copy: a lane has eight loads in flight, then adds them to its sums in LDS one after another; with many bins, LDS leaves few
// waves besides (256 bytes a bin, so up to 256 bins).
#include "common.h"

namespace marius {

constexpr int BIN_MAX = 256, BIN_MAX_WG = 2048, BIN_UN = 8;

// entries per workgroup and workgroups: as many waves as find room in LDS (160 KB a compute unit), with some work each
static int64_t bin_groups(int64_t T, int bins) {
    const int64_t room = 256 * (640 / bins < 8 ? 640 / bins : 8), want = cdiv(T, 256);
    const int64_t most = room < BIN_MAX_WG ? room : BIN_MAX_WG;
    return want < 1 ? 1 : want < most ? want : most;
}

__global__ __launch_bounds__(64) void bin_sum_kernel(const float* __restrict__ g, const int64_t* __restrict__ bin, int64_t T, int64_t per, int H, int bins, float* __restrict__ partial) {
    extern __shared__ float sums[];  // [bins][64]
    const int lane = threadIdx.x, h0 = blockIdx.y * 64, heads = H - h0 < 64 ? H - h0 : 64, slots = 64 / heads, slot = lane / heads, h = h0 + lane - slot * heads;
    for (int b = 0; b < bins; ++b) sums[b * 64 + lane] = 0.f;
    const int64_t from = blockIdx.x * per, to = from + per < T ? from + per : T;
    if (slot < slots) {
        for (int64_t t = from + slot; t < to; t += slots * BIN_UN) {
            float v[BIN_UN];
            int at[BIN_UN];
#pragma unroll
            for (int u = 0; u < BIN_UN; ++u) {
                const int64_t e = t + u * slots < to ? t + u * slots : t;
                const int64_t b = bin[e];
                v[u] = g[e * H + h];
                at[u] = t + u * slots < to && b >= 0 && b < bins ? (int)b * 64 + lane : -1;  // (an entry of no bin is left out)
            }
#pragma unroll
            for (int u = 0; u < BIN_UN; ++u)
                if (at[u] >= 0) sums[at[u]] += v[u];
        }
    }
    __syncthreads();
    for (int i = lane; i < bins * heads; i += 64) {
        const int b = i / heads, hh = i - b * heads;
        float s = 0.f;
        for (int k = 0; k < slots; ++k) s += sums[b * 64 + k * heads + hh];
        partial[((int64_t)blockIdx.x * bins + b) * H + h0 + hh] = s;
    }
}

// 32 outputs a workgroup, 32 threads each over the partial sums
__global__ __launch_bounds__(1024) void bin_join_kernel(const float* __restrict__ partial, int groups, int64_t n, float* __restrict__ out) {
    __shared__ float red[32][33];
    const int o = threadIdx.x & 31, part = threadIdx.x >> 5;
    const int64_t i = (int64_t)blockIdx.x * 32 + o;
    float s = 0.f;
    if (i < n) {
#pragma unroll 8
        for (int p = part; p < groups; p += 32) s += partial[(int64_t)p * n + i];
    }
    red[part][o] = s;
    __syncthreads();
    if (part != 0 || i >= n) return;
    for (int p = 1; p < 32; ++p) s += red[p][o];
    out[i] = s;
}

}  // namespace marius

using namespace marius;

extern "C" size_t marius_bin_sum_workspace_bytes(int64_t T, int32_t heads, int32_t bins) {
    return T >= 0 && heads > 0 && bins > 0 && bins <= BIN_MAX ? (size_t)bin_groups(T, bins) * bins * heads * sizeof(float) : 0;
}

extern "C" int marius_bin_sum(const float* values, const int64_t* bin, int64_t T, int32_t heads, int32_t bins, float* out, void* workspace, size_t workspace_bytes,
                              marius_stream_t stream) {
    MARIUS_REQUIRE(T >= 0 && heads > 0 && heads <= 1024, "bin_sum: rows of 1 to 1024 elements");
    MARIUS_REQUIRE(bins > 0 && bins <= BIN_MAX, "bin_sum: 1 to %d bins", BIN_MAX);
    MARIUS_REQUIRE(out && (T == 0 || (values && bin)), "bin_sum: null pointer");
    MARIUS_REQUIRE(workspace && workspace_bytes >= marius_bin_sum_workspace_bytes(T, heads, bins), "bin_sum: workspace too small");
    const int64_t groups = bin_groups(T, bins), n = (int64_t)bins * heads;
    hipStream_t st = as_stream(stream);
    bin_sum_kernel<<<dim3((unsigned)groups, (unsigned)cdiv(heads, 64)), dim3(64), (size_t)bins * 64 * sizeof(float), st>>>(values, bin, T, cdiv(T, groups), heads, bins,
                                                                                                                              (float*)workspace);
    bin_join_kernel<<<dim3((unsigned)cdiv(n, 32)), dim3(1024), 0, st>>>((const float*)workspace, (int)groups, n, out);
    return check_launch("bin_sum");
}
