// The lists of a neighbour attention in both directions, made once for a graph (a sampled batch, or a whole graph that many passes use) and checked:
// every kernel that walks a plan may take its entries as they are.
//
//   marius_nbr_plan_lists    one list per target out of up to three parts — list a, list b (outgoing + incoming), the target's own row — as 32-bit offsets,
//                            row indices and owners, with the checks (ascending offsets that cover their list, indices inside the rows)
//   marius_nbr_plan_reverse  the same entries grouped by row (from marius_sort_unique over the row indices, which keeps their order): the backward
//                            pass sums a row's gradients over its own list, no atomics
//   marius_nbr_plan_items    work items of at most `chunk` entries: a list longer than that is split, its parts get slots for partial results; the longest
//                            items first, in list order among those of one length: items side by side in a wave end together, and none starts last that
//                            lasts long (a training pass over 200,000 entries 100 -> 84 us, over 1.5 M of a power-law graph 1048 -> 994 us)
//
// Bound by latency: 31 short launches (for 900,000 entries 285 us of kernels, 127 of them the sort of the reverse lists) and two readbacks (status, counts).  The plan of 64 targets with 15 entries 204 us, of 900,000 entries
// over 800,000 rows 341 us, of 1.5 M entries 430 us, where their bytes (each list read once, the entries written in both directions) take 0, 7 and 7 us at the rate of a copy: a
// plan pays where several passes use it.  4-byte entries, because every pass over the graph reads them.
#include "common.h"

namespace marius {

constexpr int NP_T = 256, NP_ITEMS = 4, NP_TILE = NP_T * NP_ITEMS;

struct NpLists {
    const int64_t *index_a, *offsets_a, *index_b, *offsets_b;
    int64_t T_a, T_b, n, rows, self_offset;
};
// length of target i's list; *bad: offsets that do not ascend from 0 to the list's length
__device__ __forceinline__ int64_t np_part(const int64_t* offsets, int64_t T, int64_t n, int64_t i, int64_t& start, bool& bad) {
    if (!offsets) {
        start = 0;
        return 0;
    }
    start = offsets[i];
    const int64_t end = i + 1 < n ? offsets[i + 1] : T;
    if (start < 0 || end < start || end > T || (i == 0 && start != 0)) {
        bad = true;
        return 0;
    }
    return end - start;
}
__device__ __forceinline__ int64_t np_degree(const NpLists& L, int64_t i, bool& bad) {
    int64_t s;
    return np_part(L.offsets_a, L.T_a, L.n, i, s, bad) + np_part(L.offsets_b, L.T_b, L.n, i, s, bad) + (L.self_offset >= 0 ? 1 : 0);
}

// the value of element i that the scans below add up: three counters, the last two used by the items only
struct NpCount {
    int32_t v[3];
};
struct NpSource {
    NpLists lists;          // mode 0: v[0] = length of list i
    const int32_t* offsets; // mode 1: v = (work items, slots, split lists) of list i
    int64_t n;
    int mode, chunk;
    int32_t* status;
};
__device__ __forceinline__ NpCount np_value(const NpSource& S, int64_t i) {
    NpCount c{{0, 0, 0}};
    if (i >= S.n) return c;
    if (S.mode == 0) {
        bool bad = false;
        c.v[0] = (int32_t)np_degree(S.lists, i, bad);
        if (bad) atomicOr(S.status, 1);
    } else {
        const int len = S.offsets[i + 1] - S.offsets[i], parts = len > S.chunk ? (len + S.chunk - 1) / S.chunk : 1;
        c.v[0] = parts;
        c.v[1] = parts > 1 ? parts : 0;
        c.v[2] = parts > 1 ? 1 : 0;
    }
    return c;
}
__global__ __launch_bounds__(NP_T) void np_tile_sums_kernel(NpSource S, int32_t* __restrict__ tiles) {
    __shared__ int32_t red[3 * NP_T / 64];
    NpCount mine{{0, 0, 0}};
    for (int r = 0; r < NP_ITEMS; ++r) {
        const NpCount c = np_value(S, (int64_t)blockIdx.x * NP_TILE + r * NP_T + threadIdx.x);
        for (int k = 0; k < 3; ++k) mine.v[k] += c.v[k];
    }
    for (int o = 32; o > 0; o >>= 1)
        for (int k = 0; k < 3; ++k) mine.v[k] += __shfl_xor(mine.v[k], o, 64);
    if ((threadIdx.x & 63) == 0)
        for (int k = 0; k < 3; ++k) red[3 * (threadIdx.x >> 6) + k] = mine.v[k];
    __syncthreads();
    if (threadIdx.x < 3) {
        int32_t s = 0;
        for (int w = 0; w < NP_T / 64; ++w) s += red[3 * w + threadIdx.x];
        tiles[3 * blockIdx.x + threadIdx.x] = s;
    }
}
// exclusive scan of the tiles' sums in place, one workgroup; the totals -> totals[0 .. 3)
__global__ __launch_bounds__(NP_T) void np_scan_tiles_kernel(int32_t* __restrict__ tiles, int ntiles, int32_t* __restrict__ totals) {
    __shared__ int32_t wsum[3][NP_T / 64];
    int32_t carry[3] = {0, 0, 0};
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int b = 0; b < ntiles; b += NP_T) {
        const int i = b + threadIdx.x;
        int32_t v[3], x[3];
        for (int k = 0; k < 3; ++k) x[k] = v[k] = i < ntiles ? tiles[3 * i + k] : 0;
        for (int o = 1; o < 64; o <<= 1)
            for (int k = 0; k < 3; ++k) {
                const int32_t y = __shfl_up(x[k], o, 64);
                if (lane >= o) x[k] += y;
            }
        __syncthreads();
        if (lane == 63)
            for (int k = 0; k < 3; ++k) wsum[k][wave] = x[k];
        __syncthreads();
        for (int k = 0; k < 3; ++k) {
            int32_t before = carry[k] + x[k] - v[k];
            for (int w = 0; w < wave; ++w) before += wsum[k][w];
            if (i < ntiles) tiles[3 * i + k] = before;
            for (int w = 0; w < NP_T / 64; ++w) carry[k] += wsum[k][w];
        }
    }
    if (threadIdx.x < 3) totals[threadIdx.x] = carry[threadIdx.x];
}
struct NpOut {
    int32_t* offsets;  // mode 0: [n + 1]
    int4 *items, *splits;  // mode 1: {list, first entry, end, slot or -1}, {list, first slot, parts, 0}
    int32_t max_items, max_splits;
};
__global__ __launch_bounds__(NP_T) void np_emit_kernel(NpSource S, const int32_t* __restrict__ tiles, NpOut O) {
    __shared__ int32_t wsum[3][NP_T / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t i0 = (int64_t)blockIdx.x * NP_TILE + (int64_t)threadIdx.x * NP_ITEMS;  // a thread's elements are consecutive
    NpCount c[NP_ITEMS];
    int32_t mine[3] = {0, 0, 0}, x[3];
    for (int r = 0; r < NP_ITEMS; ++r) {
        c[r] = np_value(S, i0 + r);
        for (int k = 0; k < 3; ++k) mine[k] += c[r].v[k];
    }
    for (int k = 0; k < 3; ++k) x[k] = mine[k];
    for (int o = 1; o < 64; o <<= 1)
        for (int k = 0; k < 3; ++k) {
            const int32_t y = __shfl_up(x[k], o, 64);
            if (lane >= o) x[k] += y;
        }
    if (lane == 63)
        for (int k = 0; k < 3; ++k) wsum[k][wave] = x[k];
    __syncthreads();
    int32_t at[3];
    for (int k = 0; k < 3; ++k) {
        at[k] = tiles[3 * blockIdx.x + k] + x[k] - mine[k];
        for (int w = 0; w < wave; ++w) at[k] += wsum[k][w];
    }
    for (int r = 0; r < NP_ITEMS; ++r) {
        const int64_t i = i0 + r;
        if (i < S.n) {
            if (S.mode == 0) {
                O.offsets[i] = at[0];
                if (i == S.n - 1) O.offsets[S.n] = at[0] + c[r].v[0];
            } else {
                const int t0 = S.offsets[i], t1 = S.offsets[i + 1], parts = c[r].v[0];
                for (int p = 0; p < parts; ++p)
                    if (at[0] + p >= 0 && at[0] + p < O.max_items)
                        O.items[at[0] + p] = make_int4((int)i, t0 + p * S.chunk, parts > 1 ? min(t1, t0 + (p + 1) * S.chunk) : t1, parts > 1 ? at[1] + p : -1);
                if (parts > 1 && at[2] >= 0 && at[2] < O.max_splits) O.splits[at[2]] = make_int4((int)i, at[1], parts, 0);
            }
        }
        for (int k = 0; k < 3; ++k) at[k] += c[r].v[k];
    }
}

// ---- items by length: a counting sort by class, stable.  Classes: blocks of four entries one by one up to eight, then in steps; class 0 is the longest
constexpr int NP_CLASSES = 16;
__device__ __forceinline__ int np_class(const int4& it) {
    const int b = (it.z - it.y + 3) >> 2;
    return 13 - (b <= 8 ? b : b <= 12 ? 9 : b <= 16 ? 10 : b <= 24 ? 11 : b <= 32 ? 12 : 13);
}
__global__ __launch_bounds__(NP_T) void np_class_counts_kernel(const int4* __restrict__ items, const int32_t* __restrict__ count, int max_items, int ntiles, int32_t* __restrict__ hist) {
    __shared__ int32_t h[NP_CLASSES];
    const int n = min(*count, max_items);
    if (threadIdx.x < NP_CLASSES) h[threadIdx.x] = 0;
    __syncthreads();
    for (int r = 0; r < NP_ITEMS; ++r) {
        const int i = blockIdx.x * NP_TILE + r * NP_T + threadIdx.x;
        if (i < n) atomicAdd(&h[np_class(items[i])], 1);
    }
    __syncthreads();
    if (threadIdx.x < NP_CLASSES) hist[threadIdx.x * ntiles + blockIdx.x] = h[threadIdx.x];
}
// exclusive scan in place, one workgroup
__global__ __launch_bounds__(NP_T) void np_scan_kernel(int32_t* __restrict__ v, int n) {
    __shared__ int32_t wsum[NP_T / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int32_t carry = 0;
    for (int b = 0; b < n; b += NP_T * NP_ITEMS) {
        int32_t own[NP_ITEMS], mine = 0;
        for (int r = 0; r < NP_ITEMS; ++r) {
            const int i = b + threadIdx.x * NP_ITEMS + r;
            own[r] = i < n ? v[i] : 0;
            mine += own[r];
        }
        int32_t x = mine;
        for (int o = 1; o < 64; o <<= 1) {
            const int32_t y = __shfl_up(x, o, 64);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 63) wsum[wave] = x;
        __syncthreads();
        int32_t at = carry + x - mine;
        for (int w = 0; w < wave; ++w) at += wsum[w];
        for (int w = 0; w < NP_T / 64; ++w) carry += wsum[w];
        for (int r = 0; r < NP_ITEMS; ++r) {
            const int i = b + threadIdx.x * NP_ITEMS + r;
            if (i < n) v[i] = at;
            at += own[r];
        }
    }
}
__global__ __launch_bounds__(NP_T) void np_class_place_kernel(const int4* __restrict__ items, const int32_t* __restrict__ count, int max_items, int ntiles,
                                                              const int32_t* __restrict__ hist, int4* __restrict__ out) {
    __shared__ int32_t base[NP_CLASSES], waves[NP_T / 64][NP_CLASSES];
    const int n = min(*count, max_items), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x < NP_CLASSES) base[threadIdx.x] = hist[threadIdx.x * ntiles + blockIdx.x];
    for (int r = 0; r < NP_ITEMS; ++r) {
        if (threadIdx.x < NP_T / 64 * NP_CLASSES) waves[threadIdx.x / NP_CLASSES][threadIdx.x % NP_CLASSES] = 0;
        __syncthreads();
        const int i = blockIdx.x * NP_TILE + r * NP_T + threadIdx.x;
        const bool in = i < n;
        int4 it = make_int4(0, 0, 0, 0);
        if (in) it = items[i];
        const int c = np_class(it);
        unsigned long long same = __ballot(in);  // lanes of this lane's class
        for (int b = 1; b < NP_CLASSES; b <<= 1) {
            const unsigned long long m = __ballot((c & b) != 0);
            same &= (c & b) ? m : ~m;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        if (in && rank == 0) waves[wave][c] = __popcll(same);
        __syncthreads();
        int32_t at = base[c] + rank;
        for (int w = 0; w < wave; ++w) at += waves[w][c];
        if (in && at >= 0 && at < max_items) out[at] = it;
        __syncthreads();
        if (threadIdx.x < NP_CLASSES)
            for (int w = 0; w < NP_T / 64; ++w) base[threadIdx.x] += waves[w][threadIdx.x];
        __syncthreads();
    }
}

// one thread per entry: its list by binary search in the offsets, its row from the part that it falls into
__global__ __launch_bounds__(256) void np_entries_kernel(NpLists L, const int32_t* __restrict__ offsets, int64_t T, int32_t* __restrict__ index, int32_t* __restrict__ owner,
                                                         int64_t* __restrict__ keys, int32_t* __restrict__ status) {
    for (int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; t < T; t += (int64_t)gridDim.x * blockDim.x) {
        int64_t lo = 0, hi = L.n;
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (offsets[mid] <= t) lo = mid;
            else hi = mid;
        }
        int64_t k = t - offsets[lo], start, row = -1;
        bool bad = false;
        const int64_t na = np_part(L.offsets_a, L.T_a, L.n, lo, start, bad);
        if (k < 0) {  // (lists that do not ascend: already reported)
            bad = true;
        } else if (k < na) {
            row = L.index_a[start + k];
        } else {
            k -= na;
            const int64_t nb = np_part(L.offsets_b, L.T_b, L.n, lo, start, bad);
            if (k < nb) row = L.index_b[start + k];
            else if (k - nb == 0 && L.self_offset >= 0) row = L.self_offset + lo;
        }
        if (row < 0 || row >= L.rows) {
            atomicOr(status, 2);
            row = 0;
        }
        index[t] = (int32_t)row;
        owner[t] = (int32_t)lo;
        keys[t] = row;
    }
}
__global__ __launch_bounds__(256) void np_check_total_kernel(const int32_t* __restrict__ offsets, int64_t n, int64_t T, int32_t* __restrict__ status) {
    if (n > 0 && offsets[n] != T) atomicOr(status, 1);
}

// offsets of the reverse lists: the first run whose key is >= j starts row j's list
__global__ __launch_bounds__(256) void np_reverse_offsets_kernel(const int64_t* __restrict__ uniq, const int32_t* __restrict__ seg, const int64_t* __restrict__ count, int64_t rows,
                                                                 int64_t T, int32_t* __restrict__ offsets) {
    const int64_t U = T > 0 ? *count : 0;
    for (int64_t j = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; j <= rows; j += (int64_t)gridDim.x * blockDim.x) {
        int64_t lo = 0, hi = U;
        while (lo < hi) {
            const int64_t mid = (lo + hi) >> 1;
            if (uniq[mid] < j) lo = mid + 1;
            else hi = mid;
        }
        offsets[j] = lo < U ? seg[lo] : (int32_t)T;
    }
}
__global__ __launch_bounds__(256) void np_reverse_entries_kernel(const int32_t* __restrict__ perm, const int32_t* __restrict__ owner, int64_t T, int32_t* __restrict__ r_owner) {
    for (int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; t < T; t += (int64_t)gridDim.x * blockDim.x) r_owner[t] = owner[perm[t]];
}

static unsigned np_blocks(int64_t n) {
    const int64_t b = cdiv(n > 0 ? n : 1, 256);
    return (unsigned)(b > 65536 ? 65536 : b);
}
static int np_scan(const NpSource& S, const NpOut& O, int32_t* tiles, int32_t* totals, hipStream_t st) {
    const int64_t ntiles = cdiv(S.n, NP_TILE);
    if (ntiles > 0) np_tile_sums_kernel<<<dim3((unsigned)ntiles), dim3(NP_T), 0, st>>>(S, tiles);
    np_scan_tiles_kernel<<<dim3(1), dim3(NP_T), 0, st>>>(tiles, (int)ntiles, totals);
    if (ntiles > 0) np_emit_kernel<<<dim3((unsigned)ntiles), dim3(NP_T), 0, st>>>(S, tiles, O);
    return check_launch("nbr_plan");
}

}  // namespace marius

using namespace marius;

extern "C" size_t marius_nbr_plan_workspace_bytes(int64_t n) { return (size_t)(3 * (cdiv(n > 0 ? n : 1, NP_TILE) + 1)) * sizeof(int32_t); }

extern "C" int marius_nbr_plan_lists(const int64_t* index_a, const int64_t* offsets_a, int64_t T_a, const int64_t* index_b, const int64_t* offsets_b, int64_t T_b, int64_t n,
                                     int64_t rows, int64_t self_offset, int32_t* offsets, int32_t* index, int32_t* owner, int64_t* keys, int32_t* status,
                                     void* workspace, size_t workspace_bytes, marius_stream_t stream) {
    const int64_t T = T_a + T_b + (self_offset >= 0 ? n : 0), most = (1ll << 31) - 1;
    MARIUS_REQUIRE(n >= 0 && rows >= 0 && T_a >= 0 && T_b >= 0, "nbr_plan_lists: bad sizes");
    MARIUS_REQUIRE(n < most && rows < most && T < most - (1 << 20), "nbr_plan_lists: at most 2^31 targets, rows and entries");
    MARIUS_REQUIRE(n > 0 || T == 0, "nbr_plan_lists: entries without a target");
    MARIUS_REQUIRE(self_offset < 0 || self_offset + n <= rows, "nbr_plan_lists: a target's own row lies behind the rows");
    MARIUS_REQUIRE((T_a == 0 || (index_a && offsets_a)) && (T_b == 0 || (index_b && offsets_b)) && offsets && status && (T == 0 || (index && owner && keys)),
                   "nbr_plan_lists: null pointer");
    MARIUS_REQUIRE(workspace && workspace_bytes >= marius_nbr_plan_workspace_bytes(n), "nbr_plan_lists: workspace too small");
    hipStream_t st = as_stream(stream);
    NpSource S{};
    S.lists = NpLists{index_a, T_a > 0 ? offsets_a : nullptr, index_b, T_b > 0 ? offsets_b : nullptr, T_a, T_b, n, rows, self_offset};
    S.n = n;
    S.status = status;
    NpOut O{};
    O.offsets = offsets;
    const int rc = np_scan(S, O, (int32_t*)workspace, status + 1, st);
    if (rc) return rc;
    if (n > 0) np_check_total_kernel<<<dim3(1), dim3(1), 0, st>>>(offsets, n, T, status);
    if (T > 0) np_entries_kernel<<<dim3(np_blocks(T)), dim3(256), 0, st>>>(S.lists, offsets, T, index, owner, keys, status);
    return check_launch("nbr_plan_lists");
}

extern "C" int marius_nbr_plan_reverse(const int64_t* uniq, const int32_t* seg_offsets, const int64_t* num_unique_dev, const int32_t* perm, const int32_t* owner, int64_t T,
                                       int64_t rows, int32_t* r_offsets, int32_t* r_owner, marius_stream_t stream) {
    MARIUS_REQUIRE(T >= 0 && rows >= 0 && r_offsets && (T == 0 || (uniq && seg_offsets && num_unique_dev && perm && owner && r_owner)), "nbr_plan_reverse: bad arguments");
    hipStream_t st = as_stream(stream);
    np_reverse_offsets_kernel<<<dim3(np_blocks(rows + 1)), dim3(256), 0, st>>>(uniq, seg_offsets, num_unique_dev, rows, T, r_offsets);
    if (T > 0) np_reverse_entries_kernel<<<dim3(np_blocks(T)), dim3(256), 0, st>>>(perm, owner, T, r_owner);
    return check_launch("nbr_plan_reverse");
}

extern "C" size_t marius_nbr_plan_items_workspace_bytes(int64_t n, int32_t max_items) {
    const size_t scan = (marius_nbr_plan_workspace_bytes(n) + 15) & ~(size_t)15, most = max_items > 0 ? max_items : 0;
    return scan + most * sizeof(int4) + (size_t)cdiv((int64_t)most, NP_TILE) * NP_CLASSES * sizeof(int32_t);
}

extern "C" int marius_nbr_plan_items(const int32_t* offsets, int64_t n, int32_t chunk, int32_t* items, int32_t max_items, int32_t* splits, int32_t max_splits, int32_t* totals,
                                     void* workspace, size_t workspace_bytes, marius_stream_t stream) {
    MARIUS_REQUIRE(n >= 0 && chunk > 0 && max_items >= 0 && max_splits >= 0 && totals && offsets, "nbr_plan_items: bad arguments");
    MARIUS_REQUIRE((max_items == 0 || items) && (max_splits == 0 || splits), "nbr_plan_items: null pointer");
    MARIUS_REQUIRE(workspace && workspace_bytes >= marius_nbr_plan_items_workspace_bytes(n, max_items), "nbr_plan_items: workspace too small");
    hipStream_t st = as_stream(stream);
    int4* unsorted = (int4*)((char*)workspace + ((marius_nbr_plan_workspace_bytes(n) + 15) & ~(size_t)15));
    int32_t* hist = (int32_t*)(unsorted + max_items);
    NpSource S{};
    S.offsets = offsets;
    S.n = n;
    S.mode = 1;
    S.chunk = chunk;
    NpOut O{};
    O.items = unsorted;
    O.splits = (int4*)splits;
    O.max_items = max_items;
    O.max_splits = max_splits;
    const int rc = np_scan(S, O, (int32_t*)workspace, totals, st);
    if (rc || max_items == 0) return rc;
    const int ntiles = (int)cdiv(max_items, NP_TILE);
    np_class_counts_kernel<<<dim3((unsigned)ntiles), dim3(NP_T), 0, st>>>(unsorted, totals, max_items, ntiles, hist);
    np_scan_kernel<<<dim3(1), dim3(NP_T), 0, st>>>(hist, ntiles * NP_CLASSES);
    np_class_place_kernel<<<dim3((unsigned)ntiles), dim3(NP_T), 0, st>>>(unsorted, totals, max_items, ntiles, hist, (int4*)items);
    return check_launch("nbr_plan_items");
}
