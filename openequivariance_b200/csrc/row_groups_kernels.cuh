// Row groups: a stable counting sort of the rows of a batch by their group, the offsets of the groups among the sorted rows
// and the table of blocks of up to 64 sorted rows of one group.
//
//   order[p] = the row at sorted position p, slots[r] = the position of row r, offsets[g] = rows of groups before g.
//   Rows whose group is not in 0..groups-1 come last (key `groups`).
//
// A warp takes a run of rows, 32 at a time.  Lanes with the same key find each other by a ballot for each bit of the keys (match_any
// takes a round for each key that occurs: 0.6 us for 32 rows of 89 groups): a row's rank is the number of earlier rows of its key
// in the run, counted in shared memory, plus those of lower lanes, so equal keys keep their order, and every result is the same in every run.
//   * up to 65 536 rows: a cluster of up to eight CTAs counts, scans and places in one launch, the CTAs' counts read from one another's
//     shared memory (row_groups_cluster);
//   * more rows or many groups: count (a histogram per run), scan (the runs' histograms, a key per lane), place (every CTA adds up the keys).
// Measured between two events: 27 rows 10 us (a call among others 11-12), 20 000 rows 12-15, 1 M rows in 89 groups 27-30 (11 + 6 + 19 us under ncu), bound by the latency of a few dependent steps.
#pragma once
#include <cooperative_groups.h>

#include "oeq_common.cuh"

namespace oeq {

constexpr int RG_BLOCK = 64;                    // rows of an entry of the block table
constexpr int RG_SMALL_WARPS = 32, RG_WARPS = 4, RG_RUNS = 1184;           // most runs: eight warps an SM

// Blocks of a group of n rows (up to 2^31 - 1 of them: n + 63 would leave the range of an int).
__host__ __device__ constexpr int rg_group_blocks(int n) { return n / RG_BLOCK + (n % RG_BLOCK != 0); }
static_assert(rg_group_blocks(0) == 0 && rg_group_blocks(1) == 1 && rg_group_blocks(64) == 1 && rg_group_blocks(65) == 2, "blocks of a group");
static_assert(rg_group_blocks(0x7fffffff) == 1 << 25 && rg_group_blocks(0x7fffffff - 63) == (1 << 25) - 1, "blocks of a group");

__device__ __forceinline__ int rg_key(const long long* __restrict__ index, long long r, int groups) {
    const long long g = index[r];
    return g >= 0 && g < groups ? (int)g : groups;
}

// Exclusive sums over a[0..n) in shared memory, a[n] = total, by all threads of the CTA; `part` holds 33 ints.
__device__ __forceinline__ void rg_scan(int* a, int n, int* part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int before = 0;
    for (int i0 = 0; i0 < n; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x, v = i < n ? a[i] : 0;
        int s = v;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, s, off);
            if (lane >= off) s += t;
        }
        if (lane == 31) part[warp] = s;
        __syncthreads();
        if (warp == 0) {
            int t = lane < warps ? part[lane] : 0;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, t, off);
                if (lane >= off) t += u;
            }
            if (lane < warps) part[lane] = t;
        }
        __syncthreads();
        const int up = before + (warp ? part[warp - 1] : 0) + s - v;
        before += part[warps - 1];
        if (i < n) a[i] = up;
        __syncthreads();
    }
    if (threadIdx.x == 0) a[n] = before;
    __syncthreads();
}

// The last i with a[i] <= v, of a[0..n] ascending with a[0] <= v.
__device__ __forceinline__ int rg_find(const int* a, int n, int v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a[mid] <= v) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Offsets and the threads' share of the block table, from offsets[0..groups] in shared memory; `first` (groups + 1 ints) is
// overwritten with the number of blocks before each group's.
__device__ __forceinline__ void rg_tables(const int* offsets, int* first, int* part, int groups, int blocks, long long* __restrict__ offsets_out,
                                          int* __restrict__ table, long long thread, long long threads) {
    for (int g = threadIdx.x; g < groups; g += blockDim.x) first[g] = rg_group_blocks(offsets[g + 1] - offsets[g]);
    __syncthreads();
    rg_scan(first, groups, part);
    for (long long g = thread; g <= groups; g += threads) offsets_out[g] = offsets[g];
    for (long long b = thread; b < blocks; b += threads) {
        int g = -1, p = 0, n = 0;
        if (b < first[groups]) {
            g = rg_find(first, groups, (int)b);         // (of groups without rows between, the last starts at the same block)
            p = offsets[g] + ((int)b - first[g]) * RG_BLOCK;
            n = min(RG_BLOCK, offsets[g + 1] - p);
        }
        table[3 * b] = g;
        table[3 * b + 1] = p;
        table[3 * b + 2] = n;
    }
}

constexpr int RG_AHEAD = 8;                     // rows of a lane whose keys are loaded together
template <class F>
__device__ __forceinline__ void rg_rows(const long long* __restrict__ index, long long lo, long long hi, int groups, F&& rows) {
    const int lane = threadIdx.x & 31;
    for (long long r0 = lo; r0 < hi; r0 += 32 * RG_AHEAD) {
        int key[RG_AHEAD];
#pragma unroll
        for (int i = 0; i < RG_AHEAD; ++i) key[i] = r0 + 32 * i + lane < hi ? rg_key(index, r0 + 32 * i + lane, groups) : -1;
#pragma unroll
        for (int i = 0; i < RG_AHEAD; ++i) {
            if (r0 + 32 * i >= hi) break;
            rows(r0 + 32 * i + lane, key[i]);
        }
    }
}
// Counts of the keys of rows [lo, hi) into the warp's count[].
__device__ __forceinline__ void rg_count(const long long* __restrict__ index, long long lo, long long hi, int groups, int* count) {
    rg_rows(index, lo, hi, groups, [&](long long, int key) {
        if (key >= 0) atomicAdd(count + key, 1);
    });
    __syncwarp();
}
// visit(row, key, position) of rows [lo, hi), count[] being the position of the first row of each key.
template <class F>
__device__ __forceinline__ void rg_place(const long long* __restrict__ index, long long lo, long long hi, int groups, int* count, F&& visit) {
    const int lane = threadIdx.x & 31, bits = 32 - __clz(groups);
    rg_rows(index, lo, hi, groups, [&](long long r, int key) {
        unsigned same = __ballot_sync(0xffffffffu, key >= 0);
        for (int b = 0; b < bits; ++b) {
            const unsigned set = __ballot_sync(0xffffffffu, key >> b & 1);
            same &= key >> b & 1 ? set : ~set;
        }
        const unsigned lower = same & ((1u << lane) - 1);
        const int before = key >= 0 ? count[key] : 0;
        __syncwarp();
        if (key >= 0) {
            visit(r, key, before + __popc(lower));
            if (lower == 0) count[key] = before + __popc(same);
        }
        __syncwarp();
    });
}

// ---- a cluster of CTAs.  Shared memory: [32 warps][groups + 1] counts, [groups + 1] totals of the CTA, [groups + 2] offsets, [groups + 2]
// blocks, 33 ints
__global__ void __launch_bounds__(32 * RG_SMALL_WARPS) oeq_row_groups_cluster(const long long* __restrict__ index, int rows, int groups, int blocks,
                                                                                long long* __restrict__ order, long long* __restrict__ slots,
                                                                                long long* __restrict__ offsets, int* __restrict__ table) {
    extern __shared__ int rg_smem[];
    const auto cluster = cooperative_groups::this_cluster();
    const int ctas = (int)cluster.num_blocks(), cta = (int)cluster.block_rank();
    const int keys = groups + 1, tid = threadIdx.x, warp = tid >> 5;
    int *totals = rg_smem + RG_SMALL_WARPS * keys, *offs = totals + keys, *first = offs + keys + 1, *part = first + keys + 1;
    for (int i = tid; i < RG_SMALL_WARPS * keys; i += blockDim.x) rg_smem[i] = 0;
    __syncthreads();
    const int run = (rows + 32 * RG_SMALL_WARPS * ctas - 1) / (32 * RG_SMALL_WARPS * ctas) * 32;
    const int lo = (int)min((long long)(cta * RG_SMALL_WARPS + warp) * run, (long long)rows), hi = min(lo + run, rows);
    int* mine = rg_smem + warp * keys;
    rg_count(index, lo, hi, groups, mine);
    __syncthreads();
    for (int k = tid; k < keys; k += blockDim.x) {          // warps' counts -> rows of the key in the warps before
        int s = 0;
        for (int w = 0; w < RG_SMALL_WARPS; ++w) {
            const int n = rg_smem[w * keys + k];
            rg_smem[w * keys + k] = s;
            s += n;
        }
        totals[k] = s;
    }
    cluster.sync();
    for (int k = tid; k < keys; k += blockDim.x) {
        int all = 0, before = 0;
        for (int c = 0; c < ctas; ++c) {
            const int n = *cluster.map_shared_rank(totals + k, c);
            before += c < cta ? n : 0;
            all += n;
        }
        offs[k] = all;
        for (int w = 0; w < RG_SMALL_WARPS; ++w) rg_smem[w * keys + k] += before;
    }
    cluster.sync();                             // (a CTA's totals are read until here)
    rg_scan(offs, keys, part);
    for (int k = tid & 31; k < keys; k += 32) mine[k] += offs[k];
    __syncwarp();
    rg_place(index, lo, hi, groups, mine, [&](long long r, int, int p) {
        order[p] = r;
        slots[r] = p;
    });
    rg_tables(offs, first, part, groups, blocks, offsets, table, (long long)cta * blockDim.x + tid, (long long)ctas * blockDim.x);
}

// ---- many rows: runs of `run` rows (a multiple of 32), one per warp; counts [runs][groups + 1], totals [groups + 1]
__global__ void __launch_bounds__(32 * RG_WARPS) oeq_row_groups_count(const long long* __restrict__ index, long long rows, long long run, int runs,
                                                                      int groups, int* __restrict__ counts) {
    extern __shared__ int rg_smem[];
    const int keys = groups + 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockIdx.x * RG_WARPS + warp;
    int* mine = rg_smem + warp * keys;
    for (int k = lane; k < keys; k += 32) mine[k] = 0;
    __syncwarp();
    if (n >= runs) return;
    const long long lo = n * run, hi = min(lo + run, rows);
    rg_count(index, lo, hi, groups, mine);
    for (int k = lane; k < keys; k += 32) counts[(long long)n * keys + k] = mine[k];
}

// counts[n][k] -> rows of key k in the runs before n.  A CTA takes eight keys, eight threads of each of 128 spans of the runs.
// (32 keys and 32 spans a CTA: 13 us for 1 184 runs of 90 keys, three CTAs.)
__global__ void __launch_bounds__(1024) oeq_row_groups_scan(int* __restrict__ counts, int* __restrict__ totals, int runs, int keys) {
    constexpr int SPANS = 128, EACH = (RG_RUNS + SPANS - 1) / SPANS;
    __shared__ int sums[8][SPANS + 4];
    const int key = threadIdx.x & 7, span = threadIdx.x >> 3, k = blockIdx.x * 8 + key, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int each = (runs + SPANS - 1) / SPANS, lo = min(span * each, runs), hi = min(lo + each, runs);
    int c[EACH], s = 0;                         // all on the way at once
#pragma unroll
    for (int i = 0; i < EACH; ++i) c[i] = lo + i < hi && k < keys ? counts[(long long)(lo + i) * keys + k] : 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) s += c[i];
    sums[key][span] = s;
    __syncthreads();
    if (warp < 8) {                             // spans of key `warp`, four a lane
        int v[4], all = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = all;
            all += sums[warp][4 * lane + i];
        }
        int up = all;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, up, off);
            if (lane >= off) up += t;
        }
        if (lane == 31 && blockIdx.x * 8 + warp < keys) totals[blockIdx.x * 8 + warp] = up;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[warp][4 * lane + i] = up - all + v[i];
    }
    __syncthreads();
    int before = sums[key][span];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        if (lo + i < hi && k < keys) counts[(long long)(lo + i) * keys + k] = before;
        before += c[i];
    }
}

// Shared memory: [RG_WARPS][groups + 1] counts, [groups + 2] offsets, [groups + 2] blocks, 33 ints
__global__ void __launch_bounds__(32 * RG_WARPS) oeq_row_groups_place(const long long* __restrict__ index, long long rows, long long run, int runs,
                                                                      int groups, int blocks, const int* __restrict__ counts,
                                                                      const int* __restrict__ totals, long long* __restrict__ order,
                                                                      long long* __restrict__ slots, long long* __restrict__ offsets,
                                                                      int* __restrict__ table) {
    extern __shared__ int rg_smem[];
    const int keys = groups + 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockIdx.x * RG_WARPS + warp;
    int *offs = rg_smem + RG_WARPS * keys, *first = offs + keys + 1, *part = first + keys + 1, *mine = rg_smem + warp * keys;
    for (int k = threadIdx.x; k < keys; k += blockDim.x) offs[k] = totals[k];
    __syncthreads();
    rg_scan(offs, keys, part);
    if (n < runs) {
        for (int k = lane; k < keys; k += 32) mine[k] = offs[k] + counts[(long long)n * keys + k];
        __syncwarp();
        const long long lo = n * run, hi = min(lo + run, rows);
        rg_place(index, lo, hi, groups, mine, [&](long long r, int, int p) {
            order[p] = r;
            slots[r] = p;
        });
    }
    rg_tables(offs, first, part, groups, blocks, offsets, table, (long long)blockIdx.x * blockDim.x + threadIdx.x, (long long)gridDim.x * blockDim.x);
}

// ---- rows that lie in the order of their groups, from the number of rows of each: groups that begin behind the last row end
// there, and rows behind the last group belong to none.  Shared memory: [groups + 1] offsets, [groups + 2] blocks, 33 ints
__global__ void __launch_bounds__(512) oeq_row_groups_counts(const long long* __restrict__ counts, long long rows, int groups, int blocks,
                                                             long long* __restrict__ index, long long* __restrict__ offsets, int* __restrict__ table) {
    extern __shared__ int rg_smem[];
    int *offs = rg_smem, *first = offs + groups + 2, *part = first + groups + 2;
    // (counts are clamped one by one and their sum stays below 2^31 by the scan of clamped partial sums below)
    __shared__ long long carry[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    long long before = 0;
    for (int i0 = 0; i0 < groups; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x;
        long long v = i < groups ? counts[i] : 0;
        v = v < 0 ? 0 : (v > rows ? rows : v);
        long long s = v;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const long long t = __shfl_up_sync(0xffffffffu, s, off);
            if (lane >= off) s += t;
        }
        if (lane == 31) carry[warp] = s;
        __syncthreads();
        long long up = before, all = before;
        for (int w = 0; w < warps; ++w) {
            if (w < warp) up += carry[w];
            all += carry[w];
        }
        if (i < groups) offs[i + 1] = (int)min(up + s, rows);
        before = all;
        __syncthreads();
    }
    if (threadIdx.x == 0) offs[0] = 0;
    __syncthreads();
    const long long thread = (long long)blockIdx.x * blockDim.x + threadIdx.x, threads = (long long)gridDim.x * blockDim.x;
    rg_tables(offs, first, part, groups, blocks, offsets, table, thread, threads);
    for (long long r = thread; r < rows; r += threads) {
        const int g = rg_find(offs, groups, (int)r);
        index[r] = g < groups ? g : -1;
    }
}

}  // namespace oeq
