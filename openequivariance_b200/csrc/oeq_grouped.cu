// Row groups and linear maps with the weights of a row's group: the host side behind include/oeq_b200.h.
//
// The kernels are compiled with the library (their shapes are run-time values); nothing here allocates device memory, synchronises or
// keeps anything of a call.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <string>
#include <vector>

#include "../../include/oeq_b200.h"
#include "oeq_internal.h"
#include "grouped_kernels.cuh"
#include "grouped_tc_dw_kernels.cuh"
#include "grouped_tc_kernels.cuh"
#include "row_groups_kernels.cuh"

using namespace oeq;

namespace {

#define OEQ_CUDA(expr)                                                                                                  \
    do {                                                                                                                \
        cudaError_t e_ = (expr);                                                                                        \
        if (e_ != cudaSuccess) return oeq_fail(OEQ_ERR_CUDA, std::string(#expr) + ": " + cudaGetErrorString(e_));       \
    } while (0)

constexpr int64_t MOST_ROWS = (int64_t(1) << 31) - 1;
constexpr int MOST_GRID_Y = 65535;
constexpr size_t SMEM_MOST = 227 * 1024, WORKSPACE_ALIGN = 32;

size_t elem_bytes(int dtype) { return dtype == OEQ_F64 ? 8 : (dtype == OEQ_F32 ? 4 : 2); }
bool known_dtype(int dtype) { return dtype == OEQ_F32 || dtype == OEQ_F64 || dtype == OEQ_BF16 || dtype == OEQ_F16; }

constexpr int KNOWN_DEVICES = 64;       // what is kept of a device; of others it is asked for at every call
int sm_count(int& n) {
    static std::atomic<int> counts[KNOWN_DEVICES];
    int dev = 0;
    OEQ_CUDA(cudaGetDevice(&dev));
    n = dev < KNOWN_DEVICES ? counts[dev].load(std::memory_order_relaxed) : 0;
    if (n) return OEQ_OK;
    OEQ_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    if (dev < KNOWN_DEVICES) counts[dev].store(n, std::memory_order_relaxed);
    return OEQ_OK;
}

// Shared memory beyond 48 KB has to be allowed for a kernel on every device that it runs on: up to the most that any call asks for, at
// the first call there.
template <auto KERNEL>
int allow_smem(size_t most) {
    static std::atomic<uint64_t> done{0};       // a bit for each device
    int dev = 0;
    OEQ_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = dev < KNOWN_DEVICES ? uint64_t(1) << dev : 0;
    if (done.load(std::memory_order_acquire) & bit) return OEQ_OK;
    OEQ_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    done.fetch_or(bit, std::memory_order_release);
    return OEQ_OK;
}

int check_groups(int64_t rows, int64_t groups) {
    if (rows < 0 || rows > MOST_ROWS) return oeq_fail(OEQ_ERR_INVALID, "rows must be in 0 .. 2^31 - 1");
    if (groups < 1 || groups > OEQ_MOST_GROUPS) return oeq_fail(OEQ_ERR_INVALID, "groups must be in 1 .. " + std::to_string(OEQ_MOST_GROUPS));
    return OEQ_OK;
}

// ---------------------------------------------------------------------------- row groups
size_t table_smem(int64_t groups) { return (2 * (groups + 2) + 33) * sizeof(int); }
size_t walk_smem(int64_t groups) { return RG_WARPS * (groups + 1) * sizeof(int); }
size_t small_smem(int64_t groups) { return (RG_SMALL_WARPS + 1) * (groups + 1) * sizeof(int) + table_smem(groups); }
// A cluster's warps walk 32 rows a step each; beyond these many rows the runs of many CTAs are faster (89 groups, cluster / runs: 50 000 rows
// 17 / 20 us, 262 144 rows 41 / 21).
bool small_groups(int64_t rows, int64_t groups) { return rows <= 65536 && small_smem(groups) <= SMEM_MOST; }
struct Runs {
    int64_t run;        // rows of a run
    int runs;
};
Runs runs_of(int64_t rows) {
    const int64_t run = std::max<int64_t>(256, ((rows + RG_RUNS - 1) / RG_RUNS + 31) / 32 * 32);
    return {run, (int)std::max<int64_t>(1, (rows + run - 1) / run)};
}

}  // namespace

// ---------------------------------------------------------------------------- linear maps

struct oeq_grouped {
    GpProblem forward, backward, weights;       // X -> Z, dZ -> dX, and X -> Z with the paths in the order of their weights
    int d_max = 0;
};

namespace {

int column_count(const GpProblem& gp) {
    int n = 0;
    for (int t = 0; t < gp.n_targets; ++t) n += (gp.target[t].mul + GP_TILE - 1) / GP_TILE * gp.target[t].d;
    return n;
}

template <class T>
int simt_product(const GpProblem& gp, int64_t rows, int64_t groups, const void* X, const void* W, const int64_t* order, const int64_t* offsets,
                 const int32_t* blocks, void* Z, cudaStream_t st) {
    const int n = (int)oeq_row_groups_blocks(rows, groups), columns = column_count(gp);
    if (columns == 0) return OEQ_OK;
    int sms = 0;
    if (int rc = sm_count(sms)) return rc;
    for (int first = 0; first < columns; first += MOST_GRID_Y) {       // (the zeros with the first columns)
        const dim3 grid((unsigned)(n + (first ? 0 : (sms + columns - 1) / columns)), (unsigned)std::min(columns - first, MOST_GRID_Y));
        oeq_grouped_simt<T><<<grid, GP_SIMT_THREADS, 0, st>>>(gp, (const T*)X, (const T*)W, (const long long*)order, (const long long*)offsets, blocks, n, rows,
                                                              (int)groups, first, (T*)Z);
        OEQ_CUDA(cudaGetLastError());
    }
    return OEQ_OK;
}

// Ranges of rows: about four CTAs an SM, 64 rows and more each.
GpSplit simt_split(const GpProblem& gp, int64_t rows, int sms) {
    GpSplit s{};
    int columns = 0;
    auto tiles = [&](int p) { return (gp.path[p].src_mul + GP_TILE - 1) / GP_TILE * ((gp.target[gp.path[p].dst].mul + GP_TILE - 1) / GP_TILE); };
    for (int p = 0; p < gp.n_paths; ++p) columns += tiles(p);
    const int parts = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(GP_PARTS, (4 * sms + columns - 1) / std::max(1, columns)), rows / 64));
    for (int p = 0; p < gp.n_paths; ++p) {
        s.parts[p] = parts;
        s.first[p + 1] = s.first[p] + tiles(p) * parts;
    }
    return s;
}

// The workspace of a weight gradient: the starts of the CTAs' ranges, then their partial tiles, of which a path in one range has none.
size_t partial_ctas(const GpProblem& gp, const GpSplit& split) {
    int n = 0;
    for (int p = 0; p < gp.n_paths; ++p)
        if (split.parts[p] > 1) n = split.first[p + 1];
    return (size_t)n;
}
size_t positions_bytes(const GpProblem& gp, const GpSplit& split) { return ((size_t)split.first[gp.n_paths] * sizeof(GpStart) + 255) / 256 * 256; }

template <class T, int TILE>
int join(const GpProblem& gp, const GpSplit& split, int64_t rows, int64_t groups, const int64_t* offsets, void* dW, const void* ws, cudaStream_t st) {
    const int ctas = split.first[gp.n_paths], zero_ctas = (int)std::min<int64_t>(groups, 296);
    oeq_grouped_join<T, TILE><<<TILE / 4 * ctas + zero_ctas, 256, 0, st>>>(gp, split, (const long long*)offsets, rows, (int)groups, zero_ctas,
                                                                         (const typename GpAcc<T>::type*)((const char*)ws + positions_bytes(gp, split)), (const GpStart*)ws, (T*)dW);
    OEQ_CUDA(cudaGetLastError());
    return OEQ_OK;
}

template <class T>
int simt_weights(const GpProblem& gp, int64_t rows, int64_t groups, const void* X, const void* dZ, const int64_t* order, const int64_t* offsets, void* dW,
                 void* ws, cudaStream_t st) {
    int sms = 0;
    if (int rc = sm_count(sms)) return rc;
    const GpSplit split = simt_split(gp, rows, sms);
    oeq_grouped_simt_dw<T><<<split.first[gp.n_paths], GP_SIMT_THREADS, 0, st>>>(gp, split, (const T*)X, (const T*)dZ, (const long long*)order,
                                                                                (const long long*)offsets, rows, (int)groups, (T*)dW,
                                                                                (typename GpAcc<T>::type*)((char*)ws + positions_bytes(gp, split)), (GpStart*)ws);
    OEQ_CUDA(cudaGetLastError());
    return join<T, GP_TILE>(gp, split, rows, groups, offsets, dW, ws, st);
}

// ---- tensor cores
constexpr int MOST_PARTS = GP_PARTS;    // ranges of rows
// The time of a group's weights, in (row, component) pairs.  FP32, whose weights are split: 160 instead of 96 takes 4 999 rows of 128x(0e+1o+2e) in 89 groups
// from 41.0 to 36.9 us (64: 50, 240: 42) and 50 000 rows in 10 groups from 219 to 221.  In 16 bits, where they are copied, 64 and 96 are equal (143 us, 100 000 rows
// in 256 groups) and 160 takes 148.  The weight gradient of the first: 54 / 47 / 50 / 54 us with 64 / 96 / 160 / 240.
template <class T> constexpr int group_pairs() { return GtType<T>::SPLIT ? 160 : 96; }
constexpr int GROUP_PAIRS_DW = 96;
// The CTAs, one for each SM, are dealt to the tiles of channels by the time that they take: for every (row, component) pair, and for
// those that a group's weights count for, the channels read and written and a fixed part.  (By the rows alone 4 999 rows in 89
// groups take 58 us: an output of scalars, with as many weights as the others, has a ninth of the CTAs.)
template <class T>
int tc_plan(const GpProblem& gp, int64_t rows, int64_t groups, int sms, GtProblem& gt, int& ctas, size_t& smem) {
    gt.gp = gp;
    const size_t fixed = GT_CONTROL + GT_EPI_GROUPS * GT_STAGING, room = SMEM_MOST - fixed;
    double cost[GP_BLOCKS] = {};
    ctas = 0;
    for (int t = 0; t < gp.n_targets; ++t) {
        const GpTarget& to = gp.target[t];
        GtTarget& x = gt.target[t];
        x = {};
        if (to.mul == 0) continue;
        x.parts = 1;
        int k = 0;
        for (int p = to.path_begin; p < to.path_end; ++p) {
            k += gp.path[p].src_mul;
            x.chunks += (gp.path[p].src_mul + GtType<T>::KC - 1) / GtType<T>::KC;
        }
        // Channels of a tile.  Every tile reads the rows again, and a tile whose weights do not stay in shared memory fills them in again for
        // every 128 pairs: n / 128 of the work that the rows are.
        double least = 0;
        for (int most = GtType<T>::N_MAX; most >= GtType<T>::N_MAX / 4; most /= 2) {
            const int tiles = (to.mul + most - 1) / most, n = ((to.mul + tiles - 1) / tiles + 15) / 16 * 16;
            const bool stays = 2 * (size_t)GtType<T>::A_BYTES + (size_t)x.chunks * GtType<T>::b_bytes(n) <= room;
            const double work = ((to.mul + n - 1) / n) * (1.0 + (stays ? 0.0 : n / 128.0));
            if (x.n == 0 || work < least) {
                x.n = n;
                least = work;
            }
        }
        x.n_tiles = (to.mul + x.n - 1) / x.n;
        x.extra = group_pairs<T>() / to.d;
        cost[t] = ((double)rows * to.d + (double)std::min(rows, groups) * group_pairs<T>()) * (k + x.n + 32);
        ctas += x.n_tiles;
    }
    double all = 0;
    for (int t = 0; t < gp.n_targets; ++t) all += cost[t] * gt.target[t].n_tiles;
    ctas = 0;
    for (int t = 0; t < gp.n_targets; ++t) {            // (whole shares first: the rest takes a few steps)
        GtTarget& x = gt.target[t];
        if (x.parts) x.parts = (int)std::max(1.0, std::min((double)std::min<int64_t>(rows, MOST_PARTS), std::floor(sms * cost[t] / all)));
        ctas += x.parts * x.n_tiles;
    }
    for (;;) {                          // the tile whose ranges take longest gets another CTA
        int most = -1;
        for (int t = 0; t < gp.n_targets; ++t)
            if (gt.target[t].parts && gt.target[t].parts < std::min<int64_t>(rows, MOST_PARTS) && (most < 0 || cost[t] / gt.target[t].parts > cost[most] / gt.target[most].parts)) most = t;
        if (most < 0 || ctas + gt.target[most].n_tiles > sms) break;
        ++gt.target[most].parts;
        ctas += gt.target[most].n_tiles;
    }
    smem = 0;
    ctas = 0;
    for (int t = 0; t < gp.n_targets; ++t) {
        GtTarget& x = gt.target[t];
        x.first = ctas;
        ctas += x.n_tiles * x.parts;
        if (!x.parts) continue;
        const size_t a = GtType<T>::A_BYTES, b = GtType<T>::b_bytes(x.n);
        if (2 * a + x.chunks * b <= room) {     // a group's weights stay in shared memory
            x.slots = std::max(1, x.chunks);
            x.stages = (int)std::min<size_t>(GT_STAGES, (room - x.slots * b) / a);
        } else {
            x.slots = x.stages = (int)std::min<size_t>(GT_STAGES, room / (a + b));
        }
        smem = std::max(smem, x.stages * a + x.slots * b);
    }
    smem = std::max<size_t>(smem + fixed, 120 * 1024);         // (one CTA an SM: it takes all of the tensor memory)
    return OEQ_OK;
}

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

template <class T, bool TRANS, bool FAST, bool LONG>
int tc_launch(const GtProblem& gt, const GtArgs& args, int ctas, size_t smem, cudaStream_t st) {
    if (int rc = allow_smem<oeq_grouped_tc<T, TRANS, FAST, LONG>>(SMEM_MOST)) return rc;
    oeq_grouped_tc<T, TRANS, FAST, LONG><<<ctas, GT_THREADS, smem, st>>>(gt, args);
    OEQ_CUDA(cudaGetLastError());
    return OEQ_OK;
}

template <class T, bool TRANS>
int tc_product(const GpProblem& gp, int64_t rows, int64_t groups, const void* X, const void* W, const int64_t* order, const int64_t* offsets, void* Z,
               cudaStream_t st) {
    int sms = 0, ctas = 0;
    size_t smem = 0;
    if (int rc = sm_count(sms)) return rc;
    GtProblem gt{};
    if (int rc = tc_plan<T>(gp, rows, groups, sms, gt, ctas, smem)) return rc;
    if (ctas == 0) return OEQ_OK;
    const GtArgs args{X, W, (const long long*)order, (const long long*)offsets, Z, rows, (int)groups, aligned(Z, 16) && gp.dst_dim * sizeof(T) % 16 == 0};
    constexpr int V = 16 / sizeof(T);
    bool fast = aligned(X, 16) && aligned(W, 16) && gp.src_dim % V == 0 && gp.w_numel % V == 0;
    for (int p = 0; p < gp.n_paths; ++p) fast &= gp.path[p].src_off % V == 0 && gp.path[p].src_mul % V == 0 && gp.path[p].w_off % V == 0 && gp.path[p].w_ld % V == 0;
    if constexpr (GtType<T>::SPLIT) {
        bool is_long = false;
        for (int t = 0; t < gp.n_targets; ++t) is_long |= gt.target[t].chunks > GT_CHAIN;
        if (is_long) return fast ? tc_launch<T, TRANS, true, true>(gt, args, ctas, smem, st) : tc_launch<T, TRANS, false, true>(gt, args, ctas, smem, st);
    }
    return fast ? tc_launch<T, TRANS, true, false>(gt, args, ctas, smem, st) : tc_launch<T, TRANS, false, false>(gt, args, ctas, smem, st);
}

// CTAs of the tiles of the weight gradient, one for each SM, dealt by the time that a range of rows takes.
GpSplit tc_split(const GpProblem& gp, int64_t rows, int64_t groups, int sms) {
    GpSplit s{};
    int tiles[GP_PATHS], ctas = 0;
    double cost[GP_PATHS];
    for (int p = 0; p < gp.n_paths; ++p) {
        const GpTarget& to = gp.target[gp.path[p].dst];
        tiles[p] = (gp.path[p].src_mul + GD_TILE - 1) / GD_TILE * ((to.mul + GD_TILE - 1) / GD_TILE);
        cost[p] = ((double)rows * to.d + (double)std::min(rows, groups) * GROUP_PAIRS_DW) * (std::min(GD_TILE, gp.path[p].src_mul) + std::min(GD_TILE, to.mul) + 64);
        s.parts[p] = 1;
        ctas += tiles[p];
    }
    double all = 0;
    for (int p = 0; p < gp.n_paths; ++p) all += cost[p] * tiles[p];
    ctas = 0;
    for (int p = 0; p < gp.n_paths; ++p) {
        s.parts[p] = (int)std::max(1.0, std::min((double)std::min<int64_t>(rows, MOST_PARTS), std::floor(sms * cost[p] / all)));
        ctas += s.parts[p] * tiles[p];
    }
    for (;;) {
        int most = -1;
        for (int p = 0; p < gp.n_paths; ++p)
            if (s.parts[p] < std::min<int64_t>(rows, MOST_PARTS) && (most < 0 || cost[p] / s.parts[p] > cost[most] / s.parts[most])) most = p;
        if (most < 0 || ctas + tiles[most] > sms) break;
        ++s.parts[most];
        ctas += tiles[most];
    }
    for (int p = 0; p < gp.n_paths; ++p) s.first[p + 1] = s.first[p] + tiles[p] * s.parts[p];
    return s;
}

template <class T>
int tc_weights(const GpProblem& gp, int64_t rows, int64_t groups, const void* X, const void* dZ, const int64_t* order, const int64_t* offsets, void* dW, void* ws,
               cudaStream_t st) {
    int sms = 0;
    if (int rc = sm_count(sms)) return rc;
    GdProblem gd{gp, tc_split(gp, rows, groups, sms), {}};
    for (int p = 0; p < gp.n_paths; ++p) gd.extra[p] = GROUP_PAIRS_DW / gp.target[gp.path[p].dst].d;
    const GdArgs args{X, dZ, (const long long*)order, (const long long*)offsets, dW, (float*)((char*)ws + positions_bytes(gp, gd.split)), (GpStart*)ws, rows, (int)groups,
                      aligned(dW, 16) && gp.w_numel * sizeof(T) % 16 == 0};
    constexpr int V = 16 / sizeof(T);
    bool fast = aligned(X, 16) && aligned(dZ, 16) && gp.src_dim % V == 0 && gp.dst_dim % V == 0;
    for (int p = 0; p < gp.n_paths; ++p) {
        const GpTarget& to = gp.target[gp.path[p].dst];
        fast &= gp.path[p].src_off % V == 0 && gp.path[p].src_mul % V == 0 && to.off % V == 0 && to.mul % V == 0;
    }
    if (fast) {
        if (int rc = allow_smem<oeq_grouped_tc_dw<T, true>>(GD_SMEM)) return rc;
        oeq_grouped_tc_dw<T, true><<<gd.split.first[gp.n_paths], GD_THREADS, GD_SMEM, st>>>(gd, args);
    } else {
        if (int rc = allow_smem<oeq_grouped_tc_dw<T, false>>(GD_SMEM)) return rc;
        oeq_grouped_tc_dw<T, false><<<gd.split.first[gp.n_paths], GD_THREADS, GD_SMEM, st>>>(gd, args);
    }
    OEQ_CUDA(cudaGetLastError());
    return join<T, GD_TILE>(gp, gd.split, rows, groups, offsets, dW, ws, st);
}

// One thread polls a barrier that nothing completes, gives up and records the code, as a kernel whose wait runs out does.
__global__ void oeq_grouped_wait_probe(unsigned polls) {
    __shared__ unsigned long long bar;
    if (threadIdx.x != 0) return;
    mbar_init(&bar, 1);
    fence_mbar_init();
    for (unsigned i = 0; i < polls; ++i)
        if (mbar_try_wait(&bar, 0u)) return;
    atomicCAS(&gt_status, 0, ERR_GT_FULL);
}

int check_call(const oeq_grouped* h, int dtype, int64_t rows, int64_t groups) {
    if (!h) return oeq_fail(OEQ_ERR_INVALID, "null handle");
    if (!known_dtype(dtype)) return oeq_fail(OEQ_ERR_INVALID, "unknown dtype");
    return check_groups(rows, groups);
}

template <bool TRANS>
int product(const oeq_grouped* h, int dtype, int64_t rows, int64_t groups, const void* X, const void* W, const int64_t* order, const int64_t* offsets,
            const int32_t* blocks, void* Z, void* stream) {
    const GpProblem& gp = TRANS ? h->backward : h->forward;
    if (rows == 0 || gp.dst_dim == 0) return OEQ_OK;
    if (!offsets || !blocks || !Z || (gp.src_dim && !X) || (gp.w_numel && !W)) return oeq_fail(OEQ_ERR_INVALID, "null pointer");
    const cudaStream_t st = (cudaStream_t)stream;
    const bool tc = h->d_max <= GT_D_MAX;
    switch (dtype) {
        case OEQ_F64: return simt_product<double>(gp, rows, groups, X, W, order, offsets, blocks, Z, st);
        case OEQ_F32: return tc ? tc_product<float, TRANS>(gp, rows, groups, X, W, order, offsets, Z, st)
                                : simt_product<float>(gp, rows, groups, X, W, order, offsets, blocks, Z, st);
        case OEQ_BF16: return tc ? tc_product<__nv_bfloat16, TRANS>(gp, rows, groups, X, W, order, offsets, Z, st)
                                 : simt_product<__nv_bfloat16>(gp, rows, groups, X, W, order, offsets, blocks, Z, st);
        default: return tc ? tc_product<__half, TRANS>(gp, rows, groups, X, W, order, offsets, Z, st)
                           : simt_product<__half>(gp, rows, groups, X, W, order, offsets, blocks, Z, st);
    }
}

}  // namespace

extern "C" {

int64_t oeq_row_groups_blocks(int64_t rows, int64_t groups) { return rows / RG_BLOCK + std::min(rows, groups); }

size_t oeq_row_groups_workspace_bytes(int64_t rows, int64_t groups) {
    if (rows < 0 || groups < 1 || small_groups(rows, groups)) return 0;
    return ((size_t)runs_of(rows).runs + 1) * (size_t)(groups + 1) * sizeof(int);
}

int oeq_row_groups(int64_t rows, int64_t groups, const int64_t* index, int64_t* order, int64_t* slots, int64_t* offsets, int32_t* blocks, void* workspace,
                   size_t workspace_bytes, void* stream) {
    if (int rc = check_groups(rows, groups)) return rc;
    if (!offsets || (rows > 0 && (!index || !order || !slots || !blocks))) return oeq_fail(OEQ_ERR_INVALID, "null pointer");
    if (oeq_row_groups_workspace_bytes(rows, groups) > workspace_bytes || (oeq_row_groups_workspace_bytes(rows, groups) && !workspace))
        return oeq_fail(OEQ_ERR_INVALID, "workspace too small");
    const cudaStream_t st = (cudaStream_t)stream;
    const int n = (int)oeq_row_groups_blocks(rows, groups), keys = (int)groups + 1;
    const long long* in = (const long long*)index;
    long long *ord = (long long*)order, *slt = (long long*)slots, *off = (long long*)offsets;
    if (small_groups(rows, groups)) {
        const size_t smem = small_smem(groups);
        if (int rc = allow_smem<oeq_row_groups_cluster>(SMEM_MOST)) return rc;
        int ctas = 1;                   // two steps of a warp as long as there are CTAs for that
        while (ctas < 8 && rows > (int64_t)ctas * 64 * RG_SMALL_WARPS) ctas *= 2;
        cudaLaunchAttribute cluster;
        cluster.id = cudaLaunchAttributeClusterDimension;
        cluster.val.clusterDim.x = (unsigned)ctas;
        cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3((unsigned)ctas);
        config.blockDim = dim3(32 * RG_SMALL_WARPS);
        config.dynamicSmemBytes = smem;
        config.stream = st;
        config.attrs = &cluster;
        config.numAttrs = 1;
        OEQ_CUDA(cudaLaunchKernelEx(&config, oeq_row_groups_cluster, in, (int)rows, (int)groups, n, ord, slt, off, (int*)blocks));
    } else {
        const Runs r = runs_of(rows);
        int *counts = (int*)workspace, *totals = counts + (size_t)r.runs * keys;
        const unsigned ctas = (unsigned)((r.runs + RG_WARPS - 1) / RG_WARPS);
        const size_t smem = walk_smem(groups), smem_place = smem + table_smem(groups);
        if (int rc = allow_smem<oeq_row_groups_count>(walk_smem(OEQ_MOST_GROUPS))) return rc;
        if (int rc = allow_smem<oeq_row_groups_place>(walk_smem(OEQ_MOST_GROUPS) + table_smem(OEQ_MOST_GROUPS))) return rc;
        oeq_row_groups_count<<<ctas, 32 * RG_WARPS, smem, st>>>(in, rows, r.run, r.runs, (int)groups, counts);
        OEQ_CUDA(cudaGetLastError());
        oeq_row_groups_scan<<<(unsigned)((keys + 7) / 8), 1024, 0, st>>>(counts, totals, r.runs, keys);
        OEQ_CUDA(cudaGetLastError());
        oeq_row_groups_place<<<ctas, 32 * RG_WARPS, smem_place, st>>>(in, rows, r.run, r.runs, (int)groups, n, counts, totals, ord, slt, off, blocks);
    }
    OEQ_CUDA(cudaGetLastError());
    return OEQ_OK;
}

int oeq_row_groups_from_counts(int64_t rows, int64_t groups, const int64_t* counts, int64_t* index, int64_t* offsets, int32_t* blocks, void* stream) {
    if (int rc = check_groups(rows, groups)) return rc;
    if (!counts || !offsets || (rows > 0 && (!index || !blocks))) return oeq_fail(OEQ_ERR_INVALID, "null pointer");
    const int n = (int)oeq_row_groups_blocks(rows, groups);
    const size_t smem = table_smem(groups);
    if (int rc = allow_smem<oeq_row_groups_counts>(table_smem(OEQ_MOST_GROUPS))) return rc;
    const unsigned ctas = (unsigned)std::min<int64_t>(296, std::max<int64_t>(1, (rows + 511) / 512));
    oeq_row_groups_counts<<<ctas, 512, smem, (cudaStream_t)stream>>>((const long long*)counts, rows, (int)groups, n, (long long*)index, (long long*)offsets, blocks);
    OEQ_CUDA(cudaGetLastError());
    return OEQ_OK;
}

int oeq_grouped_create(const oeq_irrep* in, int n_in, const oeq_irrep* out, int n_out, oeq_grouped** handle) {
    if (!handle || n_in < 0 || n_out < 0 || (n_in && !in) || (n_out && !out)) return oeq_fail(OEQ_ERR_INVALID, "null or negative argument");
    *handle = nullptr;
    if (n_in > GP_BLOCKS || n_out > GP_BLOCKS)
        return oeq_fail(OEQ_ERR_UNSUPPORTED, "at most " + std::to_string(GP_BLOCKS) + " blocks of irreps on each side (join blocks of one irrep)");
    struct Block { int64_t off; int mul, l, parity; };
    std::vector<Block> a, b;
    auto lay_out = [](const oeq_irrep* src, int n, std::vector<Block>& to, int64_t& dim) {
        dim = 0;
        for (int i = 0; i < n; ++i) {
            if (src[i].mul < 0 || src[i].l < 0 || src[i].l > 64 || (src[i].parity != 1 && src[i].parity != -1)) return false;
            to.push_back({dim, src[i].mul, src[i].l, src[i].parity});
            dim += (int64_t)src[i].mul * (2 * src[i].l + 1);
        }
        return dim < (int64_t(1) << 24);
    };
    int64_t a_dim = 0, b_dim = 0, numel = 0;
    if (!lay_out(in, n_in, a, a_dim) || !lay_out(out, n_out, b, b_dim)) return oeq_fail(OEQ_ERR_INVALID, "malformed irreps");
    struct Path { int i, o; int64_t w; };
    std::vector<Path> paths;
    for (int i = 0; i < n_in; ++i)
        for (int o = 0; o < n_out; ++o)
            if (a[i].l == b[o].l && a[i].parity == b[o].parity && a[i].mul && b[o].mul) {
                paths.push_back({i, o, numel});
                numel += (int64_t)a[i].mul * b[o].mul;
            }
    if (paths.size() > (size_t)GP_PATHS) return oeq_fail(OEQ_ERR_UNSUPPORTED, "at most " + std::to_string(GP_PATHS) + " paths (join blocks of one irrep)");
    if (numel >= (int64_t(1) << 30)) return oeq_fail(OEQ_ERR_UNSUPPORTED, "2^30 weights of a group or more");
    // 1 / sqrt(channels that are summed): the same for every path of an irrep, so that the gradients have it too
    auto scale = [&](const Block& x) {
        int64_t n = 0;
        for (const Block& y : a) n += y.l == x.l && y.parity == x.parity ? y.mul : 0;
        return n ? 1.0 / std::sqrt((double)n) : 0.0;
    };
    oeq_grouped* h = new oeq_grouped();
    auto fill = [&](GpProblem& gp, const std::vector<Block>& dst, int64_t src_dim, int64_t dst_dim, bool transposed) {
        gp.n_targets = (int)dst.size();
        gp.src_dim = (int)src_dim;
        gp.dst_dim = (int)dst_dim;
        gp.w_numel = (int)numel;
        gp.transposed = transposed;
        int n = 0;
        for (int t = 0; t < gp.n_targets; ++t) {
            GpTarget& to = gp.target[t];
            to = {(int)dst[t].off, dst[t].mul, 2 * dst[t].l + 1, n, n, scale(dst[t])};
            for (const Path& p : paths)
                if ((transposed ? p.i : p.o) == t) {
                    const Block& src = transposed ? b[p.o] : a[p.i];
                    gp.path[n++] = {transposed ? p.o : p.i, src.mul, (int)src.off, (int)p.w, b[p.o].mul, t};
                }
            to.path_end = n;
        }
        gp.n_paths = n;
    };
    fill(h->forward, b, a_dim, b_dim, false);
    fill(h->backward, a, b_dim, a_dim, true);
    h->weights = h->forward;
    std::sort(h->weights.path, h->weights.path + h->weights.n_paths, [](const GpPath& x, const GpPath& y) { return x.w_off < y.w_off; });
    for (const Path& p : paths) h->d_max = std::max(h->d_max, 2 * a[p.i].l + 1);
    *handle = h;
    return OEQ_OK;
}

int oeq_grouped_destroy(oeq_grouped* h) {
    delete h;
    return OEQ_OK;
}

int64_t oeq_grouped_weight_numel(const oeq_grouped* h) { return h ? h->forward.w_numel : 0; }

int oeq_grouped_forward(oeq_grouped* h, int dtype, int64_t rows, int64_t groups, const void* X, const void* W, const int64_t* order, const int64_t* offsets,
                        const int32_t* blocks, void* Z, void* stream) {
    if (int rc = check_call(h, dtype, rows, groups)) return rc;
    return product<false>(h, dtype, rows, groups, X, W, order, offsets, blocks, Z, stream);
}

int oeq_grouped_backward_input(oeq_grouped* h, int dtype, int64_t rows, int64_t groups, const void* dZ, const void* W, const int64_t* order,
                               const int64_t* offsets, const int32_t* blocks, void* dX, void* stream) {
    if (int rc = check_call(h, dtype, rows, groups)) return rc;
    return product<true>(h, dtype, rows, groups, dZ, W, order, offsets, blocks, dX, stream);
}

size_t oeq_grouped_workspace_bytes(const oeq_grouped* h, int dtype, int64_t rows, int64_t groups) {
    int sms = 0;
    if (!h || rows < 0 || !known_dtype(dtype) || h->weights.n_paths == 0 || sm_count(sms)) return 0;
    const GpProblem& gp = h->weights;
    const bool tc = dtype != OEQ_F64 && h->d_max <= GT_D_MAX;
    const GpSplit s = tc ? tc_split(gp, rows, groups, sms) : simt_split(gp, rows, sms);
    const size_t tile = tc ? GD_TILE * GD_TILE * sizeof(float) : GP_TILE * GP_TILE * std::max<size_t>(4, elem_bytes(dtype));
    return positions_bytes(gp, s) + partial_ctas(gp, s) * 2 * tile;
}

int oeq_grouped_backward_weights(oeq_grouped* h, int dtype, int64_t rows, int64_t groups, const void* X, const void* dZ, const int64_t* order,
                                 const int64_t* offsets, void* dW, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_call(h, dtype, rows, groups)) return rc;
    const GpProblem& gp = h->weights;
    if (gp.w_numel == 0) return OEQ_OK;
    if (!offsets || !dW || (rows > 0 && (!X || !dZ))) return oeq_fail(OEQ_ERR_INVALID, "null pointer");
    // (partial sums are written and joined in pieces of 16 bytes, four FP64 sums at a time)
    if (!aligned(workspace, WORKSPACE_ALIGN)) return oeq_fail(OEQ_ERR_INVALID, "workspace must be aligned to " + std::to_string(WORKSPACE_ALIGN) + " bytes");
    const size_t want = oeq_grouped_workspace_bytes(h, dtype, rows, groups);
    if (want == 0 || workspace_bytes < want || !workspace) return oeq_fail(OEQ_ERR_INVALID, "workspace too small");
    const cudaStream_t st = (cudaStream_t)stream;
    const bool tc = h->d_max <= GT_D_MAX;
    switch (dtype) {
        case OEQ_F64: return simt_weights<double>(gp, rows, groups, X, dZ, order, offsets, dW, workspace, st);
        case OEQ_F32: return tc ? tc_weights<float>(gp, rows, groups, X, dZ, order, offsets, dW, workspace, st)
                                : simt_weights<float>(gp, rows, groups, X, dZ, order, offsets, dW, workspace, st);
        case OEQ_BF16: return tc ? tc_weights<__nv_bfloat16>(gp, rows, groups, X, dZ, order, offsets, dW, workspace, st)
                                 : simt_weights<__nv_bfloat16>(gp, rows, groups, X, dZ, order, offsets, dW, workspace, st);
        default: return tc ? tc_weights<__half>(gp, rows, groups, X, dZ, order, offsets, dW, workspace, st)
                           : simt_weights<__half>(gp, rows, groups, X, dZ, order, offsets, dW, workspace, st);
    }
}

// (the copy alone is ordered behind the default stream and the streams that block with it: the device is waited for)
int oeq_grouped_check(void) {
    int code = 0;
    OEQ_CUDA(cudaDeviceSynchronize());
    OEQ_CUDA(cudaMemcpyFromSymbol(&code, gt_status, sizeof code));
    if (code == 0) return OEQ_OK;
    const int none = 0;
    OEQ_CUDA(cudaMemcpyToSymbol(gt_status, &none, sizeof none));
    return oeq_fail(OEQ_ERR_DEVICE_WAIT, "a kernel abandoned a bounded wait (code " + std::to_string(code) + ")");
}

int oeq_selftest_grouped_issue(void* stream) {
    if (int rc = allow_smem<oeq_grouped_issue_probe>(GT_PROBE_SMEM)) return rc;
    GtProblem gt{};
    gt.gp.n_targets = gt.gp.n_paths = 1;
    gt.gp.target[0] = {0, 16, 1, 0, 1, 1.0};
    gt.gp.path[0] = {0, 16, 0, 0, 16, 0};
    gt.target[0] = {1, 16, 1, 0, GT_PROBE_STAGES, 1, 1, 0};
    oeq_grouped_issue_probe<<<1, 32, GT_PROBE_SMEM, (cudaStream_t)stream>>>(gt);
    OEQ_CUDA(cudaGetLastError());
    return OEQ_OK;
}

int oeq_selftest_grouped_drain(int warp, void* stream) {
    if (warp < -1 || warp >= GT_EPI) return oeq_fail(OEQ_ERR_INVALID, "warp must be in -1 .. " + std::to_string(GT_EPI - 1));
    for (const int channels : {16, GT_PROBE_COLUMNS}) {         // one chunk of a tile (a group has none in turn) and three
        GtProblem gt{};
        gt.gp.n_targets = gt.gp.n_paths = 1;
        gt.gp.dst_dim = channels;
        gt.gp.target[0] = {0, channels, 1, 0, 1, 1.0};
        gt.target[0] = {1, channels, 1, 0, 1, 1, 1, 0};
        oeq_grouped_drain_probe<<<1, 32 * GT_EPI, 0, (cudaStream_t)stream>>>(gt, warp);
        OEQ_CUDA(cudaGetLastError());
    }
    return OEQ_OK;
}

int oeq_selftest_grouped_wait(int polls, void* stream) {
    if (polls < 1 || polls > (1 << 20)) return oeq_fail(OEQ_ERR_INVALID, "polls must be in 1 .. 2^20");
    oeq_grouped_wait_probe<<<1, 32, 0, (cudaStream_t)stream>>>((unsigned)polls);
    OEQ_CUDA(cudaGetLastError());
    return OEQ_OK;
}

}  // extern "C"
