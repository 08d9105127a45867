// Linear maps of irreps with one set of weights for each group of rows, without tcgen05: FP64, and in every
// type the maps that have a path of l = 4 or above, all of their paths.
//
//   Z[r,o,w,k] = c_o sum_{i,u} W_g[i,o][u,w] X[r,i,u,k],  g = group of row r          (product; dX with W transposed)
//   dW_g[i,o][u,w] = c_o sum_{r in g, k} X[r,i,u,k] dZ[r,o,w,k]                        (weight gradient)
//
// Both kernels are 64 x 64 products in registers, 16 values of a thread; 16 steps of the sum are staged in shared memory while the next 16
// are on their way in registers.  FP64 goes through mma.m8n8k4 (there is no FP64 kind of tcgen05.mma): 10 007 rows of 64x(0e+1o+2e) 61 us, weight
// gradient 60 and 20 for the join, 12 and 9 TFLOP/s; with FMAs 102 and 129.  Bound by latency with two or three CTAs an SM: issue 42 %, load and store unit 49 %, FP64 tensor
// pipe 35 %.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "oeq_common.cuh"

namespace oeq {

constexpr int GP_BLOCKS = 32, GP_PATHS = 64;    // blocks of an Irreps and paths that fit the kernels' parameters

struct GpPath {
    int src, src_mul, src_off;  // source block, its multiplicity and first column
    int w_off, w_ld;            // first weight; weights between neighbouring input channels
    int dst;                    // target block
};
struct GpTarget {
    int off, mul, d;            // first column, multiplicity, components
    int path_begin, path_end;
    double scale;
};
// A linear map from a source row to a target row.
struct GpProblem {
    int n_targets, n_paths, src_dim, dst_dim, w_numel;
    bool transposed;            // the sum runs over the weights' output channels
    GpTarget target[GP_BLOCKS];
    GpPath path[GP_PATHS];
};

// ---- types: sums are held in FP32, those of FP64 values in FP64
template <class T> struct GpAcc { typedef float type; };
template <> struct GpAcc<double> { typedef double type; };
__device__ __forceinline__ float gp_load(const float* p) { return __ldg(p); }
__device__ __forceinline__ double gp_load(const double* p) { return __ldg(p); }
__device__ __forceinline__ float gp_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float gp_load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void gp_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void gp_store(double* p, double v) { *p = v; }
__device__ __forceinline__ void gp_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void gp_store(__half* p, float v) { *p = __float2half_rn(v); }

// The last group g in [0, groups) with offsets[g] <= p; p < offsets[groups].
__device__ __forceinline__ int gp_group(const long long* __restrict__ offsets, int groups, long long p) {
    int lo = 0, hi = groups - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(offsets + mid) <= p) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
__device__ __forceinline__ long long gp_row(const long long* __restrict__ order, long long p) { return order ? __ldg(order + p) : p; }

// The grouped rows are cut into `parts` equal ranges of sorted positions.
__device__ __forceinline__ long long gp_cut(long long n, int part, int parts) { return (long long)((unsigned long long)n * part / parts); }
constexpr int GP_TILE = 64, GP_STEP = 16, GP_SIMT_THREADS = 256;
// A 64 x 64 product by 256 threads, 16 values each, over GP_STEP staged steps.  PITCH of a staged step: 16 steps by two rows, which a warp
// writes, and what it reads lie in different banks, or two at most to a bank (a pitch of 64 values: 120 us instead of 102 with FMAs).
// LONG: a sum of many terms is added up in chains of 512: the error of one chain grows with its length (FP32, relative, norm: 36 000 terms 3.4e-6, in
// chains 4.3e-7).  The chains' sum is in shared memory, where it costs no registers (in registers: three CTAs an SM instead of four, 10 000 rows
// of 256x4e FP32 571 us instead of 526, product).  For FP32 results; 16-bit ones are rounded by up to 2^-8 and 2^-11.
constexpr int GP_CHAIN = 512 / GP_STEP;         // steps
template <class A, bool LONG> struct GpProduct {            // FMA: 4 rows by 4 columns of a thread
    static constexpr int PITCH = GP_TILE + 2;
    A acc[16] = {};
    int steps = 0;
    static __device__ A* chains() {             // of the thread, GP_SIMT_THREADS apart
        __shared__ A sum[16 * GP_SIMT_THREADS];
        return sum + threadIdx.x;
    }
    __device__ A result(int i) const {
        if (LONG && steps >= GP_CHAIN) return chains()[i * GP_SIMT_THREADS] + acc[i];
        return acc[i];
    }
    static __device__ int row(int i) { return threadIdx.x / 16 * 4 + (i >> 2); }
    static __device__ int col(int i) { return threadIdx.x % 16 * 4 + (i & 3); }
    __device__ void multiply(const A (*a)[PITCH], const A (*b)[PITCH]) {
#pragma unroll
        for (int k = 0; k < GP_STEP; ++k) {
            A x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = a[k][row(4 * i)];
                y[i] = b[k][col(i)];
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[i] += x[i >> 2] * y[i & 3];
        }
        if (!LONG || ++steps % GP_CHAIN) return;
        A* sum = chains();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            sum[i * GP_SIMT_THREADS] = steps == GP_CHAIN ? acc[i] : sum[i * GP_SIMT_THREADS] + acc[i];
            acc[i] = A(0);
        }
    }
};
// FP64: mma.m8n8k4, rounded as FMAs are; a warp has 16 rows by 32 columns, six values to read for eight products of 8 x 8 x 4 where the FMAs
// of a thread read eight for sixteen.
template <bool LONG> struct GpProduct<double, LONG> {
    static constexpr int PITCH = GP_TILE + 10;
    double acc[16] = {};
    __device__ double result(int i) const { return acc[i]; }
    static __device__ int row(int i) { return (threadIdx.x >> 6) * 16 + (i >> 3) * 8 + (threadIdx.x & 31) / 4; }
    static __device__ int col(int i) { return (threadIdx.x >> 5 & 1) * 32 + (i >> 1 & 3) * 8 + 2 * (threadIdx.x & 3) + (i & 1); }
    __device__ void multiply(const double (*a)[PITCH], const double (*b)[PITCH]) {
        const int k0 = threadIdx.x & 3, m0 = row(0), n0 = (threadIdx.x >> 5 & 1) * 32 + (threadIdx.x & 31) / 4;
#pragma unroll
        for (int k = 0; k < GP_STEP; k += 4) {
            double x[2], y[4];
#pragma unroll
            for (int i = 0; i < 2; ++i) x[i] = a[k + k0][m0 + 8 * i];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = b[k + k0][n0 + 8 * j];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    double* c = acc + 8 * i + 2 * j;
                    asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};" : "+d"(c[0]), "+d"(c[1]) : "d"(x[i]), "d"(y[j]));
                }
        }
    }
};

// ---------------------------------------------------------------------------- product
// CTA (x, y): entry x of the block table and column first_column + y; a column is a target block, 64 of its channels and 64 of the block's up
// to 64 d (row, component) pairs.  Row y of the grid behind the table writes the zeros of the rows without a group.
template <class T>
__global__ void __launch_bounds__(GP_SIMT_THREADS, sizeof(T) == 4 ? 4 : 0) oeq_grouped_simt(const __grid_constant__ GpProblem gp, const T* __restrict__ X, const T* __restrict__ W,
                                                                    const long long* __restrict__ order, const long long* __restrict__ offsets,
                                                                    const int* __restrict__ table, int blocks, long long rows, int groups,
                                                                    int first_column, T* __restrict__ Z) {
    typedef typename GpAcc<T>::type A;
    typedef GpProduct<A, sizeof(T) == 4> Product;
    __shared__ __align__(16) A sa[GP_STEP][Product::PITCH], sb[GP_STEP][Product::PITCH];
    const int tid = threadIdx.x;
    if ((int)blockIdx.x >= blocks) {            // rows without a group: zeros
        const long long n = min(__ldg(offsets + groups), rows), part = (long long)(blockIdx.x - blocks) * gridDim.y + blockIdx.y;
        const long long parts = (long long)(gridDim.x - blocks) * gridDim.y;
        for (long long i = part * blockDim.x + tid; i < (rows - n) * gp.dst_dim; i += parts * blockDim.x)
            gp_store(Z + gp_row(order, n + i / gp.dst_dim) * gp.dst_dim + i % gp.dst_dim, A(0));
        return;
    }
    const int g = table[3 * blockIdx.x], n_rows = table[3 * blockIdx.x + 2];
    const long long first = table[3 * blockIdx.x + 1];
    if (g < 0) return;
    int t = 0, column = first_column + (int)blockIdx.y;
    for (; t < gp.n_targets; ++t) {
        const int n = (gp.target[t].mul + GP_TILE - 1) / GP_TILE * gp.target[t].d;
        if (column < n) break;
        column -= n;
    }
    const GpTarget& to = gp.target[t];
    const int d = to.d, pair0 = column % d * GP_TILE, pairs = n_rows * d, c_tile = column / d * GP_TILE;
    if (pair0 >= pairs) return;
    // staging: thread -> (step, 4 rows apart) of A and of B
    const int k_a = tid % GP_STEP, r_a = tid / GP_STEP;
    const T* x_row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int pair = pair0 + r_a + 16 * i;
        x_row[i] = pair < pairs ? X + gp_row(order, first + pair / d) * gp.src_dim + pair % d : nullptr;
    }
    const T* w_group = W + (long long)g * gp.w_numel;
    const int kb = gp.transposed ? tid % GP_STEP : tid / 16 % GP_STEP, cb = gp.transposed ? tid / GP_STEP : tid % 16;
    Product product;
    A a[4], b[4];
    int p = to.path_begin, u0 = 0;
    auto fetch = [&]() {
        const GpPath& path = gp.path[p];
        const T* w = w_group + path.w_off;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int u = u0 + k_a;
            a[i] = x_row[i] && u < path.src_mul ? (A)gp_load(x_row[i] + path.src_off + u * d) : A(0);
            const int v = u0 + kb, c = c_tile + cb + 16 * i;
            b[i] = v < path.src_mul && c < to.mul ? (A)gp_load(w + (gp.transposed ? (long long)c * path.w_ld + v : (long long)v * path.w_ld + c)) : A(0);
        }
        u0 += GP_STEP;
        if (u0 >= path.src_mul) {
            ++p;
            u0 = 0;
        }
    };
    if (p < to.path_end) fetch();
    for (bool more = to.path_begin < to.path_end; more;) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sa[k_a][r_a + 16 * i] = a[i];
            sb[kb][cb + 16 * i] = b[i];
        }
        __syncthreads();
        more = p < to.path_end;
        if (more) fetch();
        product.multiply(sa, sb);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int pair = pair0 + product.row(i), c = c_tile + product.col(i);
        if (pair >= pairs || c >= to.mul) continue;
        gp_store(Z + gp_row(order, first + pair / d) * gp.dst_dim + to.off + pair % d + c * d, (A)(product.result(i) * (A)to.scale));
    }
}

// ---------------------------------------------------------------------------- weight gradient
// A CTA has a path, a tile of its weights and a range of the sorted rows.  A group that lies within the range is complete; the part of
// one that began before it goes to slot 0 of the CTA's two partial tiles, the part of one that goes on behind it to slot 1.
// oeq_grouped_join adds the parts in the order of the ranges: no atomics, the same sums in every run.
constexpr int GP_PARTS = 1024;                  // most ranges of a path
// First sorted position of a CTA's range, and its group.
struct GpStart { int lo, group; };
struct GpSplit {
    int parts[GP_PATHS];        // ranges of each path
    int first[GP_PATHS + 1];    // its first CTA
};
template <class T>
__global__ void __launch_bounds__(GP_SIMT_THREADS, sizeof(T) == 4 ? 4 : 0) oeq_grouped_simt_dw(const __grid_constant__ GpProblem gp, const __grid_constant__ GpSplit split,
                                                                       const T* __restrict__ X, const T* __restrict__ dZ,
                                                                       const long long* __restrict__ order, const long long* __restrict__ offsets,
                                                                       long long rows, int groups, T* __restrict__ dW,
                                                                       typename GpAcc<T>::type* __restrict__ partial, GpStart* __restrict__ starts) {
    typedef typename GpAcc<T>::type A;
    typedef GpProduct<A, sizeof(T) == 4> Product;
    __shared__ __align__(16) A sa[GP_STEP][Product::PITCH], sb[GP_STEP][Product::PITCH];
    const int tid = threadIdx.x;
    int p = 0;
    while ((int)blockIdx.x >= split.first[p + 1]) ++p;
    const GpPath& path = gp.path[p];
    const GpTarget& to = gp.target[path.dst];
    const int parts = split.parts[p], part = ((int)blockIdx.x - split.first[p]) % parts, tile_of = ((int)blockIdx.x - split.first[p]) / parts;
    const int w_tiles = (to.mul + GP_TILE - 1) / GP_TILE, u_tile = tile_of / w_tiles * GP_TILE, w_tile = tile_of % w_tiles * GP_TILE, d = to.d;
    const long long n = min(__ldg(offsets + groups), rows), lo = gp_cut(n, part, parts), hi = gp_cut(n, part + 1, parts);
    int g = lo < n ? gp_group(offsets, groups, lo) : 0;
    if (tid == 0) starts[blockIdx.x] = {(int)lo, g};
    if (lo >= hi) return;
    const int k_s = tid / 16, c_s = tid % 16;
    for (long long at = lo; at < hi;) {
        long long begin = __ldg(offsets + g), end = __ldg(offsets + g + 1);
        if (end <= at) {                        // (a group without rows)
            ++g;
            continue;
        }
        const long long stop = min(end, hi);
        const long long pairs = (stop - at) * d;
        Product product;
        A a[4], b[4];
        auto fetch = [&](long long k0) {
            const long long k = k0 + k_s;
            const bool in = k < pairs;
            const long long row = in ? gp_row(order, at + k / d) : 0;
            const T *x = X + row * gp.src_dim + path.src_off + k % d, *z = dZ + row * gp.dst_dim + to.off + k % d;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int u = u_tile + c_s + 16 * i, w = w_tile + c_s + 16 * i;
                a[i] = in && u < path.src_mul ? (A)gp_load(x + u * d) : A(0);
                b[i] = in && w < to.mul ? (A)gp_load(z + w * d) : A(0);
            }
        };
        fetch(0);
        for (long long k0 = 0; k0 < pairs; k0 += GP_STEP) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sa[k_s][c_s + 16 * i] = a[i];
                sb[k_s][c_s + 16 * i] = b[i];
            }
            __syncthreads();
            if (k0 + GP_STEP < pairs) fetch(k0 + GP_STEP);
            product.multiply(sa, sb);
        }
        const bool whole = begin >= lo && end <= hi;
        A* tile = whole ? nullptr : partial + ((long long)blockIdx.x * 2 + (begin < lo ? 0 : 1)) * (GP_TILE * GP_TILE);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = product.row(i), c = product.col(i), u = u_tile + r, w = w_tile + c;
            if (!whole) tile[r * GP_TILE + c] = product.result(i);
            else if (u < path.src_mul && w < to.mul) gp_store(dW + (long long)g * gp.w_numel + path.w_off + (long long)u * path.w_ld + w, (A)(product.result(i) * (A)to.scale));
        }
        at = stop;
        ++g;
    }
}

// Gradients of the groups that no single range has, which are those with the first row of some range behind their own: a CTA for each
// range and four rows of its tile.  The CTA of the first such range adds up the group's parts, 256 / TILE threads to four weights, in a fixed
// order.  Behind them `zero_ctas` CTAs write the zeros of the groups without rows.  (A CTA for every tile and group takes 25 us for 89 groups
// and three paths of 128 x 128, most of it to find that a group is complete.)
template <class T, int TILE>
__global__ void __launch_bounds__(256) oeq_grouped_join(const __grid_constant__ GpProblem gp, const __grid_constant__ GpSplit split,
                                                        const long long* __restrict__ offsets, long long rows, int groups, int zero_ctas,
                                                        const typename GpAcc<T>::type* __restrict__ partial, const GpStart* __restrict__ starts, T* __restrict__ dW) {
    typedef typename GpAcc<T>::type A;
    constexpr int SLICE = 4, SLICES = TILE / SLICE, SHARES = 256 / TILE;
    struct alignas(4 * sizeof(A)) Four { A v[4]; };
    __shared__ int list[GP_PARTS + 2];          // partial tiles that are added, and their number
    __shared__ Four sums[256];
    const long long n = min(__ldg(offsets + groups), rows);
    const int ctas = split.first[gp.n_paths];
    if ((int)blockIdx.x >= ctas * SLICES) {
        for (int g = blockIdx.x - ctas * SLICES; g < groups; g += zero_ctas)
            if (min(__ldg(offsets + g), n) >= min(__ldg(offsets + g + 1), n))
                for (int i = threadIdx.x; i < gp.w_numel; i += 256) gp_store(dW + (long long)g * gp.w_numel + i, A(0));
        return;
    }
    const int c = blockIdx.x / SLICES, u_slice = blockIdx.x % SLICES * SLICE;
    int p = 0;
    while (c >= split.first[p + 1]) ++p;
    const int parts = split.parts[p], j = (c - split.first[p]) % parts, tile = (c - split.first[p]) / parts;
    if (j == 0 || starts[c].lo >= n) return;
    const int lo = starts[c].lo, g = starts[c].group;
    const GpStart* of = starts + (c - j);       // of the tile's ranges
    const int begin = (int)__ldg(offsets + g), end = (int)min(__ldg(offsets + g + 1), n);
    if (begin >= lo || of[j - 1].lo > begin) return;        // no group goes on here, or an earlier range has seen to it
    const GpPath& path = gp.path[p];
    const GpTarget& to = gp.target[path.dst];
    const int w_tiles = (to.mul + TILE - 1) / TILE, u0 = tile / w_tiles * TILE + u_slice, w0 = tile % w_tiles * TILE, nu = min(SLICE, path.src_mul - u0), nw = min(TILE, to.mul - w0);
    if (nu <= 0) return;
    if (threadIdx.x < 32) {                     // the first range's part, then those of the others that have rows of the group
        int count = 1;
        if (threadIdx.x == 0) list[0] = 2 * (j - 1) + 1;
        for (int i = j;; i += 32) {
            const int k = i + threadIdx.x;
            const bool in = k < parts && of[k].lo < end, some = in && (k + 1 == parts || of[k + 1].lo > of[k].lo);
            const unsigned all = __ballot_sync(0xffffffffu, some);
            if (some) list[count + __popc(all & ((1u << threadIdx.x) - 1))] = 2 * k;
            count += __popc(all);
            if (!__all_sync(0xffffffffu, in)) break;
        }
        if (threadIdx.x == 0) list[GP_PARTS + 1] = count;
    }
    __syncthreads();
    const int count = list[GP_PARTS + 1], i = 4 * (threadIdx.x % TILE), share = threadIdx.x / TILE;
    const A* at = partial + (long long)(c - j) * 2 * (TILE * TILE) + u_slice * TILE + i;
    Four s = {};
#pragma unroll 8
    for (int k = share; k < count; k += SHARES) {
        const Four v = *reinterpret_cast<const Four*>(at + (long long)list[k] * (TILE * TILE));
#pragma unroll
        for (int e = 0; e < 4; ++e) s.v[e] += v.v[e];
    }
    sums[threadIdx.x] = s;
    __syncthreads();
    const int u = i / TILE;
    if (share > 0 || u >= nu) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int w = i % TILE + e;
        if (w >= nw) break;
        A all = s.v[e];
        for (int k = 1; k < SHARES; ++k) all += sums[threadIdx.x + k * TILE].v[e];
        gp_store(dW + (long long)g * gp.w_numel + path.w_off + (long long)(u0 + u) * path.w_ld + w0 + w, (A)(all * (A)to.scale));
    }
}

}  // namespace oeq
