// Linear maps of irreps with one set of weights for each group of rows, on the 5th-generation tensor cores: FP32 (3xTF32),
// BF16 and FP16, up to GT_D_MAX components.  FP32 accumulators.
//
//   Z[r,o,w,k] = c_o sum_{i,u} W_g[i,o][u,w] X[r,i,u,k],  g = group of row r; dX is the same with W transposed.
//
// As a matrix product: M = (row, component) pairs of sorted rows of one group, N = channels of one output block, K = channels of
// the input blocks with its irrep.  A CTA has one output block (or a tile of its channels) and one range of the sorted rows, the
// CTAs being dealt to the output blocks by cost, so a CTA meets few groups and keeps a group's weights in shared memory.
//   * 12 producer warps: a lane reads the 16 d bytes of V = 4 (16-bit types: 8) channels of a row, [channel][component], and writes
//     d pieces of 16 bytes, one per (row, component), K-major with the 128-byte swizzle.  The transposition that the layout of irreps
//     asks for costs no extra pass, rows are gathered in sorted order, and FP32 values are split into TF32 hi and lo on the way.
//     Three sets of four warps take the chunks of K in turn: each has its chunk on the way in registers before it waits for a stage, and the
//     time of a load, some 2 000 cycles, passes once for three chunks.  (With fewer stages than sets the sets wait for their stages one after
//     the other, by a barrier that goes round: a set that waited out of turn could not tell a stage's phases apart.)
//     Weights have their output channels along memory: "MN-major" tiles for Z, K-major for dX; neither is transposed.
//   * one warp, in step, issues the MMAs.  FP32: hi.hi and hi.lo as one MMA over the weights' hi channels followed by lo, lo.hi
//     into hi.lo's columns: the large and the small products have accumulators of their own.
//   * 8 epilogue warps, in two groups, add those, scale, and write rows through shared memory, so that a row's values leave in order.
//   * 3 warps prefetch rows and weights to L2, up to two tiles ahead of the MMAs: a producer's loads are half of its time, and registers for
//     more of them on the way there are none.
// Two accumulators: a tile (FP32: up to 256 channels of its sum) drains while the next is computed.  Every wait is bounded; on expiry a role records a code and all
// leave, the drain by way of its barriers and the MMA warp once its MMAs are over.
// Measured from a cold L2, 50 000 rows in 10 groups, 128x(0e+1o+2e+3o) FP32: 227 us (3.6 TB/s of rows in and out, 115 TFLOP/s); 100 000 rows in 256
// groups, 128x(0e+1o+2e) BF16: 145 us (3.3 TB/s).  The load and store unit bounds it (71 % of its wavefronts: rows of several components are read
// with a stride of 16 d bytes, results staged with two lanes to a bank), then issue (42 %); the tensor pipe is at 34 % (BF16 9 %).
#pragma once
#include "grouped_kernels.cuh"
#include "tc_common.cuh"

namespace oeq {

constexpr int GT_D_MAX = 7;
constexpr int GT_SETS = 3, GT_SET = 4, GT_PW = GT_SETS * GT_SET, GT_EPI_GROUPS = 2, GT_EPI = 4 * GT_EPI_GROUPS, GT_AHEAD = 3, GT_THREADS = (GT_PW + GT_EPI + 1 + GT_AHEAD) * 32;
constexpr int GT_STAGES = 6;                    // most stages of A
// FP32: chunks of the sum in one accumulator, 32 additions of eight channels each.  The additions are cut off, not rounded, and all of them
// one way: relative error (norm) 6.4e-7 at 256 channels, in one chain 4.9e-6 at 2 048 and 9.6e-6 at 4 096, in chains 6.6e-7 at most.  What the
// drains of more than one chain cost, product: 65 536 rows of 512x0e 277 us instead of 260, 20 000 of 1024x0e 328 instead of 293, 30 000 of 300x1o 225
// instead of 178 (chains of five and five chunks instead of eight and two: 226).  Kernels of their own (LONG): with the loop in all of them dX of
// 50 000 rows of 128x(0e+1o+2e+3o) took 225 us instead of 219.  16-bit results are rounded by up to 2^-8 and 2^-11, and an
// addition takes 16 channels: one chain, short by 5e-6 at 4 096 channels.
constexpr int GT_CHAIN = 8;
constexpr int GT_STAGING = 42 * 100 * 4;        // 32 channels of a tile's pairs (three components take most), for each epilogue group
constexpr int GT_CONTROL = 1536;                // barriers, rows of the tiles that drain, the CTA's range
constexpr int ERR_GT_EMPTY = 81, ERR_GT_FULL = 82, ERR_GT_ACC_FULL = 83, ERR_GT_ACC_EMPTY = 84, ERR_GT_TURN = 85, ERR_GT_DONE = 86;

// Set by a kernel whose bounded wait ran out; read by oeq_grouped_check.
__device__ int gt_status;

struct GtTarget {
    int n_tiles, n;             // tiles of its channels, channels of a tile (a multiple of 16)
    int parts, first;           // ranges of rows, first CTA
    int stages, slots;          // of A, of B
    int chunks;                 // of the sum
    int extra;                  // time of a group's weights, in rows
};
struct GtProblem {
    GpProblem gp;
    GtTarget target[GP_BLOCKS];
};

// Rows of a tile.  Seven components: 16 rows (112 of 128 pairs) are one piece for every lane of a set, 18 would be two.
__host__ __device__ constexpr int gt_tile_rows(int d) { return d == 7 ? 16 : 128 / d; }

template <class T> struct GtType {              // 16-bit
    static constexpr int V = 8, KC = 64, KSTEP = 16, A_BYTES = 16384, N_MAX = 256;
    static constexpr bool SPLIT = false;
    __host__ __device__ static constexpr int b_bytes(int n) { return (n + 63) / 64 * 8192; }
    __host__ __device__ static constexpr int acc(int n) { return n; }
};
template <> struct GtType<float> {
    static constexpr int V = 4, KC = 32, KSTEP = 8, A_BYTES = 32768, N_MAX = 128;
    static constexpr bool SPLIT = true;
    __host__ __device__ static constexpr int b_bytes(int n) { return n * 256; }
    __host__ __device__ static constexpr int acc(int n) { return 2 * n; }
};

// ---- instruction descriptor and MMA of the type; A is K-major
template <class T, bool B_MN> __device__ __forceinline__ unsigned gt_idesc(int n) {
    const unsigned fmt = GtType<T>::SPLIT ? 2u : (sizeof(T) == 2 && __is_same(T, __nv_bfloat16) ? 1u : 0u);
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (B_MN ? 1u << 16 : 0u) | ((unsigned)(n >> 3) << 17) | (8u << 24);
}
template <class T>
__device__ __forceinline__ void gt_mma(unsigned leader, unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, unsigned accumulate) {
    if constexpr (GtType<T>::SPLIT) {
        tc_mma_if(leader, d, a, b, idesc, accumulate);
    } else {
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u), "r"(leader)
            : "memory");
    }
}
// ---- operand B [n channels] x [KC steps of the sum]
// K-major: rows of 128 bytes per channel, FP32: hi channels, then lo.  MN-major, FP32: per 8 steps, blocks of 32 channels by 8 steps
// (128-byte rows, 32-byte atoms swizzled over four rows), hi channels then lo; 16-bit: per 8 steps, blocks of 64 channels by 8 steps.
template <class T>
__device__ __forceinline__ int gt_place_mn(int n, int ch, int k) {
    if constexpr (GtType<T>::SPLIT) return (k >> 3) * (n * 64) + (ch >> 5) * 1024 + (k & 7) * 128 + (((ch & 31) * 4) ^ ((k & 3) << 5));
    else return (k >> 3) * ((n + 63) / 64 * 1024) + (ch >> 6) * 1024 + (k & 7) * 128 + ((((ch >> 3) & 7) ^ (k & 7)) << 4);
}
template <class T, bool B_MN>
__device__ __forceinline__ unsigned long long gt_desc_b(unsigned addr, int n) {
    const unsigned long long base = (unsigned long long)((addr >> 4) & 0x3fff) | (unsigned long long)(1024 >> 4) << 16 | 1ull << 46;
    if constexpr (!B_MN) return tc_smem_desc(addr);
    else if constexpr (GtType<T>::SPLIT) return base | (unsigned long long)(512 >> 4) << 32 | 1ull << 61;
    else return base | (unsigned long long)((n + 63) / 64 * 1024 >> 4) << 32 | 2ull << 61;
}
// bytes between two MMAs' steps
template <class T, bool B_MN> __device__ __forceinline__ int gt_step_b(int n) {
    if constexpr (!B_MN) return 32;
    else return GtType<T>::SPLIT ? n * 64 : 2 * ((n + 63) / 64 * 1024);
}

// ---- values
__device__ __forceinline__ void gt_split(const float4& v, float4& hi, float4& lo) {
    hi = make_float4(tf32_hi(v.x), tf32_hi(v.y), tf32_hi(v.z), tf32_hi(v.w));
    lo = make_float4(v.x - hi.x, v.y - hi.y, v.z - hi.z, v.w - hi.w);         // exact; read as TF32 by the MMA
}
// V channels of D components, as 16-byte words: `left` of the channels exist, the others are zero.  FAST: sixteen bytes at a time, for
// blocks of whole pieces; no branch, so that the loads of several pieces are on the way together.
template <class T, int D, bool FAST>
__device__ __forceinline__ void gt_read(uint4 (&v)[D], const T* __restrict__ src, int left) {
    if constexpr (FAST) {
#pragma unroll
        for (int i = 0; i < D; ++i) v[i] = left > 0 ? __ldg(reinterpret_cast<const uint4*>(src) + i) : make_uint4(0, 0, 0, 0);
    } else if constexpr (sizeof(T) == 4) {
        unsigned* w = reinterpret_cast<unsigned*>(v);
#pragma unroll
        for (int i = 0; i < 4 * D; ++i) w[i] = i / D < left ? __float_as_uint(__ldg(reinterpret_cast<const float*>(src) + i)) : 0u;
    } else {
        unsigned* w = reinterpret_cast<unsigned*>(v);
        const unsigned short* h = reinterpret_cast<const unsigned short*>(src);
#pragma unroll
        for (int i = 0; i < 4 * D; ++i)
            w[i] = (2 * i / D < left ? (unsigned)__ldg(h + 2 * i) : 0u) | ((2 * i + 1) / D < left ? (unsigned)__ldg(h + 2 * i + 1) << 16 : 0u);
    }
}
// 16 bytes to shared memory without a register on the way; zeros where !in.
__device__ __forceinline__ void gt_copy(void* dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void gt_copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void gt_copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// Byte offset of 16-byte piece c of row `row` of a K-major tile (128-byte rows, 128-byte swizzle).
__device__ __forceinline__ int gt_place_k(int row, int c) { return row * 128 + (((row ^ c) & 7) << 4); }
// The V channels of component k.
template <class T, int D>
__device__ __forceinline__ uint4 gt_component(const uint4 (&v)[D], int k) {
    const unsigned* w = reinterpret_cast<const unsigned*>(v);
    if constexpr (sizeof(T) == 4) {
        return make_uint4(w[k], w[D + k], w[2 * D + k], w[3 * D + k]);
    } else {
        unsigned o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int a = 2 * j * D + k, b = a + D;
            o[j] = __byte_perm(w[a >> 1], w[b >> 1], (a & 1 ? 0x32 : 0x10) | (b & 1 ? 0x7600 : 0x5400));
        }
        return make_uint4(o[0], o[1], o[2], o[3]);
    }
}

// ---- a CTA's tiles: up to 128 / d sorted rows of one group
struct GtWalk {
    int pos, hi, end;           // next position, end of the range, end of the group within it
    int g, rows;
    __device__ static int end_of(const long long* offsets, int g) { return (int)__ldg(offsets + g + 1); }
    __device__ GtWalk(const long long* offsets, int g_, int lo, int hi_) : pos(lo), hi(hi_), end(0), g(g_), rows(0) {
        if (lo < hi) end = min(end_of(offsets, g), hi);
    }
    __device__ bool more() const { return pos < hi; }
    __device__ void tile(int most) { rows = min(most, end - pos); }
    __device__ void next(const long long* offsets, int groups) {
        pos += rows;
        if (pos >= end && pos < hi) {
            ++g;
            end = end_of(offsets, g);
            if (end <= pos) {                   // groups without rows between
                g = gp_group(offsets, groups, pos);
                end = end_of(offsets, g);
            }
            end = min(end, hi);
        }
    }
};

// The CTA's range of sorted rows, by all threads: part `part` of `parts` equal lengths on an axis where every row has length 1
// and every group with rows `extra` more, in front of it: the time that its weights take.
struct GtRange {
    long long lo, hi;
    int g;                      // the group that row lo is in
    int sums[33];
};
__device__ __forceinline__ void gt_range(GtRange& out, const long long* __restrict__ offsets, int groups, long long rows, int part, int parts, int extra) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const int each = (groups + blockDim.x - 1) / blockDim.x, g0 = min(tid * each, groups), g1 = min(g0 + each, groups);
    const long long n = min(__ldg(offsets + groups), rows);
    int used = 0;
    long long at = g0 < g1 ? min(__ldg(offsets + g0), n) : n;
    const long long first = at;
    for (int g = g0; g < g1; ++g) {
        const long long end = min(__ldg(offsets + g + 1), n);
        used += end > at;
        at = end;
    }
    int s = used;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, s, off);
        if (lane >= off) s += t;
    }
    if (lane == 31) out.sums[warp] = s;
    if (tid == 0) out.lo = out.hi = n, out.g = 0;
    __syncthreads();
    int before = s - used, all = 0;
    for (int w = 0; w < warps; ++w) {
        before += w < warp ? out.sums[w] : 0;
        all += out.sums[w];
    }
    const long long length = n + (long long)all * extra, lo = gp_cut(length, part, parts), hi = gp_cut(length, part + 1, parts);
    at = first;
    for (int g = g0; g < g1; ++g) {
        const long long end = min(__ldg(offsets + g + 1), n);
        if (end > at) {
            const long long v = at + (long long)before * extra, w = v + extra + (end - at);         // the group's piece of the axis
            if (lo >= v && lo < w) {
                const long long p = at + max(lo - v - extra, 0ll);
                out.lo = p;
                out.g = g;
            }
            if (hi >= v && hi < w) out.hi = at + max(hi - v - extra, 0ll);
            ++before;
        }
        at = end;
    }
    __syncthreads();
}

struct GtArgs {
    const void *X, *W;
    const long long *order, *offsets;
    void* Z;
    long long rows;
    int groups;
    int z_vec;                  // rows of Z in 16-byte pieces
};
struct GtBars {
    unsigned long long *full, *empty, *acc_full, *acc_empty, *turn, *done;
    unsigned* tmem;
    volatile int* progress;     // tiles whose MMAs are on their way
    int* rows;                  // of the tile that drains, for each epilogue group
    __device__ explicit GtBars(unsigned char* control) {
        full = reinterpret_cast<unsigned long long*>(control);
        empty = full + GT_STAGES;
        acc_full = empty + GT_STAGES;
        acc_empty = acc_full + 2;
        turn = acc_empty + 2;
        done = turn + GT_SETS;
        tmem = reinterpret_cast<unsigned*>(done + 1);
        progress = reinterpret_cast<volatile int*>(tmem + 1);
        rows = reinterpret_cast<int*>(control + 512);      // (behind the range)
    }
};

// ---------------------------------------------------------------------------- producers
// A chunk of weights by the threads of a set, four pieces of 16 bytes of a lane on the way at once.
template <class T, bool TRANS, bool FAST>
__device__ __forceinline__ void gt_fill_b(unsigned char* dst, const T* __restrict__ w, int ld, int n, int n_left, int k_left, int k_fill, float scale, int member) {
    constexpr int V = GtType<T>::V, AT_ONCE = 4;
    const int across = TRANS ? 8 : n / V, pieces = TRANS ? n * 8 : k_fill * across;     // K-major: (channel, piece of K); MN-major: (k, piece of channels)
    const unsigned magic = (65536 + across - 1) / across;       // i / across for i < 2048, across <= 32
    if constexpr (FAST && !GtType<T>::SPLIT) {  // (16-bit weights are copied as they are)
        for (int i = member; i < pieces; i += GT_SET * 32) {
            const int row = TRANS ? i >> 3 : (int)((i * magic) >> 16), c = TRANS ? i & 7 : i - row * across;
            const bool in = TRANS ? row < n_left && c * V < k_left : row < k_left && c * V < n_left;
            gt_copy(dst + (TRANS ? gt_place_k(row, c) : gt_place_mn<T>(n, c * V, row)), in ? w + (long long)row * ld + c * V : w, in);
        }
    } else
#pragma unroll 1
    for (int i0 = member; i0 < pieces; i0 += AT_ONCE * GT_SET * 32) {
        uint4 v[AT_ONCE][1];
        int row[AT_ONCE], c[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const int i = min(i0 + j * GT_SET * 32, pieces - 1);        // (the last piece again: the same value to the same place)
            row[j] = TRANS ? i >> 3 : (int)((i * magic) >> 16);
            c[j] = TRANS ? i & 7 : i - row[j] * across;
            gt_read<T, 1, FAST>(v[j], w + (long long)row[j] * ld + c[j] * V, TRANS ? (row[j] < n_left ? k_left - c[j] * V : 0) : (row[j] < k_left ? n_left - c[j] * V : 0));
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const int at = TRANS ? gt_place_k(row[j], c[j]) : gt_place_mn<T>(n, c[j] * V, row[j]);
            if constexpr (GtType<T>::SPLIT) {
                float4 hi, lo;
                float4 x = *reinterpret_cast<const float4*>(v[j]);
                x = make_float4(x.x * scale, x.y * scale, x.z * scale, x.w * scale);        // (FP32 weights carry the scale; 16-bit ones would be rounded again)
                gt_split(x, hi, lo);
                *reinterpret_cast<float4*>(dst + at) = hi;
                *reinterpret_cast<float4*>(dst + (TRANS ? at + n * 128 : gt_place_mn<T>(n, n + c[j] * V, row[j]))) = lo;
            } else {
                *reinterpret_cast<uint4*>(dst + at) = v[j][0];
            }
        }
    }
}

template <class T, bool TRANS, bool FAST, int D>
__device__ __forceinline__ void gt_produce(const GtProblem& gt, const GtArgs& p, const GtTarget& tile_of, const GpTarget& to, int n0, unsigned char* a_base,
                                           unsigned char* b_base, const GtBars& bars, GtWalk walk, int tid) {
    constexpr int V = GtType<T>::V, KC = GtType<T>::KC, KSTEP = GtType<T>::KSTEP, TILE_ROWS = gt_tile_rows(D), THREADS = GT_SET * 32;
    constexpr int PIECES = (TILE_ROWS * 8 + THREADS - 1) / THREADS;             // of V channels by D components, of a lane
    const int set = tid / THREADS, member = tid % THREADS, lane = tid & 31, c = lane & 7, r0 = member >> 3, n = tile_of.n;
    const bool resident = tile_of.chunks <= tile_of.slots, in_turn = tile_of.stages < GT_SETS;
    int it = 0, stage = 0, use = 0, slot = 0, have = -1;        // chunks so far; the group whose weights are in shared memory
    int turn = 0;                               // set that has the next chunk
    // One component of a 16-bit type goes to its stage as it is: copies without registers, two chunks of a set on the way at once.
    constexpr bool ASYNC = FAST && !GtType<T>::SPLIT && D == 1;
    int held = -1;                              // the stage of the chunk before, whose copies are on their way
    auto arrive = [&](int at) {
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars.full + at);
    };
    auto hand_over = [&]() {
        if (held < 0) return;
        gt_copies_wait<0>();
        arrive(held);
        held = -1;
    };
    for (; walk.more(); walk.next(p.offsets, p.groups)) {
        walk.tile(TILE_ROWS);
        const T* w_group = static_cast<const T*>(p.W) + (long long)walk.g * gt.gp.w_numel;
        const bool load_b = !resident || have != walk.g;
        have = walk.g;
        if (resident) slot = 0;
        int row[PIECES];                        // (past the tile's rows: the last one again)
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int at = walk.pos + min(r0 + i * (THREADS / 8), walk.rows - 1);
            row[i] = p.order ? (int)__ldg(p.order + at) : at;
        }
        for (int path_no = to.path_begin; path_no < to.path_end; ++path_no) {
            const GpPath& path = gt.gp.path[path_no];
            for (int u0 = 0; u0 < path.src_mul; u0 += KC) {
                if (turn == set) {
                    const int left = path.src_mul - u0, k_fill = left >= KC ? KC : (left + KSTEP - 1) / KSTEP * KSTEP;
                    const T* x = static_cast<const T*>(p.X) + path.src_off + (u0 + V * c) * D;
                    uint4 v[PIECES][D];
                    if constexpr (!ASYNC) {
#pragma unroll
                        for (int i = 0; i < PIECES; ++i) gt_read<T, D, FAST>(v[i], x + (long long)row[i] * gt.gp.src_dim, left - V * c);
                    }
                    bool ok = true;
                    const int last = load_b ? it - (resident ? tile_of.chunks : tile_of.slots) : -1;     // the chunk that used the slot before
                    const bool wait_b = last >= 0 && last > it - tile_of.stages;
                    if constexpr (ASYNC) {
                        // a set that has to wait hands over first what it holds: the MMAs that it waits for may need it
                        bool now = use == 0 || mbar_test(bars.empty + stage, (unsigned)(use - 1) & 1);
                        if (!__all_sync(0xffffffffu, now && !wait_b && !in_turn)) hand_over();
                    }
                    if (in_turn && it > 0) ok = warp_wait(ok, bars.turn + set, (unsigned)(it / GT_SETS - (set == 0)) & 1, &gt_status, ERR_GT_TURN);
                    if (use > 0) ok = warp_wait(ok, bars.empty + stage, (unsigned)(use - 1) & 1, &gt_status, ERR_GT_EMPTY);
                    if (wait_b) ok = warp_wait(ok, bars.empty + last % tile_of.stages, (unsigned)(last / tile_of.stages) & 1, &gt_status, ERR_GT_EMPTY);
                    if (!ok) {
                        if constexpr (!GtType<T>::SPLIT) gt_copies_wait<0>();
                        return;
                    }
                    if (in_turn && lane == 0) mbar_arrive(bars.turn + (set + 1) % GT_SETS);
                    unsigned char* a = a_base + stage * GtType<T>::A_BYTES;
                    const T* w = w_group + path.w_off + (TRANS ? (long long)n0 * path.w_ld + u0 : (long long)u0 * path.w_ld + n0);
                    unsigned char* b = b_base + slot * GtType<T>::b_bytes(n);
                    if constexpr (ASYNC) {
                        if (load_b) gt_fill_b<T, TRANS, FAST>(b, w, path.w_ld, n, to.mul - n0, left, k_fill, (float)to.scale, member);
#pragma unroll
                        for (int i = 0; i < PIECES; ++i) {
                            const bool in = left > V * c;
                            gt_copy(a + gt_place_k(r0 + i * (THREADS / 8), c), in ? x + (long long)row[i] * gt.gp.src_dim : static_cast<const T*>(p.X), in);
                        }
                        gt_copies_commit();
                        if (held >= 0) {
                            gt_copies_wait<1>();
                            arrive(held);
                        }
                        held = stage;
                    } else {
#pragma unroll
                        for (int i = 0; i < PIECES; ++i) {
                            const int r = r0 + i * (THREADS / 8);
                            if (r < walk.rows) {
#pragma unroll
                                for (int k = 0; k < D; ++k) {
                                    const uint4 piece = gt_component<T, D>(v[i], k);
                                    unsigned char* at = a + gt_place_k(r * D + k, c);
                                    if constexpr (GtType<T>::SPLIT) {
                                        float4 hi, lo;
                                        gt_split(*reinterpret_cast<const float4*>(&piece), hi, lo);
                                        *reinterpret_cast<float4*>(at) = hi;
                                        *reinterpret_cast<float4*>(at + 16384) = lo;
                                    } else {
                                        *reinterpret_cast<uint4*>(at) = piece;
                                    }
                                }
                            }
                        }
                        if (load_b) {
                            gt_fill_b<T, TRANS, FAST>(b, w, path.w_ld, n, to.mul - n0, left, k_fill, (float)to.scale, member);
                            if constexpr (!GtType<T>::SPLIT) {
                                gt_copies_commit();
                                gt_copies_wait<0>();
                            }
                        }
                        arrive(stage);
                    }
                }
                if (++turn == GT_SETS) turn = 0;
                ++it;
                if (++stage == tile_of.stages) {
                    stage = 0;
                    ++use;
                }
                if (++slot == tile_of.slots) slot = 0;
            }
        }
    }
    if constexpr (ASYNC) hand_over();
}

// ---------------------------------------------------------------------------- MMA
// After a wait that ran out: MMAs that are on their way read shared memory and write tensor memory, which the CTA gives back when it ends.
__device__ __forceinline__ void gt_settle(unsigned leader, unsigned long long* done) {
    tc_commit_if(leader, done);
    warp_wait(true, done, 0, &gt_status, ERR_GT_DONE);
}
template <class T, bool TRANS, bool LONG, class Wait>
__device__ __forceinline__ void gt_multiply(const GtProblem& gt, const GtArgs& p, const GtTarget& tile_of, const GpTarget& to, unsigned char* a_base,
                                            unsigned char* b_base, const GtBars& bars, GtWalk walk, int tile_rows, unsigned tmem, unsigned leader, Wait&& acc_wait) {
    constexpr int KC = GtType<T>::KC, KSTEP = GtType<T>::KSTEP;
    constexpr bool B_MN = !TRANS;
    const int n = tile_of.n, acc = GtType<T>::acc(n), step_b = gt_step_b<T, B_MN>(n) >> 4;
    const bool resident = tile_of.chunks <= tile_of.slots;
    const unsigned wide = gt_idesc<T, B_MN>(acc), narrow = gt_idesc<T, B_MN>(n);
    const unsigned long long a0 = tc_smem_desc(smem_u32(a_base)), b0 = gt_desc_b<T, B_MN>(smem_u32(b_base), n);
    int stage = 0, use = 0, slot = 0, tiles = 0, accs = 0;
    for (; walk.more(); walk.next(p.offsets, p.groups), ++tiles) {
        walk.tile(tile_rows);
        bool ok = true;
        if (accs >= 2) ok = acc_wait(accs & 1, (unsigned)(accs / 2 - 1) & 1);
        unsigned accumulate = 0;
        int in_chain = 0;
        if (resident) slot = 0;
        for (int path_no = to.path_begin; path_no < to.path_end && ok; ++path_no) {
            const int mul = gt.gp.path[path_no].src_mul;
            for (int u0 = 0; u0 < mul && ok; u0 += KC) {
                if (LONG && in_chain++ == GT_CHAIN) {       // the next accumulator
                    tc_commit_if(leader, bars.acc_full + (accs & 1));
                    ++accs;
                    if (accs >= 2 && !acc_wait(accs & 1, (unsigned)(accs / 2 - 1) & 1)) {
                        ok = false;
                        break;
                    }
                    accumulate = 0;
                    in_chain = 1;
                }
                const unsigned d = tmem + (unsigned)((accs & 1) * 256);
                ok = warp_wait(ok, bars.full + stage, (unsigned)use & 1, &gt_status, ERR_GT_FULL);
                if (!ok) break;
                tc_fence_after();
                const int steps = (min(KC, mul - u0) + KSTEP - 1) / KSTEP;
                unsigned long long a = a0 + (unsigned long long)(stage * (GtType<T>::A_BYTES >> 4));
                unsigned long long b = b0 + (unsigned long long)(slot * (GtType<T>::b_bytes(n) >> 4));
                for (int s = 0; s < steps; ++s, a += 2, b += step_b) {
                    gt_mma<T>(leader, d, a, b, wide, accumulate);
                    if constexpr (GtType<T>::SPLIT) gt_mma<T>(leader, d + (unsigned)n, a + (16384 >> 4), b, narrow, 1);
                    accumulate = 1;
                }
                tc_commit_if(leader, bars.empty + stage);
                if (++stage == tile_of.stages) {
                    stage = 0;
                    ++use;
                }
                if (++slot == tile_of.slots) slot = 0;
            }
        }
        if (!ok) return gt_settle(leader, bars.done);
        tc_commit_if(leader, bars.acc_full + (accs & 1));
        ++accs;
        if (leader) *bars.progress = tiles + 1;
    }
}

// ---------------------------------------------------------------------------- rows of results
template <class T> struct GtPair { static __device__ unsigned of(float, float) { return 0; } };
template <> struct GtPair<__nv_bfloat16> {
    static __device__ unsigned of(float a, float b) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const unsigned*>(&v);
    }
};
template <> struct GtPair<__half> {
    static __device__ unsigned of(float a, float b) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const unsigned*>(&v);
    }
};

// The staged values of a tile's rows, [row][channel][component] of 32 channels: rows of 128 bytes whose 16-byte pieces are swizzled (one
// component: a lane writes whole pieces), else rows with 16 bytes of padding (a lane writes single values; two lanes meet in a bank).
template <int D> __host__ __device__ constexpr int gt_pitch() { return D == 1 ? 32 : 32 * D + 4; }
template <int D> __device__ __forceinline__ int gt_staged(int r, int i) { return D == 1 ? r * 32 + ((i ^ (4 * (r & 7)))) : r * gt_pitch<D>() + i; }

// Rows of a tile, added to what stands there: each value by the thread that wrote it (gt_write; the same group of warps), so that no other
// thread has to see it and the additions have one order.
template <int D, bool VEC>
__device__ __forceinline__ void gt_add(const float* staging, const int* rows_of, int rows, float* z_col, int dim, int values, int thread) {
    constexpr int V = VEC ? 4 : 1, ROW = 32 * D / V;
#pragma unroll 2
    for (int i = thread; i < rows * ROW; i += 128) {
        const int r = i / ROW, c = (i - r * ROW) * V;
        if (c >= values) continue;
        float* z = z_col + (long long)rows_of[r] * dim + c;
        if constexpr (VEC) {
            const float4 v = *reinterpret_cast<const float4*>(staging + gt_staged<D>(r, c));
            float4 s = *reinterpret_cast<const float4*>(z);
            s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
            *reinterpret_cast<float4*>(z) = s;
        } else {
            *z += staging[gt_staged<D>(r, c)];
        }
    }
}

// Rows of a tile from shared memory by the 128 threads of a group.  VEC: 16 bytes a thread; U of them are on the way together, past the
// last one the last one again (the same values to the same place).
template <class T, int D, bool VEC>
__device__ __forceinline__ void gt_write(const float* staging, const int* rows_of, int rows, T* __restrict__ z_col, int dim, int values, int thread) {
    if constexpr (VEC) {
        constexpr int V = 16 / sizeof(T), ROW = 32 * D / V, U = sizeof(T) == 4 ? 4 : 2;          // pieces of a row
        const int pieces = rows * ROW;
#pragma unroll 1
        for (int i0 = thread; i0 < pieces; i0 += U * 128) {
            float4 v[U][V / 4];
            T* z[U];
            bool in[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int i = min(i0 + 128 * j, pieces - 1), r = i / ROW, c = (i - r * ROW) * V;
#pragma unroll
                for (int h = 0; h < V / 4; ++h) v[j][h] = *reinterpret_cast<const float4*>(staging + gt_staged<D>(r, c + 4 * h));
                z[j] = z_col + (long long)rows_of[r] * dim + c;
                in[j] = c < values;
            }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                if (!in[j]) continue;
                if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(z[j]) = v[j][0];
                else *reinterpret_cast<uint4*>(z[j]) = make_uint4(GtPair<T>::of(v[j][0].x, v[j][0].y), GtPair<T>::of(v[j][0].z, v[j][0].w),
                                                                  GtPair<T>::of(v[j][1].x, v[j][1].y), GtPair<T>::of(v[j][1].z, v[j][1].w));
            }
        }
    } else {
        constexpr int ROW = 32 * D;
        for (int i = thread; i < rows * ROW; i += 128) {
            const int r = i / ROW, c = i - r * ROW;
            if (c < values) gp_store(z_col + (long long)rows_of[r] * dim + c, staging[gt_staged<D>(r, c)]);
        }
    }
}

// ---------------------------------------------------------------------------- prefetch
__device__ __forceinline__ void gt_prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
// `len` values of sorted rows [pos, pos + rows), from `base` on in each: 1 << lp lanes a row, four rows' numbers on the way together.
template <class T>
__device__ __forceinline__ void gt_prefetch_rows(const T* base, int dim, int len, const long long* __restrict__ order, int pos, int rows, int tid) {
    constexpr int LINE = 128 / sizeof(T), U = 4;
    int lp = 0;
    while (lp < 3 && (LINE << lp) < len) ++lp;
    const int step = GT_AHEAD * 32 >> lp, i0 = (tid & ((1 << lp) - 1)) * LINE;
    for (int r0 = tid >> lp; r0 < rows; r0 += U * step) {
        int row[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int at = pos + min(r0 + j * step, rows - 1);
            row[j] = order ? (int)__ldg(order + at) : at;
        }
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (r0 + j * step < rows)
                for (int i = i0; i < len; i += LINE << lp) gt_prefetch(base + (long long)row[j] * dim + i);
    }
}
// Waits until `progress` is at least `least`, after a while no longer.  Whether work `item` is still ahead: what is late is left out.
// (Nothing depends on what a prefetch does.)
__device__ __forceinline__ bool gt_follow(volatile int* progress, int item, int distance) {
    int now = 0;
    for (int i = 0; i < 1 << 14; ++i) {
        now = __shfl_sync(0xffffffffu, *progress, 0);
        if (now >= item - distance) break;
        __nanosleep(100);
    }
    return now < item;
}
template <class T, bool TRANS>
__device__ __forceinline__ void gt_ahead(const GtProblem& gt, const GtArgs& p, const GtTarget& tile_of, const GpTarget& to, int n0, const GtBars& bars, GtWalk walk,
                                         int tile_rows, int tid) {
    constexpr int LINE = 128 / sizeof(T), THREADS = GT_AHEAD * 32;
    int have = -1, tiles = 0;
    for (; walk.more(); walk.next(p.offsets, p.groups), ++tiles) {
        walk.tile(tile_rows);
        if (!gt_follow(bars.progress, tiles, 2)) continue;
        for (int path_no = to.path_begin; path_no < to.path_end; ++path_no) {
            const GpPath& path = gt.gp.path[path_no];
            if (walk.g != have) {               // weights
                const int n = min(tile_of.n, to.mul - n0), rows = TRANS ? n : path.src_mul, len = TRANS ? path.src_mul : n;
                const T* w = static_cast<const T*>(p.W) + (long long)walk.g * gt.gp.w_numel + path.w_off + (TRANS ? (long long)n0 * path.w_ld : n0);
                for (int r = tid >> 2; r < rows; r += THREADS / 4)
                    for (int i = (tid & 3) * LINE; i < len; i += 4 * LINE) gt_prefetch(w + (long long)r * path.w_ld + i);
            }
            if (n0 == 0)                        // (the CTAs of an output block's other channels read the same rows)
                gt_prefetch_rows<T>(static_cast<const T*>(p.X) + path.src_off, gt.gp.src_dim, path.src_mul * to.d, p.order, walk.pos, walk.rows, tid);
        }
        have = walk.g;
    }
}

// ---------------------------------------------------------------------------- drain
// The chunks of 32 channels of all tiles go to the two groups of four warps in turn.  FP32: a tile whose sum has several chains comes as
// as many accumulators; the results of the first are written and the others added to them, a chunk of channels by the same group each time.
// acc_wait(buffer, parity): the warp's wait for an accumulator.  A warp whose wait ran out reads and writes nothing more but comes to every
// barrier of its group: each warp counts its own polls, so the other three may have seen the accumulator complete, and a hardware barrier
// waits without limit.  (It keeps the rows' numbers up to date: the others write the rows that stand there.)
template <class T, bool TRANS, bool LONG, int D, class Wait>
__device__ __forceinline__ void gt_drain(const GtProblem& gt, const GtArgs& p, const GtTarget& tile_of, const GpTarget& to, int n0, float* staging,
                                         const GtBars& bars, GtWalk walk, unsigned tmem, int group, int warp, int lane, Wait&& acc_wait) {
    constexpr int TILE_ROWS = gt_tile_rows(D), PITCH = gt_pitch<D>();
    const int n = tile_of.n, mul = min(n, to.mul - n0), pair = warp * 32 + lane, r_of = pair / D, k_of = pair % D;
    const float scale = (float)to.scale;
    const unsigned quarter = tmem + ((unsigned)(warp * 32) << 16);
    int* rows_of = bars.rows + 128 * group;
    staging += group * (GT_STAGING / 4);
    const int chains = LONG ? (tile_of.chunks + GT_CHAIN - 1) / GT_CHAIN : 1;
    int accs = 0, first_turn = 0;
    bool alive = true;
    for (; walk.more(); walk.next(p.offsets, p.groups)) {
        walk.tile(TILE_ROWS);
        if (pair < walk.rows) rows_of[pair] = (int)gp_row(p.order, walk.pos + pair);         // (read behind the first barrier below)
        int turn = first_turn;
        for (int chain = 0; chain < chains; ++chain, ++accs) {
            const int buf = accs & 1;
            alive = alive && acc_wait(buf, (unsigned)(accs / 2) & 1);
            tc_fence_after();
            bool mine = false;
            turn = first_turn;
            for (int w0 = 0; w0 < mul; w0 += 32, turn ^= 1) {
                if (turn != group) continue;
                mine = true;
                const bool last = w0 + 32 * GT_EPI_GROUPS >= mul;       // the group has read its part of the accumulator then
                float* to_smem = staging + r_of * PITCH + k_of;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    unsigned v[16], u[GtType<T>::SPLIT ? 16 : 1];
                    const unsigned at = quarter + (unsigned)(buf * 256 + w0 + 16 * h);
                    if (alive && w0 + 16 * h < n) {
                        tc_load16(at, v);
                        if constexpr (GtType<T>::SPLIT) tc_load16(at + n, u);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    }
                    if (alive && last && h == 1) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bars.acc_empty + buf);
                    }
                    if (alive && w0 + 16 * h < n && r_of < walk.rows) {
                        float s[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            if constexpr (GtType<T>::SPLIT) s[j] = __uint_as_float(v[j]) + __uint_as_float(u[j]);
                            else s[j] = __uint_as_float(v[j]) * scale;
                        }
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            if constexpr (D == 1) *reinterpret_cast<float4*>(staging + gt_staged<1>(r_of, 16 * h + j)) = make_float4(s[j], s[j + 1], s[j + 2], s[j + 3]);
                            else {
#pragma unroll
                                for (int i = j; i < j + 4; ++i) to_smem[(16 * h + i) * D] = s[i];
                            }
                        }
                    }
                }
                group_sync(1 + group, 128);
                const int values = min(32, mul - w0) * D;
                T* z = static_cast<T*>(p.Z) + to.off + (n0 + w0) * D;
                const bool vec = p.z_vec && (to.off | values) % (16 / (int)sizeof(T)) == 0;
                if (alive && chain == 0) {
                    if (vec) gt_write<T, D, true>(staging, rows_of, walk.rows, z, gt.gp.dst_dim, values, pair);
                    else gt_write<T, D, false>(staging, rows_of, walk.rows, z, gt.gp.dst_dim, values, pair);
                } else if (alive) {
                    if constexpr (LONG) {
                        if (vec) gt_add<D, true>(staging, rows_of, walk.rows, z, gt.gp.dst_dim, values, pair);
                        else gt_add<D, false>(staging, rows_of, walk.rows, z, gt.gp.dst_dim, values, pair);
                    }
                }
                group_sync(1 + group, 128);
            }
            if (!mine) {
                __syncwarp();
                if (alive && lane == 0) mbar_arrive(bars.acc_empty + buf);
                group_sync(1 + group, 128);     // (rows_of is written again by all four warps)
            }
        }
        first_turn = turn;
    }
}

// What a role does for blocks of D components.
template <class T, bool TRANS, bool FAST, bool LONG, int D>
__device__ __forceinline__ void gt_roles(const GtProblem& gt, const GtArgs& p, const GtTarget& tile_of, const GpTarget& to, int n0, unsigned char* a_base,
                                         unsigned char* b_base, float* staging, const GtBars& bars, const GtWalk& walk, unsigned tmem, int warp, int tid) {
    if (warp < GT_PW) gt_produce<T, TRANS, FAST, D>(gt, p, tile_of, to, n0, a_base, b_base, bars, walk, tid);
    else gt_drain<T, TRANS, LONG, D>(gt, p, tile_of, to, n0, staging, bars, walk, tmem, (warp - GT_PW) >> 2, warp & 3, tid & 31, [&](int buf, unsigned parity) {
        return warp_wait(true, bars.acc_full + buf, parity, &gt_status, ERR_GT_ACC_FULL);
    });
}

// Self-test: the MMAs of three tiles of one row, of zeros.  The third finds no accumulator free; the MMAs of the first two are over when the
// warp comes back.
constexpr int GT_PROBE_STAGES = 2, GT_PROBE_SMEM = GT_PROBE_STAGES * GtType<float>::A_BYTES + GtType<float>::b_bytes(16) + GT_CONTROL;
__device__ const long long gt_probe_offsets[] = {0, 1, 2, 3};
__global__ void __launch_bounds__(32) oeq_grouped_issue_probe(const __grid_constant__ GtProblem gt) {
    extern __shared__ __align__(1024) unsigned char gt_smem[];
    const int lane = threadIdx.x;
    unsigned char *b = gt_smem + GT_PROBE_STAGES * GtType<float>::A_BYTES, *control = b + GtType<float>::b_bytes(16);
    const GtBars bars(control);
    for (int i = lane; i < (GT_PROBE_SMEM - GT_CONTROL) / 16; i += 32) reinterpret_cast<uint4*>(gt_smem)[i] = make_uint4(0, 0, 0, 0);
    fence_async_smem();
    if (lane == 0) {
        for (int i = 0; i < GT_PROBE_STAGES; ++i) {
            mbar_init(bars.full + i, 1);
            mbar_init(bars.empty + i, 1);
            mbar_init(bars.acc_full + i, 1);
        }
        mbar_init(bars.done, 1);
        fence_mbar_init();
        for (int i = 0; i < GT_PROBE_STAGES; ++i) mbar_arrive(bars.full + i);
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(bars.tmem)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
    __syncwarp();
    tc_fence_after();
    const unsigned tmem = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile unsigned*>(bars.tmem), 0);
    const GtArgs p{nullptr, nullptr, nullptr, gt_probe_offsets, nullptr, 3, 3, 0};
    gt_multiply<float, false, false>(gt, p, gt.target[0], gt.gp.target[0], gt_smem, b, bars, GtWalk(gt_probe_offsets, 0, 0, 3), 128, tmem, elect_lane(), [&](int, unsigned) { return false; });
    const bool over = mbar_test(bars.done, 0);
    if (lane == 0) atomicCAS(&gt_status, 0, over ? ERR_GT_ACC_EMPTY : ERR_GT_DONE);
    tc_fence_before();
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
}

// Self-test: the drain of three tiles of one row, whose accumulators hold anything.  Warp `lost` has its waits run out, the others have
// theirs complete; all come back.
constexpr int GT_PROBE_ROWS = 3, GT_PROBE_COLUMNS = 80;
__device__ float gt_probe_z[GT_PROBE_ROWS * GT_PROBE_COLUMNS];
__global__ void __launch_bounds__(32 * GT_EPI) oeq_grouped_drain_probe(const __grid_constant__ GtProblem gt, int lost) {
    __shared__ __align__(1024) unsigned char smem[GT_EPI_GROUPS * GT_STAGING + GT_CONTROL];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const GtBars bars(smem + GT_EPI_GROUPS * GT_STAGING);
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) mbar_init(bars.acc_empty + i, GT_EPI);
        fence_mbar_init();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(bars.tmem)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile unsigned*>(bars.tmem), 0);
    const GtArgs p{nullptr, nullptr, nullptr, gt_probe_offsets, gt_probe_z, GT_PROBE_ROWS, GT_PROBE_ROWS, 0};
    gt_drain<float, false, false, 1>(gt, p, gt.target[0], gt.gp.target[0], 0, reinterpret_cast<float*>(smem), bars, GtWalk(gt_probe_offsets, 0, 0, GT_PROBE_ROWS), tmem, warp >> 2,
                              warp & 3, lane, [&](int, unsigned) {
                                  if (warp == lost && lane == 0) atomicCAS(&gt_status, 0, ERR_GT_ACC_FULL);
                                  return warp != lost;
                              });
    tc_fence_before();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
}

// FAST: every block of rows and weights, of all paths, is made of whole, aligned 16-byte pieces; else values are read one by one (16-bit types
// with spills then: 68 bytes for the product, 12 for dX).  LONG (FP32): some sum has more than one chain.
template <class T, bool TRANS, bool FAST, bool LONG>
__global__ void __launch_bounds__(GT_THREADS, 1) oeq_grouped_tc(const __grid_constant__ GtProblem gt, const GtArgs p) {
    extern __shared__ __align__(1024) unsigned char gt_smem[];
    unsigned char* smem = gt_smem;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    int t = 0;
    while (t + 1 < gt.gp.n_targets && (int)blockIdx.x >= gt.target[t + 1].first) ++t;
    const GpTarget& to = gt.gp.target[t];
    const GtTarget& tile_of = gt.target[t];
    const int local = (int)blockIdx.x - tile_of.first, part = local / tile_of.n_tiles, n0 = local % tile_of.n_tiles * tile_of.n, d = to.d;
    unsigned char *a_base = smem, *b_base = a_base + tile_of.stages * GtType<T>::A_BYTES;
    float* staging = reinterpret_cast<float*>(b_base + tile_of.slots * GtType<T>::b_bytes(tile_of.n));
    unsigned char* control = reinterpret_cast<unsigned char*>(staging) + GT_EPI_GROUPS * GT_STAGING;
    const GtBars bars(control);
    if (tid == 0) {
        for (int i = 0; i < GT_STAGES; ++i) {
            mbar_init(bars.full + i, GT_SET);
            mbar_init(bars.empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bars.acc_full + i, 1);
            mbar_init(bars.acc_empty + i, GT_EPI);
        }
        for (int i = 0; i < GT_SETS; ++i) mbar_init(bars.turn + i, GT_SET);
        mbar_init(bars.done, 1);
        *bars.progress = 0;
        fence_mbar_init();
    }
    constexpr int MMA_WARP = GT_PW + GT_EPI;
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(bars.tmem)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const bool work = to.path_begin < to.path_end;              // (a block without a path is zero in every row)
    GtRange& range = *reinterpret_cast<GtRange*>(control + 256);
    tc_fence_before();
    gt_range(range, p.offsets, p.groups, p.rows, part, tile_of.parts, tile_of.extra);       // (two barriers)
    tc_fence_after();
    const unsigned tmem = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile unsigned*>(bars.tmem), 0);
    const GtWalk walk(p.offsets, range.g, work ? (int)range.lo : 0, work ? (int)range.hi : 0);
    if (warp > MMA_WARP) gt_ahead<T, TRANS>(gt, p, tile_of, to, n0, bars, walk, gt_tile_rows(d), tid - (MMA_WARP + 1) * 32);
    else if (warp == MMA_WARP) gt_multiply<T, TRANS, LONG>(gt, p, tile_of, to, a_base, b_base, bars, walk, gt_tile_rows(d), tmem, elect_lane(), [&](int buf, unsigned parity) {
        return warp_wait(true, bars.acc_empty + buf, parity, &gt_status, ERR_GT_ACC_EMPTY);
    });
    else if (d == 1) gt_roles<T, TRANS, FAST, LONG, 1>(gt, p, tile_of, to, n0, a_base, b_base, staging, bars, walk, tmem, warp, tid);
    else if (d == 3) gt_roles<T, TRANS, FAST, LONG, 3>(gt, p, tile_of, to, n0, a_base, b_base, staging, bars, walk, tmem, warp, tid);
    else if (d == 5) gt_roles<T, TRANS, FAST, LONG, 5>(gt, p, tile_of, to, n0, a_base, b_base, staging, bars, walk, tmem, warp, tid);
    else gt_roles<T, TRANS, FAST, LONG, 7>(gt, p, tile_of, to, n0, a_base, b_base, staging, bars, walk, tmem, warp, tid);
    // zeros: the rows without a group, every row where the block has no path
    {
        const long long from = work ? min(__ldg(p.offsets + p.groups), p.rows) : 0, count = p.rows - from;
        const long long lo = from + gp_cut(count, part, tile_of.parts), hi = from + gp_cut(count, part + 1, tile_of.parts);
        const int values = min(tile_of.n, to.mul - n0) * d;
        for (long long at = lo + warp; at < hi; at += GT_THREADS / 32) {
            T* z = static_cast<T*>(p.Z) + gp_row(p.order, at) * gt.gp.dst_dim + to.off + n0 * d;
            for (int i = lane; i < values; i += 32) gp_store(z + i, 0.f);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
}

}  // namespace oeq
