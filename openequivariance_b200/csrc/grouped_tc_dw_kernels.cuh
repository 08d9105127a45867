// Weight gradient of the linear maps with one set of weights for each group of rows, on the 5th-generation tensor cores: FP32 (3xTF32),
// BF16 and FP16, up to GT_D_MAX components.  FP32 sums.
//
//   dW_g[i,o][u,w] = c_o sum_{r in g, k} X[r,i,u,k] dZ[r,o,w,k]
//
// M = 128 input channels u, N = up to 128 output channels w of one path, and the sum runs over rows and components.  Both operands have their
// channels along memory, so both are "MN-major": a lane reads the 16 d bytes of V channels of a row and writes d pieces, one into
// the slot of each component.  A slot has one component of GdType::ROWS sorted rows of one group, X and dZ, 16 KB; four of them are
// a bundle, and there are two bundles (16-bit types of one component: four of two, which are filled by copies without registers, two of a
// set on the way at once).
//   * 16 producer warps.  One and three components: two sets of eight take units of rows in turn, each with a bundle of its own, a lane the same
//     channels of X and dZ.  Five and seven: one set, half of it for X and half for dZ, the components of a unit in two bundles;
//   * one warp, in step, issues the MMAs of a bundle, as many as there are between two waits (a wait for each slot: 575 cycles a slot, where its
//     MMAs take 192): FP32 hi.hi and hi.lo as one, lo.hi into hi.lo's columns;
//   * 8 warps add the accumulators to sums in shared memory at the end of a group and after CHAIN slots: an MMA's additions are cut off, not
//     rounded, and the error grows with the length of a chain (relative, one chain of 750 slots: 1e-5).  The two accumulators alternate.
//   * 3 warps prefetch rows to L2, up to two units ahead of the MMAs.
// Measured from a cold L2 with the sum over ranges, 50 000 rows in 10 groups of 128x(0e+1o+2e+3o) FP32: 235 us (3.5 TB/s); 100 000 rows of 128x(0e+1o+2e)
// BF16 in 256 groups 133 us; 65 536 rows of 512x0e with 1024x0e BF16 248 us (32 tiles of 128 x 128 read 1.1 GB through L2).  Loads on their way bound it (long
// scoreboard), with the load and store unit at 56 % and the tensor pipe at 32 %.
// A CTA has one tile of one path and a range of the sorted rows (gt_range); groups that go beyond the range leave a partial tile for
// oeq_grouped_join.  Every wait is bounded.
#pragma once
#include "grouped_tc_kernels.cuh"

namespace oeq {

constexpr int GD_TILE = 128, GD_SLOT = 16384, GD_RING = 8, GD_BUNDLES = 4, GD_SUMS = GD_TILE * GD_TILE * 4;
constexpr int GD_PW = 16, GD_EPI = 8, GD_THREADS = (GD_PW + GD_EPI + 1 + GT_AHEAD) * 32;
constexpr int GD_SMEM = GD_RING * GD_SLOT + GD_SUMS + 1024;
constexpr int ERR_GD_EMPTY = 91, ERR_GD_FULL = 92, ERR_GD_ACC_FULL = 93, ERR_GD_ACC_EMPTY = 94;

template <class T> struct GdType { static constexpr int ROWS = 32, CHAIN = 32; };
template <> struct GdType<float> { static constexpr int ROWS = 8, CHAIN = 32; };
__host__ __device__ constexpr int gd_sets(int d) { return d <= 3 ? 2 : 1; }     // of producers
template <class T> __host__ __device__ constexpr int gd_bundles(int d) { return sizeof(T) == 2 && d == 1 ? 4 : 2; }
template <class T> __host__ __device__ constexpr int gd_bundle(int d) { return GD_RING / gd_bundles<T>(d); }       // slots
// rows of a unit: with one component a bundle of slots, else one slot of each component
template <class T> __host__ __device__ constexpr int gd_unit(int d) { return d == 1 ? gd_bundle<T>(d) * GdType<T>::ROWS : GdType<T>::ROWS; }
// components of a unit's first bundle
__host__ __device__ constexpr int gd_first(int d) { return d <= 4 ? d : (d + 1) / 2; }

struct GdProblem {
    GpProblem gp;               // paths in the order of their weights
    GpSplit split;
    int extra[GP_PATHS];        // time of a group, in rows
};
struct GdArgs {
    const void *X, *dZ;
    const long long *order, *offsets;
    void* dW;
    float* partial;             // [CTAs][2][128][128]
    GpStart* starts;            // [CTAs]
    long long rows;
    int groups;
    int w_vec;                  // weights of dW in 16-byte pieces
};

// byte offset of V channels from ch of row r (of the slot's) in an operand with `blocks` blocks of channels
template <class T>
__device__ __forceinline__ int gd_place(int ch, int r, int blocks) {
    if constexpr (GtType<T>::SPLIT) return (ch >> 5) * 1024 + r * 128 + (((ch & 31) * 4) ^ ((r & 3) << 5));
    else return (r >> 3) * (blocks * 1024) + (ch >> 6) * 1024 + (r & 7) * 128 + ((((ch >> 3) & 7) ^ (r & 7)) << 4);
}
template <class T>
__device__ __forceinline__ unsigned long long gd_desc(unsigned addr, int blocks) {
    const unsigned long long base = (unsigned long long)((addr >> 4) & 0x3fff) | (unsigned long long)(1024 >> 4) << 16 | 1ull << 46;
    if constexpr (GtType<T>::SPLIT) return base | (unsigned long long)(512 >> 4) << 32 | 1ull << 61;
    else return base | (unsigned long long)(blocks * 1024 >> 4) << 32 | 2ull << 61;
}

struct GdBars {
    unsigned long long *full, *empty, *acc_full, *acc_empty, *done;
    unsigned* tmem;
    volatile int* progress;     // units whose MMAs are on their way
    __device__ explicit GdBars(unsigned char* control) {
        full = reinterpret_cast<unsigned long long*>(control);
        empty = full + GD_BUNDLES;
        acc_full = empty + GD_BUNDLES;
        acc_empty = acc_full + 2;
        done = acc_empty + 2;
        tmem = reinterpret_cast<unsigned*>(done + 1);
        progress = reinterpret_cast<volatile int*>(tmem + 1);
    }
};

// A unit's place in the chain of sums.
template <class T> struct GdChain {
    int slots = 0;              // since the accumulator was begun
    bool begins = true;         // the unit begins an accumulator
    bool ends = false, piece_ends = false;              // the unit ends it; ends the group's rows in this range
    __device__ int unit(const GtWalk& walk, int d) {
        const int n = (walk.rows + GdType<T>::ROWS - 1) / GdType<T>::ROWS * d;
        begins = slots == 0;
        slots += n;
        piece_ends = walk.pos + walk.rows >= walk.end;
        ends = piece_ends || slots >= GdType<T>::CHAIN;
        if (ends) slots = 0;
        return n;
    }
};

// ---------------------------------------------------------------------------- producers
// The operands of a unit: 1 << lp lanes take a row, V channels each.
struct GdLane {
    int lp, r0, ch;             // lanes of a row; the lane's first row, its channel
    int x_left, z_left;         // channels of X and dZ from there on (0: another lane's)
};
// Components [K0, K1) of V channels, to the slots from `dst` on.
template <class T, int D, int K0, int K1>
__device__ __forceinline__ void gd_put(const uint4 (&v)[D], unsigned char* dst, int lo) {
#pragma unroll
    for (int k = K0; k < K1; ++k) {
        const uint4 a = gt_component<T, D>(v, k);
        if constexpr (GtType<T>::SPLIT) {
            float4 hi, lo4;
            gt_split(*reinterpret_cast<const float4*>(&a), hi, lo4);
            *reinterpret_cast<float4*>(dst + (k - K0) * GD_SLOT) = hi;
            *reinterpret_cast<float4*>(dst + (k - K0) * GD_SLOT + lo) = lo4;
        } else {
            *reinterpret_cast<uint4*>(dst + (k - K0) * GD_SLOT) = a;
        }
    }
}
// A unit of rows.  `bundle`: that of the first components; `parity` of the wait for it to be free again (no wait: the first use).
template <class T, int D, bool FAST>
__device__ __forceinline__ bool gd_fill(const GdArgs& p, const GpProblem& gp, const GtWalk& walk, const GdLane& l, const T* x, const T* z, int n, unsigned char* ring,
                                        const GdBars& bars, int bundle, int use) {
    constexpr bool BOTH = gd_sets(D) == 2;      // a lane reads both operands
    // Rows of a lane on the way together.  Two of 16 bits with components instead of one: 122 us instead of 126 for 300 000 rows of 128x1o and 132 instead of
    // 136 for 100 000 rows in 256 groups, but 152 instead of 134 for 200 000 of 128x2e, 130 instead of 122 for 120 000 of 128x3o, and 259 instead of 249 for 65 536 of 512x0e
    // with 1024x0e: all widths share the kernel's registers, 72 at most, which spilled.
    constexpr int PASS = D == 1 ? 4 : 1;
    constexpr int ROWS = GdType<T>::ROWS, THREADS = 256, FIRST = gd_first(D), BUNDLE = gd_bundle<T>(D);
    const int rows = (walk.rows + ROWS - 1) / ROWS * ROWS, step = THREADS >> l.lp, blocks = (n + 63) / 64, lane = threadIdx.x & 31;
    const bool is_x = l.x_left > 0;
    auto free_again = [&](int b) { return use == 0 || warp_wait(true, bars.empty + b, (unsigned)(use - 1) & 1, &gt_status, ERR_GD_EMPTY); };
    auto filled = [&](int b) {
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars.full + b);
    };
    bool waited = false;
#pragma unroll 1
    for (int q0 = 0; q0 < rows; q0 += PASS * step) {
        uint4 v[PASS][D], w[BOTH ? PASS : 1][D];
        int row[PASS];
#pragma unroll
        for (int j = 0; j < PASS; ++j) {
            const int at = walk.pos + min(l.r0 + q0 + j * step, walk.rows - 1);
            row[j] = p.order ? (int)__ldg(p.order + at) : at;
        }
#pragma unroll
        for (int j = 0; j < PASS; ++j) {
            const bool in = l.r0 + q0 + j * step < walk.rows;           // rows behind the group's last: zeros
            if constexpr (BOTH) {
                gt_read<T, D, FAST>(v[j], x + (long long)row[j] * gp.src_dim, in ? l.x_left : 0);
                gt_read<T, D, FAST>(w[j], z + (long long)row[j] * gp.dst_dim, in ? l.z_left : 0);
            } else {
                gt_read<T, D, FAST>(v[j], is_x ? x + (long long)row[j] * gp.src_dim : z + (long long)row[j] * gp.dst_dim, in ? (is_x ? l.x_left : l.z_left) : 0);
            }
        }
        if (!waited && !free_again(bundle)) return false;
        auto place = [&](int j, bool of_x, unsigned char*& dst, int& lo) {
            const int q = l.r0 + q0 + j * step, r = q % ROWS;
            const int at = of_x ? gd_place<T>(l.ch, r, GD_TILE / 64) : 8192 + gd_place<T>(l.ch, r, blocks);
            dst = ring + (bundle * BUNDLE + q / ROWS * (D == 1)) * GD_SLOT + at;
            lo = of_x ? 4096 : 8192 + gd_place<T>(l.ch + n, r, 0) - at;
            return q < rows && (of_x ? l.x_left : l.z_left) > 0;
        };
#pragma unroll
        for (int j = 0; j < PASS; ++j) {
            unsigned char* dst;
            int lo;
            if (BOTH || is_x) {
                if (place(j, true, dst, lo)) gd_put<T, D, 0, FIRST>(v[j], dst, lo);
            }
            if (BOTH || !is_x) {
                if (place(j, false, dst, lo)) gd_put<T, D, 0, FIRST>(BOTH ? w[j] : v[j], dst, lo);
            }
        }
        if constexpr (FIRST < D) {
            if (q0 + PASS * step >= rows) filled(bundle);
            if (!waited && !free_again(bundle ^ 1)) return false;
#pragma unroll
            for (int j = 0; j < PASS; ++j) {
                unsigned char* dst;
                int lo;
                if (place(j, is_x, dst, lo)) gd_put<T, D, FIRST, D>(v[j], dst + (1 - 2 * bundle) * (BUNDLE * GD_SLOT), lo);
            }
        }
        waited = true;
    }
    filled(FIRST < D ? bundle ^ 1 : bundle);
    return true;
}

// A unit of one component of a 16-bit type: copies.  Rows behind the group's last are zeros.
template <class T>
__device__ __forceinline__ void gd_copy(const GdArgs& p, const GpProblem& gp, const GtWalk& walk, const GdLane& l, const T* x, const T* z, int n, unsigned char* dst) {
    constexpr int ROWS = GdType<T>::ROWS, U = 4;
    const int rows = (walk.rows + ROWS - 1) / ROWS * ROWS, step = 256 >> l.lp, blocks = (n + 63) / 64;
#pragma unroll 1
    for (int q0 = l.r0; q0 < rows; q0 += U * step) {
        int row[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int at = walk.pos + min(q0 + j * step, walk.rows - 1);
            row[j] = p.order ? (int)__ldg(p.order + at) : at;
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int q = q0 + j * step;
            if (q >= rows) continue;
            unsigned char* slot = dst + q / ROWS * GD_SLOT;
            const bool in = q < walk.rows;
            if (l.x_left > 0) gt_copy(slot + gd_place<T>(l.ch, q % ROWS, GD_TILE / 64), x + (long long)row[j] * gp.src_dim, in);
            if (l.z_left > 0) gt_copy(slot + 8192 + gd_place<T>(l.ch, q % ROWS, blocks), z + (long long)row[j] * gp.dst_dim, in);
        }
    }
    gt_copies_commit();
}

template <class T, bool FAST, int D>
__device__ __forceinline__ void gd_produce(const GdArgs& p, const GpProblem& gp, const GpPath& path, const GpTarget& to, int u0, int w0, int mu, int mw, int n,
                                           unsigned char* ring, const GdBars& bars, GtWalk walk, int tid) {
    constexpr int V = GtType<T>::V, SETS = gd_sets(D), UNIT = gd_unit<T>(D);
    const int half = tid >> 8, member = tid & 255;
    GdLane l;
    l.lp = 0;
    while ((V << l.lp) < max(mu, mw)) ++l.lp;
    l.r0 = member >> l.lp;
    l.ch = (member & ((1 << l.lp) - 1)) * V;
    l.x_left = SETS == 2 || half == 0 ? mu - l.ch : 0;
    l.z_left = SETS == 2 || half == 1 ? mw - l.ch : 0;
    const T *x = static_cast<const T*>(p.X) + path.src_off + (u0 + l.ch) * D, *z = static_cast<const T*>(p.dZ) + to.off + (w0 + l.ch) * D;
    constexpr int BUNDLES = gd_bundles<T>(D);
    constexpr bool ASYNC = FAST && BUNDLES == 4;
    int held = -1;                              // the bundle whose copies are on their way
    auto hand_over = [&](bool all) {
        if (held < 0) return;
        if (all) gt_copies_wait<0>();
        else gt_copies_wait<1>();
        fence_async_smem();
        __syncwarp();
        if ((tid & 31) == 0) mbar_arrive(bars.full + held);
        held = -1;
    };
    int units = 0;
    for (; walk.more(); walk.next(p.offsets, p.groups), ++units) {
        walk.tile(UNIT);
        if (SETS == 2 && (units & 1) != half) continue;
        const int bundle = SETS == 1 ? 0 : units % BUNDLES, use = SETS == 1 ? units : units / BUNDLES;
        if constexpr (ASYNC) {
            // a set that has to wait hands over first what it holds: the MMAs that it waits for may need it
            if (use > 0 && !__all_sync(0xffffffffu, mbar_test(bars.empty + bundle, (unsigned)(use - 1) & 1))) {
                hand_over(true);
                if (!warp_wait(true, bars.empty + bundle, (unsigned)(use - 1) & 1, &gt_status, ERR_GD_EMPTY)) return;
            }
            gd_copy<T>(p, gp, walk, l, x, z, n, ring + bundle * gd_bundle<T>(D) * GD_SLOT);
            hand_over(false);
            held = bundle;
        } else {
            if (!gd_fill<T, D, FAST>(p, gp, walk, l, x, z, n, ring, bars, bundle, use)) return;
        }
    }
    if constexpr (ASYNC) hand_over(true);
}

// ---------------------------------------------------------------------------- MMA
template <class T>
__device__ __forceinline__ void gd_multiply(const GdArgs& p, int d, int unit, int n, unsigned char* ring, const GdBars& bars, GtWalk walk, unsigned tmem, unsigned leader) {
    constexpr unsigned MN = 1u << 15 | 1u << 16;
    const int blocks = (n + 63) / 64;
    const unsigned wide = gt_idesc<T, false>(GtType<T>::acc(n)) | MN, narrow = gt_idesc<T, false>(n) | MN;
    const unsigned long long a0 = gd_desc<T>(smem_u32(ring), GD_TILE / 64), b0 = gd_desc<T>(smem_u32(ring) + 8192, blocks);
    const int first = gd_first(d), bundles = first < d ? 2 : 1, sets = gd_sets(d), turns = gd_bundles<T>(d), bundle_bytes = gd_bundle<T>(d) * GD_SLOT;
    GdChain<T> chain;
    int units = 0, accs = 0;
    unsigned accumulate = 0;
    bool ok = true;
    for (; walk.more() && ok; walk.next(p.offsets, p.groups), ++units) {
        walk.tile(unit);
        const int slots = chain.unit(walk, d), buf = accs & 1;
        if (chain.begins) {
            if (accs >= 2) ok = warp_wait(ok, bars.acc_empty + buf, (unsigned)(accs / 2 - 1) & 1, &gt_status, ERR_GD_ACC_EMPTY);
            accumulate = 0;
        }
        const unsigned acc = tmem + (unsigned)(buf * 256);
        for (int i = 0; i < bundles && ok; ++i) {
            const int bundle = sets == 2 ? units % turns : i, n_slots = bundles == 1 ? slots : (i == 0 ? first : d - first);
            ok = warp_wait(ok, bars.full + bundle, (unsigned)(sets == 2 ? units / turns : units) & 1, &gt_status, ERR_GD_FULL);
            if (!ok) break;
            tc_fence_after();
            unsigned long long a = a0 + (unsigned long long)(bundle * (bundle_bytes >> 4)), b = b0 + (unsigned long long)(bundle * (bundle_bytes >> 4));
#pragma unroll
            for (int s = 0; s < 4; ++s, a += GD_SLOT >> 4, b += GD_SLOT >> 4) {
                if (s >= n_slots) break;
                if constexpr (GtType<T>::SPLIT) {
                    gt_mma<T>(leader, acc, a, b, wide, accumulate);
                    gt_mma<T>(leader, acc + (unsigned)n, a + (4096 >> 4), b, narrow, 1);
                    accumulate = 1;
                } else {
#pragma unroll
                    for (int h = 0; h < GdType<T>::ROWS / 16; ++h) {
                        gt_mma<T>(leader, acc, a + (unsigned long long)(h * (2 * (GD_TILE / 64) * 1024 >> 4)), b + (unsigned long long)(h * (2 * blocks * 1024 >> 4)), wide, accumulate);
                        accumulate = 1;
                    }
                }
            }
            tc_commit_if(leader, bars.empty + bundle);
        }
        if (leader) *bars.progress = units + 1;
        if (ok && chain.ends) {
            tc_commit_if(leader, bars.acc_full + buf);
            ++accs;
        }
    }
    if (!ok) gt_settle(leader, bars.done);
}

// ---------------------------------------------------------------------------- prefetch
template <class T>
__device__ __forceinline__ void gd_ahead(const GdArgs& p, const GpProblem& gp, const GpPath& path, const GpTarget& to, int d, int unit, int u0, int w0, int mu, int mw,
                                         const GdBars& bars, GtWalk walk, int tid) {
    for (int units = 0; walk.more(); walk.next(p.offsets, p.groups), ++units) {
        walk.tile(unit);
        if (!gt_follow(bars.progress, units, 2)) continue;
        gt_prefetch_rows<T>(static_cast<const T*>(p.X) + path.src_off + u0 * d, gp.src_dim, mu * d, p.order, walk.pos, walk.rows, tid);
        gt_prefetch_rows<T>(static_cast<const T*>(p.dZ) + to.off + w0 * d, gp.dst_dim, mw * d, p.order, walk.pos, walk.rows, tid);
    }
}

// ---------------------------------------------------------------------------- sums
// A lane has one input channel and 64 output channels; sums [output channel][input channel].
template <class T>
__device__ __forceinline__ void gd_sum(const GdArgs& p, const GpProblem& gp, const GpPath& path, const GpTarget& to, int d, int unit, int u0, int w0, int mu, int mw, int n,
                                       const GdBars& bars, float* sums, GtWalk walk, unsigned tmem, int warp, int lane) {
    const int lo = walk.pos, hi = walk.hi;
    constexpr int COLS = GD_TILE / 2;
    const int quarter = warp & 3, c0 = (warp >> 2) * COLS, u = quarter * 32 + lane;
    const unsigned at = tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)c0;
    const float scale = (float)to.scale;
    GdChain<T> chain;
    float* sum = sums + c0 * GD_TILE + u;
    bool begun = false;         // the group's sums hold something
    int accs = 0;
    for (; walk.more(); walk.next(p.offsets, p.groups)) {
        walk.tile(unit);
        chain.unit(walk, d);
        if (!chain.ends) continue;
        const int buf = accs & 1;
        if (!warp_wait(true, bars.acc_full + buf, (unsigned)(accs / 2) & 1, &gt_status, ERR_GD_ACC_FULL)) return;
        tc_fence_after();
#pragma unroll 1
        for (int j = 0; j < COLS && c0 + j < n; j += 16) {
            unsigned v[16], w[GtType<T>::SPLIT ? 16 : 1];
            tc_load16(at + (unsigned)(buf * 256 + j), v);
            if constexpr (GtType<T>::SPLIT) tc_load16(at + (unsigned)(buf * 256 + n + j), w);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float s = __uint_as_float(v[i]);
                if constexpr (GtType<T>::SPLIT) s += __uint_as_float(w[i]);
                sum[(j + i) * GD_TILE] = begun ? sum[(j + i) * GD_TILE] + s : s;
            }
        }
        begun = true;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars.acc_empty + buf);
        ++accs;
        if (!chain.piece_ends) continue;
        const int begin = (int)__ldg(p.offsets + walk.g), end = GtWalk::end_of(p.offsets, walk.g);
        begun = false;
        if (u >= mu) continue;
        if (begin >= lo && end <= hi) {
            T* out = static_cast<T*>(p.dW) + (long long)walk.g * gp.w_numel + path.w_off + (long long)(u0 + u) * path.w_ld + w0 + c0;
            auto value = [&](int j) { return sum[j * GD_TILE] * scale; };
            if (p.w_vec && (path.w_off | path.w_ld) % GtType<T>::V == 0) {
#pragma unroll 2
                for (int j = 0; j < COLS && c0 + j < mw; j += GtType<T>::V) {
                    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(out + j) = make_float4(value(j), value(j + 1), value(j + 2), value(j + 3));
                    else *reinterpret_cast<uint4*>(out + j) = make_uint4(GtPair<T>::of(value(j), value(j + 1)), GtPair<T>::of(value(j + 2), value(j + 3)),
                                                                         GtPair<T>::of(value(j + 4), value(j + 5)), GtPair<T>::of(value(j + 6), value(j + 7)));
                }
            } else {
                for (int j = 0; j < COLS && c0 + j < mw; ++j) gp_store(out + j, value(j));
            }
        } else {
            float* out = p.partial + ((long long)blockIdx.x * 2 + (begin < lo ? 0 : 1)) * (GD_TILE * GD_TILE) + u * GD_TILE + c0;
#pragma unroll 4
            for (int j = 0; j < COLS && c0 + j < mw; j += 4)            // (whole pieces: the tile has room)
                *reinterpret_cast<float4*>(out + j) = make_float4(sum[j * GD_TILE], sum[(j + 1) * GD_TILE], sum[(j + 2) * GD_TILE], sum[(j + 3) * GD_TILE]);
        }
    }
}

template <class T, bool FAST>
__global__ void __launch_bounds__(GD_THREADS, 1) oeq_grouped_tc_dw(const __grid_constant__ GdProblem gd, const GdArgs p) {
    extern __shared__ __align__(1024) unsigned char gt_smem[];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    int path_no = 0;
    while ((int)blockIdx.x >= gd.split.first[path_no + 1]) ++path_no;
    const GpPath& path = gd.gp.path[path_no];
    const GpTarget& to = gd.gp.target[path.dst];
    const int parts = gd.split.parts[path_no], local = (int)blockIdx.x - gd.split.first[path_no], tile = local / parts, part = local % parts, d = to.d;
    const int w_tiles = (to.mul + GD_TILE - 1) / GD_TILE, u0 = tile / w_tiles * GD_TILE, w0 = tile % w_tiles * GD_TILE;
    const int mu = min(GD_TILE, path.src_mul - u0), mw = min(GD_TILE, to.mul - w0), n = (mw + 15) / 16 * 16;
    float* sums = reinterpret_cast<float*>(gt_smem + GD_RING * GD_SLOT);
    unsigned char* control = gt_smem + GD_RING * GD_SLOT + GD_SUMS;
    const GdBars bars(control);
    GtRange& range = *reinterpret_cast<GtRange*>(control + 512);
    constexpr int MMA_WARP = GD_PW + GD_EPI;
    if (tid == 0) {
        for (int i = 0; i < GD_BUNDLES; ++i) {
            mbar_init(bars.full + i, GD_PW / gd_sets(d));
            mbar_init(bars.empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bars.acc_full + i, 1);
            mbar_init(bars.acc_empty + i, GD_EPI);
        }
        mbar_init(bars.done, 1);
        *bars.progress = 0;
        fence_mbar_init();
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(bars.tmem)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    gt_range(range, p.offsets, p.groups, p.rows, part, parts, gd.extra[path_no]);
    tc_fence_after();
    const unsigned tmem = __shfl_sync(0xffffffffu, *reinterpret_cast<volatile unsigned*>(bars.tmem), 0);
    const long long lo = range.lo, hi = range.hi;
    if (tid == 0) p.starts[blockIdx.x] = {(int)lo, range.g};
    const GtWalk walk(p.offsets, range.g, (int)lo, (int)hi);
    if (warp > MMA_WARP) {
        gd_ahead<T>(p, gd.gp, path, to, d, gd_unit<T>(d), u0, w0, mu, mw, bars, walk, tid - (MMA_WARP + 1) * 32);
    } else if (warp == MMA_WARP) {
        gd_multiply<T>(p, d, gd_unit<T>(d), n, gt_smem, bars, walk, tmem, elect_lane());
    } else if (warp >= GD_PW) {
        gd_sum<T>(p, gd.gp, path, to, d, gd_unit<T>(d), u0, w0, mu, mw, n, bars, sums, walk, tmem, warp - GD_PW, lane);
    } else {
        if (d == 1) gd_produce<T, FAST, 1>(p, gd.gp, path, to, u0, w0, mu, mw, n, gt_smem, bars, walk, tid);
        else if (d == 3) gd_produce<T, FAST, 3>(p, gd.gp, path, to, u0, w0, mu, mw, n, gt_smem, bars, walk, tid);
        else if (d == 5) gd_produce<T, FAST, 5>(p, gd.gp, path, to, u0, w0, mu, mw, n, gt_smem, bars, walk, tid);
        else gd_produce<T, FAST, 7>(p, gd.gp, path, to, u0, w0, mu, mw, n, gt_smem, bars, walk, tid);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
}

}  // namespace oeq
