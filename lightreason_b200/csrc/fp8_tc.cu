// The FP8 products on the 5th-generation tensor cores: one persistent kernel
// for a plain product and for the two grouped products of the routed experts.
//
// Mathematics.  Within a 128-column group g both scales are constants of the
// row and of the 128-row weight block, so
//   out[m, n] = sum_g  xs[m, g] * ws[n / 128, g] * (sum over the group of xq wq).
// tcgen05.mma (kind::f8f6f4) forms the inner sum of one group, four products of
// 32 columns, in one of several TMEM buffers; eight warps read it while the
// next buffers fill and add it, times the two scales, to FP32 registers.  The
// scales are any FP32 values, so they cannot ride in the tensor core's own
// power-of-two block scales.
//
// An item is a tile of rows (of one expert) by 256 weight rows: 128 gate and
// the 128 up rows of the same columns, or 256 rows of down or of a plain
// weight.  Two layouts:
//  * BN = 0, rows as M: tiles of 128 rows against N = 256 weight rows.  An
//    accumulator lane is one row, so a group's factor is one number per thread,
//    gate and up of a column meet in one thread, and warps without rows of a
//    partial tile skip.  Large plain products run them on CTA
//    pairs (PAIR): each CTA holds 128 of an item's 256 rows and 128 of its
//    weight rows, multiplied by tcgen05.mma.cta_group::2 (M = 256), a third less
//    to load for the same work.  The first CTA issues the products; both CTAs'
//    loads complete on its barriers, its commits arrive on both CTAs', and all
//    sixteen epilogue warps hand its buffers back.
//  * BN = 16, 32 (64 for a plain product), weights as M: the two blocks of 128
//    weight rows against N = BN rows.  A lane is one weight row and the tile's few
//    rows are its columns: at a few rows per expert all eight warps share the epilogue
//    instead of one row's pair of warps doing it.
// A stage is one group: the 256 weight rows (32 KB, two boxes; a pair's CTA 128
// rows, 16 KB, one box) and the tile's rows (gathered by TMA from the token rows
// for gate/up; boxes of 16 when the tile is partial).  Three to six stages keep 96
// to 192 KB of weights in flight per SM, which is what streams the banks at small
// and middle widths (a pair's four stages 64 KB: there the products bound).
//
// The experts are one launch: gate/up items, then down items, fetched in order
// from a counter.  A down item's weights are requested at once, its rows when
// the expert's gate/up items have counted in (done[e]); every such wait is for
// an item that a running CTA already has, whatever else the GPU runs.
//
// What bounds it: the weight stream up to a few hundred rows per expert; above,
// reading the sums: a group's four products take 512 cycles, with the eight
// warps reading 128 KB of TMEM beside them 583 (each alone: 512 and 385).
//
// Warps: 0 items and weight tiles, 1 MMA, 2 and 3 row tiles and scales (four
// groups at a time, up to four such requests in flight), 4-11 epilogue; the
// first four hand registers to the others (72 and 216, the experts' 104 and
// 200, a thread of 168 at launch: 64,512 a CTA either way).  Every wait for loads,
// products, rows or items is bounded (the barriers of a CTA or cluster are not: all
// their warps come to them, having given up or not); a timeout raises *status,
// drains what is in flight and returns, and leaves NaN: in a linear's tiles of that
// CTA or pair, in all of an experts call's output.
#include <algorithm>
#include <atomic>
#include <cmath>

#include <math_constants.h>

#include "fp8_kernels.cuh"
#include "sm100.cuh"

namespace lrb {
namespace {

using fp8::kGroup;

constexpr int kBM = 128, kBN = 256;
constexpr int kBTile = kBN * kGroup;
constexpr int kThreads = 12 * 32;
constexpr int kScaleSlots = 4;  // of four groups each
constexpr int kRing = 4;        // items on their way to the warps
constexpr int kMaxExperts = 1024;
constexpr uint64_t kDrainNs = 2000000000ull;  // for products in flight, when a wait gave up

// LIN: the plain product; otherwise the experts.  PAIR: two CTAs share an item.
template <bool LIN, int BN, bool PAIR = false>
struct Shape {
    static constexpr bool kSwap = BN != 0;
    static constexpr int kRows = kSwap ? BN : kBM;  // rows of a tile
    static constexpr int kB = PAIR ? kBTile / 2 : kBTile;  // a CTA's weight bytes of a stage
    static constexpr int kATile = kRows * kGroup, kStage = kATile + kB;
    static constexpr int kStages = kSwap ? (BN == 64 ? 5 : 6) : LIN && !PAIR ? 3 : 4;
    static constexpr int kBufs = kSwap ? 4 : 2;
    static constexpr int kBufCols = kSwap ? 2 * BN : kBN;
    // an epilogue warp's output buffer: 32 rows of 256 bytes (stored by TMA) or of 64
    static constexpr int kPiece = kSwap ? 0 : LIN ? 8192 : 2048;
    struct Tail {
        // rows as M: a row's four factors together; weights as M: a group's rows together
        float row_scale[kScaleSlots][kRows * 4];
        float4 block_scale[kScaleSlots][2];
        float top[2][kSwap ? 4 : 2][kSwap ? 64 : kBM];
        int4 ring[kRing][2];
        uint64_t full[kStages], empty[kStages], tfull[kBufs], tempty[kBufs], sfull[kScaleSlots], sempty[kScaleSlots],
            ifull[kRing], iempty[kRing], half[4], drain;
        int abort, other_abort;  // this CTA, the other of its pair gave up
        uint32_t tmem;
        int32_t scan[16];
        int32_t tiles[LIN ? 1 : kMaxExperts + 1];  // row tiles of the experts before e
    };
    static constexpr int kSmem = kStages * kStage + 8 * kPiece + static_cast<int>(sizeof(Tail)) + 1024;
    static_assert(kSmem <= 232448, "shared memory of one SM");
};

struct Params {
    // linear
    const float *x_scales, *w_scales;  // [T, groups], [blocks, groups]
    int rows, n, k;                    // T, weight rows, columns
    void *out;                         // [T, n]
    int out_f32;
    int split;                         // CTAs of a cluster that share an item's groups
    bool pair;                         // two CTAs share an item's 256 rows and its weights
    // experts
    const float *act_scales_in, *down_scales;  // phase 2: [R, I / 128], [E, blocks, I / 128]
    const int32_t *offsets;                    // [E + 1]
    const int32_t *row_token;                  // [R] route -> token
    int experts, hidden, inner;
    uint8_t *act;       // [R, I] e4m3
    float *act_scales;  // [R, I / 128]
    void *y;            // [R, H] BF16 or FP32
    int y_f32;
    int32_t *work;      // items handed out so far (zero at launch)
    int32_t *done;      // [E] epilogue warps that finished an item of phase 1 (zero at launch)
    int32_t *gave_up;   // set to 1 when a wait gave up (zero at launch)
    int32_t *status;
    uint64_t wait_ns;   // the longest that a wait may take; 0: give up before the first product
};

__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
// How long a wait may take, and the CTA's flag that one took longer.
struct Patience {
    volatile int *abort;
    uint64_t ns;
};
// Bounded wait; false once the CTA has given up.  The epilogue warps do not
// leave on false: from then on their waits return after a few looks and they
// run to the end on whatever is there, together.  A look that fails takes the
// hardware 4 us; the flag and the clock are looked at after every eighth (after
// each, the kernel is 2% slower where no look fails).  CLUSTER: what the other
// CTA of a cluster did before it arrived is seen too.
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_bar(uint64_t *bar, uint32_t parity, const Patience &patience) {
    uint64_t t0 = 0;
    for (uint32_t i = 1;
         !(CLUSTER ? sm100::mbar_try_wait_cluster(bar, parity) : sm100::mbar_try_wait(bar, parity)); ++i) {
        if (i & 7) continue;
        if (*patience.abort) return false;
        const uint64_t t = now_ns();
        if (t0 == 0) t0 = t;
        if (t - t0 > patience.ns) {
            *patience.abort = 1;
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ bool wait_warp(uint64_t *bar, uint32_t parity, const Patience &patience) {
    return __all_sync(0xffffffffu, wait_bar(bar, parity, patience));
}

struct Item {
    int phase, e, row0, count, n, mt;  // 1 gate/up, 2 down or linear, 0 none; expert; first row, rows; weight tile; the expert's row tiles
};

template <int BYTES>
__device__ __forceinline__ void copy_async(void *dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(sm100::smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
}
// This thread arrives on `bar` once its copies so far are complete.
__device__ __forceinline__ void copy_async_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(sm100::smem_u32(bar)) : "memory");
}

// N (8 or 16) TMEM columns of this warp's lanes.
template <int N>
__device__ __forceinline__ void load_cols(uint32_t at, float (&v)[N]) {
    static_assert(N == 8 || N == 16, "columns");
    if constexpr (N == 16) {
        sm100::tmem_ld16(at, v);
    } else {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                     : "r"(at)
                     : "memory");
    }
}
// Completes this warp's TMEM loads; the values pass through, so no use of them
// can be moved before it.
template <int N>
__device__ __forceinline__ void wait_cols(float (&v)[N]) {
    if constexpr (N == 16)
        asm volatile("tcgen05.wait::ld.sync.aligned;"
                     : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                       "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]),
                       "+f"(v[15])
                     :
                     : "memory");
    else
        asm volatile("tcgen05.wait::ld.sync.aligned;"
                     : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7])
                     :
                     : "memory");
}

// A warp's 32 rows of 64 bytes, one row a lane, to global memory as whole
// 64-byte pieces: through 2 KB of shared memory, four lanes a row (a store of
// 16 bytes per lane to 32 rows at once costs a pass of the load/store unit for
// each row).  The 16-byte units of a row are permuted by its number, so neither
// side has bank conflicts.  Rows from `rows` on, and units from `units` on, are
// not stored.
__device__ __forceinline__ void store_rows64(uint8_t *buf, const uint32_t (&v)[16], uint8_t *dst, int64_t pitch,
                                             int rows, int units) {
    const int lane = threadIdx.x & 31;
    __syncwarp();  // the previous piece has been read
#pragma unroll
    for (int u = 0; u < 4; ++u)
        *reinterpret_cast<uint4 *>(buf + lane * 64 + ((u ^ ((lane >> 1) & 3)) * 16)) =
            make_uint4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
    __syncwarp();
    const int u = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = (lane >> 2) + 8 * i;
        const uint4 w = *reinterpret_cast<const uint4 *>(buf + r * 64 + ((u ^ ((r >> 1) & 3)) * 16));
        if (r < rows && u < units) *reinterpret_cast<uint4 *>(dst + r * pitch + u * 16) = w;
    }
}

// x / (1 + exp(-x)) from the fast exponential and quotient: off by 2^-23 times
// (4.5 + 1.2 |x|) of the value at most (their documented 2 + 1.2 |x| and 2 units in
// the last place and the sum's rounding), below what the FP32 sums behind x leave;
// below x = -87.3, where the divisor passes 2^126, it is 0 for a value of 2^-119
// at most.
__device__ __forceinline__ float silu_fast(float x) { return __fdividef(x, 1.0f + __expf(-x)); }

// A warp's 32 rows of 256 bytes (128 BF16 columns), one row a lane, staged for
// two TMA stores of 128 bytes a row under the 128-byte swizzle.
__device__ __forceinline__ void stage_row256(uint8_t *buf, const float (&acc)[128]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int u = 0; u < 16; ++u)
        *reinterpret_cast<uint4 *>(buf + (u >> 3) * 4096 + lane * 128 + (((u & 7) ^ (lane & 7)) * 16)) =
            make_uint4(fp8::pack_bf16(acc[8 * u], acc[8 * u + 1]), fp8::pack_bf16(acc[8 * u + 2], acc[8 * u + 3]),
                       fp8::pack_bf16(acc[8 * u + 4], acc[8 * u + 5]), fp8::pack_bf16(acc[8 * u + 6], acc[8 * u + 7]));
}

// 32 bytes to a 32-byte boundary: a whole sector, so that a lane can store its
// own row's columns without staging.
__device__ __forceinline__ void store32(void *p, const uint32_t *v) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// tm_x: linear, the row tiles; experts, the token rows (gathered).  tm_r, tm_r16:
// full and 16-row boxes of the rows of linear or phase 2.  tm_w, tm_w2: weights
// of linear or phase 1, and of phase 2.  tm_out: linear's BF16 output.
template <bool LIN, int BN, bool SPLIT, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_tile_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_r,
                    const __grid_constant__ CUtensorMap tm_r16, const __grid_constant__ CUtensorMap tm_w,
                    const __grid_constant__ CUtensorMap tm_w2, const __grid_constant__ CUtensorMap tm_out,
                    const Params P) {
    static_assert(LIN || !SPLIT, "only the plain product is split");
    static_assert(!PAIR || (LIN && BN == 0 && !SPLIT), "pairs have 128 rows each of a plain product");
    using S = Shape<LIN, BN, PAIR>;
    constexpr bool kSwap = S::kSwap;
    constexpr int kRows = S::kRows, kItemRows = (PAIR ? 2 : 1) * kRows;  // rows of a CTA's part, of an item
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    // a stage: the weight tile, then the rows (both on 1024-byte boundaries)
    uint8_t *pieces = smem + S::kStages * S::kStage;
    typename S::Tail *tail = reinterpret_cast<typename S::Tail *>(pieces + 8 * S::kPiece);
    volatile int *abort = &tail->abort;
    const Patience patience{abort, P.wait_ns};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // gate/up rows as M: two warps gather a tile's rows
    constexpr int kGatherWarps = kSwap ? 1 : 2;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            sm100::mbar_init(&tail->full[s], LIN ? 2 : 1 + kGatherWarps);  // the warps that load into it
            sm100::mbar_init(&tail->empty[s], 1);
        }
        for (int b = 0; b < S::kBufs; ++b) {
            sm100::mbar_init(&tail->tfull[b], 1);
            sm100::mbar_init(&tail->tempty[b], PAIR ? 16 : 8);  // the epilogue warps, of both CTAs
        }
        for (int s = 0; s < kScaleSlots; ++s) {
            sm100::mbar_init(&tail->sfull[s], 32);  // the lanes of warp 3
            sm100::mbar_init(&tail->sempty[s], 8);
        }
        for (int s = 0; s < kRing; ++s) {
            sm100::mbar_init(&tail->ifull[s], 1);
            sm100::mbar_init(&tail->iempty[s], 11);  // every warp but 0
        }
        for (int q = 0; q < 4; ++q) sm100::mbar_init(&tail->half[q], kSwap ? 4 : 2);
        sm100::mbar_init(&tail->drain, 1);
        tail->abort = P.wait_ns == 0;
        tail->other_abort = 0;
        sm100::fence_barrier_init();
        sm100::tma_prefetch_map(&tm_x);
        sm100::tma_prefetch_map(&tm_w);
        if constexpr (!LIN) {
            sm100::tma_prefetch_map(&tm_w2);
            sm100::tma_prefetch_map(&tm_r);
        }
        sm100::tma_prefetch_map(&tm_r16);
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            sm100::tmem_alloc_pair(&tail->tmem, 512);
            sm100::tmem_relinquish_pair();
        } else {
            sm100::tmem_alloc(&tail->tmem, 512);
            sm100::tmem_relinquish();
        }
    }
    sm100::tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) sm100::cluster_sync();  // the other CTA's barriers are there
    sm100::tc_fence_after();
    const uint32_t tmem = tail->tmem;
    grid_dependency_wait();
    grid_dependency_trigger();

    // groups and weight tiles of the two phases (linear is a phase 2)
    const int kbs1 = LIN ? 0 : fp8::groups(P.hidden), kbs2 = fp8::groups(LIN ? P.k : P.inner);
    const int n2 = LIN ? P.n : P.hidden;
    const int nt1 = LIN ? 0 : P.inner / kGroup, nt2 = (n2 + kBN - 1) / kBN;
    int items1 = 0, total;
    if constexpr (LIN) {
        total = nt2 * ((P.rows + kItemRows - 1) / kItemRows);
    } else {
        // tiles[e]: an exclusive scan of the experts' row tiles, a few
        // neighbouring experts a thread
        constexpr int kPer = (kMaxExperts + kThreads) / kThreads;
        int tiles[kPer], sum = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = threadIdx.x * kPer + i;
            tiles[i] = e < P.experts ? (P.offsets[e + 1] - P.offsets[e] + kRows - 1) / kRows : 0;
            sum += tiles[i];
        }
        int incl = sum;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, s);
            if (lane >= s) incl += v;
        }
        if (lane == 31) tail->scan[warp] = incl;
        __syncthreads();
        int at = incl - sum;
        for (int w = 0; w < warp; ++w) at += tail->scan[w];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = threadIdx.x * kPer + i;
            if (e <= P.experts) tail->tiles[e] = at;
            at += tiles[i];
        }
        __syncthreads();
        items1 = nt1 * tail->tiles[P.experts];
        total = items1 + nt2 * tail->tiles[P.experts];
    }
    // SPLIT: this CTA's groups of its cluster's one item; else all of an item's
    const int rank = SPLIT || PAIR ? static_cast<int>(sm100::cluster_ctarank()) : 0;
    const int split0 = SPLIT ? kbs2 * rank / P.split : 0, split1 = SPLIT ? kbs2 * (rank + 1) / P.split : kbs2;
    auto decode = [&](int item) {
        Item r;
        if (item >= total) {
            r.phase = 0;
            return r;
        }
        if constexpr (LIN) {
            r.mt = (P.rows + kItemRows - 1) / kItemRows;
            r.phase = 2;
            r.e = 0;
            r.n = item / r.mt;
            // (of a pair's second CTA perhaps past the rows: count is then not positive)
            r.row0 = (item % r.mt) * kItemRows + (PAIR ? rank * kRows : 0);
            r.count = min(kRows, P.rows - r.row0);
        } else {
            r.phase = item < items1 ? 1 : 2;
            const int nt = r.phase == 1 ? nt1 : nt2;
            const int x = r.phase == 1 ? item : item - items1, u = x / nt;
            int lo = __popc(__ballot_sync(0xffffffffu, 32 * lane <= P.experts && tail->tiles[min(32 * lane, P.experts)] <= u));
            lo = 32 * (lo - 1);
            lo += __popc(__ballot_sync(0xffffffffu, lo + lane < P.experts && tail->tiles[min(lo + lane, P.experts)] <= u)) - 1;
            const int begin = P.offsets[lo], count = P.offsets[lo + 1] - begin;
            // the tiles of one weight tile are neighbours
            r.mt = (count + kRows - 1) / kRows;
            const int at = x - nt * tail->tiles[lo];
            r.e = lo;
            r.n = at / r.mt;
            const int m = at % r.mt;
            r.row0 = begin + m * kRows;
            r.count = min(kRows, count - m * kRows);
        }
        return r;
    };
    // The item after the last one this warp took: linear, the CTA's next of a
    // fixed order; experts, from the ring that warp 0 fills.
    int take_at = SPLIT ? blockIdx.x / P.split : PAIR ? blockIdx.x / 2 : LIN ? blockIdx.x : 0;
    auto take_item = [&]() {
        if constexpr (LIN) {
            const Item r = decode(take_at);
            take_at += SPLIT ? total : PAIR ? gridDim.x / 2 : gridDim.x;
            return r;
        } else {
            const int slot = take_at % kRing;
            Item r;
            r.phase = 0;
            if (wait_warp(&tail->ifull[slot], (take_at / kRing) & 1, patience)) {
                const int4 a = tail->ring[slot][0], b = tail->ring[slot][1];
                r = Item{a.x, a.y, a.z, a.w, b.x, b.y};
            }
            __syncwarp();
            sm100::mbar_arrive_if(&tail->iempty[slot], lane == 0);
            ++take_at;
            return r;
        }
    };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(LIN ? 72 : 104));
        uint32_t stage = 0, phase = 0;
        auto next_stage = [&] {
            if (++stage == S::kStages) {
                stage = 0;
                phase ^= 1;
            }
        };
        if (warp == 0) {
            // ---------------------------------------------- items, weight tiles
            sm100::fence_proxy_async_global();  // the weights may have been written by the kernel before
            const uint64_t once = sm100::l2_evict_first_policy(), keep = sm100::l2_evict_normal_policy();
            const uint32_t one = sm100::elect_one();
            bool ok = true;
            int put_at = 0, fetched = 0;
            // the next item, also handed to the other warps (one ahead of the
            // item whose weights are being loaded)
            auto fetch = [&]() {
                if constexpr (LIN) {
                    return take_item();
                } else {
                    if (lane == 0) fetched = atomicAdd(P.work, 1);
                    fetched = __shfl_sync(0xffffffffu, fetched, 0);
                    const Item r = decode(fetched);
                    const int slot = put_at % kRing;
                    ok = wait_warp(&tail->iempty[slot], ((put_at / kRing) & 1) ^ 1, patience);
                    if (lane == 0) {
                        tail->ring[slot][0] = make_int4(r.phase, r.e, r.row0, r.count);
                        tail->ring[slot][1] = make_int4(r.n, r.mt, 0, 0);
                        sm100::mbar_arrive(&tail->ifull[slot]);
                    }
                    __syncwarp();
                    ++put_at;
                    return r;
                }
            };
            Item next = fetch();
            while (ok && next.phase) {
                const Item it = next;
                next = fetch();
                if (!ok) break;
                const bool p1 = !LIN && it.phase == 1;
                const uint64_t policy = it.mt > 1 ? keep : once;  // other tiles read the same weight rows
                const int kbs = p1 ? kbs1 : split1;
                const int r0 = it.n * (p1 ? kGroup : kBN), r1 = p1 ? P.inner + r0 : r0 + 128;
                for (int kb = split0; kb < kbs; ++kb) {
                    ok = wait_warp(&tail->empty[stage], phase ^ 1, patience);
                    if (!ok) break;
                    uint8_t *b = smem + stage * S::kStage;
                    uint64_t *bar = &tail->full[stage];
                    if (one) {
                        // a pair's loads complete on the first CTA's barrier
                        if (!PAIR || rank == 0) sm100::mbar_expect_tx(bar, kBTile);
                        if constexpr (PAIR) {
                            sm100::tma_load_2d_pair(b, &tm_w, sm100::mapa(bar, 0), kb * kGroup, r0 + 128 * rank, policy);
                        } else if constexpr (LIN) {
                            sm100::tma_load_2d_hint(b, &tm_w, bar, kb * kGroup, r0, policy);
                            sm100::tma_load_2d_hint(b + kBTile / 2, &tm_w, bar, kb * kGroup, r1, policy);
                        } else if (p1) {
                            sm100::tma_load_3d_hint(b, &tm_w, bar, kb * kGroup, r0, it.e, policy);
                            sm100::tma_load_3d_hint(b + kBTile / 2, &tm_w, bar, kb * kGroup, r1, it.e, policy);
                        } else {
                            sm100::tma_load_3d_hint(b, &tm_w2, bar, kb * kGroup, r0, it.e, policy);
                            sm100::tma_load_3d_hint(b + kBTile / 2, &tm_w2, bar, kb * kGroup, r1, it.e, policy);
                        }
                    }
                    __syncwarp();
                    next_stage();
                }
            }
            // the first CTA's products read this CTA's stages and arrive on its
            // barriers: all of them have before it may leave
            if constexpr (PAIR)
                for (int i = 0; ok && i < S::kStages; ++i) {
                    ok = wait_warp(&tail->empty[stage], phase ^ 1, patience);
                    next_stage();
                }
        } else if (warp == 1) {
            // ----------------------------------------------------- MMA issuer
            const uint32_t one = sm100::elect_one();
            uint32_t buf = 0, bphase = 0;
            bool ok = !*abort, any = false;
            for (Item it = take_item(); ok && it.phase && (!PAIR || rank == 0); it = take_item()) {
                const int kbs = !LIN && it.phase == 1 ? kbs1 : split1 - split0;
                const uint32_t idesc = sm100::idesc_e4m3_f32(PAIR ? 2 * kBM : kBM, kSwap ? (it.count + 15) & ~15 : kBN);
                for (int kb = 0; kb < kbs; ++kb) {
                    ok = wait_bar<PAIR>(&tail->tempty[buf], bphase ^ 1, patience) &&
                         wait_bar<PAIR>(&tail->full[stage], phase, patience);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    sm100::tc_fence_after();
                    const uint32_t base = sm100::smem_u32(smem + stage * S::kStage), d = tmem + buf * S::kBufCols;
                    const uint64_t w = sm100::desc_kmajor_sw128(base), w1 = sm100::desc_kmajor_sw128(base + kBTile / 2);
                    const uint64_t r = sm100::desc_kmajor_sw128(base + S::kB);
                    if constexpr (kSwap) {
                        sm100::mma_e4m3<false>(d, w, r, idesc, one);
                        sm100::mma_e4m3<false>(d + BN, w1, r, idesc, one);
#pragma unroll
                        for (int kk = 1; kk < 4; ++kk) {
                            sm100::mma_e4m3<true>(d, w + 2 * kk, r + 2 * kk, idesc, one);
                            sm100::mma_e4m3<true>(d + BN, w1 + 2 * kk, r + 2 * kk, idesc, one);
                        }
                    } else if constexpr (PAIR) {
                        sm100::mma_e4m3_pair<false>(d, r, w, idesc, one);
#pragma unroll
                        for (int kk = 1; kk < 4; ++kk) sm100::mma_e4m3_pair<true>(d, r + 2 * kk, w + 2 * kk, idesc, one);
                    } else {
                        sm100::mma_e4m3<false>(d, r, w, idesc, one);
#pragma unroll
                        for (int kk = 1; kk < 4; ++kk) sm100::mma_e4m3<true>(d, r + 2 * kk, w + 2 * kk, idesc, one);
                    }
                    if constexpr (PAIR) {
                        sm100::mma_commit_pair_if(&tail->tfull[buf], one);
                        sm100::mma_commit_pair_if(&tail->empty[stage], one);
                    } else {
                        sm100::mma_commit_if(&tail->tfull[buf], one);
                        sm100::mma_commit_if(&tail->empty[stage], one);
                    }
                    __syncwarp();
                    any = true;
                    next_stage();
                    if (++buf == S::kBufs) {
                        buf = 0;
                        bphase ^= 1;
                    }
                }
            }
            if (*abort && any) {
                if (one) {
                    if constexpr (PAIR) sm100::mma_commit_pair(&tail->drain, 1);
                    else sm100::mma_commit(&tail->drain);
                }
                const uint64_t t0 = now_ns();
                while (!sm100::mbar_try_wait(&tail->drain, 0) && now_ns() - t0 < kDrainNs) {
                }
            }
            __syncwarp();
        } else {
            // --------------------------------------------- row tiles, scales
            // Warp 2 loads the rows: gathered four a lane, or one box, or
            // boxes of 16 rows one a lane.  Warp 3 requests the scales, and
            // with 128-row tiles gathers the second 64 rows: a warp's lanes
            // issue their gathers one after another, two warps halve that time.
            sm100::fence_proxy_async_global();
            const uint64_t rows_policy = sm100::l2_evict_normal_policy();
            constexpr int kPerWarp = kRows / kGatherWarps;  // gathered rows of a warp
            const int g0 = kPerWarp * (warp - 2) + 4 * lane;
            uint32_t slot = 0, sphase = 0;
            // warp 3, lane l: the scales of rows l, l + 32, ... of the tile
            constexpr int kScaleRows = (kRows + 31) / 32;
            auto copy4 = [&](float *dst, int step, const float *src, int kb, int kbs, bool quads) {
                if (quads && step == 1) {
                    copy_async<16>(dst, src + kb);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (kb + i < kbs) copy_async<4>(dst + i * step, src + kb + i);
                }
            };
            Item next = take_item();
            int next_gather[4] = {}, next_scaled[kScaleRows] = {};
            auto rows_of = [&](const Item &it) {
                if (!it.phase) return;
                const bool p1 = !LIN && it.phase == 1;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (p1) next_gather[i] = P.row_token[it.row0 + min(g0 + i, it.count - 1)];
#pragma unroll
                for (int j = 0; j < kScaleRows; ++j) {
                    const int r = it.row0 + min(lane + 32 * j, it.count - 1);
                    next_scaled[j] = p1 ? (warp == 3 ? P.row_token[r] : 0) : r;
                }
            };
            rows_of(next);
            bool ok = true;
            while (ok && next.phase) {
                const Item it = next;
                int gather[4], scaled[kScaleRows];
#pragma unroll
                for (int i = 0; i < 4; ++i) gather[i] = next_gather[i];
#pragma unroll
                for (int j = 0; j < kScaleRows; ++j) scaled[j] = next_scaled[j];
                next = take_item();
                rows_of(next);
                const bool p1 = !LIN && it.phase == 1;
                const int kbs = p1 ? kbs1 : kbs2;
                const float *rs = LIN || p1 ? P.x_scales : P.act_scales_in;
                const float *bs = LIN || p1 ? P.w_scales : P.down_scales;
                const bool quads = kbs % 4 == 0 && ((reinterpret_cast<uintptr_t>(rs) | reinterpret_cast<uintptr_t>(bs)) & 15) == 0 &&
                                   (!SPLIT || split0 % 4 == 0);
                if (!LIN && !p1) {
                    // the expert's activations: every epilogue warp of its phase-1 items
                    const int need = 8 * nt1 * it.mt;
                    const uint64_t t0 = now_ns();
                    while (sm100::ld_acquire(P.done + it.e) < need) {
                        if (*abort || now_ns() - t0 >= P.wait_ns) {
                            *abort = 1;
                            break;
                        }
                        __nanosleep(32);
                    }
                    ok = __all_sync(0xffffffffu, !*abort);
                    if (!ok) break;
                    sm100::fence_proxy_async_global();
                }
                const bool loads = warp == 2 || (p1 && kGatherWarps == 2);
                // lanes that load, and what a lane loads
                const int boxes = p1 ? min(kPerWarp / 4, (max(0, it.count - kPerWarp * (warp - 2)) + 3) / 4)
                                     : it.count == kRows ? 1 : (it.count + 15) / 16;
                const int box_bytes = p1 ? 4 * kGroup : it.count == kRows ? S::kATile : 16 * kGroup;
                for (int kb = split0; kb < (p1 ? kbs1 : split1); ++kb) {
                    if (warp == 3 && ((kb - split0) & 3) == 0) {
                        // the scales of groups kb .. kb + 3, on their way from here
                        ok = wait_warp(&tail->sempty[slot], sphase ^ 1, patience);
                        if (!ok) break;
#pragma unroll
                        for (int j = 0; j < kScaleRows; ++j) {
                            const int r = lane + 32 * j;
                            if (r < kRows)
                                copy4(&tail->row_scale[slot][kSwap ? r : 4 * r], kSwap ? kRows : 1,
                                      rs + static_cast<int64_t>(scaled[j]) * kbs, kb, kbs, quads);
                        }
                        // lanes 0 and 1: the item's two weight blocks (gate and
                        // up, or the two halves of the 256 weight rows; one
                        // past the matrix is never used)
                        if (lane < 2) {
                            const int per = fp8::groups(n2);
                            const int64_t blk = p1 ? static_cast<int64_t>(it.e) * 2 * nt1 + it.n + lane * nt1
                                                   : static_cast<int64_t>(it.e) * per + min(2 * it.n + lane, per - 1);
                            copy4(&tail->block_scale[slot][lane].x, 1, bs + blk * kbs, kb, kbs, quads);
                        }
                        copy_async_arrive(&tail->sfull[slot]);
                        if (++slot == kScaleSlots) {
                            slot = 0;
                            sphase ^= 1;
                        }
                    }
                    if (warp == 3 && (LIN || kGatherWarps == 1)) continue;
                    ok = wait_warp(&tail->empty[stage], phase ^ 1, patience);
                    if (!ok) break;
                    uint8_t *a = smem + stage * S::kStage + S::kB;
                    uint64_t *bar = &tail->full[stage];
                    if constexpr (PAIR) {
                        if (lane == 0) {
                            if (rank == 0) sm100::mbar_expect_tx(bar, 2 * S::kATile);
                            sm100::tma_load_2d_pair(a, &tm_r, sm100::mapa(bar, 0), kb * kGroup, it.row0, rows_policy);
                        }
                        __syncwarp();
                        next_stage();
                        continue;
                    }
                    if (lane == 0) {
                        if (loads) sm100::mbar_expect_tx(bar, boxes * box_bytes);
                        else sm100::mbar_arrive(bar);
                    }
                    __syncwarp();
                    if (loads && lane < boxes) {
                        if (p1) sm100::tma_gather4(a + g0 * kGroup, &tm_x, bar, kb * kGroup, gather);
                        else sm100::tma_load_2d(a + lane * box_bytes, it.count == kRows ? &tm_r : &tm_r16, bar,
                                                kb * kGroup, it.row0 + lane * 16);
                    }
                    next_stage();
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
    } else {
        // ----------------------------------------------------------- epilogue
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(LIN ? 216 : 200));
        const int q = warp & 3, h = warp >= 8;  // TMEM lanes 32q..; half of the columns
        const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * q) << 16);
        float *partial = reinterpret_cast<float *>(smem);  // SPLIT: the stages, when all of them are used
        uint32_t slot = 0, sphase = 0, buf = 0, bphase = 0, iphase = 0;
        auto release_buf = [&] {
            sm100::tc_fence_before();
            __syncwarp();
            if constexpr (PAIR) sm100::mbar_arrive_cluster_if(sm100::mapa(&tail->tempty[buf], 0), lane == 0);
            else sm100::mbar_arrive_if(&tail->tempty[buf], lane == 0);
        };
        auto next_buf = [&] {
            if (++buf == S::kBufs) {
                buf = 0;
                bphase ^= 1;
            }
        };
        auto next_slot = [&] {
            __syncwarp();
            sm100::mbar_arrive_if(&tail->sempty[slot], lane == 0);
            if (++slot == kScaleSlots) {
                slot = 0;
                sphase ^= 1;
            }
        };
        // this warp's part of a phase-1 item is stored
        auto count_in = [&](const Item &it) {
            __syncwarp();
            if (lane == 0)
                asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(P.done + it.e) : "memory");
        };
        if constexpr (kSwap) {
            // This warp: weight rows 32q + lane of both blocks, rows NJ h .. of the tile.
            constexpr int NJ = BN / 2, NL = NJ < 16 ? NJ : 16;
            const int j0 = NJ * h;
            for (Item it = take_item(); it.phase; it = take_item()) {
                const bool p1 = !LIN && it.phase == 1;
                const int kbs = p1 ? kbs1 : split1 - split0;
                const bool active = j0 < it.count;
                float acc0[NJ], acc1[NJ];
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc0[j] = acc1[j] = 0.f;
                for (int kb = 0; kb < kbs; ++kb) {
                    if ((kb & 3) == 0) wait_bar(&tail->sfull[slot], sphase, patience);
                    const float b0 = reinterpret_cast<const float *>(&tail->block_scale[slot][0])[kb & 3];
                    const float b1 = reinterpret_cast<const float *>(&tail->block_scale[slot][1])[kb & 3];
                    wait_bar(&tail->tfull[buf], bphase, patience);
                    sm100::tc_fence_after();
                    if (active) {
                        const uint32_t at = lanes + buf * S::kBufCols + j0;
#pragma unroll
                        for (int c = 0; c < NJ; c += NL) {
                            float t0[NL], t1[NL], s[NL];
                            load_cols<NL>(at + c, t0);
                            load_cols<NL>(at + BN + c, t1);
#pragma unroll
                            for (int j = 0; j < NL; j += 4)
                                *reinterpret_cast<float4 *>(&s[j]) = *reinterpret_cast<const float4 *>(
                                    &tail->row_scale[slot][(kb & 3) * kRows + j0 + c + j]);
                            wait_cols(t0);
                            wait_cols(t1);
#pragma unroll
                            for (int j = 0; j < NL; ++j) {
                                acc0[c + j] = fmaf(t0[j], s[j] * b0, acc0[c + j]);
                                acc1[c + j] = fmaf(t1[j], s[j] * b1, acc1[c + j]);
                            }
                        }
                    }
                    release_buf();
                    next_buf();
                    if ((kb & 3) == 3 || kb + 1 == kbs) next_slot();
                }
                const int left = it.count - j0;  // rows of this warp, if below NJ
                if (p1) {
                    if (active) {
                        // |h| over the 128 lanes of the block: bit patterns of
                        // magnitudes order like the values, NaN above all
#pragma unroll
                        for (int j = 0; j < NJ; ++j) {
                            acc0[j] = silu_fast(acc0[j]) * acc1[j];
                            const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(acc0[j])));
                            if (lane == (j & 31)) tail->top[iphase][q][j0 + j] = __uint_as_float(m);
                        }
                        __syncwarp();
                        sm100::mbar_arrive_if(&tail->half[h], lane == 0);
                        wait_bar(&tail->half[h], iphase, patience);
                        uint8_t *dst = P.act + static_cast<int64_t>(it.row0 + j0) * P.inner + it.n * kGroup + 32 * q + lane;
#pragma unroll
                        for (int j = 0; j < NJ; ++j) {
                            float top = fp8::kTiny;
#pragma unroll
                            for (int i = 0; i < 4; ++i) top = fp8::max_nan(top, tail->top[iphase][i][j0 + j]);
                            const fp8::Divisor f(top);
                            if (j < left) {
                                dst[static_cast<int64_t>(j) * P.inner] = static_cast<uint8_t>(fp8::pack2(f(acc0[j]), 0.f));
                                if (q == 0 && lane == (j & 31))
                                    P.act_scales[static_cast<int64_t>(it.row0 + j0 + j) * nt1 + it.n] = fp8::scale_of(top);
                            }
                        }
                        iphase ^= 1;
                    }
                    count_in(it);
                } else if (SPLIT) {
                    // partial sums [row][weight row] for the cluster
#pragma unroll
                    for (int j = 0; j < NJ; ++j) {
                        partial[(j0 + j) * kBN + 32 * q + lane] = acc0[j];
                        partial[(j0 + j) * kBN + 128 + 32 * q + lane] = acc1[j];
                    }
                } else if (active) {
                    const int c0 = it.n * kBN + 32 * q + lane;
                    const bool f32 = LIN ? P.out_f32 : P.y_f32;
                    void *base = LIN ? P.out : P.y;
                    const int64_t at = static_cast<int64_t>(it.row0 + j0) * n2 + c0;
                    uint16_t *y = static_cast<uint16_t *>(base) + at;
                    float *z = static_cast<float *>(base) + at;
#pragma unroll
                    for (int j = 0; j < NJ; ++j) {
                        if (j >= left) break;
                        const int64_t o = static_cast<int64_t>(j) * n2;
                        if (f32) {
                            if (c0 < n2) z[o] = acc0[j];
                            if (c0 + 128 < n2) z[o + 128] = acc1[j];
                        } else {
                            if (c0 < n2) y[o] = f2bf(acc0[j]);
                            if (c0 + 128 < n2) y[o + 128] = f2bf(acc1[j]);
                        }
                    }
                }
            }
        } else {
            const int r = 32 * q + lane;
            uint8_t *piece = pieces + (warp - 4) * S::kPiece;
            // the factors of the next four groups: row scale x weight scale (gate's and up's)
            float s0[4], s1[4];
            auto take_scales = [&](bool p1) {
                wait_bar(&tail->sfull[slot], sphase, patience);
                const float4 rs = *reinterpret_cast<const float4 *>(&tail->row_scale[slot][4 * r]);
                const float4 b0 = tail->block_scale[slot][p1 ? 0 : h];
                s0[0] = rs.x * b0.x, s0[1] = rs.y * b0.y, s0[2] = rs.z * b0.z, s0[3] = rs.w * b0.w;
                if constexpr (!LIN) {
                    const float4 b1 = tail->block_scale[slot][p1 ? 1 : h];
                    s1[0] = rs.x * b1.x, s1[1] = rs.y * b1.y, s1[2] = rs.z * b1.z, s1[3] = rs.w * b1.w;
                }
                next_slot();
            };
            Item next = take_item();
            bool ready = false;  // s0 and s1 are the next item's
            while (next.phase) {
                const Item it = next;
                const bool p1 = !LIN && it.phase == 1;
                const int kbs = p1 ? kbs1 : split1 - split0;
                const bool active = 32 * q < it.count;  // the warp has rows of the tile
                float acc[128];
#pragma unroll
                for (int i = 0; i < 128; ++i) acc[i] = 0.f;
                if (!ready) take_scales(p1);
                ready = false;
                // 16 columns at a time; gate/up: 64 of the gate block, then the
                // same 64 of the up block
                const uint32_t at = lanes + (p1 ? 64 * h : 128 * h), skip = p1 ? 64 : 0;
                for (int kb = 0; kb < kbs; ++kb) {
                    const float g0 = s0[0], g1 = LIN ? s0[0] : s1[0];
#pragma unroll
                    for (int i = 0; i < 3; ++i) {
                        s0[i] = s0[i + 1];
                        if (!LIN) s1[i] = s1[i + 1];
                    }
                    wait_bar(&tail->tfull[buf], bphase, patience);
                    sm100::tc_fence_after();
                    if (active) {
                        const uint32_t base = at + buf * kBN;
                        float t[2][16];
                        load_cols<16>(base, t[0]);
                        wait_cols(t[0]);
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            if (c < 7) load_cols<16>(base + 16 * (c + 1) + (c >= 3 ? skip : 0), t[(c + 1) & 1]);
                            else release_buf();  // all of it is in registers
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                acc[16 * c + i] = fmaf(t[c & 1][i], c < 4 ? g0 : g1, acc[16 * c + i]);
                            if (c < 7) wait_cols(t[(c + 1) & 1]);
                        }
                    }
                    if (!active) release_buf();
                    next_buf();
                    // behind the buffer's release: the products go on meanwhile
                    if ((kb & 3) == 3 && kb + 1 < kbs) take_scales(p1);
                }
                // The next item's first factors, before this one is stored --
                // unless they may be waiting for this very item's rows.
                next = take_item();
                if (next.phase && (LIN || next.phase == it.phase)) {
                    take_scales(!LIN && next.phase == 1);
                    ready = true;
                }
                const int rows = it.count - 32 * q;  // of this warp, if below 32
                const int64_t first = static_cast<int64_t>(it.row0) + 32 * q;
                if (p1) {
                    if (active) {
                        float top = fp8::kTiny;
#pragma unroll
                        for (int i = 0; i < 64; ++i) {
                            acc[i] = silu_fast(acc[i]) * acc[64 + i];
                            top = fp8::max_nan(top, fabsf(acc[i]));
                        }
                        // the group's other 64 columns are the other half's
                        tail->top[iphase][h][r] = top;
                        __syncwarp();
                        sm100::mbar_arrive_if(&tail->half[q], lane == 0);
                        wait_bar(&tail->half[q], iphase, patience);
                        top = fp8::max_nan(top, tail->top[iphase][h ^ 1][r]);
                        iphase ^= 1;
                        const fp8::Divisor f(top);
                        uint32_t v[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            v[i] = fp8::pack4(f, acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
                        store_rows64(piece, v, P.act + first * P.inner + it.n * kGroup + 64 * h, P.inner, rows, 4);
                        if (h == 0 && lane < rows) P.act_scales[(first + lane) * nt1 + it.n] = fp8::scale_of(top);
                    }
                    count_in(it);
                } else if (SPLIT) {
                    // partial sums [weight row][row] for the cluster
#pragma unroll
                    for (int i = 0; i < 128; ++i) partial[(128 * h + i) * kBM + r] = acc[i];
                } else if (active) {
                    const int n0 = it.n * kBN + 128 * h;
                    const bool f32 = LIN && P.out_f32;
                    // whole 16-byte units: 8 BF16 or 4 FP32 columns, all or none
                    // of them there (the experts' H is a multiple of 16)
                    const bool vec = !LIN || n2 % (f32 ? 4 : 8) == 0;
                    if (LIN && vec && !f32) {
                        // the map cuts rows and columns past the matrix
                        if (lane == 0) sm100::bulk_wait_read();  // the last item's stores have left the buffer
                        __syncwarp();
                        stage_row256(piece, acc);
                        sm100::fence_proxy_async_shared();
                        __syncwarp();
                        if (lane == 0) {
                            if (n0 < n2) sm100::tma_store_2d(piece, &tm_out, n0, static_cast<int>(first));
                            if (n0 + 64 < n2)
                                sm100::tma_store_2d(piece + 4096, &tm_out, n0 + 64, static_cast<int>(first));
                            sm100::bulk_commit();
                        }
                    } else if (!LIN) {
                        const int64_t o = (first + lane) * n2 + n0;
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            if (lane >= rows || n0 + 16 * c >= n2) continue;
                            uint32_t v[8];
                            if (P.y_f32) {
                                float *dst = static_cast<float *>(P.y) + o + 16 * c;
#pragma unroll
                                for (int g = 0; g < 2; ++g) {
#pragma unroll
                                    for (int i = 0; i < 8; ++i) v[i] = __float_as_uint(acc[16 * c + 8 * g + i]);
                                    store32(dst + 8 * g, v);
                                }
                            } else {
#pragma unroll
                                for (int i = 0; i < 8; ++i)
                                    v[i] = fp8::pack_bf16(acc[16 * c + 2 * i], acc[16 * c + 2 * i + 1]);
                                store32(static_cast<uint16_t *>(P.y) + o + 16 * c, v);
                            }
                        }
                    } else if (vec) {
                        float *dst = static_cast<float *>(P.out) + first * n2 + n0;
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            uint32_t v[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(acc[16 * c + i]);
                            store_rows64(piece + 2048 * (c & 3), v, reinterpret_cast<uint8_t *>(dst + 16 * c),
                                         4 * static_cast<int64_t>(n2), rows, (n2 - n0 - 16 * c) / 4);
                        }
                    } else if (lane < rows) {
                        const int64_t o = (first + lane) * n2 + n0;
#pragma unroll
                        for (int i = 0; i < 128; ++i) {
                            if (n0 + i >= n2) continue;
                            if (f32) static_cast<float *>(P.out)[o + i] = acc[i];
                            else static_cast<uint16_t *>(P.out)[o + i] = f2bf(acc[i]);
                        }
                    }
                }
            }
            if (LIN && lane == 0) sm100::bulk_wait_all();
        }
        __syncwarp();
        sm100::tc_fence_before();
    }
    if constexpr (SPLIT) {
        // Every CTA has its partial sums in shared memory; each adds up and
        // stores an equal part of the tile's columns, in rank order.
        __syncwarp();
        sm100::cluster_sync();
        if (warp >= 4) {
            const Item it = decode(blockIdx.x / P.split);
            const int tid = threadIdx.x - 128, cols = kBN / P.split;
            const uint32_t base = sm100::smem_u32(smem);
            // sums of N places, `step` apart, of every CTA: a CTA's N loads in flight together
            auto sums = [&](auto &v, int at, int step) {
#pragma unroll
                for (float &x : v) x = 0.f;
                for (int c = 0; c < P.split; ++c) {
                    const uint32_t from = sm100::mapa_u32(base, c) + 4 * at;
                    constexpr int N = sizeof(v) / sizeof(float);
                    float w[N];
#pragma unroll
                    for (int i = 0; i < N; ++i) w[i] = sm100::ld_cluster_f32(from + 4 * i * step);
#pragma unroll
                    for (int i = 0; i < N; ++i) v[i] += w[i];
                }
            };
            uint16_t *y = static_cast<uint16_t *>(P.out);
            float *z = static_cast<float *>(P.out);
            if constexpr (kSwap) {
                // column tid % cols of this CTA's; rows tid / cols, + step, ...
                const int step = 256 / cols, c = tid % cols + rank * cols, n = it.n * kBN + c;
                for (int j = tid / cols; j < it.count; j += 4 * step) {
                    float v[4];  // places past the tile's rows are still in the stages, and not stored
                    sums(v, j * kBN + c, step * kBN);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int64_t o = static_cast<int64_t>(it.row0 + j + i * step) * n2 + n;
                        if (n >= n2 || j + i * step >= it.count) continue;
                        if (P.out_f32) z[o] = v[i];
                        else y[o] = f2bf(v[i]);
                    }
                }
            } else {
                const int r = tid & 127;
                const bool vec = n2 % (P.out_f32 ? 4 : 8) == 0;
                for (int c = rank * cols + (tid >> 7) * (cols / 2), end = c + cols / 2; c < end; c += 16) {
                    const int n = it.n * kBN + c;
                    if (r >= it.count || n >= n2) continue;
                    float v[16];
                    sums(v, c * kBM + r, kBM);
                    const int64_t o = static_cast<int64_t>(it.row0 + r) * n2 + n;
                    if (vec && P.out_f32) {
#pragma unroll
                        for (int i = 0; i < 16; i += 4)
                            if (n + i < n2)
                                *reinterpret_cast<float4 *>(z + o + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    } else if (vec) {
#pragma unroll
                        for (int i = 0; i < 16; i += 8)
                            if (n + i < n2)
                                *reinterpret_cast<uint4 *>(y + o + i) =
                                    make_uint4(fp8::pack_bf16(v[i], v[i + 1]), fp8::pack_bf16(v[i + 2], v[i + 3]),
                                               fp8::pack_bf16(v[i + 4], v[i + 5]), fp8::pack_bf16(v[i + 6], v[i + 7]));
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            if (n + i >= n2) continue;
                            if (P.out_f32) z[o + i] = v[i];
                            else y[o + i] = f2bf(v[i]);
                        }
                    }
                }
            }
        }
        __syncwarp();
        sm100::cluster_sync();  // no CTA leaves while another reads its sums
    }
    __syncthreads();  // no warp issues loads or products any more
    if constexpr (PAIR) {
        // A pair gives up together: once one of its CTAs has, its epilogue warps
        // hand buffers back unread, and those count for the other's.  Nor does a
        // CTA leave while the other may arrive on its barriers.
        if (threadIdx.x == 0 && *abort) sm100::st_cluster_u32(sm100::mapa(&tail->other_abort, rank ^ 1), 1);
        __syncwarp();
        sm100::cluster_sync();
    }
    const bool gave_up = *abort || (PAIR && *static_cast<volatile int *>(&tail->other_abort));
    if (gave_up) {
        // loads and products may be in flight whose barriers will never
        // complete: give them a time far above any load's before the CTA leaves
        const uint64_t t0 = now_ns();
        while (now_ns() - t0 < 200000) __nanosleep(1000);
        __syncwarp();
    }
    if (warp == 1) {
        sm100::tc_fence_after();
        if constexpr (PAIR) sm100::tmem_dealloc_pair(tmem, 512);
        else sm100::tmem_dealloc(tmem, 512);
    }
    if (LIN && gave_up) {
        // NaN in place of this CTA's tiles (here, and not in the items' own
        // path, where the test alone cost a twentieth of the time)
        const int step = SPLIT ? total : PAIR ? gridDim.x / 2 : gridDim.x;
        for (int item = SPLIT ? blockIdx.x / P.split : PAIR ? blockIdx.x / 2 : blockIdx.x; item < total; item += step) {
            const Item it = decode(item);
            for (int i = threadIdx.x; i < it.count * kBN; i += kThreads) {
                const int n = it.n * kBN + i % kBN;
                const int64_t o = static_cast<int64_t>(it.row0 + i / kBN) * n2 + n;
                if (n >= n2) continue;
                if (P.out_f32) static_cast<float *>(P.out)[o] = CUDART_NAN_F;
                else static_cast<uint16_t *>(P.out)[o] = 0x7fff;
            }
        }
    }
    if (threadIdx.x == 0 && gave_up) {
        if (P.status) atomicExch(P.status, 1);
        if (!LIN) atomicExch(P.gave_up, 1);
    }
}

// The experts' plan, by one CTA or a cluster of eight with an equal share of
// the routes each: count the share's routes per expert in shared memory, scan
// the experts' totals over the cluster, and hand out places from one counter
// per expert.  The rows of an expert come in no fixed order; no result depends
// on it, since a row's products are its own and the weighted sum goes by
// route_pos.  Also zeroes the tile kernel's counters.
__global__ void __launch_bounds__(1024) fp8_plan_kernel(const int64_t *idx, int routes, int top_k,
                                                                int experts, int32_t *__restrict__ offsets,
                                                                int32_t *__restrict__ row_token,
                                                                int32_t *__restrict__ route_pos,
                                                                int32_t *__restrict__ counters) {
    __shared__ int32_t count[kMaxExperts], cursor[kMaxExperts], scan[32];
    const int x = threadIdx.x, lane = x & 31, warp = x >> 5;
    const int threads = blockDim.x;                // at least the experts
    const int ctas = gridDim.x, cta = blockIdx.x;  // one cluster
    count[x] = 0;
    grid_dependency_wait();
    grid_dependency_trigger();
    if (cta == 0)
        for (int i = x; i < experts + 2; i += threads) counters[i] = 0;
    __syncthreads();
    const int per = (routes + ctas - 1) / ctas, r0 = cta * per, r1 = min(routes, r0 + per);
    constexpr int kU = 4;  // routes of a thread in flight
    auto each = [&](auto &&f) {
        for (int r = r0 + x; r < r1; r += kU * threads) {
            int64_t id[kU];
#pragma unroll
            for (int u = 0; u < kU; ++u) id[u] = r + u * threads < r1 ? idx[r + u * threads] : -1;
#pragma unroll
            for (int u = 0; u < kU; ++u)
                if (r + u * threads < r1)
                    f(r + u * threads, id[u] >= 0 && id[u] < experts ? static_cast<int>(id[u]) : -1);
        }
    };
    each([&](int, int e) {
        if (e >= 0) atomicAdd(&count[e], 1);
    });
    if (ctas > 1) sm100::cluster_sync();
    else __syncthreads();
    int before = 0, total = 0;  // expert x: its routes in the CTAs before, in all
    if (x < experts) {
        for (int c = 0; c < ctas; ++c) {
            const int v = ctas > 1 ? sm100::ld_cluster_s32(sm100::mapa(&count[x], c)) : count[x];
            if (c < cta) before += v;
            total += v;
        }
    }
    int incl = total;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, s);
        if (lane >= s) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    int begin = incl - total;
    for (int w = 0; w < warp; ++w) begin += scan[w];
    if (x < experts) {
        cursor[x] = begin + before;
        if (cta == 0) {
            offsets[x] = begin;
            if (x == experts - 1) offsets[experts] = begin + total;
        }
    }
    __syncthreads();
    each([&](int r, int e) {
        const int pos = e >= 0 ? atomicAdd(&cursor[e], 1) : -1;
        if (e >= 0) row_token[pos] = r / top_k;
        route_pos[r] = pos;
    });
    if (ctas > 1) sm100::cluster_sync();  // no CTA leaves while another reads its counts
}

// out[t] = sum over the token's routes, in slot order, of weight * row, in
// FP32.  A thread per 16 bytes of a row, eight rows in flight.  The first
// routes' places and weights are there before the wait: the plan kernel and
// whatever wrote the weights were complete when the tile kernel let this one
// start.
template <class Y>
__global__ void __launch_bounds__(128) fp8_combine_kernel(const Y *y, const int32_t *route_pos,
                                                          const uint16_t *weights, const int32_t *gave_up, int tokens,
                                                          int top_k, int hidden, uint16_t *__restrict__ out) {
    constexpr int kU = 8, kCols = 16 / sizeof(Y);
    const int units = hidden / kCols;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x;
    const int64_t t = i / units;
    const int c = static_cast<int>(i % units) * kCols;
    int pos[kU];
    float w[kU];
    auto routes = [&](int k0) {
#pragma unroll
        for (int k = 0; k < kU; ++k) {
            const int64_t at = t * top_k + k0 + k;
            const bool there = t < tokens && k0 + k < top_k;
            pos[k] = there ? __ldcg(route_pos + at) : -1;
            w[k] = there ? bf2f(__ldcg(weights + at)) : 0.f;
        }
    };
    routes(0);
    grid_dependency_wait();
    grid_dependency_trigger();
    if (t >= tokens) return;
    const float zero = __ldcg(gave_up) ? CUDART_NAN_F : 0.f;
    float acc[kCols];
#pragma unroll
    for (int j = 0; j < kCols; ++j) acc[j] = zero;
    for (int k0 = 0; k0 < top_k; k0 += kU) {
        if (k0) routes(k0);
        uint4 v[kU];
#pragma unroll
        for (int k = 0; k < kU; ++k)
            v[k] = pos[k] >= 0 ? fp8::ld_once(y + static_cast<int64_t>(pos[k]) * hidden + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < kU; ++k) {
            if (pos[k] < 0) continue;  // a weight of a dropped route may be anything
            const uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (kCols == 4) {
                    acc[j] = fmaf(__uint_as_float(u[j]), w[k], acc[j]);
                } else {
                    acc[2 * j] = fmaf(bf16_lo(u[j]), w[k], acc[2 * j]);
                    acc[2 * j + 1] = fmaf(bf16_hi(u[j]), w[k], acc[2 * j + 1]);
                }
            }
        }
    }
    if constexpr (kCols == 4)
        *reinterpret_cast<uint2 *>(out + t * hidden + c) =
            make_uint2(fp8::pack_bf16(acc[0], acc[1]), fp8::pack_bf16(acc[2], acc[3]));
    else
        *reinterpret_cast<uint4 *>(out + t * hidden + c) =
            make_uint4(fp8::pack_bf16(acc[0], acc[1]), fp8::pack_bf16(acc[2], acc[3]),
                       fp8::pack_bf16(acc[4], acc[5]), fp8::pack_bf16(acc[6], acc[7]));
}

template <bool LIN, int BN>
int launch_tile(const CUtensorMap (&m)[6], const Params &P, int64_t items, cudaStream_t stream) {
    constexpr int smem = Shape<LIN, BN>::kSmem;
    if constexpr (LIN) {
        if (P.split > 1) {
            static_assert(Shape<LIN, BN>::kStages * Shape<LIN, BN>::kStage >= Shape<LIN, BN>::kRows * kBN * 4,
                          "the partial sums fit the stages");
            auto kernel = fp8_tile_kernel<LIN, BN, true, false>;
            if (int rc = ensure_dynamic_smem(kernel, smem, "cudaFuncSetAttribute(fp8_tile)")) return rc;
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(static_cast<unsigned>(items * P.split));
            cfg.blockDim = dim3(kThreads);
            cfg.dynamicSmemBytes = smem;
            cfg.stream = stream;
            cudaLaunchAttribute attr[2];
            attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[0].val.programmaticStreamSerializationAllowed = 1;
            attr[1].id = cudaLaunchAttributeClusterDimension;
            attr[1].val.clusterDim.x = P.split;
            attr[1].val.clusterDim.y = 1;
            attr[1].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 2;
            const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, m[0], m[1], m[2], m[3], m[4], m[5], P);
            return err == cudaSuccess ? MOE_OK : cuda_error(err, "fp8_tile_kernel");
        }
    }
    if constexpr (LIN && BN == 0) {
        if (P.pair) {
            auto kernel = fp8_tile_kernel<true, 0, false, true>;
            constexpr int pair_smem = Shape<true, 0, true>::kSmem;
            if (int rc = ensure_dynamic_smem(kernel, pair_smem, "cudaFuncSetAttribute(fp8_tile)")) return rc;
            const int clusters = static_cast<int>(std::min<int64_t>(items, grouped_pair_clusters()));
            return launch_pdl_cluster2(kernel, dim3(2 * clusters), dim3(kThreads), pair_smem, stream, "fp8_tile_kernel",
                                       m[0], m[1], m[2], m[3], m[4], m[5], P);
        }
    }
    auto kernel = fp8_tile_kernel<LIN, BN, false, false>;
    if (int rc = ensure_dynamic_smem(kernel, smem, "cudaFuncSetAttribute(fp8_tile)")) return rc;
    return launch_pdl(kernel, dim3(static_cast<unsigned>(std::min<int64_t>(items, sm_count()))),
                      dim3(kThreads), smem, stream, "fp8_tile_kernel", m[0], m[1], m[2], m[3], m[4], m[5], P);
}

// Rows [rows, cols] in boxes of `full` and of 16 rows.
int row_maps(CUtensorMap *m, CUtensorMap *m16, const void *base, int rows, int cols, int full) {
    const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
    const uint64_t str[1] = {static_cast<uint64_t>(cols)};
    if (int rc = make_map_u8(m, base, 2, dims, str, full)) return rc;
    return make_map_u8(m16, base, 2, dims, str, 16);
}

// One CTA up to 2048 routes; eight (9 us at 32,768 routes) above.
int launch_plan(const ExpertsFp8 &a, const ExpertsFp8Scratch &s, int routes, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(routes <= 2048 ? 1 : 8);
    cfg.blockDim = dim3((std::max(a.experts, std::min(routes, 1024)) + 31) / 32 * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cfg.gridDim.x;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cfg.gridDim.x > 1 ? 2 : 1;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, fp8_plan_kernel, a.idx, routes, a.top_k, a.experts, s.offsets,
                                               s.row_token, s.route_pos, s.counters);
    return err == cudaSuccess ? MOE_OK : cuda_error(err, "fp8_plan_kernel");
}

// BF16 output rows (cols % 8 == 0), stored 32 rows by 64 columns at a time.
int out_map(CUtensorMap *m, const void *base, int rows, int cols) {
    const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
    const uint64_t str[1] = {static_cast<uint64_t>(cols) * 2};
    return make_map_bf16(m, base, 2, dims, str, 32);
}

std::atomic<uint64_t> g_wait_ns{2000000000ull};

}  // namespace

uint64_t fp8_wait_limit(uint64_t ns) { return g_wait_ns.exchange(ns, std::memory_order_relaxed); }

// The least of a few estimates, in microseconds, fitted to graph replays on a
// B200 (weights of 1024 x 2048, 1000 x 1040, 2048 x 512, 4096 x 4096, 8192 x
// 8192 and 512 x 8192, 1 to 512 rows; off by a fifth at most):
//  - tiles: 5.5, plus a group's time for every group in a CTA's row of items, plus
//    what the tile's epilogue and, with a split, the cluster's sum take; and no
//    less than the tiles' traffic at 9 TB/s from L2.  Clusters of eight are
//    limited to eight of them: sixteen do not all fit at once.
//  - a warp per weight row, up to four rows of x: 4.2 plus the longest of the
//    multiplications, the weights from HBM, and a warp's chain of loads.
// At 77 rows of 1040 against 1000: tiles of 16 in one piece 9.1, of 128 12.7; at
// 64 of 8192 against 512: tiles of 16 split eight ways 11.1, of 64 in one piece
// 38.3; at 16 of 512 against 2048: in one piece 6.5, split in two 8.6.
LinearFp8Plan plan_linear_fp8(int tokens, int rows, int cols) {
    constexpr int kTiles[4] = {16, 32, 64, kBM};
    constexpr double kGroupUs[4] = {0.33, 0.36, 0.45, 0.55}, kEndUs[4] = {0, 0.4, 1.6, 1.7},
                     kSplitUs[4] = {2.8, 2.9, 3.3, 4.5};
    constexpr int kMostCtas[4] = {148, 148, 128, 64};  // of a split 1, 2, 4, 8
    const double kbs = fp8::groups(cols), nt = (rows + kBN - 1) / kBN;
    LinearFp8Plan best{kBM, 1, false, false};
    double least = 1e300;
    for (int i = 0; i < 4; ++i) {
        const double items = nt * ((tokens + kTiles[i] - 1) / kTiles[i]);
        const double floor = items * kbs * kGroup * (kBN + kTiles[i]) / 9e6;
        for (int p = 0; p < 4; ++p) {
            const int split = 1 << p;
            if (p && (kbs < 2 * split || items * split > kMostCtas[p])) break;
            const double waves = std::ceil(items * split / 148);
            const double us = std::max(floor, waves * std::ceil(kbs / split) * kGroupUs[i]) + 5.5 +
                              (p ? kSplitUs[i] : kEndUs[i]);
            if (us < least) {
                least = us;
                best = LinearFp8Plan{kTiles[i], split, false, false};
            }
        }
    }
    if (tokens <= kGemvTokens) {
        const double macs = static_cast<double>(rows) * cols;
        const double us = 4.2 + std::max(std::max(macs * tokens * 1.05e-7, macs / 6.4e6),
                                         cols / 2048.0 * (0.5 + 0.45 * tokens));
        best.gemv = us < least;
    }
    // Pairs where they need no more rounds than single CTAs (an odd number of
    // row tiles leaves half a pair idle: 1152 rows of 4096 against 4096 are one
    // round of 144 tiles in 22.1 us, and two of 80 pairs in 37.6; 3456 of 2048 three
    // in 32.0 and four in 39.9) and each CTA has at least 64 groups to go through.
    // The cycles of a group are the same, the power and the traffic are not
    // (8192 rows of 2048 against 4096: 75.6 us single, 72.5 in pairs, 90.6 and 87.3
    // in a run of seconds at 1000 W; 8192 of 8192 against 8192: 686 and 659), but a
    // pair takes 0.4 to 0.8 us longer to start and end (512 rows of 512 against
    // 9216: 7.1 single, 7.9 in pairs; from 64 groups on 0.95 to 1.016 of single).
    if (!best.gemv && best.tile == kBM && best.split == 1 && tokens > kBM && grouped_pair_clusters() > 0) {
        const double single = std::ceil(nt * std::ceil(tokens / (1.0 * kBM)) / sm_count());
        const double paired = std::ceil(nt * std::ceil(tokens / (2.0 * kBM)) / grouped_pair_clusters());
        best.pair = paired <= single && paired * kbs >= 64;
    }
    return best;
}

int launch_linear_fp8_tiles(const LinearFp8 &a, int32_t *status, cudaStream_t stream) {
    const LinearFp8Plan plan = plan_linear_fp8(a.tokens, a.rows, a.cols);
    const int tile = plan.tile, bn = tile == kBM ? 0 : tile;
    CUtensorMap m[6]{};
    if (int rc = row_maps(&m[1], &m[2], a.x, a.tokens, a.cols, tile)) return rc;
    m[0] = m[1];
    const uint64_t dims[2] = {static_cast<uint64_t>(a.cols), static_cast<uint64_t>(a.rows)};
    const uint64_t str[1] = {static_cast<uint64_t>(a.cols)};
    if (int rc = make_map_u8(&m[3], a.w, 2, dims, str, 128)) return rc;
    m[4] = m[3];
    m[5] = m[3];
    if (!a.out_f32 && a.rows % 8 == 0)
        if (int rc = out_map(&m[5], a.out, a.tokens, a.rows)) return rc;
    Params P{};
    P.x_scales = a.x_scales;
    P.w_scales = a.w_scales;
    P.rows = a.tokens;
    P.n = a.rows;
    P.k = a.cols;
    P.out = a.out;
    P.out_f32 = a.out_f32;
    P.status = status;
    P.wait_ns = g_wait_ns.load(std::memory_order_relaxed);
    P.split = plan.split;
    P.pair = plan.pair;
    const int item_rows = plan.pair ? 2 * tile : tile;
    const int64_t items = static_cast<int64_t>((a.tokens + item_rows - 1) / item_rows) * ((a.rows + kBN - 1) / kBN);
    LRB_REQUIRE(items < (1ll << 31), "moe_linear_fp8: too many tiles");
    switch (bn) {
        case 16: return launch_tile<true, 16>(m, P, items, stream);
        case 32: return launch_tile<true, 32>(m, P, items, stream);
        case 64: return launch_tile<true, 64>(m, P, items, stream);
        default: return launch_tile<true, 0>(m, P, items, stream);
    }
}

// The row tile by the average rows of an expert (256 experts of 2048 x 512,
// top-8, us at 96 / 256 / 384 / 512 / 768 / 896 / 1024 tokens, so 3 / 8 / 12 /
// 16 / 24 / 28 / 32 rows: tiles of 16 140 / 150 / 156 / 168 / 210 / 227 / 246, of
// 32 144 / 152 / 148 / 152 / 164 / 172 / 188, rows as M 152 / 158 / 158 / 162 /
// 166 / 168 / 168; 128 experts of 2048 x 768 cross at the same places).
int experts_fp8_tile(int routes, int experts) {
    const int mean = routes / experts;
    return mean < 10 ? 16 : mean <= 24 ? 32 : 0;
}

// FP32 rows cost nothing beside the weights on small batches; above 2048 routes
// they are rounded to BF16, half the traffic of what then takes a tenth of the
// time (256 experts of 2048 x 512, top-8, at 300 / 1024 / 4096 / 8192 tokens: 135 /
// 156 / 294 / 538 us, with FP32 rows 145 / 167 / 344 / 644).  The output's error
// against 64 bits is then 0.0024 of its size instead of the 0.0017 of its own
// rounding to BF16; the BF16 layer rounds the same rows.
bool experts_fp8_wide_rows(int routes) { return routes <= kWideRoutes; }

int launch_experts_fp8_tiles(const ExpertsFp8 &a, const ExpertsFp8Scratch &s, int32_t *status, cudaStream_t stream) {
    const int routes = a.tokens * a.top_k;
    if (int rc = launch_plan(a, s, routes, stream)) return rc;
    const int bn = experts_fp8_tile(routes, a.experts);
    const int tile = bn ? bn : kBM;
    // at most one partial tile per expert beside the full ones
    const int64_t tiles = std::min<int64_t>(a.experts, routes) + routes / tile;
    const int64_t items = tiles * (a.inner / kGroup + (a.hidden + kBN - 1) / kBN);
    LRB_REQUIRE(items < (1ll << 31) - 65536, "moe_experts_fp8: too many tiles");
    CUtensorMap m[6]{};
    const uint64_t H = a.hidden, I = a.inner, E = a.experts, T = a.tokens;
    {
        // rows gathered four at a time: the map's box is one row
        const uint64_t dims[2] = {H, T}, str[1] = {H};
        if (int rc = make_map_u8(&m[0], a.x, 2, dims, str, 1)) return rc;
    }
    if (int rc = row_maps(&m[1], &m[2], s.act, routes, a.inner, tile)) return rc;
    const uint64_t d1[3] = {H, 2 * I, E}, s1[2] = {H, 2 * I * H}, d2[3] = {I, H, E}, s2[2] = {I, H * I};
    if (int rc = make_map_u8(&m[3], a.gate_up, 3, d1, s1, 128)) return rc;
    if (int rc = make_map_u8(&m[4], a.down, 3, d2, s2, 128)) return rc;
    m[5] = m[4];
    Params P{};
    P.x_scales = a.x_scales;
    P.w_scales = a.gate_up_scales;
    P.act_scales_in = s.act_scales;
    P.down_scales = a.down_scales;
    P.offsets = s.offsets;
    P.row_token = s.row_token;
    P.experts = a.experts;
    P.hidden = a.hidden;
    P.inner = a.inner;
    P.act = s.act;
    P.act_scales = s.act_scales;
    P.y = s.y;
    P.y_f32 = experts_fp8_wide_rows(routes);
    P.work = s.counters;
    P.done = s.counters + 1;
    P.gave_up = s.counters + 1 + a.experts;
    P.status = status;
    P.wait_ns = g_wait_ns.load(std::memory_order_relaxed);
    int rc = MOE_OK;
    switch (bn) {
        case 16: rc = launch_tile<false, 16>(m, P, items, stream); break;
        case 32: rc = launch_tile<false, 32>(m, P, items, stream); break;
        default: rc = launch_tile<false, 0>(m, P, items, stream); break;
    }
    if (rc) return rc;
    const int64_t ctas = (static_cast<int64_t>(a.tokens) * (a.hidden / (P.y_f32 ? 4 : 8)) + 127) / 128;
    const dim3 grid(static_cast<unsigned>(ctas)), block(128);
    const int32_t *pos = s.route_pos, *gave_up = P.gave_up;
    if (!P.y_f32)
        return launch_pdl(fp8_combine_kernel<uint16_t>, grid, block, 0, stream, "fp8_combine_kernel",
                          static_cast<const uint16_t *>(s.y), pos, a.weights, gave_up, a.tokens, a.top_k, a.hidden, a.out);
    return launch_pdl(fp8_combine_kernel<float>, grid, block, 0, stream, "fp8_combine_kernel",
                      static_cast<const float *>(s.y), pos, a.weights, gave_up, a.tokens, a.top_k, a.hidden, a.out);
}

}  // namespace lrb
