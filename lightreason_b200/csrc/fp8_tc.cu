// The FP8 products on the 5th-generation tensor cores: one persistent kernel
// for a plain product and for the two grouped products of the routed experts.
//
// Mathematics.  A tile is 128 rows (tokens, or routes of one expert) by 256
// weight rows.  Within a 128-column group g both scales are constants of the
// row and of the 128-row weight block, so
//   out[m, n] = sum_g  xs[m, g] * ws[n / 128, g] * (sum over the group of xq wq).
// tcgen05.mma (kind::f8f6f4) forms the inner sum of one group, four products of
// 32 columns, in one of two TMEM buffers of 256 columns; eight warps read it
// while the other buffer fills and add it, times the two scales, to FP32
// registers (128 a thread).  The scales are any FP32 values, so they cannot ride
// in the tensor core's own power-of-two block scales.
//
// Layout.  Rows are the M operand: a lane of the accumulator is one row, so a
// group's factor is one number per thread, gate and up of a column meet in one
// thread, and a partial tile's missing rows cost no epilogue work (whole warps
// skip).  A stage is one group: 256 weight rows (32 KB, two boxes) and the
// tile's rows (gathered by TMA from the token rows for gate/up, in boxes of 16
// when the tile is partial), three stages deep: 96 KB of weights in flight per
// SM, which is what streams the banks at small and middle widths, where the
// M = 128 products on padding are hidden under the weight stream.
//
// What bounds it at large widths: the four products of a group take 647 cycles
// of the tensor core, and reading the group's 128 KB of sums out of TMEM takes
// 228 more from it (both run alone at 647 and 385, together at 875 a group).
//
// Warps: 0 weight tiles, 1 MMA, 2 and 3 row tiles and scales (four groups at a
// time, up to four such requests in flight), 4-11 epilogue; the first four hand registers to the
// others (104 and 200 a thread of 168 at launch, 64,512 a CTA either way).
// Every wait is bounded; a timeout raises *status, drains what is in flight and
// returns.
#include <algorithm>

#include "fp8_kernels.cuh"
#include "sm100.cuh"

namespace lrb {
namespace {

using fp8::kGroup;

constexpr int kBM = 128, kBN = 256;
constexpr int kStages = 3;
constexpr int kATile = kBM * kGroup, kBTile = kBN * kGroup, kStage = kATile + kBTile;
constexpr int kThreads = 12 * 32;
constexpr int kScaleSlots = 4;   // of four groups each
constexpr int kPiece = 8192;     // an epilogue warp's output: 32 rows of 256 bytes
constexpr int kMaxExperts = 1024;
constexpr uint64_t kWaitNs = 2000000000ull;

enum Mode { kLinear, kGateUp, kDown };

struct Tail {
    float4 row_scale[kScaleSlots][kBM];
    float4 block_scale[kScaleSlots][2];
    float top[2][2][kBM];
    uint64_t full[kStages], empty[kStages], tfull[2], tempty[2], sfull[kScaleSlots], sempty[kScaleSlots], half[4],
        drain;
    int abort;
    uint32_t tmem;
    int32_t scan[16];
    int32_t items[kMaxExperts + 1];   // first item of each expert
};
constexpr int kSmem = kStages * kStage + 8 * kPiece + static_cast<int>(sizeof(Tail)) + 1024;
static_assert(kSmem <= 232448, "shared memory of one SM");

struct Params {
    const float *row_scales;      // [rows, groups]
    const float *block_scales;    // [(E,) blocks, groups]
    const int32_t *offsets;       // [E + 1] (experts)
    const int32_t *row_token;     // [R] route -> token (gate/up)
    int rows;                     // linear: T
    int n;                        // output columns: rows of w, I (gate/up), H (down)
    int k;                        // H, H, I
    int experts;
    void *out;                    // linear: [T, n]; down: BF16 [R, n]
    int out_f32;
    uint8_t *act;                 // gate/up: [R, I] e4m3
    float *act_scales;            // gate/up: [R, I / 128]
    int32_t *status;
};

__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
// Bounded wait; false once the CTA has given up.  Warps that work as one (the
// scales' and the epilogue's) do not leave on false: from then on their waits
// return at once and they run to the end on whatever is there, together.
// The clock (and the flag) are looked at every 256th poll only: reading the
// global timer takes longer than most waits.
__device__ __forceinline__ bool wait_bar(uint64_t *bar, uint32_t parity, volatile int *abort) {
    uint64_t t0 = 0;
    for (uint32_t i = 1; !sm100::mbar_try_wait(bar, parity); ++i) {
        if (i & 255) continue;
        if (*abort) return false;
        const uint64_t t = now_ns();
        if (t0 == 0) t0 = t;
        if (t - t0 > kWaitNs) {
            *abort = 1;
            return false;
        }
    }
    return true;
}

struct Item {
    int e, row0, count, n;  // expert, first row, rows (<= 128), column tile
    bool shared_tiles;      // other tiles read the same weight rows
};

template <int MODE>
__device__ __forceinline__ Item decode(const Params &P, const Tail *tail, int item) {
    Item r;
    if constexpr (MODE == kLinear) {
        const int mt = (P.rows + kBM - 1) / kBM;
        r.e = 0;
        r.n = item / mt;
        r.row0 = (item % mt) * kBM;
        r.count = min(kBM, P.rows - r.row0);
        r.shared_tiles = mt > 1;
    } else {
        int lo = 0, hi = P.experts;  // the expert with items[e] <= item < items[e + 1]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (tail->items[mid] <= item) lo = mid;
            else hi = mid;
        }
        const int begin = P.offsets[lo], count = P.offsets[lo + 1] - begin;
        const int mt = (count + kBM - 1) / kBM, at = item - tail->items[lo];
        r.e = lo;
        r.n = at / mt;
        const int m = at % mt;
        r.row0 = begin + m * kBM;
        r.count = min(kBM, count - m * kBM);
        r.shared_tiles = mt > 1;
    }
    return r;
}

template <int BYTES>
__device__ __forceinline__ void copy_async(void *dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(sm100::smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
}
// This thread arrives on `bar` once its copies so far are complete.
__device__ __forceinline__ void copy_async_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(sm100::smem_u32(bar)) : "memory");
}

// Completes this warp's TMEM loads; the values pass through, so no use of them
// can be moved before it.
__device__ __forceinline__ void wait_ld16(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
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

// x / (1 + exp(-x)) from the fast exponential and quotient: off by 2^-24 times
// (4 + 1.2 |x|) of the value at most, below what the FP32 sums behind x leave.
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

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_tile_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_x16,
                    const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_out,
                    const Params P) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *pieces = smem + kStages * kStage;
    Tail *tail = reinterpret_cast<Tail *>(pieces + 8 * kPiece);
    volatile int *abort = &tail->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            sm100::mbar_init(&tail->full[s], MODE == kGateUp ? 3 : 2);  // the warps that load into it
            sm100::mbar_init(&tail->empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            sm100::mbar_init(&tail->tfull[b], 1);
            sm100::mbar_init(&tail->tempty[b], 8);
        }
        for (int s = 0; s < kScaleSlots; ++s) {
            sm100::mbar_init(&tail->sfull[s], MODE == kGateUp ? 64 : 32);  // lanes
            sm100::mbar_init(&tail->sempty[s], 8);
        }
        for (int q = 0; q < 4; ++q) sm100::mbar_init(&tail->half[q], 2);
        sm100::mbar_init(&tail->drain, 1);
        tail->abort = 0;
        sm100::fence_barrier_init();
        sm100::tma_prefetch_map(&tm_x);
        sm100::tma_prefetch_map(&tm_w);
    }
    if (warp == 1) {
        sm100::tmem_alloc(&tail->tmem, 512);
        sm100::tmem_relinquish();
    }
    sm100::tc_fence_before();
    __syncthreads();
    sm100::tc_fence_after();
    const uint32_t tmem = tail->tmem;
    grid_dependency_wait();
    grid_dependency_trigger();

    const int kbs = fp8::groups(P.k);
    const int nt = MODE == kGateUp ? P.n / kGroup : (P.n + kBN - 1) / kBN;
    int total;
    if constexpr (MODE == kLinear) {
        total = nt * ((P.rows + kBM - 1) / kBM);
    } else {
        // items[e]: an exclusive scan of the experts' tile counts, a few
        // neighbouring experts a thread
        constexpr int kPer = (kMaxExperts + kThreads) / kThreads;
        int tiles[kPer], sum = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = threadIdx.x * kPer + i;
            tiles[i] = e < P.experts ? nt * ((P.offsets[e + 1] - P.offsets[e] + kBM - 1) / kBM) : 0;
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
            if (e <= P.experts) tail->items[e] = at;
            at += tiles[i];
        }
        __syncthreads();
        total = tail->items[P.experts];
    }

    if (warp < 4) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
      if (warp == 0) {
        // ------------------------------------------------------ weight tiles
        const uint64_t once = sm100::l2_evict_first_policy(), keep = sm100::l2_evict_normal_policy();
        const bool one = sm100::elect_one();
        uint32_t stage = 0, phase = 0;
        bool ok = true;
        for (int item = blockIdx.x; ok && item < total; item += gridDim.x) {
            const Item it = decode<MODE>(P, tail, item);
            const uint64_t policy = it.shared_tiles ? keep : once;
            for (int kb = 0; kb < kbs; ++kb) {
                ok = __all_sync(0xffffffffu, wait_bar(&tail->empty[stage], phase ^ 1, abort));
                if (!ok) break;
                uint8_t *b = smem + stage * kStage + kATile;
                uint64_t *bar = &tail->full[stage];
                const int r0 = MODE == kGateUp ? it.n * kGroup : it.n * kBN;
                const int r1 = MODE == kGateUp ? P.n + r0 : r0 + 128;
                if (one) {
                    sm100::mbar_expect_tx(bar, kBTile);
                    if constexpr (MODE == kLinear) {
                        sm100::tma_load_2d_hint(b, &tm_w, bar, kb * kGroup, r0, policy);
                        sm100::tma_load_2d_hint(b + kBTile / 2, &tm_w, bar, kb * kGroup, r1, policy);
                    } else {
                        sm100::tma_load_3d_hint(b, &tm_w, bar, kb * kGroup, r0, it.e, policy);
                        sm100::tma_load_3d_hint(b + kBTile / 2, &tm_w, bar, kb * kGroup, r1, it.e, policy);
                    }
                }
                __syncwarp();
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
      } else if (warp >= 2) {
        // --------------------------------------------- row tiles and scales
        // gate/up: warp 2 has the tile's first 64 rows, warp 3 the others, four
        // rows a lane: gathered one instruction a lane (they issue one after
        // another, so two warps halve that time), and the lanes' scales.
        // Otherwise warp 2 loads the rows (one box, or 16-row boxes one a
        // lane) and warp 3 all scales, four rows a lane.
        constexpr bool kGather = MODE == kGateUp;
        const bool loads = kGather || warp == 2, scales = kGather || warp == 3;
        const int r0 = kGather ? 64 * (warp - 2) + 4 * lane : 4 * lane;
        const bool mine = !kGather || lane < 16;
        sm100::fence_proxy_async_global();
        uint32_t stage = 0, phase = 0, slot = 0, sphase = 0;
        auto rows_of = [&](const Item &it, int (&row)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = it.row0 + min(r0 + i, it.count - 1);
                row[i] = kGather ? P.row_token[r] : r;
            }
        };
        const bool quads = kbs % 4 == 0 && (reinterpret_cast<uintptr_t>(P.row_scales) & 15) == 0 &&
                           (reinterpret_cast<uintptr_t>(P.block_scales) & 15) == 0;
        // the scales of groups kb .. kb + 3 to `slot`, on their way when this
        // returns: up to kScaleSlots such requests are in flight
        auto copy4 = [&](float4 *dst, const float *src, int kb) {
            if (quads) {
                copy_async<16>(dst, src + kb);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (kb + i < kbs) copy_async<4>(reinterpret_cast<float *>(dst) + i, src + kb + i);
            }
        };
        auto request_scales = [&](const Item &it, const int (&row)[4], int kb) {
            if (mine) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    copy4(&tail->row_scale[slot][r0 + i], P.row_scales + static_cast<int64_t>(row[i]) * kbs, kb);
            }
            // lanes 0 and 1: the item's two weight blocks (gate and up, or the
            // two halves of the columns; one past the matrix is never used)
            if (warp == 3 && lane < 2) {
                int64_t blk;
                if constexpr (MODE == kGateUp) {
                    blk = static_cast<int64_t>(it.e) * 2 * nt + it.n + lane * nt;
                } else {
                    const int per = fp8::groups(P.n);
                    blk = static_cast<int64_t>(it.e) * per + min(2 * it.n + lane, per - 1);
                }
                copy4(&tail->block_scale[slot][lane], P.block_scales + blk * kbs, kb);
            }
            copy_async_arrive(&tail->sfull[slot]);
        };
        int item = blockIdx.x;
        Item next{};
        int next_row[4] = {};
        if (item < total) {
            next = decode<MODE>(P, tail, item);
            rows_of(next, next_row);
        }
        bool ok = true;
        for (; ok && item < total; item += gridDim.x) {
            const Item it = next;
            int row[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) row[i] = next_row[i];
            const bool more = item + static_cast<int>(gridDim.x) < total;
            if (more) {
                next = decode<MODE>(P, tail, item + gridDim.x);
                rows_of(next, next_row);
            }
            // lanes that load, and what a lane loads
            const int boxes = kGather ? min(16, (max(0, it.count - 64 * (warp - 2)) + 3) / 4)
                                      : it.count == kBM ? 1 : (it.count + 15) / 16;
            const int box_bytes = kGather ? 4 * kGroup : it.count == kBM ? kATile : 16 * kGroup;
            for (int kb = 0; kb < kbs; ++kb) {
                if (scales && (kb & 3) == 0) {
                    ok = __all_sync(0xffffffffu, wait_bar(&tail->sempty[slot], sphase ^ 1, abort));
                    if (!ok) break;
                    request_scales(it, row, kb);
                    if (++slot == kScaleSlots) {
                        slot = 0;
                        sphase ^= 1;
                    }
                }
                if (!loads) continue;
                ok = __all_sync(0xffffffffu, wait_bar(&tail->empty[stage], phase ^ 1, abort));
                if (!ok) break;
                uint8_t *a = smem + stage * kStage;
                uint64_t *bar = &tail->full[stage];
                if (lane == 0) sm100::mbar_expect_tx(bar, boxes * box_bytes);
                __syncwarp();
                if (lane < boxes) {
                    if constexpr (kGather)
                        sm100::tma_gather4(a + (r0 - 4 * lane) * kGroup + lane * box_bytes, &tm_x, bar, kb * kGroup,
                                           row);
                    else
                        sm100::tma_load_2d(a + lane * box_bytes, it.count == kBM ? &tm_x : &tm_x16, bar, kb * kGroup,
                                           it.row0 + lane * 16);
                }
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
      } else if (warp == 1) {
        // --------------------------------------------------------- MMA issuer
        constexpr uint32_t idesc = sm100::idesc_e4m3_f32(kBM, kBN);
        const bool one = sm100::elect_one();
        uint32_t stage = 0, phase = 0, buf = 0, bphase = 0;
        bool ok = true, any = false;
        for (int item = blockIdx.x; ok && item < total; item += gridDim.x) {
            for (int kb = 0; kb < kbs; ++kb) {
                ok = wait_bar(&tail->tempty[buf], bphase ^ 1, abort) && wait_bar(&tail->full[stage], phase, abort);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                sm100::tc_fence_after();
                const uint32_t base = sm100::smem_u32(smem + stage * kStage), d = tmem + buf * kBN;
                const uint64_t a = sm100::desc_kmajor_sw128(base), b = sm100::desc_kmajor_sw128(base + kATile);
                if (one) {
                    sm100::mma_e4m3<false>(d, a, b, idesc);
                    sm100::mma_e4m3<true>(d, a + 2, b + 2, idesc);
                    sm100::mma_e4m3<true>(d, a + 4, b + 4, idesc);
                    sm100::mma_e4m3<true>(d, a + 6, b + 6, idesc);
                    sm100::mma_commit(&tail->tfull[buf]);
                    sm100::mma_commit(&tail->empty[stage]);
                }
                __syncwarp();
                any = true;
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
                buf ^= 1;
                bphase ^= buf == 0;
            }
        }
        if (*abort && any) {
            if (one) sm100::mma_commit(&tail->drain);
            const uint64_t t0 = now_ns();
            while (!sm100::mbar_try_wait(&tail->drain, 0) && now_ns() - t0 < kWaitNs) {
            }
        }
        __syncwarp();
      }
    } else {
        // ----------------------------------------------------------- epilogue
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const int q = warp & 3, h = warp >= 8;  // TMEM lanes 32q.., half of the columns
        const int r = 32 * q + lane;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * q) << 16);
        uint8_t *piece = pieces + (warp - 4) * kPiece;
        uint32_t slot = 0, sphase = 0, buf = 0, bphase = 0, iphase = 0;
        // the factors of the next four groups: row scale x weight scale (gate's and up's)
        float s0[4], s1[4];
        auto take_scales = [&] {
            wait_bar(&tail->sfull[slot], sphase, abort);
            const float4 rs = tail->row_scale[slot][r];
            const float4 b0 = tail->block_scale[slot][MODE == kGateUp ? 0 : h];
            s0[0] = rs.x * b0.x, s0[1] = rs.y * b0.y, s0[2] = rs.z * b0.z, s0[3] = rs.w * b0.w;
            if constexpr (MODE == kGateUp) {
                const float4 b1 = tail->block_scale[slot][1];
                s1[0] = rs.x * b1.x, s1[1] = rs.y * b1.y, s1[2] = rs.z * b1.z, s1[3] = rs.w * b1.w;
            }
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(&tail->sempty[slot]);
            if (++slot == kScaleSlots) {
                slot = 0;
                sphase ^= 1;
            }
        };
        for (int item = blockIdx.x; item < total; item += gridDim.x) {
            const Item it = decode<MODE>(P, tail, item);
            const bool active = 32 * q < it.count;  // the warp has rows of the tile
            float acc[128];
#pragma unroll
            for (int i = 0; i < 128; ++i) acc[i] = 0.f;
            take_scales();
            for (int kb = 0; kb < kbs; ++kb) {
                const float g0 = s0[0], g1 = MODE == kGateUp ? s1[0] : s0[0];
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    s0[i] = s0[i + 1];
                    if (MODE == kGateUp) s1[i] = s1[i + 1];
                }
                const bool refill = (kb & 3) == 3 && kb + 1 < kbs;
                wait_bar(&tail->tfull[buf], bphase, abort);
                sm100::tc_fence_after();
                if (active) {
                    // 16 columns at a time; gate/up: 64 of the gate block, then
                    // the same 64 of the up block
                    const uint32_t base = lanes + buf * kBN;
                    auto col = [&](int c) {
                        return MODE == kGateUp ? base + 64 * h + 16 * (c & 3) + (c >= 4 ? 128 : 0)
                                               : base + 128 * h + 16 * c;
                    };
                    float t[2][16];
                    sm100::tmem_ld16(col(0), t[0]);
                    if (refill) take_scales();
                    wait_ld16(t[0]);
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        if (c < 7) sm100::tmem_ld16(col(c + 1), t[(c + 1) & 1]);
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            acc[16 * c + i] = fmaf(t[c & 1][i], c < 4 ? g0 : g1, acc[16 * c + i]);
                        if (c < 7) wait_ld16(t[(c + 1) & 1]);
                    }
                } else if (refill) {
                    take_scales();
                }
                sm100::tc_fence_before();
                __syncwarp();
                if (lane == 0) sm100::mbar_arrive(&tail->tempty[buf]);
                buf ^= 1;
                bphase ^= buf == 0;
            }
            if (!active) continue;
            const int rows = it.count - 32 * q;  // of this warp, if below 32
            const int64_t first = static_cast<int64_t>(it.row0) + 32 * q;
            if constexpr (MODE == kGateUp) {
                float top = fp8::kTiny;
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    acc[i] = silu_fast(acc[i]) * acc[64 + i];
                    top = fp8::max_nan(top, fabsf(acc[i]));
                }
                // the group's other 64 columns are the other half's
                tail->top[iphase][h][r] = top;
                __syncwarp();
                if (lane == 0) sm100::mbar_arrive(&tail->half[q]);
                wait_bar(&tail->half[q], iphase, abort);
                top = fp8::max_nan(top, tail->top[iphase][h ^ 1][r]);
                iphase ^= 1;
                const fp8::Divisor f(top);
                uint32_t v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    v[i] = fp8::pack4(f, acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
                store_rows64(piece, v, P.act + first * P.n + it.n * kGroup + 64 * h, P.n, rows, 4);
                if (h == 0 && lane < rows) P.act_scales[(first + lane) * nt + it.n] = fp8::scale_of(top);
            } else {
                const int n0 = it.n * kBN + 128 * h;
                const bool f32 = MODE == kLinear && P.out_f32;
                // whole 16-byte units: 8 BF16 or 4 FP32 columns, all or none of
                // them there (the down product's H is a multiple of 16)
                const bool vec = MODE == kDown || P.n % (f32 ? 4 : 8) == 0;
                if (vec && !f32 && (MODE == kLinear || rows >= 32)) {
                    // The map cuts rows and columns past the matrix; another
                    // expert's rows below a partial tile must not be written,
                    // so those take the other way.
                    if (lane == 0) sm100::bulk_wait_read();  // the last item's stores have left the buffer
                    __syncwarp();
                    stage_row256(piece, acc);
                    sm100::fence_proxy_async_shared();
                    __syncwarp();
                    if (lane == 0) {
                        if (n0 < P.n) sm100::tma_store_2d(piece, &tm_out, n0, static_cast<int>(first));
                        if (n0 + 64 < P.n) sm100::tma_store_2d(piece + 4096, &tm_out, n0 + 64, static_cast<int>(first));
                        sm100::bulk_commit();
                    }
                } else if (vec && !f32) {
                    if (lane == 0) sm100::bulk_wait_read();
                    uint16_t *dst = static_cast<uint16_t *>(P.out) + first * P.n + n0;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t v[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = fp8::pack_bf16(acc[32 * c + 2 * i], acc[32 * c + 2 * i + 1]);
                        store_rows64(piece + 2048 * c, v, reinterpret_cast<uint8_t *>(dst + 32 * c),
                                     2 * static_cast<int64_t>(P.n), rows, (P.n - n0 - 32 * c) / 8);
                    }
                } else if (vec) {
                    float *dst = static_cast<float *>(P.out) + first * P.n + n0;
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        uint32_t v[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(acc[16 * c + i]);
                        store_rows64(piece + 2048 * (c & 3), v, reinterpret_cast<uint8_t *>(dst + 16 * c),
                                     4 * static_cast<int64_t>(P.n), rows, (P.n - n0 - 16 * c) / 4);
                    }
                } else if (lane < rows) {
                    const int64_t at = (first + lane) * P.n + n0;
#pragma unroll
                    for (int i = 0; i < 128; ++i) {
                        if (n0 + i >= P.n) continue;
                        if (f32) static_cast<float *>(P.out)[at + i] = acc[i];
                        else static_cast<uint16_t *>(P.out)[at + i] = f2bf(acc[i]);
                    }
                }
            }
        }
        if (lane == 0) sm100::bulk_wait_all();
        __syncwarp();
        sm100::tc_fence_before();
    }
    if (*abort && warp < 4) {
        // loads may be in flight whose barriers will never complete: give them
        // a time far above any load's before the CTA leaves
        const uint64_t t0 = now_ns();
        while (now_ns() - t0 < 200000) __nanosleep(1000);
    }
    __syncthreads();
    if (warp == 1) {
        sm100::tc_fence_after();
        sm100::tmem_dealloc(tmem, 512);
    }
    if (threadIdx.x == 0 && *abort && P.status) atomicExch(P.status, 1);
}

// out[t] = sum over the token's routes, in slot order, of weight * row, in
// FP32.  A thread per 8 columns of a token, eight rows in flight.
__global__ void __launch_bounds__(256) fp8_combine_kernel(const uint16_t *__restrict__ y,
                                                          const int32_t *__restrict__ route_pos,
                                                          const uint16_t *__restrict__ weights, int tokens, int top_k,
                                                          int hidden, uint16_t *__restrict__ out) {
    grid_dependency_wait();
    grid_dependency_trigger();
    const int units = hidden / 8;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t t = i / units;
    if (t >= tokens) return;
    const int c = static_cast<int>(i % units) * 8;
    float acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.f;
    for (int k0 = 0; k0 < top_k; k0 += 8) {
        uint4 v[8];
        float w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t at = t * top_k + k0 + k;
            const int p = k0 + k < top_k ? route_pos[at] : -1;
            w[k] = p >= 0 ? bf2f(weights[at]) : 0.f;
            v[k] = p >= 0 ? ld_stream(y + static_cast<int64_t>(p) * hidden + c) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[2 * j] = fmaf(bf16_lo(u[j]), w[k], acc[2 * j]);
                acc[2 * j + 1] = fmaf(bf16_hi(u[j]), w[k], acc[2 * j + 1]);
            }
        }
    }
    *reinterpret_cast<uint4 *>(out + t * hidden + c) =
        make_uint4(fp8::pack_bf16(acc[0], acc[1]), fp8::pack_bf16(acc[2], acc[3]), fp8::pack_bf16(acc[4], acc[5]),
                   fp8::pack_bf16(acc[6], acc[7]));
}

template <int MODE>
int launch_tile(const CUtensorMap &x, const CUtensorMap &x16, const CUtensorMap &w, const CUtensorMap &out,
                const Params &P, int64_t items, cudaStream_t stream) {
    if (int rc = ensure_dynamic_smem(fp8_tile_kernel<MODE>, kSmem, "cudaFuncSetAttribute(fp8_tile)")) return rc;
    return launch_pdl(fp8_tile_kernel<MODE>, dim3(static_cast<unsigned>(std::min<int64_t>(items, sm_count()))),
                      dim3(kThreads), kSmem, stream, "fp8_tile_kernel", x, x16, w, out, P);
}

int row_maps(CUtensorMap *m, CUtensorMap *m16, const void *base, int rows, int cols) {
    const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
    const uint64_t str[1] = {static_cast<uint64_t>(cols)};
    if (int rc = make_map_u8(m, base, 2, dims, str, kBM)) return rc;
    return make_map_u8(m16, base, 2, dims, str, 16);
}

// BF16 output rows (cols % 8 == 0), stored 32 rows by 64 columns at a time.
int out_map(CUtensorMap *m, const void *base, int rows, int cols) {
    const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
    const uint64_t str[1] = {static_cast<uint64_t>(cols) * 2};
    return make_map_bf16(m, base, 2, dims, str, 32);
}

}  // namespace

int launch_linear_fp8_tiles(const LinearFp8 &a, int32_t *status, cudaStream_t stream) {
    CUtensorMap x{}, x16{}, w{}, out{};
    if (int rc = row_maps(&x, &x16, a.x, a.tokens, a.cols)) return rc;
    const uint64_t dims[2] = {static_cast<uint64_t>(a.cols), static_cast<uint64_t>(a.rows)};
    const uint64_t str[1] = {static_cast<uint64_t>(a.cols)};
    if (int rc = make_map_u8(&w, a.w, 2, dims, str, 128)) return rc;
    if (!a.out_f32 && a.rows % 8 == 0)
        if (int rc = out_map(&out, a.out, a.tokens, a.rows)) return rc;
    Params P{};
    P.row_scales = a.x_scales;
    P.block_scales = a.w_scales;
    P.rows = a.tokens;
    P.n = a.rows;
    P.k = a.cols;
    P.out = a.out;
    P.out_f32 = a.out_f32;
    P.status = status;
    const int64_t items = static_cast<int64_t>((a.tokens + kBM - 1) / kBM) * ((a.rows + kBN - 1) / kBN);
    LRB_REQUIRE(items < (1ll << 31), "moe_linear_fp8: too many tiles");
    return launch_tile<kLinear>(x, x16, w, out, P, items, stream);
}

int launch_experts_fp8_tiles(const ExpertsFp8 &a, const ExpertsFp8Scratch &s, int32_t *status, cudaStream_t stream) {
    const int routes = a.tokens * a.top_k;
    if (int rc = launch_permute(a.idx, a.tokens, a.top_k, a.experts, s.offsets, s.perm_token, s.perm_slot, s.route_pos,
                                s.active, s.counters, s.counters + 1, stream, s.hist))
        return rc;
    // at most one partial tile per expert beside the full ones
    const int64_t tiles = std::min<int64_t>(a.experts, routes) + routes / kBM;
    const int64_t nt1 = a.inner / kGroup, nt2 = (a.hidden + kBN - 1) / kBN;
    LRB_REQUIRE(tiles * std::max(nt1, nt2) < (1ll << 31), "moe_experts_fp8: too many tiles");
    CUtensorMap x{}, act{}, act16{}, gu{}, dn{}, y{};
    {
        // rows gathered four at a time: the map's box is one row
        const uint64_t dims[2] = {static_cast<uint64_t>(a.hidden), static_cast<uint64_t>(a.tokens)};
        const uint64_t str[1] = {static_cast<uint64_t>(a.hidden)};
        if (int rc = make_map_u8(&x, a.x, 2, dims, str, 1)) return rc;
    }
    if (int rc = row_maps(&act, &act16, s.act, routes, a.inner)) return rc;
    if (int rc = out_map(&y, s.y, routes, a.hidden)) return rc;
    {
        const uint64_t H = a.hidden, I = a.inner, E = a.experts;
        const uint64_t d1[3] = {H, 2 * I, E}, s1[2] = {H, 2 * I * H}, d2[3] = {I, H, E}, s2[2] = {I, H * I};
        if (int rc = make_map_u8(&gu, a.gate_up, 3, d1, s1, 128)) return rc;
        if (int rc = make_map_u8(&dn, a.down, 3, d2, s2, 128)) return rc;
    }
    Params P{};
    P.offsets = s.offsets;
    P.experts = a.experts;
    P.status = status;
    Params G = P;
    G.row_scales = a.x_scales;
    G.block_scales = a.gate_up_scales;
    G.row_token = s.perm_token;
    G.n = a.inner;
    G.k = a.hidden;
    G.act = s.act;
    G.act_scales = s.act_scales;
    if (int rc = launch_tile<kGateUp>(x, x, gu, y, G, tiles * nt1, stream)) return rc;
    P.row_scales = s.act_scales;
    P.block_scales = a.down_scales;
    P.n = a.hidden;
    P.k = a.inner;
    P.out = s.y;
    if (int rc = launch_tile<kDown>(act, act16, dn, y, P, tiles * nt2, stream)) return rc;
    const int64_t ctas = (static_cast<int64_t>(a.tokens) * (a.hidden / 8) + 255) / 256;
    return launch_pdl(fp8_combine_kernel, dim3(static_cast<unsigned>(ctas)), dim3(256), 0, stream,
                      "fp8_combine_kernel", static_cast<const uint16_t *>(s.y),
                      static_cast<const int32_t *>(s.route_pos), a.weights, a.tokens, a.top_k, a.hidden, a.out);
}

}  // namespace lrb
