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
// when the tile is partial), four stages deep: 128 KB of weights in flight per
// SM, which is what streams the banks at small and middle widths, where the
// M = 128 products on padding are hidden under the weight stream.
//
// Warps: 0 TMA, 1 MMA, 2 the scales (a ring of eight groups in shared memory,
// so that no epilogue thread waits for a scale), 3-10 epilogue.  Every wait is
// bounded; a timeout raises *status, drains what is in flight and returns.
#include <algorithm>

#include "fp8_kernels.cuh"
#include "sm100.cuh"

namespace lrb {
namespace {

using fp8::kGroup;

constexpr int kBM = 128, kBN = 256;
constexpr int kStages = 4;
constexpr int kATile = kBM * kGroup, kBTile = kBN * kGroup, kStage = kATile + kBTile;
constexpr int kThreads = 11 * 32;
constexpr int kScaleSlots = 8;
constexpr int kMaxExperts = 1024;
constexpr uint64_t kWaitNs = 2000000000ull;

enum Mode { kLinear, kGateUp, kDown };

struct Tail {
    uint64_t full[kStages], empty[kStages], tfull[2], tempty[2], sfull[kScaleSlots], sempty[kScaleSlots], half[4],
        drain;
    float row_scale[kScaleSlots][kBM];
    float block_scale[kScaleSlots][2];
    float top[2][2][kBM];
    int abort;
    uint32_t tmem;
    int32_t scan[16];
    int32_t items[kMaxExperts + 1];   // first item of each expert
    int32_t offsets[kMaxExperts + 1];  // first route of each expert
};
constexpr int kSmem = kStages * kStage + static_cast<int>(sizeof(Tail)) + 1024;

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
__device__ __forceinline__ bool wait_bar(uint64_t *bar, uint32_t parity, volatile int *abort) {
    if (sm100::mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = now_ns();
    for (uint32_t i = 1;; ++i) {
        if (sm100::mbar_try_wait(bar, parity)) return true;
        if (*abort) return false;
        if ((i & 63) == 0 && now_ns() - t0 > kWaitNs) {
            *abort = 1;
            return false;
        }
    }
}
// The same for a whole warp: every lane gets one answer.
__device__ __forceinline__ bool wait_warp(uint64_t *bar, uint32_t parity, volatile int *abort) {
    return __all_sync(0xffffffffu, wait_bar(bar, parity, abort));
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
        const int begin = tail->offsets[lo], count = tail->offsets[lo + 1] - begin;
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

// Completes this warp's TMEM loads; the values pass through, so no use of them
// can be moved before it.
__device__ __forceinline__ void wait_ld16(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
                 :
                 : "memory");
}

__device__ __forceinline__ void store32(void *p, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_tile_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_x16,
                    const __grid_constant__ CUtensorMap tm_w, const Params P) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Tail *tail = reinterpret_cast<Tail *>(smem + kStages * kStage);
    volatile int *abort = &tail->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            sm100::mbar_init(&tail->full[s], 1);
            sm100::mbar_init(&tail->empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            sm100::mbar_init(&tail->tfull[b], 1);
            sm100::mbar_init(&tail->tempty[b], 8);
        }
        for (int s = 0; s < kScaleSlots; ++s) {
            sm100::mbar_init(&tail->sfull[s], 1);
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
        // items[e]: an exclusive scan of the experts' tile counts, three
        // neighbouring experts a thread
        constexpr int kPer = (kMaxExperts + kThreads - 1) / kThreads;
        int tiles[kPer], sum = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = threadIdx.x * kPer + i;
            tiles[i] = 0;
            if (e < P.experts) {
                const int begin = P.offsets[e], end = P.offsets[e + 1];
                tail->offsets[e] = begin;
                if (e == P.experts - 1) tail->offsets[P.experts] = end;
                tiles[i] = nt * ((end - begin + kBM - 1) / kBM);
            }
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

    if (warp == 0) {
        // ------------------------------------------------------ TMA producer
        sm100::fence_proxy_async_global();
        const uint64_t once = sm100::l2_evict_first_policy(), keep = sm100::l2_evict_normal_policy();
        uint32_t stage = 0, phase = 0;
        uint32_t issued = 0, parity = 0;  // bit per stage
        bool ok = true;
        for (int item = blockIdx.x; ok && item < total; item += gridDim.x) {
            const Item it = decode<MODE>(P, tail, item);
            int tok[4];
            if constexpr (MODE == kGateUp) {
#pragma unroll
                for (int i = 0; i < 4; ++i) tok[i] = P.row_token[it.row0 + min(4 * lane + i, it.count - 1)];
            }
            // lanes that load: four rows each (gathered), or a box each
            const int boxes = MODE == kGateUp ? (it.count + 3) / 4 : it.count == kBM ? 1 : (it.count + 15) / 16;
            const int box_bytes = MODE == kGateUp ? 4 * kGroup : it.count == kBM ? kATile : 16 * kGroup;
            const uint64_t policy = it.shared_tiles ? keep : once;
            for (int kb = 0; kb < kbs; ++kb) {
                if (!wait_warp(&tail->empty[stage], phase ^ 1, abort)) {
                    ok = false;
                    break;
                }
                uint8_t *a = smem + stage * kStage, *b = a + kATile;
                uint64_t *bar = &tail->full[stage];
                if (lane == 0) {
                    sm100::mbar_expect_tx(bar, kBTile + boxes * box_bytes);
                    if constexpr (MODE == kLinear) {
                        sm100::tma_load_2d_hint(b, &tm_w, bar, kb * kGroup, it.n * kBN, policy);
                        sm100::tma_load_2d_hint(b + kBTile / 2, &tm_w, bar, kb * kGroup, it.n * kBN + 128, policy);
                    } else {
                        const int r0 = MODE == kGateUp ? it.n * kGroup : it.n * kBN;
                        const int r1 = MODE == kGateUp ? P.n + r0 : r0 + 128;
                        sm100::tma_load_3d_hint(b, &tm_w, bar, kb * kGroup, r0, it.e, policy);
                        sm100::tma_load_3d_hint(b + kBTile / 2, &tm_w, bar, kb * kGroup, r1, it.e, policy);
                    }
                }
                __syncwarp();
                if (lane < boxes) {
                    if constexpr (MODE == kGateUp)
                        sm100::tma_gather4(a + lane * box_bytes, &tm_x, bar, kb * kGroup, tok);
                    else
                        sm100::tma_load_2d(a + lane * box_bytes, it.count == kBM ? &tm_x : &tm_x16, bar, kb * kGroup,
                                           it.row0 + lane * 16);
                }
                issued |= 1u << stage;
                parity = (parity & ~(1u << stage)) | (phase << stage);
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
        if (*abort) {
            // let every load land before the CTA leaves
            for (int s = 0; s < kStages; ++s) {
                if (!(issued >> s & 1)) continue;
                const uint64_t t0 = now_ns();
                while (!sm100::mbar_try_wait(&tail->full[s], parity >> s & 1) && now_ns() - t0 < kWaitNs) {
                }
            }
        }
    } else if (warp == 1) {
        // --------------------------------------------------------- MMA issuer
        if (lane == 0) {
            constexpr uint32_t idesc = sm100::idesc_e4m3_f32(kBM, kBN);
            uint32_t stage = 0, phase = 0, buf = 0, bphase = 0;
            bool ok = true, any = false;
            for (int item = blockIdx.x; ok && item < total; item += gridDim.x) {
                for (int kb = 0; kb < kbs; ++kb) {
                    if (!wait_bar(&tail->tempty[buf], bphase ^ 1, abort) ||
                        !wait_bar(&tail->full[stage], phase, abort)) {
                        ok = false;
                        break;
                    }
                    sm100::tc_fence_after();
                    const uint32_t base = sm100::smem_u32(smem + stage * kStage);
                    const uint64_t a = sm100::desc_kmajor_sw128(base), b = sm100::desc_kmajor_sw128(base + kATile);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        sm100::mma_e4m3(tmem + buf * kBN, a + 2 * kk, b + 2 * kk, idesc, kk != 0);
                    sm100::mma_commit(&tail->empty[stage]);
                    sm100::mma_commit(&tail->tfull[buf]);
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
                sm100::mma_commit(&tail->drain);
                const uint64_t t0 = now_ns();
                while (!sm100::mbar_try_wait(&tail->drain, 0) && now_ns() - t0 < kWaitNs) {
                }
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        // ------------------------------------------------------------- scales
        uint32_t slot = 0, phase = 0;
        bool ok = true;
        for (int item = blockIdx.x; ok && item < total; item += gridDim.x) {
            const Item it = decode<MODE>(P, tail, item);
            const float *src[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = min(lane + 32 * j, it.count - 1);
                const int64_t row = MODE == kGateUp ? P.row_token[it.row0 + r] : it.row0 + r;
                src[j] = P.row_scales + row * kbs;
            }
            // lanes 0 and 1: the item's two weight blocks (gate and up, or the
            // two halves of the columns; one past the matrix is never used)
            const float *blk = nullptr;
            if (lane < 2) {
                if constexpr (MODE == kGateUp) {
                    blk = P.block_scales +
                          (static_cast<int64_t>(it.e) * 2 * nt + it.n + static_cast<int64_t>(lane) * nt) * kbs;
                } else {
                    const int per = fp8::groups(P.n);
                    blk = P.block_scales + (static_cast<int64_t>(it.e) * per + min(2 * it.n + lane, per - 1)) * kbs;
                }
            }
            for (int kb0 = 0; ok && kb0 < kbs; kb0 += 4) {
                float v[4][4], w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int kb = min(kb0 + i, kbs - 1);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[i][j] = src[j][kb];
                    w[i] = blk ? blk[kb] : 0.f;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (kb0 + i >= kbs) break;
                    if (!wait_warp(&tail->sempty[slot], phase ^ 1, abort)) {
                        ok = false;
                        break;
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) tail->row_scale[slot][lane + 32 * j] = v[i][j];
                    if (lane < 2) tail->block_scale[slot][lane] = w[i];
                    __syncwarp();
                    if (lane == 0) sm100::mbar_arrive(&tail->sfull[slot]);
                    if (++slot == kScaleSlots) {
                        slot = 0;
                        phase ^= 1;
                    }
                }
            }
        }
    } else {
        // ----------------------------------------------------------- epilogue
        const int q = warp & 3, h = warp >= 7;  // TMEM lanes 32q.., half of the columns
        const int r = 32 * q + lane;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * q) << 16);
        uint32_t slot = 0, sphase = 0, buf = 0, bphase = 0, iphase = 0;
        bool ok = true;
        for (int item = blockIdx.x; ok && item < total; item += gridDim.x) {
            const Item it = decode<MODE>(P, tail, item);
            const bool active = 32 * q < it.count;  // the warp has rows of the tile
            float acc[128];
#pragma unroll
            for (int i = 0; i < 128; ++i) acc[i] = 0.f;
            for (int kb = 0; kb < kbs; ++kb) {
                if (!wait_warp(&tail->sfull[slot], sphase, abort)) {
                    ok = false;
                    break;
                }
                const float rs = tail->row_scale[slot][r];
                const float s0 = rs * tail->block_scale[slot][MODE == kGateUp ? 0 : h];
                const float s1 = MODE == kGateUp ? rs * tail->block_scale[slot][1] : s0;
                __syncwarp();
                if (lane == 0) sm100::mbar_arrive(&tail->sempty[slot]);
                if (++slot == kScaleSlots) {
                    slot = 0;
                    sphase ^= 1;
                }
                if (!wait_warp(&tail->tfull[buf], bphase, abort)) {
                    ok = false;
                    break;
                }
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
                    wait_ld16(t[0]);
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        if (c < 7) sm100::tmem_ld16(col(c + 1), t[(c + 1) & 1]);
                        const float s = c < 4 ? s0 : s1;
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[16 * c + i] = fmaf(t[c & 1][i], s, acc[16 * c + i]);
                        if (c < 7) wait_ld16(t[(c + 1) & 1]);
                    }
                }
                sm100::tc_fence_before();
                __syncwarp();
                if (lane == 0) sm100::mbar_arrive(&tail->tempty[buf]);
                buf ^= 1;
                bphase ^= buf == 0;
            }
            if (!ok) break;
            const bool row = r < it.count;
            const int64_t at = static_cast<int64_t>(it.row0) + r;
            if constexpr (MODE == kGateUp) {
                if (!active) continue;
                float top = fp8::kTiny;
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    acc[i] = silu_f32(acc[i]) * acc[64 + i];
                    top = fp8::max_nan(top, fabsf(acc[i]));
                }
                // the group's other 64 columns are the other half's
                tail->top[iphase][h][r] = top;
                __syncwarp();
                if (lane == 0) sm100::mbar_arrive(&tail->half[q]);
                if (!wait_warp(&tail->half[q], iphase, abort)) {
                    ok = false;
                    break;
                }
                top = fp8::max_nan(top, tail->top[iphase][h ^ 1][r]);
                iphase ^= 1;
                if (row) {
                    const fp8::Divisor f(top);
                    uint8_t *dst = P.act + at * P.n + it.n * kGroup + 64 * h;
#pragma unroll
                    for (int i = 0; i < 64; i += 32) {
                        uint32_t v[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            v[j] = fp8::pack4(f, acc[i + 4 * j], acc[i + 4 * j + 1], acc[i + 4 * j + 2],
                                              acc[i + 4 * j + 3]);
                        store32(dst + i, v);
                    }
                    if (h == 0) P.act_scales[at * nt + it.n] = fp8::scale_of(top);
                }
            } else if constexpr (MODE == kDown) {
                // n % 16 == 0: 16 columns are 32 aligned bytes, all or none of them there
                uint16_t *dst = static_cast<uint16_t *>(P.out) + at * P.n;
                if (row) {
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const int n0 = it.n * kBN + 128 * h + 16 * c;
                        if (n0 < P.n) {
                            uint32_t v[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[j] = pack_bf16x2(acc[16 * c + 2 * j], acc[16 * c + 2 * j + 1]);
                            store32(dst + n0, v);
                        }
                    }
                }
            } else {
                const bool vec = P.n % 16 == 0;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const int n0 = it.n * kBN + 128 * h + 16 * c;
                    if (!row || n0 >= P.n) continue;
                    if (P.out_f32) {
                        float *dst = static_cast<float *>(P.out) + at * P.n + n0;
                        if (vec) {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                reinterpret_cast<float4 *>(dst)[i] =
                                    make_float4(acc[16 * c + 4 * i], acc[16 * c + 4 * i + 1], acc[16 * c + 4 * i + 2],
                                                acc[16 * c + 4 * i + 3]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (n0 + i < P.n) dst[i] = acc[16 * c + i];
                        }
                    } else {
                        uint16_t *dst = static_cast<uint16_t *>(P.out) + at * P.n + n0;
                        if (vec) {
#pragma unroll
                            for (int i = 0; i < 2; ++i)
                                reinterpret_cast<uint4 *>(dst)[i] =
                                    make_uint4(pack_bf16x2(acc[16 * c + 8 * i], acc[16 * c + 8 * i + 1]),
                                               pack_bf16x2(acc[16 * c + 8 * i + 2], acc[16 * c + 8 * i + 3]),
                                               pack_bf16x2(acc[16 * c + 8 * i + 4], acc[16 * c + 8 * i + 5]),
                                               pack_bf16x2(acc[16 * c + 8 * i + 6], acc[16 * c + 8 * i + 7]));
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (n0 + i < P.n) dst[i] = f2bf(acc[16 * c + i]);
                        }
                    }
                }
            }
        }
        sm100::tc_fence_before();
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
        make_uint4(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]), pack_bf16x2(acc[4], acc[5]),
                   pack_bf16x2(acc[6], acc[7]));
}

template <int MODE>
int launch_tile(const CUtensorMap &x, const CUtensorMap &x16, const CUtensorMap &w, const Params &P, int64_t items,
                cudaStream_t stream) {
    if (int rc = ensure_dynamic_smem(fp8_tile_kernel<MODE>, kSmem, "cudaFuncSetAttribute(fp8_tile)")) return rc;
    return launch_pdl(fp8_tile_kernel<MODE>, dim3(static_cast<unsigned>(std::min<int64_t>(items, sm_count()))),
                      dim3(kThreads), kSmem, stream, "fp8_tile_kernel", x, x16, w, P);
}

int row_maps(CUtensorMap *m, CUtensorMap *m16, const void *base, int rows, int cols) {
    const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
    const uint64_t str[1] = {static_cast<uint64_t>(cols)};
    if (int rc = make_map_u8(m, base, 2, dims, str, kBM)) return rc;
    return make_map_u8(m16, base, 2, dims, str, 16);
}

}  // namespace

int launch_linear_fp8_tiles(const LinearFp8 &a, int32_t *status, cudaStream_t stream) {
    CUtensorMap x{}, x16{}, w{};
    if (int rc = row_maps(&x, &x16, a.x, a.tokens, a.cols)) return rc;
    const uint64_t dims[2] = {static_cast<uint64_t>(a.cols), static_cast<uint64_t>(a.rows)};
    const uint64_t str[1] = {static_cast<uint64_t>(a.cols)};
    if (int rc = make_map_u8(&w, a.w, 2, dims, str, 128)) return rc;
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
    return launch_tile<kLinear>(x, x16, w, P, items, stream);
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
    CUtensorMap x{}, act{}, act16{}, gu{}, dn{};
    {
        // rows gathered four at a time: the map's box is one row
        const uint64_t dims[2] = {static_cast<uint64_t>(a.hidden), static_cast<uint64_t>(a.tokens)};
        const uint64_t str[1] = {static_cast<uint64_t>(a.hidden)};
        if (int rc = make_map_u8(&x, a.x, 2, dims, str, 1)) return rc;
    }
    if (int rc = row_maps(&act, &act16, s.act, routes, a.inner)) return rc;
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
    if (int rc = launch_tile<kGateUp>(x, x, gu, G, tiles * nt1, stream)) return rc;
    P.row_scales = s.act_scales;
    P.block_scales = a.down_scales;
    P.n = a.hidden;
    P.k = a.inner;
    P.out = s.y;
    if (int rc = launch_tile<kDown>(act, act16, dn, P, tiles * nt2, stream)) return rc;
    const int64_t ctas = (static_cast<int64_t>(a.tokens) * (a.hidden / 8) + 255) / 256;
    return launch_pdl(fp8_combine_kernel, dim3(static_cast<unsigned>(ctas)), dim3(256), 0, stream,
                      "fp8_combine_kernel", static_cast<const uint16_t *>(s.y),
                      static_cast<const int32_t *>(s.route_pos), a.weights, a.tokens, a.top_k, a.hidden, a.out);
}

}  // namespace lrb
