// e4m3 rows and weights: the residual addition and RMS norm that feed the FP8
// products (moe_rmsnorm_fp8), its norm-free form, and the block scales of
// weights (moe_quantize_fp8_blocks).
//
// The norm is the model's Qwen3_5MoeRMSNorm behind the layer's residual add
// (transformers modeling_qwen3_5_moe.py): r = bf16(x + residual),
// y = r * rsqrt(mean(r^2) + eps) * (offset + weight), the sum of squares in
// FP32; q and the scales are those of y before it is rounded to BF16.
#include "fp8_kernels.cuh"

namespace lrb {
namespace {

using fp8::Divisor;
using fp8::kGroup;

struct RowArgs {
    const uint16_t *x, *residual, *weight;
    int64_t x_stride, residual_stride;
    float offset, eps;
    int tokens, hidden;
    uint8_t *q;
    float *scales;
    uint16_t *normed, *residual_out;
};

__device__ __forceinline__ void unpack8(uint4 v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = bf16_lo(w[i]);
        f[2 * i + 1] = bf16_hi(w[i]);
    }
}

// A row per TPR threads; thread i of a row holds its 16-byte vectors i, i + TPR,
// ... (8 values each, as BF16: r is BF16 by definition, so a row costs 4
// registers per vector and is read once).  A group of 128 values is 16
// neighbouring lanes, so its maximum is four shuffles.  Needs hidden % 8 == 0
// and 16-byte rows.
template <int TPR, int VPT, bool NORM>
__global__ void __launch_bounds__(256) row_kernel(RowArgs a) {
    constexpr int kRows = 256 / TPR, kWarps = TPR / 32;  // rows of a CTA, warps of a row
    __shared__ float part[kRows][VPT * kWarps];
    grid_dependency_wait();
    grid_dependency_trigger();
    const int sub = threadIdx.x / TPR, i0 = threadIdx.x % TPR;
    const int t = blockIdx.x * kRows + sub;
    const int units = a.hidden / 8, n_groups = fp8::groups(a.hidden);
    const bool row = t < a.tokens;
    uint4 v[VPT], add[VPT];
    const uint4 *src = reinterpret_cast<const uint4 *>(a.x + static_cast<int64_t>(row ? t : 0) * a.x_stride);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int u = i0 + j * TPR;
        v[j] = row && u < units ? src[u] : make_uint4(0, 0, 0, 0);
    }
    if (NORM && a.residual) {
        const uint4 *res =
            reinterpret_cast<const uint4 *>(a.residual + static_cast<int64_t>(row ? t : 0) * a.residual_stride);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int u = i0 + j * TPR;
            add[j] = row && u < units ? res[u] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            float p[8], r[8];
            unpack8(v[j], p);
            unpack8(add[j], r);
            v[j] = make_uint4(fp8::pack_bf16(p[0] + r[0], p[1] + r[1]), fp8::pack_bf16(p[2] + r[2], p[3] + r[3]),
                              fp8::pack_bf16(p[4] + r[4], p[5] + r[5]), fp8::pack_bf16(p[6] + r[6], p[7] + r[7]));
        }
        if (a.residual_out) {
            uint4 *dst = reinterpret_cast<uint4 *>(a.residual_out + static_cast<int64_t>(t) * a.hidden);
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int u = i0 + j * TPR;
                if (row && u < units) dst[u] = v[j];
            }
        }
    }
    float inv = 1.f;
    if constexpr (NORM) {
        // one sum per 32 neighbouring vectors, those added in order
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            float p[8], b = 0.f;
            unpack8(v[j], p);
#pragma unroll
            for (int c = 0; c < 8; ++c) b = fmaf(p[c], p[c], b);
            b = warp_sum(b);
            if constexpr (TPR == 32) ss += b;
            else if ((threadIdx.x & 31) == 0) part[sub][j * kWarps + i0 / 32] = b;
        }
        if constexpr (TPR > 32) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < VPT * kWarps; ++i) ss += part[sub][i];
        }
        inv = rsqrtf(ss / static_cast<float>(a.hidden) + a.eps);
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int u = i0 + j * TPR;
        float y[8];
        unpack8(v[j], y);
        if constexpr (NORM) {
            float w[8];
            unpack8(u < units ? fp8::ld_again(a.weight + u * 8) : make_uint4(0, 0, 0, 0), w);
#pragma unroll
            for (int c = 0; c < 8; ++c) y[c] = y[c] * inv * (a.offset + w[c]);
            if (a.normed && row && u < units)
                *reinterpret_cast<uint4 *>(a.normed + static_cast<int64_t>(t) * a.hidden + u * 8) =
                    make_uint4(fp8::pack_bf16(y[0], y[1]), fp8::pack_bf16(y[2], y[3]), fp8::pack_bf16(y[4], y[5]),
                               fp8::pack_bf16(y[6], y[7]));
        }
        float top = fp8::kTiny;
        if (u < units) {
#pragma unroll
            for (int c = 0; c < 8; ++c) top = fp8::max_nan(top, fabsf(y[c]));
        }
#pragma unroll
        for (int s = 8; s; s >>= 1) top = fp8::max_nan(top, __shfl_xor_sync(0xffffffffu, top, s));
        if (row && u < units) {
            const Divisor f(top);
            *reinterpret_cast<uint2 *>(a.q + static_cast<int64_t>(t) * a.hidden + u * 8) =
                make_uint2(fp8::pack4(f, y[0], y[1], y[2], y[3]), fp8::pack4(f, y[4], y[5], y[6], y[7]));
            if ((u & 15) == 0) a.scales[static_cast<int64_t>(t) * n_groups + u / 16] = fp8::scale_of(top);
        }
    }
}

// Any width, alignment and stride, a CTA per row, one value at a time.  A row
// that does not stay in registers is read again for the output: the stored sum
// where there is one (it may have replaced the residual in place), else the
// inputs.  A warp owns each group, four values a lane.
template <bool NORM>
__global__ void __launch_bounds__(256) row_any_kernel(RowArgs a) {
    __shared__ float part[8];
    grid_dependency_wait();
    grid_dependency_trigger();
    const int64_t t = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_groups = fp8::groups(a.hidden);
    const uint16_t *x = a.x + t * a.x_stride;
    const uint16_t *res = a.residual ? a.residual + t * a.residual_stride : nullptr;
    uint16_t *sum = a.residual_out ? a.residual_out + t * a.hidden : nullptr;
    float inv = 1.f;
    if constexpr (NORM) {
        float ss = 0.f;
        // a warp visits the same groups in both passes, so each thread reads
        // back only what it stored itself
        for (int g = warp; g < n_groups; g += 8)
            for (int c = g * kGroup + lane; c < min(a.hidden, (g + 1) * kGroup); c += 32) {
                float v = bf2f(x[c]);
                if (res) {
                    const uint16_t b = f2bf(v + bf2f(res[c]));
                    if (sum) sum[c] = b;
                    v = bf2f(b);
                }
                ss = fmaf(v, v, ss);
            }
        ss = warp_sum(ss);
        if (lane == 0) part[warp] = ss;
        __syncthreads();
        ss = 0.f;
        for (int w = 0; w < 8; ++w) ss += part[w];
        inv = rsqrtf(ss / static_cast<float>(a.hidden) + a.eps);
    }
    for (int g = warp; g < n_groups; g += 8) {
        float y[4];
        float top = fp8::kTiny;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = g * kGroup + j * 32 + lane;
            y[j] = 0.f;
            if (c >= a.hidden) continue;
            if (NORM && res) y[j] = sum ? bf2f(sum[c]) : rbf(bf2f(x[c]) + bf2f(res[c]));
            else y[j] = bf2f(x[c]);
            if constexpr (NORM) {
                y[j] = y[j] * inv * (a.offset + bf2f(a.weight[c]));
                if (a.normed) a.normed[t * a.hidden + c] = f2bf(y[j]);
            }
            top = fp8::max_nan(top, fabsf(y[j]));
        }
#pragma unroll
        for (int s = 16; s; s >>= 1) top = fp8::max_nan(top, __shfl_xor_sync(0xffffffffu, top, s));
        const Divisor f(top);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = g * kGroup + j * 32 + lane;
            if (c < a.hidden) a.q[t * a.hidden + c] = static_cast<uint8_t>(fp8::pack2(f(y[j]), 0.f));
        }
        if (lane == 0) a.scales[t * n_groups + g] = fp8::scale_of(top);
    }
}

template <int TPR, int VPT, bool NORM>
int launch_rows(const RowArgs &a, cudaStream_t stream) {
    constexpr int kRows = 256 / TPR;
    return launch_pdl(row_kernel<TPR, VPT, NORM>, dim3((a.tokens + kRows - 1) / kRows), dim3(256), 0, stream,
                      "row_kernel", a);
}

bool aligned16(const void *p) { return on_boundary(p, 16); }

template <bool NORM>
int rows_for(const RowArgs &a, cudaStream_t stream) {
    const bool vec = a.hidden % 8 == 0 && a.hidden <= 16384 && a.x_stride % 8 == 0 && aligned16(a.x) &&
                     aligned16(a.weight) && aligned16(a.normed) && aligned16(a.residual_out) &&
                     (!a.residual || (a.residual_stride % 8 == 0 && aligned16(a.residual))) &&
                     (reinterpret_cast<uintptr_t>(a.q) & 7) == 0;
    if (!vec)
        return launch_pdl(row_any_kernel<NORM>, dim3(a.tokens), dim3(256), 0, stream, "row_any_kernel", a);
    // As many threads as the row has vectors, up to 256: by the width alone, so
    // that a row comes out the same in every batch (8192 rows of 2048 with the
    // residual: 28.5 us, 5.3 TB/s; a warp a row with eight vectors a lane 32.6).
    const int units = a.hidden / 8;
    if (units <= 32) return launch_rows<32, 1, NORM>(a, stream);
    if (units <= 64) return launch_rows<64, 1, NORM>(a, stream);
    if (units <= 128) return launch_rows<128, 1, NORM>(a, stream);
    if (units <= 256) return launch_rows<256, 1, NORM>(a, stream);
    if (units <= 512) return launch_rows<256, 2, NORM>(a, stream);
    if (units <= 1024) return launch_rows<256, 4, NORM>(a, stream);
    return launch_rows<256, 8, NORM>(a, stream);
}

// A CTA per 128 x 128 block of one matrix of the bank.  VEC: 16-byte loads
// (cols % 8 == 0), each thread holding eight vectors of the block in registers;
// four CTAs an SM (a few spilled registers) keep 128 KB of loads in flight
// where the 98 registers it would take allow two: one layer's gate/up bank
// (1.6 GB moved) 285 us, 5.65 TB/s, against 336.
template <bool VEC>
__global__ void __launch_bounds__(256, VEC ? 4 : 1) block_kernel(const uint16_t *w, int rows, int cols,
                                                    uint8_t *__restrict__ q, float *__restrict__ scales) {
    __shared__ float part[8];
    grid_dependency_wait();
    grid_dependency_trigger();
    const int gk = fp8::groups(cols), gn = fp8::groups(rows);
    const int kb = blockIdx.x % gk, nb = static_cast<int>(blockIdx.x / gk) % gn;
    const int64_t bank = static_cast<int64_t>(blockIdx.x) / gk / gn;
    const int64_t base = bank * rows * cols;
    float top = fp8::kTiny;
    if constexpr (VEC) {
        const int r0 = nb * kGroup + threadIdx.x / 16, c = kb * kGroup + (threadIdx.x % 16) * 8;
        uint4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = r0 + 16 * j;
            v[j] = r < rows && c < cols ? fp8::ld_once(w + base + static_cast<int64_t>(r) * cols + c)
                                        : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float f[8];
            unpack8(v[j], f);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fp8::max_nan(top, fabsf(f[i]));
        }
#pragma unroll
        for (int s = 16; s; s >>= 1) top = fp8::max_nan(top, __shfl_xor_sync(0xffffffffu, top, s));
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fp8::max_nan(top, part[i]);
        const Divisor f(top);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = r0 + 16 * j;
            float y[8];
            unpack8(v[j], y);
            if (r < rows && c < cols)
                *reinterpret_cast<uint2 *>(q + base + static_cast<int64_t>(r) * cols + c) =
                    make_uint2(fp8::pack4(f, y[0], y[1], y[2], y[3]), fp8::pack4(f, y[4], y[5], y[6], y[7]));
        }
    } else {
        const int r0 = nb * kGroup + threadIdx.x / 128, c = kb * kGroup + threadIdx.x % 128;
        for (int r = r0; r < min(rows, (nb + 1) * kGroup); r += 2)
            if (c < cols) top = fp8::max_nan(top, fabsf(bf2f(w[base + static_cast<int64_t>(r) * cols + c])));
#pragma unroll
        for (int s = 16; s; s >>= 1) top = fp8::max_nan(top, __shfl_xor_sync(0xffffffffu, top, s));
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
        __syncthreads();
        for (int i = 0; i < 8; ++i) top = fp8::max_nan(top, part[i]);
        const Divisor f(top);
        for (int r = r0; r < min(rows, (nb + 1) * kGroup); r += 2)
            if (c < cols) {
                const int64_t at = base + static_cast<int64_t>(r) * cols + c;
                q[at] = static_cast<uint8_t>(fp8::pack2(f(bf2f(w[at])), 0.f));
            }
    }
    if (threadIdx.x == 0) scales[blockIdx.x] = fp8::scale_of(top);
}

}  // namespace
}  // namespace lrb

extern "C" int moe_rmsnorm_fp8(const uint16_t *x, int64_t x_stride, const uint16_t *residual,
                               int64_t residual_stride, const uint16_t *weight, float weight_offset, float eps,
                               int tokens, int hidden, uint8_t *q, float *scales, uint16_t *normed,
                               uint16_t *residual_out, void *stream) {
    LRB_REQUIRE(tokens >= 0 && tokens <= (1 << 30) && hidden >= 1 && hidden <= (1 << 20),
                "moe_rmsnorm_fp8: bad tokens %d / hidden %d", tokens, hidden);
    LRB_REQUIRE(weight || (!residual && !normed && !residual_out),
                "moe_rmsnorm_fp8: without a norm weight there is no residual, normed or residual_out");
    LRB_REQUIRE(!residual_out || residual, "moe_rmsnorm_fp8: residual_out without residual");
    LRB_REQUIRE(tokens <= 1 || (x_stride >= hidden && (!residual || residual_stride >= hidden)),
                "moe_rmsnorm_fp8: row strides below hidden");
    LRB_REQUIRE(tokens == 0 || (x && q && scales), "moe_rmsnorm_fp8: null tensor");
    LRB_REQUIRE(lrb::on_boundary(x, 2) && lrb::on_boundary(residual, 2) && lrb::on_boundary(weight, 2) &&
                    lrb::on_boundary(normed, 2) && lrb::on_boundary(residual_out, 2) && lrb::on_boundary(scales, 4),
                "moe_rmsnorm_fp8: tensors must be aligned to their elements");
    LRB_REQUIRE(!weight || (eps >= 0.f && eps < 1.f), "moe_rmsnorm_fp8: eps outside [0, 1)");
    if (tokens == 0) return MOE_OK;
    if (int rc = lrb::require_sm100()) return rc;
    const lrb::RowArgs a{x, residual, weight, x_stride, residual_stride, weight_offset, eps, tokens, hidden, q, scales,
                         normed, residual_out};
    return weight ? lrb::rows_for<true>(a, lrb::as_stream(stream)) : lrb::rows_for<false>(a, lrb::as_stream(stream));
}

extern "C" int moe_quantize_fp8_blocks(const uint16_t *w, int banks, int rows, int cols, uint8_t *q, float *scales,
                                       void *stream) {
    LRB_REQUIRE(banks >= 0 && rows >= 1 && rows <= (1 << 30) && cols >= 1 && cols <= (1 << 30),
                "moe_quantize_fp8_blocks: bad shape [%d, %d, %d]", banks, rows, cols);
    const int64_t blocks = static_cast<int64_t>(banks) * lrb::fp8::groups(rows) * lrb::fp8::groups(cols);
    LRB_REQUIRE(blocks < (1ll << 31), "moe_quantize_fp8_blocks: too many blocks");
    LRB_REQUIRE(banks == 0 || (w && q && scales), "moe_quantize_fp8_blocks: null tensor");
    LRB_REQUIRE(lrb::on_boundary(w, 2) && lrb::on_boundary(scales, 4),
                "moe_quantize_fp8_blocks: tensors must be aligned to their elements");
    if (banks == 0) return MOE_OK;
    if (int rc = lrb::require_sm100()) return rc;
    const bool vec = cols % 8 == 0 && lrb::aligned16(w) && (reinterpret_cast<uintptr_t>(q) & 7) == 0;
    const dim3 grid(static_cast<unsigned>(blocks)), block(256);
    if (vec)
        return lrb::launch_pdl(lrb::block_kernel<true>, grid, block, 0, lrb::as_stream(stream), "block_kernel", w,
                               rows, cols, q, scales);
    return lrb::launch_pdl(lrb::block_kernel<false>, grid, block, 0, lrb::as_stream(stream), "block_kernel", w, rows,
                           cols, q, scales);
}
