// The FP8 products at the smallest sizes: a warp per weight row (or pair of
// rows), every lane a 16-byte piece of it, FP32 FMA over the e4m3 values
// (widened to FP16, whose products an FP32 FMA takes exactly).  The rows are the traffic: they are streamed once with all of a
// row's loads in flight, and the few activations come from L1 and L2.
#include "fp8_kernels.cuh"

namespace lrb {
namespace {

using fp8::dot16;
using fp8::kGroup;
using fp8::halves16;
using fp8::ld_again;
using fp8::ld_once;

constexpr int kWarps = 8;
constexpr int kChunk = 32 * 16;  // weight bytes a warp reads per load
constexpr int kUnroll = 4;       // loads of a row in flight

// A warp per output row, for up to MT tokens.
template <int MT>
__global__ void __launch_bounds__(kWarps * 32) linear_gemv_kernel(LinearFp8 a) {
    const int lane = threadIdx.x & 31;
    const int n = blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int gk = fp8::groups(a.cols);
    const bool live = n < a.rows;
    const uint8_t *w = a.w + static_cast<int64_t>(live ? n : 0) * a.cols;
    // L2 is coherent with whatever the previous kernel still writes, so asking
    // it for the row early is safe; the loads themselves wait.
    if (live && lane == 0) prefetch_l2_bulk(w, a.cols);
    grid_dependency_wait();
    grid_dependency_trigger();
    if (!live) return;
    const float *ws = a.w_scales + static_cast<int64_t>(n / kGroup) * gk;
    // one or two rows' pieces are requested with the weights' (1 x 1024 x 2048: 1.9 us
    // back to back in a graph, 2.2 without); more would leave no registers for these
    constexpr bool kAhead = MT <= 2;
    auto row = [&](int m) { return a.x + static_cast<int64_t>(min(m, a.tokens - 1)) * a.cols; };
    float acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = 0.f;
    for (int c0 = lane * 16; c0 < a.cols; c0 += kUnroll * kChunk) {
        uint4 v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int c = c0 + u * kChunk;
            v[u] = c < a.cols ? ld_again(w + c) : make_uint4(0, 0, 0, 0);
        }
        uint4 ahead[kAhead ? MT : 1][kUnroll];
        if constexpr (kAhead) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    const int c = c0 + u * kChunk;
                    ahead[m][u] = c < a.cols ? ld_again(row(m) + c) : make_uint4(0, 0, 0, 0);
                }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int c = c0 + u * kChunk;
            if (c >= a.cols) break;
            const float s = ws[c / kGroup];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                uint16_t x[16];
                halves16(kAhead ? ahead[m][u] : ld_again(row(m) + c), x);
                const float xs = a.x_scales[static_cast<int64_t>(min(m, a.tokens - 1)) * gk + c / kGroup];
                acc[m] = fmaf(dot16(v[u], x), s * xs, acc[m]);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const float r = warp_sum(acc[m]);
        if (lane == 0 && m < a.tokens) {
            const int64_t at = static_cast<int64_t>(m) * a.rows + n;
            if (a.out_f32) static_cast<float *>(a.out)[at] = r;
            else static_cast<uint16_t *>(a.out)[at] = f2bf(r);
        }
    }
}

// h[r, p] = silu(gate) * up for two neighbouring p of one route r: four rows
// of the route's expert, sharing the unpacked activations.
__global__ void __launch_bounds__(kWarps * 32) gate_up_gemv_kernel(ExpertsFp8 a, float *__restrict__ h) {
    grid_dependency_wait();
    grid_dependency_trigger();
    const int lane = threadIdx.x & 31;
    const int per_route = a.inner / 2;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    const int64_t r = item / per_route;
    if (r >= static_cast<int64_t>(a.tokens) * a.top_k) return;
    const int p = static_cast<int>(item % per_route) * 2;
    const int64_t e = a.idx[r];
    if (e < 0 || e >= a.experts) return;
    const int gk = fp8::groups(a.hidden);
    const int64_t t = r / a.top_k;
    const uint8_t *x = a.x + t * a.hidden;
    const float *xs = a.x_scales + t * gk;
    const uint8_t *w[4];
    const uint8_t *gu = a.gate_up + e * 2 * a.inner * a.hidden;
    w[0] = gu + static_cast<int64_t>(p) * a.hidden;
    w[1] = w[0] + a.hidden;
    w[2] = w[0] + static_cast<int64_t>(a.inner) * a.hidden;
    w[3] = w[2] + a.hidden;
    // inner % 128 == 0, so a pair never straddles two blocks
    const float *gs = a.gate_up_scales + (e * (2 * a.inner / kGroup) + p / kGroup) * gk;
    const float *us = gs + static_cast<int64_t>(a.inner / kGroup) * gk;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c0 = lane * 16; c0 < a.hidden; c0 += kUnroll * kChunk) {
        uint4 v[kUnroll][4];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int c = c0 + u * kChunk;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[u][i] = c < a.hidden ? ld_once(w[i] + c) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int c = c0 + u * kChunk;
            if (c >= a.hidden) break;
            uint16_t f[16];
            halves16(ld_again(x + c), f);
            const float s = xs[c / kGroup], g = s * gs[c / kGroup], up = s * us[c / kGroup];
            acc[0] = fmaf(dot16(v[u][0], f), g, acc[0]);
            acc[1] = fmaf(dot16(v[u][1], f), g, acc[1]);
            acc[2] = fmaf(dot16(v[u][2], f), up, acc[2]);
            acc[3] = fmaf(dot16(v[u][3], f), up, acc[3]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = warp_sum(acc[i]);
    if (lane == 0)
        *reinterpret_cast<float2 *>(h + r * a.inner + p) =
            make_float2(silu_f32(acc[0]) * acc[2], silu_f32(acc[1]) * acc[3]);
}

// out[t, n] over the token's routes, eight at a time, a warp per column n.
// Each CTA first brings the routes' activation rows to e4m3 in shared memory
// (the same values in every CTA).  The kernel follows gate_up_gemv_kernel,
// which has seen every earlier kernel of the stream complete before it lets
// this one start: the route ids and the weights are final then, so the first
// 512 bytes of each route's row, their scales and the routes' weights are on
// their way before the wait for h.
constexpr int kRoutes = 8;
__global__ void __launch_bounds__(kWarps * 32) down_gemv_kernel(ExpertsFp8 a, const float *__restrict__ h,
                                                                int blocks_per_token) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int gi = a.inner / kGroup, gn = fp8::groups(a.hidden);
    uint8_t *act = smem;                                                    // [8][I]
    float *acts = reinterpret_cast<float *>(smem + kRoutes * a.inner);      // [8][I / 128]
    const int lane = threadIdx.x & 31;
    const int64_t t = blockIdx.x / blocks_per_token;
    const int n = (blockIdx.x % blocks_per_token) * kWarps + (threadIdx.x >> 5);
    const bool live = n < a.hidden;
    float acc = 0.f;
    for (int k0 = 0; k0 < a.top_k; k0 += kRoutes) {
        const int count = min(kRoutes, a.top_k - k0);
        int e[kRoutes];
        uint4 v[kRoutes];
        float sc[kRoutes], rw[kRoutes];  // the lane's first scale and the weight of each route
#pragma unroll
        for (int j = 0; j < kRoutes; ++j) {
            const int64_t id = j < count ? __ldcg(a.idx + t * a.top_k + k0 + j) : -1;
            e[j] = id >= 0 && id < a.experts ? static_cast<int>(id) : -1;
        }
        auto row = [&](int j) { return a.down + (static_cast<int64_t>(e[j]) * a.hidden + n) * a.inner; };
#pragma unroll
        for (int j = 0; j < kRoutes; ++j)
            v[j] = live && e[j] >= 0 && lane * 16 < a.inner ? ld_once(row(j) + lane * 16) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < kRoutes; ++j) {
            sc[j] = live && e[j] >= 0 && lane * 16 < a.inner
                        ? __ldcg(a.down_scales + (static_cast<int64_t>(e[j]) * gn + n / kGroup) * gi + lane / 8) : 0.f;
            rw[j] = e[j] >= 0 ? bf2f(__ldcg(a.weights + t * a.top_k + k0 + j)) : 0.f;
        }
        if (k0 == 0) {
            grid_dependency_wait();
            grid_dependency_trigger();
        } else {
            __syncthreads();  // every warp is done with the previous routes
        }
        // 16 values a thread, 8 threads a group
        for (int i = threadIdx.x; i < kRoutes * a.inner / 16; i += kWarps * 32) {
            const int j = i / (a.inner / 16), c = (i % (a.inner / 16)) * 16;
            const int64_t id = j < count ? a.idx[t * a.top_k + k0 + j] : -1;
            float y[16];
            float top = fp8::kTiny;
            if (id >= 0 && id < a.experts) {
                const float4 *src =
                    reinterpret_cast<const float4 *>(h + (t * a.top_k + k0 + j) * a.inner + c);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float4 f = __ldcg(src + u);
                    y[4 * u] = f.x;
                    y[4 * u + 1] = f.y;
                    y[4 * u + 2] = f.z;
                    y[4 * u + 3] = f.w;
                }
            } else {
#pragma unroll
                for (int u = 0; u < 16; ++u) y[u] = 0.f;
            }
#pragma unroll
            for (int u = 0; u < 16; ++u) top = fp8::max_nan(top, fabsf(y[u]));
            // inner is a multiple of 128, so the 8 threads of a group are
            // neighbours in one warp and in the loop together
            const unsigned mask = 0xffu << (lane & 24);
#pragma unroll
            for (int s = 4; s; s >>= 1) top = fp8::max_nan(top, __shfl_xor_sync(mask, top, s));
            const fp8::Divisor f(top);
            *reinterpret_cast<uint4 *>(act + j * a.inner + c) =
                make_uint4(fp8::pack4(f, y[0], y[1], y[2], y[3]), fp8::pack4(f, y[4], y[5], y[6], y[7]),
                           fp8::pack4(f, y[8], y[9], y[10], y[11]), fp8::pack4(f, y[12], y[13], y[14], y[15]));
            if ((lane & 7) == 0) acts[j * gi + c / kGroup] = fp8::scale_of(top);
        }
        __syncthreads();
        if (!live) continue;
#pragma unroll
        for (int j = 0; j < kRoutes; ++j) {
            if (e[j] < 0) continue;
            const float *ws = a.down_scales + (static_cast<int64_t>(e[j]) * gn + n / kGroup) * gi;
            float part = 0.f;
            for (int c = lane * 16; c < a.inner; c += kChunk) {
                const uint4 w = c == lane * 16 ? v[j] : ld_once(row(j) + c);
                uint16_t f[16];
                halves16(*reinterpret_cast<const uint4 *>(act + j * a.inner + c), f);
                part = fmaf(dot16(w, f), (c == lane * 16 ? sc[j] : ws[c / kGroup]) * acts[j * gi + c / kGroup], part);
            }
            acc = fmaf(part, rw[j], acc);
        }
    }
    if (!live) return;
    acc = warp_sum(acc);
    if (lane == 0) a.out[t * a.hidden + n] = f2bf(acc);
}

}  // namespace

int launch_linear_fp8_gemv(const LinearFp8 &a, cudaStream_t stream) {
    const dim3 grid((a.rows + kWarps - 1) / kWarps), block(kWarps * 32);
    if (a.tokens == 1)
        return launch_pdl(linear_gemv_kernel<1>, grid, block, 0, stream, "linear_gemv_kernel", a);
    if (a.tokens == 2)
        return launch_pdl(linear_gemv_kernel<2>, grid, block, 0, stream, "linear_gemv_kernel", a);
    return launch_pdl(linear_gemv_kernel<kGemvTokens>, grid, block, 0, stream, "linear_gemv_kernel", a);
}

int launch_experts_fp8_gemv(const ExpertsFp8 &a, float *h, cudaStream_t stream) {
    const int64_t routes = static_cast<int64_t>(a.tokens) * a.top_k;
    const int64_t ctas = (routes * (a.inner / 2) + kWarps - 1) / kWarps;
    const int per_token = (a.hidden + kWarps - 1) / kWarps;
    LRB_REQUIRE(ctas < (1ll << 31) && static_cast<int64_t>(a.tokens) * per_token < (1ll << 31),
                "moe_experts_fp8: too many routes");
    if (int rc = launch_pdl(gate_up_gemv_kernel, dim3(static_cast<unsigned>(ctas)), dim3(kWarps * 32), 0, stream,
                            "gate_up_gemv_kernel", a, h))
        return rc;
    const int smem = kRoutes * (a.inner + a.inner / kGroup * 4);
    if (smem > 48 * 1024)
        if (int rc = ensure_dynamic_smem(down_gemv_kernel, smem, "cudaFuncSetAttribute(down_gemv)")) return rc;
    return launch_pdl(down_gemv_kernel, dim3(static_cast<unsigned>(a.tokens * per_token)), dim3(kWarps * 32), smem,
                      stream, "down_gemv_kernel", a, const_cast<const float *>(h), per_token);
}

}  // namespace lrb
