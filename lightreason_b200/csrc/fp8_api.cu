// C entry points of the FP8 products: argument checks, workspaces and the
// choice of kernel by size.
#include <algorithm>

#include "fp8_kernels.cuh"

namespace lrb {
namespace {

size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

int check_experts(int tokens, int experts, int top_k, int hidden, int inner) {
    LRB_REQUIRE(tokens >= 0 && experts >= 1 && experts <= 1024, "moe_experts_fp8: bad tokens %d / experts %d", tokens,
                experts);
    LRB_REQUIRE(top_k >= 1 && top_k <= 32, "moe_experts_fp8: top_k %d outside [1, 32]", top_k);
    LRB_REQUIRE(hidden >= 16 && hidden % 16 == 0 && hidden <= 65536,
                "moe_experts_fp8: hidden %d must be a multiple of 16 in [16, 65536]", hidden);
    LRB_REQUIRE(inner >= 128 && inner % 128 == 0 && inner <= 16384,
                "moe_experts_fp8: inner %d must be a multiple of 128 in [128, 16384]", inner);
    LRB_REQUIRE(static_cast<int64_t>(tokens) * top_k < (1 << 30), "moe_experts_fp8: too many routes");
    return MOE_OK;
}

// Where the scratch of moe_experts_fp8 lies in its workspace.
struct Layout {
    bool gemv;
    size_t offsets, row_token, route_pos, counters, act, act_scales, y, bytes;
};
Layout layout(int tokens, int experts, int top_k, int hidden, int inner) {
    Layout l{};
    const size_t routes = static_cast<size_t>(tokens) * top_k;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align256(bytes);
        return here;
    };
    l.gemv = routes <= kGemvRoutes;
    if (l.gemv) {
        take(routes * inner * 4);
        l.bytes = at;
        return l;
    }
    l.offsets = take(sizeof(int32_t) * (experts + 1));
    l.row_token = take(sizeof(int32_t) * routes);
    l.route_pos = take(sizeof(int32_t) * routes);
    l.counters = take(sizeof(int32_t) * (experts + 2));
    l.act = take(routes * inner);
    l.act_scales = take(routes * (inner / fp8::kGroup) * sizeof(float));
    l.y = take(routes * hidden * (experts_fp8_wide_rows(static_cast<int>(routes)) ? 4 : 2));
    l.bytes = at;
    return l;
}

}  // namespace
}  // namespace lrb

using namespace lrb;

extern "C" uint64_t moe_fp8_wait_limit(uint64_t ns) { return fp8_wait_limit(ns); }

extern "C" int moe_linear_fp8(const uint8_t *x, const float *x_scales, const uint8_t *w, const float *w_scales,
                              int tokens, int rows, int cols, void *out, int out_f32, int32_t *status,
                              void *stream) {
    LRB_REQUIRE(tokens >= 0 && tokens <= (1 << 30) && rows >= 1 && rows <= (1 << 30),
                "moe_linear_fp8: bad tokens %d / rows %d", tokens, rows);
    LRB_REQUIRE(cols >= 16 && cols % 16 == 0 && cols <= (1 << 30),
                "moe_linear_fp8: cols %d must be a positive multiple of 16 up to 2^30", cols);
    LRB_REQUIRE(out_f32 == 0 || out_f32 == 1, "moe_linear_fp8: out_f32 must be 0 or 1");
    if (tokens == 0) return MOE_OK;
    LRB_REQUIRE(x && x_scales && w && w_scales && out, "moe_linear_fp8: null tensor");
    LRB_REQUIRE(on_boundary(x, 16) && on_boundary(w, 16) && on_boundary(out, 16),
                "moe_linear_fp8: x, w and out must be 16-byte aligned");
    LRB_REQUIRE(on_boundary(x_scales, 4) && on_boundary(w_scales, 4) && on_boundary(status, 4),
                "moe_linear_fp8: scales and status must be 4-byte aligned");
    if (int rc = require_sm100()) return rc;
    const LinearFp8 a{x, x_scales, w, w_scales, tokens, rows, cols, out, out_f32};
    if (plan_linear_fp8(tokens, rows, cols).gemv) return launch_linear_fp8_gemv(a, as_stream(stream));
    return launch_linear_fp8_tiles(a, status, as_stream(stream));
}

extern "C" size_t moe_experts_fp8_workspace_bytes(int tokens, int experts, int top_k, int hidden, int inner) {
    if (check_experts(tokens, experts, top_k, hidden, inner) != MOE_OK) return 0;
    // A layout grows with the tokens up to where the next one, perhaps smaller,
    // takes over: the largest of all up to `tokens`.
    size_t bytes = 0;
    for (const int most : {tokens, kGemvRoutes / top_k, kWideRoutes / top_k})
        bytes = std::max(bytes, layout(std::min(tokens, most), experts, top_k, hidden, inner).bytes);
    return bytes;
}

extern "C" int moe_experts_fp8(const uint8_t *x, const float *x_scales, const uint8_t *gate_up,
                               const float *gate_up_scales, const uint8_t *down, const float *down_scales,
                               const int64_t *idx, const uint16_t *weights, int tokens, int experts, int top_k,
                               int hidden, int inner, uint16_t *out, void *workspace, size_t workspace_bytes,
                               int32_t *status, void *stream) {
    if (int rc = check_experts(tokens, experts, top_k, hidden, inner)) return rc;
    if (tokens == 0) return MOE_OK;
    LRB_REQUIRE(x && x_scales && gate_up && gate_up_scales && down && down_scales && idx && weights && out,
                "moe_experts_fp8: null tensor");
    LRB_REQUIRE(on_boundary(x, 16) && on_boundary(gate_up, 16) && on_boundary(down, 16) && on_boundary(out, 16),
                "moe_experts_fp8: x, the banks and out must be 16-byte aligned");
    LRB_REQUIRE(on_boundary(x_scales, 4) && on_boundary(gate_up_scales, 4) && on_boundary(down_scales, 4) && on_boundary(idx, 8) &&
                    on_boundary(weights, 2) && on_boundary(status, 4),
                "moe_experts_fp8: scales, idx, weights and status must be aligned to their elements");
    const Layout l = layout(tokens, experts, top_k, hidden, inner);
    LRB_REQUIRE(workspace && on_boundary(workspace, 256) && workspace_bytes >= l.bytes,
                "moe_experts_fp8: workspace of %zu bytes (256-byte aligned) required", l.bytes);
    if (int rc = require_sm100()) return rc;
    const ExpertsFp8 a{x, x_scales, gate_up, down, gate_up_scales, down_scales, idx, weights, tokens, experts, top_k,
                       hidden, inner, out};
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    if (l.gemv) return launch_experts_fp8_gemv(a, reinterpret_cast<float *>(ws), as_stream(stream));
    auto ints = [&](size_t at) { return reinterpret_cast<int32_t *>(ws + at); };
    ExpertsFp8Scratch s{};
    s.offsets = ints(l.offsets);
    s.row_token = ints(l.row_token);
    s.route_pos = ints(l.route_pos);
    s.counters = ints(l.counters);
    s.act = ws + l.act;
    s.act_scales = reinterpret_cast<float *>(ws + l.act_scales);
    s.y = ws + l.y;
    return launch_experts_fp8_tiles(a, s, status, as_stream(stream));
}
