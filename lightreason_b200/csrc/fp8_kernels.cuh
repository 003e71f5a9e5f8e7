// Internal launchers of the FP8 products (fp8_gemv.cu, fp8_tc.cu, fp8_api.cu).
#pragma once

#include "fp8.cuh"
#include "kernels.cuh"

namespace lrb {

// p on a boundary of `a` bytes (a power of two)
inline bool on_boundary(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// out[m, n] = sum over 128-column groups of xs[m, g] * ws[n / 128, g] * (x . w over the group)
struct LinearFp8 {
    const uint8_t *x;        // [tokens, cols] e4m3
    const float *x_scales;   // [tokens, ceil(cols / 128)]
    const uint8_t *w;        // [rows, cols] e4m3
    const float *w_scales;   // [ceil(rows / 128), ceil(cols / 128)]
    int tokens, rows, cols;
    void *out;               // [tokens, rows] BF16 or FP32
    int out_f32;
};

struct ExpertsFp8 {
    const uint8_t *x;                 // [T, H]
    const float *x_scales;            // [T, ceil(H / 128)]
    const uint8_t *gate_up, *down;    // [E, 2I, H], [E, H, I]
    const float *gate_up_scales;      // [E, 2I / 128, ceil(H / 128)]
    const float *down_scales;         // [E, ceil(H / 128), I / 128]
    const int64_t *idx;               // [T, K]; outside [0, E): dropped
    const uint16_t *weights;          // [T, K] BF16
    int tokens, experts, top_k, hidden, inner;
    uint16_t *out;                    // [T, H] BF16
};

constexpr int kGemvTokens = 4;   // tokens that the linear GEMV takes
// Routes up to which the experts take the GEMV kernels, whose weights are read
// once per route (2048 x 512 experts, top-8, us at 1 / 2 / 3 tokens: GEMV 22.7 /
// 36.9 / 49.0, tiles 28.7 / 34.7 / 36.9).
constexpr int kGemvRoutes = 12;
// up to kGemvTokens tokens
int launch_linear_fp8_gemv(const LinearFp8 &a, cudaStream_t stream);
// h: FP32 [T * K, I] scratch
int launch_experts_fp8_gemv(const ExpertsFp8 &a, float *h, cudaStream_t stream);

// The tensor-core path.  status (or null): set to 1 if a bounded wait gave up.
struct ExpertsFp8Scratch {
    int32_t *offsets;    // [E + 1]
    int32_t *row_token;  // [T * K]
    int32_t *route_pos;  // [T, K]
    int32_t *counters;   // [E + 2]: items handed out, per expert the finished parts of gate/up items, a wait gave up
    uint8_t *act;        // [T * K, I]
    float *act_scales;   // [T * K, I / 128]
    void *y;             // [T * K, H], BF16 or (experts_fp8_wide_rows) FP32
};
// Rows of the experts' tiles: 16, 32 (weights as M) or 0 for 128 (rows as M).
int experts_fp8_tile(int routes, int experts);
// Whether a route's down row is kept in FP32 until the weighted sum: up to so
// many routes of a call.
constexpr int kWideRoutes = 2048;
bool experts_fp8_wide_rows(int routes);
// How a plain product is cut: rows of x per tile, CTAs that share a tile's
// columns of x, or the GEMV kernel.
struct LinearFp8Plan {
    int tile, split;
    bool gemv, pair;
};
LinearFp8Plan plan_linear_fp8(int tokens, int rows, int cols);
// Sets the longest that one wait inside the tile kernel may take (ns, for the
// launches from now on); returns what it was.
uint64_t fp8_wait_limit(uint64_t ns);
int launch_linear_fp8_tiles(const LinearFp8 &a, int32_t *status, cudaStream_t stream);
int launch_experts_fp8_tiles(const ExpertsFp8 &a, const ExpertsFp8Scratch &s, int32_t *status, cudaStream_t stream);

}  // namespace lrb
