// C entry point of the products with bf16 or MXFP4 weights: checks and choice of kernel.
#include <algorithm>
#include <cmath>
#include <limits>

#include "expert_params.h"
#include "../../include/loraforge_amd.h"

namespace lf {
namespace expert {
namespace {

// What the tile kernel can take: MXFP4 x with 16 scales a row and, as an expert's
// weights beside it, within 32-bit offsets; four scales a row beside bf16 x.
bool tiles_fit(const lf_expert_product& a) {
  if (a.x_scales) return a.k >= 512 && std::max(a.x_rows, a.n) * (a.k / 2) < (int64_t(1) << 32);
  return !a.w_scales || a.k >= 128;
}

// Scales are loaded 16 at a time.
bool rows_fit(const lf_expert_product& a) { return !a.w_scales || a.k >= 512; }

// Times of the kernels in us, fitted to 2586 products (dense ones of 1..4096 rows,
// n 1024..24576, k 1024..8192; 8..128 experts, 1..8192 tokens), every plan of each.
struct Costs {
  struct Tile {
    float fixed, stage, busy;  // of a tile, of a stage (64 k; 256 k of MXFP4 x), and what all CUs at work add to a stage
  } tile[4][4];                // [rows / 64 - 1][columns / 64 - 1]
  struct Rows {
    float fixed, pass, k, k_busy;  // of the launch, of a pass of 16 rows, of 1024 k of it, and what two workgroups on every CU add
  } rows;
  struct Stream {
    float fixed, pass, k, k_tile, k_busy, k_tile_busy;  // the same, with a part for each 16-row tile of a pass (at most 64 rows)
  } stream[2];                                           // [16, 32 columns]
};
constexpr Costs kCosts[3] = {
    // bf16 x and weights
    {{
         {{4.63f, 0.241f, 0.077f}, {5.00f, 0.323f, 0.171f}, {6.31f, 0.415f, 0.214f}, {5.61f, 0.433f, 0.265f}},
         {{5.61f, 0.321f, 0.076f}, {6.02f, 0.367f, 0.181f}, {8.71f, 0.437f, 0.249f}, {8.34f, 0.541f, 0.324f}},
         {{6.27f, 0.423f, 0.074f}, {7.25f, 0.418f, 0.212f}, {12.50f, 0.546f, 0.267f}, {7.93f, 0.773f, 0.428f}},
         {{6.92f, 0.401f, 0.152f}, {9.45f, 0.494f, 0.321f}, {12.35f, 0.729f, 0.438f}, {10.18f, 0.934f, 0.588f}}},
     {1.74f, 0.49f, 3.02f, 18.08f},
     {{1.55f, 1.81f, 0.20f, 0.80f, 0.84f, 1.04f},
      {2.39f, 0.00f, 0.81f, 1.00f, 5.77f, 0.45f}}},
    // bf16 x, MXFP4 weights
    {{
         {{4.62f, 0.311f, 0.051f}, {4.83f, 0.363f, 0.076f}, {6.19f, 0.456f, 0.085f}, {5.67f, 0.474f, 0.134f}},
         {{5.27f, 0.431f, 0.047f}, {5.73f, 0.445f, 0.079f}, {8.63f, 0.570f, 0.082f}, {7.56f, 0.686f, 0.152f}},
         {{6.12f, 0.527f, 0.058f}, {7.12f, 0.562f, 0.097f}, {11.34f, 0.721f, 0.116f}, {9.36f, 0.904f, 0.145f}},
         {{6.75f, 0.512f, 0.106f}, {8.74f, 0.661f, 0.172f}, {15.07f, 0.922f, 0.138f}, {13.36f, 1.136f, 0.275f}}},
     {1.57f, 1.91f, 1.90f, 4.11f},
     {{1.70f, 1.40f, 0.00f, 0.73f, 0.00f, 1.11f},
      {1.48f, 2.02f, 0.20f, 0.84f, 0.24f, 1.30f}}},
    // MXFP4 x and weights
    {{
         {{5.03f, 0.339f, 0.198f}, {5.43f, 0.431f, 0.301f}, {6.33f, 0.542f, 0.361f}, {5.39f, 0.630f, 0.524f}},
         {{5.73f, 0.432f, 0.220f}, {6.25f, 0.501f, 0.296f}, {8.10f, 0.637f, 0.370f}, {7.04f, 0.731f, 0.541f}},
         {{5.87f, 0.555f, 0.242f}, {6.32f, 0.685f, 0.375f}, {10.43f, 0.744f, 0.354f}, {8.60f, 0.937f, 0.430f}},
         {{5.46f, 0.695f, 0.306f}, {7.15f, 0.788f, 0.441f}, {12.95f, 0.882f, 0.373f}, {10.37f, 1.087f, 0.625f}}},
     {2.30f, 1.56f, 1.06f, 4.08f},
     {{1.62f, 1.70f, 0.08f, 0.38f, 0.40f, 0.48f},
      {1.44f, 2.08f, 0.35f, 0.45f, 0.86f, 0.49f}}},
};

constexpr double kCus = 256;

// Passes that rows take `cap` at a time: of a dense product, or of experts whose rows
// are spread about their average as popularity spreads them (exponentially).
double passes(double each, double cap, bool grouped) {
  return grouped ? 1.0 / (1.0 - std::exp(-cap / each)) : std::ceil(each / cap);
}

double tile_us(const Costs& c, int rows, int columns, double each, double used, bool grouped, double width, double stages) {
  const double per = passes(each, rows, grouped);
  const double height = std::min(rows / 64.0, std::max(1.0, grouped ? each / per / 64.0 + 0.5 : std::ceil(std::ceil(each / per) / 64.0)));
  const int low = std::min(3, int(height)), high = std::min(4, low + 1), j = columns / 64 - 1;
  const double part = height - low;
  auto mix = [&](float Costs::Tile::*m) { return (1.0 - part) * (c.tile[low - 1][j].*m) + part * (c.tile[high - 1][j].*m); };
  const double fixed = mix(&Costs::Tile::fixed), stage = mix(&Costs::Tile::stage), busy = mix(&Costs::Tile::busy);
  const double tiles = used * per * std::ceil(width / columns);
  if (tiles <= kCus) return fixed + stages * (stage + busy * tiles / kCus);
  constexpr double kLaunch = 3.0;
  const double round = fixed - kLaunch + stages * (stage + busy);
  if (grouped) return kLaunch + (tiles / kCus + 0.5) * round;
  const double full = std::floor(tiles / kCus), rest = tiles / kCus - full;
  return kLaunch + full * round + (rest > 0 ? fixed - kLaunch + stages * (stage + busy * rest) : 0.0);
}

// The plan of least time. (Against the fastest plan of each of those products: 1.8 to
// 4.7 % slower on average by type, 61 % at most: 3 rows, n and k 1024, 7.1 and 4.4 us.)
lf_expert_plan plan_of(const lf_expert_product& a) {
  const Costs& c = kCosts[a.x_scales ? 2 : a.w_scales ? 1 : 0];
  const bool grouped = a.offsets != nullptr && a.experts > 1;
  const double rows = double(a.rows), experts = double(a.experts);
  const double used = grouped ? experts * (1.0 - std::pow(1.0 - 1.0 / experts, rows)) : 1.0;
  const double each = rows / used;  // rows of an expert that has any, on average
  const double n = double(a.n), k = double(a.k) / 1024.0;
  lf_expert_plan best{LF_EXPERT_STREAM, 0, 16};
  double least = std::numeric_limits<double>::infinity();
  // (No plan is faster than the used weights through HBM; of those that are at it, the one with less work.
  // bf16 weights of few rows come at 4.3 TB/s in tiles, 4.9 a wave for 16 of them, 5.5 streamed.)
  const double hbm = used * n * double(a.k) * (a.w_scales ? 17.0 / 32.0 : 2.0) * 1e-6;
  auto offer = [&](double us, lf_expert_plan plan) {
    const double rate = a.w_scales || plan.kernel == LF_EXPERT_STREAM ? 5.5 : plan.kernel == LF_EXPERT_ROWS ? 4.9 : 4.3;
    us = std::max(us, hbm / rate) + 0.1 * us;
    if (us < least) least = us, best = plan;
  };
  for (int i = 0; i < 2; ++i) {
    const Costs::Stream& s = c.stream[i];
    const double groups = std::ceil(n / (16 << i)) * used / 512.0, busy = std::min(1.0, groups);
    const double tiles = std::min(4.0, grouped ? std::max(1.0, each / 16.0 + 0.5) : each <= 16 ? 1.0 : each <= 32 ? 2.0 : 4.0);
    offer(s.fixed + passes(each, 64, grouped) * (s.pass + k * (s.k + s.k_tile * tiles + (s.k_busy + s.k_tile_busy * tiles) * busy)) *
                        std::max(1.0, groups),
          {LF_EXPERT_STREAM, 0, 16 << i});
  }
  if (rows_fit(a)) {
    const double groups = std::ceil(n / 128.0) * used / 512.0;
    offer(c.rows.fixed + passes(each, 16, grouped) * (c.rows.pass + k * (c.rows.k + c.rows.k_busy * std::min(1.0, groups))) *
                             std::max(1.0, groups),
          {LF_EXPERT_ROWS, 0, 128});
  }
  if (tiles_fit(a)) {
    const double stage_k = a.x_scales ? 256.0 : 64.0;
    for (int height = 64; height <= 256; height += 64)
      for (int columns = 64; columns <= 256; columns += 64)
        offer(tile_us(c, height, columns, each, used, grouped, n, std::ceil(double(a.k) / stage_k)), {LF_EXPERT_TILE, height, columns});
  }
  return best;
}

}  // namespace
}  // namespace expert
}  // namespace lf

extern "C" int lf_expert_linear(const lf_expert_product* a, void* stream) {
  LF_REQUIRE(a != nullptr, "null pointer argument");
  LF_REQUIRE(a->rows >= 0 && a->x_rows >= 0 && a->n >= 1 && a->experts >= 1, "sizes must be positive");
  LF_REQUIRE(a->rows < (int64_t(1) << 31) - 65536 && a->x_rows < (int64_t(1) << 31) && a->n < (int64_t(1) << 31) - 65536 &&
                 a->k < (int64_t(1) << 31) - 65536 && a->experts < 65536,
             "sizes must fit signed int32 indexing, experts 65535");
  const bool x_mx = a->x_scales != nullptr, w_mx = a->w_scales != nullptr;
  LF_REQUIRE(w_mx || !x_mx, "MXFP4 x needs an MXFP4 weight");
  LF_REQUIRE(a->k >= 1 && a->k % (w_mx ? 32 : 8) == 0, "k must be a multiple of 32 (MXFP4 weight) or 8 (bf16)");
  LF_REQUIRE(!a->swiglu || a->n % 2 == 0, "SwiGLU needs gate and up rows of equal number");
  LF_REQUIRE(a->offsets || (a->experts == 1 && !a->tokens), "offsets required for more than one expert or with tokens");
  if (a->rows == 0) return lf::kOk;
  LF_REQUIRE(a->x && a->w && a->y && a->x_rows > 0, "null pointer argument");
  LF_REQUIRE(a->tokens || a->x_rows >= a->rows, "x must hold a row for each row of the product");
  const int64_t width = a->swiglu ? a->n / 2 : a->n;
  LF_REQUIRE(a->y_stride >= width, "y_stride must cover the output columns");
  LF_REQUIRE(lf::aligned16(a->x) && lf::aligned16(a->w), "x and w must be 16-byte aligned");
  LF_REQUIRE(x_mx || (a->x_stride >= a->k && a->x_stride % 8 == 0), "x rows must be 16-byte aligned");
  lf::expert::Params p{};
  p.x = static_cast<const char*>(a->x);
  p.x_row = x_mx ? a->k / 2 : a->x_stride * 2;
  p.xs = a->x_scales;
  p.w = static_cast<const char*>(a->w);
  p.ws = a->w_scales;
  p.bias = a->bias;
  p.offsets = a->offsets;
  p.tokens = a->tokens;
  p.y = a->y;
  p.y_stride = a->y_stride;
  p.rows = int(a->rows);
  p.x_rows = int(a->x_rows);
  p.n = int(a->n);
  p.k = int(a->k);
  p.experts = int(a->experts);
  p.width = int(width);
  p.swiglu = a->swiglu ? 1 : 0;
  p.y_vec = lf::aligned16(a->y) && a->y_stride % 8 == 0;
  const lf_expert_plan plan = a->plan ? *a->plan : lf::expert::plan_of(*a);
  auto s = static_cast<hipStream_t>(stream);
  if (plan.kernel == LF_EXPERT_STREAM) {
    LF_REQUIRE(plan.columns == 16 || plan.columns == 32, "stream plan: 16 or 32 columns");
    return lf::expert::launch_stream(p, plan.columns / 16, s);
  }
  if (plan.kernel == LF_EXPERT_ROWS) {
    LF_REQUIRE(lf::expert::rows_fit(*a), "this product cannot run with a wave for 16 weight rows");
    return lf::expert::launch_rows(p, s);
  }
  LF_REQUIRE(plan.kernel == LF_EXPERT_TILE && lf::expert::tiles_fit(*a), "this product cannot run in tiles");
  LF_REQUIRE(plan.rows >= 64 && plan.rows <= 256 && plan.rows % 64 == 0, "tile plan: 64, 128, 192 or 256 rows");
  LF_REQUIRE(plan.columns >= 64 && plan.columns <= 256 && plan.columns % 64 == 0, "tile plan: 64, 128, 192 or 256 columns");
  if (x_mx) return lf::expert::launch_tiles_mx(p, plan.rows, plan.columns, s);
  return w_mx ? lf::expert::launch_tiles_mxw(p, plan.rows, plan.columns, s)
              : lf::expert::launch_tiles_bf16(p, plan.rows, plan.columns, s);
}

extern "C" int lf_expert_linear_plan(const lf_expert_product* a, lf_expert_plan* plan) {
  LF_REQUIRE(a != nullptr && plan != nullptr, "null pointer argument");
  LF_REQUIRE(a->rows >= 1 && a->n >= 1 && a->k >= 8 && a->experts >= 1, "sizes must be positive");
  *plan = lf::expert::plan_of(*a);
  return lf::kOk;
}
