// C entry point of the products with bf16, MXFP4 or FP8 weights: checks and choice of kernel.
#include <algorithm>
#include <cmath>
#include <limits>

#include "expert_params.h"
#include "../../include/loraforge_amd.h"

namespace lf {
namespace expert {
namespace {

// What the tile kernel can take: MXFP4 x with 16 scales a row and, as an expert's
// weights beside it, within 32-bit offsets; four scales a row beside bf16 x. (What it cannot
// take is streamed, whatever the rows: MXFP4 both, 4096 x 4096 x 480 58 us where k = 512 takes 15.5
// in tiles; 2048 rows gathered from 2^20 + 5 of k = 8192 341 us, from 2^20 - 1 45.)
bool tiles_fit(const lf_expert_product& a) {
  if (a.w_fp8_scales) {  // offsets below 2^31
    const int64_t x_row = a.x_fp8_scales ? a.k : a.x_stride * 2;
    return a.x_rows < (int64_t(1) << 31) / std::max(x_row, a.k) && (a.n + 512) * a.k < (int64_t(1) << 31);
  }
  if (a.x_scales) return a.k >= 512 && std::max(a.x_rows, a.n) * (a.k / 2) < (int64_t(1) << 32);
  return !a.w_scales || a.k >= 128;
}

// The highest tile of so many columns. (Sums of 256 x 256 products leave no registers for a block's of FP8 weights.)
int most_rows(const lf_expert_product& a, int columns) {
  if (!a.w_fp8_scales) return 256;
  return a.x_fp8_scales ? (columns == 256 ? 192 : 256) : columns == 256 ? 128 : 192;
}

// Scales are loaded 16 at a time.
bool rows_fit(const lf_expert_product& a) { return !a.w_scales || a.k >= 512; }

// Times of the kernels in us, fitted to 2586 products (dense ones of 1..4096 rows,
// n 1024..24576, k 1024..8192; 8..128 experts, 1..8192 tokens), every plan of each; with FP8 weights to 1080
// (dense ones of 1..4096 rows, n 528..24576, k 1024..12288; 8..128 experts, 2..32768 choices).
struct Costs {
  struct Tile {
    float fixed, stage, busy;  // of a tile, of a stage (64 k; 256 k of MXFP4 x; 128 k of FP8 weights), and what all CUs at work add to a stage
  } tile[4][4];                // [rows / 64 - 1][columns / 64 - 1]
  struct Rows {
    float fixed, pass, k, k_busy;  // of the launch, of a pass of 16 rows, of 1024 k of it, and what two workgroups on every CU add
  } rows;
  struct Stream {
    float fixed, pass, k, k_tile, k_busy, k_tile_busy;  // the same, with a part for each 16-row tile of a pass (at most 64 rows)
  } stream[2];                                           // [16, 32 columns]
};
constexpr Costs kCosts[5] = {
    // bf16 x and weights
    {{
         {{4.57f, 0.230f, 0.081f}, {5.02f, 0.307f, 0.177f}, {6.20f, 0.395f, 0.230f}, {5.69f, 0.424f, 0.284f}},
         {{5.61f, 0.298f, 0.078f}, {6.10f, 0.363f, 0.194f}, {8.72f, 0.436f, 0.268f}, {8.67f, 0.536f, 0.361f}},
         {{6.14f, 0.399f, 0.087f}, {7.65f, 0.407f, 0.230f}, {12.39f, 0.557f, 0.290f}, {8.45f, 0.769f, 0.468f}},
         {{6.99f, 0.407f, 0.155f}, {9.75f, 0.495f, 0.343f}, {12.54f, 0.725f, 0.466f}, {10.66f, 0.936f, 0.634f}}},
     {1.86f, 0.45f, 3.02f, 18.04f},
     {{1.54f, 1.83f, 0.19f, 0.81f, 0.86f, 1.02f},
      {2.38f, 0.00f, 0.80f, 1.01f, 5.81f, 0.42f}}},
    // bf16 x, MXFP4 weights
    {{
         {{4.65f, 0.310f, 0.046f}, {4.90f, 0.360f, 0.075f}, {6.15f, 0.442f, 0.089f}, {5.67f, 0.472f, 0.132f}},
         {{5.25f, 0.416f, 0.050f}, {5.83f, 0.440f, 0.081f}, {8.72f, 0.572f, 0.084f}, {7.54f, 0.683f, 0.164f}},
         {{6.09f, 0.510f, 0.056f}, {7.26f, 0.556f, 0.098f}, {11.39f, 0.718f, 0.127f}, {9.62f, 0.901f, 0.160f}},
         {{6.87f, 0.504f, 0.103f}, {8.78f, 0.655f, 0.195f}, {15.11f, 0.920f, 0.187f}, {13.46f, 1.123f, 0.358f}}},
     {1.57f, 1.91f, 1.91f, 4.08f},
     {{1.70f, 1.40f, 0.00f, 0.74f, 0.00f, 1.10f},
      {1.52f, 2.01f, 0.20f, 0.84f, 0.24f, 1.30f}}},
    // MXFP4 x and weights
    {{
         {{5.05f, 0.339f, 0.192f}, {5.48f, 0.420f, 0.301f}, {6.37f, 0.526f, 0.351f}, {5.35f, 0.623f, 0.517f}},
         {{5.71f, 0.418f, 0.224f}, {6.30f, 0.494f, 0.293f}, {8.21f, 0.631f, 0.376f}, {6.94f, 0.735f, 0.540f}},
         {{5.87f, 0.543f, 0.232f}, {6.32f, 0.695f, 0.356f}, {10.66f, 0.744f, 0.357f}, {8.62f, 0.935f, 0.444f}},
         {{5.59f, 0.680f, 0.308f}, {7.13f, 0.788f, 0.443f}, {12.74f, 0.884f, 0.394f}, {10.35f, 1.083f, 0.664f}}},
     {2.31f, 1.56f, 1.06f, 4.12f},
     {{1.66f, 1.68f, 0.08f, 0.38f, 0.42f, 0.48f},
      {1.47f, 2.04f, 0.35f, 0.45f, 0.91f, 0.48f}}},
    // bf16 x, FP8 weights (stages of 128 k; no tiles of those heights beside those columns where there is none)
    {{
         {{5.44f, 0.343f, 0.104f}, {6.17f, 0.511f, 0.192f}, {7.00f, 0.630f, 0.257f}, {6.96f, 0.772f, 0.352f}},
         {{4.89f, 0.594f, 0.330f}, {7.88f, 0.712f, 0.339f}, {11.23f, 0.879f, 0.438f}, {10.93f, 1.105f, 0.668f}},
         {{6.25f, 0.780f, 0.275f}, {9.50f, 0.973f, 0.402f}, {13.09f, 1.388f, 0.504f}, {}},
         {{}, {}, {}, {}}},
     {1.99f, 1.56f, 2.52f, 7.29f},
     {{1.30f, 1.81f, 0.00f, 0.79f, 0.00f, 1.19f},
      {1.11f, 2.47f, 0.18f, 0.91f, 0.31f, 1.46f}}},
    // FP8 x and weights
    {{
         {{4.73f, 0.207f, 0.179f}, {5.18f, 0.324f, 0.296f}, {6.33f, 0.424f, 0.399f}, {5.63f, 0.544f, 0.394f}},
         {{4.92f, 0.306f, 0.285f}, {6.37f, 0.438f, 0.385f}, {8.83f, 0.551f, 0.382f}, {8.12f, 0.615f, 0.551f}},
         {{5.79f, 0.414f, 0.286f}, {6.93f, 0.516f, 0.412f}, {11.29f, 0.713f, 0.377f}, {10.54f, 0.854f, 0.453f}},
         {{3.08f, 0.792f, 0.365f}, {6.74f, 0.679f, 0.480f}, {12.08f, 0.979f, 0.332f}, {}}},
     {2.65f, 0.79f, 2.10f, 7.86f},
     {{1.43f, 1.98f, 0.06f, 0.49f, 0.33f, 0.67f},
      {0.95f, 2.65f, 0.30f, 0.62f, 0.77f, 0.65f}}},
};

constexpr double kCus = 256;

// Passes that rows take `cap` at a time: of a dense product, or of experts whose rows
// are spread about their average as popularity spreads them (exponentially).
double passes(double each, double cap, bool grouped) {
  return grouped ? 1.0 / (1.0 - std::exp(-cap / each)) : std::ceil(each / cap);
}

double tile_us(const Costs& c, int rows, int columns, double each, double used, bool grouped, double width, double stages) {
  const double per = passes(each, rows, grouped);
  const double height = std::min(rows / 64.0, std::max(1.0, grouped ? (each / 64.0 + 0.5) / per : std::ceil(std::ceil(each / 64.0) / per)));
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

// The plan of least time. (Against the fastest plan of each of those products: 1.6 to
// 4.8 % slower on average by type, 63 % at most: 256 tokens over 64 experts, n and k 1024, 21 and 13 us.
// Over 80 dense products of 8..384 rows, n 528..8192: 10 % with bf16 x, 6 % with MXFP4 x, 43 % at most.
// FP8 weights: 5 % beside bf16 x, 4 beside FP8 x; 90 % at most: 384 tokens' 768 choices among 32 experts, n 1024, k 2048, 40 and 21 us.)
lf_expert_plan plan_of(const lf_expert_product& a) {
  const Costs& c = kCosts[a.w_fp8_scales ? (a.x_fp8_scales ? 4 : 3) : a.x_scales ? 2 : a.w_scales ? 1 : 0];
  const bool grouped = a.offsets != nullptr && a.experts > 1;
  const double rows = double(a.rows), experts = double(a.experts);
  const double used = grouped ? experts * (1.0 - std::pow(1.0 - 1.0 / experts, rows)) : 1.0;
  const double each = rows / used;  // rows of an expert that has any, on average
  const double n = double(a.n), k = double(a.k) / 1024.0;
  lf_expert_plan best{LF_EXPERT_STREAM, 64, 16};
  double least = std::numeric_limits<double>::infinity();
  // (No plan is faster than the used weights through HBM; of those that are at it, the one with less work.
  // bf16 weights of few rows come at 4.3 TB/s in tiles, 4.9 a wave for 16 of them, 5.5 streamed; FP8 ones at 4.4, 4.6 and 4.9.)
  const double hbm = used * n * double(a.k) * (a.w_scales ? 17.0 / 32.0 : a.w_fp8_scales ? 1.0 : 2.0) * 1e-6;
  auto offer = [&](double us, lf_expert_plan plan) {
    const bool stream = plan.kernel == LF_EXPERT_STREAM, wave = plan.kernel == LF_EXPERT_ROWS;
    const double rate = a.w_fp8_scales ? (stream ? 4.9 : wave ? 4.6 : 4.4) : a.w_scales || stream ? 5.5 : wave ? 4.9 : 4.3;
    us = std::max(us, hbm / rate) + 0.1 * us;
    if (us < least) least = us, best = plan;
  };
  // A dense product may have its rows apart in passes of 16 or 32, so that few weight
  // rows fill the CUs (87 x 528 x 7424: 12 us, in tiles 39; 64 x 2560 x 6144 20 and 28).
  for (int i = 0; i < 2; ++i)
    for (int part = grouped ? 64 : 16; part <= 64; part *= 2) {
      const Costs::Stream& s = c.stream[i];
      const double groups = std::ceil(n / (16 << i)) * used * passes(each, part, grouped) / 512.0, busy = std::min(1.0, groups);
      const double again = grouped ? 0.0 : std::ceil(each / part) - 1.0;  // times that passes read weights that others read
      const double most = std::min(each, double(part));
      const double tiles = grouped ? std::min(4.0, std::max(1.0, each / 16.0 + 0.5)) : most <= 16 ? 1.0 : most <= 32 ? 2.0 : 4.0;
      offer(s.fixed + (s.pass + k * (s.k + s.k_tile * tiles + (s.k_busy + s.k_tile_busy * tiles) * busy)) * std::max(1.0, groups) +
                again * hbm / 5.5,
            {LF_EXPERT_STREAM, part, 16 << i});
    }
  if (rows_fit(a)) {
    const double groups = std::ceil(n / 128.0) * used / 512.0;
    offer(c.rows.fixed + passes(each, 16, grouped) * (c.rows.pass + k * (c.rows.k + c.rows.k_busy * std::min(1.0, groups))) *
                             std::max(1.0, groups),
          {LF_EXPERT_ROWS, 0, 128});
  }
  if (tiles_fit(a)) {
    const double stage_k = a.x_scales ? 256.0 : a.w_fp8_scales ? 128.0 : 64.0;
    for (int height = 64; height <= 256; height += 64)
      for (int columns = 64; columns <= 256; columns += 64)
        if (height <= most_rows(a, columns))
          offer(tile_us(c, height, columns, each, used, grouped, n, std::ceil(double(a.k) / stage_k)), {LF_EXPERT_TILE, height, columns});
  }
  return best;
}

int launch(const lf_expert_product* a, Pair pair, void* stream) {
  LF_REQUIRE(a->rows >= 0 && a->x_rows >= 0 && a->n >= 1 && a->experts >= 1, "sizes must be positive");
  LF_REQUIRE(a->rows < (int64_t(1) << 31) - 65536 && a->x_rows < (int64_t(1) << 31) && a->n < (int64_t(1) << 31) - 65536 &&
                 a->k < (int64_t(1) << 30) - 65536 && a->experts < 65536,
             "sizes must fit signed int32 indexing (of a row's bytes: k below 2^30 - 2^16), experts 65535");
  const bool x_mx = a->x_scales != nullptr, w_mx = a->w_scales != nullptr;
  const bool x_f8 = a->x_fp8_scales != nullptr, w_f8 = a->w_fp8_scales != nullptr;
  LF_REQUIRE(!(x_mx && x_f8) && !(w_mx && w_f8), "an operand has scales of one type");
  LF_REQUIRE(w_mx || !x_mx, "MXFP4 x needs an MXFP4 weight");
  LF_REQUIRE(w_f8 || !x_f8, "FP8 x needs an FP8 weight");
  LF_REQUIRE(a->k >= 1 && a->k % (w_mx ? 32 : w_f8 ? 16 : 8) == 0, "k must be a multiple of 32 (MXFP4 weight), 16 (FP8) or 8 (bf16)");
  LF_REQUIRE(!a->swiglu || !w_f8 || a->n % (2 * lf::fp8::kBlock) == 0, "SwiGLU needs whole blocks of 128 FP8 gate and up rows");
  LF_REQUIRE(!a->swiglu || a->n % 2 == 0, "SwiGLU needs gate and up rows of equal number");
  LF_REQUIRE(a->offsets || (a->experts == 1 && !a->tokens), "offsets required for more than one expert or with tokens");
  if (a->rows == 0) return lf::kOk;
  LF_REQUIRE(a->x && a->w && a->y && a->x_rows > 0, "null pointer argument");
  LF_REQUIRE(a->tokens || a->x_rows >= a->rows, "x must hold a row for each row of the product");
  const int64_t width = a->swiglu ? a->n / 2 : a->n;
  LF_REQUIRE(a->y_stride >= width, "y_stride must cover the output columns");
  LF_REQUIRE(lf::aligned16(a->x) && lf::aligned16(a->w), "x and w must be 16-byte aligned");
  LF_REQUIRE(x_mx || x_f8 || (a->x_stride >= a->k && a->x_stride % 8 == 0), "x rows must be 16-byte aligned");
  lf::expert::Params p{};
  p.x = static_cast<const char*>(a->x);
  p.x_row = x_mx ? a->k / 2 : x_f8 ? a->k : a->x_stride * 2;
  p.xs = a->x_scales;
  p.w = static_cast<const char*>(a->w);
  p.ws = a->w_scales;
  p.xs8 = a->x_fp8_scales;
  p.ws8 = a->w_fp8_scales;
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
  p.pair = pair;
  const lf_expert_plan plan = a->plan ? *a->plan : lf::expert::plan_of(*a);
  auto s = static_cast<hipStream_t>(stream);
  if (plan.kernel == LF_EXPERT_STREAM) {
    LF_REQUIRE(plan.columns == 16 || plan.columns == 32, "stream plan: 16 or 32 columns");
    LF_REQUIRE(plan.rows == 0 || plan.rows == 16 || plan.rows == 32 || plan.rows == 64, "stream plan: 16, 32 or 64 rows (0: 64)");
    return lf::expert::launch_stream(p, plan.rows ? plan.rows : 64, plan.columns / 16, s);
  }
  if (plan.kernel == LF_EXPERT_ROWS) {
    LF_REQUIRE(lf::expert::rows_fit(*a), "this product cannot run with a wave for 16 weight rows");
    return lf::expert::launch_rows(p, s);
  }
  LF_REQUIRE(plan.kernel == LF_EXPERT_TILE && lf::expert::tiles_fit(*a), "this product cannot run in tiles");
  LF_REQUIRE(plan.rows >= 64 && plan.rows <= 256 && plan.rows % 64 == 0, "tile plan: 64, 128, 192 or 256 rows");
  LF_REQUIRE(plan.columns >= 64 && plan.columns <= 256 && plan.columns % 64 == 0, "tile plan: 64, 128, 192 or 256 columns");
  if (w_f8) {
    const int most = lf::expert::most_rows(*a, plan.columns);
    LF_REQUIRE(plan.rows <= most, "tile plan: at most %d rows beside %d columns of FP8 weights", most, int(plan.columns));
    return x_f8 ? lf::expert::launch_tiles_fp8(p, plan.rows, plan.columns, s) : lf::expert::launch_tiles_w8(p, plan.rows, plan.columns, s);
  }
  if (x_mx) return lf::expert::launch_tiles_mx(p, plan.rows, plan.columns, s);
  return w_mx ? lf::expert::launch_tiles_mxw(p, plan.rows, plan.columns, s)
              : lf::expert::launch_tiles_bf16(p, plan.rows, plan.columns, s);
}

}  // namespace

int launch_pairs(const lf_expert_product& a, Pair pair, hipStream_t stream) { return launch(&a, pair, stream); }

}  // namespace expert
}  // namespace lf

extern "C" int lf_expert_linear(const lf_expert_product* a, void* stream) {
  LF_REQUIRE(a != nullptr, "null pointer argument");
  return lf::expert::launch(a, lf::expert::kSingle, stream);
}

extern "C" int lf_expert_linear_plan(const lf_expert_product* a, lf_expert_plan* plan) {
  LF_REQUIRE(a != nullptr && plan != nullptr, "null pointer argument");
  LF_REQUIRE(a->rows >= 1 && a->n >= 1 && a->k >= 8 && a->experts >= 1, "sizes must be positive");
  *plan = lf::expert::plan_of(*a);
  return lf::kOk;
}
