// C entry point of the products with bf16 or MXFP4 weights: checks and choice of kernel.
#include <algorithm>

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

lf_expert_plan plan_of(const lf_expert_product& a) {
  const int64_t used = a.offsets ? std::min(a.experts, a.rows) : 1;
  const int64_t width = a.swiglu ? a.n / 2 : a.n;
  const int64_t each = (a.rows + used - 1) / used;  // rows of an expert, on average
  lf_expert_plan plan{};
  if (each > 32 && tiles_fit(a)) {
    plan.kernel = LF_EXPERT_TILE;
    plan.rows = int32_t(std::min<int64_t>(256, (each + 63) / 64 * 64));
    plan.columns = 256;
    return plan;
  }
  plan.kernel = LF_EXPERT_STREAM;
  const int64_t groups = (width + (a.swiglu ? 7 : 15)) / (a.swiglu ? 8 : 16) * used;
  plan.columns = groups >= 4 * 512 ? 64 : groups >= 2 * 512 ? 32 : 16;
  return plan;
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
    LF_REQUIRE(plan.columns == 16 || plan.columns == 32 || plan.columns == 64, "stream plan: 16, 32 or 64 columns");
    return lf::expert::launch_stream(p, plan.columns / 16, s);
  }
  if (plan.kernel == LF_EXPERT_ROWS) {
    LF_REQUIRE(lf::expert::rows_fit(*a), "this product cannot run with a wave for 16 weight rows");
    return lf::expert::launch_rows(p, s);
  }
  LF_REQUIRE(plan.kernel == LF_EXPERT_TILE && lf::expert::tiles_fit(*a), "this product cannot run in tiles");
  LF_REQUIRE(plan.rows >= 64 && plan.rows <= 256 && plan.rows % 64 == 0, "tile plan: 64, 128, 192 or 256 rows");
  LF_REQUIRE(plan.columns == 128 || plan.columns == 256 || (plan.columns == 64 && !a->swiglu),
             "tile plan: 64 (not with SwiGLU), 128 or 256 columns");
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
