// C entry point of the products with bf16 or MXFP4 weights: checks and choice of kernel.
#include "expert_params.h"
#include "../../include/loraforge_amd.h"

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
  return lf::expert::launch_stream(p, static_cast<hipStream_t>(stream));
}
