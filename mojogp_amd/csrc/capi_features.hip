// C ABI: operators of learned features on device arrays (layers.h).
// Declarations are in include/mojogp_amd.h.
#include <cmath>

#include "layers.h"
#include "mojogp_amd.h"

using namespace mgp;

namespace {

constexpr int64_t kMaxWidth = (int64_t)1 << 24;   // columns of a feature matrix
constexpr int64_t kMaxRows = (int64_t)1 << 31;

void check_rows(const char* name, const void* p, int64_t stride, int64_t rows, int64_t width) {
  if (rows == 0) return;
  MGP_REQUIRE(p != nullptr, std::string("null device array ") + name);
  MGP_REQUIRE(rows == 1 || stride >= width,
              std::string("row stride of ") + name + " is below its width");
}

void check_shape(int type, int64_t rows, int64_t width) {
  MGP_REQUIRE(valid_elem(type), "unknown element type");
  MGP_REQUIRE(rows >= 0 && rows < kMaxRows, "rows must be in [0, 2^31)");
  MGP_REQUIRE(width >= 1 && width <= kMaxWidth, "width must be in [1, 2^24]");
}

void check_workspace(const void* ws, int64_t have, size_t need) {
  MGP_REQUIRE(have >= 0 && (size_t)have >= need,
              "workspace of " + std::to_string(have) + " bytes, " + std::to_string(need) +
                  " are needed");
  MGP_REQUIRE(need == 0 || (ws != nullptr && (reinterpret_cast<uintptr_t>(ws) & 255) == 0),
              "the workspace must be 256-byte aligned");
}

NormArgs norm_args(const mgp_layer_norm_t* a) {
  MGP_REQUIRE(a != nullptr, "null arguments");
  check_shape(a->type, a->rows, a->width);
  MGP_REQUIRE(a->param_type == a->type || a->param_type == ELEM_F32,
              "weight and bias must be of the element type or float32");
  MGP_REQUIRE(std::isfinite(a->eps) && a->eps >= 0.0f, "eps must be finite and >= 0");
  check_rows("x", a->x, a->x_stride, a->rows, a->width);
  return {a->type,  a->x,    a->x_stride,
          a->rows,  a->width, a->weight,
          a->bias,  a->param_type == ELEM_F32, a->eps};
}

GatedArgs gated_args(const mgp_gated_layer_t* a) {
  MGP_REQUIRE(a != nullptr, "null arguments");
  check_shape(a->type, a->rows, a->width);
  MGP_REQUIRE(a->hidden >= 1 && a->hidden <= kMaxWidth, "hidden must be in [1, 2^24]");
  MGP_REQUIRE(valid_activation(a->activation), "unknown activation");
  check_rows("x", a->x, a->x_stride, a->rows, a->width);
  check_rows("w_gate", a->w_gate, a->w_gate_stride, a->hidden, a->width);
  check_rows("w_up", a->w_up, a->w_up_stride, a->hidden, a->width);
  return {a->type,   a->activation, a->rows,          a->width, a->hidden,      a->x,
          a->x_stride, a->w_gate,   a->w_gate_stride, a->w_up,  a->w_up_stride, a->b_gate,
          a->b_up};
}

}  // namespace

extern "C" {

int mgp_layer_norm_device(const mgp_layer_norm_t* args, void* y, int64_t y_stride, float* stats,
                          void* stream) {
  return guarded([&] {
    const NormArgs a = norm_args(args);
    check_rows("y", y, y_stride, a.rows, a.width);
    layer_norm(a, y, y_stride, stats, static_cast<hipStream_t>(stream));
  });
}

int mgp_layer_norm_backward_workspace(const mgp_layer_norm_t* args, int64_t* bytes) {
  return guarded([&] {
    MGP_REQUIRE(bytes != nullptr, "null result");
    *bytes = (int64_t)layer_norm_backward_bytes(norm_args(args));
  });
}

int mgp_layer_norm_backward_device(const mgp_layer_norm_t* args, const void* dy,
                                   int64_t dy_stride, const float* stats, void* dx,
                                   int64_t dx_stride, void* dweight, void* dbias,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded([&] {
    const NormArgs a = norm_args(args);
    check_rows("dy", dy, dy_stride, a.rows, a.width);
    MGP_REQUIRE(a.rows == 0 || stats != nullptr, "null statistics");
    if (dx) check_rows("dx", dx, dx_stride, a.rows, a.width);
    if (dweight || dbias) check_workspace(workspace, workspace_bytes, layer_norm_backward_bytes(a));
    layer_norm_backward(a, dy, dy_stride, stats, dx, dx_stride, dweight, dbias, workspace,
                        static_cast<hipStream_t>(stream));
  });
}

int mgp_dropout_device(int type, const void* x, int64_t x_stride, int64_t rows, int64_t width,
                       double rate, uint64_t seed, uint64_t offset, const void* residual,
                       int64_t residual_stride, void* y, int64_t y_stride, void* stream) {
  return guarded([&] {
    check_shape(type, rows, width);
    MGP_REQUIRE(rate >= 0.0 && rate < 1.0, "the dropout rate must be in [0, 1)");
    const double cut = std::nearbyint(rate * 65536.0);  // to even, as Python's round
    MGP_REQUIRE(cut < 65536.0, "the dropout rate rounds to 1 (steps of 2^-16)");
    check_rows("x", x, x_stride, rows, width);
    check_rows("y", y, y_stride, rows, width);
    if (residual) check_rows("residual", residual, residual_stride, rows, width);
    MGP_REQUIRE(offset <= UINT64_MAX - (uint64_t)rows * (uint64_t)width,
                "the draws' numbers pass 64 bits");
    dropout({type, x, x_stride, rows, width, (uint32_t)cut, seed, offset, residual,
             residual_stride},
            y, y_stride, static_cast<hipStream_t>(stream));
  });
}

int mgp_gated_layer_workspace(const mgp_gated_layer_t* args, int backward, int64_t* bytes) {
  return guarded([&] {
    MGP_REQUIRE(bytes != nullptr, "null result");
    *bytes = (int64_t)gated_bytes(gated_args(args), backward != 0);
  });
}

int mgp_gated_layer_device(const mgp_gated_layer_t* args, void* h, int64_t h_stride,
                           void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded([&] {
    const GatedArgs a = gated_args(args);
    check_rows("h", h, h_stride, a.rows, a.hidden);
    if (a.rows == 0) return;
    check_workspace(workspace, workspace_bytes, gated_bytes(a, false));
    gated_forward(a, h, h_stride, workspace, static_cast<hipStream_t>(stream));
  });
}

int mgp_gated_layer_backward_device(const mgp_gated_layer_t* args, const void* dh,
                                    int64_t dh_stride, void* dx, void* dw_gate, void* dw_up,
                                    void* db_gate, void* db_up, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  return guarded([&] {
    const GatedArgs a = gated_args(args);
    check_rows("dh", dh, dh_stride, a.rows, a.hidden);
    if (a.rows > 0) check_workspace(workspace, workspace_bytes, gated_bytes(a, true));
    gated_backward(a, dh, dh_stride, {dx, dw_gate, dw_up, db_gate, db_up}, workspace,
                   static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
