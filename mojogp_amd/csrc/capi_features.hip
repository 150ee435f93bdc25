// C ABI: operators of learned features on device arrays (layers.h).
// Declarations are in include/mojogp_amd.h.
#include <cmath>
#include <numeric>

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

// The bytes an array takes: rows of `width` bytes, `stride` apart.
struct Span {
  const char* name;
  const char* p;
  int64_t rows, width, stride;
};

Span span(const char* name, const void* p, int64_t rows, int64_t width, int64_t stride,
          size_t elem) {
  const int64_t e = (int64_t)elem;
  return {name, static_cast<const char*>(p), p && width > 0 ? rows : 0, width * e,
          (rows == 1 ? width : stride) * e};
}

// Whether two arrays share bytes.  Columns of one table (equal strides) are told
// apart; rows of different strides that may meet are taken to.
bool share(const Span& a, const Span& b) {
  if (a.rows == 0 || b.rows == 0) return false;
  if (a.p > b.p) return share(b, a);
  if (a.p + (a.rows - 1) * a.stride + a.width <= b.p) return false;
  if (a.rows == 1 && b.rows == 1) return true;
  const int64_t step = a.rows == 1   ? b.stride
                       : b.rows == 1 ? a.stride
                                     : std::gcd(a.stride, b.stride);
  const int64_t at = (b.p - a.p) % step;  // of b's columns beside a's
  return at < a.width || at + b.width > step;
}

// A result must not share memory with what the call reads, or (in_place) be that
// array itself.
void check_apart(const Span& out, const Span& in, bool in_place) {
  const bool same = out.p == in.p && out.rows == in.rows && out.width == in.width &&
                    out.stride == in.stride;
  MGP_REQUIRE((in_place && same) || !share(out, in),
              std::string(out.name) + " shares memory with " + in.name);
}

Span row_span(const char* name, const NormArgs& a, const void* p, int64_t stride) {
  return span(name, p, a.rows, a.width, stride, elem_bytes(a.type));
}
Span param_span(const char* name, const NormArgs& a, const void* p) {
  return span(name, p, 1, a.width, a.width, a.f32_params ? 4 : elem_bytes(a.type));
}

void check_apart(const Span& out, const GatedArgs& a) {
  const size_t e = elem_bytes(a.type);
  check_apart(out, span("x", a.x, a.rows, a.width, a.x_stride, e), false);
  check_apart(out, span("w_gate", a.w_gate, a.hidden, a.width, a.w_gate_stride, e), false);
  check_apart(out, span("w_up", a.w_up, a.hidden, a.width, a.w_up_stride, e), false);
  check_apart(out, span("b_gate", a.b_gate, 1, a.hidden, a.hidden, e), false);
  check_apart(out, span("b_up", a.b_up, 1, a.hidden, a.hidden, e), false);
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

GroupArgs group_args(const mgp_group_norm_t* a) {
  MGP_REQUIRE(a != nullptr, "null arguments");
  MGP_REQUIRE(valid_elem(a->type), "unknown element type");
  MGP_REQUIRE(a->activation == -1 || valid_activation(a->activation), "unknown activation");
  MGP_REQUIRE(a->samples >= 0 && a->samples < kMaxRows && a->positions >= 0 &&
                  a->positions < kMaxRows && a->samples * a->positions < kMaxRows,
              "samples, positions and their product must be in [0, 2^31)");
  MGP_REQUIRE(a->channels >= 1 && a->channels <= kMaxWidth, "channels must be in [1, 2^24]");
  MGP_REQUIRE(a->groups >= 1 && a->channels % a->groups == 0,
              "the channels must be a multiple of the groups");
  MGP_REQUIRE(a->param_type == a->type || a->param_type == ELEM_F32,
              "weight and bias must be of the element type or float32");
  MGP_REQUIRE(std::isfinite(a->eps) && a->eps >= 0.0f, "eps must be finite and >= 0");
  check_rows("x", a->x, a->x_stride, a->samples * a->positions, a->channels);
  return {a->type,          a->activation,   a->x,      a->x_stride, a->samples, a->positions,
          (int)a->channels, (int)a->groups, a->weight, a->bias,     a->param_type == ELEM_F32,
          a->eps};
}

Span row_span(const char* name, const GroupArgs& a, const void* p, int64_t stride) {
  return span(name, p, a.samples * a.positions, a.channels, stride, elem_bytes(a.type));
}
Span param_span(const char* name, const GroupArgs& a, const void* p) {
  return span(name, p, 1, a.channels, a.channels, a.f32_params ? 4 : elem_bytes(a.type));
}
void check_codes(const char* name, const void* p, int64_t stride, int64_t rows, int64_t width) {
  if (rows == 0) return;
  MGP_REQUIRE(p != nullptr, std::string("null device array ") + name);
  MGP_REQUIRE(aligned16(p) && stride % 16 == 0 && stride >= round_up(width, 16) &&
                  stride < ((int64_t)1 << 23),
              std::string("rows of ") + name +
                  " must be 16-byte aligned, below 8 MB and hold the width rounded up to 16");
}

Int8Args int8_args(const mgp_int8_layer_t* a) {
  MGP_REQUIRE(a != nullptr, "null arguments");
  check_shape(a->type, a->rows, a->width);
  MGP_REQUIRE(a->width <= kInt8Width, "8-bit rows have at most 131072 columns");
  MGP_REQUIRE(a->hidden >= 1 && a->hidden <= kMaxWidth, "hidden must be in [1, 2^24]");
  const bool gated = a->w_up != nullptr;
  MGP_REQUIRE(valid_activation(a->activation) || (a->activation == -1 && !gated),
              "unknown activation");
  check_rows("x", a->x, a->x_stride, a->rows, a->width);
  check_codes("w_gate", a->w_gate, a->w_stride, a->hidden, a->width);
  MGP_REQUIRE(a->s_gate != nullptr && (a->s_up != nullptr) == gated, "null scales");
  if (gated) check_codes("w_up", a->w_up, a->w_stride, a->hidden, a->width);
  return {a->type,
          a->activation,
          a->rows,
          a->width,
          a->hidden,
          a->x,
          a->x_stride,
          static_cast<const int8_t*>(a->w_gate),
          static_cast<const int8_t*>(a->w_up),
          a->w_stride,
          a->s_gate,
          a->s_up,
          a->b_gate,
          gated ? a->b_up : nullptr};
}

void check_pairs(const float* stats) {
  MGP_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7) == 0, "the statistics must be 8-byte aligned");
}
Span stats_span(const GroupArgs& a, const void* p) {
  const int64_t n = 2 * a.samples * a.groups;
  return span("stats", p, a.positions ? 1 : 0, n, n, sizeof(float));
}

}  // namespace

extern "C" {

int mgp_layer_norm_device(const mgp_layer_norm_t* args, void* y, int64_t y_stride, float* stats,
                          void* stream) {
  return guarded([&] {
    const NormArgs a = norm_args(args);
    check_rows("y", y, y_stride, a.rows, a.width);
    const Span out = row_span("y", a, y, y_stride);
    const Span moments = span("stats", stats, 1, 2 * a.rows, 2 * a.rows, sizeof(float));
    check_apart(out, row_span("x", a, a.x, a.x_stride), true);
    check_apart(moments, row_span("x", a, a.x, a.x_stride), false);
    check_apart(moments, out, false);
    for (const Span& q : {param_span("weight", a, a.weight), param_span("bias", a, a.bias)}) {
      check_apart(out, q, false);
      check_apart(moments, q, false);
    }
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
    const Span of_dy = row_span("dy", a, dy, dy_stride), of_x = row_span("x", a, a.x, a.x_stride);
    const Span of_dx = row_span("dx", a, dx, dx_stride);
    check_apart(of_dx, of_dy, true);
    check_apart(of_dx, of_x, true);
    for (const Span& out : {of_dx, param_span("dweight", a, dweight),
                            param_span("dbias", a, dbias)}) {
      if (out.name != of_dx.name) {
        check_apart(out, of_dy, false);
        check_apart(out, of_x, false);
      }
      check_apart(out, param_span("weight", a, a.weight), false);
      check_apart(out, span("stats", stats, 1, 2 * a.rows, 2 * a.rows, sizeof(float)), false);
    }
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
    const size_t e = elem_bytes(type);
    const Span out = span("y", y, rows, width, y_stride, e);
    check_apart(out, span("x", x, rows, width, x_stride, e), true);
    check_apart(out, span("residual", residual, rows, width, residual_stride, e), true);
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
    check_apart(span("h", h, a.rows, a.hidden, h_stride, elem_bytes(a.type)), a);
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
    const size_t e = elem_bytes(a.type);
    for (const Span& out : {span("dx", dx, a.rows, a.width, a.width, e),
                            span("dw_gate", dw_gate, a.hidden, a.width, a.width, e),
                            span("dw_up", dw_up, a.hidden, a.width, a.width, e),
                            span("db_gate", db_gate, 1, a.hidden, a.hidden, e),
                            span("db_up", db_up, 1, a.hidden, a.hidden, e)}) {
      check_apart(out, a);
      check_apart(out, span("dh", dh, a.rows, a.hidden, dh_stride, e), false);
    }
    gated_backward(a, dh, dh_stride, {dx, dw_gate, dw_up, db_gate, db_up}, workspace,
                   static_cast<hipStream_t>(stream));
  });
}

int mgp_group_norm_workspace(const mgp_group_norm_t* args, int backward, int64_t* bytes) {
  return guarded([&] {
    MGP_REQUIRE(bytes != nullptr, "null result");
    *bytes = (int64_t)group_norm_bytes(group_args(args), backward != 0);
  });
}

int mgp_group_norm_device(const mgp_group_norm_t* args, void* y, int64_t y_stride, float* stats,
                          void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded([&] {
    const GroupArgs a = group_args(args);
    check_rows("y", y, y_stride, a.samples * a.positions, a.channels);
    const Span out = row_span("y", a, y, y_stride), moments = stats_span(a, stats);
    const Span of_x = row_span("x", a, a.x, a.x_stride);
    check_pairs(stats);
    check_apart(out, of_x, true);
    check_apart(moments, of_x, false);
    check_apart(moments, out, false);
    for (const Span& q : {param_span("weight", a, a.weight), param_span("bias", a, a.bias)}) {
      check_apart(out, q, false);
      check_apart(moments, q, false);
    }
    check_workspace(workspace, workspace_bytes, group_norm_bytes(a, false));
    group_norm(a, y, y_stride, stats, workspace, static_cast<hipStream_t>(stream));
  });
}

int mgp_group_norm_backward_device(const mgp_group_norm_t* args, const void* dy,
                                   int64_t dy_stride, const float* stats, void* dx,
                                   int64_t dx_stride, void* dweight, void* dbias,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded([&] {
    const GroupArgs a = group_args(args);
    const int64_t rows = a.samples * a.positions;
    check_rows("dy", dy, dy_stride, rows, a.channels);
    MGP_REQUIRE(rows == 0 || stats != nullptr, "null statistics");
    check_pairs(stats);
    if (dx) check_rows("dx", dx, dx_stride, rows, a.channels);
    const Span of_dy = row_span("dy", a, dy, dy_stride), of_x = row_span("x", a, a.x, a.x_stride);
    const Span of_dx = row_span("dx", a, dx, dx_stride);
    const Span of_dw = param_span("dweight", a, dweight), of_db = param_span("dbias", a, dbias);
    check_apart(of_dx, of_dy, true);
    check_apart(of_dx, of_x, true);
    for (const Span& out : {of_dx, of_dw, of_db}) {
      if (out.name != of_dx.name) {
        check_apart(out, of_dy, false);
        check_apart(out, of_x, false);
        check_apart(out, of_dx, false);
      }
      check_apart(out, param_span("weight", a, a.weight), false);
      check_apart(out, param_span("bias", a, a.bias), false);
      check_apart(out, stats_span(a, stats), false);
    }
    check_apart(of_dw, of_db, false);
    check_workspace(workspace, workspace_bytes, group_norm_bytes(a, true));
    group_norm_backward(a, dy, dy_stride, stats, dx, dx_stride, dweight, dbias, workspace,
                        static_cast<hipStream_t>(stream));
  });
}

int mgp_int8_quantize_device(int type, const void* x, int64_t x_stride, int64_t rows,
                             int64_t width, void* codes, int64_t codes_stride, float* scales,
                             void* stream) {
  return guarded([&] {
    check_shape(type, rows, width);
    MGP_REQUIRE(width <= kInt8Width, "8-bit rows have at most 131072 columns");
    check_rows("x", x, x_stride, rows, width);
    check_codes("codes", codes, codes_stride, rows, width);
    MGP_REQUIRE(rows == 0 || scales != nullptr, "null scales");
    const Span of_x = span("x", x, rows, width, x_stride, elem_bytes(type));
    const Span of_codes = span("codes", codes, rows, round_up(width, 16), codes_stride, 1);
    const Span of_scales = span("scales", scales, 1, rows, rows, sizeof(float));
    check_apart(of_codes, of_x, false);
    check_apart(of_scales, of_x, false);
    check_apart(of_codes, of_scales, false);
    int8_quantize(type, x, x_stride, rows, width, static_cast<int8_t*>(codes), codes_stride,
                  scales, static_cast<hipStream_t>(stream));
  });
}

int mgp_int8_layer_workspace(const mgp_int8_layer_t* args, int64_t* bytes) {
  return guarded([&] {
    MGP_REQUIRE(bytes != nullptr, "null result");
    *bytes = (int64_t)int8_bytes(int8_args(args));
  });
}

int mgp_int8_layer_device(const mgp_int8_layer_t* args, void* y, int64_t y_stride,
                          void* workspace, int64_t workspace_bytes, void* stream) {
  return guarded([&] {
    const Int8Args a = int8_args(args);
    check_rows("y", y, y_stride, a.rows, a.hidden);
    if (a.rows == 0) return;
    const size_t e = elem_bytes(a.type);
    const int64_t pad = round_up(a.width, 16);
    const Span out = span("y", y, a.rows, a.hidden, y_stride, e);
    for (const Span& in : {span("x", a.x, a.rows, a.width, a.x_stride, e),
                           span("w_gate", a.w_gate, a.hidden, pad, a.w_stride, 1),
                           span("w_up", a.w_up, a.hidden, pad, a.w_stride, 1),
                           span("s_gate", a.s_gate, 1, a.hidden, a.hidden, sizeof(float)),
                           span("s_up", a.s_up, 1, a.hidden, a.hidden, sizeof(float)),
                           span("b_gate", a.b_gate, 1, a.hidden, a.hidden, e),
                           span("b_up", a.b_up, 1, a.hidden, a.hidden, e)})
      check_apart(out, in, false);
    check_workspace(workspace, workspace_bytes, int8_bytes(a));
    int8_layer(a, y, y_stride, workspace, static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
