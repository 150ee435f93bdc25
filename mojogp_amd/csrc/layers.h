// Operators of learned features (the layers in front of a kernel): layer norm,
// gated layers and dropout over device arrays the caller holds, in float32,
// bfloat16 and float16, on the caller's stream, without host synchronisation.
#pragma once

#include "mgp_common.h"

namespace mgp {

// Element types (part of the C ABI).
enum ElemType : int { ELEM_F32 = 0, ELEM_BF16 = 1, ELEM_F16 = 2 };
inline bool valid_elem(int t) { return t >= ELEM_F32 && t <= ELEM_F16; }
inline size_t elem_bytes(int t) { return t == ELEM_F32 ? 4 : 2; }

// Activations of the gated layer (part of the C ABI).
enum Activation : int { ACT_SILU = 0, ACT_GELU = 1, ACT_SIGMOID = 2, ACT_RELU = 3 };
inline bool valid_activation(int a) { return a >= ACT_SILU && a <= ACT_RELU; }

template <class T>
struct alignas(16) Vec16 {  // 16 bytes of elements
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};

// Runs f with a value of the element type's C++ type.
template <class F>
void dispatch_elem(int type, F&& f) {
  switch (type) {
    case ELEM_F32: f(float{}); break;
    case ELEM_BF16: f(__bf16{}); break;
    default: f(_Float16{}); break;
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// y = (x - mean) rstd w + b per row; stats[rows][2] = mean, rstd (or null).
struct NormArgs {
  int type;
  const void* x;
  int64_t x_stride;
  int64_t rows, width;
  const void* weight;  // [width] or null (ones), of the element type or float32
  const void* bias;    // [width] or null (zeros), as weight
  bool f32_params;
  float eps;
};
void layer_norm(const NormArgs& a, void* y, int64_t y_stride, float* stats, hipStream_t st);
// Bytes of the backward pass' workspace (block partials of dweight and dbias).
size_t layer_norm_backward_bytes(const NormArgs& a);
// dweight, dbias may be null (of the parameters' type otherwise); dx too.
void layer_norm_backward(const NormArgs& a, const void* dy, int64_t dy_stride, const float* stats,
                         void* dx, int64_t dx_stride, void* dweight, void* dbias, void* ws,
                         hipStream_t st);

// y = act((x - mean) rstd w + b), mean and rstd over a sample's positions and the
// channels of a group; x's row of sample n and position l is n positions + l.
// stats[samples][groups][2] = mean, rstd (or null).
struct GroupArgs {
  int type;
  int activation;  // or -1: none
  const void* x;
  int64_t x_stride;
  int64_t samples, positions;
  int channels, groups;
  const void* weight;  // [channels] or null (ones), of the element type or float32
  const void* bias;    // [channels] or null (zeros), as weight
  bool f32_params;
  float eps;
};
size_t group_norm_bytes(const GroupArgs& a, bool backward);
void group_norm(const GroupArgs& a, void* y, int64_t y_stride, float* stats, void* ws,
                hipStream_t st);
// dx, dweight and dbias may be null; of x's and the parameters' types.
void group_norm_backward(const GroupArgs& a, const void* dy, int64_t dy_stride, const float* stats,
                         void* dx, int64_t dx_stride, void* dweight, void* dbias, void* ws,
                         hipStream_t st);

// y = residual + x keep / (1 - rate), keep from draw offset + (row width + col).
struct DropoutArgs {
  int type;
  const void* x;
  int64_t x_stride;
  int64_t rows, width;
  uint32_t cut;  // kept where the 16-bit draw is at least this (0..65535)
  uint64_t seed;
  uint64_t offset;
  const void* residual;  // or null
  int64_t residual_stride;
};
void dropout(const DropoutArgs& a, void* y, int64_t y_stride, hipStream_t st);

struct GatedArgs {
  int type, activation;
  int64_t rows, width, hidden;
  const void* x;
  int64_t x_stride;
  const void* w_gate;
  int64_t w_gate_stride;
  const void* w_up;
  int64_t w_up_stride;
  const void* b_gate;  // [hidden] or null
  const void* b_up;
};
size_t gated_bytes(const GatedArgs& a, bool backward);
void gated_forward(const GatedArgs& a, void* h, int64_t h_stride, void* ws, hipStream_t st);
struct GatedGrads {  // contiguous, any may be null
  void *dx, *dw_gate, *dw_up, *db_gate, *db_up;
};
void gated_backward(const GatedArgs& a, const void* dh, int64_t dh_stride, const GatedGrads& g,
                    void* ws, hipStream_t st);

// Rows in 8-bit integers: codes[rows][codes_stride] (zeros from width up to the next
// multiple of 16) and a scale for each.
void int8_quantize(int type, const void* x, int64_t x_stride, int64_t rows, int64_t width,
                   int8_t* codes, int64_t codes_stride, float* scales, hipStream_t st);

// A layer whose weights are such rows; w_up null: act(x Wg^T + bg), otherwise times
// x Wu^T + bu.
struct Int8Args {
  int type, activation;  // of x, biases and the result; -1: none
  int64_t rows, width, hidden;
  const void* x;
  int64_t x_stride;
  const int8_t *w_gate, *w_up;
  int64_t w_stride;
  const float *s_gate, *s_up;
  const void *b_gate, *b_up;  // [hidden] or null
};
constexpr int64_t kInt8Width = 131072;  // 127^2 of so many are below 2^31
size_t int8_bytes(const Int8Args& a);
void int8_layer(const Int8Args& a, void* y, int64_t y_stride, void* ws, hipStream_t st);

}  // namespace mgp
