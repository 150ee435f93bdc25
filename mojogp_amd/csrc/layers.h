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

}  // namespace mgp
