// The AdamW step over many tensors at once (adamw.hip): what the host knows of
// the tensors, and what a step is.
#pragma once

#include <vector>

#include "layers.h"

namespace mgp {

constexpr int64_t kAdamBlock = 256;   // values of one scale; every tensor's states start at one
constexpr int64_t kAdamChunk = 2048;  // values of a workgroup

struct AdamTensor {
  void* param;
  int64_t size;
  float decay;
};

// Device table: the tensors, then for each workgroup its tensor and which of the
// tensor's chunks is its own.
struct AdamEntry {
  void* param;
  int64_t size;
  int64_t first;  // of its values in the states
  float decay;
  float unused;
};
struct AdamChunk {
  uint32_t tensor, chunk;
};

struct AdamPlan {
  int type, bits;
  bool master_copies;
  double beta1, beta2, eps;
  uint64_t seed;
  void *exp_avg, *exp_avg_sq;              // float, or 8-bit codes
  float *exp_avg_scale, *exp_avg_sq_scale; // [values / 256]
  float* master;
  const void* table;
  std::vector<AdamTensor> tensors;
  std::vector<int64_t> chunk_at;  // first chunk of each tensor, and the end
  int64_t values = 0;             // of the states

  void lay_out();  // chunk_at and values from the tensors
  size_t table_bytes() const {
    return tensors.size() * sizeof(AdamEntry) + (size_t)chunk_at.back() * sizeof(AdamChunk);
  }
  void write_table(void* host) const;
};

struct AdamStep {
  const void* const* grads;  // null: the tensor is left as it is
  int grad_type;             // the parameters' or ELEM_F32
  double grad_scale;
  bool norm;        // whether the norm of all gradients is formed
  double max_norm;  // infinity: none
  float* norm_out;  // or null
  int64_t step;
  const int64_t* step_device;  // or null
  float rate;
  const float* rate_device;  // or null
};
size_t adamw_bytes(const AdamPlan& p, const AdamStep& s);
void adamw_step(const AdamPlan& p, const AdamStep& s, void* ws, hipStream_t st);
void adamw_values(const AdamPlan& p, float* exp_avg, float* exp_avg_sq, hipStream_t st);

}  // namespace mgp
