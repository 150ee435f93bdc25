// The AdamW step over many tensors in one launch, with states in 32 or in 8 bits.
//
//   g = grad scale c, c = min(1, max_norm / |all grads scale|)
//   m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2
//   p = p (1 - rate decay) - rate (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// HBM bound: every value is read and written once; a workgroup takes 2048 values of
// one tensor, so that hundreds of tensors of any size are one launch.  The tensors
// lie in a table on the device; the gradients, which are new arrays every step, come as
// a launch's arguments (up to kGrads of them), without a copy to the device.
//
// 8-bit states: 256 values of a tensor share a scale, one wave's four values a lane.
// m is an OCP e4m3 value times scale (largest |m| / 448), v one of 5 exponent and 3
// mantissa bits without sign (largest 1.875, smallest 2^-33) times its own.  Both are
// rounded up with the probability of what lies above the code below, by 16 bits each of
// a counter-based word a value: rounded to nearest, v, which moves by a thousandth of
// itself a step where its codes lie an eighth apart, would not move at all.  A v above
// zero keeps code 1 at least: over the root of a zero, m's last bit would be a huge
// step.  What a code becomes is decided on 64-bit values (its place among 2^16
// draws leaves fp32 no digits), the step itself in fp32 from m and v before their
// rounding.
#include "adamw.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "philox.h"

namespace mgp {

namespace {

constexpr int kGrads = 400;  // gradients a launch: 3200 of 4096 bytes of arguments
constexpr int kNormBlocks = 256, kNormThreads = 1024;

struct Grads {
  const void* at[kGrads];
};

// What the kernels share of a step, formed on the device where the norm or the
// device's own step and rate are part of it.
struct Scalars {
  double factor;   // of the gradients
  float c1, c2;    // 1 / (1 - b1^t), 1 / (1 - b2^t)
  float rate;
  int skip;        // the norm is not finite: nothing is changed
};

// Four elements at any alignment, of which `left` exist; zeros past them.
template <class T>
struct Four {
  T v[4];
};
template <class T>
__device__ __forceinline__ Four<T> load4(const T* p, int64_t left) {
  Four<T> a;
  if (left >= 4) {
    __builtin_memcpy(&a, p, sizeof(a));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) a.v[k] = k < left ? p[k] : (T)0.0f;
  }
  return a;
}
template <class T>
__device__ __forceinline__ void store4(T* p, int64_t left, const float* v) {
  Four<T> a;
#pragma unroll
  for (int k = 0; k < 4; ++k) a.v[k] = (T)v[k];
  if (left >= 4) {
    __builtin_memcpy(p, &a, sizeof(a));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < left) p[k] = a.v[k];
  }
}

// ---------------------------------------------------------------- norm of the gradients

// part[block]: the sum of squares of a block's chunks, in 64 bits
template <class G>
__global__ __launch_bounds__(kNormThreads) void k_adamw_norm(Grads grads,
                                                             const AdamEntry* __restrict__ entries,
                                                             const AdamChunk* __restrict__ chunks,
                                                             uint32_t first, uint32_t count,
                                                             uint32_t tensor0,
                                                             double* __restrict__ part) {
  __shared__ double red[kNormThreads / 64];
  double s = 0.0;
  // two chunks of 2048 a round
  for (uint32_t c = blockIdx.x * 2 + (threadIdx.x >> 9); c < count; c += gridDim.x * 2) {
    const uint32_t at = __builtin_amdgcn_readfirstlane(first + c);
    const uint32_t t = __builtin_amdgcn_readfirstlane(chunks[at].tensor);
    const G* g = static_cast<const G*>(grads.at[t - tensor0]);
    if (g == nullptr) continue;
    const int64_t i = (int64_t)chunks[at].chunk * kAdamChunk + 4 * (threadIdx.x & 511);
    const Four<G> a = load4(g + i, entries[t].size - i);
#pragma unroll
    for (int k = 0; k < 4; ++k) s = fma((double)(float)a.v[k], (double)(float)a.v[k], s);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
#pragma unroll
  for (int w = 1; w < kNormThreads / 64; ++w) s += red[w];
  part[blockIdx.x] = s;
}

struct ScalarArgs {
  const double* part;
  int parts;  // 0: no norm
  double grad_scale, max_norm;
  float* norm_out;
  double beta1, beta2;
  int64_t step;
  const int64_t* step_device;
  float rate;
  const float* rate_device;
  Scalars* out;
};

__global__ __launch_bounds__(256) void k_adamw_scalars(ScalarArgs a) {
  __shared__ double red[4];
  double s = 0.0;
  for (int i = threadIdx.x; i < a.parts; i += 256) s += a.part[i];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  Scalars r;
  const double norm = sqrt(red[0] + red[1] + red[2] + red[3]) * fabs(a.grad_scale);
  r.factor = a.grad_scale * (norm > a.max_norm ? a.max_norm / norm : 1.0);
  r.skip = !(norm < HUGE_VAL);
  const double t = (double)(a.step_device ? *a.step_device : a.step);
  r.c1 = (float)(1.0 / (1.0 - pow(a.beta1, t)));
  r.c2 = (float)(1.0 / (1.0 - pow(a.beta2, t)));
  r.rate = a.rate_device ? *a.rate_device : a.rate;
  *a.out = r;
  if (a.norm_out) *a.norm_out = (float)norm;
}

// ---------------------------------------------------------------- 8-bit states

// x >= 0 in units of the scale -> code: 3 mantissa bits, exponents from LOWEST on
// (the field of 2^LOWEST is 1), evenly spaced below; rounded up where the cut-off
// part and (draw + 1/2) / 2^16 of a code's step pass the step.  In a double's high word
// a step is 2^17; below 2^LOWEST the value is brought into that binade first.
template <int LOWEST>
__device__ __forceinline__ int code_of(double x, uint32_t draw, int most) {
  constexpr double kLow = LOWEST == -6 ? 0x1p-6 : 0x1p-30;
  static_assert(LOWEST == -6 || LOWEST == -30, "");
  const bool low = x < kLow;
  const double y = low ? x + kLow : x;
  const uint32_t high = (uint32_t)(__double_as_longlong(y) >> 32);
  const int code = (int)((high + 2 * draw + 1) >> 17) - ((LOWEST + 1022) << 3) - (low ? 8 : 0);
  return min(code, most);
}

// Largest of 64 lanes, of the bits of |value|: NaN is above infinity.
__device__ __forceinline__ uint32_t wave_largest(uint32_t u) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) u = max(u, (uint32_t)__shfl_xor((int)u, o));
  return u;
}

// The scale of a block and the factor of its values, from the largest of them.
// Blocks that end below 2^-120 (whose factor would pass fp32) are held as zeros.
struct Scale {
  float scale, by;
};
__device__ __forceinline__ Scale scale_of(uint32_t largest, float top, float inv_top) {
  const float a = __uint_as_float(largest);
  const bool none = largest < 0x03800000u;  // 2^-120
  return {none ? 0.0f : a * inv_top, none ? 0.0f : top / a};
}

// b x + r y, every operation rounded: a scale is the fp32 rounding of the largest of
// these, and sums of 8-bit gradients and means come to lie on its ties, where a
// fused addition would make another scale of some than the formula does.
__device__ __forceinline__ double mean_of(double b, double x, double r, double y) {
#pragma clang fp contract(off)
  return b * x + r * y;
}

constexpr float kTopM = 448.0f, kTopV = 1.875f;

__device__ __forceinline__ float value_m(uint32_t codes, int k) {
  return k == 0   ? __builtin_amdgcn_cvt_f32_fp8(codes, 0)
         : k == 1 ? __builtin_amdgcn_cvt_f32_fp8(codes, 1)
         : k == 2 ? __builtin_amdgcn_cvt_f32_fp8(codes, 2)
                  : __builtin_amdgcn_cvt_f32_fp8(codes, 3);
}
__device__ __forceinline__ float value_v(uint32_t codes, int k) {
  // exponent field and mantissa where fp32 has them, subnormal codes included
  return __uint_as_float((codes >> (8 * k) & 0xffu) << 20) * 0x1p96f;
}

// ---------------------------------------------------------------- the step

struct StepArgs {
  const AdamEntry* entries;
  const AdamChunk* chunks;
  uint32_t first, tensor0;
  void *exp_avg, *exp_avg_sq;
  float *exp_avg_scale, *exp_avg_sq_scale;
  float* master;
  double b1, b2;
  float eps;
  uint64_t seed;
  int64_t step;
  const int64_t* step_device;
  Scalars host;
  const Scalars* device;  // or null: host's
};

template <class P, class G, bool EIGHT, bool MASTER>
__global__ __launch_bounds__(256) void k_adamw(Grads grads, StepArgs a) {
  constexpr int U = (int)(kAdamChunk / 1024);
  const AdamChunk ck = a.chunks[a.first + blockIdx.x];
  const AdamEntry e = a.entries[ck.tensor];
  const G* __restrict__ g = static_cast<const G*>(grads.at[ck.tensor - a.tensor0]);
  if (g == nullptr) return;
  const Scalars s = a.device ? *a.device : a.host;
  if (s.skip) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // a wave's blocks of 256 lie side by side
  const int64_t i0 = (int64_t)ck.chunk * kAdamChunk + wave * 256 + 4 * lane;
  P* __restrict__ param = static_cast<P*>(e.param);
  float* __restrict__ master = a.master + e.first;

  Four<G> gr[U];
  Four<P> pr[U];
  Four<float> wr[U], mr[U], vr[U];
  uint32_t mc[U], vc[U];
  float ms[U], vs[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = i0 + u * 1024, left = e.size - i;
    gr[u] = load4(g + i, left);
    if constexpr (MASTER)
      wr[u] = load4(master + i, left);
    else
      pr[u] = load4(param + i, left);
    if constexpr (EIGHT) {
      // the padding of a tensor's last block is there to be read and written
      const int64_t b = (e.first + i) >> 8;
      const bool in = (i & ~(int64_t)255) < e.size;
      mc[u] = in ? *reinterpret_cast<const uint32_t*>(static_cast<uint8_t*>(a.exp_avg) + e.first + i) : 0u;
      vc[u] = in ? *reinterpret_cast<const uint32_t*>(static_cast<uint8_t*>(a.exp_avg_sq) + e.first + i) : 0u;
      ms[u] = in ? a.exp_avg_scale[b] : 0.0f;
      vs[u] = in ? a.exp_avg_sq_scale[b] : 0.0f;
    } else {
      mr[u] = load4(static_cast<const float*>(a.exp_avg) + e.first + i, left);
      vr[u] = load4(static_cast<const float*>(a.exp_avg_sq) + e.first + i, left);
    }
  }
  const float keep = 1.0f - s.rate * e.decay;
  uint64_t t = 0;
  if constexpr (EIGHT) t = (uint64_t)(a.step_device ? *a.step_device : a.step);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = i0 + u * 1024, left = e.size - i;
    if ((i & ~(int64_t)255) >= e.size) continue;  // (of the whole wave)
    float m[4], v[4];
    if constexpr (EIGHT) {
      double md[4], vd[4];
      uint32_t mu = 0, vu = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const double gd = (double)(float)gr[u].v[k] * s.factor;
        md[k] = mean_of(a.b1, (double)value_m(mc[u], k) * (double)ms[u], 1.0 - a.b1, gd);
        vd[k] = mean_of(a.b2, (double)value_v(vc[u], k) * (double)vs[u], 1.0 - a.b2, gd * gd);
        if (k >= left) md[k] = vd[k] = 0.0;
        m[k] = (float)md[k];
        v[k] = (float)vd[k];
        mu = max(mu, __float_as_uint(m[k]) & 0x7fffffffu);
        vu = max(vu, __float_as_uint(v[k]) & 0x7fffffffu);
      }
      const Scale sm = scale_of(wave_largest(mu), kTopM, 1.0f / kTopM);
      const Scale sv = scale_of(wave_largest(vu), kTopV, 1.0f / kTopV);
      const Draws dr = philox((uint64_t)(e.first + i) >> 2, a.seed, t);
      uint32_t cm = 0, cv = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int x = code_of<-6>(fabs(md[k]) * (double)sm.by, dr.w[k] & 0xffffu, 126);
        int y = code_of<-30>(vd[k] * (double)sv.by, dr.w[k] >> 16, 255);
        if (vd[k] > 0.0 && sv.by > 0.0f) y = max(y, 1);
        cm |= (uint32_t)(x | (md[k] < 0.0 ? 128 : 0)) << (8 * k);
        cv |= (uint32_t)y << (8 * k);
      }
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.exp_avg) + e.first + i) = cm;
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.exp_avg_sq) + e.first + i) = cv;
      if (lane == 0) {
        a.exp_avg_scale[(e.first + i) >> 8] = sm.scale;
        a.exp_avg_sq_scale[(e.first + i) >> 8] = sv.scale;
      }
    } else {
      const float b1 = (float)a.b1, b2 = (float)a.b2;
      const float r1 = (float)(1.0 - a.b1), r2 = (float)(1.0 - a.b2), factor = (float)s.factor;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float x = (float)gr[u].v[k] * factor;
        m[k] = fmaf(b1, mr[u].v[k], r1 * x);
        v[k] = fmaf(b2, vr[u].v[k], r2 * (x * x));
      }
      store4(static_cast<float*>(a.exp_avg) + e.first + i, left, m);
      store4(static_cast<float*>(a.exp_avg_sq) + e.first + i, left, v);
    }
    float p[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      // v_sqrt_f32 and v_rcp_f32 are off by one unit in the last place of a step
      const float root = __builtin_amdgcn_sqrtf(v[k] * s.c2) + a.eps;
      const float update = m[k] * s.c1 * __builtin_amdgcn_rcpf(root);
      const float w = MASTER ? wr[u].v[k] : (float)pr[u].v[k];
      p[k] = fmaf(w, keep, -s.rate * update);
    }
    if constexpr (MASTER) store4(master + i, left, p);
    store4(param + i, left, p);
  }
}

// Values of 8-bit states, four a thread.
__global__ __launch_bounds__(256) void k_adamw_values(const uint32_t* __restrict__ m,
                                                      const float* __restrict__ ms,
                                                      const uint32_t* __restrict__ v,
                                                      const float* __restrict__ vs, int64_t quads,
                                                      float* __restrict__ out_m,
                                                      float* __restrict__ out_v) {
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < quads;
       q += (int64_t)gridDim.x * 256) {
    const uint32_t cm = m[q], cv = v[q];
    const float sm = ms[q >> 6], sv = vs[q >> 6];
    Four<float> a, b;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      a.v[k] = value_m(cm, k) * sm;
      b.v[k] = value_v(cv, k) * sv;
    }
    __builtin_memcpy(out_m + 4 * q, &a, sizeof(a));
    __builtin_memcpy(out_v + 4 * q, &b, sizeof(b));
  }
}

}  // namespace

// ---------------------------------------------------------------- host side

void AdamPlan::lay_out() {
  chunk_at.assign(1, 0);
  values = 0;
  for (const AdamTensor& t : tensors) {
    chunk_at.push_back(chunk_at.back() + ceil_div(t.size, kAdamChunk));
    values += round_up(t.size, kAdamBlock);
  }
}

void AdamPlan::write_table(void* host) const {
  AdamEntry* e = static_cast<AdamEntry*>(host);
  AdamChunk* c = reinterpret_cast<AdamChunk*>(e + tensors.size());
  int64_t first = 0;
  for (size_t t = 0; t < tensors.size(); ++t) {
    *e++ = {tensors[t].param, tensors[t].size, first, tensors[t].decay, 0.0f};
    first += round_up(tensors[t].size, kAdamBlock);
    for (int64_t k = chunk_at[t]; k < chunk_at[t + 1]; ++k)
      *c++ = {(uint32_t)t, (uint32_t)(k - chunk_at[t])};
  }
}

namespace {

inline bool on_device(const AdamStep& s) { return s.norm || s.step_device || s.rate_device; }
inline int64_t groups(const AdamPlan& p) { return ceil_div((int64_t)p.tensors.size(), (int64_t)kGrads); }

// Runs f(first tensor, the gradients, first chunk, chunks) for up to kGrads tensors
// at a time.
template <class F>
void for_groups(const AdamPlan& p, const AdamStep& s, F&& f) {
  const int64_t n = (int64_t)p.tensors.size();
  for (int64_t t0 = 0; t0 < n; t0 += kGrads) {
    const int64_t t1 = std::min(t0 + kGrads, n);
    Grads g{};
    std::copy(s.grads + t0, s.grads + t1, g.at);
    const int64_t c0 = p.chunk_at[t0], count = p.chunk_at[t1] - c0;
    f((uint32_t)t0, g, (uint32_t)c0, (uint32_t)count);
  }
}

template <class P, class G, bool EIGHT, bool MASTER>
void launch_step(const AdamPlan& p, const AdamStep& s, StepArgs a, hipStream_t st) {
  for_groups(p, s, [&](uint32_t t0, const Grads& g, uint32_t c0, uint32_t count) {
    if (count == 0) return;
    a.first = c0;
    a.tensor0 = t0;
    k_adamw<P, G, EIGHT, MASTER><<<count, 256, 0, st>>>(g, a);
  });
}

}  // namespace

size_t adamw_bytes(const AdamPlan& p, const AdamStep& s) {
  if (!on_device(s)) return 0;
  return 256 + (s.norm ? (size_t)groups(p) * kNormBlocks * sizeof(double) : 0);
}

void adamw_step(const AdamPlan& p, const AdamStep& s, void* ws, hipStream_t st) {
  const AdamEntry* entries = static_cast<const AdamEntry*>(p.table);
  const AdamChunk* chunks = reinterpret_cast<const AdamChunk*>(entries + p.tensors.size());
  const bool wide = s.grad_type == ELEM_F32;
  Scalars* scalars = nullptr;
  if (on_device(s)) {
    scalars = static_cast<Scalars*>(ws);
    double* part = reinterpret_cast<double*>(static_cast<char*>(ws) + 256);
    if (s.norm) {
      dispatch_elem(s.grad_type, [&](auto tag) {
        int64_t at = 0;
        for_groups(p, s, [&](uint32_t t0, const Grads& g, uint32_t c0, uint32_t count) {
          k_adamw_norm<decltype(tag)><<<kNormBlocks, kNormThreads, 0, st>>>(
              g, entries, chunks, c0, count, t0, part + at);
          at += kNormBlocks;
        });
      });
    }
    k_adamw_scalars<<<1, 256, 0, st>>>({part, s.norm ? (int)(groups(p) * kNormBlocks) : 0,
                                        s.grad_scale, s.max_norm, s.norm_out, p.beta1, p.beta2,
                                        s.step, s.step_device, s.rate, s.rate_device, scalars});
  }
  StepArgs a{entries,
             chunks,
             0,
             0,
             p.exp_avg,
             p.exp_avg_sq,
             p.exp_avg_scale,
             p.exp_avg_sq_scale,
             p.master,
             p.beta1,
             p.beta2,
             (float)p.eps,
             p.seed,
             s.step,
             s.step_device,
             {s.grad_scale, (float)(1.0 / (1.0 - std::pow(p.beta1, (double)s.step))),
              (float)(1.0 / (1.0 - std::pow(p.beta2, (double)s.step))), s.rate, 0},
             scalars};
  dispatch_elem(p.type, [&](auto tag) {
    using P = decltype(tag);
    auto with = [&](auto grad, auto eight) {
      using G = decltype(grad);
      if constexpr (sizeof(P) == 2) {
        if (p.master_copies) return launch_step<P, G, eight.value, true>(p, s, a, st);
      }
      launch_step<P, G, eight.value, false>(p, s, a, st);
    };
    auto of = [&](auto eight) {
      if constexpr (sizeof(P) == 2) {
        if (wide) return with(float{}, eight);
      }
      with(P{}, eight);
    };
    if (p.bits == 8)
      of(std::true_type{});
    else
      of(std::false_type{});
  });
  MGP_HIP_CHECK(hipGetLastError());
}

void adamw_values(const AdamPlan& p, float* exp_avg, float* exp_avg_sq, hipStream_t st) {
  const int64_t quads = p.values / 4;
  if (quads == 0) return;
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(quads, (int64_t)256), 16384);
  k_adamw_values<<<grid, 256, 0, st>>>(static_cast<const uint32_t*>(p.exp_avg), p.exp_avg_scale,
                                       static_cast<const uint32_t*>(p.exp_avg_sq),
                                       p.exp_avg_sq_scale, quads, exp_avg, exp_avg_sq);
  MGP_HIP_CHECK(hipGetLastError());
}

}  // namespace mgp
