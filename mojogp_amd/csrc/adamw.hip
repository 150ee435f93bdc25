// The AdamW step over many tensors in one launch, with states in 32 or in 8 bits.
//
//   g = grad scale c, c = min(1, max_norm / |all grads scale|)
//   m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2
//   p = p (1 - rate decay) - rate (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// HBM bound: every value is read and written once; a workgroup takes 2048 values of
// one tensor, so that hundreds of tensors of any size are one launch.  The tensors
// lie in a table on the device; the gradients, which are new arrays every step, come as
// a launch's arguments (up to kGrads of them), without a copy to the device.  On 67 million
// fp32 values the step takes 325 us in 32 bits (5.8 TB/s, part of the gradients from the
// last-level cache, where the norm has left them), 214 us in 8 bits
// (5.0 TB/s at 16 bytes), where the instructions for quotients, codes and draws hardly hide
// behind the memory; the norm 84 us.
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
constexpr int kNormBlocks = 2048;

struct Grads {
  const void* at[kGrads];
};

// What the kernels share of a step, formed on the device where the norm or the
// device's own step and rate are part of it.
struct Scalars {
  double factor;   // of the gradients
  float c1, c2;    // 1 / (1 - b1^t), 1 / (1 - b2^t)
  float rate;
  int skip;        // the norm is not finite, or step or rate is none: nothing is changed
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

// part[block]: the sum of squares of a block's chunks, in 64 bits.  Four chunks a round,
// their loads all out before the first is used.
template <class G>
__global__ __launch_bounds__(256) void k_adamw_norm(Grads grads,
                                                    const AdamEntry* __restrict__ entries,
                                                    const AdamChunk* __restrict__ chunks,
                                                    uint32_t first, uint32_t count,
                                                    uint32_t tensor0, double* __restrict__ part) {
  constexpr int U = 4, P = (int)(kAdamChunk / 1024);
  __shared__ double red[4];
  double s = 0.0;
  for (uint32_t c = blockIdx.x * U; c < count; c += gridDim.x * U) {
    Four<G> a[U][P];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const AdamChunk ck = chunks[first + min(c + u, count - 1)];
      const G* g = static_cast<const G*>(grads.at[ck.tensor - tensor0]);
      const int64_t i = (int64_t)ck.chunk * kAdamChunk + 4 * threadIdx.x;
      const int64_t size = g && c + u < count ? entries[ck.tensor].size : 0;
#pragma unroll
      for (int p = 0; p < P; ++p) a[u][p] = load4(g + i + p * 1024, size - i - p * 1024);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const double x = (double)(float)a[u][p].v[k];
          s = fma(x, x, s);
        }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

struct ScalarArgs {
  const double* part;
  int parts;  // 0: no norm, and its fields are not read
  double grad_scale, max_norm;
  float* norm_out;
  double beta1, beta2;
  const int64_t* step_device;
  const float* rate_device;
  Scalars host;
  Scalars* out;
};

__global__ __launch_bounds__(256) void k_adamw_scalars(ScalarArgs a) {
  __shared__ double red[4];
  double s = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < a.parts; i += 256) s += a.part[i];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  Scalars r = a.host;
  if (a.parts > 0) {
    const double norm = sqrt(red[0] + red[1] + red[2] + red[3]) * fabs(a.grad_scale);
    r.factor = a.grad_scale * (norm > a.max_norm ? a.max_norm / norm : 1.0);
    r.skip = !((float)norm < HUGE_VALF);
    if (a.norm_out) *a.norm_out = (float)norm;
  }
  if (a.step_device) {
    const int64_t step = *a.step_device;
    const double t = (double)step;
    r.skip |= step < 1;
    r.c1 = (float)(1.0 / (1.0 - pow(a.beta1, t)));
    r.c2 = (float)(1.0 / (1.0 - pow(a.beta2, t)));
  }
  if (a.rate_device) {
    r.rate = *a.rate_device;
    r.skip |= !(r.rate >= 0.0f && r.rate < HUGE_VALF);
  }
  *a.out = r;
}

// ---------------------------------------------------------------- 8-bit states

// x >= 0 in units of the scale -> code: 3 mantissa bits, exponents from LOWEST on
// (the field of 2^LOWEST is 1), evenly spaced below; rounded up where the cut-off
// part and (draw + 1/2) / 2^16 of a code's step pass the step.  In a double's high word
// a step is 2^17; below 2^LOWEST the value is brought into that binade first.
// twice: 2 draw.
template <int LOWEST>
__device__ __forceinline__ int code_of(double x, uint32_t twice, int most) {
  constexpr double kLow = LOWEST == -6 ? 0x1p-6 : 0x1p-30;
  static_assert(LOWEST == -6 || LOWEST == -30, "");
  constexpr uint32_t kField = (uint32_t)(LOWEST + 1022) << 20;
  const bool low = x < kLow;
  const uint32_t high = (uint32_t)(__double_as_longlong(low ? x + kLow : x) >> 32);
  return min((int)((high + (twice + (low ? 1u - kField - (8u << 17) : 1u - kField))) >> 17), most);
}

// Largest of 64 lanes, of the bits of |value| (NaN is above infinity): within rows of
// 16 lanes, then across them, to lane 63.
__device__ __forceinline__ uint32_t wave_largest(uint32_t u) {
  auto other = [](uint32_t v, auto control, auto rows) __attribute__((always_inline)) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, control.value, rows.value, 0xf, false);
  };
  using std::integral_constant;
  u = max(u, other(u, integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{}));
  u = max(u, other(u, integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{}));
  u = max(u, other(u, integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{}));
  u = max(u, other(u, integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{}));
  u = max(u, other(u, integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{}));
  u = max(u, other(u, integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{}));
  return (uint32_t)__builtin_amdgcn_readlane((int)u, 63);
}

// A block's scale is the fp32 rounding of the 64-bit quotient largest / top, and a code is
// decided by the 64-bit quotient of a value and that scale.  A 32-bit factor in the place
// of either quotient makes another last place of half the scales and moves a code in two
// million by a step.

// largest / top in fp32, of the largest of a lane's values: the lanes' largest is the
// block's, as roundings keep the order.  The quotient in 64 bits is that of a division (by
// 7 or 15 times a power of two no quotient lies near enough to a tie for the correction
// to miss it).  Blocks that end below 2^-120 are held as zeros.
__device__ __forceinline__ float scale_from(double largest, double top) {
  const double inv = 1.0 / top;
  double q = largest * inv;
  q = fma(fma(-q, top, largest), inv, q);
  return largest < 0x1p-120 ? 0.0f : (float)q;
}

// A block's scale from its lanes'; one that is not in fp32 is NaN.
__device__ __forceinline__ float wave_scale(float lane_scale) {
  const uint32_t u = wave_largest(__float_as_uint(lane_scale) & 0x7fffffffu);
  return __uint_as_float(u < 0x7f800000u ? u : 0x7fc00000u);
}

// x / scale in 64 bits; inv is the reciprocal to within a few last places.  (No quotient of
// 53 by 24 bits lies within 2^-25 of a last place from a tie.)
__device__ __forceinline__ double over(double x, double scale, double inv) {
  const double q = x * inv;
  return fma(fma(-q, scale, x), inv, q);
}

// 1 / x by the approximation of v_rcp_f64, squared away twice.
__device__ __forceinline__ double reciprocal(double x) {
  double r = __builtin_amdgcn_rcp(x);
  r = fma(fma(-x, r, 1.0), r, r);
  return fma(fma(-x, r, 1.0), r, r);
}

__device__ __forceinline__ double lane_value(double x, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// b x + r y, every operation rounded: sums of 8-bit gradients and means come to lie on
// the ties of their scales' roundings, where a fused addition would make another scale of
// some than the formula does.
__device__ __forceinline__ double mean_of(double b, double x, double r, double y) {
#pragma clang fp contract(off)
  return b * x + r * y;
}

constexpr double kTopM = 448.0, kTopV = 1.875;

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

// What a workgroup works on: the arrays of its chunk of a tensor.
template <class P, class G>
struct ChunkAt {
  const G* g;
  P* param;
  float *master, *m, *v;      // 32-bit states
  uint8_t *mc, *vc;           // 8-bit ones
  float *ms, *vs;
  int64_t first;              // of the chunk's values in the states
  int left;                   // values of the tensor from the chunk's first on, up to a chunk
  float keep;                 // 1 - rate decay
};

// FULL: none of the chunk's values is past the tensor's end.
template <class P, class G, bool EIGHT, bool MASTER, bool FULL>
__device__ __forceinline__ void step_chunk(const ChunkAt<P, G>& c, const StepArgs& a,
                                           const Scalars& s, uint64_t t) {
  constexpr int U = (int)(kAdamChunk / 1024);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Four<G> gr[U];
  Four<P> pr[U];
  Four<float> wr[U], mr[U], vr[U];
  uint32_t mc[U], vc[U];
  float ms[U], vs[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i0 = u * 1024 + wave * 256, i = i0 + 4 * lane;
    const int left = FULL ? 4 : c.left - i;
    gr[u] = load4(c.g + i, left);
    if constexpr (MASTER)
      wr[u] = load4(c.master + i, left);
    else
      pr[u] = load4(c.param + i, left);
    if constexpr (EIGHT) {
      // the padding of a tensor's last block is there to be read and written
      const bool in = FULL || i0 < c.left;
      mc[u] = in ? *reinterpret_cast<const uint32_t*>(c.mc + i) : 0u;
      vc[u] = in ? *reinterpret_cast<const uint32_t*>(c.vc + i) : 0u;
      ms[u] = in ? c.ms[i0 >> 8] : 0.0f;
      vs[u] = in ? c.vs[i0 >> 8] : 0.0f;
    } else {
      mr[u] = load4(c.m + i, left);
      vr[u] = load4(c.v + i, left);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i0 = u * 1024 + wave * 256, i = i0 + 4 * lane;
    const int left = FULL ? 4 : c.left - i;
    if (!FULL && i0 >= c.left) continue;
    float m[4], v[4];
    if constexpr (EIGHT) {
      double md[4], vd[4];
      double gd[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) gd[k] = (double)(float)gr[u].v[k];
      if (s.factor != 1.0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) gd[k] *= s.factor;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        md[k] = mean_of(a.b1, (double)value_m(mc[u], k) * (double)ms[u], 1.0 - a.b1, gd[k]);
        vd[k] = mean_of(a.b2, (double)value_v(vc[u], k) * (double)vs[u], 1.0 - a.b2, gd[k] * gd[k]);
        if (!FULL && k >= left) md[k] = vd[k] = 0.0;
        m[k] = (float)md[k];
        v[k] = (float)vd[k];
      }
      // the largest; and what is not finite, which a maximum may pass over, by a sum
      const double lm = fmax(fmax(fabs(md[0]), fabs(md[1])), fmax(fabs(md[2]), fabs(md[3])));
      const double lv = fmax(fmax(vd[0], vd[1]), fmax(vd[2], vd[3]));
      const double am = (md[0] + md[1]) + (md[2] + md[3]), av = (vd[0] + vd[1]) + (vd[2] + vd[3]);
      const float qm = scale_from(fma(am, 0.0, lm), kTopM), qv = scale_from(fma(av, 0.0, lv), kTopV);
      const float sm = wave_scale(qm), sv = wave_scale(qv);
      // both reciprocals at once, m's by the first 32 lanes; of a block of zeros, what is
      // left over a scale of one is below every draw's border
      const float sm1 = sm > 0.0f ? sm : 1.0f, sv1 = sv > 0.0f ? sv : 1.0f;
      const double inv = reciprocal((double)(lane < 32 ? sm1 : sv1));
      const double im = lane_value(inv, 0), iv = lane_value(inv, 63);
      const int least = sv > 0.0f ? 1 : 0;  // of a v above zero
      const Draws dr = philox((uint64_t)(c.first + i) >> 2, a.seed, t);
      uint32_t cm = 0, cv = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int x = code_of<-6>(over(fabs(md[k]), (double)sm1, im), (dr.w[k] & 0xffffu) << 1, 126);
        const uint32_t sign = (uint32_t)(__double_as_longlong(md[k]) >> 56) & 128u;
        const int y = code_of<-30>(over(vd[k], (double)sv1, iv), dr.w[k] >> 16 << 1, 255);
        cm |= ((uint32_t)x | sign) << (8 * k);
        cv |= (uint32_t)max(y, vd[k] > 0.0 ? least : 0) << (8 * k);
      }
      *reinterpret_cast<uint32_t*>(c.mc + i) = cm;
      *reinterpret_cast<uint32_t*>(c.vc + i) = cv;
      if (lane == 0) {
        c.ms[i0 >> 8] = sm;
        c.vs[i0 >> 8] = sv;
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
      store4(c.m + i, left, m);
      store4(c.v + i, left, v);
    }
    float p[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      // v_sqrt_f32 and v_rcp_f32 are off by one unit in the last place of a step
      const float root = __builtin_amdgcn_sqrtf(v[k] * s.c2) + a.eps;
      const float update = m[k] * s.c1 * __builtin_amdgcn_rcpf(root);
      const float w = MASTER ? wr[u].v[k] : (float)pr[u].v[k];
      p[k] = fmaf(w, c.keep, -s.rate * update);
      // a value in fp32: rounded to float16 together with the sum, a parameter would not
      // always be what its master copy rounds to
      asm("" : "+v"(p[k]));
    }
    if constexpr (MASTER) store4(c.master + i, left, p);
    store4(c.param + i, left, p);
  }
}

template <class P, class G, bool EIGHT, bool MASTER>
__global__ __launch_bounds__(256) void k_adamw(Grads grads, StepArgs a) {
  const AdamChunk ck = a.chunks[a.first + blockIdx.x];
  const AdamEntry e = a.entries[ck.tensor];
  const G* g = static_cast<const G*>(grads.at[ck.tensor - a.tensor0]);
  if (g == nullptr) return;
  const Scalars s = a.device ? *a.device : a.host;
  if (s.skip) return;
  const int64_t at = (int64_t)ck.chunk * kAdamChunk, first = e.first + at;
  uint64_t t = 0;
  ChunkAt<P, G> c;
  c.g = g + at;
  c.param = static_cast<P*>(e.param) + at;
  if constexpr (MASTER) c.master = a.master + first;
  if constexpr (EIGHT) {
    c.mc = static_cast<uint8_t*>(a.exp_avg) + first;
    c.vc = static_cast<uint8_t*>(a.exp_avg_sq) + first;
    c.ms = a.exp_avg_scale + (first >> 8);
    c.vs = a.exp_avg_sq_scale + (first >> 8);
    t = (uint64_t)(a.step_device ? *a.step_device : a.step);
  } else {
    c.m = static_cast<float*>(a.exp_avg) + first;
    c.v = static_cast<float*>(a.exp_avg_sq) + first;
  }
  c.first = first;
  c.left = (int)min(e.size - at, kAdamChunk);
  c.keep = 1.0f - s.rate * e.decay;
  if (c.left == (int)kAdamChunk)
    step_chunk<P, G, EIGHT, MASTER, true>(c, a, s, t);
  else
    step_chunk<P, G, EIGHT, MASTER, false>(c, a, s, t);
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
  const Scalars host{s.grad_scale, (float)(1.0 / (1.0 - std::pow(p.beta1, (double)s.step))),
                     (float)(1.0 / (1.0 - std::pow(p.beta2, (double)s.step))), s.rate, 0};
  Scalars* scalars = nullptr;
  if (on_device(s)) {
    scalars = static_cast<Scalars*>(ws);
    double* part = reinterpret_cast<double*>(static_cast<char*>(ws) + 256);
    if (s.norm) {
      dispatch_elem(s.grad_type, [&](auto tag) {
        int64_t at = 0;
        for_groups(p, s, [&](uint32_t t0, const Grads& g, uint32_t c0, uint32_t count) {
          k_adamw_norm<decltype(tag)><<<kNormBlocks, 256, 0, st>>>(
              g, entries, chunks, c0, count, t0, part + at);
          at += kNormBlocks;
        });
      });
    }
    k_adamw_scalars<<<1, 256, 0, st>>>({part, s.norm ? (int)(groups(p) * kNormBlocks) : 0,
                                        s.grad_scale, s.max_norm, s.norm_out, p.beta1, p.beta2,
                                        s.step_device, s.rate_device, host, scalars});
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
             host,
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
