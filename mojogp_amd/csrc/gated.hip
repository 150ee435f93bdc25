// The gated layer h = act(x Wg^T + bg) * (x Wu^T + bu) and its gradients.
//
//   g = x Wg^T + bg, u = x Wu^T + bu, a = act(g), h = a u
//   dg = dh u act'(g), du = dh a
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dbg = sum dg, dbu = sum du
//
// Matrix-core bound: 4 rows width hidden operations forward, 8 backward, and 4
// for g and u again: the backward pass forms them anew instead of keeping
// them, which costs no memory between the passes and no rounding of g and u
// to the element type (kept in 16 bits they would set the gradients' error),
// and below a width of about 750 also less time than writing and reading them
// in 32 bits.  One product kernel serves all steps: the forward pass and
// (dg, du) with both projections in one tile and the elementwise part as its
// epilogue, dx against the transposed weights, and the weight gradients with
// the reduction over the rows split over the device.
//
// dg and du go into the last two products as the matrix cores take them: rounded to
// bfloat16, to float16 times a power of two of their row, in float32 in three parts
// (24 bits); g, u, all sums and the bias gradients stay fp32.
#include <algorithm>
#include <type_traits>

#include "activation.h"
#include "product.h"

namespace mgp {

namespace {

// The P parts of values, each what the ones before leave, rounded to the type:
// the first at p, the others `apart` elements on each.  Only the last takes
// infinities and NaN (and what bfloat16 would round to infinity), so that no
// difference of infinities is formed and a product meets them once.
template <int P, int N, class E>
__device__ __forceinline__ void store_parts(E* p, int64_t apart, int64_t left, const float* v) {
  // (without the copies below: the backward epilogue of bf16 12007 x 391 -> 1027 is
  // scheduled 12 % faster)
  if constexpr (P == 1) return store_run<N>(p, left, v);
  constexpr float kMost = std::is_same<E, __bf16>::value ? 3.3895313892515355e38f : 65504.0f;
  float rest[N], part[N];
#pragma unroll
  for (int k = 0; k < N; ++k) rest[k] = v[k];
#pragma unroll
  for (int i = 0; i < P - 1; ++i) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      part[k] = (float)(E)fminf(fmaxf(rest[k], -kMost), kMost);
      rest[k] -= part[k];
    }
    store_run<N>(p + i * apart, left, part);
  }
  store_run<N>(p + (P - 1) * apart, left, rest);
}

// ---------------------------------------------------------------- epilogues

template <class T, int ACT>
struct ForwardEpi {
  static constexpr bool FORWARD = true;
  const T *bg, *bu;
  T* h;
  int64_t ldh, rows, hidden;
  template <class TL>
  __device__ __forceinline__ void run(f4 (&acc)[TL::TM][TL::TN], int64_t m0, int64_t n0,
                                      int64_t) const {
    constexpr int N = TL::RUN;
    const int lane = threadIdx.x & 63;
    const int64_t f = n0 + N * (lane >> 4), left = hidden - f;
    if (left <= 0) return;
    float g0[N], u0[N];
#pragma unroll
    for (int k = 0; k < N; ++k) g0[k] = u0[k] = 0.0f;
    if (bg) load_run<N>(bg + f, left, g0);
    if (bu) load_run<N>(bu + f, left, u0);
#pragma unroll
    for (int m = 0; m < TL::TM; ++m) {
      const int64_t r = m0 + m * 16 + (lane & 15);
      if (r >= rows) continue;
      float o[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float a, slope;
        activate<ACT, sizeof(T) == 2>(acc[m][k / 4][k % 4] + g0[k], a, slope);
        o[k] = a * (acc[m][TL::T1 + k / 4][k % 4] + u0[k]);
      }
      store_run<N>(h + r * ldh + f, left, o);
    }
  }
};

// dgu[row] = [dg | du], each `pad` columns (zeros past hidden);
// dbias[part][2][hidden] the column sums over a wave's rows.
// In COPIES parts: [dg | du] of the first, then of the others.  float16: times the
// row's scale.
template <class T, class E, int ACT, int COPIES>
struct BackwardEpi {
  static constexpr bool FORWARD = false;
  static constexpr bool SCALED = std::is_same<E, _Float16>::value;
  const float* scale;  // of each row
  const T *bg, *bu;
  const T* dh;
  int64_t lddh, rows, hidden, pad;
  void* dgu;
  float* dbias;  // or null
  template <class TL>
  __device__ __forceinline__ void run(f4 (&acc)[TL::TM][TL::TN], int64_t m0, int64_t n0,
                                      int64_t part) const {
    constexpr int N = TL::RUN;
    const int lane = threadIdx.x & 63;
    const int64_t f = n0 + N * (lane >> 4), left = hidden - f;
    float g0[N], u0[N], sg[N], su[N];
#pragma unroll
    for (int k = 0; k < N; ++k) g0[k] = u0[k] = sg[k] = su[k] = 0.0f;
    if (left > 0) {
      if (bg) load_run<N>(bg + f, left, g0);
      if (bu) load_run<N>(bu + f, left, u0);
    }
#pragma unroll
    for (int m = 0; m < TL::TM; ++m) {
      const int64_t r = m0 + m * 16 + (lane & 15);
      if (r >= rows || f >= pad) continue;
      float d[N], dg[N], du[N];
      load_run<N>(dh + r * lddh + f, left, d);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float a, slope;
        activate<ACT, sizeof(T) == 2>(acc[m][k / 4][k % 4] + g0[k], a, slope);
        // columns past hidden are products of the last weights: cut off
        const bool in = k < left;
        dg[k] = in ? d[k] * (acc[m][TL::T1 + k / 4][k % 4] + u0[k]) * slope : 0.0f;
        du[k] = in ? d[k] * a : 0.0f;
        sg[k] += dg[k];
        su[k] += du[k];
      }
      if constexpr (SCALED) {
        const float sc = scale[r];
#pragma unroll
        for (int k = 0; k < N; ++k) {
          dg[k] *= sc;
          du[k] *= sc;
        }
      }
      E* row = static_cast<E*>(dgu) + r * 2 * COPIES * pad + f;
      store_parts<COPIES, N>(row, 2 * pad, pad - f, dg);
      store_parts<COPIES, N>(row + pad, 2 * pad, pad - f, du);
    }
    if (dbias) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) {
          sg[k] += __shfl_xor(sg[k], o);
          su[k] += __shfl_xor(su[k], o);
        }
        if ((lane & 15) == 0 && k < left) {
          dbias[(part * 2) * hidden + f + k] = sg[k];
          dbias[(part * 2 + 1) * hidden + f + k] = su[k];
        }
      }
    }
  }
};

// One split: the result; more: part[split][rows][cols] sums.  scale: that of each
// row, to be undone, or null.
template <class T>
struct StoreEpi {
  static constexpr bool FORWARD = false;
  const float* scale;
  T* out;
  float* part;
  int64_t rows, cols;
  template <class TL>
  __device__ __forceinline__ void run(f4 (&acc)[TL::TM][TL::TN], int64_t m0, int64_t n0,
                                      int64_t) const {
    constexpr int N = TL::RUN;
    const int lane = threadIdx.x & 63;
    const int64_t c = n0 + N * (lane >> 4);
    if (c >= cols) return;
#pragma unroll
    for (int m = 0; m < TL::TM; ++m) {
      const int64_t r = m0 + m * 16 + (lane & 15);
      if (r >= rows) continue;
      float o[N];
#pragma unroll
      for (int k = 0; k < N; ++k) o[k] = acc[m][k / 4][k % 4];
      if constexpr (std::is_same<T, _Float16>::value) {
        const float sc = 1.0f / scale[r];
#pragma unroll
        for (int k = 0; k < N; ++k) o[k] *= sc;
      }
      if (part)
        store_run<N>(part + ((int64_t)blockIdx.y * rows + r) * cols + c, cols - c, o);
      else
        store_run<N>(out + r * cols + c, cols - c, o);
    }
  }
};

// Rows of [dg | du]^T x: row m < pad of dw_gate, row m - pad of dw_up.  One
// split: the gradients themselves; more: part[split][2][hidden][width] sums.
// float16: unscale undoes the scale of the sum.
template <class T>
struct WeightEpi {
  static constexpr bool FORWARD = false;
  const float* unscale;
  T *dw_gate, *dw_up;
  float* part;
  int64_t hidden, pad, width;
  template <class TL>
  __device__ __forceinline__ void run(f4 (&acc)[TL::TM][TL::TN], int64_t m0, int64_t n0,
                                      int64_t) const {
    const int lane = threadIdx.x & 63;
    float sc = 1.0f;
    if constexpr (std::is_same<T, _Float16>::value) sc = *unscale;
#pragma unroll
    for (int m = 0; m < TL::TM; ++m) {
      const int64_t r = m0 + m * 16 + (lane & 15);
      const int up = r >= pad;
      const int64_t f = r - up * pad;
      if (f >= hidden) continue;
#pragma unroll
      for (int n = 0; n < TL::TN; ++n) {
        const int64_t c = n0 + n * 16 + 4 * (lane >> 4);
        if (c >= width) continue;
        const float o[4] = {acc[m][n][0] * sc, acc[m][n][1] * sc, acc[m][n][2] * sc,
                            acc[m][n][3] * sc};
        if (part) {
          store_run<4>(part + (((int64_t)blockIdx.y * 2 + up) * hidden + f) * width + c, width - c,
                       o);
        } else {
          T* dst = up ? dw_up : dw_gate;
          if (dst) store_run<4>(dst + f * width + c, width - c, o);
        }
      }
    }
  }
};

// ---------------------------------------------------------------- helpers

// Up to three matrices of one width in one launch: dst[row][pad] = src[row][cols],
// zeros past cols.
template <class T>
struct PackSource {
  const T* src[3];
  int64_t ld[3], rows[3], cols, pad;
  T* dst[3];
};

template <class T>
__global__ __launch_bounds__(256) void k_pack_rows(PackSource<T> s) {
  constexpr int N = Vec16<T>::N;
  const int64_t per = s.pad / N, total = (s.rows[0] + s.rows[1] + s.rows[2]) * per;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total;
       q += (int64_t)gridDim.x * 256) {
    int64_t r = q / per;
    const int64_t c = (q - r * per) * N;
    int m = 0;
    if (r >= s.rows[0]) {
      r -= s.rows[0];
      m = 1;
      if (r >= s.rows[1]) {
        r -= s.rows[1];
        m = 2;
      }
    }
    const T* src = (m == 0 ? s.src[0] : m == 1 ? s.src[1] : s.src[2]) +
                   r * (m == 0 ? s.ld[0] : m == 1 ? s.ld[1] : s.ld[2]) + c;
    T* dst = (m == 0 ? s.dst[0] : m == 1 ? s.dst[1] : s.dst[2]) + r * s.pad + c;
    T v[N];
    if (c + N <= s.cols) {
      __builtin_memcpy(v, src, sizeof(v));
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = c + k < s.cols ? src[k] : (T)0.0f;
    }
    __builtin_memcpy(dst, v, sizeof(v));
  }
}

// dst[k][part pad + f] = W_part[f][k], zeros for f past hidden; 32 x 32 tiles
template <class T>
__global__ __launch_bounds__(256) void k_transpose_weights(const T* __restrict__ wg,
                                                           const T* __restrict__ wu, int64_t ld,
                                                           int64_t hidden, int64_t width,
                                                           int64_t pad, T* __restrict__ dst) {
  __shared__ T tile[32][33];
  const int64_t f0 = (int64_t)blockIdx.x * 32, k0 = (int64_t)blockIdx.y * 32;
  const T* w = blockIdx.z ? wu : wg;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const int64_t f = f0 + ty + i, k = k0 + tx;
    tile[ty + i][tx] = f < hidden && k < width ? w[f * ld + k] : (T)0.0f;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const int64_t k = k0 + ty + i, f = f0 + tx;
    if (k < width && f < pad) dst[k * 2 * pad + blockIdx.z * pad + f] = tile[tx][ty + i];
  }
}

// out0 / out1 [count] = sums over the parts of part[parts][outputs][count], in order
template <class T>
__global__ __launch_bounds__(256) void k_sum_parts(const float* __restrict__ part, int64_t parts,
                                                   int64_t count, int outputs,
                                                   T* __restrict__ out0, T* __restrict__ out1) {
  const int64_t total = outputs * count;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * 256) {
    const bool second = i >= count;
    T* dst = second ? out1 : out0;
    if (dst == nullptr) continue;
    float s = 0.0f;
#pragma unroll 8
    for (int64_t p = 0; p < parts; ++p) s += part[p * total + i];
    dst[i - (second ? count : 0)] = (T)s;
  }
}

template <class T>
void sum_parts(const float* part, int64_t parts, int64_t count, int outputs, T* out0, T* out1,
               hipStream_t st) {
  const int64_t blocks = ceil_div(outputs * count, (int64_t)256);
  k_sum_parts<T><<<(unsigned)std::min<int64_t>(blocks, 8192), 256, 0, st>>>(part, parts, count,
                                                                           outputs, out0, out1);
}

// The bias gradients: few columns, many parts; 64 columns a block, 16 waves
template <class T>
__global__ __launch_bounds__(1024) void k_sum_bias(const float* __restrict__ part, int64_t parts,
                                                   int64_t count, T* __restrict__ out_g,
                                                   T* __restrict__ out_u) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i = (int64_t)blockIdx.x * 64 + lane;
  float s = 0.0f;
  if (i < 2 * count) {
#pragma unroll 4
    for (int64_t p = wave; p < parts; p += 16) s += part[p * 2 * count + i];
  }
  red[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || i >= 2 * count) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) s += red[k][lane];
  T* dst = i < count ? out_g : out_u;
  if (dst) dst[i < count ? i : i - count] = (T)s;
}

// ---------------------------------------------------------------- little work

struct FewArgs {
  const void *x, *wg, *wu, *bg, *bu;
  int64_t ldx, ldg, ldu, ldh, rows, width, hidden;
  void* h;
};

// The forward pass where the product kernel's tiles would leave most of the
// device idle (a single point, a batch of a few hundred): a workgroup takes 16
// columns of both projections for 16 MT rows, its 8 waves share the reduction
// and read their fragments from global memory, at any alignment.  Bound by
// latency: one round of loads for a width of 512, one exchange through LDS
// (bf16, one row x 512 -> 2048: 4.2 us for 4.2 MB of weights).
template <class T, int ACT, int MT>
__global__ __launch_bounds__(512) void k_gated_few(FewArgs s) {
  constexpr int N = Vec16<T>::N, W = 8;
  __shared__ f4 red[W][2 * MT][64];
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t f0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * 16 * MT;
  // rows past the last are read as the last and not stored
  const int64_t f = min(f0 + i, s.hidden - 1);
  const T* wg = static_cast<const T*>(s.wg) + f * s.ldg;
  const T* wu = static_cast<const T*>(s.wu) + f * s.ldu;
  const T* x[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
    x[t] = static_cast<const T*>(s.x) + min(m0 + 16 * t + i, s.rows - 1) * s.ldx;
  f4 ag[MT], au[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) ag[t] = au[t] = f4{0.f, 0.f, 0.f, 0.f};
  auto frag = [&](const T* p, int64_t k) __attribute__((always_inline)) {
    T a[N];
    if (k + N <= s.width) {
      __builtin_memcpy(a, p + k, 16);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) a[e] = k + e < s.width ? p[k + e] : (T)0.0f;
    }
    Frag r;
    __builtin_memcpy(&r, a, 16);
    return r;
  };
#pragma unroll 2
  for (int64_t k0 = wave * 4 * N; k0 < s.width; k0 += W * 4 * N) {
    const int64_t k = k0 + g * N;
    const Frag pg = frag(wg, k), pu = frag(wu, k);
    Frag q[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) q[t] = frag(x[t], k);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      ag[t] = mma<T>(pg, q[t], ag[t]);
      au[t] = mma<T>(pu, q[t], au[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    red[wave][2 * t][lane] = ag[t];
    red[wave][2 * t + 1][lane] = au[t];
  }
  __syncthreads();
  if (wave >= MT) return;
  f4 sg = red[0][2 * wave][lane], su = red[0][2 * wave + 1][lane];
#pragma unroll
  for (int w = 1; w < W; ++w) {
    sg += red[w][2 * wave][lane];
    su += red[w][2 * wave + 1][lane];
  }
  const int64_t r = m0 + 16 * wave + i, c = f0 + 4 * g, left = s.hidden - c;
  if (r >= s.rows || left <= 0) return;
  float b0[4] = {0, 0, 0, 0}, b1[4] = {0, 0, 0, 0}, o[4];
  if (s.bg) load_run<4>(static_cast<const T*>(s.bg) + c, left, b0);
  if (s.bu) load_run<4>(static_cast<const T*>(s.bu) + c, left, b1);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float a, slope;
    activate<ACT, sizeof(T) == 2>(sg[e] + b0[e], a, slope);
    o[e] = a * (su[e] + b1[e]);
  }
  store_run<4>(static_cast<T*>(s.h) + r * s.ldh + c, left, o);
}

// ---------------------------------------------------------------- fp32 operands in bf16 parts

struct SplitSource {
  const float *x, *wg, *wu;
  int64_t ldx, ldg, ldu, rows, hidden, width, wpad;
  __bf16 *dx, *dwg, *dwu;  // [rows][kSplit][wpad]
};
constexpr int kSplit = 3;

__global__ __launch_bounds__(256) void k_split(SplitSource s) {
  const int64_t per = s.wpad / 8, total = (s.rows + 2 * s.hidden) * per;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total;
       q += (int64_t)gridDim.x * 256) {
    int64_t r = q / per;
    const int64_t c = (q - r * per) * 8;
    const float* src;
    __bf16* dst;
    if (r < s.rows) {
      src = s.x + r * s.ldx;
      dst = s.dx;
    } else if ((r -= s.rows) < s.hidden) {
      src = s.wg + r * s.ldg;
      dst = s.dwg;
    } else {
      r -= s.hidden;
      src = s.wu + r * s.ldu;
      dst = s.dwu;
    }
    float v[8];
    load_run<8>(src + c, s.width - c, v);
    store_parts<kSplit, 8>(dst + r * kSplit * s.wpad + c, s.wpad, 8, v);
  }
}

// dst[k][part][pad of the gate, pad of up] = parts of W[f][k]
__global__ __launch_bounds__(256) void k_transpose_split(const __bf16* __restrict__ wg,
                                                         const __bf16* __restrict__ wu,
                                                         int64_t hidden, int64_t width,
                                                         int64_t wpad, int64_t pad,
                                                         __bf16* __restrict__ dst) {
  __shared__ __bf16 tile[32][34];
  const int64_t f0 = (int64_t)blockIdx.x * 32, k0 = (int64_t)blockIdx.y * 32;
  const int up = blockIdx.z & 1, part = blockIdx.z >> 1;
  const __bf16* w = (up ? wu : wg) + part * wpad;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const int64_t f = f0 + ty + i, k = k0 + tx;
    tile[ty + i][tx] = f < hidden && k < width ? w[f * kSplit * wpad + k] : (__bf16)0.0f;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const int64_t k = k0 + ty + i, f = f0 + tx;
    if (k < width && f < pad)
      dst[k * kSplit * 2 * pad + part * 2 * pad + up * pad + f] = tile[tx][ty + i];
  }
}

// ---------------------------------------------------------------- float16 dg and du

// float16 ends at 65504 and loses bits below 2^-14, which dg and du of usual
// gradients pass at either end.  Each row of [dg | du] is stored times a power of
// two of its own, from a bound on the row that is known before its values are:
// |u|, |g| <= |x| |w| + |b|, |dg| <= 1.13 |dh| |u| and |du| <= |dh| |act(g)|,
// |act(g)| <= |g| or 1 (the sigmoid), some five of float16's 29 binades above what
// occurs.  dx takes a row's scale out again; the weight gradients, which sum over
// rows, take x over the row's scale instead of x, times the power of two that
// fits the largest.  bfloat16 and float32 have the range as they are.  Three kernels
// that read dh and x once, HBM and latency bound: backward, 128 x 256 -> 1024 42 -> 52
// us, 20000 x 256 -> 512 96 -> 126, 65536 x 1024 -> 4096 3340 -> 3660 (255 of it here, the
// rest the epilogue's).
struct ScaleSource {
  const _Float16 *x, *dh, *wg, *wu, *bg, *bu;
  int64_t ldx, lddh, ldg, ldu, rows, hidden, width, wpad;
  float act_max;
  int wblocks, blocks;  // workgroups of k_weight_sizes, of the kernels of the rows
  float* wpart;    // [2][kWeightBlocks]: largest norm of a weight row, largest bias
  float* scale;    // [rows]
  float* xpart;    // [kScaleBlocks]: largest |x| over its row's scale
  _Float16* xs;    // [rows][wpad]
  float* unscale;  // of the weight gradients
};
constexpr int kWeightBlocks = 512, kScaleBlocks = 2048;  // four rows at a time each, at most

__device__ __forceinline__ float pow2_below(float bound) {
  // the largest 2^e with 2^e bound < 2^15
  if (!(bound > 0.0f)) return 1.0f;
  return ldexpf(1.0f, min(max(14 - ilogbf(bound), -120), 120));
}

__device__ __forceinline__ float wave_max(float a) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) a = fmaxf(a, __shfl_xor(a, o));
  return a;
}

// The largest finite |value| of a row and the sum of the finite squares, over a
// wave.  Values that are not finite spoil their own row only.
__device__ __forceinline__ void row_sizes(const _Float16* p, int64_t cols, float& big,
                                          float& sum) {
  big = sum = 0.0f;
#pragma unroll 4
  for (int64_t c = 8 * (threadIdx.x & 63); c < cols; c += 512) {
    float v[8];
    load_run<8>(p + c, cols - c, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float a = fabsf(v[k]);
      a = a < INFINITY ? a : 0.0f;
      big = fmaxf(big, a);
      sum = fmaf(a, a, sum);
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    sum += __shfl_xor(sum, o);
    big = fmaxf(big, __shfl_xor(big, o));
  }
}

__device__ __forceinline__ float block_max(float a, float* red) {
  a = wave_max(a);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// the largest of count <= N partial results, every load out at once
template <int N>
__device__ __forceinline__ float largest_of(const float* part, int count) {
  const int lane = threadIdx.x & 63;
  float v[N / 64], a = 0.0f;
#pragma unroll
  for (int b = 0; b < N / 64; ++b) v[b] = b * 64 + lane < count ? part[b * 64 + lane] : 0.0f;
#pragma unroll
  for (int b = 0; b < N / 64; ++b) a = fmaxf(a, v[b]);
  return wave_max(a);
}

__global__ __launch_bounds__(256) void k_weight_sizes(ScaleSource s) {
  __shared__ float red[4];
  float norm = 0.0f, bias = 0.0f;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < 2 * s.hidden;
       r += (int64_t)gridDim.x * 4) {
    const bool up = r >= s.hidden;
    const int64_t f = up ? r - s.hidden : r;
    float big, sum;
    row_sizes(up ? s.wu + f * s.ldu : s.wg + f * s.ldg, s.width, big, sum);
    norm = fmaxf(norm, sqrtf(sum));
    const _Float16* b = up ? s.bu : s.bg;
    const float v = b ? fabsf((float)b[f]) : 0.0f;
    bias = fmaxf(bias, v < INFINITY ? v : 0.0f);
  }
  norm = block_max(norm, red);
  bias = block_max(bias, red);
  if (threadIdx.x == 0) {
    s.wpart[blockIdx.x] = norm;
    s.wpart[kWeightBlocks + blockIdx.x] = bias;
  }
}

__global__ __launch_bounds__(256) void k_row_scales(ScaleSource s) {
  __shared__ float red[4];
  const float norm = largest_of<kWeightBlocks>(s.wpart, s.wblocks);
  const float bias = largest_of<kWeightBlocks>(s.wpart + kWeightBlocks, s.wblocks);
  float most = 0.0f;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < s.rows;
       r += (int64_t)gridDim.x * 4) {
    float d, x, sum, unused;
    row_sizes(s.dh + r * s.lddh, s.hidden, d, unused);
    row_sizes(s.x + r * s.ldx, s.width, x, sum);
    const float sc = pow2_below(1.2f * d * fmaxf(fmaf(sqrtf(sum), norm, bias), s.act_max));
    if ((threadIdx.x & 63) == 0) s.scale[r] = d > 0.0f ? sc : 0.0f;
    if (d > 0.0f) most = fmaxf(most, x / sc);
  }
  most = block_max(most, red);
  if (threadIdx.x == 0) s.xpart[blockIdx.x] = most;
}

// A row with no gradient has scale 0 so far, which makes its part of xs 0; from
// here on 1.
__global__ __launch_bounds__(256) void k_scale_rows(ScaleSource s) {
  const float all = pow2_below(largest_of<kScaleBlocks>(s.xpart, s.blocks));
  if (blockIdx.x == 0 && threadIdx.x == 0) *s.unscale = 1.0f / all;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < s.rows;
       r += (int64_t)gridDim.x * 4) {
    const float sc = s.scale[r], by = sc > 0.0f ? all / sc : 0.0f;
    for (int64_t c = 8 * (threadIdx.x & 63); c < s.wpad; c += 512) {
      float v[8];
      load_run<8>(s.x + r * s.ldx + c, s.width - c, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= by;
      store_run<8>(s.xs + r * s.wpad + c, 8, v);
    }
    if ((threadIdx.x & 63) == 0 && !(sc > 0.0f)) s.scale[r] = 1.0f;
  }
}

// ---------------------------------------------------------------- host side

constexpr int64_t kMaxSplits = 64;

// fp32 layers go through the bf16 matrix cores: three parts of 8 bits hold a
// value's 24 whatever its size beside the others', as bf16 has the range of fp32
// (below 2^-100 the last part is lost), and six products make the sum, those left
// out being below 2^-25 of it.  Six times the work at 16 times the rate of the fp32
// instructions.  20000 x 256 -> 512, both passes: 494 us by fp32 instructions, 465
// so, 2.4e-7 off; two fp16 parts and three products take 320, but a common scale
// then ties every row to the largest value of all, and a scale a row still ties
// the columns of a row to its largest.

// The 16-bit types' dg and du are rounded to the type for the last two products:
// with the result's own rounding that makes dx and the weight gradients 1.41 times
// as far off as rounding alone, at any number of rows.  A second part takes that back
// and runs the two products twice.  Up to one tile of rows, where a call is its
// launches, it is worth it: bf16, 128 x 256 -> 1024, backward 31 -> 41 us, 100 x 1024 ->
// 4096 59 -> 70; at 65536 rows it would cost 1.9 of 3.2 ms.
constexpr int64_t kFewRows = 128;

enum Mode : int { PLAIN = 0, FP32_PARTS = 1, FEW_ROWS = 2 };

// What a call needs and where it lies in the workspace.
template <class T, int MODE_>
struct Plan {
  static constexpr int MODE = MODE_;
  static constexpr bool SPLIT = MODE == FP32_PARTS;
  static constexpr bool SCALED = std::is_same<T, _Float16>::value;  // dg and du, by rows
  using E = typename std::conditional<SPLIT, __bf16, T>::type;  // what the products take
  // products of the projections and of the gradients; copies of x and the
  // weights, and of dg and du
  static constexpr int PARTS = SPLIT ? 6 : 1, GRAD_PARTS = SPLIT ? 6 : MODE == FEW_ROWS ? 2 : 1;
  static constexpr int COPIES = SPLIT ? kSplit : 1;
  static constexpr int D_COPIES = SPLIT ? kSplit : MODE == FEW_ROWS ? 2 : 1;
  // width and hidden rounded to whole 16-byte chunks, or to whole stages
  static constexpr int WQ = SPLIT ? 64 : Vec16<T>::N, HQ = SPLIT ? 32 : Vec16<T>::N;
  int64_t wpad, hpad;
  bool pack_x, pack_w;
  size_t x_off = 0, wg_off = 0, wu_off = 0, wt_off = 0, dgu_off = 0, dbias_off = 0, part_off = 0;
  size_t dxp_off = 0, scale_off = 0, xs_off = 0;
  size_t bytes = 0;
  bool big_dual = false;
  Cut dx, dw;
  int64_t bias_parts = 0;

  Plan(const GatedArgs& a, bool backward) {
    wpad = round_up(a.width, WQ);
    hpad = round_up(a.hidden, HQ);
    pack_x = SPLIT || !direct<T>(a.x, a.x_stride, a.width);
    pack_w = SPLIT || !direct<T>(a.w_gate, a.w_gate_stride, a.width) ||
             !direct<T>(a.w_up, a.w_up_stride, a.width) || a.w_gate_stride != a.w_up_stride;
    auto require = [](int64_t row, const char* what) {
      MGP_REQUIRE(row * (int64_t)sizeof(E) < kRowBytes,
                  std::string("the ") + what + " of a gated layer is too large (the products "
                  "take rows of less than 8 MB)");
    };
    require(wpad * COPIES, "width");
    if (backward) require(std::max(ldd(), ldt()), "hidden width");
    auto take = [&](size_t n) {
      const size_t at = bytes;
      bytes += align_up(n);
      return at;
    };
    if (pack_x) x_off = take((size_t)a.rows * wpad * COPIES * sizeof(E));
    if (pack_w) {
      wg_off = take((size_t)a.hidden * wpad * COPIES * sizeof(E));
      wu_off = take((size_t)a.hidden * wpad * COPIES * sizeof(E));
    }
    const int64_t rows = std::max<int64_t>(a.rows, 1);
    constexpr int64_t KS = 128 / sizeof(E);
    constexpr bool may_big = MODE != FEW_ROWS;  // (which has too few rows for them)
    big_dual = cut_product(2 * a.hidden, rows, ceil_div(wpad, KS), PARTS, may_big, 1, 0.0).big;
    if (!backward) return;
    wt_off = take((size_t)a.width * ldt() * sizeof(E));
    dgu_off = take((size_t)a.rows * ldd() * sizeof(E));
    bias_parts = 2 * ceil_div(rows, (int64_t)(big_dual ? 256 : 128));
    dbias_off = take((size_t)bias_parts * 2 * a.hidden * sizeof(float));
    // the weight gradients' reduction is over the rows, dx's over hidden
    const int64_t weights = 2 * a.hidden * a.width;
    dw = cut_product(a.width, 2 * hpad, ceil_div(rows, KS), GRAD_PARTS, may_big, kMaxSplits,
                     (double)weights);
    if (dw.splits > 1) part_off = take((size_t)dw.splits * weights * sizeof(float));
    dx = cut_product(a.width, rows, ceil_div(2 * hpad, KS), GRAD_PARTS, may_big, kMaxSplits,
                     (double)a.rows * (double)a.width);
    if (dx.splits > 1) dxp_off = take((size_t)dx.splits * a.rows * a.width * sizeof(float));
    if (SCALED) {
      scale_off = take((2 * kWeightBlocks + kScaleBlocks + 1 + (size_t)a.rows) * sizeof(float));
      xs_off = take((size_t)a.rows * wpad * sizeof(E));
    }
  }
  static int64_t reduction(const Cut& c) { return c.per * (128 / (int64_t)sizeof(E)); }
  int64_t ldd() const { return 2 * hpad * D_COPIES; }  // of [dg | du]
  int64_t ldt() const { return 2 * hpad * COPIES; }    // of the transposed weights
};

template <class E>
struct Inputs {
  const E *x, *wg, *wu;
  int64_t ldx, ldw;
};

// x and the weights as the product kernel loads them.
template <class T, int MODE>
Inputs<typename Plan<T, MODE>::E> load_inputs(const GatedArgs& a, const Plan<T, MODE>& pl,
                                              char* ws, hipStream_t st) {
  using E = typename Plan<T, MODE>::E;
  E *x = reinterpret_cast<E*>(ws + pl.x_off), *wg = reinterpret_cast<E*>(ws + pl.wg_off),
    *wu = reinterpret_cast<E*>(ws + pl.wu_off);
  if constexpr (MODE == FP32_PARTS) {
    auto f = [](const void* p) { return static_cast<const float*>(p); };
    const int64_t items = (a.rows + 2 * a.hidden) * (pl.wpad / 8);
    k_split<<<(unsigned)std::min<int64_t>(ceil_div(items, (int64_t)256), 8192), 256, 0, st>>>(
        {f(a.x), f(a.w_gate), f(a.w_up), a.x_stride, a.w_gate_stride, a.w_up_stride, a.rows,
         a.hidden, a.width, pl.wpad, x, wg, wu});
    return {x, wg, wu, kSplit * pl.wpad, kSplit * pl.wpad};
  } else {
    Inputs<E> in{static_cast<const T*>(a.x), static_cast<const T*>(a.w_gate),
                 static_cast<const T*>(a.w_up), a.x_stride, a.w_gate_stride};
    PackSource<T> p{};
    p.cols = a.width;
    p.pad = pl.wpad;
    if (pl.pack_x) {
      p.src[0] = in.x;
      p.ld[0] = a.x_stride;
      p.rows[0] = a.rows;
      p.dst[0] = x;
      in.x = x;
      in.ldx = pl.wpad;
    }
    if (pl.pack_w) {
      p.src[1] = in.wg;
      p.src[2] = in.wu;
      p.ld[1] = a.w_gate_stride;
      p.ld[2] = a.w_up_stride;
      p.rows[1] = p.rows[2] = a.hidden;
      p.dst[1] = wg;
      p.dst[2] = wu;
      in.wg = wg;
      in.wu = wu;
      in.ldw = pl.wpad;
    }
    const int64_t items = (p.rows[0] + p.rows[1] + p.rows[2]) * (pl.wpad / Vec16<T>::N);
    if (items > 0)
      k_pack_rows<T><<<(unsigned)std::min<int64_t>(ceil_div(items, (int64_t)256), 8192), 256, 0,
                       st>>>(p);
    return in;
  }
}

// Scales of the rows of [dg | du], and x for the weight gradients.
template <class PL>
ScaleSource scale_rows(const GatedArgs& a, const PL& pl, const void* dh, int64_t dh_stride,
                       char* ws, hipStream_t st) {
  auto f = [](const void* p) { return static_cast<const _Float16*>(p); };
  auto blocks = [](int64_t rows, int most) {
    return (int)std::min<int64_t>(ceil_div(rows, (int64_t)4), most);
  };
  float *w = reinterpret_cast<float*>(ws + pl.scale_off), *xpart = w + 2 * kWeightBlocks;
  const ScaleSource s{f(a.x), f(dh), f(a.w_gate), f(a.w_up), f(a.b_gate), f(a.b_up), a.x_stride,
                      dh_stride, a.w_gate_stride, a.w_up_stride, a.rows, a.hidden, a.width,
                      pl.wpad, a.activation == ACT_SIGMOID ? 1.0f : 0.0f,
                      blocks(2 * a.hidden, kWeightBlocks), blocks(a.rows, kScaleBlocks), w,
                      xpart + kScaleBlocks + 1, xpart,
                      reinterpret_cast<_Float16*>(ws + pl.xs_off), xpart + kScaleBlocks};
  k_weight_sizes<<<s.wblocks, 256, 0, st>>>(s);
  k_row_scales<<<s.blocks, 256, 0, st>>>(s);
  k_scale_rows<<<s.blocks, 256, 0, st>>>(s);
  return s;
}

template <class PL, bool TR, bool DUAL, class EPI>
void launch_product(bool big, const GemmShape& s, int64_t splits, const EPI& epi,
                    hipStream_t st) {
  constexpr int PARTS = DUAL ? PL::PARTS : PL::GRAD_PARTS;
  if constexpr (PL::MODE != FEW_ROWS) {  // (which has too few for the large tiles)
    if (big)
      return launch_tiles<BigTile<typename PL::E, TR, DUAL, PARTS>>(s, splits, epi, st);
  }
  launch_tiles<SmallTile<typename PL::E, TR, DUAL, PARTS>>(s, splits, epi, st);
}

template <class PL, class EPI>
void launch_dual(const GatedArgs& a, const PL& pl, const Inputs<typename PL::E>& in,
                 const EPI& epi, hipStream_t st) {
  GemmShape s{};
  s.p = operand(in.wg, in.ldw, a.hidden, in.wu);
  s.q = operand(in.x, in.ldx, a.rows);
  s.K = s.k_split = pl.wpad;
  s.p_apart = s.q_apart = pl.wpad * (int64_t)sizeof(typename PL::E);
  launch_product<PL, false, true>(pl.big_dual, s, 1, epi, st);
}

// Forward passes by k_gated_few: up to this many of its workgroups it is the
// faster one, at any width, as either kernel's time grows with it.  Device time,
// few against tiles, by workgroups, at widths 64 / 256 / 1024: 16 bits, 256 3.4 - 4.2 /
// 4.3 - 5.9 / 8.1 - 12.2 us, 512 4.0 - 4.5 / 5.9 - 6.3 / 13.7 - 12.9, 768 5.5 - 4.7 / 8.0 - 6.6 /
// 19 - 13; fp32, against six products and the kernel before them, 512 5.2 - 12 / 10.5 -
// 26 / 30 - 78, 1024 8.4 - 13 / 18 - 27 / 56 - 83, 2048 15 - 14.5 / 32 - 31 / 106 - 87.
inline bool takes_few(const GatedArgs& a) {
  return ceil_div(a.rows, (int64_t)64) * ceil_div(a.hidden, (int64_t)16) <=
         (a.type == ELEM_F32 ? 1536 : 512);
}

template <class T, int ACT>
void launch_few(const FewArgs& s, hipStream_t st) {
  auto go = [&](auto mt) {
    constexpr int MT = decltype(mt)::value;
    k_gated_few<T, ACT, MT><<<dim3((unsigned)ceil_div(s.hidden, (int64_t)16),
                                   (unsigned)ceil_div(s.rows, (int64_t)(16 * MT))),
                              512, 0, st>>>(s);
  };
  if (s.rows <= 16)
    go(std::integral_constant<int, 1>{});
  else if (s.rows <= 32)
    go(std::integral_constant<int, 2>{});
  else
    go(std::integral_constant<int, 4>{});
  MGP_HIP_CHECK(hipGetLastError());
}

// Runs f with the element type and the mode of a pass.
template <class F>
void dispatch_layer(const GatedArgs& a, bool backward, F&& f) {
  dispatch_elem(a.type, [&](auto tag) {
    if constexpr (sizeof(tag) == 4)
      f(tag, std::integral_constant<int, FP32_PARTS>{});
    else if (backward && a.rows <= kFewRows)
      f(tag, std::integral_constant<int, FEW_ROWS>{});
    else
      f(tag, std::integral_constant<int, PLAIN>{});
  });
}

}  // namespace

size_t gated_bytes(const GatedArgs& a, bool backward) {
  if (!backward && takes_few(a)) return 0;
  size_t n = 0;
  dispatch_layer(a, backward, [&](auto tag, auto mode) {
    n = Plan<decltype(tag), mode.value>(a, backward).bytes;
  });
  return n;
}

void gated_forward(const GatedArgs& a, void* h, int64_t h_stride, void* ws, hipStream_t st) {
  if (a.rows == 0) return;
  if (takes_few(a)) {
    const FewArgs s{a.x,        a.w_gate, a.w_up, a.b_gate, a.b_up, a.x_stride, a.w_gate_stride,
                    a.w_up_stride, h_stride, a.rows, a.width, a.hidden, h};
    dispatch_elem(a.type, [&](auto tag) {
      dispatch_act(a.activation, [&](auto act) { launch_few<decltype(tag), act.value>(s, st); });
    });
    return;
  }
  dispatch_layer(a, false, [&](auto tag, auto mode) {
    using T = decltype(tag);
    const Plan<T, mode.value> pl(a, false);
    const auto in = load_inputs(a, pl, static_cast<char*>(ws), st);
    dispatch_act(a.activation, [&](auto act) {
      ForwardEpi<T, act.value> epi{static_cast<const T*>(a.b_gate),
                                   static_cast<const T*>(a.b_up),
                                   static_cast<T*>(h),
                                   h_stride,
                                   a.rows,
                                   a.hidden};
      launch_dual(a, pl, in, epi, st);
    });
  });
}

void gated_backward(const GatedArgs& a, const void* dh, int64_t dh_stride, const GatedGrads& g,
                    void* ws_v, hipStream_t st) {
  char* ws = static_cast<char*>(ws_v);
  dispatch_layer(a, true, [&](auto tag, auto mode) {
    using T = decltype(tag);
    using PL = Plan<T, mode.value>;
    using E = typename PL::E;
    T *dwg = static_cast<T*>(g.dw_gate), *dwu = static_cast<T*>(g.dw_up);
    T *dbg = static_cast<T*>(g.db_gate), *dbu = static_cast<T*>(g.db_up);
    if (a.rows == 0) {  // sums over no rows (fills by a kernel: a caller may capture them)
      if (dwg || dwu) sum_parts<T>(nullptr, 0, a.hidden * a.width, 2, dwg, dwu, st);
      if (dbg || dbu) sum_parts<T>(nullptr, 0, a.hidden, 2, dbg, dbu, st);
      MGP_HIP_CHECK(hipGetLastError());
      return;
    }
    const PL pl(a, true);
    const Inputs<E> in = load_inputs(a, pl, ws, st);
    E* dgu = reinterpret_cast<E*>(ws + pl.dgu_off);
    float* dbias = dbg || dbu ? reinterpret_cast<float*>(ws + pl.dbias_off) : nullptr;
    ScaleSource sc{};
    if constexpr (PL::SCALED) sc = scale_rows(a, pl, dh, dh_stride, ws, st);
    dispatch_act(a.activation, [&](auto act) {
      BackwardEpi<T, E, act.value, PL::D_COPIES> epi{sc.scale,
                                                     static_cast<const T*>(a.b_gate),
                                                     static_cast<const T*>(a.b_up),
                                                     static_cast<const T*>(dh),
                                                     dh_stride,
                                                     a.rows,
                                                     a.hidden,
                                                     pl.hpad,
                                                     dgu,
                                                     dbias};
      launch_dual(a, pl, in, epi, st);
    });
    if (dbias)
      k_sum_bias<T><<<(unsigned)ceil_div(2 * a.hidden, (int64_t)64), 1024, 0, st>>>(
          dbias, pl.bias_parts, a.hidden, dbg, dbu);
    const int64_t apart = 2 * pl.hpad * (int64_t)sizeof(E);
    if (g.dx) {
      E* wt = reinterpret_cast<E*>(ws + pl.wt_off);
      const unsigned gx = (unsigned)ceil_div(pl.hpad, (int64_t)32);
      const unsigned gy = (unsigned)ceil_div(a.width, (int64_t)32);
      if constexpr (PL::SPLIT)
        k_transpose_split<<<dim3(gx, gy, 2 * kSplit), 256, 0, st>>>(in.wg, in.wu, a.hidden, a.width,
                                                           pl.wpad, pl.hpad, wt);
      else
        k_transpose_weights<T><<<dim3(gx, gy, 2), 256, 0, st>>>(in.wg, in.wu, in.ldw, a.hidden,
                                                                a.width, pl.hpad, wt);
      GemmShape s{};
      s.p = operand(wt, pl.ldt(), a.width);
      s.q = operand(dgu, pl.ldd(), a.rows);
      s.K = 2 * pl.hpad;
      s.k_split = PL::reduction(pl.dx);
      s.p_apart = s.q_apart = apart;
      T* dx = static_cast<T*>(g.dx);
      float* part = pl.dx.splits > 1 ? reinterpret_cast<float*>(ws + pl.dxp_off) : nullptr;
      launch_product<PL, false, false>(
          pl.dx.big, s, pl.dx.splits,
          StoreEpi<T>{sc.scale, dx, part, a.rows, a.width}, st);
      if (part) sum_parts<T>(part, pl.dx.splits, a.rows * a.width, 1, dx, nullptr, st);
    }
    if (dwg || dwu) {
      float* part = pl.dw.splits > 1 ? reinterpret_cast<float*>(ws + pl.part_off) : nullptr;
      GemmShape s{};
      s.p = operand(in.x, in.ldx, pl.wpad);
      if constexpr (PL::SCALED) s.p = operand(static_cast<const E*>(sc.xs), pl.wpad, pl.wpad);
      s.q = operand(static_cast<const E*>(dgu), pl.ldd(), 2 * pl.hpad);
      s.K = a.rows;
      s.k_split = PL::reduction(pl.dw);
      s.p_apart = pl.wpad * (int64_t)sizeof(E);
      s.q_apart = apart;
      launch_product<PL, true, false>(pl.dw.big, s, pl.dw.splits,
                                      WeightEpi<T>{sc.unscale, dwg, dwu, part, a.hidden, pl.hpad,
                                                   a.width},
                                      st);
      if (part) sum_parts<T>(part, pl.dw.splits, a.hidden * a.width, 2, dwg, dwu, st);
    }
    MGP_HIP_CHECK(hipGetLastError());
  });
}

}  // namespace mgp
