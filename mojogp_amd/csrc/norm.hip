// Layer norm over the rows of a feature matrix, forward and backward.
//
//   xhat = (x - mean) rstd,  y = xhat w + b,  rstd = 1 / sqrt(var + eps)
//   dx = rstd (g - mean(g) - xhat mean(g xhat)),  g = dy w
//   dw = sum over rows of dy xhat,  db = sum over rows of dy
//
// HBM bound: a row stays in registers between the reduction and the result,
// so the forward pass reads x and writes y once, the backward pass reads x and
// dy and writes dx once (fp32, 250000 x 256: 91 us, 5.6 TB/s, and 153 us, 5.0 TB/s).
// Statistics and sums are fp32; the variance is that of the centred row.
#include "layers.h"

#include <algorithm>
#include <type_traits>

namespace mgp {

namespace {

constexpr int kNormThreads = 256;

template <class T>
struct Raw {  // one vector as it lies in memory
  T v[Vec16<T>::N];
};

// Vectors go at any alignment (rows of odd widths, of tables).
template <class T>
__device__ __forceinline__ Raw<T> load_raw(const T* p) {
  Raw<T> a;
  __builtin_memcpy(&a, p, sizeof(a));
  return a;
}

template <class T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
  T a[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) a[i] = (T)v[i];
  __builtin_memcpy(p, a, sizeof(a));
}

// VEC parameters from column c on, or the default
template <class T, int VEC>
__device__ __forceinline__ void load_params(const void* p, int64_t c, bool f32, float none,
                                            float* v) {
  if (p == nullptr) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = none;
  } else if (f32) {
    __builtin_memcpy(v, static_cast<const float*>(p) + c, VEC * sizeof(float));
  } else {
    const Raw<T> a = load_raw(static_cast<const T*>(p) + c);
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = (float)a.v[k];
  }
}

template <class T>
__device__ __forceinline__ float load_param(const void* p, int64_t i, bool f32) {
  return f32 ? static_cast<const float*>(p)[i] : (float)static_cast<const T*>(p)[i];
}

// Sums of two values over the L threads of a row group (L <= 64: lanes of one
// wave; L == 256: the block, through LDS, alternating two slots so that one
// barrier a sum is enough).
template <int L>
__device__ __forceinline__ void group_sum2(float& a, float& b, float (*red)[8], int& slot) {
#pragma unroll
  for (int o = (L < 64 ? L : 64) / 2; o >= 1; o >>= 1) {
    a += __shfl_xor(a, o);
    b += __shfl_xor(b, o);
  }
  if constexpr (L > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      red[slot][wave] = a;
      red[slot][4 + wave] = b;
    }
    __syncthreads();
    a = red[slot][0] + red[slot][1] + red[slot][2] + red[slot][3];
    b = red[slot][4] + red[slot][5] + red[slot][6] + red[slot][7];
    slot ^= 1;
  }
}

// Where a thread's vector i lies: column `at`, of which the first `skip` elements
// are another thread's.  RAGGED (the width is no multiple of the vector): the
// last vector of a row is moved back to end with it; what it then shares with
// its neighbour counts there and is stored by both with the same value, so that
// every access is a whole vector.
template <int L, int VEC, bool RAGGED>
struct Place {
  int at, skip;
  bool live;
  __device__ __forceinline__ Place(int i, int t, int width) {
    const int c = (i * L + t) * VEC;
    live = c < width;
    at = RAGGED ? min(c, width - VEC) : c;
    skip = RAGGED ? c - at : 0;
  }
  __device__ __forceinline__ bool mine(int k) const { return live && (!RAGGED || k >= skip); }
};

// L threads a row, NV vectors of VEC elements a thread, NV VEC <= 32.  The next
// row's loads are out while this one's sums are formed: a row takes two rounds
// of lane exchanges, and without that the kernel waits for memory in between.
template <class T, int L, int NV, bool RAGGED>
__global__ __launch_bounds__(kNormThreads) void k_norm_fwd(
    const T* __restrict__ x, int64_t ldx, int64_t rows, int width,
    const void* __restrict__ weight, const void* __restrict__ bias, int f32_params, float eps,
    T* __restrict__ y, int64_t ldy, float* __restrict__ stats) {
  constexpr int G = kNormThreads / L;  // rows a block works on at a time
  constexpr int VEC = Vec16<T>::N;
  using Pl = Place<L, VEC, RAGGED>;
  __shared__ float red[2][8];
  int slot = 0;
  const int t = threadIdx.x % L, g = threadIdx.x / L;
  const int64_t step = (int64_t)gridDim.x * G;
  Raw<T> next[NV];
  auto fetch = [&](int64_t r) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Pl p(i, t, width);
      if (r < rows && p.live) next[i] = load_raw(x + r * ldx + p.at);
    }
  };
  int64_t r = (int64_t)blockIdx.x * G + g;
  fetch(r);
  float w[NV * VEC], b[NV * VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const Pl p(i, t, width);
    if (!p.live) continue;
    load_params<T, VEC>(weight, p.at, f32_params, 1.0f, w + i * VEC);
    load_params<T, VEC>(bias, p.at, f32_params, 0.0f, b + i * VEC);
  }
  const float inv = 1.0f / (float)width;
  for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < rows; r0 += step, r += step) {
    const bool live = r < rows;
    float v[NV * VEC], s = 0.0f, none = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Pl p(i, t, width);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        v[i * VEC + k] = live && p.live ? (float)next[i].v[k] : 0.0f;
        s += p.mine(k) ? v[i * VEC + k] : 0.0f;
      }
    }
    fetch(r + step);
    group_sum2<L>(s, none, red, slot);
    const float mean = s * inv;
    float q = 0.0f, off = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Pl p(i, t, width);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        v[i * VEC + k] -= mean;
        const float d = p.mine(k) ? v[i * VEC + k] : 0.0f;
        q = fmaf(d, d, q);
        off += d;
      }
    }
    // off: what the mean's rounding left, taken out of both moments (a
    // constant row has no variance then)
    group_sum2<L>(q, off, red, slot);
    off *= inv;
    const float rstd = 1.0f / sqrtf(fmaxf(fmaf(-off, off, q * inv), 0.0f) + eps);
    if (!live) continue;
    if (stats && t == 0) {
      stats[2 * r] = mean + off;
      stats[2 * r + 1] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Pl p(i, t, width);
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        v[i * VEC + k] = fmaf((v[i * VEC + k] - off) * rstd, w[i * VEC + k], b[i * VEC + k]);
      if (p.live) store_vec<T, VEC>(y + r * ldy + p.at, v + i * VEC);
    }
  }
}

// part[block][2][width]: the block's sums of dy xhat and dy (null: not wanted).
template <class T, int L, int NV, bool RAGGED>
__global__ __launch_bounds__(kNormThreads) void k_norm_bwd(
    const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, int64_t rows,
    int width, const void* __restrict__ weight, int f32_params, const float* __restrict__ stats,
    T* __restrict__ dx, int64_t lddx, float* __restrict__ part) {
  constexpr int G = kNormThreads / L, VEC = Vec16<T>::N;
  using Pl = Place<L, VEC, RAGGED>;
  __shared__ float red[2][8];
  __shared__ float comb[G > 1 ? 2 * kNormThreads * NV * VEC : 1];
  int slot = 0;
  const int t = threadIdx.x % L, g = threadIdx.x / L;
  const int64_t step = (int64_t)gridDim.x * G;
  Raw<T> next_x[NV], next_d[NV];
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto fetch = [&](int64_t r) __attribute__((always_inline)) {
    if (r >= rows) return;
    next_mean = stats[2 * r];
    next_rstd = stats[2 * r + 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Pl p(i, t, width);
      if (!p.live) continue;
      next_x[i] = load_raw(x + r * ldx + p.at);
      next_d[i] = load_raw(dy + r * lddy + p.at);
    }
  };
  int64_t r = (int64_t)blockIdx.x * G + g;
  fetch(r);
  float w[NV * VEC], dw[NV * VEC], db[NV * VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const Pl p(i, t, width);
    if (p.live) load_params<T, VEC>(weight, p.at, f32_params, 1.0f, w + i * VEC);
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      dw[i * VEC + k] = 0.0f;
      db[i * VEC + k] = 0.0f;
    }
  }
  const float inv = 1.0f / (float)width;
  for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < rows; r0 += step, r += step) {
    const bool live = r < rows;
    const float mean = next_mean, rstd = next_rstd;
    float xh[NV * VEC], d[NV * VEC], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Pl p(i, t, width);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const int e = i * VEC + k;
        const bool in = live && p.live;
        xh[e] = in ? ((float)next_x[i].v[k] - mean) * rstd : 0.0f;
        d[e] = in ? (float)next_d[i].v[k] : 0.0f;
        dw[e] = fmaf(d[e], xh[e], dw[e]);
        db[e] += d[e];
        d[e] = in ? d[e] * w[e] : 0.0f;
        const float m = p.mine(k) ? d[e] : 0.0f;
        s1 += m;
        s2 = fmaf(m, xh[e], s2);
      }
    }
    fetch(r + step);
    if (dx == nullptr) continue;
    group_sum2<L>(s1, s2, red, slot);
    if (!live) continue;
    s1 *= inv;
    s2 *= inv;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Pl p(i, t, width);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const int e = i * VEC + k;
        d[e] = rstd * (d[e] - s1 - xh[e] * s2);
      }
      if (p.live) store_vec<T, VEC>(dx + r * lddx + p.at, d + i * VEC);
    }
  }
  if (part == nullptr) return;
  // the block's groups, in order
  float* pw = part + (int64_t)blockIdx.x * 2 * width;
  if constexpr (G > 1) {
#pragma unroll
    for (int e = 0; e < NV * VEC; ++e) {
      comb[(2 * e) * kNormThreads + threadIdx.x] = dw[e];
      comb[(2 * e + 1) * kNormThreads + threadIdx.x] = db[e];
    }
    __syncthreads();
    for (int q = threadIdx.x; q < 2 * NV * VEC * L; q += kNormThreads) {
      const int tt = q % L, e2 = q / L, e = e2 >> 1;
      const Pl p(e / VEC, tt, width);
      float s = 0.0f;
      for (int k = 0; k < G; ++k) s += comb[e2 * kNormThreads + k * L + tt];
      if (p.mine(e % VEC)) pw[(e2 & 1) * width + p.at + e % VEC] = s;
    }
  } else {
#pragma unroll
    for (int e = 0; e < NV * VEC; ++e) {
      const Pl p(e / VEC, t, width);
      if (p.mine(e % VEC)) {
        pw[p.at + e % VEC] = dw[e];
        pw[width + p.at + e % VEC] = db[e];
      }
    }
  }
}

// Rows too wide for registers, or narrower than a vector: three passes over the
// row, which the caches hold.
template <class T>
__global__ __launch_bounds__(kNormThreads) void k_norm_fwd_wide(
    const T* __restrict__ x, int64_t ldx, int64_t rows, int64_t width,
    const void* __restrict__ weight, const void* __restrict__ bias, int f32_params, float eps,
    T* __restrict__ y, int64_t ldy, float* __restrict__ stats) {
  __shared__ float red[2][8];
  int slot = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * ldx;
    float s = 0.0f, q = 0.0f, none = 0.0f;
    for (int64_t c = threadIdx.x; c < width; c += kNormThreads) s += (float)xr[c];
    group_sum2<256>(s, none, red, slot);
    float mean = s / (float)width, off = 0.0f;
    for (int64_t c = threadIdx.x; c < width; c += kNormThreads) {
      const float d = (float)xr[c] - mean;
      q = fmaf(d, d, q);
      off += d;
    }
    group_sum2<256>(q, off, red, slot);
    off /= (float)width;
    const float rstd = 1.0f / sqrtf(fmaxf(fmaf(-off, off, q / (float)width), 0.0f) + eps);
    mean += off;
    if (stats && threadIdx.x == 0) {
      stats[2 * r] = mean;
      stats[2 * r + 1] = rstd;
    }
    for (int64_t c = threadIdx.x; c < width; c += kNormThreads) {
      const float w = weight ? load_param<T>(weight, c, f32_params) : 1.0f;
      const float b = bias ? load_param<T>(bias, c, f32_params) : 0.0f;
      y[r * ldy + c] = (T)fmaf(((float)xr[c] - mean) * rstd, w, b);
    }
  }
}

template <class T>
__global__ __launch_bounds__(kNormThreads) void k_norm_bwd_wide(
    const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, int64_t rows,
    int64_t width, const void* __restrict__ weight, int f32_params,
    const float* __restrict__ stats, T* __restrict__ dx, int64_t lddx) {
  __shared__ float red[2][8];
  int slot = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *xr = x + r * ldx, *dr = dy + r * lddy;
    const float mean = stats[2 * r], rstd = stats[2 * r + 1];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t c = threadIdx.x; c < width; c += kNormThreads) {
      const float g = (float)dr[c] * (weight ? load_param<T>(weight, c, f32_params) : 1.0f);
      s1 += g;
      s2 = fmaf(g, ((float)xr[c] - mean) * rstd, s2);
    }
    group_sum2<256>(s1, s2, red, slot);
    s1 /= (float)width;
    s2 /= (float)width;
    for (int64_t c = threadIdx.x; c < width; c += kNormThreads) {
      // g rounded as in its sum: the gradient of a single column is 0
#pragma clang fp contract(off)
      const float g = (float)dr[c] * (weight ? load_param<T>(weight, c, f32_params) : 1.0f);
      dx[r * lddx + c] = (T)(rstd * (g - s1 - ((float)xr[c] - mean) * rstd * s2));
    }
  }
}

// The wide rows' column sums: part[y][2][width] over the rows y, y + gridDim.y, ...
template <class T>
__global__ __launch_bounds__(kNormThreads) void k_norm_cols_wide(
    const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx, int64_t rows,
    int64_t width, const float* __restrict__ stats, float* __restrict__ part) {
  const int64_t c = (int64_t)blockIdx.x * kNormThreads + threadIdx.x;
  if (c >= width) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float d = (float)dy[r * lddy + c];
    dw = fmaf(d, ((float)x[r * ldx + c] - stats[2 * r]) * stats[2 * r + 1], dw);
    db += d;
  }
  part[(int64_t)blockIdx.y * 2 * width + c] = dw;
  part[(int64_t)blockIdx.y * 2 * width + width + c] = db;
}

// dweight / dbias: the sum of nblk partials, 64 columns and 16 stretches of
// partials a block, in a fixed order.
template <class T>
__global__ __launch_bounds__(1024) void k_norm_sum(const float* __restrict__ part, int nblk,
                                                   int64_t width, int f32_params,
                                                   void* __restrict__ dweight,
                                                   void* __restrict__ dbias) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;  // column of [2][width]
  float s = 0.0f;
  if (c < 2 * width) {
#pragma unroll 16
    for (int b = wave; b < nblk; b += 16) s += part[(int64_t)b * 2 * width + c];
  }
  red[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || c >= 2 * width) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) s += red[k][lane];
  void* dst = c < width ? dweight : dbias;
  if (dst == nullptr) return;
  const int64_t i = c < width ? c : c - width;
  if (f32_params)
    static_cast<float*>(dst)[i] = s;
  else
    static_cast<T*>(dst)[i] = (T)s;
}

struct NormShape {
  int L;   // threads a row: 8 .. 64, or 256; 0: the wide kernels
  int NV;  // vectors a thread
};

// A row takes the fewest lanes that hold it with one vector each, up to a wave;
// beyond 16 elements a lane of a wave, or with too few rows to fill the device
// with waves, the block shares it (bf16 x 771, backward: 1000 rows 10.3 us by blocks,
// 12.1 by waves; 1500 rows 13.4, 9.3; 12007 rows 32.5, 19.7).
template <class T>
NormShape norm_shape(int64_t rows, int64_t width) {
  constexpr int VEC = Vec16<T>::N;
  const int64_t vecs = ceil_div(width, VEC);
  auto pow2 = [](int64_t v) {
    int p = 1;
    while (p < v) p *= 2;
    return p;
  };
  if (width < VEC) return {0, 0};
  if (vecs <= 64) return {std::max(8, pow2(vecs)), 1};
  const int nv_wave = pow2(ceil_div(vecs, 64));
  if (nv_wave * VEC <= 16 && rows > 1024) return {64, nv_wave};
  const int nv = pow2(ceil_div(vecs, 256));
  if (nv * VEC > 32) return {0, 0};
  return {256, nv};
}

template <int V>
using Int = std::integral_constant<int, V>;

template <class T, class F>
void pick_shape(const NormShape& s, bool ragged, F&& f) {
  constexpr int VEC = Vec16<T>::N;
#define MGP_NORM_CASE(LL, NN)                                     \
  if (s.L == LL && s.NV == NN) {                                  \
    if (ragged) return f(Int<LL>{}, Int<NN>{}, std::true_type{}); \
    return f(Int<LL>{}, Int<NN>{}, std::false_type{});            \
  }
  MGP_NORM_CASE(8, 1)
  MGP_NORM_CASE(16, 1)
  MGP_NORM_CASE(32, 1)
  MGP_NORM_CASE(64, 1)
  MGP_NORM_CASE(64, 2)
  if constexpr (VEC == 4) { MGP_NORM_CASE(64, 4) }
  MGP_NORM_CASE(256, 1)
  MGP_NORM_CASE(256, 2)
  MGP_NORM_CASE(256, 4)
  if constexpr (VEC == 4) { MGP_NORM_CASE(256, 8) }
#undef MGP_NORM_CASE
  throw Error(ST_INTERNAL, "no layer norm kernel for this shape");
}

// Blocks of the backward pass.  Each writes one set of column sums, which the
// sum over them reads: few blocks, but enough waves to keep the memory busy
// (bf16, 12007 x 771: 1024 blocks 24 us, 512 18.7; 1000 x 4096: 512 26.5, 256 19.6).
constexpr int64_t kNormBlocks = 512, kNormBlocksLeast = 256;
inline int64_t norm_blocks(int64_t groups) {
  return std::min(groups, std::max(kNormBlocksLeast, std::min(groups / 4, kNormBlocks)));
}
constexpr int64_t kNormWideRows = 64;  // row stretches of the wide column sums

}  // namespace

void layer_norm(const NormArgs& a, void* y, int64_t y_stride, float* stats, hipStream_t st) {
  if (a.rows == 0) return;
  dispatch_elem(a.type, [&](auto tag) {
    using T = decltype(tag);
    const NormShape s = norm_shape<T>(a.rows, a.width);
    const bool ragged = a.width % Vec16<T>::N != 0;
    const T* x = static_cast<const T*>(a.x);
    if (s.L == 0) {
      k_norm_fwd_wide<T><<<(unsigned)std::min<int64_t>(a.rows, 2048), kNormThreads, 0, st>>>(
          x, a.x_stride, a.rows, a.width, a.weight, a.bias, a.f32_params, a.eps,
          static_cast<T*>(y), y_stride, stats);
    } else {
      const int64_t groups = ceil_div(a.rows, (int64_t)(kNormThreads / s.L));
      pick_shape<T>(s, ragged, [&](auto L, auto NV, auto R) {
        k_norm_fwd<T, L.value, NV.value, R.value>
            <<<(unsigned)std::min<int64_t>(groups, 2048), kNormThreads, 0, st>>>(
                x, a.x_stride, a.rows, (int)a.width, a.weight, a.bias, a.f32_params, a.eps,
                static_cast<T*>(y), y_stride, stats);
      });
    }
    MGP_HIP_CHECK(hipGetLastError());
  });
}

size_t layer_norm_backward_bytes(const NormArgs& a) {
  return (size_t)std::min<int64_t>(std::max<int64_t>(a.rows, 1), kNormBlocks) * 2 *
         (size_t)a.width * sizeof(float);
}

void layer_norm_backward(const NormArgs& a, const void* dy, int64_t dy_stride, const float* stats,
                         void* dx, int64_t dx_stride, void* dweight, void* dbias, void* ws,
                         hipStream_t st) {
  const bool cols = dweight || dbias;
  if (!cols && (dx == nullptr || a.rows == 0)) return;
  float* part = cols ? static_cast<float*>(ws) : nullptr;
  dispatch_elem(a.type, [&](auto tag) {
    using T = decltype(tag);
    const NormShape s = norm_shape<T>(a.rows, a.width);
    const bool ragged = a.width % Vec16<T>::N != 0;
    const T *x = static_cast<const T*>(a.x), *d = static_cast<const T*>(dy);
    int nblk = 0;
    if (a.rows > 0 && s.L == 0) {
      if (cols) {
        nblk = (int)std::min(a.rows, kNormWideRows);
        k_norm_cols_wide<T><<<dim3((unsigned)ceil_div(a.width, (int64_t)kNormThreads),
                                   (unsigned)nblk),
                              kNormThreads, 0, st>>>(d, dy_stride, x, a.x_stride, a.rows, a.width,
                                                     stats, part);
      }
      if (dx)  // (last: dx may be dy or x)
        k_norm_bwd_wide<T><<<(unsigned)std::min<int64_t>(a.rows, 2048), kNormThreads, 0, st>>>(
            d, dy_stride, x, a.x_stride, a.rows, a.width, a.weight, a.f32_params, stats,
            static_cast<T*>(dx), dx_stride);
    } else if (a.rows > 0) {
      const int64_t groups = ceil_div(a.rows, (int64_t)(kNormThreads / s.L));
      nblk = (int)norm_blocks(groups);
      pick_shape<T>(s, ragged, [&](auto L, auto NV, auto R) {
        k_norm_bwd<T, L.value, NV.value, R.value><<<(unsigned)nblk, kNormThreads, 0, st>>>(
            d, dy_stride, x, a.x_stride, a.rows, (int)a.width, a.weight, a.f32_params, stats,
            static_cast<T*>(dx), dx_stride, part);
      });
    }
    if (cols)
      k_norm_sum<T><<<(unsigned)ceil_div(2 * a.width, (int64_t)64), 1024, 0, st>>>(
          part, nblk, a.width, a.f32_params, dweight, dbias);
    MGP_HIP_CHECK(hipGetLastError());
  });
}

}  // namespace mgp
