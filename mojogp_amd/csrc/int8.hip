// Layers in 8-bit integers, for serving: y = act(s_x s_w sum q_x q_w + b), or
// gated, act(gate) * up with both projections in one product.
//
//   q = rint(x by), by = 127 / largest |x| of the row, s = largest / 127
//
// for each row of x (a point) and of the weights (a channel).  The sums are exact 32-bit
// integers, so that nothing but the two roundings to 8 bits and that of the result is
// lost, and no order of summation shows.  rint(x by) is one fused operation: added to 1.5
// 2^23, the product x by is rounded once to a whole number, ties to even, which the
// low byte then holds.
//
// Matrix-core bound at twice the 16-bit rate: the tiled product of product.h with
// 128 columns a stage; rows are quantised by one pass of their own before it.  Few
// rows (k_int8_few) are bound by reading the weights once, at half the bytes of
// 16-bit ones, and by latency: up to 16 rows each workgroup quantises what it needs
// itself, in the one launch.
#include <algorithm>
#include <type_traits>

#include "activation.h"
#include "product.h"

namespace mgp {

namespace {

constexpr float kCodeMost = 127.0f;

struct RowScale {
  float by, scale;
};
// From the bits of the largest |value|, NaN above infinity.  Rows below 2^-120 are zeros,
// rows that are not finite make NaN of every result.
__device__ __forceinline__ RowScale scale_of(uint32_t largest) {
  const float a = __uint_as_float(largest);
  if (largest < 0x03800000u) return {0.0f, 0.0f};
  if (largest >= 0x7f800000u) return {0.0f, __uint_as_float(0x7fc00000u)};
  return {kCodeMost / a, a / kCodeMost};
}

__device__ __forceinline__ uint32_t code_bits(float x, float by) {
  return __float_as_uint(fmaf(x, by, 12582912.0f));
}
// the low bytes of four values
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u),
                               __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
}

__device__ __forceinline__ uint32_t wave_largest(uint32_t u) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) u = max(u, (uint32_t)__shfl_xor((int)u, o));
  return u;
}

// 16 elements of a row from column c on, zeros past the last.
template <class T>
struct Raw16 {
  T v[16];
};
template <class T>
__device__ __forceinline__ Raw16<T> load16(const T* p, int64_t left) {
  Raw16<T> a;
  if (left >= 16) {
    __builtin_memcpy(&a, p, sizeof(a));
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) a.v[k] = k < left ? p[k] : (T)0.0f;
  }
  return a;
}
template <class T>
__device__ __forceinline__ uint32_t largest_of(const Raw16<T>& a) {
  uint32_t u = 0;
#pragma unroll
  for (int k = 0; k < 16; ++k) u = max(u, __float_as_uint((float)a.v[k]) & 0x7fffffffu);
  return u;
}
template <class T>
__device__ __forceinline__ Frag codes_of(const Raw16<T>& a, float by) {
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q)
    w[q] = pack4(code_bits((float)a.v[4 * q], by), code_bits((float)a.v[4 * q + 1], by),
                 code_bits((float)a.v[4 * q + 2], by), code_bits((float)a.v[4 * q + 3], by));
  Frag f;
  __builtin_memcpy(&f, w, 16);
  return f;
}

// ---------------------------------------------------------------- rows to codes

// A row by L threads (a wave, or the workgroup for wide rows), 16 columns each at a
// time; the first KEPT rounds stay in registers between the two passes.  HBM bound.
template <class T, int L>
__global__ __launch_bounds__(256) void k_quantize(const T* __restrict__ x, int64_t ldx,
                                                  int64_t rows, int64_t width,
                                                  int8_t* __restrict__ codes, int64_t ldc,
                                                  float* __restrict__ scales) {
  constexpr int KEPT = 2;
  __shared__ uint32_t red[4];
  const int lane = threadIdx.x & (L - 1);
  const int64_t pad = (width + 15) / 16 * 16;
  for (int64_t r = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L; r < rows;
       r += (int64_t)gridDim.x * (256 / L)) {
    const T* px = x + r * ldx;
    Raw16<T> kept[KEPT];
    uint32_t u = 0;
#pragma unroll
    for (int k = 0; k < KEPT; ++k) {
      const int64_t c = 16 * (k * L + lane);
      kept[k] = load16(px + c, width - c);
    }
#pragma unroll
    for (int k = 0; k < KEPT; ++k) u = max(u, largest_of(kept[k]));
    for (int64_t c = 16 * (KEPT * L + lane); c < width; c += 16 * L)
      u = max(u, largest_of(load16(px + c, width - c)));
    u = wave_largest(u);
    if constexpr (L > 64) {
      __syncthreads();
      if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = u;
      __syncthreads();
      u = max(max(red[0], red[1]), max(red[2], red[3]));
    }
    const RowScale s = scale_of(u);
    int8_t* pc = codes + r * ldc;
#pragma unroll
    for (int k = 0; k < KEPT; ++k) {
      const int64_t c = 16 * (k * L + lane);
      if (c < pad) {
        const Frag f = codes_of(kept[k], s.by);
        __builtin_memcpy(pc + c, &f, 16);
      }
    }
    for (int64_t c = 16 * (KEPT * L + lane); c < pad; c += 16 * L) {
      const Frag f = codes_of(load16(px + c, width - c), s.by);
      __builtin_memcpy(pc + c, &f, 16);
    }
    if (lane == 0) scales[r] = s.scale;
  }
}

// ---------------------------------------------------------------- the product's end

struct EndArgs {
  const float *sx, *sg, *su;
  const void *bg, *bu;
  void* y;
  int64_t ldy, rows, hidden;
  int act;
};

// act in place, for an activation that is the same for all threads; -1: none
template <int N, bool FAST>
__device__ __forceinline__ void act_values(int act, float* z) {
  auto go = [&](auto which) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float a, slope;
      activate<which.value, FAST>(z[k], a, slope);
      z[k] = a;
    }
  };
  if (act >= 0) dispatch_act_device(act, go);
}

// N values of one row: the sums, scaled, biased and activated.
template <class T, int N, bool GATED>
__device__ __forceinline__ void finish(const int* g, const int* u, float sx, const float* sg,
                                       const float* su, const float* bg, const float* bu, int act,
                                       float* o) {
#pragma unroll
  for (int k = 0; k < N; ++k) o[k] = fmaf((float)g[k] * sx, sg[k], bg[k]);
  act_values<N, sizeof(T) == 2>(act, o);
  if constexpr (GATED) {
#pragma unroll
    for (int k = 0; k < N; ++k) o[k] *= fmaf((float)u[k] * sx, su[k], bu[k]);
  }
}

template <int N>
__device__ __forceinline__ void zeros(float* v) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = 0.0f;
}

template <class T, bool GATED>
struct EndEpi {
  static constexpr bool FORWARD = true;
  EndArgs a;
  template <class TL>
  __device__ __forceinline__ void run(i4 (&acc)[TL::TM][TL::TN], int64_t m0, int64_t n0,
                                      int64_t) const {
    constexpr int N = TL::RUN;
    const int lane = threadIdx.x & 63;
    const int64_t f = n0 + N * (lane >> 4), left = a.hidden - f;
    if (left <= 0) return;
    float sg[N], bg[N], su[GATED ? N : 1], bu[GATED ? N : 1];
    load_run<N>(a.sg + f, left, sg);
    zeros<N>(bg);
    if (a.bg) load_run<N>(static_cast<const T*>(a.bg) + f, left, bg);
    if constexpr (GATED) {
      load_run<N>(a.su + f, left, su);
      zeros<N>(bu);
      if (a.bu) load_run<N>(static_cast<const T*>(a.bu) + f, left, bu);
    }
#pragma unroll
    for (int m = 0; m < TL::TM; ++m) {
      const int64_t r = m0 + m * 16 + (lane & 15);
      if (r >= a.rows) continue;
      int g[N], u[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        g[k] = acc[m][k / 4][k % 4];
        u[k] = GATED ? acc[m][TL::T1 % TL::TN + k / 4][k % 4] : 0;
      }
      float o[N];
      finish<T, N, GATED>(g, u, a.sx[r], sg, su, bg, bu, a.act, o);
      store_run<N>(static_cast<T*>(a.y) + r * a.ldy + f, left, o);
    }
  }
};

// ---------------------------------------------------------------- few rows

struct FewArgs {
  EndArgs end;
  const void* x;  // FUSED: rows of elements, otherwise of codes
  int64_t ldx;
  const int8_t *wg, *wu;
  int64_t ldw, width;
};

// A workgroup takes 16 columns (of both projections) for 16 MT rows; its 8 waves share
// the reduction and read their fragments from memory.  FUSED: the rows are elements; the
// workgroup first finds their largest values.
template <class T, int MT, bool GATED, bool FUSED>
__global__ __launch_bounds__(512) void k_int8_few(FewArgs s) {
  constexpr int W = 8, P = GATED ? 2 : 1;
  __shared__ i4 red[W][P * MT][64];
  __shared__ uint32_t largest[W][16];
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const EndArgs& a = s.end;
  const int64_t f0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * 16 * MT;
  // rows past the last are read as the last and not stored
  const int64_t f = min(f0 + i, a.hidden - 1);
  const int8_t *wg = s.wg + f * s.ldw, *wu = GATED ? s.wu + f * s.ldw : nullptr;
  const int64_t pad = (s.width + 15) / 16 * 16;
  i4 sums[P * MT];
#pragma unroll
  for (int t = 0; t < P * MT; ++t) sums[t] = i4{0, 0, 0, 0};
  auto codes = [&](const int8_t* p, int64_t k) __attribute__((always_inline)) {
    Frag r{f4{0.0f, 0.0f, 0.0f, 0.0f}};
    if (k < pad) __builtin_memcpy(&r, p + k, 16);
    return r;
  };
  float sx[MT];
  if constexpr (FUSED) {
    static_assert(MT == 1, "");
    const T* px = static_cast<const T*>(s.x) + min(m0 + i, a.rows - 1) * s.ldx;
    uint32_t u = 0;
    for (int64_t k = wave * 64 + g * 16; k < s.width; k += W * 64)
      u = max(u, largest_of(load16(px + k, s.width - k)));
    u = max(u, (uint32_t)__shfl_xor((int)u, 16));
    u = max(u, (uint32_t)__shfl_xor((int)u, 32));
    if (g == 0) largest[wave][i] = u;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) u = max(u, largest[w][i]);
    const RowScale r = scale_of(u);
    sx[0] = r.scale;
    for (int64_t k0 = wave * 64; k0 < s.width; k0 += W * 64) {
      const int64_t k = k0 + g * 16;
      const Frag q = codes_of(load16(px + k, s.width - k), r.by);
      sums[0] = mma_i8(codes(wg, k), q, sums[0]);
      if constexpr (GATED) sums[1] = mma_i8(codes(wu, k), q, sums[1]);
    }
  } else {
    const int8_t* x[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int64_t r = min(m0 + 16 * t + i, a.rows - 1);
      x[t] = static_cast<const int8_t*>(s.x) + r * s.ldx;
      sx[t] = a.sx[r];
    }
#pragma unroll 2
    for (int64_t k0 = wave * 64; k0 < s.width; k0 += W * 64) {
      const int64_t k = k0 + g * 16;
      const Frag pg = codes(wg, k), pu = GATED ? codes(wu, k) : pg;
      Frag q[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) q[t] = codes(x[t], k);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        sums[P * t] = mma_i8(pg, q[t], sums[P * t]);
        if constexpr (GATED) sums[P * t + 1] = mma_i8(pu, q[t], sums[P * t + 1]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < P * MT; ++t) red[wave][t][lane] = sums[t];
  __syncthreads();
  if (wave >= MT) return;
  float scale = sx[0];
#pragma unroll
  for (int t = 1; t < MT; ++t) scale = wave == t ? sx[t] : scale;
  i4 tg = red[0][P * wave][lane], tu = red[0][P * wave + P - 1][lane];
#pragma unroll
  for (int w = 1; w < W; ++w) {
    tg += red[w][P * wave][lane];
    tu += red[w][P * wave + P - 1][lane];
  }
  const int64_t r = m0 + 16 * wave + i, c = f0 + 4 * g, left = a.hidden - c;
  if (r >= a.rows || left <= 0) return;
  float sg[4], su[4], bg[4], bu[4], o[4];
  zeros<4>(bg);
  zeros<4>(bu);
  load_run<4>(a.sg + c, left, sg);
  if (a.bg) load_run<4>(static_cast<const T*>(a.bg) + c, left, bg);
  if constexpr (GATED) {
    load_run<4>(a.su + c, left, su);
    if (a.bu) load_run<4>(static_cast<const T*>(a.bu) + c, left, bu);
  }
  const int ig[4] = {tg[0], tg[1], tg[2], tg[3]}, iu[4] = {tu[0], tu[1], tu[2], tu[3]};
  finish<T, 4, GATED>(ig, iu, scale, sg, su, bg, bu, a.act, o);
  store_run<4>(static_cast<T*>(a.y) + r * a.ldy + c, left, o);
}

// ---------------------------------------------------------------- host side

template <class T>
void launch_quantize(const T* x, int64_t ldx, int64_t rows, int64_t width, int8_t* codes,
                     int64_t ldc, float* scales, hipStream_t st) {
  const bool wide = width > 64 * 32;  // more than a wave keeps
  const int64_t blocks = wide ? rows : ceil_div(rows, (int64_t)4);
  const unsigned grid = (unsigned)std::min<int64_t>(blocks, 1 << 16);
  if (wide)
    k_quantize<T, 256><<<grid, 256, 0, st>>>(x, ldx, rows, width, codes, ldc, scales);
  else
    k_quantize<T, 64><<<grid, 256, 0, st>>>(x, ldx, rows, width, codes, ldc, scales);
}

enum Way : int { FUSED_ROWS, FEW_ROWS, TILES };

inline Way way_of(const Int8Args& a) {
  if (a.rows <= 16) return FUSED_ROWS;
  return ceil_div(a.rows, (int64_t)64) * ceil_div(a.hidden, (int64_t)16) <= 512 ? FEW_ROWS : TILES;
}

inline int64_t padded(int64_t width) { return round_up(width, 16); }

template <class T, bool GATED>
void launch_layer(const Int8Args& a, const EndArgs& end, const int8_t* codes, hipStream_t st) {
  const int64_t ldx = padded(a.width);
  const Way way = way_of(a);
  if (way != TILES) {
    FewArgs s{end, a.x, a.x_stride, a.w_gate, a.w_up, a.w_stride, a.width};
    const unsigned gx = (unsigned)ceil_div(a.hidden, (int64_t)16);
    auto go = [&](auto mt, auto fused) {
      k_int8_few<T, mt.value, GATED, fused.value>
          <<<dim3(gx, (unsigned)ceil_div(a.rows, (int64_t)(16 * mt.value))), 512, 0, st>>>(s);
    };
    if (way == FUSED_ROWS) return go(std::integral_constant<int, 1>{}, std::true_type{});
    s.x = codes;
    s.ldx = ldx;
    if (a.rows <= 32) return go(std::integral_constant<int, 2>{}, std::false_type{});
    return go(std::integral_constant<int, 4>{}, std::false_type{});
  }
  GemmShape s{};
  s.p = {reinterpret_cast<const char*>(a.w_gate), reinterpret_cast<const char*>(a.w_up), a.w_stride,
         a.hidden};
  s.q = {reinterpret_cast<const char*>(codes), nullptr, ldx, a.rows};
  s.K = s.k_split = ldx;
  const EndEpi<T, GATED> epi{end};
  const bool big = cut_product((GATED ? 2 : 1) * a.hidden, a.rows, ceil_div(ldx, (int64_t)128), 1,
                               true, 1, 0.0)
                       .big;
  if (big)
    launch_tiles<BigTile<int8_t, false, GATED, 1>>(s, 1, epi, st);
  else
    launch_tiles<SmallTile<int8_t, false, GATED, 1>>(s, 1, epi, st);
}

}  // namespace

void int8_quantize(int type, const void* x, int64_t x_stride, int64_t rows, int64_t width,
                   int8_t* codes, int64_t codes_stride, float* scales, hipStream_t st) {
  if (rows == 0) return;
  dispatch_elem(type, [&](auto tag) {
    using T = decltype(tag);
    launch_quantize<T>(static_cast<const T*>(x), x_stride, rows, width, codes, codes_stride, scales,
                       st);
  });
  MGP_HIP_CHECK(hipGetLastError());
}

size_t int8_bytes(const Int8Args& a) {
  if (a.rows == 0 || way_of(a) == FUSED_ROWS) return 0;
  return align_up((size_t)(a.rows * padded(a.width))) + align_up((size_t)a.rows * sizeof(float));
}

void int8_layer(const Int8Args& a, void* y, int64_t y_stride, void* ws, hipStream_t st) {
  if (a.rows == 0) return;
  int8_t* codes = static_cast<int8_t*>(ws);
  float* sx = nullptr;
  if (way_of(a) != FUSED_ROWS) {
    sx = reinterpret_cast<float*>(codes + align_up((size_t)(a.rows * padded(a.width))));
    int8_quantize(a.type, a.x, a.x_stride, a.rows, a.width, codes, padded(a.width), sx, st);
  }
  const EndArgs end{sx, a.s_gate, a.s_up, a.b_gate, a.b_up, y, y_stride, a.rows, a.hidden,
                    a.activation};
  dispatch_elem(a.type, [&](auto tag) {
    using T = decltype(tag);
    if (a.w_up)
      launch_layer<T, true>(a, end, codes, st);
    else
      launch_layer<T, false>(a, end, codes, st);
  });
  MGP_HIP_CHECK(hipGetLastError());
}

}  // namespace mgp
