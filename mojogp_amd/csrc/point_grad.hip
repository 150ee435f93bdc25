// Gradient of a kernel product's bilinear form with respect to the points:
//
//   out[i][q] = d/dx_iq sum_ab K(x_a, x_b) W_ab,   W_ab = sum_c Lf[c][a] Rf[c][b]
//             = -os / (s l_q) sum_b (W_ib + W_bi) h_ib (z_i - z_b)_q
//
// with z the scaled coordinates and h the lengthscale factor of value_and_h.
// With the columns of the marginal likelihood's gradient step ([-alpha / 2 |
// solves / (2 T)] against [alpha | probes]) this is the gradient that learned
// features receive.
//
// Two routes.  k_point_grad forms every pair's differences on the VALU: right
// for any points, and taken for Matern-1/2, whose h is unbounded, for points
// with large norms and for small sets.  k_point_grad_mm has the matrix cores
// form the distances (Gram form, as the tile products), the weights and the
// sums sum_b W h and sum_b W h z_b, which leaves the VALU the value alone;
// out is then z_i times the first minus the second.  Where that difference
// cancels (points in clusters, weights on near pairs) or weights are far below the
// largest, it has lost the digits that differences keep: every block of rows is
// weighed against the error of its sums, and one that falls short is formed again
// by k_point_grad.
#include "kval.h"
#include "provider.h"

#include <algorithm>
#include <type_traits>

namespace mgp {

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kPgBlock = 128;            // columns staged at a time
constexpr int kPgCols = 16;              // weight columns per pass
constexpr int kPgStride = kPgBlock + 16; // LDS stride of a weight column
constexpr int kPgRows = 128;             // rows of a workgroup (R = 2)

// part[split][i][q] = sum over the split's columns b of
// (W_ib + W_bi) h_ib (z_i - z_b)_q, ordered pairs.
// The symmetric weights of a 16 x 16 tile come from the fp32 matrix cores
// (four weight columns an instruction); result e belongs to the pair (column
// 4 (lane/16) + e, row lane%16), so a lane keeps its rows and their sums in
// registers and reads columns from LDS.  VALU bound: 3 d + ~12 instructions a
// pair (Matern-5/2, 8 dimensions, 50000 points: 3130 us, 0.8e12 pairs a second).
// wanted: for each block of rows whether it is formed (null: all are).
template <int KIND, int D, bool ARD, int R>
__global__ __launch_bounds__(256) void k_point_grad(
    const float* __restrict__ Z, int64_t n, int d, const float* __restrict__ Lf,
    const float* __restrict__ Rf, int cn, int64_t nb, int64_t bps,
    const int* __restrict__ wanted, float* __restrict__ part) {
  if (wanted && !wanted[blockIdx.x]) return;
  constexpr int B = kPgBlock, CS = kPgStride;
  constexpr int DS = D <= 2 ? D : (D + 3) / 4 * 4;  // LDS stride of a point
  __shared__ __align__(16) float sx[B * DS];
  __shared__ float sl[kPgCols * CS], sr[kPgCols * CS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lm = lane & 15, lq = lane >> 4;
  const int csteps = (cn + 3) / 4;

  // acc: the block's columns at hand; sum: all so far (two levels keep the
  // rounding of long sums down)
  float xi[R][D], lb[R][4], rb[R][4], acc[R][D], sum[R][D];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t i = (int64_t)blockIdx.x * (64 * R) + (wave * R + r) * 16 + lm;
#pragma unroll
    for (int k = 0; k < D; ++k) {
      xi[r][k] = (i < n && k < d) ? Z[i * d + k] : 0.0f;
      acc[r][k] = sum[r][k] = 0.0f;
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int c = 4 * s + lq;
      const bool in = i < n && c < cn;
      lb[r][s] = in ? Lf[(int64_t)c * n + i] : 0.0f;
      rb[r][s] = in ? Rf[(int64_t)c * n + i] : 0.0f;
    }
  }

  const int64_t b0 = (int64_t)blockIdx.y * bps, b1 = min(b0 + bps, nb);
  for (int64_t J = b0; J < b1; ++J) {
    const int64_t j0 = J * B;
    const int cnt = (int)min((int64_t)B, n - j0);
    __syncthreads();
    for (int q = threadIdx.x; q < B * D; q += 256) {
      const int jj = q / D, k = q - jj * D;
      sx[jj * DS + k] = (jj < cnt && k < d) ? Z[(j0 + jj) * d + k] : 0.0f;
    }
    for (int q = threadIdx.x; q < B * kPgCols; q += 256) {
      const int c = q / B, jj = q - c * B;
      const bool in = jj < cnt && c < cn;  // points past n carry no weight
      sr[c * CS + jj] = in ? Rf[(int64_t)c * n + j0 + jj] : 0.0f;
      sl[c * CS + jj] = in ? Lf[(int64_t)c * n + j0 + jj] : 0.0f;
    }
    __syncthreads();
    const int tiles = (cnt + 15) / 16;
#pragma unroll 1
    for (int ct = 0; ct < tiles; ++ct) {
      f4 wv[R];
#pragma unroll
      for (int r = 0; r < R; ++r) wv[r] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (s >= csteps) break;
        const float ar = sr[(4 * s + lq) * CS + 16 * ct + lm];
        const float al = sl[(4 * s + lq) * CS + 16 * ct + lm];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          wv[r] = __builtin_amdgcn_mfma_f32_16x16x4f32(ar, lb[r][s], wv[r], 0, 0, 0);
          wv[r] = __builtin_amdgcn_mfma_f32_16x16x4f32(al, rb[r][s], wv[r], 0, 0, 0);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float* xp = sx + (16 * ct + 4 * lq + e) * DS;
        float xj[DS];
        if constexpr (D <= 2) {
#pragma unroll
          for (int k = 0; k < D; ++k) xj[k] = xp[k];
        } else {
#pragma unroll
          for (int k = 0; k < DS; k += 4) {
            const f4 x = *reinterpret_cast<const f4*>(xp + k);
#pragma unroll
            for (int q = 0; q < 4; ++q) xj[k + q] = x[q];
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float df[D], r2 = 0.0f;
#pragma unroll
          for (int k = 0; k < D; ++k) {
            df[k] = xi[r][k] - xj[k];
            r2 = fmaf(df[k], df[k], r2);
          }
          float kv, h;
          value_and_h<KIND, ARD>(r2, kv, h);
          const float hw = h * wv[r][e];
#pragma unroll
          for (int k = 0; k < D; ++k) acc[r][k] = fmaf(hw, df[k], acc[r][k]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < D; ++k) {
        sum[r][k] += acc[r][k];
        acc[r][k] = 0.0f;
      }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t i = (int64_t)blockIdx.x * (64 * R) + (wave * R + r) * 16 + lm;
#pragma unroll
    for (int k = 0; k < D; ++k) {
      float v = sum[r][k];
      v += __shfl_xor(v, 16);
      v += __shfl_xor(v, 32);
      if (lq == 0 && i < n && k < d) part[((int64_t)blockIdx.y * n + i) * d + k] = v;
    }
  }
}

struct PgScale {
  float v[32];  // -os / (s l_q)
};

// out[i][q] (+)= scale_q sum over the splits of part[split][i][q], in order, of the
// blocks of kPgRows rows that are wanted (null: all)
__global__ __launch_bounds__(256) void k_point_grad_sum(const float* __restrict__ part,
                                                        int64_t splits, int64_t n, int d,
                                                        PgScale scale, int accumulate,
                                                        const int* __restrict__ wanted,
                                                        float* __restrict__ out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n * d;
       i += (int64_t)gridDim.x * 256) {
    if (wanted && !wanted[i / d / kPgRows]) continue;
    float s = 0.0f;
#pragma unroll 4
    for (int64_t p = 0; p < splits; ++p) s += part[p * n * d + i];
    s *= scale.v[i % d];
    out[i] = accumulate ? out[i] + s : s;
  }
}

using PgFn = void (*)(const float*, int64_t, int, const float*, const float*, int, int64_t,
                      int64_t, const int*, float*);

// below, 64-row blocks (300 points 12.7 -> 10.1 us, 2000 18.2 -> 16.4, 3000 31.0 -> 31.2)
constexpr int64_t kPgFewPoints = 3000;

// the dimension steps of the difference products (direct.hip)
template <int KIND, bool ARD, int R>
PgFn pick_pg_d(int d) {
#define MGP_PG_CASE(DV) \
  if (d <= DV) return k_point_grad<KIND, DV, ARD, R>;
  MGP_PG_CASE(1)
  MGP_PG_CASE(2)
  MGP_PG_CASE(3)
  MGP_PG_CASE(4)
  MGP_PG_CASE(5)
  MGP_PG_CASE(6)
  MGP_PG_CASE(8)
  MGP_PG_CASE(10)
  MGP_PG_CASE(12)
  MGP_PG_CASE(16)
  MGP_PG_CASE(20)
  MGP_PG_CASE(24)
  MGP_PG_CASE(32)
#undef MGP_PG_CASE
  return nullptr;
}

template <int R>
PgFn pick_pg(int kind, bool ard, int d) {
  switch (kind) {
    // the exponent clamp, the one thing ARD changes, is Matern-1/2's alone
    case KIND_RBF: return pick_pg_d<KIND_RBF, false, R>(d);
    case KIND_MATERN12:
      return ard ? pick_pg_d<KIND_MATERN12, true, R>(d) : pick_pg_d<KIND_MATERN12, false, R>(d);
    case KIND_MATERN32: return pick_pg_d<KIND_MATERN32, false, R>(d);
    default: return pick_pg_d<KIND_MATERN52, false, R>(d);
  }
}

// ---------------------------------------------------------------- matrix-core route

constexpr int kMmTiles = 4;       // 16-column tiles a stage
constexpr int kMmMaxBlocks = 64;  // partial maxima of a factor

// part[factor][block]: largest finite |value| of the columns of Lf and Rf
__global__ __launch_bounds__(256) void k_pg_max(const float* __restrict__ Lf,
                                                const float* __restrict__ Rf, int64_t count,
                                                float* __restrict__ part) {
  __shared__ float red[4];
  const float* src = blockIdx.y ? Rf : Lf;
  float m = 0.0f;
#pragma unroll 4
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += kMmMaxBlocks * 256) {
    const float a = fabsf(src[i]);
    m = a < INFINITY ? fmaxf(m, a) : m;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0)
    part[blockIdx.y * kMmMaxBlocks + blockIdx.x] =
        fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// The power of two that takes the largest value to just below 2^15.
__device__ __forceinline__ float pg_scale(const float* part, int lane) {
  float m = part[lane];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  return m > 0.0f ? ldexpf(1.0f, min(max(14 - ilogbf(m), -120), 120)) : 1.0f;
}

// Operands of the matrix-core route, a wave a 16-point tile: per tile 1 KB
// fragments [kb distance operands (of pts.A) | kw weight operands | dz
// coordinate operands] in col, the row side's weight operands in wrow.  The
// weights R_b L_a + L_b R_a of a pair are products over 6 ncols slots: the
// factors' two fp16 parts, high x high, high x low and low x high.
__global__ __launch_bounds__(256) void k_pg_pack(
    const uint4* __restrict__ A, const float* __restrict__ Z, const float* __restrict__ Lf,
    const float* __restrict__ Rf, int64_t n, int d, int ncols, int kb, int kw, int dz,
    int64_t ntiles, const float* __restrict__ maxima, uint4* __restrict__ col,
    uint4* __restrict__ wrow, float* __restrict__ unscale) {
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const float sl = pg_scale(maxima, lane), sr = pg_scale(maxima + kMmMaxBlocks, lane);
  if (blockIdx.x == 0 && threadIdx.x == 0) *unscale = (1.0f / sl) * (1.0f / sr);
  const int64_t tile = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= ntiles) return;
  uint4* dst = col + tile * (kb + kw + dz) * 64 + lane;
  for (int m = 0; m < kb; ++m) dst[m * 64] = A[(tile * kb + m) * 64 + lane];
  const int64_t i = tile * 16 + li;
  for (int m = 0; m < kw; ++m) {
    h8 a, b;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = 32 * m + 8 * g + e, p = k / (2 * ncols), j = k - p * 2 * ncols;
      float va = 0.0f, vb = 0.0f;
      if (p < 3 && i < n) {
        const int c = j < ncols ? j : j - ncols;
        const float l = Lf[(int64_t)c * n + i] * sl, r = Rf[(int64_t)c * n + i] * sr;
        va = j < ncols ? r : l;
        vb = j < ncols ? l : r;
      }
      const float ha = (float)(_Float16)va, hb = (float)(_Float16)vb;
      a[e] = (_Float16)(p == 2 ? va - ha : ha);
      b[e] = (_Float16)(p == 1 ? vb - hb : hb);
    }
    dst[(kb + m) * 64] = __builtin_bit_cast(uint4, a);
    wrow[(tile * kw + m) * 64 + lane] = __builtin_bit_cast(uint4, b);
  }
  // coordinate operand: lane (dimension li, points 4 g ..) of 16 dimensions
  for (int m = 0; m < dz; ++m) {
    f4 z;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t j = tile * 16 + 4 * g + e;
      const int q = 16 * m + li;
      z[e] = j < n && q < d ? Z[j * d + q] : 0.0f;
    }
    dst[(kb + kw + m) * 64] = __builtin_bit_cast(uint4, z);
  }
}

// h without its constant factor (3 or 5/3, in the closing scale).  Rounding
// takes the Gram form's smallest distances below zero, by no more than their
// error.
template <int KIND>
__device__ __forceinline__ float mm_h(float r2) {
  if constexpr (KIND == KIND_RBF) {
    return __builtin_amdgcn_exp2f(-r2);
  } else {
    const float u = __builtin_amdgcn_sqrtf(fabsf(r2));
    float m = fminf(u, kExp2Clamp);
    asm("" : "+v"(m));  // keeps the negation a source modifier of v_exp
    const float e = __builtin_amdgcn_exp2f(-m);
    return KIND == KIND_MATERN32 ? e : fmaf(u, kLn2, 1.0f) * e;
  }
}

template <int KB, int DZ>
struct MmStage {
  static constexpr int MAXKB = KB + 3 + DZ;                  // 1 KB fragments a tile
  static constexpr int BYTES = kMmTiles * MAXKB * 1024;
};

__device__ __forceinline__ void mm_load(const char* base, int fragments, char* __restrict__ buf) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, 0x7fffffff, 0x00020000);
  for (int i = wave; i < fragments; i += 4)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        r, (__attribute__((address_space(3))) void*)(buf + i * 1024), 16, lane * 16, i * 1024, 0,
        0);
}

template <int KIND, int KB, int DZ, int R>
__device__ __forceinline__ void mm_stage(const char* next, int fragments, int kw, bool more,
                                         const char* __restrict__ cur, char* __restrict__ nxt,
                                         int64_t tile0, int64_t row_tile0, const h8 (&bi)[R][KB],
                                         const h8 (&wb)[R][3], float (&sum)[R], float (&sq)[R],
                                         f4 (&hz)[R][DZ]) {
  if (more) mm_load(next, fragments, nxt);
  const int lane = threadIdx.x & 63, lm = lane & 15, lq = lane >> 4;
  float s1[R];
  f4 acc[R][DZ];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    s1[r] = 0.0f;
#pragma unroll
    for (int q = 0; q < DZ; ++q) acc[r][q] = f4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll(R == 4 ? 1 : 2)
  for (int t = 0; t < kMmTiles; ++t) {
    const char* c = cur + t * (KB + kw + DZ) * 1024 + lane * 16;
    h8 a[KB], wa[3];
    f4 z[DZ];
#pragma unroll
    for (int m = 0; m < KB; ++m) a[m] = *reinterpret_cast<const h8*>(c + m * 1024);
#pragma unroll
    for (int m = 0; m < 3; ++m)
      if (m < kw) wa[m] = *reinterpret_cast<const h8*>(c + (KB + m) * 1024);
#pragma unroll
    for (int m = 0; m < DZ; ++m)
      z[m] = *reinterpret_cast<const f4*>(c + (KB + kw + m) * 1024);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      f4 s = f4{0.f, 0.f, 0.f, 0.f}, w = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = 0; m < KB; ++m)
        s = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[m], bi[r][m], s, 0, 0, 0);
#pragma unroll
      for (int m = 0; m < 3; ++m)
        if (m < kw) w = __builtin_amdgcn_mfma_f32_16x16x32_f16(wa[m], wb[r][m], w, 0, 0, 0);
      float hw[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) hw[e] = mm_h<KIND>(s[e]) * w[e];
      // a point's own pair has no difference and by far the largest weight,
      // whose two sums would cancel to their rounding: left out
      if (tile0 + t == row_tile0 + r) {
#pragma unroll
        for (int e = 0; e < 4; ++e) hw[e] = lm == 4 * lq + e ? 0.0f : hw[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s1[r] += hw[e];
        sq[r] = fmaf(hw[e], hw[e], sq[r]);
#pragma unroll
        for (int q = 0; q < DZ; ++q)
          acc[r][q] = __builtin_amdgcn_mfma_f32_16x16x4f32(hw[e], z[q][e], acc[r][q], 0, 0, 0);
      }
    }
  }
  // two levels keep the rounding of long sums down (sq is for an estimate)
#pragma unroll
  for (int r = 0; r < R; ++r) {
    sum[r] += s1[r];
#pragma unroll
    for (int q = 0; q < DZ; ++q) hz[r][q] += acc[r][q];
  }
  __syncthreads();
}

// part[split][i][q] = sum_b W h z_bq and, from sums on, sums[split][0][i] = sum_b W h
// and sums[split][1][i] = sum_b (W h)^2 over the split's columns b.  Result e of a lane belongs to the pair (column
// 4 (lane/16) + e, row lane%16): W h is then the A operand of the sum over the
// columns as it stands, no lane exchanges it.  Bound by the VALU (Matern-5/2:
// 6 instructions, a square root and an exponential a pair, 224 cycles a 16 x 16
// tile) beside 192 cycles of matrix instructions of d <= 8; the two add up more than
// they overlap: 50000 points, 16 columns, the whole call 1700 us, 1.5e12 pairs a
// second; 1630 without the sum of squares and what follows from it.
template <int KIND, int KB, int DZ, int R>
__global__ __launch_bounds__(256, 3) void k_point_grad_mm(
    const char* __restrict__ col, const uint4* __restrict__ B, const uint4* __restrict__ wrow,
    int kw, int64_t n, int d, int64_t stages, int64_t sps, float* __restrict__ part,
    float* __restrict__ sums) {
  __shared__ __align__(1024) char b0[MmStage<KB, DZ>::BYTES];
  __shared__ __align__(1024) char b1[MmStage<KB, DZ>::BYTES];
  const int lane = threadIdx.x & 63, lm = lane & 15, lq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t rt0 = ((int64_t)blockIdx.x * 4 + wave) * R;
  h8 bi[R][KB], wb[R][3];
  float sum[R], sq[R];
  f4 hz[R][DZ];
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int m = 0; m < KB; ++m)
      bi[r][m] = __builtin_bit_cast(h8, B[((rt0 + r) * KB + m) * 64 + lane]);
#pragma unroll
    for (int m = 0; m < 3; ++m)
      if (m < kw) wb[r][m] = __builtin_bit_cast(h8, wrow[((rt0 + r) * kw + m) * 64 + lane]);
    sum[r] = sq[r] = 0.0f;
#pragma unroll
    for (int q = 0; q < DZ; ++q) hz[r][q] = f4{0.f, 0.f, 0.f, 0.f};
  }
  const int fragments = kMmTiles * (KB + kw + DZ);
  const int64_t bytes = (int64_t)fragments * 1024;
  int64_t st = (int64_t)blockIdx.y * sps;
  int64_t left = min(sps, stages - st);
  const char* at = col + st * bytes;
  int64_t tile = st * kMmTiles;
  // pairs of stages, so that each has its own buffers at compile time; an odd
  // one goes first
  if (left % 2 == 1) {
    mm_load(at, fragments, b1);
    __syncthreads();
    --left;
    mm_stage<KIND, KB, DZ, R>(at + bytes, fragments, kw, left > 0, b1, b0, tile, rt0, bi, wb, sum,
                              sq, hz);
    at += bytes;
    tile += kMmTiles;
  } else {
    mm_load(at, fragments, b0);
    __syncthreads();
  }
  for (; left > 0; left -= 2) {
    mm_stage<KIND, KB, DZ, R>(at + bytes, fragments, kw, true, b0, b1, tile, rt0, bi, wb, sum, sq,
                              hz);
    mm_stage<KIND, KB, DZ, R>(at + 2 * bytes, fragments, kw, left > 2, b1, b0, tile + kMmTiles,
                              rt0, bi, wb, sum, sq, hz);
    at += 2 * bytes;
    tile += 2 * kMmTiles;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float s = sum[r], s2 = sq[r];
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    s2 += __shfl_xor(s2, 16);
    s2 += __shfl_xor(s2, 32);
    const int64_t i0 = (rt0 + r) * 16;
    if (lq == 0 && i0 + lm < n) {
      sums[(int64_t)blockIdx.y * 2 * n + i0 + lm] = s;
      sums[((int64_t)blockIdx.y * 2 + 1) * n + i0 + lm] = s2;
    }
#pragma unroll
    for (int q = 0; q < DZ; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t i = i0 + 4 * lq + e;
        const int k = 16 * q + lm;
        if (i < n && k < d) part[((int64_t)blockIdx.y * n + i) * d + k] = hz[r][q][e];
      }
  }
}

// out[i][q] (+)= scale_q unscale v_iq, v_iq = z_iq S_i - sum of part, S_i = sum of
// sums, for a block of kPgRows rows, if its v stands out from the error that its sums
// left.  Over a row that is taken as
//   5e-7 |z_i| sqrt(Q_i) and 1e-6 |z_i| |S_i| of the closing difference, Q_i = sum_b (W h)^2,
//   share |z_i|^2 of v_i itself, as the distances' roundings grow with the norms,
// measured on 561 sets of 4100 to 26000 points of 2 to 31 dimensions: Gaussian,
// uniform, in clusters, in pairs, in order on a line and on a shell at the norm's
// bound, weights random, constant, smooth and those of a marginal likelihood.  A block
// passes below 3e-6 of its v; those that did were up to 2.9e-6 off (Matern) and, RBF,
// 4.1e-6 in 99 of 100, at most 8.2e-6 (points in order far out, smooth weights).
// And every row's weights have to stand out from the end of their two parts, 2^-25
// beside factors of up to 2^15: Q_i >= floor = (2^-10 / 1.5e-6)^2 2 ncols n.
// failed[block]: to be formed by differences.
__global__ __launch_bounds__(1024) void k_point_grad_mm_sum(
    const float* __restrict__ part, const float* __restrict__ sums, const float* __restrict__ Z,
    int64_t splits, int64_t n, int d, PgScale scale, const float* __restrict__ unscale,
    float floor, float share, int accumulate, int* __restrict__ failed,
    float* __restrict__ out) {
  __shared__ double total[kPgRows];
  __shared__ float value[kPgRows * 32], own[kPgRows], red[2][16];
  const int64_t row0 = (int64_t)blockIdx.x * kPgRows;
  const int rows = (int)min((int64_t)kPgRows, n - row0);
  float need = 0.0f, have = 0.0f;
  if ((int)threadIdx.x < rows) {
    const int64_t row = row0 + threadIdx.x;
    double s = 0.0, q = 0.0;
#pragma unroll 8
    for (int64_t p = 0; p < splits; ++p) {
      s += (double)sums[2 * p * n + row];
      q += (double)sums[(2 * p + 1) * n + row];
    }
    total[threadIdx.x] = s;
    float zz = 0.0f;
    for (int k = 0; k < d; ++k) zz = fmaf(Z[row * d + k], Z[row * d + k], zz);
    need = q >= (double)floor ? zz * (float)(q / 36.0 + s * s / 9.0) : INFINITY;
    const float lost = share / 3e-6f * zz;
    own[threadIdx.x] = fmaf(-lost, lost, 1.0f);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < rows * d; e += 1024) {
    double hz = 0.0;
#pragma unroll 8
    for (int64_t p = 0; p < splits; ++p) hz += (double)part[(p * n + row0) * d + e];
    const float v = (float)((double)Z[row0 * d + e] * total[e / d] - hz);
    value[e] = v;
    have = fmaf(v * own[e / d], v, have);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    need += __shfl_xor(need, o);
    have += __shfl_xor(have, o);
  }
  if ((threadIdx.x & 63) == 0) {
    red[0][threadIdx.x >> 6] = need;
    red[1][threadIdx.x >> 6] = have;
  }
  __syncthreads();
  need = have = 0.0f;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    need += red[0][w];
    have += red[1][w];
  }
  const bool passes = have >= need;  // (not where either is NaN)
  if (threadIdx.x == 0) failed[blockIdx.x] = !passes;
  if (!passes) return;
  const double un = *unscale;
  for (int e = threadIdx.x; e < rows * d; e += 1024) {
    const float v = (float)((double)scale.v[e % d] * un * (double)value[e]);
    float* o = out + row0 * d + e;
    *o = accumulate ? *o + v : v;
  }
}

using MmFn = void (*)(const char*, const uint4*, const uint4*, int, int64_t, int, int64_t, int64_t,
                      float*, float*);

struct MmKernel {
  MmFn fn;
  int dz, row_tiles;  // 16-row tiles of a workgroup
};

// Rows a wave: four 16-row tiles for many points (8 dimensions, 30000 points 619
// us, 647 with two; 50000 1701, 1750), two below, for more workgroups (10000 points
// 112 us, 120 with four; 20000 294, 315), and with two distance operands, where four
// leave too few registers (20000 points of 16 dimensions, without the sum of
// squares, 298, 335).
constexpr int64_t kMmFourTiles = 25000;
template <int KIND>
MmKernel pick_mm(int kb, int d, int64_t n) {
  if (kb == 1 && n <= kMmFourTiles) return {k_point_grad_mm<KIND, 1, 1, 2>, 1, 8};
  if (kb == 1) return {k_point_grad_mm<KIND, 1, 1, 4>, 1, 16};
  if (kb == 2 && d <= 16) return {k_point_grad_mm<KIND, 2, 1, 2>, 1, 8};
  if (kb == 2) return {k_point_grad_mm<KIND, 2, 2, 2>, 2, 8};
  if (kb == 3) return {k_point_grad_mm<KIND, 3, 2, 2>, 2, 8};
  return {nullptr, 0, 0};
}

MmKernel pick_mm(int kind, int kb, int d, int64_t n) {
  switch (kind) {
    case KIND_RBF: return pick_mm<KIND_RBF>(kb, d, n);
    case KIND_MATERN32: return pick_mm<KIND_MATERN32>(kb, d, n);
    case KIND_MATERN52: return pick_mm<KIND_MATERN52>(kb, d, n);
    default: return {nullptr, 0, 0};
  }
}

// Largest norm |z|^2 of the points for the matrix-core route: beyond it the rounding
// of the Gram form's distances alone comes near the bound of k_point_grad_mm_sum.
inline float mm_norm_bound(int kind) {
  return kind == KIND_RBF ? 32.0f : kind == KIND_MATERN32 ? 256.0f : 512.0f;
}
// and what their rounding takes of a row, over |z|^2 (k_point_grad_mm_sum)
inline float mm_error_share(int kind) {
  return kind == KIND_RBF ? 1.3e-7f : kind == KIND_MATERN32 ? 3.8e-8f : 1.7e-8f;
}
// The points from which the matrix cores' five kernels pay: the differences' time
// grows with the dimensions, theirs hardly.  Matern-5/2, 11 columns, differences
// against matrix cores: 2 dimensions, 8000 points 67 - 79 us, 12000 131 - 133, 20000 336 -
// 293; 4, 8000 77 - 80, 12000 150 - 133; 6, 4000 33 - 42, 6000 61 - 63, 8000 87 - 80; 8, 4000 43 -
// 43, 6000 72 - 64; 16, 4000 63 - 46.
inline int64_t mm_points(int d) { return d <= 4 ? 10000 : 4000; }

struct PgWork {
  Provider& pv;
  const float *Lf, *Rf;
  int ncols;  // of this pass
  bool accumulate;
  float* out;
  hipStream_t st;
};

struct PgSplit {
  int64_t nb, rb, bps, splits;  // column blocks, row blocks, column blocks a split, splits
};

PgSplit split_differences(int64_t n, bool few) {
  const int64_t nb = ceil_div(n, (int64_t)kPgBlock);
  const int64_t rb = ceil_div(n, (int64_t)(few ? kPgRows / 2 : kPgRows));
  // column splits until there are 2048 workgroups, one column block at least
  const int64_t bps = ceil_div(nb, std::min(nb, ceil_div(2048, rb)));
  return {nb, rb, bps, ceil_div(nb, bps)};
}

// part: splits n d floats.  wanted: of which blocks of kPgRows rows (null: all)
void gradient_differences(const PgWork& w, const PgScale& scale, const PgSplit& s, bool few,
                          float* part, const int* wanted) {
  const int64_t n = w.pv.n;
  const int d = w.pv.d;
  const PgFn fn = few ? pick_pg<1>(w.pv.kind, w.pv.ard, d) : pick_pg<2>(w.pv.kind, w.pv.ard, d);
  MGP_REQUIRE(fn != nullptr, "no input gradient kernel for this dimension");
  hipLaunchKernelGGL(fn, dim3((unsigned)s.rb, (unsigned)s.splits), dim3(256), 0, w.st,
                     w.pv.train.z.ptr, n, d, w.Lf, w.Rf, w.ncols, s.nb, s.bps, wanted, part);
  k_point_grad_sum<<<(unsigned)std::min<int64_t>(ceil_div(n * d, (int64_t)256), 4096), 256, 0,
                     w.st>>>(part, s.splits, n, d, scale, w.accumulate, wanted, w.out);
}

void gradient_differences(const PgWork& w, const PgScale& scale) {
  // few points: 64-row blocks, for more workgroups
  const bool few = w.pv.n < kPgFewPoints;
  const PgSplit s = split_differences(w.pv.n, few);
  float* part = w.pv.pg_buffer((size_t)s.splits * w.pv.n * w.pv.d);
  gradient_differences(w, scale, s, few, part, nullptr);
}

void gradient_matrix_cores(const PgWork& w, const MmKernel& kernel, const PgScale& scale) {
  Provider& pv = w.pv;
  const PackedPoints& pts = pv.train;
  const int64_t n = pv.n;
  const int d = pv.d, kw = (6 * w.ncols + 31) / 32, dz = kernel.dz;
  const double factor =
      pv.kind == KIND_MATERN32 ? 3.0 : pv.kind == KIND_MATERN52 ? 5.0 / 3.0 : 1.0;
  PgScale scaled = scale;
  for (int k = 0; k < d; ++k) scaled.v[k] = (float)(factor * (double)scale.v[k]);
  const int64_t stages = ceil_div(pts.ntiles, (int64_t)kMmTiles);
  const int64_t rb = ceil_div(pts.ntiles, (int64_t)kernel.row_tiles);
  const int64_t sps = ceil_div(stages, std::min(ceil_div(stages, 4), ceil_div(2048, rb)));
  const int64_t splits = ceil_div(stages, sps);
  // workgroups read whole blocks of tiles: the packing covers them
  const int64_t tiles = pts.ntiles_alloc;
  MGP_REQUIRE(rb * kernel.row_tiles <= tiles && stages * kMmTiles <= tiles, "packing too small");
  const PgSplit again = split_differences(n, false);
  size_t count = 0;  // of the buffer, in floats
  auto take = [&](size_t floats) {
    const size_t at = count;
    count += (size_t)round_up((int64_t)floats, 64);
    return at;
  };
  const size_t frag = 256;  // floats of a fragment
  const size_t col = take((size_t)tiles * (pts.kb + kw + dz) * frag);
  const size_t wrow = take((size_t)tiles * kw * frag), sums = take((size_t)splits * 2 * n);
  const size_t maxima = take(2 * kMmMaxBlocks), unscale = take(1);
  const size_t failed = take((size_t)again.rb);
  // the sums of either route: the first's are done with when the second's come
  const size_t part = take((size_t)std::max(splits, again.splits) * n * d);
  float* ws = pv.pg_buffer(count);
  int* fail = reinterpret_cast<int*>(ws + failed);
  k_pg_max<<<dim3(kMmMaxBlocks, 2), 256, 0, w.st>>>(w.Lf, w.Rf, n * w.ncols, ws + maxima);
  k_pg_pack<<<(unsigned)ceil_div(tiles, (int64_t)4), 256, 0, w.st>>>(
      reinterpret_cast<const uint4*>(pts.A.ptr), pts.z.ptr, w.Lf, w.Rf, n, d, w.ncols, pts.kb, kw,
      dz, tiles, ws + maxima, reinterpret_cast<uint4*>(ws + col),
      reinterpret_cast<uint4*>(ws + wrow), ws + unscale);
  hipLaunchKernelGGL(kernel.fn, dim3((unsigned)rb, (unsigned)splits), dim3(256), 0, w.st,
                     reinterpret_cast<const char*>(ws + col),
                     reinterpret_cast<const uint4*>(pts.B.ptr),
                     reinterpret_cast<const uint4*>(ws + wrow), kw, n, d, stages, sps, ws + part,
                     ws + sums);
  const float floor = 4.24e5f * 2.0f * (float)w.ncols * (float)n;  // (see the kernel)
  k_point_grad_mm_sum<<<(unsigned)again.rb, 1024, 0, w.st>>>(
      ws + part, ws + sums, pts.z.ptr, splits, n, d, scaled, ws + unscale, floor,
      mm_error_share(pv.kind), w.accumulate, fail, w.out);
  gradient_differences(w, scale, again, false, ws + part, fail);
}

}  // namespace

void point_gradient(Provider& pv, const float* Lf, const float* Rf, int ncols, float* out,
                    hipStream_t st) {
  MGP_REQUIRE(!pv.is_tree, "the input gradient does not serve kernel trees");
  MGP_REQUIRE(pv.d >= 1 && pv.d <= 32, "the input gradient supports d <= 32");
  const std::lock_guard<std::mutex> hold(pv.points_lock);
  PgScale scale;
  for (int k = 0; k < 32; ++k)
    scale.v[k] = k < pv.d ? (float)(-(double)pv.outputscale() /
                                    ((double)kernel_scale(pv.kind) * (double)pv.lengthscale(k)))
                          : 0.0f;
  const MmKernel mm = pv.n >= mm_points(pv.d) && pv.train.max_norm <= mm_norm_bound(pv.kind)
                          ? pick_mm(pv.kind, pv.train.kb, pv.d, pv.n)
                          : MmKernel{nullptr, 0, 0};
  const UseScope use(pv.points_use, st);
  for (int c0 = 0; c0 < ncols; c0 += kPgCols) {
    const PgWork w{pv, Lf + (int64_t)c0 * pv.n, Rf + (int64_t)c0 * pv.n,
                   std::min(kPgCols, ncols - c0), c0 > 0, out, st};
    if (mm.fn)
      gradient_matrix_cores(w, mm, scale);
    else
      gradient_differences(w, scale);
    MGP_HIP_CHECK(hipGetLastError());
  }
}

}  // namespace mgp
