// Gradient of a kernel product's bilinear form with respect to the points:
//
//   out[i][q] = d/dx_iq sum_ab K(x_a, x_b) W_ab,   W_ab = sum_c Lf[c][a] Rf[c][b]
//             = -os / (s l_q) sum_b (W_ib + W_bi) h_ib (z_i - z_b)_q
//
// with z the scaled coordinates and h the lengthscale factor of value_and_h.
// With the columns of the marginal likelihood's gradient step ([-alpha / 2 |
// solves / (2 T)] against [alpha | probes]) this is the gradient that learned
// features receive.  Differences are formed per dimension, never in Gram form:
// near pairs, which carry the gradient, keep full precision.
#include "kval.h"
#include "provider.h"

#include <algorithm>

namespace mgp {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kPgBlock = 128;            // points per block (rows and columns)
constexpr int kPgR = 2;                  // 16-row tiles per wave, 4 waves
constexpr int kPgCols = 16;              // weight columns per pass
constexpr int kPgStride = kPgBlock + 16; // LDS stride of a weight column

// part[split][i][q] = sum over the split's columns b of
// (W_ib + W_bi) h_ib (z_i - z_b)_q, ordered pairs.
// The symmetric weights of a 16 x 16 tile come from the fp32 matrix cores
// (four weight columns an instruction); result e belongs to the pair (column
// 4 (lane/16) + e, row lane%16), so a lane keeps its rows and their sums in
// registers and reads columns from LDS.  VALU bound: 3 d + ~12 instructions a
// pair.
template <int KIND, int D, bool ARD>
__global__ __launch_bounds__(256) void k_point_grad(
    const float* __restrict__ Z, int64_t n, int d, const float* __restrict__ Lf,
    const float* __restrict__ Rf, int ncols, int c0, int64_t nb, int64_t bps,
    float* __restrict__ part) {
  constexpr int R = kPgR, B = kPgBlock, CS = kPgStride;
  constexpr int DS = D <= 2 ? D : (D + 3) / 4 * 4;  // LDS stride of a point
  __shared__ __align__(16) float sx[B * DS];
  __shared__ float sl[kPgCols * CS], sr[kPgCols * CS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lm = lane & 15, lq = lane >> 4;
  const int cn = min(kPgCols, ncols - c0);
  const int csteps = (cn + 3) / 4;

  float xi[R][D], lb[R][4], rb[R][4], acc[R][D];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t i = (int64_t)blockIdx.x * B + (wave * R + r) * 16 + lm;
#pragma unroll
    for (int k = 0; k < D; ++k) {
      xi[r][k] = (i < n && k < d) ? Z[i * d + k] : 0.0f;
      acc[r][k] = 0.0f;
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int c = 4 * s + lq;
      const bool in = i < n && c < cn;
      lb[r][s] = in ? Lf[(int64_t)(c0 + c) * n + i] : 0.0f;
      rb[r][s] = in ? Rf[(int64_t)(c0 + c) * n + i] : 0.0f;
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
      sr[c * CS + jj] = in ? Rf[(int64_t)(c0 + c) * n + j0 + jj] : 0.0f;
      sl[c * CS + jj] = in ? Lf[(int64_t)(c0 + c) * n + j0 + jj] : 0.0f;
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
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t i = (int64_t)blockIdx.x * B + (wave * R + r) * 16 + lm;
#pragma unroll
    for (int k = 0; k < D; ++k) {
      float v = acc[r][k];
      v += __shfl_xor(v, 16);
      v += __shfl_xor(v, 32);
      if (lq == 0 && i < n && k < d) part[((int64_t)blockIdx.y * n + i) * d + k] = v;
    }
  }
}

struct PgScale {
  float v[32];  // -os / (s l_q)
};

// out[i][q] (+)= scale_q sum over the splits of part[split][i][q], in order
__global__ __launch_bounds__(256) void k_point_grad_sum(const float* __restrict__ part,
                                                        int64_t splits, int64_t n, int d,
                                                        PgScale scale, int accumulate,
                                                        float* __restrict__ out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n * d;
       i += (int64_t)gridDim.x * 256) {
    float s = 0.0f;
#pragma unroll 4
    for (int64_t p = 0; p < splits; ++p) s += part[p * n * d + i];
    s *= scale.v[i % d];
    out[i] = accumulate ? out[i] + s : s;
  }
}

using PgFn = void (*)(const float*, int64_t, int, const float*, const float*, int, int, int64_t,
                      int64_t, float*);

// the dimension steps of the difference products (direct.hip)
template <int KIND, bool ARD>
PgFn pick_pg_d(int d) {
#define MGP_PG_CASE(DV) \
  if (d <= DV) return k_point_grad<KIND, DV, ARD>;
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

PgFn pick_pg(int kind, bool ard, int d) {
  switch (kind) {
    // the exponent clamp, the one thing ARD changes, is Matern-1/2's alone
    case KIND_RBF: return pick_pg_d<KIND_RBF, false>(d);
    case KIND_MATERN12:
      return ard ? pick_pg_d<KIND_MATERN12, true>(d) : pick_pg_d<KIND_MATERN12, false>(d);
    case KIND_MATERN32: return pick_pg_d<KIND_MATERN32, false>(d);
    default: return pick_pg_d<KIND_MATERN52, false>(d);
  }
}

}  // namespace

void point_gradient(Provider& pv, const float* Lf, const float* Rf, int ncols, float* out,
                    hipStream_t st) {
  MGP_REQUIRE(!pv.is_tree, "the input gradient does not serve kernel trees");
  MGP_REQUIRE(pv.d >= 1 && pv.d <= 32, "the input gradient supports d <= 32");
  const int64_t n = pv.n;
  const int d = pv.d;
  const int64_t nb = ceil_div(n, (int64_t)kPgBlock);
  // column splits until there are 2048 workgroups, one column block at least
  const int64_t bps = ceil_div(nb, std::min(nb, ceil_div(2048, nb)));
  const int64_t splits = ceil_div(nb, bps);
  float* part = pv.pg_ws.ensure((size_t)splits * n * d);
  PgScale scale;
  for (int k = 0; k < 32; ++k)
    scale.v[k] = k < d ? (float)(-(double)pv.outputscale() /
                                 ((double)kernel_scale(pv.kind) * (double)pv.lengthscale(k)))
                       : 0.0f;
  const PgFn fn = pick_pg(pv.kind, pv.ard, d);
  MGP_REQUIRE(fn != nullptr, "no input gradient kernel for this dimension");
  for (int c0 = 0; c0 < ncols; c0 += kPgCols) {
    hipLaunchKernelGGL(fn, dim3((unsigned)nb, (unsigned)splits), dim3(256), 0, st, pv.train.z.ptr,
                       n, d, Lf, Rf, ncols, c0, nb, bps, part);
    k_point_grad_sum<<<(unsigned)std::min<int64_t>(ceil_div(n * d, (int64_t)256), 4096), 256, 0,
                       st>>>(part, splits, n, d, scale, c0 > 0 ? 1 : 0, out);
    MGP_HIP_CHECK(hipGetLastError());
  }
}

}  // namespace mgp
