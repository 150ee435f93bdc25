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
// dg and du are rounded to the element type before the last two products, as
// the matrix cores take them; g, u, all sums and the bias gradients stay fp32.
#include "layers.h"

#include <algorithm>

namespace mgp {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

#define MGP_LDS __attribute__((address_space(3)))

// ---------------------------------------------------------------- activation

// 1 / (1 + exp(-g)).  FAST (the 16-bit types): one v_exp and one v_rcp, good to
// a few fp32 roundings, where expf and a division cost ~40 instructions (the
// epilogue of 65536 x 1024 -> 4096 took a quarter of the kernel's time).
template <bool FAST>
__device__ __forceinline__ float sigmoid(float g) {
  if constexpr (FAST)
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * g));
  else
    return 1.0f / (1.0f + expf(-g));
}

// a = act(g) and its derivative
template <int ACT, bool FAST>
__device__ __forceinline__ void activate(float g, float& a, float& slope) {
  if constexpr (ACT == ACT_SILU) {
    const float s = sigmoid<FAST>(g);
    a = g * s;
    slope = s * fmaf(g, 1.0f - s, 1.0f);
  } else if constexpr (ACT == ACT_SIGMOID) {
    a = sigmoid<FAST>(g);
    slope = a * (1.0f - a);
  } else if constexpr (ACT == ACT_RELU) {
    a = g > 0.0f || g != g ? g : 0.0f;
    slope = g > 0.0f ? 1.0f : 0.0f;
  } else if constexpr (FAST) {
    // the normal integral by Abramowitz and Stegun 7.1.26 (absolute error
    // 1.5e-7, a thousandth of the 16-bit types' rounding), whose exponential
    // the derivative takes too
    const float x = fabsf(g) * 0.70710678118654752f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.0f));
    const float e = __builtin_amdgcn_exp2f(-0.5f * kLog2e * g * g);
    const float q =
        t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f),
                         -0.284496736f),
                 0.254829592f);
    const float tail = 0.5f * q * e;  // 1 - Phi(|g|)
    const float cdf = g > 0.0f ? 1.0f - tail : tail;
    a = g * cdf;
    slope = fmaf(g * 0.39894228040143268f, e, cdf);
  } else {
    const float cdf = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
    a = g * cdf;
    slope = fmaf(g * 0.39894228040143268f, expf(-0.5f * g * g), cdf);
  }
}

// N consecutive elements of a row, of which `left` exist; whole runs go as
// vectors, which the memory path takes at any alignment.
template <int N, class T>
__device__ __forceinline__ void load_run(const T* p, int64_t left, float* v) {
  if (left >= N) {
    T a[N];
    __builtin_memcpy(a, p, N * sizeof(T));
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = (float)a[k];
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = k < left ? (float)p[k] : 0.0f;
  }
}

template <int N, class T>
__device__ __forceinline__ void store_run(T* p, int64_t left, const float* v) {
  if (left >= N) {
    T a[N];
#pragma unroll
    for (int k = 0; k < N; ++k) a[k] = (T)v[k];
    __builtin_memcpy(p, a, N * sizeof(T));
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k < left) p[k] = (T)v[k];
  }
}

// ---------------------------------------------------------------- product core

// A 16-byte operand fragment: 8 narrow elements of 32 reduction steps spread
// over the lane groups, or 4 floats of 16.
struct Frag {
  f4 v;
};

template <class T>
__device__ __forceinline__ f4 mma(const Frag& a, const Frag& b, f4 c) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[k], b.v[k], c, 0, 0, 0);
    return c;
  } else if constexpr (std::is_same<T, __bf16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a.v),
                                                   __builtin_bit_cast(b8, b.v), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a.v),
                                                  __builtin_bit_cast(h8, b.v), c, 0, 0, 0);
  }
}

constexpr int kStageBytes = 128;        // reduction bytes of a row a stage
constexpr int kOutOfRange = (int)0x80000000u;  // past num_records: the load gives zeros
constexpr int kNumRecords = 0x7fffffff;

__device__ __forceinline__ void load_lds(const char* base, int voff, char* __restrict__ dst) {
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, kNumRecords, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (MGP_LDS void*)dst, 16, voff, 0, 0, 0);
}

// One operand of a product: element (row, k) at base + row ld + k (NT) or
// (k, row) at base + k ld + row (TN); rows < n, k < K.  Two: rows alternate
// between two matrices within each wave's share of a tile (gate and up).
struct Operand {
  const char* base;
  const char* base2;
  int64_t ld_bytes;
  int64_t n;
};

struct GemmShape {
  Operand p, q;       // p: the side whose rows are the output's columns
  int64_t K;          // reduction length
  int64_t tiles_p, tiles_q;
  int64_t k_split;    // reduction elements of one split (a multiple of a stage)
};

// Tile of 16 TN WN columns (p rows) by 16 TM WM rows (q rows), one wave 16 TN
// by 16 TM of it.  NT: the p rows are dealt to LDS so that a lane's results are
// RUN = 4 TN (dual: 2 TN of each matrix) consecutive columns.  Both operands go through LDS by direct loads, double
// buffered, 128 bytes of reduction a stage.  NT: 128-byte LDS rows, 16-byte
// chunk c of row r at c ^ (r / 2 % 8).  TN: LDS rows of the tile's width, one
// per reduction step, in the memory's order; 32-byte granules at g ^ (r % 8)
// (narrow types, read by the transposing LDS load), 64-byte ones at g ^ (r % 4)
// (fp32): both keep the fragment reads off each other's banks.
template <class T, int TM_, int TN_, int WM_, int WN_, bool TR_, bool DUAL_>
struct Tile {
  using Elem = T;
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_;
  static constexpr bool TR = TR_, DUAL = DUAL_;
  static constexpr int W = WM * WN, THREADS = 64 * W;
  static constexpr int BQ = 16 * TM * WM, BP = 16 * TN * WN;
  static constexpr int T1 = DUAL ? TN / 2 : TN;  // 16-row tiles of one matrix a wave
  static constexpr int RUN = 4 * T1;
  static constexpr int E = sizeof(T);
  static constexpr int KS = kStageBytes / E;       // reduction elements a stage
  static constexpr int LDS = (BP + BQ) * kStageBytes;  // one buffer
  static constexpr int IP = BP * kStageBytes / 1024 / W, IQ = BQ * kStageBytes / 1024 / W;
  static_assert(IP * W * 1024 == BP * kStageBytes && IQ * W * 1024 == BQ * kStageBytes, "");
};

// What a wave loads of a stage: I instructions a side, each 64 lanes x 16 bytes
// = 1 KB of LDS.  The instructions of a side lie a multiple of 8 LDS rows (TN:
// of 8, fp32 4, reduction rows) apart, so the lanes' offsets from each one's
// uniform base are the same; only which rows exist differs.
template <class TL>
struct Loader {
  static constexpr int I = TL::IP + TL::IQ;
  int voff[2];        // byte offset of the lane from an instruction's base
  int kpos[2];        // NT: its reduction element, TN: its reduction row within the stage
  bool exists[I];     // NT: its row is one of the matrix
  const char* base[I];

  template <bool P>
  __device__ __forceinline__ void init_side(const Operand& o, int64_t row0, int64_t k0) {
    constexpr int N = P ? TL::IP : TL::IQ, S = P ? 0 : TL::IP;
    constexpr int B = P ? TL::BP : TL::BQ;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if constexpr (!TL::TR) {
      static_assert(TL::W % 2 == 0, "");  // the swizzle is that of wave * 8 + lane / 8
      const int l8 = lane / 8;
      const int c = (lane & 7) ^ ((wave * 4 + lane / 16) & 7);
      // P: LDS row (wave w, matrix, tile t, row i) holds column
      // 16 T1 w + (i / 4) RUN + 4 t + i % 4
      const int lrow = P ? l8 / 4 * TL::RUN + l8 % 4 : l8;
      kpos[!P] = c * (16 / TL::E);
      voff[!P] = (int)(lrow * o.ld_bytes) + c * 16;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r8 = (i * TL::W + wave) * 8;
        int64_t r = row0 + r8;
        const char* from = o.base;
        if constexpr (P) {
          const int t = r8 % (16 * TL::TN) / 16;
          const bool up = t >= TL::T1;  // wave uniform
          r = row0 + r8 / (16 * TL::TN) * 16 * TL::T1 + r8 % 16 / 4 * TL::RUN +
              (up ? t - TL::T1 : t) * 4;
          if (up) from = o.base2;
        }
        exists[S + i] = r + lrow < o.n;
        base[S + i] = from + r * o.ld_bytes + k0 * TL::E;
      }
    } else {
      constexpr int RB = B * TL::E;  // bytes of an LDS row
      static_assert(TL::W * 1024 / RB % 8 == 0, "");
      const int byte = wave * 1024 + lane * 16, r = byte / RB, rb = wave * 1024 / RB;
      const int c = (byte % RB / 16) ^
                    ((TL::E == 2 ? ((r & 7) << 1) : ((r & 3) << 2)) & (RB / 16 - 1));
      const bool in = row0 + c * (16 / TL::E) < o.n;
      kpos[!P] = r;
      voff[!P] = (int)((r - rb) * o.ld_bytes) + c * 16;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        exists[S + i] = in;
        base[S + i] = o.base + (k0 + i * (TL::W * 1024 / RB) + rb) * o.ld_bytes + row0 * TL::E;
      }
    }
  }

  // Loads the stage of `left` remaining reduction elements into buf and moves on.
  __device__ __forceinline__ void load(char* __restrict__ buf, int64_t left, int64_t ldp,
                                       int64_t ldq) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l = (int)min(left, (int64_t)TL::KS);
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const bool p = i < TL::IP;
      const int j = p ? i : i - TL::IP;
      char* dst = buf + (p ? 0 : TL::BP * kStageBytes) + (j * TL::W + wave) * 1024;
      const int step = TL::TR ? j * (TL::W * 1024 / ((p ? TL::BP : TL::BQ) * TL::E)) : 0;
      load_lds(base[i], exists[i] && kpos[!p] < l - step ? voff[!p] : kOutOfRange, dst);
      base[i] += TL::TR ? (int64_t)TL::KS * (p ? ldp : ldq) : (int64_t)kStageBytes;
    }
  }
};

template <class TL, int B>
__device__ __forceinline__ Frag read_frag(const char* __restrict__ buf, int row, int ks) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  if constexpr (!TL::TR) {
    const int c = (ks * 4 + g) ^ (i >> 1);
    return {*reinterpret_cast<const f4*>(buf + (row + i) * kStageBytes + c * 16)};
  } else if constexpr (TL::E == 2) {
    // lane group g takes reduction rows 4 g .. 4 g + 3 and the same + 16; the
    // transposing load gives lane i the four rows' elements of column i
    constexpr int RB = B * TL::E, M = RB / 32 - 1;
    const int r = ks * 32 + 4 * g + (i >> 2);
    const int a = r * RB + (((row >> 4) ^ ((r & 7) & M)) * 32) + (i & 3) * 8;
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MGP_LDS s4*)(buf + a));
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MGP_LDS s4*)(buf + a + 16 * RB));
    typedef short s8 __attribute__((ext_vector_type(8)));
    const s8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return {__builtin_bit_cast(f4, v)};
  } else {
    constexpr int RB = B * TL::E;
    Frag f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = ks * 16 + 4 * k + g, col = row + i;  // r % 4 = g
      f.v[k] = *reinterpret_cast<const float*>(
          buf + r * RB + (((col >> 2) ^ ((g << 2) & (RB / 16 - 1))) << 4) + (col & 3) * 4);
    }
    return f;
  }
}

template <class TL>
__device__ __forceinline__ void compute(const char* __restrict__ cur, int wm, int wn,
                                        f4 (&acc)[TL::TM][TL::TN]) {
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    Frag p[TL::TN], q[TL::TM];
#pragma unroll
    for (int t = 0; t < TL::TN; ++t) p[t] = read_frag<TL, TL::BP>(cur, (wn * TL::TN + t) * 16, ks);
#pragma unroll
    for (int t = 0; t < TL::TM; ++t)
      q[t] = read_frag<TL, TL::BQ>(cur + TL::BP * kStageBytes, (wm * TL::TM + t) * 16, ks);
#pragma unroll
    for (int m = 0; m < TL::TM; ++m)
#pragma unroll
      for (int n = 0; n < TL::TN; ++n) acc[m][n] = mma<typename TL::Elem>(p[n], q[m], acc[m][n]);
  }
}

// One stage: the loads of the next go out before this one's fragments are
// read.  The two buffers are distinct restrict arguments, so that the reads
// need not wait for the loads in flight; the closing barrier waits for those
// and for every wave's reads.
template <class TL>
__device__ __forceinline__ void stage(Loader<TL>& ld, char* __restrict__ cur,
                                      char* __restrict__ nxt, int64_t left_next, int64_t ldp,
                                      int64_t ldq, int wm, int wn, f4 (&acc)[TL::TM][TL::TN]) {
  if (left_next > 0) ld.load(nxt, left_next, ldp, ldq);
  compute<TL>(cur, wm, wn, acc);
  __syncthreads();
}

// Workgroups go round the 8 XCDs in turn: each XCD takes a stretch of tiles of
// its own, ordered in groups of 8 tile rows, so that what its L2 holds serves
// the tiles in flight on it.
__device__ __forceinline__ void tile_of(int64_t id, int64_t tiles_p, int64_t tiles_q, int64_t& tp,
                                        int64_t& tq) {
  const int64_t total = tiles_p * tiles_q, xcd = id & 7, per = total >> 3, rest = total & 7;
  id = xcd * per + min(xcd, rest) + (id >> 3);
  const int64_t group = id / (8 * tiles_p), in = id - group * 8 * tiles_p;
  const int64_t height = min((int64_t)8, tiles_q - group * 8);
  tq = group * 8 + in % height;
  tp = in / height;
}

// acc[tm][tn][e] of lane l holds output row 16 (wm TM + tm) + l % 16 and column
// (NT, tn < T1) 16 T1 wn + RUN (l / 16) + 4 tn + e of either matrix, (TN)
// 16 (wn TN + tn) + 4 (l / 16) + e.
template <class TL, class EPI>
__global__ __launch_bounds__(TL::THREADS) void k_gemm(GemmShape s, EPI epi) {
  __shared__ __align__(1024) char b0[TL::LDS];
  __shared__ __align__(1024) char b1[TL::LDS];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % TL::WM, wn = wave / TL::WM;
  int64_t tp, tq;
  tile_of(blockIdx.x, s.tiles_p, s.tiles_q, tp, tq);
  constexpr int CP = TL::DUAL ? TL::BP / 2 : TL::BP;  // output columns a tile
  const int64_t n0 = (int64_t)tp * CP, m0 = (int64_t)tq * TL::BQ;
  const int64_t k0 = (int64_t)blockIdx.y * s.k_split;
  const int64_t K = min(s.k_split, s.K - k0);

  f4 acc[TL::TM][TL::TN];
#pragma unroll
  for (int m = 0; m < TL::TM; ++m)
#pragma unroll
    for (int n = 0; n < TL::TN; ++n) acc[m][n] = f4{0.f, 0.f, 0.f, 0.f};

  Loader<TL> ld;
  ld.template init_side<true>(s.p, n0, k0);
  ld.template init_side<false>(s.q, m0, k0);
  const int64_t ldp = s.p.ld_bytes, ldq = s.q.ld_bytes;
  // pairs of stages, so that each has its own buffers at compile time; an odd
  // one goes first
  int64_t left = K;
  if ((K + TL::KS - 1) / TL::KS % 2 == 1) {
    ld.load(b1, left, ldp, ldq);
    __syncthreads();
    left -= TL::KS;
    stage<TL>(ld, b1, b0, left, ldp, ldq, wm, wn, acc);
  } else {
    ld.load(b0, left, ldp, ldq);
    __syncthreads();
  }
  while (left > 0) {
    left -= TL::KS;
    stage<TL>(ld, b0, b1, left, ldp, ldq, wm, wn, acc);
    left -= TL::KS;
    stage<TL>(ld, b1, b0, left, ldp, ldq, wm, wn, acc);
  }
  epi.template run<TL>(acc, m0 + wm * TL::TM * 16, n0 + wn * (CP / TL::WN), tq * TL::WM + wm);
}

// ---------------------------------------------------------------- epilogues

template <class T, int ACT>
struct ForwardEpi {
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
template <class T, int ACT>
struct BackwardEpi {
  const T *bg, *bu;
  const T* dh;
  int64_t lddh, rows, hidden, pad;
  T* dgu;
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
      store_run<N>(dgu + r * 2 * pad + f, pad - f, dg);
      store_run<N>(dgu + r * 2 * pad + pad + f, pad - f, du);
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

template <class T>
struct StoreEpi {
  T* out;
  int64_t ld, rows, cols;
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
      store_run<N>(out + r * ld + c, cols - c, o);
    }
  }
};

// Rows of [dg | du]^T x: row m < pad of dw_gate, row m - pad of dw_up.  One
// split: the gradients themselves; more: part[split][2][hidden][width] sums.
template <class T>
struct WeightEpi {
  T *dw_gate, *dw_up;
  float* part;
  int64_t hidden, pad, width;
  template <class TL>
  __device__ __forceinline__ void run(f4 (&acc)[TL::TM][TL::TN], int64_t m0, int64_t n0,
                                      int64_t) const {
    const int lane = threadIdx.x & 63;
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
        float o[4] = {acc[m][n][0], acc[m][n][1], acc[m][n][2], acc[m][n][3]};
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

// dst[row][cols_pad] = src[row][cols], zeros past cols
template <class T>
__global__ __launch_bounds__(256) void k_pack_rows(const T* __restrict__ src, int64_t ld,
                                                   int64_t rows, int64_t cols, int64_t cols_pad,
                                                   T* __restrict__ dst) {
  constexpr int N = Vec16<T>::N;
  const int64_t per = cols_pad / N, total = rows * per;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total;
       q += (int64_t)gridDim.x * 256) {
    const int64_t r = q / per, c = (q - r * per) * N;
    Vec16<T> v;
#pragma unroll
    for (int k = 0; k < N; ++k) v.v[k] = c + k < cols ? src[r * ld + c + k] : (T)0.0f;
    *reinterpret_cast<Vec16<T>*>(dst + r * cols_pad + c) = v;
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

// out_g / out_u [count] = sums over the parts of part[parts][2][count], in order
template <class T>
__global__ __launch_bounds__(256) void k_sum_parts(const float* __restrict__ part, int64_t parts,
                                                   int64_t count, T* __restrict__ out_g,
                                                   T* __restrict__ out_u) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < 2 * count;
       i += (int64_t)gridDim.x * 256) {
    const bool up = i >= count;
    T* dst = up ? out_u : out_g;
    if (dst == nullptr) continue;
    float s = 0.0f;
#pragma unroll 8
    for (int64_t p = 0; p < parts; ++p) s += part[p * 2 * count + i];
    dst[i - (up ? count : 0)] = (T)s;
  }
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

// ---------------------------------------------------------------- host side

// Rows the product kernel can load directly: 16-byte aligned, whole 16-byte
// chunks, and the rows of one load within 31-bit offsets.
template <class T>
bool direct(const void* p, int64_t stride, int64_t cols) {
  return aligned16(p) && stride % Vec16<T>::N == 0 && cols % Vec16<T>::N == 0 &&
         stride * (int64_t)sizeof(T) < (int64_t)1 << 26;
}

constexpr size_t kAlign = 256;
inline size_t align_up(size_t b) { return (b + kAlign - 1) / kAlign * kAlign; }

// The two tile sizes: 256 x 256, one workgroup of 8 waves a CU, and 128 x 128,
// two workgroups of 4 waves, for what would leave CUs idle otherwise.
template <class T, bool TR, bool DUAL>
using BigTile = Tile<T, 8, 4, 2, 4, TR, DUAL>;
template <class T, bool TR, bool DUAL>
using SmallTile = Tile<T, 4, 4, 2, 2, TR, DUAL>;
constexpr int64_t kBigTiles = 512;  // 256 x 256 tiles from which on they are taken
inline bool big_tiles(int64_t p_rows, int64_t q_rows) {
  return ceil_div(p_rows, (int64_t)256) * ceil_div(q_rows, (int64_t)256) >= kBigTiles;
}
constexpr int64_t kSplitTarget = 512;  // workgroups the weight gradient aims at

// What a call needs and where it lies in the workspace.
template <class T>
struct Plan {
  int64_t wpad, hpad;  // width and hidden rounded to whole 16-byte chunks
  bool pack_x, pack_w;
  size_t x_off = 0, wg_off = 0, wu_off = 0, wt_off = 0, dgu_off = 0, dbias_off = 0, part_off = 0;
  size_t bytes = 0;
  bool big_dual = false, big_dx = false, big_dw = false;
  int64_t bias_parts = 0, splits = 1, k_split = 0;

  Plan(const GatedArgs& a, bool backward) {
    constexpr int N = Vec16<T>::N;
    wpad = round_up(a.width, N);
    hpad = round_up(a.hidden, N);
    pack_x = !direct<T>(a.x, a.x_stride, a.width);
    pack_w = !direct<T>(a.w_gate, a.w_gate_stride, a.width) ||
             !direct<T>(a.w_up, a.w_up_stride, a.width) || a.w_gate_stride != a.w_up_stride;
    auto take = [&](size_t n) {
      const size_t at = bytes;
      bytes += align_up(n);
      return at;
    };
    if (pack_x) x_off = take((size_t)a.rows * wpad * sizeof(T));
    if (pack_w) {
      wg_off = take((size_t)a.hidden * wpad * sizeof(T));
      wu_off = take((size_t)a.hidden * wpad * sizeof(T));
    }
    const int64_t rows = std::max<int64_t>(a.rows, 1);
    big_dual = big_tiles(2 * a.hidden, rows);
    if (!backward) return;
    big_dx = big_tiles(a.width, rows);
    wt_off = take((size_t)a.width * 2 * hpad * sizeof(T));
    dgu_off = take((size_t)a.rows * 2 * hpad * sizeof(T));
    bias_parts = 2 * ceil_div(rows, (int64_t)(big_dual ? 256 : 128));
    dbias_off = take((size_t)bias_parts * 2 * a.hidden * sizeof(float));
    // split the reduction over the rows until the tiles fill the device; each
    // split's sums cost a write and a read of the gradients in fp32
    constexpr int64_t KS = kStageBytes / sizeof(T);
    const int64_t stages = ceil_div(rows, KS);
    auto split_to = [&](int64_t side) {
      const int64_t tiles = ceil_div(2 * hpad, side) * ceil_div(a.width, side);
      return std::max<int64_t>(1, std::min(ceil_div(kSplitTarget, tiles),
                                           ceil_div(stages, (int64_t)16)));
    };
    big_dw = 2 * hpad * a.width >= (int64_t)16 * 256 * 256 && stages >= 64;
    splits = split_to(big_dw ? 256 : 128);
    const int64_t per = ceil_div(stages, splits);
    splits = ceil_div(stages, per);
    k_split = per * KS;
    if (splits > 1) part_off = take((size_t)splits * 2 * a.hidden * a.width * sizeof(float));
  }
};

template <class T>
void pack_rows(const void* src, int64_t ld, int64_t rows, int64_t cols, int64_t pad, T* dst,
               hipStream_t st) {
  const int64_t items = rows * (pad / Vec16<T>::N);
  k_pack_rows<T><<<(unsigned)std::min<int64_t>(ceil_div(items, (int64_t)256), 8192), 256, 0, st>>>(
      static_cast<const T*>(src), ld, rows, cols, pad, dst);
}

template <class T>
struct Inputs {
  const T *x, *wg, *wu;
  int64_t ldx, ldw;
};

// x and the weights as the product kernel loads them.
template <class T>
Inputs<T> load_inputs(const GatedArgs& a, const Plan<T>& pl, char* ws, hipStream_t st) {
  Inputs<T> in{static_cast<const T*>(a.x), static_cast<const T*>(a.w_gate),
               static_cast<const T*>(a.w_up), a.x_stride, a.w_gate_stride};
  if (pl.pack_x) {
    T* x = reinterpret_cast<T*>(ws + pl.x_off);
    pack_rows<T>(a.x, a.x_stride, a.rows, a.width, pl.wpad, x, st);
    in.x = x;
    in.ldx = pl.wpad;
  }
  if (pl.pack_w) {
    T *g = reinterpret_cast<T*>(ws + pl.wg_off), *u = reinterpret_cast<T*>(ws + pl.wu_off);
    pack_rows<T>(a.w_gate, a.w_gate_stride, a.hidden, a.width, pl.wpad, g, st);
    pack_rows<T>(a.w_up, a.w_up_stride, a.hidden, a.width, pl.wpad, u, st);
    in.wg = g;
    in.wu = u;
    in.ldw = pl.wpad;
  }
  return in;
}

template <class TL, class EPI>
void launch_gemm(const GemmShape& s, int64_t splits, const EPI& epi, hipStream_t st) {
  k_gemm<TL, EPI><<<dim3((unsigned)(s.tiles_p * s.tiles_q), (unsigned)splits), TL::THREADS, 0,
                    st>>>(s, epi);
  MGP_HIP_CHECK(hipGetLastError());
}

template <class TL, class EPI>
void launch_tiles(GemmShape s, int64_t splits, const EPI& epi, hipStream_t st) {
  s.tiles_p = ceil_div(s.p.n, (int64_t)(TL::DUAL ? TL::BP / 2 : TL::BP));
  s.tiles_q = ceil_div(s.q.n, (int64_t)TL::BQ);
  launch_gemm<TL>(s, splits, epi, st);
}

template <class T, bool TR, bool DUAL, class EPI>
void launch_product(bool big, const GemmShape& s, int64_t splits, const EPI& epi,
                    hipStream_t st) {
  if (big)
    launch_tiles<BigTile<T, TR, DUAL>>(s, splits, epi, st);
  else
    launch_tiles<SmallTile<T, TR, DUAL>>(s, splits, epi, st);
}

template <class T, class EPI>
void launch_dual(const GatedArgs& a, const Plan<T>& pl, const Inputs<T>& in, const EPI& epi,
                 hipStream_t st) {
  GemmShape s{};
  s.p = {reinterpret_cast<const char*>(in.wg), reinterpret_cast<const char*>(in.wu),
         in.ldw * (int64_t)sizeof(T), a.hidden};
  s.q = {reinterpret_cast<const char*>(in.x), nullptr, in.ldx * (int64_t)sizeof(T), a.rows};
  s.K = s.k_split = pl.wpad;
  launch_product<T, false, true>(pl.big_dual, s, 1, epi, st);
}

template <class F>
void dispatch_act(int act, F&& f) {
  switch (act) {
    case ACT_SILU: f(std::integral_constant<int, ACT_SILU>{}); break;
    case ACT_GELU: f(std::integral_constant<int, ACT_GELU>{}); break;
    case ACT_SIGMOID: f(std::integral_constant<int, ACT_SIGMOID>{}); break;
    default: f(std::integral_constant<int, ACT_RELU>{}); break;
  }
}

}  // namespace

size_t gated_bytes(const GatedArgs& a, bool backward) {
  size_t n = 0;
  dispatch_elem(a.type, [&](auto tag) { n = Plan<decltype(tag)>(a, backward).bytes; });
  return n;
}

void gated_forward(const GatedArgs& a, void* h, int64_t h_stride, void* ws, hipStream_t st) {
  if (a.rows == 0) return;
  dispatch_elem(a.type, [&](auto tag) {
    using T = decltype(tag);
    const Plan<T> pl(a, false);
    const Inputs<T> in = load_inputs<T>(a, pl, static_cast<char*>(ws), st);
    dispatch_act(a.activation, [&](auto act) {
      ForwardEpi<T, act.value> epi{static_cast<const T*>(a.b_gate), static_cast<const T*>(a.b_up),
                                   static_cast<T*>(h), h_stride, a.rows, a.hidden};
      launch_dual<T>(a, pl, in, epi, st);
    });
  });
}

void gated_backward(const GatedArgs& a, const void* dh, int64_t dh_stride, const GatedGrads& g,
                    void* ws_v, hipStream_t st) {
  char* ws = static_cast<char*>(ws_v);
  dispatch_elem(a.type, [&](auto tag) {
    using T = decltype(tag);
    T *dwg = static_cast<T*>(g.dw_gate), *dwu = static_cast<T*>(g.dw_up);
    T *dbg = static_cast<T*>(g.db_gate), *dbu = static_cast<T*>(g.db_up);
    if (a.rows == 0) {  // sums over no rows (fills by a kernel: a caller may capture them)
      const unsigned grid =
          (unsigned)std::min<int64_t>(ceil_div(2 * a.hidden * a.width, (int64_t)256), 4096);
      if (dwg || dwu)
        k_sum_parts<T><<<grid, 256, 0, st>>>(nullptr, 0, a.hidden * a.width, dwg, dwu);
      if (dbg || dbu) k_sum_parts<T><<<grid, 256, 0, st>>>(nullptr, 0, a.hidden, dbg, dbu);
      MGP_HIP_CHECK(hipGetLastError());
      return;
    }
    const Plan<T> pl(a, true);
    const Inputs<T> in = load_inputs<T>(a, pl, ws, st);
    T* dgu = reinterpret_cast<T*>(ws + pl.dgu_off);
    float* dbias = dbg || dbu ? reinterpret_cast<float*>(ws + pl.dbias_off) : nullptr;
    dispatch_act(a.activation, [&](auto act) {
      BackwardEpi<T, act.value> epi{static_cast<const T*>(a.b_gate), static_cast<const T*>(a.b_up),
                                    static_cast<const T*>(dh), dh_stride, a.rows, a.hidden,
                                    pl.hpad, dgu, dbias};
      launch_dual<T>(a, pl, in, epi, st);
    });
    if (dbias)
      k_sum_bias<T><<<(unsigned)ceil_div(2 * a.hidden, (int64_t)64), 1024, 0, st>>>(
          dbias, pl.bias_parts, a.hidden, dbg, dbu);
    const int64_t ldd = 2 * pl.hpad * (int64_t)sizeof(T);
    if (g.dx) {
      T* wt = reinterpret_cast<T*>(ws + pl.wt_off);
      k_transpose_weights<T><<<dim3((unsigned)ceil_div(pl.hpad, (int64_t)32),
                                    (unsigned)ceil_div(a.width, (int64_t)32), 2),
                               256, 0, st>>>(in.wg, in.wu, in.ldw, a.hidden, a.width,
                                             pl.hpad, wt);
      GemmShape s{};
      s.p = {reinterpret_cast<const char*>(wt), nullptr, ldd, a.width};
      s.q = {reinterpret_cast<const char*>(dgu), nullptr, ldd, a.rows};
      s.K = s.k_split = 2 * pl.hpad;
      launch_product<T, false, false>(
          pl.big_dx, s, 1, StoreEpi<T>{static_cast<T*>(g.dx), a.width, a.rows, a.width}, st);
    }
    if (dwg || dwu) {
      float* part = pl.splits > 1 ? reinterpret_cast<float*>(ws + pl.part_off) : nullptr;
      GemmShape s{};
      s.p = {reinterpret_cast<const char*>(in.x), nullptr, in.ldx * (int64_t)sizeof(T), pl.wpad};
      s.q = {reinterpret_cast<const char*>(dgu), nullptr, ldd, 2 * pl.hpad};
      s.K = a.rows;
      s.k_split = pl.k_split;
      launch_product<T, true, false>(pl.big_dw, s, pl.splits,
                                     WeightEpi<T>{dwg, dwu, part, a.hidden, pl.hpad, a.width}, st);
      if (part)
        k_sum_parts<T><<<(unsigned)std::min<int64_t>(
                             ceil_div(2 * a.hidden * a.width, (int64_t)256), 8192),
                         256, 0, st>>>(part, pl.splits, a.hidden * a.width, dwg, dwu);
    }
    MGP_HIP_CHECK(hipGetLastError());
  });
}

}  // namespace mgp
