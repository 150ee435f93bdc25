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
#include "layers.h"

#include <algorithm>
#include <type_traits>

namespace mgp {

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

#define MGP_LDS __attribute__((address_space(3)))

// ---------------------------------------------------------------- activation

// exp(x + tail) by v_exp_f32.  FAST (the 16-bit types): the exponent's rounding
// makes a relative error of 2^-24 |x|; fp32 takes it out to first order.  A
// library expf and a division made ~40 instructions of each sigmoid, and the
// epilogue of 65536 x 1024 -> 4096 a quarter of the kernel's time.
template <bool FAST>
__device__ __forceinline__ float exp_of(float x, float tail = 0.0f) {
  if constexpr (FAST) return __builtin_amdgcn_exp2f(kLog2e * x);
  constexpr float kLog2eLow = 1.92596299e-8f;  // log2(e) - kLog2e
  x = x < -126.0f ? -126.0f : x;  // beyond, 0 and infinity all the same; NaN stays
  x = x > 126.0f ? 126.0f : x;
  const float t = x * kLog2e;
  const float r = fmaf(x, kLog2e, -t) + fmaf(x, kLog2eLow, tail * kLog2e);
  return __builtin_amdgcn_exp2f(t) * fmaf(r, kLn2, 1.0f);
}

// 1 - Phi(x) over exp(-x^2 / 2) for x = sqrt(2) v, v >= 0: a polynomial in
// 1 / (1 + p v), p and the coefficients fitted by least squares reweighted
// towards the smallest largest relative error over 0 <= v <= 9.5: 5.2e-6 (six
// terms, the 16-bit types), 3.8e-8 (nine; 3.5e-7 as fp32 evaluates it).
template <bool FAST>
__device__ __forceinline__ float normal_tail(float v) {
  if constexpr (FAST) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.44f, v, 1.0f));
    float q = -0.0730530247092247f;
    q = fmaf(q, t, 0.17532674968242645f);
    q = fmaf(q, t, 0.020365050062537193f);
    q = fmaf(q, t, 0.13179342448711395f);
    q = fmaf(q, t, 0.12128471583127975f);
    return fmaf(q, t, 0.12428051233291626f) * t;
  } else {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, v, 1.0f));
    float q = -0.06471703946590424f;
    q = fmaf(q, t, 0.24254822731018066f);
    q = fmaf(q, t, -0.2556132376194f);
    q = fmaf(q, t, 0.2731975317001343f);
    q = fmaf(q, t, -0.04681563004851341f);
    q = fmaf(q, t, 0.10721813887357712f);
    q = fmaf(q, t, 0.07424121350049973f);
    q = fmaf(q, t, 0.08534596860408783f);
    return fmaf(q, t, 0.08459480851888657f) * t;
  }
}

// a = act(g) and its derivative
template <int ACT, bool FAST>
__device__ __forceinline__ void activate(float g, float& a, float& slope) {
  if constexpr (ACT == ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.0f + exp_of<FAST>(-g));
    a = g * s;
    slope = s * fmaf(g, 1.0f - s, 1.0f);
  } else if constexpr (ACT == ACT_SIGMOID) {
    a = __builtin_amdgcn_rcpf(1.0f + exp_of<FAST>(-g));
    slope = a * (1.0f - a);
  } else if constexpr (ACT == ACT_RELU) {
    a = g > 0.0f || g != g ? g : 0.0f;
    slope = g > 0.0f ? 1.0f : 0.0f;
  } else {
    // fp32: from |g| = 40 on e is 0, and a square that passes fp32 has no remainder
    const float c = FAST ? g : fminf(fabsf(g), 40.0f);
    const float g2 = c * c;
    const float e = exp_of<FAST>(-0.5f * g2, -0.5f * fmaf(c, c, -g2));
    const float tail = normal_tail<FAST>(fabsf(g) * 0.70710678118654752f) * e;  // 1 - Phi(|g|)
    const float cdf = g > 0.0f ? 1.0f - tail : tail;
    a = g * cdf;
    slope = fmaf(g * 0.39894228040143268f, e, cdf);
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

// ---------------------------------------------------------------- product core

// A 16-byte operand fragment: 8 narrow elements of 32 reduction steps spread
// over the lane groups, or 4 floats of 16 (k_gated_few alone).
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

constexpr int kOutOfRange = (int)0x80000000u;  // past num_records: the load gives zeros
constexpr int kNumRecords = 0x7fffffff;

// base: wave uniform; soff (too): not part of the range check, so an offset out
// of range stays it
__device__ __forceinline__ void load_lds(const char* base, int voff, int soff,
                                         char* __restrict__ dst) {
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, kNumRecords, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (MGP_LDS void*)dst, 16, voff, soff, 0, 0);
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
  int64_t p_apart, q_apart; // operands in parts: byte distance of one part from the next
};

// The products a sum is made of where operands come in parts: the parts of p and
// q of each, in order.  6: both in three parts; the smallest products first, so that
// the larger ones alone meet the rounding of the whole sum, and without those
// below 2^-25 of the largest.  2: q in two.
template <int PARTS>
struct PartOrder {
  static constexpr int p[1] = {0}, q[1] = {0};
};
template <>
struct PartOrder<2> {
  static constexpr int p[2] = {0, 0}, q[2] = {0, 1};
};
template <>
struct PartOrder<6> {
  static constexpr int p[6] = {2, 0, 1, 1, 0, 0}, q[6] = {0, 2, 1, 0, 1, 0};
};
// how many parts on the next product's operand lies, 4 bits a step, 2 for none
template <int PARTS>
constexpr uint32_t part_steps(bool of_p) {
  using O = PartOrder<PARTS>;
  uint32_t v = 0;
  for (int i = 0; i + 1 < PARTS; ++i)
    v |= (uint32_t)((of_p ? O::p[i + 1] - O::p[i] : O::q[i + 1] - O::q[i]) + 2) << (4 * i);
  return v;
}

// Tile of 16 TN WN columns (p rows) by 16 TM WM rows (q rows), one wave 16 TN
// by 16 TM of it.  NT: the p rows are dealt to LDS so that a lane's results are
// RUN = 4 TN (dual: 2 TN of each matrix) consecutive columns.  Both operands go
// through LDS by direct loads, double buffered, 128 bytes of reduction a stage.
// NT: 128-byte LDS rows, 16-byte chunk c of row r at c ^ (r / 2 % 8).  TN: LDS rows of the tile's width, one
// per reduction step, in the memory's order, their 32-byte granules at g ^ (r % 8)
// and read by the transposing LDS load.  Both keep the fragment reads off each
// other's banks.
template <class T, int TM_, int TN_, int WM_, int WN_, bool TR_, bool DUAL_, int PARTS_>
struct Tile {
  using Elem = T;
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_;
  static constexpr bool TR = TR_, DUAL = DUAL_;
  static constexpr int PARTS = PARTS_;  // products a sum is made of (PartOrder)
  static constexpr int W = WM * WN, THREADS = 64 * W;
  static constexpr int BQ = 16 * TM * WM, BP = 16 * TN * WN;
  static constexpr int T1 = DUAL ? TN / 2 : TN;  // 16-row tiles of one matrix a wave
  static constexpr int RUN = 4 * T1;
  static constexpr int E = sizeof(T);  // 2
  static constexpr int SB = 128;                   // reduction bytes of a row a stage
  static constexpr int KS = SB / E;                // reduction elements a stage
  static constexpr int LDS = (BP + BQ) * SB;  // one buffer
  static constexpr int IP = BP * SB / 1024 / W, IQ = BQ * SB / 1024 / W;
  static_assert(IP * W * 1024 == BP * SB && IQ * W * 1024 == BQ * SB, "");
};

// What a wave loads of a stage: I instructions, each 64 lanes x 16 bytes = 1 KB
// of LDS.  The instructions of a side lie a multiple of 8 LDS rows apart, so the
// lanes' offsets from each one's uniform start are the same; only which rows
// exist differs.
template <class TL>
struct Loader {
  static constexpr int I = TL::IP + TL::IQ;
  int voff[2];           // byte offset of the lane from an instruction's start
  int kpos[2];           // NT: its reduction element, TN: its reduction row within the stage
  bool exists[I];        // NT: its row is one of the matrix
  int soff[I];           // bytes from the side's base to the instruction's start
  const char* base[3];   // of p, of q, of p's second matrix
  int64_t step[2];       // bytes of a stage
  int64_t apart[2], back[2];  // bytes from one part to the next, and of a part's stages
  int64_t length, left;  // reduction elements of a part, and those still to load
  int part;

  // Whether instruction i of p loads the second matrix, for one wave: with 8
  // waves that is the wave's (its base is then base[0]), with 4 it is i's.
  static constexpr bool second(int i) { return TL::DUAL && TL::W == 4 && i % 2 == 1; }

  __device__ __forceinline__ void init(const GemmShape& s, int64_t n0, int64_t m0, int64_t k0,
                                       int64_t K) {
    init_side<true>(s.p, n0, k0);
    init_side<false>(s.q, m0, k0);
    step[0] = TL::TR ? TL::KS * s.p.ld_bytes : TL::SB;
    step[1] = TL::TR ? TL::KS * s.q.ld_bytes : TL::SB;
    length = left = K;
    if constexpr (TL::PARTS > 1) {
      apart[0] = s.p_apart;
      apart[1] = s.q_apart;
      back[0] = (K + TL::KS - 1) / TL::KS * step[0];
      back[1] = (K + TL::KS - 1) / TL::KS * step[1];
      using O = PartOrder<TL::PARTS>;
      base[0] += O::p[0] * apart[0];
      base[1] += O::q[0] * apart[1];
      if constexpr (second(1)) base[2] += O::p[0] * apart[0];
      part = 0;
    }
  }

  template <bool P>
  __device__ __forceinline__ void init_side(const Operand& o, int64_t row0, int64_t k0) {
    constexpr int N = P ? TL::IP : TL::IQ, S = P ? 0 : TL::IP;
    constexpr int B = P ? TL::BP : TL::BQ;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ld = (int)o.ld_bytes;
    if constexpr (!TL::TR) {
      static_assert(TL::W % 2 == 0, "");  // the swizzle is that of wave * 8 + lane / 8
      const int l8 = lane / 8;
      const int c = (lane & 7) ^ ((wave * 4 + lane / 16) & 7);
      // P: LDS row (wave w, matrix, tile t, row i) holds column
      // 16 T1 w + (i / 4) RUN + 4 t + i % 4
      const int lrow = P ? l8 / 4 * TL::RUN + l8 % 4 : l8;
      kpos[!P] = c * (16 / TL::E);
      voff[!P] = lrow * ld + c * 16;
      const char* from = o.base;
      if constexpr (P && TL::DUAL) {
        static_assert(TL::TN == 4 && (TL::W == 8 || TL::W == 4), "");
        base[2] = o.base2 + row0 * o.ld_bytes + k0 * TL::E;
        if (TL::W == 8 && wave >= 4) from = o.base2;
      }
      base[!P] = from + row0 * o.ld_bytes + k0 * TL::E;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r8 = (i * TL::W + wave) * 8;
        int r = r8;
        if constexpr (P) {
          const int t = r8 % (16 * TL::TN) / 16;
          r = r8 / (16 * TL::TN) * 16 * TL::T1 + r8 % 16 / 4 * TL::RUN + t % TL::T1 * 4;
        }
        exists[S + i] = row0 + r + lrow < o.n;
        soff[S + i] = r * ld;
      }
    } else {
      constexpr int RB = B * TL::E;  // bytes of an LDS row
      static_assert(TL::W * 1024 / RB % 8 == 0, "");
      const int byte = wave * 1024 + lane * 16, r = byte / RB;
      const int c = (byte % RB / 16) ^ (((r & 7) << 1) & (RB / 16 - 1));
      const bool in = row0 + c * (16 / TL::E) < o.n;
      kpos[!P] = r;
      voff[!P] = r * ld + c * 16;
      base[!P] = o.base + k0 * o.ld_bytes + row0 * TL::E;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        exists[S + i] = in;
        soff[S + i] = i * (TL::W * 1024 / RB) * ld;
      }
    }
  }

  // Loads the next stage into buf.
  __device__ __forceinline__ void load(char* __restrict__ buf) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l = (int)min(left, (int64_t)TL::KS);
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const bool p = i < TL::IP;
      const int j = p ? i : i - TL::IP;
      char* dst = buf + (p ? 0 : TL::BP * TL::SB) + (j * TL::W + wave) * 1024;
      const int at = TL::TR ? j * (TL::W * 1024 / ((p ? TL::BP : TL::BQ) * TL::E)) : 0;
      load_lds(base[p ? (second(i) ? 2 : 0) : 1],
               exists[i] && kpos[!p] < l - at ? voff[!p] : kOutOfRange, soff[i], dst);
    }
    left -= TL::KS;
    const bool turn = TL::PARTS > 1 && left <= 0 && part < TL::PARTS - 1;
#pragma unroll
    for (int b = 0; b < (second(1) ? 3 : 2); ++b) {
      base[b] += step[b & 1];
      if constexpr (TL::PARTS > 1) {
        if (turn) {
          const uint32_t steps = b & 1 ? part_steps<TL::PARTS>(false) : part_steps<TL::PARTS>(true);
          const int64_t on = (int)(steps >> (4 * part) & 15) - 2;
          base[b] += on * apart[b & 1] - back[b & 1];
        }
      }
    }
    if (turn) {
      left = length;
      ++part;
    }
  }
};

template <class TL, int B>
__device__ __forceinline__ Frag read_frag(const char* __restrict__ buf, int row, int ks) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  if constexpr (!TL::TR) {
    const int c = (ks * 4 + g) ^ (i >> 1);
    return {*reinterpret_cast<const f4*>(buf + (row + i) * TL::SB + c * 16)};
  } else {
    // lane group g takes reduction rows 4 g .. 4 g + 3 and the same + 16; the
    // transposing load gives lane i the four rows' elements of column i
    constexpr int RB = B * TL::E, M = RB / 32 - 1;
    const int r = ks * 32 + 4 * g + (i >> 2);
    // tiles differ in the granule alone: one address, and an exclusive or a
    // tile made where it is used (kept over the loop they would spill)
    int a = r * RB + ((r & 7 & M) * 32) + (i & 3) * 8;
    asm volatile("" : "+v"(a));
    a ^= (row >> 4) * 32;
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MGP_LDS s4*)(buf + a));
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((MGP_LDS s4*)(buf + a + 16 * RB));
    typedef short s8 __attribute__((ext_vector_type(8)));
    const s8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return {__builtin_bit_cast(f4, v)};
  }
}

// One stage: the loads of the next go out behind the first half's fragment
// reads (before them, the reads wait in the queue: 4 % of the product's time).
// The two buffers are distinct restrict arguments, so that the reads
// need not wait for the loads in flight; the closing barrier waits for those
// and for every wave's reads.
template <class TL>
__device__ __forceinline__ void stage(Loader<TL>& ld, const char* __restrict__ cur,
                                      char* __restrict__ nxt, bool more, int wm, int wn,
                                      f4 (&acc)[TL::TM][TL::TN]) {
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    Frag p[TL::TN], q[TL::TM];
#pragma unroll
    for (int t = 0; t < TL::TN; ++t) p[t] = read_frag<TL, TL::BP>(cur, (wn * TL::TN + t) * 16, ks);
#pragma unroll
    for (int t = 0; t < TL::TM; ++t)
      q[t] = read_frag<TL, TL::BQ>(cur + TL::BP * TL::SB, (wm * TL::TM + t) * 16, ks);
    if (ks == 0) {
      __builtin_amdgcn_sched_barrier(0);
      if (more) ld.load(nxt);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int m = 0; m < TL::TM; ++m)
#pragma unroll
      for (int n = 0; n < TL::TN; ++n) acc[m][n] = mma<typename TL::Elem>(p[n], q[m], acc[m][n]);
  }
  __syncthreads();
}

// Workgroups go round the 8 XCDs in turn: each XCD takes a stretch of tiles of
// its own, ordered in groups of 8 tile rows, so that what its L2 holds serves
// the tiles in flight on it.
__device__ __forceinline__ void tile_of(uint32_t id, uint32_t tiles_p, uint32_t tiles_q,
                                        uint32_t& tp, uint32_t& tq) {
  const uint32_t total = tiles_p * tiles_q, xcd = id & 7, per = total >> 3, rest = total & 7;
  id = xcd * per + min(xcd, rest) + (id >> 3);
  const uint32_t group = id / (8 * tiles_p), in = id - group * 8 * tiles_p;
  const uint32_t height = min(8u, tiles_q - group * 8);
  tq = group * 8 + in % height;
  tp = in / height;
}

// Whether a workgroup goes on to further tiles (of its XCD: the grid is a
// multiple of 8 then), the first stage of which it loads before the epilogue of
// the one before. For the big tile, alone on its CU, in the forward pass: bf16,
// 65536 x 1024 -> 4096 1005 -> 988 us, 30000 x 768 -> 2304 224 -> 216, 32768 x 256 ->
// 1024 55.4 -> 52.4, a single round of tiles (8192 x 1024 -> 1024) 33.5 -> 34.4; the
// backward pass' longer epilogue has no registers to spare (65536 rows: 1328 ->
// 1347), the gradients' products have many stages or one round (dx 916 -> 909).
template <class TL, class EPI>
constexpr bool stays = TL::W == 8 && EPI::FORWARD;

// acc[tm][tn][e] of lane l holds output row 16 (wm TM + tm) + l % 16 and column
// (NT, tn < T1) 16 T1 wn + RUN (l / 16) + 4 tn + e of either matrix, (TN)
// 16 (wn TN + tn) + 4 (l / 16) + e.
//
// Bound by the matrix cores' feeding: of 65536 x 1024 -> 4096 in bf16 the forward
// pass takes 1070 us (1030 TFLOP/s), g, u, dg and du 1480 (740: the epilogue reads and
// writes 1.6 GB), dx 920 (1195) and the weight gradients 975 (1130), all in turn, where
// a plain large product reaches 1420; the forward pass alone 990.  The big
// tile leaves room for one workgroup a CU, whose epilogue nothing covers; two of the
// small one cover each other, but read twice the operands from LDS and the L1 cache.
template <class TL, class EPI>
__global__ __launch_bounds__(TL::THREADS) void k_gemm(GemmShape s, EPI epi) {
  __shared__ __align__(1024) char b0[TL::LDS];
  __shared__ __align__(1024) char b1[TL::LDS];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % TL::WM, wn = wave / TL::WM;
  constexpr int CP = TL::DUAL ? TL::BP / 2 : TL::BP;  // output columns a tile
  constexpr bool STAYS = stays<TL, EPI>;
  const uint32_t tiles = (uint32_t)(s.tiles_p * s.tiles_q);
  const int64_t k0 = (int64_t)blockIdx.y * s.k_split;
  const int64_t K = min(s.k_split, s.K - k0);
  const int64_t all = (K + TL::KS - 1) / TL::KS * TL::PARTS;

  uint32_t tp, tq;
  tile_of(blockIdx.x, (uint32_t)s.tiles_p, (uint32_t)s.tiles_q, tp, tq);
  Loader<TL> ld;
  ld.init(s, (int64_t)tp * CP, (int64_t)tq * TL::BQ, k0, K);
  // pairs of stages, so that each has its own buffers at compile time; an odd
  // one goes first
  const bool odd = all % 2 == 1;
  ld.load(odd ? b1 : b0);
  __syncthreads();
  for (uint32_t id = blockIdx.x;;) {
    const int64_t n0 = (int64_t)tp * CP + wn * (CP / TL::WN);
    const int64_t m0 = (int64_t)tq * TL::BQ + wm * TL::TM * 16, part = (int64_t)tq * TL::WM + wm;
    const bool next = STAYS && id + gridDim.x < tiles;
    id += gridDim.x;
    f4 acc[TL::TM][TL::TN];
#pragma unroll
    for (int m = 0; m < TL::TM; ++m)
#pragma unroll
      for (int n = 0; n < TL::TN; ++n) acc[m][n] = f4{0.f, 0.f, 0.f, 0.f};
    const auto to_next = [&] {
      tile_of(id, (uint32_t)s.tiles_p, (uint32_t)s.tiles_q, tp, tq);
      ld.init(s, (int64_t)tp * CP, (int64_t)tq * TL::BQ, k0, K);
    };
    int64_t stages = all;
    if (odd) stage<TL>(ld, b1, b0, --stages > 0, wm, wn, acc);
    for (; stages > 0; stages -= 2) {
      stage<TL>(ld, b0, b1, true, wm, wn, acc);
      bool more = stages > 2;
      if (STAYS && !more && next && !odd) {
        to_next();
        more = true;
      }
      stage<TL>(ld, b1, b0, more, wm, wn, acc);
    }
    if (STAYS && next && odd) {
      to_next();
      ld.load(b1);
    }
    epi.template run<TL>(acc, m0, n0, part);
    if (!STAYS || !next) return;
    if (odd) __syncthreads();
  }
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

// Rows the product kernel can load directly: 16-byte aligned, whole 16-byte
// chunks, and a tile's rows within 31-bit offsets.
constexpr int64_t kRowBytes = (int64_t)1 << 23;  // 256 rows, the most of a tile, in 2^31 bytes
template <class T>
bool direct(const void* p, int64_t stride, int64_t cols) {
  return aligned16(p) && stride % Vec16<T>::N == 0 && cols % Vec16<T>::N == 0 &&
         stride * (int64_t)sizeof(T) < kRowBytes;
}

constexpr size_t kAlign = 256;
inline size_t align_up(size_t b) { return (b + kAlign - 1) / kAlign * kAlign; }

// The two tile sizes: 256 x 256, one workgroup of 8 waves a CU, and 128 x 128,
// two workgroups of 4 waves, for what would leave CUs idle otherwise.
template <class T, bool TR, bool DUAL, int PARTS>
using BigTile = Tile<T, 8, 4, 2, 4, TR, DUAL, PARTS>;
template <class T, bool TR, bool DUAL, int PARTS>
using SmallTile = Tile<T, 4, 4, 2, 2, TR, DUAL, PARTS>;
// How a product is cut: the tile, and into how many parts its reduction, whose
// sums are then written and read once each in fp32.  By the time as measured:
// whole rounds of the device (512 small tiles or 256 big ones at a time), each
// that of a tile's prologue and epilogue and of its stages (small, 4 / 7 / 16
// stages: 7.1 / 11 / 19 us a round; big: 13.8 / 19 / 34), and the parts' sums at
// 4.5 TB/s.  So 8192 rows x 1024 -> 1024 bf16 go by big tiles (34.4 us forward, 38.1
// by small ones), 12007 x 392 -> 1024 by small ones (33.1, 38.7); the weight
// gradient of 4096 x 1024 -> 4096 by small ones in one part (70 us; big ones in two
// 102, in four 143), that of 65536 rows by big ones in two.
struct Cut {
  bool big = false;
  int64_t splits = 1, per = 0;  // parts, and stages of each
};
inline Cut cut_product(int64_t p_rows, int64_t q_rows, int64_t stages, int64_t parts_a_stage,
                       bool may_big, int64_t max_splits, double outputs) {
  Cut best;
  double least = 0.0;
  for (int big = 0; big <= (may_big ? 1 : 0); ++big) {
    const int64_t side = big ? 256 : 128;
    const int64_t tiles = ceil_div(p_rows, side) * ceil_div(q_rows, side);
    for (int64_t want = 1; want <= std::min(max_splits, std::max<int64_t>(1, stages / 4)); ++want) {
      const int64_t per = ceil_div(stages, want), splits = ceil_div(stages, per);
      const double rounds = (double)ceil_div(tiles * splits, (int64_t)(big ? 256 : 512));
      const double work = (double)(per * parts_a_stage);
      const double us = rounds * (big ? 7.1 + 1.7 * work : 3.3 + 1.0 * work) +
                        (splits > 1 ? 5.0 + (double)splits * outputs * 8.0 / 4.5e6 : 0.0);
      if ((big == 0 && want == 1) || us < least) {
        least = us;
        best.big = big != 0;
        best.splits = splits;
        best.per = per;
      }
    }
  }
  return best;
}
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

template <class TL, class EPI>
void launch_tiles(GemmShape s, int64_t splits, const EPI& epi, hipStream_t st) {
  s.tiles_p = ceil_div(s.p.n, (int64_t)(TL::DUAL ? TL::BP / 2 : TL::BP));
  s.tiles_q = ceil_div(s.q.n, (int64_t)TL::BQ);
  int64_t blocks = s.tiles_p * s.tiles_q;
  if (stays<TL, EPI>) blocks = std::min(blocks, (int64_t)256);  // (never split)
  k_gemm<TL, EPI><<<dim3((unsigned)blocks, (unsigned)splits), TL::THREADS, 0, st>>>(s, epi);
  MGP_HIP_CHECK(hipGetLastError());
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

template <class E>
Operand operand(const E* p, int64_t ld, int64_t n, const E* p2 = nullptr) {
  return {reinterpret_cast<const char*>(p), reinterpret_cast<const char*>(p2),
          ld * (int64_t)sizeof(E), n};
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

template <class F>
void dispatch_act(int act, F&& f) {
  switch (act) {
    case ACT_SILU: f(std::integral_constant<int, ACT_SILU>{}); break;
    case ACT_GELU: f(std::integral_constant<int, ACT_GELU>{}); break;
    case ACT_SIGMOID: f(std::integral_constant<int, ACT_SIGMOID>{}); break;
    default: f(std::integral_constant<int, ACT_RELU>{}); break;
  }
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
