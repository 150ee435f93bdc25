// The tiled matrix product of the layers: operands through LDS by direct loads, a
// tile's sums in registers, an epilogue of the caller's.
#pragma once

#include <algorithm>
#include <type_traits>

#include "layers.h"

namespace mgp {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

#define MGP_LDS __attribute__((address_space(3)))

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

// ---------------------------------------------------------------- host side

// Rows the product kernel can load directly: 16-byte aligned, whole 16-byte
// chunks, and a tile's rows within 31-bit offsets.
constexpr int64_t kRowBytes = (int64_t)1 << 23;  // 256 rows, the most of a tile, in 2^31 bytes
template <class T>
inline bool direct(const void* p, int64_t stride, int64_t cols) {
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
template <class TL, class EPI>
void launch_tiles(GemmShape s, int64_t splits, const EPI& epi, hipStream_t st) {
  s.tiles_p = ceil_div(s.p.n, (int64_t)(TL::DUAL ? TL::BP / 2 : TL::BP));
  s.tiles_q = ceil_div(s.q.n, (int64_t)TL::BQ);
  int64_t blocks = s.tiles_p * s.tiles_q;
  if (stays<TL, EPI>) blocks = std::min(blocks, (int64_t)256);  // (never split)
  k_gemm<TL, EPI><<<dim3((unsigned)blocks, (unsigned)splits), TL::THREADS, 0, st>>>(s, epi);
  MGP_HIP_CHECK(hipGetLastError());
}

template <class E>
Operand operand(const E* p, int64_t ld, int64_t n, const E* p2 = nullptr) {
  return {reinterpret_cast<const char*>(p), reinterpret_cast<const char*>(p2),
          ld * (int64_t)sizeof(E), n};
}

}  // namespace mgp
