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
// Matrix-core bound, at up to twice the 16-bit rate; rows are quantised by one pass
// of their own before the product.  65536 x 1024 -> 2 x 4096 bf16: codes 40 us, product 670
// (1640 TOPS; of it matrix instructions alone 403, waiting for loads 120, a tile's end 150).
// Few rows (k_int8_few) are bound by reading the weights once, at half the bytes of
// 16-bit ones, and by latency: up to 16 rows, as long as that is the shorter way (way_of),
// each workgroup quantises what it needs itself, in the one launch (1 x 512 -> 2 x 2048
// bf16 4.0 us a call in a row of them, 4.7 as a kernel trace has it).
#include <algorithm>
#include <type_traits>

#include "activation.h"
#include "product.h"
#include "sym_common.h"

namespace mgp {

namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef int i16 __attribute__((ext_vector_type(16)));

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

// ---------------------------------------------------------------- tiles

// Tile of 32 TN WN columns (weight rows) by 32 TM WM rows, one wave 32 TN by 32 TM of it
// in 32 x 32 x 32 matrix instructions.  Both operands go through LDS by direct loads, SB
// columns a stage, two buffers; 16-byte chunk c of row r at c ^ (r / (256 / SB) %
// CHUNKS).  The weight rows are dealt to LDS so that a lane's results are 16 consecutive
// columns of 32 (of each projection: gated, half of a wave's rows are up's).
template <int TM_, int TN_, int WM_, int WN_, int SB_, bool GATED_>
struct ByteTile {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, SB = SB_;
  static constexpr bool GATED = GATED_;
  static constexpr int W = WM * WN, THREADS = 64 * W;
  static constexpr int BQ = 32 * TM * WM, BP = 32 * TN * WN;
  static constexpr int T1 = GATED ? TN / 2 : TN;
  static constexpr int CP = GATED ? BP / 2 : BP;  // output columns of a tile
  static constexpr int LDS = (BP + BQ) * SB, CHUNKS = SB / 16;
  static constexpr int ROWS = 1024 / SB;                        // of LDS, a load
  static constexpr int IP = BP / ROWS / W, IQ = BQ / ROWS / W;  // loads a stage
  static constexpr int FRAGS = TM + TN, STEPS = SB / 32;
  // the loads' rows of one projection: a wave's own, or every second load's
  static constexpr bool BY_WAVE = W * ROWS == 64;
  static_assert(TN == 2 && (BY_WAVE || W * ROWS == 32) && (STEPS == 2 || STEPS == 4), "");
  static __device__ __forceinline__ int chunk(int r, int c) {
    return (c ^ (r / (256 / SB))) & (CHUNKS - 1);
  }
};

struct ByteShape {
  const int8_t *wg, *wu, *x;
  int ldw, ldx;
  int64_t hidden, rows;
  int K;
  uint32_t tiles_p, tiles_q;
};

// What a wave loads of a stage: 64 lanes x 16 bytes an instruction.
template <class TL>
struct ByteLoader {
  int vp, vq;         // byte offset of a lane from an instruction's first row
  int kpos;           // its column within the stage
  int soff[TL::IP + TL::IQ];
  bool exists[TL::IP + TL::IQ];
  const char *bp[2], *bq;
  int left;           // columns still to load

  __device__ __forceinline__ void init(const ByteShape& s, uint32_t tp, uint32_t tq) {
    const int lane = threadIdx.x & 63, lr = lane / TL::CHUNKS;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = TL::chunk(wave * TL::ROWS + lr, lane & (TL::CHUNKS - 1));
    const int64_t n0 = (int64_t)tp * TL::CP, m0 = (int64_t)tq * TL::BQ;
    kpos = c * 16;
    const int prow = lr / 4 % 2 * 16 + lr / 8 * 4 + lr % 4;
    vp = prow * s.ldw + kpos;
    vq = lr * s.ldx + kpos;
    bp[0] = reinterpret_cast<const char*>(s.wg) + n0 * s.ldw;
    bp[1] = TL::GATED ? reinterpret_cast<const char*>(s.wu) + n0 * s.ldw : bp[0];
    if (TL::GATED && TL::BY_WAVE && wave >= TL::W / 2) bp[0] = bp[1];
    bq = reinterpret_cast<const char*>(s.x) + m0 * s.ldx;
#pragma unroll
    for (int i = 0; i < TL::IP; ++i) {
      const int first = (i * TL::W + wave) * TL::ROWS, in = first % (32 * TL::TN);
      const int r = first / (32 * TL::TN) * 32 * TL::T1 + in / 32 % TL::T1 * 32 + in % 32 / 8 * 4;
      soff[i] = r * s.ldw;
      exists[i] = n0 + r + prow < s.hidden;
    }
#pragma unroll
    for (int i = 0; i < TL::IQ; ++i) {
      const int r = (i * TL::W + wave) * TL::ROWS;
      soff[TL::IP + i] = r * s.ldx;
      exists[TL::IP + i] = m0 + r + lr < s.rows;
    }
    left = s.K;
  }

  // Loads the next stage into buf.
  __device__ __forceinline__ void load(char* __restrict__ buf) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool in = kpos < left;
#pragma unroll
    for (int i = 0; i < TL::IP; ++i)
      load_lds(bp[TL::GATED && !TL::BY_WAVE ? i % 2 : 0], in && exists[i] ? vp : kOutOfRange, soff[i],
               buf + (i * TL::W + wave) * 1024);
#pragma unroll
    for (int i = 0; i < TL::IQ; ++i)
      load_lds(bq, in && exists[TL::IP + i] ? vq : kOutOfRange, soff[TL::IP + i],
               buf + TL::BP * TL::SB + (i * TL::W + wave) * 1024);
    left -= TL::SB;
    bp[0] += TL::SB;
    bp[1] += TL::SB;
    bq += TL::SB;
  }
};

// The fragments of 32 columns: those of the wave's weight rows, then of its rows of x.
template <class TL>
struct ByteFrags {
  Frag f[TL::FRAGS];
  __device__ __forceinline__ void read(const char* __restrict__ buf, int step, int wm, int wn) {
    const int lane = threadIdx.x & 63, i = lane & 31;
    const int at = i * TL::SB + TL::chunk(i, step * 2 + (lane >> 5)) * 16;
#pragma unroll
    for (int t = 0; t < TL::TN; ++t)
      f[t].v = *reinterpret_cast<const f4*>(buf + (wn * TL::TN + t) * 32 * TL::SB + at);
#pragma unroll
    for (int t = 0; t < TL::TM; ++t)
      f[TL::TN + t].v = *reinterpret_cast<const f4*>(buf + (TL::BP + (wm * TL::TM + t) * 32) * TL::SB + at);
    __builtin_amdgcn_sched_barrier(0);
  }
  __device__ __forceinline__ void multiply(i16 (&acc)[TL::TM][TL::TN]) const {
#pragma unroll
    for (int m = 0; m < TL::TM; ++m)
#pragma unroll
      for (int n = 0; n < TL::TN; ++n)
        acc[m][n] = __builtin_amdgcn_mfma_i32_32x32x32_i8(
            __builtin_bit_cast(i4, f[n].v), __builtin_bit_cast(i4, f[TL::TN + m].v), acc[m][n], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  }
};

// The barrier of a stage: a wave's own loads into LDS and its reads from it have
// ended, then every wave's.  The waits stand here as the compiler's are not to be
// relied on (it adds one for such loads where it takes buffers to alias).  A counter
// of loads counts stores too: behind a tile's end, whose stores were issued after
// these loads had ended, only the reads are waited for (drained), and the stores have
// until the next barrier.
__device__ __forceinline__ void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void arrive(bool drained) {
  if (!drained) loads_done();
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// One stage of the running sum.  even holds the fragments of its first 32 columns.  The
// barrier stands before the last products: behind it, under them, go the loads of
// the stage after the next, into the buffer that every wave has read by then, and
// the reads of the next stage's first fragments.
template <class TL, class Load>
__device__ __forceinline__ void byte_stage(const char* __restrict__ cur,
                                           const char* __restrict__ nxt, bool real, bool more,
                                           bool next_real, bool drained, int wm, int wn, ByteFrags<TL>& even,
                                           i16 (&acc)[TL::TM][TL::TN], Load&& load) {
  ByteFrags<TL> odd;
  if (real) {
    odd.read(cur, 1, wm, wn);
    even.multiply(acc);
    if constexpr (TL::STEPS == 4) {
      even.read(cur, 2, wm, wn);
      odd.multiply(acc);
      odd.read(cur, 3, wm, wn);
      even.multiply(acc);
    }
  }
  if (more) {
    arrive(drained);
    if (next_real) even.read(nxt, 0, wm, wn);
    load();
    __builtin_amdgcn_sched_barrier(0);
  }
  if (real) odd.multiply(acc);
}

// The results of a wave: acc[m][n][e] of lane l is row 32 m + l % 32 and, of matrix
// n / T1, column 32 (n % T1) + 16 (l / 32) + e.  A row's 32 columns meet in LDS (out,
// the wave's own), so that they are written together: stored from where they are,
// in halves of 16 bytes a row, they took longer than the products.
template <class T, class TL>
__device__ __forceinline__ void byte_end(const EndArgs& a, const i16 (&acc)[TL::TM][TL::TN],
                                         int64_t m0, int64_t n0, char* out) {
  constexpr int N = 8, ROW = 32 * sizeof(T), CHUNKS = ROW / 16, V = 16 / sizeof(T);
  const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
  float sx[TL::TM];
#pragma unroll
  for (int m = 0; m < TL::TM; ++m) sx[m] = a.sx[min(m0 + i + 32 * m, a.rows - 1)];
#pragma unroll
  for (int t = 0; t < TL::T1; ++t) {
    const int64_t f = n0 + 32 * t;
    if (f >= a.hidden) {
      if (t == 0) loads_done();
      break;
    }
    T o[TL::TM][16];
#pragma unroll
    for (int q = 0; q < 16; q += N) {
      const int64_t c = f + 16 * h + q, left = a.hidden - c;
      float sg[N], bg[N], su[N], bu[N];
      zeros<N>(sg);
      zeros<N>(bg);
      zeros<N>(su);
      zeros<N>(bu);
      if (left > 0) {
        load_run<N>(a.sg + c, left, sg);
        if (a.bg) load_run<N>(static_cast<const T*>(a.bg) + c, left, bg);
        if constexpr (TL::GATED) {
          load_run<N>(a.su + c, left, su);
          if (a.bu) load_run<N>(static_cast<const T*>(a.bu) + c, left, bu);
        }
      }
#pragma unroll
      for (int m = 0; m < TL::TM; ++m) {
        int g[N], u[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
          g[k] = acc[m][t][q + k];
          u[k] = acc[m][TL::TN - 1][q + k];
        }
        float v[N];
        finish<T, N, TL::GATED>(g, u, sx[m], sg, su, bg, bu, a.act, v);
#pragma unroll
        for (int k = 0; k < N; ++k) o[m][q + k] = (T)v[k];
      }
    }
    if (t == 0) loads_done();  // before the first store
#pragma unroll
    for (int m = 0; m < TL::TM; ++m) {
      // 16-byte chunk c of row r at c ^ (r / (256 / ROW) % CHUNKS): off each other's banks
      auto at = [&](int r, int c) __attribute__((always_inline)) {
        return reinterpret_cast<f4*>(out + r * ROW + ((c ^ (r / (256 / ROW))) % CHUNKS) * 16);
      };
#pragma unroll
      for (int c = 0; c < CHUNKS / 2; ++c) {
        f4 x;
        __builtin_memcpy(&x, &o[m][c * V], 16);
        *at(i, h * (CHUNKS / 2) + c) = x;
      }
      wave_lds_sync();
      const int64_t c0 = f + lane % CHUNKS * V, left = a.hidden - c0;
#pragma unroll
      for (int r = lane / CHUNKS; r < 32; r += 64 / CHUNKS) {
        const f4 x = *at(r, lane % CHUNKS);
        const int64_t row = m0 + 32 * m + r;
        T* to = static_cast<T*>(a.y) + row * a.ldy + c0;
        if (row < a.rows && left > 0) {
          if (left >= V) {
            __builtin_memcpy(to, &x, 16);
          } else {
            T e[V];
            __builtin_memcpy(e, &x, 16);
#pragma unroll
            for (int k = 0; k < V; ++k)
              if (k < left) to[k] = e[k];
          }
        }
      }
      wave_lds_sync();
    }
  }
}

// Workgroups go on to further tiles of their XCD; the loads of the next tile's first
// stages are out before the end of the one before.  An odd number of stages is
// made even by an empty one, so that each has its buffer at compile time.
template <class T, class TL>
__global__ __launch_bounds__(TL::THREADS)
    __attribute__((amdgpu_waves_per_eu(2, 2))) void k_int8_tiles(ByteShape s, EndArgs a) {
  __shared__ __align__(1024) char b0[TL::LDS];
  __shared__ __align__(1024) char b1[TL::LDS];
  __shared__ __align__(1024) char out[TL::W][32 * 32 * sizeof(T)];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % TL::WM, wn = wave / TL::WM;
  const uint32_t tiles = s.tiles_p * s.tiles_q;
  const int stages = (s.K + TL::SB - 1) / TL::SB, pairs = (stages + 1) / 2;

  uint32_t tp, tq;
  tile_of(blockIdx.x, s.tiles_p, s.tiles_q, tp, tq);
  ByteLoader<TL> ld;
  ld.init(s, tp, tq);
  ld.load(b0);
  if (stages > 1) ld.load(b1);
  arrive(false);
  ByteFrags<TL> even;
  even.read(b0, 0, wm, wn);
  for (uint32_t id = blockIdx.x;;) {
    const bool drained = id != blockIdx.x;  // the end of a tile has waited for the loads
    const int64_t n0 = (int64_t)tp * TL::CP + wn * 32 * TL::T1;
    const int64_t m0 = (int64_t)tq * TL::BQ + wm * 32 * TL::TM;
    id += gridDim.x;
    const bool next = id < tiles;
    i16 acc[TL::TM][TL::TN];
#pragma unroll
    for (int m = 0; m < TL::TM; ++m)
#pragma unroll
      for (int n = 0; n < TL::TN; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[m][n][e] = 0;
    for (int p = 0; p < pairs; ++p) {
      const bool last = p + 1 == pairs, both = 2 * p + 1 < stages;
      byte_stage<TL>(b0, b1, true, both || next, both, drained && p == 0, wm, wn, even, acc, [&] {
        if (!last) {
          ld.load(b0);
        } else if (next) {
          tile_of(id, s.tiles_p, s.tiles_q, tp, tq);
          ld.init(s, tp, tq);
          ld.load(b0);
        }
      });
      byte_stage<TL>(b1, b0, both, !last || next, !last, false, wm, wn, even, acc, [&] {
        if (2 * p + 3 < stages || (last && next && stages > 1)) ld.load(b1);
      });
    }
    byte_end<T, TL>(a, acc, m0, n0, out[wave]);
    if (!next) return;
    even.read(b0, 0, wm, wn);
  }
}

// ---------------------------------------------------------------- few rows

struct FewArgs {
  EndArgs end;
  const void* x;  // FUSED: rows of elements, otherwise of codes
  int64_t ldx;
  const int8_t *wg, *wu;
  int64_t ldw, width;
};

__device__ __forceinline__ i4 mma_i8(const Frag& a, const Frag& b, i4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4, a.v),
                                               __builtin_bit_cast(i4, b.v), c, 0, 0, 0);
}

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

// Up to 16 rows in the one launch where it costs each round of 256 workgroups less to
// quantise them than a second launch takes: 1 x 512 -> 2 x 2048 bf16 4.0 us (with codes
// of their own 6.0), 16 x 512 5.7 (6.4), but 16 x 1024 8.5 (6.7), 16 x 4096 27.6 (11.8), 4 x
// 2048 8.7 (7.6), 1 x 2048 6.9 (7.2), 1 x 4096 13.6 (10.3); to 2 x 16384, 1 x 512 7.6 (8.8),
// 16 x 256 9.0 (8.1).  More rows by few up to 512 workgroups: 128 x 1024 -> 4096 10.1 us
// (tiles 11.3), 192 x 1024 -> 4096 12.6 (11.5), 500 x 64 -> 512 6.1 (7.9).
inline Way way_of(const Int8Args& a) {
  if (a.rows <= 16 && (a.rows + 4) * a.width * ceil_div(a.hidden, (int64_t)4096) <= 12288)
    return FUSED_ROWS;
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
  auto tiles = [&](auto tile, int64_t at_once) {
    using TL = decltype(tile);
    const ByteShape s{a.w_gate,
                      a.w_up,
                      codes,
                      (int)a.w_stride,
                      (int)ldx,
                      a.hidden,
                      a.rows,
                      (int)ldx,
                      (uint32_t)ceil_div(a.hidden, (int64_t)TL::CP),
                      (uint32_t)ceil_div(a.rows, (int64_t)TL::BQ)};
    const int64_t all = (int64_t)s.tiles_p * s.tiles_q;
    k_int8_tiles<T, TL><<<(unsigned)std::min(all, at_once), TL::THREADS, 0, st>>>(s, end);
  };
  // 256 x 256 by 8 waves where cut_product finds rounds of them the shorter (its stages
  // are of as many bytes and instructions here); below 256 tiles of 128 x 128, half that
  // many rows a tile, which leave no CU idle.  Device time, 64 x 128 / 128 x 128 / 256 x
  // 256: 500 x 1024 -> 4096 10.9 / 13.3 us, 1500 x 256 -> 1024 7.2 / 9.1, 1500 x 1024 ->
  // 4096 21.5 / 18.5, 4000 x 1024 -> 2 x 4096 47 (big) / 56.7
  const int64_t cols = (GATED ? 2 : 1) * a.hidden;
  if (cut_product(cols, a.rows, ceil_div(ldx, (int64_t)128), 1, true, 1, 0.0).big)
    tiles(ByteTile<4, 2, 2, 4, 128, GATED>{}, 256);
  else if (ceil_div(cols, (int64_t)128) * ceil_div(a.rows, (int64_t)128) > 256)
    tiles(ByteTile<2, 2, 2, 2, 128, GATED>{}, 512);
  else
    tiles(ByteTile<1, 2, 2, 2, 128, GATED>{}, 512);
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
