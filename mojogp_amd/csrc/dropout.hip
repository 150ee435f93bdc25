// Dropout whose mask is a function of (seed, element number): the backward
// pass draws it again, nothing is stored.
//
// Element e of the array takes draw offset + e of the stream `seed`: draw q is
// 16-bit half q % 2 of word (q % 8) / 2 of the Philox4x32-10 block of counter
// (q / 8, 0) and key seed (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011).  Sixteen bits a draw make one block
// serve eight elements: with 32 bits the ten rounds (two 32 x 32 -> 64 bit
// products each) would take longer than the array's transfer.  HBM bound: bf16,
// 250000 x 1024 with a residual 300 us (5.1 TB/s), without 193 (5.3).
#include "layers.h"

#include <algorithm>
#include <type_traits>

namespace mgp {

namespace {

struct Draws {
  uint32_t w[4];
  __device__ __forceinline__ uint32_t half(int i) const {
    return (w[i >> 1] >> (16 * (i & 1))) & 0xffffu;
  }
};

__device__ __forceinline__ Draws philox(uint64_t block, uint64_t seed) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = 0, c3 = 0;
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    const uint32_t n0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0, n2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

__device__ __forceinline__ float kept(float x, uint32_t draw, uint32_t cut, float scale) {
  // a dropped element is 0 whatever it held, infinities and NaN included
  return draw >= cut ? x * scale : 0.0f;
}

// Eight elements at any alignment (the memory path takes it).
template <class T>
__device__ __forceinline__ void load8(const T* p, float* v) {
  T a[8];
  __builtin_memcpy(a, p, sizeof(a));
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = (float)a[k];
}

// A thread takes the up to eight elements of one block of draws, loaded before
// the rounds so that those run while the loads do.  FLAT: contiguous arrays;
// otherwise rows of their own strides, eight elements of one row at a time
// where the block lies in one.
template <class T, bool FLAT, bool RES>
__global__ __launch_bounds__(256) void k_dropout(const T* __restrict__ x, int64_t ldx,
                                                 const T* __restrict__ residual, int64_t ldr,
                                                 int64_t total, int64_t width, uint32_t cut,
                                                 float scale, uint64_t seed, uint64_t offset,
                                                 T* __restrict__ y, int64_t ldy) {
  const int head = (int)(offset & 7);  // draws of the first block before element 0
  const int64_t blocks = (total + head + 7) / 8;
  for (int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x; b < blocks;
       b += (int64_t)gridDim.x * 256) {
    const int64_t first = b * 8 - head;
    int64_t row = 0, col = first > 0 ? first : 0;
    if constexpr (!FLAT) {
      row = col / width;
      col -= row * width;
    }
    const bool whole = first >= 0 && first + 8 <= total && (FLAT || col + 8 <= width);
    const T *px = x + row * ldx + col, *pr = RES ? residual + row * ldr + col : nullptr;
    float v[8], r[8];
    if (whole) {
      load8(px, v);
      if constexpr (RES) load8(pr, r);
    }
    const Draws dr = philox((offset >> 3) + (uint64_t)b, seed);
    if (whole) {
      T a[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float f = kept(v[k], dr.half(k), cut, scale);
        if constexpr (RES) f += r[k];
        a[k] = (T)f;
      }
      __builtin_memcpy(y + row * ldy + col, a, sizeof(a));
      continue;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (first + k < 0 || first + k >= total) continue;
      float f = kept((float)x[row * ldx + col], dr.half(k), cut, scale);
      if constexpr (RES) f += (float)residual[row * ldr + col];
      y[row * ldy + col] = (T)f;
      if (++col == width && !FLAT) {
        col = 0;
        ++row;
      }
    }
  }
}

}  // namespace

void dropout(const DropoutArgs& a, void* y, int64_t y_stride, hipStream_t st) {
  const int64_t total = a.rows * a.width;
  if (total == 0) return;
  const float scale = 65536.0f / (float)(65536 - a.cut);
  dispatch_elem(a.type, [&](auto tag) {
    using T = decltype(tag);
    auto flat = [&](int64_t stride) { return stride == a.width || a.rows == 1; };
    const T *x = static_cast<const T*>(a.x), *r = static_cast<const T*>(a.residual);
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(total / 8 + 2, (int64_t)256), 8192);
    auto go = [&](auto fl, auto res) {
      k_dropout<T, fl.value, res.value><<<grid, 256, 0, st>>>(
          x, a.x_stride, r, a.residual_stride, total, a.width, a.cut, scale, a.seed, a.offset,
          static_cast<T*>(y), y_stride);
    };
    const bool all = flat(a.x_stride) && flat(y_stride) && (!r || flat(a.residual_stride));
    if (all && r) go(std::true_type{}, std::true_type{});
    if (all && !r) go(std::true_type{}, std::false_type{});
    if (!all && r) go(std::false_type{}, std::true_type{});
    if (!all && !r) go(std::false_type{}, std::false_type{});
    MGP_HIP_CHECK(hipGetLastError());
  });
}

}  // namespace mgp
