// Dropout whose mask is a function of (seed, element number): the backward
// pass draws it again, nothing is stored.
//
// Element e of the array takes draw offset + e of the stream `seed`: draw q is
// 16-bit half q % 2 of word (q % 8) / 2 of the Philox4x32-10 block of counter
// (q / 8, 0) and key seed (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011).  Sixteen bits a draw make one block
// serve eight elements: with 32 bits the ten rounds (two 32 x 32 -> 64 bit
// products each) would take longer than the array's transfer.
#include "layers.h"

#include <algorithm>

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

// Contiguous, 16-byte aligned arrays with offset % 8 == 0: a thread takes the
// eight elements of a block.
template <class T, bool RES>
__global__ __launch_bounds__(256) void k_dropout(const T* __restrict__ x,
                                                 const T* __restrict__ residual, int64_t total,
                                                 uint32_t cut, float scale, uint64_t seed,
                                                 uint64_t block0, T* __restrict__ y) {
  constexpr int N = Vec16<T>::N, NV = 8 / N;
  const int64_t blocks = (total + 7) / 8;
  for (int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x; b < blocks;
       b += (int64_t)gridDim.x * 256) {
    const Draws dr = philox(block0 + (uint64_t)b, seed);
    const int64_t e0 = b * 8;
    if (e0 + 8 <= total) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        Vec16<T> a = *reinterpret_cast<const Vec16<T>*>(x + e0 + v * N), r;
        if constexpr (RES) r = *reinterpret_cast<const Vec16<T>*>(residual + e0 + v * N);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          float f = kept((float)a.v[k], dr.half(v * N + k), cut, scale);
          if constexpr (RES) f += (float)r.v[k];
          a.v[k] = (T)f;
        }
        *reinterpret_cast<Vec16<T>*>(y + e0 + v * N) = a;
      }
    } else {
      for (int k = 0; e0 + k < total; ++k) {
        float f = kept((float)x[e0 + k], dr.half(k), cut, scale);
        if constexpr (RES) f += (float)residual[e0 + k];
        y[e0 + k] = (T)f;
      }
    }
  }
}

// Any strides, alignment and offset: a thread takes the elements of one block,
// an element at a time.
template <class T>
__global__ __launch_bounds__(256) void k_dropout_any(const T* __restrict__ x, int64_t ldx,
                                                     const T* __restrict__ residual, int64_t ldr,
                                                     int64_t total, int64_t width, uint32_t cut,
                                                     float scale, uint64_t seed, uint64_t offset,
                                                     T* __restrict__ y, int64_t ldy) {
  const int head = (int)(offset & 7);  // draws of the first block before element 0
  const int64_t blocks = (total + head + 7) / 8;
  for (int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x; b < blocks;
       b += (int64_t)gridDim.x * 256) {
    const Draws dr = philox((offset >> 3) + (uint64_t)b, seed);
    const int64_t first = b * 8 - head;
    int64_t row = (first > 0 ? first : 0) / width, col = (first > 0 ? first : 0) - row * width;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t e = first + k;
      if (e < 0 || e >= total) continue;
      float f = kept((float)x[row * ldx + col], dr.half(k), cut, scale);
      if (residual) f += (float)residual[row * ldr + col];
      y[row * ldy + col] = (T)f;
      if (++col == width) {
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
    auto flat = [&](const void* p, int64_t stride) {
      return p == nullptr || (aligned16(p) && (stride == a.width || a.rows == 1));
    };
    const T *x = static_cast<const T*>(a.x), *r = static_cast<const T*>(a.residual);
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(total / 8 + 2, (int64_t)256), 8192);
    if (flat(a.x, a.x_stride) && flat(a.residual, a.residual_stride) && flat(y, y_stride) &&
        a.offset % 8 == 0) {
      if (r)
        k_dropout<T, true><<<grid, 256, 0, st>>>(x, r, total, a.cut, scale, a.seed, a.offset / 8,
                                                 static_cast<T*>(y));
      else
        k_dropout<T, false><<<grid, 256, 0, st>>>(x, r, total, a.cut, scale, a.seed, a.offset / 8,
                                                  static_cast<T*>(y));
    } else {
      k_dropout_any<T><<<grid, 256, 0, st>>>(x, a.x_stride, r, a.residual_stride, total, a.width,
                                             a.cut, scale, a.seed, a.offset, static_cast<T*>(y),
                                             y_stride);
    }
    MGP_HIP_CHECK(hipGetLastError());
  });
}

}  // namespace mgp
