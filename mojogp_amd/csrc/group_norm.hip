// Group norm with an activation over features with positions, channels last.
//
//   x [samples][positions][channels], groups of `size` channels, m = positions size
//   xhat = (x - mean) rstd over a sample's group, z = xhat w + b, y = act(z)
//   dz = dy act'(z); A, B: a sample's sums of dz and dz xhat over the positions
//   dw = sum B, db = sum A over the samples
//   dx = rstd (w dz - (sum_group w A + xhat sum_group w B) / m)
//
// HBM bound.  A thread owns 16 bytes of channels, the same for every row that it takes,
// so that parameters and channel sums stay in its registers at any channel count and
// group size.  Where a workgroup's registers hold whole samples (k_group_fwd,
// k_group_bwd: up to 128 KB a sample forward, 64 KB backward), x and dy are read
// once: z is formed anew in the backward pass, nothing but mean and rstd is kept.
// Larger samples go in stretches of rows (k_group_part, k_group_merge,
// k_group_apply), which read them twice.  Statistics are fp32 means and centred
// squares, merged by counts: a level far above the spread costs no digits.
#include <algorithm>
#include <type_traits>

#include "activation.h"

namespace mgp {

namespace {

template <class T>
struct Raw {  // one vector as it lies in memory
  T v[Vec16<T>::N];
};

// Vectors go at any alignment; of a row's last one `left` elements exist.
template <class T>
__device__ __forceinline__ Raw<T> load_raw(const T* p, int left) {
  constexpr int V = Vec16<T>::N;
  Raw<T> a;
  if (left >= V) {
    __builtin_memcpy(&a, p, sizeof(a));
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) a.v[k] = k < left ? p[k] : (T)0.0f;
  }
  return a;
}

template <class T>
__device__ __forceinline__ void store_raw(T* p, int left, const float* v) {
  constexpr int V = Vec16<T>::N;
  Raw<T> a;
#pragma unroll
  for (int k = 0; k < V; ++k) a.v[k] = (T)v[k];
  if (left >= V) {
    __builtin_memcpy(p, &a, sizeof(a));
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < left) p[k] = a.v[k];
  }
}

// V parameters from channel c on, or the default
template <class T>
__device__ __forceinline__ void load_params(const void* p, int64_t c, int left, bool f32,
                                            float none, float* v) {
#pragma unroll
  for (int k = 0; k < Vec16<T>::N; ++k)
    v[k] = p == nullptr || k >= left ? none
           : f32                     ? static_cast<const float*>(p)[c + k]
                                     : (float)static_cast<const T*>(p)[c + k];
}

// z -> act(z); and with its derivative.
template <class T>
__device__ __forceinline__ void act_values(int act, float* z) {
  constexpr int V = Vec16<T>::N;
  auto go = [&](auto which) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float a, slope;
      activate<which.value, sizeof(T) == 2>(z[k], a, slope);
      z[k] = a;
    }
  };
  if (act >= 0) dispatch_act_device(act, go);
}
template <class T>
__device__ __forceinline__ void act_slopes(int act, const float* z, float* slopes) {
  constexpr int V = Vec16<T>::N;
  auto go = [&](auto which) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float a;
      activate<which.value, sizeof(T) == 2>(z[k], a, slopes[k]);
    }
  };
  if (act >= 0) {
    dispatch_act_device(act, go);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) slopes[k] = 1.0f;
  }
}

struct GroupKernel {
  GroupArgs a;
  const void* dy;
  int64_t ldy;  // of dy (backward) or y (forward)
  void* out;    // y, or dx (or null)
  int64_t ldo;
  float2* stats;   // [samples][groups]: mean, rstd (forward: or null)
  float2* part;    // partial results of channels
  float2* coef;    // [samples][groups]: the two group sums over m
  float inv_m;     // 1 / m
  // whole samples: vectors of a row, rows at a time, samples at a time, threads a
  // group (its sums)
  int cv, rows, at_a_time, lanes;
  int64_t batches;
  // stretches: rows of one, how many a sample, column blocks of 256 vectors
  int64_t stretch;
  int stretches, blocks;
};

// How a sample's group sums come together in a workgroup that holds whole samples:
// through LDS from an entry for each channel or each vector (whose channels are all of
// one group), or, of single positions, by lane exchanges (groups of vectors) or within
// a thread (several groups a vector).
constexpr int kMostThreads = 512;
enum Join : int { CHANNELS = 0, VECTORS = 1, LANES = 2, THREAD = 3 };
// Statistics that a vector's channels have: one, or each its own.
template <class T, int JOIN>
constexpr int kStats = JOIN == CHANNELS || JOIN == THREAD ? Vec16<T>::N : 1;

// What a thread is in such a workgroup.
template <class T, int R, int JOIN>
struct Place {
  static constexpr int V = Vec16<T>::N;
  int slot, col, left, sample, row;  // sample: among those at a time; row: its first
  int slots;                         // rows at a time that are taken, of one sample
  bool active;
  __device__ __forceinline__ explicit Place(const GroupKernel& s) {
    slot = threadIdx.x / s.cv;
    col = (threadIdx.x - slot * s.cv) * V;
    left = s.a.channels - col;
    const int positions = (int)min(s.a.positions, (int64_t)1 << 30);
    slots = min(s.rows, positions);
    sample = slot / slots;
    row = slot - sample * slots;
    active = sample < s.at_a_time;
  }
};

// Sums of a thread's values over blocks of `size` (a power of two up to V).
template <int V>
__device__ __forceinline__ void block_sums(float* v, int size) {
#pragma unroll
  for (int o = 1; o < V; o <<= 1) {
    if (size > o) {
      float w[V];
#pragma unroll
      for (int k = 0; k < V; ++k) w[k] = v[k] + v[k ^ o];
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = w[k];
    }
  }
}

// Where the entries of a pair (sample at a time, group) lie in LDS: runs of `run` from
// `at` on, one for each of the sample's slots, `width` apart.
template <class T, int JOIN>
struct Entries {
  int run, width;
  __device__ __forceinline__ explicit Entries(const GroupKernel& s) {
    constexpr int V = Vec16<T>::N;
    const int size = s.a.channels / s.a.groups;
    run = JOIN == VECTORS ? size / V : size;
    width = JOIN == VECTORS ? s.cv : s.cv * V;
  }
};

__device__ __forceinline__ float lane_sum(float v, int lanes) {
  for (int o = lanes >> 1; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

template <class T, int R, int JOIN>
__global__ __launch_bounds__(kMostThreads) void k_group_fwd(GroupKernel s) {
  constexpr int V = Vec16<T>::N;
  extern __shared__ float2 lds[];
  const Place<T, R, JOIN> at(s);
  const int size = s.a.channels / s.a.groups;
  const int64_t L = s.a.positions;
  float w[V], b[V];
  load_params<T>(s.a.weight, at.col, at.left, s.a.f32_params, 1.0f, w);
  load_params<T>(s.a.bias, at.col, at.left, s.a.f32_params, 0.0f, b);
  for (int64_t batch = blockIdx.x; batch < s.batches; batch += gridDim.x) {
    const int64_t n = batch * s.at_a_time + at.sample;
    const bool in = at.active && n < s.a.samples;
    const T* px = static_cast<const T*>(s.a.x) + (n * L + at.row) * s.a.x_stride + at.col;
    Raw<T> x[R];
    int count = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool has = in && at.row + r * at.slots < L;
      x[r] = load_raw(px + (int64_t)r * at.slots * s.a.x_stride, has ? at.left : 0);
      count += has;
    }
    constexpr int MV = kStats<T, JOIN>;
    float mean[MV], rstd[MV];
    if constexpr (JOIN == THREAD || JOIN == LANES) {
      // of V sums those of a thread's groups
      auto join = [&](const float (&v)[V], float (&sum)[MV]) __attribute__((always_inline)) {
        if constexpr (JOIN == THREAD) {
#pragma unroll
          for (int k = 0; k < V; ++k) sum[k] = v[k];
          block_sums<V>(sum, size);
        } else {
          sum[0] = 0.0f;
#pragma unroll
          for (int k = 0; k < V; ++k) sum[0] += v[k];
          sum[0] = lane_sum(sum[0], s.lanes);
        }
      };
      float v[V], base[MV];  // a value of each group's
      if constexpr (JOIN == THREAD) {
#pragma unroll
        for (int k = 0; k < V; ++k)
          base[k] = (float)(size == 1 ? x[0].v[k] : size == 2 ? x[0].v[k & ~1] : x[0].v[k & ~3]);
      } else {
        base[0] = __shfl((float)x[0].v[0], (threadIdx.x & 63) & ~(s.lanes - 1));
      }
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = (float)x[0].v[k] - base[k % MV];
      join(v, mean);
#pragma unroll
      for (int k = 0; k < MV; ++k) mean[k] = fmaf(mean[k], s.inv_m, base[k]);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        v[k] = (float)x[0].v[k] - mean[k % MV];
        v[k] *= v[k];
      }
      join(v, rstd);
#pragma unroll
      for (int k = 0; k < MV; ++k) rstd[k] = 1.0f / sqrtf(fmaf(rstd[k], s.inv_m, s.a.eps));
      if (s.stats && in && (JOIN == THREAD || at.col % size == 0)) {
#pragma unroll
        for (int k = 0; k < MV; ++k)
          if (k % size == 0 && k < at.left)
            s.stats[n * s.a.groups + (at.col + k) / size] = {mean[k], rstd[k]};
      }
    } else {
      const Entries<T, JOIN> e(s);
      float2* group = lds + (blockDim.x / s.cv) * e.width;  // a pair's mean and rstd
      if (JOIN == VECTORS) {
        const float base = (float)x[0].v[0];
        float m = 0.0f, q = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (r < count) {
#pragma unroll
            for (int k = 0; k < V; ++k) m += (float)x[r].v[k] - base;
          }
        }
        m = base + (count ? m / (float)(count * V) : 0.0f);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (r < count) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
              const float d = (float)x[r].v[k] - m;
              q = fmaf(d, d, q);
            }
          }
        }
        if (at.active) lds[at.slot * e.width + at.col / V] = {m, q};
      } else if (at.active) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float base = (float)x[0].v[k];
          float m = 0.0f, q = 0.0f;
#pragma unroll
          for (int r = 0; r < R; ++r) m += r < count ? (float)x[r].v[k] - base : 0.0f;
          m = base + (count ? m / (float)count : 0.0f);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float d = r < count ? (float)x[r].v[k] - m : 0.0f;
            q = fmaf(d, d, q);
          }
          lds[at.slot * e.width + at.col + k] = {m, q};
        }
      }
      __syncthreads();
      const int pairs = s.at_a_time * s.a.groups;
      const int lane = threadIdx.x & (s.lanes - 1);
      const int teams = blockDim.x / s.lanes;
      const int all = at.slots * e.run;
      for (int p0 = 0; p0 < pairs; p0 += teams) {
        const int p = p0 + threadIdx.x / s.lanes;
        const bool has = p < pairs;
        const int q = p / s.a.groups, g = p - q * s.a.groups;
        const float2* from = lds + q * at.slots * e.width + g * e.run;
        auto sweep = [&](auto f) __attribute__((always_inline)) {
          float t = 0.0f;
          if (has) {
            for (int i = lane; i < all; i += s.lanes) {
              const int slot = i / e.run;
              const int c = ((int)L - slot + at.slots - 1) / at.slots;
              t += f(from[slot * e.width + i - slot * e.run],
                     (float)c * (JOIN == VECTORS ? V : 1));
            }
          }
          return lane_sum(t, s.lanes);
        };
        const float base = has ? from[0].x : 0.0f;
        const float m =
            fmaf(sweep([&](float2 v, float c) { return (v.x - base) * c; }), s.inv_m, base);
        const float var = sweep([&](float2 v, float c) {
                            return fmaf(c * (v.x - m), v.x - m, v.y);
                          }) * s.inv_m;
        if (has && lane == 0) {
          const float2 r = {m, 1.0f / sqrtf(var + s.a.eps)};
          group[p] = r;
          const int64_t to = batch * s.at_a_time + q;
          if (s.stats && to < s.a.samples) s.stats[to * s.a.groups + g] = r;
        }
      }
      __syncthreads();
      if (at.active) {
#pragma unroll
        for (int k = 0; k < MV; ++k) {
          const int c = min(at.col + k, s.a.channels - 1);
          const float2 r = group[at.sample * s.a.groups + c / size];
          mean[k] = r.x;
          rstd[k] = r.y;
        }
      }
    }
    if (in) {
      T* py = static_cast<T*>(s.out) + (n * L + at.row) * s.ldo + at.col;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r < count) {
          float z[V];
#pragma unroll
          for (int k = 0; k < V; ++k)
            z[k] = fmaf(((float)x[r].v[k] - mean[k % MV]) * rstd[k % MV], w[k], b[k]);
          act_values<T>(s.a.activation, z);
          store_raw(py + (int64_t)r * at.slots * s.ldo, at.left, z);
        }
      }
    }
  }
}

// dz of one vector, and what z it had: xhat.
template <class T, int MV>
__device__ __forceinline__ void vector_dz(const GroupArgs& a, const Raw<T>& x, const Raw<T>& dy,
                                          const float (&mean)[MV], const float (&rstd)[MV],
                                          const float* w, const float* b, float* xhat, float* dz) {
  constexpr int V = Vec16<T>::N;
  float z[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    xhat[k] = ((float)x.v[k] - mean[k % MV]) * rstd[k % MV];
    z[k] = fmaf(xhat[k], w[k], b[k]);
  }
  act_slopes<T>(a.activation, z, dz);
#pragma unroll
  for (int k = 0; k < V; ++k) dz[k] *= (float)dy.v[k];
}

// mean and rstd of a vector's channels
template <int MV>
__device__ __forceinline__ void load_stats(const GroupArgs& a, const float2* stats, int64_t n,
                                           int col, float (&mean)[MV], float (&rstd)[MV]) {
  const int size = a.channels / a.groups;
#pragma unroll
  for (int k = 0; k < MV; ++k) {
    const int c = min(col + k, a.channels - 1);
    const float2 r = stats[n * a.groups + c / size];
    mean[k] = r.x;
    rstd[k] = r.y;
  }
}

// part[block][channels]: sums of dz and dz xhat over the block's samples.
template <class T, int R, int JOIN>
__global__ __launch_bounds__(kMostThreads) void k_group_bwd(GroupKernel s) {
  constexpr int V = Vec16<T>::N;
  extern __shared__ float2 lds[];
  const Place<T, R, JOIN> at(s);
  const int size = s.a.channels / s.a.groups;
  const int64_t L = s.a.positions;
  float w[V], b[V], sum_a[V], sum_b[V];
  load_params<T>(s.a.weight, at.col, at.left, s.a.f32_params, 1.0f, w);
  load_params<T>(s.a.bias, at.col, at.left, s.a.f32_params, 0.0f, b);
#pragma unroll
  for (int k = 0; k < V; ++k) sum_a[k] = sum_b[k] = 0.0f;
  for (int64_t batch = blockIdx.x; batch < s.batches; batch += gridDim.x) {
    const int64_t n = batch * s.at_a_time + at.sample;
    const bool in = at.active && n < s.a.samples;
    const int64_t row0 = n * L + at.row;
    const T* px = static_cast<const T*>(s.a.x) + row0 * s.a.x_stride + at.col;
    const T* pd = static_cast<const T*>(s.dy) + row0 * s.ldy + at.col;
    Raw<T> x[R], dy[R];
    int count = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool has = in && at.row + r * at.slots < L;
      x[r] = load_raw(px + (int64_t)r * at.slots * s.a.x_stride, has ? at.left : 0);
      dy[r] = load_raw(pd + (int64_t)r * at.slots * s.ldy, has ? at.left : 0);
      count += has;
    }
    constexpr int MV = kStats<T, JOIN>;
    float mean[MV], rstd[MV], t1[MV], t2[MV];  // t1, t2: the sample's group sums
    if (in) {
      load_stats(s.a, s.stats, n, at.col, mean, rstd);
    } else {
#pragma unroll
      for (int k = 0; k < MV; ++k) mean[k] = rstd[k] = 0.0f;
    }
    {
      float a1[V], a2[V];
#pragma unroll
      for (int k = 0; k < V; ++k) a1[k] = a2[k] = 0.0f;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r < count) {
          float xhat[V], dz[V];
          vector_dz(s.a, x[r], dy[r], mean, rstd, w, b, xhat, dz);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            if (k >= at.left) dz[k] = 0.0f;
            a1[k] += dz[k];
            a2[k] = fmaf(dz[k], xhat[k], a2[k]);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < MV; ++k) t1[k] = t2[k] = 0.0f;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        sum_a[k] += a1[k];
        sum_b[k] += a2[k];
        t1[k % MV] = fmaf(a1[k], w[k], t1[k % MV]);
        t2[k % MV] = fmaf(a2[k], w[k], t2[k % MV]);
      }
    }
    if (s.out == nullptr) continue;
    if constexpr (JOIN == THREAD) {
      block_sums<V>(t1, size);
      block_sums<V>(t2, size);
    } else if constexpr (JOIN == LANES) {
      t1[0] = lane_sum(t1[0], s.lanes);
      t2[0] = lane_sum(t2[0], s.lanes);
    } else {
      const Entries<T, JOIN> e(s);
      float2* group = lds + (blockDim.x / s.cv) * e.width;
      if (at.active) {
#pragma unroll
        for (int k = 0; k < MV; ++k)
          lds[at.slot * e.width + (JOIN == VECTORS ? at.col / V : at.col + k)] = {t1[k], t2[k]};
      }
      __syncthreads();
      const int pairs = s.at_a_time * s.a.groups;
      const int lane = threadIdx.x & (s.lanes - 1);
      const int teams = blockDim.x / s.lanes;
      const int all = at.slots * e.run;
      for (int p0 = 0; p0 < pairs; p0 += teams) {
        const int p = p0 + threadIdx.x / s.lanes;
        const int q = p / s.a.groups, g = p - q * s.a.groups;
        const float2* from = lds + q * at.slots * e.width + g * e.run;
        float2 t = {0.0f, 0.0f};
        if (p < pairs) {
          for (int i = lane; i < all; i += s.lanes) {
            const int slot = i / e.run;
            const float2 v = from[slot * e.width + i - slot * e.run];
            t.x += v.x;
            t.y += v.y;
          }
        }
        t.x = lane_sum(t.x, s.lanes);
        t.y = lane_sum(t.y, s.lanes);
        if (p < pairs && lane == 0) group[p] = t;
      }
      __syncthreads();
      if (at.active) {
#pragma unroll
        for (int k = 0; k < MV; ++k) {
          const int c = min(at.col + k, s.a.channels - 1);
          const float2 r = group[at.sample * s.a.groups + c / size];
          t1[k] = r.x;
          t2[k] = r.y;
        }
      }
    }
    if (in) {
      T* po = static_cast<T*>(s.out) + row0 * s.ldo + at.col;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r < count) {
          float xhat[V], dz[V];
          vector_dz(s.a, x[r], dy[r], mean, rstd, w, b, xhat, dz);
#pragma unroll
          for (int k = 0; k < V; ++k)
            dz[k] = rstd[k % MV] *
                    fmaf(w[k], dz[k], -s.inv_m * fmaf(xhat[k], t2[k % MV], t1[k % MV]));
          store_raw(po + (int64_t)r * at.slots * s.ldo, at.left, dz);
        }
      }
    }
    if constexpr (JOIN == CHANNELS || JOIN == VECTORS) __syncthreads();
  }
  if (s.part == nullptr) return;
  // the slots' sums of each channel
  const int width = s.cv * V, taken = at.slots * s.at_a_time;
  if (at.active) {
#pragma unroll
    for (int k = 0; k < V; ++k) lds[at.slot * width + at.col + k] = {sum_a[k], sum_b[k]};
  }
  __syncthreads();
  for (int c = threadIdx.x; c < s.a.channels; c += blockDim.x) {
    float2 t = lds[c];
    for (int q = 1; q < taken; ++q) {
      const float2 v = lds[q * width + c];
      t.x += v.x;
      t.y += v.y;
    }
    s.part[(int64_t)blockIdx.x * s.a.channels + c] = t;
  }
}

// ---------------------------------------------------------------- samples in stretches

constexpr int kPartThreads = 256;

// A stretch of rows of one sample, in one block of columns.
template <class T>
struct Piece {
  static constexpr int V = Vec16<T>::N;
  int64_t n, row0, rows;  // first row within the sample
  int64_t chunk;
  int col, cv, slots, slot, left, base;  // vectors of the block, rows at a time; base: its first channel
  bool active;
  __device__ __forceinline__ Piece(const GroupKernel& s, int64_t item) {
    const int64_t block = item % s.blocks, at = item / s.blocks;
    chunk = at % s.stretches;
    n = at / s.stretches;
    row0 = chunk * s.stretch;
    rows = min(s.stretch, s.a.positions - row0);
    base = (int)block * kPartThreads * V;
    cv = min(kPartThreads, (s.a.channels - base + V - 1) / V);
    slots = kPartThreads / cv;
    slot = threadIdx.x / cv;
    col = base + (threadIdx.x - slot * cv) * V;
    left = s.a.channels - col;
    active = slot < slots;
  }
  __device__ __forceinline__ int64_t count_of(int slot_) const {  // its rows
    return rows > slot_ ? (rows - slot_ + slots - 1) / slots : 0;
  }
};

// part[sample][stretch][channels]: mean and centred squares of a channel; BACK: its
// sums of dz and dz xhat.
template <class T, bool BACK, int MV>
__global__ __launch_bounds__(kPartThreads) void k_group_part(GroupKernel s, int64_t items) {
  constexpr int V = Vec16<T>::N, U = 4;
  __shared__ float2 lds[kPartThreads * V];
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const Piece<T> at(s, item);
    const int64_t row = at.n * s.a.positions + at.row0 + at.slot;
    const T* px = static_cast<const T*>(s.a.x) + row * s.a.x_stride + at.col;
    const int64_t sx = (int64_t)at.slots * s.a.x_stride;
    const int64_t count = at.active ? at.count_of(at.slot) : 0;
    float m[V], q[V];  // or the two sums
#pragma unroll
    for (int k = 0; k < V; ++k) m[k] = q[k] = 0.0f;
    if constexpr (!BACK) {
      int64_t done = 0;
      const Raw<T> base = load_raw(px, count ? at.left : 0);  // means are formed from here
      for (; done + U <= count; done += U) {
        Raw<T> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = load_raw(px + (done + u) * sx, at.left);
        const float n1 = (float)done, share = (float)U / (float)(done + U);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          float v[U];
#pragma unroll
          for (int u = 0; u < U; ++u) v[u] = (float)x[u].v[k] - (float)base.v[k];
          const float mean = ((v[0] + v[1]) + (v[2] + v[3])) * 0.25f;
          float sq = 0.0f;
#pragma unroll
          for (int u = 0; u < U; ++u) sq = fmaf(v[u] - mean, v[u] - mean, sq);
          const float d = mean - m[k];
          m[k] = fmaf(d, share, m[k]);
          q[k] += fmaf(d * d, n1 * share, sq);
        }
      }
      for (; done < count; ++done) {
        const Raw<T> x = load_raw(px + done * sx, at.left);
        const float n1 = (float)done, share = 1.0f / (float)(done + 1);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float d = ((float)x.v[k] - (float)base.v[k]) - m[k];
          m[k] = fmaf(d, share, m[k]);
          q[k] = fmaf(d * d, n1 * share, q[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < V; ++k) m[k] += (float)base.v[k];
    } else if (at.active) {
      const T* pd = static_cast<const T*>(s.dy) + row * s.ldy + at.col;
      const int64_t sd = (int64_t)at.slots * s.ldy;
      float w[V], b[V], mean[MV], rstd[MV];
      load_params<T>(s.a.weight, at.col, at.left, s.a.f32_params, 1.0f, w);
      load_params<T>(s.a.bias, at.col, at.left, s.a.f32_params, 0.0f, b);
      load_stats(s.a, s.stats, at.n, at.col, mean, rstd);
      auto add = [&](const Raw<T>& x, const Raw<T>& dy) __attribute__((always_inline)) {
        float xhat[V], dz[V];
        vector_dz(s.a, x, dy, mean, rstd, w, b, xhat, dz);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          m[k] += dz[k];
          q[k] = fmaf(dz[k], xhat[k], q[k]);
        }
      };
      int64_t done = 0;
      for (; done + U <= count; done += U) {
        Raw<T> x[U], dy[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          x[u] = load_raw(px + (done + u) * sx, at.left);
          dy[u] = load_raw(pd + (done + u) * sd, at.left);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) add(x[u], dy[u]);
      }
      for (; done < count; ++done)
        add(load_raw(px + done * sx, at.left), load_raw(pd + done * sd, at.left));
    }
    const int width = at.cv * V;
    if (at.active) {
#pragma unroll
      for (int k = 0; k < V; ++k) lds[at.slot * width + at.col - at.base + k] = {m[k], q[k]};
    }
    __syncthreads();
    float2* to = s.part + (at.n * s.stretches + at.chunk) * s.a.channels + at.base;
    const int used = (int)min((int64_t)at.slots, at.rows);
    for (int c = threadIdx.x; c < min(width, s.a.channels - at.base); c += kPartThreads) {
      float2 t = lds[c];
      if constexpr (BACK) {
        for (int k = 1; k < used; ++k) {
          const float2 v = lds[k * width + c];
          t.x += v.x;
          t.y += v.y;
        }
      } else {
        // rows of the first `more` slots: one more than of the others
        const float few = (float)(at.rows / at.slots);
        const int more = (int)(at.rows - at.rows / at.slots * at.slots);
        float sum = 0.0f;
        for (int k = 1; k < used; ++k)
          sum = fmaf(lds[k * width + c].x - t.x, few + (k < more ? 1.0f : 0.0f), sum);
        const float mean = t.x + sum / (float)at.rows;
        float sq = 0.0f;
        for (int k = 0; k < used; ++k) {
          const float2 v = lds[k * width + c];
          sq += fmaf((v.x - mean) * (v.x - mean), few + (k < more ? 1.0f : 0.0f), v.y);
        }
        t = {mean, sq};
      }
      to[c] = t;
    }
    __syncthreads();
  }
}

// A wave a group: its mean and rstd, or (BACK) the two sums over m.
template <class T, bool BACK>
__global__ __launch_bounds__(256) void k_group_merge(GroupKernel s) {
  const int lane = threadIdx.x & 63;
  const int size = s.a.channels / s.a.groups;
  const int64_t pairs = s.a.samples * s.a.groups, all = (int64_t)s.stretches * size;
  for (int64_t p = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); p < pairs;
       p += (int64_t)gridDim.x * 4) {
    const int64_t n = p / s.a.groups;
    const int g = (int)(p - n * s.a.groups);
    const float2* from = s.part + n * s.stretches * s.a.channels + (int64_t)g * size;
    auto sweep = [&](auto f) __attribute__((always_inline)) {
      float t = 0.0f;
      for (int64_t i = lane; i < all; i += 64) {
        const int64_t chunk = i / size;
        const int d = (int)(i - chunk * size);
        t += f(from[chunk * s.a.channels + d],
               (float)min(s.stretch, s.a.positions - chunk * s.stretch), g * size + d);
      }
      return lane_sum(t, 64);
    };
    if constexpr (!BACK) {
      const float base = from[0].x;
      const float m =
          fmaf(sweep([&](float2 v, float c, int) { return (v.x - base) * c; }), s.inv_m, base);
      const float var = sweep([&](float2 v, float c, int) {
                          return fmaf(c * (v.x - m), v.x - m, v.y);
                        }) * s.inv_m;
      if (lane == 0) s.stats[p] = {m, 1.0f / sqrtf(var + s.a.eps)};
    } else {
      auto weight = [&](int c) __attribute__((always_inline)) {
        return s.a.weight == nullptr ? 1.0f
               : s.a.f32_params      ? static_cast<const float*>(s.a.weight)[c]
                                     : (float)static_cast<const T*>(s.a.weight)[c];
      };
      const float t1 = sweep([&](float2 v, float, int c) { return v.x * weight(c); });
      const float t2 = sweep([&](float2 v, float, int c) { return v.y * weight(c); });
      if (lane == 0) s.coef[p] = {t1 * s.inv_m, t2 * s.inv_m};
    }
  }
}

// y, or (BACK) dx, of a stretch.
template <class T, bool BACK, int MV>
__global__ __launch_bounds__(kPartThreads) void k_group_apply(GroupKernel s, int64_t items) {
  constexpr int V = Vec16<T>::N, U = BACK ? 2 : 4;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const Piece<T> at(s, item);
    if (!at.active) continue;
    const int64_t row = at.n * s.a.positions + at.row0 + at.slot, count = at.count_of(at.slot);
    const T* px = static_cast<const T*>(s.a.x) + row * s.a.x_stride + at.col;
    T* po = static_cast<T*>(s.out) + row * s.ldo + at.col;
    const int64_t sx = (int64_t)at.slots * s.a.x_stride, so = (int64_t)at.slots * s.ldo;
    float w[V], b[V], mean[MV], rstd[MV];
    load_params<T>(s.a.weight, at.col, at.left, s.a.f32_params, 1.0f, w);
    load_params<T>(s.a.bias, at.col, at.left, s.a.f32_params, 0.0f, b);
    load_stats(s.a, s.stats, at.n, at.col, mean, rstd);
    if constexpr (!BACK) {
      auto put = [&](const Raw<T>& x, int64_t i) __attribute__((always_inline)) {
        float z[V];
#pragma unroll
        for (int k = 0; k < V; ++k)
          z[k] = fmaf(((float)x.v[k] - mean[k % MV]) * rstd[k % MV], w[k], b[k]);
        act_values<T>(s.a.activation, z);
        store_raw(po + i * so, at.left, z);
      };
      int64_t i = 0;
      for (; i + U <= count; i += U) {
        Raw<T> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = load_raw(px + (i + u) * sx, at.left);
#pragma unroll
        for (int u = 0; u < U; ++u) put(x[u], i + u);
      }
      for (; i < count; ++i) put(load_raw(px + i * sx, at.left), i);
    } else {
      const T* pd = static_cast<const T*>(s.dy) + row * s.ldy + at.col;
      const int64_t sd = (int64_t)at.slots * s.ldy;
      float c1[MV], c2[MV];
      load_stats(s.a, s.coef, at.n, at.col, c1, c2);
      auto put = [&](const Raw<T>& x, const Raw<T>& dy, int64_t i) __attribute__((always_inline)) {
        float xhat[V], dz[V];
        vector_dz(s.a, x, dy, mean, rstd, w, b, xhat, dz);
#pragma unroll
        for (int k = 0; k < V; ++k)
          dz[k] = rstd[k % MV] * fmaf(w[k], dz[k], -fmaf(xhat[k], c2[k % MV], c1[k % MV]));
        store_raw(po + i * so, at.left, dz);
      };
      int64_t i = 0;
      for (; i + U <= count; i += U) {
        Raw<T> x[U], dy[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          x[u] = load_raw(px + (i + u) * sx, at.left);
          dy[u] = load_raw(pd + (i + u) * sd, at.left);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) put(x[u], dy[u], i + u);
      }
      for (; i < count; ++i)
        put(load_raw(px + i * sx, at.left), load_raw(pd + i * sd, at.left), i);
    }
  }
}

// dweight, dbias: sums of the partial results in a fixed order, 16 channels a
// workgroup.
template <class P>
__global__ __launch_bounds__(1024) void k_group_params(const float2* __restrict__ part,
                                                       int64_t parts, int channels,
                                                       P* __restrict__ dweight,
                                                       P* __restrict__ dbias) {
  __shared__ float2 red[64][16];
  const int c = threadIdx.x & 15, line = threadIdx.x >> 4, channel = blockIdx.x * 16 + c;
  float2 t = {0.0f, 0.0f};
  if (channel < channels) {
#pragma unroll 4
    for (int64_t p = line; p < parts; p += 64) {
      const float2 v = part[p * channels + channel];
      t.x += v.x;
      t.y += v.y;
    }
  }
  red[line][c] = t;
  __syncthreads();
  for (int o = 32; o >= 1; o >>= 1) {
    if (line < o) {
      red[line][c].x += red[line + o][c].x;
      red[line][c].y += red[line + o][c].y;
    }
    __syncthreads();
  }
  if (line != 0 || channel >= channels) return;
  if (dbias) dbias[channel] = (P)red[0][c].x;
  if (dweight) dweight[channel] = (P)red[0][c].y;
}

// ---------------------------------------------------------------- host side

constexpr int64_t kBackBlocks = 1024;  // partial results of whole samples, at most

struct Cut {
  bool whole;  // samples in a workgroup's registers
  int join = CHANNELS, r = 1, threads = 256;
  size_t lds = 0;
};

inline int pow2_at_most(int64_t v) {
  int p = 1;
  while (2 * (int64_t)p <= v) p *= 2;
  return p;
}

// Fills in how the call is cut.
Cut cut_of(GroupKernel& s, bool back) {
  const GroupArgs& a = s.a;
  const int V = a.type == ELEM_F32 ? 4 : 8;
  const int size = a.channels / a.groups, most = back ? 8 : 16;
  const int64_t cv = ceil_div((int64_t)a.channels, (int64_t)V), L = a.positions;
  s.inv_m = (float)(1.0 / ((double)L * size));
  Cut c{};
  int threads = 256;
  while (threads < kMostThreads && (cv > threads || ceil_div(L, (int64_t)(threads / cv)) > 4)) threads *= 2;
  c.whole = cv <= threads && ceil_div(L, (int64_t)(threads / cv)) <= most;
  if (!c.whole) {
    s.blocks = (int)ceil_div(cv, (int64_t)kPartThreads);
    // about eight workgroups a CU, each thread at least eight rows
    const int64_t slots = std::max<int64_t>(1, kPartThreads / cv);
    const int64_t want = ceil_div((int64_t)2048, a.samples * s.blocks);
    s.stretches = (int)std::max<int64_t>(1, std::min(want, L / (8 * slots)));
    s.stretch = ceil_div(L, (int64_t)s.stretches);
    s.stretches = (int)ceil_div(L, s.stretch);
    return c;
  }
  s.cv = (int)cv;
  s.rows = threads / s.cv;
  c.threads = threads;
  s.at_a_time = (int)std::max<int64_t>(1, s.rows / L);
  s.batches = ceil_div(a.samples, (int64_t)s.at_a_time);
  const int64_t r = ceil_div(L, (int64_t)s.rows);
  c.r = r <= 1 ? 1 : r <= 4 ? 4 : most;
  const bool pow2 = (size & (size - 1)) == 0;
  if (L == 1 && pow2 && size < V) {
    c.join = THREAD;
    s.lanes = 1;
  } else if (L == 1 && pow2 && size / V <= 64) {
    c.join = LANES;
    s.lanes = size / V;
  } else {
    c.join = size % V == 0 ? VECTORS : CHANNELS;
    const int64_t slots = std::min<int64_t>(s.rows, L);
    const int64_t entries = slots * (c.join == VECTORS ? size / V : size);
    const int64_t pairs = (int64_t)s.at_a_time * a.groups;
    s.lanes = std::min({64, pow2_at_most(2 * entries - 1),
                        pow2_at_most(std::max<int64_t>(1, threads / pairs))});
    c.lds = ((size_t)s.rows * s.cv * (c.join == VECTORS ? 1 : V) + (size_t)pairs) * sizeof(float2);
  }
  if (back) c.lds = std::max(c.lds, (size_t)s.rows * s.cv * V * sizeof(float2));
  return c;
}

inline unsigned back_blocks(const GroupKernel& s) {
  return (unsigned)std::min<int64_t>(s.batches, kBackBlocks);
}

template <class T, bool BACK, class F>
void dispatch_whole(const Cut& c, F&& f) {
  auto with = [&](auto r) {
    if (c.join == CHANNELS)
      f(r, std::integral_constant<int, CHANNELS>{});
    else
      f(r, std::integral_constant<int, VECTORS>{});
  };
  if (c.join == THREAD) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, THREAD>{});
  if (c.join == LANES) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, LANES>{});
  if (c.r == 1)
    with(std::integral_constant<int, 1>{});
  else if (c.r == 4)
    with(std::integral_constant<int, 4>{});
  else
    with(std::integral_constant<int, BACK ? 8 : 16>{});
}

template <class T, bool BACK>
void launch_stretches(GroupKernel& s, hipStream_t st) {
  const int64_t items = s.a.samples * s.stretches * s.blocks;
  const unsigned grid = (unsigned)std::min<int64_t>(items, 1 << 16);
  const unsigned waves =
      (unsigned)std::min<int64_t>(ceil_div(s.a.samples * s.a.groups, (int64_t)4), 1 << 14);
  auto go = [&](auto mv) {
    k_group_part<T, BACK, mv.value><<<grid, kPartThreads, 0, st>>>(s, items);
    if (BACK && s.out == nullptr) return;
    k_group_merge<T, BACK><<<waves, 256, 0, st>>>(s);
    k_group_apply<T, BACK, mv.value><<<grid, kPartThreads, 0, st>>>(s, items);
  };
  constexpr int V = Vec16<T>::N;
  if (s.a.channels / s.a.groups % V == 0)  // a vector's channels are of one group
    go(std::integral_constant<int, 1>{});
  else
    go(std::integral_constant<int, V>{});
}

inline size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }
inline size_t pairs_bytes(const GroupArgs& a) {
  return aligned((size_t)(a.samples * a.groups) * sizeof(float2));
}

}  // namespace

size_t group_norm_bytes(const GroupArgs& a, bool back) {
  if (a.samples * a.positions == 0) return 0;
  GroupKernel s{};
  s.a = a;
  const Cut c = cut_of(s, back);
  const size_t row = (size_t)a.channels * sizeof(float2);
  if (c.whole) return back ? aligned(back_blocks(s) * row) : 0;
  return aligned((size_t)(a.samples * s.stretches) * row) + pairs_bytes(a);
}

void group_norm(const GroupArgs& a, void* y, int64_t y_stride, float* stats, void* ws,
                hipStream_t st) {
  if (a.samples * a.positions == 0) return;
  GroupKernel s{};
  s.a = a;
  s.out = y;
  s.ldo = y_stride;
  s.stats = reinterpret_cast<float2*>(stats);
  const Cut c = cut_of(s, false);
  dispatch_elem(a.type, [&](auto tag) {
    using T = decltype(tag);
    if (!c.whole) {
      s.part = static_cast<float2*>(ws);
      if (!stats)
        s.stats = s.part + aligned((size_t)(a.samples * s.stretches) * a.channels * sizeof(float2)) /
                               sizeof(float2);
      launch_stretches<T, false>(s, st);
      return;
    }
    const unsigned grid = (unsigned)std::min<int64_t>(s.batches, 1 << 16);
    dispatch_whole<T, false>(c, [&](auto r, auto join) {
      k_group_fwd<T, r.value, join.value><<<grid, c.threads, c.lds, st>>>(s);
    });
  });
  MGP_HIP_CHECK(hipGetLastError());
}

void group_norm_backward(const GroupArgs& a, const void* dy, int64_t dy_stride, const float* stats,
                         void* dx, int64_t dx_stride, void* dweight, void* dbias, void* ws,
                         hipStream_t st) {
  GroupKernel s{};
  s.a = a;
  s.dy = dy;
  s.ldy = dy_stride;
  s.out = dx;
  s.ldo = dx_stride;
  s.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  const bool params = dweight || dbias;
  int64_t parts = 0;
  if (a.samples * a.positions > 0) {
    const Cut c = cut_of(s, true);
    dispatch_elem(a.type, [&](auto tag) {
      using T = decltype(tag);
      s.part = static_cast<float2*>(ws);
      if (!c.whole) {
        parts = a.samples * s.stretches;
        s.coef = s.part + aligned((size_t)parts * a.channels * sizeof(float2)) / sizeof(float2);
        launch_stretches<T, true>(s, st);
        return;
      }
      parts = back_blocks(s);
      if (!params) s.part = nullptr;
      dispatch_whole<T, true>(c, [&](auto r, auto join) {
        k_group_bwd<T, r.value, join.value><<<(unsigned)parts, c.threads, c.lds, st>>>(s);
      });
    });
  }
  if (params) {
    const unsigned grid = (unsigned)ceil_div((int64_t)a.channels, (int64_t)16);
    const float2* part = static_cast<const float2*>(ws);
    dispatch_elem(a.f32_params ? ELEM_F32 : a.type, [&](auto tag) {
      using P = decltype(tag);
      k_group_params<P><<<grid, 1024, 0, st>>>(part, parts, a.channels, static_cast<P*>(dweight),
                                               static_cast<P*>(dbias));
    });
  }
  MGP_HIP_CHECK(hipGetLastError());
}

}  // namespace mgp
