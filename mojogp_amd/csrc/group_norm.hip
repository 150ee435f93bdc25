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
//
// Measured: 250000 x 1 x 256 bf16 by 8 channels, silu, forward 72 us, backward 96 (4.4 and 4.6
// TB/s with the statistics); 32 x 4096 x 512 bf16 in stretches, forward 38 + 53 us,
// backward 52 + 76 (3.6 to 7 TB/s, the second reads partly from the last-level cache).
// Samples in registers wait on VALU too: 3000 x 64 x 512 bf16 by 16 channels, forward 111 us
// (3.5 TB/s), backward 255.
#include <algorithm>
#include <type_traits>

#include "activation.h"
#include "product.h"

namespace mgp {

namespace {

// How a kernel reads: elements of type T, V channels a thread (16 bytes of them, or
// one where a row has fewer).
template <class E, int V_>
struct Kind {
  using T = E;
  static constexpr int V = V_;
};

template <class K>
struct Raw {  // one vector as it lies in memory
  typename K::T v[K::V];
};

// Vectors go at any alignment.
template <class K>
__device__ __forceinline__ Raw<K> load_raw(const typename K::T* p) {
  Raw<K> a;
  __builtin_memcpy(&a, p, sizeof(a));
  return a;
}

// The elements of a vector from the `from`th on.
template <class K>
__device__ __forceinline__ void store_raw(typename K::T* p, int from, const float* v) {
  Raw<K> a;
#pragma unroll
  for (int k = 0; k < K::V; ++k) a.v[k] = (typename K::T)v[k];
  if (from == 0) {
    __builtin_memcpy(p, &a, sizeof(a));
  } else {
#pragma unroll
    for (int k = 0; k < K::V; ++k)
      if (k >= from) p[k] = a.v[k];
  }
}

// V parameters from channel c on, or the default
template <class K>
__device__ __forceinline__ void load_params(const void* p, int c, bool f32, float none, float* v) {
  if (p == nullptr) {
#pragma unroll
    for (int k = 0; k < K::V; ++k) v[k] = none;
  } else if (f32) {
    load_run<K::V>(static_cast<const float*>(p) + c, K::V, v);
  } else {
    load_run<K::V>(static_cast<const typename K::T*>(p) + c, K::V, v);
  }
}

// xhat and z of a vector, by the same operations in every pass: a slope is that of the
// value that the forward pass activated, at the jump of relu's too.
template <class K, int MV>
__device__ __forceinline__ void normalise(const Raw<K>& x, const float (&mean)[MV],
                                          const float (&rstd)[MV], const float* w, const float* b,
                                          float* xhat, float* z) {
#pragma unroll
  for (int k = 0; k < K::V; ++k) {
    xhat[k] = ((float)x.v[k] - mean[k % MV]) * rstd[k % MV];
    z[k] = fmaf(xhat[k], w[k], b[k]);
  }
}

// z -> act(z); and with its derivative.
template <class K>
__device__ __forceinline__ void act_values(int act, float* z) {
  constexpr int V = K::V;
  auto go = [&](auto which) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float a, slope;
      activate<which.value, sizeof(typename K::T) == 2>(z[k], a, slope);
      z[k] = a;
    }
  };
  if (act >= 0) dispatch_act_device(act, go);
}
template <class K>
__device__ __forceinline__ void act_slopes(int act, const float* z, float* slopes) {
  constexpr int V = K::V;
  auto go = [&](auto which) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      float a;
      activate<which.value, sizeof(typename K::T) == 2>(z[k], a, slopes[k]);
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
  bool apart;      // the result shares no memory with what is read
  // in registers: vectors of a row, rows of a sample at a time, samples at a time, threads
  // a group (its sums), and of them on the entries of one row
  int cv, slots, at_a_time, lanes, run_lanes;
  int64_t batches;
  // blocks of groups a sample is dealt out in; in the kernels a.groups and a.channels are
  // a block's, and these a sample's
  int group_blocks, all_groups, all_channels;
  // stretches: rows of one, how many a sample, column blocks of cv vectors
  int stretch, short_stretch;  // of partial results, and of the results
  int stretches, shorts, blocks;
};

// What a workgroup that holds samples, or one block of groups of them, takes: batches of
// samples from `first` on, `step` apart.  Neighbouring groups, which share lines of
// memory, go to workgroups of one XCD.
struct Share {
  int64_t first, step;
};
template <class T>
__device__ __forceinline__ Share share_of(GroupKernel& s) {
  if (s.group_blocks == 1) return {blockIdx.x, gridDim.x};
  const uint32_t total = gridDim.x, xcd = blockIdx.x & 7, per = total >> 3, rest = total & 7;
  const uint32_t unit = xcd * per + min(xcd, rest) + (blockIdx.x >> 3);
  const uint32_t n = unit / (uint32_t)s.group_blocks, block = unit - n * s.group_blocks;
  const int col = (int)block * s.a.channels;
  const auto on = [&](const void* p, bool f32) {
    return p == nullptr ? p
           : f32        ? static_cast<const void*>(static_cast<const float*>(p) + col)
                        : static_cast<const void*>(static_cast<const T*>(p) + col);
  };
  s.a.x = on(s.a.x, false);
  s.dy = on(s.dy, false);
  s.out = const_cast<void*>(on(s.out, false));
  s.a.weight = on(s.a.weight, s.a.f32_params);
  s.a.bias = on(s.a.bias, s.a.f32_params);
  if (s.stats) s.stats += block * s.a.groups;
  if (s.part) s.part += (int64_t)n * s.all_channels + col;
  return {n, total / (uint32_t)s.group_blocks};
}

// How a sample's group sums come together in a workgroup that holds whole samples:
// through LDS from an entry for each vector (whose channels are all of one group) or for
// each group that has channels of it, or, of single positions, by lane exchanges
// (groups of vectors) or within a thread (several groups a vector).
constexpr int kMostThreads = 512;
enum Join : int { SEGMENTS = 0, VECTORS = 1, LANES = 2, THREAD = 3 };
// Statistics that a vector's channels have: one, or each its own.
template <class K, int JOIN>
constexpr int kStats = JOIN == SEGMENTS || JOIN == THREAD ? K::V : 1;

// The channels of a thread: vector j of those from `base` on.  The last one of a row
// ends with it, and shares its first `dup` channels with the one before, so that rows of
// any width are read as vectors.  A result in the place of what is read is stored by
// one thread (from): the shared channels may be read when the other has written
// them, and are not used.
template <class K>
struct Columns {
  int vector, col, dup, from;
  __device__ __forceinline__ Columns(const GroupKernel& s, int base, int j) : vector(j) {
    const int first = base + j * K::V;
    dup = max(first + K::V - s.a.channels, 0);
    col = first - dup;
    from = s.apart ? 0 : dup;
  }
};

// What a thread is in such a workgroup.
template <class K>
struct Place : Columns<K> {
  int slot, sample, row;  // sample: among those at a time; row: its first
  int slots;              // rows at a time that are taken, of one sample
  int rows;               // its rows of a sample
  bool active;
  __device__ __forceinline__ explicit Place(const GroupKernel& s)
      : Columns<K>(s, 0, (int)threadIdx.x - (int)threadIdx.x / s.cv * s.cv) {
    slot = threadIdx.x / s.cv;
    slots = s.slots;
    sample = slot / slots;
    row = slot - sample * slots;
    active = sample < s.at_a_time;
    rows = ((int)min(s.a.positions, (int64_t)1 << 30) - row + slots - 1) / slots;
  }
  // Elements from the batch's first row to the thread's; how many rows it has in one.
  __device__ __forceinline__ int64_t offset(const GroupKernel& s, int64_t stride) const {
    return (sample * s.a.positions + row) * stride + this->col;
  }
  __device__ __forceinline__ int count(const GroupKernel& s, int64_t batch) const {
    const int live = (int)min((int64_t)s.at_a_time, s.a.samples - batch * s.at_a_time);
    return active && sample < live ? rows : 0;
  }
};

// Elements from the first row to a batch's.
__device__ __forceinline__ int64_t batch_offset(const GroupKernel& s, int64_t batch,
                                                int64_t stride) {
  return batch * s.at_a_time * s.a.positions * stride;
}

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

// Groups that V consecutive channels belong to, at most; vectors that hold channels of a
// group.
__host__ __device__ constexpr int most_groups(int V, int size) {
  return (V + size - 2) / size + 1 < V ? (V + size - 2) / size + 1 : V;
}
__host__ __device__ constexpr int vectors_of(int join, int V, int size) {
  return join == VECTORS ? (size + V - 1) / V : (size + V - 2) / V + 1;
}

// The entries in LDS: `each` for a vector of a slot (of the groups from that of the
// vector's own first channel on), `plane` apart, so that neighbouring threads write
// neighbouring ones.  (Planes are 64 bytes off each other's banks, as neighbouring groups
// are read together, but for the widest, which fill 64 KB with the groups' results.)
__host__ __device__ constexpr int plane_of(int threads) {
  return (threads + 31) / 32 * 32 + (threads <= 256 ? 8 : 0);
}
template <class K, int JOIN>
struct Entries {
  int size, run, plane, all;
  int few, more;  // rows of a slot: one more than few in the first `more` slots
  __device__ __forceinline__ Entries(const GroupKernel& s, int size_, int slots) : size(size_) {
    run = vectors_of(JOIN, K::V, size);
    plane = plane_of(slots * s.at_a_time * s.cv);
    all = plane * (JOIN == VECTORS ? 1 : most_groups(K::V, size));
    few = (int)s.a.positions / slots;
    more = (int)s.a.positions - few * slots;
  }
  // the first entry of group g in a slot
  __device__ __forceinline__ int first_of(int g) const {
    const int j0 = g * size / K::V;
    return j0 + (JOIN == VECTORS ? 0 : (g - j0 * K::V / size) * plane);
  }
  // f(entry, its values) of group g for a sample whose first slot is `first`,
  // dealt out among the pair's lanes.
  template <class F>
  __device__ __forceinline__ void each_of(const GroupKernel& s, const float2* first, int slots,
                                          int lane, int g, F&& f) const {
    constexpr int V = K::V;
    const int c0 = g * size, j0 = c0 / V, at0 = first_of(g);
    const int rows = s.lanes / s.run_lanes, slot0 = lane / s.run_lanes;
    for (int in = lane & (s.run_lanes - 1); in < run; in += s.run_lanes) {
      const int v0 = (j0 + in) * V, n = min(v0 + V, c0 + size) - max(v0, c0);
      if (n <= 0) break;
      const float2* from = first + (in == 0 ? at0 : j0 + in) + slot0 * s.cv;
      const float less = (float)(few * n), greater = (float)((few + 1) * n);
      for (int slot = slot0; slot < slots; slot += rows, from += rows * s.cv)
        f(*from, slot < more ? greater : less);
    }
  }
};

// Runs add(k, n) for each of a vector's own channels, n being how many of its group
// went before in the vector, and end(t) behind the last one of each group.
template <int V, class A, class E>
__device__ __forceinline__ void segments(int size, int within, int dup, A&& add, E&& end) {
  int n = 0, t = 0;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const bool last = ++within == size;
    if (k >= dup) {
      add(k, n);
      ++n;
      if (last || k == V - 1) {
        end(t);
        ++t;
        n = 0;
      }
    }
    if (last) within = 0;
  }
}

// mean and rstd of a vector's channels, the first of which is the `in`th of group g;
// row: those of the sample
template <int MV>
__device__ __forceinline__ void load_stats(int size, const float2* row, int g, int in,
                                           float (&mean)[MV], float (&rstd)[MV]) {
#pragma unroll
  for (int k = 0; k < MV; ++k) {
    const float2 r = row[g];
    mean[k] = r.x;
    rstd[k] = r.y;
    if (++in == size && k + 1 < MV) {
      in = 0;
      ++g;
    }
  }
}

__device__ __forceinline__ float lane_sum(float v, int lanes) {
  for (int o = lanes >> 1; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

template <class K, int R, int JOIN>
__global__ __launch_bounds__(kMostThreads) void k_group_fwd(GroupKernel s) {
  using T = typename K::T;
  constexpr int V = K::V;
  extern __shared__ float2 lds[];
  const Share mine = share_of<T>(s);
  const Place<K> at(s);
  const int size = s.a.channels / s.a.groups;
  float w[V], b[V];
  load_params<K>(s.a.weight, at.col, s.a.f32_params, 1.0f, w);
  load_params<K>(s.a.bias, at.col, s.a.f32_params, 0.0f, b);
  const Entries<K, JOIN> e(s, size, at.slots);
  const int first_group = at.col / size, within = at.col - first_group * size;
  const int64_t off = at.offset(s, s.a.x_stride), off_y = at.offset(s, s.ldo);
  auto load = [&](int64_t batch, Raw<K> (&x)[R]) __attribute__((always_inline)) {
    const T* px = static_cast<const T*>(s.a.x) + batch_offset(s, batch, s.a.x_stride) + off;
    const int count = at.count(s, batch);
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (r < count) x[r] = load_raw<K>(px + (int64_t)r * at.slots * s.a.x_stride);
    return count;
  };
  auto one = [&](int64_t batch, Raw<K> (&x)[R], int count) __attribute__((always_inline)) {
    const int64_t n = batch * s.at_a_time + at.sample;
    const bool in = count > 0;
    constexpr int MV = kStats<K, JOIN>;
    float mean[MV], rstd[MV];
    if constexpr (JOIN == THREAD || JOIN == LANES) {
      if (!in) x[0] = Raw<K>{};
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
        base[0] = (float)x[0].v[0];
        if (s.lanes > 1) base[0] = __shfl(base[0], (threadIdx.x & 63) & ~(s.lanes - 1));
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
          if (k % size == 0 && k >= at.dup)
            s.stats[n * s.all_groups + (at.col + k) / size] = {mean[k], rstd[k]};
      }
    } else {
      float2* group = lds + e.all;  // a pair's mean and rstd
      if (JOIN == VECTORS) {
        const float base = (float)x[0].v[V - 1];
        float m = 0.0f, q = 0.0f;
        auto moments = [&](auto odd) __attribute__((always_inline)) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            if (r < count) {
#pragma unroll
              for (int k = 0; k < V; ++k)
                m += !odd.value || k >= at.dup ? (float)x[r].v[k] - base : 0.0f;
            }
          }
          m = base + (count ? m / (float)(count * (V - at.dup)) : 0.0f);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            if (r < count) {
#pragma unroll
              for (int k = 0; k < V; ++k) {
                const float d = !odd.value || k >= at.dup ? (float)x[r].v[k] - m : 0.0f;
                q = fmaf(d, d, q);
              }
            }
          }
        };
        if (s.a.channels % V == 0)  // no vector shares channels
          moments(std::false_type{});
        else
          moments(std::true_type{});
        if (at.active) lds[threadIdx.x] = {m, q};
      } else if (at.active) {
        const float share = count ? 1.0f / (float)count : 0.0f;
        float mean_of = 0.0f, sq_of = 0.0f;  // of a group's channels so far
        segments<V>(
            size, within, at.dup,
            [&](int k, int n) __attribute__((always_inline)) {
              const float base = (float)x[0].v[k];
              float m = 0.0f, q = 0.0f;
              if constexpr (R == 1) {
                m = base;
              } else {
#pragma unroll
                for (int r = 0; r < R; ++r) m += r < count ? (float)x[r].v[k] - base : 0.0f;
                m = fmaf(m, share, base);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                  const float d = r < count ? (float)x[r].v[k] - m : 0.0f;
                  q = fmaf(d, d, q);
                }
              }
              const float part = __builtin_amdgcn_rcpf((float)(n + 1));
              const float d = n ? m - mean_of : 0.0f;
              mean_of = n ? fmaf(d, part, mean_of) : m;
              sq_of = fmaf(d * d, (float)(n * count) * part, n ? sq_of + q : q);
            },
            [&](int t) __attribute__((always_inline)) {
              lds[t * e.plane + threadIdx.x] = {mean_of, sq_of};
            });
      }
      __syncthreads();
      const int pairs = s.at_a_time * s.a.groups;
      const int lane = threadIdx.x & (s.lanes - 1);
      const int teams = blockDim.x / s.lanes;
      for (int p0 = 0; p0 < pairs; p0 += teams) {
        const int p = p0 + threadIdx.x / s.lanes;
        const bool has = p < pairs;
        const int q = p / s.a.groups, g = p - q * s.a.groups;
        const float2* from = lds + q * at.slots * s.cv;
        // a lane's entries from the mean of its first one, then the lanes'
        float base = 0.0f, sum = 0.0f, sq = 0.0f, n = 0.0f;
        if (has)
          e.each_of(s, from, at.slots, lane, g, [&](float2 v, float c) __attribute__((always_inline)) {
            base = n == 0.0f ? v.x : base;
            const float d = v.x - base;
            sum = fmaf(c, d, sum);
            sq += fmaf(c * d, d, v.y);
            n += c;
          });
        float m = 0.0f;
        if (n > 0.0f) {
          const float d = sum * __builtin_amdgcn_rcpf(n);
          m = base + d;
          sq = fmaf(-sum, d, sq);
        }
        for (int o = s.lanes >> 1; o >= 1; o >>= 1) {
          const float n2 = __shfl_xor(n, o), m2 = __shfl_xor(m, o), sq2 = __shfl_xor(sq, o);
          if (n == 0.0f) m = m2;
          const float d = n2 == 0.0f ? 0.0f : m2 - m, part = n2 * __builtin_amdgcn_rcpf(n + n2);
          if (n2 > 0.0f) m = fmaf(d, part, m);
          sq += fmaf(d * d, n * (n2 > 0.0f ? part : 0.0f), sq2);
          n += n2;
        }
        if (has && lane == 0) {
          // (below 0 by rounding; NaN stays)
          const float2 r = {m, 1.0f / sqrtf(fmaf(sq < 0.0f ? 0.0f : sq, s.inv_m, s.a.eps))};
          group[p] = r;
          const int64_t to = batch * s.at_a_time + q;
          if (s.stats && to < s.a.samples) s.stats[to * s.all_groups + g] = r;
        }
      }
      __syncthreads();
      if (at.active)
        load_stats(size, group + at.sample * s.a.groups, first_group, within, mean, rstd);
    }
    if (in) {
      T* py = static_cast<T*>(s.out) + batch_offset(s, batch, s.ldo) + off_y;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r < count) {
          float xhat[V], z[V];
          normalise<K>(x[r], mean, rstd, w, b, xhat, z);
          act_values<K>(s.a.activation, z);
          store_raw<K>(py + (int64_t)r * at.slots * s.ldo, at.from, z);
        }
      }
    }
  };
  if constexpr (R == 1) {  // single rows: U batches at a time, the next ones loaded ahead
    constexpr int U = JOIN == LANES ? 2 : 1;
    const int64_t step = mine.step;
    Raw<K> ahead[U][R];
    int counts[U];
#pragma unroll
    for (int u = 0; u < U; ++u) counts[u] = load(mine.first + u * step, ahead[u]);
    for (int64_t batch = mine.first; batch < s.batches; batch += U * step) {
      Raw<K> x[U][R];
      int count[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[u][0] = ahead[u][0];
        count[u] = counts[u];
        counts[u] = load(batch + (U + u) * step, ahead[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) one(batch + u * step, x[u], count[u]);
    }
  } else {
    for (int64_t batch = mine.first; batch < s.batches; batch += mine.step) {
      Raw<K> x[R];
      const int count = load(batch, x);
      one(batch, x, count);
    }
  }
}

// dz of one vector, and what z it had: xhat.
template <class K, int MV>
__device__ __forceinline__ void vector_dz(const GroupArgs& a, const Raw<K>& x, const Raw<K>& dy,
                                          const float (&mean)[MV], const float (&rstd)[MV],
                                          const float* w, const float* b, float* xhat, float* dz) {
  constexpr int V = K::V;
  float z[V];
  normalise<K>(x, mean, rstd, w, b, xhat, z);
  act_slopes<K>(a.activation, z, dz);
#pragma unroll
  for (int k = 0; k < V; ++k) dz[k] *= (float)dy.v[k];
}

// part[block][channels]: sums of dz and dz xhat over the block's samples.
template <class K, int R, int JOIN>
__global__ __launch_bounds__(kMostThreads)
    __attribute__((amdgpu_waves_per_eu(R == 1 && kStats<K, JOIN> == 1 ? 4 : 2))) void k_group_bwd(GroupKernel s) {
  using T = typename K::T;
  constexpr int V = K::V;
  extern __shared__ float2 lds[];
  const Share mine = share_of<T>(s);
  const Place<K> at(s);
  const int size = s.a.channels / s.a.groups;
  float w[V], b[V], sum_a[V], sum_b[V];
  load_params<K>(s.a.weight, at.col, s.a.f32_params, 1.0f, w);
  load_params<K>(s.a.bias, at.col, s.a.f32_params, 0.0f, b);
#pragma unroll
  for (int k = 0; k < V; ++k) sum_a[k] = sum_b[k] = 0.0f;
  constexpr int MV = kStats<K, JOIN>;
  struct Rows {
    Raw<K> x[R], dy[R];
    float mean[MV], rstd[MV];
    int count;
  };
  const int64_t off_x = at.offset(s, s.a.x_stride), off_d = at.offset(s, s.ldy),
                off_o = at.offset(s, s.ldo);
  const int group = at.col / size, within = at.col - group * size;
  const Entries<K, JOIN> e(s, size, at.slots);
  auto load = [&](int64_t batch, Rows& v) __attribute__((always_inline)) {
    const T* px = static_cast<const T*>(s.a.x) + batch_offset(s, batch, s.a.x_stride) + off_x;
    const T* pd = static_cast<const T*>(s.dy) + batch_offset(s, batch, s.ldy) + off_d;
    v.count = at.count(s, batch);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r < v.count) {
        v.x[r] = load_raw<K>(px + (int64_t)r * at.slots * s.a.x_stride);
        v.dy[r] = load_raw<K>(pd + (int64_t)r * at.slots * s.ldy);
      }
    }
    if (v.count > 0)
      load_stats(size, s.stats + (batch * s.at_a_time + at.sample) * s.all_groups, group, within,
                 v.mean, v.rstd);
  };
  Rows ahead;  // single rows: the next ones are loaded ahead
  if constexpr (R == 1) load(mine.first, ahead);
  for (int64_t batch = mine.first; batch < s.batches; batch += mine.step) {
    Rows now;
    if constexpr (R == 1) {
      now = ahead;
      load(batch + mine.step, ahead);
    } else {
      load(batch, now);
    }
    const auto &x = now.x, &dy = now.dy;
    const auto &mean = now.mean, &rstd = now.rstd;
    const int count = now.count;
    const bool in = count > 0;
    float t1[MV], t2[MV];   // the sample's group sums
    float xhat[V], dz[V];   // single rows keep them, dz times the weight
#pragma unroll
    for (int k = 0; k < MV; ++k) t1[k] = t2[k] = 0.0f;
    if constexpr (R == 1) {
      if (in) {
        vector_dz<K>(s.a, x[0], dy[0], mean, rstd, w, b, xhat, dz);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          sum_a[k] += dz[k];
          sum_b[k] = fmaf(dz[k], xhat[k], sum_b[k]);
          dz[k] *= w[k];
          const float g = JOIN != VECTORS || k >= at.dup ? dz[k] : 0.0f;
          t1[k % MV] += g;
          t2[k % MV] = fmaf(g, xhat[k], t2[k % MV]);
        }
      }
    } else {
      float a1[V], a2[V];
#pragma unroll
      for (int k = 0; k < V; ++k) a1[k] = a2[k] = 0.0f;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r < count) {
          vector_dz<K>(s.a, x[r], dy[r], mean, rstd, w, b, xhat, dz);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            a1[k] += dz[k];
            a2[k] = fmaf(dz[k], xhat[k], a2[k]);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        sum_a[k] += a1[k];
        sum_b[k] += a2[k];
        const float g = JOIN != VECTORS || k >= at.dup ? w[k] : 0.0f;
        t1[k % MV] = fmaf(a1[k], g, t1[k % MV]);
        t2[k % MV] = fmaf(a2[k], g, t2[k % MV]);
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
      float2* sums = lds + e.all;
      if (at.active) {
        if constexpr (JOIN == VECTORS) {
          lds[threadIdx.x] = {t1[0], t2[0]};
        } else {
          float2 sum = {0.0f, 0.0f};
          segments<V>(
              size, within, at.dup,
              [&](int k, int n) __attribute__((always_inline)) {
                sum.x = n ? sum.x + t1[k] : t1[k];
                sum.y = n ? sum.y + t2[k] : t2[k];
              },
              [&](int t) __attribute__((always_inline)) { lds[t * e.plane + threadIdx.x] = sum; });
        }
      }
      __syncthreads();
      const int pairs = s.at_a_time * s.a.groups;
      const int lane = threadIdx.x & (s.lanes - 1);
      const int teams = blockDim.x / s.lanes;
      for (int p0 = 0; p0 < pairs; p0 += teams) {
        const int p = p0 + threadIdx.x / s.lanes;
        const int q = p / s.a.groups, g = p - q * s.a.groups;
        float2 t = {0.0f, 0.0f};
        if (p < pairs)
          e.each_of(s, lds + q * at.slots * s.cv, at.slots, lane, g,
                    [&](float2 v, float) __attribute__((always_inline)) {
                      t.x += v.x;
                      t.y += v.y;
                    });
        t.x = lane_sum(t.x, s.lanes);
        t.y = lane_sum(t.y, s.lanes);
        if (p < pairs && lane == 0) sums[p] = t;
      }
      __syncthreads();
      if (at.active) load_stats(size, sums + at.sample * s.a.groups, group, within, t1, t2);
    }
    if (in) {
      T* po = static_cast<T*>(s.out) + batch_offset(s, batch, s.ldo) + off_o;
#pragma unroll
      for (int k = 0; k < MV; ++k) {
        t1[k] *= s.inv_m * rstd[k];
        t2[k] *= s.inv_m * rstd[k];
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r < count) {
          if constexpr (R > 1) vector_dz<K>(s.a, x[r], dy[r], mean, rstd, w, b, xhat, dz);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const float g = R > 1 ? dz[k] * w[k] : dz[k];
            dz[k] = fmaf(g, rstd[k % MV], -fmaf(xhat[k], t2[k % MV], t1[k % MV]));
          }
          store_raw<K>(po + (int64_t)r * at.slots * s.ldo, at.from, dz);
        }
      }
    }
    if constexpr (JOIN == SEGMENTS || JOIN == VECTORS) __syncthreads();
  }
  if (s.part == nullptr) return;
  // the slots' sums of each channel
  const int width = s.cv * V, taken = at.slots * s.at_a_time;
  if (at.active) {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k >= at.dup) lds[at.slot * width + at.col + k] = {sum_a[k], sum_b[k]};
  }
  __syncthreads();
  for (int c = threadIdx.x; c < s.a.channels; c += blockDim.x) {
    float2 t = lds[c];
    for (int q = 1; q < taken; ++q) {
      const float2 v = lds[q * width + c];
      t.x += v.x;
      t.y += v.y;
    }
    s.part[(s.group_blocks == 1 ? (int64_t)blockIdx.x * s.all_channels : 0) + c] = t;
  }
}

// ---------------------------------------------------------------- samples in stretches

constexpr int kPartThreads = 256;

// A stretch of rows of a sample, in one block of columns.
template <class K, bool APPLY>
struct Piece : Columns<K> {
  int chunk, slots, slot, base, cv;  // rows at a time; base, cv: first channel, vectors of the block
  int row0, rows;                    // first row within the sample
  bool active;
  static __device__ __forceinline__ int vectors(const GroupKernel& s, int block) {
    return min(s.cv, (s.a.channels + K::V - 1) / K::V - block * s.cv);
  }
  __device__ __forceinline__ Piece(const GroupKernel& s, int block)
      : Columns<K>(s, block * s.cv * K::V, (int)threadIdx.x % vectors(s, block)) {
    chunk = s.blocks == 1 ? (int)blockIdx.x : (int)(blockIdx.x / s.blocks);
    const int stretch = APPLY ? s.short_stretch : s.stretch;
    row0 = chunk * stretch;
    rows = min(stretch, (int)s.a.positions - row0);
    base = block * s.cv * K::V;
    cv = vectors(s, block);
    slots = kPartThreads / cv;
    slot = threadIdx.x / cv;
    active = slot < slots;
  }
  __device__ __forceinline__ int count_of(int slot_) const {  // its rows
    return rows > slot_ ? (rows - slot_ + slots - 1) / slots : 0;
  }
};

// U rows of a thread at a time, the next ones loaded ahead.  Rows past the last are
// read as the last.
template <class K, int U, bool BACK>
struct Stream {
  using T = typename K::T;
  const T *px, *pd;
  int64_t sx, sd;
  int last;
  Raw<K> x[U], dy[BACK ? U : 1];
  __device__ __forceinline__ void load(int i) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = min(i + u, last);
      x[u] = load_raw<K>(px + r * sx);
      if constexpr (BACK) dy[u] = load_raw<K>(pd + r * sd);
    }
  }
  // of the `count` > 0 rows of sample n
  template <class P>
  __device__ __forceinline__ Stream(const GroupKernel& s, const P& at, int64_t n, int count)
      : sx((int64_t)at.slots * s.a.x_stride), sd((int64_t)at.slots * s.ldy), last(count - 1) {
    const int64_t row = n * s.a.positions + at.row0 + at.slot;
    px = static_cast<const T*>(s.a.x) + row * s.a.x_stride + at.col;
    pd = BACK ? static_cast<const T*>(s.dy) + row * s.ldy + at.col : nullptr;
    load(0);
  }
};

// part[sample][stretch][channels]: mean and centred squares of a channel; BACK: its
// sums of dz and dz xhat.
template <class K, bool BACK, int MV>
__global__ __launch_bounds__(kPartThreads) void k_group_part(GroupKernel s) {
  constexpr int V = K::V, U = BACK ? 2 : 4;
  __shared__ float2 lds[kPartThreads * V];
  const Piece<K, false> at(s, s.blocks == 1 ? 0 : (int)(blockIdx.x % s.blocks));
  const int count = at.active ? at.count_of(at.slot) : 0;
  float w[V], b[V];
  if constexpr (BACK) {
    load_params<K>(s.a.weight, at.col, s.a.f32_params, 1.0f, w);
    load_params<K>(s.a.bias, at.col, s.a.f32_params, 0.0f, b);
  }
  for (int64_t n = blockIdx.y; n < s.a.samples; n += gridDim.y) {
    float m[V], q[V];  // or the two sums
#pragma unroll
    for (int k = 0; k < V; ++k) m[k] = q[k] = 0.0f;
    if (count > 0) {
      Stream<K, U, BACK> rows(s, at, n, count);
      if constexpr (!BACK) {
        const Raw<K> base = rows.x[0];  // means are formed from here
        int done = 0;
        for (; done + U <= count; done += U) {
          Raw<K> x[U];
#pragma unroll
          for (int u = 0; u < U; ++u) x[u] = rows.x[u];
          rows.load(done + U);
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
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (done + u < count) {
            const float n1 = (float)(done + u), share = 1.0f / (n1 + 1.0f);
#pragma unroll
            for (int k = 0; k < V; ++k) {
              const float d = ((float)rows.x[u].v[k] - (float)base.v[k]) - m[k];
              m[k] = fmaf(d, share, m[k]);
              q[k] = fmaf(d * d, n1 * share, q[k]);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < V; ++k) m[k] += (float)base.v[k];
      } else {
        float mean[MV], rstd[MV];
        const int size = s.a.channels / s.a.groups, g = at.col / size;
        load_stats(size, s.stats + n * s.a.groups, g, at.col - g * size, mean, rstd);
        auto add = [&](const Raw<K>& x, const Raw<K>& dy) __attribute__((always_inline)) {
          float xhat[V], dz[V];
          vector_dz<K>(s.a, x, dy, mean, rstd, w, b, xhat, dz);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            m[k] += dz[k];
            q[k] = fmaf(dz[k], xhat[k], q[k]);
          }
        };
        for (int done = 0; done < count; done += U) {
          Raw<K> x[U], dy[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            x[u] = rows.x[u];
            dy[u] = rows.dy[u];
          }
          rows.load(done + U);
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (done + u < count) add(x[u], dy[u]);
        }
      }
    }
    const int width = at.cv * V;
    if (at.active) {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (k >= at.dup) lds[at.slot * width + at.col - at.base + k] = {m[k], q[k]};
    }
    __syncthreads();
    float2* to = s.part + (n * s.stretches + at.chunk) * s.a.channels + at.base;
    const int used = min(at.slots, at.rows);
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
        const int more = at.rows - at.rows / at.slots * at.slots;
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

__device__ __forceinline__ float block_sum(float v, float* red) {
  v = lane_sum(v, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// A workgroup a group: its mean and rstd, or (BACK) the two sums over m.  The first
// 2048 partial results stay in registers between the two sweeps.
template <class T, bool BACK>
__global__ __launch_bounds__(256) void k_group_merge(GroupKernel s) {
  constexpr int KEPT = 8;
  __shared__ float red[4];
  const int size = s.a.channels / s.a.groups;
  const int64_t pairs = s.a.samples * s.a.groups;
  const int64_t all = (int64_t)s.stretches * size;
  for (int64_t p = blockIdx.x; p < pairs; p += gridDim.x) {
    const int64_t n = p / s.a.groups;
    const int g = (int)(p - n * s.a.groups);
    const float2* from = s.part + n * s.stretches * s.a.channels + (int64_t)g * size;
    struct Entry {
      float2 v;
      float by;  // its rows, or its channel's weight
    };
    auto entry = [&](int64_t i) __attribute__((always_inline)) {
      Entry e{{0.0f, 0.0f}, 0.0f};
      if (i < all) {
        const int chunk = (int)(i / size), d = (int)(i - (int64_t)chunk * size), c = g * size + d;
        e.v = from[(int64_t)chunk * s.a.channels + d];
        if constexpr (BACK)
          e.by = s.a.weight == nullptr ? 1.0f
                 : s.a.f32_params      ? static_cast<const float*>(s.a.weight)[c]
                                       : (float)static_cast<const T*>(s.a.weight)[c];
        else
          e.by = (float)min(s.stretch, (int)s.a.positions - chunk * s.stretch);
      }
      return e;
    };
    Entry kept[KEPT];
#pragma unroll
    for (int k = 0; k < KEPT; ++k) kept[k] = entry(threadIdx.x + 256 * k);
    auto sweep = [&](auto f) __attribute__((always_inline)) {
      float t = 0.0f;
#pragma unroll
      for (int k = 0; k < KEPT; ++k) t += f(kept[k]);
      for (int64_t i = threadIdx.x + 256 * KEPT; i < all; i += 256) t += f(entry(i));
      return block_sum(t, red);
    };
    if constexpr (!BACK) {
      const float base = from[0].x;
      const float m = fmaf(sweep([&](const Entry& e) { return (e.v.x - base) * e.by; }), s.inv_m,
                           base);
      const float var = sweep([&](const Entry& e) {
                          return fmaf(e.by * (e.v.x - m), e.v.x - m, e.v.y);
                        }) * s.inv_m;
      if (threadIdx.x == 0) s.stats[p] = {m, 1.0f / sqrtf(var + s.a.eps)};
    } else {
      const float t1 = sweep([](const Entry& e) { return e.v.x * e.by; });
      const float t2 = sweep([](const Entry& e) { return e.v.y * e.by; });
      if (threadIdx.x == 0) s.coef[p] = {t1 * s.inv_m, t2 * s.inv_m};
    }
  }
}

// y, or (BACK) dx, of a stretch.
template <class K, bool BACK, int MV>
__global__ __launch_bounds__(kPartThreads) void k_group_apply(GroupKernel s) {
  using T = typename K::T;
  constexpr int V = K::V, U = BACK ? 2 : 4;
  const Piece<K, true> at(s, s.blocks == 1 ? 0 : (int)(blockIdx.x % s.blocks));
  const int count = at.active ? at.count_of(at.slot) : 0;
  if (count == 0) return;
  const int64_t so = (int64_t)at.slots * s.ldo;
  const int size = s.a.channels / s.a.groups, g = at.col / size;
  float w[V], b[V];
  load_params<K>(s.a.weight, at.col, s.a.f32_params, 1.0f, w);
  load_params<K>(s.a.bias, at.col, s.a.f32_params, 0.0f, b);
  for (int64_t n = blockIdx.y; n < s.a.samples; n += gridDim.y) {
    Stream<K, U, BACK> rows(s, at, n, count);
    T* po = static_cast<T*>(s.out) + (n * s.a.positions + at.row0 + at.slot) * s.ldo + at.col;
    float mean[MV], rstd[MV], c1[MV], c2[MV];
    load_stats(size, s.stats + n * s.a.groups, g, at.col - g * size, mean, rstd);
    float wr[V];
    if constexpr (BACK) {
      load_stats(size, s.coef + n * s.a.groups, g, at.col - g * size, c1, c2);
#pragma unroll
      for (int k = 0; k < MV; ++k) {
        c1[k] *= rstd[k];
        c2[k] *= rstd[k];
      }
#pragma unroll
      for (int k = 0; k < V; ++k) wr[k] = w[k] * rstd[k % MV];
    }
    for (int i = 0; i < count; i += U) {
      Raw<K> x[U], dy[BACK ? U : 1];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[u] = rows.x[u];
        if constexpr (BACK) dy[u] = rows.dy[u];
      }
      rows.load(i + U);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u >= count) continue;
        float xhat[V], z[V];
        if constexpr (BACK) {
          vector_dz<K>(s.a, x[u], dy[u], mean, rstd, w, b, xhat, z);
#pragma unroll
          for (int k = 0; k < V; ++k)
            z[k] = fmaf(wr[k], z[k], -fmaf(xhat[k], c2[k % MV], c1[k % MV]));
        } else {
          normalise<K>(x[u], mean, rstd, w, b, xhat, z);
          act_values<K>(s.a.activation, z);
        }
        store_raw<K>(po + (i + u) * so, at.from, z);
      }
    }
  }
}

// dweight, dbias: sums of the partial results in a fixed order, kParamChannels channels
// (64 bytes of partial results) a workgroup.
constexpr int kParamChannels = 8;
template <class P>
__global__ __launch_bounds__(1024) void k_group_params(const float2* __restrict__ part,
                                                       int64_t parts, int channels,
                                                       P* __restrict__ dweight,
                                                       P* __restrict__ dbias) {
  __shared__ float2 red[1024 / kParamChannels][kParamChannels];
  constexpr int LINES = 1024 / kParamChannels;
  const int c = threadIdx.x % kParamChannels, line = threadIdx.x / kParamChannels;
  const int channel = blockIdx.x * kParamChannels + c;
  float2 t = {0.0f, 0.0f};
  if (channel < channels) {
#pragma unroll 8
    for (int64_t p = line; p < parts; p += LINES) {
      const float2 v = part[p * channels + channel];
      t.x += v.x;
      t.y += v.y;
    }
  }
  red[line][c] = t;
  __syncthreads();
  for (int o = LINES / 2; o >= 1; o >>= 1) {
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

constexpr int kForwardRows = 16, kBackRows = 8;  // of a thread, in registers
constexpr int64_t kBackBlocks = 1024;  // partial results of whole samples, at most
constexpr int64_t kStretches = 1024;    // workgroups of samples in stretches

struct GroupCut {
  bool whole;  // samples in a workgroup's registers
  int join = SEGMENTS, r = 1, threads = 256;
  size_t lds = 0;
};

// Channels of a thread: 16 bytes, or one in rows that have fewer.
inline int lane_channels(const GroupArgs& a) {
  const int v = a.type == ELEM_F32 ? 4 : 8;
  return a.channels < v ? 1 : v;
}

inline int pow2_at_most(int64_t v) {
  int p = 1;
  while (2 * (int64_t)p <= v) p *= 2;
  return p;
}

// Threads of a workgroup that holds `cv` vectors of `positions` rows, or 0.  256 of them up
// to 8 rows a thread: two such workgroups on a CU overlap where one of 512 threads would
// wait (4000 x 16 x 1024 bf16, forward and backward 231 us; by 512 threads of 4 rows
// 259).
inline int threads_of(int64_t cv, int64_t positions, int most) {
  int threads = 256;
  while (threads < kMostThreads && (cv > threads || ceil_div(positions, threads / cv) > 8))
    threads *= 2;
  return cv <= threads && ceil_div(positions, threads / cv) <= most ? threads : 0;
}

// Groups a workgroup takes of a sample (a divisor of them), 0: none fit.  All of a
// small sample's; otherwise as many as leave every CU a workgroup, in rows of 512 bytes
// at least: narrower ones read memory in parts of lines (32 x 4096 x 512 bf16, forward,
// by single groups of 32 bytes a row 147 us, in stretches of whole rows 97; 2417 x 1 x
// 3776 fp32, 7.5 KB a row 55 us, in stretches 268).
inline int groups_of(const GroupArgs& a, int V, int size, int most) {
  const int64_t row = size * (int64_t)elem_bytes(a.type);
  const bool small = a.positions * a.groups * row <= 32768;
  int best = 0;
  // (more than the threads' vectors hold never fit)
  for (int gb = std::min(a.groups, std::max(1, kMostThreads * V / size)); gb >= 1; --gb) {
    if (a.groups % gb != 0) continue;
    if (!threads_of(ceil_div((int64_t)gb * size, (int64_t)V), a.positions, most)) continue;
    if (gb < a.groups && (gb * size < V || gb * row < 512)) break;  // (rows hold a vector)
    best = gb;
    if (small || a.samples * (a.groups / gb) >= 256) break;
  }
  return best;
}

// Fills in how the call is cut.
GroupCut cut_of(GroupKernel& s, bool back) {
  const int64_t L = s.a.positions;
  const int V = lane_channels(s.a), size = s.a.channels / s.a.groups;
  s.inv_m = (float)(1.0 / ((double)L * size));
  s.all_groups = s.a.groups;
  s.all_channels = s.a.channels;
  GroupCut c{};
  const int most = back ? kBackRows : kForwardRows, gb = groups_of(s.a, V, size, most);
  c.whole = gb > 0;
  if (!c.whole) {
    const GroupArgs& a = s.a;
    const int64_t cv = ceil_div((int64_t)a.channels, (int64_t)V);
    s.blocks = (int)ceil_div(cv, (int64_t)kPartThreads);
    s.cv = (int)ceil_div(cv, (int64_t)s.blocks);
    s.blocks = (int)ceil_div(cv, (int64_t)s.cv);
    // about four workgroups a CU, each thread at least eight rows
    const int64_t slots = std::max<int64_t>(1, kPartThreads / s.cv);
    const int64_t want = ceil_div((int64_t)kStretches, a.samples * s.blocks);
    s.stretches = (int)std::max<int64_t>(1, std::min(want, L / (8 * slots)));
    s.stretch = (int)ceil_div(L, (int64_t)s.stretches);
    s.stretches = (int)ceil_div(L, (int64_t)s.stretch);
    // the results', which leave no partial ones behind: more of them, of four rows a thread
    const int64_t more = std::max<int64_t>(1, std::min(2 * want, L / (4 * slots)));
    s.short_stretch = (int)ceil_div(L, more);
    s.shorts = (int)ceil_div(L, (int64_t)s.short_stretch);
    return c;
  }
  s.group_blocks = s.a.groups / gb;
  s.a.groups = gb;
  s.a.channels = gb * size;
  const GroupArgs& a = s.a;
  const int64_t cv = ceil_div((int64_t)a.channels, (int64_t)V);
  const int threads = threads_of(cv, L, most);
  s.cv = (int)cv;
  // as many rows a thread in every slot, and no waves without rows
  const int64_t r = ceil_div(L, (int64_t)(threads / s.cv));
  s.slots = (int)ceil_div(L, r);
  s.at_a_time = s.group_blocks > 1 ? 1 : threads / s.cv / s.slots;
  s.batches = ceil_div(a.samples, (int64_t)s.at_a_time);
  const int slots = s.slots, taken = slots * s.at_a_time;
  c.threads = (int)round_up(taken * s.cv, 64);
  c.r = r <= 1 ? 1 : r <= 2 ? 2 : r <= 4 ? 4 : r <= 8 ? 8 : 16;
  const bool pow2 = (size & (size - 1)) == 0;
  if (L == 1 && pow2 && size < V) {
    c.join = THREAD;
    s.lanes = 1;
  } else if (L == 1 && pow2 && size / V <= 64) {
    c.join = LANES;
    s.lanes = size / V;
  } else {
    c.join = size % V == 0 || gb == 1 ? VECTORS : SEGMENTS;
    const int run = vectors_of(c.join, V, size);
    const int64_t pairs = (int64_t)s.at_a_time * a.groups;
    s.lanes = std::min({64, pow2_at_most(2 * (int64_t)slots * run - 1),
                        pow2_at_most(std::max<int64_t>(1, c.threads / pairs))});
    // the fewest rounds over a pair's entries
    int fewest = 0;
    for (int on = s.lanes; on >= 1; on /= 2) {
      const int rounds = ceil_div(slots, s.lanes / on) * ceil_div(run, on);
      if (fewest == 0 || rounds < fewest) {
        fewest = rounds;
        s.run_lanes = on;
      }
    }
    const int each = c.join == VECTORS ? 1 : most_groups(V, size);
    c.lds = ((size_t)plane_of(taken * s.cv) * each + (size_t)pairs) * sizeof(float2);
  }
  if (back) c.lds = std::max(c.lds, (size_t)taken * s.cv * V * sizeof(float2));
  return c;
}

// Workgroups that share the samples out among them, for each block of groups: of the
// backward pass, also the rows of partial results.  (Blocks, forward: as many as samples
// up to 2^20 workgroups, which start as others end.)
inline int64_t sharers(const GroupKernel& s, bool back) {
  const int64_t most = back                   ? kBackBlocks
                       : s.group_blocks > 1 ? (int64_t)1 << 20
                                              : 2048;
  return std::min<int64_t>(s.batches, std::max<int64_t>(1, most / s.group_blocks));
}
inline unsigned workgroups(const GroupKernel& s, bool back) {
  return (unsigned)(sharers(s, back) * s.group_blocks);
}

// Runs f with a kernel's rows a thread and join.
template <class K, bool BACK, class F>
void dispatch_whole(const GroupCut& c, F&& f) {
  using std::integral_constant;
  auto with = [&](auto r) {
    if constexpr (K::V > 1) {  // (of one channel a thread, channels are vectors)
      if (c.join == SEGMENTS) return f(r, integral_constant<int, SEGMENTS>{});
    }
    f(r, integral_constant<int, VECTORS>{});
  };
  if constexpr (K::V > 1) {
    if (c.join == THREAD) return f(integral_constant<int, 1>{}, integral_constant<int, THREAD>{});
  }
  if (c.join == LANES) return f(integral_constant<int, 1>{}, integral_constant<int, LANES>{});
  if (c.r == 1) return with(integral_constant<int, 1>{});
  if (c.r == 2) return with(integral_constant<int, 2>{});
  if (c.r == 4) return with(integral_constant<int, 4>{});
  if (c.r == 8) return with(integral_constant<int, 8>{});
  if constexpr (!BACK) with(integral_constant<int, 16>{});
}

// Runs f with the call's Kind.
template <class F>
void dispatch_kind(const GroupArgs& a, F&& f) {
  dispatch_elem(a.type, [&](auto tag) {
    using T = decltype(tag);
    if (lane_channels(a) == 1)
      f(Kind<T, 1>{});
    else
      f(Kind<T, Vec16<T>::N>{});
  });
}

template <class K, bool BACK>
void launch_stretches(GroupKernel& s, hipStream_t st) {
  auto grid = [&](int stretches) {
    const int x = stretches * s.blocks;
    return dim3((unsigned)x, (unsigned)std::min<int64_t>(s.a.samples, std::max(1, (1 << 15) / x)));
  };
  const unsigned pairs = (unsigned)std::min<int64_t>(s.a.samples * s.a.groups, 1 << 16);
  auto go = [&](auto mv) {
    k_group_part<K, BACK, mv.value><<<grid(s.stretches), kPartThreads, 0, st>>>(s);
    if (BACK && s.out == nullptr) return;
    k_group_merge<typename K::T, BACK><<<pairs, 256, 0, st>>>(s);
    k_group_apply<K, BACK, mv.value><<<grid(s.shorts), kPartThreads, 0, st>>>(s);
  };
  if (s.a.channels / s.a.groups % K::V == 0)  // a vector's channels are of one group
    go(std::integral_constant<int, 1>{});
  else
    go(std::integral_constant<int, K::V>{});
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
  const GroupCut c = cut_of(s, back);
  const size_t row = (size_t)a.channels * sizeof(float2);
  if (c.whole) return back ? aligned((size_t)sharers(s, true) * row) : 0;
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
  s.apart = y != a.x;
  const GroupCut c = cut_of(s, false);
  dispatch_kind(a, [&](auto kind) {
    using K = decltype(kind);
    if (!c.whole) {
      s.part = static_cast<float2*>(ws);
      if (!stats)
        s.stats = s.part + aligned((size_t)(a.samples * s.stretches) * a.channels * sizeof(float2)) /
                               sizeof(float2);
      launch_stretches<K, false>(s, st);
      return;
    }
    dispatch_whole<K, false>(c, [&](auto r, auto join) {
      k_group_fwd<K, r.value, join.value><<<workgroups(s, false), c.threads, c.lds, st>>>(s);
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
  s.apart = dx != a.x && dx != dy;
  const bool params = dweight || dbias;
  int64_t parts = 0;
  if (a.samples * a.positions > 0) {
    const GroupCut c = cut_of(s, true);
    dispatch_kind(a, [&](auto kind) {
      using K = decltype(kind);
      s.part = static_cast<float2*>(ws);
      if (!c.whole) {
        parts = a.samples * s.stretches;
        s.coef = s.part + aligned((size_t)parts * a.channels * sizeof(float2)) / sizeof(float2);
        launch_stretches<K, true>(s, st);
        return;
      }
      parts = sharers(s, true);
      if (!params) s.part = nullptr;
      dispatch_whole<K, true>(c, [&](auto r, auto join) {
        k_group_bwd<K, r.value, join.value><<<workgroups(s, true), c.threads, c.lds, st>>>(s);
      });
    });
  }
  if (params) {
    const unsigned grid = (unsigned)ceil_div((int64_t)a.channels, (int64_t)kParamChannels);
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
