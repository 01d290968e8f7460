// Group norm with an activation on channels-last data (batch, positions, channels), forward and backward.
//
//   xhat = (x - mean) rstd over the positions and the channels of a group, z = xhat w + b, y = act(z)
//   dz = dy act'(z), db = sum dz, dw = sum dz xhat, dx = rstd (dz w - mean(dz w) - xhat mean(dz w xhat))
//
// Memory bound: forward x and y once, backward x, dy and dx once is the floor.  Three ways, by what of a sample fits where:
// a team of lanes (norm_rows), a workgroup's registers (norm_tile), or several passes over memory.  Statistics are fp32 (mean, sum of squared
// deviations) pairs that are merged, never a difference of sums of squares.  With lengths, positions at and past
// lengths[n] * inner are padding: not read, zeros in y and dx.
#include "model_ops.h"
#include "activations.h"

#include <algorithm>
#include <type_traits>

namespace tfa {

// a vector as it lies in memory, so that one waits in registers at its own size
template <typename T, int V>
struct __attribute__((aligned(V * sizeof(T)))) Raw {
  unsigned w[V * sizeof(T) / 4];
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    const unsigned u = w[i / 2];
    if constexpr (std::is_same_v<T, __bf16>)
      return __uint_as_float(i % 2 ? u & 0xffff0000u : u << 16);
    else
      return (float)__builtin_bit_cast(_Float16, (unsigned short)(i % 2 ? u >> 16 : u));
  }
};

// (past the caches where these may still hold what the next rows' loads want)
template <typename T, int V>
__device__ __forceinline__ void stream_pack(T* p, const float (&x)[V]) {
  if constexpr (V * sizeof(T) == 16) {
    typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
    Pack<T, V> u;
#pragma unroll
    for (int i = 0; i < V; ++i) u.v[i] = from_f32<T>(x[i]);
    __builtin_nontemporal_store(__builtin_bit_cast(uintx4, u), reinterpret_cast<uintx4*>(p));
  } else {
    store_pack<T, V>(p, x);
  }
}

__device__ __forceinline__ long long live_positions(const NormArgs& a, long long n) {
  if (!a.lengths) return a.positions;
  return min(max(a.lengths[n], 0LL), a.positions / a.inner) * a.inner;
}

// (mean, M2, count) of two sets joined
__device__ __forceinline__ void merge(float& mean, float& m2, float& count, float mean_b, float m2_b, float count_b) {
  const float total = count + count_b;
  if (count_b == 0.0f) return;
  const float d = mean_b - mean, f = count_b / total;
  mean = __builtin_fmaf(d, f, mean);
  m2 += m2_b + d * d * count * f;
  count = total;
}

// Passes over memory: statistics, join, result; backward sums, join, weights' gradients, result.  A workgroup takes rows [r0, r1) of one
// sample and up to 256 vectors of V channels (V = 16 bytes, or 1 where the channels are no multiple of that); a thread keeps its
// channels over its rows, `lanes` apart.  32 x 160882 x 32 (330 MB of bf16, more than the caches hold): statistics
// 69 us, 4.8 TB/s, result 140 us, 4.7 TB/s; a large copy reaches 5.0.
constexpr int kNormThreads = 256;
struct Slab {
  int col, lane, lanes;  // first channel of the thread's vector, row lane, row lanes
  bool on;
};
template <int V>
__device__ __forceinline__ Slab slab_of(int channels) {
  const int vecs = channels / V, tile = min(vecs - (int)blockIdx.z * kNormThreads, kNormThreads);
  Slab s;
  s.lanes = kNormThreads / tile;
  s.lane = threadIdx.x / tile;
  s.col = ((int)blockIdx.z * kNormThreads + threadIdx.x % tile) * V;
  s.on = s.lane < s.lanes;
  return s;
}

// partial (mean, M2) of each channel over the workgroup's rows: part[((n * splits + split) * 2 + {0, 1}) * channels + c]
template <typename T, int V>
__global__ __launch_bounds__(kNormThreads) void norm_stats_kernel(NormArgs a, long long rows_each, unsigned splits) {
  __shared__ float red[3][kNormThreads * V];
  const Slab s = slab_of<V>(a.channels);
  const long long n = blockIdx.x / splits, live = live_positions(a, n);
  const long long r0 = (blockIdx.x % splits) * rows_each, r1 = min(r0 + rows_each, live);
  const T* x = static_cast<const T*>(a.x) + n * a.positions * a.channels + s.col;
  float mean[V] = {}, m2[V] = {}, count = 0.0f;
  constexpr int U = 8;
  if (s.on)
    for (long long r = r0 + s.lane; r < r1; r += (long long)U * s.lanes) {
      float v[U][V];
      const bool whole = r + (long long)(U - 1) * s.lanes < r1;
      const int full = whole ? U : (int)((r1 - r + s.lanes - 1) / s.lanes);
      if (whole) {
#pragma unroll
        for (int u = 0; u < U; ++u) load_pack<T, V>(x + (r + (long long)u * s.lanes) * a.channels, v[u]);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int i = 0; i < V; ++i) v[u][i] = 0.0f;
          if (u < full) load_pack<T, V>(x + (r + (long long)u * s.lanes) * a.channels, v[u]);
        }
      }
      const float inv = 1.0f / (float)full, f = (float)full / (count + (float)full);
      auto add = [&](auto all) {
        constexpr bool ALL = decltype(all)::value;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float sum = 0.0f, sq = 0.0f;
#pragma unroll
          for (int u = 0; u < U; ++u) sum += v[u][i];
          sum *= inv;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const float d = ALL || u < full ? v[u][i] - sum : 0.0f;
            sq = __builtin_fmaf(d, d, sq);
          }
          const float d = sum - mean[i];
          mean[i] = __builtin_fmaf(d, f, mean[i]);
          m2[i] += sq + d * d * count * f;
        }
      };
      if (whole)
        add(std::true_type{});
      else
        add(std::false_type{});
      count += (float)full;
    }
  if (s.on)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      red[0][threadIdx.x * V + i] = mean[i];
      red[1][threadIdx.x * V + i] = m2[i];
      red[2][threadIdx.x * V + i] = count;
    }
  __syncthreads();
  const int vecs = a.channels / V, width = min(vecs - (int)blockIdx.z * kNormThreads, kNormThreads) * V;
  float* out = a.ws + (size_t)blockIdx.x * 2 * a.channels + (size_t)blockIdx.z * kNormThreads * V;
  for (int c = threadIdx.x; c < width; c += kNormThreads) {
    float mm = 0.0f, mq = 0.0f, mc = 0.0f;
    for (int l = 0; l < s.lanes; ++l) merge(mm, mq, mc, red[0][l * width + c], red[1][l * width + c], red[2][l * width + c]);
    out[c] = mm;
    out[a.channels + c] = mq;
  }
}

__device__ __forceinline__ float rows_of(long long split, long long rows_each, long long live) {
  return (float)max(0LL, min(rows_each, live - split * rows_each));
}

// Joins the partials of one (sample, group).  A wave takes them where they are few; else 1024 threads, several splits on their way
// each: 1 x 160882 x 32 in 8 groups, 8 joins of 4096 partials, 30 us, with a wave each 38 (more with more splits); 64 x 2000 x 512 in 32
// groups, 2048 joins of 256 partials, 80 us, with 1024 threads each 88.
constexpr int kJoinFew = 512;
template <int THREADS>
__global__ __launch_bounds__(THREADS) void norm_join_kernel(NormArgs a, int splits, long long rows_each) {
  __shared__ float red[3][THREADS / 64];
  const long long n = blockIdx.x / a.groups;
  const int g = (int)(blockIdx.x % a.groups), each = a.channels / a.groups;
  const long long live = live_positions(a, n);
  const int width = min(each, THREADS), lanes = THREADS / width, lane = threadIdx.x / width;
  // (means as distances from the first one: merging rounds the distance, not a mean far from zero)
  const float pivot = a.ws[n * splits * 2 * a.channels + g * each];
  float mean = 0.0f, m2 = 0.0f, count = 0.0f;
  constexpr int U = 4;
  if (lane < lanes)
    for (int c = threadIdx.x % width; c < each; c += width)
      for (int s = lane; s < splits; s += U * lanes) {
        float x[U], q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float* src = a.ws + (n * splits + min(s + u * lanes, splits - 1)) * 2 * a.channels + g * each + c;
          x[u] = src[0] - pivot, q[u] = src[a.channels];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (s + u * lanes < splits) merge(mean, m2, count, x[u], q[u], rows_of(s + u * lanes, rows_each, live));
      }
#pragma unroll
  for (int o = 32; o > 0; o /= 2) {
    const float mb = __shfl_down(mean, o), qb = __shfl_down(m2, o), cb = __shfl_down(count, o);
    merge(mean, m2, count, mb, qb, cb);
  }
  if (threadIdx.x % 64 == 0) red[0][threadIdx.x / 64] = mean, red[1][threadIdx.x / 64] = m2, red[2][threadIdx.x / 64] = count;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < THREADS / 64; ++w) merge(mean, m2, count, red[0][w], red[1][w], red[2][w]);
    a.mean[blockIdx.x] = count > 0.0f ? pivot + mean : 0.0f;
    a.rstd[blockIdx.x] = 1.0f / sqrtf((count > 0.0f ? m2 / count : 0.0f) + a.eps);
  }
}

// (from the last rows to the first: what the statistics read last is still in the Infinity Cache; and results past it, so that they
// do not displace it: with both 200 to 207 us for the above, with neither 227)
template <typename T, int V>
__global__ __launch_bounds__(kNormThreads) void norm_apply_kernel(NormArgs a, long long rows_each, unsigned splits) {
  const Slab s = slab_of<V>(a.channels);
  if (!s.on) return;
  const unsigned block = gridDim.x - 1 - blockIdx.x;
  const long long n = block / splits, live = live_positions(a, n);
  const long long r0 = (block % splits) * rows_each, r1 = min(r0 + rows_each, a.positions);
  const int each = a.channels / a.groups;
  float mean[V], mul[V], add[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const long long g = n * a.groups + (s.col + i) / each;
    mean[i] = a.mean[g];
    mul[i] = a.rstd[g] * (a.weight ? a.weight[s.col + i] : 1.0f);
    add[i] = a.bias ? a.bias[s.col + i] : 0.0f;
  }
  const size_t at = (size_t)n * a.positions * a.channels + s.col;
  const T* x = static_cast<const T*>(a.x) + at;
  T* y = static_cast<T*>(a.y) + at;
  constexpr int U = 4;
  for (long long r = r0 + s.lane; r < r1; r += (long long)U * s.lanes) {
    Pack<T, V> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long q = r + (long long)u * s.lanes;
      if (q < r1 && q < live) v[u] = *reinterpret_cast<const Pack<T, V>*>(x + q * a.channels);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long q = r + (long long)u * s.lanes;
      if (q >= r1) break;
      float z[V] = {};
      if (q < live)
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = activate(__builtin_fmaf(to_f32(v[u].v[i]) - mean[i], mul[i], add[i]), a.act);
      stream_pack<T, V>(y + q * a.channels, z);
    }
  }
}

// partial sums of dz and dz xhat over the workgroup's rows, laid out as the statistics' partials
template <typename T, int V>
__global__ __launch_bounds__(kNormThreads) void norm_grad_sums_kernel(NormArgs a, long long rows_each, unsigned splits) {
  __shared__ float red[2][kNormThreads * V];
  const Slab s = slab_of<V>(a.channels);
  const long long n = blockIdx.x / splits, live = live_positions(a, n);
  const long long r0 = (blockIdx.x % splits) * rows_each, r1 = min(r0 + rows_each, live);
  const int each = a.channels / a.groups;
  const size_t at = (size_t)n * a.positions * a.channels + s.col;
  const T* x = static_cast<const T*>(a.x) + at;
  const T* dy = static_cast<const T*>(a.dy) + at;
  float s1[V] = {}, s2[V] = {};
  if (s.on) {
    float mean[V], rstd[V], w[V], b[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const long long g = n * a.groups + (s.col + i) / each;
      mean[i] = a.mean[g];
      rstd[i] = a.rstd[g];
      w[i] = a.weight ? a.weight[s.col + i] : 1.0f;
      b[i] = a.bias ? a.bias[s.col + i] : 0.0f;
    }
    for (long long r = r0 + s.lane; r < r1; r += s.lanes) {
      float v[V], d[V];
      load_pack<T, V>(x + r * a.channels, v);
      load_pack<T, V>(dy + r * a.channels, d);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xh = (v[i] - mean[i]) * rstd[i];
        const float dz = d[i] * activation_slope(__builtin_fmaf(xh, w[i], b[i]), a.act);
        s1[i] += dz;
        s2[i] = __builtin_fmaf(dz, xh, s2[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      red[0][threadIdx.x * V + i] = s1[i];
      red[1][threadIdx.x * V + i] = s2[i];
    }
  }
  __syncthreads();
  const int vecs = a.channels / V, width = min(vecs - (int)blockIdx.z * kNormThreads, kNormThreads) * V;
  float* out = a.ws + (size_t)blockIdx.x * 2 * a.channels + (size_t)blockIdx.z * kNormThreads * V;
  for (int c = threadIdx.x; c < width; c += kNormThreads) {
    float u = 0.0f, q = 0.0f;
    for (int l = 0; l < s.lanes; ++l) u += red[0][l * width + c], q += red[1][l * width + c];
    out[c] = u;
    out[a.channels + c] = q;
  }
}

// mean(dz w) and mean(dz w xhat) of one (sample, group): a wave each, behind the partials
template <int THREADS>
__global__ __launch_bounds__(THREADS) void norm_grad_join_kernel(NormArgs a, int splits, float* joined) {
  __shared__ float red[2][THREADS / 64];
  const long long n = blockIdx.x / a.groups;
  const int g = (int)(blockIdx.x % a.groups), each = a.channels / a.groups;
  const int width = min(each, THREADS), lanes = THREADS / width, lane = threadIdx.x / width;
  float u = 0.0f, q = 0.0f;
  if (lane < lanes)
    for (int c = threadIdx.x % width; c < each; c += width) {
      const float w = a.weight ? a.weight[g * each + c] : 1.0f;
      float cu = 0.0f, cq = 0.0f;
#pragma unroll 4
      for (int s = lane; s < splits; s += lanes) {
        const float* src = a.ws + (n * splits + s) * 2 * a.channels + g * each + c;
        cu += src[0], cq += src[a.channels];
      }
      u = __builtin_fmaf(w, cu, u), q = __builtin_fmaf(w, cq, q);
    }
#pragma unroll
  for (int o = 32; o > 0; o /= 2) u += __shfl_down(u, o), q += __shfl_down(q, o);
  if (threadIdx.x % 64 == 0) red[0][threadIdx.x / 64] = u, red[1][threadIdx.x / 64] = q;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < THREADS / 64; ++w) u += red[0][w], q += red[1][w];
    const float count = (float)live_positions(a, n) * (float)each;
    joined[2 * blockIdx.x] = count > 0.0f ? u / count : 0.0f;
    joined[2 * blockIdx.x + 1] = count > 0.0f ? q / count : 0.0f;
  }
}

// dbias[c], dweight[c]: 32 channels a workgroup, the partials of all samples and splits in a fixed order
__global__ __launch_bounds__(1024) void norm_weight_grad_kernel(const float* __restrict__ partial, float* __restrict__ dweight,
                                                                float* __restrict__ dbias, int channels, long long parts) {
  __shared__ float red[2][32][33];
  const int cl = threadIdx.x % 32, c = blockIdx.x * 32 + cl, lane = threadIdx.x / 32;
  constexpr int U = 8;
  float u = 0.0f, q = 0.0f;
  if (c < channels)
    for (long long i = lane; i < parts; i += 32 * U) {
      float p[U], r[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const bool in = i + 32 * k < parts;
        const float* src = partial + (i + 32 * k) * 2 * channels + c;
        p[k] = in ? src[0] : 0.0f;
        r[k] = in ? src[channels] : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < U; ++k) u += p[k], q += r[k];
    }
  red[0][lane][cl] = u;
  red[1][lane][cl] = q;
  __syncthreads();
  if (lane == 0 && c < channels) {
    for (int l = 1; l < 32; ++l) u += red[0][l][cl], q += red[1][l][cl];
    if (dbias) dbias[c] = u;
    if (dweight) dweight[c] = q;
  }
}

template <typename T, int V>
__global__ __launch_bounds__(kNormThreads) void norm_grad_kernel(NormArgs a, long long rows_each, unsigned splits, const float* joined) {
  const Slab s = slab_of<V>(a.channels);
  if (!s.on) return;
  const unsigned block = gridDim.x - 1 - blockIdx.x;
  const long long n = block / splits, live = live_positions(a, n);
  const long long r0 = (block % splits) * rows_each, r1 = min(r0 + rows_each, a.positions);
  const int each = a.channels / a.groups;
  float mean[V], rstd[V], w[V], b[V], c1[V], c2[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const long long g = n * a.groups + (s.col + i) / each;
    mean[i] = a.mean[g];
    rstd[i] = a.rstd[g];
    w[i] = a.weight ? a.weight[s.col + i] : 1.0f;
    b[i] = a.bias ? a.bias[s.col + i] : 0.0f;
    c1[i] = joined[2 * g];
    c2[i] = joined[2 * g + 1];
  }
  const size_t at = (size_t)n * a.positions * a.channels + s.col;
  const T* x = static_cast<const T*>(a.x) + at;
  const T* dy = static_cast<const T*>(a.dy) + at;
  T* dx = static_cast<T*>(a.y) + at;
  for (long long r = r0 + s.lane; r < r1; r += s.lanes) {
    float v[V] = {}, d[V];
    if (r < live) {
      load_pack<T, V>(x + r * a.channels, v);
      load_pack<T, V>(dy + r * a.channels, d);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xh = (v[i] - mean[i]) * rstd[i];
        const float u = d[i] * activation_slope(__builtin_fmaf(xh, w[i], b[i]), a.act) * w[i];
        v[i] = rstd[i] * (u - c1[i] - xh * c2[i]);
      }
    }
    store_pack<T, V>(dx + r * a.channels, v);
  }
}

// ------------------------------------------------------------------------------------------------
// Samples that fit a workgroup's registers: one launch, every value read once (64 x 1000 x 512 in 32 groups, bf16: 33 us, 3.9 TB/s;
// in passes 63; 64 x 626 x 512 29 against 45, a training pass with all of its host work 118 against 136; past 1024 positions of such a tile only passes remain).  A workgroup takes whole groups of one
// sample, some 128 bytes of each position (a cache line), K 16-byte vectors a thread.  Statistics are two passes over the
// registers.  Gradients keep x and dy; the activation's slope is computed twice, which is cheaper than keeping it.
// ------------------------------------------------------------------------------------------------

struct NormTile {
  int threads, vecs, lanes, groups, k;  // vectors of a position in the tile, as lanes: a power of two; groups of a tile; K
  unsigned tiles;
};

// (sum over the rows and the group's vectors of two values a thread; lanes of one vector are `lanes` apart)
template <int W>
__device__ __forceinline__ void group_sum(float& u, float& q, float (*red)[64][2], int lanes, int col, int group_vecs, int vecs) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int o = lanes; o < 64; o *= 2) u += __shfl_xor(u, o), q += __shfl_xor(q, o);
  __syncthreads();
  if (lane < lanes) red[wave][lane][0] = u, red[wave][lane][1] = q;
  __syncthreads();
  u = q = 0.0f;
  const int c0 = col / group_vecs * group_vecs;
  if (col < vecs)
    for (int w = 0; w < W; ++w)
      for (int c = 0; c < group_vecs; ++c) u += red[w][c0 + c][0], q += red[w][c0 + c][1];
}

template <typename T, int V, int K, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_whole_kernel(NormArgs a, NormTile t) {
  __shared__ float red[THREADS / 64][64][2];
  const long long n = blockIdx.x / t.tiles;
  const int each = a.channels / a.groups, group_vecs = each / V;
  const int g0 = (int)(blockIdx.x % t.tiles) * t.groups, vecs = min(t.groups, a.groups - g0) * group_vecs;
  const int col = threadIdx.x % t.lanes, row = threadIdx.x / t.lanes, rows = THREADS / t.lanes;
  const int live = (int)live_positions(a, n), positions = (int)a.positions;
  const bool on = col < vecs;
  const int ch = g0 * each + col * V, g = g0 + (on ? col / group_vecs : 0);
  const size_t at = (size_t)n * a.positions * a.channels + ch;
  const T* x = static_cast<const T*>(a.x) + at;
  Raw<T, V> v[K];
  float sum = 0.0f, unused = 0.0f;
  // (sums are of distances from one of the group's values: a mean far from zero costs nothing)
  const float pivot = on && live ? to_f32(static_cast<const T*>(a.x)[(size_t)n * a.positions * a.channels + g * each]) : 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    for (unsigned& w : v[k].w) w = 0;
    const int r = row + k * rows;
    if (on && r < live) v[k] = *reinterpret_cast<const Raw<T, V>*>(x + (size_t)r * a.channels);
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (on && row + k * rows < live)
#pragma unroll
      for (int i = 0; i < V; ++i) sum += v[k].at(i) - pivot;
  group_sum<THREADS / 64>(sum, unused, red, t.lanes, col, group_vecs, vecs);
  const float count = (float)live * (float)each, mean = live ? pivot + sum / count : 0.0f;
  float m2 = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (row + k * rows < live)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = v[k].at(i) - mean;
        m2 = __builtin_fmaf(d, d, m2);
      }
  if (!on) m2 = 0.0f;
  group_sum<THREADS / 64>(m2, unused, red, t.lanes, col, group_vecs, vecs);
  const float rstd = 1.0f / sqrtf((live ? m2 / count : 0.0f) + a.eps);
  if (!on) return;
  if (row == 0 && col % group_vecs == 0) {
    a.mean[n * a.groups + g] = mean;
    a.rstd[n * a.groups + g] = rstd;
  }
  float mul[V], add[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    mul[i] = rstd * (a.weight ? a.weight[ch + i] : 1.0f);
    add[i] = a.bias ? a.bias[ch + i] : 0.0f;
  }
  T* y = static_cast<T*>(a.y) + at;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    __builtin_amdgcn_sched_barrier(0);  // (one vector at a time: registers)
    const int r = row + k * rows;
    if (r >= positions) break;
    float z[V] = {};
    if (r < live)
#pragma unroll
      for (int i = 0; i < V; ++i) z[i] = activate(__builtin_fmaf(v[k].at(i) - mean, mul[i], add[i]), a.act);
    store_pack<T, V>(y + (size_t)r * a.channels, z);
  }
}

// the same for the gradients; partial sums of dz and dz xhat by channel at ws[(n * 2 + {0, 1}) * channels + c]
template <typename T, int V, int K, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_whole_grad_kernel(NormArgs a, NormTile t) {
  __shared__ float red[THREADS / 64][64][2];
  __shared__ float part[THREADS / 64][64 * V];
  const long long n = blockIdx.x / t.tiles;
  const int each = a.channels / a.groups, group_vecs = each / V;
  const int g0 = (int)(blockIdx.x % t.tiles) * t.groups, vecs = min(t.groups, a.groups - g0) * group_vecs;
  const int col = threadIdx.x % t.lanes, row = threadIdx.x / t.lanes, rows = THREADS / t.lanes;
  const int live = (int)live_positions(a, n), positions = (int)a.positions;
  const bool on = col < vecs;
  const int ch = on ? g0 * each + col * V : g0 * each, g = g0 + (on ? col / group_vecs : 0);
  const size_t at = (size_t)n * a.positions * a.channels + ch;
  const T* x = static_cast<const T*>(a.x) + at;
  const T* dy = static_cast<const T*>(a.dy) + at;
  Raw<T, V> v[K], d[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int r = row + k * rows;
    if (on && r < live) {
      v[k] = *reinterpret_cast<const Raw<T, V>*>(x + (size_t)r * a.channels);
      d[k] = *reinterpret_cast<const Raw<T, V>*>(dy + (size_t)r * a.channels);
    }
  }
  const float mean = a.mean[n * a.groups + g], rstd = a.rstd[n * a.groups + g];
  float w[V], b[V], s1[V] = {}, s2[V] = {};
#pragma unroll
  for (int i = 0; i < V; ++i) {
    w[i] = a.weight ? a.weight[ch + i] : 1.0f;
    b[i] = a.bias ? a.bias[ch + i] : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    __builtin_amdgcn_sched_barrier(0);  // (one vector at a time: registers)
    if (on && row + k * rows < live)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xh = (v[k].at(i) - mean) * rstd;
        const float dz = d[k].at(i) * activation_slope(__builtin_fmaf(xh, w[i], b[i]), a.act);
        s1[i] += dz;
        s2[i] = __builtin_fmaf(dz, xh, s2[i]);
      }
  }
  float u = 0.0f, q = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) u = __builtin_fmaf(w[i], s1[i], u), q = __builtin_fmaf(w[i], s2[i], q);
  group_sum<THREADS / 64>(u, q, red, t.lanes, col, group_vecs, vecs);
  const float count = (float)live * (float)each;
  const float c1 = live ? u / count : 0.0f, c2 = live ? q / count : 0.0f;
  if (a.dweight || a.dbias) {
#pragma unroll
    for (int z = 0; z < 2; ++z) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float s = z ? s2[i] : s1[i];
        for (int o = t.lanes; o < 64; o *= 2) s += __shfl_xor(s, o);
        if ((int)(threadIdx.x & 63) < t.lanes) part[threadIdx.x >> 6][(threadIdx.x & 63) * V + i] = s;
      }
      __syncthreads();
      for (int c = threadIdx.x; c < vecs * V; c += THREADS) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < THREADS / 64; ++k) s += part[k][c];
        a.ws[(n * 2 + z) * a.channels + g0 * each + c] = s;
      }
      __syncthreads();
    }
  }
  if (!on) return;
  // (as new values: xhat and the slope are computed again, not kept for all of K in registers)
  float mean2 = mean, rstd2 = rstd;
  asm volatile("" : "+v"(mean2), "+v"(rstd2));
  T* dx = static_cast<T*>(a.y) + at;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    __builtin_amdgcn_sched_barrier(0);
    const int r = row + k * rows;
    if (r >= positions) break;
    float z[V] = {};
    if (r < live)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xh = (v[k].at(i) - mean2) * rstd2;
        const float e = d[k].at(i) * activation_slope(__builtin_fmaf(xh, w[i], b[i]), a.act) * w[i];
        z[i] = rstd2 * (e - c1 - xh * c2);
      }
    store_pack<T, V>(dx + (size_t)r * a.channels, z);
  }
}

// ------------------------------------------------------------------------------------------------
// Samples of few positions (a frame of a stream, or every frame normalised by itself): several to a wave.  A team of S <= 64 lanes takes one
// tile of one sample, K vectors a lane; its sums are lane exchanges, without shared memory or barriers.  Teams go on to
// further samples of the same tile, and so sum the weights' gradients in registers: the partial sums that reach memory are one row a
// workgroup, where a row a sample would be twice as much as x itself.  40064 samples of 256 features, bf16: 24 us in one group, 17 in 4
// (a workgroup a sample and 8 vectors: 372 and 728); with gradients 65 and 56 (814 and 1707).  For what it takes it is never slower.
// ------------------------------------------------------------------------------------------------

struct NormRows {
  int slot, lanes, rows, groups, k;  // lanes of a group (a power of two), of a tile, positions at a time; groups of a tile; K (0: not taken)
  unsigned tiles, parts;             // workgroups of a tile: rows of the weights' partial sums
};
constexpr int kRowsThreads = 256;

struct TeamLane {
  int row, ch, g;
  long long n, step;  // first sample of the team, samples apart
  bool on, first;     // has channels; is its group's first lane
};
template <int V>
__device__ __forceinline__ TeamLane team_lane(const NormArgs& a, const NormRows& t) {
  const int size = t.lanes * t.rows, lane = threadIdx.x % size % t.lanes, each = a.channels / a.groups;
  const int teams = kRowsThreads / size, group = (int)(blockIdx.x % t.tiles) * t.groups + lane / t.slot, vec = lane % t.slot;
  TeamLane m;
  m.row = threadIdx.x % size / t.lanes;
  m.on = group < a.groups && vec * V < each;
  m.first = vec == 0 && m.row == 0;
  m.g = m.on ? group : 0;
  m.ch = m.on ? group * each + vec * V : 0;
  m.n = (long long)(blockIdx.x / t.tiles) * teams + threadIdx.x / size;
  m.step = (long long)t.parts * teams;
  return m;
}
__device__ __forceinline__ float team_sum(float u, const NormRows& t) {
  for (int o = 1; o < t.slot; o *= 2) u += __shfl_xor(u, o);
  for (int o = t.lanes; o < t.lanes * t.rows; o *= 2) u += __shfl_xor(u, o);
  return u;
}

template <typename T, int V, int K>
__global__ __launch_bounds__(kRowsThreads) void norm_rows_kernel(NormArgs a, NormRows t) {
  const TeamLane m = team_lane<V>(a, t);
  const int each = a.channels / a.groups, positions = (int)a.positions;
  float w[V], b[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    w[i] = a.weight ? a.weight[m.ch + i] : 1.0f;
    b[i] = a.bias ? a.bias[m.ch + i] : 0.0f;
  }
  for (long long n = m.n; n < a.batch; n += m.step) {
    const int live = (int)live_positions(a, n);
    const size_t at = (size_t)n * a.positions * a.channels + m.ch;
    const T* x = static_cast<const T*>(a.x) + at;
    Raw<T, V> v[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      for (unsigned& u : v[k].w) u = 0;
      const int r = m.row + k * t.rows;
      if (m.on && r < live) v[k] = *reinterpret_cast<const Raw<T, V>*>(x + (size_t)r * a.channels);
    }
    // (distances from the group's first value, as above)
    const float pivot = __shfl(v[0].at(0), (int)(threadIdx.x & 63) / (t.lanes * t.rows) * (t.lanes * t.rows) + threadIdx.x % t.lanes / t.slot * t.slot);
    float sum = 0.0f, m2 = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (m.on && m.row + k * t.rows < live)
#pragma unroll
        for (int i = 0; i < V; ++i) sum += v[k].at(i) - pivot;
    const float count = (float)live * (float)each, mean = live ? pivot + team_sum(sum, t) / count : 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (m.on && m.row + k * t.rows < live)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = v[k].at(i) - mean;
          m2 = __builtin_fmaf(d, d, m2);
        }
    m2 = team_sum(m2, t);
    const float rstd = 1.0f / sqrtf((live ? m2 / count : 0.0f) + a.eps);
    if (m.on && m.first) {
      a.mean[n * a.groups + m.g] = mean;
      a.rstd[n * a.groups + m.g] = rstd;
    }
    T* y = static_cast<T*>(a.y) + at;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int r = m.row + k * t.rows;
      if (!m.on || r >= positions) continue;
      float z[V] = {};
      if (r < live)
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = activate(__builtin_fmaf(v[k].at(i) - mean, rstd * w[i], b[i]), a.act);
      store_pack<T, V>(y + (size_t)r * a.channels, z);
    }
  }
}

// the same for the gradients; partial sums of dz and dz xhat by channel at ws[(part * 2 + {0, 1}) * channels + c]
template <typename T, int V, int K>
__global__ __launch_bounds__(kRowsThreads) void norm_rows_grad_kernel(NormArgs a, NormRows t) {
  __shared__ float part[kRowsThreads / 64][64 * V];
  const TeamLane m = team_lane<V>(a, t);
  const int each = a.channels / a.groups, positions = (int)a.positions;
  float w[V], b[V], db[V] = {}, dw[V] = {};
#pragma unroll
  for (int i = 0; i < V; ++i) {
    w[i] = a.weight ? a.weight[m.ch + i] : 1.0f;
    b[i] = a.bias ? a.bias[m.ch + i] : 0.0f;
  }
  for (long long n = m.n; n < a.batch; n += m.step) {
    const int live = (int)live_positions(a, n);
    const size_t at = (size_t)n * a.positions * a.channels + m.ch;
    const T* x = static_cast<const T*>(a.x) + at;
    const T* dy = static_cast<const T*>(a.dy) + at;
    Raw<T, V> v[K], d[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int r = m.row + k * t.rows;
      if (m.on && r < live) {
        v[k] = *reinterpret_cast<const Raw<T, V>*>(x + (size_t)r * a.channels);
        d[k] = *reinterpret_cast<const Raw<T, V>*>(dy + (size_t)r * a.channels);
      }
    }
    const float mean = a.mean[n * a.groups + m.g], rstd = a.rstd[n * a.groups + m.g];
    float e[K][V], xh[K][V], u = 0.0f, q = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        e[k][i] = xh[k][i] = 0.0f;
        if (m.on && m.row + k * t.rows < live) {
          xh[k][i] = (v[k].at(i) - mean) * rstd;
          const float dz = d[k].at(i) * activation_slope(__builtin_fmaf(xh[k][i], w[i], b[i]), a.act);
          db[i] += dz;
          dw[i] = __builtin_fmaf(dz, xh[k][i], dw[i]);
          e[k][i] = dz * w[i];
          u += e[k][i];
          q = __builtin_fmaf(e[k][i], xh[k][i], q);
        }
      }
    const float count = (float)live * (float)each;
    u = team_sum(u, t), q = team_sum(q, t);
    const float c1 = live ? u / count : 0.0f, c2 = live ? q / count : 0.0f;
    T* dx = static_cast<T*>(a.y) + at;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int r = m.row + k * t.rows;
      if (!m.on || r >= positions) continue;
      float z[V] = {};
      if (r < live)
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = rstd * (e[k][i] - c1 - xh[k][i] * c2);
      store_pack<T, V>(dx + (size_t)r * a.channels, z);
    }
  }
  if (!a.dweight && !a.dbias) return;
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int z = 0; z < 2; ++z) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float s = z ? dw[i] : db[i];
      for (int o = t.lanes; o < 64; o *= 2) s += __shfl_xor(s, o);
      if (lane < t.lanes) part[threadIdx.x >> 6][lane * V + i] = s;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < t.lanes * V; c += kRowsThreads) {
      const int own = c / V, group = (int)(blockIdx.x % t.tiles) * t.groups + own / t.slot, at = own % t.slot * V;
      if (group < a.groups && at < each)
        a.ws[((size_t)(blockIdx.x / t.tiles) * 2 + z) * a.channels + group * each + at + c % V] = part[0][c] + part[1][c] + part[2][c] + part[3][c];
    }
    __syncthreads();
  }
}

// The tile of a sample that a team takes, where four vectors a lane hold all positions.
static NormRows norm_rows(const NormArgs& a, int size) {
  NormRows t{};
  const int V = 16 / size, each = a.channels / a.groups;
  if (each % V || each / V > 64) return t;
  for (t.slot = 1; t.slot < each / V;) t.slot *= 2;
  for (t.groups = 1; t.groups < a.groups && t.groups * t.slot < 8;) t.groups *= 2;  // (128 bytes of a position, a cache line)
  t.lanes = t.groups * t.slot;
  for (t.rows = 1; t.rows < a.positions && t.rows * t.lanes < 64;) t.rows *= 2;
  const long long k = (a.positions + t.rows - 1) / t.rows;
  if (k > 4) return t;
  t.k = k == 1 ? 1 : 4;
  t.tiles = (unsigned)((a.groups + t.groups - 1) / t.groups);
  const long long teams = kRowsThreads / (t.lanes * t.rows), need = (a.batch + teams - 1) / teams;
  t.parts = (unsigned)std::min(need, std::max(1LL, 2048LL / t.tiles));  // (2048: eight waves a SIMD)
  return t;
}

// The tile of a sample that a workgroup can hold (threads = 0: none can): K vectors a thread, of one tensor or two. Few threads with many vectors
// leave room for several workgroups a compute unit, which cover each other's reductions (1024 threads of 5 vectors: one fits)
static NormTile norm_tile(const NormArgs& a, int size) {
  NormTile t{};
  const int V = 16 / size, each = a.channels / a.groups;
  if (a.channels % V || each % V || each / V > 64) return t;
  const int group_vecs = each / V;
  t.groups = std::min(a.groups, std::max(1, 8 / group_vecs));
  t.vecs = t.groups * group_vecs;
  t.lanes = 1;
  while (t.lanes < t.vecs) t.lanes *= 2;
  t.tiles = (unsigned)((a.groups + t.groups - 1) / t.groups);
  for (const int threads : {256, 512}) {
    const long long rows = threads / t.lanes, k = (a.positions + rows - 1) / rows;
    if (k > (threads == 256 ? 20 : 16)) continue;  // (20: the most that leaves the backward two waves a SIMD)
    t.threads = threads;
    t.k = threads == 512 ? 16 : k <= 2 ? 2 : k <= 8 ? 8 : k <= 14 ? 14 : 20;
    break;
  }
  return t;
}

// ------------------------------------------------------------------------------------------------

// Rows of a workgroup: about 1024 workgroups in all, at least 32 rows each, at most 65535 splits.  bf16, forward, with 1024, 2048 and 4096:
// 1 x 160882 x 32 in 8 groups 30, 43 and 61 us (the joins), 64 x 2000 x 512 in 32 82, 89 and 113; 32 x 160882 x 32 203, 203
// and 207, its training pass 562, 539 and 544.
static long long norm_rows_each(const NormArgs& a) {
  const long long want = std::max(1LL, 1024 / std::max(1LL, a.batch));
  const long long splits = std::min({want, std::max(1LL, a.positions / 32), 65535LL});
  return (a.positions + splits - 1) / splits;
}
static long long norm_splits(const NormArgs& a) {
  const long long each = norm_rows_each(a);
  return (a.positions + each - 1) / each;
}

template <typename T>
static bool norm_vectors(const NormArgs& a) {
  return a.channels % (16 / (int)sizeof(T)) == 0;
}

bool norm_aligned(const NormArgs& a) {
  const uintptr_t any = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.dy);
  return any % 16 == 0;
}

size_t norm_workspace_bytes(const NormArgs& a, bool backward) {
  if (a.batch == 0 || a.positions == 0) return 0;
  const int size = a.dtype == 0 ? 4 : 2;
  if (const NormRows t = norm_rows(a, size); t.k) return backward ? sizeof(float) * (size_t)t.parts * 2 * a.channels : 0;
  if (norm_tile(a, size).threads) return backward ? sizeof(float) * (size_t)a.batch * 2 * a.channels : 0;
  const size_t parts = (size_t)a.batch * norm_splits(a) * 2 * a.channels;
  return sizeof(float) * (parts + (backward ? (size_t)a.batch * a.groups * 2 : 0));
}

static void weight_grad_launch(const NormArgs& a, long long parts) {
  hipLaunchKernelGGL(norm_weight_grad_kernel, dim3((a.channels + 31) / 32), dim3(1024), 0, a.stream, a.ws, a.dweight, a.dbias,
                     a.channels, parts);
}

// The samples [first, first + most) of a, whose workspace holds `parts` rows of partial sums a sample.
template <typename T>
static NormArgs samples_of(NormArgs a, long long first, long long most, long long parts) {
  const size_t at = (size_t)first * a.positions * a.channels;
  a.x = static_cast<const T*>(a.x) + at;
  a.y = static_cast<T*>(a.y) + at;
  if (a.dy) a.dy = static_cast<const T*>(a.dy) + at;
  a.mean += first * a.groups;
  a.rstd += first * a.groups;
  if (a.lengths) a.lengths += first;
  if (a.ws) a.ws += (size_t)first * parts * 2 * a.channels;
  a.batch = std::min(most, a.batch - first);
  return a;
}

template <typename T, int V, int K, int THREADS>
static hipError_t whole_launch(const NormArgs& all, const NormTile& t, bool backward) {
  const long long most = max_blocks(THREADS) / t.tiles;  // samples of a launch (tiles are below 2^20)
  for (long long first = 0; first < all.batch; first += most) {
    const NormArgs a = samples_of<T>(all, first, most, 1);
    const dim3 grid((unsigned)a.batch * t.tiles), block(THREADS);
    if (!backward)
      hipLaunchKernelGGL((norm_whole_kernel<T, V, K, THREADS>), grid, block, 0, a.stream, a, t);
    else
      hipLaunchKernelGGL((norm_whole_grad_kernel<T, V, K, THREADS>), grid, block, 0, a.stream, a, t);
  }
  if (backward && (all.dweight || all.dbias)) weight_grad_launch(all, all.batch);
  return hipGetLastError();
}

template <typename T, int V, int K>
static hipError_t rows_launch(const NormArgs& a, const NormRows& t, bool backward) {
  const dim3 grid(t.parts * t.tiles), block(kRowsThreads);
  if (!backward) {
    hipLaunchKernelGGL((norm_rows_kernel<T, V, K>), grid, block, 0, a.stream, a, t);
  } else {
    hipLaunchKernelGGL((norm_rows_grad_kernel<T, V, K>), grid, block, 0, a.stream, a, t);
    if (a.dweight || a.dbias) weight_grad_launch(a, t.parts);
  }
  return hipGetLastError();
}

template <typename T, int V>
static hipError_t whole_sizes(const NormArgs& a, const NormTile& t, bool backward) {
  if (t.threads == 512) return whole_launch<T, V, 16, 512>(a, t, backward);
  if (t.k <= 8) return t.k == 2 ? whole_launch<T, V, 2, 256>(a, t, backward) : whole_launch<T, V, 8, 256>(a, t, backward);
  return t.k == 14 ? whole_launch<T, V, 14, 256>(a, t, backward) : whole_launch<T, V, 20, 256>(a, t, backward);
}

// In passes: the samples of a launch (one always fits: splits are below 2^16, groups 2^20 at most)
static long long pass_samples(const NormArgs& a, long long splits, bool few) {
  return std::min(max_blocks(kNormThreads) / splits, max_blocks(few ? 64 : 1024) / a.groups);
}

template <typename T, int V>
static hipError_t forward_launch(const NormArgs& all) {
  const long long each = norm_rows_each(all), splits = norm_splits(all);
  const int vecs = all.channels / V;
  const bool few = splits * (all.channels / all.groups) <= kJoinFew;
  const long long most = pass_samples(all, splits, few);
  for (long long first = 0; first < all.batch; first += most) {
    const NormArgs a = samples_of<T>(all, first, most, splits);
    const dim3 grid((unsigned)(splits * a.batch), 1, (unsigned)((vecs + kNormThreads - 1) / kNormThreads)), block(kNormThreads);
    hipLaunchKernelGGL((norm_stats_kernel<T, V>), grid, block, 0, a.stream, a, each, (unsigned)splits);
    const dim3 joins((unsigned)(a.batch * a.groups));
    if (few)
      hipLaunchKernelGGL(norm_join_kernel<64>, joins, dim3(64), 0, a.stream, a, (int)splits, each);
    else
      hipLaunchKernelGGL(norm_join_kernel<1024>, joins, dim3(1024), 0, a.stream, a, (int)splits, each);
    hipLaunchKernelGGL((norm_apply_kernel<T, V>), grid, block, 0, a.stream, a, each, (unsigned)splits);
  }
  return hipGetLastError();
}

template <typename T, int V>
static hipError_t backward_launch(const NormArgs& all) {
  const long long each = norm_rows_each(all), splits = norm_splits(all);
  const int vecs = all.channels / V;
  const bool few = splits * (all.channels / all.groups) <= kJoinFew;
  const long long most = pass_samples(all, splits, few);
  float* const joins_at = all.ws + (size_t)all.batch * splits * 2 * all.channels;
  for (long long first = 0; first < all.batch; first += most) {
    const NormArgs a = samples_of<T>(all, first, most, splits);
    const dim3 grid((unsigned)(splits * a.batch), 1, (unsigned)((vecs + kNormThreads - 1) / kNormThreads)), block(kNormThreads);
    float* const joined = joins_at + (size_t)first * a.groups * 2;
    hipLaunchKernelGGL((norm_grad_sums_kernel<T, V>), grid, block, 0, a.stream, a, each, (unsigned)splits);
    const dim3 joins((unsigned)(a.batch * a.groups));
    if (few)
      hipLaunchKernelGGL(norm_grad_join_kernel<64>, joins, dim3(64), 0, a.stream, a, (int)splits, joined);
    else
      hipLaunchKernelGGL(norm_grad_join_kernel<1024>, joins, dim3(1024), 0, a.stream, a, (int)splits, joined);
    hipLaunchKernelGGL((norm_grad_kernel<T, V>), grid, block, 0, a.stream, a, each, (unsigned)splits, joined);
  }
  if (all.dweight || all.dbias) weight_grad_launch(all, all.batch * splits);
  return hipGetLastError();
}

template <typename T>
static hipError_t norm_typed(const NormArgs& a, bool backward) {
  constexpr int V = 16 / sizeof(T);
  if (norm_vectors<T>(a)) {
    if (const NormRows t = norm_rows(a, sizeof(T)); t.k)
      return t.k == 1 ? rows_launch<T, V, 1>(a, t, backward) : rows_launch<T, V, 4>(a, t, backward);
    const NormTile t = norm_tile(a, sizeof(T));
    if (t.threads) return whole_sizes<T, V>(a, t, backward);
    return backward ? backward_launch<T, V>(a) : forward_launch<T, V>(a);
  }
  return backward ? backward_launch<T, 1>(a) : forward_launch<T, 1>(a);
}

static hipError_t norm_any(const NormArgs& a, bool backward) {
  if (a.dtype == 0) return norm_typed<float>(a, backward);
  return a.dtype == 1 ? norm_typed<__bf16>(a, backward) : norm_typed<_Float16>(a, backward);
}

hipError_t launch_norm_forward(const NormArgs& a) { return norm_any(a, false); }
hipError_t launch_norm_backward(const NormArgs& a) { return norm_any(a, true); }

}  // namespace tfa
