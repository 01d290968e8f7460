// Group norm with an activation on channels-last data (batch, positions, channels), forward and backward.
//
//   xhat = (x - mean) rstd over the positions and the channels of a group, z = xhat w + b, y = act(z)
//   dz = dy act'(z), db = sum dz, dw = sum dz xhat, dx = rstd (dz w - mean(dz w) - xhat mean(dz w xhat))
//
// Memory bound: forward x and y once, backward x, dy and dx once is the floor.  Statistics are fp32 (mean, sum of squared
// deviations) pairs that are merged, never a difference of sums of squares.  With lengths, positions at and past
// lengths[n] * inner are padding: not read, zeros in y and dx.
#include "model_ops.h"

#include <algorithm>

namespace tfa {

enum { kActNone = 0, kActSilu = 1, kActGelu = 2, kActRelu = 3 };

__device__ __forceinline__ float activate(float z, int act) {
  if (act == kActSilu) return z / (1.0f + expf(-z));
  if (act == kActGelu) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  if (act == kActRelu) return z > 0.0f ? z : z != z ? z : 0.0f;  // NaN stays
  return z;
}

__device__ __forceinline__ float activation_slope(float z, int act) {
  if (act == kActSilu) {
    const float s = 1.0f / (1.0f + expf(-z));
    return s * (1.0f + z * (1.0f - s));
  }
  if (act == kActGelu)
    return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * expf(-0.5f * z * z);
  if (act == kActRelu) return z > 0.0f ? 1.0f : 0.0f;
  return 1.0f;
}

template <typename T, int V>
struct __attribute__((aligned(V * sizeof(T)))) Pack {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_pack(const T* p, float (&x)[V]) {
  const Pack<T, V> u = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = to_f32(u.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const float (&x)[V]) {
  Pack<T, V> u;
#pragma unroll
  for (int i = 0; i < V; ++i) u.v[i] = from_f32<T>(x[i]);
  *reinterpret_cast<Pack<T, V>*>(p) = u;
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

// A workgroup takes rows [r0, r1) of one sample and up to 256 vectors of V channels; a thread keeps its channels
// over its rows: kLane rows apart.
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
      const int full = (int)min((long long)U, (r1 - r + s.lanes - 1) / s.lanes);
#pragma unroll
      for (int u = 0; u < U; ++u)  // (rows past the end repeat the last: in bounds, weight 0)
        load_pack<T, V>(x + (r + (long long)min(u, full - 1) * s.lanes) * a.channels, v[u]);
      const float inv = 1.0f / (float)full, f = (float)full / (count + (float)full);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float sum = 0.0f, sq = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) sum += u < full ? v[u][i] : 0.0f;
        sum *= inv;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float d = u < full ? v[u][i] - sum : 0.0f;
          sq = __builtin_fmaf(d, d, sq);
        }
        const float d = sum - mean[i];
        mean[i] = __builtin_fmaf(d, f, mean[i]);
        m2[i] += sq + d * d * count * f;
      }
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

// joins the partials of one (sample, group): a wave each
__global__ __launch_bounds__(64) void norm_join_kernel(NormArgs a, int splits, long long rows_each) {
  const long long n = blockIdx.x / a.groups;
  const int g = (int)(blockIdx.x % a.groups), each = a.channels / a.groups;
  const long long live = live_positions(a, n);
  float mean = 0.0f, m2 = 0.0f, count = 0.0f;
  for (long long i = threadIdx.x; i < (long long)splits * each; i += 64) {
    const long long split = i / each;
    const float* src = a.ws + (n * splits + split) * 2 * a.channels + g * each + i % each;
    merge(mean, m2, count, src[0], src[a.channels], rows_of(split, rows_each, live));
  }
#pragma unroll
  for (int o = 32; o > 0; o /= 2) {
    const float mb = __shfl_down(mean, o), qb = __shfl_down(m2, o), cb = __shfl_down(count, o);
    merge(mean, m2, count, mb, qb, cb);
  }
  if (threadIdx.x == 0) {
    a.mean[blockIdx.x] = mean;
    a.rstd[blockIdx.x] = 1.0f / sqrtf((count > 0.0f ? m2 / count : 0.0f) + a.eps);
  }
}

template <typename T, int V>
__global__ __launch_bounds__(kNormThreads) void norm_apply_kernel(NormArgs a, long long rows_each, unsigned splits) {
  const Slab s = slab_of<V>(a.channels);
  if (!s.on) return;
  const long long n = blockIdx.x / splits, live = live_positions(a, n);
  const long long r0 = (blockIdx.x % splits) * rows_each, r1 = min(r0 + rows_each, a.positions);
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
  for (long long r = r0 + s.lane; r < r1; r += s.lanes) {
    float v[V] = {};
    if (r < live) {
      load_pack<T, V>(x + r * a.channels, v);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = activate(__builtin_fmaf(v[i] - mean[i], mul[i], add[i]), a.act);
    }
    store_pack<T, V>(y + r * a.channels, v);
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
__global__ __launch_bounds__(64) void norm_grad_join_kernel(NormArgs a, int splits, float* joined) {
  const long long n = blockIdx.x / a.groups;
  const int g = (int)(blockIdx.x % a.groups), each = a.channels / a.groups;
  float u = 0.0f, q = 0.0f;
  for (long long i = threadIdx.x; i < (long long)splits * each; i += 64) {
    const int c = g * each + (int)(i % each);
    const float* src = a.ws + (n * splits + i / each) * 2 * a.channels + c;
    const float w = a.weight ? a.weight[c] : 1.0f;
    u = __builtin_fmaf(w, src[0], u);
    q = __builtin_fmaf(w, src[a.channels], q);
  }
#pragma unroll
  for (int o = 32; o > 0; o /= 2) u += __shfl_down(u, o), q += __shfl_down(q, o);
  if (threadIdx.x == 0) {
    const float count = (float)live_positions(a, n) * (float)each;
    joined[2 * blockIdx.x] = count > 0.0f ? u / count : 0.0f;
    joined[2 * blockIdx.x + 1] = count > 0.0f ? q / count : 0.0f;
  }
}

// dbias[c], dweight[c]: 32 channels a workgroup, the partials of all samples and splits in a fixed order
__global__ __launch_bounds__(256) void norm_weight_grad_kernel(NormArgs a, long long parts) {
  __shared__ float red[2][8][32];
  const int c = blockIdx.x * 32 + threadIdx.x % 32, lane = threadIdx.x / 32;
  float u = 0.0f, q = 0.0f;
  if (c < a.channels)
    for (long long i = lane; i < parts; i += 8) {
      const float* src = a.ws + i * 2 * a.channels + c;
      u += src[0];
      q += src[a.channels];
    }
  red[0][lane][threadIdx.x % 32] = u;
  red[1][lane][threadIdx.x % 32] = q;
  __syncthreads();
  if (lane == 0 && c < a.channels) {
    for (int l = 1; l < 8; ++l) u += red[0][l][threadIdx.x], q += red[1][l][threadIdx.x];
    if (a.dbias) a.dbias[c] = u;
    if (a.dweight) a.dweight[c] = q;
  }
}

template <typename T, int V>
__global__ __launch_bounds__(kNormThreads) void norm_grad_kernel(NormArgs a, long long rows_each, unsigned splits, const float* joined) {
  const Slab s = slab_of<V>(a.channels);
  if (!s.on) return;
  const long long n = blockIdx.x / splits, live = live_positions(a, n);
  const long long r0 = (blockIdx.x % splits) * rows_each, r1 = min(r0 + rows_each, a.positions);
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

// rows of a workgroup: about 2048 workgroups in all, at least 32 rows each, at most 65535 splits
static long long norm_rows_each(const NormArgs& a) {
  const long long want = std::max(1LL, 2048 / std::max(1LL, a.batch));
  const long long splits = std::min({want, std::max(1LL, a.positions / 32), 65535LL});
  return (a.positions + splits - 1) / splits;
}
static long long norm_splits(const NormArgs& a) {
  const long long each = norm_rows_each(a);
  return (a.positions + each - 1) / each;
}

size_t norm_workspace_bytes(const NormArgs& a, bool backward) {
  if (a.batch == 0 || a.positions == 0) return 0;
  const size_t parts = (size_t)a.batch * norm_splits(a) * 2 * a.channels;
  return sizeof(float) * (parts + (backward ? (size_t)a.batch * a.groups * 2 : 0));
}

template <typename T>
static bool norm_vectors(const NormArgs& a) {
  constexpr int V = 16 / sizeof(T);
  const uintptr_t any = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.dy);
  return a.channels % V == 0 && any % 16 == 0;
}

template <typename T, int V>
static hipError_t forward_launch(const NormArgs& a) {
  const long long each = norm_rows_each(a), splits = norm_splits(a);
  const int vecs = a.channels / V;
  const dim3 grid((unsigned)(splits * a.batch), 1, (unsigned)((vecs + kNormThreads - 1) / kNormThreads)), block(kNormThreads);
  hipLaunchKernelGGL((norm_stats_kernel<T, V>), grid, block, 0, a.stream, a, each, (unsigned)splits);
  hipLaunchKernelGGL(norm_join_kernel, dim3((unsigned)(a.batch * a.groups)), dim3(64), 0, a.stream, a, (int)splits, each);
  hipLaunchKernelGGL((norm_apply_kernel<T, V>), grid, block, 0, a.stream, a, each, (unsigned)splits);
  return hipGetLastError();
}

template <typename T, int V>
static hipError_t backward_launch(const NormArgs& a) {
  const long long each = norm_rows_each(a), splits = norm_splits(a);
  const int vecs = a.channels / V;
  const dim3 grid((unsigned)(splits * a.batch), 1, (unsigned)((vecs + kNormThreads - 1) / kNormThreads)), block(kNormThreads);
  float* joined = a.ws + (size_t)a.batch * splits * 2 * a.channels;
  hipLaunchKernelGGL((norm_grad_sums_kernel<T, V>), grid, block, 0, a.stream, a, each, (unsigned)splits);
  hipLaunchKernelGGL(norm_grad_join_kernel, dim3((unsigned)(a.batch * a.groups)), dim3(64), 0, a.stream, a, (int)splits, joined);
  if (a.dweight || a.dbias)
    hipLaunchKernelGGL(norm_weight_grad_kernel, dim3((a.channels + 31) / 32), dim3(256), 0, a.stream, a, a.batch * splits);
  hipLaunchKernelGGL((norm_grad_kernel<T, V>), grid, block, 0, a.stream, a, each, (unsigned)splits, joined);
  return hipGetLastError();
}

template <typename T>
static hipError_t norm_typed(const NormArgs& a, bool backward) {
  constexpr int V = 16 / sizeof(T);
  if (norm_vectors<T>(a)) return backward ? backward_launch<T, V>(a) : forward_launch<T, V>(a);
  return backward ? backward_launch<T, 1>(a) : forward_launch<T, 1>(a);
}

static hipError_t norm_any(const NormArgs& a, bool backward) {
  if (a.dtype == 0) return norm_typed<float>(a, backward);
  return a.dtype == 1 ? norm_typed<__bf16>(a, backward) : norm_typed<_Float16>(a, backward);
}

hipError_t launch_norm_forward(const NormArgs& a) { return norm_any(a, false); }
hipError_t launch_norm_backward(const NormArgs& a) { return norm_any(a, true); }

}  // namespace tfa
