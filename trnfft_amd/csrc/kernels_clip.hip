// The global norm of many tensors' gradients and their clipping, in few launches.
//
//   norm = sqrt(sum of all g^2),  g = g min(1, max_norm / (norm + 1e-6))
//
// Squares are summed in 64 bits: they neither overflow nor vanish for any finite fp32 gradient, and a sum over 10^8 of them
// is exact to the norm's last bit (conversions and 64-bit products run at the vector units' ordinary rate, and one a value is
// far below what the memory's rate leaves room for).  Every workgroup leaves one sum; they are added in one order: the
// norm does not depend on timing.  Memory bound: one reading for the norm, one reading and writing where gradients are scaled.
// 120M bf16 values in 320 tensors: 51 us for the squares (4.7 TB/s), 80 for scaling (6.0 TB/s: a part is in the caches still); 24 tensors of 0.5M
// fp32 values together 4.0 and 4.3, which is two launches.
#include "model_ops.h"

#include <algorithm>

namespace tfa {

constexpr int kGradTensors = 180;  // per launch: their table travels in the kernel's arguments (4 KB at most)
// Values of a workgroup: as many as make about kGradBlocks workgroups (small models: no fewer than keep the compute units busy; large ones: the
// loads of a next batch cover the sums of this one)
constexpr int kLeastChunk = 4096, kMostChunk = 65536;
constexpr long long kGradBlocks = 2048;
// Parts that every scaling workgroup adds up by itself; more are added in a launch of its own before.  bf16, norm and scaling: 120M values (1831
// parts) 126 us both ways, 12M fp32 17 by themselves and 19 in a launch, 1000M (15258) 1185 and 1181, 2000M (30517) 2366 and 2277, 7000M (106811)
// 10283 and 7903: together they read the square of their number.
constexpr long long kGradParts = 16384;

struct GradTable {
  GradTensor t[kGradTensors];
  unsigned first[kGradTensors];  // first workgroup
  int count, chunk;
};
static_assert(sizeof(GradTable) <= 3900, "kernel arguments");

__device__ __forceinline__ int grad_tensor_of(const GradTable& tab, unsigned block) {
  int lo = 0, hi = tab.count;  // the last tensor whose first workgroup is not past this one
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (tab.first[mid] <= block)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// sum over the workgroup's 256 threads, in all of them
__device__ __forceinline__ double block_sum(double x) {
  __shared__ double parts[4];
#pragma unroll
  for (int d = 32; d; d /= 2) x += __shfl_xor(x, d, 64);
  if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = x;
  __syncthreads();
  return parts[0] + parts[1] + parts[2] + parts[3];
}

// a workgroup's stretch of a tensor: `head` values up to a 16-byte boundary, `vectors` of 16 bytes, and what is left behind them
template <typename T>
struct GradStretch {
  static constexpr int V = 16 / (int)sizeof(T);
  T* p;
  int n, head, vectors;
  __device__ __forceinline__ GradStretch(const GradTable& tab) {
    const int k = grad_tensor_of(tab, blockIdx.x);
    const long long base = (long long)(blockIdx.x - tab.first[k]) * tab.chunk;
    p = static_cast<T*>(tab.t[k].p) + base;
    n = (int)min((long long)tab.chunk, tab.t[k].n - base);
    head = min(n, (int)((16 - reinterpret_cast<uintptr_t>(p) % 16) % 16 / sizeof(T)));
    vectors = (n - head) / V;
  }
  // f on every value that is in no vector
  template <typename F>
  __device__ __forceinline__ void rest(F f) const {
    const int behind = head + vectors * V;
    if ((int)threadIdx.x < head) f(p[threadIdx.x]);
    if ((int)threadIdx.x < n - behind) f(p[behind + threadIdx.x]);  // (less than a vector)
  }
};
constexpr int kGradBatch = 4;  // vectors of a thread whose loads are on their way together

template <typename T>
__global__ __launch_bounds__(256) void grad_squares_kernel(GradTable tab, double* parts) {
  constexpr int V = GradStretch<T>::V;
  const GradStretch<T> s(tab);
  const Pack<T, V>* const v = reinterpret_cast<const Pack<T, V>*>(s.p + s.head);
  const auto load = [&](int i, Pack<T, V>(&x)[kGradBatch]) {
#pragma unroll
    for (int u = 0; u < kGradBatch; ++u) {
      const int at = i + u * 256 + threadIdx.x;
      x[u] = at < s.vectors ? v[at] : Pack<T, V>{};
    }
  };
  double sum = 0.0;
  Pack<T, V> x[kGradBatch], next[kGradBatch];
  load(0, x);
  for (int i = 0; i < s.vectors; i += kGradBatch * 256) {
    load(i + kGradBatch * 256, next);
#pragma unroll
    for (int u = 0; u < kGradBatch; ++u) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const double g = to_f32(x[u].v[j]);
        sum = __builtin_fma(g, g, sum);
      }
      x[u] = next[u];
    }
  }
  s.rest([&](const T& value) {
    const double g = to_f32(value);
    sum = __builtin_fma(g, g, sum);
  });
  sum = block_sum(sum);
  if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

__device__ __forceinline__ double sum_of_parts(const double* parts, long long count) {
  double sum = 0.0;
#pragma unroll 8
  for (long long i = threadIdx.x; i < count; i += 256) sum += parts[i];
  return block_sum(sum);
}
__device__ __forceinline__ double norm_of_parts(const double* parts, long long count) { return sqrt(sum_of_parts(parts, count)); }

__global__ __launch_bounds__(256) void grad_norm_kernel(const double* parts, long long count, float* norm) {
  const double root = norm_of_parts(parts, count);
  if (threadIdx.x == 0) norm[0] = (float)root;
}

// the sum in place of the first part
__global__ __launch_bounds__(256) void grad_sum_kernel(double* parts, long long count) {
  const double sum = sum_of_parts(parts, count);
  if (threadIdx.x == 0) parts[0] = sum;
}

// Every workgroup adds the parts itself, in the same order: one launch less, for up to kGradParts values out of the caches.
template <typename T>
__global__ __launch_bounds__(256) void grad_scale_kernel(GradTable tab, const double* parts, long long count, double max_norm, float* norm) {
  constexpr int V = GradStretch<T>::V;
  const double root = norm_of_parts(parts, count), ratio = max_norm / (root + 1e-6);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)root;
  if (ratio >= 1.0) return;  // times one: what is there  (a norm that is NaN makes every gradient NaN)
  const float c = (float)ratio;
  const GradStretch<T> s(tab);
  Pack<T, V>* const v = reinterpret_cast<Pack<T, V>*>(s.p + s.head);
  for (int i = threadIdx.x; i < s.vectors; i += kGradBatch * 256) {
    Pack<T, V> x[kGradBatch];
#pragma unroll
    for (int u = 0; u < kGradBatch; ++u)
      if (i + u * 256 < s.vectors) x[u] = v[i + u * 256];
#pragma unroll
    for (int u = 0; u < kGradBatch; ++u) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[u].v[j] = from_f32<T>(to_f32(x[u].v[j]) * c);
      if (i + u * 256 < s.vectors) v[i + u * 256] = x[u];
    }
  }
  s.rest([&](T& value) { value = from_f32<T>(to_f32(value) * c); });
}

static int grad_chunk(const GradLists& g) {
  long long total = 0;
  for (int d = 0; d < 3; ++d)
    for (long long i = 0; i < g.count[d]; ++i) total += g.tensors[d][i].n;
  int chunk = kLeastChunk;
  while (chunk < kMostChunk && total / chunk > kGradBlocks) chunk *= 2;
  return chunk;
}
// (a chunk is a power of two: a division a tensor in every loop over them took longer than the launches)
static long long chunks_of(const GradTensor& t, int chunk) { return (t.n + chunk - 1) >> __builtin_ctz(chunk); }

long long grad_parts(const GradLists& g) {
  const int chunk = grad_chunk(g);
  long long total = 0;
  for (int d = 0; d < 3; ++d)
    for (long long i = 0; i < g.count[d]; ++i) total += chunks_of(g.tensors[d][i], chunk);
  return std::max(1LL, total);
}

// f(table, workgroups, workgroups before it) for all tensors of a dtype, as many in a launch as the arguments and the grid hold
template <typename F>
static hipError_t each_table(const GradTensor* tensors, long long count, int chunk, long long& before, F f) {
  for (long long i = 0; i < count;) {
    GradTable tab;
    tab.count = 0;
    tab.chunk = chunk;
    long long blocks = 0;
    while (i < count && tab.count < kGradTensors) {
      const long long more = chunks_of(tensors[i], chunk);
      if (blocks + more > max_blocks(256)) break;
      if (more) {
        tab.t[tab.count] = tensors[i];
        tab.first[tab.count++] = (unsigned)blocks;
        blocks += more;
      }
      ++i;
    }
    if (!tab.count) {
      if (i < count) return hipErrorInvalidValue;  // one tensor past the grid
      break;
    }
    f(tab, (unsigned)blocks, before);
    before += blocks;
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_grad_norm(const GradLists& g, double* parts, float* norm, bool scale, double max_norm, hipStream_t stream) {
  const int chunk = grad_chunk(g);
  long long done = 0;
  for (int d = 0; d < 3; ++d) {
    const hipError_t e = each_table(g.tensors[d], g.count[d], chunk, done, [&](const GradTable& tab, unsigned blocks, long long before) {
      const auto kernel = d == 0 ? grad_squares_kernel<float> : d == 1 ? grad_squares_kernel<__bf16> : grad_squares_kernel<_Float16>;
      hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, stream, tab, parts + before);
    });
    if (e != hipSuccess) return e;
  }
  if (!scale || !done) {
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(256), 0, stream, parts, done, norm);
    return hipGetLastError();
  }
  if (done > kGradParts) {
    hipLaunchKernelGGL(grad_sum_kernel, dim3(1), dim3(256), 0, stream, parts, done);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    done = 1;
  }
  for (int d = 0; d < 3; ++d) {
    long long before = 0;
    const hipError_t e = each_table(g.tensors[d], g.count[d], chunk, before, [&](const GradTable& tab, unsigned blocks, long long) {
      const auto kernel = d == 0 ? grad_scale_kernel<float> : d == 1 ? grad_scale_kernel<__bf16> : grad_scale_kernel<_Float16>;
      hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, stream, tab, parts, done, max_norm, norm);
    });
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace tfa
