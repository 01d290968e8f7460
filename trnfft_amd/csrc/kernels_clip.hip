// The global norm of many tensors' gradients and their clipping, in few launches.
//
//   norm = sqrt(sum of all g^2),  g = g min(1, max_norm / (norm + 1e-6))
//
// Squares are summed in 64 bits: they neither overflow nor vanish for any finite fp32 gradient, and a sum over 10^8 of them
// is exact to the norm's last bit (conversions and 64-bit products run at the vector units' ordinary rate, and one a value is
// far below what the memory's rate leaves room for).  Every workgroup leaves one sum; they are added in one order by one workgroup: the
// norm does not depend on timing.  Memory bound: one reading for the norm, one reading and writing where gradients are scaled.
#include "model_ops.h"

namespace tfa {

constexpr int kGradTensors = 180;  // per launch: their table travels in the kernel's arguments (4 KB at most)
constexpr int kGradChunk = 16384;  // values of a workgroup

struct GradTable {
  GradTensor t[kGradTensors];
  unsigned first[kGradTensors];  // first workgroup
  int count;
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

// sum over the workgroup's 256 threads, in thread 0
__device__ __forceinline__ double block_sum(double x) {
  __shared__ double parts[4];
#pragma unroll
  for (int d = 32; d; d /= 2) x += __shfl_xor(x, d, 64);
  if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = x;
  __syncthreads();
  return parts[0] + parts[1] + parts[2] + parts[3];
}

template <typename T>
__global__ __launch_bounds__(256) void grad_squares_kernel(GradTable tab, double* parts) {
  constexpr int V = 16 / sizeof(T);
  const int k = grad_tensor_of(tab, blockIdx.x);
  const long long base = (long long)(blockIdx.x - tab.first[k]) * kGradChunk;
  const T* const p = static_cast<const T*>(tab.t[k].p) + base;
  const int n = (int)min((long long)kGradChunk, tab.t[k].n - base);
  double sum = 0.0;
  if (n == kGradChunk && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
    constexpr int U = 8;
#pragma unroll
    for (int i = 0; i < kGradChunk; i += U * V * 256) {
      Pack<T, V> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const Pack<T, V>*>(p + i + (u * 256 + threadIdx.x) * V);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const double g = to_f32(v[u].v[j]);
          sum = __builtin_fma(g, g, sum);
        }
    }
  } else {
    for (int i = threadIdx.x; i < n; i += 256) {
      const double g = to_f32(p[i]);
      sum = __builtin_fma(g, g, sum);
    }
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

// out[0] the norm, coef[0] what gradients are multiplied with
__global__ __launch_bounds__(256) void grad_norm_kernel(const double* parts, long long count, double max_norm, float* norm, float* coef) {
  double sum = 0.0;
  for (long long i = threadIdx.x; i < count; i += 256) sum += parts[i];
  sum = block_sum(sum);
  if (threadIdx.x == 0) {
    const double root = sqrt(sum);
    norm[0] = (float)root;
    const double c = max_norm / (root + 1e-6);
    if (coef) coef[0] = c < 1.0 || c != c ? (float)c : 1.0f;  // (a norm that is NaN makes every gradient NaN)
  }
}

template <typename T>
__global__ __launch_bounds__(256) void grad_scale_kernel(GradTable tab, const float* coef) {
  constexpr int V = 16 / sizeof(T);
  const float c = coef[0];
  if (c == 1.0f) return;  // times one: what is there
  const int k = grad_tensor_of(tab, blockIdx.x);
  const long long base = (long long)(blockIdx.x - tab.first[k]) * kGradChunk;
  T* const p = static_cast<T*>(tab.t[k].p) + base;
  const int n = (int)min((long long)kGradChunk, tab.t[k].n - base);
  if (n == kGradChunk && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
    constexpr int U = 8;
#pragma unroll
    for (int i = 0; i < kGradChunk; i += U * V * 256) {
      Pack<T, V> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const Pack<T, V>*>(p + i + (u * 256 + threadIdx.x) * V);
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[u].v[j] = from_f32<T>(to_f32(v[u].v[j]) * c);
        *reinterpret_cast<Pack<T, V>*>(p + i + (u * 256 + threadIdx.x) * V) = v[u];
      }
    }
  } else {
    for (int i = threadIdx.x; i < n; i += 256) p[i] = from_f32<T>(to_f32(p[i]) * c);
  }
}

static long long chunks_of(const GradTensor& t) { return (t.n + kGradChunk - 1) / kGradChunk; }

long long grad_parts(const GradLists& g) {
  long long total = 0;
  for (int d = 0; d < 3; ++d)
    for (long long i = 0; i < g.count[d]; ++i) total += chunks_of(g.tensors[d][i]);
  return total + 1;  // (and the factor)
}

// f(table, workgroups, workgroups before it) for all tensors of a dtype, as many in a launch as the arguments and the grid hold
template <typename F>
static hipError_t each_table(const GradTensor* tensors, long long count, long long& before, F f) {
  for (long long i = 0; i < count;) {
    GradTable tab;
    tab.count = 0;
    long long blocks = 0;
    while (i < count && tab.count < kGradTensors) {
      const long long more = chunks_of(tensors[i]);
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
  long long done = 0;
  for (int d = 0; d < 3; ++d) {
    const hipError_t e = each_table(g.tensors[d], g.count[d], done, [&](const GradTable& tab, unsigned blocks, long long before) {
      if (d == 0) hipLaunchKernelGGL(grad_squares_kernel<float>, dim3(blocks), dim3(256), 0, stream, tab, parts + before);
      if (d == 1) hipLaunchKernelGGL(grad_squares_kernel<__bf16>, dim3(blocks), dim3(256), 0, stream, tab, parts + before);
      if (d == 2) hipLaunchKernelGGL(grad_squares_kernel<_Float16>, dim3(blocks), dim3(256), 0, stream, tab, parts + before);
    });
    if (e != hipSuccess) return e;
  }
  float* const coef = scale ? reinterpret_cast<float*>(parts + done) : nullptr;
  hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(256), 0, stream, parts, done, max_norm, norm, coef);
  hipError_t e = hipGetLastError();
  for (int d = 0; d < 3 && scale && e == hipSuccess; ++d) {
    long long before = 0;
    e = each_table(g.tensors[d], g.count[d], before, [&](const GradTable& tab, unsigned blocks, long long) {
      if (d == 0) hipLaunchKernelGGL(grad_scale_kernel<float>, dim3(blocks), dim3(256), 0, stream, tab, coef);
      if (d == 1) hipLaunchKernelGGL(grad_scale_kernel<__bf16>, dim3(blocks), dim3(256), 0, stream, tab, coef);
      if (d == 2) hipLaunchKernelGGL(grad_scale_kernel<_Float16>, dim3(blocks), dim3(256), 0, stream, tab, coef);
    });
  }
  return e;
}

}  // namespace tfa
