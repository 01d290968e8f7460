// AdamW (decoupled weight decay) over many tensors in few launches.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// States are fp32, or 8-bit codes with one fp32 scale s (the largest magnitude) per block of 256 values:
//   m = s sgn(c) (c / 127)^2,  v = s (c / 255)^4,   c = round(127 sqrt(|m| / s)),  c = round(255 (v / s)^(1/4)).
// (c over its top is c times the rounded reciprocal.)  The square law spends the codes where moments are (their logarithm is what varies): a step is 1.6 % of a value at the
// top of a block and values down to 6e-5 (m) and 2e-10 (v) of it keep a code; v's are the squares of m's in range, so that
// a value's m rounds to zero before its v does.  A step decodes, updates in fp32 from the decoded values, uses the
// unrounded m and v for the parameter, and only then encodes.  Every operation is one IEEE fp32 operation in
// the written order (no contraction): codes do not depend on the compiler.
// Memory bound: 28 bytes a value with fp32 parameters and states, 16 with 8-bit states.
#include "model_ops.h"

#pragma clang fp contract(off)

namespace tfa {

constexpr int kQBlock = 256;       // values of a scale
constexpr int kAdamChunk = 4096;   // values of a workgroup: 4 waves of 4 blocks
constexpr int kAdamTensors = 52;   // per launch: their table travels in the kernel's arguments (4 KB at most)

struct AdamTable {
  AdamTensor t[kAdamTensors];
  unsigned first[kAdamTensors];  // first workgroup
  int count;
};
static_assert(sizeof(AdamTable) + sizeof(AdamArgs) <= 4000, "kernel arguments");

__device__ __forceinline__ float load_as_f32(const void* p, int dtype, long long i) {
  if (dtype == 0) return static_cast<const float*>(p)[i];
  return dtype == 1 ? to_f32(static_cast<const __bf16*>(p)[i]) : to_f32(static_cast<const _Float16*>(p)[i]);
}
__device__ __forceinline__ void store_from_f32(void* p, int dtype, long long i, float x) {
  if (dtype == 0)
    static_cast<float*>(p)[i] = x;
  else if (dtype == 1)
    static_cast<__bf16*>(p)[i] = from_f32<__bf16>(x);
  else
    static_cast<_Float16*>(p)[i] = from_f32<_Float16>(x);
}

__device__ __forceinline__ float code_value(int c, float top, float s, bool fourth) {
  float t = (float)c * (1.0f / top);  // the rounded reciprocal: part of the format
  t = t * fabsf(t);
  if (fourth) t = t * t;
  return t * s;
}
// magnitudes compare as their bits; a NaN is above infinity, so it becomes the block's scale and the block decodes to NaN
__device__ __forceinline__ unsigned wave_max(unsigned x) {
#pragma unroll
  for (int o = 32; o > 0; o /= 2) x = max(x, (unsigned)__shfl_xor((int)x, o));
  return x;
}
__device__ __forceinline__ int value_code(float x, float s, float top, bool fourth) {
  const float r = s > 0.0f ? fabsf(x) / s : 0.0f;
  float t = sqrtf(r);
  if (fourth) t = sqrtf(t);
  t = rintf(t * top);
  return t <= top ? (x < 0.0f ? -(int)t : (int)t) : 0;  // NaN: 0 (the scale says it)
}

__device__ __forceinline__ int tensor_of(const unsigned* first, int count, unsigned block) {
  int lo = 0, hi = count;  // the last tensor whose first workgroup is not past this one
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first[mid] <= block)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

template <int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(AdamTable tab, AdamArgs a) {
  const int k = tensor_of(tab.first, tab.count, blockIdx.x);
  const AdamTensor& t = tab.t[k];
  const long long base = (long long)(blockIdx.x - tab.first[k]) * kAdamChunk;
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  for (int q = wave; q < kAdamChunk / kQBlock; q += 4) {
    const long long start = base + (long long)q * kQBlock;
    if (start >= t.n) break;
    float ms = 0.0f, vs = 0.0f;
    if (BITS == 8) ms = t.m_scale[start / kQBlock], vs = t.v_scale[start / kQBlock];
    float mm[4], vv[4];
    unsigned top_m = 0, top_v = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long i = start + lane * 4 + j;
      mm[j] = vv[j] = 0.0f;
      if (i >= t.n) continue;
      const float g = load_as_f32(t.g, a.g_dtype, i);
      float m, v;
      if (BITS == 8) {
        m = code_value(static_cast<const signed char*>(t.m)[i], 127.0f, ms, false);
        v = code_value(static_cast<const unsigned char*>(t.v)[i], 255.0f, vs, true);
      } else {
        m = static_cast<const float*>(t.m)[i];
        v = static_cast<const float*>(t.v)[i];
      }
      m = m * a.beta1 + g * a.one_beta1;
      v = v * a.beta2 + (g * g) * a.one_beta2;
      float p = t.master ? t.master[i] : load_as_f32(t.p, a.p_dtype, i);
      p = p * a.decay - a.step_size * (m / (sqrtf(v) / a.root_bc2 + a.eps));
      if (t.master) t.master[i] = p;
      store_from_f32(t.p, a.p_dtype, i, p);
      if (BITS == 32) {
        static_cast<float*>(t.m)[i] = m;
        static_cast<float*>(t.v)[i] = v;
      }
      mm[j] = m;
      vv[j] = v;
      top_m = max(top_m, __float_as_uint(fabsf(m)));
      top_v = max(top_v, __float_as_uint(fabsf(v)));
    }
    if (BITS == 8) {
      const float sm = __uint_as_float(wave_max(top_m)), sv = __uint_as_float(wave_max(top_v));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long i = start + lane * 4 + j;
        if (i >= t.n) continue;
        static_cast<signed char*>(t.m)[i] = (signed char)value_code(mm[j], sm, 127.0f, false);
        static_cast<unsigned char*>(t.v)[i] = (unsigned char)value_code(vv[j], sv, 255.0f, true);
      }
      if (lane == 0) {
        t.m_scale[start / kQBlock] = sm;
        t.v_scale[start / kQBlock] = sv;
      }
    }
  }
}

hipError_t launch_adamw(const AdamTensor* tensors, long long count, const AdamArgs& a, hipStream_t stream) {
  for (long long i = 0; i < count;) {
    AdamTable tab;
    tab.count = 0;
    unsigned long long blocks = 0;
    while (i < count && tab.count < kAdamTensors) {
      const AdamTensor& t = tensors[i];
      const unsigned long long more = (unsigned long long)((t.n + kAdamChunk - 1) / kAdamChunk);
      if (blocks + more > 0x7fffffffull) break;
      if (more) {
        tab.t[tab.count] = t;
        tab.first[tab.count++] = (unsigned)blocks;
        blocks += more;
      }
      ++i;
    }
    if (!tab.count) {
      if (i < count) return hipErrorInvalidValue;  // one tensor past the grid
      break;
    }
    if (a.bits == 8)
      hipLaunchKernelGGL(adamw_kernel<8>, dim3((unsigned)blocks), dim3(256), 0, stream, tab, a);
    else
      hipLaunchKernelGGL(adamw_kernel<32>, dim3((unsigned)blocks), dim3(256), 0, stream, tab, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

constexpr int kCodeTensors = 104;
struct CodeTable {
  CodeTensor t[kCodeTensors];
  unsigned first[kCodeTensors];
  int count;
};
static_assert(sizeof(CodeTable) <= 4000, "kernel arguments");

template <bool SQUARES>
__global__ __launch_bounds__(256) void adam_values_kernel(CodeTable tab) {
  const int k = tensor_of(tab.first, tab.count, blockIdx.x);
  const CodeTensor& t = tab.t[k];
  const long long base = (long long)(blockIdx.x - tab.first[k]) * kAdamChunk;
  for (long long i = base + threadIdx.x; i < min(base + kAdamChunk, t.n); i += 256) {
    const int c = SQUARES ? (int)static_cast<const unsigned char*>(t.codes)[i] : (int)static_cast<const signed char*>(t.codes)[i];
    t.out[i] = code_value(c, SQUARES ? 255.0f : 127.0f, t.scales[i / kQBlock], SQUARES);
  }
}

hipError_t launch_adam_values(const CodeTensor* tensors, long long count, bool squares, hipStream_t stream) {
  for (long long i = 0; i < count;) {
    CodeTable tab;
    tab.count = 0;
    unsigned long long blocks = 0;
    while (i < count && tab.count < kCodeTensors) {
      const unsigned long long more = (unsigned long long)((tensors[i].n + kAdamChunk - 1) / kAdamChunk);
      if (blocks + more > 0x7fffffffull) break;
      if (more) {
        tab.t[tab.count] = tensors[i];
        tab.first[tab.count++] = (unsigned)blocks;
        blocks += more;
      }
      ++i;
    }
    if (!tab.count) {
      if (i < count) return hipErrorInvalidValue;
      break;
    }
    if (squares)
      hipLaunchKernelGGL(adam_values_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, stream, tab);
    else
      hipLaunchKernelGGL(adam_values_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, stream, tab);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace tfa
