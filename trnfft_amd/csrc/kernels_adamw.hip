// AdamW (decoupled weight decay) over many tensors in few launches.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// States are fp32, or 8-bit codes with one fp32 scale s (the largest magnitude) per block of 256 values:
//   m = s sgn(c) (c / 127)^2,  v = s (c / 255)^4,   c = round(127 sqrt(|m| / s)),  c = round(255 (v / s)^(1/4)), 1 at least where v > 0.
// (c over its top is c times the rounded reciprocal.)  The square law spends the codes where moments are (their logarithm is what varies): a step is 1.6 % of a value at the
// top of a block and values down to 6e-5 (m) and 2e-10 (v) of it keep a code.  v's are the squares of m's in range, but the two scales
// fall at different rates (beta1, beta2): behind an outlier a value's m has a code again long before its v would have one, and an update by
// m over a v of zero is thousands of lr.  So no v is lost: the least one stands for 2e-10 of the block's largest, and smaller ones update by
// less.  (What codes to nearest still do: v stays where a step changes it by less than half a code, so that a value next to one 1e3 to 1e5 times
// larger may update by up to 13 lr where fp32 states give 1, until the larger one's share of the scale is forgotten.)
// A step decodes, updates in fp32 from the decoded values, uses the
// unrounded m and v for the parameter, and only then encodes.  m, v and the codes are what IEEE fp32 operations in the
// written order give (no contraction): they do not depend on the compiler.
// Memory bound: 28 bytes a value with fp32 parameters and states, 16 with 8-bit states.
#include <type_traits>

#include "model_ops.h"

#pragma clang fp contract(off)

namespace tfa {

constexpr int kQBlock = 256;       // values of a scale
constexpr int kAdamChunk = 4096;   // values of a workgroup: 4 waves of 4 blocks; with 8-bit states 2 blocks
constexpr int adam_chunk(int bits) { return bits == 8 ? kAdamChunk / 2 : kAdamChunk; }
constexpr int kAdamTensors = 52;   // per launch: their table travels in the kernel's arguments (4 KB at most)

struct AdamTable {
  AdamTensor t[kAdamTensors];
  unsigned first[kAdamTensors];  // first workgroup
  int count;
};
static_assert(sizeof(AdamTable) + sizeof(AdamArgs) <= 4000, "kernel arguments");

// four consecutive values: one access where `whole` (aligned, all inside), else one by one below n
template <typename T>
struct __attribute__((aligned(4 * sizeof(T)))) Four {
  T v[4];
};
template <typename T>
__device__ __forceinline__ Four<T> load4(const T* p, long long i, long long n, bool whole) {
  if (whole) return *reinterpret_cast<const Four<T>*>(p + i);
  Four<T> x;
#pragma unroll
  for (int j = 0; j < 4; ++j) x.v[j] = i + j < n ? p[i + j] : T(0);
  return x;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, long long i, long long n, bool whole, const Four<T>& x) {
  if (whole) {
    *reinterpret_cast<Four<T>*>(p + i) = x;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) p[i + j] = x.v[j];
  }
}

__device__ __forceinline__ float code_value(int c, float top, float s, bool fourth) {
  float t = (float)c * (1.0f / top);  // the rounded reciprocal: part of the format
  t = t * fabsf(t);
  if (fourth) t = t * t;
  return t * s;
}
// Magnitudes compare as their bits; a NaN is above infinity, so it becomes the block's scale and the block decodes to NaN.
// Within rows of 16 lanes by lane permutations, over the rows in scalar registers: no shared memory.
__device__ __forceinline__ unsigned wave_max(unsigned x) {
  x = max(x, (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 15, 15, true));   // lanes 1 apart
  x = max(x, (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 15, 15, true));   // 2 apart
  x = max(x, (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x141, 15, 15, true));  // mirrored halves of a row
  x = max(x, (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x140, 15, 15, true));  // mirrored rows
  const unsigned a = __builtin_amdgcn_readlane((int)x, 0), b = __builtin_amdgcn_readlane((int)x, 16);
  const unsigned c = __builtin_amdgcn_readlane((int)x, 32), d = __builtin_amdgcn_readlane((int)x, 48);
  return max(max(a, b), max(c, d));
}
// the code by its definition: IEEE division, roots and product, each rounded
__device__ __forceinline__ int code_of_place(float c, float x, float top) {
  return c <= top ? (x < 0.0f ? -(int)c : (int)c) : 0;  // NaN: 0 (the scale says it)
}
__device__ __forceinline__ int root_place(float x, float s, float top, bool fourth) {
  float t = sqrtf(fabsf(x) / s);
  if (fourth) t = sqrtf(t);
  float c = s > 0.0f ? rintf(t * top) : 0.0f;
  if (fourth && c == 0.0f && x > 0.0f && s < __builtin_inff()) c = 1.0f;
  return code_of_place(c, x, top);
}
// four codes by the definition, a byte each (out of line: seldom run)
template <bool SQUARES>
__device__ __noinline__ unsigned root_places(float x0, float x1, float x2, float x3, float s) {
  constexpr float top = SQUARES ? 255.0f : 127.0f;
  unsigned r = root_place(x0, s, top, SQUARES) & 255;
  r |= (root_place(x1, s, top, SQUARES) & 255) << 8;
  r |= (root_place(x2, s, top, SQUARES) & 255) << 16;
  return r | (unsigned)root_place(x3, s, top, SQUARES) << 24;
}
// The same four codes by approximate division and roots wherever they are kDoubt of a step and more from the middle between two codes
// (relative errors of 2^-23 for the quotient, each root and the product, halved by each root: 2e-4 of a
// step at most); where one of a wave's is not, by the definition: one wave's block in seven.  inv: approximate 1 / s, 0
// where s is 0 or not normal enough for it (the definition decides then).
constexpr float kDoubt = 2.5e-4f;
template <bool SQUARES>
__device__ __forceinline__ unsigned value_codes(const float (&x)[4], float s, float inv) {
  constexpr float top = SQUARES ? 255.0f : 127.0f;
  unsigned r = 0;
  float least = 1.0f;  // distance from a middle
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float t = __builtin_amdgcn_sqrtf(fabsf(x[j]) * inv);
    if (SQUARES) t = __builtin_amdgcn_sqrtf(t);
    const float u = t * top;
    least = fminf(least, fabsf(__builtin_amdgcn_fractf(u) - 0.5f));
    int c = (int)rintf(u);
    if (SQUARES) c = max(c, x[j] > 0.0f ? 1 : 0);
    r |= (unsigned)((!SQUARES && x[j] < 0.0f ? -c : c) & 255) << (8 * j);
  }
  if (__any(!(least > kDoubt)) || inv == 0.0f) r = root_places<SQUARES>(x[0], x[1], x[2], x[3], s);
  return r;
}
__device__ __forceinline__ float scale_inverse(float s) { return s > 1e-30f && s < 1e30f ? __builtin_amdgcn_rcpf(s) : 0.0f; }

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
struct StateTypes {
  typedef float M;
  typedef float V;
};
template <>
struct StateTypes<8> {
  typedef signed char M;
  typedef unsigned char V;
};

// A wave takes blocks of 256 of one tensor, a lane four neighbours of each: 16-byte accesses for fp32, and all of a wave's loads
// ahead of its arithmetic, with fp32 states four blocks.  With 8-bit states two: their arithmetic (five roots and reciprocals
// a value) then leaves eight waves a SIMD to overlap it with other waves' loads; four blocks took 457 us where two take 350
// (50 tensors of 2.4M fp32 values: 5.5 TB/s), and the wave's whole block decides by itself whether its codes need the
// definition (a branch for each value took 100 us more).  bfloat16 parameters and gradients: 353 us, bound by that arithmetic.
// fp32 states: 5.0 TB/s, as a large copy (17.4M values with bf16 parameters and masters 97 us).
template <int BITS, typename P, typename G>
__global__ __launch_bounds__(256) void adamw_kernel(AdamTable tab, AdamArgs a) {
  typedef typename StateTypes<BITS>::M M;
  typedef typename StateTypes<BITS>::V V;
  constexpr int kChunk = adam_chunk(BITS), U = kChunk / kQBlock / 4;
  const int k = tensor_of(tab.first, tab.count, blockIdx.x);
  const AdamTensor& t = tab.t[k];
  const long long n = t.n, base = (long long)(blockIdx.x - tab.first[k]) * kChunk;
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  P* const tp = static_cast<P*>(t.p);
  const G* const tg = static_cast<const G*>(t.g);
  M* const tm = static_cast<M*>(t.m);
  V* const tv = static_cast<V*>(t.v);
  float* const master = t.master;
  const uintptr_t odd = reinterpret_cast<uintptr_t>(tp) % (4 * sizeof(P)) | reinterpret_cast<uintptr_t>(tg) % (4 * sizeof(G)) |
                        reinterpret_cast<uintptr_t>(tm) % (4 * sizeof(M)) | reinterpret_cast<uintptr_t>(tv) % (4 * sizeof(V)) |
                        reinterpret_cast<uintptr_t>(master) % 16;
  const bool whole = odd == 0 && base + kChunk <= n;

  Four<P> p4[U];
  Four<float> w4[U];
  Four<G> g4[U];
  Four<M> m4[U];
  Four<V> v4[U];
  float ms[U], vs[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long start = base + (wave + 4 * u) * kQBlock, i = start + lane * 4;
    if (master)
      w4[u] = load4(master, i, n, whole);
    else
      p4[u] = load4(tp, i, n, whole);
    g4[u] = load4(tg, i, n, whole);
    m4[u] = load4(tm, i, n, whole);
    v4[u] = load4(tv, i, n, whole);
    ms[u] = vs[u] = 0.0f;
    if (BITS == 8 && start < n) ms[u] = t.m_scale[start / kQBlock], vs[u] = t.v_scale[start / kQBlock];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long start = base + (wave + 4 * u) * kQBlock, i = start + lane * 4;
    if (start >= n) break;
    Four<float> mo, vo, po;
    unsigned top_m = 0, top_v = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float g = to_f32(g4[u].v[j]);
      float m = BITS == 8 ? code_value((int)m4[u].v[j], 127.0f, ms[u], false) : (float)m4[u].v[j];
      float v = BITS == 8 ? code_value((int)v4[u].v[j], 255.0f, vs[u], true) : (float)v4[u].v[j];
      m = m * a.beta1 + g * a.one_beta1;
      v = v * a.beta2 + (g * g) * a.one_beta2;
      const float p = master ? w4[u].v[j] : to_f32(p4[u].v[j]);
      // (root and quotient of the step are the hardware's, 1 ulp each: 1e-7 of a step)
      po.v[j] = p * a.decay - a.step_size * (m * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v) * a.inv_root_bc2 + a.eps));
      mo.v[j] = m;
      vo.v[j] = v;
      if (i + j < n) {  // (past the end: nothing may enter the block's scale)
        top_m = max(top_m, __float_as_uint(fabsf(m)));
        top_v = max(top_v, __float_as_uint(fabsf(v)));
      }
    }
    if (master) store4(master, i, n, whole, po);
    Four<P> pr;
#pragma unroll
    for (int j = 0; j < 4; ++j) pr.v[j] = from_f32<P>(po.v[j]);
    store4(tp, i, n, whole, pr);
    if constexpr (BITS == 32) {
      store4(tm, i, n, whole, mo);
      store4(tv, i, n, whole, vo);
    } else {
      const float sm = __uint_as_float(wave_max(top_m)), sv = __uint_as_float(wave_max(top_v));
      const float im = scale_inverse(sm), iv = scale_inverse(sv);
      store4(tm, i, n, whole, __builtin_bit_cast(Four<M>, value_codes<false>(mo.v, sm, im)));
      store4(tv, i, n, whole, __builtin_bit_cast(Four<V>, value_codes<true>(vo.v, sv, iv)));
      if (lane == 0) {
        t.m_scale[start / kQBlock] = sm;
        t.v_scale[start / kQBlock] = sv;
      }
    }
  }
}

template <int BITS, typename P>
static void adamw_typed(const AdamTable& tab, const AdamArgs& a, unsigned blocks, hipStream_t stream) {
  if (a.g_dtype == a.p_dtype)
    hipLaunchKernelGGL((adamw_kernel<BITS, P, P>), dim3(blocks), dim3(256), 0, stream, tab, a);
  else
    hipLaunchKernelGGL((adamw_kernel<BITS, P, float>), dim3(blocks), dim3(256), 0, stream, tab, a);
}
template <int BITS>
static void adamw_bits(const AdamTable& tab, const AdamArgs& a, unsigned blocks, hipStream_t stream) {
  if (a.p_dtype == 0)
    hipLaunchKernelGGL((adamw_kernel<BITS, float, float>), dim3(blocks), dim3(256), 0, stream, tab, a);
  else if (a.p_dtype == 1)
    adamw_typed<BITS, __bf16>(tab, a, blocks, stream);
  else
    adamw_typed<BITS, _Float16>(tab, a, blocks, stream);
}

hipError_t launch_adamw(const AdamTensor* tensors, long long count, const AdamArgs& a, hipStream_t stream) {
  const int chunk = adam_chunk(a.bits);
  for (long long i = 0; i < count;) {
    AdamTable tab;
    tab.count = 0;
    long long blocks = 0;
    while (i < count && tab.count < kAdamTensors) {
      const AdamTensor& t = tensors[i];
      const long long more = (t.n + chunk - 1) / chunk;
      if (blocks + more > max_blocks(256)) break;
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
      adamw_bits<8>(tab, a, (unsigned)blocks, stream);
    else
      adamw_bits<32>(tab, a, (unsigned)blocks, stream);
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
  typedef typename StateTypes<8>::M S;
  typedef typename StateTypes<8>::V U;
  typedef std::conditional_t<SQUARES, U, S> Code;
  const Code* codes = static_cast<const Code*>(t.codes);
  const bool whole = base + kAdamChunk <= t.n && reinterpret_cast<uintptr_t>(codes) % 4 == 0 && reinterpret_cast<uintptr_t>(t.out) % 16 == 0;
  Four<Code> c[4];
  float s[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const long long i = base + u * 1024 + threadIdx.x * 4;
    c[u] = load4(codes, i, t.n, whole);
    s[u] = i < t.n ? t.scales[i / kQBlock] : 0.0f;
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const long long i = base + u * 1024 + threadIdx.x * 4;
    Four<float> x;
#pragma unroll
    for (int j = 0; j < 4; ++j) x.v[j] = code_value((int)c[u].v[j], SQUARES ? 255.0f : 127.0f, s[u], SQUARES);
    store4(t.out, i, t.n, whole, x);
  }
}

hipError_t launch_adam_values(const CodeTensor* tensors, long long count, bool squares, hipStream_t stream) {
  for (long long i = 0; i < count;) {
    CodeTable tab;
    tab.count = 0;
    long long blocks = 0;
    while (i < count && tab.count < kCodeTensors) {
      const long long more = (tensors[i].n + kAdamChunk - 1) / kAdamChunk;
      if (blocks + more > max_blocks(256)) break;
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
