// Causal convolution along frames with a short filter for each channel, channels last, and an activation.
//
//   pre_t = bias + sum_j w_j x_{t - W + 1 + j},  y_t = act(pre_t);  frames before the first come from a state (the last W - 1 inputs)
//   dpre_t = dy_t act'(pre_t),  dx_s = sum_j w_j dpre_{s + W - 1 - j},  dw_j = sum_t dpre_t x_{t - W + 1 + j},  db = sum_t dpre_t
//
// Memory bound: x and y once forward; x, dy and dx once backward, where pre is computed again from x.  A thread takes a vector of
// channels over a run of frames, with its window of frames in registers, so a frame is read once but for the W - 1 in front of
// (and, backward, behind) a run.  Each filter width is a kernel of its own: a wider one with taps of zero would make NaN of
// infinities outside the filter.  Frames at and past lengths[n] are padding: not read, zeros in y and dx.
#include "model_ops.h"
#include "activations.h"

#include <algorithm>

namespace tfa {

// Tokens of a thread's run: as many as leave about kConvThreads threads, the fewer the smaller the call.
constexpr long long kConvThreads = 128 << 10;
constexpr int kRunMost = 32;

__device__ __forceinline__ long long conv_end(const long long* lengths, long long row, long long tokens) {
  return lengths ? min(max(lengths[row], 0LL), tokens) : tokens;
}

// values of frame t >= -(W - 1) of a row: of the state where it is before the first, zeros where there is none
template <typename T, int V, int W>
__device__ __forceinline__ void conv_frame(const T* x, long long st, const T* state, long long channels, long long t, float (&v)[V]) {
  if (t >= 0) {
    load_pack<T, V>(x + t * st, v);
  } else if (state) {
    load_pack<T, V>(state + (t + W - 1) * channels, v);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.0f;
  }
}

template <typename T, int V, int W>
__global__ __launch_bounds__(256) void conv_forward_kernel(ConvArgs a, int vectors, long long runs, int run, long long first) {
  const long long id = (first + blockIdx.x) * 256 + threadIdx.x;
  const long long cell = id / vectors, row = cell / runs;
  if (row >= a.batch) return;
  const int c = (int)(id % vectors) * V;
  const long long t0 = cell % runs * run, t1 = min(t0 + run, a.tokens), end = conv_end(a.lengths, row, a.tokens);
  const T* const x = static_cast<const T*>(a.x) + row * a.x_sb + c;
  const T* const state = a.state_in ? static_cast<const T*>(a.state_in) + row * (W - 1) * a.channels + c : nullptr;
  T* const y = static_cast<T*>(a.y) + row * a.tokens * a.channels + c;
  if (a.state_out && t0 == 0) {  // the last W - 1 frames up to the end
    T* const out = static_cast<T*>(a.state_out) + row * (W - 1) * a.channels + c;
    for (int j = 0; j < W - 1; ++j) {
      float v[V];
      conv_frame<T, V, W>(x, a.x_st, state, a.channels, end + j - (W - 1), v);
      store_pack<T, V>(out + (long long)j * a.channels, v);
    }
  }
  float w[V][W], b[V], win[W][V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int j = 0; j < W; ++j) w[i][j] = a.weight[(long long)(c + i) * W + j];
    b[i] = a.bias ? a.bias[c + i] : 0.0f;
  }
  const long long live = min(t1, end);
  if (t0 < live) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j) conv_frame<T, V, W>(x, a.x_st, state, a.channels, t0 + j - (W - 1), win[j]);
  }
#pragma unroll 4
  for (long long t = t0; t < live; ++t) {
    load_pack<T, V>(x + t * a.x_st, win[W - 1]);
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float s = b[i];
#pragma unroll
      for (int j = 0; j < W; ++j) s = __builtin_fmaf(w[i][j], win[j][i], s);
      z[i] = activate(s, a.act);
#pragma unroll
      for (int j = 0; j < W - 1; ++j) win[j][i] = win[j + 1][i];
    }
    store_pack<T, V>(y + t * a.channels, z);
  }
  const float none[V] = {};
  for (long long t = max(t0, live); t < t1; ++t) store_pack<T, V>(y + t * a.channels, none);
}

// A workgroup: `lanes` vectors of channels (a power of two) by 256 / lanes runs, whose filter gradients are added in LDS.
// parts: (workgroups along the runs, channels, W + 1)
template <typename T, int V, int W>
__global__ __launch_bounds__(256) void conv_backward_kernel(ConvArgs a, int vectors, int lanes, int across, long long runs, int run, long long first) {
  const long long block = first + blockIdx.x;
  const int lane = threadIdx.x % lanes, slot = threadIdx.x / lanes, slots = 256 / lanes;
  const int vec = (int)(block % across) * lanes + lane;
  const long long part = block / across, cell = part * slots + slot, row = cell / runs;
  const int c = vec * V;
  float dw[V][W], db[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int j = 0; j < W; ++j) dw[i][j] = 0.0f;
    db[i] = 0.0f;
  }
  if (vec < vectors && row < a.batch) {
    const long long t0 = cell % runs * run, t1 = min(t0 + run, a.tokens), end = conv_end(a.lengths, row, a.tokens);
    const T* const x = static_cast<const T*>(a.x) + row * a.x_sb + c;
    const T* const state = a.state_in ? static_cast<const T*>(a.state_in) + row * (W - 1) * a.channels + c : nullptr;
    const T* const dy = static_cast<const T*>(a.dy) + row * a.tokens * a.channels + c;
    const T* const dlast = a.dstate_out ? static_cast<const T*>(a.dstate_out) + row * (W - 1) * a.channels + c : nullptr;
    T* const dx = a.dx ? static_cast<T*>(a.dx) + row * a.tokens * a.channels + c : nullptr;
    T* const dstate = a.dstate_in ? static_cast<T*>(a.dstate_in) + row * (W - 1) * a.channels + c : nullptr;
    float w[V][W], b[V], win[W][V], dpre[W][V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int j = 0; j < W; ++j) {
        w[i][j] = a.weight[(long long)(c + i) * W + j];
        dpre[j][i] = 0.0f;
      }
      b[i] = a.bias ? a.bias[c + i] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      const long long t = t0 + j - (W - 1);
      if (t < end) {
        conv_frame<T, V, W>(x, a.x_st, state, a.channels, t, win[j]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) win[j][i] = 0.0f;
      }
    }
    // frame s = t - (W - 1) is complete with dpre_t
#pragma unroll 2
    for (long long t = t0; t < t1 + W - 1; ++t) {
      float g[V];
      const bool in = t < end;
      if (in) {
        load_pack<T, V>(x + t * a.x_st, win[W - 1]);
        load_pack<T, V>(dy + t * a.channels, g);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float s = b[i];
#pragma unroll
        for (int j = 0; j < W; ++j) s = __builtin_fmaf(w[i][j], win[j][i], s);
        dpre[W - 1][i] = in ? g[i] * activation_slope(s, a.act) : 0.0f;
        if (in && t < t1) {
#pragma unroll
          for (int j = 0; j < W; ++j) dw[i][j] = __builtin_fmaf(dpre[W - 1][i], win[j][i], dw[i][j]);
          db[i] += dpre[W - 1][i];
        }
#pragma unroll
        for (int j = 0; j < W - 1; ++j) win[j][i] = win[j + 1][i];
      }
      const long long s = t - (W - 1);
      const bool own = s >= t0 || t0 == 0;
      if (own && (s >= 0 ? dx != nullptr : dstate != nullptr)) {
        float d[V], last[V];
        const long long k = s + (W - 1) - end;  // its place in the state at the end
        const bool kept = dlast && k >= 0 && k < W - 1 && s < end;
        if (kept) load_pack<T, V>(dlast + k * a.channels, last);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          d[i] = 0.0f;
#pragma unroll
          for (int j = 0; j < W; ++j) d[i] = __builtin_fmaf(w[i][j], dpre[W - 1 - j][i], d[i]);
          if (kept) d[i] += last[i];
        }
        store_pack<T, V>(s >= 0 ? dx + s * a.channels : dstate + (s + W - 1) * a.channels, d);
      }
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int j = 0; j < W - 1; ++j) dpre[j][i] = dpre[j + 1][i];
    }
  }
  if (!a.dweight && !a.dbias) return;
  // the runs' sums, in their order
  __shared__ float sums[256][V + 1];
#pragma unroll
  for (int j = 0; j <= W; ++j) {
#pragma unroll
    for (int i = 0; i < V; ++i) sums[threadIdx.x][i] = j < W ? dw[i][j < W ? j : 0] : db[i];
    __syncthreads();
    for (int i = threadIdx.x; i < lanes * V; i += 256) {
      float s = 0.0f;
      for (int k = 0; k < slots; ++k) s += sums[k * lanes + i / V][i % V];
      const int channel = (int)(block % across) * lanes * V + i;
      if (channel < a.channels) a.ws[(part * a.channels + channel) * (W + 1) + j] = s;
    }
    __syncthreads();
  }
}

// Sums over the parts: a workgroup takes 32 neighbouring values, a team of 8 threads for each
__global__ __launch_bounds__(256) void conv_join_kernel(const float* parts, long long count, int channels, int width, float* dweight, float* dbias) {
  __shared__ float sums[8][32];
  const long long values = (long long)channels * (width + 1), i = (long long)blockIdx.x * 32 + threadIdx.x % 32;
  float s = 0.0f;
  if (i < values)
    for (long long k = threadIdx.x / 32; k < count; k += 8) s += parts[k * values + i];
  sums[threadIdx.x / 32][threadIdx.x % 32] = s;
  __syncthreads();
  if (threadIdx.x >= 32 || i >= values) return;
  s = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) s += sums[k][threadIdx.x];
  const int c = (int)(i / (width + 1)), j = (int)(i % (width + 1));
  if (j < width) {
    if (dweight) dweight[(long long)c * width + j] = s;
  } else if (dbias) {
    dbias[c] = s;
  }
}

template <typename T, int V, int W>
__global__ __launch_bounds__(256) void conv_step_kernel(ConvArgs a, int vectors, long long first) {
  const long long id = (first + blockIdx.x) * 256 + threadIdx.x, row = id / vectors;
  if (row >= a.batch) return;
  const int c = (int)(id % vectors) * V;
  T* const state = static_cast<T*>(a.state_out) + row * (W - 1) * a.channels + c;
  float win[W][V], z[V];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) load_pack<T, V>(state + (long long)j * a.channels, win[j]);
  load_pack<T, V>(static_cast<const T*>(a.x) + row * a.x_sb + c, win[W - 1]);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float s = a.bias ? a.bias[c + i] : 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) s = __builtin_fmaf(a.weight[(long long)(c + i) * W + j], win[j][i], s);
    z[i] = activate(s, a.act);
  }
#pragma unroll
  for (int j = 0; j < W - 1; ++j) store_pack<T, V>(state + (long long)j * a.channels, win[j + 1]);
  store_pack<T, V>(static_cast<T*>(a.y) + row * a.channels + c, z);
}

struct ConvRuns {
  int run, vectors, lanes, across;
  long long runs, parts;
};
// `v` values a vector
static ConvRuns conv_runs(const ConvArgs& a, int v) {
  ConvRuns r;
  r.vectors = (a.channels + v - 1) / v;
  r.run = kRunMost;
  while (r.run > 4 && a.batch * ((a.tokens + r.run - 1) / r.run) * r.vectors < kConvThreads) r.run /= 2;
  r.runs = std::max(1LL, (a.tokens + r.run - 1) / r.run);
  r.lanes = 64;
  while (r.lanes > 1 && r.lanes / 2 >= r.vectors) r.lanes /= 2;
  r.across = (r.vectors + r.lanes - 1) / r.lanes;
  const long long slots = 256 / r.lanes;
  r.parts = (a.batch * r.runs + slots - 1) / slots;
  return r;
}

static size_t type_size(int dtype) { return dtype == 0 ? 4 : 2; }

// whether vectors of v values can be read and written
static bool conv_whole(const ConvArgs& a, int v) {
  const uintptr_t bytes = v * type_size(a.dtype);
  const void* const all[] = {a.x, a.y, a.state_in, a.state_out, a.dy, a.dstate_out, a.dx, a.dstate_in};
  for (const void* p : all)
    if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
  return a.channels % v == 0 && a.x_sb % v == 0 && a.x_st % v == 0;
}
// Values a vector backward: 4, so that the windows of x and dpre, the filters and their gradients stay in registers
constexpr int kConvBackwardVector = 4;
static int conv_backward_vector(const ConvArgs& a) { return a.channels % kConvBackwardVector == 0 ? kConvBackwardVector : 1; }

size_t conv_workspace_bytes(const ConvArgs& a) {
  // (the vector that the addresses allow may be narrower than the sizes do: as many parts as the more of both)
  const long long parts = std::max(conv_runs(a, conv_backward_vector(a)).parts, conv_runs(a, 1).parts);
  return (size_t)parts * a.channels * (a.width + 1) * sizeof(float);
}

// f(first workgroup, workgroups) until all are launched
template <typename F>
static hipError_t conv_launches(long long blocks, F f) {
  for (long long first = 0; first < blocks; first += max_blocks(256)) {
    f(first, (unsigned)std::min(blocks - first, max_blocks(256)));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

enum ConvMode { kConvForward, kConvBackward, kConvStep };

template <ConvMode MODE, typename T, int V, int W>
static hipError_t conv_width(const ConvArgs& a) {
  const ConvRuns r = conv_runs(a, V);
  const long long threads = a.batch * r.vectors * (MODE == kConvStep ? 1 : r.runs), blocks = (threads + 255) / 256;
  if constexpr (MODE == kConvForward) {
    return conv_launches(blocks, [&](long long first, unsigned n) {
      hipLaunchKernelGGL((conv_forward_kernel<T, V, W>), dim3(n), dim3(256), 0, a.stream, a, r.vectors, r.runs, r.run, first);
    });
  } else if constexpr (MODE == kConvStep) {
    return conv_launches(blocks, [&](long long first, unsigned n) {
      hipLaunchKernelGGL((conv_step_kernel<T, V, W>), dim3(n), dim3(256), 0, a.stream, a, r.vectors, first);
    });
  } else {
    const hipError_t e = conv_launches(r.parts * r.across, [&](long long first, unsigned n) {
      hipLaunchKernelGGL((conv_backward_kernel<T, V, W>), dim3(n), dim3(256), 0, a.stream, a, r.vectors, r.lanes, r.across, r.runs, r.run, first);
    });
    if (e != hipSuccess || (!a.dweight && !a.dbias)) return e;
    const long long values = (long long)a.channels * (W + 1);
    hipLaunchKernelGGL(conv_join_kernel, dim3((unsigned)((values + 31) / 32)), dim3(256), 0, a.stream, a.ws, r.parts, a.channels, W, a.dweight, a.dbias);
    return hipGetLastError();
  }
}

template <ConvMode MODE, typename T, int V>
static hipError_t conv_vector(const ConvArgs& a) {
  switch (a.width) {
    case 1: return conv_width<MODE, T, V, 1>(a);
    case 2: return conv_width<MODE, T, V, 2>(a);
    case 3: return conv_width<MODE, T, V, 3>(a);
    case 4: return conv_width<MODE, T, V, 4>(a);
    case 5: return conv_width<MODE, T, V, 5>(a);
    case 6: return conv_width<MODE, T, V, 6>(a);
    case 7: return conv_width<MODE, T, V, 7>(a);
    case 8: return conv_width<MODE, T, V, 8>(a);
  }
  return hipErrorInvalidValue;
}

template <ConvMode MODE, typename T>
static hipError_t conv_typed(const ConvArgs& a) {
  constexpr int V = MODE == kConvBackward ? kConvBackwardVector : 16 / (int)sizeof(T);
  return conv_whole(a, V) ? conv_vector<MODE, T, V>(a) : conv_vector<MODE, T, 1>(a);
}

template <ConvMode MODE>
static hipError_t conv_mode(const ConvArgs& a) {
  return a.dtype == 0 ? conv_typed<MODE, float>(a) : a.dtype == 1 ? conv_typed<MODE, __bf16>(a) : conv_typed<MODE, _Float16>(a);
}

hipError_t launch_conv_forward(const ConvArgs& a) { return conv_mode<kConvForward>(a); }
hipError_t launch_conv_backward(const ConvArgs& a) { return conv_mode<kConvBackward>(a); }
hipError_t launch_conv_step(const ConvArgs& a) { return conv_mode<kConvStep>(a); }

}  // namespace tfa
