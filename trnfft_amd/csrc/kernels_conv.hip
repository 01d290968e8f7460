// Causal convolution along frames with a short filter for each channel, channels last, and an activation.
//
//   pre_t = bias + sum_j w_j x_{t - W + 1 + j},  y_t = act(pre_t);  frames before the first come from a state (the last W - 1 inputs)
//   dpre_t = dy_t act'(pre_t),  dx_s = sum_j w_j dpre_{s + W - 1 - j},  dw_j = sum_t dpre_t x_{t - W + 1 + j},  db = sum_t dpre_t
//
// Memory bound: x and y once forward; x, dy and dx once backward, where pre is computed again from x.  A thread takes a vector of
// channels over a run of frames, with its window of frames in registers, so a frame is read once but for the W - 1 in front of
// (and, backward, behind) a run.  Each filter width is a kernel of its own: a wider one with taps of zero would make NaN of
// infinities outside the filter.  Frames at and past lengths[n] are padding: not read, zeros in y and dx.
// 8 x 4096 tokens of 2048 channels, bf16, 4 taps: forward 52 us (5.1 TB/s, the rate of a copy), backward 101 and its join 5 (4.0 TB/s);
// 64 x 626 of 1024 with rows of all lengths 32.
// Numbers of channels that are no multiple of 8 (4 in fp32, and backward) go one value a thread: 2047 channels 81 forward and 254 in training
// (2048: 52 and 152), 2044 78 and 211.  Widths 5 to 8 take more registers for their windows and leave the backward three waves a SIMD (5) or
// two: forward 53 to 65, training 195 to 242.
#include "model_ops.h"
#include "activations.h"

#include <algorithm>
#include <type_traits>

namespace tfa {

// Tokens of a thread's run: as many as leave about kConvThreads threads, the fewer the smaller the call.
constexpr long long kConvThreads = 256 << 10;
constexpr int kRunMost = 64;
// Tokens whose loads are on their way together: forward 4 (8 and 2 are the same), backward 2, which leaves registers for more waves (8 x 4096
// tokens of 2048 bf16 channels and 4 taps: 101 us, 4 tokens 122)
constexpr int kConvBatch = 4, kConvBackBatch = 2;

// V neighbouring values in one access, which the memory takes at any address of an element
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> pack_at(const T* p) {
  Pack<T, V> u;
  __builtin_memcpy(&u, p, sizeof(u));
  return u;
}
template <typename T, int V>
__device__ __forceinline__ void load_any(const T* p, float (&x)[V]) {
  const Pack<T, V> u = pack_at<T, V>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = to_f32(u.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_any(T* p, const float (&x)[V]) {
  Pack<T, V> u;
#pragma unroll
  for (int i = 0; i < V; ++i) u.v[i] = from_f32<T>(x[i]);
  __builtin_memcpy(p, &u, sizeof(u));
}

__device__ __forceinline__ long long conv_end(const long long* lengths, long long row, long long tokens) {
  return lengths ? min(max(lengths[row], 0LL), tokens) : tokens;
}

// values of frame t >= -(W - 1) of a row: of the state where it is before the first, zeros where there is none
template <typename T, int V, int W>
__device__ __forceinline__ void conv_frame(const T* x, long long st, const T* state, long long channels, long long t, float (&v)[V]) {
  if (t >= 0) {
    load_any<T, V>(x + t * st, v);
  } else if (state) {
    load_any<T, V>(state + (t + W - 1) * channels, v);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.0f;
  }
}

// A workgroup takes `lanes` neighbouring vectors of channels (a power of two) over 256 / lanes runs.
struct ConvPlace {
  int vec, lane, slot;
  long long part, row, t0, t1;
};
__device__ __forceinline__ ConvPlace conv_place(long long block, int lanes, int across, long long runs, int run, long long tokens) {
  ConvPlace s;
  s.lane = threadIdx.x % lanes;
  s.slot = threadIdx.x / lanes;
  s.vec = (int)(block % across) * lanes + s.lane;
  s.part = block / across;
  const long long cell = s.part * (256 / lanes) + s.slot;
  s.row = cell / runs;
  s.t0 = cell % runs * run;
  s.t1 = min(s.t0 + run, tokens);
  return s;
}
// The workgroup's filters through LDS: read in their order in memory, by their channels from there (each lane its 16 W V bytes at once
// touched 64 cache lines an instruction).
template <int V, int W>
constexpr int kFilterWords = 64 * (V * W + 1);
template <int V, int W>
__device__ __forceinline__ void conv_filters(const ConvArgs& a, int lanes, int first, const ConvPlace& s, float* lds, float (&w)[V][W], float (&b)[V]) {
  const int count = min(lanes * V, a.channels - first) * W;
  for (int i = threadIdx.x; i < count; i += 256) lds[i / (V * W) * (V * W + 1) + i % (V * W)] = a.weight[(long long)first * W + i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = min(s.vec * V + i, a.channels - 1);
#pragma unroll
    for (int j = 0; j < W; ++j) w[i][j] = lds[min(s.lane, (a.channels - first - 1) / V) * (V * W + 1) + i * W + j];
    b[i] = a.bias ? a.bias[c] : 0.0f;
  }
}

template <typename T, int V, int W>
__global__ __launch_bounds__(256) void conv_forward_kernel(ConvArgs a, int vectors, int lanes, int across, long long runs, int run, long long first) {
  __shared__ float filters[kFilterWords<V, W>];
  const ConvPlace s = conv_place(first + blockIdx.x, lanes, across, runs, run, a.tokens);
  float w[V][W], b[V], win[W][V];
  conv_filters<V, W>(a, lanes, (s.vec - s.lane) * V, s, filters, w, b);
  if (s.vec >= vectors || s.row >= a.batch) return;
  const int c = s.vec * V;
  const long long end = conv_end(a.lengths, s.row, a.tokens), live = min(s.t1, end);
  const T* const x = static_cast<const T*>(a.x) + s.row * a.x_sb + c;
  const T* const state = a.state_in ? static_cast<const T*>(a.state_in) + s.row * (W - 1) * a.channels + c : nullptr;
  T* const y = static_cast<T*>(a.y) + s.row * a.tokens * a.channels + c;
  if (a.state_out && s.t0 == 0) {  // the last W - 1 frames up to the end
    T* const out = static_cast<T*>(a.state_out) + s.row * (W - 1) * a.channels + c;
    for (int j = 0; j < W - 1; ++j) {
      float v[V];
      conv_frame<T, V, W>(x, a.x_st, state, a.channels, end + j - (W - 1), v);
      store_any<T, V>(out + (long long)j * a.channels, v);
    }
  }
  if (s.t0 < live) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j) conv_frame<T, V, W>(x, a.x_st, state, a.channels, s.t0 + j - (W - 1), win[j]);
  }
  const auto token = [&](long long t, const Pack<T, V>& u) {
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      win[W - 1][i] = to_f32(u.v[i]);
      float sum = b[i];
#pragma unroll
      for (int j = 0; j < W; ++j) sum = __builtin_fmaf(w[i][j], win[j][i], sum);
      z[i] = activate(sum, a.act);
#pragma unroll
      for (int j = 0; j < W - 1; ++j) win[j][i] = win[j + 1][i];
    }
    store_any<T, V>(y + t * a.channels, z);
  };
  long long t = s.t0;
  for (; t + kConvBatch <= live; t += kConvBatch) {
    Pack<T, V> u[kConvBatch];
#pragma unroll
    for (int k = 0; k < kConvBatch; ++k) u[k] = pack_at<T, V>(x + (t + k) * a.x_st);
#pragma unroll
    for (int k = 0; k < kConvBatch; ++k) token(t + k, u[k]);
  }
  for (; t < live; ++t) token(t, pack_at<T, V>(x + t * a.x_st));
  const float none[V] = {};
  for (t = max(s.t0, live); t < s.t1; ++t) store_any<T, V>(y + t * a.channels, none);
}

// The workgroup's filter gradients are added in LDS.  parts: (workgroups along the runs, channels, W + 1)
template <typename T, int V, int W>
__global__ __launch_bounds__(256) void conv_backward_kernel(ConvArgs a, int vectors, int lanes, int across, long long runs, int run, long long first) {
  constexpr int kSums = 256 * (V + 1);
  __shared__ float lds[kSums > kFilterWords<V, W> ? kSums : kFilterWords<V, W>];
  const ConvPlace s = conv_place(first + blockIdx.x, lanes, across, runs, run, a.tokens);
  const int head = (s.vec - s.lane) * V;
  float dw[V][W], db[V], w[V][W], b[V];
  conv_filters<V, W>(a, lanes, head, s, lds, w, b);
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int j = 0; j < W; ++j) dw[i][j] = 0.0f;
    db[i] = 0.0f;
  }
  if (s.vec < vectors && s.row < a.batch) {
    const int c = s.vec * V;
    const long long end = conv_end(a.lengths, s.row, a.tokens), live = min(s.t1, end);
    const T* const x = static_cast<const T*>(a.x) + s.row * a.x_sb + c;
    const T* const state = a.state_in ? static_cast<const T*>(a.state_in) + s.row * (W - 1) * a.channels + c : nullptr;
    const T* const dy = static_cast<const T*>(a.dy) + s.row * a.tokens * a.channels + c;
    const T* const dlast = a.dstate_out ? static_cast<const T*>(a.dstate_out) + s.row * (W - 1) * a.channels + c : nullptr;
    T* const dx = a.dx ? static_cast<T*>(a.dx) + s.row * a.tokens * a.channels + c : nullptr;
    T* const dstate = a.dstate_in ? static_cast<T*>(a.dstate_in) + s.row * (W - 1) * a.channels + c : nullptr;
    float win[W][V], dpre[W][V];
#pragma unroll
    for (int j = 0; j < W; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) win[j][i] = dpre[j][i] = 0.0f;
      if (j < W - 1 && s.t0 + j - (W - 1) < end) conv_frame<T, V, W>(x, a.x_st, state, a.channels, s.t0 + j - (W - 1), win[j]);
    }
    // dpre_t of a token before the end; `counts`: one of the run's own, whose filter gradients are its
    const auto token = [&](const Pack<T, V>& u, const Pack<T, V>& g, auto counts) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        win[W - 1][i] = to_f32(u.v[i]);
        float sum = b[i];
#pragma unroll
        for (int j = 0; j < W; ++j) sum = __builtin_fmaf(w[i][j], win[j][i], sum);
        const float d = to_f32(g.v[i]) * activation_slope(sum, a.act);
        dpre[W - 1][i] = d;
        if constexpr (counts) {
#pragma unroll
          for (int j = 0; j < W; ++j) dw[i][j] = __builtin_fmaf(d, win[j][i], dw[i][j]);
          db[i] += d;
        }
#pragma unroll
        for (int j = 0; j < W - 1; ++j) win[j][i] = win[j + 1][i];
      }
    };
    // the gradient of frame t - (W - 1), which is complete with dpre_t; then the next token's place
    const auto frame = [&](T* to, const float (&more)[V]) {
      float d[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        d[i] = more[i];
#pragma unroll
        for (int j = 0; j < W; ++j) d[i] = __builtin_fmaf(w[i][j], dpre[W - 1 - j][i], d[i]);
#pragma unroll
        for (int j = 0; j < W - 1; ++j) dpre[j][i] = dpre[j + 1][i];
      }
      if (to) store_any<T, V>(to, d);
    };
    const float none[V] = {};
    // The first W - 1 tokens complete frames of the run before, or of the state before the first
    long long t = s.t0;
    for (; t < live && t < s.t0 + W - 1; ++t) {
      token(pack_at<T, V>(x + t * a.x_st), pack_at<T, V>(dy + t * a.channels), std::true_type());
      frame(s.t0 == 0 && dstate ? dstate + t * a.channels : nullptr, none);
    }
    for (; t + kConvBackBatch <= live; t += kConvBackBatch) {
      Pack<T, V> u[kConvBackBatch], g[kConvBackBatch];
#pragma unroll
      for (int k = 0; k < kConvBackBatch; ++k) {
        u[k] = pack_at<T, V>(x + (t + k) * a.x_st);
        g[k] = pack_at<T, V>(dy + (t + k) * a.channels);
      }
#pragma unroll
      for (int k = 0; k < kConvBackBatch; ++k) {
        token(u[k], g[k], std::true_type());
        frame(dx ? dx + (t + k - (W - 1)) * a.channels : nullptr, none);
      }
    }
    // the rest of the run, the W - 1 tokens behind it, and padding
    for (; t < s.t1 + W - 1; ++t) {
      if (t < end) {
        const Pack<T, V> u = pack_at<T, V>(x + t * a.x_st), g = pack_at<T, V>(dy + t * a.channels);
        if (t < s.t1)
          token(u, g, std::true_type());
        else
          token(u, g, std::false_type());
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) dpre[W - 1][i] = 0.0f;
      }
      const long long at = t - (W - 1), k = t - end;  // the frame, and its place in the state at the end
      float more[V] = {};
      if (dlast && k >= 0 && k < W - 1) load_any<T, V>(dlast + k * a.channels, more);
      T* to = nullptr;
      if (at >= 0 ? at >= s.t0 : s.t0 == 0) to = at >= 0 ? (dx ? dx + at * a.channels : nullptr) : (dstate ? dstate + (at + W - 1) * a.channels : nullptr);
      frame(to, more);
    }
  }
  if (!a.dweight && !a.dbias) return;
  // the runs' sums, in their order
  const int slots = 256 / lanes;
#pragma unroll
  for (int j = 0; j <= W; ++j) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) lds[threadIdx.x * (V + 1) + i] = j < W ? dw[i][j < W ? j : 0] : db[i];
    __syncthreads();
    for (int i = threadIdx.x; i < lanes * V; i += 256) {
      float sum = 0.0f;
      for (int k = 0; k < slots; ++k) sum += lds[(k * lanes + i / V) * (V + 1) + i % V];
      const int channel = head + i;
      if (channel < a.channels) a.ws[(s.part * a.channels + channel) * (W + 1) + j] = sum;
    }
  }
}

// Sums over the parts: a workgroup takes 32 neighbouring values, a team of 8 threads for each
__global__ __launch_bounds__(256) void conv_join_kernel(const float* parts, long long count, int channels, int width, float* dweight, float* dbias) {
  __shared__ float sums[8][32];
  const long long values = (long long)channels * (width + 1), i = (long long)blockIdx.x * 32 + threadIdx.x % 32;
  float s = 0.0f;
  if (i < values) {
#pragma unroll 8
    for (long long k = threadIdx.x / 32; k < count; k += 8) s += parts[k * values + i];
  }
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
  for (int j = 0; j < W - 1; ++j) load_any<T, V>(state + (long long)j * a.channels, win[j]);
  load_any<T, V>(static_cast<const T*>(a.x) + row * a.x_sb + c, win[W - 1]);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float s = a.bias ? a.bias[c + i] : 0.0f;
#pragma unroll
    for (int j = 0; j < W; ++j) s = __builtin_fmaf(a.weight[(long long)(c + i) * W + j], win[j][i], s);
    z[i] = activate(s, a.act);
  }
#pragma unroll
  for (int j = 0; j < W - 1; ++j) store_any<T, V>(state + (long long)j * a.channels, win[j + 1]);
  store_any<T, V>(static_cast<T*>(a.y) + row * a.channels + c, z);
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

// Values a vector backward: 4, so that the windows of x and dpre, the filters and their gradients stay in registers
constexpr int kConvBackwardVector = 4;
static int conv_backward_vector(const ConvArgs& a) { return a.channels % kConvBackwardVector == 0 ? kConvBackwardVector : 1; }

size_t conv_workspace_bytes(const ConvArgs& a) {
  const long long parts = conv_runs(a, conv_backward_vector(a)).parts;
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
  if constexpr (MODE == kConvForward) {
    return conv_launches(r.parts * r.across, [&](long long first, unsigned n) {
      hipLaunchKernelGGL((conv_forward_kernel<T, V, W>), dim3(n), dim3(256), 0, a.stream, a, r.vectors, r.lanes, r.across, r.runs, r.run, first);
    });
  } else if constexpr (MODE == kConvStep) {
    return conv_launches((a.batch * r.vectors + 255) / 256, [&](long long first, unsigned n) {
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
  return a.channels % V == 0 ? conv_vector<MODE, T, V>(a) : conv_vector<MODE, T, 1>(a);
}

template <ConvMode MODE>
static hipError_t conv_mode(const ConvArgs& a) {
  return a.dtype == 0 ? conv_typed<MODE, float>(a) : a.dtype == 1 ? conv_typed<MODE, __bf16>(a) : conv_typed<MODE, _Float16>(a);
}

hipError_t launch_conv_forward(const ConvArgs& a) { return conv_mode<kConvForward>(a); }
hipError_t launch_conv_backward(const ConvArgs& a) { return conv_mode<kConvBackward>(a); }
hipError_t launch_conv_step(const ConvArgs& a) { return conv_mode<kConvStep>(a); }

}  // namespace tfa
