// The selective scan's step for one token of every stream, and what joins the parts of whole sequences (scan_blocks.h).
#include "scan_blocks.h"

namespace tfa {

// The states that segments start from, in place of their own sums; reversed, the gradients that they end with.  A thread takes a lane of a
// wave's states over the segments, one after the other.
template <int R>
__global__ __launch_bounds__(64) void scan_join_kernel(ScanArgs p, int lanes, bool reverse, long long first) {
  const long long unit = first + blockIdx.x;
  const int lane = threadIdx.x, channels = 64 / lanes, q = lane / channels, each = p.channels / p.groups;
  const int tiles = (each + channels - 1) / channels;
  const long long units = p.batch * p.groups * tiles;
  if (unit >= units) return;
  const int own = (int)(unit % tiles) * channels + lane % channels;
  const long long row = unit / tiles / p.groups;
  const bool valid = own < each;
  const int channel = (int)(unit / tiles % p.groups) * each + (valid ? own : 0);
  States<R> a = load_states<R>(p.a + (long long)channel * p.n, p.n, q, valid);
#pragma unroll
  for (int r = 0; r < R; ++r) a.v[r] = rate_of(a.v[r]);
  const float* from = reverse ? p.dstate_out : p.state_in;
  States<R> s = {};
  if (from) s = load_states<R>(from + (row * p.channels + channel) * p.n, p.n, q, valid);
  // sixteen segments' sums on their way at a time
  constexpr int U = 16;
  const int parts = p.segments * p.fine, sums = parts - p.fine;  // (the last segment's have none)
  for (int k0 = 0; k0 <= sums; k0 += U) {
    States<R> sum[U];
    float steps[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int k = min(k0 + i, sums - 1);
      const long long at = ((reverse ? parts - 1 - k : k) * units + unit) * 64 + lane;
      sum[i] = reinterpret_cast<const States<R>*>(p.seg_state)[at];
      steps[i] = p.seg_steps[at];
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int k = k0 + i;
      if (k > sums) break;
      reinterpret_cast<States<R>*>(p.seg_state)[((reverse ? parts - 1 - k : k) * units + unit) * 64 + lane] = s;
#pragma unroll
      for (int r = 0; r < R; ++r) s.v[r] = __builtin_fmaf(__builtin_amdgcn_exp2f(steps[i] * a.v[r]), s.v[r], sum[i].v[r]);
    }
  }
}

// db and dc from the workgroups' shares (of `states` states, n and what fills up the lanes): a thread for each value, zeros where there is padding
template <typename T>
__global__ __launch_bounds__(256) void scan_shares_kernel(ScanArgs p, int states, long long parts, long long first) {
  const long long id = (first + blockIdx.x) * 256 + threadIdx.x, width = (long long)p.groups * 2 * states, cells = p.batch * p.tokens;
  const long long cell = id / width;
  if (cell >= cells) return;
  const int at = (int)(id % width), group = at / (2 * states), which = at / states % 2, k = at % states;
  T* const out = static_cast<T*>(which ? p.dc : p.db);
  if (!out || k >= p.n) return;
  float sum = 0.0f;
  if (cell % p.tokens < scan_end(p, cell / p.tokens)) {
#pragma unroll 8
    for (long long i = 0; i < parts; ++i) sum += p.shared_parts[i * cells * width + id];
  }
  out[(cell * p.groups + group) * p.n + k] = from_f32<T>(sum);
}

// da, dd and ddt_bias from the rows' and segments' sums: a workgroup for a wave's channels, whose waves take every kSumWaves-th sum.  Many sums are
// added in two passes: `span` neighbours by a workgroup, which leaves theirs in place of the first, then (span 0) every `step`-th.
// 8 x 4096 tokens of 2048 channels 4.9 us; 10000 rows of 64 channels 20 in two passes, 241 in one, 1273 by one thread for all sums of a state.
constexpr int kSumWaves = 16;
constexpr long long kSumsAtOnce = 256;
template <int R>
__global__ __launch_bounds__(64 * kSumWaves) void scan_channels_kernel(ScanArgs p, int lanes, long long span, long long step) {
  __shared__ States<R> of_a[kSumWaves][64];
  __shared__ States<2> of_rest[kSumWaves][64];
  const int channels = 64 / lanes, each = p.channels / p.groups, tiles = (each + channels - 1) / channels;
  const int tile = (int)(blockIdx.x % (p.groups * tiles)), lane = threadIdx.x % 64, wave = threadIdx.x / 64, q = lane / channels;
  const int own = tile % tiles * channels + lane % channels;
  const long long of_row = (long long)p.groups * tiles * 64, id = tile * 64LL + lane;
  const long long count = p.segments * p.batch, all = count * of_row;
  const long long begin = blockIdx.x / (p.groups * tiles) * span, end = span ? min(begin + span, count) : count;
  States<R> da = {};
  States<2> rest = {};
#pragma unroll 4
  for (long long i = begin + wave * step; i < end; i += kSumWaves * step) {
    const long long at = i * of_row + id;
    const States<R> v = reinterpret_cast<const States<R>*>(p.channel_parts)[at];
#pragma unroll
    for (int r = 0; r < R; ++r) da.v[r] += v.v[r];
    rest.v[0] += p.channel_parts[R * all + at];
    rest.v[1] += p.channel_parts[(R + 1) * all + at];
  }
  of_a[wave][lane] = da;
  of_rest[wave][lane] = rest;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < kSumWaves; ++w) {
#pragma unroll
    for (int r = 0; r < R; ++r) da.v[r] += of_a[w][lane].v[r];
    rest.v[0] += of_rest[w][lane].v[0], rest.v[1] += of_rest[w][lane].v[1];
  }
  if (span) {
    const long long at = begin * of_row + id;
    reinterpret_cast<States<R>*>(p.channel_parts)[at] = da;
    p.channel_parts[R * all + at] = rest.v[0];
    p.channel_parts[(R + 1) * all + at] = rest.v[1];
    return;
  }
  if (own >= each) return;
  const int channel = tile / tiles * each + own;
  if (p.da) store_states<R>(p.da + (long long)channel * p.n, p.n, q, true, da);
  if (q == 0 && p.dd) p.dd[channel] = rest.v[0];
  if (q == 0 && p.ddt_bias) p.ddt_bias[channel] = rest.v[1];
}

template <int BLOCK = 256, typename F>
static hipError_t scan_launches(long long threads, F f) {
  const long long blocks = (threads + BLOCK - 1) / BLOCK;
  for (long long first = 0; first < blocks; first += max_blocks(BLOCK)) {
    f(first, (unsigned)std::min(blocks - first, max_blocks(BLOCK)));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

static hipError_t scan_mode(const ScanArgs& p, ScanMode mode) {
  return p.dtype == 0 ? scan_f32(p, mode) : p.dtype == 1 ? scan_bf16(p, mode) : scan_f16(p, mode);
}

static long long scan_tiles(const ScanArgs& p) {
  const int channels = 64 / scan_shape(p.n).lanes;
  return (p.channels / p.groups + channels - 1) / channels;
}
long long scan_waves(const ScanArgs& p) { return p.batch * p.groups * scan_tiles(p); }

bool scan_has_pairs(const ScanArgs& p) { return scan_shape(p.n).lanes == 4 && scan_shape(p.n).each == 4; }

static long long share_parts(const ScanArgs& p) {
  const int lanes = scan_shape(p.n).lanes, waves = lanes == 4 ? kBackWaves<4> : lanes == 8 ? kBackWaves<8> : kBackWaves<16>;
  return (scan_tiles(p) + waves - 1) / waves;
}

ScanSizes scan_sizes(const ScanArgs& p) {
  ScanSizes s;
  const ScanShape shape = scan_shape(p.n);
  const size_t lanes = (size_t)scan_waves(p) * 64, of_segments = p.segments > 1 ? p.segments * p.fine * lanes : 0;
  s.kept = p.tokens > 0 ? (p.tokens - 1) / kScanStretch * lanes * shape.each * sizeof(float) : 0;
  s.seg_state = of_segments * shape.each * sizeof(float);
  s.seg_steps = of_segments * sizeof(float);
  s.shared_parts = (size_t)share_parts(p) * p.batch * p.tokens * p.groups * 2 * shape.lanes * shape.each * sizeof(float);
  s.channel_parts = (size_t)p.segments * lanes * (shape.each + 2) * sizeof(float);
  return s;
}

static hipError_t scan_segments(const ScanArgs& p, bool reverse) {
  if (p.segments == 1) return hipSuccess;
  const hipError_t e = scan_mode(p, reverse ? kScanBackSums : kScanSums);
  if (e != hipSuccess) return e;
  const ScanShape s = scan_shape(p.n);
  return scan_launches<64>(scan_waves(p) * 64, [&](long long first, unsigned n) {
    const auto kernel = s.each == 1 ? scan_join_kernel<1> : s.each == 2 ? scan_join_kernel<2> : scan_join_kernel<4>;
    hipLaunchKernelGGL(kernel, dim3(n), dim3(64), 0, p.stream, p, s.lanes, reverse, first);
  });
}

hipError_t launch_scan_forward(const ScanArgs& p) {
  const hipError_t e = scan_segments(p, false);
  return e != hipSuccess ? e : scan_mode(p, kScanForward);
}

hipError_t launch_scan_backward(const ScanArgs& p) {
  hipError_t e = scan_segments(p, true);
  if (e != hipSuccess) return e;
  e = scan_mode(p, kScanBackward);
  if (e != hipSuccess) return e;
  const ScanShape s = scan_shape(p.n);
  if (p.shared_parts) {
    const int states = s.lanes * s.each;
    e = scan_launches(p.batch * p.tokens * p.groups * 2 * states, [&](long long first, unsigned n) {
      const auto kernel = p.dtype == 0 ? scan_shares_kernel<float> : p.dtype == 1 ? scan_shares_kernel<__bf16> : scan_shares_kernel<_Float16>;
      hipLaunchKernelGGL(kernel, dim3(n), dim3(256), 0, p.stream, p, states, share_parts(p), first);
    });
    if (e != hipSuccess) return e;
  }
  if (!p.da && !p.dd && !p.ddt_bias) return hipSuccess;
  const auto kernel = s.each == 1 ? scan_channels_kernel<1> : s.each == 2 ? scan_channels_kernel<2> : scan_channels_kernel<4>;
  const long long tiles = p.groups * scan_tiles(p), count = p.segments * p.batch;
  long long step = 1;
  if (count > kSumsAtOnce) {
    // (as many workgroups as a grid holds, of 64 sums at least)
    step = std::max({64LL, (count + kSumsAtOnce - 1) / kSumsAtOnce, count / std::max(1LL, max_blocks(64 * kSumWaves) / tiles - 1)});
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles * ((count + step - 1) / step))), dim3(64 * kSumWaves), 0, p.stream, p, s.lanes, step, 1LL);
    if (const hipError_t failed = hipGetLastError(); failed != hipSuccess) return failed;
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles), dim3(64 * kSumWaves), 0, p.stream, p, s.lanes, 0LL, step);
  return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------

// sum over Q neighbouring lanes, in all of them
template <int Q>
__device__ __forceinline__ float sum_lanes(float v) {
  if constexpr (Q >= 2) v += lane_xor<1>(v);
  if constexpr (Q >= 4) v += lane_xor<2>(v);
  if constexpr (Q >= 8) v += lane_xor<7>(v);
  if constexpr (Q >= 16) v += lane_xor<8>(v);
  return v;
}

// Q neighbouring lanes a channel, 4 states each, so that a wave reads and writes its states in one piece; ROWS streams a thread, whose states
// are on their way together and for which a, d and dt_bias are read once.  Memory bound by the states.  256 streams of 2048 channels of 16
// states, bf16: 16.9 us (72 MB); with one stream a thread 19.0, four 19.7, eight 28.0.
// States, a, b and c are read by fours where n is a multiple of that: the memory takes one access at any address of an element.
template <typename T, int Q, int ROWS>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanStep p, long long first) {
  const long long id = ((first + blockIdx.x) * 256 + threadIdx.x) / Q, row0 = id / p.channels * ROWS;
  const int q = threadIdx.x % Q;
  if (row0 >= p.batch) return;
  const int channel = (int)(id % p.channels), group = channel / (p.channels / p.groups), k0 = 4 * q;
  const bool all = p.n % 4 == 0 && k0 < p.n;
  const auto states_of = [&](const float* at) {
    if (!all) return load_states<4>(at, p.n, q, true);
    Four32 v;
    __builtin_memcpy(v.v, at + k0, sizeof(v));
    return v;
  };
  const auto rows_of = [&](const void* base, long long at) {
    const T* const from = static_cast<const T*>(base) + at;
    Four32 v;
    if (all) {
      T u[4];
      __builtin_memcpy(u, from + k0, sizeof(u));
#pragma unroll
      for (int r = 0; r < 4; ++r) v.v[r] = to_f32(u[r]);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) v.v[r] = k0 + r < p.n ? to_f32(from[k0 + r]) : 0.0f;
    }
    return v;
  };
  Four32 h[ROWS], b[ROWS], c[ROWS];
  float x[ROWS], dt[ROWS], z[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const long long row = min(row0 + i, p.batch - 1);
    h[i] = states_of(p.state + (row * p.channels + channel) * p.n);
    b[i] = rows_of(p.b, row * p.b_sb + group * p.b_sg);
    c[i] = rows_of(p.c, row * p.c_sb + group * p.c_sg);
    x[i] = to_f32(static_cast<const T*>(p.x)[row * p.x_sb + channel]);
    dt[i] = to_f32(static_cast<const T*>(p.dt)[row * p.dt_sb + channel]);
    z[i] = p.z ? to_f32(static_cast<const T*>(p.z)[row * p.z_sb + channel]) : 0.0f;
  }
  Four32 a = states_of(p.a + (long long)channel * p.n);
#pragma unroll
  for (int r = 0; r < 4; ++r) a.v[r] = rate_of(a.v[r]);
  const float skip = p.d ? p.d[channel] : 0.0f, bias = p.dt_bias ? p.dt_bias[channel] : 0.0f;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const long long row = row0 + i;
    if (ROWS > 1 && row >= p.batch) break;
    float s = dt[i] + bias, slope;
    if (p.softplus) s = softplus(s, slope);
    const float u = s * x[i];
    float y = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (k0 + r >= p.n) continue;  // (nothing of what fills a lane up: it may not be finite)
      h[i].v[r] = __builtin_fmaf(decay_of(s, a.v[r]), h[i].v[r], u * b[i].v[r]);
      y = __builtin_fmaf(c[i].v[r], h[i].v[r], y);
    }
    float* const state = p.state + (row * p.channels + channel) * p.n;
    if (all)
      __builtin_memcpy(state + k0, h[i].v, sizeof(h[i]));
    else
      store_states<4>(state, p.n, q, true, h[i]);
    y = sum_lanes<Q>(y);
    if (q) continue;
    y = __builtin_fmaf(skip, x[i], y);
    if (p.z) y *= activate(z[i], kActSilu);
    static_cast<T*>(p.y)[row * p.channels + channel] = from_f32<T>(y);
  }
}

template <typename T, int Q, int ROWS>
static hipError_t step_rows(const ScanStep& p) {
  return scan_launches((p.batch + ROWS - 1) / ROWS * p.channels * Q, [&](long long first, unsigned n) {
    hipLaunchKernelGGL((scan_step_kernel<T, Q, ROWS>), dim3(n), dim3(256), 0, p.stream, p, first);
  });
}
// Two streams a thread where that leaves 2048 waves
template <typename T, int Q>
static hipError_t step_lanes(const ScanStep& p) {
  return p.batch / 2 * p.channels * Q >= 2048 * 64 ? step_rows<T, Q, 2>(p) : step_rows<T, Q, 1>(p);
}
template <typename T>
static hipError_t step_typed(const ScanStep& p) {
  if (p.n <= 4) return step_lanes<T, 1>(p);
  if (p.n <= 8) return step_lanes<T, 2>(p);
  if (p.n <= 16) return step_lanes<T, 4>(p);
  return p.n <= 32 ? step_lanes<T, 8>(p) : step_lanes<T, 16>(p);
}
hipError_t launch_scan_step(const ScanStep& p) {
  return p.dtype == 0 ? step_typed<float>(p) : p.dtype == 1 ? step_typed<__bf16>(p) : step_typed<_Float16>(p);
}

}  // namespace tfa
