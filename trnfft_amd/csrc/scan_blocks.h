// The selective scan over whole sequences and its gradients (kernels_scan_{f32,bf16,f16}.hip instantiate it by type).
//
//   s_t = softplus(dt_t + dt_bias),  h_t[n] = exp(s_t a[n]) h_{t-1}[n] + s_t x_t b_t[n],  y_t = (sum_n c_t[n] h_t[n] + d x_t) silu(z_t)
// for every channel, b and c shared by the channels of a group.  With e = exp(s_t a), v_t = dy_t silu(z_t):
//   g_t[n] = v_t c_t[n] + e_{t+1}[n] g_{t+1}[n],  db_t[n] = sum over channels of g_t[n] s_t x_t,  dc_t[n] = the same of v_t h_t[n],
//   ds_t = x_t sum_n g_t[n] b_t[n] + sum_n a[n] f_t[n],  dx_t = s_t sum_n g_t[n] b_t[n] + d v_t,  da[n] = sum_t s_t f_t[n],
//   where f_t = g_t e_t h_{t-1},  dz_t = dy_t silu'(z_t) (sum_n c_t[n] h_t[n] + d x_t)
//
// A wave takes 64 / Q channels of a row and group, Q lanes a channel with 4 states each (Q the least power of two that holds n), and walks
// along the tokens in tiles of 16.  For what belongs to a channel and token alone (softplus, gates, loads, stores) lane q of a channel takes
// every Q-th token, so nothing of it is done twice; the tokens' s and s x go to the channel's lanes through LDS, as do b and
// c, whose rows all channels of a group share.  Sums over the lanes of a channel are folded: Q tokens' sums at once, each ending in
// the lane of its token.
#pragma once
#include "scan_device.h"

#include <algorithm>

namespace tfa {

struct alignas(16) Four32 {
  float v[4];
};

// where a lane stands
template <int Q>
struct ScanPlace {
  static constexpr int kChannels = 64 / Q;
  int lane, q, c;            // c: channel of the tile
  long long row;
  int group, tile, channel;  // channel of the row
  bool valid;                // whether there is such a channel
  long long unit, units;
  int seg;
};

template <int Q>
__device__ __forceinline__ ScanPlace<Q> scan_place(const ScanArgs& p, long long block, int waves) {
  ScanPlace<Q> s;
  const int each = p.channels / p.groups, tiles = (each + s.kChannels - 1) / s.kChannels, across = (tiles + waves - 1) / waves;
  s.lane = threadIdx.x % 64;
  s.q = s.lane / s.kChannels;
  s.c = s.lane % s.kChannels;
  s.tile = (int)(block % across) * waves + threadIdx.x / 64;
  block /= across;
  s.group = (int)(block % p.groups);
  block /= p.groups;
  s.row = block % p.batch;
  s.seg = (int)(block / p.batch);
  const int own = s.tile * s.kChannels + s.c;
  s.valid = own < each;
  s.channel = s.group * each + (s.valid ? own : 0);
  s.units = p.batch * p.groups * tiles;
  s.unit = (s.row * p.groups + s.group) * tiles + min(s.tile, tiles - 1);
  return s;
}

// A wave's own LDS: nothing but the order of its instructions is needed between its lanes' writes and reads.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

constexpr int kPlaneRow = kScanTile + 4;  // words of a channel's tokens: rows at 16 bytes that spread over the banks

// A value of every channel and token of the tile: lane q puts tokens q, q + Q, ...; all lanes of a channel read four neighbours.
template <int Q>
struct ScanPlane {
  float own[Q == 1 ? kScanTile : 1];
  __device__ __forceinline__ void put(float* lds, int q, int c, int i, float v) {
    if constexpr (Q == 1)
      own[i] = v;
    else
      lds[c * kPlaneRow + q + Q * i] = v;
  }
  __device__ __forceinline__ Four32 four(const float* lds, int c, int k) const {
    if constexpr (Q == 1)
      return {own[4 * k], own[4 * k + 1], own[4 * k + 2], own[4 * k + 3]};
    else
      return *reinterpret_cast<const Four32*>(lds + c * kPlaneRow + 4 * k);
  }
};
template <int Q>
constexpr int kPlaneWords = Q == 1 ? 0 : 64 / Q * kPlaneRow;

// a tile's tokens q, q + Q, ... of one operand
template <typename T, int Q>
struct ScanTokens {
  T v[kScanTile / Q];
  // p: token t0 + q of the channel
  __device__ __forceinline__ void load(const T* p, long long st, long long first, long long end, bool valid) {
#pragma unroll
    for (int i = 0; i < kScanTile / Q; ++i) v[i] = valid && first + Q * i < end ? p[i * Q * st] : T(0);
  }
};
// a tile's rows of b or c, 16 by 4 Q with zeros past n and past the end: lane l has elements l, l + 64, ...
template <typename T, int Q>
struct ScanRows {
  T v[Q];
  // p: token t0 of the row and group
  __device__ __forceinline__ void load(const T* p, long long st, int n, int lane, long long t0, long long end) {
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      const int at = lane + 64 * i, t = at / (4 * Q), k = at % (4 * Q);
      v[i] = k < n && t0 + t < end ? p[t * st + k] : T(0);
    }
  }
  __device__ __forceinline__ void put(float* lds, int lane) const {
#pragma unroll
    for (int i = 0; i < Q; ++i) lds[lane + 64 * i] = to_f32(v[i]);
  }
};

// sums over a channel's lanes of Q values: lane q receives the q-th
template <int Q, int MASK = 32>
__device__ __forceinline__ float fold_states(const float (&v)[Q]) {
  if constexpr (Q == 1) {
    return v[0];
  } else {
    float w[Q / 2];
#pragma unroll
    for (int i = 0; i < Q / 2; ++i) w[i] = fold<MASK>(v[i], v[i + Q / 2]);
    return fold_states<Q / 2, MASK / 2>(w);
  }
}
// the sum over a channel's lanes, in all of them
template <int Q, int MASK = 32>
__device__ __forceinline__ float sum_states(float v) {
  if constexpr (Q == 1)
    return v;
  else
    return sum_states<Q / 2, MASK / 2>(fold<MASK>(v));
}

// four states of a channel in (channels, n) fp32
__device__ __forceinline__ Four32 load_states(const float* p, int n, int q, bool valid) {
  Four32 s;
#pragma unroll
  for (int r = 0; r < 4; ++r) s.v[r] = valid && 4 * q + r < n ? p[4 * q + r] : 0.0f;
  return s;
}
__device__ __forceinline__ void store_states(float* p, int n, int q, bool valid, const Four32& s) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (valid && 4 * q + r < n) p[4 * q + r] = s.v[r];
}

__device__ __forceinline__ long long scan_end(const ScanArgs& p, long long row) {
  return p.lengths ? min(max(p.lengths[row], 0LL), p.tokens) : p.tokens;
}
__device__ __forceinline__ long long kept_states(const ScanArgs& p) { return p.tokens > 0 ? (p.tokens - 1) / kScanStretch : 0; }

// s_t and, where asked for, its slope by dt_t
__device__ __forceinline__ float step_of(float dt, float bias, bool soft, float& slope) {
  slope = 1.0f;
  return soft ? softplus(dt + bias, slope) : dt + bias;
}

constexpr int kScanWaves = 4;  // of a workgroup of the forward and the sums

// OUT: the sequences, or their segments from seg_state's states.  Else the segments' own sums from zero, and their steps' sums.
template <typename T, int Q, bool OUT>
__global__ __launch_bounds__(64 * kScanWaves) void scan_forward_kernel(ScanArgs p, long long first_block) {
  constexpr int kOwn = kScanTile / Q;
  __shared__ float rows[kScanWaves][2][64 * Q];
  __shared__ float planes[kScanWaves][2][Q == 1 ? 1 : kPlaneWords<Q>];
  const ScanPlace<Q> s = scan_place<Q>(p, first_block + blockIdx.x, kScanWaves);
  if (s.tile * s.kChannels >= p.channels / p.groups) return;
  const int wave = threadIdx.x / 64;
  float *const lb = rows[wave][0], *const lc = rows[wave][1], *const ls = planes[wave][0], *const lu = planes[wave][1];
  const long long seg_begin = s.seg * p.seg_tokens, seg_end = min(p.tokens, seg_begin + p.seg_tokens), end = min(scan_end(p, s.row), seg_end);

  const T* px = static_cast<const T*>(p.x) + s.row * p.x_sb + (seg_begin + s.q) * p.x_st + s.channel;
  const T* pdt = static_cast<const T*>(p.dt) + s.row * p.dt_sb + (seg_begin + s.q) * p.dt_st + s.channel;
  const T* pz = p.z ? static_cast<const T*>(p.z) + s.row * p.z_sb + (seg_begin + s.q) * p.z_st + s.channel : nullptr;
  const T* pb = static_cast<const T*>(p.b) + s.row * p.b_sb + seg_begin * p.b_st + s.group * p.b_sg;
  const T* pc = static_cast<const T*>(p.c) + s.row * p.c_sb + seg_begin * p.c_st + s.group * p.c_sg;
  T* py = OUT ? static_cast<T*>(p.y) + (s.row * p.tokens + seg_begin + s.q) * p.channels + s.channel : nullptr;

  Four32 a = load_states(p.a + (long long)s.channel * p.n, p.n, s.q, s.valid), h = {};
#pragma unroll
  for (int r = 0; r < 4; ++r) a.v[r] *= kLog2E;
  const float bias = p.dt_bias ? p.dt_bias[s.channel] : 0.0f, skip = p.d ? p.d[s.channel] : 0.0f;
  if (OUT) {
    if (p.segments > 1)
      h = reinterpret_cast<const Four32*>(p.seg_state)[(s.seg * s.units + s.unit) * 64 + s.lane];
    else if (p.state_in)
      h = load_states(p.state_in + (s.row * p.channels + s.channel) * p.n, p.n, s.q, s.valid);
  }
  float steps = 0.0f;
  ScanTokens<T, Q> x, dt, z;
  ScanRows<T, Q> b, c;
  const auto fetch = [&](long long t0) {
    x.load(px, p.x_st, t0 + s.q, end, s.valid);
    dt.load(pdt, p.dt_st, t0 + s.q, end, s.valid);
    b.load(pb, p.b_st, p.n, s.lane, t0, end);
    if (OUT) {
      c.load(pc, p.c_st, p.n, s.lane, t0, end);
      if (pz) z.load(pz, p.z_st, t0 + s.q, end, s.valid), pz += kScanTile * p.z_st;
    }
    px += kScanTile * p.x_st, pdt += kScanTile * p.dt_st, pb += kScanTile * p.b_st, pc += kScanTile * p.c_st;
  };
  fetch(seg_begin);
  for (long long t0 = seg_begin; t0 < end; t0 += kScanTile) {
    if (OUT && p.kept && t0 > 0 && t0 % kScanStretch == 0)
      reinterpret_cast<Four32*>(p.kept)[(s.unit * kept_states(p) + t0 / kScanStretch - 1) * 64 + s.lane] = h;
    ScanPlane<Q> step, in;
    float xs[kOwn], zs[kOwn];
    wave_order();
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      float slope;
      xs[i] = to_f32(x.v[i]);
      const float v = s.valid && t0 + s.q + Q * i < end ? step_of(to_f32(dt.v[i]), bias, p.softplus, slope) : 0.0f;
      step.put(ls, s.q, s.c, i, v);
      in.put(lu, s.q, s.c, i, v * xs[i]);
      steps += v;
      if (OUT && pz) zs[i] = to_f32(z.v[i]);
    }
    b.put(lb, s.lane);
    if (OUT) c.put(lc, s.lane);
    wave_order();
    fetch(t0 + kScanTile);
    float part[kScanTile];
#pragma unroll
    for (int k = 0; k < kScanTile / 4; ++k) {
      const Four32 st = step.four(ls, s.c, k), u = in.four(lu, s.c, k);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = 4 * k + j;
        const Four32 bt = *reinterpret_cast<const Four32*>(lb + t * 4 * Q + 4 * s.q);
        Four32 ct;
        if (OUT) ct = *reinterpret_cast<const Four32*>(lc + t * 4 * Q + 4 * s.q);
        float y = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          h.v[r] = __builtin_fmaf(decay_of(st.v[j], a.v[r]), h.v[r], u.v[j] * bt.v[r]);
          if (OUT) y = __builtin_fmaf(ct.v[r], h.v[r], y);
        }
        part[t] = y;
      }
    }
    if (!OUT) continue;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      float sums[Q];
#pragma unroll
      for (int j = 0; j < Q; ++j) sums[j] = part[i * Q + j];
      float y = __builtin_fmaf(skip, xs[i], fold_states<Q>(sums));
      if (pz) y *= activate(zs[i], kActSilu);
      if (s.valid && t0 + s.q + Q * i < end) py[(long long)i * Q * p.channels] = from_f32<T>(y);
    }
    py += (long long)kScanTile * p.channels;
  }
  if (!OUT) {
    reinterpret_cast<Four32*>(p.seg_state)[(s.seg * s.units + s.unit) * 64 + s.lane] = h;
    p.seg_steps[(s.seg * s.units + s.unit) * 64 + s.lane] = sum_states<Q>(steps);
    return;
  }
  T* const y = static_cast<T*>(p.y) + s.row * p.tokens * p.channels + s.channel;
  for (long long t = max(end, seg_begin) + s.q; t < seg_end; t += Q)
    if (s.valid) y[t * p.channels] = T(0);
  if (p.state_out && s.seg == p.segments - 1)
    store_states(p.state_out + (s.row * p.channels + s.channel) * p.n, p.n, s.q, s.valid, h);
}

// Waves of a workgroup of the backward: their channels' shares of db and dc are added in LDS, so at least 32 channels
template <int Q>
constexpr int kBackWaves = Q <= 4 ? 4 : 8;

// The gradients, tile by tile from the last: a tile's states are computed again from the kept one before it.
// SUM: the segments' own sums of e g from zero at their ends, and their steps' sums.
template <typename T, int Q, bool SUM>
__global__ __launch_bounds__(64 * kBackWaves<Q>) void scan_backward_kernel(ScanArgs p, long long first_block) {
  constexpr int kOwn = kScanTile / Q, kWaves = kBackWaves<Q>, kChannels = 64 / Q;
  __shared__ float rows[kWaves][2][64 * Q];
  __shared__ float planes[kWaves][3][Q == 1 ? 1 : kPlaneWords<Q>];
  __shared__ float shares[SUM ? 1 : kWaves][SUM ? 1 : kScanTile * 8 * Q];
  const ScanPlace<Q> s = scan_place<Q>(p, first_block + blockIdx.x, kWaves);
  const bool idle = s.tile * kChannels >= p.channels / p.groups;  // (takes part in the barriers)
  if (SUM && idle) return;
  const int wave = threadIdx.x / 64;
  float *const lb = rows[wave][0], *const lc = rows[wave][1];
  float *const ls = planes[wave][0], *const lu = planes[wave][1], *const lv = planes[wave][2];
  const long long seg_begin = s.seg * p.seg_tokens, seg_end = min(p.tokens, seg_begin + p.seg_tokens), end = min(scan_end(p, s.row), seg_end);

  const T* const px = static_cast<const T*>(p.x) + s.row * p.x_sb + s.channel;
  const T* const pdt = static_cast<const T*>(p.dt) + s.row * p.dt_sb + s.channel;
  const T* const pz = p.z ? static_cast<const T*>(p.z) + s.row * p.z_sb + s.channel : nullptr;
  const T* const pb = static_cast<const T*>(p.b) + s.row * p.b_sb + s.group * p.b_sg;
  const T* const pc = static_cast<const T*>(p.c) + s.row * p.c_sb + s.group * p.c_sg;
  const long long plane = s.row * p.tokens * p.channels + s.channel;  // of contiguous (batch, tokens, channels)
  const T* const pdy = static_cast<const T*>(p.dy) + plane;
  const Four32* const kept = reinterpret_cast<const Four32*>(p.kept) + s.unit * kept_states(p) * 64 + s.lane;

  Four32 a = load_states(p.a + (long long)s.channel * p.n, p.n, s.q, s.valid), carry = {}, da = {};
#pragma unroll
  for (int r = 0; r < 4; ++r) a.v[r] *= kLog2E;
  const float bias = p.dt_bias ? p.dt_bias[s.channel] : 0.0f, skip = p.d ? p.d[s.channel] : 0.0f;
  if (!SUM) {
    if (p.segments > 1)
      carry = reinterpret_cast<const Four32*>(p.seg_state)[(s.seg * s.units + s.unit) * 64 + s.lane];
    else if (p.dstate_out)
      carry = load_states(p.dstate_out + (s.row * p.channels + s.channel) * p.n, p.n, s.q, s.valid);
  }
  float steps = 0.0f, dskip = 0.0f, dbias = 0.0f;
  ScanTokens<T, Q> x, dt, z, dy;
  ScanRows<T, Q> b, c;
  Four32 h0 = {};
  const auto fetch = [&](long long t0) {
    const long long t = t0 + s.q;
    dt.load(pdt + t * p.dt_st, p.dt_st, t, end, s.valid);
    dy.load(pdy + t * p.channels, p.channels, t, end, s.valid);
    c.load(pc + t0 * p.c_st, p.c_st, p.n, s.lane, t0, end);
    if (pz) z.load(pz + t * p.z_st, p.z_st, t, end, s.valid);
    if (!SUM) {
      x.load(px + t * p.x_st, p.x_st, t, end, s.valid);
      b.load(pb + t0 * p.b_st, p.b_st, p.n, s.lane, t0, end);
      if (t0 > 0)
        h0 = s.valid ? kept[(t0 / kScanStretch - 1) * 64] : Four32{};
      else
        h0 = p.state_in ? load_states(p.state_in + (s.row * p.channels + s.channel) * p.n, p.n, s.q, s.valid) : Four32{};
    }
  };
  const long long last = end > seg_begin ? seg_begin + (end - 1 - seg_begin) / kScanTile * kScanTile : seg_begin - kScanTile;
  if (last >= seg_begin) fetch(last);
  for (long long t0 = last; t0 >= seg_begin; t0 -= kScanTile) {
    ScanPlane<Q> step, in, out;
    float xs[kOwn], ss[kOwn], slope[kOwn], vs[kOwn], zs[kOwn];  // zs: dy silu'(z)
    wave_order();
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const bool live = s.valid && t0 + s.q + Q * i < end;
      const float v = step_of(to_f32(dt.v[i]), bias, p.softplus, slope[i]);
      ss[i] = live ? v : 0.0f;
      step.put(ls, s.q, s.c, i, ss[i]);
      steps += ss[i];
      vs[i] = to_f32(dy.v[i]);
      zs[i] = 0.0f;
      if (pz) {
        const float zi = to_f32(z.v[i]);
        zs[i] = vs[i] * activation_slope(zi, kActSilu);
        vs[i] *= activate(zi, kActSilu);
      }
      out.put(lv, s.q, s.c, i, vs[i]);
      if (!SUM) {
        xs[i] = to_f32(x.v[i]);
        in.put(lu, s.q, s.c, i, ss[i] * xs[i]);
      }
    }
    c.put(lc, s.lane);
    if (!SUM) b.put(lb, s.lane);
    wave_order();
    const Four32 start = h0;
    if (t0 > seg_begin) fetch(t0 - kScanTile);
    if constexpr (SUM) {
#pragma unroll
      for (int k = kScanTile / 4 - 1; k >= 0; --k) {
        const Four32 st = step.four(ls, s.c, k), vt = out.four(lv, s.c, k);
#pragma unroll
        for (int j = 3; j >= 0; --j) {
          const Four32 ct = *reinterpret_cast<const Four32*>(lc + (4 * k + j) * 4 * Q + 4 * s.q);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            carry.v[r] = decay_of(st.v[j], a.v[r]) * __builtin_fmaf(ct.v[r], vt.v[j], carry.v[r]);
        }
      }
    } else {
      Four32 hs[kScanTile], h = start, da_tile = {};
#pragma unroll
      for (int k = 0; k < kScanTile / 4; ++k) {
        const Four32 st = step.four(ls, s.c, k), u = in.four(lu, s.c, k);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const Four32 bt = *reinterpret_cast<const Four32*>(lb + (4 * k + j) * 4 * Q + 4 * s.q);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            h.v[r] = __builtin_fmaf(decay_of(st.v[j], a.v[r]), h.v[r], u.v[j] * bt.v[r]);
          hs[4 * k + j] = h;
        }
      }
      float sum_b[kScanTile], sum_a[kScanTile], sum_y[kScanTile];
#pragma unroll
      for (int k = kScanTile / 4 - 1; k >= 0; --k) {
        const Four32 st = step.four(ls, s.c, k), u = in.four(lu, s.c, k), vt = out.four(lv, s.c, k);
#pragma unroll
        for (int j = 3; j >= 0; --j) {
          const int t = 4 * k + j;
          const Four32 bt = *reinterpret_cast<const Four32*>(lb + t * 4 * Q + 4 * s.q);
          const Four32 ct = *reinterpret_cast<const Four32*>(lc + t * 4 * Q + 4 * s.q);
          const Four32 before = t ? hs[t ? t - 1 : 0] : start;
          float v[8];
          sum_b[t] = sum_a[t] = sum_y[t] = 0.0f;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float g = __builtin_fmaf(ct.v[r], vt.v[j], carry.v[r]);
            carry.v[r] = decay_of(st.v[j], a.v[r]) * g;
            const float flow = carry.v[r] * before.v[r];
            sum_b[t] = __builtin_fmaf(g, bt.v[r], sum_b[t]);
            sum_a[t] = __builtin_fmaf(flow, a.v[r], sum_a[t]);
            sum_y[t] = __builtin_fmaf(ct.v[r], hs[t].v[r], sum_y[t]);
            da_tile.v[r] = __builtin_fmaf(flow, st.v[j], da_tile.v[r]);
            v[r] = g * u.v[j];
            v[4 + r] = vt.v[j] * hs[t].v[r];
          }
          // over the channels: db's and dc's shares part at the first level, their states at the next two
          constexpr int kTop = kChannels / 2 == 4 ? 7 : kChannels / 2, kMid = kChannels / 4 == 4 ? 7 : kChannels / 4;
          float w[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) w[r] = fold<kTop>(v[r], v[r + 4]);
          w[0] = fold<kMid>(w[0], w[2]);
          w[1] = fold<kMid>(w[1], w[3]);
          const int which = s.c / (kChannels / 2), half = s.c / (kChannels / 4) % 2;
          float* const to = shares[wave] + t * 8 * Q + which * 4 * Q + 4 * s.q + 2 * half;
          if constexpr (kChannels == 4) {
            to[0] = w[0];
            to[1] = w[1];
          } else {
            constexpr int kLow = kChannels / 8 == 4 ? 7 : kChannels / 8;
            float sum = fold<kLow>(w[0], w[1]);
            if constexpr (kChannels >= 64) sum = fold<7>(sum);
            if constexpr (kChannels >= 32) sum = fold<2>(sum);
            if constexpr (kChannels >= 16) sum = fold<1>(sum);
            if (s.c % (kChannels / 8) == 0) to[s.c / (kChannels / 8) % 2] = sum;
          }
        }
      }
      float dskip_tile = 0.0f, dbias_tile = 0.0f;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        float vb[Q], va[Q], vy[Q];
#pragma unroll
        for (int j = 0; j < Q; ++j) vb[j] = sum_b[i * Q + j], va[j] = sum_a[i * Q + j], vy[j] = sum_y[i * Q + j];
        const float gb = fold_states<Q>(vb), ga = fold_states<Q>(va) * (1.0f / kLog2E);
        const float y = pz ? __builtin_fmaf(skip, xs[i], fold_states<Q>(vy)) : 0.0f;
        const float ddt = __builtin_fmaf(xs[i], gb, ga) * slope[i];
        if (s.valid && t0 + s.q + Q * i < end) {
          const long long at = plane + (t0 + s.q + Q * i) * p.channels;
          if (p.dx) static_cast<T*>(p.dx)[at] = from_f32<T>(__builtin_fmaf(ss[i], gb, skip * vs[i]));
          if (p.ddt) static_cast<T*>(p.ddt)[at] = from_f32<T>(ddt);
          if (p.dz) static_cast<T*>(p.dz)[at] = from_f32<T>(zs[i] * y);
          dskip_tile = __builtin_fmaf(vs[i], xs[i], dskip_tile);
          dbias_tile += ddt;
        }
      }
      // (a tile's terms by themselves first: long sums keep their last bits)
      dskip += dskip_tile;
      dbias += dbias_tile;
#pragma unroll
      for (int r = 0; r < 4; ++r) da.v[r] += da_tile.v[r];
      if (p.shared_parts) {
        __syncthreads();
        const long long part = s.tile / kWaves;
        float* const to = p.shared_parts + ((part * p.batch + s.row) * p.tokens + t0) * p.groups * 8 * Q + s.group * 8 * Q;
        for (int i = threadIdx.x; i < kScanTile * 8 * Q; i += 64 * kWaves) {
          if (t0 + i / (8 * Q) >= end) break;
          float sum = 0.0f;
#pragma unroll
          for (int w = 0; w < kWaves; ++w) sum += shares[w][i];
          to[(long long)(i / (8 * Q)) * p.groups * 8 * Q + i % (8 * Q)] = sum;
        }
        __syncthreads();
      }
    }
  }
  if (SUM) {
    reinterpret_cast<Four32*>(p.seg_state)[(s.seg * s.units + s.unit) * 64 + s.lane] = carry;
    p.seg_steps[(s.seg * s.units + s.unit) * 64 + s.lane] = sum_states<Q>(steps);
    return;
  }
  if (idle) return;
  if (s.valid)
    for (long long t = max(end, seg_begin) + s.q; t < seg_end; t += Q) {
      const long long at = plane + t * p.channels;
      if (p.dx) static_cast<T*>(p.dx)[at] = T(0);
      if (p.ddt) static_cast<T*>(p.ddt)[at] = T(0);
      if (p.dz) static_cast<T*>(p.dz)[at] = T(0);
    }
  if (p.dstate_in && s.seg == 0)
    store_states(p.dstate_in + (s.row * p.channels + s.channel) * p.n, p.n, s.q, s.valid, carry);
  if (p.channel_parts) {
    // (seg, unit, lane): four of da, then dd and ddt_bias
    const long long at = (s.seg * s.units + s.unit) * 64 + s.lane, all = p.segments * s.units * 64;
    reinterpret_cast<Four32*>(p.channel_parts)[at] = da;
    p.channel_parts[4 * all + at] = sum_states<Q>(dskip);
    p.channel_parts[5 * all + at] = sum_states<Q>(dbias);
  }
}

enum ScanMode { kScanSums, kScanForward, kScanBackSums, kScanBackward };

template <typename T, int Q>
hipError_t scan_launch(const ScanArgs& p, ScanMode mode) {
  const int waves = mode == kScanBackSums || mode == kScanBackward ? kBackWaves<Q> : kScanWaves;
  const long long tiles = (p.channels / p.groups + 64 / Q - 1) / (64 / Q);
  const long long blocks = (tiles + waves - 1) / waves * p.groups * p.batch * p.segments;
  for (long long first = 0; first < blocks; first += max_blocks(64 * waves)) {
    const dim3 grid((unsigned)std::min(blocks - first, max_blocks(64 * waves))), block(64 * waves);
    if (mode == kScanSums) hipLaunchKernelGGL((scan_forward_kernel<T, Q, false>), grid, block, 0, p.stream, p, first);
    if (mode == kScanForward) hipLaunchKernelGGL((scan_forward_kernel<T, Q, true>), grid, block, 0, p.stream, p, first);
    if (mode == kScanBackSums) hipLaunchKernelGGL((scan_backward_kernel<T, Q, true>), grid, block, 0, p.stream, p, first);
    if (mode == kScanBackward) hipLaunchKernelGGL((scan_backward_kernel<T, Q, false>), grid, block, 0, p.stream, p, first);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// lanes of a channel
inline int scan_lanes(int n) { return n <= 4 ? 1 : n <= 8 ? 2 : n <= 16 ? 4 : n <= 32 ? 8 : 16; }

template <typename T>
hipError_t scan_typed(const ScanArgs& p, ScanMode mode) {
  switch (scan_lanes(p.n)) {
    case 1: return scan_launch<T, 1>(p, mode);
    case 2: return scan_launch<T, 2>(p, mode);
    case 4: return scan_launch<T, 4>(p, mode);
    case 8: return scan_launch<T, 8>(p, mode);
  }
  return scan_launch<T, 16>(p, mode);
}

hipError_t scan_f32(const ScanArgs& p, ScanMode mode);
hipError_t scan_bf16(const ScanArgs& p, ScanMode mode);
hipError_t scan_f16(const ScanArgs& p, ScanMode mode);

}  // namespace tfa
