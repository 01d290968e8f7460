// The selective scan over whole sequences and its gradients (kernels_scan_{f32,bf16,f16}.hip instantiate it by type).
//
//   s_t = softplus(dt_t + dt_bias),  h_t[n] = exp(s_t a[n]) h_{t-1}[n] + s_t x_t b_t[n],  y_t = (sum_n c_t[n] h_t[n] + d x_t) silu(z_t)
// for every channel, b and c shared by the channels of a group.  With e = exp(s_t a), v_t = dy_t silu(z_t):
//   g_t[n] = v_t c_t[n] + e_{t+1}[n] g_{t+1}[n],  db_t[n] = sum over channels of g_t[n] s_t x_t,  dc_t[n] = the same of v_t h_t[n],
//   ds_t = x_t sum_n g_t[n] b_t[n] + sum_n a[n] f_t[n],  dx_t = s_t sum_n g_t[n] b_t[n] + d v_t,  da[n] = sum_t s_t f_t[n],
//   where f_t = g_t e_t h_{t-1},  dz_t = dy_t silu'(z_t) (sum_n c_t[n] h_t[n] + d x_t)
//
// A wave takes 64 / Q channels of a row and group, Q lanes a channel with R states each (4 x 1, 2 or 4 up to 16 states, 8 and 16 x 4 above), and walks
// along the tokens in tiles of 16.  For what belongs to a channel and token alone (softplus, gates, loads, stores) lane q of a channel takes
// every Q-th token, so nothing of it is done twice; the tokens' s and s x go to the channel's lanes through LDS, as do b and
// c, whose rows all channels of a group share.  Sums over the lanes of a channel are folded: Q tokens' sums at once, each ending in
// the lane of its token.
//
// Bound by vector instructions (an exponential takes two instructions' time), not by memory.  A token and wave of 16 channels of 16 states take 39
// of them forward, 24 for the recurrence and its dot products alone, and about 100 backward.  8 x 4096 tokens of 2048 channels, bf16: backward
// 900 to 924 us in two segments (and 130 to 134 for their sums), forward 443 with one wave a SIMD, 400 in scan_pairs.h; 1 x 65536 of 1024 in 64
// segments, four waves a SIMD, 317 and 222 for the sums.  Products b u by 4 x 4 matrix instructions are 16 instructions fewer in two tokens and took
// the same time, 8 lanes a channel of two states 557 and 1190 us.
// The backward also runs out of scalar registers: 54 to 70 of them (34 to 39 at 33 to 64 states) lie in lanes of vector registers and are read back
// in every tile, a part of its instructions.  At 33 to 64 states its LDS of 106 KB leaves a compute unit one workgroup, one wave a SIMD, and 16
// channels whose shares of db and dc are added there: 32 B of workspace a value of the sequence where up to 16 states take 2.
// A group of channels that does not fill a workgroup (4 waves, 8 at 17 to 32 states) leaves waves without channels, which backward run the pass for
// its barriers: 64 x 626 tokens of 64 channels of 16 states, bf16, training 112 us in one group, 231 in four of 16 channels.
#pragma once
#include "scan_device.h"

#include <algorithm>

namespace tfa {

template <int R>
struct alignas(4 * R) States {
  float v[R];
};
typedef States<4> Four32;

// Where a wave and its lane stand.  What is one for the wave is kept where the compiler sees it (scalar registers): addresses are a scalar
// part and 32 bits of the lane's own.
template <int Q>
struct ScanPlace {
  static constexpr int kChannels = 64 / Q;
  int wave, lane, q, c;       // c: channel of the tile
  long long row;
  int group, tile, base;      // base: the tile's first channel
  int own;                    // c, or where there is no such channel the last that there is
  bool valid;                 // whether there is such a channel
  bool idle;                  // whether there is no such tile
  long long unit, units;
  int seg;
};

// Ragged rows are given out by length, so that the compute units' sums of them are about the same: the longest first, and every other layer
// of workgroups over the 256 compute units from the shortest on (a wave that starts late has little to do).  64 rows of up to 626 tokens, 512
// channels of 16 states by scan_forward_kernel, two workgroups a compute unit: 80.5 us, in their own order 88.6.  Batches of more rows than threads
// keep their order.
template <int THREADS>
__device__ __forceinline__ long long scan_row(const ScanArgs& p, long long slot, int blocks) {
  if (!p.lengths || p.batch > THREADS || p.batch == 1) return slot;
  __shared__ int found;
  // (layers 0, 2, ... take the ranks from the front, 1, 3, ... from the back)
  const int layer_rows = max(1, 256 / blocks), layer = (int)slot / layer_rows, first = layer * layer_rows;
  const int in = (int)slot - first, rank = layer % 2 == 0 ? layer / 2 * layer_rows + in : (int)p.batch - 1 - (layer / 2 * layer_rows + in);
  const int t = threadIdx.x;
  if (t < p.batch) {
    const long long own = p.lengths[t];
    int before = 0;
    for (int i = 0; i < (int)p.batch; ++i) {
      const long long other = p.lengths[i];
      before += other > own || (other == own && i < t);
    }
    if (before == rank) found = t;
  }
  __syncthreads();
  return found;
}

template <int Q, int WAVES, int SPLIT = 1>
__device__ __forceinline__ ScanPlace<Q> scan_place(const ScanArgs& p, long long block) {
  ScanPlace<Q> s;
  const int each = p.channels / p.groups, tiles = (each + s.kChannels - 1) / s.kChannels, across = (tiles + WAVES / SPLIT - 1) / (WAVES / SPLIT);
  s.wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  s.lane = threadIdx.x % 64;
  s.q = s.lane / s.kChannels;
  s.c = s.lane % s.kChannels;
  s.tile = (int)(block % across) * (WAVES / SPLIT) + s.wave / SPLIT;
  block /= across;
  s.group = (int)(block % p.groups);
  block /= p.groups;
  s.row = __builtin_amdgcn_readfirstlane((int)scan_row<64 * WAVES>(p, block % p.batch, across * p.groups));
  s.seg = (int)(block / p.batch);
  s.idle = s.tile >= tiles;
  const int tile = min(s.tile, tiles - 1), left = each - tile * s.kChannels;
  s.valid = !s.idle && s.c < left;
  s.own = min(s.c, left - 1);
  s.base = s.group * each + tile * s.kChannels;
  s.units = p.batch * p.groups * tiles;
  s.unit = (s.row * p.groups + s.group) * tiles + tile;
  return s;
}

// A wave's own LDS: nothing but the order of its instructions is needed between its lanes' writes and reads.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A workgroup's barrier for what it shares in LDS: loads and stores of memory stay on their way.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

constexpr int kPlaneRow = kScanTile + 4;  // words of a channel's tokens: rows at 16 bytes that spread over the banks

// A value of every channel and token of the tile in LDS: lane q puts tokens q, q + Q, ...; all lanes of a channel read four neighbours.
template <int Q>
__device__ __forceinline__ void put_token(float* lds, int q, int c, int i, float v) {
  lds[c * kPlaneRow + q + Q * i] = v;
}
__device__ __forceinline__ Four32 four_tokens(const float* lds, int c, int k) {
  return *reinterpret_cast<const Four32*>(lds + c * kPlaneRow + 4 * k);
}
template <int Q>
constexpr int kPlaneWords = 64 / Q * kPlaneRow;

// p, the same for a wave, and a lane's own 32 bits of an address: one register and no arithmetic in 64 bits.  (The compiler must not see that
// the lane's part stays as it is from tile to tile: it would keep the sums of both, in 64 bits, in vector registers.)
template <typename T>
__device__ __forceinline__ T* lane_address(T* p, unsigned bytes) {
  asm volatile("" : "+v"(bytes));
  typedef std::conditional_t<std::is_const_v<T>, const char, char> Byte;
  return reinterpret_cast<T*>(reinterpret_cast<Byte*>(p) + bytes);
}

// The tokens q, q + Q, ... of a tile of one operand; those past the end are the last one's again.
template <typename T, int Q>
struct ScanTokens {
  T v[kScanTile / Q];
  // p: the tile's first channel at its first token; left: tokens from there to the end, at least one
  __device__ __forceinline__ void load(const T* p, long long st, const ScanPlace<Q>& s, int left) {
    if (left >= kScanTile) {
      const unsigned at = (s.q * (unsigned)st + s.own) * sizeof(T);
#pragma unroll
      for (int i = 0; i < kScanTile / Q; ++i) v[i] = *lane_address(p + i * Q * st, at);
    } else {
#pragma unroll
      for (int i = 0; i < kScanTile / Q; ++i) v[i] = *lane_address(p, (__umul24(min(s.q + Q * i, left - 1), st) + s.own) * (unsigned)sizeof(T));
      // (keeps the compiler from making one load of both ways' with an address in 64 bits of registers)
      asm volatile("");
    }
  }
};
// A tile's rows of b or c, 16 by Q R, zeros past n and past the end.  With 4 lanes a channel a row of 16 lanes has one q: lane l of it
// keeps the R states of token l % 16, and products take them from there.  Else they go through LDS.
template <typename T, int Q, int R>
struct ScanRows {
  static constexpr int kParts = Q == 4 ? 1 : Q / 4, kBytes = R * (int)sizeof(T), kWords = kBytes < 4 ? 1 : kBytes / 4;
  unsigned w[kParts][kWords];  // as they lie in memory, so that nothing waits for them before they are put to use
  static __device__ __forceinline__ int token(int lane, int i) { return Q == 4 ? lane % 16 : (lane + 64 * i) / Q; }
  static __device__ __forceinline__ int state(int lane, int i) { return (Q == 4 ? lane / 16 : (lane + 64 * i) % Q) * R; }
  // p: the tile's first token; first: the state that lane 0 begins with; n: all states, at least R.  Behind the last R a lane reads these.
  __device__ __forceinline__ void load(const T* p, long long st, int n, int first, int lane, int left) {
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const unsigned at = __umul24(min(token(lane, i), left - 1), st);
      // (one access, which the memory takes at any address of an element)
      const T* const from = lane_address(p, (at + min(first + state(lane, i), n - R)) * (unsigned)sizeof(T));
      if constexpr (kBytes < 4)
        w[i][0] = *reinterpret_cast<const unsigned short*>(from);
      else
        __builtin_memcpy(w[i], from, kBytes);
    }
  }
  // `ahead` values more from the front dropped
  __device__ __forceinline__ void drop(int i, int ahead) {
    if constexpr (R == 4 && sizeof(T) == 2) {
      const unsigned long long v = (w[i][0] | (unsigned long long)w[i][1] << 32) >> 16 * (ahead & 3);
      w[i][0] = (unsigned)v, w[i][1] = (unsigned)(v >> 32);
    } else if constexpr (R == 2 && sizeof(T) == 2) {
      w[i][0] >>= 16 * (ahead & 1);
    } else if constexpr (R > 1) {
      // (by masks: a choice between two of them would become a choice between their places in memory)
      const unsigned one = -(unsigned)(ahead & 1), two = -(unsigned)(ahead >> 1 & 1);
#pragma unroll
      for (int r = 0; r < R - 1; ++r) w[i][r] = (w[i][r + 1] & one) | (w[i][r] & ~one);
      if constexpr (R == 4) w[i][0] = (w[i][2] & two) | (w[i][0] & ~two), w[i][1] = (w[i][3] & two) | (w[i][1] & ~two);
    }
  }
  __device__ __forceinline__ float value(int i, int r) const {
    if constexpr (sizeof(T) == 4)
      return __uint_as_float(w[i][r]);
    else
      return to_f32(__builtin_bit_cast(T, (unsigned short)(w[i][r / 2] >> 16 * (r % 2))));
  }
};
template <int Q, int R>
struct ScanBank {
  States<R> own;
  template <typename T>
  __device__ __forceinline__ void put(ScanRows<T, Q, R> rows, float* lds, int n, int first, int lane, int left) {
    const bool all = n - first >= Q * R && left == kScanTile;
#pragma unroll
    for (int i = 0; i < rows.kParts; ++i) {
      const int t = rows.token(lane, i), k = first + rows.state(lane, i);
      if (n % R) rows.drop(i, max(k + R - n, 0));  // (the lane that has the last states has read some before its own)
#pragma unroll
      for (int r = 0; r < R; ++r) own.v[r] = rows.value(i, r);
      if (!all) {
#pragma unroll
        for (int r = 0; r < R; ++r) own.v[r] = k + r < n && t < left ? own.v[r] : 0.0f;
      }
      if (Q > 4) *reinterpret_cast<States<R>*>(lds + R * (lane + 64 * i)) = own;
    }
  }
  __device__ __forceinline__ States<R> at(const float* lds, int t, int q) const {
    return *reinterpret_cast<const States<R>*>(lds + (t * Q + q) * R);
  }
  // with the values of a lane's states at tokens t and t + 1: their products with u0 and u1, and the dot products with x0 and x1
  template <int t>
  __device__ __forceinline__ void products(const float* lds, int q, float u0, float u1, float (&out0)[R], float (&out1)[R]) const {
    if constexpr (Q == 4) {
      RowLane<t>::products(own.v, u0, u1, out0, out1);
    } else {
      const States<R> v0 = at(lds, t, q), v1 = at(lds, t + 1, q);
#pragma unroll
      for (int r = 0; r < R; ++r) out0[r] = v0.v[r] * u0, out1[r] = v1.v[r] * u1;
    }
  }
  template <int t>
  __device__ __forceinline__ void dots(const float* lds, int q, const float (&x0)[R], const float (&x1)[R], float& sum0, float& sum1) const {
    if constexpr (Q == 4) {
      RowLane<t>::dots(own.v, x0, x1, sum0, sum1);
    } else {
      const States<R> v0 = at(lds, t, q), v1 = at(lds, t + 1, q);
      sum0 = sum1 = 0.0f;
#pragma unroll
      for (int r = 0; r < R; ++r) sum0 = __builtin_fmaf(v0.v[r], x0[r], sum0), sum1 = __builtin_fmaf(v1.v[r], x1[r], sum1);
    }
  }
  // token t's products with u, added to sums
  template <int t>
  __device__ __forceinline__ void add(const float* lds, int q, float u, float (&sum)[R]) const {
    if constexpr (Q == 4) {
      RowLane<t>::add(own.v, u, sum);
    } else {
      const States<R> v = at(lds, t, q);
#pragma unroll
      for (int r = 0; r < R; ++r) sum[r] = __builtin_fmaf(v.v[r], u, sum[r]);
    }
  }
};
// g += c_t u, then b_t . g and c_t . h
template <int t, int Q, int R>
__device__ __forceinline__ void reverse_token(const ScanBank<Q, R>& b, const float* lb, const ScanBank<Q, R>& c, const float* lc, int q, float u,
                                              const States<R>& h, States<R>& g, float& sum_b, float& sum_c) {
  if constexpr (Q == 4) {
    RowLane<t>::reverse(b.own.v, c.own.v, u, h.v, g.v, sum_b, sum_c);
  } else {
    const States<R> bt = b.at(lb, t, q), ct = c.at(lc, t, q);
    sum_b = sum_c = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      g.v[r] = __builtin_fmaf(ct.v[r], u, g.v[r]);
      sum_b = __builtin_fmaf(bt.v[r], g.v[r], sum_b);
      sum_c = __builtin_fmaf(ct.v[r], h.v[r], sum_c);
    }
  }
}
template <int Q, int R>
constexpr int kBankWords = Q == 4 ? 1 : 16 * Q * R;

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

// a lane's states of a channel in (channels, n) fp32
template <int R>
__device__ __forceinline__ States<R> load_states(const float* p, int n, int q, bool valid) {
  States<R> s;
#pragma unroll
  for (int r = 0; r < R; ++r) s.v[r] = valid && R * q + r < n ? p[R * q + r] : 0.0f;
  return s;
}
template <int R>
__device__ __forceinline__ void store_states(float* p, int n, int q, bool valid, const States<R>& s) {
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (valid && R * q + r < n) p[R * q + r] = s.v[r];
}

__device__ __forceinline__ long long scan_end(const ScanArgs& p, long long row) {
  return p.lengths ? min(max(p.lengths[row], 0LL), p.tokens) : p.tokens;
}
__device__ __forceinline__ long long kept_states(const ScanArgs& p) { return p.tokens > 0 ? (p.tokens - 1) / kScanStretch : 0; }

// a tile's own steps s_t and their slopes by dt_t
template <typename T, int Q>
__device__ __forceinline__ void steps_of(const ScanTokens<T, Q>& dt, float bias, bool soft, float (&step)[kScanTile / Q], float (&slope)[kScanTile / Q]) {
#pragma unroll
  for (int i = 0; i < kScanTile / Q; ++i) step[i] = to_f32(dt.v[i]) + bias, slope[i] = 1.0f;
  if (soft) {
#pragma unroll
    for (int i = 0; i < kScanTile / Q; ++i) step[i] = softplus(step[i], slope[i]);
  }
}
// zeros in the tokens past the end and the channels past the last, which take no part in anything that is shared
template <int Q>
__device__ __forceinline__ void clear_dead(const ScanPlace<Q>& s, int left, float (&v)[kScanTile / Q]) {
#pragma unroll
  for (int i = 0; i < kScanTile / Q; ++i) v[i] = s.valid && s.q + Q * i < left ? v[i] : 0.0f;
}
// The same tokens to a contiguous (batch, tokens, channels) operand; p as above; all: the wave has all of its channels and tokens.
template <typename T, int Q>
__device__ __forceinline__ void store_tokens(T* p, int st, const ScanPlace<Q>& s, int left, bool all, const float (&v)[kScanTile / Q]) {
  const unsigned at = (s.q * (unsigned)st + s.own) * sizeof(T);
  if (all) {
#pragma unroll
    for (int i = 0; i < kScanTile / Q; ++i) *lane_address(p + (long long)i * Q * st, at) = from_f32<T>(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kScanTile / Q; ++i)
      if (s.valid && s.q + Q * i < left) *lane_address(p + (long long)i * Q * st, at) = from_f32<T>(v[i]);
  }
}
// Zeros in the tokens from `from` to `to`; p: the wave's first channel at token 0
template <typename T, int Q>
__device__ __forceinline__ void zero_tokens(T* p, int st, const ScanPlace<Q>& s, long long from, long long to) {
  if (s.valid)
    for (long long t = from + s.q; t < to; t += Q) p[t * st + s.own] = T(0);
}
__device__ __forceinline__ int tile_left(long long end, long long t0) { return (int)min(end - t0, (long long)kScanTile); }

constexpr int kScanWaves = 4;  // of a workgroup of the forward and the sums

// OUT: the sequences, or their segments from seg_state's states.  Else the segments' own sums from zero, and their steps' sums.
template <typename T, int Q, int R, bool OUT>
__global__ __launch_bounds__(64 * kScanWaves) void scan_forward_kernel(ScanArgs p, long long first_block) {
  constexpr int kOwn = kScanTile / Q;
  __shared__ float rows[kScanWaves][2][kBankWords<Q, R>];
  __shared__ float planes[kScanWaves][2][kPlaneWords<Q>];
  const ScanPlace<Q> s = scan_place<Q, kScanWaves>(p, first_block + blockIdx.x);
  if (s.idle) return;
  float *const lb = rows[s.wave][0], *const lc = rows[s.wave][1], *const ls = planes[s.wave][0], *const lu = planes[s.wave][1];
  const long long seg_tokens = OUT ? p.seg_tokens : p.seg_tokens / p.fine;
  const long long seg_begin = s.seg * seg_tokens, seg_end = min(p.tokens, seg_begin + seg_tokens), end = min(scan_end(p, s.row), seg_end);

  const T* px = static_cast<const T*>(p.x) + s.row * p.x_sb + seg_begin * p.x_st + s.base;
  const T* pdt = static_cast<const T*>(p.dt) + s.row * p.dt_sb + seg_begin * p.dt_st + s.base;
  const T* pz = p.z ? static_cast<const T*>(p.z) + s.row * p.z_sb + seg_begin * p.z_st + s.base : nullptr;
  const T* pb = static_cast<const T*>(p.b) + s.row * p.b_sb + seg_begin * p.b_st + s.group * p.b_sg;
  const T* pc = static_cast<const T*>(p.c) + s.row * p.c_sb + seg_begin * p.c_st + s.group * p.c_sg;
  T* const y = OUT ? static_cast<T*>(p.y) + s.row * p.tokens * p.channels + s.base : nullptr;
  const int channel = s.base + s.own;

  States<R> a = load_states<R>(p.a + (long long)channel * p.n, p.n, s.q, s.valid), h = {};
#pragma unroll
  for (int r = 0; r < R; ++r) a.v[r] = rate_of(a.v[r]);
  const float bias = p.dt_bias ? p.dt_bias[channel] : 0.0f, skip = p.d ? p.d[channel] : 0.0f;
  if (OUT) {
    if (p.segments > 1)
      h = reinterpret_cast<const States<R>*>(p.seg_state)[(s.seg * p.fine * s.units + s.unit) * 64 + s.lane];
    else if (p.state_in)
      h = load_states<R>(p.state_in + (s.row * p.channels + channel) * p.n, p.n, s.q, s.valid);
  }
  States<R>* const kept = OUT && p.kept ? reinterpret_cast<States<R>*>(p.kept) + s.unit * kept_states(p) * 64 : nullptr;
  const bool all_valid = __all(s.valid);
  float steps = 0.0f;
  ScanTokens<T, Q> x, dt, z;
  ScanRows<T, Q, R> b, c;
  // the next tile, from where the pointers stand, of `left` tokens to the end
  const auto fetch = [&](int left) {
    x.load(px, p.x_st, s, left);
    dt.load(pdt, p.dt_st, s, left);
    b.load(pb, p.b_st, p.n, 0, s.lane, left);
    if (OUT) {
      c.load(pc, p.c_st, p.n, 0, s.lane, left);
      if (pz) z.load(pz, p.z_st, s, left), pz += kScanTile * p.z_st;
    }
    px += kScanTile * p.x_st, pdt += kScanTile * p.dt_st, pb += kScanTile * p.b_st, pc += kScanTile * p.c_st;
  };
  if (seg_begin < end) fetch(tile_left(end, seg_begin));
  // A tile's results wait in registers until the next one's loads have come: stores and loads are waited for in their order, and stores
  // right ahead of the next tile would be waited for at once.
  float ys[kOwn];
  for (long long t0 = seg_begin; t0 < end; t0 += kScanTile) {
    if (OUT && kept && t0 > 0) *lane_address(kept + (t0 / kScanStretch - 1) * 64, s.lane * (unsigned)sizeof(h)) = h;
    const int left = tile_left(end, t0);
    const bool full = all_valid && left == kScanTile;
    float xs[kOwn], zs[kOwn], own[kOwn], slope[kOwn];
    steps_of<T, Q>(dt, bias, p.softplus, own, slope);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) xs[i] = to_f32(x.v[i]), zs[i] = 1.0f;
    if (!full) clear_dead<Q>(s, left, own), clear_dead<Q>(s, left, xs);
    wave_order();
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      put_token<Q>(ls, s.q, s.c, i, own[i]);
      put_token<Q>(lu, s.q, s.c, i, own[i] * xs[i]);
      if (!OUT) steps += own[i];
    }
    ScanBank<Q, R> bs, cs;
    bs.put(b, lb, p.n, 0, s.lane, left);
    if (OUT) {
      cs.put(c, lc, p.n, 0, s.lane, left);
      if (pz) {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) zs[i] = activate(to_f32(z.v[i]), kActSilu);
      }
    }
    wave_order();
    if (OUT && t0 > seg_begin) store_tokens<T, Q>(y + (t0 - kScanTile) * p.channels, p.channels, s, kScanTile, all_valid, ys);
    if (t0 + kScanTile < end) fetch(tile_left(end, t0 + kScanTile));
    float part[kScanTile];
    Four32 st, u;
    for_each<kScanTile / 2>([&](auto index) TFA_INLINE {
      constexpr int t = 2 * index, j = t % 4;
      if constexpr (j == 0) st = four_tokens(ls, s.c, t / 4), u = four_tokens(lu, s.c, t / 4);
      float in0[R], in1[R];
      bs.template products<t>(lb, s.q, u.v[j], u.v[j + 1], in0, in1);
      States<R> h0 = h;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        h0.v[r] = __builtin_fmaf(decay_of(st.v[j], a.v[r]), h.v[r], in0[r]);
        h.v[r] = __builtin_fmaf(decay_of(st.v[j + 1], a.v[r]), h0.v[r], in1[r]);
      }
      if constexpr (OUT) cs.template dots<t>(lc, s.q, h0.v, h.v, part[t], part[t + 1]);
    });
    if (!OUT) continue;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      float sums[Q];
#pragma unroll
      for (int j = 0; j < Q; ++j) sums[j] = part[i * Q + j];
      settle(sums);
      ys[i] = __builtin_fmaf(skip, xs[i], fold_states<Q>(sums)) * zs[i];
    }
  }
  if (!OUT) {
    reinterpret_cast<States<R>*>(p.seg_state)[(s.seg * s.units + s.unit) * 64 + s.lane] = h;
    p.seg_steps[(s.seg * s.units + s.unit) * 64 + s.lane] = sum_states<Q>(steps);
    return;
  }
  if (seg_begin < end) {
    const long long t0 = seg_begin + (end - 1 - seg_begin) / kScanTile * kScanTile;
    const int left = tile_left(end, t0);
    store_tokens<T, Q>(y + t0 * p.channels, p.channels, s, left, all_valid && left == kScanTile, ys);
  }
  zero_tokens<T, Q>(y, p.channels, s, max(end, seg_begin), seg_end);
  if (p.state_out && s.seg == p.segments - 1)
    store_states<R>(p.state_out + (s.row * p.channels + channel) * p.n, p.n, s.q, s.valid, h);
}

// Waves of a workgroup of the backward: their channels' shares of db and dc are added in LDS, those of 64 channels where LDS holds them
template <int Q>
constexpr int kBackWaves = Q == 8 ? 8 : 4;

// The gradients, tile by tile from the last: a tile's states are computed again from the kept one before it.
// SUM: the segments' own sums of e g from zero at their ends, and their steps' sums.
template <typename T, int Q, int R, bool SUM>
__global__ __launch_bounds__(64 * kBackWaves<Q>, 2) void scan_backward_kernel(ScanArgs p, long long first_block) {
  constexpr int kOwn = kScanTile / Q, kWaves = kBackWaves<Q>, kChannels = 64 / Q;
  __shared__ float rows[kWaves][2][kBankWords<Q, R>];
  __shared__ float planes[kWaves][SUM ? 2 : 6][kPlaneWords<Q>];
  __shared__ float shares[2][SUM ? 1 : kWaves][SUM ? 1 : kScanTile * 2 * Q * R];  // of this tile and the one before
  ScanPlace<Q> s = scan_place<Q, kWaves>(p, first_block + blockIdx.x);
  if (SUM) s.seg += p.fine;  // (nothing comes before the first segment)
  if (SUM && s.idle) return;  // (else it takes part in the barriers)
  float *const lb = rows[s.wave][0], *const lc = rows[s.wave][1];
  // of every channel and token: s, dy silu(z), s x, and what its own lane needs again: x, the slope of s by dt, dy silu'(z)
  float *const ls = planes[s.wave][0], *const lv = planes[s.wave][1], *const lu = planes[s.wave][SUM ? 0 : 2];
  float *const lx = planes[s.wave][SUM ? 0 : 3], *const lslope = planes[s.wave][SUM ? 0 : 4], *const lz = planes[s.wave][SUM ? 0 : 5];
  const long long seg_tokens = SUM ? p.seg_tokens / p.fine : p.seg_tokens;
  const long long seg_begin = s.seg * seg_tokens, seg_end = min(p.tokens, seg_begin + seg_tokens), end = min(scan_end(p, s.row), seg_end);

  const T* const px = static_cast<const T*>(p.x) + s.row * p.x_sb + s.base;
  const T* const pdt = static_cast<const T*>(p.dt) + s.row * p.dt_sb + s.base;
  const T* const pz = p.z ? static_cast<const T*>(p.z) + s.row * p.z_sb + s.base : nullptr;
  const T* const pb = static_cast<const T*>(p.b) + s.row * p.b_sb + s.group * p.b_sg;
  const T* const pc = static_cast<const T*>(p.c) + s.row * p.c_sb + s.group * p.c_sg;
  const long long plane = s.row * p.tokens * p.channels + s.base;  // of contiguous (batch, tokens, channels)
  const T* const pdy = static_cast<const T*>(p.dy) + plane;
  const States<R>* const kept = reinterpret_cast<const States<R>*>(p.kept) + s.unit * kept_states(p) * 64;
  const int channel = s.base + s.own;

  States<R> a = load_states<R>(p.a + (long long)channel * p.n, p.n, s.q, s.valid), carry = {}, da = {};
#pragma unroll
  for (int r = 0; r < R; ++r) a.v[r] = rate_of(a.v[r]);
  const float bias = p.dt_bias ? p.dt_bias[channel] : 0.0f, skip = p.d ? p.d[channel] : 0.0f;
  if (!SUM) {
    if (p.segments > 1)
      carry = reinterpret_cast<const States<R>*>(p.seg_state)[(((long long)(s.seg + 1) * p.fine - 1) * s.units + s.unit) * 64 + s.lane];
    else if (p.dstate_out)
      carry = load_states<R>(p.dstate_out + (s.row * p.channels + channel) * p.n, p.n, s.q, s.valid);
  }
  const bool all_valid = __all(s.valid);
  float steps = 0.0f, dskip = 0.0f, dbias = 0.0f;
  ScanTokens<T, Q> x, dt, z, dy;
  ScanRows<T, Q, R> b, c;
  States<R> h0 = {};
  unsigned kept_lane = s.lane * (unsigned)sizeof(h0);
  const auto fetch = [&](long long t0) {
    const int left = tile_left(end, t0);
    asm volatile("" : "+v"(kept_lane));
    dt.load(pdt + t0 * p.dt_st, p.dt_st, s, left);
    dy.load(pdy + t0 * p.channels, p.channels, s, left);
    c.load(pc + t0 * p.c_st, p.c_st, p.n, 0, s.lane, left);
    if (pz) z.load(pz + t0 * p.z_st, p.z_st, s, left);
    if (!SUM) {
      x.load(px + t0 * p.x_st, p.x_st, s, left);
      b.load(pb + t0 * p.b_st, p.b_st, p.n, 0, s.lane, left);
      if (t0 > 0)
        // (kept_lane: a register of its own.  An address in one that the other way loads into is waited for, and with it the loads above.)
        h0 = *reinterpret_cast<const States<R>*>(reinterpret_cast<const char*>(kept + (t0 / kScanStretch - 1) * 64) + kept_lane);
      else
        h0 = p.state_in ? load_states<R>(p.state_in + (s.row * p.channels + channel) * p.n, p.n, s.q, s.valid) : States<R>{};
    }
  };
  // Results of the tile at t0, which wait in registers and LDS until the next one's loads have come (as in the forward)
  float gb[kOwn], ga[kOwn], ys[kOwn];
  int turn = 0;  // the half of `shares` that is written next
  const auto results = [&](long long t0) {
    const int left = tile_left(end, t0);
    const bool all = all_valid && left == kScanTile;
    const long long at = plane + t0 * p.channels;
    if (p.dx) store_tokens<T, Q>(static_cast<T*>(p.dx) + at, p.channels, s, left, all, gb);
    if (p.ddt) store_tokens<T, Q>(static_cast<T*>(p.ddt) + at, p.channels, s, left, all, ga);
    if (p.dz) store_tokens<T, Q>(static_cast<T*>(p.dz) + at, p.channels, s, left, all, ys);
    if (!p.shared_parts) return;
    lds_barrier();
    constexpr int kRow = 2 * Q * R;
    float* const to = p.shared_parts + (((s.tile / kWaves * p.batch + s.row) * p.tokens + t0) * p.groups + s.group) * kRow;
    for (int i = threadIdx.x; i < left * kRow; i += 64 * kWaves) {
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) sum += shares[turn ^ 1][w][i];
      to[(long long)(i / kRow) * p.groups * kRow + i % kRow] = sum;
    }
  };
  // Sums over the channels of two tokens' shares of db (the first R) and dc: these part at the first level, their states at the next ones.
  // (Lanes with the same sum write the same bits.)
  const auto fold_channels = [&](const float(&v)[2][2 * R], int t) TFA_INLINE {
    float* const to = shares[turn][s.wave] + (2 * t + s.c / (kChannels / 2)) * Q * R + R * s.q;
    constexpr int kNext = 2 * Q * R;  // from a token to the next
    if constexpr (R == 4 && kChannels == 16) {
      const int at = s.c / 4 % 2 * 2 + s.c / 2 % 2;
      float sum0, sum1;
      fold_row(v[0], v[1], 0xCCCCCCCCCCCCCCCCull, sum0, sum1);
      to[at] = sum0;
      to[kNext + at] = sum1;
    } else {
      constexpr int kTop = kChannels / 2 == 4 ? 7 : kChannels / 2, kMid = kChannels / 4 == 4 ? 7 : kChannels / 4;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float w[R];
#pragma unroll
        for (int r = 0; r < R; ++r) w[r] = fold<kTop>(v[i][r], v[i][R + r]);
        float* const half = to + i * kNext;
        if constexpr (R == 1) {
          half[0] = fold<1>(fold<2>(fold<kMid>(w[0])));
        } else if constexpr (R == 2) {
          half[s.c / (kChannels / 4) % 2] = fold<1>(fold<2>(fold<kMid>(w[0], w[1])));
        } else {
          const int first = s.c / (kChannels / 4) % 2 * 2;
          const float x0 = fold<kMid>(w[0], w[2]), x1 = fold<kMid>(w[1], w[3]);
          if constexpr (kChannels == 4) {
            half[first] = x0;
            half[first + 1] = x1;
          } else {
            half[first + s.c % 2] = fold<1>(x0, x1);
          }
        }
      }
    }
  };
  const long long last = end > seg_begin ? seg_begin + (end - 1 - seg_begin) / kScanTile * kScanTile : seg_begin - kScanTile;
  if (last >= seg_begin) fetch(last);
  for (long long t0 = last; t0 >= seg_begin; t0 -= kScanTile) {
    const int left = tile_left(end, t0);
    const bool full = all_valid && left == kScanTile;
    float xs[kOwn], own[kOwn], slope[kOwn], vs[kOwn], zs[kOwn];
    steps_of<T, Q>(dt, bias, p.softplus, own, slope);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) vs[i] = to_f32(dy.v[i]), zs[i] = 0.0f;
    if (pz) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const float zi = to_f32(z.v[i]), gate = sigmoid(zi);
        zs[i] = vs[i] * gate * __builtin_fmaf(zi, 1.0f - gate, 1.0f);
        vs[i] *= zi * gate;
      }
    }
#pragma unroll
    for (int i = 0; i < kOwn; ++i) xs[i] = SUM ? 0.0f : to_f32(x.v[i]);
    if (!full) clear_dead<Q>(s, left, own), clear_dead<Q>(s, left, vs), clear_dead<Q>(s, left, xs), clear_dead<Q>(s, left, slope);
    wave_order();
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      put_token<Q>(ls, s.q, s.c, i, own[i]);
      put_token<Q>(lv, s.q, s.c, i, vs[i]);
      if (SUM) {
        steps += own[i];
      } else {
        put_token<Q>(lu, s.q, s.c, i, own[i] * xs[i]);
        put_token<Q>(lx, s.q, s.c, i, xs[i]);
        put_token<Q>(lslope, s.q, s.c, i, slope[i]);
        put_token<Q>(lz, s.q, s.c, i, zs[i]);
      }
    }
    ScanBank<Q, R> bs, cs;
    cs.put(c, lc, p.n, 0, s.lane, left);
    if (!SUM) bs.put(b, lb, p.n, 0, s.lane, left);
    wave_order();
    const States<R> start = s.valid ? h0 : States<R>{};
    if (!SUM && t0 < last) results(t0 + kScanTile);
    if (t0 > seg_begin) fetch(t0 - kScanTile);
    if constexpr (SUM) {
      Four32 st, vt;
      for_each<kScanTile>([&](auto index) TFA_INLINE {
        constexpr int t = kScanTile - 1 - index;
        if constexpr (t % 4 == 3) st = four_tokens(ls, s.c, t / 4), vt = four_tokens(lv, s.c, t / 4);
        cs.template add<t>(lc, s.q, vt.v[t % 4], carry.v);
#pragma unroll
        for (int r = 0; r < R; ++r) carry.v[r] *= decay_of(st.v[t % 4], a.v[r]);
      });
    } else {
      States<R> hs[kScanTile], es[kScanTile], h = start, da_tile = {};
      // (the next four tokens' values are read while these are worked on)
      Four32 st = four_tokens(ls, s.c, 0), u = four_tokens(lu, s.c, 0), vt = {}, st_next = {}, u_next = {}, vt_next = {};
      for_each<kScanTile / 2>([&](auto index) TFA_INLINE {
        constexpr int t = 2 * index, k = t / 4, j = t % 4;
        if constexpr (j == 0 && k + 1 < kScanTile / 4) st_next = four_tokens(ls, s.c, k + 1), u_next = four_tokens(lu, s.c, k + 1);
        if constexpr (j == 0 && k + 1 == kScanTile / 4) vt = four_tokens(lv, s.c, k);
        float in0[R], in1[R];
        bs.template products<t>(lb, s.q, u.v[j], u.v[j + 1], in0, in1);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          es[t].v[r] = decay_of(st.v[j], a.v[r]);
          es[t + 1].v[r] = decay_of(st.v[j + 1], a.v[r]);
          hs[t].v[r] = __builtin_fmaf(es[t].v[r], h.v[r], in0[r]);
          hs[t + 1].v[r] = __builtin_fmaf(es[t + 1].v[r], hs[t].v[r], in1[r]);
        }
        h = hs[t + 1];
        if constexpr (j == 2) {
          if constexpr (k + 1 < kScanTile / 4) st = st_next, u = u_next;
          __builtin_amdgcn_sched_barrier(0);
        }
      });
      // sums over the states for a token: of Q tokens at least before they are folded
      float sum_b[Q], sum_a[Q], sum_y[Q];
      float v[2][2 * R];  // what two tokens' gradients by b and c sum up over the channels
      for_each<kScanTile>([&](auto index) TFA_INLINE {
        constexpr int t = kScanTile - 1 - index, k = t / 4, j = t % 4, at = t % Q;
        if constexpr (j == 3 && k > 0)
          st_next = four_tokens(ls, s.c, k - 1), u_next = four_tokens(lu, s.c, k - 1), vt_next = four_tokens(lv, s.c, k - 1);
        const States<R>& before = t ? hs[t ? t - 1 : 0] : start;
        float(&own)[2 * R] = v[t % 2];
        reverse_token<t>(bs, lb, cs, lc, s.q, vt.v[j], hs[t], carry, sum_b[at], sum_y[at]);  // (carry is now g)
        sum_a[at] = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          own[r] = carry.v[r] * u.v[j];
          own[R + r] = vt.v[j] * hs[t].v[r];
          carry.v[r] *= es[t].v[r];
          const float flow = carry.v[r] * before.v[r];
          sum_a[at] = __builtin_fmaf(flow, a.v[r], sum_a[at]);
          da_tile.v[r] = __builtin_fmaf(flow, st.v[j], da_tile.v[r]);
        }
        if constexpr (t % 2 == 0) fold_channels(v, t);
        if constexpr (at == 0) {
          settle(sum_b), settle(sum_y);
          gb[t / Q] = fold_states<Q>(sum_b), ga[t / Q] = fold_states<Q>(sum_a), ys[t / Q] = fold_states<Q>(sum_y);
        }
        if constexpr (j == 0) {
          st = st_next, u = u_next, vt = vt_next;
          __builtin_amdgcn_sched_barrier(0);
        }
      });
      float dskip_tile = 0.0f, dbias_tile = 0.0f;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int at = s.c * kPlaneRow + s.q + Q * i;
        const float xi = lx[at], vi = lv[at];
        ys[i] = lz[at] * __builtin_fmaf(skip, xi, ys[i]);
        // (a slope of 0, past the end and where steps are masked: no gradient, also where a rate of no memory has made an infinity of the sum)
        const float slope_i = lslope[at], of_step = __builtin_fmaf(xi, gb[i], ga[i] * (1.0f / kLog2E)) * slope_i;
        ga[i] = slope_i == 0.0f ? 0.0f : of_step;
        gb[i] = __builtin_fmaf(ls[at], gb[i], skip * vi);
        dskip_tile = __builtin_fmaf(vi, xi, dskip_tile);
        dbias_tile += ga[i];
      }
      // (a tile's terms by themselves first: long sums keep their last bits)
      dskip += dskip_tile;
      dbias += dbias_tile;
#pragma unroll
      for (int r = 0; r < R; ++r) da.v[r] += da_tile.v[r];
      turn ^= 1;
    }
  }
  if (!SUM && last >= seg_begin) results(seg_begin);
  if (SUM) {
    reinterpret_cast<States<R>*>(p.seg_state)[(s.seg * s.units + s.unit) * 64 + s.lane] = carry;
    p.seg_steps[(s.seg * s.units + s.unit) * 64 + s.lane] = sum_states<Q>(steps);
    return;
  }
  if (s.idle) return;
  for (void* const out : {p.dx, p.ddt, p.dz})
    if (out) zero_tokens<T, Q>(static_cast<T*>(out) + plane, p.channels, s, max(end, seg_begin), seg_end);
  if (p.dstate_in && s.seg == 0)
    store_states<R>(p.dstate_in + (s.row * p.channels + channel) * p.n, p.n, s.q, s.valid, carry);
  if (p.channel_parts) {
    // (seg, unit, lane): those of da, then dd and ddt_bias
    const long long at = (s.seg * s.units + s.unit) * 64 + s.lane, all = p.segments * s.units * 64;
    reinterpret_cast<States<R>*>(p.channel_parts)[at] = da;
    p.channel_parts[R * all + at] = sum_states<Q>(dskip);
    p.channel_parts[(R + 1) * all + at] = sum_states<Q>(dbias);
  }
}

enum ScanMode { kScanSums, kScanForward, kScanBackSums, kScanBackward };

// Lanes of a channel, and the states that each has
struct ScanShape {
  int lanes, each;
};
inline ScanShape scan_shape(int n) {
  return n <= 4 ? ScanShape{4, 1} : n <= 8 ? ScanShape{4, 2} : n <= 16 ? ScanShape{4, 4} : n <= 32 ? ScanShape{8, 4} : ScanShape{16, 4};
}

hipError_t scan_f32(const ScanArgs& p, ScanMode mode);
hipError_t scan_bf16(const ScanArgs& p, ScanMode mode);
hipError_t scan_f16(const ScanArgs& p, ScanMode mode);

}  // namespace tfa
