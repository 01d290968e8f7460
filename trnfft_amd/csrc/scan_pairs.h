// The selective scan over whole sequences for 9 to 16 states where one wave for 16 channels would leave a SIMD a single wave or two: two waves
// take the same 16 channels, each 8 of the states.
//
// A wave alone on its SIMD has nothing to issue behind its own instructions' latencies: a token of 16 channels takes it 250 clocks, two waves on one
// SIMD 330 for a token each.  Segments would make more waves, for a pass of sums over all of them but one.  Here what belongs to a channel and token
// alone (softplus, gates, loads, stores) is shared out as well: of a tile's 16 tokens wave `half` takes the 8 from 8 half on.  The pair meets at one
// barrier a tile: behind it both find the tile's s and s x in LDS, and what the other wave's states have added to the tile before.  Buffers
// alternate from tile to tile, so nothing is written that is still read.
//
// Bound by issue: some 380 instructions a tile and wave, 3500 clocks for two waves' (8 x 4096 tokens of 2048 channels, bf16: 400 us, and 418 to 426 with
// states kept).  Loads two tiles ahead made it no faster.
//
// States that are kept or handed on lie as the kernels of four states a lane (scan_blocks.h) lay them out.
#pragma once
#include "scan_blocks.h"

namespace tfa {

constexpr int kPairWaves = 4;  // of a workgroup: two pairs
constexpr int kPairOwn = 2;    // tokens of a lane

// Tokens 8 half + q and 4 later of a tile of one operand, as ScanTokens.
template <typename T>
struct PairTokens {
  // a register each, as they come from memory: two of 16 bits in one register would be waited for where they are put together
  typedef std::conditional_t<sizeof(T) == 4, unsigned, unsigned short> Word;
  Word w[kPairOwn];
  __device__ __forceinline__ float value(int i) const {
    Word v = w[i];
    asm volatile("" : "+v"(v));  // (else the compiler converts where it loads, and waits there)
    if constexpr (sizeof(T) == 4)
      return __uint_as_float(v);
    else
      return to_f32(__builtin_bit_cast(T, v));
  }
  __device__ __forceinline__ void load(const T* p, unsigned (&at)[kPairOwn]) {
#pragma unroll
    for (int i = 0; i < kPairOwn; ++i) {
      asm volatile("" : "+v"(at[i]));  // (as in lane_address)
      w[i] = *reinterpret_cast<const Word*>(reinterpret_cast<const char*>(p) + at[i]);
    }
  }
};
// Where a lane's tokens are in a tile of `left` tokens to the end, in bytes from its first; those past the end are the last one's again.  Kept from
// tile to tile: loads are the same instructions whether the tile is whole or not.
template <typename T>
__device__ __forceinline__ void pair_offsets(unsigned (&at)[kPairOwn], long long st, const ScanPlace<4>& s, int half, int left) {
#pragma unroll
  for (int i = 0; i < kPairOwn; ++i) at[i] = (__umul24(min(8 * half + s.q + 4 * i, left - 1), st) + s.own) * (unsigned)sizeof(T);
}
template <typename T>
__device__ __forceinline__ void store_pair_tokens(T* p, int st, const ScanPlace<4>& s, int half, int left, bool all, const float (&v)[kPairOwn]) {
  const unsigned at = (s.q * (unsigned)st + s.own) * sizeof(T);
#pragma unroll
  for (int i = 0; i < kPairOwn; ++i)
    if (all || (s.valid && 8 * half + s.q + 4 * i < left)) *lane_address(p + (long long)(8 * half + 4 * i) * st, at) = from_f32<T>(v[i]);
}
__device__ __forceinline__ void clear_dead(const ScanPlace<4>& s, int half, int left, float (&v)[kPairOwn]) {
#pragma unroll
  for (int i = 0; i < kPairOwn; ++i) v[i] = s.valid && 8 * half + s.q + 4 * i < left ? v[i] : 0.0f;
}
__device__ __forceinline__ void steps_of(float bias, bool soft, float (&step)[kPairOwn], float (&slope)[kPairOwn]) {
#pragma unroll
  for (int i = 0; i < kPairOwn; ++i) step[i] += bias, slope[i] = 1.0f;
  if (soft) {
#pragma unroll
    for (int i = 0; i < kPairOwn; ++i) step[i] = softplus(step[i], slope[i]);
  }
}
__device__ __forceinline__ void put_pair_token(float* lds, const ScanPlace<4>& s, int half, int i, float v) {
  lds[s.c * kPlaneRow + 8 * half + s.q + 4 * i] = v;
}
template <typename T>
__device__ __forceinline__ void zero_pair_tokens(T* p, int st, const ScanPlace<4>& s, int half, long long from, long long to) {
  if (s.valid)
    for (long long t = from + 4 * half + s.q; t < to; t += 8) p[t * st + s.own] = T(0);
}
// A tile's sums over this wave's states, by the lanes of their tokens: the wave's own tokens' stay, the others' are given to the other wave.
__device__ __forceinline__ void share_out(const float (&sum)[4], int half, float (&own)[kPairOwn], float (*given)[64], int lane) {
#pragma unroll
  for (int i = 0; i < kPairOwn; ++i) {
    own[i] = half ? sum[2 + i] : sum[i];
    given[i][lane] = half ? sum[i] : sum[2 + i];
  }
}
// bytes into a unit's 64 lanes of four states where this lane's two are
__device__ __forceinline__ unsigned pair_states(const ScanPlace<4>& s, int half) { return ((2 * half + s.q / 2) * 16 + s.c) * 16 + s.q % 2 * 8; }

template <typename T>
__global__ __launch_bounds__(64 * kPairWaves) void scan_pair_kernel(ScanArgs p, long long first_block) {
  __shared__ float planes[kPairWaves / 2][2][2][kPlaneWords<4>];
  __shared__ float given[kPairWaves][2][kPairOwn][64];
  const ScanPlace<4> s = scan_place<4, kPairWaves, 2>(p, first_block + blockIdx.x);
  const int half = s.wave % 2, n = half ? p.n - 8 : 8;
  const long long end = scan_end(p, s.row);
  const T* px = static_cast<const T*>(p.x) + s.row * p.x_sb + s.base;
  const T* pdt = static_cast<const T*>(p.dt) + s.row * p.dt_sb + s.base;
  const T* pz = p.z ? static_cast<const T*>(p.z) + s.row * p.z_sb + s.base : nullptr;
  const T* pb = static_cast<const T*>(p.b) + s.row * p.b_sb + s.group * p.b_sg;
  const T* pc = static_cast<const T*>(p.c) + s.row * p.c_sb + s.group * p.c_sg;
  T* const y = static_cast<T*>(p.y) + s.row * p.tokens * p.channels + s.base;
  const int channel = s.base + s.own;
  const long long states = (s.row * p.channels + channel) * p.n + 8 * half;

  States<2> a = load_states<2>(p.a + (long long)channel * p.n + 8 * half, n, s.q, s.valid), h = {};
#pragma unroll
  for (int r = 0; r < 2; ++r) a.v[r] = rate_of(a.v[r]);
  const float bias = p.dt_bias ? p.dt_bias[channel] : 0.0f, skip = p.d ? p.d[channel] : 0.0f;
  if (p.state_in) h = load_states<2>(p.state_in + states, n, s.q, s.valid);
  char* const kept = p.kept && !s.idle ? reinterpret_cast<char*>(p.kept) + s.unit * kept_states(p) * 1024 : nullptr;
  const unsigned kept_lane = pair_states(s, half);
  const bool all_valid = __all(s.valid);
  struct Operands {
    PairTokens<T> x, dt, z;
    ScanRows<T, 4, 2> b, c;
  } o;
  unsigned x_at[kPairOwn], dt_at[kPairOwn], z_at[kPairOwn];
  const auto place = [&](int left) TFA_INLINE {
    pair_offsets<T>(x_at, p.x_st, s, half, left), pair_offsets<T>(dt_at, p.dt_st, s, half, left), pair_offsets<T>(z_at, p.z_st, s, half, left);
  };
  place(kScanTile);
  const auto fetch = [&](int left) TFA_INLINE {
    if (left < kScanTile) place(left);
    o.x.load(px, x_at);
    o.dt.load(pdt, dt_at);
    o.b.load(pb, p.b_st, p.n, 8 * half, s.lane, left);
    o.c.load(pc, p.c_st, p.n, 8 * half, s.lane, left);
    if (pz) o.z.load(pz, z_at), pz += kScanTile * p.z_st;
    px += kScanTile * p.x_st, pdt += kScanTile * p.dt_st, pb += kScanTile * p.b_st, pc += kScanTile * p.c_st;
  };
  if (end > 0) fetch(tile_left(end, 0));
  float sums[kPairOwn], x_of[kPairOwn], gates[kPairOwn];  // of the tile before
  // y of the tile at t0, behind the barrier that follows it
  const auto results = [&](int turn, long long t0) TFA_INLINE {
    const int left = tile_left(end, t0);
    float ys[kPairOwn];
#pragma unroll
    for (int i = 0; i < kPairOwn; ++i) ys[i] = __builtin_fmaf(skip, x_of[i], sums[i] + given[s.wave ^ 1][turn][i][s.lane]) * gates[i];
    store_pair_tokens<T>(y + t0 * p.channels, p.channels, s, half, left, all_valid && left == kScanTile, ys);
  };
  int turn = 0;
  for (long long t0 = 0; t0 < end; t0 += kScanTile) {
    const int left = tile_left(end, t0);
    const bool full = all_valid && left == kScanTile;
    float *const ls = planes[s.wave / 2][turn][0], *const lu = planes[s.wave / 2][turn][1];
    float xs[kPairOwn], zs[kPairOwn], own[kPairOwn], slope[kPairOwn];
#pragma unroll
    for (int i = 0; i < kPairOwn; ++i) own[i] = o.dt.value(i), xs[i] = o.x.value(i), zs[i] = 1.0f;
    steps_of(bias, p.softplus, own, slope);
    if (!full) clear_dead(s, half, left, own), clear_dead(s, half, left, xs);
#pragma unroll
    for (int i = 0; i < kPairOwn; ++i) {
      put_pair_token(ls, s, half, i, own[i]);
      put_pair_token(lu, s, half, i, own[i] * xs[i]);
    }
    ScanBank<4, 2> bs, cs;
    bs.put(o.b, nullptr, p.n, 8 * half, s.lane, left);
    cs.put(o.c, nullptr, p.n, 8 * half, s.lane, left);
    if (pz) {
#pragma unroll
      for (int i = 0; i < kPairOwn; ++i) zs[i] = activate(o.z.value(i), kActSilu);
    }
    lds_barrier();
    if (kept && t0 > 0) *reinterpret_cast<States<2>*>(lane_address(kept + (t0 / kScanStretch - 1) * 1024, kept_lane)) = h;
    if (t0 > 0) results(turn ^ 1, t0 - kScanTile);
    if (t0 + kScanTile < end) fetch(tile_left(end, t0 + kScanTile));
#pragma unroll
    for (int i = 0; i < kPairOwn; ++i) x_of[i] = xs[i], gates[i] = zs[i];
    float part[kScanTile];
    Four32 st, u;
    for_each<kScanTile / 2>([&](auto index) TFA_INLINE {
      constexpr int t = 2 * index, j = t % 4;
      if constexpr (j == 0) st = four_tokens(ls, s.c, t / 4), u = four_tokens(lu, s.c, t / 4);
      float in0[2], in1[2];
      RowLane<t>::products(bs.own.v, u.v[j], u.v[j + 1], in0, in1);
      States<2> h0 = h;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        h0.v[r] = __builtin_fmaf(decay_of(st.v[j], a.v[r]), h.v[r], in0[r]);
        h.v[r] = __builtin_fmaf(decay_of(st.v[j + 1], a.v[r]), h0.v[r], in1[r]);
      }
      RowLane<t>::dots(cs.own.v, h0.v, h.v, part[t], part[t + 1]);
    });
    float folded[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float four[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) four[j] = part[4 * i + j];
      settle(four);
      folded[i] = fold_states<4>(four);
    }
    share_out(folded, half, sums, given[s.wave][turn], s.lane);
    turn ^= 1;
  }
  if (end > 0) {
    lds_barrier();
    results(turn ^ 1, (end - 1) / kScanTile * kScanTile);
  }
  zero_pair_tokens<T>(y, p.channels, s, half, end, p.tokens);
  if (p.state_out) store_states<2>(p.state_out + states, n, s.q, s.valid, h);
}

// Sequences that are walked whole, of up to 10 waves (of 16 channels) a compute unit; beyond that one wave finds enough beside it.  16 states, forward
// without and with two waves, us: 8 x 4096 tokens of 2048 channels (1024 waves) 443 and 400, fp32 550 and 463; 12 x 2048 of 2048 (1536) 309 and 260;
// 64 x 626 of 512 with rows of all lengths (2048) 83 and 65; 20 x 2048 of 2048 (2560) 421 and 392, 24 rows 422 and 442, 32 rows 536 and 571.
// Backwards the same was built, and won between 950 and 1024 waves alone (923 + 176 in two segments, 1050 in pairs): it is not here.
constexpr long long kPairMost = 2560;

template <typename F>
hipError_t scan_grid(const ScanArgs& p, int channels, int tiles_each, int waves, int segments, F launch) {
  const long long tiles = (p.channels / p.groups + channels - 1) / channels;
  const long long blocks = (tiles + tiles_each - 1) / tiles_each * p.groups * p.batch * segments;
  for (long long first = 0; first < blocks; first += max_blocks(64 * waves)) {
    launch(dim3((unsigned)std::min(blocks - first, max_blocks(64 * waves))), dim3(64 * waves), first);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, int Q, int R>
hipError_t scan_launch(const ScanArgs& p, ScanMode mode) {
  if constexpr (Q == 4 && R == 4) {
    if (mode == kScanForward && p.segments == 1 && scan_waves(p) <= kPairMost)
      return scan_grid(p, 16, kPairWaves / 2, kPairWaves, 1, [&](dim3 grid, dim3 block, long long first) {
        hipLaunchKernelGGL((scan_pair_kernel<T>), grid, block, 0, p.stream, p, first);
      });
  }
  const int waves = mode == kScanBackSums || mode == kScanBackward ? kBackWaves<Q> : kScanWaves;
  // (the last segment's sums are not needed, nor are the first's backwards)
  const int segments = mode == kScanSums || mode == kScanBackSums ? (p.segments - 1) * p.fine : p.segments;
  return scan_grid(p, 64 / Q, waves, waves, segments, [&](dim3 grid, dim3 block, long long first) {
    if (mode == kScanSums) hipLaunchKernelGGL((scan_forward_kernel<T, Q, R, false>), grid, block, 0, p.stream, p, first);
    if (mode == kScanForward) hipLaunchKernelGGL((scan_forward_kernel<T, Q, R, true>), grid, block, 0, p.stream, p, first);
    if (mode == kScanBackSums) hipLaunchKernelGGL((scan_backward_kernel<T, Q, R, true>), grid, block, 0, p.stream, p, first);
    if (mode == kScanBackward) hipLaunchKernelGGL((scan_backward_kernel<T, Q, R, false>), grid, block, 0, p.stream, p, first);
  });
}

template <typename T>
hipError_t scan_typed(const ScanArgs& p, ScanMode mode) {
  const ScanShape s = scan_shape(p.n);
  if (s.lanes == 4 && s.each == 1) return scan_launch<T, 4, 1>(p, mode);
  if (s.lanes == 4 && s.each == 2) return scan_launch<T, 4, 2>(p, mode);
  if (s.lanes == 4) return scan_launch<T, 4, 4>(p, mode);
  return s.lanes == 8 ? scan_launch<T, 8, 4>(p, mode) : scan_launch<T, 16, 4>(p, mode);
}

}  // namespace tfa
