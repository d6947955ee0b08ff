// A diagonal state space whose step, input and output maps depend on the token,
// and its gradient.  Per channel c (of group g) and state n:
//
//   d = softplus(dt + dt_bias),  a = exp(d A[c][n])
//   h'= a h + d u B[n],  y = sum_n C[n] h' + D u,  out = y z sigmoid(z)
//   G = C dy + X',  X = a G:  the gradient of h' and what it hands to the token before
//   dC[n] = sum_c dy h', dB[n] = sum_c G d u, dA = sum d X h, du = d sum_n G B + D dy, dd = sum_n A X h + u sum_n G B
//
// The tokens are cut into tiles of 32, tiles into chunks, and the chunks are
// walked side by side: a first pass leaves each chunk's state from zero and the
// sum of its steps d (its decay is exp(A sum d)), a second carries states from
// chunk to chunk, a third walks the chunks again from where they really start.
// Where channels alone fill the card there is one chunk and only the third.
// Backward, X goes through the first two passes from the end, a tile a chunk; a
// tile then has its entering h (kept by the forward pass) and X and is worked
// out on its own.  States, sums and statistics are fp32; tokens from a
// sequence's length on take no step (d = 0), are never read and give zeros.
#include <type_traits>
#include <utility>

#include "bmx_common.h"

using namespace bmx;

namespace {

constexpr int K = 32;             // tokens of a tile
constexpr int kRow = K + 4;       // LDS row of a state's map over a tile: 16-byte reads along the tokens, no conflicts
constexpr int kChannelRow = K + 2;  // LDS row of a channel: reads without conflicts, transposing writes two on a bank
constexpr int kWalk = 64;         // channels of a block that walks chunks, four lanes each
constexpr int kSlice = 32;        // channels that the gradient stages at a time
constexpr int kMaxSpan = 6144;    // channels x states of a gradient block (its dA in LDS)
constexpr float kLog2e = 1.4426950408889634f;

struct Operand {
  const void* p;
  int64_t sb, st, sg;  // strides of a batch element, a token and a group, in elements
};
struct Scan {
  Operand u, dt, z, B, C;
  const float *A, *D, *dt_bias, *state;
  const void *lengths, *dout;
  void* out;
  float *state_out, *raw;   // raw: y before its gate, for the gradient
  float *carry, *steps;     // [batch][chunks][channels][states] and [batch][chunks][channels]
  float* saved;             // [batch][tiles][channels][states]: h at every tile's start
  const float *h_in, *x_in;
  void *du, *ddt, *dz;
  float *dB, *dC;           // [spans][batch][tokens][groups][states], or the results where there is one span
  void *dB_out, *dC_out;
  float *dA, *dD, *dbias;   // partial sums, [batch * ranges][channels]([states])
  int64_t batch, tokens, tiles, chunks, chunk_tiles, blocks;
  int channels, groups, group_channels, states, cblocks, lengths64, softplus;
  int span, spans, ranges, range_tiles, whole;
};

// ------------------------------------------------------------------ elements

__device__ __forceinline__ int64_t length_of(const Scan& s, int64_t b) {
  if (!s.lengths) return s.tokens;
  const int64_t n = s.lengths64 ? ((const int64_t*)s.lengths)[b] : (int64_t)((const int32_t*)s.lengths)[b];
  return n < 0 ? 0 : n < s.tokens ? n : s.tokens;
}

// softplus(x) = max(x, 0) + log1p(e), e = exp(-|x|), with log(1 + e) = 2 atanh(r), r = e / (2 + e) <= 1 / 3, by the
// series of atanh to r^13: what is left is below 2^-25 of it, however small e is.
__device__ __forceinline__ float step_of(float x) {
  const float e = __builtin_amdgcn_exp2f(-fabsf(x) * kLog2e);
  const float r = e * __builtin_amdgcn_rcpf(2.f + e), q = r * r;
  float s = 2.f / 13.f;
  s = s * q + 2.f / 11.f;
  s = s * q + 2.f / 9.f;
  s = s * q + 2.f / 7.f;
  s = s * q + 2.f / 5.f;
  s = s * q + 2.f / 3.f;
  s = s * q + 2.f;
  return s * r + fmaxf(x, 0.f);
}

// v of the lane that a DPP control word names, as an operand of the instruction that uses it.
template <int kCtrl>
__device__ __forceinline__ float from_lane(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), kCtrl, 0xF, 0xF, true));
}
template <int kLane>
__device__ __forceinline__ float from_quad(float v) {  // lane kLane of each quad
  return from_lane<0x55 * kLane>(v);
}
template <int kLane>
__device__ __forceinline__ float from_row(float v) {  // lane kLane of each 16
  return from_lane<0x150 + kLane>(v);
}
template <typename F, int... I>
__device__ __forceinline__ void unrolled(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int kCount, typename F>
__device__ __forceinline__ void unrolled(F f) {
  unrolled(f, std::make_integer_sequence<int, kCount>());
}

__device__ __forceinline__ float xor16(float v) {
  return __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(v), 0x401F));
}
__device__ __forceinline__ float xor32_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Sums of four values over a quad; lane j gets the one of value j.
__device__ __forceinline__ float quad_sums(const f32x4& p, int lane) {
  const bool odd = lane & 1, high = lane & 2;
  const float a = (odd ? p[1] : p[0]) + from_lane<0xB1>(odd ? p[0] : p[1]);
  const float b = (odd ? p[3] : p[2]) + from_lane<0xB1>(odd ? p[2] : p[3]);
  return (high ? b : a) + from_lane<0x4E>(high ? a : b);
}

// Sums of 16 values over the 16 lanes of a row, one value after another; lane j gets the one of value rev4(j), j's four
// bits reversed.  Level by level two values become one, a lane keeping the first or the second by one of its bits; the
// exchange partner (15 - j, 7 - j, j xor 2, j xor 1) has the other value of that bit, and the earlier ones' equal.
__device__ __forceinline__ int rev4(int j) { return (j & 1) << 3 | (j & 2) << 1 | (j & 4) >> 1 | (j & 8) >> 3; }
struct RowSum {
  float held[4];
  template <int kIndex>
  __device__ __forceinline__ void add(float v, int lane) {  // values in the order 0 .. 15; the last leaves its sum in held[3]
    level<kIndex, 0>(v, lane);
  }
  template <int kIndex, int kLevel>
  __device__ __forceinline__ void level(float v, int lane) {
    if constexpr (kLevel < 4) {
      if constexpr ((kIndex >> kLevel) & 1) {
        constexpr int ctrl[4] = {0x140, 0x141, 0x4E, 0xB1};
        const bool second = lane & (8 >> kLevel);
        const float sum = (second ? v : held[kLevel]) + from_lane<ctrl[kLevel]>(second ? held[kLevel] : v);
        level<kIndex, kLevel + 1>(sum, lane);
      } else {
        held[kLevel] = v;
      }
    } else {
      held[3] = v;
    }
  }
};

// Four channels of one token as fp32; zeros where they are not there.
template <typename T>
__device__ __forceinline__ f32x4 row4(const Operand& o, int64_t b, int64_t t, int c, bool there) {
  return there ? load4((const T*)o.p + b * o.sb + t * o.st + c) : f32x4{0.f, 0.f, 0.f, 0.f};
}

// ------------------------------------------------------------ walking chunks

// kLocal: from zero states to each chunk's own, forward; kOut: the outputs; kBack: the same as kLocal for X, from the
// chunk's end, of dy in the place of d u and of C in the place of B.
enum Mode { kLocal, kOut, kBack };

template <typename T, int N, int kMode>
__global__ __launch_bounds__(256) void scan_walk_kernel(Scan s) {
  constexpr int S = N / 4, kPer = kWalk * K / 4 / 256, kMaps = (N * K / 4 + 255) / 256;
  __shared__ float sd[kWalk * kChannelRow], sv[kWalk * kChannelRow], sy[kMode == kOut ? kWalk * kChannelRow : 4];
  __shared__ __align__(16) float sB[N * kRow], sC[kMode == kOut ? N * kRow : 4];
  uint32_t block = block_index();
  if (block >= s.blocks) return;
  const int cblock = (int)(block % (uint32_t)s.cblocks);
  block /= (uint32_t)s.cblocks;
  const int group = (int)(block % (uint32_t)s.groups);
  block /= (uint32_t)s.groups;
  const int64_t chunk = block % (uint32_t)s.chunks, b = block / (uint32_t)s.chunks;
  const int c_first = group * s.group_channels + cblock * kWalk;
  const int c_end = min(c_first + kWalk, (group + 1) * s.group_channels);
  const int64_t length = length_of(s, b);
  const int lane = lane_id(), j = threadIdx.x & 3, c_local = threadIdx.x >> 2, c = c_first + c_local;
  const bool live = c < c_end;

  const int64_t tile0 = chunk * s.chunk_tiles, tile1 = min(tile0 + s.chunk_tiles, s.tiles);
  const int64_t start = kMode == kBack ? tile1 - 1 : tile0;
  // this thread's elements of a tile: four channels of kPer tokens, and of the maps four states of kMaps tokens
  const int e = threadIdx.x % (kWalk / 4) * 4, et = threadIdx.x / (kWalk / 4), cc = c_first + e;
  const int en = threadIdx.x % (N / 4) * 4, ent = threadIdx.x / (N / 4);
  const bool mine = cc < c_end;
  const int64_t dense = (b * s.tokens + start * K + et) * s.channels + cc;
  const T *dt = (const T*)s.dt.p + b * s.dt.sb + (start * K + et) * s.dt.st + cc, *u = (const T*)s.u.p, *z = (const T*)s.z.p;
  u = kMode == kBack ? (const T*)s.dout + dense : u + b * s.u.sb + (start * K + et) * s.u.st + cc;
  z = z ? z + b * s.z.sb + (start * K + et) * s.z.st + cc : nullptr;
  const int64_t u_st = kMode == kBack ? s.channels : s.u.st;
  const T* B = (const T*)s.B.p + b * s.B.sb + (start * K + ent) * s.B.st + group * s.B.sg + en;
  const T* C = (const T*)s.C.p + b * s.C.sb + (start * K + ent) * s.C.st + group * s.C.sg + en;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 ru[kPer], rdt[kPer], rz[kPer], rB[kMaps], rC[kMaps];
  auto fetch = [&](int64_t tile) {
    const int64_t left = length - tile * K;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int t = i * (K / kPer);
      const bool there = mine && et + t < left;
      rdt[i] = there ? load4(dt + t * s.dt.st) : zero;
      ru[i] = there ? load4(u + t * u_st) : zero;
      if (kMode != kLocal) rz[i] = there && z ? load4(z + t * s.z.st) : zero;
    }
#pragma unroll
    for (int i = 0; i < kMaps; ++i) {
      const int t = i * (1024 / N);
      const bool there = ent + t < K && ent + t < left;
      if (kMode != kBack) rB[i] = there ? load4(B + t * s.B.st) : zero;
      if (kMode != kLocal) rC[i] = there ? load4(C + t * s.C.st) : zero;
    }
    const int64_t step = kMode == kBack ? -K : K;
    dt += step * s.dt.st, u += step * u_st, B += step * s.B.st, C += step * s.C.st;
    if (z) z += step * s.z.st;
  };
  fetch(start);

  f32x4 bias = zero, skip = zero;
  if (mine && s.dt_bias) bias = load4(s.dt_bias + cc);
  if (kMode == kOut && mine && s.D) skip = load4(s.D + cc);
  float A2[S], h[S], total = 0.f;
  const float* from = nullptr;
  if (kMode == kOut)
    from = s.chunks > 1 ? s.carry + ((b * s.chunks + chunk) * s.channels + c) * N
           : s.state    ? s.state + (b * s.channels + c) * N
                        : nullptr;
#pragma unroll
  for (int i = 0; i < S; ++i) {
    A2[i] = live ? s.A[(int64_t)c * N + j * S + i] * kLog2e : 0.f;
    h[i] = live && from ? from[j * S + i] : 0.f;
  }

  for (int64_t k = tile0; k < tile1; ++k) {
    const int64_t tile = kMode == kBack ? tile0 + tile1 - 1 - k : k, left = length - tile * K;
    // d, and d u (kBack: dy), of the tile to LDS, along the tokens; a token that is not there takes no step
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int t = et + i * (K / kPer);
      f32x4 d = rdt[i] + bias;
      if (s.softplus) {
#pragma unroll
        for (int q = 0; q < 4; ++q) d[q] = step_of(d[q]);
      }
      d = d * (mine && t < left ? 1.f : 0.f);
      f32x4 v = kMode == kBack ? ru[i] : d * ru[i];
      if (kMode == kBack && s.z.p) {
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] *= silu_f(rz[i][q]);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        sd[(e + q) * kChannelRow + t] = d[q];
        sv[(e + q) * kChannelRow + t] = v[q];
      }
    }
#pragma unroll
    for (int i = 0; i < kMaps; ++i) {
      const int t = ent + i * (1024 / N);
      if (t >= K) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        sB[(en + q) * kRow + t] = kMode == kBack ? rC[i][q] : rB[i][q];
        if (kMode == kOut) sC[(en + q) * kRow + t] = rC[i][q];
      }
    }
    __syncthreads();
    f32x4 keep_u[kPer], keep_z[kPer];
    if (kMode == kOut) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) keep_u[i] = ru[i], keep_z[i] = rz[i];
    }
    if (k + 1 < tile1) fetch(kMode == kBack ? tile - 1 : tile + 1);
    if (kMode == kOut && s.saved && live) {
      float* to = s.saved + ((b * s.tiles + tile) * s.channels + c) * N + j * S;
#pragma unroll
      for (int i = 0; i < S; ++i) to[i] = h[i];
    }

    // Four tokens at a time: lane j of a channel's quad holds token j's d and d u, which the others take from it.
#pragma unroll 2
    for (int step = 0; step < K; step += 4) {
      const int t = kMode == kBack ? K - 4 - step : step;
      const float d = sd[c_local * kChannelRow + t + j], v = sv[c_local * kChannelRow + t + j];
      f32x4 p = zero;
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const f32x4 m = *(const f32x4*)(sB + (j * S + i) * kRow + t);
        f32x4 r = zero;
        if (kMode == kOut) r = *(const f32x4*)(sC + (j * S + i) * kRow + t);
        unrolled<4>([&](auto index) {
          constexpr int q = kMode == kBack ? 3 - decltype(index)::value : decltype(index)::value;
          const float a = __builtin_amdgcn_exp2f(from_quad<q>(d) * A2[i]);
          if (kMode == kBack) {
            h[i] = a * __builtin_fmaf(from_quad<q>(v), m[q], h[i]);
          } else {
            h[i] = __builtin_fmaf(from_quad<q>(v), m[q], a * h[i]);
            if (kMode == kOut) p[q] = __builtin_fmaf(r[q], h[i], p[q]);
          }
        });
      }
      if (kMode != kOut)
        total += d;
      else
        sy[c_local * kChannelRow + t + j] = quad_sums(p, lane);
    }
    __syncthreads();
    if (kMode == kOut) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int t = et + i * (K / kPer);
        const int64_t token = tile * K + t;
        if (!mine || token >= s.tokens) continue;
        const bool there = t < left;
        f32x4 y;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          y[q] = there ? sy[(e + q) * kChannelRow + t] + skip[q] * keep_u[i][q] : 0.f;
        const int64_t to = (b * s.tokens + token) * s.channels + cc;
        if (s.raw) store4(s.raw + to, y);
        if (s.z.p) {
#pragma unroll
          for (int q = 0; q < 4; ++q) y[q] = there ? y[q] * silu_f(keep_z[i][q]) : 0.f;
        }
        store4((T*)s.out + to, y);
      }
    }
  }
  if (kMode == kOut) {
    if (live && s.state_out && chunk == s.chunks - 1) {
#pragma unroll
      for (int i = 0; i < S; ++i) s.state_out[(b * s.channels + c) * N + j * S + i] = h[i];
    }
    return;
  }
  total += from_lane<0xB1>(total);
  total += from_lane<0x4E>(total);
  if (!live) return;
  const int64_t at = (b * s.chunks + chunk) * s.channels + c;
#pragma unroll
  for (int i = 0; i < S; ++i) s.carry[at * N + j * S + i] = h[i];
  if (j == 0) s.steps[at] = total;
}

// The second pass: from each chunk's own states and the sum of its steps to what enters it, in place; forward from the
// given state (or zeros), backward from the gradient of the last one.
template <bool kReverse>
__global__ __launch_bounds__(256) void scan_carry_kernel(Scan s, const float* first, float* last) {
  const int64_t item = (int64_t)block_index() * 256 + threadIdx.x, per = (int64_t)s.channels * s.states;
  if (item >= s.batch * per) return;
  const int64_t b = item / per, cn = item - b * per, c = cn / s.states;
  const float A2 = s.A[cn] * kLog2e;
  float carry = first ? first[item] : 0.f;
  constexpr int kAhead = 8;
  for (int64_t k0 = 0; k0 < s.chunks; k0 += kAhead) {
    float own[kAhead], d[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t k = min(k0 + i, s.chunks - 1), at = b * s.chunks + (kReverse ? s.chunks - 1 - k : k);
      own[i] = s.carry[at * per + cn];
      d[i] = s.steps[at * s.channels + c];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (k0 + i >= s.chunks) break;
      const int64_t at = b * s.chunks + (kReverse ? s.chunks - 1 - (k0 + i) : k0 + i);
      s.carry[at * per + cn] = carry;
      carry = __builtin_amdgcn_exp2f(A2 * d[i]) * carry + own[i];
    }
  }
  if (last) last[item] = carry;
}

// One token: four states a thread.
template <typename T, int N>
__global__ __launch_bounds__(256) void scan_step_kernel(Scan s) {
  constexpr int L = N / 4;
  const int64_t item = (int64_t)block_index() * 256 + threadIdx.x, row = item / L;
  if (row >= s.batch * s.channels) return;  // whole channels leave
  const int64_t b = row / s.channels;
  const int c = (int)(row - b * s.channels), j = (int)(item - row * L), n = 4 * j, group = c / s.group_channels;
  f32x4 h = s.state ? *(const f32x4*)(s.state + row * N + n) : f32x4{0.f, 0.f, 0.f, 0.f};
  const bool there = length_of(s, b) > 0;
  float y = 0.f, u = 0.f;
  if (there) {
    const f32x4 A = *(const f32x4*)(s.A + (int64_t)c * N + n);
    const f32x4 B = load4((const T*)s.B.p + b * s.B.sb + group * s.B.sg + n);
    const f32x4 C = load4((const T*)s.C.p + b * s.C.sb + group * s.C.sg + n);
    u = (float)((const T*)s.u.p)[b * s.u.sb + c];
    float d = (float)((const T*)s.dt.p)[b * s.dt.sb + c] + (s.dt_bias ? s.dt_bias[c] : 0.f);
    if (s.softplus) d = step_of(d);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[i] = __builtin_amdgcn_exp2f(d * (A[i] * kLog2e)) * h[i] + d * u * B[i];
      y += C[i] * h[i];
    }
  }
  if (L >= 2) y += dpp<0xB1>(y);
  if (L >= 4) y += dpp<0x4E>(y);
  if (L >= 8) y += dpp<0x141>(y);
  if (L >= 16) y += dpp<0x140>(y);
  if (s.state_out) *(f32x4*)(s.state_out + row * N + n) = h;
  if (j) return;
  if (there) {
    y += s.D ? s.D[c] * u : 0.f;
    if (s.z.p) y *= silu_f((float)((const T*)s.z.p)[b * s.z.sb + c]);
  }
  ((T*)s.out)[row] = (T)y;
}

// ------------------------------------------------------------------ gradient

// A block takes a span of a group's channels and a range of tiles.  A lane has one state (of 8 states every second lane
// none) and, pass by pass, channel after channel: the sums dB, dC of its state stay in its registers over a tile, h and a
// of a channel over its 32 tokens.  A token's d, d u and dy stay with lane t % 16 of each row of 16, from where the others
// take them.  dA, dD and the bias's sums stay in LDS over the range.
template <typename T, int N>
__global__ __launch_bounds__(256, 2) void scan_bwd_kernel(Scan s) {
  constexpr int NP = N < 16 ? 16 : N, kSlots = 64 / NP, kPasses = kSlice / (4 * kSlots);
  constexpr int kStage = 5 * kSlice * kRow, kJoin = 4 * K * N;
  __shared__ __align__(16) float lds[kStage > kJoin ? kStage : kJoin];
  __shared__ __align__(16) float sB[NP * kRow], sC[NP * kRow];
  extern __shared__ __align__(16) float span_sums[];  // dA [span][N], dD [span], dbias [span]
  float *sd = lds, *sv = sd + kSlice * kRow, *sy = sv + kSlice * kRow, *s1 = sy + kSlice * kRow, *s2 = s1 + kSlice * kRow;
  float *aA = span_sums, *aD = aA + s.span * N, *ab = aD + s.span;
  uint32_t block = block_index();
  if (block >= s.blocks) return;
  const int span = (int)(block % (uint32_t)s.spans);
  block /= (uint32_t)s.spans;
  const int group = (int)(block % (uint32_t)s.groups);
  block /= (uint32_t)s.groups;
  const int range = (int)(block % (uint32_t)s.ranges);
  const int64_t b = block / (uint32_t)s.ranges, length = length_of(s, b);
  const int c_first = group * s.group_channels + span * s.span;
  const int c_end = min(c_first + s.span, (group + 1) * s.group_channels);
  const int lane = lane_id(), wave = threadIdx.x >> 6, n = lane % NP, slot = lane / NP, r = lane & 15;
  const bool held = n < N;
  for (int i = threadIdx.x; i < s.span * (N + 2); i += 256) span_sums[i] = 0.f;

  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const int e = threadIdx.x % (kSlice / 4) * 4, et = threadIdx.x / (kSlice / 4);  // this thread's element of a slice
  const int64_t tile0 = (int64_t)range * s.range_tiles, tile1 = min(tile0 + s.range_tiles, s.tiles);
  for (int64_t tile = tile0; tile < tile1; ++tile) {
    const int64_t token = tile * K + et;
    const int64_t maps = (((int64_t)(s.whole ? 0 : span) * s.batch + b) * s.tokens + tile * K) * s.groups * N + group * N;
    if (tile * K >= length) {  // nothing here depends on anything
      if (token < s.tokens) {
        for (int cc = c_first + e; cc < c_end; cc += kSlice) {
          const int64_t at = (b * s.tokens + token) * s.channels + cc;
          if (s.du) store4((T*)s.du + at, zero);
          if (s.ddt) store4((T*)s.ddt + at, zero);
          if (s.dz) store4((T*)s.dz + at, zero);
        }
      }
      for (int i = threadIdx.x; i < K * N; i += 256) {
        if (tile * K + i / N >= s.tokens) continue;
        const int64_t at = maps + (int64_t)(i / N) * s.groups * N + i % N;
        if (s.whole) {
          if (s.dB_out) ((T*)s.dB_out)[at] = (T)0.f;
          if (s.dC_out) ((T*)s.dC_out)[at] = (T)0.f;
        } else {
          s.dB[at] = 0.f, s.dC[at] = 0.f;
        }
      }
      continue;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < K * NP; i += 256) {
      const int t = i / NP, m = i % NP;
      const int64_t at = tile * K + t;
      const bool there = at < length && m < N;
      sB[m * kRow + t] = there ? load_f((const T*)s.B.p + b * s.B.sb + at * s.B.st + group * s.B.sg + m) : 0.f;
      sC[m * kRow + t] = there ? load_f((const T*)s.C.p + b * s.C.sb + at * s.C.st + group * s.C.sg + m) : 0.f;
    }
    float accB[K], accC[K];
#pragma unroll
    for (int t = 0; t < K; ++t) accB[t] = accC[t] = 0.f;
    // uniform addresses of the tile and this thread's offsets from them (a token's stride is below 2^26 elements)
    const int64_t first = b * s.tokens + tile * K;
    const T *u_at = (const T*)s.u.p + b * s.u.sb + tile * K * s.u.st + c_first;
    const T *dt_at = (const T*)s.dt.p + b * s.dt.sb + tile * K * s.dt.st + c_first;
    const T *z_at = (const T*)s.z.p + b * s.z.sb + tile * K * s.z.st + c_first;
    const uint32_t u_of = (uint32_t)et * (uint32_t)s.u.st + e, dt_of = (uint32_t)et * (uint32_t)s.dt.st + e;
    const uint32_t z_of = (uint32_t)et * (uint32_t)s.z.st + e, of = (uint32_t)et * (uint32_t)s.channels + e;
    const bool here = token < length;
    for (int c0 = 0; c0 < c_end - c_first; c0 += kSlice) {
      const bool mine = c0 + e < c_end - c_first, there = here && mine, inside = token < s.tokens && mine;
      const int64_t row = first * s.channels + c_first + c0;
      f32x4 u = zero, x = zero, dy = zero, z = zero, raw = zero, bias = zero;
      if (there) {
        u = load4(u_at + c0 + u_of), x = load4(dt_at + c0 + dt_of), dy = load4((const T*)s.dout + row + of);
        if (s.dt_bias) bias = load4(s.dt_bias + c_first + c0 + e);
        if (s.z.p) z = load4(z_at + c0 + z_of), raw = load4(s.raw + row + of);
      }
      __syncthreads();
      // a token that is not there has u, dy and z zero, and takes no step
      x += bias;
      f32x4 d = x;
      if (s.softplus) {
#pragma unroll
        for (int q = 0; q < 4; ++q) d[q] = step_of(x[q]);
      }
      d = d * (there ? 1.f : 0.f);
      if (s.z.p) {
        f32x4 dz;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float sg = sigmoid_f(z[q]);
          dz[q] = dy[q] * raw[q] * (sg + z[q] * sg * (1.f - sg));
          dy[q] = dy[q] * z[q] * sg;
        }
        if (s.dz && inside) store4((T*)s.dz + row + of, dz);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        sd[(e + q) * kRow + et] = d[q];
        sv[(e + q) * kRow + et] = d[q] * u[q];
        sy[(e + q) * kRow + et] = dy[q];
      }
      __syncthreads();
      for (int pass = 0; pass < kPasses; ++pass) {
        const int cl = (pass * 4 + wave) * kSlots + slot, c = c_first + c0 + cl;
        const bool live = c < c_end && held;
        const int64_t from = ((b * s.tiles + tile) * s.channels + c) * N + n;
        const float A = live ? s.A[(int64_t)c * N + n] : 0.f, A2 = A * kLog2e;
        const float h0 = live ? s.h_in[from] : 0.f;
        float X = live ? s.x_in[from] : 0.f, dA = 0.f;
        // d as an operand from the lanes of a row in the exponent; in multiply-adds, which take none, from LDS
        const float dl[2] = {sd[cl * kRow + r], sd[cl * kRow + 16 + r]};
        float h[K], a[K], last = h0;
        unrolled<K / 4>([&](auto quad) {
          constexpr int t0 = decltype(quad)::value * 4;
          const f32x4 v = *(const f32x4*)(sv + cl * kRow + t0), m = *(const f32x4*)(sB + n * kRow + t0);
          unrolled<4>([&](auto index) {
            constexpr int q = decltype(index)::value, t = t0 + q;
            a[t] = __builtin_amdgcn_exp2f(from_row<t % 16>(dl[t / 16]) * A2);
            h[t] = last = __builtin_fmaf(v[q], m[q], a[t] * last);
          });
          __builtin_amdgcn_sched_barrier(0);
        });
        RowSum sum1, sum2;
        unrolled<K / 4>([&](auto quad) {
          constexpr int t0 = K - 4 - decltype(quad)::value * 4;
          const f32x4 m = *(const f32x4*)(sB + n * kRow + t0), o = *(const f32x4*)(sC + n * kRow + t0);
          const f32x4 d = *(const f32x4*)(sd + cl * kRow + t0), v = *(const f32x4*)(sv + cl * kRow + t0);
          const f32x4 y = *(const f32x4*)(sy + cl * kRow + t0);
          unrolled<4>([&](auto index) {
            constexpr int q = 3 - decltype(index)::value, t = t0 + q, in = t % 16;
            const float G = __builtin_fmaf(y[q], o[q], X);
            accC[t] = __builtin_fmaf(y[q], h[t], accC[t]);
            accB[t] = __builtin_fmaf(v[q], G, accB[t]);
            asm volatile("" : "+v"(accB[t]), "+v"(accC[t]));  // here, not sunk behind the pass with all that they need
            X = a[t] * G;
            const float back = X * (t ? h[t ? t - 1 : 0] : h0);
            dA = __builtin_fmaf(d[q], back, dA);
            sum1.add<15 - in>(G * m[q], lane);
            sum2.add<15 - in>(A * back, lane);
          });
          if constexpr (t0 % 16 == 0) {
            float r1 = sum1.held[3], r2 = sum2.held[3];
            if (N >= 32) r1 += xor16(r1), r2 += xor16(r2);
            if (N == 64) r1 = xor32_sum(r1), r2 = xor32_sum(r2);
            if (N <= 16 || n < 16) {
              s1[cl * kRow + t0 + 15 - rev4(r)] = r1;
              s2[cl * kRow + t0 + 15 - rev4(r)] = r2;
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        });
        if (live) aA[(c - c_first) * N + n] += dA;
      }
      __syncthreads();
      {
        f32x4 du, ddt, skip = zero;
        if (s.D && mine) skip = load4(s.D + c_first + c0 + e);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int i = (e + q) * kRow + et;
          const float g = s1[i], y = sy[i];
          du[q] = there ? sd[i] * g + skip[q] * y : 0.f;
          ddt[q] = there ? u[q] * g + s2[i] : 0.f;
          s1[i] = there ? y * u[q] : 0.f;
        }
        if (s.softplus) {
#pragma unroll
          for (int q = 0; q < 4; ++q) ddt[q] *= sigmoid_f(x[q]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) s2[(e + q) * kRow + et] = ddt[q];
        if (inside && s.du) store4((T*)s.du + row + of, du);
        if (inside && s.ddt) store4((T*)s.ddt + row + of, ddt);
      }
      __syncthreads();
      // sums over the tile's tokens: four lanes a channel, 8 tokens each; dD by the first two waves, the bias's by the others
      {
        const int which = threadIdx.x >> 7, cl = threadIdx.x % 128 / 4, quarter = threadIdx.x % 4;
        const float* from = (which ? s2 : s1) + cl * kRow + 8 * quarter;
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) v += from[i];
        v += from_lane<0xB1>(v);
        v += from_lane<0x4E>(v);
        if (quarter == 0 && c_first + c0 + cl < c_end) (which ? ab : aD)[c0 + cl] += v;
      }
    }
    // the slots' and waves' sums of dB, then dC
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int t = 0; t < K; ++t) {
        float v = which ? accC[t] : accB[t];
        if (NP == 16) v += xor16(v);
        if (NP <= 32) v = xor32_sum(v);
        if (slot == 0 && held) lds[(wave * K + t) * N + n] = v;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < K * N; i += 256) {
        const float v = (lds[i] + lds[K * N + i]) + (lds[2 * K * N + i] + lds[3 * K * N + i]);
        if (tile * K + i / N >= s.tokens) continue;
        const int64_t at = maps + (int64_t)(i / N) * s.groups * N + i % N;
        if (!s.whole)
          (which ? s.dC : s.dB)[at] = v;
        else if (which ? s.dC_out : s.dB_out)
          ((T*)(which ? s.dC_out : s.dB_out))[at] = (T)v;
      }
    }
  }
  __syncthreads();
  const int64_t part = b * s.ranges + range;
  for (int i = threadIdx.x; i < (c_end - c_first) * N; i += 256) s.dA[(part * s.channels + c_first) * N + i] = aA[i];
  for (int i = threadIdx.x; i < c_end - c_first; i += 256) {
    s.dD[part * s.channels + c_first + i] = aD[i];
    s.dbias[part * s.channels + c_first + i] = ab[i];
  }
}

// Sums of partial rows, 16 columns by 16 slices of the rows a block: out[i] = sum over r of from[r * columns + i].
struct RowSums {
  const float* from[5];
  void* out[5];
  int64_t columns[5], rows[5];
  int bf16_out[5];
};
__global__ __launch_bounds__(256) void scan_sums_kernel(RowSums s) {
  __shared__ float lds[16][17];
  const int which = blockIdx.y, col = threadIdx.x % 16, slice = threadIdx.x / 16;
  if (!s.out[which]) return;
  for (int64_t first = (int64_t)blockIdx.x * 16; first < s.columns[which]; first += (int64_t)gridDim.x * 16) {
    const int64_t i = first + col;
    float v = 0.f;
    if (i < s.columns[which])
      for (int64_t r = slice; r < s.rows[which]; r += 16) v += s.from[which][r * s.columns[which] + i];
    __syncthreads();
    lds[slice][col] = v;
    __syncthreads();
    if (slice || i >= s.columns[which]) continue;
    v = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) v += lds[k][col];
    if (s.bf16_out[which])
      ((bf16*)s.out[which])[i] = (bf16)v;
    else
      ((float*)s.out[which])[i] = v;
  }
}

// ---------------------------------------------------------------------- host

template <typename Go>
void with_states(int64_t states, Go go) {
  using std::integral_constant;
  if (states == 8) return go(integral_constant<int, 8>());
  if (states == 16) return go(integral_constant<int, 16>());
  if (states == 32) return go(integral_constant<int, 32>());
  return go(integral_constant<int, 64>());
}

struct Chunks {
  int64_t chunks, tiles;  // tiles of a chunk
};
// One chunk where the channels alone make 768 blocks (three waves a SIMD), else about 1536 blocks.
Chunks plan_chunks(int64_t batch, int64_t tokens, int64_t channels, int64_t states, int64_t groups) {
  const int64_t tiles = (tokens + K - 1) / K, blocks = batch * groups * ((channels / groups + kWalk - 1) / kWalk);
  if (blocks >= 768 || tiles <= 2) return {1, tiles};
  int64_t chunks = (1536 + blocks - 1) / blocks;
  if (chunks > tiles) chunks = tiles;
  const int64_t each = (tiles + chunks - 1) / chunks;
  return {(tiles + each - 1) / each, each};
}

struct Spans {
  int64_t span, spans, ranges, range_tiles, whole;
};
// Spans of a group's channels and ranges of tiles of the gradient's blocks: about 1024 blocks.
Spans plan_spans(int64_t batch, int64_t tokens, int64_t channels, int64_t states, int64_t groups) {
  const int64_t tiles = (tokens + K - 1) / K, group = channels / groups;
  const int64_t most = kMaxSpan / states / kSlice * kSlice;
  Spans p;
  p.spans = (group + most - 1) / most;
  p.span = ((group + p.spans - 1) / p.spans + kSlice - 1) / kSlice * kSlice;
  p.spans = (group + p.span - 1) / p.span;
  const int64_t blocks = batch * groups * p.spans;
  int64_t ranges = (1024 + blocks - 1) / blocks;
  if (ranges > tiles) ranges = tiles;
  p.range_tiles = (tiles + ranges - 1) / ranges;
  p.ranges = (tiles + p.range_tiles - 1) / p.range_tiles;
  p.whole = p.spans == 1;
  return p;
}

int setup(Scan& s, const void* u, const void* dt, const float* A, const void* B, const void* C, const float* D,
          const void* z, const float* dt_bias, const void* lengths, int dtype, int lengths64, const int64_t* shape,
          const int64_t* strides, int softplus) {
  BMX_REQUIRE(dtype == kF32 || dtype == kBF16, "selective_scan: dtype must be fp32 or bf16");
  BMX_REQUIRE(shape && strides, "selective_scan: null shape or strides");
  for (int i = 0; i < 5; ++i) BMX_REQUIRE(shape[i] >= 0, "selective_scan: negative size");
  const int64_t channels = shape[2], states = shape[3], groups = shape[4];
  BMX_REQUIRE(states == 8 || states == 16 || states == 32 || states == 64, "selective_scan: states must be 8, 16, 32 or 64");
  BMX_REQUIRE(groups >= 1 && channels >= 8 && channels < (1 << 20) && channels % (8 * groups) == 0,
              "selective_scan: channels must be a multiple of 8 per group, below 2^20");
  BMX_REQUIRE(shape[0] < (1ll << 31) && shape[1] < (1ll << 31) && (shape[1] == 0 || shape[0] < (1ll << 31) / shape[1]),
              "selective_scan: expected fewer than 2^31 rows");
  for (int i = 0; i < 12; ++i)
    BMX_REQUIRE(strides[i] % 4 == 0, "selective_scan: strides must be multiples of 4");
  s.u = {u, strides[0], strides[1], 0}, s.dt = {dt, strides[2], strides[3], 0}, s.z = {z, strides[4], strides[5], 0};
  s.B = {B, strides[6], strides[7], strides[8]}, s.C = {C, strides[9], strides[10], strides[11]};
  s.A = A, s.D = D, s.dt_bias = dt_bias, s.lengths = lengths, s.lengths64 = lengths64, s.softplus = softplus != 0;
  s.batch = shape[0], s.tokens = shape[1], s.channels = (int)channels, s.states = (int)states, s.groups = (int)groups;
  s.group_channels = (int)(channels / groups), s.tiles = (s.tokens + K - 1) / K;
  return BMX_OK;
}

bool aligned(int to, std::initializer_list<const void*> pointers) {
  uintptr_t bits = 0;
  for (const void* p : pointers) bits |= (uintptr_t)p;
  return bits % to == 0;
}

int check_inputs(const Scan& s, int dtype) {
  BMX_REQUIRE(s.u.p && s.dt.p && s.A && s.B.p && s.C.p, "selective_scan: null pointer");
  BMX_REQUIRE(aligned(dtype == kF32 ? 16 : 8, {s.u.p, s.dt.p, s.z.p, s.B.p, s.C.p}),
              "selective_scan: tensors must be aligned to four elements");
  BMX_REQUIRE(aligned(16, {s.A, s.state, s.state_out, s.raw, s.saved}), "selective_scan: fp32 tensors must be 16-byte aligned");
  return BMX_OK;
}

template <typename T, int kMode>
int walk(Scan s, hipStream_t stream) {
  int rc = BMX_OK;
  with_states(s.states, [&](auto n) {
    constexpr int N = decltype(n)::value;
    s.cblocks = (s.group_channels + kWalk - 1) / kWalk;
    s.blocks = s.batch * s.chunks * s.groups * s.cblocks;
    if (s.blocks >= (1ll << 31)) {
      rc = set_error(BMX_EINVAL, "selective_scan: too many rows");
      return;
    }
    scan_walk_kernel<T, N, kMode><<<fold_grid(s.blocks, 256), 256, 0, stream>>>(s);
  });
  return rc ? rc : check_launch("selective_scan");
}

template <bool kReverse>
int carry(const Scan& s, const float* first, float* last, hipStream_t stream) {
  const int64_t blocks = (s.batch * s.channels * s.states + 255) / 256;
  BMX_REQUIRE(blocks < (1ll << 31), "selective_scan: too many states");
  scan_carry_kernel<kReverse><<<fold_grid(blocks, 256), 256, 0, stream>>>(s, first, last);
  return check_launch("selective_scan carry");
}

template <typename T>
int forward(Scan& s, hipStream_t stream) {
  if (s.tokens == 1 && !s.saved) {
    with_states(s.states, [&](auto n) {
      constexpr int N = decltype(n)::value;
      const int64_t blocks = (s.batch * s.channels * (N / 4) + 255) / 256;
      scan_step_kernel<T, N><<<fold_grid(blocks, 256), 256, 0, stream>>>(s);
    });
    return check_launch("selective_scan step");
  }
  if (s.chunks > 1) {
    if (int rc = walk<T, kLocal>(s, stream)) return rc;
    if (int rc = carry<false>(s, s.state, nullptr, stream)) return rc;
  }
  return walk<T, kOut>(s, stream);
}

template <typename T>
int gradient(Scan& s, const float* dstate_out, float* dstate, hipStream_t stream) {
  if (int rc = walk<T, kBack>(s, stream)) return rc;
  if (int rc = carry<true>(s, dstate_out, dstate, stream)) return rc;
  with_states(s.states, [&](auto n) {
    constexpr int N = decltype(n)::value;
    scan_bwd_kernel<T, N><<<fold_grid(s.blocks, 256), 256, s.span * (N + 2) * sizeof(float), stream>>>(s);
  });
  return check_launch("selective_scan_bwd");
}

// Floats of the gradient's workspace, part by part.
struct BackSpace {
  int64_t carry, steps, maps, dA, dD;
  BackSpace(int64_t batch, int64_t tokens, int64_t channels, int64_t states, int64_t groups, const Spans& p) {
    const int64_t tiles = (tokens + K - 1) / K, parts = batch * p.ranges;
    carry = batch * tiles * channels * states, steps = batch * tiles * channels;
    maps = p.whole ? 0 : p.spans * batch * tokens * groups * states;
    dA = parts * channels * states, dD = parts * channels;
  }
  int64_t floats() const { return carry + steps + 2 * maps + dA + 2 * dD; }
};

bool sizes_ok(int64_t batch, int64_t tokens, int64_t channels, int64_t states, int64_t groups) {
  return batch > 0 && tokens > 0 && groups > 0 && channels >= groups && states >= 8 && states <= 64;
}

}  // namespace

extern "C" size_t bmx_selective_scan_saved_bytes(int64_t batch, int64_t tokens, int64_t channels, int64_t states) {
  if (batch <= 0 || tokens <= 0 || channels <= 0 || states <= 0) return 0;
  return (size_t)(batch * ((tokens + K - 1) / K) * channels * states) * sizeof(float);
}

extern "C" size_t bmx_selective_scan_workspace_bytes(int64_t batch, int64_t tokens, int64_t channels, int64_t states,
                                                     int64_t groups) {
  if (!sizes_ok(batch, tokens, channels, states, groups)) return 0;
  const Chunks p = plan_chunks(batch, tokens, channels, states, groups);
  return p.chunks > 1 ? (size_t)(batch * p.chunks * channels * (states + 1)) * sizeof(float) : 0;
}

extern "C" int bmx_selective_scan_fwd(const void* u, const void* dt, const float* A, const void* B, const void* C,
                                      const float* D, const void* z, const float* dt_bias, const float* state,
                                      const void* lengths, int dtype, int lengths64, const int64_t* shape,
                                      const int64_t* strides, int softplus, void* out, float* state_out, float* saved,
                                      float* raw, void* workspace, size_t workspace_bytes, void* stream) {
  Scan s = {};
  if (int rc = setup(s, u, dt, A, B, C, D, z, dt_bias, lengths, dtype, lengths64, shape, strides, softplus)) return rc;
  if (s.batch == 0 || s.tokens == 0) {
    BMX_REQUIRE(s.batch == 0 || !state_out, "selective_scan: the state of no tokens is the caller's");
    return BMX_OK;
  }
  s.state = state, s.state_out = state_out, s.out = out, s.saved = saved, s.raw = raw;
  if (int rc = check_inputs(s, dtype)) return rc;
  BMX_REQUIRE(out && aligned(16, {out}), "selective_scan: out must be given, 16-byte aligned");
  BMX_REQUIRE(!raw || z, "selective_scan: raw needs z");
  const Chunks p = plan_chunks(s.batch, s.tokens, s.channels, s.states, s.groups);
  s.chunks = p.chunks, s.chunk_tiles = p.tiles;
  if (p.chunks > 1) {
    BMX_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 &&
                    workspace_bytes >=
                        bmx_selective_scan_workspace_bytes(s.batch, s.tokens, s.channels, s.states, s.groups),
                "selective_scan: workspace too small or not 16-byte aligned");
    s.carry = (float*)workspace;
    s.steps = s.carry + s.batch * p.chunks * s.channels * s.states;
  }
  return dtype == kF32 ? forward<float>(s, (hipStream_t)stream) : forward<bf16>(s, (hipStream_t)stream);
}

extern "C" size_t bmx_selective_scan_bwd_workspace_bytes(int64_t batch, int64_t tokens, int64_t channels, int64_t states,
                                                         int64_t groups) {
  if (!sizes_ok(batch, tokens, channels, states, groups)) return 0;
  const Spans p = plan_spans(batch, tokens, channels, states, groups);
  return (size_t)BackSpace(batch, tokens, channels, states, groups, p).floats() * sizeof(float);
}

extern "C" int bmx_selective_scan_bwd(const void* u, const void* dt, const float* A, const void* B, const void* C,
                                      const float* D, const void* z, const float* dt_bias, const void* lengths, int dtype,
                                      int lengths64, const int64_t* shape, const int64_t* strides, int softplus,
                                      const float* saved, const float* raw, const void* dout, const float* dstate_out,
                                      void* du, void* ddt, float* dA, void* dB, void* dC, float* dD, void* dz,
                                      float* ddt_bias, float* dstate, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  Scan s = {};
  if (int rc = setup(s, u, dt, A, B, C, D, z, dt_bias, lengths, dtype, lengths64, shape, strides, softplus)) return rc;
  BMX_REQUIRE(s.batch > 0 && s.tokens > 0, "selective_scan_bwd: expected rows");
  if (int rc = check_inputs(s, dtype)) return rc;
  BMX_REQUIRE(saved && dout && (!z || raw), "selective_scan_bwd: null pointer");
  BMX_REQUIRE((D || !dD) && (z || !dz) && (dt_bias || !ddt_bias), "selective_scan_bwd: gradient of an absent operand");
  BMX_REQUIRE(aligned(16, {saved, raw, dout, du, ddt, dz}), "selective_scan: tensors must be 16-byte aligned");
  const Spans p = plan_spans(s.batch, s.tokens, s.channels, s.states, s.groups);
  const BackSpace space(s.batch, s.tokens, s.channels, s.states, s.groups, p);
  BMX_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= (size_t)space.floats() * sizeof(float),
              "selective_scan_bwd: workspace too small or not 16-byte aligned");
  s.dout = dout, s.h_in = saved, s.raw = const_cast<float*>(raw), s.du = du, s.ddt = ddt, s.dz = dz;
  s.carry = (float*)workspace, s.steps = s.carry + space.carry, s.x_in = s.carry;
  s.dB = s.steps + space.steps, s.dC = s.dB + space.maps, s.dB_out = dB, s.dC_out = dC;
  s.dA = s.dC + space.maps, s.dD = s.dA + space.dA, s.dbias = s.dD + space.dD;
  s.chunks = s.tiles, s.chunk_tiles = 1;
  s.span = (int)p.span, s.spans = (int)p.spans, s.ranges = (int)p.ranges, s.range_tiles = (int)p.range_tiles;
  s.whole = (int)p.whole;
  s.blocks = s.batch * s.groups * p.spans * p.ranges;
  BMX_REQUIRE(s.blocks < (1ll << 31), "selective_scan: too many rows");
  hipStream_t hs = (hipStream_t)stream;
  if (int rc = dtype == kF32 ? gradient<float>(s, dstate_out, dstate, hs) : gradient<bf16>(s, dstate_out, dstate, hs))
    return rc;
  const int64_t parts = s.batch * p.ranges, maps = s.batch * s.tokens * s.groups * s.states;
  const RowSums sums = {{s.dA, s.dD, s.dbias, s.dB, s.dC},
                        {dA, dD, ddt_bias, p.whole ? nullptr : dB, p.whole ? nullptr : dC},
                        {(int64_t)s.channels * s.states, s.channels, s.channels, maps, maps},
                        {parts, parts, parts, p.spans, p.spans},
                        {0, 0, 0, dtype == kBF16, dtype == kBF16}};
  int64_t columns = (int64_t)s.channels * s.states;
  if (!p.whole && maps > columns) columns = maps;
  const int64_t blocks = (columns + 15) / 16;
  scan_sums_kernel<<<dim3((unsigned)(blocks < 16384 ? blocks : 16384), 5), 256, 0, hs>>>(sums);
  return check_launch("selective_scan_bwd sums");
}
