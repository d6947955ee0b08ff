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

#include "bmx_common.h"

using namespace bmx;

namespace {

constexpr int K = 32;             // tokens of a tile
constexpr int kRow = K + 4;       // LDS row of a channel or state over a tile: 16-byte reads along the tokens, no conflicts
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

// softplus(x) = max(x, 0) + log1p(exp(-|x|)); `slope` is its derivative, sigmoid(x).
__device__ __forceinline__ float step_of(float x, int softplus) {
  return softplus ? fmaxf(x, 0.f) + log1pf(__builtin_amdgcn_exp2f(-fabsf(x) * kLog2e)) : x;
}

// Lanes of one channel: L of them share its states, in the low bits of the lane, except that eight take the bits 0, 1
// and 3: a sum over them then is two exchanges within quads and one over 8 lanes of a row.
template <int L>
__device__ __forceinline__ int lane_state(int lane) {
  return L == 8 ? (lane & 3) | (lane >> 1 & 4) : lane % L;
}
template <int L>
__device__ __forceinline__ int lane_slot(int lane) {
  return L == 8 ? (lane >> 2 & 1) | (lane >> 3 & 6) : lane / L;
}
__device__ __forceinline__ float xor16(float v) {
  return __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(v), 0x401F));
}
__device__ __forceinline__ float xor32_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Sums of four values over the L >= 4 lanes of a channel; lane j gets the one of value j % 4.
template <int L>
__device__ __forceinline__ float sum4(const f32x4& p, int lane) {
  const bool odd = lane & 1, high = lane & 2;
  const float a = (odd ? p[1] : p[0]) + dpp<0xB1>(odd ? p[0] : p[1]);
  const float b = (odd ? p[3] : p[2]) + dpp<0xB1>(odd ? p[2] : p[3]);
  float v = (high ? b : a) + dpp<0x4E>(high ? a : b);
  if (L == 16 || L >= 32) v += dpp<0x124>(v);  // row_ror:4
  if (L >= 8) v += dpp<0x128>(v);              // row_ror:8
  if (L >= 32) v += xor16(v);
  if (L == 64) v = xor32_sum(v);
  return v;
}

// Four channels of one token as fp32; zeros where they are not there.
template <typename T>
__device__ __forceinline__ f32x4 row4(const Operand& o, int64_t b, int64_t t, int c, bool there) {
  return there ? load4((const T*)o.p + b * o.sb + t * o.st + c) : f32x4{0.f, 0.f, 0.f, 0.f};
}

// ------------------------------------------------------------ walking chunks

// kLocal: from zero states to each chunk's own, forward; kOut: the outputs; kBack: the same as kLocal for X, from the
// chunk's end, of dy in the place of d u and of C in the place of B.
enum Mode { kLocal, kOut, kBack };

template <typename T, int N, int L, int kMode>
__global__ __launch_bounds__(256) void scan_walk_kernel(Scan s) {
  constexpr int S = N / L, kChannels = 256 / L, kPer = (kChannels * K / 4 + 255) / 256, kMaps = (N * K / 4 + 255) / 256;
  __shared__ __align__(16) float sd[kChannels * kRow], sv[kChannels * kRow], sy[kMode == kOut ? kChannels * kRow : 4];
  __shared__ __align__(16) float sB[N * kRow], sC[kMode == kOut ? N * kRow : 4];
  int64_t block = block_index();
  if (block >= s.blocks) return;
  const int cblock = (int)(block % s.cblocks);
  block /= s.cblocks;
  const int group = (int)(block % s.groups);
  block /= s.groups;
  const int64_t chunk = block % s.chunks, b = block / s.chunks;
  const int c_first = group * s.group_channels + cblock * kChannels;
  const int c_end = min(c_first + kChannels, (group + 1) * s.group_channels);
  const int64_t length = length_of(s, b);
  const int lane = lane_id(), j = lane_state<L>(lane);
  const int c_local = (threadIdx.x >> 6) * (64 / L) + lane_slot<L>(lane), c = c_first + c_local;
  const bool live = c < c_end;

  float A2[S], h[S], total = 0.f;
#pragma unroll
  for (int i = 0; i < S; ++i) {
    A2[i] = live ? s.A[(int64_t)c * N + j * S + i] * kLog2e : 0.f;
    h[i] = 0.f;
  }
  if (kMode == kOut && live) {
    const float* from = s.chunks > 1 ? s.carry + ((b * s.chunks + chunk) * s.channels + c) * N
                        : s.state    ? s.state + (b * s.channels + c) * N
                                     : nullptr;
#pragma unroll
    for (int i = 0; i < S; ++i) h[i] = from ? from[j * S + i] : 0.f;
  }

  const int64_t tile0 = chunk * s.chunk_tiles, tile1 = min(tile0 + s.chunk_tiles, s.tiles);
  // this thread's elements of a tile: four channels of one token
  f32x4 ru[kPer], rdt[kPer], rz[kPer], rB[kMaps], rC[kMaps];
  auto fetch = [&](int64_t tile) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int at = threadIdx.x + 256 * i, e = at % (kChannels / 4) * 4, cc = c_first + e;
      const int64_t t = tile * K + at / (kChannels / 4);
      const bool there = at < kChannels / 4 * K && t < length && cc < c_end;
      rdt[i] = row4<T>(s.dt, b, t, cc, there);
      if (kMode == kBack)
        ru[i] = there ? load4((const T*)s.dout + (b * s.tokens + t) * s.channels + cc) : f32x4{0.f, 0.f, 0.f, 0.f};
      else
        ru[i] = row4<T>(s.u, b, t, cc, there);
      if (kMode != kLocal) rz[i] = row4<T>(s.z, b, t, cc, there && s.z.p);
    }
#pragma unroll
    for (int i = 0; i < kMaps; ++i) {
      const int at = threadIdx.x + 256 * i, n = at % (N / 4) * 4;
      const int64_t t = tile * K + at / (N / 4);
      const bool there = at < N / 4 * K && t < length;
      rB[i] = there && kMode != kBack ? load4((const T*)s.B.p + b * s.B.sb + t * s.B.st + group * s.B.sg + n)
                                      : f32x4{0.f, 0.f, 0.f, 0.f};
      rC[i] = there && kMode != kLocal ? load4((const T*)s.C.p + b * s.C.sb + t * s.C.st + group * s.C.sg + n)
                                       : f32x4{0.f, 0.f, 0.f, 0.f};
    }
  };

  fetch(kMode == kBack ? tile1 - 1 : tile0);
  for (int64_t k = tile0; k < tile1; ++k) {
    const int64_t tile = kMode == kBack ? tile0 + tile1 - 1 - k : k;
    // d, and d u (kBack: dy), of the tile to LDS, along the tokens; a token that is not there takes no step
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int at = threadIdx.x + 256 * i, e = at % (kChannels / 4) * 4, t = at / (kChannels / 4);
      if (at >= kChannels / 4 * K) continue;
      const bool there = tile * K + t < length && c_first + e < c_end;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float bias = s.dt_bias && there ? s.dt_bias[c_first + e + q] : 0.f;
        const float d = there ? step_of(rdt[i][q] + bias, s.softplus) : 0.f;
        sd[(e + q) * kRow + t] = d;
        if (kMode == kBack)
          sv[(e + q) * kRow + t] = s.z.p ? ru[i][q] * silu_f(rz[i][q]) : ru[i][q];
        else
          sv[(e + q) * kRow + t] = d * ru[i][q];
      }
    }
#pragma unroll
    for (int i = 0; i < kMaps; ++i) {
      const int at = threadIdx.x + 256 * i, n = at % (N / 4) * 4, t = at / (N / 4);
      if (at >= N / 4 * K) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        sB[(n + q) * kRow + t] = kMode == kBack ? rC[i][q] : rB[i][q];
        if (kMode == kOut) sC[(n + q) * kRow + t] = rC[i][q];
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
#pragma unroll
      for (int i = 0; i < S; ++i) s.saved[((b * s.tiles + tile) * s.channels + c) * N + j * S + i] = h[i];
    }

#pragma unroll 2
    for (int step = 0; step < K; step += 4) {
      const int t = kMode == kBack ? K - 4 - step : step;
      const f32x4 d = *(const f32x4*)(sd + c_local * kRow + t), v = *(const f32x4*)(sv + c_local * kRow + t);
      f32x4 p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const f32x4 m = *(const f32x4*)(sB + (j * S + i) * kRow + t);
        if (kMode == kBack) {
#pragma unroll
          for (int q = 3; q >= 0; --q) h[i] = __builtin_amdgcn_exp2f(d[q] * A2[i]) * (m[q] * v[q] + h[i]);
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            h[i] = __builtin_amdgcn_exp2f(d[q] * A2[i]) * h[i] + m[q] * v[q];
            if (kMode == kOut) p[q] += sC[(j * S + i) * kRow + t + q] * h[i];
          }
        }
      }
      if (kMode != kOut) {
        total += (d[0] + d[1]) + (d[2] + d[3]);
      } else {
        const float y = sum4<L>(p, lane);
        if (j < 4) sy[c_local * kRow + t + j] = y;
      }
    }
    __syncthreads();
    if (kMode == kOut) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int at = threadIdx.x + 256 * i, e = at % (kChannels / 4) * 4, t = at / (kChannels / 4);
        const int64_t token = tile * K + t;
        if (at >= kChannels / 4 * K || token >= s.tokens || c_first + e >= c_end) continue;
        const bool there = token < length;
        f32x4 y;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          y[q] = sy[(e + q) * kRow + t] + (s.D ? s.D[c_first + e + q] * keep_u[i][q] : 0.f);
          if (!there) y[q] = 0.f;
        }
        const int64_t to = (b * s.tokens + token) * s.channels + c_first + e;
        if (s.raw) store4(s.raw + to, y);
        if (s.z.p) {
#pragma unroll
          for (int q = 0; q < 4; ++q) y[q] = there ? y[q] * silu_f(keep_z[i][q]) : 0.f;
        }
        store4((T*)s.out + to, y);
      }
    }
  }
  if (!live) return;
  if (kMode == kOut) {
    if (s.state_out && chunk == s.chunks - 1) {
#pragma unroll
      for (int i = 0; i < S; ++i) s.state_out[(b * s.channels + c) * N + j * S + i] = h[i];
    }
    return;
  }
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
    const float d = step_of((float)((const T*)s.dt.p)[b * s.dt.sb + c] + (s.dt_bias ? s.dt_bias[c] : 0.f), s.softplus);
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

// A block takes a span of a group's channels and a range of tiles.  A lane has one state and, wave by wave, channel
// after channel: B, C and the sums dB, dC of its state stay in its registers over a tile, h and a of a channel over its
// 32 tokens.  dA, dD and the bias's sums stay in LDS over the range.
template <typename T, int N>
__global__ __launch_bounds__(256, 2) void scan_bwd_kernel(Scan s) {
  constexpr int kSlots = 64 / N, kPasses = kSlice / (4 * kSlots);
  constexpr int kStage = 5 * kSlice * kRow, kJoin = 4 * K * N;
  __shared__ __align__(16) float lds[kStage > kJoin ? kStage : kJoin];
  extern __shared__ __align__(16) float span_sums[];  // dA [span][N], dD [span], dbias [span]
  float *sd = lds, *sv = sd + kSlice * kRow, *sy = sv + kSlice * kRow, *s1 = sy + kSlice * kRow, *s2 = s1 + kSlice * kRow;
  float *aA = span_sums, *aD = aA + s.span * N, *ab = aD + s.span;
  int64_t block = block_index();
  if (block >= s.blocks) return;
  const int span = (int)(block % s.spans);
  block /= s.spans;
  const int group = (int)(block % s.groups);
  block /= s.groups;
  const int range = (int)(block % s.ranges);
  const int64_t b = block / s.ranges, length = length_of(s, b);
  const int c_first = group * s.group_channels + span * s.span;
  const int c_end = min(c_first + s.span, (group + 1) * s.group_channels);
  const int lane = lane_id(), wave = threadIdx.x >> 6, n = lane_state<N>(lane), slot = lane_slot<N>(lane);
  for (int i = threadIdx.x; i < s.span * (N + 2); i += 256) span_sums[i] = 0.f;

  const int e = threadIdx.x % (kSlice / 4) * 4, et = threadIdx.x / (kSlice / 4);  // this thread's element of a slice
  const int64_t tile0 = (int64_t)range * s.range_tiles, tile1 = min(tile0 + s.range_tiles, s.tiles);
  for (int64_t tile = tile0; tile < tile1; ++tile) {
    const int64_t token = tile * K + et;
    if (tile * K >= length) {  // nothing here depends on anything
      const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
      if (token < s.tokens) {
        for (int cc = c_first + e; cc < c_end; cc += kSlice) {
          const int64_t at = (b * s.tokens + token) * s.channels + cc;
          if (s.du) store4((T*)s.du + at, zero);
          if (s.ddt) store4((T*)s.ddt + at, zero);
          if (s.dz) store4((T*)s.dz + at, zero);
        }
      }
      for (int i = threadIdx.x; i < K * N; i += 256) {
        const int64_t t = tile * K + i / N;
        if (t >= s.tokens) continue;
        const int64_t at = (((int64_t)(s.whole ? 0 : span) * s.batch + b) * s.tokens + t) * s.groups * N + group * N + i % N;
        if (s.whole) {
          if (s.dB_out) ((T*)s.dB_out)[at] = (T)0.f;
          if (s.dC_out) ((T*)s.dC_out)[at] = (T)0.f;
        } else {
          s.dB[at] = 0.f, s.dC[at] = 0.f;
        }
      }
      continue;
    }
    float Bm[K], Cm[K], accB[K], accC[K];
#pragma unroll
    for (int t = 0; t < K; ++t) {
      const int64_t at = tile * K + t;
      const bool there = at < length;
      Bm[t] = there ? load_f((const T*)s.B.p + b * s.B.sb + at * s.B.st + group * s.B.sg + n) : 0.f;
      Cm[t] = there ? load_f((const T*)s.C.p + b * s.C.sb + at * s.C.st + group * s.C.sg + n) : 0.f;
      accB[t] = accC[t] = 0.f;
    }
    for (int c0 = c_first; c0 < c_end; c0 += kSlice) {
      const bool there = token < length && c0 + e < c_end, inside = token < s.tokens && c0 + e < c_end;
      const int64_t at = (b * s.tokens + token) * s.channels + c0 + e;
      const f32x4 u = row4<T>(s.u, b, token, c0 + e, there), z = row4<T>(s.z, b, token, c0 + e, there && s.z.p);
      f32x4 x = row4<T>(s.dt, b, token, c0 + e, there), d, dy, dz;
      dy = there && s.dout ? load4((const T*)s.dout + at) : f32x4{0.f, 0.f, 0.f, 0.f};
      const f32x4 raw = there && s.z.p ? load4(s.raw + at) : f32x4{0.f, 0.f, 0.f, 0.f};
      __syncthreads();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        x[q] += there && s.dt_bias ? s.dt_bias[c0 + e + q] : 0.f;
        d[q] = there ? step_of(x[q], s.softplus) : 0.f;
        if (s.z.p) {
          const float sg = sigmoid_f(z[q]);
          dz[q] = there ? dy[q] * raw[q] * (sg + z[q] * sg * (1.f - sg)) : 0.f;
          dy[q] = there ? dy[q] * z[q] * sg : 0.f;
        }
        sd[(e + q) * kRow + et] = d[q];
        sv[(e + q) * kRow + et] = d[q] * u[q];
        sy[(e + q) * kRow + et] = dy[q];
      }
      if (s.dz && inside) store4((T*)s.dz + at, dz);
      __syncthreads();
      for (int pass = 0; pass < kPasses; ++pass) {
        const int cl = (pass * 4 + wave) * kSlots + slot, c = c0 + cl;
        const bool live = c < c_end;
        const int64_t from = ((b * s.tiles + tile) * s.channels + c) * N + n;
        const float A = live ? s.A[(int64_t)c * N + n] : 0.f, A2 = A * kLog2e;
        const float h0 = live ? s.h_in[from] : 0.f;
        float X = live ? s.x_in[from] : 0.f, dA = 0.f;
        float h[K], a[K];
#pragma unroll
        for (int t = 0; t < K; t += 4) {
          const f32x4 dl = *(const f32x4*)(sd + cl * kRow + t), vl = *(const f32x4*)(sv + cl * kRow + t);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            a[t + q] = __builtin_amdgcn_exp2f(dl[q] * A2);
            h[t + q] = a[t + q] * (t + q ? h[t + q ? t + q - 1 : 0] : h0) + Bm[t + q] * vl[q];
          }
        }
#pragma unroll
        for (int t = K - 4; t >= 0; t -= 4) {
          const f32x4 dl = *(const f32x4*)(sd + cl * kRow + t), vl = *(const f32x4*)(sv + cl * kRow + t);
          const f32x4 yl = *(const f32x4*)(sy + cl * kRow + t);
          f32x4 p1, p2;
#pragma unroll
          for (int q = 3; q >= 0; --q) {
            const float G = Cm[t + q] * yl[q] + X;
            accC[t + q] += yl[q] * h[t + q];
            accB[t + q] += G * vl[q];
            p1[q] = G * Bm[t + q];
            X = a[t + q] * G;
            const float back = X * (t + q ? h[t + q ? t + q - 1 : 0] : h0);
            dA += dl[q] * back;
            p2[q] = A * back;
          }
          const float r1 = sum4<N>(p1, lane), r2 = sum4<N>(p2, lane);
          if (n < 4) {
            s1[cl * kRow + t + n] = r1;
            s2[cl * kRow + t + n] = r2;
          }
        }
        if (live) aA[(c - c_first) * N + n] += dA;
      }
      __syncthreads();
      f32x4 du, ddt;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float g = s1[(e + q) * kRow + et], D = s.D && inside ? s.D[c0 + e + q] : 0.f;
        du[q] = there ? d[q] * g + D * dy[q] : 0.f;
        float slope = 1.f;
        if (s.softplus) slope = sigmoid_f(x[q]);
        ddt[q] = there ? (u[q] * g + s2[(e + q) * kRow + et]) * slope : 0.f;
        s1[(e + q) * kRow + et] = there ? dy[q] * u[q] : 0.f;
        s2[(e + q) * kRow + et] = ddt[q];
      }
      if (inside && s.du) store4((T*)s.du + at, du);
      if (inside && s.ddt) store4((T*)s.ddt + at, ddt);
      __syncthreads();
      // sums over the tile's tokens: four lanes a channel, 8 tokens each; dD by the first two waves, the bias's by the others
      {
        const int which = threadIdx.x >> 7, cl = threadIdx.x % 128 / 4, quarter = threadIdx.x % 4;
        const float* from = (which ? s2 : s1) + cl * kRow + 8 * quarter;
        const f32x4 p = *(const f32x4*)from, q = *(const f32x4*)(from + 4);
        float v = ((p[0] + p[1]) + (p[2] + p[3])) + ((q[0] + q[1]) + (q[2] + q[3]));
        v += dpp<0xB1>(v);
        v += dpp<0x4E>(v);
        if (quarter == 0 && c0 + cl < c_end) (which ? ab : aD)[c0 - c_first + cl] += v;
      }
    }
    // the slots' and waves' sums of dB, then dC
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int t = 0; t < K; ++t) {
        float v = which ? accC[t] : accB[t];
        if (N == 8) v += __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(v), 0x101F));  // xor 4
        if (N <= 16) v += xor16(v);
        if (N <= 32) v = xor32_sum(v);
        if (slot == 0) lds[(wave * K + t) * N + n] = v;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < K * N; i += 256) {
        const float v = (lds[i] + lds[K * N + i]) + (lds[2 * K * N + i] + lds[3 * K * N + i]);
        const int64_t t = tile * K + i / N;
        if (t >= s.tokens) continue;
        const int64_t to = (((int64_t)(s.whole ? 0 : span) * s.batch + b) * s.tokens + t) * s.groups * N + group * N + i % N;
        if (!s.whole)
          (which ? s.dC : s.dB)[to] = v;
        else if (which ? s.dC_out : s.dB_out)
          ((T*)(which ? s.dC_out : s.dB_out))[to] = (T)v;
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

// Lanes of a channel where chunks are walked: four states each (of eight states two).
constexpr int walk_lanes(int states) { return states <= 16 ? 4 : states / 4; }

struct Chunks {
  int64_t chunks, tiles;  // tiles of a chunk
};
// One chunk where the channels alone make 768 blocks (three waves a SIMD), else about 1536 blocks.
Chunks plan_chunks(int64_t batch, int64_t tokens, int64_t channels, int64_t states, int64_t groups) {
  const int64_t per = 256 / walk_lanes((int)states), tiles = (tokens + K - 1) / K;
  const int64_t blocks = batch * groups * ((channels / groups + per - 1) / per);
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
    constexpr int N = decltype(n)::value, L = walk_lanes(N);
    s.cblocks = (s.group_channels + 256 / L - 1) / (256 / L);
    s.blocks = s.batch * s.chunks * s.groups * s.cblocks;
    if (s.blocks >= (1ll << 31)) {
      rc = set_error(BMX_EINVAL, "selective_scan: too many rows");
      return;
    }
    scan_walk_kernel<T, N, L, kMode><<<fold_grid(s.blocks, 256), 256, 0, stream>>>(s);
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
