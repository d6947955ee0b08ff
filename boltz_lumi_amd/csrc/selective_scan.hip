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
// Backward, X goes through the first two passes from the end; a chunk then has the
// X that comes to it and, tile by tile, the h that the forward pass kept, and is
// worked out on its own.  States, sums and statistics are fp32; tokens from a
// sequence's length on take no step (d = 0), are never read and give zeros.
//
// What bounds it is vector instructions, an exp (2.6 slots of the 38.5e12 lanes
// a second) per state and token and four around it in a walk, 16 to 20 in the
// gradient, so that a second walk costs more than its bytes.  bf16, four ragged
// sequences of up to 2048 tokens, 1536 channels of 16 states, us (its
// instructions alone): kLocal 41 (30), kOut 58 (41), kBack 47 (34), gradient 160
// (106), both carries 15, sums 7; 45 would be the bytes of all.  With 16 lanes a
// channel instead of four and no chunks the outputs take 166.
#include <type_traits>
#include <utility>

#include "bmx_common.h"

using namespace bmx;

namespace {

constexpr int K = 32;             // tokens of a tile
constexpr int kRow = K + 4;       // LDS row of a state's map over a tile: 16-byte reads along the tokens, no conflicts
constexpr int KG = 16;            // tokens of a tile of the gradient, which keeps that many states and decays in registers
constexpr int kGradRow = KG + 4;
constexpr int kChannelRow = K + 2;  // LDS row of a channel: reads without conflicts, transposing writes two on a bank
constexpr int kSlice = 16;        // channels that a wave of the gradient stages at a time
// Channels x states of a gradient block (X and dA in LDS), but at least 64 channels.  4 x 2048 tokens, 1536 channels of 16
// states, both ways: 324 us; with 4096 368 (one block less a compute unit), with 1024 347 (more partial sums dB, dC).
constexpr int kMaxSpan = 2048;
constexpr int64_t kRound = 4 * 256;  // blocks of a walk that the card holds
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
  float* saved;             // [batch][grad_tiles][channels][states]: h where every tile of the gradient begins
  const float *h_in, *x_in;
  void *du, *ddt, *dz;
  float *dB, *dC;           // partial sums, [spans][batch][tokens][groups][states]; unused where there is one span
  void *dB_out, *dC_out;    // the results
  float *dA, *dD, *dbias;   // partial sums, [batch * ranges][channels]([states])
  int64_t batch, tokens, tiles, grad_tiles, chunks, chunk_tiles, blocks;
  int channels, groups, group_channels, states, cblocks, lengths64, softplus;
  int span, spans, ranges, range_tiles, whole;
};

// ------------------------------------------------------------------ elements

__device__ __forceinline__ int64_t length_of(const Scan& s, int64_t b) {
  if (!s.lengths) return s.tokens;
  const int64_t n = s.lengths64 ? ((const int64_t*)s.lengths)[b] : (int64_t)((const int32_t*)s.lengths)[b];
  return n < 0 ? 0 : n < s.tokens ? n : s.tokens;
}

// softplus(x) = max(x, 0) + log1p(e), e = exp(-|x|), with log(1 + e) = 2 atanh(r), r = e / (2 + e) <= 1 / 3, and
// 2 atanh(r) / r a polynomial of degree four in r^2, within 1.6e-08 of it on [0, 1 / 9] (7.8e-09 relative, an eighth of a
// rounding): log1p(e) is held relative to itself, however small e is.  e is off by its exponent's roundings, up to 1.3 |x|
// of 2^-24 (seen: 17 at x = -20, 65 at -87), and a small step with it.
__device__ __forceinline__ float step_of(float x) {
  const float e = __builtin_amdgcn_exp2f(-fabsf(x) * kLog2e);
  const float r = e * __builtin_amdgcn_rcpf(2.f + e), q = r * r;
  float s = 0.281783193f;
  s = s * q + 0.279606074f;
  s = s * q + 0.400249094f;
  s = s * q + 0.66666317f;
  s = s * q + 2.f;
  return s * r + __builtin_amdgcn_fmed3f(x, 0.f, __builtin_inff());
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

// L lanes of a channel share its states, in the low bits of the lane, except that eight take the bits 0, 1 and 3: a sum
// over them then is two exchanges within quads and one over 8 lanes of a row.
template <int L>
__device__ __forceinline__ int lane_state(int lane) {
  return L == 8 ? (lane & 3) | (lane >> 1 & 4) : lane % L;
}
template <int L>
__device__ __forceinline__ int lane_slot(int lane) {
  return L == 8 ? (lane >> 2 & 1) | (lane >> 3 & 6) : lane / L;
}

// Sums of four values over the L >= 4 lanes of a channel; lane j gets the one of value j % 4.
template <int L>
__device__ __forceinline__ float sum4(const f32x4& p, int lane) {
  const bool odd = lane & 1, high = lane & 2;
  const float a = (odd ? p[1] : p[0]) + from_lane<0xB1>(odd ? p[0] : p[1]);
  const float b = (odd ? p[3] : p[2]) + from_lane<0xB1>(odd ? p[2] : p[3]);
  float v = (high ? b : a) + from_lane<0x4E>(high ? a : b);
  if (L >= 16) v += from_lane<0x124>(v);  // row_ror:4
  if (L >= 8) v += from_lane<0x128>(v);   // row_ror:8
  if (L >= 32) v += xor16(v);
  if (L == 64) v = xor32_sum(v);
  return v;
}

// Sums of 16 values over the 16 lanes of a row, one value after another; lane j gets the one of value rev4(j), j's four
// bits reversed.  Level by level two values become one, a lane keeping the first or the second by one of its bits; the
// exchange partner (15 - j, 7 - j, j xor 2, j xor 1) has the other value of that bit, and the earlier ones' equal.
__device__ __forceinline__ int rev4(int j) { return (j & 1) << 3 | (j & 2) << 1 | (j & 4) >> 1 | (j & 8) >> 3; }
struct RowSum {
  float held[4];
  template <int kIndex>
  __device__ __forceinline__ void add(float v, int lane) {  // in the order 0 .. 15; the last leaves its sum in held[3]
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

// Four values as they lie in memory: a load in flight holds no more registers than it has bytes.  Addresses are a uniform
// base and a lane's bytes from it, which fit 32 bits (a token's stride is below 2^25 elements, a tile 32 tokens).
template <typename T>
struct Four;
template <>
struct Four<float> {
  f32x4 v;
  __device__ __forceinline__ f32x4 wide() const { return v; }
};
template <>
struct Four<bf16> {
  bf16x4 v;
  __device__ __forceinline__ f32x4 wide() const { return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]}; }
};
template <typename T>
__device__ __forceinline__ Four<T> four(const T* base, uint32_t bytes, bool there) {
  Four<T> o = {};
  if (there) o = *(const Four<T>*)((const char*)base + bytes);
  return o;
}
template <typename T>
__device__ __forceinline__ void put4(T* base, uint32_t bytes, const f32x4& v) {
  store4((T*)((char*)base + bytes), v);
}

// Between a wave's LDS writes and its other lanes' reads: the LDS keeps a wave's order, the compiler has to.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// v, as a value that the compiler does not know: what is worked out of it is not kept in registers over the loops around.
__device__ __forceinline__ int again(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// The same for a value that all lanes share, in a scalar register: an address of it and a lane's constant offset takes
// no vector registers of its own.
__device__ __forceinline__ int uniform(int v) {
  v = __builtin_amdgcn_readfirstlane(v);
  asm volatile("" : "+s"(v));
  return v;
}

// ------------------------------------------------------------ walking chunks

// kLocal: from zero states to each chunk's own, forward; kOut: the outputs; kBack: the same as kLocal for X, from the
// chunk's end, of dy in the place of d u and of C in the place of B.
enum Mode { kLocal, kOut, kBack };

template <typename T, int N, int L, int kMode>
__global__ __launch_bounds__(256, 4) void scan_walk_kernel(Scan s) {
  constexpr int S = N / L, kWalk = 256 / L, kPer = (kWalk * K / 4 + 255) / 256, kMaps = (N * K / 4 + 255) / 256;
  constexpr int kStep = K / kPer, kMapStep = 1024 / N;  // tokens between a thread's elements, and between its maps'
  __shared__ float sd[kWalk * kChannelRow], sv[kWalk * kChannelRow], sy[kMode == kOut ? kWalk * kChannelRow : 4];
  __shared__ __align__(16) float sB[N * kRow], sC[kMode == kOut ? N * kRow : 4];
  // Neighbours in channels read the same lines (below 64 bf16 channels a block): four at a time are dealt to an XCD.
  // Longer runs would give an XCD whole sequences, whose lengths differ.
  uint32_t block = block_index();
  block = (block / 32 * 8 + block % 8) * 4 + block / 8 % 4;
  if (block >= s.blocks) return;
  const int cblock = (int)(block % (uint32_t)s.cblocks);
  block /= (uint32_t)s.cblocks;
  const int group = (int)(block % (uint32_t)s.groups);
  block /= (uint32_t)s.groups;
  const int64_t chunk = block % (uint32_t)s.chunks, b = block / (uint32_t)s.chunks;
  const int c_first = group * s.group_channels + cblock * kWalk;
  const int c_end = min(c_first + kWalk, (group + 1) * s.group_channels);
  const int64_t length = length_of(s, b);
  const int lane = lane_id(), j = lane_state<L>(lane), jq = lane & 3;
  const int c_local = (threadIdx.x >> 6) * (64 / L) + lane_slot<L>(lane), c = c_first + c_local;
  const bool live = c < c_end;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};

  // tiles of this chunk that have tokens, and those behind them, which states pass
  const int64_t tile0 = chunk * s.chunk_tiles, tile1 = min(tile0 + s.chunk_tiles, s.tiles);
  const int64_t tile_end = max(tile0, min(tile1, (length + K - 1) / K));

  // this thread's elements of a tile: four channels of kPer tokens, and of the maps four states of kMaps tokens
  const int e = threadIdx.x % (kWalk / 4) * 4, et = threadIdx.x / (kWalk / 4), cc = c_first + e;
  const int en = threadIdx.x % (N / 4) * 4, ent = threadIdx.x / (N / 4);
  const bool mine = cc < c_end && et < K;
  const uint32_t size = sizeof(T), u_st = kMode == kBack ? s.channels : (uint32_t)s.u.st;
  const uint32_t u_of = (et * u_st + e) * size, dt_of = (et * (uint32_t)s.dt.st + e) * size;
  const uint32_t z_of = (et * (uint32_t)s.z.st + e) * size, of = et * (uint32_t)s.channels + e;
  const uint32_t B_of = (ent * (uint32_t)s.B.st + en) * size, C_of = (ent * (uint32_t)s.C.st + en) * size;
  const bool gate_grad = kMode == kBack && s.dz;
  Four<T> ru[kPer], rdt[kPer], rz[kPer], rB[kMaps], rC[kMaps];
  f32x4 rraw[kPer];
  auto fetch = [&](int64_t tile) {
    const int left = (int)min(length - tile * K, (int64_t)K);
    const int64_t row = (b * s.tokens + tile * K) * s.channels + c_first;
    const T* u = kMode == kBack ? (const T*)s.dout + row : (const T*)s.u.p + b * s.u.sb + tile * K * s.u.st + c_first;
    const T* dt = (const T*)s.dt.p + b * s.dt.sb + tile * K * s.dt.st + c_first;
    const T* z = (const T*)s.z.p + b * s.z.sb + tile * K * s.z.st + c_first;
    const T* B = (const T*)s.B.p + b * s.B.sb + tile * K * s.B.st + group * s.B.sg;
    const T* C = (const T*)s.C.p + b * s.C.sb + tile * K * s.C.st + group * s.C.sg;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const bool there = mine && et + i * kStep < left;
      rdt[i] = four(dt + i * kStep * s.dt.st, dt_of, there);
      ru[i] = four(u + (int64_t)(i * kStep) * u_st, u_of, there);
      if (kMode != kLocal) rz[i] = four(z + i * kStep * s.z.st, z_of, there && s.z.p);
      if (kMode == kBack)
        rraw[i] = four(s.raw + row + (int64_t)(i * kStep) * s.channels, of * 4, there && gate_grad).wide();
    }
#pragma unroll
    for (int i = 0; i < kMaps; ++i) {
      const bool there = ent + i * kMapStep < left;
      if (kMode != kBack) rB[i] = four(B + i * kMapStep * s.B.st, B_of, there);
      if (kMode != kLocal) rC[i] = four(C + i * kMapStep * s.C.st, C_of, there);
    }
  };
  if (tile_end > tile0) fetch(kMode == kBack ? tile_end - 1 : tile0);

  f32x4 bias = zero, skip = zero;
  if (mine && s.dt_bias) bias = load4(s.dt_bias + cc);
  if (kMode == kOut && mine && s.D) skip = load4(s.D + cc);
  typedef float States __attribute__((ext_vector_type(S)));
  const float* from = nullptr;
  if (kMode == kOut)
    from = s.chunks > 1 ? s.carry + ((b * s.chunks + chunk) * s.channels + c) * N
           : s.state    ? s.state + (b * s.channels + c) * N
                        : nullptr;
  States A = {}, h = {};
  if (live) A = *(const States*)(s.A + (int64_t)c * N + j * S);
  if (live && from) h = *(const States*)(from + j * S);
  const States A2 = A * kLog2e;
  float total = 0.f;
  int own[S];
#pragma unroll
  for (int i = 0; i < S; ++i) own[i] = again(c_local * kChannelRow + jq);
  auto save = [&](int64_t tile, int part) {  // h where a tile of the gradient begins
    const int64_t at = tile * (K / KG) + part;
    if (kMode != kOut || !s.saved || !live || at >= s.grad_tiles) return;
    *(States*)(s.saved + ((b * s.grad_tiles + at) * s.channels + c) * N + j * S) = h;
  };

  for (int64_t k = tile0; k < tile_end; ++k) {
    const int64_t tile = kMode == kBack ? tile0 + tile_end - 1 - k : k;
    const int64_t row = (b * s.tokens + tile * K) * s.channels + c_first;
    const int left = (int)min(length - tile * K, (int64_t)K), inside = (int)min(s.tokens - tile * K, (int64_t)K);
    // d, and d u (kBack: dy), of the tile to LDS, along the tokens; a token that is not there takes no step
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int t = et + i * kStep;
      f32x4 d = rdt[i].wide() + bias, v = ru[i].wide();
      if (s.softplus) {
#pragma unroll
        for (int q = 0; q < 4; ++q) d[q] = step_of(d[q]);
      }
      d = d * (mine && t < left ? 1.f : 0.f);
      if (kMode != kBack) {
        v = v * d;
      } else if (s.z.p) {
        const f32x4 z = rz[i].wide();
        f32x4 dz;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float sg = sigmoid_f(z[q]);
          dz[q] = v[q] * rraw[i][q] * (sg + z[q] * sg * (1.f - sg));
          v[q] *= z[q] * sg;
        }
        if (gate_grad && mine && t < inside)
          put4((T*)s.dz + row + (int64_t)(i * kStep) * s.channels, of * size, dz);
      }
      if (kPer * 256 > kWalk * K / 4 && et >= K) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        sd[(e + q) * kChannelRow + t] = d[q];
        sv[(e + q) * kChannelRow + t] = v[q];
      }
    }
#pragma unroll
    for (int i = 0; i < kMaps; ++i) {
      const int t = ent + i * kMapStep;
      if (t >= K) continue;
      const f32x4 m = (kMode == kBack ? rC[i] : rB[i]).wide();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        sB[(en + q) * kRow + t] = m[q];
        if (kMode == kOut) sC[(en + q) * kRow + t] = rC[i].wide()[q];
      }
    }
    __syncthreads();
    Four<T> keep_u[kPer], keep_z[kPer];
    if (kMode == kOut) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) keep_u[i] = ru[i], keep_z[i] = rz[i];
    }
    if (k + 1 < tile_end) fetch(kMode == kBack ? tile - 1 : tile + 1);

    // Four tokens at a time: lane i of a quad holds token i's d and d u, which the others take from it as an operand.
    // Each state reads them for itself: were they one value, it would be moved to every lane by an instruction of its own.
#pragma unroll 2
    for (int step = 0; step < K; step += 4) {
      if (step % KG == 0) save(tile, step / KG);
      const int t = kMode == kBack ? K - 4 - step : step;
      f32x4 p = zero;
#pragma unroll
      for (int i = 0; i < S; ++i) {
        const float d = sd[own[i] + t], v = sv[own[i] + t];
        if (kMode != kOut && i == 0) total += d;
        const f32x4 m = *(const f32x4*)(sB + (j * S + i) * kRow + t);
        f32x4 r = zero;
        if (kMode == kOut) r = *(const f32x4*)(sC + (j * S + i) * kRow + t);
        unrolled<4>([&](auto index) {
          constexpr int q = kMode == kBack ? 3 - decltype(index)::value : decltype(index)::value;
          const float a = __builtin_amdgcn_exp2f(from_quad<q>(d) * A2[i]);
          const float into = from_quad<q>(v) * m[q];  // not fused: a multiply-add takes no other lane's operand
          if (kMode == kBack) {
            h[i] = a * (into + h[i]);
          } else {
            h[i] = __builtin_fmaf(a, h[i], into);
            if (kMode == kOut) p[q] = __builtin_fmaf(r[q], h[i], p[q]);
          }
        });
      }
      if (kMode == kOut) {
        const float y = sum4<L>(p, lane);
        if (L == 4 || j < 4) sy[own[0] + t] = y;
      }
    }
    __syncthreads();
    if (kMode == kOut) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int t = et + i * kStep;
        if (!mine || t >= inside) continue;
        const bool there = t < left;
        const f32x4 u = keep_u[i].wide();
        f32x4 y;
#pragma unroll
        for (int q = 0; q < 4; ++q) y[q] = there ? sy[(e + q) * kChannelRow + t] + skip[q] * u[q] : 0.f;
        const int64_t to = row + (int64_t)(i * kStep) * s.channels;
        if (s.raw) put4(s.raw + to, of * 4, y);
        if (s.z.p) {
          const f32x4 z = keep_z[i].wide();
#pragma unroll
          for (int q = 0; q < 4; ++q) y[q] = there ? y[q] * silu_f(z[q]) : 0.f;
        }
        put4((T*)s.out + to, of * size, y);
      }
    }
  }

  for (int64_t tile = tile_end; tile < tile1; ++tile) {
    if (kMode == kLocal || (kMode == kBack && !gate_grad)) continue;
    const int64_t row = (b * s.tokens + tile * K) * s.channels + c_first;
    const int inside = (int)min(s.tokens - tile * K, (int64_t)K);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (!mine || et + i * kStep >= inside) continue;
      const int64_t to = row + (int64_t)(i * kStep) * s.channels;
      if (kMode == kOut && s.raw) put4(s.raw + to, of * 4, zero);
      put4((T*)(kMode == kOut ? s.out : s.dz) + to, of * size, zero);
    }
  }
  if (kMode == kOut) {
    if (live && s.state_out && chunk == s.chunks - 1)
      *(States*)(s.state_out + (b * s.channels + c) * N + j * S) = h;
    return;
  }
  total += from_lane<0xB1>(total);
  total += from_lane<0x4E>(total);
  if (!live) return;
  const int64_t at = (b * s.chunks + chunk) * s.channels + c;
  *(States*)(s.carry + at * N + j * S) = h;
  if (j == 0) s.steps[at] = total;
}

// The second pass: from each chunk's own states and the sum of its steps to what enters it, in place; forward from the
// given state (or zeros), backward from the gradient of the last one.  A block takes 256 states one chunk after
// another or, where they are few, 32 by eight runs of chunks: each run's own states and decay first, then from what the
// runs before it make of `first` (384 channels of 8 states, 251 chunks: 32 -> 8.5 us; 98304 states, 16 chunks: 5.5 ->
// 11.5, so not there).
// A state after a run of tokens that decays by 2^x and adds `own`.  The power is taken in halves: a growing state (A > 0)
// may be finite behind a run whose own power is not, and one that is zero stays so.
__device__ __forceinline__ float after_run(float state, float x, float own) {
  const float half = __builtin_amdgcn_exp2f(0.5f * x);
  return state == 0.f ? own : state * half * half + own;
}
template <bool kReverse, int kRuns>
__global__ __launch_bounds__(256) void scan_carry_kernel(Scan s, const float* first, float* last) {
  constexpr int kAhead = 8, kColumns = 256 / kRuns;
  __shared__ float decay[kRuns][kColumns], state[kRuns][kColumns];
  const int col = threadIdx.x % kColumns, run = threadIdx.x / kColumns;
  const int64_t item = (int64_t)block_index() * kColumns + col, per = (int64_t)s.channels * s.states;  // a multiple of 64
  if (item >= s.batch * per) return;  // whole blocks leave where there are runs
  const int64_t b = item / per, cn = item - b * per, c = cn / s.states;
  const float A2 = s.A[cn] * kLog2e;
  const int64_t each = (s.chunks + kRuns - 1) / kRuns, k_first = run * each, k_last = min(k_first + each, s.chunks);
  float own[kAhead], d[kAhead];
  auto at = [&](int64_t k) { return b * s.chunks + (kReverse ? s.chunks - 1 - k : k); };
  auto load = [&](int64_t k0) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const bool there = k0 + i < k_last;
      own[i] = there ? s.carry[at(k0 + i) * per + cn] : 0.f;
      d[i] = there ? s.steps[at(k0 + i) * s.channels + c] : 0.f;  // no step: the state passes
    }
  };
  float carry = first ? first[item] : 0.f;
  if (kRuns > 1) {
    float total = 0.f, mine = 0.f;
    for (int64_t k0 = k_first; k0 < k_last; k0 += kAhead) {
      load(k0);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        mine = after_run(mine, A2 * d[i], own[i]);
        total += d[i];
      }
    }
    decay[run][col] = A2 * total;
    state[run][col] = mine;
    __syncthreads();
    for (int i = 0; i < run; ++i) carry = after_run(carry, decay[i][col], state[i][col]);
  }
  for (int64_t k0 = k_first; k0 < k_last; k0 += kAhead) {
    if (kRuns == 1 || each > kAhead) load(k0);  // else they are still there
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (k0 + i >= k_last) break;
      s.carry[at(k0 + i) * per + cn] = carry;
      carry = after_run(carry, A2 * d[i], own[i]);
    }
  }
  if (last && run == kRuns - 1) last[item] = carry;
}

// One token: four states a thread (64 x 1536 channels of 16 states: 5.1 us; a walk would take 17.6).
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

// LDS of a block in floats: four parts of a slice for each wave, or the tile's sums that meet there; the maps; and what
// is kept for the span, of at most grad_span() channels.
constexpr int kGradStage = 4 * 4 * kSlice * kGradRow > 256 * KG ? 4 * 4 * kSlice * kGradRow : 256 * KG;
constexpr int grad_span(int states) {
  constexpr int unit = 4 * kSlice;
  return kMaxSpan / states < unit ? unit : kMaxSpan / states / unit * unit;
}
constexpr int grad_span_floats(int states) { return 2 * states + 4; }  // of a channel
constexpr int grad_lds_bytes(int states) {
  return (kGradStage + 2 * (states < 16 ? 16 : states) * kGradRow + grad_span(states) * grad_span_floats(states)) * 4;
}
static_assert(grad_lds_bytes(8) <= 65536 && grad_lds_bytes(16) <= 65536 && grad_lds_bytes(32) <= 65536 &&
                  grad_lds_bytes(64) <= 65536,
              "a launch gets no more LDS than this");
// Blocks that the card holds: three a compute unit by their registers; by their LDS too, but two of 64 states (64512 bytes).
constexpr int64_t grad_round(int states) {
  return 256 * (163840 / grad_lds_bytes(states) < 3 ? 163840 / grad_lds_bytes(states) : 3);
}

// A block takes a span of a group's channels and a range of tiles; its waves take slices of 16 channels in turn, each in
// its own part of LDS, and wait for each other only at a tile's ends.  The range's tiles go from the last to the first, X
// handed on in LDS.  A lane has one state (of 8 states every second lane none) and, pass by pass, channel after channel:
// the sums dB, dC of its state stay in its registers over a tile, h and a of a channel over its 16 tokens.  dA, dD and the
// bias's sums stay in LDS over the range.  Three waves a SIMD, at which a few registers are spilled (bf16 2 at 8 and 16
// states, 12 at 32; fp32 10 and 17): 159 us at 4 x 2048 x 1536 x 16; two, without spills, 189, four, with the sums spilled,
// 263.  Of 64 states the LDS holds two; the 28 (bf16 20) registers that three would have to spill are spilled there too.
template <typename T, int N>
__global__ __launch_bounds__(256, 3) void scan_bwd_kernel(Scan s) {
  constexpr int NP = N < 16 ? 16 : N, kSlots = 64 / NP, kPasses = kSlice / kSlots, R = kGradRow;
  constexpr int kPart = kSlice * R;
  __shared__ __align__(16) float lds[kGradStage];
  __shared__ __align__(16) float sB[NP * R], sC[NP * R];
  extern __shared__ __align__(16) float span_sums[];  // X [span][N], dA [span][N], dD, dbias, D and the bias [span]
  float *aX = span_sums, *aA = aX + s.span * N, *aD = aA + s.span * N, *ab = aD + s.span, *skips = ab + s.span;
  float* biases = skips + s.span;
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
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // uniform, as what is worked out of it
  const int lane = lane_id(), n = lane % NP, slot = lane / NP, r = lane & 15;
  const bool held = n < N;
  // d, d u, dy and the sums G B of a slice; the sums A X h take the place of the d u that they have used
  float *sd = lds + wave * 4 * kPart, *sv = sd + kPart, *sy = sv + kPart, *s1 = sy + kPart, *s2 = sv;
  const float* x_at = s.x_in + ((b * s.ranges + range) * s.channels + c_first) * N;
  for (int i = threadIdx.x; i < s.span * N; i += 256) aX[i] = i < (c_end - c_first) * N ? x_at[i] : 0.f;
  for (int i = threadIdx.x; i < s.span * (N + 2); i += 256) aA[i] = 0.f;
  for (int i = threadIdx.x; i < s.span; i += 256) {
    skips[i] = s.D && c_first + i < c_end ? s.D[c_first + i] : 0.f;
    biases[i] = s.dt_bias && c_first + i < c_end ? s.dt_bias[c_first + i] : 0.f;
  }

  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const int e = lane % (kSlice / 4) * 4, et = lane / (kSlice / 4);  // a lane's element of a slice
  const uint32_t size = sizeof(T), u_of = (et * (uint32_t)s.u.st + e) * size, dt_of = (et * (uint32_t)s.dt.st + e) * size;
  const uint32_t z_of = (et * (uint32_t)s.z.st + e) * size, of = et * (uint32_t)s.channels + e;
  const int64_t tile0 = (int64_t)range * s.range_tiles * (K / KG);
  int64_t tile1 = min(tile0 + (int64_t)s.range_tiles * (K / KG), s.grad_tiles);
  const int64_t map_row = (s.whole ? 0 : (int64_t)span * s.batch + b) * s.tokens + (s.whole ? b * s.tokens : 0);
  for (; tile1 > tile0 && (tile1 - 1) * KG >= length; --tile1) {  // nothing there depends on anything
    const int64_t token = (tile1 - 1) * KG, first = b * s.tokens + token;
    const int inside = (int)min(s.tokens - token, (int64_t)KG);
    for (int cc = again(c_first + wave * kSlice + e); et < inside && cc < c_end; cc += 4 * kSlice) {
      if (s.du) store4((T*)s.du + (first + et) * s.channels + cc, zero);
      if (s.ddt) store4((T*)s.ddt + (first + et) * s.channels + cc, zero);
    }
    for (int i = again(threadIdx.x); i < inside * N; i += 256) {
      const int64_t at = ((map_row + token + i / N) * s.groups + group) * N + i % N;
      if (!s.whole) s.dB[at] = 0.f, s.dC[at] = 0.f;
      if (s.whole && s.dB_out) ((T*)s.dB_out)[at] = (T)0.f;
      if (s.whole && s.dC_out) ((T*)s.dC_out)[at] = (T)0.f;
    }
  }

  // a slice's elements, and a pass's A and entering h, are asked for a slice and a pass before, a tile's maps and its
  // first slice before the tile behind it is summed up
  Four<T> u, x, dy, z;
  auto ask_slice = [&](int64_t tile_of, int c_of) {
    const int64_t tile = uniform((int)tile_of);
    const int c0 = uniform(c_of);
    const bool there = c0 + e < c_end && et < length - tile * KG;
    u = four((const T*)s.u.p + b * s.u.sb + tile * KG * s.u.st + c0, u_of, there);
    x = four((const T*)s.dt.p + b * s.dt.sb + tile * KG * s.dt.st + c0, dt_of, there);
    dy = four((const T*)s.dout + (b * s.tokens + tile * KG) * s.channels + c0, of * size, there);
    z = four((const T*)s.z.p + b * s.z.sb + tile * KG * s.z.st + c0, z_of, there && s.z.p);
  };
  float nA = 0.f, nh = 0.f;
  const uint32_t state_of = slot * N + n;
  auto ask = [&](int64_t tile_of, int c_of) {  // of the channels from c_of on, a slot each
    const int64_t tile = uniform((int)tile_of);
    const int c0 = uniform(c_of);
    const bool live = c0 + slot < c_end && held;
    const float* A = s.A + (int64_t)c0 * N;
    const float* h = s.h_in + ((b * s.grad_tiles + tile) * s.channels + c0) * N;
    nA = nh = 0.f;
    if (live) nA = A[state_of], nh = h[state_of];
  };
  constexpr int kMaps = KG * NP / 256;
  T map_B[kMaps], map_C[kMaps];
  const uint32_t map_m = threadIdx.x % NP, map_t = threadIdx.x / NP;
  auto ask_tile = [&](int64_t tile_of) {
    const int64_t tile = uniform((int)tile_of);
    const T* B = (const T*)s.B.p + b * s.B.sb + tile * KG * s.B.st + group * s.B.sg;
    const T* C = (const T*)s.C.p + b * s.C.sb + tile * KG * s.C.st + group * s.C.sg;
#pragma unroll
    for (int i = 0; i < kMaps; ++i) {
      const uint32_t t = map_t + i * (256 / NP);
      const bool there = t < length - tile * KG && map_m < N;
      map_B[i] = map_C[i] = (T)0.f;
      if (there) map_B[i] = B[t * (uint32_t)s.B.st + map_m], map_C[i] = C[t * (uint32_t)s.C.st + map_m];
    }
    ask_slice(tile, c_first + wave * kSlice);
    ask(tile, c_first + wave * kSlice);
  };
  if (tile1 > tile0) ask_tile(tile1 - 1);
  for (int64_t tile = tile1 - 1; tile >= tile0; --tile) {
    const int left = (int)min(length - tile * KG, (int64_t)KG), inside = (int)min(s.tokens - tile * KG, (int64_t)KG);
    const int64_t row = (b * s.tokens + tile * KG) * s.channels;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMaps; ++i) {
      const int at = map_m * R + map_t + i * (256 / NP);
      sB[at] = (float)map_B[i];
      sC[at] = (float)map_C[i];
    }
    __syncthreads();
    float accB[KG], accC[KG];
#pragma unroll
    for (int t = 0; t < KG; ++t) accB[t] = accC[t] = 0.f;
    for (int c_of = c_first + wave * kSlice; c_of < c_end; c_of += 4 * kSlice) {
      const int c0 = uniform(c_of);
      const bool mine = c0 + e < c_end, there = mine && et < left;
      const f32x4 bias = *(const f32x4*)(biases + c0 - c_first + e);
      const Four<T> u_kept = u, x_kept = x;
      {
        // a token that is not there has u, dy and z zero, and takes no step
        f32x4 d = x.wide() + bias, y = dy.wide();
        const f32x4 uw = u.wide(), zw = z.wide();
        if (s.softplus) {
#pragma unroll
          for (int q = 0; q < 4; ++q) d[q] = step_of(d[q]);
        }
        d = d * (there ? 1.f : 0.f);
        if (s.z.p) {
#pragma unroll
          for (int q = 0; q < 4; ++q) y[q] *= silu_f(zw[q]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          sd[(e + q) * R + et] = d[q];
          sv[(e + q) * R + et] = d[q] * uw[q];
          sy[(e + q) * R + et] = y[q];
        }
      }
      wave_fence();
      for (int pass = 0; pass < kPasses; ++pass) {
        const int cl = pass * kSlots + slot, c = c0 + cl;
        const bool live = c < c_end && held;
        float A = nA, h0 = nh;
        asm volatile("" : "+v"(A), "+v"(h0));
        const float A2 = A * kLog2e;
        float X = live ? aX[(c - c_first) * N + n] : 0.f, dA = 0.f;
        // behind the use of what was asked for before: loads come back in their order, and a pass waits for all of them
        __builtin_amdgcn_sched_barrier(0);
        if (pass == 0) ask_slice(tile, c0 + 4 * kSlice);
        ask(tile, pass + 1 < kPasses ? c0 + (pass + 1) * kSlots : c0 + 4 * kSlice);
        // d as an operand from the lanes of a row in the exponent; in multiply-adds, which take none, from LDS
        const float dl = sd[cl * R + r];
        float h[KG], a[KG], last = h0;
        unrolled<KG / 4>([&](auto quad) {
          constexpr int t0 = decltype(quad)::value * 4;
          const f32x4 v = *(const f32x4*)(sv + cl * R + t0), m = *(const f32x4*)(sB + n * R + t0);
          unrolled<4>([&](auto index) {
            constexpr int q = decltype(index)::value, t = t0 + q;
            a[t] = __builtin_amdgcn_exp2f(from_row<t>(dl) * A2);
            h[t] = last = __builtin_fmaf(v[q], m[q], a[t] * last);
          });
          __builtin_amdgcn_sched_barrier(0);
        });
        RowSum sum1, sum2;
        unrolled<KG / 4>([&](auto quad) {
          constexpr int t0 = KG - 4 - decltype(quad)::value * 4;
          const f32x4 m = *(const f32x4*)(sB + n * R + t0), o = *(const f32x4*)(sC + n * R + t0);
          const f32x4 d = *(const f32x4*)(sd + cl * R + t0), v = *(const f32x4*)(sv + cl * R + t0);
          const f32x4 y = *(const f32x4*)(sy + cl * R + t0);
          unrolled<4>([&](auto index) {
            constexpr int q = 3 - decltype(index)::value, t = t0 + q;
            const float G = __builtin_fmaf(y[q], o[q], X);
            accC[t] = __builtin_fmaf(y[q], h[t], accC[t]);
            accB[t] = __builtin_fmaf(v[q], G, accB[t]);
            asm volatile("" : "+v"(accB[t]), "+v"(accC[t]));  // here, not sunk behind the pass with all that they need
            X = a[t] * G;
            const float back = X * (t ? h[t ? t - 1 : 0] : h0);
            dA = __builtin_fmaf(d[q], back, dA);
            sum1.add<15 - t>(G * m[q], lane);
            sum2.add<15 - t>(A * back, lane);
          });
          __builtin_amdgcn_sched_barrier(0);
        });
        float r1 = sum1.held[3], r2 = sum2.held[3];
        if (N >= 32) r1 += xor16(r1), r2 += xor16(r2);
        if (N == 64) r1 = xor32_sum(r1), r2 = xor32_sum(r2);
        if (N <= 16 || n < 16) {
          s1[cl * R + 15 - rev4(r)] = r1;
          s2[cl * R + 15 - rev4(r)] = r2;
        }
        if (live) {
          aA[(c - c_first) * N + n] += dA;
          aX[(c - c_first) * N + n] = X;
        }
      }
      wave_fence();
      {
        const f32x4 skip = *(const f32x4*)(skips + c0 - c_first + e);
        f32x4 du, ddt;
        const f32x4 uw = u_kept.wide(), xw = x_kept.wide() + bias;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int at = (e + q) * R + et;
          const float g = s1[at], y = sy[at];
          du[q] = there ? sd[at] * g + skip[q] * y : 0.f;
          ddt[q] = there ? uw[q] * g + s2[at] : 0.f;
          s1[at] = there ? y * uw[q] : 0.f;
        }
        if (s.softplus) {
#pragma unroll
          for (int q = 0; q < 4; ++q) ddt[q] *= sigmoid_f(xw[q]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) s2[(e + q) * R + et] = ddt[q];
        if (mine && et < inside) {
          if (s.du) put4((T*)s.du + row + c0, of * size, du);
          if (s.ddt) put4((T*)s.ddt + row + c0, of * size, ddt);
        }
      }
      wave_fence();
      // sums over the tile's tokens: two lanes a channel, 8 tokens each; dD by the lower half of the wave, the bias's by
      // the upper
      {
        const int cl = (lane & 31) >> 1;
        const float* from = (lane & 32 ? s2 : s1) + cl * R + 8 * (lane & 1);
        const f32x4 v = *(const f32x4*)from + *(const f32x4*)(from + 4);
        float total = (v[0] + v[1]) + (v[2] + v[3]);
        total += from_lane<0xB1>(total);
        if (!(lane & 1) && c0 + cl < c_end) (lane & 32 ? ab : aD)[c0 - c_first + cl] += total;
      }
      wave_fence();
    }
    if (tile > tile0) ask_tile(tile - 1);
    // the slots' and waves' sums of dB, then dC
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int t = 0; t < KG; ++t) lds[t * 256 + threadIdx.x] = which ? accC[t] : accB[t];
      __syncthreads();
      for (int i = again(threadIdx.x); i < inside * N; i += 256) {
        const float* from = lds + i / N * 256 + i % N;
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < 4 * kSlots; ++k) v += from[k * NP];
        const int64_t at = ((map_row + tile * KG + i / N) * s.groups + group) * N + i % N;
        if (!s.whole)
          (which ? s.dC : s.dB)[at] = v;
        else if (which ? s.dC_out : s.dB_out)
          ((T*)(which ? s.dC_out : s.dB_out))[at] = (T)v;
      }
    }
  }
  __syncthreads();
  const int64_t part = b * s.ranges + range;
  for (int i = again(threadIdx.x); i < (c_end - c_first) * N; i += 256) s.dA[(part * s.channels + c_first) * N + i] = aA[i];
  for (int i = again(threadIdx.x); i < c_end - c_first; i += 256) {
    s.dD[part * s.channels + c_first + i] = aD[i];
    s.dbias[part * s.channels + c_first + i] = ab[i];
  }
}

// Sums of partial rows, 64 columns by 16 slices of the rows a block: out[i] = sum over r of from[r * columns + i].
struct RowSums {
  const float* from[5];
  void* out[5];
  int64_t columns[5], rows[5];  // columns are multiples of 4
  int bf16_out[5];
};
__global__ __launch_bounds__(256) void scan_sums_kernel(RowSums s) {
  __shared__ f32x4 lds[16][17];
  const int which = blockIdx.y, col = threadIdx.x % 16, slice = threadIdx.x / 16;
  if (!s.out[which]) return;
  const int64_t columns = s.columns[which], rows = s.rows[which];
  for (int64_t first = (int64_t)blockIdx.x * 64; first < columns; first += (int64_t)gridDim.x * 64) {
    const int64_t i = first + 4 * col;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (i < columns) {
#pragma unroll 4
      for (int64_t r = slice; r < rows; r += 16) v += *(const f32x4*)(s.from[which] + r * columns + i);
    }
    __syncthreads();
    lds[slice][col] = v;
    __syncthreads();
    if (slice || i >= columns) continue;
#pragma unroll
    for (int k = 1; k < 16; ++k) v += lds[k][col];
    if (s.bf16_out[which])
      store4((bf16*)s.out[which] + i, v);
    else
      store4((float*)s.out[which] + i, v);
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

// Chunks of a forward call.  One where its blocks keep the card busy (a round of them takes as long with 288 as with 480;
// us at 1536 channels of 16 states, 512 tokens, one chunk against several: 384 blocks 96 and 104, 480 97 and 139, 288 97
// and 87) or where there is little to walk (96 tokens: 17 and 19; 128: 21 and 20).  Else about three rounds of the four
// blocks that a compute unit holds: 2 x 4096 tokens take 111 with three or four rounds, 118 with two, 115 to 122 with one.
// Two tiles a chunk at least, as the carry is read and written per chunk (2 x 4096: 102, with one 107; 16001 x 384 of 8
// states: 47 and 55), but one where all tiles are a round's blocks (1 x 512 x 768: 23 with two, 16 with one; 1 x 2048: 31
// and 27; at 1536 blocks equal).  Longer calls draw the same line, with a few per cent lost on it (one chunk against
// several: 8192 tokens, 384 blocks 1483 and 1426, 480 1486 and 1851, 768 1938 and 2877; 2048 tokens 375 and 368, 375 and 483,
// 483 and 722).
struct Chunks {
  int64_t chunks, tiles;  // tiles of a chunk
};
Chunks plan_chunks(int64_t batch, int64_t tokens, int64_t channels, int64_t states, int64_t groups) {
  const int64_t tiles = (tokens + K - 1) / K, per = 256 / walk_lanes((int)states);
  const int64_t blocks = batch * groups * ((channels / groups + per - 1) / per);
  if (blocks >= 384 || tiles <= 3) return {1, tiles};
  const int64_t most = blocks * tiles <= kRound ? tiles : tiles / 2;
  int64_t chunks = (3 * kRound + blocks - 1) / blocks;
  if (chunks > most) chunks = most;
  const int64_t each = (tiles + chunks - 1) / chunks;
  return {(tiles + each - 1) / each, each};
}

struct Spans {
  int64_t span, spans, ranges, range_tiles, whole;
};
// Spans of a group's channels and ranges of tiles of the gradient's blocks: two tiles (of 32) a range, for half the states
// to carry, where that still is a round of blocks (both ways, us at 2048 tokens x 1536 channels of 16 states with two and
// one: batch 8 655 and 690, 2 204 and 211, 1 142 and 125, as a wave then waits for every tile; with four 338 for 325;
// backward, 512 channels of 64 states in 8 groups, where a round is 512 blocks: 1024 of them 160 and 170, 768 151 and 142).
Spans plan_spans(int64_t batch, int64_t tokens, int64_t channels, int64_t states, int64_t groups) {
  const int64_t tiles = (tokens + K - 1) / K, group = channels / groups, unit = 4 * kSlice;
  const int64_t most = grad_span((int)states);
  Spans p;
  p.spans = (group + most - 1) / most;
  p.span = ((group + p.spans - 1) / p.spans + unit - 1) / unit * unit;
  p.spans = (group + p.span - 1) / p.span;
  const int64_t m = batch * groups * p.spans * tiles >= 2 * grad_round((int)states) ? 2 : 1, ranges = (tiles + m - 1) / m;
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
  for (int i : {1, 3, 5, 7, 10})
    BMX_REQUIRE(strides[i] >= 0 && strides[i] < (1 << 25), "selective_scan: a token's stride must be below 2^25");
  s.u = {u, strides[0], strides[1], 0}, s.dt = {dt, strides[2], strides[3], 0}, s.z = {z, strides[4], strides[5], 0};
  s.B = {B, strides[6], strides[7], strides[8]}, s.C = {C, strides[9], strides[10], strides[11]};
  s.A = A, s.D = D, s.dt_bias = dt_bias, s.lengths = lengths, s.lengths64 = lengths64, s.softplus = softplus != 0;
  s.batch = shape[0], s.tokens = shape[1], s.channels = (int)channels, s.states = (int)states, s.groups = (int)groups;
  s.group_channels = (int)(channels / groups), s.tiles = (s.tokens + K - 1) / K;
  s.grad_tiles = (s.tokens + KG - 1) / KG;
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
  BMX_REQUIRE(aligned(16, {s.A, s.D, s.dt_bias, s.state, s.state_out, s.raw, s.saved}),
              "selective_scan: fp32 tensors must be 16-byte aligned");
  return BMX_OK;
}

template <typename T, int kMode>
int walk(Scan s, hipStream_t stream) {
  int rc = BMX_OK;
  with_states(s.states, [&](auto n) {
    constexpr int N = decltype(n)::value, L = walk_lanes(N);
    s.cblocks = (s.group_channels + 256 / L - 1) / (256 / L);
    s.blocks = s.batch * s.chunks * s.groups * s.cblocks;
    if (s.blocks >= (1ll << 31) - 32) {
      rc = set_error(BMX_EINVAL, "selective_scan: too many rows");
      return;
    }
    scan_walk_kernel<T, N, L, kMode><<<fold_grid((s.blocks + 31) / 32 * 32, 256), 256, 0, stream>>>(s);
  });
  return rc ? rc : check_launch("selective_scan");
}

template <bool kReverse>
int carry(const Scan& s, const float* first, float* last, hipStream_t stream) {
  const int64_t states = s.batch * s.channels * s.states;
  BMX_REQUIRE(states / 32 < (1ll << 31), "selective_scan: too many states");
  if (states >= 65536)
    scan_carry_kernel<kReverse, 1><<<fold_grid((states + 255) / 256, 256), 256, 0, stream>>>(s, first, last);
  else
    scan_carry_kernel<kReverse, 8><<<fold_grid(states / 32, 256), 256, 0, stream>>>(s, first, last);
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
    scan_bwd_kernel<T, N><<<fold_grid(s.blocks, 256), 256, s.span * grad_span_floats(N) * sizeof(float), stream>>>(s);
  });
  return check_launch("selective_scan_bwd");
}

// Floats of the gradient's workspace, part by part.
struct BackSpace {
  int64_t carry, steps, maps, dA, dD;
  BackSpace(int64_t batch, int64_t tokens, int64_t channels, int64_t states, int64_t groups, const Spans& p) {
    const int64_t parts = batch * p.ranges;
    carry = parts * channels * states, steps = parts * channels;
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
  return (size_t)(batch * ((tokens + KG - 1) / KG) * channels * states) * sizeof(float);
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
  BMX_REQUIRE(aligned(16, {saved, raw, dout, du, ddt, dz, dA, dB, dC, dD, ddt_bias}),
              "selective_scan: tensors must be 16-byte aligned");
  const Spans p = plan_spans(s.batch, s.tokens, s.channels, s.states, s.groups);
  const BackSpace space(s.batch, s.tokens, s.channels, s.states, s.groups, p);
  BMX_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= (size_t)space.floats() * sizeof(float),
              "selective_scan_bwd: workspace too small or not 16-byte aligned");
  s.dout = dout, s.h_in = saved, s.raw = const_cast<float*>(raw), s.du = du, s.ddt = ddt, s.dz = dz;
  s.carry = (float*)workspace, s.steps = s.carry + space.carry, s.x_in = s.carry;
  s.dB = s.steps + space.steps, s.dC = s.dB + space.maps, s.dB_out = dB, s.dC_out = dC;
  s.dA = s.dC + space.maps, s.dD = s.dA + space.dA, s.dbias = s.dD + space.dD;
  s.chunks = p.ranges, s.chunk_tiles = p.range_tiles;
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
  const int64_t blocks = (columns + 63) / 64;
  scan_sums_kernel<<<dim3((unsigned)(blocks < 16384 ? blocks : 16384), 5), 256, 0, hs>>>(sums);
  return check_launch("selective_scan_bwd sums");
}
