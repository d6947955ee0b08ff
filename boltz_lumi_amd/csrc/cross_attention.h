// Tiles and operands shared by the cross attention kernels (cross_attention.hip,
// cross_attention_bwd.hip).
//
// Query rows of the `group` heads that share one key / value head are one list: row r of
// key head c is query r % m of head c * group + r / m, so a key tile serves all of them and a
// single query of a shared head still fills MFMA columns.
//
// Operand layout (v_mfma_f32_32x32x16_bf16, or v_mfma_f32_32x32x2f32 for fp32; lane l, half
// h = l / 32): a product tile holds column l % 32 and, in register r, row 8 (r / 4) + 4 h + r % 4. A
// logits tile S^T (keys x queries) is then itself the B operand of the next product over its keys:
// registers 8 t .. 8 t + 7 are the 16 keys of bf16 step t, and register r the keys of fp32 step r.
#pragma once

#include "bmx_common.h"

namespace bmx {

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaskChunk = 4096;  // keys whose mask words are in LDS at a time

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct CrossArgs {
  const void *q, *k, *v, *bias;
  const uint8_t* mask;
  int64_t sq[3], sk[3], sv[3];  // batch, token, head strides
  int64_t sb[3], smask;         // bias: batch, head, query strides; keys dense
  int64_t batch, m, n;
  int heads, kv_heads, group, dim, rows;  // rows = group * m
  float scale;
  void *out, *out_lo;
  float2* stats;  // [batch][heads][m]: row maximum of the logits and log2 of the sum of exp(logit - maximum)
  // work split
  int row_blocks, splits;
  int64_t split_keys;
  float* part_o;   // [split][batch * kv_heads][rows][dim] sums before the division
  float2* part_ml;  // [split][batch * kv_heads][rows] maximum and sum
  // backward
  const void* dout;
  float* delta;
  void *dq, *dk, *dv, *dbias;
  int64_t sdb[3];  // dbias: batch (0: shared), head (0: shared), query strides
};

// Blocks go round the XCDs in turn: block b of `total` becomes a position such that each XCD
// works through consecutive ones, whose keys then stay in its own L2.
__device__ __forceinline__ int64_t xcd_position(int64_t b, int64_t total) {
  const int64_t per = total / 8, whole = per * 8;
  return b < whole ? (b % 8) * per + b / 8 : b;
}

// ---- LDS tiles -----------------------------------------------------------
// Rows of DP elements in 16-byte chunks, chunk c of row r at c ^ twist(r). Two kinds of read meet: 16 rows at one
// chunk (operands with the row in the lane) and, for bf16, four rows r .. r + 3 (r % 4 == 0) at four
// chunks (the transposing read); the twist puts both on different banks.
template <typename T, int DP>
struct Tile {
  static constexpr int kElems = 16 / sizeof(T);           // elements of a chunk
  static constexpr int kChunks = DP / kElems;             // chunks with data
  static constexpr int kRow = kChunks <= 4 ? 4 : kChunks <= 8 ? 8 : kChunks <= 16 ? 16 : 32;  // chunks of a row
  static constexpr int kRowBytes = kRow * 16;

  static __device__ __forceinline__ int twist(int r) {
    if (kRow == 4) return (r >> 2) & 3;
    if (kRow == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    return ((r & 3) << 2) | ((r >> 2) & 3);
  }
  static __device__ __forceinline__ int at(int r, int c) { return r * kRowBytes + ((c ^ twist(r)) << 4); }
};

// Operand with the row in the lane, from global memory: 16 bytes per step, zeros past dim.
template <typename T, int DP>
struct RowOperand {
  static constexpr int kSteps = Tile<T, DP>::kChunks / 2;  // each half of the wave takes every other chunk
  u32x4 c[kSteps];

  __device__ __forceinline__ void load(const T* row, int dim, int half) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = (2 * s + half) * Tile<T, DP>::kElems;
      const u32x4 x = *(const u32x4*)(row + (d < dim ? d : 0));
      c[s] = d < dim ? x : u32x4{0, 0, 0, 0};
    }
  }
};

__device__ __forceinline__ f32x16 mfma_step(const bf16*, u32x4 a, u32x4 b, f32x16 acc) {
  return mfma32(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc);
}
__device__ __forceinline__ f32x16 mfma_step(const float*, u32x4 a, u32x4 b, f32x16 acc) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), acc, 0, 0, 0);
  return acc;
}

// acc += tile rows row0 .. row0 + 31 (A) times the operand's columns (B), over the channels.
template <typename T, int DP>
__device__ __forceinline__ f32x16 product(const char* tile, int row0, const RowOperand<T, DP>& b, f32x16 acc) {
  const int r = row0 + (lane_id() & 31), h = lane_id() >> 5;
#pragma unroll
  for (int s = 0; s < RowOperand<T, DP>::kSteps; ++s)
    acc = mfma_step((const T*)nullptr, *(const u32x4*)(tile + Tile<T, DP>::at(r, 2 * s + h)), b.c[s], acc);
  return acc;
}

// A 32 x 32 product tile as the B operand of a product over its rows.
template <typename T>
struct Weights;
template <>
struct Weights<bf16> {
  bf16x8 v[2];
  __device__ __forceinline__ void set(const f32x16& p) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[t][e] = (bf16)p[8 * t + e];
  }
  // Sum of the rounded values: what the product over them adds up.
  __device__ __forceinline__ float sum(float acc) const {
    const bf16x2 one = {(bf16)1.f, (bf16)1.f};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 8; e += 2)
        acc = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{v[t][e], v[t][e + 1]}, one, acc, false);
    return acc;
  }
};
template <>
struct Weights<float> {
  f32x16 v;
  __device__ __forceinline__ void set(const f32x16& p) { v = p; }
  __device__ __forceinline__ float sum(float acc) const {
#pragma unroll
    for (int r = 0; r < 16; ++r) acc += v[r];
    return acc;
  }
};

// acc[dt] += (tile rows row0 .. row0 + 31)^T (channels 32 dt .. as rows) times the weights, over those rows.
template <int DP>
__device__ __forceinline__ void transposed_product(const char* tile, int row0, const Weights<bf16>& w,
                                                   f32x16 (&acc)[DP / 32]) {
  const int l = lane_id(), h = l >> 5, i = l & 15;
  const int chunk = 2 * ((l >> 4) & 1) + ((i & 3) >> 1), byte = 8 * (i & 1);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int r = row0 + 16 * t + 4 * h + (i >> 2);
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) {
      union {
        s16x4 half[2];
        bf16x8 all;
      } a;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        a.half[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(tile + Tile<bf16, DP>::at(r + 8 * u, 4 * dt + chunk) + byte));
      acc[dt] = mfma32(a.all, w.v[t], acc[dt]);
    }
  }
}
template <int DP>
__device__ __forceinline__ void transposed_product(const char* tile, int row0, const Weights<float>& w,
                                                   f32x16 (&acc)[DP / 32]) {
  const int l = lane_id(), h = l >> 5, i = l & 31;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = row0 + 8 * (r >> 2) + 4 * h + (r & 3);
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) {
      const float a = *(const float*)(tile + Tile<float, DP>::at(row, 8 * dt + (i >> 2)) + 4 * (i & 3));
      acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, w.v[r], acc[dt], 0, 0, 0);
    }
  }
}

// ---- staging -------------------------------------------------------------
// ROWS rows of a [.., tokens, .., dim] tensor through registers into an LDS tile, by THREADS threads.
template <typename T, int DP, int ROWS, int THREADS>
struct Stage {
  using L = Tile<T, DP>;
  static constexpr int kCount = (ROWS * L::kChunks + THREADS - 1) / THREADS;
  u32x4 v[kCount];

  // row(r): pointer to row r, always readable; channels past dim read the row's first ones.
  template <typename Row>
  __device__ __forceinline__ void load(int t, int dim, Row row) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int at = t + i * THREADS, r = at / L::kChunks, d = (at % L::kChunks) * L::kElems;
      if ((ROWS * L::kChunks) % THREADS == 0 || r < ROWS) v[i] = *(const u32x4*)(row(r) + (d < dim ? d : 0));
    }
  }
  // live(r): rows that hold data; the others, and channels past dim, are stored as zeros.
  template <typename Live>
  __device__ __forceinline__ void store(int t, int dim, char* tile, Live live) const {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int at = t + i * THREADS, r = at / L::kChunks, c = at % L::kChunks;
      if ((ROWS * L::kChunks) % THREADS != 0 && r >= ROWS) continue;
      const bool ok = c * L::kElems < dim && live(r);
      *(u32x4*)(tile + L::at(r, c)) = ok ? v[i] : u32x4{0, 0, 0, 0};
    }
  }
};

// Orders a wave's LDS writes and its other lanes' reads where no barrier does: the LDS serves a wave in order, so
// only the compiler has to keep them.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// ---- key mask ------------------------------------------------------------
// Bit words of a chunk of keys: bit j of word w is key c0 + 64 w + j present (inside the mask and below end).
// All threads call fill (two barriers); key c0 is a multiple of 64.
struct KeyWords {
  uint64_t* words;  // LDS [kMaskChunk / 64]
  const uint8_t* mask;
  int64_t c0, end;

  __device__ __forceinline__ void fill(int64_t first, int64_t stop) {
    c0 = first, end = stop;
    if (!mask) return;
    __syncthreads();
    const int64_t left = min(stop - first, (int64_t)kMaskChunk);
    for (int w = threadIdx.x >> 6; 64 * w < left; w += blockDim.x >> 6) {
      const int64_t key = first + 64 * w + lane_id();
      const bool on = key < stop && mask[key < stop ? key : stop - 1] != 0;
      const uint64_t bits = __ballot(on);
      if (lane_id() == 0) words[w] = bits;
    }
    __syncthreads();
  }
  // Presence of the `count` (32 or 64) keys from `key` on, the same in every lane; key - c0 a multiple of count.
  __device__ __forceinline__ uint64_t bits(int64_t key, int count) const {
    const uint64_t all = count == 64 ? ~0ull : 0xffffffffull;
    const int64_t left = end - key;
    if (left <= 0) return 0;
    uint64_t b = left >= count ? all : (1ull << left) - 1;
    if (mask) {
      const int at = (int)(key - c0);
      const uint64_t w = words[at >> 6] >> (at & 63);
      b &= (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)w) |
           (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(w >> 32)) << 32;
    }
    return b;
  }
};

// ---- bias ----------------------------------------------------------------
// Four consecutive bias values at any element alignment.
typedef uint32_t u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_at2 __attribute__((ext_vector_type(2), aligned(2)));
__device__ __forceinline__ f32x4 bias4(const float* p) { return __builtin_bit_cast(f32x4, (u32x4) * (const u32x4_at4*)p); }
__device__ __forceinline__ f32x4 bias4(const bf16* p) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  const bf16x4 v = __builtin_bit_cast(bf16x4, (u32x2) * (const u32x2_at2*)p);
  return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
}

// Bias of the lane's query at the 16 keys of a logits tile from key `key` on, in register order; keys from n on
// read the last one (they are masked).
template <typename T>
__device__ __forceinline__ f32x16 bias_tile(const T* row, int64_t key, int64_t n) {
  f32x16 b;
  const int64_t k = key + 4 * (lane_id() >> 5);
  if (key + 32 <= n) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 v = bias4(row + k + 8 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e) b[4 * g + e] = v[e];
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) b[r] = (float)row[min(k + 8 * (r >> 2) + (r & 3), n - 1)];
  }
  return b;
}

// Bit of register r's key in a logits tile whose 32 keys are `bits`, already shifted by 4 h.
__device__ __forceinline__ bool key_bit(uint32_t bits, int r) { return (bits >> (8 * (r >> 2) + (r & 3))) & 1; }

// Maximum / sum over the two halves of the wave, per column.
__device__ __forceinline__ float halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

int cross_setup(CrossArgs& a, int dtype, const int64_t* shape, const int64_t* strides, float scale, bool has_bias);

}  // namespace bmx
