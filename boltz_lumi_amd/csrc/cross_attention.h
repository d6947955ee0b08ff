// Tiles and operands shared by the cross attention kernels (cross_attention.hip,
// cross_attention_bwd.hip).
//
// Query rows of the `group` heads that share one key / value head are one list: row r of
// key head c is query r % m of head c * group + r / m, so a key tile serves all of them and a
// single query of a shared head still fills MFMA columns.
//
// Operand layout (v_mfma_f32_32x32x16_bf16, or v_mfma_f32_32x32x2f32 for fp32; lane l, half
// h = l / 32): a product tile holds column l % 32 and, in register r, row 8 (r / 4) + 4 h + r % 4. The
// A operand's rows are read in the order that makes this row 16 h + r of the LDS tile (tile_row), so a
// lane's 16 values are 16 rows in a run: of keys, whose bias lies in a run too. A logits tile S^T
// (keys x queries) is then itself the B operand of the next product over its keys: registers 8 t .. 8 t + 7 are
// bf16 step t, register r is fp32 step r.
#pragma once

#include <type_traits>

#include "bmx_common.h"

namespace bmx {

constexpr float kLog2E = 1.4426950408889634f;
constexpr int kFewRows = 32;      // a decoding step's rows of one key head, at most
constexpr int kMaskChunk = 4096;  // keys whose mask words are in LDS at a time

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct CrossArgs {
  const void *q, *k, *v, *bias;
  const uint8_t* mask;
  int64_t sq[3], sk[3], sv[3];  // batch, token, head strides
  int64_t sb[3], smask;         // bias: batch, head, query strides; keys dense
  int64_t batch, m;
  int n, heads, kv_heads, group, dim, rows;  // rows = group * m
  float scale;
  void *out, *out_lo;
  float2* stats;  // [batch][heads][m]: reference point (without a bias before the scale) and log2 of the sum against it
  // work split
  bool exact;       // bf16: weights of 16 bits instead of 8 in the products over them
  int batch_first;  // a bias shared by the batch: its elements' blocks follow each other, so that it stays in L2
  uint32_t blocks;  // of the launch
  int row_blocks, splits;
  int split_keys;  // or, of dK and dV, tiles of 32 queries
  float* part_o;   // [split][batch * kv_heads][rows][dim] sums before the division; backward: [split] gradients
  float2* part_ml;  // [split][batch * kv_heads][rows] maximum and sum
  // backward
  const void* dout;
  float* delta;
  void *dq, *dk, *dv, *dbias;
  int64_t sdb[3];  // dbias: batch (0: shared), head (0: shared), query strides
};

// Blocks go round the XCDs in turn: block b of `total` becomes a position such that each XCD
// works through consecutive ones, whose keys then stay in its own L2.
__device__ __forceinline__ uint32_t xcd_position(uint32_t b, uint32_t total) {
  const uint32_t per = total / 8, whole = per * 8;
  return b < whole ? (b % 8) * per + b / 8 : b;
}
// at % n, with at / n left in at: one axis of a block's position.
__device__ __forceinline__ int take(uint32_t& at, uint32_t n) {
  const uint32_t q = at / n, r = at - q * n;
  at = q;
  return (int)r;
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

// Tile row of A-operand row i.
__device__ __forceinline__ int tile_row(int i) { return 16 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3); }

// Where a lane reads its parts of a 32-row tile. kKeep: every offset in a register, worked out once; with the tile's
// position a constant of an unrolled loop a read is then that register and an immediate. Else the first
// one, from which the others differ by an exclusive or with a constant (one instruction with the tile's position added):
// for kernels that are short of registers.
template <typename T, int DP, bool kKeep = true>
struct RowReads {
  int off[kKeep ? RowOperand<T, DP>::kSteps : 1];
  int steps;  // fp32: with channels below dim, the others are passed over (four MFMA a step)
  __device__ __forceinline__ void init(int dim) {
    steps = (dim + 2 * Tile<T, DP>::kElems - 1) / (2 * Tile<T, DP>::kElems);
    const int r = tile_row(lane_id() & 31), h = lane_id() >> 5;
#pragma unroll
    for (int s = 0; s < (kKeep ? RowOperand<T, DP>::kSteps : 1); ++s) off[s] = Tile<T, DP>::at(r, 2 * s + h);
  }
  __device__ __forceinline__ int at(int s) const { return kKeep ? off[s] : off[0] ^ (s << 5); }
  // In a loop: keeps the compiler from working the others out before it.
  __device__ __forceinline__ void renew() { asm volatile("" : "+v"(off[0])); }
};

// Tile rows (A) times the operand's columns (B), over the channels.
template <typename T, int DP, bool kKeep>
__device__ __forceinline__ f32x16 product(const char* tile, const RowReads<T, DP, kKeep>& reads,
                                          const RowOperand<T, DP>& b) {
  f32x16 acc = zero16();
  auto step = [&](int s) { acc = mfma_step((const T*)nullptr, *(const u32x4*)(tile + reads.at(s)), b.c[s], acc); };
  if (sizeof(T) == 2 || reads.steps == RowOperand<T, DP>::kSteps) {
#pragma unroll
    for (int s = 0; s < RowOperand<T, DP>::kSteps; ++s) step(s);
  } else {
#pragma unroll
    for (int s = 0; s < RowOperand<T, DP>::kSteps; ++s)
      if (s < reads.steps) step(s);
  }
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
  // p cut off to its upper half, and into rest what that left.
  __device__ __forceinline__ void cut(const f32x16& p, Weights& rest) {
    uint32_t word[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      word[i] = __builtin_amdgcn_perm(__float_as_uint(p[2 * i + 1]), __float_as_uint(p[2 * i]), 0x07060302);
    __builtin_memcpy(v, word, 32);
    f32x16 left;
#pragma unroll
    for (int r = 0; r < 16; ++r) left[r] = p[r] - __uint_as_float(__float_as_uint(p[r]) & 0xffff0000u);
    rest.set(left);
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

// acc[dt] += (tile rows)^T (channels 32 dt .. as rows) times the weights, over the rows.
template <typename T, int DP, bool kKeep = true>
struct ColumnReads;
template <int DP, bool kKeep>
struct ColumnReads<bf16, DP, kKeep> {
  int off[4][kKeep ? DP / 32 : 1];  // of four rows each
  __device__ __forceinline__ void init() {
    const int l = lane_id(), h = l >> 5, i = l & 15, chunk = 2 * ((l >> 4) & 1) + ((i & 3) >> 1);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int dt = 0; dt < (kKeep ? DP / 32 : 1); ++dt)
        off[u][dt] = Tile<bf16, DP>::at(16 * h + 4 * u + (i >> 2), 4 * dt + chunk) + 8 * (i & 1);
  }
  __device__ __forceinline__ int at(int u, int dt) const { return kKeep ? off[u][dt] : off[u][0] ^ (dt << 6); }
  __device__ __forceinline__ void renew() {
#pragma unroll
    for (int u = 0; u < 4; ++u) asm volatile("" : "+v"(off[u][0]));
  }
};
template <int DP, bool kKeep>
__device__ __forceinline__ void transposed_product(const char* tile, const ColumnReads<bf16, DP, kKeep>& reads,
                                                   const Weights<bf16>& w, f32x16 (&acc)[DP / 32]) {
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) {
      union {
        s16x4 half[2];
        bf16x8 all;
      } a;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        a.half[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)(tile + reads.at(2 * t + u, dt)));
      acc[dt] = mfma32(a.all, w.v[t], acc[dt]);
    }
}
template <int DP, bool kKeep>
struct ColumnReads<float, DP, kKeep> {
  __device__ __forceinline__ void init() {}
  __device__ __forceinline__ void renew() {}
};
template <int DP, bool kKeep>
__device__ __forceinline__ void transposed_product(const char* tile, const ColumnReads<float, DP, kKeep>&,
                                                   const Weights<float>& w, f32x16 (&acc)[DP / 32]) {
  const int l = lane_id(), h = l >> 5, i = l & 31;
#pragma unroll
  for (int r = 0; r < 16; ++r)
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) {
      const float a = *(const float*)(tile + Tile<float, DP>::at(16 * h + r, 8 * dt + (i >> 2)) + 4 * (i & 3));
      acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, w.v[r], acc[dt], 0, 0, 0);
    }
}

// transposed_product over the weights p, with kExact to 16 bits (two products); their sum to *sum.
template <typename T, int DP, bool kExact, bool kKeep>
__device__ __forceinline__ void weighted_sum(const char* tile, const ColumnReads<T, DP, kKeep>& reads, const f32x16& p,
                                             f32x16 (&acc)[DP / 32], float* sum = nullptr) {
  Weights<T> w;
  if constexpr (kExact) {
    Weights<T> rest;
    w.cut(p, rest);
    if (sum) {
#pragma unroll
      for (int r = 0; r < 16; ++r) *sum += p[r];
    }
    transposed_product<DP>(tile, reads, rest, acc);
  } else {
    w.set(p);
    if (sum) *sum = w.sum(*sum);
  }
  transposed_product<DP>(tile, reads, w, acc);
}

// f(std::bool_constant): kernels with kExact are their own, as a branch in their loops would cost the others 4%.
template <typename T, typename F>
void with_exact(const CrossArgs& a, F f) {
  if constexpr (sizeof(T) == 2) {
    if (a.exact) return f(std::true_type());
  }
  f(std::false_type());
}

// ---- staging -------------------------------------------------------------
// ROWS rows of a tensor through registers into an LDS tile, by THREADS threads. Every load is unconditional (a load in
// a branch of its own would wait for all others): channels past dim read the row's first ones and are stored as zeros.
// Offsets within a tile are 32 bits (a row stride is below kMaxStride elements), so a load is a scalar base and
// one register.
constexpr int64_t kMaxStride = 1 << 22;

template <typename T, int DP, int ROWS, int THREADS>
struct Stage {
  using L = Tile<T, DP>;
  static constexpr int kCount = (ROWS * L::kChunks + THREADS - 1) / THREADS;
  static constexpr bool kEven = (ROWS * L::kChunks) % THREADS == 0;
  u32x4 v[kCount];
  uint32_t off[kCount];

  static __device__ __forceinline__ int row(int t, int i) { return min((t + i * THREADS) / L::kChunks, ROWS - 1); }
  static __device__ __forceinline__ int chunk(int t, int i) { return (t + i * THREADS) % L::kChunks; }

  __device__ __forceinline__ uint32_t offset(int t, int i, int last, int dim, int64_t stride) const {
    const int c = chunk(t, i);
    return (uint32_t)(min(row(t, i), last) * (int)(stride * sizeof(T)) + (c * L::kElems < dim ? c : 0) * 16);
  }
  __device__ __forceinline__ void init(int t, int dim, int64_t stride) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) off[i] = offset(t, i, ROWS - 1, dim, stride);
  }
  // Rows 0 .. ROWS - 1 from `base` on; of a tile with `rows` < ROWS of them the last one again.
  __device__ __forceinline__ void load(int t, const T* base, int rows, int dim, int64_t stride) {
    const char* p = (const char*)base;
    if (rows >= ROWS) {
#pragma unroll
      for (int i = 0; i < kCount; ++i) v[i] = *(const u32x4*)(p + off[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kCount; ++i) v[i] = *(const u32x4*)(p + offset(t, i, rows - 1, dim, stride));
    }
  }
  // live: the tile's rows that hold data (bits); the others are stored as zeros.
  __device__ __forceinline__ void store(int t, char* tile, uint64_t live, int dim) const {
    constexpr uint64_t all = ROWS == 64 ? ~0ull : (1ull << (ROWS & 63)) - 1;
    if (live == all && dim == DP) {
#pragma unroll
      for (int i = 0; i < kCount; ++i)
        if (kEven || t + i * THREADS < ROWS * L::kChunks) *(u32x4*)(tile + L::at(row(t, i), chunk(t, i))) = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < kCount; ++i) {
        const bool ok = ((live >> row(t, i)) & 1) && chunk(t, i) * L::kElems < dim;
        if (kEven || t + i * THREADS < ROWS * L::kChunks)
          *(u32x4*)(tile + L::at(row(t, i), chunk(t, i))) = ok ? v[i] : u32x4{0, 0, 0, 0};
      }
    }
  }
};

// LDS DMA of 64 lanes x 16 bytes, each from base + its off, to lds_addr + 16 * lane (base and lds_addr uniform). It reads
// M0 and the base's SGPRs: one wait state must lie between M0's write and the read, five after a vector write
// of the SGPRs (s_nop 4). The compiler does not see into the asm, nor does it wait for the copy. Every
// wave waits for its own copies of a tile (wait_copies) before the barrier that publishes the tile, and a tile is
// overwritten only after a barrier that every wave reached with its reads of it done.
__device__ __forceinline__ void lds_copy16(const void* base, uint32_t off, unsigned lds_addr) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uintptr_t)base);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)((uintptr_t)base >> 32));
  const void* at = (const void*)((uintptr_t)hi << 32 | lo);
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(at), "{m0}"(lds_addr) : "memory");
}
__device__ __forceinline__ void wait_copies() { __builtin_amdgcn_s_waitcnt(0x0F70); }  // vmcnt(0)
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// ROWS rows of a tensor into an LDS tile by WAVES waves' DMA. A copy writes its lanes' 16 bytes in a run, so the twist is
// in the addresses read. Chunks past dim are not copied: clear_tiles zeroes them once, before the first copy.
template <typename T, int DP, int ROWS, int WAVES>
struct Copy {
  using L = Tile<T, DP>;
  static constexpr int kTotal = ROWS * L::kRow / 64, kPer = (kTotal + WAVES - 1) / WAVES;
  static_assert(ROWS * L::kRow % 64 == 0, "whole copies");
  uint32_t off[kPer];  // ~0: past dim

  static __device__ __forceinline__ uint32_t offset(int part, int last, int dim, int64_t stride) {
    const int p = part * 64 + lane_id(), r = p / L::kRow, c = (p % L::kRow) ^ L::twist(r);
    return c * L::kElems < dim ? (uint32_t)(min(r, last) * (int)(stride * sizeof(T)) + c * 16) : ~0u;
  }
  __device__ __forceinline__ void init(int wave, int dim, int64_t stride) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) off[j] = offset(wave + j * WAVES, ROWS - 1, dim, stride);
  }
  // Rows 0 .. ROWS - 1 from `base` on; of a tile with `rows` < ROWS of them the last one again. wave and tile are uniform.
  __device__ __forceinline__ void issue(int wave, const T* base, int rows, int dim, int64_t stride, unsigned tile) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int part = wave + j * WAVES;
      if (kTotal % WAVES != 0 && part >= kTotal) break;
      const uint32_t o = rows >= ROWS ? off[j] : offset(part, rows - 1, dim, stride);
      if (o != ~0u) lds_copy16(base, o, tile + part * 1024);
    }
  }
};

// Zeros in `bytes` of LDS by THREADS threads, where tiles have chunks past dim.
template <typename T, int DP, int THREADS>
__device__ __forceinline__ void clear_tiles(int t, char* lds, int bytes, int dim) {
  if (dim == DP) return;  // chunks past DP are never read
  for (int at = 16 * t; at < bytes; at += 16 * THREADS) *(u32x4*)(lds + at) = u32x4{0, 0, 0, 0};
  __syncthreads();
}

// Zeros in the tile rows whose bit is not set, by THREADS threads.
template <typename T, int DP, int ROWS, int THREADS>
__device__ __forceinline__ void clear_rows(int t, char* tile, uint64_t live) {
  constexpr int kRow = Tile<T, DP>::kRow;
  for (int at = t; at < ROWS * kRow; at += THREADS)
    if (!((live >> (at / kRow)) & 1)) *(u32x4*)(tile + at * 16) = u32x4{0, 0, 0, 0};
}

// Orders a wave's LDS writes and its other lanes' reads where no barrier does: the LDS serves a wave in order, so
// only the compiler has to keep them.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// ---- key mask ------------------------------------------------------------
// Bit words of a chunk of keys: bit j of word w is key c0 + 32 w + j present (inside the mask and below end).
// All threads call fill (two barriers); key c0 is a multiple of 32.
struct KeyWords {
  uint32_t* words;  // LDS [kMaskChunk / 32]
  const uint8_t* mask;
  int c0, end;

  __device__ __forceinline__ void fill(int first, int stop) {
    c0 = first, end = stop;
    if (!mask) return;
    __syncthreads();
    const int left = min(stop - first, kMaskChunk);
    for (int w = threadIdx.x >> 6; 64 * w < left; w += blockDim.x >> 6) {
      const int key = first + 64 * w + lane_id();
      const bool on = key < stop && mask[key < stop ? key : stop - 1] != 0;
      const uint64_t bits = __ballot(on);
      if (lane_id() < 2) words[2 * w + lane_id()] = (uint32_t)(bits >> (32 * lane_id()));
    }
    __syncthreads();
  }
  // Presence of the 32 keys from `key` on, the same in every lane; key - c0 a multiple of 32.
  __device__ __forceinline__ uint32_t bits(int key) const {
    if (key >= end) return 0;
    if (mask) return (uint32_t)__builtin_amdgcn_readfirstlane((int)words[(key - c0) >> 5]);
    return end - key >= 32 ? ~0u : (1u << (end - key)) - 1;
  }
  // The next 32 keys from `key` on that hold a present one, or the first past `last`.
  __device__ __forceinline__ int next(int key, int last) const {
    if (mask)
      while (key < last && bits(key) == 0) key += 32;
    return key;
  }
};

// ---- bias ----------------------------------------------------------------
// Bias of a lane's query at the 16 keys of a logits tile, in register order, as it lies in memory: loaded a tile ahead,
// together with the tile's copies, whose wait is then its own. bf16 rows at an odd element (an odd number of keys) are read
// from the dword before and shifted: 16-byte loads at 2-byte alignment took 109 us against 74 at 1531 keys.
__device__ __forceinline__ bool bias_odd(const CrossArgs& a) {
  return (((int)((uintptr_t)a.bias >> 1) | (int)a.sb[0] | (int)a.sb[1] | (int)a.sb[2]) & 1) != 0;
}

template <typename T>
struct BiasTile;
template <>
struct BiasTile<float> {
  typedef uint32_t u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
  u32x4 v[4];

  // Keys from `key` on; those from n on repeat the last one (they are masked).
  __device__ __forceinline__ void load(const float* row, int key, int n) {
    const int k = key + 16 * (lane_id() >> 5);
    if (key + 32 <= n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *(const u32x4_at4*)(row + k + 4 * i);
    } else {
      asm volatile("" : "+s"(n));  // keeps a loop's compiler from holding all these addresses over it
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r >> 2][r & 3] = __float_as_uint(row[min(k + r, n - 1)]);
    }
  }
  __device__ __forceinline__ void ready(bool) {}
  __device__ __forceinline__ float at(int r) const { return __uint_as_float(v[r >> 2][r & 3]); }
};
template <>
struct BiasTile<bf16> {
  typedef uint32_t u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
  u32x4 v[2];
  uint32_t last, shift;

  __device__ __forceinline__ void load(const bf16* row, int key, int n) {
    const int k = key + 16 * (lane_id() >> 5);
    if (key + 32 <= n) {
      const uintptr_t at = (uintptr_t)(row + k), odd = at & 2;
      const uint32_t* p = (const uint32_t*)(at - odd);  // every dword read holds one of the keys' values
#pragma unroll
      for (int i = 0; i < 2; ++i) v[i] = *(const u32x4_at4*)(p + 4 * i);
      last = p[odd ? 8 : 7];
      shift = (uint32_t)odd * 8;
    } else {
      asm volatile("" : "+s"(n));
      uint16_t x[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) x[r] = __builtin_bit_cast(uint16_t, row[min(k + r, n - 1)]);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i >> 2][i & 3] = x[2 * i] | (uint32_t)x[2 * i + 1] << 16;
      last = shift = 0;
    }
  }
  // Shifts the words into place, before the first at(); odd: some row of the bias may need it (uniform).
  __device__ __forceinline__ void ready(bool odd) {
    if (!odd) return;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i >> 2][i & 3] = __builtin_amdgcn_alignbit(i < 7 ? v[(i + 1) >> 2][(i + 1) & 3] : last, v[i >> 2][i & 3], shift);
  }
  __device__ __forceinline__ float at(int r) const {
    const uint32_t w = v[r >> 3][(r >> 1) & 3];
    return __uint_as_float(r & 1 ? w & 0xffff0000u : w << 16);
  }
};

// Bit of register r's key in a logits tile whose 32 keys are `bits`, already shifted by 16 h.
__device__ __forceinline__ bool key_bit(uint32_t bits, int r) { return (bits >> r) & 1; }

// Maximum / sum over the two halves of the wave, per column.
__device__ __forceinline__ float halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---- reference point -----------------------------------------------------
// A row's weights are taken against one of its logits, `top` (with a bias in natural units, without one before the scale;
// c0 takes either to base 2). fp32: exp2((x - top) c0). bf16 saves the subtraction, exp2(x c - S) in one multiply-add with
// S = top c rounded once: whatever that rounding is, all weights of the row share it, so sums
// against another reference point are moved by the difference of the two S, and what is kept for the gradients is
// corrected to top itself. From 2^29 on two logits differ by nothing or by at least 2^5, the weights are zeros and
// ones in any unit, and one in which S is exact keeps the shared factor from leaving fp32's range (below it is 2^32 at most).
__device__ __forceinline__ float logit_unit(float top, float c0) {
  const float t = fabsf(top);
  if (t * c0 <= 0x1p29f) return c0;
  const float p = __uint_as_float(__float_as_uint(c0) & 0x7f800000u);  // the power of two below
  return t > 0x1p64f ? fminf(p, 1.f) : p;
}
// S: the product on its own, not a part of a multiply-add.
__device__ __forceinline__ float reference_shift(float top, float c) {
  float s = top * c;
  asm("" : "+v"(s));
  return s;
}
// What sums taken against `from` (-inf: none yet) are multiplied by to be against `to` (finite).
template <typename T>
__device__ __forceinline__ float rescale(float from, float to, float c0) {
  if (sizeof(T) == 4) return __builtin_amdgcn_exp2f((from - to) * c0);
  const float c = logit_unit(from, c0), d = logit_unit(to, c0);
  return __builtin_amdgcn_exp2f(c == d ? reference_shift(from, c) - reference_shift(to, d) : (from - to) * fminf(c, d));
}

int cross_setup(CrossArgs& a, int dtype, const int64_t* shape, const int64_t* strides, float scale, bool has_bias);

}  // namespace bmx
