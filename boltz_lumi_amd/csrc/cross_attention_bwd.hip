// Gradients of cross attention (cross_attention.hip), from the row statistics
// that the forward pass kept:
//
//   P = exp(S - max) / sum;  dV = P^T dO;  dP = dO V^T;  delta = rowsum(dO O)
//   dS = P (dP - delta);  dQ = scale dS K;  dK = scale dS^T Q;  dbias = dS summed over its shared axes
//
// No logits are kept: each kernel recomputes S and dP for its tiles.  Three
// kernels instead of one, because each sums over another axis and keeps its sum in
// registers: no atomics, and the same bits on every run.  P and dS are rounded to
// the operand's type for the products over them (small elements: to two of them),
// and where the forward pass summed rounded weights, P is divided by that sum: half a step
// more at most, of a row that one weight dominates.  delta is taken from the output
// before its rounding (out + out_lo), so that dP - delta cancels as it does in the formula.
#include <algorithm>
#include <type_traits>

#include "cross_attention.h"

using namespace bmx;

namespace {

// Offset of list row r of key head c: query i of head c * group + g.
struct RowAt {
  int64_t head;
  int i;
  __device__ __forceinline__ RowAt(const CrossArgs& a, int c, int row) {
    const int r = min(row, a.rows - 1), g = r / (int)a.m;
    i = r - g * (int)a.m;
    head = (int64_t)c * a.group + g;
  }
  __device__ __forceinline__ int64_t q(const CrossArgs& a, int64_t b) const {
    return b * a.sq[0] + i * a.sq[1] + head * a.sq[2];
  }
  __device__ __forceinline__ int64_t dense(const CrossArgs& a, int64_t b) const {  // out, dout, dq
    return ((b * a.m + i) * a.heads + head) * a.dim;
  }
  __device__ __forceinline__ int64_t stat(const CrossArgs& a, int64_t b) const { return (b * a.heads + head) * a.m + i; }
  __device__ __forceinline__ int64_t bias(const CrossArgs& a, int64_t b) const {
    return b * a.sb[0] + head * a.sb[1] + i * a.sb[2];
  }
};

// delta: 16 lanes per row of [batch, m, heads], written as [batch][heads][m].
template <typename T>
__global__ __launch_bounds__(256) void cross_attention_delta(CrossArgs a) {
  const int64_t at = (int64_t)block_index() * 16 + (threadIdx.x >> 4), total = a.batch * a.m * a.heads;
  const int l = threadIdx.x & 15;
  float sum = 0.f;
  if (at < total) {
    for (int d = 4 * l; d < a.dim; d += 64) {
      const int64_t p = at * a.dim + d;
      f32x4 o = load4((const T*)a.out + p);
      if (a.out_lo) o += load4((const T*)a.out_lo + p);
      const f32x4 g = load4((const T*)a.dout + p);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += o[e] * g[e];
    }
  }
  sum += dpp<0xB1>(sum);
  sum += dpp<0x4E>(sum);
  sum += dpp<0x141>(sum);
  sum += dpp<0x140>(sum);
  if (at >= total || l != 0) return;
  const int64_t bi = at / a.heads, head = at - bi * a.heads, b = bi / a.m, i = bi - b * a.m;
  a.delta[(b * a.heads + head) * a.m + i] = sum;
}

// Four channels of a gradient row.
template <typename T>
__device__ __forceinline__ void store_rows(T* row, int dim, const f32x16& acc, int dt, float f, bool live) {
  const int h = lane_id() >> 5;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int d = 32 * dt + 8 * g + 4 * h;
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = live ? acc[4 * g + e] * f : 0.f;
    if (d < dim) store4(row + d, v);
  }
}

// The 16 values of a run of keys of one row, at any element alignment.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
template <typename T>
__device__ __forceinline__ void store_keys(T* row, int key, int n, const f32x16& v) {
  if (key + 16 <= n) {
    constexpr int kElems = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 16 / kElems; ++i) {
      T x[kElems];
#pragma unroll
      for (int e = 0; e < kElems; ++e) x[e] = (T)v[i * kElems + e];
      u32x4 word;
      __builtin_memcpy(&word, x, 16);
      *(u32x4_any*)(row + key + i * kElems) = word;
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (key + r < n) row[key + r] = (T)v[r];
  }
}

// Without a bias bf16 weights are one multiply-add and an exponential, exp2(x c - (top c + log)), where that sum's rounding
// stays below 2^-16. A row further from zero takes the difference x - top first, as rows with a bias and fp32 do.
__device__ __forceinline__ bool far_row(const CrossArgs& a, float2 st) {
  return fabsf(st.x) * (a.scale * kLog2E) > 256.f;
}

// P of a logits tile whose column is a query: reference point and log2 of the sum are the lane's. far: of some row.
template <typename T, bool kBias>
__device__ __forceinline__ void weights_of(const CrossArgs& a, f32x16& s, const BiasTile<T>& b, float2 st, bool far) {
  const float c = a.scale * kLog2E;
  if (kBias) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f((s[r] * a.scale + b.at(r) - st.x) * kLog2E - st.y);
  } else if (sizeof(T) == 4 || far) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f((s[r] - st.x) * c - st.y);
  } else {
    const float shift = -(st.x * c + st.y);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] * c + shift);
  }
}

// dQ: four waves of 32 rows over all keys, as the forward pass runs (batch 2, 32 / 8 heads, 2048 x 4096, D = 128: 377 us,
// 1090 TF/s; the choice of far rows costs 1 to 3%).
template <typename T, int DP, bool kBias, bool kExact>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 64 ? 1 : 2) void cross_attention_dq(CrossArgs a) {
  constexpr int kTile = 32 * Tile<T, DP>::kRowBytes;
  __shared__ __attribute__((aligned(16))) char lds[4 * kTile + kMaskChunk / 8];
  if (block_index() >= a.blocks) return;
  uint32_t at = xcd_position(block_index(), a.blocks);
  int64_t b = a.batch_first ? take(at, a.batch) : 0;
  const int row_block = take(at, a.row_blocks), split = take(at, a.splits), c = take(at, a.kv_heads);
  if (!a.batch_first) b = at;
  const int first = split * a.split_keys, stop = min(first + a.split_keys, a.n);
  const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), h = lane_id() >> 5;
  const int row = row_block * 128 + w * 32 + (t & 31);
  const RowAt ra(a, c, row);
  RowOperand<T, DP> q, g;
  q.load((const T*)a.q + ra.q(a, b), a.dim, h);
  g.load((const T*)a.dout + ra.dense(a, b), a.dim, h);
  const float2 st = a.stats[ra.stat(a, b)];
  const float delta = a.delta[ra.stat(a, b)];
  const bool far = !kBias && sizeof(T) == 2 && __any(far_row(a, st));
  const T* bias_row = (const T*)a.bias + ra.bias(a, b);
  RowReads<T, DP> rr;
  ColumnReads<T, DP> cr;
  rr.init(a.dim);
  cr.init();
  f32x16 dq[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) dq[dt] = zero16();
  const T* k = (const T*)a.k + b * a.sk[0] + c * a.sk[2];
  const T* v = (const T*)a.v + b * a.sv[0] + c * a.sv[2];
  KeyWords words{(uint32_t*)(lds + 4 * kTile), a.mask ? a.mask + b * a.smask : nullptr};
  Copy<T, DP, 32, 4> ck, cv;
  ck.init(w, a.dim, a.sk[1]);
  cv.init(w, a.dim, a.sv[1]);
  const unsigned lds0 = lds_address(lds);
  clear_tiles<T, DP, 256>(t, lds, 4 * kTile, a.dim);
  const int chunk = a.mask ? kMaskChunk : stop - first;
  for (int c0 = first; c0 < stop; c0 += chunk) {
    words.fill(c0, stop);  // its barrier also ends the last chunk's reads of the tiles
    const int end = min(c0 + chunk, stop);
    auto copy = [&](int key, unsigned tile) {
      ck.issue(w, k + key * a.sk[1], a.n - key, a.dim, a.sk[1], tile);
      cv.issue(w, v + key * a.sv[1], a.n - key, a.dim, a.sv[1], tile + kTile);
    };
    int key = words.next(c0, end);
    BiasTile<T> bias[2];
    auto step = [&](auto B) {
      constexpr int kAt = decltype(B)::value * 2 * kTile, kOther = 2 * kTile - kAt;
      const char *kt = lds + kAt, *vt = lds + kAt + kTile;
      const uint32_t bits = words.bits(key);
      const int after = words.next(key + 32, end);
      wait_copies();
      __syncthreads();
      if (after < end) {
        copy(after, lds0 + kOther);
        if (kBias) bias[1 - decltype(B)::value].load(bias_row, after, a.n);
      }
      if (bits != ~0u) {  // what a left-out key holds must not meet its zero dS
        clear_rows<T, DP, 32, 256>(t, lds + kAt, bits);
        __syncthreads();
      }
      f32x16 s = product<T, DP>(kt, rr, q);
      const f32x16 dp = product<T, DP>(vt, rr, g);
      if (kBias) bias[decltype(B)::value].ready(true);
      weights_of<T, kBias>(a, s, bias[decltype(B)::value], st, far);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] *= dp[r] - delta;
      if (bits != ~0u) {
        const uint32_t mine = bits >> (16 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!key_bit(mine, r)) s[r] = 0.f;
      }
      weighted_sum<T, DP, kExact>(kt, cr, s, dq);
      key = after;
      return key < end;
    };
    if (key < end) {
      copy(key, lds0);
      if (kBias) bias[0].load(bias_row, key, a.n);
      while (step(std::integral_constant<int, 0>()) && step(std::integral_constant<int, 1>())) {
      }
    }
  }
  if (row >= a.rows) return;
  float* part = a.part_o + split * a.batch * a.m * a.heads * a.dim + ra.dense(a, b);
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) {
    if (a.splits > 1)
      store_rows(part, a.dim, dq[dt], dt, a.scale, true);
    else
      store_rows((T*)a.dq + ra.dense(a, b), a.dim, dq[dt], dt, a.scale, true);
  }
}

// dK and dV: four waves of 32 keys (in the lanes, in tile_row order) over all rows of the group's heads in
// tiles of 32 queries of one head, so a shared key head's gradient is one sum in row order.
// Queries past the last repeat it with weights of zero. A wave's K, and V for narrow heads, are in registers;
// bf16 heads past 64 channels keep V in LDS, which makes room for two waves on a SIMD.
// A bias of its own for every head and batch element has its gradient written here, as dS is at hand (kGrad).
// Bound by the MFMA (batch 2, 32 / 8 heads, 2048 x 4096, D = 128: 518 us, 1060 TF/s), with a bias by
// the work between the products at two waves a SIMD (batch 5, 16 heads, 1024 x 1531, D = 64: 116 us, 550 TF/s; its 16
// two-byte loads a lane are not it: whole runs of keys turned through LDS took 124). Two waves a SIMD leave 256
// registers: bf16 with D = 128 spills 3 of them, 11 with 16-bit weights and 20 to 39 with a bias, fp32 with D = 64
// and a shared bias 26.
template <typename T, int DP, bool kBias, bool kGrad, bool kExact>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 64 ? 1 : 2) void cross_attention_dkv(CrossArgs a) {
  constexpr bool kValuesInLds = sizeof(T) == 2 && DP > 64;
  constexpr bool kFirst = kBias || sizeof(T) == 4;
  constexpr int kTile = 32 * Tile<T, DP>::kRowBytes;
  constexpr int kStat = 32 * 3 * 4;  // of a row: reference point (or the whole shift), log2 of the sum, delta
  constexpr int kValues = 4 * kTile + 2 * kStat + 16;  // V of the block's 128 keys
  __shared__ __attribute__((aligned(16))) char lds[kValues + (kValuesInLds ? 4 * kTile : 0)];
  const int key_blocks = (a.n + 127) / 128;
  if (block_index() >= a.blocks) return;
  uint32_t at = xcd_position(block_index(), a.blocks);
  int64_t b = a.batch_first ? take(at, a.batch) : 0;
  const int first = take(at, key_blocks) * 128, split = take(at, a.splits), c = take(at, a.kv_heads);
  if (!a.batch_first) b = at;
  const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), l = lane_id(), h = l >> 5;
  const int lane_key = tile_row(l & 31), key = first + w * 32 + lane_key, safe = min(key, a.n - 1);
  KeyWords words{(uint32_t*)(lds + 4 * kTile + 2 * kStat), a.mask ? a.mask + b * a.smask : nullptr};
  words.fill(first, min(first + 128, a.n));
  const bool live = (words.bits(first + w * 32) >> lane_key) & 1;
  uint32_t any = kGrad;  // left-out keys have a gradient of zero to write
#pragma unroll
  for (int i = 0; i < 4; ++i) any |= words.bits(first + 32 * i);
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) dk[dt] = zero16(), dv[dt] = zero16();
  if (any) {
    RowOperand<T, DP> kf, vf;
    kf.load((const T*)a.k + b * a.sk[0] + safe * a.sk[1] + c * a.sk[2], a.dim, h);
    if (!kValuesInLds) vf.load((const T*)a.v + b * a.sv[0] + safe * a.sv[1] + c * a.sv[2], a.dim, h);
    RowReads<T, DP, !kValuesInLds> rr;
    ColumnReads<T, DP, !kValuesInLds> cr;
    rr.init(a.dim);
    cr.init();
    const int64_t row_step = (int64_t)a.heads * a.dim;
    Copy<T, DP, 32, 4> cq, cg;
    cq.init(w, a.dim, a.sq[1]);
    cg.init(w, a.dim, row_step);
    const unsigned lds0 = lds_address(lds);
    clear_tiles<T, DP, 256>(t, lds, 4 * kTile, a.dim);
    if (kValuesInLds) {  // waited for with the first tile; each wave reads the 32 rows of its keys
      Copy<T, DP, 128, 4> values;
      values.init(w, a.dim, a.sv[1]);
      if (a.dim != DP) {
        for (int z = 16 * t; z < 4 * kTile; z += 16 * 256) *(u32x4*)(lds + kValues + z) = u32x4{0, 0, 0, 0};
        __syncthreads();
      }
      values.issue(w, (const T*)a.v + b * a.sv[0] + first * a.sv[1] + c * a.sv[2], a.n - first, a.dim, a.sv[1],
                   lds0 + kValues);
    }
    const int m = (int)a.m, head_tiles = (m + 31) / 32;
    int tile_at = split * a.split_keys;
    const int tile_end = min(tile_at + a.split_keys, a.group * head_tiles);
    float2 st;
    float delta;
    auto copy = [&](int g, int i, unsigned tile) {
      const int64_t head = (int64_t)c * a.group + g;
      cq.issue(w, (const T*)a.q + b * a.sq[0] + i * a.sq[1] + head * a.sq[2], m - i, a.dim, a.sq[1], tile);
      cg.issue(w, (const T*)a.dout + ((b * a.m + i) * a.heads + head) * a.dim, m - i, a.dim, row_step, tile + kTile);
    };
    auto load_stats = [&](int g, int i) {
      const int64_t stat = (b * a.heads + (int64_t)c * a.group + g) * a.m + min(i + (t & 31), m - 1);
      st = a.stats[stat], delta = a.delta[stat];
      if (i + (t & 31) >= m) st = make_float2(0.f, INFINITY), delta = 0.f;
    };
    T bias[16];  // of the lane's key and 16 queries, a tile ahead
    const uint32_t bias_lane = (uint32_t)(16 * h * a.sb[2]) + safe;
    auto load_bias = [&](int g, int i) {
      const T* at = (const T*)a.bias + b * a.sb[0] + ((int64_t)c * a.group + g) * a.sb[1];
      if (i + 32 <= m) {
#pragma unroll
        for (int r = 0; r < 16; ++r) bias[r] = (at + (i + r) * a.sb[2])[bias_lane];
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) bias[r] = at[min(i + 16 * h + r, m - 1) * a.sb[2] + safe];
      }
    };
    int g = __builtin_amdgcn_readfirstlane(tile_at / head_tiles), i = (tile_at - g * head_tiles) * 32;
    auto step = [&](auto buffer) {  // one tile; false after the last
      const int buf = buffer;
      if (kValuesInLds) rr.renew(), cr.renew();
      const char *qt = lds + buf * 2 * kTile, *gt = qt + kTile;
      float* stat = (float*)(lds + 4 * kTile + buf * kStat);
      const bool far = !kFirst && __any(far_row(a, st));  // the same in all waves
      if (t < 32) {
        stat[t] = kFirst || far ? st.x : st.x * (a.scale * kLog2E) + st.y;
        stat[32 + t] = st.y;
        stat[64 + t] = delta;
      }
      T* dbias = nullptr;
      int left = 0;  // of the lane's 16 queries
      if (kGrad) {
        dbias = (T*)a.dbias + b * a.sdb[0] + ((int64_t)c * a.group + g) * a.sdb[1] + (i + 16 * h) * a.sdb[2] + key;
        left = key < a.n ? m - i - 16 * h : 0;
      }
      i += 32;
      if (i >= m) i = 0, ++g;
      const bool more = ++tile_at < tile_end;
      wait_copies();
      __syncthreads();
      float x[16];
      if (kBias) {
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = (float)bias[r];
      }
      if (more) {
        copy(g, i, lds0 + (buf ^ 1) * 2 * kTile);
        load_stats(g, i);
        if (kBias) load_bias(g, i);
      }
      f32x16 s = product<T, DP>(qt, rr, kf), dp;
      if (!kValuesInLds) dp = product<T, DP>(gt, rr, vf);
      auto weigh = [&](auto first) {
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const f32x4 top = *(const f32x4*)(stat + 4 * g4 + 16 * h);
          f32x4 log;
          if (first) log = *(const f32x4*)(stat + 32 + 4 * g4 + 16 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * g4 + e;
            if (kBias)
              s[r] = __builtin_amdgcn_exp2f((s[r] * a.scale + x[r] - top[e]) * kLog2E - log[e]);
            else if (first)
              s[r] = __builtin_amdgcn_exp2f((s[r] - top[e]) * (a.scale * kLog2E) - log[e]);
            else
              s[r] = __builtin_amdgcn_exp2f(s[r] * (a.scale * kLog2E) - top[e]);
          }
        }
      };
      if (kFirst || far)
        weigh(std::true_type());
      else
        weigh(std::bool_constant<kFirst>());
      if (kValuesInLds) __builtin_amdgcn_sched_barrier(0);
      weighted_sum<T, DP, kExact>(gt, cr, s, dv);
      if (kValuesInLds) __builtin_amdgcn_sched_barrier(0);
      if (kValuesInLds) {
        dp = zero16();
#pragma unroll
        for (int u = 0; u < RowOperand<T, DP>::kSteps; ++u) {
          dp = mfma_step((const T*)nullptr, *(const u32x4*)(gt + rr.at(u)),
                         *(const u32x4*)(lds + kValues + w * kTile + rr.at(u)), dp);
          if (u % 2) __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        const f32x4 dl = *(const f32x4*)(stat + 64 + 4 * g4 + 16 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * g4 + e] *= dp[4 * g4 + e] - dl[e];
      }
      if (kGrad) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (r < left) dbias[r * a.sdb[2]] = live ? (T)s[r] : (T)0.f;
      }
      if (kValuesInLds) __builtin_amdgcn_sched_barrier(0);
      weighted_sum<T, DP, kExact>(qt, cr, s, dk);
      return more;
    };
    copy(g, i, lds0);
    load_stats(g, i);
    if (kBias) load_bias(g, i);
    if (kValuesInLds) {
      for (int buf = 0; step(buf); buf ^= 1) {
      }
    } else {
      while (step(std::integral_constant<int, 0>()) && step(std::integral_constant<int, 1>())) {
      }
    }
  }
  if (key >= a.n) return;
  const int64_t out = ((b * a.n + key) * a.kv_heads + c) * a.dim, whole = a.batch * a.n * a.kv_heads * a.dim;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) {
    if (a.splits > 1) {
      if (a.dk) store_rows(a.part_o + split * whole + out, a.dim, dk[dt], dt, a.scale, live);
      if (a.dv) store_rows(a.part_o + (a.splits + split) * whole + out, a.dim, dv[dt], dt, 1.f, live);
    } else {
      if (a.dk) store_rows((T*)a.dk + out, a.dim, dk[dt], dt, a.scale, live);
      if (a.dv) store_rows((T*)a.dv + out, a.dim, dv[dt], dt, 1.f, live);
    }
  }
}

// dbias of a bias that batch elements or heads share: a block holds 128 queries x kBiasKeys keys of one bias plane in
// registers and walks the batch elements and heads that share the plane, in order. A step is short, so what bounds it is
// the chain of its loads: the next step's operands are copied while one is computed, its mask an element earlier, and
// the bias is loaded once if it is the same in all steps (batch 5, 16 heads, 1024 x 1531, D = 64: 127 -> 102 us).
// bf16 has all four operands in LDS by DMA. Up to 64 channels four waves and 64 keys take 64 KB, K and V in two buffers:
// two blocks on a compute unit (before the copies ran ahead: eight waves and 128 keys 155 us, four and 128 spill: 250).
// Past 64 channels eight waves, four by the queries and two by the keys, and 128 keys take 128 KB (batch 2, 16 heads,
// 1024 x 2048, D = 128: 105 us; four waves and 64 keys with the queries read into registers 154). fp32: four waves
// and 32 keys, the queries' operands read straight into registers.
template <typename T, int DP>
constexpr int kBiasWaves = sizeof(T) == 2 && DP > 64 ? 8 : 4;
template <typename T, int DP>
constexpr int kBiasKeys = sizeof(T) == 4 ? 32 : DP > 64 ? 128 : 64;

template <typename T, int DP>
__global__ __launch_bounds__((64 * kBiasWaves<T, DP>), sizeof(T) == 4 && DP > 64 ? 1 : 2)
void cross_attention_dbias(CrossArgs a) {
  constexpr bool kRowsInLds = sizeof(T) == 2;
  constexpr int kWaves = kBiasWaves<T, DP>, kThreads = 64 * kWaves, KT = kBiasKeys<T, DP>;
  constexpr int kParts = KT / 32 / (kWaves / 4);  // of 32 keys, of a wave
  constexpr int kRowBytes = Tile<T, DP>::kRowBytes, kTile = KT * kRowBytes, kRowTile = kRowsInLds ? 128 * kRowBytes : 0;
  constexpr bool kDouble = !kRowsInLds || DP <= 64;  // K and V in two buffers
  constexpr int kKeyTiles = kDouble ? 4 * kTile : 2 * kTile, kAll = kKeyTiles + 2 * kRowTile, kMasks = (KT + 63) / 64;
  __shared__ __attribute__((aligned(16))) char lds[kAll];
  const int key_blocks = (a.n + KT - 1) / KT, query_blocks = (int)((a.m + 127) / 128);
  if (block_index() >= a.blocks) return;
  uint32_t at = xcd_position(block_index(), a.blocks);
  const int key = take(at, key_blocks) * KT, q0 = take(at, query_blocks) * 128;
  const int64_t ph = take(at, a.sdb[1] ? a.heads : 1), pb = at;
  const int64_t b0 = a.sdb[0] ? pb : 0, b1 = a.sdb[0] ? pb + 1 : a.batch;
  const int h0 = a.sdb[1] ? (int)ph : 0, h1 = a.sdb[1] ? (int)ph + 1 : a.heads;
  const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), l = lane_id(), h = l >> 5;
  const int rows_at = (w & 3) * 32, keys_at = (w >> 2) * 32 * kParts;  // of the wave, in the block's
  const int m = (int)a.m, i = q0 + rows_at + tile_row(l & 31), safe = min(i, m - 1);
  f32x16 sum[kParts];
#pragma unroll
  for (int u = 0; u < kParts; ++u) sum[u] = zero16();
  RowReads<T, DP> rr;
  rr.init(a.dim);
  const int64_t row_step = (int64_t)a.heads * a.dim;
  Copy<T, DP, KT, kWaves> ck, cv;
  Copy<T, DP, 128, kWaves> cq, cg;
  ck.init(w, a.dim, a.sk[1]);
  cv.init(w, a.dim, a.sv[1]);
  if (kRowsInLds) {
    cq.init(w, a.dim, a.sq[1]);
    cg.init(w, a.dim, row_step);
  }
  const unsigned lds0 = lds_address(lds);
  clear_tiles<T, DP, kThreads>(t, lds, kAll, a.dim);

  // Presence of the keys in a batch element, whose mask is loaded an element ahead.
  uint8_t ahead[kMasks];
  uint64_t bits[kMasks];
  auto load_mask = [&](int64_t b) {
#pragma unroll
    for (int u = 0; u < kMasks; ++u)
      ahead[u] = a.mask ? a.mask[min(b, b1 - 1) * a.smask + min(key + 64 * u + l, a.n - 1)] : 1;
  };
  auto find = [&](int64_t b) {  // the first element from b on (whose mask is in `ahead`) with a present key
    for (; b < b1; ++b) {
      uint64_t any = 0;
#pragma unroll
      for (int u = 0; u < kMasks; ++u) {
        const int k = 64 * u + l;
        any |= bits[u] = __ballot(ahead[u] != 0 && k < KT && key + k < a.n);
      }
      load_mask(b + 1);
      if (any) break;
    }
    return b;
  };
  // A step's operands: one batch element and head. The next step's are on their way while a step is computed.
  float2 next_st;
  float next_delta;
  BiasTile<T> bias[kParts];
  auto issue_keys = [&](int64_t b, int head, unsigned tile) {
    const int c = head / a.group;
    ck.issue(w, (const T*)a.k + b * a.sk[0] + c * a.sk[2] + key * a.sk[1], a.n - key, a.dim, a.sk[1], tile);
    cv.issue(w, (const T*)a.v + b * a.sv[0] + c * a.sv[2] + key * a.sv[1], a.n - key, a.dim, a.sv[1], tile + kTile);
  };
  auto issue_rows = [&](int64_t b, int head) {
    const int64_t stat = (b * a.heads + head) * a.m + safe;
    next_st = a.stats[stat], next_delta = a.delta[stat];
    if (!kRowsInLds) return;
    cq.issue(w, (const T*)a.q + b * a.sq[0] + head * a.sq[2] + q0 * a.sq[1], m - q0, a.dim, a.sq[1], lds0 + kKeyTiles);
    cg.issue(w, (const T*)a.dout + (b * a.m * a.heads + head) * a.dim + q0 * row_step, m - q0, a.dim, row_step,
             lds0 + kKeyTiles + kRowTile);
  };
  auto load_bias = [&](int64_t b, int head) {
    const T* row = (const T*)a.bias + b * a.sb[0] + head * a.sb[1] + safe * a.sb[2];
#pragma unroll
    for (int u = 0; u < kParts; ++u) {
      bias[u].load(row, min(key + keys_at + 32 * u, a.n - 1), a.n);
      bias[u].ready(true);
    }
  };
  load_mask(b0);
  int64_t b = find(b0);
  int head = h0, buf = 0;
  if (b < b1) {
    load_bias(b, head);
    issue_rows(b, head);
    issue_keys(b, head, lds0);
  }
  while (b < b1) {
    uint64_t mine[kMasks];
#pragma unroll
    for (int u = 0; u < kMasks; ++u) mine[u] = bits[u];
    wait_copies();
    __syncthreads();
    const float2 st = next_st;
    const float delta = next_delta;
    RowOperand<T, DP> q, g;
    if (kRowsInLds) {
#pragma unroll
      for (int s = 0; s < RowOperand<T, DP>::kSteps; ++s) {
        q.c[s] = *(const u32x4*)(lds + kKeyTiles + rows_at * kRowBytes + rr.at(s));
        g.c[s] = *(const u32x4*)(lds + kKeyTiles + kRowTile + rows_at * kRowBytes + rr.at(s));
      }
      __syncthreads();  // every wave has its rows: the next step's may come
    } else {
      q.load((const T*)a.q + b * a.sq[0] + head * a.sq[2] + safe * a.sq[1], a.dim, h);
      g.load((const T*)a.dout + (b * a.m * a.heads + head) * a.dim + safe * row_step, a.dim, h);
    }
    const int64_t this_b = b;
    if (++head == h1) head = h0, b = find(b + 1);
    if (b < b1) {
      issue_rows(b, head);
      if (kDouble) issue_keys(b, head, lds0 + (buf ^ 1) * 2 * kTile);
    }
#pragma unroll
    for (int u = 0; u < kParts; ++u) {
      const char* kt = lds + buf * 2 * kTile + (keys_at + 32 * u) * kRowBytes;
      f32x16 s = product<T, DP>(kt, rr, q);
      const f32x16 dp = product<T, DP>(kt + kTile, rr, g);
      weights_of<T, true>(a, s, bias[u], st, false);
      const uint32_t keys = (uint32_t)(mine[(keys_at + 32 * u) / 64] >> ((keys_at + 32 * u) % 64)) >> (16 * h);
#pragma unroll
      for (int r = 0; r < 16; ++r) sum[u][r] += key_bit(keys, r) ? s[r] * (dp[r] - delta) : 0.f;
      __builtin_amdgcn_sched_barrier(0);  // one part's operands at a time: all of them spill
    }
    if (b >= b1) break;
    if (kDouble) {
      buf ^= 1;
    } else {
      __syncthreads();  // every wave is done with the keys
      issue_keys(b, head, lds0);
    }
    if ((a.sb[0] != 0 && b != this_b) || (a.sb[1] != 0 && h1 - h0 > 1)) load_bias(b, head);
  }
  if (i >= m) return;
  T* out = (T*)a.dbias + pb * a.sdb[0] + ph * a.sdb[1] + i * a.sdb[2];
#pragma unroll
  for (int u = 0; u < kParts; ++u) store_keys(out, key + keys_at + 32 * u + 16 * h, a.n, sum[u]);
}

// out = the splits' parts added in order, loaded kAhead at a time: of dQ, or (blockIdx.y) of dK and dV.
template <typename T>
__global__ __launch_bounds__(256) void cross_attention_sum(const float* part, int splits, int64_t quads, T* out0, T* out1) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  T* out = blockIdx.y ? out1 : out0;
  if (at >= quads || !out) return;
  part += blockIdx.y * splits * quads * 4;
  constexpr int kAhead = 4;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < splits; s0 += kAhead) {
    f32x4 x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) x[u] = *(const f32x4*)(part + 4 * (min(s0 + u, splits - 1) * quads + at));
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (s0 + u >= splits) break;
      v += x[u];
    }
  }
  store4(out + 4 * at, v);
}

struct Split {
  int splits, size;
};

// Splits of a block's `units` (keys, or query tiles) by what they cost: rounds of blocks over the 256 compute units, where
// a lone block (one wave a SIMD) takes 1.4 times its share of a pair's time, against writing and adding the parts.
// whole: us of an unsplit block; part_bytes: of one split's parts. fp32, D = 48, 96 blocks of dQ over 1134 keys: 3 splits
// 74 us, 5 splits 53; D = 128, 32 blocks of dK and dV: 107 and 69; bf16, D = 64, 16 blocks of dK and dV: 37 and 30.
Split plan(int64_t blocks, int64_t units, int64_t least, int64_t round, double whole, double part_bytes) {
  Split best = {1, (int)std::max<int64_t>(units, 1)};
  double best_us = 0;
  for (int64_t want = 1; want == 1 || (want <= 512 / blocks + 3 && want * least <= units); ++want) {
    const int64_t size = std::max<int64_t>((units + want - 1) / want + round - 1, round) / round * round;
    const int64_t splits = std::max<int64_t>((units + size - 1) / size, 1), all = blocks * splits;
    const double rounds = all <= 256 ? 1.4 : (double)((all + 255) / 256);
    const double us = rounds * whole * std::min<double>(size, units) / (double)std::max<int64_t>(units, 1) +
                      (splits > 1 ? 4 + 2 * part_bytes * splits / 3e6 : 0);
    if (want == 1 || us < best_us) best = {(int)splits, (int)size}, best_us = us;
  }
  return best;
}
// A block's products over `flops` at what a compute unit reaches (fp32 110 TF/s of the whole card, bf16 700).
double block_us(int dtype, double flops) { return flops / (dtype == kF32 ? 110e6 : 700e6) * 256; }
Split plan_dq(int dtype, int64_t batch, int64_t kv_heads, int64_t rows, int64_t n, int64_t dim) {
  return plan((rows + 127) / 128 * batch * kv_heads, n, 128, 32, block_us(dtype, 6. * 128 * n * dim),
              4. * batch * kv_heads * rows * dim);
}
Split plan_dkv(int dtype, int64_t batch, int64_t kv_heads, int64_t group, int64_t m, int64_t n, int64_t dim) {
  const int64_t tiles = group * ((m + 31) / 32);
  return plan((n + 127) / 128 * batch * kv_heads, tiles, 3, 1, block_us(dtype, 8. * 128 * 32 * tiles * dim),
              8. * batch * kv_heads * n * dim);
}

// Floats of the workspace: delta, then the parts of dQ or of dK and dV, whichever is more.
int64_t workspace_floats(int dtype, int64_t batch, int64_t m, int64_t n, int64_t heads, int64_t kv_heads, int64_t dim,
                         int64_t* parts) {
  const int64_t group = heads / kv_heads, delta = (batch * m * heads + 3) / 4 * 4;
  const Split q = plan_dq(dtype, batch, kv_heads, group * m, n, dim);
  const Split kv = plan_dkv(dtype, batch, kv_heads, group, m, n, dim);
  const int64_t pq = q.splits > 1 ? q.splits * batch * m * heads * dim : 0;
  const int64_t pkv = kv.splits > 1 ? 2 * kv.splits * batch * n * kv_heads * dim : 0;
  if (parts) *parts = delta;
  return delta + (pq > pkv ? pq : pkv);
}

template <typename T, int DP>
int launch(CrossArgs& a, hipStream_t stream) {
  const int64_t lists = a.batch * a.kv_heads, key_blocks = (a.n + 127) / 128;
  a.row_blocks = (a.rows + 127) / 128;
  constexpr int dtype = sizeof(T) == 4 ? kF32 : kBF16;
  const Split q = plan_dq(dtype, a.batch, a.kv_heads, a.rows, a.n, a.dim);
  const Split kv = plan_dkv(dtype, a.batch, a.kv_heads, a.group, a.m, a.n, a.dim);
  const int64_t planes = (a.sdb[0] ? a.batch : 1) * (a.sdb[1] ? a.heads : 1);
  // Shared by batch elements or heads: a kernel of its own; otherwise dK and dV's writes it.
  const bool shared = a.dbias && ((!a.sdb[0] && a.batch > 1) || (!a.sdb[1] && a.heads > 1));
  constexpr int KT = kBiasKeys<T, DP>;
  const int64_t bias_blocks = planes * ((a.m + 127) / 128) * ((a.n + KT - 1) / KT);
  const int64_t delta_blocks = (a.batch * a.m * a.heads + 15) / 16;
  const int64_t q_quads = a.batch * a.m * a.heads * a.dim / 4, k_quads = a.batch * a.n * a.kv_heads * a.dim / 4;
  constexpr int64_t most = 1ll << 31, threads = 0xffffff00ll;
  BMX_REQUIRE(lists * a.row_blocks * q.splits < most && lists * key_blocks * kv.splits < most && bias_blocks < most &&
                  delta_blocks < most && (q.splits < 2 || q_quads < threads) && (kv.splits < 2 || k_quads < threads),
              "cross_attention_bwd: too many blocks");
  cross_attention_delta<T><<<fold_grid(delta_blocks, 256), 256, 0, stream>>>(a);
  auto sum = [&](const Split& s, int64_t quads, void* out0, void* out1) {
    const dim3 grid((unsigned)((quads + 255) / 256), out1 ? 2 : 1);
    if (s.splits > 1) cross_attention_sum<<<grid, 256, 0, stream>>>(a.part_o, s.splits, quads, (T*)out0, (T*)out1);
  };
  if (a.dq) {
    a.splits = q.splits, a.split_keys = q.size;
    a.blocks = (uint32_t)(lists * a.row_blocks * q.splits);
    const dim3 grid = fold_grid(a.blocks, 256);
    with_exact<T>(a, [&](auto exact) {
      constexpr bool kExact = decltype(exact)::value;
      a.bias ? cross_attention_dq<T, DP, true, kExact><<<grid, 256, 0, stream>>>(a)
             : cross_attention_dq<T, DP, false, kExact><<<grid, 256, 0, stream>>>(a);
    });
    sum(q, q_quads, a.dq, nullptr);
  }
  if (a.dk || a.dv || (a.dbias && !shared)) {
    a.splits = kv.splits, a.split_keys = kv.size;
    a.blocks = (uint32_t)(lists * key_blocks * kv.splits);
    const dim3 grid = fold_grid(a.blocks, 256);
    with_exact<T>(a, [&](auto exact) {
      constexpr bool kExact = decltype(exact)::value;
      if (a.dbias && !shared)
        cross_attention_dkv<T, DP, true, true, kExact><<<grid, 256, 0, stream>>>(a);
      else if (a.bias)
        cross_attention_dkv<T, DP, true, false, kExact><<<grid, 256, 0, stream>>>(a);
      else
        cross_attention_dkv<T, DP, false, false, kExact><<<grid, 256, 0, stream>>>(a);
    });
    sum(kv, k_quads, a.dk, a.dv);
  }
  if (shared) {
    constexpr int threads = 64 * kBiasWaves<T, DP>;
    a.blocks = (uint32_t)bias_blocks;
    cross_attention_dbias<T, DP><<<fold_grid(bias_blocks, threads), threads, 0, stream>>>(a);
  }
  return check_launch("cross_attention_bwd");
}

template <typename T>
int launch_dim(CrossArgs& a, hipStream_t stream) {
  const int dp = (a.dim + 31) / 32;
  return dp == 1 ? launch<T, 32>(a, stream) : dp == 2 ? launch<T, 64>(a, stream)
         : dp == 3 ? launch<T, 96>(a, stream) : launch<T, 128>(a, stream);
}

}  // namespace

extern "C" size_t bmx_cross_attention_bwd_workspace_bytes(int64_t batch, int64_t m, int64_t n, int64_t heads,
                                                          int64_t kv_heads, int64_t dim) {
  if (batch < 1 || m < 1 || n < 1 || heads < 1 || kv_heads < 1 || dim < 1) return 0;
  return (size_t)std::max(workspace_floats(kF32, batch, m, n, heads, kv_heads, dim, nullptr),
                          workspace_floats(kBF16, batch, m, n, heads, kv_heads, dim, nullptr)) *
         sizeof(float);
}

extern "C" int bmx_cross_attention_bwd(const void* q, const void* k, const void* v, const void* mask, const void* bias,
                                       int dtype, const int64_t* shape, const int64_t* strides, float scale,
                                       const void* out, const void* out_lo, const float* stats, const void* dout,
                                       void* dq, void* dk, void* dv, void* dbias, const int64_t* dbias_strides,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  CrossArgs a = {};
  if (int rc = cross_setup(a, dtype, shape, strides, scale, bias != nullptr)) return rc;
  BMX_REQUIRE(a.batch > 0 && a.rows > 0 && a.n > 0, "cross_attention_bwd: empty");
  BMX_REQUIRE(q && k && v && out && stats && dout, "cross_attention_bwd: null pointer");
  BMX_REQUIRE(dtype == kF32 || out_lo, "cross_attention_bwd: bf16 needs out_lo");
  BMX_REQUIRE(!dbias || (bias && dbias_strides), "cross_attention_bwd: dbias needs a bias and its strides");
  BMX_REQUIRE(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)out_lo | (uintptr_t)dout |
               (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) % 16 == 0,
              "cross_attention_bwd: tensors must be 16-byte aligned");
  BMX_REQUIRE((uintptr_t)stats % 8 == 0, "cross_attention_bwd: stats must be 8-byte aligned");
  BMX_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 &&
                  workspace_bytes >= bmx_cross_attention_bwd_workspace_bytes(a.batch, a.m, a.n, a.heads, a.kv_heads, a.dim),
              "cross_attention_bwd: workspace too small or not 16-byte aligned");
  a.q = q, a.k = k, a.v = v, a.mask = (const uint8_t*)mask, a.bias = bias;
  a.out = (void*)out, a.out_lo = dtype == kBF16 ? (void*)out_lo : nullptr, a.stats = (float2*)stats, a.dout = dout;
  int64_t parts = 0;
  workspace_floats(dtype, a.batch, a.m, a.n, a.heads, a.kv_heads, a.dim, &parts);
  a.part_o = (float*)workspace + parts;
  a.delta = (float*)workspace, a.dq = dq, a.dk = dk, a.dv = dv, a.dbias = dbias;
  for (int i = 0; i < 3; ++i) a.sdb[i] = dbias ? dbias_strides[i] : 0;
  hipStream_t hs = (hipStream_t)stream;
  return dtype == kF32 ? launch_dim<float>(a, hs) : launch_dim<bf16>(a, hs);
}
