// Gradients of cross attention (cross_attention.hip), from the row statistics
// that the forward pass kept:
//
//   P = exp(S - max) / sum;  dV = P^T dO;  dP = dO V^T;  delta = rowsum(dO O)
//   dS = P (dP - delta);  dQ = scale dS K;  dK = scale dS^T Q;  dbias = dS summed over its shared axes
//
// No logits are kept: each kernel recomputes S and dP for its tiles.  Three
// kernels instead of one, because each sums over another axis and keeps its sum in
// registers: no atomics, and the same bits on every run.  P and dS are rounded to
// the operand's type for the products over them; delta is taken from the output before its rounding
// (out + out_lo), so that dP - delta cancels as it does in the formula.
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
  const int64_t at = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4), total = a.batch * a.m * a.heads;
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

// P of a logits tile whose column is a query: maximum and log2 of the sum are the lane's.
template <typename T, bool kBias>
__device__ __forceinline__ void weights_of(const CrossArgs& a, f32x16& s, const T* bias, int64_t key, float2 st) {
  if (kBias) {
    const f32x16 b = bias_tile(bias, min(key, a.n - 1), a.n);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f((s[r] * a.scale + b[r] - st.x) * kLog2E - st.y);
  } else if (sizeof(T) == 4) {  // as the forward pass: the difference first
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f((s[r] * a.scale - st.x) * kLog2E - st.y);
  } else {
    const float c = a.scale * kLog2E, shift = -(st.x * kLog2E + st.y);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] * c + shift);
  }
}

template <typename T>
constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;

// dQ: four waves of 32 rows over all keys, as the forward pass runs.
template <typename T, int DP, bool kBias>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 64 ? 1 : 2) void cross_attention_dq(CrossArgs a) {
  constexpr int KT = kKeys<T>, kTile = KT * Tile<T, DP>::kRowBytes;
  __shared__ __attribute__((aligned(16))) char lds[4 * kTile + kMaskChunk / 8];
  int64_t at = xcd_position(blockIdx.x, gridDim.x);
  const int row_block = (int)(at % a.row_blocks);
  at /= a.row_blocks;
  const int c = (int)(at % a.kv_heads);
  const int64_t b = at / a.kv_heads;
  const int t = threadIdx.x, row = row_block * 128 + (t >> 6) * 32 + (t & 31), h = lane_id() >> 5;
  const RowAt ra(a, c, row);
  RowOperand<T, DP> q, g;
  q.load((const T*)a.q + ra.q(a, b), a.dim, h);
  g.load((const T*)a.dout + ra.dense(a, b), a.dim, h);
  const float2 st = a.stats[ra.stat(a, b)];
  const float delta = a.delta[ra.stat(a, b)];
  const T* bias = (const T*)a.bias + ra.bias(a, b);
  f32x16 dq[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) dq[dt] = zero16();
  const T* k = (const T*)a.k + b * a.sk[0] + c * a.sk[2];
  const T* v = (const T*)a.v + b * a.sv[0] + c * a.sv[2];
  KeyWords words{(uint64_t*)(lds + 4 * kTile), a.mask ? a.mask + b * a.smask : nullptr};
  Stage<T, DP, KT, 256> sk, sv;
  int buf = 0;
  for (int64_t c0 = 0; c0 < a.n; c0 += kMaskChunk) {
    words.fill(c0, a.n);
    const int64_t end = min(c0 + kMaskChunk, a.n);
    auto next = [&](int64_t key) {
      while (key < end && words.bits(key, KT) == 0) key += KT;
      return key;
    };
    auto load = [&](int64_t key) {
      sk.load(t, a.dim, [&](int r) { return k + min(key + r, a.n - 1) * a.sk[1]; });
      sv.load(t, a.dim, [&](int r) { return v + min(key + r, a.n - 1) * a.sv[1]; });
    };
    int64_t key = next(c0);
    if (key < end) load(key);
    while (key < end) {
      const uint64_t bits = words.bits(key, KT);
      char* kt = lds + buf * 2 * kTile;
      auto live = [&](int r) { return (bits >> r) & 1; };
      sk.store(t, a.dim, kt, live);
      sv.store(t, a.dim, kt + kTile, live);
      const int64_t after = next(key + KT);
      if (after < end) load(after);
      __syncthreads();
#pragma unroll
      for (int u = 0; u < KT / 32; ++u) {
        const uint32_t sub = (uint32_t)(bits >> (32 * u));
        f32x16 s = product<T, DP>(kt, 32 * u, q, zero16());
        const f32x16 dp = product<T, DP>(kt + kTile, 32 * u, g, zero16());
        weights_of<T, kBias>(a, s, bias, key + 32 * u, st);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= dp[r] - delta;
        if (sub != 0xffffffffu) {
          const uint32_t mine = sub >> (4 * h);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!key_bit(mine, r)) s[r] = 0.f;
        }
        Weights<T> w;
        w.set(s);
        transposed_product<DP>(kt, 32 * u, w, dq);
      }
      buf ^= 1, key = after;
    }
  }
  if (row >= a.rows) return;
  T* out = (T*)a.dq + ra.dense(a, b);
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) store_rows(out, a.dim, dq[dt], dt, a.scale, true);
}

// dK and dV: four waves of 32 keys (in the lanes, their K and V in registers) over all rows of the group's
// heads in tiles of 32, so a shared key head's gradient is one sum in row order.
template <typename T, int DP, bool kBias>
__global__ __launch_bounds__(256, DP > 64 ? 1 : 2) void cross_attention_dkv(CrossArgs a) {
  constexpr bool kFirst = kBias || sizeof(T) == 4;
  constexpr int kTile = 32 * Tile<T, DP>::kRowBytes;
  constexpr int kStat = 32 * 3 * 4 + 32 * 8;  // maximum (or the whole shift), log2 of the sum, delta; bias offset
  __shared__ __attribute__((aligned(16))) char lds[4 * kTile + 2 * kStat + kMaskChunk / 8];
  const int key_blocks = (int)((a.n + 127) / 128);
  int64_t at = xcd_position(blockIdx.x, gridDim.x);
  const int64_t first = (at % key_blocks) * 128;
  at /= key_blocks;
  const int c = (int)(at % a.kv_heads);
  const int64_t b = at / a.kv_heads;
  const int t = threadIdx.x, l = lane_id(), h = l >> 5;
  const int64_t key = first + (t >> 6) * 32 + (l & 31), safe = min(key, a.n - 1);
  KeyWords words{(uint64_t*)(lds + 4 * kTile + 2 * kStat), a.mask ? a.mask + b * a.smask : nullptr};
  words.fill(first, min(first + 128, a.n));
  const uint64_t lo = words.bits(first, 64), hi = words.bits(first + 64, 64);
  const bool live = ((t >> 7 ? hi : lo) >> (t >> 6 & 1 ? 32 + (l & 31) : l & 31)) & 1;
  RowOperand<T, DP> kf, vf;
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) dk[dt] = zero16(), dv[dt] = zero16();
  if ((lo | hi) != 0) {
    kf.load((const T*)a.k + b * a.sk[0] + safe * a.sk[1] + c * a.sk[2], a.dim, h);
    vf.load((const T*)a.v + b * a.sv[0] + safe * a.sv[1] + c * a.sv[2], a.dim, h);
    Stage<T, DP, 32, 256> sq, sg;
    float2 st;
    float delta;
    int64_t bias_at;
    auto load = [&](int row0) {
      sq.load(t, a.dim, [&](int r) { return (const T*)a.q + RowAt(a, c, row0 + r).q(a, b); });
      sg.load(t, a.dim, [&](int r) { return (const T*)a.dout + RowAt(a, c, row0 + r).dense(a, b); });
      if (t < 32) {
        const RowAt ra(a, c, row0 + t);
        st = a.stats[ra.stat(a, b)], delta = a.delta[ra.stat(a, b)];
        if (kBias) bias_at = ra.bias(a, b);
        if (row0 + t >= a.rows) st = make_float2(0.f, INFINITY), delta = 0.f;
      }
    };
    load(0);
    int buf = 0;
    for (int row0 = 0; row0 < a.rows; row0 += 32, buf ^= 1) {
      char* qt = lds + buf * 2 * kTile;
      char* gt = qt + kTile;
      float* stat = (float*)(lds + 4 * kTile + buf * kStat);
      int64_t* offs = (int64_t*)(stat + 96);
      auto in = [&](int r) { return row0 + r < a.rows; };
      sq.store(t, a.dim, qt, in);
      sg.store(t, a.dim, gt, in);
      if (t < 32) {
        stat[t] = kFirst ? st.x : st.x * kLog2E + st.y;
        stat[32 + t] = st.y;
        stat[64 + t] = delta;
        if (kBias) offs[t] = bias_at;
      }
      if (row0 + 32 < a.rows) load(row0 + 32);
      __syncthreads();
      f32x16 s = product<T, DP>(qt, 0, kf, zero16());
      const f32x16 dp = product<T, DP>(gt, 0, vf, zero16());
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 top = *(const f32x4*)(stat + 8 * g + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          if (kFirst) {
            const float x = kBias ? (float)((const T*)a.bias)[offs[8 * g + 4 * h + e] + safe] : 0.f;
            s[r] = __builtin_amdgcn_exp2f((s[r] * a.scale + x - top[e]) * kLog2E - stat[32 + 8 * g + 4 * h + e]);
          } else {
            s[r] = __builtin_amdgcn_exp2f(s[r] * (a.scale * kLog2E) - top[e]);
          }
        }
      }
      Weights<T> w;
      w.set(s);
      transposed_product<DP>(gt, 0, w, dv);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 dl = *(const f32x4*)(stat + 64 + 8 * g + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * g + e] *= dp[4 * g + e] - dl[e];
      }
      w.set(s);
      transposed_product<DP>(qt, 0, w, dk);
    }
  }
  if (key >= a.n) return;
  const int64_t out = ((b * a.n + key) * a.kv_heads + c) * a.dim;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) {
    if (a.dk) store_rows((T*)a.dk + out, a.dim, dk[dt], dt, a.scale, live);
    if (a.dv) store_rows((T*)a.dv + out, a.dim, dv[dt], dt, 1.f, live);
  }
}

// dbias: a block holds 128 queries x 64 (fp32: 32) keys of one bias plane in registers and walks the batch elements and
// heads that share the plane, in order.
template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 64 ? 1 : 2) void cross_attention_dbias(CrossArgs a) {
  constexpr int KT = kKeys<T>, kTile = KT * Tile<T, DP>::kRowBytes;
  __shared__ __attribute__((aligned(16))) char lds[4 * kTile + kMaskChunk / 8];
  const int key_blocks = (int)((a.n + KT - 1) / KT), query_blocks = (int)((a.m + 127) / 128);
  int64_t at = xcd_position(blockIdx.x, gridDim.x);
  const int64_t key = (at % key_blocks) * KT;
  at /= key_blocks;
  const int q0 = (int)(at % query_blocks) * 128;
  at /= query_blocks;
  const int plane_heads = a.sdb[1] ? a.heads : 1;
  const int64_t ph = at % plane_heads, pb = at / plane_heads;
  const int64_t b0 = a.sdb[0] ? pb : 0, b1 = a.sdb[0] ? pb + 1 : a.batch;
  const int h0 = a.sdb[1] ? (int)ph : 0, h1 = a.sdb[1] ? (int)ph + 1 : a.heads;
  const int t = threadIdx.x, h = lane_id() >> 5;
  const int64_t i = q0 + (t >> 6) * 32 + (t & 31), safe = min(i, a.m - 1);
  f32x16 sum[KT / 32];
#pragma unroll
  for (int u = 0; u < KT / 32; ++u) sum[u] = zero16();
  KeyWords words{(uint64_t*)(lds + 4 * kTile), nullptr};
  Stage<T, DP, KT, 256> sk, sv;
  int buf = 0;
  for (int64_t b = b0; b < b1; ++b) {
    words.mask = a.mask ? a.mask + b * a.smask : nullptr;
    words.fill(key, min(key + KT, a.n));
    const uint64_t bits = words.bits(key, KT);
    if (bits == 0) continue;
    for (int head = h0; head < h1; ++head) {
      const int c = head / a.group;
      const T* k = (const T*)a.k + b * a.sk[0] + c * a.sk[2];
      const T* v = (const T*)a.v + b * a.sv[0] + c * a.sv[2];
      sk.load(t, a.dim, [&](int r) { return k + min(key + r, a.n - 1) * a.sk[1]; });
      sv.load(t, a.dim, [&](int r) { return v + min(key + r, a.n - 1) * a.sv[1]; });
      RowOperand<T, DP> q, g;
      q.load((const T*)a.q + b * a.sq[0] + safe * a.sq[1] + head * a.sq[2], a.dim, h);
      g.load((const T*)a.dout + ((b * a.m + safe) * a.heads + head) * a.dim, a.dim, h);
      const int64_t stat = (b * a.heads + head) * a.m + safe;
      const float2 st = a.stats[stat];
      const float delta = a.delta[stat];
      const T* bias = (const T*)a.bias + b * a.sb[0] + head * a.sb[1] + safe * a.sb[2];
      char* kt = lds + buf * 2 * kTile;
      auto live = [&](int r) { return (bits >> r) & 1; };
      sk.store(t, a.dim, kt, live);
      sv.store(t, a.dim, kt + kTile, live);
      __syncthreads();
#pragma unroll
      for (int u = 0; u < KT / 32; ++u) {
        const uint32_t mine = (uint32_t)(bits >> (32 * u)) >> (4 * h);
        f32x16 s = product<T, DP>(kt, 32 * u, q, zero16());
        const f32x16 dp = product<T, DP>(kt + kTile, 32 * u, g, zero16());
        weights_of<T, true>(a, s, bias, key + 32 * u, st);
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[u][r] += key_bit(mine, r) ? s[r] * (dp[r] - delta) : 0.f;
      }
      buf ^= 1;
    }
  }
  if (i >= a.m) return;
  T* out = (T*)a.dbias + pb * a.sdb[0] + ph * a.sdb[1] + i * a.sdb[2];
#pragma unroll
  for (int u = 0; u < KT / 32; ++u)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int64_t at_key = key + 32 * u + 8 * (r >> 2) + 4 * h + (r & 3);
      if (at_key < a.n) out[at_key] = (T)sum[u][r];
    }
}

template <typename T, int DP>
int launch(CrossArgs& a, hipStream_t stream) {
  const int64_t lists = a.batch * a.kv_heads, key_blocks = (a.n + 127) / 128;
  a.row_blocks = (a.rows + 127) / 128;
  const int64_t planes = (a.sdb[0] ? a.batch : 1) * (a.sdb[1] ? a.heads : 1);
  const int64_t bias_blocks = planes * ((a.m + 127) / 128) * ((a.n + kKeys<T> - 1) / kKeys<T>);
  const int64_t delta_blocks = (a.batch * a.m * a.heads + 15) / 16;
  BMX_REQUIRE(lists * a.row_blocks < (1ll << 31) && lists * key_blocks < (1ll << 31) && bias_blocks < (1ll << 31) &&
                  delta_blocks < (1ll << 31),
              "cross_attention_bwd: too many blocks");
  cross_attention_delta<T><<<dim3((unsigned)delta_blocks), 256, 0, stream>>>(a);
  if (a.dq) {
    const dim3 grid((unsigned)(lists * a.row_blocks));
    a.bias ? cross_attention_dq<T, DP, true><<<grid, 256, 0, stream>>>(a)
           : cross_attention_dq<T, DP, false><<<grid, 256, 0, stream>>>(a);
  }
  if (a.dk || a.dv) {
    const dim3 grid((unsigned)(lists * key_blocks));
    a.bias ? cross_attention_dkv<T, DP, true><<<grid, 256, 0, stream>>>(a)
           : cross_attention_dkv<T, DP, false><<<grid, 256, 0, stream>>>(a);
  }
  if (a.dbias) cross_attention_dbias<T, DP><<<dim3((unsigned)bias_blocks), 256, 0, stream>>>(a);
  return check_launch("cross_attention_bwd");
}

template <typename T>
int launch_dim(CrossArgs& a, hipStream_t stream) {
  const int dp = (a.dim + 31) / 32;
  return dp == 1 ? launch<T, 32>(a, stream) : dp == 2 ? launch<T, 64>(a, stream)
         : dp == 3 ? launch<T, 96>(a, stream) : launch<T, 128>(a, stream);
}

}  // namespace

extern "C" size_t bmx_cross_attention_bwd_workspace_bytes(int64_t batch, int64_t m, int64_t heads) {
  return batch < 1 || m < 1 || heads < 1 ? 0 : (size_t)(batch * m * heads) * sizeof(float);
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
                  workspace_bytes >= bmx_cross_attention_bwd_workspace_bytes(a.batch, a.m, a.heads),
              "cross_attention_bwd: workspace too small or not 16-byte aligned");
  a.q = q, a.k = k, a.v = v, a.mask = (const uint8_t*)mask, a.bias = bias;
  a.out = (void*)out, a.out_lo = dtype == kBF16 ? (void*)out_lo : nullptr, a.stats = (float2*)stats, a.dout = dout;
  a.delta = (float*)workspace, a.dq = dq, a.dk = dk, a.dv = dv, a.dbias = dbias;
  for (int i = 0; i < 3; ++i) a.sdb[i] = dbias ? dbias_strides[i] : 0;
  hipStream_t hs = (hipStream_t)stream;
  return dtype == kF32 ? launch_dim<float>(a, hs) : launch_dim<bf16>(a, hs);
}
