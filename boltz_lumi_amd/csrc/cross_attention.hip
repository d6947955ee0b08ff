// Softmax attention of one sequence's queries over another's keys and values,
// with a key mask, an additive bias and key / value heads shared by groups of
// query heads (bf16 or fp32, head dims up to 128).
//
//   S = scale q k^T + bias, masked keys left out;  out = softmax(S) v
//
// One pass over the keys with a running maximum and sum (fp32).  A wave holds 32 query
// rows: S^T = K Q^T puts a query in a lane, so maximum and sum are one lane's
// registers plus one exchange between the halves, and the weights in registers are the next product's
// operand as they stand (out^T += V^T P^T, V read transposed from LDS).  The
// weights are rounded to the operand's type (small elements: to two of them), and their sum is taken over the rounded
// values, so a row's weights add up to one: the error is a rounding of each weight against the others.
//
// A row without keys (masked, or -inf bias throughout) gives zeros.
#include <algorithm>
#include <type_traits>

#include "cross_attention.h"

using namespace bmx;

namespace {

// State of a wave's 32 rows: lane l holds row l % 32, in both halves.
template <typename T, int DP, bool kBias, bool kExact>
struct Rows {
  // The weight of a logit x (without a bias q k^T, with one the logit in natural units): see the reference point.
  static constexpr bool kFirst = sizeof(T) == 4;
  RowOperand<T, DP> q;
  RowReads<T, DP> kr;
  ColumnReads<T, DP> vr;
  f32x16 o[DP / 32];
  float top, sum;  // maximum that the weights refer to; this half's share of their sum
  float limit;     // the maximum moves when a logit passes this
  float shift;     // of the exponent: -S, or (fp32) top
  float c;         // logits to base 2, or the unit of rows far from zero
  const T* bias;
  bool odd;  // some bias rows start at an odd element

  __device__ __forceinline__ void init(const CrossArgs& a, int64_t b, int kv, int row) {
    const int r = min(row, a.rows - 1), g = r / (int)a.m, i = r - g * (int)a.m;
    const int64_t head = (int64_t)kv * a.group + g;
    q.load((const T*)a.q + b * a.sq[0] + i * a.sq[1] + head * a.sq[2], a.dim, lane_id() >> 5);
    bias = (const T*)a.bias + b * a.sb[0] + head * a.sb[1] + i * a.sb[2];
    kr.init(a.dim);
    vr.init();
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt) o[dt] = zero16();
    top = limit = -INFINITY, sum = shift = 0.f;
    c = (kBias ? 1.f : a.scale) * kLog2E;
    odd = bias_odd(a);
  }

  // 32 keys: rows of the tiles, presence bits, bias.
  __device__ __forceinline__ void attend(const CrossArgs& a, const char* kt, const char* vt, uint32_t bits,
                                         BiasTile<T>& b) {
    f32x16 s = product<T, DP>(kt, kr, q);
    if (kBias) {
      b.ready(odd);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = s[r] * a.scale + b.at(r);
    }
    if (bits != ~0u) {
      const uint32_t mine = bits >> (16 * (lane_id() >> 5));
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!key_bit(mine, r)) s[r] = -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
    // bf16 moves the maximum (and scales the sums) only when a logit passes it by 2^6: the weights' rounding is relative, and
    // their sums stay far inside fp32. After the first tiles that hardly happens, so the halves' exchange, the
    // factor and the products with it are off the common path.
    if (__any(mx > limit)) {
      mx = fmaxf(halves_max(mx), top);
      const float base = mx == -INFINITY ? 0.f : mx, c0 = (kBias ? 1.f : a.scale) * kLog2E;
      const float f = rescale<T>(top, base, c0);
      sum *= f;
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) o[dt] *= f;
      top = mx;
      if (!kFirst) c = logit_unit(base, c0);
      limit = kFirst ? mx : mx + 6.f / c;
      shift = kFirst ? base : -reference_shift(base, c);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(kFirst ? (s[r] - shift) * c : s[r] * c + shift);
    weighted_sum<T, DP, kExact>(vt, vr, s, o, &sum);
  }
};

// Four channels of a row, rounded; and what the rounding left, for the gradient's row sums.
template <typename T>
__device__ __forceinline__ void store_out(const CrossArgs& a, int64_t at, f32x4 v);
template <>
__device__ __forceinline__ void store_out<bf16>(const CrossArgs& a, int64_t at, f32x4 v) {
  bf16x4 hi, lo;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    hi[e] = (bf16)v[e];
    lo[e] = (bf16)(v[e] - (float)hi[e]);
  }
  *(bf16x4*)((bf16*)a.out + at) = hi;
  if (a.out_lo) *(bf16x4*)((bf16*)a.out_lo + at) = lo;
}
template <>
__device__ __forceinline__ void store_out<float>(const CrossArgs& a, int64_t at, f32x4 v) {
  *(f32x4*)((float*)a.out + at) = v;
}

// A row without keys. A row whose logits are all NaN has no maximum either, but a sum that is NaN, and stays NaN.
__device__ __forceinline__ bool no_keys(float top, float sum) { return top == -INFINITY && sum == sum; }

// Reference point and log2 of the sum against it; a row without keys gets weights exp2(-inf) = 0.
template <typename T>
__device__ __forceinline__ float2 row_stats(float top, float sum, float c0) {
  if (no_keys(top, sum)) return make_float2(0.f, INFINITY);
  float log = __builtin_amdgcn_logf(sum);
  if (sizeof(T) == 2) {  // bf16's sum is against S, which is off top c by what its rounding left
    const float c = logit_unit(top, c0);
    log += fmaf(-top, c, reference_shift(top, c));
  }
  return make_float2(top, log);
}

// The lane's row of a wave's result: to out (and stats), or as a partial sum of its split.
template <typename T, int DP>
__device__ __forceinline__ void write_rows(const CrossArgs& a, int64_t b, int c, int split, int row,
                                           const f32x16 (&o)[DP / 32], float top, float sum, float c0) {
  if (row >= a.rows) return;
  const int h = lane_id() >> 5;
  if (a.splits > 1) {
    const int64_t at = ((int64_t)split * a.batch * a.kv_heads + b * a.kv_heads + c) * a.rows + row;
    if (h == 0) a.part_ml[at] = make_float2(top, sum);
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * dt + 8 * g + 4 * h;
        if (d < a.dim)
          *(f32x4*)(a.part_o + at * a.dim + d) = f32x4{o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
      }
    return;
  }
  const int g0 = row / (int)a.m, i = row - g0 * (int)a.m;
  const int64_t head = (int64_t)c * a.group + g0;
  const int64_t at = ((b * a.m + i) * a.heads + head) * a.dim;
  const bool none = no_keys(top, sum);
  const float f = none ? 0.f : 1.f / sum;
  if (a.stats && h == 0) a.stats[(b * a.heads + head) * a.m + i] = row_stats<T>(top, sum, c0);
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * dt + 8 * g + 4 * h;
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = none ? 0.f : o[dt][4 * g + e] * f;
      if (d < a.dim) store_out<T>(a, at + d, v);
    }
}

// Position of a block: row block, split, key head, batch element.
struct Place {
  int row_block, split, c, first, stop;  // keys of the split
  int64_t b;
  __device__ __forceinline__ Place(const CrossArgs& a) {
    uint32_t at = xcd_position(block_index(), a.blocks);
    b = a.batch_first ? take(at, a.batch) : 0;
    row_block = take(at, a.row_blocks), split = take(at, a.splits), c = take(at, a.kv_heads);
    if (!a.batch_first) b = at;
    first = split * a.split_keys;
    stop = min(first + a.split_keys, a.n);
  }
};

// Many rows: four waves of 32 rows share tiles of 32 keys in two LDS buffers, copied there by DMA: the next tile's
// copies are in flight while a tile is attended, one barrier per tile. No staging registers and small tiles leave room
// for two to four blocks on a compute unit, so one wave's exponentials run under another's MFMA. Tiles without a
// present key are passed over. Bound: D = 128 by the MFMA (batch 2, 32 / 8 heads, 2048 x 4096: 300 us, 920 TF/s;
// blocks of two waves, three waves a SIMD, or a wave of its own for the copies took 377 to 440), narrower heads by the
// exponentials and conversions between the products (D = 64: 2 x 16 heads, 2048 x 4096, 90 us, 765 TF/s; 6 x 32 heads
// 477 us, 865), with a bias by those and the bias's reads. Heads of 24 and 48 run as 32 and 64 do (2 x 16 heads: 91 and
// 88 us).
template <typename T, int DP, bool kBias, bool kExact>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DP > 64 ? 1 : sizeof(T) == 4 || kBias || DP == 128 ? 2 : 3)
void cross_attention_wide(CrossArgs a) {
  constexpr int kTile = 32 * Tile<T, DP>::kRowBytes;
  __shared__ __attribute__((aligned(16))) char lds[4 * kTile + kMaskChunk / 8];
  if (block_index() >= a.blocks) return;
  const Place p(a);
  const int t = threadIdx.x, w = __builtin_amdgcn_readfirstlane(t >> 6), row = (p.row_block * 4 + w) * 32 + (t & 31);
  Rows<T, DP, kBias, kExact> rows;
  rows.init(a, p.b, p.c, row);
  const T* k = (const T*)a.k + p.b * a.sk[0] + p.c * a.sk[2];
  const T* v = (const T*)a.v + p.b * a.sv[0] + p.c * a.sv[2];
  KeyWords words{(uint32_t*)(lds + 4 * kTile), a.mask ? a.mask + p.b * a.smask : nullptr};
  Copy<T, DP, 32, 4> ck, cv;
  ck.init(w, a.dim, a.sk[1]);
  cv.init(w, a.dim, a.sv[1]);
  const unsigned lds0 = lds_address(lds);
  clear_tiles<T, DP, 256>(t, lds, 4 * kTile, a.dim);
  const int chunk = a.mask ? kMaskChunk : p.stop - p.first;  // c0 + chunk stays below 2^31, as the keys do
  for (int c0 = p.first; c0 < p.stop; c0 += chunk) {
    words.fill(c0, p.stop);  // its barrier also ends the last chunk's reads of the tiles
    const int end = min(c0 + chunk, p.stop);
    auto copy = [&](int key, unsigned tile) {
      ck.issue(w, k + key * a.sk[1], a.n - key, a.dim, a.sk[1], tile);
      cv.issue(w, v + key * a.sv[1], a.n - key, a.dim, a.sv[1], tile + kTile);
    };
    int key = words.next(c0, end);
    BiasTile<T> bias[2];
    // One tile in the buffer at B; false after the last.
    auto step = [&](auto B) {
      constexpr int kAt = decltype(B)::value * 2 * kTile, kOther = 2 * kTile - kAt;
      const uint32_t bits = words.bits(key);
      const int after = words.next(key + 32, end);
      wait_copies();
      __syncthreads();
      if (after < end) {
        copy(after, lds0 + kOther);
        if (kBias) bias[1 - decltype(B)::value].load(rows.bias, after, a.n);
      }
      if (bits != ~0u) {  // what a left-out value holds must not meet its weight of zero
        clear_rows<T, DP, 32, 256>(t, lds + kAt + kTile, bits);
        __syncthreads();
      }
      rows.attend(a, lds + kAt, lds + kAt + kTile, bits, bias[decltype(B)::value]);
      key = after;
      return key < end;
    };
    if (key < end) {
      copy(key, lds0);
      if (kBias) bias[0].load(rows.bias, key, a.n);
      while (step(std::integral_constant<int, 0>()) && step(std::integral_constant<int, 1>())) {
      }
    }
  }
  write_rows<T, DP>(a, p.b, p.c, p.split, row, rows.o, rows.top, halves_sum(rows.sum),
                    (kBias ? 1.f : a.scale) * kLog2E);
}

// Up to kFewRows rows (a decoding step): the four waves take 32 keys in turn, each through a tile of its own without
// barriers, so every wave keeps its next 32 keys' loads in flight, and merge their sums at the end. The bound
// is the read of the keys and values (batch 32, 32 / 8 heads, 4096 keys of 128 channels, 537 MB: 102 us, 5.3 TB/s).
template <typename T, int DP, bool kBias>
__global__ __launch_bounds__(256, sizeof(T) == 4 || DP == 128 ? 1 : DP == 96 ? 2 : DP == 64 ? 3 - kBias : 4)
void cross_attention_few(CrossArgs a) {
  constexpr int kTile = 32 * Tile<T, DP>::kRowBytes;
  __shared__ __attribute__((aligned(16))) char lds[8 * kTile + kMaskChunk / 8 + 4 * 32 * 4];
  if (block_index() >= a.blocks) return;
  const Place p(a);
  const int t = threadIdx.x, w = t >> 6, l = t & 63, row = l & 31;
  Rows<T, DP, kBias, sizeof(T) == 2> rows;
  rows.init(a, p.b, p.c, row);
  const T* k = (const T*)a.k + p.b * a.sk[0] + p.c * a.sk[2];
  const T* v = (const T*)a.v + p.b * a.sv[0] + p.c * a.sv[2];
  char* kt = lds + w * 2 * kTile;
  KeyWords words{(uint32_t*)(lds + 8 * kTile), a.mask ? a.mask + p.b * a.smask : nullptr};
  Stage<T, DP, 32, 64> sk, sv;
  sk.init(l, a.dim, a.sk[1]);
  sv.init(l, a.dim, a.sv[1]);
  for (int c0 = p.first; c0 < p.stop; c0 += kMaskChunk) {
    words.fill(c0, p.stop);
    const int end = min(c0 + kMaskChunk, p.stop);
    auto next = [&](int key) {
      while (key < end && words.bits(key) == 0) key += 128;
      return key;
    };
    auto load = [&](int key) {
      sk.load(l, k + key * a.sk[1], a.n - key, a.dim, a.sk[1]);
      sv.load(l, v + key * a.sv[1], a.n - key, a.dim, a.sv[1]);
    };
    int key = next(c0 + 32 * w);
    BiasTile<T> bias, ahead;
    if (key < end) {
      load(key);
      if (kBias) ahead.load(rows.bias, key, a.n);
    }
    while (key < end) {
      const uint32_t bits = words.bits(key);
      sk.store(l, kt, bits, a.dim);
      sv.store(l, kt + kTile, bits, a.dim);
      bias = ahead;
      const int after = next(key + 128);
      if (after < end) {
        load(after);
        if (kBias) ahead.load(rows.bias, after, a.n);
      }
      wave_order();
      rows.attend(a, kt, kt + kTile, bits, bias);
      wave_order();
      key = after;
    }
  }
  // Merge: the common maximum, then the waves' sums and outputs added in order.
  float* ml = (float*)(lds + 8 * kTile + kMaskChunk / 8);  // [4][32] maxima
  float sum = halves_sum(rows.sum);
  if (l < 32) ml[w * 32 + row] = rows.top;
  __syncthreads();  // also: every wave is done with its tiles
  float top = ml[row];
#pragma unroll
  for (int i = 1; i < 4; ++i) top = fmaxf(top, ml[i * 32 + row]);
  const float base = top == -INFINITY ? 0.f : top;
  const float c0 = (kBias ? 1.f : a.scale) * kLog2E, f = rescale<T>(rows.top, base, c0);  // 0 for a wave without keys
  sum *= f;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt) rows.o[dt] *= f;
  // Waves 1 .. 3 leave [register][lane] values; wave 0 adds them.
  float* part = (float*)lds;
  constexpr int kPart = (DP / 2 + 1) * 64;
  static_assert(3 * kPart * 4 <= 8 * kTile, "the merge fits the tiles");
  if (w > 0) {
    float* mine = part + (w - 1) * kPart;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) mine[(16 * dt + r) * 64 + l] = rows.o[dt][r];
    mine[(DP / 2) * 64 + l] = sum;
  }
  __syncthreads();
  if (w > 0) return;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const float* other = part + i * kPart;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) rows.o[dt][r] += other[(16 * dt + r) * 64 + l];
    sum += other[(DP / 2) * 64 + l];
  }
  write_rows<T, DP>(a, p.b, p.c, p.split, row, rows.o, top, sum, c0);
}

// Joins the splits: a thread per four channels of a row.
template <typename T>
__global__ __launch_bounds__(256) void cross_attention_join(CrossArgs a, int bias) {
  const int quads = a.dim / 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, lists = a.batch * a.kv_heads;
  const int64_t at = id / quads;  // (batch, key head, row)
  if (at >= lists * a.rows) return;
  const int d = (int)(id - at * quads) * 4;
  const int64_t step = lists * a.rows;
  // Loads go out kAhead splits at a time (those past the last repeat it, unused): one after another, 32
  // splits of a few rows took longer than the attention itself.
  constexpr int kAhead = 8;
  float top = -INFINITY;
  for (int s0 = 0; s0 < a.splits; s0 += kAhead) {
    float x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) x[u] = a.part_ml[min(s0 + u, a.splits - 1) * step + at].x;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) top = fmaxf(top, x[u]);
  }
  const float c0 = (bias ? 1.f : a.scale) * kLog2E, base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < a.splits; s0 += kAhead) {
    float2 ml[kAhead];
    f32x4 part[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t i = min(s0 + u, a.splits - 1) * step + at;
      ml[u] = a.part_ml[i];
      part[u] = *(const f32x4*)(a.part_o + i * a.dim + d);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (s0 + u >= a.splits) break;
      const float f = rescale<T>(ml[u].x, base, c0);
      sum += ml[u].y * f;
      o += part[u] * f;
    }
  }
  const int64_t list = at / a.rows, b = list / a.kv_heads;
  const int row = (int)(at - list * a.rows), g = row / (int)a.m, i = row - g * (int)a.m;
  const int64_t head = (list - b * a.kv_heads) * a.group + g;
  const bool none = no_keys(top, sum);
  if (a.stats && d == 0) a.stats[(b * a.heads + head) * a.m + i] = row_stats<T>(top, sum, c0);
  const float f = none ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = none ? 0.f : o[e] * f;
  store_out<T>(a, ((b * a.m + i) * a.heads + head) * a.dim + d, o);
}

struct Split {
  bool few;
  int row_blocks, splits;
  int keys;  // per split, a multiple of 128
};

// Few rows run as many splits as give every compute unit a block, each of at least 128 keys (one tile a wave), past 16
// splits 512, since a short split costs less than joining another (one query, 32 / 8 heads, D = 128, 4096 keys: 32 splits
// 23.8 us, 16 splits 18.6; batch 8: two blocks a compute unit 36 us, one 30).
// Many rows split where their blocks leave compute units idle, or, for a second wave on every SIMD, where the keys
// are many enough to pay for writing and joining the parts (bf16, 256 blocks, D = 64: 1024 keys 26 us whole and
// 30 in two, 4096 keys 77 and 57; fp32's keys cost several times as much: 96 blocks of 1134 keys 63 in two, 50 in five).
Split plan(int dtype, int64_t batch, int64_t kv_heads, int64_t rows, int64_t n) {
  Split s;
  s.few = rows <= kFewRows;
  s.row_blocks = s.few ? 1 : (int)((rows + 127) / 128);
  const int64_t blocks = (int64_t)s.row_blocks * batch * kv_heads;
  auto fill = [&](int64_t want, int64_t least) { return blocks ? std::min(want / blocks, (n + least - 1) / least) : 1; };
  int64_t splits = s.few ? std::min<int64_t>(fill(256, 128), std::max<int64_t>(16, fill(256, 512)))
                   : dtype == kF32 ? fill(512, 256) : std::max(fill(256, 256), fill(512, 1024));
  if (splits < 1) splits = 1;
  s.keys = (int)(((n + splits - 1) / splits + 127) / 128 * 128);
  if (s.keys == 0) s.keys = 128;
  s.splits = (int)(n > 0 ? (n + s.keys - 1) / s.keys : 1);
  return s;
}

template <typename T, int DP, bool kBias>
void launch(const CrossArgs& a, bool few, hipStream_t stream) {
  const dim3 grid = fold_grid(a.blocks, 256);
  if (few) {
    cross_attention_few<T, DP, kBias><<<grid, 256, 0, stream>>>(a);
  } else {
    with_exact<T>(a, [&](auto exact) {
      cross_attention_wide<T, DP, kBias, decltype(exact)::value><<<grid, 256, 0, stream>>>(a);
    });
  }
}

template <typename T>
void launch_dim(const CrossArgs& a, bool few, hipStream_t stream) {
  const int dp = (a.dim + 31) / 32;
  if (a.bias) {
    dp == 1 ? launch<T, 32, true>(a, few, stream) : dp == 2 ? launch<T, 64, true>(a, few, stream)
    : dp == 3 ? launch<T, 96, true>(a, few, stream) : launch<T, 128, true>(a, few, stream);
  } else {
    dp == 1 ? launch<T, 32, false>(a, few, stream) : dp == 2 ? launch<T, 64, false>(a, few, stream)
    : dp == 3 ? launch<T, 96, false>(a, few, stream) : launch<T, 128, false>(a, few, stream);
  }
}

}  // namespace

namespace bmx {

int cross_setup(CrossArgs& a, int dtype, const int64_t* shape, const int64_t* strides, float scale, bool has_bias) {
  BMX_REQUIRE(dtype == kF32 || dtype == kBF16, "cross_attention: dtype must be fp32 or bf16");
  BMX_REQUIRE(shape && strides, "cross_attention: null shape or strides");
  for (int i = 0; i < 6; ++i) BMX_REQUIRE(shape[i] >= 0, "cross_attention: negative size");
  BMX_REQUIRE(shape[2] < (1ll << 31) - (1 << 20), "cross_attention: too many keys");
  a.batch = shape[0], a.m = shape[1], a.n = (int)shape[2];
  const int64_t heads = shape[3], kv = shape[4], dim = shape[5];
  BMX_REQUIRE(dim >= 8 && dim <= 128 && dim % 8 == 0, "cross_attention: head dim must be a multiple of 8 in [8, 128]");
  BMX_REQUIRE(heads >= 1 && heads <= 65536 && kv >= 1 && heads % kv == 0,
              "cross_attention: the query heads must be a multiple of the key heads");
  const int64_t rows = heads / kv * a.m;
  BMX_REQUIRE(a.batch < (1ll << 31) && a.m < (1ll << 31) && rows < (1ll << 30), "cross_attention: too many query rows");
  // Its product with log2(e) is a number that fp32 holds to all its bits (denormals are flushed).
  BMX_REQUIRE(scale >= 0x1p-126f && scale <= 0x1p127f, "cross_attention: scale must be in [2^-126, 2^127]");
  const int vec = dtype == kF32 ? 4 : 8;
  for (int i = 0; i < 3; ++i) {
    a.sq[i] = strides[i], a.sk[i] = strides[3 + i], a.sv[i] = strides[6 + i], a.sb[i] = has_bias ? strides[10 + i] : 0;
    BMX_REQUIRE(a.sq[i] % vec == 0 && a.sk[i] % vec == 0 && a.sv[i] % vec == 0,
                "cross_attention: strides must be multiples of 16 bytes");
  }
  BMX_REQUIRE(a.sq[1] >= 0 && a.sk[1] >= 0 && a.sv[1] >= 0 && a.sq[1] < kMaxStride && a.sk[1] < kMaxStride &&
                  a.sv[1] < kMaxStride && heads * dim < kMaxStride,
              "cross_attention: token strides must be below 2^22 elements");
  BMX_REQUIRE(a.sb[2] >= 0 && a.sb[2] < (1ll << 26), "cross_attention: the bias's query stride must be below 2^26 elements");
  a.smask = strides[9];
  a.heads = (int)heads, a.kv_heads = (int)kv, a.group = (int)(heads / kv), a.dim = (int)dim, a.rows = (int)rows;
  a.scale = scale;
  // The weights' rounding moves a result by as much as its own rounding does, and over few keys the output's error does not
  // average out before the gradients' differences dP - delta meet it. Weights of 16 bits leave the result's rounding alone:
  // in decoding steps, which are bound by reading the keys (batch 32, 32 / 8 heads, 4096 keys, D = 128: 95.7 us with 8
  // bits, 96.6 with 16; 16 heads, 2048 keys, D = 64: 45.7 and 47.3, D = 32 with a bias, the worst, 26.6 and 31.8),
  // and where an element's products are few, whatever the batch: its neighbours must not decide its error, and one such
  // element alone is mostly latency (300 queries, 500 keys, 16 heads, D = 64: forward 15.4 and 16.1 us, dQ, dK and dV 23.5
  // and 26.5). Large batches of them pay for the added products (32 of that size: forward 42 and 51 us, dQ 50 and 60, dK
  // and dV 75 and 91; 16 x 250 queries, 500 keys, 16 / 4 heads, D = 128: 31 and 36, 37 and 42, 57 and 92), as calls over up
  // to 256 keys do (2048 queries, D = 128: dK and dV 46 and 55), where the few weights' errors average out least. Large
  // elements would pay as much on top of more work, and their rows have the most keys to average over.
  a.exact = dtype == kBF16 && (rows <= kFewRows || a.n <= 256 || (double)heads * a.m * a.n * dim <= 1ll << 28);
  a.batch_first = has_bias && a.batch > 1 && a.sb[0] == 0;
  return BMX_OK;
}

}  // namespace bmx

extern "C" size_t bmx_cross_attention_workspace_bytes(int dtype, int64_t batch, int64_t m, int64_t n, int64_t heads,
                                                      int64_t kv_heads, int64_t dim) {
  if (batch < 1 || m < 1 || n < 1 || heads < 1 || kv_heads < 1 || dim < 1) return 0;
  const int64_t rows = heads / kv_heads * m;
  const Split s = plan(dtype, batch, kv_heads, rows, n);
  return s.splits < 2 ? 0 : (size_t)(s.splits * batch * kv_heads * rows) * (dim + 2) * sizeof(float);
}

extern "C" int bmx_cross_attention_fwd(const void* q, const void* k, const void* v, const void* mask, const void* bias,
                                       int dtype, const int64_t* shape, const int64_t* strides, float scale, void* out,
                                       void* out_lo, float* stats, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  CrossArgs a = {};
  if (int rc = cross_setup(a, dtype, shape, strides, scale, bias != nullptr)) return rc;
  if (a.batch == 0 || a.rows == 0) return BMX_OK;
  BMX_REQUIRE(q && out && (a.n == 0 || (k && v)), "cross_attention: null pointer");
  BMX_REQUIRE(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)out_lo) % 16 == 0,
              "cross_attention: q, k, v and out must be 16-byte aligned");
  BMX_REQUIRE(!stats || (uintptr_t)stats % 8 == 0, "cross_attention: stats must be 8-byte aligned");
  const Split s = plan(dtype, a.batch, a.kv_heads, a.rows, a.n);
  const size_t need = bmx_cross_attention_workspace_bytes(dtype, a.batch, a.m, a.n, a.heads, a.kv_heads, a.dim);
  BMX_REQUIRE(need == 0 || (workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need),
              "cross_attention: workspace too small or not 16-byte aligned");
  a.q = q, a.k = k, a.v = v, a.mask = (const uint8_t*)mask, a.bias = bias;
  a.out = out, a.out_lo = dtype == kBF16 ? out_lo : nullptr, a.stats = (float2*)stats;
  a.row_blocks = s.row_blocks, a.splits = s.splits, a.split_keys = s.keys;
  const int64_t lists = (int64_t)s.splits * a.batch * a.kv_heads;
  const int64_t threads = a.batch * a.kv_heads * a.rows * (a.dim / 4);  // of the join
  BMX_REQUIRE(lists * s.row_blocks < (1ll << 31) && (s.splits < 2 || threads < 0xffffff00ll),
              "cross_attention: too many blocks");
  a.blocks = (uint32_t)(lists * s.row_blocks);
  a.part_o = (float*)workspace;
  a.part_ml = (float2*)((float*)workspace + lists * a.rows * a.dim);
  hipStream_t hs = (hipStream_t)stream;
  dtype == kF32 ? launch_dim<float>(a, s.few, hs) : launch_dim<bf16>(a, s.few, hs);
  if (s.splits > 1) {
    const dim3 grid((unsigned)((threads + 255) / 256));
    if (dtype == kF32)
      cross_attention_join<float><<<grid, 256, 0, hs>>>(a, bias != nullptr);
    else
      cross_attention_join<bf16><<<grid, 256, 0, hs>>>(a, bias != nullptr);
  }
  return check_launch("cross_attention");
}
