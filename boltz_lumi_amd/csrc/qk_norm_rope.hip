// RMS norm of every query and key head and the rotation by position, one pass
// over both tensors, and its gradient.
//
//   y = R(pos) (x r w),  r = 1 / sqrt(mean(x^2) + eps)      per head vector x[D]
//   R turns the channel pairs (i, i + R) (or (2 i, 2 i + 1)) of the first 2 R
//   channels by pos * inv_freq[i]; the others pass.
//   g = R(-pos) dy:  dw = sum g x r,  dx = r (g w - x r mean(g w x r))
//
// A row of D values is held by L = 2^k >= D / 8 lanes, 8 values each: two runs
// of four, placed so that both members of a pair sit in one lane (4 p and
// R + 4 p for split pairs, 8 p and 8 p + 4 for adjacent ones): the rotation
// needs no exchange.  A lane group takes one token and kRows of its heads, so
// that its four angles are computed once for kRows rows.  The angle is
// pos * inv_freq in 64 bits, reduced to a fraction of a turn there and rounded
// to 32 bits after: a position of 10^6 loses nothing.  Sums are fp32, and there is one
// rounding, to the output's type.  The bound is HBM: 168 MB of bf16 (2 x 4096 tokens, 32 + 8 heads of 128) take
// 36 us, 4.7 TB/s (a copy of that size: 5.3); one token 4 us, a launch.
#include <type_traits>

#include "bmx_common.h"

using namespace bmx;

namespace {

constexpr int kBwdBlocks = 1024;  // of a tensor's gradient at most: four per compute unit

// One of the two tensors: x [batch, tokens, heads, D] at element strides, y dense.
struct HeadRows {
  const void *x, *w, *dy;
  void* y;          // forward: the result; backward: dx, or null
  float* partial;   // backward: [blocks][D] sums of g x r, or null
  const void* pos;
  int64_t sb, st, sh, pos_sb;
  int64_t tokens, items;  // tokens of a batch element; items = batch * tokens * chunks of heads
  int heads, chunks, blocks;
};
struct NormRope {
  HeadRows q, k;
  const void* inv_freq;
  int inv_freq64, pos64, w_bf16, dim, half, interleaved;
  float eps;
};

template <int L>
__device__ __forceinline__ float group_sum(float v) {
  if (L >= 2) v += dpp<0xB1>(v);
  if (L >= 4) v += dpp<0x4E>(v);
  if (L >= 8) v += dpp<0x141>(v);
  if (L >= 16) v += dpp<0x140>(v);
  if (L >= 32) v += __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(v), 0x401F));
  return v;
}

// A lane's 8 values: channels a .. a + 3 and b .. b + 3.
struct Eight {
  f32x4 a, b;
};
__device__ __forceinline__ float dot(const Eight& x, const Eight& y) {
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) v += x.a[i] * y.a[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) v += x.b[i] * y.b[i];
  return v;
}

struct Lane {
  int a, b;  // first channels of the lane's two runs of four
  bool live, turns;
  Eight w;
};

template <int L>
__device__ __forceinline__ Lane lane_channels(const NormRope& s, const void* w) {
  Lane c;
  const int p = threadIdx.x & (L - 1);
  c.live = 8 * p < s.dim;
  c.turns = 4 * p < s.half;
  const bool split = c.turns && !s.interleaved;
  c.a = c.live ? (split ? 4 * p : 8 * p) : 0;
  c.b = c.live ? (split ? s.half + 4 * p : 8 * p + 4) : 4;
  c.w.a = c.w.b = f32x4{1.f, 1.f, 1.f, 1.f};
  if (w) {
    c.w.a = s.w_bf16 ? load4((const bf16*)w + c.a) : load4((const float*)w + c.a);
    c.w.b = s.w_bf16 ? load4((const bf16*)w + c.b) : load4((const float*)w + c.b);
  }
  return c;
}

// cos and sin of the lane's four pairs at one token.
struct Angles {
  f32x4 c, s;
};
template <int L>
__device__ __forceinline__ Angles lane_angles(const NormRope& s, const HeadRows& t, const Lane& c, int64_t batch,
                                              int64_t token) {
  Angles out = {{1.f, 1.f, 1.f, 1.f}, {0.f, 0.f, 0.f, 0.f}};
  if (!c.turns) return out;
  const int64_t at = batch * t.pos_sb + token;
  const double pos = s.pos64 ? (double)((const int64_t*)t.pos)[at] : (double)((const int32_t*)t.pos)[at];
  const int f = 4 * (threadIdx.x & (L - 1));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double freq = s.inv_freq64 ? ((const double*)s.inv_freq)[f + i] : (double)((const float*)s.inv_freq)[f + i];
    double turn = pos * freq * 0.15915494309189533577;  // 1 / (2 pi)
    turn -= rint(turn);
    float sn, cs;
    sincospif(2.f * (float)turn, &sn, &cs);
    out.c[i] = cs, out.s[i] = sn;
  }
  return out;
}

// The rotation of a lane's 8 values; the transpose takes -s.
__device__ __forceinline__ Eight rotate(const NormRope& s, const Eight& v, const Angles& t) {
  if (!s.interleaved) return {v.a * t.c - v.b * t.s, v.a * t.s + v.b * t.c};
  Eight o;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    o.a[2 * i] = v.a[2 * i] * t.c[i] - v.a[2 * i + 1] * t.s[i];
    o.a[2 * i + 1] = v.a[2 * i] * t.s[i] + v.a[2 * i + 1] * t.c[i];
    o.b[2 * i] = v.b[2 * i] * t.c[2 + i] - v.b[2 * i + 1] * t.s[2 + i];
    o.b[2 * i + 1] = v.b[2 * i] * t.s[2 + i] + v.b[2 * i + 1] * t.c[2 + i];
  }
  return o;
}

// Lanes past the head's channels read its first ones and count as zeros.
template <typename T>
__device__ __forceinline__ Eight load8(const T* row, const Lane& c) {
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const f32x4 a = load4(row + c.a), b = load4(row + c.b);
  return {c.live ? a : zero, c.live ? b : zero};
}
template <typename T>
__device__ __forceinline__ void store8(T* row, const Lane& c, const Eight& v) {
  if (!c.live) return;
  store4(row + c.a, v.a);
  store4(row + c.b, v.b);
}

template <typename T, int L, int kRows>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(NormRope s) {
  const bool second = (int)blockIdx.x >= s.q.blocks;
  const HeadRows& t = second ? s.k : s.q;
  const int64_t item = ((int64_t)blockIdx.x - (second ? s.q.blocks : 0)) * (256 / L) + threadIdx.x / L;
  if (item >= t.items) return;  // whole groups leave; no exchange crosses a group
  const Lane c = lane_channels<L>(s, t.w);
  const int64_t row = item / t.chunks, batch = row / t.tokens, token = row % t.tokens;
  const int h0 = (int)(item % t.chunks) * kRows, last = t.heads - 1;
  const T* x = (const T*)t.x + batch * t.sb + token * t.st;
  T* y = (T*)t.y + row * t.heads * s.dim;
  Eight v[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) v[u] = load8(x + min(h0 + u, last) * t.sh, c);
  const Angles turn = lane_angles<L>(s, t, c, batch, token);
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const float r = 1.f / sqrtf(group_sum<L>(dot(v[u], v[u])) / (float)s.dim + s.eps);
    Eight n = {v[u].a * r * c.w.a, v[u].b * r * c.w.b};
    if (c.turns) n = rotate(s, n, turn);
    if (h0 + u <= last) store8(y + (h0 + u) * s.dim, c, n);
  }
}

// Gradient: the blocks of a tensor walk its items; each lane keeps the weight
// gradient of its 8 channels, the block's groups add theirs in a fixed order (79 MB of fp32: 18 us, 4.3 TB/s).
template <typename T, int L, int kRows>
__global__ __launch_bounds__(256) void qk_norm_rope_bwd_kernel(NormRope s) {
  __shared__ float sums[256 * 8];
  const bool second = (int)blockIdx.x >= s.q.blocks;
  const HeadRows& t = second ? s.k : s.q;
  const int block = (int)blockIdx.x - (second ? s.q.blocks : 0), groups = 256 / L;
  const Lane c = lane_channels<L>(s, t.w);
  Eight dw = {};
  for (int64_t item = (int64_t)block * groups + threadIdx.x / L; item < t.items;
       item += (int64_t)t.blocks * groups) {
    const int64_t row = item / t.chunks, batch = row / t.tokens, token = row % t.tokens;
    const int h0 = (int)(item % t.chunks) * kRows, last = t.heads - 1;
    const T* x = (const T*)t.x + batch * t.sb + token * t.st;
    const T* dy = (const T*)t.dy + row * t.heads * s.dim;
    T* dx = t.y ? (T*)t.y + row * t.heads * s.dim : nullptr;
    Eight v[kRows], g[kRows];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      v[u] = load8(x + min(h0 + u, last) * t.sh, c);
      g[u] = load8(dy + min(h0 + u, last) * s.dim, c);
    }
    Angles turn = lane_angles<L>(s, t, c, batch, token);
    turn.s = -turn.s;
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      if (h0 + u > last) continue;  // the same in every lane of a group
      if (c.turns) g[u] = rotate(s, g[u], turn);
      const float r = 1.f / sqrtf(group_sum<L>(dot(v[u], v[u])) / (float)s.dim + s.eps);
      const Eight n = {v[u].a * r, v[u].b * r};
      dw.a += g[u].a * n.a, dw.b += g[u].b * n.b;
      const Eight gw = {g[u].a * c.w.a, g[u].b * c.w.b};
      const float mean = group_sum<L>(dot(gw, n)) / (float)s.dim;
      if (dx) store8(dx + (h0 + u) * s.dim, c, Eight{r * (gw.a - n.a * mean), r * (gw.b - n.b * mean)});
    }
  }
  if (!t.partial) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sums[i * 256 + threadIdx.x] = dw.a[i];
    sums[(4 + i) * 256 + threadIdx.x] = dw.b[i];
  }
  __syncthreads();
  // thread (i, p): value i of lane p over the groups
  for (int at = threadIdx.x; at < 8 * L; at += 256) {
    const int i = at / L, p = at % L;
    if (8 * p >= s.dim) continue;
    float v = 0.f;
    for (int g = 0; g < groups; ++g) v += sums[i * 256 + g * L + p];
    const bool split = 4 * p < s.half && !s.interleaved;
    const int channel = split ? (i < 4 ? 4 * p + i : s.half + 4 * p + i - 4) : 8 * p + i;
    t.partial[(int64_t)block * s.dim + channel] = v;
  }
}

// Weight gradients of both tensors in one launch: a block per four channels, its 256 threads' partial rows
// in flight together, added over the lanes and then the waves.
struct WeightGrads {
  const float* partial[2];
  void* out[2];
  int blocks[2];  // partial rows
  int dim, out_bf16;
};
__global__ __launch_bounds__(256) void norm_weight_grad_kernel(WeightGrads s) {
  __shared__ float sums[4][4];
  const int quads = s.dim / 4, which = (int)blockIdx.x / quads, d = 4 * ((int)blockIdx.x % quads);
  if (!s.out[which]) return;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < kBwdBlocks / 256; ++u) {
    const int row = threadIdx.x + 256 * u;
    if (row < s.blocks[which]) v += *(const f32x4*)(s.partial[which] + (int64_t)row * s.dim + d);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float x = wave_sum_full(v[e]);
    if (lane_id() == 0) sums[threadIdx.x >> 6][e] = x;
  }
  __syncthreads();
  if (threadIdx.x >= 4) return;
  const float x = sums[0][threadIdx.x] + sums[1][threadIdx.x] + sums[2][threadIdx.x] + sums[3][threadIdx.x];
  if (s.out_bf16)
    ((bf16*)s.out[which])[d + threadIdx.x] = (bf16)x;
  else
    ((float*)s.out[which])[d + threadIdx.x] = x;
}


// Items of a tensor at `rows` heads per item, and its blocks (at most `most`).
int64_t plan(HeadRows& t, int64_t batch, int rows, int groups, int64_t most) {
  t.chunks = (t.heads + rows - 1) / rows;
  t.items = batch * t.tokens * t.chunks;
  const int64_t blocks = (t.items + groups - 1) / groups;
  t.blocks = (int)(blocks < most ? blocks : most);
  return blocks;
}

int lanes_of(int64_t dim) {
  int lanes = 1;
  while (8 * lanes < dim) lanes *= 2;
  return lanes;
}

template <typename T, int kRows>
void launch(bool backward, int lanes, const NormRope& s, hipStream_t stream) {
  const dim3 grid(s.q.blocks + s.k.blocks);
  auto go = [&](auto L) {
    constexpr int l = decltype(L)::value;
    if (backward)
      qk_norm_rope_bwd_kernel<T, l, kRows><<<grid, 256, 0, stream>>>(s);
    else
      qk_norm_rope_kernel<T, l, kRows><<<grid, 256, 0, stream>>>(s);
  };
  switch (lanes) {
    case 1: return go(std::integral_constant<int, 1>());
    case 2: return go(std::integral_constant<int, 2>());
    case 4: return go(std::integral_constant<int, 4>());
    case 8: return go(std::integral_constant<int, 8>());
    case 16: return go(std::integral_constant<int, 16>());
    default: return go(std::integral_constant<int, 32>());
  }
}

// Checks shared by both directions; fills everything but the tensors' pointers.
int setup(NormRope& s, int dtype, const int64_t* shape, const int64_t* strides, int w_dtype, int pos64,
          const void* inv_freq, int inv_freq64, int64_t half, int interleaved, float eps) {
  BMX_REQUIRE(dtype == kF32 || dtype == kBF16, "qk_norm_rope: dtype must be fp32 or bf16");
  BMX_REQUIRE(w_dtype == kF32 || w_dtype == kBF16, "qk_norm_rope: weight dtype must be fp32 or bf16");
  BMX_REQUIRE(shape && strides, "qk_norm_rope: null shape or strides");
  for (int i = 0; i < 6; ++i) BMX_REQUIRE(shape[i] >= 0, "qk_norm_rope: negative size");
  const int64_t dim = shape[5];
  BMX_REQUIRE(dim >= 8 && dim <= 256 && dim % 8 == 0, "qk_norm_rope: head dim must be a multiple of 8 in [8, 256]");
  BMX_REQUIRE(half >= 0 && half % 4 == 0 && 2 * half <= dim,
              "qk_norm_rope: the rotated pairs must be a multiple of 4, at most half the head dim");
  BMX_REQUIRE(half == 0 || inv_freq, "qk_norm_rope: null inv_freq");
  BMX_REQUIRE(eps >= 0x1p-126f, "qk_norm_rope: eps must be positive, at least 2^-126");  // below it is flushed to zero
  BMX_REQUIRE(shape[3] < (1 << 20) && shape[4] < (1 << 20), "qk_norm_rope: too many heads");
  for (int i = 0; i < 6; ++i) BMX_REQUIRE(strides[i] % 4 == 0, "qk_norm_rope: strides must be multiples of 4");
  s.inv_freq = inv_freq, s.inv_freq64 = inv_freq64, s.pos64 = pos64, s.w_bf16 = w_dtype == kBF16;
  s.dim = (int)dim, s.half = (int)half, s.interleaved = interleaved, s.eps = eps;
  s.q.tokens = shape[1], s.k.tokens = shape[2];
  s.q.heads = (int)shape[3], s.k.heads = (int)shape[4];
  s.q.sb = strides[0], s.q.st = strides[1], s.q.sh = strides[2], s.q.pos_sb = strides[6];
  s.k.sb = strides[3], s.k.st = strides[4], s.k.sh = strides[5], s.k.pos_sb = strides[7];
  return BMX_OK;
}

int check_tensor(const HeadRows& t, int64_t batch, int64_t half, int elem, bool backward) {
  if (batch * t.tokens * t.heads == 0) return BMX_OK;
  BMX_REQUIRE(t.x && (backward ? t.dy : t.y) && (half == 0 || t.pos), "qk_norm_rope: null pointer");
  const uintptr_t bits = (uintptr_t)t.x | (uintptr_t)t.y | (uintptr_t)t.dy | (uintptr_t)t.w;
  BMX_REQUIRE(bits % (4 * elem) == 0 && (uintptr_t)t.w % 16 == 0,
              "qk_norm_rope: tensors must be aligned to four elements, weights to 16 bytes");
  return BMX_OK;
}

}  // namespace

extern "C" int bmx_qk_norm_rope_fwd(const void* q, const void* k, int dtype, const int64_t* shape,
                                    const int64_t* strides, const void* q_weight, const void* k_weight, int w_dtype,
                                    const void* q_pos, const void* k_pos, int pos64, const void* inv_freq,
                                    int inv_freq64, int64_t half, int interleaved, float eps, void* q_out, void* k_out,
                                    void* stream) {
  NormRope s = {};
  if (int rc = setup(s, dtype, shape, strides, w_dtype, pos64, inv_freq, inv_freq64, half, interleaved, eps)) return rc;
  s.q.x = q, s.q.w = q_weight, s.q.pos = q_pos, s.q.y = q_out;
  s.k.x = k, s.k.w = k_weight, s.k.pos = k_pos, s.k.y = k_out;
  const int64_t batch = shape[0];
  const int elem = dtype == kF32 ? 4 : 2;
  if (int rc = check_tensor(s.q, batch, half, elem, false)) return rc;
  if (int rc = check_tensor(s.k, batch, half, elem, false)) return rc;
  const int lanes = lanes_of(s.dim), groups = 256 / lanes;
  // Four heads share a token's angles; a few tokens take one head a group, for the latency of one.
  const int64_t rows = batch * (s.q.tokens * s.q.heads + s.k.tokens * s.k.heads);
  const bool few = rows * lanes < 256 * 1024;
  const int64_t most = (1 << 24) - 1;  // a launch takes fewer than 2^32 threads
  const int64_t total = plan(s.q, batch, few ? 1 : 4, groups, most) + plan(s.k, batch, few ? 1 : 4, groups, most);
  BMX_REQUIRE(total <= most, "qk_norm_rope: too many rows");
  if (total == 0) return BMX_OK;
  hipStream_t hs = (hipStream_t)stream;
  if (dtype == kF32)
    few ? launch<float, 1>(false, lanes, s, hs) : launch<float, 4>(false, lanes, s, hs);
  else
    few ? launch<bf16, 1>(false, lanes, s, hs) : launch<bf16, 4>(false, lanes, s, hs);
  return check_launch("qk_norm_rope");
}

extern "C" size_t bmx_qk_norm_rope_workspace_bytes(int64_t dim) {
  return dim > 0 ? (size_t)2 * kBwdBlocks * dim * sizeof(float) : 0;
}

extern "C" int bmx_qk_norm_rope_bwd(const void* q, const void* k, int dtype, const int64_t* shape,
                                    const int64_t* strides, const void* q_weight, const void* k_weight, int w_dtype,
                                    const void* q_pos, const void* k_pos, int pos64, const void* inv_freq,
                                    int inv_freq64, int64_t half, int interleaved, float eps, const void* dq_out,
                                    const void* dk_out, void* dq, void* dk, void* dq_weight, void* dk_weight,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  NormRope s = {};
  if (int rc = setup(s, dtype, shape, strides, w_dtype, pos64, inv_freq, inv_freq64, half, interleaved, eps)) return rc;
  s.q.x = q, s.q.w = q_weight, s.q.pos = q_pos, s.q.dy = dq_out, s.q.y = dq;
  s.k.x = k, s.k.w = k_weight, s.k.pos = k_pos, s.k.dy = dk_out, s.k.y = dk;
  if (!dq && !dq_weight) s.q.tokens = 0;  // a tensor without a gradient to write takes no part
  if (!dk && !dk_weight) s.k.tokens = 0;
  const int64_t batch = shape[0];
  const int elem = dtype == kF32 ? 4 : 2;
  if (int rc = check_tensor(s.q, batch, half, elem, true)) return rc;
  if (int rc = check_tensor(s.k, batch, half, elem, true)) return rc;
  BMX_REQUIRE(!(dq_weight && !q_weight) && !(dk_weight && !k_weight), "qk_norm_rope: gradient of an absent weight");
  if (dq_weight || dk_weight)
    BMX_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 &&
                    workspace_bytes >= bmx_qk_norm_rope_workspace_bytes(s.dim),
                "qk_norm_rope: workspace too small or not 16-byte aligned");
  s.q.partial = dq_weight ? (float*)workspace : nullptr;
  s.k.partial = dk_weight ? (float*)workspace + (int64_t)kBwdBlocks * s.dim : nullptr;
  const int lanes = lanes_of(s.dim), groups = 256 / lanes;
  const int64_t rows = batch * (s.q.tokens * s.q.heads + s.k.tokens * s.k.heads);
  const bool few = rows * lanes < 256 * 1024;
  plan(s.q, batch, few ? 1 : 4, groups, kBwdBlocks);
  plan(s.k, batch, few ? 1 : 4, groups, kBwdBlocks);
  hipStream_t hs = (hipStream_t)stream;
  if (s.q.blocks + s.k.blocks > 0) {
    if (dtype == kF32)
      few ? launch<float, 1>(true, lanes, s, hs) : launch<float, 4>(true, lanes, s, hs);
    else
      few ? launch<bf16, 1>(true, lanes, s, hs) : launch<bf16, 4>(true, lanes, s, hs);
  }
  if (dq_weight || dk_weight) {  // without rows: no partial rows, a gradient of zeros
    const WeightGrads w = {{s.q.partial, s.k.partial}, {dq_weight, dk_weight}, {s.q.blocks, s.k.blocks}, s.dim,
                           w_dtype == kBF16};
    norm_weight_grad_kernel<<<dim3(s.dim / 4 * 2), 256, 0, hs>>>(w);
  }
  return check_launch("qk_norm_rope_bwd");
}
