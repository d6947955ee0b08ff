// Short causal convolution of every channel on its own, with SiLU, and its
// gradient.
//
//   p[t] = bias + sum_j weight[j] x[t - (W - 1) + j],  y = p sigmoid(p)
//   dp = dy s (1 + p (1 - s));  dx[t] = sum_j weight[j] dp[t + W - 1 - j]
//   dweight[j] = sum dp[t] x[t - (W - 1) + j];  dbias = sum dp
//
// Before the first token stand the W - 1 rows of `state` (or zeros); the last
// W - 1 rows before a sequence's end are the next call's state.  Rows from a
// sequence's length on are never read and give zeros.
//
// A thread takes 16 bytes of channels (8 bf16, 4 fp32) of a run of kRun tokens
// with all its rows in flight at once; the W - 1 rows before (backward: and
// behind) a run come from the neighbours' cache lines.  Sums are fp32.
//
// Bound by HBM forward in fp32 (16001 x 768: 17 us, 5.7 TB/s, part of it cached).
// In bf16 (4 x 2048 x 1536, ragged: 44.7 MB in 15 us, 2.9 TB/s) by neither HBM nor
// instructions (6 of the 15): 768 blocks are three a compute unit, one round, in
// which loads, arithmetic and stores follow each other.  Backward (the same: 32 us,
// 17 of them instructions, and 4 for the partial rows) by the loads that the
// registers let be in flight: two waves a SIMD, 25 rows asked for per 16 that are
// needed.  32 single tokens: 4 us.
#include <type_traits>
#include <utility>

#include "bmx_common.h"

using namespace bmx;

namespace {

constexpr int kRun = 8;       // tokens of a thread (4 x 2048 x 1536: 15 us; with 16 23, with 4 15.5)
constexpr int kBwdVec = 4, kBwdRun = 8;
constexpr int kBwdVecs = 32;  // a gradient's block: 32 runs of channels by 8 runs of tokens

template <typename F, int... I>
__device__ __forceinline__ void each_of(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int kCount, typename F>
__device__ __forceinline__ void each_of(F f) {
  each_of(f, std::make_integer_sequence<int, kCount>());
}

struct Conv {
  const void *x, *w, *bias, *state, *lengths, *dy, *dnext;
  void *y, *next, *dx, *dstate;
  float* partial;  // [parts][W + 1][channels]
  int64_t sb, st, tokens, batch;
  int64_t blocks;
  int channels, vecs, runs, lengths64, silu, w_bf16, b_bf16;
};

// V channels of one token as they lie in memory, and as fp32.
template <typename T, int V>
struct Run {
  typedef T Vec __attribute__((ext_vector_type(V)));
  Vec v;
  __device__ __forceinline__ float operator[](int i) const { return (float)v[i]; }
};
template <int V>
struct Vals {
  float v[V];
};
template <typename T, int V>
__device__ __forceinline__ void put(T* p, const Vals<V>& a) {
  Run<T, V> o;
#pragma unroll
  for (int i = 0; i < V; ++i) o.v[i] = (T)a.v[i];
  *(Run<T, V>*)p = o;
}

__device__ __forceinline__ int64_t length_of(const void* lengths, int lengths64, int64_t b, int64_t tokens) {
  if (!lengths) return tokens;
  const int64_t n = lengths64 ? ((const int64_t*)lengths)[b] : (int64_t)((const int32_t*)lengths)[b];
  return n < 0 ? 0 : n < tokens ? n : tokens;
}

// The taps of a thread's channels and the bias: weight is [channels][W], V W values in a row.
template <int W, int V>
struct Taps {
  float w[V][W], b[V];
  template <typename T, int kCount>
  static __device__ __forceinline__ void load(const void* from, int at, float* to) {
#pragma unroll
    for (int i = 0; i < kCount; i += 4) {
      const f32x4 q = load4((const T*)from + at + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) to[i + k] = q[k];
    }
  }
  __device__ __forceinline__ Taps(const Conv& s, int c) {
    if (s.w_bf16)
      load<bf16, V * W>(s.w, c * W, &w[0][0]);
    else
      load<float, V * W>(s.w, c * W, &w[0][0]);
#pragma unroll
    for (int i = 0; i < V; ++i) b[i] = 0.f;
    if (s.bias) s.b_bf16 ? load<bf16, V>(s.bias, c, b) : load<float, V>(s.bias, c, b);
  }
};

// Row t of a sequence: the state's rows before token 0, zeros from its length on.
template <typename T, int W, int V>
__device__ __forceinline__ Run<T, V> input_row(const Conv& s, int64_t b, int64_t t, int64_t length, int c) {
  Run<T, V> o = {};
  if (t >= length) return o;
  if (t >= 0)
    o = *(const Run<T, V>*)((const T*)s.x + b * s.sb + t * s.st + c);
  else if (s.state)
    o = *(const Run<T, V>*)((const T*)s.state + (b * (W - 1) + t + W - 1) * s.channels + c);
  return o;
}

template <typename T, int W, int V, int R>
__global__ __launch_bounds__(256) void causal_conv_kernel(Conv s) {
  const int64_t item = (int64_t)block_index() * 256 + threadIdx.x;
  const int64_t row = item / s.vecs, b = row / s.runs;
  if (b >= s.batch) return;
  const int c = (int)(item - row * s.vecs) * V;
  const int64_t t0 = (row - b * s.runs) * R, length = length_of(s.lengths, s.lengths64, b, s.tokens);
  Run<T, V> raw[R + W - 1];
#pragma unroll
  for (int i = 0; i < R + W - 1; ++i) raw[i] = input_row<T, W, V>(s, b, t0 + i - (W - 1), length, c);
  if (s.next && t0 == 0) {
    // The thread of the first tokens alone looks at the state, so that the next one may take its place.
    Run<T, V> last[W - 1];
#pragma unroll
    for (int i = 0; i < W - 1; ++i) last[i] = input_row<T, W, V>(s, b, length + i - (W - 1), length, c);
#pragma unroll
    for (int i = 0; i < W - 1; ++i) *(Run<T, V>*)((T*)s.next + (b * (W - 1) + i) * s.channels + c) = last[i];
  }
  const Taps<W, V> taps(s, c);
  T* y = (T*)s.y + (b * s.tokens + t0) * s.channels + c;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (t0 + i >= s.tokens) break;
    Vals<V> p;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      p.v[e] = taps.b[e];
#pragma unroll
      for (int j = 0; j < W; ++j) p.v[e] += taps.w[e][j] * raw[i + j][e];
      if (s.silu) p.v[e] = silu_f(p.v[e]);
      if (t0 + i >= length) p.v[e] = 0.f;
    }
    put<T, V>(y + (int64_t)i * s.channels, p);
  }
}

// Gradient: a thread works dp out for its run and the W - 1 tokens behind it, four channels (eight of bf16 need more
// registers than two waves a SIMD have: 50 us for 16 at 4 x 2048 x 1536).  Its eight token-run neighbours add their sums
// for the weights in LDS; a block leaves one partial row per weight.
template <typename T, int W>
__global__ __launch_bounds__(256) void causal_conv_bwd_kernel(Conv s) {
  constexpr int V = kBwdVec, R = kBwdRun, kRows = 256 / kBwdVecs;
  __shared__ __align__(16) f32x4 sums[kRows][kBwdVecs];
  const int64_t block = block_index();
  if (block >= s.blocks) return;
  const int cblocks = (s.vecs + kBwdVecs - 1) / kBwdVecs, tblocks = (s.runs + kRows - 1) / kRows;
  const int64_t part = block / cblocks, b = part / tblocks;
  const int v = threadIdx.x % kBwdVecs, group = threadIdx.x / kBwdVecs;
  const int vec = (int)(block % cblocks) * kBwdVecs + v;
  const int64_t t0 = ((part % tblocks) * kRows + group) * R;
  const bool live = vec < s.vecs && t0 < s.tokens;
  const int c = live ? vec * V : 0;
  const int64_t length = live ? length_of(s.lengths, s.lengths64, b, s.tokens) : 0;
  Run<T, V> raw[R + 2 * (W - 1)], back[R + W - 1];
#pragma unroll
  for (int i = 0; i < R + 2 * (W - 1); ++i) raw[i] = input_row<T, W, V>(s, b, t0 + i - (W - 1), length, c);
#pragma unroll
  for (int i = 0; i < R + W - 1; ++i) {
    back[i] = {};
    if (s.dy && t0 + i < length) back[i] = *(const Run<T, V>*)((const T*)s.dy + (b * s.tokens + t0 + i) * s.channels + c);
  }
  const Taps<W, V> taps(s, c);
  f32x4 dw[W + 1];
#pragma unroll
  for (int j = 0; j <= W; ++j) dw[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  Vals<V> dp[R + W - 1];
#pragma unroll
  for (int i = 0; i < R + W - 1; ++i) {
    const bool there = t0 + i < length;  // a row that is not there has dp 0, whatever an infinite p does
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float d = back[i][e];
      if (s.silu) {
        float p = taps.b[e];
#pragma unroll
        for (int j = 0; j < W; ++j) p += taps.w[e][j] * raw[i + j][e];
        const float sg = sigmoid_f(p);
        d *= sg + p * sg * (1.f - sg);
      }
      dp[i].v[e] = there ? d : 0.f;
      if (i < R) {
#pragma unroll
        for (int j = 0; j < W; ++j) dw[j][e] += there ? d * raw[i + j][e] : 0.f;
        dw[W][e] += dp[i].v[e];
      }
    }
  }
  // dx of row t (the state's rows where t < 0): the taps that it went into, and its place in the next state.
  auto dx_row = [&](auto index, int64_t t, T* to) {  // index: dp's of row t
    constexpr int i = decltype(index)::value;
    Vals<V> dx;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      dx.v[e] = 0.f;
#pragma unroll
      for (int j = 0; j < W; ++j)
        if (i + W - 1 - j >= 0) dx.v[e] += taps.w[e][j] * dp[i + W - 1 - j >= 0 ? i + W - 1 - j : 0].v[e];
    }
    const int64_t at = t - (length - (W - 1));
    if (s.dnext && at >= 0 && at < W - 1) {
      const Run<T, V> d = *(const Run<T, V>*)((const T*)s.dnext + (b * (W - 1) + at) * s.channels + c);
#pragma unroll
      for (int e = 0; e < V; ++e) dx.v[e] += d[e];
    }
    put<T, V>(to, dx);
  };
  if (live && s.dx) {
    T* dx = (T*)s.dx + (b * s.tokens + t0) * s.channels + c;
    each_of<R>([&](auto i) {
      if (t0 + i < s.tokens) dx_row(i, t0 + i, dx + (int64_t)i * s.channels);
    });
  }
  if (live && s.dstate && t0 == 0)
    each_of<W - 1>([&](auto i) {
      dx_row(std::integral_constant<int, decltype(i)::value - (W - 1)>(), i - (W - 1),
             (T*)s.dstate + (b * (W - 1) + i) * s.channels + c);
    });
  if (!s.partial) return;
#pragma unroll
  for (int j = 0; j <= W; ++j) {
    __syncthreads();
    sums[group][v] = live ? dw[j] : f32x4{0.f, 0.f, 0.f, 0.f};
    __syncthreads();
    if (group == 0 && vec < s.vecs) {
      f32x4 total = sums[0][v];
#pragma unroll
      for (int g = 1; g < kRows; ++g) total += sums[g][v];
      *(f32x4*)(s.partial + (part * (W + 1) + j) * s.channels + vec * V) = total;
    }
  }
}

// Sums of the partial rows: a block per 16 channels of one tap (the last: the bias), 16 threads over the rows of each.
struct ConvSums {
  const float* partial;
  void *dw, *db;
  int64_t parts;
  int channels, width, w_bf16, b_bf16;
};
__global__ __launch_bounds__(256) void causal_conv_sums_kernel(ConvSums s) {
  __shared__ float lds[16][17];
  const int j = blockIdx.y, col = threadIdx.x % 16, slice = threadIdx.x / 16, c = (int)blockIdx.x * 16 + col;
  float v = 0.f;
  if (c < s.channels)
    for (int64_t row = slice; row < s.parts; row += 16) v += s.partial[(row * (s.width + 1) + j) * s.channels + c];
  lds[slice][col] = v;
  __syncthreads();
  if (slice || c >= s.channels) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) v += lds[i][col];
  void* out = j < s.width ? s.dw : s.db;
  if (!out) return;
  const int at = j < s.width ? c * s.width + j : c;
  if (j < s.width ? s.w_bf16 : s.b_bf16)
    ((bf16*)out)[at] = (bf16)v;
  else
    ((float*)out)[at] = v;
}

template <typename T>
constexpr int kVec = 16 / sizeof(T);  // channels of a thread, forward

template <typename Go>
int with_width(int64_t width, Go go) {
  using std::integral_constant;
  if (width == 2) return go(integral_constant<int, 2>());
  if (width == 3) return go(integral_constant<int, 3>());
  return go(integral_constant<int, 4>());
}

template <typename T>
int forward(Conv& s, int64_t width, hipStream_t stream) {
  s.vecs = s.channels / kVec<T>;
  // Few rows go in short runs, for the latency of one (1 x 1024 x 1536: 5.0 us, with kRun 6.5; 1 x 2048: 6.6 and 7.3;
  // 4 x 2048: 15.5 and 14.8).  Either covers the W - 1 tokens that read the state, so that one thread reads it and may
  // write the next one over it.
  const bool few = s.tokens <= 4 || s.batch * s.tokens * s.vecs < 512 * 1024;
  const int run = few ? 4 : kRun;
  s.runs = (int)((s.tokens + run - 1) / run);
  const int64_t blocks = (s.batch * s.runs * s.vecs + 255) / 256;
  BMX_REQUIRE(blocks < (1ll << 31), "causal_conv: too many rows");
  return with_width(width, [&](auto w) {
    constexpr int W = decltype(w)::value;
    if (few)
      causal_conv_kernel<T, W, kVec<T>, 4><<<fold_grid(blocks, 256), 256, 0, stream>>>(s);
    else
      causal_conv_kernel<T, W, kVec<T>, kRun><<<fold_grid(blocks, 256), 256, 0, stream>>>(s);
    return check_launch("causal_conv");
  });
}

int64_t bwd_parts(int64_t batch, int64_t tokens) {
  const int64_t runs = (tokens + kBwdRun - 1) / kBwdRun, rows = 256 / kBwdVecs;
  return batch * ((runs + rows - 1) / rows);
}

template <typename T>
int backward(Conv& s, int64_t width, hipStream_t stream) {
  s.vecs = s.channels / kBwdVec;
  s.runs = (int)((s.tokens + kBwdRun - 1) / kBwdRun);
  s.blocks = bwd_parts(s.batch, s.tokens) * ((s.vecs + kBwdVecs - 1) / kBwdVecs);
  BMX_REQUIRE(s.blocks < (1ll << 31), "causal_conv: too many rows");
  return with_width(width, [&](auto w) {
    causal_conv_bwd_kernel<T, decltype(w)::value><<<fold_grid(s.blocks, 256), 256, 0, stream>>>(s);
    return check_launch("causal_conv_bwd");
  });
}

int setup(Conv& s, const void* x, int dtype, const int64_t* shape, const int64_t* strides, const void* weight, int w_dtype,
          const void* bias, int bias_dtype, const void* state, const void* lengths, int lengths64, int silu) {
  BMX_REQUIRE(dtype == kF32 || dtype == kBF16, "causal_conv: dtype must be fp32 or bf16");
  BMX_REQUIRE((w_dtype == kF32 || w_dtype == kBF16) && (bias_dtype == kF32 || bias_dtype == kBF16),
              "causal_conv: weight and bias dtypes must be fp32 or bf16");
  BMX_REQUIRE(shape && strides, "causal_conv: null shape or strides");
  for (int i = 0; i < 4; ++i) BMX_REQUIRE(shape[i] >= 0, "causal_conv: negative size");
  BMX_REQUIRE(shape[2] >= 8 && shape[2] % 8 == 0 && shape[2] < (1 << 20),
              "causal_conv: channels must be a multiple of 8 in [8, 2^20)");
  BMX_REQUIRE(shape[3] >= 2 && shape[3] <= 4, "causal_conv: width must be 2, 3 or 4");
  BMX_REQUIRE(shape[0] < (1ll << 31) && shape[1] < (1ll << 31) && (shape[1] == 0 || shape[0] < (1ll << 31) / shape[1]),
              "causal_conv: expected fewer than 2^31 rows");
  const int unit = dtype == kF32 ? 4 : 8;
  BMX_REQUIRE(strides[0] % unit == 0 && strides[1] % unit == 0, "causal_conv: strides must be multiples of 16 bytes");
  s.x = x, s.w = weight, s.bias = bias, s.state = state, s.lengths = lengths, s.lengths64 = lengths64;
  s.sb = strides[0], s.st = strides[1], s.batch = shape[0], s.tokens = shape[1], s.channels = (int)shape[2];
  s.silu = silu != 0, s.w_bf16 = w_dtype == kBF16, s.b_bf16 = bias_dtype == kBF16;
  return BMX_OK;
}

bool aligned16(std::initializer_list<const void*> pointers) {
  uintptr_t bits = 0;
  for (const void* p : pointers) bits |= (uintptr_t)p;
  return bits % 16 == 0;
}

}  // namespace

extern "C" int bmx_causal_conv_fwd(const void* x, int dtype, const int64_t* shape, const int64_t* strides,
                                   const void* weight, int w_dtype, const void* bias, int bias_dtype, const void* state,
                                   const void* lengths, int lengths64, int silu, void* y, void* state_out, void* stream) {
  Conv s = {};
  if (int rc = setup(s, x, dtype, shape, strides, weight, w_dtype, bias, bias_dtype, state, lengths, lengths64, silu))
    return rc;
  if (s.batch == 0 || s.tokens == 0) {
    BMX_REQUIRE(s.batch == 0 || !state_out, "causal_conv: the state of no tokens is the caller's");
    return BMX_OK;
  }
  BMX_REQUIRE(x && weight && y, "causal_conv: null pointer");
  BMX_REQUIRE(aligned16({x, weight, bias, state, y, state_out}), "causal_conv: tensors must be 16-byte aligned");
  s.y = y, s.next = state_out;
  return dtype == kF32 ? forward<float>(s, shape[3], (hipStream_t)stream) : forward<bf16>(s, shape[3], (hipStream_t)stream);
}

extern "C" size_t bmx_causal_conv_workspace_bytes(int64_t batch, int64_t tokens, int64_t channels, int64_t width) {
  if (batch <= 0 || tokens <= 0 || channels <= 0 || width <= 0) return 0;
  return (size_t)(bwd_parts(batch, tokens) * (width + 1) * channels) * sizeof(float);
}

extern "C" int bmx_causal_conv_bwd(const void* x, int dtype, const int64_t* shape, const int64_t* strides,
                                   const void* weight, int w_dtype, const void* bias, int bias_dtype, const void* state,
                                   const void* lengths, int lengths64, int silu, const void* dy, const void* dstate_out,
                                   void* dx, void* dweight, void* dbias, void* dstate, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  Conv s = {};
  if (int rc = setup(s, x, dtype, shape, strides, weight, w_dtype, bias, bias_dtype, state, lengths, lengths64, silu))
    return rc;
  BMX_REQUIRE(s.batch > 0 && s.tokens > 0, "causal_conv_bwd: expected rows");
  BMX_REQUIRE(x && weight, "causal_conv: null pointer");
  BMX_REQUIRE((bias || !dbias) && (state || !dstate), "causal_conv_bwd: gradient of an absent bias or state");
  BMX_REQUIRE(aligned16({x, weight, bias, state, dy, dstate_out, dx, dstate}), "causal_conv: tensors must be 16-byte aligned");
  s.dy = dy, s.dnext = dstate_out, s.dx = dx, s.dstate = dstate;
  if (dweight || dbias) {
    BMX_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 &&
                    workspace_bytes >= bmx_causal_conv_workspace_bytes(s.batch, s.tokens, s.channels, shape[3]),
                "causal_conv_bwd: workspace too small or not 16-byte aligned");
    s.partial = (float*)workspace;
  }
  hipStream_t hs = (hipStream_t)stream;
  if (int rc = dtype == kF32 ? backward<float>(s, shape[3], hs) : backward<bf16>(s, shape[3], hs)) return rc;
  if (s.partial) {
    const ConvSums c = {s.partial, dweight, dbias, bwd_parts(s.batch, s.tokens), s.channels, (int)shape[3], s.w_bf16,
                        s.b_bf16};
    causal_conv_sums_kernel<<<dim3((s.channels + 15) / 16, (int)shape[3] + 1), 256, 0, hs>>>(c);
  }
  return check_launch("causal_conv_bwd");
}
