// The frame between two blocks of a sequence stack in one pass: RMS norm of the
// block's result y, its gate and residual scale, the residual add and the next
// block's RMS norm; and its gradient.
//
//   m = y rho_y yw,  rho_y = 1 / sqrt(mean(y^2) + eps)   (without the norm: m = y)
//   r = x + scale s m,  s = sigmoid(gate)
//   h = r rho_r w,  rho_r = 1 / sqrt(mean(r^2) + eps)
//   e = dh w:  dR = dr + rho_r (e - r rho_r^2 mean(e r)) = dx;  dw = sum dh r rho_r
//   f = dR s scale yw:  dy = rho_y (f - y rho_y^2 mean(f y))
//   dscale = sum dR s m;  dgate = dR scale m s (1 - s);  dyw = sum dR s scale y rho_y
//
// A row lies in the registers of L threads, V runs of 8 channels each, from its
// only read to its only write; the backward pass works r and both norms out
// again instead of keeping them.  h comes from r before its rounding.  All sums
// are fp32 and in a fixed order.
//
// Bound by HBM: 2 x 8192 rows of 2048 (fp32 stream, bf16 block and gate) take 90
// us, 5.2 TB/s where a copy reaches 4.8; the gradient of 4 x 2048 such rows 72
// us, 5.1 TB/s, and 5 more for the weights' partial rows.  32 rows of 768: 4 us.
#include <type_traits>

#include "bmx_common.h"

using namespace bmx;

namespace {

constexpr int kMaxDim = 8192;
// Threads of the gradient at most: two waves a SIMD.  A block leaves a partial row per weight, so not twice as many (2^24
// values of 4096 a row, both ways: 114 us, 119); with half of them 157.
constexpr int kBwdThreads = 512 * 256;

struct Rows {
  const void* p;
  int64_t sb, st;  // strides of a batch element and a token, in elements
};
struct Frame {
  Rows x, y, gate;
  const void *yw, *scale, *w, *dr, *dh;
  void *r, *h, *dx, *dy, *dgate;
  float *partial, *gate_partial;  // [blocks][3][dim] sums for yw, scale, w; [units][dim] for a shared gate
  int64_t rows, tokens, units, unit_rows, splits;  // units: runs of rows, `splits` per batch element where it has its gate
  int dim, w_bf16, post, pre, shared;
  float eps, inv_dim;
};

// 8 consecutive values as fp32, and back.
struct Oct {
  f32x4 a, b;
};
__device__ __forceinline__ Oct load_oct(const float* p) { return {*(const f32x4*)p, *(const f32x4*)(p + 4)}; }
__device__ __forceinline__ Oct load_oct(const bf16* p) {
  const bf16x8 v = *(const bf16x8*)p;
  return {f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]},
          f32x4{(float)v[4], (float)v[5], (float)v[6], (float)v[7]}};
}
__device__ __forceinline__ void store_oct(float* p, const Oct& v) { *(f32x4*)p = v.a, *(f32x4*)(p + 4) = v.b; }
__device__ __forceinline__ void store_oct(bf16* p, const Oct& v) {
  *(bf16x8*)p = bf16x8{(bf16)v.a[0], (bf16)v.a[1], (bf16)v.a[2], (bf16)v.a[3],
                       (bf16)v.b[0], (bf16)v.b[1], (bf16)v.b[2], (bf16)v.b[3]};
}
// The same as they lie in memory: a row that is on its way holds no more registers than it has bytes.
template <typename T>
struct RawOct;
template <>
struct RawOct<float> {
  Oct v;
  __device__ __forceinline__ Oct wide() const { return v; }
};
template <>
struct RawOct<bf16> {
  bf16x8 v;
  __device__ __forceinline__ Oct wide() const {
    return {f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]},
            f32x4{(float)v[4], (float)v[5], (float)v[6], (float)v[7]}};
  }
};
template <typename T>
__device__ __forceinline__ RawOct<T> load_raw(const T* p, bool there) {
  RawOct<T> o = {};
  if (there) o = *(const RawOct<T>*)p;
  return o;
}
__device__ __forceinline__ Oct fill(float v) { return {f32x4{v, v, v, v}, f32x4{v, v, v, v}}; }
__device__ __forceinline__ Oct operator*(const Oct& x, const Oct& y) { return {x.a * y.a, x.b * y.b}; }
__device__ __forceinline__ Oct operator+(const Oct& x, const Oct& y) { return {x.a + y.a, x.b + y.b}; }
__device__ __forceinline__ Oct operator-(const Oct& x, const Oct& y) { return {x.a - y.a, x.b - y.b}; }
__device__ __forceinline__ Oct operator*(const Oct& x, float s) { return {x.a * s, x.b * s}; }
__device__ __forceinline__ float dot(const Oct& x, const Oct& y) {
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) v += x.a[i] * y.a[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) v += x.b[i] * y.b[i];
  return v;
}
__device__ __forceinline__ Oct sigmoid(const Oct& x) {
  Oct o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o.a[i] = sigmoid_f(x.a[i]), o.b[i] = sigmoid_f(x.b[i]);
  return o;
}
// 1 - s of a gate's s = sigmoid(x), relative to itself, as a factor of s (1 - s): exp(-x) s.  Of 1 less an s that is
// rounded to nearly 1 little or (from x = 17 on) nothing would be left.  Where exp(-x) is infinite, s is zero.
__device__ __forceinline__ Oct shut(const Oct& x, const Oct& s) {
  Oct o;
  auto one = [](float x, float s) {
    return __builtin_amdgcn_fmed3f(__builtin_amdgcn_exp2f(x * -1.4426950408889634f), 0.f, 0x1p126f) * s;
  };
#pragma unroll
  for (int i = 0; i < 4; ++i) o.a[i] = one(x.a[i], s.a[i]), o.b[i] = one(x.b[i], s.b[i]);
  return o;
}
__device__ __forceinline__ Oct load_weight(const void* w, int w_bf16, int at) {
  if (!w) return fill(1.f);
  return w_bf16 ? load_oct((const bf16*)w + at) : load_oct((const float*)w + at);
}

// Sum over the L threads of a row, in every one of them.  Rows of several waves meet in LDS: `turn` alternates
// between two buffers, so that one barrier a sum is enough.
template <int L>
__device__ __forceinline__ float row_sum(float v, float (&lds)[2][16], int& turn) {
  if (L == 16) {
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    v += dpp<0x140>(v);
    return v;
  }
  v = wave_sum_full(v);
  if (L == 64) return v;
  if (lane_id() == 0) lds[turn][threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < L / 64; ++i) v += lds[turn][i];
  turn ^= 1;
  return v;
}

// The same for two values, one barrier for both.
template <int L>
__device__ __forceinline__ void row_sums(float& v, float& w, float (&lds)[2][16], int& turn) {
  if (L <= 64) {
    v = row_sum<L>(v, lds, turn), w = row_sum<L>(w, lds, turn);
    return;
  }
  v = wave_sum_full(v), w = wave_sum_full(w);
  if (lane_id() == 0) lds[turn][threadIdx.x >> 6] = v, lds[turn][8 + (threadIdx.x >> 6)] = w;
  __syncthreads();
  v = w = 0.f;
#pragma unroll
  for (int i = 0; i < L / 64; ++i) v += lds[turn][i], w += lds[turn][8 + i];
  turn ^= 1;
}

// Threads of a block: rows of up to a wave share one, others have one of their own (they meet at barriers).
template <int L>
constexpr int threads_of() {
  return L > 64 ? L : 256;
}

__device__ __forceinline__ float rho(float sum, const Frame& s) { return 1.f / sqrtf(sum * s.inv_dim + s.eps); }

template <typename X, typename Y, int L, int V>
__global__ __launch_bounds__(threads_of<L>()) void residual_norm_kernel(Frame s) {
  __shared__ float lds[2][16];
  int turn = 0;
  const int lane = threadIdx.x % L;
  const int64_t row = (int64_t)block_index() * (threads_of<L>() / L) + threadIdx.x / L;
  if (row >= s.rows) return;  // whole rows leave; a row of several waves is its block's only one
  const int64_t b = row / s.tokens, t = row - b * s.tokens;
  const X* x = (const X*)s.x.p + b * s.x.sb + t * s.x.st;
  const Y* y = (const Y*)s.y.p + b * s.y.sb + t * s.y.st;
  const Y* gate = s.gate.p ? (const Y*)s.gate.p + b * s.gate.sb + t * s.gate.st : nullptr;
  Oct xv[V], m[V], g[V];
  float sum = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = 8 * (lane + v * L);
    const bool live = c < s.dim;
    xv[v] = live ? load_oct(x + c) : fill(0.f);
    m[v] = live ? load_oct(y + c) : fill(0.f);
    g[v] = live && gate ? load_oct(gate + c) : fill(0.f);
    sum += dot(m[v], m[v]);
  }
  const float ry = s.post ? rho(row_sum<L>(sum, lds, turn), s) : 1.f;
  sum = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = 8 * (lane + v * L);
    if (c >= s.dim) continue;
    Oct k = load_weight(s.scale, s.w_bf16, c);
    if (gate) k = k * sigmoid(g[v]);
    xv[v] = xv[v] + m[v] * ry * load_weight(s.yw, s.w_bf16, c) * k;
    sum += dot(xv[v], xv[v]);
    store_oct((X*)s.r + row * s.dim + c, xv[v]);
  }
  if (!s.pre) return;
  const float rr = rho(row_sum<L>(sum, lds, turn), s);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = 8 * (lane + v * L);
    if (c < s.dim) store_oct((Y*)s.h + row * s.dim + c, xv[v] * rr * load_weight(s.w, s.w_bf16, c));
  }
}

// Gradient.  A block walks units of rows, its L-thread groups taking every (256 / L)-th row of a unit; each thread
// keeps the weights' sums of its channels over all of them, a shared gate's over the unit.
template <typename X, typename Y, int L, int V>
__global__ __launch_bounds__(threads_of<L>()) void residual_norm_bwd_kernel(Frame s) {
  constexpr int groups = threads_of<L>() / L;
  __shared__ float lds[2][16];
  __shared__ float sums[groups > 1 ? groups : 1][groups > 1 ? 8 * L * V : 1];
  int turn = 0;
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  Oct dyw[V], dscale[V], dw[V], dgate[V];
#pragma unroll
  for (int v = 0; v < V; ++v) dyw[v] = dscale[v] = dw[v] = dgate[v] = fill(0.f);
  // the weights stay in registers where there is room; channels that are not there have no part in a row's sums
  Oct kept[3] = {fill(0.f), fill(0.f), fill(0.f)};
  if (V == 1 && 8 * lane < s.dim) {
    kept[0] = load_weight(s.yw, s.w_bf16, 8 * lane), kept[1] = load_weight(s.scale, s.w_bf16, 8 * lane);
    kept[2] = load_weight(s.w, s.w_bf16, 8 * lane);
  }
  auto weight = [&](int which, int v) {
    const int c = 8 * (lane + v * L);
    if (V == 1) return kept[which];
    return c < s.dim ? load_weight(which == 0 ? s.yw : which == 1 ? s.scale : s.w, s.w_bf16, c) : fill(0.f);
  };

  // The groups' sums of one quantity, added in their order, to `out` (its row of dim values).
  auto put = [&](const Oct (&v)[V], auto* out) {
    if constexpr (groups == 1) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (8 * (lane + i * L) < s.dim) store_oct(out + 8 * (lane + i * L), v[i]);
      return;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) store_oct(&sums[group][8 * (lane + i * L)], v[i]);
    __syncthreads();
    for (int c = threadIdx.x; c < s.dim; c += threads_of<L>()) {
      float total = 0.f;
#pragma unroll
      for (int i = 0; i < groups; ++i) total += sums[i][c];
      using Out = std::remove_pointer_t<decltype(out)>;
      out[c] = (Out)total;
    }
  };

  for (int64_t unit = blockIdx.x; unit < s.units; unit += gridDim.x) {
    const int64_t element = s.shared ? unit / s.splits : 0, part = s.shared ? unit % s.splits : unit;
    const int64_t limit = s.shared ? s.tokens : s.rows;
    const int64_t first = part * s.unit_rows, last = min(first + s.unit_rows, limit);
    // a row's operands are asked for while the row before is worked on (with two runs a thread there is no room)
    RawOct<X> nx[V], ndr[V];
    RawOct<Y> ny[V], ng[V], ndh[V];
    auto ask = [&](int64_t i) {
      const int64_t row = element * s.tokens + i, b = row / s.tokens, t = row - b * s.tokens;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = 8 * (lane + v * L);
        const bool live = c < s.dim && i < last;
        nx[v] = load_raw((const X*)s.x.p + b * s.x.sb + t * s.x.st + c, live);
        ny[v] = load_raw((const Y*)s.y.p + b * s.y.sb + t * s.y.st + c, live);
        ng[v] = load_raw((const Y*)s.gate.p + b * s.gate.sb + t * s.gate.st + c, live && s.gate.p);
        ndr[v] = load_raw((const X*)s.dr + row * s.dim + c, live && s.dr);
        ndh[v] = load_raw((const Y*)s.dh + row * s.dim + c, live && s.dh);
      }
    };
    if (V == 1) ask(first + group);
    for (int64_t i = first + group; i < last; i += groups) {
      const int64_t row = element * s.tokens + i;
      const bool gate = s.gate.p;
      if (V > 1) ask(i);
      Oct r[V], n[V], g[V], dr[V], dh[V];
      float sum = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        r[v] = nx[v].wide(), n[v] = ny[v].wide(), g[v] = ng[v].wide(), dr[v] = ndr[v].wide(), dh[v] = ndh[v].wide();
        sum += dot(n[v], n[v]);
      }
      if (V == 1) ask(i + groups);
      const float ry = s.post ? rho(row_sum<L>(sum, lds, turn), s) : 1.f;
      float rr = 0.f, er = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        Oct k = weight(1, v);
        if (gate) k = k * sigmoid(g[v]);
        n[v] = n[v] * ry;
        r[v] = r[v] + n[v] * weight(0, v) * k;
        rr += dot(r[v], r[v]);
        er += dot(dh[v] * weight(2, v), r[v]);
      }
      if (s.pre) {
        row_sums<L>(rr, er, lds, turn);
        rr = rho(rr, s), er *= s.inv_dim * rr * rr;
      }
      float fn = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = 8 * (lane + v * L);
        const bool live = c < s.dim;
        if (s.pre) {
          dr[v] = dr[v] + (dh[v] * weight(2, v) - r[v] * er) * rr;
          dw[v] = dw[v] + dh[v] * r[v] * rr;
        }
        if (s.dx && live) store_oct((X*)s.dx + row * s.dim + c, dr[v]);
        const Oct gated = gate ? dr[v] * sigmoid(g[v]) : dr[v];  // dR s
        const Oct block = gated * n[v];
        dscale[v] = dscale[v] + block * weight(0, v);
        const Oct back = gated * weight(1, v);
        dyw[v] = dyw[v] + back * n[v];
        dr[v] = back * weight(0, v);
        if (gate) {
          const Oct dg = dr[v] * n[v] * shut(g[v], sigmoid(g[v]));
          if (s.shared)
            dgate[v] = dgate[v] + dg;
          else if (s.dgate && live)
            store_oct((Y*)s.dgate + row * s.dim + c, dg);
        }
        fn += dot(dr[v], n[v]);
      }
      if (s.post) fn = row_sum<L>(fn, lds, turn) * s.inv_dim;
      if (s.dy) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int c = 8 * (lane + v * L);
          if (c < s.dim) store_oct((Y*)s.dy + row * s.dim + c, s.post ? (dr[v] - n[v] * fn) * ry : dr[v]);
        }
      }
    }
    if (s.shared && s.dgate) {
      if (s.splits == 1)
        put(dgate, (Y*)s.dgate + unit * s.dim);
      else
        put(dgate, s.gate_partial + unit * s.dim);
#pragma unroll
      for (int v = 0; v < V; ++v) dgate[v] = fill(0.f);
    }
  }
  if (!s.partial) return;
  float* out = s.partial + (int64_t)blockIdx.x * 3 * s.dim;
  put(dyw, out);
  put(dscale, out + s.dim);
  put(dw, out + 2 * s.dim);
}

// Column sums of partial rows: a block per 32 columns of one result, 32 slices of the rows, four columns a thread.
struct ColumnSums {
  const float* partial[4];
  void* out[4];
  int64_t row_stride[4], batch_stride[4];
  int rows[4], bf16_out[4], batches[4];
  int dim;
};
__global__ __launch_bounds__(256) void residual_norm_sums_kernel(ColumnSums s) {
  __shared__ f32x4 lds[32][9];
  const int which = blockIdx.y;
  if (!s.out[which]) return;
  const int col = threadIdx.x % 8, part = threadIdx.x / 8, c = (int)blockIdx.x * 32 + 4 * col;
  for (int64_t batch = blockIdx.z; batch < s.batches[which]; batch += gridDim.z) {
    const float* from = s.partial[which] + batch * s.batch_stride[which] + c;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (c < s.dim) {
#pragma unroll 8
      for (int row = part; row < s.rows[which]; row += 32) v += *(const f32x4*)(from + row * s.row_stride[which]);
    }
    __syncthreads();
    lds[part][col] = v;
    __syncthreads();
    if (part == 0 && c < s.dim) {
#pragma unroll
      for (int i = 1; i < 32; ++i) v += lds[i][col];
      if (s.bf16_out[which])
        store4((bf16*)s.out[which] + batch * s.dim + c, v);
      else
        store4((float*)s.out[which] + batch * s.dim + c, v);
    }
  }
}

// A row's threads and runs of 8 channels each: as few threads as hold it with one run each (a wave for 128 channels
// instead of 16 lanes: 79 us for 36 at 131072 rows), as a row of several waves meets at a barrier a sum, but two runs
// cost as much (64 rows of 1024: 128 threads 3.4 us, 64 with two runs 4.2) and in the gradient, where they leave one
// wave a SIMD, more (2^24 values, both ways: 1024 106 and 125 us, 4096 114 and 143).  Forward, rows past 2048 lose
// more to idle threads (8160 rows of 2056: 512 threads 50 us, 256 with two runs 42; of 4096: 38 and 37).
template <bool kBackward, typename Go>
void with_layout(int dim, Go go) {
  using std::integral_constant;
  if (dim <= 128) return go(integral_constant<int, 16>(), integral_constant<int, 1>());
  if (dim <= 512) return go(integral_constant<int, 64>(), integral_constant<int, 1>());
  if (dim <= 1024) return go(integral_constant<int, 128>(), integral_constant<int, 1>());
  if (dim <= 2048) return go(integral_constant<int, 256>(), integral_constant<int, 1>());
  if (dim <= 4096) return go(integral_constant<int, kBackward ? 512 : 256>(), integral_constant<int, kBackward ? 1 : 2>());
  return go(integral_constant<int, 512>(), integral_constant<int, 2>());
}

template <typename X, typename Y>
void launch(const Frame& s, hipStream_t stream) {
  with_layout<false>(s.dim, [&](auto l, auto v) {
    constexpr int L = decltype(l)::value, V = decltype(v)::value, threads = threads_of<L>(), per = threads / L;
    residual_norm_kernel<X, Y, L, V><<<fold_grid((s.rows + per - 1) / per, threads), threads, 0, stream>>>(s);
  });
}
template <typename X, typename Y>
void launch_bwd(const Frame& s, int blocks, hipStream_t stream) {
  with_layout<true>(s.dim, [&](auto l, auto v) {
    constexpr int L = decltype(l)::value, V = decltype(v)::value;
    residual_norm_bwd_kernel<X, Y, L, V><<<blocks, threads_of<L>(), 0, stream>>>(s);
  });
}

// Units of the gradient's rows and the blocks that walk them.  About 8 rows a group, at most kBwdThreads threads; with
// a gate per batch element, whole elements or equal parts of them.
struct Units {
  int64_t units, unit_rows, splits;
  int blocks;
};
Units plan_units(int64_t batch, int64_t tokens, int64_t dim, bool shared) {
  int64_t per = 1, most = 1;
  with_layout<true>((int)dim, [&](auto l, auto) {
    constexpr int L = decltype(l)::value, threads = threads_of<L>();
    per = 8 * (threads / L), most = kBwdThreads / threads;
  });
  const int64_t rows = batch * tokens, length = shared ? tokens : rows, elements = shared ? batch : 1;
  int64_t splits = elements >= most ? 1 : most / elements;
  const int64_t enough = (length + per - 1) / per;
  if (splits > enough) splits = enough;
  if (splits < 1) splits = 1;
  Units u;
  u.unit_rows = (length + splits - 1) / splits;
  u.splits = u.unit_rows ? (length + u.unit_rows - 1) / u.unit_rows : 1;
  u.units = elements * u.splits;
  u.blocks = (int)(u.units < most ? u.units : most);
  return u;
}

int setup(Frame& s, int x_dtype, int dtype, const int64_t* shape, const int64_t* strides, int gate, int w_dtype, int post,
          int pre, float eps) {
  BMX_REQUIRE((x_dtype == kF32 || x_dtype == kBF16) && (dtype == kF32 || dtype == kBF16) &&
                  (x_dtype == kF32 || dtype == kBF16),
              "residual_norm: x and y must be fp32 or bf16, fp32 x where y is fp32");
  BMX_REQUIRE(w_dtype == kF32 || w_dtype == kBF16, "residual_norm: weight dtype must be fp32 or bf16");
  BMX_REQUIRE(shape && strides, "residual_norm: null shape or strides");
  BMX_REQUIRE(gate >= 0 && gate <= 2, "residual_norm: gate must be 0 (none), 1 (per token) or 2 (per batch element)");
  for (int i = 0; i < 3; ++i) BMX_REQUIRE(shape[i] >= 0, "residual_norm: negative size");
  BMX_REQUIRE(shape[2] >= 8 && shape[2] <= kMaxDim && shape[2] % 8 == 0,
              "residual_norm: dim must be a multiple of 8 in [8, 8192]");
  BMX_REQUIRE(shape[0] < (1ll << 31) && shape[1] < (1ll << 31) && (shape[1] == 0 || shape[0] < (1ll << 31) / shape[1]),
              "residual_norm: expected fewer than 2^31 rows");
  BMX_REQUIRE(eps >= 0x1p-126f, "residual_norm: eps must be positive, at least 2^-126");
  for (int i = 0; i < 6; ++i) BMX_REQUIRE(strides[i] % 8 == 0, "residual_norm: strides must be multiples of 8");
  s.rows = shape[0] * shape[1], s.tokens = shape[1], s.dim = (int)shape[2];
  s.x.sb = strides[0], s.x.st = strides[1], s.y.sb = strides[2], s.y.st = strides[3];
  s.gate.sb = strides[4], s.gate.st = gate == 2 ? 0 : strides[5];
  s.w_bf16 = w_dtype == kBF16, s.post = post != 0, s.pre = pre != 0, s.shared = gate == 2;
  s.eps = eps, s.inv_dim = 1.f / (float)s.dim;
  return BMX_OK;
}

bool aligned16(std::initializer_list<const void*> pointers) {
  uintptr_t bits = 0;
  for (const void* p : pointers) bits |= (uintptr_t)p;
  return bits % 16 == 0;
}

}  // namespace

extern "C" int bmx_residual_norm_fwd(const void* x, const void* y, const void* gate, int x_dtype, int dtype,
                                     const int64_t* shape, const int64_t* strides, int gate_kind, const void* y_weight,
                                     const void* scale, const void* weight, int w_dtype, int post_norm, int pre_norm,
                                     float eps, void* r, void* h, void* stream) {
  Frame s = {};
  if (int rc = setup(s, x_dtype, dtype, shape, strides, gate_kind, w_dtype, post_norm, pre_norm, eps)) return rc;
  if (s.rows == 0) return BMX_OK;
  BMX_REQUIRE(x && y && r && (!s.pre || h) && (gate_kind == 0 || gate), "residual_norm: null pointer");
  BMX_REQUIRE(aligned16({x, y, gate, y_weight, scale, weight, r, h}), "residual_norm: tensors must be 16-byte aligned");
  s.x.p = x, s.y.p = y, s.gate.p = gate_kind ? gate : nullptr;
  s.yw = s.post ? y_weight : nullptr, s.scale = scale, s.w = weight, s.r = r, s.h = h;
  hipStream_t hs = (hipStream_t)stream;
  if (dtype == kF32)
    launch<float, float>(s, hs);
  else if (x_dtype == kF32)
    launch<float, bf16>(s, hs);
  else
    launch<bf16, bf16>(s, hs);
  return check_launch("residual_norm");
}

extern "C" size_t bmx_residual_norm_workspace_bytes(int64_t batch, int64_t tokens, int64_t dim, int gate_kind) {
  if (batch <= 0 || tokens <= 0 || dim < 8 || dim > kMaxDim) return 0;
  const Units u = plan_units(batch, tokens, dim, gate_kind == 2);
  return (size_t)((int64_t)u.blocks * 3 + (gate_kind == 2 && u.splits > 1 ? u.units : 0)) * dim * sizeof(float);
}

extern "C" int bmx_residual_norm_bwd(const void* x, const void* y, const void* gate, int x_dtype, int dtype,
                                     const int64_t* shape, const int64_t* strides, int gate_kind, const void* y_weight,
                                     const void* scale, const void* weight, int w_dtype, int post_norm, int pre_norm,
                                     float eps, const void* dr, const void* dh, void* dx, void* dy, void* dgate,
                                     void* dy_weight, void* dscale, void* dweight, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  Frame s = {};
  if (int rc = setup(s, x_dtype, dtype, shape, strides, gate_kind, w_dtype, post_norm, pre_norm, eps)) return rc;
  BMX_REQUIRE(s.rows > 0, "residual_norm_bwd: expected rows");
  BMX_REQUIRE(x && y && (gate_kind == 0 || gate), "residual_norm: null pointer");
  BMX_REQUIRE(gate_kind != 0 || !dgate, "residual_norm_bwd: gradient of an absent gate");
  BMX_REQUIRE((y_weight || !dy_weight) && (scale || !dscale) && (weight || !dweight),
              "residual_norm_bwd: gradient of an absent weight");
  BMX_REQUIRE(aligned16({x, y, gate, y_weight, scale, weight, dr, dh, dx, dy, dgate, dy_weight, dscale, dweight}),
              "residual_norm: tensors must be 16-byte aligned");
  const Units u = plan_units(shape[0], shape[1], s.dim, s.shared);
  const bool weights = dy_weight || dscale || dweight, gates = s.shared && dgate && u.splits > 1;
  if (weights || gates)
    BMX_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 &&
                    workspace_bytes >= bmx_residual_norm_workspace_bytes(shape[0], shape[1], s.dim, gate_kind),
                "residual_norm_bwd: workspace too small or not 16-byte aligned");
  s.x.p = x, s.y.p = y, s.gate.p = gate_kind ? gate : nullptr;
  s.yw = s.post ? y_weight : nullptr, s.scale = scale, s.w = weight;
  s.dr = dr, s.dh = s.pre ? dh : nullptr, s.dx = dx, s.dy = dy, s.dgate = dgate;
  s.units = u.units, s.unit_rows = u.unit_rows, s.splits = u.splits;
  s.partial = weights ? (float*)workspace : nullptr;
  s.gate_partial = gates ? (float*)workspace + (int64_t)u.blocks * 3 * s.dim : nullptr;
  hipStream_t hs = (hipStream_t)stream;
  if (dtype == kF32)
    launch_bwd<float, float>(s, u.blocks, hs);
  else if (x_dtype == kF32)
    launch_bwd<float, bf16>(s, u.blocks, hs);
  else
    launch_bwd<bf16, bf16>(s, u.blocks, hs);
  if (weights || gates) {
    ColumnSums c = {};
    void* outs[3] = {dy_weight, dscale, dweight};
    for (int i = 0; i < 3; ++i) {
      c.partial[i] = s.partial + i * s.dim, c.out[i] = weights ? outs[i] : nullptr;
      c.row_stride[i] = 3 * s.dim, c.rows[i] = u.blocks, c.bf16_out[i] = s.w_bf16, c.batches[i] = 1;
    }
    c.partial[3] = s.gate_partial, c.out[3] = gates ? dgate : nullptr;
    c.row_stride[3] = s.dim, c.batch_stride[3] = u.splits * s.dim, c.rows[3] = (int)u.splits;
    c.bf16_out[3] = dtype == kBF16, c.batches[3] = (int)shape[0];
    c.dim = s.dim;
    const int z = gates ? (int)(shape[0] < 64 ? shape[0] : 64) : 1;
    residual_norm_sums_kernel<<<dim3((s.dim + 31) / 32, 4, z), 256, 0, hs>>>(c);
  }
  return check_launch("residual_norm_bwd");
}
