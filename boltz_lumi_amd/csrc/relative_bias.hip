// Learned relative-position bias by buckets, and the gradient of its table.
//
//   bias[b][h][i][j] = table[bucket(k_pos[b][j] - q_pos[b][i])][h]
//   dtable[c][h]     = sum of dbias[b][h][i][j] over the (b, i, j) of bucket c
//
// A bucket is counted from whole-number thresholds t_1 <= t_2 <= .. that the
// host gives: bucket(d) = #{t_i <= n} with n = max(-d, 0) (one direction), or n =
// |d| and side = #thresholds + 1 added for d > 0 (two directions).  No
// logarithm is taken here, so a distance at a border cannot round to the other side.
#include "bmx_common.h"

using namespace bmx;

namespace {

constexpr int kMaxSide = 256;             // thresholds travel in the kernel arguments
constexpr int kMaxBuckets = 256;
constexpr int kMaxDistance = 0x7ffffffe;  // distances are cut here, above every threshold

struct Relative {
  const void *q_pos, *k_pos;
  int64_t q_sb, k_sb;  // batch strides of the positions
  int64_t m, n;
  int pos64, heads, buckets, bidirectional, count, exact;  // exact: the first thresholds are 1, 2, .., exact
  int32_t t[kMaxSide];
};

__device__ __forceinline__ int64_t position(const void* p, int wide, int64_t i) {
  return wide ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

// Signed distance cut to +-kMaxDistance.
__device__ __forceinline__ int distance(int64_t k, int64_t q) {
  const int64_t d = k - q;
  return (int)(d > kMaxDistance ? kMaxDistance : d < -kMaxDistance ? -kMaxDistance : d);
}

// Thresholds in LDS: n < exact is its own bucket, the others are searched.
__device__ __forceinline__ int bucket_of(const Relative& s, const int* t, int d) {
  int n = d < 0 ? -d : (s.bidirectional ? d : 0);
  int lo = 0;
  if (n < s.exact) {
    lo = n;
  } else {
    int hi = s.count;  // thresholds t[lo - 1] <= n < t[hi]
    lo = s.exact;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (t[mid] <= n)
        lo = mid + 1;
      else
        hi = mid;
    }
  }
  return lo + (s.bidirectional && d > 0 ? s.count + 1 : 0);
}

// 16 bytes at any element alignment: rows of an odd number of keys.
typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));

// A thread holds the buckets of 16 bytes' worth of consecutive keys of one query row
// and writes them for `per` heads from the table in LDS: the positions are looked at once,
// a store is 16 bytes, and the floor is the write of the result (16 heads, 2048 x 2048, fp32, 268 MB: 46 us, 5.8 TB/s).
template <typename U>  // the element's bits: uint32_t (fp32) or uint16_t (bf16); values are copied, not rounded
__global__ __launch_bounds__(256) void relative_bias_kernel(Relative s, const U* table, int64_t batch, int per, U* out) {
  constexpr int V = 16 / sizeof(U);
  extern __shared__ int lds[];
  int* edges = lds;
  U* tab = (U*)(lds + kMaxSide);  // [per][buckets]
  const int h0 = blockIdx.y * per, heads = min(per, s.heads - h0);
  for (int i = threadIdx.x; i < s.count; i += 256) edges[i] = s.t[i];
  for (int i = threadIdx.x; i < heads * s.buckets; i += 256) {
    const int h = i / s.buckets, c = i - h * s.buckets;
    tab[i] = table[(int64_t)c * s.heads + h0 + h];
  }
  __syncthreads();
  const int64_t chunks = (s.n + V - 1) / V, total = batch * s.m * chunks;
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < total; id += (int64_t)gridDim.x * 256) {
    const int64_t row = id / chunks, j0 = (id - row * chunks) * V, b = row / s.m, i = row - b * s.m;
    const int64_t qp = position(s.q_pos, s.pos64, b * s.q_sb + i);
    int at[V];
#pragma unroll
    for (int e = 0; e < V; ++e)
      at[e] = bucket_of(s, edges, distance(position(s.k_pos, s.pos64, b * s.k_sb + min(j0 + e, s.n - 1)), qp));
    U* dst = out + ((b * s.heads + h0) * s.m + i) * s.n + j0;
    const U* src = tab;
    for (int h = 0; h < heads; ++h, dst += s.m * s.n, src += s.buckets) {
      union {
        U e[V];
        u32x4_u v;
      } w;
#pragma unroll
      for (int e = 0; e < V; ++e) w.e[e] = src[at[e]];
      if (j0 + V <= s.n) {
        *(u32x4_u*)dst = w.v;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (j0 + e < s.n) dst[e] = w.e[e];
      }
    }
  }
}

// Gradient.  A block sums a strip of columns over every row_blocks-th row of one (b, h)
// plane: a wave reads 64 x 16 bytes of a row, four rows in flight. Where a wave's columns all lie past the last
// threshold on one side of the row's position, which is most of a plane of running positions, the row is added
// to one sum in registers. Otherwise every thread adds to its own bin per bucket in LDS (bins[bucket][thread],
// consecutive threads in consecutive banks). Nothing is shared, so there is no atomic and the order of every
// sum is fixed. A distance's bucket comes from a byte table where the last threshold is below kLut. The bound is the
// read of dbias (16 heads, 2048 x 2048, fp32, 268 MB: 72 us, 3.7 TB/s, as a plain sum over it; right behind the forward
// pass, whose result is then still on its way to HBM, 110; LDS atomics instead of own bins 350).
constexpr int kLut = 2048, kAhead = 4;

__device__ __forceinline__ int64_t wave_extreme(int64_t v, bool largest) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const int64_t o = __shfl_xor((long long)v, m, kWave);
    v = (o > v) == largest ? o : v;
  }
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

template <typename T>
__global__ __launch_bounds__(256) void relative_bias_bwd_kernel(Relative s, const T* dbias, int waves_across,
                                                                int64_t row_blocks, int64_t col_blocks,
                                                                uint32_t blocks, float* partial) {
  constexpr int V = 16 / sizeof(T);
  extern __shared__ int lds[];
  const int threads = blockDim.x, t = threadIdx.x;
  const uint32_t block = block_index();
  if (block >= blocks) return;
  int* edges = lds;
  uint8_t* lut = (uint8_t*)(lds + kMaxSide);
  float* bins = (float*)(lds + kMaxSide + kLut / 4);
  for (int i = t; i < s.count; i += threads) edges[i] = s.t[i];
  for (int i = t; i < s.buckets * threads; i += threads) bins[i] = 0.f;
  __syncthreads();
  const int last = s.count ? s.t[s.count - 1] : 1;  // every distance from here on is in one bucket
  const bool small = last < kLut;
  if (small)
    for (int i = t; i <= last; i += threads) lut[i] = (uint8_t)bucket_of(s, edges, -i);
  __syncthreads();
  const int64_t cb = block % col_blocks, rest = block / col_blocks;
  const int64_t rb = rest % row_blocks, plane = rest / row_blocks, b = plane / s.heads;
  // The row blocks take rows in turn, so that rows near the diagonal, which cost more, are dealt to all of them.
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6), down = threads / 64 / waves_across;
  const int64_t step = down * row_blocks;
  const int64_t j0 = ((cb * waves_across + wave % waves_across) * 64 + lane_id()) * V;
  const int held = (int)max(min(s.n - j0, (int64_t)V), (int64_t)0);  // the lane's columns
  const bool whole = __all(held == V);
  int64_t kp[V], least = INT64_MAX, most = INT64_MIN;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    kp[e] = position(s.k_pos, s.pos64, b * s.k_sb + min(j0 + e, s.n - 1));
    least = min(least, kp[e]), most = max(most, kp[e]);
  }
  // Rows up to `ahead` have every column past the thresholds ahead of them, rows from `behind` on behind them.
  const int64_t ahead = wave_extreme(least, false) - (s.bidirectional ? last : 1), behind = wave_extreme(most, true) + last;
  float far_ahead = 0.f, far_behind = 0.f;
  auto add = [&](int64_t qp, const float (&v)[V]) {
    if (qp <= ahead || qp >= behind) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) sum += v[e];
      qp <= ahead ? far_ahead += sum : far_behind += sum;
      return;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int d = distance(kp[e], qp);
      const int n = d < 0 ? -d : (s.bidirectional ? d : 0);
      const int c = small ? lut[min(n, last)] + (s.bidirectional && d > 0 ? s.count + 1 : 0) : bucket_of(s, edges, d);
      bins[c * threads + t] += v[e];
    }
  };
  const T* src = dbias + plane * s.m * s.n;
  int64_t i = rb * down + wave / waves_across;
  if (whole) {
    for (; i < s.m; i += kAhead * step) {  // rows past the plane read its last one and add nothing
      union {
        T e[V];
        u32x4_u v;
      } w[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) w[u].v = *(const u32x4_u*)(src + min(i + u * step, s.m - 1) * s.n + j0);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (i + u * step >= s.m) break;
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (float)w[u].e[e];
        add(position(s.q_pos, s.pos64, b * s.q_sb + i + u * step), v);
      }
    }
  } else {
    for (; i < s.m; i += step) {
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = e < held ? (float)src[i * s.n + j0 + e] : 0.f;
      add(position(s.q_pos, s.pos64, b * s.q_sb + i), v);
    }
  }
  bins[s.count * threads + t] += far_behind;
  bins[(s.bidirectional ? 2 * s.count + 1 : 0) * threads + t] += far_ahead;
  __syncthreads();
  // one wave per bucket in turn
  const int lane = t & 63, waves = threads / 64;
  for (int c = t / 64; c < s.buckets; c += waves) {
    float v = 0.f;
    for (int i = lane; i < threads; i += 64) v += bins[c * threads + i];
    v = wave_sum_full(v);
    if (lane == 0) partial[(int64_t)block * s.buckets + c] = v;
  }
}

// dtable[c][h] from the partial rows of all blocks of head h: a block per (h, c), in a fixed order.
template <typename T>
__global__ __launch_bounds__(64) void relative_table_grad_kernel(const float* partial, int64_t batch, int heads,
                                                                 int buckets, int64_t blocks, T* dtable) {
  const int h = blockIdx.x % heads, c = blockIdx.x / heads;
  float v = 0.f;
  for (int64_t i = threadIdx.x; i < batch * blocks; i += 64) {
    const int64_t b = i / blocks, at = (b * heads + h) * blocks + (i - b * blocks);
    v += partial[at * buckets + c];
  }
  v = wave_sum_full(v);
  if (threadIdx.x == 0) dtable[(int64_t)c * heads + h] = (T)v;
}

struct BwdPlan {
  int threads, across;  // waves of a block side by side
  int64_t row_blocks, col_blocks, blocks;
};

// Threads by the bins' LDS (64 KB at most); waves of a block side by side as the plane is wide,
// rows so that a wave reads about 64, fewer where that leaves under four blocks a compute unit.
BwdPlan bwd_plan(int dtype, int64_t buckets, int64_t planes, int64_t m, int64_t n) {
  BwdPlan p;
  const int64_t wide = 64 * (dtype == kF32 ? 4 : 8);
  p.threads = buckets <= 64 ? 256 : buckets <= 128 ? 128 : 64;
  p.across = p.threads / 64;
  while (p.across > 1 && p.across / 2 * wide >= n) p.across /= 2;
  p.col_blocks = (n + p.across * wide - 1) / (p.across * wide);
  const int64_t step = p.threads / 64 / p.across;
  int64_t turns = 64;
  while (turns > 4 && planes * p.col_blocks * ((m + step * turns - 1) / (step * turns)) < 1024) turns /= 2;
  p.row_blocks = (m + step * turns - 1) / (step * turns);
  p.blocks = p.row_blocks * p.col_blocks;
  return p;
}

int setup(Relative& s, int dtype, int64_t buckets, int64_t heads, const void* q_pos, const void* k_pos, int pos64,
          int64_t batch, int64_t m, int64_t n, int64_t q_sb, int64_t k_sb, const int32_t* thresholds, int count,
          int bidirectional) {
  BMX_REQUIRE(dtype == kF32 || dtype == kBF16, "relative_bias: dtype must be fp32 or bf16");
  BMX_REQUIRE(buckets >= 1 && buckets <= kMaxBuckets, "relative_bias: buckets must be in [1, %d]", kMaxBuckets);
  BMX_REQUIRE(heads >= 1 && heads <= 65535, "relative_bias: heads must be in [1, 65535]");
  BMX_REQUIRE(batch >= 0 && m >= 0 && n >= 0, "relative_bias: negative size");
  BMX_REQUIRE(count >= 0 && count < kMaxSide && (count == 0 || thresholds), "relative_bias: bad thresholds");
  BMX_REQUIRE((bidirectional ? 2 : 1) * (int64_t)(count + 1) == buckets,
              "relative_bias: the thresholds do not give this many buckets");
  for (int i = 0; i < count; ++i)
    BMX_REQUIRE(thresholds[i] >= 1 && thresholds[i] <= kMaxDistance && (i == 0 || thresholds[i - 1] <= thresholds[i]),
                "relative_bias: thresholds must be positive and rising");
  s.q_pos = q_pos, s.k_pos = k_pos, s.pos64 = pos64, s.q_sb = q_sb, s.k_sb = k_sb, s.m = m, s.n = n;
  s.heads = (int)heads, s.buckets = (int)buckets, s.bidirectional = bidirectional != 0, s.count = count, s.exact = 0;
  for (int i = 0; i < count; ++i) {
    s.t[i] = thresholds[i];
    if (s.exact == i && thresholds[i] == i + 1) s.exact = i + 1;
  }
  return BMX_OK;
}

}  // namespace

extern "C" int bmx_relative_bias_fwd(const void* table, int dtype, int64_t buckets, int64_t heads, const void* q_pos,
                                     const void* k_pos, int pos64, int64_t batch, int64_t m, int64_t n, int64_t q_sb,
                                     int64_t k_sb, const int32_t* thresholds, int count, int bidirectional, void* out,
                                     void* stream) {
  Relative s;
  if (int rc = setup(s, dtype, buckets, heads, q_pos, k_pos, pos64, batch, m, n, q_sb, k_sb, thresholds, count,
                     bidirectional))
    return rc;
  if (batch == 0 || m == 0 || n == 0) return BMX_OK;
  BMX_REQUIRE(table && q_pos && k_pos && out, "relative_bias: null pointer");
  const int elem = dtype == kF32 ? 4 : 2, vec = 16 / elem;
  const int64_t blocks = (batch * m * ((n + vec - 1) / vec) + 255) / 256;
  // Heads of a thread: all that 32 KB of table hold, fewer where that leaves less than four blocks a compute unit
  // (a single query row writes in one short wave of blocks, one head each).
  int64_t per = 32768 / (elem * buckets);
  per = per < heads ? per : heads;
  while (per > 1 && blocks * ((heads + per - 1) / per) < 1024) per = (per + 1) / 2;
  const size_t lds = kMaxSide * 4 + (size_t)per * buckets * elem;
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)), (unsigned)((heads + per - 1) / per));
  hipStream_t hs = (hipStream_t)stream;
  if (dtype == kF32)
    relative_bias_kernel<uint32_t><<<grid, 256, lds, hs>>>(s, (const uint32_t*)table, batch, (int)per, (uint32_t*)out);
  else
    relative_bias_kernel<uint16_t><<<grid, 256, lds, hs>>>(s, (const uint16_t*)table, batch, (int)per, (uint16_t*)out);
  return check_launch("relative_bias");
}

extern "C" size_t bmx_relative_bias_workspace_bytes(int dtype, int64_t buckets, int64_t heads, int64_t batch, int64_t m,
                                                    int64_t n) {
  if (buckets < 1 || heads < 1 || batch < 1 || m < 1 || n < 1) return 0;
  return (size_t)(bwd_plan(dtype, buckets, batch * heads, m, n).blocks * batch * heads * buckets) * sizeof(float);
}

extern "C" int bmx_relative_bias_bwd(const void* dbias, int dtype, int64_t buckets, int64_t heads, const void* q_pos,
                                     const void* k_pos, int pos64, int64_t batch, int64_t m, int64_t n, int64_t q_sb,
                                     int64_t k_sb, const int32_t* thresholds, int count, int bidirectional,
                                     void* dtable, void* workspace, size_t workspace_bytes, void* stream) {
  Relative s;
  if (int rc = setup(s, dtype, buckets, heads, q_pos, k_pos, pos64, batch, m, n, q_sb, k_sb, thresholds, count,
                     bidirectional))
    return rc;
  BMX_REQUIRE(dtable, "relative_bias_bwd: null pointer");
  const bool any = batch > 0 && m > 0 && n > 0;
  BwdPlan p = {};
  hipStream_t hs = (hipStream_t)stream;
  if (any) {
    BMX_REQUIRE(dbias && q_pos && k_pos, "relative_bias_bwd: null pointer");
    BMX_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0 &&
                    workspace_bytes >= bmx_relative_bias_workspace_bytes(dtype, buckets, heads, batch, m, n),
                "relative_bias_bwd: workspace too small or not 16-byte aligned");
    p = bwd_plan(dtype, buckets, batch * heads, m, n);
    const int64_t blocks = p.blocks * batch * heads;
    BMX_REQUIRE(blocks < (1ll << 31), "relative_bias_bwd: too many elements");
    const size_t lds = kMaxSide * 4 + kLut + (size_t)buckets * p.threads * 4;
    const dim3 grid = fold_grid(blocks, p.threads);
    if (dtype == kF32)
      relative_bias_bwd_kernel<float><<<grid, p.threads, lds, hs>>>(s, (const float*)dbias, p.across, p.row_blocks,
                                                                    p.col_blocks, (uint32_t)blocks, (float*)workspace);
    else
      relative_bias_bwd_kernel<bf16><<<grid, p.threads, lds, hs>>>(s, (const bf16*)dbias, p.across, p.row_blocks,
                                                                   p.col_blocks, (uint32_t)blocks, (float*)workspace);
  }
  const dim3 grid((unsigned)(heads * buckets));
  const int64_t rows = any ? batch : 0;  // nothing to sum: a gradient of zeros
  if (dtype == kF32)
    relative_table_grad_kernel<<<grid, 64, 0, hs>>>((const float*)workspace, rows, (int)heads, (int)buckets, p.blocks,
                                                    (float*)dtable);
  else
    relative_table_grad_kernel<<<grid, 64, 0, hs>>>((const float*)workspace, rows, (int)heads, (int)buckets, p.blocks,
                                                    (bf16*)dtable);
  return check_launch("relative_bias_bwd");
}
