// Softmax cross entropy of points against centroids, and its gradients.
//
//   z[n, k] = scale * x[n] . c[k],   d[n, k] = z[n, k] - z[n, y_n]
//   loss[n] = log sum_k exp(d[n, k]) = log1p(sum_{k != y} exp(d))   (d <= 0)
//   dz[n, k] = w_n (softmax(z[n])[k] - [k == y_n])
//   dx = scale * dz . c,   dc = scale * dz^T . x
//
// The (N, K) scores never reach memory.  The forward pass is one product whose
// epilogue keeps each row's running maximum and sum of exponentials over the
// centroids other than the label; a small kernel joins the column chunks.  The
// label's term stays out of the sum because a well-fitted row's loss is
// log1p of what the others add, and 1 + that in 32 bits would round it away.
//
// The backward pass goes over the centroids in pieces.  For each it recomputes
// the scores, writes dz of the piece rounded to 16 bits (the operand type of
// the tensor cores: one rounding of half a step at most, next to the rounding
// of the 16-bit gradients themselves; what it takes from the label's entry is
// added to dx again) and runs the two products that read it,
// in one launch whose workers finish together; accumulators are float32
// throughout.  That is 8 N K D operations instead of the 6 N K D of a pass that
// keeps N x K scores.
//
// Measured alone at 16384 x 32768 x 1024 bfloat16 with 15 % of the rows ignored:
// forward product 580 us, combine 19, four pieces of 158 (scores again, dz) and
// 324 to 338 (both gradients), 1.5 PFLOP/s; back to back the power cap stretches
// the 2.7 ms to 3.1.  With 128 features (32444 x 8192) the forward product keeps
// the special-function units 74 % busy (108 us); each of two backward pieces writes
// 0.2 GB of dz to memory (80 us) and reads it twice, 0.38 GB of that from memory
// (94 us).
//
// float32 inputs are split exactly into three bf16 parts, and the six products
// of parts down to 2^-16 of the leading one are accumulated, smallest first:
// the terms left out are below 2^-24 of |x||c|.  That costs what 3xTF32 costs
// and keeps one kernel, MN-major operands included (8192 x 1024 x 512, loss and
// gradients: 0.23 ms, errors a fifth of plain float32's).
#include <algorithm>
#include <cmath>

#include "fk_head_launch.cuh"

namespace fk {
namespace head {

// 16-bit P elements of a piece: 256 MB, so that a piece's products have whole
// waves of tiles, and the float32 sums carried between pieces are few.
constexpr int64_t kPieceElems = 1ll << 27;
constexpr int64_t kMaxRowChunk = 16384;

int encode_operand(CUtensorMap* map, const Operand& o, uint32_t box_rows) {
  const int64_t eb = o.dtype == FK_I8 ? 1 : 2;
  const uint32_t box0 = o.dtype == FK_I8 ? 128 : 64;
  // (one matrix: its distance to the next is never used, but has to be encodable)
  return encode_tmap_3d(map, o.p, o.dtype, o.inner, o.rows, o.mats, o.ld * eb,
                        (o.mats > 1 ? o.mat : o.ld) * eb, box0, box_rows);
}

// ------------------------------------------------------------ operand copies
// Rows of x as the tensor cores read them: padded to 16 bytes, zeros past D,
// float32 as three bf16 parts.  With labels, ignored rows become zeros, so that
// whatever a padded position holds (NaN included) adds nothing to dc.
__device__ __forceinline__ void split3(float v, uint16_t (&p)[3]) {
  uint32_t h = pack_bf16(v, 0.0f) & 0xffffu;
  if ((h & 0x7f80u) == 0x7f80u && fabsf(v) <= 3.40282347e38f)
    h = __float_as_uint(v) >> 16;  // would round past the largest bf16: truncate
  p[0] = static_cast<uint16_t>(h);
  const float hf = __uint_as_float(h << 16);
  float r = fabsf(v) <= 3.40282347e38f ? v - hf : 0.0f;  // inf, NaN: all in the first part
  h = pack_bf16(r, 0.0f) & 0xffffu;
  p[1] = static_cast<uint16_t>(h);
  r -= __uint_as_float(h << 16);
  p[2] = static_cast<uint16_t>(pack_bf16(r, 0.0f) & 0xffffu);
}

struct Labels {
  const void* p = nullptr;
  int dtype = FK_I32;
  int64_t sb = 0, sn = 0;
  int64_t ignore = -100;
};

struct RowsJob {        // one tensor to copy; units = 0 for none
  const void* x;
  int64_t sb, sn, sd;
  int vec;              // rows can be read 16 bytes at a time
  uint16_t* out;
  int64_t part;         // elements from one part to the next
  int N, D, Dp;
  int64_t units;        // of eight elements
  Labels y;             // p: ignored rows become zeros
  const int32_t* map;   // gathered rows: row r of the copy is row map[r] of x
  const int32_t* live;  // and there are this many, zeros up to the next 128 behind them
};
struct RowsJobs {
  RowsJob job[2];
};

template <typename T>
__global__ void head_rows_kernel(const RowsJobs jobs) {
  pdl_wait_then_release();
  const RowsJob& j = jobs.job[blockIdx.y];
  const T* x = static_cast<const T*>(j.x);
  const int per = j.Dp / 8, D = j.D;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; u < j.units;
       u += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t row = u / per;
    const int d0 = static_cast<int>(u - row * per) * 8;
    int64_t b = row / j.N, n = row - b * j.N;
    T v[8];
    bool zero = j.y.p && load_label(j.y.p, b * j.y.sb + n * j.y.sn, j.y.dtype) == j.y.ignore;
    if (j.map) {
      const int live = *j.live;
      if (row >= (static_cast<int64_t>(live) + 127) / 128 * 128) break;
      zero = row >= live;
      b = 0;
      n = zero ? 0 : j.map[row];
    }
    const T* src = x + b * j.sb + n * j.sn;
    if (zero) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = Elem<T>::from_f(0.0f);
    } else if (j.vec && d0 + 8 <= D) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
        reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(src + d0)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = d0 + i < D ? src[(d0 + i) * j.sd] : Elem<T>::from_f(0.0f);
    }
    uint16_t* dst = j.out + row * j.Dp + d0;
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(v);
    } else {
      uint16_t p[8][3];
#pragma unroll
      for (int i = 0; i < 8; ++i) split3(v[i], p[i]);
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        uint4 w;
        uint32_t* ww = &w.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) ww[i] = p[2 * i][q] | static_cast<uint32_t>(p[2 * i + 1][q]) << 16;
        *reinterpret_cast<uint4*>(dst + q * j.part) = w;
      }
    }
  }
}

static RowsJob rows_job(const void* x, int dtype, int64_t B, int64_t N, int64_t D, const int64_t* xs,
                        uint16_t* out, int64_t Dp, const Labels* y) {
  RowsJob j = {};
  if (!out) return j;
  const int64_t eb = dtype_bytes(dtype);
  j.x = x;
  j.sb = xs[0];
  j.sn = xs[1];
  j.sd = xs[2];
  j.vec = (xs[2] == 1 || D == 1) && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
          (N == 1 || xs[1] * eb % 16 == 0) && (B == 1 || xs[0] * eb % 16 == 0);
  j.out = out;
  j.part = B * N * Dp;
  j.N = static_cast<int>(N);
  j.D = static_cast<int>(D);
  j.Dp = static_cast<int>(Dp);
  j.units = B * N * (Dp / 8);
  if (y) j.y = *y;
  return j;
}

// Both copies in one launch.
static int rows_copy(int dtype, const RowsJob& a, const RowsJob& b, cudaStream_t s) {
  RowsJobs jobs = {{a.units ? a : b, b}};
  const int n = (a.units ? 1 : 0) + (b.units ? 1 : 0);
  if (n == 0) return FK_OK;
  const int sms = sm_count_current();
  const int64_t cap = (sms > 0 ? sms : 148) * 16ll;
  const dim3 grid(static_cast<unsigned>(std::min(ceil_div(std::max(a.units, b.units), 256), cap)), n);
  switch (dtype) {
    case FK_F16: return launch_plain("head_rows_kernel", head_rows_kernel<__half>, grid, 256, s, jobs);
    case FK_BF16: return launch_plain("head_rows_kernel", head_rows_kernel<__nv_bfloat16>, grid, 256, s, jobs);
    default: return launch_plain("head_rows_kernel", head_rows_kernel<float>, grid, 256, s, jobs);
  }
}

// ------------------------------------------------------------------ combine
// Sixteen warps join the column chunks of 32 rows and sum the label's score of
// two rows each; block sums of the losses go to `block_part`, and the last
// block adds them up in block order, so the result does not depend on which
// block came last.  What bounds this kernel is the chain of dependent loads
// (label, centroid row, partial results), so a warp's rows and chunks are in flight
// together.
constexpr int kCombineWarps = 16;
constexpr int kRowsPerWarp = 32 / kCombineWarps;

struct CombineParams {
  const float2* partial;   // [batch][pieces][N]
  const void *x, *c;       // for the label's score
  int dtype, D, vec;       // vec: rows of both can be read 16 bytes at a time
  int64_t xs[3], cs[3];
  float scale, scale2;     // scale2: times log2(e)
  const void* labels;
  int label_dtype;
  int64_t lb, ln, ignore;
  int64_t K;
  int N, pieces, row_blocks;
  int reduction;           // 0 none, 1 mean, 2 sum
  float* loss;             // rows [batch][N], or one value
  RowStat* stat;           // optional
  int32_t* count;          // rows that are not ignored
  double2* block_part;     // (sum, count) of each block
  uint32_t* ticket;        // zero before the launch
  const int32_t *map, *live;  // gathered rows (see xent_live_kernel), null: all, in order
  uint16_t* copy;          // optional: x's rows, 16-bit, Dp apart, ignored ones as zeros
  int Dp;
  int* status;
};

// x[n] . c[y] of a warp's rows, in float32 (each lane's partial sum, then a tree).
template <typename T>
__device__ __forceinline__ void row_dots(const CombineParams& p, int b, const int64_t (&n)[kRowsPerWarp],
                                         const int64_t (&y)[kRowsPerWarp], const bool (&on)[kRowsPerWarp],
                                         int lane, float (&z)[kRowsPerWarp]) {
  constexpr int E = 16 / sizeof(T);
  const T *x[kRowsPerWarp], *c[kRowsPerWarp];
#pragma unroll
  for (int i = 0; i < kRowsPerWarp; ++i) {
    x[i] = static_cast<const T*>(p.x) + (on[i] ? b * p.xs[0] + n[i] * p.xs[1] : 0);
    c[i] = static_cast<const T*>(p.c) + (on[i] ? b * p.cs[0] + y[i] * p.cs[1] : 0);
    z[i] = 0.0f;
  }
  int d = 0;
  if (p.vec) {
    for (d = lane * E; d + E <= p.D; d += 32 * E) {
      uint4 a[kRowsPerWarp], w[kRowsPerWarp];
#pragma unroll
      for (int i = 0; i < kRowsPerWarp; ++i)
        if (on[i]) {
          a[i] = *reinterpret_cast<const uint4*>(x[i] + d);
          w[i] = *reinterpret_cast<const uint4*>(c[i] + d);
        }
#pragma unroll
      for (int i = 0; i < kRowsPerWarp; ++i)
        if (on[i]) {
          const T *pa = reinterpret_cast<const T*>(&a[i]), *pb = reinterpret_cast<const T*>(&w[i]);
#pragma unroll
          for (int k = 0; k < E; ++k) z[i] = fmaf(Elem<T>::to_f(pa[k]), Elem<T>::to_f(pb[k]), z[i]);
        }
    }
    d = p.D / E * E;
  }
  for (d += lane; d < p.D; d += 32)
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i)
      if (on[i]) z[i] = fmaf(Elem<T>::to_f(x[i][d * p.xs[2]]), Elem<T>::to_f(c[i][d * p.cs[2]]), z[i]);
#pragma unroll
  for (int i = 0; i < kRowsPerWarp; ++i) z[i] = warp_sum(z[i]);
}

__global__ void __launch_bounds__(kCombineWarps * 32) xent_combine_kernel(const CombineParams p) {
  __shared__ float2 sm[kCombineWarps][33];
  __shared__ float z_label[32];
  __shared__ double2 red[kCombineWarps];
  __shared__ bool last;
  pdl_wait_then_release();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / p.row_blocks;
  const int row = (blockIdx.x % p.row_blocks) * 32 + lane;
  const int rows = p.live ? *p.live : p.N;
  const float2* part = p.partial + static_cast<int64_t>(b) * p.pieces * p.N + row;
  float m = -INFINITY, s = 0.0f;
  if (row < rows) {
    for (int i0 = warp; i0 < p.pieces; i0 += 4 * kCombineWarps) {
      float2 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = i0 + i * kCombineWarps;
        v[i] = k < p.pieces ? part[static_cast<int64_t>(k) * p.N] : make_float2(-INFINITY, 0.0f);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float mn = fmaxf(m, v[i].x);
        const float mu = mn == -INFINITY ? 0.0f : mn;
        // a piece whose exponents were NaN has a NaN sum, which stays
        s = s * ex2((m - mu) * p.scale2) + v[i].y * ex2((v[i].x - mu) * p.scale2);
        m = mn;
      }
    }
  }
  sm[warp][lane] = make_float2(m, s);
  {
    int64_t n[kRowsPerWarp], y[kRowsPerWarp];
    bool on[kRowsPerWarp];
    float z[kRowsPerWarp];
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) {
      n[i] = (blockIdx.x % p.row_blocks) * 32 + warp * kRowsPerWarp + i;
      on[i] = n[i] < rows;
      if (on[i] && p.map) n[i] = p.map[n[i]];
    }
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i)
      y[i] = on[i] ? load_label(p.labels, b * p.lb + n[i] * p.ln, p.label_dtype) : p.ignore;
#pragma unroll
    for (int i = 0; i < kRowsPerWarp; ++i) on[i] = on[i] && y[i] != p.ignore && y[i] >= 0 && y[i] < p.K;
    if (p.copy) {
      // the backward pass's copy of x (see head_rows_kernel), while the rows are at hand
#pragma unroll
      for (int i = 0; i < kRowsPerWarp; ++i) {
        if (n[i] >= p.N) continue;
        const uint16_t* src = static_cast<const uint16_t*>(p.x) + b * p.xs[0] + n[i] * p.xs[1];
        uint16_t* dst = p.copy + (static_cast<int64_t>(b) * p.N + n[i]) * p.Dp;
        for (int d = lane * 8; d < p.Dp; d += 256) {
          uint4 u = make_uint4(0, 0, 0, 0);
          if (y[i] != p.ignore) {
            if (d + 8 <= p.D) {
              u = *reinterpret_cast<const uint4*>(src + d);
            } else {
              uint16_t* v = reinterpret_cast<uint16_t*>(&u);
#pragma unroll
              for (int k = 0; k < 8; ++k)
                if (d + k < p.D) v[k] = src[d + k];
            }
          }
          *reinterpret_cast<uint4*>(dst + d) = u;
        }
      }
    }
    if (p.dtype == FK_F32) row_dots<float>(p, b, n, y, on, lane, z);
    else if (p.dtype == FK_F16) row_dots<__half>(p, b, n, y, on, lane, z);
    else row_dots<__nv_bfloat16>(p, b, n, y, on, lane, z);
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < kRowsPerWarp; ++i) z_label[warp * kRowsPerWarp + i] = z[i];
  }
  __syncthreads();
  double sum = 0.0, cnt = 0.0;
  if (warp == 0) {
    for (int w = 1; w < kCombineWarps; ++w) {
      const float2 v = sm[w][lane];
      const float mn = fmaxf(m, v.x);
      const float mu = mn == -INFINITY ? 0.0f : mn;
      s = s * ex2((m - mu) * p.scale2) + v.y * ex2((v.x - mu) * p.scale2);
      m = mn;
    }
    if (row < rows) {
      const int64_t n = p.map ? p.map[row] : row;
      const int64_t r = static_cast<int64_t>(b) * p.N + n;
      const int64_t y = load_label(p.labels, b * p.lb + n * p.ln, p.label_dtype);
      const bool ignored = y == p.ignore;
      RowStat st = {0.0f, 0.0f, 0.0f, -1};
      float loss = 0.0f;
      if (!ignored && (y < 0 || y >= p.K)) {
        loss = NAN;
        st = {0.0f, NAN, NAN, -1};
        if (p.status) atomicCAS(p.status, 0, FK_DEV_BAD_LABEL);
      } else if (!ignored) {
        const float ty = z_label[lane];
        const float d = m - ty;  // -inf for K = 1
        // sum over the others, relative to the larger of the label's term and theirs
        const float top = fmaxf(m, ty);
        const float others = s * ex2((m - top) * p.scale2);
        const float own = ex2((ty - top) * p.scale2);
        loss = d > 0.0f ? fmaf(d, p.scale, logf(others + own)) : log1pf(others);
        if (!(s == s) || !(ty < INFINITY)) loss = NAN;  // NaN scores, or inf - inf
        st.top = top;
        st.coef = 1.0f / (others + own);
        st.at_label = expm1f(-loss);
        st.label = static_cast<int>(y);
        if (!(loss == loss)) st.coef = st.at_label = NAN;
      }
      if (p.stat) p.stat[r] = st;
      if (p.reduction == 0) p.loss[r] = loss;
      sum = loss;
      cnt = ignored ? 0.0 : 1.0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      cnt += __shfl_xor_sync(0xffffffffu, cnt, o);
    }
    if (lane == 0) {
      p.block_part[blockIdx.x] = make_double2(sum, cnt);
      __threadfence();
      last = atomicAdd(p.ticket, 1u) == gridDim.x - 1;
    }
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  sum = cnt = 0.0;
  for (int i = threadIdx.x; i < static_cast<int>(gridDim.x); i += kCombineWarps * 32) {
    const double2 v = __ldcg(p.block_part + i);
    sum += v.x;
    cnt += v.y;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    cnt += __shfl_xor_sync(0xffffffffu, cnt, o);
  }
  if (lane == 0) red[warp] = make_double2(sum, cnt);
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = cnt = 0.0;
    for (int w = 0; w < kCombineWarps; ++w) {
      sum += red[w].x;
      cnt += red[w].y;
    }
    if (p.reduction == 1) *p.loss = static_cast<float>(sum / cnt);  // no row left: 0 / 0
    if (p.reduction == 2) *p.loss = static_cast<float>(sum);
    *p.count = static_cast<int32_t>(cnt);
  }
}

// --------------------------------------------------------- row weights (none)
// Losses that stay per row arrive with one upstream gradient g each, which goes
// into the row's weight.
__global__ void xent_weight_kernel(const float* g, const RowStat* stat, int64_t rows, RowStat* out) {
  pdl_wait_then_release();
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < rows;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    RowStat st = stat[i];
    const bool ignored = st.label < 0 && st.coef == 0.0f;
    if (!ignored) {
      st.coef *= g[i];
      st.at_label *= g[i];
    }
    out[i] = st;
  }
}

// float16 has 40 powers of two, which the softmax of one row alone can fill.  So
// only the part of g within [1, 2) goes into P.  The power of two is a factor of
// the row in dx; in dc, where the rows are summed, it goes into a copy of x:
// relative to the largest power of two times |x| of all rows, which sits at the
// upper end of float16 there (below 2^16; powers of two round nothing but what
// falls under 2^-14).  Gradients of every size keep their softmax that way: with
// g itself in P, a row whose gradient was 2^-20 of the largest lost the softmax
// of 40000 centroids.  The two passes over x take 75 us of 728 at 65536 x 1024 x
// 1024, 30 of 540 at 16384 x 8192 x 512.
__device__ __forceinline__ float power_of_two(int e) {   // of a normal number
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// A warp has a row; `reach` is 512 + the largest exponent found, 0 for none.
__global__ void xent_weight16_kernel(const float* g, const RowStat* stat, int64_t rows, RowStat* out,
                                     float* power, const uint16_t* x, int Dp, const int32_t* map,
                                     const int32_t* live, uint32_t* reach) {
  pdl_wait_then_release();
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  const int64_t used = live ? *live : rows;
  uint32_t most = 0;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); r < used; r += warps) {
    const int64_t i = map ? map[r] : r;
    RowStat st = stat[i];
    const bool ignored = st.label < 0 && st.coef == 0.0f;
    const float w = ignored ? 0.0f : g[i];
    const uint32_t bits = __float_as_uint(w) & 0x7fffffffu;
    const bool finite = bits < 0x7f800000u && bits != 0;
    // (a gradient below the normal numbers is left with 2^-126)
    const int e = finite ? max(static_cast<int>(bits >> 23), 1) - 127 : 0;
    if (lane == 0) {
      if (!ignored) {
        // (in two steps: 2^-127 is no normal number)
        const float m = w * power_of_two(-(e / 2)) * power_of_two(e / 2 - e);
        st.coef *= m;
        st.at_label *= m;
      }
      out[i] = st;
      power[i] = bits ? power_of_two(e) : 0.0f;
    }
    if (!x || !finite) continue;
    uint32_t top = 0;
    for (int d = lane * 8; d < Dp; d += 256) {
      const uint4 u = *reinterpret_cast<const uint4*>(x + r * Dp + d);
      const uint32_t v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t lo = v[k] & 0x7fffu, hi = (v[k] >> 16) & 0x7fffu;
        if (lo < 0x7c00u) top = max(top, lo);   // infinities and NaN stay what they are
        if (hi < 0x7c00u) top = max(top, hi);
      }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (top == 0) continue;
    int ex;
    frexpf(__half2float(__ushort_as_half(static_cast<unsigned short>(top))), &ex);
    most = max(most, static_cast<uint32_t>(512 + e + ex));
  }
  if (lane == 0 && most) atomicMax(reach, most);
}

__global__ void xent_scale16_kernel(const uint16_t* x, int64_t rows, int Dp, const float* power, const int32_t* map,
                                    const int32_t* live, const uint32_t* reach, uint16_t* out, float* factor) {
  pdl_wait_then_release();
  // |x| 2^e < 2^E: what is written is below 2^16
  const uint32_t most = *reach;
  const int E = most ? max(static_cast<int>(most) - 512, -100) : 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *factor = power_of_two(E - 16);
  const int per = Dp / 8;
  const int64_t units = rows * per;
  const int64_t used = live ? *live : rows;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; u < units;
       u += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t r = u / per;
    if (r >= (used + 127) / 128 * 128) break;
    // (rows of weight 0 are not among those that E bounds; behind the last row
    // that counts the copy holds zeros)
    const float w = r < used ? power[map ? map[r] : r] : 0.0f;
    const int e = static_cast<int>(__float_as_uint(w) >> 23) - 127;
    const float by = w > 0.0f ? power_of_two(min(max(e - E + 16, -126), 127)) : 0.0f;
    uint4 v = reinterpret_cast<const uint4*>(x)[u];
    __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = __half22float2(h[k]);
      h[k] = __floats2half2_rn(f.x * by, f.y * by);
    }
    reinterpret_cast<uint4*>(out)[u] = v;
  }
}

// ------------------------------------------------------------ rows that count
// The rows that are not ignored, in order (map[r] is the r-th of them) and how
// many there are; the losses, statistics and gradients of the others, where
// wanted, are set to zero here.  A block has a segment of the rows.  What lies
// before it is counted by a launch in front (`counts`, one a segment) or, where
// the labels are few, by the block itself.
constexpr int kLiveThreads = 1024;
constexpr int kLiveSegments = 128;

// Sum of all threads' v, in the first warp's lanes.
__device__ __forceinline__ int block_count(int v, int (&sm)[32]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  v = __reduce_add_sync(0xffffffffu, v);
  if (lane == 0) sm[warp] = v;
  __syncthreads();
  return warp == 0 ? __reduce_add_sync(0xffffffffu, sm[lane]) : 0;
}

__global__ void __launch_bounds__(kLiveThreads) xent_count_kernel(const Labels y, int64_t N, int64_t segment,
                                                                  int32_t* counts) {
  __shared__ int sm[32];
  pdl_wait_then_release();
  const int64_t first = blockIdx.x * segment, last = min(first + segment, N);
  int n = 0;
#pragma unroll 4
  for (int64_t i = first + threadIdx.x; i < last; i += kLiveThreads)
    n += load_label(y.p, i * y.sn, y.dtype) != y.ignore;
  n = block_count(n, sm);
  if (threadIdx.x == 0) counts[blockIdx.x] = n;
}

__global__ void __launch_bounds__(kLiveThreads) xent_live_kernel(const Labels y, int64_t N, int64_t segment,
                                                                 const int32_t* counts,
                                                                 int32_t* map, int32_t* live, float* loss,
                                                                 RowStat* stat, void* gx, int64_t gx_row,
                                                                 int64_t gx_bytes, int gx_vec) {
  __shared__ int sm[32];
  __shared__ int base;
  pdl_wait_then_release();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t first = blockIdx.x * segment, last = min(first + segment, N);
  int before = 0;
  if (counts) {
    if (tid < static_cast<int>(blockIdx.x)) before = counts[tid];
  } else {
#pragma unroll 4
    for (int64_t n = tid; n < first; n += kLiveThreads) before += load_label(y.p, n * y.sn, y.dtype) != y.ignore;
  }
  before = block_count(before, sm);
  if (tid == 0) base = before;
  __syncthreads();
  for (int64_t n0 = first; n0 < last; n0 += kLiveThreads) {
    const int64_t n = n0 + tid;
    const bool on = n < last && load_label(y.p, n * y.sn, y.dtype) != y.ignore;
    const uint32_t votes = __ballot_sync(0xffffffffu, on);
    if (lane == 0) sm[warp] = __popc(votes);
    __syncthreads();
    int at = base;
    for (int w = 0; w < warp; ++w) at += sm[w];
    if (on) map[at + __popc(votes & ((1u << lane) - 1))] = static_cast<int32_t>(n);
    if (n < last && !on) {
      if (loss) loss[n] = 0.0f;
      if (stat) stat[n] = {0.0f, 0.0f, 0.0f, -1};
    }
    if (gx) {
      for (uint32_t off = __ballot_sync(0xffffffffu, n < last && !on); off; off &= off - 1) {
        uint8_t* row = static_cast<uint8_t*>(gx) + (n0 + warp * 32 + __ffs(off) - 1) * gx_row;
        if (gx_vec) {
          for (int64_t k = lane * 16; k < gx_bytes; k += 512)
            *reinterpret_cast<uint4*>(row + k) = make_uint4(0, 0, 0, 0);
        } else {
          for (int64_t k = lane * 2; k < gx_bytes; k += 64) *reinterpret_cast<uint16_t*>(row + k) = 0;
        }
      }
    }
    __syncthreads();
    if (tid == 0) {
      int t = base;
      for (int w = 0; w < 32; ++w) t += sm[w];
      base = t;
    }
    __syncthreads();
  }
  if (tid == 0 && last == N) *live = base;
}

// -------------------------------------------------------------------- plans
struct Bump {  // workspace layout: the same walk sizes it and hands it out
  uint8_t* base;
  size_t used = 0;
  template <typename T>
  T* take(int64_t n) {
    T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += align_up(static_cast<size_t>(n) * sizeof(T), 256);
    return p;
  }
};

struct Xent {
  const void *x, *c;
  int dtype;
  int64_t B, N, K, D;
  int64_t xs[3], cs[3];
  Labels y;
  float scale;
  int reduction;

  int parts() const { return dtype == FK_F32 ? 3 : 1; }
  int mma_dtype() const { return dtype == FK_F16 ? FK_F16 : FK_BF16; }
  int64_t Dp() const { return ceil_div(D, 8) * 8; }
  int64_t Bc() const { return cs[0] == 0 ? 1 : B; }  // batches with centroids of their own
};

// Operand over a caller's tensor (used in place) or its copy in the workspace.
static bool in_place(const void* p, int dtype, int64_t B, int64_t M, int64_t D, const int64_t* st) {
  if (dtype == FK_F32 || (B > 1 && st[0] == 0)) return false;
  int64_t s[3] = {st[0], st[1], D == 1 ? 1 : st[2]};
  if (M == 1) s[1] = ceil_div(D, 8) * 8;
  if (B == 1) s[0] = M * s[1];
  return fk_tma_compatible(p, dtype, D, s) != 0;
}

static Operand operand(const Xent& q, const void* p, const uint16_t* copy, int64_t B, int64_t M,
                       const int64_t* st, bool mn, int64_t off) {
  Operand o;
  o.dtype = q.mma_dtype();
  o.inner = q.D;
  o.rows = M;
  o.mn = mn;
  o.off = off;
  if (copy) {
    o.p = copy;
    o.ld = q.Dp();
    o.mat = M * q.Dp();
    o.mats = B * q.parts();
    o.part_step = static_cast<int>(B);
  } else {
    o.p = p;
    o.ld = M == 1 ? q.Dp() : st[1];
    o.mat = st[0];
    o.mats = B;
    o.part_step = 0;
  }
  o.batch_step = B > 1 ? 1 : 0;
  return o;
}

static int check_args(const Xent& q, const char* who) {
  if (q.B < 0 || q.N < 0 || q.K <= 0 || q.D <= 0) return fail(FK_ERR_INVALID_ARG, "%s: bad sizes", who);
  if (q.dtype != FK_F16 && q.dtype != FK_BF16 && q.dtype != FK_F32)
    return fail(FK_ERR_INVALID_ARG, "%s: unsupported dtype %d", who, q.dtype);
  if (q.y.dtype != FK_I32 && q.y.dtype != FK_I64)
    return fail(FK_ERR_INVALID_ARG, "%s: labels must be int32 or int64", who);
  if (q.reduction < 0 || q.reduction > 2) return fail(FK_ERR_INVALID_ARG, "%s: bad reduction", who);
  if (!(q.scale > 0.0f) || !std::isfinite(q.scale) || !std::isfinite(q.scale * 1.44269504f))
    return fail(FK_ERR_INVALID_ARG, "%s: scale must be positive and finite", who);
  if (q.N >= (1ll << 30) || q.K >= (1ll << 30) || q.D >= (1ll << 30) || q.B * 3 >= (1ll << 30) ||
      q.B * q.N >= (1ll << 31))
    return fail(FK_ERR_UNSUPPORTED, "%s: sizes exceed 32-bit", who);
  // (expanded centroids can have any size: no workspace may wrap around)
  if (static_cast<double>(q.B) * static_cast<double>(q.K) * static_cast<double>(q.D) >= 0x1p58)
    return fail(FK_ERR_UNSUPPORTED, "%s: sizes exceed 64-bit", who);
  return FK_OK;
}

static int check_workspace(const void* ws, size_t have, size_t need, const char* who) {
  if (need == 0) return FK_OK;
  if (!ws || have < need || reinterpret_cast<uintptr_t>(ws) % 256)
    return fail(FK_ERR_WORKSPACE, "%s: workspace of %zu bytes (256-byte aligned) needed, %zu given", who,
                need, have);
  return FK_OK;
}

// Whether ignored rows are left out of the products.  Finding them takes 10 us;
// where x is copied in any case (the backward pass, float32) gathering adds
// nothing to that.  Loss and gradients with none / a tenth / half of the rows
// ignored, gathered to not: 16384 x 8192 x 512 bfloat16 1.00 / 0.98 / 0.63, 65536
// x 256 x 4096 1.06 / 1.00 / 0.65; the largest loss seen, 1.10 / 1.02 / 0.67, was at
// 2^20 x 1024 x 128.  Below 2^36 products a call is too short for the 10 us.
// Separate codebooks keep one block of rows for each batch, and go without.
static bool gathers(const Xent& q) { return q.B == 1 && q.N >= 1024 && q.N * q.K >= (1ll << 36) / q.D; }

// The forward pass alone reads 16-bit rows in place, and gathering them costs a
// copy of x, which does not shrink with the centroids as the products do: with
// none / a tenth / half of the rows ignored, gathered to not, 65536 x 256 x 4096
// takes 1.89 / 1.85 / 1.27, 65536 x 1024 x 1024 1.45 / 1.43 / 0.97, 65536 x 4096 x 1024
// 1.15 / 1.2 / 0.70, 16384 x 8192 x 512 1.13 / 1.12 / 0.73, 16384 x 32768 x 1024 1.04 /
// 1.0 / 0.58.
static bool gathers_forward(const Xent& q) {
  return gathers(q) && (q.K >= 8192 || !in_place(q.x, q.dtype, q.B, q.N, q.D, q.xs));
}

// The rows' indices, their number, and the segments' counts.
static int64_t map_words(const Xent& q) { return q.N + 1 + kLiveSegments; }

// Rows up to which a block counts all labels before its own: the last one reads
// nearly all of them, which takes longer than a launch that counts them from
// 65536 int64 labels on (5 us longer; 25 at 262144, 125 at 2^20; none at 16384).
constexpr int64_t kLiveAlone = 32768;

// Finds the rows that count: map gets N + 1 words, their number the last.
static int find_live(const Xent& q, int32_t* map, float* loss, RowStat* stat, void* gx, int64_t gx_row,
                     cudaStream_t s) {
  const int64_t segment = ceil_div(ceil_div(q.N, kLiveSegments), kLiveThreads) * kLiveThreads;
  const dim3 blocks(static_cast<unsigned>(ceil_div(q.N, segment)));
  int32_t* counts = q.N > kLiveAlone ? map + q.N + 1 : nullptr;
  if (counts) {
    const int st = launch_plain("xent_count_kernel", xent_count_kernel, blocks, kLiveThreads, s, q.y, q.N, segment,
                                counts);
    if (st != FK_OK) return st;
  }
  const int64_t eb = dtype_bytes(q.dtype);
  const bool vec = reinterpret_cast<uintptr_t>(gx) % 16 == 0 && gx_row * eb % 16 == 0 && q.D * eb % 16 == 0;
  return launch_plain("xent_live_kernel", xent_live_kernel, blocks, kLiveThreads, s, q.y, q.N, segment, counts, map,
                      map + q.N, loss, stat, gx, gx_row * eb, q.D * eb, vec ? 1 : 0);
}

// Copies of the operands made by the caller of a pass; see fk_xent_loss_grad.
struct Copies {
  uint16_t *x_forward, *x_backward, *c;   // null: used in place (x_forward, c)
  int32_t* map;                           // gathered rows, which the copies of x hold then; or null
};

struct ForwardPlan {
  ShapeChoice sh;
  int chunks;
  int64_t row_blocks;
  uint16_t *xc, *cc;
  int32_t* map;
  float2* partial;
  double2* block_part;
  uint32_t* ticket;
  size_t bytes;
};

static ForwardPlan plan_forward(const Xent& q, void* ws, const Copies* given = nullptr) {
  ForwardPlan f;
  Bump b{static_cast<uint8_t*>(ws)};
  f.sh = choose_shape(q.N, q.K, q.B, q.parts() > 1);
  f.chunks = choose_chunks(q.B * ceil_div(q.N, f.sh.bm()), ceil_div(q.K, f.sh.bn), slots_of(f.sh),
                           2 * slots_of(f.sh), 0.25);
  f.row_blocks = ceil_div(q.N, 32);
  const bool gather = given ? given->map != nullptr : gathers_forward(q);
  f.map = given ? given->map : gather ? b.take<int32_t>(map_words(q)) : nullptr;
  if (given) {
    f.xc = given->x_forward;
    f.cc = given->c;
  } else {
    f.xc = !gather && in_place(q.x, q.dtype, q.B, q.N, q.D, q.xs)
               ? nullptr
               : b.take<uint16_t>(q.parts() * q.B * q.N * q.Dp());
    f.cc = in_place(q.c, q.dtype, q.Bc(), q.K, q.D, q.cs)
               ? nullptr
               : b.take<uint16_t>(q.parts() * q.Bc() * q.K * q.Dp());
  }
  f.partial = b.take<float2>(q.B * f.chunks * parts_of(kEpiLse, f.sh.bn) * q.N);
  f.block_part = b.take<double2>(q.B * f.row_blocks);
  f.ticket = b.take<uint32_t>(1);
  f.bytes = b.used;
  return f;
}

static int forward(const Xent& q, float* loss, RowStat* stat, int32_t* count, void* ws, size_t ws_bytes,
                   int* status, cudaStream_t s, const Copies* given = nullptr) {
  const ForwardPlan f = plan_forward(q, ws, given);
  if (const int bad = check_workspace(ws, ws_bytes, f.bytes, "fk_xent_forward")) return bad;
  int st = FK_OK;
  const int32_t* live = f.map ? f.map + q.N : nullptr;
  if (!given) {
    if (f.map) st = find_live(q, f.map, q.reduction == 0 ? loss : nullptr, stat, nullptr, 0, s);
    RowsJob xj = rows_job(q.x, q.dtype, q.B, q.N, q.D, q.xs, f.xc, q.Dp(), nullptr);
    xj.map = f.map;
    xj.live = live;
    if (st == FK_OK)
      st = rows_copy(q.dtype, xj, rows_job(q.c, q.dtype, q.Bc(), q.K, q.D, q.cs, f.cc, q.Dp(), nullptr), s);
  }
  if (st != FK_OK) return st;
  Params<1> prm = {};
  prm.count = 1;
  Problem& p = prm.p[0];
  p.M = static_cast<int>(q.N);
  p.N = static_cast<int>(q.K);
  p.batches = static_cast<int>(q.B);
  p.chunks = f.chunks;
  p.scale2 = q.scale * 1.44269504f;
  p.labels = q.y.p;
  p.label_dtype = q.y.dtype;
  p.label_sb = q.y.sb;
  p.label_sn = q.y.sn;
  p.ignore_index = q.y.ignore;
  p.live = live;
  p.live_cap = p.M;
  p.row_map = f.map;
  p.partial = f.partial;
  p.zero = f.ticket;
  p.zero_n = 1;
  p.status = status;
  st = set_problem<kEpiLse>(prm, 0, operand(q, q.x, f.xc, q.B, q.N, q.xs, false, 0),
                            operand(q, q.c, f.cc, q.Bc(), q.K, q.cs, false, 0), q.D, f.sh);
  if (st == FK_OK) st = launch<kEpiLse>(prm, f.sh, s);
  if (st != FK_OK) return st;
  CombineParams cp = {};
  cp.partial = f.partial;
  cp.x = q.x;
  cp.c = q.c;
  cp.dtype = q.dtype;
  for (int i = 0; i < 3; ++i) {
    cp.xs[i] = q.xs[i];
    cp.cs[i] = q.cs[i];
  }
  cp.D = static_cast<int>(q.D);
  cp.scale = q.scale;
  cp.scale2 = q.scale * 1.44269504f;
  const int64_t eb = dtype_bytes(q.dtype);
  auto aligned = [&](const void* t, int64_t B, int64_t M, const int64_t* st) {
    return (st[2] == 1 || q.D == 1) && reinterpret_cast<uintptr_t>(t) % 16 == 0 &&
           (M == 1 || st[1] * eb % 16 == 0) && (B == 1 || st[0] * eb % 16 == 0);
  };
  cp.vec = aligned(q.x, q.B, q.N, q.xs) && aligned(q.c, q.B, q.K, q.cs);
  cp.labels = q.y.p;
  cp.label_dtype = q.y.dtype;
  cp.lb = q.y.sb;
  cp.ln = q.y.sn;
  cp.ignore = q.y.ignore;
  cp.K = q.K;
  cp.N = static_cast<int>(q.N);
  cp.pieces = f.chunks * parts_of(kEpiLse, f.sh.bn);
  cp.row_blocks = static_cast<int>(f.row_blocks);
  cp.reduction = q.reduction;
  cp.loss = loss;
  cp.stat = stat;
  cp.count = count;
  cp.block_part = f.block_part;
  cp.ticket = f.ticket;
  cp.map = f.map;
  cp.live = live;
  if (given && !given->x_forward) {
    cp.copy = given->x_backward;
    cp.Dp = static_cast<int>(q.Dp());
  }
  cp.status = status;
  return launch_plain("xent_combine_kernel", xent_combine_kernel,
                      dim3(static_cast<unsigned>(q.B * f.row_blocks)), kCombineWarps * 32, s, cp);
}

struct BackwardPlan {
  int64_t R, Kp;               // rows and centroids of a piece
  int64_t n_chunks, n_pieces;
  ShapeChoice sh_p, sh;          // of P, of the two gradient products
  int split_x, split_c;
  int64_t ld;                  // of the float32 accumulators
  uint16_t *xc, *cc, *P;
  float *acc_x, *acc_c;        // null: the product writes the output itself
  uint32_t *join_x, *join_c;   // arrival counters of split products
  int64_t joins;               // of both, from join_x on
  RowStat* weighted;
  int32_t* map;                // gathered rows, their number behind it
  float* power;                // float16 row losses: each row's power of two,
  uint32_t* reach;             // the largest with x's and the factor that it gives,
  uint16_t* xs;                // and the copy of x that holds it
  size_t bytes;
};

// Tile shape and splits of the two gradient products: dx is Mx x D over steps_x
// steps, dc Mc x D over steps_c (0: not wanted).  A product with few tiles and a
// long contraction is split along it; each split costs a write and a read of
// float32 partial sums, counted in steps of a tile's contraction.
static void plan_products(const Xent& q, int64_t Mx, int64_t steps_x, int64_t Mc, int64_t steps_c,
                          BackwardPlan* f) {
  const bool exact = q.parts() > 1;
  const int wide = exact || q.D <= 128 ? 128 : 256;
  auto tiles = [&](int64_t M, int64_t steps, int64_t bm, int64_t bn) {
    return steps ? q.B * ceil_div(M, bm) * ceil_div(q.D, bn) : 0;
  };
  // work in shares of a megabyte of operands, the least that is worth a worker
  const int64_t share = exact ? 3 : 8;
  auto shares = [&](int64_t bm, int64_t bn) {
    return tiles(Mx, steps_x, bm, bn) * std::max<int64_t>(1, steps_x / share) +
           tiles(Mc, steps_c, bm, bn) * std::max<int64_t>(1, steps_c / share);
  };
  if (std::max(Mx, Mc) > 128 && shares(256, wide) >= 74) f->sh = {2, wide, exact};
  else if (!exact && q.D > 64 && shares(128, 128) >= 100) f->sh = {1, 128, exact};
  else f->sh = {1, 64, exact};
  f->split_x = f->split_c = 1;
  const int64_t slots = slots_of(f->sh);
  const int64_t tx = tiles(Mx, steps_x, f->sh.bm(), f->sh.bn), tc = tiles(Mc, steps_c, f->sh.bm(), f->sh.bn);
  if (tx + tc >= 8 * slots) return;
  static const int tries[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32};
  const double us = f->sh.step_us();
  double best = 1e300;
  for (int sx : tries) {
    if (sx > 1 && (sx > steps_x || tx * sx > 4 * slots)) break;
    for (int sc : tries) {
      if (sc > 1 && (sc > steps_c || tc * sc > 4 * slots)) break;
      const double cx = tile_cost(ceil_div(steps_x, sx)), cc = tile_cost(ceil_div(steps_c, sc));
      const int64_t n = tx * sx + tc * sc, workers = std::min(n, slots);
      const double span = cx >= cc ? fill(tx * sx, cx, tc * sc, cc, workers).span
                                   : fill(tc * sc, cc, tx * sx, cx, workers).span;
      const double bytes = (sx > 1 ? 4.0 * q.B * Mx * q.D * (2 * sx) : 0.0) + (sc > 1 ? 4.0 * q.B * Mc * q.D * (2 * sc) : 0.0);
      // the last split's warp reads the others' sums one after another
      const double chain = 0.7 * (sx > 1 || sc > 1 ? std::max(sx, sc) : 0) * (f->sh.bn == 256 ? 2 : 1);
      const double join = (chain + bytes / 4e6) / us;
      if (span + join < best * 0.999) {
        best = span + join;
        f->split_x = sx;
        f->split_c = sc;
      }
    }
  }
}

static BackwardPlan plan_backward(const Xent& q, bool want_x, bool want_c, void* ws,
                                  const Copies* given = nullptr) {
  BackwardPlan f;
  Bump b{static_cast<uint8_t*>(ws)};
  const int64_t budget = std::max<int64_t>(kPieceElems / q.parts() / q.B, 256 * 128);
  const int64_t kall = ceil_div(q.K, 256) * 256;
  f.R = std::min(q.N, kMaxRowChunk);
  f.Kp = std::min(kall, std::max<int64_t>(256, budget / std::max<int64_t>(f.R, 128) / 256 * 256));
  f.R = std::min(q.N, std::max<int64_t>(128, budget / f.Kp / 128 * 128));
  f.n_pieces = ceil_div(q.K, f.Kp);
  f.Kp = ceil_div(ceil_div(q.K, f.n_pieces), 256) * 256;
  f.n_pieces = ceil_div(q.K, f.Kp);
  f.n_chunks = ceil_div(q.N, f.R);
  f.R = std::min(q.N, ceil_div(ceil_div(q.N, f.n_chunks), 128) * 128);
  f.n_chunks = ceil_div(q.N, f.R);
  const int64_t kw = std::min(f.Kp, q.K);
  f.sh_p = choose_shape(f.R, kw, q.B, q.parts() > 1);
  const int64_t steps_x = ceil_div(kw, 64), steps_c = ceil_div(f.R, 64);
  plan_products(q, f.R, want_x ? steps_x : 0, kw, want_c ? steps_c : 0, &f);
  f.ld = ceil_div(q.D, 4) * 4;
  if (given) {
    f.xc = given->x_backward;
    f.cc = given->c;
  } else {
    f.xc = b.take<uint16_t>(q.parts() * q.B * q.N * q.Dp());
    f.cc = in_place(q.c, q.dtype, q.Bc(), q.K, q.D, q.cs)
               ? nullptr
               : b.take<uint16_t>(q.parts() * q.Bc() * q.K * q.Dp());
  }
  f.map = given ? given->map : gathers(q) ? b.take<int32_t>(map_words(q)) : nullptr;
  f.P = b.take<uint16_t>(q.parts() * q.B * f.R * f.Kp);
  f.acc_x = f.acc_c = nullptr;
  if (want_x && (f.n_pieces > 1 || f.split_x > 1)) f.acc_x = b.take<float>(f.split_x * q.B * q.N * f.ld);
  if (want_c && (f.n_chunks > 1 || f.split_c > 1)) f.acc_c = b.take<float>(f.split_c * q.B * f.Kp * f.ld);
  // 32 warps a tile at most
  auto counters = [&](int64_t M, int splits) {
    return splits > 1 ? q.B * ceil_div(M, f.sh.bm()) * ceil_div(q.D, f.sh.bn) * 32 : 0;
  };
  const int64_t jx = want_x ? counters(f.R, f.split_x) : 0, jc = want_c ? counters(kw, f.split_c) : 0;
  f.joins = jx + jc;
  f.join_x = f.joins ? b.take<uint32_t>(f.joins) : nullptr;
  f.join_c = f.join_x ? f.join_x + jx : nullptr;
  f.weighted = q.reduction == 0 ? b.take<RowStat>(q.B * q.N) : nullptr;
  const bool weigh16 = q.reduction == 0 && q.dtype == FK_F16;
  f.power = weigh16 ? b.take<float>(q.B * q.N) : nullptr;
  f.reach = weigh16 ? b.take<uint32_t>(2) : nullptr;
  f.xs = weigh16 && want_c ? b.take<uint16_t>(q.B * q.N * q.Dp()) : nullptr;
  f.bytes = b.used;
  return f;
}

struct Grad {
  void* p;
  int64_t sb, sr;
};

// One gradient product over a piece, into the accumulator or the output.
static int grad_problem(const Xent& q, Params<2>& prm, uint32_t* join, const Problem& base, const Operand& a,
                        const Operand& b, int64_t M, int64_t kdim, ShapeChoice sh, int splits, float* acc,
                        int64_t acc_rows, int64_t acc_row0, int64_t ld, bool first, bool last, const Grad& g,
                        int64_t out_row0) {
  Problem& p = prm.p[prm.count];
  p = base;
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(q.D);
  const int64_t steps = ceil_div(kdim, 64);
  p.chunks = static_cast<int>(std::min<int64_t>(splits, steps));
  const int eb = dtype_bytes(q.dtype);
  // gathered rows go where the map says, counted from the first row
  p.out = static_cast<uint8_t*>(g.p) + (p.row_map ? 0 : out_row0 * g.sr * eb);
  p.out_dtype = q.dtype;
  p.out_sb = g.sb;
  p.out_sr = g.sr;
  p.out_vec = reinterpret_cast<uintptr_t>(p.out) % (4 * eb) == 0 && g.sr % 4 == 0 && g.sb % 4 == 0;
  if (acc) {
    p.acc = acc + acc_row0 * ld;
    p.acc_ld = ld;
    p.acc_batch = acc_rows * ld;
    p.acc_split = q.B * acc_rows * ld;
    p.acc_read = !first;
    p.acc_write = splits > 1 || !last;
  }
  if (splits > 1 && last) {
    // a short last piece may have fewer steps than splits: the others hold
    // earlier pieces' sums, or were never written if this is the only piece
    p.join = join;
    p.join_splits = first ? p.chunks : splits;
  }
  return set_problem<kEpiOut>(prm, prm.count++, a, b, kdim, sh);
}

static int backward(const Xent& q, const RowStat* stat, const int32_t* count, const float* g,
                    const Grad& gx, const Grad& gc, void* ws, size_t ws_bytes, int* status,
                    cudaStream_t s, const Copies* given = nullptr) {
  const BackwardPlan f = plan_backward(q, gx.p != nullptr, gc.p != nullptr, ws, given);
  if (const int bad = check_workspace(ws, ws_bytes, f.bytes, "fk_xent_backward")) return bad;
  const int64_t rows = q.B * q.N;
  const bool f16 = q.dtype == FK_F16;
  // float16 P is kept times 2^14: a softmax over 2^20 centroids then still has
  // ten bits above float16's smallest subnormal, and 2 * 2^14 is in range (see
  // xent_weight16_kernel)
  const float p_scale = f16 ? 16384.0f : 1.0f;
  int st = FK_OK;
  const int32_t* live = f.map ? f.map + q.N : nullptr;
  if (!given) {
    if (f.map) st = find_live(q, f.map, nullptr, nullptr, gx.p, gx.sr, s);
    RowsJob xj = rows_job(q.x, q.dtype, q.B, q.N, q.D, q.xs, f.xc, q.Dp(), f.map ? nullptr : &q.y);
    xj.map = f.map;
    xj.live = live;
    if (st == FK_OK)
      st = rows_copy(q.dtype, xj, rows_job(q.c, q.dtype, q.Bc(), q.K, q.D, q.cs, f.cc, q.Dp(), nullptr), s);
  }
  if (st != FK_OK) return st;
  const float* factor_c = nullptr;
  if (q.reduction == 0) {
    const int blocks = static_cast<int>(std::min<int64_t>(ceil_div(rows, 256), 1024));
    if (f.power) {
      const cudaError_t e = cudaMemsetAsync(f.reach, 0, 2 * sizeof(uint32_t), s);
      if (e != cudaSuccess) return fail(FK_ERR_CUDA, "cudaMemsetAsync: %s", cudaGetErrorString(e));
      const int many = static_cast<int>(std::min<int64_t>(ceil_div(rows, 8), 2048));
      const int Dp = static_cast<int>(q.Dp());
      st = launch_plain("xent_weight16_kernel", xent_weight16_kernel, dim3(many), 256, s, g, stat, rows, f.weighted,
                        f.power, f.xs ? f.xc : nullptr, Dp, f.map, live, f.reach);
      if (st == FK_OK && f.xs) {
        factor_c = reinterpret_cast<const float*>(f.reach + 1);
        const int wide = static_cast<int>(std::min<int64_t>(ceil_div(rows * (Dp / 8), 256), 2048));
        st = launch_plain("xent_scale16_kernel", xent_scale16_kernel, dim3(wide), 256, s, f.xc, rows, Dp, f.power,
                          f.map, live, f.reach, f.xs, reinterpret_cast<float*>(f.reach + 1));
      }
    } else {
      st = launch_plain("xent_weight_kernel", xent_weight_kernel, dim3(blocks), 256, s, g, stat, rows, f.weighted);
    }
    if (st != FK_OK) return st;
    stat = f.weighted;
  }

  for (int64_t piece = 0; piece < f.n_pieces; ++piece) {
    const int64_t k0 = piece * f.Kp, kw = std::min(f.Kp, q.K - k0);
    for (int64_t chunk = 0; chunk < f.n_chunks; ++chunk) {
      const int64_t r0 = chunk * f.R, rw = std::min(f.R, q.N - r0);
      // dz of the piece
      Params<1> prm = {};
      prm.count = 1;
      Problem& p = prm.p[0];
      p.M = static_cast<int>(rw);
      p.N = static_cast<int>(kw);
      p.batches = static_cast<int>(q.B);
      p.chunks = 1;
      p.status = status;
      p.live = live;
      p.live_off = static_cast<int>(r0);
      p.live_cap = static_cast<int>(rw);
      p.row_map = f.map;
      p.scale2 = q.scale * 1.44269504f;
      p.stat = stat;
      p.stat_rows = q.N;
      p.stat_off = r0;
      p.col_off = static_cast<int>(k0);
      p.p_scale = p_scale;
      p.p_out = f.P;
      p.p_ld = f.Kp;
      p.p_batch = f.R * f.Kp;
      p.p_part = q.B * f.R * f.Kp;
      p.p_bf16 = !f16;
      if (piece == 0 && chunk == 0) {
        p.zero = f.join_x;
        p.zero_n = static_cast<int>(f.joins);
      }
      st = set_problem<kEpiGrad>(prm, 0, operand(q, q.x, f.xc, q.B, q.N, q.xs, false, r0),
                                 operand(q, q.c, f.cc, q.Bc(), q.K, q.cs, false, k0), q.D, f.sh_p);
      if (st == FK_OK) st = launch<kEpiGrad>(prm, f.sh_p, s);
      if (st != FK_OK) return st;

      Operand po;  // P by rows (for dx); its valid width and height bound the products
      po.p = f.P;
      po.dtype = q.mma_dtype();
      po.inner = kw;
      po.rows = rw;
      po.ld = f.Kp;
      po.mat = f.R * f.Kp;
      po.mats = q.parts() * q.B;
      po.batch_step = 1;
      po.part_step = static_cast<int>(q.B);
      po.mn = false;
      po.off = 0;
      Problem base = {};
      base.batches = static_cast<int>(q.B);
      base.status = status;
      base.fscale = q.scale / p_scale;
      base.stat = stat;
      base.stat_rows = q.N;
      base.p_scale = p_scale;
      base.f_den = q.reduction == 1 ? count : nullptr;
      base.live = live;
      base.live_off = static_cast<int>(r0);
      base.live_cap = static_cast<int>(rw);
      Params<2> pair = {};
      auto add_x = [&]() {
        const Operand co = operand(q, q.c, f.cc, q.Bc(), q.K, q.cs, true, k0);
        base.live_steps = 0;
        base.row_map = f.map;
        base.f_num = q.reduction == 0 ? nullptr : g;
        base.row_factor = f.power;
        base.label_rows = nullptr;
        if (q.dtype != FK_F32 && piece == 0) {
          base.label_rows = static_cast<const uint16_t*>(co.p);
          base.label_ld = co.ld;
          base.label_batch = co.batch_step ? co.mat : 0;
        }
        return grad_problem(q, pair, f.join_x, base, po, co, rw, kw, f.sh, f.split_x, f.acc_x, q.N, r0, f.ld,
                            piece == 0, piece + 1 == f.n_pieces, gx, r0);
      };
      auto add_c = [&]() {
        Operand pt = po;
        pt.mn = true;
        const Operand xo = operand(q, q.x, f.xs ? f.xs : f.xc, q.B, q.N, q.xs, true, r0);
        base.live_steps = 1;
        base.row_map = nullptr;
        base.f_num = q.reduction == 0 ? factor_c : g;
        base.row_factor = nullptr;
        base.label_rows = nullptr;
        return grad_problem(q, pair, f.join_c, base, pt, xo, kw, rw, f.sh, f.split_c, f.acc_c, f.Kp, 0, f.ld,
                            chunk == 0, chunk + 1 == f.n_chunks, gc, k0);
      };
      // the product with the longer tiles first
      const bool x_first = ceil_div(kw, 64) / f.split_x >= ceil_div(rw, 64) / f.split_c;
      st = FK_OK;
      if (gx.p && x_first) st = add_x();
      if (st == FK_OK && gc.p) st = add_c();
      if (st == FK_OK && gx.p && !x_first) st = add_x();
      const bool own = f.power || (gx.p && q.dtype != FK_F32 && piece == 0);
      if (st == FK_OK) st = own ? launch<kEpiOutRows>(pair, f.sh, s) : launch<kEpiOut>(pair, f.sh, s);
      if (st != FK_OK) return st;
    }
  }
  return FK_OK;
}

// Loss and gradients in one call: the operands' copies serve both passes, and a
// 16-bit x that the forward pass reads in place is copied by its combine kernel.
struct LossGradPlan {
  Copies copies;
  RowStat* stat;
  int32_t* count;
  uint8_t* rest;               // scratch of the passes, one after the other
  size_t rest_bytes, bytes;
};

static LossGradPlan plan_loss_grad(const Xent& q, bool want_x, bool want_c, void* ws) {
  LossGradPlan f;
  Bump b{static_cast<uint8_t*>(ws)};
  f.copies.x_backward = b.take<uint16_t>(q.parts() * q.B * q.N * q.Dp());
  f.copies.map = gathers(q) ? b.take<int32_t>(map_words(q)) : nullptr;
  f.copies.c = in_place(q.c, q.dtype, q.Bc(), q.K, q.D, q.cs)
                   ? nullptr
                   : b.take<uint16_t>(q.parts() * q.Bc() * q.K * q.Dp());
  f.copies.x_forward =
      !gathers(q) && in_place(q.x, q.dtype, q.B, q.N, q.D, q.xs) ? nullptr : f.copies.x_backward;
  f.stat = b.take<RowStat>(q.B * q.N);
  f.count = b.take<int32_t>(1);
  f.rest = b.base ? b.base + b.used : nullptr;
  f.rest_bytes = std::max(plan_forward(q, nullptr, &f.copies).bytes,
                          plan_backward(q, want_x, want_c, nullptr, &f.copies).bytes);
  f.bytes = b.used + f.rest_bytes;
  return f;
}

static int loss_grad(const Xent& q, float* loss, const float* g, const Grad& gx, const Grad& gc, void* ws,
                     size_t ws_bytes, int* status, cudaStream_t s) {
  const LossGradPlan f = plan_loss_grad(q, gx.p != nullptr, gc.p != nullptr, ws);
  if (const int bad = check_workspace(ws, ws_bytes, f.bytes, "fk_xent_loss_grad")) return bad;
  int st = FK_OK;
  int32_t* map = f.copies.map;
  if (map) st = find_live(q, map, q.reduction == 0 ? loss : nullptr, f.stat, gx.p, gx.sr, s);
  RowsJob xj = rows_job(q.x, q.dtype, q.B, q.N, q.D, q.xs, f.copies.x_forward, q.Dp(), map ? nullptr : &q.y);
  xj.map = map;
  xj.live = map ? map + q.N : nullptr;
  if (st == FK_OK)
    st = rows_copy(q.dtype, xj,
                   rows_job(q.c, q.dtype, q.Bc(), q.K, q.D, q.cs, f.copies.c, q.Dp(), nullptr), s);
  if (st == FK_OK) st = forward(q, loss, f.stat, f.count, f.rest, f.rest_bytes, status, s, &f.copies);
  if (st == FK_OK)
    st = backward(q, f.stat, f.count, g, gx, gc, f.rest, f.rest_bytes, status, s, &f.copies);
  return st;
}

static int make(Xent& q, const void* x, const void* c, const void* labels, int dtype, int labels_dtype,
                int64_t B, int64_t N, int64_t K, int64_t D, const int64_t* xs, const int64_t* cs,
                const int64_t* ls, float scale, int64_t ignore_index, int reduction, const char* who) {
  q.x = x;
  q.c = c;
  q.dtype = dtype;
  q.B = B;
  q.N = N;
  q.K = K;
  q.D = D;
  q.y.p = labels;
  q.y.dtype = labels_dtype;
  q.y.ignore = ignore_index;
  q.scale = scale;
  q.reduction = reduction;
  if (!xs || !cs || !ls) return fail(FK_ERR_INVALID_ARG, "%s: null strides", who);
  for (int i = 0; i < 3; ++i) {
    q.xs[i] = xs[i];
    q.cs[i] = cs[i];
  }
  q.y.sb = ls[0];
  q.y.sn = ls[1];
  return check_args(q, who);
}

}  // namespace head
}  // namespace fk

using namespace fk;
using namespace fk::head;

static int check_grads(int64_t D, const void* gx, const void* gc, const int64_t* gxs, const int64_t* gcs,
                       const char* who) {
  if ((gx && !gxs) || (gc && !gcs)) return fail(FK_ERR_INVALID_ARG, "%s: null strides", who);
  if ((gx && D > 1 && gxs[2] != 1) || (gc && D > 1 && gcs[2] != 1))
    return fail(FK_ERR_UNSUPPORTED, "%s: gradient rows must have unit stride", who);
  return FK_OK;
}

static int no_rows_grad(int64_t B, int64_t K, int64_t D, int dtype, void* gc, const int64_t* gcs,
                        cudaStream_t s) {
  if (!gc) return FK_OK;
  const int64_t eb = dtype_bytes(dtype);
  for (int64_t b = 0; b < B; ++b) {
    const cudaError_t e = cudaMemset2DAsync(static_cast<uint8_t*>(gc) + b * gcs[0] * eb,
                                            static_cast<size_t>(std::max(gcs[1], D) * eb), 0,
                                            static_cast<size_t>(D * eb), static_cast<size_t>(K), s);
    if (e != cudaSuccess) return fail(FK_ERR_CUDA, "cudaMemset2DAsync: %s", cudaGetErrorString(e));
  }
  return FK_OK;
}

static int no_rows_loss(int reduction, float* loss, int32_t* count, cudaStream_t s) {
  // a sum of 0, a mean of 0 / 0 (all bits set is a NaN)
  cudaError_t e = count ? cudaMemsetAsync(count, 0, sizeof(int32_t), s) : cudaSuccess;
  if (e == cudaSuccess && reduction != 0) e = cudaMemsetAsync(loss, reduction == 1 ? 0xff : 0, sizeof(float), s);
  return e == cudaSuccess ? FK_OK : fail(FK_ERR_CUDA, "cudaMemsetAsync: %s", cudaGetErrorString(e));
}

extern "C" size_t fk_xent_workspace_size(const void* x, const void* centroids, int dtype, int64_t B,
                                         int64_t N, int64_t K, int64_t D, const int64_t* x_strides3,
                                         const int64_t* c_strides3, int reduction, int backward_x,
                                         int backward_c) {
  Xent q;
  const int64_t ls[2] = {0, 0};
  if (make(q, x, centroids, nullptr, dtype, FK_I32, B, N, K, D, x_strides3, c_strides3, ls, 1.0f, 0,
           reduction, "fk_xent_workspace_size") != FK_OK ||
      B == 0 || N == 0)
    return 0;
  return backward_x || backward_c ? plan_backward(q, backward_x != 0, backward_c != 0, nullptr).bytes
                                  : plan_forward(q, nullptr).bytes;
}

extern "C" int fk_xent_forward(const void* x, const void* centroids, const void* labels, int dtype,
                               int labels_dtype, int64_t B, int64_t N, int64_t K, int64_t D,
                               const int64_t* x_strides3, const int64_t* c_strides3,
                               const int64_t* l_strides2, float scale, int64_t ignore_index,
                               int reduction, float* loss, float* row_stats, int32_t* count,
                               void* workspace, size_t workspace_bytes, int32_t* dev_status,
                               void* stream) {
  Xent q;
  int st = make(q, x, centroids, labels, dtype, labels_dtype, B, N, K, D, x_strides3, c_strides3,
                l_strides2, scale, ignore_index, reduction, "fk_xent_forward");
  if (st != FK_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!count || (!loss && (B * N > 0 || reduction != 0)))
    return fail(FK_ERR_INVALID_ARG, "fk_xent_forward: null pointer");
  if (B == 0 || N == 0) return no_rows_loss(reduction, loss, count, s);
  if (!x || !centroids || !labels) return fail(FK_ERR_INVALID_ARG, "fk_xent_forward: null pointer");
  if (reinterpret_cast<uintptr_t>(row_stats) % 16)
    return fail(FK_ERR_INVALID_ARG, "fk_xent_forward: row_stats must be 16-byte aligned");
  return forward(q, loss, reinterpret_cast<RowStat*>(row_stats), count, workspace, workspace_bytes,
                 dev_status, s);
}

extern "C" size_t fk_xent_loss_grad_workspace_size(const void* x, const void* centroids, int dtype,
                                                   int64_t B, int64_t N, int64_t K, int64_t D,
                                                   const int64_t* x_strides3, const int64_t* c_strides3,
                                                   int reduction, int want_x, int want_c) {
  Xent q;
  const int64_t ls[2] = {0, 0};
  if (make(q, x, centroids, nullptr, dtype, FK_I32, B, N, K, D, x_strides3, c_strides3, ls, 1.0f, 0,
           reduction, "fk_xent_loss_grad_workspace_size") != FK_OK ||
      B == 0 || N == 0)
    return 0;
  return plan_loss_grad(q, want_x != 0, want_c != 0, nullptr).bytes;
}

extern "C" int fk_xent_loss_grad(const void* x, const void* centroids, const void* labels, int dtype,
                                 int labels_dtype, int64_t B, int64_t N, int64_t K, int64_t D,
                                 const int64_t* x_strides3, const int64_t* c_strides3,
                                 const int64_t* l_strides2, float scale, int64_t ignore_index,
                                 int reduction, float* loss, const float* grad_loss, void* grad_x,
                                 void* grad_centroids, const int64_t* gx_strides3,
                                 const int64_t* gc_strides3, void* workspace, size_t workspace_bytes,
                                 int32_t* dev_status, void* stream) {
  Xent q;
  int st = make(q, x, centroids, labels, dtype, labels_dtype, B, N, K, D, x_strides3, c_strides3,
                l_strides2, scale, ignore_index, reduction, "fk_xent_loss_grad");
  if (st != FK_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  st = check_grads(D, grad_x, grad_centroids, gx_strides3, gc_strides3, "fk_xent_loss_grad");
  if (st != FK_OK) return st;
  if (!loss && (B * N > 0 || reduction != 0))
    return fail(FK_ERR_INVALID_ARG, "fk_xent_loss_grad: null pointer");
  if (B == 0 || N == 0) {
    st = no_rows_loss(reduction, loss, nullptr, s);
    return st == FK_OK ? no_rows_grad(B, K, D, dtype, grad_centroids, gc_strides3, s) : st;
  }
  if (!x || !centroids || !labels || (!grad_x && !grad_centroids) || (reduction == 0 && !grad_loss))
    return fail(FK_ERR_INVALID_ARG, "fk_xent_loss_grad: null pointer");
  Grad gx{grad_x, grad_x ? gx_strides3[0] : 0, grad_x ? gx_strides3[1] : 0};
  Grad gc{grad_centroids, grad_centroids ? gc_strides3[0] : 0, grad_centroids ? gc_strides3[1] : 0};
  return loss_grad(q, loss, grad_loss, gx, gc, workspace, workspace_bytes, dev_status, s);
}

extern "C" int fk_xent_backward(const void* x, const void* centroids, const void* labels, int dtype,
                                int labels_dtype, int64_t B, int64_t N, int64_t K, int64_t D,
                                const int64_t* x_strides3, const int64_t* c_strides3,
                                const int64_t* l_strides2, float scale, int64_t ignore_index,
                                int reduction, const float* row_stats, const int32_t* count,
                                const float* grad_loss, void* grad_x, void* grad_centroids,
                                const int64_t* gx_strides3, const int64_t* gc_strides3,
                                void* workspace, size_t workspace_bytes, int32_t* dev_status,
                                void* stream) {
  Xent q;
  int st = make(q, x, centroids, labels, dtype, labels_dtype, B, N, K, D, x_strides3, c_strides3,
                l_strides2, scale, ignore_index, reduction, "fk_xent_backward");
  if (st != FK_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  st = check_grads(D, grad_x, grad_centroids, gx_strides3, gc_strides3, "fk_xent_backward");
  if (st != FK_OK || (!grad_x && !grad_centroids)) return st;
  if (B == 0 || N == 0) return no_rows_grad(B, K, D, dtype, grad_centroids, gc_strides3, s);
  if (!x || !centroids || !labels || !row_stats || !count || (reduction == 0 && !grad_loss))
    return fail(FK_ERR_INVALID_ARG, "fk_xent_backward: null pointer");
  if (reinterpret_cast<uintptr_t>(row_stats) % 16)
    return fail(FK_ERR_INVALID_ARG, "fk_xent_backward: row_stats must be 16-byte aligned");
  Grad gx{grad_x, grad_x ? gx_strides3[0] : 0, grad_x ? gx_strides3[1] : 0};
  Grad gc{grad_centroids, grad_centroids ? gc_strides3[0] : 0, grad_centroids ? gc_strides3[1] : 0};
  return backward(q, reinterpret_cast<const RowStat*>(row_stats), count, grad_loss, gx, gc, workspace,
                  workspace_bytes, dev_status, s);
}
