// Scores of points against centroids from 8-bit integers, one scale for each
// point and each centroid:
//
//   z[n, k] = ((sum_d x[n, d] c[k, d]) * sx[n]) * sc[k] (+ bias[k])
//
// The integer sum is exact (tcgen05 kind::i8, int32 accumulators); the scaling
// is two float32 products and a sum in this order, each rounded, so scores and
// argmax agree to the bit with the formula.  fk_int8_scores stores z rounded
// once to its output type; fk_int8_assign keeps only each row's argmax.
//
// A 256 x 256 tile needs the same bytes per step as with 16-bit operands in half
// the time, so long products are bound by the L2: 4096 x 8192 x 4096 takes 95 us
// (2.9 POP/s, 11 TB/s from the L2).  One token against 32768 x 4096 streams the
// codebook at 4.8 TB/s (28 us); 604800 points against 1000 centroids of 128
// features are bound by the argmax's scaling (255 us, see argmax_epilogue).
#include <algorithm>
#include <type_traits>

#include "fk_head_launch.cuh"

namespace fk {
namespace head {

// A row is quantised to zeros with scale 0 when its largest magnitude is below
// this: 127 / most would leave float32.
constexpr float kTiny = 1e-36f;
constexpr int64_t kMaxD8 = 65536;   // 127^2 * D stays below 2^30

// -------------------------------------------------------------- quantisation
// One group of threads per row: the largest magnitude, then
// round-to-nearest-even of x * (127 / most) and the scale most / 127.  Rows of up
// to eight 16-byte loads a thread stay in registers between the two.
// Magnitudes compare as their bits do, NaN and infinity above the rest, so the
// largest one is taken on the bits, two 16-bit values at a time; rounding adds
// 1.5 * 2^23, whose mantissa then ends in the integer's low byte.  (With a
// conversion each way the kernel was bound by the instructions: 60 us for
// 65537 x 1024 bfloat16, which 31 us would read and write.)
template <typename T>
__device__ __forceinline__ uint32_t most_bits(uint4 u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    else m = max(m, w[i] & 0x7fffffffu);
  }
  return m;
}
template <typename T>
__device__ __forceinline__ uint32_t join_bits(uint32_t a, uint32_t b) {
  if constexpr (sizeof(T) == 2) return __vmaxu2(a, b);
  else return max(a, b);
}
// the two halves of a 16-bit pair, as float32 bits
template <typename T>
__device__ __forceinline__ uint32_t float_bits(uint32_t m) {
  if constexpr (sizeof(T) == 4) return m;
  const uint32_t h = max(m & 0xffffu, m >> 16);
  if constexpr (std::is_same_v<T, __nv_bfloat16>) return h << 16;
  else return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(h))));
}
template <typename T>
__device__ __forceinline__ void floats_of(uint4 u, float (&f)[16 / sizeof(T)]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
}

// STEPS: 16-byte loads of a thread that hold its whole share of the row in
// registers, all in flight at once; 0 for longer rows, which are read twice.
template <typename T, int STEPS>
__global__ void __launch_bounds__(256) quantize_rows_kernel(
    const T* x, int64_t sb, int64_t sn, int64_t sd, int vec, int8_t* q, int64_t qb, int64_t qn, int Dq,
    int qvec, float* scale, int64_t scb, int64_t scn, int N,
    int D, int64_t rows, int lanes) {
  // `lanes` threads per row: a power of two up to a block
  __shared__ uint32_t sm[8];
  pdl_wait_then_release();
  constexpr int E = 16 / sizeof(T);
  constexpr int kHeld = STEPS > 0 ? STEPS : 1;
  const int sub = threadIdx.x & (lanes - 1);
  const int64_t row = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / lanes;
  const bool ok = row < rows;
  const int64_t b = ok ? row / N : 0, n = ok ? row - b * N : 0;
  const T* src = x + b * sb + n * sn;
  auto load = [&](int d) -> uint4 {
    uint4 u = make_uint4(0, 0, 0, 0);
    if (vec && d + E <= D) {
      u = *reinterpret_cast<const uint4*>(src + d);
    } else {
      T* v = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (d + i < D) v[i] = src[(d + i) * sd];
    }
    return u;
  };
  uint32_t most = 0;
  uint4 held[kHeld];
  if constexpr (STEPS > 0) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) held[s] = ok ? load((s * lanes + sub) * E) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) most = join_bits<T>(most, most_bits<T>(held[s]));
  } else if (ok) {
    for (int d = sub * E; d < D; d += lanes * E) most = join_bits<T>(most, most_bits<T>(load(d)));
  }
  most = float_bits<T>(most);
  for (int o = min(lanes, 32) >> 1; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  if (lanes > 32) {
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = most;
    __syncthreads();
    const int w0 = (threadIdx.x & ~(lanes - 1)) >> 5;
    for (int w = 0; w < lanes / 32; ++w) most = max(most, sm[w0 + w]);
  }
  if (!ok) return;
  const float m = __uint_as_float(most);
  // NaN and infinity sort above every finite magnitude: such a row has no
  // scale, and NaN in its place makes every score of it NaN
  const bool bad = most >= 0x7f800000u, zero = !bad && m < kTiny;
  const float inv = bad || zero ? 0.0f : __fdiv_rn(127.0f, m);
  if (sub == 0) scale[b * scb + n * scn] = bad ? __uint_as_float(0x7fc00000u) : zero ? 0.0f : __fdiv_rn(m, 127.0f);
  int8_t* dst = q + b * qb + n * qn;
  auto store = [&](int d, uint4 u) {
    if (d >= Dq) return;
    float f[E];
    floats_of<T>(u, f);
    uint32_t w[E / 4];
#pragma unroll
    for (int j = 0; j < E / 4; ++j) {
      uint32_t r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)   // |x * inv| is at most 127 and a rounding
        r[i] = __float_as_uint(__fadd_rn(__fmul_rn(f[j * 4 + i], inv), 12582912.0f));
      w[j] = __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
      if (bad) w[j] = 0;
    }
    if (qvec && d + E <= Dq) {
      if constexpr (E == 8) *reinterpret_cast<uint2*>(dst + d) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(dst + d) = w[0];
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (d + i < Dq) dst[d + i] = static_cast<int8_t>(w[i / 4] >> (8 * (i % 4)));
    }
  };
  if constexpr (STEPS > 0) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) store((s * lanes + sub) * E, held[s]);
  } else {
    for (int d = sub * E; d < Dq; d += lanes * E) store(d, load(d));
  }
}

// q's first Dq elements of a row are written (zeros from D on).
template <typename T>
static int quantize_typed(const void* x, int64_t B, int64_t N, int64_t D, const int64_t* xs, int8_t* q,
                          int64_t qb, int64_t qn, int64_t Dq, float* scale, int64_t scb, int64_t scn,
                          cudaStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const int vec = (xs[2] == 1 || D == 1) && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                  (N == 1 || xs[1] * sizeof(T) % 16 == 0) && (B == 1 || xs[0] * sizeof(T) % 16 == 0);
  const int qvec = reinterpret_cast<uintptr_t>(q) % E == 0 && (N == 1 || qn % E == 0) && (B == 1 || qb % E == 0);
  // a warp's lanes first, then up to eight loads each, then more warps; few
  // long rows (a token's call) take whole blocks at once
  const int64_t rows = B * N;
  int lanes = 1;
  while (lanes < 32 && static_cast<int64_t>(lanes) * E < Dq) lanes *= 2;
  const int held = rows < 1024 ? 2 : 8;
  while (lanes < 256 && static_cast<int64_t>(lanes) * E * held < Dq) lanes *= 2;
  const int64_t steps = ceil_div(Dq, static_cast<int64_t>(lanes) * E);
  const int64_t blocks = ceil_div(rows * lanes, 256);
  if (blocks >= (1ll << 31)) return fail(FK_ERR_UNSUPPORTED, "fk_quantize_rows: too many rows");
  auto kern = steps <= 1   ? quantize_rows_kernel<T, 1>
              : steps <= 2 ? quantize_rows_kernel<T, 2>
              : steps <= 4 ? quantize_rows_kernel<T, 4>
              : steps <= 8 ? quantize_rows_kernel<T, 8>
                           : quantize_rows_kernel<T, 0>;
  return launch_plain("quantize_rows_kernel", kern, dim3(static_cast<unsigned>(blocks)), 256, s,
                      static_cast<const T*>(x), xs[0], xs[1], xs[2], vec, q, qb, qn, static_cast<int>(Dq), qvec,
                      scale, scb, scn, static_cast<int>(N), static_cast<int>(D), rows, lanes);
}

static int quantize(const void* x, int dtype, int64_t B, int64_t N, int64_t D, const int64_t* xs,
                    int8_t* q, int64_t qb, int64_t qn, int64_t Dp, float* scale, int64_t scb, int64_t scn,
                    cudaStream_t s) {
  switch (dtype) {
    case FK_F16: return quantize_typed<__half>(x, B, N, D, xs, q, qb, qn, Dp, scale, scb, scn, s);
    case FK_BF16: return quantize_typed<__nv_bfloat16>(x, B, N, D, xs, q, qb, qn, Dp, scale, scb, scn, s);
    default: return quantize_typed<float>(x, B, N, D, xs, q, qb, qn, Dp, scale, scb, scn, s);
  }
}

// 8-bit rows that are not 16-byte addressable, copied to padded ones; x's and
// the centroids' in one launch.
struct Pack8 {
  const int8_t* x;
  int64_t sb, sn, sd;
  int8_t* out;
  int N, D, Dp;
  int64_t units;     // of 16 bytes; 0 for none
};
struct Pack8Jobs {
  Pack8 job[2];
};

__global__ void pack8_kernel(const Pack8Jobs jobs) {
  pdl_wait_then_release();
  const Pack8& j = jobs.job[blockIdx.y];
  const int per = j.Dp / 16;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; u < j.units;
       u += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t row = u / per;
    const int d0 = static_cast<int>(u - row * per) * 16;
    const int64_t b = row / j.N, n = row - b * j.N;
    const int8_t* src = j.x + b * j.sb + n * j.sn;
    int8_t v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = d0 + i < j.D ? src[(d0 + i) * j.sd] : 0;
    *reinterpret_cast<uint4*>(j.out + row * j.Dp + d0) = *reinterpret_cast<const uint4*>(v);
  }
}

static Pack8 pack8_job(const void* x, int64_t B, int64_t N, int64_t D, const int64_t* xs, int8_t* out,
                       int64_t Dp) {
  Pack8 j = {};
  if (out)
    j = {static_cast<const int8_t*>(x), xs[0], xs[1], xs[2], out, static_cast<int>(N), static_cast<int>(D),
         static_cast<int>(Dp), B * N * (Dp / 16)};
  return j;
}

static int pack8(const Pack8& a, const Pack8& b, cudaStream_t s) {
  const Pack8Jobs jobs = {{a.units ? a : b, b}};
  const int n = (a.units ? 1 : 0) + (b.units ? 1 : 0);
  if (n == 0) return FK_OK;
  const int sms = sm_count_current();
  const int64_t blocks = std::min<int64_t>(ceil_div(std::max(a.units, b.units), 256), (sms > 0 ? sms : 148) * 16ll);
  return launch_plain("pack8_kernel", pack8_kernel, dim3(static_cast<unsigned>(blocks), n), 256, s, jobs);
}

// Joins the column chunks of a row's argmax.
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(kJoinWarps * 32) argmax_join_kernel(const float2* partial, int pieces, int N,
                                                                      int row_blocks, int32_t* out, int64_t ob, int64_t on) {
  __shared__ float2 sm[kJoinWarps][33];
  pdl_wait_then_release();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / row_blocks;
  const int row = (blockIdx.x % row_blocks) * 32 + lane;
  float m = -INFINITY;
  int i = INT_MAX;
  if (row < N) {
    for (int p = warp; p < pieces; p += kJoinWarps) {
      const float2 v = partial[(static_cast<int64_t>(b) * pieces + p) * N + row];
      if (argmax_better(v.x, __float_as_int(v.y), m, i)) {
        m = v.x;
        i = __float_as_int(v.y);
      }
    }
  }
  sm[warp][lane] = make_float2(m, __int_as_float(i));
  __syncthreads();
  if (warp || row >= N) return;
  for (int w = 1; w < kJoinWarps; ++w) {
    const float2 v = sm[w][lane];
    if (argmax_better(v.x, __float_as_int(v.y), m, i)) {
      m = v.x;
      i = __float_as_int(v.y);
    }
  }
  out[b * ob + row * on] = i;
}

struct Scores {
  const void *x, *c;
  int x_dtype;                 // FK_I8, or a float type quantised within the call
  int64_t B, N, K, D;
  int64_t xs[3], cs[3];
  int64_t Dp() const { return ceil_div(D, 16) * 16; }
  int64_t Bc() const { return cs[0] == 0 ? 1 : B; }
};

static bool in_place8(const void* p, int64_t B, int64_t M, int64_t D, const int64_t* st) {
  if (B > 1 && st[0] == 0) return false;
  if (reinterpret_cast<uintptr_t>(p) % 16 || (D > 1 && st[2] != 1)) return false;
  if (M > 1 && (st[1] % 16 || st[1] < D || st[1] >= (1ll << 40))) return false;
  return B == 1 || (st[0] % 16 == 0 && st[0] > 0 && st[0] < (1ll << 40));
}

static Operand operand8(const Scores& q, const void* p, const int8_t* copy, int64_t B, int64_t M,
                        const int64_t* st) {
  Operand o;
  o.dtype = FK_I8;
  o.inner = q.D;
  o.rows = M;
  o.mn = false;
  o.off = 0;
  o.p = copy ? copy : p;
  o.ld = copy || M == 1 ? q.Dp() : st[1];
  o.mat = copy ? M * q.Dp() : st[0];
  o.mats = B;
  o.batch_step = B > 1 ? 1 : 0;
  o.part_step = 0;
  return o;
}

struct ScoresPlan {
  ShapeChoice sh;
  int chunks;
  int8_t *xq, *cq;
  float* sx;
  float2* partial;
  size_t bytes;
};

static ScoresPlan plan_scores(const Scores& q, bool argmax, void* ws) {
  ScoresPlan f = {};
  size_t used = 0;
  auto take = [&](int64_t bytes) -> void* {
    void* p = ws ? static_cast<uint8_t*>(ws) + used : nullptr;
    used += align_up(static_cast<size_t>(bytes), 256);
    return p;
  };
  f.sh = choose_shape(q.N, q.K, q.B, false);
  f.chunks = argmax ? choose_chunks(q.B * ceil_div(q.N, f.sh.bm()), ceil_div(q.K, f.sh.bn), slots_of(f.sh),
                                    2 * slots_of(f.sh), 0.25)
                    : 1;
  if (q.x_dtype != FK_I8 || !in_place8(q.x, q.B, q.N, q.D, q.xs))
    f.xq = static_cast<int8_t*>(take(q.B * q.N * q.Dp()));
  if (q.x_dtype != FK_I8) f.sx = static_cast<float*>(take(q.B * q.N * 4));
  if (!in_place8(q.c, q.Bc(), q.K, q.D, q.cs)) f.cq = static_cast<int8_t*>(take(q.Bc() * q.K * q.Dp()));
  if (f.chunks > 1) f.partial = static_cast<float2*>(take(q.B * f.chunks * parts_of(kEpiArgmax, f.sh.bn) * q.N * 8));
  f.bytes = used;
  return f;
}

static int make8(Scores& q, const void* x, const void* c, int x_dtype, int64_t B, int64_t N, int64_t K,
                 int64_t D, const int64_t* xs, const int64_t* cs, const char* who) {
  if (B < 0 || N < 0 || K <= 0 || D <= 0) return fail(FK_ERR_INVALID_ARG, "%s: bad sizes", who);
  if (x_dtype != FK_I8 && x_dtype != FK_F16 && x_dtype != FK_BF16 && x_dtype != FK_F32)
    return fail(FK_ERR_INVALID_ARG, "%s: unsupported dtype %d", who, x_dtype);
  if (!xs || !cs) return fail(FK_ERR_INVALID_ARG, "%s: null strides", who);
  if (D > kMaxD8)
    return fail(FK_ERR_UNSUPPORTED, "%s: D above %lld could overflow the int32 sums", who,
                static_cast<long long>(kMaxD8));
  if (N >= (1ll << 30) || K >= (1ll << 30) || B >= (1ll << 30) || B * N >= (1ll << 31))
    return fail(FK_ERR_UNSUPPORTED, "%s: sizes exceed 32-bit", who);
  // (expanded centroids can have any size: no workspace may wrap around)
  if (static_cast<double>(B) * static_cast<double>(K) * static_cast<double>(D) >= 0x1p58)
    return fail(FK_ERR_UNSUPPORTED, "%s: sizes exceed 64-bit", who);
  q.x = x;
  q.c = c;
  q.x_dtype = x_dtype;
  q.B = B;
  q.N = N;
  q.K = K;
  q.D = D;
  for (int i = 0; i < 3; ++i) {
    q.xs[i] = xs[i];
    q.cs[i] = cs[i];
  }
  return FK_OK;
}

struct Scales {
  const float *x, *c, *bias;
  const int64_t *xs, *cs, *bs;
};

template <int EPI>
static int run8(const Scores& q, const Scales& sc, Problem base, void* ws, size_t ws_bytes,
                int32_t* label_out, const int64_t* ls, int* status, cudaStream_t s, const char* who) {
  const bool argmax = EPI == kEpiArgmax;
  const ScoresPlan f = plan_scores(q, argmax, ws);
  if (f.bytes && (!ws || ws_bytes < f.bytes || reinterpret_cast<uintptr_t>(ws) % 256))
    return fail(FK_ERR_WORKSPACE, "%s: workspace of %zu bytes (256-byte aligned) needed, %zu given", who,
                f.bytes, ws_bytes);
  int st = FK_OK;
  if (q.x_dtype != FK_I8)
    st = quantize(q.x, q.x_dtype, q.B, q.N, q.D, q.xs, f.xq, q.N * q.Dp(), q.Dp(), q.Dp(), f.sx, q.N, 1, s);
  if (st == FK_OK)
    st = pack8(pack8_job(q.x, q.B, q.N, q.D, q.xs, q.x_dtype == FK_I8 ? f.xq : nullptr, q.Dp()),
               pack8_job(q.c, q.Bc(), q.K, q.D, q.cs, f.cq, q.Dp()), s);
  if (st != FK_OK) return st;
  Params<1> prm = {};
  prm.count = 1;
  Problem& p = prm.p[0];
  p = base;
  p.M = static_cast<int>(q.N);
  p.N = static_cast<int>(q.K);
  p.batches = static_cast<int>(q.B);
  p.chunks = f.chunks;
  p.a_scale = f.sx ? f.sx : sc.x;
  p.as_sb = f.sx ? q.N : sc.xs[0];
  p.as_sn = f.sx ? 1 : sc.xs[1];
  p.b_scale = sc.c;
  p.bs_sb = sc.cs[0];
  p.bs_sn = sc.cs[1];
  p.bias = sc.bias;
  p.bias_sb = sc.bias ? sc.bs[0] : 0;
  p.bias_sn = sc.bias ? sc.bs[1] : 0;
  p.unit = 1.0f;
  p.partial = f.partial;
  p.label_out = label_out;
  p.lo_sb = ls ? ls[0] : 0;
  p.lo_sn = ls ? ls[1] : 0;
  p.status = status;
  st = set_problem<EPI>(prm, 0, operand8(q, q.x, f.xq, q.B, q.N, q.xs),
                        operand8(q, q.c, f.cq, q.Bc(), q.K, q.cs), q.D, f.sh);
  if (st == FK_OK) st = launch<EPI>(prm, f.sh, s);
  if (st != FK_OK || !f.partial) return st;
  const int64_t row_blocks = ceil_div(q.N, 32);
  return launch_plain("argmax_join_kernel", argmax_join_kernel, dim3(static_cast<unsigned>(q.B * row_blocks)),
                      kJoinWarps * 32, s, f.partial, f.chunks * parts_of(kEpiArgmax, f.sh.bn), static_cast<int>(q.N),
                      static_cast<int>(row_blocks), label_out, ls[0], ls[1]);
}

}  // namespace head
}  // namespace fk

using namespace fk;
using namespace fk::head;

extern "C" int fk_quantize_rows(const void* x, int dtype, int64_t B, int64_t N, int64_t D,
                                const int64_t* x_strides3, int8_t* q, const int64_t* q_strides3,
                                float* scale, const int64_t* scale_strides2, void* stream) {
  if (B < 0 || N < 0 || D <= 0) return fail(FK_ERR_INVALID_ARG, "fk_quantize_rows: bad sizes");
  if (dtype != FK_F16 && dtype != FK_BF16 && dtype != FK_F32)
    return fail(FK_ERR_INVALID_ARG, "fk_quantize_rows: unsupported dtype %d", dtype);
  if (B == 0 || N == 0) return FK_OK;
  if (!x || !q || !scale || !x_strides3 || !q_strides3 || !scale_strides2)
    return fail(FK_ERR_INVALID_ARG, "fk_quantize_rows: null pointer");
  if (D > 1 && q_strides3[2] != 1)
    return fail(FK_ERR_UNSUPPORTED, "fk_quantize_rows: rows of q must have unit stride");
  if (N >= (1ll << 31) || D >= (1ll << 30)) return fail(FK_ERR_UNSUPPORTED, "fk_quantize_rows: sizes exceed 32-bit");
  return quantize(x, dtype, B, N, D, x_strides3, q, q_strides3[0], q_strides3[1], D, scale,
                  scale_strides2[0], scale_strides2[1], static_cast<cudaStream_t>(stream));
}

extern "C" size_t fk_int8_workspace_size(const void* x, const int8_t* centroids, int x_dtype, int64_t B,
                                         int64_t N, int64_t K, int64_t D, const int64_t* x_strides3,
                                         const int64_t* c_strides3, int argmax) {
  Scores q;
  if (make8(q, x, centroids, x_dtype, B, N, K, D, x_strides3, c_strides3, "fk_int8_workspace_size") != FK_OK ||
      B == 0 || N == 0)
    return 0;
  return plan_scores(q, argmax != 0, nullptr).bytes;
}

static int check8(const void* x, const void* c, int x_dtype, const Scales& sc, const char* who) {
  if (!x || !c || !sc.c || !sc.cs) return fail(FK_ERR_INVALID_ARG, "%s: null pointer", who);
  if (x_dtype == FK_I8 && (!sc.x || !sc.xs))
    return fail(FK_ERR_INVALID_ARG, "%s: 8-bit x needs its scales", who);
  if (x_dtype != FK_I8 && sc.x)
    return fail(FK_ERR_INVALID_ARG, "%s: x_scale goes with 8-bit x only", who);
  if (sc.bias && !sc.bs) return fail(FK_ERR_INVALID_ARG, "%s: null strides", who);
  return FK_OK;
}

extern "C" int fk_int8_scores(const void* x, const int8_t* centroids, const float* x_scale,
                              const float* c_scale, const float* bias, void* out, int x_dtype,
                              int out_dtype, int64_t B, int64_t N, int64_t K, int64_t D,
                              const int64_t* x_strides3, const int64_t* c_strides3,
                              const int64_t* xs_strides2, const int64_t* cs_strides2,
                              const int64_t* bias_strides2, const int64_t* out_strides3,
                              void* workspace, size_t workspace_bytes, int32_t* dev_status,
                              void* stream) {
  Scores q;
  int st = make8(q, x, centroids, x_dtype, B, N, K, D, x_strides3, c_strides3, "fk_int8_scores");
  if (st != FK_OK) return st;
  if (out_dtype != FK_F16 && out_dtype != FK_BF16 && out_dtype != FK_F32)
    return fail(FK_ERR_INVALID_ARG, "fk_int8_scores: unsupported output dtype %d", out_dtype);
  if (B == 0 || N == 0) return FK_OK;
  const Scales sc{x_scale, c_scale, bias, xs_strides2, cs_strides2, bias_strides2};
  if ((st = check8(x, centroids, x_dtype, sc, "fk_int8_scores")) != FK_OK) return st;
  if (!out || !out_strides3) return fail(FK_ERR_INVALID_ARG, "fk_int8_scores: null pointer");
  if (K > 1 && out_strides3[2] != 1)
    return fail(FK_ERR_UNSUPPORTED, "fk_int8_scores: rows of out must have unit stride");
  const int eb = dtype_bytes(out_dtype);
  Problem base = {};
  base.out = out;
  base.out_dtype = out_dtype;
  base.out_sb = out_strides3[0];
  base.out_sr = out_strides3[1];
  base.out_vec = reinterpret_cast<uintptr_t>(out) % (4 * eb) == 0 && (N == 1 || out_strides3[1] % 4 == 0) &&
                 (B == 1 || out_strides3[0] % 4 == 0);
  return run8<kEpiScores>(q, sc, base, workspace, workspace_bytes, nullptr, nullptr, dev_status,
                          static_cast<cudaStream_t>(stream), "fk_int8_scores");
}

extern "C" int fk_int8_assign(const void* x, const int8_t* centroids, const float* x_scale,
                              const float* c_scale, const float* bias, int32_t* out, int x_dtype,
                              int64_t B, int64_t N, int64_t K, int64_t D, const int64_t* x_strides3,
                              const int64_t* c_strides3, const int64_t* xs_strides2,
                              const int64_t* cs_strides2, const int64_t* bias_strides2,
                              const int64_t* out_strides2, void* workspace, size_t workspace_bytes,
                              int32_t* dev_status, void* stream) {
  Scores q;
  int st = make8(q, x, centroids, x_dtype, B, N, K, D, x_strides3, c_strides3, "fk_int8_assign");
  if (st != FK_OK) return st;
  if (B == 0 || N == 0) return FK_OK;
  const Scales sc{x_scale, c_scale, bias, xs_strides2, cs_strides2, bias_strides2};
  if ((st = check8(x, centroids, x_dtype, sc, "fk_int8_assign")) != FK_OK) return st;
  if (!out || !out_strides2) return fail(FK_ERR_INVALID_ARG, "fk_int8_assign: null pointer");
  return run8<kEpiArgmax>(q, sc, Problem{}, workspace, workspace_bytes, out, out_strides2, dev_status,
                          static_cast<cudaStream_t>(stream), "fk_int8_assign");
}
