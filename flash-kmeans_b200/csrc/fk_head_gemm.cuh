// Matrix product core of the cluster head (cross entropy over centroids and
// 8-bit scores): a persistent, warp-specialised tcgen05 kernel whose epilogue
// consumes the accumulator tile instead of storing the scores.
//
//   acc[m, n] = sum_k A[m, k] B[n, k]
//
// A and B are 16-bit (float32 accumulator) or 8-bit integers (int32
// accumulator).  Each operand is K-major (rows of the contraction axis) or,
// for 16-bit types, MN-major (the contraction axis is the row axis in memory),
// so x.c^T, P.c and P^T.x all run without a transposed copy.
//
// Warp roles: warp 0 TMA producer, warp 1 MMA issuer (one thread), warps 4-11
// epilogue (four TMEM lane quarters x two column halves).  With CG = 2 two
// CTAs of a cluster form one 256 x 256 tile (cta_group::2): each loads its own
// 128 rows of A and its own half of B, so a CTA moves 32 KB per 64 columns of
// the contraction instead of the 48 KB of a 128 x 256 tile, which is what
// keeps the L2 feed below the tensor core's pace.  CG = 1 (128 x 128, 128 x 64
// tiles) serves problems with too few tiles to fill 74 pairs.
//
// Two accumulators alternate in TMEM, so the epilogue of one tile overlaps the
// products of the next.  Every wait is bounded (fk_ptx.cuh).
#pragma once
#include <climits>

#include "fk_common.cuh"
#include "fk_ptx.cuh"

namespace fk {
namespace head {

constexpr int kMaxPairs = 6;
constexpr int kCtlWarps = 4;
constexpr int kEpiWarps = 8;
constexpr int kThreads = (kCtlWarps + kEpiWarps) * 32;
constexpr int kStageRowBytes = 128;            // one swizzle row: 64 16-bit or 128 8-bit elements
constexpr int kStagingBytes = kEpiWarps * 4096;  // 32 rows x 128 bytes for each epilogue warp

constexpr int kTableBytes = 2 * 2 * 256 * 4;     // two tables of 256 column scales and biases
constexpr int kSlotBytes = 128 * 8;              // one (value, index) for each row of the tile

enum Epilogue {
  kEpiLse = 0,     // running maximum and sum of exp2 over the columns
  kEpiGrad = 1,    // (softmax - one-hot) * weight, rounded to 16 bits, into a piece
  kEpiOut = 2,     // scaled accumulator, kept in float32 or cast to the output
  kEpiScores = 3,  // int32 -> scaled scores
  kEpiArgmax = 4   // int32 -> index of the largest scaled score
};
__host__ __device__ constexpr bool running(int epi) { return epi == kEpiLse || epi == kEpiArgmax; }
__host__ __device__ constexpr bool integer(int epi) { return epi == kEpiScores || epi == kEpiArgmax; }

// What the backward pass needs of a row: P = exp2((z - top) * scale2) * coef at
// other columns, `at_label` at the label's.  An ignored row has coef = at_label = 0.
struct RowStat {
  float top;       // largest x.c of the row, the label's included
  float coef;      // weight / sum_k exp2((z_k - top) * scale2)
  float at_label;  // weight * (softmax - 1) at the label
  int label;       // the label's column, -1 for none
};

struct Problem {
  int M, N;                 // valid rows and columns of acc
  int m_tiles, n_tiles;     // tiles of this instance's shape
  int batches;
  int chunks;               // running epilogues: column chunks of a row block; else splits of the contraction
  int kblocks;              // 128-byte steps of the contraction, for each operand pair
  int npairs;               // operand parts multiplied: 1, or 6 for float32 split into three bf16 parts
  int pa[kMaxPairs], pb[kMaxPairs];
  int a_mn, b_mn;           // MN-major operands
  int a_batch, b_batch;     // z coordinate = batch * this + part * a_part
  int a_part, b_part;
  int a_off, b_off;         // first row (K-major) or first contraction index (MN-major)
  int a_rows;               // rows of A's box (K-major)
  int group;                // row blocks that share a sweep over the columns
  int window;               // running epilogues: column tiles among which row blocks start apart
  uint32_t idesc;

  // ---- epilogue
  float scale2;             // scale * log2(e)
  const void* labels;       // kEpiLse
  int label_dtype;
  int64_t label_sb, label_sn;
  int64_t ignore_index;
  float2* partial;          // kEpiLse / kEpiArgmax: [batch][chunk * 2 + half][row]
  const RowStat* stat;      // kEpiGrad: [batch][stat_rows], the row block starts at stat_off
  int64_t stat_rows;
  int64_t stat_off;
  int col_off;              // first column of the piece
  float p_scale;            // kEpiGrad: power of two that keeps float16 P out of its subnormals
  void* p_out;              // kEpiGrad: [part][batch][M][p_ld] 16-bit
  int64_t p_ld, p_part, p_batch;
  int p_parts, p_bf16;
  float fscale;             // kEpiOut: factor, times *f_num, over max(*f_den, 1)
  const float* f_num;
  const int32_t* f_den;
  float* acc;               // kEpiOut: float32 accumulator [split][batch][row][acc_ld]
  int64_t acc_ld, acc_batch, acc_split;
  int acc_read, acc_write;
  void* out;                // kEpiOut final / kEpiScores: [batch][row][col]
  int out_dtype, out_vec;   // out_vec: 4 elements of a row can be stored at once
  int64_t out_sb, out_sr;
  const float* a_scale;     // integer epilogues: per row of A, per row of B, optional bias
  const float* b_scale;
  const float* bias;
  int64_t as_sb, as_sn, bs_sb, bs_sn, bias_sb, bias_sn;
  int small_acc;            // |acc| < 2^22: conversion by an integer add
  int32_t* label_out;       // kEpiArgmax with one chunk: labels
  int64_t lo_sb, lo_sn;
  uint32_t* zero;           // words cleared for the kernel that follows
  int zero_n;
  int* status;
};

struct Params {
  CUtensorMap a, b;
  Problem p;
};

template <int CG, int BN, int EPI>
struct Shape {
  static constexpr int kBM = 128 * CG;
  static constexpr int kARows = 128;             // of one CTA
  static constexpr int kBRows = BN / CG;         // of one CTA
  static constexpr int kABytes = kARows * kStageRowBytes;
  static constexpr int kBBytes = kBRows * kStageRowBytes;
  static constexpr int kStageBytes = kABytes + kBBytes;
  // the argmax keeps column tables and the best chunk of every row besides
  static constexpr int kStages = (EPI == kEpiArgmax ? 160 : 192) * 1024 / kStageBytes;
  static constexpr int kExtra = EPI == kEpiArgmax ? kTableBytes + kSlotBytes : 0;
  static constexpr int kTmemCols = 2 * BN;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kStagingBytes + kExtra + 512;
  static_assert(kSmem <= 232448, "shared memory");
};

// ------------------------------------------------------------------ helpers
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float fmax3(float a, float b, float c) { return fmaxf(a, fmaxf(b, c)); }

__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Two floats rounded to nearest even as packed bf16 / f16, `lo` in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Where a tile sits.  Running epilogues visit the column tiles of a
// (batch, row block, chunk) item in turn; the others one tile per item.
struct Tile {
  int b, m, n, chunk;
  int it0, it1;        // steps of the flattened (pair, kblock) contraction
  bool first, last;    // of the item
};

template <int EPI>
struct Walk {
  const Problem& p;
  int64_t item, total;
  int step;
  int j, j_begin, j_end;

  __device__ Walk(const Problem& q, int64_t first, int stride) : p(q), item(first), step(stride) {
    total = static_cast<int64_t>(p.batches) * p.chunks * p.m_tiles * (running(EPI) ? 1 : p.n_tiles);
    begin();
  }
  __device__ void begin() {
    if (running(EPI) && item < total) {
      const int c = static_cast<int>(item % p.chunks);
      j_begin = static_cast<int>(static_cast<int64_t>(p.n_tiles) * c / p.chunks);
      j_end = static_cast<int>(static_cast<int64_t>(p.n_tiles) * (c + 1) / p.chunks);
      j = j_begin;
    }
  }
  __device__ bool get(Tile& t) const {
    if (item >= total) return false;
    const int steps = p.npairs * p.kblocks;
    if constexpr (running(EPI)) {
      t.chunk = static_cast<int>(item % p.chunks);
      const int64_t r = item / p.chunks;
      t.m = static_cast<int>(r % p.m_tiles);
      t.b = static_cast<int>(r / p.m_tiles);
      // row blocks start at different tiles of a window, so that they do not
      // all read the same centroids from the same L2 slices at once
      const int rel = j - j_begin;
      const int w0 = rel / p.window * p.window;
      const int wl = min(p.window, j_end - j_begin - w0);
      t.n = j_begin + w0 + (rel - w0 + t.m) % wl;
      t.it0 = 0;
      t.it1 = steps;
      t.first = j == j_begin;
      t.last = j + 1 == j_end;
    } else {
      const int per = p.m_tiles * p.n_tiles;
      const int64_t r = item / per;
      int i = static_cast<int>(item % per);
      t.chunk = static_cast<int>(r % p.chunks);
      t.b = static_cast<int>(r / p.chunks);
      const int band = p.group * p.n_tiles;
      const int g0 = i / band * p.group;
      const int gl = min(p.group, p.m_tiles - g0);
      i -= g0 * p.n_tiles;
      t.m = g0 + i % gl;
      t.n = i / gl;
      t.it0 = static_cast<int>(static_cast<int64_t>(steps) * t.chunk / p.chunks);
      t.it1 = static_cast<int>(static_cast<int64_t>(steps) * (t.chunk + 1) / p.chunks);
      t.first = t.last = true;
    }
    return true;
  }
  __device__ void next() {
    if constexpr (running(EPI)) {
      if (++j < j_end) return;
    }
    item += step;
    begin();
  }
};

__device__ __forceinline__ int64_t load_label(const void* p, int64_t i, int dt) {
  return dt == FK_I64 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// acc (int32) as float: exact for |acc| < 2^22 by placing it in the mantissa of
// 1.5 * 2^23 (an add on the integer pipe, an add on the float pipe; the
// conversion instruction runs at an eighth of their rate), else converted.
__device__ __forceinline__ float acc_to_f(uint32_t v, bool small) {
  return small ? __uint_as_float(v + 0x4B400000u) - 12582912.0f
               : static_cast<float>(static_cast<int32_t>(v));
}

// Maximum that a NaN wins, as argmax counts it.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Whether (v, i) comes before (m, j): NaN first, then the larger value, then the lower index.
__device__ __forceinline__ bool argmax_better(float v, int i, float m, int j) {
  if (v > m) return true;
  if (v < m) return false;
  if (v == m) return i < j;
  return v != v && (m == m || i < j);
}

// Barrier of the epilogue warps alone.
__device__ __forceinline__ void epilogue_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory");
}

// ------------------------------------------------------------------- kernel
// EXACT: the tensor core adds to its float32 accumulator with truncation, a
// bias of up to 2^-24 of the partial sum for every 16 elements.  16-bit inputs
// leave it at that (the label's score, which the loss hangs on most, is summed
// in ordinary float32 by the combine kernel); float32 inputs move the
// accumulator to registers every kSegment steps and add there, rounded.  Their
// tiles are 128 columns wide: 64 sums a thread leave the epilogue its registers.
constexpr int kSegment = 4;       // of 64 elements: 16 truncated additions

template <int CG, int BN, int EPI, bool EXACT>
__global__ void __launch_bounds__(kThreads, 1) head_gemm(const __grid_constant__ Params prm) {
  using S = Shape<CG, BN, EPI>;
  const Problem& p = prm.p;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* staging = smem + S::kStages * S::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + kStagingBytes + S::kExtra);
  uint64_t* empty = full + S::kStages;
  uint64_t* acc_full = empty + S::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  const bool leader = rank == 0;
  const int first = blockIdx.x / CG;
  const int stride = gridDim.x / CG;

  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&prm.a);
    tma_prefetch_desc(&prm.b);
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kEpiWarps * CG);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 2) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(tmem_slot, S::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, S::kTmemCols);
      tmem_relinquish();
    }
  }
  if (warp == 3 && blockIdx.x == 0)
    for (int i = lane; i < p.zero_n; i += 32) p.zero[i] = 0;
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      const uint32_t tx = static_cast<uint32_t>(
          (p.a_mn ? S::kABytes : p.a_rows * kStageRowBytes) + S::kBBytes) * CG;
      const int kstep = integer(EPI) ? 128 : 64;
      int stage = 0;
      uint32_t phase = 0;
      Walk<EPI> walk(p, first, stride);
      bool ok = true;
      for (Tile t; ok && walk.get(t); walk.next()) {
        int pair = t.it0 / p.kblocks, kb = t.it0 % p.kblocks;
        for (int it = t.it0; it < t.it1; ++it) {
          if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, p.status, FK_DEV_WAIT_TIMEOUT)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + stage * S::kStageBytes;
          uint8_t* sb = sa + S::kABytes;
          if (leader) mbar_arrive_expect_tx(&full[stage], tx);
          const uint32_t bar = CG == 2 ? map_to_rank(&full[stage], 0) : smem_u32(&full[stage]);
          const int az = t.b * p.a_batch + p.pa[pair] * p.a_part;
          const int bz = t.b * p.b_batch + p.pb[pair] * p.b_part;
          const int am = t.m * S::kBM + static_cast<int>(rank) * S::kARows;
          const int bn = t.n * BN + static_cast<int>(rank) * S::kBRows;
          if (p.a_mn) {
#pragma unroll
            for (int g = 0; g < S::kARows / 64; ++g)
              tma_load_3d_cg<CG>(sa + g * 8192, &prm.a, bar, am + g * 64, p.a_off + kb * 64, az);
          } else {
            tma_load_3d_cg<CG>(sa, &prm.a, bar, kb * kstep, p.a_off + am, az);
          }
          if (p.b_mn) {
#pragma unroll
            for (int g = 0; g < S::kBRows / 64; ++g)
              tma_load_3d_cg<CG>(sb + g * 8192, &prm.b, bar, bn + g * 64, p.b_off + kb * 64, bz);
          } else {
            tma_load_3d_cg<CG>(sb, &prm.b, bar, kb * kstep, p.b_off + bn, bz);
          }
          if (++stage == S::kStages) {
            stage = 0;
            phase ^= 1;
          }
          if (++kb == p.kblocks) {
            kb = 0;
            ++pair;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (lane == 0 && leader) {
      const uint32_t idesc = p.idesc;
      const uint32_t a_step = p.a_mn ? 2048 : 32, b_step = p.b_mn ? 2048 : 32;
      int stage = 0, buf = 0;
      uint32_t phase = 0, aphase = 0;
      Walk<EPI> walk(p, first, stride);
      bool ok = true;
      for (Tile t; ok && walk.get(t); walk.next()) {
        uint32_t accumulate = 0;
        for (int it = t.it0; it < t.it1; ++it) {
          if (accumulate == 0) {
            if (!mbar_wait_cluster(&acc_empty[buf], aphase ^ 1, abort_flag, p.status,
                                   FK_DEV_WAIT_TIMEOUT)) {
              ok = false;
              break;
            }
            tc_fence_after();
          }
          const uint32_t d = tmem + buf * BN;
          if (!mbar_wait(&full[stage], phase, abort_flag, p.status, FK_DEV_WAIT_TIMEOUT)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(smem + stage * S::kStageBytes);
          const uint32_t b0 = a0 + S::kABytes;
          uint64_t ad = p.a_mn ? smem_desc_sw128_mn(a0, 8192, 1024) : smem_desc_sw128(a0);
          uint64_t bd = p.b_mn ? smem_desc_sw128_mn(b0, 8192, 1024) : smem_desc_sw128(b0);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (integer(EPI)) mma_i8_cg<CG>(d, ad, bd, idesc, accumulate);
            else mma_f16_cg<CG>(d, ad, bd, idesc, accumulate);
            accumulate = 1;
            ad += a_step >> 4;
            bd += b_step >> 4;
          }
          mma_commit_cg<CG>(&empty[stage]);
          if (++stage == S::kStages) {
            stage = 0;
            phase ^= 1;
          }
          if (it + 1 == t.it1 || (EXACT && (it + 1 - t.it0) % kSegment == 0)) {
            mma_commit_cg<CG>(&acc_full[buf]);
            buf ^= 1;
            if (buf == 0) aphase ^= 1;
            accumulate = 0;
          }
        }
      }
    }
  } else if (warp >= kCtlWarps) {
    // ------------------------------------------------------------ epilogue
    const int ew = warp - kCtlWarps;
    const int half = ew >> 2;
    const int quarter = warp & 3;
    constexpr int kCols = BN / 2;          // columns of this warp
    constexpr int kChunks = kCols / 32;
    uint8_t* stg = staging + ew * 4096;
    int buf = 0;
    uint32_t aphase = 0;
    Walk<EPI> walk(p, first, stride);

    // running state of a row
    float run_m = -INFINITY, run_s = 0.0f;
    int run_i = 0;
    int64_t label = -1;
    float xs = 0.0f;
    float fac = 0.0f;
    if constexpr (EPI == kEpiOut) {
      fac = p.fscale;
      if (p.f_num) fac *= *p.f_num;
      if (p.f_den) fac /= static_cast<float>(max(*p.f_den, 1));
    }

    for (Tile t; walk.get(t); walk.next()) {
      const int row = t.m * S::kBM + static_cast<int>(rank) * 128 + quarter * 32 + lane;
      const int row0 = row - lane;
      const bool row_ok = row < p.M;
      const int col0 = t.n * BN + half * kCols;

      if constexpr (EPI == kEpiLse) {
        if (t.first) {
          run_m = -INFINITY;
          run_s = 0.0f;
          label = -1;
          if (row_ok) {
            const int64_t y = load_label(p.labels, t.b * p.label_sb + row * p.label_sn, p.label_dtype);
            label = y == p.ignore_index ? -1 : y;
          }
        }
      }
      RowStat st = {0.0f, 0.0f, 0.0f, -1};
      if constexpr (EPI == kEpiGrad) {
        if (row_ok) {
          st = p.stat[t.b * p.stat_rows + p.stat_off + row];
          st.coef *= p.p_scale;
          st.at_label *= p.p_scale;
        }
      }
      if constexpr (integer(EPI)) {
        if (t.first) xs = row_ok ? p.a_scale[t.b * p.as_sb + row * p.as_sn] : 0.0f;
      }
      float* table = reinterpret_cast<float*>(staging + kStagingBytes);
      if constexpr (EPI == kEpiArgmax) {
        if (t.first) {
          run_m = -INFINITY;
          run_i = INT_MAX;
        }
        // this tile's column scales and biases, two tables in turn; the
        // barrier also keeps the tile before last's readers ahead of the writes
        table += buf * (2 * 256);
        const int c = (warp - kCtlWarps) * 32 + lane;
        if (c < BN) {
          const int col = t.n * BN + c;
          const bool ok = col < p.N;
          table[c] = ok ? p.b_scale[t.b * p.bs_sb + col * p.bs_sn] : 0.0f;
          table[256 + c] = ok && p.bias ? p.bias[t.b * p.bias_sb + col * p.bias_sn] : 0.0f;
        }
        epilogue_sync();
      }

      // one chunk of 32 columns, accumulators in v
      auto chunk = [&](const int c, uint32_t (&v)[32]) {
        const int cc = col0 + c * 32;

        if constexpr (EPI == kEpiLse) {
          const int left = p.N - cc;
          if (left < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i >= left) v[i] = 0xff800000u;  // -inf past the last centroid
          }
          const int64_t rel = label - cc;
          if (rel >= 0 && rel < 32 && rel < left) {
            // the label's own term stays out of the sum
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (rel == i) v[i] = 0xff800000u;
          }
          float mx[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) mx[i] = __uint_as_float(v[i]);
#pragma unroll
          for (int i = 4; i < 32; i += 8)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              mx[q] = i + 4 + q < 32 ? fmax3(mx[q], __uint_as_float(v[i + q]), __uint_as_float(v[i + 4 + q]))
                                     : fmaxf(mx[q], __uint_as_float(v[i + q]));
          // differences of scores first, then the scale: exact near the maximum,
          // and never above 0, however large the scores are
          const float m_new = fmaxf(run_m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
          const float m_use = m_new == -INFINITY ? 0.0f : m_new;
          const uint64_t s2 = pack2(p.scale2, p.scale2), nm = pack2(-m_use, -m_use);
          uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float e0, e1;
            unpack2(mul2(add2(pack2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), nm), s2), e0, e1);
            sum[(i >> 1) & 3] = add2(sum[(i >> 1) & 3], pack2(ex2(e0), ex2(e1)));
          }
          float s0, s1;
          unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), s0, s1);
          run_s = run_s * ex2((run_m - m_use) * p.scale2) + (s0 + s1);
          run_m = m_new;
        } else if constexpr (EPI == kEpiGrad) {
          // softmax minus one-hot, times the row's weight
          const int rel = st.label - p.col_off - cc;
          const uint64_t s2 = pack2(p.scale2, p.scale2), nm = pack2(-st.top, -st.top);
          float e[32];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            unpack2(mul2(add2(pack2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), nm), s2), e[i], e[i + 1]);
            e[i] = ex2(e[i]) * st.coef;
            e[i + 1] = ex2(e[i + 1]) * st.coef;
          }
          if (rel >= 0 && rel < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (rel == i) e[i] = st.at_label;
          }
          for (int part = 0; part < p.p_parts; ++part) {
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int k = q * 8 + i * 2;
                w[i] = p.p_bf16 ? pack_bf16(e[k], e[k + 1]) : pack_f16(e[k], e[k + 1]);
                if (p.p_parts > 1) {  // what this part leaves for the next
                  e[k] -= __uint_as_float(w[i] << 16);
                  e[k + 1] -= __uint_as_float(w[i] & 0xffff0000u);
                }
              }
              *reinterpret_cast<uint4*>(stg + lane * 64 + ((q ^ ((lane >> 1) & 3)) * 16)) =
                  make_uint4(w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
            uint8_t* dst = static_cast<uint8_t*>(p.p_out) +
                           2 * (part * p.p_part + t.b * p.p_batch);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int rr = i * 8 + (lane >> 2), q = lane & 3;
              if (row0 + rr < p.M && cc < p.p_ld)
                *reinterpret_cast<uint4*>(dst + 2 * ((row0 + rr) * p.p_ld + cc + q * 8)) =
                    *reinterpret_cast<const uint4*>(stg + rr * 64 + ((q ^ ((rr >> 1) & 3)) * 16));
            }
          }
        } else if constexpr (EPI == kEpiOut || EPI == kEpiScores) {
          const bool small = p.small_acc != 0;
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            float4 f;
            float* ff = &f.x;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              ff[i] = EPI == kEpiScores ? acc_to_f(v[q * 4 + i], small) * xs
                                        : __uint_as_float(v[q * 4 + i]) * fac;
            *reinterpret_cast<float4*>(stg + lane * 128 + ((q ^ (lane & 7)) * 16)) = f;
          }
          __syncwarp();
          const int q = lane & 7;
          const int col = cc + q * 4;
          float sc[4], bi[4];
          if constexpr (EPI == kEpiScores) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              sc[i] = col + i < p.N ? p.b_scale[t.b * p.bs_sb + (col + i) * p.bs_sn] : 0.0f;
              bi[i] = col + i < p.N && p.bias ? p.bias[t.b * p.bias_sb + (col + i) * p.bias_sn] : 0.0f;
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int rr = i * 4 + (lane >> 3);
            const int64_t grow = row0 + rr;
            if (grow >= p.M || col >= p.N) continue;
            float4 f = *reinterpret_cast<const float4*>(stg + rr * 128 + ((q ^ (rr & 7)) * 16));
            if constexpr (EPI == kEpiScores) {
              float* ff = &f.x;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                ff[k] = __fmul_rn(ff[k], sc[k]);
                if (p.bias) ff[k] = __fadd_rn(ff[k], bi[k]);
              }
            } else if (p.acc) {
              float* a = p.acc + t.chunk * p.acc_split + t.b * p.acc_batch + grow * p.acc_ld + col;
              if (p.acc_read) {
                const float4 o = *reinterpret_cast<const float4*>(a);
                f.x += o.x;
                f.y += o.y;
                f.z += o.z;
                f.w += o.w;
              }
              if (p.acc_write) {
                *reinterpret_cast<float4*>(a) = f;
                continue;
              }
            }
            const int64_t o = t.b * p.out_sb + grow * p.out_sr + col;
            if (p.out_vec && col + 4 <= p.N) {
              if (p.out_dtype == FK_F32) {
                *reinterpret_cast<float4*>(static_cast<float*>(p.out) + o) = f;
              } else {
                uint2 w;
                w.x = p.out_dtype == FK_BF16 ? pack_bf16(f.x, f.y) : pack_f16(f.x, f.y);
                w.y = p.out_dtype == FK_BF16 ? pack_bf16(f.z, f.w) : pack_f16(f.z, f.w);
                *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + o) = w;
              }
            } else {
              const float* ff = &f.x;
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (col + k < p.N) store_f(p.out, o + k, p.out_dtype, ff[k]);
            }
          }
        } else {  // kEpiArgmax
          const float* sc = table + half * kCols + c * 32;
          const float* bi = sc + 256;
          const bool small = p.small_acc != 0;
          const uint64_t x2 = pack2(xs, xs);
          float z[32];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 s4 = *reinterpret_cast<const float4*>(sc + i);
            uint64_t z0 = mul2(mul2(pack2(acc_to_f(v[i], small), acc_to_f(v[i + 1], small)), x2),
                               pack2(s4.x, s4.y));
            uint64_t z1 = mul2(mul2(pack2(acc_to_f(v[i + 2], small), acc_to_f(v[i + 3], small)), x2),
                               pack2(s4.z, s4.w));
            if (p.bias) {
              const float4 b4 = *reinterpret_cast<const float4*>(bi + i);
              z0 = add2(z0, pack2(b4.x, b4.y));
              z1 = add2(z1, pack2(b4.z, b4.w));
            }
            unpack2(z0, z[i], z[i + 1]);
            unpack2(z1, z[i + 2], z[i + 3]);
          }
          const int left = p.N - cc;
          if (left < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i >= left) z[i] = -INFINITY;
          }
          float mx[4] = {z[0], z[1], z[2], z[3]};
#pragma unroll
          for (int i = 4; i < 32; ++i) mx[i & 3] = max_nan(mx[i & 3], z[i]);
          const float m = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3]));
          if (left > 0 && argmax_better(m, cc, run_m, run_i)) {
            // keep the chunk: which of its columns won is looked up once, at
            // the end of the row, instead of at every improvement
            run_m = m;
            run_i = cc;
#pragma unroll
            for (int q = 0; q < 8; ++q)
              *reinterpret_cast<float4*>(stg + lane * 128 + ((q ^ (lane & 7)) * 16)) =
                  make_float4(z[q * 4], z[q * 4 + 1], z[q * 4 + 2], z[q * 4 + 3]);
          }
        }
      };

      bool got = true;
      if constexpr (EXACT) {
        float sum[kChunks][32];
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) sum[c][i] = 0.0f;
        for (int it = t.it0; it < t.it1; it += kSegment) {
          got = __all_sync(0xffffffffu, mbar_wait(&acc_full[buf], aphase, abort_flag, p.status,
                                                  FK_DEV_WAIT_TIMEOUT));
          if (!got) break;
          tc_fence_after();
          const uint32_t taddr =
              tmem + buf * BN + half * kCols + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            uint32_t v[32];
            tmem_ld32(taddr + c * 32, v);
            tmem_ld_wait(v);
#pragma unroll
            for (int i = 0; i < 32; i += 2)
              unpack2(add2(pack2(sum[c][i], sum[c][i + 1]),
                           pack2(__uint_as_float(v[i]), __uint_as_float(v[i + 1]))),
                      sum[c][i], sum[c][i + 1]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cg<CG>(&acc_empty[buf]);
          buf ^= 1;
          if (buf == 0) aphase ^= 1;
        }
        if (!got) break;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          uint32_t v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(sum[c][i]);
          chunk(c, v);
        }
      } else {
        got = __all_sync(0xffffffffu, mbar_wait(&acc_full[buf], aphase, abort_flag, p.status,
                                                FK_DEV_WAIT_TIMEOUT));
        if (!got) {
          if constexpr (EPI == kEpiArgmax) {
            // the other warps meet at the barriers of every tile: keep to them
            if (t.last && p.chunks == 1) epilogue_sync();
            buf ^= 1;
            if (buf == 0) aphase ^= 1;
            continue;
          } else {
            break;
          }
        }
        tc_fence_after();
        const uint32_t taddr =
            tmem + buf * BN + half * kCols + (static_cast<uint32_t>(quarter * 32) << 16);
        uint32_t r[2][32];
        tmem_ld32(taddr, r[0]);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          tmem_ld_wait(r[c & 1]);
          if (c + 1 < kChunks) {
            tmem_ld32(taddr + (c + 1) * 32, r[(c + 1) & 1]);
          } else {
            // the accumulator is in registers: hand it back
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cg<CG>(&acc_empty[buf]);
          }
          chunk(c, r[c & 1]);
        }
        buf ^= 1;
        if (buf == 0) aphase ^= 1;
      }

      if constexpr (EPI == kEpiLse) {
        if (t.last && row_ok)
          p.partial[(static_cast<int64_t>(t.b) * p.chunks * 2 + t.chunk * 2 + half) * p.M + row] =
              make_float2(run_m, run_s);
      }
      if constexpr (EPI == kEpiArgmax) {
        if (t.last) {
          if (run_i != INT_MAX) {
            int at = 0;
#pragma unroll
            for (int q = 7; q >= 0; --q) {
              const float4 f = *reinterpret_cast<const float4*>(stg + lane * 128 + ((q ^ (lane & 7)) * 16));
              const float* ff = &f.x;
#pragma unroll
              for (int i = 3; i >= 0; --i)
                if (ff[i] == run_m || ff[i] != ff[i]) at = q * 4 + i;
            }
            run_i += at;
          }
          if (p.chunks == 1) {
            // the two column halves of a row meet in shared memory
            float2* slot = reinterpret_cast<float2*>(staging + kStagingBytes + kTableBytes) +
                           (quarter * 32 + lane);
            if (half == 1) *slot = make_float2(run_m, __int_as_float(run_i));
            epilogue_sync();
            if (half == 0 && row_ok) {
              const float2 o = *slot;
              if (argmax_better(o.x, __float_as_int(o.y), run_m, run_i)) run_i = __float_as_int(o.y);
              p.label_out[t.b * p.lo_sb + row * p.lo_sn] = run_i;
            }
          } else if (row_ok) {
            p.partial[(static_cast<int64_t>(t.b) * p.chunks * 2 + t.chunk * 2 + half) * p.M + row] =
                make_float2(run_m, __int_as_float(run_i));
          }
        }
      }
    }
  }

  // A role that gave up may have copies or products in flight: let them land
  // before the memory they write goes away.
  __syncthreads();
  if (*abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  tc_fence_after();
  if (warp == 2) {
    if constexpr (CG == 2) tmem_dealloc_pair(tmem, S::kTmemCols);
    else tmem_dealloc(tmem, S::kTmemCols);
  }
}

}  // namespace head
}  // namespace fk
