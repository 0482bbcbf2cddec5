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
// Warp roles: warp 0 TMA producer, warp 1 MMA issuer (one thread), warps 4 and
// up epilogue (four TMEM lane quarters x two or four column parts).  With CG = 2 two
// CTAs of a cluster form one 256 x 256 tile (cta_group::2): each loads its own
// 128 rows of A and its own half of B, so a CTA moves 32 KB per 64 columns of
// the contraction instead of the 48 KB of a 128 x 256 tile.  That matters: with
// all SMs reading, the L2 delivers 11 to 12 TB/s, and a 256 x 256 pair tile needs
// 32 KB for 0.38 us of products (16384 x 32768 x 1024 forward: 658 us, 1.67
// PFLOP/s alone; 128 x 128 tiles took 1.6 times as long).  CG = 1 (128 x 128,
// 128 x 64 tiles) serves problems with too few tiles to fill 74 pairs.
//
// Two or four accumulators alternate in TMEM, so the epilogue of one tile
// overlaps the products of the next.  Every wait is bounded (fk_ptx.cuh).
#pragma once
#include <climits>
#include <type_traits>

#include "fk_common.cuh"
#include "fk_ptx.cuh"

namespace fk {
namespace head {

constexpr int kCtlWarps = 4;
constexpr int kStageRowBytes = 128;            // one swizzle row: 64 16-bit or 128 8-bit elements
constexpr int kSlotBytes = 2 * 128 * 8;        // (value, index) of two items' rows from the other column part

enum Epilogue {
  kEpiLse = 0,     // running maximum and sum of exp2 over the columns
  kEpiGrad = 1,    // (softmax - one-hot) * weight, rounded to 16 bits, into a piece
  kEpiOut = 2,     // scaled accumulator, kept in float32 or cast to the output
  kEpiScores = 3,  // int32 -> scaled scores
  kEpiArgmax = 4,  // int32 -> index of the largest scaled score
  kEpiOutRows = 5  // kEpiOut with what rows have of their own (testing for it would cost kEpiOut 1 %)
};
__host__ __device__ constexpr bool output(int epi) { return epi == kEpiOut || epi == kEpiOutRows; }
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
  int kblocks;              // 128-byte steps of the contraction
  int a_mn;                 // MN-major A (B is MN-major in the output epilogues alone)
  int a_batch, b_batch;     // z coordinate = batch * this + part * a_part
  int a_part, b_part;
  int a_off, b_off;         // first row (K-major) or first contraction index (MN-major)
  int a_rows;               // rows of A's box (K-major)
  int group;                // row blocks that share a sweep over the columns
  int window;               // running epilogues: column tiles among which row blocks start apart
  uint32_t idesc;
  // kEpiLse, kEpiGrad, kEpiOut: only the rows that are not ignored take part,
  // gathered; their number is known on the device alone
  const int32_t* live;      // that number; null: all rows
  int live_off, live_cap;   // this chunk's first row (of all rows, with none), its rows at most
  int live_steps;           // the rows are the contraction, not the rows of A
  const int32_t* row_map;   // gathered row live_off + r is row row_map[live_off + r] of the call

  // ---- epilogue
  float scale2;             // scale * log2(e)
  const void* labels;       // kEpiLse
  int label_dtype;
  int64_t label_sb, label_sn;
  int64_t ignore_index;
  float2* partial;          // kEpiLse / kEpiArgmax: [batch][chunk][part][row]
  const RowStat* stat;      // kEpiGrad: [batch][stat_rows], the row block starts at stat_off
  int64_t stat_rows;
  int64_t stat_off;
  int col_off;              // first column of the piece
  float p_scale;            // kEpiGrad: power of two that keeps float16 P out of its subnormals
  void* p_out;              // kEpiGrad: [part][batch][M][p_ld] 16-bit
  int64_t p_ld, p_part, p_batch;
  int p_bf16;
  float fscale;             // kEpiOut: factor, times *f_num, over max(*f_den, 1)
  const float* f_num;
  const int32_t* f_den;
  // kEpiOutRows: what rounding took from P at the label, times that centroid, is
  // added to the row (stat, stat_rows and p_scale as for kEpiGrad); null: none
  const uint16_t* label_rows;   // the centroids, 16 bytes from aligned row to row
  int64_t label_ld, label_batch;
  const float* row_factor;  // kEpiOutRows: and times that of the row, or null: [batch][stat_rows]
  float* acc;               // kEpiOut: float32 accumulator [split][batch][row][acc_ld]
  int64_t acc_ld, acc_batch, acc_split;
  int acc_read, acc_write;
  uint32_t* join;           // kEpiOut, splits that are added up here: an arrival counter for each
  int join_splits;          // warp of a tile, zero on entry and on exit; null otherwise
  void* out;                // kEpiOut final / kEpiScores: [batch][row][col]
  int out_dtype, out_vec;   // out_vec: 4 elements of a row can be stored at once
  int64_t out_sb, out_sr;
  const float* a_scale;     // integer epilogues: per row of A, per row of B, optional bias
  const float* b_scale;
  const float* bias;
  int64_t as_sb, as_sn, bs_sb, bs_sn, bias_sb, bias_sn;
  float unit;               // kEpiArgmax: 1 (see add2_rounded)
  int32_t* label_out;       // kEpiArgmax with one chunk: labels
  int64_t lo_sb, lo_sn;
  uint32_t* zero;           // words cleared for the kernel that follows
  int zero_n;
  int* status;
};

// kEpiOut runs the two gradient products of a piece in one launch, the one with
// the longer tiles first; its workers then take the other's tiles so that all
// finish together.  In the second product every worker has `all` tiles, the
// workers from `short_from` on (one tile of the first product behind) `more`
// others, and the last `rest` workers one more.
constexpr int problems_of(int epi) { return output(epi) ? 2 : 1; }

template <int NP>
struct Params {
  CUtensorMap a[NP], b[NP];
  Problem p[NP];
  int count;
  int all, short_from, more, rest;
};

template <int CG, int BN, int EPI, bool EXACT>
struct Shape {
  static constexpr int kBM = 128 * CG;
  static constexpr int kARows = 128;             // of one CTA
  static constexpr int kBRows = BN / CG;         // of one CTA
  static constexpr int kABytes = kARows * kStageRowBytes;
  static constexpr int kBBytes = kBRows * kStageRowBytes;
  // EXACT: a step brings the three parts of both operands, used by six products
  static constexpr int kOps = EXACT ? 3 : 1;
  static constexpr int kStageBytes = kOps * (kABytes + kBBytes);
  // Epilogue warps: four TMEM lane quarters x column parts.  Four parts give
  // each scheduler four warps, which is what hides the exponentials' and the
  // accumulator loads' latency (two left 70 % of the issue slots empty).
  // The argmax has work at every row's end that each part adds to: with four, 302400
  // x 1000 x 128 took 126 us against 129, 604800 x 256 x 64 93 against 83.
  static constexpr int kParts = BN >= 128 && EPI != kEpiArgmax ? 4 : 2;
  static constexpr int kEpiWarps = 4 * kParts;
  static constexpr int kThreads = (kCtlWarps + kEpiWarps) * 32;
  // shared memory of an epilogue warp: 32 rows of 128 bytes (64 for P)
  static constexpr int kStaging =
      EPI == kEpiLse ? 0 : EPI == kEpiGrad ? 2048 : 4096;
  static constexpr int kStagingBytes = kEpiWarps * kStaging;
  // the argmax's column scales and biases, of this tile and of the next, by warp
  static constexpr int kTable = 2 * (BN / kParts) * 4;
  static constexpr int kTables = kEpiWarps * 2 * kTable;
  static constexpr int kExtra = EPI == kEpiArgmax ? kTables + kSlotBytes : 0;
  static constexpr int kRoom = 232448 - 1024 - 512 - kStagingBytes - kExtra;
  static constexpr int kStages = kRoom / kStageBytes > 8 ? 8 : kRoom / kStageBytes;
  // accumulators in turn: the more, the less a tile waits for the one before
  static constexpr int kBufs = BN >= 256 ? 2 : 4;
  static constexpr int kTmemCols = kBufs * BN;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kStagingBytes + kExtra + 512;
  static_assert(kStages >= (EXACT ? 2 : 4) && kSmem <= 232448, "shared memory");
};

template <int CG, int BN, int EPI, bool EXACT>
constexpr int threads_of() { return Shape<CG, BN, EPI, EXACT>::kThreads; }
// column parts that write partial results of a row
inline int parts_of(int epi, int bn) { return bn >= 128 && epi != kEpiArgmax ? 4 : 2; }

// ------------------------------------------------------------------ helpers
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float fmax3(float a, float b, float c) { return fmaxf(a, fmaxf(b, c)); }

__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void sts32(uint32_t at, uint32_t a) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(a) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 u;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(at) : "memory");
  return u;
}

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
// a + b where a is a product that has to be rounded first: mul2 and add2 in
// sequence came out as one fused step, for all their .rn.  `one` holds 1 twice,
// which the compiler must not know.
__device__ __forceinline__ uint64_t add2_rounded(uint64_t a, uint64_t one, uint64_t b) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(one), "l"(b));
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
  int q;               // which problem
  int b, m, n, chunk;
  int it0, it1;        // steps of the contraction
  bool first, last;    // of the item
};

// Every role walks the tiles by itself, in one thread: the decoding is kept to
// 32-bit divisions, once per item (64-bit ones at every tile took 2000 cycles,
// more than a short tile's products).
template <int EPI, int BM>
struct Walk {
  static constexpr int NP = problems_of(EPI);
  static constexpr bool kLive = EPI == kEpiLse || EPI == kEpiGrad || output(EPI);
  const Params<NP>& prm;
  uint32_t item, total;
  const uint32_t slot, slots;
  Tile t;
  int j_begin, j_end, w_end, wl, w0, j;
  int m_tiles[NP], steps[NP];
  int all, short_from, more, rest;

  __device__ Walk(const Params<NP>& q, int first, int stride) : prm(q), slot(first), slots(stride) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const Problem& p = prm.p[i];
      m_tiles[i] = p.m_tiles;
      steps[i] = p.kblocks;
      if (kLive && p.live) {
        const int rows = live_rows(p);
        if (p.live_steps) steps[i] = (rows + 63) / 64;
        else m_tiles[i] = (rows + BM - 1) / BM;
      }
    }
    all = prm.all;
    short_from = prm.short_from;
    more = prm.more;
    rest = prm.rest;
    if constexpr (NP > 1) {
      if (prm.count > 1 && prm.p[0].live) {
        // the shares that the host worked out (fill) for the rows that are left
        const uint32_t n0 = items_of(0), n1 = items_of(1);
        const uint32_t c0 = steps[0] / prm.p[0].chunks + 3, c1 = steps[1] / prm.p[1].chunks + 3;
        short_from = n0 % slots;
        const uint32_t behind = slots - short_from, want = short_from ? c0 / c1 : 0;
        const uint32_t got = min(want, n1 / behind), left = n1 - got * behind;
        more = got;
        all = got < want ? 0 : left / slots;
        rest = left - all * slots;
      }
    }
    t.q = 0;
    item = slot;
    total = items_of(0);
    j = -1;
    if (NP > 1 && item >= total) second();
    decode();
  }
  __device__ static int live_rows(const Problem& p) {
    return min(max(*p.live - p.live_off, 0), p.live_cap);
  }
  // rows of A that count, and those of P that are written
  __device__ static int rows_of(const Problem& p) {
    return kLive && p.live && !p.live_steps ? live_rows(p) : p.M;
  }
  __device__ uint32_t items_of(int i) const {
    const Problem& p = prm.p[i];
    return static_cast<uint32_t>(p.batches) * p.chunks * m_tiles[i] * (running(EPI) ? 1 : p.n_tiles);
  }
  // this worker's next tile of the second problem
  __device__ void second() {
    t.q = NP - 1;
    total = prm.count > 1 ? items_of(NP - 1) : 0;
    ++j;
    const uint32_t behind = short_from, tail = slots - rest;
    if (j < all) {
      item = j * slots + slot;
      return;
    }
    const int k = j - all;
    const int mine = slot >= behind ? more : 0;
    item = all * slots;
    if (k < mine) item += k * (slots - behind) + slot - behind;
    else if (k == mine && slot >= tail) item += more * (slots - behind) + slot - tail;
    else item = total;
  }
  // Row blocks start at different tiles of a window, so that they do not all
  // read the same centroids from the same L2 slices at once.
  __device__ void window(int from) {
    w0 = from;
    wl = min(prm.p[0].window, j_end - from);
    w_end = from + wl;
    t.n = w0 + static_cast<int>(static_cast<uint32_t>(t.m) % static_cast<uint32_t>(wl));
  }
  __device__ void decode() {
    if (item >= total) return;
    const Problem& p = prm.p[NP > 1 ? t.q : 0];
    const int steps = this->steps[NP > 1 ? t.q : 0], m_tiles = this->m_tiles[NP > 1 ? t.q : 0];
    if constexpr (running(EPI)) {
      uint32_t r = item;
      uint32_t c = 0;
      if (p.chunks > 1) {
        r = item / static_cast<uint32_t>(p.chunks);
        c = item - r * p.chunks;
      }
      t.chunk = c;
      t.b = r / static_cast<uint32_t>(m_tiles);
      t.m = r - t.b * m_tiles;
      j_begin = static_cast<int>(static_cast<uint32_t>(p.n_tiles) * c / static_cast<uint32_t>(p.chunks));
      j_end = static_cast<int>(static_cast<uint32_t>(p.n_tiles) * (c + 1) / static_cast<uint32_t>(p.chunks));
      t.it0 = 0;
      t.it1 = steps;
      t.first = true;
      t.last = j_begin + 1 == j_end;
      window(j_begin);
      j = j_begin;
    } else {
      const uint32_t per = static_cast<uint32_t>(m_tiles) * p.n_tiles;
      const uint32_t r = item / per;
      uint32_t i = item - r * per;
      t.b = r;
      t.chunk = 0;
      t.it0 = 0;
      t.it1 = steps;
      if (p.chunks > 1) {
        t.b = r / static_cast<uint32_t>(p.chunks);
        t.chunk = r - t.b * p.chunks;
        t.it0 = static_cast<int>(static_cast<uint32_t>(steps) * t.chunk / static_cast<uint32_t>(p.chunks));
        t.it1 = static_cast<int>(static_cast<uint32_t>(steps) * (t.chunk + 1) / static_cast<uint32_t>(p.chunks));
      }
      const uint32_t g = i / static_cast<uint32_t>(p.group * p.n_tiles);
      const int g0 = g * p.group;
      const uint32_t gl = min(p.group, m_tiles - g0);
      i -= static_cast<uint32_t>(g0) * p.n_tiles;
      t.n = i / gl;
      t.m = g0 + i - t.n * gl;
      t.first = t.last = true;
    }
  }
  __device__ bool get(Tile& out) const {
    out = t;
    return item < total;
  }
  __device__ void next() {
    if constexpr (running(EPI)) {
      if (++j < j_end) {
        t.first = false;
        t.last = j + 1 == j_end;
        if (j == w_end) window(j);
        else if (++t.n == w_end) t.n = w0;
        return;
      }
    }
    if (NP > 1 && t.q > 0) {
      second();
    } else {
      item += slots;
      if (NP > 1 && item >= total) second();
    }
    decode();
  }
};

__device__ __forceinline__ int64_t load_label(const void* p, int64_t i, int dt) {
  return dt == FK_I64 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// 32 int32 accumulators as floats, in place.
__device__ __forceinline__ void acc_to_f(uint32_t (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(static_cast<float>(static_cast<int32_t>(v[i])));
}

// Maximum that a NaN wins, as argmax counts it.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Whether (v, i) comes before (m, j): NaN first, then the larger value, then the lower index.
__device__ __forceinline__ bool argmax_better(float v, int i, float m, int j) {
  if (v > m) return true;
  if (v < m) return false;
  if (v == m) return i < j;
  return v != v && (m == m || i < j);
}

// Put into a branch that is seldom taken: the compiler would otherwise turn its
// 32 conditional moves into selects that every chunk pays for (they were more
// than half of the epilogues' instructions).
__device__ __forceinline__ void keep_branch() { asm volatile(""); }

// Barrier of the epilogue warps that share a lane quarter, hence rows.
template <int THREADS>
__device__ __forceinline__ void quarter_sync(int quarter) {
  asm volatile("bar.sync %0, %1;" ::"r"(1 + quarter), "n"(THREADS) : "memory");
}

// ------------------------------------------------------------------- kernel
// Epilogue of the argmax.  The scores' scaling and comparing bounds it (2400 scores
// a ns at 604800 x 1000 x 128: 255 us, of which the products need 47), so a row
// keeps only its best score and the 32 scores of the chunk that it came from, in
// shared memory; which column of it won is looked up once, at the end of the
// row.  A column's scale and bias come from shared memory, 16 bytes to all lanes
// at a time.  (Two rows a thread, to load each of those once for both, needs
// tiles of 128 columns to keep its accumulators in turn: the same time up to 256
// features, 31 us against 25 for 65537 x 500 x 512.)
template <int CG, int BN>
__device__ __forceinline__ void argmax_epilogue(const Params<1>& prm, uint8_t* staging, uint32_t tmem,
                                                uint64_t* acc_full, uint64_t* acc_empty,
                                                volatile int* abort_flag, int ew, int lane, uint32_t rank,
                                                int first, int stride) {
  using S = Shape<CG, BN, kEpiArgmax, false>;
  static_assert(S::kParts == 2, "one slot a row");
  const Problem& p = prm.p[0];
  constexpr int kCols = BN / S::kParts;      // columns of this warp
  constexpr int kChunks = kCols / 32;
  const int part = ew >> 2, quarter = ew & 3;
  const uint32_t save = smem_u32(staging + ew * S::kStaging) + lane * 128 + (lane & 7) * 16;
  const uint32_t tables = smem_u32(staging + S::kStagingBytes) + ew * 2 * S::kTable;
  constexpr int kBias = kCols * 4;           // the biases, behind the scales
  float2* slot = reinterpret_cast<float2*>(staging + S::kStagingBytes + S::kTables) + quarter * 32 + lane;
  int buf = 0, tab = 0, turn = 0;
  uint32_t aphase = 0;
  Walk<kEpiArgmax, S::kBM> walk(prm, first, stride);
  Tile t;
  bool more = walk.get(t);

  float run_m = -INFINITY, xs = 0.0f, xs_next = 0.0f, sc_next[kChunks], bi_next[kChunks];
  int run_i = INT_MAX;
  // The next tile's columns, and at an item's start its rows' scales: fetched a
  // tile ahead, as their latency would stand between the accumulator and its use.
  auto fetch = [&]() {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int64_t col = t.n * BN + part * kCols + c * 32 + lane;
      sc_next[c] = col < p.N ? p.b_scale[t.b * p.bs_sb + col * p.bs_sn] : 0.0f;
      bi_next[c] = col < p.N && p.bias ? p.bias[t.b * p.bias_sb + col * p.bias_sn] : 0.0f;
    }
    if (t.first) {
      const int64_t row = t.m * S::kBM + static_cast<int>(rank) * 128 + quarter * 32 + lane;
      xs_next = row < p.M ? p.a_scale[t.b * p.as_sb + row * p.as_sn] : 0.0f;
    }
  };
  // A row's end: its label, or what its chunk of the columns found.
  auto finish = [&](const Tile& now) {
    const int row = now.m * S::kBM + static_cast<int>(rank) * 128 + quarter * 32 + lane;
    if (p.chunks == 1) {
      // the two column parts of a row meet in shared memory
      // (in turn in two slots: the item after the next one writes this one again,
      // behind the next one's barrier)
      if (part == 1) slot[turn] = make_float2(run_m, __int_as_float(run_i));
      quarter_sync<S::kParts * 32>(quarter);
      if (part == 0) {
        const float2 o = slot[turn];
        if (argmax_better(o.x, __float_as_int(o.y), run_m, run_i)) run_i = __float_as_int(o.y);
        if (row < p.M) p.label_out[now.b * p.lo_sb + row * p.lo_sn] = run_i;
      }
      turn ^= 128;
    } else if (row < p.M) {
      p.partial[((static_cast<int64_t>(now.b) * p.chunks + now.chunk) * S::kParts + part) * p.M + row] =
          make_float2(run_m, __int_as_float(run_i));
    }
  };
  if (more) fetch();
  while (more) {
    const Tile now = t;
    walk.next();
    more = walk.get(t);
    if (now.first) {
      run_m = -INFINITY;
      run_i = INT_MAX;
      xs = xs_next;
    }
    const uint32_t table = tables + tab * S::kTable;
    tab ^= 1;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      sts32(table + (c * 32 + lane) * 4, __float_as_uint(sc_next[c]));
      sts32(table + kBias + (c * 32 + lane) * 4, __float_as_uint(bi_next[c]));
    }
    __syncwarp();
    if (more) fetch();

    const bool got = mbar_wait(&acc_full[buf], aphase, abort_flag, p.status, FK_DEV_WAIT_TIMEOUT);
    if (!__all_sync(0xffffffffu, got)) {
      // The labels from here on are -1, in a loop of its own: a flag looked at in
      // this one cost 2 %.  (NaN comes first, and of NaNs the lowest index.)
      for (Tile left = now;; left = t, walk.next(), more = walk.get(t)) {
        run_m = __uint_as_float(0x7fc00000u);
        run_i = -1;
        if (left.last) finish(left);
        if (!more) return;
      }
    }
    tc_fence_after();
    const uint32_t taddr = tmem + buf * BN + part * kCols + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint64_t x2 = pack2(xs, xs), one2 = pack2(p.unit, p.unit);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int cc = now.n * BN + part * kCols + c * 32, left = p.N - cc;
      uint32_t v[32];
      tmem_ld32(taddr + c * 32, v);
      tmem_ld_wait(v);
      if (c + 1 == kChunks) {
        // the accumulator is in registers: hand it back
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cg<CG>(&acc_empty[buf]);
      }
      if (left <= 0) continue;
      acc_to_f(v);
      float z[32];
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        // without a bias the table holds zeros: no branch for every column
        const uint4 s4 = lds128(table + (c * 32 + i) * 4), b4 = lds128(table + kBias + (c * 32 + i) * 4);
        const uint32_t* su = &s4.x;
        const uint32_t* bu = &b4.x;
#pragma unroll
        for (int k = 0; k < 4; k += 2)
          unpack2(add2_rounded(mul2(mul2(pack2(__uint_as_float(v[i + k]), __uint_as_float(v[i + k + 1])), x2),
                                    pack2(__uint_as_float(su[k]), __uint_as_float(su[k + 1]))),
                               one2, pack2(__uint_as_float(bu[k]), __uint_as_float(bu[k + 1]))),
                  z[i + k], z[i + k + 1]);
      }
      if (left < 32) {
        keep_branch();
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i >= left) z[i] = -INFINITY;
      }
      float mx[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        mx[q] = max_nan3(z[q], z[q + 4], z[q + 8]);
        mx[q] = max_nan3(mx[q], z[q + 12], z[q + 16]);
        mx[q] = max_nan(max_nan3(mx[q], z[q + 20], z[q + 24]), z[q + 28]);
      }
      const float m = max_nan(max_nan3(mx[0], mx[1], mx[2]), mx[3]);
      if (!(m < run_m) && argmax_better(m, cc, run_m, run_i)) {
        run_m = m;
        run_i = cc;
#pragma unroll
        for (int q = 0; q < 8; ++q)
          sts128(save ^ (q * 16), __float_as_uint(z[q * 4]), __float_as_uint(z[q * 4 + 1]),
                 __float_as_uint(z[q * 4 + 2]), __float_as_uint(z[q * 4 + 3]));
      }
    }
    if (++buf == S::kBufs) {
      buf = 0;
      aphase ^= 1;
    }
    if (!now.last) continue;

    if (run_i != INT_MAX) {
      int at = 0;
#pragma unroll
      for (int q = 7; q >= 0; --q) {
        const uint4 f = lds128(save ^ (q * 16));
        const uint32_t* fu = &f.x;
#pragma unroll
        for (int i = 3; i >= 0; --i) {
          const float g = __uint_as_float(fu[i]);
          if (g == run_m || g != g) at = q * 4 + i;
        }
      }
      run_i += at;
    }
    finish(now);
  }
}

// ------------------------------------------------------------------- kernel
// EXACT: float32 operands as three bf16 parts each.  A step loads the six part
// tiles once and issues the six products that reach above 2^-24 of the leading
// one, smallest first; loading a pair of parts per product instead fetched twice
// the bytes and was bound by the L2 (8192 x 1024 x 512 forward 71 -> 49 us).  The tensor core
// adds to its float32 accumulator with truncation, a bias of up to 2^-24 of the
// partial sum for every 16 elements.  16-bit inputs leave it at that (the
// label's score, which the loss hangs on most, is summed in ordinary float32 by
// the combine kernel); here the accumulator moves to registers after every step
// and is added there, rounded.  The tiles are 128 columns wide: 32 sums a thread
// leave the epilogue its registers.
constexpr int kSegment = 1;       // steps of 64 elements: 24 truncated additions
__device__ constexpr int kPairA[6] = {2, 0, 1, 1, 0, 0};
__device__ constexpr int kPairB[6] = {0, 2, 1, 0, 1, 0};

template <int CG, int BN, int EPI, bool EXACT>
__global__ void __launch_bounds__(threads_of<CG, BN, EPI, EXACT>(), 1) head_gemm(const __grid_constant__ Params<problems_of(EPI)> prm) {
  constexpr int NP = problems_of(EPI);
  using S = Shape<CG, BN, EPI, EXACT>;
  const Problem& p0 = prm.p[0];
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* staging = smem + S::kStages * S::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + S::kStagingBytes + S::kExtra);
  uint64_t* empty = full + S::kStages;
  uint64_t* acc_full = empty + S::kStages;
  uint64_t* acc_empty = acc_full + S::kBufs;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + S::kBufs);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  const bool leader = rank == 0;
  const int first = blockIdx.x / CG;
  const int stride = gridDim.x / CG;

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < NP; ++i) {
      tma_prefetch_desc(&prm.a[i]);
      tma_prefetch_desc(&prm.b[i]);
    }
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < S::kBufs; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], S::kEpiWarps * CG);
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
  pdl_wait_then_release();
  if (warp == 3)
    for (int i = blockIdx.x * 32 + lane; i < p0.zero_n; i += gridDim.x * 32) p0.zero[i] = 0;
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    // One thread issues every load of the CTA, one step of the contraction
    // after another: what it executes per step bounds the kernel, so all that
    // does not change from step to step is computed outside.
    if (lane == 0) {
      constexpr int kstep = integer(EPI) ? 128 : 64;
      const uint32_t smem0 = smem_u32(smem), empty0 = smem_u32(empty);
      const uint32_t full0 = smem_u32(full);                               // of this CTA
      const uint32_t bar0 = CG == 2 ? map_to_rank(full, 0) : full0;        // of the pair's first
      int stage = 0;
      uint32_t phase = 0;
      Walk<EPI, S::kBM> walk(prm, first, stride);
      bool ok = true;
      for (Tile t; ok && walk.get(t); walk.next()) {
        const Problem& p = prm.p[NP > 1 ? t.q : 0];
        const CUtensorMap *ma = &prm.a[NP > 1 ? t.q : 0], *mb = &prm.b[NP > 1 ? t.q : 0];
        const int am = t.m * S::kBM + static_cast<int>(rank) * S::kARows;
        const int bn = t.n * BN + static_cast<int>(rank) * S::kBRows;
        auto load = [&](auto a_mn, auto b_mn) {
          constexpr bool kA = decltype(a_mn)::value, kB = decltype(b_mn)::value;
          const uint32_t tx = static_cast<uint32_t>(
              (kA ? S::kABytes : p.a_rows * kStageRowBytes) + S::kBBytes) * CG * S::kOps;
          const int a_at = kA ? am : p.a_off + am, b_at = kB ? bn : p.b_off + bn;
          const int a_k = kA ? p.a_off : 0, b_k = kB ? p.b_off : 0;
          const int az = t.b * p.a_batch, bz = t.b * p.b_batch;
          const int ap = p.a_part, bp = p.b_part;
          int c = t.it0 * kstep;
          for (int i = t.it0; i < t.it1; ++i, c += kstep) {
            if (!mbar_wait_at<false>(empty0 + stage * 8, phase ^ 1, abort_flag, p0.status,
                                     FK_DEV_WAIT_TIMEOUT)) {
              ok = false;
              return;
            }
            const uint32_t sa = smem0 + stage * S::kStageBytes, sb = sa + S::kOps * S::kABytes;
            if (leader) mbar_expect_at(full0 + stage * 8, tx);
            const uint32_t bar = bar0 + stage * 8;
#pragma unroll
            for (int o = 0; o < S::kOps; ++o) {
              if constexpr (kA) {
#pragma unroll
                for (int g = 0; g < S::kARows / 64; ++g)
                  tma_load_3d_cg<CG>(sa + o * S::kABytes + g * 8192, ma, bar, a_at + g * 64, a_k + c, az + o * ap);
              } else {
                tma_load_3d_cg<CG>(sa + o * S::kABytes, ma, bar, c, a_at, az + o * ap);
              }
              if constexpr (kB) {
#pragma unroll
                for (int g = 0; g < S::kBRows / 64; ++g)
                  tma_load_3d_cg<CG>(sb + o * S::kBBytes + g * 8192, mb, bar, b_at + g * 64, b_k + c, bz + o * bp);
              } else {
                tma_load_3d_cg<CG>(sb + o * S::kBBytes, mb, bar, c, b_at, bz + o * bp);
              }
            }
            if (++stage == S::kStages) {
              stage = 0;
              phase ^= 1;
            }
          }
        };
        if constexpr (output(EPI)) {
          // dx: P by rows, centroids by columns; dc: both by columns
          if (p.a_mn) load(std::true_type{}, std::true_type{});
          else load(std::false_type{}, std::true_type{});
        } else {
          load(std::false_type{}, std::false_type{});
        }
      }
      // The last products' commits still arrive on this CTA's barriers, from
      // the pair's other CTA too: stay until they have.
      for (int i = 0; ok && i < S::kStages; ++i) {
        ok = mbar_wait_at<false>(empty0 + stage * 8, phase ^ 1, abort_flag, p0.status, FK_DEV_WAIT_TIMEOUT);
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (lane == 0 && leader) {
      const uint32_t full0 = smem_u32(full), empty0 = smem_u32(empty);
      const uint32_t acc_full0 = smem_u32(acc_full), acc_empty0 = smem_u32(acc_empty);
      const uint32_t smem0 = smem_u32(smem);
      int stage = 0, buf = 0;
      uint32_t phase = 0, aphase = 0;
      Walk<EPI, S::kBM> walk(prm, first, stride);
      bool ok = true;
      for (Tile t; ok && walk.get(t); walk.next()) {
        const Problem& p = prm.p[NP > 1 ? t.q : 0];
        const uint32_t idesc = p.idesc;
        const bool a_mn = output(EPI) && p.a_mn;
        constexpr bool b_mn = output(EPI);
        const uint64_t ad0 = a_mn ? smem_desc_sw128_mn(smem0, 8192, 1024) : smem_desc_sw128(smem0);
        const uint64_t bd0 = b_mn ? smem_desc_sw128_mn(smem0 + S::kOps * S::kABytes, 8192, 1024)
                                  : smem_desc_sw128(smem0 + S::kOps * S::kABytes);
        const uint32_t a_step = (a_mn ? 2048 : 32) >> 4;
        constexpr uint32_t b_step = (b_mn ? 2048 : 32) >> 4;
        int left = t.it1 - t.it0;
        while (ok && left > 0) {
          // one accumulator: a segment (EXACT) or the whole tile
          const int n = EXACT ? min(left, kSegment) : left;
          left -= n;
          if (!mbar_wait_at<true>(acc_empty0 + buf * 8, aphase ^ 1, abort_flag, p0.status,
                                  FK_DEV_WAIT_TIMEOUT)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem + buf * BN;
          for (int i = 0; i < n; ++i) {
            if (!mbar_wait_at<false>(full0 + stage * 8, phase, abort_flag, p0.status,
                                     FK_DEV_WAIT_TIMEOUT)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t at = stage * (S::kStageBytes >> 4);
#pragma unroll
            for (int o = 0; o < (EXACT ? 6 : 1); ++o) {
              uint64_t ad = ad0 + at, bd = bd0 + at;
              if constexpr (EXACT) {
                ad += kPairA[o] * (S::kABytes >> 4);
                bd += kPairB[o] * (S::kBBytes >> 4);
              }
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t accumulate = o > 0 || k > 0 || i > 0;
                if constexpr (integer(EPI)) mma_i8_cg<CG>(d, ad, bd, idesc, accumulate);
                else mma_f16_cg<CG>(d, ad, bd, idesc, accumulate);
                ad += a_step;
                bd += b_step;
              }
            }
            mma_commit_cg<CG>(empty0 + stage * 8);
            if (++stage == S::kStages) {
              stage = 0;
              phase ^= 1;
            }
          }
          if (!ok) break;
          mma_commit_cg<CG>(acc_full0 + buf * 8);
          if (++buf == S::kBufs) {
            buf = 0;
            aphase ^= 1;
          }
        }
      }
      // and so do the epilogues' arrivals on the accumulators' barriers
      for (int i = 0; ok && i < S::kBufs; ++i) {
        ok = mbar_wait_at<true>(acc_empty0 + buf * 8, aphase ^ 1, abort_flag, p0.status, FK_DEV_WAIT_TIMEOUT);
        if (++buf == S::kBufs) {
          buf = 0;
          aphase ^= 1;
        }
      }
    }
  } else if (EPI == kEpiArgmax && warp >= kCtlWarps) {
    if constexpr (EPI == kEpiArgmax)
      argmax_epilogue<CG, BN>(prm, staging, tmem, acc_full, acc_empty, abort_flag, warp - kCtlWarps, lane, rank,
                              first, stride);
  } else if (warp >= kCtlWarps) {
    // ------------------------------------------------------------ epilogue
    const int ew = warp - kCtlWarps;
    const int part = ew >> 2;
    const int quarter = warp & 3;
    constexpr int kCols = BN / S::kParts;  // columns of this warp
    constexpr int kChunks = kCols / 32;
    uint8_t* stg = staging + ew * S::kStaging;
    int buf = 0;
    uint32_t aphase = 0;
    Walk<EPI, S::kBM> walk(prm, first, stride);

    // running state of a row
    float run_m = -INFINITY, run_s = 0.0f;
    int label = -1;
    float xs = 0.0f;
    float fac = 0.0f;
    if constexpr (EPI == kEpiOut) {   // (the same for both problems)
      fac = p0.fscale;
      if (p0.f_num) fac *= *p0.f_num;
      if (p0.f_den) fac /= static_cast<float>(max(*p0.f_den, 1));
    }

    // Once a wait has run out, what this warp still has to write becomes NaN: left
    // as it is, memory that nobody wrote would pass for a loss or a gradient.  (By
    // a factor of each value, and only that of this epilogue: choosing the values
    // cost narrow losses 4 %, all factors the gradients' products 1 %.)
    bool dead = false;
    auto spoil = [&](RowStat& st) {
      if (!dead) return;
      keep_branch();
      const float nan = __uint_as_float(0x7fc00000u);
      if constexpr (output(EPI)) fac = nan;
      else run_s = xs = st.coef = st.at_label = nan;
    };

    // What the epilogue needs from memory besides the accumulator is fetched a
    // tile ahead: its latency would stand between the accumulator and its use.
    Tile t, nt;
    bool more = walk.get(nt);
    RowStat st_next = {0.0f, 0.0f, 0.0f, -1};
    float xs_next = 0.0f;
    auto fetch = [&]() {
      const Problem& p = p0;
      const int64_t row = nt.m * S::kBM + static_cast<int>(rank) * 128 + quarter * 32 + lane;
      if constexpr (EPI == kEpiGrad) {
        st_next = {0.0f, 0.0f, 0.0f, -1};
        if (row < Walk<EPI, S::kBM>::rows_of(p)) {
          const float4 f = *reinterpret_cast<const float4*>(p.stat + nt.b * p.stat_rows + (p.row_map ? p.row_map[p.stat_off + row] : p.stat_off + row));
          st_next = {f.x, f.y, f.z, __float_as_int(f.w)};
        }
      }
      if constexpr (integer(EPI)) xs_next = row < p.M ? p.a_scale[nt.b * p.as_sb + row * p.as_sn] : 0.0f;
    };
    if (more) fetch();
    while (more) {
      t = nt;
      walk.next();
      more = walk.get(nt);
      const Problem& p = prm.p[NP > 1 ? t.q : 0];
      const int row = t.m * S::kBM + static_cast<int>(rank) * 128 + quarter * 32 + lane;
      const int row0 = row - lane;
      const int rows = Walk<EPI, S::kBM>::rows_of(p);
      const bool row_ok = row < rows;
      const int col0 = t.n * BN + part * kCols;
      if constexpr (EPI == kEpiOutRows) {
        fac = p.fscale;
        if (p.f_num) fac *= *p.f_num;
        if (p.f_den) fac /= static_cast<float>(max(*p.f_den, 1));
        if (p.row_factor && row_ok) {
          const int n = p.live_off + row;
          fac *= p.row_factor[t.b * p.stat_rows + (p.row_map ? p.row_map[n] : n)];
        }
      }

      if constexpr (EPI == kEpiLse) {
        if (t.first) {
          run_m = -INFINITY;
          run_s = 0.0f;
          label = -1;
          if (row_ok) {
            const int64_t n = p.row_map ? p.row_map[row] : row;
            const int64_t y = load_label(p.labels, t.b * p.label_sb + n * p.label_sn, p.label_dtype);
            label = y == p.ignore_index || y < 0 || y >= p.N ? -1 : static_cast<int>(y);
          }
        }
      }
      RowStat st = st_next;
      st.coef *= p.p_scale;
      st.at_label *= p.p_scale;
      xs = xs_next;
      if (more) fetch();
      // this lane's columns of every chunk
      float sc[kChunks][4], bi[kChunks][4];
      if constexpr (EPI == kEpiScores) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int64_t col = col0 + c * 32 + (lane & 7) * 4 + i;
            sc[c][i] = col < p.N ? p.b_scale[t.b * p.bs_sb + col * p.bs_sn] : 0.0f;
            bi[c][i] = col < p.N && p.bias ? p.bias[t.b * p.bias_sb + col * p.bias_sn] : 0.0f;
          }
      }

      // four columns of an output row, rounded
      auto emit = [&](const int64_t grow, const int col, const float4 f) {
        const int64_t at = output(EPI) && p.row_map ? p.row_map[p.live_off + grow] : grow;
        const int64_t o = t.b * p.out_sb + at * p.out_sr + col;
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
      };

      // P's entry at the label outweighs the row's others, and what its rounding
      // takes is missing by the same share from all of dx's row; so this lane's row
      // adds it, times the label's centroid, to the first piece's sums.  (Errors of
      // dx, of float32 rounded once, before and now: 32444 x 8192 x 128 float16 2.07,
      // 3.00 and 2.08e-4, 16384 x 32768 x 1024 bfloat16 1.66, 2.40 and 1.66e-3.  It
      // takes 6 of 475 and 10 of 2750 us.)
      float lost = 0.0f;
      const uint16_t* label_row = nullptr;
      if constexpr (EPI == kEpiOutRows) {
        if (p.label_rows && t.chunk == 0 && row_ok) {
          const int n = p.live_off + row;
          const float4 f = *reinterpret_cast<const float4*>(p.stat + t.b * p.stat_rows + (p.row_map ? p.row_map[n] : n));
          const float at_label = f.z * p.p_scale;
          if (__float_as_int(f.w) >= 0) {
            lost = at_label - (p.out_dtype == FK_BF16 ? __uint_as_float(pack_bf16(at_label, 0.0f) << 16)
                                                      : __half2float(__float2half_rn(at_label)));
            label_row = p.label_rows + t.b * p.label_batch + __float_as_int(f.w) * p.label_ld;
          }
        }
      }

      // one chunk of 32 columns, accumulators in v
      auto chunk = [&](const int c, uint32_t (&v)[32]) {
        const int cc = col0 + c * 32;

        if constexpr (EPI == kEpiLse) {
          const int left = p.N - cc;
          if (left < 32) {
            keep_branch();
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i >= left) v[i] = 0xff800000u;  // -inf past the last centroid
          }
          const int rel = label - cc;
          if (rel >= 0 && rel < 32) {
            keep_branch();
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
          const uint64_t co = pack2(st.coef, st.coef);
          float e[32];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            unpack2(mul2(add2(pack2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), nm), s2), e[i], e[i + 1]);
            unpack2(mul2(pack2(ex2(e[i]), ex2(e[i + 1])), co), e[i], e[i + 1]);
          }
          if (rel >= 0 && rel < 32) {
            keep_branch();
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (rel == i) e[i] = st.at_label;
          }
          // rows of this warp in P, four lanes to a row of 64 bytes
          uint8_t* dst = static_cast<uint8_t*>(p.p_out) +
                         2 * (t.b * p.p_batch + (row0 + (lane >> 2)) * p.p_ld + cc + (lane & 3) * 8);
          const int64_t step8 = 16 * p.p_ld;
          const uint32_t wr = smem_u32(stg) + lane * 64, wx = (lane >> 1) & 3;
          const uint32_t rd = smem_u32(stg) + (lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) * 16);
          const bool in = cc < p.p_ld;
          // with gathered rows, zeros up to the next step of the contraction over them
          const int rows_p = p.live ? min(p.M, (rows + 63) & ~63) : rows;
          auto put = [&](auto bf16, const int pp) {
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int k = q * 8 + i * 2;
                w[i] = decltype(bf16)::value ? pack_bf16(e[k], e[k + 1]) : pack_f16(e[k], e[k + 1]);
                if constexpr (EXACT) {  // what this part leaves for the next
                  e[k] -= __uint_as_float(w[i] << 16);
                  e[k + 1] -= __uint_as_float(w[i] & 0xffff0000u);
                }
              }
              sts128(wr + ((q ^ wx) * 16), w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
            uint8_t* d = dst + 2 * pp * p.p_part;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint4 u = lds128(rd + i * 512);
              if (in && row0 + i * 8 + (lane >> 2) < rows_p) *reinterpret_cast<uint4*>(d + i * step8) = u;
            }
          };
          if constexpr (EXACT) {
            for (int pp = 0; pp < 3; ++pp) put(std::true_type{}, pp);
          } else if (p.p_bf16) {
            keep_branch();
            put(std::true_type{}, 0);
          } else {
            keep_branch();
            put(std::false_type{}, 0);
          }
        } else if constexpr (output(EPI) || EPI == kEpiScores) {
          if constexpr (EPI == kEpiScores) acc_to_f(v);
          if constexpr (EPI == kEpiOutRows) {
            if (lost != 0.0f) {
              keep_branch();
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                uint16_t h[8] = {};
                if (cc + q * 8 + 8 <= p.N) {
                  *reinterpret_cast<uint4*>(h) = *reinterpret_cast<const uint4*>(label_row + cc + q * 8);
                } else {
#pragma unroll
                  for (int i = 0; i < 8; ++i)
                    if (cc + q * 8 + i < p.N) h[i] = label_row[cc + q * 8 + i];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const float ci = p.out_dtype == FK_BF16 ? __uint_as_float(static_cast<uint32_t>(h[i]) << 16)
                                                          : __half2float(__ushort_as_half(h[i]));
                  v[q * 8 + i] = __float_as_uint(fmaf(lost, ci, __uint_as_float(v[q * 8 + i])));
                }
              }
            }
          }
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            float4 f;
            float* ff = &f.x;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              ff[i] = __uint_as_float(v[q * 4 + i]) * (EPI == kEpiScores ? xs : fac);
            *reinterpret_cast<float4*>(stg + lane * 128 + ((q ^ (lane & 7)) * 16)) = f;
          }
          __syncwarp();
          const int q = lane & 7;
          const int col = cc + q * 4;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int rr = i * 4 + (lane >> 3);
            const int64_t grow = row0 + rr;
            if (grow >= rows || col >= p.N) continue;
            float4 f = *reinterpret_cast<const float4*>(stg + rr * 128 + ((q ^ (rr & 7)) * 16));
            if constexpr (EPI == kEpiScores) {
              float* ff = &f.x;
#pragma unroll
              for (int k = 0; k < 4; ++k) ff[k] = __fadd_rn(__fmul_rn(ff[k], sc[c][k]), bi[c][k]);
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
            emit(grow, col, f);
          }
        }
      };

      if constexpr (EXACT) {
        float sum[kChunks][32];
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) sum[c][i] = 0.0f;
        for (int it = t.it0; it < t.it1; it += kSegment) {
          dead = dead || !__all_sync(0xffffffffu, mbar_wait(&acc_full[buf], aphase, abort_flag, p0.status,
                                                            FK_DEV_WAIT_TIMEOUT));
          if (dead) break;
          tc_fence_after();
          const uint32_t taddr =
              tmem + buf * BN + part * kCols + (static_cast<uint32_t>(quarter * 32) << 16);
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
          if (++buf == S::kBufs) {
            buf = 0;
            aphase ^= 1;
          }
        }
        spoil(st);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          uint32_t v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(sum[c][i]);
          chunk(c, v);
        }
      } else {
        // no gathered row in this split of them: nothing comes, nothing is added
        const bool none = output(EPI) && t.it0 == t.it1;
        if (!none && !dead &&
            !__all_sync(0xffffffffu, mbar_wait(&acc_full[buf], aphase, abort_flag, p0.status, FK_DEV_WAIT_TIMEOUT)))
          dead = true;
        spoil(st);
        tc_fence_after();
        const uint32_t taddr =
            tmem + buf * BN + part * kCols + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          uint32_t v[32];
          if (none) {
            keep_branch();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0;
          } else {
            tmem_ld32(taddr + c * 32, v);
            tmem_ld_wait(v);
          }
          if (c + 1 == kChunks && !none && !dead) {
            // the accumulator is in registers: hand it back
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cg<CG>(&acc_empty[buf]);
          }
          chunk(c, v);
        }
        if (!none && ++buf == S::kBufs) {
          buf = 0;
          aphase ^= 1;
        }
      }

      if constexpr (output(EPI)) {
        if (p.join) {
          // Partial sums of a split contraction: whichever split's warp arrives
          // last adds all of them up, in the order of the splits, so the result
          // does not depend on which one that is.
          __threadfence();
          __syncwarp();
          const int64_t tile = (static_cast<int64_t>(t.b) * p.m_tiles + t.m) * p.n_tiles + t.n;
          uint32_t* arrived = p.join + (tile * CG + rank) * S::kEpiWarps + ew;
          uint32_t n = 0;
          if (lane == 0) n = atomicAdd(arrived, 1u) + 1;
          n = __shfl_sync(0xffffffffu, n, 0);
          if (n == static_cast<uint32_t>(p.chunks)) {
            __threadfence();
            if (lane == 0) *arrived = 0;
            // eight loads in flight a lane: the sums are a chain of `splits` of them
            constexpr int kQuads = kCols / 4, kRows = 32 / kQuads;
#pragma unroll 1
            for (int r = 0; r < 32; r += 8 * kRows) {
              const int grow = row0 + r + lane / kQuads;
              const int col = col0 + lane % kQuads * 4;
              if (grow >= rows || col >= p.N) continue;
              // rows past the last one load it again: no branch between the loads
              const float* a = p.acc + t.b * p.acc_batch + col;
              int64_t at[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) at[i] = min(grow + i * kRows, rows - 1) * p.acc_ld;
              float4 f[8] = {};
              for (int k = 0; k < p.join_splits; ++k, a += p.acc_split) {
                float4 o[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = __ldcg(reinterpret_cast<const float4*>(a + at[i]));
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  f[i].x += o[i].x;
                  f[i].y += o[i].y;
                  f[i].z += o[i].z;
                  f[i].w += o[i].w;
                }
              }
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (grow + i * kRows < rows) emit(grow + i * kRows, col, f[i]);
            }
          }
        }
      }
      if constexpr (EPI == kEpiLse) {
        if (t.last && row_ok)
          p.partial[((static_cast<int64_t>(t.b) * p.chunks + t.chunk) * S::kParts + part) * p.M + row] =
              make_float2(run_m, run_s);
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
