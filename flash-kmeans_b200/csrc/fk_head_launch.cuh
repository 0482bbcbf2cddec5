// Host side of the cluster head's products: operand maps, tile shapes and
// launches of head_gemm.
#pragma once
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "fk_head_gemm.cuh"

namespace fk {
namespace head {

// One operand: `parts` x `batches` matrices of `rows` rows of `inner` valid
// elements, `ld` elements apart, laid out in part-major order `mat` elements
// apart.  16-bit (FK_F16 / FK_BF16) or FK_I8.
struct Operand {
  const void* p;
  int dtype;
  int64_t inner, rows, ld, mat;
  int64_t mats;        // parts * batches
  int batch_step;      // matrices from one batch to the next (0: shared)
  int part_step;       // matrices from one part to the next
  bool mn;             // the contraction runs over rows
  int64_t off;         // first row / first contraction index
};

struct ShapeChoice {
  int cg, bn;
  bool exact;          // float32 operands in three parts: 256 x 128 or 128 x 64
  int bm() const { return 128 * cg; }
  // microseconds of a step: its bytes at what the L2 gives an SM (78 KB a
  // microsecond with all of them reading), and no less than the issue takes
  double step_us() const { return std::max(0.2, (16.0 + bn / cg / 8.0) * (exact ? 3 : 1) / 78.0); }
};

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// 256 x 256 tiles on CTA pairs once they give half of the 74 pairs a tile; below
// that 128 x 128 tiles, and 128 x 64 ones when even those leave a third of the
// SMs idle.  Losses of bfloat16 rows in us, as pairs / 128 / 64: 1024 x 4096 x
// 1024 19.3 / 21.1 / 28.2, 512 x 4096 x 1024 17.5 / 16.0 / 19.1, 512 x 1000 x 128
// 11.9 / 10.4 / 9.8, 1 x 32768 x 1024 28.2 / 21.1 / 27.3.
inline ShapeChoice choose_shape(int64_t M, int64_t N, int64_t batches, bool exact) {
  const int wide = exact ? 128 : 256;
  if (M > 128 && ceil_div(M, 256) * ceil_div(N, wide) * batches >= 37) return {2, wide, exact};
  if (!exact && ceil_div(M, 128) * ceil_div(N, 128) * batches >= 100) return {1, 128, exact};
  return {1, 64, exact};
}

// Number of equal chunks of `units` for which `slots` workers finish `items`
// items first; every chunk also costs `extra` units.
inline int choose_chunks(int64_t items, int64_t units, int64_t slots, int64_t most, double extra) {
  int best = 1;
  double best_cost = 1e300;
  if (most > units) most = units;
  for (int64_t c = 1; c <= most;) {
    const int64_t per = ceil_div(units, c);
    const double cost =
        static_cast<double>(ceil_div(items * c, slots)) * (per + extra) + (c > 1 ? extra : 0.0);
    if (cost < best_cost * 0.999) {
      best_cost = cost;
      best = static_cast<int>(c);
    }
    if (per == 1) break;
    c = ceil_div(units, per - 1);    // the next count with shorter chunks
  }
  return best;
}

// How `workers` share the tiles of two problems, those of the first (n0 of cost
// c0 >= c1) dealt out in turn: see Params.
struct Fill {
  int all, short_from, more, rest;
  double span;   // cost of the longest worker
};
inline double tile_cost(int64_t steps) { return static_cast<double>(steps) + 3.0; }
inline double tile_cost(const Problem& p) {
  return tile_cost(ceil_div(p.kblocks, p.chunks));
}
inline Fill fill(int64_t n0, double c0, int64_t n1, double c1, int64_t workers) {
  Fill f = {};
  const int64_t ahead = n0 % workers;            // workers with one tile more
  const int64_t behind = workers - ahead;
  int64_t more = ahead ? static_cast<int64_t>(c0 / c1) : 0;
  if (more * behind > n1) more = n1 / behind;
  const int64_t left = n1 - more * behind;
  const int64_t all = more < (ahead ? static_cast<int64_t>(c0 / c1) : 0) ? 0 : left / workers;
  const int64_t rest = left - all * workers;
  f.all = static_cast<int>(all);
  f.short_from = static_cast<int>(ahead);
  f.more = static_cast<int>(more);
  f.rest = static_cast<int>(rest);
  const double base = static_cast<double>(n0 / workers) * c0 + static_cast<double>(all) * c1;
  const double low = base + static_cast<double>(more) * c1;
  f.span = std::max(ahead ? base + c0 + (rest > behind ? c1 : 0.0) : 0.0, low + (rest > 0 ? c1 : 0.0));
  return f;
}

// Launch of a kernel that begins with pdl_wait_then_release().
template <typename... Args>
int launch_plain(const char* what, void (*kern)(Args...), dim3 grid, int threads, cudaStream_t s,
                 std::common_type_t<Args>... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(FK_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
  }
  return FK_OK;
}

int encode_operand(CUtensorMap* map, const Operand& o, uint32_t box_rows);

template <int CG, int BN, int EPI, bool EXACT>
int launch_shape(Params<problems_of(EPI)>& prm, cudaStream_t s) {
  using S = Shape<CG, BN, EPI, EXACT>;
  auto kern = head_gemm<CG, BN, EPI, EXACT>;
  const int dev = current_device();
  if (dev < 0 || dev >= 64) return fail(FK_ERR_CUDA, "bad current device %d", dev);
  static std::atomic<bool> ready[64];
  if (!ready[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return fail(FK_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    ready[dev].store(true, std::memory_order_release);
  }
  const int sms = sm_count_current();
  if (sms <= 0) return fail(FK_ERR_CUDA, "no SM count for device %d", dev);
  const int64_t slots = sms / CG;
  int64_t items = 0, first = 0;
  for (int i = 0; i < prm.count; ++i) {
    const Problem& p = prm.p[i];
    const int64_t n = static_cast<int64_t>(p.batches) * p.chunks * p.m_tiles * (running(EPI) ? 1 : p.n_tiles);
    items += n;
    if (i == 0) first = n;
    if (items >= (1ll << 31) || static_cast<int64_t>(p.n_tiles) * p.chunks >= (1ll << 31) ||
        static_cast<int64_t>(p.kblocks) * p.chunks >= (1ll << 31))
      return fail(FK_ERR_UNSUPPORTED, "head_gemm: %lld tiles exceed 32-bit", static_cast<long long>(items));
  }
  const int64_t workers = items < slots ? items : slots;
  const unsigned grid = static_cast<unsigned>(workers * CG);
  if (prm.count > 1) {
    const Fill f = fill(first, tile_cost(prm.p[0]), items - first, tile_cost(prm.p[1]), workers);
    prm.all = f.all;
    prm.short_from = f.short_from;
    prm.more = f.more;
    prm.rest = f.rest;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = CG;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CG > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, prm);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(FK_ERR_CUDA, "head_gemm launch failed: %s", cudaGetErrorString(e));
  }
  return FK_OK;
}

// The tiles and maps of prm's problem i.  `kdim` elements are contracted; p.M,
// p.N, p.batches, p.chunks and the epilogue's fields are set.
template <int EPI>
int set_problem(Params<problems_of(EPI)>& prm, int i, const Operand& a, const Operand& b, int64_t kdim,
                ShapeChoice sh) {
  Problem& p = prm.p[i];
  const int step = integer(EPI) ? 128 : 64;
  p.m_tiles = static_cast<int>(ceil_div(p.M, sh.bm()));
  p.n_tiles = static_cast<int>(ceil_div(p.N, sh.bn));
  p.kblocks = static_cast<int>(ceil_div(kdim, step));
  p.a_mn = a.mn;
  p.a_batch = a.batch_step;
  p.b_batch = b.batch_step;
  p.a_part = a.part_step;
  p.b_part = b.part_step;
  p.a_off = static_cast<int>(a.off);
  p.b_off = static_cast<int>(b.off);
  // a short A is loaded in a box of its own height: the rows below it hold
  // what the last stage left, and nothing reads their accumulators
  p.a_rows = sh.cg == 1 && p.M < 128 ? static_cast<int>(ceil_div(p.M, 8) * 8) : 128;
  p.group = 8;
  const int64_t tile_bytes = static_cast<int64_t>(sh.bn) * p.kblocks * kStageRowBytes;
  p.window = static_cast<int>(std::max<int64_t>(1, (16 << 20) / tile_bytes));
  if (integer(EPI)) {
    p.idesc = instr_desc_i8(128 * sh.cg, sh.bn);
  } else {
    p.idesc = instr_desc(a.dtype == FK_BF16 ? 1 : 0, 128 * sh.cg, sh.bn) |
              (a.mn ? 1u << 15 : 0u) | (b.mn ? 1u << 16 : 0u);
  }
  const int st = encode_operand(&prm.a[i], a, a.mn ? 64 : p.a_rows);
  if (st != FK_OK) return st;
  return encode_operand(&prm.b[i], b, b.mn ? 64 : sh.bn / sh.cg);
}

template <int EPI>
int launch(Params<problems_of(EPI)>& prm, ShapeChoice sh, cudaStream_t s) {
  if constexpr (!integer(EPI) && EPI != kEpiOutRows) {   // (16-bit operands only)
    if (sh.exact) {
      if (sh.cg == 2) return launch_shape<2, 128, EPI, true>(prm, s);
      return launch_shape<1, 64, EPI, true>(prm, s);
    }
  }
  if constexpr (output(EPI)) {
    if (sh.cg == 2 && sh.bn == 128) return launch_shape<2, 128, EPI, false>(prm, s);
  }
  if (sh.cg == 2) return launch_shape<2, 256, EPI, false>(prm, s);
  if (sh.bn == 128) return launch_shape<1, 128, EPI, false>(prm, s);
  return launch_shape<1, 64, EPI, false>(prm, s);
}

inline int64_t slots_of(ShapeChoice sh) {
  const int sms = sm_count_current();
  return (sms > 0 ? sms : 148) / sh.cg;
}

}  // namespace head
}  // namespace fk
