// C-ABI entry points of the operators around a dictionary that is trained inside a language model (include/flexsae_amd.h): layer
// norm, the lookup of a table's rows by token, distillation from a teacher's top logits.  Argument validation, plans and launches; no
// allocation, no synchronisation, no global state.
#include <hip/hip_runtime.h>
#include <math.h>

#include "distill_kernels.hpp"
#include "layer_norm_kernels.hpp"
#include "lookup_kernels.hpp"

using namespace flexsae;

namespace {

constexpr size_t kAlign = 256;
constexpr int64_t kComputeUnits = 256;
constexpr int64_t kMostRows = int64_t{1} << 32, kMostCols = int64_t{1} << 29;
constexpr int64_t kMostNormCols = int64_t{1} << 27;  // (a grid's threads along an axis: 16 for each column)

bool valid_dtype(int d) { return d == FLEXSAE_F32 || d == FLEXSAE_BF16 || d == FLEXSAE_F16; }
size_t dtype_size(int d) { return d == FLEXSAE_F32 ? 4 : 2; }
bool aligned(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
bool placed(const void *p, int dtype) { return aligned(p, dtype_size(dtype)); }
int64_t ceil_div(int64_t a, int64_t b) { return a / b + (a % b != 0); }
size_t round_up(size_t a) { return (a + kAlign - 1) / kAlign * kAlign; }
int launch_status() { return hipGetLastError() == hipSuccess ? FLEXSAE_OK : FLEXSAE_ERR_LAUNCH; }
hipStream_t as_stream(void *s) { return static_cast<hipStream_t>(s); }

// (rows of the grid are counted in 16 bits: 2^36 blocks and more are refused before)
dim3 grid_of(int64_t blocks) {
  const int64_t x = blocks < kGridRow ? blocks : kGridRow;
  return dim3(static_cast<unsigned>(x), static_cast<unsigned>(ceil_div(blocks, x)));
}
constexpr int64_t kMostBlocks = kGridRow * 32768;

int check_workspace(const void *workspace, size_t have, size_t need) {
  return workspace && aligned(workspace, kAlign) && have >= need ? FLEXSAE_OK : FLEXSAE_ERR_WORKSPACE;
}

// ---- layer norm ----------------------------------------------------------------------------

int check_norm(const flexsae_norm *n) {
  if (!n || n->rows < 0 || n->cols <= 0 || !valid_dtype(n->dtype) || !valid_dtype(n->weight_dtype) || !valid_dtype(n->bias_dtype))
    return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (!(n->eps >= 0.f) || !isfinite(n->eps) || n->x_stride < 0 || n->dy_stride < 0) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (n->rows >= kMostRows || n->cols >= kMostNormCols) return FLEXSAE_ERR_UNSUPPORTED;
  return FLEXSAE_OK;
}

using NormKernel = void (*)(const NormArgs);

// How rows are shared out: kernel, threads of a block, rows that it has at a time.
struct NormPlan {
  NormKernel kernel = nullptr;
  int threads = 0, groups = 0;
  bool held = true;  // false: rows that no block holds
};

template <typename T, int LANES, int UNITS, bool WHOLE = true>
NormPlan norm_shared(bool backward) {
  return {backward ? layer_norm_bwd_kernel<T, LANES, UNITS, WHOLE> : layer_norm_fwd_kernel<T, LANES, UNITS, WHOLE>, kNormThreads,
          kNormThreads / LANES};
}
template <typename T, int UNITS>
NormPlan norm_block(int64_t units, bool backward) {
  return {backward ? layer_norm_bwd_kernel<T, 0, UNITS, true> : layer_norm_fwd_kernel<T, 0, UNITS, true>,
          static_cast<int>(ceil_div(units, kWave * UNITS)) * kWave, 1};
}

template <typename T>
NormPlan norm_plan(int64_t cols, bool backward) {
  constexpr int64_t N = kUnitOf<T>;
  constexpr int kEight = 8 / N, kSixteen = 16 / N;  // units of 8 and 16 elements
  const int64_t units = ceil_div(cols, N);
  if (cols < N) return norm_shared<T, 16, 1, false>(backward);
  if (units <= 16) return norm_shared<T, 16, 1>(backward);
  if (units <= 32) return norm_shared<T, 32, 1>(backward);
  if (units <= 64) return norm_shared<T, 64, 1>(backward);
  if (units <= 64 * kEight) return norm_shared<T, 64, kEight>(backward);
  if (units <= 64 * kSixteen) return norm_shared<T, 64, kSixteen>(backward);
  // Sixteen elements a lane leave fewer wavefronts to join (us of the forward, 65536 x 2304 bf16: 158 with eight, 142 with sixteen);
  // the backward, with the sums of its columns, has the registers for eight while a block's wavefronts hold a row that way (8192 columns
  // of 16-bit numbers; 16384 x 8192 bf16 165 us, 4.9 TB/s).  Beyond that it has sixteen too, and spills 8 registers of a lane, 39 of fp32:
  // 16384 x 12288 bf16 276 us, 4.4 TB/s, 8192 x 16384 206, 3.9; rows that no block holds are read again, 8192 x 16392 326, 2.5.
  if (backward && units <= kNormMostWaves * 64 * kEight) return norm_block<T, kEight>(units, backward);
  if (units <= kNormMostWaves * 64 * kSixteen) return norm_block<T, kSixteen>(units, backward);
  return {backward ? layer_norm_bwd_long_kernel<T> : layer_norm_fwd_long_kernel<T>, 1024, 1, false};
}

NormPlan norm_plan(const flexsae_norm &n, bool backward) {
  return n.dtype == FLEXSAE_F32    ? norm_plan<float>(n.cols, backward)
         : n.dtype == FLEXSAE_BF16 ? norm_plan<bf16_t>(n.cols, backward)
                                   : norm_plan<f16_t>(n.cols, backward);
}

NormArgs norm_args(const flexsae_norm &n) {
  NormArgs a{};
  a.rows = n.rows;
  a.cols = n.cols;
  a.x_stride = n.x_stride;
  a.dy_stride = n.dy_stride;
  a.eps = n.eps;
  a.weight_dtype = n.weight_dtype;
  a.bias_dtype = n.bias_dtype;
  a.per_block = 1;
  return a;
}

// Blocks of the backward pass, each of which leaves a row of partial sums.
int64_t norm_parts(const flexsae_norm &n, const NormPlan &plan) {
  if (!plan.held) return n.rows < 64 ? n.rows : 64;
  const int64_t blocks = ceil_div(n.rows, plan.groups), most = kComputeUnits * (plan.threads < 1024 ? 1024 / plan.threads : 1);
  return blocks < most ? blocks : most;
}

}  // namespace

extern "C" {

int flexsae_layer_norm_fwd(const flexsae_norm *n, const void *x, const void *weight, const void *bias, void *y, float *mean,
                           float *rstd, void *stream) {
  if (const int rc = check_norm(n)) return rc;
  if (n->rows == 0) return FLEXSAE_OK;
  if (!x || !y) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (!placed(x, n->dtype) || !placed(y, n->dtype) || !placed(weight, n->weight_dtype) || !placed(bias, n->bias_dtype) ||
      !aligned(mean, 4) || !aligned(rstd, 4))
    return FLEXSAE_ERR_ALIGNMENT;
  NormArgs a = norm_args(*n);
  a.x = x;
  a.weight = weight;
  a.bias = bias;
  a.y = y;
  a.mean = mean;
  a.rstd = rstd;
  const NormPlan plan = norm_plan(*n, false);
  if (plan.held) {
    // rows of a block one after another, where there are blocks enough for eight rounds of them
    const int64_t rounds = n->rows / (plan.groups * kComputeUnits * (2048 / plan.threads) * 8);
    a.per_block = rounds < 1 ? 1 : rounds > 8 ? 8 : rounds;
  }
  const int64_t blocks = ceil_div(n->rows, plan.groups * a.per_block);
  plan.kernel<<<grid_of(blocks), plan.threads, 0, as_stream(stream)>>>(a);
  return launch_status();
}

size_t flexsae_layer_norm_bwd_workspace_bytes(const flexsae_norm *n) {
  if (check_norm(n)) return 0;
  return round_up(static_cast<size_t>(norm_parts(*n, norm_plan(*n, true))) * 2 * static_cast<size_t>(n->cols) * sizeof(float));
}

int flexsae_layer_norm_bwd(const flexsae_norm *n, const void *x, const void *dy, const void *weight, const float *mean,
                           const float *rstd, void *dx, void *dweight, void *dbias, void *workspace, size_t workspace_bytes,
                           void *stream) {
  if (const int rc = check_norm(n)) return rc;
  if (!dx && !dweight && !dbias) return FLEXSAE_OK;
  if (n->rows > 0 && (!x || !dy || !mean || !rstd)) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (!placed(x, n->dtype) || !placed(dy, n->dtype) || !placed(dx, n->dtype) || !placed(weight, n->weight_dtype) ||
      !placed(dweight, n->weight_dtype) || !placed(dbias, n->bias_dtype) || !aligned(mean, 4) || !aligned(rstd, 4))
    return FLEXSAE_ERR_ALIGNMENT;
  const bool sums = dweight || dbias;
  if (sums && n->rows > 0)
    if (const int rc = check_workspace(workspace, workspace_bytes, flexsae_layer_norm_bwd_workspace_bytes(n))) return rc;
  const hipStream_t s = as_stream(stream);
  const NormPlan plan = norm_plan(*n, true);
  const int64_t parts = norm_parts(*n, plan);
  NormArgs a = norm_args(*n);
  a.x = x;
  a.dy = dy;
  a.weight = weight;
  a.mean = const_cast<float *>(mean);
  a.rstd = const_cast<float *>(rstd);
  a.y = dx;
  a.partial = sums ? static_cast<float *>(workspace) : nullptr;
  if (n->rows > 0) {
    if (plan.held) {
      const size_t lds = sums && plan.groups > 1 ? static_cast<size_t>(plan.groups) * 2 * static_cast<size_t>(n->cols) * sizeof(float) : 0;
      plan.kernel<<<static_cast<unsigned>(parts), plan.threads, lds, s>>>(a);
      if (const int rc = launch_status()) return rc;
    } else {
      if (dx) {
        plan.kernel<<<grid_of(n->rows), plan.threads, 0, s>>>(a);
        if (const int rc = launch_status()) return rc;
      }
      if (sums) {
        const int64_t per = static_cast<int64_t>(kNormThreads) * (n->dtype == FLEXSAE_F32 ? 4 : 8);
        const dim3 grid(static_cast<unsigned>(ceil_div(n->cols, per)), static_cast<unsigned>(parts));
        (n->dtype == FLEXSAE_F32    ? layer_norm_columns_kernel<float>
         : n->dtype == FLEXSAE_BF16 ? layer_norm_columns_kernel<bf16_t>
                                    : layer_norm_columns_kernel<f16_t>)<<<grid, kNormThreads, 0, s>>>(a);
        if (const int rc = launch_status()) return rc;
      }
    }
  }
  if (!sums) return FLEXSAE_OK;
  const dim3 grid(static_cast<unsigned>(ceil_div(n->cols, kWave)), 2);
  layer_norm_finish_kernel<<<grid, 1024, 0, s>>>(a.partial, n->rows > 0 ? parts : 0, n->cols, dweight, n->weight_dtype, dbias,
                                                 n->bias_dtype);
  return launch_status();
}

}  // extern "C"

// ---- lookup --------------------------------------------------------------------------------

namespace {

int check_lookup(const flexsae_lookup *l) {
  if (!l || l->n < 0 || l->vocab <= 0 || l->cols <= 0 || !valid_dtype(l->dtype) || !valid_dtype(l->scale_dtype))
    return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (l->weight_stride < 0 || l->dout_stride < 0 || !isfinite(l->factor)) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (l->n >= kMostRows || l->vocab >= (int64_t{1} << 31) || l->cols >= kMostCols) return FLEXSAE_ERR_UNSUPPORTED;
  return FLEXSAE_OK;
}

constexpr int kLookupRows = 4;          // rows of a group of lanes ...
constexpr int64_t kLookupMany = 8192;  // ... where there are this many blocks without
using LookupKernel = void (*)(const LookupArgs);
struct LookupPlan {
  LookupKernel fwd, fwd_rows, pieces, pieces_dots, bwd, bwd_dots, bwd_rows, bwd_rows_dots, dots;
  int64_t groups, tiles, width;  // of a block, of a row, columns of whole tiles
};

template <typename T, int LANES, int UNITS, bool WHOLE = true>
LookupPlan lookup_shared(int64_t cols) {
  constexpr int64_t kTile = int64_t{LANES} * UNITS * kUnitOf<T>;
  const int64_t tiles = ceil_div(cols, kTile);
  return {lookup_fwd_kernel<T, LANES, UNITS, WHOLE, 1>,
          lookup_fwd_kernel<T, LANES, UNITS, WHOLE, kLookupRows>,
          lookup_pieces_kernel<T, LANES, UNITS, WHOLE, false>,
          lookup_pieces_kernel<T, LANES, UNITS, WHOLE, true>,
          lookup_bwd_kernel<T, LANES, UNITS, WHOLE, false, 1>,
          lookup_bwd_kernel<T, LANES, UNITS, WHOLE, true, 1>,
          lookup_bwd_kernel<T, LANES, UNITS, WHOLE, false, kLookupRows>,
          lookup_bwd_kernel<T, LANES, UNITS, WHOLE, true, kLookupRows>,
          lookup_dots_kernel<T, LANES, UNITS, WHOLE>,
          kLookupThreads / LANES,
          tiles,
          tiles * kTile};
}

template <typename T>
LookupPlan lookup_plan(int64_t cols) {
  const int64_t units = ceil_div(cols, kUnitOf<T>);
  if (cols < kUnitOf<T>) return lookup_shared<T, 16, 1, false>(cols);
  if (units <= 16) return lookup_shared<T, 16, 1>(cols);
  if (units <= 32) return lookup_shared<T, 32, 1>(cols);
  return lookup_shared<T, 64, 1>(cols);
}

LookupPlan lookup_plan(const flexsae_lookup &l) {
  return l.dtype == FLEXSAE_F32    ? lookup_plan<float>(l.cols)
         : l.dtype == FLEXSAE_BF16 ? lookup_plan<bf16_t>(l.cols)
                                   : lookup_plan<f16_t>(l.cols);
}

LookupArgs lookup_args(const flexsae_lookup &l, const LookupPlan &plan, const int64_t *tokens, const void *weight, const void *scale) {
  LookupArgs a{};
  a.tokens = tokens;
  a.weight = weight;
  a.scale = scale;
  a.n = l.n;
  a.vocab = l.vocab;
  a.cols = l.cols;
  a.weight_stride = l.weight_stride;
  a.dout_stride = l.dout_stride;
  a.factor = l.factor;
  a.scale_dtype = l.scale_dtype;
  a.tiles = plan.tiles;
  return a;
}

// (tasks of groups of lanes are counted in 32 bits)
bool too_many(int64_t items, const LookupPlan &plan) { return items >= ((int64_t{1} << 32) - kLookupThreads) / plan.tiles; }
bool many(int64_t items, const LookupPlan &plan) { return items * plan.tiles >= kLookupMany * plan.groups; }
int64_t lookup_blocks(int64_t items, bool rows, const LookupPlan &plan) {
  return ceil_div(ceil_div(items, rows ? kLookupRows : 1) * plan.tiles, plan.groups);
}

// Where the parts of a backward's workspace lie.
struct LookupSpace {
  size_t begin, map, csr, csr_bytes, pieces, dots, bytes;
};
LookupSpace lookup_space(const flexsae_lookup &l, const LookupPlan &plan) {
  LookupSpace s{};
  auto take = [&](size_t bytes) {
    const size_t at = s.bytes;
    s.bytes += round_up(bytes);
    return at;
  };
  const size_t n = static_cast<size_t>(l.n);
  s.begin = take((static_cast<size_t>(l.vocab) + 1) * 4);
  s.map = take(n * 4);
  s.csr_bytes = l.n > 0 ? flexsae_csr_workspace_bytes(l.n, 1, l.vocab) : 0;
  s.csr = take(s.csr_bytes);
  s.pieces = take(l.n > kLookupChunk ? static_cast<size_t>(ceil_div(l.n, kLookupChunk)) * 2 * static_cast<size_t>(plan.width) * 4 : 0);
  s.dots = take(n * static_cast<size_t>(plan.tiles) * 4);
  return s;
}

}  // namespace

extern "C" {

int flexsae_lookup_fwd(const flexsae_lookup *l, const int64_t *tokens, const void *weight, const void *scale, void *out,
                       int *status_flag, void *stream) {
  if (const int rc = check_lookup(l)) return rc;
  if (l->n == 0) return FLEXSAE_OK;
  if (!tokens || !weight || !out) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (!aligned(tokens, 8) || !placed(weight, l->dtype) || !placed(out, l->dtype) || !placed(scale, l->scale_dtype))
    return FLEXSAE_ERR_ALIGNMENT;
  const LookupPlan plan = lookup_plan(*l);
  if (too_many(l->n, plan)) return FLEXSAE_ERR_UNSUPPORTED;
  LookupArgs a = lookup_args(*l, plan, tokens, weight, scale);
  a.out = out;
  a.flag = status_flag;
  const bool rows = many(l->n, plan);
  (rows ? plan.fwd_rows : plan.fwd)<<<grid_of(lookup_blocks(l->n, rows, plan)), kLookupThreads, 0, as_stream(stream)>>>(a);
  return launch_status();
}

size_t flexsae_lookup_bwd_workspace_bytes(const flexsae_lookup *l) {
  if (check_lookup(l)) return 0;
  return lookup_space(*l, lookup_plan(*l)).bytes;
}

int flexsae_lookup_bwd(const flexsae_lookup *l, const int64_t *tokens, const void *weight, const void *scale, const void *dout,
                       void *dweight, void *dscale, void *workspace, size_t workspace_bytes, void *stream) {
  if (const int rc = check_lookup(l)) return rc;
  if (!dweight && !dscale) return FLEXSAE_OK;
  if (l->n > 0 && (!tokens || !dout)) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (dscale && l->n > 0 && (!weight || !scale)) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (!aligned(tokens, 8) || !placed(weight, l->dtype) || !placed(scale, l->scale_dtype) || !placed(dout, l->dtype) ||
      !placed(dweight, l->dtype) || !placed(dscale, l->scale_dtype))
    return FLEXSAE_ERR_ALIGNMENT;
  const LookupPlan plan = lookup_plan(*l);
  if (too_many(l->n, plan) || too_many(l->vocab, plan)) return FLEXSAE_ERR_UNSUPPORTED;
  const LookupSpace space = lookup_space(*l, plan);
  if (const int rc = check_workspace(workspace, workspace_bytes, space.bytes)) return rc;
  const hipStream_t s = as_stream(stream);
  uint8_t *const ws = static_cast<uint8_t *>(workspace);
  LookupArgs a = lookup_args(*l, plan, tokens, weight, scale);
  a.dout = dout;
  a.dots = dscale ? reinterpret_cast<float *>(ws + space.dots) : nullptr;
  a.dscale = dscale;
  a.out = dweight;
  if (dweight) {
    if (l->n > 0) {
      uint32_t *const begin = reinterpret_cast<uint32_t *>(ws + space.begin), *const map = reinterpret_cast<uint32_t *>(ws + space.map);
      if (const int rc = flexsae_csr_build(tokens, l->n, 1, l->vocab, begin, map, ws + space.csr, space.csr_bytes, nullptr, stream)) return rc;
      a.begin = begin;
      a.map = map;
      a.pieces = reinterpret_cast<float *>(ws + space.pieces);
      if (l->n > kLookupChunk) {
        const int64_t stretches = ceil_div(l->n, kLookupChunk);
        (dscale ? plan.pieces_dots : plan.pieces)<<<grid_of(ceil_div(stretches * plan.tiles, plan.groups)), kLookupThreads, 0, s>>>(a);
        if (const int rc = launch_status()) return rc;
      }
    }
    const bool rows = many(l->vocab, plan);
    (rows ? dscale ? plan.bwd_rows_dots : plan.bwd_rows : dscale ? plan.bwd_dots : plan.bwd)<<<
        grid_of(lookup_blocks(l->vocab, rows, plan)), kLookupThreads, 0, s>>>(a);
    if (const int rc = launch_status()) return rc;
  } else if (l->n > 0) {
    plan.dots<<<grid_of(ceil_div(l->n * plan.tiles, plan.groups)), kLookupThreads, 0, s>>>(a);
    if (const int rc = launch_status()) return rc;
  }
  if (!dscale || l->n == 0) return FLEXSAE_OK;
  lookup_dscale_kernel<<<grid_of(ceil_div(l->n, kLookupThreads)), kLookupThreads, 0, s>>>(a);
  return launch_status();
}

}  // extern "C"

// ---- distillation --------------------------------------------------------------------------

namespace {

int check_distill(const flexsae_distill *d) {
  if (!d || d->rows <= 0 || d->vocab <= 0 || d->k <= 0 || d->logits_stride < 0 || !valid_dtype(d->dtype) || !valid_dtype(d->top_dtype))
    return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (!(d->temperature > 0.f) || !isfinite(d->temperature) || !isfinite(kLog2e / d->temperature) ||
      !isfinite(d->temperature * d->temperature))
    return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (d->flags & ~FLEXSAE_DISTILL_BY_ROW) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (d->rows >= (int64_t{1} << 31) || d->vocab >= (int64_t{1} << 31) || d->k >= (int64_t{1} << 31)) return FLEXSAE_ERR_UNSUPPORTED;
  return FLEXSAE_OK;
}

// Parts of a row, so that there are blocks for the whole chip; a part has whole units of 16 bytes and, but for the last, the same size.
struct DistillSplit {
  int splits;
  int64_t part;
};
DistillSplit distill_split(const flexsae_distill &d) {
  constexpr int64_t kBlocks = 2048, kLeast = 4096;
  int64_t splits = ceil_div(kBlocks, d.rows);
  const int64_t most = ceil_div(d.vocab, kLeast);
  if (splits > most) splits = most;
  if (splits > kDistillSplits) splits = kDistillSplits;
  const int64_t part = ceil_div(ceil_div(d.vocab, splits), 8) * 8;
  return {static_cast<int>(ceil_div(d.vocab, part)), part};
}

struct DistillSpace {
  size_t parts, row_loss, bytes;
};
DistillSpace distill_space(const flexsae_distill &d) {
  DistillSpace s{};
  s.parts = 0;
  s.row_loss = round_up(static_cast<size_t>(d.rows) * static_cast<size_t>(distill_split(d).splits) * sizeof(float2));
  s.bytes = s.row_loss + round_up(static_cast<size_t>(d.rows) * sizeof(float));
  return s;
}

int check_tensors(const flexsae_distill *d, const void *logits, const void *top, const int64_t *index, const float *row_weights,
                  const float *stats) {
  if (!logits || !top || !index || !stats) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (!placed(logits, d->dtype) || !placed(top, d->top_dtype) || !aligned(index, 8) || !aligned(row_weights, 4) || !aligned(stats, 16))
    return FLEXSAE_ERR_ALIGNMENT;
  return FLEXSAE_OK;
}

// Slots of a block's table of stored entries: twice the places, to a power of two, up to what leaves two blocks a compute unit.
int distill_slots(int64_t k) {
  int slots = 64;
  while (slots < 2 * kStoredMost && slots < 2 * k) slots *= 2;
  return slots;
}

DistillArgs distill_args(const flexsae_distill &d, const void *logits, const void *top, const int64_t *index, const float *row_weights,
                         float *stats) {
  const DistillSplit split = distill_split(d);
  DistillArgs a{};
  a.logits = logits;
  a.top = top;
  a.index = index;
  a.row_weights = row_weights;
  a.stats = reinterpret_cast<float4 *>(stats);
  a.rows = d.rows;
  a.vocab = d.vocab;
  a.k = d.k;
  a.stride = d.logits_stride;
  a.part = split.part;
  a.splits = split.splits;
  a.slots = distill_slots(d.k);
  a.t = d.temperature;
  a.inv_t = 1.f / d.temperature;
  a.top_dtype = d.top_dtype;
  a.by_row = d.flags & FLEXSAE_DISTILL_BY_ROW;
  return a;
}

using DistillKernel = void (*)(const DistillArgs);
// A row in the registers of a block of so many threads: where it fits there (131072 entries of 16 bits, 65536 of fp32), and each of the
// teacher's places has a thread.  Longer rows take passes of their own for statistics and gradient: us of a mean with its gradient,
// 8192 x 131072 bf16 948, x 131080 1415; 4096 x 65536 fp32 415, x 65544 678.
struct DistillHeld {
  DistillKernel kernel = nullptr;
  int threads = 0;
};
struct DistillKernels {
  DistillKernel parts, rows, grad;
  DistillHeld held;
};
template <typename T>
DistillHeld distill_held(int64_t vocab, int64_t k) {
  const int64_t units = ceil_div(vocab, kUnitOf<T>);
  if (vocab < kUnitOf<T>) return {};
  if (units <= 256 * 4 && k <= 256) return {distill_held_kernel<T, 256, 4>, 256};
  if (units <= 256 * 16 && k <= 256) return {distill_held_kernel<T, 256, 16>, 256};
  if (units <= 512 * 16 && k <= 512) return {distill_held_kernel<T, 512, 16>, 512};
  if (units <= 1024 * 16 && k <= 1024) return {distill_held_kernel<T, 1024, 16>, 1024};
  return {};
}
template <typename T>
DistillKernels distill_kernels_of(const flexsae_distill &d) {
  const DistillKernel grad = d.top_dtype == FLEXSAE_F32    ? distill_grad_kernel<T, float>
                             : d.top_dtype == FLEXSAE_BF16 ? distill_grad_kernel<T, bf16_t>
                                                           : distill_grad_kernel<T, f16_t>;
  return {distill_parts_kernel<T>, distill_rows_kernel<T>, grad, distill_held<T>(d.vocab, d.k)};
}
DistillKernels distill_kernels(const flexsae_distill &d) {
  return d.dtype == FLEXSAE_F32    ? distill_kernels_of<float>(d)
         : d.dtype == FLEXSAE_BF16 ? distill_kernels_of<bf16_t>(d)
                                   : distill_kernels_of<f16_t>(d);
}

}  // namespace

extern "C" {

size_t flexsae_distill_workspace_bytes(const flexsae_distill *d) { return check_distill(d) ? 0 : distill_space(*d).bytes; }

int flexsae_distill_fwd(const flexsae_distill *d, const void *logits, const void *top, const int64_t *index, const float *row_weights,
                        float *loss, float *stats, void *dlogits, void *workspace, size_t workspace_bytes, int *status_flag,
                        void *stream) {
  if (const int rc = check_distill(d)) return rc;
  if (const int rc = check_tensors(d, logits, top, index, row_weights, stats)) return rc;
  if (!loss) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (!aligned(loss, 4) || !placed(dlogits, d->dtype)) return FLEXSAE_ERR_ALIGNMENT;
  const DistillSpace space = distill_space(*d);
  if (const int rc = check_workspace(workspace, workspace_bytes, space.bytes)) return rc;
  DistillArgs a = distill_args(*d, logits, top, index, row_weights, stats);
  if (a.rows > kMostBlocks / a.splits) return FLEXSAE_ERR_UNSUPPORTED;
  uint8_t *const ws = static_cast<uint8_t *>(workspace);
  a.parts = reinterpret_cast<float2 *>(ws + space.parts);
  a.row_loss = a.by_row ? loss : reinterpret_cast<float *>(ws + space.row_loss);
  a.loss = loss;
  a.dlogits = dlogits;
  a.flag = status_flag;
  const hipStream_t s = as_stream(stream);
  const DistillKernels k = distill_kernels(*d);
  const auto finish = [&]() {
    if (a.by_row) return static_cast<int>(FLEXSAE_OK);
    distill_mean_kernel<<<1, 1024, 0, s>>>(a);
    return launch_status();
  };
  if (!a.by_row && row_weights) {
    distill_weights_kernel<<<1, 1024, 0, s>>>(a);
    if (const int rc = launch_status()) return rc;
  }
  if (dlogits && k.held.kernel && (a.rows >= kComputeUnits || k.held.threads == 256)) {
    k.held.kernel<<<grid_of(a.rows), k.held.threads, 0, s>>>(a);
    if (const int rc = launch_status()) return rc;
    return finish();
  }
  k.parts<<<grid_of(a.rows * a.splits), kDistillThreads, 0, s>>>(a);
  if (const int rc = launch_status()) return rc;
  k.rows<<<grid_of(ceil_div(a.rows, kDistillThreads / kWave)), kDistillThreads, 0, s>>>(a);
  if (const int rc = launch_status()) return rc;
  if (dlogits) {
    k.grad<<<grid_of(a.rows * a.splits), kDistillThreads, a.slots * kStoredBytes, s>>>(a);
    if (const int rc = launch_status()) return rc;
  }
  return finish();
}

int flexsae_distill_bwd(const flexsae_distill *d, const void *logits, const void *top, const int64_t *index, const float *row_weights,
                        const float *stats, const float *grad, int skip_if_one, void *dlogits, void *stream) {
  if (const int rc = check_distill(d)) return rc;
  if (const int rc = check_tensors(d, logits, top, index, row_weights, stats)) return rc;
  if (!grad || !dlogits || (skip_if_one && (d->flags & FLEXSAE_DISTILL_BY_ROW))) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (!aligned(grad, 4) || !placed(dlogits, d->dtype)) return FLEXSAE_ERR_ALIGNMENT;
  DistillArgs a = distill_args(*d, logits, top, index, row_weights, const_cast<float *>(stats));
  if (a.rows > kMostBlocks / a.splits) return FLEXSAE_ERR_UNSUPPORTED;
  a.grad = grad;
  a.dlogits = dlogits;
  a.skip_if_one = skip_if_one != 0;
  distill_kernels(*d).grad<<<grid_of(a.rows * a.splits), kDistillThreads, a.slots * kStoredBytes, as_stream(stream)>>>(a);
  return launch_status();
}

}  // extern "C"
