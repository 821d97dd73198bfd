// C-ABI entry points of the optimiser (include/flexsae_amd.h): argument validation, tables of tensors and launches.  No
// allocation, no synchronisation, no global state.
#include <hip/hip_runtime.h>
#include <math.h>

#include "adamw_kernels.hpp"

using namespace flexsae;

namespace {

bool valid_dtype(int d) { return d == FLEXSAE_F32 || d == FLEXSAE_BF16 || d == FLEXSAE_F16; }
size_t dtype_size(int d) { return d == FLEXSAE_F32 ? 4 : 2; }
bool aligned(const void *p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
int64_t ceil_div(int64_t a, int64_t b) { return a / b + (a % b != 0); }
int launch_status() { return hipGetLastError() == hipSuccess ? FLEXSAE_OK : FLEXSAE_ERR_LAUNCH; }

constexpr int64_t kMostElements = int64_t{1} << 40;  // of a tensor: tiles are counted in 32 bits

constexpr int64_t kMostTiles = int64_t{1} << 31;  // of a launch
// Large steps with 32-bit states ask for LDS that they do not use, so that two blocks share a compute unit instead of eight: fewer
// places of memory under way at once.  TB/s with two / eight: 20M fp32 parameters 5.70 / 5.65, 40M 5.88 / 5.76, 320M 5.94 / 5.60,
// 320M bf16 ones with masters 5.96 / 5.64.  Steps that have arithmetic to hide lose by it (302M bf16 parameters with 8-bit states:
// 818 / 508 us; rows of 1538 columns 5.10 / 5.31 TB/s).
constexpr int64_t kStreamTiles = 16384;
constexpr size_t kTwoBlocks = 79 << 10;  // of 160 KiB
constexpr int64_t kNormBlocks = 1024;  // each takes one tile after another, and leaves one partial sum

unsigned blocks_for(int64_t tiles, int64_t most) { return static_cast<unsigned>(tiles < 1 ? 1 : tiles > most ? most : tiles); }

int check_tensor(const flexsae_adamw_tensor &t, const flexsae_adamw_config &c) {
  const bool unit = c.flags & FLEXSAE_ADAMW_UNIT_ROWS;
  if (t.rows < 0 || t.cols < 0 || !valid_dtype(t.dtype)) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (!(t.lr >= 0.f) || !(t.weight_decay >= 0.f)) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (t.rows == 0 || t.cols == 0) return FLEXSAE_OK;
  if (t.rows > kMostElements / t.cols || (unit && (t.cols >= (int64_t{1} << 29) || t.rows >= (int64_t{1} << 32)))) return FLEXSAE_ERR_UNSUPPORTED;
  if (!t.param || !t.grad || !t.state0 || !t.state1) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (t.master && t.dtype == FLEXSAE_F32) return FLEXSAE_ERR_INVALID_ARGUMENT;
  const size_t es = dtype_size(t.dtype);
  if (!aligned(t.param, es) || !aligned(t.grad, es) || !aligned(t.master, 4)) return FLEXSAE_ERR_ALIGNMENT;
  if (c.state_bits == 32 ? !aligned(t.state0, 4) || !aligned(t.state1, 4) : !aligned(t.state0, 2) || !aligned(t.state1, 8))
    return FLEXSAE_ERR_ALIGNMENT;
  return FLEXSAE_OK;
}

int check_config(const flexsae_adamw_config *c) {
  if (!c || !c->counter) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (c->state_bits != 32 && c->state_bits != 8) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (!(c->beta1 >= 0. && c->beta1 < 1.) || !(c->beta2 >= 0. && c->beta2 < 1.) || !(c->eps >= 0.)) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (!(c->grad_scale > 0.f) || !isfinite(c->grad_scale) || !isfinite(1.f / c->grad_scale)) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (!(c->max_norm >= 0.f) || (c->max_norm > 0.f && !c->grad_norm)) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (!aligned(c->counter, 8) || !aligned(c->grad_norm, 4) || !aligned(c->lr, 4)) return FLEXSAE_ERR_ALIGNMENT;
  return FLEXSAE_OK;
}

AdamwTable table_of(const flexsae_adamw_config &c) {
  AdamwTable a{};
  a.beta1 = static_cast<float>(c.beta1);
  a.one_minus_beta1 = static_cast<float>(1. - c.beta1);
  a.beta2 = static_cast<float>(c.beta2);
  a.one_minus_beta2 = static_cast<float>(1. - c.beta2);
  a.eps = static_cast<float>(c.eps);
  a.inv_scale = 1.f / c.grad_scale;
  a.max_norm = c.max_norm;
  a.grad_norm = c.grad_norm;
  a.lr = c.lr;
  a.bias = reinterpret_cast<const float2 *>(c.counter + 1);
  return a;
}

using Kernel = void (*)(const AdamwTable);

// How the rows of a tensor are shared out.
struct RowPlan {
  Kernel kernel;
  int threads, rows;  // of a block
};

template <typename T, bool MASTER, bool EIGHT, int WAVES, int UNITS>
RowPlan held_by() {
  return {adamw_rows_kernel<T, MASTER, EIGHT, WAVES, kWave, UNITS>, rows_threads(WAVES), rows_threads(WAVES) / (WAVES * kWave)};
}

// A row goes to as few lanes as hold it in four units each, since what a wavefront does for the row (its sums, its places) is shared
// by what it holds; and to no fewer, since registers then leave too few wavefronts to cover memory and arithmetic with each other.
// us with 1 / 4 / 8 wavefronts a row (40M fp32 elements): 1024 columns, states in 8 bits 116 / 115 / 214, in 32 189 / 198 / 183;
// 2304 columns 214 / 125 / 143 and 204 / 189 / 189; 4096 columns - / 124 / 126 and - / 190 / 187.  Walked three times instead of held,
// from 1.5 times as long (8192 columns, 32 bits 350 / 198) on.
template <typename T, bool MASTER, bool EIGHT>
RowPlan row_plan(int64_t cols) {
  constexpr int N = kUnit<T, MASTER, EIGHT>;
  if (cols <= 16 * N) return {adamw_rows_kernel<T, MASTER, EIGHT, 1, 16, 1>, 256, 16};
  if (cols <= 32 * N) return {adamw_rows_kernel<T, MASTER, EIGHT, 1, 32, 1>, 256, 8};
  switch (ceil_div(cols, 64 * N)) {  // stretches of a wavefront
    case 1: return held_by<T, MASTER, EIGHT, 1, 1>();
    case 2: return held_by<T, MASTER, EIGHT, 1, 2>();
    case 3: return held_by<T, MASTER, EIGHT, 1, 3>();
    case 4: return held_by<T, MASTER, EIGHT, 1, 4>();
    case 5: case 6: case 7: case 8: return held_by<T, MASTER, EIGHT, 4, 2>();
    case 9: case 10: case 11: case 12: return held_by<T, MASTER, EIGHT, 4, 3>();
    case 13: case 14: case 15: case 16: return held_by<T, MASTER, EIGHT, 4, 4>();
    default: break;
  }
  if (cols <= 24 * 64 * N) return held_by<T, MASTER, EIGHT, 8, 3>();
  if (cols <= 32 * 64 * N) return held_by<T, MASTER, EIGHT, 8, 4>();
  if (cols <= 64 * 64 * N) return held_by<T, MASTER, EIGHT, 16, 4>();
  return held_by<T, MASTER, EIGHT, 16, 0>();
}

template <bool EIGHT>
RowPlan row_plan(const flexsae_adamw_tensor &t) {
  if (t.dtype == FLEXSAE_F32) return row_plan<float, false, EIGHT>(t.cols);
  if (t.dtype == FLEXSAE_BF16) return t.master ? row_plan<bf16_t, true, EIGHT>(t.cols) : row_plan<bf16_t, false, EIGHT>(t.cols);
  return t.master ? row_plan<f16_t, true, EIGHT>(t.cols) : row_plan<f16_t, false, EIGHT>(t.cols);
}

// Adds a tensor of `tiles` tiles; false: the table is full.
bool add(AdamwTable &a, const flexsae_adamw_tensor &t, int64_t tiles, bool flat) {
  if (a.count == kAdamwTensors || a.first[a.count] + tiles > kMostTiles) return false;
  a.tensor[a.count] = {t.param, t.grad, t.state0, t.state1, static_cast<float *>(t.master),
                       flat ? sized(t.rows * t.cols, t.dtype) : static_cast<uint64_t>(t.cols) << 32 | static_cast<uint64_t>(t.rows),
                       t.lr, t.weight_decay};
  a.first[a.count + 1] = a.first[a.count] + static_cast<uint32_t>(tiles);
  ++a.count;
  return true;
}

// A tile is a block's work: blocks that loop over the chip-wide grid reach 4.3 TB/s where one after another in memory's order
// they reach 5.7 (302M bf16 parameters with masters), and two or four tiles in a row are slower too (2.1e9 bf16 parameters with
// 8-bit states: 3646 us, 3892, 3946).
int launch(const RowPlan &plan, AdamwTable &a, hipStream_t stream) {
  const int64_t tiles = a.first[a.count];
  if (tiles == 0) return FLEXSAE_OK;
  const size_t lds = plan.kernel == adamw_kernel<false> && tiles > kStreamTiles ? kTwoBlocks : 0;
  const int64_t most = (int64_t{1} << 31) / plan.threads;  // (a grid's threads are counted in 32 bits)
  a.per_block = static_cast<uint32_t>(ceil_div(tiles, most));
  plan.kernel<<<static_cast<unsigned>(ceil_div(tiles, a.per_block)), plan.threads, lds, stream>>>(a);
  a.count = 0;
  return launch_status();
}

// Tiles of the tensor in the kernels' sense.
struct Work {
  RowPlan plan;
  int64_t tiles;
};
Work work_of(const flexsae_adamw_tensor &t, bool eight, bool unit) {
  if (!unit) return {{eight ? adamw_kernel<true> : adamw_kernel<false>, kAdamwThreads, 1}, ceil_div(t.rows * t.cols, kAdamwTile)};
  const RowPlan plan = eight ? row_plan<true>(t) : row_plan<false>(t);
  return {plan, ceil_div(t.rows, plan.rows)};
}

// Partial sums of all gradients: `sums` of them.
template <int TENSORS>
int launch_norms(const flexsae_grad *grads, int64_t count, double *partial, int64_t &sums, hipStream_t stream) {
  NormTable<TENSORS> a;
  a.count = 0;
  a.first[0] = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (grads[i].n > 0) {
      a.tensor[a.count] = {grads[i].grad, sized(grads[i].n, grads[i].dtype)};
      a.first[a.count + 1] = a.first[a.count] + static_cast<uint32_t>(ceil_div(grads[i].n, kNormTile));
      ++a.count;
    }
    if (a.count == 0 || (a.count < TENSORS && i + 1 < count)) continue;
    a.partial = partial + sums;
    const unsigned blocks = blocks_for(a.first[a.count], kNormBlocks);
    norm_partial_kernel<TENSORS><<<blocks, kAdamwThreads, 0, stream>>>(a);
    if (const int rc = launch_status()) return rc;
    sums += blocks;
    a.count = 0;
  }
  return FLEXSAE_OK;
}

}  // namespace

extern "C" {

int flexsae_adamw_check(const flexsae_adamw_tensor *tensors, int64_t count, const flexsae_adamw_config *config) {
  if (const int rc = check_config(config)) return rc;
  if (count < 0 || (count > 0 && !tensors)) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (config->flags & ~FLEXSAE_ADAMW_UNIT_ROWS) return FLEXSAE_ERR_INVALID_ARGUMENT;
  const bool eight = config->state_bits == 8, unit = config->flags & FLEXSAE_ADAMW_UNIT_ROWS;
  for (int64_t i = 0; i < count; ++i) {
    if (const int rc = check_tensor(tensors[i], *config)) return rc;
    if (tensors[i].rows == 0 || tensors[i].cols == 0) continue;
    if (work_of(tensors[i], eight, unit).tiles > kMostTiles) return FLEXSAE_ERR_UNSUPPORTED;
  }
  return FLEXSAE_OK;
}

int flexsae_adamw_step(const flexsae_adamw_tensor *tensors, int64_t count, const flexsae_adamw_config *config, void *stream) {
  if (const int rc = flexsae_adamw_check(tensors, count, config)) return rc;
  const bool eight = config->state_bits == 8, unit = config->flags & FLEXSAE_ADAMW_UNIT_ROWS;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  AdamwTable a = table_of(*config);
  // (of a beta of zero: minus infinity, whose exponential is zero)
  adamw_count_kernel<<<1, 1, 0, s>>>(config->counter, config->grad_norm, log(config->beta1), log(config->beta2));
  if (const int rc = launch_status()) return rc;
  // Tensors that the same kernel takes go into one launch; a table that is full, or another kernel's turn, ends a launch.
  RowPlan plan = {eight ? adamw_kernel<true> : adamw_kernel<false>, kAdamwThreads, 1};
  for (int64_t i = 0; i < count; ++i) {
    const flexsae_adamw_tensor &t = tensors[i];
    if (t.rows == 0 || t.cols == 0) continue;
    const Work w = work_of(t, eight, unit);
    if (a.count > 0 && w.plan.kernel != plan.kernel)
      if (const int rc = launch(plan, a, s)) return rc;
    plan = w.plan;
    if (add(a, t, w.tiles, !unit)) continue;
    if (const int rc = launch(plan, a, s)) return rc;
    (void)add(a, t, w.tiles, !unit);
  }
  return launch(plan, a, s);
}

size_t flexsae_grad_norm_workspace_bytes(int64_t count) {
  if (count < 0) return 0;
  return static_cast<size_t>(ceil_div(count > 0 ? count : 1, kNormTensors)) * kNormBlocks * sizeof(double);
}

int flexsae_grad_norm(const flexsae_grad *grads, int64_t count, float *norm, void *workspace, size_t workspace_bytes, void *stream) {
  if (count < 0 || (count > 0 && !grads) || !norm) return FLEXSAE_ERR_INVALID_ARGUMENT;
  if (!aligned(norm, 4)) return FLEXSAE_ERR_ALIGNMENT;
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < flexsae_grad_norm_workspace_bytes(count)) return FLEXSAE_ERR_WORKSPACE;
  int64_t all = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (grads[i].n < 0 || !valid_dtype(grads[i].dtype)) return FLEXSAE_ERR_INVALID_ARGUMENT;
    if (grads[i].n > kMostElements - all) return FLEXSAE_ERR_UNSUPPORTED;
    all += grads[i].n;
    if (grads[i].n > 0 && !grads[i].grad) return FLEXSAE_ERR_INVALID_ARGUMENT;
    if (!aligned(grads[i].grad, dtype_size(grads[i].dtype))) return FLEXSAE_ERR_ALIGNMENT;
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  double *const partial = static_cast<double *>(workspace);
  int64_t sums = 0;
  const int rc = count <= kNormFew ? launch_norms<kNormFew>(grads, count, partial, sums, s) : launch_norms<kNormTensors>(grads, count, partial, sums, s);
  if (rc) return rc;
  norm_finish_kernel<<<1, kAdamwThreads, 0, s>>>(partial, sums, norm);
  return launch_status();
}

int flexsae_adamw8_moments(const flexsae_adamw8_state *states, int64_t count, int dtype, void *stream) {
  if (count < 0 || (count > 0 && !states) || !valid_dtype(dtype)) return FLEXSAE_ERR_INVALID_ARGUMENT;
  for (int64_t i = 0; i < count; ++i) {
    const flexsae_adamw8_state &t = states[i];
    if (t.rows < 0 || t.cols < 0) return FLEXSAE_ERR_INVALID_ARGUMENT;
    if (t.rows == 0 || t.cols == 0) continue;
    if (t.rows > kMostElements / t.cols) return FLEXSAE_ERR_UNSUPPORTED;
    if (!t.codes || !t.absmax || !t.exp_avg || !t.exp_avg_sq) return FLEXSAE_ERR_INVALID_ARGUMENT;
    if (!aligned(t.codes, 2) || !aligned(t.absmax, 8) || !aligned(t.exp_avg, dtype_size(dtype)) || !aligned(t.exp_avg_sq, dtype_size(dtype)))
      return FLEXSAE_ERR_ALIGNMENT;
  }
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const auto kernel = dtype == FLEXSAE_F32 ? adamw8_moments_kernel<float> : dtype == FLEXSAE_BF16 ? adamw8_moments_kernel<bf16_t>
                                                                                                   : adamw8_moments_kernel<f16_t>;
  MomentsTable a;
  a.count = 0;
  a.first[0] = 0;
  auto launch_moments = [&]() {
    if (a.count == 0) return static_cast<int>(FLEXSAE_OK);
    kernel<<<blocks_for(a.first[a.count], int64_t{1} << 20), kAdamwThreads, 0, s>>>(a);
    a.count = 0;
    return launch_status();
  };
  for (int64_t i = 0; i < count; ++i) {
    const flexsae_adamw8_state &t = states[i];
    if (t.rows == 0 || t.cols == 0) continue;
    const bool flat = t.cols % kAdamwQuant == 0;  // blocks do not ask where rows begin
    const int64_t rows = flat ? 1 : t.rows, cols = flat ? t.rows * t.cols : t.cols;
    const int64_t tiles = ceil_div(rows * cols, kAdamwTile);
    if (a.count == kMomentsTensors || a.first[a.count] + tiles > kMostTiles)
      if (const int rc = launch_moments()) return rc;
    a.tensor[a.count] = {t.codes, t.absmax, t.exp_avg, t.exp_avg_sq, rows, cols};
    a.first[a.count + 1] = a.first[a.count] + static_cast<uint32_t>(tiles);
    ++a.count;
  }
  return launch_moments();
}

}  // extern "C"
