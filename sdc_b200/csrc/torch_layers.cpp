// Torch operators of the layers beside the protected GEMMs (head norm with
// rotation, low-rank adapters, distillation loss): extensions of the
// `sdc_cutlass` library that the reference does not have. As in
// torch_ops.cpp each op validates, allocates its outputs and scratch with the
// caching allocator and enqueues the C ABI on the current CUDA stream. Their
// derivatives are registered here as well: a training step's small layers
// are bound by the host, and a C++ node costs a fraction of a Python one.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <limits>
#include <optional>
#include <tuple>

#include "sdc_b200.h"

namespace {

using at::Tensor;
using OptTensor = const std::optional<Tensor>&;

void check_status(int rc) { TORCH_CHECK(rc == SDC_OK, sdc_last_error()); }
cudaStream_t stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

int element_type(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: TORCH_CHECK(false, what, " must be FP32, BF16 or FP16");
  }
}

void check_cuda(const Tensor& t, const Tensor& like, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.layout() == at::kStrided, what,
              " must be a strided CUDA tensor on the operand device");
}

// Rows of contiguous elements (any row stride).
bool unit_rows(const Tensor& t) { return t.dim() == 0 || t.numel() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1; }
// The tensorwise FP8 projections' outputs, and what is computed from them, are
// column-major: copied to rows before a kernel that streams rows.
Tensor as_rows(const Tensor& t) { return unit_rows(t) ? t : t.contiguous(); }
const void* data_of(OptTensor t) { return t.has_value() ? t->const_data_ptr() : nullptr; }

// ------------------------------------------------- head norm and rotation ----

struct Heads {
  int64_t batch, sequence;
  int heads, dim;
  int64_t strides[3];
};

// [tokens, heads, dim] or [batch, sequence, heads, dim] with a unit last stride.
Heads heads_of(const Tensor& t, const char* what) {
  TORCH_CHECK(t.dim() == 3 || t.dim() == 4, what, " must be [tokens, heads, dim] or [batch, sequence, heads, dim]");
  const bool batched = t.dim() == 4;
  TORCH_CHECK(t.size(-1) <= 512 && t.size(-2) <= std::numeric_limits<int>::max() / 512, what,
              " has too large heads or too many of them");
  Heads h{batched ? t.size(0) : 1, t.size(-3), static_cast<int>(t.size(-2)), static_cast<int>(t.size(-1)), {}};
  h.strides[0] = batched ? t.stride(0) : 0;
  h.strides[1] = t.stride(-3);
  h.strides[2] = t.stride(-2);
  return h;
}

struct RotaryArgs {
  Heads q, k;
  int dtype, weight_f32;
  int64_t position_strides[2];
};

RotaryArgs check_rotary(const Tensor& q, const Tensor& k, const Tensor& table, const Tensor& positions,
                        OptTensor q_weight, OptTensor k_weight) {
  TORCH_CHECK(q.is_cuda() && q.layout() == at::kStrided, "q must be a strided CUDA tensor");
  check_cuda(k, q, "k");
  check_cuda(table, q, "the rotation table");
  check_cuda(positions, q, "positions");
  RotaryArgs a{heads_of(q, "q"), heads_of(k, "k"), element_type(q, "q and k"), 0, {0, 0}};
  TORCH_CHECK(k.scalar_type() == q.scalar_type(), "q and k must have the same dtype");
  TORCH_CHECK(q.dim() == k.dim() && a.q.batch == a.k.batch && a.q.sequence == a.k.sequence && a.q.dim == a.k.dim,
              "q and k must agree in tokens and head dimension");
  TORCH_CHECK(a.q.heads > 0 && a.k.heads > 0, "q and k need at least one head");
  TORCH_CHECK(table.scalar_type() == at::kFloat && table.dim() == 2 && table.is_contiguous() && table.size(0) > 0,
              "the rotation table must be contiguous FP32 [positions, rotary]");
  TORCH_CHECK(table.size(1) <= 512, "rotary dimension must be even and within the head");
  TORCH_CHECK(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong,
              "positions must be int32 or int64");
  const bool batched = q.dim() == 4;
  TORCH_CHECK((positions.dim() == 1 && positions.size(0) == a.q.sequence) ||
                  (batched && positions.dim() == 2 && positions.size(0) == a.q.batch &&
                   positions.size(1) == a.q.sequence),
              "positions must be [tokens], or [sequence] or [batch, sequence] for batched heads");
  a.position_strides[0] = positions.dim() == 2 ? positions.stride(0) : 0;
  a.position_strides[1] = positions.stride(-1);
  TORCH_CHECK(q_weight.has_value() == k_weight.has_value(),
              "head norm weights must be given for both q and k, or for neither");
  if (q_weight.has_value()) {
    for (const Tensor* w : {&*q_weight, &*k_weight}) {
      check_cuda(*w, q, "head norm weights");
      TORCH_CHECK(w->dim() == 1 && w->size(0) == a.q.dim && w->is_contiguous(),
                  "head norm weights must be contiguous [dim]");
      TORCH_CHECK(w->scalar_type() == q_weight->scalar_type() &&
                      (w->scalar_type() == q.scalar_type() || w->scalar_type() == at::kFloat),
                  "head norm weights must both be FP32 or both the heads' dtype");
    }
    a.weight_f32 = q_weight->scalar_type() == at::kFloat;
  }
  return a;
}

std::tuple<Tensor, Tensor> head_norm_rotary(const Tensor& q_in, const Tensor& k_in, const Tensor& table,
                                            const Tensor& positions, OptTensor q_weight, OptTensor k_weight,
                                            double eps, bool interleaved) {
  const Tensor q = as_rows(q_in), k = as_rows(k_in);
  const RotaryArgs a = check_rotary(q, k, table, positions, q_weight, k_weight);
  const c10::cuda::CUDAGuard guard(q.device());
  auto q_out = at::empty(q.sizes(), q.options());
  auto k_out = at::empty(k.sizes(), k.options());
  check_status(sdc_head_norm_rotary(
      a.dtype, q.const_data_ptr(), a.q.strides, k.const_data_ptr(), a.k.strides, a.q.batch, a.q.sequence, a.q.heads,
      a.k.heads, a.q.dim, table.const_data_ptr<float>(), table.size(0), static_cast<int>(table.size(1)), interleaved,
      positions.const_data_ptr(), positions.scalar_type() == at::kLong, a.position_strides, data_of(q_weight),
      data_of(k_weight), a.weight_f32, static_cast<float>(eps), q_out.data_ptr(), k_out.data_ptr(), stream_of(q)));
  return {q_out, k_out};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> head_norm_rotary_backward(
    const Tensor& dq_in, const Tensor& dk_in, const Tensor& q_in, const Tensor& k_in, const Tensor& table,
    const Tensor& positions, OptTensor q_weight, OptTensor k_weight, double eps, bool interleaved) {
  const Tensor q = as_rows(q_in), k = as_rows(k_in), dq_out = as_rows(dq_in), dk_out = as_rows(dk_in);
  const RotaryArgs a = check_rotary(q, k, table, positions, q_weight, k_weight);
  check_cuda(dq_out, q, "gradients");
  check_cuda(dk_out, q, "gradients");
  TORCH_CHECK(dq_out.sizes() == q.sizes() && dk_out.sizes() == k.sizes() && dq_out.scalar_type() == q.scalar_type() &&
                  dk_out.scalar_type() == k.scalar_type(),
              "gradients must have the shapes and dtype of q and k");
  const Heads gq = heads_of(dq_out, "the gradient of q"), gk = heads_of(dk_out, "the gradient of k");
  const c10::cuda::CUDAGuard guard(q.device());
  auto dq = at::empty(q.sizes(), q.options());
  auto dk = at::empty(k.sizes(), k.options());
  Tensor dq_weight, dk_weight, workspace;
  size_t bytes = 0;
  if (q_weight.has_value()) {
    dq_weight = at::empty_like(*q_weight);
    dk_weight = at::empty_like(*k_weight);
    bytes = sdc_head_norm_rotary_workspace_bytes(a.q.batch, a.q.sequence, a.q.heads, a.k.heads, a.q.dim);
    workspace = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
  }
  check_status(sdc_head_norm_rotary_backward(
      a.dtype, dq_out.const_data_ptr(), gq.strides, dk_out.const_data_ptr(), gk.strides, q.const_data_ptr(),
      a.q.strides, k.const_data_ptr(), a.k.strides, a.q.batch, a.q.sequence, a.q.heads, a.k.heads, a.q.dim,
      table.const_data_ptr<float>(), table.size(0), static_cast<int>(table.size(1)), interleaved,
      positions.const_data_ptr(), positions.scalar_type() == at::kLong, a.position_strides, data_of(q_weight),
      data_of(k_weight), a.weight_f32, static_cast<float>(eps), dq.data_ptr(), dk.data_ptr(),
      q_weight.has_value() ? dq_weight.data_ptr() : nullptr, q_weight.has_value() ? dk_weight.data_ptr() : nullptr,
      bytes > 0 ? workspace.data_ptr() : nullptr, bytes, stream_of(q)));
  if (!q_weight.has_value()) {
    dq_weight = at::empty({0}, q.options());
    dk_weight = at::empty({0}, q.options());
  }
  return {dq, dk, dq_weight, dk_weight};
}

// ------------------------------------------------------ low-rank adapters ----

struct AdapterArgs {
  int64_t tokens, k, n, slots, active_tiles, tiles;
  int dtype, adapters, rank, tile_rows;
};

void check_matrix(const Tensor& t, const Tensor& like, int64_t rows, int64_t columns, const char* what) {
  check_cuda(t, like, what);
  TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) == columns, what, " must be [", rows, ", ", columns, "]");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), what, " must have the adapters' dtype");
}

// rows int32 [tokens]: tokens grouped by adapter, those without one last.
// groups int32 [adapters + 1]: slots of each adapter. tiles int32 [n, 3]:
// {slot, count, adapter}; the first `active` of them have an adapter.
AdapterArgs check_adapters(const Tensor& x, const Tensor& a, const Tensor& b, OptTensor scale, const Tensor& rows,
                           const Tensor& groups, const Tensor& tiles, int64_t slots, int64_t active,
                           int64_t tile_rows) {
  TORCH_CHECK(x.is_cuda() && x.layout() == at::kStrided && x.dim() == 2, "adapter input must be a CUDA matrix");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf,
              "low-rank adapters compute BF16 or FP16");
  for (const Tensor* w : {&a, &b}) {
    check_cuda(*w, x, "adapter weights");
    TORCH_CHECK(w->dim() == 3 && w->is_contiguous() && w->scalar_type() == x.scalar_type(),
                "adapter weights must be contiguous [adapters, rank, in] and [adapters, out, rank] of the input's dtype");
  }
  TORCH_CHECK(a.size(0) == b.size(0) && a.size(1) == b.size(2) && a.size(2) == x.size(1),
              "adapter weights must be [adapters, rank, in] and [adapters, out, rank]");
  TORCH_CHECK(a.size(0) >= 1 && a.size(0) <= 65535 && a.size(1) >= 1 && a.size(1) <= 256,
              "low-rank adapters take 1 to 65535 adapters of rank 1 to 256");
  if (scale.has_value()) {
    check_cuda(*scale, x, "adapter scales");
    TORCH_CHECK(scale->scalar_type() == at::kFloat && scale->dim() == 1 && scale->size(0) == a.size(0) &&
                    scale->is_contiguous(),
                "adapter scales must be contiguous FP32 [adapters]");
  }
  for (const Tensor* t : {&rows, &groups, &tiles}) {
    check_cuda(*t, x, "the adapter batch");
    TORCH_CHECK(t->scalar_type() == at::kInt && t->is_contiguous(), "the adapter batch must be contiguous int32");
  }
  TORCH_CHECK(rows.dim() == 1 && rows.size(0) == x.size(0) && groups.dim() == 1 && groups.size(0) == a.size(0) + 1 &&
                  tiles.dim() == 2 && tiles.size(1) == 3,
              "the adapter batch was made for another number of tokens or adapters");
  TORCH_CHECK(slots >= 0 && slots <= x.size(0) && active >= 0 && active <= tiles.size(0) &&
                  (tile_rows == 16 || tile_rows == 128),
              "the adapter batch is inconsistent");
  return {x.size(0), x.size(1), b.size(1), slots, active, tiles.size(0), x.scalar_type() == at::kBFloat16 ? 1 : 2,
          static_cast<int>(a.size(0)), static_cast<int>(a.size(1)), static_cast<int>(tile_rows)};
}

Tensor low_rows(const Tensor& x, const AdapterArgs& s) {
  const int64_t padded = (s.rank + 15) / 16 * 16;
  return at::empty({2, s.slots, padded}, x.options());
}

void run_shrink(const AdapterArgs& s, const Tensor& x, const Tensor& rows, const Tensor& tiles, const Tensor& weight,
                int64_t width, bool rank_minor, OptTensor scale, Tensor& low) {
  check_status(sdc_adapter_shrink(
      s.dtype, x.const_data_ptr(), x.stride(0), s.tokens, rows.const_data_ptr<int32_t>(),
      tiles.const_data_ptr<int32_t>(), s.active_tiles, s.tile_rows, weight.const_data_ptr(), s.adapters, s.rank, width,
      rank_minor, scale.has_value() ? scale->const_data_ptr<float>() : nullptr, low.data_ptr(), s.slots,
      stream_of(x)));
}

void run_expand(const AdapterArgs& s, const void* base, int64_t base_stride, const Tensor& rows, const Tensor& tiles,
                int64_t tile_count, const Tensor& weight, int64_t width, bool rank_minor, const Tensor& low,
                Tensor& out) {
  check_status(sdc_adapter_expand(
      s.dtype, base, base_stride, s.tokens, rows.const_data_ptr<int32_t>(), tiles.const_data_ptr<int32_t>(),
      tile_count, s.tile_rows, weight.const_data_ptr(), s.adapters, s.rank, width, rank_minor, low.const_data_ptr(),
      s.slots, s.active_tiles > 0, out.data_ptr(), out.stride(0), stream_of(out)));
}

// The adapters' sum with base, and the low-rank rows that the backward pass reads.
std::tuple<Tensor, Tensor> low_rank_adapters(const Tensor& base_in, const Tensor& x_in, const Tensor& a,
                                             const Tensor& b, OptTensor scale, const Tensor& rows,
                                             const Tensor& groups, const Tensor& tiles, int64_t slots, int64_t active,
                                             int64_t tile_rows) {
  const AdapterArgs s = check_adapters(x_in, a, b, scale, rows, groups, tiles, slots, active, tile_rows);
  check_matrix(base_in, x_in, s.tokens, s.n, "the projection's output");
  const c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor base = as_rows(base_in), x = as_rows(x_in);
  Tensor low = low_rows(x, s);
  Tensor out = at::empty({s.tokens, s.n}, x.options());
  if (s.tokens == 0 || s.n == 0) return {out, low};
  run_shrink(s, x, rows, tiles, a, s.k, false, scale, low);
  run_expand(s, base.const_data_ptr(), base.stride(0), rows, tiles, s.tiles, b, s.n, true, low, out);
  return {out, low};
}

// The same, added to the projection's output in place: rows without an adapter are not touched.
Tensor low_rank_adapters_(Tensor& base, const Tensor& x_in, const Tensor& a, const Tensor& b, OptTensor scale,
                          const Tensor& rows, const Tensor& groups, const Tensor& tiles, int64_t slots, int64_t active,
                          int64_t tile_rows) {
  const AdapterArgs s = check_adapters(x_in, a, b, scale, rows, groups, tiles, slots, active, tile_rows);
  check_matrix(base, x_in, s.tokens, s.n, "the projection's output");
  at::assert_no_internal_overlap(base);
  const c10::cuda::CUDAGuard guard(x_in.device());
  if (!unit_rows(base)) {
    auto [out, low] = low_rank_adapters(base, x_in, a, b, scale, rows, groups, tiles, slots, active, tile_rows);
    base.copy_(out);
    return low;
  }
  TORCH_CHECK(s.tokens <= 1 || base.stride(0) >= s.n, "the projection's output must not overlap itself");
  const Tensor x = as_rows(x_in);
  Tensor low = low_rows(x, s);
  if (s.tokens == 0 || s.n == 0) return low;
  run_shrink(s, x, rows, tiles, a, s.k, false, scale, low);
  run_expand(s, base.const_data_ptr(), base.stride(0), rows, tiles, s.active_tiles, b, s.n, true, low, base);
  return low;
}

std::tuple<Tensor, Tensor, Tensor> low_rank_adapters_backward(
    const Tensor& grad_in, const Tensor& x_in, const Tensor& a, const Tensor& b, OptTensor scale, const Tensor& low,
    const Tensor& rows, const Tensor& groups, const Tensor& tiles, int64_t slots, int64_t active, int64_t tile_rows,
    bool need_x, bool need_a, bool need_b) {
  const AdapterArgs s = check_adapters(x_in, a, b, scale, rows, groups, tiles, slots, active, tile_rows);
  check_matrix(grad_in, x_in, s.tokens, s.n, "the output's gradient");
  check_cuda(low, x_in, "the low-rank rows");
  const int64_t padded = (s.rank + 15) / 16 * 16;
  TORCH_CHECK(low.scalar_type() == x_in.scalar_type() && low.is_contiguous() && low.dim() == 3 && low.size(0) == 2 &&
                  low.size(1) == s.slots && low.size(2) == padded,
              "the low-rank rows must be those of the forward pass");
  const c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor grad = as_rows(grad_in), x = as_rows(x_in);
  Tensor dx = at::empty({need_x ? s.tokens : 0, s.k}, x.options());
  Tensor da = need_a ? at::empty_like(a) : at::empty({0}, a.options());
  Tensor db = need_b ? at::empty_like(b) : at::empty({0}, b.options());
  if (need_x || need_a) {
    Tensor dlow = low_rows(x, s);
    run_shrink(s, grad, rows, tiles, b, s.n, true, scale, dlow);
    if (need_x && s.tokens > 0) run_expand(s, nullptr, 0, rows, tiles, s.tiles, a, s.k, false, dlow, dx);
    if (need_a) {
      check_status(sdc_adapter_outer(s.dtype, x.const_data_ptr(), x.stride(0), s.tokens,
                                     rows.const_data_ptr<int32_t>(), groups.const_data_ptr<int32_t>(), s.adapters,
                                     dlow.const_data_ptr(), s.slots, s.rank, s.k, 0, da.data_ptr(), stream_of(x)));
    }
  }
  if (need_b) {
    check_status(sdc_adapter_outer(s.dtype, grad.const_data_ptr(), grad.stride(0), s.tokens,
                                   rows.const_data_ptr<int32_t>(), groups.const_data_ptr<int32_t>(), s.adapters,
                                   low.const_data_ptr(), s.slots, s.rank, s.n, 1, db.data_ptr(), stream_of(x)));
  }
  return {dx, da, db};
}

// ----------------------------------------------------------- distillation ----

struct DistillArgs {
  int dtype, teacher_dtype, top;
  int64_t rows, vocab;
};

DistillArgs check_distill(const Tensor& logits, const Tensor& indices, const Tensor& teacher) {
  TORCH_CHECK(logits.is_cuda() && logits.layout() == at::kStrided && logits.dim() == 2,
              "student logits must be a CUDA matrix [rows, vocabulary]");
  TORCH_CHECK(logits.size(1) > 0, "student logits must have a vocabulary");
  check_cuda(indices, logits, "teacher indices");
  check_cuda(teacher, logits, "teacher logits");
  TORCH_CHECK(indices.scalar_type() == at::kInt || indices.scalar_type() == at::kLong,
              "teacher indices must be int32 or int64");
  TORCH_CHECK(indices.dim() == 2 && indices.size(0) == logits.size(0) && indices.size(1) >= 1 &&
                  indices.size(1) <= 1024 && teacher.sizes() == indices.sizes(),
              "teacher indices and logits must be [rows, top] with top from 1 to 1024");
  return {element_type(logits, "student logits"), element_type(teacher, "teacher logits"),
          static_cast<int>(indices.size(1)), logits.size(0), logits.size(1)};
}

std::tuple<Tensor, Tensor> distill_loss(const Tensor& logits_in, const Tensor& indices_in, const Tensor& teacher_in,
                                        double temperature) {
  const DistillArgs a = check_distill(logits_in, indices_in, teacher_in);
  const c10::cuda::CUDAGuard guard(logits_in.device());
  const Tensor logits = as_rows(logits_in), indices = as_rows(indices_in), teacher = as_rows(teacher_in);
  auto loss = at::empty({a.rows}, logits.options().dtype(at::kFloat));
  auto stats = at::empty({a.rows, 4}, loss.options());
  check_status(sdc_distill_loss(a.dtype, logits.const_data_ptr(), a.rows, a.vocab, logits.stride(0),
                                indices.const_data_ptr(), indices.scalar_type() == at::kLong, indices.stride(0),
                                teacher.const_data_ptr(), a.teacher_dtype, teacher.stride(0), a.top,
                                static_cast<float>(temperature), loss.data_ptr<float>(), stats.data_ptr<float>(),
                                stream_of(logits)));
  return {loss, stats};
}

Tensor distill_reduce(const Tensor& loss, const Tensor& stats, bool mean) {
  TORCH_CHECK(loss.is_cuda() && loss.scalar_type() == at::kFloat && loss.dim() == 1 && loss.is_contiguous() &&
                  stats.is_cuda() && stats.device() == loss.device() && stats.scalar_type() == at::kFloat &&
                  stats.dim() == 2 && stats.size(0) == loss.size(0) && stats.size(1) == 4 && stats.is_contiguous(),
              "distillation losses and statistics must be contiguous CUDA FP32 [rows] and [rows, 4]");
  const c10::cuda::CUDAGuard guard(loss.device());
  auto out = at::empty({2}, loss.options());
  check_status(sdc_distill_reduce(loss.const_data_ptr<float>(), stats.const_data_ptr<float>(), loss.size(0), mean,
                                  out.data_ptr<float>(), stream_of(loss)));
  return out;
}

// The upstream gradient: none, one value, or one a row.
int64_t upstream_stride(OptTensor grad_loss, const Tensor& logits) {
  if (!grad_loss.has_value()) return 0;
  check_cuda(*grad_loss, logits, "the loss gradient");
  TORCH_CHECK(grad_loss->scalar_type() == at::kFloat &&
                  (grad_loss->dim() == 0 || (grad_loss->dim() == 1 && grad_loss->size(0) == logits.size(0))),
              "the loss gradient must be an FP32 scalar or [rows]");
  if (grad_loss->dim() == 0 || grad_loss->size(0) <= 1) return 0;
  TORCH_CHECK(grad_loss->stride(0) == 0 || grad_loss->stride(0) == 1, "the loss gradient must be contiguous or expanded");
  return grad_loss->stride(0);
}

Tensor distill_backward(const Tensor& logits_in, const Tensor& indices_in, const Tensor& teacher_in,
                        double temperature, const Tensor& stats, OptTensor grad_loss, OptTensor grad_scale) {
  const DistillArgs a = check_distill(logits_in, indices_in, teacher_in);
  const c10::cuda::CUDAGuard guard(logits_in.device());
  const Tensor logits = as_rows(logits_in), indices = as_rows(indices_in), teacher = as_rows(teacher_in);
  check_cuda(stats, logits, "distillation statistics");
  TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.dim() == 2 && stats.size(0) == a.rows && stats.size(1) == 4 &&
                  stats.is_contiguous(),
              "distillation statistics must be contiguous FP32 [rows, 4]");
  const int64_t stride = upstream_stride(grad_loss, logits);
  if (grad_scale.has_value()) {
    check_cuda(*grad_scale, logits, "the loss scale");
    TORCH_CHECK(grad_scale->scalar_type() == at::kFloat && grad_scale->numel() == 1, "the loss scale must be one FP32 value");
  }
  auto grad = at::empty({a.rows, a.vocab}, logits.options());
  check_status(sdc_distill_backward(
      a.dtype, logits.const_data_ptr(), a.rows, a.vocab, logits.stride(0), indices.const_data_ptr(),
      indices.scalar_type() == at::kLong, indices.stride(0), teacher.const_data_ptr(), a.teacher_dtype,
      teacher.stride(0), a.top, static_cast<float>(temperature), stats.const_data_ptr<float>(),
      static_cast<const float*>(data_of(grad_loss)), stride, static_cast<const float*>(data_of(grad_scale)),
      grad.data_ptr(), a.vocab, stream_of(logits)));
  return grad;
}

Tensor loss_and_grad_into(const Tensor& logits, const Tensor& indices_in, const Tensor& teacher_in, double temperature,
                          OptTensor grad_loss, Tensor& grad) {
  const DistillArgs a = check_distill(logits, indices_in, teacher_in);
  const Tensor indices = as_rows(indices_in), teacher = as_rows(teacher_in);
  const int64_t stride = upstream_stride(grad_loss, logits);
  auto loss = at::empty({a.rows}, logits.options().dtype(at::kFloat));
  auto stats = at::empty({a.rows, 4}, loss.options());
  check_status(sdc_distill_loss_and_grad(
      a.dtype, logits.const_data_ptr(), a.rows, a.vocab, logits.stride(0), indices.const_data_ptr(),
      indices.scalar_type() == at::kLong, indices.stride(0), teacher.const_data_ptr(), a.teacher_dtype,
      teacher.stride(0), a.top, static_cast<float>(temperature), static_cast<const float*>(data_of(grad_loss)), stride,
      loss.data_ptr<float>(), stats.data_ptr<float>(), grad.data_ptr(), grad.stride(0), stream_of(logits)));
  return loss;
}

std::tuple<Tensor, Tensor> distill_loss_and_grad(const Tensor& logits, const Tensor& indices, const Tensor& teacher,
                                                 double temperature, OptTensor grad_loss) {
  check_distill(logits, indices, teacher);
  const c10::cuda::CUDAGuard guard(logits.device());
  auto grad = at::empty({logits.size(0), logits.size(1)}, logits.options());
  auto loss = loss_and_grad_into(as_rows(logits), indices, teacher, temperature, grad_loss, grad);
  return {loss, grad};
}

// The gradient replaces the logits.
Tensor distill_loss_and_grad_(Tensor& logits, const Tensor& indices, const Tensor& teacher, double temperature,
                              OptTensor grad_loss) {
  check_distill(logits, indices, teacher);
  TORCH_CHECK(unit_rows(logits), "student logits must have contiguous rows to be replaced in place");
  TORCH_CHECK(logits.size(0) <= 1 || logits.stride(0) >= logits.size(1), "student logits must not overlap themselves");
  const c10::cuda::CUDAGuard guard(logits.device());
  return loss_and_grad_into(logits, indices, teacher, temperature, grad_loss, logits);
}

// ---------------------------------------------------------------- autograd ----

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

std::optional<Tensor> optional_of(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
Tensor tensor_of(OptTensor t) { return t.has_value() ? *t : Tensor(); }
bool differentiates(OptTensor t) { return t.has_value() && t->requires_grad(); }

// The derivatives here are those of backward passes. A dual tensor's tangent
// would be lost where nothing else asks for a gradient.
template <typename... Tensors>
void refuse_tangents(const Tensors&... inputs) {
  auto dual = [](OptTensor t) { return t.has_value() && t->defined() && t->_fw_grad(0).defined(); };
  TORCH_CHECK_NOT_IMPLEMENTED(!(dual(inputs) || ...), "the layer operators have no forward-mode derivatives");
}

// The backward kernels have no derivatives: a second differentiation raises.
variable_list once_differentiable(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a layer operator that is only once differentiable",
      static_cast<int64_t>(grads.size()));
  variable_list tracked;
  for (Tensor& g : grads) {
    if (g.defined()) g = g.detach().requires_grad_(true);  // an edge for the error to hang on
    tracked.push_back(g);
  }
  return (*error)(std::move(tracked));
}

struct HeadNormRotary : torch::autograd::Function<HeadNormRotary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& table,
                               const Tensor& positions, OptTensor q_weight, OptTensor k_weight, double eps,
                               bool interleaved) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({q, k, table, positions, tensor_of(q_weight), tensor_of(k_weight)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->set_materialize_grads(false);
    auto [q_out, k_out] = head_norm_rotary(q, k, table, positions, q_weight, k_weight, eps, interleaved);
    return {q_out, k_out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(8);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      for (int i = 0; i < 2; ++i) {  // an output that was not used
        grads[i] = grads[i].defined() ? grads[i] : at::zeros(saved[i].sizes(), saved[i].options());
      }
      auto [dq, dk, dq_weight, dk_weight] = head_norm_rotary_backward(
          grads[0], grads[1], saved[0], saved[1], saved[2], saved[3], optional_of(saved[4]), optional_of(saved[5]),
          ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool());
      out[0] = dq;
      out[1] = dk;
      if (saved[4].defined()) {
        out[4] = dq_weight;
        out[5] = dk_weight;
      }
    }
    return once_differentiable(std::move(out));
  }
};

std::tuple<Tensor, Tensor> head_norm_rotary_autograd(const Tensor& q, const Tensor& k, const Tensor& table,
                                                     const Tensor& positions, OptTensor q_weight, OptTensor k_weight,
                                                     double eps, bool interleaved) {
  refuse_tangents(q, k, table, q_weight, k_weight);
  TORCH_CHECK(!(at::GradMode::is_enabled() && table.requires_grad()), "the rotation table is not differentiable");
  if (at::GradMode::is_enabled() &&
      (q.requires_grad() || k.requires_grad() || differentiates(q_weight) || differentiates(k_weight))) {
    variable_list out = HeadNormRotary::apply(q, k, table, positions, q_weight, k_weight, eps, interleaved);
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return head_norm_rotary(q, k, table, positions, q_weight, k_weight, eps, interleaved);
}

// In place (low_out given) base is the only output: autograd takes no other
// beside one that may be a view.
struct LowRankAdapters : torch::autograd::Function<LowRankAdapters> {
  static variable_list forward(AutogradContext* ctx, const Tensor& base, const Tensor& x, const Tensor& a,
                               const Tensor& b, OptTensor scale, const Tensor& rows, const Tensor& groups,
                               const Tensor& tiles, int64_t slots, int64_t active, int64_t tile_rows, Tensor* low_out) {
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor out = base, low;
    if (low_out != nullptr) {
      *low_out = low = low_rank_adapters_(out, x, a, b, scale, rows, groups, tiles, slots, active, tile_rows);
      ctx->mark_dirty({base});
    } else {
      std::tie(out, low) = low_rank_adapters(base, x, a, b, scale, rows, groups, tiles, slots, active, tile_rows);
      ctx->mark_non_differentiable({low});
    }
    ctx->save_for_backward({x, a, b, tensor_of(scale), low, rows, groups, tiles});
    ctx->saved_data["slots"] = slots;
    ctx->saved_data["active"] = active;
    ctx->saved_data["tile_rows"] = tile_rows;
    ctx->set_materialize_grads(false);  // no zeros for `low`
    if (low_out != nullptr) return {out};
    return {out, low};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const bool need_base = ctx->needs_input_grad(0), need_x = ctx->needs_input_grad(1);
    const bool need_a = ctx->needs_input_grad(2), need_b = ctx->needs_input_grad(3);
    variable_list out(12);
    if (!grads[0].defined()) return out;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      auto [dx, da, db] = low_rank_adapters_backward(
          grads[0], saved[0], saved[1], saved[2], optional_of(saved[3]), saved[4], saved[5], saved[6],
          saved[7], ctx->saved_data["slots"].toInt(), ctx->saved_data["active"].toInt(),
          ctx->saved_data["tile_rows"].toInt(), need_x, need_a, need_b);
      if (need_x) out[1] = dx;
      if (need_a) out[2] = da;
      if (need_b) out[3] = db;
    }
    out = once_differentiable(std::move(out));
    if (need_base) out[0] = grads[0];  // the identity differentiates by itself
    return out;
  }
};

bool adapters_differentiate(const Tensor& base, const Tensor& x, const Tensor& a, const Tensor& b, OptTensor scale) {
  refuse_tangents(base, x, a, b, scale);
  if (!at::GradMode::is_enabled()) return false;
  TORCH_CHECK(!differentiates(scale), "adapter scales are not differentiable");
  return base.requires_grad() || x.requires_grad() || a.requires_grad() || b.requires_grad();
}

std::tuple<Tensor, Tensor> low_rank_adapters_autograd(const Tensor& base, const Tensor& x, const Tensor& a,
                                                      const Tensor& b, OptTensor scale, const Tensor& rows,
                                                      const Tensor& groups, const Tensor& tiles, int64_t slots,
                                                      int64_t active, int64_t tile_rows) {
  if (adapters_differentiate(base, x, a, b, scale)) {
    variable_list out = LowRankAdapters::apply(base, x, a, b, scale, rows, groups, tiles, slots, active, tile_rows,
                                               static_cast<Tensor*>(nullptr));
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return low_rank_adapters(base, x, a, b, scale, rows, groups, tiles, slots, active, tile_rows);
}

Tensor low_rank_adapters_autograd_(Tensor& base, const Tensor& x, const Tensor& a, const Tensor& b, OptTensor scale,
                                   const Tensor& rows, const Tensor& groups, const Tensor& tiles, int64_t slots,
                                   int64_t active, int64_t tile_rows) {
  if (adapters_differentiate(base, x, a, b, scale)) {
    torch::autograd::check_inplace(base, true);  // before base is changed
    Tensor low;
    LowRankAdapters::apply(base, x, a, b, scale, rows, groups, tiles, slots, active, tile_rows, &low);
    return low;
  }
  at::AutoDispatchBelowADInplaceOrView below;
  Tensor low = low_rank_adapters_(base, x, a, b, scale, rows, groups, tiles, slots, active, tile_rows);
  if (!base.is_inference()) torch::autograd::impl::bump_version(base);
  return low;
}

// loss: one value a row, or the sum or mean of them.
enum Reduction : int64_t { kNone = 0, kSum = 1, kMean = 2 };

// {loss, statistics, factor of a row's loss in it (undefined: 1)}.
variable_list reduced_loss(const Tensor& logits, const Tensor& indices, const Tensor& teacher, double temperature,
                           int64_t reduction) {
  auto [loss, stats] = distill_loss(logits, indices, teacher, temperature);
  if (reduction == kNone) return {loss, stats, Tensor()};
  const Tensor both = distill_reduce(loss, stats, reduction == kMean);
  return {both[0], stats, both[1]};
}

struct DistillationLoss : torch::autograd::Function<DistillationLoss> {
  static Variable forward(AutogradContext* ctx, const Tensor& logits, const Tensor& indices, const Tensor& teacher,
                          double temperature, int64_t reduction) {
    at::AutoDispatchBelowADInplaceOrView below;
    const variable_list out = reduced_loss(logits, indices, teacher, temperature, reduction);
    ctx->save_for_backward({logits, indices, teacher, out[1], out[2]});
    ctx->saved_data["temperature"] = temperature;
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(5);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      Tensor upstream = grads[0];
      if (upstream.dim() == 1 && upstream.size(0) > 1 && upstream.stride(0) > 1) upstream = upstream.contiguous();
      out[0] = distill_backward(saved[0], saved[1], saved[2], ctx->saved_data["temperature"].toDouble(), saved[3],
                                upstream, optional_of(saved[4]));
    }
    return once_differentiable(std::move(out));
  }
};

Tensor distillation_loss_cuda(const Tensor& logits, const Tensor& indices, const Tensor& teacher, double temperature,
                              int64_t reduction) {
  TORCH_CHECK(reduction >= kNone && reduction <= kMean, "distillation reduction must be 0 (none), 1 (sum) or 2 (mean)");
  return reduced_loss(logits, indices, teacher, temperature, reduction)[0];
}

Tensor distillation_loss_autograd(const Tensor& logits, const Tensor& indices, const Tensor& teacher,
                                  double temperature, int64_t reduction) {
  TORCH_CHECK(reduction >= kNone && reduction <= kMean, "distillation reduction must be 0 (none), 1 (sum) or 2 (mean)");
  refuse_tangents(logits, teacher);
  TORCH_CHECK(!(at::GradMode::is_enabled() && teacher.requires_grad()),
              "distillation is not differentiable in the teacher's logits");
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    return DistillationLoss::apply(logits, indices, teacher, temperature, reduction);
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return distillation_loss_cuda(logits, indices, teacher, temperature, reduction);
}

// Losses and gradients as values, not recorded.
std::tuple<Tensor, Tensor> distill_loss_and_grad_autograd(const Tensor& logits, const Tensor& indices,
                                                          const Tensor& teacher, double temperature,
                                                          OptTensor grad_loss) {
  refuse_tangents(logits, teacher, grad_loss);
  at::AutoDispatchBelowADInplaceOrView below;
  return distill_loss_and_grad(logits, indices, teacher, temperature, grad_loss);
}

// No derivative: the logits become their gradient, which anything that saved them has to notice.
Tensor distill_loss_and_grad_autograd_(Tensor& logits, const Tensor& indices, const Tensor& teacher,
                                       double temperature, OptTensor grad_loss) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && logits.requires_grad()),
              "in-place distillation replaces the logits and is not differentiable");
  refuse_tangents(logits, teacher, grad_loss);
  at::AutoDispatchBelowADInplaceOrView below;
  Tensor loss = distill_loss_and_grad_(logits, indices, teacher, temperature, grad_loss);
  if (!logits.is_inference()) torch::autograd::impl::bump_version(logits);
  return loss;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(sdc_cutlass, lib) {
  lib.def("head_norm_rotary(Tensor q, Tensor k, Tensor table, Tensor positions, Tensor? q_weight, Tensor? k_weight, float eps, bool interleaved) -> (Tensor, Tensor)");
  lib.def("head_norm_rotary_backward(Tensor dq_out, Tensor dk_out, Tensor q, Tensor k, Tensor table, Tensor positions, Tensor? q_weight, Tensor? k_weight, float eps, bool interleaved) -> (Tensor, Tensor, Tensor, Tensor)");
  lib.def("low_rank_adapters(Tensor base, Tensor x, Tensor a, Tensor b, Tensor? scale, Tensor rows, Tensor groups, Tensor tiles, int slots, int active, int tile_rows) -> (Tensor, Tensor)");
  lib.def("low_rank_adapters_(Tensor(a!) base, Tensor x, Tensor a, Tensor b, Tensor? scale, Tensor rows, Tensor groups, Tensor tiles, int slots, int active, int tile_rows) -> Tensor");
  lib.def("low_rank_adapters_backward(Tensor grad, Tensor x, Tensor a, Tensor b, Tensor? scale, Tensor low, Tensor rows, Tensor groups, Tensor tiles, int slots, int active, int tile_rows, bool need_x, bool need_a, bool need_b) -> (Tensor, Tensor, Tensor)");
  lib.def("distillation_loss(Tensor logits, Tensor indices, Tensor teacher, float temperature, int reduction) -> Tensor");
  lib.def("distill_loss(Tensor logits, Tensor indices, Tensor teacher, float temperature) -> (Tensor, Tensor)");
  lib.def("distill_reduce(Tensor loss, Tensor stats, bool mean) -> Tensor");
  lib.def("distill_backward(Tensor logits, Tensor indices, Tensor teacher, float temperature, Tensor stats, Tensor? grad_loss, Tensor? grad_scale) -> Tensor");
  lib.def("distill_loss_and_grad(Tensor logits, Tensor indices, Tensor teacher, float temperature, Tensor? grad_loss) -> (Tensor, Tensor)");
  lib.def("distill_loss_and_grad_(Tensor(a!) logits, Tensor indices, Tensor teacher, float temperature, Tensor? grad_loss) -> Tensor");
}

TORCH_LIBRARY_IMPL(sdc_cutlass, CUDA, lib) {
  lib.impl("head_norm_rotary", &head_norm_rotary);
  lib.impl("head_norm_rotary_backward", &head_norm_rotary_backward);
  lib.impl("low_rank_adapters", &low_rank_adapters);
  lib.impl("low_rank_adapters_", &low_rank_adapters_);
  lib.impl("low_rank_adapters_backward", &low_rank_adapters_backward);
  lib.impl("distillation_loss", &distillation_loss_cuda);
  lib.impl("distill_loss", &distill_loss);
  lib.impl("distill_reduce", &distill_reduce);
  lib.impl("distill_backward", &distill_backward);
  lib.impl("distill_loss_and_grad", &distill_loss_and_grad);
  lib.impl("distill_loss_and_grad_", &distill_loss_and_grad_);
}

TORCH_LIBRARY_IMPL(sdc_cutlass, AutogradCUDA, lib) {
  lib.impl("head_norm_rotary", &head_norm_rotary_autograd);
  lib.impl("low_rank_adapters", &low_rank_adapters_autograd);
  lib.impl("low_rank_adapters_", &low_rank_adapters_autograd_);
  lib.impl("distillation_loss", &distillation_loss_autograd);
  lib.impl("distill_loss_and_grad", &distill_loss_and_grad_autograd);
  lib.impl("distill_loss_and_grad_", &distill_loss_and_grad_autograd_);
}
