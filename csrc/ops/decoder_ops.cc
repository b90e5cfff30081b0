// torch.ops.nnsx.qk_norm_rope / paged_append / paged_attention / rope_table: the
// operators of a token model's decoder layer (kernels/rope.hip,
// kernels/attn.hip), beside the convolution ops of torch_ops.cc: TorchScript
// models call them from tensor_filter and, qk_norm_rope with its gradient, from
// tensor_trainer.  CPU implementations are the fp32 numerics reference.
//
// The cache is two tensors [pages, kv heads, page size, head dim]; a sequence's
// pages are a row of page_table [sequences, pages of a sequence].  cu_seqlens
// [sequences + 1] says where each sequence's new tokens start among the token
// rows, kv_lens [sequences] how many keys it has with them, so its i-th of n
// new tokens stands at position kv_lens - n + i.  Token rows from
// cu_seqlens[-1] on are padding: their outputs are zero, nothing of them is
// stored.  All three are int32 on the tensors' device and are not copied to the
// host: a captured graph may be replayed after they change.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/TensorIndexing.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include <cmath>
#include <limits>
#include <tuple>

#include "kernels/attn.h"

namespace {

using nnsx::kernels::AttnType;
using OptTensor = c10::optional<at::Tensor>;

hipStream_t cur_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

AttnType type_of(const at::Tensor& t, const char* op) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return AttnType::kBF16;
    case at::kHalf: return AttnType::kF16;
    case at::kFloat: return AttnType::kF32;
    default: break;
  }
  TORCH_CHECK(false, op, ": bfloat16, float16 or float32, got ", t.scalar_type());
}

void check_like(const at::Tensor& t, const at::Tensor& q, const char* op, const char* name) {
  TORCH_CHECK(t.scalar_type() == q.scalar_type(), op, ": ", name, " is ", t.scalar_type(), ", expected ", q.scalar_type());
  TORCH_CHECK(t.device() == q.device(), op, ": ", name, " is on ", t.device(), ", expected ", q.device());
}

void check_ints(const at::Tensor& t, const at::Tensor& q, int64_t n, const char* op, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous() &&
                  t.device() == q.device(),
              op, ": ", name, " is a contiguous int32 tensor [", n, "] on ", q.device(), ", got ", t.scalar_type(), " ",
              t.sizes(), " on ", t.device());
}

void check_head_dim(int64_t d, const char* op) {
  TORCH_CHECK(d > 0 && d <= 256 && d % 8 == 0, op, ": head dim ", d, " (a multiple of 8 up to 256)");
}

// rows of at least `bytes` alignment: the tensor itself, or a packed copy
at::Tensor rows_aligned(const at::Tensor& t, int64_t bytes) {
  const int64_t es = t.element_size();
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) * es % bytes == 0);
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

int64_t row_bytes(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? 16 : 8; }

struct Cache {
  int64_t pages, heads, page, dim;
};

// (a launch counts its threads in 32 bits: up to 512 of them for a token)
constexpr int64_t kMaxTokens = (1 << 23) - 1;

Cache check_cache(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                  const at::Tensor& cu, const at::Tensor& len, const char* op) {
  check_like(k, q, op, "k_cache");
  check_like(v, q, op, "v_cache");
  TORCH_CHECK(k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes(), op,
              ": k_cache and v_cache are both [pages, kv heads, page size, head dim], got ", k.sizes(), " and ", v.sizes());
  const Cache c{k.size(0), k.size(1), k.size(2), k.size(3)};
  TORCH_CHECK(c.heads > 0 && c.page > 0, op, ": the cache has no heads or an empty page");
  check_head_dim(c.dim, op);
  for (const auto* t : {&k, &v}) {
    bool ok = t->stride(3) == 1 && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0;
    for (int64_t i = 0; i < 3; ++i) ok = ok && (t->size(i) <= 1 || t->stride(i) * t->element_size() % 16 == 0);
    TORCH_CHECK(ok, op, ": rows of the cache start at multiples of 16 bytes and are packed, got strides ", t->strides());
    TORCH_CHECK((t->size(0) <= 1 || t->stride(0) * t->element_size() <= (int64_t{1} << 31)) &&
                    (t->size(2) <= 1 || t->stride(2) * t->element_size() <= (int64_t{1} << 28)),
                op, ": pages of the cache are at most 2 GiB apart and rows 256 MiB, got strides ", t->strides());
  }
  TORCH_CHECK(table.scalar_type() == at::kInt && table.dim() == 2 && table.device() == q.device() &&
                  (table.size(1) <= 1 || table.stride(1) == 1),
              op, ": page_table is an int32 tensor [sequences, pages of a sequence] on ", q.device(), ", got ",
              table.scalar_type(), " ", table.sizes(), " on ", table.device());
  check_ints(len, q, table.size(0), op, "kv_lens");
  check_ints(cu, q, table.size(0) + 1, op, "cu_seqlens");
  // (a launch counts its threads in 32 bits: 256 of them for 32 rows, 512 for a sequence)
  TORCH_CHECK(c.pages <= std::numeric_limits<int>::max() && c.page <= (1 << 30) && table.size(1) <= (1 << 30) / c.page &&
                  q.size(0) <= kMaxTokens && q.size(0) * q.size(1) <= (1 << 27) &&
                  (table.size(0) + 1) * c.heads <= (1 << 20),
              op, ": ", q.size(0), " tokens of ", table.size(0), " sequences, tables of ", table.size(1),
              " pages: more than one call takes");
  return c;
}

void fill_batch(nnsx::kernels::PagedBatch* p, const Cache& c, const at::Tensor& table, const at::Tensor& cu,
                const at::Tensor& len, int64_t tokens) {
  p->table = table.data_ptr<int>();
  p->cu = cu.data_ptr<int>();
  p->len = len.data_ptr<int>();
  p->tstride = table.stride(0);
  p->B = static_cast<int>(table.size(0));
  p->T = static_cast<int>(tokens);
  p->width = static_cast<int>(table.size(1));
  p->page = static_cast<int>(c.page);
  p->pages = static_cast<int>(c.pages);
}

// offsets of a CPU batch, checked: they ascend from 0 and stay within the rows
std::vector<int64_t> offsets(const at::Tensor& cu, int64_t tokens, const char* op) {
  const int* p = cu.data_ptr<int>();
  std::vector<int64_t> o(p, p + cu.numel());
  TORCH_CHECK(o[0] == 0, op, ": cu_seqlens starts with 0");
  for (size_t i = 1; i < o.size(); ++i)
    TORCH_CHECK(o[i] >= o[i - 1] && o[i] <= tokens, op, ": cu_seqlens ascends and ends within the token rows");
  return o;
}

// ------------------------------------------------------- paged_attention ----
struct AttnCall {
  Cache c;
  double scale;
};

AttnCall check_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                         const at::Tensor& cu, const at::Tensor& len, c10::optional<double> scale, int64_t window) {
  const char* op = "paged_attention";
  TORCH_CHECK(q.dim() == 3, op, ": q is [tokens, heads, head dim], got ", q.sizes());
  type_of(q, op);
  AttnCall r;
  r.c = check_cache(q, k, v, table, cu, len, op);
  TORCH_CHECK(q.size(2) == r.c.dim && q.size(1) > 0 && q.size(1) % r.c.heads == 0, op, ": q ", q.sizes(),
              " does not fit a cache of ", r.c.heads, " heads of ", r.c.dim);
  r.scale = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(r.c.dim));
  TORCH_CHECK(std::isfinite(r.scale) && r.scale > 0 && std::isnormal(static_cast<float>(r.scale)), op, ": scale ", r.scale,
              " (a positive number)");
  TORCH_CHECK(window >= 0, op, ": window ", window, " (0: none)");
  return r;
}

at::Tensor paged_attention_cuda(const at::Tensor& q0, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                                const at::Tensor& cu, const at::Tensor& len, c10::optional<double> scale, bool causal,
                                int64_t window) {
  const AttnCall call = check_attention(q0, k, v, table, cu, len, scale, window);
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(q0.device());
  at::Tensor out = at::empty(q0.sizes(), q0.options().memory_format(at::MemoryFormat::Contiguous));
  if (out.numel() == 0) return out;
  const at::Tensor q = rows_aligned(q0, 16);
  nnsx::kernels::PagedAttnArgs a;
  fill_batch(&a.p, call.c, table, cu, len, q.size(0));
  a.type = type_of(q, "paged_attention");
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.o = out.data_ptr();
  a.qt = q.stride(0);
  a.qh = q.stride(1);
  a.kp = k.stride(0);
  a.kh = k.stride(1);
  a.kr = k.stride(2);
  a.vp = v.stride(0);
  a.vh = v.stride(1);
  a.vr = v.stride(2);
  a.hq = static_cast<int>(q.size(1));
  a.hkv = static_cast<int>(call.c.heads);
  a.d = static_cast<int>(call.c.dim);
  a.scale = static_cast<float>(call.scale);
  a.causal = causal ? 1 : 0;
  a.window = static_cast<int>(std::min<int64_t>(window, std::numeric_limits<int>::max()));  // (no position is farther)
  at::Tensor ws;
  if (const size_t bytes = nnsx::kernels::paged_attn_workspace_bytes(a)) {
    ws = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
    a.ws = ws.data_ptr();
  }
  nnsx::kernels::paged_attn(a, cur_stream());
  return out;
}

at::Tensor paged_attention_cpu(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                               const at::Tensor& cu, const at::Tensor& len, c10::optional<double> scale, bool causal,
                               int64_t window) {
  const AttnCall call = check_attention(q, k, v, table, cu, len, scale, window);
  const Cache& c = call.c;
  const auto off = offsets(cu, q.size(0), "paged_attention");
  at::Tensor out = at::zeros(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  const int64_t group = q.size(1) / c.heads;
  for (int64_t b = 0; b < table.size(0); ++b) {
    const int64_t n = off[b + 1] - off[b], total = std::max(len.data_ptr<int>()[b], 0);
    const int64_t keys = std::min(total, table.size(1) * c.page);
    if (n == 0 || keys == 0) continue;
    const at::Tensor j = at::arange(keys, table.options().dtype(at::kLong));
    at::Tensor page = table[b].to(at::kLong).index_select(0, at::floor_divide(j, c.page));
    const at::Tensor there = page.ge(0).logical_and(page.lt(c.pages));
    if (!there.any().item<bool>()) continue;
    page = page.masked_fill(there.logical_not(), 0);
    auto rows = [&](const at::Tensor& t) {  // [heads, keys, dim] f32, absent keys zero
      return t.index({page, at::indexing::Slice(), j.remainder(c.page)})
          .to(at::kFloat)
          .masked_fill(there.logical_not().view({-1, 1, 1}), 0)
          .transpose(0, 1)
          .contiguous();
    };
    const at::Tensor kk = rows(k), vv = rows(v);
    const at::Tensor pos = at::arange(total - n, total, j.options()).view({-1, 1});
    at::Tensor sees = there.expand({n, keys});
    if (causal) sees = sees.logical_and(j.le(pos));
    if (window > 0) sees = sees.logical_and(j.gt(pos - window));
    for (int64_t h = 0; h < q.size(1); ++h) {
      at::Tensor s = at::matmul(q.slice(0, off[b], off[b + 1]).select(1, h).to(at::kFloat), kk[h / group].t()) * call.scale;
      s = s.masked_fill(sees.logical_not(), -std::numeric_limits<float>::infinity());
      at::Tensor w = s - std::get<0>(s.max(1, true)).clamp_min(std::numeric_limits<float>::lowest());
      w = w.exp().masked_fill(sees.logical_not(), 0);
      const at::Tensor sum = w.sum(1, true);
      at::Tensor o = at::matmul(w, vv[h / group]);
      // a hidden key's weight 0 times an infinite or NaN value is nothing, not NaN: add such keys one by one
      const at::Tensor bad = vv[h / group].isfinite().all(1).logical_not();
      if (bad.any().item<bool>()) {
        o = at::matmul(w, vv[h / group].masked_fill(bad.view({-1, 1}), 0));
        const at::Tensor idx = bad.nonzero().view({-1});
        for (int64_t i = 0; i < idx.numel(); ++i) {
          const int64_t key = idx[i].item<int64_t>();
          o = at::where(sees.select(1, key).view({-1, 1}), o + w.select(1, key).view({-1, 1}) * vv[h / group][key], o);
        }
      }
      o = at::where(sum.eq(0), at::zeros({}, o.options()), o / sum);
      out.slice(0, off[b], off[b + 1]).select(1, h).copy_(o);
    }
  }
  return out;
}

// ---------------------------------------------------- norm and rotation ----
at::Tensor rope_table(int64_t positions, int64_t dim, double base) {
  TORCH_CHECK(positions >= 0 && dim > 0 && dim % 2 == 0 && std::isfinite(base) && base > 0, "rope_table: ", positions,
              " positions, dim ", dim, " (even), base ", base, " (positive)");
  const auto f64 = at::TensorOptions().dtype(at::kDouble);
  // angles in 64 bits: in 32 a far position times a frequency has no fraction left
  const at::Tensor freq = at::pow(base, at::arange(0, dim, 2, f64) * (-1.0 / static_cast<double>(dim)));
  const at::Tensor angle = at::arange(positions, f64).view({-1, 1}) * freq;
  return at::cat({angle.cos(), angle.sin()}, 1).to(at::kFloat);
}

void check_rope(const at::Tensor& rope, const at::Tensor& q, int64_t dim, const char* op) {
  TORCH_CHECK(rope.scalar_type() == at::kFloat && rope.dim() == 2 && rope.device() == q.device(), op,
              ": rope is a float32 table [positions, rotated columns] on ", q.device(), ", got ", rope.scalar_type(), " ",
              rope.sizes(), " on ", rope.device());
  TORCH_CHECK(rope.size(1) > 0 && rope.size(1) % 8 == 0 && rope.size(1) <= dim, op, ": ", rope.size(1),
              " rotated columns (a multiple of 8 up to the head dim ", dim, ")");
  TORCH_CHECK(rope.size(0) <= std::numeric_limits<int>::max(), op, ": too many positions");
}

void check_weight(const OptTensor& w, const at::Tensor& q, int64_t dim, const char* op, const char* name) {
  if (!given(w)) return;
  TORCH_CHECK((w->scalar_type() == q.scalar_type() || w->scalar_type() == at::kFloat) && w->dim() == 1 &&
                  w->size(0) == dim && w->device() == q.device(),
              op, ": ", name, " is [", dim, "] of the rows' type or float32 on ", q.device(), ", got ", w->scalar_type(), " ",
              w->sizes(), " on ", w->device());
}

void check_weights(const OptTensor& qw, const OptTensor& kw, const at::Tensor& q, int64_t dim, const char* op) {
  check_weight(qw, q, dim, op, "q_weight");
  check_weight(kw, q, dim, op, "k_weight");
  TORCH_CHECK(!given(qw) || !given(kw) || qw->scalar_type() == kw->scalar_type(), op,
              ": q_weight and k_weight have one type, got ", qw->scalar_type(), " and ", kw->scalar_type());
}

void check_eps(double eps, const char* op) {
  TORCH_CHECK(std::isfinite(eps) && eps >= 0, op, ": eps ", eps, " (not negative)");
}

// [tokens, heads, dim] or [batch, tokens, heads, dim], positions [tokens] or [batch, tokens]
void check_norm(const at::Tensor& q, const at::Tensor& k, const OptTensor& qw, const OptTensor& kw, const at::Tensor& pos,
                const at::Tensor& rope, double eps, const char* op) {
  type_of(q, op);
  check_like(k, q, op, "k");
  TORCH_CHECK((q.dim() == 3 || q.dim() == 4) && k.dim() == q.dim(), op,
              ": q and k are both [tokens, heads, head dim] or [batch, tokens, heads, head dim], got ", q.sizes(), " and ",
              k.sizes());
  const int64_t n = q.dim();
  bool same = q.size(n - 1) == k.size(n - 1);
  for (int64_t i = 0; i < n - 2; ++i) same = same && q.size(i) == k.size(i);
  TORCH_CHECK(same && q.size(n - 2) > 0 && k.size(n - 2) > 0, op, ": q ", q.sizes(), " and k ", k.sizes(),
              " differ in more than their heads, or have none");
  check_head_dim(q.size(n - 1), op);
  check_weights(qw, kw, q, q.size(n - 1), op);
  check_rope(rope, q, q.size(n - 1), op);
  check_eps(eps, op);
  TORCH_CHECK((pos.scalar_type() == at::kInt || pos.scalar_type() == at::kLong) && pos.device() == q.device(), op,
              ": positions are int32 or int64 on ", q.device(), ", got ", pos.scalar_type(), " on ", pos.device());
  const bool fits = (pos.dim() == 1 && pos.size(0) == q.size(n - 3)) ||
                    (n == 4 && pos.dim() == 2 && pos.size(0) == q.size(0) && pos.size(1) == q.size(1));
  TORCH_CHECK(fits, op, ": positions ", pos.sizes(), " do not fit q ", q.sizes());
  TORCH_CHECK(q.numel() / (q.size(n - 1) * q.size(n - 2)) <= kMaxTokens && q.size(n - 2) + k.size(n - 2) <= 65535, op,
              ": more tokens or heads than one call takes, got q ", q.sizes(), " and k ", k.sizes());
}

void fill_rows(nnsx::kernels::RopeRows* r, const at::Tensor& x) {
  r->x = x.data_ptr();
  r->sb = x.dim() == 4 ? x.stride(0) : 0;
  r->ss = x.stride(x.dim() - 3);
  r->sh = x.stride(x.dim() - 2);
  r->heads = static_cast<int>(x.size(x.dim() - 2));
}

void fill_grad(nnsx::kernels::RopeRows* r, const at::Tensor& g) {
  r->g = g.data_ptr();
  r->gb = g.dim() == 4 ? g.stride(0) : 0;
  r->gs = g.stride(g.dim() - 3);
  r->gh = g.stride(g.dim() - 2);
}

// the weights' storage must outlive the launch call: packed copies go to `keep`
void fill_weights(nnsx::kernels::RopeArgs* a, const OptTensor& qw, const OptTensor& kw, std::vector<at::Tensor>* keep) {
  auto one = [&](const OptTensor& w) -> const void* {
    if (!given(w)) return nullptr;
    a->w_f32 = w->scalar_type() == at::kFloat ? 1 : 0;
    keep->push_back(rows_aligned(*w, 16));
    return keep->back().data_ptr();
  };
  a->q.w = one(qw);
  a->k.w = one(kw);
}

void fill_norm(nnsx::kernels::RopeArgs* a, const at::Tensor& q, const at::Tensor& k, const OptTensor& qw,
               const OptTensor& kw, const at::Tensor& pos, const at::Tensor& rope, double eps, bool interleaved,
               std::vector<at::Tensor>* keep) {
  a->type = type_of(q, "qk_norm_rope");
  fill_rows(&a->q, q);
  fill_rows(&a->k, k);
  fill_weights(a, qw, kw, keep);
  a->B = q.dim() == 4 ? static_cast<int>(q.size(0)) : 1;
  a->S = static_cast<int>(q.size(q.dim() - 3));
  a->d = static_cast<int>(q.size(q.dim() - 1));
  a->rot = static_cast<int>(rope.size(1));
  a->interleaved = interleaved ? 1 : 0;
  a->norm = 1;
  a->eps = static_cast<float>(eps);
  keep->push_back(rows_aligned(rope, 16));
  a->rope = keep->back().data_ptr<float>();
  a->rstride = keep->back().stride(0);
  a->positions = static_cast<int>(rope.size(0));
  a->pos = pos.data_ptr();
  a->pos64 = pos.scalar_type() == at::kLong ? 1 : 0;
  a->pb = pos.dim() == 2 ? pos.stride(0) : 0;
  a->ps = pos.stride(pos.dim() - 1);
}

at::Tensor packed_like(const at::Tensor& t) {
  return at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous));
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope_cuda(const at::Tensor& q0, const at::Tensor& k0, const OptTensor& qw,
                                                     const OptTensor& kw, const at::Tensor& pos, const at::Tensor& rope,
                                                     double eps, bool interleaved) {
  check_norm(q0, k0, qw, kw, pos, rope, eps, "qk_norm_rope");
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(q0.device());
  at::Tensor yq = packed_like(q0), yk = packed_like(k0);
  if (yq.numel() == 0) return {yq, yk};
  const at::Tensor q = rows_aligned(q0, row_bytes(q0)), k = rows_aligned(k0, row_bytes(k0));
  nnsx::kernels::RopeArgs a;
  std::vector<at::Tensor> keep;
  fill_norm(&a, q, k, qw, kw, pos, rope, eps, interleaved, &keep);
  a.q.y = yq.data_ptr();
  a.k.y = yk.data_ptr();
  nnsx::kernels::qk_norm_rope(a, cur_stream());
  return {yq, yk};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_norm_rope_backward_cuda(
    const at::Tensor& gq0, const at::Tensor& gk0, const at::Tensor& q0, const at::Tensor& k0, const OptTensor& qw,
    const OptTensor& kw, const at::Tensor& pos, const at::Tensor& rope, double eps, bool interleaved) {
  const char* op = "qk_norm_rope_backward";
  check_norm(q0, k0, qw, kw, pos, rope, eps, op);
  check_like(gq0, q0, op, "grad_q");
  check_like(gk0, q0, op, "grad_k");
  TORCH_CHECK(gq0.sizes() == q0.sizes() && gk0.sizes() == k0.sizes(), op, ": gradients have their outputs' sizes");
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(q0.device());
  at::Tensor dq = packed_like(q0), dk = packed_like(k0);
  const auto f32 = q0.options().dtype(at::kFloat);
  auto like_weight = [&](const OptTensor& w) {
    return given(w) ? at::empty({w->size(0)}, f32.dtype(w->scalar_type())) : at::empty({0}, f32);
  };
  at::Tensor dwq = like_weight(qw), dwk = like_weight(kw);
  if (dq.numel() == 0) return {dq, dk, dwq.zero_(), dwk.zero_()};
  const at::Tensor q = rows_aligned(q0, row_bytes(q0)), k = rows_aligned(k0, row_bytes(k0));
  const at::Tensor gq = rows_aligned(gq0, row_bytes(q0)), gk = rows_aligned(gk0, row_bytes(k0));
  nnsx::kernels::RopeArgs a;
  std::vector<at::Tensor> keep;
  fill_norm(&a, q, k, qw, kw, pos, rope, eps, interleaved, &keep);
  fill_grad(&a.q, gq);
  fill_grad(&a.k, gk);
  a.q.y = dq.data_ptr();
  a.k.y = dk.data_ptr();
  at::Tensor ws;
  if (given(qw) || given(kw)) {
    ws = at::empty({static_cast<int64_t>(nnsx::kernels::qk_norm_rope_backward_workspace_bytes(a) / sizeof(float))}, f32);
    a.ws = ws.data_ptr<float>();
    a.dwq = given(qw) ? dwq.data_ptr() : nullptr;
    a.dwk = given(kw) ? dwk.data_ptr() : nullptr;
  }
  nnsx::kernels::qk_norm_rope_backward(a, cur_stream());
  return {dq, dk, dwq, dwk};
}

// cosines and sines [.., 1, rot / 2] of the tokens, and which rows the table holds
struct Angles {
  at::Tensor cos, sin, there;
};

Angles angles(const at::Tensor& pos, const at::Tensor& rope) {
  Angles a;
  at::Tensor p = pos.to(at::kLong);
  a.there = p.ge(0).logical_and(p.lt(rope.size(0)));
  p = p.masked_fill(a.there.logical_not(), 0);
  auto sizes = p.sizes().vec();
  sizes.push_back(rope.size(1));
  const at::Tensor rows = rope.size(0) ? rope.index({p}) : at::zeros(sizes, rope.options());
  a.cos = rows.slice(-1, 0, rope.size(1) / 2).unsqueeze(-2);
  a.sin = rows.slice(-1, rope.size(1) / 2).unsqueeze(-2);
  a.there = a.there.unsqueeze(-1).unsqueeze(-1);
  return a;
}

at::Tensor turned(const at::Tensor& x, const Angles& a, bool interleaved, double sign) {
  const int64_t half = a.cos.size(-1), d = x.size(-1);
  const at::Tensor sin = a.sin * sign;
  const at::Tensor rest = x.slice(-1, 2 * half, d);
  if (interleaved) {
    const at::Tensor u = x.slice(-1, 0, 2 * half, 2), w = x.slice(-1, 1, 2 * half, 2);
    return at::cat({at::stack({u * a.cos - w * sin, w * a.cos + u * sin}, -1).flatten(-2), rest}, -1);
  }
  const at::Tensor u = x.slice(-1, 0, half), w = x.slice(-1, half, 2 * half);
  return at::cat({u * a.cos - w * sin, w * a.cos + u * sin, rest}, -1);
}

at::Tensor normed(const at::Tensor& x, const OptTensor& w, double eps) {
  const at::Tensor y = x * at::rsqrt((x * x).mean(-1, true) + eps);
  return given(w) ? y * w->to(at::kFloat) : y;
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope_cpu(const at::Tensor& q, const at::Tensor& k, const OptTensor& qw,
                                                    const OptTensor& kw, const at::Tensor& pos, const at::Tensor& rope,
                                                    double eps, bool interleaved) {
  check_norm(q, k, qw, kw, pos, rope, eps, "qk_norm_rope");
  const Angles a = angles(pos, rope);
  auto one = [&](const at::Tensor& x, const OptTensor& w) {
    return turned(normed(x.to(at::kFloat), w, eps), a, interleaved, 1.0)
        .masked_fill(a.there.logical_not(), 0)
        .to(x.scalar_type())
        .contiguous();
  };
  return {one(q, qw), one(k, kw)};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_norm_rope_backward_cpu(
    const at::Tensor& gq, const at::Tensor& gk, const at::Tensor& q, const at::Tensor& k, const OptTensor& qw,
    const OptTensor& kw, const at::Tensor& pos, const at::Tensor& rope, double eps, bool interleaved) {
  const char* op = "qk_norm_rope_backward";
  check_norm(q, k, qw, kw, pos, rope, eps, op);
  check_like(gq, q, op, "grad_q");
  check_like(gk, q, op, "grad_k");
  TORCH_CHECK(gq.sizes() == q.sizes() && gk.sizes() == k.sizes(), op, ": gradients have their outputs' sizes");
  const Angles a = angles(pos, rope);
  auto one = [&](const at::Tensor& x0, const at::Tensor& g0, const OptTensor& w) {
    const at::Tensor x = x0.to(at::kFloat);
    at::Tensor g = turned(g0.to(at::kFloat), a, interleaved, -1.0);
    const at::Tensor inv = at::rsqrt((x * x).mean(-1, true) + eps);
    at::Tensor dw = at::empty({0}, x.options());
    if (given(w)) {
      dw = (g * x * inv).masked_fill(a.there.logical_not(), 0).flatten(0, -2).sum(0).to(w->scalar_type());
      g = g * w->to(at::kFloat);
    }
    const at::Tensor dx = inv * (g - x * inv * inv * (g * x).mean(-1, true));
    return std::make_pair(dx.masked_fill(a.there.logical_not(), 0).to(x0.scalar_type()).contiguous(), dw);
  };
  auto [dq, dwq] = one(q, gq, qw);
  auto [dk, dwk] = one(k, gk, kw);
  return {dq, dk, dwq, dwk};
}

// ---------------------------------------------------------- paged_append ----
// do the memory ranges of two tensors meet?
bool meets(const at::Tensor& a, const at::Tensor& b) {
  auto end = [](const at::Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return static_cast<const char*>(t.data_ptr()) + (last + 1) * t.element_size();
  };
  return a.numel() > 0 && b.numel() > 0 && static_cast<const char*>(a.data_ptr()) < end(b) &&
         static_cast<const char*>(b.data_ptr()) < end(a);
}

Cache check_append(const OptTensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache,
                   const at::Tensor& v_cache, const at::Tensor& table, const at::Tensor& cu, const at::Tensor& len,
                   const OptTensor& rope, bool norm, const OptTensor& qw, const OptTensor& kw, double eps) {
  const char* op = "paged_append";
  type_of(k, op);
  TORCH_CHECK(k.dim() == 3 && v.sizes() == k.sizes(), op, ": k and v are both [tokens, kv heads, head dim], got ", k.sizes(),
              " and ", v.sizes());
  check_like(v, k, op, "v");
  const Cache c = check_cache(k, k_cache, v_cache, table, cu, len, op);
  TORCH_CHECK(k.size(1) == c.heads && k.size(2) == c.dim, op, ": k ", k.sizes(), " does not fit a cache of ", c.heads,
              " heads of ", c.dim);
  for (const auto* t : {&k_cache, &v_cache})
    TORCH_CHECK(at::has_internal_overlap(*t) != at::MemOverlap::Yes, op, ": rows of the cache lie on each other");
  const auto both = at::get_overlap_status(k_cache, v_cache);
  TORCH_CHECK((k_cache.numel() == 0 || k_cache.data_ptr() != v_cache.data_ptr()) && both != at::MemOverlapStatus::Full &&
                  both != at::MemOverlapStatus::Partial,
              op, ": k_cache and v_cache are one");
  for (const at::Tensor* t : {&k, &v, given(q) ? &*q : &k})
    TORCH_CHECK(!meets(*t, k_cache) && !meets(*t, v_cache), op, ": the new rows are a part of the cache");
  if (given(q)) {
    check_like(*q, k, op, "q");
    TORCH_CHECK(q->dim() == 3 && q->size(0) == k.size(0) && q->size(1) > 0 && q->size(2) == c.dim, op, ": q ", q->sizes(),
                " does not fit k ", k.sizes());
    TORCH_CHECK(q->size(1) + 2 * c.heads <= 65535, op, ": more heads than one call takes");
  }
  if (given(rope)) check_rope(*rope, k, c.dim, op);
  TORCH_CHECK(norm || (!given(qw) && !given(kw)), op, ": weights without norm");
  TORCH_CHECK(given(q) || !given(qw), op, ": q_weight without q");
  check_weights(qw, kw, k, c.dim, op);
  check_eps(eps, op);
  return c;
}

at::Tensor paged_append_cuda(const OptTensor& q0, const at::Tensor& k0, const at::Tensor& v0, at::Tensor& k_cache,
                             at::Tensor& v_cache, const at::Tensor& table, const at::Tensor& cu, const at::Tensor& len,
                             const OptTensor& rope, bool norm, const OptTensor& qw, const OptTensor& kw, double eps,
                             bool interleaved) {
  const Cache c = check_append(q0, k0, v0, k_cache, v_cache, table, cu, len, rope, norm, qw, kw, eps);
  const c10::hip::OptionalHIPGuardMasqueradingAsCUDA guard(k0.device());
  at::Tensor out = given(q0) ? packed_like(*q0) : at::empty({0}, k0.options());
  if (k0.size(0) == 0) return out;
  const at::Tensor k = rows_aligned(k0, row_bytes(k0)), v = rows_aligned(v0, row_bytes(v0));
  const at::Tensor q = given(q0) ? rows_aligned(*q0, row_bytes(*q0)) : at::Tensor();
  nnsx::kernels::RopeArgs a;
  std::vector<at::Tensor> keep;
  a.type = type_of(k, "paged_append");
  if (q.defined()) {
    fill_rows(&a.q, q);
    a.q.y = out.data_ptr();
  }
  fill_rows(&a.k, k);
  fill_rows(&a.v, v);
  fill_weights(&a, qw, kw, &keep);
  a.S = static_cast<int>(k.size(0));
  a.d = static_cast<int>(c.dim);
  if (given(rope)) {
    a.rot = static_cast<int>(rope->size(1));
    keep.push_back(rows_aligned(*rope, 16));
    a.rope = keep.back().data_ptr<float>();
    a.rstride = keep.back().stride(0);
    a.positions = static_cast<int>(rope->size(0));
  }
  a.interleaved = interleaved ? 1 : 0;
  a.norm = norm ? 1 : 0;
  a.eps = static_cast<float>(eps);
  fill_batch(&a.p, c, table, cu, len, k.size(0));
  a.kc = k_cache.data_ptr();
  a.vc = v_cache.data_ptr();
  a.kp = k_cache.stride(0);
  a.kh = k_cache.stride(1);
  a.kr = k_cache.stride(2);
  a.vp = v_cache.stride(0);
  a.vh = v_cache.stride(1);
  a.vr = v_cache.stride(2);
  nnsx::kernels::paged_append(a, cur_stream());
  return out;
}

at::Tensor paged_append_cpu(const OptTensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor& k_cache,
                            at::Tensor& v_cache, const at::Tensor& table, const at::Tensor& cu, const at::Tensor& len,
                            const OptTensor& rope, bool norm, const OptTensor& qw, const OptTensor& kw, double eps,
                            bool interleaved) {
  const Cache c = check_append(q, k, v, k_cache, v_cache, table, cu, len, rope, norm, qw, kw, eps);
  const auto off = offsets(cu, k.size(0), "paged_append");
  at::Tensor out = given(q) ? at::zeros(q->sizes(), q->options().memory_format(at::MemoryFormat::Contiguous))
                            : at::empty({0}, k.options());
  for (int64_t b = 0; b < table.size(0); ++b) {
    const int64_t n = off[b + 1] - off[b], total = std::max(len.data_ptr<int>()[b], 0);
    if (n == 0) continue;
    const at::Tensor pos = at::arange(total - n, total, table.options().dtype(at::kLong));
    Angles ang;
    if (given(rope)) {
      ang = angles(pos, *rope);
    } else {
      ang.there = pos.ge(0).view({-1, 1, 1});
    }
    auto ready = [&](const at::Tensor& x, const OptTensor& w) {
      at::Tensor y = x.slice(0, off[b], off[b + 1]).to(at::kFloat);
      if (norm) y = normed(y, w, eps);
      if (given(rope)) y = turned(y, ang, interleaved, 1.0);
      return y.masked_fill(ang.there.logical_not(), 0).to(x.scalar_type());
    };
    if (given(q)) out.slice(0, off[b], off[b + 1]).copy_(ready(*q, qw));
    const at::Tensor kk = ready(k, kw);
    for (int64_t i = 0; i < n; ++i) {
      const int64_t p = total - n + i;
      if (!ang.there[i].item<bool>() || p >= table.size(1) * c.page) continue;
      const int64_t id = table[b][p / c.page].item<int64_t>();
      if (id < 0 || id >= c.pages) continue;
      k_cache.select(0, id).select(1, p % c.page).copy_(kk[i]);
      v_cache.select(0, id).select(1, p % c.page).copy_(v[off[b] + i]);
    }
  }
  return out;
}

// -------------------------------------------------------------- autograd ----
// (A node of its own: the host's part of a small forward and backward takes 84 us, 89 us as a torch::autograd::Function.)
struct QkNormRopeBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable q, k, qw, kw, pos, rope;
  double eps = 0;
  bool interleaved = false;

  std::string name() const override { return "QkNormRopeBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto* v : {&q, &k, &qw, &kw, &pos, &rope}) v->reset_data();
  }

  torch::autograd::variable_list apply(torch::autograd::variable_list&& g) override {
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("nnsx::qk_norm_rope_backward", "")
                               .typed<decltype(qk_norm_rope_backward_cuda)>();
    std::lock_guard<std::mutex> lock(mutex_);
    if (!g[0].defined() && !g[1].defined()) return torch::autograd::variable_list(4);
    const auto self = shared_from_this();
    const at::Tensor x = q.unpack(self), y = k.unpack(self), wx = qw.unpack(self), wy = kw.unpack(self);
    auto opt = [](const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    auto [dq, dk, dwq, dwk] = op.call(g[0].defined() ? g[0] : at::zeros_like(x), g[1].defined() ? g[1] : at::zeros_like(y), x, y,
                                      opt(wx), opt(wy), pos.unpack(self), rope.unpack(self), eps, interleaved);
    return {dq, dk, wx.defined() ? dwq : at::Tensor(), wy.defined() ? dwk : at::Tensor()};
  }
};

// a tangent would be dropped unnoticed
void no_forward_gradient(const char* op, std::initializer_list<const at::Tensor*> ts) {
  for (const auto* t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), op, " has no forward-mode gradient");
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope_autograd(const at::Tensor& q, const at::Tensor& k, const OptTensor& qw,
                                                         const OptTensor& kw, const at::Tensor& pos,
                                                         const at::Tensor& rope, double eps, bool interleaved) {
  using torch::autograd::SavedVariable;
  TORCH_CHECK(!at::GradMode::is_enabled() || !rope.requires_grad(), "qk_norm_rope: no gradient for the table of angles");
  const at::Tensor wq = given(qw) ? *qw : at::Tensor(), wk = given(kw) ? *kw : at::Tensor();
  no_forward_gradient("qk_norm_rope", {&q, &k, &wq, &wk, &rope});
  std::shared_ptr<QkNormRopeBackward> node;
  if (torch::autograd::compute_requires_grad(q, k, wq, wk)) {
    node = std::shared_ptr<QkNormRopeBackward>(new QkNormRopeBackward, torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(q, k, wq, wk));
    node->q = SavedVariable(q, false);
    node->k = SavedVariable(k, false);
    if (wq.defined()) node->qw = SavedVariable(wq, false);
    if (wk.defined()) node->kw = SavedVariable(wk, false);
    node->pos = SavedVariable(pos, false);
    node->rope = SavedVariable(rope, false);
    node->eps = eps;
    node->interleaved = interleaved;
  }
  at::Tensor yq, yk;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("nnsx::qk_norm_rope", "")
                               .typed<decltype(qk_norm_rope_cpu)>();
    std::tie(yq, yk) = op.call(q, k, qw, kw, pos, rope, eps, interleaved);
  }
  if (node) {
    torch::autograd::set_history(yq, node);
    torch::autograd::set_history(yk, node);
  }
  return {yq, yk};
}

// an operator without a derivative says so where one would be recorded
void no_gradient(const char* op, std::initializer_list<const at::Tensor*> ts) {
  no_forward_gradient(op, ts);
  if (!at::GradMode::is_enabled()) return;
  for (const auto* t : ts)
    TORCH_CHECK(!t->defined() || !t->requires_grad(), op, " has no gradient: call it under torch.no_grad(), or on detached tensors");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_norm_rope_backward_autograd(
    const at::Tensor& gq, const at::Tensor& gk, const at::Tensor& q, const at::Tensor& k, const OptTensor& qw,
    const OptTensor& kw, const at::Tensor& pos, const at::Tensor& rope, double eps, bool interleaved) {
  const at::Tensor none;
  no_gradient("qk_norm_rope_backward", {&gq, &gk, &q, &k, given(qw) ? &*qw : &none, given(kw) ? &*kw : &none, &rope});
  at::AutoDispatchBelowADInplaceOrView below;
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("nnsx::qk_norm_rope_backward", "")
                             .typed<decltype(qk_norm_rope_backward_cpu)>();
  return op.call(gq, gk, q, k, qw, kw, pos, rope, eps, interleaved);
}

at::Tensor paged_attention_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                                    const at::Tensor& cu, const at::Tensor& len, c10::optional<double> scale, bool causal,
                                    int64_t window) {
  no_gradient("paged_attention", {&q, &k, &v});
  at::AutoDispatchBelowADInplaceOrView below;
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("nnsx::paged_attention", "")
                             .typed<decltype(paged_attention_cpu)>();
  return op.call(q, k, v, table, cu, len, scale, causal, window);
}

const auto& append_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("nnsx::paged_append", "")
                             .typed<decltype(paged_append_cpu)>();
  return op;
}

at::Tensor paged_append_autograd(const OptTensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor& k_cache,
                                 at::Tensor& v_cache, const at::Tensor& table, const at::Tensor& cu, const at::Tensor& len,
                                 const OptTensor& rope, bool norm, const OptTensor& qw, const OptTensor& kw, double eps,
                                 bool interleaved) {
  const at::Tensor none;
  no_gradient("paged_append", {given(q) ? &*q : &none, &k, &v, &k_cache, &v_cache, given(qw) ? &*qw : &none,
                               given(kw) ? &*kw : &none, given(rope) ? &*rope : &none});
  at::AutoDispatchBelowAutograd below;
  return append_op().call(q, k, v, k_cache, v_cache, table, cu, len, rope, norm, qw, kw, eps, interleaved);
}

// what an earlier operation keeps of the cache for its gradient has changed
at::Tensor paged_append_inplace(const OptTensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor& k_cache,
                                at::Tensor& v_cache, const at::Tensor& table, const at::Tensor& cu, const at::Tensor& len,
                                const OptTensor& rope, bool norm, const OptTensor& qw, const OptTensor& kw, double eps,
                                bool interleaved) {
  for (const auto* t : {&k_cache, &v_cache})  // (the count of changes below would refuse it, after the change)
    TORCH_CHECK(!t->is_inference() || c10::InferenceMode::is_enabled(),
                "paged_append: a cache made in inference mode can be changed in inference mode only");
  at::Tensor out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = append_op().call(q, k, v, k_cache, v_cache, table, cu, len, rope, norm, qw, kw, eps, interleaved);
  }
  torch::autograd::impl::bump_version(k_cache);
  torch::autograd::impl::bump_version(v_cache);
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(nnsx, m) {
  m.def("rope_table(int positions, int dim, float base=10000.0) -> Tensor", rope_table);
  m.def("qk_norm_rope(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor positions, Tensor rope, "
        "float eps=1e-6, bool interleaved=False) -> (Tensor, Tensor)");
  m.def("qk_norm_rope_backward(Tensor grad_q, Tensor grad_k, Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, "
        "Tensor positions, Tensor rope, float eps=1e-6, bool interleaved=False) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("paged_append(Tensor? q, Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor page_table, "
        "Tensor cu_seqlens, Tensor kv_lens, Tensor? rope=None, bool norm=False, Tensor? q_weight=None, "
        "Tensor? k_weight=None, float eps=1e-6, bool interleaved=False) -> Tensor");
  m.def("paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor cu_seqlens, "
        "Tensor kv_lens, float? scale=None, bool causal=True, int window=0) -> Tensor");
}

TORCH_LIBRARY_IMPL(nnsx, CUDA, m) {
  m.impl("qk_norm_rope", qk_norm_rope_cuda);
  m.impl("qk_norm_rope_backward", qk_norm_rope_backward_cuda);
  m.impl("paged_append", paged_append_cuda);
  m.impl("paged_attention", paged_attention_cuda);
}

TORCH_LIBRARY_IMPL(nnsx, CPU, m) {
  m.impl("qk_norm_rope", qk_norm_rope_cpu);
  m.impl("qk_norm_rope_backward", qk_norm_rope_backward_cpu);
  m.impl("paged_append", paged_append_cpu);
  m.impl("paged_attention", paged_attention_cpu);
}

TORCH_LIBRARY_IMPL(nnsx, Autograd, m) {
  m.impl("qk_norm_rope", qk_norm_rope_autograd);
  m.impl("qk_norm_rope_backward", qk_norm_rope_backward_autograd);
  m.impl("paged_append", paged_append_autograd);
  m.impl("paged_attention", paged_attention_autograd);
}

TORCH_LIBRARY_IMPL(nnsx, ADInplaceOrView, m) { m.impl("paged_append", paged_append_inplace); }
