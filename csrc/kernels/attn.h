// Attention over a paged key/value cache (attn.hip) and the per-head norm,
// position rotation and cache append that feed it (rope.hip).
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

namespace nnsx {
namespace kernels {

enum class AttnType : int { kBF16 = 0, kF16 = 1, kF32 = 2 };

// A batch of sequences over a paged cache.  Sequence b owns the new tokens
// cu[b] .. cu[b + 1] - 1 (cu[0] counts as 0) and has len[b] keys with them, so its
// i-th new token stands at position len[b] - n + i; key j lives in page
// table[b * width + j / page] at row j % page.  A page id outside
// [0, pages) and a key behind the table's last page are not there: they are
// neither read nor written.
struct PagedBatch {
  const int* table = nullptr;
  const int* cu = nullptr;
  const int* len = nullptr;
  int64_t tstride = 0;  // table row stride
  int B = 0, T = 0;     // sequences, token rows (rows from cu[B] on belong to nobody)
  int width = 0, page = 1, pages = 0;
};

struct PagedAttnArgs {
  PagedBatch p;
  AttnType type = AttnType::kBF16;
  const void* q = nullptr;  // [T][hq][d], strides qt / qh elements
  const void* k = nullptr;  // [pages][hkv][page][d], strides kp / kh / kr
  const void* v = nullptr;
  void* o = nullptr;  // [T][hq][d] contiguous
  int64_t qt = 0, qh = 0, kp = 0, kh = 0, kr = 0, vp = 0, vh = 0, vr = 0;
  int hq = 0, hkv = 0, d = 0;
  float scale = 1.f;
  int causal = 1;
  int window = 0;       // 0: no window; else only keys from position - window + 1 on (up to the last, unless causal)
  void* ws = nullptr;   // paged_attn_workspace_bytes(a)
  // derived by the launcher: rows a token, and how the keys are split (attn.hip, plan)
  int group = 1, target = 0, min_chunk = 1, slots = 0, pairs = 0, parts = 0, apart = 1, one_round = 0, item_cost = 0, rows_lo = 0, rows_hi = 0;
  void* plan = nullptr;
  int* chunk = nullptr;  // key blocks of a split, left by the attention for the join
};
// bytes of scratch memory the call needs (0: none)
size_t paged_attn_workspace_bytes(const PagedAttnArgs& a);
// d % 8 == 0, d <= 256, 16-byte aligned rows; rows without a key become zero
void paged_attn(const PagedAttnArgs& a, hipStream_t s);

// Rows of queries and keys (and values, which only a cache append takes):
// x[b][s][head][d] with strides sb / ss / sh, rows of d elements aligned to 16 bytes,
// or to 8 where the type has 16 bits.
struct RopeRows {
  const void* x = nullptr;
  const void* g = nullptr;  // backward: gradient of the output rows, strides gb / gs / gh
  void* y = nullptr;        // forward: output rows; backward: gradient of x; [B][S][heads][d] contiguous
  const void* w = nullptr;  // [d] norm weight, or null
  int64_t sb = 0, ss = 0, sh = 0, gb = 0, gs = 0, gh = 0;
  int heads = 0;
};

struct RopeArgs {
  AttnType type = AttnType::kBF16;
  int w_f32 = 0;            // weights are fp32 (else the rows' type)
  RopeRows q, k, v;         // v: append only
  int B = 1, S = 0;         // append: B = 1, S = token rows
  int d = 0, rot = 0;       // d % 8 == 0, d <= 256; rot % 8 == 0, rot <= d
  int interleaved = 0, norm = 1;
  float eps = 0.f;
  const float* rope = nullptr;  // [positions][rot]: cosines, then sines
  int64_t rstride = 0;
  int positions = 0;
  const void* pos = nullptr;  // qk_norm_rope: [B][S], strides pb / ps; int64 or int32
  int pos64 = 0;
  int64_t pb = 0, ps = 0;
  // append
  PagedBatch p;
  void* kc = nullptr;
  void* vc = nullptr;
  int64_t kp = 0, kh = 0, kr = 0, vp = 0, vh = 0, vr = 0;
  // backward: gradients of the weights ([d] each in the weights' type, null: not wanted) and their scratch
  void* dwq = nullptr;
  void* dwk = nullptr;
  float* ws = nullptr;
};
// y = R(position) (w . x / sqrt(mean x^2 + eps)) for every head of q and k; a row
// whose position the table does not hold becomes zero
void qk_norm_rope(const RopeArgs& a, hipStream_t s);
// its gradient: q.y / k.y from q.g / k.g, and dwq / dwk
size_t qk_norm_rope_backward_workspace_bytes(const RopeArgs& a);
void qk_norm_rope_backward(const RopeArgs& a, hipStream_t s);
// q -> q.y and k, v -> cache rows, by the batch's positions
void paged_append(const RopeArgs& a, hipStream_t s);

}  // namespace kernels
}  // namespace nnsx
