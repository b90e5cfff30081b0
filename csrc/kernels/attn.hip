// Attention of new tokens over a paged key/value cache, gfx950.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j   over the keys j that row i sees
//
// Rows: the new tokens of one sequence times the query heads that share one
// key/value head, packed token-major (row = token * group + head in group), so
// a key is fetched once for the whole group.  Both products run transposed on
// 32 x 32 matrix instructions,
//
//   S^T = K Q^T   (A = 32 keys, B = 32 rows)    O^T = V^T P^T   (A = V^T, B = P^T),
//
// so that a lane holds one row's scores: 16 of a block's 32 keys, the lane 32
// further the other 16.  The running maximum and sum of the softmax are then
// one exchange between two lanes per block, the rescale of O^T is one factor
// per lane, and P^T is already where the second product wants it -- the order
// of the summed index is free as long as V^T uses the same one (slot j of lane
// half h = key 16 s + 8 (j / 4) + 4 h + j % 4).  Scores, maxima, sums and O are
// fp32; for the second product P is rounded to the cache's type, each weight by
// at most half a step of itself, as the output is: without that the matrix
// instruction of 16-bit operands could not take it, and two parts a weight would
// double the second product.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "kernels/attn.h"

namespace nnsx {
namespace kernels {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kRows = 32;   // rows of one item
constexpr int kKeys = 32;   // keys of one block
constexpr int kCus = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_huge_valf();

struct BF16 {};
struct F16 {};
struct F32 {};

// 8 slots of the summed index for one lane: 16-bit types
template <typename T>
__device__ __forceinline__ f32x16 mfma16(u32x4 a, u32x4 b, f32x16 c);
template <>
__device__ __forceinline__ f32x16 mfma16<BF16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 mfma16<F16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<BF16>(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}
template <>
__device__ __forceinline__ uint32_t pack2<F16>(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
}
// A word's values that are infinite or NaN: their sign bits set in `infinite`
// (the exponent's bits all ones carry into it), `finite_part` the word with them 0.
template <typename T>
struct Bits;
template <>
struct Bits<BF16> { static constexpr uint32_t exp = 0x7f807f80u, low = 0x00800080u, sign = 0x80008000u; };
template <>
struct Bits<F16> { static constexpr uint32_t exp = 0x7c007c00u, low = 0x04000400u, sign = 0x80008000u; };
template <>
struct Bits<F32> { static constexpr uint32_t exp = 0x7f800000u, low = 0x00800000u, sign = 0x80000000u; };
template <typename T>
__device__ __forceinline__ uint32_t infinite(uint32_t x) {
  return (x & Bits<T>::exp) + Bits<T>::low;
}
template <typename T>
__device__ __forceinline__ uint32_t finite_part(uint32_t x) {
  const uint32_t f = infinite<T>(x) & Bits<T>::sign;
  if constexpr (std::is_same_v<T, F32>) return f ? 0u : x;
  return x & ~((f >> 15) * 0xffffu);
}
// Weights are e^(score - maximum) times 2^kLift: fp16 has no values below 2^-24, and
// a hundred thousand keys of less weight each are not nothing
template <typename T>
constexpr float kLift = std::is_same_v<T, F16> ? 7.f : 0.f;
// value number e of a word
template <typename T>
__device__ __forceinline__ float value_of(uint32_t x, int e);
template <>
__device__ __forceinline__ float value_of<BF16>(uint32_t x, int e) {
  return __uint_as_float(e ? x & 0xffff0000u : x << 16);
}
template <>
__device__ __forceinline__ float value_of<F16>(uint32_t x, int e) {
  return static_cast<float>(__builtin_bit_cast(f16x2, x)[e]);
}
template <>
__device__ __forceinline__ float value_of<F32>(uint32_t x, int) {
  return __uint_as_float(x);
}

// the low (0) or high (1) 16 bits of two words, the first's below
__device__ __forceinline__ uint32_t interleave(uint32_t a, uint32_t b, int high) {
  return __builtin_amdgcn_perm(b, a, high ? 0x07060302u : 0x05040100u);
}
// max(a, b) as one instruction, the middle of a, b and infinity (fmaxf first quiets both
// operands, and so would this if the compiler knew the constant); a NaN loses
__device__ __forceinline__ float max2(float a, float b, float inf) { return __builtin_amdgcn_fmed3f(a, b, inf); }
__device__ __forceinline__ float opaque_infinity() {
  float inf;
  asm volatile("s_mov_b32 %0, 0x7f800000" : "=s"(inf));
  return inf;
}
// max(a, b, c) likewise, of results that no matrix instruction wrote (the compiler keeps no distance for asm)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// over the two lanes of a row, 32 apart
__device__ __forceinline__ float row_max(float x, float inf) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return max2(__uint_as_float(r[0]), __uint_as_float(r[1]), inf);
}
__device__ __forceinline__ float row_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Scores times `c` are rounded before their maximum is taken, but fused into the exponent's subtraction: the
// largest key's exponent is off by half a step of the maximum.  From 2^20 on that may be more than 2^-4 (from 2^28 on
// it would leave fp16's range), and the products are rounded first there too, so that it is 0.
constexpr float kFar = 1048576.f;
__device__ __forceinline__ bool any_far(float max) { return __any(fabsf(max) >= kFar && max != kNegInf); }
__device__ __forceinline__ float far_exponent(float s, float c, float max, float lift) {
  float x = s * c;
  asm("" : "+v"(x));  // (a product by itself)
  return x - max + lift;
}

// ------------------------------------------------------------------- plan ----
// Work is cut into items: (sequence, tile of rows, split of its key blocks).
// Lengths live on the device, so every wave derives its own item from them (of many
// sequences, from what one workgroup has summed up before): the
// key blocks of all (sequence, tile) pairs are summed, a split is chosen so long
// that about `target` items result (more only because every pair has at least
// one), and the item's pair is found by a running sum over the sequences.
// target = 0: no split.
struct Item {
  int b;        // sequence; -1: nothing to do.  B: the rows behind the last sequence
  int tile, split, splits;
  int part;     // of the scratch memory, if split
  int chunk;    // key blocks of a split
  int n, t0;    // new tokens, first token row
  int len, keys;  // length; keys that the table can hold of them
};

struct Seq {
  int n, t0, len, keys, tiles, blocks;
};

template <int ROWS, int KEYS>
__device__ __forceinline__ Seq seq_of(const PagedAttnArgs& a, int b) {
  Seq s;
  const int T = a.p.T, B = a.p.B;
  // (three loads at once; the last entry stands for the rows behind the last sequence)
  const int c0 = a.p.cu[b], c1 = a.p.cu[min(b + 1, B)], len = B > 0 ? a.p.len[min(b, B - 1)] : 0;
  s.t0 = b == 0 ? 0 : min(max(c0, 0), T);
  const int t1 = b < B ? min(max(c1, 0), T) : T;
  s.n = max(t1 - s.t0, 0);
  s.len = b < B ? max(len, 0) : 0;
  s.keys = min(s.len, a.p.width * a.p.page);
  const int rows = s.n * a.group;  // (T * hq < 2^31)
  if (rows <= a.rows_lo || rows > a.rows_hi) s.n = 0;  // (the other form's)
  s.tiles = s.n > 0 ? static_cast<int>((static_cast<uint32_t>(rows) + ROWS - 1) / ROWS) : 0;
  const int64_t first = static_cast<int64_t>(s.len) - s.n - a.window + 1;
  const int lo = a.window > 0 ? static_cast<int>(min(max(first, static_cast<int64_t>(0)), static_cast<int64_t>(s.keys))) : 0;
  s.blocks = s.n > 0 ? static_cast<int>(static_cast<uint32_t>(s.keys + KEYS - 1) / KEYS - static_cast<uint32_t>(lo) / KEYS) : 0;
  return s;
}

// sum of the lanes up to this one
template <typename V>
__device__ __forceinline__ V wave_scan(V x) {
  auto shifted = [&](auto ctrl, auto rows) {
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value,
                                                             decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  x += shifted(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});  // row_shr 1, 2, 4, 8
  x += shifted(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  x += shifted(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  x += shifted(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  x += shifted(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // row_bcast 15, 31
  x += shifted(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return x;
}
// the least of all lanes, in the last one
__device__ __forceinline__ float wave_least(float x) {
  auto other = [&](auto ctrl, auto rows) {  // (where there is none: itself)
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, x), __builtin_bit_cast(int, x),
                                                                 decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  x = fminf(x, other(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{}));
  x = fminf(x, other(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{}));
  x = fminf(x, other(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{}));
  x = fminf(x, other(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{}));
  x = fminf(x, other(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{}));
  x = fminf(x, other(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{}));
  return x;
}
template <typename V>
__device__ __forceinline__ V last_lane(V x) {
  return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// key blocks of a split: the items of all pairs stay within `target` more than the pairs
__device__ __forceinline__ int chunk_of(const PagedAttnArgs& a, float blocks) {
  if (a.target == 0) return 1 << 28;
  // (a float sum of few terms is off by less than the 1e-4 that is added; no sequence has 2^25 blocks)
  const float c = blocks * 1.0001f / static_cast<float>(a.target);
  return max(static_cast<int>(fminf(c, 33554432.f)) + 1, a.min_chunk);
}

// pairs, items beyond one a pair << 16 | items of split pairs (both below 2 target)
struct Count {
  int pairs;
  uint32_t split;
};
__device__ __forceinline__ Count count_of(const Seq& s, int splits) {
  return {s.tiles, splits > 1 ? static_cast<uint32_t>(s.tiles) * (static_cast<uint32_t>(splits - 1) << 16 | splits) : 0u};
}
__device__ __forceinline__ int splits_of(const Seq& s, int chunk) {
  return s.blocks > chunk ? static_cast<int>(static_cast<uint32_t>(s.blocks + chunk - 1) / static_cast<uint32_t>(chunk)) : 1;
}

// Many sequences: what stands before each, [B + 1], and behind them the key blocks of a split, all
// written by one workgroup in a launch before the others.  (Where every wave looked through all sequences instead,
// 64 at a time: 1024 single tokens after 512 655 us, 408 by the plan; 256 136 and 119; 64 after 1024, which
// were not weighed then, 70 and 54.)
struct PlanEntry {
  int pairs;
  uint32_t split;  // as in Count
};

// item number `rel` of a sequence, `first_split` before it
template <bool PAIRS>
__device__ __forceinline__ Item item_of(const PagedAttnArgs& a, int b, const Seq& s, int rel, int splits, int chunk, uint32_t first_split) {
  Item it;
  it.splits = splits;
  const int tile = PAIRS ? rel : rel / splits;
  it.split = PAIRS ? 0 : rel - tile * splits;
  it.tile = s.tiles - 1 - tile;  // the tiles with the most keys first: the short ones fill the tail
  it.part = static_cast<int>(first_split & 0xffff) + tile * splits + it.split;
  it.chunk = chunk;
  it.n = s.n;
  it.t0 = s.t0;
  it.len = s.len;
  it.keys = s.keys;
  // (offsets that do not ascend may make more items than planned for: those are left out)
  it.b = splits == 1 || (it.part >= 0 && it.part <= a.parts - (PAIRS ? splits : 1)) ? b : -1;
  return it;
}

template <int ROWS, int KEYS, bool PAIRS>
__device__ __forceinline__ Item find_planned(const PagedAttnArgs& a, int index) {
  const PlanEntry* plan = static_cast<const PlanEntry*>(a.plan);
  const int lane = threadIdx.x & 63, B1 = a.p.B + 1;
  auto first_of = [&](const PlanEntry& e) { return PAIRS ? e.pairs : e.pairs + static_cast<int>(e.split >> 16); };
  // the last sequence that begins at or before the item, by 64 steps at a time
  int lo = 0;
  for (int n = B1, step = 0; step != 1; n = min(step, B1 - lo)) {
    step = (n + 63) / 64;
    const int i = lane * step;
    const int c = __popcll(__ballot(i < n && first_of(plan[lo + min(i, n - 1)]) <= index));
    lo += max(c - 1, 0) * step;
  }
  const PlanEntry e = plan[lo];
  const int chunk = plan[B1].pairs;
  const Seq s = seq_of<ROWS, KEYS>(a, lo);
  const int splits = splits_of(s, chunk), rel = index - first_of(e);
  if (rel < 0 || rel >= s.tiles * (PAIRS ? 1 : splits)) {
    Item none;
    none.b = -1;
    return none;
  }
  return item_of<PAIRS>(a, lo, s, rel, splits, chunk, e.split);
}

// The card takes `one_round` items of a kv head at once: items just beyond a round take a whole
// one more, and each has a cost of its own.  So of the splits 1, 1 1/8, .. 8 7/8 times as long
// as the shortest, one a lane, the one with the least rounds times blocks is taken (by estimate:
// products with reciprocals).
__device__ __forceinline__ int longer(int chunk, int lane) { return chunk + chunk / 8 * lane + chunk % 8 * lane / 8; }
__device__ __forceinline__ float items_by(int tiles, int blocks, float of_chunk) {
  return static_cast<float>(tiles) * fmaxf(ceilf(static_cast<float>(blocks) * of_chunk - 1e-3f), 1.f);
}
// this lane's items of the wave's sequences
__device__ __forceinline__ float weigh_wave(const Seq& s, int chunk) {
  const float of = __builtin_amdgcn_rcpf(static_cast<float>(chunk));
  float items = 0.f;
  for (uint64_t left = __ballot(s.tiles > 0); left != 0; left &= left - 1) {
    const int l = __builtin_ctzll(left);
    items += items_by(__builtin_amdgcn_readlane(s.tiles, l), __builtin_amdgcn_readlane(s.blocks, l), of);
  }
  return items;
}
__device__ __forceinline__ int best_of(const PagedAttnArgs& a, int chunk, float items) {
  const float round = __builtin_amdgcn_rcpf(static_cast<float>(a.one_round));
  const float cost = ceilf(items * round - 1e-3f) * static_cast<float>(chunk + a.item_cost);
  return __builtin_amdgcn_readlane(chunk, __builtin_ctzll(__ballot(cost == last_lane(wave_least(cost)))));
}

// PAIRS false: `index` counts items; PAIRS true: (sequence, tile) pairs, and
// the item is the pair's first split.  Up to 64 sequences with the rows behind the last: each wave
// finds it by itself among them.  The split comes from sums of floats, which another kernel's code might round
// otherwise (products fused into sums or not): the join takes the one that the attention has left in a.chunk.
template <int ROWS, int KEYS, bool PAIRS>
__device__ Item find_item(const PagedAttnArgs& a, int index) {
  if (a.plan != nullptr) return find_planned<ROWS, KEYS, PAIRS>(a, index);
  const int lane = threadIdx.x & 63;
  Seq s{};
  if (lane <= a.p.B) s = seq_of<ROWS, KEYS>(a, lane);
  int chunk;
  if constexpr (PAIRS) {
    chunk = *a.chunk;
  } else {
    chunk = chunk_of(a, last_lane(wave_scan(static_cast<float>(s.tiles) * static_cast<float>(s.blocks))));
    if (a.target > 0) {  // (chunk < 2^26)
      const float items = last_lane(wave_scan(items_by(s.tiles, s.blocks, __builtin_amdgcn_rcpf(static_cast<float>(chunk)))));
      if (items > static_cast<float>(a.one_round) + 0.5f) {
        const int c = longer(chunk, lane);
        chunk = best_of(a, c, weigh_wave(s, c));
      }
    }
  }
  const int splits = splits_of(s, chunk);
  const Count mine = count_of(s, splits);
  const int first_pair = wave_scan(mine.pairs) - mine.pairs;
  const uint32_t first_split = a.target > 0 ? static_cast<uint32_t>(wave_scan(static_cast<int>(mine.split))) - mine.split : 0u;
  const int first = PAIRS ? first_pair : first_pair + static_cast<int>(first_split >> 16);
  const uint64_t here = __ballot(index >= first && index - first < s.tiles * (PAIRS ? 1 : splits));
  if (here == 0) {
    Item none;
    none.b = -1;
    none.chunk = chunk;
    return none;
  }
  const int l = __builtin_ctzll(here);
  auto get = [&](int x) { return __builtin_amdgcn_readlane(x, l); };
  const Seq found{get(s.n), get(s.t0), get(s.len), get(s.keys), get(s.tiles), get(s.blocks)};
  return item_of<PAIRS>(a, l, found, index - get(first), get(splits), chunk, static_cast<uint32_t>(get(static_cast<int>(first_split))));
}

constexpr int kPlanThreads = 1024;

template <int ROWS, int KEYS>
__device__ void make_plan(const PagedAttnArgs& a) {
  constexpr int kWaves = kPlanThreads / 64;
  __shared__ float sums[kWaves];
  __shared__ float weighed[kWaves][64];
  __shared__ int tiles[kPlanThreads], blocks[kPlanThreads];
  __shared__ Count ends[kWaves];
  PlanEntry* plan = static_cast<PlanEntry*>(a.plan);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, B1 = a.p.B + 1;
  // (a sequence a thread is kept from loop to loop)
  auto load = [&](int b) {
    Seq s{};
    if (b < B1) s = seq_of<ROWS, KEYS>(a, b);
    return s;
  };
  const Seq mine0 = load(threadIdx.x);
  auto seq_at = [&](int b0) { return b0 == 0 ? mine0 : load(b0 + static_cast<int>(threadIdx.x)); };
  float work = 0.f;
  if (a.target > 0)
    for (int b0 = 0; b0 < B1; b0 += kPlanThreads) {
      const Seq s = seq_at(b0);
      work += static_cast<float>(s.tiles) * static_cast<float>(s.blocks);
    }
  work = wave_scan(work);
  if (lane == 63) sums[wave] = work;
  __syncthreads();
  work = 0.f;
  for (int w = 0; w < kWaves; ++w) work += sums[w];
  int chunk = chunk_of(a, work);
  if (a.target > 0) {
    const int c = longer(chunk, lane);
    const float of = __builtin_amdgcn_rcpf(static_cast<float>(c));
    float items = 0.f;
    for (int b0 = 0; b0 < B1; b0 += kPlanThreads) {  // (every wave takes some of the sequences)
      const Seq s = seq_at(b0);
      __syncthreads();
      tiles[threadIdx.x] = s.tiles;
      blocks[threadIdx.x] = s.blocks;
      __syncthreads();
      for (int i = wave; i < min(B1 - b0, kPlanThreads); i += kWaves)
        if (tiles[i] > 0) items += items_by(tiles[i], blocks[i], of);
    }
    weighed[wave][lane] = items;
    __syncthreads();
    items = 0.f;
    for (int w = 0; w < kWaves; ++w) items += weighed[w][lane];
    chunk = best_of(a, c, items);
  }
  Count before{0, 0};
  for (int b0 = 0; b0 < B1; b0 += kPlanThreads) {
    const int b = b0 + static_cast<int>(threadIdx.x);
    const Seq s = seq_at(b0);
    const Count mine = count_of(s, splits_of(s, chunk));
    const int pairs = wave_scan(mine.pairs);
    const uint32_t split = static_cast<uint32_t>(wave_scan(static_cast<int>(mine.split)));
    if (lane == 63) ends[wave] = {pairs, split};
    __syncthreads();
    Count here = before;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) {
        here.pairs += ends[w].pairs;
        here.split += ends[w].split;
      }
      before.pairs += ends[w].pairs;
      before.split += ends[w].split;
    }
    if (b < B1) plan[b] = {here.pairs + pairs - mine.pairs, here.split + split - mine.split};
    __syncthreads();
  }
  if (threadIdx.x == 0) plan[B1] = {chunk, 0u};
}

// keys [lo, hi) that the tokens i0 .. i1 of an item see
__device__ __forceinline__ void key_range(const PagedAttnArgs& a, const Item& it, int i0, int i1, int* lo, int* hi) {
  const int64_t first = static_cast<int64_t>(it.len) - it.n;
  *hi = a.causal ? static_cast<int>(min(max(first + i1 + 1, static_cast<int64_t>(0)), static_cast<int64_t>(it.keys)))
                 : it.keys;
  *lo = a.window > 0 ? static_cast<int>(min(max(first + i0 - a.window + 1, static_cast<int64_t>(0)),
                                            static_cast<int64_t>(it.keys)))
                     : 0;
  if (*hi < *lo) *hi = *lo;
}

// A key's page id (as the table has it, -1 behind the item's keys) and row in the page.  Only
// fetched here: a use of the id would wait for every load issued before it.
struct KeyRow {
  int id, off;
};
__device__ __forceinline__ KeyRow key_row(const PagedAttnArgs& a, const int* table, int key, int keys) {
  KeyRow r{-1, 0};
  if (key < keys) {
    const int p = key / a.p.page;
    r.off = key - p * a.p.page;
    r.id = table[p];
  }
  return r;
}
__device__ __forceinline__ bool is_there(const PagedAttnArgs& a, const KeyRow& r) {
  return static_cast<uint32_t>(r.id) < static_cast<uint32_t>(a.p.pages);
}

// scratch memory of a split call: for an item of a split pair and a kv head, rows x (max, sum, d columns)
__host__ __device__ __forceinline__ size_t part_floats(int rows, int d) { return static_cast<size_t>(rows) * (d + 2); }

// ------------------------------------------------------------ stream kernel ----
// One workgroup per item of 32 rows; its waves take key blocks in turn,
// each on its own (no barrier in the loop) and straight from global memory into
// the matrix instructions' registers: a lane loads 16 bytes of a key for S^T;
// for O^T the lanes of a half load a whole row of V (DP / 32 neighbouring
// columns each, so column = (DP / 32) * row of the tile + tile) and eight rows'
// halves are interleaved with byte permutes.  The waves' partial (max, sum,
// O) are joined through LDS at the end.
// Bound by the reads of the cache: 64 single tokens after 100 to 8192, 8 heads of 128 columns, bf16: 1.10 GB in
// 222 us, 5.0 TB/s, as a large copy; two after 131072 and 120001, fp16: 1.03 GB in 186 us, 5.5 TB/s.  One after
// 4096: 9.5 us, the plan and a few round trips to memory.  In fp32 64 single tokens take 611 us (2.21 GB, 3.6 TB/s), and a
// prompt of 2048 tokens, 32 heads of 128 columns, 477 us: 72 TFLOP/s of the pairs that count, a large product 153.
// The matrix unit is busy for 46 % of that: a workgroup fills the registers of a SIMD's one wave, so that reads of K
// and V (each again for every 32 rows), softmax and products mostly take turns.
template <typename T>
struct Elem { using type = uint16_t; static constexpr bool wide = false; };
template <>
struct Elem<F32> { using type = float; static constexpr bool wide = true; };

// QUAD: pages hold whole groups of four keys, so four neighbouring rows of V
// are addressed from the first one's offset.
template <typename T, int DP, bool QUAD, int kWaves>
__device__ __forceinline__ void stream_item(const PagedAttnArgs& a, unsigned index) {
  using E = typename Elem<T>::type;
  constexpr bool WIDE = Elem<T>::wide;
  constexpr int NB = DP / 32;            // 32-column tiles of O^T
  constexpr int KC = WIDE ? DP / 8 : DP / 16;  // 16-byte pieces of a key per lane
  constexpr int PIECE = WIDE ? 4 : 8;    // elements of a piece
  __shared__ float sh_ml[kWaves][2][kRows];
  __shared__ float sh_o[kWaves / 2][NB * 16][64];
  constexpr bool QLDS = DP * sizeof(E) > 256;
  __shared__ u32x4 sh_q[QLDS ? KC : 1][64];

  const int head = static_cast<int>(index % a.hkv);
  const int slot = static_cast<int>(index / a.hkv);
  const Item it = find_item<kRows, kKeys, false>(a, slot);
  if (index == 0 && threadIdx.x == 0 && a.chunk != nullptr) *a.chunk = it.chunk;
  if (it.b < 0) return;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int rows = it.n * a.group;  // (fits: T * hq < 2^31)
  const int row = it.tile * kRows + col;
  const bool live = row < rows;
  const int tok = row / a.group, gh = row - tok * a.group;
  // what this lane's row sees
  int rlo, rhi, tlo, thi;
  key_range(a, it, tok, tok, &rlo, &rhi);
  if (!live) rhi = rlo = 0;
  {
    const int i0 = it.tile * kRows / a.group, i1 = min((it.tile * kRows + kRows - 1) / a.group, it.n - 1);
    key_range(a, it, i0, i1, &tlo, &thi);
  }
  int blk0 = tlo / kKeys, blk1 = (thi + kKeys - 1) / kKeys;
  {  // this split's blocks
    const int64_t s0 = blk0 + static_cast<int64_t>(it.split) * it.chunk;
    const int64_t s1 = s0 + it.chunk;
    blk0 = static_cast<int>(min(s0, static_cast<int64_t>(blk1)));
    blk1 = static_cast<int>(min(s1, static_cast<int64_t>(blk1)));
  }

  const E* qp = static_cast<const E*>(a.q) + static_cast<int64_t>(it.t0 + tok) * a.qt +
                static_cast<int64_t>(head * a.group + gh) * a.qh;
  const E* kbase = static_cast<const E*>(a.k) + head * a.kh;
  const E* vbase = static_cast<const E*>(a.v) + head * a.vh;
  const int* table = a.p.table + static_cast<int64_t>(it.b) * a.p.tstride;

  // Q: in registers where they suffice, else in LDS (every wave reads the same rows)
  u32x4 q[QLDS ? 1 : KC];
  if constexpr (QLDS) {
    for (int s = wave; s < KC; s += kWaves) {
      const int d = (2 * s + half) * PIECE;
      sh_q[s][lane] = live && d < a.d ? *reinterpret_cast<const u32x4*>(qp + d) : (u32x4)(0u);
    }
    __syncthreads();
  } else {
#pragma unroll
    for (int s = 0; s < KC; ++s) {
      const int d = (2 * s + half) * PIECE;
      q[s] = (u32x4)(0u);
      if (live && d < a.d) q[s] = *reinterpret_cast<const u32x4*>(qp + d);
    }
  }
  auto q_piece = [&](int s) { return QLDS ? sh_q[QLDS ? s : 0][lane] : q[QLDS ? 0 : s]; };

  f32x16 o[NB];
#pragma unroll
  for (int m = 0; m < NB; ++m) o[m] = (f32x16)(0.f);
  float mx = kNegInf, sum = 0.f;
  bool distant = false;  // some row's maximum is
  const float c = a.scale * kLog2e, inf = opaque_infinity();

  u32x4 k[KC];
  // V: 16 rows a lane half, NB neighbouring columns: NB / 2 words (16 bit) or NB (32 bit)
  constexpr int VW = WIDE ? NB : NB / 2;
  uint32_t v[16][VW];
  const int vcol = NB * col;

  // this lane's key (lane & 31) of a block
  auto row_of = [&](int blk) { return key_row(a, table, blk < blk1 ? blk * kKeys + col : it.keys, it.keys); };
  auto load_k = [&](const KeyRow& r) {
    const bool there = is_there(a, r);
    const E* p = kbase + r.id * a.kp + r.off * a.kr;
#pragma unroll
    for (int s = 0; s < KC; ++s) {
      const int d = (2 * s + half) * PIECE;
      k[s] = (u32x4)(0u);
      if (there && d < a.d) k[s] = *reinterpret_cast<const u32x4*>(p + d);
    }
  };
  auto load_v = [&](const KeyRow& r) {
    const uint32_t there = static_cast<uint32_t>(__ballot(is_there(a, r))) >> (4 * half);
    const E* first = vbase;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int kk = 8 * (i / 4) + i % 4;
      if (!QUAD || i % 4 == 0)
        first = vbase + __shfl(r.id, kk + 4 * half) * a.vp + __shfl(r.off, kk + 4 * half) * a.vr + vcol;
      const E* p = first + (QUAD ? (i % 4) * a.vr : 0);
#pragma unroll
      for (int w = 0; w < VW; ++w) v[i][w] = 0u;
      if ((there >> kk & 1) && vcol < a.d) {
        if constexpr (VW == 1) {
          v[i][0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (VW == 2) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(p);
          v[i][0] = x[0];
          v[i][1] = x[1];
        } else {
#pragma unroll
          for (int w = 0; w < VW; w += 4) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(p + w * (WIDE ? 1 : 2));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][w + e] = x[e];
          }
        }
      }
    }
  };

  int blk = blk0 + wave;
  KeyRow here = row_of(blk), then = row_of(blk + kWaves);
  // (fp32 rows of 256 columns: K and V of a block share registers, nothing is loaded ahead)
  constexpr bool LOAD_AHEAD = DP * sizeof(E) <= 512;
  if (LOAD_AHEAD && blk < blk1) {
    load_k(here);
    load_v(here);
  }
  while (blk < blk1) {
    if (!LOAD_AHEAD) load_k(here);
    const int next = blk + kWaves;
    const int key0 = blk * kKeys;
    const uint32_t there = static_cast<uint32_t>(__ballot(is_there(a, here)));  // (lanes 0 .. 31: the block's keys)
    f32x16 s = (f32x16)(0.f);
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < KC; ++i)
        if (2 * i * PIECE < a.d) {  // (256 cycles)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k[i][e]), __uint_as_float(q_piece(i)[e]), s, 0, 0, 0);
        }
    } else {
#pragma unroll
      for (int i = 0; i < KC; ++i) s = mfma16<T>(k[i], q_piece(i), s);
    }
    if (!LOAD_AHEAD)
      load_v(here);
    else if (next < blk1)
      load_k(then);
    // every row of the tile sees every key of the block?
    const bool full = there == 0xffffffffu && __all(!live || (rlo <= key0 && key0 + kKeys <= rhi));
    if (!full) {
      const int lo = rlo - key0 - 4 * half, hi = rhi - key0 - 4 * half;
      const uint32_t bits = there >> (4 * half);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int kk = 8 * (i / 4) + i % 4;
        if (!(kk >= lo && kk < hi && (bits >> kk & 1))) s[i] = kNegInf;
      }
    }
    float bm = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) bm = max2(bm, s[i], inf);
    bm = row_max(bm, inf);
    const float nm = fmaxf(mx, bm * c);
    const float to = nm == kNegInf ? 0.f : nm;  // (a row may have seen nothing yet)
    if (__any(nm > mx)) {
      const float f = __builtin_amdgcn_exp2f(mx - to);
      sum *= f;
#pragma unroll
      for (int m = 0; m < NB; ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[m][i] *= f;
      mx = nm;
      distant = any_far(mx);
    }
    float by = c, base = to - kLift<T>;
    if (distant) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = far_exponent(s[i], c, to, kLift<T>);
      by = 1.f;
      base = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(s[i] * by - base);
      sum += s[i];
    }

    // O^T += V^T P^T.  Where a key is hidden from some rows only, its weight
    // is 0 there, but 0 times an infinite or NaN value is not: in such a block
    // those values are taken out of V and added to the rows that see their key.
    if (!full) {
      uint32_t odd = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int w = 0; w < VW; ++w) odd |= infinite<T>(v[i][w]);
      if (__any((odd & Bits<T>::sign) != 0)) {
#pragma unroll 1
        for (int kk = 0; kk < kKeys; ++kk) {
          if (!(there >> kk & 1)) continue;
          const int key = key0 + kk;
          const bool sees = key >= rlo && key < rhi;
          const E* p = vbase + __shfl(here.id, kk) * a.vp + __shfl(here.off, kk) * a.vr;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int d = NB * (8 * (i / 4) + 4 * half + i % 4);
            if (sees && d < a.d) {
#pragma unroll
              for (int m = 0; m < NB; m += WIDE ? 1 : 2) {
                const uint32_t x = *reinterpret_cast<const uint32_t*>(p + d + m);
                const uint32_t f = infinite<T>(x) & Bits<T>::sign;
#pragma unroll
                for (int e = 0; e < (WIDE ? 1 : 2); ++e)
                  if (f >> (WIDE ? 31 : 15 + 16 * e) & 1) o[m + e][i] += value_of<T>(x, e);
              }
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
          for (int w = 0; w < VW; ++w) v[i][w] = finite_part<T>(v[i][w]);
      }
    }
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int m = 0; m < NB; ++m)
          o[m] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(v[i][m]), s[i], o[m], 0, 0, 0);
    } else {
      u32x4 p[2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) p[t][e] = pack2<T>(s[8 * t + 2 * e], s[8 * t + 2 * e + 1]);
#pragma unroll
      for (int m = 0; m < NB; ++m)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          u32x4 vt;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            vt[e] = interleave(v[8 * t + 2 * e][m / 2], v[8 * t + 2 * e + 1][m / 2], m % 2);
          o[m] = mfma16<T>(vt, p[t], o[m]);
        }
    }
    if (LOAD_AHEAD && next < blk1) load_v(then);
    here = then;
    then = row_of(next + kWaves);
    blk = next;
  }
  sum = row_sum(sum);

  // join the waves: a common maximum, then O in rounds, the upper half of the waves to the lower
  if (half == 0) {
    sh_ml[wave][0][col] = mx;
    sh_ml[wave][1][col] = sum;
  }
  __syncthreads();
  float M = kNegInf, L = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) M = fmaxf(M, sh_ml[w][0][col]);
  const float Mb = M == kNegInf ? 0.f : M;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) L += sh_ml[w][1][col] * __builtin_amdgcn_exp2f(sh_ml[w][0][col] - Mb);
  const float f = __builtin_amdgcn_exp2f(mx - Mb);
#pragma unroll
  for (int m = 0; m < NB; ++m)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[m][i] *= f;
#pragma unroll
  for (int r = kWaves / 2; r >= 1; r >>= 1) {
    if (wave >= r && wave < 2 * r) {
#pragma unroll
      for (int m = 0; m < NB; ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i) sh_o[wave - r][m * 16 + i][lane] = o[m][i];
    }
    __syncthreads();
    if (wave < r) {
#pragma unroll
      for (int m = 0; m < NB; ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[m][i] += sh_o[wave][m * 16 + i][lane];
    }
    __syncthreads();
  }
  if (wave != 0 || !live) return;

  if (it.splits > 1) {
    float* ws = static_cast<float*>(a.ws) + (static_cast<size_t>(it.part) * a.hkv + head) * part_floats(kRows, a.d);
    if (half == 0) {
      ws[col] = M;
      ws[kRows + col] = L;
    }
    float* wo = ws + 2 * kRows + static_cast<size_t>(col) * a.d;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int d = NB * (8 * (i / 4) + 4 * half + i % 4);
      if (d < a.d) {
#pragma unroll
        for (int m = 0; m < NB; ++m) wo[d + m] = o[m][i];
      }
    }
    return;
  }
  const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
  E* op = static_cast<E*>(a.o) + (static_cast<int64_t>(it.t0 + tok) * a.hq + head * a.group + gh) * a.d;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int d = NB * (8 * (i / 4) + 4 * half + i % 4);
    if (d < a.d) {
      if constexpr (WIDE) {
#pragma unroll
        for (int m = 0; m < NB; ++m) op[d + m] = o[m][i] * inv;
      } else {
        uint32_t* ow = reinterpret_cast<uint32_t*>(op + d);
#pragma unroll
        for (int m = 0; m < NB; m += 2) ow[m / 2] = pack2<T>(o[m][i] * inv, o[m + 1][i] * inv);
      }
    }
  }
}

template <typename T, int DP, bool QUAD>
__global__ __launch_bounds__(kThreads, (DP <= 128 && !Elem<T>::wide) ? 2 : 1) void paged_attn_stream(PagedAttnArgs a) {
  stream_item<T, DP, QUAD, kThreads / 64>(a, blockIdx.x);
}

// -------------------------------------------------------------- tile kernel ----
// Many rows of one sequence: a workgroup of WAVES waves takes 32 rows each and
// all walk over the same key blocks of 64, staged through LDS in two buffers: a
// block's rows are loaded straight to LDS while the one before it is worked on,
// with one barrier a block.  K rows are read as 16-byte pieces; V^T comes out of
// the row-major tile through the transposing LDS read (ds_read_b64_tr_b16: 16
// lanes read 4 keys x 16 columns and each gets one column's 4 keys).  Pieces of
// a row are stored at piece ^ turn(row), such that the 16 lanes of a read (K:
// 16 rows, one piece; V: 4 rows, 4 pieces) touch every bank once.
// Bound by the matrix unit and what the waves issue beside it (a block of 128 columns: a softmax of 32
// scores a lane, 48 LDS reads, the loads' addresses): 8192 tokens, 32 heads of 128 columns, bf16, causal: 540 to 570 us, 0.96 to 1.02
// PFLOP/s of the pairs that count, where a large matrix product reaches 1.15; 4096 tokens, 16 heads of
// 256 columns: 176 to 190 us, 0.72 to 0.78, the matrix unit busy for a third of the cycles: O, Q and the scores leave a
// SIMD one wave, whose softmax runs beside nobody's products; 8192 tokens, 32 heads of 64 columns: 342 us, 0.80 (as many exponentials for half
// the products).  Four pieces of V^T and six of K read ahead (two of V^T: 592 us, six: 582; four or eight of K: 578, 585).
constexpr int kTileKeys = 64;

// A row of 128 bytes shares the 256 bytes that the banks hold with its neighbour.
template <int DP>
__device__ __forceinline__ int turn(int row) {
  return (DP >= 128 ? row & 3 : row >> 1 & 1) << 2 | (row >> 2 & 3);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
#define NNSX_LDS __attribute__((address_space(3)))
#define NNSX_GLOBAL __attribute__((address_space(1)))

// Waves of a workgroup.  64 columns: three workgroups of 4 waves on a compute unit (by registers) are faster
// than one of 8 (8192 tokens, 32 heads: 342 us for 371; 4096, 16 kv heads: 75 for 93); 128 columns: one of 8 (8192 tokens,
// 32 heads: 551 us, 579 by two of 4, which share less; 700 and 512 tokens among single ones: 164 and 206, as only
// one fits beside the stream form's LDS); 256: one of 4, as O fills the registers of a SIMD's one wave.
template <int DP>
constexpr int kTileWaves = DP == 128 ? 8 : 4;
template <int DP>
constexpr int kTileRows = kTileWaves<DP> * kRows;

template <typename T, int DP, bool ONE_PAGE>
__device__ __forceinline__ void tile_item(const PagedAttnArgs& a, unsigned index) {
  using E = uint16_t;
  constexpr int WAVES = kTileWaves<DP>;
  constexpr int ROWS = WAVES * 32, NB = DP / 32, KC = DP / 16, P = DP / 8;
  constexpr int PASS = WAVES * 64 / P;       // rows of a block that the workgroup loads at once,
  constexpr int RUN = 64 / P;                // a wave's of them (1 KiB)
  constexpr int PASSES = kTileKeys / PASS;
  static_assert(PASS * PASSES == kTileKeys && RUN * P == 64 && PASSES <= 64, "tile");
  // K and V of two blocks, an array each: the compiler keeps them apart, so that a read of one
  // does not wait for the loads into another.  Rows are aligned to their size, so that pieces
  // of a row are reached by exclusive or.
  constexpr int ROW = DP * 2, TILE = kTileKeys * ROW;
  __shared__ __attribute__((aligned(1024))) char sh_k0[TILE], sh_k1[TILE], sh_v0[TILE], sh_v1[TILE];
  const int head = static_cast<int>(index % a.hkv);
  const int slot = static_cast<int>(index / a.hkv);
  const Item it = find_item<ROWS, kTileKeys, false>(a, slot);
  if (index == 0 && threadIdx.x == 0 && a.chunk != nullptr) *a.chunk = it.chunk;
  if (it.b < 0) return;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int rows = it.n * a.group;
  const int row = it.tile * ROWS + wave * 32 + col;
  const bool live = row < rows;
  const int tok = row / a.group, gh = row - tok * a.group;
  // keys that this lane's row sees; that some row of the tile sees; that every
  // row of the tile (t_in) and of the wave (w_in) sees
  int rlo, rhi, tlo, thi, t_in_lo, t_in_hi, w_in_lo = 0, w_in_hi = 0x7fffffff, x;
  key_range(a, it, tok, tok, &rlo, &rhi);
  if (!live) rhi = rlo = 0;
  {
    const int f = it.tile * ROWS, l = min(f + ROWS, rows) - 1;
    key_range(a, it, f / a.group, l / a.group, &tlo, &thi);
    key_range(a, it, f / a.group, f / a.group, &x, &t_in_hi);
    key_range(a, it, l / a.group, l / a.group, &t_in_lo, &x);
    const int wf = f + wave * 32, wl = min(wf + 32, rows) - 1;
    if (wf < rows) {  // (else nothing of the wave matters)
      key_range(a, it, wf / a.group, wf / a.group, &x, &w_in_hi);
      key_range(a, it, wl / a.group, wl / a.group, &w_in_lo, &x);
    }
  }
  int blk0 = tlo / kTileKeys, blk1 = (thi + kTileKeys - 1) / kTileKeys;
  {
    const int64_t s0 = blk0 + static_cast<int64_t>(it.split) * it.chunk;
    const int64_t s1 = s0 + it.chunk;
    blk0 = static_cast<int>(min(s0, static_cast<int64_t>(blk1)));
    blk1 = static_cast<int>(min(s1, static_cast<int64_t>(blk1)));
  }

  const E* qp = static_cast<const E*>(a.q) + static_cast<int64_t>(it.t0 + tok) * a.qt +
                static_cast<int64_t>(head * a.group + gh) * a.qh;
  const E* kbase = static_cast<const E*>(a.k) + head * a.kh;
  const E* vbase = static_cast<const E*>(a.v) + head * a.vh;
  const int* table = a.p.table + static_cast<int64_t>(it.b) * a.p.tstride;

  u32x4 q[KC];
#pragma unroll
  for (int s = 0; s < KC; ++s) {
    const int d = (2 * s + half) * 8;
    q[s] = (u32x4)(0u);
    if (live && d < a.d) q[s] = *reinterpret_cast<const u32x4*>(qp + d);
  }
  f32x16 o[NB];
#pragma unroll
  for (int m = 0; m < NB; ++m) o[m] = (f32x16)(0.f);
  float mx = kNegInf, sum = 0.f;
  int distant = 0;  // some row's maximum is
  const float c = a.scale * kLog2e, inf = opaque_infinity();

  if (a.p.pages == 0) blk1 = blk0;
  const int keys1 = min(it.keys, blk1 * kTileKeys);
  // Does the table name a page that is not there, among the item's?  (Hardly ever: then blocks are looked over one by one.)
  bool missing = false;
  if (blk0 < blk1) {
    for (int p = blk0 * kTileKeys / a.p.page + threadIdx.x; p <= (keys1 - 1) / a.p.page; p += WAVES * 64)
      missing |= static_cast<uint32_t>(table[p]) >= static_cast<uint32_t>(a.p.pages);
    missing = __syncthreads_or(missing);
  }
  auto there_of = [&](int blk) {
    const int key = blk * kTileKeys + lane;
    return __ballot(key >= keys1 || static_cast<uint32_t>(table[key / a.p.page]) < static_cast<uint32_t>(a.p.pages));
  };

  // This wave's loads: in every pass the RUN rows from i PASS + wave RUN on; lane: slot lane % P
  // of LDS row lane / P, which holds piece (lane % P) ^ turn.  A row behind the last key or of a
  // page that is not there is some other row of the cache: its key is hidden from every row of the tile.
  const int lrow = lane / P;
  const int piece[2] = {(lane % P) ^ turn<DP>(wave * RUN + lrow), (lane % P) ^ turn<DP>(PASS + wave * RUN + lrow)};
  auto piece_of = [&](int i) { return piece[i % 2]; };  // (the turn repeats every 16 rows, two passes at most)
  static_assert(PASS % 16 == 0 || 2 * PASS % 16 == 0, "tile");
  const int last_page = blk0 < blk1 ? (keys1 - 1) / a.p.page : 0;
  // ONE_PAGE: the rows of a run share a page; lane i looks after pass i.  Else every lane after its
  // own rows, of every pass.  (4096 tokens after none, 16 heads of 256 columns, 8 passes: 191 us, 205 us by
  // the latter; of 128 columns and less, 1 or 2 passes, the latter is as fast and the only one.)
  constexpr int WALKS = ONE_PAGE ? 1 : PASSES;
  int walk_p[WALKS], walk_off[WALKS], id[WALKS], off[WALKS];
  const int dp = kTileKeys / a.p.page, doff = kTileKeys - dp * a.p.page;
#pragma unroll
  for (int i = 0; i < WALKS; ++i) {
    const int key = blk0 * kTileKeys + wave * RUN + (ONE_PAGE ? lane % PASSES * PASS : i * PASS + lrow);
    walk_p[i] = key / a.p.page;
    walk_off[i] = key - walk_p[i] * a.p.page;
  }
  auto fetch = [&]() __attribute__((always_inline)) {  // page ids of the next block
#pragma unroll
    for (int i = 0; i < WALKS; ++i) {
      id[i] = table[min(walk_p[i], last_page)];
      off[i] = walk_off[i];
      walk_p[i] += dp;
      walk_off[i] += doff;
      if (walk_off[i] >= a.p.page) {
        walk_off[i] -= a.p.page;
        ++walk_p[i];
      }
    }
  };
  const uint32_t page_k = static_cast<uint32_t>(a.kp) * 2, row_k = static_cast<uint32_t>(a.kr) * 2;  // bytes
  const uint32_t page_v = static_cast<uint32_t>(a.vp) * 2, row_v = static_cast<uint32_t>(a.vr) * 2;
  uint64_t from_k[WALKS], from_v[WALKS];
  auto locate = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < WALKS; ++i) {
      const uint32_t x = static_cast<uint32_t>(id[i]) < static_cast<uint32_t>(a.p.pages) ? id[i] : 0;
      from_k[i] = reinterpret_cast<uint64_t>(kbase) + static_cast<uint64_t>(x) * page_k + static_cast<uint64_t>(static_cast<uint32_t>(off[i])) * row_k;
      from_v[i] = reinterpret_cast<uint64_t>(vbase) + static_cast<uint64_t>(x) * page_v + static_cast<uint64_t>(static_cast<uint32_t>(off[i])) * row_v;
    }
  };
  const uint32_t lane_k = ONE_PAGE ? lrow * row_k : 0, lane_v = ONE_PAGE ? lrow * row_v : 0;
  auto load = [&](char* to, const uint64_t* from, uint32_t lane_off) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      uint64_t x = from[ONE_PAGE ? 0 : i];
      if constexpr (ONE_PAGE)
        x = static_cast<uint64_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(x >> 32), i)) << 32 |
            static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(x), i));
      const char* p = reinterpret_cast<const char*>(x) + (lane_off + piece_of(i) * 16);
      if (piece_of(i) * 8 < a.d)  // (else the piece stays 0)
        __builtin_amdgcn_global_load_lds((const NNSX_GLOBAL void*)p, (NNSX_LDS void*)(to + (i * WAVES + wave) * 1024), 16, 0, 0);
    }
  };
  // Addresses to read in a buffer
  const uint32_t kread = col * ROW + ((half ^ turn<DP>(col)) << 4);
  const int vrow = 4 * half + (lane & 15) / 4, vx = 2 * (lane >> 4 & 1) + (lane & 3) / 2;
  uint32_t vread[2];
#pragma unroll
  for (int g = 0; g < 2; ++g)
    vread[g] = (vrow + 8 * g) * ROW + ((vx ^ turn<DP>(vrow + 8 * g)) << 4) + (lane & 1) * 8;

  // A hidden key's weight is 0, but 0 times an infinite or NaN value is not: in
  // a block that hides a key from some row, those values are added to the rows
  // that see their key and taken out of the block.
  auto take_infinite = [&](char* v, int key0, uint64_t there) __attribute__((always_inline)) {
    uint32_t odd = 0;
    for (int i = threadIdx.x; i < TILE / 4; i += WAVES * 64) odd |= infinite<T>(reinterpret_cast<uint32_t*>(v)[i]);
    if (!__syncthreads_or((odd & Bits<T>::sign) != 0)) return;
#pragma unroll 1
    for (int kk = 0; kk < kTileKeys; ++kk) {
      const bool sees = key0 + kk >= rlo && key0 + kk < rhi && (there >> kk & 1);
#pragma unroll
      for (int m = 0; m < NB; ++m)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const int d = 32 * m + 8 * (i / 4) + 4 * half + i % 4;
          const uint32_t x = *reinterpret_cast<const uint32_t*>(v + kk * ROW + ((d / 8 ^ turn<DP>(kk)) << 4) + d % 8 * 2);
          const uint32_t f = sees ? infinite<T>(x) & Bits<T>::sign : 0u;
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (f >> (15 + 16 * e) & 1) o[m][i + e] += value_of<T>(x, e);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < TILE / 4; i += WAVES * 64) {
      uint32_t* w = reinterpret_cast<uint32_t*>(v) + i;
      *w = finite_part<T>(*w);
    }
    __syncthreads();
  };

  // Block blk from k and v, while the next one is loaded to kn and vn
  auto step = [&](char* k, char* v, char* kn, char* vn, int blk) __attribute__((always_inline)) {
    const int key0 = blk * kTileKeys;
    __builtin_amdgcn_s_waitcnt(0x0f70);  // this wave's loads of the block have arrived (vmcnt 0)
    __syncthreads();                     // every wave's have, and the other buffers are read
    locate();
    load(kn, from_k, lane_k);
    f32x16 s[2];
    constexpr int NK = 2 * KC, AHEAD = 6;  // matrix instructions of the scores, pieces of K read ahead
    u32x4 kf[AHEAD];
    auto read_k = [&](int j) __attribute__((always_inline)) {
      kf[j % AHEAD] = *reinterpret_cast<const u32x4*>(k + ((kread ^ (j / 2) << 5) + j % 2 * 32 * ROW));
    };
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) read_k(j);
    s[0] = s[1] = (f32x16)(0.f);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      s[j % 2] = mfma16<T>(kf[j % AHEAD], q[j / 2], s[j % 2]);
      if (j + AHEAD < NK) read_k(j + AHEAD);
      __builtin_amdgcn_sched_barrier(0);
    }
    uint64_t there = ~0ull;
    if (missing) there = there_of(blk);
    load(vn, from_v, lane_v);
    fetch();
    if (there != ~0ull || key0 < w_in_lo || key0 + kTileKeys > w_in_hi) {
      const int lo = rlo - key0 - 4 * half, hi = rhi - key0 - 4 * half;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint32_t bits = static_cast<uint32_t>(there >> (32 * b)) >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int kk = 8 * (i / 4) + i % 4;
          if (!(32 * b + kk >= lo && 32 * b + kk < hi && (bits >> kk & 1))) s[b][i] = kNegInf;
        }
      }
    }
    float bm = max2(s[0][0], s[1][0], inf);
#pragma unroll
    for (int i = 1; i < 15; i += 2) bm = max3(bm, max2(s[0][i], s[1][i], inf), max2(s[0][i + 1], s[1][i + 1], inf));
    const float nm = fmaxf(mx, row_max(max2(bm, max2(s[0][15], s[1][15], inf), inf), inf) * c);
    // the maximum that weights are relative to follows only steps of more than
    // 2^8: weights stay within [0, 2^15 and a sixteenth], inside every type's range, and the
    // rescale of O is rare (8192 tokens, 32 heads of 128 columns: 580 us, 605 us with every step followed)
    if (__any(nm > mx + (distant ? 0.f : 8.f))) {
      const float f = __builtin_amdgcn_exp2f(mx - (nm == kNegInf ? 0.f : nm));
      sum *= f;
#pragma unroll
      for (int m = 0; m < NB; ++m)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[m][i] *= f;
      mx = nm;
      distant = __builtin_amdgcn_readfirstlane(any_far(mx));
    }
    if (there != ~0ull || key0 < t_in_lo || key0 + kTileKeys > t_in_hi) take_infinite(v, key0, there);
    float by = c, base = (mx == kNegInf ? 0.f : mx) - kLift<T>;  // (a row may have seen nothing yet)
    if (distant) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][i] = far_exponent(s[b][i], c, mx == kNegInf ? 0.f : mx, kLift<T>);
      by = 1.f;
      base = 0.f;
    }
    u32x4 p[4];
    auto weigh = [&](int t) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          w[h] = __builtin_amdgcn_exp2f(s[t / 2][8 * (t % 2) + 2 * e + h] * by - base);
          sum += w[h];
        }
        p[t][e] = pack2<T>(w[0], w[1]);
      }
    };
    constexpr int NV = 4 * NB, VAHEAD = 4;  // matrix instructions of the values, pieces of V^T read ahead
    u32x4 vf[VAHEAD];
    auto read_v = [&](int j) __attribute__((always_inline)) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (NNSX_LDS s16x4*)(v + ((vread[g] ^ (j % NB) << 6) + j / NB * 16 * ROW))));
        vf[j % VAHEAD][2 * g] = x[0];
        vf[j % VAHEAD][2 * g + 1] = x[1];
      }
    };
#pragma unroll
    for (int j = 0; j < VAHEAD; ++j) read_v(j);
    weigh(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int m = 0; m < NB; ++m) {
        const int j = t * NB + m;
        o[m] = mfma16<T>(vf[j % VAHEAD], p[t], o[m]);
        if (j + VAHEAD < NV) read_v(j + VAHEAD);
      }
      if (t < 3) weigh(t + 1);  // (while the matrix unit works)
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // (columns from d on are never loaded: they stay 0)
  for (int i = threadIdx.x; i < TILE / 16; i += WAVES * 64)
    for (char* x : {sh_k0, sh_k1, sh_v0, sh_v1}) reinterpret_cast<u32x4*>(x)[i] = (u32x4)(0u);
  if (blk0 < blk1) {
    fetch();
    __syncthreads();
    locate();
    load(sh_k0, from_k, lane_k);
    load(sh_v0, from_v, lane_v);
    fetch();
  }
  for (int blk = blk0; blk < blk1; blk += 2) {
    step(sh_k0, sh_v0, sh_k1, sh_v1, blk);
    if (blk + 1 >= blk1) break;
    step(sh_k1, sh_v1, sh_k0, sh_v0, blk + 1);
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // (the last block loaded one too many)
  sum = row_sum(sum);
  if (!live) return;

  if (it.splits > 1) {
    float* ws = static_cast<float*>(a.ws) + (static_cast<size_t>(it.part) * a.hkv + head) * part_floats(ROWS, a.d);
    const int r = wave * 32 + col;
    if (half == 0) {
      ws[r] = mx;
      ws[ROWS + r] = sum;
    }
    float* wo = ws + 2 * ROWS + static_cast<size_t>(r) * a.d;
#pragma unroll
    for (int m = 0; m < NB; ++m)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int d = 32 * m + 2 * i + 4 * half;
        if (d < a.d) *reinterpret_cast<f32x4*>(wo + d) = (f32x4){o[m][i], o[m][i + 1], o[m][i + 2], o[m][i + 3]};
      }
    return;
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  E* op = static_cast<E*>(a.o) + (static_cast<int64_t>(it.t0 + tok) * a.hq + head * a.group + gh) * a.d;
#pragma unroll
  for (int m = 0; m < NB; ++m)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int d = 32 * m + 2 * i + 4 * half;
      if (d < a.d)
        *reinterpret_cast<u32x2*>(op + d) = (u32x2){pack2<T>(o[m][i] * inv, o[m][i + 1] * inv),
                                                    pack2<T>(o[m][i + 2] * inv, o[m][i + 3] * inv)};
    }
}

template <typename T, int DP, bool ONE_PAGE>
__global__ __launch_bounds__(kTileWaves<DP> * 64, DP <= 64 ? 3 : DP <= 128 ? 2 : 1) void paged_attn_tile(PagedAttnArgs a) {
  tile_item<T, DP, ONE_PAGE>(a, blockIdx.x);
}

// A batch of long and short pieces: the tile form's items first, the stream form's after them, one launch.
// (700 tokens, 512 after 8488, 14 sequences of 1 and 5 tokens: 163 us with the join; the two long ones alone
// 131 us, the others alone 42 us.  What is left is the tiles of unequal lengths, which the splits take as alike.)
template <typename T, int DP, bool QUAD>
__global__ __launch_bounds__(kTileWaves<DP> * 64, DP <= 64 ? 3 : 2) void paged_attn_both(PagedAttnArgs t, PagedAttnArgs s, unsigned tiles) {
  if (blockIdx.x < tiles)
    tile_item<T, DP, false>(t, blockIdx.x);
  else
    stream_item<T, DP, QUAD, kTileWaves<DP>>(s, blockIdx.x - tiles);
}

// ------------------------------------------------------------------- join ----
// Joins the splits of one (sequence, tile, kv head):
//   M = max_s m_s,  o = sum_s e^(m_s - M) o_s / sum_s e^(m_s - M) l_s.
// LG lanes hold a row's columns, four each; the workgroup's 256 / LG such
// groups divide the live rows and, where there are few, a row's splits, whose
// parts are added through LDS in a fixed order.  A pair's rows are dealt out to
// a.apart workgroups: few pairs are spread over more of the card.  4 to 7 us, a launch, the plan and a round
// trip; 13 us for the tiles of that mixed batch.
constexpr int kJoinThreads = 256;

template <typename T, int ROWS, int KEYS, int LG>
__device__ __forceinline__ void join_pair(const PagedAttnArgs& a, unsigned index) {
  using E = typename Elem<T>::type;
  constexpr int NG = kJoinThreads / LG;
  __shared__ f32x4 sh_o[NG][LG];
  __shared__ float sh_ml[NG][2];
  const int apart = a.apart, mine = static_cast<int>(index % apart);
  const int head = static_cast<int>(index / apart % a.hkv);
  const Item it = find_item<ROWS, KEYS, true>(a, static_cast<int>(index / apart / a.hkv));
  if (it.b < 0 || it.splits == 1) return;
  const int lg = threadIdx.x % LG, grp = threadIdx.x / LG;
  const int all = min(it.n * a.group - it.tile * ROWS, ROWS);
  const int live = (all - mine + apart - 1) / apart;  // rows of this workgroup
  if (live <= 0) return;
  int per_row = NG;  // groups of a row: a power of two
  while (per_row > 1 && per_row * live > NG) per_row >>= 1;
  const int rows_at_once = NG / per_row, part = grp % per_row;
  const size_t step = static_cast<size_t>(a.hkv) * part_floats(ROWS, a.d);
  const float* ws = static_cast<const float*>(a.ws) + (static_cast<size_t>(it.part) * a.hkv + head) * part_floats(ROWS, a.d);
  for (int r0 = 0; r0 < live; r0 += rows_at_once) {
    const int i0 = r0 + grp / per_row, r = i0 * apart + mine;
    f32x4 acc = (f32x4)(0.f);
    float M = kNegInf, L = 0.f;
    if (i0 < live) {
      // some splits at a time: all their loads first, then one step of the running maximum
      constexpr int U = 8;
      for (int s0 = part; s0 < it.splits; s0 += U * per_row) {
        float m[U], l[U];
        f32x4 x[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
          m[i] = kNegInf;
          l[i] = 0.f;
          x[i] = (f32x4)(0.f);
          const int s = s0 + i * per_row;
          if (s < it.splits) {
            const float* w = ws + s * step;
            m[i] = w[r];
            l[i] = w[ROWS + r];
            if (4 * lg < a.d) x[i] = *reinterpret_cast<const f32x4*>(w + 2 * ROWS + static_cast<size_t>(r) * a.d + 4 * lg);
          }
        }
        float nm = M;
#pragma unroll
        for (int i = 0; i < U; ++i) nm = fmaxf(nm, m[i]);
        const float base = nm == kNegInf ? 0.f : nm, f = __builtin_amdgcn_exp2f(M - base);
        M = nm;
        L *= f;
        acc *= f;
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const float g = __builtin_amdgcn_exp2f(m[i] - base);
          L += g * l[i];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] += g * x[i][e];
        }
      }
    }
    if (per_row > 1) {  // (the same in every thread)
      __syncthreads();
      sh_o[grp][lg] = acc;
      if (lg == 0) {
        sh_ml[grp][0] = M;
        sh_ml[grp][1] = L;
      }
      __syncthreads();
      if (part == 0) {
        float nm = M;
        for (int i = 1; i < per_row; ++i) nm = fmaxf(nm, sh_ml[grp + i][0]);
        const float base = nm == kNegInf ? 0.f : nm, f = __builtin_amdgcn_exp2f(M - base);
        L *= f;
        acc *= f;
        for (int i = 1; i < per_row; ++i) {
          const float g = __builtin_amdgcn_exp2f(sh_ml[grp + i][0] - base);
          L += g * sh_ml[grp + i][1];
          const f32x4 x = sh_o[grp + i][lg];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] += g * x[e];
        }
      }
    }
    if (part != 0 || i0 >= live || 4 * lg >= a.d) continue;
    const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
    const int row = it.tile * ROWS + r, tok = row / a.group, gh = row - tok * a.group;
    E* op = static_cast<E*>(a.o) + (static_cast<int64_t>(it.t0 + tok) * a.hq + head * a.group + gh) * a.d + 4 * lg;
    if constexpr (Elem<T>::wide)
      *reinterpret_cast<f32x4*>(op) = (f32x4){acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
    else
      *reinterpret_cast<u32x2*>(op) = (u32x2){pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv)};
  }
}

template <int TILE_ROWS>
__global__ __launch_bounds__(kPlanThreads) void paged_attn_plan(PagedAttnArgs t, PagedAttnArgs s) {
  if (blockIdx.x == 0) {
    if (s.plan != nullptr) make_plan<kRows, kKeys>(s);
  } else {
    if (t.plan != nullptr) make_plan<TILE_ROWS, kTileKeys>(t);
  }
}

// `tiles` workgroups for the tile form's pairs, then the stream form's
template <typename T, int TILE_ROWS, int LG>
__global__ __launch_bounds__(kJoinThreads) void paged_attn_join(PagedAttnArgs t, PagedAttnArgs s, unsigned tiles) {
  if constexpr (TILE_ROWS > 0) {
    if (blockIdx.x < tiles) return join_pair<T, TILE_ROWS, kTileKeys, LG>(t, blockIdx.x);
  }
  join_pair<T, kRows, kKeys, LG>(s, blockIdx.x - tiles);
}

// (60 tokens after 8192, 8 heads of 128 columns: 371 us, 394 us with every row of V addressed by itself)
template <typename T, int DP>
void launch_stream(const PagedAttnArgs& a, unsigned grid, hipStream_t s) {
  if (a.p.page % 4 == 0)
    paged_attn_stream<T, DP, true><<<grid, kThreads, 0, s>>>(a);
  else
    paged_attn_stream<T, DP, false><<<grid, kThreads, 0, s>>>(a);
}

template <typename T, int DP>
void launch_tile(const PagedAttnArgs& a, unsigned grid, hipStream_t s) {
  constexpr int threads = kTileWaves<DP> * 64;
  if (DP > 128 && a.p.page % (512 / DP) == 0)  // (the keys of 1 KiB)
    paged_attn_tile<T, DP, (DP > 128)><<<grid, threads, 0, s>>>(a);
  else
    paged_attn_tile<T, DP, false><<<grid, threads, 0, s>>>(a);
}

// (sequence, tile) pairs a call can have: every sequence, and the rows behind the last, may end in a partial tile
int64_t pairs_bound(const PagedAttnArgs& a, int rows) {
  return static_cast<int64_t>(a.p.T) * a.group / rows + std::min<int64_t>(a.p.B + 1, a.p.T);
}

int tile_rows(const PagedAttnArgs& a) { return a.d <= 64 ? kTileRows<64> : a.d <= 128 ? kTileRows<128> : kTileRows<256>; }

// Either form's part of a call: which sequences it takes (by their rows), and
// how its keys are split: for about `target` items a kv head (0: no split), of at least `min_chunk` key blocks.
PagedAttnArgs part_of(const PagedAttnArgs& a0, int rows, int64_t pairs, int rows_lo, int rows_hi, int target, int min_chunk) {
  PagedAttnArgs a = a0;
  // (no more items than the longest sequence that the tables can hold gives each pair)
  const int keys = rows == kRows ? kKeys : kTileKeys, blocks = (a.p.width * a.p.page + keys - 1) / keys;
  const int most = std::max((blocks + min_chunk - 1) / min_chunk, 1);
  a.rows_lo = rows_lo;
  a.rows_hi = rows_hi;
  a.target = most > 1 ? (target + a.hkv - 1) / a.hkv : 0;
  a.min_chunk = min_chunk;
  a.pairs = static_cast<int>(pairs);
  a.slots = static_cast<int>(std::min<int64_t>(pairs + a.target, pairs * most));
  a.parts = std::min(2 * a.target, a.slots);  // (items of split pairs)
  a.apart = static_cast<int>(std::clamp<int64_t>(rows / kRows * 4 * kCus / (static_cast<int64_t>(a.pairs) * a.hkv), 1,
                                                 rows > kRows ? rows / 32 : kRows));
  return a;
}

size_t part_bytes(const PagedAttnArgs& a, int rows) {
  return static_cast<size_t>(a.parts) * a.hkv * part_floats(rows, a.d) * sizeof(float);
}

// workgroups of the tile form, or of both, that a compute unit holds
int tile_units(const PagedAttnArgs& a) { return a.d <= 64 ? 3 : 1; }

// Sequences from which on a plan is made
constexpr int kPlanned = 64;  // (find_item: a lane for each, and the rows behind the last)
size_t plan_bytes(const PagedAttnArgs& a) { return (static_cast<size_t>(a.p.B) + 2) * sizeof(PlanEntry); }

constexpr int kAllRows = 0x7fffffff;
// Rows of a sequence up to which the stream form takes it: one item's.  (30 x 16 tokens, 64 rows, beside 2 x 1024,
// all after 4096: 289 us; 397 us if the stream form takes them, which then reads each key twice.)
constexpr int kStreamRows = 32;

struct Plan {
  bool stream, tile;
  PagedAttnArgs s, t;
};

Plan plan_of(PagedAttnArgs a) {
  a.group = a.hq / a.hkv;
  Plan p;
  const int64_t rows = static_cast<int64_t>(a.p.T) * a.group;
  // Measured with 32 query and 8 kv heads of 128 columns (rows = 4 times the tokens), us.
  // One sequence: up to 32 rows the stream form (8 tokens after 65536: 54, tile form 79), beyond the
  // tile form (9 tokens: 81, stream form 80; 32 tokens: 96, 180).
  // Several: as many tokens as sequences (single tokens, as a rule), or no more rows than one tile has:
  // the stream form takes all (8 single tokens after 4096: 34, 40 by both; 2 x 16 tokens
  // after 8192: 33, 37).  Else both run, each on its own sequences (8 x 16 tokens after 4096: 58, stream form 71).
  // Single tokens with rows of padding behind them run both, with fewer splits (64 tokens after 2048: 107 without padding,
  // 124 with 1 to 64 rows of it; 64 after 100 to 8192: 224 and 253; 8 after 4096: 38 either way), and a chunk among as
  // many tokens as slots takes the stream form (200 tokens after 4096, 56 single ones, 199 empty slots: 122; 119
  // by both, with one row more).
  if (a.type == AttnType::kF32)
    p.tile = false;
  else if (a.p.B == 1)
    p.tile = rows > kStreamRows;
  else
    p.tile = a.p.T != a.p.B && rows > tile_rows(a);
  p.stream = !p.tile || a.p.B > 1;
  // The stream form always splits: a sequence much longer than the others is spread over the card.  Up to 6 items a
  // compute unit, of which the rounds decide (60 single tokens after 8192: 362 us, always 2 a unit 516 us, as
  // 480 items are nearly a round already; 8 after 4096: 35 us, always 8 a unit 48 us; 1 after 131072: 105 and
  // 125 us; 64 after 1024: 54 and 70 us).  One workgroup of 256 columns fills a unit's registers, and each has
  // twice the rows to join: 2 (64 single tokens after 2048, 4 heads: 110 us, 192 us by 8; 128 us by 3).
  const int per_cu = p.tile ? 2 * tile_units(a) : a.type == AttnType::kF32 ? 3 : a.d > 128 ? 2 : 6;
  const int64_t pairs = p.tile ? static_cast<int64_t>(a.p.B) + 1 : pairs_bound(a, kRows);  // (with the tile form: one a sequence)
  p.s = part_of(a, kRows, pairs, 0, p.tile ? kStreamRows : kAllRows, per_cu * kCus, p.tile ? 8 : 4);
  const int units = p.tile ? tile_units(a) : a.d > (a.type == AttnType::kF32 ? 64 : 128) ? 1 : 2;
  p.s.one_round = (units * kCus + a.hkv - 1) / a.hkv;
  p.s.item_cost = a.type == AttnType::kF32 ? 6 : 12;
  // The tile form splits where whole tiles do not fill the card (1300 tokens after 8192, 168 tiles: 212 us,
  // 317 us whole; 3600 tokens after 16384, 456 tiles: 852 us, 1065 us if those split too: a
  // split's rows go through memory twice).  Splits of less than 8 blocks cost more than they give
  // (4 x 100 tokens alone: 25.7 us, 29.1 us with splits of 4).
  // 64 columns and less: three times as many tiles fill it, but from twice as many on whole ones are faster
  // (4096 tokens, 16 heads: 75 us, 90 us split; 1500 tokens after 16384: 281 us, 330 us whole).
  const int64_t tiles = (rows + tile_rows(a) - 1) / tile_rows(a) * a.hkv;
  const int slots = tile_units(a) * kCus, full = std::min(slots, 2 * kCus);
  p.t = part_of(a, tile_rows(a), pairs_bound(a, tile_rows(a)), p.stream ? kStreamRows : 0, kAllRows,
                tiles >= full ? 0 : 2 * slots, 8);
  p.t.one_round = (slots + a.hkv - 1) / a.hkv;
  p.t.item_cost = 8;
  char* ws = static_cast<char*>(a.ws) + (p.stream ? part_bytes(p.s, kRows) : 0);
  p.t.ws = ws;
  ws += p.tile ? part_bytes(p.t, tile_rows(a)) : 0;
  p.s.plan = p.t.plan = nullptr;
  p.s.chunk = p.t.chunk = nullptr;
  if (a.p.B >= kPlanned) {
    if (p.stream) p.s.plan = ws;
    if (p.tile) p.t.plan = ws + plan_bytes(a);
  } else {
    if (p.stream && p.s.target > 0) p.s.chunk = reinterpret_cast<int*>(ws);
    if (p.tile && p.t.target > 0) p.t.chunk = reinterpret_cast<int*>(ws) + 1;
  }
  return p;
}

unsigned grid_of(const PagedAttnArgs& a) { return static_cast<unsigned>(static_cast<int64_t>(a.slots) * a.hkv); }

template <typename T, int DP>
void launch_join(const Plan& p, hipStream_t s) {
  const auto wgs = [](bool runs, const PagedAttnArgs& a) {
    return runs && a.target > 0 ? static_cast<unsigned>(static_cast<int64_t>(a.pairs) * a.hkv * a.apart) : 0u;
  };
  const unsigned tiles = wgs(p.tile, p.t), grid = tiles + wgs(p.stream, p.s);
  if (grid > 0) paged_attn_join<T, Elem<T>::wide ? 0 : kTileRows<DP>, DP / 4><<<grid, kJoinThreads, 0, s>>>(p.t, p.s, tiles);
}

template <typename T, int DP>
void launch_both(const Plan& p, hipStream_t s) {
  const unsigned tiles = grid_of(p.t), grid = tiles + grid_of(p.s);
  constexpr int threads = kTileWaves<DP> * 64;
  if (p.t.p.page % 4 == 0)
    paged_attn_both<T, DP, true><<<grid, threads, 0, s>>>(p.t, p.s, tiles);
  else
    paged_attn_both<T, DP, false><<<grid, threads, 0, s>>>(p.t, p.s, tiles);
}

template <typename T, int DP>
void launch(const Plan& p, hipStream_t s) {
  if (p.s.p.B >= kPlanned)
    paged_attn_plan<Elem<T>::wide ? kRows : kTileRows<DP>><<<p.tile ? 2 : 1, kPlanThreads, 0, s>>>(p.t, p.s);
  if constexpr (!Elem<T>::wide) {
    if constexpr (DP <= 128) {
      if (p.tile && p.stream) {
        launch_both<T, DP>(p, s);
        return launch_join<T, DP>(p, s);
      }
    }  // (else the two forms' LDS does not fit one workgroup)
    if (p.tile) launch_tile<T, DP>(p.t, grid_of(p.t), s);
  }
  if (p.stream) launch_stream<T, DP>(p.s, grid_of(p.s), s);
  launch_join<T, DP>(p, s);
}

template <typename T>
void launch(const Plan& p, hipStream_t s) {
  if (p.s.d <= 64)
    launch<T, 64>(p, s);
  else if (p.s.d <= 128)
    launch<T, 128>(p, s);
  else
    launch<T, 256>(p, s);
}

}  // namespace

size_t paged_attn_workspace_bytes(const PagedAttnArgs& a) {
  const Plan p = plan_of(a);
  const size_t parts = (p.stream ? part_bytes(p.s, kRows) : 0) + (p.tile ? part_bytes(p.t, tile_rows(a)) : 0);
  return parts + (a.p.B >= kPlanned ? 2 * plan_bytes(a) : parts > 0 ? 2 * sizeof(int) : 0);
}

void paged_attn(const PagedAttnArgs& a, hipStream_t s) {
  const Plan p = plan_of(a);
  if (a.type == AttnType::kBF16)
    launch<BF16>(p, s);
  else if (a.type == AttnType::kF16)
    launch<F16>(p, s);
  else
    launch<F32>(p, s);
}

}  // namespace kernels
}  // namespace nnsx
