// Norm of queries and keys for each head with the position rotation in the same
// pass, its gradient, and the same rows appended to a paged cache, gfx950.
//
//   r = 1 / sqrt(mean_d x_d^2 + eps),  u_d = w_d x_d r,
//   y = R(p) u:  (y_a, y_b) = (u_a cos t - u_b sin t, u_b cos t + u_a sin t)
//
// for the pairs (a, b) = (i, i + rot / 2), or (2 i, 2 i + 1) when interleaved,
// with cos t and sin t of position p and pair i from a table; what lies behind
// the first rot columns is not turned.  Backward, with h = R(-p) gy:
//
//   dw_d = sum_rows h_d x_d r,   dx_d = r (w_d h_d - x_d r^2 mean_e(w_e h_e x_e)).
//
// Everything is computed in fp32 and rounded once, at the store.
//
// The kernels move bytes: a row is read once and written once.  A lane holds
// two pieces of VEC neighbouring columns such that both members of each of its
// pairs are its own (piece i and the piece rot / 2 columns further), so the
// rotation needs no exchange and the norm one butterfly over the LPR lanes of
// a row.  A workgroup is one token: the lanes of all its heads.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "kernels/attn.h"

namespace nnsx {
namespace kernels {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct BF16 { using E = uint16_t; };
struct F16 { using E = uint16_t; };
struct F32 { using E = float; };

template <typename T>
__device__ __forceinline__ f32x2 unpack2(uint32_t x);
template <>
__device__ __forceinline__ f32x2 unpack2<BF16>(uint32_t x) {
  return (f32x2){__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)};
}
template <>
__device__ __forceinline__ f32x2 unpack2<F16>(uint32_t x) {
  return __builtin_convertvector(__builtin_bit_cast(f16x2, x), f32x2);
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

template <typename T, int VEC>
__device__ __forceinline__ void load_piece(const typename T::E* p, float* x) {
  if constexpr (sizeof(typename T::E) == 4) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(p + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i + e] = v[e];
    }
  } else {
    uint32_t w[VEC / 2];
    if constexpr (VEC == 8) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = v[e];
    } else {
      const u32x2 v = *reinterpret_cast<const u32x2*>(p);
      w[0] = v[0];
      w[1] = v[1];
    }
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) {
      const f32x2 v = unpack2<T>(w[e]);
      x[2 * e] = v[0];
      x[2 * e + 1] = v[1];
    }
  }
}

// A piece as loaded: several can be under way before the first is unpacked
template <typename T, int VEC>
struct Raw {
  static constexpr int W = VEC * sizeof(typename T::E) / 4;
  uint32_t w[W];
  __device__ __forceinline__ void load(const typename T::E* p) {
    if constexpr (W == 4) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = v[e];
    } else {
      const u32x2 v = *reinterpret_cast<const u32x2*>(p);
      w[0] = v[0];
      w[1] = v[1];
    }
  }
  __device__ __forceinline__ void unpack(float* x) const {
#pragma unroll
    for (int e = 0; e < W; ++e) {
      if constexpr (sizeof(typename T::E) == 4) {
        x[e] = __uint_as_float(w[e]);
      } else {
        const f32x2 v = unpack2<T>(w[e]);
        x[2 * e] = v[0];
        x[2 * e + 1] = v[1];
      }
    }
  }
};

template <typename T, int VEC>
__device__ __forceinline__ void store_piece(typename T::E* p, const float* x) {
  if constexpr (sizeof(typename T::E) == 4) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4)
      *reinterpret_cast<f32x4*>(p + i) = (f32x4){x[i], x[i + 1], x[i + 2], x[i + 3]};
  } else {
    uint32_t w[VEC / 2];
#pragma unroll
    for (int e = 0; e < VEC / 2; ++e) w[e] = pack2<T>(x[2 * e], x[2 * e + 1]);
    if constexpr (VEC == 8)
      *reinterpret_cast<u32x4*>(p) = (u32x4){w[0], w[1], w[2], w[3]};
    else
      *reinterpret_cast<u32x2*>(p) = (u32x2){w[0], w[1]};
  }
}

// what one lane holds of a row: columns c[0] .. + VEC and c[1] .. + VEC
template <int VEC>
struct Lane {
  int c[2];
  bool has[2];
  bool turns;   // half-split: (piece 0, piece 1) is a pair of pieces that turns
  int pair;     // its first pair
};

template <int VEC, bool INTER>
__device__ __forceinline__ Lane<VEC> lane_of(int j, int d, int rot) {
  Lane<VEC> l;
  if (INTER) {
    l.c[0] = 2 * j * VEC;
    l.c[1] = l.c[0] + VEC;
    l.turns = false;
    l.pair = 0;
  } else {
    const int n = rot / (2 * VEC);  // lanes that turn
    l.turns = j < n;
    l.pair = j * VEC;
    l.c[0] = l.turns ? j * VEC : rot + 2 * (j - n) * VEC;
    l.c[1] = l.turns ? l.c[0] + rot / 2 : l.c[0] + VEC;
  }
  l.has[0] = l.c[0] < d;
  l.has[1] = l.c[1] < d;
  return l;
}

// cosines and sines of this lane's pairs: cs[0] / sn[0] .. for half-split pieces
// VEC pairs; interleaved pieces hold VEC / 2 pairs each.  Of pieces that do not
// turn: nothing.
template <int VEC, bool INTER>
__device__ __forceinline__ void load_angles(const float* row, const Lane<VEC>& l, int rot, float* cs, float* sn) {
  if (row == nullptr) return;
  if constexpr (INTER) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (l.c[h] < rot) {
#pragma unroll
        for (int i = 0; i < VEC / 2; i += 2) {  // (rot % 8 == 0, so rot / 2 and the pairs are even)
          const f32x2 c = *reinterpret_cast<const f32x2*>(row + l.c[h] / 2 + i);
          const f32x2 s = *reinterpret_cast<const f32x2*>(row + rot / 2 + l.c[h] / 2 + i);
          cs[h * VEC / 2 + i] = c[0];
          cs[h * VEC / 2 + i + 1] = c[1];
          sn[h * VEC / 2 + i] = s[0];
          sn[h * VEC / 2 + i + 1] = s[1];
        }
      }
  } else if (l.turns) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const f32x4 c = *reinterpret_cast<const f32x4*>(row + l.pair + i);
      const f32x4 s = *reinterpret_cast<const f32x4*>(row + rot / 2 + l.pair + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        cs[i + e] = c[e];
        sn[i + e] = s[e];
      }
    }
  }
}

// x[0 .. VEC) and x[VEC .. 2 VEC) turned by the angles (sign 1) or back (-1), where they turn at all: by an
// angle of 0, an infinite value would make the one beside it NaN
template <int VEC, bool INTER>
__device__ __forceinline__ void turn(const Lane<VEC>& l, int rot, float* x, const float* cs, const float* sn, float sign) {
  if constexpr (INTER) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (l.c[h] < rot) {  // (a piece of 4 or 8 columns turns or does not: rot % 8 == 0)
#pragma unroll
        for (int i = h * VEC / 2; i < (h + 1) * VEC / 2; ++i) {
          const float a = x[2 * i], b = x[2 * i + 1];
          x[2 * i] = a * cs[i] - sign * b * sn[i];
          x[2 * i + 1] = b * cs[i] + sign * a * sn[i];
        }
      }
  } else if (l.turns) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float a = x[i], b = x[VEC + i];
      x[i] = a * cs[i] - sign * b * sn[i];
      x[VEC + i] = b * cs[i] + sign * a * sn[i];
    }
  }
}

// over the LPR lanes of a row: neighbours, pairs, then the mirrored halves of 8 and of 16 lanes
template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
  auto other = [&](auto ctrl) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  x += other(std::integral_constant<int, 0xb1>{});
  if constexpr (LPR >= 4) x += other(std::integral_constant<int, 0x4e>{});
  if constexpr (LPR >= 8) x += other(std::integral_constant<int, 0x141>{});
  if constexpr (LPR >= 16) x += other(std::integral_constant<int, 0x140>{});
  if constexpr (LPR >= 32) x += __shfl_xor(x, 16);
  return x;
}

template <typename T, int VEC>
__device__ __forceinline__ void load_weight(const void* w, int f32, const Lane<VEC>& l, float* x) {
#pragma unroll
  for (int i = 0; i < 2 * VEC; ++i) x[i] = 1.f;
  if (w == nullptr) return;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (l.has[h]) {
      if (f32)
        load_piece<F32, VEC>(static_cast<const float*>(w) + l.c[h], x + h * VEC);
      else
        load_piece<T, VEC>(static_cast<const typename T::E*>(w) + l.c[h], x + h * VEC);
    }
}

__device__ __forceinline__ int64_t position_of(const RopeArgs& a, int b, int s) {
  const int64_t i = b * a.pb + s * a.ps;
  return a.pos64 ? static_cast<const int64_t*>(a.pos)[i] : static_cast<const int*>(a.pos)[i];
}

// --------------------------------------------------------------- forward ----
// blockIdx.x: token, blockIdx.y: slice of the heads (q, then k, then v).
// Bound by its bytes: 8192 tokens, 40 heads of 128 columns, bf16: 172 MB in 38 us, 4.6 TB/s
// (a large copy: 5.0; 28 us where the caches hold the rows); as an append of 8192 fp16 tokens, 48 heads: 206 MB in 48 us, 4.3 TB/s.
// 8 tokens: 5 us, the launch and one round trip to memory.
template <typename T, int VEC, int LPR, bool INTER, bool APPEND>
__global__ __launch_bounds__(512) void rope_forward(RopeArgs a) {
  using E = typename T::E;
  const int j = threadIdx.x % LPR;
  const int head = static_cast<int>(blockIdx.y * (blockDim.x / LPR) + threadIdx.x / LPR);
  const int b = APPEND ? 0 : static_cast<int>(blockIdx.x / a.S), s = APPEND ? static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x % a.S);
  const int heads = a.q.heads + a.k.heads + (APPEND ? a.v.heads : 0);
  const bool is_q = head < a.q.heads, is_v = APPEND && head >= a.q.heads + a.k.heads;
  const int h = is_q ? head : is_v ? head - a.q.heads - a.k.heads : head - a.q.heads;
  const RopeRows& r = is_q ? a.q : is_v ? a.v : a.k;
  const Lane<VEC> l = lane_of<VEC, INTER>(j, a.d, a.rot);

  const E* xp = static_cast<const E*>(r.x) + b * r.sb + s * r.ss + h * r.sh;
  Raw<T, VEC> xr[2]{};
  float w[2 * VEC];
  if constexpr (APPEND) {
    // the row and its weight are under way while the position is found, three loads one after the other
    // (8192 tokens of five sequences: 48 us, 55 us with the row after them)
    if (head < heads) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (l.has[e]) xr[e].load(xp + l.c[e]);
      if (a.norm && !is_v) load_weight<T, VEC>(r.w, a.w_f32, l, w);
    }
  }

  // where the token stands, and the cache row its key and value go to
  int64_t pos;
  int64_t krow = -1, vrow = -1;
  if constexpr (APPEND) {
    // sequence: the last that starts at or before the token, by 64 steps at a time
    const int lane = threadIdx.x & 63;
    int seq = 0;
    for (int n = a.p.B + 1, step = 0; step != 1; n = min(step, a.p.B + 1 - seq)) {
      step = (n + 63) / 64;
      const int i = lane * step, at = seq + min(i, n - 1);
      const int c = __popcll(__ballot(i < n && (at == 0 || a.p.cu[at] <= s)));
      seq += max(c - 1, 0) * step;
    }
    pos = -1;
    if (seq < a.p.B) {
      const int t0 = seq == 0 ? 0 : min(max(a.p.cu[seq], 0), a.p.T), t1 = min(max(a.p.cu[seq + 1], 0), a.p.T);
      pos = static_cast<int64_t>(max(a.p.len[seq], 0)) - (t1 - t0) + (s - t0);
      if (s < t0) pos = -1;  // (offsets that do not ascend)
      if (a.rope != nullptr && pos >= a.positions) pos = -1;
      if (pos >= 0 && pos < static_cast<int64_t>(a.p.width) * a.p.page) {
        const int ip = static_cast<int>(pos) / a.p.page, off = static_cast<int>(pos) - ip * a.p.page;
        const int id = a.p.table[seq * a.p.tstride + ip];
        if (id >= 0 && id < a.p.pages) {
          krow = id * a.kp + off * a.kr;
          vrow = id * a.vp + off * a.vr;
        }
      }
    }
  } else {
    pos = position_of(a, b, s);
    if (pos >= a.positions) pos = -1;
  }
  if (head >= heads) return;

  float x[2 * VEC];
  if constexpr (!APPEND) {
    if (pos >= 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (l.has[e]) xr[e].load(xp + l.c[e]);
    }
  }
  float cs[VEC], sn[VEC];
  const bool turns = !is_v && pos >= 0;
  if (turns) {  // (every load before the first use)
    load_angles<VEC, INTER>(a.rope == nullptr ? nullptr : a.rope + pos * a.rstride, l, a.rot, cs, sn);
    if (!APPEND && a.norm) load_weight<T, VEC>(r.w, a.w_f32, l, w);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) xr[e].unpack(x + e * VEC);
  if (APPEND && pos < 0) {  // (whatever the row holds)
#pragma unroll
    for (int i = 0; i < 2 * VEC; ++i) x[i] = 0.f;
  }
  if (turns) {
    if (a.norm) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * VEC; ++i) ss += x[i] * x[i];
      const float inv = rsqrtf(row_sum<LPR>(ss) / a.d + a.eps);
#pragma unroll
      for (int i = 0; i < 2 * VEC; ++i) x[i] *= inv * w[i];
    }
    turn<VEC, INTER>(l, a.rot, x, cs, sn, 1.f);
  }
  E* yp;
  if (!APPEND || is_q) {
    yp = static_cast<E*>(r.y) + ((static_cast<int64_t>(b) * a.S + s) * r.heads + h) * a.d;
  } else {
    if (krow < 0) return;
    yp = is_v ? static_cast<E*>(a.vc) + vrow + h * a.vh : static_cast<E*>(a.kc) + krow + h * a.kh;
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (l.has[e]) store_piece<T, VEC>(yp + l.c[e], x + e * VEC);
}

// -------------------------------------------------------------- backward ----
// A workgroup keeps its heads and walks over tokens, so each lane adds the
// weight gradient of its own columns in registers; at the end the workgroup's
// rows are added in LDS in a fixed order and its partial sums stored, and a second kernel
// adds the workgroups' -- no atomics, the same result every time.
// 8192 tokens, 40 heads of 128 columns, bf16: 256 MB in 67 us with the sum of 4, 4.1 TB/s (51 us where the caches
// hold the rows).  More waves, more rows loaded ahead and consecutive tokens for a workgroup were all slower
// (87, 70 and 71 us).
template <typename T, int VEC, int LPR, bool INTER>
__global__ __launch_bounds__(512, 4) void rope_backward(RopeArgs a) {
  using E = typename T::E;
  extern __shared__ float sh[];  // [rows of the workgroup][d]
  const int j = threadIdx.x % LPR, grp = threadIdx.x / LPR, groups = blockDim.x / LPR;
  const int head = static_cast<int>(blockIdx.y) * groups + grp;
  const int heads = a.q.heads + a.k.heads;
  const bool is_q = head < a.q.heads, live = head < heads;
  const int h = is_q ? head : head - a.q.heads;
  const RopeRows& r = is_q ? a.q : a.k;
  const Lane<VEC> l = lane_of<VEC, INTER>(j, a.d, a.rot);
  float w[2 * VEC], dw[2 * VEC];
  load_weight<T, VEC>(r.w, a.w_f32, l, w);
#pragma unroll
  for (int i = 0; i < 2 * VEC; ++i) dw[i] = 0.f;
  const int tokens = a.B * a.S;
  // A token's rows are loaded while the one before it is worked on; the rows'
  // offsets go on by additions as long as the sequence lasts
  Raw<T, VEC> xr[2]{}, gr[2]{};
  int64_t pos = -1;
  int b = static_cast<int>(blockIdx.x) / a.S, s = static_cast<int>(blockIdx.x) - b * a.S;
  const int64_t x_step = gridDim.x * r.ss, g_step = gridDim.x * r.gs;
  int64_t xo = b * r.sb + s * r.ss + h * r.sh, go = b * r.gb + s * r.gs + h * r.gh;
  auto fetch = [&]() {
    pos = position_of(a, b, s);
    const E* xp = static_cast<const E*>(r.x) + xo;
    const E* gp = static_cast<const E*>(r.g) + go;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (l.has[e]) {
        xr[e].load(xp + l.c[e]);
        gr[e].load(gp + l.c[e]);
      }
  };
  auto advance = [&]() {
    s += gridDim.x;
    xo += x_step;
    go += g_step;
    if (s >= a.S) {
      b += s / a.S;
      s %= a.S;
      xo = b * r.sb + s * r.ss + h * r.sh;
      go = b * r.gb + s * r.gs + h * r.gh;
    }
  };
  if (live) {
    E* yp = static_cast<E*>(r.y) + (static_cast<int64_t>(blockIdx.x) * r.heads + h) * a.d;
    const int64_t y_step = static_cast<int64_t>(gridDim.x) * r.heads * a.d;
    const float per_d = 1.f / a.d;
    fetch();
    for (int t = blockIdx.x; t < tokens; t += gridDim.x) {
      float x[2 * VEC], g[2 * VEC], cs[VEC], sn[VEC];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        xr[e].unpack(x + e * VEC);
        gr[e].unpack(g + e * VEC);
      }
      const bool there = pos >= 0 && pos < a.positions;
      if (there) load_angles<VEC, INTER>(a.rope + pos * a.rstride, l, a.rot, cs, sn);
      if (t + static_cast<int>(gridDim.x) < tokens) {
        advance();
        fetch();
      }
      if (there) {
        turn<VEC, INTER>(l, a.rot, g, cs, sn, -1.f);
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * VEC; ++i) ss += x[i] * x[i];
        const float inv = rsqrtf(row_sum<LPR>(ss) * per_d + a.eps);
#pragma unroll
        for (int i = 0; i < 2 * VEC; ++i) {
          x[i] *= inv;
          dw[i] += g[i] * x[i];
          g[i] *= w[i];
          dot += g[i] * x[i];
        }
        const float f = row_sum<LPR>(dot) * per_d;
#pragma unroll
        for (int i = 0; i < 2 * VEC; ++i) g[i] = inv * (g[i] - x[i] * f);
      } else {
#pragma unroll
        for (int i = 0; i < 2 * VEC; ++i) g[i] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (l.has[e]) store_piece<T, VEC>(yp + l.c[e], g + e * VEC);
      yp += y_step;
    }
  }
  if (a.ws == nullptr) return;
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (l.has[e]) store_piece<F32, VEC>(sh + grp * a.d + l.c[e], dw + e * VEC);
  __syncthreads();
  const int first_k = min(max(a.q.heads - static_cast<int>(blockIdx.y) * groups, 0), groups);
  const int last = min(max(heads - static_cast<int>(blockIdx.y) * groups, 0), groups);
  float* out = a.ws + (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * 2 * a.d;
  for (int c = threadIdx.x; c < a.d; c += blockDim.x) {
    float sq = 0.f, sk = 0.f;
    for (int i = 0; i < first_k; ++i) sq += sh[i * a.d + c];
    for (int i = first_k; i < last; ++i) sk += sh[i * a.d + c];
    out[c] = sq;
    out[a.d + c] = sk;
  }
}

// column sums of the workgroups' partial weight gradients [n][2 d], in the
// weights' type: a workgroup takes 8 columns, each of its 128 rows of threads
// every 128th partial sum; then the rows in order
template <typename T>
__global__ __launch_bounds__(1024) void rope_dw_sum(const float* ws, int n, int d, typename T::E* dwq, typename T::E* dwk) {
  __shared__ float sh[128][9], part[16][9];
  const int c = threadIdx.x & 7, col = blockIdx.x * 8 + c, row = threadIdx.x >> 3;
  float x = 0.f;
#pragma unroll 16
  for (int i = row; i < n; i += 128) x += ws[static_cast<int64_t>(i) * 2 * d + col];
  sh[row][c] = x;
  __syncthreads();
  if (row < 16) {
    x = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x += sh[row * 8 + i][c];
    part[row][c] = x;
  }
  __syncthreads();
  if (row != 0) return;
  x = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) x += part[i][c];
  typename T::E* out = col < d ? dwq : dwk;
  if (out == nullptr) return;
  out += col < d ? col : col - d;
  if constexpr (sizeof(typename T::E) == 4)
    *out = x;
  else
    *out = static_cast<uint16_t>(pack2<T>(x, 0.f));
}

// ---------------------------------------------------------------- launch ----
// 16-byte pieces where every row and pair of pieces allows them, else 8-byte
// ones (16-bit types: rot / 2 not a multiple of 8, or rows aligned to 8 bytes only).
// (8192 tokens, 40 heads of 128 columns, bf16: forward 28 us, 33 us by 8-byte pieces; backward 51 us by both)
bool wide_pieces(const RopeArgs& a, bool rows16) {
  return a.type != AttnType::kF32 && rows16 && (a.interleaved || a.rot % 16 == 0);
}

bool aligned16(const RopeArgs& a, const RopeRows& r) {
  auto odd = [](const void* p, int64_t x, int64_t y, int64_t z) {
    return reinterpret_cast<uintptr_t>(p) % 16 != 0 || x % 8 != 0 || y % 8 != 0 || z % 8 != 0;
  };
  return !odd(r.x, r.sb, r.ss, r.sh) && !odd(r.g, r.gb, r.gs, r.gh);
}

template <int VEC, typename F>
void by_lanes(int d, F f) {
  const int n = (d / VEC + 1) / 2;  // lanes that hold something, <= 256 / (2 VEC)
  if (n <= 2)
    f(std::integral_constant<int, 2>{});
  else if (n <= 4)
    f(std::integral_constant<int, 4>{});
  else if (n <= 8)
    f(std::integral_constant<int, 8>{});
  else if (VEC == 8 || n <= 16)
    f(std::integral_constant<int, 16>{});
  else if constexpr (VEC < 8)
    f(std::integral_constant<int, 32>{});
}

template <typename F>
void by_type(const RopeArgs& a, bool rows16, F f) {
  auto pieces = [&](auto t) {
    using T = decltype(t);
    auto shape = [&](auto vec) {
      by_lanes<decltype(vec)::value>(a.d, [&](auto lpr) {
        if (a.interleaved)
          f(t, vec, lpr, std::true_type{});
        else
          f(t, vec, lpr, std::false_type{});
      });
    };
    if constexpr (sizeof(typename T::E) == 2) {
      if (wide_pieces(a, rows16)) return shape(std::integral_constant<int, 8>{});
    }
    shape(std::integral_constant<int, 4>{});
  };
  if (a.type == AttnType::kBF16)
    pieces(BF16{});
  else if (a.type == AttnType::kF16)
    pieces(F16{});
  else
    pieces(F32{});
}

// workgroup: whole waves that hold `heads` rows, at most `limit` threads; slices: blockIdx.y
void block_of(int heads, int lpr, int limit, int* threads, int* slices) {
  const int per_wave = 64 / lpr, waves = (heads + per_wave - 1) / per_wave, most = limit / 64;
  *slices = (waves + most - 1) / most;
  *threads = (waves + *slices - 1) / *slices * 64;
}

template <bool APPEND>
void forward(const RopeArgs& a, hipStream_t s) {
  const int heads = a.q.heads + a.k.heads + (APPEND ? a.v.heads : 0);
  const int64_t tokens = static_cast<int64_t>(a.B) * a.S;
  if (tokens == 0 || heads == 0) return;
  const bool rows16 = aligned16(a, a.q) && aligned16(a, a.k) && (!APPEND || aligned16(a, a.v));
  by_type(a, rows16, [&](auto t, auto vec, auto lpr, auto inter) {
    int threads, slices;
    block_of(heads, decltype(lpr)::value, 512, &threads, &slices);
    rope_forward<decltype(t), decltype(vec)::value, decltype(lpr)::value, decltype(inter)::value, APPEND>
        <<<dim3(static_cast<unsigned>(tokens), static_cast<unsigned>(slices)), threads, 0, s>>>(a);
  });
}

// Workgroups along the tokens of the backward kernel: about ten waves a compute unit in all, one round
// (8192 tokens x 40 heads x 128 bf16: 512 workgroups of 5 waves 67 us with the sum, 256 97 us, 768 82 us, 1024 86 us)
int backward_blocks(const RopeArgs& a, int threads, int slices) {
  const int waves = threads / 64 * slices;
  return static_cast<int>(std::min<int64_t>(static_cast<int64_t>(a.B) * a.S, std::max(2560 / waves, 1)));
}

}  // namespace

void qk_norm_rope(const RopeArgs& a, hipStream_t s) { forward<false>(a, s); }

void paged_append(const RopeArgs& a, hipStream_t s) { forward<true>(a, s); }

size_t qk_norm_rope_backward_workspace_bytes(const RopeArgs& a) {
  size_t bytes = 0;
  const bool rows16 = aligned16(a, a.q) && aligned16(a, a.k);
  by_type(a, rows16, [&](auto, auto, auto lpr, auto) {
    int threads, slices;
    block_of(a.q.heads + a.k.heads, decltype(lpr)::value, 512, &threads, &slices);
    bytes = static_cast<size_t>(backward_blocks(a, threads, slices)) * slices * 2 * a.d * sizeof(float);
  });
  return bytes;
}

void qk_norm_rope_backward(const RopeArgs& a, hipStream_t s) {
  const int heads = a.q.heads + a.k.heads;
  int n = 0;
  const bool rows16 = aligned16(a, a.q) && aligned16(a, a.k);
  if (static_cast<int64_t>(a.B) * a.S > 0 && heads > 0)
    by_type(a, rows16, [&](auto t, auto vec, auto lpr, auto inter) {
      constexpr int LPR = decltype(lpr)::value;
      int threads, slices;
      block_of(heads, LPR, 512, &threads, &slices);
      const int blocks = backward_blocks(a, threads, slices);
      n = blocks * slices;
      const size_t lds = a.ws != nullptr ? static_cast<size_t>(threads / LPR) * a.d * sizeof(float) : 0;
      rope_backward<decltype(t), decltype(vec)::value, LPR, decltype(inter)::value>
          <<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(slices)), threads, lds, s>>>(a);
    });
  if (a.dwq == nullptr && a.dwk == nullptr) return;
  auto sum = [&](auto t) {
    using T = decltype(t);
    using E = typename T::E;
    rope_dw_sum<T><<<2 * a.d / 8, 1024, 0, s>>>(a.ws, n, a.d, static_cast<E*>(a.dwq), static_cast<E*>(a.dwk));
  };
  if (a.w_f32 || a.type == AttnType::kF32)
    sum(F32{});
  else if (a.type == AttnType::kBF16)
    sum(BF16{});
  else
    sum(F16{});
}

}  // namespace kernels
}  // namespace nnsx
