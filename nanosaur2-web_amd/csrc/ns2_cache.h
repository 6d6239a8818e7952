// Shared by the cache kernels (ns2_cache.hip, ns2_cache_rows.hip, ns2_cache_prompt.hip): the layout of a
// cache, its 4-bit values, which keys a tile of query columns sees, and the softmax's running state.
//
// Attention runs transposed: S^T = K Q^T and O^T = V^T P^T, both with v_mfma_f32_16x16x32_f16. A product's
// result holds one query per lane column (lane % 16) and four rows per lane (4 (lane / 16) + r), so that
// the weights p of two 16-key score tiles are, in place, the B operand of the second product: operand
// element j of lane group grp is key 4 grp + j of the first tile (j < 4) or of the second (j >= 4). V^T's
// operand takes its keys in the same order. A "column" is one (token, query head) pair of a K/V head, token
// by token, so that the heads of a group share every key that is loaded.
#pragma once

#include <type_traits>

#include "ns2_common.h"

namespace ns2cache {

using namespace ns2dev;

typedef float float2_t __attribute__((ext_vector_type(2)));
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kGroup = 32;  // values per step and offset of a 4-bit cache

struct AttnArgs {
  const void* q;
  const int* pos;
  const void *k, *v;
  const half2_t *kg, *vg;  // (step, offset) of a 4-bit cache
  void* o;
  float* part_o;   // splits > 1: [splits][batch*KH][R][D] sums over a split's keys
  float2* part_s;  // and their (maximum, sum of weights)
  long long kvBatch;
  int ldq, ldo, ldkv, L, H, KH, cap, window, sinks, q_fmt, batch, splits;
  float scale;  // the caller's times log2(e)
};

struct Plan {
  bool prompt;  // ns2_cache_prompt.hip, else ns2_cache_rows.hip
  int splits;
};

int launch_rows(const AttnArgs& a, int D, hipStream_t s);
int launch_prompt(const AttnArgs& a, int D, hipStream_t s);

// ---- 4-bit values ----------------------------------------------------------------------------

// Four nibbles of each 16-bit half of x -> the half2 pairs (n0, n0'), (n1, n1') ...: 0x6400 | n is the half
// 1024 + n (and 0x6400 | 16 n is 1024 + 16 n), taking 1024 off (or a sixteenth, less 64) is exact, and the fused
// multiply-add rounds offset + n * step once.
__device__ __forceinline__ void dequant4(uint32_t x, half2_t s, half2_t o, uint32_t r[4]) {
  nibbles4(x, half2_t{-1024.f, -1024.f}, half2_t{-64.f, -64.f}, r);
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2_t, r[i]), s, o));
}

// A word's eight values in the order 0 4 1 5 2 6 3 7 (operand elements; Q's are put in the same order).
__device__ __forceinline__ half8_t dequant8(uint32_t w, half2_t so) {
  uint32_t r[4];
  dequant4(w, half2_t{so[0], so[0]}, half2_t{so[1], so[1]}, r);
  return __builtin_bit_cast(half8_t, make_uint4(r[0], r[1], r[2], r[3]));
}

// (low half of a, low half of b) and (high half of a, high half of b)
__device__ __forceinline__ uint32_t pair_lo(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t pair_hi(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// ---- columns and the keys they see --------------------------------------------------------------

template <int CTRL>
__device__ __forceinline__ int dpp_i(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false);
}
__device__ __forceinline__ int row16_max(int v) {
  v = max(v, dpp_i<kDppXor1>(v));
  v = max(v, dpp_i<kDppXor2>(v));
  v = max(v, dpp_i<kDppHalfMirror>(v));
  return max(v, dpp_i<kDppRowMirror>(v));
}
// Maximum over the four lanes that hold one column (lane % 16).
__device__ __forceinline__ float column_max(float v) {
  float a = v, b = v;
  permlane16_swap(a, b);
  a = fmaxf(a, b);
  b = a;
  permlane32_swap(a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float column_sum(float v) {
  float a = v, b = v;
  permlane16_swap(a, b);
  a = a + b;
  b = a;
  permlane32_swap(a, b);
  return a + b;
}

// Position of column m (-1: padding, or past the last column).
__device__ __forceinline__ int column_pos(const AttnArgs& a, int b, int m) {
  const int G = a.H / a.KH;
  if (m >= a.L * G) return -1;
  const int p = a.pos[(long long)b * a.L + m / G];
  return p < a.cap ? p : -1;
}

// The keys that some column of a block sees, as tiles of KT: the first tokens [0, first) that are outside
// every window, then [lo, last].
struct Keys {
  int pmin, pmax, lo, first, tiles_first, tiles;
};

template <int KT>
__device__ __forceinline__ Keys keys_of(const AttnArgs& a, int pmin, int pmax) {
  Keys k;
  k.pmin = pmin;
  k.pmax = pmax;
  k.lo = a.window && pmin >= a.window ? pmin - a.window + 1 : 0;
  k.first = a.sinks < k.lo ? a.sinks : k.lo;
  k.tiles_first = (k.first + KT - 1) / KT;
  k.tiles = k.tiles_first + (pmax - k.lo) / KT + 1;
  return k;
}

struct Tile {
  int key0, end;  // keys [key0, end) of the tile exist; loads past them repeat the last one
  bool whole;     // every column sees every key
};

template <int KT>
__device__ __forceinline__ Tile tile_of(const AttnArgs& a, const Keys& k, int t) {
  Tile r;
  const bool first = t < k.tiles_first;
  r.key0 = first ? t * KT : k.lo + (t - k.tiles_first) * KT;
  r.end = first ? k.first : k.pmax + 1;
  const int last = r.key0 + KT - 1;
  r.whole = last < r.end && last <= k.pmin && (!a.window || r.key0 > k.pmax - a.window || last < a.sinks);
  return r;
}

// What a column at position p (-1: nothing) sees of a tile: keys [from, from + n) and keys below `below`. (In a
// tile of first tokens, those below its end; else its window, and first tokens that lie inside another
// column's window.)
struct Sight {
  int from;
  unsigned n;
  int below;
  __device__ __forceinline__ bool operator()(int key) const { return (unsigned)(key - from) < n || key < below; }
};
__device__ __forceinline__ Sight sight_of(const AttnArgs& a, const Keys& k, int t, int p) {
  const bool first = t < k.tiles_first;
  const int from = a.window && p >= a.window ? p - a.window + 1 : 0;
  Sight s;
  s.from = from;
  s.n = first ? 0u : (unsigned)(p + 1 - from);
  s.below = min(first ? k.first : a.sinks, p + 1);
  return s;
}

// A tile's first row, from which lanes count in 32 bits (rows are at most 2^24 values apart).
__device__ __forceinline__ const char* tile_rows(const void* cache, long long base, int key0, int ldkv, bool i4) {
  const long long at = base + (long long)key0 * ldkv;
  return static_cast<const char*>(cache) + (i4 ? at / 2 : at * 2);
}

__device__ __forceinline__ const half2_t* tile_groups(const half2_t* groups, long long base, int key0, int ldkv) {
  return groups + (base + (long long)key0 * ldkv) / kGroup;
}

// ---- queries -------------------------------------------------------------------------------------

// Element e of operand step t of lane group grp is dimension qdim(t, grp) + e (fp16 cache: e in order, 4-bit:
// in the order of dequant8). A lane's K values are 8 apart from its neighbours' in an fp16 row, and one
// contiguous quarter of a 4-bit row.
template <int D, bool I4>
__device__ __forceinline__ int qdim(int t, int grp) {
  return I4 ? grp * (D / 4) + 8 * t : 32 * t + 8 * grp;
}

// Column m's query (zeros for padding), negated for a negative scale. fp32 queries are scaled by a power of two to
// below 2^14 and taken as two halves that keep 21 bits.
template <int D, bool I4, bool F32>
struct Query {
  static constexpr int QT = D / 32;
  float4 x[F32 ? QT : 1][2];
  half8_t h[F32 ? 1 : QT];
  float sign;

  __device__ __forceinline__ void load(const AttnArgs& a, int b, int g, int m, bool live, int grp) {
    const int G = a.H / a.KH, i = live ? m / G : 0, hd = live ? m - i * G : 0;
    const long long e = ((long long)b * a.L + i) * a.ldq + (long long)(g * G + hd) * D;
    sign = a.scale < 0.f ? -1.f : 1.f;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const int d = qdim<D, I4>(t, grp);
      if constexpr (F32) {
        const float* q = static_cast<const float*>(a.q) + e + d;
        x[t][0] = live ? *reinterpret_cast<const float4*>(q) : make_float4(0.f, 0.f, 0.f, 0.f);
        x[t][1] = live ? *reinterpret_cast<const float4*>(q + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
      } else {
        h[t] = live ? *reinterpret_cast<const half8_t*>(static_cast<const half_t*>(a.q) + e + d) : half8_t{0, 0, 0, 0, 0, 0, 0, 0};
      }
    }
  }
  // The exponent of the scaling, the same in the column's lanes.
  __device__ __forceinline__ int up() const {
    if constexpr (!F32) return 0;
    float top = 0.f;
#pragma unroll
    for (int t = 0; t < (F32 ? QT : 0); ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        top = fmaxf(top, fmaxf(fmaxf(fabsf(x[t][i].x), fabsf(x[t][i].y)), fmaxf(fabsf(x[t][i].z), fabsf(x[t][i].w))));
    top = column_max(top);
    return top > 0.f && top < INFINITY ? min(14 - __builtin_amdgcn_frexp_expf(top), 120) : 0;
  }
  // What takes a score to a base-2 logarithm: above 0, so that -inf stays -inf for a scale of 0.
  __device__ __forceinline__ static float mult(const AttnArgs& a, int up) { return fmaxf(ldexpf(fabsf(a.scale), -up), 1e-37f); }
  // The B operand of step t; PERM: in the order of dequant8.
  template <bool PERM>
  __device__ __forceinline__ void operand(int t, int up, half8_t& hi, half8_t& lo) const {
    constexpr int order[8] = {0, PERM ? 4 : 1, PERM ? 1 : 2, PERM ? 5 : 3, PERM ? 2 : 4, PERM ? 6 : 5, PERM ? 3 : 6, 7};
    if constexpr (!F32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) hi[e] = h[t][order[e]] * (half_t)sign;
    } else {
      const float y[8] = {x[t][0].x, x[t][0].y, x[t][0].z, x[t][0].w, x[t][1].x, x[t][1].y, x[t][1].z, x[t][1].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // both of z's sign unless it is 0 (they are fp16's smallest at least, 2^-38 of the largest), so that two products
        // with an infinity agree
        const float z = ldexpf(sign * y[order[e]], up), least = z == 0.f ? 0.f : copysignf(0x1p-24f, z);
        const half_t h = (half_t)__builtin_amdgcn_cvt_pkrtz(z, z)[0];
        const half_t l = (half_t)(z - (float)h);
        hi[e] = h == (half_t)0.f ? (half_t)least : h;
        lo[e] = h == (half_t)0.f || l == (half_t)0.f ? (half_t)least : l;
      }
    }
  }
};

// ---- the softmax's running state -------------------------------------------------------------------

// The reference m of a column trails its maximum by up to 2^kSlack: only a score above m + kSlack moves it
// and rescales the sums, so that most tiles leave the accumulators alone. Weights are 2^(score - m + kLift),
// at most 2^(kSlack + kLift): far enough below fp16's largest value, and as far as that allows above its
// smallest (what a weight's two halves leave is off by up to 2^-25, 2^-31 of the weight of the reference).
constexpr float kSlack = 8.f, kLift = 6.f;

// Scores s[N] (-inf where masked; times mult > 0 they are base-2 logarithms) of the lane's column -> weights in
// place; returns whether the lane's column moved its reference, with the factor for what was summed before.
template <int N>
__device__ __forceinline__ bool soften(float (&s)[N], float mult, float& m, float& l, float& corr) {
  float top = s[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, s[i]);
  top = column_max(top) * mult;
  const bool moves = top > m + kSlack;
  corr = moves && m > -INFINITY ? __builtin_amdgcn_exp2f(m - top) : moves ? 0.f : 1.f;
  m = moves ? top : m;
  const float ref = m == -INFINITY ? 0.f : m - kLift;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], mult, -ref));
    sum += s[i];
  }
  l = l * corr + sum;
  return moves;
}

__device__ __forceinline__ float4_t mfma(half8_t a, half8_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float4_t mfma(half4_t a, half4_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
}

// The B operand of the second product: the weights as two halves that keep 21 bits, the first one step below the weight
// cut off, the second what that left (one mixed-precision multiply-add; the factor hides from the compiler, which would
// make a conversion and a subtraction of it). For fp16 queries too: with one half per weight, the sum of weights that
// divides the output would have to be one of rounded weights, and the output's error is half as large again as that of
// its own rounding (2.9e-4 against 2.1e-4). Both halves are positive where the weight is (from 2^-23 on, 2^-29 of the
// weight of the reference), so that two products with an infinity agree.
template <int N, class H>
__device__ __forceinline__ void weights(const float (&p)[N], H& hi, H& lo) {
  float one = 1.f;
  asm("" : "+s"(one));
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    const ushort2_t u = __builtin_bit_cast(ushort2_t, __builtin_amdgcn_cvt_pkrtz(p[e], p[e + 1]));
    const half2_t h = __builtin_bit_cast(half2_t, __builtin_elementwise_sub_sat(u, ushort2_t{1, 1}));
    const half2_t l = __builtin_convertvector(
        float2_t{__builtin_fmaf(-(float)h[0], one, p[e]), __builtin_fmaf(-(float)h[1], one, p[e + 1])}, half2_t);
    hi[e] = h[0];
    hi[e + 1] = h[1];
    lo[e] = l[0];
    lo[e + 1] = l[1];
  }
}

// Values that are not finite must reach the columns that see them and no others, but 0 * inf is NaN: they are
// taken out of the product, and a second product of marks (1 for inf, 64 for -inf, 4096 for NaN) with the
// columns' visible keys (1 or 0) tells each output what it has seen (at most 32 of each per product). What was
// seen is kept aside and put into the outputs at the end.
template <class H>
__device__ __forceinline__ H without_marked(H v, H& mark) {
#pragma unroll
  for (int e = 0; e < (int)(sizeof(H) / 2); ++e) {
    const half_t x = v[e];  // (a bit cast of the element itself would read element 0)
    const uint16_t u = __builtin_bit_cast(uint16_t, x), size = u & 0x7fffu;
    mark[e] = size < 0x7c00u ? (half_t)0.f : size > 0x7c00u ? (half_t)4096.f : u == size ? (half_t)1.f : (half_t)64.f;
    v[e] = size < 0x7c00u ? x : (half_t)0.f;
  }
  return v;
}
// Two bits per output: 1 inf, 2 -inf, 3 NaN (and what both infinities add up to).
__device__ __forceinline__ uint32_t seen_bits(float4_t count) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = (int)count[i];
    w |= (uint32_t)((c & 63 ? 1 : 0) | (c & 0xfc0 ? 2 : 0) | (c >= 4096 ? 3 : 0)) << (2 * i);
  }
  return w;
}
__device__ __forceinline__ float4_t with_seen(float4_t o, uint32_t bits) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = (bits >> (2 * i)) & 3u;
    if (b) o[i] += b == 1 ? INFINITY : b == 2 ? -INFINITY : NAN;
  }
  return o;
}

// Adds 0 * v: NaN once v held an infinity or a NaN.
__device__ __forceinline__ void spot(uint32_t v, half2_t& z) {
  z = __builtin_elementwise_fma(__builtin_bit_cast(half2_t, v), half2_t{0.f, 0.f}, z);
}
__device__ __forceinline__ void spot(half4_t v, half2_t& z) {
  const uint2 w = __builtin_bit_cast(uint2, v);
  spot(w.x, z);
  spot(w.y, z);
}
__device__ __forceinline__ void spot(half8_t v, half2_t& z) {
  const uint4 w = __builtin_bit_cast(uint4, v);
  spot(w.x, z);
  spot(w.y, z);
  spot(w.z, z);
  spot(w.w, z);
}

}  // namespace ns2cache

#define NS2_CACHE_D(D, LAUNCH)  \
  switch (D) {                  \
    case 64: LAUNCH(64) break;   \
    case 96: LAUNCH(96) break;   \
    case 128: LAUNCH(128) break; \
    default: LAUNCH(256) break;  \
  }
