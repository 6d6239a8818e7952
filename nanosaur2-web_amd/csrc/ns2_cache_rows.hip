// Attention of few query columns over a cache: single tokens, and short runs of them.
//
// The cache is read once and that bounds it: 2 D values per key and K/V head for at most 16 columns. A block
// takes 16 columns of one K/V head and one split of their keys; its four waves take tiles of 32 keys in
// turn, straight from memory into operand registers, each with a softmax state and accumulators of its own,
// and merge them through LDS at the end (of 16 keys for fp16 heads of 256, where 32 would take more registers
// than two waves per SIMD have). A tile's next K rows are requested as soon as the scores have used
// the last ones, its next V rows after the second product, so that a wave always has loads in flight.
//
// Measured, with the join of the splits: 16 fp16 tokens of 16 heads on 16384 fp16 keys of 4 heads of 128 98 us (the
// cache at 5.5 TB/s, a copy reads and writes 5.2); 32 tokens of 4 heads on up to 16000 4-bit keys of one head of 256
// 38 us (2.9 TB/s: eight 4-bit values of a lane take 13 instructions, the VALU is busy 60 % of the time); one fp32
// token on a window of 516 fp16 keys of 256 10.6 us, the chain of two launches (position, keys, merge; sums, output).
#include "ns2_cache.h"

using namespace ns2cache;

namespace {

constexpr int kWaves = 4;
// 16-key steps of a wave's tile
template <int D, bool I4>
constexpr int steps() {
  return D == 256 && !I4 ? 1 : 2;
}
// Operand element j of lane group grp is this key of the tile.
__device__ __forceinline__ int key_of(int grp, int j) { return 4 * grp + (j < 4 ? j : 12 + j); }

// The K operands of a tile: rows key0 + 16 s + lane % 16 of step t.
template <int D, bool I4>
struct KTile {
  static constexpr int NS = steps<D, I4>();
  half8_t x[NS][D / 32];
  __device__ __forceinline__ void load(const AttnArgs& a, long long base, const Tile& t, int col, int grp) {
    const char* rows = tile_rows(a.k, base, t.key0, a.ldkv, false);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const uint32_t at = (uint32_t)(min(16 * s + col, t.end - 1 - t.key0) * a.ldkv + 8 * grp);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) x[s][i] = *reinterpret_cast<const half8_t*>(rows + 2u * at + 64 * i);
    }
  }
  __device__ __forceinline__ half8_t operand(int s, int t, int) const { return x[s][t]; }
};

template <int D>
struct KTile<D, true> {
  static constexpr int W = D / 32, NG = D == 96 ? 3 : D == 256 ? 2 : 1;  // words and groups of a lane's D / 4 values
  uint32_t w[2][W];
  half2_t so[2][NG];
  __device__ __forceinline__ void load(const AttnArgs& a, long long base, const Tile& t, int col, int grp) {
    const char* rows = tile_rows(a.k, base, t.key0, a.ldkv, true);
    const half2_t* groups = tile_groups(a.kg, base, t.key0, a.ldkv);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint32_t at = (uint32_t)(min(16 * s + col, t.end - 1 - t.key0) * a.ldkv);
      const char* row = rows + (at / 2 + grp * (D / 8));
      if constexpr (D == 96) {
#pragma unroll
        for (int i = 0; i < W; ++i) w[s][i] = reinterpret_cast<const uint32_t*>(row)[i];
      } else if constexpr (D == 64) {
        const uint2 x = *reinterpret_cast<const uint2*>(row);
        w[s][0] = x.x;
        w[s][1] = x.y;
      } else {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(row + 4 * i);
          w[s][i] = x.x;
          w[s][i + 1] = x.y;
          w[s][i + 2] = x.z;
          w[s][i + 3] = x.w;
        }
      }
#pragma unroll
      for (int i = 0; i < NG; ++i) so[s][i] = groups[at / kGroup + (grp * (D / 4) + (D == 96 ? 8 : 32) * i) / kGroup];
    }
  }
  __device__ __forceinline__ half8_t operand(int s, int t, int) const { return dequant8(w[s][t], so[s][D == 96 ? t : t / 4]); }
};

// The V^T operands of a tile: lane column c holds dimensions vdim(t, c) of eight keys, a contiguous piece of
// each row, so that 16 lanes read a row; two keys' halves are paired in registers.
template <int D, bool I4>
__device__ __forceinline__ int vdim(int t, int c) {
  return I4 && D == 96 ? (t < 4 ? 4 * c + t : 64 + 2 * c + t - 4) : D / 16 * c + t;
}

template <int D, bool I4>
struct VTile {
  static constexpr int DT = D / 16, NK = 4 * steps<D, I4>();
  uint32_t x[NK][DT / 2];
  __device__ __forceinline__ void load(const AttnArgs& a, long long base, const Tile& t, int col, int grp) {
    const char* rows = tile_rows(a.v, base, t.key0, a.ldkv, false);
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      const char* row = rows + 2u * (uint32_t)(min(key_of(grp, j), t.end - 1 - t.key0) * a.ldkv + DT * col);
      if constexpr (DT % 8 == 0) {
#pragma unroll
        for (int i = 0; i < DT / 2; i += 4) {
          const uint4 y = *reinterpret_cast<const uint4*>(row + 4 * i);
          x[j][i] = y.x;
          x[j][i + 1] = y.y;
          x[j][i + 2] = y.z;
          x[j][i + 3] = y.w;
        }
      } else if constexpr (DT == 4) {
        const uint2 y = *reinterpret_cast<const uint2*>(row);
        x[j][0] = y.x;
        x[j][1] = y.y;
      } else {
#pragma unroll
        for (int i = 0; i < DT / 2; ++i) x[j][i] = reinterpret_cast<const uint32_t*>(row)[i];
      }
    }
  }
  // makes the next each() start from the loaded values again, instead of keeping every operand of the last
  __device__ __forceinline__ void again() {
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
      for (int i = 0; i < DT / 2; ++i) asm volatile("" : "+v"(x[j][i]));
  }
  // calls f(t, operand) for every step of 16 dimensions
  template <class F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      uint32_t r[NK / 2];
#pragma unroll
      for (int i = 0; i < NK / 2; ++i) r[i] = t & 1 ? pair_hi(x[2 * i][t / 2], x[2 * i + 1][t / 2]) : pair_lo(x[2 * i][t / 2], x[2 * i + 1][t / 2]);
      if constexpr (NK == 8) f(t, __builtin_bit_cast(half8_t, make_uint4(r[0], r[1], r[2], r[3])));
      else f(t, __builtin_bit_cast(half4_t, make_uint2(r[0], r[1])));
    }
  }
};

template <int D>
struct VTile<D, true> {
  static constexpr int DT = D / 16, W = D == 256 ? 2 : D == 96 ? 2 : 1, NG = D == 96 ? 2 : 1;
  uint32_t w[8][W];
  uint32_t so[8][NG];
  __device__ __forceinline__ void load(const AttnArgs& a, long long base, const Tile& t, int col, int grp) {
    const char* rows = tile_rows(a.v, base, t.key0, a.ldkv, true);
    const uint32_t* groups = reinterpret_cast<const uint32_t*>(tile_groups(a.vg, base, t.key0, a.ldkv));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t at = (uint32_t)(min(key_of(grp, j), t.end - 1 - t.key0) * a.ldkv);
      const char* row = rows + at / 2;
      const uint32_t* gr = groups + at / kGroup;
      if constexpr (D == 256) {
        const uint2 y = *reinterpret_cast<const uint2*>(row + 8 * col);
        w[j][0] = y.x;
        w[j][1] = y.y;
      } else if constexpr (D == 128) {
        w[j][0] = *reinterpret_cast<const uint32_t*>(row + 4 * col);
      } else {
        w[j][0] = *reinterpret_cast<const uint16_t*>(row + 2 * col);
        if constexpr (D == 96) w[j][1] = *reinterpret_cast<const uint8_t*>(row + 32 + col);
      }
      so[j][0] = gr[vdim<D, true>(0, col) / kGroup];
      if constexpr (NG == 2) so[j][1] = gr[2];
    }
  }
  __device__ __forceinline__ void again() {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < W; ++i) asm volatile("" : "+v"(w[j][i]));
  }
  // four dimensions u, u + 1.. of the key pairs (2 i, 2 i + 1), taken from the pairs' 16-bit pieces
  template <class F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int u = 0; u < (DT + 3) / 4; ++u) {
      uint32_t r[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int word = D == 96 ? u : u / 2, gi = NG == 2 ? u : 0;
        const uint32_t x = D >= 128 && u & 1 ? pair_hi(w[2 * i][word], w[2 * i + 1][word]) : pair_lo(w[2 * i][word], w[2 * i + 1][word]);
        dequant4(x, __builtin_bit_cast(half2_t, pair_lo(so[2 * i][gi], so[2 * i + 1][gi])),
                 __builtin_bit_cast(half2_t, pair_hi(so[2 * i][gi], so[2 * i + 1][gi])), r[i]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (4 * u + e < DT) f(4 * u + e, __builtin_bit_cast(half8_t, make_uint4(r[0][e], r[1][e], r[2][e], r[3][e])));
    }
  }
};

template <int D, bool I4, bool F32>
__global__ __launch_bounds__(64 * kWaves, 2) void cache_rows_kernel(AttnArgs a) {
  constexpr int DT = D / 16, QT = D / 32, OS = D + 4, NS = steps<D, I4>(), NK = 4 * NS, kTile = 16 * NS;
  typedef typename std::conditional<NS == 2, half8_t, half4_t>::type Part;  // of the second product's operands
  // the queries' operands and which values were not finite; after the last tile the waves' outputs
  __shared__ __attribute__((aligned(16))) float smem[kWaves * 16 * OS];
  constexpr int kQueries = (F32 ? 2 : 1) * QT * 64 * sizeof(half8_t);
  static_assert(sizeof(smem) >= kQueries + kWaves * DT * 64, "both fit");
  half8_t(*q_s)[QT][64] = reinterpret_cast<half8_t(*)[QT][64]>(smem);
  uint8_t(*seen_s)[DT][64] = reinterpret_cast<uint8_t(*)[DT][64]>(reinterpret_cast<char*>(smem) + kQueries);
  float(*o_s)[16][OS] = reinterpret_cast<float(*)[16][OS]>(smem);
  __shared__ float m_s[kWaves][16], l_s[kWaves][16];
  __shared__ int p_s[16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 15, grp = lane >> 4;
  const int heads = a.batch * a.KH, z = blockIdx.x / heads, bg = blockIdx.x - z * heads;
  const int b = bg / a.KH, g = bg - b * a.KH;
  const int m0 = blockIdx.y * 16, G = a.H / a.KH, R = a.L * G;
  const int p = column_pos(a, b, m0 + col);
  const int pmax = __builtin_amdgcn_readfirstlane(row16_max(p));
  if (pmax < 0) return;
  const int pmin = __builtin_amdgcn_readfirstlane(-row16_max(p < 0 ? -pmax : -p));
  const Keys keys = keys_of<kTile>(a, pmin, pmax);
  const int per = (keys.tiles + a.splits - 1) / a.splits;
  const int t_end = min(keys.tiles, (z + 1) * per);
  if (a.splits > 1 && z * per >= keys.tiles) {
    // a split without keys says so
    if (threadIdx.x < 16 && m0 + threadIdx.x < R)
      a.part_s[((long long)z * heads + bg) * R + m0 + threadIdx.x] = make_float2(-INFINITY, 0.f);
    return;
  }
  const long long base = (long long)b * a.kvBatch + (long long)g * D;

  // the queries are asked for first, and waited for while the first tile's rows come
  Query<D, I4, F32> query;
  query.load(a, b, g, m0 + col, p >= 0, grp);
  __builtin_amdgcn_sched_barrier(0);
  int t = z * per + wave;
  Tile tile = tile_of<kTile>(a, keys, t < t_end ? t : keys.tiles - 1);
  KTile<D, I4> kx;
  VTile<D, I4> vx;
  if (t < t_end) {
    kx.load(a, base, tile, col, grp);
    vx.load(a, base, tile, col, grp);
  }
  __builtin_amdgcn_sched_barrier(0);
  const int up = query.up();
  const float mult = query.mult(a, up);
#pragma unroll
  for (int i = 0; i < QT; ++i)
    if (i % kWaves == wave) {
      half8_t hi, lo;
      query.template operand<I4>(i, up, hi, lo);
      q_s[0][i][lane] = hi;
      if constexpr (F32) q_s[1][i][lane] = lo;
    }
  if (wave == 0 && grp == 0) p_s[col] = p;
  __syncthreads();

  float4_t o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = float4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  bool seen = false;
  while (t < t_end) {
    const int tn = t + kWaves;
    float s[NK];
    {
      float4_t sc[NS];
#pragma unroll
      for (int h = 0; h < NS; ++h) sc[h] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < QT; ++i) {
        const half8_t qh = q_s[0][i][lane];
#pragma unroll
        for (int h = 0; h < NS; ++h) {
          const half8_t k8 = kx.operand(h, i, 0);
          sc[h] = mfma(k8, qh, sc[h]);
          if constexpr (F32) sc[h] = mfma(k8, q_s[1][i][lane], sc[h]);
        }
      }
#pragma unroll
      for (int i = 0; i < NK; ++i) s[i] = sc[i >> 2][i & 3];
    }
    const Tile next = tile_of<kTile>(a, keys, tn < t_end ? tn : t);
    const Sight sight = sight_of(a, keys, t, p);
    if (tn < t_end) kx.load(a, base, next, col, grp);
    if (!tile.whole) {
      int key = tile.key0 + 4 * grp;
      asm volatile("" : "+v"(key));  // (keeps the comparisons below out of whole tiles' way)
#pragma unroll
      for (int i = 0; i < NK; ++i)
        if (!sight(key + (i < 4 ? i : 12 + i))) s[i] = -INFINITY;
    }
    float corr;
    const bool moves = soften(s, mult, m, l, corr);
    if (__builtin_amdgcn_ballot_w64(moves)) {
#pragma unroll
      for (int i = 0; i < DT; ++i) o[i] *= corr;
    }
    Part ph, pl;
    weights(s, ph, pl);
    bool apart = false;
    if (!tile.whole) {
      half2_t zz = {0.f, 0.f};
      vx.each([&](int, Part v) { spot(v, zz); });
      apart = __builtin_amdgcn_ballot_w64(!(zz[0] == 0.f && zz[1] == 0.f)) != 0;
      vx.again();
    }
    if (!apart) {
      vx.each([&](int i, Part v) {
        o[i] = mfma(v, ph, o[i]);
        o[i] = mfma(v, pl, o[i]);
      });
    } else {
      Part vis;
#pragma unroll
      for (int j = 0; j < NK; ++j) vis[j] = sight(tile.key0 + key_of(grp, j)) ? (half_t)1.f : (half_t)0.f;
      if (!seen) {
#pragma unroll 1
        for (int i = 0; i < DT; ++i) seen_s[wave][i][lane] = 0;
        seen = true;
      }
      vx.each([&](int i, Part v) {
        Part mark;
        v = without_marked(v, mark);
        o[i] = mfma(v, ph, o[i]);
        o[i] = mfma(v, pl, o[i]);
        seen_s[wave][i][lane] |= seen_bits(mfma(mark, vis, float4_t{0.f, 0.f, 0.f, 0.f}));
        __builtin_amdgcn_sched_barrier(0);
      });
    }
    if (tn < t_end) vx.load(a, base, next, col, grp);
    tile = next;
    t = tn;
  }

  // merge the waves: outputs by column, then whole rows
  l = column_sum(l);
  if (seen) {
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = with_seen(o[i], seen_s[wave][i][lane]);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) o_s[wave][col][vdim<D, I4>(i, 4 * grp + r)] = o[i][r];
  if (grp == 0) {
    m_s[wave][col] = m;
    l_s[wave][col] = l;
  }
  __syncthreads();
  for (int e = threadIdx.x * 4; e < 16 * D; e += 256 * 4) {
    const int c = e / D, d = e - c * D;
    const int mc = m0 + c;
    if (mc >= R) break;
    float top = m_s[0][c];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, m_s[w][c]);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f, r[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(m_s[w][c] - ref);
      const float4 x = *reinterpret_cast<const float4*>(&o_s[w][c][d]);
      sum += f * l_s[w][c];
      r[0] += f * x.x;
      r[1] += f * x.y;
      r[2] += f * x.z;
      r[3] += f * x.w;
    }
    if (a.splits > 1) {
      const long long row = ((long long)z * heads + bg) * R + mc;
      *reinterpret_cast<float4*>(a.part_o + row * D + d) = make_float4(r[0], r[1], r[2], r[3]);
      if (d == 0) a.part_s[row] = make_float2(top, sum);
    } else if (p_s[c] >= 0) {
      const float inv = 1.f / sum;
      const int i = mc / G;
      const long long at = ((long long)b * a.L + i) * a.ldo + (long long)(g * G + mc - i * G) * D + d;
      if constexpr (F32)
        *reinterpret_cast<float4*>(static_cast<float*>(a.o) + at) = make_float4(r[0] * inv, r[1] * inv, r[2] * inv, r[3] * inv);
      else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at) = make_uint2(pack_half2(r[0] * inv, r[1] * inv), pack_half2(r[2] * inv, r[3] * inv));
    }
  }
}

}  // namespace

int ns2cache::launch_rows(const AttnArgs& a, int D, hipStream_t s) {
  const dim3 grid((unsigned)(a.batch * a.KH * a.splits), (unsigned)((a.L * (a.H / a.KH) + 15) / 16));
#define NS2_ROWS(D_)                                                                             \
  if (a.kg && !a.q_fmt) cache_rows_kernel<D_, true, true><<<grid, 64 * kWaves, 0, s>>>(a);        \
  else if (a.kg) cache_rows_kernel<D_, true, false><<<grid, 64 * kWaves, 0, s>>>(a);              \
  else if (!a.q_fmt) cache_rows_kernel<D_, false, true><<<grid, 64 * kWaves, 0, s>>>(a);          \
  else cache_rows_kernel<D_, false, false><<<grid, 64 * kWaves, 0, s>>>(a);
  NS2_CACHE_D(D, NS2_ROWS)
#undef NS2_ROWS
  NS2_LAUNCHED("cache_rows");
  return NS2_OK;
}
