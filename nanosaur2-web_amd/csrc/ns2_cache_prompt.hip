// Attention of many query columns over a cache: prompts and their continuations.
//
// The two products bound it. A block takes 64 CT columns of one K/V head (CT tiles of 16 in each of its four
// waves, queries and accumulators in registers) and runs over the keys they see in tiles of 64. A tile's K
// and V rows go to LDS once for all waves, as operand fragments: K as it lies, V transposed in registers on
// the way (8 keys x 8 dimensions per thread, one byte permutation per pair of values), 4-bit values turned
// into fp16 there. The next tile's rows are requested before this one's products. Fragments are 1 KB, lane by
// lane; the 16-byte slots inside one are exchanged (xor) by a pattern of the fragment so that the threads
// of a row write to different banks.
#include "ns2_cache.h"

using namespace ns2cache;

namespace {

constexpr int kTile = 64;  // keys
constexpr int kThreads = 256;

// What one thread brings of a tile from memory to LDS: NK pieces of 8 dimensions of a K row and NV blocks of
// 8 keys x 8 dimensions of V.
template <int D, bool I4>
struct Stage {
  static constexpr int C = D / 8;                                 // 8-dimension pieces of a row
  static constexpr int NK = (kTile * C + kThreads - 1) / kThreads;  // pieces of K per thread
  static constexpr int VB = 8 * C;                                // 8x8 blocks of V
  static constexpr int NV = (VB + kThreads - 1) / kThreads;
  typename std::conditional<I4, uint32_t, uint4>::type k[NK], v[NV][8];
  uint32_t ks[I4 ? NK : 1], vs[I4 ? NV : 1][8];

  __device__ __forceinline__ void load(const AttnArgs& a, long long base, const Tile& t) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int u = tid + kThreads * i, key = t.key0 + u / C, c = u % C;
      if (kTile * C % kThreads == 0 || u < kTile * C) {
        const long long at = base + (long long)(key < t.end ? key : t.end - 1) * a.ldkv + 8 * c;
        if constexpr (I4) {
          k[i] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.k) + at / 2);
          ks[i] = reinterpret_cast<const uint32_t*>(a.kg)[at / kGroup];
        } else {
          k[i] = *reinterpret_cast<const uint4*>(static_cast<const half_t*>(a.k) + at);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = tid + kThreads * i, c = u % C, q = u / C;  // q = 4 (key step) + lane group
      if (VB % kThreads == 0 || u < VB) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = t.key0 + 32 * (q >> 2) + 4 * (q & 3) + (j < 4 ? j : 12 + j);
          const long long at = base + (long long)(key < t.end ? key : t.end - 1) * a.ldkv + 8 * c;
          if constexpr (I4) {
            v[i][j] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.v) + at / 2);
            vs[i][j] = reinterpret_cast<const uint32_t*>(a.vg)[at / kGroup];
          } else {
            v[i][j] = *reinterpret_cast<const uint4*>(static_cast<const half_t*>(a.v) + at);
          }
        }
      }
    }
  }

  // K fragment (key tile kt, step t): lane (key % 16, grp) holds dimensions 32 t + 8 grp ..; V fragment (step t,
  // key step ks): lane (dimension % 16, grp) holds the eight keys of grp. Returns NaN if a V value is not finite.
  __device__ __forceinline__ half2_t store(half8_t* ksm, half8_t* vsm, bool check) const {
    const int tid = threadIdx.x;
    half2_t z = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int u = tid + kThreads * i, key = u / C, c = u % C;
      if (kTile * C % kThreads == 0 || u < kTile * C) {
        half8_t x;
        if constexpr (I4) x = dequant8(k[i], __builtin_bit_cast(half2_t, ks[i]));
        else x = __builtin_bit_cast(half8_t, k[i]);
        ksm[((key >> 4) * (D / 32) + (c >> 2)) * 64 + (c & 3) * 16 + ((key ^ c) & 15)] = x;
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = tid + kThreads * i, c = u % C, q = u / C;
      if (VB % kThreads == 0 || u < VB) {
        uint32_t r[8][4];  // [dimension][key pair]
        if constexpr (I4) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const half2_t s = __builtin_bit_cast(half2_t, pair_lo(vs[i][2 * j], vs[i][2 * j + 1]));
            const half2_t o = __builtin_bit_cast(half2_t, pair_hi(vs[i][2 * j], vs[i][2 * j + 1]));
            uint32_t x[4], y[4];
            dequant4(pair_lo(v[i][2 * j], v[i][2 * j + 1]), s, o, x);
            dequant4(pair_hi(v[i][2 * j], v[i][2 * j + 1]), s, o, y);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              r[e][j] = x[e];
              r[4 + e][j] = y[e];
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t x[4] = {v[i][2 * j].x, v[i][2 * j].y, v[i][2 * j].z, v[i][2 * j].w};
            const uint32_t y[4] = {v[i][2 * j + 1].x, v[i][2 * j + 1].y, v[i][2 * j + 1].z, v[i][2 * j + 1].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              r[2 * e][j] = pair_lo(x[e], y[e]);
              r[2 * e + 1][j] = pair_hi(x[e], y[e]);
            }
          }
        }
        const int t = c >> 1;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const half8_t x = __builtin_bit_cast(half8_t, make_uint4(r[e][0], r[e][1], r[e][2], r[e][3]));
          if (check) spot(x, z);
          vsm[(t * 2 + (q >> 2)) * 64 + (q & 3) * 16 + (((c & 1) * 8 + e) ^ (t & 7))] = x;
        }
      }
    }
    return z;
  }
};

template <int D, bool I4, bool F32, int CT>
__global__ __launch_bounds__(kThreads) void cache_prompt_kernel(AttnArgs a) {
  constexpr int DT = D / 16, QT = D / 32;
  __shared__ __attribute__((aligned(16))) half8_t k_s[4 * QT * 64];
  __shared__ __attribute__((aligned(16))) half8_t v_s[DT * 2 * 64];
  __shared__ int bad_s;  // 1 + the last tile with a V value that is not finite
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int col = lane & 15, grp = lane >> 4;
  const int G = a.H / a.KH, R = a.L * G;
  const int z = blockIdx.x % a.splits, bg = blockIdx.x / a.splits;
  const int b = bg / a.KH, g = bg - b * a.KH;
  const int m0 = (gridDim.y - 1 - blockIdx.y) * (64 * CT);  // the columns with the most keys first

  // the block's first and last position
  int hi_p = -1, lo_p = INT32_MAX;
#pragma unroll
  for (int i = 0; i < CT; ++i) {
    const int p = column_pos(a, b, m0 + 64 * i + lane);
    hi_p = max(hi_p, p);
    lo_p = p < 0 ? lo_p : min(lo_p, p);
  }
  for (int i = 1; i < 64; i <<= 1) {
    hi_p = max(hi_p, __shfl_xor(hi_p, i));
    lo_p = min(lo_p, __shfl_xor(lo_p, i));
  }
  hi_p = __builtin_amdgcn_readfirstlane(hi_p);
  lo_p = __builtin_amdgcn_readfirstlane(lo_p);
  if (hi_p < 0) return;
  const Keys keys = keys_of<kTile>(a, lo_p, hi_p);
  const int per = (keys.tiles + a.splits - 1) / a.splits;
  const int t0 = z * per, t1 = min(keys.tiles, t0 + per);
  const long long base = (long long)b * a.kvBatch + (long long)g * D;

  Stage<D, I4> st;
  Tile tile = tile_of<kTile>(a, keys, t0 < t1 ? t0 : 0);
  if (t0 < t1) st.load(a, base, tile);
  half8_t qh[CT][QT], ql[CT][F32 ? QT : 1];
  Query<F32> query[CT];
  float m[CT], l[CT];
  int p[CT];
  float4_t o[CT][DT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int mc = m0 + (wave * CT + c) * 16 + col;
    p[c] = column_pos(a, b, mc);
    query[c].template open<D, false>(a, b, g, mc, p[c] >= 0, grp);
#pragma unroll
    for (int i = 0; i < QT; ++i) query[c].template operand<D, false, I4>(i, grp, qh[c][i], ql[c][F32 ? i : 0]);
    m[c] = -INFINITY;
    l[c] = 0.f;
#pragma unroll
    for (int i = 0; i < DT; ++i) o[c][i] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
  if (threadIdx.x == 0) bad_s = 0;

  for (int t = t0; t < t1; ++t) {
    __syncthreads();  // the last tile's fragments are used
    {
      const half2_t zz = st.store(k_s, v_s, !tile.whole);
      if (!(zz[0] == 0.f && zz[1] == 0.f)) bad_s = t + 1;
    }
    __syncthreads();
    const Tile next = tile_of<kTile>(a, keys, t + 1 < t1 ? t + 1 : t);
    if (t + 1 < t1) st.load(a, base, next);

    float4_t s[CT][4];
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) s[c][kt] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < QT; ++i)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        const half8_t k8 = k_s[(kt * QT + i) * 64 + grp * 16 + ((col ^ (4 * i + grp)) & 15)];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          s[c][kt] = mfma(k8, qh[c][i], s[c][kt]);
          if constexpr (F32) s[c][kt] = mfma(k8, ql[c][i], s[c][kt]);
        }
      }
    half8_t ph[CT][2], pl[CT][2];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      float w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = s[c][i >> 2][i & 3] * query[c].mult;
      if (!tile.whole) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!sees(a, p[c], tile.key0 + 16 * (i >> 2) + 4 * grp + (i & 3), tile.end)) w[i] = -INFINITY;
      }
      float corr;
      const bool moves = soften(w, m[c], l[c], corr);
      if (__builtin_amdgcn_ballot_w64(moves)) {
#pragma unroll
        for (int i = 0; i < DT; ++i) o[c][i] *= corr;
      }
      weights<F32>(w, ph[c][0], pl[c][0]);
      weights<F32>(w + 8, ph[c][1], pl[c][1]);
    }
    const bool apart = !tile.whole && bad_s == t + 1;
    if (!apart) {
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const half8_t v8 = v_s[(i * 2 + ks) * 64 + grp * 16 + (col ^ (i & 7))];
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            o[c][i] = mfma(v8, ph[c][ks], o[c][i]);
            if constexpr (F32) o[c][i] = mfma(v8, pl[c][ks], o[c][i]);
          }
        }
    } else {
#pragma unroll 1
      for (int ks = 0; ks < 2; ++ks) {
        half8_t vis[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
          for (int j = 0; j < 8; ++j)
            vis[c][j] = sees(a, p[c], tile.key0 + 32 * ks + 4 * grp + (j < 4 ? j : 12 + j), tile.end) ? (half_t)1.f : (half_t)0.f;
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          half8_t mark;
          const half8_t v8 = without_marked(v_s[(i * 2 + ks) * 64 + grp * 16 + (col ^ (i & 7))], mark);
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            o[c][i] = mfma(v8, ks ? ph[c][1] : ph[c][0], o[c][i]);
            if constexpr (F32) o[c][i] = mfma(v8, ks ? pl[c][1] : pl[c][0], o[c][i]);
            o[c][i] = with_seen(o[c][i], mfma(mark, vis[c], float4_t{0.f, 0.f, 0.f, 0.f}));
          }
        }
      }
    }
    tile = next;
  }

#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const float sum = column_sum(l[c]);
    const int mc = m0 + (wave * CT + c) * 16 + col;
    if (p[c] < 0) continue;
    if (a.splits > 1) {
      const long long row = ((long long)z * a.batch * a.KH + bg) * R + mc;
#pragma unroll
      for (int i = 0; i < DT; ++i)
        *reinterpret_cast<float4*>(a.part_o + row * D + 16 * i + 4 * grp) = make_float4(o[c][i][0], o[c][i][1], o[c][i][2], o[c][i][3]);
      if (grp == 0) a.part_s[row] = make_float2(m[c], sum);
    } else {
      const float inv = 1.f / sum;
      const int i0 = mc / G;
      const long long at = ((long long)b * a.L + i0) * a.ldo + (long long)(g * G + mc - i0 * G) * D + 4 * grp;
#pragma unroll
      for (int i = 0; i < DT; ++i) {
        const float4_t r = o[c][i] * inv;
        if constexpr (F32) *reinterpret_cast<float4*>(static_cast<float*>(a.o) + at + 16 * i) = make_float4(r[0], r[1], r[2], r[3]);
        else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at + 16 * i) = make_uint2(pack_half2(r[0], r[1]), pack_half2(r[2], r[3]));
      }
    }
  }
}

template <int D, bool I4, bool F32>
void launch(const AttnArgs& a, hipStream_t s) {
  const int R = a.L * (a.H / a.KH);
  const unsigned x = (unsigned)(a.batch * a.KH * a.splits);
  // two column tiles per wave where that leaves every CU a block (and the registers hold them)
  if constexpr (D < 256) {
    if ((long long)x * ((R + 127) / 128) >= 256) {
      cache_prompt_kernel<D, I4, F32, 2><<<dim3(x, (R + 127) / 128), kThreads, 0, s>>>(a);
      return;
    }
  }
  cache_prompt_kernel<D, I4, F32, 1><<<dim3(x, (R + 63) / 64), kThreads, 0, s>>>(a);
}

}  // namespace

int ns2cache::launch_prompt(const AttnArgs& a, int D, hipStream_t s) {
#define NS2_PROMPT(D_)                                \
  if (a.kg && !a.q_fmt) launch<D_, true, true>(a, s);  \
  else if (a.kg) launch<D_, true, false>(a, s);        \
  else if (!a.q_fmt) launch<D_, false, true>(a, s);    \
  else launch<D_, false, false>(a, s);
  NS2_CACHE_D(D, NS2_PROMPT)
#undef NS2_PROMPT
  NS2_LAUNCHED("cache_prompt");
  return NS2_OK;
}
