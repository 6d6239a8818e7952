// Attention of many query columns over a cache: prompts and their continuations.
//
// The two products bound it. A block takes 64 CT columns of one K/V head and runs over the keys they see in
// tiles of 64. Its eight waves are four groups of columns (CT tiles of 16 each, queries and accumulators in
// registers) times two halves of every tile, with a softmax state each; the halves are merged at the end. So
// every SIMD has two waves to choose from where one block fills a CU, and a wave reads from LDS only its half
// of a tile. A tile's K and V rows go to LDS once for all waves, as operand fragments, every thread bringing the
// same share of both (the tile ends with the slowest wave): K as it lies, V transposed in registers on the way
// (4 keys x VD dimensions per thread, one byte permutation per pair of values), 4-bit values turned into fp16
// there. The next tile's rows are requested before this one's products. Fragments are 1 KB, lane by lane; the
// 16-byte slots inside one are exchanged (xor) by a pattern of the fragment so that the threads of a row write to
// different banks.
//
// Measured: 2 x 3001 fp32 queries of 16 heads of 128 on 1003 to 4003 4-bit keys of 4 heads 254 us (373 TFLOP/s, and
// twice that in products, since fp32 takes two), 4096 fp16 queries of 4 heads of 256 in a window of 512 28 us (290
// TFLOP/s, and half as much again in products: the weights take two). A tile of the first takes a wave about 5200
// cycles, of which 2048 keep the matrix cores busy; the rest is mostly VALU work of the two waves of a SIMD (300
// instructions each: 4-bit values 115, softmax and weights 134).
// Heads of 256 wait for LDS most: their 64 columns read each fragment four times (2048 of about 4400 cycles a tile,
// products 1536). Four waves of 32 columns, which read it twice, leave a SIMD one wave and took 39 us (with weights
// of one half, where the kernel took 26).
#include "ns2_cache.h"

using namespace ns2cache;

namespace {

constexpr int kTile = 64;  // keys

constexpr int kWaves = 8, kThreads = 64 * kWaves, kGroups = kWaves / 2;  // (groups of columns)

// What one of the T threads brings of a tile from memory to LDS: NK pieces of 8 dimensions of K rows, and NV blocks of
// 4 keys x VD dimensions of V.
template <int D, bool I4>
struct Stage {
  static constexpr int T = kThreads;
  static constexpr int C = D / 8, KU = kTile * C, NK = (KU + T - 1) / T;  // pieces of a K row, of a tile, of a thread
  static constexpr int VD = D == 256 ? 8 : D >= 96 ? 4 : 2, VC = D / VD, VU = kTile / 4 * VC, NV = (VU + T - 1) / T;
  uint32_t k[NK][I4 ? 1 : 4], kg[I4 ? NK : 1], v[NV][I4 ? 4 : 2 * VD], vg[I4 ? NV : 1][4];

  static __device__ __forceinline__ bool has_k(int u) { return KU % T == 0 || u < KU; }
  static __device__ __forceinline__ bool has_v(int u) { return VU % T == 0 || u < VU; }
  // Block u: four keys from 32 (q / 4) + 4 (q % 4) + 16 h on, where 2 q + h is the half fragment it goes to. (The two
  // halves are neighbours, so that 16 lanes write 16 different 8-byte banks; the last threads start, since the first
  // have a K piece more where T does not divide them.)
  static __device__ __forceinline__ int block_of(int tid, int i) { return T - 1 - tid + T * i; }
  static __device__ __forceinline__ int column_of(int u) { return (u >> 1) % VC; }
  static __device__ __forceinline__ int q_of(int u) { return (u >> 1) / VC; }
  static __device__ __forceinline__ int key_of(int u) { return 32 * (q_of(u) >> 2) + 4 * (q_of(u) & 3) + 16 * (u & 1); }

  __device__ __forceinline__ void load(const AttnArgs& a, long long base, const Tile& t, int tid) {
    const int last = t.end - 1 - t.key0;
    {
      const char* rows = tile_rows(a.k, base, t.key0, a.ldkv, I4);
      const half2_t* groups = I4 ? tile_groups(a.kg, base, t.key0, a.ldkv) : nullptr;
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const int u = tid + T * i;
        if (!has_k(u)) continue;
        const uint32_t at = (uint32_t)(min(u / C, last) * a.ldkv + 8 * (u % C));
        if constexpr (I4) {
          k[i][0] = *reinterpret_cast<const uint32_t*>(rows + at / 2);
          kg[i] = __builtin_bit_cast(uint32_t, groups[at / kGroup]);
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(rows + 2u * at);
          k[i][0] = x.x;
          k[i][1] = x.y;
          k[i][2] = x.z;
          k[i][3] = x.w;
        }
      }
    }
    const char* rows = tile_rows(a.v, base, t.key0, a.ldkv, I4);
    const half2_t* groups = I4 ? tile_groups(a.vg, base, t.key0, a.ldkv) : nullptr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = block_of(tid, i);
      if (!has_v(u)) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t at = (uint32_t)(min(key_of(u) + j, last) * a.ldkv + VD * column_of(u));
        if constexpr (I4) {
          v[i][j] = VD == 8   ? *reinterpret_cast<const uint32_t*>(rows + at / 2)
                    : VD == 4 ? *reinterpret_cast<const uint16_t*>(rows + at / 2)
                              : *reinterpret_cast<const uint8_t*>(rows + at / 2);
          vg[i][j] = __builtin_bit_cast(uint32_t, groups[at / kGroup]);
        } else if constexpr (VD == 8) {
          const uint4 x = *reinterpret_cast<const uint4*>(rows + 2u * at);
          v[i][4 * j] = x.x;
          v[i][4 * j + 1] = x.y;
          v[i][4 * j + 2] = x.z;
          v[i][4 * j + 3] = x.w;
        } else if constexpr (VD == 4) {
          const uint2 x = *reinterpret_cast<const uint2*>(rows + 2u * at);
          v[i][2 * j] = x.x;
          v[i][2 * j + 1] = x.y;
        } else {
          v[i][j] = *reinterpret_cast<const uint32_t*>(rows + 2u * at);
        }
      }
    }
  }

  // K fragment (key tile kt, step t): lane (key % 16, grp) holds dimensions 32 t + 8 grp ..
  __device__ __forceinline__ void store_k(half8_t* ksm, int tid) const {
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int u = tid + T * i, key = u / C, c = u % C;
      if (!has_k(u)) continue;
      half8_t x;
      if constexpr (I4) x = dequant8(k[i][0], __builtin_bit_cast(half2_t, kg[i]));
      else x = __builtin_bit_cast(half8_t, make_uint4(k[i][0], k[i][1], k[i][2], k[i][3]));
      ksm[((key >> 4) * (D / 32) + (c >> 2)) * 64 + (c & 3) * 16 + ((key ^ c) & 15)] = x;
    }
  }

  // V fragment (step t, tile half): lane (dimension % 16, grp) holds the eight keys of grp. Returns NaN if a value
  // is not finite and `check` is set.
  static __device__ __forceinline__ int v_slot(int t, int d) { return d ^ (t & (VD - 1)) ^ ((d >> 3) * (VD / 2)); }
  __device__ __forceinline__ half2_t store_v(half8_t* vsm, int tid, bool check) const {
    half2_t z = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = block_of(tid, i), c = column_of(u), q = q_of(u);
      if (!has_v(u)) continue;
      uint32_t r[VD][2];  // [dimension][key pair]
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (I4) {
          const half2_t s = __builtin_bit_cast(half2_t, pair_lo(vg[i][2 * j], vg[i][2 * j + 1]));
          const half2_t o = __builtin_bit_cast(half2_t, pair_hi(vg[i][2 * j], vg[i][2 * j + 1]));
#pragma unroll
          for (int h = 0; h < (VD + 3) / 4; ++h) {
            uint32_t x[4];
            dequant4(h ? pair_hi(v[i][2 * j], v[i][2 * j + 1]) : pair_lo(v[i][2 * j], v[i][2 * j + 1]), s, o, x);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (4 * h + e < VD) r[4 * h + e][j] = x[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < VD / 2; ++e) {
            const uint32_t x = v[i][2 * j * (VD / 2) + e], y = v[i][(2 * j + 1) * (VD / 2) + e];
            r[2 * e][j] = pair_lo(x, y);
            r[2 * e + 1][j] = pair_hi(x, y);
          }
        }
      }
      const int t = VD * c >> 4;
#pragma unroll
      for (int e = 0; e < VD; ++e) {
        const uint2 x = make_uint2(r[e][0], r[e][1]);
        if (check) spot(__builtin_bit_cast(half4_t, x), z);
        reinterpret_cast<uint2*>(vsm + (t * 2 + (q >> 2)) * 64 + (q & 3) * 16 + v_slot(t, (VD * c & 15) + e))[u & 1] = x;
      }
    }
    return z;
  }
};

template <int D, bool I4, bool F32, int CT>
__global__ __launch_bounds__(kThreads, 2) void cache_prompt_kernel(AttnArgs a) {
  typedef Stage<D, I4> Bring;
  constexpr int DT = D / 16, QT = D / 32, kColumns = 16 * CT * kGroups;
  constexpr int kFrags = 4 * QT + 2 * DT, kMerge = kGroups * CT * (DT + 1);  // KB of a tile; of the second halves' sums
  __shared__ __attribute__((aligned(16))) half8_t smem[(2 * kFrags > kMerge ? 2 * kFrags : kMerge) * 64];
  __shared__ uint8_t seen_s[kWaves][CT * DT][64];  // values that were not finite
  __shared__ int bad_s[2];                    // 1 + the last tile in this buffer with such a V value
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int half = wave / kGroups, wc = wave - half * kGroups;  // of a tile; column group
  const int col = lane & 15, grp = lane >> 4;
  const int G = a.H / a.KH, R = a.L * G;
  // Blocks go to the eight dies in turn, the columns with the most keys first. A die would see few of the
  // heads then (fewer keys for its cache) but also few of the sequences, which may differ in length: every four
  // column blocks the sequences move on by one (8 sequences of 333 to 1000 tokens on a cache of 1003: 168 us
  // without, 120 with; of equal lengths the same). In a window, where neighbours share keys, each die takes a run of
  // columns (27.0 us without, 26.0 with, 4096 tokens and heads of 256).
  int by = gridDim.y - 1 - blockIdx.y, bx = (blockIdx.x + blockIdx.y / 4 * (a.KH * a.splits)) % gridDim.x;
  if (a.window) {
    const int n = gridDim.x * gridDim.y, id = blockIdx.x + gridDim.x * blockIdx.y, even = n / 8, odd = n - 8 * even;
    const int die = id & 7, at = die * even + min(die, odd) + (id >> 3);
    bx = at / gridDim.y;
    by = at - bx * gridDim.y;
  }
  const int z = bx % a.splits, bg = bx / a.splits;
  const int b = bg / a.KH, g = bg - b * a.KH;
  const int m0 = by * kColumns;

  // the block's first and last position
  int hi_p = -1, lo_p = INT32_MAX;
#pragma unroll
  for (int i = 0; i < kColumns / 64; ++i) {
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

  Bring st;
  Tile tile = tile_of<kTile>(a, keys, t0 < t1 ? t0 : 0);
  if (t0 < t1) st.load(a, base, tile, threadIdx.x);
  half8_t qh[CT][QT], ql[CT][F32 ? QT : 1];
  float mult[CT], m[CT], l[CT];
  int p[CT];
  float4_t o[CT][DT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int mc = m0 + (wc * CT + c) * 16 + col;
    p[c] = column_pos(a, b, mc);
    Query<D, false, F32> query;
    query.load(a, b, g, mc, p[c] >= 0, grp);
    const int up = query.up();
    mult[c] = query.mult(a, up);
#pragma unroll
    for (int i = 0; i < QT; ++i) query.template operand<I4>(i, up, qh[c][i], ql[c][F32 ? i : 0]);
    m[c] = -INFINITY;
    l[c] = 0.f;
#pragma unroll
    for (int i = 0; i < DT; ++i) o[c][i] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
  bool seen = false;
  // tile t + 1's fragments are written while tile t's are used: one barrier per tile
  auto store = [&](int t, const Tile& tl) {
    half8_t* k_s = smem + ((t - t0) & 1) * (kFrags * 64);
    st.store_k(k_s, threadIdx.x);
    const half2_t zz = st.store_v(k_s + 4 * QT * 64, threadIdx.x, !tl.whole);
    if (!(zz[0] == 0.f && zz[1] == 0.f)) bad_s[(t - t0) & 1] = t + 1;
  };
  if (threadIdx.x < 2) bad_s[threadIdx.x] = 0;
  __syncthreads();
  Tile next = tile_of<kTile>(a, keys, t0 + 1 < t1 ? t0 + 1 : t0);
  if (t0 < t1) store(t0, tile);
  if (t0 + 1 < t1) st.load(a, base, next, threadIdx.x);
  __syncthreads();

  for (int t = t0; t < t1; ++t) {
    const half8_t* k_s = smem + ((t - t0) & 1) * (kFrags * 64);
    half8_t* v_s = smem + ((t - t0) & 1) * (kFrags * 64) + 4 * QT * 64;
    float4_t s[CT][2];
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) s[c][kt] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < QT; ++i)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const half8_t k8 = k_s[((2 * half + kt) * QT + i) * 64 + grp * 16 + ((col ^ (4 * i + grp)) & 15)];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          s[c][kt] = mfma(k8, qh[c][i], s[c][kt]);
          if constexpr (F32) s[c][kt] = mfma(k8, ql[c][i], s[c][kt]);
        }
      }
    const Tile after = tile_of<kTile>(a, keys, t + 2 < t1 ? t + 2 : t);
    if (t + 1 < t1) {
      store(t + 1, next);
      if (t + 2 < t1) st.load(a, base, after, threadIdx.x);
    }
    half8_t ph[CT], pl[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = s[c][i >> 2][i & 3];
      if (!tile.whole) {
        const Sight sight = sight_of(a, keys, t, p[c]);
        int key = tile.key0 + 32 * half + 4 * grp;
        asm volatile("" : "+v"(key));  // (keeps the comparisons below out of whole tiles' way)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!sight(key + 16 * (i >> 2) + (i & 3))) w[i] = -INFINITY;
      }
      float corr;
      const bool moves = soften(w, mult[c], m[c], l[c], corr);
      if (__builtin_amdgcn_ballot_w64(moves)) {
#pragma unroll
        for (int i = 0; i < DT; ++i) o[c][i] *= corr;
      }
      weights(w, ph[c], pl[c]);
    }
    if (!tile.whole && bad_s[(t - t0) & 1] == t + 1) {  // (for all waves)
      half8_t vis[CT];
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        const Sight sight = sight_of(a, keys, t, p[c]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          vis[c][j] = sight(tile.key0 + 32 * half + 4 * grp + (j < 4 ? j : 12 + j)) ? (half_t)1.f : (half_t)0.f;
      }
#pragma unroll 1
      for (int i = 0; i < DT; ++i) {
        half8_t mark;
        without_marked(v_s[(i * 2 + half) * 64 + grp * 16 + Bring::v_slot(i, col)], mark);
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          uint8_t* w = &seen_s[wave][c * DT + i][lane];
          *w = (seen ? *w : 0) | seen_bits(mfma(mark, vis[c], float4_t{0.f, 0.f, 0.f, 0.f}));
        }
      }
      seen = true;
      __syncthreads();  // every wave has the marks: the values go
#pragma unroll 1
      for (int i = threadIdx.x; i < 2 * DT * 64; i += kThreads) {
        half8_t mark;
        v_s[i] = without_marked(v_s[i], mark);
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      const half8_t v8 = v_s[(i * 2 + half) * 64 + grp * 16 + Bring::v_slot(i, col)];
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        o[c][i] = mfma(v8, ph[c], o[c][i]);
        o[c][i] = mfma(v8, pl[c], o[c][i]);
      }
    }
    tile = next;
    next = after;
    __syncthreads();
  }

  if (seen) {
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int i = 0; i < DT; ++i) o[c][i] = with_seen(o[c][i], seen_s[wave][c * DT + i][lane]);
  }

  // the second halves' sums through LDS to the first's
  float4_t* o_s = reinterpret_cast<float4_t*>(smem) + wc * (CT * DT * 64);
  float2* ml_s = reinterpret_cast<float2*>(reinterpret_cast<float4_t*>(smem) + kGroups * CT * DT * 64) + wc * (CT * 64);
  if (half) {
#pragma unroll
    for (int c = 0; c < CT; ++c) {
#pragma unroll
      for (int i = 0; i < DT; ++i) o_s[(c * DT + i) * 64 + lane] = o[c][i];
      ml_s[c * 64 + lane] = make_float2(m[c], l[c]);
    }
  }
  __syncthreads();
  if (half) return;
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const float2 ml = ml_s[c * 64 + lane];
    const float top = fmaxf(m[c], ml.x), ref = top == -INFINITY ? 0.f : top;
    const float f0 = __builtin_amdgcn_exp2f(m[c] - ref), f1 = __builtin_amdgcn_exp2f(ml.x - ref);
    const float sum = column_sum(f0 * l[c] + f1 * ml.y);
    const int mc = m0 + (wave * CT + c) * 16 + col;
    if (p[c] < 0) continue;
    const int i0 = mc / G;
    const long long row = ((long long)z * a.batch * a.KH + bg) * R + mc;
    const long long at = ((long long)b * a.L + i0) * a.ldo + (long long)(g * G + mc - i0 * G) * D + 4 * grp;
    const float inv = a.splits > 1 ? 1.f : 1.f / sum;
    if (a.splits > 1 && grp == 0) a.part_s[row] = make_float2(top, sum);
#pragma unroll
    for (int i = 0; i < DT; ++i) {
      const float4_t r = (o[c][i] * f0 + o_s[(c * DT + i) * 64 + lane] * f1) * inv;
      if (a.splits > 1)
        *reinterpret_cast<float4*>(a.part_o + row * D + 16 * i + 4 * grp) = make_float4(r[0], r[1], r[2], r[3]);
      else if constexpr (F32)
        *reinterpret_cast<float4*>(static_cast<float*>(a.o) + at + 16 * i) = make_float4(r[0], r[1], r[2], r[3]);
      else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at + 16 * i) = make_uint2(pack_half2(r[0], r[1]), pack_half2(r[2], r[3]));
    }
  }
}

template <int D, bool I4, bool F32>
void launch(const AttnArgs& a, hipStream_t s) {
  const int R = a.L * (a.H / a.KH);
  const unsigned x = (unsigned)(a.batch * a.KH * a.splits);
  // two column tiles per wave where that leaves every CU a block and the registers hold them (2 x 3001 queries of 16
  // heads of 128: 342 us with one, 244 with two; 1200 queries, 40 blocks x 4 heads: 27, 35)
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
