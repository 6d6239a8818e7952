// A key/value cache: new tokens enter it (head norms, rotation to their positions, fp16 or 4-bit
// storage), and attention of queries at given positions reads it through a causal window with
// first tokens that stay visible.
//
// Cache row (b, j, g) is the D values of K/V head g at position j of sequence b, at value
// b*kvBatch + j*ldkv + g*D. An fp16 cache holds them as they are. A 4-bit cache holds codes c two
// to a byte (the even value in the low four bits) and, per 32 values, an fp16 step s and offset o;
// it stands for the fp16 values half(o + c*s).
#include <algorithm>
#include <cmath>

#include "ns2_cache.h"

using namespace ns2cache;

namespace {

inline bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// ---- new tokens -> queries and cache -----------------------------------------------------------

struct WriteArgs {
  const float* x;  // [rows][ldx]: H query heads, KH key heads, KH value heads of D
  const int* pos;
  const float *w_q, *w_k, *cs;
  void *q, *k, *v;
  half2_t *kg, *vg;
  long long sin_off, kvBatch;
  unsigned units;  // heads of all tokens
  int ldx, ldq, ldkv, L, H, KH, cap, rope_rows, q_fmt;
  float eps;
};

__device__ __forceinline__ float unit8_sum(float v) {
  v += dpp<kDppXor1>(v);
  v += dpp<kDppXor2>(v);
  return v + dpp<kDppHalfMirror>(v);
}

// The same in 64 bits.
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint64_t lo = (uint32_t)dpp_i<CTRL>((int)(uint32_t)u), hi = (uint32_t)dpp_i<CTRL>((int)(u >> 32));
  return __builtin_bit_cast(double, hi << 32 | lo);
}
__device__ __forceinline__ double unit8_sum(double v) {
  v += dpp64<kDppXor1>(v);
  v += dpp64<kDppXor2>(v);
  return v + dpp64<kDppHalfMirror>(v);
}
__device__ __forceinline__ double unit8_min(double v) {
  v = fmin(v, dpp64<kDppXor1>(v));
  v = fmin(v, dpp64<kDppXor2>(v));
  return fmin(v, dpp64<kDppHalfMirror>(v));
}
// Four values of a group of 32 (eight lanes): its step and offset, and their codes, lowest first. A NaN or an
// infinity makes both NaN.
__device__ __forceinline__ uint32_t codes_of(const double (&y)[4], half_t& step, half_t& offset) {
  float bad = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) bad += (float)y[e] - (float)y[e];
  bad = unit8_sum(bad);
  const double lo = unit8_min(fmin(fmin(y[0], y[1]), fmin(y[2], y[3])));
  const double hi = -unit8_min(-fmax(fmax(y[0], y[1]), fmax(y[2], y[3])));
  step = (half_t)((float)((hi - lo) * (1.0 / 15.0)) + bad);
  offset = (half_t)((float)lo + bad);
  const float s = (float)step, inv = s > 0.f ? 1.f / s : 0.f;
  const double s64 = s, o64 = (double)(float)offset;
  uint32_t c = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    // the code next to the quotient in 32 bits, moved where the rest says that another is nearer
    const double d = y[e] - o64;
    float q = rintf((float)d * inv);
    const double rest = 2.0 * fma(-(double)q, s64, d);
    const bool odd = (int)fminf(fmaxf(q, 0.f), 15.f) & 1;
    if (rest > s64 || (rest == s64 && odd)) q += 1.f;
    if (rest < -s64 || (rest == -s64 && odd)) q -= 1.f;
    c |= (uint32_t)(int)(s > 0.f ? fminf(fmaxf(q, 0.f), 15.f) : 0.f) << (4 * e);
  }
  return c;
}

// D / 4 lanes hold one head of one token, four consecutive values each, so that a wave takes 256 / D heads at a
// time: the sum of squares runs over units of 8 lanes (DPP) and then over the head's D / 32 units, the rotation's
// partner i +- D/2 is D / 8 lanes away, and a 4-bit group is one unit of 8 lanes. Every value is read once and
// written once, which bounds it; U times as many heads per wave, all asked for at once, keep the memory busy
// where there are enough of them (8191 tokens x 24 heads of 128 to fp16, the same rows again: 30.6 us with one, 29.7
// with four; rows that come from memory 35.6, 4.3 TB/s; 2048 tokens 9.0, 9.8).
//
// What becomes 4-bit codes is computed in 64 bits, keys from the norm on: a value's last bits in fp32 would decide
// between two codes, a step of the whole value apart, wherever it lies near their border. (Value heads go through the
// norm's sums with the keys and leave the result.) 2400 tokens x 6 heads of 256 8.4 us, in fp32 7.4.
template <int D, bool I4, int U>
__global__ __launch_bounds__(256) void cache_write_kernel(WriteArgs a) {
  constexpr int T = D / 4, HPW = 256 / D;
  const int lane = threadIdx.x & 63;
  const int sub = lane / T, t = lane % T, base = sub * T;
  const unsigned heads = a.H + 2 * a.KH;
  const unsigned u0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * (HPW * U) + sub;
  const bool low = t < T / 2;
  unsigned row[U], h[U];
  bool lives[U];
  int p[U];
  float4 xs[U], cs[U], sn[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    unsigned u = u0 + HPW * i;
    lives[i] = sub < HPW && u < a.units;
    if (!lives[i]) u = 0;  // idle lanes repeat the first head, for the shuffles, and store nothing
    row[i] = u / heads;
    h[i] = u - row[i] * heads;
    p[i] = a.pos[row[i]];
    xs[i] = *reinterpret_cast<const float4*>(a.x + (long long)row[i] * a.ldx + h[i] * D + 4 * t);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    cs[i] = make_float4(1.f, 1.f, 1.f, 1.f);
    sn[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.cs && h[i] < (unsigned)(a.H + a.KH) && p[i] >= 0 && p[i] < a.rope_rows) {
      const long long at = (long long)p[i] * (D / 2) + 4 * (low ? t : t - T / 2);
      cs[i] = *reinterpret_cast<const float4*>(a.cs + at);
      sn[i] = *reinterpret_cast<const float4*>(a.cs + a.sin_off + at);
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    float x[4] = {xs[i].x, xs[i].y, xs[i].z, xs[i].w};
    const bool is_v = h[i] >= (unsigned)(a.H + a.KH), is_q = h[i] < (unsigned)a.H;
    if (!I4 || __builtin_amdgcn_ballot_w64(is_q)) {
      const float* w = is_q ? a.w_q : is_v ? nullptr : a.w_k;
      // (multiply-adds are written out, so that a token's bits do not depend on U)
      const float ss = unit8_sum(fmaf(x[0], x[0], x[1] * x[1]) + fmaf(x[2], x[2], x[3] * x[3]));
      float sum = 0.f;
  #pragma unroll
      for (int n = 0; n < D / 32; ++n) sum += __shfl(ss, (base + 8 * n) & 63);
      if (w) {
        const float r = rsqrtf(fmaf(sum, 1.0f / D, a.eps));
        const float4 w4 = *reinterpret_cast<const float4*>(w + 4 * t);
        x[0] = x[0] * r * w4.x;
        x[1] = x[1] * r * w4.y;
        x[2] = x[2] * r * w4.z;
        x[3] = x[3] * r * w4.w;
      }
      {
        const int partner = (base + (low ? t + T / 2 : t - T / 2)) & 63;
        const float c[4] = {cs[i].x, cs[i].y, cs[i].z, cs[i].w}, s[4] = {sn[i].x, sn[i].y, sn[i].z, sn[i].w};
        float o[4];
  #pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __shfl(x[e], partner);
        if (a.cs && !is_v && p[i] >= 0 && p[i] < a.rope_rows) {
  #pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = fmaf(x[e], c[e], (low ? -o[e] : o[e]) * s[e]);
        }
      }
    }
    const bool held = lives[i] && p[i] >= 0 && p[i] < a.cap;
    uint32_t code = 0;
    half_t step = 0, offset = 0;
    if constexpr (I4) {
      // (lanes of queries take part in the exchanges of the others)
      if (__builtin_amdgcn_ballot_w64(!is_q)) {
        double y[4] = {xs[i].x, xs[i].y, xs[i].z, xs[i].w};
        if (a.w_k) {
          const double s8 = unit8_sum(fma(y[0], y[0], y[1] * y[1]) + fma(y[2], y[2], y[3] * y[3]));
          double all = 0.0;
#pragma unroll
          for (int n = 0; n < D / 32; ++n) all += __shfl(s8, (base + 8 * n) & 63);
          const float4 w4 = *reinterpret_cast<const float4*>(a.w_k + 4 * t);
          const double scale = rsqrt(all / D + (double)a.eps);
          if (!is_v) {
            y[0] *= scale * w4.x;
            y[1] *= scale * w4.y;
            y[2] *= scale * w4.z;
            y[3] *= scale * w4.w;
          }
        }
        const int partner = (base + (low ? t + T / 2 : t - T / 2)) & 63;
        const float c[4] = {cs[i].x, cs[i].y, cs[i].z, cs[i].w}, sv[4] = {sn[i].x, sn[i].y, sn[i].z, sn[i].w};
        double o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __shfl(y[e], partner);
        if (a.cs && !is_v && p[i] >= 0 && p[i] < a.rope_rows) {
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = fma(y[e], (double)c[e], (low ? -o[e] : o[e]) * sv[e]);
        }
        code = codes_of(y, step, offset);
      }
    }
    if (is_q) {
      const long long at = (long long)row[i] * a.ldq + h[i] * D + 4 * t;
      if (held) {
        if (a.q_fmt)
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.q) + at) = make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
        else
          *reinterpret_cast<float4*>(static_cast<float*>(a.q) + at) = make_float4(x[0], x[1], x[2], x[3]);
      }
      continue;
    }
    const unsigned g = is_v ? h[i] - a.H - a.KH : h[i] - a.H;
    const long long at = (long long)(row[i] / (unsigned)a.L) * a.kvBatch + (long long)p[i] * a.ldkv + g * D + 4 * t;
    void* cache = is_v ? a.v : a.k;
    if constexpr (!I4) {
      if (held)
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(cache) + at) = make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
    } else {
      if (held) {
        *reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(cache) + at / 2) = (uint16_t)code;
        if ((t & 7) == 0) (is_v ? a.vg : a.kg)[at / kGroup] = half2_t{step, offset};
      }
    }
  }
}

// ---- attention: the splits joined, and which kernel runs ---------------------------------------------

// One block per column: the splits' sums weighted to their common maximum. D / 4 lanes hold a row of D, so that
// the block's Z groups of lanes take a split each, four at a time in flight; the groups are added in order. What a
// split that saw no key (maximum -inf, sum 0) left as its sums is not taken.
constexpr int kMaxSplits = 64;

template <int D>
__global__ __launch_bounds__(256) void cache_join_kernel(AttnArgs a) {
  constexpr int T = D / 4, PW = 64 / T, Z = 4 * PW;
  __shared__ float4 o_s[Z][T];
  __shared__ float f_s[kMaxSplits];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int G = a.H / a.KH, R = a.L * G;
  const long long columns = (long long)a.batch * a.KH * R, u = blockIdx.x;
  const int bg = (int)(u / R), mc = (int)(u - (long long)bg * R), b = bg / a.KH, g = bg - b * a.KH;
  // everything is asked for at once: the column's position, the splits' statistics and their first sums
  const int p = column_pos(a, b, mc);
  const float2 ml = lane < a.splits ? a.part_s[lane * columns + u] : make_float2(-INFINITY, 0.f);
  const int sub = lane / T, t = lane - sub * T, zg = wave * PW + sub;
  float4 x[4];
  auto load = [&](int z0) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = sub < PW && z0 + i * Z < a.splits ? *reinterpret_cast<const float4*>(a.part_o + ((z0 + i * Z) * columns + u) * D + 4 * t)
                                               : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  load(zg);
  if (p < 0) return;
  float top = ml.x;
  for (int i = 1; i < 64; i <<= 1) top = fmaxf(top, __shfl_xor(top, i));
  const float f = __builtin_amdgcn_exp2f(ml.x - (top == -INFINITY ? 0.f : top));
  const float sum = wave_sum(f * ml.y);
  if (wave == 0) f_s[lane] = ml.x == -INFINITY && ml.y == 0.f ? -1.f : f;
  __syncthreads();
  float r[4] = {0.f, 0.f, 0.f, 0.f};
  for (int z0 = zg; z0 < a.splits; z0 += 4 * Z) {
    if (z0 != zg) load(z0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w = z0 + i * Z < a.splits ? f_s[z0 + i * Z] : -1.f;
      if (w >= 0.f || w != w) {
        r[0] += w * x[i].x;
        r[1] += w * x[i].y;
        r[2] += w * x[i].z;
        r[3] += w * x[i].w;
      }
    }
  }
  if (sub < PW) o_s[zg][t] = make_float4(r[0], r[1], r[2], r[3]);
  __syncthreads();
  if (threadIdx.x >= T) return;
  float4 q = o_s[0][t];
#pragma unroll
  for (int i = 1; i < Z; ++i) {
    const float4 x = o_s[i][t];
    q.x += x.x;
    q.y += x.y;
    q.z += x.z;
    q.w += x.w;
  }
  const float inv = 1.f / sum;
  const int i = mc / G;
  const long long at = ((long long)b * a.L + i) * a.ldo + (long long)(g * G + mc - i * G) * D + 4 * t;
  if (a.q_fmt)
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at) = make_uint2(pack_half2(q.x * inv, q.y * inv), pack_half2(q.z * inv, q.w * inv));
  else
    *reinterpret_cast<float4*>(static_cast<float*>(a.o) + at) = make_float4(q.x * inv, q.y * inv, q.z * inv, q.w * inv);
}

// Columns of a K/V head up to which its keys are streamed past 16 at a time, though they are read again for every 16.
// us, streamed | tiles in LDS: 8 sequences of 4 fp16 heads of 256 on 4096 fp16 keys, 32 columns 18.5 | 18.8, 64 21.9 |
// 22.6, 80 25.1 | 22.7, 128 30.9 | 25.2; 16 heads of 128 over 4 4-bit ones, 32 20.2 | 27.6, 64 28.1 | 29.7, 80 34.6 |
// 35.3, 96 45.9 | 36.2; fp32 queries and long caches of few sequences gain a little more by streaming.
constexpr int kRowsColumns = 64;
constexpr long long kCUs = 256;

Plan plan_of(int batch, int L, int H, int KH, int cap, int window, int sinks) {
  const long long R = (long long)L * (H / KH);
  // keys that a block may have to read
  const long long keys = window ? std::min<long long>(cap, (long long)window + sinks + L) : cap;
  Plan p;
  p.prompt = R > kRowsColumns;
  // enough blocks for the CUs: one each, of few columns two (32 single tokens on 16000 4-bit keys: 34.2 us, with one
  // block each 41.6)
  const long long full = p.prompt ? kCUs : 2 * kCUs;
  const long long heads = std::min((long long)batch * KH, full), tiles = std::min(p.prompt ? (R + 63) / 64 : (R + 15) / 16, full);
  const long long want = full / (heads * tiles);
  // at least 64 keys per split
  const long long most = std::min<long long>(kMaxSplits, std::max<long long>(1, keys / 64));
  p.splits = (int)std::max<long long>(1, std::min(want, most));
  return p;
}

// Whether rows of x (wx bytes, ldx bytes apart) and of y share a byte. Rows that lie between each other's, at one
// distance, do not; at different distances, ranges that meet count as sharing.
bool rows_meet(const void* x, long long ldx, long long wx, const void* y, long long ldy, long long wy, long long rows) {
  const uintptr_t a = (uintptr_t)x, b = (uintptr_t)y;
  if (a + (uintptr_t)((rows - 1) * ldx + wx) <= b || b + (uintptr_t)((rows - 1) * ldy + wy) <= a) return false;
  if (ldx != ldy) return true;
  const long long from = (long long)(b >= a ? (b - a) % ldx : (ldx - (a - b) % ldx) % ldx);  // y's row within x's
  return from < wx || from + wy > ldx;
}

// The argument checks that both entry points share.
int check_cache(const char* fn, const void* q, const int* pos, const void* k, const void* v, const void* kg, const void* vg,
                int batch, int L, int H, int KH, int D, int ldq, int cap, int ldkv, long long kvBatch, int q_fmt) {
  NS2_REQUIRE(q && pos && k && v, "%s: null q, pos, k or v", fn);
  NS2_REQUIRE(D == 64 || D == 96 || D == 128 || D == 256, "%s: head dim %d is not 64, 96, 128 or 256", fn, D);
  NS2_REQUIRE(H > 0 && KH > 0 && H % KH == 0 && (long long)H * D <= INT32_MAX, "%s: H=%d is not a positive multiple of KH=%d", fn, H,
              KH);
  NS2_REQUIRE(cap > 0 && cap <= 1 << 30 && ldq >= H * D && ldkv >= (long long)KH * D && ldkv <= 1 << 24 && kvBatch >= 0,
              "%s: bad sizes or strides (cap=%d, ldq=%d, ldkv=%d)", fn, cap, ldq, ldkv);
  NS2_REQUIRE((long long)batch * L <= INT32_MAX && (long long)batch * L * (H / KH) <= INT32_MAX - 256 && (long long)batch * KH <= 1 << 22,
              "%s: batch=%d, L=%d, H=%d are too many for one launch", fn, batch, L, H);
  NS2_REQUIRE(!kg == !vg, "%s: a 4-bit cache needs the groups of both k and v", fn);
  NS2_REQUIRE(q_fmt == 0 || q_fmt == 1, "%s: q_fmt %d is not 0 (fp32) or 1 (fp16)", fn, q_fmt);
  NS2_REQUIRE(aligned(q, 16) && ldq % (q_fmt ? 8 : 4) == 0 && aligned(pos, 4), "%s: the rows of q must be 16-byte aligned", fn);
  const int unit = kg ? kGroup : 8;
  NS2_REQUIRE(aligned(k, 16) && aligned(v, 16) && aligned(kg, 4) && aligned(vg, 4) && ldkv % unit == 0 && kvBatch % unit == 0,
              "%s: cache rows must be 16-byte aligned (ldkv, kvBatch multiples of %d)", fn, unit);
  return NS2_OK;
}

}  // namespace

extern "C" {

int ns2_head_norm_cache(const float* X, int ldx, const int* pos, const float* w_q, const float* w_k, const float* cs,
                        long long sin_off, int rope_rows, float eps, void* q, int q_fmt, int ldq, void* k, void* v,
                        uint16_t* k_groups, uint16_t* v_groups, int batch, int L, int H, int KH, int D, int cap, int ldkv,
                        long long kvBatch) {
  NS2_READY();
  if (batch <= 0 || L <= 0) return NS2_OK;
  const char* fn = "ns2_head_norm_cache";
  if (int rc = check_cache(fn, q, pos, k, v, k_groups, v_groups, batch, L, H, KH, D, ldq, cap, ldkv, kvBatch, q_fmt)) return rc;
  NS2_REQUIRE(X && aligned(X, 16) && ldx % 4 == 0 && ldx >= (H + 2LL * KH) * D,
              "%s: X must hold 16-byte aligned rows of (H + 2 KH) * D values (ldx=%d)", fn, ldx);
  NS2_REQUIRE(aligned(w_q, 16) && aligned(w_k, 16), "%s: the norm weights must be 16-byte aligned", fn);
  // (in place a lane overwrites what it has read itself, and nothing else, only in rows of the same type and distance)
  const long long rows = (long long)batch * L, wx = 4 * (H + 2LL * KH) * D, wq = (q_fmt ? 2LL : 4LL) * H * D;
  NS2_REQUIRE((q == X && !q_fmt && ldq == ldx) || !rows_meet(X, 4LL * ldx, wx, q, (q_fmt ? 2LL : 4LL) * ldq, wq, rows),
              "%s: q overlaps X (q may be X itself as fp32 with ldq == ldx)", fn);
  if (cs)
    NS2_REQUIRE(aligned(cs, 16) && sin_off % 4 == 0 && rope_rows >= 0 && sin_off >= 0, "%s: the rotation table must be 16-byte aligned",
                fn);
  NS2_REQUIRE(batch == 1 || kvBatch >= (cap - 1LL) * ldkv + KH * D, "%s: the sequences' caches overlap (kvBatch)", fn);
  const long long units = (long long)batch * L * (H + 2LL * KH);  // (below 2^55: batch * L and H + 2 KH are)
  NS2_REQUIRE(units <= INT32_MAX, "%s: %lld heads are too many for one launch", fn, units);
  WriteArgs a{X,  pos, w_q, w_k,  cs,   q, k, v, reinterpret_cast<half2_t*>(k_groups), reinterpret_cast<half2_t*>(v_groups), sin_off, kvBatch,
              (unsigned)units, ldx, ldq, ldkv, L, H, KH, cap, rope_rows, q_fmt, eps};
  // four heads per lane group where that still leaves every SIMD sixteen waves
  const long long waves = (units + 256 / D - 1) / (256 / D);
  const bool four = waves >= 4 * 16 * 4 * kCUs;
  const unsigned grid = (unsigned)((waves + (four ? 15 : 3)) / (four ? 16 : 4));
  hipStream_t s = ns2::stream();
  ns2::ProfScope prof_("head_norm_cache");
#define NS2_WRITE(D_)                                                                    \
  if (k_groups && four) cache_write_kernel<D_, true, 4><<<grid, 256, 0, s>>>(a);          \
  else if (k_groups) cache_write_kernel<D_, true, 1><<<grid, 256, 0, s>>>(a);             \
  else if (four) cache_write_kernel<D_, false, 4><<<grid, 256, 0, s>>>(a);                \
  else cache_write_kernel<D_, false, 1><<<grid, 256, 0, s>>>(a);
  NS2_CACHE_D(D, NS2_WRITE)
#undef NS2_WRITE
  NS2_LAUNCHED("head_norm_cache");
  return NS2_OK;
}

size_t ns2_attention_cache_bytes(int batch, int L, int H, int KH, int D, int cap, int window, int sinks) {
  if (batch <= 0 || L <= 0 || H <= 0 || KH <= 0 || H % KH || D <= 0 || cap <= 0 || window < 0 || sinks < 0) return 0;
  const int splits = plan_of(batch, L, H, KH, cap, window, sinks).splits;
  return splits > 1 ? (size_t)splits * batch * L * H * (D + 2) * sizeof(float) : 0;
}

int ns2_attention_cache(const void* q, int q_fmt, int ldq, const int* pos, const void* k, const void* v, const uint16_t* k_groups,
                        const uint16_t* v_groups, void* o, int ldo, int batch, int L, int H, int KH, int D, int cap, int ldkv,
                        long long kvBatch, int window, int sinks, float scale, void* work, size_t work_bytes) {
  NS2_READY();
  if (batch <= 0 || L <= 0) return NS2_OK;
  const char* fn = "ns2_attention_cache";
  if (int rc = check_cache(fn, q, pos, k, v, k_groups, v_groups, batch, L, H, KH, D, ldq, cap, ldkv, kvBatch, q_fmt)) return rc;
  NS2_REQUIRE(o && aligned(o, 16) && ldo >= H * D && ldo % (q_fmt ? 8 : 4) == 0,
              "%s: o must hold 16-byte aligned rows of H * D values (ldo=%d)", fn, ldo);
  NS2_REQUIRE(window >= 0 && sinks >= 0, "%s: negative window or sinks", fn);
  NS2_REQUIRE(std::isfinite(scale * kLog2e), "%s: the scale is not a finite number", fn);
  const size_t need = ns2_attention_cache_bytes(batch, L, H, KH, D, cap, window, sinks);
  NS2_REQUIRE(work_bytes >= need && (!need || (work && aligned(work, 16))),
              "%s: the call needs %zu bytes of 16-byte aligned work memory (ns2_attention_cache_bytes), got %zu", fn, need, work_bytes);
  const Plan plan = plan_of(batch, L, H, KH, cap, window, sinks);
  NS2_REQUIRE((long long)L * (H / KH) <= 64LL * 65535, "%s: L=%d is too many tokens for one launch", fn, L);
  AttnArgs a{};
  a.q = q;
  a.pos = pos;
  a.k = k;
  a.v = v;
  a.kg = reinterpret_cast<const half2_t*>(k_groups);
  a.vg = reinterpret_cast<const half2_t*>(v_groups);
  a.o = o;
  a.part_o = static_cast<float*>(work);
  if (plan.splits > 1) a.part_s = reinterpret_cast<float2*>(a.part_o + (size_t)plan.splits * batch * L * H * D);
  a.kvBatch = kvBatch;
  a.ldq = ldq;
  a.ldo = ldo;
  a.ldkv = ldkv;
  a.L = L;
  a.H = H;
  a.KH = KH;
  a.cap = cap;
  a.window = window;
  a.sinks = sinks;
  a.q_fmt = q_fmt;
  a.batch = batch;
  a.splits = plan.splits;
  a.scale = scale * kLog2e;
  hipStream_t s = ns2::stream();
  ns2::ProfScope prof_(plan.prompt ? "attention_cache_prompt" : "attention_cache_rows");
  if (int rc = plan.prompt ? launch_prompt(a, D, s) : launch_rows(a, D, s)) return rc;
  if (plan.splits > 1) {
    const long long columns = (long long)batch * L * H;
#define NS2_JOIN(D_) cache_join_kernel<D_><<<(unsigned)columns, 256, 0, s>>>(a);
    NS2_CACHE_D(D, NS2_JOIN)
#undef NS2_JOIN
    NS2_LAUNCHED("cache_join");
  }
  return NS2_OK;
}

}  // extern "C"
