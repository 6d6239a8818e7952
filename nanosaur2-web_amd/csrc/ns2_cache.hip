// A key/value cache: new tokens enter it (head norms, rotation to their positions, fp16 or 4-bit
// storage), and attention of queries at given positions reads it through a causal window with
// first tokens that stay visible.
//
// Cache row (b, j, g) is the D values of K/V head g at position j of sequence b, at value
// b*kvBatch + j*ldkv + g*D. An fp16 cache holds them as they are. A 4-bit cache holds codes c two
// to a byte (the even value in the low four bits) and, per 32 values, an fp16 step s and offset o;
// it stands for the fp16 values half(o + c*s).
#include "ns2_common.h"

using namespace ns2dev;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kGroup = 32;  // values per step and offset of a 4-bit cache

inline bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// ---- new tokens -> queries and cache -----------------------------------------------------------

struct WriteArgs {
  const float* x;  // [rows][ldx]: H query heads, KH key heads, KH value heads of D
  const int* pos;
  const float *w_q, *w_k, *cs;
  void *q, *k, *v;
  half2_t *kg, *vg;
  long long sin_off, kvBatch, rows;
  int ldx, ldq, ldkv, L, H, KH, cap, rope_rows, q_fmt;
  float eps;
};

__device__ __forceinline__ float unit8_sum(float v) {
  v += dpp<kDppXor1>(v);
  v += dpp<kDppXor2>(v);
  return v + dpp<kDppHalfMirror>(v);
}
__device__ __forceinline__ float unit8_min(float v) {
  v = fminf(v, dpp<kDppXor1>(v));
  v = fminf(v, dpp<kDppXor2>(v));
  return fminf(v, dpp<kDppHalfMirror>(v));
}

// D / 4 lanes hold one head of one token, four consecutive values each, so that a wave takes
// 256 / D heads: the sum of squares runs over units of 8 lanes (DPP) and then over the head's
// D / 32 units, the rotation's partner i +- D/2 is D / 8 lanes away, and a 4-bit group is one unit
// of 8 lanes. Every value is read once and written once.
template <int D, bool I4>
__global__ __launch_bounds__(256) void cache_write_kernel(WriteArgs a) {
  constexpr int T = D / 4, HPW = 64 / T;
  const int lane = threadIdx.x & 63;
  const int sub = lane / T, t = lane % T, base = sub * T;
  const int heads = a.H + 2 * a.KH;
  long long u = ((long long)blockIdx.x * 4 + (threadIdx.x >> 6)) * HPW + sub;
  const bool lives = sub < HPW && u < a.rows * heads;
  if (!lives) u = 0;  // idle lanes repeat the first head, for the shuffles, and store nothing
  const long long row = u / heads;
  const int h = (int)(u - row * heads);
  const int p = a.pos[row];
  const float4 x4 = *reinterpret_cast<const float4*>(a.x + row * a.ldx + (long long)h * D + 4 * t);
  float x[4] = {x4.x, x4.y, x4.z, x4.w};
  const bool is_v = h >= a.H + a.KH;
  const float* w = h < a.H ? a.w_q : is_v ? nullptr : a.w_k;
  {
    const float ss = unit8_sum((x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3]));
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) sum += __shfl(ss, (base + 8 * i) & 63);
    if (w) {
      const float r = rsqrtf(sum / (float)D + a.eps);
      const float4 w4 = *reinterpret_cast<const float4*>(w + 4 * t);
      x[0] = x[0] * r * w4.x;
      x[1] = x[1] * r * w4.y;
      x[2] = x[2] * r * w4.z;
      x[3] = x[3] * r * w4.w;
    }
  }
  {
    const bool low = t < T / 2;
    const int partner = (base + (low ? t + T / 2 : t - T / 2)) & 63;
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __shfl(x[i], partner);
    if (a.cs && !is_v && p >= 0 && p < a.rope_rows) {
      const long long at = (long long)p * (D / 2) + 4 * (low ? t : t - T / 2);
      const float4 c = *reinterpret_cast<const float4*>(a.cs + at);
      const float4 s = *reinterpret_cast<const float4*>(a.cs + a.sin_off + at);
      const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = x[i] * cc[i] + (low ? -o[i] : o[i]) * ss[i];
    }
  }
  const bool held = lives && p >= 0 && p < a.cap;
  if (h < a.H) {
    if (!held) return;
    const long long at = row * a.ldq + (long long)h * D + 4 * t;
    if (a.q_fmt) {
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.q) + at) = make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
    } else {
      *reinterpret_cast<float4*>(static_cast<float*>(a.q) + at) = make_float4(x[0], x[1], x[2], x[3]);
    }
    return;
  }
  const int g = is_v ? h - a.H - a.KH : h - a.H;
  const long long at = (row / a.L) * a.kvBatch + (long long)p * a.ldkv + (long long)g * D + 4 * t;
  void* cache = is_v ? a.v : a.k;
  if constexpr (!I4) {
    if (held)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(cache) + at) = make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
  } else {
    // offset = the least value, step = range / 15, both rounded to fp16 before the codes are taken;
    // a NaN or an infinity (x - x is then NaN) makes the group's offset NaN
    const float bad = unit8_sum(((x[0] - x[0]) + (x[1] - x[1])) + ((x[2] - x[2]) + (x[3] - x[3])));
    const float lo = unit8_min(fminf(fminf(x[0], x[1]), fminf(x[2], x[3])));
    const float hi = -unit8_min(-fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    const half_t sh = (half_t)((hi - lo) / 15.0f), oh = (half_t)(lo + bad);
    const float s = (float)sh, o = (float)oh;
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float q = s > 0.f ? fminf(fmaxf(rintf((x[i] - o) / s), 0.f), 15.f) : 0.f;
      c |= (uint32_t)(int)q << (4 * i);
    }
    if (held) {
      *reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(cache) + at / 2) = (uint16_t)c;
      if ((t & 7) == 0) (is_v ? a.vg : a.kg)[at / kGroup] = half2_t{sh, oh};
    }
  }
}

// ---- attention over the cache --------------------------------------------------------------------

struct CacheAttnArgs {
  const void* q;
  const int* pos;
  const void *k, *v;
  const half2_t *kg, *vg;
  void* o;
  long long kvBatch, rows;
  int ldq, ldo, ldkv, L, H, KH, cap, window, sinks, q_fmt;
  float scale;  // times log2(e)
};

// 8 cached values from value index `at` (a multiple of 8)
template <bool I4>
__device__ __forceinline__ half8_t cached8(const void* c, const half2_t* g, long long at) {
  if constexpr (!I4) {
    return *reinterpret_cast<const half8_t*>(static_cast<const half_t*>(c) + at);
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(c) + at / 2);
    const half2_t so = g[at / kGroup];
    half8_t r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __builtin_fmaf16((half_t)(float)((w >> (4 * i)) & 15), so[0], so[1]);
    return r;
  }
}

// One wave per (token, query head): 64 visible keys at a time, a key per lane for the scores and
// D / 64 output values per lane for the sum.
template <int D, bool I4>
__global__ __launch_bounds__(256) void cache_attn_kernel(CacheAttnArgs a) {
  constexpr int DL = (D + 63) / 64;
  __shared__ float q_s[4][D];
  __shared__ float p_s[4][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long long u = (long long)blockIdx.x * 4 + wave;
  if (u >= a.rows * a.H) return;
  const long long row = u / a.H;
  const int h = (int)(u - row * a.H), g = h / (a.H / a.KH);
  const int p = a.pos[row];
  if (p < 0 || p >= a.cap) return;
  for (int d = lane; d < D; d += 64) {
    const long long at = row * a.ldq + (long long)h * D + d;
    q_s[wave][d] = a.q_fmt ? (float)static_cast<const half_t*>(a.q)[at] : static_cast<const float*>(a.q)[at];
  }
  const int lo = a.window && p >= a.window ? p - a.window + 1 : 0;
  const int first = a.sinks < lo ? a.sinks : lo;
  const int n = first + p - lo + 1;
  const long long base = (row / a.L) * a.kvBatch + (long long)g * D;
  float m = -INFINITY, l = 0.f, o[DL];
#pragma unroll
  for (int i = 0; i < DL; ++i) o[i] = 0.f;
  for (int t0 = 0; t0 < n; t0 += 64) {
    const int cnt = n - t0 < 64 ? n - t0 : 64;
    const int t = t0 + (lane < cnt ? lane : 0);
    const int key = t < first ? t : lo + t - first;
    float s = 0.f;
    for (int d = 0; d < D; d += 8) {
      const half8_t k8 = cached8<I4>(a.k, a.kg, base + (long long)key * a.ldkv + d);
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf((float)k8[i], q_s[wave][d + i], s);
    }
    s = lane < cnt ? s * a.scale : -INFINITY;
    float mx = s;
    for (int i = 1; i < 64; i <<= 1) mx = fmaxf(mx, __shfl_xor(mx, i));
    const float mn = fmaxf(m, mx);
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float corr = exp2f(m - ref);
    const float e = exp2f(s - ref);
    l = l * corr + wave_sum(e);
    m = mn;
    __builtin_amdgcn_wave_barrier();
    p_s[wave][lane] = e;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < DL; ++i) o[i] *= corr;
    for (int c = 0; c < cnt; ++c) {
      const int tc = t0 + c;
      const long long at = base + (long long)(tc < first ? tc : lo + tc - first) * a.ldkv;
      const float e = p_s[wave][c];
#pragma unroll
      for (int i = 0; i < DL; ++i) {
        const int d = lane + 64 * i;
        if (d < D) {
          const half8_t v8 = cached8<I4>(a.v, a.vg, at + (d & ~7));
          o[i] = fmaf(e, (float)v8[d & 7], o[i]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < DL; ++i) {
    const int d = lane + 64 * i;
    if (d < D) {
      const long long at = row * a.ldo + (long long)h * D + d;
      if (a.q_fmt) static_cast<half_t*>(a.o)[at] = (half_t)(o[i] / l);
      else static_cast<float*>(a.o)[at] = o[i] / l;
    }
  }
}

// The argument checks that both entry points share.
int check_cache(const char* fn, const void* q, const int* pos, const void* k, const void* v, const void* kg, const void* vg,
                int batch, int L, int H, int KH, int D, int ldq, int cap, int ldkv, long long kvBatch, int q_fmt) {
  NS2_REQUIRE(q && pos && k && v, "%s: null q, pos, k or v", fn);
  NS2_REQUIRE(D == 64 || D == 96 || D == 128 || D == 256, "%s: head dim %d is not 64, 96, 128 or 256", fn, D);
  NS2_REQUIRE(H > 0 && KH > 0 && H % KH == 0 && (long long)H * D <= INT32_MAX, "%s: H=%d is not a positive multiple of KH=%d", fn, H,
              KH);
  NS2_REQUIRE(cap > 0 && ldq >= H * D && ldkv >= (long long)KH * D && kvBatch >= 0, "%s: bad sizes or strides", fn);
  NS2_REQUIRE(!kg == !vg, "%s: a 4-bit cache needs the groups of both k and v", fn);
  NS2_REQUIRE(q_fmt == 0 || q_fmt == 1, "%s: q_fmt %d is not 0 (fp32) or 1 (fp16)", fn, q_fmt);
  NS2_REQUIRE(aligned(q, 16) && ldq % (q_fmt ? 8 : 4) == 0 && aligned(pos, 4), "%s: the rows of q must be 16-byte aligned", fn);
  const int unit = kg ? kGroup : 8;
  NS2_REQUIRE(aligned(k, 16) && aligned(v, 16) && aligned(kg, 4) && aligned(vg, 4) && ldkv % unit == 0 && kvBatch % unit == 0,
              "%s: cache rows must be 16-byte aligned (ldkv, kvBatch multiples of %d)", fn, unit);
  return NS2_OK;
}

}  // namespace

#define NS2_CACHE_D(D, LAUNCH)            \
  switch (D) {                            \
    case 64: LAUNCH(64) break;            \
    case 96: LAUNCH(96) break;            \
    case 128: LAUNCH(128) break;          \
    default: LAUNCH(256) break;           \
  }

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
  if (cs)
    NS2_REQUIRE(aligned(cs, 16) && sin_off % 4 == 0 && rope_rows >= 0 && sin_off >= 0, "%s: the rotation table must be 16-byte aligned",
                fn);
  NS2_REQUIRE(batch == 1 || kvBatch >= (cap - 1LL) * ldkv + KH * D, "%s: the sequences' caches overlap (kvBatch)", fn);
  WriteArgs a{X, pos, w_q, w_k, cs, q, k, v, reinterpret_cast<half2_t*>(k_groups), reinterpret_cast<half2_t*>(v_groups), sin_off,
              kvBatch, (long long)batch * L, ldx, ldq, ldkv, L, H, KH, cap, rope_rows, q_fmt, eps};
  const long long units = a.rows * (H + 2 * KH);
  const int per = 4 * (256 / D);  // heads of a block: 256 / D in each of its four waves
  NS2_REQUIRE((units + per - 1) / per <= INT32_MAX, "%s: %lld heads are too many for one launch", fn, units);
  const unsigned grid = (unsigned)((units + per - 1) / per);
  hipStream_t s = ns2::stream();
  ns2::ProfScope prof_("head_norm_cache");
#define NS2_WRITE(D_)                                                        \
  if (k_groups) cache_write_kernel<D_, true><<<grid, 256, 0, s>>>(a);        \
  else cache_write_kernel<D_, false><<<grid, 256, 0, s>>>(a);
  NS2_CACHE_D(D, NS2_WRITE)
#undef NS2_WRITE
  NS2_LAUNCHED("head_norm_cache");
  return NS2_OK;
}

size_t ns2_attention_cache_bytes(int batch, int L, int H, int KH, int D, int cap, int window, int sinks) { return 0; }

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
  const size_t need = ns2_attention_cache_bytes(batch, L, H, KH, D, cap, window, sinks);
  NS2_REQUIRE(work_bytes >= need && (!need || (work && aligned(work, 16))),
              "%s: the call needs %zu bytes of 16-byte aligned work memory (ns2_attention_cache_bytes), got %zu", fn, need, work_bytes);
  CacheAttnArgs a{q, pos, k, v, reinterpret_cast<const half2_t*>(k_groups), reinterpret_cast<const half2_t*>(v_groups), o, kvBatch,
                  (long long)batch * L, ldq, ldo, ldkv, L, H, KH, cap, window, sinks, q_fmt, scale * kLog2e};
  const long long units = a.rows * H;
  NS2_REQUIRE((units + 3) / 4 <= INT32_MAX, "%s: %lld query heads are too many for one launch", fn, units);
  const unsigned grid = (unsigned)((units + 3) / 4);
  hipStream_t s = ns2::stream();
  ns2::ProfScope prof_("attention_cache");
#define NS2_ATTN(D_)                                                        \
  if (k_groups) cache_attn_kernel<D_, true><<<grid, 256, 0, s>>>(a);        \
  else cache_attn_kernel<D_, false><<<grid, 256, 0, s>>>(a);
  NS2_CACHE_D(D, NS2_ATTN)
#undef NS2_ATTN
  NS2_LAUNCHED("attention_cache");
  return NS2_OK;
}

}  // extern "C"
