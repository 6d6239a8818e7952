// Linears on 4-bit weights with group scales, and the quantizer that makes such weights from bf16.
//
// W[n][k] = scale[n][k / G] * (code[n][k] - 8), codes 0..15 two to a byte (the even column in the
// low four bits), one fp16 scale per G = 32, 64 or 128 columns of a row.
#include "ns2_common.h"

using namespace ns2dev;

namespace {

struct I4Args {
  const void* A;  // fp32 or fp16 [M][lda]
  const uint8_t* W;
  const half_t* scale;
  const float* bias;
  const float* add;
  float* C;
  const float* gate;
  long long cOff, gOff;
  int lda, ldc, M, N, K, group;
  float alpha;
  int act, resid;
};

// Epilogue of one output element, as every linear's (gemm.js:159-164).
__device__ __forceinline__ void store_i4(const I4Args& p, int m, int n, float acc, float bi, float gt) {
  float r = acc * p.alpha + bi;
  if (p.add) r += p.add[(long long)m * p.N + n];
  r = apply_act(r, p.act);
  float* c = p.C + p.cOff + (long long)m * p.ldc + n;
  if (!p.resid) *c = r;
  else if (!p.gate) *c = *c + r;
  else *c = *c + gt * r;
}

// One wave per output column, 32 columns of k (16 bytes of codes, inside one group) per lane and
// step, four rows of A per pass over the weights.
template <bool A16>
__global__ __launch_bounds__(256) void linear_i4_kernel(I4Args p) {
  const int lane = threadIdx.x & 63;
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= p.N) return;
  const uint8_t* wr = p.W + (long long)n * (p.K / 2);
  const half_t* sr = p.scale + (long long)n * (p.K / p.group);
  const float bi = p.bias ? p.bias[n] : 0.f;
  const float gt = p.gate ? p.gate[p.gOff + n] : 1.f;
  for (int m0 = 0; m0 < p.M; m0 += 4) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k = lane * 32; k < p.K; k += 2048) {
      const uint4 w4 = *reinterpret_cast<const uint4*>(wr + k / 2);
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
      const float s = (float)sr[k / p.group];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = m0 + i < p.M ? m0 + i : p.M - 1;
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const long long at = (long long)m * p.lda + k + 8 * j + e;
            const float x = A16 ? (float)static_cast<const half_t*>(p.A)[at] : static_cast<const float*>(p.A)[at];
            t = fmaf(x, (float)((int)((w[j] >> (4 * e)) & 15) - 8), t);
          }
        acc[i] = fmaf(t, s, acc[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float sum = wave_sum(acc[i]);
      if (lane == 0 && m0 + i < p.M) store_i4(p, m0 + i, n, sum, bi, gt);
    }
  }
}

// One thread per group: the group's largest magnitude a goes to code 1 or 15 with step
// s = half(a / 7), code = 8 + clamp(rint(w / s), -7, 7); a group of zeros (or whose step rounds to
// 0) is all code 8. Division and rounding are exact, so the codes are a function of the weight.
// A group that holds a NaN or an infinity gets a NaN scale.
__global__ __launch_bounds__(256) void quantize_i4_kernel(const uint16_t* __restrict__ W, uint8_t* __restrict__ codes,
                                                           half_t* __restrict__ scale, long long groups, int G) {
  const long long g = (long long)blockIdx.x * 256 + threadIdx.x;
  if (g >= groups) return;
  const uint16_t* w = W + g * G;
  float a = 0.f, bad = 0.f;
  for (int i = 0; i < G; ++i) {
    const float x = __builtin_bit_cast(float, (uint32_t)w[i] << 16);
    a = fmaxf(a, fabsf(x));
    bad += x - x;
  }
  const half_t sh = (half_t)(a / 7.0f + bad);
  const float s = (float)sh;
  scale[g] = sh;
  for (int i = 0; i < G; i += 2) {
    uint32_t b = 0;
    for (int e = 0; e < 2; ++e) {
      const float x = __builtin_bit_cast(float, (uint32_t)w[i + e] << 16);
      const float q = s > 0.f ? fminf(fmaxf(rintf(x / s), -7.f), 7.f) : 0.f;
      b |= (uint32_t)((int)q + 8) << (4 * e);
    }
    codes[(g * G + i) / 2] = (uint8_t)b;
  }
}

inline bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace

extern "C" {

int ns2_quantize_i4(const uint16_t* W, uint8_t* codes, uint16_t* scale, int N, int K, int group) {
  NS2_READY();
  if (N == 0) return NS2_OK;
  NS2_REQUIRE(W && codes && scale, "ns2_quantize_i4: null W, codes or scale");
  NS2_REQUIRE(group == 32 || group == 64 || group == 128, "ns2_quantize_i4: group %d is not 32, 64 or 128", group);
  NS2_REQUIRE(N > 0 && K > 0 && K % group == 0, "ns2_quantize_i4: N=%d, K=%d must be positive, K a multiple of the group %d", N, K,
              group);
  const long long groups = (long long)N * (K / group);
  NS2_REQUIRE((groups + 255) / 256 <= INT32_MAX, "ns2_quantize_i4: %lld groups are too many for one launch", groups);
  ns2::ProfScope prof_("quantize_i4");
  quantize_i4_kernel<<<(unsigned)((groups + 255) / 256), 256, 0, ns2::stream()>>>(W, codes, reinterpret_cast<half_t*>(scale),
                                                                                 groups, group);
  NS2_LAUNCHED("quantize_i4");
  return NS2_OK;
}

int ns2_linear_i4(const void* A, int a_fmt, int lda, const uint8_t* W, const uint16_t* scale, const float* bias,
                  const float* add, float* C, int M, int N, int K, int group, int ldc, long long cOff, float alpha, int act,
                  int resid, const float* gate, long long gOff) {
  NS2_READY();
  if (M == 0) return NS2_OK;
  const char* fn = "ns2_linear_i4";
  NS2_REQUIRE(A && W && scale && C, "%s: null A, W, scale or C", fn);
  NS2_REQUIRE(a_fmt == 0 || a_fmt == 1, "%s: a_fmt %d is not 0 (fp32) or 1 (fp16)", fn, a_fmt);
  NS2_REQUIRE(group == 32 || group == 64 || group == 128, "%s: group %d is not 32, 64 or 128", fn, group);
  NS2_REQUIRE(M > 0 && N > 0 && K > 0 && K % group == 0, "%s: M=%d, N=%d, K=%d must be positive, K a multiple of the group %d", fn,
              M, N, K, group);
  NS2_REQUIRE(lda >= K && ldc >= N && cOff >= 0 && gOff >= 0, "%s: lda=%d, ldc=%d must cover K and N, offsets be non-negative", fn,
              lda, ldc);
  NS2_REQUIRE(act >= NS2_ACT_NONE && act <= NS2_ACT_GELU_TANH, "%s: unknown activation %d", fn, act);
  NS2_REQUIRE(aligned(A, 16) && lda % (a_fmt ? 8 : 4) == 0 && aligned(W, 16) && aligned(scale, 2),
              "%s: the rows of A and W must be 16-byte aligned (lda a multiple of %d)", fn, a_fmt ? 8 : 4);
  I4Args p{A,  W,   reinterpret_cast<const half_t*>(scale), bias, add, C, gate, cOff, gOff, lda, ldc, M, N, K, group, alpha,
           act, resid};
  ns2::ProfScope prof_("linear_i4");
  const unsigned grid = (unsigned)((N + 3LL) / 4);
  if (a_fmt) linear_i4_kernel<true><<<grid, 256, 0, ns2::stream()>>>(p);
  else linear_i4_kernel<false><<<grid, 256, 0, ns2::stream()>>>(p);
  NS2_LAUNCHED("linear_i4");
  return NS2_OK;
}

}  // extern "C"
