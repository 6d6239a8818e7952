// Linears on 4-bit weights with group scales, and the quantizer that makes such weights from bf16.
//
// W[n][k] = scale[n][k / G] * (code[n][k] - 8), codes 0..15 two to a byte (the even column in the
// low four bits), one fp16 scale per G = 32, 64 or 128 columns of a row.
#include <algorithm>

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
  int slab;  // columns of k whose rows of x are in LDS at a time
};

// The power of two that takes a row's largest finite magnitude to below 2^14.
__device__ __forceinline__ int i4_up(float top) {
  const int up = 14 - __builtin_amdgcn_frexp_expf(top);
  return top > 0.f ? (up < 120 ? up : 120) : 0;
}

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

// ---- the product --------------------------------------------------------------------------------
//
// v_mfma_f32_16x16x32_f16 with A = 16 rows of x, B = 16 columns of W^T as the exact halves code - 8, so that a
// product over one group needs its scale only once, in fp32, after the sum. An fp32 row of x is scaled by a
// power of two to below 2^14 and split into two halves that keep 22 of its bits (two products); fp16 rows go in
// as they are. The weights bound it where rows are few: 16 weight rows are read 64 bytes of each at a time (16
// per lane, 128 columns of k, a "chunk"), and since the four lanes of a row then hold one 32-column step each
// where the product wants a quarter of each step, the words change lanes (4 x 4, four row swaps). Within a
// word, codes come out in the order 0 4 1 5 2 6 3 7; x is stored in that order.
//
// A row of A and the same row of D are apart: row 4 a + b of A is x row a + 4 b, whose results are then register
// b of lane group a, so that up to 4 (8) rows take only one (two) of the four result registers through the
// scales.

// Four registers of the four 16-lane rows transposed: register j of row g becomes register g of row j.
__device__ __forceinline__ void transpose_rows(uint32_t w[4]) {
  permlane32_swap(w[0], w[2]);
  permlane32_swap(w[1], w[3]);
  permlane16_swap(w[0], w[1]);
  permlane16_swap(w[2], w[3]);
}

// code - 8 of a word's eight codes
__device__ __forceinline__ half8_t codes8(uint32_t w) {
  uint32_t r[4];
  nibbles4(w, half2_t{-1032.f, -1032.f}, half2_t{-72.f, -72.f}, r);
  return __builtin_bit_cast(half8_t, make_uint4(r[0], r[1], r[2], r[3]));
}

constexpr int kChunk = 128;  // columns of k per load
// Waves of a block, and its LDS for the rows of x.
template <int WK>
constexpr int waves() {
  return WK == 16 ? 16 : 4;
}
// (one block to a CU where sixteen waves run, else three); pieces of 8 columns of fp32 rows that a thread holds.
template <int WK>
constexpr int slab_bytes() {
  return WK == 16 ? 60 * 1024 : 52 * 1024;
}
template <int WK>
constexpr int pieces() {
  return WK == 16 ? 2 : 6;
}
// Places of a piece of 8 columns in LDS: an odd number, since threads that write pieces of one row would meet in the
// same banks otherwise (16 x 4096 x 1536 fp32 8.7 us, so 7.3).
__host__ __device__ constexpr int places(int rows) { return rows | 1; }

// A block takes 16 RT rows and, with WK = 1, 64 CT columns (16 CT per wave) over all of K; with WK = 4 or 16, 16 CT
// columns whose chunks its WK waves take in turn and add up at the end. NR: result registers in use (4 NR rows of
// each 16).
// SG: 32-column steps per group. The block's rows of x go to LDS a slab of p.slab columns at a time: operand
// (step, lane group, row), places(rows) apart, hi then lo.
template <bool A16, int SG, int RT, int NR, int CT, int WK>
__global__ __launch_bounds__((64 * waves<WK>())) void linear_i4_kernel(I4Args p) {
  constexpr int kWaves = waves<WK>();
  extern __shared__ __attribute__((aligned(16))) char smem[];
  half8_t* x_s = reinterpret_cast<half8_t*>(smem);
  __shared__ uint32_t top_s[16 * RT];
  __shared__ int infinite_s;  // a row of the slab holds an infinity
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c16 = lane & 15, g = lane >> 4;
  const int m0 = blockIdx.y * (16 * RT);
  const int rows = p.M - m0 < 16 * RT ? p.M - m0 : 16 * RT;
  const int n0 = (WK == 1 ? blockIdx.x * kWaves + wave : blockIdx.x) * (16 * CT);
  const int kb = p.K / 2, kg = p.K / (32 * SG);

  const uint8_t* wr[CT];
  const half_t* sr[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int n = n0 + 16 * c + c16 < p.N ? n0 + 16 * c + c16 : p.N - 1;
    wr[c] = p.W + (long long)n * kb;
    sr[c] = p.scale + (long long)n * kg;
  }
  // the wave's next PD chunks are on their way
  constexpr int PD = CT == 1 ? 4 : 2;
  uint4 w[PD][CT];
  half_t sc[PD][CT];
  auto load = [&](int s, int chunk) {
    int k = chunk * kChunk + 32 * g;
    k = k < p.K ? k : 0;  // (a step past K meets zeros of x)
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      w[s][c] = *reinterpret_cast<const uint4*>(wr[c] + k / 2);
      sc[s][c] = sr[c][k / (32 * SG)];
    }
  };

  float tot[RT][CT][NR] = {};
  int arow[RT];  // this lane's rows of the A operand
#pragma unroll
  for (int i = 0; i < RT; ++i) arow[i] = min(16 * i + (c16 >> 2) + 4 * (c16 & 3), rows - 1);

  for (int k0 = 0; k0 < p.K; k0 += p.slab) {
    const int ks = p.K - k0 < p.slab ? p.K - k0 : p.slab;
    const int n8 = (ks + kChunk - 1) / kChunk * (kChunk / 8), items = rows * n8, pad = places(rows);  // (zeros behind K, to the end of its chunk)
    half8_t* lo_s = x_s + pad * n8;
    const int first = k0 / kChunk + (WK == 1 ? 0 : wave), last = (k0 + ks + kChunk - 1) / kChunk;
#pragma unroll
    for (int s = 0; s < PD; ++s)
      if (first + s * WK < last) load(s, first + s * WK);
    if (k0) __syncthreads();  // the last slab is used
    if constexpr (A16) {
      for (int u = threadIdx.x; u < items; u += 64 * kWaves) {
        const int r = u / n8, k8 = u - r * n8;
        half8_t v = {0, 0, 0, 0, 0, 0, 0, 0};
        if (8 * k8 < ks) v = *reinterpret_cast<const half8_t*>(static_cast<const half_t*>(p.A) + (long long)(m0 + r) * p.lda + k0 + 8 * k8);
        x_s[k8 * pad + r] = half8_t{v[0], v[4], v[1], v[5], v[2], v[6], v[3], v[7]};
      }
    } else {
      constexpr int NI = pieces<WK>();
      float4 x[NI][2];
      for (int u = threadIdx.x; u < rows; u += 64 * kWaves) top_s[u] = 0u;
      if (threadIdx.x == 0) infinite_s = 0;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int u = threadIdx.x + 64 * kWaves * i, r = u / n8, k8 = u - r * n8;
        x[i][0] = x[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (u < items && 8 * k8 < ks) {
          const float* a = static_cast<const float*>(p.A) + (long long)(m0 + r) * p.lda + k0 + 8 * k8;
          x[i][0] = *reinterpret_cast<const float4*>(a);
          x[i][1] = *reinterpret_cast<const float4*>(a + 4);
        }
      }
      __syncthreads();
      // magnitudes order as their bits do; four neighbours share a row (n8 is a multiple of 4)
      bool infinite = false;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int u = threadIdx.x + 64 * kWaves * i;
        const float4 a = x[i][0], b = x[i][1];
        float top = fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))),
                          fmaxf(fmaxf(fabsf(b.x), fabsf(b.y)), fmaxf(fabsf(b.z), fabsf(b.w))));
        infinite |= top == INFINITY;
        top = fmaxf(top, dpp<kDppXor1>(top));
        top = fmaxf(top, dpp<kDppXor2>(top));
        if (u < items && (threadIdx.x & 3) == 0) atomicMax(&top_s[u / n8], __builtin_bit_cast(uint32_t, top));
      }
      if (infinite) infinite_s = 1;
      __syncthreads();
      infinite = __builtin_amdgcn_readfirstlane(infinite_s) != 0;
      if (infinite) {  // what is finite decides the scaling
        for (int u = threadIdx.x; u < rows; u += 64 * kWaves) top_s[u] = 0u;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int u = threadIdx.x + 64 * kWaves * i;
          const float4 a = x[i][0], b = x[i][1];
          const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
          float top = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.f);
          if (u < items) atomicMax(&top_s[u / n8], __builtin_bit_cast(uint32_t, top));
        }
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int u = threadIdx.x + 64 * kWaves * i, r = u / n8, k8 = u - r * n8;
        if (u < items) {
          const float4 a = x[i][0], b = x[i][1];
          const float v[8] = {a.x, b.x, a.y, b.y, a.z, b.z, a.w, b.w};
          const int up = i4_up(__builtin_bit_cast(float, top_s[r]));
          half8_t hi, lo;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float t = ldexpf(v[e], up);
            hi[e] = (half_t)t;
            lo[e] = (half_t)(t - (float)hi[e]);
          }
          if (infinite) {  // an infinity is all in hi
#pragma unroll
            for (int e = 0; e < 8; ++e) lo[e] = fabsf(v[e]) == INFINITY ? (half_t)0.f : lo[e];
          }
          x_s[k8 * pad + r] = hi;
          lo_s[k8 * pad + r] = lo;
        }
      }
    }
    __syncthreads();

    float acc[RT][CT][NR] = {};
    for (int chunk = first; chunk < last; chunk += PD * WK) {
#pragma unroll
      for (int sl = 0; sl < PD; ++sl) {
        const int ch = chunk + sl * WK;
        if (ch < last) {  // uniform
          uint32_t t[CT][4];
          float s[CT][4];
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            t[c][0] = w[sl][c].x;
            t[c][1] = w[sl][c].y;
            t[c][2] = w[sl][c].z;
            t[c][3] = w[sl][c].w;
            const float f = ch * kChunk + 32 * g < p.K ? (float)sc[sl][c] : 0.f;
            uint32_t a = __builtin_bit_cast(uint32_t, f), b = a;
            permlane32_swap(a, b);  // the scales of steps 0, 1 | 2, 3
            uint32_t a1 = a, b1 = b;
            permlane16_swap(a, a1);
            permlane16_swap(b, b1);
            s[c][0] = __builtin_bit_cast(float, a);
            s[c][1] = __builtin_bit_cast(float, a1);
            s[c][2] = __builtin_bit_cast(float, b);
            s[c][3] = __builtin_bit_cast(float, b1);
          }
#pragma unroll
          for (int c = 0; c < CT; ++c) transpose_rows(t[c]);
          if (ch + PD * WK < last) load(sl, ch + PD * WK);
          const int base = (ch * kChunk - k0) / 8 + g;
          float4_t d[RT][CT];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            half8_t xh[RT], xl[RT];
#pragma unroll
            for (int i = 0; i < RT; ++i) {
              xh[i] = x_s[(base + 4 * j) * pad + arow[i]];
              if constexpr (!A16) xl[i] = lo_s[(base + 4 * j) * pad + arow[i]];
            }
#pragma unroll
            for (int c = 0; c < CT; ++c) {
              const half8_t q = codes8(t[c][j]);
#pragma unroll
              for (int i = 0; i < RT; ++i) {
                if (j % SG == 0) d[i][c] = float4_t{0.f, 0.f, 0.f, 0.f};
                d[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh[i], q, d[i][c], 0, 0, 0);
                if constexpr (!A16) d[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xl[i], q, d[i][c], 0, 0, 0);
                if (j % SG == SG - 1) {
#pragma unroll
                  for (int r = 0; r < NR; ++r) acc[i][c][r] = fmaf(s[c][j], d[i][c][r], acc[i][c][r]);
                }
              }
            }
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        float back = 1.f;
        if constexpr (!A16) back = ldexpf(1.f, -i4_up(__builtin_bit_cast(float, top_s[min(16 * i + g + 4 * r, rows - 1)])));
#pragma unroll
        for (int c = 0; c < CT; ++c) tot[i][c][r] = fmaf(acc[i][c][r], back, tot[i][c][r]);
      }
  }

  if constexpr (WK > 1) {
    float* red = reinterpret_cast<float*>(smem);  // [wave][c][r][lane]
    constexpr int T = CT * NR;
    static_assert(RT == 1, "K is split for few rows only");
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int r = 0; r < NR; ++r) red[(wave * T + c * NR + r) * 64 + lane] = tot[0][c][r];
    __syncthreads();
    for (int u = wave; u < T; u += kWaves) {
      float sum = 0.f;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) sum += red[(v * T + u) * 64 + lane];
      const int m = m0 + g + 4 * (u % NR), n = n0 + 16 * (u / NR) + c16;
      if (m < m0 + rows && n < p.N) store_i4(p, m, n, sum, p.bias ? p.bias[n] : 0.f, p.gate ? p.gate[p.gOff + n] : 1.f);
    }
  } else {
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int n = n0 + 16 * c + c16;
      if (n < p.N) {
        const float bi = p.bias ? p.bias[n] : 0.f, gt = p.gate ? p.gate[p.gOff + n] : 1.f;
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            const int m = m0 + 16 * i + g + 4 * r;
            if (m < m0 + rows) store_i4(p, m, n, tot[i][c][r], bi, gt);
          }
      }
    }
  }
}

template <bool A16, int SG, int RT, int NR, int CT, int WK>
void launch_rows(I4Args p, hipStream_t s) {
  const int rows = p.M < 16 * RT ? p.M : 16 * RT, size = A16 ? 2 : 4;  // (of a value of x)
  const int room = slab_bytes<WK>() / (places(rows) * size), held = A16 ? room : pieces<WK>() * waves<WK>() * 512 / rows;
  const int most = std::min(room, held) / kChunk, chunks = (p.K + kChunk - 1) / kChunk;
  // slabs of about the same number of chunks, if possible as many for each wave
  const int slabs = (chunks + most - 1) / most, each = (chunks + slabs - 1) / slabs, even = (each + WK - 1) / WK * WK;
  p.slab = (even <= most && even < chunks ? even : each) * kChunk;
  constexpr int kWaves = waves<WK>();
  const size_t red = WK > 1 ? sizeof(float) * kWaves * CT * NR * 64 : 0;
  const size_t lds = std::max<size_t>((size_t)p.slab * places(rows) * size, red);
  const int cols = 16 * CT * (WK == 1 ? kWaves : 1);
  const dim3 grid((unsigned)((p.N + cols - 1LL) / cols), (unsigned)((p.M + 16 * RT - 1) / (16 * RT)));
  linear_i4_kernel<A16, SG, RT, NR, CT, WK><<<grid, 64 * kWaves, lds, s>>>(p);
}
template <bool A16, int SG, int CT, int WK>
void launch_i4(const I4Args& p, hipStream_t s) {
  if (p.M <= 4) launch_rows<A16, SG, 1, 1, CT, WK>(p, s);
  else if (p.M <= 8) launch_rows<A16, SG, 1, 2, CT, WK>(p, s);
  else launch_rows<A16, SG, 1, 4, CT, WK>(p, s);
}

// By the number of 16 x 16 tiles of the output (us, "a | b": fp16 | fp32 x):
//  - many tiles: all of K in a wave of 32 columns, loads two chunks ahead (256 x 4096 x 640 9.9 | 11.3, over four
//    waves 10.9 | 18.3; 12 x 32768 x 2048 16.7 | 18.9, 18.4 | 24.5); with up to four fp16 rows, whose products cost
//    least, 16 columns and loads four chunks ahead (1 x 262144 x 640 18.2, with 32 columns 19.9); with many fp16 rows
//    32 of them per block, unless that leaves an eighth of the blocks' rows empty (32 x 65536 x 2048 34.5, with 16
//    50; 300 x 27000 x 1536 82, 102; 48 x 65600 x 640 26.9, 24.4. fp32 rows take the same either way, 128 and 131);
//  - few tiles and a K that gives sixteen waves work: over sixteen waves (1 x 8192 x 1536 4.1 | 4.8, over four 4.6 |
//    4.9; 16 x 8192 x 1536 5.3 | 8.2, 7.3 | 10.0), of 16 columns up to one block per CU or where rows cost least
//    (16 x 4096 x 1536 fp32 7.4, with 32 columns 7.9), else of 32 (16 x 8192 x 1536 fp32 8.2, with 16 12.6);
//  - between: over four waves of 32 columns (8 x 16384 x 4096 fp32 21.4, with 16 columns 28.6; in one wave 27.8).
// The bytes bound a table (1 x 262144 x 640: 90 MB at 5.0 TB/s); the smallest calls are a launch and two round trips
// to memory; many rows are bound by the VALU, which decodes the weights again for every block of rows (300 x 27000 x
// 1536: 300 TFLOP/s, fp32 190).
template <bool A16, int SG>
void choose_i4(const I4Args& p, hipStream_t s) {
  const long long high = (p.M + 15LL) / 16, tiles = (p.N + 15) / 16 * high;
  const bool light = A16 && p.M <= 4, deep = p.K > 4 * kChunk;
  if (tiles >= (A16 ? 1792 : 1536)) {
    if constexpr (A16) {
      if (light) return launch_rows<A16, SG, 1, 1, 1, 1>(p, s);
      if (high > 1 && tiles >= 8192 && 8 * high >= 14 * ((high + 1) / 2)) return launch_rows<A16, SG, 2, 4, 2, 1>(p, s);
    }
    launch_i4<A16, SG, 2, 1>(p, s);
  } else if (deep && tiles <= (light ? 512 : 256)) launch_i4<A16, SG, 1, 16>(p, s);
  else if (deep && tiles <= 512) launch_i4<A16, SG, 2, 16>(p, s);
  else launch_i4<A16, SG, 2, 4>(p, s);
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
  NS2_REQUIRE(groups <= UINT32_MAX - 255LL, "ns2_quantize_i4: %lld groups are too many for one launch", groups);
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
  NS2_REQUIRE(M <= 16LL * 65535 && N <= 1 << 29 && K <= 1 << 30, "%s: M=%d, N=%d, K=%d are too many for one launch", fn, M, N, K);
  I4Args p{A,  W,   reinterpret_cast<const half_t*>(scale), bias, add, C, gate, cOff, gOff, lda, ldc, M, N, K, group, alpha,
           act, resid};
  ns2::ProfScope prof_("linear_i4");
  hipStream_t s = ns2::stream();
  if (group == 32) a_fmt ? choose_i4<true, 1>(p, s) : choose_i4<false, 1>(p, s);
  else if (group == 64) a_fmt ? choose_i4<true, 2>(p, s) : choose_i4<false, 2>(p, s);
  else a_fmt ? choose_i4<true, 4>(p, s) : choose_i4<false, 4>(p, s);
  NS2_LAUNCHED("linear_i4");
  return NS2_OK;
}

}  // extern "C"
