// Products of few rows with 4-bit weights, and the quantiser that makes them.
//
// out[m][n] = sum over groups of scale[group][n] * sum_k (code[n][k] - 8) x[m][k]. Bound: memory, half a byte for every weight; at that
// rate an SM gets 46 weights a clock, too many for multiply-adds of every row (128 lanes a clock), so the products are m16n8k16 matrix
// instructions with 16 outputs as rows and 8 tokens as columns, on codes turned into 16-bit floats in registers. Order of k within a
// tile is free as long as both operands agree: a lane takes 16 consecutive inputs (k steps of 4), so it loads 16 bytes of weights
// (8 of outputs r and of r + 8) and 16 inputs in a row.
//  - Weights are exact: a field of 4 bits or-ed into the mantissa of a power of two, less what that adds. (Sums that start at -136 sum x
//    in place of the subtraction are off by a part of the inputs' size even where the weights are zero.)
//  - BF16 inputs are exact operands. A product with zeros, once for all the outputs of a pass, makes the sums of a row with a NaN or an infinity
//    start at NaN.
//  - FP32 inputs are pairs of FP16 numbers, scaled by a power of two for every 64 inputs of a row, the rests' products first, then the
//    others' into the same accumulator: FP32 grade.
// A group's sums are FP32, times the scale once per 64 inputs.
// A CTA has a range of the tiles of 16 outputs and goes over it in passes of up to R tiles, so that 64 inputs once loaded serve R tiles. Its
// warps take every WARPS-th tile of 64 inputs and are added up in shared memory, in order.
// Measured: 28672 x 8192, BF16, 8 rows 42 us (3.0 TB/s), 16 rows 53 us, FP32 54 and 75 us, 19 us by bytes: two warps a scheduler, whose
// chains of shifts, masks, subtractions and matrix instructions leave half of the cycles free. The subtraction is 4 and 5 us of the BF16 times; multiply-adds
// that also save the shifts (fields in bits 4-7 taken as numbers below 2^-125) were slower, 59 us at 16 rows. 2304 x 768, one row: 2.2 us, a launch.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "device_util.cuh"
#include "serving.h"

namespace pg {
namespace {

template <bool PAIR>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
  if (PAIR)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Weights code - 8 of inputs 2 i and 2 i + 1 of a word of 8 codes as 16-bit floats: BF16 128 + code less 136, FP16 1024 + code (or 64 + code,
// from the field one place further up) less the rest, all exact.
template <bool PAIR>
__device__ __forceinline__ uint32_t weights2(uint32_t word, int i) {
  if (PAIR) {
    const uint32_t u = ((i < 2 ? word : word >> 8) & (i & 1 ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;
    const __half2 h = *reinterpret_cast<const __half2*>(&u);
    const __half2 w = i & 1 ? __hfma2(h, __float2half2_rn(0.0625f), __float2half2_rn(-72.f)) : __hsub2(h, __float2half2_rn(1032.f));
    return *reinterpret_cast<const uint32_t*>(&w);
  }
  const uint32_t u = ((word >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
  const __nv_bfloat162 w = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), __float2bfloat162_rn(136.f));
  return *reinterpret_cast<const uint32_t*>(&w);
}

// 16 inputs of one row: as they come, and as operand words (word 2 s + e: inputs 4 s + 2 e and 4 s + 2 e + 1).
template <typename T>
struct Raw {
  uint4 v[sizeof(T)];
  __device__ __forceinline__ void load(const T* p, int live, bool wide) {
    constexpr int N = 16 / sizeof(T);
    if (live <= 0 || (wide && live >= 16)) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); ++i) v[i] = live > 0 ? *reinterpret_cast<const uint4*>(p + i * N) : make_uint4(0, 0, 0, 0);
    } else {
      union {
        uint4 u[sizeof(T)];
        T t[16];
      } x;
#pragma unroll
      for (int i = 0; i < 16; ++i) x.t[i] = i < live ? p[i] : from_f32<T>(0.f);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); ++i) v[i] = x.u[i];
    }
  }
};
template <typename T>
struct Operand;
template <>
struct Operand<__nv_bfloat16> {
  uint32_t w[1][8];
  __device__ __forceinline__ float make(const Raw<__nv_bfloat16>& r) {
    w[0][0] = r.v[0].x; w[0][1] = r.v[0].y; w[0][2] = r.v[0].z; w[0][3] = r.v[0].w;
    w[0][4] = r.v[1].x; w[0][5] = r.v[1].y; w[0][6] = r.v[1].z; w[0][7] = r.v[1].w;
    return 1.f;
  }
};
template <>
struct Operand<float> {
  uint32_t w[2][8];
  // What the row's sums of these 64 inputs are to be multiplied with.
  __device__ __forceinline__ float make(const Raw<float>& r) {
    float v[16], m = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[4 * i] = __uint_as_float(r.v[i].x); v[4 * i + 1] = __uint_as_float(r.v[i].y);
      v[4 * i + 2] = __uint_as_float(r.v[i].z); v[4 * i + 3] = __uint_as_float(r.v[i].w);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(v[i]));
    m = fmaxf(m, __shfl_xor_sync(ALL_LANES, m, 1));
    m = fmaxf(m, __shfl_xor_sync(ALL_LANES, m, 2));
    // exponents within +-126 keep both the factor and its inverse normal numbers, and the largest input, 2^128, below 4
    const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -126), 126);
    const float s = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = v[2 * i] * s, b = v[2 * i + 1] * s;
      const __half2 h = __floats2half2_rn(a, b);
      const float2 q = __half22float2(h);
      const __half2 l = __floats2half2_rn(a - q.x, b - q.y);
      w[0][i] = *reinterpret_cast<const uint32_t*>(&h);
      w[1][i] = *reinterpret_cast<const uint32_t*>(&l);
    }
    return __uint_as_float((uint32_t)(127 + e) << 23);
  }
};

// 64 inputs of NT groups of 8 tokens as the column operand, and what the accumulators start from.
template <typename T, int NT>
struct Tokens {
  static constexpr bool PAIR = std::is_same<T, float>::value;
  static constexpr int PARTS = PAIR ? 2 : 1;
  Operand<T> x[NT];
  float base[NT][4], back[NT][2];
  __device__ __forceinline__ Tokens(const Raw<T> (&raw)[NT], int c) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float b = x[t].make(raw[t]);
      if (PAIR) {  // columns 2 c and 2 c + 1 are the tokens of lanes 8 c and 8 c + 4
        back[t][0] = __shfl_sync(ALL_LANES, b, c * 8);
        back[t][1] = __shfl_sync(ALL_LANES, b, c * 8 + 4);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) base[t][e] = 0.f;
      if constexpr (!PAIR) {
        const uint32_t f[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int s = 0; s < 4; ++s) mma16<PAIR>(base[t], f, x[t].w[0][2 * s], x[t].w[0][2 * s + 1], base[t]);
      }
    }
  }
  // 16 outputs: this lane's codes, the scales of outputs g and g + 8.
  __device__ __forceinline__ void add(const uint4& w, uint16_t scale_a, uint16_t scale_b, float (&acc)[NT][4]) const {
    // inputs 4 s .. 4 s + 3 of outputs g (words x, y) and g + 8 (z, w)
    uint32_t f[4][4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const uint32_t wa = s < 2 ? w.x : w.y, wb = s < 2 ? w.z : w.w;
      const int i = (s & 1) * 2;
      f[s][0] = weights2<PAIR>(wa, i);
      f[s][1] = weights2<PAIR>(wb, i);
      f[s][2] = weights2<PAIR>(wa, i + 1);
      f[s][3] = weights2<PAIR>(wb, i + 1);
    }
    float d[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int p = PARTS - 1; p >= 0; --p)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          if (p == PARTS - 1 && s == 0) mma16<PAIR>(d[t], f[s], x[t].w[p][2 * s], x[t].w[p][2 * s + 1], base[t]);
          else mma16<PAIR>(d[t], f[s], x[t].w[p][2 * s], x[t].w[p][2 * s + 1], d[t]);
        }
    const float sa = __uint_as_float((uint32_t)scale_a << 16), sb = __uint_as_float((uint32_t)scale_b << 16);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(PAIR ? d[t][e] * back[t][e & 1] : d[t][e], e < 2 ? sa : sb, acc[t][e]);
  }
};

// NT: groups of 8 tokens. R: tiles of 16 outputs of a pass.
template <typename T, int NT, int WARPS, int R>
__global__ void __launch_bounds__(WARPS * 32, 1) linear_q4_kernel(Q4Args a) {
  constexpr int THREADS = WARPS * 32, LD = NT * 8 + 1;
  extern __shared__ float sums[];  // [WARPS][R * 16][LD]
  grid_dep_launch();
  grid_dep_wait();
  const int tid = threadIdx.x, warp = __shfl_sync(ALL_LANES, tid >> 5, 0), lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int row_tiles = (a.n + 15) >> 4, k_tiles = (a.k + 63) >> 6, ld = row_tiles * 16, shift = a.group == 128 ? 1 : 0;
  // this CTA's tiles, cut into passes of nearly equal size
  const int each = row_tiles / gridDim.x, more = row_tiles - each * gridDim.x;
  const int t_first = blockIdx.x * each + min((int)blockIdx.x, more), t_count = each + ((int)blockIdx.x < more ? 1 : 0);
  const int passes = (t_count + R - 1) / R, per_pass = (t_count + passes - 1) / passes;
  const bool wide = ((uintptr_t)a.x & 15) == 0 && (a.x_row * sizeof(T)) % 16 == 0;

  struct Loads {
    uint4 w[R];
    uint16_t s[R][2];
    Raw<T> x[NT];
  };
  auto load = [&](Loads& l, int t0, int kt) {
    // (the same for all lanes but the last term, which keeps the addresses in uniform registers)
    const uint8_t* w = a.packed + ((int64_t)t0 * k_tiles + kt) * 512;
    const uint16_t* s = a.scales + (int64_t)(kt >> shift) * ld + t0 * 16;
    const int tiles = min(per_pass, t_first + t_count - t0);
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (r == 0 || r < tiles) {
        l.w[r] = __ldg(reinterpret_cast<const uint4*>(w + (int64_t)r * k_tiles * 512) + lane);
        l.s[r][0] = __ldg(s + r * 16 + g);
        l.s[r][1] = __ldg(s + r * 16 + 8 + g);
      }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int tok = t * 8 + g, from = kt * 64 + c * 16;
      l.x[t].load((const T*)a.x + min(tok, a.m - 1) * a.x_row + from, tok < a.m ? a.k - from : 0, wide);
    }
  };
  Loads now, next;
  if (warp < k_tiles) load(now, t_first, warp);
#pragma unroll 1
  for (int t0 = t_first; t0 < t_first + t_count; t0 += per_pass) {
    const int tiles = min(per_pass, t_first + t_count - t0);
    float acc[R][NT][4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][t][e] = 0.f;
    auto add = [&](const Loads& l) {
      const Tokens<T, NT> x(l.x, c);
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r == 0 || r < tiles) x.add(l.w[r], l.s[r][0], l.s[r][1], acc[r]);
    };
#pragma unroll 1
    for (int kt = warp; kt < k_tiles; kt += WARPS) {
      // the next tile of inputs, or the next pass's first one
      if (kt + WARPS < k_tiles) load(next, t0, kt + WARPS);
      else if (t0 + per_pass < t_first + t_count) load(next, t0 + per_pass, warp);
      add(now);
      now = next;
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (r < tiles)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) sums[(warp * R * 16 + r * 16 + g + (e < 2 ? 0 : 8)) * LD + t * 8 + 2 * c + (e & 1)] = acc[r][t][e];
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < tiles * 16 * a.m; i += THREADS) {
      const int tok = i / (tiles * 16), o = i - tok * (tiles * 16), n = t0 * 16 + o;
      if (n >= a.n) continue;
      float v = a.bias ? to_f32(((const T*)a.bias)[n]) : 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) v += sums[(w * R * 16 + o) * LD + tok];
      ((T*)a.out)[tok * a.out_row + n] = from_f32<T>(v);
    }
    __syncthreads();
  }
}

constexpr int THREADS = 256;  // of the quantiser

// One thread for 16 inputs of one output; the threads of a group are neighbours in a warp. Once for a matrix, and a third of the memory's rate is enough for
// that: 28672 x 8192 FP32 444 us, BF16 300 us (162 and 90 by bytes).
template <typename T>
__global__ void __launch_bounds__(THREADS) quantize_q4_kernel(const T* w, int64_t w_row, int n, int k, int group, uint8_t* packed, uint16_t* scales) {
  const int k_tiles = (k + 63) >> 6, row_tiles = (n + 15) >> 4, pieces = ((k + 127) >> 7) * 8;  // 16 inputs each, whole groups of 128
  const int64_t at = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  const int64_t r64 = at / pieces;
  const int r = (int)r64, p = (int)(at - r64 * pieces);
  const bool row_ok = r64 < row_tiles * 16ll;
  float v[16], m = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int kk = p * 16 + i;
    v[i] = row_ok && r < n && kk < k ? to_f32(w[(size_t)r * w_row + kk]) : 0.f;
    m = fmaxf(m, fabsf(v[i]));
  }
  for (int o = 1; o < group / 16; o <<= 1) m = fmaxf(m, __shfl_xor_sync(ALL_LANES, m, o));
  const __nv_bfloat16 sb = __float2bfloat16_rn(__fdiv_rn(m, 7.f));
  const float s = __bfloat162float(sb);
  if (!row_ok) return;
  if (p % (group / 16) == 0 && p * 16 < k) scales[(size_t)(p * 16 / group) * (row_tiles * 16) + r] = *reinterpret_cast<const uint16_t*>(&sb);
  if (p >= k_tiles * 4) return;
  uint32_t words[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int code = s > 0.f ? min(max((int)rintf(__fdiv_rn(v[i], s)), -8), 7) + 8 : 8;
    words[i >> 3] |= (uint32_t)code << (4 * (((i & 7) >> 1) + (i & 1) * 4));
  }
  uint8_t* to = packed + ((size_t)(r >> 4) * k_tiles + (p >> 2)) * 512 + ((r & 7) * 4 + (p & 3)) * 16 + ((r >> 3) & 1) * 8;
  *reinterpret_cast<uint2*>(to) = make_uint2(words[0], words[1]);
}

template <typename T, int NT, int WARPS, int R>
struct Variant {
  static constexpr int SMEM = WARPS * R * 16 * (NT * 8 + 1) * 4;
  static cudaError_t allow() { return cudaFuncSetAttribute(linear_q4_kernel<T, NT, WARPS, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM); }
  static cudaError_t run(const Q4Args& a, int sms, cudaStream_t s) {
    return launch_kernel(linear_q4_kernel<T, NT, WARPS, R>, dim3(std::min((a.n + 15) / 16, sms)), dim3(WARPS * 32), SMEM, s, true, a);
  }
};
// Few tiles of outputs for a CTA: 16 warps share the inputs' length, which is latency. Many: 8 warps, whose registers hold more tiles, so
// that what is done once for 64 inputs serves more outputs. us with few / many (444 tiles are 7104 outputs on 148 SMs; weights through a ring of
// shared memory, bulk copies, were as fast as these loads into registers):
//                  rows:  1            8            16              rows:  1            8           16
//   4096 x 4096    BF16 5.0 / 7.2    5.1 / 7.2    6.8 / 8.8      FP32 6.1 / 9.1    6.4 / 9.2   10.0 / 13.5
//   6400 x 1600    BF16 3.7 / 4.5    3.9 / 4.7    5.2 / 5.7      FP32 5.6 / 5.6    6.3 / 6.0   10.0 / 8.3
//   7600 x 2000    BF16 5.4 / 5.4    5.6 / 5.6    7.9 / 7.2      FP32 6.6 / 6.7    7.6 / 7.1   12.1 / 10.1
//   16384 x 4096   BF16 14.1 / 12.9  14.5 / 13.2  19.4 / 16.7    FP32 19.3 / 15.9  22.1 / 16.4  35.6 / 23.1
template <typename T, int NT>
struct Choice {
  static constexpr bool PAIR = std::is_same<T, float>::value;
  using Few = Variant<T, NT, PAIR && NT == 2 ? 8 : 16, PAIR ? 2 : 3>;
  using Many = Variant<T, NT, 8, 8>;
  static cudaError_t run(const Q4Args& a, int sms, cudaStream_t s) { return (a.n + 15) / 16 <= 3 * sms ? Few::run(a, sms, s) : Many::run(a, sms, s); }
  static cudaError_t allow() {
    const cudaError_t e = Few::allow();
    return e != cudaSuccess ? e : Many::allow();
  }
};

}  // namespace

cudaError_t init_q4_attributes() {
  for (cudaError_t e : {Choice<float, 1>::allow(), Choice<float, 2>::allow(), Choice<__nv_bfloat16, 1>::allow(), Choice<__nv_bfloat16, 2>::allow()})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

cudaError_t launch_linear_q4(const Q4Args& a, int dtype, int sms, cudaStream_t s) {
  if (dtype == PG_DTYPE_F32) return a.m <= 8 ? Choice<float, 1>::run(a, sms, s) : Choice<float, 2>::run(a, sms, s);
  return a.m <= 8 ? Choice<__nv_bfloat16, 1>::run(a, sms, s) : Choice<__nv_bfloat16, 2>::run(a, sms, s);
}

cudaError_t launch_quantize_q4(const void* w, int64_t w_row, int dtype, int n, int k, int group, uint8_t* packed, uint16_t* scales, cudaStream_t s) {
  const int64_t threads = (int64_t)((n + 15) / 16 * 16) * (((k + 127) / 128) * 8);
  const dim3 grid((unsigned)((threads + THREADS - 1) / THREADS));
  if (dtype == PG_DTYPE_F32)
    return launch_kernel(quantize_q4_kernel<float>, grid, dim3(THREADS), 0, s, false, (const float*)w, w_row, n, k, group, packed, scales);
  return launch_kernel(quantize_q4_kernel<__nv_bfloat16>, grid, dim3(THREADS), 0, s, false, (const __nv_bfloat16*)w, w_row, n, k, group, packed, scales);
}

}  // namespace pg
