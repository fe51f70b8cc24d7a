// Products of few rows with 4-bit weights, and the quantiser that makes them.
//
// out[m][n] = sum over groups of scale[group][n] * sum_k (code[n][k] - 8) x[m][k]. Bound: memory, half a byte for every weight; at that
// rate an SM gets 46 weights a clock, too many for multiply-adds of every row (128 lanes a clock), so the products are m16n8k16 matrix
// instructions with 16 outputs as rows and 8 tokens as columns, on codes turned into 16-bit floats in registers: a field of 4 bits or-ed
// into the mantissa of 2^7 (BF16) or 2^10 (FP16) is that power plus the code, one subtraction gives the exact weight. Order of k
// within a tile is free as long as both operands agree: a lane takes 16 consecutive inputs (k steps of 4), so it loads 16 bytes of
// weights (8 of outputs r and of r + 8) and 16 inputs in a row.
// BF16 inputs are exact operands. FP32 inputs are pairs of FP16 numbers, scaled by a power of two for every 64 inputs of a row, whose
// two halves are separate columns: FP32 grade. A group's sums are FP32, times the scale once per 64 inputs.
// A CTA has R tiles of 16 outputs; its warps take every eighth tile of 64 inputs and are added up in shared memory, in order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "device_util.cuh"
#include "serving.h"

namespace pg {
namespace {

constexpr int WARPS = 8, THREADS = WARPS * 32;

template <bool PAIR>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (PAIR)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Inputs 2 i and 2 i + 1 of a word of 8 codes, as exact 16-bit floats.
template <bool PAIR>
__device__ __forceinline__ uint32_t weights2(uint32_t word, int i) {
  if (PAIR) {
    const uint32_t u = ((word >> (4 * i)) & 0x000F000Fu) | 0x64006400u;  // 1024 + code
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __float2half2_rn(1032.f));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const uint32_t u = ((word >> (4 * i)) & 0x000F000Fu) | 0x43004300u;  // 128 + code
  const __nv_bfloat162 h = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), __float2bfloat162_rn(136.f));
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 16 inputs of one row as operand words: word 2 s + e holds inputs 4 s + 2 e and 4 s + 2 e + 1.
template <typename T>
struct Inputs;
template <>
struct Inputs<__nv_bfloat16> {
  uint32_t w[8];
  __device__ __forceinline__ void load(const __nv_bfloat16* p, int live, bool wide) {
    if (wide && live >= 16) {
      const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 8);
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
      w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    } else {
      const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = (2 * i < live ? (uint32_t)u[2 * i] : 0u) | (2 * i + 1 < live ? (uint32_t)u[2 * i + 1] << 16 : 0u);
    }
  }
};
template <>
struct Inputs<float> {
  uint32_t hi[8], lo[8];
  float back;  // what the row's sums of these 64 inputs are to be multiplied with
  __device__ __forceinline__ void load(const float* p, int live, bool wide) {
    float v[16];
    if (wide && live >= 16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 f = *reinterpret_cast<const float4*>(p + 4 * i);
        v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = i < live ? p[i] : 0.f;
    }
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(v[i]));
    m = fmaxf(m, __shfl_xor_sync(ALL_LANES, m, 1));
    m = fmaxf(m, __shfl_xor_sync(ALL_LANES, m, 2));
    const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -100), 100);
    const float s = __uint_as_float((uint32_t)(127 - e) << 23);
    back = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = v[2 * i] * s, b = v[2 * i + 1] * s;
      const __half2 h = __floats2half2_rn(a, b);
      const float2 f = __half22float2(h);
      const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
      hi[i] = *reinterpret_cast<const uint32_t*>(&h);
      lo[i] = *reinterpret_cast<const uint32_t*>(&l);
    }
  }
};

// NT: groups of 8 tokens.
template <typename T, int NT, int R>
__global__ void __launch_bounds__(THREADS) linear_q4_kernel(Q4Args a) {
  constexpr bool PAIR = std::is_same<T, float>::value;
  __shared__ float sums[WARPS][R * 16][NT * 8 + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int row_tiles = (a.n + 15) >> 4, k_tiles = (a.k + 63) >> 6, t0 = blockIdx.x * R, ld = row_tiles * 16, shift = a.group == 128 ? 1 : 0;
  const bool wide = ((uintptr_t)a.x & 15) == 0 && (a.x_row * sizeof(T)) % 16 == 0;
  float acc[R][NT][4];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[r][t][e] = 0.f;

  for (int kt = warp; kt < k_tiles; kt += WARPS) {
    uint4 w[R];
    float sa[R], sb[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int t = min(t0 + r, row_tiles - 1);
      w[r] = __ldg(reinterpret_cast<const uint4*>(a.packed + ((size_t)t * k_tiles + kt) * 512) + lane);
      const uint16_t* s = a.scales + (size_t)(kt >> shift) * ld + t * 16 + g;
      sa[r] = __uint_as_float((uint32_t)__ldg(s) << 16);
      sb[r] = __uint_as_float((uint32_t)__ldg(s + 8) << 16);
    }
    Inputs<T> x[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int tok = t * 8 + g, from = kt * 64 + c * 16;
      x[t].load((const T*)a.x + (size_t)min(tok, a.m - 1) * a.x_row + from, tok < a.m ? a.k - from : 0, wide);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float hi[NT][4], lo[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) hi[t][e] = lo[t][e] = 0.f;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        // inputs 4 s .. 4 s + 3 of outputs g (words x, y) and g + 8 (z, w)
        const uint32_t wa = s < 2 ? w[r].x : w[r].y, wb = s < 2 ? w[r].z : w[r].w;
        const uint32_t f[4] = {weights2<PAIR>(wa, (s & 1) * 2), weights2<PAIR>(wb, (s & 1) * 2), weights2<PAIR>(wa, (s & 1) * 2 + 1),
                               weights2<PAIR>(wb, (s & 1) * 2 + 1)};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (PAIR) {
            mma16<true>(hi[t], f, x[t].hi[2 * s], x[t].hi[2 * s + 1]);
            mma16<true>(lo[t], f, x[t].lo[2 * s], x[t].lo[2 * s + 1]);
          } else {
            mma16<false>(hi[t], f, x[t].w[2 * s], x[t].w[2 * s + 1]);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float b0 = 1.f, b1 = 1.f;
        if constexpr (PAIR) {  // columns 2 c and 2 c + 1 are the tokens of lanes 8 c and 8 c + 4
          b0 = __shfl_sync(ALL_LANES, x[t].back, c * 8);
          b1 = __shfl_sync(ALL_LANES, x[t].back, c * 8 + 4);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = PAIR ? (hi[t][e] + lo[t][e]) * (e & 1 ? b1 : b0) : hi[t][e];
          acc[r][t][e] = fmaf(v, e < 2 ? sa[r] : sb[r], acc[r][t][e]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[warp][r * 16 + g + (e < 2 ? 0 : 8)][t * 8 + 2 * c + (e & 1)] = acc[r][t][e];
  __syncthreads();
  for (int i = tid; i < R * 16 * a.m; i += THREADS) {
    const int tok = i / (R * 16), o = i - tok * (R * 16), n = t0 * 16 + o;
    if (n >= a.n) continue;
    float v = a.bias ? to_f32(((const T*)a.bias)[n]) : 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += sums[w][o][tok];
    ((T*)a.out)[(size_t)tok * a.out_row + n] = from_f32<T>(v);
  }
}

// One thread for 16 inputs of one output; the threads of a group are neighbours in a warp.
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

template <typename T, int NT, int R>
cudaError_t run(const Q4Args& a, cudaStream_t s) {
  return launch_kernel(linear_q4_kernel<T, NT, R>, dim3(((a.n + 15) / 16 + R - 1) / R), dim3(THREADS), 0, s, false, a);
}
template <typename T>
cudaError_t run_of(const Q4Args& a, cudaStream_t s) {
  return a.m <= 8 ? run<T, 1, 1>(a, s) : run<T, 2, 1>(a, s);
}

}  // namespace

cudaError_t init_q4_attributes() { return cudaSuccess; }

cudaError_t launch_linear_q4(const Q4Args& a, int dtype, int sms, cudaStream_t s) {
  (void)sms;
  return dtype == PG_DTYPE_F32 ? run_of<float>(a, s) : run_of<__nv_bfloat16>(a, s);
}

cudaError_t launch_quantize_q4(const void* w, int64_t w_row, int dtype, int n, int k, int group, uint8_t* packed, uint16_t* scales, cudaStream_t s) {
  const int64_t threads = (int64_t)((n + 15) / 16 * 16) * (((k + 127) / 128) * 8);
  const dim3 grid((unsigned)((threads + THREADS - 1) / THREADS));
  if (dtype == PG_DTYPE_F32)
    return launch_kernel(quantize_q4_kernel<float>, grid, dim3(THREADS), 0, s, false, (const float*)w, w_row, n, k, group, packed, scales);
  return launch_kernel(quantize_q4_kernel<__nv_bfloat16>, grid, dim3(THREADS), 0, s, false, (const __nv_bfloat16*)w, w_row, n, k, group, packed, scales);
}

}  // namespace pg
