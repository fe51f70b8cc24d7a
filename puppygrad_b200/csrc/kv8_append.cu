// Appending to the 8-bit paged cache: rotation, the blocks' scales, e4m3 codes.
//
// A block is one page's keys or values of one head. Its scale is a power of two, so that a later, larger token only moves the
// exponents of the codes that are there (a code that becomes subnormal is rounded once more), and code = e4m3(x / scale) rounds x
// once. Each block that gets tokens belongs to one CTA, which therefore needs no atomics: it stages the new tokens in shared
// memory as FP32, turns them, takes the largest magnitude, and writes keys by token and values by head entry, the order in which
// the attention's matrix instructions take them. Queries are turned by CTAs of their own in the same launch.
// Bound: memory (every value read once, every code written once); a step of few tokens is launch latency.
#include <cfloat>

#include "kv8.cuh"

namespace pg {
namespace {

constexpr int THREADS = 128;
constexpr int MIN_EXP = -100;  // of a scale: below every magnitude that matters, above FP32's subnormals in both directions

// (cos, sin) of pos * base^(-2 i / rot). The angle is formed and reduced in 64 bits: at position 10^5 an FP32 angle is off by 0.01.
__device__ __forceinline__ float2 turn_of(int pos, int i, double step) {
  double s, c;
  sincos((double)pos * exp2(step * i), &s, &c);
  return make_float2((float)c, (float)s);
}
// Products rounded one by one: an append is the same whatever the compiler fuses.
__device__ __forceinline__ float2 turned(float a, float b, float2 cs) {
  return make_float2(__fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y)), __fadd_rn(__fmul_rn(b, cs.x), __fmul_rn(a, cs.y)));
}

// Smallest power of two that keeps `amax` within 448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)(max(e, MIN_EXP) + 127) << 23);
}

template <typename T>
__device__ void turn_queries(const Kv8AppendArgs& a, int row, float2* cs) {
  const Kv8View& c = a.c;
  int pos;
  if (a.row_start) {
    // the sequence of this row: the last one that starts at or before it
    int lo = 0, hi = c.seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.row_start[mid] <= row) lo = mid;
      else hi = mid;
    }
    const SeqRows r = seq_rows(a.row_start, a.rows, lo);
    if (row < r.first || row >= r.first + r.n) return;
    pos = a.lens[lo] - r.n + (row - r.first);
  } else {
    pos = a.lens[row] - 1;
  }
  const int half = a.rot_dims >> 1, tid = threadIdx.x;
  for (int i = tid; i < half; i += THREADS) cs[i] = turn_of(pos, i, a.turn_step);
  __syncthreads();
  const T* q = (const T*)a.q + (size_t)row * a.q_row;
  T* o = (T*)a.q_out + (size_t)row * a.q_out_row;
  const int per = c.dim - half;  // pairs first, then the entries that stay
  for (int x = tid; x < a.heads * per; x += THREADS) {
    const int h = x / per, i = x - h * per;
    const size_t at = (size_t)h * c.dim + i;
    if (i < half) {
      const float2 t = turned(to_f32(q[at]), to_f32(q[at + half]), cs[i]);
      o[at] = from_f32<T>(t.x);
      o[at + half] = from_f32<T>(t.y);
    } else {
      o[at + half] = q[at + half];
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) kv8_append_kernel(Kv8AppendArgs a, int slots, int most) {
  extern __shared__ float sm[];  // [most][dim + 1] values, [most][rot_dims / 2] turns; most: new tokens of a page
  const Kv8View& c = a.c;
  const int tid = threadIdx.x, blocks = slots * c.kv_heads * 2;
  if ((int)blockIdx.x >= blocks) {
    turn_queries<T>(a, blockIdx.x - blocks, reinterpret_cast<float2*>(sm));
    return;
  }
  const int side = blockIdx.x & 1, h = (blockIdx.x >> 1) % c.kv_heads, slot = (blockIdx.x >> 1) / c.kv_heads;
  // sequence b has the page slots from row_start[b] / P + 2 b on: as many as its rows can touch, or more
  int b = slot, local = 0;
  if (a.row_start) {
    int lo = 0, hi = c.seqs;
    auto first_slot = [&](int s) { return (min(max(a.row_start[s], 0), a.rows) >> c.page_shift) + 2 * s; };
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first_slot(mid) <= slot) lo = mid;
      else hi = mid;
    }
    b = lo;
    local = slot - first_slot(b);
  }
  const SeqRows r = seq_rows(a.row_start, a.rows, b);
  const int len = a.lens[b], start = len - r.n, from = max(start, 0);  // new positions: from .. len - 1
  const int lp = (from >> c.page_shift) + local, p = c.page_tokens;
  if (r.n <= 0 || len <= from || local < 0 || lp > (len - 1) >> c.page_shift) return;
  const int page = page_of(c, b, lp);
  if (page < 0) return;
  const int base = lp << c.page_shift, o0 = max(from - base, 0), o1 = min(len - base, p), n = o1 - o0;
  const int row0 = r.first + (base + o0 - start);

  const int dim = c.dim, ld = dim + 1, half = side == 0 ? a.rot_dims >> 1 : 0;
  float2* cs = reinterpret_cast<float2*>(sm + ((most * ld + 1) & ~1));
  const T* src = side == 0 ? (const T*)a.k + (size_t)h * dim : (const T*)a.v + (size_t)h * dim;
  const int64_t step = side == 0 ? a.k_row : a.v_row;
  for (int x = tid; x < n * dim; x += THREADS) {
    const int t = x / dim, d = x - t * dim;
    sm[t * ld + d] = to_f32(src[(row0 + t) * step + d]);
  }
  if (half) {
    for (int x = tid; x < n * half; x += THREADS) {
      const int t = x / half, i = x - t * half;
      cs[x] = turn_of(base + o0 + t, i, a.turn_step);
    }
  }
  __syncthreads();
  if (half) {
    for (int x = tid; x < n * half; x += THREADS) {
      const int t = x / half, i = x - t * half;
      float* v = sm + t * ld + i;
      const float2 o = turned(v[0], v[half], cs[x]);
      v[0] = o.x;
      v[half] = o.y;
    }
    __syncthreads();
  }
  float amax = 0.f;
  bool finite = true;
  for (int x = tid; x < n * dim; x += THREADS) {
    const int t = x / dim;
    const float v = fabsf(sm[t * ld + (x - t * dim)]);
    amax = fmaxf(amax, v);
    finite = finite && v <= FLT_MAX;
  }
  __shared__ float red[THREADS / 32];
  amax = lane_max(amax);
  if ((tid & 31) == 0) red[tid >> 5] = amax;
  finite = __syncthreads_and(finite);
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) amax = fmaxf(amax, red[w]);

  float* scale_at = c.scales + ((size_t)page * c.kv_heads + h) * 2 + side;
  const float old = o0 ? *scale_at : 0.f;
  float scale = scale_for(amax);
  if (old > scale) scale = old;
  const bool ok = finite && old == old;
  if (!ok) scale = __uint_as_float(0x7FC00000u);
  __syncthreads();  // everybody has read the old scale
  if (tid == 0) *scale_at = scale;
  const float inv = ok ? 1.f / scale : 0.f;

  const int dp = kv8_padded(dim);
  uint8_t* blk = c.pool + (((size_t)page * c.kv_heads + h) * 2 + side) * (size_t)(p * dp);
  if (o0 && ok && old != scale) {  // earlier tokens in the new scale
    const float ratio = old * inv;
    for (int x = tid; x < o0 * dp; x += THREADS) {
      const size_t at = side == 0 ? (size_t)x : (size_t)(x / o0) * p + x % o0;
      const uint32_t f = e4m3x2_to_f16x2(blk[at]);
      blk[at] = (uint8_t)f32x2_to_e4m3x2(__half2float(__ushort_as_half((unsigned short)f)) * ratio, 0.f);
    }
  }
  auto value = [&](int t, int d) { return ok && d < dim ? sm[t * ld + d] * inv : 0.f; };
  if (side == 0) {
    const int quads = dp >> 2;
    for (int x = tid; x < n * quads; x += THREADS) {
      const int t = x / quads, d = (x - t * quads) * 4;
      *reinterpret_cast<uint32_t*>(blk + (size_t)(o0 + t) * dp + d) = f32x4_to_e4m3x4(value(t, d), value(t, d + 1), value(t, d + 2), value(t, d + 3));
    }
  } else {
    const int q0 = o0 >> 2, quads = ((o1 + 3) >> 2) - q0;
    for (int x = tid; x < dp * quads; x += THREADS) {
      const int d = x / quads, t = (q0 + (x - d * quads)) * 4;  // tokens t .. t + 3 of the page
      uint8_t* to = blk + (size_t)d * p + t;
      if (t >= o0 && t + 4 <= o1) {
        *reinterpret_cast<uint32_t*>(to) = f32x4_to_e4m3x4(value(t - o0, d), value(t + 1 - o0, d), value(t + 2 - o0, d), value(t + 3 - o0, d));
      } else {
        for (int i = 0; i < 4; ++i)
          if (t + i >= o0 && t + i < o1) to[i] = (uint8_t)f32x2_to_e4m3x2(value(t + i - o0, d), 0.f);
      }
    }
  }
}

}  // namespace

cudaError_t init_kv8_append_attributes() {
  const int most = (64 * 257 + 1) * 4 + 64 * 128 * 8;
  cudaError_t e = cudaFuncSetAttribute(kv8_append_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  return e != cudaSuccess ? e : cudaFuncSetAttribute(kv8_append_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
}

cudaError_t launch_kv8_append(const Kv8AppendArgs& a, int dtype, cudaStream_t s) {
  const int slots = a.row_start ? (a.rows >> a.c.page_shift) + 2 * a.c.seqs : a.c.seqs, most = a.row_start ? a.c.page_tokens : 1;
  const unsigned grid = (unsigned)slots * a.c.kv_heads * 2 + (a.q ? a.rows : 0);
  const size_t smem = (size_t)((most * (a.c.dim + 1) + 1) & ~1) * 4 + (size_t)most * (a.rot_dims / 2) * 8;
  auto k = dtype == PG_DTYPE_F32 ? kv8_append_kernel<float> : kv8_append_kernel<__nv_bfloat16>;
  return launch_kernel(k, dim3(grid), dim3(THREADS), smem, s, false, a, slots, most);
}

}  // namespace pg
