// Appending to the 8-bit paged cache: rotation, the blocks' scales, e4m3 codes.
//
// A block is one page's keys or values of one head. Its scale is a power of two, so that a later, larger token only moves the
// exponents of the codes that are there (a code that becomes subnormal is rounded once more), and code = e4m3(x / scale) rounds x
// once. Each block that gets tokens belongs to one CTA (or warp), which therefore needs no atomics: it holds the new tokens as FP32,
// turned, takes the largest magnitude, and writes keys by token and values by head entry, the order in which the attention's
// matrix instructions take them.
//  - one token for every sequence: a warp for each block and each query head, an entry for every lane;
//  - more, rows on 16-byte boundaries: a CTA for each block, eight entries for a thread at a time, in registers;
//  - more, any rows: a CTA for each block, values staged in shared memory.
// Bound: memory (every value read once, every code written once); a step of few tokens is launch latency. Measured: 8 prompts of up to 2047
// tokens, 46 us (21 by bytes: instructions of the conversions, and a block's loads, maximum and stores one after the other); 64 single tokens
// 4.8 us, one 2.2 us.
#include "kv8.cuh"

namespace pg {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int MIN_EXP = -100;  // of a scale: below every magnitude that matters, above FP32's subnormals in both directions

// Turns a position makes of entry i: base^(-2 i / rot) / 2 pi.
__device__ __forceinline__ double turns_of(const Kv8AppendArgs& a, int i) { return exp2(a.turn_step * i) * 0.15915494309189534; }
// (cos, sin) of a position's angle. The angle is formed and reduced in 64 bits (at position 10^5 an FP32 angle is off by 0.01), what
// the reduced angle's rounding to FP32 leaves out is put back to first order.
__device__ __forceinline__ float2 turn_at(int pos, double turns) {
  double t = (double)pos * turns;
  t = 2.0 * (t - rint(t));  // in half turns, -1 .. 1
  const float h = (float)t, rest = (float)(t - (double)h) * 3.14159265f;
  float s, c;
  sincospif(h, &s, &c);
  return make_float2(fmaf(-rest, s, c), fmaf(rest, c, s));
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

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
// The block's scale with the new tokens: the one it has, where it holds earlier tokens, or what the new ones need. NaN where either
// is not finite. `inv`: what values are multiplied with, 0 for NaN.
struct BlockScale {
  float scale, inv;
  bool ok;
  // `top`: the largest of the new values' magnitude bits, which are in the order of the magnitudes, infinity and NaN above all
  __device__ __forceinline__ BlockScale(float old, uint32_t top) {
    scale = scale_for(__uint_as_float(top));
    if (old > scale) scale = old;
    ok = top < 0x7F800000u && old == old;
    inv = ok ? 1.f / scale : 0.f;
    if (!ok) scale = __uint_as_float(0x7FC00000u);
  }
};

__device__ __forceinline__ uint8_t in_new_scale(uint8_t code, float ratio) {
  const uint32_t f = e4m3x2_to_f16x2(code);
  return (uint8_t)f32x2_to_e4m3x2(__half2float(__ushort_as_half((unsigned short)f)) * ratio, 0.f);
}
// Earlier tokens of a block, places 0 .. o0 - 1, in its new scale.
__device__ __forceinline__ void rescale(uint8_t* blk, int side, int o0, int p, int dp, float ratio, int first, int step) {
  for (int x = first; x < o0 * dp; x += step) {
    const size_t at = side == 0 ? (size_t)x : (size_t)(x / o0) * p + x % o0;
    blk[at] = in_new_scale(blk[at], ratio);
  }
}

// The page that page slot `slot` of the call stands for: sequence b has the slots from row_start[b] / P + 2 b on, as many as its
// rows can touch, or more.
struct PageRows {
  int page, o0, n, row0, pos0;  // -1: none; its first new place, how many, the first one's row and position
  __device__ __forceinline__ PageRows(const Kv8AppendArgs& a, int slot) {
    const Kv8View& c = a.c;
    page = -1;
    auto first_slot = [&](int s) { return (min(max(a.row_start[s], 0), a.rows) >> c.page_shift) + 2 * s; };
    int lo = 0, hi = c.seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first_slot(mid) <= slot) lo = mid;
      else hi = mid;
    }
    const SeqRows r = seq_rows(a.row_start, a.rows, lo);
    const int len = a.lens[lo], start = len - r.n, from = max(start, 0);  // new positions: from .. len - 1
    const int local = slot - first_slot(lo), lp = (from >> c.page_shift) + local;
    if (r.n <= 0 || len <= from || local < 0 || lp > (len - 1) >> c.page_shift) return;
    const int base = lp << c.page_shift;
    o0 = max(from - base, 0);
    n = min(len - base, c.page_tokens) - o0;
    pos0 = base + o0;
    row0 = r.first + (pos0 - start);
    page = page_of(c, lo, lp);
  }
};

// Position of a row, or -1 where it belongs to no sequence.
__device__ __forceinline__ int row_position(const Kv8AppendArgs& a, int row, bool* any) {
  int lo = 0, hi = a.c.seqs;  // the last sequence that starts at or before the row
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.row_start[mid] <= row) lo = mid;
    else hi = mid;
  }
  const SeqRows r = seq_rows(a.row_start, a.rows, lo);
  *any = row >= r.first && row < r.first + r.n;
  return a.lens[lo] - r.n + (row - r.first);
}

// ------------------------------------------------------------------ one token for every sequence
template <typename T>
__global__ void __launch_bounds__(THREADS) kv8_append_step_kernel(Kv8AppendArgs a) {
  __shared__ float2 cs[128];
  grid_dep_launch();
  grid_dep_wait();
  const Kv8View& c = a.c;
  const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, half = a.rot_dims >> 1;
  const int item = blockIdx.y * WARPS + warp, dim = c.dim;  // keys of every head, values of every head, query heads
  const bool any = item < 2 * c.kv_heads + (a.q ? a.heads : 0);
  const int side = item < c.kv_heads ? 0 : item < 2 * c.kv_heads ? 1 : 2, h = item - side * c.kv_heads;
  // everything that can be asked for at once: the values, then length, page and scale one after the other
  const T* x = side == 0 ? (const T*)a.k + b * a.k_row : side == 1 ? (const T*)a.v + b * a.v_row : (const T*)a.q + b * a.q_row;
  x += (size_t)h * dim;
  float v[8], o[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int d = lane + 32 * k;
    v[k] = any && d < dim ? to_f32(x[d]) : 0.f;
    o[k] = any && side != 1 && d < 2 * half ? to_f32(x[d < half ? d + half : d - half]) : 0.f;
  }
  const int pos = a.lens[b] - 1, p = c.page_tokens, o0 = pos & (p - 1);
  const int page = !any || side == 2 || pos < 0 ? -1 : page_of(c, b, pos >> c.page_shift);
  float* scale_at = c.scales + ((size_t)max(page, 0) * c.kv_heads + (side == 2 ? 0 : h)) * 2 + (side & 1);
  const float old = page >= 0 && o0 ? *scale_at : 0.f;
  if (tid < half) cs[tid] = turn_at(pos, turns_of(a, tid));
  __syncthreads();
  if (!any) return;
  if (side != 1) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int d = lane + 32 * k;
      if (d >= 2 * half) continue;
      const float2 t = d < half ? turned(v[k], o[k], cs[d]) : turned(o[k], v[k], cs[d - half]);
      v[k] = d < half ? t.x : t.y;
    }
  }
  if (side == 2) {
    T* to = (T*)a.q_out + b * a.q_out_row + (size_t)h * dim;
    __syncwarp();  // q_out may be q: every lane has read its partners
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (lane + 32 * k < dim) to[lane + 32 * k] = from_f32<T>(v[k]);
    return;
  }
  if (page < 0) return;
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, magnitude(v[k]));
  top = __reduce_max_sync(ALL_LANES, top);
  const int dp = kv8_padded(dim);
  const BlockScale s(old, top);
  if (lane == 0) *scale_at = s.scale;
  uint8_t* blk = c.pool + (((size_t)page * c.kv_heads + h) * 2 + side) * (size_t)(p * dp);
  if (o0 && s.ok && old != s.scale) rescale(blk, side, o0, p, dp, old * s.inv, lane, 32);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int d = lane + 32 * k;
    if (d < dp) blk[side == 0 ? (size_t)o0 * dp + d : (size_t)d * p + o0] = (uint8_t)f32x2_to_e4m3x2(s.ok ? v[k] * s.inv : 0.f, 0.f);
  }
}

// ------------------------------------------------------------------ portions, rows on 16-byte boundaries
// (cos, sin) of n tokens from pos0 on: cs[t][half].
__device__ __forceinline__ void turn_table(const Kv8AppendArgs& a, double* turns, float2* cs, int n, int half, int pos0, const int* positions) {
  for (int i = threadIdx.x; i < half; i += THREADS) turns[i] = turns_of(a, i);
  __syncthreads();
  for (int x = threadIdx.x; x < n * half; x += THREADS) {
    const int t = x / half, i = x - t * half;
    cs[x] = turn_at(positions ? positions[t] : pos0 + t, turns[i]);
  }
  __syncthreads();
}
// The same in the order in which neighbouring threads, which have neighbouring groups of 8 entries, take them 16 bytes at a time
// (`half` a multiple of 8): [t][entry pair of the group][group] of two (cos, sin).
__device__ __forceinline__ void turn_table_by_eights(const Kv8AppendArgs& a, double* turns, float2* cs, int n, int half, int pos0, const int* positions) {
  for (int i = threadIdx.x; i < half; i += THREADS) turns[i] = turns_of(a, i);
  __syncthreads();
  const int groups = half >> 3;
  for (int x = threadIdx.x; x < n * half; x += THREADS) {
    const int t = x / half, i = x - t * half;
    cs[((t * 4 + ((i & 7) >> 1)) * groups + (i >> 3)) * 2 + (i & 1)] = turn_at(positions ? positions[t] : pos0 + t, turns[i]);
  }
  __syncthreads();
}
// Group i of a table row, applied to entries u (first half) and w (second half).
__device__ __forceinline__ void turn_eight(const float2* cs, int t, int groups, int i, float (&u)[8], float (&w)[8]) {
  const float4* at = reinterpret_cast<const float4*>(cs) + t * 4 * groups + i;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float4 f = at[e * groups];
    const float2 x = turned(u[2 * e], w[2 * e], make_float2(f.x, f.y)), y = turned(u[2 * e + 1], w[2 * e + 1], make_float2(f.z, f.w));
    u[2 * e] = x.x;
    w[2 * e] = x.y;
    u[2 * e + 1] = y.x;
    w[2 * e + 1] = y.y;
  }
}
// Entries d .. d + 7 of row x, turned by table row t.
template <typename T>
__device__ __forceinline__ void eight_turned(const T* x, int d, int half, const float2* cs, int t, float (&v)[8]) {
  load8(x + d, v);
  if (d >= 2 * half) return;
  float o[8];
  if (d < half) {
    load8(x + d + half, o);
    turn_eight(cs, t, half >> 3, d >> 3, v, o);
  } else {
    load8(x + d - half, o);
    turn_eight(cs, t, half >> 3, (d - half) >> 3, o, v);
  }
}

constexpr int QUERY_ROWS = 8;  // of a CTA that turns queries

template <int DP, typename T>
__global__ void __launch_bounds__(THREADS, DP <= 128 ? 4 : 2) kv8_append_block_kernel(Kv8AppendArgs a, int slots) {
  extern __shared__ __align__(16) float2 cs[];  // [tokens][rot_dims / 2]
  __shared__ double turns[128];
  __shared__ uint32_t red[WARPS];
  __shared__ int positions[QUERY_ROWS], there[QUERY_ROWS];
  grid_dep_launch();
  grid_dep_wait();
  const Kv8View& c = a.c;
  const int tid = threadIdx.x, blocks = slots * c.kv_heads * 2, dim = c.dim;
  // CTAs of blocks, which compute more, and of queries, which move more, in turn
  const int both = min(blocks, (int)gridDim.x - blocks), bx = blockIdx.x;
  const bool queries = bx < 2 * both ? bx & 1 : blocks == both;
  const int number = bx < 2 * both ? bx >> 1 : bx - both;
  if (queries) {
    const int row0 = number * QUERY_ROWS, n = min(QUERY_ROWS, a.rows - row0), half = a.rot_dims >> 1;
    // an item: entries 8 i .. and their partners together (q_out may be q), of several rows, which are on their way at once; the first
    // item's before the positions are known
    constexpr int AT_ONCE = sizeof(T) == 2 ? 4 : 2, VECS = sizeof(T) / 2;  // rows; 16-byte words of 8 values
    const int pairs = half >> 3, per = pairs + ((dim - 2 * half) >> 3), across = a.heads * per, items = across * ((n + AT_ONCE - 1) / AT_ONCE);
    uint4 u[AT_ONCE][VECS], w[AT_ONCE][VECS];
    struct Item {
      int t0, i;
      int64_t at;
    };
    auto item_at = [&](int y) {
      const int t = y / across, x = y - t * across, h = x / per, i = x - h * per;
      return Item{t * AT_ONCE, i, (int64_t)h * dim + (i < pairs ? i * 8 : 2 * half + (i - pairs) * 8)};
    };
    auto ask = [&](const Item& m) {
      const T* q = (const T*)a.q + row0 * a.q_row + m.at;
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k)
        if (m.t0 + k < n)
#pragma unroll
          for (int e = 0; e < VECS; ++e) {
            u[k][e] = reinterpret_cast<const uint4*>(q + (m.t0 + k) * a.q_row)[e];
            if (m.i < pairs) w[k][e] = reinterpret_cast<const uint4*>(q + (m.t0 + k) * a.q_row + half)[e];
          }
    };
    Item m{};
    if (tid < items) {
      m = item_at(tid);
      ask(m);
    }
    if (tid < n) {
      bool any;
      positions[tid] = row_position(a, row0 + tid, &any);
      there[tid] = any;
    }
    __syncthreads();
    turn_table_by_eights(a, turns, cs, n, half, 0, positions);
    for (int y = tid; y < items; y += THREADS) {
      if (y != tid) {
        m = item_at(y);
        ask(m);
      }
      T* o = (T*)a.q_out + row0 * a.q_out_row + m.at;
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        if (m.t0 + k >= n || !there[m.t0 + k]) continue;
        T* to = o + (m.t0 + k) * a.q_out_row;
        if (m.i < pairs) {
          float f[8], g[8];
          load8(reinterpret_cast<const T*>(u[k]), f);
          load8(reinterpret_cast<const T*>(w[k]), g);
          turn_eight(cs, m.t0 + k, pairs, m.i, f, g);
          store4(to, make_float4(f[0], f[1], f[2], f[3]));
          store4(to + 4, make_float4(f[4], f[5], f[6], f[7]));
          store4(to + half, make_float4(g[0], g[1], g[2], g[3]));
          store4(to + half + 4, make_float4(g[4], g[5], g[6], g[7]));
        } else {
#pragma unroll
          for (int e = 0; e < VECS; ++e) reinterpret_cast<uint4*>(to)[e] = u[k][e];
        }
      }
    }
    return;
  }
  const int side = number & 1, h = (number >> 1) % c.kv_heads;
  const PageRows pr(a, (number >> 1) / c.kv_heads);
  if (pr.page < 0) return;
  const int p = c.page_tokens, half = side == 0 ? a.rot_dims >> 1 : 0, n = pr.n, o0 = pr.o0;
  if (half) turn_table_by_eights(a, turns, cs, n, half, pr.pos0, nullptr);

  // keys: item (token, 8 entries), values: item (8 entries, 4 tokens), all of a thread's in registers
  constexpr int KI = DP / 32, VI = (DP + 127) / 128;  // at most, with pages of 64
  float v[KI > 4 * VI ? KI : 4 * VI][8];
  uint32_t top = 0;
  auto look = [&](const float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, magnitude(x[e]));
  };
  if (side == 0) {
    const T* src = (const T*)a.k + (size_t)h * dim;
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int x = i * THREADS + tid, t = x / (DP / 8), d = (x - t * (DP / 8)) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
      if (t < n && d < dim) eight_turned(src + (pr.row0 + t) * a.k_row, d, half, cs, t, v[i]);
      look(v[i]);
    }
  } else {
    const T* src = (const T*)a.v + (size_t)h * dim;
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int x = i * THREADS + tid, d = (x / (p >> 2)) * 8, t = (x & ((p >> 2) - 1)) * 4 - o0;  // t: from the first new token
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[4 * i + k][e] = 0.f;
        if (t + k >= 0 && t + k < n && d < dim) load8(src + (pr.row0 + t + k) * a.v_row + d, v[4 * i + k]);
        look(v[4 * i + k]);
      }
    }
  }
  top = __reduce_max_sync(ALL_LANES, top);
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) top = max(top, red[w]);
  float* scale_at = c.scales + ((size_t)pr.page * c.kv_heads + h) * 2 + side;
  const float old = o0 ? *scale_at : 0.f;
  const BlockScale s(old, top);
  uint8_t* blk = c.pool + (((size_t)pr.page * c.kv_heads + h) * 2 + side) * (size_t)(p * DP);
  __syncthreads();  // everybody has read the old scale
  if (tid == 0) *scale_at = s.scale;
  if (o0 && s.ok && old != s.scale) rescale(blk, side, o0, p, DP, old * s.inv, tid, THREADS);
  auto code = [&](float x) { return s.ok ? x * s.inv : 0.f; };
  if (side == 0) {
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int x = i * THREADS + tid, t = x / (DP / 8), d = (x - t * (DP / 8)) * 8;
      if (t >= n) continue;
      uint2 w;
      w.x = f32x4_to_e4m3x4(code(v[i][0]), code(v[i][1]), code(v[i][2]), code(v[i][3]));
      w.y = f32x4_to_e4m3x4(code(v[i][4]), code(v[i][5]), code(v[i][6]), code(v[i][7]));
      *reinterpret_cast<uint2*>(blk + (size_t)(o0 + t) * DP + d) = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int x = i * THREADS + tid, d = (x / (p >> 2)) * 8, at = (x & ((p >> 2) - 1)) * 4, t = at - o0;
      if (d >= DP || t + 3 < 0 || t >= n) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint8_t* to = blk + (size_t)(d + e) * p + at;
        const uint32_t w = f32x4_to_e4m3x4(code(v[4 * i][e]), code(v[4 * i + 1][e]), code(v[4 * i + 2][e]), code(v[4 * i + 3][e]));
        if (t >= 0 && t + 4 <= n) {
          *reinterpret_cast<uint32_t*>(to) = w;
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (t + k >= 0 && t + k < n) to[k] = (uint8_t)(w >> (8 * k));
        }
      }
    }
  }
}

// ------------------------------------------------------------------ portions, any rows
template <typename T>
__device__ void turn_queries(const Kv8AppendArgs& a, int row, float2* cs) {
  const Kv8View& c = a.c;
  bool any;
  const int pos = row_position(a, row, &any);
  if (!any) return;
  const int half = a.rot_dims >> 1, tid = threadIdx.x;
  for (int i = tid; i < half; i += THREADS) cs[i] = turn_at(pos, turns_of(a, i));
  __syncthreads();
  const T* q = (const T*)a.q + row * a.q_row;
  T* o = (T*)a.q_out + row * a.q_out_row;
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
__global__ void __launch_bounds__(THREADS) kv8_append_any_kernel(Kv8AppendArgs a, int slots) {
  extern __shared__ __align__(16) float sm[];  // [page_tokens][dim + 1] values, [page_tokens][rot_dims / 2] turns
  __shared__ double turns[128];
  __shared__ uint32_t red[WARPS];
  grid_dep_launch();
  grid_dep_wait();
  const Kv8View& c = a.c;
  const int tid = threadIdx.x, blocks = slots * c.kv_heads * 2;
  if ((int)blockIdx.x >= blocks) {
    turn_queries<T>(a, blockIdx.x - blocks, reinterpret_cast<float2*>(sm));
    return;
  }
  const int side = blockIdx.x & 1, h = (blockIdx.x >> 1) % c.kv_heads;
  const PageRows pr(a, (blockIdx.x >> 1) / c.kv_heads);
  if (pr.page < 0) return;
  const int p = c.page_tokens, o0 = pr.o0, n = pr.n, o1 = o0 + n;
  const int dim = c.dim, ld = dim + 1, half = side == 0 ? a.rot_dims >> 1 : 0;
  float2* cs = reinterpret_cast<float2*>(sm + ((p * ld + 1) & ~1));
  const T* src = side == 0 ? (const T*)a.k + (size_t)h * dim : (const T*)a.v + (size_t)h * dim;
  const int64_t step = side == 0 ? a.k_row : a.v_row;
  for (int x = tid; x < n * dim; x += THREADS) {
    const int t = x / dim, d = x - t * dim;
    sm[t * ld + d] = to_f32(src[(pr.row0 + t) * step + d]);
  }
  __syncthreads();
  if (half) {
    turn_table(a, turns, cs, n, half, pr.pos0, nullptr);
    for (int x = tid; x < n * half; x += THREADS) {
      const int t = x / half, i = x - t * half;
      float* v = sm + t * ld + i;
      const float2 o = turned(v[0], v[half], cs[x]);
      v[0] = o.x;
      v[half] = o.y;
    }
    __syncthreads();
  }
  uint32_t top = 0;
  for (int x = tid; x < n * dim; x += THREADS) {
    const int t = x / dim;
    top = max(top, magnitude(sm[t * ld + (x - t * dim)]));
  }
  top = __reduce_max_sync(ALL_LANES, top);
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) top = max(top, red[w]);
  float* scale_at = c.scales + ((size_t)pr.page * c.kv_heads + h) * 2 + side;
  const float old = o0 ? *scale_at : 0.f;
  const BlockScale s(old, top);
  __syncthreads();  // everybody has read the old scale
  if (tid == 0) *scale_at = s.scale;
  const int dp = kv8_padded(dim);
  uint8_t* blk = c.pool + (((size_t)pr.page * c.kv_heads + h) * 2 + side) * (size_t)(p * dp);
  if (o0 && s.ok && old != s.scale) rescale(blk, side, o0, p, dp, old * s.inv, tid, THREADS);
  auto value = [&](int t, int d) { return s.ok && d < dim ? sm[t * ld + d] * s.inv : 0.f; };
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

template <int DP, typename T>
cudaError_t run_blocks(const Kv8AppendArgs& a, int slots, cudaStream_t s) {
  const unsigned grid = (unsigned)slots * a.c.kv_heads * 2 + (a.q ? (a.rows + QUERY_ROWS - 1) / QUERY_ROWS : 0);
  return launch_kernel(kv8_append_block_kernel<DP, T>, dim3(grid), dim3(THREADS), (size_t)a.c.page_tokens * (a.rot_dims / 2) * 8, s, true, a, slots);
}
template <typename T>
cudaError_t run(const Kv8AppendArgs& a, cudaStream_t s) {
  const Kv8View& c = a.c;
  if (!a.row_start) {
    const int items = 2 * c.kv_heads + (a.q ? a.heads : 0);
    return launch_kernel(kv8_append_step_kernel<T>, dim3(c.seqs, (items + WARPS - 1) / WARPS), dim3(THREADS), 0, s, true, a);
  }
  const int slots = (a.rows >> c.page_shift) + 2 * c.seqs;
  auto wide = [](const void* p, int64_t row) { return (((uintptr_t)p | (uintptr_t)(row * (int64_t)sizeof(T))) & 15) == 0; };
  if (c.dim % 8 == 0 && a.rot_dims % 16 == 0 && wide(a.k, a.k_row) && wide(a.v, a.v_row) && (!a.q || (wide(a.q, a.q_row) && wide(a.q_out, a.q_out_row)))) {
    switch (kv8_padded(c.dim)) {
      case 64: return run_blocks<64, T>(a, slots, s);
      case 128: return run_blocks<128, T>(a, slots, s);
      case 192: return run_blocks<192, T>(a, slots, s);
      default: return run_blocks<256, T>(a, slots, s);
    }
  }
  const unsigned grid = (unsigned)slots * c.kv_heads * 2 + (a.q ? a.rows : 0);
  const size_t smem = (size_t)((c.page_tokens * (c.dim + 1) + 1) & ~1) * 4 + (size_t)c.page_tokens * (a.rot_dims / 2) * 8;
  return launch_kernel(kv8_append_any_kernel<T>, dim3(grid), dim3(THREADS), smem, s, true, a, slots);
}

template <typename F>
cudaError_t allow(F* kernel, int bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

}  // namespace

cudaError_t init_kv8_append_attributes() {
  const int turns = 64 * 128 * 8, values = (64 * 257 + 1) * 4 + turns;
  cudaError_t all[] = {allow(kv8_append_any_kernel<float>, values), allow(kv8_append_any_kernel<__nv_bfloat16>, values),
                       allow(kv8_append_block_kernel<192, float>, turns), allow(kv8_append_block_kernel<256, float>, turns),
                       allow(kv8_append_block_kernel<192, __nv_bfloat16>, turns), allow(kv8_append_block_kernel<256, __nv_bfloat16>, turns)};
  for (cudaError_t e : all)
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

cudaError_t launch_kv8_append(const Kv8AppendArgs& a, int dtype, cudaStream_t s) {
  return dtype == PG_DTYPE_F32 ? run<float>(a, s) : run<__nv_bfloat16>(a, s);
}

}  // namespace pg
