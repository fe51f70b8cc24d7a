// Attention over the 8-bit paged cache for few rows of a sequence (a step's single token, several guesses of one).
//
// Work: a tile is up to 16 (FP32: 8) rows that share a key / value head, i.e. (token, query head of the group) pairs; a unit is a tile
// times 64 consecutive positions. All units of a call, in the order sequence, head, tile, position, are cut into equal contiguous
// shares, one for each CTA of a persistent grid, and a CTA's into one for each warp: every SM reads the same number of bytes whatever
// the lengths are. A tile that several warps share is put together in shared memory, one that several CTAs share by the CTA that
// arrives last, in the order of the positions (the result does not hang on who that is).
//
// A unit: S = Q K^T and O += P V by m16n8k16 FP16 matrix instructions, codes turned into FP16 (exact) in registers. The k index of a
// product may be permuted as long as both operands agree, so a lane takes 16 consecutive bytes of a key row (4 k steps) and 16
// consecutive tokens of a value row (values lie by head entry), and column n of score tile j stands for token 16 (n / 2) + 2 j +
// (n & 1): a lane's probabilities are then those of the tokens whose values it holds, and no data passes between lanes.
//
// Softmax with the blocks' scales: the key scale multiplies the score, the value scale is part of the exponent, w = 2^(s log2 e +
// log2 scale_v - m), so that O = sum w code and the weights stay within [0, 1] however the scales differ; the denominator adds w /
// scale_v. m is the running maximum of that exponent. FP32 queries: rows 0..7 of the instruction's tile hold the FP16 parts hi of
// q and of the weights, rows 8..15 the rests lo, their sums are added afterwards: FP32 grade at the price of one instruction.
// Rounding: BF16 queries are exact in FP16 after the row's scaling to [1, 2), their weights round to FP16 (2^-12 of the largest).
#include <type_traits>

#include "kv8.cuh"

namespace pg {
namespace {

constexpr int UNIT = 64;  // positions

template <int DP>
struct Shape {
  static constexpr int WARPS = DP <= 128 ? 8 : 4;  // partial tiles of all warps fit shared memory
  static constexpr int THREADS = WARPS * 32;
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Pieces of 64 positions that any row of a sequence sees: [0, keep) and [low, high).
struct Span {
  int keep, low, high;
  __device__ __forceinline__ int units() const { return keep + high - low; }
};
__device__ __forceinline__ Span span_of(const Kv8AttnArgs& a, int len, int n) {
  Span s;
  s.high = (min(len, a.c.pages_per_seq << a.c.page_shift) + UNIT - 1) / UNIT;
  s.low = a.window > 0 ? min(max(len - n - a.window + 1, 0) / UNIT, s.high) : 0;
  s.keep = min((min(a.keep, len) + UNIT - 1) / UNIT, s.low);
  if (s.units() <= 0) s.high = s.low + 1;  // rows that see nothing still get their zeros
  return s;
}

template <int DP, typename T>
__global__ void __launch_bounds__(Shape<DP>::THREADS) kv8_step_kernel(Kv8AttnArgs a) {
  constexpr bool PAIR = std::is_same<T, float>::value;
  constexpr int WARPS = Shape<DP>::WARPS, THREADS = Shape<DP>::THREADS, ROWS = PAIR ? 8 : 16, PART = ROWS * (DP + 2);
  constexpr int KC = DP / 64, NT = DP / 8;
  extern __shared__ __align__(16) uint8_t smem[];
  // [WARPS][DP / 16][32] uint4 queries, [WARPS][2][PART] floats, then the units' and the counters' prefix of the sequences
  uint4* qf = reinterpret_cast<uint4*>(smem) + (threadIdx.x >> 5) * (DP / 16) * 32;
  float* parts = reinterpret_cast<float*>(smem + WARPS * (DP / 16) * 512);
  int* unit_end = reinterpret_cast<int*>(parts + WARPS * 2 * PART);
  __shared__ int scan[Shape<DP>::THREADS];
  __shared__ int part_tile[WARPS * 2];  // counter of the tile that a partial belongs to, -1: none
  __shared__ int last_here;

  const Kv8View& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, cc = lane & 3;

  auto tiles_of = [&](const SeqRows& r) { return (r.n * a.group + ROWS - 1) / ROWS; };
  // ---- units of every sequence, summed up
  {
    const int per = (c.seqs + THREADS - 1) / THREADS, b0 = min(tid * per, c.seqs), b1 = min(b0 + per, c.seqs);
    int sum = 0;
    for (int b = b0; b < b1; ++b) {
      const SeqRows r = seq_rows(a.row_start, a.rows, b);
      if (r.n) sum += tiles_of(r) * c.kv_heads * span_of(a, max(a.lens[b], 0), r.n).units();
      unit_end[b] = sum;
    }
    scan[tid] = sum;
    __syncthreads();
    for (int o = 1; o < THREADS; o <<= 1) {
      const int v = tid >= o ? scan[tid - o] : 0;
      __syncthreads();
      scan[tid] += v;
      __syncthreads();
    }
    const int before = tid ? scan[tid - 1] : 0;
    for (int b = b0; b < b1; ++b) unit_end[b] += before;
    if (tid < WARPS * 2) part_tile[tid] = -1;
    __syncthreads();
  }
  const int units = unit_end[c.seqs - 1];
  const int ctas = min((int)gridDim.x, units);
  if ((int)blockIdx.x >= ctas) return;
  auto cta_begin = [&](int i) { return (int)((int64_t)units * i / ctas); };
  const int c0 = cta_begin(blockIdx.x), c1 = cta_begin(blockIdx.x + 1);
  const int u0 = c0 + (int)((int64_t)(c1 - c0) * warp / WARPS), u1 = c0 + (int)((int64_t)(c1 - c0) * (warp + 1) / WARPS);

  // writes one row of a finished tile: `value(d)` is the sum of weighted codes, `l` the denominator
  for (int u = u0; u < u1;) {
    // ---- the tile of unit u
    int lo = 0, hi = c.seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (unit_end[mid] > u) hi = mid;
      else lo = mid + 1;
    }
    const int b = lo;
    const SeqRows r = seq_rows(a.row_start, a.rows, b);
    const int len = max(a.lens[b], 0), have = min(len, c.pages_per_seq << c.page_shift);
    const Span span = span_of(a, len, r.n);
    const int n = span.units(), tiles = tiles_of(r);
    const int in_seq = u - (b ? unit_end[b - 1] : 0), tile_i = in_seq / n, x0 = in_seq - tile_i * n;
    const int head = tile_i / tiles, tile = tile_i - head * tiles;
    const int x1 = min(n, x0 + (u1 - u));
    const int row0 = tile * ROWS, rows = min(ROWS, r.n * a.group - row0);  // in (token, head of the group) pairs
    // positions of this lane's rows g and g + 8 (FP32: both halves are row g)
    auto pos_of = [&](int i) { return len - r.n + (row0 + min(i, rows - 1)) / a.group; };
    const int pos_a = pos_of(g), pos_b = PAIR ? pos_a : pos_of(g + 8);
    const int pos_low = pos_of(0), pos_high = pos_of(rows - 1);

    // ---- queries into fragments, each row scaled by a power of two to [1, 2)
    float fa, fb;  // what brings a row's product back, times scale log2 e
    {
      auto query = [&](int i) -> const T* {
        const int x = row0 + i, t = x / a.group;
        return (const T*)a.q + (size_t)(r.first + t) * a.q_row + (size_t)(head * a.group + (x - t * a.group)) * c.dim;
      };
      const T* qa = g < rows ? query(g) : nullptr;
      const T* qb = !PAIR && g + 8 < rows ? query(g + 8) : nullptr;
      auto at = [&](const T* q, int d) { return q && d < c.dim ? to_f32(q[d]) : 0.f; };
      float ma = 0.f, mb = 0.f;
      for (int d = cc; d < c.dim; d += 4) {
        ma = fmaxf(ma, fabsf(at(qa, d)));
        mb = fmaxf(mb, fabsf(at(qb, d)));
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        ma = fmaxf(ma, __shfl_xor_sync(ALL_LANES, ma, o));
        mb = fmaxf(mb, __shfl_xor_sync(ALL_LANES, mb, o));
      }
      // exponents within +-100 keep both the factor and its inverse normal numbers
      auto exponent = [](float m) { return min(max((int)(__float_as_uint(m) >> 23) - 127, -100), 100); };
      const int ea = exponent(ma), eb = exponent(mb);
      const float sa = __uint_as_float((uint32_t)(127 - ea) << 23), sb = __uint_as_float((uint32_t)(127 - eb) << 23);
      fa = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 + ea) << 23);
      fb = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 + eb) << 23);
      for (int i = 0; i < DP / 16; ++i) {
        const int d = (i >> 2) * 64 + cc * 16 + (i & 3) * 4;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = at(qa, d + e) * sa;
        uint4 f;
        f.x = pack_f16(v[0], v[1]);
        f.z = pack_f16(v[2], v[3]);
        if (PAIR) {
          const float2 p = __half22float2(*reinterpret_cast<__half2*>(&f.x)), q = __half22float2(*reinterpret_cast<__half2*>(&f.z));
          f.y = pack_f16(v[0] - p.x, v[1] - p.y);
          f.w = pack_f16(v[2] - q.x, v[3] - q.y);
        } else {
          f.y = pack_f16(at(qb, d) * sb, at(qb, d + 1) * sb);
          f.w = pack_f16(at(qb, d + 2) * sb, at(qb, d + 3) * sb);
        }
        qf[i * 32 + lane] = f;
      }
      __syncwarp();
    }

    float o[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;

    for (int x = x0; x < x1; ++x) {
      const int t0 = (x < span.keep ? x : span.low + x - span.keep) * UNIT;
      if (t0 > pos_high) break;  // later pieces are later positions: none of the tile's rows sees them
      // this lane's 16 tokens: their page and scales
      const int tok = t0 + cc * 16;
      const int page = tok < have ? page_of(c, b, tok >> c.page_shift) : -1;
      float ks = 0.f, ev = 0.f, inv_v = 1.f;
      if (page >= 0) {
        const float2 s = *reinterpret_cast<const float2*>(c.scales + ((size_t)page * c.kv_heads + head) * 2);
        ks = s.x;
        ev = __log2f(fmaxf(s.y, 7.888609e-31f));  // 2^-100, the least scale that an append writes
        inv_v = 1.f / fmaxf(s.y, 7.888609e-31f);
        if (s.y != s.y) ev = s.y, inv_v = 1.f;
      }
      const size_t block = (size_t)(DP << c.page_shift);
      const int page_k = __shfl_sync(ALL_LANES, page, g >> 1);  // of the keys that this lane loads: chunk g / 2
      const int off_k = ((t0 + (g >> 1) * 16) & (c.page_tokens - 1)) + (g & 1);
      const uint8_t* kp = c.pool + ((size_t)max(page_k, 0) * c.kv_heads + head) * 2 * block + (size_t)off_k * DP + cc * 16;
      const uint8_t* vp = c.pool + (((size_t)max(page, 0) * c.kv_heads + head) * 2 + 1) * block + (tok & (c.page_tokens - 1)) + ((size_t)g << c.page_shift);

      float s[8][4];
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        uint4 kv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) kv[j] = __ldg(reinterpret_cast<const uint4*>(kp + (size_t)2 * j * DP + i * 64));
        uint4 q[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = qf[(i * 4 + e) * 32 + lane];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t w[4] = {kv[j].x, kv[j].y, kv[j].z, kv[j].w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            mma_f16(s[j], q[e].x, q[e].y, q[e].z, q[e].w, e4m3x2_to_f16x2(w[e] & 0xFFFFu), e4m3x2_to_f16x2(w[e] >> 16));
        }
      }
      // ---- exponents; masked ones are -infinity whatever the bytes were
      const float xa = fa * ks, xb = fb * ks;
      const bool whole = __all_sync(ALL_LANES, page >= 0) && t0 + UNIT - 1 <= pos_low && t0 + UNIT <= have &&
                         (a.window == 0 || t0 > pos_high - a.window || t0 + UNIT <= a.keep);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (PAIR) {
          s[j][0] += s[j][2];
          s[j][1] += s[j][3];
        }
        s[j][0] = fmaf(s[j][0], xa, ev);
        s[j][1] = fmaf(s[j][1], xa, ev);
        s[j][2] = PAIR ? -INFINITY : fmaf(s[j][2], xb, ev);
        s[j][3] = PAIR ? -INFINITY : fmaf(s[j][3], xb, ev);
      }
      if (!whole) {
        auto seen = [&](int t, int pos) { return page >= 0 && t <= pos && t < have && (a.window == 0 || t > pos - a.window || t < a.keep); };
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int t = tok + 2 * j + e;
            if (!seen(t, pos_a)) s[j][e] = -INFINITY;
            if (!PAIR && !seen(t, pos_b)) s[j][2 + e] = -INFINITY;
          }
      }
      // ---- running maximum and denominator
      float na = m_a, nb = m_b;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        na = fmaxf(na, fmaxf(s[j][0], s[j][1]));
        nb = fmaxf(nb, fmaxf(s[j][2], s[j][3]));
      }
#pragma unroll
      for (int off = 1; off < 4; off <<= 1) {
        na = fmaxf(na, __shfl_xor_sync(ALL_LANES, na, off));
        nb = fmaxf(nb, __shfl_xor_sync(ALL_LANES, nb, off));
      }
      const float ua = na == -INFINITY ? 0.f : na, ub = nb == -INFINITY ? 0.f : nb;
      const float ra = ex2(m_a - ua), rb = ex2(m_b - ub);
      m_a = na;
      m_b = nb;
      float sum_a = 0.f, sum_b = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[j][0] = ex2(s[j][0] - ua);
        s[j][1] = ex2(s[j][1] - ua);
        sum_a += s[j][0] + s[j][1];
        if (!PAIR) {
          s[j][2] = ex2(s[j][2] - ub);
          s[j][3] = ex2(s[j][3] - ub);
          sum_b += s[j][2] + s[j][3];
        }
      }
      l_a = fmaf(sum_a, inv_v, l_a * ra);
      if (!PAIR) l_b = fmaf(sum_b, inv_v, l_b * rb);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        o[i][0] *= ra;
        o[i][1] *= ra;
        o[i][2] *= PAIR ? ra : rb;
        o[i][3] *= PAIR ? ra : rb;
      }
      uint32_t p[4][4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float *x = s[2 * e], *y = s[2 * e + 1];
        p[e][0] = pack_f16(x[0], x[1]);
        p[e][2] = pack_f16(y[0], y[1]);
        if (PAIR) {
          const float2 hx = __half22float2(*reinterpret_cast<__half2*>(&p[e][0])), hy = __half22float2(*reinterpret_cast<__half2*>(&p[e][2]));
          p[e][1] = pack_f16(x[0] - hx.x, x[1] - hx.y);
          p[e][3] = pack_f16(y[0] - hy.x, y[1] - hy.y);
        } else {
          p[e][1] = pack_f16(x[2], x[3]);
          p[e][3] = pack_f16(y[2], y[3]);
        }
      }
      // bytes behind the sequence's end may be anything, and 0 times NaN is NaN
      const int live = page >= 0 ? have - tok : 0;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        uint4 v = __ldg(reinterpret_cast<const uint4*>(vp + ((size_t)(8 * i) << c.page_shift)));
        if (!whole) {
          auto keep_bytes = [&](uint32_t w, int from) { return live >= from + 4 ? w : live <= from ? 0u : w & ((1u << 8 * (live - from)) - 1); };
          v.x = keep_bytes(v.x, 0);
          v.y = keep_bytes(v.y, 4);
          v.z = keep_bytes(v.z, 8);
          v.w = keep_bytes(v.w, 12);
        }
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          mma_f16(o[i], p[e][0], p[e][1], p[e][2], p[e][3], e4m3x2_to_f16x2(w[e] & 0xFFFFu), e4m3x2_to_f16x2(w[e] >> 16));
      }
    }
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
      l_a += __shfl_xor_sync(ALL_LANES, l_a, off);
      l_b += __shfl_xor_sync(ALL_LANES, l_b, off);
    }
    if (PAIR) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        o[i][0] += o[i][2];
        o[i][1] += o[i][3];
      }
    }

    // ---- a tile that is complete goes out, a part of one to shared memory
    if (x0 == 0 && x1 == n) {
      auto put = [&](int i, float l, float v0, float v1, int d) {
        if (i >= rows || d >= c.dim) return;
        const int x = row0 + i, t = x / a.group;
        T* to = (T*)a.out + (size_t)(r.first + t) * a.out_row + (size_t)(head * a.group + (x - t * a.group)) * c.dim + d;
        to[0] = from_f32<T>(l == 0.f ? 0.f : v0 / l);
        to[1] = from_f32<T>(l == 0.f ? 0.f : v1 / l);
      };
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        put(g, l_a, o[i][0], o[i][1], 8 * i + 2 * cc);
        if (!PAIR) put(g + 8, l_b, o[i][2], o[i][3], 8 * i + 2 * cc);
      }
    } else {
      const int slot = warp * 2 + (x0 == 0 ? 1 : 0);
      float* w = parts + slot * PART;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        *reinterpret_cast<float2*>(w + g * DP + 8 * i + 2 * cc) = make_float2(o[i][0], o[i][1]);
        if (!PAIR) *reinterpret_cast<float2*>(w + (g + 8) * DP + 8 * i + 2 * cc) = make_float2(o[i][2], o[i][3]);
      }
      if (cc == 0) {
        w[ROWS * DP + g] = m_a;
        w[ROWS * (DP + 1) + g] = l_a;
        if (!PAIR) {
          w[ROWS * DP + g + 8] = m_b;
          w[ROWS * (DP + 1) + g + 8] = l_b;
        }
      }
      // the first unit of the tile names it
      if (lane == 0) part_tile[slot] = u - x0;
    }
    u += x1 - x0;
    __syncwarp();
  }
  __syncthreads();

  // ---- parts of this CTA's warps, tile by tile; they are in the order of the positions
  for (int first = 0; first < WARPS * 2;) {
    const int at = part_tile[first];
    if (at < 0) {
      ++first;
      continue;
    }
    int end = first + 1;
    while (end < WARPS * 2 && (part_tile[end] < 0 || part_tile[end] == at)) ++end;
    int lo = 0, hi = c.seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (unit_end[mid] > at) hi = mid;
      else lo = mid + 1;
    }
    const int b = lo;
    const SeqRows r = seq_rows(a.row_start, a.rows, b);
    const Span span = span_of(a, max(a.lens[b], 0), r.n);
    const int n = span.units(), tiles = tiles_of(r), tile_i = (at - (b ? unit_end[b - 1] : 0)) / n;
    const int head = tile_i / tiles, tile = tile_i - head * tiles, row0 = tile * ROWS, rows = min(ROWS, r.n * a.group - row0);
    const bool alone = at >= c0 && at + n <= c1;
    auto put = [&](int i, int d, float l, float v) {
      const int x = row0 + i, t = x / a.group;
      T* to = (T*)a.out + (size_t)(r.first + t) * a.out_row + (size_t)(head * a.group + (x - t * a.group)) * c.dim + d;
      *to = from_f32<T>(l == 0.f ? 0.f : v / l);
    };
    float* mine = a.partials + (size_t)(blockIdx.x * 2 + (at >= c0 ? 1 : 0)) * PART;
    for (int x = tid; x < rows * DP; x += THREADS) {
      const int i = x / DP, d = x - i * DP;
      float m = -INFINITY, l = 0.f, v = 0.f;
      for (int s = first; s < end; ++s) {
        if (part_tile[s] < 0) continue;
        const float* w = parts + s * PART;
        m = fmaxf(m, w[ROWS * DP + i]);
      }
      for (int s = first; s < end; ++s) {
        if (part_tile[s] < 0) continue;
        const float* w = parts + s * PART;
        const float f = m == -INFINITY ? 0.f : ex2(w[ROWS * DP + i] - m);
        l = fmaf(w[ROWS * (DP + 1) + i], f, l);
        v = fmaf(w[i * DP + d], f, v);
      }
      if (alone) {
        if (d < c.dim) put(i, d, l, v);
      } else {
        __stcg(mine + i * DP + d, v);
        if (d == 0) {
          __stcg(mine + ROWS * DP + i, m);
          __stcg(mine + ROWS * (DP + 1) + i, l);
        }
      }
    }
    if (!alone) {
      // CTAs that hold a part of the tile: those of its first to its last unit
      const int first_cta = (int)((((int64_t)at + 1) * ctas - 1) / units), last_cta = (int)((((int64_t)at + n) * ctas - 1) / units);
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        unsigned* counter = a.counters + (size_t)((r.first * (int64_t)a.group / ROWS + b) + tile) * c.kv_heads + head;
        const bool last = atomicAdd(counter, 1u) == (unsigned)(last_cta - first_cta);
        if (last) *counter = 0;  // ready for the next call
        __threadfence();
        last_here = last;
      }
      __syncthreads();
      if (last_here) {
        auto part_of = [&](int i) { return a.partials + (size_t)(i * 2 + (at >= cta_begin(i) ? 1 : 0)) * PART; };
        for (int x = tid; x < rows * c.dim; x += THREADS) {
          const int i = x / c.dim, d = x - i * c.dim;
          float m = -INFINITY, l = 0.f, v = 0.f;
          for (int s = first_cta; s <= last_cta; ++s) m = fmaxf(m, __ldcg(part_of(s) + ROWS * DP + i));
          for (int s = first_cta; s <= last_cta; ++s) {
            const float* w = part_of(s);
            const float f = m == -INFINITY ? 0.f : ex2(__ldcg(w + ROWS * DP + i) - m);
            l = fmaf(__ldcg(w + ROWS * (DP + 1) + i), f, l);
            v = fmaf(__ldcg(w + i * DP + d), f, v);
          }
          put(i, d, l, v);
        }
      }
      __syncthreads();
    }
    first = end;
  }
}

template <int DP, typename T>
size_t step_smem(int seqs) {
  constexpr int WARPS = Shape<DP>::WARPS, ROWS = std::is_same<T, float>::value ? 8 : 16;
  return (size_t)WARPS * (DP / 16) * 512 + (size_t)WARPS * 2 * ROWS * (DP + 2) * 4 + (size_t)seqs * 4;
}

template <int DP, typename T>
cudaError_t run(const Kv8AttnArgs& a, int grid, cudaStream_t s) {
  return launch_kernel(kv8_step_kernel<DP, T>, dim3(grid), dim3(Shape<DP>::THREADS), step_smem<DP, T>(a.c.seqs), s, false, a);
}
template <int DP, typename T>
cudaError_t allow() {
  return cudaFuncSetAttribute(kv8_step_kernel<DP, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)step_smem<DP, T>(KV8_MAX_SEQS));
}
template <typename T>
cudaError_t run_of(const Kv8AttnArgs& a, int grid, cudaStream_t s) {
  switch (kv8_padded(a.c.dim)) {
    case 64: return run<64, T>(a, grid, s);
    case 128: return run<128, T>(a, grid, s);
    case 192: return run<192, T>(a, grid, s);
    default: return run<256, T>(a, grid, s);
  }
}

}  // namespace

cudaError_t init_kv8_step_attributes() {
  cudaError_t all[] = {allow<64, float>(), allow<128, float>(), allow<192, float>(), allow<256, float>(),
                       allow<64, __nv_bfloat16>(), allow<128, __nv_bfloat16>(), allow<192, __nv_bfloat16>(), allow<256, __nv_bfloat16>()};
  for (cudaError_t e : all)
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

cudaError_t launch_kv8_attention_step(const Kv8AttnArgs& a, int dtype, int sms, cudaStream_t s) {
  const int grid = sms < KV8_MAX_CTAS ? sms : KV8_MAX_CTAS;
  return dtype == PG_DTYPE_F32 ? run_of<float>(a, grid, s) : run_of<__nv_bfloat16>(a, grid, s);
}

}  // namespace pg
