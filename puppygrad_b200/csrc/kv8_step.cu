// Attention over the 8-bit paged cache for few rows of a sequence (a step's single token, several guesses of one).
//
// Work: a tile is 8 or 16 rows that share a key / value head, i.e. (token, query head of the group) pairs; a unit is a tile times 64
// consecutive positions. All units of a call, in the order sequence, head, tile, position, are cut into equal contiguous shares,
// one for each CTA of a persistent grid, and a CTA's into one for each warp: every SM reads the same number of bytes whatever the
// lengths are. Parts of a tile that several warps share are merged by their CTA, those of several CTAs by the one that arrives
// last, in the order of the positions (the result does not hang on who that is).
//
// A unit: S^T = K Q^T and O^T += V^T P^T by m16n8k16 FP16 matrix instructions: 16 tokens (or head entries) as rows, 8 of the tile's
// rows as columns, codes turned into FP16 (exact) in registers. With the tokens as rows, a tile of 8 wastes nothing and costs half the
// instructions and accumulators of the other order. The k index of a product may be permuted as long as both operands agree: a
// lane takes 16 consecutive bytes of a key (4 k steps) and 16 consecutive tokens of a value row (values lie by head entry). Row r of
// score tile s is token 16 ((r % 8) / 2) + 4 s + 2 (r / 8) + r % 2, so that a transposition of 8x8 blocks (movmatrix) makes the
// weights the operand that goes with the values a lane holds.
//
// Softmax with the blocks' scales: the key scale multiplies the score, the value scale is part of the exponent, w = 2^(s log2 e +
// log2 scale_v - m), so that O = sum w code and the weights stay within [0, 1] however the scales differ; the denominator adds w /
// scale_v. m is the running maximum of that exponent, rounded up, less 15: FP16 holds up to 2^16, and what rounds to nothing at its lower end
// is then below 2^-40 of the largest. FP32 queries and their weights are pairs of FP16 numbers, two instructions into one accumulator: FP32
// grade. Rounding: BF16 queries are exact in FP16 after their row's scaling to [1, 2) (entries below 2^-17 of the largest: to 2^-25 of it), their weights
// round to FP16 (2^-11 of each).
//
// Bound by bytes: 31 us for 64 sequences with 32 query and 8 key / value heads of 128 (202 MB). Measured: 71 us, 135000 cycles, of which an SM is active
// 100000 on average, 126000 at most: equal shares end a quarter apart. Of its time an SM takes 4300 cycles until it asks for the first bytes (units
// counted, page table, scales) and 10000 to merge cut tiles; the 85000 in between are half as many again as HBM's rate would need, for a reason that is
// not established (schedulers issue in 32 of 100 cycles and wait for bytes, at the end for other warps). Two sequences of 131000 positions 68 us
// (41 by bytes), one of 777 10.9 us, 64 FP32 rows 81 us.
#include <algorithm>
#include <type_traits>

#include "kv8.cuh"

namespace pg {
namespace {

constexpr int UNIT = 64;  // positions
constexpr float LOWER = 0x1p-15f;  // 2^-WEIGHT_BITS: denominators are without that factor, which keeps them in FP32's range

// Bytes come through a ring of slots for every warp, 64 tokens times 64 head entries (4 KB) each, keys of a unit first, then its
// values: all but one are on their way while that one is worked on, 128 KB for an SM.
template <int DP, int NB>
struct Shape {
  static constexpr int KC = DP / 64;                                    // key slots (and value slots) of a unit
  static constexpr int WARPS = DP == 64 || (DP == 128 && NB == 1) ? 16 : 8;  // by registers
  static constexpr int THREADS = WARPS * 32;
  static constexpr int SLOT = 4096, SLOTS = WARPS == 16 ? 3 : 2 * KC + 1 < 6 ? 2 * KC + 1 : 6, AHEAD = SLOTS - 1;
  static constexpr int ROWS = 8 * NB, PART = ROWS * (DP + 2);
  static constexpr int SMEM = WARPS * SLOTS * SLOT;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {  // an 8x8 block of FP16
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Pieces of 64 positions that any row of a sequence sees: [0, keep) and [low, high).
struct Span {
  int keep, low, high;
  __device__ __forceinline__ int units() const { return keep + high - low; }
};
__device__ __forceinline__ Span span_of(const Kv8AttnArgs& a, int len, int n) {
  Span s;
  const int have = min(len, a.c.pages_per_seq << a.c.page_shift);
  s.high = (have + UNIT - 1) / UNIT;
  s.low = a.window > 0 ? min(max(len - n - a.window + 1, 0) / UNIT, s.high) : 0;
  s.keep = min((min(a.keep, have) + UNIT - 1) / UNIT, s.low);
  if (s.units() <= 0) s.high = s.low + 1;  // rows that see nothing still get their zeros
  return s;
}

// 16 bytes from global to shared memory, asynchronously; zeros where `live` is false (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t to, const uint8_t* from, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 shared16(uint32_t from) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
  return v;
}
// 16 consecutive values of a row, zeros from `dim` on (and where there is no row).
template <typename T>
struct Sixteen {
  uint4 w[sizeof(T)];
  __device__ __forceinline__ void load(const T* q, int d, int dim, bool wide) {
    if (wide) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); ++i) {
        constexpr int N = 16 / sizeof(T);
        w[i] = q && d + (i + 1) * N <= dim ? *reinterpret_cast<const uint4*>(q + d + i * N) : make_uint4(0, 0, 0, 0);
      }
    } else {
      union {
        uint4 u[sizeof(T)];
        T t[16];
      } x;
#pragma unroll
      for (int e = 0; e < 16; ++e) x.t[e] = q && d + e < dim ? q[d + e] : from_f32<T>(0.f);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); ++i) w[i] = x.u[i];
    }
  }
  __device__ __forceinline__ float2 two(int i) const {  // values 2 i and 2 i + 1
    const uint32_t r[4] = {w[i / (8 / sizeof(T))].x, w[i / (8 / sizeof(T))].y, w[i / (8 / sizeof(T))].z, w[i / (8 / sizeof(T))].w};
    if (sizeof(T) == 4) return make_float2(__uint_as_float(r[2 * (i & 1)]), __uint_as_float(r[2 * (i & 1) + 1]));
    return make_float2(__uint_as_float(r[i & 3] << 16), __uint_as_float(r[i & 3] & 0xFFFF0000u));
  }
};

// A tile of rows, and where its units lie among all units.
struct Tile {
  int b, head, row0, rows, first_row, n_rows, len, have, first_unit, units;
  Span span;
};
// Equal shares of the units: share i begins at floor(i * units / n), without 64-bit divisions. Shares of equal tiles begin where
// tiles do if n is a multiple of their number.
struct Shares {
  int units, n, each, more;
  __device__ __forceinline__ Shares(int u, int k) : units(u), n(k), each(u / k), more(u - u / k * k) {}
  __device__ __forceinline__ int begin(int i) const { return i * each + i * more / n; }
  __device__ __forceinline__ int of(int u) const {
    int i = min((int)(((float)u + 0.5f) / (float)units * (float)n), n - 1);
#pragma unroll 1
    while (begin(i) > u) --i;
#pragma unroll 1
    while (i + 1 < n && begin(i + 1) <= u) ++i;
    return i;
  }
};

template <int DP, typename T, int NB>
__global__ void __launch_bounds__(Shape<DP, NB>::THREADS, 1) kv8_step_kernel(Kv8AttnArgs a) {
  constexpr bool PAIR = std::is_same<T, float>::value;
  using S = Shape<DP, NB>;
  constexpr int WARPS = S::WARPS, THREADS = S::THREADS, ROWS = S::ROWS, PART = S::PART, KC = S::KC, SLOT = S::SLOT, AHEAD = S::AHEAD, MT = DP / 16;
  static_assert(PART * 4 <= S::SLOTS * SLOT, "a warp's last part takes the place of its ring");
  static_assert(AHEAD <= 2 * KC, "the ring reaches into the next unit at most");
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int scan[THREADS];  // units of the sequences up to thread t's last
  __shared__ int wsum[WARPS];
  __shared__ int part_tile[WARPS * 2];  // first unit of the tile that a part belongs to, -1: none
  __shared__ Tile part_of_tile[WARPS * 2];
  __shared__ float factor[ROWS][KV8_MAX_CTAS], row_max[ROWS], row_sum[ROWS];
  __shared__ int last_here;

  const Kv8View& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, cc = lane & 3;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem + warp * S::SLOTS * SLOT) + lane * 16;  // this lane's 16 bytes of every 512
  // parts: a warp's last one in its ring, one before it (of another tile) in global memory
  auto last_part = [&](int w) { return reinterpret_cast<float*>(smem + w * S::SLOTS * SLOT); };
  float* const warp_parts = a.partials + (size_t)gridDim.x * 2 * PART;
  auto early_part = [&](int w) { return warp_parts + ((size_t)blockIdx.x * WARPS + w) * PART; };

  // ---- units of every sequence, summed up: thread t has sequences per * t and following
  auto tiles_of = [&](int n) { return (n * a.group + ROWS - 1) / ROWS; };
  auto units_of = [&](int b) {
    const int n = seq_rows(a.row_start, a.rows, b).n;
    return n && (int64_t)n * a.group <= a.step_rows ? tiles_of(n) * c.kv_heads * span_of(a, max(a.lens[b], 0), n).units() : 0;
  };
  grid_dep_launch();
  grid_dep_wait();
  // the page table will be asked for as soon as the lengths are known
#pragma unroll 1
  for (int64_t i = (int64_t)tid * 32; i < (int64_t)c.seqs * c.pages_per_seq && i < THREADS * 32; i += THREADS * 32)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(c.table + i));
  const int per = c.seqs <= THREADS ? 1 : (c.seqs + THREADS - 1) / THREADS;
  {
    int sum = 0;
    bool disorder = false;
#pragma unroll 1
    for (int b = tid * per; b < min(tid * per + per, c.seqs); ++b) {
      sum += units_of(b);
      disorder |= a.row_start && a.row_start[b + 1] < a.row_start[b];
    }
    int up = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(ALL_LANES, up, o);
      if (lane >= o) up += v;
    }
    if (lane == 31) wsum[warp] = up;
    scan[tid] = up;
    if (tid < WARPS * 2) part_tile[tid] = -1;
    // rows of two sequences at once would make more units than can be numbered
    if (__syncthreads_or(disorder)) return;
  }
  int total = lane < WARPS ? wsum[lane] : 0;  // lane i: units up to those of warp i's threads
#pragma unroll
  for (int o = 1; o < WARPS; o <<= 1) {
    const int v = __shfl_up_sync(ALL_LANES, total, o);
    if (lane >= o) total += v;
  }
  const int units = __shfl_sync(ALL_LANES, total, WARPS - 1);
  if (units == 0) return;
  // no more CTAs than give each warp a unit; for a single sequence a number that lets CTAs begin where tiles do
  int ctas = min((int)gridDim.x, (units + WARPS - 1) / WARPS);
  if (c.seqs == 1) {
    const int tiles = tiles_of(seq_rows(a.row_start, a.rows, 0).n) * c.kv_heads;
    if (tiles <= (int)gridDim.x) ctas = min((int)gridDim.x / tiles, (units / tiles + WARPS - 1) / WARPS) * tiles;
  }
  if ((int)blockIdx.x >= ctas) return;
  const Shares shares(units, ctas);
  const int c0 = shares.begin(blockIdx.x), c1 = shares.begin(blockIdx.x + 1);
  const int u0 = c0 + (c1 - c0) * warp / WARPS, u1 = c0 + (c1 - c0) * (warp + 1) / WARPS;

  auto tile_at = [&](int u) {  // by the whole warp
    const int w = __ffs(__ballot_sync(ALL_LANES, lane < WARPS && total > u)) - 1;
    int before = w ? __shfl_sync(ALL_LANES, total, w - 1) : 0;
    const int up = scan[w * 32 + lane];
    const int i = __ffs(__ballot_sync(ALL_LANES, before + up > u)) - 1;
    if (i) before += __shfl_sync(ALL_LANES, up, i - 1);
    Tile t;
    t.b = (w * 32 + i) * per;
#pragma unroll 1
    for (int k = 1; k < per; ++k) {
      const int n = units_of(t.b);
      if (before + n > u) break;
      before += n;
      ++t.b;
    }
    const SeqRows r = seq_rows(a.row_start, a.rows, t.b);
    t.first_row = r.first;
    t.n_rows = r.n;
    t.len = max(a.lens[t.b], 0);
    t.have = min(t.len, c.pages_per_seq << c.page_shift);
    t.span = span_of(a, t.len, r.n);
    t.units = t.span.units();
    const int tiles = tiles_of(r.n), x = (u - before) / t.units;
    t.first_unit = before + x * t.units;
    t.head = tiles == 1 ? x : x / tiles;
    const int tile = x - t.head * tiles;
    t.row0 = tile * ROWS;
    t.rows = min(ROWS, r.n * a.group - t.row0);
    return t;
  };
  auto start_of = [&](const Span& s, int x) { return (x < s.keep ? x : s.low + x - s.keep) * UNIT; };

  const size_t block = (size_t)DP << c.page_shift;
#pragma unroll 1
  for (int u = u0; u < u1;) {
    const Tile t = tile_at(u);
    const int x0 = u - t.first_unit, x1 = min(t.units, x0 + (u1 - u));
    // ---- fetching runs AHEAD slots in front of computing, and the look-up of a unit's pages a unit in front of that
    struct Source {
      const uint8_t *k, *v;  // of this lane's first 16 bytes
      bool k_live, v_live;
      int page;      // of this lane's scores: tokens 16 (g / 2) and following
      float2 scale;  // of that page: keys, values
    };
    int fx = x0, f_page = -1;  // next unit to fetch, its page
    auto look_up = [&] {
      const int tok = start_of(t.span, fx) + (g >> 1) * 16;
      f_page = fx < x1 && tok < t.have ? c.table[(size_t)t.b * c.pages_per_seq + (tok >> c.page_shift)] : -1;
    };
    auto next_source = [&](Source& s) {
      const int f_t0 = start_of(t.span, fx), mask = c.page_tokens - 1;
      s.page = (unsigned)f_page < (unsigned)c.n_pages ? f_page : -1;
      const int page_v = __shfl_sync(ALL_LANES, s.page, cc * 8);  // of the values: tokens 16 cc and following
      s.k = c.pool + ((size_t)max(s.page, 0) * c.kv_heads + t.head) * 2 * block + (size_t)(((f_t0 + (g >> 1) * 16) & mask) + (g & 1)) * DP + cc * 16;
      s.v = c.pool + (((size_t)max(page_v, 0) * c.kv_heads + t.head) * 2 + 1) * block + ((f_t0 + cc * 16) & mask) + ((size_t)g << c.page_shift);
      s.k_live = s.page >= 0;
      s.v_live = page_v >= 0;
      s.scale = make_float2(0.f, 1.f);
      if (s.k_live) s.scale = *reinterpret_cast<const float2*>(c.scales + ((size_t)s.page * c.kv_heads + t.head) * 2);
      ++fx;
      look_up();
    };
    int wr = 0, rd = 0;  // ring positions, in bytes
    auto fetch = [&](const Source& s, int i) {  // slot i of a unit
      const uint32_t to = ring + wr;
      wr = wr == (S::SLOTS - 1) * SLOT ? 0 : wr + SLOT;
      if (i < KC) {
#pragma unroll
        for (int j = 0; j < 8; ++j) copy16(to + j * 512, s.k + 2 * j * DP + i * 64, s.k_live);
      } else {
        const uint8_t* from = s.v + ((size_t)((i - KC) * 64) << c.page_shift);
#pragma unroll
        for (int j = 0; j < 8; ++j) copy16(to + j * 512, from + ((j * 8) << c.page_shift), s.v_live);
      }
    };
    Source cur, nxt;
    look_up();
    next_source(cur);
    nxt = cur;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      fetch(cur, i);
      copy_commit();
    }
    // ---- queries: lane (g, cc) takes row g; behind the first keys and values, which take longer
    const bool wide = (((uintptr_t)a.q | (uintptr_t)(a.q_row * sizeof(T)) | (uintptr_t)(c.dim * sizeof(T))) & 15) == 0;
    Sixteen<T> raw[NB][KC];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int x = t.row0 + n * 8 + g, r = t.n_rows == 1 ? 0 : x / a.group;
      const T* q = n * 8 + g < t.rows ? (const T*)a.q + (size_t)(t.first_row + r) * a.q_row + (size_t)(t.head * a.group + (x - r * a.group)) * c.dim : nullptr;
#pragma unroll
      for (int i = 0; i < KC; ++i) raw[n][i].load(q, i * 64 + cc * 16, c.dim, wide);
    }
    auto pos_of = [&](int i) { return t.n_rows == 1 ? t.len - 1 : t.len - t.n_rows + (t.row0 + min(i, t.rows - 1)) / a.group; };
    const int pos_low = pos_of(0), pos_high = pos_of(t.rows - 1);
    int pos[NB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) pos[n][e] = pos_of(n * 8 + cc * 2 + e);

    // ---- queries as the column operand, each row scaled by a power of two to [1, 2)
    uint32_t qh[NB][MT][2], ql[PAIR ? NB : 1][PAIR ? MT : 1][2];
    float back[NB][2];  // what brings the products of rows 2 cc and 2 cc + 1 back, times scale log2 e
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < KC; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 v = raw[n][i].two(e);
          m = fmaxf(m, fmaxf(fabsf(v.x), fabsf(v.y)));
        }
      m = fmaxf(m, __shfl_xor_sync(ALL_LANES, m, 1));
      m = fmaxf(m, __shfl_xor_sync(ALL_LANES, m, 2));
      // exponents within +-126 keep both the factor and its inverse normal numbers, and the largest entry, 2^128, below 4
      const int ex = min(max((int)(__float_as_uint(m) >> 23) - 127, -126), 126);
      // the sign of the score's factor goes to the queries, so that the largest product is the largest score
      const float f = copysignf(__uint_as_float((uint32_t)(127 - ex) << 23), a.scale);
      const float b = fabsf(a.scale) * 1.4426950408889634f * __uint_as_float((uint32_t)(127 + ex) << 23);
      back[n][0] = __shfl_sync(ALL_LANES, b, cc * 8);
      back[n][1] = __shfl_sync(ALL_LANES, b, cc * 8 + 4);
#pragma unroll
      for (int i = 0; i < KC; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 v = raw[n][i].two(e);
          const uint32_t h = pack_f16(v.x * f, v.y * f);
          qh[n][i * 4 + e / 2][e & 1] = h;
          if constexpr (PAIR) {
            const float2 r = unpack_f16(h);
            ql[n][i * 4 + e / 2][e & 1] = pack_f16(v.x * f - r.x, v.y * f - r.y);
          }
        }
    }

    float o[MT][NB][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][n][e] = 0.f;
    float m[NB][2], l[NB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;

#pragma unroll 1
    for (int x = x0; x < x1; ++x, ++u) {
      const int t0 = start_of(t.span, x), tok = t0 + (g >> 1) * 16 + (g & 1);  // this lane's scores: tok + 2 j, j = 0..7
      // waits for slot i, has the one AHEAD of it sent for, and gives its place
      auto slot = [&](int i) {
        copy_wait<AHEAD - 1>();
        const uint32_t from = ring + rd;
        rd = rd == (S::SLOTS - 1) * SLOT ? 0 : rd + SLOT;
        const int k = i + AHEAD;
        if (k < 2 * KC) {
          fetch(cur, k);
        } else {
          if (x + 1 < x1) {
            if (k == 2 * KC) next_source(nxt);
            fetch(nxt, k - 2 * KC);
          }
        }
        copy_commit();
        return from;
      };
      float s[4][NB][4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][n][e] = 0.f;
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const uint32_t from = slot(i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // tokens of rows r and r + 8: key rows 2 j and 2 j + 1 of the lane
          const uint4 k0 = shared16(from + 2 * j * 512), k1 = shared16(from + (2 * j + 1) * 512);
          const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
          uint32_t f[4][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f[e][0] = e4m3x2_to_f16x2(w0[e] & 0xFFFFu);
            f[e][1] = e4m3x2_to_f16x2(w1[e] & 0xFFFFu);
            f[e][2] = e4m3x2_to_f16x2(w0[e] >> 16);
            f[e][3] = e4m3x2_to_f16x2(w1[e] >> 16);
          }
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            if constexpr (PAIR) {  // the rests first, and the sum in registers: the instruction cuts off what it adds
              float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int e = 0; e < 4; ++e) mma_f16(d, f[e][0], f[e][1], f[e][2], f[e][3], ql[n][i * 4 + e][0], ql[n][i * 4 + e][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e) mma_f16(d, f[e][0], f[e][1], f[e][2], f[e][3], qh[n][i * 4 + e][0], qh[n][i * 4 + e][1]);
#pragma unroll
              for (int e = 0; e < 4; ++e) s[j][n][e] += d[e];
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) mma_f16(s[j][n], f[e][0], f[e][1], f[e][2], f[e][3], qh[n][i * 4 + e][0], qh[n][i * 4 + e][1]);
            }
          }
        }
      }
      // ---- exponents; masked ones are -infinity whatever the bytes were
      const float sv = fmaxf(cur.scale.y, 7.888609e-31f);  // 2^-100, the least scale that an append writes
      const bool odd = cur.scale.y != cur.scale.y;
      const float ev = odd ? cur.scale.y : __log2f(sv), inv_v = odd ? 1.f : LOWER / sv;
      const bool whole = __all_sync(ALL_LANES, cur.page >= 0) && t0 + UNIT - 1 <= pos_low && t0 + UNIT <= t.have &&
                         (a.window == 0 || t0 > pos_high - a.window || t0 + UNIT <= a.keep);
      uint32_t ph[NB][8], pl[PAIR ? NB : 1][8];
      float down[NB][2];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float f0 = back[n][0] * cur.scale.x, f1 = back[n][1] * cur.scale.x, add = ev;
        if (!whole) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int k = tok + 4 * j + (e & 2), p = pos[n][e & 1];
              const bool seen = cur.page >= 0 && k <= p && k < t.have && (a.window == 0 || k > p - a.window || k < a.keep);
              s[j][n][e] = seen ? fmaf(s[j][n][e], e & 1 ? f1 : f0, ev) : -INFINITY;
            }
          f0 = f1 = 1.f;
          add = 0.f;
        }
        // ---- running maximum and denominator; the maximum rounded up to a whole number, so that less the blocks' exponents it is exact
        float raw[2] = {fmaxf(s[0][n][0], s[0][n][2]), fmaxf(s[0][n][1], s[0][n][3])};
#pragma unroll
        for (int j = 1; j < 4; ++j) {
          raw[0] = fmaxf(raw[0], fmaxf(s[j][n][0], s[j][n][2]));
          raw[1] = fmaxf(raw[1], fmaxf(s[j][n][1], s[j][n][3]));
        }
        float top[2] = {fmaxf(m[n][0], ceilf(__fmaf_ru(raw[0], f0, add))), fmaxf(m[n][1], ceilf(__fmaf_ru(raw[1], f1, add)))};
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          top[0] = fmaxf(top[0], __shfl_xor_sync(ALL_LANES, top[0], off));
          top[1] = fmaxf(top[1], __shfl_xor_sync(ALL_LANES, top[1], off));
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float base = top[e] == -INFINITY ? 0.f : top[e];
          down[n][e] = ex2(m[n][e] - base);
          m[n][e] = top[e];
          top[e] = __fadd_rd(__fsub_rd(add, base), WEIGHT_BITS);
        }
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[j][n][e] = ex2(fmaf(s[j][n][e], e & 1 ? f1 : f0, top[e & 1]));
            sum[e & 1] += s[j][n][e];
          }
          const uint32_t h0 = pack_f16(s[j][n][0], s[j][n][1]), h1 = pack_f16(s[j][n][2], s[j][n][3]);
          ph[n][2 * j] = transposed(h0);
          ph[n][2 * j + 1] = transposed(h1);
          if constexpr (PAIR) {
            const float2 r0 = unpack_f16(h0), r1 = unpack_f16(h1);
            pl[n][2 * j] = transposed(pack_f16(s[j][n][0] - r0.x, s[j][n][1] - r0.y));
            pl[n][2 * j + 1] = transposed(pack_f16(s[j][n][2] - r1.x, s[j][n][3] - r1.y));
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) l[n][e] = fmaf(sum[e], inv_v, l[n][e] * down[n][e]);
      }
      // bytes behind the sequence's end may be anything, and 0 times NaN is NaN
      const int live = t.have - t0 - cc * 16;
      const bool cut = !whole && live < 16;
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        const uint32_t from = slot(KC + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // head entries of rows r and r + 8
          uint4 v0 = shared16(from + 2 * j * 512), v1 = shared16(from + (2 * j + 1) * 512);
          if (cut) {
            auto keep_bytes = [&](uint32_t& w, int k) { w = live >= k + 4 ? w : live <= k ? 0u : w & ((1u << 8 * (live - k)) - 1); };
            keep_bytes(v0.x, 0); keep_bytes(v0.y, 4); keep_bytes(v0.z, 8); keep_bytes(v0.w, 12);
            keep_bytes(v1.x, 0); keep_bytes(v1.y, 4); keep_bytes(v1.z, 8); keep_bytes(v1.w, 12);
          }
          const uint32_t w0[4] = {v0.x, v0.y, v0.z, v0.w}, w1[4] = {v1.x, v1.y, v1.z, v1.w};
          uint32_t f[4][4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f[e][0] = e4m3x2_to_f16x2(w0[e] & 0xFFFFu);
            f[e][1] = e4m3x2_to_f16x2(w1[e] & 0xFFFFu);
            f[e][2] = e4m3x2_to_f16x2(w0[e] >> 16);
            f[e][3] = e4m3x2_to_f16x2(w1[e] >> 16);
          }
#pragma unroll
          for (int n = 0; n < NB; ++n) {  // a unit's sums start from zero and join the others in registers
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            if constexpr (PAIR) {
#pragma unroll
              for (int e = 0; e < 4; ++e) mma_f16(d, f[e][0], f[e][1], f[e][2], f[e][3], pl[n][2 * e], pl[n][2 * e + 1]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) mma_f16(d, f[e][0], f[e][1], f[e][2], f[e][3], ph[n][2 * e], ph[n][2 * e + 1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i * 4 + j][n][e] = fmaf(o[i * 4 + j][n][e], down[n][e & 1], d[e]);
          }
        }
      }
      cur = nxt;
    }
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[n][e] += __shfl_xor_sync(ALL_LANES, l[n][e], off);

    // ---- a tile that is complete goes out, a part of one waits for the others
    if (x0 == 0 && x1 == t.units) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = n * 8 + cc * 2 + e, x = t.row0 + row, r = t.n_rows == 1 ? 0 : x / a.group;
          if (row >= t.rows) continue;
          T* to = (T*)a.out + (size_t)(t.first_row + r) * a.out_row + (size_t)(t.head * a.group + (x - r * a.group)) * c.dim;
          const float f = l[n][e] == 0.f ? 0.f : LOWER / l[n][e];
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            if (16 * i + g < c.dim) to[16 * i + g] = from_f32<T>(o[i][n][e] * f);
            if (16 * i + g + 8 < c.dim) to[16 * i + g + 8] = from_f32<T>(o[i][n][e + 2] * f);
          }
        }
    } else {
      __syncwarp();  // all lanes have read their last bytes of the ring
      float* w = u == u1 ? last_part(warp) : early_part(warp);
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = n * 8 + cc * 2 + e;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            w[row * DP + 16 * i + g] = o[i][n][e];
            w[row * DP + 16 * i + g + 8] = o[i][n][e + 2];
          }
          if (g == 0) {
            w[ROWS * DP + row] = m[n][e];
            w[ROWS * (DP + 1) + row] = l[n][e];
          }
        }
      if (lane == 0) {
        part_tile[warp * 2 + (u == u1 ? 1 : 0)] = t.first_unit;
        part_of_tile[warp * 2 + (u == u1 ? 1 : 0)] = t;
      }
    }
    copy_wait<0>();  // (nothing but empty groups)
  }
  __syncthreads();  // parts in global memory too are read by this block alone

  auto put = [&](const Tile& t, int i, int d, const float4& v, float l) {
    const int x = t.row0 + i, r = t.n_rows == 1 ? 0 : x / a.group;
    T* to = (T*)a.out + (size_t)(t.first_row + r) * a.out_row + (size_t)(t.head * a.group + (x - r * a.group)) * c.dim + d;
    const float f = l == 0.f ? 0.f : LOWER / l;
    const float w[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < c.dim) to[e] = from_f32<T>(w[e]);
  };
  auto add_part = [](float4& v, const float4& p, float f) {
    v.x = fmaf(p.x, f, v.x);
    v.y = fmaf(p.y, f, v.y);
    v.z = fmaf(p.z, f, v.z);
    v.w = fmaf(p.w, f, v.w);
  };
  // ---- parts of this CTA's warps, tile by tile; they are in the order of the positions
  const int id = lane < WARPS * 2 ? part_tile[lane] : -1;
  unsigned todo = __ballot_sync(ALL_LANES, id >= 0);
#pragma unroll 1
  while (todo) {
    const int at = __shfl_sync(ALL_LANES, id, __ffs(todo) - 1);
    const unsigned these = __ballot_sync(ALL_LANES, id == at);
    todo &= ~these;
    const Tile& t = part_of_tile[__ffs(these) - 1];
    const bool alone = at >= c0 && at + t.units <= c1;
    auto part = [&](int s) -> const float* { return s & 1 ? last_part(s >> 1) : early_part(s >> 1); };
    // a warp for a row, a lane for a part: the row's maximum, what each part is to be multiplied with, the denominator
#pragma unroll 1
    for (int row = warp; row < t.rows; row += WARPS) {
      const bool in = these >> lane & 1;
      const float* w = part(in ? lane : __ffs(these) - 1) + ROWS * DP + row;
      const float m = in ? w[0] : -INFINITY, top = lane_max(m), f = top == -INFINITY || !in ? 0.f : ex2(m - top);
      const float l = lane_sum(in ? w[ROWS] * f : 0.f);
      factor[row][lane] = f;
      if (lane == 0) row_max[row] = top, row_sum[row] = l;
    }
    __syncthreads();
    float* whole = a.partials + (size_t)(blockIdx.x * 2 + (at >= c0 ? 1 : 0)) * PART;
#pragma unroll 1
    for (int x = tid; x < t.rows * (DP / 4); x += THREADS) {
      const int row = x / (DP / 4), d = (x - row * (DP / 4)) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (unsigned rest = these; rest; rest &= rest - 1) {
        const int s = __ffs(rest) - 1;
        add_part(v, *reinterpret_cast<const float4*>(part(s) + row * DP + d), factor[row][s]);
      }
      if (alone) put(t, row, d, v, row_sum[row]);
      else __stcg(reinterpret_cast<float4*>(whole + row * DP + d), v);
    }
    if (!alone) {
      if (tid < t.rows) {
        __stcg(whole + ROWS * DP + tid, row_max[tid]);
        __stcg(whole + ROWS * (DP + 1) + tid, row_sum[tid]);
      }
      const int first_cta = shares.of(at), n = shares.of(at + t.units - 1) - first_cta + 1;  // CTAs that hold a part of the tile
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        // that of the CTA in which the tile begins; no other tile reaches from there into the next one
        unsigned* counter = a.counters + first_cta;
        const bool last = atomicAdd(counter, 1u) == (unsigned)(n - 1);
        if (last) *counter = 0;  // ready for the next call
        __threadfence();
        last_here = last;
      }
      __syncthreads();
      if (last_here) {
        // the tile begins in the first one's share, whose last tile it is, and before the others' shares
        auto part_of = [&](int i) { return a.partials + (size_t)((first_cta + i) * 2 + (i == 0 ? 1 : 0)) * PART; };
#pragma unroll 1
        for (int row = warp; row < t.rows; row += WARPS) {
          float top = -INFINITY, l = 0.f;
#pragma unroll 1
          for (int i = lane; i < n; i += 32) top = fmaxf(top, __ldcg(part_of(i) + ROWS * DP + row));
          top = lane_max(top);
#pragma unroll 1
          for (int i = lane; i < n; i += 32) {
            const float f = top == -INFINITY ? 0.f : ex2(__ldcg(part_of(i) + ROWS * DP + row) - top);
            l = fmaf(__ldcg(part_of(i) + ROWS * (DP + 1) + row), f, l);
            factor[row][i] = f;
          }
          l = lane_sum(l);
          if (lane == 0) row_sum[row] = l;
        }
        __syncthreads();
#pragma unroll 1
        for (int x = tid; x < t.rows * (DP / 4); x += THREADS) {
          const int row = x / (DP / 4), d = (x - row * (DP / 4)) * 4;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
          for (int i = 0; i < n; ++i) add_part(v, __ldcg(reinterpret_cast<const float4*>(part_of(i) + row * DP + d)), factor[row][i]);
          put(t, row, d, v, row_sum[row]);
        }
      }
    }
    __syncthreads();
  }
}

template <int DP, typename T, int NB>
cudaError_t run(const Kv8AttnArgs& a, int sms, cudaStream_t s) {
  using S = Shape<DP, NB>;
  return launch_kernel(kv8_step_kernel<DP, T, NB>, dim3(std::min(sms, KV8_MAX_CTAS)), dim3(S::THREADS), S::SMEM, s, true, a);
}
template <int DP, typename T, int NB>
cudaError_t allow() {
  return cudaFuncSetAttribute(kv8_step_kernel<DP, T, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DP, NB>::SMEM);
}
// Tiles of 16 rows read the cache once for what two tiles of 8 would read twice; where registers allow and there are more than 8. us
// with tiles of 16 / of 8: 64 sequences of 2000 positions, 8 heads of 128, 16 rows each 81 / 125, 32 rows 140 / 216; 12 heads of 64 84 / 108;
// one sequence of 8000, 32 rows 22 / 25 (12 heads of 64, 22 / 20).
template <typename T, int NB>
cudaError_t run_of(const Kv8AttnArgs& a, int sms, cudaStream_t s) {
  switch (kv8_padded(a.c.dim)) {
    case 64: return run<64, T, NB>(a, sms, s);
    case 128: return run<128, T, NB>(a, sms, s);
    case 192: return run<192, T, 1>(a, sms, s);
    default: return run<256, T, 1>(a, sms, s);
  }
}

}  // namespace

cudaError_t init_kv8_step_attributes() {
  cudaError_t all[] = {allow<64, float, 1>(), allow<128, float, 1>(), allow<192, float, 1>(), allow<256, float, 1>(), allow<64, __nv_bfloat16, 1>(),
                       allow<128, __nv_bfloat16, 1>(), allow<192, __nv_bfloat16, 1>(), allow<256, __nv_bfloat16, 1>(),
                       allow<64, __nv_bfloat16, 2>(), allow<128, __nv_bfloat16, 2>()};
  for (cudaError_t e : all)
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

cudaError_t launch_kv8_attention_step(const Kv8AttnArgs& a, int dtype, int sms, cudaStream_t s) {
  if (dtype == PG_DTYPE_F32) return run_of<float, 1>(a, sms, s);
  return (int64_t)a.group * a.max_rows > 8 ? run_of<__nv_bfloat16, 2>(a, sms, s) : run_of<__nv_bfloat16, 1>(a, sms, s);
}

}  // namespace pg
