// Attention over the 8-bit paged cache for sequences with many new rows: portions of prompts.
//
// A CTA has one or two tiles of 128 (token, query head of the group) rows that share a key / value head, and walks the pieces of 64
// positions that any of them sees. Both products are tcgen05 instructions on FP16 operands: S = Q K^T with both in shared memory, O += P V
// with P in tensor memory in the place of S and O in tensor memory. Producer warps load codes (sent for one piece ahead, in
// registers), turn them into FP16 (exact) and store them with the operands' 128-byte swizzle: keys lie by token, values by head entry,
// so both are K-major as they come. Four softmax warps for each tile have a row for every thread, which needs no exchange between
// threads; one warp issues the products, the scores of a piece in front of the values of the one before it, so that the tensor pipe
// works while the softmax of the next scores is computed. Two tiles share the producers' work at head_dim 128 (1500 rows behind 2600
// positions of two sequences, 32 query heads: 238 us, 282 us with one tile a CTA and two CTAs an SM); at 64 two CTAs with a tile each are
// better (1000 rows of four sequences, 12 heads: 42 us, 55 us), above 128 tensor memory has room for one.
// The instruction cuts off what it adds to O, up to 5*10^-8 of it each time, and always towards zero, so that sums of one sign drift: 4*10^-4 over 65536
// positions of FP32 rows. Theirs therefore join sums in memory (a place of the workspace for each CTA that is running) after every 32 pieces, by rounded
// additions, and O starts anew: within 10^-5 for 11% of the time (16 pieces: 3*10^-6, 14%). BF16 rows, with half as many
// products, drift by less than their result's rounding up to 10^6 positions and are left.
// Where the tiles are too few for the chip, each is cut along the positions (grid y); the parts, FP32 with their maxima and sums, are
// merged by a kernel of their own in the order of the positions.
//
// Scales, weights and the running maximum are those of the step kernel: the value scale is part of the exponent, the denominator
// divides it out. The maximum that weights refer to (a whole number: less the blocks' exponents it is exact) moves only when a row
// outgrows it by 2^3, which spares most passes over O; weights are up to 2^12 there, which leaves those to FP16's range. FP32 rows are pairs
// of FP16 numbers, queries and weights alike: two products into the same accumulator.
//
// Bound: 64 exponentials for every 64 * 2 * head_dim multiply-adds of a row keep the special-function and the tensor pipe equally busy at
// head_dim 128, 1024 cycles for 256 rows and 64 positions. Measured there: 2700 cycles. A softmax warp takes 400 for the maximum, 250 to
// get the scores, 1200 for exponentials, sums and stores, and two of them share a scheduler and its special functions; 0.6 PFLOP/s, 238 us
// for the portions above (384 CTAs, so that an SM is active for four fifths of it), 449 us with FP32 rows. Three producer warps are too few at 128 (321 us), seven no better than four (249 us);
// above 128 eight are better than four (head_dim 256, 1000 rows of four sequences: 158 us, 168 us).
#include <algorithm>
#include <type_traits>

#include "kv8.cuh"
#include "tc_common.cuh"

namespace pg {
namespace {

constexpr int ROWS = 128, TOKENS = 64, TILE_WARPS = 4;
constexpr float LAG = 3.f, LIFT = WEIGHT_BITS - LAG;  // a row's weights are up to 2^LIFT where its maximum is up to date
constexpr float LOWER = 0x1p-12f;                     // 2^-LIFT: denominators are without that factor, which keeps them in FP32's range
static_assert(LIFT == 12.f, "LOWER");

template <int DP, typename T>
struct PortionShape {
  static constexpr bool PAIR = std::is_same<T, float>::value;
  static constexpr int KC = DP / 64, TILES = DP == 128 ? 2 : 1;
  static constexpr int PRODUCER_WARPS = DP == 64 ? 3 : DP == 128 ? 4 : 8;  // (3: two CTAs of eight warps have 128 registers a thread)
  static constexpr int SOFTMAX_WARPS = TILES * TILE_WARPS, THREADS = (SOFTMAX_WARPS + 1 + PRODUCER_WARPS) * 32;
  static constexpr int TILE_QUERIES = (PAIR ? 2 : 1) * KC * 16384, QUERIES = TILES * TILE_QUERIES, HALF = KC * 8192, STAGE = 2 * HALF;  // bytes
  static constexpr int STAGES = QUERIES + 3 * STAGE <= (DP == 64 ? 100 : 192) * 1024 ? 3 : QUERIES + 2 * STAGE <= 192 * 1024 ? 2 : 1;
  static constexpr int SMEM = QUERIES + STAGES * STAGE + 1024;
  static constexpr int CTAS = DP == 64 ? 2 : 1;       // for an SM
  static constexpr int KEEP = 32;                     // pieces after which the sums of FP32 rows join those in memory
  static constexpr int PLACES = KV8_MAX_CTAS * CTAS;  // for those
  static_assert(TILES * ROWS * CTAS * (DP + 1) == kv8_held(DP) && PLACES <= KV8_PLACES, "the workspace");
  static constexpr int COLS = 512 / CTAS;  // tensor memory: for each tile O, then two places for scores and weights
  static_assert(TILES * (DP + 128) <= COLS, "tensor memory");
};

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// 64 columns of this warp's 32 rows.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&v)[64]) {
  uint32_t r[4][16];
#pragma unroll
  for (int i = 0; i < 4; ++i) tmem_ld16_issue(taddr + i * 16, r[i]);
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i >> 4][i & 15]);
}
__device__ __forceinline__ unsigned long long add_two(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// True in one lane of a converged warp; what the others compute beside it stays in uniform registers, which the products' operands need.
__device__ __forceinline__ bool elected() {
  uint32_t p;
  asm volatile("{\n.reg .pred q;\nelect.sync _|q, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, q;\n}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A warp's 32 rows of COLS sums out of tensor memory, times a factor for each, to rows of `dim` entries at to(row) (null: none). A thread has
// a row there, and neighbouring threads get neighbouring 16 bytes of one here: through shared memory (32 * COLS * sizeof(E) bytes). Where
// there are no sums (any = false) the rows get `fill`, and that memory, which may still be in use, is left alone. `held` (or null): more sums of this thread's
// row, a column every `step`, to be multiplied with f.
template <typename E, int COLS, typename F>
__device__ __forceinline__ void rows_out(uint8_t* mine, uint32_t taddr, bool any, float fill, const float* held, int step, float f, float by, int dim,
                                         bool wide, F to) {
  constexpr int PER = 16 / sizeof(E), VECS = COLS / PER;
  static_assert(VECS % 8 == 0, "places are swapped among eight");
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int d = 0; d < COLS && any; d += 16) {
    float o[16];
    tmem_ld16(taddr + d, o);
    if (held) {
#pragma unroll
      for (int e = 0; e < 16; ++e) o[e] = fmaf(__ldcg(held + (d + e) * step), f, o[e]);
    }
    union {
      uint4 u[16 / PER];
      E t[16];
    } x;
#pragma unroll
    for (int e = 0; e < 16; ++e) x.t[e] = from_f32<E>(o[e] * by);
#pragma unroll
    for (int k = 0; k < 16 / PER; ++k) *reinterpret_cast<uint4*>(mine + (lane * VECS + ((d / PER + k) ^ (lane & 7))) * 16) = x.u[k];
  }
  __syncwarp();
#pragma unroll 4
  for (int k = lane; k < 32 * VECS; k += 32) {  // (all lanes as often: to() may exchange)
    const int row = k / VECS, d = (k - row * VECS) * PER;
    E* p = to(row);
    if (!p) continue;
    union {
      uint4 u;
      E t[PER];
    } x;
    if (any) {
      x.u = *reinterpret_cast<const uint4*>(mine + (row * VECS + ((d / PER) ^ (row & 7))) * 16);
    } else {
#pragma unroll
      for (int e = 0; e < PER; ++e) x.t[e] = from_f32<E>(fill);
    }
    if (wide && d + PER <= dim) {
      *reinterpret_cast<uint4*>(p + d) = x.u;
    } else {
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (d + e < dim) p[d + e] = x.t[e];
    }
  }
  __syncwarp();
}

// Rows of one CTA (slot) and the pieces of 64 positions that they see: [0, kept) and [low, high). A sequence has the slots from
// floor(its first row * group / size) + its number on; the last rows, which see most, come first.
struct Portion {
  SeqRows r;
  int b, row0, rows, len, have, pos_low, pos_high, low, kept, pieces, parts;
  __device__ __forceinline__ Portion(const Kv8AttnArgs& a, int slot, int size, int most_parts) {
    const Kv8View& c = a.c;
    auto first_slot = [&](int s) { return (int)((int64_t)min(max(a.row_start[s], 0), a.rows) * a.group / size) + s; };
    int lo = 0, hi = c.seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first_slot(mid) <= slot) lo = mid;
      else hi = mid;
    }
    b = lo;
    r = seq_rows(a.row_start, a.rows, b);
    row0 = (slot - first_slot(b)) * size;
    rows = min(size, r.n * a.group - row0);
    if (row0 < 0 || r.n * a.group <= a.step_rows) rows = 0;  // none, or so few that the step kernel has them
    if (rows <= 0) return;
    len = max(a.lens[b], 0);
    have = min(len, c.pages_per_seq << c.page_shift);
    pos_low = len - r.n + row0 / a.group;
    pos_high = len - r.n + (row0 + rows - 1) / a.group;
    const int high = (max(min(pos_high + 1, have), 0) + TOKENS - 1) / TOKENS;
    low = a.window > 0 ? min(max(pos_low - a.window + 1, 0) / TOKENS, high) : 0;
    kept = min((min(a.keep, have) + TOKENS - 1) / TOKENS, low);
    pieces = kept + high - low;
    parts = max(1, min(most_parts, pieces / 4));  // not so many that a part is all beginning and end
  }
};

template <int DP, typename T>
__global__ void __launch_bounds__(PortionShape<DP, T>::THREADS, PortionShape<DP, T>::CTAS) kv8_portion_kernel(Kv8AttnArgs a, int slots) {
  using S = PortionShape<DP, T>;
  constexpr bool PAIR = S::PAIR;
  constexpr int KC = S::KC, STAGES = S::STAGES, TILES = S::TILES, SOFTMAX_WARPS = S::SOFTMAX_WARPS;
  constexpr int PRODUCERS = S::PRODUCER_WARPS * 32, COUNT = DP * 4, ITEMS = (COUNT + PRODUCERS - 1) / PRODUCERS;  // 16-byte items of keys (and of values): in all, for a thread
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t q_full[TILES], full[STAGES], empty[STAGES], s_full[TILES][2], p_full[TILES][2], o_done[TILES];
  __shared__ uint32_t tmem_slot;
  __shared__ int failed_flag, place;  // place: of this CTA's sums in memory
  __shared__ float4 info[STAGES][3];  // of a stage's four pieces of 16 tokens: key scale, log2 of the value scale, 2^-LIFT times its inverse
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* stages = base + S::QUERIES;
  volatile int* failed = &failed_flag;
  const Kv8View& c = a.c;
  const int tid = threadIdx.x, warp = __shfl_sync(ALL_LANES, tid >> 5, 0), lane = tid & 31;
  grid_dep_launch();
  grid_dep_wait();

  const int slot = slots - 1 - (int)(blockIdx.x / c.kv_heads), head = blockIdx.x % c.kv_heads;
  const Portion w(a, slot, TILES * ROWS, gridDim.y);
  if (w.rows <= 0 || (int)blockIdx.y >= w.parts) return;
  const int b = w.b, row0 = w.row0, rows = w.rows, len = w.len, have = w.have, pos_low = w.pos_low, pos_high = w.pos_high, low = w.low, kept = w.kept;
  const SeqRows r = w.r;
  // this CTA's pieces, numbered from 0
  const int first = w.pieces * (int)blockIdx.y / w.parts, pieces = w.pieces * ((int)blockIdx.y + 1) / w.parts - first;
  const int tiles = rows > ROWS ? TILES : 1;  // that have rows
  auto start_of = [&](int j) { return (first + j < kept ? first + j : low + first + j - kept) * TOKENS; };

  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], S::PRODUCER_WARPS);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < TILES; ++i) {
      mbar_init(&q_full[i], TILE_WARPS);
      mbar_init(&s_full[i][0], 1);
      mbar_init(&s_full[i][1], 1);
      mbar_init(&p_full[i][0], TILE_WARPS);
      mbar_init(&p_full[i][1], TILE_WARPS);
      mbar_init(&o_done[i], 1);
    }
    failed_flag = 0;
    place = -1;
    if (PAIR && pieces > S::KEEP) {
      // there are as many places as CTAs can run at once, so one is free
      for (int i = 0, p = blockIdx.x % S::PLACES; i < S::PLACES && place < 0; ++i, p = p + 1 == S::PLACES ? 0 : p + 1)
        if (atomicCAS(a.places + p, 0u, 1u) == 0u) place = p;
      __threadfence();
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == SOFTMAX_WARPS) tmem_alloc(&tmem_slot, S::COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  auto o_of = [&](int t) { return tmem + (uint32_t)(t * (DP + 128)); };
  bool ok = !PAIR || place >= 0 || pieces <= S::KEEP;

  if (warp < SOFTMAX_WARPS) {
    // ---- a row for every thread
    const int tile = warp / TILE_WARPS, in_tile = tid & (ROWS - 1);
    const bool used = tile < tiles;
    const int i = tile * ROWS + in_tile, own = row0 + min(i, rows - 1), tok = own / a.group, pos = len - r.n + tok;
    const int64_t entry = (int64_t)(head * a.group + own - tok * a.group) * c.dim;  // of the thread's own row, behind its token's first
    auto wide_of = [&](const void* p, int64_t row) {
      return (((uintptr_t)p | (uintptr_t)(row * (int64_t)sizeof(T)) | (uintptr_t)(c.dim * sizeof(T))) & 15) == 0;
    };
    const bool wide_rows = wide_of(a.q, a.q_row);
    const uint32_t lane_addr = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tmem_o = o_of(tile) + lane_addr, tmem_s = tmem_o + DP;
    float back = 0.f;
    if (used) {
      // a warp has 32 rows; neighbouring lanes take 8 entries each of the same one, so that it comes in whole lines
      constexpr int ACROSS = DP == 64 ? 8 : DP == 128 ? 16 : 32, AT_ONCE = 32 / ACROSS;  // lanes for a row, rows at a time
      const int u = lane % ACROSS;
      const int64_t from = (int64_t)(r.first + tok) * a.q_row + entry;
#pragma unroll 4
      for (int k = 0; k < 32; k += AT_ONCE) {
        const int row = (warp & 3) * 32 + k + lane / ACROSS;
        const T* q = (const T*)a.q + __shfl_sync(ALL_LANES, from, k + lane / ACROSS) + u * 8;
        float v[8], top = 0.f;
        if (wide_rows && u * 8 + 8 <= c.dim) {
          load8(q, v);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = u * 8 + e < c.dim ? to_f32(q[e]) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));
#pragma unroll
        for (int o = 1; o < ACROSS; o <<= 1) top = fmaxf(top, __shfl_xor_sync(ALL_LANES, top, o));
        // the sign of the score's factor goes to the queries, so that the largest product is the largest score
        // (exponents within +-126: both the factor and its inverse are normal numbers, and the largest entry, 2^128, becomes less than 4)
        const int ex = min(max((int)(__float_as_uint(top) >> 23) - 127, -126), 126);
        const float f = copysignf(__uint_as_float((uint32_t)(127 - ex) << 23), a.scale);
        const int mine = __shfl_sync(ALL_LANES, ex, lane % AT_ONCE * ACROSS);  // of this thread's own row
        if (k == lane / AT_ONCE * AT_ONCE) back = __uint_as_float((uint32_t)(127 + mine) << 23);
        if (u >= DP / 8) continue;
        uint8_t* to = base + tile * S::TILE_QUERIES + (u >> 3) * 16384 + row * 128 + (((u & 7) ^ (row & 7)) << 4);
        uint32_t h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          h[e] = pack_f16(v[2 * e] * f, v[2 * e + 1] * f);
          const float2 p = unpack_f16(h[e]);
          l[e] = pack_f16(v[2 * e] * f - p.x, v[2 * e + 1] * f - p.y);
        }
        *reinterpret_cast<uint4*>(to) = make_uint4(h[0], h[1], h[2], h[3]);
        if (PAIR) *reinterpret_cast<uint4*>(to + KC * 16384) = make_uint4(l[0], l[1], l[2], l[3]);
      }
      back = fabsf(a.scale) * 1.4426950408889634f * back;
      fence_async_proxy();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[tile]);
    }

    float m_ref = -INFINITY, sum = 0.f;
    // sums in memory, then the maximum that they refer to: [column][row], so that lanes are neighbours
    constexpr int NEXT = TILES * ROWS;
    auto held_at = [&] { return a.held + (size_t)max(place, 0) * (DP + 1) * NEXT + tile * ROWS + in_tile; };
    auto held_factor = [&](const float* held) {
      const float m = __ldcg(held + DP * NEXT);
      return m == -INFINITY ? 0.f : ex2(m - m_ref);
    };
    int stage = 0;
    for (int j = 0; j < pieces && used; ++j) {
      const uint32_t s_at = tmem_s + (uint32_t)(j & 1) * 64;
      ok = __all_sync(ALL_LANES, ok && mbar_wait(&s_full[tile][j & 1], (j >> 1) & 1, failed, nullptr, 0));
      if (!ok) break;
      tc_fence_after();
      const int t0 = start_of(j);
      const float4 k4 = info[stage][0], e4 = info[stage][1], i4 = info[stage][2];
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      float kf[4] = {k4.x * back, k4.y * back, k4.z * back, k4.w * back}, ev[4] = {e4.x, e4.y, e4.z, e4.w};
      const float inv[4] = {i4.x, i4.y, i4.z, i4.w};
      float v[64];
      tmem_ld64(s_at, v);
      if (!(t0 + TOKENS - 1 <= pos_low && t0 + TOKENS <= have && (a.window == 0 || t0 > pos_high - a.window || t0 + TOKENS <= a.keep))) {
        const int hi_i = min(pos, have - 1) - t0, lo_i = a.window > 0 ? pos - a.window + 1 - t0 : -1, keep_i = a.keep - t0;
#pragma unroll
        for (int e = 0; e < 64; ++e) {
          const bool hidden = e > hi_i || (e < lo_i && e >= keep_i);
          v[e] = hidden ? -INFINITY : fmaf(v[e], kf[e / 16], ev[e / 16]);  // whatever the scales are
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) kf[h] = 1.f, ev[h] = 0.f;
      }
      float t_max = -INFINITY;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        float m = fmaxf(v[h * 16], v[h * 16 + 1]);
#pragma unroll
        for (int e = 2; e < 16; e += 2) m = fmaxf(m, fmaxf(v[h * 16 + e], v[h * 16 + e + 1]));
        t_max = fmaxf(t_max, __fmaf_ru(m, kf[h], ev[h]));
      }
      if (__any_sync(ALL_LANES, t_max > __fadd_rd(m_ref, LAG))) {
        const float m_new = fmaxf(m_ref, ceilf(t_max)), corr = m_ref == -INFINITY ? 0.f : ex2(m_ref - m_new);
        m_ref = m_new;
        sum *= corr;
        if (j > 0) {
          ok = __all_sync(ALL_LANES, mbar_wait(&o_done[tile], (j - 1) & 1, failed, nullptr, 0));
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int d = 0; d < DP; d += 16) {
            float o[16];
            tmem_ld16(tmem_o + d, o);
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(o[e] * corr);
            tmem_st16(tmem_o + d, w);
          }
        }
      }
      const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const float b = __fadd_rd(__fsub_rd(ev[h], m_use), LIFT);
        const unsigned long long k2 = pack2(kf[h], kf[h]), b2 = pack2(b, b);
        unsigned long long part = pack2(0.f, 0.f);
        uint32_t hi16[8], lo16[8];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          float p0, p1;
          unpack2(fma2(pack2(v[h * 16 + e], v[h * 16 + e + 1]), k2, b2), p0, p1);
          p0 = ex2(p0);
          p1 = ex2(p1);
          part = add_two(part, pack2(p0, p1));
          hi16[e / 2] = pack_f16(p0, p1);
          if (PAIR) {
            const float2 p = unpack_f16(hi16[e / 2]);
            lo16[e / 2] = pack_f16(p0 - p.x, p1 - p.y);
          }
        }
        float a0, a1;
        unpack2(part, a0, a1);
        sum = fmaf(a0 + a1, inv[h], sum);
        // (the scores are in registers: any order of storing is fine)
        tmem_st8(s_at + (h >> 1) * 32 + (h & 1) * 8, hi16);
        if (PAIR) tmem_st8(s_at + (h >> 1) * 32 + 16 + (h & 1) * 8, lo16);
      }
      // each product is waited for before the next one can be issued: a wait by parity knows two phases apart no more (by now it is done)
      if (j > 0) ok = __all_sync(ALL_LANES, mbar_wait(&o_done[tile], (j - 1) & 1, failed, nullptr, 0));
      if (!ok) break;
      if (PAIR && j > 0 && j % S::KEEP == 0) {
        tc_fence_after();
        float* held = held_at();
        const float f = j == S::KEEP ? 0.f : held_factor(held);
#pragma unroll 1
        for (int d = 0; d < DP; d += 16) {
          float o[16], h[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) h[e] = j == S::KEEP ? 0.f : __ldcg(held + (d + e) * NEXT);
          tmem_ld16(tmem_o + d, o);
#pragma unroll
          for (int e = 0; e < 16; ++e) __stcg(held + (d + e) * NEXT, fmaf(h[e], f, o[e]));
        }
        __stcg(held + DP * NEXT, m_ref);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[tile][j & 1]);  // (two in turn: the next one's may come before this one is waited for)
    }
    if (ok && used && pieces > 0) ok = __all_sync(ALL_LANES, mbar_wait(&o_done[tile], (pieces - 1) & 1, failed, nullptr, 0));
    if (used) {
      tc_fence_after();
      const float fill = ok ? 0.f : __uint_as_float(0x7FC00000u);  // a wait ran out: no result, one that shows, and a word that says so
      if (!ok && lane == 0) atomicExch(a.status, 1u);
      sum += fill;
      uint8_t* mine = base + tile * S::TILE_QUERIES + (warp & 3) * (S::TILE_QUERIES / 4);  // the queries are not needed any more
      const int row_w = tile * ROWS + (warp & 3) * 32;  // the warp's first row
      const bool any = pieces > 0 && ok;
      const float* more = PAIR && pieces > S::KEEP && ok ? held_at() : nullptr;
      const float f = more ? held_factor(more) : 0.f;
      if (w.parts > 1) {
        float* to = a.partials + ((size_t)blockIdx.x * gridDim.y + blockIdx.y) * (TILES * ROWS) * (DP + 2);
        if (i < rows) *reinterpret_cast<float2*>(to + (size_t)TILES * ROWS * DP + 2 * i) = make_float2(m_ref, sum);
#pragma unroll 1
        for (int d = 0; d < DP; d += DP / 2)
          rows_out<float, DP / 2>(mine, tmem_o + d, any, fill, more ? more + d * NEXT : nullptr, NEXT, f, 1.f, DP / 2, true,
                                  [&](int k) { return row_w + k < rows ? to + (row_w + k) * DP + d : nullptr; });
      } else {
        const int64_t at = (int64_t)(r.first + tok) * a.out_row + entry;
        rows_out<T, DP>(mine, tmem_o, any, fill, more, NEXT, f, sum == 0.f ? 0.f : LOWER / sum, c.dim, wide_of(a.out, a.out_row), [&](int k) {
          T* p = (T*)a.out + __shfl_sync(ALL_LANES, at, k);
          return row_w + k < rows ? p : nullptr;
        });
      }
    }
    tc_fence_before();
  } else if (warp == SOFTMAX_WARPS) {
    // ---- products
    if (pieces > 0) {
      constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(TOKENS >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
      constexpr uint32_t idesc_o = (1u << 4) | ((uint32_t)(DP >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
      const uint64_t q_desc = umma_desc_sw128(base), kv_desc = umma_desc_sw128(stages);
      RingCursor ahead, now;  // the stage whose scores are next, and the one whose values are
      auto scores = [&](int j) {
        if (!__all_sync(ALL_LANES, mbar_wait(&full[ahead.stage], ahead.parity, failed, nullptr, 0))) return false;
        tc_fence_after();
        const uint64_t dk = kv_desc + ahead.stage * (S::STAGE >> 4);
        for (int t = 0; t < tiles; ++t) {
          const uint32_t to = o_of(t) + DP + (uint32_t)(j & 1) * 64;
          const uint64_t dq = q_desc + (uint32_t)t * (S::TILE_QUERIES >> 4);
          if (elected()) {
#pragma unroll
            for (int p = PAIR ? 1 : 0; p >= 0; --p)  // the rests first: the sums are cut off
#pragma unroll
              for (int k = 0; k < DP / 16; ++k)
                umma_bf16_ss(to, dq + (uint32_t)((p * KC + (k >> 2)) * (16384 >> 4) + (k & 3) * 2), dk + (uint32_t)((k >> 2) * (8192 >> 4) + (k & 3) * 2),
                             idesc_s, p != (PAIR ? 1 : 0) || k != 0);
            umma_commit(&s_full[t][j & 1]);
          }
          __syncwarp();
        }
        ahead.next(STAGES);
        return true;
      };
      for (int t = 0; t < tiles && ok; ++t) ok = __all_sync(ALL_LANES, mbar_wait(&q_full[t], 0, failed, nullptr, 0));
      if (ok && STAGES > 1) ok = scores(0);
      for (int j = 0; j < pieces && ok; ++j) {
        if (STAGES > 1) {
          if (j + 1 < pieces) ok = scores(j + 1);
        } else {
          ok = scores(j);
        }
        const uint64_t dv = kv_desc + (uint32_t)(now.stage * (S::STAGE >> 4) + (S::HALF >> 4));
        for (int t = 0; t < tiles && ok; ++t) {
          ok = __all_sync(ALL_LANES, mbar_wait(&p_full[t][j & 1], (j >> 1) & 1, failed, nullptr, 0));
          if (!ok) break;
          tc_fence_after();
          const uint32_t to = o_of(t), from = to + DP + (uint32_t)(j & 1) * 64;
          if (elected()) {
#pragma unroll
            for (int p = PAIR ? 1 : 0; p >= 0; --p)
#pragma unroll
              for (int k = 0; k < TOKENS / 16; ++k)
                umma_bf16_ts(to, from + (uint32_t)((k >> 1) * 32 + p * 16 + (k & 1) * 8), dv + (uint32_t)(k * 2), idesc_o,
                             (PAIR ? j % S::KEEP : j) != 0 || p != (PAIR ? 1 : 0) || k != 0);
            umma_commit(&o_done[t]);
            if (t == tiles - 1) umma_commit(&empty[now.stage]);
          }
          __syncwarp();
        }
        now.next(STAGES);
      }
    }
    __syncwarp();
  } else {
    // ---- producers: keys and values of a piece as FP16, one piece ahead in registers
    const int p_tid = tid - (SOFTMAX_WARPS + 1) * 32, mask = c.page_tokens - 1;
    const size_t block = (size_t)DP << c.page_shift;
    auto look_up = [&](int j) {  // the page of 16 tokens, of piece lane % 4
      if (j >= pieces) return -1;
      const int tok = start_of(j) + (lane & 3) * 16;
      return tok < have ? page_of(c, b, tok >> c.page_shift) : -1;
    };
    uint4 kr[ITEMS], vr[ITEMS];
    int page = look_up(0);
    float2 scale;
    auto load = [&](int j) {
      const int t0 = start_of(j);
      scale = make_float2(0.f, 0.f);
      if (page >= 0) scale = *reinterpret_cast<const float2*>(c.scales + ((size_t)page * c.kv_heads + head) * 2);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int idx = i * PRODUCERS + p_tid, t = idx / (DP / 16), d = (idx - t * (DP / 16)) * 16;
        const int pg_k = __shfl_sync(ALL_LANES, page, (t >> 4) & 3);
        kr[i] = make_uint4(0, 0, 0, 0);
        if (pg_k >= 0 && idx < COUNT)
          kr[i] = *reinterpret_cast<const uint4*>(c.pool + ((size_t)pg_k * c.kv_heads + head) * 2 * block + (size_t)((t0 + t) & mask) * DP + d);
      }
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int idx = i * PRODUCERS + p_tid;  // head entry idx / 4; piece idx % 4 = lane % 4: this lane's own page
        vr[i] = make_uint4(0, 0, 0, 0);
        if (page >= 0 && idx < COUNT)
          vr[i] = *reinterpret_cast<const uint4*>(c.pool + (((size_t)page * c.kv_heads + head) * 2 + 1) * block + ((size_t)(idx >> 2) << c.page_shift) +
                                                 ((t0 + (lane & 3) * 16) & mask));
      }
    };
    auto halves = [](const uint4& v, uint4& x, uint4& y) {
      x = make_uint4(e4m3x2_to_f16x2(v.x & 0xFFFFu), e4m3x2_to_f16x2(v.x >> 16), e4m3x2_to_f16x2(v.y & 0xFFFFu), e4m3x2_to_f16x2(v.y >> 16));
      y = make_uint4(e4m3x2_to_f16x2(v.z & 0xFFFFu), e4m3x2_to_f16x2(v.z >> 16), e4m3x2_to_f16x2(v.w & 0xFFFFu), e4m3x2_to_f16x2(v.w >> 16));
    };
    if (pieces > 0) load(0);
    RingCursor at;
    for (int j = 0; j < pieces; ++j, at.next(STAGES)) {
      const int next_page = look_up(j + 1), stage = at.stage;
      ok = __all_sync(ALL_LANES, ok && mbar_wait(&empty[stage], at.parity ^ 1, failed, nullptr, 0));
      if (!ok) break;
      uint8_t* ks = stages + stage * S::STAGE;
      uint8_t* vs = ks + S::HALF;
      const int live = have - (start_of(j) + (lane & 3) * 16);  // of this lane's 16 tokens of values; bytes behind them may be anything
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int idx = i * PRODUCERS + p_tid, t = idx / (DP / 16), u = idx - t * (DP / 16);
        if (idx >= COUNT) continue;
        uint4 x, y;
        halves(kr[i], x, y);
        uint8_t* to = ks + (u >> 2) * 8192 + t * 128;
        *reinterpret_cast<uint4*>(to + ((((u & 3) * 2) ^ (t & 7)) << 4)) = x;
        *reinterpret_cast<uint4*>(to + ((((u & 3) * 2 + 1) ^ (t & 7)) << 4)) = y;
      }
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int idx = i * PRODUCERS + p_tid, d = idx >> 2;
        if (idx >= COUNT) continue;
        if (live < 16) {
          auto keep_bytes = [&](uint32_t& w, int k) { w = live >= k + 4 ? w : live <= k ? 0u : w & ((1u << 8 * (live - k)) - 1); };
          keep_bytes(vr[i].x, 0);
          keep_bytes(vr[i].y, 4);
          keep_bytes(vr[i].z, 8);
          keep_bytes(vr[i].w, 12);
        }
        uint4 x, y;
        halves(vr[i], x, y);
        *reinterpret_cast<uint4*>(vs + d * 128 + ((((lane & 3) * 2) ^ (d & 7)) << 4)) = x;
        *reinterpret_cast<uint4*>(vs + d * 128 + ((((lane & 3) * 2 + 1) ^ (d & 7)) << 4)) = y;
      }
      if (p_tid < 4) {  // a piece without a page is not seen
        const float sv = fmaxf(scale.y, 7.888609e-31f);  // 2^-100, the least scale that an append writes
        const bool odd = scale.y != scale.y;
        float* to = reinterpret_cast<float*>(&info[stage][0]) + p_tid;
        to[0] = page < 0 ? 1.f : scale.x;
        to[4] = page < 0 ? -INFINITY : odd ? scale.y : __log2f(sv);
        to[8] = page < 0 || odd ? 1.f : LOWER / sv;
      }
      fence_async_proxy();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[stage]);
      page = next_page;
      if (j + 1 < pieces) load(j + 1);
    }
  }
  // ---- all products are done: the softmax warps have waited for the last one, or a wait ran out, which happens to none that was issued
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == SOFTMAX_WARPS) tmem_dealloc(tmem, S::COLS);
  if (PAIR && tid == 0 && place >= 0) {
    __threadfence();
    atomicExch(a.places + place, 0u);
  }
}

// Puts the parts of a row together: a warp for a row.
template <int DP, typename T>
__global__ void __launch_bounds__(128) kv8_portion_merge_kernel(Kv8AttnArgs a, int slots, int most_parts) {
  constexpr int SIZE = PortionShape<DP, T>::TILES * ROWS;
  grid_dep_launch();
  grid_dep_wait();
  const Kv8View& c = a.c;
  const int slot = slots - 1 - (int)(blockIdx.x / c.kv_heads), head = blockIdx.x % c.kv_heads;
  const Portion w(a, slot, SIZE, most_parts);
  const int i = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= w.rows || w.parts <= 1) return;
  const float* from = a.partials + (size_t)blockIdx.x * most_parts * SIZE * (DP + 2) + (size_t)i * DP;
  const size_t step = (size_t)SIZE * (DP + 2);
  // a lane for a part (at most 32): its maximum, what it is to be multiplied with
  const float2 ml = lane < w.parts ? *reinterpret_cast<const float2*>(from + lane * step + (size_t)(SIZE - i) * DP + 2 * i) : make_float2(-INFINITY, 0.f);
  const float top = lane_max(ml.x), f = ml.x == -INFINITY ? (ml.y == ml.y ? 0.f : ml.y) : ex2(ml.x - top), sum = lane_sum(ml.y * f);
  const float by = sum == 0.f ? 0.f : LOWER / sum;
  const int x = w.row0 + i, tok = x / a.group;
  T* out = (T*)a.out + (size_t)(w.r.first + tok) * a.out_row + (size_t)(head * a.group + (x - tok * a.group)) * c.dim;
  float o[DP / 32];
#pragma unroll
  for (int k = 0; k < DP / 32; ++k) o[k] = 0.f;
#pragma unroll 4
  for (int z = 0; z < w.parts; ++z) {
    const float fz = __shfl_sync(ALL_LANES, f, z);
#pragma unroll
    for (int k = 0; k < DP / 32; ++k)
      if (lane + 32 * k < c.dim) o[k] = fmaf(from[z * step + lane + 32 * k], fz, o[k]);
  }
#pragma unroll
  for (int k = 0; k < DP / 32; ++k)
    if (lane + 32 * k < c.dim) out[lane + 32 * k] = from_f32<T>(o[k] * by);
}

template <int DP, typename T>
cudaError_t run(const Kv8AttnArgs& a, cudaStream_t s) {
  using S = PortionShape<DP, T>;
  constexpr int SIZE = S::TILES * ROWS;
  const int slots = (int)((int64_t)a.rows * a.group / SIZE) + a.c.seqs;
  // parts of a tile along the positions: as many as give every SM a CTA, no more than the workspace and a warp's lanes hold
  const int64_t ctas = (int64_t)slots * a.c.kv_heads;
  const int parts = (int)std::max<int64_t>(1, std::min<int64_t>(32, KV8_MAX_CTAS / ctas));
  const cudaError_t e = launch_kernel(kv8_portion_kernel<DP, T>, dim3((unsigned)ctas, parts), dim3(S::THREADS), S::SMEM, s, true, a, slots);
  if (e != cudaSuccess || parts == 1) return e;
  return launch_kernel(kv8_portion_merge_kernel<DP, T>, dim3((unsigned)ctas, SIZE / 4), dim3(128), 0, s, true, a, slots, parts);
}
template <int DP, typename T>
cudaError_t allow() {
  return cudaFuncSetAttribute(kv8_portion_kernel<DP, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, PortionShape<DP, T>::SMEM);
}
template <typename T>
cudaError_t run_of(const Kv8AttnArgs& a, cudaStream_t s) {
  switch (kv8_padded(a.c.dim)) {
    case 64: return run<64, T>(a, s);
    case 128: return run<128, T>(a, s);
    case 192: return run<192, T>(a, s);
    default: return run<256, T>(a, s);
  }
}

}  // namespace

cudaError_t init_kv8_portion_attributes() {
  cudaError_t all[] = {allow<64, float>(), allow<128, float>(), allow<192, float>(), allow<256, float>(),
                       allow<64, __nv_bfloat16>(), allow<128, __nv_bfloat16>(), allow<192, __nv_bfloat16>(), allow<256, __nv_bfloat16>()};
  for (cudaError_t e : all)
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

cudaError_t launch_kv8_attention_portion(const Kv8AttnArgs& a, int dtype, cudaStream_t s) {
  return dtype == PG_DTYPE_F32 ? run_of<float>(a, s) : run_of<__nv_bfloat16>(a, s);
}

}  // namespace pg
