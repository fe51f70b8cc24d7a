// Scores of rows of logits: log probability of a given token, entropy, the most likely alternatives.
//
// One pass over a row: every thread keeps a running maximum m, S = sum e^(x - m), U = sum (x - m) e^(x - m) over its entries, and the
// place of the largest entry it met; then lp = x_t - M - log S and H = log S - U / S. The alternatives need no second pass over the
// row: the k-th largest of the threads' maxima, tau, is a lower bound of the k-th largest entry, and every entry from tau on was met by
// one of the k threads whose maxima are the largest, so only what those k threads met is read again (from L2). Entries are ordered by
// (value, lower id first) as one 64-bit key, which makes the order total and the k threads unambiguous.
// Bound: bytes, 40 us for 4096 x 32000 BF16 and 80 in FP32; measured 53 (schedulers issue in 74 of 100 cycles, the special functions are busy in 61)
// and 85. In BF16 one exponential for two bytes takes 30 us of the special functions, so the rest is kept to a few instructions: maximum and
// minimum of two entries at once, multiply-adds of two at once. Entries that are masked (-infinity, the type's lowest value) would
// give 0 * infinity in U: where a batch has one so low, its exponents are clamped. Alternatives are the expensive part: sorts and merges of a row's candidates
// across lanes, 17 us for five of each of those rows; 37000 x 1000 FP32 with 20 takes 195 us, 24 by bytes.
// A row is a warp's where there are many rows (no barriers, and every SM has dozens of rows on their way), four warps' where there are
// fewer, a block's or a cluster of up to 8 blocks' where they are few.
#include <cfloat>

#include <cooperative_groups.h>

#include "device_util.cuh"
#include "serving.h"

namespace cg = cooperative_groups;

namespace pg {
namespace {

constexpr int MAX_CLUSTER = 8, LOADS = 4;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LOWEST = -300.f;  // 2^-300 is 0 in FP32, and 0 * -300 no NaN

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float ex2_of(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 16 bytes of a row: maximum (NaN if there is one), minimum, values.
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  float v[4];
  __device__ __forceinline__ void load(const float* p) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  }
  __device__ __forceinline__ float top() const { return max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3])); }
  __device__ __forceinline__ float low() const { return fminf(fminf(v[0], v[1]), fminf(v[2], v[3])); }
  __device__ __forceinline__ float at(int i) const { return v[i]; }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  uint32_t w[4];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ __forceinline__ float top() const {
    const uint32_t m = max2(max2(w[0], w[1]), max2(w[2], w[3]));
    return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u));
  }
  __device__ __forceinline__ float low() const {
    const uint32_t m = min2(min2(w[0], w[1]), min2(w[2], w[3]));
    return fminf(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u));
  }
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16); }
};

// Running statistics of some entries: maximum (NaN once one was met), S, and U in units of log 2.
struct Stats {
  float m, s, u;
  // The same relative to a maximum `to` >= m (or NaN).
  __device__ __forceinline__ void rise(float to) {
    if (s > 0.f) {
      const float d = fmaxf((m - to) * LOG2E, LOWEST), f = ex2_of(d);
      u = f * fmaf(d, s, u);
      s *= f;
    }
    m = to;
  }
  __device__ __forceinline__ void add(float x) {
    const float d = fmaxf((x - m) * LOG2E, LOWEST), e = ex2_of(d);
    s += e;
    u = fmaf(d, e, u);
  }
  __device__ __forceinline__ void join(Stats o) {
    const float to = max_nan(m, o.m);
    rise(to);
    o.rise(to);
    s += o.s;
    u += o.u;
  }
  __device__ __forceinline__ void join_lanes() {
#pragma unroll 1
    for (int o = 16; o; o >>= 1) join({__shfl_xor_sync(ALL_LANES, m, o), __shfl_xor_sync(ALL_LANES, s, o), __shfl_xor_sync(ALL_LANES, u, o)});
  }
};

// (value, id) as a key that is larger for larger values and, among equal ones, for lower ids; 0 is less than every entry's.
__device__ __forceinline__ uint64_t key_of(float x, int id) {
  uint32_t u = __float_as_uint(x + 0.f);  // -0 equals 0
  u = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (uint64_t)u << 32 | (uint32_t)~id;
}
__device__ __forceinline__ int id_of(uint64_t k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float value_of(uint64_t k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}

__device__ __forceinline__ uint64_t swap_with(uint64_t k, int mask, bool keep_large) {
  const uint64_t o = __shfl_xor_sync(ALL_LANES, k, mask);
  return (k > o) == keep_large ? k : o;
}
// Keys of a warp, largest in lane 0.
__device__ __forceinline__ uint64_t sort_keys(uint64_t k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o; o >>= 1) k = swap_with(k, o, ((lane & o) == 0) == ((lane & size) == 0));
  return k;
}
// The 32 largest of two sorted lists, sorted.
__device__ __forceinline__ uint64_t merge_keys(uint64_t a, uint64_t b, int lane) {
  const uint64_t r = __shfl_xor_sync(ALL_LANES, b, 31);  // smallest first
  uint64_t k = a > r ? a : r;
#pragma unroll
  for (int o = 16; o; o >>= 1) k = swap_with(k, o, (lane & o) == 0);
  return k;
}
// The threads that share a row, or a part of one.
template <int WARPS>
struct Team {
  static constexpr int THREADS = WARPS * 32;
  static __device__ __forceinline__ void sync() {
    if (WARPS > 1) __syncthreads();
    else __syncwarp();
  }
  // The 32 largest of all warps' sorted lists, in every warp.
  static __device__ __forceinline__ uint64_t merge(uint64_t k, uint64_t (*lists)[32], int warp, int lane) {
    if constexpr (WARPS > 1) {
#pragma unroll 1
      for (int o = WARPS / 2; o; o >>= 1) {
        if (warp >= o && warp < 2 * o) lists[warp][lane] = k;
        __syncthreads();
        if (warp < o) k = merge_keys(k, lists[warp + o][lane], lane);
      }
      if (warp == 0) lists[0][lane] = k;
      __syncthreads();
      k = lists[0][lane];
    }
    return k;
  }
};

template <typename T, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 256 : WARPS * 32) token_logprobs_kernel(LogprobArgs a) {
  using M = Team<WARPS>;
  constexpr int N = Vec<T>::N, THREADS = M::THREADS;
  __shared__ Stats wstats[WARPS];
  __shared__ uint64_t lists[WARPS == 1 ? 1 : WARPS][32], found[WARPS == 1 ? 8 : WARPS][64];
  grid_dep_launch();
  grid_dep_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, parts = WARPS == 16 ? gridDim.x : 1, part = WARPS == 16 ? blockIdx.x : 0;
  // of the team: threads, warps
  const int tid = WARPS == 1 ? lane : threadIdx.x, warp = WARPS == 1 ? 0 : threadIdx.x >> 5;
  const int64_t row = WARPS == 1 ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : WARPS == 4 ? blockIdx.x : blockIdx.y;
  if (row >= a.rows) return;  // whole teams
  const T* x = (const T*)a.logits + row * a.row;
  // entries before the first 16-byte boundary, vectors, entries behind the last; the vectors are shared out over the parts
  const int head = min(a.vocab, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
  const int vecs = (a.vocab - head) / N, tail = a.vocab - head - vecs * N;
  const int per = (vecs + parts - 1) / parts, v0 = min(part * per, vecs), v1 = min(v0 + per, vecs);
  const bool ends = part == parts - 1;  // the entries outside the vectors

  Stats st{-INFINITY, 0.f, 0.f};
  float best = -INFINITY;  // largest entry of this thread and the vector that has it: -1 head, -2 tail, -3 none
  int best_at = -3;
  if (ends && tid < head) {
    st.m = best = to_f32(x[tid]);
    st.add(best);
    best_at = -1;
  }
  auto batch = [&](const Vec<T> (&r)[LOADS], int v, int n) {
    float top = st.m, low = INFINITY;
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      if (i < n) {
        const float t = r[i].top();
        top = max_nan(top, t);
        low = fminf(low, r[i].low());
        if (t > best || best_at == -3) {
          best = t;
          best_at = v + i * THREADS;
        }
      }
    if (!(top <= st.m)) st.rise(top);
    if ((low - st.m) * LOG2E > LOWEST) {  // (false where the maximum is NaN or infinite)
      const unsigned long long k2 = pack2(LOG2E, LOG2E), m2 = pack2(-st.m, -st.m);
      unsigned long long s2 = pack2(st.s, 0.f), u2 = pack2(st.u, 0.f);
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        if (i < n)
#pragma unroll
          for (int e = 0; e < N; e += 2) {
            const unsigned long long d2 = mul2(add2(pack2(r[i].at(e), r[i].at(e + 1)), m2), k2);  // x - m first: exact where it matters
            float d0, d1;
            unpack2(d2, d0, d1);
            const unsigned long long e2 = pack2(ex2_of(d0), ex2_of(d1));
            s2 = add2(s2, e2);
            u2 = fma2(d2, e2, u2);
          }
      float y0, y1;
      unpack2(s2, y0, y1);
      st.s = y0 + y1;
      unpack2(u2, y0, y1);
      st.u = y0 + y1;
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        if (i < n)
#pragma unroll
          for (int e = 0; e < N; ++e) st.add(r[i].at(e));
    }
  };
  // the next batch is asked for while one is worked on
  auto ask = [&](Vec<T> (&r)[LOADS], int v) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      if (v + i * THREADS < v1) r[i].load(x + head + (size_t)(v + i * THREADS) * N);
  };
  Vec<T> now[LOADS], next[LOADS];
  ask(now, v0 + tid);
#pragma unroll 1
  for (int v = v0 + tid; v < v1; v += THREADS * LOADS) {
    ask(next, v + THREADS * LOADS);
    batch(now, v, min(LOADS, (v1 - v + THREADS - 1) / THREADS));
#pragma unroll
    for (int i = 0; i < LOADS; ++i) now[i] = next[i];
  }
  if (ends && tid < tail) {
    const float t = to_f32(x[head + (size_t)vecs * N + tid]);
    const float to = max_nan(st.m, t);
    if (!(to <= st.m)) st.rise(to);
    st.add(t);
    if (t > best || best_at == -3) {
      best = t;
      best_at = -2;
    }
  }
  // ---- statistics of the team, in a fixed order
  st.join_lanes();
  if (WARPS > 1) {
    if (lane == 0) wstats[warp] = st;
    __syncthreads();
    if (warp == 0) {
      st = lane < WARPS ? wstats[lane] : Stats{-INFINITY, 0.f, 0.f};
      st.join_lanes();
    }
  }

  uint64_t k = 0;
  if (a.top_k) {
    // entries of this thread: its vectors v0 + tid + i * THREADS, and perhaps one of the head or tail
    auto first_at = [&](int at, float value) {  // lowest id in that place with that value
      if (at == -1) return tid;
      if (at == -2) return head + vecs * N + tid;
      Vec<T> r;
      r.load(x + head + (size_t)at * N);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (r.at(e) == value) return head + at * N + e;
      return head + at * N;  // there is a NaN: the row has no distribution
    };
    const uint64_t merged = M::merge(sort_keys(best_at == -3 ? 0 : key_of(best, first_at(best_at, best)), lane), lists, warp, lane);
    const uint64_t tau = __shfl_sync(ALL_LANES, merged, a.top_k - 1);
    // ---- what the k threads with the largest maxima met: entries from tau on are collected, sorted and merged 32 at a time
    uint64_t* mine = found[threadIdx.x >> 5];
    int n = 0;
    auto take = [&](int count) {  // the first 32 (or all `count` < 32) of the collected ones
      __syncwarp();
      k = merge_keys(k, sort_keys(lane < count ? mine[lane] : 0, lane), lane);
      const uint64_t rest = mine[32 + lane];
      __syncwarp();
      mine[lane] = rest;
      __syncwarp();
    };
    auto offer = [&](float value, int at, bool live) {
      const uint64_t c = live ? key_of(value, at) : 0;
      const bool in = live && c >= tau && value == value;
      const unsigned hits = __ballot_sync(ALL_LANES, in);
      if (!hits) return;
      if (in) mine[n + __popc(hits & ((1u << lane) - 1))] = c;
      n += __popc(hits);
      if (n >= 32) {
        take(32);
        n -= 32;
      }
    };
#pragma unroll 1
    for (int w = warp; w < a.top_k; w += WARPS) {
      const uint64_t win = __shfl_sync(ALL_LANES, merged, w);
      if (win == 0) break;  // fewer threads than k have entries
      const int id = id_of(win);
      const int owner = id < head ? id : id >= head + vecs * N ? id - head - vecs * N : ((id - head) / N - v0) % THREADS;
#pragma unroll 1
      for (int v = v0 + owner; v < v1; v += THREADS * 32) {
        const int at = v + lane * THREADS;
        Vec<T> r{};
        if (at < v1) r.load(x + head + (size_t)at * N);
        // a warp where no entry reaches tau has nothing to offer
        if (!__any_sync(ALL_LANES, at < v1 && key_of(r.top(), 0) >= tau)) continue;
#pragma unroll
        for (int e = 0; e < N; ++e) offer(at < v1 ? r.at(e) : 0.f, head + at * N + e, at < v1);
      }
      if (ends) {
        const int at = lane == 0 ? owner : head + vecs * N + owner;
        const bool live = lane == 0 ? owner < head : lane == 1 && owner < tail;
        offer(live ? to_f32(x[at]) : 0.f, at, live);
      }
    }
    if (n) take(n);
    M::sync();
    k = M::merge(k, lists, warp, lane);
  }
  if (WARPS == 16 && parts > 1) {
    if (threadIdx.x == 0) wstats[0] = st;
    cluster.sync();
    if (part == 0) {
      // a warp for a part's list, a lane for its statistics
      if (a.top_k) {
        k = warp < parts ? *cluster.map_shared_rank(&lists[0][lane], warp) : 0;
        __syncthreads();  // lists[0] has been read here
        uint64_t (*other)[32] = lists + 1;
#pragma unroll 1
        for (int o = MAX_CLUSTER / 2; o; o >>= 1) {
          if (warp >= o && warp < 2 * o) other[warp][lane] = k;
          __syncthreads();
          if (warp < o) k = merge_keys(k, other[warp + o][lane], lane);
        }
      }
      if (warp == 0) {
        st = lane < parts ? *cluster.map_shared_rank(&wstats[0], lane) : Stats{-INFINITY, 0.f, 0.f};
        st.join_lanes();
      }
    }
  }
  if (part == 0 && warp == 0) {
    const bool ok = st.m <= FLT_MAX && st.m >= -FLT_MAX;
    const float nan = __uint_as_float(0x7FC00000u), log_s = logf(st.s);
    if (lane == 0) {
      if (a.logprobs) {
        const int t = a.targets[row];
        a.logprobs[row] = t == -1 ? 0.f : !ok || (unsigned)t >= (unsigned)a.vocab ? nan : to_f32(x[t]) - st.m - log_s;
      }
      if (a.entropy) a.entropy[row] = ok ? log_s - st.u / st.s * LN2 : nan;
    }
    if (lane < a.top_k) {
      a.top_ids[row * a.top_k + lane] = ok ? id_of(k) : -1;
      a.top_logprobs[row * a.top_k + lane] = ok ? value_of(k) - st.m - log_s : nan;
    }
  }
  if (WARPS == 16 && parts > 1) cluster.sync();  // the other parts' shared memory is read until here
}

template <typename T>
cudaError_t run(const LogprobArgs& a, int sms, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // Measured, us with a warp / four warps / a block for a row: 37000 x 3400 BF16 64 / 99 / 385; with five alternatives 8000 x 8000 FP32 74 / 75 / 207,
  // 3000 x 20000 BF16 59 / 48 / 97, 1200 x 50257 FP32 127 / 51 / 69, 500 x 30000 BF16 39 / 25 / 22; with 20 400 x 160000 FP32 719 / 133 / 71.
  if (a.rows >= 12 * sms && (int64_t)a.vocab * (int)sizeof(T) <= 16384) {
    cfg.gridDim = dim3((a.rows + 7) / 8);
    cfg.blockDim = dim3(256);
    return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, 1>, a);
  }
  if (a.rows >= 6 * sms) {
    cfg.gridDim = dim3(a.rows);
    cfg.blockDim = dim3(128);
    return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, 4>, a);
  }
  // parts of a row: doubled while that leaves SMs without a block, and each thread two vectors to load
  int parts = 1;
  while (parts < MAX_CLUSTER && (int64_t)a.rows * parts * 2 <= sms && (int64_t)a.vocab * (int)sizeof(T) / 16 >= (int64_t)parts * 2 * 512 * 2) parts *= 2;
  cfg.gridDim = dim3(parts, a.rows);
  cfg.blockDim = dim3(512);
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)parts, 1, 1};
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, 16>, a);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobArgs& a, int dtype, int sms, cudaStream_t s) {
  return dtype == PG_DTYPE_F32 ? run<float>(a, sms, s) : run<__nv_bfloat16>(a, sms, s);
}

}  // namespace pg
