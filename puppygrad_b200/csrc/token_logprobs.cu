// Scores of rows of logits: log probability of a given token, entropy, the most likely alternatives.
//
// One pass over a row: every thread keeps a running maximum m, S = sum e^(x - m), U = sum (x - m) e^(x - m) over its entries, and the
// largest entry it met; then lp = x_t - M - log S and H = log S - U / S. The alternatives need no second pass over the row: the k-th
// largest of the threads' maxima, tau, is a lower bound of the k-th largest entry, and every entry from tau on was met by one of the
// k threads whose maxima are the largest, so only what those k threads met is read again (from L2). Entries are ordered by (value, lower
// id first) as one 64-bit key, which makes the order total and the k threads unambiguous.
// Bound: memory. A row belongs to a cluster of 1 to 8 CTAs, as many as it takes to fill the chip when rows are few.
#include <cfloat>

#include <cooperative_groups.h>

#include "device_util.cuh"
#include "serving.h"

namespace cg = cooperative_groups;

namespace pg {
namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32, MAX_CLUSTER = 8, LOADS = 4;
constexpr float LOG2E = 1.4426950408889634f;

template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  float v[N];
  __device__ __forceinline__ void load(const T* p) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (sizeof(T) == 4) {
        v[i] = __uint_as_float(w[i]);
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    }
  }
};

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

// Running statistics of some entries: maximum (NaN once one was met), S and U.
struct Stats {
  float m, s, u;
  __device__ __forceinline__ void rise(float to) {  // to >= m, or NaN
    if (s > 0.f) {
      const float d = fmaxf(m - to, -200.f), f = ex2_of(d * LOG2E);
      u = f * fmaf(d, s, u);
      s *= f;
    }
    m = to;
  }
  // masked entries are -infinity or the type's lowest value: e^-200 is 0 in FP32 and 0 * -200 is no NaN
  __device__ __forceinline__ void add(float x) {
    const float d = fmaxf(x - m, -200.f), e = ex2_of(d * LOG2E);
    s += e;
    u = fmaf(d, e, u);
  }
  __device__ __forceinline__ void join(const Stats& o) {
    const float to = max_nan(m, o.m);
    Stats b = o;
    if (b.s > 0.f) {
      const float d = fmaxf(b.m - to, -200.f), f = ex2_of(d * LOG2E);
      b.u = f * fmaf(d, b.s, b.u);
      b.s *= f;
    }
    if (s > 0.f) {
      const float d = fmaxf(m - to, -200.f), f = ex2_of(d * LOG2E);
      u = f * fmaf(d, s, u);
      s *= f;
    }
    m = to;
    s += b.s;
    u += b.u;
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
// The 32 largest of all warps' sorted lists, in warp 0 (and `lists`).
__device__ uint64_t merge_warps(uint64_t k, uint64_t (*lists)[32], int warp, int lane) {
  for (int o = WARPS / 2; o; o >>= 1) {
    if (warp >= o && warp < 2 * o) lists[warp][lane] = k;
    __syncthreads();
    if (warp < o) k = merge_keys(k, lists[warp + o][lane], lane);
    __syncthreads();
  }
  if (warp == 0) lists[0][lane] = k;
  __syncthreads();
  return lists[0][lane];
}

template <typename T>
__global__ void __launch_bounds__(THREADS) token_logprobs_kernel(LogprobArgs a) {
  constexpr int N = Vec<T>::N;
  __shared__ Stats wstats[WARPS];
  __shared__ uint64_t lists[WARPS][32];
  __shared__ uint64_t winners[32];
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = gridDim.x, part = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  if (row >= a.rows) return;  // whole clusters
  const T* x = (const T*)a.logits + row * a.row;
  // entries before the first 16-byte boundary, vectors, entries behind the last; the vectors are shared out over the parts
  const int head = min(a.vocab, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
  const int vecs = (a.vocab - head) / N, tail = a.vocab - head - vecs * N;
  const int per = (vecs + parts - 1) / parts, v0 = min(part * per, vecs), v1 = min(v0 + per, vecs);
  const bool ends = part == parts - 1;  // the entries outside the vectors

  Stats st{-INFINITY, 0.f, 0.f};
  float best = -INFINITY;  // largest entry of this thread (no NaN) and the vector that has it: -1 head, -2 tail, -3 none
  int best_at = -3;
  if (ends && tid < head) {
    st.m = max_nan(st.m, to_f32(x[tid]));
    st.add(to_f32(x[tid]));
    best = fmaxf(best, to_f32(x[tid]));
    best_at = -1;
  }
  for (int v = v0 + tid; v < v1; v += THREADS * LOADS) {
    Vec<T> r[LOADS];
    const int n = min(LOADS, (v1 - v + THREADS - 1) / THREADS);
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      if (i < n) r[i].load(x + head + (size_t)(v + i * THREADS) * N);
    float top = st.m;
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      if (i < n) {
        float t = r[i].v[0], tn = r[i].v[0];
#pragma unroll
        for (int e = 1; e < N; ++e) {
          t = fmaxf(t, r[i].v[e]);
          tn = max_nan(tn, r[i].v[e]);
        }
        top = max_nan(top, tn);
        if (t > best || best_at == -3) {
          best = t;
          best_at = v + i * THREADS;
        }
      }
    if (!(top <= st.m)) st.rise(top);
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      if (i < n)
#pragma unroll
        for (int e = 0; e < N; ++e) st.add(r[i].v[e]);
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
  // ---- statistics of the block, in a fixed order
#pragma unroll
  for (int o = 16; o; o >>= 1) st.join({__shfl_xor_sync(ALL_LANES, st.m, o), __shfl_xor_sync(ALL_LANES, st.s, o), __shfl_xor_sync(ALL_LANES, st.u, o)});
  if (lane == 0) wstats[warp] = st;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < WARPS; ++w) st.join(wstats[w]);
    wstats[0] = st;
  }

  if (a.top_k) {
    // entries of this thread: its vectors v0 + tid + i * THREADS, and perhaps one of the head or tail
    auto first_at = [&](int at, float value) {  // lowest id in that place with that value
      if (at == -1) return tid;
      if (at == -2) return head + vecs * N + tid;
      Vec<T> r;
      r.load(x + head + (size_t)at * N);
      for (int e = 0; e < N; ++e)
        if (r.v[e] == value) return head + at * N + e;
      return head + at * N;  // nothing but NaN: the row has no distribution
    };
    uint64_t k = best_at == -3 ? 0 : key_of(best, first_at(best_at, best));
    const uint64_t merged = merge_warps(sort_keys(k, lane), lists, warp, lane);
    const uint64_t tau = __shfl_sync(ALL_LANES, merged, a.top_k - 1);
    if (warp == 0) winners[lane] = merged;
    __syncthreads();
    // ---- what the k threads with the largest maxima met
    k = 0;
    for (int w = warp; w < a.top_k; w += WARPS) {
      const uint64_t win = winners[w];
      if (win == 0) break;  // fewer threads than k have entries
      const int id = id_of(win);
      const int owner = id < head ? id : id >= head + vecs * N ? id - head - vecs * N : ((id - head) / N - v0) % THREADS;
      auto offer = [&](float value, int at, bool live) {
        const uint64_t c = live ? key_of(value, at) : 0;
        const uint64_t least = __shfl_sync(ALL_LANES, k, 31);
        const bool in = c >= tau && c > least && value == value;
        if (__any_sync(ALL_LANES, in)) k = merge_keys(k, sort_keys(in ? c : 0, lane), lane);
      };
      for (int v = v0 + owner; v < v1; v += THREADS * 32) {
        const int mine = v + lane * THREADS;
        Vec<T> r;
        if (mine < v1) r.load(x + head + (size_t)mine * N);
        for (int e = 0; e < N; ++e) offer(mine < v1 ? r.v[e] : 0.f, head + mine * N + e, mine < v1);
      }
      if (ends) {
        const int at = lane == 0 ? owner : head + vecs * N + owner;
        const bool live = lane == 0 ? owner < head : lane == 1 && owner < tail;
        offer(live ? to_f32(x[at]) : 0.f, at, live);
      }
    }
    merge_warps(k, lists, warp, lane);
  }
  cluster.sync();
  if (part == 0) {
    if (warp == 0) {
      Stats all = wstats[0];
      uint64_t k = a.top_k ? lists[0][lane] : 0;
      for (int p = 1; p < parts; ++p) {
        all.join(*cluster.map_shared_rank(&wstats[0], p));
        if (a.top_k) k = merge_keys(k, *cluster.map_shared_rank(&lists[0][lane], p), lane);
      }
      const bool ok = all.m <= FLT_MAX && all.m >= -FLT_MAX;
      const float nan = __uint_as_float(0x7FC00000u), log_s = logf(all.s);
      if (lane == 0) {
        if (a.logprobs) {
          const int t = a.targets[row];
          a.logprobs[row] = t == -1 ? 0.f : !ok || (unsigned)t >= (unsigned)a.vocab ? nan : to_f32(x[t]) - all.m - log_s;
        }
        if (a.entropy) a.entropy[row] = ok ? log_s - all.u / all.s : nan;
      }
      if (lane < a.top_k) {
        a.top_ids[row * a.top_k + lane] = ok ? id_of(k) : -1;
        a.top_logprobs[row * a.top_k + lane] = ok ? value_of(k) - all.m - log_s : nan;
      }
    }
  }
  cluster.sync();  // the other parts' shared memory is read until here
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobArgs& a, int dtype, int sms, cudaStream_t s) {
  const int size = dtype == PG_DTYPE_F32 ? 4 : 2;
  // parts of a row: doubled while that leaves SMs without a block, and each thread two vectors to load
  int parts = 1;
  while (parts < MAX_CLUSTER && (int64_t)a.rows * parts * 2 <= sms && (int64_t)a.vocab * size / 16 >= (int64_t)parts * 2 * THREADS * 2) parts *= 2;
  cudaLaunchConfig_t cfg = {};
  const unsigned y = a.rows < 65535 ? a.rows : 65535;
  cfg.gridDim = dim3(parts, y, (a.rows + y - 1) / y);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)parts, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return dtype == PG_DTYPE_F32 ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<float>, a) : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<__nv_bfloat16>, a);
}

}  // namespace pg
