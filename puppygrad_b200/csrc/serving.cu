// Entry points of the serving operators: checks of what the host can see, then the launch. The kernels are in kv8_append.cu,
// kv8_step.cu, kv8_portion.cu, linear_q4.cu and token_logprobs.cu.
#include "serving.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "common.h"

namespace pg {
int ensure_device(int device);  // model.cu

namespace {

// Makes `device` current for one call and puts the caller's device back.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if (device < 0 || device >= MAX_DEVICES) {
      rc_ = set_error(PG_INVALID_INPUT, "device " + std::to_string(device) + " out of range");
      return;
    }
    if (cudaGetDevice(&before_) != cudaSuccess) before_ = -1;
    sms_ = sms_of_[device].load(std::memory_order_acquire);
    if (sms_ && before_ == device) {  // nothing to change, nothing to put back
      before_ = -1;
      return;
    }
    rc_ = ensure_device(device);
    if (rc_ == PG_OK && !sms_) rc_ = init(device);
  }
  ~DeviceScope() {
    if (before_ >= 0) cudaSetDevice(before_);
  }
  int rc() const { return rc_; }
  int sms() const { return sms_; }

 private:
  static constexpr int MAX_DEVICES = 64;
  static std::atomic<int> sms_of_[MAX_DEVICES];  // 0: no call on that device yet
  int init(int device) {
    cudaError_t e = cudaDeviceGetAttribute(&sms_, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = init_kv8_append_attributes();
    if (e == cudaSuccess) e = init_kv8_step_attributes();
    if (e == cudaSuccess) e = init_kv8_portion_attributes();
    if (e == cudaSuccess) e = init_q4_attributes();
    if (e != cudaSuccess) return set_error(PG_CUDA, std::string("CUDA error: ") + cudaGetErrorString(e));
    sms_of_[device].store(sms_, std::memory_order_release);
    return PG_OK;
  }
  int before_ = -1, rc_ = PG_OK, sms_ = 0;
};
std::atomic<int> DeviceScope::sms_of_[MAX_DEVICES];

int launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return PG_OK;
  cudaGetLastError();  // a refused launch must not be reported again by the caller's next check
  return set_error(PG_CUDA, std::string("CUDA error: ") + cudaGetErrorString(e) + " (" + what + ")");
}

int bad(const std::string& what) { return set_error(PG_INVALID_INPUT, what); }

bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
size_t dtype_size(int dtype) { return dtype == PG_DTYPE_F32 ? 4 : 2; }
int check_dtype(int dtype) {
  return dtype == PG_DTYPE_F32 || dtype == PG_DTYPE_BF16 ? PG_OK : bad("dtype " + std::to_string(dtype) + " must be PG_DTYPE_F32 or PG_DTYPE_BF16");
}
int check_rows(const char* name, const void* p, int64_t row, int64_t width, int dtype) {
  if (!p) return bad(std::string(name) + " is null");
  if (!aligned(p, dtype_size(dtype))) return bad(std::string(name) + " is not aligned to its type");
  if (row < width) return bad(std::string(name) + ": distance between rows " + std::to_string(row) + " is less than a row of " + std::to_string(width));
  return PG_OK;
}

int check_cache_sizes(int n_pages, int page_tokens, int kv_heads, int head_dim) {
  if (n_pages < 1) return bad("n_pages must be > 0");
  if (page_tokens != 16 && page_tokens != 32 && page_tokens != 64) return bad("page_tokens " + std::to_string(page_tokens) + " must be 16, 32 or 64");
  if (kv_heads < 1 || kv_heads > 1024) return bad("kv_heads " + std::to_string(kv_heads) + " must be in 1..1024");
  if (head_dim < 2 || head_dim > 256 || head_dim % 2) return bad("head_dim " + std::to_string(head_dim) + " must be even and in 2..256");
  return PG_OK;
}
int check_cache(const pg_kv8_cache* c) {
  if (!c) return bad("cache is null");
  if (!c->pool || !c->scales || !c->page_table) return bad("cache: null pool, scales or page_table");
  if (int r = check_cache_sizes(c->n_pages, c->page_tokens, c->kv_heads, c->head_dim)) return r;
  if (c->seqs < 1 || c->seqs > KV8_MAX_SEQS) return bad("cache: seqs " + std::to_string(c->seqs) + " must be in 1.." + std::to_string(KV8_MAX_SEQS));
  if (c->pages_per_seq < 1 || (int64_t)c->pages_per_seq * c->page_tokens > INT32_MAX / 2)
    return bad("cache: pages_per_seq " + std::to_string(c->pages_per_seq) + " must be > 0 and hold less than 2^30 positions");
  if (!aligned(c->pool, 16)) return bad("cache: pool is not 16-byte aligned");
  if (!aligned(c->scales, 8) || !aligned(c->page_table, 4)) return bad("cache: scales or page_table is not aligned");
  return PG_OK;
}
int check_heads(const pg_kv8_cache* c, int heads) {
  if (heads < 1 || heads % c->kv_heads || heads / c->kv_heads > 128)
    return bad("heads " + std::to_string(heads) + " must be 1 to 128 times kv_heads " + std::to_string(c->kv_heads));
  return PG_OK;
}
int check_row_map(const pg_kv8_cache* c, int rows, const int32_t* row_start, const int32_t* lens) {
  if (rows < 0) return bad("rows must not be negative");
  if (!lens) return bad("lens is null");
  if (!row_start && rows != c->seqs) return bad("rows " + std::to_string(rows) + " without row_start must be seqs " + std::to_string(c->seqs));
  return PG_OK;
}
Kv8View view(const pg_kv8_cache* c) {
  return {(uint8_t*)c->pool, c->scales, c->page_table, c->n_pages, c->page_tokens, c->page_tokens == 64 ? 6 : c->page_tokens == 32 ? 5 : 4,
          c->kv_heads, c->head_dim, c->seqs, c->pages_per_seq};
}

// A workspace: a word that says whether a wait ran out, counters of the step kernel, one for each of its CTAs, and which of the portion
// kernel's places are taken; for FP32 rows the sums in those places; then parts of tiles: two for every CTA of the step kernel and one for each of its warps, of which there are 16 with tiles of 8
// rows, 8 with tiles of 16. Where the words lie that have to be zero between calls is the same for all calls: parts that one leaves are
// never what the next one counts with.
constexpr size_t COUNTERS_AT = 256, PLACES_AT = 1024, SUMS_AT = 4096;
static_assert(PLACES_AT >= COUNTERS_AT + KV8_MAX_CTAS * 4 && SUMS_AT >= PLACES_AT + KV8_PLACES * 4, "a counter for each CTA, a word for each place");
size_t held_bytes(const pg_kv8_cache* c, int dtype) {
  return dtype == PG_DTYPE_F32 ? ((size_t)KV8_MAX_CTAS * kv8_held(kv8_padded(c->head_dim)) * 4 + 255) / 256 * 256 : 0;
}
size_t partial_bytes(const pg_kv8_cache* c) {
  const int padded = kv8_padded(c->head_dim), rows = padded == 64 ? (2 + 16) * 16 : std::max((2 + 16) * 8, (2 + 8) * 16);
  // (the portion kernel, which runs behind the step kernel, cuts its tiles of 128 or 256 rows into as many parts)
  return (size_t)KV8_MAX_CTAS * std::max(rows, padded == 128 ? 256 : 128) * (padded + 2) * 4;
}

}  // namespace
}  // namespace pg
using namespace pg;

extern "C" {

uint64_t pg_kv8_pool_bytes(int32_t n_pages, int32_t page_tokens, int32_t kv_heads, int32_t head_dim) {
  if (check_cache_sizes(n_pages, page_tokens, kv_heads, head_dim)) return 0;
  return (uint64_t)n_pages * kv_heads * 2 * page_tokens * kv8_padded(head_dim);
}

int pg_kv8_append(const pg_kv8_cache* cache, const void* k, int64_t k_row, const void* v, int64_t v_row, const void* q,
                  int64_t q_row, void* q_out, int64_t q_out_row, int32_t dtype, int32_t heads, int32_t rows,
                  const int32_t* row_start, const int32_t* lens, int32_t rot_dims, double rot_base, void* stream) {
  if (int r = check_cache(cache)) return r;
  if (int r = check_dtype(dtype)) return r;
  if (int r = check_row_map(cache, rows, row_start, lens)) return r;
  const int64_t width = (int64_t)cache->kv_heads * cache->head_dim;
  if (rot_dims < 0 || rot_dims % 2 || rot_dims > cache->head_dim)
    return bad("rot_dims " + std::to_string(rot_dims) + " must be even and in 0.." + std::to_string(cache->head_dim));
  if (rot_dims && !(rot_base > 0 && std::isfinite(rot_base))) return bad("rot_base must be > 0");
  if (!q != !q_out) return bad("q and q_out must be given together");
  if (q)
    if (int r = check_heads(cache, heads)) return r;
  if (rows == 0) return PG_OK;
  if (int r = check_rows("k", k, k_row, width, dtype)) return r;
  if (int r = check_rows("v", v, v_row, width, dtype)) return r;
  if (q) {
    if (int r = check_rows("q", q, q_row, (int64_t)heads * cache->head_dim, dtype)) return r;
    if (int r = check_rows("q_out", q_out, q_out_row, (int64_t)heads * cache->head_dim, dtype)) return r;
    if (q == q_out && q_row != q_out_row) return bad("q_out in place of q must have its distance between rows");
  }
  if (((int64_t)rows / cache->page_tokens + 2 * cache->seqs) * cache->kv_heads * 2 + rows > INT32_MAX) return bad("rows " + std::to_string(rows) + " are too many for one call");
  DeviceScope scope(cache->device);
  if (scope.rc()) return scope.rc();
  Kv8AppendArgs a{view(cache), k, v, q, q_out, k_row, v_row, q_row, q_out_row, heads, rows, row_start, lens, rot_dims,
                  rot_dims ? -2.0 / rot_dims * std::log2(rot_base) : 0.0};
  return launched(launch_kv8_append(a, dtype, (cudaStream_t)stream), "kv8_append");
}

uint64_t pg_kv8_attention_workspace_bytes(const pg_kv8_cache* cache, int32_t rows, int32_t heads, int32_t dtype) {
  if (check_cache(cache) || check_dtype(dtype) || check_heads(cache, heads)) return 0;
  if (rows < 0) return bad("rows must not be negative"), 0;
  return SUMS_AT + held_bytes(cache, dtype) + partial_bytes(cache);
}

int pg_kv8_attention(const pg_kv8_cache* cache, const void* q, int64_t q_row, void* out, int64_t out_row, int32_t dtype,
                     int32_t heads, int32_t rows, int32_t max_rows, const int32_t* row_start, const int32_t* lens, float scale,
                     int32_t window, int32_t keep_first, void* workspace, uint64_t workspace_bytes, void* stream) {
  if (int r = check_cache(cache)) return r;
  if (int r = check_dtype(dtype)) return r;
  if (int r = check_heads(cache, heads)) return r;
  if (int r = check_row_map(cache, rows, row_start, lens)) return r;
  if (!std::isfinite(scale)) return bad("scale must be finite");
  if (window < 0 || keep_first < 0) return bad("window and keep_first must not be negative");
  if (rows == 0) return PG_OK;
  if (max_rows < 1) return bad("max_rows must be > 0");
  const int64_t width = (int64_t)heads * cache->head_dim;
  if (int r = check_rows("q", q, q_row, width, dtype)) return r;
  if (int r = check_rows("out", out, out_row, width, dtype)) return r;
  const size_t need = pg_kv8_attention_workspace_bytes(cache, rows, heads, dtype);
  if (!workspace || workspace_bytes < need)
    return bad("workspace of " + std::to_string(workspace ? workspace_bytes : 0) + " bytes, " + std::to_string(need) + " needed");
  if (!aligned(workspace, 256)) return bad("workspace is not 256-byte aligned");
  // rows of a key / value head, and pieces of 64 tokens of all tiles of rows, are numbered with 31 bits
  const int group = heads / cache->kv_heads;
  const int64_t tiles = ((int64_t)rows * group / 8 + cache->seqs) * cache->kv_heads;
  if ((int64_t)rows * group > INT32_MAX / 2 || tiles * (((int64_t)cache->pages_per_seq * cache->page_tokens + 63) / 64) > INT32_MAX)
    return bad("rows " + std::to_string(rows) + " with tables of " + std::to_string(cache->pages_per_seq) + " pages are too many for one call");
  DeviceScope scope(cache->device);
  if (scope.rc()) return scope.rc();
  if (window > INT32_MAX / 2) window = 0;  // wider than any table: its arithmetic stays within 32 bits
  // rows that fill less than half a tile of the portion kernel, and all of them where it has no table of rows
  const bool portions = row_start && (int64_t)group * max_rows > KV8_STEP_ROWS;
  char *const base = (char*)workspace, *const sums = base + SUMS_AT;
  Kv8AttnArgs a{view(cache), q, out, q_row, out_row, heads, group, rows, max_rows, row_start, lens, scale, window, window > 0 ? keep_first : 0,
                portions ? KV8_STEP_ROWS : INT32_MAX, (unsigned*)base, (unsigned*)(base + COUNTERS_AT), (unsigned*)(base + PLACES_AT),
                (float*)(sums + held_bytes(cache, dtype)), (float*)sums};
  if (!portions) return launched(launch_kv8_attention_step(a, dtype, scope.sms(), (cudaStream_t)stream), "kv8_attention");
  a.max_rows = std::min(max_rows, (KV8_STEP_ROWS + group - 1) / group);
  if (int r = launched(launch_kv8_attention_step(a, dtype, scope.sms(), (cudaStream_t)stream), "kv8_attention")) return r;
  return launched(launch_kv8_attention_portion(a, dtype, (cudaStream_t)stream), "kv8_attention");
}

uint64_t pg_q4_packed_bytes(int32_t n, int32_t k) {
  if (n < 1 || k < 1) return bad("n and k must be > 0"), 0;
  return (uint64_t)((n + 15ll) / 16) * ((k + 63ll) / 64) * 512;
}
uint64_t pg_q4_scale_bytes(int32_t n, int32_t k, int32_t group) {
  if (n < 1 || k < 1) return bad("n and k must be > 0"), 0;
  if (group != 64 && group != 128) return bad("group " + std::to_string(group) + " must be 64 or 128"), 0;
  return (uint64_t)((k + (int64_t)group - 1) / group) * ((n + 15ll) / 16 * 16) * 2;
}

static int check_q4(const void* packed, const void* scales, int n, int k, int group) {
  if (n < 1 || k < 1 || n > (1 << 28) || k > (1 << 28)) return bad("n and k must be in 1..2^28");
  if (group != 64 && group != 128) return bad("group " + std::to_string(group) + " must be 64 or 128");
  if (!packed || !scales) return bad("packed or scales is null");
  if (!aligned(packed, 16) || !aligned(scales, 16)) return bad("packed or scales is not 16-byte aligned");
  return PG_OK;
}

int pg_quantize_q4(const void* w, int64_t w_row, int32_t dtype, int32_t n, int32_t k, int32_t group, void* packed, void* scales,
                   int32_t device, void* stream) {
  if (int r = check_dtype(dtype)) return r;
  if (int r = check_q4(packed, scales, n, k, group)) return r;
  if (int r = check_rows("w", w, w_row, k, dtype)) return r;
  DeviceScope scope(device);
  if (scope.rc()) return scope.rc();
  return launched(launch_quantize_q4(w, w_row, dtype, n, k, group, (uint8_t*)packed, (uint16_t*)scales, (cudaStream_t)stream), "quantize_q4");
}

int pg_linear_q4(const void* x, int64_t x_row, const void* packed, const void* scales, const void* bias, int32_t dtype, int32_t m,
                 int32_t n, int32_t k, int32_t group, void* out, int64_t out_row, int32_t device, void* stream) {
  if (int r = check_dtype(dtype)) return r;
  if (int r = check_q4(packed, scales, n, k, group)) return r;
  if (m < 1 || m > 16) return bad("m " + std::to_string(m) + " must be in 1..16");
  if (int r = check_rows("x", x, x_row, k, dtype)) return r;
  if (int r = check_rows("out", out, out_row, n, dtype)) return r;
  if (bias && !aligned(bias, dtype_size(dtype))) return bad("bias is not aligned to its type");
  DeviceScope scope(device);
  if (scope.rc()) return scope.rc();
  Q4Args a{x, bias, (const uint8_t*)packed, (const uint16_t*)scales, out, x_row, out_row, m, n, k, group};
  return launched(launch_linear_q4(a, dtype, scope.sms(), (cudaStream_t)stream), "linear_q4");
}

int pg_token_logprobs(const void* logits, int64_t row, int32_t dtype, int32_t rows, int32_t vocab, const int32_t* targets,
                      float* logprobs, float* entropy, int32_t top_k, int32_t* top_ids, float* top_logprobs, int32_t device,
                      void* stream) {
  if (int r = check_dtype(dtype)) return r;
  if (rows < 0) return bad("rows must not be negative");
  if (vocab < 1 || vocab > (1 << 30)) return bad("vocab " + std::to_string(vocab) + " must be in 1..2^30");
  if (!targets != !logprobs) return bad("targets and logprobs must be given together");
  if (top_k < 0 || top_k > 32 || top_k > vocab) return bad("top_k " + std::to_string(top_k) + " must be in 0..min(32, vocab)");
  if (top_k && (!top_ids || !top_logprobs)) return bad("top_ids or top_logprobs is null");
  if (rows == 0) return PG_OK;
  if (int r = check_rows("logits", logits, row, vocab, dtype)) return r;
  for (const void* p : {(const void*)targets, (const void*)logprobs, (const void*)entropy, (const void*)top_ids, (const void*)top_logprobs})
    if (!aligned(p, 4)) return bad("targets or an output is not 4-byte aligned");
  if (!logprobs && !entropy && !top_k) return bad("no output is asked for");
  DeviceScope scope(device);
  if (scope.rc()) return scope.rc();
  LogprobArgs a{logits, row, rows, vocab, top_k, targets, logprobs, entropy, top_ids, top_logprobs};
  return launched(launch_token_logprobs(a, dtype, scope.sms(), (cudaStream_t)stream), "token_logprobs");
}

}  // extern "C"
