// Launches of the serving operators on device buffers (serving.cu has the entry points and their checks).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "puppygrad_b200.h"

namespace pg {

constexpr int KV8_MAX_SEQS = 4096;
// Rows of a (sequence, head) up to which the step kernel has them. us, step / portion kernel:
//   rows                                    16         32         40         48         64
//   16 sequences of 2000, 8 heads of 128,   38 / 47    50 / 49    64 / 51    65 / 51    78 / 51     FP32  49 / 70    73 / 72    88 / 72    101 / 73   127 / 73
//   64 of them                              83 / 214   142 / 229  198 / 229  202 / 230  252 / 232   FP32  145 / 271  262 / 288  306 / 288  376 / 288  492 / 290
//   64 of 2000, 12 heads of 64              77 / 170   135 / 179  173 / 180  174 / 180  238 / 182   FP32  107 / 192  182 / 202  211 / 202  251 / 203  306 / 205
//   one of 8000, 8 heads of 128             20 / 38    23 / 41    28 / 41    28 / 41    32 / 42     FP32  22 / 49    29 / 51    35 / 51    35 / 51    43 / 51
//   8 of 4000, 4 heads of 256               45 / 53    62 / 57    73 / 59    84 / 67    101 / 70    FP32  55 / 85    76 / 89    89 / 89    103 / 108  124 / 111
// The two cross between 32 and 64 rows, at other places for other loads (and not yet for a single sequence). One number for all of them: at
// 40 rows up to a quarter is lost (16 sequences), at 48 a seventh (64 BF16 sequences), half as much again as the step kernel's time for a single one.
constexpr int KV8_STEP_ROWS = 40;
constexpr int KV8_MAX_CTAS = 160;  // of the step kernel's persistent grid: the size of its workspace does not hang on the device
constexpr int KV8_PLACES = 2 * KV8_MAX_CTAS;  // for sums in memory of CTAs of the portion kernel, of which two run on an SM at head_dim 64

__host__ __device__ inline int kv8_padded(int head_dim) { return (head_dim + 63) / 64 * 64; }
// Floats of those sums for an SM: of 256 rows (128 above head_dim 128), with a maximum for each.
__host__ __device__ constexpr int kv8_held(int padded) { return (padded <= 128 ? 256 : 128) * (padded + 1); }

// The cache as the kernels see it.
struct Kv8View {
  uint8_t* pool;
  float* scales;
  const int* table;
  int n_pages, page_tokens, page_shift, kv_heads, dim, seqs, pages_per_seq;
};
struct Kv8AppendArgs {
  Kv8View c;
  const void *k, *v, *q;
  void* q_out;
  int64_t k_row, v_row, q_row, q_out_row;
  int heads, rows;
  const int *row_start, *lens;
  int rot_dims;
  double turn_step;  // entry i turns by position * 2^(turn_step * i)
};
struct Kv8AttnArgs {
  Kv8View c;
  const void* q;
  void* out;
  int64_t q_row, out_row;
  int heads, group, rows, max_rows;
  const int *row_start, *lens;
  float scale;
  int window, keep;
  int step_rows;  // sequences of at most so many (token, head of the group) rows are the step kernel's, the others the portion kernel's
  unsigned *status, *counters, *places;
  float *partials, *held;
};
struct Q4Args {
  const void *x, *bias;
  const uint8_t* packed;
  const uint16_t* scales;
  void* out;
  int64_t x_row, out_row;
  int m, n, k, group;
};
struct LogprobArgs {
  const void* logits;
  int64_t row;
  int rows, vocab, top_k;
  const int* targets;
  float *logprobs, *entropy;
  int* top_ids;
  float* top_logprobs;
};

cudaError_t init_kv8_append_attributes();
cudaError_t init_kv8_step_attributes();
cudaError_t init_kv8_portion_attributes();
cudaError_t init_q4_attributes();
cudaError_t launch_kv8_append(const Kv8AppendArgs& a, int dtype, cudaStream_t s);
cudaError_t launch_kv8_attention_step(const Kv8AttnArgs& a, int dtype, int sms, cudaStream_t s);
cudaError_t launch_kv8_attention_portion(const Kv8AttnArgs& a, int dtype, cudaStream_t s);
cudaError_t launch_quantize_q4(const void* w, int64_t w_row, int dtype, int n, int k, int group, uint8_t* packed, uint16_t* scales, cudaStream_t s);
cudaError_t launch_linear_q4(const Q4Args& a, int dtype, int sms, cudaStream_t s);
cudaError_t launch_token_logprobs(const LogprobArgs& a, int dtype, int sms, cudaStream_t s);

}  // namespace pg
