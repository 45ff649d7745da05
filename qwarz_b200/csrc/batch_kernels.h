// Host-side launch interface of the operators that serve many requests from
// one NVFP4 pool and of the token log probabilities (internal; the public C
// ABI is include/qwz_b200.h).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace qwz {

// A step needs more pages than the pool has free (device error word).
constexpr int kErrPoolEmpty = 16;

// Attention of many requests over one NVFP4 pool (batch_few.cu, batch_rows.cu).
struct BatchAttnParams {
  const void* q;                 // [rows, q_heads, dim] FP16/BF16, row stride q_stride
  void* out;                     // same type, row stride out_stride
  const uint8_t* k_codes;        // [P, 256, kv_heads, dim / 2]
  const uint8_t* v_codes;
  const uint8_t* k_scales;       // [P, 256, kv_heads, dim / 16] E4M3
  const uint8_t* v_scales;
  const int32_t* block_table;    // [requests, table_width]
  const int32_t* cu_rows;        // [requests + 1] first row of each request
  const int32_t* kv_lens;        // [requests] tokens after the step
  float* records;                // partial records of batch_few.cu, two per CTA
  float* row_records;            // and of batch_rows.cu
  int32_t* meta;                 // [2][kBatchMaxCtas][kBatchMeta] what the combines have to do
  long long q_stride, out_stride;  // elements
  int requests, rows, table_width, num_pages, kv_heads, group;
  int max_rows;                  // upper bound of a request's rows
  int few_cols;                  // most (row, head) columns a KV head of batch_few.cu has
  int col_groups;                // groups of eight of them
  float sm_scale_log2;           // sm_scale * log2(e)
  // attention behind shared prefixes (the plan of batch_prefix.cu)
  const int32_t* cu_shared;      // [requests + 1] request g is the prefix of the rows shared_rows[cu_shared[g] ..]
  const int32_t* reads;          // [requests] the prefix a request reads (-1: none)
  const int32_t* alone;          // [requests] the only request that reads this one (-1: none, or several do)
  const int32_t* shared_rows;    // [rows] rows by prefix
  int32_t* direct;               // [requests] whether those that read this prefix do so by themselves
  long long* few_starts;         // [col_groups][requests + 1] weighed units of batch_few.cu before each request
  int32_t* busy;                 // [1 + kv_heads * col_groups] CTAs with work of batch_tiles.cu, of batch_few.cu's columns
  // the parts of a row, of its prefix and of its own tokens: [2][rows, q_heads]
  uint32_t* where;               // BatchWhere
  float* part_ml;                // reference maximum and sum of a whole part
  float* part_o;                 // and its unnormalised output [2][rows, q_heads, dim]
};
constexpr int kShareMaxRequests = 1 << 14;
// What a launch of batch_few.cu does: all of a request's tokens
// into out (kBatchPlain), or the parts that batch_join.cu merges (kBatchShared).
enum BatchMode : int { kBatchPlain = 0, kBatchShared = 1 };
// Where a part is: bits 0-1 what, 2-11 first CTA (split) of its records, 12-21 their
// number less one, 22-29 its row in them.  A whole part of a prefix has the row's place in
// shared_rows from bit 2 on (2^30 rows have workspaces of 575 GB), one in records has it for
// its reference maximum.
enum BatchWhere : uint32_t { kWhereDone = 0, kWhereWhole = 1, kWhereFew = 2, kWhereRows = 3 };
constexpr int kBatchMeta = 8;    // int32 words per CTA
constexpr int kBatchMaxSms = 256;
constexpr int kBatchMaxCtas = 4 * kBatchMaxSms;  // batch_few.cu has up to 4 CTAs an SM

// TMA descriptors of the pool's codes as [P * 256 rows, kv_heads * dim / 2
// bytes], boxes of one head's dim / 2 bytes x batch_few_box_rows(dim) rows.
struct alignas(64) BatchPoolMaps {
  CUtensorMap k, v;
};
int batch_few_box_rows(int dim);
constexpr int kBatchFewCols = 8;
constexpr size_t kBatchMetaBytes = 2 * (size_t)kBatchMaxCtas * kBatchMeta * 4;
size_t batch_few_record_bytes(int dim);  // all records of batch_few.cu
size_t batch_workspace_bytes(int dim);
// What attention behind shared prefixes adds to it.
struct BatchSharedSpace {
  int64_t starts, direct, busy, where, ml, o, bytes;  // offsets
  BatchSharedSpace(int dim, int64_t rows, int64_t q_heads) {
    const int64_t pairs = 2 * rows * q_heads;
    starts = 0;
    direct = starts + 2 * 8 * ((int64_t)kShareMaxRequests + 1);
    busy = direct + 4 * (int64_t)kShareMaxRequests;
    where = busy + 4 * 1024;
    ml = where + (4 * pairs + 15) / 16 * 16;
    o = ml + 8 * pairs;
    bytes = o + 4 * pairs * dim;
  }
};

// Paging of many requests (batch_tables.cu).
struct BatchTablesParams {
  const int32_t* lengths;        // [requests] tokens before the step
  const int32_t* new_rows;       // [requests] rows of the step; < 0: the request ends
  const int32_t* held;           // [requests] pages held
  const int32_t* ring_state;     // [2] first free place, free count
  int32_t* ring;                 // [ring_size] page ids
  int32_t* block_table;          // [requests, table_width]
  int32_t* cu_rows;              // [requests + 1]
  int32_t* kv_lens;              // [requests]
  int32_t* held_out;             // [requests]
  int32_t* ring_out;             // [2]
  int32_t* slots;                // [rows]
  int32_t* positions;            // [rows]
  int32_t* request_of;           // [rows]
  int requests, table_width, ring_size;
  long long rows;
};

struct BatchAppendParams {
  const void* k;                 // [rows, kv_heads, dim] FP16/BF16, row stride k_stride
  const void* v;
  uint8_t* k_cache;
  uint8_t* v_cache;
  uint8_t* k_scales;
  uint8_t* v_scales;
  const int32_t* slots;          // [rows] page * 256 + offset; < 0: not stored
  void* k_held;                  // [rows, kv_heads, dim] what the cache stands for, or null
  void* v_held;
  long long rows, k_stride, v_stride;  // strides in elements
  int kv_heads, dim, num_pages;
};

// The step's rows by the prefix they read (batch_prefix.cu).
struct BatchShareParams {
  const int32_t* prefix_of;      // [requests]
  const int32_t* kv_lens;        // [requests]
  const int32_t* cu_rows;        // [requests + 1]
  const int32_t* positions;      // [rows]
  const int32_t* request_of;     // [rows]
  int32_t* cu_shared;            // [requests + 1]
  int32_t* reads;                // [requests]
  int32_t* alone;                // [requests]
  int32_t* shared_rows;          // [rows]
  int32_t* positions_out;        // [rows]
  int requests, rows;
};

constexpr int kRotMaxHeads = 64 * 256;  // of Q
// Q and K normed and rotated, K and V quantised into their slots (batch_prefix.cu).
struct BatchRotateParams {
  BatchAppendParams kv;          // k before the norm and the rotation
  const void* q;                 // [rows, q_heads, dim]
  void* q_out;
  const int32_t* positions;      // [rows]
  const float* inv_freq;         // [freqs] radians a position
  const float* q_weight;         // [dim] of the head norm, or null
  const float* k_weight;
  long long q_stride, q_out_stride;
  int q_heads, freqs, neighbours;  // neighbours: pairs (2i, 2i + 1), otherwise (i, i + freqs)
  float eps;
};

// Token log probabilities (token_logprobs.cu).
struct LogprobParams {
  const void* logits;            // [rows, vocab], row stride `stride` elements
  const void* ids;               // [rows] int32 or int64
  float* logprob;                // [rows]
  float* entropy;                // [rows]
  float* top_logprobs;           // [rows, top]
  int32_t* top_ids;              // [rows, top]
  void* workspace;               // records of parts of rows
  long long stride;
  int rows, vocab, top;
  int ids64;
  int row_tiles, ctas;           // set by the launch: tiles of a row, CTAs of the first kernel
};
enum : int { kDtypeF32 = 2 };    // logits only
long long logprob_records(int rows);
size_t logprob_record_bytes(int top);
cudaError_t launch_token_logprobs(LogprobParams p, int dtype, int sms, cudaStream_t stream);

cudaError_t launch_batch_tables(const BatchTablesParams& p, int sms, cudaStream_t stream);
cudaError_t launch_batch_append(const BatchAppendParams& p, int dtype, cudaStream_t stream);
cudaError_t launch_batch_attend(const BatchAttnParams& p, const BatchPoolMaps& maps, int dim, int dtype, int sms,
                                cudaStream_t stream);
cudaError_t launch_batch_attend_shared(const BatchAttnParams& p, const BatchPoolMaps& maps, int dim, int dtype, int sms,
                                       cudaStream_t stream);
cudaError_t launch_batch_share(const BatchShareParams& p, int sms, cudaStream_t stream);
cudaError_t launch_batch_rotate(const BatchRotateParams& p, int dtype, cudaStream_t stream);

}  // namespace qwz
