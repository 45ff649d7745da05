// C ABI of the operators that serve many requests from one NVFP4 pool
// (batch_tables.cu, batch_few.cu) and of the token log probabilities
// (token_logprobs.cu).  Part of the single translation unit qwz_b200.cu; it
// uses the argument checks of capi.cu.

#include "qwz_common.cuh"
#include "batch_kernels.h"
#include "qwz_kernels.h"
#include "../../include/qwz_b200.h"

namespace {

int check_batch_pool(const void* kc, const void* vc, const void* ks, const void* vs, int32_t num_pages,
                     int32_t kv_heads, int32_t dim) {
  const int rc = check_nvfp4_cache(kc, vc, ks, vs, num_pages);
  if (rc) return rc;
  if (kv_heads < 1 || kv_heads > 256) return fail(QWZ_EINVAL, "num_kv_heads must be in 1..256");
  if (dim != 64 && dim != 128 && dim != 256) return fail(QWZ_EINVAL, "head_dim must be 64, 128 or 256");
  return QWZ_OK;
}

int check_row_stride(int64_t stride, int64_t width, const char* what) {
  if (stride < width || stride % 8 != 0)
    return fail(QWZ_EINVAL, "%s: the row stride must be a multiple of 8 elements and hold a row", what);
  return QWZ_OK;
}

// SMs of the current device (0: none).
int batch_sms() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return sms < qwz::kBatchMaxSms ? sms : qwz::kBatchMaxSms;
}

}  // namespace

extern "C" {

int qwz_batch_tables(const int32_t* lengths, const int32_t* new_rows, const int32_t* held, int32_t* ring,
                     const int32_t* ring_state, int32_t* block_table, int32_t* cu_rows, int32_t* kv_lens,
                     int32_t* held_out, int32_t* ring_out, int32_t* slots, int32_t* positions, int32_t* request_of,
                     int32_t requests, int32_t table_width, int32_t ring_size, int64_t rows, void* stream) {
  if (!lengths || !new_rows || !held || !ring || !ring_state || !block_table || !cu_rows || !kv_lens || !held_out ||
      !ring_out)
    return fail(QWZ_EINVAL, "request, ring, table and output arrays are required (non-null)");
  if (rows < 0 || rows > 0x7fffffff) return fail(QWZ_EINVAL, "rows must be in 0..2^31-1");
  if (rows > 0 && (!slots || !positions || !request_of))
    return fail(QWZ_EINVAL, "slots, positions and request_of are required");
  if (requests < 1 || requests > (1 << 20)) return fail(QWZ_EINVAL, "requests must be in 1..2^20");
  if (table_width < 1 || table_width > (1 << 22)) return fail(QWZ_EINVAL, "table_width must be in 1..2^22");
  if (ring_size < 1) return fail(QWZ_EINVAL, "ring_size must be positive");
  // every CTA reads all of the inputs while others write
  struct Array {
    const int32_t* at;
    int64_t n;
  };
  const Array both[] = {{ring, ring_size}, {block_table, (int64_t)requests * table_width}};  // read and written
  const Array reads[] = {{lengths, requests}, {new_rows, requests}, {held, requests}, {ring_state, 2}};
  const Array writes[] = {{cu_rows, requests + 1}, {kv_lens, requests}, {held_out, requests}, {ring_out, 2},
                          {slots, rows},           {positions, rows},   {request_of, rows}};
  auto shared = [](const Array& a, const Array& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
    return a.n > 0 && b.n > 0 && x < y + 4 * (uintptr_t)b.n && y < x + 4 * (uintptr_t)a.n;
  };
  bool clash = shared(both[0], both[1]);
  for (const Array& r : reads) {
    for (const Array& w : writes) clash |= shared(r, w);
    for (const Array& w : both) clash |= shared(r, w);
  }
  for (const Array& r : both)
    for (const Array& w : writes) clash |= shared(r, w);
  if (clash) return fail(QWZ_EINVAL, "outputs must not share storage with inputs");
  const int sms = batch_sms();
  if (sms <= 0) return fail(QWZ_ELAUNCH, "no CUDA device");
  qwz::BatchTablesParams p{lengths, new_rows, held, ring_state, ring, block_table, cu_rows, kv_lens, held_out,
                           ring_out, slots, positions, request_of, requests, table_width, ring_size, rows};
  return launched(qwz::launch_batch_tables(p, sms, as_stream(stream)), "qwz_batch_tables");
}

int qwz_batch_append(const void* k, const void* v, void* k_cache, void* v_cache, void* k_scales, void* v_scales,
                     const int32_t* slots, void* k_held, void* v_held, int64_t rows, int64_t k_stride,
                     int64_t v_stride, int32_t num_kv_heads, int32_t head_dim, int32_t num_pages, int32_t dtype,
                     void* stream) {
  int rc = check_dtype(dtype);
  if (rc) return rc;
  rc = check_batch_pool(k_cache, v_cache, k_scales, v_scales, num_pages, num_kv_heads, head_dim);
  if (rc) return rc;
  if (rows < 0 || rows > (1 << 24)) return fail(QWZ_EINVAL, "rows must be in 0..2^24");
  if (rows == 0) return QWZ_OK;
  if (!k || !v || !slots) return fail(QWZ_EINVAL, "k, v and slots are required");
  if (!aligned(k, 16) || !aligned(v, 16) || (k_held && !aligned(k_held, 16)) || (v_held && !aligned(v_held, 16)))
    return fail(QWZ_EINVAL, "k, v, k_held and v_held must be 16-byte aligned");
  const int64_t width = (int64_t)num_kv_heads * head_dim;
  if ((rc = check_row_stride(k_stride, width, "k"))) return rc;
  if ((rc = check_row_stride(v_stride, width, "v"))) return rc;
  qwz::BatchAppendParams p{};
  p.k = k;
  p.v = v;
  p.k_cache = static_cast<uint8_t*>(k_cache);
  p.v_cache = static_cast<uint8_t*>(v_cache);
  p.k_scales = static_cast<uint8_t*>(k_scales);
  p.v_scales = static_cast<uint8_t*>(v_scales);
  p.slots = slots;
  p.k_held = k_held;
  p.v_held = v_held;
  p.rows = rows;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.kv_heads = num_kv_heads;
  p.dim = head_dim;
  p.num_pages = num_pages;
  return launched(qwz::launch_batch_append(p, dtype, as_stream(stream)), "qwz_batch_append");
}

int64_t qwz_batch_attend_workspace_bytes(int32_t head_dim) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
  return (int64_t)qwz::batch_workspace_bytes(head_dim);
}

int qwz_batch_attend(const void* q, const void* k_cache, const void* v_cache, const void* k_scales,
                     const void* v_scales, const int32_t* block_table, const int32_t* cu_rows,
                     const int32_t* kv_lens, void* out, void* workspace, int64_t workspace_bytes, int32_t rows,
                     int32_t requests, int32_t max_rows, int32_t table_width, int32_t num_pages,
                     int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int64_t q_stride,
                     int64_t out_stride, float sm_scale, int32_t dtype, void* stream) {
  int rc = check_dtype(dtype);
  if (rc) return rc;
  rc = check_batch_pool(k_cache, v_cache, k_scales, v_scales, num_pages, num_kv_heads, head_dim);
  if (rc) return rc;
  if (rows < 0 || requests < 0 || requests > (1 << 20)) return fail(QWZ_EINVAL, "rows and requests must be >= 0 (requests at most 2^20)");
  if (max_rows < 1) return fail(QWZ_EINVAL, "max_rows must be positive");
  if (table_width < 1 || table_width > (1 << 22)) return fail(QWZ_EINVAL, "table_width must be in 1..2^22");
  if (num_q_heads < num_kv_heads || num_q_heads % num_kv_heads != 0 || num_q_heads / num_kv_heads > 64)
    return fail(QWZ_EINVAL, "num_q_heads must be 1 to 64 times num_kv_heads");
  const int64_t width = (int64_t)num_q_heads * head_dim;
  if ((rc = check_row_stride(q_stride, width, "q"))) return rc;
  if ((rc = check_row_stride(out_stride, width, "out"))) return rc;
  if (!(sm_scale > 0.f) || !std::isfinite(sm_scale)) return fail(QWZ_EINVAL, "sm_scale must be positive and finite");
  if (rows == 0 || requests == 0) return QWZ_OK;
  if (!q || !out || !aligned(q, 16) || !aligned(out, 16)) return fail(QWZ_EINVAL, "q and out must be non-null 16-byte aligned pointers");
  if (!block_table || !cu_rows || !kv_lens) return fail(QWZ_EINVAL, "block_table, cu_rows and kv_lens are required");
  if (!workspace || !aligned(workspace, 16)) return fail(QWZ_EINVAL, "workspace must be a non-null 16-byte aligned pointer");
  if (workspace_bytes < (int64_t)qwz::batch_workspace_bytes(head_dim))
    return fail(QWZ_EINVAL, "workspace smaller than qwz_batch_attend_workspace_bytes(head_dim)");
  const int sms = batch_sms();
  if (sms <= 0) return fail(QWZ_ELAUNCH, "no CUDA device");
  qwz::BatchPoolMaps maps;
  const uint64_t pool_rows = (uint64_t)num_pages * qwz::kPage, row_bytes = (uint64_t)num_kv_heads * head_dim / 2;
  const CUtensorMapSwizzle swizzle = head_dim == 256   ? CU_TENSOR_MAP_SWIZZLE_128B
                                     : head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                       : CU_TENSOR_MAP_SWIZZLE_32B;
  const uint32_t box_rows = (uint32_t)qwz::batch_few_box_rows(head_dim);
  rc = encode_2d(&maps.k, k_cache, row_bytes, pool_rows, head_dim / 2, box_rows, swizzle);
  if (!rc) rc = encode_2d(&maps.v, v_cache, row_bytes, pool_rows, head_dim / 2, box_rows, swizzle);
  if (rc) return rc;
  qwz::BatchAttnParams p{};
  p.q = q;
  p.out = out;
  p.k_codes = static_cast<const uint8_t*>(k_cache);
  p.v_codes = static_cast<const uint8_t*>(v_cache);
  p.k_scales = static_cast<const uint8_t*>(k_scales);
  p.v_scales = static_cast<const uint8_t*>(v_scales);
  p.block_table = block_table;
  p.cu_rows = cu_rows;
  p.kv_lens = kv_lens;
  p.meta = static_cast<int32_t*>(workspace);
  p.records = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + qwz::kBatchMetaBytes);
  p.row_records = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + qwz::kBatchMetaBytes +
                                          qwz::batch_few_record_bytes(head_dim));
  p.q_stride = q_stride;
  p.out_stride = out_stride;
  p.requests = requests;
  p.rows = rows;
  p.table_width = table_width;
  p.num_pages = num_pages;
  p.kv_heads = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.max_rows = max_rows;
  // Decode rows of 9 to 16 heads a KV head are two groups of columns in batch_few.cu:
  // 8 requests of 32,768 tokens, 48/4/256: 124 us against 193 in batch_rows.cu; 512 of
  // 512 tokens, 96/8/64: 124 against 316.  What has more columns goes to batch_rows.cu.
  // The group of heads alone decides, so that a request's result does not depend on
  // max_rows.  With fewer heads a launch for two groups would gain on windows of 9 to
  // 16 columns and lose on decode rows, whose CTAs it halves: 16 requests of 4,096 to
  // 32,768 tokens, 24/4/256, 2 rows 109 us against 176, 1 row 108 against 63; 32/8/128,
  // 3 rows 122 against 201, 1 row 120 against 71.
  p.col_groups = p.group > qwz::kBatchFewCols && p.group <= 2 * qwz::kBatchFewCols ? 2 : 1;
  p.few_cols = p.col_groups * qwz::kBatchFewCols;
  p.sm_scale_log2 = sm_scale * kLog2e;
  return launched(qwz::launch_batch_attend(p, maps, head_dim, dtype, sms, as_stream(stream)), "qwz_batch_attend");
}

int64_t qwz_token_logprobs_workspace_bytes(int32_t rows, int32_t vocab, int32_t top, int32_t dtype) {
  if (rows < 0 || vocab < 1 || vocab > (1 << 30) || top < 0 || top > 32 || dtype < 0 || dtype > QWZ_DTYPE_F32) return 0;
  return qwz::logprob_records(rows) * (int64_t)qwz::logprob_record_bytes(top);
}

int qwz_token_logprobs(const void* logits, const void* ids, int32_t ids64, float* logprob, float* entropy,
                       float* top_logprobs, int32_t* top_ids, void* workspace, int64_t workspace_bytes, int32_t rows,
                       int32_t vocab, int32_t top, int64_t stride, int32_t dtype, void* stream) {
  if (dtype < 0 || dtype > QWZ_DTYPE_F32)
    return fail(QWZ_EINVAL, "dtype must be QWZ_DTYPE_F16 (0), QWZ_DTYPE_BF16 (1) or QWZ_DTYPE_F32 (2)");
  if (rows < 0) return fail(QWZ_EINVAL, "rows must be >= 0");
  if (vocab < 1 || vocab > (1 << 30)) return fail(QWZ_EINVAL, "vocab must be in 1..2^30");
  if (top < 0 || top > 32 || top > vocab) return fail(QWZ_EINVAL, "top must be in 0..32 and at most vocab");
  if (rows == 0) return QWZ_OK;
  if (!logits || !ids || !logprob || !entropy) return fail(QWZ_EINVAL, "logits, ids, logprob and entropy are required");
  if (top > 0 && (!top_logprobs || !top_ids)) return fail(QWZ_EINVAL, "top_logprobs and top_ids are required");
  const int item = dtype == QWZ_DTYPE_F32 ? 4 : 2;
  if (!aligned(logits, item)) return fail(QWZ_EINVAL, "logits must be aligned to their element");
  if (stride < vocab && stride != 0 && rows > 1) return fail(QWZ_EINVAL, "the row stride must hold a row (or be 0)");
  if (!workspace || !aligned(workspace, 16)) return fail(QWZ_EINVAL, "workspace must be a non-null 16-byte aligned pointer");
  if (workspace_bytes < qwz_token_logprobs_workspace_bytes(rows, vocab, top, dtype))
    return fail(QWZ_EINVAL, "workspace smaller than qwz_token_logprobs_workspace_bytes");
  const int sms = batch_sms();
  if (sms <= 0) return fail(QWZ_ELAUNCH, "no CUDA device");
  qwz::LogprobParams p{logits, ids, logprob, entropy, top_logprobs, top_ids, workspace, stride, rows, vocab, top, ids64,
                       0, 0};
  return launched(qwz::launch_token_logprobs(p, dtype, sms, as_stream(stream)), "qwz_token_logprobs");
}

}  // extern "C"
