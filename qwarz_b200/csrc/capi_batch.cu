// C ABI of the operators that serve many requests from one NVFP4 pool
// (batch_tables.cu, batch_few.cu, batch_prefix.cu) and of the token log
// probabilities (token_logprobs.cu).  Part of the single translation unit qwz_b200.cu; it
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

// Whether bytes [a, a + n) and [b, b + m) meet.
bool meet(const void* a, int64_t n, const void* b, int64_t m) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && n > 0 && m > 0 && x < y + (uintptr_t)m && y < x + (uintptr_t)n;
}

// Whether rows of `width` elements at `a` and of `other` at `b` meet: rows of one
// stride lie side by side in a packed projection's rows.
bool rows_meet(const void* a, int64_t width, int64_t stride, const void* b, int64_t other, int64_t other_stride,
               int64_t rows) {
  if (!meet(a, 2 * ((rows - 1) * stride + width), b, 2 * ((rows - 1) * other_stride + other))) return false;
  if (stride != other_stride) return true;
  const int64_t pitch = 2 * stride;
  int64_t off = (int64_t)(reinterpret_cast<uintptr_t>(b) - reinterpret_cast<uintptr_t>(a)) % pitch;
  if (off < 0) off += pitch;
  return off < 2 * width || off + 2 * other > pitch;
}

// The same of such rows and bytes [b, b + n), which may lie between two rows.
bool row_meets(const void* a, int64_t width, int64_t stride, int64_t rows, const void* b, int64_t n) {
  if (!meet(a, 2 * ((rows - 1) * stride + width), b, n)) return false;
  const int64_t off = (int64_t)(reinterpret_cast<uintptr_t>(b) - reinterpret_cast<uintptr_t>(a)), pitch = 2 * stride;
  const int64_t row = off < 2 * width ? 0 : (off - 2 * width) / pitch + 1;  // the first that ends behind b
  return row < rows && row * pitch < off + n;
}

// SMs of the current device (0: none).
int batch_sms() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return sms < qwz::kBatchMaxSms ? sms : qwz::kBatchMaxSms;
}

}  // namespace

extern "C" int64_t qwz_batch_shared_workspace_bytes(int32_t, int32_t, int32_t);

namespace {

// Checks and packs what the two writers have in common.
int append_checked(qwz::BatchAppendParams& p, const void* k, const void* v, void* k_cache, void* v_cache, void* k_scales, void* v_scales,
                     const int32_t* slots, void* k_held, void* v_held, int64_t rows, int64_t k_stride,
                     int64_t v_stride, int32_t num_kv_heads, int32_t head_dim, int32_t num_pages, int32_t dtype) {
  int rc = check_dtype(dtype);
  if (rc) return rc;
  rc = check_batch_pool(k_cache, v_cache, k_scales, v_scales, num_pages, num_kv_heads, head_dim);
  if (rc) return rc;
  if (rows < 0 || rows > (1 << 24)) return fail(QWZ_EINVAL, "rows must be in 0..2^24");
  if (rows == 0) return QWZ_OK;  // nothing to launch: p stays empty
  if (!k || !v || !slots) return fail(QWZ_EINVAL, "k, v and slots are required");
  if (!aligned(k, 16) || !aligned(v, 16) || (k_held && !aligned(k_held, 16)) || (v_held && !aligned(v_held, 16)))
    return fail(QWZ_EINVAL, "k, v, k_held and v_held must be 16-byte aligned");
  const int64_t width = (int64_t)num_kv_heads * head_dim;
  if ((rc = check_row_stride(k_stride, width, "k"))) return rc;
  if ((rc = check_row_stride(v_stride, width, "v"))) return rc;
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
  return QWZ_OK;
}

// qwz_batch_attend, and with a plan qwz_batch_attend_shared.
int attend_checked(const char* what, const int32_t* plan, bool shared, const void* q, const void* k_cache, const void* v_cache, const void* k_scales,
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
  if (shared && requests > qwz::kShareMaxRequests) return fail(QWZ_EINVAL, "requests must be at most 2^14");
  if (rows == 0 || requests == 0) return QWZ_OK;
  if (!q || !out || !aligned(q, 16) || !aligned(out, 16)) return fail(QWZ_EINVAL, "q and out must be non-null 16-byte aligned pointers");
  if (!block_table || !cu_rows || !kv_lens) return fail(QWZ_EINVAL, "block_table, cu_rows and kv_lens are required");
  if (shared && !plan) return fail(QWZ_EINVAL, "plan is required");
  if (!workspace || !aligned(workspace, 16)) return fail(QWZ_EINVAL, "workspace must be a non-null 16-byte aligned pointer");
  if (!shared && workspace_bytes < (int64_t)qwz::batch_workspace_bytes(head_dim))
    return fail(QWZ_EINVAL, "workspace smaller than qwz_batch_attend_workspace_bytes(head_dim)");
  if (shared && workspace_bytes < qwz_batch_shared_workspace_bytes(head_dim, rows, num_q_heads))
    return fail(QWZ_EINVAL, "workspace smaller than qwz_batch_shared_workspace_bytes(head_dim, rows, num_q_heads)");
  if (shared && rows_meet(q, width, q_stride, out, width, out_stride, rows))
    return fail(QWZ_EINVAL, "out must not share storage with q");
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
  if (!shared) return launched(qwz::launch_batch_attend(p, maps, head_dim, dtype, sms, as_stream(stream)), what);
  p.cu_shared = plan;
  p.reads = p.cu_shared + requests + 1;
  p.alone = p.reads + requests;
  p.shared_rows = p.alone + requests;
  uint8_t* space = static_cast<uint8_t*>(workspace) + qwz::batch_workspace_bytes(head_dim);
  const qwz::BatchSharedSpace at(head_dim, rows, num_q_heads);
  p.few_starts = reinterpret_cast<long long*>(space + at.starts);
  p.direct = reinterpret_cast<int32_t*>(space + at.direct);
  p.busy = reinterpret_cast<int32_t*>(space + at.busy);
  p.where = reinterpret_cast<uint32_t*>(space + at.where);
  p.part_ml = reinterpret_cast<float*>(space + at.ml);
  p.part_o = reinterpret_cast<float*>(space + at.o);
  return launched(qwz::launch_batch_attend_shared(p, maps, head_dim, dtype, sms, as_stream(stream)), what);
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
  qwz::BatchAppendParams p{};
  const int rc = append_checked(p, k, v, k_cache, v_cache, k_scales, v_scales, slots, k_held, v_held, rows, k_stride,
                                v_stride, num_kv_heads, head_dim, num_pages, dtype);
  if (rc || p.rows == 0) return rc;
  return launched(qwz::launch_batch_append(p, dtype, as_stream(stream)), "qwz_batch_append");
}

int qwz_batch_append_rotated(const void* q, const void* k, const void* v, void* q_out, void* k_cache, void* v_cache,
                             void* k_scales, void* v_scales, const int32_t* slots, const int32_t* positions,
                             const float* inv_freq, const float* q_weight, const float* k_weight, void* k_held,
                             void* v_held, int64_t rows, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                             int64_t q_out_stride, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                             int32_t num_freqs, int32_t neighbours, float eps, int32_t num_pages, int32_t dtype,
                             void* stream) {
  qwz::BatchRotateParams p{};
  int rc = append_checked(p.kv, k, v, k_cache, v_cache, k_scales, v_scales, slots, k_held, v_held, rows, k_stride,
                          v_stride, num_kv_heads, head_dim, num_pages, dtype);
  if (rc) return rc;
  if (num_q_heads < 1 || num_q_heads > qwz::kRotMaxHeads) return fail(QWZ_EINVAL, "num_q_heads must be in 1..16384");
  if (num_freqs < 0 || num_freqs % 8 != 0 || 2 * num_freqs > head_dim)
    return fail(QWZ_EINVAL, "num_freqs must be a multiple of 8, at most head_dim / 2");
  if (!(eps >= 0.f) || !std::isfinite(eps)) return fail(QWZ_EINVAL, "eps must be finite and >= 0");
  if (rows == 0) return QWZ_OK;
  if (!q || !q_out || !aligned(q, 16) || !aligned(q_out, 16))
    return fail(QWZ_EINVAL, "q and q_out must be non-null 16-byte aligned pointers");
  if (!positions || (num_freqs > 0 && !inv_freq)) return fail(QWZ_EINVAL, "positions and inv_freq are required");
  if ((q_weight && !aligned(q_weight, 16)) || (k_weight && !aligned(k_weight, 16)))
    return fail(QWZ_EINVAL, "q_weight and k_weight must be 16-byte aligned");
  const int64_t width = (int64_t)num_q_heads * head_dim, kv_width = (int64_t)num_kv_heads * head_dim;
  if ((rc = check_row_stride(q_stride, width, "q"))) return rc;
  if ((rc = check_row_stride(q_out_stride, width, "q_out"))) return rc;
  // q may be rotated in place; nothing else that is read may be written
  if (!(q == q_out && q_stride == q_out_stride) && rows_meet(q, width, q_stride, q_out, width, q_out_stride, rows))
    return fail(QWZ_EINVAL, "q_out must be q itself or share no storage with it");
  if (rows_meet(q_out, width, q_out_stride, k, kv_width, k_stride, rows) ||
      rows_meet(q_out, width, q_out_stride, v, kv_width, v_stride, rows))
    return fail(QWZ_EINVAL, "q_out must not share storage with k or v");
  const void* held[] = {k_held, v_held};
  for (const void* h : held)
    if (row_meets(k, kv_width, k_stride, rows, h, 2 * rows * kv_width) ||
        row_meets(v, kv_width, v_stride, rows, h, 2 * rows * kv_width) ||
        row_meets(q, width, q_stride, rows, h, 2 * rows * kv_width) ||
        row_meets(q_out, width, q_out_stride, rows, h, 2 * rows * kv_width))
      return fail(QWZ_EINVAL, "k_held and v_held must not share storage with q, k, v or q_out");
  if (meet(k_held, 2 * rows * kv_width, v_held, 2 * rows * kv_width))
    return fail(QWZ_EINVAL, "k_held and v_held must not share storage");
  const struct {
    const void* at;
    int64_t n;
  } small[] = {{slots, 4 * rows}, {positions, 4 * rows}, {inv_freq, 4 * (int64_t)num_freqs}, {q_weight, 4 * (int64_t)head_dim},
               {k_weight, 4 * (int64_t)head_dim}},
    pool[] = {{k_cache, num_pages * qwz::kPage * kv_width / 2}, {v_cache, num_pages * qwz::kPage * kv_width / 2},
              {k_scales, num_pages * qwz::kPage * kv_width / 16}, {v_scales, num_pages * qwz::kPage * kv_width / 16}};
  bool clash = false;
  for (const auto& in : small) {
    clash |= row_meets(q_out, width, q_out_stride, rows, in.at, in.n);
    for (const void* h : held) clash |= meet(h, 2 * rows * kv_width, in.at, in.n);
    for (const auto& c : pool) clash |= meet(c.at, c.n, in.at, in.n);
  }
  for (const auto& c : pool) {
    clash |= row_meets(q, width, q_stride, rows, c.at, c.n) || row_meets(q_out, width, q_out_stride, rows, c.at, c.n) ||
             row_meets(k, kv_width, k_stride, rows, c.at, c.n) || row_meets(v, kv_width, v_stride, rows, c.at, c.n);
    for (const void* h : held) clash |= meet(h, 2 * rows * kv_width, c.at, c.n);
    for (const auto& d : pool) clash |= &c < &d && meet(c.at, c.n, d.at, d.n);
  }
  if (clash) return fail(QWZ_EINVAL, "outputs must not share storage with inputs or with each other");
  p.q = q;
  p.q_out = q_out;
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.q_stride = q_stride;
  p.q_out_stride = q_out_stride;
  p.q_heads = num_q_heads;
  p.freqs = num_freqs;
  p.neighbours = neighbours;
  p.eps = eps;
  return launched(qwz::launch_batch_rotate(p, dtype, as_stream(stream)), "qwz_batch_append_rotated");
}

int64_t qwz_batch_attend_workspace_bytes(int32_t head_dim) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
  return (int64_t)qwz::batch_workspace_bytes(head_dim);
}

int64_t qwz_batch_shared_workspace_bytes(int32_t head_dim, int32_t rows, int32_t num_q_heads) {
  if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || rows < 0 || num_q_heads < 1 || num_q_heads > 64 * 256)
    return 0;
  return (int64_t)qwz::batch_workspace_bytes(head_dim) + qwz::BatchSharedSpace(head_dim, rows, num_q_heads).bytes;
}

int qwz_batch_attend(const void* q, const void* k_cache, const void* v_cache, const void* k_scales,
                     const void* v_scales, const int32_t* block_table, const int32_t* cu_rows,
                     const int32_t* kv_lens, void* out, void* workspace, int64_t workspace_bytes, int32_t rows,
                     int32_t requests, int32_t max_rows, int32_t table_width, int32_t num_pages,
                     int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int64_t q_stride,
                     int64_t out_stride, float sm_scale, int32_t dtype, void* stream) {
  return attend_checked("qwz_batch_attend", nullptr, false, q, k_cache, v_cache, k_scales, v_scales, block_table, cu_rows,
                        kv_lens, out, workspace, workspace_bytes, rows, requests, max_rows, table_width, num_pages,
                        num_q_heads, num_kv_heads, head_dim, q_stride, out_stride, sm_scale, dtype, stream);
}

int qwz_batch_attend_shared(const void* q, const void* k_cache, const void* v_cache, const void* k_scales,
                            const void* v_scales, const int32_t* block_table, const int32_t* cu_rows,
                            const int32_t* kv_lens, const int32_t* plan, void* out, void* workspace,
                            int64_t workspace_bytes, int32_t rows, int32_t requests, int32_t max_rows,
                            int32_t table_width, int32_t num_pages, int32_t num_q_heads, int32_t num_kv_heads,
                            int32_t head_dim, int64_t q_stride, int64_t out_stride, float sm_scale, int32_t dtype,
                            void* stream) {
  return attend_checked("qwz_batch_attend_shared", plan, true, q, k_cache, v_cache, k_scales, v_scales, block_table,
                        cu_rows, kv_lens, out, workspace, workspace_bytes, rows, requests, max_rows, table_width,
                        num_pages, num_q_heads, num_kv_heads, head_dim, q_stride, out_stride, sm_scale, dtype, stream);
}

int qwz_batch_share_prefixes(const int32_t* prefix_of, const int32_t* kv_lens, const int32_t* cu_rows,
                             const int32_t* positions, const int32_t* request_of, int32_t* plan, int32_t* positions_out,
                             int32_t requests, int32_t rows, void* stream) {
  if (!prefix_of || !kv_lens || !cu_rows || !plan) return fail(QWZ_EINVAL, "prefix_of, kv_lens, cu_rows and plan are required");
  if (rows < 0) return fail(QWZ_EINVAL, "rows must be >= 0");
  if (rows > 0 && (!positions || !request_of || !positions_out))
    return fail(QWZ_EINVAL, "positions, request_of and positions_out are required");
  if (requests < 1 || requests > qwz::kShareMaxRequests) return fail(QWZ_EINVAL, "requests must be in 1..2^14");
  // every CTA reads all requests while others write (a row's position is read and written by one thread)
  const int64_t r4 = 4 * (int64_t)requests, t4 = 4 * (int64_t)rows, plan4 = 3 * r4 + 4 + t4;
  bool clash = meet(plan, plan4, positions_out, t4) || meet(plan, plan4, positions, t4) ||
               meet(positions_out, t4, request_of, t4) || meet(plan, plan4, request_of, t4) ||
               (positions_out != positions && meet(positions_out, t4, positions, t4));
  const struct {
    const int32_t* at;
    int64_t n;
  } reads[] = {{prefix_of, r4}, {kv_lens, r4}, {cu_rows, r4 + 4}};
  for (const auto& in : reads) clash |= meet(plan, plan4, in.at, in.n) || meet(positions_out, t4, in.at, in.n);
  if (clash) return fail(QWZ_EINVAL, "outputs must not share storage with inputs");
  const int sms = batch_sms();
  if (sms <= 0) return fail(QWZ_ELAUNCH, "no CUDA device");
  qwz::BatchShareParams p{};
  p.prefix_of = prefix_of;
  p.kv_lens = kv_lens;
  p.cu_rows = cu_rows;
  p.positions = positions;
  p.request_of = request_of;
  p.cu_shared = plan;
  p.reads = p.cu_shared + requests + 1;
  p.alone = p.reads + requests;
  p.shared_rows = p.alone + requests;
  p.positions_out = positions_out;
  p.requests = requests;
  p.rows = rows;
  return launched(qwz::launch_batch_share(p, sms, as_stream(stream)), "qwz_batch_share_prefixes");
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
