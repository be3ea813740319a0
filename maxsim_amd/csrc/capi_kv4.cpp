// capi_kv4.cpp -- C ABI of the 4-bit key/value cache (kv4_rows.hip,
// kv4_attend.hip, kv4_keep.hip): argument checks and launches.  The pool, the batch and the
// workspace are the caller's device memory.
#include <algorithm>
#include <climits>
#include <cmath>

#include "capi_internal.hpp"
#include "kv4.hpp"

using namespace msim;

namespace {

constexpr int64_t kMaxRows = int64_t{1} << 26;  // of a call: keeps every launch within the grid limits
constexpr double kLog2e = 1.4426950408889634;
// The kernels hold key positions in 32 bits and look ahead of a sequence's end by up
// to 640 keys (the tiles on their way, the page numbers of the next ones).
constexpr int64_t kMostKeys = INT_MAX - 4096;

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

Kv4Pool check_pool(const msim_kv4_pool* p) {
  if (p == nullptr) throw InvalidArgument("pool must not be NULL");
  if (p->dim != 64 && p->dim != 96 && p->dim != 128 && p->dim != 192 && p->dim != 256)
    throw NotSupported("head_dim must be 64, 96, 128, 192 or 256");
  if (p->page_size < 16 || p->page_size > 65536 || (p->page_size & (p->page_size - 1)) != 0)
    throw InvalidArgument("page_size must be a power of two from 16 to 65536");
  if (p->num_pages < 1 || p->num_pages > INT_MAX) throw InvalidArgument("num_pages must be positive");
  if (p->kv_heads < 1 || p->kv_heads > 1024) throw InvalidArgument("kv_heads must be between 1 and 1024");
  if (!p->k_codes || !p->v_codes || !p->k_scales || !p->v_scales)
    throw InvalidArgument("pool pointers must not be NULL");
  if (!aligned(p->k_codes, 16) || !aligned(p->v_codes, 16) || !aligned(p->k_scales, 16) || !aligned(p->v_scales, 16))
    throw InvalidArgument("pool pointers must be 16-byte aligned");
  Kv4Pool pool{};
  pool.codes[0] = p->k_codes;
  pool.codes[1] = p->v_codes;
  pool.scales[0] = p->k_scales;
  pool.scales[1] = p->v_scales;
  pool.num_pages = (int32_t)p->num_pages;
  pool.page_shift = __builtin_ctz((unsigned)p->page_size);
  pool.kv_heads = p->kv_heads;
  pool.dim = p->dim;
  return pool;
}

Kv4Batch check_batch(const Kv4Pool& pool, const int32_t* table, const int32_t* lengths, const int32_t* offsets,
                     int64_t batch, int64_t max_pages, int64_t rows) {
  if (batch < 0 || rows < 0 || max_pages < 0) throw InvalidArgument("batch, max_pages and rows must not be negative");
  if (rows > kMaxRows || batch > kMaxRows) throw NotSupported("a call takes at most 2^26 rows and sequences");
  if (max_pages > kMostKeys >> pool.page_shift)
    throw NotSupported("a page table holds sequences of less than 2^31 - 4096 tokens");
  if (offsets == nullptr && rows != batch)
    throw InvalidArgument("without offsets there is one row per sequence");
  if (batch > 0 && (lengths == nullptr || (table == nullptr && max_pages > 0)))
    throw InvalidArgument("page_table and lengths must not be NULL");
  return Kv4Batch{table, lengths, offsets, (int32_t)batch, (int32_t)max_pages, (int32_t)rows};
}

Kv4Type check_type(int type) {
  if (type != MSIM_F32 && type != MSIM_F16 && type != MSIM_BF16)
    throw InvalidArgument("type must be MSIM_F32, MSIM_F16 or MSIM_BF16");
  return static_cast<Kv4Type>(type);
}

void check_rows(const void* p, Kv4Type type, const char* what) {
  if (p == nullptr) throw InvalidArgument(std::string(what) + " must not be NULL");
  if (!aligned(p, type == kKv4F32 ? 4 : 2)) throw InvalidArgument(std::string(what) + " must be aligned to its type");
}

void check_heads(const Kv4Pool& pool, const Kv4Batch& batch, int64_t heads) {
  if (heads < 1 || heads % pool.kv_heads != 0) throw InvalidArgument("heads must be a multiple of kv_heads");
  if (heads > 16384 || ((int64_t)batch.rows + batch.batch) * heads >= int64_t{1} << 30)
    throw NotSupported("at most 16384 heads, and less than 2^30 of (rows + batch) * heads");
}

int rows_call(const msim_kv4_pool* pool, const int32_t* table, const int32_t* lengths, const int32_t* offsets,
              int64_t batch, int64_t max_pages, int64_t rows, const Kv4Rows kv[2], int type, bool append,
              void* stream) {
  return guarded([&] {
    const Kv4Pool p = check_pool(pool);
    const Kv4Batch b = check_batch(p, table, lengths, offsets, batch, max_pages, rows);
    const Kv4Type t = check_type(type);
    if (rows == 0) return;
    check_rows(kv[0].ptr, t, "k");
    check_rows(kv[1].ptr, t, "v");
    check_hip(append ? launch_kv4_append(p, b, kv, t, as_stream(stream)) : launch_kv4_read(p, b, kv, t, as_stream(stream)),
              append ? "launch cache append kernel" : "launch cache read kernel");
  });
}

}  // namespace

extern "C" int msim_kv4_append_async(const msim_kv4_pool* pool, const int32_t* page_table, const int32_t* lengths,
                                     const int32_t* offsets, int64_t batch, int64_t max_pages, int64_t rows,
                                     const void* k, int64_t k_row_stride, int64_t k_head_stride, const void* v,
                                     int64_t v_row_stride, int64_t v_head_stride, int type, void* stream) {
  const Kv4Rows kv[2] = {{const_cast<void*>(k), k_row_stride, k_head_stride},
                         {const_cast<void*>(v), v_row_stride, v_head_stride}};
  return rows_call(pool, page_table, lengths, offsets, batch, max_pages, rows, kv, type, true, stream);
}

extern "C" int msim_kv4_read_async(const msim_kv4_pool* pool, const int32_t* page_table, const int32_t* lengths,
                                   const int32_t* offsets, int64_t batch, int64_t max_pages, int64_t rows, void* k,
                                   int64_t k_row_stride, int64_t k_head_stride, void* v, int64_t v_row_stride,
                                   int64_t v_head_stride, int type, void* stream) {
  const Kv4Rows kv[2] = {{k, k_row_stride, k_head_stride}, {v, v_row_stride, v_head_stride}};
  return rows_call(pool, page_table, lengths, offsets, batch, max_pages, rows, kv, type, false, stream);
}

extern "C" int msim_kv4_attend_workspace(const msim_kv4_pool* pool, int64_t batch, int64_t max_pages, int64_t rows,
                                         int64_t heads, uint64_t* bytes) {
  return msim_kv4_attend_ex_workspace(pool, batch, max_pages, rows, heads, 0, bytes);
}

extern "C" int msim_kv4_attend_ex_workspace(const msim_kv4_pool* pool, int64_t batch, int64_t max_pages, int64_t rows,
                                            int64_t heads, int parents, uint64_t* bytes) {
  return guarded([&] {
    if (bytes == nullptr) throw InvalidArgument("bytes must not be NULL");
    const Kv4Pool p = check_pool(pool);
    static const int32_t present = 0;  // only the sizes count here
    const Kv4Batch b = check_batch(p, &present, &present, &present, batch, max_pages, rows);
    check_heads(p, b, heads);
    *bytes = kv4_attend_workspace(p, b, (int)heads, parents != 0, device_cu_count());
  });
}

extern "C" int msim_kv4_attend_async(const msim_kv4_pool* pool, const int32_t* page_table, const int32_t* lengths,
                                     const int32_t* offsets, int64_t batch, int64_t max_pages, int64_t rows,
                                     const void* q, int64_t q_row_stride, int64_t q_head_stride, int64_t heads,
                                     int type, double scale, int causal, int64_t window, const uint8_t* mask,
                                     int64_t mask_row_stride, int64_t mask_width, void* out, int64_t out_row_stride,
                                     int64_t out_head_stride, float* lse, void* workspace, uint64_t workspace_bytes,
                                     void* stream) {
  return msim_kv4_attend_ex_async(pool, page_table, lengths, offsets, batch, max_pages, rows, q, q_row_stride,
                                  q_head_stride, heads, type, scale, causal, window, mask, mask_row_stride, mask_width,
                                  0, nullptr, out, out_row_stride, out_head_stride, lse, workspace, workspace_bytes,
                                  stream);
}

extern "C" int msim_kv4_attend_ex_async(const msim_kv4_pool* pool, const int32_t* page_table, const int32_t* lengths,
                                        const int32_t* offsets, int64_t batch, int64_t max_pages, int64_t rows,
                                        const void* q, int64_t q_row_stride, int64_t q_head_stride, int64_t heads,
                                        int type, double scale, int causal, int64_t window, const uint8_t* mask,
                                        int64_t mask_row_stride, int64_t mask_width, int64_t sinks,
                                        const int32_t* parents, void* out, int64_t out_row_stride,
                                        int64_t out_head_stride, float* lse, void* workspace, uint64_t workspace_bytes,
                                        void* stream) {
  return guarded([&] {
    const Kv4Pool p = check_pool(pool);
    const Kv4Batch b = check_batch(p, page_table, lengths, offsets, batch, max_pages, rows);
    const Kv4Type t = check_type(type);
    check_heads(p, b, heads);
    const float scale_log2 = (float)(scale * kLog2e);
    if (!std::isfinite(scale_log2)) throw InvalidArgument("scale must be finite in single precision");
    if (window < 0) throw InvalidArgument("window must not be negative");
    if (mask != nullptr && mask_width < 0) throw InvalidArgument("mask width must not be negative");
    if (sinks < 0) throw InvalidArgument("sinks must not be negative");
    if (parents != nullptr && causal == 0) throw InvalidArgument("parents need a causal call");
    if (rows == 0) return;
    check_rows(q, t, "q");
    check_rows(out, t, "out");
    const int cus = device_cu_count();
    size_t need = kv4_attend_workspace(p, b, (int)heads, false, cus);
    if (parents != nullptr) need = std::min(need, kv4_attend_workspace(p, b, (int)heads, true, cus));
    if (need > 0 && (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < need))
      throw InvalidArgument("workspace is smaller than msim_kv4_attend_workspace asks for, or not 16-byte aligned");
    Kv4AttendArgs a{};
    a.q = q;
    a.q_row_stride = q_row_stride;
    a.q_head_stride = q_head_stride;
    a.out = out;
    a.out_row_stride = out_row_stride;
    a.out_head_stride = out_head_stride;
    a.lse = lse;
    a.mask = mask;
    a.mask_row_stride = mask_row_stride;
    a.mask_width = mask_width;
    const int64_t size = t == kKv4F32 ? 4 : 2;
    a.q_wide = aligned(q, 16) && q_row_stride * size % 16 == 0 && q_head_stride * size % 16 == 0;
    a.out_wide = aligned(out, 4 * size) && out_row_stride % 4 == 0 && out_head_stride % 4 == 0;
    a.heads = (int32_t)heads;
    a.causal = causal != 0;
    a.window = window == 0 || window > INT_MAX ? INT_MAX : (int32_t)window;
    a.sinks = a.window == INT_MAX ? 0 : (int32_t)std::min<int64_t>(sinks, INT_MAX);
    a.parents = parents;
    a.scale_log2 = scale_log2;
    check_hip(launch_kv4_attend(p, b, a, t, workspace, workspace_bytes, cus, as_stream(stream)),
              "launch cache attention kernels");
  });
}

extern "C" int msim_kv4_keep_async(const msim_kv4_pool* pool, const int32_t* page_table, const int32_t* lengths,
                                   const int32_t* offsets, int64_t batch, int64_t max_pages, int64_t rows,
                                   const int32_t* kept, int64_t width, int32_t* new_lengths, void* stream) {
  return guarded([&] {
    const Kv4Pool p = check_pool(pool);
    const Kv4Batch b = check_batch(p, page_table, lengths, offsets, batch, max_pages, rows);
    if (width < 0) throw InvalidArgument("width must not be negative");
    if (width > kMaxRows || batch > int64_t{1} << 20) throw NotSupported("a call keeps rows of at most 2^20 sequences");
    if (batch == 0) return;
    if (new_lengths == nullptr || (kept == nullptr && width > 0))
      throw InvalidArgument("kept and new_lengths must not be NULL");
    check_hip(launch_kv4_keep(p, b, kept, (int)width, new_lengths, as_stream(stream)), "launch cache keep kernel");
  });
}
