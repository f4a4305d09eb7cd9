// The gawee_kv entry points of include/gawee_cuda.h: argument checks, scratch
// memory and launches of the paged key/value cache kernels.
#include <cuda_runtime.h>

#include <cstdint>
#include <exception>
#include <string>

#include "../../../include/gawee_cuda.h"
#include "../kernels/paged_kv.h"

namespace gawee {
void set_thread_error(const std::string& msg);  // runtime.cpp: read back by gawee_last_error(NULL, ...)
std::string device_status_text(int st);
}  // namespace gawee

struct gawee_kv {
  gawee_kv_desc desc{};
  gawee::kern::PageGeom geom{};
  int device = -1;
  int sms = 0;
  void* memory = nullptr;      // one allocation, of which the rest are parts
  int* status = nullptr;       // first error a kernel reported (kern::Status)
  int32_t* plan = nullptr;     // [max_batch][2]: evict's lengths before and after
  float* stats = nullptr;      // [max_batch][heads][2], with desc.weights
  float* scores = nullptr;     // [max_batch][heads][max_pages * page_size], with desc.weights
  float* parts = nullptr;      // attend's partial states
  int2* info = nullptr;        // attend's segments and the blocks that share them
  int2* splits = nullptr;      // .. and its blocks and the segments that they leave unfinished
  ~gawee_kv() { cudaFree(memory); }
};

namespace {

using gawee::kern::PageGeom;

gawee_status fail(gawee_status st, const std::string& what) {
  gawee::set_thread_error(what);
  return st;
}

// No exception crosses the C interface.
template <class F>
gawee_status guarded(const char* name, F&& f) {
  try {
    return f();
  } catch (const std::exception& e) {
    return fail(GAWEE_ERR_INVALID, std::string(name) + ": " + e.what());
  } catch (...) {
    return fail(GAWEE_ERR_INVALID, std::string(name) + ": unknown error");
  }
}

// Makes the handle's device current and puts the caller's back.
struct DeviceScope {
  int before = -1;
  cudaError_t err;
  explicit DeviceScope(int device) {
    err = cudaGetDevice(&before);
    if (err == cudaSuccess && before != device) err = cudaSetDevice(device);
    else before = -1;
  }
  ~DeviceScope() {
    if (before >= 0) cudaSetDevice(before);
  }
};

bool is_act(int dt) { return dt == GAWEE_F32 || dt == GAWEE_F16 || dt == GAWEE_BF16; }
int size_of(int dt) { return dt == GAWEE_F32 ? 4 : 2; }
bool aligned(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(n - 1)) == 0; }

// What every call has: pages and a table for `batch` sequences.
std::string check_common(const gawee_kv* kv, const void* k_pages, const void* v_pages, int batch,
                         const int32_t* table, int64_t table_stride, int table_cols) {
  if (batch == 0) return "";
  if (!k_pages || !v_pages) return "null pages";
  if (!aligned(k_pages, 16) || !aligned(v_pages, 16)) return "pages are not 16-byte aligned";
  if (k_pages == v_pages) return "k_pages and v_pages are the same";
  if (batch < 0 || batch > kv->desc.max_batch)
    return "batch " + std::to_string(batch) + " outside 0 .. " + std::to_string(kv->desc.max_batch);
  if (!table || !aligned(table, 4)) return "null or unaligned block table";
  if (table_cols < 1 || table_cols > kv->desc.max_pages)
    return "table_cols " + std::to_string(table_cols) + " outside 1 .. " + std::to_string(kv->desc.max_pages);
  if (table_stride < table_cols && batch > 1) return "block table rows overlap";
  return "";
}

// A weights array [batch][kv_heads][cols]: rows that do not overlap.
std::string check_weights(const gawee_kv* kv, const void* p, int64_t stride, int64_t batch_stride, int64_t cols,
                          int batch, const char* name) {
  if (!aligned(p, 4)) return std::string(name) + " is not 4-byte aligned";
  if (cols < 1) return "weights_cols is below 1";
  if ((kv->geom.kv_heads > 1 && stride < cols) || stride < 0) return std::string(name) + " rows overlap";
  if (batch > 1 && batch_stride < (kv->geom.kv_heads - 1) * stride + cols) return std::string(name) + " sequences overlap";
  return "";
}

gawee_status finish(const char* name, cudaError_t e) {
  if (e == cudaSuccess) return GAWEE_OK;
  return fail(GAWEE_ERR_CUDA, std::string(name) + ": launch: " + cudaGetErrorString(e));
}

template <class F>
gawee_status run_on(const gawee_kv* kv, const char* name, F&& launch) {
  if (kv->device < 0) return fail(GAWEE_ERR_CUDA, std::string(name) + ": the handle has no device");
  DeviceScope scope(kv->device);
  if (scope.err != cudaSuccess) return finish(name, scope.err);
  return finish(name, launch());
}

}  // namespace

extern "C" {

gawee_status gawee_kv_create(const gawee_kv_desc* desc, int device, gawee_kv** out) {
  static const char* kName = "gawee_kv_create";
  if (!out) return fail(GAWEE_ERR_INVALID, std::string(kName) + ": null out");
  *out = nullptr;
  return guarded(kName, [&]() -> gawee_status {
    auto bad = [&](const std::string& m) { return fail(GAWEE_ERR_INVALID, std::string(kName) + ": " + m); };
    if (!desc) return bad("null desc");
    const gawee_kv_desc& d = *desc;
    if (!is_act(d.dtype)) return bad("dtype must be f32, f16 or bf16");
    if (d.kv_heads < 1 || d.heads < d.kv_heads || d.heads > 4096 || d.heads % d.kv_heads)
      return bad("heads must be a positive multiple of kv_heads, up to 4096");
    if (d.head_dim < 8 || d.head_dim > 256 || d.head_dim % 8) return bad("head_dim must be a multiple of 8 up to 256");
    if (d.page_size < 1 || d.page_size > 65536) return bad("page_size must be 1 .. 65536");
    if (d.num_pages < 1 || d.num_pages > INT32_MAX) return bad("num_pages must be 1 .. 2^31 - 1");
    const int64_t page = (int64_t)d.kv_heads * d.page_size * d.head_dim;
    const int64_t stride = d.page_stride ? d.page_stride : page;
    if (stride < page) return bad("page_stride is below the page's size");
    if (stride * size_of(d.dtype) % 16) return bad("page_stride is not a multiple of 16 bytes");
    if (stride > (INT64_MAX / 4) / d.num_pages) return bad("the pages pass 2^63 bytes");
    if (d.max_batch < 1 || d.max_batch > 65535) return bad("max_batch must be 1 .. 65535");
    // lengths are int32; the kernels step past the last row by less than 2^20
    if (d.max_pages < 1 || (int64_t)d.max_pages * d.page_size > INT32_MAX - (1 << 20))
      return bad("max_pages * page_size must be 1 .. 2^31 - 2^20");
    auto kv = new gawee_kv();
    struct Drop {
      gawee_kv* kv;
      ~Drop() { delete kv; }
    } drop{kv};
    kv->desc = d;
    kv->geom = PageGeom{stride, d.num_pages, d.kv_heads, d.page_size, d.head_dim};
    kv->device = device;
    if (device == -1) {
      *out = kv;
      drop.kv = nullptr;
      return GAWEE_OK;
    }
    int n = 0;
    cudaError_t e = cudaGetDeviceCount(&n);
    if (e != cudaSuccess) return fail(GAWEE_ERR_CUDA, std::string(kName) + ": " + cudaGetErrorString(e));
    if (device < 0 || device >= n) return bad("invalid device index");
    DeviceScope scope(device);
    e = scope.err;
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&kv->sms, cudaDevAttrMultiProcessorCount, device);
    const int group = d.heads / d.kv_heads;
    const size_t rows = (size_t)d.max_batch * d.heads;
    size_t bytes = 0;
    auto place = [&](size_t n) {
      const size_t at = bytes;
      bytes += (n + 255) / 256 * 256;
      return at;
    };
    const size_t status = place(sizeof(int)), plan = place(sizeof(int32_t) * 2 * d.max_batch);
    const size_t parts = place(sizeof(float) * gawee::kern::kv_parts_floats(kv->sms, group, d.head_dim));
    const size_t info = place(sizeof(int2) * gawee::kern::kv_segments(d.max_batch, d.kv_heads, group));
    const size_t splits = place(sizeof(int2) * gawee::kern::kv_blocks(kv->sms));
    const size_t stats = place(d.weights ? sizeof(float) * 2 * rows : 0);
    const size_t scores = place(d.weights ? sizeof(float) * rows * d.max_pages * d.page_size : 0);
    if (e == cudaSuccess) e = cudaMalloc(&kv->memory, bytes);
    if (e == cudaSuccess) {
      char* m = static_cast<char*>(kv->memory);
      kv->status = reinterpret_cast<int*>(m + status);
      kv->plan = reinterpret_cast<int32_t*>(m + plan);
      kv->parts = reinterpret_cast<float*>(m + parts);
      kv->info = reinterpret_cast<int2*>(m + info);
      kv->splits = reinterpret_cast<int2*>(m + splits);
      if (d.weights) {
        kv->stats = reinterpret_cast<float*>(m + stats);
        kv->scores = reinterpret_cast<float*>(m + scores);
      }
      e = cudaMemset(kv->status, 0, sizeof(int));
    }
    if (e == cudaSuccess) e = cudaStreamSynchronize(nullptr);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return fail(e == cudaErrorMemoryAllocation ? GAWEE_ERR_OOM : GAWEE_ERR_CUDA,
                  std::string(kName) + ": " + cudaGetErrorString(e));
    }
    *out = kv;
    drop.kv = nullptr;
    return GAWEE_OK;
  });
}

void gawee_kv_destroy(gawee_kv* kv) {
  if (!kv) return;
  if (kv->device < 0) {
    delete kv;
    return;
  }
  DeviceScope scope(kv->device);
  cudaDeviceSynchronize();
  delete kv;
}

gawee_status gawee_kv_append(gawee_kv* kv, const gawee_kv_append_args* a, void* stream) {
  static const char* kName = "gawee_kv_append";
  return guarded(kName, [&]() -> gawee_status {
    auto bad = [&](const std::string& m) { return fail(GAWEE_ERR_INVALID, std::string(kName) + ": " + m); };
    if (!kv || !a) return bad("null handle or arguments");
    std::string m = check_common(kv, a->k_pages, a->v_pages, a->batch, a->block_table, a->table_stride, a->table_cols);
    if (!m.empty()) return bad(m);
    if (!is_act(a->dtype)) return bad("dtype must be f32, f16 or bf16");
    if (a->batch == 0 && a->tokens > 0) return bad("tokens without a sequence");
    if (a->tokens < 0 || a->tokens > INT32_MAX) return bad("tokens outside 0 .. 2^31 - 1");
    if (a->tokens == 0) return GAWEE_OK;
    if (!a->k || !a->v || !a->positions) return bad("null k, v or positions");
    if (!aligned(a->k, size_of(a->dtype)) || !aligned(a->v, size_of(a->dtype)))
      return bad("k or v is not aligned to its type");
    if (!aligned(a->positions, 4) || !aligned(a->sequences, 4)) return bad("positions or sequences is not 4-byte aligned");
    if (!a->sequences && a->tokens > a->batch) return bad("more tokens than sequences, and no `sequences`");
    const int64_t row = (int64_t)kv->geom.kv_heads * kv->geom.head_dim;
    if (a->tokens > 1 && (a->k_stride < row || a->v_stride < row)) return bad("k or v rows overlap");
    gawee::kern::KvAppendParams p{};
    p.geom = kv->geom;
    p.k_pages = a->k_pages;
    p.v_pages = a->v_pages;
    p.page_dt = kv->desc.dtype;
    p.k = a->k;
    p.v = a->v;
    p.dt = a->dtype;
    p.k_stride = a->k_stride;
    p.v_stride = a->v_stride;
    p.tokens = a->tokens;
    p.sequences = a->sequences;
    p.positions = a->positions;
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.table_cols = a->table_cols;
    p.batch = a->batch;
    p.status = kv->status;
    return run_on(kv, kName, [&] { return launch_kv_append(p, static_cast<cudaStream_t>(stream)); });
  });
}

gawee_status gawee_kv_attend(gawee_kv* kv, const gawee_kv_attend_args* a, void* stream) {
  static const char* kName = "gawee_kv_attend";
  return guarded(kName, [&]() -> gawee_status {
    auto bad = [&](const std::string& m) { return fail(GAWEE_ERR_INVALID, std::string(kName) + ": " + m); };
    if (!kv || !a) return bad("null handle or arguments");
    std::string m = check_common(kv, a->k_pages, a->v_pages, a->batch, a->block_table, a->table_stride, a->table_cols);
    if (!m.empty()) return bad(m);
    if (!is_act(a->dtype)) return bad("dtype must be f32, f16 or bf16");
    if (a->batch == 0) return GAWEE_OK;
    if (!a->q || !a->out || !a->lengths) return bad("null q, out or lengths");
    const int es = size_of(a->dtype);
    if (!aligned(a->q, es) || !aligned(a->out, es) || !aligned(a->k, es) || !aligned(a->v, es))
      return bad("q, out, k or v is not aligned to its type");
    if (!aligned(a->lengths, 4)) return bad("lengths is not 4-byte aligned");
    if (!(a->scale == a->scale) || a->scale - a->scale != 0.f) return bad("scale is not finite");
    const int64_t qrow = (int64_t)kv->desc.heads * kv->geom.head_dim, row = (int64_t)kv->geom.kv_heads * kv->geom.head_dim;
    if (a->batch > 1 && (a->q_stride < qrow || a->out_stride < qrow)) return bad("q or out rows overlap");
    if (!a->k != !a->v) return bad("k without v");
    if (a->k && a->batch > 1 && (a->k_stride < row || a->v_stride < row)) return bad("k or v rows overlap");
    int64_t max_len = (int64_t)a->table_cols * kv->geom.page_size;
    if (a->mask) {
      if (!aligned(a->mask, 4)) return bad("mask is not 4-byte aligned");
      if (a->mask_cols < 1) return bad("mask_cols is below 1");
      // stride 0: one mask for every sequence
      if (a->batch > 1 && a->mask_stride != 0 && a->mask_stride < a->mask_cols) return bad("mask rows overlap");
      max_len = max_len < a->mask_cols ? max_len : a->mask_cols;
    }
    if (a->weights && !a->weights_out) return bad("weights without weights_out");
    if (a->weights_out) {
      if (!kv->desc.weights) return bad("the handle was created without `weights`");
      m = check_weights(kv, a->weights_out, a->weights_out_stride, a->weights_out_batch_stride, a->weights_cols, a->batch,
                        "weights_out");
      if (m.empty() && a->weights)
        m = check_weights(kv, a->weights, a->weights_stride, a->weights_batch_stride, a->weights_cols, a->batch, "weights");
      if (!m.empty()) return bad(m);
      if (a->weights == a->weights_out && (a->weights_stride != a->weights_out_stride ||
                                           a->weights_batch_stride != a->weights_out_batch_stride))
        return bad("weights in place with other strides");
      max_len = max_len < a->weights_cols ? max_len : a->weights_cols;
    }
    gawee::kern::KvAttendParams p{};
    p.geom = kv->geom;
    p.k_pages = a->k_pages;
    p.v_pages = a->v_pages;
    p.page_dt = kv->desc.dtype;
    p.q = a->q;
    p.out = a->out;
    p.dt = a->dtype;
    p.q_stride = a->q_stride;
    p.out_stride = a->out_stride;
    p.batch = a->batch;
    p.heads = kv->desc.heads;
    p.scale = a->scale;
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.table_cols = a->table_cols;
    p.lengths = a->lengths;
    p.max_len = max_len;
    p.k = a->k;
    p.v = a->v;
    p.k_stride = a->k_stride;
    p.v_stride = a->v_stride;
    p.mask = a->mask;
    p.mask_stride = a->mask_stride;
    p.weights = a->weights;
    p.weights_out = a->weights_out;
    p.w_stride = a->weights_stride;
    p.w_batch = a->weights_batch_stride;
    p.wo_stride = a->weights_out_stride;
    p.wo_batch = a->weights_out_batch_stride;
    p.scores = kv->scores;
    p.stats = kv->stats;
    p.parts = kv->parts;
    p.info = kv->info;
    p.splits = kv->splits;
    p.device = kv->device;
    p.sms = kv->sms;
    p.page_shift = gawee::kern::page_shift_of(kv->geom.page_size);
    p.status = kv->status;
    return run_on(kv, kName, [&] { return launch_kv_attend(p, static_cast<cudaStream_t>(stream)); });
  });
}

gawee_status gawee_kv_evict(gawee_kv* kv, const gawee_kv_evict_args* a, void* stream) {
  static const char* kName = "gawee_kv_evict";
  return guarded(kName, [&]() -> gawee_status {
    auto bad = [&](const std::string& m) { return fail(GAWEE_ERR_INVALID, std::string(kName) + ": " + m); };
    if (!kv || !a) return bad("null handle or arguments");
    std::string m = check_common(kv, a->k_pages, a->v_pages, a->batch, a->block_table, a->table_stride, a->table_cols);
    if (!m.empty()) return bad(m);
    // the kernels step past the last kept row by less than 2^24
    if (a->budget < 1 || a->budget > INT32_MAX - (1 << 24)) return bad("budget is below 1, or 2^31 - 2^24 or more");
    if (a->recent < 0 || a->recent > a->budget) return bad("recent outside 0 .. budget");
    if (a->batch == 0) return GAWEE_OK;
    if (!a->weights || !a->weights_out || !a->lengths || !a->lengths_out || !a->kept)
      return bad("null weights, weights_out, lengths, lengths_out or kept");
    if (!aligned(a->lengths, 4) || !aligned(a->lengths_out, 4) || !aligned(a->kept, 4))
      return bad("lengths, lengths_out or kept is not 4-byte aligned");
    m = check_weights(kv, a->weights, a->weights_stride, a->weights_batch_stride, a->weights_cols, a->batch, "weights");
    if (m.empty())
      m = check_weights(kv, a->weights_out, a->weights_out_stride, a->weights_out_batch_stride, a->weights_cols, a->batch,
                        "weights_out");
    if (!m.empty()) return bad(m);
    if (a->weights == a->weights_out && (a->weights_stride != a->weights_out_stride ||
                                         a->weights_batch_stride != a->weights_out_batch_stride))
      return bad("weights in place with other strides");
    int64_t max_len = (int64_t)a->table_cols * kv->geom.page_size;
    max_len = max_len < a->weights_cols ? max_len : a->weights_cols;
    if (a->to_table) {
      if (!aligned(a->to_table, 4)) return bad("to_table is not 4-byte aligned");
      if (a->to_table == a->block_table) return bad("to_table is block_table: leave it out to evict in place");
      if (a->to_cols < 1 || a->to_cols > kv->desc.max_pages) return bad("to_cols outside 1 .. max_pages");
      if (a->batch > 1 && a->to_stride < a->to_cols) return bad("to_table rows overlap");
    }
    gawee::kern::KvEvictParams p{};
    p.geom = kv->geom;
    p.k_pages = a->k_pages;
    p.v_pages = a->v_pages;
    p.page_dt = kv->desc.dtype;
    p.weights = a->weights;
    p.weights_out = a->weights_out;
    p.w_stride = a->weights_stride;
    p.w_batch = a->weights_batch_stride;
    p.wo_stride = a->weights_out_stride;
    p.wo_batch = a->weights_out_batch_stride;
    p.table = a->block_table;
    p.table_stride = a->table_stride;
    p.table_cols = a->table_cols;
    p.to_table = a->to_table;
    p.to_stride = a->to_stride;
    p.to_cols = a->to_cols;
    p.lengths = a->lengths;
    p.lengths_out = a->lengths_out;
    p.max_len = max_len;
    p.batch = a->batch;
    p.budget = a->budget;
    p.recent = a->recent;
    p.kept = a->kept;
    p.plan = kv->plan;
    p.sms = kv->sms;
    p.status = kv->status;
    return run_on(kv, kName, [&] { return launch_kv_evict(p, static_cast<cudaStream_t>(stream)); });
  });
}

gawee_status gawee_kv_synchronize(gawee_kv* kv, void* stream) {
  static const char* kName = "gawee_kv_synchronize";
  return guarded(kName, [&]() -> gawee_status {
    if (!kv) return fail(GAWEE_ERR_INVALID, std::string(kName) + ": null handle");
    int st = 0;
    const gawee_status ok = run_on(kv, kName, [&] {
      cudaStream_t s = static_cast<cudaStream_t>(stream);
      cudaError_t e = cudaStreamSynchronize(s);
      if (e == cudaSuccess) e = cudaMemcpyAsync(&st, kv->status, sizeof(int), cudaMemcpyDeviceToHost, s);
      if (e == cudaSuccess) e = cudaStreamSynchronize(s);
      if (e == cudaSuccess && st) e = cudaMemsetAsync(kv->status, 0, sizeof(int), s);
      if (e == cudaSuccess && st) e = cudaStreamSynchronize(s);
      return e;
    });
    if (ok != GAWEE_OK) return ok;
    return st ? fail(GAWEE_ERR_DEVICE, gawee::device_status_text(st)) : GAWEE_OK;
  });
}

}  // extern "C"
