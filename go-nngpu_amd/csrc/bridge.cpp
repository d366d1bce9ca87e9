// bridge.cpp — extern "C" entry points of libgonngpu.so (declared in include/gonngpu.h).
// Part 1 keeps the reference bridge's names, signatures and return codes
// (internal/cgo/metal_bridge*.m); Part 2 is the device-pointer API.
#include <atomic>
#include <chrono>
#include <cstdlib>
#include <cstring>
#include <memory>
#include <thread>
#include <unordered_map>
#include <vector>

#include "common.h"
#include "adjust.h"
#include "int8.h"
#include "logits.h"
#include "mxfp4.h"

using gn::Buffer;
using gn::set_error;

namespace {

struct Scratch {  // device scratch released on scope exit (after the stream is synchronized)
  void *p = nullptr;
  ~Scratch() { gn::dev_free(p); }
};

// Idle completion events of sync(), created on demand and kept for the life of the process
// (one per thread that has waited at the same time).
std::mutex g_sync_mu;
std::vector<hipEvent_t> g_sync_events;

hipError_t take_sync_event(hipEvent_t *ev) {
  {
    std::lock_guard<std::mutex> lk(g_sync_mu);
    if (!g_sync_events.empty()) {
      *ev = g_sync_events.back();
      g_sync_events.pop_back();
      return hipSuccess;
    }
  }
  return hipEventCreateWithFlags(ev, hipEventDisableTiming);
}

void give_sync_event(hipEvent_t ev) {
  std::lock_guard<std::mutex> lk(g_sync_mu);
  g_sync_events.push_back(ev);
}

// Waits for the work enqueued on s, as the reference's waitUntilCompleted does. A timing-free
// event recorded behind that work is polled for up to 5 ms, then waited on: the blocking wait's
// wake-up is slower (the C5 SpMM through perform_sparse_dense_matmul took 0.400 ms per
// synchronous call with it alone and 0.385 ms with the polling, against 0.366 ms of kernels), and
// polling the stream itself (hipStreamQuery) is slower still for short work: a 1-element kernel's
// synchronous round trip took 26.6 us that way against 12.7 us through the event, the C5 SpMV
// 27.7 against 22.2 us. A capturing stream has no completion to wait for and is an error, as
// hipStreamQuery reports it.
int sync(hipStream_t s, CError *err, int code) {
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  hipError_t e = hipStreamIsCapturing(s, &cap);
  if (e == hipSuccess && cap != hipStreamCaptureStatusNone) e = hipErrorStreamCaptureUnsupported;
  hipEvent_t ev = nullptr;
  if (e == hipSuccess) e = take_sync_event(&ev);
  if (e == hipSuccess) e = hipEventRecord(ev, s);
  if (e == hipSuccess) {
    const auto t0 = std::chrono::steady_clock::now();
    while ((e = hipEventQuery(ev)) == hipErrorNotReady) {
      if (std::chrono::steady_clock::now() - t0 > std::chrono::milliseconds(5)) {
        e = hipEventSynchronize(ev);
        break;
      }
      std::this_thread::yield();  // threads waiting side by side leave the CPU to each other
    }
  }
  if (ev) give_sync_event(ev);
  (void)hipGetLastError();  // the polls' hipErrorNotReady must not reach a later launch check
  if (e != hipSuccess) return gn::hip_error(err, code, "device execution", e);
  return 0;
}

// The Part-1 SpMV uses the grouped layout (spmv_grouped.hip) for cached structures from this
// many stored entries: below it the kernel is launch-bound and the layout's memory and one-time
// build do not pay.
constexpr long kGroupedSpmvMinNnz = 1L << 18;

bool fits(const Buffer *b, long rows, long cols, size_t esz) {
  size_t n;
  return gn::matrix_bytes(rows, cols, esz, &n) && n <= b->bytes;
}

// ---------------------------------------------------------------- CSR index cache
// The Part-1 sparse entries receive the index arrays as host pointers on every call
// (sparse-matrix.go:167-170), while the values already live in a GPUPtr buffer. The
// device copy of the indices is kept with that values buffer: the first call uploads
// and validates them, later calls with the same buffer, the same host arrays and the
// same row pointers reuse the copy and skip the validation read-back. The entry goes
// when the values buffer is released (a new EnsureGPU makes a new buffer and a new
// entry), or when gn_csr_indices_changed is called for it. Row pointers are compared
// on every call (4(rows+1) bytes); column indices changed in place under an unchanged
// values buffer need gn_csr_indices_changed, just as changed values need a new upload.
// The validation checks the indices against the call's column count (K), so an entry
// counts as validated only for the K it was checked against: a call with another K
// validates again.
// GONNGPU_CSR_CACHE=0 turns the cache off (upload and validate on every call).
struct CsrEntry {
  const int *host_rp = nullptr, *host_col = nullptr;
  long rows = 0, nnz = 0;
  std::vector<int> rp_copy;
  void *d_rp = nullptr, *d_col = nullptr;
  std::atomic<long> validated_bound{-1};  // the K the indices were checked against (-1: none)
  // The grouped SpMV layout of this structure, built by the first SpMV that finds the entry
  // validated, for that K (spmv_for: the K the build was tried for; an empty layout then
  // means the structure does not take it). Under layout_mu.
  std::mutex layout_mu;
  gn::SpmvLayout spmv;
  long spmv_for = -1;
  ~CsrEntry() {  // stream-ordered: after every call already enqueued with this entry
    gn::free_spmv_layout(&spmv, gn::resolve_stream(nullptr));
    gn::dev_free(d_rp);
    gn::dev_free(d_col);
  }
};

std::mutex g_csr_mu;
std::unordered_map<const Buffer *, std::shared_ptr<CsrEntry>> &csr_cache() {
  static auto *m = new std::unordered_map<const Buffer *, std::shared_ptr<CsrEntry>>();
  return *m;
}

bool csr_cache_enabled() {
  static const bool on = [] {
    const char *v = getenv("GONNGPU_CSR_CACHE");
    return !(v && v[0] == '0');
  }();
  return on;
}

// The cached device copy of (rowptr, cols) for values buffer `key`, uploading it when
// there is none or it no longer matches the caller's arrays.
std::shared_ptr<CsrEntry> csr_lookup(const Buffer *key) {
  std::lock_guard<std::mutex> lk(g_csr_mu);
  auto it = csr_cache().find(key);
  return it != csr_cache().end() ? it->second : nullptr;
}

std::shared_ptr<CsrEntry> csr_entry(const Buffer *key, const int *rowptr, long rows, const int *cols, long nnz,
                                    hipStream_t s, CError *err) {
  const size_t rp_bytes = sizeof(int) * (size_t)(rows + 1);
  std::shared_ptr<CsrEntry> cached;
  {
    std::lock_guard<std::mutex> lk(g_csr_mu);
    auto it = csr_cache().find(key);
    if (it != csr_cache().end()) cached = it->second;
  }
  // Entries are immutable once published, so the comparison needs no lock.
  if (cached && cached->host_rp == rowptr && cached->host_col == cols && cached->rows == rows &&
      cached->nnz == nnz && memcmp(cached->rp_copy.data(), rowptr, rp_bytes) == 0)
    return cached;
  auto e = std::make_shared<CsrEntry>();
  e->host_rp = rowptr;
  e->host_col = cols;
  e->rows = rows;
  e->nnz = nnz;
  e->rp_copy.assign(rowptr, rowptr + rows + 1);
  e->d_rp = gn::dev_alloc(rp_bytes, err);
  if (!e->d_rp) return nullptr;
  if (nnz > 0) {
    e->d_col = gn::dev_alloc(sizeof(int) * (size_t)nnz, err);
    if (!e->d_col) return nullptr;
  }
  if (gn::upload(e->d_rp, rowptr, rp_bytes, s, err)) return nullptr;
  if (nnz > 0 && gn::upload(e->d_col, cols, sizeof(int) * (size_t)nnz, s, err)) return nullptr;
  std::lock_guard<std::mutex> lk(g_csr_mu);
  csr_cache()[key] = e;  // replaces a stale entry (freed once its last user lets go)
  return e;
}

void csr_cache_forget(const Buffer *key, const CsrEntry *only) {
  std::lock_guard<std::mutex> lk(g_csr_mu);
  auto it = csr_cache().find(key);
  if (it != csr_cache().end() && (!only || it->second.get() == only)) csr_cache().erase(it);
}

// Uploads host CSR index arrays (or takes the cached copy kept with the values buffer
// `values`, when there is one), runs fn, which enqueues the work on s (no
// synchronisation), waits for it, and converts the kernel's validation flags into the
// reference's error convention. fn must only write its outputs, so enqueuing it a second
// time gives the same result. fn's last argument is the cache entry when the indices it gets
// are the entry's (so fn may keep data derived from them with it, such as the grouped SpMV
// layout), else nullptr; its flags argument is nullptr once they are validated for this
// call's bound.
template <typename Fn>
int with_csr(const Buffer *values, const int *rowptr, long rows, const int *cols, long nnz, long bound,
             hipStream_t s, CError *err, Fn fn) {
  const auto bad = [&](int f0, int f1) {
    if (f0) return set_error(err, -3, "malformed CSR: row pointers are not monotone within [0, nnz]");
    if (f1) return set_error(err, -3, "malformed CSR: column index outside [0, cols)");
    return 0;
  };
  if (values && csr_cache_enabled()) {
    // A validated entry for the same host arrays runs before its row pointers are
    // compared, so the comparison (4(rows + 1) bytes on the host) overlaps the kernels.
    // On a mismatch the entry is dropped and the work enqueued again on a fresh copy;
    // stream order makes that second result the one the caller sees. The speculative run
    // stays in bounds: the stale indices were validated for the same rows and nnz, and
    // the kernels check every column against this call's K.
    std::shared_ptr<CsrEntry> cur = csr_lookup(values);
    if (cur && cur->validated_bound.load(std::memory_order_acquire) == bound && cur->host_rp == rowptr &&
        cur->host_col == cols && cur->rows == rows && cur->nnz == nnz) {
      if (int rc = fn(static_cast<const int32_t *>(cur->d_rp), static_cast<const int32_t *>(cur->d_col), nullptr,
                      cur.get()))
        return rc;
      if (memcmp(cur->rp_copy.data(), rowptr, sizeof(int) * (size_t)(rows + 1)) == 0) return sync(s, err, -6);
      csr_cache_forget(values, cur.get());
    }
    std::shared_ptr<CsrEntry> e = csr_entry(values, rowptr, rows, cols, nnz, s, err);
    if (!e) return -3;
    const int32_t *d_rp = static_cast<const int32_t *>(e->d_rp), *d_col = static_cast<const int32_t *>(e->d_col);
    if (e->validated_bound.load(std::memory_order_acquire) == bound) {
      if (int rc = fn(d_rp, d_col, nullptr, e.get())) return rc;
      return sync(s, err, -6);
    }
    Scratch d_flags;
    d_flags.p = gn::dev_alloc(2 * sizeof(int), err);
    if (!d_flags.p) return -3;
    if (int rc = gn::launch_zero_i32(static_cast<int *>(d_flags.p), 2, s, err)) return rc;
    if (int rc = fn(d_rp, d_col, static_cast<int *>(d_flags.p), e.get())) return rc;
    if (int rc = sync(s, err, -6)) return rc;
    int flags[2] = {0, 0};
    if (int rc = gn::download(flags, d_flags.p, sizeof(flags), s, err)) return rc;
    if (int rc = bad(flags[0], flags[1])) {
      csr_cache_forget(values, e.get());
      return rc;
    }
    e->validated_bound.store(bound, std::memory_order_release);
    return 0;
  }
  Scratch d_rp, d_col, d_flags;
  d_rp.p = gn::dev_alloc(sizeof(int) * (size_t)(rows + 1), err);
  if (!d_rp.p) return -3;
  if (nnz > 0) {
    d_col.p = gn::dev_alloc(sizeof(int) * (size_t)nnz, err);
    if (!d_col.p) return -3;
  }
  d_flags.p = gn::dev_alloc(2 * sizeof(int), err);
  if (!d_flags.p) return -3;
  if (int rc = gn::upload(d_rp.p, rowptr, sizeof(int) * (size_t)(rows + 1), s, err)) return rc;
  if (nnz > 0)
    if (int rc = gn::upload(d_col.p, cols, sizeof(int) * (size_t)nnz, s, err)) return rc;
  if (int rc = gn::launch_zero_i32(static_cast<int *>(d_flags.p), 2, s, err)) return rc;
  if (int rc = fn(static_cast<const int32_t *>(d_rp.p), static_cast<const int32_t *>(d_col.p),
                  static_cast<int *>(d_flags.p), nullptr))
    return rc;
  if (int rc = sync(s, err, -6)) return rc;
  int flags[2] = {0, 0};
  if (int rc = gn::download(flags, d_flags.p, sizeof(flags), s, err)) return rc;
  return bad(flags[0], flags[1]);
}

// Device copy of a host array (n elements of T), released on scope exit.
template <typename T>
int upload_array(Scratch &dst, const T *src, long n, hipStream_t s, CError *err) {
  if (n <= 0) return 0;
  dst.p = gn::dev_alloc(sizeof(T) * (size_t)n, err);
  if (!dst.p) return -3;
  return gn::upload(dst.p, src, sizeof(T) * (size_t)n, s, err);
}

int alloc_scratch(Scratch &dst, size_t bytes, CError *err) {
  if (bytes == 0) return 0;
  dst.p = gn::dev_alloc(bytes, err);
  return dst.p ? 0 : -3;
}

// Reads back the kernels' validation flags (after everything on s has run).
int check_flags(const Scratch &flags, hipStream_t s, CError *err, const char *ptrs_msg, const char *index_msg) {
  int f[2] = {0, 0};
  if (int rc = gn::download(f, flags.p, sizeof(f), s, err)) return rc;
  if (f[0]) return set_error(err, -3, "%s", ptrs_msg);
  if (f[1]) return set_error(err, -3, "%s", index_msg);
  return 0;
}

// Exclusive prefix sum of per-row counts on the host; returns the total.
long exclusive_scan(std::vector<long> &v) {
  long run = 0;
  for (long &x : v) {
    const long c = x;
    x = run;
    run += c;
  }
  return run;
}

// Copies a device COO result (n entries) into the caller's host arrays.
int download_coo(const Scratch &ri, const Scratch &ci, const Scratch &vv, long n, int *rows, int *cols, float *vals,
                 hipStream_t s, CError *err) {
  if (n <= 0) return 0;
  if (int rc = gn::download(rows, ri.p, sizeof(int) * (size_t)n, s, err)) return rc;
  if (int rc = gn::download(cols, ci.p, sizeof(int) * (size_t)n, s, err)) return rc;
  return gn::download(vals, vv.p, sizeof(float) * (size_t)n, s, err);
}

}  // namespace

void gn::csr_cache_drop(const Buffer *b) { csr_cache_forget(b, nullptr); }
int gn::sync_stream(hipStream_t s, CError *err, int code) { return sync(s, err, code); }
bool gn::buffer_fits(const Buffer *b, long rows, long cols, size_t esz) { return fits(b, rows, cols, esz); }

extern "C" {

// =========================================================================== Part 1

int create_gpu_buffer(float *data, long length_bytes, GPUPtr *outGPUPtr, DevicePtr *outDevicePtr, CError *err) {
  gn::Context *ctx = gn::context(err);
  if (!ctx) return -1;
  if (length_bytes < 0 || !outGPUPtr) return set_error(err, -3, "Could not create GPU buffer: invalid length or output");
  void *d = gn::dev_alloc((size_t)length_bytes, err);
  if (!d) return -3;
  int rc = 0;
  if (length_bytes > 0) {
    if (data) {
      rc = gn::upload(d, data, (size_t)length_bytes, ctx->stream, err);
    } else {
      hipError_t e = hipMemsetAsync(d, 0, (size_t)length_bytes, ctx->stream);
      if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
      if (e != hipSuccess) rc = gn::hip_error(err, -4, "zero fill", e);
    }
  }
  if (rc) {
    gn::dev_free(d);
    return rc;
  }
  *outGPUPtr = gn::register_buffer(d, (size_t)length_bytes);
  if (outDevicePtr) *outDevicePtr = ctx;
  return 0;
}

int retrieve_gpu_buffer_data(GPUPtr gpuPtr, float *data, long length_bytes, CError *err) {
  Buffer *b = gn::as_buffer(gpuPtr);
  if (!b) return set_error(err, -1, "Invalid GPU buffer pointer.");
  if (length_bytes < 0 || (size_t)length_bytes > b->bytes)
    return set_error(err, -2, "Buffer length mismatch during retrieval.");
  if (length_bytes == 0) return 0;
  if (!data) return set_error(err, -1, "Invalid host pointer.");
  gn::Context *ctx = gn::context(err);
  if (!ctx) return -1;
  return gn::download(data, b->dptr, (size_t)length_bytes, ctx->stream, err);
}

int release_gpu_buffer(GPUPtr gpuPtr) {
  if (!gpuPtr) return 0;
  Buffer *b = gn::as_buffer(gpuPtr);
  if (!b) return 0;
  void *d = b->dptr;
  if (gn::unregister_buffer(b)) {
    gn::csr_cache_drop(b);
    gn::dev_free(d);  // stream-ordered: reused only after the library stream's work so far
    delete b;
  }
  return 0;
}

int perform_mps_matrix_multiplication(GPUPtr aMatrixPtr, long aRows, long aCols, GPUPtr bMatrixPtr, long bRows,
                                      long bCols, GPUPtr resultMatrixPtr, long resultRows, long resultCols,
                                      DevicePtr mtlDevicePtr, CError *err) {
  (void)mtlDevicePtr;
  gn::Context *ctx = gn::context(err);
  if (!ctx) return -1;
  Buffer *a = gn::as_buffer(aMatrixPtr), *b = gn::as_buffer(bMatrixPtr), *c = gn::as_buffer(resultMatrixPtr);
  if (!a || !b || !c) return set_error(err, -2, "Invalid input or output buffer pointers.");
  if (aRows < 0 || aCols < 0 || bCols < 0 || aCols != bRows || resultRows != aRows || resultCols != bCols)
    return set_error(err, -3, "Invalid matrix dimensions: A %ldx%ld, B %ldx%ld, C %ldx%ld", aRows, aCols, bRows, bCols,
                     resultRows, resultCols);
  if (!fits(a, aRows, aCols, 4) || !fits(b, bRows, bCols, 4) || !fits(c, resultRows, resultCols, 4))
    return set_error(err, -3, "Buffer smaller than the matrix it describes.");
  gn::GemmDesc d{GN_F32, false, false, aRows, bCols, aCols, 1.0f, 0.0f, a->dptr, aCols, 0, b->dptr, bCols, 0,
                 static_cast<float *>(c->dptr), bCols, 0, 1, nullptr, GN_ACT_NONE, 0.0f};
  if (int rc = gn::launch_gemm(d, ctx->stream, err)) return rc == -1 ? -3 : rc;
  return sync(ctx->stream, err, -6);
}

int perform_mps_matrix_transpose(GPUPtr inputMatrixPtr, long inputRows, long inputCols, GPUPtr outputMatrixPtr,
                                 long outputRows, long outputCols, DevicePtr mtlDevicePtr, CError *err) {
  (void)mtlDevicePtr;
  gn::Context *ctx = gn::context(err);
  if (!ctx) return -1;
  if (inputRows != outputCols || inputCols != outputRows || inputRows < 0 || inputCols < 0)
    return set_error(err, -2, "Invalid transpose dimensions.");
  Buffer *in = gn::as_buffer(inputMatrixPtr), *out = gn::as_buffer(outputMatrixPtr);
  if (!in || !out) return set_error(err, -3, "Invalid input or output buffer pointers.");
  if (!fits(in, inputRows, inputCols, 4) || !fits(out, outputRows, outputCols, 4))
    return set_error(err, -3, "Buffer smaller than the matrix it describes.");
  if (int rc = gn::launch_transpose_f32(static_cast<const float *>(in->dptr), inputRows, inputCols,
                                        static_cast<float *>(out->dptr), ctx->stream, err))
    return rc == -1 ? -3 : rc;
  return sync(ctx->stream, err, -6);
}

static int batched_gemm(GPUPtr aPtr, GPUPtr bPtr, GPUPtr cPtr, long batch, long M, long N, long K, float alpha,
                        float beta, CError *err) {
  gn::Context *ctx = gn::context(err);
  if (!ctx) return -1;
  Buffer *a = gn::as_buffer(aPtr), *b = gn::as_buffer(bPtr), *c = gn::as_buffer(cPtr);
  if (!a || !b || !c) return set_error(err, -2, "Invalid buffer pointers");
  if (batch < 0 || M < 0 || N < 0 || K < 0) return set_error(err, -3, "Invalid GEMM sizes");
  if (batch == 0) return 0;
  long bM, bK;
  if (__builtin_mul_overflow(batch, M, &bM) || __builtin_mul_overflow(batch, K, &bK))
    return set_error(err, -3, "Invalid GEMM sizes");
  if (!fits(a, bM, K, 4) || !fits(b, bK, N, 4) || !fits(c, bM, N, 4))
    return set_error(err, -3, "Buffer smaller than the matrices it describes.");
  gn::GemmDesc d{GN_F32, false, false, M, N, K, alpha, beta, a->dptr, K, M * K, b->dptr, N, K * N,
                 static_cast<float *>(c->dptr), N, M * N, batch, nullptr, GN_ACT_NONE, 0.0f};
  if (int rc = gn::launch_gemm(d, ctx->stream, err)) return rc == -1 ? -3 : -4;
  return sync(ctx->stream, err, -4);
}

int perform_optimized_gemm(GPUPtr aPtr, GPUPtr bPtr, GPUPtr cPtr, long M, long N, long K, float alpha, float beta,
                           DevicePtr mtlDevicePtr, CError *err) {
  (void)mtlDevicePtr;
  return batched_gemm(aPtr, bPtr, cPtr, 1, M, N, K, alpha, beta, err);
}

int perform_batch_matmul_optimized(GPUPtr aPtr, GPUPtr bPtr, GPUPtr cPtr, long batchSize, long M, long N, long K,
                                   DevicePtr mtlDevicePtr, CError *err) {
  (void)mtlDevicePtr;
  return batched_gemm(aPtr, bPtr, cPtr, batchSize, M, N, K, 1.0f, 0.0f, err);
}

int perform_fused_linear_activation(GPUPtr input, long batch_size, long input_size, GPUPtr weight, long output_size,
                                    GPUPtr bias, int activation_type, float alpha, GPUPtr output, DevicePtr device,
                                    CError *error) {
  (void)device;
  gn::Context *ctx = gn::context(error);
  if (!ctx) return -1;
  Buffer *x = gn::as_buffer(input), *w = gn::as_buffer(weight), *y = gn::as_buffer(output);
  Buffer *bb = bias ? gn::as_buffer(bias) : nullptr;
  if (!x || !w || !y || (bias && !bb)) return set_error(error, -1, "Invalid GPU buffers");
  if (activation_type == GN_ACT_NONE || !gn::act_supported(activation_type))
    return set_error(error, -1, "Unsupported activation type %d", activation_type);
  if (batch_size < 0 || input_size < 0 || output_size < 0) return set_error(error, -1, "Invalid sizes");
  if (!fits(x, batch_size, input_size, 4) || !fits(w, input_size, output_size, 4) ||
      !fits(y, batch_size, output_size, 4) || (bb && !fits(bb, 1, output_size, 4)))
    return set_error(error, -1, "Buffer smaller than the tensor it describes.");
  gn::GemmDesc d{GN_F32, false, false, batch_size, output_size, input_size, 1.0f, 0.0f, x->dptr, input_size, 0,
                 w->dptr, output_size, 0, static_cast<float *>(y->dptr), output_size, 0, 1,
                 bb ? static_cast<const float *>(bb->dptr) : nullptr, activation_type, alpha};
  if (gn::launch_gemm(d, ctx->stream, error)) return -1;
  return sync(ctx->stream, error, -1);
}

int perform_sparse_dense_matmul(GPUPtr aValuesPtr, int *aRowPtr, long aRowPtrLen, int *aColIndices,
                                long aColIndicesLen, long aRows, long aCols, long aNNZ, GPUPtr bMatrixPtr,
                                long bRows, long bCols, GPUPtr resultMatrixPtr, long resultRows, long resultCols,
                                DevicePtr mtlDevicePtr, CError *err) {
  (void)mtlDevicePtr;
  gn::Context *ctx = gn::context(err);
  if (!ctx) return -1;
  Buffer *v = aValuesPtr ? gn::as_buffer(aValuesPtr) : nullptr;
  Buffer *b = gn::as_buffer(bMatrixPtr), *c = gn::as_buffer(resultMatrixPtr);
  if (!b || !c || (aNNZ > 0 && !v) || (aValuesPtr && !v))
    return set_error(err, -1, "Invalid buffer pointers for sparse-dense multiplication.");
  if (aRows < 0 || aCols < 0 || aNNZ < 0 || aRowPtrLen != aRows + 1 || aColIndicesLen < aNNZ || aCols != bRows ||
      resultRows != aRows || resultCols != bCols || !aRowPtr || (aNNZ > 0 && !aColIndices))
    return set_error(err, -2, "Incompatible dimensions for sparse-dense multiplication.");
  if (!fits(b, bRows, bCols, 4) || !fits(c, resultRows, resultCols, 4) || (v && !fits(v, 1, aNNZ, 4)))
    return set_error(err, -2, "Buffer smaller than the matrix it describes.");
  const float *vals = v ? static_cast<const float *>(v->dptr) : nullptr;
  return with_csr(v, aRowPtr, aRows, aColIndices, aNNZ, aCols, ctx->stream, err,
                  [&](const int32_t *rp, const int32_t *col, int *flags, CsrEntry *) -> int {
                    int rc = gn::launch_spmm(aRows, bCols, aCols, aNNZ, rp, col, vals,
                                             static_cast<const float *>(b->dptr), bCols,
                                             static_cast<float *>(c->dptr), resultCols, flags, ctx->stream, err);
                    return rc ? (rc == -1 ? -2 : rc) : 0;
                  });
}

int perform_sparse_matvec(GPUPtr aValuesPtr, int *aRowPtr, long aRowPtrLen, int *aColIndices, long aColIndicesLen,
                          long aRows, long aCols, long aNNZ, GPUPtr xVectorPtr, long xSize, GPUPtr resultVectorPtr,
                          long resultSize, DevicePtr mtlDevicePtr, CError *err) {
  (void)mtlDevicePtr;
  if (aCols != xSize || aRows != resultSize)  // metal_bridge_sparse.m:306-309
    return set_error(err, -1, "Incompatible dimensions for sparse matrix-vector multiplication.");
  gn::Context *ctx = gn::context(err);
  if (!ctx) return -1;
  Buffer *v = aValuesPtr ? gn::as_buffer(aValuesPtr) : nullptr;
  Buffer *x = gn::as_buffer(xVectorPtr), *y = gn::as_buffer(resultVectorPtr);
  if (!x || !y || (aNNZ > 0 && !v) || (aValuesPtr && !v))
    return set_error(err, -1, "Invalid buffer pointers for sparse matrix-vector multiplication.");
  if (aRows < 0 || aCols < 0 || aNNZ < 0 || aRowPtrLen != aRows + 1 || aColIndicesLen < aNNZ || !aRowPtr ||
      (aNNZ > 0 && !aColIndices))
    return set_error(err, -1, "Incompatible CSR arrays for sparse matrix-vector multiplication.");
  if (!fits(x, 1, xSize, 4) || !fits(y, 1, resultSize, 4) || (v && !fits(v, 1, aNNZ, 4)))
    return set_error(err, -1, "Buffer smaller than the vector it describes.");
  const float *vals = v ? static_cast<const float *>(v->dptr) : nullptr;
  const float *xp = static_cast<const float *>(x->dptr);
  float *yp = static_cast<float *>(y->dptr);
  return with_csr(v, aRowPtr, aRows, aColIndices, aNNZ, aCols, ctx->stream, err,
                  [&](const int32_t *rp, const int32_t *col, int *flags, CsrEntry *entry) -> int {
                    // A cached structure of at least kGroupedSpmvMinNnz entries gets the grouped
                    // layout, built by its first call for this K (the validating one, which then
                    // reads the grouped kernel's column flag), so every call gives the same bits.
                    // The layout needs row pointers that are non-decreasing within [0, nnz]:
                    // checked on the host copy first; malformed ones keep the flat kernel, whose
                    // flag reports them.
                    if (entry && aNNZ >= kGroupedSpmvMinNnz && gn::spmv_grouped_supported(aRows, aCols, aNNZ)) {
                      std::lock_guard<std::mutex> lk(entry->layout_mu);
                      if (entry->spmv_for != aCols) {
                        gn::free_spmv_layout(&entry->spmv, ctx->stream);
                        const std::vector<int> &h = entry->rp_copy;
                        bool monotone = true;
                        for (long r = 0; r < aRows && monotone; ++r)
                          monotone = h[r] >= 0 && h[r + 1] >= h[r] && h[r + 1] <= aNNZ;
                        // an allocation failure leaves no layout: the flat kernel serves
                        if (monotone)
                          (void)gn::build_spmv_layout(aRows, aCols, aNNZ, h.data(), col, ctx->num_cus, ctx->stream,
                                                      &entry->spmv, nullptr);
                        entry->spmv_for = aCols;
                      }
                      if (entry->spmv.blk) return gn::launch_spmv_grouped(entry->spmv, rp, vals, xp, yp, flags,
                                                                          ctx->stream, err);
                    }
                    return gn::launch_spmv(aRows, aCols, aNNZ, rp, col, vals, xp, yp, flags, ctx->stream, err);
                  });
}

// ActivationForward entries (metal_bridge_activation.m forwards): a device kernel over
// the buffers, then a synchronisation as every Part-1 call.
static int activation_forward(GPUPtr inputPtr, GPUPtr outputPtr, long rows, long cols, int act, float alpha,
                              const char *name, CError *err) {
  gn::Context *ctx = gn::context(err);
  if (!ctx) return -1;
  Buffer *in = gn::as_buffer(inputPtr), *out = gn::as_buffer(outputPtr);
  if (!in || !out) return set_error(err, -1, "Invalid buffer pointers for %s forward.", name);
  if (rows < 0 || cols < 0) return set_error(err, -1, "Invalid size for %s forward.", name);
  if (!fits(in, rows, cols, 4) || !fits(out, rows, cols, 4))
    return set_error(err, -1, "Buffer smaller than the %ld values of %s forward.", rows * cols, name);
  const float *x = static_cast<const float *>(in->dptr);
  float *y = static_cast<float *>(out->dptr);
  const int rc = act == 3 ? gn::launch_softmax_rows(x, y, rows, cols, ctx->stream, err)
                          : gn::launch_act_forward(x, y, rows * cols, act, alpha, ctx->stream, err);
  if (rc) return -1;
  return sync(ctx->stream, err, -1);
}

int perform_activation_relu_forward(GPUPtr inputPtr, long size, GPUPtr outputPtr, DevicePtr, CError *err) {
  return activation_forward(inputPtr, outputPtr, 1, size, 0, 0.0f, "ReLU", err);
}
int perform_activation_sigmoid_forward(GPUPtr inputPtr, long size, GPUPtr outputPtr, DevicePtr, CError *err) {
  return activation_forward(inputPtr, outputPtr, 1, size, 1, 0.0f, "Sigmoid", err);
}
int perform_activation_tanh_forward(GPUPtr inputPtr, long size, GPUPtr outputPtr, DevicePtr, CError *err) {
  return activation_forward(inputPtr, outputPtr, 1, size, 2, 0.0f, "Tanh", err);
}
int perform_activation_softmax_1d_forward(GPUPtr inputPtr, long size, GPUPtr outputPtr, DevicePtr, CError *err) {
  return activation_forward(inputPtr, outputPtr, 1, size, 3, 0.0f, "Softmax 1D", err);
}
int perform_activation_softmax_2d_forward(GPUPtr inputPtr, long batchSize, long features, GPUPtr outputPtr,
                                          DevicePtr, CError *err) {
  return activation_forward(inputPtr, outputPtr, batchSize, features, 3, 0.0f, "Softmax 2D", err);
}
int perform_activation_leaky_relu_forward(GPUPtr inputPtr, long size, float alpha, GPUPtr outputPtr, DevicePtr,
                                          CError *err) {
  return activation_forward(inputPtr, outputPtr, 1, size, 4, alpha, "Leaky ReLU", err);
}
int perform_activation_elu_forward(GPUPtr inputPtr, long size, float alpha, GPUPtr outputPtr, DevicePtr,
                                   CError *err) {
  return activation_forward(inputPtr, outputPtr, 1, size, 5, alpha, "ELU", err);
}
int perform_activation_swish_forward(GPUPtr inputPtr, long size, GPUPtr outputPtr, DevicePtr, CError *err) {
  return activation_forward(inputPtr, outputPtr, 1, size, 6, 0.0f, "Swish", err);
}
int perform_activation_gelu_forward(GPUPtr inputPtr, long size, GPUPtr outputPtr, DevicePtr, CError *err) {
  return activation_forward(inputPtr, outputPtr, 1, size, 7, 0.0f, "GELU", err);
}

void free_c_error_message(char *message) { free(message); }

// ---------------------------------------------------------------- remaining sparse entries
// perform_sparse_sparse_matmul (metal_bridge.h:169-176): CSR A x CSC B -> dense.
int perform_sparse_sparse_matmul(GPUPtr aValuesPtr, int *aRowPtr, long aRowPtrLen, int *aColIndices,
                                 long aColIndicesLen, long aRows, long aCols, long aNNZ, GPUPtr bValuesPtr,
                                 int *bColPtr, long bColPtrLen, int *bRowIndices, long bRowIndicesLen, long bRows,
                                 long bCols, long bNNZ, GPUPtr resultMatrixPtr, long resultRows, long resultCols,
                                 DevicePtr mtlDevicePtr, CError *err) {
  (void)mtlDevicePtr;
  gn::Context *ctx = gn::context(err);
  if (!ctx) return -1;
  Buffer *av = aValuesPtr ? gn::as_buffer(aValuesPtr) : nullptr;
  Buffer *bv = bValuesPtr ? gn::as_buffer(bValuesPtr) : nullptr;
  Buffer *c = gn::as_buffer(resultMatrixPtr);
  if (!c || (aNNZ > 0 && !av) || (aValuesPtr && !av) || (bNNZ > 0 && !bv) || (bValuesPtr && !bv))
    return set_error(err, -1, "Invalid buffer pointers for sparse-sparse multiplication.");
  if (aRows < 0 || aCols < 0 || aNNZ < 0 || bRows < 0 || bCols < 0 || bNNZ < 0 || aRowPtrLen != aRows + 1 ||
      bColPtrLen != bCols + 1 || aColIndicesLen < aNNZ || bRowIndicesLen < bNNZ || aCols != bRows ||
      resultRows != aRows || resultCols != bCols || !aRowPtr || !bColPtr || (aNNZ > 0 && !aColIndices) ||
      (bNNZ > 0 && !bRowIndices))
    return set_error(err, -2, "Incompatible dimensions for sparse-sparse multiplication.");
  if (!fits(c, resultRows, resultCols, 4) || (av && !fits(av, 1, aNNZ, 4)) || (bv && !fits(bv, 1, bNNZ, 4)))
    return set_error(err, -2, "Buffer smaller than the matrix it describes.");
  const hipStream_t s = ctx->stream;
  Scratch arp, acol, bcp, brow, flags;
  int rc = upload_array(arp, aRowPtr, aRows + 1, s, err);
  if (!rc) rc = upload_array(acol, aColIndices, aNNZ, s, err);
  if (!rc) rc = upload_array(bcp, bColPtr, bCols + 1, s, err);
  if (!rc) rc = upload_array(brow, bRowIndices, bNNZ, s, err);
  if (!rc) rc = alloc_scratch(flags, 2 * sizeof(int), err);
  if (!rc) rc = gn::launch_zero_i32(static_cast<int *>(flags.p), 2, s, err);
  if (!rc)
    rc = gn::launch_spgemm_csr_csc(aRows, bCols, aNNZ, bNNZ, static_cast<const int32_t *>(arp.p),
                                   static_cast<const int32_t *>(acol.p),
                                   av ? static_cast<const float *>(av->dptr) : nullptr,
                                   static_cast<const int32_t *>(bcp.p), static_cast<const int32_t *>(brow.p),
                                   bv ? static_cast<const float *>(bv->dptr) : nullptr, static_cast<float *>(c->dptr),
                                   resultCols, static_cast<int *>(flags.p), s, err);
  if (rc) return rc;
  return check_flags(flags, s, err, "malformed sparse operand: row/column pointers are not monotone within [0, nnz]",
                     "malformed sparse operand");
}

// perform_dense_sparse_matmul (metal_bridge.h:190-197): dense A x CSC B -> dense. Runs
// as C^T = B^T A^T: B's CSC arrays are the CSR arrays of B^T, so the CSR SpMM kernel
// computes C^T from A^T, accumulating each output over B's column entries in order
// (the reference's order, metal_bridge_sparse.m:163-176), and C is transposed back.
int perform_dense_sparse_matmul(GPUPtr aMatrixPtr, long aRows, long aCols, GPUPtr bValuesPtr, int *bColPtr,
                                long bColPtrLen, int *bRowIndices, long bRowIndicesLen, long bRows, long bCols,
                                long bNNZ, GPUPtr resultMatrixPtr, long resultRows, long resultCols,
                                DevicePtr mtlDevicePtr, CError *err) {
  (void)mtlDevicePtr;
  gn::Context *ctx = gn::context(err);
  if (!ctx) return -1;
  Buffer *a = gn::as_buffer(aMatrixPtr), *c = gn::as_buffer(resultMatrixPtr);
  Buffer *bv = bValuesPtr ? gn::as_buffer(bValuesPtr) : nullptr;
  if (!a || !c || (bNNZ > 0 && !bv) || (bValuesPtr && !bv))
    return set_error(err, -1, "Invalid buffer pointers for dense-sparse multiplication.");
  if (aRows < 0 || aCols < 0 || bRows < 0 || bCols < 0 || bNNZ < 0 || bColPtrLen != bCols + 1 ||
      bRowIndicesLen < bNNZ || aCols != bRows || resultRows != aRows || resultCols != bCols || !bColPtr ||
      (bNNZ > 0 && !bRowIndices))
    return set_error(err, -2, "Incompatible dimensions for dense-sparse multiplication.");
  if (!fits(a, aRows, aCols, 4) || !fits(c, resultRows, resultCols, 4) || (bv && !fits(bv, 1, bNNZ, 4)))
    return set_error(err, -2, "Buffer smaller than the matrix it describes.");
  if (aRows == 0 || bCols == 0) return 0;
  const hipStream_t s = ctx->stream;
  Scratch at, ct;
  int rc = alloc_scratch(at, sizeof(float) * (size_t)aRows * (size_t)std::max(aCols, 1L), err);
  if (!rc) rc = alloc_scratch(ct, sizeof(float) * (size_t)aRows * (size_t)bCols, err);
  if (!rc && aCols > 0)
    rc = gn::launch_transpose_f32(static_cast<const float *>(a->dptr), aRows, aCols, static_cast<float *>(at.p), s,
                                  err);
  if (rc) return rc;
  const float *vals = bv ? static_cast<const float *>(bv->dptr) : nullptr;
  rc = with_csr(bv, bColPtr, bCols, bRowIndices, bNNZ, aCols, s, err,
                [&](const int32_t *cp, const int32_t *rows, int *flags, CsrEntry *) -> int {
                  int r = gn::launch_spmm(bCols, aRows, aCols, bNNZ, cp, rows, vals, static_cast<const float *>(at.p),
                                          aRows, static_cast<float *>(ct.p), aRows, flags, s, err);
                  if (!r) r = gn::launch_transpose_f32(static_cast<const float *>(ct.p), bCols, aRows,
                                                       static_cast<float *>(c->dptr), s, err);
                  return r ? (r == -1 ? -2 : r) : 0;
                });
  return rc;
}

// perform_sparse_add (metal_bridge.h:200-209): CSR + CSR -> COO in host arrays.
int perform_sparse_add(GPUPtr aValuesPtr, int *aRowPtr, long aRowPtrLen, int *aColIndices, long aColIndicesLen,
                       long aRows, long aCols, long aNNZ, GPUPtr bValuesPtr, int *bRowPtr, long bRowPtrLen,
                       int *bColIndices, long bColIndicesLen, long bRows, long bCols, long bNNZ,
                       int *resultRowIndices, int *resultColIndices, float *resultValues, long *actualNNZ,
                       long maxResultNNZ, DevicePtr mtlDevicePtr, CError *err) {
  (void)mtlDevicePtr;
  if (aRows != bRows || aCols != bCols)  // metal_bridge_sparse.m:196-199
    return set_error(err, -1, "Matrix dimensions must match for addition.");
  gn::Context *ctx = gn::context(err);
  if (!ctx) return -1;
  Buffer *av = aValuesPtr ? gn::as_buffer(aValuesPtr) : nullptr;
  Buffer *bv = bValuesPtr ? gn::as_buffer(bValuesPtr) : nullptr;
  if ((aNNZ > 0 && !av) || (aValuesPtr && !av) || (bNNZ > 0 && !bv) || (bValuesPtr && !bv))
    return set_error(err, -1, "Invalid buffer pointers for sparse addition.");
  if (aRows < 0 || aCols < 0 || aNNZ < 0 || bNNZ < 0 || aRowPtrLen != aRows + 1 || bRowPtrLen != bRows + 1 ||
      aColIndicesLen < aNNZ || bColIndicesLen < bNNZ || !aRowPtr || !bRowPtr || (aNNZ > 0 && !aColIndices) ||
      (bNNZ > 0 && !bColIndices) || !actualNNZ || maxResultNNZ < 0 ||
      (maxResultNNZ > 0 && (!resultRowIndices || !resultColIndices || !resultValues)))
    return set_error(err, -1, "Invalid arguments for sparse addition.");
  if ((av && !fits(av, 1, aNNZ, 4)) || (bv && !fits(bv, 1, bNNZ, 4)))
    return set_error(err, -1, "Buffer smaller than the values it describes.");
  *actualNNZ = 0;
  if (aRows == 0) return 0;
  const hipStream_t s = ctx->stream;
  Scratch arp, acol, brp, bcol, flags, counts, offs, ri, ci, vv;
  int rc = upload_array(arp, aRowPtr, aRows + 1, s, err);
  if (!rc) rc = upload_array(acol, aColIndices, aNNZ, s, err);
  if (!rc) rc = upload_array(brp, bRowPtr, bRows + 1, s, err);
  if (!rc) rc = upload_array(bcol, bColIndices, bNNZ, s, err);
  if (!rc) rc = alloc_scratch(flags, 2 * sizeof(int), err);
  if (!rc) rc = alloc_scratch(counts, sizeof(long) * (size_t)aRows, err);
  if (!rc) rc = gn::launch_zero_i32(static_cast<int *>(flags.p), 2, s, err);
  const float *a_vals = av ? static_cast<const float *>(av->dptr) : nullptr;
  const float *b_vals = bv ? static_cast<const float *>(bv->dptr) : nullptr;
  auto pass = [&](bool write) {
    return gn::launch_spadd(write, aRows, aCols, aNNZ, bNNZ, static_cast<const int32_t *>(arp.p),
                            static_cast<const int32_t *>(acol.p), a_vals, static_cast<const int32_t *>(brp.p),
                            static_cast<const int32_t *>(bcol.p), b_vals, static_cast<long *>(counts.p),
                            static_cast<const long *>(offs.p), static_cast<int32_t *>(ri.p),
                            static_cast<int32_t *>(ci.p), static_cast<float *>(vv.p), static_cast<int *>(flags.p), s,
                            err);
  };
  if (!rc) rc = pass(false);
  if (rc) return rc;
  if (int f = check_flags(flags, s, err, "malformed CSR: row pointers are not monotone within [0, nnz]",
                          "malformed CSR: column index outside [0, cols)"))
    return f;
  std::vector<long> off((size_t)aRows);
  if (int r = gn::download(off.data(), counts.p, sizeof(long) * (size_t)aRows, s, err)) return r;
  const long total = exclusive_scan(off);
  if (total > maxResultNNZ) return set_error(err, -2, "Result matrix exceeds maximum allocated space.");
  if (total > 0) {
    rc = upload_array(offs, off.data(), aRows, s, err);
    if (!rc) rc = alloc_scratch(ri, sizeof(int32_t) * (size_t)total, err);
    if (!rc) rc = alloc_scratch(ci, sizeof(int32_t) * (size_t)total, err);
    if (!rc) rc = alloc_scratch(vv, sizeof(float) * (size_t)total, err);
    if (!rc) rc = pass(true);
    if (!rc) rc = download_coo(ri, ci, vv, total, resultRowIndices, resultColIndices, resultValues, s, err);
    if (rc) return rc;
  }
  *actualNNZ = total;
  return 0;
}

// perform_sparse_scalar_multiply (metal_bridge.h:212-218): values *= scalar in place.
int perform_sparse_scalar_multiply(GPUPtr valuesPtr, int *rowPtr, long rowPtrLen, int *colIndices,
                                   long colIndicesLen, long rows, long cols, long nnz, float scalar,
                                   DevicePtr mtlDevicePtr, CError *err) {
  (void)mtlDevicePtr;
  (void)rowPtr;
  (void)rowPtrLen;
  (void)colIndices;
  (void)colIndicesLen;
  (void)rows;
  (void)cols;
  gn::Context *ctx = gn::context(err);
  if (!ctx) return -1;
  Buffer *v = valuesPtr ? gn::as_buffer(valuesPtr) : nullptr;
  if (nnz < 0 || (nnz > 0 && !v) || (valuesPtr && !v))
    return set_error(err, -1, "Invalid buffer pointer for sparse scalar multiplication.");
  if (v && !fits(v, 1, nnz, 4)) return set_error(err, -1, "Buffer smaller than the values it describes.");
  if (nnz == 0) return 0;
  int rc = gn::launch_scale_f32(static_cast<float *>(v->dptr), nnz, scalar, ctx->stream, err);
  return rc ? rc : sync(ctx->stream, err, -6);
}

// perform_sparse_to_dense (metal_bridge.h:231-236): CSR -> dense (later duplicates win).
int perform_sparse_to_dense(GPUPtr valuesPtr, int *rowPtr, long rowPtrLen, int *colIndices, long colIndicesLen,
                            long rows, long cols, long nnz, GPUPtr denseMatrixPtr, long denseRows, long denseCols,
                            DevicePtr mtlDevicePtr, CError *err) {
  (void)mtlDevicePtr;
  if (rows != denseRows || cols != denseCols)  // metal_bridge_sparse.m:353-356
    return set_error(err, -1, "Dimension mismatch in sparse to dense conversion.");
  gn::Context *ctx = gn::context(err);
  if (!ctx) return -1;
  Buffer *v = valuesPtr ? gn::as_buffer(valuesPtr) : nullptr;
  Buffer *d = gn::as_buffer(denseMatrixPtr);
  if (!d || (nnz > 0 && !v) || (valuesPtr && !v))
    return set_error(err, -1, "Invalid buffer pointers for sparse to dense conversion.");
  if (rows < 0 || cols < 0 || nnz < 0 || rowPtrLen != rows + 1 || colIndicesLen < nnz || !rowPtr ||
      (nnz > 0 && !colIndices))
    return set_error(err, -1, "Incompatible CSR arrays for sparse to dense conversion.");
  if (!fits(d, rows, cols, 4) || (v && !fits(v, 1, nnz, 4)))
    return set_error(err, -1, "Buffer smaller than the matrix it describes.");
  if (rows == 0 || cols == 0) return 0;
  const float *vals = v ? static_cast<const float *>(v->dptr) : nullptr;
  return with_csr(v, rowPtr, rows, colIndices, nnz, cols, ctx->stream, err,
                  [&](const int32_t *rp, const int32_t *col, int *flags, CsrEntry *) -> int {
                    return gn::launch_csr_to_dense(rows, cols, nnz, rp, col, vals, static_cast<float *>(d->dptr), flags,
                                                   ctx->stream, err);
                  });
}

// perform_dense_to_sparse (metal_bridge.h:240-246): dense -> COO (|v| > threshold) in
// host arrays, row-major order.
int perform_dense_to_sparse(GPUPtr denseMatrixPtr, long rows, long cols, float threshold, int *rowIndices,
                            int *colIndices, float *values, long *actualNNZ, long maxNNZ, DevicePtr mtlDevicePtr,
                            CError *err) {
  (void)mtlDevicePtr;
  gn::Context *ctx = gn::context(err);
  if (!ctx) return -1;
  Buffer *d = gn::as_buffer(denseMatrixPtr);
  if (!d) return set_error(err, -1, "Invalid buffer pointer for dense to sparse conversion.");
  if (rows < 0 || cols < 0 || !actualNNZ || maxNNZ < 0 || (maxNNZ > 0 && (!rowIndices || !colIndices || !values)))
    return set_error(err, -1, "Invalid arguments for dense to sparse conversion.");
  if (!fits(d, rows, cols, 4)) return set_error(err, -1, "Buffer smaller than the matrix it describes.");
  *actualNNZ = 0;
  if (rows == 0 || cols == 0) return 0;
  const hipStream_t s = ctx->stream;
  const float *D = static_cast<const float *>(d->dptr);
  Scratch counts, offs, ri, ci, vv;
  int rc = alloc_scratch(counts, sizeof(long) * (size_t)rows, err);
  if (!rc)
    rc = gn::launch_dense_to_coo(false, rows, cols, D, threshold, static_cast<long *>(counts.p), nullptr, nullptr,
                                 nullptr, nullptr, s, err);
  if (rc) return rc;
  std::vector<long> off((size_t)rows);
  if (int r = gn::download(off.data(), counts.p, sizeof(long) * (size_t)rows, s, err)) return r;
  const long total = exclusive_scan(off);
  if (total > maxNNZ) return set_error(err, -2, "Too many non-zero elements, exceeds allocated space.");
  if (total > 0) {
    rc = upload_array(offs, off.data(), rows, s, err);
    if (!rc) rc = alloc_scratch(ri, sizeof(int32_t) * (size_t)total, err);
    if (!rc) rc = alloc_scratch(ci, sizeof(int32_t) * (size_t)total, err);
    if (!rc) rc = alloc_scratch(vv, sizeof(float) * (size_t)total, err);
    if (!rc)
      rc = gn::launch_dense_to_coo(true, rows, cols, D, threshold, nullptr, static_cast<const long *>(offs.p),
                                   static_cast<int32_t *>(ri.p), static_cast<int32_t *>(ci.p),
                                   static_cast<float *>(vv.p), s, err);
    if (!rc) rc = download_coo(ri, ci, vv, total, rowIndices, colIndices, values, s, err);
    if (rc) return rc;
  }
  *actualNNZ = total;
  return 0;
}

// =========================================================================== Part 2

const char *gn_version(void) { return "gonngpu-mi355x 0.1 (gfx950)"; }

int gn_init(CError *err) { return gn::context(err) ? 0 : -1; }

void *gn_stream(void) {
  gn::Context *ctx = gn::context(nullptr);
  return ctx ? (void *)ctx->stream : nullptr;
}

int gn_device(void) {
  gn::Context *ctx = gn::context(nullptr);
  return ctx ? ctx->device : -1;
}

void *gn_buffer_device_ptr(GPUPtr buf) {
  Buffer *b = gn::as_buffer(buf);
  return b ? b->dptr : nullptr;
}

long gn_buffer_bytes(GPUPtr buf) {
  Buffer *b = gn::as_buffer(buf);
  return b ? (long)b->bytes : -1;
}

void gn_memory_stats(long *current_bytes, long *peak_bytes, long *num_allocations) {
  gn::memory_stats(current_bytes, peak_bytes, num_allocations);
}

int gn_malloc(void **ptr, size_t bytes, CError *err) {
  if (!ptr) return set_error(err, -1, "gn_malloc: NULL output");
  *ptr = gn::dev_alloc(bytes, err);
  return *ptr ? 0 : -3;
}

int gn_free(void *ptr) {
  if (!ptr) return 0;
  // Device-wide: the block may have been used on any stream (the caller's own included).
  if (hipDeviceSynchronize() != hipSuccess) {
    (void)hipGetLastError();  // e.g. a stream capture in progress: keep the block, report it
    return -1;
  }
  gn::dev_free(ptr);
  return 0;
}

int gn_csr_indices_changed(GPUPtr valuesPtr) {
  Buffer *b = gn::as_buffer(valuesPtr);
  if (b) gn::csr_cache_drop(b);
  return 0;
}

int gn_free_async(void *ptr, void *stream) {
  if (!ptr) return 0;
  const hipStream_t s = gn::resolve_stream(stream);
  // The release records an event that is queried later, which a capturing stream cannot do.
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(s, &cap) != hipSuccess || cap != hipStreamCaptureStatusNone) {
    (void)hipGetLastError();
    return -1;
  }
  gn::dev_free_on(ptr, s);
  return 0;
}

int gn_synchronize(void *stream, CError *err) {
  if (!gn::context(err)) return -1;
  return sync(gn::resolve_stream(stream), err, -6);
}

int gn_gemm(int dtype, int transA, int transB, long M, long N, long K, float alpha, const void *A, long lda,
            long strideA, const void *B, long ldb, long strideB, float beta, float *C, long ldc, long strideC,
            long batch, const float *bias, int act, float act_alpha, void *stream, CError *err) {
  if (!gn::context(err)) return -1;
  gn::GemmDesc d{dtype, transA != 0, transB != 0, M, N, K, alpha, beta, A, lda, strideA, B, ldb, strideB,
                 C, ldc, strideC, batch, bias, act, act_alpha};
  return gn::launch_gemm(d, gn::resolve_stream(stream), err);
}

int gn_cast_f32_f16(const float *in, uint16_t *out, size_t n, int round_mode, void *stream, CError *err) {
  if (!gn::context(err)) return -1;
  return gn::launch_cast_f32_f16(in, out, n, round_mode, gn::resolve_stream(stream), err);
}

int gn_cast_f16_f32(const uint16_t *in, float *out, size_t n, void *stream, CError *err) {
  if (!gn::context(err)) return -1;
  return gn::launch_cast_f16_f32(in, out, n, gn::resolve_stream(stream), err);
}

int gn_activation_backward(const float *grad_out, const float *pre, long rows, long cols, int act, float alpha,
                           float scale, float *grad_in, float *grad_bias, void *stream, CError *err) {
  if (!gn::context(err)) return -1;
  return gn::launch_act_backward(grad_out, pre, rows, cols, act, alpha, scale, grad_in, grad_bias,
                                 gn::resolve_stream(stream), err);
}

int gn_activation_backward_noalloc(const float *grad_out, const float *pre, long rows, long cols, int act,
                                   float alpha, float scale, float *grad_in, float *grad_bias, void *stream,
                                   CError *err) {
  if (!gn::context(err)) return -1;
  return gn::launch_act_backward_noalloc(grad_out, pre, rows, cols, act, alpha, scale, grad_in, grad_bias,
                                         gn::resolve_stream(stream), err);
}

int gn_activation_forward(const float *in, float *out, long n, int act, float alpha, void *stream, CError *err) {
  if (!gn::context(err)) return -1;
  return gn::launch_act_forward(in, out, n, act, alpha, gn::resolve_stream(stream), err);
}

int gn_softmax_rows(const float *in, float *out, long rows, long cols, void *stream, CError *err) {
  if (!gn::context(err)) return -1;
  return gn::launch_softmax_rows(in, out, rows, cols, gn::resolve_stream(stream), err);
}

int gn_transpose_f32(const float *in, long rows, long cols, float *out, void *stream, CError *err) {
  if (!gn::context(err)) return -1;
  return gn::launch_transpose_f32(in, rows, cols, out, gn::resolve_stream(stream), err);
}

int gn_add_bias_cyclic_f32(float *y, long n, const float *bias, long len, void *stream, CError *err) {
  if (!gn::context(err)) return -1;
  if (n > 0 && (!y || !bias)) return set_error(err, -1, "cyclic bias add: NULL pointer");
  return gn::launch_add_cyclic_f32(y, n, bias, len, gn::resolve_stream(stream), err);
}

int gn_mxfp4_size(long rows, long cols, size_t *data_bytes, size_t *scale_bytes, CError *err) {
  if (!data_bytes || !scale_bytes) return set_error(err, -1, "mxfp4 size: NULL output");
  if (!gn::mxfp4_size(rows, cols, data_bytes, scale_bytes))
    return set_error(err, -1, "mxfp4 size: invalid size %ld x %ld", rows, cols);
  return 0;
}

int gn_mxfp4_quantize(int dtype, const void *x, long rows, long cols, long ldx, void *data, void *scales,
                      void *stream, CError *err) {
  if (int rc = gn::check_mxfp4_quantize(dtype, x, rows, cols, ldx, data, scales, err)) return rc;
  if (!gn::context(err)) return -1;
  return gn::launch_mxfp4_quantize(dtype, x, rows, cols, ldx, data, scales, gn::resolve_stream(stream), err);
}

int gn_mxfp4_dequantize(const void *data, const void *scales, long rows, long cols, int dtype, void *out, long ldo,
                        void *stream, CError *err) {
  if (int rc = gn::check_mxfp4_dequantize(data, scales, rows, cols, dtype, out, ldo, err)) return rc;
  if (!gn::context(err)) return -1;
  return gn::launch_mxfp4_dequantize(data, scales, rows, cols, dtype, out, ldo, gn::resolve_stream(stream), err);
}

int gn_mxfp4_gemm(int a_dtype, long M, long N, long K, float alpha, const void *A, long lda, const void *a_scales,
                  const void *B, const void *b_scales, float beta, float *C, long ldc, const float *bias, int act,
                  float act_alpha, void *stream, CError *err) {
  const gn::MxGemmDesc d{a_dtype, M, N, K, alpha, beta, A, lda, a_scales, B, b_scales, C, ldc, bias, act, act_alpha};
  if (int rc = gn::check_mxfp4_gemm(d, err)) return rc;
  if (!gn::context(err)) return -1;
  return gn::launch_mxfp4_gemm(d, gn::resolve_stream(stream), err);
}

int gn_int8_quantize(int dtype, const void *x, long rows, long cols, long ldx, const float *col_scale, int8_t *q, long ldq,
                     float *scales, void *stream, CError *err) {
  const gn::Int8QuantizeDesc d{dtype, x, rows, cols, ldx, col_scale, q, ldq, scales};
  if (int rc = gn::check_int8_quantize(d, err)) return rc;
  if (!gn::context(err)) return -1;
  return gn::launch_int8_quantize(d, gn::resolve_stream(stream), err);
}

int gn_int8_dequantize(const int8_t *q, const float *scales, long rows, long cols, long ldq, int dtype, void *out, long ldo,
                       void *stream, CError *err) {
  if (int rc = gn::check_int8_dequantize(q, scales, rows, cols, ldq, dtype, out, ldo, err)) return rc;
  if (!gn::context(err)) return -1;
  return gn::launch_int8_dequantize(q, scales, rows, cols, ldq, dtype, out, ldo, gn::resolve_stream(stream), err);
}

int gn_int8_gemm(long M, long N, long K, float alpha, const int8_t *A, long lda, const float *a_scales, const int8_t *B,
                 long ldb, const float *b_scales, float beta, float *C, long ldc, const float *bias, int act, float act_alpha,
                 void *stream, CError *err) {
  const gn::Int8GemmDesc d{M, N, K, alpha, beta, A, lda, a_scales, B, ldb, b_scales, C, ldc, bias, act, act_alpha};
  if (int rc = gn::check_int8_gemm(d, err)) return rc;
  if (!gn::context(err)) return -1;
  return gn::launch_int8_gemm(d, gn::resolve_stream(stream), err);
}

size_t gn_int8_linear_workspace(long M, long N, long K) { return gn::int8_linear_workspace(M, N, K); }

int gn_int8_linear(int dtype, long M, long N, long K, float alpha, const void *x, long ldx, const float *col_scale,
                   const int8_t *B, long ldb, const float *b_scales, float beta, float *C, long ldc, const float *bias, int act,
                   float act_alpha, void *workspace, size_t workspace_bytes, void *stream, CError *err) {
  const gn::Int8LinearDesc d{dtype, x, ldx, col_scale,
                             {M, N, K, alpha, beta, nullptr, 0, nullptr, B, ldb, b_scales, C, ldc, bias, act, act_alpha},
                             workspace, workspace_bytes};
  if (int rc = gn::check_int8_linear(d, err)) return rc;
  if (!gn::context(err)) return -1;
  return gn::launch_int8_linear(d, gn::resolve_stream(stream), err);
}

int gn_adjust_logits(int dtype, const void *logits, long rows, long cols, long ld, const int64_t *history, long history_len,
                     const int64_t *prompt, const float *repetition, const float *frequency, const float *presence,
                     const int64_t *bias_ids, const float *bias, int biases, const uint32_t *mask, long ldmask, void *out,
                     long ldo, void *stream, CError *err) {
  const gn::AdjustDesc d{dtype, logits, rows, cols, ld, history, history_len, prompt, repetition, frequency, presence,
                         bias_ids, bias, biases, mask, ldmask, out, ldo};
  if (int rc = gn::check_adjust(d, err)) return rc;
  if (!gn::context(err)) return -1;
  return gn::launch_adjust(d, gn::resolve_stream(stream), err);
}

int gn_adjust_logits_backward(int dtype, const void *logits, long rows, long cols, long ld, const void *grad_out, long ldg,
                              const int64_t *history, long history_len, const float *repetition, const uint32_t *mask,
                              long ldmask, void *grad_logits, long ldo, void *stream, CError *err) {
  const gn::AdjustGradDesc d{dtype, logits, rows, cols, ld, grad_out, ldg, history, history_len, repetition, mask, ldmask,
                             grad_logits, ldo};
  if (int rc = gn::check_adjust_backward(d, err)) return rc;
  if (!gn::context(err)) return -1;
  return gn::launch_adjust_backward(d, gn::resolve_stream(stream), err);
}

size_t gn_logits_workspace(long rows, long cols, int k) { return gn::logits_workspace(rows, cols, k); }

int gn_token_logprobs(int dtype, const void *logits, long rows, long cols, long ld, float temperature,
                      const int64_t *targets, float *logprob, float *lse, float *entropy, int k, int64_t *top_ids,
                      float *top_logprobs, void *workspace, size_t workspace_bytes, void *stream, CError *err) {
  const gn::LogprobsDesc d{{dtype, logits, rows, cols, ld, temperature}, targets, logprob, lse, entropy, k, top_ids,
                           top_logprobs, workspace, workspace_bytes};
  if (int rc = gn::check_token_logprobs(d, err)) return rc;
  if (!gn::context(err)) return -1;
  return gn::launch_token_logprobs(d, gn::resolve_stream(stream), err);
}

int gn_token_logprobs_backward(int dtype, const void *logits, long rows, long cols, long ld, float temperature,
                               const int64_t *targets, const float *lse, const float *entropy,
                               const float *grad_logprob, const float *grad_entropy, void *grad_logits, long ldg,
                               void *stream, CError *err) {
  const gn::LogprobsGradDesc d{{dtype, logits, rows, cols, ld, temperature}, targets, lse, entropy, grad_logprob,
                               grad_entropy, grad_logits, ldg};
  if (int rc = gn::check_token_logprobs_backward(d, err)) return rc;
  if (!gn::context(err)) return -1;
  return gn::launch_token_logprobs_backward(d, gn::resolve_stream(stream), err);
}

int gn_distill_forward(int dtype, const void *logits, long rows, long cols, long ld, float temperature,
                       const int64_t *ids, const float *teacher, int k, float *loss, float *lse, void *workspace,
                       size_t workspace_bytes, void *stream, CError *err) {
  const gn::DistillDesc d{{dtype, logits, rows, cols, ld, temperature}, ids, teacher, k, loss, lse, workspace,
                          workspace_bytes, nullptr, nullptr, nullptr, 0};
  if (int rc = gn::check_distill_forward(d, err)) return rc;
  if (!gn::context(err)) return -1;
  return gn::launch_distill_forward(d, gn::resolve_stream(stream), err);
}

int gn_distill_backward(int dtype, const void *logits, long rows, long cols, long ld, float temperature,
                        const int64_t *ids, const float *teacher, int k, const float *lse, const float *grad_loss,
                        void *grad_logits, long ldg, void *stream, CError *err) {
  const gn::DistillDesc d{{dtype, logits, rows, cols, ld, temperature}, ids, teacher, k, nullptr, nullptr, nullptr, 0,
                          lse, grad_loss, grad_logits, ldg};
  if (int rc = gn::check_distill_backward(d, err)) return rc;
  if (!gn::context(err)) return -1;
  return gn::launch_distill_backward(d, gn::resolve_stream(stream), err);
}

int gn_spmm_csr(long M, long N, long K, long nnz, const int32_t *rowptr, const int32_t *col, const float *val,
                const float *D, long ldd, float *C, long ldc, int *error_flags, void *stream, CError *err) {
  if (!gn::context(err)) return -1;
  return gn::launch_spmm(M, N, K, nnz, rowptr, col, val, D, ldd, C, ldc, error_flags, gn::resolve_stream(stream),
                         err);
}

int gn_spmv_csr(long M, long K, long nnz, const int32_t *rowptr, const int32_t *col, const float *val,
                const float *x, float *y, int *error_flags, void *stream, CError *err) {
  if (!gn::context(err)) return -1;
  return gn::launch_spmv(M, K, nnz, rowptr, col, val, x, y, error_flags, gn::resolve_stream(stream), err);
}

}  // extern "C"

namespace {
struct SpmvPlan {
  uint64_t magic;
  long M, K, nnz;
  const int32_t *rowptr, *col;
  gn::SpmvLayout layout;  // empty: the plain kernel (no stored entries)
};
constexpr uint64_t kSpmvPlanMagic = 0x676E73706D76504CULL;  // "gnspmvPL"
}  // namespace

extern "C" {

int gn_spmv_plan_create(long M, long K, long nnz, const int32_t *rowptr, const int32_t *col, void **plan,
                        void *stream, CError *err) {
  if (!plan) return set_error(err, -1, "spmv plan: NULL plan pointer");
  *plan = nullptr;
  gn::Context *ctx = gn::context(err);
  if (!ctx) return -1;
  if (M < 0 || K < 0 || nnz < 0) return set_error(err, -1, "spmv plan: negative size");
  if (!rowptr || (nnz > 0 && !col)) return set_error(err, -1, "spmv plan: NULL pointer");
  if (nnz > 0x7FFFFFFFL || M > 0x7FFFFFF0L) return set_error(err, -1, "spmv plan: exceeds int32 CSR indexing");
  hipStream_t s = gn::resolve_stream(stream);
  std::vector<int32_t> h_rp((size_t)M + 1);
  if (int rc = gn::download(h_rp.data(), rowptr, sizeof(int32_t) * h_rp.size(), s, err)) return rc;
  for (long r = 0; r < M; ++r)
    if (h_rp[r] < 0 || h_rp[r + 1] < h_rp[r] || h_rp[r + 1] > nnz)
      return set_error(err, -1, "malformed CSR: row pointers are not monotone within [0, nnz]");
  auto *p = new SpmvPlan{kSpmvPlanMagic, M, K, nnz, rowptr, col, {}};
  // A structure that does not take the layout (build returns 1) keeps the flat kernel.
  if (int rc = gn::build_spmv_layout(M, K, nnz, h_rp.data(), col, ctx->num_cus, s, &p->layout, err); rc < 0) {
    delete p;
    return rc;
  }
  *plan = p;
  return 0;
}

int gn_spmv_plan_run(const void *plan, const float *val, const float *x, float *y, int *error_flags, void *stream,
                     CError *err) {
  if (!gn::context(err)) return -1;
  const SpmvPlan *p = static_cast<const SpmvPlan *>(plan);
  if (!p || p->magic != kSpmvPlanMagic) return set_error(err, -1, "spmv plan: not a live plan");
  hipStream_t s = gn::resolve_stream(stream);
  if (p->M == 0) return 0;
  if (!y || (p->nnz > 0 && !val) || (p->K > 0 && !x)) return set_error(err, -1, "spmv plan: NULL pointer");
  if (!p->layout.blk)
    return gn::launch_spmv(p->M, p->K, p->nnz, p->rowptr, p->col, val, x, y, error_flags, s, err);
  return gn::launch_spmv_grouped(p->layout, p->rowptr, val, x, y, error_flags, s, err);
}

void gn_spmv_plan_release(void *plan, void *stream) {
  SpmvPlan *p = static_cast<SpmvPlan *>(plan);
  if (!p || p->magic != kSpmvPlanMagic) return;
  gn::free_spmv_layout(&p->layout, gn::resolve_stream(stream));
  p->magic = 0;
  delete p;
}

int gn_fill_uniform_f32(float *out, size_t n, uint64_t seed, uint64_t stream_id, float lo, float hi, void *stream,
                        CError *err) {
  if (!gn::context(err)) return -1;
  return gn::launch_fill_uniform(out, n, seed, stream_id, lo, hi, gn::resolve_stream(stream), err);
}

int gn_fill_normal_f32(float *out, size_t n, uint64_t seed, uint64_t stream_id, float mean, float stddev,
                       void *stream, CError *err) {
  if (!gn::context(err)) return -1;
  return gn::launch_fill_normal(out, n, seed, stream_id, mean, stddev, gn::resolve_stream(stream), err);
}

}  // extern "C"
