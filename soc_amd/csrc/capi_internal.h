// capi_internal.h - pieces shared by the translation units that implement the C ABI: the device context, the guard
// that turns C++ exceptions into status codes, and the check of caller pointers before a kernel reads them.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <new>
#include <stdexcept>

#include "soc_hip.h"
#include "status.h"

#define SOC_API_BEGIN try {
#define SOC_API_END                                                         \
  }                                                                         \
  catch (const std::bad_alloc&) {                                           \
    return soc::fail(SOC_ERR_NOMEM, "host allocation failed");              \
  }                                                                         \
  catch (const std::exception& e) {                                         \
    return soc::fail(SOC_ERR_INVALID, e.what());                            \
  }

struct soc_ctx {
  int device = 0;
  int num_cus = 0;
  hipStream_t stream = nullptr;
  hipEvent_t ev0 = nullptr, ev1 = nullptr;
  bool timing = false;          // between soc_ctx_timer_start and _stop
  bool stop_recorded = false;   // a forward recorded ev1 before its final synchronisation
  uint32_t* scratch = nullptr;  // device address of this device's copy of `scratch` (soc_decode_steps_noalloc)
  void* sample_ws = nullptr;    // soc_sample_topk: candidate search workspace and its output block
  size_t sample_ws_bytes = 0;
  int* sample_out = nullptr;
  int* sample_host = nullptr;   // pinned host copy of the output block (hipHostMalloc)
  int* sample_host_dev = nullptr;  // the address kernels use for it
  // pinned host words a decode step's readback kernel writes (next token, wait error, token id error), then a batch's
  // ids, slots and positions on their way in and tokens on their way out, with the address kernels use for them
  int32_t* readback = nullptr;
  int32_t* readback_dev = nullptr;
  // op-level attention (soc_attention_decode): split-key partials and arrival counters, grown on demand
  float* op_part = nullptr;
  size_t op_part_floats = 0;
  int* op_counters = nullptr;
  size_t op_counter_ints = 0;
  // paged serving operators (soc_paged_*, soc_logprobs): partial results and arrival counters, grown on demand; every
  // kernel leaves the counters at zero
  char* serve_ws = nullptr;
  size_t serve_ws_bytes = 0;
  int* serve_counters = nullptr;
  size_t serve_counter_ints = 0;
  // soc_forward with token ids in device memory: set by the staging kernel when an id lies outside [0, vocab)
  int* id_err = nullptr;
};


namespace soc {

// Where `bytes` bytes at p lie. kDeviceRange: in memory a kernel may read (a hipMalloc'd or managed allocation that
// holds the whole range, or pinned host memory mapped for the device). kPageable: host memory the device cannot read
// (a kernel reading it faults on devices without XNACK). kOutside: device memory whose allocation ends before
// p + bytes.
enum class MemRange { kDeviceRange, kPageable, kOutside };
MemRange classify_range(const void* p, size_t bytes);

// SOC_OK when every (pointer, bytes) of a caller's device operands lies inside one device allocation (null pointers
// with 0 bytes pass); otherwise SOC_ERR_INVALID naming the operand. Called before any kernel reads caller memory.
int check_device_operand(const char* what, const void* p, size_t bytes);

// The operands of one call in device memory: each checked to lie inside one allocation of the context's device. What the
// runtime answers about an allocation serves the call's further operands in it.
class Operands {
 public:
  explicit Operands(const soc_ctx* ctx) : ctx_(ctx) {}
  // `rows` rows of `width` elements of `size` bytes, `stride` elements apart (at least width), aligned to an element.
  int rows(const char* what, const void* p, int64_t rows, int64_t stride, int64_t width, int size);
  // `count` elements of `size` bytes
  int array(const char* what, const void* p, int64_t count, int size) { return rows(what, p, 1, count, count, size); }

 private:
  struct Range {
    const char *begin, *end;
  };
  const soc_ctx* ctx_;
  Range known_[8];
  int count_ = 0;
};

// Grows the context's serve_ws to `bytes` and its zeroed serve_counters to `ints`.
int ensure_serve_ws(soc_ctx* ctx, size_t bytes, size_t ints);

// Makes the context's device current for the calling thread while it lives: streams and allocations belong to it.
class DeviceScope {
 public:
  explicit DeviceScope(const soc_ctx* ctx) {
    if (hipGetDevice(&before_) != hipSuccess) before_ = ctx->device;
    if (before_ != ctx->device && hipSetDevice(ctx->device) == hipSuccess) changed_ = true;
  }
  ~DeviceScope() {
    if (changed_) (void)hipSetDevice(before_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;

 private:
  int before_ = 0;
  bool changed_ = false;
};

}  // namespace soc
