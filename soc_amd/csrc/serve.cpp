// serve.cpp - what the paged serving entry points share on the host: the checks of strided operands and of a cache, and the
// context's workspace.
#include <string>

#include "paged_host.h"

namespace soc {

int Operands::rows(const char* what, const void* p, int64_t rows, int64_t stride, int64_t width, int size) {
  if (rows <= 0 || width <= 0) return SOC_OK;
  if (p == nullptr) return fail(SOC_ERR_INVALID, std::string(what) + ": null device pointer");
  if (stride < width || stride > (int64_t{1} << 40))
    return fail(SOC_ERR_INVALID, std::string(what) + ": row stride below the row's width, or beyond 2^40");
  if (reinterpret_cast<uintptr_t>(p) % size != 0)
    return fail(SOC_ERR_INVALID, std::string(what) + " is not aligned to its elements");
  // rows < 2^31 and stride <= 2^40 could pass 64 bits of bytes: no allocation is that large
  const unsigned __int128 bytes =
      (static_cast<unsigned __int128>(rows - 1) * static_cast<uint64_t>(stride) + static_cast<uint64_t>(width)) * size;
  const char* begin = static_cast<const char*>(p);
  const Range* in = nullptr;
  for (int i = 0; i < count_ && in == nullptr; ++i)
    if (begin >= known_[i].begin && begin < known_[i].end) in = &known_[i];
  Range asked{nullptr, nullptr};
  if (in == nullptr) {
    hipPointerAttribute_t attr{};
    if (hipPointerGetAttributes(&attr, p) != hipSuccess) {
      (void)hipGetLastError();
      return fail(SOC_ERR_INVALID, std::string(what) + " is not in device memory");
    }
    if ((attr.type == hipMemoryTypeHost && attr.devicePointer != p) ||
        (attr.type != hipMemoryTypeDevice && attr.type != hipMemoryTypeManaged && attr.type != hipMemoryTypeHost))
      return fail(SOC_ERR_INVALID, std::string(what) + " is not in device memory");
    if (attr.type == hipMemoryTypeDevice && attr.device != ctx_->device)
      return fail(SOC_ERR_INVALID, std::string(what) + " is memory of another device than the context's");
    void* base = nullptr;
    size_t held = 0;
    if (hipMemGetAddressRange(&base, &held, const_cast<void*>(p)) != hipSuccess) {
      (void)hipGetLastError();
      return fail(SOC_ERR_INVALID, std::string(what) + " extends past the end of its device allocation");
    }
    asked = Range{static_cast<const char*>(base), static_cast<const char*>(base) + held};
    in = &asked;
    if (count_ < static_cast<int>(sizeof(known_) / sizeof(known_[0]))) known_[count_++] = asked;
  }
  if (bytes > static_cast<uint64_t>(in->end - begin))
    return fail(SOC_ERR_INVALID, std::string(what) + " extends past the end of its device allocation");
  return SOC_OK;
}

int shift_of(int page_size) {
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

int check_page_size(int32_t page_size) {
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128 && page_size != 256)
    return fail(SOC_ERR_INVALID, "paged cache: page_size must be 16, 32, 64, 128 or 256");
  return SOC_OK;
}

int check_cache_shape(const soc_paged_cache* c) {
  if (c == nullptr) return fail(SOC_ERR_INVALID, "null paged cache");
  SOC_TRY(check_page_size(c->page_size));
  if (c->head_dim != 64 && c->head_dim != 128) return fail(SOC_ERR_INVALID, "paged cache: head_dim must be 64 or 128");
  if (c->kv_heads <= 0 || c->kv_heads > 1024 || c->num_pages <= 0)
    return fail(SOC_ERR_INVALID, "paged cache: need num_pages > 0 and 1 to 1024 kv_heads");
  if (static_cast<int64_t>(c->num_pages) * c->page_size > INT32_MAX)
    return fail(SOC_ERR_INVALID, "paged cache: num_pages * page_size must be below 2^31");
  const int64_t page = static_cast<int64_t>(c->kv_heads) * c->page_size * c->head_dim;
  if (c->page_stride != 0 && (c->page_stride < page || c->page_stride % 8 != 0))
    return fail(SOC_ERR_INVALID, "paged cache: page_stride must be 0 or a multiple of 8 that holds a page");
  if (reinterpret_cast<uintptr_t>(c->keys) % 16 != 0 || reinterpret_cast<uintptr_t>(c->values) % 16 != 0)
    return fail(SOC_ERR_INVALID, "paged cache: keys and values must be 16-byte aligned");
  return SOC_OK;
}

int64_t page_stride(const soc_paged_cache* c) {
  return c->page_stride != 0 ? c->page_stride : static_cast<int64_t>(c->kv_heads) * c->page_size * c->head_dim;
}

int check_cache_memory(Operands& operands, const soc_paged_cache* c) {
  const int64_t page = static_cast<int64_t>(c->kv_heads) * c->page_size * c->head_dim;
  SOC_TRY(operands.rows("paged cache keys", c->keys, c->num_pages, page_stride(c), page, 2));
  return operands.rows("paged cache values", c->values, c->num_pages, page_stride(c), page, 2);
}

int hip_status(hipError_t e, const char* what) {
  return e == hipSuccess ? SOC_OK : fail(SOC_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

int ensure_serve_ws(soc_ctx* ctx, size_t bytes, size_t ints) {
  // kernels in flight may still use what is replaced
  if (ctx->serve_ws_bytes < bytes) {
    SOC_HIP_TRY(hipStreamSynchronize(ctx->stream));
    (void)hipFree(ctx->serve_ws);
    ctx->serve_ws = nullptr;
    ctx->serve_ws_bytes = 0;
    if (hipMalloc(&ctx->serve_ws, bytes) != hipSuccess) {
      (void)hipGetLastError();
      return fail(SOC_ERR_NOMEM, "allocation of " + std::to_string(bytes) + " bytes of workspace failed");
    }
    ctx->serve_ws_bytes = bytes;
  }
  if (ctx->serve_counter_ints < ints) {
    SOC_HIP_TRY(hipStreamSynchronize(ctx->stream));
    (void)hipFree(ctx->serve_counters);
    ctx->serve_counters = nullptr;
    ctx->serve_counter_ints = 0;
    if (hipMalloc(&ctx->serve_counters, ints * sizeof(int)) != hipSuccess) {
      (void)hipGetLastError();
      ctx->serve_counters = nullptr;
      return fail(SOC_ERR_NOMEM, "allocation of the workspace counters failed");
    }
    // on the kernels' stream, so that it lands before the first of them
    const hipError_t e = hipMemsetAsync(ctx->serve_counters, 0, ints * sizeof(int), ctx->stream);
    if (e != hipSuccess) {
      (void)hipFree(ctx->serve_counters);
      ctx->serve_counters = nullptr;
      return fail(SOC_ERR_HIP, std::string("workspace counters: ") + hipGetErrorString(e));
    }
    ctx->serve_counter_ints = ints;
  }
  return SOC_OK;
}

}  // namespace soc
