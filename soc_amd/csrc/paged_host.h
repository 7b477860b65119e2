// paged_host.h - host side of the paged cache's entry points: checks of its shape and memory (serve.cpp).
#pragma once

#include "capi_internal.h"

namespace soc {

// log2 of a page size
int shift_of(int page_size);
int check_page_size(int32_t page_size);
int check_cache_shape(const soc_paged_cache* c);
// Elements from one page to the next.
int64_t page_stride(const soc_paged_cache* c);
int check_cache_memory(Operands& operands, const soc_paged_cache* c);
int hip_status(hipError_t e, const char* what);

}  // namespace soc
