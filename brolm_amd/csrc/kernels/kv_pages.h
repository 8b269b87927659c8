// Shared by the kernels of the paged 8-bit KV cache (kv_pages.hip, attention_q8.hip).
#pragma once

#include "common.h"

namespace bx {

constexpr int kPlanMaxReq = 4096;   // requests of a plan: its prefix sums are held in LDS

inline bool kv_page_ok(int page) { return page == 16 || page == 32 || page == 64 || page == 128; }

// Checks of the cache arguments that the entry points share.
int kv_cache_check(const char* what, int n_kv, int hd, int page, int n_pages, const int8_t* Kc, const int8_t* Vc,
                   const float* ks, const float* vs);

}  // namespace bx
