// The paged K/V cache's host-side checks, shared by the entry points that write and read it.
#pragma once
#include <algorithm>

#include "host.h"

namespace mimo {

// tokens of one request that a page table may hold: key numbers a tile past the last stay below 2^31
constexpr int64_t kMaxTokens = 0x7fff0000;

int check_cache(const mimo_kv_cache* c, const char* what);

}  // namespace mimo
