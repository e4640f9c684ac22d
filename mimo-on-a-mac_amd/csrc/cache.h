// The paged K/V cache's host-side checks, shared by the entry points that write and read it.
#pragma once
#include <algorithm>

#include "host.h"

namespace mimo {

// tokens of one request that a page table may hold: key numbers a tile past the last stay below 2^31
constexpr int64_t kMaxTokens = 0x7fff0000;
// blocks of 256 threads of one launch: its threads stay below 2^32
constexpr int64_t kMaxBlocks = (1 << 24) - 1;

inline bool overlap(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + nb && y < x + na;
}

int check_cache(const mimo_kv_cache* c, const char* what);

}  // namespace mimo
