// The paged K/V cache's host-side checks, shared by the entry points that write and read it.
#pragma once
#include <algorithm>

#include "host.h"

namespace mimo {

int check_cache(const mimo_kv_cache* c, const char* what);

}  // namespace mimo
