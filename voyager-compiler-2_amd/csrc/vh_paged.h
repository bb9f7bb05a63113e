// The paged cache as kernels see it.
//
// Slot s holds the keys and values of one token, in page s / page at row
// s % page.  Codes are [pages][kv][page][dim] (a head's rows of a page
// contiguous, so attention reads whole lines), scales [pages][kv][page]
// float32, one a row.  int8 codes are held as code + 128.
#pragma once

#include <stdint.h>

#include "../../include/voyager_hip.h"

enum { CACHE_E4M3 = VH_CACHE_E4M3, CACHE_INT8 = VH_CACHE_INT8, CACHE_F16 = VH_CACHE_F16, CACHE_BF16 = VH_CACHE_BF16 };

// Checks what every entry point needs of a cache; VH_OK or VH_EINVAL.
int vh_cache_check(const vh_cache* c, const char* what);
