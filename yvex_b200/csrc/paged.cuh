// What the entries of a serving step over a paged cache share.
#pragma once
#include <stdint.h>

#include <type_traits>

#include "common.cuh"

namespace yb {

// Host checks of a cache (types, alignment, limits) and of a step's sizes; 0 or a refusal.
int check_cache(const yvex_b200_kv_cache *c);
int check_step(const yvex_b200_kv_step *t);

}  // namespace yb
