// causal_walk_host.cpp with the plans of a cache of int8.
#include "../hexanima_amd/csrc/causal_walk.h"

namespace {
inline CachedPlan q8_plan(const hxa_kv_cache &c, int T, int Hq, bool ws, long places) { return cached_plan(c, T, Hq, ws, places, true); }
}  // namespace
#define cached_plan q8_plan
#include "causal_walk_host.cpp"
