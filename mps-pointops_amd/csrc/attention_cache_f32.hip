// Attention over caches in the tokens' own type, f32.
#include "attention_cache.hpp"

namespace pointops {
namespace attn {
template hipError_t launch_cache_form<float, kAligned>(const CacheArgs&, const CachePlan&, void*, float*, hipStream_t);
template hipError_t launch_cache_form<float, kAny>(const CacheArgs&, const CachePlan&, void*, float*, hipStream_t);
}  // namespace attn
}  // namespace pointops
