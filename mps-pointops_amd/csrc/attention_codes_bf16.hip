// Attention over caches in 8 and 4 bits, queries and results in bf16.
#include "attention_cache.hpp"

namespace pointops {
namespace attn {
template hipError_t launch_cache_form<bf16, kEight>(const CacheArgs&, const CachePlan&, void*, float*, hipStream_t);
template hipError_t launch_cache_form<bf16, kFour>(const CacheArgs&, const CachePlan&, void*, float*, hipStream_t);
}  // namespace attn
}  // namespace pointops
