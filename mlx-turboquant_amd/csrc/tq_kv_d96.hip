// Attention over 8-bit and uncompressed KV caches, head dim 96.
#include "tq_kv_chunk.h"
#include "tq_kv_decode.h"

namespace tq {
namespace kv {
template hipError_t launch_decode<96>(const Params&, bool, int, hipStream_t);
template hipError_t launch_chunk<96>(const Params&, bool, int, hipStream_t);
}  // namespace kv
}  // namespace tq
