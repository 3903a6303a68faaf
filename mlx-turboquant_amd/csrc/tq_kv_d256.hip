// Attention over 8-bit and uncompressed KV caches, head dim 256.
#include "tq_kv_chunk.h"
#include "tq_kv_decode.h"

namespace tq {
namespace kv {
template hipError_t launch_decode<256>(const Params&, bool, int, hipStream_t);
template hipError_t launch_chunk<256>(const Params&, bool, int, hipStream_t);
}  // namespace kv
}  // namespace tq
