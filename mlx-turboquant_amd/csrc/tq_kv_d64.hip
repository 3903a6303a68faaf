// Attention over 8-bit and uncompressed KV caches, head dim 64.
#include "tq_kv_chunk.h"
#include "tq_kv_decode.h"

namespace tq {
namespace kv {
template hipError_t launch_decode<64>(const Params&, bool, int, hipStream_t);
template hipError_t launch_chunk<64>(const Params&, bool, int, hipStream_t);
}  // namespace kv
}  // namespace tq
