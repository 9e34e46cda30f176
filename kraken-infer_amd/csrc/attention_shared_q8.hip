// Causal attention of a ragged batch over 8-bit KV pages whose sequences share prefixes.
#include <hip/hip_runtime.h>

#include "context_internal.hpp"
#include "paged_q8_internal.hpp"

namespace kraken {

size_t attention_shared_q8_workspace_bytes(const PagedAttentionArgs& a, const SharedPrefixArgs&,
                                           int cu_count) {
  return attention_paged_q8_workspace_bytes(a, cu_count);
}

// Each sequence by itself: a shared page is read once for each.
hipError_t launch_attention_shared_q8(const PagedAttentionArgs& a, const SharedPrefixArgs&,
                                      int cu_count, void* workspace, hipStream_t stream) {
  return launch_attention_paged_q8(a, cu_count, workspace, stream);
}

}  // namespace kraken
