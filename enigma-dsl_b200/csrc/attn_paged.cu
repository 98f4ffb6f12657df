// attn_paged.cu — one new token per sequence over a paged cache with a shared prefix.
#include "attn_serving.cuh"

namespace enigma {

size_t sdpa_shared_prefix_workspace(const enigma_sdpa_shared_prefix_desc&) { return 0; }

cudaError_t sdpa_shared_prefix_launch(const enigma_sdpa_shared_prefix_desc& d, cudaStream_t s) {
  return sdpa_paged_simt_launch(d, s);
}

}  // namespace enigma
