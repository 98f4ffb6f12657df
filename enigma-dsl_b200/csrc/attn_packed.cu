// attn_packed.cu — attention over packed prompts.
#include "attn_serving.cuh"

namespace enigma {

cudaError_t sdpa_packed_launch(const enigma_sdpa_packed_desc& d, cudaStream_t s) {
  return sdpa_packed_simt_launch(d, s);
}

}  // namespace enigma
