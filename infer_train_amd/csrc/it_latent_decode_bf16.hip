// it_latent_decode_bf16.hip -- absorbed latent attention over BF16 rows.
#include "it_latent_decode.hpp"

hipError_t itkv::latent_decode_bf16(const LatentDecodeArgs& a, const LatentSplitPlan& p, int qg, hipStream_t s) {
  return launch_latent_decode<true>(a, p, qg, s);
}
