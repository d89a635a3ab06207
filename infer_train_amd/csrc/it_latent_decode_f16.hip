// it_latent_decode_f16.hip -- absorbed latent attention over F16 rows.
#include "it_latent_decode.hpp"

hipError_t itkv::latent_decode_f16(const LatentDecodeArgs& a, const LatentSplitPlan& p, int qg, hipStream_t s) {
  return launch_latent_decode<false>(a, p, qg, s);
}
