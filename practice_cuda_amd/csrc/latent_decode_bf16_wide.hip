// latent_decode_bf16_wide.hip - decode kernels: bf16 queries, latent width 512, rotary width 64.
#include "latent_decode_inst.h"

namespace pcamd {
namespace decode {
template int launch<kBF16, 512, 64>(const Args&, Shape, bool, hipStream_t);
}  // namespace decode
}  // namespace pcamd
