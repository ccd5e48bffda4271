// latent_decode_f16_wide.hip - decode kernels: f16 queries, latent width 512, rotary width 64.
#include "latent_decode_inst.h"

namespace pcamd {
namespace decode {
template int launch<kF16, 512, 64>(const Args&, Shape, bool, hipStream_t);
}  // namespace decode
}  // namespace pcamd
