// latent_decode_f16_narrow.hip - decode kernels: f16 queries, latent width 256, rotary width 32.
#include "latent_decode_inst.h"

namespace pcamd {
namespace decode {
template int launch<kF16, 256, 32>(const Args&, Shape, bool, hipStream_t);
}  // namespace decode
}  // namespace pcamd
