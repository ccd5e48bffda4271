// latent_decode_bf16_narrow.hip - decode kernels: bf16 queries, latent width 256, rotary width 32.
#include "latent_decode_inst.h"

namespace pcamd {
namespace decode {
template int launch<kBF16, 256, 32>(const Args&, Shape, bool, hipStream_t);
}  // namespace decode
}  // namespace pcamd
