// latent_decode_inst.h - the decode kernels of one element type and geometry.
#pragma once

#include <atomic>

#include "abi_util.h"
#include "latent_decode.h"

namespace pcamd {
namespace decode {

template <int DT, bool FP8, int DL, int DR, int MR, int WR, int SPLIT>
int launch_shape(const Args& a, hipStream_t st) {
  static std::atomic<uint64_t> done{0};
  typedef Kernel<DT, FP8, DL, DR, MR, WR, SPLIT> K;
  const auto kern = decode_kernel<DT, FP8, DL, DR, MR, WR, SPLIT>;
  const int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(kern), K::LDS, st, done);
  if (rc != PCAMD_OK) return rc;
  kern<<<a.groups * SPLIT, NT, K::LDS, st>>>(a);
  return check_launch("decode_kernel");
}

template <int DT, int DL, int DR>
int launch(const Args& a, Shape shape, bool fp8, hipStream_t st) {
  int rc;
  if (shape.split == 2) rc = fp8 ? launch_shape<DT, true, DL, DR, 32, 2, 2>(a, st) : launch_shape<DT, false, DL, DR, 32, 2, 2>(a, st);
  else if (shape.mr == 32) rc = fp8 ? launch_shape<DT, true, DL, DR, 32, 4, 1>(a, st) : launch_shape<DT, false, DL, DR, 32, 4, 1>(a, st);
  else if (shape.wr == 4) rc = fp8 ? launch_shape<DT, true, DL, DR, 16, 4, 1>(a, st) : launch_shape<DT, false, DL, DR, 16, 4, 1>(a, st);
  else if (shape.wr == 2) rc = fp8 ? launch_shape<DT, true, DL, DR, 16, 2, 1>(a, st) : launch_shape<DT, false, DL, DR, 16, 2, 1>(a, st);
  else rc = fp8 ? launch_shape<DT, true, DL, DR, 16, 1, 1>(a, st) : launch_shape<DT, false, DL, DR, 16, 1, 1>(a, st);
  if (rc != PCAMD_OK || !a.parts) return rc;
  // as many workgroups as the joins can keep busy: one at most a boundary between pieces
  const int64_t tiles = a.batch * a.row_tiles, joins = tiles < a.groups - 1 ? tiles : a.groups - 1;
  const int64_t units = joins * shape.tile_rows() * DL / 256;  // of 1 KB
  const auto kern = shape.mr == 32 ? combine_kernel<DT, DL, 32> : combine_kernel<DT, DL, 16>;
  kern<<<static_cast<uint32_t>(units < kJoinGroups ? units : kJoinGroups), kJoinThreads, 0, st>>>(a, shape.tile_rows());
  return check_launch("combine_kernel");
}

}  // namespace decode
}  // namespace pcamd
