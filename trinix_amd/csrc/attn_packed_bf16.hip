// Packed-sequence attention kernels, bf16.
#include "attn_packed16.h"
#include "attn_packed_generic.h"

namespace trinix {

hipError_t launch_packed_fwd_bf16(const PackedParams& p, int D, PackedShape shape, int grid, hipStream_t st) {
  return launch_packed_fwd16<BF16>(p, D, shape, grid, st);
}
hipError_t launch_packed_dkdv_bf16(const PackedParams& p, int D, int grid, hipStream_t st) {
  switch (D) {
    case 64: return launch_packed_dkdv_g<Ops16<BF16, 64>, 2, 1>(p, grid, st);
    case 128: return launch_packed_dkdv_g<Ops16<BF16, 128>, 1, 1>(p, grid, st);
    case 256: return launch_packed_dkdv_g<Ops16<BF16, 256>, 1, 2>(p, grid, st);
  }
  return hipErrorNotSupported;
}
hipError_t launch_packed_dq_bf16(const PackedParams& p, int D, int grid, hipStream_t st) {
  switch (D) {
    case 64: return launch_packed_dq_g<Ops16<BF16, 64>, 2, 1>(p, grid, st);
    case 128: return launch_packed_dq_g<Ops16<BF16, 128>, 1, 1>(p, grid, st);
    case 256: return launch_packed_dq_g<Ops16<BF16, 256>, 1, 2>(p, grid, st);
  }
  return hipErrorNotSupported;
}

}  // namespace trinix
