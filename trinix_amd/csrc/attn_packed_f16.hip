// Packed-sequence attention kernels, f16.
#include "attn_packed16.h"
#include "attn_packed_generic.h"

namespace trinix {

hipError_t launch_packed_fwd_f16(const PackedParams& p, int D, PackedShape shape, int grid, hipStream_t st) {
  return launch_packed_fwd16<F16>(p, D, shape, grid, st);
}
hipError_t launch_packed_dkdv_f16(const PackedParams& p, int D, int grid, hipStream_t st) {
  switch (D) {
    case 64: return launch_packed_dkdv_g<Ops16<F16, 64>, 2, 1>(p, grid, st);
    case 128: return launch_packed_dkdv_g<Ops16<F16, 128>, 1, 1>(p, grid, st);
    case 256: return launch_packed_dkdv_g<Ops16<F16, 256>, 1, 2>(p, grid, st);
  }
  return hipErrorNotSupported;
}
hipError_t launch_packed_dq_f16(const PackedParams& p, int D, int grid, hipStream_t st) {
  switch (D) {
    case 64: return launch_packed_dq_g<Ops16<F16, 64>, 2, 1>(p, grid, st);
    case 128: return launch_packed_dq_g<Ops16<F16, 128>, 1, 1>(p, grid, st);
    case 256: return launch_packed_dq_g<Ops16<F16, 256>, 1, 2>(p, grid, st);
  }
  return hipErrorNotSupported;
}

}  // namespace trinix
