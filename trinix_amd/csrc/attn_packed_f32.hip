// Packed-sequence attention kernels, fp32.
#include "attn_packed_generic.h"

namespace trinix {

hipError_t launch_packed_fwd_f32(const PackedParams& p, int D, PackedShape, int grid, hipStream_t st) {
  const dim3 g((unsigned)grid), b(256);
  switch (D) {
    case 64: return launch_kernel(&packed_fwd_generic<Ops32<64>, BF16, 2>, g, b, 0, st, p);
    case 128: return launch_kernel(&packed_fwd_generic<Ops32<128>, BF16, 1>, g, b, 0, st, p);
    case 256: return launch_kernel(&packed_fwd_generic<Ops32<256>, BF16, 1>, g, b, 0, st, p);
  }
  return hipErrorNotSupported;
}
hipError_t launch_packed_dkdv_f32(const PackedParams& p, int D, int grid, hipStream_t st) {
  switch (D) {
    case 64: return launch_packed_dkdv_g<Ops32<64>, 2, 1>(p, grid, st);
    case 128: return launch_packed_dkdv_g<Ops32<128>, 1, 1>(p, grid, st);
    case 256: return launch_packed_dkdv_g<Ops32<256>, 1, 4>(p, grid, st);  // as bwd_dkdv_generic: registers
  }
  return hipErrorNotSupported;
}
hipError_t launch_packed_dq_f32(const PackedParams& p, int D, int grid, hipStream_t st) {
  switch (D) {
    case 64: return launch_packed_dq_g<Ops32<64>, 2, 1>(p, grid, st);
    case 128: return launch_packed_dq_g<Ops32<128>, 1, 1>(p, grid, st);
    case 256: return launch_packed_dq_g<Ops32<256>, 1, 2>(p, grid, st);
  }
  return hipErrorNotSupported;
}

}  // namespace trinix
