// Packed-sequence attention kernels, bf16.
#include "attn_packed16.h"
#include "attn_packed_bwd16.h"
#include "attn_packed_generic.h"

namespace trinix {

hipError_t launch_packed_fwd_bf16(const PackedParams& p, int C, PackedShape shape, int grid, hipStream_t st) {
  return launch_packed_fwd16<BF16>(p, C, shape, grid, st);
}
hipError_t launch_packed_bwd_bf16(const PackedParams& p, int C, int n_kv, int n_q, hipStream_t st) {
  return launch_packed_bwd16<BF16>(p, C, n_kv, n_q, st);
}
hipError_t launch_packed_dkdv_bf16(const PackedParams& p, int ks, int grid, hipStream_t st) {
  using O = Ops16<BF16, 256>;
  return ks == 2 ? launch_packed_dkdv_g<O, 1, 2, 2>(p, grid, st) : launch_packed_dkdv_g<O, 1, 2, 1>(p, grid, st);
}
hipError_t launch_packed_dq_bf16(const PackedParams& p, int ks, int grid, hipStream_t st) {
  using O = Ops16<BF16, 256>;
  return ks == 2 ? launch_packed_dq_g<O, 1, 1, 2>(p, grid, st) : launch_packed_dq_g<O, 1, 1, 1>(p, grid, st);
}

}  // namespace trinix
