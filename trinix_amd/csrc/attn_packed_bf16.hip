// Packed-sequence attention kernels, bf16.
#include "attn_packed16.h"
#include "attn_packed_bwd16.h"
#include "attn_packed_generic.h"

namespace trinix {

hipError_t launch_packed_fwd_bf16(const PackedParams& p, int C, PackedShape shape, int grid, hipStream_t st) {
  return launch_packed_fwd16<BF16>(p, C, shape, grid, st);
}
hipError_t launch_packed_chunks_bf16(const PackedParams& p, int C, int grid, hipStream_t st) {
  return launch_packed_chunks16<BF16>(p, C, grid, st);
}
hipError_t launch_packed_bwd_bf16(const PackedParams& p, int C, int n_kv, int n_q, hipStream_t st) {
  if (C == 256) return launch_packed_bwd_g<Ops16<BF16, 256>, 1, 2, 1, 1>(p, n_kv, n_q, st);
  return launch_packed_bwd16<BF16>(p, C, n_kv, n_q, st);
}

}  // namespace trinix
