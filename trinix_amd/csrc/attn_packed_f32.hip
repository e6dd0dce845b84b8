// Packed-sequence attention kernels, fp32.
#include "attn_packed_generic.h"

namespace trinix {

// ks: wavefronts per 32 rows (keys); head_dim 256 (registers, LDS): 1
hipError_t launch_packed_fwd_f32(const PackedParams& p, int C, int ks, int grid, hipStream_t st) {
  const dim3 g((unsigned)grid), b(256);
  switch (C) {
    case 64:
      return ks == 2 ? launch_kernel(&packed_fwd_f32<Ops32<64>, 2, 2>, g, b, 0, st, p)
                     : launch_kernel(&packed_fwd_f32<Ops32<64>, 2, 1>, g, b, 0, st, p);
    case 96:
      return ks == 2 ? launch_kernel(&packed_fwd_f32<Ops32<128, 96>, 1, 2>, g, b, 0, st, p)
                     : launch_kernel(&packed_fwd_f32<Ops32<128, 96>, 1, 1>, g, b, 0, st, p);
    case 128:
      return ks == 2 ? launch_kernel(&packed_fwd_f32<Ops32<128>, 1, 2>, g, b, 0, st, p)
                     : launch_kernel(&packed_fwd_f32<Ops32<128>, 1, 1>, g, b, 0, st, p);
    case 256: return launch_kernel(&packed_fwd_f32<Ops32<256>, 1, 1>, g, b, 0, st, p);
  }
  return hipErrorNotSupported;
}
hipError_t launch_packed_bwd_f32(const PackedParams& p, int C, int ks, int n_kv, int n_q, hipStream_t st) {
  switch (C) {
    case 64:
      return ks == 2 ? launch_packed_bwd_g<Ops32<64>, 2, 1, 1, 2>(p, n_kv, n_q, st)
                     : launch_packed_bwd_g<Ops32<64>, 2, 1, 1, 1>(p, n_kv, n_q, st);
    case 96:
      return ks == 2 ? launch_packed_bwd_g<Ops32<128, 96>, 1, 1, 1, 2>(p, n_kv, n_q, st)
                     : launch_packed_bwd_g<Ops32<128, 96>, 1, 1, 1, 1>(p, n_kv, n_q, st);
    case 128:
      return ks == 2 ? launch_packed_bwd_g<Ops32<128>, 1, 1, 1, 2>(p, n_kv, n_q, st)
                     : launch_packed_bwd_g<Ops32<128>, 1, 1, 1, 1>(p, n_kv, n_q, st);
    case 256: return launch_packed_bwd_g<Ops32<256>, 1, 4, 2, 1>(p, n_kv, n_q, st);  // K and V rows fill the registers
  }
  return hipErrorNotSupported;
}

}  // namespace trinix
