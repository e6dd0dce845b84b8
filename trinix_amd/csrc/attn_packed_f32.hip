// Packed-sequence attention kernels, fp32.
#include "attn_packed_generic.h"
#include "attn_packed_merge.h"

namespace trinix {

// ks: wavefronts per 32 rows (keys); head_dim 256 (registers, LDS): 1
hipError_t launch_packed_fwd_f32(const PackedParams& p, int C, int ks, int grid, hipStream_t st) {
  const dim3 g((unsigned)grid), b(256);
  switch (C) {
    case 64:
      return ks == 2 ? launch_kernel(&packed_fwd_f32<Ops32<64>, 2, 2, false>, g, b, 0, st, p)
                     : launch_kernel(&packed_fwd_f32<Ops32<64>, 2, 1, false>, g, b, 0, st, p);
    case 96:
      return ks == 2 ? launch_kernel(&packed_fwd_f32<Ops32<128, 96>, 1, 2, false>, g, b, 0, st, p)
                     : launch_kernel(&packed_fwd_f32<Ops32<128, 96>, 1, 1, false>, g, b, 0, st, p);
    case 128:
      return ks == 2 ? launch_kernel(&packed_fwd_f32<Ops32<128>, 1, 2, false>, g, b, 0, st, p)
                     : launch_kernel(&packed_fwd_f32<Ops32<128>, 1, 1, false>, g, b, 0, st, p);
    case 256: return launch_kernel(&packed_fwd_f32<Ops32<256>, 1, 1, false>, g, b, 0, st, p);
  }
  return hipErrorNotSupported;
}
template <class O, int OCC, int KS>
hipError_t launch_chunks(const PackedParams& p, int grid, hipStream_t st) {
  constexpr int D = O::kD;
  const hipError_t e = launch_kernel(&packed_fwd_f32<O, OCC, KS, true>, dim3((unsigned)(grid * p.n_chunks)), dim3(256), 0, st, p);
  if (e != hipSuccess) return e;
  return launch_kernel(&packed_fwd_merge<float, D, 128 / KS, kTileRows, kPackedF32Slots<D>>, dim3((unsigned)grid), dim3(256), 0, st, p);
}
hipError_t launch_packed_chunks_f32(const PackedParams& p, int C, int grid, hipStream_t st) {
  switch (C) {
    case 64: return launch_chunks<Ops32<64>, 2, 2>(p, grid, st);
    case 96: return launch_chunks<Ops32<128, 96>, 1, 2>(p, grid, st);
    case 128: return launch_chunks<Ops32<128>, 1, 2>(p, grid, st);
    case 256: return launch_chunks<Ops32<256>, 1, 1>(p, grid, st);
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
