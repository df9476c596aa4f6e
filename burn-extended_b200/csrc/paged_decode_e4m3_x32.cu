// paged_decode_e4m3_x32.cu -- the attention kernel of paged_decode.cuh over a cache of
// 8-bit floats (E4M3), 32-bit queries or outputs.
#include "paged_decode.cuh"

namespace mxmoe {

cudaError_t launch_attend_e4m3_x32(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st) {
  if (p.c.head_dim <= 64) return decode::launch<decode::E4m3<64, true>, 64>(p, ws, plan, st);
  if (p.c.head_dim <= 96) return decode::launch<decode::E4m3<96, true>, 96>(p, ws, plan, st);
  if (p.c.head_dim <= 128) return decode::launch<decode::E4m3<128, true>, 128>(p, ws, plan, st);
  return decode::launch<decode::E4m3<256, true>, 256>(p, ws, plan, st);
}

}  // namespace mxmoe
