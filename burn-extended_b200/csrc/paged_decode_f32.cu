// paged_decode_f32.cu -- the attention kernel of paged_decode.cuh over a cache of
// 32-bit floats.
#include "paged_decode.cuh"

namespace mxmoe {

cudaError_t launch_attend_f32(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st) {
  if (p.c.head_dim <= 64) return decode::launch<decode::F32<64, true>, 64>(p, ws, plan, st);
  if (p.c.head_dim <= 80) return decode::launch<decode::F32<80, true>, 80>(p, ws, plan, st);
  if (p.c.head_dim <= 96) return decode::launch<decode::F32<96, true>, 96>(p, ws, plan, st);
  if (p.c.head_dim <= 128) return decode::launch<decode::F32<128, true>, 128>(p, ws, plan, st);
  return decode::launch<decode::F32<256, true>, 256>(p, ws, plan, st);
}

}  // namespace mxmoe
