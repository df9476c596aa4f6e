// paged_decode_bf16_x32.cu -- the attention kernel of paged_decode.cuh over a cache of
// bf16, 32-bit queries or outputs.
#include "paged_decode.cuh"

namespace mxmoe {

cudaError_t launch_attend_bf16_x32(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st) {
  if (p.c.head_dim <= 64) return decode::launch<decode::Bf16<64, true>, 64>(p, ws, plan, st);
  if (p.c.head_dim <= 80) return decode::launch<decode::Bf16<80, true>, 80>(p, ws, plan, st);
  if (p.c.head_dim <= 96) return decode::launch<decode::Bf16<96, true>, 96>(p, ws, plan, st);
  if (p.c.head_dim <= 128) return decode::launch<decode::Bf16<128, true>, 128>(p, ws, plan, st);
  return decode::launch<decode::Bf16<256, true>, 256>(p, ws, plan, st);
}

}  // namespace mxmoe
