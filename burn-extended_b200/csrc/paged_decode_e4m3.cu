// paged_decode_e4m3.cu -- the attention kernel of paged_decode.cuh over a cache of
// 8-bit floats (E4M3), bf16 queries and outputs.
#include "paged_decode.cuh"

namespace mxmoe {

cudaError_t launch_attend_e4m3(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st) {
  if (p.c.head_dim <= 64) return decode::launch<decode::E4m3<64, false>, 64>(p, ws, plan, st);
  if (p.c.head_dim <= 96) return decode::launch<decode::E4m3<96, false>, 96>(p, ws, plan, st);
  if (p.c.head_dim <= 128) return decode::launch<decode::E4m3<128, false>, 128>(p, ws, plan, st);
  return decode::launch<decode::E4m3<256, false>, 256>(p, ws, plan, st);
}

}  // namespace mxmoe
