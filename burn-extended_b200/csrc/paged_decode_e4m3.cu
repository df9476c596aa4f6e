// paged_decode_e4m3.cu -- the attention kernel of paged_decode.cuh over a cache of 8-bit floats (E4M3).
#include "paged_decode.cuh"

namespace mxmoe {

cudaError_t launch_attend_e4m3(const DecodeParams& p, const DecodeScratch& ws, const DecodePlan& plan, cudaStream_t st) {
  // 32-bit queries or outputs keep 22 bits and more of queries and shares
  if (p.q_dtype == MXMOE_F32 || p.out_dtype == MXMOE_F32) {
    if (p.c.head_dim <= 64) return decode::launch<decode::E4m3<64, true>, 64>(p, ws, plan, st);
    if (p.c.head_dim <= 128) return decode::launch<decode::E4m3<128, true>, 128>(p, ws, plan, st);
    return decode::launch<decode::E4m3<256, true>, 256>(p, ws, plan, st);
  }
  if (p.c.head_dim <= 64) return decode::launch<decode::E4m3<64, false>, 64>(p, ws, plan, st);
  if (p.c.head_dim <= 128) return decode::launch<decode::E4m3<128, false>, 128>(p, ws, plan, st);
  return decode::launch<decode::E4m3<256, false>, 256>(p, ws, plan, st);
}

}  // namespace mxmoe
