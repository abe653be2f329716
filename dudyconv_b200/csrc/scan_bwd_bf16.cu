// scan_bwd_bf16.cu -- the selective scan's gradients for __nv_bfloat16 tensors (scan_bwd.cuh).
#include "scan_bwd.cuh"

namespace dudy {
namespace scan {

int bwd_chain_bf16(int lpc, bool four, const Bwd &a, const Shape &s, int64_t tiles,
                   cudaStream_t st) {
  return bwd_chain_by<__nv_bfloat16>(lpc, four, a, s, tiles, st);
}

}  // namespace scan
}  // namespace dudy
