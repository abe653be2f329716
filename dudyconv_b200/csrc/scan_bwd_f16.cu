// scan_bwd_f16.cu -- the selective scan's gradients for __half tensors (scan_bwd.cuh).
#include "scan_bwd.cuh"

namespace dudy {
namespace scan {

int bwd_chain_f16(int lpc, bool four, const Bwd &a, const Shape &s, int64_t tiles,
                  cudaStream_t st) {
  return bwd_chain_by<__half>(lpc, four, a, s, tiles, st);
}

}  // namespace scan
}  // namespace dudy
