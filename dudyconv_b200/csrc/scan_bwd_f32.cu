// scan_bwd_f32.cu -- the selective scan's gradients for float tensors (scan_bwd.cuh).
#include "scan_bwd.cuh"

namespace dudy {
namespace scan {

int bwd_chain_f32(int lpc, bool four, const Bwd &a, const Shape &s, int64_t tiles,
                  cudaStream_t st) {
  return bwd_chain_by<float>(lpc, four, a, s, tiles, st);
}

}  // namespace scan
}  // namespace dudy
