// The kernels of block_norm.cuh for float (one type a file: they compile side by side).
#include "block_norm.cuh"

namespace adops {
cudaError_t start_norm_f32(const NormArgs& a, bool grad, bool gen, bool vec, unsigned blocks, int sms, cudaStream_t s) {
  return start_norm_typed<float>(a, grad, gen, vec, blocks, sms, s);
}
}  // namespace adops
