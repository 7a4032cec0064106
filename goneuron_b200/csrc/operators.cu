// operators.cu -- operators of language models on device memory (C ABI: the last part of goneuron_cuda.h).
#include "device_ops.cuh"
#include "op_qk_norm_rope.cuh"
#include "op_distill.cuh"
#include "op_embedding.cuh"
#include "op_gated_ffn.cuh"

namespace gn {
__global__ void op_status_clear_kernel(int bits) { op_begin(); atomicAnd(&op_status_word, ~bits); }
}  // namespace gn

extern "C" int gn_op_status(gn_ctx* ctx, void* stream) {
  using namespace gn;
  GN_OP_BEGIN("op_status", nullptr);
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  GN_CUDA(cudaStreamIsCapturing((cudaStream_t)stream, &cap));
  if (cap != cudaStreamCaptureStatusNone) return fail(GN_ERR_INVALID_ARG, "op_status: the stream is being captured");
  int bits = 0;
  GN_CUDA(cudaMemcpyFromSymbolAsync(&bits, op_status_word, sizeof bits, 0, cudaMemcpyDeviceToHost, (cudaStream_t)stream));
  GN_CUDA(cudaStreamSynchronize((cudaStream_t)stream));
  if (bits == 0) return GN_OK;
  GN_TRY(op_launch("op_status", stream, op_status_clear_kernel, dim3(1), dim3(1), 0, 0, bits));
  GN_CUDA(cudaStreamSynchronize((cudaStream_t)stream));
  if (bits & OP_TIMEOUT) return fail(GN_ERR_TIMEOUT, "a bounded device-side wait of an operator gave up: its outputs are not valid");
  return fail(GN_ERR_INVALID_ARG, "an operator met an index out of range and treated it as -1");
}
