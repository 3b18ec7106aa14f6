// pa_decode_mma.cu — pa_decode's instantiations of the decode kernel
// (pa_decode_kernel.cuh): fp16 / bf16, plain, cascade and fused gather.
#include "pa_decode_kernel.cuh"

namespace pa {

size_t decode_mma_smem_bytes(int D, int B, int stages, bool cascade) {
  const size_t stage_bytes = 2u * 16u * (size_t)D * 2u;
  return 1024 + (size_t)kDecodeWarps * stages * stage_bytes + (size_t)kDecodeWarps * stages * 8 +
         (size_t)((cascade ? 4 : 3) * B + 2) * 4;
}

template <typename T, int D, int kMode>
static cudaError_t launch_mma_impl(const DecodeParams& p, const CUtensorMap& tmk,
                                   const CUtensorMap& tmv, int grid, size_t smem, bool pdl,
                                   cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kDecodeWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl ? attr : nullptr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, decode_mma_kernel<T, D, kMode>, tmk, tmv, p);
}

template <int kMode>
static cudaError_t launch_mma(const DecodeParams& p, const CUtensorMap& tmk, const CUtensorMap& tmv, int dtype,
                              int grid, size_t smem, bool pdl, cudaStream_t stream) {
  if (dtype == PA_DTYPE_BFLOAT16) {
    if (p.D == 128) return launch_mma_impl<__nv_bfloat16, 128, kMode>(p, tmk, tmv, grid, smem, pdl, stream);
    if (p.D == 64) return launch_mma_impl<__nv_bfloat16, 64, kMode>(p, tmk, tmv, grid, smem, pdl, stream);
  } else if (dtype == PA_DTYPE_FLOAT16) {
    if (p.D == 128) return launch_mma_impl<__half, 128, kMode>(p, tmk, tmv, grid, smem, pdl, stream);
    if (p.D == 64) return launch_mma_impl<__half, 64, kMode>(p, tmk, tmv, grid, smem, pdl, stream);
  }
  return cudaErrorInvalidValue;
}

cudaError_t launch_decode_mma(const DecodeParams& p, const CUtensorMap& tmk, const CUtensorMap& tmv,
                              int dtype, int grid, size_t smem, bool pdl, cudaStream_t stream) {
  if (p.out_ranks != nullptr) return launch_mma<2>(p, tmk, tmv, dtype, grid, smem, pdl, stream);
  if (p.seq_group != nullptr) return launch_mma<1>(p, tmk, tmv, dtype, grid, smem, pdl, stream);
  return launch_mma<0>(p, tmk, tmv, dtype, grid, smem, pdl, stream);
}

template <int kMode>
static const void* decode_fn(int dtype, int D) {
  if (dtype == PA_DTYPE_BFLOAT16)
    return D == 128 ? (const void*)decode_mma_kernel<__nv_bfloat16, 128, kMode>
                    : (const void*)decode_mma_kernel<__nv_bfloat16, 64, kMode>;
  return D == 128 ? (const void*)decode_mma_kernel<__half, 128, kMode>
                  : (const void*)decode_mma_kernel<__half, 64, kMode>;
}

cudaError_t decode_mma_prepare(int dtype, int D, size_t smem) {
  const void* fns[3] = {decode_fn<0>(dtype, D), decode_fn<1>(dtype, D), decode_fn<2>(dtype, D)};
  for (const void* fn : fns) {
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace pa
