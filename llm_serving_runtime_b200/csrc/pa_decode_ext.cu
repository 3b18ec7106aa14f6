// pa_decode_ext.cu — pa_decode_ext's instantiations of the decode kernel
// (pa_decode_kernel.cuh): 8-bit caches, changed scores, and both.
#include "pa_decode_kernel.cuh"

namespace pa {

size_t decode_ext_smem_bytes(int D, int B, int stages, bool eight, bool scored) {
  const size_t stage_bytes = 2u * 16u * (size_t)D * 2u;  // 16 tokens of 2 bytes, or 32 of 1
  return 1024 + (size_t)kDecodeWarps * stages * (stage_bytes + 8 + (eight ? 32 : 0)) +
         ((size_t)decode_seq_tables(false, scored) * B + 2) * 4;
}

namespace {

template <typename T, int D, typename KV, bool kScored>
cudaError_t launch(const DecodeParams& p, const CUtensorMap& tmk, const CUtensorMap& tmv, int grid, size_t smem,
                   bool pdl, cudaStream_t stream) {
  // Shared memory beyond the default limit, once per device (the largest a block may have).
  static bool prepared[64] = {false};
  int dev = 0, most = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!prepared[dev]) {
    e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
    if (e != cudaSuccess) return e;
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, decode_mma_kernel<T, D, 0, KV, kScored>);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(decode_mma_kernel<T, D, 0, KV, kScored>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             most - (int)fa.sharedSizeBytes);
    if (e != cudaSuccess) return e;
    prepared[dev] = true;
  }
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
  return cudaLaunchKernelEx(&cfg, decode_mma_kernel<T, D, 0, KV, kScored>, tmk, tmv, p);
}

template <typename T, int D>
cudaError_t pick(const DecodeParams& p, const CUtensorMap& tmk, const CUtensorMap& tmv, int grid, size_t smem,
                 bool pdl, cudaStream_t stream) {
  if (p.k_scales == nullptr) return launch<T, D, T, true>(p, tmk, tmv, grid, smem, pdl, stream);
  if (p.scored) return launch<T, D, e4m3_t, true>(p, tmk, tmv, grid, smem, pdl, stream);
  return launch<T, D, e4m3_t, false>(p, tmk, tmv, grid, smem, pdl, stream);
}

}  // namespace

cudaError_t launch_decode_ext(const DecodeParams& p, const CUtensorMap& tmk, const CUtensorMap& tmv, int dtype,
                              int grid, size_t smem, bool pdl, cudaStream_t stream) {
  if (dtype == PA_DTYPE_BFLOAT16)
    return p.D == 128 ? pick<__nv_bfloat16, 128>(p, tmk, tmv, grid, smem, pdl, stream)
                      : pick<__nv_bfloat16, 64>(p, tmk, tmv, grid, smem, pdl, stream);
  return p.D == 128 ? pick<__half, 128>(p, tmk, tmv, grid, smem, pdl, stream)
                    : pick<__half, 64>(p, tmk, tmv, grid, smem, pdl, stream);
}

}  // namespace pa
