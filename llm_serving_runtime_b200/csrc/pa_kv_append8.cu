// pa_kv_append8.cu — append new K/V rows to a cache held in 8 bits (e4m3) with
// one scale for each block of tokens and KV head.
//
//   value of a code = code * scale[block, head]
//   need  = 2^e, the smallest e in [-100, 120] with amax <= 448 * 2^e
//           (amax: largest finite |x| of the block's new rows of one head)
//   scale = max(scale held, need); need alone when offset 0 of the block is
//           written, which starts the block anew
//   new codes = round(x / scale) (nearest even; infinities saturate, NaN stays)
//   held codes of the block's other tokens, when its scale grows:
//           round(code * held scale / scale)
//
// A scale that only ever grows by a power of two costs e4m3 nothing: codes move
// down whole binades and lose bits only where they become subnormal (below
// 2^-6 * scale).  A scale found in the cache need not be a power of two.
//
// A block's codes and scale have to be written together, so the work item is a
// run: all tokens of one call for one block.  One CTA takes a run, its warps
// take (head, K or V) pairs in turn.  Through a block table a row's runs follow
// from its position; through slot_mapping the CTA of each token looks whether
// that token opens a run (the row's previous slot lies in another block).  Two
// runs of one call in one block would race, so a CTA looks for an earlier run in
// its block first; it then leaves its own unwritten and flags it.  The runs'
// bytes are few, so latency decides; measured figures stand at the launcher.
#include <cuda_fp8.h>
#include <math.h>

#include "pa_common.cuh"
#include "pa_internal.h"

namespace pa {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxBlock = 256;  // tokens of a block

template <typename T>
__device__ __forceinline__ float widen(T x);
template <>
__device__ __forceinline__ float widen<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ float widen<__half>(__half x) {
  return __half2float(x);
}
template <>
__device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 x) {
  return __bfloat162float(x);
}

// Eight neighbouring elements; kWide: as 16-byte loads.
template <typename T, bool kWide>
__device__ __forceinline__ void load8(const T* src, float (&x)[8]) {
  if constexpr (kWide) {
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8 / N; ++i) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + i);
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int j = 0; j < N; ++j) x[i * N + j] = widen<T>(e[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = widen<T>(__ldg(src + i));
  }
}

__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

__device__ __forceinline__ float2 two_values(uint32_t codes) {
  __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

// 2^e with the smallest e in [-100, 120] for which amax <= 448 * 2^e = 1.75 * 2^(e + 8).
__device__ __forceinline__ float needed_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = max(e, -100);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Block of token i of the call through the block table, logical block lb of row b; -1: none.
__device__ __forceinline__ long long table_block(const AppendParams& p, int b, long long lb) {
  if (lb >= p.max_blocks) return -1;
  return p.block_tables[(long long)b * p.bt_stride + lb];
}

__device__ __forceinline__ long long first_position(const AppendParams& p, int b) {
  return (p.positions_is_int64 ? static_cast<const int64_t*>(p.positions)[b]
                               : (long long)static_cast<const int32_t*>(p.positions)[b]) +
         p.position_offset;
}

}  // namespace

template <typename T, bool kWide>
__global__ void __launch_bounds__(kThreads) kv_append8_kernel(const AppendParams p, const ScaleParams sc,
                                                              const int runs_per_row, const int bs_log2) {
  // the attention that follows may start its prologue; it waits for every write below
  pdl_launch_dependents();
  __shared__ int s_token[kMaxBlock];  // token of the row written at each offset, -1: none
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / runs_per_row, k = blockIdx.x - b * runs_per_row;
  const int bs = 1 << bs_log2;
  for (int o = tid; o < bs; o += kThreads) s_token[o] = -1;
  __syncthreads();

  long long blk;
  bool earlier = false;  // another run of the call writes this block before this one
  if (p.slot_mapping == nullptr) {
    const long long pos0 = first_position(p, b);
    if (pos0 < 0 && k == 0 && tid == 0) raise_flag(p.error_flags, PA_DEVERR_SLOT_RANGE);
    const long long lb = ((pos0 < 0 ? 0 : pos0) >> bs_log2) + k;
    const long long t0 = max(0LL, (lb << bs_log2) - pos0), t1 = min((long long)p.q_len, ((lb + 1) << bs_log2) - pos0);
    if (t0 >= t1) return;
    if (lb >= p.max_blocks) {
      if (tid == 0) raise_flag(p.error_flags, PA_DEVERR_TABLE_UNDERRUN);
      return;
    }
    blk = table_block(p, b, lb);
    for (long long t = t0 + tid; t < t1; t += kThreads) s_token[(int)((pos0 + t) & (bs - 1))] = (int)t;
    for (int r = tid; r < (int)blockIdx.x; r += kThreads) {
      const int b2 = r / runs_per_row;
      const long long q0 = first_position(p, b2);
      const long long lb2 = ((q0 < 0 ? 0 : q0) >> bs_log2) + (r - b2 * runs_per_row);
      if (((lb2 << bs_log2) < q0 + p.q_len) && q0 + p.q_len > 0) earlier |= table_block(p, b2, lb2) == blk;
    }
  } else {
    const int64_t* row = p.slot_mapping + (long long)b * p.q_len;
    if (row[k] < 0) return;  // padding
    blk = row[k] >> bs_log2;
    int prev = k - 1;
    while (prev >= 0 && row[prev] < 0) --prev;
    if (prev >= 0 && (row[prev] >> bs_log2) == blk) return;  // not the first token of its run
    // the run: up to the next slot of another block
    int end = k + 1;
    while (end < p.q_len && (row[end] < 0 || (row[end] >> bs_log2) == blk)) ++end;
    for (int t = k + tid; t < end; t += kThreads)
      if (row[t] >= 0) atomicMax(&s_token[(int)(row[t] & (bs - 1))], t);  // a slot given twice: the last one
    for (int i = tid; i < (int)blockIdx.x; i += kThreads)
      earlier |= p.slot_mapping[i] >= 0 && (p.slot_mapping[i] >> bs_log2) == blk;
  }
  const bool any_earlier = __syncthreads_or(earlier);  // also: s_token is complete
  if (blk < 0 || blk >= p.num_blocks) {
    if (tid == 0)
      raise_flag(p.error_flags, p.slot_mapping != nullptr ? PA_DEVERR_SLOT_RANGE : PA_DEVERR_BLOCK_ID_RANGE);
    return;
  }
  if (any_earlier) {
    if (tid == 0) raise_flag(p.error_flags, PA_DEVERR_BLOCK_CONFLICT);
    return;
  }
  const bool fresh = s_token[0] >= 0;
  const int chunks = p.D >> 3;  // of 8 elements
  const int items = bs * chunks;

  for (int hv = warp; hv < 2 * p.Hkv; hv += kThreads / 32) {
    const int h = hv >> 1;
    const bool is_v = hv & 1;
    const T* src = is_v ? static_cast<const T*>(p.value) + (long long)b * p.v_sb + (long long)h * p.v_sh
                        : static_cast<const T*>(p.key) + (long long)b * p.k_sb + (long long)h * p.k_sh;
    const int64_t src_t = is_v ? p.v_st : p.k_st;
    uint8_t* dst = is_v ? static_cast<uint8_t*>(p.v_cache) + blk * p.vc_sblk + (long long)h * p.vc_sh
                        : static_cast<uint8_t*>(p.k_cache) + blk * p.kc_sblk + (long long)h * p.kc_sh;
    const int64_t dst_t = is_v ? p.vc_st : p.kc_st;
    float* scale_at = is_v ? sc.v_scales + blk * sc.vs_sblk + h * sc.vs_sh
                           : sc.k_scales + blk * sc.ks_sblk + h * sc.ks_sh;
    float held = *scale_at;
    held = (!fresh && held > 0.f && held < INFINITY) ? held : 0.f;

    float amax = 0.f;
    for (int i = lane; i < items; i += 32) {
      const int o = i / chunks, t = s_token[o];
      if (t < 0) continue;
      float x[8];
      load8<T, kWide>(src + t * src_t + (i - o * chunks) * 8, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = fabsf(x[j]);
        if (a < INFINITY) amax = fmaxf(amax, a);  // not for NaN either
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float scale = fmaxf(held, needed_scale(amax));
    const bool pow2 = (__float_as_uint(scale) & 0x7fffffu) == 0u;
    const float inv = 1.f / scale;  // exact where scale is a power of two
    for (int i = lane; i < items; i += 32) {
      const int o = i / chunks, t = s_token[o];
      if (t < 0) continue;
      float x[8];
      load8<T, kWide>(src + t * src_t + (i - o * chunks) * 8, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = pow2 ? x[j] * inv : __fdiv_rn(x[j], scale);
      *reinterpret_cast<uint2*>(dst + o * dst_t + (i - o * chunks) * 8) =
          make_uint2(codes4(x[0], x[1], x[2], x[3]), codes4(x[4], x[5], x[6], x[7]));
    }
    if (!fresh && scale != held) {
      const float ratio = __fdiv_rn(held, scale);
      for (int i = lane; i < items; i += 32) {
        const int o = i / chunks;
        if (s_token[o] >= 0) continue;
        uint2* at = reinterpret_cast<uint2*>(dst + o * dst_t + (i - o * chunks) * 8);
        const uint2 c = *at;
        float2 f[4] = {two_values(c.x), two_values(c.x >> 16), two_values(c.y), two_values(c.y >> 16)};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[j].x *= ratio;
          f[j].y *= ratio;
        }
        *at = make_uint2(codes4(f[0].x, f[0].y, f[1].x, f[1].y), codes4(f[2].x, f[2].y, f[3].x, f[3].y));
      }
    }
    if (lane == 0 && (fresh || scale != held)) *scale_at = scale;
  }
}

template <typename T>
static cudaError_t launch_typed(const AppendParams& p, const ScaleParams& sc, bool wide, int runs, int bs_log2,
                                cudaStream_t stream) {
  const unsigned grid = (unsigned)((long long)p.B * runs);
  if (wide)
    kv_append8_kernel<T, true><<<grid, kThreads, 0, stream>>>(p, sc, runs, bs_log2);
  else
    kv_append8_kernel<T, false><<<grid, kThreads, 0, stream>>>(p, sc, runs, bs_log2);
  return cudaGetLastError();
}

cudaError_t launch_kv_append8(const AppendParams& p, const ScaleParams& sc, int dtype, cudaStream_t stream) {
  int bs_log2 = 0;
  while ((1 << bs_log2) < p.bs) ++bs_log2;
  const int runs = p.slot_mapping != nullptr ? p.q_len : (p.q_len + p.bs - 2) / p.bs + 1;
  auto ok_str = [&](int64_t s) { return (s * p.elem_bytes) % 16 == 0; };
  const bool wide = reinterpret_cast<uintptr_t>(p.key) % 16 == 0 && reinterpret_cast<uintptr_t>(p.value) % 16 == 0 &&
                    ok_str(p.k_sb) && ok_str(p.k_sh) && ok_str(p.k_st) && ok_str(p.v_sb) && ok_str(p.v_sh) &&
                    ok_str(p.v_st);
  if (dtype == PA_DTYPE_BFLOAT16) return launch_typed<__nv_bfloat16>(p, sc, wide, runs, bs_log2, stream);
  if (dtype == PA_DTYPE_FLOAT16) return launch_typed<__half>(p, sc, wide, runs, bs_log2, stream);
  return launch_typed<float>(p, sc, wide, runs, bs_log2, stream);
}

}  // namespace pa
