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
// run: all tokens of one call for one block.  A CTA takes a run and up to eight
// (head, K or V) pairs of it, a warp each.  Through a block table a row's runs follow
// from its position; through slot_mapping a CTA looks which of a block's number of
// tokens open a run (the row's previous slot lies in another block) and takes those.  Two
// runs of one call in one block would race, so a CTA looks for an earlier run in
// its block first; it then leaves its own unwritten and flags it.
//
// The bytes are few, so latency decides: a warp loads its share of the run (up to
// 256 pieces of 8 elements, a 16-token block of 128 columns) into registers at once,
// before the look at the other runs, and rounds it from there; longer runs
// are read twice.  Four CTAs an SM (64 registers) hold a prefill chunk in one wave.
// Measured: 8 x 509 tokens, 8 heads of 128 (25 MB) 8.6 us (18.5 with a warp reading
// piece by piece for two pairs, 20.9 with two CTAs an SM); 64 rows of one token 4.1 us.
// The look at other runs grows with the square of their number, in the slot form of
// the tokens: 8192 tokens of one row 19 us through tables, 29 through slots; 131,072
// tokens 368 and 1017.  A long prompt is written through tables.
#include <cuda_fp8.h>
#include <limits.h>
#include <math.h>

#include "pa_common.cuh"
#include "pa_internal.h"
#include "pa_tile_math.cuh"

namespace pa {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxBlock = 256;  // tokens of a block
constexpr int kBatch = 8;       // pieces of 8 elements that a lane holds
constexpr int kHeld = 4;        // and of codes that are rounded again

// Eight neighbouring elements as they are in memory, and widened; kWide: loaded
// 16 bytes at a time.
template <typename T>
struct Piece {
  static constexpr int kWords = 8 * sizeof(T) / 4;
  uint32_t w[kWords];

  template <bool kWide>
  __device__ __forceinline__ void load(const T* src) {
    if constexpr (kWide) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + i);
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(__ldg(src + i));
    } else {
      const unsigned short* u = reinterpret_cast<const unsigned short*>(src);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__ldg(u + 2 * i) | ((uint32_t)__ldg(u + 2 * i + 1) << 16);
    }
  }
  __device__ __forceinline__ void widen(float (&x)[8]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = lo_half<T>(w[i]);
        x[2 * i + 1] = hi_half<T>(w[i]);
      }
    }
  }
};

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

// kSlots: through slot_mapping; a CTA takes the runs that open among one block's number of
// neighbouring tokens of a row, one after the other.
template <typename T, bool kWide, bool kSlots>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 4 : 2)
    kv_append8_kernel(const AppendParams p, const ScaleParams sc, const int runs_per_row, const int bs_log2,
                      const int chunks_log2) {
  // the attention that follows may start its prologue; it waits for every write below
  pdl_launch_dependents();
  // The run's tokens: offset in the block (low byte) and token of the row, in any
  // order; and which offsets of the block they take.
  __shared__ int2 s_run[kMaxBlock];
  __shared__ int s_token[kSlots ? kMaxBlock : 1];       // token of the row at each offset, -1: none
  __shared__ long long s_block[kSlots ? kMaxBlock : 1];  // block of each of the CTA's tokens, -1: padding
  __shared__ int s_open[kSlots ? kMaxBlock : 1];         // tokens that open a run
  __shared__ int s_count, s_found, s_opens;
  __shared__ uint32_t s_taken[kMaxBlock / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x;
  const int b = blockIdx.x / runs_per_row, k = blockIdx.x - b * runs_per_row;
  const int bs = 1 << bs_log2;

  // Block of run r of the call (-1: none), for the look at earlier runs.
  auto block_of_run = [&](int r) -> long long {
    const int b2 = r / runs_per_row;
    const long long q0 = first_position(p, b2);
    const long long lb2 = ((q0 < 0 ? 0 : q0) >> bs_log2) + (r - b2 * runs_per_row);
    return ((lb2 << bs_log2) < q0 + p.q_len) && q0 + p.q_len > 0 ? table_block(p, b2, lb2) : -1;
  };
  const int64_t* row = kSlots ? p.slot_mapping + (long long)b * p.q_len : nullptr;
  // kReach slots of each thread at a time: padding between a run's tokens may be
  // long (a padded batch)
  [[maybe_unused]] constexpr int kReach = 8;
  if constexpr (kSlots) {
    const int k0 = k << bs_log2, span = min(bs, p.q_len - k0);
    if (tid == 0) {
      s_opens = 0;
      s_found = -1;
    }
    int any = 0;
    for (int i = tid; i < span; i += threads) {
      const int64_t at = row[k0 + i];
      s_block[i] = at < 0 ? -1 : at >> bs_log2;
      any |= at >= 0;
    }
    if (!__syncthreads_or(any)) return;
    // the block before: of the row's last slot that is no padding
    for (int base = k0 - 1; base >= 0; base -= threads * kReach) {
      if (base == k0 - 1 && row[base] >= 0) {  // as a rule the neighbour's
        if (tid == 0) s_found = base;
        __syncthreads();
        break;
      }
      int last = -1;
#pragma unroll
      for (int j = 0; j < kReach; ++j) {
        const int i = base - (j * threads + tid);
        if (i >= 0 && row[i] >= 0) last = max(last, i);
      }
      if (last >= 0) atomicMax(&s_found, last);
      __syncthreads();
      const int found = s_found;
      __syncthreads();
      if (found >= 0) break;
    }
    const long long before = s_found >= 0 ? row[s_found] >> bs_log2 : -1;
    for (int i = tid; i < span; i += threads) {
      if (s_block[i] < 0) continue;
      int j = i - 1;
      while (j >= 0 && s_block[j] < 0) --j;
      if ((j >= 0 ? s_block[j] : before) != s_block[i]) s_open[atomicAdd(&s_opens, 1)] = k0 + i;
    }
    __syncthreads();
  }

  for (int turn = 0; turn < (kSlots ? s_opens : 1); ++turn) {
    long long blk, other = -1;
    int count, first_index = blockIdx.x;  // of the run: nothing of the call before it may lie in its block
    if constexpr (!kSlots) {
      if (tid < (int)blockIdx.x) other = block_of_run(tid);  // in flight beside this run's own
      const long long pos0 = first_position(p, b);
      if (pos0 < 0 && k == 0 && tid == 0 && blockIdx.y == 0 && !empty_row(p, pos0 - p.position_offset))
        raise_flag(p.error_flags, PA_DEVERR_SLOT_RANGE);
      const long long lb = ((pos0 < 0 ? 0 : pos0) >> bs_log2) + k;
      const long long t0 = max(0LL, (lb << bs_log2) - pos0), t1 = min((long long)p.q_len, ((lb + 1) << bs_log2) - pos0);
      if (t0 >= t1) return;
      if (lb >= p.max_blocks) {
        if (tid == 0 && blockIdx.y == 0) raise_flag(p.error_flags, PA_DEVERR_TABLE_UNDERRUN);
        return;
      }
      blk = table_block(p, b, lb);
      count = (int)(t1 - t0);
      for (int i = tid; i < count; i += threads) s_run[i] = make_int2((int)((pos0 + t0 + i) & (bs - 1)), (int)t0 + i);
      if (tid < kMaxBlock / 32) {  // offsets first .. first + count - 1
        const int first = (int)((pos0 + t0) & (bs - 1)) - 32 * tid, last = first + count;
        const uint32_t from = first <= 0 ? ~0u : first >= 32 ? 0u : ~0u << first;
        const uint32_t to = last >= 32 ? ~0u : last <= 0 ? 0u : ~(~0u << last);
        s_taken[tid] = from & to;
      }
    } else {
      const int k_open = s_open[turn];
      first_index = b * p.q_len + k_open;
      blk = s_block[k_open - (k << bs_log2)];
      __syncthreads();  // the run before is done
      for (int o = tid; o < bs; o += threads) s_token[o] = -1;
      if (tid < kMaxBlock / 32) s_taken[tid] = 0u;
      if (tid == 0) {
        s_count = 0;
        s_found = INT_MAX;
      }
      __syncthreads();
      // the next slot of another block ends the run
      for (int base = k_open + 1; base < p.q_len; base += threads * kReach) {
        int next = INT_MAX;
#pragma unroll
        for (int j = 0; j < kReach; ++j) {
          const int i = base + j * threads + tid;
          if (i < p.q_len && row[i] >= 0 && (row[i] >> bs_log2) != blk) next = min(next, i);
        }
        if (next < INT_MAX) atomicMin(&s_found, next);
        __syncthreads();
        const int found = s_found;
        __syncthreads();
        if (found < INT_MAX) break;
      }
      const int end = min(s_found, p.q_len);
      for (int t = k_open + tid; t < end; t += threads)
        if (row[t] >= 0) atomicMax(&s_token[(int)(row[t] & (bs - 1))], t);  // a slot given twice: the last one
      __syncthreads();
      for (int o = tid; o < bs; o += threads)
        if (s_token[o] >= 0) {
          s_run[atomicAdd(&s_count, 1)] = make_int2(o, s_token[o]);
          atomicOr(&s_taken[o >> 5], 1u << (o & 31));
        }
      __syncthreads();
      count = s_count;
    }
    __syncthreads();  // the run is complete

    // ---- this warp's pair: K or V of one head ----
    const int hv = blockIdx.y * (kThreads / 32) + warp;
    const bool mine = hv < 2 * p.Hkv;
    const int h = hv >> 1;
    const bool is_v = hv & 1;
    const int chunks = p.D >> 3;  // of 8 elements
    const int items = mine ? count * chunks : 0;
    const T* src = is_v ? static_cast<const T*>(p.value) + (long long)b * p.v_sb + (long long)h * p.v_sh
                        : static_cast<const T*>(p.key) + (long long)b * p.k_sb + (long long)h * p.k_sh;
    const int64_t src_t = is_v ? p.v_st : p.k_st;
    // Piece i of the run: 8 elements from column 8 c of its i / chunks-th token.
    auto token_of = [&](int i) -> int { return chunks_log2 >= 0 ? i >> chunks_log2 : i / chunks; };
    Piece<T> x[kBatch];
    auto load = [&](int base) {
#pragma unroll
      for (int n = 0; n < kBatch; ++n) {
        const int i = base + n * 32 + lane;
        if (i >= items) continue;
        const int r = token_of(i);
        x[n].template load<kWide>(src + s_run[r].y * src_t + (i - r * chunks) * 8);
      }
    };
    load(0);
    const bool in_pool = blk >= 0 && blk < p.num_blocks;
    float* scale_at = is_v ? sc.v_scales + blk * sc.vs_sblk + h * sc.vs_sh
                           : sc.k_scales + blk * sc.ks_sblk + h * sc.ks_sh;
    float held = in_pool && mine ? *scale_at : 0.f;

    bool earlier = other == blk && blk >= 0;  // another run of the call writes this block before this one
    if constexpr (!kSlots) {
#pragma unroll 4
      for (int r = tid + threads; r < (int)blockIdx.x; r += threads) earlier |= block_of_run(r) == blk;
    } else {
#pragma unroll 4
      for (int i = tid; i < first_index; i += threads)
        earlier |= p.slot_mapping[i] >= 0 && (p.slot_mapping[i] >> bs_log2) == blk;
    }
    const bool any_earlier = __syncthreads_or(earlier);
    if (!in_pool) {
      if (tid == 0 && blockIdx.y == 0)
        raise_flag(p.error_flags, kSlots ? PA_DEVERR_SLOT_RANGE : PA_DEVERR_BLOCK_ID_RANGE);
      continue;
    }
    if (any_earlier) {
      if (tid == 0 && blockIdx.y == 0) raise_flag(p.error_flags, PA_DEVERR_BLOCK_CONFLICT);
      continue;
    }
    if (!mine) continue;
    const bool fresh = s_taken[0] & 1u;
    uint8_t* dst = is_v ? static_cast<uint8_t*>(p.v_cache) + blk * p.vc_sblk + (long long)h * p.vc_sh
                        : static_cast<uint8_t*>(p.k_cache) + blk * p.kc_sblk + (long long)h * p.kc_sh;
    const int64_t dst_t = is_v ? p.vc_st : p.kc_st;
    held = (!fresh && held > 0.f && held < INFINITY) ? held : 0.f;

    float amax = 0.f;
    for (int base = 0; base < items; base += kBatch * 32) {
      if (base > 0) load(base);
#pragma unroll
      for (int n = 0; n < kBatch; ++n) {
        if (base + n * 32 + lane >= items) continue;
        float v[8];
        x[n].widen(v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float a = fabsf(v[j]);
          if (a < INFINITY) amax = fmaxf(amax, a);  // not for NaN either
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float scale = fmaxf(held, needed_scale(amax));
    if ((__float_as_uint(scale) & 0x7fffffu) == 0u) {
      const float inv = 1.f / scale;  // exact: a power of two
      for (int base = 0; base < items; base += kBatch * 32) {
        if (items > kBatch * 32) load(base);
#pragma unroll
        for (int n = 0; n < kBatch; ++n) {
          const int i = base + n * 32 + lane;
          if (i >= items) continue;
          float v[8];
          x[n].widen(v);
          const int r = token_of(i);
          *reinterpret_cast<uint2*>(dst + s_run[r].x * dst_t + (i - r * chunks) * 8) =
              make_uint2(codes4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                         codes4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
        }
      }
    } else {
      // a scale that was found in the cache; short code (the kernel runs once, its fetch counts)
#pragma unroll 1
      for (int i = lane; i < items; i += 32) {
        const int r = token_of(i);
        Piece<T> y;
        y.template load<kWide>(src + s_run[r].y * src_t + (i - r * chunks) * 8);
        float v[8];
        y.widen(v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fdiv_rn(v[j], scale);
        *reinterpret_cast<uint2*>(dst + s_run[r].x * dst_t + (i - r * chunks) * 8) =
            make_uint2(codes4(v[0], v[1], v[2], v[3]), codes4(v[4], v[5], v[6], v[7]));
      }
    }
    if (!fresh && scale != held) {
      // the block's other tokens to the new scale
      const float ratio = __fdiv_rn(held, scale);
      for (int base = 0; base < bs * chunks; base += kHeld * 32) {
        uint2 c[kHeld];
#pragma unroll
        for (int n = 0; n < kHeld; ++n) {
          const int i = base + n * 32 + lane, o = token_of(i);
          if (i < bs * chunks && !((s_taken[o >> 5] >> (o & 31)) & 1u))
            c[n] = *reinterpret_cast<const uint2*>(dst + o * dst_t + (i - o * chunks) * 8);
        }
#pragma unroll
        for (int n = 0; n < kHeld; ++n) {
          const int i = base + n * 32 + lane, o = token_of(i);
          if (i >= bs * chunks || ((s_taken[o >> 5] >> (o & 31)) & 1u)) continue;
          float2 f[4] = {two_values(c[n].x), two_values(c[n].x >> 16), two_values(c[n].y), two_values(c[n].y >> 16)};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            f[j].x *= ratio;
            f[j].y *= ratio;
          }
          *reinterpret_cast<uint2*>(dst + o * dst_t + (i - o * chunks) * 8) =
              make_uint2(codes4(f[0].x, f[0].y, f[1].x, f[1].y), codes4(f[2].x, f[2].y, f[3].x, f[3].y));
        }
      }
    }
    if (lane == 0 && (fresh || scale != held)) *scale_at = scale;
  }
}

template <typename T>
static cudaError_t launch_typed(const AppendParams& p, const ScaleParams& sc, bool wide, int runs, int bs_log2,
                                cudaStream_t stream) {
  const int pairs = 2 * p.Hkv, warps = kThreads / 32;
  const dim3 grid((unsigned)((long long)p.B * runs), (unsigned)((pairs + warps - 1) / warps));
  const int threads = pairs < warps ? 32 * pairs : kThreads;
  const int chunks = p.D / 8;
  int chunks_log2 = -1;  // of a power of two
  if ((chunks & (chunks - 1)) == 0)
    for (chunks_log2 = 0; (1 << chunks_log2) < chunks;) ++chunks_log2;
  const auto through_slots = wide ? kv_append8_kernel<T, true, true> : kv_append8_kernel<T, false, true>;
  const auto through_tables = wide ? kv_append8_kernel<T, true, false> : kv_append8_kernel<T, false, false>;
  const auto kernel = p.slot_mapping != nullptr ? through_slots : through_tables;
  kernel<<<grid, threads, 0, stream>>>(p, sc, runs, bs_log2, chunks_log2);
  return cudaGetLastError();
}

cudaError_t launch_kv_append8(const AppendParams& p, const ScaleParams& sc, int dtype, cudaStream_t stream) {
  int bs_log2 = 0;
  while ((1 << bs_log2) < p.bs) ++bs_log2;
  const int runs = p.slot_mapping != nullptr ? (p.q_len + p.bs - 1) / p.bs : (p.q_len + p.bs - 2) / p.bs + 1;
  auto ok_str = [&](int64_t s) { return (s * p.elem_bytes) % 16 == 0; };
  const bool wide = reinterpret_cast<uintptr_t>(p.key) % 16 == 0 && reinterpret_cast<uintptr_t>(p.value) % 16 == 0 &&
                    ok_str(p.k_sb) && ok_str(p.k_sh) && ok_str(p.k_st) && ok_str(p.v_sb) && ok_str(p.v_sh) &&
                    ok_str(p.v_st);
  if (dtype == PA_DTYPE_BFLOAT16) return launch_typed<__nv_bfloat16>(p, sc, wide, runs, bs_log2, stream);
  if (dtype == PA_DTYPE_FLOAT16) return launch_typed<__half>(p, sc, wide, runs, bs_log2, stream);
  return launch_typed<float>(p, sc, wide, runs, bs_log2, stream);
}

}  // namespace pa
