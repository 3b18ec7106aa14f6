// pa_decode_direct.cu — pa_decode_ext for few rows, or rows that cannot be long: a
// row (sequence, KV head, group of 16 query rows) gets CTAs of its own.
//
// The stream-K kernel (pa_decode_kernel.cuh) balances any batch, but a warp that
// crosses rows pays for each start and end, a warp's least share is several units,
// and a long row's many pieces are merged by one warp.  None of that is needed here:
// CTA (row, s) takes the s-th of S equal ranges of the row's units, its warps an equal
// part of it each (their own ring of TMA tiles, as there), and merges their states in shared memory; the last CTA
// of a row to finish merges the S partial states, all threads together, with the
// log-sum-exp rule, in the order of the ranges.  S is at most the launch's second
// dimension and leaves every CTA chunk_units units or more (known on the device
// only: further CTAs leave at once).  The rule on shapes and sizes that calls it
// is in pa_capi.cu, with what was measured.
//
// Bound: issue and latency of a unit's chain (products, maxima, exponentials; 170
// registers leave 12 warps an SM), then what a row pays once.  96 x 4 tokens of 16
// to 2048 cached ones, 8 KV heads (768 rows, 90 MB of codes) 38 us at 1.7 instructions
// a clock; a CTA pays 3 us for lengths, table, first tile and merge, and its queries
// and output.  128 rows with a window of 1024 (16-bit, 441 MB) 77 us, 5.7 TB/s; one row of
// 32k 20 us, 3.3 TB/s.
#include "pa_common.cuh"
#include "pa_internal.h"
#include "pa_tile_ext.cuh"
#include "pa_tile_math.cuh"

namespace pa {

namespace {
constexpr int kMaxSplits = kDirectMaxSplits;
// Warps of a CTA, and CTAs an SM is built for.  Few rows: one CTA with all warps,
// so that a row's share is spread widest.  Many rows: several smaller CTAs, whose
// starts and ends overlap the others' work.
template <typename KV, bool kMany>
struct Shape {
  static constexpr int kWarps = kIs8<KV>::value ? (kMany ? 4 : 12) : (kMany ? 6 : 8);
  static constexpr int kCtas = kMany ? (kIs8<KV>::value ? 3 : 2) : 1;
};
}  // namespace

template <typename T, int D, typename KV, bool kScored, bool kMany>
__global__ void __launch_bounds__(Shape<KV, kMany>::kWarps * 32, Shape<KV, kMany>::kCtas)
    decode_direct_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                         const DecodeParams p) {
  constexpr bool k8 = kIs8<KV>::value;
  constexpr int kWarps = Shape<KV, kMany>::kWarps;
  using TL = TileLayout<KV, D>;
  constexpr int UT = TL::kTokens;
  constexpr int HALVES = TL::kHalves;
  constexpr uint32_t TILE_BYTES = TL::kTileBytes;
  constexpr uint32_t STAGE_BYTES = 2 * TILE_BYTES;
  // Rows of the CTA's shared arrays, padded so that the fragments' accesses (8 rows x
  // 4 lanes) fall into different banks: staged query rows (words; the merge's weights
  // take their place), and a warp's accumulator (floats).
  constexpr int WT = k8 ? 72 : 68;
  constexpr int AS = D + 8;
  static_assert(D / 2 <= 64 && kMaxSplits <= 64, "rows of s_wt");
  static_assert(16 * AS * 4 <= 2 * STAGE_BYTES, "an accumulator lies in two stages");

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_addr(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  const int stages = p.stages;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (size_t)kWarps * stages * STAGE_BYTES);
  float4* s_scales = reinterpret_cast<float4*>(bars + kWarps * stages);
  __shared__ float s_m[kWarps][16], s_l[kWarps][16];
  __shared__ __align__(16) float s_wt[16][WT];
  __shared__ const T* s_qrow[16];
  __shared__ T* s_orow[16];
  __shared__ float s_ref[16], s_norm[16];
  __shared__ int s_min_start, s_last;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane & 3;
  const int row = blockIdx.x, split = blockIdx.y;
  const int mg = row % p.NMG, h = (row / p.NMG) % p.Hkv, b = row / (p.NMG * p.Hkv);
  const int rows_here = min(16, p.GQ - 16 * mg);
  const int t_first = 16 * mg / p.G, t_last = (16 * mg + rows_here - 1) / p.G;

  int L = p.context_lens[b] + p.len_offset;
  if (lane < stages) mbar_init(smem_addr(&bars[warp * stages + lane]), k8 ? 9 : 1);
  if (tid < rows_here) {
    const int t = (16 * mg + tid) / p.G, hq = h * p.G + (16 * mg + tid - t * p.G);
    s_qrow[tid] = static_cast<const T*>(p.q) + (long long)b * p.q_sb + (long long)hq * p.q_sh + (long long)t * p.q_st;
    s_orow[tid] = static_cast<T*>(p.out) + (long long)b * p.o_sb + (long long)hq * p.o_sh + (long long)t * p.o_st;
  }
  if (tid == 0) {
    prefetch_tensormap(&tmk);
    prefetch_tensormap(&tmv);
    s_min_start = p.key_starts != nullptr ? INT_MAX : 0;
  }
  fence_mbar_init();
  __syncthreads();

  // ---- the row's units, and this warp's share ----
  const int cap = p.max_blocks * p.bs;
  if (L > cap) {
    if (tid == 0 && h == 0 && mg == 0 && split == 0) raise_flag(p.status, PA_DEVERR_TABLE_UNDERRUN);
    L = cap;
  }
  if (L < 0) L = 0;
  int lo = 0, hi;
  if constexpr (kScored) {
    const int prefix = p.prefix_lens != nullptr ? __ldg(&p.prefix_lens[b]) : 0;
    if (p.key_starts != nullptr) {
      if (warp == 0)
        for (int t = t_first + lane; t <= t_last; t += 32)
          atomicMin(&s_min_start, __ldg(&p.key_starts[b * p.kst_sb + t * p.kst_st]));
      __syncthreads();
    }
    lo = key_range(L, p.q_len, t_first, p.window, s_min_start, prefix).first;
    hi = key_range(L, p.q_len, t_last, 0, 0, prefix).end;
  } else {
    hi = key_range(L, p.q_len, t_last, 0, 0, 0).end;
  }
  const int u_first = lo / UT;
  const int n = hi > lo ? (hi + UT - 1) / UT - u_first : 0;
  const int S = max(1, min((int)gridDim.y, (n + p.chunk_units - 1) / p.chunk_units));
  if (split >= S) return;
  const int c0 = (int)((long long)n * split / S), c1 = (int)((long long)n * (split + 1) / S);
  const int w0 = u_first + c0 + (c1 - c0) * warp / kWarps, w1 = u_first + c0 + (c1 - c0) * (warp + 1) / kWarps;

  const int bs = p.bs, bs_log2 = 31 - __clz(bs);
  const uint32_t ring = smem_addr(smem) + (uint32_t)(warp * stages) * STAGE_BYTES;
  const uint32_t my_bars = smem_addr(&bars[warp * stages]);
  const uint64_t kv_policy = l2_policy_evict_first();
  int win_base = 0, win_val = -1;
  auto load_window = [&](int lb) {
    win_base = lb;
    const int e = lb + lane;
    win_val = e < p.max_blocks ? __ldg(&p.block_tables[(long long)b * p.bt_stride + e]) : -1;
  };
  if (w0 < w1) load_window((w0 * UT) >> bs_log2);

  // Everything below reads what the previous kernel may write.
  pdl_wait_previous();

  // The 16 query rows, once a CTA: whole rows a load instruction (each warp loading its
  // fragments itself took 2.6 us of a verify call's 14.6 a CTA).
  constexpr int kThreads = kWarps * 32, kWords = 16 * (D / 2), kLoads = (kWords + kThreads - 1) / kThreads;
  uint32_t qw[kLoads];
#pragma unroll
  for (int n = 0; n < kLoads; ++n) {
    const int i = tid + n * kThreads, r = i / (D / 2), w = i % (D / 2);
    qw[n] = r < rows_here && 2 * w < p.Dv ? __ldg(reinterpret_cast<const unsigned int*>(s_qrow[r]) + w) : 0u;
  }

  // Lane roles as in pa_decode_kernel.cuh.
  auto issue = [&](int u, int slot) {
    const uint32_t stage = ring + (uint32_t)slot * STAGE_BYTES;
    const uint32_t bar = my_bars + (uint32_t)slot * 8u;
    const int tok0 = u * UT;
    const int lb0 = tok0 >> bs_log2;
    if (lb0 + max(1, UT >> bs_log2) > win_base + 32) load_window(lb0);
    const int g = k8 ? 8 * (lane & 3) : (lane / (2 * HALVES)) * bs;
    const int kv = k8 ? (lane >> 2) & 1 : (lane / HALVES) & 1;
    const int hf = k8 ? 0 : lane % HALVES;
    const int lb = (tok0 + g) >> bs_log2;
    const int y = (tok0 + g) & (bs - 1);
    const int phys = __shfl_sync(0xffffffffu, win_val, (lb - win_base) & 31);
    const bool mine = k8 ? lane < 8 : lane < 2 * HALVES * (bs < UT ? UT >> bs_log2 : 1);
    const bool want = mine && (lb << bs_log2) < L && ((lb + 1) << bs_log2) > lo;
    const bool ok = phys >= 0 && phys < p.num_blocks;
    const bool box = want && (!k8 || (lane & 3) == 0 || y == 0);
    const uint32_t boxes = __ballot_sync(0xffffffffu, box);
    if (want && !ok) raise_flag(p.status, PA_DEVERR_BLOCK_ID_RANGE);
    if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)__popc(boxes) * (uint32_t)min(bs, UT) * TL::kRowBytes);
    __syncwarp();
    if (box)  // a bad id is out of the map's range: TMA fills zeros
      tma_load_4d_policy(stage + (uint32_t)kv * TILE_BYTES + (uint32_t)hf * TL::kHalfBytes +
                             (uint32_t)g * TL::kRowBytes,
                         kv ? &tmv : &tmk, bar, hf * 64, y, h, phys, kv_policy);
    if constexpr (k8) {
      if (lane < 8) {
        const bool use = want && ok;
        const long long blk = use ? phys : 0;
        const float* from = kv ? p.v_scales + blk * p.vs_sblk + h * p.vs_sh : p.k_scales + blk * p.ks_sblk + h * p.ks_sh;
        cp_async_4_zfill(smem_addr(&s_scales[2 * (warp * stages + slot)]) + 4u * lane, from, use ? 4u : 0u);
        cp_async_mbar_arrive_noinc(bar);
      }
    }
    __syncwarp();
  };
  int next = w0;
  for (int s = 0; s < stages && next < w1; ++s, ++next) issue(next, s);

  // ---- the warp's query rows and its units ----
  const int qr0 = 16 * mg + (lane >> 2);
#pragma unroll
  for (int n = 0; n < kLoads; ++n) {
    const int i = tid + n * kThreads;
    if (kWords % kThreads == 0 || i < kWords) s_wt[i / (D / 2)][i % (D / 2)] = __uint_as_float(qw[n]);
  }
  __syncthreads();
  uint32_t qa[D / 16][4];
  float o_acc[D / 8][4];
  RowState st;
  int tok_lo, tok_hi, full_lo, full_hi;
  if constexpr (k8) {
    float qinv[2];
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint2 v = *reinterpret_cast<const uint2*>(&s_wt[(lane >> 2) + 8 * r][ks * 8 + 2 * quad]);
        qa[ks][r] = v.x;
        qa[ks][r + 2] = v.y;
      }
    scale_query_frags_8<T, D>(qa, qinv);
    st.c[0] = p.scale_log2 * qinv[0];
    st.c[1] = p.scale_log2 * qinv[1];
  } else {
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        qa[ks][i] = __float_as_uint(s_wt[(lane >> 2) + 8 * (i & 1)][ks * 8 + quad + 4 * (i >> 1)]);
    st.c[0] = st.c[1] = p.scale_log2;
  }
  init_rows<kScored>(st, p, b, h, L, qr0, tok_lo, tok_hi, full_lo, full_hi);
#pragma unroll
  for (int nd = 0; nd < D / 8; ++nd) o_acc[nd][0] = o_acc[nd][1] = o_acc[nd][2] = o_acc[nd][3] = 0.f;
  int slot = 0;
  uint32_t phase = 0;
  for (int u = w0; u < w1; ++u) {
    if (!mbar_test_then_wait(my_bars + (uint32_t)slot * 8u, (phase >> slot) & 1u)) {
      if (lane == 0) raise_flag(p.status, PA_DEVERR_WAIT_TIMEOUT);
      // wait (bounded) for this warp's copies still in flight, then go on to the merge
      for (int k = u; k < next; ++k) {
        mbar_wait_bounded(my_bars + (uint32_t)slot * 8u, (phase >> slot) & 1u);
        slot = slot + 1 == stages ? 0 : slot + 1;
      }
      break;
    }
    phase ^= 1u << slot;
    const uint32_t kbase = ring + (uint32_t)slot * STAGE_BYTES;
    if constexpr (k8)
      attend_unit_8<T, D, kScored, true>(kbase, kbase + TILE_BYTES, qa, o_acc, st, u * UT, tok_lo, tok_hi, full_lo, full_hi,
                                   s_scales[2 * (warp * stages + slot)], s_scales[2 * (warp * stages + slot) + 1], p,
                                   lane);
    else
      attend_unit_scored<T, D, true>(kbase, kbase + TILE_BYTES, qa, o_acc, st, u * UT, tok_lo, tok_hi, full_lo, full_hi, p,
                               lane);
    __syncwarp();
    if (next < w1) {
      fence_proxy_async_smem();
      issue(next, slot);
      ++next;
    }
    slot = slot + 1 == stages ? 0 : slot + 1;
  }

  // ---- the CTA's state: (m, l, acc) of its warps, acc in each warp's own ring ----
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float l = st.l[r] + __shfl_xor_sync(0xffffffffu, st.l[r], 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (quad == 0) {
      s_m[warp][(lane >> 2) + 8 * r] = st.m[r];
      s_l[warp][(lane >> 2) + 8 * r] = l;
    }
  }
  float* acc = reinterpret_cast<float*>(smem + (size_t)(warp * stages) * STAGE_BYTES);
#pragma unroll
  for (int nd = 0; nd < D / 8; ++nd) {
    const int d = nd * 8 + 2 * quad;
    *reinterpret_cast<float2*>(acc + (lane >> 2) * AS + d) = make_float2(o_acc[nd][0], o_acc[nd][1]);
    *reinterpret_cast<float2*>(acc + ((lane >> 2) + 8) * AS + d) = make_float2(o_acc[nd][2], o_acc[nd][3]);
  }
  __syncthreads();
  auto sees = [&](int r) -> bool {
    const KeyRange kr = row_keys<kScored>(p, b, L, (16 * mg + r) / p.G);
    return kr.first < kr.end;
  };
  if (tid < 16) {
    float M = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w][tid]);
    const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(s_m[w][tid] - base);
      s_wt[tid][w] = f;
      l = fmaf(f, s_l[w][tid], l);
    }
    s_ref[tid] = M;
    s_norm[tid] = S > 1 ? l : tid < rows_here ? row_norm<KV>(l, sees(tid)) : 0.f;
  }
  __syncthreads();
  auto out_pair = [&](int r, int d, float2 a, float inv) {
    if (d < p.Dv) *reinterpret_cast<uint32_t*>(s_orow[r] + d) = pack2<T>(a.x * inv, a.y * inv);
  };
  const int slot_floats = p.slot_rows * (2 + D);
  float* part = p.partials + ((long long)row * gridDim.y + split) * slot_floats;
#pragma unroll 2
  for (int i = tid; i < rows_here * (D / 4); i += kThreads) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = s_wt[r][w];
      const float4 v = *reinterpret_cast<const float4*>(smem + (size_t)(w * stages) * STAGE_BYTES + (r * AS + d) * 4);
      a.x = fmaf(f, v.x, a.x);
      a.y = fmaf(f, v.y, a.y);
      a.z = fmaf(f, v.z, a.z);
      a.w = fmaf(f, v.w, a.w);
    }
    if (S == 1) {
      out_pair(r, d, make_float2(a.x, a.y), s_norm[r]);
      out_pair(r, d + 2, make_float2(a.z, a.w), s_norm[r]);
    } else {
      float2* to = reinterpret_cast<float2*>(part + 2 * p.slot_rows + r * D + d);
      to[0] = make_float2(a.x, a.y);
      to[1] = make_float2(a.z, a.w);
    }
  }
  if (S == 1) return;
  if (tid < rows_here) {
    part[tid] = s_ref[tid];
    part[p.slot_rows + tid] = s_norm[tid];
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(&p.counters[row], 1) == S - 1;
  __syncthreads();
  if (!s_last) return;

  // ---- the row's last CTA: log-sum-exp merge of its S partial states ----
  __threadfence();
  const float* first_part = p.partials + (long long)row * gridDim.y * slot_floats;
  for (int r = warp; r < rows_here; r += kWarps) {
    float m[kMaxSplits / 32], M = -INFINITY, l = 0.f;
#pragma unroll
    for (int k = 0; k < kMaxSplits / 32; ++k) {
      const int s = lane + 32 * k;
      m[k] = s < S ? __ldcg(first_part + (long long)s * slot_floats + r) : -INFINITY;
      M = fmaxf(M, m[k]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int k = 0; k < kMaxSplits / 32; ++k) {
      const int s = lane + 32 * k;
      if (s >= S) continue;
      const float f = ex2(m[k] - base);
      s_wt[r][s] = f;
      l = fmaf(f, __ldcg(first_part + (long long)s * slot_floats + p.slot_rows + r), l);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) s_norm[r] = row_norm<KV>(l, sees(r));
  }
  __syncthreads();
  for (int i = tid; i < rows_here * (D / 2); i += kWarps * 32) {
    const int r = i / (D / 2), d = 2 * (i - r * (D / 2));
    const float* from = first_part + 2 * p.slot_rows + r * D + d;
    float2 a = make_float2(0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < S; ++s) {
      const float f = s_wt[r][s];
      const float2 v = __ldcg(reinterpret_cast<const float2*>(from + (long long)s * slot_floats));
      a.x = fmaf(f, v.x, a.x);
      a.y = fmaf(f, v.y, a.y);
    }
    out_pair(r, d, a, s_norm[r]);
  }
  if (tid == 0) atomicExch(&p.counters[row], 0);
}

DirectShape decode_direct_shape(bool eight, bool many) {
  DirectShape d;
  d.warps = eight ? (many ? Shape<e4m3_t, true>::kWarps : Shape<e4m3_t, false>::kWarps)
                  : (many ? Shape<__half, true>::kWarps : Shape<__half, false>::kWarps);
  d.ctas_per_sm = eight ? (many ? Shape<e4m3_t, true>::kCtas : Shape<e4m3_t, false>::kCtas)
                        : (many ? Shape<__half, true>::kCtas : Shape<__half, false>::kCtas);
  return d;
}

size_t decode_direct_smem_bytes(int D, int stages, int warps, bool eight) {
  const size_t stage_bytes = 2u * 16u * (size_t)D * 2u;  // 16 tokens of 2 bytes, or 32 of 1
  return 1024 + (size_t)warps * stages * (stage_bytes + 8 + (eight ? 32 : 0));
}

namespace {

template <typename T, int D, typename KV, bool kScored, bool kMany>
cudaError_t launch(const DecodeParams& p, const CUtensorMap& tmk, const CUtensorMap& tmv, int splits, size_t smem,
                   bool pdl, cudaStream_t stream) {
  const auto kernel = decode_direct_kernel<T, D, KV, kScored, kMany>;
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
    e = cudaFuncGetAttributes(&fa, kernel);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most - (int)fa.sharedSizeBytes);
    if (e != cudaSuccess) return e;
    prepared[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.B * p.Hkv * p.NMG), (unsigned)splits);
  cfg.blockDim = dim3(Shape<KV, kMany>::kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl ? attr : nullptr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, tmk, tmv, p);
}

template <typename T, int D, bool kMany>
cudaError_t pick(const DecodeParams& p, const CUtensorMap& tmk, const CUtensorMap& tmv, int splits, size_t smem,
                 bool pdl, cudaStream_t stream) {
  if (p.k_scales == nullptr) return launch<T, D, T, true, kMany>(p, tmk, tmv, splits, smem, pdl, stream);
  if (p.scored) return launch<T, D, e4m3_t, true, kMany>(p, tmk, tmv, splits, smem, pdl, stream);
  return launch<T, D, e4m3_t, false, kMany>(p, tmk, tmv, splits, smem, pdl, stream);
}

template <typename T>
cudaError_t pick_width(const DecodeParams& p, const CUtensorMap& tmk, const CUtensorMap& tmv, int splits, bool many,
                       size_t smem, bool pdl, cudaStream_t stream) {
  if (p.D == 128)
    return many ? pick<T, 128, true>(p, tmk, tmv, splits, smem, pdl, stream)
                : pick<T, 128, false>(p, tmk, tmv, splits, smem, pdl, stream);
  return many ? pick<T, 64, true>(p, tmk, tmv, splits, smem, pdl, stream)
              : pick<T, 64, false>(p, tmk, tmv, splits, smem, pdl, stream);
}

}  // namespace

cudaError_t launch_decode_direct(const DecodeParams& p, const CUtensorMap& tmk, const CUtensorMap& tmv, int dtype,
                                 int splits, bool many, size_t smem, bool pdl, cudaStream_t stream) {
  if (splits < 1 || splits > kMaxSplits) return cudaErrorInvalidValue;
  return dtype == PA_DTYPE_BFLOAT16 ? pick_width<__nv_bfloat16>(p, tmk, tmv, splits, many, smem, pdl, stream)
                                    : pick_width<__half>(p, tmk, tmv, splits, many, smem, pdl, stream);
}

}  // namespace pa
