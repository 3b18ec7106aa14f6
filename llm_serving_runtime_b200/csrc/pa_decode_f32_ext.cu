// pa_decode_f32_ext.cu — pa_decode_ext over fp32 caches: changed scores on CUDA cores
// (TF32 tensor cores would not keep fp32's digits).
//
//   s = scale * (q . k_j);  s = c * tanh(s / c);  s -= slope * |i - j|
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)  over the keys the row sees
//
// A CTA takes up to 8 query rows of one (sequence, KV head) and the s-th of S equal
// ranges of the 16-token tiles they see (from the first visible key's on; what
// lies before is not read).  Its warps take an equal part of it each, two tiles in
// flight (cp.async), merge their states in shared memory, and the row group's last
// CTA merges the S partial states in order.  In a warp, lane (half, t) scores token t
// over half of the columns for all rows; each half then keeps the softmax state of
// half of the rows, and for P V lanes span the columns.  K rows are 4 floats longer than
// the head in shared memory, so 16-byte reads of eight tokens hit all banks.
//
// Latency bounds it at the sizes fp32 is served at, shared-memory reads (five
// 16-byte ones for 16 multiply-adds a lane with four rows) beyond.  Measured against the
// plain fp32 kernel's form, one CTA a (sequence, head) that stages a block at a
// time: four rows of 1 to 512 tokens, 8/2 heads of 64, 10.5 us for 17.8; one of 1500
// tokens, 8 heads, 12.4 for 58.7; 128 of 46 to 1500, 32/8 heads of 128, 275 for 378 (1.6 TB/s).
#include <limits.h>
#include <math.h>

#include "pa_common.cuh"
#include "pa_internal.h"

namespace pa {

namespace {

constexpr int kTile = 16;  // tokens
constexpr int kSplitsMost = kDirectMaxSplits;

// Warps of a CTA: what two tiles in flight for each leave room for.
constexpr int f32_warps(int D) { return D == 128 ? 4 : 8; }
constexpr int f32_pitch(int D) { return D + 4; }
// Floats of a warp's two tiles of K and V.
constexpr int f32_warp_floats(int D) { return 2 * kTile * (f32_pitch(D) + D); }

__device__ __forceinline__ KeyRange keys_of(const DecodeParams& p, int b, int L, int t) {
  const int start = p.key_starts != nullptr ? __ldg(&p.key_starts[b * p.kst_sb + t * p.kst_st]) : 0;
  const int prefix = p.prefix_lens != nullptr ? __ldg(&p.prefix_lens[b]) : 0;
  return key_range(L, p.q_len, t, p.window, start, prefix);
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait_group() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace

// DPL: head width / 32; R: rows of a CTA; kVec: floats of a copy (4: rows 16-byte
// aligned and a head_dim that is a multiple of 4).
template <int DPL, int R, int kVec>
__global__ void __launch_bounds__(f32_warps(DPL * 32) * 32) decode_f32_ext_kernel(const DecodeParams p) {
  constexpr int D = DPL * 32, W = f32_warps(D), PITCH = f32_pitch(D), H2 = R / 2;
  extern __shared__ float f32e_smem[];
  float* s_q = f32e_smem;  // [R][D]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float* s_k = s_q + R * D + warp * f32_warp_floats(D);  // [2][kTile][PITCH]
  float* s_v = s_k + 2 * kTile * PITCH;                  // [2][kTile][D]
  __shared__ float s_p[W][R][kTile];                     // weights; -1: hidden
  __shared__ float s_m[W][R], s_l[W][R], s_wt[R][kSplitsMost], s_ref[R], s_norm[R];
  __shared__ int s_lo, s_hi, s_last;

  const int groups = (p.GQ + R - 1) / R;
  const int row = blockIdx.x, split = blockIdx.y;
  const int grp = row % groups, h = (row / groups) % p.Hkv, b = row / (groups * p.Hkv);
  const int r0 = grp * R, rows = min(R, p.GQ - r0);

  if (tid == 0) {
    s_lo = INT_MAX;
    s_hi = 0;
  }
  // columns past the head's stay zero in every tile
  if (p.Dv < D)
    for (int i = lane; i < f32_warp_floats(D); i += 32) s_k[i] = 0.f;
  __syncthreads();
  pdl_wait_previous();
  int L = p.context_lens[b] + p.len_offset;
  const int cap = p.max_blocks * p.bs;
  if (L > cap) {
    if (tid == 0 && h == 0 && grp == 0 && split == 0) raise_flag(p.status, PA_DEVERR_TABLE_UNDERRUN);
    L = cap;
  }
  if (L < 0) L = 0;
  // Query row r0 + r: head g, token t (head-major, as the plain fp32 kernel orders them).
  if (tid < rows) {
    const KeyRange kr = keys_of(p, b, L, (r0 + tid) % p.q_len);
    if (kr.first < kr.end) {
      atomicMin(&s_lo, kr.first);
      atomicMax(&s_hi, kr.end);
    }
  }
  for (int i = tid; i < R * D; i += W * 32) {
    const int r = i / D, d = i - r * D, qr = r0 + r;
    float v = 0.f;
    if (r < rows && d < p.Dv)
      v = static_cast<const float*>(p.q)[(long long)b * p.q_sb + (long long)(h * p.G + qr / p.q_len) * p.q_sh +
                                         (long long)(qr % p.q_len) * p.q_st + d];
    s_q[i] = v;
  }
  __syncthreads();
  const int lo = s_lo, hi = s_hi;
  const int u_first = lo < hi ? lo / kTile : 0;
  const int n = lo < hi ? (hi + kTile - 1) / kTile - u_first : 0;
  const int S = max(1, min((int)gridDim.y, (n + W - 1) / W));
  if (split >= S) return;
  const int c0 = (int)((long long)n * split / S), c1 = (int)((long long)n * (split + 1) / S);
  const int w0 = u_first + c0 + (c1 - c0) * warp / W, w1 = u_first + c0 + (c1 - c0) * (warp + 1) / W;

  const float* kc = static_cast<const float*>(p.k_cache);
  const float* vc = static_cast<const float*>(p.v_cache);
  auto issue = [&](int u, int buf) {
    // lane t < 16: block and offset of token t
    const int tok = u * kTile + (lane & 15);
    long long ko = -1, vo = 0;
    bool zero = false;  // of a block outside the pool: zeros, as TMA fills them for the other types
    if (tok >= lo && tok < hi) {
      const int lb = tok / p.bs, off = tok - lb * p.bs;
      const int phys = __ldg(&p.block_tables[(long long)b * p.bt_stride + lb]);
      if (phys < 0 || phys >= p.num_blocks) {
        raise_flag(p.status, PA_DEVERR_BLOCK_ID_RANGE);
        zero = true;
      } else {
        ko = phys * p.k_sblk + h * p.k_sh + off * p.k_st;
        vo = phys * p.v_sblk + h * p.v_sh + off * p.v_st;
      }
    }
    for (uint32_t left = __ballot_sync(0xffffffffu, zero) & 0xffffu; left != 0u; left &= left - 1) {
      const int t = __ffs(left) - 1;
      for (int c = lane; c < D; c += 32) {
        s_k[buf * kTile * PITCH + t * PITCH + c] = 0.f;
        s_v[buf * kTile * D + t * D + c] = 0.f;
      }
    }
    constexpr int PER = D / kVec;  // copies of a row
    const uint32_t kd = smem_addr(s_k + buf * kTile * PITCH), vd = smem_addr(s_v + buf * kTile * D);
#pragma unroll 4
    for (int i = lane; i < kTile * PER; i += 32) {
      const int t = i / PER, c = (i - t * PER) * kVec;
      const long long ka = __shfl_sync(0xffffffffu, ko, t), va = __shfl_sync(0xffffffffu, vo, t);
      if (ka < 0 || c >= p.Dv) continue;
      if constexpr (kVec == 4) {
        cp_async_16(kd + 4u * (t * PITCH + c), kc + ka + c);
        cp_async_16(vd + 4u * (t * D + c), vc + va + c);
      } else {
        cp_async_4(kd + 4u * (t * PITCH + c), kc + ka + c);
        cp_async_4(vd + 4u * (t * D + c), vc + va + c);
      }
    }
    cp_async_commit();
  };
  if (w0 < w1) issue(w0, 0);

  // this lane's rows in the softmax: half * H2 ..
  const int half = lane >> 4, t = lane & 15;
  float m[H2], l[H2], slope[H2], acc[R][DPL];
  int first[H2], end[H2], pos[H2];
#pragma unroll
  for (int i = 0; i < H2; ++i) {
    const int r = half * H2 + i, qr = r0 + r;
    m[i] = -INFINITY;
    l[i] = 0.f;
    slope[i] = 0.f;
    first[i] = 0;
    end[i] = INT_MAX;  // rows past the group's last see everything and are not stored
    pos[i] = 0;
    if (r < rows) {
      const KeyRange kr = keys_of(p, b, L, qr % p.q_len);
      first[i] = kr.first;
      end[i] = kr.end;
      pos[i] = L - p.q_len + qr % p.q_len;
      if (p.alibi_slopes != nullptr) slope[i] = __ldg(&p.alibi_slopes[h * p.G + qr / p.q_len]);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < DPL; ++j) acc[r][j] = 0.f;

  for (int u = w0; u < w1; ++u) {
    const int buf = (u - w0) & 1;
    if (u + 1 < w1) {
      issue(u + 1, buf ^ 1);
      cp_async_wait_group<1>();
    } else {
      cp_async_wait_group<0>();
    }
    __syncwarp();
    const float* kr = s_k + buf * kTile * PITCH + t * PITCH + half * (D / 2);
    const float* qh = s_q + half * (D / 2);
    float sc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) sc[r] = 0.f;
#pragma unroll 4
    for (int d = 0; d < D / 2; d += 4) {
      const float4 kv = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float4 qv = *reinterpret_cast<const float4*>(qh + r * D + d);
        sc[r] = fmaf(qv.x, kv.x, fmaf(qv.y, kv.y, fmaf(qv.z, kv.z, fmaf(qv.w, kv.w, sc[r]))));
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) sc[r] += __shfl_xor_sync(0xffffffffu, sc[r], 16);
    const int tok = u * kTile + t;
    bool any_hidden = false;
    float alpha[H2];
#pragma unroll
    for (int i = 0; i < H2; ++i) {
      float s = (half ? sc[H2 + i] : sc[i]) * p.scale;
      if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
      if (p.alibi_slopes != nullptr) s -= slope[i] * fabsf((float)(pos[i] - tok));
      const bool hidden = tok < first[i] || tok >= end[i];
      any_hidden |= hidden;
      float mx = hidden ? -INFINITY : s;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float mn = fmaxf(m[i], mx), base = mn == -INFINITY ? 0.f : mn;
      alpha[i] = m[i] == -INFINITY ? 0.f : expf(m[i] - base);
      const float w = hidden ? 0.f : expf(s - base);
      float ws = w;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
      l[i] = l[i] * alpha[i] + ws;
      m[i] = mn;
      s_p[warp][half * H2 + i][t] = hidden ? -1.f : w;
    }
    any_hidden = __any_sync(0xffffffffu, any_hidden || tok < lo || tok >= hi);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float a = __shfl_sync(0xffffffffu, alpha[r % H2], (r / H2) * 16);
#pragma unroll
      for (int j = 0; j < DPL; ++j) acc[r][j] *= a;
    }
    __syncwarp();
    const float* vr = s_v + buf * kTile * D + lane;
    if (!any_hidden) {
#pragma unroll
      for (int t4 = 0; t4 < kTile; t4 += 4) {
        float v[4][DPL];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int j = 0; j < DPL; ++j) v[k][j] = vr[(t4 + k) * D + 32 * j];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float4 w = *reinterpret_cast<const float4*>(&s_p[warp][r][t4]);
#pragma unroll
          for (int j = 0; j < DPL; ++j)
            acc[r][j] = fmaf(w.w, v[3][j], fmaf(w.z, v[2][j], fmaf(w.y, v[1][j], fmaf(w.x, v[0][j], acc[r][j]))));
        }
      }
    } else {
      // a key a row does not see must not reach it, whatever V holds there (0 * inf)
      for (int k = 0; k < kTile; ++k) {
        const int at = u * kTile + k;
        if (at < lo || at >= hi) continue;  // not even copied
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float w = s_p[warp][r][k];
          if (w < 0.f) continue;
#pragma unroll
          for (int j = 0; j < DPL; ++j) acc[r][j] = fmaf(w, vr[k * D + 32 * j], acc[r][j]);
        }
      }
    }
    __syncwarp();
  }

  // ---- the CTA's state ----
  if (t == 0) {
#pragma unroll
    for (int i = 0; i < H2; ++i) {
      s_m[warp][half * H2 + i] = m[i];
      s_l[warp][half * H2 + i] = l[i];
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < DPL; ++j) s_k[r * D + lane + 32 * j] = acc[r][j];
  __syncthreads();
  // 1 / l; zero for a row that sees no key, NaN where all its scores are -inf
  auto norm = [&](int r, float sum) -> float {
    if (sum > 0.f) return 1.f / sum;
    const KeyRange kr = keys_of(p, b, L, (r0 + r) % p.q_len);
    return sum == 0.f && kr.first >= kr.end ? 0.f : __int_as_float(0x7fffffff);
  };
  if (tid < rows) {
    float M = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, s_m[w][tid]);
    const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = s_m[w][tid] == -INFINITY ? 0.f : expf(s_m[w][tid] - base);
      s_wt[tid][w] = f;
      sum = fmaf(f, s_l[w][tid], sum);
    }
    s_ref[tid] = M;
    s_norm[tid] = S > 1 ? sum : norm(tid, sum);
  }
  __syncthreads();
  auto out_at = [&](int r, int d) -> float* {
    const int qr = r0 + r;
    return static_cast<float*>(p.out) + (long long)b * p.o_sb + (long long)(h * p.G + qr / p.q_len) * p.o_sh +
           (long long)(qr % p.q_len) * p.o_st + d;
  };
  constexpr int kSlot = R * (2 + D);
  float* part = p.partials + ((long long)row * gridDim.y + split) * kSlot;
  const float* all = s_q + R * D;
  for (int i = tid; i < rows * D; i += W * 32) {
    const int r = i / D, d = i - r * D;
    float a = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) a = fmaf(s_wt[r][w], all[w * f32_warp_floats(D) + i], a);
    if (S > 1)
      part[2 * R + i] = a;
    else if (d < p.Dv)
      *out_at(r, d) = a * s_norm[r];
  }
  if (S == 1) return;
  if (tid < rows) {
    part[tid] = s_ref[tid];
    part[R + tid] = s_norm[tid];
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(&p.counters[row], 1) == S - 1;
  __syncthreads();
  if (!s_last) return;

  // ---- the group's last CTA: merge of its S partial states ----
  __threadfence();
  const float* parts = p.partials + (long long)row * gridDim.y * kSlot;
  if (tid < rows) {
    float M = -INFINITY, sum = 0.f;
    for (int s = 0; s < S; ++s) M = fmaxf(M, __ldcg(parts + s * kSlot + tid));
    const float base = M == -INFINITY ? 0.f : M;
    for (int s = 0; s < S; ++s) {
      const float ms = __ldcg(parts + s * kSlot + tid);
      const float f = ms == -INFINITY ? 0.f : expf(ms - base);
      s_wt[tid][s] = f;
      sum = fmaf(f, __ldcg(parts + s * kSlot + R + tid), sum);
    }
    s_norm[tid] = norm(tid, sum);
  }
  __syncthreads();
  for (int i = tid; i < rows * D; i += W * 32) {
    const int r = i / D, d = i - r * D;
    float a = 0.f;
#pragma unroll 8
    for (int s = 0; s < S; ++s) a = fmaf(s_wt[r][s], __ldcg(parts + s * kSlot + 2 * R + i), a);
    if (d < p.Dv) *out_at(r, d) = a * s_norm[r];
  }
  if (tid == 0) atomicExch(&p.counters[row], 0);
}

namespace {

// Row groups times splits of a launch: two CTAs an SM, as far as splits go.  Both fit
// into the shared memory at a head width of 32; from 64 on an SM holds one (132 to 134
// KB), and a launch that uses all its splits runs in two rounds.  With one an SM
// single rows are faster (us, 8 heads: 4000 tokens, 128 wide, 29 for 40; 8000, 64 wide,
// 20 for 26; 32,000, 128 wide, 117 for 131), several are not (4 of 8000, 128 wide, 128 for
// 120; 2 of 20,000 with 4 tokens, 64 wide, 156 for 149).
constexpr int kCtasPerSm = 2;

int f32_rows(const DecodeParams& p) { return p.GQ <= 4 ? 4 : 8; }

template <int DPL, int R, int kVec>
cudaError_t launch(const DecodeParams& p, int splits, bool pdl, cudaStream_t stream) {
  constexpr int D = DPL * 32, W = f32_warps(D);
  const auto kernel = decode_f32_ext_kernel<DPL, R, kVec>;
  const size_t smem = sizeof(float) * ((size_t)R * D + (size_t)W * f32_warp_floats(D));
  static bool prepared[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!prepared[dev]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    prepared[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)p.B * p.Hkv * ((p.GQ + R - 1) / R)), (unsigned)splits);
  cfg.blockDim = dim3(W * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl ? attr : nullptr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int DPL>
cudaError_t pick(const DecodeParams& p, bool vec, int splits, bool pdl, cudaStream_t stream) {
  if (f32_rows(p) == 4)
    return vec ? launch<DPL, 4, 4>(p, splits, pdl, stream) : launch<DPL, 4, 1>(p, splits, pdl, stream);
  return vec ? launch<DPL, 8, 4>(p, splits, pdl, stream) : launch<DPL, 8, 1>(p, splits, pdl, stream);
}

}  // namespace

size_t f32_ext_partial_bytes(int num_sms) { return (size_t)kCtasPerSm * num_sms * 8 * (2 + 128) * sizeof(float); }

cudaError_t launch_decode_f32_ext(const DecodeParams& p, int num_sms, bool pdl, cudaStream_t stream) {
  const int R = f32_rows(p);
  const long long groups = (long long)p.B * p.Hkv * ((p.GQ + R - 1) / R);
  if (groups > INT_MAX) return cudaErrorInvalidValue;
  long long splits = (long long)kCtasPerSm * num_sms / groups;
  splits = splits < 1 ? 1 : splits > kSplitsMost ? kSplitsMost : splits;
  auto aligned = [](const void* ptr, int64_t a, int64_t b, int64_t c) {
    return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && ((a | b | c) & 3) == 0;
  };
  const bool vec = p.Dv % 4 == 0 && aligned(p.k_cache, p.k_sblk, p.k_sh, p.k_st) &&
                   aligned(p.v_cache, p.v_sblk, p.v_sh, p.v_st);
  switch (p.D) {
    case 32:
      return pick<1>(p, vec, (int)splits, pdl, stream);
    case 64:
      return pick<2>(p, vec, (int)splits, pdl, stream);
    case 128:
      return pick<4>(p, vec, (int)splits, pdl, stream);
    default:
      return cudaErrorInvalidValue;
  }
}

}  // namespace pa
