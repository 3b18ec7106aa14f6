// pa_tile_ext.cuh — one warp's attention over one 16-token unit for the two
// extensions of the plain tile (pa_tile_math.cuh): caches held in 8 bits (e4m3
// with one scale per block of tokens and KV head) and changed scores (tanh cap,
// distance bias, sliding window, document starts, prefix mask).
//
// With x = log2(e) * s the score of a query at position i and a key at j, and
// first <= j < end the keys the row sees:
//   s = scale * (q . k_j),  capped c * tanh(s / c),  minus slope * |i - j|
//   out = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m)
//
// 8-bit caches (attend_unit_8, 32 tokens at a time).  k_j = ks * c_j and v_j =
// vs * d_j with codes c, d and the block's scales ks, vs.  Codes widen to fp16
// without rounding, so both products run as fp16 MMAs whatever the query's type
// (mma.sync has no 8-bit float unit here: an e4m3 MMA expands to two fp16 ones and
// ten conversions, measured 0.17 a clock against 0.40 for fp16); ks multiplies the
// finished dot product.  A bf16 query row is brought to fp16 by a power of two of
// its own that puts its largest element into [2^14, 2^15): 8-bit significands fit
// fp16's 11, and only elements 2^29 below the row's largest lose bits.  V comes
// out of a byte transpose (ldmatrix b8).  vs goes into the weights, and the running
// reference is that of the weighted values:
//   m = max_j (x_j + log2 vs_j) - 14,  w_j = 2^(x_j + log2 vs_j - m)
//   out = sum_j w_j d_j / (2^14 sum_j 2^-14 w_j / vs_j)
// so a block of large scale and little weight cannot push the others' weights
// out of fp16's range, and one exponential serves both sums.  w is rounded to
// fp16 for the product (at most 2^-11 of each weight; normal down to 2^-28 of the
// largest, nothing below 2^-39 of it), the norm takes it unrounded.  The norm's fp32 range
// holds as long as the V scales of a row's blocks lie within 2^100 of one another.  Scales
// up to 2^-100, the least that the append writes (a block of zeros), would not beside
// values above 3e10: such blocks' values count as 0 (they are below 4e-28), and their
// weights go into the norm by way of a scale of 2^-40.
//
// What a mask hides never reaches a row: hidden scores are -inf whatever K
// holds, and in units where rows see different keys (or none), V rows that are not
// finite (0 * inf) are added row by row and then, like rows nobody sees, zeroed in
// shared memory before the MMA (or masked out of it where other warps read the tile).
#pragma once

#include <limits.h>

#include "pa_common.cuh"
#include "pa_internal.h"
#include "pa_tile_math.cuh"

namespace pa {

// Cache element of 8-bit caches (an e4m3 code).
struct e4m3_t {
  uint8_t bits;
};

template <bool b>
struct Bool {
  static constexpr bool value = b;
};

template <typename C>
struct kIs8 {
  static constexpr bool value = sizeof(C) == 1;
};

// Two e4m3 codes (bits 0-15, or 16-31) to two fp16 values, exactly.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t codes) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(d) : "r"(codes));
  return d;
}
__device__ __forceinline__ uint32_t e4m3x2_hi_to_f16x2(uint32_t codes) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(d) : "r"(codes));
  return d;
}

// log2 (approximate instruction).
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Tokens of an 8-bit unit: two k-steps of the P.V product, so that a unit's fixed
// work (barrier, copies, maxima) is spread over the same bytes as a 16-bit one's.
constexpr int kUnit8Tokens = 32;

// 1 / x (approximate instruction; 1 / inf = 0).
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Element layout of a unit's tile in shared memory.  16-bit: 64-element column
// halves of 16 rows x 128 bytes, 128-byte swizzle.  8-bit: 32 rows of D bytes,
// swizzled over 128 bytes (D = 128) or 64 bytes (D = 64).
template <typename C, int D>
struct TileLayout {
  static constexpr bool k8 = kIs8<C>::value;
  static constexpr int kHalves = k8 ? 1 : D / 64;           // TMA boxes across a row
  static constexpr uint32_t kRowBytes = k8 ? D : 128;       // bytes of a box row
  static constexpr int kTokens = k8 ? kUnit8Tokens : kUnitTokens;
  static constexpr uint32_t kHalfBytes = kTokens * kRowBytes;
  static constexpr uint32_t kTileBytes = kHalves * kHalfBytes;
};

// Byte address of 16-byte chunk `chunk` of row `tok` in a tile at `base`.
template <typename C, int D>
__device__ __forceinline__ uint32_t tile_chunk_addr(uint32_t base, int tok, int chunk) {
  using L = TileLayout<C, D>;
  if constexpr (L::kRowBytes == 128)
    return base + (uint32_t)(chunk >> 3) * L::kHalfBytes + (uint32_t)tok * 128u +
           ((uint32_t)((chunk & 7) ^ (tok & 7)) << 4);
  else
    return base + (uint32_t)tok * 64u + ((uint32_t)(chunk ^ ((tok >> 1) & 3)) << 4);
}

// tile_chunk_addr() of a lane's chunk c ^ i for even i (c: the lane's own, 0 or 1 more
// than an even one) is this with i << 4 exchanged: tiles are aligned to
// the swizzle, so the chunk is a field of the address.
__device__ __forceinline__ uint32_t flip_chunk(uint32_t addr, int i) { return addr ^ ((uint32_t)i << 4); }

// Running state of a warp's rows lane/4 (index 0) and lane/4 + 8 (index 1).
struct RowState {
  float m[2], l[2];    // the softmax's reference and norm
  float c[2];          // dot product -> x (scale * log2 e, and the query row's power of two)
  int first[2], end[2];  // keys the row sees
  float slope[2];      // distance bias, log2 domain
  int pos[2];          // the row's own position
};

// Keys that query token t of sequence b (attended length L) sees.
template <bool kScored>
__device__ __forceinline__ KeyRange row_keys(const DecodeParams& p, int b, int L, int t) {
  if constexpr (kScored) {
    const int start = p.key_starts != nullptr ? __ldg(&p.key_starts[b * p.kst_sb + t * p.kst_st]) : 0;
    const int prefix = p.prefix_lens != nullptr ? __ldg(&p.prefix_lens[b]) : 0;
    return key_range(L, p.q_len, t, p.window, start, prefix);
  }
  return key_range(L, p.q_len, t, 0, 0, 0);
}

// Fresh state of rows qr0 and qr0 + 8 of KV head h (st.c is the caller's), and of
// the tile's 16 rows: keys that some row sees lie in [tok_lo, tok_hi), keys in
// [full_lo, full_hi) are seen by every row.
template <bool kScored>
__device__ __forceinline__ void init_rows(RowState& st, const DecodeParams& p, int b, int h, int L, int qr0,
                                          int& tok_lo, int& tok_hi, int& full_lo, int& full_hi) {
  tok_lo = full_hi = INT_MAX;
  tok_hi = full_lo = 0;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int qr = qr0 + 8 * r;
    st.m[r] = -INFINITY;
    st.l[r] = 0.f;
    st.first[r] = 0;  // rows past the group's last see everything and are not stored
    st.end[r] = INT_MAX;
    st.slope[r] = 0.f;
    st.pos[r] = 0;
    if (qr < p.GQ) {
      const int t = qr / p.G, g = qr - t * p.G;
      const KeyRange kr = row_keys<kScored>(p, b, L, t);
      if (kScored && p.alibi_slopes != nullptr)
        st.slope[r] = __ldg(&p.alibi_slopes[h * p.G + g]) * 1.4426950408889634f;
      st.first[r] = kr.first;
      st.end[r] = kr.end;
      st.pos[r] = L - p.q_len + t;
      tok_lo = min(tok_lo, kr.first);
      tok_hi = max(tok_hi, kr.end);
      full_lo = max(full_lo, kr.first);
      full_hi = min(full_hi, kr.end);
    }
  }
  tok_lo = __reduce_min_sync(0xffffffffu, tok_lo);
  tok_hi = __reduce_max_sync(0xffffffffu, tok_hi);
  full_lo = __reduce_max_sync(0xffffffffu, full_lo);
  full_hi = __reduce_min_sync(0xffffffffu, full_hi);
}

// Query fragments of an 8-bit tile: k-step ks holds columns 16 ks + 4 quad, +1
// (registers 0, 1) and +2, +3 (registers 2, 3), the order in which ldmatrix
// hands out four neighbouring codes.  Here they become fp16: each row times a power
// of two of its own, which qinv takes back out of its dot products.
template <typename T, int D>
__device__ __forceinline__ void scale_query_frags_8(uint32_t (&qa)[D / 16][4], float (&qinv)[2]) {
  qinv[0] = qinv[1] = 1.f;
  if constexpr (sizeof(T) == 2 && !kSplitProbabilities<T>::value) return;  // fp16 already
  float mx[2] = {0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      mx[i & 1] = fmaxf(mx[i & 1], fmaxf(fabsf(lo_half<T>(qa[ks][i])), fabsf(hi_half<T>(qa[ks][i]))));
  float mul[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
    mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
    const int e = (int)(__float_as_uint(mx[r]) >> 23);  // biased exponent: mx in [2^(e-127), 2^(e-126))
    // 2^(14 + 127 - e), within what fp32 holds; rows of 0 or with an infinity stay as they are
    const int k = (e == 0 || e == 255) ? 0 : min(max(14 + 127 - e, -120), 100);
    mul[r] = __uint_as_float((uint32_t)(127 + k) << 23);
    qinv[r] = __uint_as_float((uint32_t)(127 - k) << 23);
  }
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      qa[ks][i] = pack2<__half>(lo_half<T>(qa[ks][i]) * mul[i & 1], hi_half<T>(qa[ks][i]) * mul[i & 1]);
}

// The same from the rows qp0 and qp1 (null: 0) in memory.
template <typename T, int D>
__device__ __forceinline__ void load_query_frags_8(uint32_t (&qa)[D / 16][4], const T* qp0, const T* qp1, int quad,
                                                   int Dv, float (&qinv)[2]) {
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
    const int d = ks * 16 + 4 * quad;
    const bool in = d < Dv;  // Dv is a multiple of 16
    qa[ks][0] = (qp0 && in) ? __ldg(reinterpret_cast<const unsigned int*>(qp0 + d)) : 0u;
    qa[ks][1] = (qp1 && in) ? __ldg(reinterpret_cast<const unsigned int*>(qp1 + d)) : 0u;
    qa[ks][2] = (qp0 && in) ? __ldg(reinterpret_cast<const unsigned int*>(qp0 + d + 2)) : 0u;
    qa[ks][3] = (qp1 && in) ? __ldg(reinterpret_cast<const unsigned int*>(qp1 + d + 2)) : 0u;
  }
  scale_query_frags_8<T, D>(qa, qinv);
}

// c * tanh(x / c) in the log2 domain (cap, inv_cap = 1 / cap, both of it), with
// tanh y = 1 - 2 / (1 + e^2y).  Near 0 that is off by 2^-22 of the cap (the
// exponential's and the division's error), so up to kDirectCap a score is off by
// less than 4e-5, far below the rounding of its weight.
constexpr float kDirectCap = 128.f;
__device__ __forceinline__ float softcap_direct(float x, float cap, float inv_cap) {
  return fmaf(-2.f * cap, rcp_approx(1.f + ex2(x * inv_cap * 2.8853900817779268f)), cap);
}

// The same for larger caps: near 0 the odd Taylor series y - y^3/3 + 2y^5/15 -
// 17y^7/315 takes over (at |y| <= 0.25 its first left-out term, 62y^9/2835, is
// 3.4e-7 of y).
__device__ __forceinline__ float softcap_log2(float x, float cap, float inv_cap) {
  const float y = x * inv_cap;
  const float y2 = y * y;
  const float p = fmaf(y2, fmaf(y2, fmaf(y2, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);
  // NaN fails the comparison and comes out of the series' argument
  return fabsf(y) > 0.25f ? softcap_direct(x, cap, inv_cap) : x * p;
}

// Token (within a unit) of a lane's element i of n-tile n.  The two n-tiles of an
// 8-bit unit's 16 tokens follow the order in which ldmatrix b8 hands out V's rows,
// chosen so that neither K's nor V's loads conflict (see v_row_8): the second
// tile's halves are exchanged.
template <bool k8>
__device__ __forceinline__ int frag_token(int n, int i, int quad) {
  const int c = 2 * quad + (i & 1);
  return n * 8 + (k8 && (n & 1) ? c ^ 4 : c);
}

// Capped and biased scores of n-tiles of 8 tokens (log2 domain).
template <int N, bool k8>
__device__ __forceinline__ void change_scores(float (&x)[N][4], const RowState& st, int tok_base,
                                              const DecodeParams& p, int quad) {
  if (p.softcap_log2 > 0.f) {
    const float cap = p.softcap_log2, inv = p.inv_softcap_log2;
    if (p.softcap <= kDirectCap) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[n][i] = softcap_direct(x[n][i], cap, inv);
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[n][i] = softcap_log2(x[n][i], cap, inv);
    }
  }
  if (p.alibi_slopes != nullptr) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = tok_base + frag_token<k8>(n, i, quad);
        x[n][i] = fmaf(-st.slope[i >> 1], fabsf((float)(st.pos[i >> 1] - tok)), x[n][i]);
      }
  }
}

// -inf for the keys a row does not see.
template <int N, bool k8>
__device__ __forceinline__ void hide_keys(float (&x)[N][4], const RowState& st, int tok_base, int quad) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int tok = tok_base + frag_token<k8>(n, i, quad);
      if (tok < st.first[i >> 1] || tok >= st.end[i >> 1]) x[n][i] = -INFINITY;
    }
}

// Once a row's reference settles, alpha is exactly 1: the accumulator is only
// rescaled when some row of the warp moved its reference.
template <int D>
__device__ __forceinline__ void rescale_rows(float (&o_acc)[D / 8][4], const float (&alpha)[2]) {
  if (!__any_sync(0xffffffffu, (alpha[0] != 1.f) | (alpha[1] != 1.f))) return;
#pragma unroll
  for (int nd = 0; nd < D / 8; ++nd) {
    o_acc[nd][0] *= alpha[0];
    o_acc[nd][1] *= alpha[0];
    o_acc[nd][2] *= alpha[1];
    o_acc[nd][3] *= alpha[1];
  }
}

__device__ __forceinline__ uint4 load_chunk(uint32_t addr) {
  uint4 w;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(addr));
  return w;
}

// Whether one of two 16-bit values (four codes) is not finite.
template <typename T>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
  const uint32_t em = kSplitProbabilities<T>::value ? 0x7f80u : 0x7c00u;
  return (w & em) == em || (w & (em << 16)) == (em << 16);
}
__device__ __forceinline__ bool nan4(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0u; }

// Mask of a register of two 16-bit values, tokens t and t + 1 of a unit whose
// dropped tokens are the set bits.
__device__ __forceinline__ uint32_t keep_pair(uint32_t dropped, int t) {
  return (((dropped >> t) & 1u) ? 0u : 0x0000ffffu) | (((dropped >> t) & 2u) ? 0u : 0xffff0000u);
}

__device__ __forceinline__ void zero_chunk(uint32_t addr) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(addr), "r"(0u) : "memory");
}

// One 16-token unit of a 16-bit cache with changed scores.
// tok_base: position of the unit's first token; tokens before tok_lo or at or
// past tok_hi are seen by no row of the tile (their V may be anything); units
// outside [full_lo, full_hi) hold keys that some row does not see.  kOwnTile: no
// other warp reads the tile, so rows to be left out can be zeroed in place; else
// their registers are masked.
template <typename T, int D, bool kOwnTile>
__device__ __forceinline__ void attend_unit_scored(uint32_t kbase, uint32_t vbase, const uint32_t (&qa)[D / 16][4],
                                                   float (&o_acc)[D / 8][4], RowState& st, int tok_base, int tok_lo,
                                                   int tok_hi, int full_lo, int full_hi, const DecodeParams& p,
                                                   int lane) {
  constexpr int NDT = D / 8;
  const int quad = lane & 3;

  // ---- S = Q K^T ----
  float x[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  {
    const int tok = ((lane >> 4) << 3) | (lane & 7);
    const uint32_t at = tile_chunk_addr<T, D>(kbase, tok, (lane >> 3) & 1);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t r0, r1, r2, r3;
      ldsm_x4(flip_chunk(at, (2 * kk) & 7) + (kk >> 2) * TileLayout<T, D>::kHalfBytes, r0, r1, r2, r3);
      Mma16816<T>::run(x[0], qa[kk], r0, r1);
      Mma16816<T>::run(x[1], qa[kk], r2, r3);
    }
  }

  // ---- scores in the log2 domain ----
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) x[n][i] *= st.c[i >> 1];
  change_scores<2, false>(x, st, tok_base, p, quad);
  const bool boundary = tok_base < full_lo || tok_base + kUnitTokens > full_hi;
  if (boundary) hide_keys<2, false>(x, st, tok_base, quad);

  // ---- online softmax ----
  float alpha[2], w[2][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float mx = fmaxf(fmaxf(x[0][2 * r], x[0][2 * r + 1]), fmaxf(x[1][2 * r], x[1][2 * r + 1]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float mn = fmaxf(st.m[r], mx);
    const float base = mn == -INFINITY ? 0.f : mn;
    alpha[r] = ex2(st.m[r] - base);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[r][i] = ex2(x[i >> 1][2 * r + (i & 1)] - base);
    st.l[r] = st.l[r] * alpha[r] + ((w[r][0] + w[r][1]) + (w[r][2] + w[r][3]));
    st.m[r] = mn;
  }
  rescale_rows<D>(o_acc, alpha);

  [[maybe_unused]] uint32_t dropped = 0;  // tokens left out of the MMA
  if (boundary) {
    // Lane pair 2t, 2t+1 looks over V row t.
    const int t = lane >> 1;
    const bool seen = tok_base + t >= tok_lo && tok_base + t < tok_hi;
    bool odd = false;
#pragma unroll
    for (int ch = 0; ch < D / 16; ++ch) {
      const uint4 v = load_chunk(tile_chunk_addr<T, D>(vbase, t, 2 * ch + (lane & 1)));
      odd |= not_finite2<T>(v.x) | not_finite2<T>(v.y) | not_finite2<T>(v.z) | not_finite2<T>(v.w);
    }
    const uint32_t pairs = __ballot_sync(0xffffffffu, odd && seen);
    uint32_t left = (pairs | (pairs >> 1)) & 0x55555555u;  // bit 2t: token t
    const uint32_t drop = __ballot_sync(0xffffffffu, !seen) | left | (left << 1);
    while (left) {
      const int to = (__ffs(left) - 1) >> 1;
      left &= left - 1;
      const int src = (lane & ~3) | ((to & 7) >> 1);  // the quad lane that holds column to
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float lo = (to >> 3) ? w[r][2] : w[r][0], hi = (to >> 3) ? w[r][3] : w[r][1];
        const float wt = __shfl_sync(0xffffffffu, (to & 1) ? hi : lo, src);
        if (tok_base + to < st.first[r] || tok_base + to >= st.end[r]) continue;
#pragma unroll
        for (int nd = 0; nd < NDT; ++nd)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int col = nd * 8 + 2 * quad + j;
            const uint32_t addr = tile_chunk_addr<T, D>(vbase, to, col / 8) + (uint32_t)(col % 8 * 2);
            unsigned short h;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(addr) : "memory");
            o_acc[nd][2 * r + j] = fmaf(wt, lo_half<T>((uint32_t)h), o_acc[nd][2 * r + j]);
          }
      }
    }
    if constexpr (kOwnTile) {
      __syncwarp();
      if ((drop >> lane) & 1u) {
#pragma unroll
        for (int ch = 0; ch < D / 16; ++ch) zero_chunk(tile_chunk_addr<T, D>(vbase, t, 2 * ch + (lane & 1)));
      }
      __syncwarp();
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) dropped |= ((drop >> (2 * j)) & 1u) << j;
    }
  }

  // ---- O += P V ----
  uint32_t pa[4] = {pack2<T>(w[0][0], w[0][1]), pack2<T>(w[1][0], w[1][1]), pack2<T>(w[0][2], w[0][3]),
                    pack2<T>(w[1][2], w[1][3])};
  constexpr bool kSplitP = kSplitProbabilities<T>::value;
  uint32_t plo[4] = {0u, 0u, 0u, 0u};
  if constexpr (kSplitP) {
    plo[0] = pack2<T>(w[0][0] - lo_half<T>(pa[0]), w[0][1] - hi_half<T>(pa[0]));
    plo[1] = pack2<T>(w[1][0] - lo_half<T>(pa[1]), w[1][1] - hi_half<T>(pa[1]));
    plo[2] = pack2<T>(w[0][2] - lo_half<T>(pa[2]), w[0][3] - hi_half<T>(pa[2]));
    plo[3] = pack2<T>(w[1][2] - lo_half<T>(pa[3]), w[1][3] - hi_half<T>(pa[3]));
  }
  const uint32_t vat = tile_chunk_addr<T, D>(vbase, (((lane >> 3) & 1) << 3) | (lane & 7), lane >> 4);
  auto pv = [&](auto masked) {
    constexpr bool kMasked = decltype(masked)::value;
    const uint32_t vm0 = kMasked ? keep_pair(dropped, 2 * quad) : 0u;
    const uint32_t vm1 = kMasked ? keep_pair(dropped, 2 * quad + 8) : 0u;
#pragma unroll
    for (int nd = 0; nd < NDT; nd += 2) {
      uint32_t v0, v1, v2, v3;
      ldsm_x4_trans(flip_chunk(vat, nd & 7) + (nd >> 3) * TileLayout<T, D>::kHalfBytes, v0, v1, v2, v3);
      if constexpr (kMasked) v0 &= vm0, v1 &= vm1, v2 &= vm0, v3 &= vm1;
      Mma16816<T>::run(o_acc[nd], pa, v0, v1);
      Mma16816<T>::run(o_acc[nd + 1], pa, v2, v3);
      if constexpr (kSplitP) {
        Mma16816<T>::run(o_acc[nd], plo, v0, v1);
        Mma16816<T>::run(o_acc[nd + 1], plo, v2, v3);
      }
    }
  };
  if (kOwnTile || !boundary)
    pv(Bool<false>{});
  else
    pv(Bool<true>{});
}

// m16n8k16 fp16 MMA on a zero accumulator.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// Two transposed 16 x 16 byte matrices, row addresses from lanes 0-15 and 16-31.
// A lane gets bytes (rows 4 (lane % 4) .. + 3, column lane / 4) and the same of
// column lane / 4 + 8 of each.
__device__ __forceinline__ void ldsm_b8_x2_trans(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2,
                                                 uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}

// Token (of 16) that V's matrix row i holds.  A lane's four bytes are rows 4q ..
// 4q + 3; with i = (q1, q0, j, e) in bits, bytes 0, 1 (j = 0) become the B operand's
// first register, whose k are columns 2q, 2q + 1 of the first score tile, bytes 2, 3
// (j = 1) the second.  Tokens 8 j + 4 (q1 ^ j) + 2 q0 + e: any 8 rows loaded
// together (fixed q1), and any 8 of a score tile (fixed j), differ modulo 8, which
// is what the swizzles keep apart.
__device__ __forceinline__ int v_row_8(int i) {
  const int e = i & 1, j = (i >> 1) & 1, q0 = (i >> 2) & 1, q1 = (i >> 3) & 1;
  return 8 * j + 4 * (q1 ^ j) + 2 * q0 + e;
}

// One 32-token unit of an 8-bit cache (parameters as above).  ks4 / vs4: the
// scales of its four groups of 8 tokens.
template <typename T, int D, bool kScored, bool kOwnTile>
__device__ __forceinline__ void attend_unit_8(uint32_t kbase, uint32_t vbase, const uint32_t (&qa)[D / 16][4],
                                              float (&o_acc)[D / 8][4], RowState& st, int tok_base, int tok_lo,
                                              int tok_hi, int full_lo, int full_hi, const float4 ks4,
                                              const float4 vs4, const DecodeParams& p, int lane) {
  constexpr int NDT = D / 8;
  const int quad = lane & 3;
  const float ks[4] = {ks4.x, ks4.y, ks4.z, ks4.w}, vs[4] = {vs4.x, vs4.y, vs4.z, vs4.w};

  // ---- S = Q K^T: n-tile n holds tokens 8n .. 8n + 7 (frag_token) ----
  float x[4][4];
  {
    // matrices: (tile 0, chunk 2kp), (0, 2kp + 1), (1, 2kp), (1, 2kp + 1)
    const int second = lane >> 4;
    const int tok = 8 * second + ((lane & 7) ^ (4 * second));
    const uint32_t at = tile_chunk_addr<e4m3_t, D>(kbase, tok, (lane >> 3) & 1);
#pragma unroll
    for (int kp = 0; kp < D / 32; ++kp)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t r[4];
        ldsm_x4(flip_chunk(at, 2 * kp) + 16u * h * TileLayout<e4m3_t, D>::kRowBytes, r[0], r[1], r[2], r[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t b0 = e4m3x2_to_f16x2(r[j]), b1 = e4m3x2_hi_to_f16x2(r[j]);
          if (kp == 0 && (j & 1) == 0)
            mma_f16_first(x[2 * h + (j >> 1)], qa[0], b0, b1);
          else
            Mma16816<__half>::run(x[2 * h + (j >> 1)], qa[2 * kp + (j & 1)], b0, b1);
        }
      }
  }

  // ---- scores in the log2 domain ----
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const float c0 = st.c[0] * ks[n], c1 = st.c[1] * ks[n];
    x[n][0] *= c0;
    x[n][1] *= c0;
    x[n][2] *= c1;
    x[n][3] *= c1;
  }
  if constexpr (kScored) change_scores<4, true>(x, st, tok_base, p, quad);
  const bool boundary = tok_base < full_lo || tok_base + kUnit8Tokens > full_hi;
  if (boundary) hide_keys<4, true>(x, st, tok_base, quad);

  // ---- online softmax, weighted by the V scales ----
  // (a comparison that NaN fails keeps a NaN scale's NaN)
  float lvs[4], ivs[4];
  constexpr float kZeros = 7.8886090522101181e-31f;  // 2^-100
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    lvs[n] = vs[n] <= kZeros ? -40.f : lg2(vs[n]);
    ivs[n] = (vs[n] <= kZeros ? 1.099511627776e12f : rcp_approx(vs[n])) * 6.103515625e-05f;  // 2^-14 / vs
  }
  float alpha[2], w[2][8];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float mx = -INFINITY;
#pragma unroll
    for (int n = 0; n < 4; ++n) mx = fmaxf(mx, fmaxf(x[n][2 * r], x[n][2 * r + 1]) + lvs[n]);
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float mn = fmaxf(st.m[r], mx - 14.f);  // the reference, lowered so that weights reach 2^14
    const float base = mn == -INFINITY ? 0.f : mn;
    alpha[r] = ex2(st.m[r] - base);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const float off = lvs[n] - base;
      w[r][2 * n] = ex2(x[n][2 * r] + off);
      w[r][2 * n + 1] = ex2(x[n][2 * r + 1] + off);
    }
    st.l[r] *= alpha[r];
    st.m[r] = mn;
  }
  rescale_rows<D>(o_acc, alpha);

  [[maybe_unused]] uint32_t dropped = 0;  // tokens left out of the MMA
  if (!boundary) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      st.l[0] = fmaf(w[0][2 * n] + w[0][2 * n + 1], ivs[n], st.l[0]);
      st.l[1] = fmaf(w[1][2 * n] + w[1][2 * n + 1], ivs[n], st.l[1]);
    }
  } else {
    // a hidden score has no weight, and no part in the norm, beside any scale
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        if (x[n][2 * r] == -INFINITY) w[r][2 * n] = 0.f;
        if (x[n][2 * r + 1] == -INFINITY) w[r][2 * n + 1] = 0.f;
        const float g = w[r][2 * n] + w[r][2 * n + 1];
        if (g != 0.f) st.l[r] = fmaf(g, ivs[n], st.l[r]);
      }
    // Lane t looks over V row t.
    const bool seen = tok_base + lane >= tok_lo && tok_base + lane < tok_hi;
    bool odd = false;
#pragma unroll
    for (int ch = 0; ch < D / 16; ++ch) {
      const uint4 v = load_chunk(tile_chunk_addr<e4m3_t, D>(vbase, lane, ch));
      odd |= nan4(v.x) | nan4(v.y) | nan4(v.z) | nan4(v.w);
    }
    uint32_t left = __ballot_sync(0xffffffffu, odd && seen);
    const bool drop = !seen || odd;
    while (left) {
      const int t = __ffs(left) - 1;
      left &= left - 1;
      const int c = (t & 7) ^ ((t >> 1) & 4);  // its column in tile t / 8
      const int src = (lane & ~3) | (c >> 1);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const bool second = c & 1, g1 = t & 8, g2 = t & 16;
        const float p0 = second ? w[r][1] : w[r][0], p1 = second ? w[r][3] : w[r][2];
        const float p2 = second ? w[r][5] : w[r][4], p3 = second ? w[r][7] : w[r][6];
        float wt = __shfl_sync(0xffffffffu, g2 ? (g1 ? p3 : p2) : (g1 ? p1 : p0), src);
        if (tok_base + t < st.first[r] || tok_base + t >= st.end[r]) continue;
        if ((g2 ? (g1 ? vs[3] : vs[2]) : (g1 ? vs[1] : vs[0])) <= kZeros) wt = 0.f;
#pragma unroll
        for (int nd = 0; nd < NDT; ++nd)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int col = nd * 8 + 2 * quad + j;
            const uint32_t addr = tile_chunk_addr<e4m3_t, D>(vbase, t, col / 16) + (uint32_t)(col % 16);
            uint32_t code;
            asm volatile("ld.shared.u8 %0, [%1];" : "=r"(code) : "r"(addr) : "memory");
            o_acc[nd][2 * r + j] = fmaf(wt, lo_half<__half>(e4m3x2_to_f16x2(code)), o_acc[nd][2 * r + j]);
          }
      }
    }
    if constexpr (kOwnTile) {
      __syncwarp();
      if (drop) {
#pragma unroll
        for (int ch = 0; ch < D / 16; ++ch) zero_chunk(tile_chunk_addr<e4m3_t, D>(vbase, lane, ch));
      }
      __syncwarp();
    } else {
      dropped = __ballot_sync(0xffffffffu, drop);
    }
  }

  // ---- O += P V: two k-steps of 16 tokens ----
  uint32_t pa[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    pa[h][0] = pack2<__half>(w[0][4 * h], w[0][4 * h + 1]);
    pa[h][1] = pack2<__half>(w[1][4 * h], w[1][4 * h + 1]);
    pa[h][2] = pack2<__half>(w[0][4 * h + 2], w[0][4 * h + 3]);
    pa[h][3] = pack2<__half>(w[1][4 * h + 2], w[1][4 * h + 3]);
  }
  if (fminf(fminf(vs[0], vs[1]), fminf(vs[2], vs[3])) <= kZeros) {  // blocks of zeros
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (vs[n] <= kZeros) pa[n >> 1][2 * (n & 1)] = pa[n >> 1][2 * (n & 1) + 1] = 0u;
  }
  const uint32_t vat = tile_chunk_addr<e4m3_t, D>(vbase, v_row_8(lane & 15), lane >> 4);
  auto pv = [&](auto masked) {
    constexpr bool kMasked = decltype(masked)::value;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t vm0 = kMasked ? keep_pair(dropped, 16 * h + 2 * quad) : 0u;
      const uint32_t vm1 = kMasked ? keep_pair(dropped, 16 * h + 8 + ((2 * quad) ^ 4)) : 0u;
#pragma unroll
      for (int c = 0; c < D / 16; c += 2) {
        uint32_t r[4];  // chunk c: columns 0-7, 8-15; chunk c + 1: the same
        ldsm_b8_x2_trans(flip_chunk(vat, c) + 16u * h * TileLayout<e4m3_t, D>::kRowBytes, r[0], r[1], r[2], r[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t b0 = e4m3x2_to_f16x2(r[j]), b1 = e4m3x2_hi_to_f16x2(r[j]);
          if constexpr (kMasked) b0 &= vm0, b1 &= vm1;
          Mma16816<__half>::run(o_acc[2 * c + j], pa[h], b0, b1);
        }
      }
    }
  };
  if (kOwnTile || !boundary)
    pv(Bool<false>{});
  else
    pv(Bool<true>{});
}

// 1 / l of a finished row.  A row without weight is zero when it sees no key, and
// NaN (0 / 0) when all its scores are -inf; so is one whose sum is NaN.
template <typename KV>
__device__ __forceinline__ float row_norm(float l, bool sees_a_key) {
  constexpr float lift = kIs8<KV>::value ? 6.103515625e-05f : 1.f;  // the weights' 2^14, which only the sum carries
  return l > 0.f ? 1.f / l * lift : (l == 0.f && !sees_a_key) ? 0.f : __int_as_float(0x7fffffff);
}

// store_rows with the norms inv0 / inv1.
template <typename T, int D>
__device__ __forceinline__ void store_rows_ext(T* op0, T* op1, const float (&o_acc)[D / 8][4], float inv0, float inv1,
                                               int quad, int Dv) {
#pragma unroll
  for (int nd = 0; nd < D / 8; ++nd) {
    const int d = nd * 8 + 2 * quad;
    if (d >= Dv) break;
    if (op0) *reinterpret_cast<uint32_t*>(op0 + d) = pack2<T>(o_acc[nd][0] * inv0, o_acc[nd][1] * inv0);
    if (op1) *reinterpret_cast<uint32_t*>(op1 + d) = pack2<T>(o_acc[nd][2] * inv1, o_acc[nd][3] * inv1);
  }
}

}  // namespace pa
