// pa_pages.cu — pages of a paged cache, moved and accounted for on the device:
// copies, and the free / fork / reserve / compact steps of a table of sequences.
//
// A sequence slot s holds seq_lens[s] tokens in the pages block_tables[s, 0 ..
// ceil(len / bs)); further entries are -1.  ref_counts[page] counts the table
// entries that hold a page (0: free).  Every step leaves these three right
// without the host: a captured decode loop can fork, free and grow.
//
//   copy     page src[i] -> page dst[i] in every given cache
//   free     each slot's pages lose a holder, the slot becomes empty
//   fork     an empty child gets its parent's tokens: full pages are shared, a
//            page in use is copied to a page of the child's own, so that a page
//            two sequences hold is never written to again
//   reserve  room for further tokens: new pages at the end of the slot's table
//   compact  the live pages move to ids [0, live): the k-th live page at or above
//            `live`, in ascending order, goes to the k-th free page below it, and
//            tables and counts follow
//
// New pages are the lowest free ids, handed out in the order of the arguments, so
// results do not depend on timing.  A call whose pages run out leaves the slots
// that did not get all of theirs as they were and flags it.
//
// Bound: copies by memory (16-byte loads, four of a thread in flight), the rest by
// latency.  48 pages of a 4-layer pool (25 MB moved) 6.7 us; 4096 pages compacted to
// 2458 live ones (525 MB moved) 97 us, of it plan 6, tables 4, copies 83 (6.3 TB/s).  The
// planning kernels are one CTA each: a prefix sum over counts in tiles of 4096, the
// next tile's loads issued before the current one is summed.  64 beams replaced by
// forks over 6000 pages: free 4, fork 8 + 6, reserve 8 us with cold caches, some 14 us
// in a row, mostly launches (marks and lists in shared memory saved 0.2).
#include <limits.h>

#include "pa_common.cuh"
#include "pa_internal.h"

namespace pa {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;
constexpr int kInvalid = -2;  // a pair or slot the plan refused

// Exclusive prefix sum over the block; total returned to every thread.
__device__ __forceinline__ int block_exclusive(int v, int* s_warp, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  __syncthreads();  // s_warp is free
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  const int w = s_warp[lane];  // kPlanThreads / 32 == 32 warps
  int wi = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, wi, o);
    if (lane >= o) wi += u;
  }
  total = __shfl_sync(0xffffffffu, wi, 31);
  const int before = __shfl_sync(0xffffffffu, wi - w, warp);
  return before + incl - v;
}

// Four neighbouring counts from id `at`; ids past the pool count as -1.
__device__ __forceinline__ int4 load_counts(const int32_t* refs, int at, int n, bool vec) {
  if (vec && at + 4 <= n) return *reinterpret_cast<const int4*>(refs + at);
  int4 v;
  v.x = at < n ? refs[at] : -1;
  v.y = at + 1 < n ? refs[at + 1] : -1;
  v.z = at + 2 < n ? refs[at + 2] : -1;
  v.w = at + 3 < n ? refs[at + 3] : -1;
  return v;
}

// The lowest free ids, ascending, into list[0 .. min(want, free)); returns how
// many there are, at most want.  The whole block calls it.
__device__ int collect_free(const int32_t* refs, int n, int want, int32_t* list, int* s_warp) {
  const bool vec = (reinterpret_cast<uintptr_t>(refs) & 15) == 0;
  int found = 0;
  constexpr int kTile = kPlanThreads * 4;
  int4 next = load_counts(refs, threadIdx.x * 4, n, vec);
  for (int base = 0; base < n && found < want; base += kTile) {
    const int at = base + threadIdx.x * 4;
    const int4 c = next;
    if (base + kTile < n) next = load_counts(refs, at + kTile, n, vec);
    const bool f[4] = {c.x == 0, c.y == 0, c.z == 0, c.w == 0};
    int total;
    int k = found + block_exclusive((int)f[0] + f[1] + f[2] + f[3], s_warp, total);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (f[j]) {
        if (k < want) list[k] = at + j;
        ++k;
      }
    found += total;
  }
  return min(found, want);
}

// Marks the first argument that names each slot: afterwards mark[slot] is its
// index.  Arguments outside [0, slots) are passed over, and so are those whose
// partner (null: none) is negative: such a pair is padding and claims nothing.  The
// whole block calls it.
__device__ void mark_first(const int32_t* arg, const int32_t* partner, int n, int slots, int32_t* mark) {
  auto names = [&](int i) { return arg[i] >= 0 && arg[i] < slots && (partner == nullptr || partner[i] >= 0); };
  for (int i = threadIdx.x; i < n; i += blockDim.x)
    if (names(i)) mark[arg[i]] = INT_MAX;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x)
    if (names(i)) atomicMin(&mark[arg[i]], i);
  __syncthreads();
}

__device__ __forceinline__ int pages_of(int len, int bs) { return (len + bs - 1) / bs; }

// Page copy of one CTA's share: bytes [lo, hi) of the pages' joint bytes (views one after the other).
template <typename V>
__device__ __forceinline__ void copy_span(const PageViews& pv, long long src, long long dst, long long lo,
                                          long long hi) {
  constexpr int kStep = kCopyThreads * (int)sizeof(V);
  long long start = 0;
  for (int v = 0; v < pv.n; ++v) {
    const PageView& w = pv.v[v];
    const long long bytes = w.segments * w.segment_bytes;
    const long long a = max(lo, start) - start, z = min(hi, start + bytes) - start;
    start += bytes;
    if (a >= z) continue;
    const char* from = static_cast<const char*>(w.data) + src * w.stride_block;
    char* to = static_cast<char*>(w.data) + dst * w.stride_block;
    for (long long o = a + (long long)threadIdx.x * sizeof(V); o < z; o += (long long)kStep * kCopyUnroll) {
      V x[kCopyUnroll];
      long long at[kCopyUnroll];
#pragma unroll
      for (int j = 0; j < kCopyUnroll; ++j) {
        const long long oj = o + (long long)j * kStep;
        at[j] = oj;
        if (w.segments > 1) {
          const long long seg = oj / w.segment_bytes;
          at[j] = seg * w.stride_segment + (oj - seg * w.segment_bytes);
        }
        if (oj < z) x[j] = *reinterpret_cast<const V*>(from + at[j]);
      }
#pragma unroll
      for (int j = 0; j < kCopyUnroll; ++j)
        if (o + (long long)j * kStep < z) *reinterpret_cast<V*>(to + at[j]) = x[j];
    }
  }
}

}  // namespace

// Copies pairs (src[i], dst[i]).  Checked (kChecked): a pair with a negative id is
// passed over, one outside the pool is flagged, and so is one whose destination
// another pair reads or an earlier pair writes: those pairs are left out, so the
// result does not depend on the order in which pairs are copied.  n_dev, when
// given, holds the number of pairs on the device.  The pairs' bytes are one line,
// cut into spans of at most span bytes (a multiple of the vector) that never
// cross a pair; CTAs take neighbouring spans, so a pair is checked once a CTA.
template <typename V, bool kChecked>
__global__ void __launch_bounds__(kCopyThreads) pages_copy_kernel(const PageViews pv, const int32_t* src,
                                                                  const int32_t* dst, int n, const int32_t* n_dev,
                                                                  int num_blocks, long long span, int spans_per_page,
                                                                  uint32_t* flags) {
  pdl_wait_previous();
  if (n_dev != nullptr) n = *n_dev;
  const long long total = (long long)n * spans_per_page;
  const long long first = total * blockIdx.x / gridDim.x, last = total * (blockIdx.x + 1) / gridDim.x;
  long long pair = -1;
  bool ok = false;
  long long s = 0, d = 0;
  for (long long k = first; k < last; ++k) {
    const long long i = k / spans_per_page;
    if (i != pair) {
      pair = i;
      s = src[i];
      d = dst[i];
      ok = s >= 0 && d >= 0;
      if constexpr (kChecked) {
        if (ok && (s >= num_blocks || d >= num_blocks)) {
          ok = false;
          if (threadIdx.x == 0) raise_flag(flags, PA_DEVERR_BLOCK_ID_RANGE);
        }
        bool clash = false;
        if (ok)
          for (int j = threadIdx.x; j < n; j += kCopyThreads) {
            const long long sj = src[j], dj = dst[j];
            if (sj < 0 || dj < 0) continue;
            clash |= (j != i && sj == d) || (j < i && dj == d);
          }
        clash = __syncthreads_or(clash);
        if (clash) {
          ok = false;
          if (threadIdx.x == 0) raise_flag(flags, PA_DEVERR_BLOCK_CONFLICT);
        }
      }
      ok = ok && s != d;
    }
    if (!ok) continue;
    const long long lo = (k - i * spans_per_page) * span;
    copy_span<V>(pv, s, d, lo, lo + span);
  }
}

__global__ void __launch_bounds__(256) pages_free_kernel(const PageTables t, const int32_t* slots, int n) {
  const int i = blockIdx.x;
  const int slot = slots[i];
  if (slot < 0) return;
  if (slot >= t.num_seqs) {
    if (threadIdx.x == 0) raise_flag(t.flags, PA_DEVERR_SEQUENCE);
    return;
  }
  bool before = false;  // freed by an earlier argument
  for (int j = threadIdx.x; j < i; j += blockDim.x) before |= slots[j] == slot;
  if (__syncthreads_or(before)) return;
  int32_t* row = t.tables + (long long)slot * t.stride;
  for (int j = threadIdx.x; j < t.max_blocks; j += blockDim.x) {
    const int page = row[j];
    if (page < 0) continue;
    if (page >= t.num_blocks)
      raise_flag(t.flags, PA_DEVERR_BLOCK_ID_RANGE);
    else if (atomicSub(&t.refs[page], 1) <= 0) {
      atomicAdd(&t.refs[page], 1);  // nobody held it: the table and the counts disagree
      raise_flag(t.flags, PA_DEVERR_SEQUENCE);
    }
    row[j] = -1;
  }
  if (threadIdx.x == 0) t.lens[slot] = 0;
}

// Plan of a fork: fresh[i] = the child's own page for the parent's page in use, -1
// when there is none to copy, kInvalid when pair i is passed over; len[i] = the
// parent's length.
__global__ void __launch_bounds__(kPlanThreads) pages_fork_plan_kernel(const PageTables t, const int32_t* parents,
                                                                       const int32_t* children, int n) {
  __shared__ int s_warp[32];
  int32_t* mark = t.scratch;
  int32_t* fresh = mark + t.num_seqs;
  int32_t* len = fresh + t.num_seqs;
  int32_t* list = len + t.num_seqs;
  mark_first(children, parents, n, t.num_seqs, mark);
  int want = 0;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int need = 0, f = kInvalid, l = 0;
    if (i < n) {
      const int p = parents[i], c = children[i];
      if (p >= 0 && c >= 0) {
        bool ok = p < t.num_seqs && c < t.num_seqs;
        ok = ok && mark[c] == i && t.lens[c] == 0 && t.tables[(long long)c * t.stride] < 0;
        if (ok) {
          l = t.lens[p];
          ok = l >= 0 && pages_of(l, t.bs) <= t.max_blocks;
        }
        if (!ok)
          raise_flag(t.flags, PA_DEVERR_SEQUENCE);
        else {
          f = -1;
          need = l % t.bs != 0;
        }
      }
    }
    int total;
    const int k = want + block_exclusive(need, s_warp, total);
    if (i < n) {
      fresh[i] = need ? k : f;  // the rank of its page, for now
      len[i] = need ? ~l : l;   // complemented: waits for a page
    }
    want += total;
  }
  const int have = collect_free(t.refs, t.num_blocks, want, list, s_warp);
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    if (len[i] >= 0) continue;
    len[i] = ~len[i];
    const int k = fresh[i];
    if (k < have) {
      fresh[i] = list[k];
    } else {
      fresh[i] = kInvalid;
      raise_flag(t.flags, PA_DEVERR_PAGES_EXHAUSTED);
    }
  }
}

// A fork's tables, counts and page copies, from its plan.  CTA (i, y): span y of
// pair i's page; y = 0 also writes the child's row.
template <typename V>
__global__ void __launch_bounds__(kCopyThreads) pages_fork_kernel(const PageTables t, const int32_t* parents,
                                                                  const int32_t* children, const PageViews pv,
                                                                  long long span) {
  pdl_wait_previous();
  const int i = blockIdx.x;
  const int32_t* fresh = t.scratch + t.num_seqs;
  const int f = fresh[i], l = fresh[t.num_seqs + i];
  if (f == kInvalid || l == 0) return;
  const int full = l / t.bs;
  const int32_t* from = t.tables + (long long)parents[i] * t.stride;
  const long long tail = f >= 0 ? from[full] : 0;
  if (f >= 0 && (tail < 0 || tail >= t.num_blocks)) {
    if (threadIdx.x == 0 && blockIdx.y == 0) raise_flag(t.flags, PA_DEVERR_BLOCK_ID_RANGE);
  } else if (f >= 0 && pv.n > 0) {
    const long long lo = span * blockIdx.y;
    copy_span<V>(pv, tail, f, lo, lo + span);
  }
  if (blockIdx.y != 0) return;
  int32_t* row = t.tables + (long long)children[i] * t.stride;
  for (int j = threadIdx.x; j < full; j += kCopyThreads) {
    const int page = from[j];
    row[j] = page;
    if (page >= 0 && page < t.num_blocks)
      atomicAdd(&t.refs[page], 1);
    else
      raise_flag(t.flags, PA_DEVERR_BLOCK_ID_RANGE);
  }
  if (threadIdx.x == 0) {
    if (f >= 0) {
      row[full] = f;
      t.refs[f] = 1;
    }
    t.lens[children[i]] = l;
  }
}

__global__ void __launch_bounds__(kPlanThreads) pages_reserve_kernel(const PageTables t, const int32_t* slots,
                                                                     const int32_t* tokens, int n) {
  __shared__ int s_warp[32];
  int32_t* mark = t.scratch;
  int32_t* rank = mark + t.num_seqs;
  int32_t* list = rank + 2 * t.num_seqs;
  mark_first(slots, nullptr, n, t.num_seqs, mark);
  long long want = 0;  // pages asked for; at most n * max_blocks
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int need = 0, ok = 0;
    if (i < n && slots[i] >= 0) {
      const int s = slots[i], more = tokens[i];
      if (s >= t.num_seqs || mark[s] != i || more < 0 || t.lens[s] < 0) {
        raise_flag(t.flags, PA_DEVERR_SEQUENCE);
      } else {
        const long long len = (long long)t.lens[s] + more;
        if (len > (long long)t.max_blocks * t.bs)
          raise_flag(t.flags, PA_DEVERR_TABLE_UNDERRUN);
        else {
          ok = 1;
          need = (int)((len + t.bs - 1) / t.bs) - pages_of(t.lens[s], t.bs);
        }
      }
    }
    int total;
    const int before = block_exclusive(need, s_warp, total);
    // past the pool's size a rank only says that there are no pages for it
    if (i < n) rank[i] = ok ? (int)min(want + before, (long long)t.num_blocks + 1) : kInvalid;
    want += total;
  }
  const int have = collect_free(t.refs, t.num_blocks, (int)min(want, (long long)t.num_blocks), list, s_warp);
  __syncthreads();
  // a warp for each slot
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < n; i += kPlanThreads / 32) {
    const int k = rank[i];
    if (k == kInvalid) continue;
    const int s = slots[i], len = t.lens[s];
    const int old = pages_of(len, t.bs), need = pages_of(len + tokens[i], t.bs) - old;
    __syncwarp();
    if (need > have - k) {
      if (need > 0) {
        if (lane == 0) raise_flag(t.flags, PA_DEVERR_PAGES_EXHAUSTED);
        continue;
      }
    }
    int32_t* row = t.tables + (long long)s * t.stride + old;
    for (int j = lane; j < need; j += 32) {
      const int page = list[k + j];
      row[j] = page;
      t.refs[page] = 1;
    }
    if (lane == 0) t.lens[s] = len + tokens[i];
  }
}

// Plan of a compaction: pairs (src, dst) and their number, the map old id -> new
// id, and the counts moved.
__global__ void __launch_bounds__(kPlanThreads) pages_compact_plan_kernel(const PageTables t, int32_t* live_out) {
  __shared__ int s_warp[32];
  const int n = t.num_blocks;
  int32_t* map = t.scratch;
  int32_t* src = map + n;
  int32_t* dst = src + n / 2 + 1;
  int32_t* count = dst + n / 2 + 1;
  const bool vec = (reinterpret_cast<uintptr_t>(t.refs) & 15) == 0;
  int mine = 0;
  for (int at = threadIdx.x * 4; at < n; at += kPlanThreads * 4) {
    const int4 c = load_counts(t.refs, at, n, vec);
    mine += (c.x > 0) + (c.y > 0) + (c.z > 0) + (c.w > 0);
  }
  int live;
  block_exclusive(mine, s_warp, live);
  int holes = 0, high = 0;
  int4 next = load_counts(t.refs, threadIdx.x * 4, n, vec);
  for (int base = 0; base < n; base += kPlanThreads * 4) {
    const int at = base + threadIdx.x * 4;
    const int4 c4 = next;
    if (base + kPlanThreads * 4 < n) next = load_counts(t.refs, at + kPlanThreads * 4, n, vec);
    const int c[4] = {c4.x, c4.y, c4.z, c4.w};
    int h = 0, g = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (at + j >= n) continue;
      if (at + j < live)
        h += c[j] <= 0;
      else
        g += c[j] > 0;
    }
    // one sum for both: each is below 2^16 in a tile
    int total;
    const int before = block_exclusive(h | (g << 16), s_warp, total);
    int kh = holes + (before & 0xffff), kg = high + (before >> 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (at + j >= n) continue;
      if (at + j < live) {
        if (c[j] <= 0) dst[kh++] = at + j;
      } else if (c[j] > 0) {
        src[kg++] = at + j;
      }
      map[at + j] = at + j;
    }
    holes += total & 0xffff;
    high += total >> 16;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < high; i += kPlanThreads) {
    const int s = src[i], d = dst[i];
    map[s] = d;
    t.refs[d] = t.refs[s];
    t.refs[s] = 0;
  }
  if (threadIdx.x == 0) {
    *count = high;
    *live_out = live;
  }
}

__global__ void __launch_bounds__(256) pages_remap_kernel(const PageTables t) {
  pdl_launch_dependents();
  pdl_wait_previous();
  const long long total = (long long)t.num_seqs * t.max_blocks;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const long long s = i / t.max_blocks;
    int32_t* at = t.tables + s * t.stride + (i - s * t.max_blocks);
    const int page = *at;
    if (page < 0) continue;
    if (page >= t.num_blocks)
      raise_flag(t.flags, PA_DEVERR_BLOCK_ID_RANGE);
    else
      *at = t.scratch[page];
  }
}

namespace {

long long page_bytes(const PageViews& pv) {
  long long b = 0;
  for (int v = 0; v < pv.n; ++v) b += pv.v[v].segments * pv.v[v].segment_bytes;
  return b;
}

// Widest vector (16, 4 or 1 bytes) that every address and length is a multiple of.
int view_vector(const PageViews& pv) {
  int vec = 16;
  for (int v = 0; v < pv.n; ++v) {
    const PageView& w = pv.v[v];
    const uintptr_t all = reinterpret_cast<uintptr_t>(w.data) | (uintptr_t)w.stride_block |
                          (uintptr_t)w.stride_segment | (uintptr_t)w.segment_bytes;
    while (all % vec != 0) vec /= 4;  // 16, 4, 1
  }
  return vec;
}

// Bytes of a page that one CTA copies at a time.
constexpr long long kSpan = (long long)kCopyThreads * kCopyUnroll * 16;

template <typename... A>
cudaError_t launch_pdl(void (*kernel)(A...), dim3 grid, int threads, bool pdl, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = pdl ? attr : nullptr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename V>
cudaError_t copy_typed(const PageViews& pv, const int32_t* src, const int32_t* dst, int n, const int32_t* n_dev,
                       int most, int num_blocks, bool checked, bool pdl, int num_sms, uint32_t* flags,
                       cudaStream_t stream) {
  const int spans = (int)((page_bytes(pv) + kSpan - 1) / kSpan);
  const long long want = (long long)most * spans;
  const unsigned grid = (unsigned)(want < num_sms * 8LL ? (want > 0 ? want : 1) : num_sms * 8LL);
  auto kernel = checked ? pages_copy_kernel<V, true> : pages_copy_kernel<V, false>;
  return launch_pdl(kernel, dim3(grid), kCopyThreads, pdl, stream, pv, src, dst, n, n_dev, num_blocks, kSpan, spans,
                    flags);
}

cudaError_t copy_any(const PageViews& pv, const int32_t* src, const int32_t* dst, int n, const int32_t* n_dev,
                     int most, int num_blocks, bool checked, bool pdl, int num_sms, uint32_t* flags,
                     cudaStream_t stream) {
  switch (view_vector(pv)) {
    case 16:
      return copy_typed<uint4>(pv, src, dst, n, n_dev, most, num_blocks, checked, pdl, num_sms, flags, stream);
    case 4:
      return copy_typed<uint32_t>(pv, src, dst, n, n_dev, most, num_blocks, checked, pdl, num_sms, flags, stream);
    default:
      return copy_typed<uint8_t>(pv, src, dst, n, n_dev, most, num_blocks, checked, pdl, num_sms, flags, stream);
  }
}

}  // namespace

cudaError_t launch_pages_copy(const PageViews& pv, const int32_t* src, const int32_t* dst, int n, int num_blocks,
                              int num_sms, uint32_t* flags, cudaStream_t stream) {
  return copy_any(pv, src, dst, n, nullptr, n, num_blocks, true, false, num_sms, flags, stream);
}

cudaError_t launch_pages_free(const PageTables& t, const int32_t* slots, int n, cudaStream_t stream) {
  pages_free_kernel<<<n, 256, 0, stream>>>(t, slots, n);
  return cudaGetLastError();
}

cudaError_t launch_pages_fork(const PageTables& t, const int32_t* parents, const int32_t* children, int n,
                              const PageViews& pv, cudaStream_t stream) {
  pages_fork_plan_kernel<<<1, kPlanThreads, 0, stream>>>(t, parents, children, n);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const long long spans = (page_bytes(pv) + kSpan - 1) / kSpan;
  const dim3 grid((unsigned)n, (unsigned)(spans > 0 ? spans : 1));
  switch (view_vector(pv)) {
    case 16:
      return launch_pdl(pages_fork_kernel<uint4>, grid, kCopyThreads, true, stream, t, parents, children, pv, kSpan);
    case 4:
      return launch_pdl(pages_fork_kernel<uint32_t>, grid, kCopyThreads, true, stream, t, parents, children, pv,
                        kSpan);
    default:
      return launch_pdl(pages_fork_kernel<uint8_t>, grid, kCopyThreads, true, stream, t, parents, children, pv,
                        kSpan);
  }
}

cudaError_t launch_pages_reserve(const PageTables& t, const int32_t* slots, const int32_t* tokens, int n,
                                 cudaStream_t stream) {
  pages_reserve_kernel<<<1, kPlanThreads, 0, stream>>>(t, slots, tokens, n);
  return cudaGetLastError();
}

cudaError_t launch_pages_compact(const PageTables& t, const PageViews& pv, int32_t* live, int num_sms,
                                 cudaStream_t stream) {
  pages_compact_plan_kernel<<<1, kPlanThreads, 0, stream>>>(t, live);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const long long entries = (long long)t.num_seqs * t.max_blocks;
  const long long blocks = (entries + 255) / 256;
  e = launch_pdl(pages_remap_kernel, dim3((unsigned)(blocks < num_sms * 8LL ? blocks : num_sms * 8LL)), 256, true,
                 stream, t);
  if (e != cudaSuccess || pv.n == 0) return e;
  const int n = t.num_blocks;
  const int32_t* src = t.scratch + n;
  const int32_t* dst = src + n / 2 + 1;
  return copy_any(pv, src, dst, 0, dst + n / 2 + 1, n / 2 + 1, n, false, true, num_sms, t.flags, stream);
}

}  // namespace pa
