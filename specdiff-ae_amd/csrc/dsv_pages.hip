// dsv_pages.hip — page operations of a paged KV cache on gfx950: fork, extend,
// free and compact, on device tables and reference counts.
//
// Bookkeeping.  A pool of P pages is shared by B sequences: page_table
// [B, n_log] names each sequence's pages (-1: none), refcount [P] counts the
// tables' entries (0: free), seqlens [B] holds the tokens.  Every operation
// reads and writes these on the device, so a serving loop needs no host round
// trip.  Pages are taken in ascending order, for the requests in ascending
// order: results do not depend on which thread comes first (reference counts
// change by integer atomics, whose order does not matter).
//
// Split.  fork and compact are two launches: a plan by one workgroup (who gets
// which page: prefix sums over the counts, 4 bytes a page), then the copies by
// the whole chip.  extend is the plan alone, free one launch over the entries.
// The plan is latency (fork and extend 5 to 7 us, compact of 2048 pages 7); the
// copies are bound by HBM: each page is read and written once, in 16-byte pieces,
// eight in flight per thread.  92 pages of 2 MiB of 23 parents: 57 us, 6.8 TB/s of
// reads and writes together (a parent's page comes from the cache after the first
// time); 507 pages of 512 KiB moved: 101 to 114 us, 4.7 to 5.2 TB/s.
//
// Reference: core/kv_cache/paged_kv.py:81-166 (allocation, sharing with copy
// on write, release) and :364-402 (defragmentation) keep this on the host.

#include "dsv_internal.h"

namespace dsv {

namespace {

constexpr int kPT = kPlanThreads;
constexpr int kPW = kPT / 64;       // waves of the planning workgroup
constexpr int kScanStep = 4 * kPT;  // pages of a scan step
constexpr int kFewPages = 8;        // pages that one thread hands to a sequence

__device__ __forceinline__ int64_t get(const PageIndex& x, int64_t i) {
  return x.is64 ? reinterpret_cast<const int64_t*>(x.p)[i * x.stride]
                : (int64_t) reinterpret_cast<const int32_t*>(x.p)[i * x.stride];
}
__device__ __forceinline__ int64_t seqlen(const PageBook& b, int64_t i) {
  return b.lens_i64 ? reinterpret_cast<const int64_t*>(b.lens)[i] : (int64_t) reinterpret_cast<const int32_t*>(b.lens)[i];
}
__device__ __forceinline__ void set_seqlen(const PageBook& b, int64_t i, int64_t n) {
  if (b.lens_i64)
    reinterpret_cast<int64_t*>(b.lens)[i] = n;
  else
    reinterpret_cast<int32_t*>(b.lens)[i] = (int32_t)n;
}

// x of the lane that DPP control CTRL names, 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t dpp(int64_t x) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)((uint64_t)x >> 32), CTRL, ROWS, 0xf, false);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// Exclusive scan of one value per thread over the planning workgroup.
__device__ __forceinline__ int64_t scan1(int64_t x, int64_t* scratch, int64_t& total) {
  // Shifts by 1, 2, 4, 8 inside the rows of 16, then the last lanes of rows 0 and
  // 2, then of row 1, handed on.
  int64_t inc = x;
  inc += dpp<0x111, 0xf>(inc);
  inc += dpp<0x112, 0xf>(inc);
  inc += dpp<0x114, 0xf>(inc);
  inc += dpp<0x118, 0xf>(inc);
  inc += dpp<0x142, 0xa>(inc);
  inc += dpp<0x143, 0xc>(inc);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) scratch[threadIdx.x >> 6] = inc;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll 1
  for (int i = 0; i < kPW; ++i) {
    if (i == (int)(threadIdx.x >> 6)) before = total;
    total += scratch[i];
  }
  return before + inc - x;
}

// The counts of this thread's four pages of the scan step at s0 (0 behind the pool).
typedef int32_t i32x4 __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ i32x4 refs_at(const PageBook& b, int64_t s0) {
  const int64_t i = s0 + 4 * (int)threadIdx.x;
  if (i + 4 <= b.P) return *reinterpret_cast<const i32x4*>(b.ref + i);
  i32x4 r = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (i + e < b.P) r[e] = b.ref[i + e];
  return r;
}

// Visits the pages of [lo, hi) whose number and count satisfy pred in ascending
// order: each calls emit(index, rank), rank counted from 0; stops after the step
// in which `limit` were found.  Returns how many were found (more than limit
// possible).  Steps start at multiples of kScanStep; `first` holds the counts of
// the first one, read once for all of a plan's scans.  What a plan of a few
// hundred pages takes is mostly the fetching of its code from memory: four pages
// a thread and loops that are not unrolled (16 a thread, unrolled: 2 to 4 times the
// code; compact's plan of 2048 pages took 10 us, so 7).
template <typename Pred, typename Emit>
__device__ __forceinline__ int64_t scan_pages(const PageBook& b, const i32x4& first, int64_t lo, int64_t hi, int64_t limit,
                                              int32_t* cnt, Pred pred, Emit emit) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t below = (1ull << lane) - 1ull;
  int64_t found = 0;
#pragma unroll 1
  for (int64_t s0 = lo - lo % kScanStep; s0 < hi && found < limit; s0 += kScanStep) {
    const int64_t i = s0 + 4 * (int)threadIdx.x;
    const i32x4 ref = s0 == 0 ? first : refs_at(b, s0);
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e >= lo && i + e < hi && pred(i + e, ref[e])) bits |= 1u << e;
    // The number of entries before this thread's, from the bits of the numbers.
    const int n = __builtin_popcount(bits);
    const uint64_t b0 = __ballot(n & 1), b1 = __ballot(n & 2), b2 = __ballot(n & 4);
    __syncthreads();  // the previous step's counts have been read
    if (lane == 0) cnt[wave] = __builtin_popcountll(b0) + 2 * __builtin_popcountll(b1) + 4 * __builtin_popcountll(b2);
    __syncthreads();
    int before = __builtin_popcountll(b0 & below) + 2 * __builtin_popcountll(b1 & below) + 4 * __builtin_popcountll(b2 & below);
    int all = 0;
#pragma unroll 1
    for (int w = 0; w < kPW; ++w) {
      before += w < wave ? cnt[w] : 0;
      all += cnt[w];
    }
    int64_t at = found + before;
#pragma unroll 1
    for (int e = 0; e < 4; ++e)
      if ((bits >> e) & 1u) emit(i + e, at++);
    found += all;
  }
  return found;
}

// ---- copies ---------------------------------------------------------------

constexpr int kCopyT = 256;
constexpr int kCopyN = 8;                          // 16-byte chunks per thread and piece
constexpr int kCopyPiece = kCopyT * kCopyN;        // chunks of a piece

// Copies page src[i] to dst[i] of every slab for the pairs [0, n), the pieces
// shared out over the workgroups [wg, wg + step, ..).  Pairs with dst < 0 are
// skipped.
template <bool CONTIG>
__device__ __forceinline__ void copy_pages(const PageData& d, const int32_t* src, const int32_t* dst, int64_t n,
                                           int64_t wg, int64_t step) {
  const int chunks = d.n1 * d.n2 * d.row16;
  const int pieces = (chunks + kCopyPiece - 1) / kCopyPiece;
  const int64_t slabs = 2 * (int64_t)d.n_l;
  const int64_t items = n * slabs * pieces;
  for (int64_t it = wg; it < items; it += step) {
    const int piece = (int)(it % pieces);
    const int64_t r = it / pieces;
    const int64_t slab = r % slabs, i = r / slabs;
    const int32_t to = dst[i], from = src[i];
    if (to < 0) continue;
    char* base = d.kv + (slab >> 1) * d.s_l + (slab & 1) * d.s_h;
    const char* s = base + from * d.s_p;
    char* t = base + to * d.s_p;
    u32x4 x[kCopyN];
    int64_t off[kCopyN];
#pragma unroll
    for (int k = 0; k < kCopyN; ++k) {
      const int c = piece * kCopyPiece + k * kCopyT + (int)threadIdx.x;
      if (CONTIG) {
        off[k] = (int64_t)c * 16;
      } else {
        const int row = c / d.row16;
        off[k] = (int64_t)(row / d.n2) * d.s_1 + (int64_t)(row % d.n2) * d.s_2 + (int64_t)(c - row * d.row16) * 16;
      }
      if (c < chunks) x[k] = *reinterpret_cast<const u32x4*>(s + off[k]);
    }
#pragma unroll
    for (int k = 0; k < kCopyN; ++k)
      if (piece * kCopyPiece + k * kCopyT + (int)threadIdx.x < chunks) *reinterpret_cast<u32x4*>(t + off[k]) = x[k];
  }
}

// ---- fork -------------------------------------------------------------------

// Checks the pairs, finds the pages for the copies of partly filled last
// pages and, if all is well, takes them; otherwise nothing changes.
__global__ void __launch_bounds__(kPT) fork_plan_kernel(const ForkArgs a) {
  __shared__ uint32_t is_child[kPageMaxSeqs / 32], is_parent[kPageMaxSeqs / 32];
  __shared__ int64_t scratch[kPW];
  __shared__ int32_t cnt[kPW];
  __shared__ int32_t bad;
  const PageBook& b = a.book;
  const i32x4 first = refs_at(b, 0);
  const int64_t ps = 1ll << b.ps_shift;
  for (int64_t i = threadIdx.x; i < (b.B + 31) / 32; i += kPT) is_child[i] = is_parent[i] = 0;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  for (int64_t i = threadIdx.x; i < a.n; i += kPT) {
    const int64_t p = get(a.parents, i), c = get(a.children, i);
    bool ok = p >= 0 && p < b.B && c >= 0 && c < b.B && p != c;
    if (ok) {
      const int64_t len = seqlen(b, p);
      ok = len >= 0 && len <= b.n_log * ps && seqlen(b, c) == 0;
      ok = (atomicOr(&is_child[c >> 5], 1u << (c & 31)) >> (c & 31) & 1u) == 0 && ok;
      atomicOr(&is_parent[p >> 5], 1u << (p & 31));
    }
    if (!ok) atomicAdd(&bad, 1);
  }
  __syncthreads();
  // A child that is also a parent of this call: its state would depend on the order.
  for (int64_t i = threadIdx.x; i < a.n; i += kPT) {
    const int64_t c = get(a.children, i);
    if (c >= 0 && c < b.B && (is_parent[c >> 5] >> (c & 31) & 1u)) atomicAdd(&bad, 1);
  }
  __syncthreads();
  const int refused = bad;
  // The pairs with a partly filled last page, in order: src, and in dst the rank.
  int64_t want = 0;
  if (refused == 0) {
    for (int64_t i0 = 0; i0 < a.n; i0 += kPT) {
      const int64_t i = i0 + threadIdx.x;
      int32_t page = -1;
      if (i < a.n) {
        const int64_t p = get(a.parents, i), len = seqlen(b, p);
        if ((len & (ps - 1)) != 0) {
          page = b.table[p * b.t_sb + (len >> b.ps_shift)];
          if (page < 0 || page >= b.P) page = -1;
        }
      }
      int64_t total;
      const int64_t rank = want + scan1(page >= 0 ? 1 : 0, scratch, total);
      if (i < a.n) {
        a.src[i] = page;
        a.dst[i] = page >= 0 ? (int32_t)rank : -1;
      }
      want += total;
    }
  }
  // list[rank] = page, kept behind the pairs.
  int32_t* list = a.dst + a.n;
  const int64_t found = scan_pages(
      b, first, 0, b.P, want, cnt, [](int64_t, int32_t ref) { return ref == 0; },
      [&](int64_t i, int64_t r) {
        if (r < want) list[r] = (int32_t)i;
      });
  const bool go = refused == 0 && found >= want;
  __syncthreads();
  if (threadIdx.x == 0) {
    a.state[0] = go ? (int32_t)a.n : 0;
    a.info[0] = go ? (int32_t)want : 0;
    a.info[1] = go ? 0 : (int32_t)(want > found ? want - found : 0);
    a.info[2] = refused;
  }
  if (!go) return;
  for (int64_t i = threadIdx.x; i < a.n; i += kPT) {
    if (a.dst[i] >= 0) {
      const int32_t page = list[a.dst[i]];
      a.dst[i] = page;
      b.ref[page] = 1;
    }
    set_seqlen(b, get(a.children, i), seqlen(b, get(a.parents, i)));
  }
}

template <bool CONTIG>
__global__ void __launch_bounds__(kCopyT) fork_kernel(const ForkArgs a, int64_t rows_wg) {
  const int64_t n = a.state[0];
  const PageBook& b = a.book;
  if (blockIdx.x < rows_wg) {
    // The children's table rows and the shared pages' counts.
    const int64_t ps = 1ll << b.ps_shift;
    for (int64_t x = (int64_t)blockIdx.x * kCopyT + threadIdx.x; x < n * b.n_log; x += rows_wg * kCopyT) {
      const int64_t i = x / b.n_log, j = x - i * b.n_log;
      const int64_t p = get(a.parents, i), len = seqlen(b, p);
      int32_t page = j * ps < len ? b.table[p * b.t_sb + j] : -1;
      if ((j + 1) * ps <= len) {
        if (page >= 0 && page < b.P) atomicAdd(&b.ref[page], 1);
      } else if (page >= 0 && a.dst[i] >= 0) {
        page = a.dst[i];
      }
      b.table[get(a.children, i) * b.t_sb + j] = page;
    }
    return;
  }
  copy_pages<CONTIG>(a.data, a.src, a.dst, n, blockIdx.x - rows_wg, gridDim.x - rows_wg);
}

// ---- extend ----------------------------------------------------------------

// Pages that a sequence's row already names behind its tokens stay its own (those
// of drafted tokens that were rejected); the missing ones are taken.
__global__ void __launch_bounds__(kPT) extend_kernel(const ExtendArgs a) {
  __shared__ int64_t scratch[kPW];
  __shared__ int32_t cnt[kPW];
  __shared__ int32_t bad, many;
  const PageBook& b = a.book;
  const int64_t ps = 1ll << b.ps_shift;
  const i32x4 first = refs_at(b, 0);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) bad = many = 0;
  __syncthreads();
  auto pages_of = [&](int64_t n) { return (n >> b.ps_shift) + ((n & (ps - 1)) != 0 ? 1 : 0); };
  auto missing = [&](int64_t i, int64_t j) {
    const int32_t page = b.table[i * b.t_sb + j];
    return page < 0 || page >= b.P;
  };
  // Which of up to kFewPages entries from lo on are missing.
  auto missing_few = [&](int64_t i, int64_t lo, int n) {
    int32_t page[kFewPages];
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < kFewPages; ++j) page[j] = j < n ? b.table[i * b.t_sb + lo + j] : 0;
#pragma unroll
    for (int j = 0; j < kFewPages; ++j) bits |= (page[j] < 0 || page[j] >= b.P ? 1u : 0u) << j;
    return bits;
  };
  // The pages that sequences lack: a thread counts a few, a wave many.
  int64_t want = 0, lo = 0, hi = 0;
  uint32_t few = 0;
  for (int64_t i0 = 0; i0 < b.B; i0 += kPT) {
    const int64_t i = i0 + threadIdx.x;
    lo = hi = 0;
    if (i < b.B) {
      const int64_t len = seqlen(b, i), n = get(a.newlens, i);
      if (n > len) {
        if (len < 0 || n > b.n_log * ps) {
          atomicAdd(&bad, 1);
        } else {
          lo = pages_of(len);
          hi = pages_of(n);
        }
      }
    }
    const bool is_many = hi - lo > kFewPages;
    few = is_many ? 0u : missing_few(i, lo, (int)(hi - lo));
    int64_t need = __builtin_popcount(few);
    if (__syncthreads_or(is_many) != 0) {
      if (threadIdx.x == 0) many = 1;
      for (uint64_t left = __ballot(is_many); left != 0; left &= left - 1) {
        const int src = __builtin_ctzll(left);
        const int64_t l = __shfl((long long)lo, src), h = __shfl((long long)hi, src), s = __shfl((long long)i, src);
        int found = 0;
        for (int64_t j = l + lane; j - lane < h; j += 64) found += __builtin_popcountll(__ballot(j < h && missing(s, j)));
        if (lane == src) need = found;
      }
    }
    int64_t total;
    const int64_t at = want + scan1(need, scratch, total);
    if (i < b.B) a.off[i] = at;
    want += total;
  }
  __syncthreads();
  const int refused = bad;
  const int64_t limit = refused == 0 ? want : 0;
  const int64_t found = scan_pages(
      b, first, 0, b.P, limit, cnt, [](int64_t, int32_t ref) { return ref == 0; },
      [&](int64_t i, int64_t r) {
        if (r < limit) a.list[r] = (int32_t)i;
      });
  const bool go = refused == 0 && found >= want;
  __syncthreads();
  if (threadIdx.x == 0) {
    a.info[0] = go ? (int32_t)want : 0;
    a.info[1] = refused == 0 && want > found ? (int32_t)(want - found) : 0;
    a.info[2] = refused;
  }
  if (!go) return;
  const bool again = b.B > kPT;  // (else lo, hi and few are this thread's sequence's)
  for (int64_t i = threadIdx.x; i < b.B; i += kPT) {
    const int64_t n = get(a.newlens, i);
    if (again) {
      const int64_t len = seqlen(b, i);
      lo = n > len ? pages_of(len) : 0;
      hi = n > len ? pages_of(n) : 0;
      few = hi - lo > kFewPages ? 0u : missing_few(i, lo, (int)(hi - lo));
    }
    if (hi - lo > kFewPages) continue;
    int64_t at = a.off[i];
#pragma unroll 1
    for (uint32_t left = few; left != 0; left &= left - 1) {
      const int32_t page = a.list[at++];
      b.table[i * b.t_sb + lo + __builtin_ctz(left)] = page;
      b.ref[page] = 1;
    }
    if (n > seqlen(b, i)) set_seqlen(b, i, n);
  }
  __syncthreads();
  if (many == 0) return;
  for (int64_t i = wave; i < b.B; i += kPW) {
    const int64_t len = seqlen(b, i), n = get(a.newlens, i);
    if (n <= len) continue;  // (those done above among them)
    const int64_t l = pages_of(len), h = pages_of(n);
    int64_t at = a.off[i];
    for (int64_t j = l + lane; j - lane < h; j += 64) {
      const bool take = j < h && missing(i, j);
      const uint64_t all = __ballot(take);
      if (take) {
        const int32_t page = a.list[at + __builtin_popcountll(all & ((1ull << lane) - 1ull))];
        b.table[i * b.t_sb + j] = page;
        b.ref[page] = 1;
      }
      at += __builtin_popcountll(all);
    }
    // Every lane has read the length before it changes.
    __builtin_amdgcn_wave_barrier();
    if (lane == 0) set_seqlen(b, i, n);
  }
}

// ---- free -------------------------------------------------------------------

__global__ void __launch_bounds__(256) free_kernel(const FreeArgs a) {
  const PageBook& b = a.book;
  const int64_t ps = 1ll << b.ps_shift;
  for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < a.n * b.n_log; x += (int64_t)gridDim.x * 256) {
    const int64_t i = x / b.n_log, j = x - i * b.n_log;
    const int64_t s = get(a.seqs, i);
    if (s < 0 || s >= b.B) continue;
    // Behind the window: every token of the page lies after the sinks and is
    // out of sight of the next token, at position len, which sees n > len - window.
    const bool gone = a.window == 0 || (j * ps >= a.sinks && (j + 1) * ps <= seqlen(b, s) - a.window + 1);
    if (gone) {
      // A sequence named twice gives its pages back once.
      const int32_t page = atomicExch(&b.table[s * b.t_sb + j], -1);
      if (page >= 0 && page < b.P && atomicSub(&b.ref[page], 1) <= 0) atomicAdd(&b.ref[page], 1);
    }
    if (a.window == 0 && j == 0) set_seqlen(b, s, 0);
  }
}

// ---- compact ----------------------------------------------------------------

// The pages in use at or behind n = their number move, in order, into the
// free pages below n.
__global__ void __launch_bounds__(kPT) compact_plan_kernel(const CompactArgs a) {
  __shared__ int64_t scratch[kPW];
  __shared__ int32_t cnt[kPW];
  const PageBook& b = a.book;
  const i32x4 first = refs_at(b, 0);
  int64_t mine = 0;
#pragma unroll 1
  for (int64_t s0 = 0; s0 < b.P; s0 += kScanStep) {
    const i32x4 ref = s0 == 0 ? first : refs_at(b, s0);
#pragma unroll
    for (int e = 0; e < 4; ++e) mine += ref[e] > 0 ? 1 : 0;
  }
  int64_t n;
  scan1(mine, scratch, n);
  // (As many as are moved: n pages are in use, those below n and the moved ones.)
  scan_pages(
      b, first, 0, n, b.P, cnt, [](int64_t, int32_t ref) { return ref <= 0; }, [&](int64_t i, int64_t r) { a.dst[r] = (int32_t)i; });
  const int64_t moved = scan_pages(
      b, first, n, b.P, b.P, cnt,
      [&](int64_t i, int32_t ref) {
        a.to[i] = (int32_t)i;
        return ref > 0;
      },
      [&](int64_t i, int64_t r) { a.src[r] = (int32_t)i; });
  __syncthreads();
  for (int64_t r = threadIdx.x; r < moved; r += kPT) {
    const int32_t s = a.src[r], d = a.dst[r];
    a.to[s] = d;
    b.ref[d] = b.ref[s];
    b.ref[s] = 0;
  }
  if (threadIdx.x == 0) {
    a.state[0] = (int32_t)n;
    a.state[1] = (int32_t)moved;
    a.info[0] = (int32_t)n;
    a.info[1] = (int32_t)moved;
    a.info[2] = 0;
  }
}

template <bool CONTIG>
__global__ void __launch_bounds__(kCopyT) compact_kernel(const CompactArgs a, int64_t rows_wg) {
  const PageBook& b = a.book;
  if (blockIdx.x < rows_wg) {
    const int64_t n = a.state[0];
    for (int64_t x = (int64_t)blockIdx.x * kCopyT + threadIdx.x; x < b.B * b.n_log; x += rows_wg * kCopyT) {
      const int64_t i = x / b.n_log, j = x - i * b.n_log;
      int32_t* e = &b.table[i * b.t_sb + j];
      const int32_t page = *e;
      if (page >= n && page < b.P) *e = a.to[page];
    }
    return;
  }
  copy_pages<CONTIG>(a.data, a.src, a.dst, a.state[1], blockIdx.x - rows_wg, gridDim.x - rows_wg);
}

// Workgroups for the table's entries and for the copies (at most pairs pairs).
int64_t entry_wgs(int64_t entries) {
  const int64_t n = (entries + kCopyT - 1) / kCopyT;
  return n < 1 ? 1 : (n > 256 ? 256 : n);
}
int64_t copy_wgs(const PageData& d, int64_t pairs) {
  const int64_t pieces = ((int64_t)d.n1 * d.n2 * d.row16 + kCopyPiece - 1) / kCopyPiece;
  const int64_t n = pairs * 2 * d.n_l * pieces;
  return n > 2048 ? 2048 : n;
}

}  // namespace

hipError_t launch_fork(const ForkArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kPT), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t rows = entry_wgs(a.n * a.book.n_log);
  const dim3 grid((unsigned)(rows + copy_wgs(a.data, a.n)));
  if (a.data.contiguous)
    hipLaunchKernelGGL(fork_kernel<true>, grid, dim3(kCopyT), 0, s, a, rows);
  else
    hipLaunchKernelGGL(fork_kernel<false>, grid, dim3(kCopyT), 0, s, a, rows);
  return hipGetLastError();
}

hipError_t launch_extend(const ExtendArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(extend_kernel, dim3(1), dim3(kPT), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_free(const FreeArgs& a, hipStream_t s) {
  const int64_t n = (a.n * a.book.n_log + 255) / 256;
  if (n <= 0) return hipSuccess;
  hipLaunchKernelGGL(free_kernel, dim3((unsigned)(n > 2048 ? 2048 : n)), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_compact(const CompactArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPT), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t rows = entry_wgs(a.book.B * a.book.n_log);
  const dim3 grid((unsigned)(rows + copy_wgs(a.data, a.book.P / 2)));
  if (a.data.contiguous)
    hipLaunchKernelGGL(compact_kernel<true>, grid, dim3(kCopyT), 0, s, a, rows);
  else
    hipLaunchKernelGGL(compact_kernel<false>, grid, dim3(kCopyT), 0, s, a, rows);
  return hipGetLastError();
}

}  // namespace dsv
