// dsv_window.h — launch arguments and key geometry of the windowed attention
// (dsv_window.hip, dsv_window_tile.hip).
#pragma once

#include <stdint.h>

#include "dsv_attn_geo.h"
#include "dsv_internal.h"

namespace dsv {

struct WinArgs {
  int dtype;                               // dsv_dtype of q, k, v
  const uint16_t* q;                       // (element strides; fp32 data too)
  int64_t q_sb, q_sm, q_sh;
  const uint16_t* k; int64_t k_sb, k_sp, k_sh, k_st;
  const uint16_t* v; int64_t v_sb, v_sp, v_sh, v_st;
  const void* pt; int pt_i64, ps_shift;    // page table (nullptr: dense)
  int64_t pt_sb, n_phys;
  const void* seqlens; int seqlens_i64;    // optional [B]
  int64_t n_keys;                          // keys of the cache (lengths are clamped to it)
  int B, M, H, Hk, G, R;                   // R = G * M rows per KV head, row m * G + g
  int W, S;                                // window (>= 1) and sinks, at most kWinMaxKeys
  float scale_log2;                        // log2(e) / sqrt(D)
  const void* parent; int par_i64;         // tree: [B, M] parents (nullptr: causal)
  int64_t par_sb, par_sm;
  int MW;                                  // tree: 64-bit words of a row's set
  int rows_per_block, n_rb, splits;
  float* opart;                            // [B, Hk, splits, R, D] (splits > 1), relative to the maximum
  float2* ml;                              // [B, Hk, splits, R] (maximum in log2 units, sum)
  void* out; int out_dtype, out_vec;       // out_vec: rows take vector stores
  int64_t o_sb, o_sm, o_sh;
  float* lse; int64_t l_sb, l_sm, l_sh;
};

// Keys of a sequence at most: token numbers, positions and their differences
// are 32-bit (byte offsets are not).
constexpr int64_t kWinMaxKeys = (int64_t)1 << 30;

// Bits [0, x) of a 32-bit word, x clamped to [0, 32].
DSV_HD uint32_t win_below(int x) { return x <= 0 ? 0u : (x >= 32 ? ~0u : (1u << x) - 1u); }

// The keys of a block of rows: [0, sink) and [lo, hi), as nt tiles of 32: nst
// tiles from key 0, the others from lo_al (a multiple of 32).  Where the two
// meet, nst is 0 and lo_al is 0.
struct WinKeys {
  int lo, hi, sink, lo_al;
  int nst, nt;
  DSV_HD int base(int t) const { return t < nst ? 32 * t : lo_al + 32 * (t - nst); }
  // Key n, or where no row sees it one that some row does: what is read in its
  // place (its own page may be gone).
  DSV_HD int read(int n) const {
    if (n < sink) return n;
    n = n > lo ? n : lo;
    return n < hi ? n : hi - 1;
  }
  // The tiles [first_whole(), end_whole()) hold only keys that some row sees (others
  // may): the window's.
  DSV_HD int first_whole() const { return nst + (lo > lo_al ? (lo - lo_al + 31) >> 5 : 0); }
  DSV_HD int end_whole() const { return nst + ((hi - lo_al) >> 5); }
  // The tiles [first_seen(), end_seen()) are seen whole by every row between
  // positions pmin and pmax (others may be).
  DSV_HD int first_seen(int pmax, int W) const {
    const int x = (pmax - W + 1 - lo_al + 31) >> 5;
    return nst + (x > 0 ? x : 0);
  }
  DSV_HD int end_seen(int pmin, int n0, bool tree) const { return nst + (((tree ? n0 : pmin + 1) - lo_al) >> 5); }
  // Is every key of the tile seen by every row between positions pmin and pmax?
  DSV_HD bool seen_by_all(int kb, int pmin, int pmax, int W, int S, int n0, bool tree) const {
    return (tree ? kb + 32 <= n0 : kb + 31 <= pmin) && (kb > pmax - W || kb + 32 <= S);
  }
};

// The keys of rows [r0, r0 + nrows) of a sequence whose new tokens start at n0.
DSV_HD WinKeys win_keys(int M, int G, int R, int W, int S, bool tree, int n0, int r0, int nrows) {
  WinKeys k;
  const int rl = (r0 + nrows < R ? r0 + nrows : R) - 1;
  // Positions of the first and last row; a tree's rows lie anywhere from n0 on.
  const int pmin = tree ? n0 : n0 + r0 / G, pmax = tree ? n0 + M - 1 : n0 + rl / G;
  k.hi = pmax + 1 > 0 ? pmax + 1 : 0;
  if (tree && n0 < 0) k.hi = 0;
  k.lo = pmin - W + 1;
  if (k.lo < 0) k.lo = 0;
  if (k.lo > k.hi) k.lo = k.hi;
  k.sink = S < k.hi ? S : k.hi;
  const int sink_al = (k.sink + 31) & ~31;
  k.lo_al = k.lo & ~31;
  k.nst = 0;
  if (k.lo_al > sink_al)
    k.nst = sink_al >> 5;
  else if (k.sink > 0)
    k.lo_al = 0;
  k.nt = k.nst + (k.hi > k.lo_al ? (k.hi - k.lo_al + 31) >> 5 : 0);
  return k;
}

// The kernel for many rows (rows_per_block 256, 16-bit, pages of at least 8 keys).
hipError_t launch_window_tile(const WinArgs& a, int D, hipStream_t s);
hipError_t launch_window(const WinArgs& a, int D, hipStream_t s);

}  // namespace dsv
