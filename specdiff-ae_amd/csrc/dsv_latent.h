// dsv_latent.h — launch arguments and work sharing of the latent attention
// (dsv_latent.hip, dsv_latent_tile.hip, dsv_latent_f32.hip).
#pragma once

#include <stdint.h>

#include "dsv_attn_geo.h"
#include "dsv_internal.h"

namespace dsv {

// One of the key or value arrays: element (b, h, n) at p + b*sb + h*sh + n*st, or,
// in a page pool, page*sp + (n mod page size)*st (element strides).
struct LatSrc {
  const void* p;
  int64_t sb, sp, sh, st;
};

struct LatArgs {
  int dtype;                               // dsv_dtype of q, keys and values
  int dn, dr, dv;                          // widths: keys without their rotated part, that part, values
  const void* q;
  int64_t q_sb, q_sm, q_sh;
  LatSrc kn, kr, v;
  const void* pt; int pt_i64, ps_shift;    // page table (nullptr: dense)
  int64_t pt_sb, n_phys;
  const void* seqlens; int seqlens_i64;    // optional [B]
  int64_t n_keys;                          // keys of the cache (lengths are clamped to it)
  int B, M, H, Hk, G, R;                   // R = G * M rows per key head, row m * G + g
  int causal;
  float scale_log2;                        // log2(e) * softmax scale
  const void* parent; int par_i64;         // tree: [B, M] parents (nullptr: none)
  int64_t par_sb, par_sm;
  int MW;                                  // tree: 64-bit words of a row's set
  int rpb, n_rb, W;                        // rows per block, blocks, ranges (see LatCut)
  float* opart;                            // [Hk, n_rb, W, 2, rpb, dv], relative to the maximum
  float2* ml;                              // [Hk, n_rb, W, 2, rpb] (maximum as a score, sum)
  void* out; int out_dtype, out_vec;       // out_vec: rows take vector stores
  int64_t o_sb, o_sm, o_sh;
  float* lse; int64_t l_sb, l_sm, l_sh;
};

// Keys of a sequence at most (token numbers are 32-bit, byte offsets are not).
constexpr int64_t kLatMaxKeys = (int64_t)1 << 30;

// Keys [0, end(len)) of a sequence are those that some row of a block sees; in tiles of
// 2^sh, at least one, so that every sequence's rows are somebody's.
struct LatEnd {
  int off, least;   // end = len + off, none below `least` tokens
  DSV_HD LatEnd(const LatArgs& a, int rb) {
    const int rl = ((rb + 1) * a.rpb < a.R ? (rb + 1) * a.rpb : a.R) - 1;
    off = a.causal && a.parent == nullptr ? rl / a.G + 1 - a.M : 0;
    least = a.parent != nullptr ? a.M : -off;
  }
  DSV_HD int operator()(int len) const { return len >= least ? len + off : 0; }
  DSV_HD int tiles(int len, int sh) const {
    const int t = (operator()(len) + (1 << sh) - 1) >> sh;
    return t > 0 ? t : 1;
  }
};

// Work sharing.  For each unit (key head, block of rows) the sequences' tiles
// stand in one line, which W workgroups share out evenly: the first total % W ranges
// hold a tile more than the others.  A range holds pieces of one or more sequences.
// Where a piece is all of its sequence's tiles the workgroup writes the output, else a
// partial: number 0 for the piece that the range begins with, 1 for another, which its
// end cuts (so at most two per range).  The line is below 2^31 tiles.
struct LatCut {
  int q, r;  // total / W, total % W
  DSV_HD LatCut(int total, int W) : q(total / W), r(total - q * W) {}
  DSV_HD int begin(int j) const { return j * q + (j < r ? j : r); }
  DSV_HD int range_of(int tile) const {
    const int head = r * (q + 1);
    return tile < head ? tile / (q + 1) : r + (tile - head) / q;
  }
};

// Shapes that the kernels are built for.
bool latent_widths(int dc, int dr);
bool expanded_widths(int dn, int dr);

hipError_t launch_latent(const LatArgs& a, hipStream_t s);
hipError_t launch_latent_tile(const LatArgs& a, hipStream_t s);
hipError_t launch_latent_f32(const LatArgs& a, hipStream_t s);
hipError_t launch_latent_merge(const LatArgs& a, int sh, hipStream_t s);

// Keys per tile of the three kernels, as powers of two.
constexpr int kLatTile = 6, kLatTileExp = 5, kLatTileF32 = 6;

}  // namespace dsv
