// dsv_window_tile.hip — windowed attention for many rows (chunks of prompts,
// trees): the matrix-bound side of dsv_window.hip, whose mathematics and row
// packing it shares.
//
// A workgroup of 8 waves owns 256 rows of a KV head (256 / G positions, so the
// keys outside a row's window are few), each wave 32.  K and V tiles of 32 keys
// go HBM -> LDS by LDS-DMA into a ring of four tiles, and every tile feeds all
// 256 rows.  The schedule is that of dsv_attn.hip: waves 0-3 issue the K half of
// the DMA and waves 4-7 the V half, and on each SIMD one wave runs its softmax on
// the VALU while the other's MFMAs run.  Differences: the tiles are the sinks'
// and the window's (tile t -> key by WinKeys::base), rows and masks are the
// window's, addresses are 64-bit per lane, so a cache of any size and stride
// takes the one path, and pages of at least one DMA instruction's keys are
// resolved from a register window of 64 tiles.
//
// Bound by the matrix products and the softmax between them, about 1.0 us a tile
// of 256 rows and D = 128 with all CUs at work.  8192 rows through 4096 keys (32
// query heads, 8 key heads of 128, bf16): 504 to 536 us by card, 1.03 to 1.09
// PFLOP/s, 84 to 89% of what a large library product reaches (on one card 512, and
// 529 with the tests of each barrier's loads in the long loop).  Two trees of 64
// nodes through 8192 keys (one block of rows per key head, 16 splits): 39 us, of
// which the 16 tiles take 19, arguments, length, pages and first tile 7, the fp32
// partials 3 and the launch the rest; the merge follows with 8.

#include "dsv_attn_geo.h"
#include "dsv_dma.h"
#include "dsv_window_dev.h"

namespace dsv {

namespace {

// The running maximum used for the exponentials may lag the true one by kRescaleTau
// (log2 units) on masked tiles; unmasked ones are redone with the true one when a
// lane's 16 probabilities sum to more than kSumBound.  fp16 probabilities (times
// 2^10) stay below what the type holds either way: 2^(10 + 5) and kSumBound, and
// with the true maximum a lane sums to 2^14 at most, so nothing is redone twice.
template <typename T>
constexpr float kRescaleTau = 8.0f;
template <>
constexpr float kRescaleTau<F16> = 5.0f;
template <typename T>
constexpr float kSumBound = 65536.f;
template <>
constexpr float kSumBound<F16> = 32768.f;

template <typename T>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c);
template <>
__device__ __forceinline__ f32x16 mfma32<BF16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 mfma32<F16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ float xor32_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor32_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// A lane's 16 scores (NaN-propagating).
__device__ __forceinline__ float max16(const f32x16& s) {
  float m = __builtin_elementwise_maximum(s[0], s[1]);
#pragma unroll
  for (int v = 2; v < 16; ++v) m = __builtin_elementwise_maximum(m, s[v]);
  return m;
}

// x, computed again at every use: what is derived from it is not held in
// registers across the loop.
__device__ __forceinline__ int again(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

template <bool B>
struct BoolC {
  static constexpr bool value = B;
};

template <typename T, int D, bool PAGED>
__global__ void __launch_bounds__(512, 2) win_tile_kernel(const WinArgs a) {
  using G = Geo<D>;
  constexpr int NW = 8;
  constexpr int KS = D / 16;
  constexpr int DT = D / 32;
  constexpr int CH = G::CH;
  constexpr int SHIFT = kProbShift<T, 10>;
  constexpr int IPW = 2 * G::NINS / NW;  // DMA instructions per wave and tile
  static_assert(IPW * NW == 2 * G::NINS && G::NINS % IPW == 0, "K and V DMA halves map to wave halves");
  static_assert(G::STAGES == 4 && NW * 32 * D * 2 <= G::RING, "");
  // One LDS allocation, the DMA ring at its start (destinations below 64 KiB).
  __shared__ __attribute__((aligned(1024))) uint8_t smem[G::RING + sizeof(TreeLds<256>)];
  TreeLds<256>& tl = *reinterpret_cast<TreeLds<256>*>(smem + G::RING);

  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, lj = lane & 31, lg = lane >> 5;

  // Dispatch ids go round-robin over the 8 XCDs: give each a contiguous eighth,
  // so that the row blocks that share keys share an L2.
  const int nblk = gridDim.x;
  int w = (nblk & 7) == 0 ? (int)(blockIdx.x & 7) * (nblk >> 3) + (int)(blockIdx.x >> 3) : (int)blockIdx.x;
  const int rb = w % a.n_rb;
  w /= a.n_rb;
  const int split = w % a.splits;
  w /= a.splits;
  const int kvh = w % a.Hk, b = w / a.Hk;

  const bool tree = a.parent != nullptr;
  const int n0 = uniform(len_of(a, b) - a.M);
  const WinKeys kl = win_keys(a.M, a.G, a.R, a.W, a.S, tree, n0, rb * 256, 256);
  const int t_lo = (int)((int64_t)kl.nt * split / a.splits);
  const int ntiles = (int)((int64_t)kl.nt * (split + 1) / a.splits) - t_lo;

  // ---- this wave's rows: Q fragments (B operand of S^T = K . Q^T) ------------
  const int row0 = rb * 256 + wid * 32;
  const bool wave_active = row0 < a.R;
  const int r_me = row0 + lj;
  u32x4 qf[KS];
  int pos;
  {
    const Row row = row_of(a, min(r_me, a.R - 1));
    pos = n0 + row.m;
    const uint16_t* qp = a.q + b * a.q_sb + (int64_t)row.m * a.q_sm + (int64_t)(kvh * a.G + row.g) * a.q_sh + lg * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const u32x4*>(qp + ks * 16);
  }
  const TreeParents<512> parents(a, tree ? b : -1);

  // ---- DMA of one tile into its ring stage --------------------------------------
  // Instruction x of this wave covers keys [j*KPI, (j+1)*KPI) of the tile's K
  // (waves 0-3) or V half; lane p fills key j*KPI + p/CH, slot p%CH, which holds
  // global chunk slot ^ swizzle(key).  Tile t goes into stage t & 3.
  const bool v_wave = wid >= NW / 2;
  const int64_t st2 = 2 * (v_wave ? a.v_st : a.k_st), sp2 = 2 * (v_wave ? a.v_sp : a.k_sp);
  const char* hbase = reinterpret_cast<const char*>(v_wave ? a.v : a.k) +
                      2 * (v_wave ? b * a.v_sb + kvh * a.v_sh : b * a.k_sb + kvh * a.k_sh);
  const int j0 = uniform(wid % (NW / 2) * IPW);  // this wave's first instruction of its half
  const uint32_t dst0 = lds_addr(smem) + (uint32_t)uniform(v_wave ? G::TILE : 0) + (uint32_t)j0 * 1024;
  auto chunk_of = [&](int x, int l) {
    const int key_t = (j0 + x) * G::KPI + l / CH;
    return v_wave ? v_slot(CH, key_t, l % CH) : k_slot(CH, key_t, l % CH);
  };
  // In a tile that the block's rows see whole: a uniform 64-bit offset plus the
  // lane's 32-bit one (from the tile's first key; paged: from the instruction's).
  uint32_t lane_off[IPW];
#pragma unroll
  for (int x = 0; x < IPW; ++x)
    lane_off[x] = (uint32_t)(((PAGED ? 0 : (j0 + x) * G::KPI) + lane / CH) * st2) + (uint32_t)(chunk_of(x, lane) * 16);
  const uint32_t reach = (uint32_t)((PAGED ? G::KPI - 1 : 31) * st2) + 2 * D;
  // The tiles [whole0, whole1) are such (others may be: whole() tells).
  const int whole0 = kl.first_whole() - t_lo, whole1 = kl.end_whole() - t_lo;
  // Paged: lane l holds the offset of instruction x's keys in tile pgw_t0 + l.
  uint32_t pgw_lo[IPW], pgw_hi[IPW];
  int pgw_t0 = -64;
#pragma unroll
  for (int x = 0; x < IPW; ++x) pgw_lo[x] = pgw_hi[x] = 0;
  auto fill_pgw = [&](int t0) {
    pgw_t0 = t0;
#pragma unroll
    for (int x = 0; x < IPW; ++x) {
      const int n = kl.read(kl.base(t_lo + min(t0 + again(lane), ntiles - 1)) + (j0 + x) * G::KPI);
      const uint64_t o = (uint64_t)key_off(a, PAGED, sp2, st2, n, page_of(a, b, n));
      pgw_lo[x] = (uint32_t)o;
      pgw_hi[x] = (uint32_t)(o >> 32);
    }
  };
  auto issue_tile = [&](int t) {
    if (PAGED && t - pgw_t0 >= 64) fill_pgw(t);
    const uint32_t dst = dst0 + (uint32_t)(t & 3) * (2 * G::TILE);
    const int kb = kl.base(t_lo + t);
    if ((uint32_t)(t - whole0) < (uint32_t)(whole1 - whole0) && whole1 > whole0) {
#pragma unroll
      for (int x = 0; x < IPW; ++x) {
        int64_t off;
        if (PAGED)
          off = (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)pgw_hi[x], t - pgw_t0) << 32) |
                          (uint32_t)__builtin_amdgcn_readlane((int)pgw_lo[x], t - pgw_t0));
        else
          off = kb * st2;
        dma_rs<false>(dst + x * 1024, make_rsrc(hbase + off, reach), lane_off[x]);
      }
    } else {
      // At a border: a key that some row sees, through its own page.
#pragma unroll
      for (int x = 0; x < IPW; ++x) {
        const int l = again(lane);
        const int n = kl.read(kb + (j0 + x) * G::KPI + l / CH);
        dma_lane<false>(dst + x * 1024, hbase + key_off(a, PAGED, sp2, st2, n, PAGED ? page_of(a, b, n) : 0) + chunk_of(x, l) * 16);
      }
    }
  };

  f32x16 acc[DT];
  float mx = kNegInf, lsum = 0.f;
  uint32_t odd = 0;  // infinite or NaN entries of V in tiles that some row drops keys of, far scores
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16{};

  // Per-lane LDS offsets of the operand reads within a tile: K's of k-step ks is
  // kofs ^ (ks << 5) and V's of d tile dt is vofs ^ (dt << 6) (the swizzles are
  // XORs of whole chunks) plus the stage: one register each, so that the loop is
  // not unrolled over the ring and nothing spills.
  uint32_t kofs, vofs;
  {
    const int bl = lane >> 4, bi = lane & 15;
    const int vkey = 4 * (bl >> 1) + (bi >> 2);
    const int vcol = 16 * (bl & 1) + 4 * (bi & 3);
    kofs = lj * (2 * D) + k_slot(CH, lj, lg) * 16;
    vofs = vkey * (2 * D) + v_slot(CH, vkey, vcol >> 3) * 16 + (vcol & 7) * 2;
  }

  auto sync = [&](int k) {
    if (k + 2 < ntiles)
      wait_vmcnt<IPW>();
    else
      wait_vmcnt<0>();
    barrier_lds();
    if (k + 3 < ntiles) issue_tile(k + 3);
  };

  // The same in the long loop, where three tiles follow and the third is whole.
  int64_t next_off = 0;  // dense: that tile's offset
  auto sync_steady = [&](int k) {
    wait_vmcnt<IPW>();
    barrier_lds();
    const int t = k + 3;
    if (PAGED && t - pgw_t0 >= 64) fill_pgw(t);
    const uint32_t dst = dst0 + (uint32_t)(t & 3) * (2 * G::TILE);
#pragma unroll
    for (int x = 0; x < IPW; ++x) {
      int64_t off = next_off;
      if (PAGED)
        off = (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)pgw_hi[x], t - pgw_t0) << 32) |
                        (uint32_t)__builtin_amdgcn_readlane((int)pgw_lo[x], t - pgw_t0));
      dma_rs<false>(dst + x * 1024, make_rsrc(hbase + off, reach), lane_off[x]);
    }
    next_off += 32 * st2;
  };

  f32x16 s_cur = f32x16{};
  auto read_k = [&](int t, u32x4 (&kf)[KS]) {
    const uint32_t o = kofs + (uint32_t)(t & 3) * (2 * G::TILE);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kf[ks] = *reinterpret_cast<const u32x4*>(smem + (o ^ (ks << 5)));
  };
  // V^T operands of half hh (keys 16*hh .. 16*hh+15) of a tile.
  auto read_vh = [&](int t, int hh, u32x4 (&vf)[2][DT]) {
    const uint32_t o = vofs + (uint32_t)(t & 3) * (2 * G::TILE) + G::TILE;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const uint8_t* p = smem + (o ^ (dt << 6)) + hh * 16 * (2 * D);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * (2 * D)));
      const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
      vf[hh][dt] = u32x4{l2[0], l2[1], h2[0], h2[1]};
    }
  };
  const float scale_log2 = a.scale_log2;

  int pmin = pos, pmax = pos;  // of the wave's rows

  auto step = [&](auto masked_c, int k) {
    constexpr bool MASKED = decltype(masked_c)::value;
    if (!v_wave && (!MASKED || k > 0)) MASKED ? sync(k) : sync_steady(k);
    u32x4 kf[KS], vf[2][DT];
    u32x4 pk[2];
    {
      read_k(k + 1, kf);
      bool drops = false;
      if constexpr (MASKED) {
       const int kb = kl.base(t_lo + k);
       drops = !kl.seen_by_all(kb, pmin, pmax, a.W, a.S, n0, tree);
       if (drops) {
        const uint32_t keep = keep_word(a, tl.vis + (wid * 32 + (again(lane) & 31)) * kTreeMaxW, again(pos), kb, n0);
        // Bit v of a lane <-> key 8 * (v / 4) + 4 * lg + v % 4.
        const uint32_t vb = keep >> (again(lane) >> 5 << 2);
        const uint32_t kv = (vb & 0xFu) | ((vb >> 4) & 0xF0u) | ((vb >> 8) & 0xF00u) | ((vb >> 12) & 0xF000u);
#pragma unroll
        for (int v = 0; v < 16; ++v) s_cur[v] = ((kv >> v) & 1u) ? s_cur[v] : kNegInf;
       }
      }
      auto rescale = [&](float tau) {
        const float mt = xor32_max(max16(s_cur)) * scale_log2;
        if (__ballot(mt > mx + tau) != 0ull) {
          const float mn = __builtin_elementwise_maximum(mx, mt);
          const float al = (mn == mx) ? 1.f : __builtin_amdgcn_exp2f(mx - mn);
          mx = mn;
          odd |= far_score(mx) ? 1u : 0u;
          lsum *= al;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) acc[dt] *= al;
        }
      };
      if (MASKED && (drops || __ballot(mx == kNegInf) != 0ull)) rescale(kRescaleTau<T>);
      auto exps = [&](bool with_v) {
        const float ms = (mx == kNegInf) ? 0.f : mx - (float)SHIFT;
        float ts = 0.f;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          if (with_v) {
            __builtin_amdgcn_sched_barrier(0);
            read_vh(k, hh, vf);
            __builtin_amdgcn_sched_barrier(0);
          }
          uint32_t w4[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s_cur[hh * 8 + 2 * e], scale_log2, -ms));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(s_cur[hh * 8 + 2 * e + 1], scale_log2, -ms));
            w4[e] = pack2<T>(p0, p1);
            ts += p0 + p1;
          }
          pk[hh] = u32x4{w4[0], w4[1], w4[2], w4[3]};
        }
        return ts;
      };
      float ts = exps(true);
      if (!drops && __ballot(!(ts <= kSumBound<T>)) != 0ull) {
        rescale(0.f);
        ts = exps(false);
      }
      lsum += ts;
      if (MASKED && drops) {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) odd |= nonfinite2<T>(vf[hh][dt][e]);
      }
    }
    if (v_wave) MASKED ? sync(k) : sync_steady(k);
    {
      f32x16 sn = f32x16{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) sn = mfma32<T>(kf[ks], qf[ks], sn);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] = mfma32<T>(vf[hh][dt], pk[hh], acc[dt]);
      s_cur = sn;
    }
  };

  // ---- prologue: K(0..2) and V(0..1) issued, barrier 0, S(0) ---------------------
  if (ntiles > 0) issue_tile(0);
  if (ntiles > 1) issue_tile(1);
  if (ntiles > 2 && !v_wave) issue_tile(2);
  // The tree is walked while the first tiles come in.
  if (tree) {
    tree_rows<256, 512>(a, parents, n0, rb * 256, tl);
    pos = n0 + tl.depth[wid * 32 + lj];
  }
  pmin = pmax = pos;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    pmin = min(pmin, __shfl_xor(pmin, o));
    pmax = max(pmax, __shfl_xor(pmax, o));
  }
  pmin = uniform(pmin);
  pmax = uniform(pmax);
  // The tiles [seen0, seen1) are seen whole by every row of the wave (others may be).
  const int seen0 = kl.first_seen(pmax, a.W) - t_lo, seen1 = kl.end_seen(pmin, n0, tree) - t_lo;
  // The Q fragments and the score scale are complete before the loop: waits
  // placed at a first use inside it would wait for the DMA in flight there.
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" ::"v"(qf[ks]));
  asm volatile("" ::"s"(scale_log2));
  if (ntiles > 0) {
    if (v_wave ? ntiles > 1 : ntiles > 2)
      wait_vmcnt<IPW>();
    else
      wait_vmcnt<0>();
    barrier_lds();
    if (v_wave) {
      if (ntiles > 2) issue_tile(2);
    } else {
      if (ntiles > 3) issue_tile(3);
    }
    if (wave_active) {
      u32x4 kf[KS];
      read_k(0, kf);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s_cur = mfma32<T>(kf[ks], qf[ks], s_cur);
    }
  }
  if (wave_active) {
    // Three loops, so that the long one in the middle holds no mask and no first
    // maximum (one of its tiles comes before it; a row that then still has none,
    // all its scores -inf, keeps the wave out of it).  Unrolled: the accumulators
    // stay in place.
    const int k0 = min(max(seen0, 0) + 1, ntiles);
    int k = 0;
    for (; k < k0; ++k) step(BoolC<true>{}, k);
    if (__ballot(mx == kNegInf) == 0ull) {
      if (!PAGED) next_off = (int64_t)kl.base(t_lo + min(k + 3, ntiles - 1)) * st2;
      const int k1 = k + 3 >= whole0 ? min(seen1, min(whole1, ntiles) - 3) : 0;
      for (; k + 4 <= k1; k += 4) {
        step(BoolC<false>{}, k);
        step(BoolC<false>{}, k + 1);
        step(BoolC<false>{}, k + 2);
        step(BoolC<false>{}, k + 3);
      }
    }
    for (; k < ntiles; ++k) step(BoolC<true>{}, k);
  } else {
    // A wave without rows does its share of the DMA and meets the barriers.  (A
    // loop of its own: tests inside the other one cost 20 registers.)
    for (int k = v_wave ? 0 : 1; k < ntiles; ++k) sync(k);
  }
  // K waves meet the last barrier (V waves met it after the softmax of the last tile).
  if (ntiles > 0 && !v_wave) {
    wait_vmcnt<0>();
    barrier_lds();
  }

  // ---- epilogue -------------------------------------------------------------------
  __syncthreads();
  if (!wave_active) return;
  const WinArgs& z = args_again();
  // (Derived again, so that the loop keeps one register for all of them.)
  int tid_ep = threadIdx.x;
  asm volatile("" : "+v"(tid_ep));
  const int le = tid_ep & 63, lje = le & 31, lge = le >> 5;
  const int r_ep = row0 + lje;
  const bool rvalid = r_ep < z.R;
  if (__ballot(odd != 0) != 0ull) {
    exact_rows<T, D, 256>(&z, &tl, b, kvh, split, rb, t_lo, t_lo + ntiles, wid * 32, wid * 32 + 32, 1);
    return;
  }
  // (Sums as without the factor: by exact products.)
  constexpr float kBack = 1.f / (1 << SHIFT);
  const float ltot = xor32_sum(lsum) * kBack;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] *= kBack;
  const Row row = row_of(z, min(r_ep, z.R - 1));
  const int h = kvh * z.G + row.g;
  // Accumulator value v of d tile dt holds d = 32*dt + 8*(v/4) + 4*lge + v%4.
  if (z.splits > 1) {
    const int64_t pr = ((int64_t)(b * z.Hk + kvh) * z.splits + split) * z.R + r_ep;
    if (!rvalid) return;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *reinterpret_cast<f32x4*>(z.opart + pr * D + 32 * dt + 8 * q4 + 4 * lge) =
            f32x4{acc[dt][4 * q4], acc[dt][4 * q4 + 1], acc[dt][4 * q4 + 2], acc[dt][4 * q4 + 3]};
    if (lge == 0) z.ml[pr] = make_float2(mx, ltot);
    return;
  }
  const float inv = ltot > 0.f ? 1.f / ltot : (ltot == 0.f ? 0.f : ltot);
  const int64_t off = b * z.o_sb + (int64_t)row.m * z.o_sm + (int64_t)h * z.o_sh;
  if (rvalid && lge == 0 && z.lse != nullptr)
    z.lse[b * z.l_sb + (int64_t)row.m * z.l_sm + (int64_t)h * z.l_sh] = ltot == 0.f ? kNegInf : (mx + __log2f(ltot)) * kLn2;
  if (z.out_dtype == 2 || !z.out_vec) {
    if (!rvalid) return;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const float x[4] = {acc[dt][4 * q4] * inv, acc[dt][4 * q4 + 1] * inv, acc[dt][4 * q4 + 2] * inv, acc[dt][4 * q4 + 3] * inv};
        store_out(a, off + 32 * dt + 8 * q4 + 4 * lge, x);
      }
    return;
  }
  // Rows through the ring, so that a store instruction writes whole rows.
  constexpr int CHR = D / 8;
  uint8_t* stage = smem + wid * (32 * D * 2);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const float x0 = acc[dt][4 * q4] * inv, x1 = acc[dt][4 * q4 + 1] * inv, x2 = acc[dt][4 * q4 + 2] * inv, x3 = acc[dt][4 * q4 + 3] * inv;
      const u32x2 val = z.out_dtype == 0 ? u32x2{pack2<BF16>(x0, x1), pack2<BF16>(x2, x3)} : u32x2{pack2<F16>(x0, x1), pack2<F16>(x2, x3)};
      const int c = 4 * dt + q4;
      *reinterpret_cast<u32x2*>(stage + lje * (2 * D) + ((c ^ (lje % CHR)) * 16) + 8 * lge) = val;
    }
  wave_lds_fence();
#pragma unroll
  for (int k = 0; k < CHR / 2; ++k) {
    const int f = k * 64 + le, r = f / CHR, i = f % CHR;
    const u32x4 chunk = *reinterpret_cast<const u32x4*>(stage + r * (2 * D) + ((i ^ (r % CHR)) * 16));
    const int64_t o = __shfl((long long)off, r);
    if (row0 + r < z.R) *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(z.out) + o + i * 8) = chunk;
  }
}

template <typename T, int D>
hipError_t launch_t(const WinArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.B * a.Hk * a.n_rb * a.splits));
  if (a.pt != nullptr)
    hipLaunchKernelGGL((win_tile_kernel<T, D, true>), grid, dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL((win_tile_kernel<T, D, false>), grid, dim3(512), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_window_tile(const WinArgs& a, int D, hipStream_t s) {
  if (a.dtype == 0) return D == 64 ? launch_t<BF16, 64>(a, s) : launch_t<BF16, 128>(a, s);
  return D == 64 ? launch_t<F16, 64>(a, s) : launch_t<F16, 128>(a, s);
}

}  // namespace dsv
