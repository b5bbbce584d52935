// dsv_latent_tile.hip — attention over keys and values expanded per head from the
// latent cache (prompts and chunks of them), bf16 and fp16, on gfx950.
//
// Mathematics: s = scale * (q[:dn] . kn_h + q[dn:] . kr), the second part of the key
// shared by the heads; out = sum softmax(s) v_h.  Per (row, key) 2 (2 dn + dr)
// operations, 3.4 times fewer than over the latent rows themselves at 512 + 64 and
// 128 + 64, against the expansion's own once per key: the form for many rows.
//
// A workgroup of 8 waves owns 256 rows of a head, each wave 32; tiles of 32 keys (key
// parts and values) go HBM -> LDS by LDS-DMA into a ring of four and feed all rows.
// Waves 0-3 issue the keys' DMA and waves 4-7 the values'; the two kinds meet the
// tile's barrier before and after their softmax, so that on each SIMD one wave's
// softmax runs on the VALU while the other's matrix products run (the schedule of
// dsv_window_tile.hip).  Sequences and their tiles are shared out evenly over the
// workgroups as in dsv_latent.hip.
//
// The running maximum may lag behind the true one: on tiles that all of a wave's rows
// see whole no maximum is taken, and a tile is redone with it where a lane's 16
// probabilities sum to more than kExpBound.  An exponent is one product and sum,
// s * scale - max * scale; where the second rounds to whole bits (2^21 and more), the
// difference is taken first.
//
// Registers: 256 a wave (two on a SIMD).  Tiles' addresses are uniform plus a lane's
// offset, the values' second half is read behind the barrier: nothing is spilled.
//
// Measured (a large bf16 product reaches 1309 TFLOP/s, fp16 1294): a prompt of 8192 tokens,
// 16 heads of 128 + 64, 344 GFLOP: 327-362 us by card, 0.95-1.05 PFLOP/s; the matrix units are
// busy in 48 % of the cycles of the counters' reference clock (the shader clock under this
// load was not measured, so their share of its own cycles is open).  Chunks of
// 1001 tokens of two sequences through 5000 to 12007 keys, 8 heads, fp16, 116 GFLOP: 132 us
// and 16 for joining the partials (33 MB of fp32 written and read).  No bank conflicts.

#include "dsv_dma.h"
#include "dsv_latent_dev.h"

namespace dsv {

namespace {

template <typename T>
constexpr float kExpTau = 8.0f;
template <>
constexpr float kExpTau<F16> = 5.0f;
template <typename T>
constexpr float kExpBound = 65536.f;
template <>
constexpr float kExpBound<F16> = 32768.f;

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

__device__ __forceinline__ float halves_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// x, computed again at every use: what is derived from it is not held in registers
// across the loop.
__device__ __forceinline__ uint32_t again(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Chunk c of key k stands at slot c ^ of these: operand reads without bank conflicts.
template <int CH>
__device__ __forceinline__ int kswz(int key) {
  return CH >= 16 ? key & 15 : CH == 8 ? (key >> 1) & 7 : (key >> 2) & 3;
}
template <int CH>
__device__ __forceinline__ int vswz(int key) {
  return ((key & 3) << 2) & (CH - 1);
}

template <bool B>
struct BoolC {
  static constexpr bool value = B;
};

template <int DN, int DR>
struct ExpLds {
  static constexpr int DV = DN;
  static constexpr int KN = 32 * DN * 2, KR = 32 * DR * 2, VT = 32 * DV * 2;
  static constexpr int STAGE = KN + KR + VT;
  uint8_t ring[4 * STAGE];
  uint32_t flag[8];
  LatSpan span;
};

template <typename T, int DN, int DR>
__global__ void __launch_bounds__(512, 2) expanded_kernel(const LatArgs a) {
  using L = ExpLds<DN, DR>;
  constexpr int DV = DN, KT = 1 << kLatTileExp;
  constexpr int KSN = DN / 16, KSR = DR / 16, DT = DV / 32;
  constexpr int CHN = DN / 8, CHR = DR / 8, CHV = DV / 8;
  constexpr int SHIFT = kProbShift<T, 10>;
  constexpr int IPN = DN / 64, IPV = DV / 64;      // DMA instructions per wave and tile
  constexpr int IPK = IPN + 1;
  static_assert(8 * 32 * DV * 2 <= 4 * L::STAGE, "the output rows are staged in the ring");
  __shared__ __attribute__((aligned(1024))) L lds;
  uint8_t* const ring = lds.ring;

  lat_touch_args();
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, lj = lane & 31, lg = lane >> 5;

  // Dispatch ids go round-robin over the 8 XCDs: give each a contiguous eighth of the
  // heads, whose row blocks share keys in that XCD's L2; the last row blocks, which see
  // most keys when causal, first.
  const int nblk = gridDim.x;
  int w = (nblk & 7) == 0 ? (int)(blockIdx.x & 7) * (nblk >> 3) + (int)(blockIdx.x >> 3) : (int)blockIdx.x;
  const int rj = w % a.W;
  w /= a.W;
  const int rb = a.n_rb - 1 - w % a.n_rb, kvh = w / a.n_rb;

  const LatEnd ends(a, rb);
  const int total = lat_line<512>(a, ends, kLatTileExp, rj, -1, lds.span);
  const LatCut cut(total, a.W);
  const int start = cut.begin(rj), stop = cut.begin(rj + 1);
  if (start >= stop) return;
  int b = __builtin_amdgcn_readfirstlane(lds.span.b);
  int tb = __builtin_amdgcn_readfirstlane(lds.span.off);

  const int row0 = rb * 256 + wid * 32;
  const bool wave_active = row0 < a.R;
  const int m_me = min(row0 + lj, a.R - 1);       // (one head per key head: a row is a position)
  const int m_lo = rb * 256;                      // of the block
  const bool v_wave = wid >= 4;
  const int w4 = wid & 3;
  const float scale = a.scale_log2;

  // Operand addresses within a stage.
  const uint32_t kofs = lj * (2 * DN) + ((lg ^ kswz<CHN>(lj)) << 4);
  const uint32_t rofs = L::KN + lj * (2 * DR) + ((lg ^ kswz<CHR>(lj)) << 4);
  uint32_t vofs;
  {
    const int bl = lane >> 4, bi = lane & 15;
    const int vkey = 4 * (bl >> 1) + (bi >> 2);
    const int vcol = 16 * (bl & 1) + 4 * (bi & 3);
    vofs = L::KN + L::KR + vkey * (2 * DV) + (((vcol >> 3) ^ vswz<CHV>(vkey)) << 4) + (vcol & 7) * 2;
  }

  // DMA: this wave's instructions of a tile and a lane's offsets in them.
  constexpr int KPN = 1024 / (2 * DN), KPR = 1024 / (2 * DR), NR = DR / 16;
  const int wr = w4 % NR;  // (two waves load the same rows where there are fewer instructions than waves)
  const int64_t nstep = 2 * (v_wave ? a.v.st : a.kn.st), rstep = 2 * a.kr.st;
  const bool near = nstep < (1 << 25) && rstep < (1 << 25);
  const uint32_t nst2 = (uint32_t)nstep, rst2 = (uint32_t)rstep;
  const uint32_t dst0 = lds_addr(ring) + (v_wave ? L::KN + L::KR : 0) + w4 * IPN * 1024, dst1 = lds_addr(ring) + L::KN + wr * 1024;
  uint32_t noff[IPN], roff;
#pragma unroll
  for (int x = 0; x < IPN; ++x) {
    const int k = (w4 * IPN + x) * KPN + lane / CHN;
    noff[x] = k * nst2 + (((lane % CHN) ^ (v_wave ? vswz<CHV>(k) : kswz<CHN>(k))) << 4);
  }
  {
    const int k = wr * KPR + lane / CHR;
    roff = k * rst2 + (((lane % CHR) ^ kswz<CHR>(k)) << 4);
  }

  for (int at = start; at < stop;) {
    const int len = __builtin_amdgcn_readfirstlane(len_of(a, b));
    const int tiles = ends.tiles(len, kLatTileExp);
    const int te = min(tiles, tb + (stop - at));
    LatPiece pc;
    pc.b = b;
    pc.len = len;
    pc.t0 = tb;
    pc.t1 = te;
    pc.slot = tb == 0 && te == tiles ? -1 : (((int64_t)kvh * a.n_rb + rb) * a.W + rj) * 2 + (at == start ? 0 : 1);
    const int end = ends(len);
    const int ntiles = end > 0 ? te - tb : 0;
    const int n0 = len - a.M;

    u32x4 qf[KSN + KSR];
    {
      const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + b * a.q_sb + (int64_t)m_me * a.q_sm + (int64_t)kvh * a.q_sh + lg * 8;
#pragma unroll
      for (int ks = 0; ks < KSN + KSR; ++ks) qf[ks] = *reinterpret_cast<const u32x4*>(qp + ks * 16);
    }

    // ---- DMA of a tile's keys (waves 0-3) or values (waves 4-7) ---------------------
    // Where rows see the whole tile, a uniform address plus the lane's offset; at the end of
    // the keys, the last one in the place of those behind it.
    const uint64_t nbase = (uint64_t)(v_wave ? a.v.p : a.kn.p) + 2 * (v_wave ? b * a.v.sb + kvh * a.v.sh : b * a.kn.sb + kvh * a.kn.sh);
    const uint64_t rbase = (uint64_t)a.kr.p + 2 * (b * a.kr.sb);
    auto issue_tile = [&](int t) {
      const int kb = (tb + t) * KT;
      const uint32_t st = (uint32_t)(t & 3) * L::STAGE;
      if (kb + KT <= end && near) {
        const uint64_t at = nbase + (uint64_t)(uint32_t)kb * nst2;
#pragma unroll
        for (int x = 0; x < IPN; ++x) dma_off(dst0 + st + x * 1024, at, noff[x]);
        if (!v_wave) dma_off(dst1 + st, rbase + (uint64_t)(uint32_t)kb * rst2, roff);
      } else {
        const int l = again(lane);
#pragma unroll 1
        for (int x = 0; x < IPN; ++x) {
          const int k = (w4 * IPN + x) * KPN + l / CHN;
          const int c = (l % CHN) ^ (v_wave ? vswz<CHV>(k) : kswz<CHN>(k));
          dma_lane<false>(dst0 + st + x * 1024, (const char*)nbase + min(kb + k, end - 1) * nstep + c * 16);
        }
        if (!v_wave) {
          const int k = wr * KPR + l / CHR;
          dma_lane<false>(dst1 + st, (const char*)rbase + min(kb + k, end - 1) * rstep + ((l % CHR) ^ kswz<CHR>(k)) * 16);
        }
      }
    };
    auto wait_one = [&]() { v_wave ? wait_vmcnt<IPV>() : wait_vmcnt<IPK>(); };

    f32x16 acc[DT];
    float mx = kNegInf, lsum = 0.f;
    // Probabilities are 2^(s * scale - ms + SHIFT), ms the maximum times the scale, rounded (with
    // the shift, too: far below zero their sum has a bit less): a row's sums share a factor
    // 2^-err, err = ms - mx * scale, which the end of the piece takes back.  Where that grows to bits (far), they are 2^((s - mx) * scale + SHIFT), an
    // instruction more each, and err is 0.
    float nms = (float)SHIFT, err = 0.f;
    bool far = false;
    uint32_t odd = 0;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16{};

    auto sync = [&](int k) {
      if (k + 2 < ntiles)
        wait_one();
      else
        wait_vmcnt<0>();
      barrier_lds();
      if (k + 3 < ntiles) issue_tile(k + 3);
    };

    f32x16 s_cur = f32x16{};
    // (Stages are multiples of 1 KiB: XORs within a row leave them alone.)
    auto read_k = [&](int t, int ks) {
      const uint32_t o = (uint32_t)(t & 3) * L::STAGE;
      return ks < KSN ? *reinterpret_cast<const u32x4*>(ring + ((kofs + o) ^ (ks << 5)))
                      : *reinterpret_cast<const u32x4*>(ring + ((rofs + o) ^ ((ks - KSN) << 5)));
    };
    auto read_vh = [&](int t, int hh, u32x4 (&vf)[DT]) {
      const uint32_t o = vofs + (uint32_t)(t & 3) * L::STAGE;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const uint8_t* p = ring + (o ^ (dt << 6)) + hh * 16 * (2 * DV);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * (2 * DV)));
        const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
        vf[dt] = u32x4{l2[0], l2[1], h2[0], h2[1]};
      }
    };

    // The keys that all of this wave's rows see: below `seen`.
    const int seen = a.causal ? n0 + row0 + 1 : len;
    // The last key that this lane's row sees.
    const int last = a.causal ? n0 + m_me : len - 1;

    auto step = [&](auto masked_c, int k) {
      constexpr bool MASKED = decltype(masked_c)::value;
      if (!v_wave && k > 0) sync(k);
      u32x4 kf[KSN], vf[DT];
      u32x4 pk[2];
#pragma unroll
      for (int ks = 0; ks < KSN; ++ks) kf[ks] = read_k(k + 1, ks);
      bool drops = false;
      if constexpr (MASKED) {
        const int kb = (tb + k) * KT;
        drops = kb + KT > seen;
        if (drops) {
#pragma unroll
          for (int v = 0; v < 16; ++v) s_cur[v] = kb + 8 * (v / 4) + 4 * lg + v % 4 <= last ? s_cur[v] : kNegInf;
        }
      }
      auto rescale = [&](float tau) {
        float mt = s_cur[0];
#pragma unroll
        for (int v = 1; v < 16; ++v) mt = fmaxf(mt, s_cur[v]);
        mt = halves_max(mt);
        if (__ballot((mt - mx) * scale > tau) != 0ull) {
          const float mn = fmaxf(mx, mt);
          float top = mn == kNegInf ? 0.f : mn * scale;
          asm("" : "+v"(top));  // (rounded here, not with the sum below)
          far = __ballot(fabsf(top) >= 2097152.f) != 0ull;
          nms = (float)SHIFT - top;
          const float ms = (float)SHIFT - nms;  // exact: what the shifted sum, rounded again, took off
          const float e = far || mn == kNegInf ? 0.f : fmaf(-mn, scale, ms);
          const float al = mn == kNegInf ? 1.f : __builtin_amdgcn_exp2f((mn == mx ? 0.f : (mx - mn) * scale) + (err - e));
          mx = mn;
          err = e;
          lsum *= al;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) acc[dt] *= al;
        }
      };
      if (MASKED && (drops || __ballot(mx == kNegInf) != 0ull)) rescale(kExpTau<T>);
      auto exps_of = [&](auto far_c) {
        constexpr bool FAR = decltype(far_c)::value;
        const float m0 = mx == kNegInf ? 0.f : mx;
        float ts = 0.f;
        auto p1 = [&](float x) { return __builtin_amdgcn_exp2f(FAR ? fmaf(x - m0, scale, (float)SHIFT) : fmaf(x, scale, nms)); };
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          uint32_t w4x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a0 = p1(s_cur[hh * 8 + 2 * e]), a1 = p1(s_cur[hh * 8 + 2 * e + 1]);
            w4x[e] = pack2<T>(a0, a1);
            ts += a0 + a1;
          }
          pk[hh] = u32x4{w4x[0], w4x[1], w4x[2], w4x[3]};
        }
        return ts;
      };
      auto exps = [&]() { return far ? exps_of(BoolC<true>{}) : exps_of(BoolC<false>{}); };
      float ts = exps();
      if (!drops && __ballot(!(ts <= kExpBound<T>)) != 0ull) {
        rescale(0.f);
        ts = exps();
      }
      lsum += ts;
      __builtin_amdgcn_sched_barrier(0);
      read_vh(k, 0, vf);
      if (v_wave) {
        // (The second half of the values after the barrier, while the products run: the
        // stage is overwritten a barrier later.)
        sync(k);
      }
      {
        f32x16 sn = f32x16{};
#pragma unroll
        for (int ks = 0; ks < KSN; ++ks) sn = mfma32<T>(kf[ks], qf[ks], sn);
        __builtin_amdgcn_sched_barrier(0);
        u32x4 vg[DT];
        read_vh(k, 1, vg);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] = mfma32<T>(vf[dt], pk[0], acc[dt]);
        __builtin_amdgcn_sched_barrier(0);
        u32x4 kr[KSR];
#pragma unroll
        for (int ks = 0; ks < KSR; ++ks) kr[ks] = read_k(k + 1, KSN + ks);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] = mfma32<T>(vg[dt], pk[1], acc[dt]);
        // (Behind the last tile these products are of an old one and not used.)
#pragma unroll
        for (int ks = 0; ks < KSR; ++ks) sn = mfma32<T>(kr[ks], qf[KSN + ks], sn);
        s_cur = sn;
        if (MASKED && drops) {
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int e = 0; e < 4; ++e) odd |= nonfinite2<T>(vf[dt][e]) | nonfinite2<T>(vg[dt][e]);
        }
      }
    };

    // ---- prologue: keys of tiles 0..2 and values of 0..1 issued, barrier 0, scores of 0 ----
    if (ntiles > 0) issue_tile(0);
    if (ntiles > 1) issue_tile(1);
    if (ntiles > 2 && !v_wave) issue_tile(2);
#pragma unroll
    for (int ks = 0; ks < KSN + KSR; ++ks) asm volatile("" ::"v"(qf[ks]));
    if (ntiles > 0) {
      if (v_wave ? ntiles > 1 : ntiles > 2)
        wait_one();
      else
        wait_vmcnt<0>();
      barrier_lds();
      if (v_wave) {
        if (ntiles > 2) issue_tile(2);
      } else {
        if (ntiles > 3) issue_tile(3);
      }
      if (wave_active) {
#pragma unroll
        for (int ks = 0; ks < KSN + KSR; ++ks) s_cur = mfma32<T>(read_k(0, ks), qf[ks], s_cur);
      }
    }
    if (wave_active) {
      const int k0 = min(1, ntiles);
      int k = 0;
      for (; k < k0; ++k) step(BoolC<true>{}, k);
      if (__ballot(mx == kNegInf) == 0ull) {
        const int k1 = min(ntiles, seen / KT - tb);
        for (; k < k1; ++k) step(BoolC<false>{}, k);
      }
      for (; k < ntiles; ++k) step(BoolC<true>{}, k);
    } else {
      for (int k = v_wave ? 0 : 1; k < ntiles; ++k) sync(k);
    }
    // Waves 0-3 meet the last barrier (waves 4-7 met it after their last softmax).
    if (ntiles > 0 && !v_wave) {
      wait_vmcnt<0>();
      barrier_lds();
    }

    // ---- the piece's results ---------------------------------------------------------
    __syncthreads();
    if (wave_active) {
      const float kBack = __builtin_amdgcn_exp2f(err - (float)SHIFT);
      const int row = row0 + lj;
      if (__ballot(odd != 0) != 0ull) {
        lat_exact_rows<T, DV>(lat_args(), pc, kvh, rb, KT, m_lo, nullptr, wid * 32, wid * 32 + 32, 1);
      } else {
        const float l = halves_sum(lsum) * kBack;
        // Value v of output tile dt is column 32 dt + 8 (v / 4) + 4 lg + v % 4.
        if (pc.slot >= 0) {
          if (row < a.R) {
            const int64_t prow = pc.slot * 256 + wid * 32 + lj;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int q4 = 0; q4 < 4; ++q4)
                *reinterpret_cast<f32x4*>(a.opart + prow * DV + 32 * dt + 8 * q4 + 4 * lg) =
                    f32x4{acc[dt][4 * q4], acc[dt][4 * q4 + 1], acc[dt][4 * q4 + 2], acc[dt][4 * q4 + 3]} * kBack;
            if (lg == 0) a.ml[prow] = make_float2(mx, l);
          }
        } else {
          const float inv = l > 0.f ? kBack / l : (l == 0.f ? 0.f : l);
          const int64_t off = b * a.o_sb + (int64_t)m_me * a.o_sm + (int64_t)kvh * a.o_sh;
          if (row < a.R) {
            if (lg == 0 && a.lse != nullptr) a.lse[b * a.l_sb + (int64_t)m_me * a.l_sm + (int64_t)kvh * a.l_sh] = lat_lse(a, mx, l);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int q4 = 0; q4 < 4; ++q4) {
                const float x[4] = {acc[dt][4 * q4] * inv, acc[dt][4 * q4 + 1] * inv, acc[dt][4 * q4 + 2] * inv, acc[dt][4 * q4 + 3] * inv};
                store4(a, off + 32 * dt + 8 * q4 + 4 * lg, x);
              }
          }
        }
      }
    }
    // Stores are done, and the ring is free, before the next piece's loads.
    wait_vmcnt<0>();
    __syncthreads();
    at += te - tb;
    tb = 0;
    ++b;
  }
}

template <typename T>
void launch_w(const LatArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.Hk * a.n_rb * a.W)), block(512);
  if (a.dn == 128) {
    if (a.dr == 64)
      hipLaunchKernelGGL((expanded_kernel<T, 128, 64>), grid, block, 0, s, a);
    else
      hipLaunchKernelGGL((expanded_kernel<T, 128, 32>), grid, block, 0, s, a);
  } else {
    if (a.dr == 64)
      hipLaunchKernelGGL((expanded_kernel<T, 64, 64>), grid, block, 0, s, a);
    else
      hipLaunchKernelGGL((expanded_kernel<T, 64, 32>), grid, block, 0, s, a);
  }
}

}  // namespace

bool expanded_widths(int dn, int dr) { return (dn == 64 || dn == 128) && (dr == 32 || dr == 64); }

hipError_t launch_latent_tile(const LatArgs& a, hipStream_t s) {
  a.dtype == 0 ? launch_w<BF16>(a, s) : launch_w<F16>(a, s);
  return hipGetLastError();
}

}  // namespace dsv
