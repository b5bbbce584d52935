// dsv_latent.hip — attention over a cache of one latent vector per token (absorbed
// form), bf16 and fp16, on gfx950.
//
// Mathematics.  A token's cache row x (dc + dr wide) is the key of every head, and
// its first dc entries are the value of every head: s = scale * q . x, out = sum
// softmax(s) x[:dc].  The M new tokens of a sequence stand at the end of its cache;
// row m sees the keys up to its own position, or, of a drafted tree, its ancestors
// and itself.
//
// All heads share the keys, so the rows of a sequence (m, h) are packed, row m * H +
// h, in blocks of 16, 32 or 64; a tile of 64 cache rows comes into LDS once and
// serves both products.  Of a tile, wave w of four computes the scores of keys
// [16w, 16w + 16) for all rows (S^T = X . Q^T, the queries in registers), and, of the
// output, the columns [w dc / 4, (w + 1) dc / 4) for all rows and keys (O^T = X^T . P^T);
// the probabilities go between them through LDS.  So each wave reads every cache
// row's quarter once as a key and once as a value: 64 rows a workgroup read 22 bytes
// of LDS per key and 64 flops.  That decides the split: waves that own rows instead
// would each read the whole tile twice.
//
// The running maximum is common to the waves and may lag behind the true one by
// kLatTau (log2 units); a wave whose scores exceed it raises a flag beside its
// probabilities, and only then do the waves exchange maxima and rescale.  The
// exponent is (s - max) * scale, a difference of scores, so that it holds for scores
// of any size.  Scores, sums and maxima are fp32; probabilities are rounded to the
// cache's type for the second product (half a step of each; fp16 holds them times
// 2^10, see kProbShift); their sum takes them unrounded.
//
// Tiles go HBM -> LDS by LDS-DMA into two buffers; the next tile's loads are issued
// before the present one's are waited for, so that the memory is never idle.
// Sequences and their tiles are shared out evenly over the workgroups (LatRange),
// whatever their lengths; latent_merge_kernel joins the partials.

#include "dsv_dma.h"
#include "dsv_latent_dev.h"

namespace dsv {

namespace {

template <typename T>
constexpr float kLatTau = 8.0f;
template <>
constexpr float kLatTau<F16> = 5.0f;

template <typename T>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mfma16<BF16>(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mfma16<F16>(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ float groups_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float groups_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// x, computed again at every use: what is derived from it is not held in registers
// across the loop.
__device__ __forceinline__ uint32_t again(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// LDS image of a tile: the rows' first dc entries, then their last dr.  Chunk c (16
// bytes) of key k stands at slot c ^ swz(k): 16 keys read at one chunk (scores) and
// four keys read at two neighbouring chunks (values, transposed) fall on distinct
// banks.
__device__ __forceinline__ int swz_n(int key) { return ((key & 7) << 1) | ((key >> 3) & 1); }
template <int DR>
__device__ __forceinline__ int swz_r(int key) {
  return DR == 64 ? (key >> 1) & 7 : (key >> 2) & 3;
}

template <int DC, int DR, int ROWS>
struct LatLds {
  static constexpr int KT = kLatTile;
  static constexpr int NB = DC * 2, RB = DR * 2;
  static constexpr int TILE = KT * (NB + RB);
  // Sets of tree keys: a block's rows of H heads belong to at most ROWS nodes, of
  // H >= 2 heads to ROWS / 2 + 1 (lat_block).
  static constexpr int VIS = 36 * (kTreeMaxM / 64) * 8;
  uint8_t ring[2 * TILE];
  uint8_t p[ROWS * KT * 2];
  uint64_t vis[VIS / 8];
  float red[4][ROWS];
  uint32_t flag[4];
  LatSpan span;
};

template <typename T, int DC, int DR, int ROWS>
__global__ void __launch_bounds__(256, 1) latent_kernel(const LatArgs a) {
  using L = LatLds<DC, DR, ROWS>;
  // Scores: KG groups of KB x 16 keys, RG groups of QR x 16 rows, a wave each.
  constexpr int RG = ROWS == 64 ? 2 : 1, KG = 4 / RG, KB = 4 / KG, QR = ROWS / 16 / RG;
  constexpr int KT = L::KT, RB = ROWS / 16, KSN = DC / 32, KSR = DR / 32, KS = KSN + KSR;
  constexpr int CB = DC / 64;              // blocks of 16 output columns per wave
  constexpr int SHIFT = kProbShift<T, 10>;
  constexpr int KPI = 1024 / L::NB;        // keys per DMA instruction of the first part
  constexpr int IPN = 16 / KPI;            // such instructions per wave and tile
  static_assert(KPI <= 2, "");
  constexpr int KPR = 1024 / L::RB;        // the same of the second part
  constexpr int IPR = 16 * L::RB / 1024;
  static_assert(L::TILE % 1024 == 0, "XORs within a row leave the buffer alone");
  static_assert(sizeof(L) <= 163840, "LDS of a CU");
  static_assert(2 * kTreeMaxM <= ROWS * KT * 2, "the parents are staged in p");
  __shared__ __attribute__((aligned(1024))) L lds;

  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;

  // Dispatch ids go round-robin over the 8 XCDs: give each a contiguous eighth, so
  // that the row blocks of a range, which read the same keys, share an L2.
  const int nblk = gridDim.x;
  const int w = (nblk & 7) == 0 ? (int)(blockIdx.x & 7) * (nblk >> 3) + (int)(blockIdx.x >> 3) : (int)blockIdx.x;
  const int rb = w % a.n_rb, rj = w / a.n_rb;

  lat_line<256>(a, rb, KT, rj, -1, lds.span);
  const int64_t total = lds.span.total;
  const int64_t start = lat_cut(total, rj, a.W), stop = lat_cut(total, rj + 1, a.W);
  int b = __builtin_amdgcn_readfirstlane(lds.span.b);
  int t0 = __builtin_amdgcn_readfirstlane(lds.span.off);
  if (start >= stop) return;

  const int m_lo = rb * ROWS / a.G, m_hi = (min((rb + 1) * ROWS, a.R) - 1) / a.G;
  // Operand addresses within a tile (the swizzles are XORs of whole chunks).
  const int kg = wid % KG, rg = wid / KG;
  const uint32_t qofs = li * L::NB + ((lg ^ swz_n(li)) << 4);
  const uint32_t qrofs = KT * L::NB + li * L::RB + ((lg ^ swz_r<DR>(li)) << 4);
  const uint32_t kofs = kg * KB * 16 * L::NB + qofs, rofs = kg * KB * 16 * L::RB + qrofs;
  const int vkey = 4 * lg + (li >> 2);
  const uint32_t vofs = vkey * L::NB + (((wid * (DC / 32) + ((li & 3) >> 1)) ^ swz_n(vkey)) << 4) + (li & 1) * 8;
  // Probabilities: of 32 keys, lane group g holds 4g .. 4g + 3 and 16 + 4g .. 16 + 4g + 3 as
  // one chunk, which is the order in which the values are read.
  const uint32_t pw = rg * QR * 2048 + li * 128 + (((kg * KB >> 1) * 4 + lg) ^ (li >> 1)) * 16 + (KB == 1 ? (kg & 1) * 8 : 0);
  const uint32_t pr = li * 128 + ((lg ^ (li >> 1)) << 4);
  const uint32_t ring0 = lds_addr(lds.ring);
  const float scale = a.scale_log2;

  for (int64_t at = start; at < stop;) {
    const int len = __builtin_amdgcn_readfirstlane(len_of(a, b));
    const int tiles = lat_tiles(a, len, rb, KT);
    const int t1 = (int)min((int64_t)tiles, t0 + (stop - at));
    LatPiece pc;
    pc.b = b;
    pc.len = len;
    pc.t0 = t0;
    pc.t1 = t1;
    pc.slot = t0 == 0 && t1 == tiles ? -1 : ((int64_t)rb * a.W + rj) * 2 + (at == start ? 0 : 1);
    const int end = lat_end(a, len, rb);
    const char* base = reinterpret_cast<const char*>(a.kn.p) + 2 * (b * a.kn.sb);

    if (a.parent != nullptr) lat_tree<256>(a, b, m_lo, m_hi - m_lo + 1, reinterpret_cast<int16_t*>(lds.p), lds.vis);

    // ---- DMA of 16 rows of this wave into a buffer: lane l knows row l % 16 ----------
    auto issue_rows = [&](int buf, const char* src, int64_t off) {
      const uint32_t dst = ring0 + (uint32_t)buf * L::TILE + wid * 16 * L::NB;
      const int lo = (int)(uint32_t)off, hi = (int)(off >> 32);
      const uint32_t ln = again(lane);
      auto row = [&](int k) {
        return src + (((int64_t)__builtin_amdgcn_readlane(hi, k) << 32) | (uint32_t)__builtin_amdgcn_readlane(lo, k));
      };
      // (One instruction's address at a time: the registers are full.)
#pragma unroll
      for (int x = 0; x < IPN; ++x) {
        if constexpr (KPI == 1) {
          dma_off<false>(dst + x * 1024, row(x), (ln ^ swz_n(x)) << 4);
        } else {
          const int k = 2 * x + (lane >> 5);
          const char* r = lane < 32 ? row(2 * x) : row(2 * x + 1);
          dma_lane<false>(dst + x * 1024, r + (((lane & 31) ^ swz_n(k)) << 4));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      const uint32_t dst2 = ring0 + (uint32_t)buf * L::TILE + KT * L::NB + wid * 16 * L::RB;
#pragma unroll
      for (int x = 0; x < IPR; ++x) {
        const int k = x * KPR + lane / (64 / KPR);
        const int64_t o = __shfl((long long)off, k);
        dma_lane<false>(dst2 + x * 1024, src + o + L::NB + (((lane % (64 / KPR)) ^ swz_r<DR>(k)) << 4));
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // A tile's keys; those at or behind the end are replaced by the last one (no row
    // sees them).
    auto issue = [&](int t) {
      const int n = min(t * KT + wid * 16 + li, end - 1);
      issue_rows(t & 1, base, 2 * key_off(a, a.kn, n, a.pt != nullptr ? page_of(a, b, n) : 0));
    };

    u32x4 qf[QR][KS];
    f32x4 acc[RB][CB];
    float mx[RB], ls[QR];
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      mx[i] = kNegInf;
#pragma unroll
      for (int c = 0; c < CB; ++c) acc[i][c] = f32x4{};
    }
#pragma unroll
    for (int i = 0; i < QR; ++i) ls[i] = 0.f;
    uint32_t odd = 0;
    if (end > 0) {
      issue(t0);
      // The queries come through the other buffer (a load that ends in registers would
      // be waited for at its first use, in the loop, and the tiles in flight with it).
      if (wid * 16 < ROWS) {
        const int r = min(rb * ROWS + wid * 16 + li, a.R - 1), m = r / a.G;
        issue_rows((t0 + 1) & 1, reinterpret_cast<const char*>(a.q), 2 * (b * a.q_sb + (int64_t)m * a.q_sm + (int64_t)(r - m * a.G) * a.q_sh));
      }
      wait_vmcnt<0>();
      barrier_lds();
      const uint8_t* qt = lds.ring + ((t0 + 1) & 1) * L::TILE;
#pragma unroll
      for (int i = 0; i < QR; ++i)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          qf[i][ks] = ks < KSN ? *reinterpret_cast<const u32x4*>(qt + (rg * QR + i) * 16 * L::NB + (qofs ^ (ks << 6)))
                               : *reinterpret_cast<const u32x4*>(qt + (rg * QR + i) * 16 * L::RB + (qrofs ^ ((ks - KSN) << 6)));
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      for (int t = t0; t < t1; ++t) {
        // The other buffer is free once every wave is done with tile t - 1.
        barrier_lds();
        if (t + 1 < t1) {
          issue(t + 1);
          wait_vmcnt<IPN + IPR>();
        } else {
          wait_vmcnt<0>();
        }
        // (Waves that share keys wait for each other's loads.)
        if constexpr (KB > 1) barrier_lds();
        asm volatile("" ::: "memory");
        const uint32_t stage = (uint32_t)(t & 1) * L::TILE;
        // ---- scores of this wave's keys and rows ----------------------------------------
        f32x4 s[QR][KB];
#pragma unroll
        for (int i = 0; i < QR; ++i)
#pragma unroll
          for (int k = 0; k < KB; ++k) s[i][k] = f32x4{};
        const uint32_t ko = again(kofs) + stage, ro = again(rofs) + stage;
        auto read_k = [&](int x) {
          const int ks = x / KB, k = x % KB;
          return ks < KSN ? *reinterpret_cast<const u32x4*>(lds.ring + (ko ^ (ks << 6)) + k * 16 * L::NB)
                          : *reinterpret_cast<const u32x4*>(lds.ring + (ro ^ ((ks - KSN) << 6)) + k * 16 * L::RB);
        };
        u32x4 kf[4];
#pragma unroll
        for (int x = 0; x < 3; ++x) kf[x] = read_k(x);
#pragma unroll
        for (int x = 0; x < KS * KB; ++x) {
          if (x + 3 < KS * KB) kf[(x + 3) % 4] = read_k(x + 3);
#pragma unroll
          for (int i = 0; i < QR; ++i) s[i][x % KB] = mfma16<T>(kf[x % 4], qf[i][x / KB], s[i][x % KB]);
          __builtin_amdgcn_sched_barrier(0);
        }
        const int kb = t * KT;
        const bool whole = lat_whole(a, len, m_lo, kb, KT);
        if (!whole) {
          // (Loops, so that it costs no registers.)
          uint32_t keep = 0;
#pragma unroll 1
          for (int i = 0; i < QR; ++i) {
            const int m = min(rb * ROWS + (rg * QR + i) * 16 + li, a.R - 1) / a.G;
#pragma unroll 1
            for (int v = 0; v < 4 * KB; ++v)
              keep |= (lat_sees(a, len, m, lds.vis + (m - m_lo) * a.MW, kb + (kg * KB + v / 4) * 16 + 4 * lg + v % 4) ? 1u : 0u)
                      << (4 * KB * i + v);
          }
#pragma unroll
          for (int i = 0; i < QR; ++i)
#pragma unroll
            for (int v = 0; v < 4 * KB; ++v) s[i][v / 4][v % 4] = ((keep >> (4 * KB * i + v)) & 1u) ? s[i][v / 4][v % 4] : kNegInf;
        }
        // ---- probabilities, relative to the maximum so far ------------------------------
        float ps[QR];
        auto top = [&](int i) {
          float m = fmaxf(fmaxf(s[i][0][0], s[i][0][1]), fmaxf(s[i][0][2], s[i][0][3]));
          if constexpr (KB > 1) m = fmaxf(m, fmaxf(fmaxf(s[i][KB - 1][0], s[i][KB - 1][1]), fmaxf(s[i][KB - 1][2], s[i][KB - 1][3])));
          return m;
        };
        auto max_of = [&](int i) { return RG > 1 && rg != 0 ? mx[QR * (RG - 1) + i] : mx[i]; };
        auto probs = [&]() {
#pragma unroll
          for (int i = 0; i < QR; ++i) {
            const float m = max_of(i), m0 = m == kNegInf ? 0.f : m;
            float p[4 * KB], sum = 0.f;
            uint32_t w2[2 * KB];
#pragma unroll
            for (int v = 0; v < 4 * KB; ++v) {
              p[v] = __builtin_amdgcn_exp2f(fmaf(s[i][v / 4][v % 4] - m0, scale, (float)SHIFT));
              sum += p[v];
            }
#pragma unroll
            for (int v = 0; v < 2 * KB; ++v) w2[v] = pack2<T>(p[2 * v], p[2 * v + 1]);
            ps[i] = sum;
            if constexpr (KB == 1)
              *reinterpret_cast<u32x2*>(lds.p + i * 2048 + pw) = u32x2{w2[0], w2[1]};
            else
              *reinterpret_cast<u32x4*>(lds.p + i * 2048 + pw) = u32x4{w2[0], w2[1], w2[2 * KB - 2], w2[2 * KB - 1]};
          }
        };
        bool over = false;
#pragma unroll
        for (int i = 0; i < QR; ++i) over |= (top(i) - max_of(i)) * scale > kLatTau<T>;
        probs();
        if (lane == 0) lds.flag[wid] = 0;
        if (__ballot(over) != 0ull && lane == 0) lds.flag[wid] = 1;
        barrier_after_lds();
        const u32x4 fl = *reinterpret_cast<const u32x4*>(lds.flag);
        if (__builtin_amdgcn_readfirstlane(fl[0] | fl[1] | fl[2] | fl[3]) != 0) {
#pragma unroll
          for (int i = 0; i < QR; ++i) {
            const float m = groups_max(top(i));
            if (lg == 0) lds.red[kg][(rg * QR + i) * 16 + li] = m;
          }
          barrier_after_lds();
#pragma unroll
          for (int i = 0; i < RB; ++i) {
            float mn = mx[i];
#pragma unroll
            for (int k = 0; k < KG; ++k) mn = fmaxf(mn, lds.red[k][i * 16 + li]);
            const float al = mn == mx[i] ? 1.f : __builtin_amdgcn_exp2f((mx[i] - mn) * scale);
            mx[i] = mn;
            if (i / QR == rg) ls[i % QR] *= al;
#pragma unroll
            for (int c = 0; c < CB; ++c) acc[i][c] *= al;
          }
          probs();
          barrier_after_lds();
        }
#pragma unroll
        for (int i = 0; i < QR; ++i) ls[i] += ps[i];
        // ---- this wave's columns -------------------------------------------------------
        u32x4 pf[2][RB], vf[3];
        const uint32_t vo = again(vofs) + stage;
        auto read_p = [&](int k2) {
#pragma unroll
          for (int i = 0; i < RB; ++i) pf[k2][i] = *reinterpret_cast<const u32x4*>(lds.p + i * 2048 + (pr ^ (k2 << 6)));
        };
        auto read_v = [&](int x) {
          const uint8_t* vp = lds.ring + (vo ^ ((x % CB) << 5)) + x / CB * 32 * L::NB;
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)vp);
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vp + 16 * L::NB));
          const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
          return u32x4{l2[0], l2[1], h2[0], h2[1]};
        };
        read_p(0);
        vf[0] = read_v(0);
        vf[1] = read_v(1);
#pragma unroll
        for (int x = 0; x < 2 * CB; ++x) {
          if (x == CB - 2) read_p(1);
          if (x + 2 < 2 * CB) vf[(x + 2) % 3] = read_v(x + 2);
          const u32x4 v = vf[x % 3];
          if (!whole && m_hi > m_lo) odd |= nonfinite2<T>(v[0]) | nonfinite2<T>(v[1]) | nonfinite2<T>(v[2]) | nonfinite2<T>(v[3]);
#pragma unroll
          for (int i = 0; i < RB; ++i) acc[i][x % CB] = mfma16<T>(v, pf[x / CB][i], acc[i][x % CB]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }

    // ---- the piece's results ---------------------------------------------------------
    constexpr float kBack = 1.f / (1 << SHIFT);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < QR; ++i) {
      const float x = groups_sum(ls[i]);
      if (lg == 0) lds.red[kg][(rg * QR + i) * 16 + li] = x;
    }
    if (lane == 0) lds.flag[wid] = 0;
    if (__ballot(odd != 0) != 0ull && lane == 0) lds.flag[wid] = 1;
    __syncthreads();
    const u32x4 fl = *reinterpret_cast<const u32x4*>(lds.flag);
    if (__builtin_amdgcn_readfirstlane(fl[0] | fl[1] | fl[2] | fl[3]) != 0) {
      lat_exact_rows<T, DC>(lat_args(), pc, 0, rb, KT, m_lo, lds.vis, wid, ROWS, 4);
    } else {
#pragma unroll
      for (int i = 0; i < RB; ++i) {
        const int r = i * 16 + li, row = rb * ROWS + r;
        float l = 0.f;
#pragma unroll
        for (int k = 0; k < KG; ++k) l += lds.red[k][r];
        l *= kBack;
        if (row >= a.R) continue;
        if (pc.slot >= 0) {
          const int64_t prow = pc.slot * ROWS + r;
#pragma unroll
          for (int c = 0; c < CB; ++c)
            *reinterpret_cast<f32x4*>(a.opart + prow * DC + wid * (DC / 4) + c * 16 + lg * 4) = acc[i][c] * kBack;
          if (wid == 0 && lg == 0) a.ml[prow] = make_float2(mx[i], l);
          continue;
        }
        const float inv = l > 0.f ? kBack / l : (l == 0.f ? 0.f : l);
        const int m = row / a.G, h = row - m * a.G;
        const int64_t off = b * a.o_sb + (int64_t)m * a.o_sm + (int64_t)h * a.o_sh + wid * (DC / 4) + lg * 4;
#pragma unroll
        for (int c = 0; c < CB; ++c) {
          const float x[4] = {acc[i][c][0] * inv, acc[i][c][1] * inv, acc[i][c][2] * inv, acc[i][c][3] * inv};
          store4(a, off + c * 16, x);
        }
        if (wid == 0 && lg == 0 && a.lse != nullptr)
          a.lse[b * a.l_sb + (int64_t)m * a.l_sm + (int64_t)h * a.l_sh] = lat_lse(a, mx[i], l);
      }
    }
    // Stores are done before the next piece counts its loads.
    wait_vmcnt<0>();
    __syncthreads();
    at += t1 - t0;
    t0 = 0;
    ++b;
  }
}

// ---- the partials joined -------------------------------------------------------------
// A workgroup takes (sequence, unit, 4 rows) at a time: 64 lanes a row, DV / 64 columns
// each.
template <int DV>
__device__ __forceinline__ void merge_rows(const LatArgs& a, int kt, int64_t x, LatSpan& span) {
  constexpr int N = DV / 64;
  const int parts = a.rpb / 4;
  const int part = (int)(x % parts);
  x /= parts;
  const int rb = (int)(x % a.n_rb);
  x /= a.n_rb;
  const int kvh = (int)(x % a.Hk), b = (int)(x / a.Hk);
  lat_line<256>(a, rb, kt, 0, b, span);
  const int64_t total = span.total, at = span.at;
  const int tiles = lat_tiles(a, len_of(a, b), rb, kt);
  const int j0 = lat_range_of(total, at, a.W), j1 = lat_range_of(total, at + tiles - 1, a.W);
  if (j0 == j1) return;  // one piece: written by its workgroup
  const int lane = threadIdx.x & 63;
  const int i = part * 4 + (threadIdx.x >> 6), row = rb * a.rpb + i;
  if (row >= a.R) return;
  constexpr int U = 8;  // partials in flight
  float m = kNegInf, l = 0.f, o[N];
#pragma unroll
  for (int e = 0; e < N; ++e) o[e] = 0.f;
  const int64_t unit = (int64_t)kvh * a.n_rb + rb;
  for (int s0 = j0; s0 <= j1; s0 += U) {
    float2 ml[U];
    float p[U][N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = min(s0 + u, j1);
      const int64_t begin = lat_cut(total, j, a.W);
      const int64_t pr = ((unit * a.W + j) * 2 + (begin >= at ? 0 : 1)) * a.rpb + i;
      // (Ranges of nothing, where there are more ranges than tiles, hold no partial.)
      const bool none = s0 + u > j1 || begin == lat_cut(total, j + 1, a.W);
      ml[u] = none ? make_float2(kNegInf, 0.f) : a.ml[pr];
#pragma unroll
      for (int e = 0; e < N; ++e) p[u][e] = none ? 0.f : a.opart[pr * DV + lane * N + e];
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u) mn = fmaxf(mn, ml[u].x);
    const float f0 = mn == m ? 1.f : __builtin_amdgcn_exp2f((m - mn) * a.scale_log2);
    l *= f0;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] *= f0;
    m = mn;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (ml[u].y == 0.f) continue;  // a piece without a key of this row
      const float f = __builtin_amdgcn_exp2f((ml[u].x - mn) * a.scale_log2);
      l += ml[u].y * f;
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = fmaf(p[u][e], f, o[e]);
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  const int mm = row / a.G, h = kvh * a.G + row - mm * a.G;
  const int64_t off = b * a.o_sb + (int64_t)mm * a.o_sm + (int64_t)h * a.o_sh + lane * N;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float y = o[e] * inv;
    if (a.out_dtype == 2)
      reinterpret_cast<float*>(a.out)[off + e] = y;
    else
      reinterpret_cast<uint16_t*>(a.out)[off + e] = (uint16_t)(a.out_dtype == 0 ? pack2<BF16>(y, y) : pack2<F16>(y, y));
  }
  if (lane == 0 && a.lse != nullptr) a.lse[b * a.l_sb + (int64_t)mm * a.l_sm + (int64_t)h * a.l_sh] = lat_lse(a, m, l);
}

template <int DV>
__global__ void __launch_bounds__(256) latent_merge_kernel(const LatArgs a, int kt, int64_t n) {
  __shared__ LatSpan span;
  for (int64_t x = blockIdx.x; x < n; x += gridDim.x) {
    merge_rows<DV>(a, kt, x, span);
    __syncthreads();
  }
}

template <typename T, int DC, int DR>
void launch_rows(const LatArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.n_rb * a.W)), block(256);
  if (a.rpb == 64)
    hipLaunchKernelGGL((latent_kernel<T, DC, DR, 64>), grid, block, 0, s, a);
  else if (a.rpb == 32)
    hipLaunchKernelGGL((latent_kernel<T, DC, DR, 32>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((latent_kernel<T, DC, DR, 16>), grid, block, 0, s, a);
}

template <typename T>
void launch_widths(const LatArgs& a, hipStream_t s) {
  if (a.dn == 512)
    a.dr == 64 ? launch_rows<T, 512, 64>(a, s) : launch_rows<T, 512, 32>(a, s);
  else
    a.dr == 64 ? launch_rows<T, 256, 64>(a, s) : launch_rows<T, 256, 32>(a, s);
}

}  // namespace

bool latent_widths(int dc, int dr) { return (dc == 256 || dc == 512) && (dr == 32 || dr == 64); }

hipError_t launch_latent(const LatArgs& a, hipStream_t s) {
  if (a.dtype == 0)
    launch_widths<BF16>(a, s);
  else
    launch_widths<F16>(a, s);
  return hipGetLastError();
}

hipError_t launch_latent_merge(const LatArgs& a, int kt, hipStream_t s) {
  if (a.W == 1) return hipSuccess;
  const int64_t n = (int64_t)a.B * a.Hk * a.n_rb * (a.rpb / 4);
  const dim3 grid((unsigned)(n < (1 << 20) ? n : 1 << 20)), block(256);
  switch (a.dv) {
    case 64: hipLaunchKernelGGL(latent_merge_kernel<64>, grid, block, 0, s, a, kt, n); break;
    case 128: hipLaunchKernelGGL(latent_merge_kernel<128>, grid, block, 0, s, a, kt, n); break;
    case 256: hipLaunchKernelGGL(latent_merge_kernel<256>, grid, block, 0, s, a, kt, n); break;
    default: hipLaunchKernelGGL(latent_merge_kernel<512>, grid, block, 0, s, a, kt, n); break;
  }
  return hipGetLastError();
}

}  // namespace dsv
