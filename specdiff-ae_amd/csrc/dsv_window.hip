// dsv_window.hip — attention through a sliding window with a few first tokens
// that stay visible (sinks), over a dense or paged cache, on gfx950.
//
// Mathematics.  The M new tokens of a sequence of len tokens sit at the end of
// its cache, n0 = len - M.  Row m has position p = n0 + m (causal), or n0 +
// its depth in the drafted tree, and sees key n of its past at position pos(n)
// iff pos(n) > p - W or pos(n) < S; the past is n <= p, or, with a tree, every
// n < n0 and the row's ancestors and itself.  out = sum softmax(q.k / sqrt D)
// v, lse = ln sum exp; a row without a key writes zeros and -inf.
//
// The G query heads of a KV head and neighbouring rows see nearly the same
// keys, so rows are packed row-major over (m, g), r = m * G + g: a workgroup's
// rows read each key once.  A workgroup's keys are the sinks' tiles followed by
// the tiles from its first row's window to its last row's position (32 keys a
// tile); what lies between is never read.  Only tiles at either border or in
// the tree are masked: one keep word of 32 bits per row, from comparisons of
// positions, so a mask costs no memory.
//
// Scores, sums and running maxima are fp32 (log2 domain); the probabilities
// are rounded to the inputs' 16-bit type for the second matrix product, the type
// of the values that they weigh (off by half a step of each: 2^-8 of it in bf16,
// 2^-11 in fp16, which holds them times a power of two, see kProbShift); their sum
// takes them unrounded.  Partial outputs of splits are fp32.
//
// Values of keys that a row does not see never reach it, whatever they hold: a
// masked score is replaced, keys that no row of a workgroup sees are not read (a
// seen one is, in their place), and where V holds infinities or NaN in a tile of
// which some row drops keys, the rows are computed once more without matrix
// products (exact_rows; in the product 0 * inf would be NaN).  So are rows whose
// scores are beyond 2^22, where the exponents lose their last bits before the point.
//
// win_rows_kernel (up to 16 rows: single tokens, short chunks): bound by
// reading K and V.  Eight waves share a workgroup's tiles, each with a softmax of
// its own, merged in LDS at the end, so no barrier stands in the loop.  A tile
// goes memory -> registers in whole rows (16 bytes a lane, the next tile in flight
// while this one is used) -> the wave's own LDS -> MFMA operands: K rows by
// ds_read_b128, V transposed by ds_read_b64_tr_b16.  Splits over the keys fill
// the GPU when there are few rows; win_merge_kernel joins them.  64 sequences of
// one token through 4096 keys (32 query heads, 8 key heads of 128, pages of 64):
// 179 us, 5.5 TB/s, 88% of what a kernel that only reads reaches (6.2).  One
// sequence through 1024 keys: 15 us, 5 of them arguments, length and page; in the
// rest 8 workgroups read 0.5 MB each, what one CU fetches (more workgroups would
// need the merge, a launch more).  (Each lane
// computing the offsets of the keys that it loads took 17.5: 64-bit products.)
//
// Reference context: runtime/attention_compat.py:103-132 (the cache call whose
// layouts are kept), runtime/cache_state.py:52-66 (the tree behind the prefix),
// draft/draft_network.py:1250-1331 (a working cache of first and recent
// tokens).

#include "dsv_internal.h"
#include "dsv_window_dev.h"

namespace dsv {

namespace {

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

// Over the four lanes of a row (lane ^ 16, lane ^ 32).
__device__ __forceinline__ float row_max(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float row_sum(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Eight waves, two per SIMD, each with a tile's loads in flight: the batch of 64
// above takes 179 us; with four waves a workgroup it took 230, and 16 do not have
// the registers (they spill).
constexpr int kRowWaves = 8;

// ---- few rows ------------------------------------------------------------------

template <typename T, int D, bool PAGED>
__global__ void __launch_bounds__(kRowWaves * 64) win_rows_kernel(const WinArgs a) {
  constexpr int NW = kRowWaves;
  constexpr int CH = D / 8;           // 16-byte chunks per key
  constexpr int KPI = 64 / CH;        // keys per load instruction
  constexpr int NL = 32 / KPI;        // load instructions per tile and half
  constexpr int KS = D / 32;          // k-steps of Q.K^T
  constexpr int DT = D / 16;          // d tiles of P.V
  constexpr int SHIFT = kProbShift<T, 15>;  // (the maximum is exact: probabilities are at most 2^15)
  // Row strides of the LDS images: K rows shift by 4 banks a key (b128 reads
  // of 16 keys), V rows by 8 (transposed reads of 16 keys x 32 bytes): free of
  // bank conflicts.  K, then V, then the wave's partial output use one region.
  constexpr int KST = 2 * D + 16, VST = 2 * D + 32, OST = (D + 4) * 4;
  constexpr int REGION = 32 * VST;
  static_assert(16 * OST <= REGION && 32 * KST <= REGION, "one region per wave");
  __shared__ __attribute__((aligned(16))) uint8_t smem[NW * REGION];
  __shared__ float sm_m[NW][16], sm_l[NW][16];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int lr = lane & 15, lg = lane >> 4;
  uint8_t* mine = smem + wave * REGION;

  int w = blockIdx.x;
  const int split = w % a.splits;
  w /= a.splits;
  const int rb = w % a.n_rb;
  w /= a.n_rb;
  const int kvh = w % a.Hk, b = w / a.Hk;
  const int n0 = len_of(a, b) - a.M;
  const int r0 = rb * 16;
  const WinKeys kl = win_keys(a.M, a.G, a.R, a.W, a.S, a.parent != nullptr, n0, r0, 16);
  const int t_end = (int)((int64_t)kl.nt * (split + 1) / a.splits);
  int t = (int)((int64_t)kl.nt * split / a.splits) + wave;

  // This lane's rows: Q fragments (B operand): row lr, elements 32 ks + 8 lg ..
  __shared__ TreeLds<16> tl;
  int pos;
  u32x4 qf[KS];
  {
    const Row row = row_of(a, min(r0 + lr, a.R - 1));
    const uint16_t* q = a.q + b * a.q_sb + (int64_t)row.m * a.q_sm + (int64_t)(kvh * a.G + row.g) * a.q_sh + 8 * lg;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const u32x4*>(q + 32 * ks);
    pos = n0 + row.m;
  }
  if (a.parent != nullptr) {
    tree_rows<16, kRowWaves * 64>(a, TreeParents<kRowWaves * 64>(a, b), n0, r0, tl);
    pos = n0 + tl.depth[lr];
  }
  int pmin = pos, pmax = pos;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    pmin = min(pmin, __shfl_xor(pmin, o));
    pmax = max(pmax, __shfl_xor(pmax, o));
  }

  float mx = kNegInf, ls = 0.f;
  uint32_t odd = 0;  // infinite or NaN entries of V in tiles that some row drops keys of, far scores
  f32x4 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x4{};

  const uint16_t* kbase = a.k + b * a.k_sb + kvh * a.k_sh + (lane % CH) * 8;
  const uint16_t* vbase = a.v + b * a.v_sb + kvh * a.v_sh + (lane % CH) * 8;
  // Lane l holds the page of key l (mod 32) of a tile, read a tile ahead.
  auto tile_pages = [&](int tt) -> int32_t {
    if (!PAGED || tt >= t_end) return 0;
    return page_of(a, b, kl.read(kl.base(tt) + (lane & 31)));
  };
  u32x4 kr[NL], vr[NL];
  // It works out that key's offsets for the others.
  auto load_tile = [&](int tt, int32_t pg) {
    const int n = kl.read(kl.base(tt) + (lane & 31));
    const long long ko = key_off(a, PAGED, a.k_sp, a.k_st, n, pg), vo = key_off(a, PAGED, a.v_sp, a.v_st, n, pg);
#pragma unroll
    for (int j = 0; j < NL; ++j) kr[j] = *reinterpret_cast<const u32x4*>(kbase + __shfl(ko, j * KPI + lane / CH));
#pragma unroll
    for (int j = 0; j < NL; ++j) vr[j] = *reinterpret_cast<const u32x4*>(vbase + __shfl(vo, j * KPI + lane / CH));
  };

  int32_t pg = tile_pages(t);
  if (t < t_end) load_tile(t, pg);
  pg = tile_pages(t + NW);
  for (; t < t_end; t += NW) {
    const int kb = kl.base(t);
    // ---- S^T = K . Q^T
#pragma unroll
    for (int j = 0; j < NL; ++j)
      *reinterpret_cast<u32x4*>(mine + (j * KPI + lane / CH) * KST + (lane % CH) * 16) = kr[j];
    wave_lds_fence();
    f32x4 s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] = f32x4{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u32x4 kf = *reinterpret_cast<const u32x4*>(mine + (16 * h + lr) * KST + (4 * ks + lg) * 16);
        s[h] = mfma16<T>(kf, qf[ks], s[h]);
      }
    }
    wave_lds_fence();
    // ---- V into LDS
    const bool masked = !kl.seen_by_all(kb, pmin, pmax, a.W, a.S, n0, a.parent != nullptr);
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      const int i = j * KPI + lane / CH;
      if (masked) odd |= nonfinite2<T>(vr[j][0]) | nonfinite2<T>(vr[j][1]) | nonfinite2<T>(vr[j][2]) | nonfinite2<T>(vr[j][3]);
      *reinterpret_cast<u32x4*>(mine + i * VST + (lane % CH) * 16) = vr[j];
    }
    wave_lds_fence();
    // ---- the next tile's loads
    if (t + NW < t_end) load_tile(t + NW, pg);
    pg = tile_pages(t + 2 * NW);
    // ---- mask and softmax
    if (masked) {
      const uint32_t keep = keep_word(a, tl.vis + lr * kTreeMaxW, pos, kb, n0);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!((keep >> (16 * (e >> 2) + 4 * lg + (e & 3))) & 1u)) s[e >> 2][e & 3] = kNegInf;
    }
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = s[e >> 2][e & 3];
    float mt = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mt = fmaxf(mt, x[e]);
    const float mn = fmaxf(mx, row_max(mt) * a.scale_log2);
    if (__ballot(mn > mx) != 0ull) {
      const float al = mx == kNegInf ? 0.f : __builtin_amdgcn_exp2f(mx - mn);
      ls *= al;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] *= al;
      mx = mn;
      odd |= far_score(mx) ? 0x80008000u : 0u;
    }
    const float ms = mx == kNegInf ? 0.f : mx - (float)SHIFT;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], a.scale_log2, -ms));
      ls += x[e];
    }
    const u32x4 pf = {pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7])};
    // ---- O^T += V^T . P^T; element e of lane group lg is key 16 (e / 4) + 4 lg + e % 4.
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const uint8_t* p = mine + (4 * lg + (lr >> 2)) * VST + (16 * d + 4 * (lr & 3)) * 2;
      const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
      const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 16 * VST)));
      const u32x4 vf = {lo[0], lo[1], hi[0], hi[1]};
      acc[d] = mfma16<T>(vf, pf, acc[d]);
    }
    wave_lds_fence();
  }

  if (__syncthreads_or((int)(odd & 0x80008000u)) != 0) {
    exact_rows<T, D, 16>(&args_again(), &tl, b, kvh, split, rb, (int)((int64_t)kl.nt * split / a.splits), t_end, wave, 16, NW);
    return;
  }
  // ---- the waves' rows joined (sums as without the factor: by exact products)
  constexpr float kBack = 1.f / (1 << SHIFT);
  const float lt = row_sum(ls) * kBack;
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] *= kBack;
  if (lg == 0) {
    sm_m[wave][lr] = mx;
    sm_l[wave][lr] = lt;
  }
#pragma unroll
  for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(mine + lr * OST + (16 * d + 4 * lg) * 4) = acc[d];
  __syncthreads();
  constexpr int N = 4;  // elements per thread
  constexpr int TPR = D / N;
  const int rr = threadIdx.x / TPR, d0 = threadIdx.x % TPR * N;
  if (rr < 16) {
    float m = sm_m[0][rr];
#pragma unroll
    for (int x = 1; x < NW; ++x) m = fmaxf(m, sm_m[x][rr]);
    const float ms = m == kNegInf ? 0.f : m;
    float l = 0.f, o[N];
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      if (sm_l[x][rr] == 0.f) continue;  // a wave without a key of this row
      const float f = __builtin_amdgcn_exp2f(sm_m[x][rr] - ms);
      l += sm_l[x][rr] * f;
      const f32x4* p = reinterpret_cast<const f32x4*>(smem + x * REGION + rr * OST + d0 * 4);
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] += p[e / 4][e % 4] * f;
    }
    const int r = r0 + rr;
    if (r < a.R) {
      if (a.splits == 1) {
        const int mm = r / a.G, h = kvh * a.G + r - mm * a.G;
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] *= inv;
        store_out(a, b * a.o_sb + mm * a.o_sm + h * a.o_sh + d0, o);
        if (d0 == 0 && a.lse != nullptr)
          a.lse[b * a.l_sb + mm * a.l_sm + h * a.l_sh] = l == 0.f ? kNegInf : (m + __log2f(l)) * kLn2;
      } else {
        const int64_t pr = ((int64_t)(b * a.Hk + kvh) * a.splits + split) * a.R + r;
#pragma unroll
        for (int e = 0; e < N; e += 4) *reinterpret_cast<f32x4*>(a.opart + pr * D + d0 + e) = f32x4{o[e], o[e + 1], o[e + 2], o[e + 3]};
        if (d0 == 0) a.ml[pr] = make_float2(m, l);
      }
    }
  }
}

// ---- fp32 ------------------------------------------------------------------------
// The same walk over tiles with v_mfma_f32_16x16x4_f32, 16 rows and 32 keys a
// step.  K's operand takes a lane's 16 bytes as four k-steps (the order of the
// head dimension in the product is free as long as Q's agrees), V's operand a
// lane's 16 bytes as four tiles of columns (tile d's row i is column 64 (d / 4) + 4 i
// + d % 4), so nothing passes through LDS but the join of the waves.
// Three chunks of 37 rows through 777 keys (14 query heads, 2 key heads of 64):
// 20 us, of which 102 workgroups of three or four tiles a wave spend 4.5 before the
// first tile and a third in fp32 MFMA (a tile: 64 of 32 cycles, two waves a SIMD).
template <int D, bool PAGED>
__global__ void __launch_bounds__(kRowWaves * 64) win_rows_f32_kernel(const WinArgs a) {
  constexpr int NW = kRowWaves;
  constexpr int KC = D / 16;          // 16-byte chunks per lane and key
  constexpr int DT = D / 16;
  constexpr int OST = D + 4;
  __shared__ __attribute__((aligned(16))) float smem[NW][16 * OST];
  __shared__ float sm_m[NW][16], sm_l[NW][16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int lr = lane & 15, lg = lane >> 4;
  int w = blockIdx.x;
  const int split = w % a.splits;
  w /= a.splits;
  const int rb = w % a.n_rb;
  w /= a.n_rb;
  const int kvh = w % a.Hk, b = w / a.Hk;
  const int n0 = len_of(a, b) - a.M;
  const int r0 = rb * 16;
  const WinKeys kl = win_keys(a.M, a.G, a.R, a.W, a.S, a.parent != nullptr, n0, r0, 16);
  const int t_end = (int)((int64_t)kl.nt * (split + 1) / a.splits);
  const float* kbase = reinterpret_cast<const float*>(a.k) + b * a.k_sb + kvh * a.k_sh;
  const float* vbase = reinterpret_cast<const float*>(a.v) + b * a.v_sb + kvh * a.v_sh;

  __shared__ TreeLds<16> tl;
  const Row row = row_of(a, min(r0 + lr, a.R - 1));
  f32x4 qf[KC];
  const float* q = reinterpret_cast<const float*>(a.q) + b * a.q_sb + (int64_t)row.m * a.q_sm + (int64_t)(kvh * a.G + row.g) * a.q_sh;
#pragma unroll
  for (int c = 0; c < KC; ++c) qf[c] = *reinterpret_cast<const f32x4*>(q + 16 * c + 4 * lg);
  int pos = n0 + row.m;
  if (a.parent != nullptr) {
    tree_rows<16, kRowWaves * 64>(a, TreeParents<kRowWaves * 64>(a, b), n0, r0, tl);
    pos = n0 + tl.depth[lr];
  }
  int pmin = pos, pmax = pos;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    pmin = min(pmin, __shfl_xor(pmin, o));
    pmax = max(pmax, __shfl_xor(pmax, o));
  }
  float mx = kNegInf, ls = 0.f;
  bool odd = false;
  f32x4 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x4{};

  // Lane l holds the page of key l (mod 32) of a tile, read a tile ahead.
  auto tile_pages = [&](int tt) -> int32_t {
    if (!PAGED || tt >= t_end) return 0;
    return page_of(a, b, kl.read(kl.base(tt) + (lane & 31)));
  };
  int t = (int)((int64_t)kl.nt * split / a.splits) + wave;
  // Keys 16 h + lr of K (operand A), 16 (e / 4) + 4 lg + e % 4 of V; the next tile's
  // are loaded as soon as this one's have been used.
  f32x4 kf[2][KC];
  f32x4 vf[8][DT / 4];
  // Lane l works out the offsets of key l (mod 32) for the others.
  auto load_k = [&](int tt, int32_t pg) {
    const long long ko = key_off(a, PAGED, a.k_sp, a.k_st, kl.read(kl.base(tt) + (lane & 31)), pg);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float* k = kbase + __shfl(ko, 16 * h + lr) + 4 * lg;
#pragma unroll
      for (int c = 0; c < KC; ++c) kf[h][c] = *reinterpret_cast<const f32x4*>(k + 16 * c);
    }
  };
  auto load_v = [&](int tt, int32_t pg) {
    const long long vo = key_off(a, PAGED, a.v_sp, a.v_st, kl.read(kl.base(tt) + (lane & 31)), pg);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float* v = vbase + __shfl(vo, 16 * (e >> 2) + 4 * lg + (e & 3)) + 4 * lr;
#pragma unroll
      for (int d = 0; d < DT / 4; ++d) vf[e][d] = *reinterpret_cast<const f32x4*>(v + 64 * d);
    }
  };
  int32_t pg = tile_pages(t);
  if (t < t_end) {
    load_k(t, pg);
    load_v(t, pg);
  }
  pg = tile_pages(t + NW);
  for (; t < t_end; t += NW) {
    const int kb = kl.base(t);
    const bool masked = !kl.seen_by_all(kb, pmin, pmax, a.W, a.S, n0, a.parent != nullptr);
    const uint32_t keep = masked ? keep_word(a, tl.vis + lr * kTreeMaxW, pos, kb, n0) : ~0u;
    f32x4 s[2] = {f32x4{}, f32x4{}};
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int h = 0; h < 2; ++h) s[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[h][c][e], qf[c][e], s[h], 0, 0, 0);
    if (t + NW < t_end) load_k(t + NW, pg);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = s[e >> 2][e & 3];
      if (masked && !((keep >> (16 * (e >> 2) + 4 * lg + (e & 3))) & 1u)) x[e] = kNegInf;
    }
    float mt = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mt = fmaxf(mt, x[e]);
    const float mn = fmaxf(mx, row_max(mt) * a.scale_log2);
    if (__ballot(mn > mx) != 0ull) {
      const float al = mx == kNegInf ? 0.f : __builtin_amdgcn_exp2f(mx - mn);
      ls *= al;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] *= al;
      mx = mn;
      odd |= far_score(mx);
    }
    const float ms = mx == kNegInf ? 0.f : mx;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], a.scale_log2, -ms));
      ls += x[e];
    }
    if (masked) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int d = 0; d < DT; ++d) odd |= !(vf[e][d / 4][d % 4] - vf[e][d / 4][d % 4] == 0.f);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[e][d / 4][d % 4], x[e], acc[d], 0, 0, 0);
    if (t + NW < t_end) load_v(t + NW, pg);
    pg = tile_pages(t + 2 * NW);
  }
  if (__syncthreads_or((int)odd) != 0) {
    exact_rows<float, D, 16>(&args_again(), &tl, b, kvh, split, rb, (int)((int64_t)kl.nt * split / a.splits), t_end, wave, 16, NW);
    return;
  }

  const float lt = row_sum(ls);
  if (lg == 0) {
    sm_m[wave][lr] = mx;
    sm_l[wave][lr] = lt;
  }
#pragma unroll
  for (int d = 0; d < DT; d += 4)
#pragma unroll
    for (int v = 0; v < 4; ++v)
      *reinterpret_cast<f32x4*>(&smem[wave][lr * OST + 16 * d + 16 * lg + 4 * v]) =
          f32x4{acc[d][v], acc[d + 1][v], acc[d + 2][v], acc[d + 3][v]};
  __syncthreads();
  constexpr int N = 4, TPR = D / N;
  const int rr = threadIdx.x / TPR, d0 = threadIdx.x % TPR * N;
  if (rr >= 16) return;
  float m = sm_m[0][rr];
#pragma unroll
  for (int y = 1; y < NW; ++y) m = fmaxf(m, sm_m[y][rr]);
  const float ms = m == kNegInf ? 0.f : m;
  float l = 0.f, o[N];
#pragma unroll
  for (int e = 0; e < N; ++e) o[e] = 0.f;
#pragma unroll
  for (int y = 0; y < NW; ++y) {
    if (sm_l[y][rr] == 0.f) continue;
    const float f = __builtin_amdgcn_exp2f(sm_m[y][rr] - ms);
    l += sm_l[y][rr] * f;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] += smem[y][rr * OST + d0 + e] * f;
  }
  const int r = r0 + rr;
  if (r >= a.R) return;
  if (a.splits == 1) {
    const int mm = r / a.G, hh = kvh * a.G + r - mm * a.G;
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] *= inv;
    store_out(a, b * a.o_sb + mm * a.o_sm + hh * a.o_sh + d0, o);
    if (d0 == 0 && a.lse != nullptr)
      a.lse[b * a.l_sb + mm * a.l_sm + hh * a.l_sh] = l == 0.f ? kNegInf : (m + __log2f(l)) * kLn2;
  } else {
    const int64_t pr = ((int64_t)(b * a.Hk + kvh) * a.splits + split) * a.R + r;
#pragma unroll
    for (int e = 0; e < N; e += 4) *reinterpret_cast<f32x4*>(a.opart + pr * D + d0 + e) = f32x4{o[e], o[e + 1], o[e + 2], o[e + 3]};
    if (d0 == 0) a.ml[pr] = make_float2(m, l);
  }
}

// ---- the splits joined -------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(256) win_merge_kernel(const WinArgs a) {
  constexpr int TPR = D / 4;  // threads per row, four elements each
  const int64_t x = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  const int d0 = (threadIdx.x % TPR) * 4;
  if (x >= (int64_t)a.B * a.Hk * a.R) return;
  const int64_t bh = x / a.R;
  const int r = (int)(x - bh * a.R);
  const int b = (int)(bh / a.Hk), kvh = (int)(bh % a.Hk);
  // Eight splits' loads in flight (16 splits of 4096 rows: 12 us with four, 8 with
  // eight).
  constexpr int U = 8;
  float m = kNegInf, l = 0.f;
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  const int64_t p0 = bh * a.splits * a.R + r;
  for (int s0 = 0; s0 < a.splits; s0 += U) {
    float2 ml[U];
    f32x4 p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t pr = p0 + (int64_t)min(s0 + u, a.splits - 1) * a.R;
      ml[u] = a.ml[pr];
      p[u] = *reinterpret_cast<const f32x4*>(a.opart + pr * D + d0);
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u >= a.splits) ml[u] = make_float2(kNegInf, 0.f);
      mn = fmaxf(mn, ml[u].x);
    }
    const float ms = mn == kNegInf ? 0.f : mn, f0 = __builtin_amdgcn_exp2f(m - ms);
    l *= f0;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= f0;
    m = mn;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (ml[u].y == 0.f) continue;  // a split without a key of this row
      const float f = __builtin_amdgcn_exp2f(ml[u].x - ms);
      l += ml[u].y * f;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += p[u][e] * f;
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] *= inv;
  const int mm = r / a.G, h = kvh * a.G + r - mm * a.G;
  store_out(a, b * a.o_sb + mm * a.o_sm + h * a.o_sh + d0, o);
  if (d0 == 0 && a.lse != nullptr)
    a.lse[b * a.l_sb + mm * a.l_sm + h * a.l_sh] = l == 0.f ? kNegInf : (m + __log2f(l)) * kLn2;
}

template <typename T, int D>
hipError_t launch_rows(const WinArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.B * a.Hk * a.n_rb * a.splits)), block(kRowWaves * 64);
  if (a.pt != nullptr)
    hipLaunchKernelGGL((win_rows_kernel<T, D, true>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((win_rows_kernel<T, D, false>), grid, block, 0, s, a);
  return hipGetLastError();
}

template <int D>
hipError_t launch_rows_f32(const WinArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.B * a.Hk * a.n_rb * a.splits)), block(kRowWaves * 64);
  if (a.pt != nullptr)
    hipLaunchKernelGGL((win_rows_f32_kernel<D, true>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((win_rows_f32_kernel<D, false>), grid, block, 0, s, a);
  return hipGetLastError();
}

template <int D>
hipError_t launch_d(const WinArgs& a, hipStream_t s) {
  hipError_t e;
  if (a.dtype == 2) {
    e = launch_rows_f32<D>(a, s);
  } else if (a.rows_per_block == 256) {
    e = launch_window_tile(a, D, s);
  } else {
    e = a.dtype == 0 ? launch_rows<BF16, D>(a, s) : launch_rows<F16, D>(a, s);
  }
  if (e != hipSuccess || a.splits == 1) return e;
  const int64_t rows = (int64_t)a.B * a.Hk * a.R;
  const int per = 256 / (D / 4);
  hipLaunchKernelGGL(win_merge_kernel<D>, dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_window(const WinArgs& a, int D, hipStream_t s) { return D == 64 ? launch_d<64>(a, s) : launch_d<128>(a, s); }

}  // namespace dsv
