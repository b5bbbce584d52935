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
// serves both products, S^T = X . Q^T and O^T = X^T . P^T.  Of the output, wave w of
// four has the columns [w dc / 4, (w + 1) dc / 4) for all rows and keys.  Of the scores
// of 16 or 32 rows it has the keys [16w, 16w + 16) for all rows, in 16x16x32 products;
// of 64 rows, 32 keys of 32 rows (waves 2 x 2), in 32x32x16 products, whose operands
// serve twice the flops.  The probabilities go between the two through LDS.  So each
// cache row is read from LDS once (64 rows: twice) as a key and once as a value; waves
// that own rows would each read the whole tile twice.
//
// The running maximum is common to the waves and may lag behind the true one by
// kLatTau (log2 units); a wave whose scores exceed it raises a flag beside its
// probabilities, and only then do the waves exchange maxima and rescale.  The
// exponent is (s - max) * scale, a difference of scores, so that it holds for scores
// of any size.  Scores, sums and maxima are fp32; probabilities are rounded to the
// cache's type for the second product (half a step of each; fp16 holds them times
// 2^10, see kProbShift); their sum takes them unrounded.
//
// Registers: a wave alone on its SIMD has 512.  At 512 + 64 and 64 rows the queries
// (144) stand in the upper half, which only the matrix products read, and the output
// (128), the scores and the operands ahead in the lower.  The queries come through LDS:
// a load that ends in registers would be waited for with the tiles in flight behind it.
//
// Tiles go HBM -> LDS by LDS-DMA into two buffers.  Where a block of rows has the keys
// to itself, the next tile's loads are issued as soon as its buffer is free, so that the
// memory is never idle; where several blocks share them, between the products (measured
// with 128 heads: 92 -> 84 us; issued at once, 72 loads take the CU 1700 cycles).
// Sequences and their tiles are shared out evenly over the workgroups (LatCut),
// whatever their lengths; latent_merge_kernel joins the partials.
//
// Measured at rows of 512 + 64 (a large copy reaches 4.95 TB/s, a large bf16 product
// 1309 TFLOP/s).  64 sequences of up to 16384 keys, 16 heads, 652 MB: 126 + 6.5 us (the
// join), 4.9 TB/s, bound by HBM.  One sequence of 2900 keys, 128 heads: 15 + 5.5 us, bound by
// latencies: arguments, lengths, pages, first tile, and the code itself as it is fetched.
// 32 sequences of 1000 to 8192 keys, 128 heads, fp16: 77 + 11 to 14 us; 8 trees of 64 nodes, 32
// heads: 194 + 16 us, 56 % of the large product's rate: a wave alone on its SIMD does its
// products, exponents and barriers one after the other (of 4300 cycles a tile the products'
// own are 2200); a second wave's registers are the output's and the queries'.

#include "dsv_dma.h"
#include "dsv_latent_dev.h"

namespace dsv {

namespace {

template <typename T>
constexpr float kLatTau = 8.0f;
template <>
constexpr float kLatTau<F16> = 5.0f;

// Products: 16x16x32 into four values a lane, 32x32x16 into sixteen.
template <typename T>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (__is_same(T, BF16))
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (__is_same(T, BF16))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <bool WIDE>
struct LatAcc {
  typedef f32x4 type;
};
template <>
struct LatAcc<true> {
  typedef f32x16 type;
};

// Over the lanes that hold one row (TR lanes apart).
template <int TR>
__device__ __forceinline__ float groups_max(float x) {
  if constexpr (TR == 16) x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
template <int TR>
__device__ __forceinline__ float groups_sum(float x) {
  if constexpr (TR == 16) x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// x, computed again at every use: what is derived from it is not held in registers
// across the loop.
__device__ __forceinline__ uint32_t again(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

// LDS image of a tile: the rows' first dc entries, then their last dr.  Chunk c (16
// bytes) of key k stands at slot c ^ swz(k): keys read at one chunk (scores) and four
// keys read at neighbouring chunks (values, transposed) fall on distinct banks in the
// reads of 64 rows' products (conflict cycles 5 % of the LDS's).  Those of 16 and 32 rows
// read eight keys at once, two on a bank (45 %, beside loads that take longer).
__device__ __forceinline__ int swz_n(int key) { return ((key & 3) << 2) | ((key >> 2) & 3); }
template <int DR>
__device__ __forceinline__ int swz_r(int key) {
  return DR == 64 ? (key >> 1) & 7 : (key >> 2) & 3;
}

template <int DC, int DR, int ROWS>
struct LatLds {
  static constexpr int KT = 1 << kLatTile;
  static constexpr int NB = DC * 2, RB = DR * 2;
  static constexpr int TILE = KT * (NB + RB);
  // Sets of tree keys: a block's rows of H heads belong to at most ROWS nodes, of
  // H >= 2 heads to ROWS / 2 + 1 (the plan takes blocks of 32 where that does not fit).
  static constexpr int VIS = 36 * (kTreeMaxM / 64) * 8;
  uint8_t ring[2 * TILE];          // tiles; at the end the output rows in fp32
  uint8_t p[ROWS * KT * 2];
  uint64_t vis[VIS / 8];
  float red[4][ROWS];
  float m[ROWS];
  uint32_t flag[4];
  LatSpan span;
  static_assert(TILE % 1024 == 0, "XORs within a row leave the buffer alone");
  static_assert(ROWS * DC * 4 <= 2 * TILE, "");
  static_assert(2 * kTreeMaxM <= ROWS * KT * 2, "the parents are staged in p");
};

// DMA of one wave's 16 rows of a tile: keys [16w, 16w + 16).  (Instructions are what a
// lone wave on a SIMD is short of: one is issued every four cycles at most.)
template <int DC, int DR>
struct LatLoader {
  using L = LatLds<DC, DR, 16>;
  static constexpr int KPI = 1024 / L::NB;         // keys per instruction of the first part
  static constexpr int IPN = 16 / KPI;             // such instructions per tile
  static constexpr int KPR = 1024 / L::RB;         // the same of the second part
  static constexpr int IPR = 16 * L::RB / 1024;
  static constexpr int N = IPN + IPR;
  static_assert(KPI <= 2, "");
  const LatArgs& a;
  int wid, lane;
  uint32_t dstn, dstr;
  bool run_ok;                                     // a wave's 16 keys lie at even, 32-bit distances
  int b, end;
  uint64_t base;
  int32_t pwin;                                    // lane l: physical page of the sequence's page pw0 + l
  int pw0;
  int shift, mask;                                 // of the page size (a dense cache is one page, number 0)
  uint64_t sp2;
  uint32_t kst2;

  __device__ __forceinline__ LatLoader(const LatArgs& args, int w, int l, uint32_t ring) : a(args), wid(w), lane(l) {
    dstn = ring + w * 16 * L::NB;
    dstr = ring + L::KT * L::NB + w * 16 * L::RB;
    shift = a.pt != nullptr ? a.ps_shift : 30;
    mask = (1 << shift) - 1;
    sp2 = (uint64_t)(2 * a.kn.sp);
    kst2 = (uint32_t)(2 * a.kn.st);
    run_ok = (a.pt == nullptr || a.ps_shift >= 4) && a.kn.st > 0 && a.kn.st <= (1 << 24);
  }
  __device__ __forceinline__ void sequence(int b_, int end_) {
    b = b_;
    end = end_;
    base = (uint64_t)a.kn.p + 2 * (b * a.kn.sb);
    pw0 = a.pt != nullptr ? -64 : 0;
    pwin = 0;
  }
  // A wave's rows: 16 at even distances st2 from a uniform address, or (st2 = 0) anywhere,
  // lane l knowing the address of row l % 16.
  uint64_t from;
  uint32_t st2;
  // Instruction x of such rows.
  __device__ __forceinline__ void one(uint32_t buf, int x, uint32_t ln) const {
    if (x < IPN) {
      const uint32_t k = KPI > 1 ? ln / (64 / KPI) : 0, c = ln % (64 / KPI);
      dma_off(dstn + buf + x * 1024, from, (x * KPI + k) * st2 + ((c ^ swz_n(x * KPI + k)) << 4));
    } else {
      const uint32_t k = (x - IPN) * KPR + ln / (64 / KPR), c = ln % (64 / KPR);
      dma_off(dstr + buf + (x - IPN) * 1024, from + L::NB, k * st2 + ((c ^ swz_r<DR>(k)) << 4));
    }
  }
  __device__ __forceinline__ void all(uint32_t buf, uint64_t addr) const {
    const uint32_t ln = again(lane);
    if (st2 != 0) {
#pragma unroll 2
      for (int x = 0; x < N; ++x) one(buf, x, ln);
      return;
    }
#pragma unroll 4
    for (int x = 0; x < IPN; ++x) {
      const int k = x * KPI + ln / (64 / KPI);
      const char* r = (const char*)__shfl((long long)addr, k);
      dma_lane<false>(dstn + buf + x * 1024, r + (((ln % (64 / KPI)) ^ swz_n(k)) << 4));
    }
#pragma unroll
    for (int x = 0; x < IPR; ++x) {
      const int k = x * KPR + ln / (64 / KPR);
      const char* r = (const char*)__shfl((long long)addr, k);
      dma_lane<false>(dstr + buf + x * 1024, r + L::NB + (((ln % (64 / KPR)) ^ swz_r<DR>(k)) << 4));
    }
  }
  __device__ __forceinline__ static uint64_t uniform64(uint64_t x) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)x);
  }
  // The keys [kb, kb + 64); those at or behind the end are replaced by the last one (no row
  // sees them).  Page numbers are kept in a window: a load at the use would be waited for,
  // and the tiles in flight with it.  Returns a lane's address where they lie apart.
  __device__ __forceinline__ uint64_t keys(int kb) {
    const int n0 = kb + wid * 16;
    if (!run_ok || n0 + 15 >= end || (uint32_t)((n0 >> shift) - pw0) >= 64u) return keys_slow(kb);
    run(n0);
    return 0;
  }
  __device__ __forceinline__ void run(int n0) {
    const uint32_t pg = (uint32_t)__builtin_amdgcn_readlane(pwin, (n0 >> shift) - pw0);
    from = base + (uint64_t)pg * sp2 + (uint64_t)(uint32_t)(n0 & mask) * kst2;
    st2 = kst2;
  }
  __device__ __forceinline__ uint64_t keys_slow(int kb) {
    const int n0 = min(kb + wid * 16, end - 1), n1 = min(kb + wid * 16 + 15, end - 1);
    const int p0 = n0 >> shift;
    if (a.pt != nullptr && (p0 < pw0 || n1 >> shift >= pw0 + 64)) {
      pw0 = p0;
      pwin = (int32_t)page_of(a, b, (int)min((int64_t)(p0 + lane) << shift, (int64_t)end - 1));
      asm volatile("" : "+v"(pwin));  // (waited for here)
    }
    if (run_ok && n1 == n0 + 15) {
      run(n0);
      return 0;
    }
    st2 = 0;
    const int n = min(n0 + (lane & 15), end - 1);
    return base + 2 * key_off(a, a.kn, n, a.pt != nullptr ? __shfl(pwin, (n >> shift) - pw0) : 0);
  }
  // The query rows [row0, row0 + 16) of this wave; those behind the last are replaced by it.
  __device__ __forceinline__ uint64_t queries(int row0) {
    const int r = min(row0 + wid * 16 + (lane & 15), a.R - 1), m = r / a.G;
    const uint64_t at = (uint64_t)a.q + 2 * (b * a.q_sb + (int64_t)m * a.q_sm + (int64_t)(r - m * a.G) * a.q_sh);
    st2 = 0;
    if (row0 + wid * 16 + 15 < a.R && (a.M == 1 || a.q_sm == a.G * a.q_sh) && a.q_sh > 0 && a.q_sh <= (1 << 24)) {
      from = uniform64(at);
      st2 = (uint32_t)(2 * a.q_sh);
    }
    return at;
  }
};

// Rows of a block from LDS (fp32, chunk c of row r at c ^ (r & 15)) into the output or a
// partial.  red: [groups][ROWS] sums; off, fac: room for a row's place and factor.  Called
// by every thread; the caller's next barrier ends it.
template <int DC, int ROWS, int GROUPS>
__device__ __forceinline__ void lat_store_rows(const LatArgs& a, const LatPiece& pc, int rb, const uint8_t* acc, const float* m,
                                               const float (*red)[ROWS], float back, int64_t* off, float* fac) {
  const bool part = pc.slot >= 0;
  const int rows = min(ROWS, a.R - rb * ROWS);
  if ((int)threadIdx.x < rows) {
    const int r = threadIdx.x, row = rb * ROWS + r, pos = row / a.G, h = row - pos * a.G;
    float l = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) l += red[g][r];
    l *= back;
    const int64_t pr = pc.slot * ROWS + r;
    off[r] = part ? pr * DC : b_off(a, pc.b, pos, h);
    fac[r] = part ? back : l > 0.f ? back / l : (l == 0.f ? 0.f : l);
    if (part)
      a.ml[pr] = make_float2(m[r], l);
    else if (a.lse != nullptr)
      a.lse[pc.b * a.l_sb + (int64_t)pos * a.l_sm + (int64_t)h * a.l_sh] = lat_lse(a, m[r], l);
  }
  __syncthreads();
  auto chunk = [&](int r, int c) { return *reinterpret_cast<const f32x4*>(acc + r * DC * 4 + ((c ^ (r & 15)) << 4)) * fac[r]; };
  if (part || (a.out_dtype == 2 && a.out_vec)) {
    float* o = part ? a.opart : reinterpret_cast<float*>(a.out);
#pragma unroll 4
    for (int x = threadIdx.x; x < rows * (DC / 4); x += 256) {
      const int r = x / (DC / 4), c = x % (DC / 4);
      *reinterpret_cast<f32x4*>(o + off[r] + c * 4) = chunk(r, c);
    }
  } else if (a.out_vec) {
#pragma unroll 2
    for (int x = threadIdx.x; x < rows * (DC / 8); x += 256) {
      const int r = x / (DC / 8), c = x % (DC / 8);
      const f32x4 u = chunk(r, 2 * c), v = chunk(r, 2 * c + 1);
      u32x4 w;
      if (a.out_dtype == 0)
        w = u32x4{pack2<BF16>(u[0], u[1]), pack2<BF16>(u[2], u[3]), pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3])};
      else
        w = u32x4{pack2<F16>(u[0], u[1]), pack2<F16>(u[2], u[3]), pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3])};
      *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(a.out) + off[r] + c * 8) = w;
    }
  } else {
    // (An output whose rows take no vector stores: element by element.)
#pragma unroll 1
    for (int x = threadIdx.x; x < rows * DC; x += 256) {
      const int r = x / DC, d = x % DC;
      store1(a, off[r] + d, *reinterpret_cast<const float*>(acc + r * DC * 4 + (((d >> 2) ^ (r & 15)) << 4) + (d & 3) * 4) * fac[r]);
    }
  }
}

template <int ROWS, bool WIDE>
struct LatShape;
// 16x16x32 products.  Scores: wave w has keys [16w, 16w + 16) for all rows.
template <int ROWS>
struct LatShape<ROWS, false> {
  static constexpr int KG = 4, RG = 1, QR = ROWS / 16, RB = ROWS / 16, TR = 16;
};
// 32x32x16 products, of 64 rows: wave w has keys [32 (w % 2), + 32) for rows [32 (w / 2), + 32).
template <>
struct LatShape<64, true> {
  static constexpr int KG = 2, RG = 2, QR = 1, RB = 2, TR = 32;
};

template <typename T, int DC, int DR, int ROWS>
__global__ void __launch_bounds__(256, 1) latent_kernel(const LatArgs a) {
  using L = LatLds<DC, DR, ROWS>;
  using Loader = LatLoader<DC, DR>;
  constexpr bool WIDE = ROWS == 64;
  using S = LatShape<ROWS, WIDE>;
  // TR rows a product; scores of QR such row groups per wave, outputs of all RB.
  constexpr int KT = L::KT, KG = S::KG, QR = S::QR, RB = S::RB, TR = S::TR;
  constexpr int DS = WIDE ? 16 : 32;               // depth of a product
  constexpr int KSN = DC / DS, KSR = DR / DS, KS = KSN + KSR;
  constexpr int CB = DC / 4 / TR;                  // output tiles of TR columns per wave
  constexpr int NV = WIDE ? 16 : 4;                // values of a product's result per lane
  constexpr int SHIFT = kProbShift<T, 10>;
  using Acc = typename LatAcc<WIDE>::type;
  static_assert(sizeof(L) <= 163840, "LDS of a CU");
  __shared__ __attribute__((aligned(1024))) L lds;

  lat_touch_args();
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, li = lane & (TR - 1), lg = lane / TR;

  // Dispatch ids go round-robin over the 8 XCDs: give each a contiguous eighth, so
  // that the row blocks of a range, which read the same keys, share an L2.
  const int nblk = gridDim.x;
  const int w = (nblk & 7) == 0 ? (int)(blockIdx.x & 7) * (nblk >> 3) + (int)(blockIdx.x >> 3) : (int)blockIdx.x;
  const int rb = w % a.n_rb, rj = w / a.n_rb;

  const LatEnd ends(a, rb);
  const LatCut cut(lat_line<256>(a, ends, kLatTile, rj, -1, lds.span), a.W);
  const int start = cut.begin(rj), stop = cut.begin(rj + 1);
  if (start >= stop) return;
  int b = __builtin_amdgcn_readfirstlane(lds.span.b);
  int t0 = __builtin_amdgcn_readfirstlane(lds.span.off);

  const int m_lo = rb * ROWS / a.G, m_hi = (min((rb + 1) * ROWS, a.R) - 1) / a.G;

  // Operand addresses within a tile (the swizzles are XORs of whole chunks).
  const int kg = wid % KG, rg = wid / KG;
  const uint32_t qofs = li * L::NB + ((lg ^ swz_n(li)) << 4);
  const uint32_t qrofs = KT * L::NB + li * L::RB + ((lg ^ swz_r<DR>(li)) << 4);
  const uint32_t kofs = kg * (KT / KG) * L::NB + qofs, rofs = kg * (KT / KG) * L::RB + qrofs;
  uint32_t vofs;
  {
    const int bl = lane >> 4, bi = lane & 15;
    const int vkey = 4 * (WIDE ? bl >> 1 : bl) + (bi >> 2), vcol = wid * (DC / 4) + (WIDE ? 16 * (bl & 1) : 0) + 4 * (bi & 3);
    vofs = vkey * L::NB + (((vcol >> 3) ^ swz_n(vkey)) << 4) + (vcol & 7) * 2;
  }
  // Probabilities: a row's chunk holds what a lane needs for a product, of keys that the
  // reading of the values gives it: of 16 keys (WIDE) 4g .. 4g + 3 and 8 + 4g .., which
  // are a lane's own scores; of 32 keys 4g .. 4g + 3 and 16 + 4g ...
  const int prow = rg * QR * TR + li, psw = (li >> 1) & 7;
  const uint32_t pw = prow * 128 + (((WIDE ? kg * 4 + lg : (kg >> 1) * 4 + lg) ^ psw) << 4) + (WIDE ? 0 : (kg & 1) * 8);
  const uint32_t pr = li * 128 + ((lg ^ psw) << 4);
  const float scale = a.scale_log2;
  Loader ld(a, wid, lane, lds_addr(lds.ring));
  const bool early = !WIDE || a.n_rb == 1;
  static_assert(!WIDE || Loader::N <= KS / 3 + KT / DS * CB / 2, "the loads are out before the next addresses come");

  for (int at = start; at < stop;) {
    const int len = __builtin_amdgcn_readfirstlane(len_of(a, b));
    const int tiles = ends.tiles(len, kLatTile);
    const int t1 = min(tiles, t0 + (stop - at));
    LatPiece pc;
    pc.b = b;
    pc.len = len;
    pc.t0 = t0;
    pc.t1 = t1;
    pc.slot = t0 == 0 && t1 == tiles ? -1 : ((int64_t)rb * a.W + rj) * 2 + (at == start ? 0 : 1);
    const int end = ends(len);
    ld.sequence(b, end);

    if (a.parent != nullptr) lat_tree<256>(a, b, m_lo, m_hi - m_lo + 1, reinterpret_cast<int16_t*>(lds.p), lds.vis);

    u32x4 qf[QR][KS];
    Acc acc[RB][CB];
    float mx[RB], ls[QR];
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      mx[i] = kNegInf;
#pragma unroll
      for (int c = 0; c < CB; ++c) acc[i][c] = Acc{};
    }
#pragma unroll
    for (int i = 0; i < QR; ++i) ls[i] = 0.f;
    bool hides = false;
    if (end > 0) {
      // The queries come through the other buffer (a load that ends in registers would be
      // waited for at its first use, in the loop, and the tiles in flight with it).
      const uint32_t other = (uint32_t)((t0 + 1) & 1) * L::TILE;
      if (wid * 16 < ROWS) {
        const uint64_t at = ld.queries(rb * ROWS);
        ld.all(other, at);
      }
      const uint64_t at = ld.keys(t0 * KT);
      ld.all((uint32_t)(t0 & 1) * L::TILE, at);
      wait_vmcnt<0>();
      barrier_lds();
      const uint8_t* qt = lds.ring + other;
#pragma unroll
      for (int i = 0; i < QR; ++i)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int x = ks < KSN ? ks * DS / 8 : (ks - KSN) * DS / 8;
          qf[i][ks] = ks < KSN ? *reinterpret_cast<const u32x4*>(qt + (rg * QR + i) * TR * L::NB + (qofs ^ ((x & 15) << 4)) + (x >> 4) * 256)
                               : *reinterpret_cast<const u32x4*>(qt + (rg * QR + i) * TR * L::RB + (qrofs ^ (x << 4)));
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      // (The upper half of the registers: products read it, other instructions do not.)
      if constexpr (WIDE && DC == 512) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+a"(qf[0][ks]));
      }
    }
    uint64_t apart = 0;  // a lane's address in the next tile, where they lie apart
    if (t0 + 1 < t1 && end > 0) apart = ld.keys((t0 + 1) * KT);
    for (int t = t0; t < t1 && end > 0; ++t) {
      // The next tile's loads go out as soon as its buffer is free (every wave done with
      // tile t - 1), before this tile's are waited for, so that the memory is never idle;
      // or, where several row blocks share the keys and the products take longer than the
      // memory, between the products, whose time covers theirs (72 of them take the vector
      // memory path of a CU 1700 cycles at once).
      const uint32_t next = (uint32_t)((t + 1) & 1) * L::TILE, stage = (uint32_t)(t & 1) * L::TILE;
      bool between = false;
      if (early || t + 1 == t1) barrier_lds();
      if (t + 1 < t1) {
        if (!early) {
          wait_vmcnt<0>();
          barrier_lds();
        }
        between = !early && ld.st2 != 0;
        if (!between) ld.all(next, apart);
        if (early) wait_vmcnt<Loader::N>();
      } else {
        wait_vmcnt<0>();
      }
      if (WIDE && (early || t + 1 == t1)) barrier_lds();  // (waves that share keys wait for each other's loads)
      asm volatile("" ::: "memory");
      // ---- scores of this wave's keys and rows ----------------------------------------
      Acc s[QR];
#pragma unroll
      for (int i = 0; i < QR; ++i) s[i] = Acc{};
      const uint32_t ko = again(kofs) + stage, ro = again(rofs) + stage;
      // The swizzle reaches the 16 chunks of 256 bytes; beyond, an offset.
      auto read_k = [&](int ks) {
        const int x = ks < KSN ? ks * DS / 8 : (ks - KSN) * DS / 8;
        return ks < KSN ? *reinterpret_cast<const u32x4*>(lds.ring + (ko ^ ((x & 15) << 4)) + (x >> 4) * 256)
                        : *reinterpret_cast<const u32x4*>(lds.ring + (ro ^ (x << 4)));
      };
      const uint32_t ln = again(lane);
      constexpr int KA = 6;  // operands ahead
      u32x4 kf[KA + 1];
#pragma unroll
      for (int x = 0; x < KA; ++x) kf[x] = read_k(x);
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        if (x + KA < KS) kf[(x + KA) % (KA + 1)] = read_k(x + KA);
#pragma unroll
        for (int i = 0; i < QR; ++i) s[i] = mfma<T>(kf[x % (KA + 1)], qf[i][x], s[i]);
        if (WIDE && x % 3 == 2 && x / 3 < Loader::N && between) ld.one(next, x / 3, ln);
        __builtin_amdgcn_sched_barrier(0);
      }
      const int kb = t * KT;
      const bool whole = lat_whole(a, len, m_lo, kb, KT);
      // Value v of a result is key 8 (v / 4) + 4 lg + v % 4 of the wave's.
      hides |= !whole;
      if (!whole) {
        uint32_t keep = 0;
#pragma unroll 1
        for (int i = 0; i < QR; ++i) {
          const int m = min(rb * ROWS + (rg * QR + i) * TR + li, a.R - 1) / a.G;
#pragma unroll 1
          for (int v = 0; v < NV; ++v)
            keep |= (lat_sees(a, len, m, lds.vis + (m - m_lo) * a.MW, kb + kg * (KT / KG) + 8 * (v / 4) + 4 * lg + v % 4) ? 1u : 0u)
                    << (NV * i + v);
        }
#pragma unroll
        for (int i = 0; i < QR; ++i)
#pragma unroll
          for (int v = 0; v < NV; ++v) s[i][v] = ((keep >> (NV * i + v)) & 1u) ? s[i][v] : kNegInf;
      }
      // ---- probabilities, relative to the maximum so far ------------------------------
      float ps[QR];
      auto top = [&](int i) {
        float m = s[i][0];
#pragma unroll
        for (int v = 1; v < NV; ++v) m = fmaxf(m, s[i][v]);
        return m;
      };
      auto max_of = [&](int i) { return WIDE && rg != 0 ? mx[RB - 1] : mx[i]; };
      auto probs = [&]() {
#pragma unroll
        for (int i = 0; i < QR; ++i) {
          const float m = max_of(i), m0 = m == kNegInf ? 0.f : m;
          float sum = 0.f;
          uint32_t w2[NV / 2];
#pragma unroll
          for (int v = 0; v < NV / 2; ++v) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[i][2 * v] - m0, scale, (float)SHIFT));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(s[i][2 * v + 1] - m0, scale, (float)SHIFT));
            sum += p0 + p1;
            w2[v] = pack2<T>(p0, p1);
          }
          ps[i] = sum;
          if constexpr (WIDE) {
            *reinterpret_cast<u32x4*>(lds.p + pw) = u32x4{w2[0], w2[1], w2[2], w2[3]};
            *reinterpret_cast<u32x4*>(lds.p + (pw ^ 32)) = u32x4{w2[NV / 2 - 4], w2[NV / 2 - 3], w2[NV / 2 - 2], w2[NV / 2 - 1]};
          } else {
            *reinterpret_cast<u32x2*>(lds.p + i * 2048 + pw) = u32x2{w2[0], w2[1]};
          }
        }
      };
      bool over = false;
#pragma unroll
      for (int i = 0; i < QR; ++i) over |= (top(i) - max_of(i)) * scale > kLatTau<T>;
      probs();
      const uint32_t up = __ballot(over) != 0ull ? 1 : 0;
      if (lane == 0) lds.flag[wid] = up;
      // The first operands of the output come while the waves meet.
      constexpr int PK = KT / DS, VA = 3;
      u32x4 pf[RB], pn[RB], vf[VA + 1];
      const uint32_t vo = again(vofs) + stage;
      auto read_p = [&](int k, u32x4 (&f)[RB]) {
#pragma unroll
        for (int i = 0; i < RB; ++i) f[i] = *reinterpret_cast<const u32x4*>(lds.p + i * TR * 128 + (pr ^ (k * DS * 2)));
      };
      auto read_v = [&](int x) {
        const uint8_t* vp = lds.ring + x / CB * DS * L::NB;
        const uint32_t o = vo ^ ((x % CB) * TR * 2), o8 = DS == 16 ? o ^ 32 : o;  // (the swizzle of keys 8 on)
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vp + o));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(vp + o8 + DS / 2 * L::NB));
        const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
        return u32x4{l2[0], l2[1], h2[0], h2[1]};
      };
      barrier_after_lds();
      const u32x4 fl = *reinterpret_cast<const u32x4*>(lds.flag);
      read_p(0, pf);
#pragma unroll
      for (int x = 0; x < VA; ++x) vf[x] = read_v(x);
      if (__builtin_amdgcn_readfirstlane(fl[0] | fl[1] | fl[2] | fl[3]) != 0) {
#pragma unroll
        for (int i = 0; i < QR; ++i) {
          const float m = groups_max<TR>(top(i));
          if (lg == 0) lds.red[kg][(rg * QR + i) * TR + li] = m;
        }
        barrier_after_lds();
#pragma unroll
        for (int i = 0; i < RB; ++i) {
          float mn = mx[i];
#pragma unroll
          for (int k = 0; k < KG; ++k) mn = fmaxf(mn, lds.red[k][i * TR + li]);
          const float al = mn == mx[i] ? 1.f : __builtin_amdgcn_exp2f((mx[i] - mn) * scale);
          mx[i] = mn;
          if (i / QR == rg) ls[i % QR] *= al;
#pragma unroll
          for (int c = 0; c < CB; ++c) acc[i][c] *= al;
        }
        probs();
        barrier_after_lds();
        read_p(0, pf);
      }
#pragma unroll
      for (int i = 0; i < QR; ++i) ls[i] += ps[i];
      // ---- this wave's columns -------------------------------------------------------
#pragma unroll
      for (int x = 0; x < PK * CB; ++x) {
        if (x % CB == 0 && x / CB + 1 < PK) read_p(x / CB + 1, (x / CB) % 2 ? pf : pn);
        if (x + VA < PK * CB) vf[(x + VA) % (VA + 1)] = read_v(x + VA);
        const u32x4 v = vf[x % (VA + 1)];
#pragma unroll
        for (int i = 0; i < RB; ++i) acc[i][x % CB] = mfma<T>(v, (x / CB) % 2 ? pn[i] : pf[i], acc[i][x % CB]);
        if (WIDE && KS / 3 + x < Loader::N && between) ld.one(next, KS / 3 + x, ln);
        // (The addresses of the tile after the next, while the products run.)
        if (x == PK * CB / 2 && t + 2 < t1) apart = ld.keys((t + 2) * KT);
        __builtin_amdgcn_sched_barrier(0);
      }
    }

    // ---- the piece's results ---------------------------------------------------------
    __syncthreads();
#pragma unroll
    for (int i = 0; i < QR; ++i) {
      const float x = groups_sum<TR>(ls[i]);
      if (lg == 0) lds.red[kg][(rg * QR + i) * TR + li] = x;
    }
    if (wid == 0 && lg == 0) {
#pragma unroll
      for (int i = 0; i < RB; ++i) lds.m[i * TR + li] = mx[i];
    }
    // An infinite or NaN value of a hidden key makes 0 * inf = NaN of rows that do not see it.
    float bad = 0.f;
    if (hides) {
#pragma unroll
      for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int c = 0; c < CB; ++c)
#pragma unroll
          for (int v = 0; v < NV; ++v) bad = fmaf(acc[i][c][v], 0.f, bad);  // (NaN of an infinite sum, too)
    }
    const uint32_t any = __ballot(bad != 0.f) != 0ull ? 1 : 0;
    if (lane == 0) lds.flag[wid] = any;
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int q4 = 0; q4 < NV / 4; ++q4) {
          const int r = i * TR + li, ch = wid * (DC / 16) + c * (TR / 4) + 2 * q4 + lg;
          *reinterpret_cast<f32x4*>(lds.ring + r * DC * 4 + ((ch ^ (r & 15)) << 4)) =
              f32x4{acc[i][c][4 * q4], acc[i][c][4 * q4 + 1], acc[i][c][4 * q4 + 2], acc[i][c][4 * q4 + 3]};
        }
    __syncthreads();
    const u32x4 fl = *reinterpret_cast<const u32x4*>(lds.flag);
    bool spreads = false;
    if (__builtin_amdgcn_readfirstlane(fl[0] | fl[1] | fl[2] | fl[3]) != 0)
      spreads = __builtin_amdgcn_readfirstlane(lat_spreads<T, DC>(lat_args(), pc, 0, rb, KT, m_lo, lds.span.wave));
    if (spreads)
      lat_exact_rows<T, DC>(lat_args(), pc, 0, rb, KT, m_lo, lds.vis, wid, ROWS, 4);
    else
      lat_store_rows<DC, ROWS, KG>(a, pc, rb, lds.ring, lds.m, lds.red, 1.f / (1 << SHIFT), reinterpret_cast<int64_t*>(lds.p),
                                   reinterpret_cast<float*>(lds.p + ROWS * 8));
    // Stores are done before the next piece counts its loads.
    wait_vmcnt<0>();
    __syncthreads();
    at += t1 - t0;
    t0 = 0;
    ++b;
  }
}

// ---- the partials joined -------------------------------------------------------------
// A workgroup takes (sequence, unit, `per` rows) at a time, a wave a row of DV / 64 values
// a lane, eight partials in flight; of one row (per = 1), the waves take eight partials each
// in turn and their sums are joined through LDS.  The sequences of a unit are all of them
// (cuts = 0), each sought among the lengths, or those that the starts of the ranges 1 to
// cuts = W - 1 cut, whichever are fewer: the lengths are read W times a unit at most, not B
// times (131072 sequences of up to four keys, both launches: 61.5 ms, now 2.0; 600 of up to 400,
// 128 heads: 170 us, now 156).
template <int N>
struct Count {
  static constexpr int value = N;
};
template <int DV>
__global__ void __launch_bounds__(256) latent_merge_kernel(const LatArgs a, int sh, uint32_t n, int per, int cuts) {
  constexpr int N = DV / 64;
  typedef float Row __attribute__((ext_vector_type(N)));
  __shared__ LatSpan span;
  __shared__ __attribute__((aligned(16))) float part[3 * DV];
  __shared__ float2 part_ml[3];
  lat_touch_args();
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const bool split = per == 1;
#pragma unroll 1
  for (uint32_t x = blockIdx.x; x < n; x += gridDim.x) {
    const uint32_t parts = (uint32_t)a.rpb / (uint32_t)per;
    uint32_t y = x / parts;
    const int i0 = (int)(x - y * parts) * per;
    const uint32_t unit = y % (uint32_t)(a.n_rb * a.Hk), item = y / (uint32_t)(a.n_rb * a.Hk);
    const int kvh = unit / (uint32_t)a.n_rb, rb = unit % (uint32_t)a.n_rb;
    const LatEnd ends(a, rb);
    const int total = lat_line<256>(a, ends, sh, cuts != 0 ? (int)item + 1 : 0, cuts != 0 ? -1 : (int)item, span);
    const LatCut cut(total, a.W);
    if (cuts != 0 && cut.begin((int)item + 1) >= total) continue;  // (a range of nothing)
    const int at = span.at, b = __builtin_amdgcn_readfirstlane(span.b);
    __syncthreads();
    const int j0 = cut.range_of(at), j1 = cut.range_of(at + ends.tiles(len_of(a, b), sh) - 1);
    // (One piece: written by its workgroup.  Of the ranges that begin within a sequence the first
    // one's workgroup joins it.)
    if (j0 == j1 || (cuts != 0 && j0 != (int)item)) continue;
#pragma unroll 1
    for (int i = split ? i0 : i0 + wid; i < i0 + per && rb * a.rpb + i < a.R; i += 4) {
      const int row = rb * a.rpb + i;
      // A range behind the first one begins with this sequence.
      const int64_t base = ((int64_t)unit * a.W * 2) * a.rpb + i;
      const int64_t first = cut.begin(j0) >= at ? 0 : a.rpb;
      float m = kNegInf, l = 0.f;
      Row o{};
      auto join = [&](auto count, int s0) {
        constexpr int U = decltype(count)::value;
        float2 ml[U];
        Row p[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int j = min(s0 + u, j1);
          const int64_t pr = base + (int64_t)j * 2 * a.rpb + (j == j0 ? first : 0);
          ml[u] = a.ml[pr];
          p[u] = *reinterpret_cast<const Row*>(a.opart + pr * DV + lane * N);
        }
        // (All in flight before the first is used: the compiler moves them to their uses.)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float t = p[u][N - 1];
          asm volatile("" : "+v"(t));
          p[u][N - 1] = t;
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < U; ++u) mn = fmaxf(mn, ml[u].x);
        const float f0 = mn == m ? 1.f : __builtin_amdgcn_exp2f((m - mn) * a.scale_log2);
        l *= f0;
        o *= f0;
        m = mn;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          // (Behind the last: nothing.  A piece without a key of this row holds zeros; one whose
          // maximum is -inf may hold NaN: of NaN scores, or of infinite values of no weight.)
          const bool none = s0 + u > j1;
          const float f = ml[u].x == mn ? 1.f : __builtin_amdgcn_exp2f((ml[u].x - mn) * a.scale_log2);
          l = fmaf(none ? 0.f : ml[u].y, f, l);
#pragma unroll
          for (int e = 0; e < N; ++e) o[e] = fmaf(none ? 0.f : p[u][e], f, o[e]);
        }
      };
      // (Two at once where there are no more: loads of nothing cost as much.)
      if (!split && j1 - j0 < 2) {
        join(Count<2>{}, j0);
      } else {
#pragma unroll 1
        for (int s0 = split ? j0 + 8 * wid : j0; s0 <= j1; s0 += split ? 32 : 8) join(Count<8>{}, s0);
      }
      if (split) {
        if (wid != 0) {
          *reinterpret_cast<Row*>(part + (wid - 1) * DV + lane * N) = o;
          if (lane == 0) part_ml[wid - 1] = make_float2(m, l);
        }
        __syncthreads();
        if (wid != 0) break;
        float mn = m;
#pragma unroll
        for (int u = 0; u < 3; ++u) mn = fmaxf(mn, part_ml[u].x);
        const float f0 = mn == m ? 1.f : __builtin_amdgcn_exp2f((m - mn) * a.scale_log2);
        l *= f0;
        o *= f0;
        m = mn;
#pragma unroll
        for (int u = 0; u < 3; ++u) {
          const float2 ml = part_ml[u];
          const float f = ml.x == mn ? 1.f : __builtin_amdgcn_exp2f((ml.x - mn) * a.scale_log2);
          l = fmaf(ml.y, f, l);
          o += *reinterpret_cast<const Row*>(part + u * DV + lane * N) * f;
        }
      }
      o *= l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
      const int pos = row / a.G, h = kvh * a.G + row - pos * a.G;
      const int64_t off = b_off(a, b, pos, h) + lane * N;
      if (a.out_vec && a.out_dtype == 2) {
        *reinterpret_cast<Row*>(reinterpret_cast<float*>(a.out) + off) = o;
      } else if (a.out_vec && N > 1) {
        uint32_t w[(N + 1) / 2];
#pragma unroll
        for (int e = 0; e + 1 < N; e += 2) w[e / 2] = a.out_dtype == 0 ? pack2<BF16>(o[e], o[e + 1]) : pack2<F16>(o[e], o[e + 1]);
        uint32_t* p = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + off);
        typedef uint32_t Out __attribute__((ext_vector_type((N + 1) / 2)));
        Out v;
#pragma unroll
        for (int e = 0; e < N / 2; ++e) v[e] = w[e];
        *reinterpret_cast<Out*>(p) = v;
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) store1(a, off + e, o[e]);
      }
      if (lane == 0 && a.lse != nullptr) a.lse[b * a.l_sb + (int64_t)pos * a.l_sm + (int64_t)h * a.l_sh] = lat_lse(a, m, l);
    }
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

hipError_t launch_latent_merge(const LatArgs& a, int sh, hipStream_t s) {
  if (a.W == 1) return hipSuccess;
  // One row a workgroup where rows are few and have many partials (both launches, in us: one
  // sequence of 32768 keys, 16 heads 29.3, with four rows 51.9; 2900 keys, 128 heads 19.8, 23.0),
  // four where there are some (40 of 2000 keys, 16 heads 32.7, with one 33.4, with 16 37.7; 32 of
  // 4000, 128 heads 72.3, 87.4, 73.3), 16 where the search of their pieces counts (8 trees of 64
  // nodes, 32 heads 153.5, with four 161.0).
  const int64_t units = (int64_t)a.Hk * a.n_rb, rows = a.B * units * a.rpb;
  int per = rows <= 1024 && a.W >= 8 * a.B ? 1 : (rows <= 8192 ? 4 : 16);
  const int cuts = a.W - 1 < a.B ? a.W - 1 : 0;
  const int64_t blocks = units * (cuts != 0 ? cuts : a.B);
  while (blocks * (a.rpb / per) > 0x7fffffff) per *= 2;  // (blocks are fewer than 2^30: the plan's range)
  const uint32_t n = (uint32_t)(blocks * (a.rpb / per));
  const dim3 grid((unsigned)(n < (1 << 20) ? n : 1 << 20)), block(256);
  switch (a.dv) {
    case 64: hipLaunchKernelGGL(latent_merge_kernel<64>, grid, block, 0, s, a, sh, n, per, cuts); break;
    case 128: hipLaunchKernelGGL(latent_merge_kernel<128>, grid, block, 0, s, a, sh, n, per, cuts); break;
    case 256: hipLaunchKernelGGL(latent_merge_kernel<256>, grid, block, 0, s, a, sh, n, per, cuts); break;
    default: hipLaunchKernelGGL(latent_merge_kernel<512>, grid, block, 0, s, a, sh, n, per, cuts); break;
  }
  return hipGetLastError();
}

}  // namespace dsv
