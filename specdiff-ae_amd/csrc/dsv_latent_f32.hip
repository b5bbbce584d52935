// dsv_latent_f32.hip — latent attention in fp32, absorbed and expanded, on gfx950.
//
// The mathematics of dsv_latent.hip with keys of two parts, [kn | kr], and values of
// their own: absorbed, all three are the cache row (kr its end, v its beginning);
// expanded, kn and v are a head's and kr is shared.  Blocks of 16 rows of a key head,
// tiles of 64 keys.  Every product is an fp32 matrix product (16x16x4): wave w of four
// computes the scores of 16 keys and then a quarter of the output's columns.  Operands
// come straight from the caches (a wave's load takes 16 rows x 64 bytes, a tile's in flight
// together): no copy in LDS but the probabilities, held in fp32, and the tile's addresses.
// That is the form for few rows: nothing but its neighbours covers a tile's load, and each
// block of 16 rows reads all keys for itself.
//
// Measured (a large fp32 product reaches 153 TFLOP/s): three chunks of 5 tokens through up
// to 3001 keys, 20 heads, 256 + 32 wide: 24 + 5.5 us for the join, floor 3.7: a workgroup
// has one or two tiles, whose loads take a round trip and its products 4 us.  Four
// prompts of 77 tokens, 5 heads of 64 + 32: 15 + 5 us, bound by the same latencies.  Of many
// rows: four chunks of 64 tokens through 2000 keys, 16 heads of 512 + 64, 18 GFLOP: 304 us,
// 59 TFLOP/s (14 to 31 registers spill at 512); two of 200 tokens through 2000, 16 heads of 128 +
// 64, 7.8 GFLOP: 198 us, 39 TFLOP/s.

#include "dsv_latent_dev.h"

namespace dsv {

namespace {

constexpr float kTau = 8.0f;

template <int DN, int DR, int DV>
__global__ void __launch_bounds__(256, 1) latent_f32_kernel(const LatArgs a) {
  constexpr int KT = 1 << kLatTileF32, ROWS = 16;
  constexpr int SN = DN / 16, SR = DR / 16, CB = DV / 64;
  constexpr int PST = KT + 4;  // floats per row of probabilities
  __shared__ __attribute__((aligned(16))) float p_lds[ROWS * PST];
  __shared__ uint64_t vis[ROWS * (kTreeMaxM / 64)];
  __shared__ int16_t par[kTreeMaxM];
  __shared__ int64_t voff[KT];
  __shared__ float red[4][ROWS];
  __shared__ uint32_t flag[4];
  __shared__ LatSpan span;

  lat_touch_args();
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  int w = (int)blockIdx.x;
  const int rb = w % a.n_rb;
  w /= a.n_rb;
  const int kvh = w % a.Hk, rj = w / a.Hk;
  const LatEnd ends(a, rb);
  const int total = lat_line<256>(a, ends, kLatTileF32, rj, -1, span);
  const LatCut cut(total, a.W);
  const int start = cut.begin(rj), stop = cut.begin(rj + 1);
  if (start >= stop) return;
  int b = __builtin_amdgcn_readfirstlane(span.b);
  int t0 = __builtin_amdgcn_readfirstlane(span.off);

  const int m_lo = rb * ROWS / a.G, m_hi = (min((rb + 1) * ROWS, a.R) - 1) / a.G;
  const int row = rb * ROWS + li, r_me = min(row, a.R - 1), m_me = r_me / a.G, h_me = kvh * a.G + r_me - m_me * a.G;
  const float scale = a.scale_log2;

  for (int at = start; at < stop;) {
    const int len = __builtin_amdgcn_readfirstlane(len_of(a, b));
    const int tiles = ends.tiles(len, kLatTileF32);
    const int t1 = min(tiles, t0 + (stop - at));
    LatPiece pc;
    pc.b = b;
    pc.len = len;
    pc.t0 = t0;
    pc.t1 = t1;
    pc.slot = t0 == 0 && t1 == tiles ? -1 : (((int64_t)kvh * a.n_rb + rb) * a.W + rj) * 2 + (at == start ? 0 : 1);
    const int end = ends(len);
    if (a.parent != nullptr) lat_tree<256>(a, b, m_lo, m_hi - m_lo + 1, par, vis);
    const float* kn = reinterpret_cast<const float*>(a.kn.p) + b * a.kn.sb + kvh * a.kn.sh;
    const float* kr = reinterpret_cast<const float*>(a.kr.p) + b * a.kr.sb + kvh * a.kr.sh;
    const float* vb = reinterpret_cast<const float*>(a.v.p) + b * a.v.sb + kvh * a.v.sh;

    // A lane holds four consecutive entries of its row per step of 16 (the order of the
    // reduction is the same for both operands).
    f32x4 qf[SN + SR];
    const float* q = reinterpret_cast<const float*>(a.q) + b * a.q_sb + (int64_t)m_me * a.q_sm + (int64_t)h_me * a.q_sh + lg * 4;
#pragma unroll
    for (int s = 0; s < SN + SR; ++s) qf[s] = *reinterpret_cast<const f32x4*>(q + s * 16);
    f32x4 acc[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c) acc[c] = f32x4{};
    float mx = kNegInf, ls = 0.f;
    bool hides = false;

    auto key_at = [&](int t) { return min(t * KT + wid * 16 + li, end - 1); };
    int64_t page = a.pt != nullptr && end > 0 ? page_of(a, b, key_at(t0)) : 0;
    for (int t = t0; t < t1 && end > 0; ++t) {
      const int kb = t * KT;
      // ---- loads: the values' places go round through LDS, all of a tile in flight ------
      const int n = key_at(t);
      const float* k1 = kn + key_off(a, a.kn, n, page) + lg * 4;
      const float* k2 = kr + key_off(a, a.kr, n, page) + lg * 4;
      if (lg == 0) voff[wid * 16 + li] = key_off(a, a.v, n, page);
      __syncthreads();
      const float* vc = vb + wid * (DV / 4) + li;
      float vf[KT / 4][CB];
#pragma unroll
      for (int k4 = 0; k4 < KT / 4; ++k4) {
        const float* vr = vc + voff[k4 * 4 + lg];
#pragma unroll
        for (int c = 0; c < CB; ++c) vf[k4][c] = vr[c * 16];
      }
      f32x4 kf[SN + SR];
#pragma unroll
      for (int x = 0; x < SN + SR; ++x) kf[x] = *reinterpret_cast<const f32x4*>(x < SN ? k1 + x * 16 : k2 + (x - SN) * 16);
      if (a.pt != nullptr && t + 1 < t1) page = page_of(a, b, key_at(t + 1));
      // ---- scores of this wave's 16 keys -----------------------------------------------
      // (In sums of 64 products, added up with one in between, so that no add waits for a product:
      // a single chain of all of them rounds its partial sums, up to 8 times as large, as often.)
      f32x4 s{}, before{};
#pragma unroll
      for (int x = 0; x < SN + SR; x += 4) {
        f32x4 part{};
#pragma unroll
        for (int y = x; y < x + 4 && y < SN + SR; ++y) {
#pragma unroll
          for (int e = 0; e < 4; ++e) part = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[y][e], qf[y][e], part, 0, 0, 0);
        }
        s += before;
        before = part;
        __builtin_amdgcn_sched_barrier(0);  // (in the order in which the keys arrive)
      }
      s += before;
      const bool whole = lat_whole(a, len, m_lo, kb, KT);
      hides |= !whole;
      if (!whole) {
#pragma unroll
        for (int v = 0; v < 4; ++v)
          if (!lat_sees(a, len, m_me, vis + (m_me - m_lo) * a.MW, kb + wid * 16 + 4 * lg + v)) s[v] = kNegInf;
      }
      // ---- probabilities ---------------------------------------------------------------
      float ps = 0.f;
      auto probs = [&]() {
        const float m0 = mx == kNegInf ? 0.f : mx;
        float p[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) p[v] = __builtin_amdgcn_exp2f((s[v] - m0) * scale);
        ps = (p[0] + p[1]) + (p[2] + p[3]);
        *reinterpret_cast<f32x4*>(p_lds + li * PST + wid * 16 + lg * 4) = f32x4{p[0], p[1], p[2], p[3]};
      };
      const float m4 = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
      probs();
      const bool over = __ballot((m4 - mx) * scale > kTau) != 0ull;
      if (lane == 0) flag[wid] = over ? 1 : 0;
      __syncthreads();
      if ((flag[0] | flag[1] | flag[2] | flag[3]) != 0) {
        float mw = fmaxf(m4, __shfl_xor(m4, 16));
        mw = fmaxf(mw, __shfl_xor(mw, 32));
        if (lg == 0) red[wid][li] = mw;
        __syncthreads();
        const float mn = fmaxf(mx, fmaxf(fmaxf(red[0][li], red[1][li]), fmaxf(red[2][li], red[3][li])));
        const float al = mn == mx ? 1.f : __builtin_amdgcn_exp2f((mx - mn) * scale);
        mx = mn;
        ls *= al;
#pragma unroll
        for (int c = 0; c < CB; ++c) acc[c] *= al;
        probs();
        __syncthreads();
      }
      ls += ps;
      // ---- this wave's columns -----------------------------------------------------------
#pragma unroll
      for (int k4 = 0; k4 < KT / 4; ++k4) {
        const float pf = p_lds[li * PST + k4 * 4 + lg];
#pragma unroll
        for (int c = 0; c < CB; ++c) acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[k4][c], pf, acc[c], 0, 0, 0);
      }
      __syncthreads();
    }

    // ---- the piece's results ---------------------------------------------------------
    float lw = ls + __shfl_xor(ls, 16);
    lw += __shfl_xor(lw, 32);
    if (lg == 0) red[wid][li] = lw;
    // An infinite or NaN value of a hidden key makes 0 * inf = NaN of rows that do not see it.
    float bad = 0.f;
    if (hides) {
#pragma unroll
      for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int v = 0; v < 4; ++v) bad = fmaf(acc[c][v], 0.f, bad);  // (NaN of an infinite sum, too)
    }
    const bool any = __ballot(bad != 0.f) != 0ull;
    if (lane == 0) flag[wid] = any ? 1 : 0;
    __syncthreads();
    bool spreads = false;
    if ((flag[0] | flag[1] | flag[2] | flag[3]) != 0) spreads = lat_spreads<float, DV>(lat_args(), pc, kvh, rb, KT, m_lo, span.wave);
    if (spreads) {
      lat_exact_rows<float, DV>(lat_args(), pc, kvh, rb, KT, m_lo, vis, wid, ROWS, 4);
    } else if (row < a.R) {
      const float l = red[0][li] + red[1][li] + red[2][li] + red[3][li];
      if (pc.slot >= 0) {
        const int64_t prow = pc.slot * ROWS + li;
#pragma unroll
        for (int c = 0; c < CB; ++c) *reinterpret_cast<f32x4*>(a.opart + prow * DV + wid * (DV / 4) + c * 16 + lg * 4) = acc[c];
        if (wid == 0 && lg == 0) a.ml[prow] = make_float2(mx, l);
      } else {
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        const int64_t off = b * a.o_sb + (int64_t)m_me * a.o_sm + (int64_t)h_me * a.o_sh + wid * (DV / 4) + lg * 4;
#pragma unroll
        for (int c = 0; c < CB; ++c) {
          const float x[4] = {acc[c][0] * inv, acc[c][1] * inv, acc[c][2] * inv, acc[c][3] * inv};
          store4(a, off + c * 16, x);
        }
        if (wid == 0 && lg == 0 && a.lse != nullptr)
          a.lse[b * a.l_sb + (int64_t)m_me * a.l_sm + (int64_t)h_me * a.l_sh] = lat_lse(a, mx, l);
      }
    }
    __syncthreads();
    at += t1 - t0;
    t0 = 0;
    ++b;
  }
}

template <int DN, int DR, int DV>
void launch_w(const LatArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.n_rb * a.Hk * a.W));
  hipLaunchKernelGGL((latent_f32_kernel<DN, DR, DV>), grid, dim3(256), 0, s, a);
}

template <int DN>
void launch_dr(const LatArgs& a, hipStream_t s) {
  a.dr == 64 ? launch_w<DN, 64, DN>(a, s) : launch_w<DN, 32, DN>(a, s);
}

}  // namespace

hipError_t launch_latent_f32(const LatArgs& a, hipStream_t s) {
  switch (a.dn) {
    case 64: launch_dr<64>(a, s); break;
    case 128: launch_dr<128>(a, s); break;
    case 256: launch_dr<256>(a, s); break;
    default: launch_dr<512>(a, s); break;
  }
  return hipGetLastError();
}

}  // namespace dsv
