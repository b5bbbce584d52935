// dsv_spec.hip — verification of drafted tokens against the target's
// probabilities, from given random numbers, on gfx950.
//
// Mathematics.  From the root, a node's children x_1, x_2, .. (index order)
// are tested in turn.  With w_0 = p, c_0 = 0, S_0 = 1 (p the target's row, q
// the draft's), child j is accepted iff u_j * S_{j-1} * q(x_j) < w_{j-1}(x_j);
// after a rejection the weights become w_j = max(w_{j-1} - S_{j-1} q, 0).
// Since max(max(a - b, 0) - c, 0) = max(a - b - c, 0) for b, c >= 0,
//     w_j = max(p - c_j q, 0),  c_j = c_{j-1} + S_{j-1},  S_j = sum w_j:
// the whole recursion is one scalar c, and a row is swept only for the mass
// S_j that a further sibling's test needs (none on a chain).  Without draft
// probabilities every child is a certain proposal (q one at its token):
// accepted iff u_j * R < p(x_j), R = 1 - the rejected children's
// probabilities, and the weights are p without those tokens.  Where no child
// is accepted the next token is the first v whose cumulative weight exceeds
// u_root * W.
//
// Everything is summed in 64 bits: an fp32 sum over 128256 entries is off by
// more than a token's mass, which would change the drawn token.  Sums run in a
// fixed order, so a call gives the same result every time.
//
// Layout.  The acceptance tests read two scalars a node; all M nodes' are
// gathered at once and wave 0 walks in LDS.  The last row's sweep is the large
// read.  One CU sweeps a row pair of 128256 entries in about 17 us, so with few
// trees a long row is shared out over several workgroups of 16 waves, each walking
// the tree by itself (no wait stands between the walk and the sweep), and a second
// launch, one wave a tree, draws from their sums; with a tree per CU, or a short
// row, the one workgroup draws as well.  64 chains of 5 over 128256 fp32 entries:
// one workgroup each 27 us, four each 19.5 (16.5 + 3.8).  The mass that a further
// sibling's test needs is not shared out: every workgroup of the tree sweeps the
// whole row for it (sampled trees of 64 nodes over 128256 entries, in a graph: one
// 23 to 25 us, four 38 to 48).  A wave sums a contiguous
// slot of the row, 8 entries a lane at a time with the next ones in flight.
//
// Reference context: draft/tree_verification.py:100-182 (the walk whose
// outputs are kept alike: path, tokens, winner, accept length, next token).

#include "dsv_internal.h"

namespace dsv {

namespace {

constexpr int kT = kSpecThreads;
constexpr int kW = kT / 64;
constexpr int kPer = kSpecSeg / 64;  // entries per lane and round of a sweep
template <typename E>
struct Load;
template <>
struct Load<float> {
  static __device__ __forceinline__ float at(const float* p) { return *p; }
};
template <>
struct Load<__bf16> {
  static __device__ __forceinline__ float at(const __bf16* p) { return (float)*p; }
};
template <>
struct Load<_Float16> {
  static __device__ __forceinline__ float at(const _Float16* p) { return (float)*p; }
};

// A probability entry: negative, infinite and NaN entries count as 0.
__device__ __forceinline__ float prob(float x) { return x > 0.f && x < __builtin_huge_valf() ? x : 0.f; }

// A given number in [0, 1): others are clamped (NaN to 0).
__device__ __forceinline__ double unit(float u) {
  const float hi = 0.99999994f;  // the largest fp32 below 1
  return u >= 0.f ? (double)(u < hi ? u : hi) : 0.0;
}

// x of the lane that DPP control CTRL names, 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
// Inclusive scan over a wave: shifts by 1, 2, 4, 8 inside the rows of 16, then
// the last lanes of rows 0 and 2, then of row 1, handed on.  (Through LDS
// permutes the six steps took 10 times as long, and a draw has four scans in a
// row.)
__device__ __forceinline__ double wave_scan(double x) {
  x += dpp<0x111, 0xf>(x);
  x += dpp<0x112, 0xf>(x);
  x += dpp<0x114, 0xf>(x);
  x += dpp<0x118, 0xf>(x);
  x += dpp<0x142, 0xa>(x);
  x += dpp<0x143, 0xc>(x);
  return x;
}

// x of a lane that the wave agrees on.
__device__ __forceinline__ double lane_of(double x, int l) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, l);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), l);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// What the remaining weights of a row are: max(p - c q, 0), or p without the
// rejected tokens.
template <typename E>
struct Rows {
  const E* p;
  const E* q;
  double c;
  const int32_t* rej;
  int nrej;
  int64_t V;
};

// N entries that a lane holds of 64 N consecutive ones that its wave covers from
// v0 on.  ROWS: 16-byte loads side by side over the lanes (whole lines; the order
// of a sum is free), else N consecutive entries per lane (the draw walks them in
// the vocabulary's order).  Rows need no alignment; entries past V are 0.
template <typename E, int N, bool ROWS>
struct Piece {
  static constexpr int VE = 16 / (int)sizeof(E) < N ? 16 / (int)sizeof(E) : N;
  static constexpr int NV = N / VE;
  typedef E vec __attribute__((ext_vector_type(VE), aligned(sizeof(E))));
  vec x[NV];
  static __device__ __forceinline__ int index(int e) {
    const int lane = threadIdx.x & 63;
    return ROWS ? (e / VE) * (64 * VE) + lane * VE + e % VE : lane * N + e;
  }
  __device__ __forceinline__ void load(const E* row, int64_t v0, int64_t V) {
    if (v0 + 64 * N <= V) {
#pragma unroll
      for (int k = 0; k < NV; ++k) x[k] = *reinterpret_cast<const vec*>(row + v0 + index(k * VE));
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) x[e / VE][e % VE] = v0 + index(e) < V ? row[v0 + index(e)] : (E)0.f;
    }
  }
  __device__ __forceinline__ float at(int e) const { return (float)x[e / VE][e % VE]; }
};

// Weights of this lane's entries of the wave's piece at v0.  CHECK: infinite
// entries count as 0; without it they are assumed absent (negative ones and NaN
// are 0 either way, p's by the maximum behind the product).
template <typename E, bool Q, bool CHECK, int N, bool ROWS>
__device__ __forceinline__ void weights(const Rows<E>& r, const Piece<E, N, ROWS>& p, const Piece<E, N, ROWS>& q, int64_t v0,
                                        double (&w)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    w[e] = (double)(CHECK ? prob(p.at(e)) : (Q ? p.at(e) : fmaxf(p.at(e), 0.f)));
    if constexpr (Q) w[e] = fmax(fma(-r.c, (double)(CHECK ? prob(q.at(e)) : fmaxf(q.at(e), 0.f)), w[e]), 0.0);
  }
  if constexpr (!Q) {
    // The rejected tokens among the wave's entries, found 64 at a time.
    const int lane = threadIdx.x & 63;
    for (int i = 0; i < r.nrej; i += 64) {
      const int64_t d = i + lane < r.nrej ? (int64_t)r.rej[i + lane] - v0 : -1;
      for (uint64_t in = __ballot(d >= 0 && d < 64 * N); in != 0; in &= in - 1) {
        const int at = __shfl((int)d, __builtin_ctzll(in));
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (Piece<E, N, ROWS>::index(e) == at) w[e] = 0.0;
      }
    }
  }
}

// The sums of the workgroup's 16 own slots (own per wave, step segments each, from
// slot first on) into LDS, their total in every thread, in a fixed order.  Bound by
// its VALU operations, 64-bit ones among them (a pair of 64000 entries takes one
// workgroup 4 us more than of 32000, in bf16 as in fp32): the check for infinite
// entries is one maximum over all of them, and the sweep runs again with the full
// check only if there is one.
template <typename E, bool Q, bool CHECK>
__device__ __forceinline__ double sweep_as(const Rows<E>& r, int first, int own, int step, double* sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  typedef Piece<E, kPer, true> Pc;
  const int64_t w0 = ((int64_t)first + wave * own) * step * kSpecSeg;
  const int64_t w1 = min(w0 + (int64_t)own * step * kSpecSeg, r.V);
  float mx = 0.f;
  Pc p, q, pn, qn;
  auto fetch = [&](int64_t v, Pc& x, Pc& y) {
    x.load(r.p, v, r.V);
    if (Q && r.c != 0.0) y.load(r.q, v, r.V);
  };
#pragma unroll
  for (int k = 0; k < Pc::NV; ++k) p.x[k] = pn.x[k] = q.x[k] = qn.x[k] = (E)0.f;
  if (w0 < w1) fetch(w0, p, q);
  __syncthreads();  // the sums before these have been read
  int64_t v = w0;
  for (int k = 0; k < own; ++k) {
    double s0 = 0.0, s1 = 0.0;
    for (int j = 0; j < step && v < w1; ++j, v += kSpecSeg) {
      if (v + kSpecSeg < w1) fetch(v + kSpecSeg, pn, qn);
      double w[kPer];
      weights<E, Q, CHECK, kPer, true>(r, p, q, v, w);
      if constexpr (!CHECK) {
#pragma unroll
        for (int e = 0; e < kPer; e += Q ? 1 : 2) mx = fmaxf(fmaxf(mx, p.at(e)), Q ? q.at(e) : p.at(e + 1));
      }
#pragma unroll
      for (int e = 0; e < kPer; e += 2) {
        s0 += w[e];
        s1 += w[e + 1];
      }
      p = pn;
      q = qn;
    }
    const double s = lane_of(wave_scan(s0 + s1), 63);
    if (lane == 0) sums[wave * own + k] = s;
  }
  // (Infinite entries are marked by an infinite sum.)
  const bool inf = __ballot(mx == __builtin_huge_valf()) != 0ull;
  if (lane == 0 && inf) sums[wave * own] = __builtin_huge_val();
  __syncthreads();
  static_assert(kSpecSlots == 64, "a lane per slot at most");
  return lane_of(wave_scan(lane < kW * own ? sums[lane] : 0.0), 63);
}

template <typename E, bool Q>
__device__ __forceinline__ double sweep(const Rows<E>& r, int first, int own, int step, double* sums) {
  const double s = sweep_as<E, Q, false>(r, first, own, step, sums);
  return s < __builtin_huge_val() ? s : sweep_as<E, Q, true>(r, first, own, step, sums);
}

// The next token from the remaining weights, whose nslot sums of step segments
// are given (in LDS or memory): the first v whose cumulative weight exceeds u W,
// W the total (the last one with a weight if rounding left none); -1 if W is 0.
// One wave: no barriers, and little code, which a kernel of this length fetches
// from memory line by line (by 4 waves with block scans it took 7 us, by 16 ten).
template <typename E, bool Q>
__device__ __forceinline__ int64_t draw(const Rows<E>& r, const double* sums, int nslot, int step, double u) {
  const int lane = threadIdx.x & 63;
  const int per = (nslot + 63) / 64;
  double mine = 0.0;
  for (int k = 0; k < per; ++k) mine += lane * per + k < nslot ? sums[lane * per + k] : 0.0;
  double inc = wave_scan(mine);
  const double W = lane_of(inc, 63);
  if (!(W > 0.0)) return -1;
  const double tau = u * W;
  // The lane whose slots carry the cumulative weight past tau, then the slot.
  uint64_t some = __ballot(mine > 0.0), past = __ballot(mine > 0.0 && inc > tau);
  int owner = past != 0 ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
  double run = lane_of(inc - mine, owner), base = run;
  int slot = 0;
  for (int k = 0; k < per; ++k) {
    const int i = owner * per + k;
    const double s = i < nslot ? sums[i] : 0.0;
    if (s > 0.0) {
      slot = i;
      base = run;
      if (run + s > tau) break;
    }
    run += s;
  }
  int64_t tok = 0;
  const int64_t v1 = min((int64_t)(slot + 1) * step * kSpecSeg, r.V);
  for (int64_t v = (int64_t)slot * step * kSpecSeg; v < v1; v += kSpecSeg) {
    typedef Piece<E, kPer, false> Pc;
    Pc p, q;
#pragma unroll
    for (int k = 0; k < Pc::NV; ++k) q.x[k] = (E)0.f;
    p.load(r.p, v, r.V);
    if (Q && r.c != 0.0) q.load(r.q, v, r.V);
    double w[kPer];
    weights<E, Q, true, kPer, false>(r, p, q, v, w);
    mine = 0.0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) mine += w[e];
    inc = wave_scan(mine);
    some = __ballot(mine > 0.0);
    past = __ballot(mine > 0.0 && base + inc > tau);
    if (some != 0) {
      owner = past != 0 ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
      // The owner's entry, in every lane for its own.
      double cum = base + (inc - mine);
      int at = 0;
      bool done = false;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        cum += w[e];
        if (w[e] > 0.0 && !done) {
          at = e;
          done = cum > tau;
        }
      }
      tok = v + owner * kPer + __builtin_amdgcn_readlane(at, owner);
      if (past != 0) return tok;
    }
    base += lane_of(inc, 63);
  }
  return tok;
}

// Where nothing is left of the weights (the target never exceeds the draft's
// share, or all of it was rejected) the token is drawn from the target's own
// row, and it is 0 if that has no weight either.  One wave, any waves beside it.
template <typename E>
__device__ __noinline__ int64_t draw_row(const E* p, int64_t V, double u) {
  const Rows<E> r{p, nullptr, 0.0, nullptr, 0, V};
  double W = 0.0;
  for (int64_t v = 0; v < V; v += kSpecSeg) {
    Piece<E, kPer, false> x;
    x.load(p, v, V);
    double w[kPer], mine = 0.0;
    weights<E, false, true, kPer, false>(r, x, x, v, w);
#pragma unroll
    for (int e = 0; e < kPer; ++e) mine += w[e];
    W += lane_of(wave_scan(mine), 63);
  }
  const int64_t nseg = (V + kSpecSeg - 1) / kSpecSeg;
  if (!(W > 0.0)) return 0;
  const int64_t t = draw<E, false>(r, &W, 1, (int)nseg, u);
  return t < 0 ? 0 : t;
}

struct Walk {
  double c, mass;   // share of q taken, mass of the remaining weights
  int node;         // the node whose children are being tested
  int next;         // first child index not tested yet
  int len;          // path length
  int nrej;         // rejected tokens of this node (given tokens)
  int sweep;        // the mass of the weights at c is needed
};

template <typename E, bool Q>
__global__ void __launch_bounds__(kT) spec_kernel(const SpecArgs a) {
  const int t = blockIdx.x / a.nwg, wg = blockIdx.x % a.nwg, M = a.M;
  const int64_t V = a.V;
  __shared__ int32_t par[kSpecMaxM], tok[kSpecMaxM], rej[kSpecMaxM];
  __shared__ float px[kSpecMaxM], qx[kSpecMaxM], un[kSpecMaxM];
  __shared__ int16_t path[kSpecMaxM];
  __shared__ double sums[kSpecSlots];
  __shared__ Walk wk;
  const E* P = reinterpret_cast<const E*>(a.target) + (int64_t)t * a.t_st;
  const E* Dp = Q ? reinterpret_cast<const E*>(a.dprobs) + (int64_t)t * a.q_st : nullptr;

  for (int i = threadIdx.x; i < M; i += kT) {
    int pe = -1;
    if (i > 0) {
      const int64_t r = a.parent[(int64_t)t * a.p_st + (int64_t)(i - 1) * a.p_sm];
      // -1 and the node's own place mean the root; others out of range: no parent.
      pe = r == -1 || r == i - 1 ? 0 : (r >= 0 && r < M - 1 ? (int)r + 1 : -1);
    }
    const int64_t x = a.draft[(int64_t)t * a.d_st + (int64_t)i * a.d_sm];
    const bool in = x >= 0 && x < V;
    par[i] = pe;
    tok[i] = in ? (int)x : -1;
    un[i] = a.uniform[(int64_t)t * a.u_st + (int64_t)i * a.u_sm];
    float p = 0.f, q = 0.f;
    if (pe >= 0 && in) {
      p = prob(Load<E>::at(P + (int64_t)pe * a.t_sm + x));
      if constexpr (Q) q = prob(Load<E>::at(Dp + (int64_t)pe * a.q_sm + x));
    }
    px[i] = p;
    qx[i] = q;
  }
  if (threadIdx.x == 0) {
    wk = Walk{0.0, 1.0, 0, 1, 1, 0, 0};
    path[0] = 0;
  }
  __syncthreads();

  // The walk: wave 0 in LDS; the whole workgroup joins for a mass.
  while (true) {
    if (threadIdx.x < 64) {
      const int lane = threadIdx.x;
      Walk w = wk;
      w.sweep = 0;
      for (int base = w.next & ~63; base < M && w.sweep == 0;) {
        const int i = base + lane;
        uint64_t kids = __ballot(i < M && i >= w.next && par[i] == w.node);
        bool moved = false;
        while (kids != 0) {
          const int k = base + __builtin_ctzll(kids);
          kids &= kids - 1;
          double wx;
          if constexpr (Q) {
            const double d = (double)px[k] - w.c * (double)qx[k];
            wx = d > 0.0 ? d : 0.0;
          } else {
            bool gone = false;  // a sibling with this token was rejected
            for (int r = lane; r < w.nrej; r += 64) gone |= rej[r] == tok[k];
            wx = __ballot(gone) != 0 ? 0.0 : (double)px[k];
          }
          const double qk = Q ? (double)qx[k] : 1.0;
          if (unit(un[k]) * w.mass * qk < wx) {
            w = Walk{0.0, 1.0, k, 1, w.len + 1, 0, 0};
            if (lane == 0) path[w.len - 1] = (int16_t)k;
            moved = true;
            break;
          }
          w.next = k + 1;
          if constexpr (Q) {
            w.c += w.mass;
            // The mass is needed if another child follows.
            bool more = false;
            for (int b2 = base; b2 < M && !more; b2 += 64) {
              const int j = b2 + lane;
              more = __ballot(j < M && j > k && par[j] == w.node) != 0;
            }
            if (more) {
              w.sweep = 1;
              break;
            }
          } else {
            if (wx > 0.0) {
              w.mass -= wx;
              if (lane == 0) rej[w.nrej] = tok[k];
              ++w.nrej;
              // Lanes read what lane 0 wrote.
              __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
              __builtin_amdgcn_wave_barrier();
              __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            }
          }
        }
        base = moved ? 0 : base + 64;
      }
      if (lane == 0) wk = w;
    }
    __syncthreads();
    if (!Q || wk.sweep == 0) break;
    if constexpr (Q) {
      const Rows<E> r{P + (int64_t)wk.node * a.t_sm, Dp + (int64_t)wk.node * a.q_sm, wk.c, rej, 0, V};
      const double s = sweep<E, Q>(r, 0, 1, a.step1, sums);
      if (threadIdx.x == 0) wk.mass = s;
      __syncthreads();
    }
  }

  const int node = wk.node, len = wk.len, nrej = Q ? 0 : wk.nrej;
  int64_t* info = a.out_info + (int64_t)t * a.oi_st;
  if (wg == 0) {
    for (int i = threadIdx.x; i < M; i += kT) {
      const int id = i < len ? path[i] : -1;
      a.out_path[(int64_t)t * a.op_st + i] = id;
      a.out_tok[(int64_t)t * a.ot_st + i] = id >= 0 ? a.draft[(int64_t)t * a.d_st + (int64_t)id * a.d_sm] : -1;
    }
    if (threadIdx.x == 0) {
      info[0] = node;
      info[1] = len - 1;
      info[3] = len;
    }
  }
  // The last node's remaining weights.
  Rows<E> r{P + (int64_t)node * a.t_sm, Q ? Dp + (int64_t)node * a.q_sm : nullptr, wk.c, rej, nrej, V};
  const int nsum = kW * a.own;
  sweep<E, Q>(r, wg * nsum, a.own, a.step, sums);
  if (a.nwg == 1) {
    if (threadIdx.x >= 64) return;
    int64_t tok = draw<E, Q>(r, sums, nsum, a.step, unit(un[0]));
    if (tok < 0) tok = draw_row<E>(r.p, V, unit(un[0]));
    if (threadIdx.x == 0) info[2] = tok;
    return;
  }
  if (threadIdx.x < nsum) a.part[((int64_t)t * a.nwg + wg) * nsum + threadIdx.x] = sums[threadIdx.x];
  if (wg == 0) {
    if (threadIdx.x == 0) a.state[t] = SpecState{wk.c, node, nrej};
    for (int i = threadIdx.x; i < nrej; i += kT) a.rej[(int64_t)t * M + i] = rej[i];
  }
}

// The draw from the sums that a tree's workgroups left.
template <typename E, bool Q>
__global__ void __launch_bounds__(64) spec_draw_kernel(const SpecArgs a) {
  const int t = blockIdx.x, nslot = a.nwg * kW * a.own;
  const SpecState st = a.state[t];
  const double u = unit(a.uniform[(int64_t)t * a.u_st]);
  const Rows<E> r{reinterpret_cast<const E*>(a.target) + (int64_t)t * a.t_st + (int64_t)st.node * a.t_sm,
                  Q ? reinterpret_cast<const E*>(a.dprobs) + (int64_t)t * a.q_st + (int64_t)st.node * a.q_sm : nullptr,
                  st.c, a.rej + (int64_t)t * a.M, st.nrej, a.V};
  int64_t tok = draw<E, Q>(r, a.part + (int64_t)t * nslot, nslot, a.step, u);
  if (tok < 0) tok = draw_row<E>(r.p, a.V, u);
  if (threadIdx.x == 0) a.out_info[(int64_t)t * a.oi_st + 2] = tok;
}

template <typename E, bool Q>
hipError_t launch_q(const SpecArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((spec_kernel<E, Q>), dim3((unsigned)(a.T * a.nwg)), dim3(kT), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.nwg == 1) return e;
  hipLaunchKernelGGL((spec_draw_kernel<E, Q>), dim3((unsigned)a.T), dim3(64), 0, s, a);
  return hipGetLastError();
}

template <typename E>
hipError_t launch_e(const SpecArgs& a, hipStream_t s) {
  return a.dprobs != nullptr ? launch_q<E, true>(a, s) : launch_q<E, false>(a, s);
}

}  // namespace

hipError_t launch_spec(const SpecArgs& a, hipStream_t s) {
  switch (a.dtype) {
    case 0: return launch_e<__bf16>(a, s);
    case 1: return launch_e<_Float16>(a, s);
    default: return launch_e<float>(a, s);
  }
}

}  // namespace dsv
