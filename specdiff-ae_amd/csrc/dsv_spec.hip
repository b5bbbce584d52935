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
// gathered at once and the walk runs in LDS.  The last row's sweep is the only
// large read: it is cut into sub-blocks of kSpecSub entries that the
// workgroups of a tree share out, each walking the tree by itself (the walk
// needs no other workgroup, so no launch or wait stands between it and the
// sweep).  A second launch, one workgroup a tree, finds the sub-block and the
// token.  The memory traffic is the last row of p (and q).
//
// Reference context: draft/tree_verification.py:100-182 (the walk whose
// outputs are kept alike: path, tokens, winner, accept length, next token).

#include "dsv_internal.h"

namespace dsv {

namespace {

constexpr int kT = kSpecThreads;
constexpr int kPer = kSpecSub / kT;  // entries per thread and sub-block

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

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// The sum of x over the workgroup, in every thread (scratch: one per wave).
__device__ __forceinline__ double block_sum(double x, double* scratch) {
  x = wave_sum(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
  __syncthreads();
  double s = scratch[0];
#pragma unroll
  for (int i = 1; i < kT / 64; ++i) s += scratch[i];
  return s;
}

// The inclusive scan of x over the workgroup's threads, and its total.
__device__ __forceinline__ double block_scan(double x, double* scratch, double& total) {
  double inc = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(inc, o);
    if ((int)(threadIdx.x & 63) >= o) inc += y;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 63) scratch[threadIdx.x >> 6] = inc;
  __syncthreads();
  total = 0.0;
  double before = 0.0;
#pragma unroll
  for (int i = 0; i < kT / 64; ++i) {
    if (i == (int)(threadIdx.x >> 6)) before = total;
    total += scratch[i];
  }
  return before + inc;
}

// kPer consecutive-by-vector entries of a row's sub-block: entry e of thread
// tid is v0 + (e / VE) * kT * VE + tid * VE + e % VE (VE entries per 16-byte
// load; rows need no alignment).  Entries past the row read as 0.
template <typename E>
struct Vec {
  static constexpr int VE = 16 / (int)sizeof(E);
  static constexpr int NV = kPer / VE;
  typedef E vec __attribute__((ext_vector_type(VE), aligned(sizeof(E))));
  static __device__ __forceinline__ int64_t index(int64_t v0, int e) {
    return v0 + (int64_t)(e / VE) * (kT * VE) + threadIdx.x * VE + e % VE;
  }
  static __device__ __forceinline__ void load(const E* row, int64_t v0, int64_t V, float (&x)[kPer]) {
    if (v0 + kSpecSub <= V) {
      vec t[NV];
#pragma unroll
      for (int k = 0; k < NV; ++k) t[k] = *reinterpret_cast<const vec*>(row + index(v0, k * VE));
#pragma unroll
      for (int e = 0; e < kPer; ++e) x[e] = prob((float)t[e / VE][e % VE]);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int64_t v = index(v0, e);
        x[e] = v < V ? prob(Load<E>::at(row + v)) : 0.f;
      }
    }
  }
};

// Weights of a sub-block's entries of this thread: max(p - c q, 0), or p
// without the dropped tokens (bits of the sub-block).
template <typename E, bool Q>
__device__ __forceinline__ void weights(const E* p, const E* q, double c, const uint32_t* drop, int64_t v0, int64_t V,
                                        double (&w)[kPer]) {
  float x[kPer];
  if constexpr (Q) {
    float y[kPer];
    Vec<E>::load(p, v0, V, x);
    if (c != 0.0) {
      Vec<E>::load(q, v0, V, y);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e) y[e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const double d = (double)x[e] - c * (double)y[e];
      w[e] = d > 0.0 ? d : 0.0;
    }
  } else {
    Vec<E>::load(p, v0, V, x);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      w[e] = (double)x[e];
      if (drop != nullptr) {
        const int i = (int)(Vec<E>::index(v0, e) - v0);
        if ((drop[i >> 5] >> (i & 31)) & 1u) w[e] = 0.0;
      }
    }
  }
}

// Bits of the rejected tokens inside a sub-block (every thread calls it).
__device__ __forceinline__ void mark_dropped(uint32_t* drop, const int32_t* rej, int nrej, int64_t v0) {
  __syncthreads();
  for (int i = threadIdx.x; i < kSpecSub / 32; i += kT) drop[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < nrej; i += kT) {
    const int64_t d = (int64_t)rej[i] - v0;
    if (d >= 0 && d < kSpecSub) atomicOr(&drop[d >> 5], 1u << (d & 31));
  }
  __syncthreads();
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
__global__ void __launch_bounds__(kT) spec_walk_kernel(const SpecArgs a) {
  const int t = blockIdx.x / a.nwg, wg = blockIdx.x % a.nwg, M = a.M;
  const int64_t V = a.V;
  __shared__ int32_t par[kSpecMaxM], tok[kSpecMaxM], rej[kSpecMaxM];
  __shared__ float px[kSpecMaxM], qx[kSpecMaxM], un[kSpecMaxM];
  __shared__ int16_t path[kSpecMaxM];
  __shared__ uint32_t drop[kSpecSub / 32];
  __shared__ double scratch[kT / 64];
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
      const E* p = P + (int64_t)wk.node * a.t_sm;
      const E* q = Dp + (int64_t)wk.node * a.q_sm;
      const double c = wk.c;
      double s = 0.0;
      for (int64_t v0 = 0; v0 < V; v0 += kSpecSub) {
        double w[kPer];
        weights<E, Q>(p, q, c, nullptr, v0, V, w);
#pragma unroll
        for (int e = 0; e < kPer; ++e) s += w[e];
      }
      s = block_sum(s, scratch);
      if (threadIdx.x == 0) wk.mass = s;
      __syncthreads();
    }
  }

  const int node = wk.node, len = wk.len, nrej = wk.nrej;
  const double c = wk.c;
  if (wg == 0) {
    for (int i = threadIdx.x; i < M; i += kT) {
      const int id = i < len ? path[i] : -1;
      a.out_path[(int64_t)t * a.op_st + i] = id;
      a.out_tok[(int64_t)t * a.ot_st + i] = id >= 0 ? a.draft[(int64_t)t * a.d_st + (int64_t)id * a.d_sm] : -1;
    }
    int32_t* rj = a.rej + (int64_t)t * M;
    if constexpr (!Q)
      for (int i = threadIdx.x; i < nrej; i += kT) rj[i] = rej[i];
    if (threadIdx.x == 0) {
      a.state[t] = SpecState{c, node, len, nrej, 0};
      int64_t* info = a.out_info + (int64_t)t * a.oi_st;
      info[0] = node;
      info[1] = len - 1;
      info[3] = len;
    }
  }

  // The last row's weights, one sum per sub-block.
  const E* p = P + (int64_t)node * a.t_sm;
  const E* q = Q ? Dp + (int64_t)node * a.q_sm : nullptr;
  for (int64_t j = wg; j < a.nsub; j += a.nwg) {
    const int64_t v0 = j * kSpecSub;
    if (!Q && nrej > 0) mark_dropped(drop, rej, nrej, v0);
    double w[kPer], s = 0.0;
    weights<E, Q>(p, q, c, !Q && nrej > 0 ? drop : nullptr, v0, V, w);
#pragma unroll
    for (int e = 0; e < kPer; ++e) s += w[e];
    s = block_sum(s, scratch);
    if (threadIdx.x == 0) a.part[(int64_t)t * a.nsub + j] = s;
  }
}

// The first entry of sub-block v0 whose cumulative weight exceeds tau, in
// the order of the vocabulary; the last entry with a weight if rounding left
// none; -1 if no entry has one.
template <typename E>
__device__ int64_t pick(const double (&w)[kPer], int64_t v0, double tau, double* scratch, int32_t* found) {
  using L = Vec<E>;
  // Vector k of every thread covers VE consecutive entries; the vectors of the
  // workgroup follow one another, then k + 1.
  double run = 0.0;
  if (threadIdx.x == 0) {
    found[0] = 0x7fffffff;
    found[1] = -1;
  }
  __syncthreads();
  int last = -1, hit = 0x7fffffff;
#pragma unroll
  for (int k = 0; k < L::NV; ++k) {
    double mine = 0.0;
#pragma unroll
    for (int e = 0; e < L::VE; ++e) mine += w[k * L::VE + e];
    double all = 0.0;
    const double inc = block_scan(mine, scratch, all);
    double cum = run + (inc - mine);
    run += all;
#pragma unroll
    for (int e = 0; e < L::VE; ++e) {
      const int i = (int)(L::index(v0, k * L::VE + e) - v0);
      cum += w[k * L::VE + e];
      if (w[k * L::VE + e] > 0.0) {
        last = i;
        if (cum > tau && hit == 0x7fffffff) hit = i;
      }
    }
  }
  atomicMin(&found[0], hit);
  atomicMax(&found[1], last);
  __syncthreads();
  const int h = found[0] != 0x7fffffff ? found[0] : found[1];
  return h < 0 ? -1 : v0 + h;
}

template <typename E, bool Q>
__global__ void __launch_bounds__(kT) spec_pick_kernel(const SpecArgs a) {
  const int t = blockIdx.x;
  const int64_t V = a.V;
  __shared__ uint32_t drop[kSpecSub / 32];
  __shared__ double scratch[kT / 64];
  __shared__ int32_t found[2];
  __shared__ int64_t sel;
  __shared__ double base_s;
  const SpecState st = a.state[t];
  const E* p = reinterpret_cast<const E*>(a.target) + (int64_t)t * a.t_st + (int64_t)st.node * a.t_sm;
  const E* q = Q ? reinterpret_cast<const E*>(a.dprobs) + (int64_t)t * a.q_st + (int64_t)st.node * a.q_sm : nullptr;
  const int32_t* rej = a.rej + (int64_t)t * a.M;
  double* part = a.part + (int64_t)t * a.nsub;
  const double u = unit(a.uniform[(int64_t)t * a.u_st]);
  double c = st.c;
  int nrej = Q ? 0 : st.nrej;

  // Thread i owns sub-blocks [i * nper, (i + 1) * nper): its sum, the
  // cumulative sum up to its end and the total.
  const int64_t nper = (a.nsub + kT - 1) / kT;
  double own = 0.0, inc = 0.0;
  auto total = [&]() {
    own = 0.0;
    for (int64_t j = 0; j < nper; ++j) {
      const int64_t x = threadIdx.x * nper + j;
      if (x < a.nsub) own += part[x];
    }
    double w = 0.0;
    inc = block_scan(own, scratch, w);
    return w;
  };
  double W = total();
  if (!(W > 0.0)) {
    // Nothing is left of the row (the target never exceeds the draft's share,
    // or all of it was rejected): the target's own row is drawn from.
    c = 0.0;
    nrej = 0;
    for (int64_t j = 0; j < a.nsub; ++j) {
      double w[kPer], s = 0.0;
      weights<E, Q>(p, q, c, nullptr, j * kSpecSub, V, w);
#pragma unroll
      for (int e = 0; e < kPer; ++e) s += w[e];
      s = block_sum(s, scratch);
      if (threadIdx.x == 0) part[j] = s;
    }
    __syncthreads();
    W = total();
  }
  const double tau = u * W;
  // The first owner whose end passes tau (the last one with a weight if
  // rounding left none), then its sub-block.
  if (threadIdx.x == 0) {
    found[0] = kT;
    found[1] = -1;
    sel = -1;
  }
  __syncthreads();
  if (own > 0.0) {
    if (inc > tau) atomicMin(&found[0], (int)threadIdx.x);
    atomicMax(&found[1], (int)threadIdx.x);
  }
  __syncthreads();
  if ((int)threadIdx.x == (found[0] < kT ? found[0] : found[1])) {
    double r = inc - own;
    for (int64_t j = 0; j < nper; ++j) {
      const int64_t x = threadIdx.x * nper + j;
      if (x >= a.nsub) break;
      const double s = part[x];
      if (s > 0.0) {
        sel = x;
        base_s = r;
        if (r + s > tau) break;
      }
      r += s;
    }
  }
  __syncthreads();
  int64_t tok = 0;  // a row without a positive entry draws token 0
  if (sel >= 0) {
    const int64_t v0 = sel * kSpecSub;
    if (nrej > 0) mark_dropped(drop, rej, nrej, v0);
    double w[kPer];
    weights<E, Q>(p, q, c, nrej > 0 ? drop : nullptr, v0, V, w);
    const int64_t r = pick<E>(w, v0, tau - base_s, scratch, found);
    if (r >= 0) tok = r;
  }
  if (threadIdx.x == 0) a.out_info[(int64_t)t * a.oi_st + 2] = tok;
}

template <typename E, bool Q>
hipError_t launch_q(const SpecArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.nwg * a.T));
  hipLaunchKernelGGL((spec_walk_kernel<E, Q>), grid, dim3(kT), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((spec_pick_kernel<E, Q>), dim3((unsigned)a.T), dim3(kT), 0, s, a);
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
