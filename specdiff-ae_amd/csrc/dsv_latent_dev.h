// dsv_latent_dev.h — device helpers of the latent attention's kernels.
#pragma once

#include "dsv_latent.h"
#include "dsv_window_dev.h"

namespace dsv {

// (Small code throughout: a kernel's instructions come from memory at its first pass
// over them, 64 bytes a time, which is most of what a short call takes.)
__device__ __forceinline__ int len_of(const LatArgs& a, int b) {
  if (a.seqlens == nullptr) return (int)a.n_keys;
  const int32_t* p = reinterpret_cast<const int32_t*>(a.seqlens) + ((int64_t)b << a.seqlens_i64);
  const int32_t lo = p[0], hi = a.seqlens_i64 ? p[1] : lo >> 31, n = (int)a.n_keys;
  return hi < 0 ? 0 : (hi > 0 || (uint32_t)lo > (uint32_t)n ? n : lo);
}

// Physical page of key n, clamped to the pool.
__device__ __forceinline__ int64_t page_of(const LatArgs& a, int b, int n) {
  const int64_t i = (int64_t)b * a.pt_sb + (n >> a.ps_shift);
  const int64_t p = a.pt_i64 ? reinterpret_cast<const int64_t*>(a.pt)[i] : (int64_t) reinterpret_cast<const int32_t*>(a.pt)[i];
  return p < 0 ? 0 : (p >= a.n_phys ? a.n_phys - 1 : p);
}

// Element offset of key n of a source, sequence and head aside.
__device__ __forceinline__ int64_t key_off(const LatArgs& a, const LatSrc& s, int n, int64_t page) {
  return a.pt != nullptr ? page * s.sp + (int64_t)(n & ((1 << a.ps_shift) - 1)) * s.st : (int64_t)n * s.st;
}

// Where a workgroup's range begins (or a sequence's tiles lie): filled by one thread.
struct LatSpan {
  int at;              // tiles before a sequence
  int b, off;          // sequence, tile within it
  int wave[16];        // scratch of the scan
};

// The line of a unit's tiles over the sequences: returns their number, and finds the
// sequence and tile at which range j begins (find_b < 0; none for a range of nothing),
// or the place of sequence find_b (`at`).
// Every thread of the workgroup calls it; ends with a barrier.
template <int NT>
__device__ __forceinline__ int lat_line(const LatArgs& a, const LatEnd& end, int sh, int j, int find_b, LatSpan& s) {
  const int per = (a.B + NT - 1) / NT;
  const int lo = min((int)threadIdx.x * per, a.B), hi = min(lo + per, a.B);
  int sum = 0;
#pragma unroll 1
  for (int b = lo; b < hi; ++b) sum += end.tiles(len_of(a, b), sh);
  int pre = sum, total = 0;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  if (a.B > 1) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(pre, o);
      if (lane >= o) pre += x;
    }
  }
  if (lane == (a.B > 1 ? 63 : 0)) s.wave[wid] = pre;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wid) pre += s.wave[w];
    total += s.wave[w];
  }
  pre -= sum;  // tiles before this thread's sequences
  // The thread that has it walks to it.
  const int start = LatCut(total, a.W).begin(j);
  if (find_b >= 0 ? find_b >= lo && find_b < hi : start >= pre && start < pre + sum) {
    int b = lo;
#pragma unroll 1
    for (;; ++b) {
      const int t = end.tiles(len_of(a, b), sh);
      if (find_b >= 0 ? b == find_b : start < pre + t) break;
      pre += t;
    }
    s.b = b;
    s.at = pre;
    s.off = start - pre;
  }
  __syncthreads();
  return total;
}

// The trees of a workgroup: parents of one sequence's nodes and, of the nodes
// [m0, m0 + n) that its rows belong to, the set of tree keys that each sees
// (itself and its ancestors), MW 64-bit words a node.  At most M steps a walk, so a
// cycle of parents ends it.  Called by every thread; ends with a barrier.
template <int NT>
__device__ __forceinline__ void lat_tree(const LatArgs& a, int b, int m0, int n, int16_t* par, uint64_t* vis) {
  for (int i = threadIdx.x; i < a.M; i += NT) {
    const int64_t o = (int64_t)b * a.par_sb + (int64_t)i * a.par_sm;
    const int64_t x = a.par_i64 ? reinterpret_cast<const int64_t*>(a.parent)[o]
                                : (int64_t) reinterpret_cast<const int32_t*>(a.parent)[o];
    par[i] = x >= 0 && x < a.M && x != i ? (int16_t)x : (int16_t)-1;
  }
  __syncthreads();
  if ((int)threadIdx.x < n) {
    uint64_t* v = vis + threadIdx.x * a.MW;
    for (int w = 0; w < a.MW; ++w) v[w] = 0;
    int h = 0;
    for (int x = m0 + threadIdx.x; x >= 0 && h < a.M; x = par[x], ++h) v[x >> 6] |= 1ull << (x & 63);
  }
  __syncthreads();
}

// Does the row of position m (tree: with set vis) see key n of a sequence?
__device__ __forceinline__ bool lat_sees(const LatArgs& a, int len, int m, const uint64_t* vis, int n) {
  const int n0 = len - a.M;
  if (!a.causal) return n < len;
  if (a.parent == nullptr) return n <= n0 + m;
  if (n < n0) return true;
  const int i = n - n0;
  return i >= 0 && i < a.M && n0 >= 0 && ((vis[i >> 6] >> (i & 63)) & 1);
}

// Is every key of the tile at kb seen by every row of positions m >= m_lo?
__device__ __forceinline__ bool lat_whole(const LatArgs& a, int len, int m_lo, int kb, int kt) {
  const int n0 = len - a.M;
  if (!a.causal) return kb + kt <= len;
  return a.parent != nullptr ? kb + kt <= n0 : kb + kt - 1 <= n0 + m_lo;
}

// A row's piece of `x` (four consecutive values at d0): the output's, or a partial's.
__device__ __forceinline__ void store4(const LatArgs& a, int64_t off, const float (&x)[4]) {
  if (a.out_dtype == 2) {
    float* o = reinterpret_cast<float*>(a.out) + off;
    if (a.out_vec) {
      *reinterpret_cast<f32x4*>(o) = f32x4{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = x[i];
    }
    return;
  }
  uint16_t* o = reinterpret_cast<uint16_t*>(a.out) + off;
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = a.out_dtype == 0 ? pack2<BF16>(x[2 * i], x[2 * i + 1]) : pack2<F16>(x[2 * i], x[2 * i + 1]);
  if (a.out_vec) {
    *reinterpret_cast<u32x2*>(o) = u32x2{w[0], w[1]};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
  }
}

// Element offset of an output row.
__device__ __forceinline__ int64_t b_off(const LatArgs& a, int b, int m, int h) {
  return b * a.o_sb + (int64_t)m * a.o_sm + (int64_t)h * a.o_sh;
}

__device__ __forceinline__ void store1(const LatArgs& a, int64_t off, float x) {
  if (a.out_dtype == 2)
    reinterpret_cast<float*>(a.out)[off] = x;
  else
    reinterpret_cast<uint16_t*>(a.out)[off] = (uint16_t)(a.out_dtype == 0 ? pack2<BF16>(x, x) : pack2<F16>(x, x));
}

// ln sum exp of a row from its maximum (a score) and its sum relative to it.
__device__ __forceinline__ float lat_lse(const LatArgs& a, float m, float l) {
  return l == 0.f ? kNegInf : (m * a.scale_log2 + __log2f(l)) * kLn2;
}

// The kernel's arguments where they lie (a pointer to the parameter itself would put
// a copy into scratch memory).
__device__ __forceinline__ const LatArgs* lat_args() {
  typedef const LatArgs __attribute__((address_space(4))) * Ptr;
  Ptr p = (Ptr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return (const LatArgs*)p;
}

// Touches every line of the arguments at once: they lie in host memory, and a load at
// each first use costs a round trip of its own.
__device__ __forceinline__ void lat_touch_args() {
  typedef const uint32_t __attribute__((address_space(4))) * Ptr;
  Ptr p = (Ptr)__builtin_amdgcn_kernarg_segment_ptr();
  constexpr int LINES = (sizeof(LatArgs) + 63) / 64;
  static_assert(LINES <= 8, "");
  uint32_t x[LINES];
#pragma unroll
  for (int i = 0; i < LINES; ++i) x[i] = p[min(i * 16, (int)sizeof(LatArgs) / 4 - 1)];
#pragma unroll
  for (int i = 0; i < LINES; ++i) asm volatile("" ::"s"(x[i]));
}

// One piece of a range: tiles [t0, t1) of sequence b of len keys, `slot` its
// partial (-1: the piece is all of its sequence's tiles).
struct LatPiece {
  int b, len, t0, t1;
  int64_t slot;
};

// Does a piece hold a value that its products spread to rows that do not see it, 0 * inf = NaN?
// Of the keys that some row of the block (positions from m_lo) does not see, any infinite or
// NaN one; of the last key, which stands in for those behind the end, an infinite one (what is
// NaN there is NaN anyway).  So NaN queries and NaN keys that all rows see need no second pass.
// A wave takes every fourth key; called by all 256 threads, behind a barrier.
template <typename T, int DV>
__device__ __noinline__ bool lat_spreads(const LatArgs* ap, const LatPiece pc, int kvh, int rb, int kt, int m_lo, int* flags) {
  typedef Elem<T> El;
  typedef typename El::type E;
  constexpr int N = DV / 64;
  const LatArgs& a = *ap;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, end = LatEnd(a, rb)(pc.len), n0 = pc.len - a.M;
  // The first key that not every row sees (of a tree, its first).
  const int hidden = !a.causal || (a.parent != nullptr && a.M == 1) ? end : a.parent != nullptr ? n0 : n0 + m_lo + 1;
  const E* vb = reinterpret_cast<const E*>(a.v.p) + pc.b * a.v.sb + kvh * a.v.sh;
  float odd = 0.f;
  for (int n = max(min(hidden, end - 1), pc.t0 * kt) + wid; n < min(end, pc.t1 * kt); n += 4) {
    const E* v = vb + key_off(a, a.v, n, a.pt != nullptr ? page_of(a, pc.b, n) : 0) + lane * N;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float x = El::get(v[e]);
      if (n >= hidden || x == x) odd = fmaf(x, 0.f, odd);
    }
  }
  const bool any = __ballot(odd != 0.f) != 0ull;
  if (lane == 0) flags[wid] = any ? 1 : 0;
  __syncthreads();
  return (flags[0] | flags[1] | flags[2] | flags[3]) != 0;
}

// Rows [i0, i1) by step of a block once more, by one wave, from memory and without
// matrix products: where a value that some rows see and others do not is infinite or
// NaN (in the product 0 * inf would reach those others).  A lane takes a key of 64
// for the scores and DV / 64 columns for the sums.
template <typename T, int DV>
__device__ __noinline__ void lat_exact_rows(const LatArgs* ap, const LatPiece pc, int kvh, int rb, int kt, int m0, const uint64_t* vis,
                                            int i0, int i1, int step) {
  typedef Elem<T> El;
  typedef typename El::type E;
  constexpr int N = DV / 64;
  const LatArgs& a = *ap;
  const int lane = threadIdx.x & 63, b = pc.b;
  const int end = min(LatEnd(a, rb)(pc.len), pc.t1 * kt);
  const E* kn = reinterpret_cast<const E*>(a.kn.p) + b * a.kn.sb + kvh * a.kn.sh;
  const E* kr = reinterpret_cast<const E*>(a.kr.p) + b * a.kr.sb + kvh * a.kr.sh;
  const E* vb = reinterpret_cast<const E*>(a.v.p) + b * a.v.sb + kvh * a.v.sh;
  for (int i = i0; i < i1; i += step) {
    const int r = rb * a.rpb + i;
    if (r >= a.R) break;
    const int m = r / a.G, h = kvh * a.G + r - m * a.G;
    const E* q = reinterpret_cast<const E*>(a.q) + b * a.q_sb + (int64_t)m * a.q_sm + (int64_t)h * a.q_sh;
    float mx = kNegInf, l = 0.f, o[N];
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = 0.f;
    for (int n0 = pc.t0 * kt; n0 < end; n0 += 64) {
      const int n = min(n0 + lane, end - 1);
      const bool seen = n0 + lane < end && lat_sees(a, pc.len, m, vis + (m - m0) * a.MW, n);
      const int64_t page = a.pt != nullptr ? page_of(a, b, n) : 0;
      const int64_t vo = key_off(a, a.v, n, page);
      float s = kNegInf;
      if (seen) {
        s = 0.f;
        const E* k = kn + key_off(a, a.kn, n, page);
        for (int d = 0; d < a.dn; ++d) s = fmaf(El::get(q[d]), El::get(k[d]), s);
        k = kr + key_off(a, a.kr, n, page);
        for (int d = 0; d < a.dr; ++d) s = fmaf(El::get(q[a.dn + d]), El::get(k[d]), s);
      }
      float mt = s;
#pragma unroll
      for (int y = 1; y < 64; y <<= 1) mt = fmaxf(mt, __shfl_xor(mt, y));
      const float mn = fmaxf(mx, mt), ms = mn == kNegInf ? 0.f : mn;
      const float al = mx == kNegInf ? 0.f : __builtin_amdgcn_exp2f((mx - mn) * a.scale_log2);
      mx = mn;
      const float p = seen ? __builtin_amdgcn_exp2f((s - ms) * a.scale_log2) : 0.f;
      float ps = p;
#pragma unroll
      for (int y = 1; y < 64; y <<= 1) ps += __shfl_xor(ps, y);
      l = l * al + ps;
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] *= al;
      for (uint64_t left = __ballot(seen); left != 0; left &= left - 1) {
        const int src = __builtin_ctzll(left);
        const float pn = __shfl(p, src);
        const E* v = vb + (int64_t)__shfl((long long)vo, src) + lane * N;
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = fmaf(pn, El::get(v[e]), o[e]);
      }
    }
    if (pc.slot >= 0) {
      const int64_t pr = pc.slot * a.rpb + i;
#pragma unroll
      for (int e = 0; e < N; ++e) a.opart[pr * DV + lane * N + e] = o[e];
      if (lane == 0) a.ml[pr] = make_float2(mx, l);
      continue;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    const int64_t off = b * a.o_sb + (int64_t)m * a.o_sm + (int64_t)h * a.o_sh + lane * N;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float x = o[e] * inv;
      if (a.out_dtype == 2)
        reinterpret_cast<float*>(a.out)[off + e] = x;
      else
        reinterpret_cast<uint16_t*>(a.out)[off + e] = (uint16_t)(a.out_dtype == 0 ? pack2<BF16>(x, x) : pack2<F16>(x, x));
    }
    if (lane == 0 && a.lse != nullptr) a.lse[b * a.l_sb + (int64_t)m * a.l_sm + (int64_t)h * a.l_sh] = lat_lse(a, mx, l);
  }
}

}  // namespace dsv
