// dsv_window_dev.h — device helpers of the windowed attention's kernels.
#pragma once

#include "dsv_window.h"

namespace dsv {

constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kLn2 = 0.69314718055994530942f;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<BF16>(float lo, float hi) {
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  bf2 r = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(uint32_t, r);
}
template <>
__device__ __forceinline__ uint32_t pack2<F16>(float lo, float hi) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  h2 r = {(_Float16)lo, (_Float16)hi};
  return __builtin_bit_cast(uint32_t, r);
}
template <typename T>
__device__ __forceinline__ float unpack1(uint16_t x);
template <>
__device__ __forceinline__ float unpack1<BF16>(uint16_t x) {
  return __uint_as_float((uint32_t)x << 16);
}
template <>
__device__ __forceinline__ float unpack1<F16>(uint16_t x) {
  return (float)__builtin_bit_cast(_Float16, x);
}
// Nonzero where a half of x is infinite or NaN (bits 15 and 31).
template <typename T>
__device__ __forceinline__ uint32_t nonfinite2(uint32_t x);
template <>
__device__ __forceinline__ uint32_t nonfinite2<BF16>(uint32_t x) {
  return ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}
template <>
__device__ __forceinline__ uint32_t nonfinite2<F16>(uint32_t x) {
  return ((x & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}

// fp16 probabilities are held times 2^N of this, N the power that a kernel's own
// bound on them leaves room for: below 2^-14 fp16 loses bits and below 2^-25 all of
// them, and a key 17 above 2^18 others (whose sum is 2^18 e^-17 = 0.01 of its own
// weight) would hide them.  bf16 has fp32's range.
template <typename T, int N>
constexpr int kProbShift = 0;
template <int N>
constexpr int kProbShift<F16, N> = N;

// A running maximum from here on: the product of a score and the exponent's scale is
// off by 2^-24 of itself, so a probability by 2^0.25 at 2^22 (a factor that a row's
// sum shares) and by more than fp16, later fp32, holds beyond.  Such rows are
// computed by exact_rows, which takes differences of scores.
__device__ __forceinline__ bool far_score(float m) {
  return fabsf(m) >= 4194304.f && fabsf(m) < __builtin_huge_valf();
}

// Lanes of a wave read LDS that other lanes of it wrote (LDS operations of a
// wave execute in order; this keeps the compiler from moving them).
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// One query row.
struct Row {
  int m, g;
};
__device__ __forceinline__ Row row_of(const WinArgs& a, int r) {
  Row w;
  w.m = r / a.G;
  w.g = r - w.m * a.G;
  return w;
}

// A workgroup's rows of a tree, in LDS: each row's depth and the set of tree keys
// that it sees, MW = ceil(M / 64) words.  Every workgroup walks up its rows'
// parents by itself (about a microsecond beside the latencies of its first
// loads; a kernel of its own before the attention took 5 us and a launch).
template <int ROWS>
struct TreeLds {
  int16_t par[kTreeMaxM];
  int depth[ROWS];
  uint64_t vis[ROWS * kTreeMaxW];
};

// A barrier behind the waves' LDS operations alone: loads into LDS stay in flight.
__device__ __forceinline__ void barrier_after_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// This thread's parents, of up to kTreeMaxM in the workgroup (a parent < 0, >= M or
// equal to the node: -1); none for b < 0.
template <int NT>
struct TreeParents {
  static constexpr int N = (kTreeMaxM + NT - 1) / NT;
  int16_t p[N];
  __device__ __forceinline__ TreeParents(const WinArgs& a, int b) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = k * NT + (int)threadIdx.x;
      p[k] = -1;
      if (b < 0 || i >= a.M) continue;
      const int64_t o = b * a.par_sb + (int64_t)i * a.par_sm;
      const int64_t x = a.par_i64 ? reinterpret_cast<const int64_t*>(a.parent)[o]
                                  : (int64_t) reinterpret_cast<const int32_t*>(a.parent)[o];
      if (x >= 0 && x < a.M && x != i) p[k] = (int16_t)x;
    }
  }
};

// The walks, at most M nodes each (a row that leads into a cycle has depth M - 1).  Every thread of the workgroup calls it; ends
// with a barrier.
template <int ROWS, int NT>
__device__ __forceinline__ void tree_rows(const WinArgs& a, const TreeParents<NT>& mine, int n0, int r0, TreeLds<ROWS>& t) {
  const int M = a.M;
#pragma unroll
  for (int k = 0; k < TreeParents<NT>::N; ++k)
    if (k * NT + (int)threadIdx.x < M) t.par[k * NT + threadIdx.x] = mine.p[k];
  barrier_after_lds();
  if (threadIdx.x < ROWS) {
    const int m = min(r0 + (int)threadIdx.x, a.R - 1) / a.G;
    uint64_t* vis = t.vis + threadIdx.x * kTreeMaxW;
    for (int w = 0; w < a.MW; ++w) vis[w] = 0;
    // The ancestor at h hops stands h positions before the row: seen for h < W.
    uint64_t word = 0;
    int at = m >> 6, h = 0;
    for (int x = m; x >= 0 && h < M; x = t.par[x], ++h) {
      if (x >> 6 != at) {
        vis[at] |= word;
        word = 0;
        at = x >> 6;
      }
      if (h < a.W) word |= 1ull << (x & 63);
    }
    vis[at] |= word;
    const int depth = h - 1;
    t.depth[threadIdx.x] = depth;
    // And those at positions below the sinks' end.
    if (n0 < a.S) {
      h = 0;
      for (int x = m; x >= 0 && h <= depth; x = t.par[x], ++h)
        if (n0 + depth - h < a.S) vis[x >> 6] |= 1ull << (x & 63);
    }
  }
  barrier_after_lds();
}

// The keep word of a row at position pos for the tile at key kb: bit i = key
// kb + i is seen (vis: the row's tree keys, where there is a tree).
__device__ __forceinline__ uint32_t keep_word(const WinArgs& a, const uint64_t* vis, int pos, int kb, int n0) {
  const uint32_t win = ~win_below(pos - a.W + 1 - kb) | win_below(a.S - kb);
  if (a.parent == nullptr) return win & win_below(pos + 1 - kb);
  uint32_t keep = win & win_below(n0 - kb);
  if (kb + 32 > n0) {
    // Tree keys: bits [kb - n0, kb - n0 + 32) of the row's set.
    const int at = kb - n0;
    uint64_t x = 0;
    if (at < 0) {
      x = vis[0] << -at;
    } else if ((at >> 6) < a.MW) {
      const int i = at >> 6, sh = at & 63;
      x = vis[i] >> sh;
      if (sh > 32 && i + 1 < a.MW) x |= vis[i + 1] << (64 - sh);
    }
    keep |= (uint32_t)x;
  }
  return keep;
}

// Element offset of key n of the K or V half, for its physical page.
__device__ __forceinline__ int64_t key_off(const WinArgs& a, bool paged, int64_t sp, int64_t st, int n, int32_t page) {
  return paged ? page * sp + (n & ((1 << a.ps_shift) - 1)) * st : n * st;
}
__device__ __forceinline__ int32_t page_of(const WinArgs& a, int b, int n) {
  const int64_t i = (int64_t)b * a.pt_sb + (n >> a.ps_shift);
  int64_t p = a.pt_i64 ? reinterpret_cast<const int64_t*>(a.pt)[i] : (int64_t) reinterpret_cast<const int32_t*>(a.pt)[i];
  p = p < 0 ? 0 : (p >= a.n_phys ? a.n_phys - 1 : p);
  return (int32_t)p;
}

__device__ __forceinline__ int len_of(const WinArgs& a, int b) {
  int64_t n = a.n_keys;
  if (a.seqlens != nullptr) {
    const int64_t x = a.seqlens_i64 ? reinterpret_cast<const int64_t*>(a.seqlens)[b]
                                    : (int64_t) reinterpret_cast<const int32_t*>(a.seqlens)[b];
    n = x < 0 ? 0 : (x < n ? x : n);
  }
  return (int)n;
}

// Writes four consecutive output elements.
__device__ __forceinline__ void store_out(const WinArgs& a, int64_t off, const float (&x)[4]) {
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

// The kernel's arguments, loaded again where they are needed: what the epilogue
// reads does not stay in registers through the loop.
__device__ __forceinline__ const WinArgs& args_again() {
  typedef const WinArgs __attribute__((address_space(4))) * Ptr;
  Ptr p = (Ptr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const WinArgs*)p;
}

// Rows [i0, i1) by step of a workgroup once more, by one wave, from memory and
// without matrix products, where V holds infinities or NaN in keys that some of
// the rows do not see (in the product 0 * inf would reach those rows), or where a
// row's scores are so large that their product with the exponent's scale is off by
// powers of two (the maximum is held and subtracted as a score).  A lane takes a key
// of 64 for the scores and D / 64 columns for the sums.
template <typename T>
struct Elem {
  typedef uint16_t type;
  static __device__ __forceinline__ float get(uint16_t x) { return unpack1<T>(x); }
};
template <>
struct Elem<float> {
  typedef float type;
  static __device__ __forceinline__ float get(float x) { return x; }
};
template <typename T, int D, int ROWS>
__device__ __noinline__ void exact_rows(const WinArgs* ap, const TreeLds<ROWS>* tl, int b, int kvh, int split, int rb, int t0, int t1,
                                        int i0, int i1, int step) {
  typedef Elem<T> El;
  typedef typename El::type E;
  constexpr int N = D / 64;
  const WinArgs& a = *ap;
  const int n0 = len_of(a, b) - a.M;
  const WinKeys kl = win_keys(a.M, a.G, a.R, a.W, a.S, a.parent != nullptr, n0, rb * ROWS, ROWS);
  const int lane = threadIdx.x & 63;
  const E* kbase = reinterpret_cast<const E*>(a.k) + b * a.k_sb + kvh * a.k_sh;
  const E* vbase = reinterpret_cast<const E*>(a.v) + b * a.v_sb + kvh * a.v_sh;
  for (int i = i0; i < i1; i += step) {
    const int r = rb * ROWS + i;
    if (r >= a.R) break;
    const Row row = row_of(a, r);
    const int pos = n0 + (a.parent != nullptr ? tl->depth[i] : row.m);
    const int h = kvh * a.G + row.g;
    const E* q = reinterpret_cast<const E*>(a.q) + b * a.q_sb + (int64_t)row.m * a.q_sm + (int64_t)h * a.q_sh;
    float m = kNegInf, l = 0.f, o[N];
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = 0.f;
    for (int t = t0; t < t1; t += 2) {
      const int tt = t + (lane >> 5), x = lane & 31;
      const int kb = kl.base(min(tt, t1 - 1));
      const bool seen = tt < t1 && ((keep_word(a, tl->vis + i * kTreeMaxW, pos, kb, n0) >> x) & 1u);
      const int n = kl.read(kb + x);
      const bool paged = a.pt != nullptr;
      const int32_t page = paged ? page_of(a, b, n) : 0;
      const E* k = kbase + key_off(a, paged, a.k_sp, a.k_st, n, page);
      const int64_t vo = key_off(a, paged, a.v_sp, a.v_st, n, page);
      float s = kNegInf;
      if (seen) {
        s = 0.f;
#pragma unroll 4
        for (int d = 0; d < D; ++d) s = fmaf(El::get(q[d]), El::get(k[d]), s);
      }
      float mt = s;
#pragma unroll
      for (int y = 1; y < 64; y <<= 1) mt = fmaxf(mt, __shfl_xor(mt, y));
      const float mn = fmaxf(m, mt), ms = mn == kNegInf ? 0.f : mn;
      const float al = m == kNegInf ? 0.f : __builtin_amdgcn_exp2f((m - mn) * a.scale_log2);
      m = mn;
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
        const E* v = vbase + (int64_t)__shfl((long long)vo, src) + lane * N;
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = fmaf(pn, El::get(v[e]), o[e]);
      }
    }
    m *= a.scale_log2;
    if (a.splits > 1) {
      const int64_t pr = ((int64_t)(b * a.Hk + kvh) * a.splits + split) * a.R + r;
#pragma unroll
      for (int e = 0; e < N; ++e) a.opart[pr * D + lane * N + e] = o[e];
      if (lane == 0) a.ml[pr] = make_float2(m, l);
      continue;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    const int64_t off = b * a.o_sb + (int64_t)row.m * a.o_sm + (int64_t)h * a.o_sh + lane * N;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float x = o[e] * inv;
      if (a.out_dtype == 2)
        reinterpret_cast<float*>(a.out)[off + e] = x;
      else
        reinterpret_cast<uint16_t*>(a.out)[off + e] = (uint16_t)(a.out_dtype == 0 ? pack2<BF16>(x, x) : pack2<F16>(x, x));
    }
    if (lane == 0 && a.lse != nullptr)
      a.lse[b * a.l_sb + (int64_t)row.m * a.l_sm + (int64_t)h * a.l_sh] = l == 0.f ? kNegInf : (m + __log2f(l)) * kLn2;
  }
}

}  // namespace dsv
