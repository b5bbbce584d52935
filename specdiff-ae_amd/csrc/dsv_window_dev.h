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

// The walks, at most M steps each (a parent < 0, >= M or equal to the node ends
// one, as in the tree split of dsv_attn.hip).  Every thread of the workgroup
// calls it; ends with a barrier.
template <int ROWS, int NT>
__device__ __forceinline__ void tree_rows(const WinArgs& a, int b, int n0, int r0, TreeLds<ROWS>& t) {
  const int M = a.M;
  for (int i = threadIdx.x; i < M; i += NT) {
    const int64_t o = b * a.par_sb + (int64_t)i * a.par_sm;
    const int64_t x = a.par_i64 ? reinterpret_cast<const int64_t*>(a.parent)[o]
                                : (int64_t) reinterpret_cast<const int32_t*>(a.parent)[o];
    t.par[i] = x < 0 || x >= M || x == i ? (int16_t)-1 : (int16_t)x;
  }
  __syncthreads();
  if (threadIdx.x < ROWS) {
    const int m = min(r0 + (int)threadIdx.x, a.R - 1) / a.G;
    uint64_t* vis = t.vis + threadIdx.x * kTreeMaxW;
    for (int w = 0; w < a.MW; ++w) vis[w] = 0;
    // The ancestor at h hops stands h positions before the row: seen for h < W.
    uint64_t word = 0;
    int at = m >> 6, h = 0;
    for (int x = m; x >= 0 && h <= M; x = t.par[x], ++h) {
      if (x >> 6 != at) {
        vis[at] |= word;
        word = 0;
        at = x >> 6;
      }
      if (h < a.W) word |= 1ull << (x & 63);
    }
    vis[at] |= word;
    const int depth = min(h - 1, M);
    t.depth[threadIdx.x] = depth;
    // And those at positions below the sinks' end.
    if (n0 < a.S) {
      h = 0;
      for (int x = m; x >= 0 && h <= depth; x = t.par[x], ++h)
        if (n0 + depth - h < a.S) vis[x >> 6] |= 1ull << (x & 63);
    }
  }
  __syncthreads();
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
__device__ __forceinline__ int64_t key_off(const WinArgs& a, int64_t sp, int64_t st, int n, int32_t page) {
  return a.pt != nullptr ? page * sp + (n & ((1 << a.ps_shift) - 1)) * st : n * st;
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

// Writes N consecutive output elements.
template <int N>
__device__ __forceinline__ void store_out(const WinArgs& a, int64_t off, const float (&x)[N]) {
  static_assert(N == 4 || N == 8, "");
  if (a.out_dtype == 2) {
    float* o = reinterpret_cast<float*>(a.out) + off;
    if (a.out_vec) {
#pragma unroll
      for (int i = 0; i < N; i += 4) *reinterpret_cast<f32x4*>(o + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = x[i];
    }
    return;
  }
  uint16_t* o = reinterpret_cast<uint16_t*>(a.out) + off;
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i)
    w[i] = a.out_dtype == 0 ? pack2<BF16>(x[2 * i], x[2 * i + 1]) : pack2<F16>(x[2 * i], x[2 * i + 1]);
  if (a.out_vec) {
    if constexpr (N == 8)
      *reinterpret_cast<u32x4*>(o) = u32x4{w[0], w[1], w[2], w[3]};
    else
      *reinterpret_cast<u32x2*>(o) = u32x2{w[0], w[1]};
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
  }
}

}  // namespace dsv
