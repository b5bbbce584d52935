// dsv_latent_append.hip — new rows of a latent cache: norm, rotation and scatter, on
// gfx950.
//
// Token t's row is [ w * c / sqrt(mean(c^2) + eps) | x * cos + partner(x) * sin ]: the
// latent vector, normalised where a weight is given, and the key's rotated part; it goes
// to slot slots[t] of the cache.  The queries' rotated parts are rotated in the same
// launch.  partner(x) is rotate_half's (-x[d/2:], x[:d/2]) or, interleaved, (-x[1],
// x[0], -x[3], x[2], ..).  All of it is computed in fp32 and rounded once, when stored.
//
// Bound by reading and writing each row once.  A wave takes a token's latent vector (16
// bytes a lane and step, held in registers between the sum of squares and the product);
// a thread takes two chunks of a rotated row, half the row apart, which holds every
// element's partner in either form.
//
// Measured: 65536 tokens of 512 + 64 and the rotated parts of 16 heads, 452 MB: 95 us, 4.76
// TB/s of the 4.95 that a large copy reaches; 64 tokens: 3.5 us (the call 17).

#include "dsv_internal.h"

namespace dsv {

namespace {

template <typename E>
struct Vec;  // 16 bytes of E as floats
struct TagBF16 {};
struct TagF16 {};
template <>
struct Vec<TagBF16> {
  static constexpr int N = 8, ES = 2;
  static __device__ __forceinline__ void load(const void* p, float (&x)[8]) {
    const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(v[i] << 16);
      x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store(void* p, const float (&x)[8]) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bf2 r = {(__bf16)x[2 * i], (__bf16)x[2 * i + 1]};
      v[i] = __builtin_bit_cast(uint32_t, r);
    }
    *reinterpret_cast<u32x4*>(p) = v;
  }
};
template <>
struct Vec<TagF16> {
  static constexpr int N = 8, ES = 2;
  static __device__ __forceinline__ void load(const void* p, float (&x)[8]) {
    const f16x8 v = *reinterpret_cast<const f16x8*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
  }
  static __device__ __forceinline__ void store(void* p, const float (&x)[8]) {
    f16x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (_Float16)x[i];
    *reinterpret_cast<f16x8*>(p) = v;
  }
};
template <>
struct Vec<float> {
  static constexpr int N = 4, ES = 4;
  static __device__ __forceinline__ void load(const void* p, float (&x)[4]) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = v[i];
  }
  static __device__ __forceinline__ void store(void* p, const float (&x)[4]) {
    *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
  }
};

// The cache row of token t, nullptr for a slot out of range.
__device__ __forceinline__ char* row_of(const LatentAppendArgs& a, int64_t t, int es) {
  const int64_t s = a.slots_i64 ? reinterpret_cast<const int64_t*>(a.slots)[t] : (int64_t) reinterpret_cast<const int32_t*>(a.slots)[t];
  if (s < 0 || s >= a.n_slots) return nullptr;
  return static_cast<char*>(a.cache) + es * ((s >> a.ps_shift) * a.s_p + (s & ((1ll << a.ps_shift) - 1)) * a.s_t);
}

// NC: 16-byte chunks per lane of a latent vector.
template <typename E, int NC>
__global__ void __launch_bounds__(256) latent_append_kernel(const LatentAppendArgs a, int64_t c_blocks) {
  using V = Vec<E>;
  constexpr int N = V::N, ES = V::ES;
  if ((int64_t)blockIdx.x < c_blocks) {
    const int lane = threadIdx.x & 63;
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= a.T) return;
    char* row = row_of(a, t, ES);
    if (row == nullptr) return;
    const char* c = static_cast<const char*>(a.c) + ES * t * a.c_st;
    const int n = a.dc / N;
    float x[NC][N], sum = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[k][i] = 0.f;
      if (k * 64 + lane < n) V::load(c + 16 * (k * 64 + lane), x[k]);
#pragma unroll
      for (int i = 0; i < N; ++i) sum = fmaf(x[k][i], x[k][i], sum);
    }
    if (a.w != nullptr) {
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
      const float f = 1.f / sqrtf(sum / (float)a.dc + a.eps);
#pragma unroll
      for (int k = 0; k < NC; ++k)
        if (k * 64 + lane < n) {
          float g[N];
          V::load(static_cast<const char*>(a.w) + 16 * (k * 64 + lane), g);
#pragma unroll
          for (int i = 0; i < N; ++i) x[k][i] = x[k][i] * f * g[i];
        }
    }
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (k * 64 + lane < n) V::store(row + 16 * (k * 64 + lane), x[k]);
    return;
  }
  // ---- rotated rows: the key's and then the heads' of every token -----------------
  const int half = a.dr / (2 * N);
  const int64_t per = (int64_t)(1 + a.H) * half;
  const int64_t x = ((int64_t)blockIdx.x - c_blocks) * 256 + threadIdx.x;
  const int64_t t = x / per;
  if (t >= a.T) return;
  const int y = (int)(x - t * per), h = y / half - 1, c0 = y % half, c1 = c0 + half;
  const char* src;
  char* dst;
  if (h < 0) {
    src = static_cast<const char*>(a.pe) + ES * t * a.pe_st;
    dst = row_of(a, t, ES);
    if (dst == nullptr) return;
    dst += ES * (int64_t)a.dc;
  } else {
    src = static_cast<const char*>(a.q) + ES * (t * a.q_st + h * a.q_sh);
    dst = static_cast<char*>(a.qo) + ES * (t * a.qo_st + h * a.qo_sh);
  }
  float u[2][N], r[2][N];
  V::load(src + 16 * c0, u[0]);
  V::load(src + 16 * c1, u[1]);
  if (a.cos != nullptr) {
    int64_t p = t;
    if (a.pos != nullptr) p = a.pos_i64 ? reinterpret_cast<const int64_t*>(a.pos)[t] : (int64_t) reinterpret_cast<const int32_t*>(a.pos)[t];
    p = p < 0 ? 0 : (p < a.n_pos ? p : a.n_pos - 1);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = k == 0 ? c0 : c1;
      float cs[N], sn[N];
      if (a.tab_f32) {
        const char* pc = static_cast<const char*>(a.cos) + 4 * (p * a.cos_st + c * N);
        const char* ps = static_cast<const char*>(a.sin) + 4 * (p * a.sin_st + c * N);
#pragma unroll
        for (int q4 = 0; q4 < N / 4; ++q4) {
          float v4[4];
          Vec<float>::load(pc + 16 * q4, v4);
#pragma unroll
          for (int i = 0; i < 4; ++i) cs[4 * q4 + i] = v4[i];
          Vec<float>::load(ps + 16 * q4, v4);
#pragma unroll
          for (int i = 0; i < 4; ++i) sn[4 * q4 + i] = v4[i];
        }
      } else {
        V::load(static_cast<const char*>(a.cos) + ES * (p * a.cos_st + c * N), cs);
        V::load(static_cast<const char*>(a.sin) + ES * (p * a.sin_st + c * N), sn);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float o = a.interleaved ? ((i & 1) ? u[k][i - 1] : -u[k][i + 1 < N ? i + 1 : i]) : (k == 0 ? -u[1][i] : u[0][i]);
        r[k][i] = fmaf(u[k][i], cs[i], o * sn[i]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      r[0][i] = u[0][i];
      r[1][i] = u[1][i];
    }
  }
  V::store(dst + 16 * c0, r[0]);
  V::store(dst + 16 * c1, r[1]);
}

template <typename E>
void launch_e(const LatentAppendArgs& a, hipStream_t s) {
  const int64_t c_blocks = (a.T + 3) / 4;
  const int64_t items = a.T * (1 + a.H) * (a.dr / (2 * Vec<E>::N));
  const dim3 grid((unsigned)(c_blocks + (items + 255) / 256)), block(256);
  const int n = a.dc / Vec<E>::N;
  if (n <= 64)
    hipLaunchKernelGGL((latent_append_kernel<E, 1>), grid, block, 0, s, a, c_blocks);
  else if (n <= 128)
    hipLaunchKernelGGL((latent_append_kernel<E, 2>), grid, block, 0, s, a, c_blocks);
  else
    hipLaunchKernelGGL((latent_append_kernel<E, 8>), grid, block, 0, s, a, c_blocks);
}

}  // namespace

hipError_t launch_latent_append(const LatentAppendArgs& a, hipStream_t s) {
  if (a.dtype == 0)
    launch_e<TagBF16>(a, s);
  else if (a.dtype == 1)
    launch_e<TagF16>(a, s);
  else
    launch_e<float>(a, s);
  return hipGetLastError();
}

}  // namespace dsv
