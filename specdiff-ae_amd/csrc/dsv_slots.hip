// dsv_slots.hip — block tables and slot maps from request lengths, on gfx950.
//
// Request i names a sequence of len tokens, of which the last k are new.  In request
// order the new tokens stand at cu[i] .. cu[i + 1]; token t of request i has position
// p = len - (cu[i + 1] - t) and its place in the page pool is page_table[p / page] *
// page + p % page.  The requests' page lists come out as rows of their own.
//
// Bound by latencies: the chain seqs -> lengths -> scan -> page -> store.  Up to
// kSlotInline requests every workgroup scans all the lengths for itself (a few KiB out
// of L2; a launch of its own for the scan would cost more), finds its tokens'
// requests by bisection in LDS and writes its share of tokens and table entries.  Beyond, a
// first launch writes cu and the second bisects in it.
//
// Measured: 48 requests with a token each 7.4 us, 512 requests with up to 1000 tokens each
// (300000 places, 5.2 MB) 8.3 us; the call from Python takes 17.  Two launches: 4000 requests
// with a token each 18 + 6 us, 131072 488 + 51: of the scan's one workgroup a thread has n / 256
// requests, one after the other.

#include "dsv_internal.h"

namespace dsv {

namespace {

__device__ __forceinline__ int64_t at(const PageIndex& x, int64_t i) {
  return x.is64 ? reinterpret_cast<const int64_t*>(x.p)[i * x.stride] : (int64_t) reinterpret_cast<const int32_t*>(x.p)[i * x.stride];
}

struct Request {
  int64_t seq;   // -1: none (an index out of range)
  int64_t len, k;
};
__device__ __forceinline__ Request request(const SlotArgs& a, int i) {
  Request r;
  r.seq = a.seqs.p != nullptr ? at(a.seqs, i) : i;
  r.len = r.k = 0;
  if (r.seq < 0 || r.seq >= a.B) {
    r.seq = -1;
    return r;
  }
  const int64_t x = a.lens_i64 ? reinterpret_cast<const int64_t*>(a.lens)[r.seq] : (int64_t) reinterpret_cast<const int32_t*>(a.lens)[r.seq];
  const int64_t most = a.n_log << a.ps_shift;
  r.len = x < 0 ? 0 : (x < most ? x : most);
  const int64_t k = at(a.news, i);
  r.k = k < 0 ? 0 : (k < r.len ? k : r.len);
  return r;
}

// Totals beyond 32 bits stay at the largest number (no capacity reaches it).
__device__ __forceinline__ int32_t sat(int64_t x) { return x < 0x7fffffff ? (int32_t)x : 0x7fffffff; }

constexpr int kThreads = 256;

// Exclusive sums of one value per thread; the total of all.
__device__ __forceinline__ int64_t scan(int64_t x, int64_t* wave, int64_t& total) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  int64_t pre = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up((long long)pre, o);
    if (lane >= o) pre += y;
  }
  if (lane == 63) wave[wid] = pre;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wid) pre += wave[w];
    total += wave[w];
  }
  return pre - x;
}

// The first launch of many requests: cu.
__global__ void __launch_bounds__(kThreads) slots_scan_kernel(const SlotArgs a) {
  __shared__ int64_t wave[kThreads / 64];
  const int per = (a.n + kThreads - 1) / kThreads;
  const int lo = min((int)threadIdx.x * per, a.n), hi = min(lo + per, a.n);
  int64_t sum = 0, total;
  for (int i = lo; i < hi; ++i) sum += request(a, i).k;
  int64_t pre = scan(sum, wave, total);
  for (int i = lo; i < hi; ++i) {
    a.cu[i] = sat(pre);
    pre += request(a, i).k;
  }
  if (threadIdx.x == 0) a.cu[a.n] = sat(total);
}

template <bool INLINE>
__global__ void __launch_bounds__(kThreads) slots_kernel(const SlotArgs a) {
  __shared__ int32_t cu_lds[INLINE ? kSlotInline + 1 : 1];
  __shared__ int64_t wave[kThreads / 64];
  const int32_t* cu = a.cu;
  if (INLINE) {
    constexpr int PER = kSlotInline / kThreads;
    int64_t k[PER], sum = 0, total;
    const int per = (a.n + kThreads - 1) / kThreads, lo = (int)threadIdx.x * per;
#pragma unroll
    for (int x = 0; x < PER; ++x) {
      k[x] = x < per && lo + x < a.n ? request(a, lo + x).k : 0;
      sum += k[x];
    }
    int64_t pre = scan(sum, wave, total);
#pragma unroll
    for (int x = 0; x < PER; ++x) {
      if (x < per && lo + x < a.n) {
        cu_lds[lo + x] = sat(pre);
        if (blockIdx.x == 0) a.cu[lo + x] = sat(pre);
      }
      pre += k[x];
    }
    if (threadIdx.x == 0) {
      cu_lds[a.n] = sat(total);
      if (blockIdx.x == 0) a.cu[a.n] = sat(total);
    }
    __syncthreads();
    cu = cu_lds;
  }
  const int64_t step = (int64_t)gridDim.x * kThreads, first = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t total = cu[a.n];
  for (int64_t t = first; t < a.cap; t += step) {
    int64_t slot = -1;
    int32_t pos = -1, req = -1;
    if (t < total) {
      int lo = 0, hi = a.n;  // cu[lo] <= t < cu[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= t)
          lo = mid;
        else
          hi = mid;
      }
      const Request r = request(a, lo);
      // (From the request's first token: the next entry may be saturated.)
      const int64_t p = r.len - r.k + (t - cu[lo]);
      const int32_t page = a.table[r.seq * a.t_sb + (p >> a.ps_shift)];
      if (page >= 0) slot = ((int64_t)page << a.ps_shift) + (p & ((1ll << a.ps_shift) - 1));
      pos = (int32_t)p;
      req = lo;
    }
    a.slots[t] = slot;
    a.pos[t] = pos;
    a.req[t] = req;
  }
  // A wave takes a request's row of the block table at a time.
  const int lane = threadIdx.x & 63;
  const int64_t nw = (int64_t)gridDim.x * (kThreads / 64);
  for (int64_t i = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); i < a.n; i += nw) {
    const Request r = request(a, (int)i);
    const int64_t used = (r.len + (1ll << a.ps_shift) - 1) >> a.ps_shift;
    for (int64_t j = lane; j < a.n_log; j += 64) a.block[i * a.b_sb + j] = j < used ? a.table[r.seq * a.t_sb + j] : -1;
    if (lane == 0) a.out_lens[i] = (int32_t)r.len;
  }
}

}  // namespace

hipError_t launch_slots(const SlotArgs& a, hipStream_t s) {
  // A thread per token, a wave per table row; at most 512 workgroups, which then loop.
  int64_t wgs = (a.cap + kThreads - 1) / kThreads;
  const int64_t rows = (a.n + 3) / 4;
  if (wgs < rows) wgs = rows;
  wgs = wgs < 1 ? 1 : (wgs > 512 ? 512 : wgs);
  if (a.n <= kSlotInline) {
    hipLaunchKernelGGL(slots_kernel<true>, dim3((unsigned)wgs), dim3(kThreads), 0, s, a);
  } else {
    hipLaunchKernelGGL(slots_scan_kernel, dim3(1), dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(slots_kernel<false>, dim3((unsigned)wgs), dim3(kThreads), 0, s, a);
  }
  return hipGetLastError();
}

}  // namespace dsv
