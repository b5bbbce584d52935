// dsv_api.hip — C ABI of libdsv.so: argument validation, split planning,
// workspace carving and kernel launches.  Declarations and the reference
// interface each entry point replaces are in include/dsv.h.

#include "dsv.h"
#include "dsv_attn_geo.h"
#include "dsv_check.h"
#include "dsv_internal.h"
#include "dsv_latent.h"
#include "dsv_window.h"

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <string>

namespace dsv {
size_t accept_walk_lds_bytes(int M);
}

namespace {

using dsv::AcceptArgs;
using dsv::AttnArgs;
using dsv::AttnExtents;
using dsv::Extent;
using dsv::KvSrc;
using dsv::MergeArgs;

thread_local std::string g_err;
thread_local int g_dry_run = 0;
thread_local int64_t g_dry_checks = 0;

// Byte span of a tensor view from its data pointer (non-negative strides),
// over dimensions [first, ndim).
int64_t span_bytes(const dsv_tensor* t, int first = 0) {
  int64_t s = 1;
  for (int i = first; i < t->ndim; ++i) {
    if (t->shape[i] == 0) return 0;
    s += (t->shape[i] - 1) * t->stride[i];
  }
  static const int es[] = {2, 2, 4, 1, 1, 1, 4, 8};
  return s * ((t->dtype >= 0 && t->dtype <= 7) ? es[t->dtype] : 1);
}

Extent extent_of(const char* name, const dsv_tensor* t) {
  if (t == nullptr || t->ndim == 0 || t->data == nullptr) return Extent{name, 0, 0};
  const uintptr_t lo = (uintptr_t)t->data;
  return Extent{name, lo, lo + (uintptr_t)span_bytes(t)};
}

Extent extent_raw(const char* name, const void* p, int64_t bytes) {
  return Extent{name, (uintptr_t)p, (uintptr_t)p + (uintptr_t)(bytes > 0 ? bytes : 0)};
}

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_err = buf;
  return code;
}

int hip_fail(hipError_t e, const char* what) {
  return fail(DSV_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

int elem_size(int dt) {
  switch (dt) {
    case DSV_BF16:
    case DSV_F16: return 2;
    case DSV_F32:
    case DSV_I32: return 4;
    case DSV_I64: return 8;
    case DSV_I8:
    case DSV_U8:
    case DSV_BOOL: return 1;
    default: return 0;
  }
}

const char* dt_name(int dt) {
  static const char* names[] = {"bf16", "f16", "f32", "int8", "uint8", "bool", "int32", "int64"};
  return (dt >= 0 && dt <= 7) ? names[dt] : "?";
}

bool present(const dsv_tensor* t) { return t != nullptr && t->ndim > 0; }

int check_nd(const dsv_tensor* t, const char* name, int ndim) {
  if (t == nullptr || t->ndim != ndim)
    return fail(DSV_ERR_INVALID, "%s must be a %d-d tensor (got %d-d)", name, ndim, t ? t->ndim : -1);
  if (t->data == nullptr) return fail(DSV_ERR_INVALID, "%s has a null data pointer", name);
  if (elem_size(t->dtype) == 0) return fail(DSV_ERR_INVALID, "%s has an unknown dtype %d", name, t->dtype);
  for (int i = 0; i < ndim; ++i) {
    if (t->shape[i] < 0) return fail(DSV_ERR_INVALID, "%s has a negative extent", name);
    if (t->stride[i] < 0) return fail(DSV_ERR_INVALID, "%s has a negative stride", name);
  }
  return DSV_OK;
}

// Attention operand (q, k, v, pages) read with 16-byte vector loads: bf16,
// f16 or f32; innermost stride 1, other strides multiples of 16 bytes,
// 16-byte aligned base.
int check_vec16(const dsv_tensor* t, const char* name, int skip_dim = -1) {
  if (t->dtype != DSV_BF16 && t->dtype != DSV_F16 && t->dtype != DSV_F32)
    return fail(DSV_ERR_UNSUPPORTED, "%s: dtype %s is not supported by the MI355X kernels (bf16, f16 or f32)",
                name, dt_name(t->dtype));
  const int per16 = 16 / elem_size(t->dtype);  // elements per 16 bytes
  if (t->stride[t->ndim - 1] != 1) return fail(DSV_ERR_INVALID, "%s: innermost stride must be 1", name);
  if ((reinterpret_cast<uintptr_t>(t->data) & 15) != 0)
    return fail(DSV_ERR_INVALID, "%s: data pointer must be 16-byte aligned", name);
  for (int i = 0; i < t->ndim - 1; ++i) {
    if (i == skip_dim) continue;
    if (t->shape[i] > 1 && (t->stride[i] % per16) != 0)
      return fail(DSV_ERR_INVALID, "%s: stride[%d]=%lld is not a multiple of %d elements (16 bytes)", name, i,
                  (long long)t->stride[i], per16);
  }
  return DSV_OK;
}

int device_cus() {
  static int cache[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (cache[dev] == 0) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cache[dev] = n;
  }
  return cache[dev];
}

struct Plan {
  int G = 0, R = 0, n_rb = 0, n_splits = 0, s_total = 0;
  int64_t kps = 0;
  size_t opart_bytes = 0, ml_bytes = 0, total = 0;
  const char* err = nullptr;  // sizes beyond the kernels' 32-bit counts (nothing planned)
};

size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

// Splits are sized so that prefix workgroups plus the tree workgroups fill
// every resident workgroup slot of the GPU exactly once.
Plan make_plan(int64_t B, int64_t M, int64_t H, int64_t Hk, int64_t D, int64_t n_keys, int64_t page_size,
               bool has_tree) {
  Plan p;
  const int rows_per_block = dsv::attn_rows_per_block();
  // Row, split and workgroup counts are 32-bit in the kernels and the merge.
  const bool in_range = B <= (1 << 20) && M <= (1 << 24) && H <= (1 << 16) && n_keys <= ((int64_t)1 << 40);
  const int64_t R = in_range ? (H / Hk) * M : 0;
  if (!in_range || R > ((int64_t)1 << 24) || B * Hk * R > ((int64_t)1 << 30)) {
    p.err = "sizes beyond the attention kernels' range (batch <= 2^20, heads <= 65536, keys <= 2^40, query heads / "
            "key heads x rows <= 2^24, batch x query heads x rows <= 2^30)";
    return p;
  }
  p.G = (int)(H / Hk);
  p.R = (int)R;
  p.n_rb = (int)((p.R + rows_per_block - 1) / rows_per_block);
  const int64_t units = B * Hk * p.n_rb;
  if (n_keys > 0) {
    const int64_t slots = (int64_t)device_cus() * dsv::attn_blocks_per_cu();
    const int64_t avail = std::max<int64_t>(slots - (has_tree ? units : 0), units);
    const int64_t s0 = std::max<int64_t>(1, avail / units);
    int64_t kps_max = 16384;
    if (page_size > 0) kps_max = std::min<int64_t>(kps_max, (int64_t)(dsv::kPageLds - 2) * page_size);
    // Whole 32-key tiles per split.
    kps_max = std::max<int64_t>(32, kps_max / 32 * 32);
    int64_t kps = ((n_keys + s0 - 1) / s0 + 31) / 32 * 32;
    kps = std::min(std::max<int64_t>(kps, 32), kps_max);
    p.kps = kps;
    const int64_t ns = (n_keys + kps - 1) / kps;
    if (units * (ns + 1) >= ((int64_t)1 << 31)) {
      p = Plan{};
      p.err = "the key splits need more than 2^31 workgroups";
      return p;
    }
    p.n_splits = (int)ns;
  }
  p.s_total = p.n_splits + (has_tree ? 1 : 0);
  const size_t rows = (size_t)p.s_total * B * Hk * p.R;
  p.opart_bytes = align_up(rows * D * sizeof(uint16_t), 256);
  p.ml_bytes = align_up(rows * sizeof(float2), 256);
  p.total = p.opart_bytes + p.ml_bytes;
  return p;
}

int log2_exact(int64_t x) {
  if (x <= 0 || (x & (x - 1)) != 0) return -1;
  int s = 0;
  while ((1ll << s) < x) ++s;
  return s;
}

// Common checks of q [B, M, H, D] and the output [B, M, H, D].
int check_q_out(const dsv_tensor* q, const dsv_tensor* out) {
  int rc;
  if ((rc = check_nd(q, "q", 4)) != DSV_OK) return rc;
  if ((rc = check_vec16(q, "q")) != DSV_OK) return rc;
  if ((rc = check_nd(out, "out", 4)) != DSV_OK) return rc;
  for (int i = 0; i < 4; ++i)
    if (out->shape[i] != q->shape[i]) return fail(DSV_ERR_INVALID, "out shape must equal q shape");
  if (out->dtype != DSV_BF16 && out->dtype != DSV_F16 && out->dtype != DSV_F32)
    return fail(DSV_ERR_INVALID, "out dtype must be bf16, f16 or f32");
  if (out->stride[3] != 1) return fail(DSV_ERR_INVALID, "out innermost stride must be 1");
  const int64_t D = q->shape[3];
  if (D != 64 && D != 128) return fail(DSV_ERR_UNSUPPORTED, "head_dim %lld is not supported (64 or 128)", (long long)D);
  return DSV_OK;
}

int check_kv_dense(const dsv_tensor* k, const dsv_tensor* v, const dsv_tensor* q, const char* kn, const char* vn) {
  int rc;
  if ((rc = check_nd(k, kn, 4)) != DSV_OK) return rc;
  if ((rc = check_nd(v, vn, 4)) != DSV_OK) return rc;
  if ((rc = check_vec16(k, kn)) != DSV_OK) return rc;
  if ((rc = check_vec16(v, vn)) != DSV_OK) return rc;
  for (int i = 0; i < 4; ++i)
    if (k->shape[i] != v->shape[i]) return fail(DSV_ERR_INVALID, "%s and %s shapes differ", kn, vn);
  if (k->dtype != q->dtype || v->dtype != q->dtype)
    return fail(DSV_ERR_INVALID, "q, %s and %s must share a dtype", kn, vn);
  if (k->shape[0] != q->shape[0]) return fail(DSV_ERR_INVALID, "%s batch differs from q", kn);
  if (k->shape[3] != q->shape[3]) return fail(DSV_ERR_INVALID, "%s head_dim differs from q", kn);
  const int64_t H = q->shape[2], Hk = k->shape[2];
  if (Hk <= 0 || H % Hk != 0)
    return fail(DSV_ERR_INVALID, "query heads (%lld) must be a multiple of key heads (%lld)", (long long)H,
                (long long)Hk);
  return DSV_OK;
}

KvSrc dense_src(const dsv_tensor* k, const dsv_tensor* v, int64_t key0) {
  KvSrc s{};
  s.k = static_cast<const uint16_t*>(k->data);
  s.v = static_cast<const uint16_t*>(v->data);
  s.k_sb = k->shape[0] > 1 ? k->stride[0] : 0;
  s.k_st = k->stride[1];
  s.k_sh = k->stride[2];
  s.v_sb = v->shape[0] > 1 ? v->stride[0] : 0;
  s.v_st = v->stride[1];
  s.v_sh = v->stride[2];
  s.pt = nullptr;
  s.key0 = key0;
  s.k_bytes = span_bytes(k);
  s.v_bytes = span_bytes(v);
  return s;
}

int check_ws(const Plan& p, void* ws, size_t ws_bytes) {
  if (p.err != nullptr) return fail(DSV_ERR_UNSUPPORTED, "%s", p.err);
  if (p.total == 0) return DSV_OK;
  if (ws == nullptr || ws_bytes < p.total)
    return fail(DSV_ERR_WORKSPACE, "workspace of %zu bytes required (got %zu)", p.total, ws_bytes);
  if ((reinterpret_cast<uintptr_t>(ws) & 255) != 0) return fail(DSV_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  return DSV_OK;
}

void fill_common(AttnArgs& a, const dsv_tensor* q, int64_t Hk, const Plan& p, void* ws) {
  a.q = static_cast<const uint16_t*>(q->data);
  a.q_sb = q->stride[0];
  a.q_sm = q->stride[1];
  a.q_sh = q->stride[2];
  a.B = (int)q->shape[0];
  a.M = (int)q->shape[1];
  a.H = (int)q->shape[2];
  a.Hk = (int)Hk;
  a.G = p.G;
  a.R = p.R;
  a.n_rb = p.n_rb;
  a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)q->shape[3]));
  a.n_splits = p.n_splits;
  a.kps = p.kps;
  a.s_total = p.s_total;
  a.opart = static_cast<uint16_t*>(ws);
  a.ml = reinterpret_cast<float2*>(static_cast<char*>(ws) + p.opart_bytes);
}

void fill_merge(MergeArgs& m, const AttnArgs& a, const dsv_tensor* out, int D) {
  m.opart = a.opart;
  m.ml = a.ml;
  m.s_total = a.s_total;
  m.B = a.B;
  m.M = a.M;
  m.H = a.H;
  m.Hk = a.Hk;
  m.G = a.G;
  m.R = a.R;
  m.D = D;
  m.row_perm = a.row_perm;
  m.out = out->data;
  m.out_dtype = out->dtype;
  m.o_sb = out->stride[0];
  m.o_sm = out->stride[1];
  m.o_sh = out->stride[2];
}

// One-shot timing events armed by dsv_set_timing_events (per thread).
thread_local hipEvent_t g_ev_start = nullptr;
thread_local hipEvent_t g_ev_stop = nullptr;

void take_events(hipEvent_t& s, hipEvent_t& e) {
  s = g_ev_start;
  e = g_ev_stop;
  g_ev_start = g_ev_stop = nullptr;
}

// Extents shared by every attention entry point (dry-run checks).
AttnExtents common_extents(const dsv_tensor* q, const dsv_tensor* out, void* ws, const Plan& p) {
  AttnExtents ex;
  ex.q = extent_of("q", q);
  ex.out = extent_of("out", out);
  ex.ws = extent_raw("workspace", ws, (int64_t)p.total);
  return ex;
}

int run(const AttnArgs& a_in, const MergeArgs& m, int dtype, int D, bool dmask, hipStream_t st,
        const AttnExtents& ex) {
  AttnArgs a = a_in;
  a.pre.fast32 = dsv::fast32_ok(a.pre, a.pre.key0 + a.n_pre) ? 1 : 0;
  a.tree.fast32 = a.has_tree && dsv::fast32_ok(a.tree, a.tree.key0 + a.M) ? 1 : 0;
  // One dense prefix split: the attention kernel writes the output itself where
  // it is 16-bit with 16-byte aligned rows (2048 x 32 rows over 8192 keys: the
  // partials' merge took 56 of 305 us, 250 without; rows are rounded once, not
  // twice) and skips the keys past a causal block's rows (4096 of 4096: 384 ->
  // 169 us).  Outputs that overlap an input go through the merge, which starts
  // when every input has been read.
  const auto apart = [](const Extent& x, const Extent& y) { return x.hi <= y.lo || y.hi <= x.lo; };
  const auto outside = [&](const Extent& o) { return apart(o, ex.q) && apart(o, ex.pre_k) && apart(o, ex.pre_v); };
  a.direct = !dmask && !a.has_tree && a.pre.pt == nullptr && a.pre.fast32 != 0 && dtype != DSV_F32 && a.s_total == 1 &&
             m.weight == nullptr && m.out_dtype != DSV_F32 && (reinterpret_cast<uintptr_t>(m.out) & 15) == 0 &&
             ((m.o_sb | m.o_sm | m.o_sh) & 7) == 0 && outside(ex.out) && outside(ex.lse);
  if (a.direct) {
    a.out = static_cast<uint16_t*>(m.out);
    a.direct = m.out_dtype == DSV_F16 ? 2 : 1;
    // Causal row blocks differ in length where a query head has more than one.
    // Within one round of the CUs every order ends with the longest block, and
    // eighths of like lengths are the faster (12 heads of 4, 4096 rows over
    // 16384 keys, 192 blocks: 418 us, 426 dealt or unsorted).
    if (a.causal != 0 && a.n_rb > a.G) a.long_first = (int64_t)a.B * a.Hk * a.n_rb > device_cus() ? 2 : 1;
    a.o_sb = m.o_sb;
    a.o_sm = m.o_sm;
    a.o_sh = m.o_sh;
    a.lse = m.lse;
    a.l_sb = m.l_sb;
    a.l_sm = m.l_sm;
    a.l_sh = m.l_sh;
  }
  if (g_dry_run) {
    std::string err;
    int64_t n = 0;
    const int rc = dsv::emulate_attention(a, m, D, dmask, dtype == DSV_F32, ex, err, &n);
    g_dry_checks = n;
    if (rc != 0) return fail(DSV_ERR_INVALID, "dry run: out-of-bounds access: %s", err.c_str());
    return DSV_OK;
  }
  hipEvent_t ev0, ev1;
  take_events(ev0, ev1);
  hipError_t e = dtype == DSV_F32 ? dsv::launch_attn_f32(a, D, dmask, st, ev0, ev1)
                                  : dsv::launch_attn(a, dtype, D, dmask, st, ev0, ev1);
  if (e != hipSuccess) return hip_fail(e, "attention kernel launch");
  if (a.direct) return DSV_OK;
  e = dsv::launch_merge(m, st);
  if (e != hipSuccess) return hip_fail(e, "merge kernel launch");
  return DSV_OK;
}

int check_byte_mask(const dsv_tensor* mask, int64_t B, int64_t M, const char* name) {
  int rc;
  if ((rc = check_nd(mask, name, 3)) != DSV_OK) return rc;
  if (mask->dtype != DSV_I8 && mask->dtype != DSV_U8 && mask->dtype != DSV_BOOL)
    return fail(DSV_ERR_INVALID, "%s must be int8, uint8 or bool (got %s)", name, dt_name(mask->dtype));
  if (mask->shape[0] != 1 && mask->shape[0] != B) return fail(DSV_ERR_INVALID, "%s batch must be 1 or B", name);
  if (mask->shape[1] != M) return fail(DSV_ERR_INVALID, "%s must have M rows", name);
  return DSV_OK;
}

// Physical page pool view: kv_pages [L, 2, P, Hk, ps, D] -> K and V halves of one layer.
int paged_src(const dsv_tensor* kv_pages, int64_t layer, const dsv_tensor* pt, int64_t B, KvSrc& s,
              int64_t& page_size, int64_t& Hk, int64_t& D, int64_t& capacity) {
  int rc;
  if ((rc = check_nd(kv_pages, "kv_pages", 6)) != DSV_OK) return rc;
  if ((rc = check_vec16(kv_pages, "kv_pages")) != DSV_OK) return rc;
  if (kv_pages->shape[1] != 2) return fail(DSV_ERR_INVALID, "kv_pages dim 1 must be 2 (K, V)");
  if (layer < 0 || layer >= kv_pages->shape[0]) return fail(DSV_ERR_INVALID, "layer_idx out of range");
  page_size = kv_pages->shape[4];
  const int sh = log2_exact(page_size);
  if (sh < 0) return fail(DSV_ERR_UNSUPPORTED, "page_size %lld must be a power of two", (long long)page_size);
  if ((rc = check_nd(pt, "page_table", pt ? pt->ndim : 1)) != DSV_OK) return rc;
  if (pt->ndim != 1 && pt->ndim != 2) return fail(DSV_ERR_INVALID, "page_table must be 1-d or 2-d");
  if (pt->dtype != DSV_I32 && pt->dtype != DSV_I64) return fail(DSV_ERR_INVALID, "page_table must be int32 or int64");
  if (pt->ndim == 2 && pt->shape[0] != B && pt->shape[0] != 1)
    return fail(DSV_ERR_INVALID, "page_table batch must be 1 or B");
  const int64_t npt = pt->shape[pt->ndim - 1];
  if (pt->stride[pt->ndim - 1] != 1) return fail(DSV_ERR_INVALID, "page_table innermost stride must be 1");
  Hk = kv_pages->shape[3];
  D = kv_pages->shape[5];
  const int es = elem_size(kv_pages->dtype);
  const char* base = static_cast<const char*>(kv_pages->data) + layer * kv_pages->stride[0] * es;
  s.k = reinterpret_cast<const uint16_t*>(base);
  s.v = reinterpret_cast<const uint16_t*>(base + kv_pages->stride[1] * es);
  s.k_sb = s.v_sb = 0;
  s.k_sp = s.v_sp = kv_pages->stride[2];
  s.k_sh = s.v_sh = kv_pages->stride[3];
  s.k_st = s.v_st = kv_pages->stride[4];
  s.pt = pt->data;
  s.pt_i64 = pt->dtype == DSV_I64;
  s.ps_shift = sh;
  s.pt_sb = (pt->ndim == 2 && pt->shape[0] > 1) ? pt->stride[0] : 0;
  s.key0 = 0;
  s.n_phys = kv_pages->shape[2];
  s.k_bytes = s.v_bytes = span_bytes(kv_pages, 2);
  capacity = npt * page_size;
  (void)B;
  return DSV_OK;
}

}  // namespace

extern "C" {

int dsv_version(void) { return 1; }

const char* dsv_last_error(void) { return g_err.c_str(); }

int dsv_set_timing_events(void* start_event, void* stop_event) {
  g_ev_start = static_cast<hipEvent_t>(start_event);
  g_ev_stop = static_cast<hipEvent_t>(stop_event);
  return DSV_OK;
}

int dsv_set_dry_run(int enable) {
  g_dry_run = enable != 0;
  return DSV_OK;
}

int64_t dsv_dry_run_checks(void) { return g_dry_checks; }

size_t dsv_attn_workspace_bytes(int64_t B, int64_t M, int64_t H, int64_t Hk, int64_t D, int64_t n_keys,
                                int64_t page_size, int has_tree) {
  if (B <= 0 || M <= 0 || H <= 0 || Hk <= 0 || D <= 0 || H % Hk != 0 || n_keys < 0) return 0;
  return make_plan(B, M, H, Hk, D, n_keys, page_size, has_tree != 0).total;
}

}  // extern "C"

namespace {

// Prefix attention with an optional per-batch length and causal mask: the
// body of dsv_prefix_attention_forward and dsv_flash_attn_with_kvcache.
int prefix_attention(const dsv_tensor* q, const dsv_tensor* k, const dsv_tensor* v, const dsv_tensor* seqlens,
                     int64_t n_keys, int causal, dsv_tensor* out, dsv_tensor* lse, void* workspace,
                     size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_q_out(q, out)) != DSV_OK) return rc;
  if ((rc = check_kv_dense(k, v, q, "k", "v")) != DSV_OK) return rc;
  const int64_t B = q->shape[0], M = q->shape[1], H = q->shape[2], D = q->shape[3];
  const int64_t N = k->shape[1], Hk = k->shape[2];
  if (n_keys < 0) n_keys = N;
  if (n_keys > N) return fail(DSV_ERR_INVALID, "n_keys (%lld) exceeds the key length (%lld)", (long long)n_keys, (long long)N);
  if (present(seqlens)) {
    if ((rc = check_nd(seqlens, "cache_seqlens", 1)) != DSV_OK) return rc;
    if ((seqlens->dtype != DSV_I32 && seqlens->dtype != DSV_I64) || seqlens->shape[0] != B || seqlens->stride[0] != 1)
      return fail(DSV_ERR_INVALID, "cache_seqlens must be a contiguous int32|int64 [B] tensor");
  }
  if (present(lse)) {
    if ((rc = check_nd(lse, "lse", 3)) != DSV_OK) return rc;
    if (lse->dtype != DSV_F32 || lse->shape[0] != B || lse->shape[1] != H || lse->shape[2] != M)
      return fail(DSV_ERR_INVALID, "lse must be float32 [B, H, M]");
  }
  const Plan p = make_plan(B, M, H, Hk, D, n_keys, 0, false);
  if ((rc = check_ws(p, workspace, workspace_bytes)) != DSV_OK) return rc;

  AttnArgs a{};
  fill_common(a, q, Hk, p, workspace);
  a.pre = dense_src(k, v, 0);
  a.n_pre = n_keys;
  if (present(seqlens)) {
    a.seqlens = seqlens->data;
    a.seqlens_i64 = seqlens->dtype == DSV_I64;
  }
  a.causal = causal != 0;
  MergeArgs m{};
  fill_merge(m, a, out, (int)D);
  if (present(lse)) {
    m.lse = static_cast<float*>(lse->data);
    m.l_sb = lse->stride[0];
    m.l_sh = lse->stride[1];
    m.l_sm = lse->stride[2];
  }
  AttnExtents ex = common_extents(q, out, workspace, p);
  ex.pre_k = extent_of("k", k);
  ex.pre_v = extent_of("v", v);
  ex.lse = extent_of("lse", lse);
  return run(a, m, q->dtype, (int)D, false, static_cast<hipStream_t>(stream), ex);
}

}  // namespace

extern "C" {

int dsv_prefix_attention_forward(const dsv_tensor* q, const dsv_tensor* k, const dsv_tensor* v, int64_t n_keys,
                                 dsv_tensor* out, dsv_tensor* lse, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  if (!present(lse)) return fail(DSV_ERR_INVALID, "lse must be float32 [B, H, M]");
  return prefix_attention(q, k, v, nullptr, n_keys, 0, out, lse, workspace, workspace_bytes, stream);
}

int dsv_flash_attn_with_kvcache(const dsv_tensor* q, const dsv_tensor* k_cache, const dsv_tensor* v_cache,
                                const dsv_tensor* cache_seqlens, int64_t n_keys, int causal, dsv_tensor* out,
                                dsv_tensor* softmax_lse, void* workspace, size_t workspace_bytes, void* stream) {
  return prefix_attention(q, k_cache, v_cache, cache_seqlens, n_keys, causal, out, softmax_lse, workspace,
                          workspace_bytes, stream);
}

int dsv_tree_attention_forward(const dsv_tensor* q, const dsv_tensor* k, const dsv_tensor* v,
                               const dsv_tensor* tree_mask, const dsv_tensor* prefix_lse, dsv_tensor* current_out,
                               dsv_tensor* weight, dsv_tensor* tree_lse, void* workspace, size_t workspace_bytes,
                               void* stream) {
  int rc;
  if ((rc = check_q_out(q, current_out)) != DSV_OK) return rc;
  if ((rc = check_kv_dense(k, v, q, "key_states", "value_states")) != DSV_OK) return rc;
  const int64_t B = q->shape[0], M = q->shape[1], H = q->shape[2], D = q->shape[3], Hk = k->shape[2];
  if (k->shape[1] != M) return fail(DSV_ERR_INVALID, "key/value must be the post-cache block of M rows");
  if (M > dsv::kTreeMaxM) return fail(DSV_ERR_UNSUPPORTED, "tree blocks larger than %d nodes are not supported", dsv::kTreeMaxM);
  if (tree_mask == nullptr || (tree_mask->ndim != 3 && tree_mask->ndim != 4))
    return fail(DSV_ERR_INVALID, "tree_mask must be [B, 1, T, T] or [B, T, T]");
  if ((rc = check_nd(tree_mask, "tree_mask", tree_mask->ndim)) != DSV_OK) return rc;
  const int nd = tree_mask->ndim;
  const int64_t T0 = tree_mask->shape[nd - 2], T1 = tree_mask->shape[nd - 1];
  if (T0 < M || T1 < M) return fail(DSV_ERR_INVALID, "tree_mask is smaller than the M x M block");
  if (tree_mask->shape[0] != B && tree_mask->shape[0] != 1) return fail(DSV_ERR_INVALID, "tree_mask batch must be 1 or B");
  if ((rc = check_nd(prefix_lse, "prefix_lse", 3)) != DSV_OK) return rc;
  if (prefix_lse->dtype != DSV_F32 || prefix_lse->shape[0] != B || prefix_lse->shape[1] != H || prefix_lse->shape[2] != M)
    return fail(DSV_ERR_INVALID, "prefix_lse must be float32 viewed as [B, H, M]");
  if ((rc = check_nd(weight, "weight", 4)) != DSV_OK) return rc;
  if (weight->shape[0] != B || weight->shape[1] != M || weight->shape[2] != H || weight->shape[3] != 1)
    return fail(DSV_ERR_INVALID, "weight must be [B, M, H, 1]");
  if (weight->dtype != DSV_BF16 && weight->dtype != DSV_F16 && weight->dtype != DSV_F32)
    return fail(DSV_ERR_INVALID, "weight dtype must be bf16, f16 or f32");
  if (present(tree_lse)) {
    if ((rc = check_nd(tree_lse, "tree_lse", 3)) != DSV_OK) return rc;
    if (tree_lse->dtype != DSV_F32 || tree_lse->shape[0] != B || tree_lse->shape[1] != M || tree_lse->shape[2] != H)
      return fail(DSV_ERR_INVALID, "tree_lse must be float32 [B, M, H]");
  }
  const Plan p = make_plan(B, M, H, Hk, D, 0, 0, true);
  if ((rc = check_ws(p, workspace, workspace_bytes)) != DSV_OK) return rc;

  AttnArgs a{};
  fill_common(a, q, Hk, p, workspace);
  a.n_pre = 0;
  a.has_tree = 1;
  a.tree = dense_src(k, v, 0);
  const int64_t es = elem_size(tree_mask->dtype);
  const int64_t sb = tree_mask->shape[0] > 1 ? tree_mask->stride[0] : 0;
  const int64_t sm = tree_mask->stride[nd - 2], sn = tree_mask->stride[nd - 1];
  a.tmask = static_cast<const char*>(tree_mask->data) + ((T0 - M) * sm + (T1 - M) * sn) * es;
  a.tmask_dtype = tree_mask->dtype;
  a.tm_sb = sb;
  a.tm_sm = sm;
  a.tm_sn = sn;
  MergeArgs m{};
  fill_merge(m, a, current_out, (int)D);
  if (present(tree_lse)) {
    m.lse = static_cast<float*>(tree_lse->data);
    m.l_sb = tree_lse->stride[0];
    m.l_sm = tree_lse->stride[1];
    m.l_sh = tree_lse->stride[2];
  }
  m.plse = static_cast<const float*>(prefix_lse->data);
  m.p_sb = prefix_lse->stride[0];
  m.p_sh = prefix_lse->stride[1];
  m.p_sm = prefix_lse->stride[2];
  m.weight = weight->data;
  m.w_dtype = weight->dtype;
  m.w_sb = weight->stride[0];
  m.w_sm = weight->stride[1];
  m.w_sh = weight->stride[2];
  AttnExtents ex = common_extents(q, current_out, workspace, p);
  ex.tree_k = extent_of("key_states", k);
  ex.tree_v = extent_of("value_states", v);
  ex.tmask = extent_of("tree_mask", tree_mask);
  ex.lse = extent_of("tree_lse", tree_lse);
  ex.plse = extent_of("prefix_lse", prefix_lse);
  ex.weight = extent_of("weight", weight);
  return run(a, m, q->dtype, (int)D, false, static_cast<hipStream_t>(stream), ex);
}

int dsv_verify_bundle(const dsv_tensor* q, const dsv_tensor* k, const dsv_tensor* v, const dsv_tensor* mask,
                      dsv_tensor* out, dsv_tensor* lse, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_q_out(q, out)) != DSV_OK) return rc;
  if ((rc = check_kv_dense(k, v, q, "k", "v")) != DSV_OK) return rc;
  const int64_t B = q->shape[0], M = q->shape[1], H = q->shape[2], D = q->shape[3];
  const int64_t N = k->shape[1], Hk = k->shape[2];
  if ((rc = check_byte_mask(mask, B, M, "mask")) != DSV_OK) return rc;
  if ((rc = check_nd(lse, "lse", 3)) != DSV_OK) return rc;
  if (lse->dtype != DSV_F32 || lse->shape[0] != B || lse->shape[1] != M || lse->shape[2] != H)
    return fail(DSV_ERR_INVALID, "lse must be float32 [B, M, H]");
  const Plan p = make_plan(B, M, H, Hk, D, N, 0, false);
  if ((rc = check_ws(p, workspace, workspace_bytes)) != DSV_OK) return rc;

  AttnArgs a{};
  fill_common(a, q, Hk, p, workspace);
  a.pre = dense_src(k, v, 0);
  a.n_pre = N;
  a.dmask = static_cast<const uint8_t*>(mask->data);
  a.dm_sb = mask->shape[0] > 1 ? mask->stride[0] : 0;
  a.dm_sm = mask->stride[1];
  a.dm_sn = mask->stride[2];
  a.dm_n = mask->shape[2];
  MergeArgs m{};
  fill_merge(m, a, out, (int)D);
  m.lse = static_cast<float*>(lse->data);
  m.l_sb = lse->stride[0];
  m.l_sm = lse->stride[1];
  m.l_sh = lse->stride[2];
  AttnExtents ex = common_extents(q, out, workspace, p);
  ex.pre_k = extent_of("k", k);
  ex.pre_v = extent_of("v", v);
  ex.dmask = extent_of("mask", mask);
  ex.lse = extent_of("lse", lse);
  return run(a, m, q->dtype, (int)D, true, static_cast<hipStream_t>(stream), ex);
}

int dsv_verify_bundle_paged(const dsv_tensor* q, const dsv_tensor* kv_pages, const dsv_tensor* page_table,
                            int64_t layer_idx, const dsv_tensor* mask, dsv_tensor* out, dsv_tensor* lse,
                            void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_q_out(q, out)) != DSV_OK) return rc;
  const int64_t B = q->shape[0], M = q->shape[1], H = q->shape[2], D = q->shape[3];
  KvSrc s{};
  int64_t ps = 0, Hk = 0, Dk = 0, cap = 0;
  if ((rc = paged_src(kv_pages, layer_idx, page_table, B, s, ps, Hk, Dk, cap)) != DSV_OK) return rc;
  if (kv_pages->dtype != q->dtype) return fail(DSV_ERR_INVALID, "q and kv_pages must share a dtype");
  if (Dk != D) return fail(DSV_ERR_INVALID, "kv_pages head_dim differs from q");
  if (H % Hk != 0) return fail(DSV_ERR_INVALID, "query heads must be a multiple of kv_pages heads");
  if ((rc = check_byte_mask(mask, B, M, "mask")) != DSV_OK) return rc;
  const int64_t N = mask->shape[2];
  if (N > cap) return fail(DSV_ERR_INVALID, "mask covers %lld tokens but the page table maps %lld", (long long)N, (long long)cap);
  if ((rc = check_nd(lse, "lse", 3)) != DSV_OK) return rc;
  if (lse->dtype != DSV_F32 || lse->shape[0] != B || lse->shape[1] != M || lse->shape[2] != H)
    return fail(DSV_ERR_INVALID, "lse must be float32 [B, M, H]");
  const Plan p = make_plan(B, M, H, Hk, D, N, ps, false);
  if ((rc = check_ws(p, workspace, workspace_bytes)) != DSV_OK) return rc;

  AttnArgs a{};
  fill_common(a, q, Hk, p, workspace);
  a.pre = s;
  a.n_pre = N;
  a.dmask = static_cast<const uint8_t*>(mask->data);
  a.dm_sb = mask->shape[0] > 1 ? mask->stride[0] : 0;
  a.dm_sm = mask->stride[1];
  a.dm_sn = mask->stride[2];
  a.dm_n = N;
  MergeArgs m{};
  fill_merge(m, a, out, (int)D);
  m.lse = static_cast<float*>(lse->data);
  m.l_sb = lse->stride[0];
  m.l_sm = lse->stride[1];
  m.l_sh = lse->stride[2];
  AttnExtents ex = common_extents(q, out, workspace, p);
  ex.pre_k = extent_raw("kv_pages[layer, 0]", s.k, s.k_bytes);
  ex.pre_v = extent_raw("kv_pages[layer, 1]", s.v, s.v_bytes);
  ex.pre_pt = extent_of("page_table", page_table);
  ex.dmask = extent_of("mask", mask);
  ex.lse = extent_of("lse", lse);
  return run(a, m, q->dtype, (int)D, true, static_cast<hipStream_t>(stream), ex);
}

}  // extern "C"

namespace {

// Scratch of the allocation-free tree verify: a file-scope device array, one
// copy per GPU for the life of the process.  The split plan fills the GPU's
// workgroup slots with (batch, KV head, row block, split) units and needs
// 2 * D + 8 bytes per (split, batch, KV head, query row), about
// slots x 256 rows x (2 * D + 8) bytes (17 MiB at D = 128 on 256 CUs) until
// the 16384-key cap on a split adds splits.  At D = 128, 8 KV heads, 256 CUs
// 32 MiB holds one tree of <= 64 nodes up to 512K prefix tokens, <= 128
// nodes up to 256K, <= 256 nodes up to 128K, and 8 trees of 64 nodes at 64K.
constexpr size_t kNoAllocScratchBytes = DSV_NOALLOC_SCRATCH_BYTES;
static __device__ __align__(256) uint8_t scratch[kNoAllocScratchBytes];

constexpr int kMaxDevices = 64;
std::mutex g_scratch_mu;

// Per GPU: the scratch array's device address, and the guard that orders
// calls made on different streams: an event recorded after each call's
// kernels and the stream it was recorded on.  A call on another stream first
// makes its stream wait for that event, so two calls never use the array at
// the same time unless a caller hides them from the guard (graph capture,
// see dsv.h).
struct NoAllocDevice {
  void* scratch = nullptr;
  hipEvent_t done = nullptr;
  hipStream_t last = nullptr;
  bool used = false;
};
NoAllocDevice g_noalloc[kMaxDevices];

// Set-up, once per device with that device current: the scratch array's
// address (its name is a host-side stand-in and may not be passed to a
// kernel or a copy) and the guard's event.  Called with g_scratch_mu held.
int noalloc_device(NoAllocDevice** out) {
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return hip_fail(e, "hipGetDevice");
  if (dev < 0 || dev >= kMaxDevices) return fail(DSV_ERR_UNSUPPORTED, "device ordinal %d beyond %d", dev, kMaxDevices);
  NoAllocDevice& d = g_noalloc[dev];
  if (d.scratch == nullptr) {
    void* p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    if (e != hipSuccess) return hip_fail(e, "hipGetSymbolAddress(scratch)");
    if (p == nullptr || (reinterpret_cast<uintptr_t>(p) & 255) != 0)
      return fail(DSV_ERR_HIP, "scratch array at an unusable address");
    e = hipEventCreateWithFlags(&d.done, hipEventDisableTiming);
    if (e != hipSuccess) return hip_fail(e, "hipEventCreateWithFlags (allocation-free entry point set-up)");
    d.scratch = p;
  }
  *out = &d;
  return DSV_OK;
}

int tree_verify_impl(const dsv_tensor* q, const dsv_tensor* k, const dsv_tensor* v, const dsv_tensor* page_table,
                     int64_t n_prefix, const dsv_tensor* parent, const dsv_tensor* row_perm, dsv_tensor* out,
                     dsv_tensor* lse, void* workspace, size_t workspace_bytes, bool noalloc, void* stream) {
  int rc;
  if ((rc = check_q_out(q, out)) != DSV_OK) return rc;
  const int64_t B = q->shape[0], M = q->shape[1], H = q->shape[2], D = q->shape[3];
  if (M > dsv::kTreeMaxM) return fail(DSV_ERR_UNSUPPORTED, "trees larger than %d nodes are not supported", dsv::kTreeMaxM);
  if (n_prefix < 0) return fail(DSV_ERR_INVALID, "n_prefix must be >= 0");
  KvSrc src{};
  int64_t Hk = 0, ps = 0, cap = 0;
  if (present(page_table)) {
    // k, v: [P, Hk, ps, D] page-pool halves.
    if ((rc = check_nd(k, "k_pages", 4)) != DSV_OK) return rc;
    if ((rc = check_nd(v, "v_pages", 4)) != DSV_OK) return rc;
    if ((rc = check_vec16(k, "k_pages")) != DSV_OK) return rc;
    if ((rc = check_vec16(v, "v_pages")) != DSV_OK) return rc;
    for (int i = 0; i < 4; ++i)
      if (k->shape[i] != v->shape[i]) return fail(DSV_ERR_INVALID, "k_pages and v_pages shapes differ");
    if (k->dtype != q->dtype || v->dtype != q->dtype) return fail(DSV_ERR_INVALID, "q and pages must share a dtype");
    if (k->shape[3] != D) return fail(DSV_ERR_INVALID, "page head_dim differs from q");
    ps = k->shape[2];
    const int sh = log2_exact(ps);
    if (sh < 0) return fail(DSV_ERR_UNSUPPORTED, "page_size %lld must be a power of two", (long long)ps);
    if ((rc = check_nd(page_table, "page_table", page_table->ndim)) != DSV_OK) return rc;
    if (page_table->ndim != 1 && page_table->ndim != 2) return fail(DSV_ERR_INVALID, "page_table must be 1-d or 2-d");
    if (page_table->dtype != DSV_I32 && page_table->dtype != DSV_I64)
      return fail(DSV_ERR_INVALID, "page_table must be int32 or int64");
    if (page_table->ndim == 2 && page_table->shape[0] != B && page_table->shape[0] != 1)
      return fail(DSV_ERR_INVALID, "page_table batch must be 1 or B");
    if (page_table->stride[page_table->ndim - 1] != 1) return fail(DSV_ERR_INVALID, "page_table innermost stride must be 1");
    Hk = k->shape[1];
    src.k = static_cast<const uint16_t*>(k->data);
    src.v = static_cast<const uint16_t*>(v->data);
    src.k_sp = k->stride[0];
    src.k_sh = k->stride[1];
    src.k_st = k->stride[2];
    src.v_sp = v->stride[0];
    src.v_sh = v->stride[1];
    src.v_st = v->stride[2];
    src.pt = page_table->data;
    src.pt_i64 = page_table->dtype == DSV_I64;
    src.ps_shift = sh;
    src.pt_sb = (page_table->ndim == 2 && page_table->shape[0] > 1) ? page_table->stride[0] : 0;
    src.n_phys = k->shape[0];
    src.k_bytes = span_bytes(k);
    src.v_bytes = span_bytes(v);
    cap = page_table->shape[page_table->ndim - 1] * ps;
  } else {
    if ((rc = check_kv_dense(k, v, q, "k_cache", "v_cache")) != DSV_OK) return rc;
    Hk = k->shape[2];
    src = dense_src(k, v, 0);
    cap = k->shape[1];
  }
  if (H % Hk != 0) return fail(DSV_ERR_INVALID, "query heads must be a multiple of key heads");
  if (n_prefix + M > cap)
    return fail(DSV_ERR_INVALID, "cache holds %lld tokens, n_prefix + M = %lld", (long long)cap, (long long)(n_prefix + M));
  if (parent == nullptr || (parent->ndim != 1 && parent->ndim != 2))
    return fail(DSV_ERR_INVALID, "parent must be [M] or [B, M]");
  if ((rc = check_nd(parent, "parent", parent->ndim)) != DSV_OK) return rc;
  if (parent->dtype != DSV_I32 && parent->dtype != DSV_I64) return fail(DSV_ERR_INVALID, "parent must be int32 or int64");
  if (parent->shape[parent->ndim - 1] != M) return fail(DSV_ERR_INVALID, "parent must have M entries per tree");
  if (parent->ndim == 2 && parent->shape[0] != B && parent->shape[0] != 1)
    return fail(DSV_ERR_INVALID, "parent batch must be 1 or B");
  if (present(row_perm)) {
    if ((rc = check_nd(row_perm, "row_perm", 1)) != DSV_OK) return rc;
    if (row_perm->dtype != DSV_I32 || row_perm->shape[0] != M || row_perm->stride[0] != 1)
      return fail(DSV_ERR_INVALID, "row_perm must be a contiguous int32 [M] permutation");
  }
  if (present(lse)) {
    if ((rc = check_nd(lse, "lse", 3)) != DSV_OK) return rc;
    if (lse->dtype != DSV_F32 || lse->shape[0] != B || lse->shape[1] != M || lse->shape[2] != H)
      return fail(DSV_ERR_INVALID, "lse must be float32 [B, M, H]");
  }
  const Plan p = make_plan(B, M, H, Hk, D, n_prefix, ps, true);
  // The allocation-free entry point holds g_scratch_mu from here to the end
  // of its launches, so that the guard's wait, the kernels and the record of
  // the guard's event are one step for other threads.
  std::unique_lock<std::mutex> lock(g_scratch_mu, std::defer_lock);
  NoAllocDevice* nad = nullptr;
  bool guard = false;
  if (noalloc) {
    if (p.total > kNoAllocScratchBytes)
      return fail(DSV_ERR_UNSUPPORTED,
                  "this shape needs %zu bytes of split scratch, above the %zu bytes of the allocation-free entry "
                  "point; use dsv_tree_verify with a workspace",
                  p.total, kNoAllocScratchBytes);
    lock.lock();
    if ((rc = noalloc_device(&nad)) != DSV_OK) return rc;
    workspace = nad->scratch;
    workspace_bytes = kNoAllocScratchBytes;
    // Under stream capture the guard stands aside: the captured kernels run
    // when the graph is replayed, in the order the caller gives the replays.
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    hipError_t e = hipStreamIsCapturing(static_cast<hipStream_t>(stream), &cs);
    if (e != hipSuccess) return hip_fail(e, "hipStreamIsCapturing");
    guard = cs == hipStreamCaptureStatusNone && !g_dry_run;
  }
  if ((rc = check_ws(p, workspace, workspace_bytes)) != DSV_OK) return rc;

  AttnArgs a{};
  fill_common(a, q, Hk, p, workspace);
  a.pre = src;
  a.pre.key0 = 0;
  a.n_pre = n_prefix;
  a.has_tree = 1;
  a.tree = src;
  a.tree.key0 = n_prefix;
  a.tpar = parent->data;
  a.tpar_i64 = parent->dtype == DSV_I64;
  a.tpar_sb = (parent->ndim == 2 && parent->shape[0] > 1) ? parent->stride[0] : 0;
  a.tpar_sm = parent->stride[parent->ndim - 1];
  a.row_perm = present(row_perm) ? static_cast<const int32_t*>(row_perm->data) : nullptr;
  MergeArgs m{};
  fill_merge(m, a, out, (int)D);
  if (present(lse)) {
    m.lse = static_cast<float*>(lse->data);
    m.l_sb = lse->stride[0];
    m.l_sm = lse->stride[1];
    m.l_sh = lse->stride[2];
  }
  AttnExtents ex = common_extents(q, out, workspace, p);
  ex.pre_k = ex.tree_k = extent_raw("k", src.k, src.k_bytes);
  ex.pre_v = ex.tree_v = extent_raw("v", src.v, src.v_bytes);
  ex.pre_pt = ex.tree_pt = extent_of("page_table", page_table);
  ex.tpar = extent_of("parent", parent);
  ex.perm = extent_of("row_perm", row_perm);
  ex.lse = extent_of("lse", lse);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (guard && nad->used && nad->last != st) {
    // The previous call ran on another stream: this one starts after it.
    const hipError_t e = hipStreamWaitEvent(st, nad->done, 0);
    if (e != hipSuccess) return hip_fail(e, "hipStreamWaitEvent (allocation-free entry point guard)");
  }
  rc = run(a, m, q->dtype, (int)D, false, st, ex);
  if (rc == DSV_OK && guard) {
    const hipError_t e = hipEventRecord(nad->done, st);
    if (e != hipSuccess) return hip_fail(e, "hipEventRecord (allocation-free entry point guard)");
    nad->last = st;
    nad->used = true;
  }
  return rc;
}

}  // namespace

extern "C" {

int dsv_tree_verify(const dsv_tensor* q, const dsv_tensor* k, const dsv_tensor* v, const dsv_tensor* page_table,
                    int64_t n_prefix, const dsv_tensor* parent, const dsv_tensor* row_perm, dsv_tensor* out,
                    dsv_tensor* lse, void* workspace, size_t workspace_bytes, void* stream) {
  return tree_verify_impl(q, k, v, page_table, n_prefix, parent, row_perm, out, lse, workspace, workspace_bytes,
                          false, stream);
}

int dsv_tree_verify_noalloc(const dsv_tensor* q, const dsv_tensor* k, const dsv_tensor* v,
                            const dsv_tensor* page_table, int64_t n_prefix, const dsv_tensor* parent,
                            const dsv_tensor* row_perm, dsv_tensor* out, dsv_tensor* lse, void* stream) {
  return tree_verify_impl(q, k, v, page_table, n_prefix, parent, row_perm, out, lse, nullptr, 0, true, stream);
}

// ----------------------------------------------------------------------------
// Acceptance
// ----------------------------------------------------------------------------

size_t dsv_accept_workspace_bytes(int64_t T, int64_t M, int64_t V) {
  if (T <= 0 || M <= 0 || V <= 0) return 0;
  const size_t rows = (size_t)T * M * dsv::accept_max_chunks(V);
  // per (row, range) statistics, the typical sums, and per row the sampling
  // mode's kept-set bounds
  return align_up(rows * 16, 256) + align_up(rows * 4, 256) + align_up((size_t)T * M * 16, 256);
}

int dsv_kv_append(const dsv_tensor* k, const dsv_tensor* v, const dsv_tensor* cos, const dsv_tensor* sin,
                  dsv_tensor* k_dst, dsv_tensor* v_dst, const dsv_tensor* page_table, int64_t start,
                  const dsv_tensor* q, dsv_tensor* q_out, void* stream) {
  int rc;
  // A [lead..., X, Y, D] operand with an optional leading 1: the last three dims.
  auto last3 = [&](const dsv_tensor* t, const char* name, int64_t s[3], int64_t st[3]) -> int {
    int r;
    if (t == nullptr || (t->ndim != 3 && t->ndim != 4)) return fail(DSV_ERR_INVALID, "%s must be 3-d or [1, ...] 4-d", name);
    if ((r = check_nd(t, name, t->ndim)) != DSV_OK) return r;
    if (t->ndim == 4 && t->shape[0] != 1) return fail(DSV_ERR_INVALID, "%s leading dimension must be 1", name);
    const int o = t->ndim - 3;
    for (int x = 0; x < 3; ++x) {
      s[x] = t->shape[o + x];
      st[x] = t->stride[o + x];
    }
    if (st[2] != 1) return fail(DSV_ERR_INVALID, "%s innermost stride must be 1", name);
    if ((reinterpret_cast<uintptr_t>(t->data) & 15) != 0 || (st[0] * 2) % 16 != 0 || (st[1] * 2) % 16 != 0)
      return fail(DSV_ERR_INVALID, "%s rows must be 16-byte aligned", name);
    return DSV_OK;
  };
  int64_t ks[3], kst[3], vs[3], vst[3];
  if ((rc = last3(k, "k", ks, kst)) != DSV_OK) return rc;
  if ((rc = last3(v, "v", vs, vst)) != DSV_OK) return rc;
  if (k->dtype != DSV_BF16 && k->dtype != DSV_F16) return fail(DSV_ERR_INVALID, "k must be bf16 or f16");
  if (v->dtype != k->dtype) return fail(DSV_ERR_INVALID, "k and v must share a dtype");
  const int64_t M = ks[0], Hk = ks[1], D = ks[2];
  if (vs[0] != M || vs[1] != Hk || vs[2] != D) return fail(DSV_ERR_INVALID, "v must match k");
  if (M < 1 || Hk < 1) return fail(DSV_ERR_INVALID, "empty k");
  if (D % 16 != 0) return fail(DSV_ERR_UNSUPPORTED, "head_dim %lld must be a multiple of 16", (long long)D);
  // The kernel's counts are 32-bit and its grid covers one thread per
  // 16-element chunk of every row.
  if (M > (1 << 24) || Hk > (1 << 16) || D > (1 << 12))
    return fail(DSV_ERR_UNSUPPORTED, "k is too large (M <= 2^24, key heads <= 65536, head_dim <= 4096)");
  if (start < 0) return fail(DSV_ERR_INVALID, "start must be >= 0");

  dsv::AppendArgs a{};
  a.f16 = k->dtype == DSV_F16;
  a.M = (int)M;
  a.Hk = (int)Hk;
  a.D = (int)D;
  a.start = start;
  a.k = static_cast<const uint16_t*>(k->data);
  a.k_sm = kst[0];
  a.k_sh = kst[1];
  a.v = static_cast<const uint16_t*>(v->data);
  a.v_sm = vst[0];
  a.v_sh = vst[1];
  if (present(cos) || present(sin)) {
    if (!present(cos) || !present(sin)) return fail(DSV_ERR_INVALID, "cos and sin go together");
    for (const dsv_tensor* t : {cos, sin}) {
      const char* nm = t == cos ? "cos" : "sin";
      if (t->ndim != 2 && t->ndim != 3) return fail(DSV_ERR_INVALID, "%s must be [M, D] or [1, M, D]", nm);
      if ((rc = check_nd(t, nm, t->ndim)) != DSV_OK) return rc;
      const int o = t->ndim - 2;
      if ((t->ndim == 3 && t->shape[0] != 1) || t->shape[o] != M || t->shape[o + 1] != D || t->stride[o + 1] != 1)
        return fail(DSV_ERR_INVALID, "%s must be [M, D] with innermost stride 1", nm);
      if (t->dtype != k->dtype) return fail(DSV_ERR_INVALID, "%s must have the dtype of k", nm);
      if ((reinterpret_cast<uintptr_t>(t->data) & 15) != 0 || (t->stride[o] * 2) % 16 != 0)
        return fail(DSV_ERR_INVALID, "%s rows must be 16-byte aligned", nm);
    }
    a.cos = static_cast<const uint16_t*>(cos->data);
    a.cs_m = cos->stride[cos->ndim - 2];
    a.sin = static_cast<const uint16_t*>(sin->data);
    a.sn_m = sin->stride[sin->ndim - 2];
  }
  if (present(q) || present(q_out)) {
    int64_t qs[3], qst[3], os[3], ost[3];
    if (!present(q) || !present(q_out)) return fail(DSV_ERR_INVALID, "q and q_out go together");
    if ((rc = last3(q, "q", qs, qst)) != DSV_OK) return rc;
    if ((rc = last3(q_out, "q_out", os, ost)) != DSV_OK) return rc;
    if (q->dtype != k->dtype || q_out->dtype != k->dtype) return fail(DSV_ERR_INVALID, "q and q_out must have the dtype of k");
    if (qs[0] != M || qs[2] != D || os[0] != M || os[1] != qs[1] || os[2] != D)
      return fail(DSV_ERR_INVALID, "q and q_out must be [M, H, D]");
    if (qs[1] > (1 << 16)) return fail(DSV_ERR_UNSUPPORTED, "q has more than 65536 heads");
    a.H = (int)qs[1];
    a.q = static_cast<const uint16_t*>(q->data);
    a.q_sm = qst[0];
    a.q_sh = qst[1];
    a.q_out = static_cast<uint16_t*>(q_out->data);
    a.qo_sm = ost[0];
    a.qo_sh = ost[1];
  }
  if ((2 * M * Hk + (int64_t)a.H * M) * (D / 16) > ((int64_t)1 << 31))
    return fail(DSV_ERR_UNSUPPORTED, "k, v and q hold more than 2^31 16-element chunks");
  for (dsv_tensor* t : {k_dst, v_dst}) {
    const char* nm = t == k_dst ? "k_dst" : "v_dst";
    if (t == nullptr || t->data == nullptr) return fail(DSV_ERR_INVALID, "%s missing", nm);
    if (t->dtype != k->dtype) return fail(DSV_ERR_INVALID, "%s must have the dtype of k", nm);
    if ((reinterpret_cast<uintptr_t>(t->data) & 15) != 0) return fail(DSV_ERR_INVALID, "%s must be 16-byte aligned", nm);
  }
  if (present(page_table)) {
    if ((rc = check_nd(page_table, "page_table", 1)) != DSV_OK) return rc;
    if (page_table->dtype != DSV_I32 && page_table->dtype != DSV_I64)
      return fail(DSV_ERR_INVALID, "page_table must be int32 or int64");
    if (page_table->stride[0] != 1) return fail(DSV_ERR_INVALID, "page_table stride must be 1");
    int64_t ps = 0, P = 0;
    for (dsv_tensor* t : {k_dst, v_dst}) {
      const char* nm = t == k_dst ? "k_dst" : "v_dst";
      if ((rc = check_nd(t, nm, 4)) != DSV_OK) return rc;
      if (t->shape[1] != Hk || t->shape[3] != D || t->stride[3] != 1)
        return fail(DSV_ERR_INVALID, "%s must be [P, Hk, page, D] with innermost stride 1", nm);
      for (int x = 0; x < 3; ++x)
        if ((t->stride[x] * 2) % 16 != 0) return fail(DSV_ERR_INVALID, "%s rows must be 16-byte aligned", nm);
      if (t == k_dst) {
        ps = t->shape[2];
        P = t->shape[0];
      } else if (t->shape[2] != ps || t->shape[0] != P) {
        return fail(DSV_ERR_INVALID, "k_dst and v_dst must have the same pages");
      }
    }
    const int sh = log2_exact(ps);
    if (sh < 0) return fail(DSV_ERR_UNSUPPORTED, "page size must be a power of two");
    if (start + M > page_table->shape[0] * ps) return fail(DSV_ERR_INVALID, "tokens [start, start + M) exceed the page table");
    a.pt = page_table->data;
    a.pt_i64 = page_table->dtype == DSV_I64;
    a.ps_shift = sh;
    a.n_phys = P;
    a.k_dst = static_cast<uint16_t*>(k_dst->data);
    a.kd_sp = k_dst->stride[0];
    a.kd_sh = k_dst->stride[1];
    a.kd_st = k_dst->stride[2];
    a.v_dst = static_cast<uint16_t*>(v_dst->data);
    a.vd_sp = v_dst->stride[0];
    a.vd_sh = v_dst->stride[1];
    a.vd_st = v_dst->stride[2];
  } else {
    int64_t S = -1;
    for (dsv_tensor* t : {k_dst, v_dst}) {
      const char* nm = t == k_dst ? "k_dst" : "v_dst";
      int64_t s3[3], st3[3];
      if ((rc = last3(t, nm, s3, st3)) != DSV_OK) return rc;
      if (s3[0] != Hk || s3[2] != D) return fail(DSV_ERR_INVALID, "%s must be [Hk, S, D]", nm);
      if (S >= 0 && s3[1] != S) return fail(DSV_ERR_INVALID, "k_dst and v_dst must hold the same tokens");
      S = s3[1];
      if (t == k_dst) {
        a.k_dst = static_cast<uint16_t*>(t->data);
        a.kd_sh = st3[0];
        a.kd_st = st3[1];
      } else {
        a.v_dst = static_cast<uint16_t*>(t->data);
        a.vd_sh = st3[0];
        a.vd_st = st3[1];
      }
    }
    if (start + M > S) return fail(DSV_ERR_INVALID, "tokens [start, start + M) exceed the cache");
  }
  // Aliasing: a thread reads one row's chunk pair and writes the same pair of
  // the destination row, so a row rotated in place is safe; any other overlap
  // of a read operand with a written one would let one thread overwrite what
  // another still has to read.  Exact in place: q_out == q, or (dense cache)
  // k / v already sitting in the destination's tree slots.
  {
    struct Span {
      const char* name;
      uintptr_t lo, hi;
    };
    auto span = [&](const char* nm, const dsv_tensor* t) {
      const uintptr_t lo = present(t) ? reinterpret_cast<uintptr_t>(t->data) : 0;
      return Span{nm, lo, present(t) ? lo + (uintptr_t)span_bytes(t) : lo};
    };
    auto in_place = [&](const dsv_tensor* src, const dsv_tensor* dst, int64_t dst_st, int64_t dst_sh) {
      if (!present(src) || !present(dst)) return false;
      const int o = src->ndim - 3;
      if (dst == q_out)
        return src->data == dst->data && src->stride[o] == dst->stride[dst->ndim - 3] &&
               src->stride[o + 1] == dst->stride[dst->ndim - 2];
      if (present(page_table)) return false;
      return reinterpret_cast<uintptr_t>(src->data) == reinterpret_cast<uintptr_t>(dst->data) + (uintptr_t)(start * dst_st * 2) &&
             src->stride[o] == dst_st && src->stride[o + 1] == dst_sh;
    };
    const dsv_tensor* srcs[5] = {k, v, q, cos, sin};
    const char* snames[5] = {"k", "v", "q", "cos", "sin"};
    const dsv_tensor* dsts[3] = {k_dst, v_dst, q_out};
    const char* dnames[3] = {"k_dst", "v_dst", "q_out"};
    const int64_t dst_st[3] = {a.kd_st, a.vd_st, 0}, dst_sh[3] = {a.kd_sh, a.vd_sh, 0};
    for (int si = 0; si < 5; ++si) {
      const Span s = span(snames[si], srcs[si]);
      if (s.hi == s.lo) continue;
      for (int di = 0; di < 3; ++di) {
        const Span d = span(dnames[di], dsts[di]);
        if (d.hi == d.lo || s.hi <= d.lo || d.hi <= s.lo) continue;
        if (si == di && in_place(srcs[si], dsts[di], dst_st[di], dst_sh[di])) continue;
        return fail(DSV_ERR_INVALID, "%s overlaps %s: inputs may not alias an output except row for row in place",
                    s.name, d.name);
      }
    }
    for (int i = 0; i < 3; ++i)
      for (int j = i + 1; j < 3; ++j) {
        const Span x = span(dnames[i], dsts[i]), y = span(dnames[j], dsts[j]);
        if (x.hi > x.lo && y.hi > y.lo && x.lo < y.hi && y.lo < x.hi)
          return fail(DSV_ERR_INVALID, "%s overlaps %s: outputs may not alias each other", x.name, y.name);
      }
  }
  if (g_dry_run) return DSV_OK;
  const hipError_t e = dsv::launch_append(a, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "kv append launch");
  return DSV_OK;
}

int dsv_kv_commit(const dsv_tensor* kv, const dsv_tensor* page_table, int64_t start, const dsv_tensor* path,
                  const dsv_tensor* info, int64_t tree, void* stream) {
  int rc;
  if (kv == nullptr || kv->ndim < 2 || kv->ndim > 6) return fail(DSV_ERR_INVALID, "kv must have 2..6 dimensions");
  if ((rc = check_nd(kv, "kv", kv->ndim)) != DSV_OK) return rc;
  if (kv->dtype != DSV_BF16 && kv->dtype != DSV_F16 && kv->dtype != DSV_F32)
    return fail(DSV_ERR_INVALID, "kv must be bf16, f16 or f32");
  const int nd = kv->ndim;
  const int esize = kv->dtype == DSV_F32 ? 4 : 2;
  if (kv->stride[nd - 1] != 1) return fail(DSV_ERR_INVALID, "kv innermost stride must be 1");
  const int64_t D = kv->shape[nd - 1];
  if ((D * esize) % 16 != 0) return fail(DSV_ERR_UNSUPPORTED, "token rows must be a multiple of 16 bytes");
  if ((reinterpret_cast<uintptr_t>(kv->data) & 15) != 0) return fail(DSV_ERR_INVALID, "kv must be 16-byte aligned");
  for (int d = 0; d < nd - 1; ++d)
    if ((kv->stride[d] * esize) % 16 != 0) return fail(DSV_ERR_INVALID, "kv strides must keep token rows 16-byte aligned");
  if (path == nullptr || (path->ndim != 1 && path->ndim != 2)) return fail(DSV_ERR_INVALID, "path must be [M] or [T, M]");
  if ((rc = check_nd(path, "path", path->ndim)) != DSV_OK) return rc;
  if (info == nullptr || (info->ndim != 1 && info->ndim != 2)) return fail(DSV_ERR_INVALID, "info must be [4] or [T, 4]");
  if ((rc = check_nd(info, "info", info->ndim)) != DSV_OK) return rc;
  if (path->dtype != DSV_I64 || info->dtype != DSV_I64) return fail(DSV_ERR_INVALID, "path and info must be int64");
  if (path->stride[path->ndim - 1] != 1 || info->stride[info->ndim - 1] != 1)
    return fail(DSV_ERR_INVALID, "path and info innermost stride must be 1");
  if (info->shape[info->ndim - 1] < 4) return fail(DSV_ERR_INVALID, "info rows must hold 4 entries");
  const int64_t T = path->ndim == 2 ? path->shape[0] : 1;
  if ((info->ndim == 2 ? info->shape[0] : 1) != T) return fail(DSV_ERR_INVALID, "path and info must hold the same trees");
  if (tree < 0 || tree >= T) return fail(DSV_ERR_INVALID, "tree %lld out of range", (long long)tree);
  const int64_t M = path->shape[path->ndim - 1];
  if (M < 1) return fail(DSV_ERR_INVALID, "path must hold at least one node");
  if (M * (D * esize / 16) > (int64_t)dsv::kCommitThreads * dsv::kCommitChunks)
    return fail(DSV_ERR_UNSUPPORTED, "M * row bytes above %d KiB", dsv::kCommitThreads * dsv::kCommitChunks / 64);
  if (start < 0) return fail(DSV_ERR_INVALID, "start must be >= 0");

  dsv::CommitArgs c{};
  c.data = kv->data;
  c.esize = esize;
  c.D = (int)D;
  c.start = start;
  c.M = (int)M;
  c.path = static_cast<const int64_t*>(path->data) + (path->ndim == 2 ? tree * path->stride[0] : 0);
  c.info = static_cast<const int64_t*>(info->data) + (info->ndim == 2 ? tree * info->stride[0] : 0);
  if (present(page_table)) {
    if (nd != 6) return fail(DSV_ERR_INVALID, "a paged kv must be [L, 2, P, Hk, page, D]");
    if ((rc = check_nd(page_table, "page_table", 1)) != DSV_OK) return rc;
    if (page_table->dtype != DSV_I32 && page_table->dtype != DSV_I64)
      return fail(DSV_ERR_INVALID, "page_table must be int32 or int64");
    if (page_table->stride[0] != 1) return fail(DSV_ERR_INVALID, "page_table stride must be 1");
    const int sh = log2_exact(kv->shape[4]);
    if (sh < 0) return fail(DSV_ERR_UNSUPPORTED, "page size must be a power of two");
    if (start + M > page_table->shape[0] * kv->shape[4])
      return fail(DSV_ERR_INVALID, "tokens [start, start + M) exceed the page table");
    c.nlead = 3;
    const int lead[3] = {0, 1, 3};
    c.rows = 1;
    for (int x = 0; x < 3; ++x) {
      c.lead_shape[x] = kv->shape[lead[x]];
      c.lead_stride[x] = kv->stride[lead[x]];
      c.rows *= kv->shape[lead[x]];
    }
    c.pt = page_table->data;
    c.pt_i64 = page_table->dtype == DSV_I64;
    c.ps_shift = sh;
    c.page_stride = kv->stride[2];
    c.n_phys = kv->shape[2];
    c.tok_stride = kv->stride[4];
  } else {
    if (nd < 3) return fail(DSV_ERR_INVALID, "a dense kv must be [..., S, D] with at least one leading dimension");
    if (start + M > kv->shape[nd - 2]) return fail(DSV_ERR_INVALID, "tokens [start, start + M) exceed the cache");
    c.nlead = nd - 2;
    c.rows = 1;
    for (int x = 0; x < nd - 2; ++x) {
      c.lead_shape[x] = kv->shape[x];
      c.lead_stride[x] = kv->stride[x];
      c.rows *= kv->shape[x];
    }
    c.tok_stride = kv->stride[nd - 2];
  }
  if (g_dry_run) return DSV_OK;
  const hipError_t e = dsv::launch_commit(c, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "kv commit launch");
  return DSV_OK;
}

int dsv_bundle_order(const dsv_tensor* parent, int64_t bundle_size, int64_t num_bundles, int64_t max_bundles,
                     dsv_tensor* perm, dsv_tensor* bundle_of, void* stream) {
  int rc;
  if (parent == nullptr || (parent->ndim != 1 && parent->ndim != 2)) return fail(DSV_ERR_INVALID, "parent must be [M] or [B, M]");
  if ((rc = check_nd(parent, "parent", parent->ndim)) != DSV_OK) return rc;
  if (parent->dtype != DSV_I32 && parent->dtype != DSV_I64) return fail(DSV_ERR_INVALID, "parent must be int32 or int64");
  const int nd = parent->ndim;
  const int64_t B = nd == 2 ? parent->shape[0] : 1, M = parent->shape[nd - 1];
  if (M < 1 || M > dsv::kBundleMaxNodes)
    return fail(DSV_ERR_UNSUPPORTED, "trees of %lld nodes are not supported (1..%d)", (long long)M, dsv::kBundleMaxNodes);
  if (B < 1 || B > 0x7fffffff) return fail(DSV_ERR_INVALID, "batch size out of range");
  if (num_bundles < 0 || num_bundles > 0x7fffffff) return fail(DSV_ERR_INVALID, "num_bundles must be >= 0");
  if (num_bundles == 0 && (bundle_size < 1 || bundle_size > 0x7fffffff))
    return fail(DSV_ERR_INVALID, "bundle_size must be >= 1");
  for (dsv_tensor* t : {perm, bundle_of}) {
    const char* nm = t == perm ? "perm" : "bundle_of";
    if (t == bundle_of && !present(t)) continue;
    if (t == nullptr || t->ndim != nd) return fail(DSV_ERR_INVALID, "%s must have the shape of parent", nm);
    if ((rc = check_nd(t, nm, nd)) != DSV_OK) return rc;
    if (t->dtype != DSV_I32) return fail(DSV_ERR_INVALID, "%s must be int32", nm);
    if (t->shape[nd - 1] != M || (nd == 2 && t->shape[0] != B)) return fail(DSV_ERR_INVALID, "%s must have the shape of parent", nm);
    if (t->stride[nd - 1] != 1 || (nd == 2 && B > 1 && t->stride[0] != M)) return fail(DSV_ERR_INVALID, "%s must be contiguous", nm);
  }
  dsv::BundleArgs a{};
  a.B = (int)B;
  a.M = (int)M;
  a.parent = parent->data;
  a.p_i64 = parent->dtype == DSV_I64;
  a.p_st = nd == 2 ? parent->stride[0] : 0;
  a.p_sm = parent->stride[nd - 1];
  a.bundle_size = num_bundles > 0 ? 1 : (int)bundle_size;
  a.num_bundles = (int)num_bundles;
  // The scheduler stops once it holds max_bundles bundles, checked after each
  // one is added: at least one bundle is always emitted.
  a.max_bundles = (int)std::min<int64_t>(std::max<int64_t>(max_bundles, 1), 0x7fffffff);
  a.perm = static_cast<int32_t*>(perm->data);
  a.bundle_of = present(bundle_of) ? static_cast<int32_t*>(bundle_of->data) : nullptr;
  if (g_dry_run) return DSV_OK;
  const hipError_t e = dsv::launch_bundle_order(a, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "bundle order launch");
  return DSV_OK;
}

}  // extern "C"

// Validation and arguments shared by both acceptance entry points: tree
// shape (T, M), vocabulary V, the tree tensors and the outputs.
static int accept_common(int mode, int64_t T, int64_t M, int64_t V, const dsv_tensor* draft,
                         const dsv_tensor* parent, const dsv_tensor* pos, int64_t max_hops, float temperature,
                         float posterior_threshold, float posterior_alpha, dsv_tensor* out_path,
                         dsv_tensor* out_tokens, dsv_tensor* out_info, dsv_tensor* out_next, dsv::AcceptArgs& a) {
  int rc;
  if (M < 1 || M > 1024) return fail(DSV_ERR_UNSUPPORTED, "trees of %lld nodes are not supported (1..1024)", (long long)M);
  if (T < 1 || T > (1 << 20)) return fail(DSV_ERR_INVALID, "tree count %lld out of range (1..2^20)", (long long)T);
  if (V < 1 || V > 0x7fffffff) return fail(DSV_ERR_INVALID, "vocab size out of range");
  if ((rc = check_nd(draft, "draft", 2)) != DSV_OK) return rc;
  if (draft->dtype != DSV_I64 || draft->shape[0] != T || draft->shape[1] != M)
    return fail(DSV_ERR_INVALID, "draft must be int64 [T, M]");
  // A root-only tree (M == 1) has an empty parent tensor, possibly without
  // storage; nothing reads it then.
  if (M > 1) {
    if ((rc = check_nd(parent, "parent", 2)) != DSV_OK) return rc;
  } else if (parent == nullptr || parent->ndim != 2) {
    return fail(DSV_ERR_INVALID, "parent must be int64 [T, M-1]");
  }
  if (parent->dtype != DSV_I64 || parent->shape[0] != T || parent->shape[1] != M - 1)
    return fail(DSV_ERR_INVALID, "parent must be int64 [T, M-1]");
  if (pos == nullptr || (pos->ndim != 1 && pos->ndim != 2)) return fail(DSV_ERR_INVALID, "pos must be [M] or [T, M]");
  if ((rc = check_nd(pos, "pos", pos->ndim)) != DSV_OK) return rc;
  if (pos->dtype != DSV_I64 || pos->shape[pos->ndim - 1] != M) return fail(DSV_ERR_INVALID, "pos must be int64 with M entries");
  if (pos->ndim == 2 && pos->shape[0] != T && pos->shape[0] != 1) return fail(DSV_ERR_INVALID, "pos batch must be 1 or T");
  if (max_hops < 0) return fail(DSV_ERR_INVALID, "max_hops must be >= 0");
  if (mode == DSV_ACCEPT_TYPICAL && !(temperature > 0.f)) return fail(DSV_ERR_INVALID, "temperature must be > 0");
  auto chk_out = [&](const dsv_tensor* t, const char* name, int64_t cols) -> int {
    int r;
    if ((r = check_nd(t, name, 2)) != DSV_OK) return r;
    if (t->dtype != DSV_I64 || t->shape[0] != T || t->shape[1] != cols || t->stride[1] != 1)
      return fail(DSV_ERR_INVALID, "%s must be contiguous int64 [T, %lld]", name, (long long)cols);
    return DSV_OK;
  };
  if ((rc = chk_out(out_path, "out_path", M)) != DSV_OK) return rc;
  if ((rc = chk_out(out_tokens, "out_tokens", M)) != DSV_OK) return rc;
  if ((rc = chk_out(out_info, "out_info", 4)) != DSV_OK) return rc;
  if (present(out_next) && (rc = chk_out(out_next, "out_next", M)) != DSV_OK) return rc;

  a.mode = mode;
  a.T = (int)T;
  a.M = (int)M;
  a.V = V;
  a.draft = static_cast<const int64_t*>(draft->data);
  a.d_st = draft->stride[0];
  a.d_sm = draft->stride[1];
  a.parent = static_cast<const int64_t*>(parent->data);
  a.p_st = parent->stride[0];
  a.p_sm = parent->stride[1];
  a.pos = static_cast<const int64_t*>(pos->data);
  a.pos_st = (pos->ndim == 2 && pos->shape[0] > 1) ? pos->stride[0] : 0;
  a.pos_sm = pos->stride[pos->ndim - 1];
  a.max_hops = (int)std::min<int64_t>(max_hops, 1 << 20);
  a.inv_temp = mode == DSV_ACCEPT_TYPICAL ? 1.f / temperature : 1.f;
  a.temperature = mode == DSV_ACCEPT_TYPICAL ? temperature : 1.f;  // the typical re-check's T
  a.eps = posterior_threshold;
  a.alpha = posterior_alpha;
  a.out_path = static_cast<int64_t*>(out_path->data);
  a.op_st = out_path->stride[0];
  a.out_tok = static_cast<int64_t*>(out_tokens->data);
  a.ot_st = out_tokens->stride[0];
  a.out_info = static_cast<int64_t*>(out_info->data);
  a.oi_st = out_info->stride[0];
  if (present(out_next)) {
    a.out_next = static_cast<int64_t*>(out_next->data);
    a.on_st = out_next->stride[0];
  }
  return DSV_OK;
}

extern "C" {

int dsv_tree_accept(int mode, const dsv_tensor* logits, const dsv_tensor* draft, const dsv_tensor* parent,
                    const dsv_tensor* pos, int64_t max_hops, float temperature, float posterior_threshold,
                    float posterior_alpha, dsv_tensor* out_path, dsv_tensor* out_tokens, dsv_tensor* out_info,
                    dsv_tensor* out_next, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if (mode != DSV_ACCEPT_GREEDY && mode != DSV_ACCEPT_TYPICAL) return fail(DSV_ERR_INVALID, "unknown acceptance mode %d", mode);
  if ((rc = check_nd(logits, "logits", 3)) != DSV_OK) return rc;
  if (logits->dtype != DSV_BF16 && logits->dtype != DSV_F16 && logits->dtype != DSV_F32)
    return fail(DSV_ERR_INVALID, "logits must be bf16, f16 or f32");
  if (logits->stride[2] != 1) return fail(DSV_ERR_INVALID, "logits vocab stride must be 1");
  const int64_t T = logits->shape[0], M = logits->shape[1], V = logits->shape[2];
  AcceptArgs a{};
  if ((rc = accept_common(mode, T, M, V, draft, parent, pos, max_hops, temperature, posterior_threshold,
                          posterior_alpha, out_path, out_tokens, out_info, out_next, a)) != DSV_OK)
    return rc;
  const size_t need = dsv_accept_workspace_bytes(T, M, V);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(DSV_ERR_WORKSPACE, "workspace of %zu bytes required (got %zu)", need, workspace_bytes);
  if ((reinterpret_cast<uintptr_t>(workspace) & 255) != 0) return fail(DSV_ERR_WORKSPACE, "workspace must be 256-byte aligned");

  a.logits = logits->data;
  a.l_dtype = logits->dtype;
  a.l_st = logits->stride[0];
  a.l_sm = logits->stride[1];
  dsv::accept_chunking(a, device_cus());
  const size_t rows = (size_t)T * M * a.nchunk;
  a.rstat = static_cast<float4*>(workspace);
  a.rstat2 = reinterpret_cast<float*>(static_cast<char*>(workspace) + align_up(rows * 16, 256));
  if (g_dry_run) return DSV_OK;
  hipEvent_t ev0, ev1;
  take_events(ev0, ev1);
  hipError_t e = dsv::launch_accept(a, static_cast<hipStream_t>(stream), ev0, ev1);
  if (e != hipSuccess) return hip_fail(e, "acceptance kernel launch");
  return DSV_OK;
}

int dsv_tree_accept_sample(const dsv_tensor* logits, const dsv_tensor* draft, const dsv_tensor* parent,
                           const dsv_tensor* pos, int64_t max_hops, float temperature, float top_p, int64_t top_k,
                           uint64_t seed, dsv_tensor* out_path, dsv_tensor* out_tokens, dsv_tensor* out_info,
                           dsv_tensor* out_next, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_nd(logits, "logits", 3)) != DSV_OK) return rc;
  if (logits->dtype != DSV_BF16 && logits->dtype != DSV_F16 && logits->dtype != DSV_F32)
    return fail(DSV_ERR_INVALID, "logits must be bf16, f16 or f32");
  if (logits->stride[2] != 1) return fail(DSV_ERR_INVALID, "logits vocab stride must be 1");
  // The reference builds its warpers only when temperature > 1e-5 (compared in
  // double precision, draft/tree_verification.py:21); at or below it the
  // walk is greedy (dsv_tree_accept).
  if (!((double)temperature > 1e-5) || !(temperature < __builtin_huge_valf()))
    return fail(DSV_ERR_INVALID, "temperature must be > 1e-5 (smaller temperatures are greedy acceptance)");
  if (!(top_p >= 0.f && top_p <= 1.f)) return fail(DSV_ERR_INVALID, "top_p must lie in [0, 1]");
  if (top_k < 0) return fail(DSV_ERR_INVALID, "top_k must be >= 0");
  const int64_t T = logits->shape[0], M = logits->shape[1], V = logits->shape[2];
  AcceptArgs a{};
  if ((rc = accept_common(DSV_ACCEPT_GREEDY, T, M, V, draft, parent, pos, max_hops, 1.f, 0.f, 0.f, out_path,
                          out_tokens, out_info, out_next, a)) != DSV_OK)
    return rc;
  const size_t need = dsv_accept_workspace_bytes(T, M, V);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(DSV_ERR_WORKSPACE, "workspace of %zu bytes required (got %zu)", need, workspace_bytes);
  if ((reinterpret_cast<uintptr_t>(workspace) & 255) != 0) return fail(DSV_ERR_WORKSPACE, "workspace must be 256-byte aligned");

  a.mode = 2;
  a.logits = logits->data;
  a.l_dtype = logits->dtype;
  a.l_st = logits->stride[0];
  a.l_sm = logits->stride[1];
  a.temperature = temperature;
  // The warpers that apply, as prepare_logits_processor builds them
  // (draft/tree_verification.py:15-32): top-p when 1e-8 <= top_p < 1, top-k when > 0.
  a.top_p_q = (top_p >= 1e-8f && top_p < 1.f) ? (uint32_t)std::nearbyint((double)top_p * 4294967296.0) : 0u;
  a.top_k = top_k;
  a.seed = seed;
  dsv::accept_chunking(a, device_cus());
  const size_t rows = (size_t)T * M * a.nchunk;
  char* ws = static_cast<char*>(workspace);
  a.rstat = reinterpret_cast<float4*>(ws);
  const size_t max_rows = (size_t)T * M * dsv::accept_max_chunks(V);
  a.sel = (a.top_p_q != 0 || top_k > 0)
              ? reinterpret_cast<uint4*>(ws + align_up(max_rows * 16, 256) + align_up(max_rows * 4, 256))
              : nullptr;
  (void)rows;
  if (g_dry_run) return DSV_OK;
  hipEvent_t ev0, ev1;
  take_events(ev0, ev1);
  hipError_t e = dsv::launch_sample(a, static_cast<hipStream_t>(stream), ev0, ev1);
  if (e != hipSuccess) return hip_fail(e, "sampling acceptance launch");
  return DSV_OK;
}

size_t dsv_lmhead_accept_workspace_bytes(int64_t T, int64_t M, int64_t V) {
  if (T <= 0 || M <= 0 || V <= 0) return 0;
  const size_t R = (size_t)T * M, parts = R * (size_t)dsv::lmhead_blocks(V);
  return align_up(parts * 16, 256) + align_up(parts * 4, 256) + align_up(R * 16, 256) + 2 * align_up(R * 4, 256);
}

int dsv_lmhead_accept(int mode, const dsv_tensor* hidden, const dsv_tensor* weight, const dsv_tensor* draft,
                      const dsv_tensor* parent, const dsv_tensor* pos, int64_t max_hops, float temperature,
                      float posterior_threshold, float posterior_alpha, dsv_tensor* out_path, dsv_tensor* out_tokens,
                      dsv_tensor* out_info, dsv_tensor* out_next, dsv_tensor* logits_out, void* workspace,
                      size_t workspace_bytes, void* stream) {
  int rc;
  if (mode != DSV_ACCEPT_GREEDY && mode != DSV_ACCEPT_TYPICAL) return fail(DSV_ERR_INVALID, "unknown acceptance mode %d", mode);
  if ((rc = check_nd(hidden, "hidden", 3)) != DSV_OK) return rc;
  if ((rc = check_nd(weight, "weight", 2)) != DSV_OK) return rc;
  if (hidden->dtype != DSV_BF16 || weight->dtype != DSV_BF16) return fail(DSV_ERR_UNSUPPORTED, "hidden and weight must be bf16");
  const int64_t T = hidden->shape[0], M = hidden->shape[1], Dm = hidden->shape[2], V = weight->shape[0];
  if (weight->shape[1] != Dm) return fail(DSV_ERR_INVALID, "weight must be [V, %lld]", (long long)Dm);
  if (Dm < dsv::kLmK || Dm % dsv::kLmK != 0 || Dm > (1 << 20))
    return fail(DSV_ERR_UNSUPPORTED, "hidden size %lld must be a positive multiple of %d", (long long)Dm, dsv::kLmK);
  if (hidden->stride[2] != 1 || weight->stride[1] != 1) return fail(DSV_ERR_INVALID, "hidden and weight rows must be contiguous");
  if (hidden->stride[0] != M * hidden->stride[1] && T > 1)
    return fail(DSV_ERR_INVALID, "hidden rows of all trees must share one stride ([T*M, Dm] view)");
  if ((reinterpret_cast<uintptr_t>(hidden->data) & 15) != 0 || (reinterpret_cast<uintptr_t>(weight->data) & 15) != 0 ||
      hidden->stride[1] % 8 != 0 || weight->stride[0] % 8 != 0)
    return fail(DSV_ERR_INVALID, "hidden and weight rows must be 16-byte aligned");
  AcceptArgs a{};
  if ((rc = accept_common(mode, T, M, V, draft, parent, pos, max_hops, temperature, posterior_threshold,
                          posterior_alpha, out_path, out_tokens, out_info, out_next, a)) != DSV_OK)
    return rc;
  if (present(logits_out)) {
    if ((rc = check_nd(logits_out, "logits_out", 3)) != DSV_OK) return rc;
    if (logits_out->dtype != DSV_BF16 || logits_out->shape[0] != T || logits_out->shape[1] != M ||
        logits_out->shape[2] != V || logits_out->stride[2] != 1 || (T > 1 && logits_out->stride[0] != M * logits_out->stride[1]))
      return fail(DSV_ERR_INVALID, "logits_out must be bf16 [T, M, V] with rows of one stride");
  }
  const size_t need = dsv_lmhead_accept_workspace_bytes(T, M, V);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(DSV_ERR_WORKSPACE, "workspace of %zu bytes required (got %zu)", need, workspace_bytes);
  if ((reinterpret_cast<uintptr_t>(workspace) & 255) != 0) return fail(DSV_ERR_WORKSPACE, "workspace must be 256-byte aligned");

  dsv::LmArgs lm{};
  lm.mode = mode;
  lm.h = static_cast<const uint16_t*>(hidden->data);
  lm.ldh = hidden->stride[1];
  lm.w = static_cast<const uint16_t*>(weight->data);
  lm.ldw = weight->stride[0];
  lm.R = (int)(T * M);
  lm.Dm = (int)Dm;
  lm.V = V;
  lm.T = (int)T;
  lm.M = (int)M;
  lm.draft = a.draft;
  lm.d_st = a.d_st;
  lm.d_sm = a.d_sm;
  lm.parent = a.parent;
  lm.p_st = a.p_st;
  lm.p_sm = a.p_sm;
  lm.inv_temp = a.inv_temp;
  lm.nblk = dsv::lmhead_blocks(V);
  a.cus = device_cus();
  const size_t R = (size_t)T * M, parts = R * (size_t)lm.nblk;
  char* ws = static_cast<char*>(workspace);
  lm.rstat = reinterpret_cast<float4*>(ws);
  ws += align_up(parts * 16, 256);
  lm.rstat2 = reinterpret_cast<float*>(ws);
  ws += align_up(parts * 4, 256);
  a.rstat = reinterpret_cast<float4*>(ws);
  ws += align_up(R * 16, 256);
  a.rstat2 = reinterpret_cast<float*>(ws);
  ws += align_up(R * 4, 256);
  lm.xtok = reinterpret_cast<float*>(ws);
  a.xtok = lm.xtok;
  a.nchunk = 1;
  a.chunk = V;
  if (present(logits_out)) {
    lm.lout = static_cast<uint16_t*>(logits_out->data);
    lm.lo_sr = logits_out->stride[1];
    // The typical test re-decides its near-threshold nodes from the written
    // logits (kernel 5 writes them before the walk runs, on this stream).
    a.logits = logits_out->data;
    a.l_dtype = DSV_BF16;
    a.l_st = logits_out->stride[0];
    a.l_sm = logits_out->stride[1];
  }
  if (g_dry_run) return DSV_OK;
  hipEvent_t ev0, ev1;
  take_events(ev0, ev1);
  hipError_t e;
  if (ev0 != nullptr && (e = hipEventRecord(ev0, static_cast<hipStream_t>(stream))) != hipSuccess)
    return hip_fail(e, "timing event");
  e = dsv::launch_lmhead_accept(a, lm, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "lm_head acceptance launch");
  if (ev1 != nullptr && (e = hipEventRecord(ev1, static_cast<hipStream_t>(stream))) != hipSuccess)
    return hip_fail(e, "timing event");
  return DSV_OK;
}

}  // extern "C"

// ---------------------------------------------------------------------------
// Verification of drafted tokens from given random numbers
// ---------------------------------------------------------------------------

namespace {

struct SpecPlan {
  int nwg = 1, own = 1, step = 0, step1 = 0;
  size_t state_bytes = 0, rej_bytes = 0, total = 0;
};

// Workgroups per tree: one per CU in all, at most so many that each wave has a
// segment of the row.  One up to 32768 entries: its sweep is longer by at most 2 us,
// and the second launch costs the caller 2.5 (4 chains over pairs of rows, us in a
// graph and called: 16384 entries 8.1 and 15.9 by one workgroup, 8.8 and 18.6 by
// several; 32000 10.4 and 16.0, 8.9 and 18.5; 64000 14.4 and 15.8, 8.7 and 18.4;
// 128256 22.6 and 22.9, 9.1 and 18.0).
bool spec_plan(int64_t T, int64_t M, int64_t V, SpecPlan& p) {
  if (M < 1 || M > dsv::kSpecMaxM || T < 1 || T > (1 << 20) || V < 1 || V > 0x7fffffff) return false;
  const int64_t waves = dsv::kSpecThreads / 64, nseg = (V + dsv::kSpecSeg - 1) / dsv::kSpecSeg;
  const int64_t most = nseg <= 64 ? 1 : std::min<int64_t>((nseg + waves - 1) / waves, 64);
  p.nwg = (int)std::max<int64_t>(1, std::min(most, (int64_t)device_cus() / T));
  // A wave's segments in up to 4 slots: the draw walks one slot again.
  const int64_t each = (nseg + waves * p.nwg - 1) / (waves * p.nwg);
  p.own = (int)std::min<int64_t>(each, dsv::kSpecSlots / waves);
  p.step = (int)((each + p.own - 1) / p.own);
  p.step1 = (int)((nseg + waves - 1) / waves);
  if (p.nwg > 1) {
    p.state_bytes = align_up((size_t)T * sizeof(dsv::SpecState), 256);
    p.rej_bytes = align_up((size_t)T * M * sizeof(int32_t), 256);
    p.total = p.state_bytes + p.rej_bytes + align_up((size_t)T * p.nwg * waves * p.own * sizeof(double), 256);
  }
  return true;
}

int check_workspace(size_t need, void* ws, size_t ws_bytes) {
  if (ws == nullptr || ws_bytes < need)
    return fail(DSV_ERR_WORKSPACE, "workspace of %zu bytes required (got %zu)", need, ws == nullptr ? 0 : ws_bytes);
  if ((reinterpret_cast<uintptr_t>(ws) & 255) != 0) return fail(DSV_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  return DSV_OK;
}

// Byte ranges that share an address.
bool overlap(const Extent& x, const Extent& y) { return x.lo < y.hi && y.lo < x.hi; }

}  // namespace

extern "C" {

size_t dsv_spec_workspace_bytes(int64_t T, int64_t M, int64_t V) {
  SpecPlan p;
  return spec_plan(T, M, V, p) ? p.total : 0;
}

int dsv_spec_accept(const dsv_tensor* target, const dsv_tensor* draft, const dsv_tensor* parent,
                    const dsv_tensor* uniform, const dsv_tensor* draft_probs, dsv_tensor* out_path,
                    dsv_tensor* out_tokens, dsv_tensor* out_info, void* workspace, size_t workspace_bytes,
                    void* stream) {
  int rc;
  if ((rc = check_nd(target, "target", 3)) != DSV_OK) return rc;
  if (target->dtype != DSV_BF16 && target->dtype != DSV_F16 && target->dtype != DSV_F32)
    return fail(DSV_ERR_INVALID, "target must be bf16, f16 or f32 (got %s)", dt_name(target->dtype));
  const int64_t T = target->shape[0], M = target->shape[1], V = target->shape[2];
  if (target->stride[2] != 1) return fail(DSV_ERR_INVALID, "target: vocab stride must be 1");
  SpecPlan p;
  if (!spec_plan(T, M, V, p))
    return fail(DSV_ERR_UNSUPPORTED, "sizes out of range: %lld trees (1..2^20) of %lld nodes (1..%d) over %lld tokens (1..2^31 - 1)",
                (long long)T, (long long)M, dsv::kSpecMaxM, (long long)V);
  if ((rc = check_nd(draft, "draft", 2)) != DSV_OK) return rc;
  if (draft->dtype != DSV_I64 || draft->shape[0] != T || draft->shape[1] != M)
    return fail(DSV_ERR_INVALID, "draft must be int64 [T, M]");
  // A root-only tree has an empty parent tensor, possibly without storage.
  if (M > 1 && (rc = check_nd(parent, "parent", 2)) != DSV_OK) return rc;
  if (parent == nullptr || parent->ndim != 2 || parent->dtype != DSV_I64 || parent->shape[0] != T ||
      parent->shape[1] != M - 1)
    return fail(DSV_ERR_INVALID, "parent must be int64 [T, M-1]");
  if ((rc = check_nd(uniform, "uniform", 2)) != DSV_OK) return rc;
  if (uniform->dtype != DSV_F32 || uniform->shape[0] != T || uniform->shape[1] != M)
    return fail(DSV_ERR_INVALID, "uniform must be float32 [T, M]");
  if (present(draft_probs)) {
    if ((rc = check_nd(draft_probs, "draft_probs", 3)) != DSV_OK) return rc;
    if (draft_probs->dtype != target->dtype || draft_probs->shape[0] != T || draft_probs->shape[1] != M ||
        draft_probs->shape[2] != V || draft_probs->stride[2] != 1)
      return fail(DSV_ERR_INVALID, "draft_probs must have target's dtype and shape [T, M, V], vocab stride 1");
  }
  struct Out { dsv_tensor* t; const char* name; int64_t cols; };
  const Out outs[3] = {{out_path, "out_path", M}, {out_tokens, "out_tokens", M}, {out_info, "out_info", 4}};
  const Extent ins[5] = {extent_of("target", target), extent_of("draft", draft),
                         M > 1 ? extent_of("parent", parent) : Extent{"parent", 0, 0},
                         extent_of("uniform", uniform), extent_of("draft_probs", draft_probs)};
  for (const Out& o : outs) {
    if ((rc = check_nd(o.t, o.name, 2)) != DSV_OK) return rc;
    if (o.t->dtype != DSV_I64 || o.t->shape[0] != T || o.t->shape[1] != o.cols || o.t->stride[1] != 1)
      return fail(DSV_ERR_INVALID, "%s must be int64 [T, %lld] with innermost stride 1", o.name, (long long)o.cols);
    if (T > 1 && o.t->stride[0] < o.cols) return fail(DSV_ERR_INVALID, "%s: rows overlap", o.name);
    // A tree's outputs are written while others' inputs are still read.
    for (const Extent& in : ins)
      if (overlap(extent_of(o.name, o.t), in)) return fail(DSV_ERR_INVALID, "%s overlaps %s", o.name, in.name);
  }
  if (overlap(extent_of("", out_path), extent_of("", out_tokens)) || overlap(extent_of("", out_path), extent_of("", out_info)) ||
      overlap(extent_of("", out_tokens), extent_of("", out_info)))
    return fail(DSV_ERR_INVALID, "outputs overlap each other");
  if (p.total > 0 && (rc = check_workspace(p.total, workspace, workspace_bytes)) != DSV_OK) return rc;

  dsv::SpecArgs a{};
  a.dtype = target->dtype;
  a.T = (int)T;
  a.M = (int)M;
  a.V = V;
  a.target = target->data;
  a.t_st = target->stride[0];
  a.t_sm = target->stride[1];
  if (present(draft_probs)) {
    a.dprobs = draft_probs->data;
    a.q_st = draft_probs->stride[0];
    a.q_sm = draft_probs->stride[1];
  }
  a.draft = static_cast<const int64_t*>(draft->data);
  a.d_st = draft->stride[0];
  a.d_sm = draft->stride[1];
  a.parent = static_cast<const int64_t*>(parent->data);
  a.p_st = parent->stride[0];
  a.p_sm = parent->stride[1];
  a.uniform = static_cast<const float*>(uniform->data);
  a.u_st = uniform->stride[0];
  a.u_sm = uniform->stride[1];
  a.out_path = static_cast<int64_t*>(out_path->data);
  a.op_st = out_path->stride[0];
  a.out_tok = static_cast<int64_t*>(out_tokens->data);
  a.ot_st = out_tokens->stride[0];
  a.out_info = static_cast<int64_t*>(out_info->data);
  a.oi_st = out_info->stride[0];
  a.nwg = p.nwg;
  a.own = p.own;
  a.step = p.step;
  a.step1 = p.step1;
  if (p.total > 0) {
    char* w = static_cast<char*>(workspace);
    a.state = reinterpret_cast<dsv::SpecState*>(w);
    a.rej = reinterpret_cast<int32_t*>(w + p.state_bytes);
    a.part = reinterpret_cast<double*>(w + p.state_bytes + p.rej_bytes);
  }
  if (g_dry_run) return DSV_OK;
  const hipError_t e = dsv::launch_spec(a, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "speculative acceptance launch");
  return DSV_OK;
}

}  // extern "C"

// ---------------------------------------------------------------------------
// Pages
// ---------------------------------------------------------------------------

namespace {

struct PagesPlan {
  size_t list_bytes = 0, off_bytes = 0, total = 0;
};

bool pages_plan(int64_t P, int64_t B, int64_t n, PagesPlan& p) {
  if (P < 0 || P > 0x7fffffff || B < 0 || B > dsv::kPageMaxSeqs || n < 0 || n > dsv::kPageMaxSeqs) return false;
  // Page lists: fork 3 n (source, destination, free pages), extend P, compact
  // P / 2 + P / 2 + P; behind them extend's offsets and the state words.
  p.list_bytes = align_up((size_t)std::max<int64_t>(2 * P + 2, 3 * n) * sizeof(int32_t), 256);
  p.off_bytes = align_up((size_t)B * sizeof(int64_t), 256);
  p.total = p.list_bytes + p.off_bytes + 256;
  return true;
}

int check_book(const dsv_tensor* table, const dsv_tensor* ref, const dsv_tensor* lens, int64_t page_size,
               dsv::PageBook& b) {
  int rc;
  if ((rc = check_nd(table, "page_table", 2)) != DSV_OK) return rc;
  if (table->dtype != DSV_I32 || table->stride[1] != 1)
    return fail(DSV_ERR_INVALID, "page_table must be int32 [B, n_logical] with innermost stride 1");
  if (table->shape[0] > 1 && table->stride[0] < table->shape[1])
    return fail(DSV_ERR_INVALID, "page_table rows overlap");
  if ((rc = check_nd(ref, "refcount", 1)) != DSV_OK) return rc;
  if (ref->dtype != DSV_I32 || (ref->shape[0] > 1 && ref->stride[0] != 1))
    return fail(DSV_ERR_INVALID, "refcount must be contiguous int32 [P]");
  const int sh = log2_exact(page_size);
  if (sh < 0) return fail(DSV_ERR_UNSUPPORTED, "page_size %lld must be a power of two", (long long)page_size);
  b.table = static_cast<int32_t*>(table->data);
  b.t_sb = table->stride[0];
  b.B = table->shape[0];
  b.n_log = table->shape[1];
  b.ref = static_cast<int32_t*>(ref->data);
  b.P = ref->shape[0];
  b.ps_shift = sh;
  if (b.B > dsv::kPageMaxSeqs) return fail(DSV_ERR_UNSUPPORTED, "more than %d sequences", dsv::kPageMaxSeqs);
  if (b.P > 0x7fffffff) return fail(DSV_ERR_UNSUPPORTED, "more than 2^31 - 1 pages");
  if (b.n_log > ((int64_t)1 << 40) >> sh) return fail(DSV_ERR_UNSUPPORTED, "page_table rows beyond 2^40 tokens");
  if (overlap(extent_of("", table), extent_of("", ref))) return fail(DSV_ERR_INVALID, "page_table overlaps refcount");
  if (lens != nullptr) {
    if ((rc = check_nd(lens, "seqlens", 1)) != DSV_OK) return rc;
    if ((lens->dtype != DSV_I32 && lens->dtype != DSV_I64) || lens->shape[0] != b.B ||
        (b.B > 1 && lens->stride[0] != 1))
      return fail(DSV_ERR_INVALID, "seqlens must be contiguous int32 or int64 [B]");
    if (lens->dtype == DSV_I32 && b.n_log > 0x7fffffff >> sh)
      return fail(DSV_ERR_UNSUPPORTED, "table rows beyond 2^31 tokens need int64 seqlens");
    if (overlap(extent_of("", lens), extent_of("", table)) || overlap(extent_of("", lens), extent_of("", ref)))
      return fail(DSV_ERR_INVALID, "seqlens overlaps page_table or refcount");
    b.lens = lens->data;
    b.lens_i64 = lens->dtype == DSV_I64;
  }
  return DSV_OK;
}

// An index argument: [n] int32|int64 that no output overlaps.
int check_index(const dsv_tensor* t, const char* name, int64_t n, const dsv_tensor* const* outs, int n_outs,
                dsv::PageIndex& x) {
  int rc;
  // (An empty list may come without storage; nothing reads it.)
  if ((t == nullptr || t->ndim != 1 || t->shape[0] != 0) && (rc = check_nd(t, name, 1)) != DSV_OK) return rc;
  if (t->dtype != DSV_I32 && t->dtype != DSV_I64) return fail(DSV_ERR_INVALID, "%s must be int32 or int64", name);
  if (t->shape[0] != n) return fail(DSV_ERR_INVALID, "%s must have %lld entries", name, (long long)n);
  for (int i = 0; i < n_outs; ++i)
    if (outs[i] != nullptr && overlap(extent_of("", t), extent_of("", outs[i])))
      return fail(DSV_ERR_INVALID, "%s overlaps a tensor that the call writes", name);
  x.p = t->data;
  x.is64 = t->dtype == DSV_I64;
  x.stride = t->stride[0];
  return DSV_OK;
}

int check_info(const dsv_tensor* info, const dsv_tensor* const* others, int n) {
  int rc;
  if ((rc = check_nd(info, "info", 1)) != DSV_OK) return rc;
  if (info->dtype != DSV_I32 || info->shape[0] != 3 || info->stride[0] != 1)
    return fail(DSV_ERR_INVALID, "info must be contiguous int32 [3]");
  for (int i = 0; i < n; ++i)
    if (others[i] != nullptr && overlap(extent_of("", info), extent_of("", others[i])))
      return fail(DSV_ERR_INVALID, "info overlaps another argument");
  return DSV_OK;
}

int check_page_data(const dsv_tensor* kv, int64_t P, dsv::PageData& d) {
  int rc;
  if ((rc = check_nd(kv, "kv_pages", 6)) != DSV_OK) return rc;
  if ((rc = check_vec16(kv, "kv_pages")) != DSV_OK) return rc;
  if (kv->shape[1] != 2) return fail(DSV_ERR_INVALID, "kv_pages dim 1 must be 2 (K, V)");
  if (kv->shape[2] != P)
    return fail(DSV_ERR_INVALID, "kv_pages holds %lld pages, refcount %lld", (long long)kv->shape[2], (long long)P);
  const int es = elem_size(kv->dtype);
  if ((kv->shape[5] * es) % 16 != 0) return fail(DSV_ERR_UNSUPPORTED, "token rows must be a multiple of 16 bytes");
  if (kv->shape[0] > (1 << 20)) return fail(DSV_ERR_UNSUPPORTED, "more than 2^20 layers");
  if (kv->shape[3] * kv->shape[4] * (kv->shape[5] * es / 16) > ((int64_t)1 << 26))
    return fail(DSV_ERR_UNSUPPORTED, "a page of one layer beyond 1 GiB");
  // Pages that share bytes would be copied into each other: strides from the
  // smallest up must each step over what lies below.
  int order[6];
  int nd = 0;
  for (int i = 0; i < 6; ++i)
    if (kv->shape[i] > 1) order[nd++] = i;
  std::sort(order, order + nd, [&](int x, int y) { return kv->stride[x] < kv->stride[y]; });
  int64_t extent = 1;
  for (int i = 0; i < nd; ++i) {
    const int x = order[i];
    if (kv->stride[x] < extent) return fail(DSV_ERR_INVALID, "kv_pages overlaps itself (stride[%d])", x);
    extent = kv->stride[x] * (kv->shape[x] - 1) + extent;
  }
  d.kv = static_cast<char*>(kv->data);
  d.s_l = kv->stride[0] * es;
  d.s_h = kv->stride[1] * es;
  d.s_p = kv->stride[2] * es;
  d.s_1 = kv->stride[3] * es;
  d.s_2 = kv->stride[4] * es;
  d.n_l = (int)kv->shape[0];
  d.n1 = (int)kv->shape[3];
  d.n2 = (int)kv->shape[4];
  d.row16 = (int)(kv->shape[5] * es / 16);
  d.contiguous = (d.n2 <= 1 || kv->stride[4] == kv->shape[5]) && (d.n1 <= 1 || kv->stride[3] == kv->shape[4] * kv->shape[5]);
  return DSV_OK;
}

}  // namespace

extern "C" {

size_t dsv_pages_workspace_bytes(int64_t P, int64_t B, int64_t n) {
  PagesPlan p;
  return pages_plan(P, B, n, p) ? p.total : 0;
}

int dsv_pages_fork(const dsv_tensor* kv_pages, const dsv_tensor* page_table, const dsv_tensor* refcount,
                   const dsv_tensor* seqlens, const dsv_tensor* parents, const dsv_tensor* children, dsv_tensor* info,
                   void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  dsv::ForkArgs a{};
  if (kv_pages == nullptr || kv_pages->ndim != 6) return fail(DSV_ERR_INVALID, "kv_pages must be [L, 2, P, Hk, page, D]");
  if ((rc = check_nd(seqlens, "seqlens", 1)) != DSV_OK) return rc;
  if ((rc = check_book(page_table, refcount, seqlens, kv_pages->shape[4], a.book)) != DSV_OK) return rc;
  if ((rc = check_page_data(kv_pages, a.book.P, a.data)) != DSV_OK) return rc;
  const dsv_tensor* written[5] = {kv_pages, page_table, refcount, seqlens, info};
  for (int i = 1; i < 4; ++i)
    if (overlap(extent_of("", kv_pages), extent_of("", written[i])))
      return fail(DSV_ERR_INVALID, "kv_pages overlaps the bookkeeping");
  if ((rc = check_info(info, written, 4)) != DSV_OK) return rc;
  if (parents == nullptr || parents->ndim != 1) return fail(DSV_ERR_INVALID, "parents must be a 1-d tensor");
  a.n = parents->shape[0];
  if ((rc = check_index(parents, "parents", a.n, written, 5, a.parents)) != DSV_OK) return rc;
  if ((rc = check_index(children, "children", a.n, written, 5, a.children)) != DSV_OK) return rc;
  PagesPlan p;
  if (!pages_plan(a.book.P, a.book.B, a.n, p)) return fail(DSV_ERR_UNSUPPORTED, "more than %d pairs", dsv::kPageMaxSeqs);
  if ((rc = check_workspace(p.total, workspace, workspace_bytes)) != DSV_OK) return rc;
  char* w = static_cast<char*>(workspace);
  a.info = static_cast<int32_t*>(info->data);
  a.src = reinterpret_cast<int32_t*>(w);
  a.dst = a.src + a.n;
  a.state = reinterpret_cast<int32_t*>(w + p.list_bytes + p.off_bytes);
  if (g_dry_run) return DSV_OK;
  const hipError_t e = dsv::launch_fork(a, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "page fork launch");
  return DSV_OK;
}

int dsv_pages_extend(const dsv_tensor* page_table, const dsv_tensor* refcount, const dsv_tensor* seqlens,
                     const dsv_tensor* new_lens, int64_t page_size, dsv_tensor* info, void* workspace,
                     size_t workspace_bytes, void* stream) {
  int rc;
  dsv::ExtendArgs a{};
  if ((rc = check_nd(seqlens, "seqlens", 1)) != DSV_OK) return rc;
  if ((rc = check_book(page_table, refcount, seqlens, page_size, a.book)) != DSV_OK) return rc;
  const dsv_tensor* written[4] = {page_table, refcount, seqlens, info};
  if ((rc = check_info(info, written, 3)) != DSV_OK) return rc;
  if ((rc = check_index(new_lens, "new_lens", a.book.B, written, 4, a.newlens)) != DSV_OK) return rc;
  PagesPlan p;
  if (!pages_plan(a.book.P, a.book.B, 0, p)) return fail(DSV_ERR_UNSUPPORTED, "sizes out of range");
  if ((rc = check_workspace(p.total, workspace, workspace_bytes)) != DSV_OK) return rc;
  char* w = static_cast<char*>(workspace);
  a.info = static_cast<int32_t*>(info->data);
  a.list = reinterpret_cast<int32_t*>(w);
  a.off = reinterpret_cast<int64_t*>(w + p.list_bytes);
  if (g_dry_run) return DSV_OK;
  const hipError_t e = dsv::launch_extend(a, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "page extend launch");
  return DSV_OK;
}

int dsv_pages_free(const dsv_tensor* page_table, const dsv_tensor* refcount, const dsv_tensor* seqlens,
                   const dsv_tensor* seqs, int64_t page_size, int64_t window, int64_t sinks, void* stream) {
  int rc;
  dsv::FreeArgs a{};
  if ((rc = check_nd(seqlens, "seqlens", 1)) != DSV_OK) return rc;
  if ((rc = check_book(page_table, refcount, seqlens, page_size, a.book)) != DSV_OK) return rc;
  if (window < 0 || sinks < 0) return fail(DSV_ERR_INVALID, "window and sinks must be >= 0");
  if (window == 0 && sinks != 0) return fail(DSV_ERR_INVALID, "sinks without a window: every page is freed");
  const dsv_tensor* written[3] = {page_table, refcount, seqlens};
  if (seqs == nullptr || seqs->ndim != 1) return fail(DSV_ERR_INVALID, "seqs must be a 1-d tensor");
  a.n = seqs->shape[0];
  if (a.n > ((int64_t)1 << 22)) return fail(DSV_ERR_UNSUPPORTED, "more than 2^22 sequences named");
  if ((rc = check_index(seqs, "seqs", a.n, written, 3, a.seqs)) != DSV_OK) return rc;
  a.window = std::min<int64_t>(window, (int64_t)1 << 41);
  a.sinks = std::min<int64_t>(sinks, (int64_t)1 << 41);
  if (g_dry_run) return DSV_OK;
  const hipError_t e = dsv::launch_free(a, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "page free launch");
  return DSV_OK;
}

int dsv_pages_compact(const dsv_tensor* kv_pages, const dsv_tensor* page_table, const dsv_tensor* refcount,
                      dsv_tensor* info, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  dsv::CompactArgs a{};
  if (kv_pages == nullptr || kv_pages->ndim != 6) return fail(DSV_ERR_INVALID, "kv_pages must be [L, 2, P, Hk, page, D]");
  if ((rc = check_book(page_table, refcount, nullptr, kv_pages->shape[4], a.book)) != DSV_OK) return rc;
  if ((rc = check_page_data(kv_pages, a.book.P, a.data)) != DSV_OK) return rc;
  const dsv_tensor* written[3] = {kv_pages, page_table, refcount};
  for (int i = 1; i < 3; ++i)
    if (overlap(extent_of("", kv_pages), extent_of("", written[i])))
      return fail(DSV_ERR_INVALID, "kv_pages overlaps the bookkeeping");
  if ((rc = check_info(info, written, 3)) != DSV_OK) return rc;
  PagesPlan p;
  if (!pages_plan(a.book.P, a.book.B, 0, p)) return fail(DSV_ERR_UNSUPPORTED, "sizes out of range");
  if ((rc = check_workspace(p.total, workspace, workspace_bytes)) != DSV_OK) return rc;
  char* w = static_cast<char*>(workspace);
  a.info = static_cast<int32_t*>(info->data);
  a.to = reinterpret_cast<int32_t*>(w);
  a.src = a.to + a.book.P;
  a.dst = a.src + (a.book.P + 1) / 2;
  a.state = reinterpret_cast<int32_t*>(w + p.list_bytes + p.off_bytes);
  if (g_dry_run) return DSV_OK;
  const hipError_t e = dsv::launch_compact(a, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "page compact launch");
  return DSV_OK;
}

}  // extern "C"

// ---------------------------------------------------------------------------
// Windowed attention
// ---------------------------------------------------------------------------

namespace {

struct WinPlan {
  int G = 0, R = 0, MW = 0, rpb = 0, n_rb = 0, splits = 1;
  size_t opart_bytes = 0, ml_bytes = 0, total = 0;
  const char* err = nullptr;
};

bool win_args_ok(int64_t B, int64_t M, int64_t H, int64_t Hk, int64_t D, int dtype, int64_t n_keys, int64_t window,
                 int64_t sinks) {
  return B >= 1 && M >= 1 && H >= 1 && Hk >= 1 && H % Hk == 0 && (D == 64 || D == 128) && dtype >= DSV_BF16 &&
         dtype <= DSV_F32 && n_keys >= 0 && window >= 1 && sinks >= 0;
}

WinPlan win_plan(int64_t B, int64_t M, int64_t H, int64_t Hk, int64_t D, int dtype, int64_t n_keys, int64_t window,
                 int64_t sinks, bool tree, bool no_tile) {
  WinPlan p;
  const bool in_range = B <= (1 << 20) && M <= (1 << 24) && H <= (1 << 16) && n_keys <= dsv::kWinMaxKeys;
  const int64_t R = in_range ? (H / Hk) * M : 0;
  if (!in_range || R > ((int64_t)1 << 24) || B * Hk * R > ((int64_t)1 << 30)) {
    p.err = "sizes beyond the windowed attention's range (batch <= 2^20, heads <= 65536, keys <= 2^30, query heads / "
            "key heads x rows <= 2^24, batch x query heads x rows <= 2^30)";
    return p;
  }
  // (Beyond every key, either means all of them.)
  window = std::min(window, dsv::kWinMaxKeys);
  sinks = std::min(sinks, dsv::kWinMaxKeys);
  p.G = (int)(H / Hk);
  p.R = (int)R;
  p.MW = tree ? (int)((M + 63) / 64) : 0;
  // Blocks of 256 rows from 17 rows on (32 sequences of 24 rows through 4096 keys:
  // 108 us, in blocks of 16 113; of 64 rows 122 against 196), of 16
  // below (64 sequences of 16 rows: 198 us, 219 in blocks of 256) and in fp32.
  const bool tile = dtype != DSV_F32 && R > 16 && !no_tile;
  p.rpb = tile ? 256 : 16;
  p.n_rb = (int)((R + p.rpb - 1) / p.rpb);
  if (B * Hk * p.n_rb >= (1 << 23)) {
    // (512 threads each; a launch counts fewer than 2^32.)
    p.err = "batch x key heads x blocks of rows beyond 2^23 - 1";
    return p;
  }
  // Splits over the keys until there is a workgroup per CU, of 20 tiles at
  // least (8 waves, 2 to 3 tiles each): more splits cost more in the merge than
  // they gain (bf16, one sequence through 16384 keys: 16 splits 31 us, 32 splits
  // 36; 8 sequences of 16 rows through 4096: 2 splits 75, 4 splits 86).
  const int64_t units = B * Hk * p.n_rb;
  const int64_t span = tree ? M : std::min<int64_t>(M, p.rpb / p.G + 2);
  const int64_t reach = std::min(n_keys, window + span) / 32 + 2 + std::min(n_keys, sinks) / 32;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(device_cus() / units, reach / (tile ? 4 : 20)));
  const size_t rows = p.splits > 1 ? (size_t)B * Hk * p.splits * R : 0;
  p.opart_bytes = align_up(rows * D * sizeof(float), 256);
  p.ml_bytes = align_up(rows * sizeof(float2), 256);
  p.total = p.opart_bytes + p.ml_bytes;
  return p;
}

}  // namespace

extern "C" {

size_t dsv_window_workspace_bytes(int64_t B, int64_t M, int64_t H, int64_t Hk, int64_t D, int dtype, int64_t n_keys,
                                  int64_t window, int64_t sinks, int has_tree) {
  if (!win_args_ok(B, M, H, Hk, D, dtype, n_keys, window, sinks) || (has_tree && M > dsv::kTreeMaxM)) return 0;
  // (Whatever pages and strides the call comes with.)
  const WinPlan p = win_plan(B, M, H, Hk, D, dtype, n_keys, window, sinks, has_tree != 0, false);
  const WinPlan r = win_plan(B, M, H, Hk, D, dtype, n_keys, window, sinks, has_tree != 0, true);
  return p.err != nullptr ? 0 : std::max(p.total, r.total);
}

int dsv_window_attention(const dsv_tensor* q, const dsv_tensor* k, const dsv_tensor* v, const dsv_tensor* page_table,
                         const dsv_tensor* cache_seqlens, int64_t n_keys, int64_t window, int64_t sinks,
                         const dsv_tensor* parent, dsv_tensor* out, dsv_tensor* lse, void* workspace,
                         size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_q_out(q, out)) != DSV_OK) return rc;
  const int64_t B = q->shape[0], M = q->shape[1], H = q->shape[2], D = q->shape[3];
  if (B < 1 || M < 1 || H < 1) return fail(DSV_ERR_INVALID, "q must hold at least one query");
  if (window < 1) return fail(DSV_ERR_INVALID, "window must be at least 1 (got %lld)", (long long)window);
  if (sinks < 0) return fail(DSV_ERR_INVALID, "sinks must be >= 0");
  dsv::WinArgs a{};
  int64_t Hk = 0, cap = 0;
  if (present(page_table)) {
    if ((rc = check_nd(k, "k_pages", 4)) != DSV_OK) return rc;
    if ((rc = check_nd(v, "v_pages", 4)) != DSV_OK) return rc;
    if ((rc = check_vec16(k, "k_pages")) != DSV_OK) return rc;
    if ((rc = check_vec16(v, "v_pages")) != DSV_OK) return rc;
    for (int i = 0; i < 4; ++i)
      if (k->shape[i] != v->shape[i]) return fail(DSV_ERR_INVALID, "k_pages and v_pages shapes differ");
    if (k->dtype != q->dtype || v->dtype != q->dtype) return fail(DSV_ERR_INVALID, "q and pages must share a dtype");
    if (k->shape[3] != D) return fail(DSV_ERR_INVALID, "page head_dim differs from q");
    if (k->shape[0] < 1 || k->shape[0] > 0x7fffffff) return fail(DSV_ERR_INVALID, "the pool must hold 1 to 2^31 - 1 pages");
    const int sh = log2_exact(k->shape[2]);
    if (sh < 0) return fail(DSV_ERR_UNSUPPORTED, "page_size %lld must be a power of two", (long long)k->shape[2]);
    if ((rc = check_nd(page_table, "page_table", page_table->ndim)) != DSV_OK) return rc;
    if (page_table->ndim != 1 && page_table->ndim != 2) return fail(DSV_ERR_INVALID, "page_table must be 1-d or 2-d");
    if (page_table->dtype != DSV_I32 && page_table->dtype != DSV_I64)
      return fail(DSV_ERR_INVALID, "page_table must be int32 or int64");
    if (page_table->ndim == 2 && page_table->shape[0] != B && page_table->shape[0] != 1)
      return fail(DSV_ERR_INVALID, "page_table batch must be 1 or B");
    const int64_t npt = page_table->shape[page_table->ndim - 1];
    if (npt > 1 && page_table->stride[page_table->ndim - 1] != 1)
      return fail(DSV_ERR_INVALID, "page_table innermost stride must be 1");
    Hk = k->shape[1];
    a.k_sp = k->stride[0];
    a.k_sh = k->stride[1];
    a.k_st = k->stride[2];
    a.v_sp = v->stride[0];
    a.v_sh = v->stride[1];
    a.v_st = v->stride[2];
    a.pt = page_table->data;
    a.pt_i64 = page_table->dtype == DSV_I64;
    a.ps_shift = sh;
    a.pt_sb = (page_table->ndim == 2 && page_table->shape[0] > 1) ? page_table->stride[0] : 0;
    a.n_phys = k->shape[0];
    cap = npt > ((int64_t)1 << 40) >> sh ? (int64_t)1 << 40 : npt << sh;
  } else {
    if ((rc = check_kv_dense(k, v, q, "k_cache", "v_cache")) != DSV_OK) return rc;
    Hk = k->shape[2];
    a.k_sb = B > 1 ? k->stride[0] : 0;
    a.k_st = k->stride[1];
    a.k_sh = k->stride[2];
    a.v_sb = B > 1 ? v->stride[0] : 0;
    a.v_st = v->stride[1];
    a.v_sh = v->stride[2];
    cap = k->shape[1];
  }
  if (Hk < 1 || H % Hk != 0)
    return fail(DSV_ERR_INVALID, "query heads (%lld) must be a multiple of key heads (%lld)", (long long)H, (long long)Hk);
  const int64_t n = n_keys < 0 || n_keys > cap ? cap : n_keys;
  if (present(cache_seqlens)) {
    if ((rc = check_nd(cache_seqlens, "cache_seqlens", 1)) != DSV_OK) return rc;
    if ((cache_seqlens->dtype != DSV_I32 && cache_seqlens->dtype != DSV_I64) || cache_seqlens->shape[0] != B ||
        (B > 1 && cache_seqlens->stride[0] != 1))
      return fail(DSV_ERR_INVALID, "cache_seqlens must be a contiguous int32 or int64 [B] tensor");
    a.seqlens = cache_seqlens->data;
    a.seqlens_i64 = cache_seqlens->dtype == DSV_I64;
  }
  if (present(parent)) {
    if (parent->ndim != 1 && parent->ndim != 2) return fail(DSV_ERR_INVALID, "parent must be [M] or [B, M]");
    if ((rc = check_nd(parent, "parent", parent->ndim)) != DSV_OK) return rc;
    if (parent->dtype != DSV_I32 && parent->dtype != DSV_I64) return fail(DSV_ERR_INVALID, "parent must be int32 or int64");
    if (parent->shape[parent->ndim - 1] != M) return fail(DSV_ERR_INVALID, "parent must have M entries per tree");
    if (parent->ndim == 2 && parent->shape[0] != B && parent->shape[0] != 1)
      return fail(DSV_ERR_INVALID, "parent batch must be 1 or B");
    if (M > dsv::kTreeMaxM) return fail(DSV_ERR_UNSUPPORTED, "trees larger than %d nodes are not supported", dsv::kTreeMaxM);
    a.parent = parent->data;
    a.par_i64 = parent->dtype == DSV_I64;
    a.par_sb = (parent->ndim == 2 && parent->shape[0] > 1) ? parent->stride[0] : 0;
    a.par_sm = parent->stride[parent->ndim - 1];
  }
  if (present(lse)) {
    if ((rc = check_nd(lse, "lse", 3)) != DSV_OK) return rc;
    if (lse->dtype != DSV_F32 || lse->shape[0] != B || lse->shape[1] != H || lse->shape[2] != M)
      return fail(DSV_ERR_INVALID, "lse must be float32 [B, H, M]");
    a.lse = static_cast<float*>(lse->data);
    a.l_sb = lse->stride[0];
    a.l_sh = lse->stride[1];
    a.l_sm = lse->stride[2];
  }
  // Rows are written while others' inputs are still read.
  const Extent ins[6] = {extent_of("q", q), extent_of("k", k), extent_of("v", v), extent_of("page_table", page_table),
                         extent_of("cache_seqlens", cache_seqlens), extent_of("parent", parent)};
  for (const Extent& in : ins)
    if (overlap(extent_of("out", out), in) || overlap(extent_of("lse", lse), in))
      return fail(DSV_ERR_INVALID, "out or lse overlaps %s", in.name);
  if (overlap(extent_of("out", out), extent_of("lse", lse))) return fail(DSV_ERR_INVALID, "out overlaps lse");

  // (As win_plan takes them.)
  const int64_t W = std::min<int64_t>(window, dsv::kWinMaxKeys), S = std::min<int64_t>(sinks, dsv::kWinMaxKeys);
  // The kernel for many rows reads a DMA instruction's 4 or 8 keys through one
  // page, and a tile's 32 keys with 32-bit offsets from the first.
  const bool no_tile = (present(page_table) && k->shape[2] < 8) || a.k_st > (1 << 25) || a.v_st > (1 << 25);
  const WinPlan p = win_plan(B, M, H, Hk, D, q->dtype, n, W, S, a.parent != nullptr, no_tile);
  if (p.err != nullptr) return fail(DSV_ERR_UNSUPPORTED, "%s", p.err);
  if (p.total > 0 && (rc = check_workspace(p.total, workspace, workspace_bytes)) != DSV_OK) return rc;
  a.dtype = q->dtype;
  a.q = static_cast<const uint16_t*>(q->data);
  a.q_sb = q->stride[0];
  a.q_sm = q->stride[1];
  a.q_sh = q->stride[2];
  a.k = static_cast<const uint16_t*>(k->data);
  a.v = static_cast<const uint16_t*>(v->data);
  a.n_keys = n;
  a.B = (int)B;
  a.M = (int)M;
  a.H = (int)H;
  a.Hk = (int)Hk;
  a.G = p.G;
  a.R = p.R;
  a.W = (int)W;
  a.S = (int)S;
  a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)D));
  a.rows_per_block = p.rpb;
  a.n_rb = p.n_rb;
  a.splits = p.splits;
  if (p.total > 0) {
    char* w = static_cast<char*>(workspace);
    a.opart = reinterpret_cast<float*>(w);
    a.ml = reinterpret_cast<float2*>(w + p.opart_bytes);
  }
  a.MW = p.MW;
  a.out = out->data;
  a.out_dtype = out->dtype;
  a.o_sb = out->stride[0];
  a.o_sm = out->stride[1];
  a.o_sh = out->stride[2];
  const int per16 = 16 / elem_size(out->dtype);
  a.out_vec = (reinterpret_cast<uintptr_t>(out->data) & 15) == 0 && (B == 1 || a.o_sb % per16 == 0) &&
              (M == 1 || a.o_sm % per16 == 0) && (H == 1 || a.o_sh % per16 == 0);
  if (g_dry_run) {
    dsv::WinExtents ex;
    ex.q = ins[0], ex.k = ins[1], ex.v = ins[2], ex.pt = ins[3], ex.lens = ins[4], ex.parent = ins[5];
    ex.out = extent_of("out", out);
    ex.lse = extent_of("lse", lse);
    ex.ws = extent_raw("workspace", workspace, (int64_t)workspace_bytes);
    std::string err;
    int64_t checks = 0;
    const int bad = dsv::emulate_window(a, (int)D, ex, err, &checks);
    g_dry_checks = checks;
    return bad ? fail(DSV_ERR_INVALID, "dry run: %s", err.c_str()) : DSV_OK;
  }
  const hipError_t e = dsv::launch_window(a, (int)D, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "windowed attention launch");
  return DSV_OK;
}

}  // extern "C"

// ---------------------------------------------------------------------------
// Slot maps and the latent cache's append
// ---------------------------------------------------------------------------

namespace {

// An int32 or int64 array that the call writes: contiguous, of n entries.
int check_list(const dsv_tensor* t, const char* name, int dtype, int64_t n) {
  if (t == nullptr || t->ndim != 1 || t->shape[0] != 0) {
    const int rc = check_nd(t, name, 1);
    if (rc != DSV_OK) return rc;
  }
  if (t->dtype != dtype || t->shape[0] != n || (n > 1 && t->stride[0] != 1))
    return fail(DSV_ERR_INVALID, "%s must be contiguous %s [%lld]", name, dt_name(dtype), (long long)n);
  return DSV_OK;
}

// Outputs may share no byte with an input or with each other.
int check_apart(const Extent* outs, int n_outs, const Extent* ins, int n_ins) {
  for (int i = 0; i < n_outs; ++i) {
    for (int j = 0; j < n_ins; ++j)
      if (overlap(outs[i], ins[j])) return fail(DSV_ERR_INVALID, "%s overlaps %s", outs[i].name, ins[j].name);
    for (int j = i + 1; j < n_outs; ++j)
      if (overlap(outs[i], outs[j])) return fail(DSV_ERR_INVALID, "%s overlaps %s", outs[i].name, outs[j].name);
  }
  return DSV_OK;
}

}  // namespace

extern "C" {

int dsv_token_slots(const dsv_tensor* page_table, const dsv_tensor* seqlens, const dsv_tensor* new_lens,
                    const dsv_tensor* seqs, int64_t page_size, dsv_tensor* slots, dsv_tensor* positions,
                    dsv_tensor* requests, dsv_tensor* cu_seqlens, dsv_tensor* block_table, dsv_tensor* lens,
                    void* stream) {
  int rc;
  dsv::SlotArgs a{};
  if ((rc = check_nd(page_table, "page_table", 2)) != DSV_OK) return rc;
  if (page_table->dtype != DSV_I32 || (page_table->shape[1] > 1 && page_table->stride[1] != 1))
    return fail(DSV_ERR_INVALID, "page_table must be int32 [B, n_logical] with innermost stride 1");
  const int sh = log2_exact(page_size);
  if (sh < 0) return fail(DSV_ERR_UNSUPPORTED, "page_size %lld must be a power of two", (long long)page_size);
  a.table = static_cast<const int32_t*>(page_table->data);
  a.t_sb = page_table->stride[0];
  a.B = page_table->shape[0];
  a.n_log = page_table->shape[1];
  a.ps_shift = sh;
  if (a.B > dsv::kPageMaxSeqs) return fail(DSV_ERR_UNSUPPORTED, "more than %d sequences", dsv::kPageMaxSeqs);
  if (a.n_log > 0x7fffffff >> sh) return fail(DSV_ERR_UNSUPPORTED, "page_table rows beyond 2^31 - 1 tokens");
  if ((rc = check_nd(seqlens, "seqlens", 1)) != DSV_OK) return rc;
  if ((seqlens->dtype != DSV_I32 && seqlens->dtype != DSV_I64) || seqlens->shape[0] != a.B || (a.B > 1 && seqlens->stride[0] != 1))
    return fail(DSV_ERR_INVALID, "seqlens must be contiguous int32 or int64 [B]");
  a.lens = seqlens->data;
  a.lens_i64 = seqlens->dtype == DSV_I64;
  if (new_lens == nullptr || new_lens->ndim != 1) return fail(DSV_ERR_INVALID, "new_lens must be a 1-d tensor");
  const int64_t n = new_lens->shape[0];
  if (n > dsv::kPageMaxSeqs) return fail(DSV_ERR_UNSUPPORTED, "more than %d requests", dsv::kPageMaxSeqs);
  if ((rc = check_index(new_lens, "new_lens", n, nullptr, 0, a.news)) != DSV_OK) return rc;
  if (present(seqs)) {
    if ((rc = check_index(seqs, "seqs", n, nullptr, 0, a.seqs)) != DSV_OK) return rc;
  } else if (n != a.B) {
    return fail(DSV_ERR_INVALID, "new_lens must have an entry per sequence (%lld) where no seqs are given", (long long)a.B);
  }
  a.n = (int)n;
  if (slots == nullptr || slots->ndim != 1) return fail(DSV_ERR_INVALID, "slots must be a 1-d tensor");
  a.cap = slots->shape[0];
  if (a.cap > ((int64_t)1 << 30)) return fail(DSV_ERR_UNSUPPORTED, "a capacity of more than 2^30 tokens");
  if ((rc = check_list(slots, "slots", DSV_I64, a.cap)) != DSV_OK) return rc;
  if ((rc = check_list(positions, "positions", DSV_I32, a.cap)) != DSV_OK) return rc;
  if ((rc = check_list(requests, "requests", DSV_I32, a.cap)) != DSV_OK) return rc;
  if ((rc = check_list(cu_seqlens, "cu_seqlens", DSV_I32, n + 1)) != DSV_OK) return rc;
  if ((rc = check_list(lens, "lens", DSV_I32, n)) != DSV_OK) return rc;
  if (block_table == nullptr || block_table->ndim != 2 || block_table->dtype != DSV_I32 || block_table->shape[0] != n ||
      block_table->shape[1] != a.n_log || (a.n_log > 1 && block_table->stride[1] != 1) ||
      (n > 1 && block_table->stride[0] < a.n_log))
    return fail(DSV_ERR_INVALID, "block_table must be int32 [n, n_logical] with innermost stride 1");
  if (n > 0 && a.n_log > 0 && (rc = check_nd(block_table, "block_table", 2)) != DSV_OK) return rc;
  const Extent outs[6] = {extent_of("slots", slots), extent_of("positions", positions), extent_of("requests", requests),
                          extent_of("cu_seqlens", cu_seqlens), extent_of("block_table", block_table), extent_of("lens", lens)};
  const Extent ins[4] = {extent_of("page_table", page_table), extent_of("seqlens", seqlens), extent_of("new_lens", new_lens),
                         extent_of("seqs", seqs)};
  if ((rc = check_apart(outs, 6, ins, 4)) != DSV_OK) return rc;
  a.slots = static_cast<int64_t*>(slots->data);
  a.pos = static_cast<int32_t*>(positions->data);
  a.req = static_cast<int32_t*>(requests->data);
  a.cu = static_cast<int32_t*>(cu_seqlens->data);
  a.block = static_cast<int32_t*>(block_table->data);
  a.b_sb = block_table->stride[0];
  a.out_lens = static_cast<int32_t*>(lens->data);
  if (g_dry_run) return DSV_OK;
  const hipError_t e = dsv::launch_slots(a, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "slot map launch");
  return DSV_OK;
}

int dsv_latent_append(const dsv_tensor* c, const dsv_tensor* k_pe, const dsv_tensor* norm_weight, float eps,
                      const dsv_tensor* cos, const dsv_tensor* sin, const dsv_tensor* positions, int interleaved,
                      const dsv_tensor* slots, const dsv_tensor* cache, const dsv_tensor* q_pe, dsv_tensor* q_out,
                      void* stream) {
  int rc;
  dsv::LatentAppendArgs a{};
  if ((rc = check_nd(cache, "cache", cache != nullptr && cache->ndim == 2 ? 2 : 3)) != DSV_OK) return rc;
  if ((rc = check_vec16(cache, "cache")) != DSV_OK) return rc;
  // (No tokens, as a list of capacity 0 has them: their tensors may come without storage.)
  if (c != nullptr && c->ndim == 2 && c->shape[0] == 0) {
    if (k_pe == nullptr || k_pe->ndim != 2 || k_pe->shape[0] != 0 || c->shape[1] + k_pe->shape[1] != cache->shape[cache->ndim - 1] ||
        slots == nullptr || slots->ndim != 1 || slots->shape[0] != 0)
      return fail(DSV_ERR_INVALID, "c and k_pe must be [T, dc] and [T, dr], dc + dr as wide as cache's rows, and slots [T]");
    return DSV_OK;
  }
  auto rows = [&](const dsv_tensor* t, const char* name, int nd) -> int {
    int r;
    if (t == nullptr || t->ndim != nd) return fail(DSV_ERR_INVALID, "%s must be a %d-d tensor", name, nd);
    for (int i = 0; i < nd; ++i)
      if (t->shape[i] == 0) return fail(DSV_ERR_INVALID, "%s is empty", name);
    if ((r = check_nd(t, name, nd)) != DSV_OK) return r;
    if ((r = check_vec16(t, name)) != DSV_OK) return r;
    if (t->dtype != cache->dtype) return fail(DSV_ERR_INVALID, "%s must have the cache's dtype", name);
    return DSV_OK;
  };
  if ((rc = rows(c, "c", 2)) != DSV_OK) return rc;
  if ((rc = rows(k_pe, "k_pe", 2)) != DSV_OK) return rc;
  const int64_t T = c->shape[0], dc = c->shape[1], dr = k_pe->shape[1];
  const int es = elem_size(cache->dtype), nd = cache->ndim;
  if (k_pe->shape[0] != T) return fail(DSV_ERR_INVALID, "c and k_pe must have the same tokens");
  if ((dc * es) % 16 != 0 || (dr * es) % 32 != 0)
    return fail(DSV_ERR_UNSUPPORTED, "rows of %lld + %lld entries (the latent part a multiple of 16 bytes, the rotated part of 32)",
                (long long)dc, (long long)dr);
  if (dc > 2048 || dr > 2048) return fail(DSV_ERR_UNSUPPORTED, "rows wider than 2048 + 2048 entries");
  if (cache->shape[nd - 1] != dc + dr)
    return fail(DSV_ERR_INVALID, "cache rows hold %lld entries, c and k_pe %lld", (long long)cache->shape[nd - 1], (long long)(dc + dr));
  a.dtype = cache->dtype;
  a.T = T;
  a.dc = (int)dc;
  a.dr = (int)dr;
  a.c = c->data;
  a.c_st = c->stride[0];
  a.pe = k_pe->data;
  a.pe_st = k_pe->stride[0];
  a.eps = eps;
  if (present(norm_weight)) {
    if ((rc = rows(norm_weight, "norm_weight", 1)) != DSV_OK) return rc;
    if (norm_weight->shape[0] != dc) return fail(DSV_ERR_INVALID, "norm_weight must be [%lld]", (long long)dc);
    if (!(eps >= 0.f) || !(eps < 3.4e38f)) return fail(DSV_ERR_INVALID, "eps must be finite and >= 0");
    a.w = norm_weight->data;
  }
  if (present(cos) != present(sin)) return fail(DSV_ERR_INVALID, "cos and sin go together");
  if (present(cos)) {
    for (const dsv_tensor* t : {cos, sin}) {
      const char* nm = t == cos ? "cos" : "sin";
      if ((rc = check_nd(t, nm, 2)) != DSV_OK) return rc;
      if ((rc = check_vec16(t, nm)) != DSV_OK) return rc;
      if (t->shape[1] != dr || t->shape[0] < 1 || t->shape[0] != cos->shape[0])
        return fail(DSV_ERR_INVALID, "cos and sin must be [n_pos, %lld]", (long long)dr);
      if (t->dtype != cos->dtype || (t->dtype != DSV_F32 && t->dtype != a.dtype))
        return fail(DSV_ERR_INVALID, "cos and sin must both be float32 or of the cache's dtype");
    }
    a.cos = cos->data;
    a.sin = sin->data;
    a.cos_st = cos->stride[0];
    a.sin_st = sin->stride[0];
    a.tab_f32 = cos->dtype == DSV_F32;
    a.n_pos = cos->shape[0];
    if (present(positions)) {
      dsv::PageIndex x{};
      if ((rc = check_index(positions, "positions", T, nullptr, 0, x)) != DSV_OK) return rc;
      if (T > 1 && x.stride != 1) return fail(DSV_ERR_INVALID, "positions must be contiguous");
      a.pos = x.p;
      a.pos_i64 = x.is64;
    } else if (a.n_pos != T) {
      return fail(DSV_ERR_INVALID, "cos and sin must have a row per token where no positions are given");
    }
  } else if (present(positions)) {
    return fail(DSV_ERR_INVALID, "positions without cos and sin");
  }
  a.interleaved = interleaved != 0;
  {
    dsv::PageIndex x{};
    if ((rc = check_index(slots, "slots", T, nullptr, 0, x)) != DSV_OK) return rc;
    if (T > 1 && x.stride != 1) return fail(DSV_ERR_INVALID, "slots must be contiguous");
    a.slots = x.p;
    a.slots_i64 = x.is64;
  }
  a.cache = cache->data;
  a.s_t = cache->stride[nd - 2];
  // Rows that share bytes would be written into each other.
  if (cache->shape[nd - 2] > 1 && a.s_t < dc + dr) return fail(DSV_ERR_INVALID, "cache rows overlap");
  if (nd == 3) {
    const int sh = log2_exact(cache->shape[1]);
    if (sh < 0) return fail(DSV_ERR_UNSUPPORTED, "page_size %lld must be a power of two", (long long)cache->shape[1]);
    if (cache->shape[0] > 0x7fffffff) return fail(DSV_ERR_UNSUPPORTED, "more than 2^31 - 1 pages");
    a.s_p = cache->stride[0];
    if (cache->shape[0] > 1 && a.s_p < (cache->shape[1] - 1) * a.s_t + dc + dr) return fail(DSV_ERR_INVALID, "cache pages overlap");
    a.ps_shift = sh;
    a.n_slots = cache->shape[0] << sh;
  } else {
    a.ps_shift = 62;
    a.n_slots = cache->shape[0];
  }
  if (present(q_pe) != present(q_out)) return fail(DSV_ERR_INVALID, "q_pe and q_out go together");
  bool in_place = false;
  if (present(q_pe)) {
    if ((rc = rows(q_pe, "q_pe", 3)) != DSV_OK) return rc;
    if ((rc = rows(q_out, "q_out", 3)) != DSV_OK) return rc;
    for (int i = 0; i < 3; ++i)
      if (q_out->shape[i] != q_pe->shape[i]) return fail(DSV_ERR_INVALID, "q_out must have q_pe's shape");
    if (q_pe->shape[0] != T || q_pe->shape[2] != dr) return fail(DSV_ERR_INVALID, "q_pe must be [%lld, H, %lld]", (long long)T, (long long)dr);
    if (q_pe->shape[1] > (1 << 16)) return fail(DSV_ERR_UNSUPPORTED, "more than 65536 heads");
    a.H = (int)q_pe->shape[1];
    a.q = q_pe->data;
    a.q_st = q_pe->stride[0];
    a.q_sh = q_pe->stride[1];
    a.qo = q_out->data;
    a.qo_st = q_out->stride[0];
    a.qo_sh = q_out->stride[1];
    // Rows of the output apart from each other: heads within tokens or tokens within heads.
    const int64_t H = a.H, st = T > 1 ? a.qo_st : -1, sh = H > 1 ? a.qo_sh : -1;
    const bool ok = (st < 0 || st >= dr) && (sh < 0 || sh >= dr) && (st < 0 || sh < 0 || st >= (H - 1) * sh + dr || sh >= (T - 1) * st + dr);
    if (!ok) return fail(DSV_ERR_INVALID, "q_out rows overlap");
    // A thread reads what it writes: row for row in place is safe.
    in_place = a.qo == a.q && a.qo_st == a.q_st && a.qo_sh == a.q_sh;
  }
  // (64 threads a token and one a pair: a launch counts fewer than 2^32.)
  if (T > ((int64_t)1 << 24) || T * (1 + a.H) * (dr * es / 32) > ((int64_t)1 << 31))
    return fail(DSV_ERR_UNSUPPORTED, "more than 2^24 tokens or 2^31 chunk pairs of rotated rows");
  const Extent outs[2] = {extent_of("cache", cache), extent_of("q_out", q_out)};
  const Extent ins[8] = {extent_of("c", c), extent_of("k_pe", k_pe), extent_of("norm_weight", norm_weight), extent_of("cos", cos),
                         extent_of("sin", sin), extent_of("positions", positions), extent_of("slots", slots),
                         in_place ? Extent{"q_pe", 0, 0} : extent_of("q_pe", q_pe)};
  if ((rc = check_apart(outs, 2, ins, 8)) != DSV_OK) return rc;
  if (g_dry_run) return DSV_OK;
  const hipError_t e = dsv::launch_latent_append(a, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "latent append launch");
  return DSV_OK;
}

}  // extern "C"

// ---------------------------------------------------------------------------
// Latent attention
// ---------------------------------------------------------------------------

namespace {

struct LatPlan {
  int G = 0, R = 0, MW = 0, rpb = 0, n_rb = 0, W = 1, sh = 0;
  size_t opart_bytes = 0, ml_bytes = 0, total = 0;
  const char* err = nullptr;
};

// Ranges of the expanded form's tile kernel, whose lines differ where causal (a block of
// rows sees the keys before its end): one, or as many as fill the CUs one to four times,
// whichever an estimate puts first.  In us, as measured: 1.03 a tile, 6 a piece, 2 a
// partial; lines much alike run in turns, others in the load of a CU and what its last
// range adds; joining 5 and the partials' bytes.  Against the most even use of the last
// turn alone (heads of 128 + 64): a prompt of 1500 tokens, 32 heads 94 -> 56 us, of 6000, 16
// heads 232 -> 197, of 3000, 32 heads 158 -> 142.  The constants are those of 128 + 64; narrower
// heads, whose tiles take less, were not measured by themselves and follow the same rule.
int expanded_ranges(const LatPlan& p, int64_t B, int64_t M, int64_t Hk, int64_t n_keys, bool causal) {
  const int64_t cus = device_cus(), units = Hk * p.n_rb;
  constexpr int kSamples = 32;
  const int n = std::min(p.n_rb, kSamples);
  int64_t line[kSamples];
  for (int i = 0; i < n; ++i) {
    const int64_t rb = ((int64_t)(i + 1) * p.n_rb - 1) / n, last = std::min<int64_t>((rb + 1) * p.rpb, M);
    const int64_t keys = causal ? std::max<int64_t>(0, n_keys - M + last) : n_keys;
    line[i] = B * std::max<int64_t>(1, (keys + (1 << p.sh) - 1) >> p.sh);
  }
  const bool even = line[0] > line[n - 1] * 4 / 5;
  int64_t best_w = 1;
  double best = 0;
  for (int64_t k = 0; k <= 4; ++k) {
    const int64_t w = k == 0 ? 1 : std::min(cus * k / units, line[n - 1] / 2);
    if (w < 1) continue;
    const double pieces = (double)(B + w - 1) / w, each = pieces * 6 + (w > 1 ? 2 : 0);
    double sum = 0;
    for (int i = 0; i < n; ++i) sum += (double)((line[i] - 1) / w + 1) * 1.03 + each;
    const double most = (double)((line[n - 1] - 1) / w + 1) * 1.03 + each, mean = sum / n, turns = (double)(units * w) / cus;
    double t = turns <= 1 ? most : (even ? std::ceil(turns) * most : std::max(most, (turns + 0.4) * mean));
    if (w > 1) t += 5 + (double)(units * w * p.rpb) * 900 / 4e6;
    if (k > 0 && t >= 0.95 * best) continue;
    best = t;
    best_w = w;
  }
  return (int)best_w;
}

LatPlan lat_plan(int64_t B, int64_t M, int64_t H, int64_t Hk, int64_t dv, int dtype, int64_t n_keys, bool tree, bool causal) {
  LatPlan p;
  const bool in_range = B <= (1 << 20) && M <= (1 << 24) && H <= (1 << 16) && n_keys <= dsv::kLatMaxKeys;
  const int64_t R = in_range ? (H / Hk) * M : 0;
  if (!in_range || R > ((int64_t)1 << 24) || B * Hk * R > ((int64_t)1 << 30)) {
    p.err = "sizes beyond the latent attention's range (batch <= 2^20, heads <= 65536, keys <= 2^30, rows per key head "
            "<= 2^24, batch x heads x rows <= 2^30)";
    return p;
  }
  const bool expanded = dv <= 128;
  p.G = (int)(H / Hk);
  p.R = (int)R;
  p.MW = tree ? (int)((M + 63) / 64) : 0;
  if (dtype == DSV_F32) {
    p.rpb = 16;
    p.sh = dsv::kLatTileF32;
  } else if (expanded) {
    p.rpb = 256;
    p.sh = dsv::kLatTileExp;
  } else {
    p.sh = dsv::kLatTile;
    // Blocks of 64 rows where two tiles of them and more fall to a CU (8 trees of 64 nodes, 32
    // heads: 214 us; blocks of 32 rows 360, of 16 603); of fewer rows, whose tiles and
    // partials take less time, where there is less (one token, 128 heads, 2900 keys: 15.0
    // us; blocks of 32 rows 17.2, of 64 19.9).
    const int64_t line = B * std::max<int64_t>(1, (n_keys + 63) >> 6), enough = 2 * (int64_t)device_cus();
    p.rpb = R > 32 && (R + 63) / 64 * line >= enough ? 64 : (R > 16 && (R + 31) / 32 * line >= enough ? 32 : 16);
    // The trees' sets of a block of 64 rows have room for 576 words.
    if (p.rpb == 64 && std::min<int64_t>(64, 63 / p.G + 2) * p.MW > 576) p.rpb = 32;
  }
  p.n_rb = (int)((R + p.rpb - 1) / p.rpb);
  const int64_t units = Hk * p.n_rb;
  if (units >= (1 << 23)) {
    // (512 threads each; a launch counts fewer than 2^32.)
    p.err = "key heads x blocks of rows beyond 2^23 - 1";
    return p;
  }
  const int64_t tiles = B * std::max<int64_t>(1, (n_keys + (1 << p.sh) - 1) >> p.sh);
  if (tiles >= ((int64_t)1 << 31)) {
    p.err = "batch x keys beyond 2^31 tiles of 32 or 64 keys";
    return p;
  }
  const int64_t cus = device_cus();
  if (units >= 4 * cus) {
    // (The units fill the CUs by themselves.)
  } else if (expanded && dtype != DSV_F32) {
    p.W = expanded_ranges(p, B, M, Hk, n_keys, causal);
  } else {
    // Ranges: as many workgroups as fill the CUs one to four times, whichever leaves
    // fewest idle in the last turn, of two tiles at least.  Against one turn: 2 chunks of 80
    // tokens, 128 heads, 8192 keys (160 blocks) 529 -> 421 us, 2 of 150, 64 heads, 4000 keys
    // 274 -> 227.  With one tile at least and with four, the join included: 128 heads, 2900
    // keys 19.8 us, 20.1 and 23.3; 16 heads, 8000 keys 20.9, 21.3 and 23.2; 8 sequences of 2000
    // 19.7, 20.0 and 22.8 (the other way: 1000 keys 17.0, with one 15.2; 32768 29.3, with four 26.9).
    double best = 0;
    for (int64_t k = 1; k <= 4; ++k) {
      const int64_t w = cus * k / units;
      const double use = (double)(units * w) / (double)(cus * k);
      if (w >= 1 && use > best + 0.04) {
        best = use;
        p.W = (int)w;
      }
    }
    p.W = (int)std::max<int64_t>(1, std::min<int64_t>(p.W, tiles / 2));
  }
  const size_t rows = p.W > 1 ? (size_t)units * p.W * 2 * p.rpb : 0;
  p.opart_bytes = align_up(rows * dv * sizeof(float), 256);
  p.ml_bytes = align_up(rows * sizeof(float2), 256);
  p.total = p.opart_bytes + p.ml_bytes;
  return p;
}

// The lengths, the tree, the outputs and the plan of both forms; then the launch.
int lat_common(dsv::LatArgs& a, const dsv_tensor* q, const dsv_tensor* seqlens, int64_t n, const dsv_tensor* parent, double scale,
               dsv_tensor* out, dsv_tensor* lse, const Extent* ins, int n_ins, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  const int64_t B = q->shape[0], M = q->shape[1], H = q->shape[2];
  if (!(scale > 0) || !(scale < 3.4e38)) return fail(DSV_ERR_INVALID, "the softmax scale must be finite and > 0");
  if ((rc = check_nd(out, "out", 4)) != DSV_OK) return rc;
  if (out->shape[0] != B || out->shape[1] != M || out->shape[2] != H || out->shape[3] != a.dv)
    return fail(DSV_ERR_INVALID, "out must be [B, M, H, %d]", a.dv);
  if (out->dtype != DSV_BF16 && out->dtype != DSV_F16 && out->dtype != DSV_F32)
    return fail(DSV_ERR_INVALID, "out dtype must be bf16, f16 or f32");
  if (out->stride[3] != 1) return fail(DSV_ERR_INVALID, "out innermost stride must be 1");
  if (present(seqlens)) {
    if ((rc = check_nd(seqlens, "cache_seqlens", 1)) != DSV_OK) return rc;
    if ((seqlens->dtype != DSV_I32 && seqlens->dtype != DSV_I64) || seqlens->shape[0] != B || (B > 1 && seqlens->stride[0] != 1))
      return fail(DSV_ERR_INVALID, "cache_seqlens must be a contiguous int32 or int64 [B] tensor");
    a.seqlens = seqlens->data;
    a.seqlens_i64 = seqlens->dtype == DSV_I64;
  }
  if (present(parent)) {
    if (parent->ndim != 1 && parent->ndim != 2) return fail(DSV_ERR_INVALID, "parent must be [M] or [B, M]");
    if ((rc = check_nd(parent, "parent", parent->ndim)) != DSV_OK) return rc;
    if (parent->dtype != DSV_I32 && parent->dtype != DSV_I64) return fail(DSV_ERR_INVALID, "parent must be int32 or int64");
    if (parent->shape[parent->ndim - 1] != M) return fail(DSV_ERR_INVALID, "parent must have M entries per tree");
    if (parent->ndim == 2 && parent->shape[0] != B && parent->shape[0] != 1)
      return fail(DSV_ERR_INVALID, "parent batch must be 1 or B");
    if (M > dsv::kTreeMaxM) return fail(DSV_ERR_UNSUPPORTED, "trees larger than %d nodes are not supported", dsv::kTreeMaxM);
    a.parent = parent->data;
    a.par_i64 = parent->dtype == DSV_I64;
    a.par_sb = (parent->ndim == 2 && parent->shape[0] > 1) ? parent->stride[0] : 0;
    a.par_sm = parent->stride[parent->ndim - 1];
  }
  if (present(lse)) {
    if ((rc = check_nd(lse, "lse", 3)) != DSV_OK) return rc;
    if (lse->dtype != DSV_F32 || lse->shape[0] != B || lse->shape[1] != H || lse->shape[2] != M)
      return fail(DSV_ERR_INVALID, "lse must be float32 [B, H, M]");
    a.lse = static_cast<float*>(lse->data);
    a.l_sb = lse->stride[0];
    a.l_sh = lse->stride[1];
    a.l_sm = lse->stride[2];
  }
  // Rows are written while others' inputs are still read.
  const Extent outs[2] = {extent_of("out", out), extent_of("lse", lse)};
  if ((rc = check_apart(outs, 2, ins, n_ins)) != DSV_OK) return rc;
  const LatPlan p = lat_plan(B, M, H, a.Hk, a.dv, a.dtype, n, a.parent != nullptr, a.causal != 0);
  if (p.err != nullptr) return fail(DSV_ERR_UNSUPPORTED, "%s", p.err);
  if (p.total > 0 && (rc = check_workspace(p.total, workspace, workspace_bytes)) != DSV_OK) return rc;
  const bool expanded = a.dv <= 128;
  a.q = q->data;
  a.q_sb = q->stride[0];
  a.q_sm = q->stride[1];
  a.q_sh = q->stride[2];
  a.n_keys = n;
  a.B = (int)B;
  a.M = (int)M;
  a.H = (int)H;
  a.G = p.G;
  a.R = p.R;
  a.MW = p.MW;
  a.rpb = p.rpb;
  a.n_rb = p.n_rb;
  a.W = p.W;
  a.scale_log2 = (float)(1.4426950408889634 * scale);
  if (!(a.scale_log2 > 0.f)) return fail(DSV_ERR_INVALID, "the softmax scale is too small for float32");
  if (p.total > 0) {
    char* w = static_cast<char*>(workspace);
    a.opart = reinterpret_cast<float*>(w);
    a.ml = reinterpret_cast<float2*>(w + p.opart_bytes);
  }
  a.out = out->data;
  a.out_dtype = out->dtype;
  a.o_sb = out->stride[0];
  a.o_sm = out->stride[1];
  a.o_sh = out->stride[2];
  const int per16 = 16 / elem_size(out->dtype);
  a.out_vec = (reinterpret_cast<uintptr_t>(out->data) & 15) == 0 && (B == 1 || a.o_sb % per16 == 0) &&
              (M == 1 || a.o_sm % per16 == 0) && (H == 1 || a.o_sh % per16 == 0);
  if (g_dry_run) return DSV_OK;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t e = a.dtype == DSV_F32 ? dsv::launch_latent_f32(a, s)
                 : expanded                ? dsv::launch_latent_tile(a, s)
                                                            : dsv::launch_latent(a, s);
  if (e == hipSuccess) e = dsv::launch_latent_merge(a, p.sh, s);
  if (e != hipSuccess) return hip_fail(e, "latent attention launch");
  return DSV_OK;
}

int lat_query(const dsv_tensor* q) {
  int rc;
  if ((rc = check_nd(q, "q", 4)) != DSV_OK) return rc;
  if ((rc = check_vec16(q, "q")) != DSV_OK) return rc;
  if (q->shape[0] < 1 || q->shape[1] < 1 || q->shape[2] < 1) return fail(DSV_ERR_INVALID, "q must hold at least one query");
  return DSV_OK;
}

}  // namespace

extern "C" {

size_t dsv_latent_workspace_bytes(int64_t B, int64_t M, int64_t H, int64_t v_dim, int dtype, int64_t n_keys, int has_tree,
                                  int expanded) {
  if (B < 1 || M < 1 || H < 1 || v_dim < 1 || dtype < DSV_BF16 || dtype > DSV_F32 || n_keys < 0 ||
      (has_tree && M > dsv::kTreeMaxM) || !(expanded ? dsv::expanded_widths((int)std::min<int64_t>(v_dim, 4096), 64)
                                                     : dsv::latent_widths((int)std::min<int64_t>(v_dim, 4096), 64)))
    return 0;
  // (Expanded, the plan depends on the mask, which a caller may choose later.)
  const LatPlan p = lat_plan(B, M, H, expanded ? H : 1, v_dim, dtype, n_keys, has_tree != 0, true);
  const LatPlan whole = expanded ? lat_plan(B, M, H, H, v_dim, dtype, n_keys, false, false) : p;
  return p.err != nullptr ? 0 : std::max(p.total, whole.total);
}

int dsv_latent_attention(const dsv_tensor* q, const dsv_tensor* kv, int64_t v_dim, const dsv_tensor* page_table,
                         const dsv_tensor* cache_seqlens, int64_t n_keys, double softmax_scale, const dsv_tensor* parent,
                         dsv_tensor* out, dsv_tensor* lse, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = lat_query(q)) != DSV_OK) return rc;
  if ((rc = check_nd(kv, "kv_cache", 3)) != DSV_OK) return rc;
  if ((rc = check_vec16(kv, "kv_cache")) != DSV_OK) return rc;
  const int64_t B = q->shape[0], D = q->shape[3];
  if (kv->dtype != q->dtype) return fail(DSV_ERR_INVALID, "q and kv_cache must share a dtype");
  if (kv->shape[2] != D) return fail(DSV_ERR_INVALID, "kv_cache rows hold %lld entries, q's %lld", (long long)kv->shape[2], (long long)D);
  if (v_dim < 1 || v_dim > D) return fail(DSV_ERR_INVALID, "v_dim must be in [1, %lld]", (long long)D);
  if (D > 4096 || !dsv::latent_widths((int)v_dim, (int)(D - v_dim)))
    return fail(DSV_ERR_UNSUPPORTED, "rows of %lld + %lld entries are not supported (256 or 512, and 32 or 64)", (long long)v_dim,
                (long long)(D - v_dim));
  dsv::LatArgs a{};
  int64_t cap = 0;
  dsv::LatSrc src{};
  src.p = kv->data;
  src.st = kv->stride[1];
  if (present(page_table)) {
    if (kv->shape[0] < 1 || kv->shape[0] > 0x7fffffff) return fail(DSV_ERR_INVALID, "the pool must hold 1 to 2^31 - 1 pages");
    const int sh = log2_exact(kv->shape[1]);
    if (sh < 0) return fail(DSV_ERR_UNSUPPORTED, "page_size %lld must be a power of two", (long long)kv->shape[1]);
    if (page_table->ndim != 1 && page_table->ndim != 2) return fail(DSV_ERR_INVALID, "page_table must be 1-d or 2-d");
    if ((rc = check_nd(page_table, "page_table", page_table->ndim)) != DSV_OK) return rc;
    if (page_table->dtype != DSV_I32 && page_table->dtype != DSV_I64)
      return fail(DSV_ERR_INVALID, "page_table must be int32 or int64");
    if (page_table->ndim == 2 && page_table->shape[0] != B && page_table->shape[0] != 1)
      return fail(DSV_ERR_INVALID, "page_table batch must be 1 or B");
    const int64_t npt = page_table->shape[page_table->ndim - 1];
    if (npt > 1 && page_table->stride[page_table->ndim - 1] != 1)
      return fail(DSV_ERR_INVALID, "page_table innermost stride must be 1");
    src.sp = kv->stride[0];
    a.pt = page_table->data;
    a.pt_i64 = page_table->dtype == DSV_I64;
    a.ps_shift = std::min(sh, 30);  // (keys are below 2^30)
    a.pt_sb = (page_table->ndim == 2 && page_table->shape[0] > 1) ? page_table->stride[0] : 0;
    a.n_phys = kv->shape[0];
    cap = npt > ((int64_t)1 << 40) >> sh ? (int64_t)1 << 40 : npt << sh;
  } else {
    if (kv->shape[0] != B) return fail(DSV_ERR_INVALID, "kv_cache batch differs from q");
    src.sb = B > 1 ? kv->stride[0] : 0;
    cap = kv->shape[1];
  }
  const int64_t n = n_keys < 0 || n_keys > cap ? cap : n_keys;
  a.dtype = q->dtype;
  a.dn = (int)v_dim;
  a.dr = (int)(D - v_dim);
  a.dv = (int)v_dim;
  a.kn = a.kr = a.v = src;
  a.kr.p = static_cast<const char*>(kv->data) + v_dim * elem_size(kv->dtype);
  a.Hk = 1;
  a.causal = 1;
  const Extent ins[5] = {extent_of("q", q), extent_of("kv_cache", kv), extent_of("page_table", page_table),
                         extent_of("cache_seqlens", cache_seqlens), extent_of("parent", parent)};
  return lat_common(a, q, cache_seqlens, n, parent, softmax_scale, out, lse, ins, 5, workspace, workspace_bytes, stream);
}

int dsv_latent_expanded(const dsv_tensor* q, const dsv_tensor* k, const dsv_tensor* k_pe, const dsv_tensor* v,
                        const dsv_tensor* cache_seqlens, int64_t n_keys, int causal, double softmax_scale, dsv_tensor* out,
                        dsv_tensor* lse, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = lat_query(q)) != DSV_OK) return rc;
  const int64_t B = q->shape[0], H = q->shape[2], D = q->shape[3];
  struct In { const dsv_tensor* t; const char* name; int nd; };
  for (const In& x : {In{k, "k", 4}, In{k_pe, "k_pe", 3}, In{v, "v", 4}}) {
    if ((rc = check_nd(x.t, x.name, x.nd)) != DSV_OK) return rc;
    if ((rc = check_vec16(x.t, x.name)) != DSV_OK) return rc;
    if (x.t->dtype != q->dtype) return fail(DSV_ERR_INVALID, "q and %s must share a dtype", x.name);
    if (x.t->shape[0] != B) return fail(DSV_ERR_INVALID, "%s batch differs from q", x.name);
    if (x.t->shape[1] != k->shape[1]) return fail(DSV_ERR_INVALID, "k, k_pe and v must hold the same tokens");
    if (x.nd == 4 && x.t->shape[2] != H) return fail(DSV_ERR_INVALID, "%s must have q's heads", x.name);
  }
  const int64_t dn = k->shape[3], dr = k_pe->shape[2];
  if (dn + dr != D) return fail(DSV_ERR_INVALID, "q rows hold %lld entries, k and k_pe %lld", (long long)D, (long long)(dn + dr));
  if (v->shape[3] != dn || dn > 4096 || dr > 4096 || !dsv::expanded_widths((int)dn, (int)dr))
    return fail(DSV_ERR_UNSUPPORTED, "heads of %lld + %lld entries and values of %lld are not supported (64 or 128 and 32 or 64, "
                "values as wide as the first part)", (long long)dn, (long long)dr, (long long)v->shape[3]);
  dsv::LatArgs a{};
  a.dtype = q->dtype;
  a.dn = a.dv = (int)dn;
  a.dr = (int)dr;
  a.kn = dsv::LatSrc{k->data, B > 1 ? k->stride[0] : 0, 0, k->stride[2], k->stride[1]};
  a.kr = dsv::LatSrc{k_pe->data, B > 1 ? k_pe->stride[0] : 0, 0, 0, k_pe->stride[1]};
  a.v = dsv::LatSrc{v->data, B > 1 ? v->stride[0] : 0, 0, v->stride[2], v->stride[1]};
  a.Hk = (int)std::min<int64_t>(H, 1 << 17);
  a.causal = causal != 0;
  const int64_t n = n_keys < 0 || n_keys > k->shape[1] ? k->shape[1] : n_keys;
  const Extent ins[5] = {extent_of("q", q), extent_of("k", k), extent_of("k_pe", k_pe), extent_of("v", v),
                         extent_of("cache_seqlens", cache_seqlens)};
  return lat_common(a, q, cache_seqlens, n, nullptr, softmax_scale, out, lse, ins, 5, workspace, workspace_bytes, stream);
}

}  // extern "C"
