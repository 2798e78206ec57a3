// th_rope / th_rope_append: rotary positions on queries and keys, and the
// append of rotated keys and of values to a paged cache.
#include "common.cuh"

namespace th {

// Where the heads of one token come from and go to: unit h < hq is query head
// h, then hkv keys, then (append) hkv values, which are copied.
template <typename T>
struct RopeUnit {
  const T* src;
  T* dst;   // nullptr: nothing to store
  T* dst2;  // a second copy of the result (rotated keys outside the cache), or nullptr
  bool rotate;
};

// Page slot of token t in the cache, or false (padding, or an id out of range,
// which is reported).
__device__ __forceinline__ bool rope_slot(const th_rope_args& p, int64_t t, int pos, int& page, int& slot) {
  if (pos < 0) return false;
  int64_t row = t;
  if (p.seqs) row = p.seqs[t];
  const int col = pos / p.page_size;
  if (row < 0 || row >= p.batch || col >= p.table_cols) {
    atomicOr(&g_device_error, TH_DEVERR_BAD_ARG);
    return false;
  }
  page = p.table[row * p.ld_table + col];
  slot = pos - col * p.page_size;
  if (page < 0 || page >= p.num_pages) {
    atomicOr(&g_device_error, TH_DEVERR_BAD_ARG);
    return false;
  }
  return true;
}

template <typename T, bool APPEND>
__device__ __forceinline__ RopeUnit<T> rope_unit(const th_rope_args& p, int64_t t, int h, bool cached, int page,
                                                 int slot) {
  RopeUnit<T> u;
  u.rotate = true;
  u.dst2 = nullptr;
  if (h < p.hq) {
    u.src = (const T*)p.q + t * p.q_token + h * p.q_head;
    u.dst = (T*)p.q_out + t * p.qo_token + h * p.qo_head;
    return u;
  }
  h -= p.hq;
  if (!APPEND) {
    u.src = (const T*)p.k + t * p.k_token + h * p.k_head;
    u.dst = (T*)p.k_out + t * p.ko_token + h * p.ko_head;
  } else if (h < p.hkv) {
    u.src = (const T*)p.k + t * p.k_token + h * p.k_head;
    u.dst = cached ? (T*)p.k_pages + page * p.k_page + h * p.k_phead + slot * p.k_slot : nullptr;
    u.dst2 = p.k_out ? (T*)p.k_out + t * p.ko_token + h * p.ko_head : nullptr;
  } else {
    h -= p.hkv;
    u.src = (const T*)p.v + t * p.v_token + h * p.v_head;
    u.dst = cached ? (T*)p.v_pages + page * p.v_page + h * p.v_phead + slot * p.v_slot : nullptr;
    u.rotate = false;
  }
  return u;
}

// One warp per (token, head), one element pair per lane: every stride,
// alignment and rotary width.
template <typename T, bool APPEND>
__global__ void __launch_bounds__(256) rope_any_kernel(const __grid_constant__ th_rope_args p) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, half = p.rotary_dim / 2;
  const int units = p.hq + p.hkv * (APPEND ? 2 : 1);
  const int64_t all = p.tokens * units, nw = (int64_t)gridDim.x * 8;
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < all; w += nw) {
    const int64_t t = w / units;
    const int h = (int)(w - t * units), pos = p.positions[t];
    int page = 0, slot = 0;
    bool cached = false;
    if (APPEND && h >= p.hq) cached = rope_slot(p, t, pos, page, slot);
    const bool known = pos >= 0 && pos < p.table_rows;
    if (pos >= p.table_rows && lane == 0) atomicOr(&g_device_error, TH_DEVERR_BAD_ARG);
    const RopeUnit<T> u = rope_unit<T, APPEND>(p, t, h, cached && known, page, slot);
    if (!known) {  // padding: the caller's rows are zero, the cache is left alone
      T* z = APPEND && h >= p.hq ? u.dst2 : u.dst;
      for (int i = lane; z && i < p.head_dim; i += 32) z[i] = from_f32<T>(0.f);
      continue;
    }
    if (!u.dst && !u.dst2) continue;
    const int turned = u.rotate ? half : 0;
    const float* cs = p.cos + pos * p.ld_cs;
    const float* sn = p.sin + pos * p.ld_cs;
    for (int i = lane; i < turned; i += 32) {
      const int ia = p.interleaved ? 2 * i : i, ib = p.interleaved ? 2 * i + 1 : i + half;
      const float a = to_f32(u.src[ia]), b = to_f32(u.src[ib]), c = cs[i], s = p.inverse ? -sn[i] : sn[i];
      const T ra = from_f32<T>(a * c - b * s), rb = from_f32<T>(a * s + b * c);
      if (u.dst) { u.dst[ia] = ra; u.dst[ib] = rb; }
      if (u.dst2) { u.dst2[ia] = ra; u.dst2[ib] = rb; }
    }
    for (int i = 2 * turned + lane; i < p.head_dim; i += 32) {
      const T x = u.src[i];
      if (u.dst) u.dst[i] = x;
      if (u.dst2) u.dst2[i] = x;
    }
  }
}

template <typename T, bool APPEND>
static int rope_launch(const th_rope_args* a, cudaStream_t st, const char* what) {
  const int64_t warps = a->tokens * (a->hq + a->hkv * (APPEND ? 2 : 1));
  const int64_t want = (warps + 7) / 8, cap = (int64_t)sm_count() * 64;
  launch_pdl(rope_any_kernel<T, APPEND>, dim3((unsigned)(want < cap ? want : cap)), dim3(256), 0, st, *a);
  return check_launch(what);
}

static int rope_checked(const th_rope_args* a, void* stream, bool append, const char* what) {
  if (!a || !a->positions || !a->cos || !a->sin) return fail(TH_EINVAL, "%s: NULL argument", what);
  if (a->tokens <= 0 || a->hq < 0 || a->hkv < 0 || a->hq + a->hkv <= 0 || a->head_dim <= 0 || a->table_rows <= 0)
    return fail(TH_EINVAL, "%s: bad shape", what);
  if (a->rotary_dim <= 0 || a->rotary_dim % 2 || a->rotary_dim > a->head_dim)
    return fail(TH_EINVAL, "%s: rotary_dim %d must be even, positive and at most head_dim %d", what, a->rotary_dim, a->head_dim);
  if (a->ld_cs < a->rotary_dim / 2 && a->table_rows > 1) return fail(TH_EINVAL, "%s: ld_cs too small", what);
  if (a->hq && (!a->q || !a->q_out)) return fail(TH_EINVAL, "%s: NULL q or q_out", what);
  if (a->hkv && !a->k) return fail(TH_EINVAL, "%s: NULL k", what);
  th_rope_args b = *a;
  if (append) {
    if (a->hkv <= 0 || !a->v || !a->k_pages || !a->v_pages || !a->table)
      return fail(TH_EINVAL, "%s: keys, values, pools and table are needed", what);
    if (a->batch <= 0 || a->table_cols <= 0 || a->page_size <= 0 || a->num_pages <= 0 || a->ld_table < (a->batch > 1 ? a->table_cols : 0))
      return fail(TH_EINVAL, "%s: bad cache shape", what);
    if (!a->seqs && a->tokens > a->batch) return fail(TH_EINVAL, "%s: more tokens than table rows without seqs", what);
    b.inverse = 0;
  } else if (a->hkv && !a->k_out) {
    return fail(TH_EINVAL, "%s: NULL k_out", what);
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case TH_F32: return append ? rope_launch<float, true>(&b, st, what) : rope_launch<float, false>(&b, st, what);
    case TH_BF16: return append ? rope_launch<__nv_bfloat16, true>(&b, st, what) : rope_launch<__nv_bfloat16, false>(&b, st, what);
    case TH_F16: return append ? rope_launch<__half, true>(&b, st, what) : rope_launch<__half, false>(&b, st, what);
    default: return fail(TH_EDTYPE, "%s: bad dtype %d", what, a->dtype);
  }
}

}  // namespace th

extern "C" int th_rope(const th_rope_args* a, void* stream) { return th::rope_checked(a, stream, false, "th_rope"); }

extern "C" int th_rope_append(const th_rope_args* a, void* stream) {
  return th::rope_checked(a, stream, true, "th_rope_append");
}
