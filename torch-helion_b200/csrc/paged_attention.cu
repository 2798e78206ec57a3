// th_paged_attention: attention of one new token per sequence over a paged
// key-value cache.
#include "common.cuh"

namespace th {

// One block per (sequence, query head).  Each warp takes every fourth key:
// lanes hold the head's elements, the running maximum and sum are per warp
// and the four warps join at the end.
template <typename T>
__global__ void __launch_bounds__(128) paged_attention_kernel(const __grid_constant__ th_paged_attention_args p) {
  pdl_wait();
  pdl_trigger();
  __shared__ float sm_m[4], sm_l[4], sm_o[4][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = p.head_dim;
  const int h = blockIdx.x % p.hq, b = blockIdx.x / p.hq, hk = h / (p.hq / p.hkv);
  const int64_t room = (int64_t)p.table_cols * p.page_size;
  int len = max(p.lens[b], 0);
  if (len > room) {
    if (threadIdx.x == 0) atomicOr(&g_device_error, TH_DEVERR_BAD_ARG);
    len = (int)room;
  }
  const T* q = (const T*)p.q + b * p.q_row + h * p.q_head;
  float qr[8], acc[8], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    qr[e] = lane + 32 * e < d ? to_f32(q[lane + 32 * e]) : 0.f;
    acc[e] = 0.f;
  }
  const int first = p.window > 0 ? max(0, len - p.window) : 0;
  for (int j = first + warp; j < len; j += 4) {
    const int col = j / p.page_size, slot = j - col * p.page_size;
    const int page = p.table[b * p.ld_table + col];
    if (page < 0 || page >= p.num_pages) {
      if (lane == 0) atomicOr(&g_device_error, TH_DEVERR_BAD_ARG);
      continue;
    }
    const T* k = (const T*)p.k_pages + page * p.k_page + hk * p.k_head + slot * p.k_slot;
    const T* v = (const T*)p.v_pages + page * p.v_page + hk * p.v_head + slot * p.v_slot;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (lane + 32 * e < d) s = fmaf(qr[e], to_f32(k[lane + 32 * e]), s);
    s = warp_sum(s) * p.scale;
    if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
    const float mn = fmaxf(m, s), top = mn == -INFINITY ? 0.f : mn;
    const float keep = expf(m - top), w = expf(s - top);
    l = l * keep + w;
    m = mn;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (lane + 32 * e < d) acc[e] = acc[e] * keep + w * to_f32(v[lane + 32 * e]);
  }
  if (lane == 0) { sm_m[warp] = m; sm_l[warp] = l; }
#pragma unroll
  for (int e = 0; e < 8; ++e) sm_o[warp][lane + 32 * e] = acc[e];
  __syncthreads();
  float mm = -INFINITY, ll = 0.f, f[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sm_m[w]);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = sm_m[w] == -INFINITY ? 0.f : expf(sm_m[w] - mm);
    ll += sm_l[w] * f[w];
  }
  T* o = (T*)p.o + b * p.o_row + h * p.o_head;
  for (int i = threadIdx.x; i < d; i += 128) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) x += sm_o[w][i] * f[w];
    o[i] = from_f32<T>(ll == 0.f ? 0.f : x / ll);
  }
  if (p.lse && threadIdx.x == 0) p.lse[(int64_t)b * p.hq + h] = ll == 0.f ? -INFINITY : mm + logf(ll);
}

}  // namespace th

extern "C" size_t th_paged_attention_workspace_size(int32_t hq, int32_t hkv, int32_t head_dim, int32_t dtype) {
  using namespace th;
  if (hq <= 0 || hkv <= 0 || hq % hkv || head_dim <= 0 || head_dim > 256 || dtype < TH_F32 || dtype > TH_F16 ||
      head_dim * elem_bytes(dtype) % 16)
    return 0;
  return 16;
}

extern "C" int th_paged_attention(const th_paged_attention_args* a, void* stream) {
  using namespace th;
  if (!a || !a->q || !a->o || !a->k_pages || !a->v_pages || !a->table || !a->lens || !a->workspace)
    return fail(TH_EINVAL, "th_paged_attention: NULL argument");
  if (a->batch <= 0 || a->hq <= 0 || a->hkv <= 0 || a->hq % a->hkv)
    return fail(TH_EINVAL, "th_paged_attention: bad heads/shape (hq %% hkv must be 0)");
  if (a->page_size <= 0 || a->num_pages <= 0 || a->table_cols <= 0 || a->ld_table < (a->batch > 1 ? a->table_cols : 0))
    return fail(TH_EINVAL, "th_paged_attention: bad cache shape");
  if (a->dtype < TH_F32 || a->dtype > TH_F16) return fail(TH_EDTYPE, "th_paged_attention: bad dtype %d", a->dtype);
  const int eb = elem_bytes(a->dtype);
  if (a->head_dim <= 0 || a->head_dim > 256 || a->head_dim * eb % 16)
    return fail(TH_EUNSUPPORTED, "th_paged_attention: head_dim %d (at most 256, rows of a multiple of 16 bytes)", a->head_dim);
  if (a->window < 0 || !(a->softcap >= 0.f)) return fail(TH_EINVAL, "th_paged_attention: negative window or softcap");
  const int64_t strides[] = {a->k_page, a->k_head, a->k_slot, a->v_page, a->v_head, a->v_slot};
  for (int64_t s : strides)
    if (s * eb % 16) return fail(TH_EALIGN, "th_paged_attention: pool strides must be multiples of 16 bytes");
  if (!aligned16(a->k_pages) || !aligned16(a->v_pages) || !aligned16(a->workspace))
    return fail(TH_EALIGN, "th_paged_attention: pools and workspace must be 16-byte aligned");
  const size_t need = th_paged_attention_workspace_size(a->hq, a->hkv, a->head_dim, a->dtype);
  if (a->workspace_bytes < need)
    return fail(TH_EINVAL, "th_paged_attention: workspace %zu B < %zu B", a->workspace_bytes, need);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)(a->batch * a->hq));
  if (a->dtype == TH_F32) launch_pdl(paged_attention_kernel<float>, grid, dim3(128), 0, st, *a);
  else if (a->dtype == TH_BF16) launch_pdl(paged_attention_kernel<__nv_bfloat16>, grid, dim3(128), 0, st, *a);
  else launch_pdl(paged_attention_kernel<__half>, grid, dim3(128), 0, st, *a);
  return check_launch("th_paged_attention");
}
