// th_page_copy: copies of pages, or of their first slots, inside one pool.
#include "common.cuh"

namespace th {

// One block per (pair, plane): the plane's filled slots are one run of
// contiguous bytes, moved V bytes per thread and step.
template <typename V>
__global__ void __launch_bounds__(256) page_copy_kernel(const __grid_constant__ th_page_copy_args p) {
  pdl_wait();
  pdl_trigger();
  const int64_t all = (int64_t)p.pairs * p.planes;
  for (int64_t w = blockIdx.x; w < all; w += gridDim.x) {
    const int i = (int)(w / p.planes);
    const int64_t plane = w - (int64_t)i * p.planes;
    const int src = p.src[i], dst = p.dst[i], n = p.counts ? p.counts[i] : p.page_size;
    if (src < 0 || dst < 0) continue;
    if (src >= p.num_pages || dst >= p.num_pages || n < 0 || n > p.page_size) {
      if (threadIdx.x == 0) atomicOr(&g_device_error, TH_DEVERR_BAD_ARG);
      continue;
    }
    char* base = (char*)p.pages + plane * p.plane_stride;
    const V* from = (const V*)(base + src * p.page_stride);
    V* to = (V*)(base + dst * p.page_stride);
    const int64_t run = n * p.slot_bytes / (int64_t)sizeof(V);
    for (int64_t c = threadIdx.x; c < run; c += blockDim.x) to[c] = from[c];
  }
}

}  // namespace th

extern "C" int th_page_copy(const th_page_copy_args* a, void* stream) {
  using namespace th;
  if (!a || !a->pages || !a->src || !a->dst) return fail(TH_EINVAL, "th_page_copy: NULL argument");
  if (a->pairs <= 0 || a->num_pages <= 0 || a->planes <= 0 || a->page_size <= 0 || a->slot_bytes <= 0)
    return fail(TH_EINVAL, "th_page_copy: bad shape");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // every address is base + multiples of these four: their common alignment is the widest legal access
  const uint64_t low = reinterpret_cast<uintptr_t>(a->pages) | (uint64_t)a->page_stride | (uint64_t)a->plane_stride |
                       (uint64_t)a->slot_bytes;
  const int64_t want = (int64_t)a->pairs * a->planes, cap = (int64_t)sm_count() * 64;
  const dim3 grid((unsigned)(want < cap ? want : cap));
  if (low % 16 == 0) launch_pdl(page_copy_kernel<uint4>, grid, dim3(256), 0, st, *a);
  else if (low % 4 == 0) launch_pdl(page_copy_kernel<uint32_t>, grid, dim3(256), 0, st, *a);
  else launch_pdl(page_copy_kernel<uint8_t>, grid, dim3(256), 0, st, *a);
  return check_launch("th_page_copy");
}
