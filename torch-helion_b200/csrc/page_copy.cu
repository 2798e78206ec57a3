// th_page_copy: copies of pages, or of their first slots, inside one pool.
// Bound by memory: every byte is read once and written once.  On a B200 509
// pages of 2 MB take 317 us, 6.7 TB/s of reads and writes, the rate of a plain
// copy; 64 partly filled ones of 512 planes 20 us on the device, 6.0 TB/s.  One
// block per plane with a load and a store at a time took 345 and 33 us.
#include "common.cuh"

namespace th {

constexpr int PC_FLY = 8;  // loads of V in flight per lane

// The filled slots of one plane are one run of contiguous bytes, cut into
// segments of 32 PC_FLY words V (4 KB at 16 bytes); a warp moves one segment,
// all of its loads before its first store.
template <typename V>
__global__ void __launch_bounds__(256) page_copy_kernel(const __grid_constant__ th_page_copy_args p, int segs) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int64_t items = (int64_t)p.planes * segs;
  for (int i = blockIdx.y; i < p.pairs; i += gridDim.y) {
    const int src = p.src[i], dst = p.dst[i], n = p.counts ? p.counts[i] : p.page_size;
    if (src < 0 || dst < 0) continue;
    if (src >= p.num_pages || dst >= p.num_pages || n < 0 || n > p.page_size) {
      if (threadIdx.x == 0 && blockIdx.x == 0) atomicOr(&g_device_error, TH_DEVERR_BAD_ARG);
      continue;
    }
    const int64_t run = n * (p.slot_bytes / (int64_t)sizeof(V));
    for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < items; w += (int64_t)gridDim.x * 8) {
      const int64_t plane = segs == 1 ? w : w / segs, first = (w - plane * segs) * (32 * PC_FLY) + lane;
      char* base = (char*)p.pages + plane * p.plane_stride;
      const V* from = (const V*)(base + src * p.page_stride) + first;
      V* to = (V*)(base + dst * p.page_stride) + first;
      const int64_t left = run - first;
      V v[PC_FLY];
#pragma unroll
      for (int k = 0; k < PC_FLY; ++k)
        if (k * 32 < left) v[k] = from[k * 32];
#pragma unroll
      for (int k = 0; k < PC_FLY; ++k)
        if (k * 32 < left) to[k * 32] = v[k];
    }
  }
}

template <typename V>
static void page_copy_launch(const th_page_copy_args* a, cudaStream_t st) {
  const int64_t words = a->page_size * (a->slot_bytes / (int64_t)sizeof(V));
  const int64_t segs = (words + 32 * PC_FLY - 1) / (32 * PC_FLY), blocks = (a->planes * segs + 7) / 8;
  const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536), (unsigned)(a->pairs < 65535 ? a->pairs : 65535));
  launch_pdl(page_copy_kernel<V>, grid, dim3(256), 0, st, *a, (int)segs);
}

}  // namespace th

extern "C" int th_page_copy(const th_page_copy_args* a, void* stream) {
  using namespace th;
  if (!a || !a->pages || !a->src || !a->dst) return fail(TH_EINVAL, "th_page_copy: NULL argument");
  if (a->pairs <= 0 || a->num_pages <= 0 || a->planes <= 0 || a->page_size <= 0 || a->slot_bytes <= 0)
    return fail(TH_EINVAL, "th_page_copy: bad shape");
  if (a->slot_bytes > INT32_MAX) return fail(TH_EUNSUPPORTED, "th_page_copy: slots of more than 2^31 bytes");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  // every address is base + multiples of these four: their common alignment is the widest legal access
  const uint64_t low = reinterpret_cast<uintptr_t>(a->pages) | (uint64_t)a->page_stride | (uint64_t)a->plane_stride |
                       (uint64_t)a->slot_bytes;
  if (low % 16 == 0) page_copy_launch<uint4>(a, st);
  else if (low % 4 == 0) page_copy_launch<uint32_t>(a, st);
  else page_copy_launch<uint8_t>(a, st);
  return check_launch("th_page_copy");
}
