// Pages of a cache copied in place, in all layers and planes (keys, values) of a pool at once: what a fork of a request and the
// bringing together of a pool's live pages do on the device.
//
// A pool is [layers, n_pages * (w_0 + .. )] elements: within a layer the planes lie one behind the other, plane j as n_pages
// pages of w_j elements.  Pair i copies page src[i] to page dst[i] of every plane of every layer.  Nothing is computed; what
// bounds it is memory, each page read once and written once, and for a few pages the launch.
#include "common.h"

#define COPY_THREADS 256
#define COPY_PLANES 4

typedef uint32_t copy_word4 __attribute__((ext_vector_type(4)));

struct CopyPlanes {
  size_t start[COPY_PLANES];            // bytes from a layer's start to the plane's
  uint32_t bytes[COPY_PLANES];          // of a page of the plane
  uint32_t blocks_before[COPY_PLANES + 1];   // workgroups of a page in the planes before this one
};

// One workgroup copies COPY_THREADS pieces (of sizeof(Piece) bytes) of one page of one plane of one layer, a piece a thread: the
// device holds enough of them to keep memory busy (1,600 pages of 28 layers, 2.9 GB: 565 us, 5.2 TB/s, where torch's copy of 2 GiB reaches
// 5.0; four pieces a thread 565, eight 869; nontemporal 549, but 29 us instead of 26 for what lies in the caches).  Three pages of 24
// layers: 2.4 us.  (Pieces are vectors, not the runtime's structs of four words: those, kept in an array, were put into LDS, and
// the kernel asked the launch's packet in host memory how large it is, 9 us.)
// A pair that names a page outside the pool is passed over.
template <typename Piece>
__global__ void __launch_bounds__(COPY_THREADS)
copy_pages_kernel(char* __restrict__ pool, size_t layer_bytes, CopyPlanes planes, int n_planes, const int* __restrict__ src,
                  const int* __restrict__ dst, int n_pages) {
  const int from = scalar_int(src + blockIdx.y), to = scalar_int(dst + blockIdx.y);
  if ((uint32_t)from >= (uint32_t)n_pages || (uint32_t)to >= (uint32_t)n_pages || from == to) return;
  int plane = 0;
#pragma unroll
  for (int p = 1; p < COPY_PLANES; ++p)
    if (p < n_planes && blockIdx.x >= planes.blocks_before[p]) plane = p;
  size_t start = planes.start[0];
  uint32_t bytes = planes.bytes[0], before = 0;
#pragma unroll
  for (int p = 1; p < COPY_PLANES; ++p)
    if (plane == p) { start = planes.start[p]; bytes = planes.bytes[p]; before = planes.blocks_before[p]; }
  char* base = pool + (size_t)blockIdx.z * layer_bytes + start;
  const Piece* in = reinterpret_cast<const Piece*>(base + (size_t)from * bytes);
  Piece* out = reinterpret_cast<Piece*>(base + (size_t)to * bytes);
  const uint32_t count = bytes / sizeof(Piece);
  const uint32_t at = (blockIdx.x - before) * COPY_THREADS + threadIdx.x;
  if (at < count) out[at] = in[at];
}

template <typename Piece>
static int launch_copy(char* pool, size_t layer_bytes, CopyPlanes planes, int n_planes, const int* src, const int* dst, int n_pairs,
                       int n_pages, int layers, hipStream_t stream) {
  uint32_t blocks = 0;
  for (int p = 0; p < n_planes; ++p) {
    planes.blocks_before[p] = blocks;
    const uint32_t pieces = planes.bytes[p] / sizeof(Piece);
    blocks += (pieces + COPY_THREADS - 1) / COPY_THREADS;
  }
  planes.blocks_before[n_planes] = blocks;
  // (A launch takes up to 65,535 workgroups in the directions of pairs and layers.)
  for (int pair = 0; pair < n_pairs; pair += 65535) {
    const int pairs = n_pairs - pair < 65535 ? n_pairs - pair : 65535;
    copy_pages_kernel<Piece><<<dim3(blocks, pairs, layers), COPY_THREADS, 0, stream>>>(pool, layer_bytes, planes, n_planes,
                                                                                        src + pair, dst + pair, n_pages);
    const int status = LAUNCH_STATUS();
    if (status) return status;
  }
  return 0;
}

// widths: elements a page has in each plane (host).  src, dst: int32 [n_pairs] on the device.  A page that a pair writes is neither
// read nor written by another pair.
extern "C" int ta_copy_pages(void* pool, const void* src, const void* dst, int n_pairs, int n_pages, int layers, int n_planes,
                             int width0, int width1, int width2, int width3, int dtype, hipStream_t stream) {
  if (n_pairs <= 0) return 0;
  const int widths[COPY_PLANES] = {width0, width1, width2, width3};
  if (!pool || !src || !dst || n_pages < 1 || layers < 1 || layers > 65535 || n_planes < 1 || n_planes > COPY_PLANES) return -1;
  const size_t size = dtype == DT_F32 ? 4 : 2;
  CopyPlanes planes = {};
  size_t at = 0, align = (size_t)pool | 16;
  for (int p = 0; p < n_planes; ++p) {
    const size_t bytes = (size_t)widths[p] * size;
    if (widths[p] < 1 || bytes > 0x7fffffffu) return -1;
    planes.start[p] = at;
    planes.bytes[p] = (uint32_t)bytes;
    at += bytes * n_pages;
    align |= bytes;                      // every page starts, and every layer ends, at a multiple of what all of these are
  }
  char* base = (char*)pool;
  const int *s = (const int*)src, *d = (const int*)dst;
  if (align % 16 == 0) return launch_copy<copy_word4>(base, at, planes, n_planes, s, d, n_pairs, n_pages, layers, stream);
  if (align % 4 == 0) return launch_copy<uint32_t>(base, at, planes, n_planes, s, d, n_pairs, n_pages, layers, stream);
  return launch_copy<uint16_t>(base, at, planes, n_planes, s, d, n_pairs, n_pages, layers, stream);
}
