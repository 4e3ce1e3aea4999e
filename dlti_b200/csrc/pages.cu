// Copies of cache pages: any number of caches (keys, values, scales of every layer) and pairs of pages in one launch.
//
// Nothing but memory traffic: a page is cut into pieces of 16 KB, one CTA each, whose four 16-byte loads per thread are all in flight before the
// first store: 192 pages of 128 KB in 32 layers, 1.6 GB moved, in 250 us (6.5 TB/s). Caches and pairs travel as kernel arguments, so a call needs no copy to the device, no workspace, and can be captured.
#include "common.cuh"

namespace {

constexpr int MAX_CACHES = 32, MAX_PAIRS = 300;
constexpr int PIECE = 16384;

struct Cache {
  char* base;
  long long layer, page;         // bytes from layer to layer and from page to page
  int layers, bytes;             // bytes of a page
};
struct CopyJob {
  Cache cache[MAX_CACHES];
  int2 pair[MAX_PAIRS];          // from, to
  int first[MAX_CACHES + 1];     // first piece column of a cache: layers * pieces each
  int caches;
};
static_assert(sizeof(CopyJob) <= 4000, "kernel arguments");

template <typename V>
__device__ __forceinline__ void copy_piece(const char* src, char* dst, int n) {
  constexpr int S = sizeof(V);
  for (int a = threadIdx.x * S; a < n; a += 4 * 256 * S) {
    V v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (a + i * 256 * S < n) v[i] = *reinterpret_cast<const V*>(src + a + i * 256 * S);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (a + i * 256 * S < n) *reinterpret_cast<V*>(dst + a + i * 256 * S) = v[i];
  }
}

__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyJob job) {
  const int col = blockIdx.x;
  int c = 0;
  while (col >= job.first[c + 1]) ++c;
  const Cache& k = job.cache[c];
  const int pieces = (k.bytes + PIECE - 1) / PIECE;
  const int layer = (col - job.first[c]) / pieces, at = ((col - job.first[c]) % pieces) * PIECE;
  const int n = min(PIECE, k.bytes - at);
  const int2 pr = job.pair[blockIdx.y];
  const char* src = k.base + layer * k.layer + pr.x * k.page + at;
  char* dst = k.base + layer * k.layer + pr.y * k.page + at;
  const unsigned long long low = (unsigned long long)src | (unsigned long long)dst | (unsigned)n;
  if ((low & 15) == 0) copy_piece<int4>(src, dst, n);
  else if ((low & 3) == 0) copy_piece<int>(src, dst, n);
  else copy_piece<char>(src, dst, n);
}

}  // namespace

// caches: base address, layers, bytes from layer to layer, bytes from page to page, bytes of a page, of each. Pages from[i] -> to[i] of every
// layer of every cache, all on the host; no page is written twice or both read and written (the caller's check).
DLTI_API int dlti_copy_pages(const long long* caches, int count, const int* from, const int* to, int pairs, cudaStream_t st) {
  if (pairs <= 0 || count <= 0) return 0;
  for (int c = 0; c < count; ++c) {
    const long long layers = caches[5 * c + 1], bytes = caches[5 * c + 4];
    if (bytes <= 0 || bytes > 1 << 30 || layers <= 0 || layers * ((bytes + PIECE - 1) / PIECE) > 1 << 24) {
      dlti_set_error("copy_pages: a cache without layers, with pages of nothing, or with more than 2^24 pieces of 16 KB in a page of all layers");
      return DLTI_ERR_BAD_ARG;
    }
  }
  CopyJob job;
  for (int c0 = 0; c0 < count; c0 += MAX_CACHES) {
    job.caches = count - c0 < MAX_CACHES ? count - c0 : MAX_CACHES;
    job.first[0] = 0;
    for (int c = 0; c < job.caches; ++c) {
      const long long* k = caches + 5 * (c0 + c);
      job.cache[c] = Cache{reinterpret_cast<char*>(k[0]), k[2], k[3], (int)k[1], (int)k[4]};
      job.first[c + 1] = job.first[c] + (int)k[1] * (int)((k[4] + PIECE - 1) / PIECE);
    }
    for (int p0 = 0; p0 < pairs; p0 += MAX_PAIRS) {
      const int n = pairs - p0 < MAX_PAIRS ? pairs - p0 : MAX_PAIRS;
      for (int i = 0; i < n; ++i) job.pair[i] = make_int2(from[p0 + i], to[p0 + i]);
      copy_pages_kernel<<<dim3((unsigned)job.first[job.caches], (unsigned)n), 256, 0, st>>>(job);
      dlti_count_launch();
    }
  }
  return (int)cudaGetLastError();
}
