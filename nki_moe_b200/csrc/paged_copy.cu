// Copies of whole pages inside a pool, every layer's key and value planes in
// one launch: what a fork (the last page of a sequence that two continue) and
// a compaction (pages moved to the front of the pool) need.
//
// The page ids are host data (the bookkeeping of pages is the host's), so they
// travel in the kernel's parameters: no staging buffer to keep alive, nothing
// to copy to the device first, and a captured launch keeps its own ids.
#include "paged.cuh"

namespace nkimoe {

namespace {

constexpr int kCopyThreads = 256;
constexpr int kCopyVec = 4;                                   // 16-byte pieces per thread
constexpr long long kCopyPiece = kCopyThreads * kCopyVec * 16;  // bytes per CTA

template <int N>
struct CopyParams {
  char* pages;
  long long plane_bytes, page_bytes;
  int planes, pieces;
  int src[N], dst[N];
};

// CTA (piece, plane, pair).  Bound by HBM: each page read once, written once.
// Measured: 300 pages of 64 KB in 48 planes 287 us = 6.6 TB/s = the measured
// copy; 8 pages of 16 KB in 96 planes 4.6 us.
template <int N>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyParams<N> p) {
  pdl_launch_dependents();
  pdl_wait();
  const unsigned i = blockIdx.x;
  const unsigned piece = i % p.pieces, rest = i / p.pieces;
  const unsigned plane = rest % p.planes, pair = rest / p.planes;
  char* base = p.pages + plane * p.plane_bytes + piece * kCopyPiece;
  const uint4* src = reinterpret_cast<const uint4*>(base + p.src[pair] * p.page_bytes);
  uint4* dst = reinterpret_cast<uint4*>(base + p.dst[pair] * p.page_bytes);
  const int n = static_cast<int>(min(kCopyPiece, p.page_bytes - piece * kCopyPiece) >> 4);
  uint4 v[kCopyVec];
#pragma unroll
  for (int u = 0; u < kCopyVec; ++u) {
    const int at = threadIdx.x + u * kCopyThreads;
    if (at < n) v[u] = __ldcs(src + at);
  }
#pragma unroll
  for (int u = 0; u < kCopyVec; ++u) {
    const int at = threadIdx.x + u * kCopyThreads;
    if (at < n) __stcs(dst + at, v[u]);
  }
}

template <int N>
cudaError_t copy_some(char* pages, long long planes, long long plane_bytes, long long page_bytes, const int* src,
                      const int* dst, int n, cudaStream_t s) {
  CopyParams<N> p;
  p.pages = pages;
  p.plane_bytes = plane_bytes;
  p.page_bytes = page_bytes;
  p.planes = static_cast<int>(planes);
  p.pieces = static_cast<int>((page_bytes + kCopyPiece - 1) / kCopyPiece);
  for (int i = 0; i < N; ++i) {
    p.src[i] = i < n ? src[i] : 0;
    p.dst[i] = i < n ? dst[i] : 0;
  }
  const long long grid = static_cast<long long>(n) * planes * p.pieces;
  return launch_pdl(copy_pages_kernel<N>, dim3(static_cast<unsigned>(grid)), dim3(kCopyThreads), 0, s, p);
}

}  // namespace

// Pairs per launch: the smallest of three parameter blocks that holds them
// (kernel parameters are at most 32764 bytes), and no more CTAs than a grid
// dimension takes.
cudaError_t copy_pages_launch(void* pages, long long planes, long long plane_bytes, long long page_bytes,
                              const int* src, const int* dst, long long n, cudaStream_t s) {
  const long long pieces = (page_bytes + kCopyPiece - 1) / kCopyPiece;
  const long long most = 0x7fffffffLL / (planes * pieces);
  char* base = static_cast<char*>(pages);
  for (long long at = 0; at < n;) {
    long long m = n - at < most ? n - at : most;
    if (m > 4000) m = 4000;
    const int k = static_cast<int>(m);
    cudaError_t e = k <= 32    ? copy_some<32>(base, planes, plane_bytes, page_bytes, src + at, dst + at, k, s)
                    : k <= 480 ? copy_some<480>(base, planes, plane_bytes, page_bytes, src + at, dst + at, k, s)
                               : copy_some<4000>(base, planes, plane_bytes, page_bytes, src + at, dst + at, k, s);
    if (e != cudaSuccess) return e;
    at += m;
  }
  return cudaSuccess;
}

}  // namespace nkimoe
