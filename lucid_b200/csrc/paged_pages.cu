// Data movement of the paged cache: new rows scattered into the sequences' pages, and
// whole pages copied (forking a sequence, compacting a pool).  Both read and write
// every byte once and compute nothing, so they are bound by HBM (or, for a few rows, by
// one launch and one round of dependent loads).
#include "serve_common.cuh"

namespace lb {

// One warp per (row, tensor): lanes copy 8- or 16-byte vectors of the row's D elements.
// Rows past counts[b], of sequences marked unused (negative length), past the block
// table or on an invalid page are not written.
template <int CB>
__global__ void __launch_bounds__(256) paged_append_kernel(const __grid_constant__ PagedAppendArgs a) {
  using V = typename std::conditional<CB == 16, uint4, uint2>::type;
  const int per = CB / 2, nv = a.D / per;           // vectors per row
  const int b = blockIdx.z;
  const int len = a.lengths[b], cnt = a.counts ? min(a.counts[b], a.N) : a.N;
  if (len < 0) return;
  const long long total = (long long)max(cnt, 0) * nv;  // vectors of one head
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const int n = (int)(i / nv), v = (int)(i % nv);
    const long long pos = (long long)len + n;
    const long long pi = pos / a.ps, row = pos % a.ps;
    if (pi >= a.M) {
      report(a.status, kStatusLength, kTagPagedAppend);
      continue;
    }
    const int page = a.table[(long long)b * a.t_sb + pi];
    if (page < 0 || page >= a.P) {
      report(a.status, kStatusPage, kTagPagedAppend);
      continue;
    }
    for (int h = blockIdx.y; h < a.H; h += gridDim.y) {
      const V kv = *reinterpret_cast<const V*>(a.k + (long long)b * a.k_sb + (long long)h * a.k_sh + (long long)n * a.k_sn + v * per);
      const V xv = *reinterpret_cast<const V*>(a.x + (long long)b * a.x_sb + (long long)h * a.x_sh + (long long)n * a.x_sn + v * per);
      *reinterpret_cast<V*>(a.kp.p + (long long)page * a.kp.sp + (long long)h * a.kp.sh + row * a.kp.sn + v * per) = kv;
      *reinterpret_cast<V*>(a.xp.p + (long long)page * a.xp.sp + (long long)h * a.xp.sh + row * a.xp.sn + v * per) = xv;
    }
  }
}

cudaError_t launch_paged_append(const PagedAppendArgs& a, cudaStream_t st) {
  const bool a16 = ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.x) |
                     reinterpret_cast<uintptr_t>(a.kp.p) | reinterpret_cast<uintptr_t>(a.xp.p)) & 15u) == 0 &&
                   ((a.k_sb | a.k_sh | a.k_sn | a.x_sb | a.x_sh | a.x_sn | a.kp.sp | a.kp.sh | a.kp.sn | a.xp.sp |
                     a.xp.sh | a.xp.sn | a.D) & 7) == 0;
  const long long vec = (long long)a.N * (a.D / (a16 ? 8 : 4));
  const unsigned gx = (unsigned)min((vec + 255) / 256, 1024LL);
  const dim3 grid(gx, (unsigned)min(a.H, 65535), (unsigned)a.B);
  if (a16) paged_append_kernel<16><<<grid, 256, 0, st>>>(a);
  else paged_append_kernel<8><<<grid, 256, 0, st>>>(a);
  return cudaGetLastError();
}

// One block per 16 KB segment of one (pair, layer, tensor); four vectors in flight per
// thread.
constexpr int kCopyThreads = 256, kCopyUnroll = 4;

template <typename V>
__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(const __grid_constant__ PageCopyArgs a) {
  unsigned i = blockIdx.x;
  const int seg = i % a.segs;
  i /= a.segs;
  const int tensor = i & 1;
  i >>= 1;
  const int layer = i % a.layers, pair = i / a.layers;
  char* base = a.pool[tensor] + (long long)layer * a.layer[tensor];
  const V* src = reinterpret_cast<const V*>(base + (long long)a.src[pair] * a.page[tensor]);
  V* dst = reinterpret_cast<V*>(base + (long long)a.dst[pair] * a.page[tensor]);
  const long long nv = a.bytes / (long long)sizeof(V);
  const long long v0 = (long long)seg * kCopyThreads * kCopyUnroll + threadIdx.x;
  V r[kCopyUnroll];
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u)
    if (v0 + u * kCopyThreads < nv) r[u] = src[v0 + u * kCopyThreads];
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u)
    if (v0 + u * kCopyThreads < nv) dst[v0 + u * kCopyThreads] = r[u];
}

cudaError_t launch_page_copy(const PageCopyArgs& in, cudaStream_t st) {
  PageCopyArgs a = in;
  bool a16 = a.bytes % 16 == 0;
  for (int t = 0; t < 2; ++t)
    a16 = a16 && ((reinterpret_cast<uintptr_t>(a.pool[t]) | (uintptr_t)a.layer[t] | (uintptr_t)a.page[t]) & 15u) == 0;
  const long long per = (long long)kCopyThreads * kCopyUnroll * (a16 ? 16 : 8);
  a.segs = (int)((a.bytes + per - 1) / per);
  const unsigned grid = (unsigned)((long long)a.segs * 2 * a.layers * a.pairs);
  if (a16) page_copy_kernel<uint4><<<grid, kCopyThreads, 0, st>>>(a);
  else page_copy_kernel<uint2><<<grid, kCopyThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace lb
