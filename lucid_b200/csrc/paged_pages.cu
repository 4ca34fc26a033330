// Data movement of the paged cache: new rows scattered into the sequences' pages, and
// whole pages copied (forking a sequence, compacting a pool).  Both read and write
// every byte once and compute nothing, so they are bound by HBM (or, for a few rows, by
// one launch and one round of dependent loads).
#include "serve_common.cuh"

#include <algorithm>
#include <type_traits>

namespace lb {

// A block takes 256 / nv rows at a time, nv being the 8- or 16-byte vectors of a row: a
// thread keeps its vector, finds its row's page once and copies it for HN heads of both
// pools, all loads before the stores.  Rows past counts[b], of sequences marked unused
// (negative length), past the block table or on an invalid page are not written.
template <int CB, int HN>
__global__ void __launch_bounds__(256) paged_append_kernel(const __grid_constant__ PagedAppendArgs a) {
  using V = typename std::conditional<CB == 16, uint4, uint2>::type;
  constexpr int per = CB / 2;
  const int nv = a.D / per, rows = 256 / nv;
  const int b = blockIdx.z, mine = threadIdx.x / nv, v = threadIdx.x - mine * nv;
  const int len = a.lengths[b], cnt = a.counts ? min(a.counts[b], a.N) : a.N;
  if (len < 0 || mine >= rows) return;
  const bf16* ks = a.k + (long long)b * a.k_sb + v * per;
  const bf16* xs = a.x + (long long)b * a.x_sb + v * per;
  for (long long n = (long long)blockIdx.x * rows + mine; n < cnt; n += (long long)gridDim.x * rows) {
    const long long pos = len + n;
    if (pos >= (long long)a.M * a.ps) {
      report(a.status, kStatusLength, kTagPagedAppend);
      return;
    }
    const unsigned pi = (unsigned)pos / (unsigned)a.ps, row = (unsigned)pos - pi * a.ps;
    const int page = a.table[(long long)b * a.t_sb + pi];
    if (page < 0 || page >= a.P) {
      report(a.status, kStatusPage, kTagPagedAppend);
      continue;
    }
    bf16* kd = a.kp.p + page * a.kp.sp + row * a.kp.sn + v * per;
    bf16* xd = a.xp.p + page * a.xp.sp + row * a.xp.sn + v * per;
    for (int h0 = blockIdx.y * HN; h0 < a.H; h0 += gridDim.y * HN) {
      V kv[HN], xv[HN];
#pragma unroll
      for (int u = 0; u < HN; ++u)
        if (h0 + u < a.H) {
          kv[u] = *reinterpret_cast<const V*>(ks + (h0 + u) * a.k_sh + n * a.k_sn);
          xv[u] = *reinterpret_cast<const V*>(xs + (h0 + u) * a.x_sh + n * a.x_sn);
        }
#pragma unroll
      for (int u = 0; u < HN; ++u)
        if (h0 + u < a.H) {
          *reinterpret_cast<V*>(kd + (h0 + u) * a.kp.sh) = kv[u];
          *reinterpret_cast<V*>(xd + (h0 + u) * a.xp.sh) = xv[u];
        }
    }
  }
}

cudaError_t launch_paged_append(const PagedAppendArgs& a, cudaStream_t st) {
  const bool a16 = ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.x) |
                     reinterpret_cast<uintptr_t>(a.kp.p) | reinterpret_cast<uintptr_t>(a.xp.p)) & 15u) == 0 &&
                   ((a.k_sb | a.k_sh | a.k_sn | a.x_sb | a.x_sh | a.x_sn | a.kp.sp | a.kp.sh | a.kp.sn | a.xp.sp |
                     a.xp.sh | a.xp.sn | a.D) & 7) == 0;
  const int rows = 256 / (a.D / (a16 ? 8 : 4));
  const unsigned gx = (unsigned)std::min(((long long)a.N + rows - 1) / rows, 4096LL);
  // few rows: a block per head, for the latency; many: four heads a thread
  const bool few = (long long)gx * a.B < 296;
  const dim3 grid(gx, (unsigned)std::min(few ? a.H : (a.H + 3) / 4, 65535), (unsigned)a.B);
  if (few) {
    if (a16) paged_append_kernel<16, 1><<<grid, 256, 0, st>>>(a);
    else paged_append_kernel<8, 1><<<grid, 256, 0, st>>>(a);
  } else {
    if (a16) paged_append_kernel<16, 4><<<grid, 256, 0, st>>>(a);
    else paged_append_kernel<8, 4><<<grid, 256, 0, st>>>(a);
  }
  return cudaGetLastError();
}

// One block per segment of one (pair, layer, tensor), 16 KB of it, or 8 KB where vectors are
// 8 bytes; four vectors in flight per thread.
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
