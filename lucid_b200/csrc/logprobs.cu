// Log probabilities of given tokens, entropy and the most likely alternatives of each
// row of logits, and the gradient of the first two.
//
// For a row x of V logits with maximum m, in units of log2:
//   t_i = (x_i - m) log2 e,   l = sum 2^t_i,   w = sum 2^t_i t_i
//   log p_i = x_i - m - ln l,     H = ln 2 (log2 l - w / l)
// The difference is taken before the scaling, so far-off maxima cost no digits and a row
// at its type's lowest value does not overflow.  Each thread keeps (m, l, w) over its
// elements in one pass; when its maximum grows by d:  w <- 2^-d (w - d l),  l <- 2^-d l;
// the block then joins its threads.  All sums are fp32.
//
// The k best: the maxima of 128 groups of threads are at hand after that pass; the k-th
// largest of them, T, has k elements at or above it, so the k best are among the elements
// >= T, of which there are few more than k unless the row clusters.  They are
// collected (those equal to T apart) and ranked by (value, lowest index).  If more than
// fits is above T, T is made exact by selecting byte by byte over histograms (then fewer
// than k are above it); if too many equal T, the lowest indices are taken by a scan
// in order.
#include "serve_common.cuh"

#include <algorithm>

namespace lb {

constexpr int kLpThreads = 512, kLpWarps = kLpThreads / 32;
constexpr int kLpGroups = 128;   // groups of 4 threads
constexpr int kLpCap = 512;      // list of elements above T, and of those equal to it
constexpr float kLpFloor = -200.f;  // 2^-200 is 0 in fp32; keeps 0 * -inf out of w

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<bf16>(bf16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float v) { return __float2bfloat16(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half(v); }

// a row as 16-byte vectors from the 16-byte boundary at or below its start: vector v
// holds the elements [v VE - shift, +VE); the first and last may be partial
template <typename T>
struct RowView {
  static constexpr int VE = 16 / (int)sizeof(T);
  const T* row;
  int V, shift, nvec;
  __device__ RowView(const T* r, int n) : row(r), V(n) {
    shift = (int)((reinterpret_cast<uintptr_t>(r) & 15u) / sizeof(T));
    nvec = (int)(((long long)shift + n + VE - 1) / VE);
  }
  __device__ __forceinline__ int first(int v) const { return (int)((long long)v * VE - shift); }
  __device__ __forceinline__ void load(int v, float (&x)[VE]) const {
    const int e0 = first(v);
    if (e0 >= 0 && e0 <= V - VE) {
      const uint4 u = *reinterpret_cast<const uint4*>(row + e0);
      const T* p = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < VE; ++i) x[i] = to_f32<T>(p[i]);
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) x[i] = e0 + i >= 0 && e0 + i < V ? to_f32<T>(row[e0 + i]) : -INFINITY;
    }
  }
};

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// order-preserving unsigned key (-0 and +0 alike)
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

struct LpShared {
  float gmax[kLpGroups];
  float wm[kLpWarps], wl[kLpWarps], ww[kLpWarps];
  float T;
  int na, nb, need;
  float av[kLpCap];
  int ai[kLpCap], bi[kLpCap];
  int hist[256];
  uint32_t prefix;
  int remain;
  int wcount[kLpWarps];
};

template <typename T>
__global__ void __launch_bounds__(kLpThreads) logprobs_fwd_kernel(const __grid_constant__ LogprobArgs a) {
  __shared__ LpShared sh;
  constexpr int VE = RowView<T>::VE;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long r = blockIdx.x;
  const RowView<T> row(static_cast<const T*>(a.logits) + (r / a.R1) * a.s0 + (r % a.R1) * a.s1, a.V);
  // ---- one pass: maximum, sum, entropy sum ----
  float mx = -INFINITY, l = 0.f, w = 0.f;
  for (int v = tid; v < row.nvec; v += kLpThreads) {
    float x[VE];
    row.load(v, x);
    float vm = x[0];
#pragma unroll
    for (int i = 1; i < VE; ++i) vm = max_nan(vm, x[i]);
    if (!(vm <= mx)) {            // larger, or NaN
      const float mn = max_nan(mx, vm);
      if (l > 0.f) {
        const float d = fmaxf((mx - mn) * kLog2e, kLpFloor), f = exp2f(d);
        w = f * (w + d * l);
        l *= f;
      }
      mx = mn;
    }
    if (vm == -INFINITY) continue;  // nothing to add (and mx may not be finite yet)
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const float t = fmaxf((x[i] - mx) * kLog2e, kLpFloor);
      const float p = exp2f(t);
      l += p;
      w = fmaf(p, t, w);
    }
  }
  // ---- join the block ----
  float bm = mx;
  float gm = bm;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    bm = max_nan(bm, __shfl_xor_sync(0xffffffffu, bm, o));
    if (o == 2) gm = bm;          // 4 lanes
  }
  if ((lane & 3) == 0) sh.gmax[tid >> 2] = gm;
  if (lane == 0) sh.wm[warp] = bm;
  if (tid == 0) sh.na = sh.nb = 0;
  __syncthreads();
  float M = sh.wm[0];
#pragma unroll
  for (int i = 1; i < kLpWarps; ++i) M = max_nan(M, sh.wm[i]);
  const bool ok = fabsf(M) < INFINITY;  // else no distribution: all -inf, a NaN or +inf
  float lj = 0.f, wj = 0.f;
  if (l > 0.f) {
    const float d = fmaxf((mx - M) * kLog2e, kLpFloor), f = exp2f(d);
    lj = l * f;
    wj = f * (w + d * l);
  }
  lj = warp_sum_f(lj);
  wj = warp_sum_f(wj);
  if (lane == 0) {
    sh.wl[warp] = lj;
    sh.ww[warp] = wj;
  }
  if (a.top > 0 && ok && tid < kLpGroups) {  // the top-th largest of the group maxima
    const float v = sh.gmax[tid];
    int rank = 0;
    for (int i = 0; i < kLpGroups; ++i) {
      const float o = sh.gmax[i];
      rank += o > v || (o == v && i < tid);
    }
    if (rank == a.top - 1) sh.T = v;
  }
  __syncthreads();
  float L = 0.f, W = 0.f;
#pragma unroll
  for (int i = 0; i < kLpWarps; ++i) {
    L += sh.wl[i];
    W += sh.ww[i];
  }
  const float ll = log2f(L), ln = logf(L);
  const float nan = __int_as_float(0x7fc00000);
  if (tid == 0) {
    a.entropy[r] = ok ? kLn2 * (ll - W / L) : nan;
    if (a.stats != nullptr) {
      a.stats[2 * r] = ok ? M : nan;
      a.stats[2 * r + 1] = ok ? ll : nan;
    }
    if (a.tokens != nullptr) {
      const long long tok = a.tokens[r];
      float lp = 0.f;
      if (tok >= 0 && tok < a.V) lp = ok ? (to_f32<T>(row.row[tok]) - M) - ln : nan;
      else if (tok != -100) {
        report(a.status, kStatusToken, kTagLogprobs);
        lp = nan;
      }
      a.logprobs[r] = lp;
    }
  }
  if (a.top == 0) return;
  if (!ok) {
    for (int i = tid; i < a.top; i += kLpThreads) {
      a.top_lp[r * a.top + i] = nan;
      a.top_tok[r * a.top + i] = -1;
    }
    return;
  }
  // ---- the top best ----
  float thr = sh.T;
  auto collect = [&](float t) {
    for (int v = tid; v < row.nvec; v += kLpThreads) {
      float x[VE];
      row.load(v, x);
      float vm = x[0];
#pragma unroll
      for (int i = 1; i < VE; ++i) vm = fmaxf(vm, x[i]);
      if (vm < t) continue;
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const int e = row.first(v) + i;
        if (x[i] >= t && e >= 0 && e < a.V) {
          if (x[i] > t) {
            const int at = atomicAdd(&sh.na, 1);
            if (at < kLpCap) {
              sh.av[at] = x[i];
              sh.ai[at] = e;
            }
          } else {
            const int at = atomicAdd(&sh.nb, 1);
            if (at < kLpCap) sh.bi[at] = e;
          }
        }
      }
    }
    __syncthreads();
  };
  collect(thr);
  if (sh.na > kLpCap) {  // uniform: make the threshold the exact top-th largest value
    if (tid == 0) {
      sh.prefix = 0;
      sh.remain = a.top;
    }
    for (int byte = 3; byte >= 0; --byte) {
      __syncthreads();
      if (tid < 256) sh.hist[tid] = 0;
      __syncthreads();
      const uint32_t pre = sh.prefix;
      for (int v = tid; v < row.nvec; v += kLpThreads) {
        float x[VE];
        row.load(v, x);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const int e = row.first(v) + i;
          const uint32_t key = order_key(x[i]);
          if (e >= 0 && e < a.V && (byte == 3 || (key >> (8 * byte + 8)) == pre)) atomicAdd(&sh.hist[(key >> (8 * byte)) & 255], 1);
        }
      }
      __syncthreads();
      if (tid == 0) {
        int need = sh.remain, d = 255;
        while (d > 0 && sh.hist[d] < need) need -= sh.hist[d--];
        sh.remain = need;
        sh.prefix = (pre << 8) | (uint32_t)d;
      }
    }
    __syncthreads();
    thr = key_value(sh.prefix);
    if (tid == 0) sh.na = sh.nb = 0;
    __syncthreads();
    collect(thr);
  }
  const int na = sh.na;
  int nb = sh.nb;
  if (nb > kLpCap) {  // uniform: the lowest indices equal to the threshold, by a scan in order
    const int need = max(a.top - na, 0);
    __syncthreads();
    int found = 0;
    for (int e0 = 0; e0 < a.V && found < need; e0 += kLpThreads) {
      const int e = e0 + tid;
      const bool hit = e < a.V && to_f32<T>(row.row[e]) == thr;
      const unsigned bal = __ballot_sync(0xffffffffu, hit);
      if (lane == 0) sh.wcount[warp] = __popc(bal);
      __syncthreads();
      int at = found, all = 0;
      for (int i = 0; i < kLpWarps; ++i) {
        if (i < warp) at += sh.wcount[i];
        all += sh.wcount[i];
      }
      at += __popc(bal & ((1u << lane) - 1u));
      if (hit && at < need) sh.bi[at] = e;
      found += all;
      __syncthreads();
    }
    nb = need;
  }
  // rank: values above the threshold by (value, index), those equal to it by index behind them
  for (int i = tid; i < na + nb; i += kLpThreads) {
    int rank;
    float v;
    int e;
    if (i < na) {
      v = sh.av[i];
      e = sh.ai[i];
      rank = 0;
      for (int q = 0; q < na; ++q) rank += sh.av[q] > v || (sh.av[q] == v && sh.ai[q] < e);
    } else {
      v = thr;
      e = sh.bi[i - na];
      rank = na;
      for (int q = 0; q < nb; ++q) rank += sh.bi[q] < e;
    }
    if (rank < a.top) {
      a.top_lp[r * a.top + rank] = (v - M) - ln;
      a.top_tok[r * a.top + rank] = e;
    }
  }
}

// d x_i = g_lp (1[i = tok] - p_i) - g_ent p_i (log p_i + H).  Rows with both factors 0
// (a masked token, say) are written as zeros without being read.
template <typename T>
__global__ void __launch_bounds__(kLpThreads) logprobs_bwd_kernel(const __grid_constant__ LogprobArgs a) {
  constexpr int VE = RowView<T>::VE;
  const long long r = blockIdx.x;
  const long long tok = a.tokens != nullptr ? a.tokens[r] : -100;
  const float gl = a.g_lp != nullptr && tok >= 0 ? a.g_lp[r] : 0.f;
  const float ge = a.g_ent != nullptr ? a.g_ent[r] : 0.f;
  const T* in = static_cast<const T*>(a.logits) + (r / a.R1) * a.s0 + (r % a.R1) * a.s1;
  T* out = static_cast<T*>(a.dlogits) + r * a.V;
  const bool any = gl != 0.f || ge != 0.f;
  const float M = a.stats[2 * r], ll = a.stats[2 * r + 1], H = any && ge != 0.f ? a.entropy[r] : 0.f;
  auto grad = [&](float x, int e) {
    const float t = max_nan(fmaf(x - M, kLog2e, -ll), kLpFloor);  // a row without a distribution stays NaN
    const float p = exp2f(t);
    const float d = -p * (gl + ge * fmaf(t, kLn2, H));
    return e == tok ? d + gl : d;
  };
  const RowView<T> src(in, a.V), dst(out, a.V);
  const bool same = src.shift == dst.shift;
  for (int v = threadIdx.x; v < dst.nvec; v += kLpThreads) {
    const int e0 = dst.first(v);
    const bool full = e0 >= 0 && e0 <= a.V - VE;
    float x[VE];
    if (any) {
      if (same) src.load(v, x);
      else
#pragma unroll
        for (int i = 0; i < VE; ++i) x[i] = e0 + i >= 0 && e0 + i < a.V ? to_f32<T>(in[e0 + i]) : -INFINITY;
    }
    uint4 u;
    T* o = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < VE; ++i) o[i] = from_f32<T>(any ? grad(x[i], e0 + i) : 0.f);
    if (full) *reinterpret_cast<uint4*>(out + e0) = u;
    else
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (e0 + i >= 0 && e0 + i < a.V) out[e0 + i] = o[i];
  }
}

cudaError_t launch_logprobs_fwd(const LogprobArgs& a, int dtype, cudaStream_t st) {
  const unsigned grid = (unsigned)(a.R0 * a.R1);
  if (dtype == 0) logprobs_fwd_kernel<bf16><<<grid, kLpThreads, 0, st>>>(a);
  else if (dtype == 1) logprobs_fwd_kernel<__half><<<grid, kLpThreads, 0, st>>>(a);
  else logprobs_fwd_kernel<float><<<grid, kLpThreads, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_logprobs_bwd(const LogprobArgs& a, int dtype, cudaStream_t st) {
  const unsigned grid = (unsigned)(a.R0 * a.R1);
  if (dtype == 0) logprobs_bwd_kernel<bf16><<<grid, kLpThreads, 0, st>>>(a);
  else if (dtype == 1) logprobs_bwd_kernel<__half><<<grid, kLpThreads, 0, st>>>(a);
  else logprobs_bwd_kernel<float><<<grid, kLpThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace lb
