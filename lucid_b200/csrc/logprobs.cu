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
#include <atomic>
#include <climits>

namespace lb {

constexpr int kLpThreads = 512;  // backward
constexpr int kLpGroups = 128;   // groups of threads
constexpr int kLpHold = 8;       // vectors a thread holds: 32768 bf16 logits in 512 threads
constexpr int kLpBwdHold = 4;
constexpr int kLpManyRows = 900;
constexpr int kLpWarpHold = 5;   // of a warp that has a row to itself
constexpr int kLpWarpBatches = 128;
constexpr int kLpSmallTop = 24;  // up to here 32 group maxima do
constexpr float kLpFloor = -200.f;  // 2^-200 is 0 in fp32; keeps 0 * -inf out of w

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 2^v, flushed to zero below 2^-126
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// two fp32 values side by side: one instruction for both
struct Pair {
  unsigned long long v;
};
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves(Pair p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p.v));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// A type's 16-byte vector: its VE values as VE / 2 pairs, their maximum (NaN if there is
// one), the bits of -inf, and the way back from pairs.
template <typename T>
struct Vec;
template <>
struct Vec<bf16> {
  static constexpr int VE = 8;
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  static __device__ __forceinline__ float value(bf16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ Pair get(const uint4& u, int i) {
    const uint32_t w = (&u.x)[i];
    return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float top(uint32_t w) {
    return max_nan(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  // -inf and what is near it as a number so low that its weight stays 0, but for which t
  // is finite, while |m| < kNear
  static constexpr float kNear = 1e37f;
  static __device__ __forceinline__ uint4 bounded(const uint4& u) {
    constexpr uint32_t low = 0xfe96fe96u;  // -9.97e37
    return make_uint4(max2(u.x, low), max2(u.y, low), max2(u.z, low), max2(u.w, low));
  }
  static __device__ __forceinline__ uint32_t put(Pair p) {
    const float2 f = halves(p);
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  // whether either half of a vec_max reaches v, a value of the type given in both halves
  static __device__ __forceinline__ uint32_t twice(float v) { return put(pair(v, v)); }
  static __device__ __forceinline__ bool reaches(uint32_t w, uint32_t v) {
    uint32_t r;
    asm("{\n.reg .pred p, q;\nsetp.ge.bf16x2 p|q, %1, %2;\nor.pred p, p, q;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(r) : "r"(w), "r"(v));
    return r != 0;
  }
  static __device__ __forceinline__ bf16 from(float v) { return __float2bfloat16(v); }
};
template <>
struct Vec<__half> {
  static constexpr int VE = 8;
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  static __device__ __forceinline__ float value(__half v) { return __half2float(v); }
  static __device__ __forceinline__ Pair get(const uint4& u, int i) {
    const uint32_t w = (&u.x)[i];
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return pair(f.x, f.y);
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float top(uint32_t w) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return max_nan(f.x, f.y);
  }
  static constexpr float kNear = 6e4f;
  static __device__ __forceinline__ uint4 bounded(const uint4& u) {  // -65504
    constexpr uint32_t low = 0xfbfffbffu;
    return make_uint4(max2(u.x, low), max2(u.y, low), max2(u.z, low), max2(u.w, low));
  }
  static __device__ __forceinline__ uint32_t put(Pair p) {
    const float2 f = halves(p);
    const __half2 h = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t twice(float v) { return put(pair(v, v)); }
  static __device__ __forceinline__ bool reaches(uint32_t w, uint32_t v) {
    uint32_t r;
    asm("{\n.reg .pred p, q;\nsetp.ge.f16x2 p|q, %1, %2;\nor.pred p, p, q;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(r) : "r"(w), "r"(v));
    return r != 0;
  }
  static __device__ __forceinline__ __half from(float v) { return __float2half(v); }
};
template <>
struct Vec<float> {
  static constexpr int VE = 4;
  static constexpr float kNear = 0.f;
  static constexpr uint32_t kNegInf = 0xff800000u;
  static __device__ __forceinline__ float value(float v) { return v; }
  static __device__ __forceinline__ Pair get(const uint4& u, int i) {
    return pair(__uint_as_float((&u.x)[2 * i]), __uint_as_float((&u.x)[2 * i + 1]));
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ float top(uint32_t w) { return __uint_as_float(w); }
  static __device__ __forceinline__ uint32_t twice(float v) { return __float_as_uint(v); }
  static __device__ __forceinline__ bool reaches(uint32_t w, uint32_t v) { return __uint_as_float(w) >= __uint_as_float(v); }
  static __device__ __forceinline__ float from(float v) { return v; }
};
template <typename T>
__device__ __forceinline__ uint32_t vec_max(const uint4& u) {
  return Vec<T>::max2(Vec<T>::max2(u.x, u.y), Vec<T>::max2(u.z, u.w));
}

// a row as 16-byte vectors from the 16-byte boundary at or below its start: vector v
// holds the elements [v VE - shift, +VE); the first and last may be partial
template <typename T>
struct RowView {
  static constexpr int VE = Vec<T>::VE;
  const T* row;
  int V, shift, nvec;
  __device__ RowView(const T* r, int n) : row(r), V(n) {
    shift = (int)((reinterpret_cast<uintptr_t>(r) & 15u) / sizeof(T));
    nvec = (shift + n + VE - 1) / VE;
  }
  __device__ __forceinline__ int first(int v) const { return v * VE - shift; }
  // whether the vector that starts at element e0 lies inside the row
  __device__ __forceinline__ bool whole(int e0) const { return (unsigned)e0 < (unsigned)max(V - VE + 1, 0); }
  // the bits of vector v; places outside the row hold -inf
  __device__ __forceinline__ uint4 bits(int v) const {
    const int e0 = first(v);
    return whole(e0) ? *reinterpret_cast<const uint4*>(row + e0) : edge(e0);
  }
  __device__ __noinline__ uint4 edge(int e0) const {  // rare, and long where it is inlined
    uint4 u = make_uint4(Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf);
    T* p = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < VE; ++i)
      if (e0 + i >= 0 && e0 + i < V) p[i] = row[e0 + i];
    return u;
  }
};

__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
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

// This thread's vectors of the batch at v0 into its own places next[u NT]: cp.async, and
// what lies over the row's ends with -inf outside.
// Code size matters here: blocks are at different places of it, and what the
// instruction cache cannot hold they wait for.  Rare cases are loops, not unrolled.
template <typename T, int NT, int HOLD>
__device__ __forceinline__ void lp_fetch(const RowView<T> row, int v0, int tid, uint4* next) {
  constexpr int VE = RowView<T>::VE;
  const uint32_t own = (uint32_t)__cvta_generic_to_shared(next);
  const int e0 = row.first(v0 + tid);
  const T* from = row.row + e0;
  bool all = true;
#pragma unroll
  for (int u = 0; u < HOLD; ++u) {
    const bool in = row.whole(e0 + u * NT * VE);
    all = all && in;
    if (in)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(own + u * NT * 16), "l"(from + u * NT * VE) : "memory");
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  if (!all) {
#pragma unroll 1
    for (int u = 0; u < HOLD; ++u)
      if (!row.whole(e0 + u * NT * VE)) next[u * NT] = row.edge(e0 + u * NT * VE);  // -inf outside
  }
}

// (m, l, w) of a thread
struct Sums {
  float mx = -INFINITY;
  Pair l2 = pair(0.f, 0.f), w2 = pair(0.f, 0.f);

  __device__ __forceinline__ void raise(float vm) {  // to a batch with maximum vm
    if (!(vm <= mx)) {            // larger, or NaN
      const float mn = max_nan(mx, vm);
      const float d = fmaxf((mx - mn) * kLog2e, kLpFloor), f = ex2(d);  // nothing yet: f = 0
      w2 = mul2(pair(f, f), fma2(pair(d, d), l2, w2));
      l2 = mul2(pair(f, f), l2);
      mx = mn;
    }
  }

  template <typename T, int NT, int HOLD>
  __device__ __forceinline__ void add(const RowView<T>& row, const uint4 (&raw)[HOLD], int v0, int tid, float vm) {
    constexpr int VE = RowView<T>::VE;
    const Pair nm = pair(-mx, -mx), le = pair(kLog2e, kLog2e);
    if (VE == 8 && fabsf(mx) < Vec<T>::kNear) {
      if constexpr (VE == 8) {
#pragma unroll
        for (int u = 0; u < HOLD; ++u)
          if (v0 + u * NT < row.nvec) {
            const uint4 x = Vec<T>::bounded(raw[u]);
#pragma unroll
            for (int i = 0; i < VE / 2; ++i) {
              const Pair t2 = mul2(add2(Vec<T>::get(x, i), nm), le);
              const float2 t = halves(t2);
              const Pair p = pair(ex2(t.x), ex2(t.y));
              l2 = add2(l2, p);
              w2 = fma2(p, t2, w2);
            }
          }
      }
    } else if (vm != -INFINITY) {  // else nothing to add (and mx may not be finite yet)
      auto one = [&](const uint4& x) {
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) {
          const float2 t = halves(mul2(add2(Vec<T>::get(x, i), nm), le));
          const float tx = fmaxf(t.x, kLpFloor), ty = fmaxf(t.y, kLpFloor);
          const Pair p = pair(ex2(tx), ex2(ty));
          l2 = add2(l2, p);
          w2 = fma2(p, pair(tx, ty), w2);
        }
      };
      if constexpr (VE == 4) {
#pragma unroll
        for (int u = 0; u < HOLD; ++u)
          if (v0 + u * NT < row.nvec) one(raw[u]);
      } else {                     // a maximum near the type's ends: rare
#pragma unroll 1
        for (int v = v0 + tid; v < min(row.nvec, v0 + HOLD * NT); v += NT) one(row.bits(v));
      }
    }
  }

  __device__ __forceinline__ void join_warp() {  // all lanes get the warp's
    const float l = halves(l2).x + halves(l2).y, w = halves(w2).x + halves(w2).y;
    const float M = warp_max_nan(mx);
    const float d = fmaxf((mx - M) * kLog2e, kLpFloor), f = ex2(d);  // a thread without elements: l = w = 0
    l2 = pair(warp_sum_f(l * f), 0.f);
    w2 = pair(warp_sum_f(f * fmaf(d, l, w)), 0.f);
    mx = M;
  }
};

// the warp's values sorted, largest first; the k-th of them
__device__ __forceinline__ float warp_kth(float v, int lane, int k) {
#pragma unroll
  for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
    for (int o = n >> 1; o > 0; o >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, v, o);
      v = ((lane & o) == 0) == ((lane & n) == 0) ? fmaxf(v, other) : fminf(v, other);
    }
  return __shfl_sync(0xffffffffu, v, k - 1);
}

// one row's outputs but the alternatives, from its joined sums
template <typename T>
__device__ __forceinline__ void lp_write(const LogprobArgs& a, const RowView<T>& row, long long r, bool ok, float M, float ll,
                                         float ln, float W, float L) {
  const float nan = __int_as_float(0x7fc00000), H = kLn2 * (ll - W / L);
  a.entropy[r] = ok ? H : nan;
  if (a.stats != nullptr) {
    a.stats[3 * r] = ok ? M : nan;
    a.stats[3 * r + 1] = ll;
    a.stats[3 * r + 2] = H;
  }
  if (a.tokens != nullptr) {
    const long long tok = a.tokens[r];
    float lp = 0.f;
    if (tok >= 0 && tok < a.V) lp = ok ? (Vec<T>::value(row.row[tok]) - M) - ln : nan;
    else if (tok != -100) {
      report(a.status, kStatusToken, kTagLogprobs);
      lp = nan;
    }
    a.logprobs[r] = lp;
  }
}

template <int NT, bool TOP>
struct LpShared {
  static constexpr int kCap = !TOP ? 1 : NT == 128 ? 256 : 512;   // list of elements above T, and of those equal to it
  static constexpr int kHits = !TOP ? 1 : NT == 128 ? 384 : 1024;  // list of vectors that hold any
  __align__(16) float gmax[2][TOP ? kLpGroups : 1];
  int hit[kHits];
  uint4 kept[TOP && NT != 128 ? kHits : 1];                       // their bits (the short block reads them again)
  float wm[2][NT / 32], wl[2][NT / 32], ww[2][NT / 32];
  float T, M, ln;
  int nh, na, nb;
  unsigned long long above[kCap];  // (value, lowest index first) as one key
  int equal[kCap];                 // indices
  int hist[TOP ? 256 : 1];
  uint32_t prefix;
  int remain;
  int wcount[NT / 32];
};

// blocks to an SM: 64 registers a thread, 80 for the short block with alternatives
constexpr int lp_blocks(int nt, bool top) { return nt == 128 && top ? 6 : 1024 / nt; }

// Blocks stay for many rows.  While a block works on the 8 vectors that each thread holds
// in registers (a batch), cp.async brings the thread's next 8 (of this row or the next)
// into its own places in shared memory, so loads never wait for the joins.
template <typename T, int NT, bool TOP>
__global__ void __launch_bounds__(NT, lp_blocks(NT, TOP)) logprobs_fwd_kernel(const __grid_constant__ LogprobArgs a) {
  __shared__ LpShared<NT, TOP> sh;
  extern __shared__ uint4 next[];  // [kLpHold][NT]
  constexpr int VE = RowView<T>::VE, kWarps = NT / 32, kBatch = kLpHold * NT;
  constexpr int kCap = LpShared<NT, TOP>::kCap, kHits = LpShared<NT, TOP>::kHits;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const unsigned R = (unsigned)(a.R0 * a.R1), R1 = (unsigned)a.R1;
  constexpr bool kKeep = NT != 128;
  const float nan = __int_as_float(0x7fc00000);
  auto row_of = [&](unsigned r) {
    const unsigned r0 = a.R0 == 1 ? 0 : r / R1;
    return static_cast<const T*>(a.logits) + (long long)r0 * a.s0 + (long long)(r - r0 * R1) * a.s1;
  };
  const T* at = row_of(blockIdx.x);
  lp_fetch<T, NT, kLpHold>(RowView<T>(at, a.V), 0, tid, next + tid);
  // Without alternatives a row has one barrier: a warp may be at its next row while others
  // read this row's sums, which the rows therefore keep in turn.
  int turn = 0;
  for (unsigned r = blockIdx.x; r < R; r += gridDim.x, turn ^= 1) {
    const RowView<T> row(at, a.V);
    const bool multi = row.nvec > kBatch;  // else the whole row stays in registers
    const bool small = a.top <= kLpSmallTop && row.nvec >= NT;  // 32 groups do, with a vector in each
    // the maxima so far of 32 or 128 groups of neighbouring threads (which = 0: of the first batch)
    auto publish = [&](int which, float mx) {
      constexpr int kFew = NT / 32, kMany = NT / kLpGroups;
      float gm = mx;
#pragma unroll
      for (int o = 1; o < kFew; o <<= 1)
        if (small || o < kMany) gm = max_nan(gm, __shfl_xor_sync(0xffffffffu, gm, o));
      if (small) {
        if (tid % kFew == 0) sh.gmax[which][tid / kFew] = gm;
      } else {
        if (tid % kMany == 0) sh.gmax[which][tid / kMany] = gm;
      }
    };
    // after a barrier: the top-th largest of them
    auto select = [&](int which) -> float {
      if (small) {                   // every warp sorts the 32, largest first
        return warp_kth(sh.gmax[which][lane], lane, a.top);
      }
      constexpr int kTeam = NT / kLpGroups;  // NT / 128 threads rank each of 128
      const int me = tid / kTeam;
      const float v = sh.gmax[which][me];
      int rank = 0;
#pragma unroll 8
      for (int q = tid % kTeam; q < kLpGroups / 4; q += kTeam) {
        const float4 o = *reinterpret_cast<const float4*>(&sh.gmax[which][4 * q]);
        rank += (o.x > v || (o.x == v && 4 * q < me)) + (o.y > v || (o.y == v && 4 * q + 1 < me)) +
                (o.z > v || (o.z == v && 4 * q + 2 < me)) + (o.w > v || (o.w == v && 4 * q + 3 < me));
      }
#pragma unroll
      for (int o = 1; o < kTeam; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
      if (rank == a.top - 1) sh.T = v;
      __syncthreads();
      return sh.T;
    };
    auto look = [&](const uint4 (&x)[kLpHold], int v0, float t) {  // lists this thread's vectors that reach t
      const uint32_t t2 = Vec<T>::twice(t);
      if constexpr (kKeep) {
#pragma unroll
        for (int u = 0; u < kLpHold; ++u)
          if (Vec<T>::reaches(vec_max<T>(x[u]), t2) && v0 + u * NT + tid < row.nvec) {
            const int n = atomicAdd(&sh.nh, 1);
            if (n < kHits) {
              sh.hit[n] = v0 + u * NT + tid;
              sh.kept[n] = x[u];
            }
          }
      } else {
        unsigned found = 0;
#pragma unroll
        for (int u = 0; u < kLpHold; ++u) found |= Vec<T>::reaches(vec_max<T>(x[u]), t2) ? 1u << u : 0u;
#pragma unroll 1
        for (; found; found &= found - 1) {
          const int v = v0 + (__ffs(found) - 1) * NT + tid;
          if (v >= row.nvec) break;
          const int n = atomicAdd(&sh.nh, 1);
          if (n < kHits) sh.hit[n] = v;
        }
      }
    };
    if (TOP && tid == 0) sh.nh = sh.na = sh.nb = 0;

    // ---- one pass: maximum, sum, entropy sum ----
    uint4 raw[kLpHold];
    float thr = -INFINITY;
    Sums sums;
    for (int v0 = 0; v0 < row.nvec; v0 += kBatch) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
      for (int u = 0; u < kLpHold; ++u) raw[u] = next[u * NT + tid];
      const bool last = v0 + kBatch >= row.nvec;
      if (last && r + gridDim.x < R) at = row_of(r + gridDim.x);
      if (!last || r + gridDim.x < R) lp_fetch<T, NT, kLpHold>(RowView<T>(at, a.V), last ? 0 : v0 + kBatch, tid, next + tid);
      uint32_t best = vec_max<T>(raw[0]);
#pragma unroll
      for (int u = 1; u < kLpHold; ++u) best = Vec<T>::max2(best, vec_max<T>(raw[u]));
      const float vm = Vec<T>::top(best);
      sums.raise(vm);
      sums.add<T, NT, kLpHold>(row, raw, v0, tid, vm);
      // A row of several batches lists its candidates as it goes, by the first batch's
      // threshold, which the final one is not below.
      if (TOP && multi) {      // uniform
        if (v0 == 0) {
          publish(0, sums.mx);
          __syncthreads();
          thr = select(0);
        }
        look(raw, v0, thr);
      }
    }
    // ---- join the block: warps by shuffles, the rest by the first warp ----
    if constexpr (TOP) publish(1, sums.mx);
    sums.join_warp();
    if (lane == 0) {
      sh.wm[turn][warp] = sums.mx;
      sh.wl[turn][warp] = halves(sums.l2).x;
      sh.ww[turn][warp] = halves(sums.w2).x;
    }
    __syncthreads();
    if (warp == 0) {
      const float m = lane < kWarps ? sh.wm[turn][lane] : -INFINITY;
      const float M = warp_max_nan(m);
      const bool ok = fabsf(M) < INFINITY;  // else no distribution: all -inf, a NaN or +inf
      const float d = fmaxf((m - M) * kLog2e, kLpFloor), f = ex2(d);
      const float l0 = lane < kWarps ? sh.wl[turn][lane] : 0.f, w0 = lane < kWarps ? sh.ww[turn][lane] : 0.f;
      const float L = warp_sum_f(l0 * f), W = warp_sum_f(f * fmaf(d, l0, w0));
      const float ll = log2f(L), ln = logf(L);
      if (lane == 0) {
        sh.M = ok ? M : nan;
        sh.ln = ln;
        lp_write<T>(a, row, r, ok, M, ll, ln, W, L);
      }
    }
    if constexpr (TOP) {

    // ---- the top best ----
    auto put = [&](float x, int e, float t) {
      if (x > t) {
        const int n = atomicAdd(&sh.na, 1);
        if (n < kCap) sh.above[n] = (unsigned long long)order_key(x) << 32 | (0xffffffffu - (uint32_t)e);
      } else if (x == t) {
        const int n = atomicAdd(&sh.nb, 1);
        if (n < kCap) sh.equal[n] = e;
      }
    };
    // after a barrier behind the last look: the elements of the few listed vectors, or, where
    // the list was too short, all
    auto collect = [&](float t) {
      if (sh.nh > kHits && multi) {  // uniform: listed by a threshold below t, so once more by t
        __syncthreads();
        if (tid == 0) sh.nh = 0;
        __syncthreads();
#pragma unroll 1
        for (int v = tid; v < row.nvec; v += NT) {
          const uint4 x = row.bits(v);
          if (Vec<T>::reaches(vec_max<T>(x), Vec<T>::twice(t))) {
            const int n = atomicAdd(&sh.nh, 1);
            if (n < kHits) {
              sh.hit[n] = v;
              if constexpr (kKeep) sh.kept[n] = x;
            }
          }
        }
        __syncthreads();
      }
      const int nh = sh.nh;
      if (nh <= kHits) {
        for (int i = tid; i < nh; i += NT) {
          uint4 x = kKeep ? sh.kept[i] : row.bits(sh.hit[i]);
          if (!Vec<T>::reaches(vec_max<T>(x), Vec<T>::twice(t))) continue;
          const int e0 = row.first(sh.hit[i]);
#pragma unroll 1
          for (int q = 0; q < VE; ++q) {  // the first element, then the rest moved up
            const float f = halves(Vec<T>::get(x, 0)).x;
            if (f >= t && e0 + q >= 0 && e0 + q < a.V) put(f, e0 + q, t);
            x.x = __funnelshift_rc(x.x, x.y, 128 / VE);
            x.y = __funnelshift_rc(x.y, x.z, 128 / VE);
            x.z = __funnelshift_rc(x.z, x.w, 128 / VE);
            x.w = __funnelshift_rc(x.w, 0u, 128 / VE);
          }
        }
      } else {
        for (int e = tid; e < a.V; e += NT) put(Vec<T>::value(row.row[e]), e, t);
      }
      __syncthreads();
    };
    thr = select(1);
    if (!multi) {
      look(raw, 0, thr);
      __syncthreads();
    }
    collect(thr);
    const float M = sh.M, ln = sh.ln;  // the first warp's, before the barrier above
    if (!(fabsf(M) < INFINITY)) {    // uniform
      for (int i = tid; i < a.top; i += NT) {
        a.top_lp[(long long)r * a.top + i] = nan;
        a.top_tok[(long long)r * a.top + i] = -1;
      }
    } else {
    if (sh.na > kCap) {  // uniform: make the threshold the exact top-th largest value
      if (tid == 0) {
        sh.prefix = 0;
        sh.remain = a.top;
      }
      for (int byte = 3; byte >= 0; --byte) {
        __syncthreads();
        for (int i = tid; i < 256; i += NT) sh.hist[i] = 0;
        __syncthreads();
        const uint32_t pre = sh.prefix;
        for (int v = tid; v < row.nvec; v += NT) {
          const uint4 x = row.bits(v);
#pragma unroll 1
          for (int i = 0; i < VE; ++i) {
            const int e = row.first(v) + i;
            const float2 f = halves(Vec<T>::get(x, i / 2));
            const uint32_t key = order_key(i & 1 ? f.y : f.x);
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
      for (int e = tid; e < a.V; e += NT) put(Vec<T>::value(row.row[e]), e, thr);
      __syncthreads();
    }
    const int na = min(sh.na, kCap);  // fewer than that, unless somebody changes the row meanwhile
    int nb = sh.nb;
    if (nb > kCap) {  // uniform: the lowest indices equal to the threshold, by a scan in order
      const int need = max(a.top - na, 0);
      __syncthreads();
      int found = 0;
      for (int e0 = 0; e0 < a.V && found < need; e0 += NT) {
        const int e = e0 + tid;
        const bool hit = e < a.V && Vec<T>::value(row.row[e]) == thr;
        const unsigned bal = __ballot_sync(0xffffffffu, hit);
        if (lane == 0) sh.wcount[warp] = __popc(bal);
        __syncthreads();
        int at = found, all = 0;
        for (int i = 0; i < kWarps; ++i) {
          if (i < warp) at += sh.wcount[i];
          all += sh.wcount[i];
        }
        at += __popc(bal & ((1u << lane) - 1u));
        if (hit && at < need) sh.equal[at] = e;
        found += all;
        __syncthreads();
      }
      nb = need;
    }
    // rank: values above the threshold by (value, index), those equal to it by index behind
    // them; four lanes share a candidate's rivals
    for (int c = tid >> 2; c - (lane >> 2) < na + nb; c += NT / 4) {  // uniform in the warp
      const bool above = c < na;
      const unsigned long long key = above ? sh.above[c] : 0;
      const int e = above ? (int)(0xffffffffu - (uint32_t)key) : c < na + nb ? sh.equal[c - na] : 0;
      int rank = 0;
      if (above) {
        for (int q = tid & 3; q < na; q += 4) rank += sh.above[q] > key;
      } else {
        for (int q = tid & 3; q < nb; q += 4) rank += sh.equal[q] < e;
      }
      rank += __shfl_xor_sync(0xffffffffu, rank, 1);
      rank += __shfl_xor_sync(0xffffffffu, rank, 2);
      if (!above) rank += na;
      if ((tid & 3) == 0 && c < na + nb && rank < a.top) {
        a.top_lp[(long long)r * a.top + rank] = ((above ? key_value((uint32_t)(key >> 32)) : thr) - M) - ln;
        a.top_tok[(long long)r * a.top + rank] = e;
      }
    }
    }
    __syncthreads();                 // the lists are free for the next row
    }
  }
}

// Many rows with up to kLpSmallTop alternatives: a warp (a block of 32 threads) to a row,
// without any barrier.  The lanes' maxima are the groups; their top-th largest is taken
// anew whenever the batches seen have doubled.  What is listed meanwhile is a lane's whole
// batch with its maximum, where that reaches the threshold: one test for 40 elements, and
// the final threshold drops most of the list (about 140 of a row of 25 batches, with 20
// alternatives) without a look at its elements.
// 8190 rows of 32000 bf16, 20 best: 120 us with 28 warps of 5 vectors a thread to an SM, 125
// with 24 of 8 or 28 of 4.  What bounds it: issue slots are busy 63 % of the time; 4.4 TB/s of
// logits, 4.9 with the second look at the listed batches; of the 8.9 cycles that a warp takes for an instruction 2.1 are fixed latency, 1.1
// loads, 2.0 shuffles and shared memory, 1.7 other warps' turns.
constexpr int kLpWarpBlocks = 28;
constexpr int kLpWarpHits = 320;
constexpr int kLpWarpCap = 192;  // (kLpSmallTop - 1) vectors, with lanes without one
struct LpWarpShared {
  uint4 next[kLpWarpHold * 32];
  union {
    float most[kLpWarpHits];     // a listed batch's maximum, then
    int hit[kLpWarpHits];        // the vectors that reach the final threshold
  };
  union {
    unsigned long long best[kLpWarpCap];  // elements, (value, lowest index first) as one key
    int hist[256];
  };
  int equal[kLpWarpCap];
  unsigned short from[kLpWarpHits];  // batch and lane
};

template <typename T>
__global__ void __launch_bounds__(32, kLpWarpBlocks) logprobs_warp_kernel(const __grid_constant__ LogprobArgs a) {
  __shared__ __align__(16) LpWarpShared sh;
  constexpr int VE = RowView<T>::VE, kBatch = kLpWarpHold * 32;
  const int lane = threadIdx.x;
  const unsigned below = (1u << lane) - 1u;
  const unsigned R = (unsigned)(a.R0 * a.R1), R1 = (unsigned)a.R1;
  auto row_of = [&](unsigned r) {
    const unsigned r0 = a.R0 == 1 ? 0 : r / R1;
    return static_cast<const T*>(a.logits) + (long long)r0 * a.s0 + (long long)(r - r0 * R1) * a.s1;
  };
  const T* at = row_of(blockIdx.x);
  lp_fetch<T, 32, kLpWarpHold>(RowView<T>(at, a.V), 0, lane, sh.next + lane);
  for (unsigned r = blockIdx.x; r < R; r += gridDim.x) {
    const RowView<T> row(at, a.V);
    float thr = -INFINITY;
    int nh = 0;                        // uniform, as the other counts below
    bool fresh = false;
    Sums sums;
    for (int v0 = 0, batch = 0; v0 < row.nvec; v0 += kBatch) {
      uint4 raw[kLpWarpHold];
      asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
      for (int u = 0; u < kLpWarpHold; ++u) raw[u] = sh.next[u * 32 + lane];
      const bool last = v0 + kBatch >= row.nvec;
      if (last && r + gridDim.x < R) at = row_of(r + gridDim.x);
      if (!last || r + gridDim.x < R) lp_fetch<T, 32, kLpWarpHold>(RowView<T>(at, a.V), last ? 0 : v0 + kBatch, lane, sh.next + lane);
      uint32_t best = vec_max<T>(raw[0]);
#pragma unroll
      for (int u = 1; u < kLpWarpHold; ++u) best = Vec<T>::max2(best, vec_max<T>(raw[u]));
      const float vm = Vec<T>::top(best);
      sums.raise(vm);
      const int id = batch++ * 32 + lane;
      fresh = (batch & (batch - 1)) == 0;
      if (fresh) thr = warp_kth(sums.mx, lane, a.top);
      const unsigned some = __ballot_sync(0xffffffffu, vm >= thr);
      const int n = nh + __popc(some & below);
      if (vm >= thr && n < kLpWarpHits) {
        sh.from[n] = (unsigned short)id;
        sh.most[n] = vm;
      }
      nh += __popc(some);
      sums.add<T, 32, kLpWarpHold>(row, raw, v0, lane, vm);
    }
    const float mine = sums.mx;
    sums.join_warp();
    const float M = sums.mx, L = halves(sums.l2).x, ll = log2f(L), ln = logf(L);
    const bool ok = fabsf(M) < INFINITY;  // else no distribution: all -inf, a NaN or +inf
    if (lane == 0) lp_write<T>(a, row, r, ok, M, ll, ln, halves(sums.w2).x, L);
    if (!ok) {
      for (int i = lane; i < a.top; i += 32) {
        a.top_lp[(long long)r * a.top + i] = __int_as_float(0x7fc00000);
        a.top_tok[(long long)r * a.top + i] = -1;
      }
      continue;
    }
    // ---- the listed batches that reach the final threshold ----
    if (!fresh) thr = warp_kth(mine, lane, a.top);
    const bool over = nh > kLpWarpHits;  // too many: every vector is looked at
    __syncwarp();
    if (!over) {
      const int listed = nh;
      nh = 0;
#pragma unroll 1
      for (int i = lane; i - lane < listed; i += 32) {
        const bool in = i < listed && sh.most[i] >= thr;
        const int id = i < listed ? sh.from[i] : 0;
        const unsigned some = __ballot_sync(0xffffffffu, in);
        __syncwarp();
        if (in) sh.from[nh + __popc(some & below)] = (unsigned short)id;  // at or before i: read already
        nh += __popc(some);
      }
      __syncwarp();
    }
    // ---- their vectors that do ----
    const uint32_t t2 = Vec<T>::twice(thr);
    const int looks = over ? row.nvec : nh * kLpWarpHold;
    int nv = 0;
    auto vector = [&](int i) {
      if (over) return i;
      const int id = sh.from[i / kLpWarpHold];
      return (id >> 5) * kBatch + i % kLpWarpHold * 32 + (id & 31);
    };
#pragma unroll 1
    for (int i = lane; i - lane < looks; i += 32 * 4) {
      uint4 x[4];
      int v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = i + 32 * k < looks ? vector(i + 32 * k) : row.nvec;
        x[k] = make_uint4(0u, 0u, 0u, 0u);
        if (v[k] < row.nvec) x[k] = row.bits(v[k]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool hit = v[k] < row.nvec && Vec<T>::reaches(vec_max<T>(x[k]), t2);
        const unsigned some = __ballot_sync(0xffffffffu, hit);
        const int n = nv + __popc(some & below);
        if (hit && n < kLpWarpHits) sh.hit[n] = v[k];
        nv += __popc(some);
      }
    }
    __syncwarp();
    // ---- and their elements: (value, index) in sh.best ----
    auto key_of = [](float x, int e) { return (unsigned long long)order_key(x) << 32 | (0xffffffffu - (uint32_t)e); };
    int na = 0, nb = 0;
    if (nv <= kLpWarpHits) {
#pragma unroll 1
      for (int i = lane; i - lane < nv * VE; i += 32) {
        const int e = row.first(i < nv * VE ? sh.hit[i / VE] : 0) + i % VE;
        const bool in = i < nv * VE && e >= 0 && e < a.V;
        const float x = in ? Vec<T>::value(row.row[e]) : -INFINITY;
        const unsigned some = __ballot_sync(0xffffffffu, in && x >= thr);
        const int n = na + __popc(some & below);
        if (in && x >= thr && n < kLpWarpCap) sh.best[n] = key_of(x, e);
        na += __popc(some);
      }
    }
    if (nv > kLpWarpHits || na > kLpWarpCap) {  // by scans in order, those equal to the threshold apart
      auto scan = [&]() {
        na = nb = 0;
        __syncwarp();
#pragma unroll 1
        for (int e = lane; e - lane < a.V; e += 32) {
          const float x = e < a.V ? Vec<T>::value(row.row[e]) : -INFINITY;
          const bool above = e < a.V && x > thr, equal = e < a.V && x == thr;
          const unsigned sa = __ballot_sync(0xffffffffu, above), se = __ballot_sync(0xffffffffu, equal);
          const int pa = na + __popc(sa & below), pe = nb + __popc(se & below);
          if (above && pa < kLpWarpCap) sh.best[pa] = key_of(x, e);
          if (equal && pe < kLpWarpCap) sh.equal[pe] = e;  // the lowest indices
          na += __popc(sa);
          nb += __popc(se);
        }
      };
      scan();
      if (na > kLpWarpCap) {  // make the threshold the exact top-th largest value
        uint32_t prefix = 0;
        int remain = a.top;
        for (int byte = 3; byte >= 0; --byte) {
          __syncwarp();
          for (int i = lane; i < 256; i += 32) sh.hist[i] = 0;
          __syncwarp();
#pragma unroll 1
          for (int e = lane; e < a.V; e += 32) {
            const uint32_t key = order_key(Vec<T>::value(row.row[e]));
            if (byte == 3 || (key >> (8 * byte + 8)) == prefix) atomicAdd(&sh.hist[(key >> (8 * byte)) & 255], 1);
          }
          __syncwarp();
          int d = 255;
          while (d > 0 && sh.hist[d] < remain) remain -= sh.hist[d--];
          prefix = (prefix << 8) | (uint32_t)d;
        }
        thr = key_value(prefix);
        scan();
      }
      na = min(na, kLpWarpCap);
      nb = min(nb, kLpWarpCap);
    }
    __syncwarp();
    // ---- ranks, as above ----
    for (int c = lane; c < na + nb; c += 32) {
      const bool above = c < na;
      const unsigned long long key = above ? sh.best[c] : 0;
      const int e = above ? (int)(0xffffffffu - (uint32_t)key) : sh.equal[c - na];
      int rank = 0;
      if (above) {
        for (int q = 0; q < na; ++q) rank += sh.best[q] > key;
      } else {
        rank = na;
        for (int q = 0; q < nb; ++q) rank += sh.equal[q] < e;
      }
      if (rank < a.top) {
        a.top_lp[(long long)r * a.top + rank] = ((above ? key_value((uint32_t)(key >> 32)) : thr) - M) - ln;
        a.top_tok[(long long)r * a.top + rank] = e;
      }
    }
    __syncwarp();                      // the lists are free for the next row
  }
}

// d x_i = g_lp (1[i = tok] - p_i) - g_ent p_i (log p_i + H).  Rows with both factors 0
// (a masked token, say) are written as zeros without being read.
template <typename T>
__global__ void __launch_bounds__(kLpThreads, 3) logprobs_bwd_kernel(const __grid_constant__ LogprobArgs a) {
  constexpr int VE = RowView<T>::VE;
  const long long r = blockIdx.x;
  const long long tk = a.tokens != nullptr ? a.tokens[r] : -100;
  const bool given = tk >= 0 && tk < a.V;
  const int tok = given ? (int)tk : INT_MIN;                 // anything else has no element
  float gl = a.g_lp != nullptr && tk != -100 ? a.g_lp[r] : 0.f;
  if (!given && gl != 0.f) gl = __int_as_float(0x7fc00000);  // like the log probability
  const float ge = a.g_ent != nullptr ? a.g_ent[r] : 0.f;
  const T* in = static_cast<const T*>(a.logits) + (r / a.R1) * a.s0 + (r % a.R1) * a.s1;
  T* out = static_cast<T*>(a.dlogits) + r * a.V;
  const RowView<T> src(in, a.V), dst(out, a.V);
  if (gl == 0.f && ge == 0.f) {
    for (int v = threadIdx.x; v < dst.nvec; v += kLpThreads) {
      const int e0 = dst.first(v);
      if (dst.whole(e0)) *reinterpret_cast<uint4*>(out + e0) = make_uint4(0u, 0u, 0u, 0u);
      else
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if (e0 + i >= 0 && e0 + i < a.V) out[e0 + i] = Vec<T>::from(0.f);
    }
    return;
  }
  const float M = a.stats[3 * r], ll = a.stats[3 * r + 1];
  // -p (gl + ge (ln 2 t + H)) = p (c0 + c1 t), t = log2 p
  const float c0 = ge != 0.f ? -(gl + ge * a.stats[3 * r + 2]) : -gl, c1 = -ge * kLn2;
  const Pair nm = pair(-M, -M), nl = pair(-ll, -ll), le = pair(kLog2e, kLog2e), k0 = pair(c0, c0), k1 = pair(c1, c1);
  auto grad = [&](Pair x) {
    const float2 t = halves(fma2(add2(x, nm), le, nl));
    const float tx = max_nan(t.x, kLpFloor), ty = max_nan(t.y, kLpFloor);  // a row without a distribution stays NaN
    return mul2(pair(ex2(tx), ex2(ty)), fma2(k1, pair(tx, ty), k0));
  };
  auto one = [&](float x) { return halves(grad(pair(x, x))).x; };
  if (src.shift == dst.shift) {  // both rows are vectors at the same places
    for (int v0 = threadIdx.x; v0 < dst.nvec; v0 += kLpBwdHold * kLpThreads) {
      uint4 raw[kLpBwdHold];
#pragma unroll
      for (int u = 0; u < kLpBwdHold; ++u)
        if (v0 + u * kLpThreads < dst.nvec) raw[u] = src.bits(v0 + u * kLpThreads);
#pragma unroll
      for (int u = 0; u < kLpBwdHold; ++u) {
        const int v = v0 + u * kLpThreads;
        if (v >= dst.nvec) break;
        const int e0 = dst.first(v);
        uint4 y;
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) {
          const Pair d = grad(Vec<T>::get(raw[u], i));
          if constexpr (VE == 8) {
            (&y.x)[i] = Vec<T>::put(d);
          } else {
            (&y.x)[2 * i] = __float_as_uint(halves(d).x);
            (&y.x)[2 * i + 1] = __float_as_uint(halves(d).y);
          }
        }
        if (dst.whole(e0)) *reinterpret_cast<uint4*>(out + e0) = y;
        else
#pragma unroll
          for (int i = 0; i < VE; ++i)
            if (e0 + i >= 0 && e0 + i < a.V) out[e0 + i] = reinterpret_cast<const T*>(&y)[i];
        // the given token's element gets gl too (this thread has just stored it)
        if (tok >= e0 && tok < e0 + VE) out[tok] = Vec<T>::from(one(Vec<T>::value(in[tok])) + gl);
      }
    }
  } else {
    for (int e = threadIdx.x; e < a.V; e += kLpThreads) {
      const float d = one(Vec<T>::value(in[e]));
      out[e] = Vec<T>::from(e == tok ? d + gl : d);
    }
  }
}

template <typename T, int NT, bool TOP>
static cudaError_t launch_fwd(const LogprobArgs& a, cudaStream_t st) {
  constexpr int smem = kLpHold * NT * 16, kDevices = 64;
  static std::atomic<int> known[kDevices];  // the device's SMs, once its shared memory is granted
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < kDevices) sms = known[dev].load(std::memory_order_relaxed);
  if (sms == 0) {
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(logprobs_fwd_kernel<T, NT, TOP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev < kDevices) known[dev].store(sms, std::memory_order_relaxed);
  }
  const long long rows = a.R0 * a.R1;
  const unsigned grid = (unsigned)std::min<long long>(rows, (long long)sms * lp_blocks(NT, TOP));
  logprobs_fwd_kernel<T, NT, TOP><<<grid, NT, smem, st>>>(a);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_warp(const LogprobArgs& a, cudaStream_t st) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices];
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < kDevices) sms = known[dev].load(std::memory_order_relaxed);
  if (sms == 0) {
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    if (dev < kDevices) known[dev].store(sms, std::memory_order_relaxed);
  }
  const unsigned grid = (unsigned)std::min<long long>(a.R0 * a.R1, (long long)sms * kLpWarpBlocks);
  logprobs_warp_kernel<T><<<grid, 32, 0, st>>>(a);
  return cudaGetLastError();
}

// Without alternatives.  Many rows, or short ones: 128 threads a row, 8 rows to an SM, whose
// joins hide behind one another (8190 rows of 32000 bf16: 98 us, with 512 threads 125).  Few
// rows: 512 threads a row, for the latency (900 rows: equal).
//
// With up to 24 alternatives a warp a row, once there are rows enough to hide that a warp
// needs 10 us and 4 more per 1000 vectors for its row.  20 best, bf16, us with a warp / 128 /
// 512 threads:
//   8190 x 32000   120 / 173 / 230      1200 x 32000    33 /  38 / 39      600 x 32000   29 / 25 / 25
//   4100 x 128000  200 / 640 / 270      1200 x 128000  101 / 263 / 87      600 x 16000   21 / 15 / 25
//   9000 x 2000     31 /  82 / 290       600 x 2000     10 /  10 / 27      150 x 2000     9 /  8 / 12
// fp32, where a row has twice the vectors, crosses at the same counts of them:
//   1800 x 32000    56 /  84 /  64      1200 x 32000    47 /  69 / 45       900 x 2000    12 / 14 / 27
//   2600 x 65000   119 / 411 / 133      1800 x 65000    95 / 336 / 94       600 x 2000    11 /  8 / 21
// so from 900 rows and one more for every 16 vectors of a row, or 300 where a row is two
// batches; but to 128 batches a row, whose list the doublings still fit (2500 x 160000: 183 /
// 605 / 211; 4200 x 200000, which it does not always: 478 / 1232 / 438).  Below that 128 threads
// where the rows are at least 150 for each of their batches, of which four at most (the
// first one sets the threshold for the lists: 900 x 65000: 68 and with 512 threads 49), else 512.
// More alternatives than the 32 groups serve: 512 threads (50 best of 8190 x 32000: 305 with 128
// threads and 261), but for a row of one batch (900 x 500: 86 with 512, 17 with 128).
template <typename T>
static cudaError_t launch_fwd_t(const LogprobArgs& a, cudaStream_t st) {
  constexpr int VE = RowView<T>::VE, kShort = kLpHold * 128 * VE;  // a batch of 128 threads
  const long long rows = a.R0 * a.R1;
  if (a.top == 0)
    return a.V <= kShort || rows >= kLpManyRows ? launch_fwd<T, 128, false>(a, st) : launch_fwd<T, 512, false>(a, st);
  if (a.top <= kLpSmallTop && a.V <= kLpWarpBatches * kLpWarpHold * 32 * VE &&
      rows >= (a.V <= 2 * kLpWarpHold * 32 * VE ? 300 : kLpManyRows + a.V / VE / 16))
    return launch_warp<T>(a, st);
  const bool narrow = a.V <= kShort || (a.top <= kLpSmallTop && a.V <= 4 * kShort && rows * kShort >= 150LL * a.V);
  return narrow ? launch_fwd<T, 128, true>(a, st) : launch_fwd<T, 512, true>(a, st);
}

cudaError_t launch_logprobs_fwd(const LogprobArgs& a, int dtype, cudaStream_t st) {
  return dtype == 0 ? launch_fwd_t<bf16>(a, st) : dtype == 1 ? launch_fwd_t<__half>(a, st) : launch_fwd_t<float>(a, st);
}

cudaError_t launch_logprobs_bwd(const LogprobArgs& a, int dtype, cudaStream_t st) {
  const unsigned grid = (unsigned)(a.R0 * a.R1);
  if (dtype == 0) logprobs_bwd_kernel<bf16><<<grid, kLpThreads, 0, st>>>(a);
  else if (dtype == 1) logprobs_bwd_kernel<__half><<<grid, kLpThreads, 0, st>>>(a);
  else logprobs_bwd_kernel<float><<<grid, kLpThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace lb
