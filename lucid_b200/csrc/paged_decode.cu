// Paged decoding of one new token per sequence: the LUCID step (the update of
// modeling_lucid.py:576-598 and the attention of :505-549 over the updated cache)
// and the attention alone, over a cache kept in pages.
//
// For sequence b with n cached tokens, kv head h and its gq query heads:
//   u     = sum_{t<n} exp(s k^_new . k^_t - 1/s) x_t,     x_new = bf16(v_new - u)
//   o_r   = sum_t softmax_t(s q_r . k_t) x_t              over t < n and the new token
// k^ = k / sqrt(mean(k^2) + eps).  The queries and the raw new key are the rows of one
// 16-row operand, so both sums come out of one pass over the cached rows:
//   S = A K^T (mma m16n8k16: exact bf16 products, fp32 sums), the scores scaled
//   afterwards in fp32 (softmax rows by s, the update row by s rstd_new rstd_t), and
//   acc += P X with P split into bf16 hi + lo, so that P keeps 16 bits.
// sum(k_t^2) is the diagonal of K K^T, computed by the same instruction: the B fragment
// of a key tile is also its A fragment.
//
// The cached tokens of all (sequence, kv head, row block) items are cut into tiles of
// 64 tokens; the tiles, in item order, are dealt to the CTAs in equal contiguous
// runs, so ragged batches balance whatever the lengths, which only the device
// knows.  A run's part of one item is a segment; its (max, sum, weighted sum) rows go
// to slot cta + item of the workspace (each next segment has a higher cta or item, so
// slots never collide), and the join kernel merges an item's segments in cta order:
// results do not depend on timing.
#include "serve_common.cuh"

#include <algorithm>

namespace lb {

constexpr int kPdWarps = 4, kPdThreads = 32 * kPdWarps;
constexpr int kPdTile = 16 * kPdWarps;  // tokens per tile, 16 per warp

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float2 unpack_bf16(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// cached tokens of sequence b; negative lengths mark unused places of the batch
__device__ __forceinline__ int pd_len(const PagedDecodeArgs& a, int b) {
  const int n = a.lengths[b];
  return n < 0 || (long long)n > (long long)a.M * a.ps ? 0 : n;
}
__device__ __forceinline__ int pd_tiles(int n) { return (int)(((unsigned)n + kPdTile - 1) / kPdTile); }

// tiles of the whole batch (every lane returns the sum)
__device__ __forceinline__ long long pd_total(const PagedDecodeArgs& a, int lane) {
  long long t = 0;
  for (int b = lane; b < a.B; b += 32) t += pd_tiles(pd_len(a, b));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t * a.H * a.nblk;
}

// CTAs with work: no more than tiles, so that each of them has at least one and every
// CTA from an item's first to its last holds a segment of it
__device__ __forceinline__ long long pd_ctas(const PagedDecodeArgs& a, long long T) {
  return T < a.nctas ? T : a.nctas;
}

// position in the sequence of tiles
struct PdCursor {
  int b, hb, tile, nt, n;  // sequence, h * nblk + blk, tile of the item, the item's tiles, tokens
};

__device__ __forceinline__ PdCursor pd_seek(const PagedDecodeArgs& a, long long t0, int lane) {
  PdCursor c{0, 0, 0, 0, 0};
  long long acc = 0;
  const long long per = (long long)a.H * a.nblk;
  for (int base = 0; base < a.B; base += 32) {
    const int n = base + lane < a.B ? pd_len(a, base + lane) : 0;
    const long long own = (long long)pd_tiles(n) * per;
    long long incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, acc + incl > t0);
    if (hit) {
      const int f = __ffs(hit) - 1;
      c.b = base + f;
      c.n = __shfl_sync(0xffffffffu, n, f);
      c.nt = pd_tiles(c.n);
      const long long rem = t0 - acc - __shfl_sync(0xffffffffu, incl - own, f);
      c.hb = (int)(rem / c.nt);
      c.tile = (int)(rem % c.nt);
      return c;
    }
    acc += __shfl_sync(0xffffffffu, incl, 31);
  }
  return c;
}

// the next item with at least one tile (the caller never asks past the last tile)
__device__ __forceinline__ void pd_next_item(const PagedDecodeArgs& a, PdCursor& c) {
  c.tile = 0;
  if (++c.hb == a.H * a.nblk) {
    c.hb = 0;
    do {
      ++c.b;
      c.n = c.b < a.B ? pd_len(a, c.b) : 1;
    } while (c.n == 0);
    c.nt = pd_tiles(c.n);
  }
}

// STEP: an update row behind the query rows.  R8: at most 8 rows, so rows 8-15 of the
// P operand carry the low halves of P and one mma does both.  A row's elements are cut
// into chunks of CE (16 bytes where every row is 16-byte aligned, else 8): lane j of a
// quad holds the key chunks 4 i + j (i < NK), lane group g the value chunks
// 8 c + g (c < NX); the same permutation of the inner index on both operands, and of
// the output columns, leaves the products unchanged.
template <bool STEP, bool R8, int CE, int NK, int NX>
__global__ void __launch_bounds__(kPdThreads, 2) paged_decode_kernel(const __grid_constant__ PagedDecodeArgs a) {
  constexpr int NT = NX * CE;      // 8-column output tiles
  constexpr int KR = CE / 2;       // 32-bit registers per chunk
  constexpr int KS = NK * CE / 4;  // 16-element k steps
  __shared__ float red[2][16][132];  // a warp pair's accumulator rows
  __shared__ float red_ml[kPdWarps][16][2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, j = lane & 3;
  const long long T = pd_total(a, lane);
  const long long G = pd_ctas(a, T);
  if (blockIdx.x >= G) return;
  const long long t0 = blockIdx.x * T / G, t1 = (blockIdx.x + 1) * T / G;
  PdCursor c = pd_seek(a, t0, lane);
  const float c1 = a.s * kLog2e, c2 = kLog2e / a.s, inv_d = 1.f / (float)a.D;

  for (long long t = t0; t < t1;) {
    // ---- one segment: the run's tiles of one item ----
    const int h = c.hb / a.nblk, blk = c.hb % a.nblk;
    const int r_first = blk * a.rows;                      // first query row of the block
    const int nq = min(a.gq - r_first, a.rows);            // query rows of the block
    const int upd = STEP && blk == 0 ? nq : -1;            // the update row
    const int tiles = (int)min((long long)(c.nt - c.tile), t1 - t);
    // operand A: rows g and g + 8
    uint32_t qa[KS][R8 ? 2 : 4];
    float ss = 0.f;
#pragma unroll
    for (int hf = 0; hf < (R8 ? 1 : 2); ++hf) {
      const int r = g + 8 * hf;
      const bf16* row = nullptr;
      if (r < nq) row = a.q + (long long)c.b * a.q_sb + (long long)(h * a.gq + r_first + r) * a.q_sh;
      else if (r == upd) row = a.kn + (long long)c.b * a.kn_sb + (long long)h * a.kn_sh;
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int u = 0; u < CE / 4; ++u) {
          const int e = (4 * i + j) * CE + 4 * u;
          uint2 v = make_uint2(0u, 0u);
          if (row != nullptr && e < a.D) v = *reinterpret_cast<const uint2*>(row + e);
          qa[i * (CE / 4) + u][hf] = v.x;
          qa[i * (CE / 4) + u][(R8 ? 1 : 2) + hf] = v.y;
          if (STEP && r == upd) {
            const float2 p = unpack_bf16(v.x), q2 = unpack_bf16(v.y);
            ss += p.x * p.x + p.y * p.y + q2.x * q2.x + q2.y * q2.y;
          }
        }
    }
    float rs_new = 0.f;
    if (STEP) {
      ss += __shfl_xor_sync(0xffffffffu, ss, 1);
      ss += __shfl_xor_sync(0xffffffffu, ss, 2);
      rs_new = rsqrtf(ss * inv_d + a.eps);   // meaningful in the update row's quad
    }
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[i][u] = 0.f;
    float m[2], l[2] = {0.f, 0.f};
    m[0] = STEP && g == upd ? 0.f : -INFINITY;
    m[1] = STEP && g + 8 == upd ? 0.f : -INFINITY;

    const bf16* kh = a.k.p + (long long)h * a.k.sh;
    const bf16* xh = a.x.p + (long long)h * a.x.sh;
    for (int it = 0; it < tiles; ++it) {
      const int base = (c.tile + it) * kPdTile + 16 * warp;
      if (base >= c.n) continue;             // uniform in the warp
      // page and row of token base + (lane & 15)
      const int tok = base + (lane & 15);
      int page = -1, row = 0;
      if (tok < c.n) {
        page = a.table[(long long)c.b * a.t_sb + tok / a.ps];
        row = tok % a.ps;
        if (page < 0 || page >= a.P) {
          report(a.status, kStatusPage, kTagPagedDecode);
          page = -1;
        }
      }
      // keys: operand B of both 8-key tiles
      uint32_t kr[2][NK][KR];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const int pg = __shfl_sync(0xffffffffu, page, g + 8 * kt), rw = __shfl_sync(0xffffffffu, row, g + 8 * kt);
        const bf16* p = kh + (long long)max(pg, 0) * a.k.sp + (long long)rw * a.k.sn;
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int u = 0; u < CE / 4; ++u) {
            const int e = (4 * i + j) * CE + 4 * u;
            uint2 v = make_uint2(0u, 0u);
            if (pg >= 0 && e < a.D) v = *reinterpret_cast<const uint2*>(p + e);
            kr[kt][i][2 * u] = v.x;
            kr[kt][i][2 * u + 1] = v.y;
          }
      }
      float S[2][4] = {};
      float dg[2][4] = {};
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int u = 0; u < CE / 4; ++u) {
          const int ks = i * (CE / 4) + u;
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) {
            if constexpr (R8) mma16816(S[kt], qa[ks][0], 0u, qa[ks][1], 0u, kr[kt][i][2 * u], kr[kt][i][2 * u + 1]);
            else mma16816(S[kt], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], kr[kt][i][2 * u], kr[kt][i][2 * u + 1]);
            if constexpr (STEP)
              mma16816(dg[kt], kr[0][i][2 * u], kr[1][i][2 * u], kr[0][i][2 * u + 1], kr[1][i][2 * u + 1],
                       kr[kt][i][2 * u], kr[kt][i][2 * u + 1]);
          }
        }
      // 1 / rms of this lane's four keys 2j, 2j+1, 8+2j, 9+2j: the diagonal element of
      // key q (of its tile) sits in lane 4 q + q / 2
      float rk[4] = {1.f, 1.f, 1.f, 1.f};
      if constexpr (STEP) {
        const float v0 = rsqrtf(((g & 1) ? dg[0][1] : dg[0][0]) * inv_d + a.eps);
        const float v1 = rsqrtf(((g & 1) ? dg[1][3] : dg[1][2]) * inv_d + a.eps);
        rk[0] = __shfl_sync(0xffffffffu, v0, 9 * j);
        rk[1] = __shfl_sync(0xffffffffu, v0, 9 * j + 4);
        rk[2] = __shfl_sync(0xffffffffu, v1, 9 * j);
        rk[3] = __shfl_sync(0xffffffffu, v1, 9 * j + 4);
      }
      uint32_t phi[4], plo[4];
      float al[2] = {1.f, 1.f};
#pragma unroll
      for (int hf = 0; hf < (R8 ? 1 : 2); ++hf) {
        const bool is_upd = STEP && g + 8 * hf == upd;
        float z[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float sc = S[q >> 1][2 * hf + (q & 1)];
          z[q] = is_upd ? fmaf(sc * rs_new * rk[q], c1, -c2) : sc * c1;
          if (base + 8 * (q >> 1) + 2 * j + (q & 1) >= c.n) z[q] = -INFINITY;
        }
        float mx = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = is_upd ? 0.f : fmaxf(m[hf], mx);
        const float ms = mn == -INFINITY ? 0.f : mn;
        al[hf] = exp2f(m[hf] - ms);          // 0 while nothing has been seen
        float p[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) p[q] = exp2f(z[q] - ms);
        l[hf] = l[hf] * al[hf] + ((p[0] + p[1]) + (p[2] + p[3]));
        m[hf] = mn;
        phi[2 * hf] = pack_bf16(p[0], p[1]);
        phi[2 * hf + 1] = pack_bf16(p[2], p[3]);
        const float2 h0 = unpack_bf16(phi[2 * hf]), h1 = unpack_bf16(phi[2 * hf + 1]);
        plo[2 * hf] = pack_bf16(p[0] - h0.x, p[1] - h0.y);
        plo[2 * hf + 1] = pack_bf16(p[2] - h1.x, p[3] - h1.y);
      }
      if constexpr (R8) al[1] = al[0];
      if (__any_sync(0xffffffffu, al[0] != 1.f || al[1] != 1.f)) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          acc[i][0] *= al[0];
          acc[i][1] *= al[0];
          acc[i][2] *= al[1];
          acc[i][3] *= al[1];
        }
      }
      // values: rows 2j, 2j+1, 8+2j, 9+2j, chunk 8 c + g
#pragma unroll
      for (int cx = 0; cx < NX; ++cx) {
        uint32_t xr[4][KR];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int kq = 8 * (q >> 1) + 2 * j + (q & 1);
          const int pg = __shfl_sync(0xffffffffu, page, kq), rw = __shfl_sync(0xffffffffu, row, kq);
          const bf16* p = xh + (long long)max(pg, 0) * a.x.sp + (long long)rw * a.x.sn;
#pragma unroll
          for (int u = 0; u < CE / 4; ++u) {
            const int e = (8 * cx + g) * CE + 4 * u;
            uint2 v = make_uint2(0u, 0u);
            if (pg >= 0 && e < a.D) v = *reinterpret_cast<const uint2*>(p + e);
            xr[q][2 * u] = v.x;
            xr[q][2 * u + 1] = v.y;
          }
        }
#pragma unroll
        for (int e = 0; e < CE; ++e) {
          const uint32_t sel = (e & 1) ? 0x7632u : 0x5410u;
          const uint32_t b0 = __byte_perm(xr[0][e >> 1], xr[1][e >> 1], sel);
          const uint32_t b1 = __byte_perm(xr[2][e >> 1], xr[3][e >> 1], sel);
          if constexpr (R8) {
            mma16816(acc[cx * CE + e], phi[0], plo[0], phi[1], plo[1], b0, b1);
          } else {
            mma16816(acc[cx * CE + e], phi[0], phi[2], phi[1], phi[3], b0, b1);
            mma16816(acc[cx * CE + e], plo[0], plo[2], plo[1], plo[3], b0, b1);
          }
        }
      }
    }

    // ---- the segment's rows: merge the four warps in fixed order ----
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
      l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
    }
    if constexpr (R8) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        acc[i][0] += acc[i][2];
        acc[i][1] += acc[i][3];
      }
    }
    __syncthreads();  // the previous segment's readers of red / red_ml are done
    if (j == 0) {
#pragma unroll
      for (int hf = 0; hf < (R8 ? 1 : 2); ++hf) {
        red_ml[warp][g + 8 * hf][0] = m[hf];
        red_ml[warp][g + 8 * hf][1] = l[hf];
      }
    }
    __syncthreads();
    float f[2], M[2], L[2];
#pragma unroll
    for (int hf = 0; hf < (R8 ? 1 : 2); ++hf) {
      M[hf] = -INFINITY;
#pragma unroll
      for (int w = 0; w < kPdWarps; ++w) M[hf] = fmaxf(M[hf], red_ml[w][g + 8 * hf][0]);
      const float Ms = M[hf] == -INFINITY ? 0.f : M[hf];
      L[hf] = 0.f;
#pragma unroll
      for (int w = 0; w < kPdWarps; ++w) L[hf] += exp2f(red_ml[w][g + 8 * hf][0] - Ms) * red_ml[w][g + 8 * hf][1];
      f[hf] = exp2f(m[hf] - Ms);
    }
    // (0 + 1) + (2 + 3): warps 1 and 3 store, 0 and 2 add; 2 stores, 0 adds
#pragma unroll
    for (int round = 0; round < 2; ++round) {
      const bool put = round == 0 ? (warp & 1) : warp == 2;
      const bool take = round == 0 ? !(warp & 1) : warp == 0;
      const int buf = round == 0 ? warp >> 1 : 0;
      if (round == 1) __syncthreads();  // the first round's readers are done
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int u = 0; u < (R8 ? 2 : 4); ++u) {
          const int col = ((i / CE) * 8 + 2 * j + (u & 1)) * CE + i % CE;
          if (put && col < 128) red[buf][g + 8 * (u >> 1)][col] = round == 0 ? acc[i][u] * f[u >> 1] : acc[i][u];
        }
      __syncthreads();
      if (take) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int u = 0; u < (R8 ? 2 : 4); ++u) {
            const int col = ((i / CE) * 8 + 2 * j + (u & 1)) * CE + i % CE;
            const float v = round == 0 ? acc[i][u] * f[u >> 1] : acc[i][u];
            if (col < 128) acc[i][u] = v + red[buf][g + 8 * (u >> 1)][col];
          }
      }
    }
    if (warp == 0) {
      const int nr = nq + (upd >= 0 ? 1 : 0);
      const long long item = ((long long)c.b * a.H) * a.nblk + c.hb;
      float* dst = a.part + (blockIdx.x + item) * (long long)(a.rows + (STEP ? 1 : 0)) * (a.D + 4);
#pragma unroll
      for (int hf = 0; hf < (R8 ? 1 : 2); ++hf) {
        const int r = g + 8 * hf;
        if (r >= nr) continue;
        float* d = dst + (long long)r * (a.D + 4);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int col = ((i / CE) * 8 + 2 * j + u) * CE + i % CE;
            if (col < a.D) d[col] = acc[i][2 * hf + u];
          }
        if (j == 0) {
          d[a.D] = M[hf];
          d[a.D + 1] = L[hf];
        }
      }
    }
    // ---- on to the next item ----
    t += tiles;
    c.tile += tiles;
    if (c.tile == c.nt && t < t1) pd_next_item(a, c);
  }
}

// One block of 128 threads per (sequence, kv head) and query row: merges the item's
// segments, and in the step adds the new token.
constexpr int kPdMaxCtas = 1184;

template <bool STEP>
__global__ void __launch_bounds__(128) paged_join_kernel(const __grid_constant__ PagedDecodeArgs a) {
  __shared__ float fs[kPdMaxCtas];
  __shared__ float wred[4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / a.H, h = blockIdx.x % a.H;
  const int raw = a.lengths[b];
  const bool over = (long long)raw > (long long)a.M * a.ps;
  const bool used = raw >= 0 && !over;
  if (over && tid == 0) report(a.status, kStatusLength, kTagPagedDecode);
  const int n = used ? raw : 0, nt = pd_tiles(n);
  const int pr = a.D + 4, slot_rows = a.rows + (STEP ? 1 : 0);
  // first tile of the sequence and the batch's tiles
  long long before = 0, T = 0;
  for (int i = lane; i < a.B; i += 32) {
    const int ti = pd_tiles(pd_len(a, i));
    T += ti;
    if (i < b) before += ti;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    T += __shfl_xor_sync(0xffffffffu, T, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  const long long per = (long long)a.H * a.nblk;
  T *= per;
  before *= per;
  const long long G = pd_ctas(a, T);
  auto bsum = [&](float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) wred[warp] = v;
    __syncthreads();
    return (wred[0] + wred[1]) + (wred[2] + wred[3]);
  };
  auto bmax = [&](float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if (lane == 0) wred[warp] = v;
    __syncthreads();
    return fmaxf(fmaxf(wred[0], wred[1]), fmaxf(wred[2], wred[3]));
  };
  // segments of the item (h, blk): ctas [i0, i1], slots i + item
  auto range = [&](int blk, int& i0, int& cnt, const float*& p) {
    const long long item = (long long)blockIdx.x * a.nblk + blk;
    const long long first = before + ((long long)h * a.nblk + blk) * nt, last = first + nt - 1;
    i0 = (int)(((first + 1) * G - 1) / T);
    cnt = (int)(((last + 1) * G - 1) / T) - i0 + 1;
    p = a.part + (i0 + item) * (long long)slot_rows * pr;
  };
  const int d = tid;
  float xv = 0.f, knv = 0.f;
  if constexpr (STEP) {
    float u = 0.f;
    if (nt > 0) {
      int i0, cnt;
      const float* p;
      range(0, i0, cnt, p);
      const int upd = min(a.gq, a.rows);
      if (d < a.D) {
#pragma unroll 4
        for (int i = 0; i < cnt; ++i) u += p[((long long)i * slot_rows + upd) * pr + d];
      }
    }
    bf16 xb = __float2bfloat16(0.f), kb = xb;
    if (d < a.D && used) {
      kb = a.kn[(long long)b * a.kn_sb + (long long)h * a.kn_sh + d];
      xb = __float2bfloat16(__bfloat162float(a.vn[(long long)b * a.vn_sb + (long long)h * a.vn_sh + d]) - u);
    }
    xv = __bfloat162float(xb);
    knv = __bfloat162float(kb);
    if (blockIdx.y == 0 && d < a.D) {
      a.xo[(long long)b * a.xo_sb + (long long)h * a.xo_sh + d] = xb;
      if (a.append && used) {
        const int pi = n / a.ps;
        const int page = pi < a.M ? a.table[(long long)b * a.t_sb + pi] : -1;
        if (page < 0 || page >= a.P) {
          if (d == 0) report(a.status, pi < a.M ? kStatusPage : kStatusLength, kTagPagedDecode);
        } else {
          const long long row = n % a.ps;
          a.k.p[(long long)page * a.k.sp + (long long)h * a.k.sh + row * a.k.sn + d] = kb;
          a.x.p[(long long)page * a.x.sp + (long long)h * a.x.sh + row * a.x.sn + d] = xb;
        }
      }
    }
  }
  for (int r = blockIdx.y; r < a.gq; r += gridDim.y) {
    const long long orow = (long long)b * a.o_sb + (long long)(h * a.gq + r) * a.o_sh;
    if (!used || (!STEP && nt == 0)) {   // no token to attend to
      if (d < a.D) a.o[orow + d] = __float2bfloat16(0.f);
      continue;
    }
    int i0 = 0, cnt = 0;
    const float* p = nullptr;
    if (nt > 0) range(r / a.rows, i0, cnt, p);
    const int rr = r % a.rows;
    float z = -INFINITY;
    if constexpr (STEP) {
      const float qv = d < a.D ? __bfloat162float(a.q[(long long)b * a.q_sb + (long long)(h * a.gq + r) * a.q_sh + d]) : 0.f;
      z = bsum(qv * knv) * a.s * kLog2e;
    }
    float mx = z;
    for (int i = tid; i < cnt; i += 128) mx = fmaxf(mx, p[((long long)i * slot_rows + rr) * pr + a.D]);
    const float M = bmax(mx), Ms = M == -INFINITY ? 0.f : M;
    float ls = 0.f;
    for (int i = tid; i < cnt; i += 128) {
      const float* e = p + ((long long)i * slot_rows + rr) * pr + a.D;
      const float f = exp2f(e[0] - Ms);
      fs[i] = f;
      ls += f * e[1];
    }
    float L = bsum(ls);  // its barriers also order fs
    float acc = 0.f;
    if (d < a.D) {
#pragma unroll 4
      for (int i = 0; i < cnt; ++i) acc = fmaf(fs[i], p[((long long)i * slot_rows + rr) * pr + d], acc);
    }
    if constexpr (STEP) {
      const float pn = exp2f(z - Ms);
      L += pn;
      acc = fmaf(pn, xv, acc);
    }
    if (d < a.D) a.o[orow + d] = __float2bfloat16(acc / L);
    __syncthreads();  // fs is free again
  }
}

int paged_decode_ctas() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
    cudaGetLastError();
    sms = 148;
  }
  return std::min(2 * sms, kPdMaxCtas);
}

template <bool STEP, bool R8, int CE, int NK, int NX>
static cudaError_t launch_pd(const PagedDecodeArgs& a, cudaStream_t st) {
  paged_decode_kernel<STEP, R8, CE, NK, NX><<<a.nctas, kPdThreads, 0, st>>>(a);
  return cudaGetLastError();
}

template <bool STEP, bool R8>
static cudaError_t launch_pd_d(const PagedDecodeArgs& a, cudaStream_t st) {
  const bool al16 = ((reinterpret_cast<uintptr_t>(a.k.p) | reinterpret_cast<uintptr_t>(a.x.p)) & 15u) == 0 &&
                    ((a.k.sp | a.k.sh | a.k.sn | a.x.sp | a.x.sh | a.x.sn) & 7) == 0;
  if (al16 && a.D % 8 == 0) {
    if (a.D <= 64) return launch_pd<STEP, R8, 8, 2, 1>(a, st);
    return launch_pd<STEP, R8, 8, 4, 2>(a, st);
  }
  if (a.D <= 64) return launch_pd<STEP, R8, 4, 4, 2>(a, st);
  if (a.D <= 80) return launch_pd<STEP, R8, 4, 5, 3>(a, st);
  return launch_pd<STEP, R8, 4, 8, 4>(a, st);
}

cudaError_t launch_paged_decode(const PagedDecodeArgs& a, bool step, cudaStream_t st) {
  const int rows = std::min(a.gq, a.rows) + (step ? 1 : 0);
  cudaError_t e = step ? (rows <= 8 ? launch_pd_d<true, true>(a, st) : launch_pd_d<true, false>(a, st))
                       : (rows <= 8 ? launch_pd_d<false, true>(a, st) : launch_pd_d<false, false>(a, st));
  if (e != cudaSuccess) return e;
  // one block per query row while that still fills the GPU only a few times over
  const int bh = a.B * a.H, gy = bh >= 4096 ? 1 : a.gq;
  if (step) paged_join_kernel<true><<<dim3(bh, gy), 128, 0, st>>>(a);
  else paged_join_kernel<false><<<dim3(bh, gy), 128, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace lb
