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
//   acc += P X with P split into three bf16 parts, which hold all 24 bits of an fp32
//   weight, so the products are exact.  A tile's are summed from zero by the MMAs, then added
//   to the row's sums: an MMA cuts its result off instead of rounding it, which over the
//   148 tiles of a CTA at 4 x 32765 tokens left 70 of 32768 results on the other side of a bf16
//   rounding than the exact ones, now 2.  (Two parts, 16 bits: 46.  Time on one GPU, 24
//   ragged sequences with 8 query heads per kv head / 4 x 32765 tokens with one: 31.3 / 338 us
//   a pass with the sums left to the MMAs, 32.5 / 341 as it is, 31.2 / 335 with two parts.)
// sum(k_t^2) is the diagonal of K K^T, computed by the same instructions: the B fragment
// of a key tile is also its A fragment, and with at most 8 query rows it rides in the
// rows of A that S leaves empty.
//
// The cached tokens of all (sequence, kv head, row block) items are cut into tiles of
// 64 tokens; the tiles, in item order, are dealt to the CTAs in equal contiguous
// runs, so ragged batches balance whatever the lengths, which only the device
// knows.  A run's part of one item is a segment; its (max, sum, weighted sum) rows go
// to slot cta + item of the workspace (each next segment has a higher cta or item, so
// slots never collide), and the join kernel merges an item's segments in cta order:
// results do not depend on timing.
//
// The products are mma.sync's: a kv head brings 1 to 16 rows a step, where a tcgen05 tile
// has 64 or more and would hand its scores back through tensor memory for the softmax.
// HBM bounds the pass (4 x 32765 tokens, 32 heads of 128: 2.15 GB in 333 to 349 us a call
// in runs of different length, 6.2 to 6.5 TB/s); over 4 x 8189 tokens the tensor pipe is active 30 % of it.
#include "paged_flat.h"
#include "serve_common.cuh"

#include <algorithm>
#include <atomic>

namespace lb {

constexpr int kPdWarps = 4, kPdThreads = 32 * kPdWarps;
constexpr int kPdTile = 16 * kPdWarps;  // tokens per tile, 16 per warp
constexpr float kPdSlack = 8.f;         // log2 units
constexpr int kPdItemCost = 2;          // tiles

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the same from zero
__device__ __forceinline__ void mma16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// two rounded sums in one instruction
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
  asm("{\n.reg .b64 s, t;\nmov.b64 s, {%0, %1};\nmov.b64 t, {%2, %3};\nadd.rn.f32x2 s, s, t;\nmov.b64 {%0, %1}, s;\n}"
      : "+f"(x), "+f"(y) : "f"(a), "f"(b));
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float2 unpack_bf16(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// 2^v; results below 2^-126 flush to zero, which nothing here can tell from a weight of 0
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// CB bytes from global to shared memory, the bytes at and past `bytes` zero and unread
template <int CB>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, int bytes) {
  if constexpr (CB == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// cached tokens of sequence b; negative lengths mark unused places of the batch
__device__ __forceinline__ int pd_len(const PagedDecodeArgs& a, int b) {
  const int n = a.lengths[b];
  return n < 0 || (long long)n > (long long)a.M * a.ps ? 0 : n;
}
__device__ __forceinline__ int pd_tiles(int n) { return (int)(((unsigned)n + kPdTile - 1) / kPdTile); }

// An item counts as its tiles and kPdItemCost more in front of them, about what its
// queries' loads and its merge of the warps cost: batches with many short sequences would
// otherwise give some CTAs a dozen items and others none.  24 sequences of 4 to 6007 tokens
// (4 kv heads of 68): 37.7 us without, 30.2, 25.6 and 26.6 us with 1, 2 and 4; the attention of
// 48 sequences of 0 to 8150 tokens (4 of 128): 52.8, 48.1, 47.5 and 48.2 us.
__device__ __forceinline__ int pd_units(int n) { return n > 0 ? pd_tiles(n) + kPdItemCost : 0; }

// units of the whole batch (every lane returns the sum)
__device__ __forceinline__ long long pd_total(const PagedDecodeArgs& a, int lane) {
  long long t = 0;
  for (int b = lane; b < a.B; b += 32) t += pd_units(pd_len(a, b));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t * a.H * a.nblk;
}

// CTAs with a share: no more than units, so that each of them has at least one and every
// CTA from the one of an item's first tile to that of its last holds a segment of it
__device__ __forceinline__ long long pd_ctas(const PagedDecodeArgs& a, long long T) {
  return T < a.nctas ? T : a.nctas;
}

// a / b for nonnegative a and positive b; nearly always both fit 32 bits, where the
// division is several times shorter
__device__ __forceinline__ long long pd_div(long long a, long long b) {
  if (((a | b) >> 32) == 0) return (unsigned)a / (unsigned)b;
  return a / b;
}

// position in the sequence of units
struct PdCursor {
  int b, hb, tile, nt, n;  // sequence, h * nblk + blk, tile of the item (negative: units before
};                         // the first), the item's tiles, tokens

// spends the units in front of an item's first tile; `left` may come to 0
__device__ __forceinline__ void pd_enter(PdCursor& c, int& left) {
  const int k = max(0, min(-c.tile, left));
  c.tile += k;
  left -= k;
}

__device__ __forceinline__ PdCursor pd_seek(const PagedDecodeArgs& a, long long t0, int lane) {
  PdCursor c{0, 0, 0, 0, 0};
  long long acc = 0;
  const long long per = (long long)a.H * a.nblk;
  for (int base = 0; base < a.B; base += 32) {
    const int n = base + lane < a.B ? pd_len(a, base + lane) : 0;
    const long long own = (long long)pd_units(n) * per;
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
      c.hb = (int)pd_div(rem, c.nt + kPdItemCost);
      c.tile = (int)(rem - (long long)c.hb * (c.nt + kPdItemCost)) - kPdItemCost;
      return c;
    }
    acc += __shfl_sync(0xffffffffu, incl, 31);
  }
  c.b = a.B;
  return c;
}

// the next item with at least one tile; `left` becomes 0 behind the last sequence, which a
// CTA with units left reaches only if somebody changes the lengths meanwhile
__device__ __forceinline__ void pd_next_item(const PagedDecodeArgs& a, PdCursor& c, int& left) {
  c.tile = -kPdItemCost;
  if (++c.hb == a.H * a.nblk) {
    c.hb = 0;
    do {
      if (++c.b >= a.B) {
        left = 0;
        return;
      }
      c.n = pd_len(a, c.b);
    } while (c.n == 0);
    c.nt = pd_tiles(c.n);
  }
  pd_enter(c, left);
}

template <int KR>
__device__ __forceinline__ void load_chunk(const unsigned char* p, uint32_t (&r)[KR]) {
  if constexpr (KR == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    r[0] = v.x; r[1] = v.y;
  }
}

// Shared-memory rows: 16 tokens of each pool per warp and stage, RB bytes each (128 up to
// D = 64, else 256), a chunk's place in its row swizzled so that the fragment reads below
// are free of bank conflicts (8 lanes read 16-byte, 16 lanes 8-byte chunks at a time: key
// reads take chunks 4 i + j of rows g; 16-byte value chunks are read by ldmatrix, 8 rows of
// one chunk at a time, 8-byte ones as chunks 8 c + g of rows 2 j + const).
template <int CE>
__device__ __forceinline__ int pd_kswz(int row) { return CE == 8 ? (row & 1) * 4 : (row & 3) * 4; }
template <int CE>
__device__ __forceinline__ int pd_xswz(int row) { return CE == 8 ? row & 7 : ((row >> 1) & 3) * 4; }

// B fragments (16 tokens x 8 columns) of two 8-column tiles from rows of values
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// How rows reach shared memory.  kRows: any strides, row by row.  kFull: rows of exactly
// the fragments' width, the same with constant places.  kFlat: rows that follow one another
// in pages of a multiple of 16 tokens but start on 8-byte boundaries only (an odd multiple
// of 4 elements): the 16 tokens are one run of bytes, copied 16 at a time as it is (5
// copies per lane and pool at D = 68 instead of 9), whose reads conflict up to 4-way.
enum : int { kRows = 0, kFull = 1, kFlat = 2 };

// Three CTAs of four warps per SM where the registers allow (at most 168 a thread): the
// tile loop is a chain of short dependent steps.  24 ragged sequences at D = 68 take 28.3 us
// with two CTAs and 25.6 with three; at D = 128, with three stages for two CTAs and two for
// three, 24 ragged sequences with 16 heads on 8 take 51.5 and 47.6, 4 x 32K tokens with 32 heads
// 326 and 338 in a short run, 355 and 339 under the power cap.  16 rows at D > 96, and the addresses of odd rows at D > 64, need more registers.
template <bool R8, int CE, int NK, int NX, int MODE>
struct PdShape {
  static constexpr int kCols = NX * 8 * CE;                 // columns covered
  static constexpr int kRowBytes = MODE == kFlat ? 0 : kCols <= 64 ? 128 : 256;
  static constexpr int kPool = MODE == kFlat ? 32 * flat_most_d(NK) : 16 * kRowBytes;  // bytes of a pool in a stage, at most
  static constexpr int kCtas = kCols <= 64 || MODE != kRows && (R8 || kCols <= 96) ? 3 : 2;
  static constexpr int kStages = kCtas == 2 || kPool <= 2560 ? 3 : 2;
  // reads of the columns past D may run up to 192 bytes past a flat run
  static constexpr int kSmem = kPdWarps * kStages * 2 * kPool + (MODE == kFlat ? 256 : 0);
};

// The rows stream through a ring of stages per warp, filled by cp.async across
// item borders: consecutive lanes copy consecutive chunks, so whole rows are requested at
// once.  Page numbers are looked up one tile before their copies are issued.
//
// STEP: an update row behind the query rows.  R8: at most 8 rows, so rows 8-15 of the
// P operand carry the second parts of P and one mma does both.  A row's elements are cut
// into chunks of CE (16 bytes where every row is 16-byte aligned, else 8): lane j of a
// quad holds the key chunks 4 i + j (i < NK), lane group g the value chunks
// 8 c + g (c < NX); the same permutation of the inner index on both operands, and of
// the output columns, leaves the products unchanged.
template <bool STEP, bool R8, int CE, int NK, int NX, int MODE>
__global__ void __launch_bounds__(kPdThreads, PdShape<R8, CE, NK, NX, MODE>::kCtas) paged_decode_kernel(const __grid_constant__ PagedDecodeArgs a) {
  constexpr int NT = NX * CE;      // 8-column output tiles
  constexpr int KR = CE / 2;       // 32-bit registers per chunk
  constexpr int KS = NK * CE / 4;  // 16-element k steps
  using Shape = PdShape<R8, CE, NK, NX, MODE>;
  constexpr int CB = CE * 2, RB = Shape::kRowBytes, POOL = Shape::kPool, STAGE = 2 * POOL, STAGES = Shape::kStages;
  constexpr int NU = MODE == kFull ? RB / CB / 2 : MODE == kRows ? (NK * 4 + 1) / 2 : flat_copies(NK);  // copies per lane and pool
  extern __shared__ __align__(16) unsigned char ring[];  // [warp][stage][pool]: 16 tokens
  __shared__ float red[2][R8 ? 8 : 16][132];  // a warp pair's accumulator rows
  __shared__ float red_ml[kPdWarps][16][2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, j = lane & 3;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const long long T = pd_total(a, lane);
  const long long G = pd_ctas(a, T);
  if (blockIdx.x >= G) return;
  const long long t0 = pd_div(blockIdx.x * T, G);
  int left = (int)(pd_div((blockIdx.x + 1) * T, G) - t0);  // units of this CTA
  PdCursor c = pd_seek(a, t0, lane);
  if (c.b >= a.B) return;        // the lengths have just changed
  pd_enter(c, left);
  const float c1 = a.s * kLog2e, c2 = kLog2e / a.s, inv_d = 1.f / (float)a.D;
  unsigned char* own = ring + warp * (STAGES * STAGE);
  const uint32_t own_s = (uint32_t)__cvta_generic_to_shared(own);

  // ---- the producer's side: cursor `pc` runs ahead of `c` ----
  PdCursor pc = c;
  int ahead = left;              // units from the tile whose offsets are in (koff, xoff)
  int ph = pc.hb / a.nblk;       // its kv head
  long long koff = 0, xoff = 0;  // element offsets of the row of token 16 warp + (lane & 15)
  auto look_up = [&]() {
    const int tok = pc.tile * kPdTile + 16 * warp + (lane & 15);
    if (ahead > 0 && tok < pc.n) {
      const int pi = a.ps_shift >= 0 ? tok >> a.ps_shift : tok / a.ps, row = tok - pi * a.ps;
      int page = a.table[(long long)pc.b * a.t_sb + pi];
      if (page < 0 || page >= a.P) {
        report(a.status, kStatusPage, kTagPagedDecode);
        page = 0;
      }
      koff = page * a.k.sp + ph * a.k.sh + row * a.k.sn;
      xoff = page * a.x.sp + ph * a.x.sh + row * a.x.sn;
    }
  };
  // this lane's copies by rows: element 32 u + lane of the 16 x nc chunks; packed as row,
  // element offset in the row, place of a key and of a value chunk in the stage
  const int nc = a.D / CE, inv_nc = (65535 + nc) / nc;   // e / nc = e inv_nc >> 16 for e < 2048
  uint32_t todo[MODE == kFlat ? 1 : NU] = {}, place[MODE == kFlat ? 1 : NU] = {};
  if constexpr (MODE != kFlat) {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int e = 32 * u + lane, r = MODE == kFull ? e / (RB / CB) : (e * inv_nc) >> 16;
      const int ch = MODE == kFull ? e % (RB / CB) : e - r * nc;
      todo[u] = MODE == kFull || r < 16 ? r | (ch * CE) << 8 : 0xffu;
      place[u] = (r * RB + (ch ^ pd_kswz<CE>(r)) * CB) | (POOL + r * RB + (ch ^ pd_xswz<CE>(r)) * CB) << 16;
    }
  }
  if constexpr (MODE == kRows) {  // the chunks between D and the fragments' width stay zero
    for (int i = lane; i < STAGES * STAGE / 16; i += 32) *reinterpret_cast<uint4*>(own + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
    __syncwarp();
  }
  // whole rows: consecutive u are RPU rows apart
  constexpr int RPU = MODE == kFull ? 32 * CB / RB : 1;
  const long long kfirst = (todo[0] & 0xff) * a.k.sn + (todo[0] >> 8), kstep = RPU * a.k.sn;
  const long long xfirst = (todo[0] & 0xff) * a.x.sn + (todo[0] >> 8), xstep = RPU * a.x.sn;
  const bool dense = MODE == kFull && (a.ps & 15) == 0 && a.k.sn == a.D && a.x.sn == a.D;
  const bool one_page = MODE == kFlat || (a.ps & 15) == 0;  // a warp's 16 tokens never span two pages
  auto issue = [&](int st) {     // copies of the producer's tile, then the look-up of the next
    if (ahead > 0) {
      const uint32_t dst = own_s + st * STAGE;
      const int lim = pc.n - (pc.tile * kPdTile + 16 * warp);  // tokens of this warp's 16
      long long k0 = 0, x0 = 0;
      if (one_page && lim > 0) {
        k0 = __shfl_sync(0xffffffffu, koff, 0);
        x0 = __shfl_sync(0xffffffffu, xoff, 0);
      }
      if constexpr (MODE == kFlat) {
        const uint32_t to = dst + 16 * lane;
        const bf16* kp = a.k.p + k0 + 8 * lane;
        const bf16* xp = a.x.p + x0 + 8 * lane;
        if (lim >= 16) {
#pragma unroll
          for (int u = 0; u < NU; ++u)
            if (flat_copied(NK, a.D, u, lane)) {
              copy_async<16>(to + 512 * u, kp + 256 * u, 16);
              copy_async<16>(to + POOL + 512 * u, xp + 256 * u, 16);
            }
        } else {
          const int most = max(0, lim) * a.D * 2;          // bytes of the run that are tokens
#pragma unroll 1
          for (int u = 0; u < NU; ++u) {
            const int e = 16 * (32 * u + lane), bytes = max(0, min(16, most - e));
            if (e < 32 * a.D) {                            // a page's 16 rows, inside it past `lim` too
              copy_async<16>(dst + e, kp + 256 * u, bytes);
              copy_async<16>(dst + POOL + e, xp + 256 * u, bytes);
            }
          }
        }
      } else if (MODE == kFull && dense) {  // the 16 rows are one run
        const bf16* kp = a.k.p + k0 + 8 * lane;
        const bf16* xp = a.x.p + x0 + 8 * lane;
        const uint32_t kto = dst + (place[0] & 0xffff);
        const int rl = lim - (int)(todo[0] & 0xff);
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          const int bytes = RPU * u < rl ? CB : 0;         // rows past `lim` are in the page too
          copy_async<CB>(kto + 512 * u, kp + 256 * u, bytes);
          copy_async<CB>(dst + (place[u] >> 16), xp + 256 * u, bytes);
        }
      } else if (MODE == kFull && one_page) {  // rows 2 u + lane / 16 of the page, inside it past `lim` too
        const bf16* kp = a.k.p + k0 + kfirst;
        const bf16* xp = a.x.p + x0 + xfirst;
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          const int bytes = (int)(todo[u] & 0xff) < lim ? CB : 0;
          copy_async<CB>(dst + (place[u] & 0xffff), kp, bytes);
          copy_async<CB>(dst + (place[u] >> 16), xp, bytes);
          kp += kstep;
          xp += xstep;
        }
      } else {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          const int r = todo[u] & 0xff, e = todo[u] >> 8;
          const bool in = r < lim;
          long long ko, xo;
          if (one_page) {
            ko = k0 + r * a.k.sn;
            xo = x0 + r * a.x.sn;
          } else {
            ko = __shfl_sync(0xffffffffu, koff, r & 15);
            xo = __shfl_sync(0xffffffffu, xoff, r & 15);
          }
          if (MODE == kFull || r < 16) {
            copy_async<CB>(dst + (place[u] & 0xffff), a.k.p + (in ? ko + e : 0), in ? CB : 0);
            copy_async<CB>(dst + (place[u] >> 16), a.x.p + (in ? xo + e : 0), in ? CB : 0);
          }
        }
      }
      if (--ahead > 0 && ++pc.tile == pc.nt) {
        pd_next_item(a, pc, ahead);
        ph = pc.hb / a.nblk;
      }
      look_up();
    }
    copy_commit();
  };
  look_up();
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) issue(s);
  int st = 0;                    // stage of the consumer's tile
  // ldmatrix: lane l addresses row l & 7 (+ 8 for the odd matrices) of chunk i + l / 16
  const int xat = POOL + ((lane & 7) + (lane & 8)) * RB, xsw = (lane >> 4) ^ (lane & 7);

  while (left > 0) {
    // ---- one segment: the run's tiles of one item ----
    const int h = c.hb / a.nblk, blk = c.hb % a.nblk;
    const int r_first = blk * a.rows;                      // first query row of the block
    const int nq = min(a.gq - r_first, a.rows);            // query rows of the block
    const int upd = STEP && blk == 0 ? nq : -1;            // the update row
    const bool lone = STEP && !R8 && upd == 8;             // and nothing else in rows 8-15
    const int tiles = min(c.nt - c.tile, left);
    // operand A: rows g and g + 8
    uint32_t qa[KS][R8 ? 2 : 4];
    float ss = 0.f;
#pragma unroll
    for (int hf = 0; hf < (R8 ? 1 : 2); ++hf) {
      const int r = g + 8 * hf;
      const bf16* row_q = nullptr;
      if (r < nq) row_q = a.q + (long long)c.b * a.q_sb + (long long)(h * a.gq + r_first + r) * a.q_sh;
      else if (r == upd) row_q = a.kn + (long long)c.b * a.kn_sb + (long long)h * a.kn_sh;
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int u = 0; u < CE / 4; ++u) {
          const int e = (4 * i + j) * CE + 4 * u;
          uint2 v = make_uint2(0u, 0u);
          if (row_q != nullptr && e < a.D) v = *reinterpret_cast<const uint2*>(row_q + e);
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
    m[1] = STEP && (g + 8 == upd || lone) ? 0.f : -INFINITY;

    for (int it = 0; it < tiles; ++it) {
      __syncwarp();                          // every lane has read the stage that is filled next
      issue(st == 0 ? STAGES - 1 : st - 1);
      copy_wait<STAGES - 1>();            // this lane's copies of the tile have landed,
      __syncwarp();                          // and the other lanes'
      const unsigned char* in = own + st * STAGE;
      const uint32_t in_s = own_s + st * STAGE;
      st = st + 1 == STAGES ? 0 : st + 1;
      const int base = (c.tile + it) * kPdTile + 16 * warp;
      if (base >= c.n) continue;             // uniform in the warp
      // keys: operand B of both 8-key tiles
      uint32_t kr[2][NK][KR];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          if constexpr (MODE == kFlat) {
            // a chunk past D is the next row's: not this key's
            load_chunk<KR>(in + (g + 8 * kt) * 2 * a.D + (4 * i + j) * CB, kr[kt][i]);
            if (4 * i + 3 >= (NK == 4 ? 1 : 4 * NK - 11 + (NK == 5 ? 8 : 0)) && 4 * i + j >= nc) kr[kt][i][0] = kr[kt][i][1] = 0u;
          } else {
            load_chunk<KR>(in + (g + 8 * kt) * RB + ((4 * i + j) ^ pd_kswz<CE>(g)) * CB, kr[kt][i]);
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
            const uint32_t b0 = kr[kt][i][2 * u], b1 = kr[kt][i][2 * u + 1];
            // rows 8-15 are free at 8 rows: the step puts the tile's own keys there, whose
            // squared norms then come out on the diagonal of the same instruction
            if constexpr (R8) mma16816(S[kt], qa[ks][0], STEP ? b0 : 0u, qa[ks][1], STEP ? b1 : 0u, b0, b1);
            else mma16816(S[kt], qa[ks][0], qa[ks][1], qa[ks][2], qa[ks][3], b0, b1);
            if constexpr (STEP && !R8)
              mma16816(dg[kt], kr[0][i][2 * u], kr[1][i][2 * u], kr[0][i][2 * u + 1], kr[1][i][2 * u + 1],
                       kr[kt][i][2 * u], kr[kt][i][2 * u + 1]);
          }
        }
      // 1 / rms of this lane's four keys 2j, 2j+1, 8+2j, 9+2j: the diagonal element of
      // key q (of its tile) sits in lane 4 q + q / 2
      float rk[4] = {1.f, 1.f, 1.f, 1.f};
      if constexpr (STEP) {
        const float d0 = R8 ? ((g & 1) ? S[0][3] : S[0][2]) : ((g & 1) ? dg[0][1] : dg[0][0]);
        const float d1 = R8 ? ((g & 1) ? S[1][3] : S[1][2]) : ((g & 1) ? dg[1][3] : dg[1][2]);
        const float v0 = rsqrtf(d0 * inv_d + a.eps), v1 = rsqrtf(d1 * inv_d + a.eps);
        rk[0] = __shfl_sync(0xffffffffu, v0, 9 * j);
        rk[1] = __shfl_sync(0xffffffffu, v0, 9 * j + 4);
        rk[2] = __shfl_sync(0xffffffffu, v1, 9 * j);
        rk[3] = __shfl_sync(0xffffffffu, v1, 9 * j + 4);
      }
      uint32_t phi[4], pmi[4], plo[4];
      float al[2] = {1.f, 1.f};
#pragma unroll
      for (int hf = 0; hf < (R8 ? 1 : 2); ++hf) {
        const bool is_upd = STEP && (g + 8 * hf == upd || (hf == 1 && lone));
        float z[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float sc = S[q >> 1][2 * hf + (q & 1)];
          z[q] = is_upd ? fmaf(sc * rs_new * rk[q], c1, -c2) : sc * c1;
        }
        if (base + 16 > c.n) {               // uniform: the sequence's last tokens
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (base + 8 * (q >> 1) + 2 * j + (q & 1) >= c.n) z[q] = -INFINITY;
        }
        if (!(STEP && hf == 1 && lone)) {    // uniform: the update row alone needs no maximum
          float mx = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          // the reference point moves only when a score passes it by kPdSlack: until then
          // the weights stay below 2^kPdSlack, which costs an fp32 sum no digits
          if (!is_upd && mx > m[hf] + kPdSlack) {
            al[hf] = ex2(m[hf] - mx);        // 0 while nothing has been seen
            m[hf] = mx;
          }
        }
        const float ms = m[hf] == -INFINITY ? 0.f : m[hf];
        float p[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) p[q] = ex2(z[q] - ms);
        l[hf] = l[hf] * al[hf] + ((p[0] + p[1]) + (p[2] + p[3]));
        phi[2 * hf] = pack_bf16(p[0], p[1]);
        phi[2 * hf + 1] = pack_bf16(p[2], p[3]);
        const float2 h0 = unpack_bf16(phi[2 * hf]), h1 = unpack_bf16(phi[2 * hf + 1]);
        p[0] -= h0.x; p[1] -= h0.y; p[2] -= h1.x; p[3] -= h1.y;  // exact
        pmi[2 * hf] = pack_bf16(p[0], p[1]);
        pmi[2 * hf + 1] = pack_bf16(p[2], p[3]);
        const float2 m0 = unpack_bf16(pmi[2 * hf]), m1 = unpack_bf16(pmi[2 * hf + 1]);
        plo[2 * hf] = pack_bf16(p[0] - m0.x, p[1] - m0.y);
        plo[2 * hf + 1] = pack_bf16(p[2] - m1.x, p[3] - m1.y);
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
      auto weigh = [&](float (&sum)[4], uint32_t b0, uint32_t b1) {
        float d[4];                          // the smallest parts first
        if constexpr (R8) {
          mma16816_zero(d, plo[0], 0u, plo[1], 0u, b0, b1);
          mma16816(d, phi[0], pmi[0], phi[1], pmi[1], b0, b1);
        } else {
          mma16816_zero(d, plo[0], plo[2], plo[1], plo[3], b0, b1);
          mma16816(d, pmi[0], pmi[2], pmi[1], pmi[3], b0, b1);
          mma16816(d, phi[0], phi[2], phi[1], phi[3], b0, b1);
        }
        add2(sum[0], sum[1], d[0], d[1]);
        add2(sum[2], sum[3], d[2], d[3]);
      };
      if constexpr (CE == 8) {               // columns in order: tile i holds 8 i .. 8 i + 7
#pragma unroll
        for (int i = 0; i < NT; i += 2) {
          uint32_t x[4];
          ldmatrix_x4_trans(x, in_s + xat + ((i ^ xsw) << 4));
          weigh(acc[i], x[0], x[1]);
          weigh(acc[i + 1], x[2], x[3]);
        }
      } else {                               // rows 2j, 2j+1, 8+2j, 9+2j, chunk 8 c + g
#pragma unroll
        for (int cx = 0; cx < NX; ++cx) {
          uint32_t xr[4][KR];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int r = 8 * (q >> 1) + 2 * j + (q & 1);
            if constexpr (MODE == kFlat) load_chunk<KR>(in + POOL + r * 2 * a.D + (8 * cx + g) * CB, xr[q]);
            else load_chunk<KR>(in + POOL + r * RB + ((8 * cx + g) ^ pd_xswz<CE>(2 * j)) * CB, xr[q]);
          }
#pragma unroll
          for (int e = 0; e < CE; ++e) {
            const uint32_t sel = (e & 1) ? 0x7632u : 0x5410u;
            weigh(acc[cx * CE + e], __byte_perm(xr[0][e >> 1], xr[1][e >> 1], sel),
                  __byte_perm(xr[2][e >> 1], xr[3][e >> 1], sel));
          }
        }
      }
    }

    // ---- the segment's rows: merge the four warps in fixed order ----
    auto column = [&](int i, int u) {        // of accumulator acc[i][u]
      return CE == 8 ? 8 * i + 2 * j + u : ((i / CE) * 8 + 2 * j + u) * CE + i % CE;
    };
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
      for (int w = 0; w < kPdWarps; ++w) L[hf] += ex2(red_ml[w][g + 8 * hf][0] - Ms) * red_ml[w][g + 8 * hf][1];
      f[hf] = ex2(m[hf] - Ms);
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
          const int col = column(i, u & 1);
          if (put && col < 128) red[buf][g + 8 * (u >> 1)][col] = round == 0 ? acc[i][u] * f[u >> 1] : acc[i][u];
        }
      __syncthreads();
      if (take) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int u = 0; u < (R8 ? 2 : 4); ++u) {
            const int col = column(i, u & 1);
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
            const int col = column(i, u);
            if (col < a.D) d[col] = acc[i][2 * hf + u];
          }
        if (j == 0) {
          d[a.D] = M[hf];
          d[a.D + 1] = L[hf];
        }
      }
    }
    // ---- on to the next item ----
    left -= tiles;
    c.tile += tiles;
    if (c.tile == c.nt && left > 0) pd_next_item(a, c, left);
  }
  copy_wait<0>();
}

// The join: merges an item's segments and, in the step, adds the new token.  Blocks
// (sequence and kv head, y).  Few segments: the block y = 0 gives a warp to each query row,
// lane i holding columns 4 i .. 4 i + 3.  Many (a long sequence over many CTAs): each query
// row takes a whole block, warp w the segments w, w + 8, ...  Either way a segment's row is one
// 16-byte load per lane, all of them independent, and the order of the sums is fixed.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32, kJoinFew = 16, kJoinAhead = 6;

// (max, denominator, weighted sum) of `cnt` segment rows at p, p + step, ...; the lanes
// together read the maxima first.  Lanes past D (col false) sum nothing.
struct JoinRow {
  float M, L;
  float4 acc;
};
__device__ __forceinline__ JoinRow join_rows(const float* p, long long step, int cnt, int D, bool col, int lane) {
  JoinRow r{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int i0 = 0; i0 < cnt; i0 += 32) {
    float mi = -INFINITY, li = 0.f;
    if (i0 + lane < cnt) {
      const float2 ml = *reinterpret_cast<const float2*>(p + (i0 + lane) * step + D);
      mi = ml.x;
      li = ml.y;
    }
    const int k = min(32, cnt - i0);
    float4 v[kJoinAhead];
    auto fetch = [&](int q0) {       // all loads of a group before any use
#pragma unroll
      for (int q = 0; q < kJoinAhead; ++q) {
        v[q] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (col && q0 + q < k) v[q] = *reinterpret_cast<const float4*>(p + (i0 + q0 + q) * step + 4 * lane);
      }
    };
    fetch(0);
    float mx = mi;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float mn = fmaxf(r.M, mx), ms = mn == -INFINITY ? 0.f : mn;
    const float f = ex2(mi - ms), fo = ex2(r.M - ms);
    float ls = f * li;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, o);
    r.L = r.L * fo + ls;
    r.acc.x *= fo; r.acc.y *= fo; r.acc.z *= fo; r.acc.w *= fo;
    r.M = mn;
    for (int q0 = 0; q0 < k; q0 += kJoinAhead) {
      if (q0 > 0) fetch(q0);
#pragma unroll
      for (int q = 0; q < kJoinAhead; ++q) {
        const float fq = __shfl_sync(0xffffffffu, f, (q0 + q) & 31);  // 0 past the last segment's lane
        r.acc.x = fmaf(fq, v[q].x, r.acc.x);
        r.acc.y = fmaf(fq, v[q].y, r.acc.y);
        r.acc.z = fmaf(fq, v[q].z, r.acc.z);
        r.acc.w = fmaf(fq, v[q].w, r.acc.w);
      }
    }
  }
  return r;
}
// plain sum of `cnt` rows
__device__ __forceinline__ float4 join_sum(const float* p, long long step, int cnt, bool col, int lane) {
  float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int q0 = 0; q0 < cnt; q0 += kJoinAhead) {
    float4 v[kJoinAhead];
#pragma unroll
    for (int q = 0; q < kJoinAhead; ++q) {
      v[q] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (col && q0 + q < cnt) v[q] = *reinterpret_cast<const float4*>(p + (q0 + q) * step + 4 * lane);
    }
#pragma unroll
    for (int q = 0; q < kJoinAhead; ++q) { u.x += v[q].x; u.y += v[q].y; u.z += v[q].z; u.w += v[q].w; }
  }
  return u;
}
__device__ __forceinline__ float4 load4(const bf16* p) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const float2 x = unpack_bf16(v.x), y = unpack_bf16(v.y);
  return make_float4(x.x, x.y, y.x, y.y);
}

template <bool STEP>
__global__ void __launch_bounds__(kJoinThreads, 3) paged_join_kernel(const __grid_constant__ PagedDecodeArgs a) {
  __shared__ __align__(16) float sum_a[kJoinWarps][128], sum_u[kJoinWarps][128];
  __shared__ float wm[kJoinWarps], wl[kJoinWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / a.H, h = blockIdx.x % a.H;
  const int raw = a.lengths[b];
  const bool over = (long long)raw > (long long)a.M * a.ps;
  const bool used = raw >= 0 && !over;
  if (over && tid == 0) report(a.status, kStatusLength, kTagPagedDecode);
  const int n = used ? raw : 0, nt = pd_tiles(n);
  const int pr = a.D + 4;
  const long long slot = (long long)(a.rows + (STEP ? 1 : 0)) * pr;
  // first unit of the sequence and the batch's units
  long long before = 0, T = 0;
  for (int i = lane; i < a.B; i += 32) {
    const int ti = pd_units(pd_len(a, i));
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
  // segments of the item (h, blk): ctas [i0, i0 + cnt), slots cta + item
  auto range = [&](int blk, int& cnt) -> const float* {
    cnt = 0;
    if (nt == 0) return a.part;
    const long long first = before + ((long long)h * a.nblk + blk) * (nt + kPdItemCost) + kPdItemCost;
    const long long last = first + nt - 1;
    const int i0 = (int)pd_div((first + 1) * G - 1, T);
    cnt = (int)pd_div((last + 1) * G - 1, T) - i0 + 1;
    return a.part + (i0 + (long long)blockIdx.x * a.nblk + blk) * slot;
  };
  int cnt0;
  const float* p0 = range(0, cnt0);
  const bool few = cnt0 <= kJoinFew;   // the other blocks of query rows differ by one segment at most
  if (few && blockIdx.y > 0) return;
  const bool col = 4 * lane < a.D;
  const float c1 = a.s * kLog2e;
  // what the tile pass does not write: this lane's columns of the new key and value, and
  // the place of the new row
  float4 kn = make_float4(0.f, 0.f, 0.f, 0.f), vn = kn;
  int page = -1;
  if (STEP && used && col) {
    kn = load4(a.kn + (long long)b * a.kn_sb + (long long)h * a.kn_sh + 4 * lane);
    vn = load4(a.vn + (long long)b * a.vn_sb + (long long)h * a.vn_sh + 4 * lane);
  }
  if (STEP && used && a.append && blockIdx.y == 0) {
    const int pi = n / a.ps;
    page = pi < a.M ? a.table[(long long)b * a.t_sb + pi] : -1;
    if (page < 0 || page >= a.P) {
      if (tid == 0) report(a.status, pi < a.M ? kStatusPage : kStatusLength, kTagPagedDecode);
      page = -1;
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the tile pass has ended and its stores are seen

  // x_new as the cache holds it, from the sum u; one warp of the sequence and head writes it
  auto solved = [&](const float4& u, bool write) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!col) return x;
    const uint32_t lo = pack_bf16(vn.x - u.x, vn.y - u.y), hi = pack_bf16(vn.z - u.z, vn.w - u.w);
    const float2 x0 = unpack_bf16(lo), x1 = unpack_bf16(hi);
    x = make_float4(x0.x, x0.y, x1.x, x1.y);
    if (write) {
      *reinterpret_cast<uint2*>(a.xo + (long long)b * a.xo_sb + (long long)h * a.xo_sh + 4 * lane) = make_uint2(lo, hi);
      if (page >= 0) {
        const long long row = n % a.ps;
        *reinterpret_cast<uint2*>(a.k.p + (long long)page * a.k.sp + (long long)h * a.k.sh + row * a.k.sn + 4 * lane) =
            make_uint2(pack_bf16(kn.x, kn.y), pack_bf16(kn.z, kn.w));
        *reinterpret_cast<uint2*>(a.x.p + (long long)page * a.x.sp + (long long)h * a.x.sh + row * a.x.sn + 4 * lane) =
            make_uint2(lo, hi);
      }
    }
    return x;
  };
  // the row's output from its merged sums and the new token
  auto finish = [&](int r, float M, float L, float4 acc, const float4& x) {
    if constexpr (STEP) {
      float z = 0.f;
      if (col) {
        const float4 q = load4(a.q + (long long)b * a.q_sb + (long long)(h * a.gq + r) * a.q_sh + 4 * lane);
        z = (q.x * kn.x + q.y * kn.y) + (q.z * kn.z + q.w * kn.w);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
      z *= c1;
      const float mn = fmaxf(M, z), ms = mn == -INFINITY ? 0.f : mn;
      const float f = ex2(M - ms), p = ex2(z - ms);
      L = fmaf(L, f, p);
      acc = make_float4(fmaf(acc.x, f, p * x.x), fmaf(acc.y, f, p * x.y), fmaf(acc.z, f, p * x.z), fmaf(acc.w, f, p * x.w));
    }
    const bool none = !used || (!STEP && nt == 0);  // no token to attend to
    if (col)
      *reinterpret_cast<uint2*>(a.o + (long long)b * a.o_sb + (long long)(h * a.gq + r) * a.o_sh + 4 * lane) =
          none ? make_uint2(0u, 0u) : make_uint2(pack_bf16(acc.x / L, acc.y / L), pack_bf16(acc.z / L, acc.w / L));
  };
  const long long upd = (long long)min(a.gq, a.rows) * pr;  // the update row of block 0's segments
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  bool have_x = false;
  for (int blk = 0; blk < a.nblk; ++blk) {
    int cnt;
    const float* p = range(blk, cnt);
    const int r0 = blk * a.rows, r1 = min(a.gq, r0 + a.rows);
    if (few) {
      for (int r = r0 + warp; r < r1; r += kJoinWarps) {
        float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
        if (STEP && !have_x) u = join_sum(p0 + upd, slot, cnt0, col, lane);
        const JoinRow j = join_rows(p + (r - r0) * (long long)pr, slot, cnt, a.D, col, lane);
        if (STEP && !have_x) {
          x = solved(u, r == 0);
          have_x = true;
        }
        finish(r, j.M, j.L, j.acc, x);
      }
    } else {
      if (STEP && blk == 0) {
        *reinterpret_cast<float4*>(&sum_u[warp][4 * lane]) =
            join_sum(p0 + upd + warp * slot, kJoinWarps * slot, (cnt0 - warp + kJoinWarps - 1) / kJoinWarps, col, lane);
        __syncthreads();
        float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) {
          const float4 v = *reinterpret_cast<const float4*>(&sum_u[w][4 * lane]);
          u.x += v.x; u.y += v.y; u.z += v.z; u.w += v.w;
        }
        x = solved(u, blockIdx.y == 0 && warp == 0);
      }
      for (int r = r0; r < r1; ++r) {
        if (r % (int)gridDim.y != (int)blockIdx.y) continue;
        const JoinRow j = join_rows(p + (r - r0) * (long long)pr + warp * slot, kJoinWarps * slot,
                                    (cnt - warp + kJoinWarps - 1) / kJoinWarps, a.D, col, lane);
        *reinterpret_cast<float4*>(&sum_a[warp][4 * lane]) = j.acc;
        if (lane == 0) {
          wm[warp] = j.M;
          wl[warp] = j.L;
        }
        __syncthreads();
        if (warp == 0) {
          float M = wm[0];
#pragma unroll
          for (int w = 1; w < kJoinWarps; ++w) M = fmaxf(M, wm[w]);
          const float ms = M == -INFINITY ? 0.f : M;
          float L = 0.f;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kJoinWarps; ++w) {
            const float f = ex2(wm[w] - ms);
            const float4 v = *reinterpret_cast<const float4*>(&sum_a[w][4 * lane]);
            L = fmaf(f, wl[w], L);
            acc = make_float4(fmaf(f, v.x, acc.x), fmaf(f, v.y, acc.y), fmaf(f, v.z, acc.z), fmaf(f, v.w, acc.w));
          }
          finish(r, M, L, acc, x);
        }
        __syncthreads();  // the sums are free again
      }
    }
  }
}

constexpr int kPdDevices = 64;  // devices whose attributes are remembered

static int pd_device() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    dev = kPdDevices;
  }
  return dev;
}

static int pd_sms() {
  static std::atomic<int> known[kPdDevices];
  const int dev = pd_device();
  if (dev >= kPdDevices) return 148;
  int sms = known[dev].load(std::memory_order_relaxed);
  if (sms == 0) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
      cudaGetLastError();
      return 148;
    }
    known[dev].store(sms, std::memory_order_relaxed);
  }
  return sms;
}

// the most CTAs a tile pass runs with (workspace size)
int paged_decode_ctas() { return 3 * pd_sms(); }

template <bool STEP, bool R8, int CE, int NK, int NX, int MODE>
static cudaError_t launch_pd(PagedDecodeArgs& a, cudaStream_t st) {
  using Shape = PdShape<R8, CE, NK, NX, MODE>;
  static std::atomic<bool> sized[kPdDevices];  // shared memory granted on this device
  const int dev = pd_device();
  if (dev >= kPdDevices || !sized[dev].load(std::memory_order_relaxed)) {
    const cudaError_t e = cudaFuncSetAttribute(paged_decode_kernel<STEP, R8, CE, NK, NX, MODE>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem);
    if (e != cudaSuccess) return e;
    if (dev < kPdDevices) sized[dev].store(true, std::memory_order_relaxed);
  }
  a.nctas = Shape::kCtas * pd_sms();
  paged_decode_kernel<STEP, R8, CE, NK, NX, MODE><<<a.nctas, kPdThreads, Shape::kSmem, st>>>(a);
  return cudaGetLastError();
}

template <bool STEP, bool R8>
static cudaError_t launch_pd_d(PagedDecodeArgs& a, cudaStream_t st) {
  const bool base16 = ((reinterpret_cast<uintptr_t>(a.k.p) | reinterpret_cast<uintptr_t>(a.x.p)) & 15u) == 0 &&
                      ((a.k.sp | a.k.sh | a.x.sp | a.x.sh) & 7) == 0;
  if (base16 && ((a.k.sn | a.x.sn | a.D) & 7) == 0) {
    if (a.D == 64) return launch_pd<STEP, R8, 8, 2, 1, kFull>(a, st);
    if (a.D == 128) return launch_pd<STEP, R8, 8, 4, 2, kFull>(a, st);
    if (a.D < 64) return launch_pd<STEP, R8, 8, 2, 1, kRows>(a, st);
    return launch_pd<STEP, R8, 8, 4, 2, kRows>(a, st);
  }
  if (base16 && a.k.sn == a.D && a.x.sn == a.D && a.ps % 16 == 0) {  // D is an odd multiple of 4 here
    switch (flat_chunks(a.D)) {
      case 4: return launch_pd<STEP, R8, 4, 4, 2, kFlat>(a, st);
      case 5: return launch_pd<STEP, R8, 4, 5, 3, kFlat>(a, st);
      default: return launch_pd<STEP, R8, 4, 8, 4, kFlat>(a, st);
    }
  }
  if (a.D <= 64) return launch_pd<STEP, R8, 4, 4, 2, kRows>(a, st);
  if (a.D <= 80) return launch_pd<STEP, R8, 4, 5, 3, kRows>(a, st);
  return launch_pd<STEP, R8, 4, 8, 4, kRows>(a, st);
}

cudaError_t launch_paged_decode(PagedDecodeArgs a, bool step, cudaStream_t st) {
  const int rows = std::min(a.gq, a.rows) + (step ? 1 : 0);
  cudaError_t e = step ? (rows <= 8 ? launch_pd_d<true, true>(a, st) : launch_pd_d<true, false>(a, st))
                       : (rows <= 8 ? launch_pd_d<false, true>(a, st) : launch_pd_d<false, false>(a, st));
  if (e != cudaSuccess) return e;
  // a block for each query row while that fills the GPU only a few times over.  The join's
  // blocks may start while the tile pass ends (they wait before reading its results).
  const int bh = a.B * a.H;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(bh, bh >= 4096 ? 1 : a.gq);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return step ? cudaLaunchKernelEx(&cfg, paged_join_kernel<true>, a) : cudaLaunchKernelEx(&cfg, paged_join_kernel<false>, a);
}

}  // namespace lb
