// Shared definitions of the serving kernels: paged key / solved-value cache and
// token log probabilities.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace lb {

using bf16 = __nv_bfloat16;

// Run-time status codes and kernel tags (layout of sm100.cuh: code | tag << 20),
// written to the caller's status word, which may be mapped host memory.
enum : int { kStatusPage = 4, kStatusLength = 5, kStatusToken = 6 };
enum : int { kTagPagedDecode = 16, kTagPagedAppend = 17, kTagLogprobs = 18 };

__device__ __forceinline__ void report(int* status, int code, int tag) {
  if (status != nullptr) *reinterpret_cast<volatile int*>(status) = code | (tag << 20);
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// One pool of pages: element strides of [P, H, ps, D], innermost stride 1.
struct PoolView {
  bf16* p;
  long long sp, sh, sn;
};

// Paged decoding of one new token per sequence (csrc/paged_decode.cu).
struct PagedDecodeArgs {
  int B, H, D;                 // sequences, kv heads, head dimension
  int P, ps, M;                // pool pages, page size, block table width
  int ps_shift;                // log2 of the page size, -1 if it is no power of two
  int gq, nblk, rows, nctas;   // query heads per kv head, row blocks of them, rows per block, CTAs (set by the launch)
  float s, eps;
  const bf16* q;  long long q_sb, q_sh;
  const bf16* kn; long long kn_sb, kn_sh;   // new keys (step only)
  const bf16* vn; long long vn_sb, vn_sh;   // new values (step only)
  PoolView k, x;
  const int* table; long long t_sb;
  const int* lengths;
  bf16* xo; long long xo_sb, xo_sh;         // solved new values (step only)
  bf16* o;  long long o_sb, o_sh;
  float* part;                              // [nctas + B H nblk][rows, and one in the step][D + 4]
  int* status;
  int append;                               // step: write (kn, xo) into the pages
};

struct PagedAppendArgs {
  int B, H, N, D, P, ps, M;
  const bf16* k; long long k_sb, k_sh, k_sn;
  const bf16* x; long long x_sb, x_sh, x_sn;
  PoolView kp, xp;
  const int* table; long long t_sb;
  const int* lengths;
  const int* counts;                        // null: N rows of every sequence
  int* status;
};

// Page copies: the pairs travel as kernel parameters.
constexpr int kCopyPairs = 448;
struct PageCopyArgs {
  char* pool[2];
  long long layer[2], page[2];              // byte strides
  long long bytes;                          // bytes of one page of one layer (dense)
  int layers, pairs, segs;
  int src[kCopyPairs], dst[kCopyPairs];
};

// Token log probabilities (csrc/logprobs.cu).
struct LogprobArgs {
  const void* logits;
  long long R0, R1, s0, s1;                 // rows r = r0 * R1 + r1 at element r0 s0 + r1 s1
  int V, top;
  const long long* tokens;                  // [R] or null
  float* logprobs;                          // [R] (with tokens)
  float* entropy;                           // [R]
  float* stats;                             // [R][3]: maximum, log2 of the sum, entropy (forward: or null)
  float* top_lp;                            // [R][top]
  long long* top_tok;                       // [R][top]
  const float* g_lp;                        // backward: [R] or null
  const float* g_ent;                       // backward: [R] or null
  void* dlogits;                            // backward: [R][V] contiguous
  int* status;
};

cudaError_t launch_paged_decode(PagedDecodeArgs a, bool step, cudaStream_t st);
cudaError_t launch_paged_append(const PagedAppendArgs& a, cudaStream_t st);
cudaError_t launch_page_copy(const PageCopyArgs& a, cudaStream_t st);
cudaError_t launch_logprobs_fwd(const LogprobArgs& a, int dtype, cudaStream_t st);
cudaError_t launch_logprobs_bwd(const LogprobArgs& a, int dtype, cudaStream_t st);
int paged_decode_ctas();

}  // namespace lb
