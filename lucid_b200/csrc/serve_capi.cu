// extern "C" entry points of the serving operators (include/lucid_b200.h): paged
// decoding, page movement, token log probabilities.
#include "lucid_b200.h"
#include "profile.h"
#include "serve_common.cuh"

#include <climits>
#include <cstdlib>
#include <cstring>

using namespace lb;

namespace {
constexpr int kMaxD = 128;
bool ptr_ok(const void* p, unsigned to) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
bool m4(int64_t a, int64_t b, int64_t c = 0) { return ((a | b | c) & 3) == 0; }
cudaStream_t stream_of(void* s) { return reinterpret_cast<cudaStream_t>(s); }
int done(cudaError_t e) { return e == cudaSuccess ? LUCID_OK : LUCID_ERR_LAUNCH; }

// query heads per kv head in row blocks of at most 16 operand rows (one of them the
// update row of the step)
void row_blocks(int gq, bool step, int* nblk, int* rows) {
  const int most = step ? 15 : 16;
  *nblk = (gq + most - 1) / most;
  *rows = (gq + *nblk - 1) / *nblk;
}

bool heads_ok(int B, int Hq, int Hkv, int D) {
  return B >= 0 && Hq >= 0 && Hkv > 0 && D >= 4 && D <= kMaxD && D % 4 == 0 && Hq % Hkv == 0 &&
         (long long)B * Hq <= INT_MAX;
}
bool pool_ok(int P, int ps, int M) { return P > 0 && ps > 0 && M > 0 && (long long)M * ps <= INT_MAX - 64; }

size_t decode_bytes(int B, int Hq, int Hkv, int D, bool step) {
  if (!heads_ok(B, Hq, Hkv, D) || Hq == 0) return 256;
  int nblk, rows;
  row_blocks(Hq / Hkv, step, &nblk, &rows);
  const size_t slots = (size_t)paged_decode_ctas() + (size_t)B * Hkv * nblk;
  return slots * (rows + (step ? 1 : 0)) * (D + 4) * sizeof(float) + 256;
}

int decode(bool step, int B, int Hq, int Hkv, int D, int P, int ps, int M, float scale, float eps,
           const void* q, int64_t q_sb, int64_t q_sh, const void* kn, int64_t kn_sb, int64_t kn_sh,
           const void* vn, int64_t vn_sb, int64_t vn_sh, void* kp, int64_t kp_sp, int64_t kp_sh, int64_t kp_sn,
           void* xp, int64_t xp_sp, int64_t xp_sh, int64_t xp_sn, const int* table, int64_t t_sb, const int* lengths,
           void* xo, int64_t xo_sb, int64_t xo_sh, void* o, int64_t o_sb, int64_t o_sh, int append, int* status,
           void* workspace, size_t workspace_bytes, void* stream) {
  if (!heads_ok(B, Hq, Hkv, D) || !pool_ok(P, ps, M)) return LUCID_ERR_SHAPE;
  if (B == 0 || Hq == 0) return LUCID_OK;
  if (Hq / Hkv > 65535) return LUCID_ERR_SHAPE;
  if (!ptr_ok(q, 8) || !ptr_ok(kp, 8) || !ptr_ok(xp, 8) || !ptr_ok(table, 4) || !ptr_ok(lengths, 4) || !ptr_ok(o, 8) ||
      !m4(q_sb, q_sh) || !m4(o_sb, o_sh) || !m4(kp_sp, kp_sh, kp_sn) || !m4(xp_sp, xp_sh, xp_sn))
    return LUCID_ERR_ALIGN;
  if (step && (!ptr_ok(kn, 8) || !ptr_ok(vn, 8) || !ptr_ok(xo, 8) || !m4(kn_sb, kn_sh) || !m4(vn_sb, vn_sh) ||
               !m4(xo_sb, xo_sh)))
    return LUCID_ERR_ALIGN;
  if (!ptr_ok(workspace, 16) || workspace_bytes < decode_bytes(B, Hq, Hkv, D, step)) return LUCID_ERR_WORKSPACE;
  PagedDecodeArgs a{};
  a.B = B; a.H = Hkv; a.D = D; a.P = P; a.ps = ps; a.M = M;
  a.ps_shift = -1;
  for (int s = 0; s < 31; ++s)
    if (ps == 1 << s) a.ps_shift = s;
  a.gq = Hq / Hkv;
  row_blocks(a.gq, step, &a.nblk, &a.rows);
  a.s = scale; a.eps = eps;
  a.q = static_cast<const bf16*>(q); a.q_sb = q_sb; a.q_sh = q_sh;
  a.kn = static_cast<const bf16*>(kn); a.kn_sb = kn_sb; a.kn_sh = kn_sh;
  a.vn = static_cast<const bf16*>(vn); a.vn_sb = vn_sb; a.vn_sh = vn_sh;
  a.k = PoolView{static_cast<bf16*>(kp), kp_sp, kp_sh, kp_sn};
  a.x = PoolView{static_cast<bf16*>(xp), xp_sp, xp_sh, xp_sn};
  a.table = table; a.t_sb = t_sb; a.lengths = lengths;
  a.xo = static_cast<bf16*>(xo); a.xo_sb = xo_sb; a.xo_sh = xo_sh;
  a.o = static_cast<bf16*>(o); a.o_sb = o_sb; a.o_sh = o_sh;
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + 256);
  a.status = status; a.append = append;
  ProfileScope ps_(LUCID_KERNEL_PAGED_DECODE, stream_of(stream));
  return done(launch_paged_decode(a, step, stream_of(stream)));
}
}  // namespace

extern "C" {

size_t lucid_paged_decode_workspace_bytes(int B, int Hq, int Hkv, int D, int step) {
  return decode_bytes(B, Hq, Hkv, D, step != 0);
}

int lucid_paged_decode_step(int B, int Hq, int Hkv, int D, int P, int ps, int M, float scale, float eps,
                            const void* q, int64_t q_sb, int64_t q_sh,
                            const void* k_new, int64_t kn_sb, int64_t kn_sh,
                            const void* v_new, int64_t vn_sb, int64_t vn_sh,
                            void* k_pages, int64_t kp_sp, int64_t kp_sh, int64_t kp_sn,
                            void* x_pages, int64_t xp_sp, int64_t xp_sh, int64_t xp_sn,
                            const int* block_table, int64_t t_sb, const int* lengths,
                            void* x_new, int64_t xn_sb, int64_t xn_sh,
                            void* o, int64_t o_sb, int64_t o_sh, int append, int* status,
                            void* workspace, size_t workspace_bytes, void* stream) {
  return decode(true, B, Hq, Hkv, D, P, ps, M, scale, eps, q, q_sb, q_sh, k_new, kn_sb, kn_sh, v_new, vn_sb, vn_sh,
                k_pages, kp_sp, kp_sh, kp_sn, x_pages, xp_sp, xp_sh, xp_sn, block_table, t_sb, lengths,
                x_new, xn_sb, xn_sh, o, o_sb, o_sh, append, status, workspace, workspace_bytes, stream);
}

int lucid_paged_decode_attn(int B, int Hq, int Hkv, int D, int P, int ps, int M, float scale,
                            const void* q, int64_t q_sb, int64_t q_sh,
                            const void* k_pages, int64_t kp_sp, int64_t kp_sh, int64_t kp_sn,
                            const void* x_pages, int64_t xp_sp, int64_t xp_sh, int64_t xp_sn,
                            const int* block_table, int64_t t_sb, const int* lengths,
                            void* o, int64_t o_sb, int64_t o_sh, int* status,
                            void* workspace, size_t workspace_bytes, void* stream) {
  return decode(false, B, Hq, Hkv, D, P, ps, M, scale, 0.f, q, q_sb, q_sh, nullptr, 0, 0, nullptr, 0, 0,
                const_cast<void*>(k_pages), kp_sp, kp_sh, kp_sn, const_cast<void*>(x_pages), xp_sp, xp_sh, xp_sn,
                block_table, t_sb, lengths, nullptr, 0, 0, o, o_sb, o_sh, 0, status, workspace, workspace_bytes, stream);
}

int lucid_paged_append(int B, int Hkv, int N, int D, int P, int ps, int M,
                       const void* k, int64_t k_sb, int64_t k_sh, int64_t k_sn,
                       const void* x, int64_t x_sb, int64_t x_sh, int64_t x_sn,
                       void* k_pages, int64_t kp_sp, int64_t kp_sh, int64_t kp_sn,
                       void* x_pages, int64_t xp_sp, int64_t xp_sh, int64_t xp_sn,
                       const int* block_table, int64_t t_sb, const int* lengths, const int* counts,
                       int* status, void* stream) {
  if (B < 0 || B > 65535 || Hkv < 0 || N < 0 || D < 4 || D > kMaxD || D % 4 || !pool_ok(P, ps, M)) return LUCID_ERR_SHAPE;
  if (B == 0 || Hkv == 0 || N == 0) return LUCID_OK;
  if (!ptr_ok(k, 8) || !ptr_ok(x, 8) || !ptr_ok(k_pages, 8) || !ptr_ok(x_pages, 8) || !ptr_ok(block_table, 4) ||
      !ptr_ok(lengths, 4) || (counts != nullptr && !ptr_ok(counts, 4)) || !m4(k_sb, k_sh, k_sn) || !m4(x_sb, x_sh, x_sn) ||
      !m4(kp_sp, kp_sh, kp_sn) || !m4(xp_sp, xp_sh, xp_sn))
    return LUCID_ERR_ALIGN;
  PagedAppendArgs a{B, Hkv, N, D, P, ps, M,
                    static_cast<const bf16*>(k), k_sb, k_sh, k_sn, static_cast<const bf16*>(x), x_sb, x_sh, x_sn,
                    PoolView{static_cast<bf16*>(k_pages), kp_sp, kp_sh, kp_sn},
                    PoolView{static_cast<bf16*>(x_pages), xp_sp, xp_sh, xp_sn},
                    block_table, t_sb, lengths, counts, status};
  ProfileScope ps_(LUCID_KERNEL_PAGES, stream_of(stream));
  return done(launch_paged_append(a, stream_of(stream)));
}

int lucid_copy_pages(int layers, int P, int64_t page_bytes, void* k_pages, int64_t k_layer, int64_t k_page,
                     void* x_pages, int64_t x_layer, int64_t x_page, const int* src, const int* dst, int pairs,
                     void* stream) {
  // at most one grid of blocks, one per 8 KB of a page, for a launch's pairs
  if (layers < 0 || P < 0 || page_bytes <= 0 || page_bytes % 8 || pairs < 0 ||
      (page_bytes + 8191) / 8192 > INT_MAX / 2 / kCopyPairs / (layers > 0 ? layers : 1))
    return LUCID_ERR_SHAPE;
  if (pairs == 0 || layers == 0) return LUCID_OK;
  if (src == nullptr || dst == nullptr) return LUCID_ERR_SHAPE;
  // every page written once and none of them read: the order of the copies is then free
  unsigned char* mark = static_cast<unsigned char*>(std::calloc((size_t)(P > 0 ? P : 1), 1));
  if (mark == nullptr) return LUCID_ERR_TOO_LARGE;
  bool fine = true;
  for (int i = 0; i < pairs && fine; ++i) {
    fine = src[i] >= 0 && src[i] < P && dst[i] >= 0 && dst[i] < P && !mark[dst[i]];
    if (fine) mark[dst[i]] = 1;
  }
  for (int i = 0; i < pairs && fine; ++i) fine = !mark[src[i]];
  std::free(mark);
  if (!fine) return LUCID_ERR_SHAPE;
  if (!ptr_ok(k_pages, 8) || !ptr_ok(x_pages, 8) || ((k_layer | k_page | x_layer | x_page) & 7)) return LUCID_ERR_ALIGN;
  PageCopyArgs a;
  a.pool[0] = static_cast<char*>(k_pages);
  a.pool[1] = static_cast<char*>(x_pages);
  a.layer[0] = k_layer; a.layer[1] = x_layer;
  a.page[0] = k_page; a.page[1] = x_page;
  a.bytes = page_bytes;
  a.layers = layers;
  ProfileScope ps_(LUCID_KERNEL_PAGES, stream_of(stream));
  for (int i = 0; i < pairs; i += kCopyPairs) {
    a.pairs = pairs - i < kCopyPairs ? pairs - i : kCopyPairs;
    std::memcpy(a.src, src + i, (size_t)a.pairs * sizeof(int));
    std::memcpy(a.dst, dst + i, (size_t)a.pairs * sizeof(int));
    const cudaError_t e = launch_page_copy(a, stream_of(stream));
    if (e != cudaSuccess) return LUCID_ERR_LAUNCH;
  }
  return LUCID_OK;
}

// V leaves room for the kernels' 32-bit element indexes to pass its end by a batch
static bool logprob_shape(int64_t R0, int64_t R1, int V, int dtype) {
  return R0 >= 0 && R1 >= 0 && V > 0 && V <= 1 << 30 && dtype >= 0 && dtype <= 2 &&
         (R1 == 0 || R0 <= INT_MAX / R1);
}

int lucid_token_logprobs(int64_t R0, int64_t R1, int V, int dtype, const void* logits, int64_t s0, int64_t s1,
                         const int64_t* tokens, int top, float* logprobs, float* entropy, float* stats,
                         float* top_logprobs, int64_t* top_tokens, int* status, void* stream) {
  if (!logprob_shape(R0, R1, V, dtype) || top < 0 || top > LUCID_MAX_TOP || top > V) return LUCID_ERR_SHAPE;
  if (R0 == 0 || R1 == 0) return LUCID_OK;
  if (!ptr_ok(logits, dtype == 2 ? 4 : 2) || !ptr_ok(entropy, 4) || (stats != nullptr && !ptr_ok(stats, 4)) ||
      (tokens != nullptr && (!ptr_ok(tokens, 8) || !ptr_ok(logprobs, 4))) ||
      (top > 0 && (!ptr_ok(top_logprobs, 4) || !ptr_ok(top_tokens, 8))))
    return LUCID_ERR_ALIGN;
  LogprobArgs a{};
  a.logits = logits; a.R0 = R0; a.R1 = R1; a.s0 = s0; a.s1 = s1; a.V = V; a.top = top;
  a.tokens = reinterpret_cast<const long long*>(tokens);
  a.logprobs = logprobs; a.entropy = entropy; a.stats = stats;
  a.top_lp = top_logprobs; a.top_tok = reinterpret_cast<long long*>(top_tokens);
  a.status = status;
  ProfileScope ps_(LUCID_KERNEL_LOGPROBS, stream_of(stream));
  return done(launch_logprobs_fwd(a, dtype, stream_of(stream)));
}

int lucid_token_logprobs_bwd(int64_t R0, int64_t R1, int V, int dtype, const void* logits, int64_t s0, int64_t s1,
                             const int64_t* tokens, const float* stats, const float* g_logprobs, const float* g_entropy,
                             void* dlogits, void* stream) {
  if (!logprob_shape(R0, R1, V, dtype)) return LUCID_ERR_SHAPE;
  if (R0 == 0 || R1 == 0) return LUCID_OK;
  const unsigned es = dtype == 2 ? 4 : 2;
  if (!ptr_ok(logits, es) || !ptr_ok(dlogits, es) || !ptr_ok(stats, 4) ||
      (tokens != nullptr && !ptr_ok(tokens, 8)))
    return LUCID_ERR_ALIGN;
  LogprobArgs a{};
  a.logits = logits; a.R0 = R0; a.R1 = R1; a.s0 = s0; a.s1 = s1; a.V = V;
  a.tokens = reinterpret_cast<const long long*>(tokens);
  a.stats = const_cast<float*>(stats);
  a.g_lp = g_logprobs; a.g_ent = g_entropy; a.dlogits = dlogits;
  ProfileScope ps_(LUCID_KERNEL_LOGPROBS, stream_of(stream));
  return done(launch_logprobs_bwd(a, dtype, stream_of(stream)));
}

}  // extern "C"
