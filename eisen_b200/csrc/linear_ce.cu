// Head projection and cross-entropy in pieces of the vocabulary: x = h W is never stored.
//
//   forward   every 256-column tile of the product leaves (maximum, sum of exponentials) per row, formed from
//             the f32 accumulators in the GEMM's epilogue (gemm_tc2.cu, LCE_STATS); ce_join_kernel adds them up:
//             lse = M + ln sum_t s_t exp(m_t - M),  row loss = -ln(exp(x_y - lse) + 1e-8) * normalizer.
//             2 rows k vocab FLOPs, 8 bytes per row and tile instead of 512 for the logits.
//   backward  per piece of the vocabulary the tile is formed again and leaves D = exp(x - lse) - onehot in bf16
//             (LCE_GRAD), then dH += c D W^T and dW = c H^T D with c = normalizer * grad by the library's GEMM.
//             6 rows k vocab FLOPs (4 with the logits at hand).
//
// The row statistics come from unrounded logits; a [rows, vocab] tensor of bf16 logits carries a rounding of up to
// 2^-9 of a logit, 3 % of a probability at |x| = 16.  D is the one value rounded to bf16 on the way to the
// gradients: the tensor cores take bf16 operands.
#include <algorithm>
#include <cstdio>

#include "common.cuh"
#include "errors.h"
#include "gemm_tc.h"
#include "../../include/eisen_b200.h"

namespace eisen {
namespace {

constexpr int CJ_ROWS = 32, CJ_FLIGHT = 4;

// A CTA joins the tiles of 32 rows (lane = row: a tile's statistics of successive rows lie side by side), dealt to
// SLICES warps, four loads of each in flight.  Bound by the latency of those loads where rows are few (64 rows, 125 tiles:
// 10.6 us with 8 warps that waited for one load after the other, 4.8 now), by reading 8 bytes per row and tile where they are many.
// A launch of one CTA also adds up the loss.
template <int CJ_SLICES>
__global__ void __launch_bounds__(CJ_ROWS * CJ_SLICES)
ce_join_kernel(const float2* __restrict__ stats, const float* __restrict__ target_logit, const int* __restrict__ targets,
               float* __restrict__ loss, float* __restrict__ row_loss, float* __restrict__ lse, long long rows, int tiles,
               int vocab, int ignore_index, float normalizer, int* __restrict__ bad_target_flag) {
  __shared__ float sh_m[CJ_SLICES][CJ_ROWS], sh_s[CJ_SLICES][CJ_ROWS];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const long long row = (long long)blockIdx.x * CJ_ROWS + lane;
  float m = -INFINITY, s = 0.0f;
  if (row < rows) {
    for (int t0 = slice; t0 < tiles; t0 += CJ_FLIGHT * CJ_SLICES) {
      float2 v[CJ_FLIGHT];
#pragma unroll
      for (int q = 0; q < CJ_FLIGHT; ++q) {
        const int t = t0 + q * CJ_SLICES;
        v[q] = t < tiles ? stats[(long long)t * rows + row] : make_float2(-INFINITY, 0.0f);
      }
      float nm = m;
#pragma unroll
      for (int q = 0; q < CJ_FLIGHT; ++q) nm = fmaxf(nm, v[q].x);
      const float ref = nm == -INFINITY ? 0.0f : nm;
      s *= expf(m - ref);
#pragma unroll
      for (int q = 0; q < CJ_FLIGHT; ++q) s += v[q].y * expf(v[q].x - ref);
      m = nm;
    }
  }
  sh_m[slice][lane] = m;
  sh_s[slice][lane] = s;
  __syncthreads();
  if (slice == 0) {
    float l = 0.0f;
    if (row < rows) {
      float gm = -INFINITY, gs = 0.0f;
#pragma unroll
      for (int i = 0; i < CJ_SLICES; ++i) gm = fmaxf(gm, sh_m[i][lane]);
      const float ref = gm == -INFINITY ? 0.0f : gm;
#pragma unroll
      for (int i = 0; i < CJ_SLICES; ++i) gs += sh_s[i][lane] * expf(sh_m[i][lane] - ref);
      const int t = targets[row];
      float e = 0.0f;
      if (t != ignore_index && t >= 0 && t < vocab) {
        e = ref + logf(gs);
        l = -logf(expf(target_logit[row] - e) + 1e-8f) * normalizer;
      } else if (t != ignore_index && bad_target_flag) {
        *bad_target_flag = 1;
      }
      row_loss[row] = l;
      lse[row] = e;
    }
    if (gridDim.x == 1 && loss) {
      l = warp_sum(l);
      if (lane == 0) *loss = l;
    }
  }
}

// dst [n] (op)= the sum of `slices` f32 vectors that lie n elements apart, in their order, rounded once.  Eight elements per thread.
__global__ void __launch_bounds__(256)
ce_slices_kernel(__nv_bfloat16* __restrict__ dst, const float* __restrict__ src, int slices, long long n, int accumulate) {
  for (long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 8; i < n; i += (long long)gridDim.x * blockDim.x * 8) {
    float x[8], o[8];
    ld16(src + i, *reinterpret_cast<float(*)[4]>(x));
    ld16(src + i + 4, *reinterpret_cast<float(*)[4]>(x + 4));
    for (int s = 1; s < slices; ++s) {
      ld16(src + s * n + i, *reinterpret_cast<float(*)[4]>(o));
      ld16(src + s * n + i + 4, *reinterpret_cast<float(*)[4]>(o + 4));
#pragma unroll
      for (int c = 0; c < 8; ++c) x[c] += o[c];
    }
    if (accumulate) {
      ld16(dst + i, o);
#pragma unroll
      for (int c = 0; c < 8; ++c) x[c] += o[c];
    }
    st16(dst + i, x);
  }
}

struct CePlan {
  long long piece, ld;                 // vocabulary entries of a piece, row stride of D
  long long stats_bytes, fwd_bytes;    // forward: tile statistics, then the target logits
  long long d_bytes, bwd_bytes;        // backward: D, then dH in f32
  int dh_slices;                       // f32 sums of dH, one per k slice, added up over the pieces; 0: dH leaves the product as it is
};

constexpr long long up256(long long n) { return (n + 255) & ~255LL; }

CePlan ce_plan(long long rows, long long k, long long vocab, long long piece) {
  CePlan p;
  // D of the default piece takes about CE_D_BYTES: fewer pieces are faster, and beyond that not by much.  Forward and backward
  // with an f32 weight gradient that is added to, D in 64 / 128 / 256 / 512 MB: 16384 x 2048 x 32000 8.5 / 7.7 / 7.3 / 7.0 ms;
  // 2048 x 2048 x 32000 0.99 ms / 0.95 in one piece (125 MB); 1021 x 1000 x 50001 tied, in 32 MB 0.60 ms, 0.51-0.55 in one (102 MB)
  constexpr long long CE_D_BYTES = 256LL << 20;
  const long long all = (vocab + GEMM_CE_COLS - 1) / GEMM_CE_COLS * GEMM_CE_COLS;
  if (piece <= 0) piece = CE_D_BYTES / (2 * std::max<long long>(rows, 1));
  piece = std::max<long long>(piece / GEMM_CE_COLS * GEMM_CE_COLS, GEMM_CE_COLS);
  const long long n = (all + std::min(piece, all) - 1) / std::min(piece, all);
  piece = ((all + n - 1) / n + GEMM_CE_COLS - 1) / GEMM_CE_COLS * GEMM_CE_COLS;  // pieces of about the same size
  p.piece = piece;
  p.ld = piece;
  const long long tiles = all / GEMM_CE_COLS;
  p.stats_bytes = up256(tiles * rows * 8);
  p.fwd_bytes = p.stats_bytes + up256(rows * 4);
  p.d_bytes = up256(rows * p.ld * 2);
  // Few output tiles of dH and a long sum: in k slices, with sums of their own that are added up in order at the end, so that the
  // result is the same every time (forward and backward of 64 x 384 x 8192: 58 us, 88 in one slice; of 1021 x 1000 x 50001, tied:
  // 475-483, slices that add up atomically in one place 480-499).  Their memory stays within 64 MB.
  const int most = (int)std::min<long long>(32, (64LL << 20) / (rows * k * 4));
  p.dh_slices = gemm_pair_split_k_apart(rows, k, std::min(piece, vocab), vocab, most);
  if (n == 1 && p.dh_slices == 1) p.dh_slices = 0;
  p.bwd_bytes = p.d_bytes + up256(p.dh_slices * rows * k * 4);
  return p;
}

int ce_check(const char* what, const void* h, long long ldh, const void* w, long long ldw, int trans_b, const void* targets,
             const void* workspace, long long rows, long long k, long long vocab) {
  static thread_local char msg[160];
  auto bad = [&](int code, const char* why) {
    snprintf(msg, sizeof(msg), "%s: %s", what, why);
    return fail(code, msg);
  };
  if (rows < 0 || k <= 0 || vocab <= 0) return bad(EISEN_ERR_INVALID, "rows must not be negative, k and vocab must be positive");
  if (rows > 0x7fffff00LL || k > 0x7fffff00LL || vocab > 0x7fffff00LL) return bad(EISEN_ERR_LIMIT, "a dimension exceeds 2^31 - 256");
  if (!h || !w || !targets || !workspace) return bad(EISEN_ERR_INVALID, "h, w, targets and workspace must not be null");
  if (ldh < k || ldw < (trans_b ? k : vocab)) return bad(EISEN_ERR_INVALID, "a leading dimension is shorter than its row");
  if ((ldh % 8) || (ldw % 8) || !aligned16(h) || !aligned16(w) || !aligned16(workspace))
    return bad(EISEN_ERR_INVALID, "h, w and workspace must be 16-byte aligned, leading dimensions multiples of 8");
  return 0;
}

}  // namespace
}  // namespace eisen

extern "C" {

long long eisen_linear_ce_workspace_bytes(long long rows, long long k, long long vocab, long long piece, int backward) {
  using namespace eisen;
  if (rows <= 0 || k <= 0 || vocab <= 0) return 256;
  const CePlan p = ce_plan(rows, k, vocab, piece);
  return backward ? std::max(p.fwd_bytes, p.bwd_bytes) : p.fwd_bytes;
}

int eisen_linear_ce_fwd(void* stream, const void* h, long long ldh, const void* w, long long ldw, int trans_b, const int* targets,
                        float* loss, float* row_loss, float* lse, void* workspace, long long rows, long long k, long long vocab,
                        int ignore_index, float normalizer, int* bad_target_flag, int* status) {
  using namespace eisen;
  if (rows == 0) {
    if (loss && cudaMemsetAsync(loss, 0, 4, (cudaStream_t)stream) != cudaSuccess) return fail(EISEN_ERR_CUDA, "linear_ce_fwd: memset");
    return 0;
  }
  int rc = ce_check("linear_ce_fwd", h, ldh, w, ldw, trans_b, targets, workspace, rows, k, vocab);
  if (rc) return rc;
  if (!row_loss || !lse) return fail(EISEN_ERR_INVALID, "linear_ce_fwd: row_loss and lse must not be null");
  const CePlan p = ce_plan(rows, k, vocab, 0);
  float2* stats = (float2*)workspace;
  float* target_logit = (float*)((char*)workspace + p.stats_bytes);
  const char* err = nullptr;
  rc = gemm_bf16_pair_ce((cudaStream_t)stream, trans_b ? 0 : 1, (int)rows, (int)vocab, (int)k, h, ldh, w, ldw, 0, targets,
                         ignore_index, (int)vocab, 0, stats, target_logit, nullptr, nullptr, 0, status, &err);
  if (rc) return fail(EISEN_ERR_CUDA, err ? err : "linear_ce_fwd failed");
  count_launch();
  const unsigned grid = (unsigned)((rows + CJ_ROWS - 1) / CJ_ROWS);
  const int tiles = (int)((vocab + GEMM_CE_COLS - 1) / GEMM_CE_COLS);
  if (tiles <= 32)
    ce_join_kernel<8><<<grid, CJ_ROWS * 8, 0, (cudaStream_t)stream>>>(stats, target_logit, targets, loss, row_loss, lse, rows, tiles, (int)vocab,
                                                                     ignore_index, normalizer, bad_target_flag);
  else
    ce_join_kernel<32><<<grid, CJ_ROWS * 32, 0, (cudaStream_t)stream>>>(stats, target_logit, targets, loss, row_loss, lse, rows, tiles,
                                                                       (int)vocab, ignore_index, normalizer, bad_target_flag);
  rc = check_launch("linear_ce_join");
  if (rc || !loss || grid == 1) return rc;
  return eisen_ce_loss_reduce(stream, row_loss, loss, rows);
}

int eisen_linear_ce_bwd(void* stream, const void* h, long long ldh, const void* w, long long ldw, int trans_b, const int* targets,
                        const float* lse, const float* grad_out, void* dh, int accumulate_dh, void* dw, long long lddw,
                        int dw_dtype, int accumulate_dw, void* workspace, long long rows, long long k, long long vocab,
                        long long piece, int ignore_index, float normalizer, int* status) {
  using namespace eisen;
  cudaStream_t s = (cudaStream_t)stream;
  const long long dw_rows = trans_b ? vocab : k, dw_cols = trans_b ? k : vocab;
  if (dw && (dw_dtype != DT_F32 && dw_dtype != DT_BF16)) return fail(EISEN_ERR_INVALID, "linear_ce_bwd: dw must be f32 or bf16");
  if (dw && lddw < dw_cols) return fail(EISEN_ERR_INVALID, "linear_ce_bwd: lddw is shorter than a row of dw");
  if (rows == 0) {
    const size_t es = dw_dtype == DT_F32 ? 4 : 2;
    if (dw && !accumulate_dw && dw_cols > 0 && dw_rows > 0 &&
        cudaMemset2DAsync(dw, (size_t)lddw * es, 0, (size_t)dw_cols * es, (size_t)dw_rows, s) != cudaSuccess)
      return fail(EISEN_ERR_CUDA, "linear_ce_bwd: memset");
    return 0;
  }
  int rc = ce_check("linear_ce_bwd", h, ldh, w, ldw, trans_b, targets, workspace, rows, k, vocab);
  if (rc) return rc;
  if (!lse || (!dh && !dw)) return fail(EISEN_ERR_INVALID, "linear_ce_bwd: lse and one of dh, dw must not be null");
  if (!aligned16(dh) || !aligned16(dw)) return fail(EISEN_ERR_INVALID, "linear_ce_bwd: dh and dw must be 16-byte aligned");
  if (k % 8) return fail(EISEN_ERR_INVALID, "linear_ce_bwd: k must be a multiple of 8");
  if ((dh && dh == h) || (dw && dw == w)) return fail(EISEN_ERR_INVALID, "linear_ce_bwd: a gradient may not go over its operand");
  const CePlan p = ce_plan(rows, k, vocab, piece);
  char* d = (char*)workspace;
  float* dh32 = (float*)(d + p.d_bytes);
  // C (op)= normalizer * (*grad_out) * A B^T on the paired-CTA kernel, whatever the size: its k slices fill the machine
  auto product = [&](int a_mn, int b_mn, long long M, long long N, long long K, const void* A, long long lda, const void* B,
                     long long ldb, void* C, long long ldc, int mode, int split, long long apart) {
    const PairScale scale = {grad_out, apart};
    const char* err = nullptr;
    if (gemm_bf16_tc_pair(s, a_mn, b_mn, (int)M, (int)N, (int)K, A, lda, B, ldb, C, ldc, nullptr, 0, mode, split, normalizer, status, &err,
                          &scale))
      return fail(EISEN_ERR_CUDA, err ? err : "linear_ce_bwd failed");
    count_launch();
    return 0;
  };
  for (long long c0 = 0; c0 < vocab; c0 += p.piece) {
    const long long n = std::min(p.piece, vocab - c0);
    const char* wp = (const char*)w + 2 * (trans_b ? c0 * ldw : c0);
    const char* err = nullptr;
    rc = gemm_bf16_pair_ce(s, trans_b ? 0 : 1, (int)rows, (int)n, (int)k, h, ldh, wp, ldw, 1, targets, ignore_index, (int)vocab,
                           (int)c0, nullptr, nullptr, lse, d, p.ld, status, &err);
    if (rc) return fail(EISEN_ERR_CUDA, err ? err : "linear_ce_bwd failed");
    count_launch();
    if (dh) {  // dH[rows, k] += D[rows, n] W_piece^T
      // (atomically where there is something to add to: one add per element and piece)
      const int mode = p.dh_slices ? (c0 == 0 ? GEMM_OUT_F32 : GEMM_OUT_F32_ATOMIC) : accumulate_dh ? GEMM_OUT_BF16_ACC : GEMM_OUT_BF16;
      rc = product(0, trans_b ? 1 : 0, rows, k, n, d, p.ld, wp, ldw, p.dh_slices ? (void*)dh32 : dh, k, mode, std::max(p.dh_slices, 1), rows * k);
      if (rc) return rc;
    }
    if (dw) {  // dW[k, piece] = H^T D, or with the tied table dW[piece, k] = D^T H
      char* out = (char*)dw + (dw_dtype == DT_F32 ? 4 : 2) * (trans_b ? c0 * lddw : c0);
      const int mode = dw_dtype == DT_F32 ? (accumulate_dw ? GEMM_OUT_F32_ATOMIC : GEMM_OUT_F32)
                                          : (accumulate_dw ? GEMM_OUT_BF16_ACC : GEMM_OUT_BF16);
      const int split = mode == GEMM_OUT_F32_ATOMIC && !deterministic()
                            ? gemm_pair_auto_split_k((int)(trans_b ? n : k), (int)(trans_b ? k : n), (int)rows) : 1;
      rc = trans_b ? product(1, 1, n, k, rows, d, p.ld, h, ldh, out, lddw, mode, split, 0)
                   : product(1, 1, k, n, rows, h, ldh, d, p.ld, out, lddw, mode, split, 0);
      if (rc) return rc;
    }
  }
  if (!dh || !p.dh_slices) return 0;
  ce_slices_kernel<<<grid_for(rows * k, 256 * 8, 8), 256, 0, s>>>((__nv_bfloat16*)dh, dh32, p.dh_slices, rows * k, accumulate_dh);
  return check_launch("linear_ce_bwd(dh)");
}

}  // extern "C"
