// C ABI of the FP8 blocks' operators and of layer norm (declared in include/novaq.h):
// argument validation, status codes and dispatch.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "novaq_convert.h"
#include "novaq_internal.h"

using namespace novaq;

namespace {

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
bool plain_float(int dt) { return dt == F32 || dt == F16 || dt == BF16; }
bool fp8(int dt) { return dt == E4M3 || dt == E5M2; }
constexpr int64_t INT = 0x7FFFFFFF;

// An R x C matrix in blocks: rows below 2^31, a row's bytes so that 256 of them stay
// within a buffer's 2 GiB.
int check_matrix(int64_t R, int64_t C, int block_rows) {
  if (R < 0 || C < 0 || (block_rows != 1 && block_rows != 128)) return NOVAQ_EINVAL;
  if (R >= INT || C > ((int64_t)1 << 22)) return NOVAQ_ENOTSUP;
  return NOVAQ_OK;
}
// Rows that are normalised.
int check_rows(int64_t R, int64_t D) {
  if (R < 0 || D < 0) return NOVAQ_EINVAL;
  if (D == 0) return NOVAQ_ESHAPE;
  return R >= INT || D > (1 << 20) ? NOVAQ_ENOTSUP : NOVAQ_OK;
}
int64_t tiles_of(int64_t R, int64_t C) { return ((R + 127) / 128) * ((C + 127) / 128); }

// Bytes of an R x C matrix's codes and of its exponents (block_rows 1), each on a boundary
// of 256.
size_t up256(int64_t n) { return ((size_t)n + 255) / 256 * 256; }
size_t code_bytes(int64_t R, int64_t C) { return up256(R * ((C + 127) / 128 * 128)); }
size_t exponent_bytes(int64_t R, int64_t C) { return up256(R * ((C + 511) / 512 * 4)); }

// The parts of a layer's workspaces.
struct ForwardWs {
  size_t codes = 0, exponents, product, total;
  ForwardWs(int64_t M, int64_t K, int64_t N)
      : exponents(code_bytes(M, K)),
        product(exponents + exponent_bytes(M, K)),
        total(product + block_product_workspace(M, N, K)) {}
};
struct BackwardWs {
  // the gradient's codes, the transposed ones, the input's transposed ones (where they are
  // made here), then what the column sums and the products need in turn
  size_t g = 0, ge, gt, gte, xt, xte, rest, total;
  BackwardWs(int64_t M, int64_t K, int64_t N, bool kept)
      : ge(code_bytes(M, N)),
        gt(ge + exponent_bytes(M, N)),
        gte(gt + code_bytes(N, M)),
        xt(gte + exponent_bytes(N, M)),
        xte(xt + (kept ? 0 : code_bytes(K, M))),
        rest(xte + (kept ? 0 : exponent_bytes(K, M))),
        total(rest + std::max({quantize_blocks_workspace(M, N), block_product_workspace(M, K, N),
                               block_product_workspace(N, K, M)})) {}
};

// A layer's sizes: M rows, K inputs, N outputs.
int check_layer(int64_t M, int64_t K, int64_t N) {
  if (M < 0 || K < 0 || N < 0) return NOVAQ_EINVAL;
  if (K == 0) return NOVAQ_ESHAPE;
  const int64_t most = (int64_t)1 << 22;
  if (M > most || K > most || N > most || tiles_of(M, N) >= most || tiles_of(M, K) >= most ||
      tiles_of(N, K) >= most)
    return NOVAQ_ENOTSUP;
  return NOVAQ_OK;
}

}  // namespace

extern "C" {

size_t novaq_quantize_blocks_workspace(int64_t R, int64_t C) {
  return R <= 128 || C <= 0 || R >= INT || C >= INT ? 0 : quantize_blocks_workspace(R, C);
}

int novaq_quantize_blocks(const void* x, int x_dtype, int64_t R, int64_t C, int dtype,
                          int block_rows, void* codes, void* exponents, void* codes_t,
                          void* exponents_t, float* colsum, void* workspace,
                          size_t workspace_bytes, void* stream) {
  if (!plain_float(x_dtype) || !fp8(dtype)) return NOVAQ_EDTYPE;
  int rc = check_matrix(R, C, block_rows);
  if (rc == NOVAQ_OK && codes_t) rc = check_matrix(C, R, block_rows);
  if (rc != NOVAQ_OK) return rc;
  if (!codes != !exponents || !codes_t != !exponents_t) return NOVAQ_EINVAL;
  if (colsum && block_rows != 1) return NOVAQ_EINVAL;
  if (!aligned(x, 16) || !aligned(codes, 16) || !aligned(codes_t, 16) || !aligned(exponents, 4) ||
      !aligned(exponents_t, 4) || !aligned(colsum, 4) || !aligned(workspace, 16))
    return NOVAQ_EALIGN;
  if (tiles_of(R, C) >= (1 << 23)) return NOVAQ_ENOTSUP;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (C == 0) return NOVAQ_OK;
  if (R == 0)
    return colsum ? fill_u32_launch(reinterpret_cast<uint32_t*>(colsum), 0u, (int)C, st) : NOVAQ_OK;
  if (!codes && !codes_t && !colsum) return NOVAQ_OK;
  if (!x) return NOVAQ_EINVAL;
  if (colsum && R > 128 && (!workspace || workspace_bytes < quantize_blocks_workspace(R, C)))
    return NOVAQ_EINVAL;
  return quantize_blocks_launch(x, x_dtype, R, C, dtype, block_rows, codes, exponents, codes_t,
                                exponents_t, colsum, workspace, false, st);
}

int novaq_dequantize_blocks(const void* codes, int dtype, const void* exponents, int64_t R,
                            int64_t C, int block_rows, void* out, int out_dtype, void* stream) {
  if (!fp8(dtype) || !plain_float(out_dtype)) return NOVAQ_EDTYPE;
  const int rc = check_matrix(R, C, block_rows);
  if (rc != NOVAQ_OK) return rc;
  if (!aligned(codes, 16) || !aligned(out, 16)) return NOVAQ_EALIGN;
  if (R == 0 || C == 0) return NOVAQ_OK;
  if (!codes || !exponents || !out) return NOVAQ_EINVAL;
  return dequantize_blocks_launch(codes, dtype, exponents, R, C, block_rows, out, out_dtype,
                                  static_cast<hipStream_t>(stream));
}

size_t novaq_block_product_workspace(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || M >= INT || N >= INT || K > ((int64_t)1 << 22)) return 0;
  return block_product_workspace(M, N, K);
}

int novaq_block_product(const void* x, int x_dtype, const void* x_exponents, int x_block_rows,
                        int64_t M, int64_t K, const void* w, int w_dtype,
                        const void* w_exponents, int w_block_rows, int64_t N, const float* bias,
                        void* y, int y_dtype, void* workspace, size_t workspace_bytes,
                        void* stream) {
  if (!fp8(x_dtype) || !fp8(w_dtype) || !plain_float(y_dtype)) return NOVAQ_EDTYPE;
  int rc = check_matrix(M, K, x_block_rows);
  if (rc == NOVAQ_OK) rc = check_matrix(N, K, w_block_rows);
  if (rc != NOVAQ_OK) return rc;
  if (K == 0) return NOVAQ_ESHAPE;
  if (tiles_of(M, N) >= (1 << 22)) return NOVAQ_ENOTSUP;
  if (!aligned(x, 16) || !aligned(w, 16) || !aligned(x_exponents, 4) || !aligned(w_exponents, 4) ||
      !aligned(bias, 4) || !aligned(y, 16) || !aligned(workspace, 16))
    return NOVAQ_EALIGN;
  if (M == 0 || N == 0) return NOVAQ_OK;
  if (!x || !x_exponents || !w || !w_exponents || !y) return NOVAQ_EINVAL;
  const size_t need = block_product_workspace(M, N, K);
  if (need && (!workspace || workspace_bytes < need)) return NOVAQ_EINVAL;
  return block_product_launch(x, x_dtype, x_exponents, x_block_rows, M, K, w, w_dtype, w_exponents,
                              w_block_rows, N, bias, y, y_dtype, workspace,
                              static_cast<hipStream_t>(stream));
}

size_t novaq_block_linear_workspace(int64_t M, int64_t K, int64_t N) {
  return M <= 0 || N <= 0 || check_layer(M, K, N) != NOVAQ_OK ? 0 : ForwardWs(M, K, N).total;
}

int novaq_block_linear(const void* x, int x_dtype, int64_t M, int64_t K, int q_dtype,
                       const void* w, int w_dtype, const void* w_exponents, int64_t N,
                       const float* bias, void* y, int y_dtype, void* kept,
                       void* kept_exponents, void* workspace, size_t workspace_bytes,
                       void* stream) {
  if (!plain_float(x_dtype) || !fp8(q_dtype) || !fp8(w_dtype) || !plain_float(y_dtype))
    return NOVAQ_EDTYPE;
  const int rc = check_layer(M, K, N);
  if (rc != NOVAQ_OK) return rc;
  if (!kept != !kept_exponents) return NOVAQ_EINVAL;
  if (!aligned(x, 16) || !aligned(w, 16) || !aligned(w_exponents, 4) || !aligned(bias, 4) ||
      !aligned(y, 16) || !aligned(kept, 16) || !aligned(kept_exponents, 4) ||
      !aligned(workspace, 16))
    return NOVAQ_EALIGN;
  if (M == 0) return NOVAQ_OK;
  if (!x) return NOVAQ_EINVAL;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (N == 0)
    return kept ? quantize_blocks_launch(x, x_dtype, M, K, q_dtype, 1, nullptr, nullptr, kept,
                                         kept_exponents, nullptr, nullptr, true, st)
                : NOVAQ_OK;
  const ForwardWs p(M, K, N);
  if (!w || !w_exponents || !y || !workspace || workspace_bytes < p.total) return NOVAQ_EINVAL;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int rq = quantize_blocks_launch(x, x_dtype, M, K, q_dtype, 1, ws + p.codes,
                                        ws + p.exponents, kept, kept_exponents, nullptr, nullptr, true,
                                        st);
  if (rq != NOVAQ_OK) return rq;
  return block_product_launch(ws + p.codes, q_dtype, ws + p.exponents, 1, M, K, w, w_dtype,
                              w_exponents, 128, N, bias, y, y_dtype, ws + p.product, st);
}

size_t novaq_block_linear_backward_workspace(int64_t M, int64_t K, int64_t N, int kept) {
  return M <= 0 || N <= 0 || check_layer(M, K, N) != NOVAQ_OK ? 0
                                                               : BackwardWs(M, K, N, kept).total;
}

int novaq_block_linear_backward(const void* grad, int grad_dtype, int64_t M, int64_t N,
                                int gq_dtype, const void* x, int x_dtype, int xq_dtype,
                                const void* kept, const void* kept_exponents, int64_t K,
                                const void* w_t, int w_dtype, const void* w_t_exponents,
                                void* grad_input, void* grad_weight, int gw_dtype,
                                float* grad_bias, void* workspace, size_t workspace_bytes,
                                void* stream) {
  if (!plain_float(grad_dtype) || !fp8(gq_dtype) || !fp8(xq_dtype) || !fp8(w_dtype) ||
      !plain_float(gw_dtype) || (!kept && !plain_float(x_dtype)))
    return NOVAQ_EDTYPE;
  int rc = check_layer(M, K, N);
  if (rc != NOVAQ_OK) return rc;
  if (!kept != !kept_exponents) return NOVAQ_EINVAL;
  if (!aligned(grad, 16) || !aligned(x, 16) || !aligned(kept, 16) || !aligned(kept_exponents, 4) ||
      !aligned(w_t, 16) || !aligned(w_t_exponents, 4) || !aligned(grad_input, 16) ||
      !aligned(grad_weight, 16) || !aligned(grad_bias, 4) || !aligned(workspace, 16))
    return NOVAQ_EALIGN;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (M == 0 || N == 0) return NOVAQ_ESHAPE;  // (empty sums are the caller's zeros)
  const BackwardWs p(M, K, N, kept != nullptr);
  if (!grad || (grad_weight && !kept && !x) || (grad_input && (!w_t || !w_t_exponents)) ||
      !workspace || workspace_bytes < p.total)
    return NOVAQ_EINVAL;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  rc = quantize_blocks_launch(grad, grad_dtype, M, N, gq_dtype, 1, grad_input ? ws + p.g : nullptr,
                              grad_input ? ws + p.ge : nullptr, grad_weight ? ws + p.gt : nullptr,
                              grad_weight ? ws + p.gte : nullptr, grad_bias, ws + p.rest, true, st);
  if (rc == NOVAQ_OK && grad_input)
    rc = block_product_launch(ws + p.g, gq_dtype, ws + p.ge, 1, M, N, w_t, w_dtype, w_t_exponents,
                              128, K, nullptr, grad_input, grad_dtype, ws + p.rest, st);
  if (rc != NOVAQ_OK || !grad_weight) return rc;
  if (!kept) {
    rc = quantize_blocks_launch(x, x_dtype, M, K, xq_dtype, 1, nullptr, nullptr, ws + p.xt,
                                ws + p.xte, nullptr, nullptr, true, st);
    if (rc != NOVAQ_OK) return rc;
    kept = ws + p.xt, kept_exponents = ws + p.xte;
  }
  return block_product_launch(ws + p.gt, gq_dtype, ws + p.gte, 1, N, M, kept, xq_dtype,
                              kept_exponents, 1, K, nullptr, grad_weight, gw_dtype, ws + p.rest, st);
}

int novaq_layer_norm(const void* x, int x_dtype, int64_t R, int64_t D, const float* gamma,
                     const float* beta, float eps, void* y, int y_dtype, void* exponents,
                     float* mean, float* rstd, void* stream) {
  if (!plain_float(x_dtype) || !(plain_float(y_dtype) || fp8(y_dtype))) return NOVAQ_EDTYPE;
  const int rc = check_rows(R, D);
  if (rc != NOVAQ_OK) return rc;
  if (!(eps >= 0.0f) || !mean != !rstd || !exponents != !fp8(y_dtype)) return NOVAQ_EINVAL;
  if (!aligned(x, 16) || !aligned(gamma, 16) || !aligned(beta, 16) || !aligned(y, 16) ||
      !aligned(exponents, 4) || !aligned(mean, 4) || !aligned(rstd, 4))
    return NOVAQ_EALIGN;
  if (R == 0) return NOVAQ_OK;
  if (!x || !y) return NOVAQ_EINVAL;
  return layer_norm_launch(x, x_dtype, R, D, gamma, beta, eps, y, y_dtype, exponents, mean, rstd,
                           static_cast<hipStream_t>(stream));
}

size_t novaq_layer_norm_backward_workspace(int64_t R, int64_t D) {
  return R <= 0 || check_rows(R, D) != NOVAQ_OK ? 0 : layer_norm_backward_workspace(R, D);
}

int novaq_layer_norm_backward(const void* grad, int grad_dtype, const void* x, int x_dtype,
                              int64_t R, int64_t D, const float* gamma, const float* mean,
                              const float* rstd, void* grad_input, float* grad_gamma,
                              float* grad_beta, void* workspace, size_t workspace_bytes,
                              void* stream) {
  if (!plain_float(x_dtype) || (grad_dtype != x_dtype && grad_dtype != F32)) return NOVAQ_EDTYPE;
  const int rc = check_rows(R, D);
  if (rc != NOVAQ_OK) return rc;
  if (!aligned(grad, 16) || !aligned(x, 16) || !aligned(gamma, 16) || !aligned(grad_input, 16) ||
      !aligned(grad_gamma, 4) || !aligned(grad_beta, 4) || !aligned(mean, 4) ||
      !aligned(rstd, 4) || !aligned(workspace, 16))
    return NOVAQ_EALIGN;
  if (!grad_input && !grad_gamma && !grad_beta) return NOVAQ_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (R == 0) {
    int rf = NOVAQ_OK;
    if (grad_gamma) rf = fill_u32_launch(reinterpret_cast<uint32_t*>(grad_gamma), 0u, (int)D, st);
    if (grad_beta && rf == NOVAQ_OK)
      rf = fill_u32_launch(reinterpret_cast<uint32_t*>(grad_beta), 0u, (int)D, st);
    return rf;
  }
  if (!grad || !x || !mean || !rstd || !workspace) return NOVAQ_EINVAL;
  if (workspace_bytes < layer_norm_backward_workspace(R, D)) return NOVAQ_EINVAL;
  return layer_norm_backward_launch(grad, grad_dtype, x, x_dtype, R, D, gamma, mean, rstd,
                                    grad_input, grad_gamma, grad_beta, workspace, st);
}

}  // extern "C"
