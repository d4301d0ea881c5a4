// C ABI of the token operators (declared in include/novaq.h): argument
// validation, status codes and dispatch.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <memory>
#include <new>

#include "novaq_convert.h"
#include "novaq_internal.h"
#include "token_io.h"

using namespace novaq;

namespace {

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
bool plain_float(int dt) { return dt == F32 || dt == F16 || dt == BF16; }
bool any_weight(int dt) { return dt >= F32 && dt <= E2M1; }
constexpr int64_t INT = 0x7FFFFFFF;
// The embedding's gradient: 64 threads for 16 sorted tokens, fewer than 2^32 in a
// launch, and positions (with a block's and a wave's more) in 31 bits.
constexpr int64_t MOST_TOKENS = (int64_t)1 << 30;

// A (V, D) table: its type and whether it may have a scale, its sizes (256 fp32
// rows stay within a buffer's 2 GiB).
int check_table(int w_dtype, const float* w_scale, int64_t V, int64_t D) {
  if (!any_weight(w_dtype)) return NOVAQ_EDTYPE;
  if (w_scale && !is_quant(w_dtype)) return NOVAQ_EINVAL;
  if (V < 0 || D < 0) return NOVAQ_EINVAL;
  if (V == 0 || D == 0) return NOVAQ_ESHAPE;
  if (V >= INT || D > (1 << 20)) return NOVAQ_ENOTSUP;
  return NOVAQ_OK;
}

int check_ids(const void* ids, int bits) {
  if (bits != 32 && bits != 64) return NOVAQ_EDTYPE;
  if (!aligned(ids, bits / 8)) return NOVAQ_EALIGN;
  return NOVAQ_OK;
}

// The vocabulary loss's sizes: a launch's threads stay below 2^32.  N (whose pieces of
// the vocabulary have 1024 rows at least) by the logits' tiles, V by the kernel that
// reads it as stored, 256 rows a workgroup; N and a piece of V (2^21 rows at most) with
// D by the gradients' tiles.
int check_loss_sizes(int64_t N, int64_t V, int64_t D) {
  auto tiles = [](int64_t a) { return (a + 127) / 128; };
  if (N > ((int64_t)1 << 27) || V > INT - 255) return NOVAQ_ENOTSUP;
  const int64_t piece = std::min<int64_t>(V, 1 << 21);
  if (std::max(tiles(N), tiles(piece)) * tiles(D) >= (1 << 23)) return NOVAQ_ENOTSUP;
  return NOVAQ_OK;
}

int check_loss(const void* x, int x_dtype, int64_t N, int64_t D, const void* w, int w_dtype,
               const float* w_scale, int64_t V, const void* targets, int bits, int reduction) {
  if (!plain_float(x_dtype)) return NOVAQ_EDTYPE;
  int rc = check_table(w_dtype, w_scale, V, D);
  if (rc != NOVAQ_OK) return rc;
  if (N < 0 || reduction < NOVAQ_REDUCE_NONE || reduction > NOVAQ_REDUCE_SUM) return NOVAQ_EINVAL;
  rc = check_loss_sizes(N, V, D);
  if (rc != NOVAQ_OK) return rc;
  rc = check_ids(targets, bits);
  if (rc != NOVAQ_OK) return rc;
  if (!w || (N > 0 && (!x || !targets))) return NOVAQ_EINVAL;
  if (!aligned(x, 16) || !aligned(w, 16)) return NOVAQ_EALIGN;
  return NOVAQ_OK;
}

unsigned float_size(int dt) { return dt == NOVAQ_F64 ? 8u : dt == F32 ? 4u : 2u; }

// NOVAQ_EINVAL where a clipped gradient's bytes are another one's as well, or are
// read as another gradient (or as its own, but not in place) while they are written:
// workgroups would race on them.
int check_outputs(const novaq_gradient* list, int64_t count) {
  struct Span {
    uintptr_t from, to;
    bool written;
  };
  Span few[256];  // (of up to 128 gradients: no allocation)
  std::unique_ptr<Span[]> many;
  Span* span = few;
  if (count > 128) {
    many.reset(count < INT ? new (std::nothrow) Span[2 * count] : nullptr);
    span = many.get();
    if (!span) return NOVAQ_ESCRATCH;
  }
  int64_t spans = 0;
  for (int64_t i = 0; i < count; ++i) {
    const novaq_gradient& g = list[i];
    if (g.n == 0 || !g.out) continue;
    const unsigned gb = float_size(g.grad_dtype), ob = float_size(g.out_dtype);
    const uintptr_t in = reinterpret_cast<uintptr_t>(g.grad), out = reinterpret_cast<uintptr_t>(g.out);
    span[spans++] = Span{out, out + (uintptr_t)g.n * ob, true};
    if (in != out || gb != ob) span[spans++] = Span{in, in + (uintptr_t)g.n * gb, false};
  }
  std::sort(span, span + spans, [](const Span& a, const Span& b) { return a.from < b.from; });
  uintptr_t any = 0, written = 0;  // where the spans so far, and the written ones, end
  for (int64_t i = 0; i < spans; ++i) {
    if (span[i].from < (span[i].written ? any : written)) return NOVAQ_EINVAL;
    any = std::max(any, span[i].to);
    if (span[i].written) written = std::max(written, span[i].to);
  }
  return NOVAQ_OK;
}

}  // namespace

extern "C" {

int novaq_embedding(const void* ids, int id_bits, int64_t N, const void* table, int w_dtype,
                    const float* w_scale, int64_t V, int64_t D, float factor, void* out,
                    int out_dtype, void* stream) {
  if (!plain_float(out_dtype)) return NOVAQ_EDTYPE;
  int rc = check_table(w_dtype, w_scale, V, D);
  if (rc != NOVAQ_OK) return rc;
  if (N < 0) return NOVAQ_EINVAL;
  rc = check_ids(ids, id_bits);
  if (rc != NOVAQ_OK) return rc;
  if (N == 0) return NOVAQ_OK;
  if (!ids || !table || !out) return NOVAQ_EINVAL;
  if (!aligned(table, 16) || !aligned(out, 16)) return NOVAQ_EALIGN;
  return embedding_launch(ids, id_bits, N, table, w_dtype, w_scale, V, D, factor, out, out_dtype,
                          static_cast<hipStream_t>(stream));
}

size_t novaq_embedding_backward_workspace(int64_t N, int64_t V, int64_t D) {
  if (N <= 0 || N >= MOST_TOKENS || V <= 0 || V >= INT || D <= 0 || D > (1 << 20)) return 0;
  return embedding_backward_workspace(N, V, D);
}

int novaq_embedding_backward(const void* grad, int grad_dtype, const void* ids, int id_bits,
                             int64_t N, int64_t V, int64_t D, float factor, int accumulate,
                             void* grad_table, int out_dtype, void* workspace,
                             size_t workspace_bytes, void* stream) {
  if (!plain_float(grad_dtype) || !plain_float(out_dtype)) return NOVAQ_EDTYPE;
  int rc = check_table(out_dtype, nullptr, V, D);
  if (rc != NOVAQ_OK) return rc;
  if (N < 0) return NOVAQ_EINVAL;
  if (N >= MOST_TOKENS) return NOVAQ_ENOTSUP;
  rc = check_ids(ids, id_bits);
  if (rc != NOVAQ_OK) return rc;
  if (!grad_table || (N > 0 && (!grad || !ids))) return NOVAQ_EINVAL;
  if (!aligned(grad, 16) || !aligned(grad_table, 16) || !aligned(workspace, 16)) return NOVAQ_EALIGN;
  if (N > 0 && (!workspace || workspace_bytes < embedding_backward_workspace(N, V, D)))
    return NOVAQ_EINVAL;
  return embedding_backward_launch(grad, grad_dtype, ids, id_bits, N, V, D, factor, accumulate,
                                   grad_table, out_dtype, workspace,
                                   static_cast<hipStream_t>(stream));
}

size_t novaq_linear_cross_entropy_workspace(int64_t N, int64_t D, int64_t V, int x_dtype,
                                            int w_dtype) {
  if (N <= 0 || !plain_float(x_dtype) || check_table(w_dtype, nullptr, V, D) != NOVAQ_OK ||
      check_loss_sizes(N, V, D) != NOVAQ_OK)
    return 256;
  return vocab_loss_workspace(N, D, V, x_dtype, w_dtype, false);
}

size_t novaq_linear_cross_entropy_backward_workspace(int64_t N, int64_t D, int64_t V, int x_dtype,
                                                     int w_dtype) {
  if (N <= 0 || !plain_float(x_dtype) || check_table(w_dtype, nullptr, V, D) != NOVAQ_OK ||
      check_loss_sizes(N, V, D) != NOVAQ_OK)
    return 256;
  return vocab_loss_workspace(N, D, V, x_dtype, w_dtype, true);
}

int novaq_linear_cross_entropy(const void* x, int x_dtype, int64_t N, int64_t D, const void* w_q,
                               int w_dtype, const float* w_scale, int64_t V, const void* targets,
                               int target_bits, int64_t ignore_index, int reduction, float* loss,
                               float* lse, void* workspace, size_t workspace_bytes,
                               void* stream) {
  const int rc = check_loss(x, x_dtype, N, D, w_q, w_dtype, w_scale, V, targets, target_bits,
                            reduction);
  if (rc != NOVAQ_OK) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (N == 0) {
    if (reduction == NOVAQ_REDUCE_NONE) return NOVAQ_OK;
    return loss ? fill_u32_launch(reinterpret_cast<uint32_t*>(loss), 0u, 1, st) : NOVAQ_EINVAL;
  }
  if (!loss || !lse || !workspace) return NOVAQ_EINVAL;
  if (!aligned(workspace, 16)) return NOVAQ_EALIGN;
  if (workspace_bytes < vocab_loss_workspace(N, D, V, x_dtype, w_dtype, false)) return NOVAQ_EINVAL;
  return vocab_loss_launch(x, x_dtype, N, D, w_q, w_dtype, w_scale, V, targets, target_bits,
                           ignore_index, reduction, loss, lse, workspace, st);
}

int novaq_linear_cross_entropy_backward(const void* x, int x_dtype, int64_t N, int64_t D,
                                        const void* w_q, int w_dtype, const float* w_scale,
                                        int64_t V, const void* targets, int target_bits,
                                        int64_t ignore_index, int reduction, const float* grad,
                                        const float* lse, void* grad_input, void* grad_weight,
                                        int gw_dtype, void* workspace, size_t workspace_bytes,
                                        void* stream) {
  const int rc = check_loss(x, x_dtype, N, D, w_q, w_dtype, w_scale, V, targets, target_bits,
                            reduction);
  if (rc != NOVAQ_OK) return rc;
  if (!plain_float(gw_dtype)) return NOVAQ_EDTYPE;
  if (!aligned(grad_input, 16) || !aligned(grad_weight, 16) || !aligned(workspace, 16))
    return NOVAQ_EALIGN;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (!grad_input && !grad_weight) return NOVAQ_OK;
  if (N == 0)  // an empty sum (no rows add nothing: the lookup's gradient of no tokens)
    return grad_weight ? embedding_backward_launch(nullptr, F32, nullptr, 32, 0, V, D, 1.0f, 0,
                                                   grad_weight, gw_dtype, nullptr, st)
                       : NOVAQ_OK;
  if (!lse || !workspace) return NOVAQ_EINVAL;
  if (workspace_bytes < vocab_loss_workspace(N, D, V, x_dtype, w_dtype, true)) return NOVAQ_EINVAL;
  return vocab_loss_backward_launch(x, x_dtype, N, D, w_q, w_dtype, w_scale, V, targets,
                                    target_bits, ignore_index, reduction, grad, lse, grad_input,
                                    grad_weight, gw_dtype, workspace, st);
}

size_t novaq_clip_grad_norm_workspace(int64_t count) {
  return clip_grad_norm_workspace(count < 0 ? 0 : count);
}

int novaq_clip_grad_norm(const novaq_gradient* list, int64_t count, double max_norm, double eps,
                         float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  if (count < 0 || (count > 0 && !list) || !norm || !workspace) return NOVAQ_EINVAL;
  if (!(max_norm >= 0.0) || !(eps >= 0.0)) return NOVAQ_EINVAL;
  for (int64_t i = 0; i < count; ++i) {
    const novaq_gradient& g = list[i];
    const bool has_out = g.out != nullptr;
    if (!(plain_float(g.grad_dtype) || g.grad_dtype == NOVAQ_F64)) return NOVAQ_EDTYPE;
    if (has_out && !(plain_float(g.out_dtype) || g.out_dtype == NOVAQ_F64)) return NOVAQ_EDTYPE;
    if (g.n < 0 || g.n > INT64_MAX / 16 || (g.n > 0 && !g.grad)) return NOVAQ_EINVAL;
    if (!aligned(g.grad, float_size(g.grad_dtype)) ||
        (has_out && !aligned(g.out, float_size(g.out_dtype))))
      return NOVAQ_EALIGN;
  }
  if (!aligned(workspace, 16) || !aligned(norm, 4)) return NOVAQ_EALIGN;
  if (workspace_bytes < clip_grad_norm_workspace(count)) return NOVAQ_EINVAL;
  const int rc = check_outputs(list, count);
  if (rc != NOVAQ_OK) return rc;
  return clip_grad_norm_launch(list, count, max_norm, eps, norm, workspace,
                               static_cast<hipStream_t>(stream));
}

}  // extern "C"
