/* The C-ABI library's host code under AddressSanitizer and
 * UndefinedBehaviorSanitizer: every entry point's argument checks, including
 * sizes at the edge of int64 that must be rejected before any size
 * arithmetic can overflow.  Every call here is answered on the host; none
 * reaches the device (the pointers are placeholders that are never
 * dereferenced), so the checker runs without a GPU. */
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "argcases.h"

static int sample_capi(const void* a, int b, int64_t c, int64_t d, int64_t e, const int32_t* f,
                       int64_t g, int64_t h, const uint32_t* i, int64_t j, const float* k,
                       const gtp_sampler_params* l, const uint8_t* m, int64_t n, int64_t* o,
                       float* p, float* q, int32_t* r, float* s, int32_t* t, int32_t* u) {
  return gtp_sample_rows(a, b, c, d, e, f, g, h, i, j, k, l, m, n, o, p, q, r, s, t, u, NULL, 0,
                         NULL);
}

static int sample_noalloc(const void* a, int b, int64_t c, int64_t d, int64_t e, const int32_t* f,
                          int64_t g, int64_t h, const uint32_t* i, int64_t j, const float* k,
                          const gtp_sampler_params* l, const uint8_t* m, int64_t n, int64_t* o,
                          float* p, float* q, int32_t* r, float* s, int32_t* t, int32_t* u) {
  return gtp_sample_rows_noalloc(a, b, c, d, e, f, g, h, i, j, k, l, m, n, o, p, q, r, s, t, u,
                                 NULL);
}

static int logprob_capi(const void* a, int b, int64_t c, int64_t d, int64_t e, const void* f,
                        int g, float* h, float* i, int32_t* j) {
  return gtp_logprob_entropy_rows(a, b, c, d, e, f, g, h, i, j, NULL);
}

/* Token losses from hidden states, the embedding and the clipping: one field
 * after another out of range, sizes whose products would overflow. */
static void training_step_cases(void) {
  const int I = GTP_ERR_INVALID_ARGUMENT, X = GTP_ERR_UNSUPPORTED, OK = GTP_OK;
  const char* w = "training step";
  const int64_t M = INT64_MAX;
  void* p = PH(void*);
  float* f = PH(float*);
  int64_t* c = PH(int64_t*);
  const gtp_linear_rows good = {p, p, p, GTP_DTYPE_BF16, 1, 0, 0, 2, 8, 8, 64, 1000,
                                512, 64, 64, 8, 1};
  const size_t fwd = gtp_linear_logprob_workspace_bytes(&good);
  const size_t bwd = gtp_linear_logprob_backward_workspace_bytes(&good);
  EXPECT_RC(w, fwd > 0 && bwd > 0, 1);
  EXPECT_RC(w, gtp_linear_logprob_rows(NULL, f, f, NULL, NULL, NULL, p, fwd, NULL), I);
  EXPECT_RC(w, gtp_linear_logprob_rows(&good, NULL, f, NULL, NULL, NULL, p, fwd, NULL), I);
  EXPECT_RC(w, gtp_linear_logprob_rows(&good, f, f, f, NULL, NULL, p, fwd, NULL), I);
  EXPECT_RC(w, gtp_linear_logprob_rows(&good, f, f, NULL, NULL, NULL, NULL, fwd, NULL), I);
  EXPECT_RC(w, gtp_linear_logprob_rows(&good, f, f, NULL, NULL, NULL, p, fwd - 1, NULL), I);
  EXPECT_RC(w, gtp_linear_logprob_backward(&good, NULL, f, NULL, p, p, p, bwd, NULL), I);
  EXPECT_RC(w, gtp_linear_logprob_backward(&good, f, NULL, c, p, p, p, bwd, NULL), I);
  EXPECT_RC(w, gtp_linear_logprob_backward(&good, f, f, NULL, p, p, p, bwd - 1, NULL), I);
#define LINEAR(field, value, rc)                                                          \
  do {                                                                                    \
    gtp_linear_rows r_ = good;                                                            \
    r_.field = value;                                                                     \
    EXPECT_RC(w, gtp_linear_logprob_rows(&r_, f, f, NULL, NULL, NULL, p, SIZE_MAX, NULL), rc); \
    EXPECT_RC(w, gtp_linear_logprob_backward(&r_, f, f, NULL, p, p, p, SIZE_MAX, NULL), rc);   \
    EXPECT_RC(w, gtp_linear_logprob_workspace_bytes(&r_) == 0, 1);                        \
    EXPECT_RC(w, gtp_linear_logprob_backward_workspace_bytes(&r_) == 0, 1);               \
  } while (0)
  LINEAR(hidden, NULL, I);
  LINEAR(weight, NULL, I);
  LINEAR(targets, NULL, I);
  LINEAR(B, -1, I);
  LINEAR(S, -1, I);
  LINEAR(T, 9, I);
  LINEAR(K, 0, I);
  LINEAR(V, 0, I);
  LINEAR(hidden_batch_stride, -1, I);
  LINEAR(target_row_stride, -1, I);
  LINEAR(weight_stride, 63, I);
  LINEAR(dtype, GTP_DTYPE_F32, X);
  LINEAR(weight_stride, 68, X);
  LINEAR(weight_stride, M - 7, X);
  LINEAR(weight, (void*)(uintptr_t)0x18, X);
  LINEAR(B, M, X);
  LINEAR(S, M, X);
  LINEAR(V, M, X);
  LINEAR(V, 0x7FFFFFFF, X);
#undef LINEAR

  EXPECT_RC(w, gtp_embedding_rows(p, 1, 4, M, p, 1, 10, 8, 8, 1.0f, NULL, NULL), I);
  EXPECT_RC(w, gtp_embedding_rows(p, 1, 4, -1, p, 1, 10, 8, 8, 1.0f, p, NULL), I);
  EXPECT_RC(w, gtp_embedding_rows(p, 1, 4, 1, p, 1, 10, 8, 7, 1.0f, p, NULL), I);
  EXPECT_RC(w, gtp_embedding_rows(p, 1, 4, 1, p, 1, 10, 8, M, 1.0f, p, NULL), X);
  EXPECT_RC(w, gtp_embedding_rows(p, 1, M, 1, p, 1, 10, 8, 8, 1.0f, p, NULL), X);
  EXPECT_RC(w, gtp_embedding_rows(p, 1, 4, 1, p, 1, M, 8, 8, 1.0f, p, NULL), X);
  EXPECT_RC(w, gtp_embedding_rows(p, 1, 4, 1, p, 1, 10, M, M, 1.0f, p, NULL), X);
  EXPECT_RC(w, gtp_embedding_rows(NULL, 1, 0, 1, NULL, 1, 10, 8, 8, 1.0f, NULL, NULL), OK);
  EXPECT_RC(w, gtp_embedding_order_bytes(M, 10) == 0, 1);
  EXPECT_RC(w, gtp_embedding_order_bytes(4, M) == 0, 1);
  EXPECT_RC(w, gtp_embedding_backward_workspace_bytes(1, M, 10, 8) == 0, 1);
  EXPECT_RC(w, gtp_embedding_backward_workspace_bytes(1, 4, M, M) == 0, 1);
  EXPECT_RC(w, gtp_embedding_backward_ordered_workspace_bytes(1, 4, M) == 0, 1);
  EXPECT_RC(w, gtp_embedding_rows_ordered(p, 1, 4, 1, p, 1, 10, 8, 8, 1.0f, p, -1, p, 3, NULL), I);
  EXPECT_RC(w, gtp_embedding_rows_ordered(p, 1, 4, 1, p, 1, 10, 8, 8, 1.0f, p, -1, NULL, SIZE_MAX,
                                          NULL), I);
  EXPECT_RC(w, gtp_embedding_backward(p, 1, 4, 1, p, 1, 8, 10, 8, 1.0f, -1, 0, p, p, 3, NULL), I);
  EXPECT_RC(w, gtp_embedding_backward(p, 1, 4, 1, p, 1, M, 10, 8, 1.0f, -1, 0, p, p, SIZE_MAX,
                                      NULL), X);
  EXPECT_RC(w, gtp_embedding_backward(p, 1, 4, 1, p, 1, 8, M, M, 1.0f, -1, 0, p, p, SIZE_MAX,
                                      NULL), X);
  EXPECT_RC(w, gtp_embedding_backward_ordered(p, 3, 4, p, 1, 8, 10, 8, 1.0f, 0, p, p, SIZE_MAX,
                                              NULL), I);
  EXPECT_RC(w, gtp_embedding_backward_ordered(p, SIZE_MAX, 4, p, 1, M, 10, 8, 1.0f, 0, p, p,
                                              SIZE_MAX, NULL), X);

  void* t[2] = {p, PH(void*)};
  int64_t n[2] = {8, 8};
  int32_t d[2] = {GTP_DTYPE_F32, GTP_DTYPE_BF16};
  EXPECT_RC(w, gtp_grad_norm((const void* const*)t, n, d, 2, 2, f, p, 8, NULL), I);
  EXPECT_RC(w, gtp_grad_norm((const void* const*)t, n, d, -1, 2, f, p, 64, NULL), I);
  EXPECT_RC(w, gtp_grad_norm(NULL, n, d, 2, 2, f, p, 64, NULL), I);
  EXPECT_RC(w, gtp_clip_grads(t, n, d, 2, NULL, 1.0f, NULL), I);
  n[1] = -1;
  EXPECT_RC(w, gtp_grad_norm((const void* const*)t, n, d, 2, 2, f, p, 64, NULL), I);
  n[1] = M;
  EXPECT_RC(w, gtp_grad_norm((const void* const*)t, n, d, 2, 2, f, p, 64, NULL), X);
  EXPECT_RC(w, gtp_clip_grads(t, n, d, 2, f, 1.0f, NULL), X);
  EXPECT_RC(w, gtp_grad_norm_workspace_bytes((const void* const*)t, n, d, 2) == 0, 1);
  n[1] = 8;
  d[1] = 7;
  EXPECT_RC(w, gtp_clip_grads(t, n, d, 2, f, 1.0f, NULL), I);
}

int main(void) {
  const int I = GTP_ERR_INVALID_ARGUMENT, X = GTP_ERR_UNSUPPORTED, OK = GTP_OK;
  const char* w = "capi";
  sample_arg_cases(sample_capi, "capi sampler");
  sample_arg_cases(sample_noalloc, "capi sampler noalloc");
  logprob_arg_cases(logprob_capi, "capi logprob");

  const void* L = PH(const void*);
  const void* T = PH(const void*);
  const float* F = PH(const float*);
  float* o = PH(float*);
  void* g = PH(void*);
  const gtp_sampler_params topp = {0.7f, 0, 0.9f, 1.0f};

  /* the workspace query: zero for every call that cannot run */
  {
    int32_t rt = 0, sl = 0;
    EXPECT_RC(w, gtp_sample_route(1, 4, 151936, 1, 0, 0, NULL, 0, &rt, &sl), I);
    EXPECT_RC(w, gtp_sample_route(1, 4, 151936, 1, 0, 0, &topp, 0, NULL, &sl), I);
    EXPECT_RC(w, gtp_sample_route(1, 0, 151936, 1, 0, 0, &topp, 0, &rt, &sl), I);
    EXPECT_RC(w, gtp_sample_route(1, 4, 0, 1, 0, 0, &topp, 0, &rt, &sl), I);
    EXPECT_RC(w, gtp_sample_route(1, 4, 151936, 1, -1, 0, &topp, 0, &rt, &sl), I);
    EXPECT_RC(w, gtp_sample_route(7, 4, 151936, 1, 0, 0, &topp, 0, &rt, &sl), I);
    EXPECT_RC(w, gtp_sample_route(1, 4, INT64_MAX, 1, 0, 0, &topp, 0, &rt, &sl), X);
    EXPECT_RC(w, gtp_sample_route(1, INT64_MAX, 151936, 1, 0, 0, &topp, 0, &rt, &sl), X);
    EXPECT_RC(w, gtp_sample_route(1, 4, 151936, 1, 0, 0, &topp, SIZE_MAX, &rt, NULL), OK);
    EXPECT_RC(w, rt, GTP_ROUTE_TOPP_SPLIT);
  }
  EXPECT_RC(w, (int)gtp_sample_workspace_bytes(1, 4, 100, NULL), 0);
  EXPECT_RC(w, (int)gtp_sample_workspace_bytes(1, 0, 151936, &topp), 0);
  EXPECT_RC(w, (int)gtp_sample_workspace_bytes(1, 4, 0, &topp), 0);
  EXPECT_RC(w, (int)(gtp_sample_workspace_bytes(1, INT64_MAX, 151936, &topp) != 0), 0);
  EXPECT_RC(w, (int)(gtp_sample_workspace_bytes(1, 64, INT64_MAX, &topp) != 0), 0);
  /* top-p rows of a large batch (and fp32 rows): one workgroup per row, no
     workspace */
  EXPECT_RC(w, (int)gtp_sample_workspace_bytes(1, 256, 151936, &topp), 0);
  EXPECT_RC(w, (int)gtp_sample_workspace_bytes(0, 64, 151936, &topp), 0);
  /* bf16 top-p rows of a small batch, split over S = 4 workgroups per row
     (no device here: 256 CUs assumed): 16 KB of counters, 64 x 4 headers of
     64 bytes, 64 x 4 slots of 64 KB */
  EXPECT_RC(w, (int)gtp_sample_workspace_bytes(1, 64, 151936, &topp), 16384 + 16384 + 64 * 4 * 65536);
  /* the library's own workspace is bounded: 8192 fp32 rows of 2^18 with
     top-k 128 merge more candidate lists than it holds */
  {
    const gtp_sampler_params topk = {1.0f, 128, 1.0f, 1.0f};
    EXPECT_RC(w, (int)(gtp_sample_workspace_bytes(0, 8192, 1 << 18, &topk) > GTP_NOALLOC_SCRATCH_BYTES), 1);
    EXPECT_RC(w, gtp_sample_rows_noalloc(L, 0, 8192, 1 << 18, 1 << 18, NULL, 0, 0, NULL, 0, F, &topk,
                                         NULL, 0, PH(int64_t*), NULL, NULL, NULL, NULL, NULL, NULL,
                                         NULL),
              X);
  }

  EXPECT_RC(w, gtp_lse_partial_rows(L, 1, -1, 10, 10, 0, T, 0, o, 0, NULL), I);
  EXPECT_RC(w, gtp_lse_partial_rows(L, 1, 4, 0, 10, 0, T, 0, o, 0, NULL), I);
  EXPECT_RC(w, gtp_lse_partial_rows(L, 1, 4, 10, 9, 0, T, 0, o, 0, NULL), I);
  EXPECT_RC(w, gtp_lse_partial_rows(L, 1, 4, 10, 10, -1, T, 0, o, 0, NULL), I);
  EXPECT_RC(w, gtp_lse_partial_rows(NULL, 1, 4, 10, 10, 0, T, 0, o, 0, NULL), I);
  EXPECT_RC(w, gtp_lse_partial_rows(L, 1, 4, 10, 10, 0, T, 0, NULL, 0, NULL), I);
  EXPECT_RC(w, gtp_lse_partial_rows(L, 7, 4, 10, 10, 0, T, 0, o, 0, NULL), I);
  EXPECT_RC(w, gtp_lse_partial_rows(L, 1, INT64_MAX, 10, 10, 0, T, 0, o, 0, NULL), X);
  EXPECT_RC(w, gtp_lse_partial_rows(NULL, 1, 0, 10, 10, 0, NULL, 0, NULL, 0, NULL), OK);

  EXPECT_RC(w, gtp_lse_finalize_rows(F, -1, o, NULL, NULL), I);
  EXPECT_RC(w, gtp_lse_finalize_rows(NULL, 4, o, NULL, NULL), I);
  EXPECT_RC(w, gtp_lse_finalize_rows(F, INT64_MAX, o, NULL, NULL), X);
  EXPECT_RC(w, gtp_lse_finalize_rows(NULL, 0, NULL, NULL, NULL), OK);

  EXPECT_RC(w, gtp_logprob_backward_rows(L, 1, -1, 10, 10, 0, T, 0, F, F, g, 10, NULL), I);
  EXPECT_RC(w, gtp_logprob_backward_rows(L, 1, 4, 10, 10, 0, T, 0, F, F, g, 9, NULL), I);
  EXPECT_RC(w, gtp_logprob_backward_rows(L, 1, 4, 10, 10, 0, T, 0, F, NULL, g, 10, NULL), I);
  EXPECT_RC(w, gtp_logprob_backward_rows(L, 1, 4, 10, 10, 0, T, 0, F, F, NULL, 10, NULL), I);
  EXPECT_RC(w, gtp_logprob_backward_rows(L, 8, 4, 10, 10, 0, T, 0, F, F, g, 10, NULL), I);
  EXPECT_RC(w, gtp_logprob_backward_rows(L, 1, INT64_MAX, 10, 10, 0, T, 0, F, F, g, 10, NULL), X);
  EXPECT_RC(w, gtp_logprob_backward_rows(NULL, 1, 0, 10, 10, 0, NULL, 0, NULL, NULL, NULL, 10,
                                         NULL),
            OK);

  uint16_t* h = PH(uint16_t*);
  EXPECT_RC(w, gtp_logprob_backward_split_rows(F, -1, 10, 10, 0, T, 0, F, F, h, h, 10, NULL), I);
  EXPECT_RC(w, gtp_logprob_backward_split_rows(F, 4, 10, 10, 0, T, 0, F, F, h, NULL, 10, NULL), I);
  EXPECT_RC(w, gtp_logprob_backward_split_rows(F, 4, 10, 10, 0, T, 0, F, F, h, h, 3, NULL), I);
  EXPECT_RC(w, gtp_logprob_backward_split_rows(F, INT64_MAX, 10, 10, 0, T, 0, F, F, h, h, 10,
                                               NULL),
            X);

  EXPECT_RC(w, gtp_graspo_loss_forward(F, F, F, NULL, 0, 0, 8, 0.8f, 1.2f, o, o, o, NULL), I);
  EXPECT_RC(w, gtp_graspo_loss_forward(F, F, F, NULL, 0, 4, 0, 0.8f, 1.2f, o, o, o, NULL), I);
  EXPECT_RC(w, gtp_graspo_loss_forward(F, NULL, F, NULL, 0, 4, 8, 0.8f, 1.2f, o, o, o, NULL), I);
  EXPECT_RC(w, gtp_graspo_loss_forward(F, F, F, NULL, 0, (int64_t)1 << 31, 8, 0.8f, 1.2f, o, o, o,
                                       NULL),
            X);
  EXPECT_RC(w, gtp_graspo_loss_backward(F, F, F, NULL, 0, F, F, -4, 8, 0.8f, 1.2f, o, NULL), I);
  EXPECT_RC(w, gtp_graspo_loss_backward(F, F, F, NULL, 0, NULL, F, 4, 8, 0.8f, 1.2f, o, NULL), I);
  /* B * T beyond int64, and beyond the launch grid */
  EXPECT_RC(w, gtp_graspo_loss_backward(F, F, F, NULL, 0, F, F, (int64_t)1 << 40, (int64_t)1 << 40,
                                        0.8f, 1.2f, o, NULL),
            X);
  EXPECT_RC(w, gtp_graspo_loss_backward(F, F, F, NULL, 0, F, F, 1, (int64_t)1 << 40, 0.8f, 1.2f,
                                        o, NULL),
            X);

  int64_t* ids = PH(int64_t*);
  uint8_t* fin = PH(uint8_t*);
  int32_t* flags = PH(int32_t*);
  EXPECT_RC(w, gtp_decode_update_rows(ids, NULL, -1, 2, 0, fin, NULL, 0, NULL, 0, 0, flags, NULL),
            I);
  EXPECT_RC(w, gtp_decode_update_rows(ids, NULL, 4, 2, 0, fin, NULL, 0, NULL, 0, -1, flags, NULL),
            I);
  EXPECT_RC(w, gtp_decode_update_rows(ids, NULL, 4, 2, 0, fin, NULL, 0, NULL, 0, 0, NULL, NULL),
            I);
  EXPECT_RC(w, gtp_decode_update_rows(NULL, NULL, 4, 2, 0, fin, NULL, 0, NULL, 0, 0, flags, NULL),
            I);
  EXPECT_RC(w, gtp_decode_update_rows(ids, NULL, 4, 2, 0, fin, ids, 5, NULL, 0, 5, flags, NULL),
            I);
  EXPECT_RC(w, gtp_decode_update_rows(ids, NULL, 4, 2, 0, fin, NULL, 0, fin, 3, 5, flags, NULL),
            I);
  EXPECT_RC(w, gtp_decode_update_rows(ids, NULL, INT64_MAX, 2, 0, fin, NULL, 0, NULL, 0, 0, flags,
                                      NULL),
            X);

  uint32_t* inexact = PH(uint32_t*);
  EXPECT_RC(w, gtp_f32_to_bf16_exact(F, -1, h, inexact, NULL), I);
  EXPECT_RC(w, gtp_f32_to_bf16_exact(F, 10, h, NULL, NULL), I);
  EXPECT_RC(w, gtp_f32_to_bf16_exact(NULL, 10, h, inexact, NULL), I);
  EXPECT_RC(w, gtp_f32_to_bf16_exact((const float*)(uintptr_t)0x14, INT64_MAX, h, inexact, NULL),
            X);
  EXPECT_RC(w, gtp_f32_to_bf16_exact(NULL, 0, NULL, inexact, NULL), OK);

  EXPECT_RC(w, gtp_time_next_launch(NULL, g), I);
  EXPECT_RC(w, gtp_time_next_launch(g, NULL), I);

  uint32_t* out = PH(uint32_t*);
  const void* A = (const void*)(uintptr_t)0x100;
  EXPECT_RC(w, gtp_stream_read_rows(A, -1, 16, 16, out, NULL), I);
  EXPECT_RC(w, gtp_stream_read_rows(A, 4, -16, 16, out, NULL), I);
  EXPECT_RC(w, gtp_stream_read_rows(A, 4, 32, 16, out, NULL), I);
  EXPECT_RC(w, gtp_stream_read_rows(A, 4, 32, 32, NULL, NULL), I);
  EXPECT_RC(w, gtp_stream_read_rows((const void*)(uintptr_t)0x104, 4, 32, 32, out, NULL), X);
  EXPECT_RC(w, gtp_stream_read_rows(A, 4, 24, 32, out, NULL), X);
  EXPECT_RC(w, gtp_stream_read_rows(A, INT64_MAX, 32, 32, out, NULL), X);
  EXPECT_RC(w, gtp_stream_read_rows(NULL, 0, 32, 32, NULL, NULL), OK);

  const uint16_t* HB = PH(const uint16_t*);
  const uint16_t* WB = (const uint16_t*)(uintptr_t)0x1000;
  void* wsp = PH(void*);
  const size_t wsz = gtp_lm_head_workspace_bytes(256, 1000);
  EXPECT_RC(w, wsz > 0, 1);
  EXPECT_RC(w, (int)gtp_lm_head_workspace_bytes(0, 1000), 0);
  EXPECT_RC(w, (int)gtp_lm_head_workspace_bytes(256, 0), 0);
  EXPECT_RC(w, (int)gtp_lm_head_workspace_bytes(INT64_MAX, 1000), 0);
  EXPECT_RC(w, gtp_lm_head_logprob_rows(HB, -1, 128, 128, WB, 1000, 128, T, 0, o, NULL, NULL, NULL,
                                        wsp, wsz, NULL), I);
  EXPECT_RC(w, gtp_lm_head_logprob_rows(HB, 256, 128, 128, WB, 0, 128, T, 0, o, NULL, NULL, NULL,
                                        wsp, wsz, NULL), I);
  EXPECT_RC(w, gtp_lm_head_logprob_rows(HB, 256, 0, 128, WB, 1000, 128, T, 0, o, NULL, NULL, NULL,
                                        wsp, wsz, NULL), I);
  EXPECT_RC(w, gtp_lm_head_logprob_rows(HB, 256, 128, 120, WB, 1000, 128, T, 0, o, NULL, NULL,
                                        NULL, wsp, wsz, NULL), I);
  EXPECT_RC(w, gtp_lm_head_logprob_rows(NULL, 256, 128, 128, WB, 1000, 128, T, 0, o, NULL, NULL,
                                        NULL, wsp, wsz, NULL), I);
  EXPECT_RC(w, gtp_lm_head_logprob_rows(HB, 256, 128, 128, WB, 1000, 128, NULL, 0, o, NULL, NULL,
                                        NULL, wsp, wsz, NULL), I);
  EXPECT_RC(w, gtp_lm_head_logprob_rows(HB, 256, 128, 128, WB, 1000, 128, T, 0, o, NULL, NULL,
                                        NULL, NULL, wsz, NULL), I);
  EXPECT_RC(w, gtp_lm_head_logprob_rows(HB, 256, 128, 128, WB, 1000, 128, T, 0, o, NULL, NULL,
                                        NULL, wsp, wsz - 1, NULL), I);
  EXPECT_RC(w, gtp_lm_head_logprob_rows(HB, 256, 192, 192, WB, 1000, 192, T, 0, o, NULL, NULL,
                                        NULL, wsp, wsz, NULL), X);  /* K % 128 */
  EXPECT_RC(w, gtp_lm_head_logprob_rows((const uint16_t*)(uintptr_t)0x18, 256, 128, 128, WB, 1000,
                                        128, T, 0, o, NULL, NULL, NULL, wsp, wsz, NULL), X);
  EXPECT_RC(w, gtp_lm_head_logprob_rows(HB, 256, 128, 1 << 22, WB, 1000, 128, T, 0, o, NULL, NULL,
                                        NULL, wsp, wsz, NULL), X);
  EXPECT_RC(w, gtp_lm_head_logprob_rows(HB, INT64_MAX, 128, 128, WB, 1000, 128, T, 0, o, NULL,
                                        NULL, NULL, wsp, wsz, NULL), X);
  EXPECT_RC(w, gtp_lm_head_logprob_rows(NULL, 0, 128, 128, NULL, 1000, 128, NULL, 0, NULL, NULL,
                                        NULL, NULL, NULL, 0, NULL), OK);

  float* LG = PH(float*);
  EXPECT_RC(w, gtp_lm_head_logprob_save_rows(HB, 256, 128, 128, WB, 1000, 128, T, 0, o, NULL,
                                             NULL, NULL, NULL, 256, wsp, wsz, NULL), I);
  EXPECT_RC(w, gtp_lm_head_logprob_save_rows(HB, 256, 128, 128, WB, 1000, 128, T, 0, o, NULL,
                                             NULL, NULL, LG, 255, wsp, wsz, NULL), I);
  EXPECT_RC(w, gtp_lm_head_logprob_save_rows(HB, 256, 128, 128, WB, 1000, 128, T, 0, o, NULL,
                                             NULL, NULL, (float*)(uintptr_t)0x1002, 256, wsp,
                                             wsz, NULL), X);
  EXPECT_RC(w, gtp_lm_head_logprob_save_rows(HB, 256, 128, 128, WB, 1000, 128, T, 0, o, NULL,
                                             NULL, NULL, LG, (int64_t)1 << 40, wsp, wsz, NULL), X);
  EXPECT_RC(w, gtp_lm_head_logprob_save_rows(HB, 256, 192, 192, WB, 1000, 192, T, 0, o, NULL,
                                             NULL, NULL, LG, 256, wsp, wsz, NULL), X);
  EXPECT_RC(w, gtp_lm_head_logprob_save_rows(HB, 256, 128, 128, WB, 1000, 128, T, 0, o, NULL,
                                             NULL, NULL, LG, 256, wsp, wsz - 1, NULL), I);
  EXPECT_RC(w, gtp_lm_head_logprob_save_rows(NULL, 0, 128, 128, NULL, 1000, 128, NULL, 0, NULL,
                                             NULL, NULL, NULL, NULL, 0, NULL, 0, NULL), OK);

  EXPECT_RC(w, gtp_softmax_grad_bf16_cols(F, 10, -1, 10, F, F, h, 10, NULL, 0, NULL), I);
  EXPECT_RC(w, gtp_softmax_grad_bf16_cols(F, 10, 4, 3, F, F, h, 10, NULL, 0, NULL), I);
  EXPECT_RC(w, gtp_softmax_grad_bf16_cols(F, 10, 4, 4, F, F, h, 3, NULL, 0, NULL), I);
  EXPECT_RC(w, gtp_softmax_grad_bf16_cols(F, 0, 4, 4, F, F, h, 4, NULL, 0, NULL), I);
  EXPECT_RC(w, gtp_softmax_grad_bf16_cols(F, 10, 4, 4, NULL, F, h, 4, NULL, 0, NULL), I);
  EXPECT_RC(w, gtp_softmax_grad_bf16_cols(F, 10, 4, 4, F, F, NULL, 4, NULL, 0, NULL), I);
  EXPECT_RC(w, gtp_softmax_grad_bf16_cols(F, 10, INT64_MAX, INT64_MAX, F, F, h, INT64_MAX, NULL, 0, NULL),
            X);
  EXPECT_RC(w, gtp_softmax_grad_bf16_cols(F, INT64_MAX, 4, 4, F, F, h, 4, NULL, 0, NULL), X);
  EXPECT_RC(w, gtp_softmax_grad_bf16_cols(NULL, 10, 0, 0, NULL, NULL, NULL, 0, NULL, 0, NULL), OK);
  /* the token-major output: its stride must hold V, and bound N * stride */
  EXPECT_RC(w, gtp_softmax_grad_bf16_cols(F, 10, 4, 4, F, F, NULL, 0, h, 9, NULL), I);
  EXPECT_RC(w, gtp_softmax_grad_bf16_cols(F, 10, 4, 4, F, F, h, 4, h, 9, NULL), I);
  EXPECT_RC(w, gtp_softmax_grad_bf16_cols(F, 10, 4, 4, F, F, NULL, 0, h, INT64_MAX, NULL), X);

  training_step_cases();

  EXPECT_RC(w, strstr(gtp_version(), "gfx950") != NULL, 1);

  printf("C-ABI sanitizer checks: %d run, %d failed\n", g_checks, g_fails);
  return g_fails ? 1 : 0;
}
