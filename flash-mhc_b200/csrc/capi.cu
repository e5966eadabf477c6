// C ABI (include/flashmhc.h): argument validation, path selection, launch,
// error reporting.  No device memory is allocated here.
#include <cstdarg>
#include <cstdio>

#include "../../include/flashmhc.h"
#include "fmhc_launch.h"
#include "k1_tc.h"

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int ok() {
  g_err[0] = '\0';
  return FMHC_OK;
}

int check_launch(const char *what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(FMHC_ERR_LAUNCH, "%s: launch failed: %s", what, cudaGetErrorString(e));
  return ok();
}

bool aligned(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Largest bf16 chunk width v in {8,4,2,1} with C % v == 0 and every bf16
// pointer aligned to 2*v bytes.
int pick_vec(int64_t C, std::initializer_list<const void *> ptrs) {
  for (int v : {8, 4, 2, 1}) {
    if (C % v) continue;
    bool good = true;
    for (const void *p : ptrs) good = good && aligned(p, uintptr_t(2 * v));
    if (good) return v;
  }
  return 0;
}

int check_streams(const char *what, int64_t T, int64_t n, int64_t C) {
  if (T < 0) return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: T must be >= 0 (got %lld)", what, (long long)T);
  if (n != 4) return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: supports n=4 only (got n=%lld)", what, (long long)n);
  if (C < 1 || C > (int64_t(1) << 28))
    return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: C must be in [1, 2^28] (got %lld)", what, (long long)C);
  return FMHC_OK;
}

#define FMHC_REQUIRE_PTR(what, p) \
  if ((p) == nullptr) return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: %s is NULL", what, #p)
#define FMHC_REQUIRE_ALIGN16(what, p) \
  if (!aligned((p), 16)) return fail(FMHC_ERR_ALIGNMENT, "%s: %s must be 16-byte aligned", what, #p)
#define FMHC_REQUIRE_ALIGN2(what, p) \
  if (!aligned((p), 2)) return fail(FMHC_ERR_ALIGNMENT, "%s: %s must be 2-byte aligned", what, #p)

}  // namespace

namespace fmhc {
// Records `msg` as this thread's fmhc_last_error() text and returns `code`.
int set_last_error(int code, const char *msg) { return fail(code, "%s", msg); }
}  // namespace fmhc

extern "C" {

const char *fmhc_last_error(void) { return g_err; }

const char *fmhc_version(void) { return "flashmhc-sm100 0.1.0"; }

int fmhc_check_device_error(int *code) {
  if (code == nullptr) return fail(FMHC_ERR_INVALID_ARGUMENT, "fmhc_check_device_error: code is NULL");
  if (cudaDeviceSynchronize() != cudaSuccess)
    return fail(FMHC_ERR_CUDA, "fmhc_check_device_error: %s", cudaGetErrorString(cudaGetLastError()));
  unsigned v = 0;
  unsigned v8 = 0;
  if (fmhc::read_device_error(&v) || fmhc::read_int8_linear_error(&v8))
    return fail(FMHC_ERR_CUDA, "fmhc_check_device_error: symbol copy failed");
  *code = int(v != 0 ? v : v8);
  return ok();
}

int fmhc_k3_fwd(const void *x, const float *h_pre, void *out, int64_t T, int64_t n, int64_t C,
                void *stream) {
  const char *w = "fmhc_k3_fwd";
  if (int e = check_streams(w, T, n, C)) return e;
  if (T == 0) return ok();
  FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, h_pre); FMHC_REQUIRE_PTR(w, out);
  FMHC_REQUIRE_ALIGN16(w, h_pre);
  FMHC_REQUIRE_ALIGN2(w, x); FMHC_REQUIRE_ALIGN2(w, out);
  const int vec = pick_vec(C, {x, out});
  fmhc::launch_k3_fwd(x, h_pre, out, T, int(C), vec, (cudaStream_t)stream);
  return check_launch(w);
}

int fmhc_k3_bwd(const void *grad_out, const void *x, const float *h_pre, void *grad_x,
                float *grad_h, int64_t T, int64_t n, int64_t C, void *stream) {
  const char *w = "fmhc_k3_bwd";
  if (int e = check_streams(w, T, n, C)) return e;
  if (T == 0) return ok();
  FMHC_REQUIRE_PTR(w, grad_out); FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, h_pre);
  FMHC_REQUIRE_PTR(w, grad_h);
  FMHC_REQUIRE_ALIGN16(w, h_pre); FMHC_REQUIRE_ALIGN16(w, grad_h);
  FMHC_REQUIRE_ALIGN2(w, grad_out); FMHC_REQUIRE_ALIGN2(w, x);
  if (grad_x) FMHC_REQUIRE_ALIGN2(w, grad_x);
  const int vec = grad_x ? pick_vec(C, {grad_out, x, grad_x}) : pick_vec(C, {grad_out, x});
  fmhc::launch_k3_bwd(grad_out, x, h_pre, grad_x, grad_h, T, int(C), vec, (cudaStream_t)stream);
  return check_launch(w);
}

int fmhc_mhc_grad_x_combine(const void *gx1, const void *grad_li, const float *h_pre,
                            const void *gx4, void *grad_x, int64_t T, int64_t n, int64_t C,
                            void *stream) {
  const char *w = "fmhc_mhc_grad_x_combine";
  if (int e = check_streams(w, T, n, C)) return e;
  if (T == 0) return ok();
  FMHC_REQUIRE_PTR(w, gx1); FMHC_REQUIRE_PTR(w, grad_li); FMHC_REQUIRE_PTR(w, h_pre);
  FMHC_REQUIRE_PTR(w, grad_x);
  FMHC_REQUIRE_ALIGN16(w, h_pre);
  FMHC_REQUIRE_ALIGN2(w, gx1); FMHC_REQUIRE_ALIGN2(w, grad_li); FMHC_REQUIRE_ALIGN2(w, grad_x);
  if (gx4) FMHC_REQUIRE_ALIGN2(w, gx4);
  const int vec = gx4 ? pick_vec(C, {gx1, grad_li, gx4, grad_x}) : pick_vec(C, {gx1, grad_li, grad_x});
  fmhc::launch_grad_x_combine(gx1, grad_li, h_pre, gx4, grad_x, T, int(C), vec,
                              (cudaStream_t)stream);
  return check_launch(w);
}

int fmhc_mhc_grad_x_combine_post(const void *gx1, const void *grad_li, const float *h_pre,
                                 const void *grad_out, const float *H, void *grad_x, int64_t T,
                                 int64_t n, int64_t C, void *stream) {
  const char *w = "fmhc_mhc_grad_x_combine_post";
  if (int e = check_streams(w, T, n, C)) return e;
  if (T == 0) return ok();
  FMHC_REQUIRE_PTR(w, gx1); FMHC_REQUIRE_PTR(w, grad_li); FMHC_REQUIRE_PTR(w, h_pre);
  FMHC_REQUIRE_PTR(w, grad_out); FMHC_REQUIRE_PTR(w, H); FMHC_REQUIRE_PTR(w, grad_x);
  FMHC_REQUIRE_ALIGN16(w, h_pre); FMHC_REQUIRE_ALIGN16(w, H);
  FMHC_REQUIRE_ALIGN2(w, gx1); FMHC_REQUIRE_ALIGN2(w, grad_li); FMHC_REQUIRE_ALIGN2(w, grad_out);
  FMHC_REQUIRE_ALIGN2(w, grad_x);
  const int vec = pick_vec(C, {gx1, grad_li, grad_out, grad_x});
  fmhc::launch_grad_x_combine_post(gx1, grad_li, h_pre, grad_out, H, grad_x, T, int(C), vec,
                                   (cudaStream_t)stream);
  return check_launch(w);
}

int fmhc_k4_fwd(const void *x, const void *lo, const float *H, const float *h_post, void *out,
                int64_t T, int64_t n, int64_t C, void *stream) {
  const char *w = "fmhc_k4_fwd";
  if (int e = check_streams(w, T, n, C)) return e;
  if (T == 0) return ok();
  FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, lo); FMHC_REQUIRE_PTR(w, H);
  FMHC_REQUIRE_PTR(w, h_post); FMHC_REQUIRE_PTR(w, out);
  FMHC_REQUIRE_ALIGN16(w, H); FMHC_REQUIRE_ALIGN16(w, h_post);
  FMHC_REQUIRE_ALIGN2(w, x); FMHC_REQUIRE_ALIGN2(w, lo); FMHC_REQUIRE_ALIGN2(w, out);
  const int vec = pick_vec(C, {x, lo, out});
  fmhc::launch_k4_fwd(x, lo, H, h_post, out, T, int(C), vec, (cudaStream_t)stream);
  return check_launch(w);
}

int fmhc_k4_bwd(const void *grad_out, const void *x, const void *lo, const float *H,
                const float *h_post, void *grad_x, void *grad_lo, float *grad_H,
                float *grad_hp, int64_t T, int64_t n, int64_t C, void *stream) {
  const char *w = "fmhc_k4_bwd";
  if (int e = check_streams(w, T, n, C)) return e;
  if (T == 0) return ok();
  FMHC_REQUIRE_PTR(w, grad_out); FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, lo);
  FMHC_REQUIRE_PTR(w, H); FMHC_REQUIRE_PTR(w, h_post);
  FMHC_REQUIRE_PTR(w, grad_lo); FMHC_REQUIRE_PTR(w, grad_H); FMHC_REQUIRE_PTR(w, grad_hp);
  FMHC_REQUIRE_ALIGN16(w, H); FMHC_REQUIRE_ALIGN16(w, h_post);
  FMHC_REQUIRE_ALIGN16(w, grad_H); FMHC_REQUIRE_ALIGN16(w, grad_hp);
  FMHC_REQUIRE_ALIGN2(w, grad_out); FMHC_REQUIRE_ALIGN2(w, x); FMHC_REQUIRE_ALIGN2(w, lo);
  FMHC_REQUIRE_ALIGN2(w, grad_lo);
  if (grad_x) FMHC_REQUIRE_ALIGN2(w, grad_x);  // NULL: parameter gradients only
  const int vec = grad_x ? pick_vec(C, {grad_out, x, lo, grad_x, grad_lo})
                         : pick_vec(C, {grad_out, x, lo, grad_lo});
  fmhc::launch_k4_bwd(grad_out, x, lo, H, h_post, grad_x, grad_lo, grad_H, grad_hp, T, int(C),
                      vec, (cudaStream_t)stream);
  return check_launch(w);
}

static int check_k1(const char *w, int64_t T, int64_t nC, int64_t D) {
  if (T < 0) return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: T must be >= 0 (got %lld)", w, (long long)T);
  if (nC < 1 || nC > (int64_t(1) << 28))
    return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: nC must be in [1, 2^28] (got %lld)", w, (long long)nC);
  if (D < 1 || D > 32)
    return fail(FMHC_ERR_UNSUPPORTED, "%s: D (projection width) must be in [1, 32] (got %lld)", w,
                (long long)D);
  return FMHC_OK;
}

int fmhc_k1_fwd(const void *x, const void *W, void *out, float *inv_rms, int64_t T, int64_t nC,
                int64_t D, void *stream) {
  const char *w = "fmhc_k1_fwd";
  if (int e = check_k1(w, T, nC, D)) return e;
  if (T == 0) return ok();
  FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, W); FMHC_REQUIRE_PTR(w, out);
  FMHC_REQUIRE_PTR(w, inv_rms);
  FMHC_REQUIRE_ALIGN2(w, x); FMHC_REQUIRE_ALIGN2(w, W); FMHC_REQUIRE_ALIGN2(w, out);
  if (!aligned(inv_rms, 4)) return fail(FMHC_ERR_ALIGNMENT, "%s: inv_rms must be 4-byte aligned", w);
  cudaStream_t s = (cudaStream_t)stream;
  if (T <= FMHC_K1_ROWS_MAX_T && D == 32 && nC % 8 == 0 && aligned(x, 16) && aligned(W, 16)) {
    // Few tokens: one pass over W per block of 2 tokens (split over a cluster
    // while the tokens are too few to fill the GPU) beats the tensor-core
    // kernel's serial k-loop per tile.
    const int rc = fmhc::launch_k1_fwd_rows_cluster(x, W, out, inv_rms, T, int(nC), s);
    if (rc > 0) return fail(rc, "%s: %s", w, fmhc::k1_tc_error());
    if (rc < 0) fmhc::launch_k1_fwd_rows(x, W, out, inv_rms, T, int(nC), int(D), s);
  } else if (fmhc::k1_tc_fwd_supported(x, W, out, inv_rms, T, nC, D)) {
    if (int e = fmhc::launch_k1_tc_fwd(x, W, out, inv_rms, T, int(nC), s))
      return fail(e, "%s: %s", w, fmhc::k1_tc_error());
  } else {
    const int vec = pick_vec(nC, {x, W});
    fmhc::launch_k1_fwd_simt(x, W, out, inv_rms, T, int(nC), int(D), vec == 8 ? 8 : 1, s);
  }
  return check_launch(w);
}

int fmhc_debug_k1_fwd_lost_copy(const void *x, const void *W, void *out, float *inv_rms,
                                int64_t T, int64_t nC, void *stream) {
  const char *w = "fmhc_debug_k1_fwd_lost_copy";
  if (int e = check_k1(w, T, nC, 32)) return e;
  if (T == 0) return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: needs T >= 1", w);
  FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, W); FMHC_REQUIRE_PTR(w, out);
  FMHC_REQUIRE_PTR(w, inv_rms);
  if (!fmhc::k1_tc_fwd_supported(x, W, out, inv_rms, T, nC, 32))
    return fail(FMHC_ERR_INVALID_ARGUMENT,
                "%s: needs the tensor-core K1 forward (nC %% 64 == 0, 16-byte aligned x, W, out, "
                "a B200)", w);
  if (int e = fmhc::launch_k1_tc_fwd_lost_copy(x, W, out, inv_rms, T, int(nC), (cudaStream_t)stream))
    return fail(e, "%s: %s", w, fmhc::k1_tc_error());
  return check_launch(w);
}

int fmhc_k1_bwd_dx(const void *grad_out, const void *x, const void *W, const void *proj,
                   const float *inv_rms, void *grad_x, int64_t T, int64_t nC, int64_t D,
                   void *stream) {
  const char *w = "fmhc_k1_bwd_dx";
  if (int e = check_k1(w, T, nC, D)) return e;
  if (T == 0) return ok();
  FMHC_REQUIRE_PTR(w, grad_out); FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, W);
  FMHC_REQUIRE_PTR(w, proj); FMHC_REQUIRE_PTR(w, inv_rms); FMHC_REQUIRE_PTR(w, grad_x);
  FMHC_REQUIRE_ALIGN2(w, grad_out); FMHC_REQUIRE_ALIGN2(w, x); FMHC_REQUIRE_ALIGN2(w, W);
  FMHC_REQUIRE_ALIGN2(w, proj); FMHC_REQUIRE_ALIGN2(w, grad_x);
  if (!aligned(inv_rms, 4)) return fail(FMHC_ERR_ALIGNMENT, "%s: inv_rms must be 4-byte aligned", w);
  cudaStream_t s = (cudaStream_t)stream;
  if (fmhc::k1_tc_bwd_supported(grad_out, x, W, proj, grad_x, T, nC, D)) {
    if (int e = fmhc::launch_k1_tc_bwd(grad_out, x, W, proj, inv_rms, grad_x, nullptr, nullptr, 0,
                                       T, int(nC), s))
      return fail(e, "%s: %s", w, fmhc::k1_tc_error());
  } else {
    const int vec = pick_vec(nC, {x, W, grad_x});
    fmhc::launch_k1_bwd_dx_simt(grad_out, x, W, proj, inv_rms, grad_x, T, int(nC), int(D),
                                vec == 8 ? 8 : 1, s);
  }
  return check_launch(w);
}

int64_t fmhc_k1_bwd_workspace_size(int64_t T, int64_t nC, int64_t D) {
  if (T <= 0 || nC <= 0 || D <= 0 || D > 32) return 0;
  const int64_t a = fmhc::k1_tc_bwd_workspace_bytes(T, nC);
  const int64_t b = fmhc::k1_dw_workspace_bytes(T, nC, D);
  return a > b ? a : b;
}

int fmhc_k1_bwd(const void *grad_out, const void *x, const void *W, const void *proj,
                const float *inv_rms, void *grad_x, void *grad_W, void *workspace,
                int64_t workspace_bytes, int64_t T, int64_t nC, int64_t D, void *stream) {
  const char *w = "fmhc_k1_bwd";
  if (int e = check_k1(w, T, nC, D)) return e;
  FMHC_REQUIRE_PTR(w, grad_W);
  cudaStream_t s = (cudaStream_t)stream;
  if (T == 0) {
    // Empty batch: the weight gradient is exactly zero.
    if (cudaMemsetAsync(grad_W, 0, size_t(D * nC) * 2, s) != cudaSuccess)
      return fail(FMHC_ERR_CUDA, "%s: cudaMemsetAsync failed", w);
    return ok();
  }
  FMHC_REQUIRE_PTR(w, grad_out); FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, W);
  FMHC_REQUIRE_PTR(w, proj); FMHC_REQUIRE_PTR(w, inv_rms); FMHC_REQUIRE_PTR(w, grad_x);
  FMHC_REQUIRE_PTR(w, workspace);
  FMHC_REQUIRE_ALIGN2(w, grad_out); FMHC_REQUIRE_ALIGN2(w, x); FMHC_REQUIRE_ALIGN2(w, W);
  FMHC_REQUIRE_ALIGN2(w, proj); FMHC_REQUIRE_ALIGN2(w, grad_x); FMHC_REQUIRE_ALIGN2(w, grad_W);
  if (!aligned(inv_rms, 4)) return fail(FMHC_ERR_ALIGNMENT, "%s: inv_rms must be 4-byte aligned", w);
  if (!aligned(workspace, 256)) return fail(FMHC_ERR_ALIGNMENT, "%s: workspace must be 256-byte aligned", w);
  const int64_t need = fmhc_k1_bwd_workspace_size(T, nC, D);
  if (workspace_bytes < need)
    return fail(FMHC_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", w,
                (long long)workspace_bytes, (long long)need);
  if (fmhc::k1_tc_bwd_supported(grad_out, x, W, proj, grad_x, T, nC, D)) {
    if (int e = fmhc::launch_k1_tc_bwd(grad_out, x, W, proj, inv_rms, grad_x, grad_W, workspace,
                                       workspace_bytes, T, int(nC), s))
      return fail(e, "%s: %s", w, fmhc::k1_tc_error());
  } else {
    const int vec = pick_vec(nC, {x, W, grad_x});
    fmhc::launch_k1_bwd_dx_simt(grad_out, x, W, proj, inv_rms, grad_x, T, int(nC), int(D),
                                vec == 8 ? 8 : 1, s);
    fmhc::launch_k1_dw_simt(grad_out, x, inv_rms, grad_W, (float *)workspace, T, int(nC),
                            int(D), s);
  }
  return check_launch(w);
}

int fmhc_k2_fwd(const void *proj, const float *params, const float *perm, float *h_pre,
                float *h_post, float *H_merged, int64_t T, void *stream) {
  const char *w = "fmhc_k2_fwd";
  if (T < 0) return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: T must be >= 0 (got %lld)", w, (long long)T);
  if (T == 0) return ok();
  FMHC_REQUIRE_PTR(w, proj); FMHC_REQUIRE_PTR(w, params); FMHC_REQUIRE_PTR(w, perm);
  FMHC_REQUIRE_PTR(w, h_pre); FMHC_REQUIRE_PTR(w, h_post); FMHC_REQUIRE_PTR(w, H_merged);
  FMHC_REQUIRE_ALIGN16(w, proj); FMHC_REQUIRE_ALIGN16(w, h_pre); FMHC_REQUIRE_ALIGN16(w, h_post);
  FMHC_REQUIRE_ALIGN16(w, H_merged);
  if (!aligned(params, 4) || !aligned(perm, 4)) return fail(FMHC_ERR_ALIGNMENT, "%s: params/perm must be 4-byte aligned", w);
  fmhc::launch_k2_fwd(proj, fmhc::k2_packed_params(params, perm), h_pre, h_post, H_merged, T,
                      (cudaStream_t)stream);
  return check_launch(w);
}

int fmhc_k2_fwd_typed(const void *proj, const void *alpha_pre, const void *alpha_post,
                      const void *alpha_res, const void *bias, int param_dtype, const void *perm,
                      int perm_dtype, float *h_pre, float *h_post, float *H_merged, int64_t T,
                      void *stream) {
  const char *w = "fmhc_k2_fwd_typed";
  if (T < 0) return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: T must be >= 0 (got %lld)", w, (long long)T);
  const auto dt_ok = [](int d) { return d == FMHC_DTYPE_F32 || d == FMHC_DTYPE_BF16; };
  if (!dt_ok(param_dtype) || !dt_ok(perm_dtype))
    return fail(FMHC_ERR_UNSUPPORTED, "%s: parameter dtypes must be FMHC_DTYPE_F32 or FMHC_DTYPE_BF16", w);
  if (T == 0) return ok();
  FMHC_REQUIRE_PTR(w, proj); FMHC_REQUIRE_PTR(w, alpha_pre); FMHC_REQUIRE_PTR(w, alpha_post);
  FMHC_REQUIRE_PTR(w, alpha_res); FMHC_REQUIRE_PTR(w, bias); FMHC_REQUIRE_PTR(w, perm);
  FMHC_REQUIRE_PTR(w, h_pre); FMHC_REQUIRE_PTR(w, h_post); FMHC_REQUIRE_PTR(w, H_merged);
  FMHC_REQUIRE_ALIGN16(w, proj); FMHC_REQUIRE_ALIGN16(w, h_pre); FMHC_REQUIRE_ALIGN16(w, h_post);
  FMHC_REQUIRE_ALIGN16(w, H_merged);
  const uintptr_t pa = param_dtype == FMHC_DTYPE_BF16 ? 2 : 4;
  const uintptr_t qa = perm_dtype == FMHC_DTYPE_BF16 ? 2 : 4;
  if (!aligned(alpha_pre, pa) || !aligned(alpha_post, pa) || !aligned(alpha_res, pa) ||
      !aligned(bias, pa) || !aligned(perm, qa))
    return fail(FMHC_ERR_ALIGNMENT, "%s: parameters must be aligned to their element size", w);
  const fmhc::K2Params P{alpha_pre, alpha_post, alpha_res, bias, perm,
                         param_dtype == FMHC_DTYPE_BF16 ? 1 : 0,
                         perm_dtype == FMHC_DTYPE_BF16 ? 1 : 0};
  fmhc::launch_k2_fwd(proj, P, h_pre, h_post, H_merged, T, (cudaStream_t)stream);
  return check_launch(w);
}

int fmhc_mhc_pre_fwd(const void *x, const void *W, const void *alpha_pre, const void *alpha_post,
                     const void *alpha_res, const void *bias, int param_dtype, const void *perm,
                     int perm_dtype, void *proj, float *inv_rms, float *h_pre, float *h_post,
                     float *H_merged, void *layer_input, int64_t T, int64_t n, int64_t C,
                     void *stream) {
  const char *w = "fmhc_mhc_pre_fwd";
  if (int e = check_streams(w, T, n, C)) return e;
  const int64_t nC = n * C, D = 32;
  if (int e = check_k1(w, T, nC, D)) return e;
  const auto dt_ok = [](int d) { return d == FMHC_DTYPE_F32 || d == FMHC_DTYPE_BF16; };
  if (!dt_ok(param_dtype) || !dt_ok(perm_dtype))
    return fail(FMHC_ERR_UNSUPPORTED, "%s: parameter dtypes must be FMHC_DTYPE_F32 or FMHC_DTYPE_BF16", w);
  if (T == 0) return ok();
  FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, W); FMHC_REQUIRE_PTR(w, alpha_pre);
  FMHC_REQUIRE_PTR(w, alpha_post); FMHC_REQUIRE_PTR(w, alpha_res); FMHC_REQUIRE_PTR(w, bias);
  FMHC_REQUIRE_PTR(w, perm); FMHC_REQUIRE_PTR(w, proj); FMHC_REQUIRE_PTR(w, inv_rms);
  FMHC_REQUIRE_PTR(w, h_pre); FMHC_REQUIRE_PTR(w, h_post); FMHC_REQUIRE_PTR(w, H_merged);
  FMHC_REQUIRE_ALIGN2(w, x); FMHC_REQUIRE_ALIGN2(w, W); FMHC_REQUIRE_ALIGN16(w, proj);
  FMHC_REQUIRE_ALIGN16(w, h_pre); FMHC_REQUIRE_ALIGN16(w, h_post); FMHC_REQUIRE_ALIGN16(w, H_merged);
  if (!aligned(inv_rms, 4)) return fail(FMHC_ERR_ALIGNMENT, "%s: inv_rms must be 4-byte aligned", w);
  if (layer_input) FMHC_REQUIRE_ALIGN2(w, layer_input);
  const uintptr_t pa = param_dtype == FMHC_DTYPE_BF16 ? 2 : 4;
  const uintptr_t qa = perm_dtype == FMHC_DTYPE_BF16 ? 2 : 4;
  if (!aligned(alpha_pre, pa) || !aligned(alpha_post, pa) || !aligned(alpha_res, pa) ||
      !aligned(bias, pa) || !aligned(perm, qa))
    return fail(FMHC_ERR_ALIGNMENT, "%s: parameters must be aligned to their element size", w);
  const fmhc::K2Params P{alpha_pre, alpha_post, alpha_res, bias, perm,
                         param_dtype == FMHC_DTYPE_BF16 ? 1 : 0,
                         perm_dtype == FMHC_DTYPE_BF16 ? 1 : 0};
  cudaStream_t s = (cudaStream_t)stream;
  bool pre_done = false;
  // K1 takes the kernel fmhc_k1_fwd would take for this call, with K2 (and
  // at few tokens K3) in its epilogue, so every output equals the separate
  // fmhc_k1_fwd -> fmhc_k2_fwd_typed -> fmhc_k3_fwd results bit for bit.
  if (T <= FMHC_K1_ROWS_MAX_T && nC % 8 == 0 && aligned(x, 16) && aligned(W, 16)) {
    const bool pre = layer_input && C % 8 == 0 && aligned(layer_input, 16);
    void *pre_out = pre ? layer_input : nullptr;
    const int rc = fmhc::launch_k1_fwd_rows_cluster(x, W, proj, inv_rms, T, int(nC), s, &P, h_pre,
                                                    h_post, H_merged, pre_out);
    if (rc > 0) return fail(rc, "%s: %s", w, fmhc::k1_tc_error());
    if (rc < 0)
      fmhc::launch_k1_fwd_rows(x, W, proj, inv_rms, T, int(nC), int(D), s, &P, h_pre, h_post,
                               H_merged, pre_out);
    pre_done = pre;
  } else if (fmhc::k1_tc_fwd_supported(x, W, proj, inv_rms, T, nC, D)) {
    if (int e = fmhc::launch_k1_tc_fwd(x, W, proj, inv_rms, T, int(nC), s, &P, h_pre, h_post,
                                       H_merged))
      return fail(e, "%s: %s", w, fmhc::k1_tc_error());
  } else {
    const int vec = pick_vec(nC, {x, W});
    fmhc::launch_k1_fwd_simt(x, W, proj, inv_rms, T, int(nC), int(D), vec == 8 ? 8 : 1, s);
    fmhc::launch_k2_fwd(proj, P, h_pre, h_post, H_merged, T, s);
  }
  if (layer_input && !pre_done) {
    const int vec = pick_vec(C, {x, layer_input});
    fmhc::launch_k3_fwd(x, h_pre, layer_input, T, int(C), vec, s);
  }
  return check_launch(w);
}

int64_t fmhc_k2_bwd_workspace_size(int64_t T) {
  if (T <= 0) return 0;
  return fmhc::k2_bwd_workspace_bytes(T);
}

int fmhc_k2_bwd(const void *proj, const float *params, const float *perm, const float *grad_h_pre,
                const float *grad_h_post, const float *grad_H_merged, void *grad_proj,
                float *grad_params, void *workspace, int64_t workspace_bytes, int64_t T,
                void *stream) {
  const char *w = "fmhc_k2_bwd";
  if (T < 0) return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: T must be >= 0 (got %lld)", w, (long long)T);
  FMHC_REQUIRE_PTR(w, grad_params);
  cudaStream_t s = (cudaStream_t)stream;
  if (T == 0) {
    if (cudaMemsetAsync(grad_params, 0, 35 * sizeof(float), s) != cudaSuccess)
      return fail(FMHC_ERR_CUDA, "%s: cudaMemsetAsync failed", w);
    return ok();
  }
  FMHC_REQUIRE_PTR(w, proj); FMHC_REQUIRE_PTR(w, params); FMHC_REQUIRE_PTR(w, perm);
  FMHC_REQUIRE_PTR(w, grad_h_pre); FMHC_REQUIRE_PTR(w, grad_h_post);
  FMHC_REQUIRE_PTR(w, grad_H_merged); FMHC_REQUIRE_PTR(w, grad_proj); FMHC_REQUIRE_PTR(w, workspace);
  FMHC_REQUIRE_ALIGN16(w, proj); FMHC_REQUIRE_ALIGN16(w, grad_h_pre);
  FMHC_REQUIRE_ALIGN16(w, grad_h_post); FMHC_REQUIRE_ALIGN16(w, grad_H_merged);
  FMHC_REQUIRE_ALIGN16(w, grad_proj);
  if (!aligned(workspace, 256)) return fail(FMHC_ERR_ALIGNMENT, "%s: workspace must be 256-byte aligned", w);
  if (!aligned(params, 4) || !aligned(perm, 4) || !aligned(grad_params, 4))
    return fail(FMHC_ERR_ALIGNMENT, "%s: params/perm/grad_params must be 4-byte aligned", w);
  const int64_t need = fmhc::k2_bwd_workspace_bytes(T);
  if (workspace_bytes < need)
    return fail(FMHC_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", w,
                (long long)workspace_bytes, (long long)need);
  fmhc::launch_k2_bwd(proj, fmhc::k2_packed_params(params, perm), grad_h_pre, grad_h_post,
                      grad_H_merged, grad_proj, fmhc::k2_packed_grads(grad_params),
                      (float *)workspace, T, s);
  return check_launch(w);
}

int fmhc_k2_bwd_typed(const void *proj, const void *alpha_pre, const void *alpha_post,
                      const void *alpha_res, const void *bias, int param_dtype, const void *perm,
                      int perm_dtype, const float *grad_h_pre, const float *grad_h_post,
                      const float *grad_H_merged, void *grad_proj, void *grad_alpha_pre,
                      void *grad_alpha_post, void *grad_alpha_res, void *grad_bias,
                      void *workspace, int64_t workspace_bytes, int64_t T, void *stream) {
  const char *w = "fmhc_k2_bwd_typed";
  if (T < 0) return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: T must be >= 0 (got %lld)", w, (long long)T);
  const auto dt_ok = [](int d) { return d == FMHC_DTYPE_F32 || d == FMHC_DTYPE_BF16; };
  if (!dt_ok(param_dtype) || !dt_ok(perm_dtype))
    return fail(FMHC_ERR_UNSUPPORTED, "%s: parameter dtypes must be FMHC_DTYPE_F32 or FMHC_DTYPE_BF16", w);
  FMHC_REQUIRE_PTR(w, grad_alpha_pre); FMHC_REQUIRE_PTR(w, grad_alpha_post);
  FMHC_REQUIRE_PTR(w, grad_alpha_res); FMHC_REQUIRE_PTR(w, grad_bias);
  const uintptr_t pa = param_dtype == FMHC_DTYPE_BF16 ? 2 : 4;
  const uintptr_t qa = perm_dtype == FMHC_DTYPE_BF16 ? 2 : 4;
  if (!aligned(grad_alpha_pre, pa) || !aligned(grad_alpha_post, pa) ||
      !aligned(grad_alpha_res, pa) || !aligned(grad_bias, pa))
    return fail(FMHC_ERR_ALIGNMENT, "%s: parameter gradients must be aligned to their element size", w);
  const fmhc::K2ParamGrads G{grad_alpha_pre, grad_alpha_post, grad_alpha_res, grad_bias,
                             param_dtype == FMHC_DTYPE_BF16 ? 1 : 0};
  cudaStream_t s = (cudaStream_t)stream;
  if (T == 0) {
    fmhc::launch_k2_bwd(nullptr, fmhc::K2Params{}, nullptr, nullptr, nullptr, nullptr, G, nullptr,
                        0, s);
    return check_launch(w);
  }
  FMHC_REQUIRE_PTR(w, proj); FMHC_REQUIRE_PTR(w, alpha_pre); FMHC_REQUIRE_PTR(w, alpha_post);
  FMHC_REQUIRE_PTR(w, alpha_res); FMHC_REQUIRE_PTR(w, bias); FMHC_REQUIRE_PTR(w, perm);
  FMHC_REQUIRE_PTR(w, grad_h_pre); FMHC_REQUIRE_PTR(w, grad_h_post);
  FMHC_REQUIRE_PTR(w, grad_H_merged); FMHC_REQUIRE_PTR(w, grad_proj); FMHC_REQUIRE_PTR(w, workspace);
  FMHC_REQUIRE_ALIGN16(w, proj); FMHC_REQUIRE_ALIGN16(w, grad_h_pre);
  FMHC_REQUIRE_ALIGN16(w, grad_h_post); FMHC_REQUIRE_ALIGN16(w, grad_H_merged);
  FMHC_REQUIRE_ALIGN16(w, grad_proj);
  if (!aligned(alpha_pre, pa) || !aligned(alpha_post, pa) || !aligned(alpha_res, pa) ||
      !aligned(bias, pa) || !aligned(perm, qa))
    return fail(FMHC_ERR_ALIGNMENT, "%s: parameters must be aligned to their element size", w);
  if (!aligned(workspace, 256)) return fail(FMHC_ERR_ALIGNMENT, "%s: workspace must be 256-byte aligned", w);
  const int64_t need = fmhc::k2_bwd_workspace_bytes(T);
  if (workspace_bytes < need)
    return fail(FMHC_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", w,
                (long long)workspace_bytes, (long long)need);
  const fmhc::K2Params P{alpha_pre, alpha_post, alpha_res, bias, perm,
                         param_dtype == FMHC_DTYPE_BF16 ? 1 : 0,
                         perm_dtype == FMHC_DTYPE_BF16 ? 1 : 0};
  fmhc::launch_k2_bwd(proj, P, grad_h_pre, grad_h_post, grad_H_merged, grad_proj, G,
                      (float *)workspace, T, s);
  return check_launch(w);
}

// ------------------------------------------------- 8-bit activation checkpoints
static bool fmt_ok(int f) { return f == FMHC_ACT8_INT8 || f == FMHC_ACT8_E4M3; }
static bool dtype_ok(int d) {
  return d == FMHC_DTYPE_F32 || d == FMHC_DTYPE_BF16 || d == FMHC_DTYPE_F16;
}
static uintptr_t dtype_size(int d) { return d == FMHC_DTYPE_F32 ? 4 : 2; }

static int check_rows(const char *w, int64_t rows, int64_t C) {
  if (rows < 0) return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: rows must be >= 0 (got %lld)", w, (long long)rows);
  if (C < 1 || C > (int64_t(1) << 28))
    return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: C must be in [1, 2^28] (got %lld)", w, (long long)C);
  return FMHC_OK;
}

#define FMHC_REQUIRE_FMT(w, f)                                                              \
  if (!fmt_ok(f))                                                                           \
  return fail(FMHC_ERR_UNSUPPORTED, "%s: the code format must be FMHC_ACT8_INT8 or "        \
              "FMHC_ACT8_E4M3", w)
#define FMHC_REQUIRE_DTYPE(w, d)                                                            \
  if (!dtype_ok(d))                                                                         \
  return fail(FMHC_ERR_UNSUPPORTED, "%s: the element type must be FMHC_DTYPE_F32, "         \
              "FMHC_DTYPE_BF16 or FMHC_DTYPE_F16", w)
#define FMHC_REQUIRE_ALIGN_TO(w, p, a)                                                      \
  if (!aligned((p), (a)))                                                                   \
  return fail(FMHC_ERR_ALIGNMENT, "%s: %s must be aligned to its element size", w, #p)

int fmhc_act_quantize(const void *x, int x_dtype, void *codes, int format, void *scales,
                      int64_t rows, int64_t C, void *stream) {
  const char *w = "fmhc_act_quantize";
  if (int e = check_rows(w, rows, C)) return e;
  FMHC_REQUIRE_DTYPE(w, x_dtype);
  FMHC_REQUIRE_FMT(w, format);
  if (rows == 0) return ok();
  FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, codes); FMHC_REQUIRE_PTR(w, scales);
  FMHC_REQUIRE_ALIGN_TO(w, x, dtype_size(x_dtype));
  const bool vec = C % 8 == 0 && aligned(x, 16) && aligned(codes, 8);
  fmhc::launch_act_quantize(x, x_dtype, codes, format, scales, rows, int(C), vec, (cudaStream_t)stream);
  return check_launch(w);
}

int fmhc_act_dequantize(const void *codes, int format, const void *scales, void *x, int x_dtype,
                        int64_t rows, int64_t C, void *stream) {
  const char *w = "fmhc_act_dequantize";
  if (int e = check_rows(w, rows, C)) return e;
  FMHC_REQUIRE_DTYPE(w, x_dtype);
  FMHC_REQUIRE_FMT(w, format);
  if (rows == 0) return ok();
  FMHC_REQUIRE_PTR(w, codes); FMHC_REQUIRE_PTR(w, scales); FMHC_REQUIRE_PTR(w, x);
  FMHC_REQUIRE_ALIGN_TO(w, x, dtype_size(x_dtype));
  const bool vec = C % 8 == 0 && aligned(x, 16) && aligned(codes, 8);
  fmhc::launch_act_dequantize(codes, format, scales, x, x_dtype, rows, int(C), vec, (cudaStream_t)stream);
  return check_launch(w);
}

int fmhc_k3_fwd_q8(const void *x, const float *h_pre, void *out, void *x_codes, void *x_scales,
                   int format, int64_t T, int64_t n, int64_t C, void *stream) {
  const char *w = "fmhc_k3_fwd_q8";
  if (int e = check_streams(w, T, n, C)) return e;
  FMHC_REQUIRE_FMT(w, format);
  if (T == 0) return ok();
  FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, h_pre); FMHC_REQUIRE_PTR(w, out);
  FMHC_REQUIRE_PTR(w, x_codes); FMHC_REQUIRE_PTR(w, x_scales);
  FMHC_REQUIRE_ALIGN16(w, h_pre);
  FMHC_REQUIRE_ALIGN2(w, x); FMHC_REQUIRE_ALIGN2(w, out);
  cudaStream_t s = (cudaStream_t)stream;
  const int vec = pick_vec(C, {x, out});
  if (vec == 8 && aligned(x_codes, 8)) {
    fmhc::launch_k3_fwd_q8(x, h_pre, out, x_codes, x_scales, format, T, int(C), s);
  } else {
    fmhc::launch_k3_fwd(x, h_pre, out, T, int(C), vec, s);
    fmhc::launch_act_quantize(x, FMHC_DTYPE_BF16, x_codes, format, x_scales, 4 * T, int(C),
                              C % 8 == 0 && aligned(x, 16) && aligned(x_codes, 8), s);
  }
  return check_launch(w);
}

int fmhc_k4_fwd_q8(const void *x, const void *lo, const float *H, const float *h_post, void *out,
                   void *lo_codes, void *lo_scales, int format, int64_t T, int64_t n, int64_t C,
                   void *stream) {
  const char *w = "fmhc_k4_fwd_q8";
  if (int e = check_streams(w, T, n, C)) return e;
  FMHC_REQUIRE_FMT(w, format);
  if (T == 0) return ok();
  FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, lo); FMHC_REQUIRE_PTR(w, H);
  FMHC_REQUIRE_PTR(w, h_post); FMHC_REQUIRE_PTR(w, out); FMHC_REQUIRE_PTR(w, lo_codes);
  FMHC_REQUIRE_PTR(w, lo_scales);
  FMHC_REQUIRE_ALIGN16(w, H); FMHC_REQUIRE_ALIGN16(w, h_post);
  FMHC_REQUIRE_ALIGN2(w, x); FMHC_REQUIRE_ALIGN2(w, lo); FMHC_REQUIRE_ALIGN2(w, out);
  cudaStream_t s = (cudaStream_t)stream;
  const int vec = pick_vec(C, {x, lo, out});
  if (vec == 8 && aligned(lo_codes, 8)) {
    fmhc::launch_k4_fwd_q8(x, lo, H, h_post, out, lo_codes, lo_scales, format, T, int(C), s);
  } else {
    fmhc::launch_k4_fwd(x, lo, H, h_post, out, T, int(C), vec, s);
    fmhc::launch_act_quantize(lo, FMHC_DTYPE_BF16, lo_codes, format, lo_scales, T, int(C),
                              C % 8 == 0 && aligned(lo, 16) && aligned(lo_codes, 8), s);
  }
  return check_launch(w);
}

int fmhc_k3_bwd_q8(const void *grad_out, const void *x_codes, const void *x_scales, int format,
                   float *grad_h, int64_t T, int64_t n, int64_t C, void *stream) {
  const char *w = "fmhc_k3_bwd_q8";
  if (int e = check_streams(w, T, n, C)) return e;
  FMHC_REQUIRE_FMT(w, format);
  if (T == 0) return ok();
  FMHC_REQUIRE_PTR(w, grad_out); FMHC_REQUIRE_PTR(w, x_codes); FMHC_REQUIRE_PTR(w, x_scales);
  FMHC_REQUIRE_PTR(w, grad_h);
  FMHC_REQUIRE_ALIGN16(w, grad_h); FMHC_REQUIRE_ALIGN2(w, grad_out);
  const int vec = pick_vec(C, {grad_out}) == 8 && aligned(x_codes, 8) ? 8 : 1;
  fmhc::launch_k3_bwd_q8(grad_out, x_codes, x_scales, format, grad_h, T, int(C), vec, (cudaStream_t)stream);
  return check_launch(w);
}

int fmhc_k4_bwd_q8(const void *grad_out, const void *x_codes, const void *x_scales,
                   const void *lo_codes, const void *lo_scales, int format, const float *h_post,
                   void *grad_lo, float *grad_H, float *grad_hp, int64_t T, int64_t n, int64_t C,
                   void *stream) {
  const char *w = "fmhc_k4_bwd_q8";
  if (int e = check_streams(w, T, n, C)) return e;
  FMHC_REQUIRE_FMT(w, format);
  if (T == 0) return ok();
  FMHC_REQUIRE_PTR(w, grad_out); FMHC_REQUIRE_PTR(w, x_codes); FMHC_REQUIRE_PTR(w, x_scales);
  FMHC_REQUIRE_PTR(w, lo_codes); FMHC_REQUIRE_PTR(w, lo_scales); FMHC_REQUIRE_PTR(w, h_post);
  FMHC_REQUIRE_PTR(w, grad_lo); FMHC_REQUIRE_PTR(w, grad_H); FMHC_REQUIRE_PTR(w, grad_hp);
  FMHC_REQUIRE_ALIGN16(w, h_post); FMHC_REQUIRE_ALIGN16(w, grad_H); FMHC_REQUIRE_ALIGN16(w, grad_hp);
  FMHC_REQUIRE_ALIGN2(w, grad_out); FMHC_REQUIRE_ALIGN2(w, grad_lo);
  const int vec = pick_vec(C, {grad_out, grad_lo}) == 8 && aligned(x_codes, 8) && aligned(lo_codes, 8) ? 8 : 1;
  fmhc::launch_k4_bwd_q8(grad_out, x_codes, x_scales, lo_codes, lo_scales, format, h_post, grad_lo,
                         grad_H, grad_hp, T, int(C), vec, (cudaStream_t)stream);
  return check_launch(w);
}

// Which kernel: the tcgen05 one for the widths it takes, but for little work, where
// its set-up and its second launch cost more than they gain (us, tcgen05 / any
// width: T = 32, C = 4096 14.2 / 6.4; T = 1024, C = 256 7.9 / 6.9; T = 256, C =
// 1024 8.9 / 8.6; T = 512, C = 1024 9.6 / 11.1; T = 128, C = 4096 13.8 / 17.6).
static bool k1_bwd_q8_on_tcgen05(int64_t T, int64_t nC) {
  return fmhc::k1_tc_bwd_q8_shape(T, nC) && T > 32 && T * nC > (int64_t(1) << 20);
}

int64_t fmhc_k1_bwd_q8_workspace_size(int64_t T, int64_t C) {
  if (T <= 0 || C <= 0 || C > (int64_t(1) << 26)) return 0;
  if (k1_bwd_q8_on_tcgen05(T, 4 * C)) return fmhc::k1_tc_bwd_workspace_bytes(T, 4 * C);
  return fmhc::k1_bwd_q8_any_workspace_bytes(T, int(4 * C));
}

int fmhc_k1_bwd_q8(const void *grad_out, const void *x_codes, const void *x_scales, int format,
                   const void *W, const void *proj, const float *inv_rms, void *grad_x,
                   void *grad_W, void *workspace, int64_t workspace_bytes, int64_t T, int64_t n,
                   int64_t C, void *stream) {
  const char *w = "fmhc_k1_bwd_q8";
  if (int e = check_streams(w, T, n, C)) return e;
  const int64_t nC = n * C;
  if (int e = check_k1(w, T, nC, 32)) return e;
  FMHC_REQUIRE_FMT(w, format);
  FMHC_REQUIRE_PTR(w, grad_W);
  cudaStream_t s = (cudaStream_t)stream;
  if (T == 0) return fmhc_k1_bwd(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, grad_W, nullptr,
                                 0, 0, nC, 32, stream);
  FMHC_REQUIRE_PTR(w, grad_out); FMHC_REQUIRE_PTR(w, x_codes); FMHC_REQUIRE_PTR(w, x_scales);
  FMHC_REQUIRE_PTR(w, W); FMHC_REQUIRE_PTR(w, proj); FMHC_REQUIRE_PTR(w, inv_rms);
  FMHC_REQUIRE_PTR(w, grad_x); FMHC_REQUIRE_PTR(w, workspace);
  FMHC_REQUIRE_ALIGN2(w, grad_W); FMHC_REQUIRE_ALIGN_TO(w, inv_rms, 4);
  if (!aligned(workspace, 256)) return fail(FMHC_ERR_ALIGNMENT, "%s: workspace must be 256-byte aligned", w);
  const int64_t need = fmhc_k1_bwd_q8_workspace_size(T, C);
  if (workspace_bytes < need)
    return fail(FMHC_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", w,
                (long long)workspace_bytes, (long long)need);
  FMHC_REQUIRE_ALIGN16(w, grad_out); FMHC_REQUIRE_ALIGN16(w, x_codes); FMHC_REQUIRE_ALIGN16(w, W);
  FMHC_REQUIRE_ALIGN16(w, proj); FMHC_REQUIRE_ALIGN16(w, grad_x);
  if (!aligned(x_scales, 4)) return fail(FMHC_ERR_ALIGNMENT, "%s: x_scales must be 4-byte aligned", w);
  if (k1_bwd_q8_on_tcgen05(T, nC)) {
    if (int e = fmhc::launch_k1_tc_bwd_q8(grad_out, x_codes, x_scales, format, W, proj, inv_rms,
                                          grad_x, grad_W, workspace, T, int(nC), s))
      return fail(e, "%s: %s", w, fmhc::k1_tc_error());
  } else {
    fmhc::launch_k1_bwd_q8_any(grad_out, x_codes, x_scales, format, W, proj, inv_rms, grad_x,
                               grad_W, (float *)workspace, T, int(nC), s);
  }
  return check_launch(w);
}

// ------------------------------------------------------------------ layer norm
int fmhc_layer_norm_fwd(const void *x, int x_dtype, const void *weight, const void *bias,
                        int param_dtype, float eps, void *y, float *mean, float *rstd,
                        void *x_codes, int format, void *x_scales, int64_t rows, int64_t C,
                        void *stream) {
  const char *w = "fmhc_layer_norm_fwd";
  if (int e = check_rows(w, rows, C)) return e;
  FMHC_REQUIRE_DTYPE(w, x_dtype);
  FMHC_REQUIRE_DTYPE(w, param_dtype);
  if (!(eps >= 0.f)) return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: eps must be >= 0", w);
  if (x_codes != nullptr) FMHC_REQUIRE_FMT(w, format);
  if ((x_codes == nullptr) != (x_scales == nullptr))
    return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: x_codes and x_scales go together", w);
  if (rows == 0) return ok();
  FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, y); FMHC_REQUIRE_PTR(w, mean); FMHC_REQUIRE_PTR(w, rstd);
  FMHC_REQUIRE_ALIGN_TO(w, x, dtype_size(x_dtype)); FMHC_REQUIRE_ALIGN_TO(w, y, dtype_size(x_dtype));
  FMHC_REQUIRE_ALIGN_TO(w, weight, dtype_size(param_dtype));
  FMHC_REQUIRE_ALIGN_TO(w, bias, dtype_size(param_dtype));
  FMHC_REQUIRE_ALIGN_TO(w, mean, 4); FMHC_REQUIRE_ALIGN_TO(w, rstd, 4);
  const bool vec = aligned(x, 16) && aligned(y, 16) && aligned(weight, 16) && aligned(bias, 16) &&
                   aligned(x_codes, 8);
  fmhc::launch_ln_fwd(x, x_dtype, weight, bias, param_dtype, eps, y, mean, rstd, x_codes,
                      x_codes ? format : -1, x_scales, rows, int(C), vec, (cudaStream_t)stream);
  return check_launch(w);
}

int64_t fmhc_layer_norm_bwd_workspace_size(int64_t rows, int64_t C) {
  if (rows <= 0 || C <= 0 || C > (int64_t(1) << 28)) return 0;
  return fmhc::ln_bwd_workspace_bytes(rows, int(C));
}

int fmhc_layer_norm_bwd(const void *grad_y, int x_dtype, const void *x, const void *x_codes,
                        int format, const void *x_scales, const float *mean, const float *rstd,
                        const void *weight, int param_dtype, void *grad_x, void *grad_weight,
                        void *grad_bias, void *workspace, int64_t workspace_bytes, int64_t rows,
                        int64_t C, void *stream) {
  const char *w = "fmhc_layer_norm_bwd";
  if (int e = check_rows(w, rows, C)) return e;
  FMHC_REQUIRE_DTYPE(w, x_dtype);
  FMHC_REQUIRE_DTYPE(w, param_dtype);
  if (x_codes != nullptr) FMHC_REQUIRE_FMT(w, format);
  if ((x_codes == nullptr) != (x_scales == nullptr))
    return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: x_codes and x_scales go together", w);
  FMHC_REQUIRE_ALIGN_TO(w, grad_weight, dtype_size(param_dtype));
  FMHC_REQUIRE_ALIGN_TO(w, grad_bias, dtype_size(param_dtype));
  cudaStream_t s = (cudaStream_t)stream;
  if (rows == 0) {
    // No rows: the parameters' gradients are exactly zero.
    for (void *p : {grad_weight, grad_bias})
      if (p != nullptr && cudaMemsetAsync(p, 0, size_t(C) * dtype_size(param_dtype), s) != cudaSuccess)
        return fail(FMHC_ERR_CUDA, "%s: cudaMemsetAsync failed", w);
    return ok();
  }
  if ((x == nullptr) == (x_codes == nullptr))
    return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: exactly one of x and x_codes is wanted", w);
  FMHC_REQUIRE_PTR(w, grad_y); FMHC_REQUIRE_PTR(w, mean); FMHC_REQUIRE_PTR(w, rstd);
  FMHC_REQUIRE_PTR(w, grad_x);
  FMHC_REQUIRE_ALIGN_TO(w, grad_y, dtype_size(x_dtype)); FMHC_REQUIRE_ALIGN_TO(w, x, dtype_size(x_dtype));
  FMHC_REQUIRE_ALIGN_TO(w, grad_x, dtype_size(x_dtype));
  FMHC_REQUIRE_ALIGN_TO(w, weight, dtype_size(param_dtype));
  FMHC_REQUIRE_ALIGN_TO(w, mean, 4); FMHC_REQUIRE_ALIGN_TO(w, rstd, 4);
  if (grad_weight != nullptr || grad_bias != nullptr) {
    FMHC_REQUIRE_PTR(w, workspace);
    if (!aligned(workspace, 256)) return fail(FMHC_ERR_ALIGNMENT, "%s: workspace must be 256-byte aligned", w);
    const int64_t need = fmhc_layer_norm_bwd_workspace_size(rows, C);
    if (workspace_bytes < need)
      return fail(FMHC_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", w,
                  (long long)workspace_bytes, (long long)need);
  }
  const bool vec = aligned(grad_y, 16) && aligned(x, 16) && aligned(x_codes, 8) && aligned(x_scales, 4) &&
                   aligned(weight, 16) && aligned(grad_x, 16);
  fmhc::launch_ln_bwd(grad_y, x_dtype, x_codes ? x_codes : x, x_codes ? format : -1, x_scales, mean,
                      rstd, weight, param_dtype, grad_x, grad_weight, grad_bias, (float *)workspace,
                      rows, int(C), vec, s);
  return check_launch(w);
}

// ------------------------------------------------------- root-mean-square norm
static int check_rms(const char *w, const void *x, int x_dtype, const void *residual,
                     const void *weight, int param_dtype, float eps, const void *total) {
  FMHC_REQUIRE_DTYPE(w, x_dtype);
  FMHC_REQUIRE_DTYPE(w, param_dtype);
  if (!(eps >= 0.f)) return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: eps must be >= 0", w);
  if ((residual == nullptr) != (total == nullptr))
    return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: residual and total go together", w);
  for (const void *p : {x, residual, total}) FMHC_REQUIRE_ALIGN_TO(w, p, dtype_size(x_dtype));
  FMHC_REQUIRE_ALIGN_TO(w, weight, dtype_size(param_dtype));
  return FMHC_OK;
}

int fmhc_rms_norm_fwd(const void *x, int x_dtype, const void *residual, const void *weight,
                      int param_dtype, float eps, void *y, void *total, float *rstd, int64_t rows,
                      int64_t C, void *stream) {
  const char *w = "fmhc_rms_norm_fwd";
  if (int e = check_rows(w, rows, C)) return e;
  if (int e = check_rms(w, x, x_dtype, residual, weight, param_dtype, eps, total)) return e;
  if (rows == 0) return ok();
  FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, y); FMHC_REQUIRE_PTR(w, rstd);
  FMHC_REQUIRE_ALIGN_TO(w, y, dtype_size(x_dtype)); FMHC_REQUIRE_ALIGN_TO(w, rstd, 4);
  const bool vec = aligned(x, 16) && aligned(residual, 16) && aligned(weight, 16) && aligned(y, 16) &&
                   aligned(total, 16);
  fmhc::launch_rms_fwd(x, x_dtype, residual, weight, param_dtype, eps, y, total, rstd, nullptr, 0,
                       nullptr, rows, int(C), vec, (cudaStream_t)stream);
  return check_launch(w);
}

// Rows of codes: a stride of at least C bytes.
static int check_codes(const char *w, const char *name, int64_t stride, int64_t C) {
  if (stride < C)
    return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: rows of %s must be at least %lld bytes apart (got %lld)", w, name,
                (long long)C, (long long)stride);
  return FMHC_OK;
}

int fmhc_rms_norm_fwd_int8(const void *x, int x_dtype, const void *residual, const void *weight,
                           int param_dtype, float eps, void *codes, int64_t codes_stride,
                           float *scales, void *total, int64_t rows, int64_t C, void *stream) {
  const char *w = "fmhc_rms_norm_fwd_int8";
  if (int e = check_rows(w, rows, C)) return e;
  if (int e = check_rms(w, x, x_dtype, residual, weight, param_dtype, eps, total)) return e;
  if (int e = check_codes(w, "codes", codes_stride, C)) return e;
  if (rows == 0) return ok();
  FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, codes); FMHC_REQUIRE_PTR(w, scales);
  FMHC_REQUIRE_ALIGN_TO(w, scales, 4);
  const bool vec = aligned(x, 16) && aligned(residual, 16) && aligned(weight, 16) && aligned(total, 16) &&
                   aligned(codes, 8) && codes_stride % 8 == 0;
  fmhc::launch_rms_fwd(x, x_dtype, residual, weight, param_dtype, eps, nullptr, total, nullptr, codes,
                       codes_stride, scales, rows, int(C), vec, (cudaStream_t)stream);
  return check_launch(w);
}

int64_t fmhc_rms_norm_bwd_workspace_size(int64_t rows, int64_t C) {
  if (rows <= 0 || C <= 0 || C > (int64_t(1) << 28)) return 0;
  return fmhc::rms_bwd_workspace_bytes(rows, int(C));
}

int fmhc_rms_norm_bwd(const void *grad_y, int x_dtype, const void *grad_total, const void *x,
                      const float *rstd, const void *weight, int param_dtype, void *grad_x,
                      void *grad_weight, void *workspace, int64_t workspace_bytes, int64_t rows,
                      int64_t C, void *stream) {
  const char *w = "fmhc_rms_norm_bwd";
  if (int e = check_rows(w, rows, C)) return e;
  FMHC_REQUIRE_DTYPE(w, x_dtype);
  FMHC_REQUIRE_DTYPE(w, param_dtype);
  FMHC_REQUIRE_ALIGN_TO(w, grad_weight, dtype_size(param_dtype));
  cudaStream_t s = (cudaStream_t)stream;
  if (rows == 0) {
    // No rows: the weight's gradient is exactly zero.
    if (grad_weight != nullptr &&
        cudaMemsetAsync(grad_weight, 0, size_t(C) * dtype_size(param_dtype), s) != cudaSuccess)
      return fail(FMHC_ERR_CUDA, "%s: cudaMemsetAsync failed", w);
    return ok();
  }
  FMHC_REQUIRE_PTR(w, grad_y); FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, rstd);
  FMHC_REQUIRE_PTR(w, grad_x);
  for (const void *p : {grad_y, grad_total, x, (const void *)grad_x})
    FMHC_REQUIRE_ALIGN_TO(w, p, dtype_size(x_dtype));
  FMHC_REQUIRE_ALIGN_TO(w, weight, dtype_size(param_dtype)); FMHC_REQUIRE_ALIGN_TO(w, rstd, 4);
  if (grad_weight != nullptr) {
    FMHC_REQUIRE_PTR(w, workspace);
    if (!aligned(workspace, 256)) return fail(FMHC_ERR_ALIGNMENT, "%s: workspace must be 256-byte aligned", w);
    const int64_t need = fmhc_rms_norm_bwd_workspace_size(rows, C);
    if (workspace_bytes < need)
      return fail(FMHC_ERR_WORKSPACE, "%s: workspace of %lld bytes, %lld needed", w,
                  (long long)workspace_bytes, (long long)need);
  }
  const bool vec = aligned(grad_y, 16) && aligned(grad_total, 16) && aligned(x, 16) && aligned(weight, 16) &&
                   aligned(grad_x, 16);
  fmhc::launch_rms_bwd(grad_y, x_dtype, grad_total, x, rstd, weight, param_dtype, grad_x, grad_weight,
                       (float *)workspace, rows, int(C), vec, s);
  return check_launch(w);
}

// ------------------------------------------------- rows and linear layers in int8
int fmhc_row_quantize(const void *x, int x_dtype, void *codes, int64_t codes_stride, float *scales,
                      int64_t rows, int64_t C, void *stream) {
  const char *w = "fmhc_row_quantize";
  if (int e = check_rows(w, rows, C)) return e;
  FMHC_REQUIRE_DTYPE(w, x_dtype);
  if (int e = check_codes(w, "codes", codes_stride, C)) return e;
  if (rows == 0) return ok();
  FMHC_REQUIRE_PTR(w, x); FMHC_REQUIRE_PTR(w, codes); FMHC_REQUIRE_PTR(w, scales);
  FMHC_REQUIRE_ALIGN_TO(w, x, dtype_size(x_dtype)); FMHC_REQUIRE_ALIGN_TO(w, scales, 4);
  const bool vec = aligned(x, 16) && aligned(codes, 8) && codes_stride % 8 == 0;
  fmhc::launch_row_quantize(x, x_dtype, codes, codes_stride, scales, rows, int(C), vec, (cudaStream_t)stream);
  return check_launch(w);
}

int fmhc_row_dequantize(const void *codes, int64_t codes_stride, const float *scales, void *x,
                        int x_dtype, int64_t rows, int64_t C, void *stream) {
  const char *w = "fmhc_row_dequantize";
  if (int e = check_rows(w, rows, C)) return e;
  FMHC_REQUIRE_DTYPE(w, x_dtype);
  if (int e = check_codes(w, "codes", codes_stride, C)) return e;
  if (rows == 0) return ok();
  FMHC_REQUIRE_PTR(w, codes); FMHC_REQUIRE_PTR(w, scales); FMHC_REQUIRE_PTR(w, x);
  FMHC_REQUIRE_ALIGN_TO(w, x, dtype_size(x_dtype)); FMHC_REQUIRE_ALIGN_TO(w, scales, 4);
  const bool vec = aligned(x, 16) && aligned(codes, 8) && codes_stride % 8 == 0;
  fmhc::launch_row_dequantize(codes, codes_stride, scales, x, x_dtype, rows, int(C), vec, (cudaStream_t)stream);
  return check_launch(w);
}

static int int8_linear(const char *w, const void *codes, int64_t codes_stride, const float *scales,
                       const void *weight_codes, int64_t weight_stride, const float *weight_scales,
                       const void *bias, int bias_dtype, void *y, int y_dtype, int64_t T, int64_t N,
                       int64_t K, void *stream, bool lose_copy) {
  for (int64_t n : {T, N})
    if (n < 0 || n >= (int64_t(1) << 31) - 512)  // the last tile's end fits 32 bits too
      return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: T and N must be in [0, 2^31 - 512) (got %lld)", w, (long long)n);
  if (K < 1 || K >= (int64_t(1) << 17))
    return fail(FMHC_ERR_INVALID_ARGUMENT, "%s: K must be in [1, 2^17) (got %lld)", w, (long long)K);
  FMHC_REQUIRE_DTYPE(w, bias_dtype);
  FMHC_REQUIRE_DTYPE(w, y_dtype);
  if (int e = check_codes(w, "codes", codes_stride, K)) return e;
  if (int e = check_codes(w, "weight_codes", weight_stride, K)) return e;
  if (codes_stride % 16 || weight_stride % 16)
    return fail(FMHC_ERR_ALIGNMENT, "%s: rows of codes must be a multiple of 16 bytes apart", w);
  if (T == 0 || N == 0) return ok();
  FMHC_REQUIRE_PTR(w, codes); FMHC_REQUIRE_PTR(w, scales); FMHC_REQUIRE_PTR(w, weight_codes);
  FMHC_REQUIRE_PTR(w, weight_scales); FMHC_REQUIRE_PTR(w, y);
  FMHC_REQUIRE_ALIGN16(w, codes); FMHC_REQUIRE_ALIGN16(w, weight_codes);
  FMHC_REQUIRE_ALIGN_TO(w, scales, 4); FMHC_REQUIRE_ALIGN_TO(w, weight_scales, 4);
  FMHC_REQUIRE_ALIGN_TO(w, bias, dtype_size(bias_dtype)); FMHC_REQUIRE_ALIGN_TO(w, y, dtype_size(y_dtype));
  if (int e = fmhc::launch_int8_linear(codes, codes_stride, scales, weight_codes, weight_stride,
                                       weight_scales, bias, bias_dtype, y, y_dtype, T, N, int(K),
                                       (cudaStream_t)stream, lose_copy))
    return e;
  return check_launch(w);
}

int fmhc_int8_linear(const void *codes, int64_t codes_stride, const float *scales,
                     const void *weight_codes, int64_t weight_stride, const float *weight_scales,
                     const void *bias, int bias_dtype, void *y, int y_dtype, int64_t T, int64_t N,
                     int64_t K, void *stream) {
  return int8_linear("fmhc_int8_linear", codes, codes_stride, scales, weight_codes, weight_stride,
                     weight_scales, bias, bias_dtype, y, y_dtype, T, N, K, stream, false);
}

int fmhc_debug_int8_linear_lost_copy(const void *codes, int64_t codes_stride, const float *scales,
                                     const void *weight_codes, int64_t weight_stride,
                                     const float *weight_scales, void *y, int64_t T, int64_t N,
                                     int64_t K, void *stream) {
  return int8_linear("fmhc_debug_int8_linear_lost_copy", codes, codes_stride, scales, weight_codes,
                     weight_stride, weight_scales, nullptr, FMHC_DTYPE_F32, y, FMHC_DTYPE_BF16, T, N, K,
                     stream, true);
}

}  // extern "C"
