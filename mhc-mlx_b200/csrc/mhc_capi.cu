// extern "C" boundary of libmhc_b200.so: argument validation, error codes
// and the thread-local error text, then a call into the launchers.  The
// checks mirror the ValueError conditions of the reference launchers in
// mhc_mlx/metal.py (n in [1, 64] via _validate_n metal.py:826-833, shape and
// dtype agreement, output dtype fp32 or matching a half input
// metal.py:1610-1616).
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <mutex>
#include <tuple>

#include "mhc_internal.h"
#include "mhc_sinkhorn.cuh"

namespace mhc {

static thread_local char g_err[512] = "";

int set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int check_launch(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(MHC_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
  return MHC_OK;
}

static constexpr int kMaxDevices = 64;
static int g_sm[kMaxDevices];
static int g_smem[kMaxDevices];
static std::once_flag g_once[kMaxDevices];

static int current_device() {
  int d = 0;
  if (cudaGetDevice(&d) != cudaSuccess || d < 0 || d >= kMaxDevices) d = 0;
  return d;
}

static void query(int d) {
  int v = 0;
  g_sm[d] = (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, d) == cudaSuccess && v > 0) ? v : 148;
  v = 0;
  g_smem[d] = (cudaDeviceGetAttribute(&v, cudaDevAttrMaxSharedMemoryPerBlockOptin, d) == cudaSuccess && v > 0) ? v : 48 * 1024;
}

int sm_count() {
  const int d = current_device();
  std::call_once(g_once[d], query, d);
  return g_sm[d];
}

int max_smem_optin() {
  const int d = current_device();
  std::call_once(g_once[d], query, d);
  return g_smem[d];
}

bool pdl_enabled() {
  static const bool on = [] {
    const char* v = getenv("MHC_B200_PDL");
    return !(v && *v == '0');
  }();
  return on;
}

// Launch-attribute caches keyed on (kernel, device[, block, shared bytes]).
namespace {
std::mutex g_attr_mu;
std::map<std::pair<const void*, int>, size_t> g_dyn;  // largest dynamic smem allowed so far
std::map<std::tuple<const void*, int, int, size_t>, int> g_occ;  // resident blocks per SM
}  // namespace

bool dyn_smem_cached(const void* kernel, size_t dyn) {
  std::lock_guard<std::mutex> lk(g_attr_mu);
  auto it = g_dyn.find({kernel, current_device()});
  return it != g_dyn.end() && it->second >= dyn;
}

void dyn_smem_remember(const void* kernel, size_t dyn) {
  std::lock_guard<std::mutex> lk(g_attr_mu);
  size_t& v = g_dyn[{kernel, current_device()}];
  if (dyn > v) v = dyn;
}

int occupancy_cached(const void* kernel, int threads, size_t smem) {
  std::lock_guard<std::mutex> lk(g_attr_mu);
  auto it = g_occ.find({kernel, current_device(), threads, smem});
  return it == g_occ.end() ? -1 : it->second;
}

void occupancy_remember(const void* kernel, int threads, size_t smem, int per_sm) {
  std::lock_guard<std::mutex> lk(g_attr_mu);
  g_occ[{kernel, current_device(), threads, smem}] = per_sm;
}

}  // namespace mhc

using namespace mhc;

#define MHC_TRY_BEGIN try {
#define MHC_TRY_END                                                        \
  }                                                                        \
  catch (...) {                                                            \
    return set_error(MHC_ERR_CUDA, "%s: unexpected C++ exception", __func__); \
  }

static int check_common(const char* fn, int64_t T, int n, int C) {
  if (n < 1 || n > 64) return set_error(MHC_ERR_INVALID, "%s: n=%d must be in [1, 64]", fn, n);
  if (C < 1) return set_error(MHC_ERR_INVALID, "%s: C=%d must be positive", fn, C);
  if (T < 0) return set_error(MHC_ERR_INVALID, "%s: T=%lld must be >= 0", fn, (long long)T);
  return MHC_OK;
}

static int check_dtype(const char* fn, const char* what, int dt) {
  if (!dtype_ok(dt)) return set_error(MHC_ERR_INVALID, "%s: %s dtype %d is not one of MHC_F32/F16/BF16", fn, what, dt);
  return MHC_OK;
}

#define MHC_REQ(cond, ...) \
  do { if (!(cond)) return set_error(MHC_ERR_INVALID, __VA_ARGS__); } while (0)
#define MHC_CHK(expr) \
  do { const int _r = (expr); if (_r != MHC_OK) return _r; } while (0)

extern "C" {

const char* mhc_last_error(void) { return g_err; }

int mhc_version(void) { return 10000; }  // 1.0.0

#ifndef MHC_BUILD_ID
#define MHC_BUILD_ID "unknown"
#endif
const char* mhc_build_id(void) { return MHC_BUILD_ID; }

int mhc_device_sm_count(int* out) {
  MHC_REQ(out, "mhc_device_sm_count: NULL output");
  *out = sm_count();
  return MHC_OK;
}

int mhc_selftest_reciprocal(const float* x, float* y, int64_t count, void* stream) {
  MHC_TRY_BEGIN
  MHC_REQ(count >= 0, "mhc_selftest_reciprocal: count must be >= 0");
  MHC_REQ(count == 0 || (x && y), "mhc_selftest_reciprocal: NULL pointer");
  if (count == 0) return MHC_OK;
  return launch_selftest_reciprocal(x, y, count, as_stream(stream));
  MHC_TRY_END
}

size_t mhc_sinkhorn_tape_floats(int n, int iters) {
  if (n < 1 || n > 64 || iters < 0) return 0;
  return sk_tape_floats(n, iters);
}

int mhc_params_fwd(const float* H_pre_raw, const float* H_post_raw, const float* H_res_raw, int n,
                   int iters, float eps, float* H_pre_act, float* H_post_act, float* M,
                   float* tape, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, 1, n, 1));
  MHC_REQ(iters >= 0, "%s: iters=%d must be >= 0", __func__, iters);
  MHC_REQ(!H_pre_raw == !H_pre_act, "%s: H_pre_raw and H_pre_act must both be given or both NULL", __func__);
  MHC_REQ(!H_post_raw == !H_post_act, "%s: H_post_raw and H_post_act must both be given or both NULL", __func__);
  MHC_REQ(!H_res_raw || M, "%s: M is NULL", __func__);
  return launch_params_fwd(H_pre_raw, H_post_raw, H_res_raw, n, iters, eps, H_pre_act, H_post_act,
                           M, H_res_raw ? tape : nullptr, as_stream(stream));
  MHC_TRY_END
}

int mhc_params_bwd(const float* H_pre_raw, const float* H_post_raw, const float* H_res_raw,
                   const float* tape, int n, int iters, float eps, const float* dH_pre_act,
                   const float* dH_post_act, const float* dM, float* dH_pre_raw,
                   float* dH_post_raw, float* dH_res_raw, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, 1, n, 1));
  MHC_REQ(iters >= 0, "%s: iters=%d must be >= 0", __func__, iters);
  MHC_REQ(!(H_pre_raw && dH_pre_act) || dH_pre_raw, "%s: dH_pre_raw is NULL", __func__);
  MHC_REQ(!(H_post_raw && dH_post_act) || dH_post_raw, "%s: dH_post_raw is NULL", __func__);
  if (H_res_raw && dM) {
    MHC_REQ(dH_res_raw, "%s: dH_res_raw is NULL", __func__);
    MHC_REQ(tape || iters == 0, "%s: tape is NULL (record it with mhc_params_fwd)", __func__);
  }
  return launch_params_bwd(H_pre_raw, H_post_raw, H_res_raw, tape, n, iters, eps, dH_pre_act,
                           dH_post_act, dM, dH_pre_raw, dH_post_raw, dH_res_raw,
                           as_stream(stream));
  MHC_TRY_END
}

size_t mhc_sinkhorn_batched_workspace_bytes(int64_t batch, int n, int iters) {
  if (n < 1 || n > 64 || iters < 0 || batch < 0) return 0;
  return sk_batched_ws_bytes(batch, n, iters);
}

int mhc_sinkhorn_batched_fwd(const float* H_res_raw, int64_t batch, int n, int iters, float eps,
                             float* M, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, batch, n, 1));
  MHC_REQ(iters >= 0, "%s: iters=%d must be >= 0", __func__, iters);
  MHC_REQ(batch == 0 || (H_res_raw && M), "%s: NULL pointer", __func__);
  MHC_REQ(batch * n <= (int64_t)INT32_MAX * 64, "%s: batch too large", __func__);
  return launch_sk_batched_fwd(H_res_raw, batch, n, iters, eps, M, nullptr, 0, as_stream(stream));
  MHC_TRY_END
}

int mhc_sinkhorn_batched_bwd(const float* H_res_raw, const float* dM, int64_t batch, int n,
                             int iters, float eps, float* dH_res_raw, void* workspace,
                             size_t workspace_bytes, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, batch, n, 1));
  MHC_REQ(iters >= 0, "%s: iters=%d must be >= 0", __func__, iters);
  MHC_REQ(batch == 0 || (H_res_raw && dM && dH_res_raw), "%s: NULL pointer", __func__);
  return launch_sk_batched_bwd(H_res_raw, dM, batch, n, iters, eps, dH_res_raw, workspace,
                               workspace_bytes, as_stream(stream));
  MHC_TRY_END
}

int mhc_fwd(const void* x, int x_dtype, const float* M, const float* H_pre_act,
            const float* H_post_act, const float* rms_weight, void* out, int out_dtype, int64_t T,
            int n, int C, float eps, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, T, n, C));
  MHC_CHK(check_dtype(__func__, "x", x_dtype));
  MHC_CHK(check_dtype(__func__, "out", out_dtype));
  MHC_REQ(out_dtype == MHC_F32 || out_dtype == x_dtype,
          "%s: out dtype must be fp32 or equal to x's dtype", __func__);
  MHC_REQ(M && H_pre_act && H_post_act && rms_weight, "%s: NULL parameter pointer", __func__);
  MHC_REQ(T == 0 || (x && out), "%s: NULL x/out", __func__);
  return launch_fwd(x, x_dtype, M, H_pre_act, H_post_act, rms_weight, out, out_dtype, T, n, C, eps,
                    as_stream(stream));
  MHC_TRY_END
}

size_t mhc_bwd_workspace_bytes(int64_t T, int n, int C) {
  if (n < 1 || n > 64 || C < 1 || T < 0) return 0;
  return bwd_ws_bytes(T, n, C);
}

int mhc_bwd(const void* x, int x_dtype, const void* d_out, int dout_dtype, const float* M,
            const float* H_pre_act, const float* H_post_act, const float* rms_weight, void* dx,
            int dx_dtype, int64_t T, int n, int C, float eps, void* workspace,
            size_t workspace_bytes, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, T, n, C));
  MHC_CHK(check_dtype(__func__, "x", x_dtype));
  MHC_CHK(check_dtype(__func__, "d_out", dout_dtype));
  MHC_CHK(check_dtype(__func__, "dx", dx_dtype));
  MHC_REQ(M && H_pre_act && H_post_act && rms_weight, "%s: NULL parameter pointer", __func__);
  MHC_REQ(T == 0 || (x && d_out && dx), "%s: NULL x/d_out/dx", __func__);
  return launch_bwd(x, x_dtype, d_out, dout_dtype, M, H_pre_act, H_post_act, rms_weight, dx,
                    dx_dtype, T, n, C, eps, workspace, workspace_bytes, as_stream(stream));
  MHC_TRY_END
}

int mhc_bwd_finalize(const void* workspace, int n, int C, float* dM, float* dH_pre_act,
                     float* dH_post_act, float* d_rms_weight, const float* H_pre_raw,
                     const float* H_post_raw, const float* H_res_raw, const float* tape,
                     int iters, float eps, float* dH_pre_raw, float* dH_post_raw,
                     float* dH_res_raw, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, 0, n, C));
  MHC_REQ(workspace, "%s: NULL workspace", __func__);
  MHC_REQ(iters >= 0, "%s: iters=%d must be >= 0", __func__, iters);
  if (H_res_raw && dH_res_raw)
    MHC_REQ(tape || iters == 0, "%s: tape is NULL (record it with mhc_params_fwd)", __func__);
  return launch_finalize(workspace, n, C, dM, dH_pre_act, dH_post_act, d_rms_weight, H_pre_raw,
                         H_post_raw, H_res_raw, tape, iters, eps, dH_pre_raw, dH_post_raw,
                         dH_res_raw, as_stream(stream));
  MHC_TRY_END
}

int mhc_mix_add_fwd(const void* x, int x_dtype, const float* M, const void* y_dist, int y_dtype,
                    void* out, int out_dtype, int64_t T, int n, int C, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, T, n, C));
  MHC_CHK(check_dtype(__func__, "x", x_dtype));
  MHC_CHK(check_dtype(__func__, "y_dist", y_dtype));
  MHC_CHK(check_dtype(__func__, "out", out_dtype));
  MHC_REQ(M, "%s: NULL M", __func__);
  MHC_REQ(T == 0 || (x && y_dist && out), "%s: NULL tensor pointer", __func__);
  return launch_mix_add_fwd(x, x_dtype, M, y_dist, y_dtype, out, out_dtype, T, n, C,
                            as_stream(stream));
  MHC_TRY_END
}

size_t mhc_mix_bwd_workspace_bytes(int64_t T, int n, int C) {
  if (n < 1 || n > 64 || C < 1 || T < 0) return 0;
  return mix_ws_bytes(T, n, C);
}

int mhc_mix_add_bwd(const void* x, int x_dtype, const float* M, const void* d_out, int dout_dtype,
                    void* dx, int dx_dtype, float* dM, int64_t T, int n, int C, void* workspace,
                    size_t workspace_bytes, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, T, n, C));
  MHC_CHK(check_dtype(__func__, "x", x_dtype));
  MHC_CHK(check_dtype(__func__, "d_out", dout_dtype));
  MHC_CHK(check_dtype(__func__, "dx", dx_dtype));
  MHC_REQ(M && dM, "%s: NULL M/dM", __func__);
  MHC_REQ(T == 0 || (x && d_out && dx), "%s: NULL tensor pointer", __func__);
  return launch_mix_add_bwd(x, x_dtype, M, d_out, dout_dtype, dx, dx_dtype, dM, T, n, C, workspace,
                            workspace_bytes, as_stream(stream));
  MHC_TRY_END
}

int mhc_rewire_combine_fwd(const void* x, int x_dtype, const void* y_inner, int y_dtype,
                           const float* M, const float* H_pre_act, const float* H_post_act,
                           void* out, int out_dtype, int64_t T, int n, int C, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, T, n, C));
  MHC_CHK(check_dtype(__func__, "x", x_dtype));
  MHC_CHK(check_dtype(__func__, "y_inner", y_dtype));
  MHC_CHK(check_dtype(__func__, "out", out_dtype));
  MHC_REQ(M && H_pre_act && H_post_act, "%s: NULL parameter pointer", __func__);
  MHC_REQ(T == 0 || (x && y_inner && out), "%s: NULL tensor pointer", __func__);
  return launch_rewire_fwd(x, x_dtype, y_inner, y_dtype, M, H_pre_act, H_post_act, out, out_dtype,
                           T, n, C, as_stream(stream));
  MHC_TRY_END
}

size_t mhc_rewire_bwd_workspace_bytes(int64_t T, int n, int C) {
  return mhc_mix_bwd_workspace_bytes(T, n, C);
}

int mhc_rewire_combine_bwd(const void* x, int x_dtype, const void* y_inner, int y_dtype,
                           const void* d_out, int dout_dtype, const float* M,
                           const float* H_pre_act, const float* H_post_act, void* dx, int dx_dtype,
                           void* dy_inner, int dy_dtype, float* dM, float* dH_pre_act,
                           float* dH_post_act, int64_t T, int n, int C, void* workspace,
                           size_t workspace_bytes, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, T, n, C));
  MHC_CHK(check_dtype(__func__, "x", x_dtype));
  MHC_CHK(check_dtype(__func__, "y_inner", y_dtype));
  MHC_CHK(check_dtype(__func__, "d_out", dout_dtype));
  MHC_CHK(check_dtype(__func__, "dx", dx_dtype));
  MHC_CHK(check_dtype(__func__, "dy_inner", dy_dtype));
  MHC_REQ(M && H_pre_act && H_post_act, "%s: NULL parameter pointer", __func__);
  MHC_REQ(dM && dH_pre_act && dH_post_act, "%s: NULL gradient pointer", __func__);
  MHC_REQ(T == 0 || (x && y_inner && d_out && dx && dy_inner), "%s: NULL tensor pointer", __func__);
  return launch_rewire_bwd(x, x_dtype, y_inner, y_dtype, d_out, dout_dtype, M, H_pre_act,
                           H_post_act, dx, dx_dtype, dy_inner, dy_dtype, dM, dH_pre_act,
                           dH_post_act, T, n, C, workspace, workspace_bytes, as_stream(stream));
  MHC_TRY_END
}

size_t mhc_rewire_fused_bwd_workspace_bytes(int64_t T, int n, int C) {
  if (n < 1 || n > 64 || C < 1 || T < 0) return 0;
  return rewire_fused_ws_bytes(T, n, C);
}

int mhc_rewire_bwd_dy(const void* y_inner, int y_dtype, const void* d_out, int dout_dtype,
                      const float* H_post_act, void* dy_inner, int dy_dtype, int64_t T, int n,
                      int C, void* workspace, size_t workspace_bytes, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, T, n, C));
  MHC_CHK(check_dtype(__func__, "y_inner", y_dtype));
  MHC_CHK(check_dtype(__func__, "d_out", dout_dtype));
  MHC_CHK(check_dtype(__func__, "dy_inner", dy_dtype));
  MHC_REQ(H_post_act, "%s: NULL parameter pointer", __func__);
  MHC_REQ(T == 0 || (y_inner && d_out && dy_inner), "%s: NULL tensor pointer", __func__);
  return launch_rewire_bwd_dy(y_inner, y_dtype, d_out, dout_dtype, H_post_act, dy_inner, dy_dtype,
                              T, n, C, workspace, workspace_bytes, as_stream(stream));
  MHC_TRY_END
}

int mhc_rewire_bwd_dx(const void* x, int x_dtype, const void* d_out, int dout_dtype,
                      const void* d_xpre, int dxpre_dtype, const float* M, const float* H_pre_act,
                      const float* H_post_act, void* dx, int dx_dtype, float* dM,
                      float* dH_pre_act, float* dH_post_act, const float* H_pre_raw,
                      const float* H_post_raw, const float* H_res_raw, const float* tape,
                      const float* jacobian, int iters, float eps, float* dH_pre_raw,
                      float* dH_post_raw, float* dH_res_raw, int64_t T, int n, int C,
                      void* workspace, size_t workspace_bytes, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, T, n, C));
  MHC_CHK(check_dtype(__func__, "x", x_dtype));
  MHC_CHK(check_dtype(__func__, "d_out", dout_dtype));
  MHC_CHK(check_dtype(__func__, "d_xpre", dxpre_dtype));
  MHC_CHK(check_dtype(__func__, "dx", dx_dtype));
  MHC_REQ(M && H_pre_act && H_post_act, "%s: NULL parameter pointer", __func__);
  MHC_REQ(dM && dH_pre_act && dH_post_act, "%s: NULL gradient pointer", __func__);
  MHC_REQ(T == 0 || (x && d_out), "%s: NULL tensor pointer", __func__);
  MHC_REQ(!H_pre_raw == !dH_pre_raw, "%s: H_pre_raw and dH_pre_raw must both be given or both NULL", __func__);
  MHC_REQ(!H_post_raw == !dH_post_raw, "%s: H_post_raw and dH_post_raw must both be given or both NULL", __func__);
  MHC_REQ(!H_res_raw == !dH_res_raw, "%s: H_res_raw and dH_res_raw must both be given or both NULL", __func__);
  if (H_res_raw) {
    MHC_REQ(iters >= 0, "%s: iters=%d must be >= 0", __func__, iters);
    MHC_REQ(tape || jacobian || iters == 0, "%s: tape is NULL (record it with mhc_rewire_in_fwd)", __func__);
  }
  MHC_REQ(!jacobian || sk_lane_ok(n), "%s: a Jacobian exists for n in {1, 2, 4} only (n=%d)", __func__, n);
  const ParamsBwd pb{H_pre_raw, H_post_raw, H_res_raw, tape, jacobian, iters, eps,
                     dH_pre_raw, dH_post_raw, dH_res_raw};
  return launch_rewire_bwd_dx(x, x_dtype, d_out, dout_dtype, d_xpre, dxpre_dtype, M, H_pre_act,
                              H_post_act, dx, dx_dtype, dM, dH_pre_act, dH_post_act, pb, T, n, C,
                              workspace, workspace_bytes, as_stream(stream));
  MHC_TRY_END
}

size_t mhc_rewire_jacobian_floats(int n) {
  if (n < 1 || n > 64) return 0;
  return sk_jacobian_floats(n);
}

int mhc_rewire_in_fwd(const void* x, int x_dtype, const float* H_pre_raw, const float* H_post_raw,
                      const float* H_res_raw, int iters, float eps, float* H_pre_act,
                      float* H_post_act, float* M, float* tape, float* jacobian, void* x_pre,
                      int out_dtype, int64_t T, int n, int C, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, T, n, C));
  MHC_CHK(check_dtype(__func__, "x", x_dtype));
  MHC_CHK(check_dtype(__func__, "x_pre", out_dtype));
  MHC_REQ(iters >= 0, "%s: iters=%d must be >= 0", __func__, iters);
  MHC_REQ(H_pre_raw && H_post_raw && H_res_raw, "%s: NULL raw parameter pointer", __func__);
  MHC_REQ(H_pre_act && H_post_act && M, "%s: NULL activation pointer", __func__);
  MHC_REQ(tape || iters == 0, "%s: tape is NULL", __func__);
  MHC_REQ(!jacobian || sk_lane_ok(n), "%s: a Jacobian exists for n in {1, 2, 4} only (n=%d)", __func__, n);
  MHC_REQ(T == 0 || (x && x_pre), "%s: NULL tensor pointer", __func__);
  const ParamsFwd pf{H_pre_raw, H_post_raw, H_res_raw, iters, eps, H_pre_act, H_post_act, M,
                     tape, jacobian, 0};
  return launch_rewire_in_fwd(x, x_dtype, pf, x_pre, out_dtype, T, n, C, as_stream(stream));
  MHC_TRY_END
}

int mhc_prescale_fwd(const void* x, int x_dtype, const float* H_pre_act, void* x_pre,
                     int out_dtype, int64_t T, int n, int C, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, T, n, C));
  MHC_CHK(check_dtype(__func__, "x", x_dtype));
  MHC_CHK(check_dtype(__func__, "x_pre", out_dtype));
  MHC_REQ(H_pre_act, "%s: NULL H_pre_act", __func__);
  MHC_REQ(T == 0 || (x && x_pre), "%s: NULL tensor pointer", __func__);
  return launch_prescale_fwd(x, x_dtype, H_pre_act, x_pre, out_dtype, T, n, C, as_stream(stream));
  MHC_TRY_END
}

int mhc_prescale_bwd(const void* x, int x_dtype, const void* d_xpre, int d_dtype,
                     const float* H_pre_act, void* dx, int dx_dtype, float* dH_pre_act, int64_t T,
                     int n, int C, void* workspace, size_t workspace_bytes, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, T, n, C));
  MHC_CHK(check_dtype(__func__, "x", x_dtype));
  MHC_CHK(check_dtype(__func__, "d_xpre", d_dtype));
  MHC_CHK(check_dtype(__func__, "dx", dx_dtype));
  MHC_REQ(H_pre_act && dH_pre_act, "%s: NULL parameter pointer", __func__);
  MHC_REQ(T == 0 || (x && d_xpre && dx), "%s: NULL tensor pointer", __func__);
  return launch_prescale_bwd(x, x_dtype, d_xpre, d_dtype, H_pre_act, dx, dx_dtype, dH_pre_act, T, n,
                             C, workspace, workspace_bytes, as_stream(stream));
  MHC_TRY_END
}

int mhc_qlinear_fwd(const void* x, int x_dtype, const uint32_t* w_packed, const void* scales,
                    const void* biases, int scales_dtype, const void* bias, void* y, int64_t M,
                    int N, int K, int group_size, int bits, void* stream) {
  MHC_TRY_BEGIN
  return launch_qlinear_fwd(x, x_dtype, w_packed, scales, biases, scales_dtype, bias, y, M, N, K,
                            group_size, bits, as_stream(stream));
  MHC_TRY_END
}

int mhc_qlinear_bwd_dx(const void* dy, int dy_dtype, const uint32_t* w_packed,
                       const void* scales, const void* biases, int scales_dtype, void* dx,
                       int64_t M, int N, int K, int group_size, int bits, void* stream) {
  MHC_TRY_BEGIN
  return launch_qlinear_bwd_dx(dy, dy_dtype, w_packed, scales, biases, scales_dtype, dx, M, N, K,
                               group_size, bits, as_stream(stream));
  MHC_TRY_END
}

int mhc_qlinear_transpose_pack(const uint32_t* w_packed, uint32_t* wt_packed, int N, int K,
                               void* stream) {
  MHC_TRY_BEGIN
  return launch_qlinear_transpose_pack(w_packed, wt_packed, N, K, as_stream(stream));
  MHC_TRY_END
}

int mhc_qlinear_bwd_dx_t(const void* dy, int dy_dtype, const uint32_t* wt_packed,
                         const void* scales_t, const void* biases_t, void* dx, int64_t M, int N,
                         int K, int group_size, int bits, void* stream) {
  MHC_TRY_BEGIN
  return launch_qlinear_bwd_dx_t(dy, dy_dtype, wt_packed, scales_t, biases_t, dx, M, N, K,
                                 group_size, bits, as_stream(stream));
  MHC_TRY_END
}

int mhc_residual_add_agg(const void* x, int x_dtype, const void* res, int res_dtype,
                         const float* H_pre, void* out, int out_dtype, float* y_agg, int64_t T,
                         int n, int C, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, T, n, C));
  MHC_CHK(check_dtype(__func__, "x", x_dtype));
  MHC_CHK(check_dtype(__func__, "res", res_dtype));
  MHC_CHK(check_dtype(__func__, "out", out_dtype));
  MHC_REQ(H_pre, "%s: NULL H_pre", __func__);
  MHC_REQ(T == 0 || (x && res && out && y_agg), "%s: NULL tensor pointer", __func__);
  return launch_residual_add_agg(x, x_dtype, res, res_dtype, H_pre, out, out_dtype, y_agg, T, n, C,
                                 as_stream(stream));
  MHC_TRY_END
}

int mhc_residual_add_agg_bwd(const void* out, int out_dtype, const void* d_out, int dout_dtype,
                             const float* d_y, const float* H_pre, void* dx, int dx_dtype,
                             float* dH_pre, int64_t T, int n, int C, void* workspace,
                             size_t workspace_bytes, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_common(__func__, T, n, C));
  MHC_CHK(check_dtype(__func__, "out", out_dtype));
  MHC_CHK(check_dtype(__func__, "dx", dx_dtype));
  if (d_out) MHC_CHK(check_dtype(__func__, "d_out", dout_dtype));
  MHC_REQ(H_pre && dH_pre, "%s: NULL H_pre/dH_pre", __func__);
  MHC_REQ(T == 0 || (out && dx), "%s: NULL out/dx", __func__);
  return launch_residual_add_agg_bwd(out, out_dtype, d_out, d_out ? dout_dtype : out_dtype, d_y,
                                     H_pre, dx, dx_dtype, dH_pre, T, n, C, workspace,
                                     workspace_bytes, as_stream(stream));
  MHC_TRY_END
}

// ---- losses on logits ----
static int check_logits(const char* fn, const LogitsArg& l) {
  MHC_CHK(check_dtype(fn, "logits", l.dtype));
  MHC_REQ(l.rows >= 0 && l.rows < ((int64_t)1 << 28), "%s: rows=%lld must be in [0, 2^28)", fn, (long long)l.rows);
  MHC_REQ(l.vocab >= 1 && l.vocab < ((int64_t)1 << 31), "%s: V=%lld must be in [1, 2^31)", fn, (long long)l.vocab);
  MHC_REQ(l.per_batch >= 1, "%s: rows_per_batch=%lld must be positive", fn, (long long)l.per_batch);
  MHC_REQ(l.rows == 0 || (l.logits && l.targets), "%s: NULL logits/targets", fn);
  const uintptr_t size = (uintptr_t)dtype_size(l.dtype);
  MHC_REQ(reinterpret_cast<uintptr_t>(l.logits) % size == 0, "%s: logits are not aligned to their type", fn);
  return MHC_OK;
}

int mhc_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t rows_per_batch,
                       int64_t batch_stride, int64_t row_stride, int64_t V, const int64_t* targets,
                       int64_t ignore_index, float* logp, float* stats, void* stream) {
  MHC_TRY_BEGIN
  const LogitsArg l = {logits, dtype, rows, rows_per_batch, batch_stride, row_stride, V, targets, ignore_index};
  MHC_CHK(check_logits(__func__, l));
  MHC_REQ(rows == 0 || (logp && stats), "%s: NULL logp/stats", __func__);
  MHC_REQ(aligned16(stats), "%s: stats must be 16-byte aligned", __func__);
  return launch_token_logprobs(l, logp, stats, as_stream(stream));
  MHC_TRY_END
}

int mhc_logits_grad(const void* logits, int dtype, int64_t rows, int64_t rows_per_batch,
                    int64_t batch_stride, int64_t row_stride, int64_t V, const int64_t* targets,
                    int64_t ignore_index, const float* stats, const float* coef, float scale,
                    const float* scale_ptr, int unless_one, void* dlogits, void* stream) {
  MHC_TRY_BEGIN
  const LogitsArg l = {logits, dtype, rows, rows_per_batch, batch_stride, row_stride, V, targets, ignore_index};
  MHC_CHK(check_logits(__func__, l));
  MHC_REQ(rows == 0 || (stats && coef && dlogits), "%s: NULL stats/coef/dlogits", __func__);
  MHC_REQ(!unless_one || scale_ptr, "%s: unless_one needs scale_ptr", __func__);
  MHC_REQ(aligned16(stats), "%s: stats must be 16-byte aligned", __func__);
  return launch_logits_grad(l, stats, coef, scale, scale_ptr, unless_one, dlogits, as_stream(stream));
  MHC_TRY_END
}

int mhc_preference_loss(const void* logits, int dtype, int64_t rows, int64_t rows_per_batch,
                        int64_t batch_stride, int64_t row_stride, int64_t V,
                        const int64_t* targets, int64_t ignore_index, const void* cu_seqlens,
                        int cu_is64, int64_t uniform_len, int64_t pairs, const float* ref_logp,
                        float beta, float label_smoothing, float inv_denominator,
                        float grad_scale, float* logp, float* stats, float* coef, float* margins,
                        float* loss, void* dlogits, void* stream) {
  MHC_TRY_BEGIN
  const LogitsArg l = {logits, dtype, rows, rows_per_batch, batch_stride, row_stride, V, targets, ignore_index};
  MHC_CHK(check_logits(__func__, l));
  MHC_REQ(pairs >= 1 && pairs < ((int64_t)1 << 30), "%s: pairs=%lld must be in [1, 2^30)", __func__, (long long)pairs);
  MHC_REQ(cu_seqlens || (uniform_len >= 0 && uniform_len <= rows), "%s: uniform_len=%lld must be in [0, rows]", __func__, (long long)uniform_len);
  MHC_REQ(label_smoothing >= 0.f && label_smoothing < 1.f, "%s: label_smoothing must be in [0, 1)", __func__);
  MHC_REQ(margins && loss && (rows == 0 || (ref_logp && logp && stats && coef)), "%s: NULL pointer", __func__);
  MHC_REQ(aligned16(stats), "%s: stats must be 16-byte aligned", __func__);
  const PreferenceArg a = {cu_seqlens, cu_is64, uniform_len, pairs, ref_logp, beta, label_smoothing, inv_denominator, grad_scale};
  const PreferenceOut o = {logp, stats, coef, margins, loss, dlogits};
  return launch_preference(l, a, o, as_stream(stream));
  MHC_TRY_END
}

// Workspace of the policy loss: a counter and 1 / D, then two fp64 sums for
// each cluster of blocks.
static constexpr size_t kLossHeader = 256;
size_t mhc_policy_workspace_bytes(void) {
  return kLossHeader + (size_t)sm_count() * kPolicyClustersSM * 2 * sizeof(double);
}

int mhc_policy_loss(const void* logits, int dtype, int64_t rows, int64_t rows_per_batch,
                    int64_t batch_stride, int64_t row_stride, int64_t V, const int64_t* targets,
                    int64_t ignore_index, const float* old_logp, const float* advantages,
                    const float* ref_logp, float clip_low, float clip_high, float kl_coef,
                    float inv_denominator, float grad_scale, float* logp, float* stats,
                    float* coef, float* loss, float* kl, void* dlogits, void* workspace,
                    size_t workspace_bytes, void* stream) {
  MHC_TRY_BEGIN
  const LogitsArg l = {logits, dtype, rows, rows_per_batch, batch_stride, row_stride, V, targets, ignore_index};
  MHC_CHK(check_logits(__func__, l));
  MHC_REQ(clip_low >= 0.f && clip_high >= 0.f, "%s: clip_low and clip_high must be >= 0", __func__);
  MHC_REQ(kl_coef == 0.f || ref_logp, "%s: kl_coef needs ref_logp", __func__);
  MHC_REQ(inv_denominator >= 0.f, "%s: inv_denominator must be >= 0", __func__);
  MHC_REQ(loss && kl && (rows == 0 || (old_logp && advantages && logp && stats && coef)), "%s: NULL pointer", __func__);
  if (!workspace || workspace_bytes < mhc_policy_workspace_bytes())
    return set_error(MHC_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", __func__, workspace_bytes, mhc_policy_workspace_bytes());
  MHC_REQ(aligned16(stats) && aligned16(workspace), "%s: stats and workspace must be 16-byte aligned", __func__);
  const PolicyArg a = {old_logp, advantages, ref_logp, clip_low, clip_high, kl_coef, inv_denominator, grad_scale};
  char* ws = static_cast<char*>(workspace);
  const PolicyOut o = {logp, stats, coef, loss, kl, reinterpret_cast<unsigned*>(ws),
                       reinterpret_cast<float*>(ws) + 1, reinterpret_cast<double*>(ws + kLossHeader), dlogits};
  return launch_policy(l, a, o, as_stream(stream));
  MHC_TRY_END
}

// ---- AdamW ----
int mhc_adamw_step(int count, void* const* params, const void* const* grads, const int64_t* numel,
                   const int64_t* offsets, int dtype, int state_bits, void* exp_avg,
                   float* exp_avg_scale, void* exp_avg_sq, float* exp_avg_sq_scale, float* master,
                   float beta1, float one_minus_beta1, float beta2, float one_minus_beta2,
                   float decay, float step_size, float inv_sqrt_correction, float eps,
                   const float* grad_scale, uint32_t key, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_dtype(__func__, "params", dtype));
  MHC_REQ(count >= 0, "%s: count=%d must be >= 0", __func__, count);
  MHC_REQ(state_bits == 8 || state_bits == 32, "%s: state_bits=%d must be 8 or 32", __func__, state_bits);
  MHC_REQ(!master || dtype != MHC_F32, "%s: master weights are for 16-bit parameters", __func__);
  if (count == 0) return MHC_OK;
  MHC_REQ(params && grads && numel && offsets, "%s: NULL array", __func__);
  MHC_REQ(exp_avg && exp_avg_sq, "%s: NULL state", __func__);
  MHC_REQ(state_bits == 32 || (exp_avg_scale && exp_avg_sq_scale), "%s: 8-bit state needs its scales", __func__);
  MHC_REQ(aligned16(exp_avg) && aligned16(exp_avg_sq) && aligned16(master), "%s: the state must be 16-byte aligned", __func__);
  const uintptr_t size = (uintptr_t)dtype_size(dtype);
  for (int i = 0; i < count; ++i) {
    MHC_REQ(numel[i] >= 0, "%s: numel[%d] is negative", __func__, i);
    MHC_REQ(offsets[i] >= 0 && offsets[i] % 256 == 0 && offsets[i] / 256 < ((int64_t)1 << 32), "%s: offsets[%d] must be a multiple of 256 below 2^40", __func__, i);
    MHC_REQ(numel[i] == 0 || (params[i] && grads[i]), "%s: NULL tensor %d", __func__, i);
    MHC_REQ(reinterpret_cast<uintptr_t>(params[i]) % size == 0 && reinterpret_cast<uintptr_t>(grads[i]) % size == 0, "%s: tensor %d is not aligned to its type", __func__, i);
  }
  const AdamWArg a = {count, params, grads, numel, offsets, dtype, state_bits, exp_avg, exp_avg_sq,
                      exp_avg_scale, exp_avg_sq_scale, master, beta1, one_minus_beta1, beta2,
                      one_minus_beta2, decay, step_size, inv_sqrt_correction, eps, grad_scale, key};
  return launch_adamw(a, as_stream(stream));
  MHC_TRY_END
}

// ---- linear layer with its epilogue ----
static int check_linear(const char* fn, int dtype, int act, int64_t M, int64_t N, int64_t K) {
  if (dtype != MHC_BF16 && dtype != MHC_F16)
    return set_error(dtype_ok(dtype) ? MHC_ERR_UNSUPPORTED : MHC_ERR_INVALID, "%s: dtype %d is not MHC_F16 or MHC_BF16", fn, dtype);
  MHC_REQ(act >= 0 && act <= 3, "%s: act=%d must be in [0, 3]", fn, act);
  MHC_REQ(M >= 0 && M < ((int64_t)1 << 31), "%s: M=%lld must be in [0, 2^31)", fn, (long long)M);
  MHC_REQ(N >= 1 && N < ((int64_t)1 << 31), "%s: N=%lld must be in [1, 2^31)", fn, (long long)N);
  MHC_REQ(K >= 1 && K < ((int64_t)1 << 31), "%s: K=%lld must be in [1, 2^31)", fn, (long long)K);
  return MHC_OK;
}
static int check_rows(const char* fn, const char* what, const void* p, int64_t ld, int64_t cols) {
  MHC_REQ(p, "%s: NULL %s", fn, what);
  MHC_REQ(reinterpret_cast<uintptr_t>(p) % 2 == 0, "%s: %s is not aligned to its type", fn, what);
  MHC_REQ(ld >= cols, "%s: rows of %s are %lld apart, %lld values long", fn, what, (long long)ld, (long long)cols);
  return MHC_OK;
}

size_t mhc_linear_fwd_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw,
                                      int64_t M, int64_t N, int64_t K) {
  if (M < 1 || N < 1 || K < 1) return 0;
  return linear_fwd_ws_bytes(x, ldx, w, ldw, M, N, K);
}

int mhc_linear_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                   const void* residual, int64_t ldr, int dtype, int act, float* z, int64_t ldz,
                   void* y, int64_t ldy, int64_t M, int64_t N, int64_t K, void* workspace,
                   size_t workspace_bytes, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_linear(__func__, dtype, act, M, N, K));
  if (M == 0) return MHC_OK;
  MHC_CHK(check_rows(__func__, "x", x, ldx, K));
  MHC_CHK(check_rows(__func__, "w", w, ldw, K));
  MHC_CHK(check_rows(__func__, "y", y, ldy, N));
  if (bias) MHC_CHK(check_rows(__func__, "bias", bias, N, N));
  if (residual) MHC_CHK(check_rows(__func__, "residual", residual, ldr, N));
  if (z) {
    MHC_CHK(check_rows(__func__, "z", z, ldz, N));
    MHC_REQ(aligned16(z) && ldz % 8 == 0, "%s: z must be 16-byte aligned, its rows multiples of 8", __func__);
  }
  const LinearArg l = {x, w, bias, residual, ldx, ldw, ldr, dtype, act, M, N, K, z, ldz, y, ldy, workspace, workspace ? workspace_bytes : 0};
  if (l.workspace_bytes < linear_fwd_ws_bytes(x, ldx, w, ldw, M, N, K))
    return set_error(MHC_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", __func__, l.workspace_bytes, linear_fwd_ws_bytes(x, ldx, w, ldw, M, N, K));
  MHC_REQ(aligned16(workspace), "%s: the workspace must be 16-byte aligned", __func__);
  return launch_linear_fwd(l, as_stream(stream));
  MHC_TRY_END
}

size_t mhc_linear_bwd_workspace_bytes(const void* dy, int64_t ldy, const void* x, int64_t ldx,
                                      const void* w, int64_t ldw, int act, int want_dx,
                                      int want_dw, int want_dbias, int64_t M, int64_t N,
                                      int64_t K) {
  if (M < 1 || N < 1 || K < 1) return 0;
  char some = 0;  // stands for an output that is wanted
  LinearGradArg l = {};
  l.dy = dy; l.ldy = ldy; l.x = x; l.ldx = ldx; l.w = w; l.ldw = ldw; l.act = act;
  l.M = M; l.N = N; l.K = K;
  l.dx = want_dx ? &some : nullptr;
  l.dw = want_dw ? &some : nullptr;
  l.dbias = want_dbias ? &some : nullptr;
  return linear_bwd_ws_bytes(l);
}

int mhc_linear_bwd(const void* dy, int64_t ldy, const float* z, int64_t ldz, const void* x,
                   int64_t ldx, const void* w, int64_t ldw, int dtype, int act, void* dx,
                   int64_t lddx, void* dw, int64_t lddw, void* dbias, int64_t M, int64_t N,
                   int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  MHC_TRY_BEGIN
  MHC_CHK(check_linear(__func__, dtype, act, M, N, K));
  if (dw) MHC_CHK(check_rows(__func__, "dw", dw, lddw, K));
  if (M == 0) {
    cudaError_t e = cudaSuccess;
    if (dw) e = cudaMemset2DAsync(dw, (size_t)lddw * 2, 0, (size_t)K * 2, (size_t)N, as_stream(stream));
    if (dbias && e == cudaSuccess) e = cudaMemsetAsync(dbias, 0, (size_t)N * 2, as_stream(stream));
    if (e != cudaSuccess) return set_error(MHC_ERR_CUDA, "%s: %s", __func__, cudaGetErrorString(e));
    return MHC_OK;
  }
  MHC_CHK(check_rows(__func__, "dy", dy, ldy, N));
  if (act != 0) {
    MHC_CHK(check_rows(__func__, "z", z, ldz, N));
    MHC_REQ(aligned16(z) && ldz % 8 == 0, "%s: z must be 16-byte aligned, its rows multiples of 8", __func__);
  }
  if (dx) {
    MHC_CHK(check_rows(__func__, "dx", dx, lddx, K));
    MHC_CHK(check_rows(__func__, "w", w, ldw, K));
  }
  if (dw) MHC_CHK(check_rows(__func__, "x", x, ldx, K));
  if (dbias) MHC_CHK(check_rows(__func__, "dbias", dbias, N, N));
  const LinearGradArg l = {dy, z, x, w, ldy, ldz, ldx, ldw, dtype, act, M, N, K, dx, dw, dbias, lddx, lddw, workspace, workspace ? workspace_bytes : 0};
  if (l.workspace_bytes < linear_bwd_ws_bytes(l))
    return set_error(MHC_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", __func__, l.workspace_bytes, linear_bwd_ws_bytes(l));
  MHC_REQ(aligned16(workspace), "%s: the workspace must be 16-byte aligned", __func__);
  return launch_linear_bwd(l, as_stream(stream));
  MHC_TRY_END
}

}  // extern "C"
