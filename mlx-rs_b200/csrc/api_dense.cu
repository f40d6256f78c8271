// api_dense.cu — extern "C" entry points of the dense operators (include/moe_b200.h):
// 4-bit matrix products at every MLX group size, the gated feed-forward block with its
// backward pass, and the rotary positions. Their workspace comes from the caller, so calls
// on different streams and captured graphs share nothing.
#include <cuda_runtime.h>

#include <algorithm>
#include <utility>
#include <cstdarg>
#include <cstdio>
#include <cmath>
#include <cstring>

#include "../../include/moe_b200.h"
#include "dense.cuh"

namespace moe_internal {
int ctx_device(const moe_ctx* ctx);
void* ctx_stream(const moe_ctx* ctx);
void ctx_set_error(moe_ctx* ctx, const char* msg);
}  // namespace moe_internal

namespace {

int fail(moe_ctx* ctx, int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  if (ctx) moe_internal::ctx_set_error(ctx, buf);
  return code;
}

#define DENSE_CUDA(ctx, fn, expr)                                                                       \
  do {                                                                                                  \
    cudaError_t _e = (expr);                                                                            \
    if (_e != cudaSuccess) return fail((ctx), MOE_ERR_CUDA, "%s: %s", (fn), cudaGetErrorString(_e));    \
  } while (0)

struct DeviceGuard {
  int prev = -1;
  bool ok = true;
  explicit DeviceGuard(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) ok = cudaSetDevice(dev) == cudaSuccess;
  }
  ~DeviceGuard() {
    int cur = -1;
    if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
  }
};

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int64_t up8(int64_t v) { return (v + 7) & ~int64_t(7); }

int check_format(moe_ctx* ctx, const char* fn, int dtype, int group_size, int bits) {
  if (!(bits == 2 || bits == 3 || bits == 4 || bits == 5 || bits == 6 || bits == 8))
    return fail(ctx, MOE_ERR_INVALID, "%s: bits=%d is not a valid MLX affine width", fn, bits);
  if (!(group_size == 32 || group_size == 64 || group_size == 128))
    return fail(ctx, MOE_ERR_INVALID, "%s: group_size=%d is not a valid MLX group size", fn, group_size);
  if (bits != 4) return fail(ctx, MOE_ERR_UNSUPPORTED, "%s: only bits=4 is implemented (got %d)", fn, bits);
  if (dtype == MOE_DTYPE_F32) return fail(ctx, MOE_ERR_UNSUPPORTED, "%s: f32 activations are not implemented", fn);
  if (dtype != MOE_DTYPE_BF16 && dtype != MOE_DTYPE_F16)
    return fail(ctx, MOE_ERR_INVALID, "%s: dtype=%d", fn, dtype);
  return MOE_OK;
}

int check_weight(moe_ctx* ctx, const char* fn, const char* name, const moe_qweight& q) {
  if (!q.w || !q.scales) return fail(ctx, MOE_ERR_INVALID, "%s: %s weight missing", fn, name);
  if (!aligned16(q.w) || !aligned16(q.scales) || !aligned16(q.biases))
    return fail(ctx, MOE_ERR_INVALID, "%s: %s weight pointers must be 16-byte aligned", fn, name);
  return MOE_OK;
}

moe::PackedMatrix packed(const moe_qweight& q, int64_t rows, int64_t cols) {
  return {q.w, static_cast<const uint16_t*>(q.scales), static_cast<const uint16_t*>(q.biases), rows, (int)cols};
}

// ---- workspaces, in 256-byte steps
size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

// Output columns per piece of a product over 16-bit weights: at most 32 M weights at a time
// (64 MB, which stay in the 126 MB L2 between the dequantisation and the product).
int64_t qmm_piece(int64_t N, int64_t K) {
  const int64_t n = (int64_t(32) << 20) / K / 256 * 256;
  return std::min(N, std::max<int64_t>(256, n));
}
// The 4-bit matrix product: a copy of x with rows of 16-byte pitch when K is no multiple of 8
// (possible in the direction that sums over the weights' rows); for many tokens one piece of
// 16-bit weights. A piece of weight columns would not be contiguous, so that direction takes
// 16-bit weights only where one piece holds them all.
struct QmmWs {
  bool wide;
  size_t xpad, total;
};
QmmWs qmm_workspace(int64_t M, int64_t N, int64_t K, int transpose) {
  QmmWs w{};
  w.xpad = K % 8 ? up256((size_t)M * up8(K) * sizeof(uint16_t)) : 0;
  const int64_t piece = qmm_piece(N, K);
  w.wide = M >= (transpose ? moe::kWideMinM : moe::kWideMinRowsM) && (transpose || piece == N);
  w.total = w.xpad + (w.wide ? (size_t)piece * K * sizeof(uint16_t) : 0);
  return w;
}

int check_qmm_sizes(moe_ctx* ctx, const char* fn, int64_t M, int64_t K, int64_t N, int transpose, int group_size) {
  constexpr int64_t kMost = INT32_MAX - 1024;
  if (M < 0 || N <= 0 || K <= 0 || M > kMost || N > kMost || K > kMost)
    return fail(ctx, MOE_ERR_INVALID, "%s: bad M/N/K (%lld, %lld, %lld)", fn, (long long)M, (long long)N, (long long)K);
  const int64_t inner = transpose ? K : N;
  if (inner % group_size)
    return fail(ctx, MOE_ERR_INVALID, "%s: %s=%lld must be a multiple of group_size=%d", fn, transpose ? "K" : "N",
                (long long)inner, group_size);
  return MOE_OK;
}

// ---- feed-forward block
int check_ffn(moe_ctx* ctx, const char* fn, const moe_ffn_config* c, int64_t T) {
  if (!c) return fail(ctx, MOE_ERR_INVALID, "%s: null config", fn);
  int rc = check_format(ctx, fn, c->dtype, c->group_size, c->bits);
  if (rc) return rc;
  if (c->hidden <= 0 || c->hidden % c->group_size || c->inter <= 0 || c->inter % c->group_size)
    return fail(ctx, MOE_ERR_INVALID, "%s: hidden=%d and inter=%d must be positive multiples of group_size=%d", fn,
                c->hidden, c->inter, c->group_size);
  if (c->hidden > (1 << 24) || c->inter > (1 << 24))
    return fail(ctx, MOE_ERR_INVALID, "%s: hidden=%d / inter=%d too large", fn, c->hidden, c->inter);
  if (c->activation != MOE_ACT_SILU && c->activation != MOE_ACT_GELU)
    return fail(ctx, MOE_ERR_INVALID, "%s: activation=%d", fn, c->activation);
  if (T < 0 || T > INT32_MAX - 1024) return fail(ctx, MOE_ERR_INVALID, "%s: T=%lld", fn, (long long)T);
  return MOE_OK;
}

int check_ffn_weights(moe_ctx* ctx, const char* fn, const moe_ffn_weights* w) {
  if (!w) return fail(ctx, MOE_ERR_INVALID, "%s: null weights", fn);
  int rc = check_weight(ctx, fn, "gate", w->gate);
  if (!rc) rc = check_weight(ctx, fn, "up", w->up);
  if (!rc) rc = check_weight(ctx, fn, "down", w->down);
  return rc;
}

// The forward pass keeps h [T][I] between its two products; for many tokens both passes keep
// the three matrices in 16 bits.
struct FfnWs {
  bool wide;
  size_t h, each, total;  // bytes of h, of one matrix, of all
};
FfnWs ffn_workspace(const moe_ffn_config* c, int64_t T, bool backward) {
  FfnWs w{};
  w.wide = T >= (backward ? moe::kWideMinRowsM : moe::kWideMinM);
  w.h = backward ? 0 : up256((size_t)T * c->inter * sizeof(uint16_t));
  w.each = w.wide ? up256((size_t)c->hidden * c->inter * sizeof(uint16_t)) : 0;
  w.total = w.h + 3 * w.each;
  return w;
}

// The three matrices in 16 bits, behind h in the workspace.
struct Wide {
  uint16_t *gate = nullptr, *up = nullptr, *down = nullptr;
};
cudaError_t widen(const moe_ffn_config* c, const moe_ffn_weights* w, const FfnWs& ws, void* workspace, Wide& out,
                  cudaStream_t st) {
  if (!ws.wide) return cudaSuccess;
  char* base = static_cast<char*>(workspace) + ws.h;
  out.gate = reinterpret_cast<uint16_t*>(base);
  out.up = reinterpret_cast<uint16_t*>(base + ws.each);
  out.down = reinterpret_cast<uint16_t*>(base + 2 * ws.each);
  moe::DequantArgs da{};
  da.jobs = 3;
  da.group = c->group_size;
  da.type = c->dtype;
  da.job[0] = {packed(w->gate, c->inter, c->hidden), out.gate};
  da.job[1] = {packed(w->up, c->inter, c->hidden), out.up};
  da.job[2] = {packed(w->down, c->hidden, c->inter), out.down};
  return moe::launch_dequant(da, st);
}

// Whether rows of D elements at these strides (of B, H and L) lie apart: by rising stride, each
// step is longer than all that the smaller ones reach.
bool separate_rows(int64_t B, int64_t H, int64_t L, int64_t D, const int64_t* strides) {
  std::pair<int64_t, int64_t> axis[3] = {{strides[0], B}, {strides[1], H}, {strides[2], L}};
  std::sort(axis, axis + 3);
  int64_t reach = D - 1;
  for (const auto& [stride, size] : axis) {
    if (size == 1) continue;
    if (stride <= reach || stride > (INT64_MAX / 4) / size) return false;
    reach += (size - 1) * stride;
  }
  return true;
}

int check_workspace(moe_ctx* ctx, const char* fn, const void* ws, size_t have, size_t need) {
  if (need == 0) return MOE_OK;
  if (!ws || have < need)
    return fail(ctx, MOE_ERR_INVALID, "%s: workspace of %zu bytes, %zu needed", fn, ws ? have : (size_t)0, need);
  if (reinterpret_cast<uintptr_t>(ws) & 31)
    return fail(ctx, MOE_ERR_INVALID, "%s: workspace must be 32-byte aligned", fn);
  return MOE_OK;
}

}  // namespace

extern "C" {

int moe_quantized_matmul_workspace(int dtype, int64_t M, int64_t K, int64_t N, int transpose, int group_size, int bits,
                                   size_t* bytes) {
  if (!bytes) return MOE_ERR_INVALID;
  *bytes = 0;
  int rc = check_format(nullptr, "", dtype, group_size, bits);
  if (!rc) rc = check_qmm_sizes(nullptr, "", M, K, N, transpose, group_size);
  if (rc || M == 0) return rc;
  *bytes = qmm_workspace(M, N, K, transpose).total;
  return MOE_OK;
}

int moe_quantized_matmul_ex(moe_ctx* ctx, int dtype, const void* x, int64_t M, int64_t K, const uint32_t* w,
                            const void* scales, const void* biases, int64_t N, int transpose, int group_size, int bits,
                            void* out, void* workspace, size_t workspace_bytes) {
  if (!ctx) return MOE_ERR_INVALID;
  moe_internal::ctx_set_error(ctx, "");
  const char* fn = "moe_quantized_matmul";
  int rc = check_format(ctx, fn, dtype, group_size, bits);
  if (!rc) rc = check_qmm_sizes(ctx, fn, M, K, N, transpose, group_size);
  if (rc || M == 0) return rc;
  const moe_qweight q{w, scales, biases};
  if (!x || !out) return fail(ctx, MOE_ERR_INVALID, "%s: null pointer", fn);
  rc = check_weight(ctx, fn, "w", q);
  if (rc) return rc;
  if (!aligned16(x) || !aligned16(out)) return fail(ctx, MOE_ERR_INVALID, "%s: x and out must be 16-byte aligned", fn);
  const QmmWs ws = qmm_workspace(M, N, K, transpose);
  rc = check_workspace(ctx, fn, workspace, workspace_bytes, ws.total);
  if (rc) return rc;
  DeviceGuard g(moe_internal::ctx_device(ctx));
  if (!g.ok) return fail(ctx, MOE_ERR_CUDA, "%s: cudaSetDevice failed", fn);
  const cudaStream_t st = static_cast<cudaStream_t>(moe_internal::ctx_stream(ctx));

  if (transpose && moe::qmv_fits(M, N, K, false)) {
    moe::QmvArgs a{};
    a.x = static_cast<const uint16_t*>(x);
    a.m[0] = packed(q, N, K);
    a.M = (int)M;
    a.N = N;
    a.K = (int)K;
    a.group = group_size;
    a.type = dtype;
    a.out = static_cast<uint16_t*>(out);
    DENSE_CUDA(ctx, fn, moe::launch_qmv(a, false, st));
    return MOE_OK;
  }
  moe::DenseGemm gm{};
  gm.a[0] = static_cast<const uint16_t*>(x);
  gm.lda = up8(K);
  if (gm.lda != K) {
    uint16_t* padded = static_cast<uint16_t*>(workspace);
    DENSE_CUDA(ctx, fn, moe::launch_pad_rows(gm.a[0], M, K, padded, gm.lda, st));
    gm.a[0] = padded;
  }
  gm.w[0] = packed(q, transpose ? N : K, transpose ? K : N);
  gm.pairs = 1;
  gm.rows_k = !transpose;
  gm.M = M;
  gm.N = (int)N;
  gm.K = (int)K;
  gm.group = group_size;
  gm.type = dtype;
  gm.epilogue = moe::kEpiPlain;
  gm.e.out = static_cast<uint16_t*>(out);
  gm.e.ldo = N;
  if (!ws.wide) {
    DENSE_CUDA(ctx, fn, moe::launch_dense_gemm(gm, st));
    return MOE_OK;
  }
  uint16_t* w16 = reinterpret_cast<uint16_t*>(static_cast<char*>(workspace) + ws.xpad);
  const int64_t piece = qmm_piece(N, K);
  for (int64_t n0 = 0; n0 < N; n0 += piece) {
    moe::DequantArgs da{};
    da.jobs = 1;
    da.group = group_size;
    da.type = dtype;
    moe::PackedMatrix m = gm.w[0];
    if (transpose) {  // rows n0.. of the weights
      m.rows = gm.N = (int)std::min(piece, N - n0);
      m.w += n0 * (K / 8);
      m.s += n0 * (K / group_size);
      if (m.b) m.b += n0 * (K / group_size);
    }
    da.job[0] = {m, w16};
    DENSE_CUDA(ctx, fn, moe::launch_dequant(da, st));
    gm.wide[0] = w16;
    gm.e.out = static_cast<uint16_t*>(out) + n0;
    DENSE_CUDA(ctx, fn, moe::launch_dense_gemm(gm, st));
  }
  return MOE_OK;
}

int moe_gated_ffn_workspace(const moe_ffn_config* cfg, int64_t T, int backward, size_t* bytes) {
  if (!bytes) return MOE_ERR_INVALID;
  *bytes = 0;
  int rc = check_ffn(nullptr, "", cfg, T);
  if (rc || T == 0) return rc;
  *bytes = ffn_workspace(cfg, T, backward != 0).total;
  return MOE_OK;
}

int moe_gated_ffn_forward(moe_ctx* ctx, const moe_ffn_config* cfg, const moe_ffn_weights* wts, const void* x, int64_t T,
                          const void* residual, void* gate, void* up, void* out, void* workspace,
                          size_t workspace_bytes) {
  if (!ctx) return MOE_ERR_INVALID;
  moe_internal::ctx_set_error(ctx, "");
  const char* fn = "moe_gated_ffn_forward";
  int rc = check_ffn(ctx, fn, cfg, T);
  if (!rc) rc = check_ffn_weights(ctx, fn, wts);
  if (rc || T == 0) return rc;
  if (!x || !out) return fail(ctx, MOE_ERR_INVALID, "%s: null pointer", fn);
  if (!gate != !up) return fail(ctx, MOE_ERR_INVALID, "%s: gate and up are saved together or not at all", fn);
  for (const void* p : {x, residual, (const void*)gate, (const void*)up, (const void*)out})
    if (!aligned16(p)) return fail(ctx, MOE_ERR_INVALID, "%s: tensors must be 16-byte aligned", fn);
  const FfnWs ws = ffn_workspace(cfg, T, false);
  rc = check_workspace(ctx, fn, workspace, workspace_bytes, ws.total);
  if (rc) return rc;
  uint16_t* h = static_cast<uint16_t*>(workspace);
  DeviceGuard g(moe_internal::ctx_device(ctx));
  if (!g.ok) return fail(ctx, MOE_ERR_CUDA, "%s: cudaSetDevice failed", fn);
  const cudaStream_t st = static_cast<cudaStream_t>(moe_internal::ctx_stream(ctx));
  const int H = cfg->hidden, I = cfg->inter;

  Wide wide;
  DENSE_CUDA(ctx, fn, widen(cfg, wts, ws, workspace, wide, st));
  if (moe::qmv_fits(T, I, H, true)) {
    moe::QmvArgs a{};
    a.x = static_cast<const uint16_t*>(x);
    a.m[0] = packed(wts->gate, I, H);
    a.m[1] = packed(wts->up, I, H);
    a.M = (int)T;
    a.N = I;
    a.K = H;
    a.group = cfg->group_size;
    a.type = cfg->dtype;
    a.out = h;
    a.gate = static_cast<uint16_t*>(gate);
    a.up = static_cast<uint16_t*>(up);
    a.act = cfg->activation;
    DENSE_CUDA(ctx, fn, moe::launch_qmv(a, true, st));
  } else {
    moe::DenseGemm gu{};
    gu.a[0] = static_cast<const uint16_t*>(x);
    gu.w[0] = packed(wts->gate, I, H);
    gu.w[1] = packed(wts->up, I, H);
    gu.wide[0] = wide.gate;
    gu.wide[1] = wide.up;
    gu.lda = H;
    gu.pairs = 1;
    gu.M = T;
    gu.N = I;
    gu.K = H;
    gu.group = cfg->group_size;
    gu.type = cfg->dtype;
    gu.epilogue = moe::kEpiGated;
    gu.e.out = h;
    gu.e.ldo = I;
    gu.e.gate = static_cast<uint16_t*>(gate);
    gu.e.up = static_cast<uint16_t*>(up);
    gu.e.act = cfg->activation;
    DENSE_CUDA(ctx, fn, moe::launch_dense_gemm(gu, st));
  }
  if (moe::qmv_fits(T, H, I, false)) {
    moe::QmvArgs d{};
    d.x = h;
    d.m[0] = packed(wts->down, H, I);
    d.M = (int)T;
    d.N = H;
    d.K = I;
    d.group = cfg->group_size;
    d.type = cfg->dtype;
    d.out = static_cast<uint16_t*>(out);
    d.residual = static_cast<const uint16_t*>(residual);
    d.early = 1;
    DENSE_CUDA(ctx, fn, moe::launch_qmv(d, false, st));
  } else {
    moe::DenseGemm dn{};
    dn.a[0] = h;
    dn.w[0] = packed(wts->down, H, I);
    dn.wide[0] = wide.down;
    dn.lda = I;
    dn.pairs = 1;
    dn.M = T;
    dn.N = H;
    dn.K = I;
    dn.group = cfg->group_size;
    dn.type = cfg->dtype;
    dn.early = 1;
    dn.epilogue = moe::kEpiPlain;
    dn.e.out = static_cast<uint16_t*>(out);
    dn.e.ldo = H;
    dn.e.residual = static_cast<const uint16_t*>(residual);
    DENSE_CUDA(ctx, fn, moe::launch_dense_gemm(dn, st));
  }
  return MOE_OK;
}

int moe_gated_ffn_backward(moe_ctx* ctx, const moe_ffn_config* cfg, const moe_ffn_weights* wts, const void* gate,
                           const void* up, const void* dy, int64_t T, void* dgate, void* dup, void* dx, void* workspace,
                           size_t workspace_bytes) {
  if (!ctx) return MOE_ERR_INVALID;
  moe_internal::ctx_set_error(ctx, "");
  const char* fn = "moe_gated_ffn_backward";
  int rc = check_ffn(ctx, fn, cfg, T);
  if (!rc) rc = check_ffn_weights(ctx, fn, wts);
  if (rc || T == 0) return rc;
  for (const void* p : {gate, up, dy, (const void*)dgate, (const void*)dup, (const void*)dx}) {
    if (!p) return fail(ctx, MOE_ERR_INVALID, "%s: null pointer", fn);
    if (!aligned16(p)) return fail(ctx, MOE_ERR_INVALID, "%s: tensors must be 16-byte aligned", fn);
  }
  const FfnWs ws = ffn_workspace(cfg, T, true);
  rc = check_workspace(ctx, fn, workspace, workspace_bytes, ws.total);
  if (rc) return rc;
  DeviceGuard g(moe_internal::ctx_device(ctx));
  if (!g.ok) return fail(ctx, MOE_ERR_CUDA, "%s: cudaSetDevice failed", fn);
  const cudaStream_t st = static_cast<cudaStream_t>(moe_internal::ctx_stream(ctx));
  const int H = cfg->hidden, I = cfg->inter;

  Wide wide;
  DENSE_CUDA(ctx, fn, widen(cfg, wts, ws, workspace, wide, st));
  // both products sum over the weights' rows
  moe::DenseGemm dh{};
  dh.a[0] = static_cast<const uint16_t*>(dy);
  dh.w[0] = packed(wts->down, H, I);
  dh.wide[0] = wide.down;
  dh.lda = H;
  dh.pairs = 1;
  dh.rows_k = 1;
  dh.M = T;
  dh.N = I;
  dh.K = H;
  dh.group = cfg->group_size;
  dh.type = cfg->dtype;
  dh.epilogue = moe::kEpiGatedBackward;
  dh.e.ldo = I;
  dh.e.gate = static_cast<uint16_t*>(const_cast<void*>(gate));
  dh.e.up = static_cast<uint16_t*>(const_cast<void*>(up));
  dh.e.dgate = static_cast<uint16_t*>(dgate);
  dh.e.dup = static_cast<uint16_t*>(dup);
  dh.e.act = cfg->activation;
  DENSE_CUDA(ctx, fn, moe::launch_dense_gemm(dh, st));

  moe::DenseGemm in{};  // dx = dgate . gate + dup . up: one sum over both
  in.a[0] = static_cast<const uint16_t*>(dgate);
  in.a[1] = static_cast<const uint16_t*>(dup);
  in.w[0] = packed(wts->gate, I, H);
  in.w[1] = packed(wts->up, I, H);
  in.wide[0] = wide.gate;
  in.wide[1] = wide.up;
  in.lda = I;
  in.pairs = 2;
  in.rows_k = 1;
  in.M = T;
  in.N = H;
  in.K = I;
  in.group = cfg->group_size;
  in.type = cfg->dtype;
  in.early = 1;
  in.epilogue = moe::kEpiPlain;
  in.e.out = static_cast<uint16_t*>(dx);
  in.e.ldo = H;
  DENSE_CUDA(ctx, fn, moe::launch_dense_gemm(in, st));
  return MOE_OK;
}

int moe_fast_rope(moe_ctx* ctx, const moe_rope_config* cfg, const void* x, const int64_t* x_strides, int64_t B,
                  int64_t H, int64_t L, int64_t D, int64_t offset, const void* offsets, int offsets_bits,
                  const float* freqs, void* out, const int64_t* out_strides) {
  if (!ctx) return MOE_ERR_INVALID;
  moe_internal::ctx_set_error(ctx, "");
  const char* fn = "moe_fast_rope";
  if (!cfg) return fail(ctx, MOE_ERR_INVALID, "%s: null config", fn);
  if (cfg->dtype != MOE_DTYPE_BF16 && cfg->dtype != MOE_DTYPE_F16 && cfg->dtype != MOE_DTYPE_F32)
    return fail(ctx, MOE_ERR_INVALID, "%s: dtype=%d", fn, cfg->dtype);
  if (B < 0 || H < 0 || L < 0 || D <= 0) return fail(ctx, MOE_ERR_INVALID, "%s: bad shape", fn);
  if (cfg->dims <= 0 || cfg->dims % 2 || cfg->dims > D)
    return fail(ctx, MOE_ERR_INVALID, "%s: dims=%d must be even and in 2..%lld", fn, cfg->dims, (long long)D);
  if (B == 0 || H == 0 || L == 0) return MOE_OK;
  if (D > 4096 || H > (int64_t(1) << 26) / D || B > INT32_MAX / L)
    return fail(ctx, MOE_ERR_UNSUPPORTED, "%s: shape [%lld, %lld, %lld, %lld] is too large", fn, (long long)B,
                (long long)H, (long long)L, (long long)D);
  if (!x || !x_strides || !out || !out_strides) return fail(ctx, MOE_ERR_INVALID, "%s: null pointer", fn);
  if (!separate_rows(B, H, L, D, out_strides))
    return fail(ctx, MOE_ERR_INVALID, "%s: rows of out overlap one another", fn);
  if (offset > (int64_t(1) << 53) || offset < -(int64_t(1) << 53))
    return fail(ctx, MOE_ERR_INVALID, "%s: offset=%lld is beyond 2^53", fn, (long long)offset);
  if (offsets && offsets_bits != 32 && offsets_bits != 64)
    return fail(ctx, MOE_ERR_INVALID, "%s: offsets_bits=%d", fn, offsets_bits);
  if (!freqs && !(cfg->base > 0.0 && std::isfinite(cfg->base)))
    return fail(ctx, MOE_ERR_INVALID, "%s: base must be positive and finite", fn);
  if (!std::isfinite(cfg->scale) || !std::isfinite(cfg->mscale))
    return fail(ctx, MOE_ERR_INVALID, "%s: scale and mscale must be finite", fn);
  const uintptr_t size = cfg->dtype == MOE_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(out) % size ||
      (offsets && reinterpret_cast<uintptr_t>(offsets) % (uintptr_t)(offsets_bits / 8)) ||
      (freqs && reinterpret_cast<uintptr_t>(freqs) % 4))
    return fail(ctx, MOE_ERR_INVALID, "%s: misaligned pointer", fn);
  DeviceGuard g(moe_internal::ctx_device(ctx));
  if (!g.ok) return fail(ctx, MOE_ERR_CUDA, "%s: cudaSetDevice failed", fn);
  moe::RopeArgs a{};
  a.x = x;
  a.out = out;
  for (int i = 0; i < 3; ++i) a.xs[i] = x_strides[i], a.os[i] = out_strides[i];
  a.B = B;
  a.H = H;
  a.L = L;
  a.D = (int)D;
  a.dims = cfg->dims;
  a.type = cfg->dtype;
  a.interleaved = cfg->traditional != 0;
  a.base = freqs ? 0.0 : std::log2(cfg->base);
  a.scale = cfg->scale;
  a.mscale = (float)cfg->mscale;
  a.sign = cfg->inverse ? -1.0f : 1.0f;
  a.offset = offset;
  a.offsets = offsets;
  a.offsets64 = offsets_bits == 64;
  a.freqs = freqs;
  DENSE_CUDA(ctx, fn, moe::launch_rope(a, static_cast<cudaStream_t>(moe_internal::ctx_stream(ctx))));
  return MOE_OK;
}

}  // extern "C"
