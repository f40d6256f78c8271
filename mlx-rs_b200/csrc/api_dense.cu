// api_dense.cu — extern "C" entry points of the dense operators (include/moe_b200.h):
// 4-bit matrix products at every MLX group size, the gated feed-forward block with its
// backward pass, and the rotary positions. Their workspace comes from the caller, so calls
// on different streams and captured graphs share nothing.
#include <cuda_runtime.h>

#include <algorithm>
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

struct Carve {
  char* base;
  size_t off = 0;
  template <class T>
  T* take(size_t count) {
    off = (off + 255) & ~size_t(255);
    T* p = reinterpret_cast<T*>(base ? base + off : nullptr);
    off += count * sizeof(T);
    return p;
  }
};

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

// ---- 4-bit matrix product. Weight rows are dequantised in pieces of at most this many
// elements (64 MB of 16-bit values, which stay in the 126 MB L2 for the product).
constexpr int64_t kPieceElems = int64_t(32) << 20;

// Output columns per piece.
int64_t qmm_piece(int64_t N, int64_t K) {
  const int64_t n = std::max<int64_t>(256, kPieceElems / up8(K) / 256 * 256);
  return std::min(N, n);
}

struct QmmWs {
  uint16_t* w;      // 16-bit weights: [piece][K], or [K][piece] when !transpose
  uint16_t* xpad;   // [M][K rounded up to 8] when K is no multiple of 8
  float* partial;
  size_t partial_bytes, bytes;
};
QmmWs carve_qmm(void* base, int64_t M, int64_t N, int64_t K, int transpose) {
  Carve cv{static_cast<char*>(base)};
  QmmWs w{};
  if (transpose && M <= moe::kQmvMaxM) return w;  // straight from the packed weights
  const int64_t piece = qmm_piece(N, K);
  w.w = cv.take<uint16_t>(piece * up8(K));
  if (K % 8) w.xpad = cv.take<uint16_t>(M * up8(K));
  // the last piece may split where the full ones do not
  w.partial_bytes = moe::dense_partial_bytes(M, (int)piece, (int)K, 1, false);
  if (N % piece) w.partial_bytes = std::max(w.partial_bytes, moe::dense_partial_bytes(M, (int)(N % piece), (int)K, 1, false));
  w.partial = w.partial_bytes ? cv.take<float>(w.partial_bytes / sizeof(float)) : nullptr;
  w.bytes = cv.off;
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

struct FfnWs {
  uint16_t *wg, *wu, *wd;  // 16-bit weights
  uint16_t* h;             // [T][I] (forward)
  float* partial;
  size_t partial_bytes, bytes;
};
FfnWs carve_ffn(void* base, const moe_ffn_config* c, int64_t T, bool backward) {
  Carve cv{static_cast<char*>(base)};
  FfnWs w{};
  const size_t n = (size_t)c->hidden * c->inter;
  const int H = c->hidden, I = c->inter;
  if (!backward && T <= moe::kQmvMaxM) {  // straight from the packed weights
    w.h = cv.take<uint16_t>((size_t)T * I);
    w.bytes = cv.off;
    return w;
  }
  w.wg = cv.take<uint16_t>(n);
  w.wu = cv.take<uint16_t>(n);
  w.wd = cv.take<uint16_t>(n);
  if (!backward) {
    w.h = cv.take<uint16_t>((size_t)T * I);
    w.partial_bytes = std::max(moe::dense_partial_bytes(T, I, H, 1, true), moe::dense_partial_bytes(T, H, I, 1, false));
  } else {
    w.partial_bytes =
        std::max(moe::dense_partial_bytes(T, I, H, 1, false), moe::dense_partial_bytes(T, H, I, 2, false));
  }
  w.partial = w.partial_bytes ? cv.take<float>(w.partial_bytes / sizeof(float)) : nullptr;
  w.bytes = cv.off;
  return w;
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
  *bytes = carve_qmm(nullptr, M, N, K, transpose).bytes;
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
  const QmmWs need = carve_qmm(nullptr, M, N, K, transpose);
  rc = check_workspace(ctx, fn, workspace, workspace_bytes, need.bytes);
  if (rc) return rc;
  const QmmWs ws = carve_qmm(workspace, M, N, K, transpose);
  DeviceGuard g(moe_internal::ctx_device(ctx));
  if (!g.ok) return fail(ctx, MOE_ERR_CUDA, "%s: cudaSetDevice failed", fn);
  const cudaStream_t st = static_cast<cudaStream_t>(moe_internal::ctx_stream(ctx));

  if (transpose && M <= moe::kQmvMaxM) {
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
  const int64_t ldx = up8(K);
  const uint16_t* xs = static_cast<const uint16_t*>(x);
  if (ws.xpad) {
    DENSE_CUDA(ctx, fn, moe::launch_pad_rows(xs, M, K, ws.xpad, ldx, st));
    xs = ws.xpad;
  }
  const int64_t piece = qmm_piece(N, K);
  for (int64_t n0 = 0; n0 < N; n0 += piece) {
    const int64_t n = std::min(piece, N - n0);
    moe::DequantArgs da{};
    da.jobs = 1;
    da.group = group_size;
    da.type = dtype;
    const int64_t inner = transpose ? K : N;
    moe::PackedMatrix m = packed(q, transpose ? n : K, inner);
    m.w_pitch = (int)(inner / 8);
    m.s_pitch = (int)(inner / group_size);
    if (transpose) {
      m.w += n0 * (K / 8);
      m.s += n0 * (K / group_size);
      if (m.b) m.b += n0 * (K / group_size);
    } else {
      // a piece of columns: whole words and groups (the piece is a multiple of 256)
      m.w += n0 / 8;
      m.s += n0 / group_size;
      if (m.b) m.b += n0 / group_size;
      m.cols = (int)n;
    }
    da.job[0] = {m, ws.w, transpose ? ldx : piece};
    DENSE_CUDA(ctx, fn, moe::launch_dequant(da, st));
    moe::DenseGemm gm{};
    gm.a[0] = xs;
    gm.b[0] = ws.w;
    gm.lda[0] = ldx;
    gm.ldb[0] = transpose ? ldx : piece;
    gm.b_rows_k = !transpose;
    gm.pairs = 1;
    gm.M = M;
    gm.N = (int)n;
    gm.K = (int)K;
    gm.type = dtype;
    gm.epilogue = moe::kEpiPlain;
    gm.e.out = static_cast<uint16_t*>(out) + n0;
    gm.e.ldo = N;
    gm.partial = ws.partial;
    gm.partial_bytes = ws.partial_bytes;
    DENSE_CUDA(ctx, fn, moe::launch_dense_gemm(gm, st));
  }
  return MOE_OK;
}

int moe_gated_ffn_workspace(const moe_ffn_config* cfg, int64_t T, int backward, size_t* bytes) {
  if (!bytes) return MOE_ERR_INVALID;
  *bytes = 0;
  int rc = check_ffn(nullptr, "", cfg, T);
  if (rc || T == 0) return rc;
  *bytes = carve_ffn(nullptr, cfg, T, backward != 0).bytes;
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
  const FfnWs need = carve_ffn(nullptr, cfg, T, false);
  rc = check_workspace(ctx, fn, workspace, workspace_bytes, need.bytes);
  if (rc) return rc;
  const FfnWs ws = carve_ffn(workspace, cfg, T, false);
  DeviceGuard g(moe_internal::ctx_device(ctx));
  if (!g.ok) return fail(ctx, MOE_ERR_CUDA, "%s: cudaSetDevice failed", fn);
  const cudaStream_t st = static_cast<cudaStream_t>(moe_internal::ctx_stream(ctx));
  const int H = cfg->hidden, I = cfg->inter;

  if (T <= moe::kQmvMaxM) {
    moe::QmvArgs a{};
    a.x = static_cast<const uint16_t*>(x);
    a.m[0] = packed(wts->gate, I, H);
    a.m[1] = packed(wts->up, I, H);
    a.M = (int)T;
    a.N = I;
    a.K = H;
    a.group = cfg->group_size;
    a.type = cfg->dtype;
    a.out = ws.h;
    a.gate = static_cast<uint16_t*>(gate);
    a.up = static_cast<uint16_t*>(up);
    a.act = cfg->activation;
    DENSE_CUDA(ctx, fn, moe::launch_qmv(a, true, st));
    moe::QmvArgs d{};
    d.x = ws.h;
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
    return MOE_OK;
  }
  moe::DequantArgs da{};
  da.jobs = 3;
  da.group = cfg->group_size;
  da.type = cfg->dtype;
  da.job[0] = {packed(wts->gate, I, H), ws.wg, H};
  da.job[1] = {packed(wts->up, I, H), ws.wu, H};
  da.job[2] = {packed(wts->down, H, I), ws.wd, I};
  for (auto& j : da.job) j.m.w_pitch = j.m.cols / 8, j.m.s_pitch = j.m.cols / cfg->group_size;
  DENSE_CUDA(ctx, fn, moe::launch_dequant(da, st));

  moe::DenseGemm gu{};
  gu.a[0] = static_cast<const uint16_t*>(x);
  gu.b[0] = ws.wg;
  gu.b[1] = ws.wu;
  gu.lda[0] = gu.ldb[0] = gu.ldb[1] = H;
  gu.pairs = 1;
  gu.M = T;
  gu.N = I;
  gu.K = H;
  gu.type = cfg->dtype;
  gu.epilogue = moe::kEpiGated;
  gu.e.out = ws.h;
  gu.e.ldo = I;
  gu.e.gate = static_cast<uint16_t*>(gate);
  gu.e.up = static_cast<uint16_t*>(up);
  gu.e.act = cfg->activation;
  gu.partial = ws.partial;
  gu.partial_bytes = ws.partial_bytes;
  DENSE_CUDA(ctx, fn, moe::launch_dense_gemm(gu, st));

  moe::DenseGemm dn{};
  dn.a[0] = ws.h;
  dn.b[0] = ws.wd;
  dn.lda[0] = dn.ldb[0] = I;
  dn.pairs = 1;
  dn.M = T;
  dn.N = H;
  dn.K = I;
  dn.type = cfg->dtype;
  dn.epilogue = moe::kEpiPlain;
  dn.e.out = static_cast<uint16_t*>(out);
  dn.e.ldo = H;
  dn.e.residual = static_cast<const uint16_t*>(residual);
  dn.partial = ws.partial;
  dn.partial_bytes = ws.partial_bytes;
  DENSE_CUDA(ctx, fn, moe::launch_dense_gemm(dn, st));
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
  const FfnWs need = carve_ffn(nullptr, cfg, T, true);
  rc = check_workspace(ctx, fn, workspace, workspace_bytes, need.bytes);
  if (rc) return rc;
  const FfnWs ws = carve_ffn(workspace, cfg, T, true);
  DeviceGuard g(moe_internal::ctx_device(ctx));
  if (!g.ok) return fail(ctx, MOE_ERR_CUDA, "%s: cudaSetDevice failed", fn);
  const cudaStream_t st = static_cast<cudaStream_t>(moe_internal::ctx_stream(ctx));
  const int H = cfg->hidden, I = cfg->inter;

  // the products below sum over the weights' rows
  moe::DequantArgs da{};
  da.jobs = 3;
  da.group = cfg->group_size;
  da.type = cfg->dtype;
  da.job[0] = {packed(wts->gate, I, H), ws.wg, H};
  da.job[1] = {packed(wts->up, I, H), ws.wu, H};
  da.job[2] = {packed(wts->down, H, I), ws.wd, I};
  for (auto& j : da.job) j.m.w_pitch = j.m.cols / 8, j.m.s_pitch = j.m.cols / cfg->group_size;
  DENSE_CUDA(ctx, fn, moe::launch_dequant(da, st));

  moe::DenseGemm dh{};
  dh.a[0] = static_cast<const uint16_t*>(dy);
  dh.b[0] = ws.wd;
  dh.lda[0] = H;
  dh.ldb[0] = I;
  dh.b_rows_k = 1;
  dh.pairs = 1;
  dh.M = T;
  dh.N = I;
  dh.K = H;
  dh.type = cfg->dtype;
  dh.epilogue = moe::kEpiGatedBackward;
  dh.e.ldo = I;
  dh.e.gate = static_cast<uint16_t*>(const_cast<void*>(gate));
  dh.e.up = static_cast<uint16_t*>(const_cast<void*>(up));
  dh.e.dgate = static_cast<uint16_t*>(dgate);
  dh.e.dup = static_cast<uint16_t*>(dup);
  dh.e.act = cfg->activation;
  dh.partial = ws.partial;
  dh.partial_bytes = ws.partial_bytes;
  DENSE_CUDA(ctx, fn, moe::launch_dense_gemm(dh, st));

  moe::DenseGemm dxg{};
  dxg.a[0] = static_cast<const uint16_t*>(dgate);
  dxg.a[1] = static_cast<const uint16_t*>(dup);
  dxg.b[0] = ws.wg;
  dxg.b[1] = ws.wu;
  dxg.lda[0] = dxg.lda[1] = I;
  dxg.ldb[0] = dxg.ldb[1] = H;
  dxg.b_rows_k = 1;
  dxg.pairs = 2;
  dxg.M = T;
  dxg.N = H;
  dxg.K = I;
  dxg.type = cfg->dtype;
  dxg.epilogue = moe::kEpiPlain;
  dxg.e.out = static_cast<uint16_t*>(dx);
  dxg.e.ldo = H;
  dxg.partial = ws.partial;
  dxg.partial_bytes = ws.partial_bytes;
  DENSE_CUDA(ctx, fn, moe::launch_dense_gemm(dxg, st));
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
