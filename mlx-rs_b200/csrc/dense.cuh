// dense.cuh — argument blocks, launchers and device helpers of the dense operators: 4-bit
// matrix products at every MLX group size, the gated feed-forward block with its backward
// pass, and the rotary positions. Activations are bf16 or f16 (the rotary positions f32
// too); scales and biases have the activations' type.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"
#include "kernels.cuh"

namespace moe {

enum DenseType { kBf16 = 0, kF16 = 1, kF32 = 2 };

// One packed matrix [rows][cols]: cols / 8 words and cols / group scales (biases) per row.
struct PackedMatrix {
  const uint32_t* w;
  const uint16_t* s;
  const uint16_t* b;  // may be null
  int64_t rows;
  int cols;
};

// ---- 4-bit weights to 16-bit rows [rows][cols], 32-byte aligned (dense_dequant.cu)
struct DequantJob {
  PackedMatrix m;
  uint16_t* out;
};
struct DequantArgs {
  DequantJob job[3];
  int jobs;
  int group;
  int type;
  uint32_t rows_cta;  // set by launch_dequant
};
cudaError_t launch_dequant(const DequantArgs& a, cudaStream_t st);
// Tokens from which the products take weights dequantised once by launch_dequant; below, the
// product's own warps dequantise each tile again for every 256 tokens. Per call in us, packed |
// dequantised once, at 1024, 1536, 2048, 2560 and 4096 tokens:
//   block forward, 2048 x 5632, group 64     71 | 82    91 | 95   110 | 114  148 | 142  217 | 208
//   2048 -> 32768, group 128                103 | 130  157 | 179  205 | 214  256 | 260  402 | 385
//   2048 -> 2048, group 32                   17 | 18    18 | 20    21 | 23    30 | 25    36 | 32
// so from the ninth tile of 256 tokens on; and with the weights' rows summed (the gradients):
//   block 2048 x 5632 and gradients         168 | 184  219 | 216  266 | 260  365 | 353  520 | 464
//   block 2048 x 768 and gradients           54 | 62    61 | 66    74 | 70    86 | 79   116 | 98
//   5632 -> 2048, group 32                   28 | 34    40 | 41    41 | 43    79 | 73    80 | 74
// where the two are level from the fifth tile to the eighth and the second is ahead above.
constexpr int64_t kWideMinM = 2049, kWideMinRowsM = 1025;

// out[r][0..cols) = x[r][0..cols), rows ld elements apart, the rest of each row zero
// (dense_pad.cu).
cudaError_t launch_pad_rows(const uint16_t* x, int64_t rows, int64_t cols, uint16_t* out, int64_t ld, cudaStream_t st);

// ---- 4-bit matrix product on tcgen05 with fused epilogues (dense_gemm.cu)
enum DenseEpilogue { kEpiPlain = 0, kEpiGated = 1, kEpiGatedBackward = 2 };
struct DenseEpi {
  int64_t ldo;               // row pitch of every tensor below
  uint16_t* out;             // plain: [M][N]; gated: h = act(g) * u [M][N]
  const uint16_t* residual;  // plain: [M][N] added before the rounding, or null
  uint16_t* gate;            // gated: g and u [M][N] stored when non-null; backward: read
  uint16_t* up;
  uint16_t* dgate;           // backward: [M][N]
  uint16_t* dup;
  int act;                   // 0 SiLU, 1 GELU (tanh form)
};
struct DenseGemm {
  // D[M, N] = sum over the operand pairs p of A_p[M, K] . W_p[N, K]^T (one or two pairs), or
  // . W_p[K, N] with rows_k; in the gated form one A and two W: g = A . W_0^T, u = A . W_1^T.
  const uint16_t* a[2];
  int64_t lda;   // elements, a multiple of 8
  PackedMatrix w[2];
  const uint16_t* wide[2];  // the same weights in 16 bits (M > 128), or null
  int pairs;
  int rows_k;
  int64_t M;
  int N, K;
  int group, type;  // type: kBf16 / kF16
  int early;        // the weights may be read before the launch before has completed
  int epilogue;     // DenseEpilogue
  DenseEpi e;
};
cudaError_t launch_dense_gemm(const DenseGemm& g, cudaStream_t st);
// Device status word of these kernels on the current device (bounded waits that expired: codes
// below 2^16); what it reports is cleared. Synchronises the stream.
cudaError_t dense_gemm_status(int32_t* status, cudaStream_t st);
// A wait of `limit_ns` that nothing ends: code kExpiredWait.
constexpr int32_t kExpiredWait = 256;
cudaError_t launch_expire_wait(uint64_t limit_ns, cudaStream_t st);

// ---- 4-bit products for few tokens (qmv.cu): out = x m[0]^T, or gated out = act(g) * u
struct QmvArgs {
  const uint16_t* x;  // [M][K]
  PackedMatrix m[2];
  int M, K, group, type;
  int64_t N;
  uint16_t* out;             // [M][N]
  const uint16_t* residual;  // [M][N] added before the rounding, or null (not gated)
  uint16_t* gate;            // gated: g and u [M][N] stored when non-null
  uint16_t* up;
  int act;
  int early;                 // the weights may be read before the launch before has completed
  int tiles;                 // set by launch_qmv
};
// Whether these kernels, and not dense_gemm.cu's, serve a product.
bool qmv_fits(int64_t M, int64_t N, int64_t K, bool gated);
cudaError_t launch_qmv(const QmvArgs& a, bool gated, cudaStream_t st);

// ---- rotary positions (rope.cu)
struct RopeArgs {
  const void* x;
  void* out;
  int64_t xs[3], os[3];  // element strides of batch, head, position
  int64_t B, H, L;
  int D, dims;
  int type;
  int interleaved;
  double base, scale;
  float mscale, sign;    // sign -1: the transposed rotation
  int64_t offset;
  const void* offsets;   // [B] int32 or int64 (offsets64), or null
  int offsets64;
  const float* freqs;    // [dims / 2] or null
};
cudaError_t launch_rope(const RopeArgs& a, cudaStream_t st);

// Allows `kern` its dynamic shared memory, once per device (`done`: a static of the caller).
template <class K>
cudaError_t allow_smem(K kern, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
  err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == cudaSuccess && dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return err;
}

// ---- device helpers: mbarriers. Every wait is bounded (2 s): a kernel whose wait expires
// records a code in its status word and runs to its end without waiting further.
constexpr uint64_t kWaitLimitNs = 2000ull * 1000 * 1000;
MOE_DEV uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
MOE_DEV void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count) : "memory");
}
MOE_DEV void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
MOE_DEV bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(1000u)
      : "memory");
  return ok != 0;
}
// Non-blocking (a try_wait may hold the thread until the phase completes).
MOE_DEV bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
MOE_DEV uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;\n" : "=l"(t));
  return t;
}
// Bounded wait; false when it gave up. `gone` is the CTA's abort flag: once one role has
// given up, the others stop waiting.
MOE_DEV bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* gone, uint64_t limit_ns = kWaitLimitNs) {
  if (mbar_try(bar, parity)) return true;
  const uint64_t t0 = now_ns();
  while (!mbar_try(bar, parity))
    if (*gone || now_ns() - t0 > limit_ns) return false;
  return true;
}
MOE_DEV void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}

template <int TYPE>
struct Elem;  // conversions of the 16-bit element types
template <>
struct Elem<kBf16> {
  static MOE_DEV float to_f(uint16_t v) { return bf2f(v); }
  static MOE_DEV uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  static MOE_DEV float lo(uint32_t v) { return bf_lo(v); }
  static MOE_DEV float hi(uint32_t v) { return bf_hi(v); }
};
template <>
struct Elem<kF16> {
  static MOE_DEV float to_f(uint16_t v) { return __half2float(__ushort_as_half(v)); }
  static MOE_DEV uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  static MOE_DEV float lo(uint32_t v) { return to_f((uint16_t)(v & 0xffffu)); }
  static MOE_DEV float hi(uint32_t v) { return to_f((uint16_t)(v >> 16)); }
};

// Two 4-bit fields of a word as 16 + q, exact in either type: the field becomes the top
// mantissa bits under the exponent of 16 (one shift and one LOP3).
template <int TYPE>
struct Nib;
template <>
struct Nib<kBf16> {
  static constexpr uint32_t kMask = 0x00780078u, kBase = 0x41804180u, kOne = 0x3f803f80u;
  static constexpr int kBit = 3;  // lowest mantissa bit of the field
};
template <>
struct Nib<kF16> {
  static constexpr uint32_t kMask = 0x03c003c0u, kBase = 0x4c004c00u, kOne = 0x3c003c00u;
  static constexpr int kBit = 6;
};
// fields j and j + 4 of w
template <int TYPE, int J>
MOE_DEV uint32_t fields(uint32_t w) {
  constexpr int sh = Nib<TYPE>::kBit - 4 * J;
  const uint32_t v = sh >= 0 ? w << (sh >= 0 ? sh : 0) : w >> (sh >= 0 ? 0 : -sh);
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;\n" : "=r"(r) : "r"(v), "n"(Nib<TYPE>::kMask), "n"(Nib<TYPE>::kBase));
  return r;
}
// RN(s * q + b) of a pair of fields: the subtraction of 16 is exact, the fused multiply-add
// rounds once. s2 / b2: the scale / bias in both halves.
template <int TYPE>
MOE_DEV uint32_t scale2(uint32_t f, uint32_t s2, uint32_t b2) {
  uint32_t q, r;
  if constexpr (TYPE == kBf16) {
    asm("sub.rn.bf16x2 %0, %1, %2;\n" : "=r"(q) : "r"(f), "r"(Nib<TYPE>::kBase));
    asm("fma.rn.bf16x2 %0, %1, %2, %3;\n" : "=r"(r) : "r"(q), "r"(s2), "r"(b2));
  } else {
    asm("sub.rn.f16x2 %0, %1, %2;\n" : "=r"(q) : "r"(f), "r"(Nib<TYPE>::kBase));
    asm("fma.rn.f16x2 %0, %1, %2, %3;\n" : "=r"(r) : "r"(q), "r"(s2), "r"(b2));
  }
  return r;
}
// A word's eight weights in element order.
template <int TYPE>
MOE_DEV uint4 dequant8(uint32_t w, uint32_t s2, uint32_t b2) {
  const uint32_t f0 = fields<TYPE, 0>(w), f1 = fields<TYPE, 1>(w), f2 = fields<TYPE, 2>(w), f3 = fields<TYPE, 3>(w);
  uint4 o;
  o.x = scale2<TYPE>(__byte_perm(f0, f1, 0x5410), s2, b2);
  o.y = scale2<TYPE>(__byte_perm(f2, f3, 0x5410), s2, b2);
  o.z = scale2<TYPE>(__byte_perm(f0, f1, 0x7632), s2, b2);
  o.w = scale2<TYPE>(__byte_perm(f2, f3, 0x7632), s2, b2);
  return o;
}

// 1 / (1 + exp(-x)) from the hardware base-2 exponential and reciprocal (relative error a
// few fp32 ulps, far below the 16-bit rounding that follows).
MOE_DEV float sigmoid_hw(float x) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(e) : "f"(x * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(1.0f + e));
  return r;
}
// The activation and its derivative. Both are x * sigmoid(z): SiLU with z = x, GELU's tanh
// form with z = 2 sqrt(2/pi) (x + 0.044715 x^3), since (1 + tanh(y)) / 2 = sigmoid(2 y);
// the derivative is sig + x sig (1 - sig) z'. Where z' would overflow (|x| > 1.8e19)
// x sig (1 - sig) is zero: z' is held finite, so that their product is too.
MOE_DEV float act_val(float x, int act) {
  const float z = act ? 1.5957691216057308f * x * __fmaf_rn(0.044715f * x, x, 1.0f) : x;
  return x * sigmoid_hw(z);
}
MOE_DEV void act_grad(float x, int act, float& val, float& grad) {
  const float z = act ? 1.5957691216057308f * x * __fmaf_rn(0.044715f * x, x, 1.0f) : x;
  const float zp = act ? fminf(1.5957691216057308f * __fmaf_rn(0.134145f * x, x, 1.0f), 1e30f) : 1.0f;
  const float s = sigmoid_hw(z);
  val = x * s;
  grad = __fmaf_rn(val * (1.0f - s), zp, s);
}

}  // namespace moe
