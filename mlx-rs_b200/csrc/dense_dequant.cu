// dense_dequant.cu — 4-bit weights to 16-bit rows for the dense tensor-core products.
//
// w[n][k] = RN16(scale[n][k / group] * q[n][k] + bias[n][k / group]): one fused
// multiply-add in fp32 and one rounding, to the activations' type, because a tcgen05
// product takes both operands in one 16-bit type. Bound by the bytes: 0.5 + 4 / group
// read and 2 written per weight.
#include "dense.cuh"

namespace moe {

namespace {

constexpr int kSteps = 4;  // pairs of words in flight per thread

// Thread = two words (16 weights of one group) at a time, kSteps of them 256 pairs apart, so
// that a warp reads 256 and writes 1024 contiguous bytes per step. The row and column of a
// thread's first pair take one division; the next ones follow by addition.
template <int TYPE>
__global__ void __launch_bounds__(256) dequant_kernel(const __grid_constant__ DequantArgs a) {
  const DequantJob& j = a.job[blockIdx.y];
  const uint32_t ppr = (uint32_t)j.m.cols >> 4, ppg = (uint32_t)a.group >> 4;  // pairs per row, per group
  const uint32_t rows_cta = a.rows_cta;
  const uint32_t wpr = (uint32_t)j.m.cols >> 3, gpr = (uint32_t)(j.m.cols / a.group);
  const int64_t row0 = (int64_t)blockIdx.x * rows_cta;
  if (row0 >= j.m.rows) return;
  const uint32_t rows = (uint32_t)(j.m.rows - row0 < rows_cta ? j.m.rows - row0 : rows_cta);
  const uint32_t* w = j.m.w + row0 * wpr;
  const uint16_t* s = j.m.s + row0 * gpr;
  const uint16_t* b = j.m.b ? j.m.b + row0 * gpr : nullptr;
  uint16_t* out = j.out + row0 * j.m.cols;
  uint32_t r = threadIdx.x / ppr, c = threadIdx.x - r * ppr;
  const uint32_t dr = 256 / ppr, dc = 256 - dr * ppr;
  pdl_wait();
  pdl_trigger();
  while (r < rows) {
    uint2 q[kSteps];
    uint32_t sc[kSteps], bi[kSteps], rr[kSteps], cc[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      rr[i] = r, cc[i] = c;
      if (r < rows) {
        q[i] = __ldg(reinterpret_cast<const uint2*>(w + (size_t)r * wpr) + c);
        const size_t g = (size_t)r * gpr + c / ppg;
        sc[i] = __ldg(s + g);
        bi[i] = b ? __ldg(b + g) : 0u;
      }
      r += dr, c += dc;
      if (c >= ppr) c -= ppr, ++r;
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (rr[i] >= rows) break;
      const uint32_t s2 = __byte_perm(sc[i], 0, 0x1010), b2 = __byte_perm(bi[i], 0, 0x1010);
      const uint4 lo = dequant8<TYPE>(q[i].x, s2, b2), hi = dequant8<TYPE>(q[i].y, s2, b2);
      uint16_t* o = out + (size_t)rr[i] * j.m.cols + cc[i] * 16;
      asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"l"(o), "r"(lo.x), "r"(lo.y), "r"(lo.z),
                   "r"(lo.w), "r"(hi.x), "r"(hi.y), "r"(hi.z), "r"(hi.w)
                   : "memory");
    }
  }
}

}  // namespace

cudaError_t launch_dequant(const DequantArgs& args, cudaStream_t st) {
  DequantArgs a = args;
  int64_t rows = 0;
  int cols = 0;
  for (int i = 0; i < a.jobs; ++i) {
    rows = rows > a.job[i].m.rows ? rows : a.job[i].m.rows;
    cols = cols > a.job[i].m.cols ? cols : a.job[i].m.cols;
  }
  // rows per CTA: about two rounds of a thread's steps in the widest matrix
  a.rows_cta = 256 * 2 * kSteps / (cols / 16);
  if (a.rows_cta < 1) a.rows_cta = 1;
  const dim3 grid((unsigned)((rows + a.rows_cta - 1) / a.rows_cta), a.jobs);
  return a.type == kF16 ? launch_k(dequant_kernel<kF16>, grid, dim3(256), 0, st, a)
                        : launch_k(dequant_kernel<kBf16>, grid, dim3(256), 0, st, a);
}

}  // namespace moe
