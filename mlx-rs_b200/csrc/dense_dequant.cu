// dense_dequant.cu — 4-bit weights to 16-bit rows for the dense tensor-core products.
//
// w[n][k] = RN16(scale[n][k / group] * q[n][k] + bias[n][k / group]): one fused
// multiply-add in fp32 and one rounding, to the activations' type, because a tcgen05
// product takes both operands in one 16-bit type. Bound by the bytes: 0.5 + 4 / group
// read and 2 written per weight.
#include "dense.cuh"

namespace moe {

namespace {

template <int TYPE>
MOE_DEV uint4 dequant_word(uint32_t w, float s, float b) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __fmaf_rn(s, (float)((w >> (4 * e)) & 15u), b);
  return make_uint4(Elem<TYPE>::pack(v[0], v[1]), Elem<TYPE>::pack(v[2], v[3]), Elem<TYPE>::pack(v[4], v[5]),
                    Elem<TYPE>::pack(v[6], v[7]));
}

constexpr int kWordsPerThread = 4;

// Row-major: thread = words wi, wi + 256, ... of the flattened matrix, so that a warp reads
// 128 and writes 512 contiguous bytes per step.
template <int TYPE>
__global__ void __launch_bounds__(256) dequant_rows_kernel(const __grid_constant__ DequantArgs a) {
  pdl_wait();
  const DequantJob& j = a.job[blockIdx.y];
  const int wpr = j.m.cols >> 3, wpg = a.group >> 3;
  const int64_t total = j.m.rows * wpr;
  const int64_t base = (int64_t)blockIdx.x * (256 * kWordsPerThread) + threadIdx.x;
#pragma unroll
  for (int i = 0; i < kWordsPerThread; ++i) {
    const int64_t wi = base + i * 256;
    if (wi >= total) break;
    const int64_t row = wi / wpr;
    const int c = (int)(wi - row * wpr);
    const int64_t g = row * j.m.s_pitch + c / wpg;
    const float s = Elem<TYPE>::to_f(j.m.s[g]);
    const float b = j.m.b ? Elem<TYPE>::to_f(j.m.b[g]) : 0.0f;
    *reinterpret_cast<uint4*>(j.out + row * j.ld + c * 8) = dequant_word<TYPE>(__ldg(j.m.w + row * j.m.w_pitch + c), s, b);
  }
}

// Transposed: a CTA turns 64 rows x 64 columns. Lane = a pair of rows, warp = a word of 8
// columns: the pair's elements leave as one 32-bit shared store per column (conflict-free),
// then each column's 64 rows leave as 128 contiguous bytes.
template <int TYPE>
__global__ void __launch_bounds__(256) dequant_cols_kernel(const __grid_constant__ DequantArgs a) {
  __shared__ __align__(16) uint32_t tile[64][36];  // [column][pair of rows], 144-byte rows
  pdl_wait();
  const DequantJob& j = a.job[blockIdx.z];
  const int wpr = j.m.cols >> 3, wpg = a.group >> 3;
  const int64_t n0 = (int64_t)blockIdx.x * 64;
  const int c0 = blockIdx.y * 8;
  if (n0 >= j.m.rows || c0 >= wpr) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = c0 + warp;
  if (c < wpr) {
    uint32_t v[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t row = n0 + 2 * lane + h;
      uint4 d = make_uint4(0, 0, 0, 0);
      if (row < j.m.rows) {
        const int64_t g = row * j.m.s_pitch + c / wpg;
        const float s = Elem<TYPE>::to_f(j.m.s[g]);
        const float b = j.m.b ? Elem<TYPE>::to_f(j.m.b[g]) : 0.0f;
        d = dequant_word<TYPE>(__ldg(j.m.w + row * j.m.w_pitch + c), s, b);
      }
      v[h][0] = d.x, v[h][1] = d.y, v[h][2] = d.z, v[h][3] = d.w;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      tile[warp * 8 + 2 * e][lane] = __byte_perm(v[0][e], v[1][e], 0x5410);
      tile[warp * 8 + 2 * e + 1][lane] = __byte_perm(v[0][e], v[1][e], 0x7632);
    }
  }
  __syncthreads();
  // 64 columns x 8 pieces of 16 bytes; ld is a multiple of 8 and covers the rows rounded
  // up to 8, so a piece that starts inside the rows lies inside the output row
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int p = threadIdx.x + 256 * i;
    const int col = p >> 3, piece = p & 7;
    if (c0 * 8 + col < j.m.cols && n0 + piece * 8 < j.m.rows)
      *reinterpret_cast<uint4*>(j.out + (int64_t)(c0 * 8 + col) * j.ld + n0 + piece * 8) =
          *reinterpret_cast<const uint4*>(&tile[col][piece * 4]);
  }
}

__global__ void __launch_bounds__(256) pad_rows_kernel(const uint16_t* __restrict__ x, int64_t rows, int64_t cols,
                                                       uint16_t* __restrict__ out, int64_t ld) {
  pdl_wait();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * ld) return;
  const int64_t r = i / ld, c = i - r * ld;
  out[i] = c < cols ? x[r * cols + c] : (uint16_t)0;
}

}  // namespace

cudaError_t launch_dequant(const DequantArgs& a, cudaStream_t st) {
  int64_t rows = 0, words = 0;
  int cols = 0;
  for (int i = 0; i < a.jobs; ++i) {
    rows = rows > a.job[i].m.rows ? rows : a.job[i].m.rows;
    cols = cols > a.job[i].m.cols ? cols : a.job[i].m.cols;
    const int64_t n = a.job[i].m.rows * (a.job[i].m.cols / 8);
    words = words > n ? words : n;
  }
  if (!a.transposed) {
    const int64_t per = 256 * kWordsPerThread;
    const dim3 grid((unsigned)((words + per - 1) / per), a.jobs);
    return a.type == kF16 ? launch_k(dequant_rows_kernel<kF16>, grid, dim3(256), 0, st, a)
                          : launch_k(dequant_rows_kernel<kBf16>, grid, dim3(256), 0, st, a);
  }
  const dim3 grid((unsigned)((rows + 63) / 64), (unsigned)((cols + 63) / 64), a.jobs);
  return a.type == kF16 ? launch_k(dequant_cols_kernel<kF16>, grid, dim3(256), 0, st, a)
                        : launch_k(dequant_cols_kernel<kBf16>, grid, dim3(256), 0, st, a);
}

cudaError_t launch_pad_rows(const uint16_t* x, int64_t rows, int64_t cols, uint16_t* out, int64_t ld, cudaStream_t st) {
  return launch_k(pad_rows_kernel, dim3((unsigned)((rows * ld + 255) / 256)), dim3(256), 0, st, x, rows, cols, out, ld);
}

}  // namespace moe
