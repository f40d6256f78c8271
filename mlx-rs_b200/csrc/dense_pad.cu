// dense_pad.cu — token rows whose length is no multiple of 8 elements, copied to rows that are:
// TMA needs row pitches of 16 bytes. Bound by the bytes of x, read and written once.
#include "dense.cuh"

namespace moe {

namespace {

// x is not __restrict__: the launch before may write it while this kernel already runs, so it may
// not be read by read-only loads.
__global__ void __launch_bounds__(256) pad_rows_kernel(const uint16_t* x, int64_t rows, int64_t cols, uint16_t* out,
                                                       int64_t ld) {
  pdl_wait();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * ld) return;
  const int64_t r = i / ld, c = i - r * ld;
  out[i] = c < cols ? x[r * cols + c] : (uint16_t)0;
}

}  // namespace

cudaError_t launch_pad_rows(const uint16_t* x, int64_t rows, int64_t cols, uint16_t* out, int64_t ld, cudaStream_t st) {
  return launch_k(pad_rows_kernel, dim3((unsigned)((rows * ld + 255) / 256)), dim3(256), 0, st, x, rows, cols, out, ld);
}

}  // namespace moe
