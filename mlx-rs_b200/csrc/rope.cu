// rope.cu — rotary positions: fast_rope of MLX (mlx_fast_rope) on strided [B, H, L, D] tensors.
//
// Pair i of a head at position p is turned by the angle p * scale / wavelength_i, with
// wavelength_i = base^(2 i / dims) or freqs[i]: (a, b) -> mscale (a cos - b sin, a sin + b cos).
// Pairs are (i, i + dims / 2), or (2 i, 2 i + 1) when interleaved; channels from dims on pass
// through. The transposed rotation (the gradient) has the angle's sign turned.
//
// The angle is formed in turns in 64 bits and reduced to [-1/2, 1/2] before it becomes a
// float: at position 10^6 a 32-bit angle is already off by a few hundredths of a radian.
// Bound by the bytes (one read and one write of the tensor). A CTA takes `tokens` positions
// with all of their heads: it fills a table of cosines and sines in shared memory once, one
// pair per thread, so that the 64-bit work is spread over the threads and shared by the heads,
// then moves the heads through two vectors per thread.
#include "dense.cuh"

namespace moe {

namespace {

constexpr int kRopeThreads = 256;

template <int BYTES>
struct Vec;
template <>
struct Vec<16> { using T = uint4; };
template <>
struct Vec<8> { using T = uint2; };
template <>
struct Vec<4> { using T = uint32_t; };
template <>
struct Vec<2> { using T = uint16_t; };

template <int TYPE>
MOE_DEV float get(const void* p, int i) {
  if constexpr (TYPE == kF32) return static_cast<const float*>(p)[i];
  else return Elem<TYPE>::to_f(static_cast<const uint16_t*>(p)[i]);
}
template <int TYPE>
MOE_DEV void put(void* p, int i, float v) {
  if constexpr (TYPE == kF32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = (uint16_t)(Elem<TYPE>::pack(v, 0.0f) & 0xffffu);
}

// VE: elements per vector access (16 bytes where every address allows it)
template <int TYPE, int VE, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeArgs a, int tokens) {
  constexpr int kSize = TYPE == kF32 ? 4 : 2;
  using V = typename Vec<VE * kSize>::T;
  extern __shared__ float2 table[];  // [tokens][dims / 2]: mscale cos, mscale sin
  pdl_wait();
  const int half = a.dims >> 1;
  const int64_t t0 = (int64_t)blockIdx.x * tokens, all = a.B * a.L;
  const int here = (int)(all - t0 < tokens ? all - t0 : tokens);
  for (int i = threadIdx.x; i < here * half; i += kRopeThreads) {
    const int t = i / half, k = i - t * half;
    const int64_t b = (t0 + t) / a.L, l = (t0 + t) - b * a.L;
    int64_t at = a.offset + l;
    if (a.offsets)
      at = l + (a.offsets64 ? static_cast<const int64_t*>(a.offsets)[b] : (int64_t) static_cast<const int32_t*>(a.offsets)[b]);
    // turns = position * scale / (2 pi wavelength)
    constexpr double kPerTurn = 0.15915494309189533577;  // 1 / (2 pi)
    const double rate = a.freqs ? kPerTurn / (double)a.freqs[k]
                                : kPerTurn * exp2(-2.0 * k / a.dims * a.base);  // base holds log2(base)
    const double turns = (double)at * a.scale * rate;
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    table[i] = make_float2(a.mscale * c, a.mscale * a.sign * s);
  }
  __syncthreads();
  const int nrot = half / VE, nitems = (int)((a.D - a.dims + 2 * VE - 1) / (2 * VE)) + nrot;
  const int per_token = (int)a.H * nitems;
  const char* xb = static_cast<const char*>(a.x);
  char* ob = static_cast<char*>(a.out);
  for (int i = threadIdx.x; i < here * per_token; i += kRopeThreads) {
    const int t = i / per_token, r = i - t * per_token;
    const int h = r / nitems, item = r - h * nitems;
    const int64_t b = (t0 + t) / a.L, l = (t0 + t) - b * a.L;
    const char* x = xb + (b * a.xs[0] + h * a.xs[1] + l * a.xs[2]) * kSize;
    char* o = ob + (b * a.os[0] + h * a.os[1] + l * a.os[2]) * kSize;
    const bool rot = item < nrot;
    int c0, c1;  // first channels of the two vectors
    if (rot) {
      c0 = INTER ? 2 * item * VE : item * VE;
      c1 = INTER ? c0 + VE : c0 + half;
    } else {
      c0 = a.dims + 2 * (item - nrot) * VE;
      c1 = c0 + VE;
    }
    const bool two = c1 < a.D;
    alignas(16) V v0 = *reinterpret_cast<const V*>(x + (int64_t)c0 * kSize);
    alignas(16) V v1{};
    if (two) v1 = *reinterpret_cast<const V*>(x + (int64_t)c1 * kSize);
    if (rot) {
      const float2* cs = table + t * half + item * VE;
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float2 w = cs[j];
        if constexpr (INTER) {  // pairs 2 j, 2 j + 1 of the two vectors taken as one
          void* p = 2 * j < VE ? (void*)&v0 : (void*)&v1;
          const int e = (2 * j) % VE;
          if constexpr (VE == 1) {
            const float p0 = get<TYPE>(&v0, 0), p1 = get<TYPE>(&v1, 0);
            put<TYPE>(&v0, 0, p0 * w.x - p1 * w.y);
            put<TYPE>(&v1, 0, p0 * w.y + p1 * w.x);
          } else {
            const float p0 = get<TYPE>(p, e), p1 = get<TYPE>(p, e + 1);
            put<TYPE>(p, e, p0 * w.x - p1 * w.y);
            put<TYPE>(p, e + 1, p0 * w.y + p1 * w.x);
          }
        } else {
          const float p0 = get<TYPE>(&v0, j), p1 = get<TYPE>(&v1, j);
          put<TYPE>(&v0, j, p0 * w.x - p1 * w.y);
          put<TYPE>(&v1, j, p0 * w.y + p1 * w.x);
        }
      }
    }
    *reinterpret_cast<V*>(o + (int64_t)c0 * kSize) = v0;
    if (two) *reinterpret_cast<V*>(o + (int64_t)c1 * kSize) = v1;
  }
}

// The widest vector every address of the call allows, in elements.
int vector_elems(const RopeArgs& a, int size) {
  int ve = 16 / size;
  auto fits = [&](int v) {
    const uintptr_t m = (uintptr_t)v * size - 1;
    if ((reinterpret_cast<uintptr_t>(a.x) & m) || (reinterpret_cast<uintptr_t>(a.out) & m)) return false;
    for (int i = 0; i < 3; ++i)
      if (a.xs[i] % v || a.os[i] % v) return false;
    return (a.dims / 2) % v == 0 && (a.D - a.dims) % v == 0;
  };
  while (ve > 1 && !fits(ve)) ve >>= 1;
  return ve;
}

template <int TYPE, int VE>
cudaError_t launch_v(const RopeArgs& a, cudaStream_t st) {
  // positions per CTA: one pair per thread in the table, no fewer than about four CTAs per SM
  const int64_t all = a.B * a.L;
  int tokens = 1;
  while (tokens < 16 && 2 * tokens * (a.dims / 2) <= kRopeThreads && all / (2 * tokens) >= 4 * 148) tokens *= 2;
  const size_t smem = (size_t)tokens * (a.dims / 2) * sizeof(float2);
  const dim3 grid((unsigned)((all + tokens - 1) / tokens));
  return a.interleaved ? launch_k(rope_kernel<TYPE, VE, true>, grid, dim3(kRopeThreads), smem, st, a, tokens)
                       : launch_k(rope_kernel<TYPE, VE, false>, grid, dim3(kRopeThreads), smem, st, a, tokens);
}

template <int TYPE>
cudaError_t launch_ty(const RopeArgs& a, cudaStream_t st) {
  const int ve = vector_elems(a, TYPE == kF32 ? 4 : 2);
  if constexpr (TYPE != kF32)
    if (ve == 8) return launch_v<TYPE, 8>(a, st);
  if (ve == 4) return launch_v<TYPE, 4>(a, st);
  if (ve == 2) return launch_v<TYPE, 2>(a, st);
  return launch_v<TYPE, 1>(a, st);
}

}  // namespace

cudaError_t launch_rope(const RopeArgs& a, cudaStream_t st) {
  if (a.type == kF32) return launch_ty<kF32>(a, st);
  return a.type == kF16 ? launch_ty<kF16>(a, st) : launch_ty<kBf16>(a, st);
}

}  // namespace moe
