// rope.cu — rotary positions: fast_rope of MLX (mlx_fast_rope) on strided [B, H, L, D] tensors.
//
// Pair i of a head at position p is turned by the angle p * scale / wavelength_i, with
// wavelength_i = base^(2 i / dims) or freqs[i]: (a, b) -> mscale (a cos - b sin, a sin + b cos).
// Pairs are (i, i + dims / 2), or (2 i, 2 i + 1) when interleaved; channels from dims on pass
// through. The transposed rotation (the gradient) has the angle's sign turned.
//
// The angle is formed in turns in 64 bits and reduced to [-1/2, 1/2] before it becomes a
// float: at position 10^6 a 32-bit angle is already off by a few hundredths of a radian.
// The floor is the bytes (one read and one write of the tensor; at 4096 positions the writes stay
// in L2, and neither DRAM nor the issue slots, 57 % active, are full; what bounds it has not been
// shown). A CTA takes `tokens` positions with all of their heads: it fills a table of cosines and
// sines in shared memory once, one pair per thread, so that the 64-bit work is spread over the
// threads and shared by the heads, then moves the heads through two vectors per item, the loads of
// two items in flight.
// 36 heads of 128 bf16 channels out of a fused projection: 4096 positions 15.8 us (4.8 TB/s),
// 8192 30.9 us (4.9 TB/s); one position of 64 sequences 2.5 us; 2 x 1023 x 16 heads of 80, f32,
// interleaved, 5.3 us. Measured against it, the same four in us: one item in flight 15.4, 28.1,
// 2.5, 6.3 (faster for 16-bit prompts, slower for f32); three 18.2, 36.1, 2.6, 7.1 (registers);
// one in flight as two named copies, with CTAs of 128 threads 16.5, 31.0, 2.7, 6.3, of 256 17.5,
// 34.5, 2.4, 6.1, of 512 22.1, 36.6, 2.2, 7.7; 64-bit index arithmetic 19.2, 33.1, 3.0, 6.6.
#include "dense.cuh"

namespace moe {

namespace {

constexpr int kRopeThreads = 128;
constexpr int kAhead = 2;  // items per thread whose loads are in flight

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

// n / d for n < 2^31 (a multiplication by a rounded-up reciprocal, exact with 32 + log2 d bits)
struct Divider {
  uint32_t d, mul, shift;
  explicit Divider(uint32_t v) : d(v), mul(0), shift(0) {
    while ((uint64_t(1) << shift) < v) ++shift;
    mul = (uint32_t)(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - v)) / v + 1);
  }
  MOE_DEV uint32_t operator()(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};
struct RopeParams {
  RopeArgs a;
  int tokens, nrot;           // positions per CTA; rotating items of a head
  Divider heads, items, len;  // by H, items of a head, L
};

// VE: elements per vector access (16 bytes where every address allows it). An item is two
// vectors of a head: the two halves' pairs, or 2 VE channels (interleaved pairs, and channels
// that pass through).
template <int TYPE, int VE, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ RopeParams p) {
  constexpr int kSize = TYPE == kF32 ? 4 : 2;
  using V = typename Vec<VE * kSize>::T;
  extern __shared__ __align__(16) float2 table[];  // [tokens][dims / 2]: mscale cos, mscale sin
  const RopeArgs& a = p.a;
  const int half = a.dims >> 1;
  const uint32_t t0 = blockIdx.x * (uint32_t)p.tokens, all = (uint32_t)(a.B * a.L);
  const int here = (int)(all - t0 < (uint32_t)p.tokens ? all - t0 : (uint32_t)p.tokens);
  const uint32_t total = (uint32_t)here * p.heads.d * p.items.d;
  const char* xb = static_cast<const char*>(a.x);
  char* ob = static_cast<char*>(a.out);

  struct Item {
    V v0, v1;
    int64_t o0, o1;  // byte offsets in the output
    int row, rot;    // table row of the token, first pair (negative: passes through)
    bool two;
  };
  auto fetch = [&](uint32_t i, Item& q) {
    const uint32_t r = p.items(i), item = i - r * p.items.d;
    const uint32_t t = p.heads(r), h = r - t * p.heads.d;
    const uint32_t b = p.len(t0 + t), l = t0 + t - b * p.len.d;
    int c0, c1;  // first channels of the two vectors
    q.rot = -1;
    if ((int)item < p.nrot) {
      c0 = INTER ? 2 * (int)item * VE : (int)item * VE;
      c1 = INTER ? c0 + VE : c0 + half;
      q.rot = (int)item * VE;
    } else {
      c0 = a.dims + 2 * ((int)item - p.nrot) * VE;
      c1 = c0 + VE;
    }
    q.row = (int)t * half;
    q.two = c1 < a.D;
    const int64_t x = (int64_t)b * a.xs[0] + (int64_t)h * a.xs[1] + (int64_t)l * a.xs[2];
    const int64_t o = (int64_t)b * a.os[0] + (int64_t)h * a.os[1] + (int64_t)l * a.os[2];
    q.o0 = (o + c0) * kSize, q.o1 = (o + c1) * kSize;
    q.v0 = *reinterpret_cast<const V*>(xb + (x + c0) * kSize);
    if (q.two) q.v1 = *reinterpret_cast<const V*>(xb + (x + c1) * kSize);
  };

  pdl_wait();
  pdl_trigger();
  // the first items are on their way while the table is made
  Item ring[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (threadIdx.x + k * kRopeThreads < total) fetch(threadIdx.x + k * kRopeThreads, ring[k]);
  for (int i = threadIdx.x; i < here * half; i += kRopeThreads) {
    const int t = i / half, k = i - t * half;
    const uint32_t b = p.len(t0 + t), l = t0 + t - b * p.len.d;
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
  auto turn = [&](Item& cur) {
    if (cur.rot >= 0) {
      const float2* cs = table + cur.row + cur.rot;
      if constexpr (TYPE != kF32 && VE > 1) {  // two 16-bit channels of a word at a time
        uint32_t* w0 = reinterpret_cast<uint32_t*>(&cur.v0);
        uint32_t* w1 = reinterpret_cast<uint32_t*>(&cur.v1);
#pragma unroll
        for (int j = 0; j < VE / 2; ++j) {
          const float4 w = *reinterpret_cast<const float4*>(cs + 2 * j);  // cos, sin of two pairs
          if constexpr (INTER) {  // a word is a pair; the vectors' words in turn
            uint32_t& u = 2 * j < VE / 2 ? w0[2 * j] : w1[2 * j - VE / 2];
            uint32_t& v = 2 * j + 1 < VE / 2 ? w0[2 * j + 1] : w1[2 * j + 1 - VE / 2];
            const float a0 = Elem<TYPE>::lo(u), b0 = Elem<TYPE>::hi(u), a1 = Elem<TYPE>::lo(v), b1 = Elem<TYPE>::hi(v);
            u = Elem<TYPE>::pack(a0 * w.x - b0 * w.y, a0 * w.y + b0 * w.x);
            v = Elem<TYPE>::pack(a1 * w.z - b1 * w.w, a1 * w.w + b1 * w.z);
          } else {
            const float a0 = Elem<TYPE>::lo(w0[j]), a1 = Elem<TYPE>::hi(w0[j]);
            const float b0 = Elem<TYPE>::lo(w1[j]), b1 = Elem<TYPE>::hi(w1[j]);
            w0[j] = Elem<TYPE>::pack(a0 * w.x - b0 * w.y, a1 * w.z - b1 * w.w);
            w1[j] = Elem<TYPE>::pack(a0 * w.y + b0 * w.x, a1 * w.w + b1 * w.z);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float2 w = cs[j];
          if constexpr (INTER && VE > 1) {  // pairs 2 j, 2 j + 1 of the two vectors taken as one
            void* v = 2 * j < VE ? (void*)&cur.v0 : (void*)&cur.v1;
            const int e = (2 * j) % VE;
            const float p0 = get<TYPE>(v, e), p1 = get<TYPE>(v, e + 1);
            put<TYPE>(v, e, p0 * w.x - p1 * w.y);
            put<TYPE>(v, e + 1, p0 * w.y + p1 * w.x);
          } else {  // one element of each vector
            const float p0 = get<TYPE>(&cur.v0, j), p1 = get<TYPE>(&cur.v1, j);
            put<TYPE>(&cur.v0, j, p0 * w.x - p1 * w.y);
            put<TYPE>(&cur.v1, j, p0 * w.y + p1 * w.x);
          }
        }
      }
    }
    *reinterpret_cast<V*>(ob + cur.o0) = cur.v0;
    if (cur.two) *reinterpret_cast<V*>(ob + cur.o1) = cur.v1;
  };
  for (uint32_t i = threadIdx.x; i < total; i += kAhead * kRopeThreads) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const uint32_t at = i + k * kRopeThreads;
      if (at >= total) break;
      Item cur = ring[k];
      if (at + kAhead * kRopeThreads < total) fetch(at + kAhead * kRopeThreads, ring[k]);
      turn(cur);
    }
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
  const int nrot = a.dims / 2 / VE, items = nrot + (a.D - a.dims + 2 * VE - 1) / (2 * VE);
  const RopeParams p{a, tokens, nrot, Divider((uint32_t)a.H), Divider((uint32_t)items), Divider((uint32_t)a.L)};
  const size_t smem = (size_t)tokens * (a.dims / 2) * sizeof(float2);
  const dim3 grid((unsigned)((all + tokens - 1) / tokens));
  return a.interleaved ? launch_k(rope_kernel<TYPE, VE, true>, grid, dim3(kRopeThreads), smem, st, p)
                       : launch_k(rope_kernel<TYPE, VE, false>, grid, dim3(kRopeThreads), smem, st, p);
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
