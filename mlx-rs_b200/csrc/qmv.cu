// qmv.cu — 4-bit matrix products for few tokens (decode): y = x W^T, or the gated pair
// h = act(x Wg^T) * (x Wu^T), at group sizes 32, 64 and 128.
//
// Per group of `G` weights with scale s and bias b, sum_k (s q_k + b) x_k is
//   s * D + (b - 16 s) * X,  D = sum_k (16 + q_k) x_k,  X = sum_k x_k,
// where 16 + q is exact in either 16-bit type and takes one LOP3 per two weights (the field
// becomes the top mantissa bits under the exponent of 16). D and X are mma.sync products
// with fp32 accumulators (X with a matrix of ones); the weights are never rounded.
//
// A CTA owns 16 weight rows (gated: 8 of gate and the same 8 of up, so that a thread holds
// both projections of an element) and all of K: its warps take spans of 128 columns in turn,
// add up in registers, and the CTA adds the warps' sums through shared memory in warp order.
// Lane (g, t) reads 16 bytes (32 columns) of rows g and g + 8 straight into registers: four
// lanes cover 64 contiguous bytes of a row, and every load of a batch is in flight before
// the first is used. An MMA sums over the four lanes of a row, so all of its k must lie in
// one group: the lanes first exchange words by shuffles (none at G = 128, one step at 64,
// two at 32); the tokens are read to match (x is small and stays in L1), each 16-byte piece
// permuted to the order in which the fields leave a word.
// Bound by the bytes of W for up to 8 tokens; beyond, by the MMAs and the permutations of x
// (8 tokens more share the weight fragments).
#include "dense.cuh"

namespace moe {

namespace {

template <int TYPE>
MOE_DEV void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (TYPE == kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

MOE_DEV void swap_words(uint32_t& keep_lo, uint32_t& keep_hi, bool hi, int mask) {
  // a lane with !hi gives keep_hi and takes the partner's keep_lo in its place; one with hi
  // gives keep_lo and takes the partner's keep_hi
  const uint32_t give = hi ? keep_lo : keep_hi;
  const uint32_t got = __shfl_xor_sync(0xffffffffu, give, mask);
  if (hi) keep_lo = got;
  else keep_hi = got;
}

// Words so that step i's four lanes hold words of one group (see word_of for which).
template <int G>
MOE_DEV void exchange(uint4& w, int t) {
  if constexpr (G == 64) {
    swap_words(w.x, w.z, t >= 2, 2);
    swap_words(w.y, w.w, t >= 2, 2);
  } else if constexpr (G == 32) {
    swap_words(w.x, w.y, t & 1, 1);
    swap_words(w.z, w.w, t & 1, 1);
    swap_words(w.x, w.z, t >= 2, 2);
    swap_words(w.y, w.w, t >= 2, 2);
  }
}
template <int G>
MOE_DEV int word_of(int t, int i) {
  if constexpr (G == 128) return 4 * t + i;
  if constexpr (G == 64) return 4 * ((t & 1) + (i & 2)) + (t & 2) + (i & 1);
  return 4 * i + t;
}

MOE_DEV uint4 ldg16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

template <int TYPE, int G, bool GATED, int NC>
__global__ void __launch_bounds__(512) qmv_kernel(const __grid_constant__ QmvArgs a) {
  constexpr int GP = 128 / G;           // groups per span
  constexpr int kBatch = NC == 1 ? 4 : 2;  // spans of weights in flight per warp
  extern __shared__ float red[];        // [warps][16][8 NC]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int K = a.K, spans = (K + 127) >> 7, groups = K / G;
  const int64_t n0 = (int64_t)blockIdx.x * (GATED ? 8 : 16);
  const int64_t last = a.N - 1;  // rows past the last read it again and are not stored
  const int64_t r0 = n0 + g < last ? n0 + g : last;
  const int64_t r1 = GATED ? r0 : (n0 + 8 + g < last ? n0 + 8 + g : last);
  const PackedMatrix& m1 = GATED ? a.m[1] : a.m[0];
  const uint32_t* w0 = a.m[0].w + r0 * (K >> 3) + t * 4;
  const uint32_t* w1 = m1.w + r1 * (K >> 3) + t * 4;
  const uint16_t* s0 = a.m[0].s + r0 * groups;
  const uint16_t* s1 = m1.s + r1 * groups;
  const uint16_t* b0 = a.m[0].b ? a.m[0].b + r0 * groups : nullptr;
  const uint16_t* b1 = m1.b ? m1.b + r1 * groups : nullptr;

  uint4 wa[kBatch], wb[kBatch];
  uint32_t sa[kBatch], sb[kBatch];  // scale | bias << 16 of group `span * GP + t` (t < GP)
  auto load = [&](int base) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int s = base + i * warps;
      const bool in = s < spans && s * 128 + t * 32 < K;
      wa[i] = in ? ldg16(w0 + s * 16) : make_uint4(0, 0, 0, 0);
      wb[i] = in ? ldg16(w1 + s * 16) : make_uint4(0, 0, 0, 0);
      const int gi = s * GP + (GP == 1 ? 0 : t);
      const bool sin = s < spans && (GP == 1 || t < GP) && gi < groups;
      sa[i] = sin ? (uint32_t)__ldg(s0 + gi) | (b0 ? (uint32_t)__ldg(b0 + gi) << 16 : 0u) : 0u;
      sb[i] = sin ? (uint32_t)__ldg(s1 + gi) | (b1 ? (uint32_t)__ldg(b1 + gi) << 16 : 0u) : 0u;
    }
  };
  // `early`: the launch before this one does not write the weights and let this one start
  // only after everything before it had completed (the second product of a block)
  if (a.early) load(warp);
  pdl_wait();
  pdl_trigger();
  if (!a.early) load(warp);

  const int mbase = blockIdx.y * (8 * NC);
  const uint16_t* xr[NC];
  bool xin[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int m = mbase + c * 8 + g;
    xin[c] = m < a.M;
    xr[c] = a.x + (int64_t)(xin[c] ? m : 0) * K;
  }
  float acc[NC][4] = {};
  for (int base = warp; base < spans; base += warps * kBatch) {
    if (base != warp) load(base);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int s = base + i * warps;
      if (s >= spans) break;
      exchange<G>(wa[i], t);
      exchange<G>(wb[i], t);
      const uint32_t* pa = &wa[i].x;
      const uint32_t* pb = &wb[i].x;
#pragma unroll
      for (int gr = 0; gr < GP; ++gr) {
        float d[NC][4] = {}, x1[NC][4] = {};
#pragma unroll
        for (int j = 0; j < 4 / GP; ++j) {
          const int step = gr * (4 / GP) + j;
          const int col = (s * 16 + word_of<G>(t, step)) * 8;
          const uint32_t u = pa[step], v = pb[step];
          const uint32_t u0 = fields<TYPE, 0>(u), u1 = fields<TYPE, 1>(u), u2 = fields<TYPE, 2>(u), u3 = fields<TYPE, 3>(u);
          const uint32_t v0 = fields<TYPE, 0>(v), v1 = fields<TYPE, 1>(v), v2 = fields<TYPE, 2>(v), v3 = fields<TYPE, 3>(v);
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            uint4 q = make_uint4(0, 0, 0, 0);
            if (xin[c] && col < K) q = __ldg(reinterpret_cast<const uint4*>(xr[c] + col));
            const uint32_t e0 = __byte_perm(q.x, q.z, 0x5410), e1 = __byte_perm(q.x, q.z, 0x7632);
            const uint32_t e2 = __byte_perm(q.y, q.w, 0x5410), e3 = __byte_perm(q.y, q.w, 0x7632);
            constexpr uint32_t one = Nib<TYPE>::kOne;
            mma<TYPE>(d[c], u0, v0, u1, v1, e0, e1);
            mma<TYPE>(x1[c], one, one, one, one, e0, e1);
            mma<TYPE>(d[c], u2, v2, u3, v3, e2, e3);
            mma<TYPE>(x1[c], one, one, one, one, e2, e3);
          }
        }
        const int src = (lane & ~3) | gr;
        const uint32_t qa = GP == 1 ? sa[i] : __shfl_sync(0xffffffffu, sa[i], src);
        const uint32_t qb = GP == 1 ? sb[i] : __shfl_sync(0xffffffffu, sb[i], src);
        const float sc0 = Elem<TYPE>::lo(qa), sc1 = Elem<TYPE>::lo(qb);
        const float bi0 = __fmaf_rn(-16.0f, sc0, Elem<TYPE>::hi(qa)), bi1 = __fmaf_rn(-16.0f, sc1, Elem<TYPE>::hi(qb));
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          acc[c][0] = __fmaf_rn(sc0, d[c][0], __fmaf_rn(bi0, x1[c][0], acc[c][0]));
          acc[c][1] = __fmaf_rn(sc0, d[c][1], __fmaf_rn(bi0, x1[c][1], acc[c][1]));
          acc[c][2] = __fmaf_rn(sc1, d[c][2], __fmaf_rn(bi1, x1[c][0], acc[c][2]));
          acc[c][3] = __fmaf_rn(sc1, d[c][3], __fmaf_rn(bi1, x1[c][1], acc[c][3]));
        }
      }
    }
  }
  // ---- the warps' sums, in warp order
  constexpr int kCols = 8 * NC;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float* r = red + (warp * 16 + g) * kCols + c * 8 + 2 * t;
    *reinterpret_cast<float2*>(r) = make_float2(acc[c][0], acc[c][1]);
    *reinterpret_cast<float2*>(r + 8 * kCols) = make_float2(acc[c][2], acc[c][3]);
  }
  __syncthreads();
  constexpr int kRows = GATED ? 8 : 16;
  for (int i = threadIdx.x; i < kRows * kCols; i += blockDim.x) {
    const int row = i % kRows, col = i / kRows;
    const int64_t n = n0 + row;
    const int m = mbase + col;
    if (n >= a.N || m >= a.M) continue;
    float v = 0.0f, u = 0.0f;
    for (int w = 0; w < warps; ++w) {
      v += red[(w * 16 + row) * kCols + col];
      if (GATED) u += red[(w * 16 + 8 + row) * kCols + col];
    }
    const int64_t at = (int64_t)m * a.N + n;
    if constexpr (GATED) {
      if (a.gate) {
        a.gate[at] = (uint16_t)Elem<TYPE>::pack(v, 0.0f);
        a.up[at] = (uint16_t)Elem<TYPE>::pack(u, 0.0f);
      }
      v = act_val(v, a.act) * u;
    } else if (a.residual) {
      v += Elem<TYPE>::to_f(a.residual[at]);
    }
    a.out[at] = (uint16_t)Elem<TYPE>::pack(v, 0.0f);
  }
}

template <int TYPE, int G, bool GATED, int NC>
cudaError_t launch_nc(const QmvArgs& a, cudaStream_t st) {
  const int64_t tiles = GATED ? (a.N + 7) / 8 : (a.N + 15) / 16;
  const int spans = (a.K + 127) / 128;
  // warps per CTA: a warp takes up to four spans at once; more warps with fewer spans each
  // while the tiles alone would not give the SMs 16 warps
  int warps = 4;
  while (warps < 16 && (spans > 4 * warps || (tiles * warps < 148 * 16 && spans > warps))) warps *= 2;
  const dim3 grid((unsigned)tiles, (unsigned)((a.M + 8 * NC - 1) / (8 * NC)));
  return launch_k(qmv_kernel<TYPE, G, GATED, NC>, grid, dim3(32 * warps), (size_t)warps * 16 * 8 * NC * sizeof(float),
                  st, a);
}
template <int TYPE, int G, bool GATED>
cudaError_t launch_g(const QmvArgs& a, cudaStream_t st) {
  if (a.M <= 8) return launch_nc<TYPE, G, GATED, 1>(a, st);
  if (a.M <= 16) return launch_nc<TYPE, G, GATED, 2>(a, st);
  return launch_nc<TYPE, G, GATED, 4>(a, st);
}
template <int TYPE, bool GATED>
cudaError_t launch_ty(const QmvArgs& a, cudaStream_t st) {
  if (a.group == 32) return launch_g<TYPE, 32, GATED>(a, st);
  if (a.group == 64) return launch_g<TYPE, 64, GATED>(a, st);
  return launch_g<TYPE, 128, GATED>(a, st);
}

}  // namespace

cudaError_t launch_qmv(const QmvArgs& a, bool gated, cudaStream_t st) {
  if (a.type == kF16) return gated ? launch_ty<kF16, true>(a, st) : launch_ty<kF16, false>(a, st);
  return gated ? launch_ty<kBf16, true>(a, st) : launch_ty<kBf16, false>(a, st);
}

}  // namespace moe
