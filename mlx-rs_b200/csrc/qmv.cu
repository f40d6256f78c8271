// qmv.cu — 4-bit matrix products for few tokens (decode): y = x W^T, or the gated pair
// h = act(x Wg^T) * (x Wu^T), at group sizes 32, 64 and 128.
//
// Per group of `G` weights with scale s and bias b, sum_k (s q_k + b) x_k is
//   s * D + (b - 16 s) * X,  D = sum_k (16 + q_k) x_k,  X = sum_k x_k,
// where 16 + q is exact in either 16-bit type and takes one LOP3 per two weights (the field
// becomes the top mantissa bits under the exponent of 16). D and X are mma.sync products
// with fp32 accumulators (X with a matrix of ones); the weights are never rounded. Where these
// sums leave the range of fp32, or a token holds infinities, the element is formed again in 64
// bits from the weights themselves.
//
// A CTA takes tiles of 16 weight rows (gated: 8 of gate and the same 8 of up, so that a thread
// holds both projections of an element), one after the other, and all of K: its warps take
// spans of 128 columns in turn, add up in registers, and the CTA adds the warps' sums through
// shared memory in warp order. Each warp copies its spans (16 rows x 64 bytes) ahead with
// cp.async into a ring of its own, across tile borders, so that the copies run under the
// products. An MMA sums over the four lanes of a row, so all of its k must lie in one group:
// lane (g, t) reads from the ring the words of rows g and g + 8 that make it so (16-byte piece
// j of row r lies at piece j ^ swz(r): conflict-free for reads of 16, 8 and 4 bytes a lane).
// The tokens are read to match (x is small and stays in L1), each 16-byte piece permuted to
// the order in which the fields leave a word.
// Bound by the instructions of a span (about 280 for 16 x 128 weights: 64 to extract the
// fields, 16 MMAs) and their latency (issue slots 55 %) at the 20 warps per SM that 96 registers
// allow: one token, on the device, group 128 2048 -> 32768 14.7 us (2.4 TB/s; 16.0 a call), group
// 64 2048 -> 11264 6.8 us and 5632 -> 2048 5.1 us, group 32 2048 -> 2048 3.4 us. Measured against
// earlier forms of it (16 us a call for 2048 -> 32768, 2.9 for 2048 -> 2048): a warp that does the copies of a CTA, bulk copies and scales through shared
// memory (fewer instructions, but 1.5 us more before the first product: 2048 -> 2048 4.5 us),
// 32 rows per warp (19.7 us for 2048 -> 32768), the span's tokens loaded ahead (19.2 us: the
// registers), 24 warps of 80 registers (21 us).
#include <algorithm>

#include "dense.cuh"

namespace moe {

namespace {

// d = a . b, or d += a . b (ADD)
template <int TYPE, bool ADD>
MOE_DEV void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  const float c0 = ADD ? d[0] : 0.0f, c1 = ADD ? d[1] : 0.0f, c2 = ADD ? d[2] : 0.0f, c3 = ADD ? d[3] : 0.0f;
  if constexpr (TYPE == kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// 16 bytes, or zeros
MOE_DEV void copy16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
MOE_DEV uint32_t lds4(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(v) : "r"(a) : "memory");
  return v;
}
MOE_DEV uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
MOE_DEV uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
// GP consecutive scales into whole registers, so that nothing has to wait for them before
// their use: in one access where every row allows it.
template <int GP>
MOE_DEV void ldg_scales(const uint16_t* p, bool wide, int have, uint32_t (&v)[GP]) {
  if (GP == 1) {
    asm volatile("ld.global.nc.u16 %0, [%1];\n" : "=r"(v[0]) : "l"(p));
  } else if (wide) {  // v[i]: values 2 i and 2 i + 1
    if constexpr (GP == 2) asm volatile("ld.global.nc.u32 %0, [%1];\n" : "=r"(v[0]) : "l"(p));
    if constexpr (GP == 4) asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];\n" : "=r"(v[0]), "=r"(v[1]) : "l"(p));
  } else {
#pragma unroll
    for (int i = 0; i < GP; ++i)
      if (i < have) asm volatile("ld.global.nc.u16 %0, [%1];\n" : "=r"(v[i]) : "l"(p + i));
  }
}
template <int TYPE, int GP>
MOE_DEV float scale_of(const uint32_t (&v)[GP], bool wide, int i) {
  const uint32_t x = GP > 1 && wide ? v[i >> 1] : v[i];
  return GP > 1 && wide && (i & 1) ? Elem<TYPE>::hi(x) : Elem<TYPE>::lo(x);
}

constexpr int kSms = 148;
constexpr int kRing = 6;             // spans in flight per warp
constexpr int kSpanBytes = 16 * 64;  // 16 rows x 128 weights

MOE_DEV int swz(int row) { return ((row >> 1) & 1) * 2 | ((row >> 2) & 1); }
MOE_DEV uint32_t piece_at(int row, int piece) { return (uint32_t)(row * 64 + ((piece ^ swz(row)) << 4)); }

// This lane's words of row `row` of a span for the steps of a group.
template <int G>
MOE_DEV void row_words(uint32_t span, int row, int gr, int t, uint32_t (&w)[G / 32]) {
  if constexpr (G == 128) {
    *reinterpret_cast<uint4*>(w) = lds16(span + piece_at(row, t));
  } else if constexpr (G == 64) {
    *reinterpret_cast<uint2*>(w) = lds8(span + piece_at(row, 2 * gr + (t >> 1)) + (t & 1) * 8);
  } else {
    w[0] = lds4(span + piece_at(row, gr) + t * 4);
  }
}

// sum_k (s q_k + b) x_k of one row and one token in 64 bits, over the lanes of a warp.
template <int TYPE, int G>
__device__ __noinline__ float exact_sum(const PackedMatrix& m, int row, const uint16_t* x, int K, int lane) {
  double lo = 0.0, hi = 0.0;
#pragma unroll 4
  for (int i = lane; i < K >> 3; i += 32) {
    const uint32_t q = m.w[(size_t)row * (K >> 3) + i];
    const size_t g = (size_t)row * (K / G) + i / (G / 8);
    const double s = Elem<TYPE>::to_f(m.s[g]), b = m.b ? Elem<TYPE>::to_f(m.b[g]) : 0.0f;
    const uint4 v = *reinterpret_cast<const uint4*>(x + 8 * i);
    const uint32_t t[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      lo = fma(fma((double)(q >> 8 * j & 15u), s, b), (double)Elem<TYPE>::lo(t[j]), lo);
      hi = fma(fma((double)(q >> (8 * j + 4) & 15u), s, b), (double)Elem<TYPE>::hi(t[j]), hi);
    }
  }
  double sum = lo + hi;
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return (float)sum;
}
// Whether a token holds a NaN, over the lanes of a warp: its sums are right as they are.
template <int TYPE>
__device__ __noinline__ bool has_nan(const uint16_t* x, int K, int lane) {
  bool is = false;
  for (int i = lane; i < K >> 3; i += 32) {
    const uint4 v = *reinterpret_cast<const uint4*>(x + 8 * i);
    const uint32_t t[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) is |= isnan(Elem<TYPE>::lo(t[j])) || isnan(Elem<TYPE>::hi(t[j]));
  }
  return __any_sync(0xffffffffu, is);
}

// IN_PLACE: out is the residual
template <int TYPE, int G, bool GATED, int NC, bool IN_PLACE>
__global__ void __maxnreg__(NC == 4 ? 128 : 96) qmv_kernel(const __grid_constant__ QmvArgs a) {
  constexpr int GP = 128 / G;      // groups per span
  constexpr int kSteps = G / 32;   // words of a lane per group
  constexpr int kCols = 8 * NC;
  constexpr int kChains = NC == 1 ? 2 : 1;
  extern __shared__ __align__(128) unsigned char smem[];  // [warps][kRing][1 KB] | [2][warps][16][kCols] floats
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int K = a.K, spans = (K + 127) >> 7, groups = K / G;
  const int mine = (spans - warp + warps - 1) / warps;  // this warp's spans of a tile (warps <= spans)
  const uint32_t ring = smem_u32(smem) + warp * (kRing * kSpanBytes), ring_end = ring + kRing * kSpanBytes;
  float* red = reinterpret_cast<float*>(smem + warps * (kRing * kSpanBytes));
  const int tiles = a.tiles, rows = (int)a.N;
  const bool wide = groups % GP == 0;  // every row's scales start at a multiple of GP

  // this lane's rows of a tile, g and g + 8 (gated: row g of gate and of up). Rows past the
  // last read it again and are not stored.
  auto row_of = [&](int tile, int i) {
    const int n = GATED ? tile * 8 + g : tile * 16 + g + 8 * i;
    return n < rows ? n : rows - 1;
  };
  auto mat = [&](int i) -> const PackedMatrix& { return a.m[GATED ? i : 0]; };

  // ---- copies, span by span across tiles (lane (g, t): piece t of its rows)
  int c_tile = blockIdx.x, c_i = 0;
  uint32_t c_slot = ring;
  uint32_t c_at[2];  // words into the matrix
  auto copy_next = [&]() {
    if (c_tile < tiles) {
      if (c_i == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) c_at[i] = (uint32_t)row_of(c_tile, i) * (uint32_t)(K >> 3) + warp * 16 + t * 4;
      }
      const bool in = (warp + c_i * warps) * 128 + t * 32 < K;  // the last span may be short
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        copy16(c_slot + piece_at(g + 8 * i, t), mat(i).w + (in ? c_at[i] : 0u), in);
        c_at[i] += warps * 16;
      }
      if (++c_i == mine) c_i = 0, c_tile += gridDim.x;
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
    c_slot += kSpanBytes;
    if (c_slot == ring_end) c_slot = ring;
  };
  // ---- scales and biases of a span's groups, read one span ahead
  int q_tile = blockIdx.x, q_i = 0;
  uint32_t q_at[2];  // scales into the matrix
  struct Scales {
    uint32_t s[2][GP] = {}, b[2][GP] = {};
  };
  auto read_scales = [&](Scales& v) {
    if (q_tile >= tiles) return;
    if (q_i == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) q_at[i] = (uint32_t)row_of(q_tile, i) * (uint32_t)groups + warp * GP;
    }
    const int have = groups - (warp + q_i * warps) * GP;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      ldg_scales<GP>(mat(i).s + q_at[i], wide, have, v.s[i]);
      if (mat(i).b) ldg_scales<GP>(mat(i).b + q_at[i], wide, have, v.b[i]);
      q_at[i] += warps * GP;
    }
    if (++q_i == mine) q_i = 0, q_tile += gridDim.x;
  };

  // `early`: the launch before this one does not write the weights and let this one start
  // only after everything before it had completed (the second product of a block)
  if (!a.early) {
    pdl_wait();
    pdl_trigger();
  }
#pragma unroll 1
  for (int i = 0; i < kRing - 1; ++i) copy_next();
  Scales ahead;
  read_scales(ahead);
  if (a.early) {
    pdl_wait();
    pdl_trigger();
  }

  // Columns of the MMA without a token read the last token again and are not stored. The tokens
  // are read by plain loads: the launch before may write them while this kernel already runs, so
  // they are not read-only for its lifetime, which the read-only loads of the weights ask for.
  const int mbase = blockIdx.y * kCols;
  const uint16_t* xr[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int m = mbase + c * 8 + g;
    constexpr int kLaneWords = G == 128 ? 4 : G == 64 ? 2 : 1;
    xr[c] = a.x + (int64_t)(m < a.M ? m : a.M - 1) * K + warp * 128 + t * kLaneWords * 8;
  }
  // ---- an element's epilogue
  constexpr int kOut = GATED ? 8 : 16;  // rows of a tile
  auto store = [&](int n, int m, float v, float u) {
    const int64_t at = (int64_t)m * rows + n;
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
  };
  // A sum that is not finite may have left the range only by its factors of 16 + q (tokens from
  // 2^128 / 31 on, and infinities, which give inf - inf): the lanes whose sum is `bad` get it
  // again, from the weights themselves, unless the token holds a NaN. Whole warps. known, nans:
  // columns whose token was looked at, that hold one.
  auto again = [&](bool bad, int n, int m, float& v, float& u, uint32_t& known, uint32_t& nans) {
#pragma unroll 1
    for (uint32_t todo = __ballot_sync(0xffffffffu, bad); todo; todo &= todo - 1) {
      const int src = __ffs(todo) - 1;
      const int row = __shfl_sync(0xffffffffu, n, src), token = __shfl_sync(0xffffffffu, m, src);
      const uint16_t* x = a.x + (int64_t)token * K;
      const uint32_t bit = 1u << (token - mbase);
      if (!(known & bit)) {
        known |= bit;
        if (has_nan<TYPE>(x, K, lane)) nans |= bit;
      }
      if (nans & bit) continue;
      const float ev = exact_sum<TYPE, G>(a.m[0], row, x, K, lane);
      const float eu = GATED ? exact_sum<TYPE, G>(a.m[1], row, x, K, lane) : 0.0f;
      if (lane == src) v = ev, u = eu;
    }
  };
  bool lost = false;
  uint32_t slot = ring;
  int buf = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, buf ^= 1) {
    float acc[NC][4] = {};
    for (int i = 0; i < mine; ++i) {
      copy_next();
      asm volatile("cp.async.wait_group %0;\n" ::"n"(kRing - 1) : "memory");
      __syncwarp();
      const int xoff = i * warps * 128;
      const int have = groups - (warp + i * warps) * GP;  // groups of this span
      const Scales cur = ahead;
      read_scales(ahead);
#pragma unroll
      for (int gr = 0; gr < GP; ++gr) {
        if (GP > 1 && gr >= have) break;
        uint32_t w[2][kSteps];
#pragma unroll
        for (int r = 0; r < 2; ++r) row_words<G>(slot, g + 8 * r, gr, t, w[r]);
        // two chains each for eight tokens, so that an MMA does not wait for the one before
        float d[kChains][NC][4], x1[kChains][NC][4];
        constexpr int kLast = kChains - 1;
        constexpr uint32_t one = Nib<TYPE>::kOne;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          uint32_t e[NC][4];
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const uint4 q = *reinterpret_cast<const uint4*>(xr[c] + xoff + gr * G + j * 8);
            e[c][0] = __byte_perm(q.x, q.z, 0x5410), e[c][1] = __byte_perm(q.x, q.z, 0x7632);
            e[c][2] = __byte_perm(q.y, q.w, 0x5410), e[c][3] = __byte_perm(q.y, q.w, 0x7632);
          }
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            if (j == 0) {
              mma<TYPE, false>(x1[0][c], one, one, one, one, e[c][0], e[c][1]);
              mma<TYPE, kChains == 1>(x1[kLast][c], one, one, one, one, e[c][2], e[c][3]);
            } else {
              mma<TYPE, true>(x1[0][c], one, one, one, one, e[c][0], e[c][1]);
              mma<TYPE, true>(x1[kLast][c], one, one, one, one, e[c][2], e[c][3]);
            }
          }
          const uint32_t u = w[0][j], v = w[1][j];
          const uint32_t u0 = fields<TYPE, 0>(u), u1 = fields<TYPE, 1>(u), u2 = fields<TYPE, 2>(u), u3 = fields<TYPE, 3>(u);
          const uint32_t v0 = fields<TYPE, 0>(v), v1 = fields<TYPE, 1>(v), v2 = fields<TYPE, 2>(v), v3 = fields<TYPE, 3>(v);
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            if (j == 0) {
              mma<TYPE, false>(d[0][c], u0, v0, u1, v1, e[c][0], e[c][1]);
              mma<TYPE, kChains == 1>(d[kLast][c], u2, v2, u3, v3, e[c][2], e[c][3]);
            } else {
              mma<TYPE, true>(d[0][c], u0, v0, u1, v1, e[c][0], e[c][1]);
              mma<TYPE, true>(d[kLast][c], u2, v2, u3, v3, e[c][2], e[c][3]);
            }
          }
        }
        if constexpr (kChains == 2) {
#pragma unroll
          for (int k = 0; k < 4; ++k) d[0][0][k] += d[1][0][k];
          x1[0][0][0] += x1[1][0][0], x1[0][0][1] += x1[1][0][1];
        }
        const float sc0 = scale_of<TYPE, GP>(cur.s[0], wide, gr), sc1 = scale_of<TYPE, GP>(cur.s[1], wide, gr);
        const float bi0 = __fmaf_rn(-16.0f, sc0, scale_of<TYPE, GP>(cur.b[0], wide, gr));
        const float bi1 = __fmaf_rn(-16.0f, sc1, scale_of<TYPE, GP>(cur.b[1], wide, gr));
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          acc[c][0] = __fmaf_rn(sc0, d[0][c][0], __fmaf_rn(bi0, x1[0][c][0], acc[c][0]));
          acc[c][1] = __fmaf_rn(sc0, d[0][c][1], __fmaf_rn(bi0, x1[0][c][1], acc[c][1]));
          acc[c][2] = __fmaf_rn(sc1, d[0][c][2], __fmaf_rn(bi1, x1[0][c][0], acc[c][2]));
          acc[c][3] = __fmaf_rn(sc1, d[0][c][3], __fmaf_rn(bi1, x1[0][c][1], acc[c][3]));
        }
      }
      // The slot is filled again by the copy that the next round issues: this warp's own, and
      // every word above has gone into an MMA whose sum the line before waited for.
      __syncwarp();
      slot += kSpanBytes;
      if (slot == ring_end) slot = ring;
    }
    // ---- the warps' sums, in warp order (two buffers: one barrier per tile)
    float* rb = red + buf * (warps * 16 * kCols);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float* at = rb + (warp * 16 + g) * kCols + c * 8 + 2 * t;
      *reinterpret_cast<float2*>(at) = make_float2(acc[c][0], acc[c][1]);
      *reinterpret_cast<float2*>(at + 8 * kCols) = make_float2(acc[c][2], acc[c][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kOut * kCols; i += blockDim.x) {
      const int row = i % kOut, col = i / kOut;
      const int n = tile * kOut + row;
      const int m = mbase + col;
      const bool in = n < rows && m < a.M;
      if (!IN_PLACE && !in) continue;
      float v = 0.0f, u = 0.0f;
      if (in)
        for (int w = 0; w < warps; ++w) {
          v += rb[(w * 16 + row) * kCols + col];
          if (GATED) u += rb[(w * 16 + 8 + row) * kCols + col];
        }
      const bool bad = !isfinite(v) || (GATED && !isfinite(u));
      if constexpr (IN_PLACE) {
        uint32_t known = 0, nans = 0;
        again(bad, n, m, v, u, known, nans);
      }
      lost |= bad;
      if (in) store(n, m, v, u);
    }
  }
  asm volatile("cp.async.wait_all;\n" ::: "memory");
  // Such an element's output is not finite either. Done here, and not in the tiles' loop, whose
  // registers are all taken: a call without such elements takes 0 to 3 % longer for it up to 8
  // tokens and -2 to +3 % from 9 to 32, there it would be up to 6 %. In place the output cannot be
  // formed twice. A token with an infinity, 2048 -> 32768, takes 93 us, one with a NaN 20 (14.7).
  if (!IN_PLACE && __any_sync(0xffffffffu, lost)) {
    uint32_t known = 0, nans = 0;
#pragma unroll 1
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x)
#pragma unroll 1
      for (int i = threadIdx.x; i < kOut * kCols; i += blockDim.x) {
        const int n = tile * kOut + i % kOut, m = mbase + i / kOut;
        const bool bad = n < rows && m < a.M && !isfinite(Elem<TYPE>::to_f(a.out[(int64_t)m * rows + n]));
        float v = __int_as_float(0x7fffffff), u = v;  // of a token with a NaN
        again(bad, n, m, v, u, known, nans);
        if (bad) store(n, m, v, u);
      }
  }
}

template <int TYPE, int G, bool GATED, int NC, bool IN_PLACE = false>
cudaError_t launch_nc(const QmvArgs& args, cudaStream_t st) {
  if constexpr (!GATED && !IN_PLACE)
    if (args.residual == args.out) return launch_nc<TYPE, G, GATED, NC, true>(args, st);
  QmvArgs a = args;
  const int per_tile = GATED ? 8 : 16;
  a.tiles = (int)((a.N + per_tile - 1) / per_tile);
  const int spans = (a.K + 127) / 128;
  // warps per CTA: four; more with fewer spans each while the tiles alone would not give the
  // SMs 16 warps
  int warps = spans < 4 ? spans : 4;
  while (warps < 16 && a.tiles * warps < kSms * 16 && spans >= 2 * warps) warps *= 2;
  const size_t smem = (size_t)warps * (kRing * kSpanBytes + 2 * 16 * 8 * NC * sizeof(float));
  auto kern = qmv_kernel<TYPE, G, GATED, NC, IN_PLACE>;
  static std::atomic<uint64_t> done{0};
  cudaError_t err = allow_smem(kern, 16 * (kRing * kSpanBytes + 2 * 16 * 8 * NC * (int)sizeof(float)), done);
  if (err != cudaSuccess) return err;
  // CTAs that the SMs hold at once (20 warps of 96 registers, 227 KB of shared memory)
  const int per_sm = std::max(1, std::min((NC == 4 ? 16 : 20) / warps, (int)((227 * 1024) / (smem + 1024))));
  const int m_tiles = (a.M + 8 * NC - 1) / (8 * NC);
  const int most = std::max(1, kSms * per_sm / m_tiles);
  const dim3 grid((unsigned)std::min(a.tiles, most), (unsigned)m_tiles);
  return launch_k(kern, grid, dim3(32 * warps), smem, st, a);
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

bool qmv_fits(int64_t M, int64_t N, int64_t K, bool gated) {
  // offsets into a matrix are 32-bit words
  if (M > 32 || N >= (int64_t(1) << 30) || N * (K / 8) >= (int64_t(1) << 32)) return false;
  // Up to eight tokens the weights' bytes count, and these kernels read them best. Above, a
  // warp's MMAs and permutations of x do, and the tensor-memory products are faster once they
  // have enough weights to work on (us here / there): 16 tokens, 2048 -> 11264 10.4 / 15,
  // 2048 -> 32768 29 / 26; 32 tokens, 2048 -> 2048 6.7 / 9.1, 5632 -> 2048 10.9 / 12.9,
  // 2048 -> 11264 23 / 15.
  const int64_t weights = N * (gated ? 2 : 1) * K;
  return M <= 8 || weights <= (int64_t(M <= 16 ? 48 : 12) << 20);
}

cudaError_t launch_qmv(const QmvArgs& a, bool gated, cudaStream_t st) {
  if (!qmv_fits(a.M, a.N, a.K, gated)) return cudaErrorInvalidValue;
  if (a.type == kF16) return gated ? launch_ty<kF16, true>(a, st) : launch_ty<kF16, false>(a, st);
  return gated ? launch_ty<kBf16, true>(a, st) : launch_ty<kBf16, false>(a, st);
}

}  // namespace moe
