// dense_gemm.cu — 4-bit matrix products on tcgen05 with the feed-forward block's epilogues.
//
// D[m, n] = sum_p A_p[m, :] . W_p[n, :]^T, or A_p . W_p with the weights' rows as the summed
// index (the gradient's direction), fp32 accumulators in tensor memory. Tokens are the MMA's
// rows (an epilogue thread owns one token and walks its columns), weights its columns; K runs
// in steps of 64. w = RN16(s q + b): one rounding, because a tcgen05 product takes both
// operands in one 16-bit type.
// The packed form dequantises in the product, so that no 16-bit copy of the weights exists in
// global memory; 23 warps:
//   warps 0-3   read the finished accumulator back and apply the epilogue, while the next
//               tile accumulates in the other buffer. A warp's global accesses go through a
//               1 KB buffer, so that they cover 32 contiguous bytes of 16 rows each;
//   warps 4-19  four groups, taking the K steps in turn: a thread turns the 64 weights of one
//               row (32 bytes packed, one or two quantization groups) into eight 16-byte
//               pieces of the B tile. With the rows summed, a word's eight weights are
//               neighbours along N and the tile is MN-major; the addresses are the same in
//               both layouts, only the meaning of a row differs;
//   warp 20     streams the token tile with TMA (128 bytes of each row, swizzled);
//   warp 21     allocates the tensor memory (two accumulators) and issues tcgen05.mma from one
//               lane: M = 128 (256 over a pair of CTAs), K = 16;
//   warp 22     streams the packed tiles with TMA into a ring of their own.
// The wide form (weights already in 16 bits, kWideMinM) has eight epilogue warps, then the TMA
// warp, which streams the weights' tile beside the tokens', and the MMA warp.
// CTA pairs (CG = 2, more than 128 tokens): each CTA loads its own 128 tokens and its half of
// the weight rows, once per 256 tokens; the leader (even rank) owns the full and
// accumulator-empty barriers and issues the MMAs of both. In the gated form the two halves of
// a tile's columns are gate rows and the same rows of up, so that one thread holds g and u of
// the same element.
// Few tiles (packed form): K is split over the CTAs of a cluster (up to 8). Each leaves its
// fp32 sums in its own shared memory, and after a cluster barrier every CTA adds one slice of
// the tokens over the cluster in split order (distributed shared memory; no atomics, the same
// bits on every run) and applies the epilogue to it.
// Every wait is bounded (2 s): on expiry the CTA records a code in the device's status word,
// stops working and leaves through the same barriers as the rest of its cluster.
//
// What bounds it. Packed: not the tensor pipe (active 47 % in the gated product of 512 tokens)
// nor the issue slots (46 %): a K step takes 0.3 / 0.5 us at 64 / 128 weight rows per CTA, of
// which a group of warps dequantises for about 40 %, waits for its stage for 20 % and spends
// 15 to 20 % on issuing the next scales' loads; and a round has 4.5 us of start, first loads and
// epilogue. 512 tokens of the block 2048 x 5632 44.7 us (0.79 PFLOP/s), 5632 -> 2048 20.4 us with
// the rows summed. Wide: the tensor pipe, active 87 to 93 % of the cycles in the plain and gated
// products (block 2048 x 5632, 4096 tokens, with the dequantisation: forward 208 us, 1.36
// PFLOP/s; with the gradients 464 us, 1.22). In the product with the gated gradient it is active
// 57 %: beside the operands g and u are read and dg and du written, 1.1 GB through L2 at 11.7
// TB/s. Measured against it: weights left in 16 bits by a launch before for every size (64.6 us
// for 512 tokens), cluster-scope arrivals on the step barriers (twice the time per step: each is
// a fence over global memory), 12 or 16 epilogue warps in the gated gradient and its g and u one
// or two chunks ahead (all within 0.6 %); in the packed form five stages instead of four (up to
// 2.5 % slower), scales staged in shared memory by the packing warp (9 to 88 % slower), rows
// dequantised into registers before the wait for their stage (1 to 5 % slower).
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>

#include "dense.cuh"

namespace moe {

namespace {

constexpr int kBM = 128, kBK = 64;
constexpr int kATile = kBM * kBK * 2;      // 16 KB
constexpr int kBTile = 128 * kBK * 2;      // 16 KB: this CTA's weight rows of a tile, at most 128
constexpr int kPackBytes = 128 * 32;       // 4 KB: their packed K step
constexpr int kStageBuf = 1024;            // 32 rows x 16 columns of 16 bits, per epilogue warp
constexpr int kSms = 148;

__device__ int32_t g_dense_status;

constexpr int kStageBytes = kATile + kBTile;
constexpr int kSumPitch = 260;
// The two sources of the weight tile. PACKED: dequantised by this kernel's warps; otherwise
// 16-bit weights (dense_dequant.cu wrote them) that TMA copies like the tokens.
// Shared memory: [stages][token tile, weight tile] | [slots][packed step] | [epilogue warps][1 KB]
// | full[S] empty[S] acc_full[2] acc_empty[2] pfull[P] pempty[P] | tensor-memory base.
template <bool PACKED>
struct Cfg {
  static constexpr int kEpiWarps = PACKED ? 4 : 8;
  static constexpr int kGroups = PACKED ? 4 : 0;  // of 4 dequantising warps
  static constexpr int kDeqWarp = kEpiWarps;
  static constexpr int kTmaWarp = kDeqWarp + 4 * kGroups, kMmaWarp = kTmaWarp + 1, kPackWarp = kTmaWarp + 2;
  static constexpr int kThreads = (kMmaWarp + 1 + (PACKED ? 1 : 0)) * 32;
  static constexpr int kStages = PACKED ? 4 : 6, kSlots = PACKED ? 8 : 0;
  static constexpr int kPackAt = kStages * kStageBytes;
  static constexpr int kStagingAt = kPackAt + kSlots * kPackBytes;
  static constexpr int kBarsAt = kStagingAt + kEpiWarps * kStageBuf;
  static constexpr int kNumBars = 2 * kStages + 4 + 2 * kSlots;
  static constexpr int kSmem = kBarsAt + 8 * kNumBars + 16 + 1024;
  // A group that waits for a stage has written its step kGroups before, so the stage's
  // previous use but one is over when kGroups <= kStages, and one parity bit tells the phases
  // apart; a slot belongs to one group.
  static_assert(kGroups <= kStages && (!PACKED || kSlots % (PACKED ? kGroups : 1) == 0), "phases told apart by parity");
  // the split form leaves its sums, rows of 256 floats and one 16-byte piece (so that a column
  // of rows spreads over the banks), over the operand stages and the packed slots
  static_assert(kBM * kSumPitch * 4 <= kStagingAt, "sums over the stages and slots");
};

struct WeightSide {  // scales and biases of one operand pair's weights
  const uint16_t* s;
  const uint16_t* b;
};
struct GemmParams {
  CUtensorMap a[2], w[2];
  WeightSide q[2];
  int64_t M;
  int N;
  int rows;             // weight rows of each matrix (N, or the summed K when ROWS_K)
  int s_pitch;          // scales per weight row
  int lg;               // log2 of the group size
  int gated;
  int hb;               // weight rows (columns of D) per half of a tile
  int ks0, ks;          // K steps of the first operand pair, of all
  int tiles_m, splits, spk;
  int units;            // tiles
  int a_rows;           // token rows of a box: all 128 of a tile, or those of the only tile
  int wide;             // the weights are 16-bit (w maps them), not packed
  int early;            // the weights may be read before the launch before has completed
  DenseEpi e;
};

// The address of `a` in CTA `rank` of the cluster.
MOE_DEV uint32_t map_rank(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
// Arrival on a barrier of this CTA, or of the pair's leader (an address from map_rank). CTA
// scope on purpose: what it publishes is this SM's shared memory (after fence_proxy) or tensor
// memory (after tc_before); cluster scope costs a fence over global memory in every step.
MOE_DEV void mbar_arrive_cluster(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_bar) : "memory");
}
template <int CG>
MOE_DEV void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3}], [%4];\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
MOE_DEV void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
MOE_DEV void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
MOE_DEV void fence_proxy() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
// 1 in one lane of the (converged) warp.
MOE_DEV uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}\n" : "=r"(r));
  return r;
}
template <int CG>
MOE_DEV void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
// Arrives on `bar` of every CTA in `mask` when the MMAs issued so far have completed.
template <int CG>
MOE_DEV void tc_commit(uint32_t bar, uint32_t mask) {
  if constexpr (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(
            bar),
        "h"((uint16_t)mask)
        : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
}
// K-major operand rows of 128 bytes, 128-byte swizzle, 8-row groups 1024 bytes apart.
MOE_DEV uint64_t sw128_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3fffu) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
// N-contiguous operand: 64-column blocks of 64 rows x 128 bytes (8 KB apart, the leading
// offset), 8-row groups 1024 bytes apart.
MOE_DEV uint64_t sw128_mn_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3fffu) | (uint64_t)(8192 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
MOE_DEV void tmem_ld16(uint32_t taddr, float (&r)[16]) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(taddr));
}
MOE_DEV void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }

// ---- W (4 or 8) consecutive elements of a 16-bit row, at column c of n (vec, four: rows of 16-byte
// aligned multiples of 8; otherwise element by element, columns beyond n left alone)
template <int TYPE, int W>
MOE_DEV void load_n(const uint16_t* row, int c, int n, bool vec, float (&v)[W]) {
  if (W == 4 && vec) {
    uint32_t q[W / 2];
    *reinterpret_cast<uint2*>(q) = *reinterpret_cast<const uint2*>(row + c);
#pragma unroll
    for (int i = 0; i < W / 2; ++i) v[2 * i] = Elem<TYPE>::lo(q[i]), v[2 * i + 1] = Elem<TYPE>::hi(q[i]);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = c + i < n ? Elem<TYPE>::to_f(row[c + i]) : 0.0f;
  }
}
template <int TYPE, int W>
MOE_DEV void store_n(uint16_t* row, int c, int n, bool vec, const float (&v)[W]) {
  uint32_t q[W / 2];
#pragma unroll
  for (int i = 0; i < W / 2; ++i) q[i] = Elem<TYPE>::pack(v[2 * i], v[2 * i + 1]);
  if (W == 4 && vec) {
    *reinterpret_cast<uint2*>(row + c) = make_uint2(q[0], q[1]);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (c + i < n) row[c + i] = (uint16_t)(i & 1 ? q[i >> 1] >> 16 : q[i >> 1] & 0xffffu);
  }
}

// The epilogues on columns [c, c + W) of token m (c < n). d: the sums; in the gated form the
// gate's, with u the up projection's.
template <int EPI, int TYPE, int W>
MOE_DEV void epilogue_n(const DenseEpi& e, int64_t m, int c, int n, bool vec, float (&d)[W], const float (&u)[W]) {
  const int64_t off = m * e.ldo;
  if constexpr (EPI == kEpiPlain) {
    if (e.residual) {
      float r[W];
      load_n<TYPE, W>(e.residual + off, c, n, vec, r);
#pragma unroll
      for (int i = 0; i < W; ++i) d[i] += r[i];
    }
    store_n<TYPE, W>(e.out + off, c, n, vec, d);
  } else if constexpr (EPI == kEpiGated) {
    // g and u stay in fp32 up to h, which is rounded once (the down projection's operand)
    if (e.gate) {
      store_n<TYPE, W>(e.gate + off, c, n, vec, d);
      store_n<TYPE, W>(e.up + off, c, n, vec, u);
    }
#pragma unroll
    for (int i = 0; i < W; ++i) d[i] = act_val(d[i], e.act) * u[i];
    store_n<TYPE, W>(e.out + off, c, n, vec, d);
  } else {
    // d = dh: dup = dh act(g), dgate = dh u act'(g), each rounded once
    float g[W], up[W];
    load_n<TYPE, W>(e.gate + off, c, n, vec, g);
    load_n<TYPE, W>(e.up + off, c, n, vec, up);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      float val, grad;
      act_grad(g[i], e.act, val, grad);
      const float dh = d[i];
      g[i] = dh * up[i] * grad;
      up[i] = dh * val;
    }
    store_n<TYPE, W>(e.dgate + off, c, n, vec, g);
    store_n<TYPE, W>(e.dup + off, c, n, vec, up);
  }
}

// ---- a warp's 32 rows x 16 columns through its staging buffer. 16-byte piece j of row r lies
// at piece j ^ ((r >> 2) & 1): conflict-free both by row (one lane each) and by two lanes of
// a row. cols: valid columns (a multiple of 8), rows: valid rows.
MOE_DEV uint32_t stage_off(int r, int j) { return (uint32_t)(r * 32 + ((j ^ ((r >> 2) & 1)) << 4)); }
MOE_DEV void sts16(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};\n" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
MOE_DEV uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
// into a whole register, so that nothing has to wait for the value before its use
MOE_DEV uint32_t ldg_u16(const uint16_t* p) {
  uint32_t v;
  asm volatile("ld.global.nc.u16 %0, [%1];\n" : "=r"(v) : "l"(p));
  return v;
}
MOE_DEV uint32_t ldg_u32(const uint16_t* p) {
  uint32_t v;
  asm volatile("ld.global.nc.u32 %0, [%1];\n" : "=r"(v) : "l"(p));
  return v;
}
MOE_DEV float4 lds_cluster(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}
template <int TYPE>
MOE_DEV void store_tile(uint32_t stage, const float (&v)[16], uint16_t* base, int64_t ld, int rows, int cols, int lane) {
#pragma unroll
  for (int j = 0; j < 2; ++j)
    sts16(stage + stage_off(lane, j),
          make_uint4(Elem<TYPE>::pack(v[8 * j], v[8 * j + 1]), Elem<TYPE>::pack(v[8 * j + 2], v[8 * j + 3]),
                     Elem<TYPE>::pack(v[8 * j + 4], v[8 * j + 5]), Elem<TYPE>::pack(v[8 * j + 6], v[8 * j + 7])));
  __syncwarp();
  const int j = lane & 1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 16 * i + (lane >> 1);
    const uint4 q = lds16(stage + stage_off(r, j));
    if (r < rows && 8 * j < cols) *reinterpret_cast<uint4*>(base + (int64_t)r * ld + 8 * j) = q;
  }
  __syncwarp();
}
struct TileRegs {
  uint4 q[2];
};
MOE_DEV void fetch_tile(TileRegs& t, const uint16_t* base, int64_t ld, int rows, int cols, int lane) {
  const int j = lane & 1;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 16 * i + (lane >> 1);
    t.q[i] = r < rows && 8 * j < cols ? *reinterpret_cast<const uint4*>(base + (int64_t)r * ld + 8 * j)
                                      : make_uint4(0, 0, 0, 0);
  }
}
// The fetched tile, turned: this lane's row.
template <int TYPE>
MOE_DEV void turn_tile(uint32_t stage, const TileRegs& t, float (&v)[16], int lane) {
#pragma unroll
  for (int i = 0; i < 2; ++i) sts16(stage + stage_off(16 * i + (lane >> 1), lane & 1), t.q[i]);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint4 q = lds16(stage + stage_off(lane, j));
    v[8 * j] = Elem<TYPE>::lo(q.x), v[8 * j + 1] = Elem<TYPE>::hi(q.x);
    v[8 * j + 2] = Elem<TYPE>::lo(q.y), v[8 * j + 3] = Elem<TYPE>::hi(q.y);
    v[8 * j + 4] = Elem<TYPE>::lo(q.z), v[8 * j + 5] = Elem<TYPE>::hi(q.z);
    v[8 * j + 6] = Elem<TYPE>::lo(q.w), v[8 * j + 7] = Elem<TYPE>::hi(q.w);
  }
  __syncwarp();
}

MOE_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

// CG: CTAs per tile; ROWS_K: the weights' rows are the summed index; SPLIT: a cluster per tile
template <int CG, int EPI, int TYPE, bool ROWS_K, bool SPLIT, bool PACKED>
__global__ void __launch_bounds__(Cfg<PACKED>::kThreads, 1) gemm_kernel(const __grid_constant__ GemmParams p) {
  using C = Cfg<PACKED>;
  constexpr int kStages = C::kStages, kSlots = C::kSlots, kGroups = C::kGroups, kEpiWarps = C::kEpiWarps;
  constexpr int kDeqWarp = C::kDeqWarp, kTmaWarp = C::kTmaWarp, kMmaWarp = C::kMmaWarp, kPackWarp = C::kPackWarp;
  constexpr int kPackAt = C::kPackAt, kStagingAt = C::kStagingAt, kBarsAt = C::kBarsAt;
  static_assert(PACKED || (CG == 2 && !SPLIT), "the 16-bit form serves many tokens");
  extern __shared__ unsigned char smem_raw[];
  // the same offset in every CTA of a cluster: the base of dynamic shared memory is
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar_full = sbase + kBarsAt;
  const uint32_t bar_empty = bar_full + 8 * kStages;
  const uint32_t bar_accf = bar_empty + 8 * kStages;
  const uint32_t bar_acce = bar_accf + 16;
  const uint32_t bar_pfull = bar_acce + 16;
  const uint32_t bar_pempty = bar_pfull + 8 * kSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kBarsAt + 8 * C::kNumBars);
  __shared__ int gone;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t crank = 0;
  if constexpr (CG == 2 || SPLIT) asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(crank));
  const int rank = CG == 2 ? (int)(crank & 1) : 0;   // in the pair
  const int split = SPLIT ? (int)crank / CG : 0;
  const uint32_t leader = CG == 2 ? crank & ~1u : crank;
  const int ctas = SPLIT ? CG * p.splits : CG;       // CTAs of a tile
  const int first = blockIdx.x / ctas, stride = gridDim.x / ctas;
  constexpr int kHalves = 2 / CG;                    // of a tile's weight rows in this CTA
  const int k0 = split * p.spk, k1 = k0 + p.spk < p.ks ? k0 + p.spk : p.ks;

  if (tid == 0) {
    gone = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full + 8 * s, PACKED ? 1 + 4 * CG : 1);  // the leader's expect_tx for both CTAs' bytes, a group of each
      mbar_init(bar_empty + 8 * s, 1);          // one commit
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_accf + 8 * i, 1);
      mbar_init(bar_acce + 8 * i, CG * kEpiWarps);
    }
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(bar_pfull + 8 * i, 1);
      mbar_init(bar_pempty + 8 * i, 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == kMmaWarp) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(tmem_slot))
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(tmem_slot))
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
  }
  tc_before();
  __syncthreads();
  if constexpr (CG == 2 || SPLIT) cluster_sync();
  tc_after();
  const uint32_t tmem = *tmem_slot;
  // `early`: the launch before this one writes no weights, and let this one start only after
  // everything before it had completed (a later product of one call)
  const bool weights = PACKED && ((warp >= kDeqWarp && warp < kTmaWarp) || warp == kPackWarp);
  if (!(weights && p.early)) {
    pdl_wait();
    pdl_trigger();
  }

  auto tile_m = [&](int unit) { return unit % p.tiles_m; };
  auto tile_n = [&](int unit) { return unit / p.tiles_m; };
  // first weight row (column of D) of this CTA's half h of n tile nt
  auto half_row = [&](int nt, int h) {
    const int half = CG == 2 ? rank : h;
    return p.gated ? nt * p.hb : nt * 2 * p.hb + half * p.hb;
  };

  if (warp == kTmaWarp) {
    if (lane == 0) {
      int it = 0, s = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int unit = first; ok && unit < p.units; unit += stride) {
        const int m0 = (tile_m(unit) * CG + rank) * kBM;
        const int n = half_row(tile_n(unit), 0);
        int pr = k0 >= p.ks0 ? 1 : 0, x = (k0 - (pr ? p.ks0 : 0)) * kBK;
        for (int k = k0; k < k1; ++k, ++it) {
          if (k == p.ks0) pr = 1, x = 0;
          if (!mbar_wait(bar_empty + 8 * s, phase, &gone)) {
            gone = 1;
            atomicOr(&g_dense_status, 1);
            ok = false;
            break;
          }
          uint32_t bar = bar_full + 8 * s;
          if (rank == 0) mbar_expect_tx(bar, CG * (p.a_rows + (PACKED ? 0 : p.hb)) * 128);
          if constexpr (CG == 2) bar = map_rank(bar, leader);
          const uint32_t dst = sbase + s * kStageBytes;
          tma_2d<CG>(dst, &p.a[pr], x, m0, bar);
          if constexpr (!PACKED) {
            if constexpr (ROWS_K) {  // boxes of 64 rows x 64 columns
              tma_2d<CG>(dst + kATile, &p.w[pr], n, x, bar);
              if (p.hb == 128) tma_2d<CG>(dst + kATile + kBTile / 2, &p.w[pr], n + 64, x, bar);
            } else {                 // hb rows x 64 columns
              tma_2d<CG>(dst + kATile, &p.w[p.gated ? rank : pr], x, n, bar);
            }
          }
          x += kBK;
          if (++s == kStages) s = 0, phase ^= 1;
        }
      }
      // no copy may still be landing, and no MMA's arrival still be under way, when the CTA
      // leaves: the leader's full barriers count both CTAs' bytes, and the pair leaves together
      for (int i = it - kStages < 0 ? 0 : it - kStages; ok && i < it; ++i)
        if (!mbar_wait(bar_empty + 8 * (i % kStages), (i / kStages) & 1, &gone)) {
          gone = 1;
          atomicOr(&g_dense_status, 1);
          ok = false;
        }
      if (!ok && rank == 0)
        for (int i = it - kStages < 0 ? 0 : it - kStages; i < it; ++i) {
          int never = 0;
          if (!mbar_wait(bar_full + 8 * (i % kStages), (i / kStages) & 1, &never)) atomicOr(&g_dense_status, 2);
        }
    }
  } else if (PACKED && warp == kPackWarp) {
    if constexpr (PACKED) {
      if (lane == 0) {
        int it = 0;
        bool ok = true;
        for (int unit = first; ok && unit < p.units; unit += stride) {
          const int nt = tile_n(unit);
          for (int k = k0; k < k1; ++k, ++it) {
            const int s = it % kSlots;
            if (!mbar_wait(bar_pempty + 8 * s, ((it / kSlots) & 1) ^ 1, &gone)) {
              gone = 1;
              atomicOr(&g_dense_status, 32);
              ok = false;
              break;
            }
            const uint32_t bar = bar_pfull + 8 * s;
            mbar_expect_tx(bar, kHalves * p.hb * 32);
            const int pr = k >= p.ks0 ? 1 : 0;
            const int kk = k - (pr ? p.ks0 : 0);
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
              const uint32_t dst = sbase + kPackAt + s * kPackBytes + h * p.hb * 32;
              const int n = half_row(nt, h);
              if constexpr (ROWS_K) {  // boxes of 64 rows x 64 columns
                tma_2d<1>(dst, &p.w[pr], n / 8, kk * kBK, bar);
                if (CG == 2 && p.hb == 128) tma_2d<1>(dst + 2048, &p.w[pr], n / 8 + 8, kk * kBK, bar);
              } else {                 // hb rows x 64 columns
                tma_2d<1>(dst, &p.w[p.gated ? (CG == 2 ? rank : h) : pr], kk * 8, n, bar);
              }
            }
          }
        }
        // no copy may still be landing when the CTA leaves
        for (int i = it - kSlots < 0 ? 0 : it - kSlots; i < it; ++i) {
          int never = 0;
          if (!mbar_wait(bar_pfull + 8 * (i % kSlots), (i / kSlots) & 1, &never)) atomicOr(&g_dense_status, 64);
        }
      }
    }
  } else if (PACKED && warp >= kDeqWarp && warp < kTmaWarp) {
    if constexpr (PACKED) {
      // ---- dequantisation: group wg takes steps wg, wg + kGroups, ... of this CTA's sequence
      const int wg = (warp - kDeqWarp) >> 2, wt = tid - (kDeqWarp + 4 * wg) * 32;
      // A thread owns one row of 64 weights of the tile (128 bytes of it, eight words packed):
      // row wt of this CTA's weight rows (both halves when CG = 1); with ROWS_K row wt % 64 of
      // the step, in the block wt / 64 of 64 columns. Two groups of weights at group size 32.
      const int per = k1 - k0;
      const int total = first < p.units ? (int)((p.units - first + stride - 1) / stride) * per : 0;
      const bool mine = wt < kHalves * p.hb;
      const int half = CG == 1 && wt >= p.hb ? 1 : 0;
      const bool two = p.lg == 5;
      // Both scales of a row and step in one load where every row starts at an even one (a step
      // starts at an even group): a load of 32 rows is 32 lines, whatever its width, and lengthens
      // the chain of a group's step (1000 tokens, 2048 -> 7168 at group 32: 39.7 us with two).
      // `upper` takes the second scale from where it is: the same word, the next, or the first's.
      const bool pair = two && (p.s_pitch & 1) == 0;
      const uint32_t upper = pair ? 0x3232 : two ? 0x5454 : 0x1010;
      // The scales and biases of the group's next two steps, read ahead: at_k walks the steps,
      // the pointers are those of its tile and operand pair.
      const uint16_t* ps = nullptr;
      const uint16_t* pb = nullptr;
      bool valid = false, second = false;
      int at_unit = first, at_k = k0 + wg, at_key = -1;
      while (at_k >= k1) at_k -= per, at_unit += stride;
      auto read_scales = [&](uint32_t (&vs)[2], uint32_t (&vb)[2]) {
        vs[0] = vs[1] = vb[0] = vb[1] = 0u;
        if (at_unit < p.units) {
          const int pr = at_k >= p.ks0 ? 1 : 0;
          if (at_key != 2 * at_unit + pr) {
            at_key = 2 * at_unit + pr;
            const int n = half_row(tile_n(at_unit), half) + (ROWS_K ? (CG == 2 ? wt & 64 : 0) : wt - half * p.hb);
            const WeightSide& q = p.q[p.gated ? (CG == 2 ? rank : half) : pr];
            valid = mine && n < p.N;
            second = valid && two && (!ROWS_K || n + 32 < p.N);
            const int64_t off = !valid ? 0 : ROWS_K ? (int64_t)(wt & 63) * p.s_pitch + (n >> p.lg) : (int64_t)n * p.s_pitch;
            ps = q.s + off;
            pb = q.b ? q.b + off : nullptr;
          }
          const int kk = at_k - (pr ? p.ks0 : 0);
          const int g = (kk * kBK) >> p.lg;
          const int64_t off = ROWS_K ? (int64_t)(kk * kBK) * p.s_pitch : g;
          const bool in = ROWS_K ? kk * kBK + (wt & 63) < p.rows : true;  // the first group of a step exists
          if (pair && second && in) {
            vs[0] = ldg_u32(ps + off);
            if (pb) vb[0] = ldg_u32(pb + off);
          } else if (valid && in) {
            vs[0] = ldg_u16(ps + off);
            if (pb) vb[0] = ldg_u16(pb + off);
          }
          if (!pair && second && in && (ROWS_K || g + 1 < p.s_pitch)) {
            vs[1] = ldg_u16(ps + off + 1);
            if (pb) vb[1] = ldg_u16(pb + off + 1);
          }
        }
        at_k += kGroups;
        while (at_k >= k1) at_k -= per, at_unit += stride;
      };
      uint32_t rs[2][2], rb[2][2];
      read_scales(rs[0], rb[0]);
      read_scales(rs[1], rb[1]);
      const uint32_t to = (uint32_t)wt * 128;
      bool ok = true;
      for (int it = wg; ok && it < total; it += 2 * kGroups) {
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {  // two steps per round: constant ring indexes
          const int step = it + kGroups * sub;
          if (step >= total) break;
          const int s = step % kStages, sl = step % kSlots;
          bool ready = mbar_wait(bar_pfull + 8 * sl, (step / kSlots) & 1, &gone);
          uint4 q0, q1;
          if (__all_sync(0xffffffffu, ready)) {
            const uint32_t src = sbase + kPackAt + sl * kPackBytes + wt * 32;
            q0 = lds16(src), q1 = lds16(src + 16);
            ready = mbar_wait(bar_empty + 8 * s, ((step / kStages) & 1) ^ 1, &gone);
          }
          if (!__all_sync(0xffffffffu, ready)) {
            gone = 1;
            if (lane == 0) atomicOr(&g_dense_status, 128);
            ok = false;
            break;
          }
          if (mine) {
            const uint32_t row = sbase + s * kStageBytes + kATile + to;
            const uint32_t s2 = __byte_perm(rs[sub][0], 0, 0x1010), b2 = __byte_perm(rb[sub][0], 0, 0x1010);
            const uint32_t* w = &q0.x;
#pragma unroll
            for (int c = 0; c < 4; ++c) sts16(row + (((uint32_t)c ^ (wt & 7)) << 4), dequant8<TYPE>(w[c], s2, b2));
            const uint32_t s3 = __byte_perm(rs[sub][0], rs[sub][1], upper), b3 = __byte_perm(rb[sub][0], rb[sub][1], upper);
            const uint32_t* v = &q1.x;
#pragma unroll
            for (int c = 0; c < 4; ++c) sts16(row + (((uint32_t)(4 + c) ^ (wt & 7)) << 4), dequant8<TYPE>(v[c], s3, b3));
          }
          fence_proxy();
          __syncwarp();
          // the packed words are in use by now: only here may their slot be filled again
          if (lane == 0) {
            mbar_arrive(bar_pempty + 8 * sl);
            mbar_arrive_cluster(CG == 2 ? map_rank(bar_full + 8 * s, leader) : bar_full + 8 * s);
          }
          read_scales(rs[sub], rb[sub]);
        }
      }
    }
  } else if (warp == kMmaWarp) {
    // The whole warp walks the steps, so that descriptors and addresses stay in uniform
    // registers; one elected lane issues. The next stage's barrier is asked about before this
    // stage's MMAs are issued: an answer takes about as long as two of them.
    if (rank == 0) {
      const uint32_t one = elect_one();
      const uint32_t idesc = (1u << 4) | (TYPE == kBf16 ? (1u << 7) | (1u << 10) : 0u) | (ROWS_K ? 1u << 16 : 0u) |
                             ((uint32_t)(2 * p.hb >> 3) << 17) | ((uint32_t)(CG * kBM >> 4) << 24);
      const uint32_t both = 3u << leader;
      const uint64_t ad0 = sw128_desc(sbase);
      const uint64_t bd0 = ROWS_K ? sw128_mn_desc(sbase + kATile) : sw128_desc(sbase + kATile);
      constexpr int kBStep = ROWS_K ? (16 * 128) >> 4 : 32 >> 4;  // 16 rows, or 32 bytes of each row
      int s = 0, tile = 0;
      uint32_t phase = 0;
      bool ok = true;
      bool ready = mbar_test(bar_full, 0);
      for (int unit = first; ok && unit < p.units; unit += stride, ++tile) {
        const int buf = tile & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(bar_acce + 8 * buf, ((tile >> 1) & 1) ^ 1, &gone))) {
          gone = 1;
          if (lane == 0) atomicOr(&g_dense_status, 4);
          break;
        }
        tc_after();
        for (int k = k0; k < k1; ++k) {
          if (!ready) ready = mbar_wait(bar_full + 8 * s, phase, &gone);
          if (!__all_sync(0xffffffffu, ready)) {
            gone = 1;
            if (lane == 0) atomicOr(&g_dense_status, 8);
            ok = false;
            break;
          }
          tc_after();
          const int next = s + 1 == kStages ? 0 : s + 1;
          const uint32_t next_phase = next ? phase : phase ^ 1;
          ready = mbar_test(bar_full + 8 * next, next_phase);
          const uint32_t at = (uint32_t)(s * kStageBytes) >> 4;
          if (one) {
#pragma unroll
            for (int j = 0; j < kBK / 16; ++j)
              tc_mma<CG>(tmem + buf * 256, ad0 + at + 2 * j, bd0 + at + kBStep * j, idesc, (k > k0 || j > 0) ? 1u : 0u);
            tc_commit<CG>(bar_empty + 8 * s, both);
            if (k == k1 - 1) tc_commit<CG>(bar_accf + 8 * buf, both);
          }
          __syncwarp();
          s = next;
          phase = next_phase;
        }
      }
    }
  } else {
    // ---- epilogue warps
    const int quad = warp & 3;
    constexpr int kChunkStep = kEpiWarps / 4;  // warps that share a lane quadrant take chunks in turn
    const bool vec = ((p.N | p.e.ldo) & 7) == 0;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t stage = sbase + kStagingAt + warp * kStageBuf;
    const int chunks = (EPI == kEpiGated ? p.hb : 2 * p.hb) / 16;  // of 16 output columns
    // chunks of gate / up (residual) fetched ahead: the first ones before the accumulator is ready
    constexpr int kAhead = PACKED ? 1 : 2;
    int tile = 0;
    for (int unit = first; unit < p.units; unit += stride, ++tile) {
      const int nt = tile_n(unit);
      const int buf = tile & 1;
      const uint32_t acc = tmem + buf * 256 + lanes;
      const int64_t mrow = (int64_t)(tile_m(unit) * CG + rank) * kBM + quad * 32;  // the warp's first row
      const int rows = p.M - mrow < 32 ? (int)(p.M - mrow) : 32;  // may be <= 0
      const int64_t ld = p.e.ldo;
      const int n0 = EPI == kEpiGated ? nt * p.hb : nt * 2 * p.hb;
      TileRegs tg[kAhead], tu[kAhead];
      auto fetch = [&](int q, int slot) {
        if (q >= chunks) return;
        const int n = n0 + 16 * q;
        const int64_t at = mrow * ld + n;
        if constexpr (EPI == kEpiGatedBackward) {
          fetch_tile(tg[slot], p.e.gate + at, ld, rows, p.N - n, lane);
          fetch_tile(tu[slot], p.e.up + at, ld, rows, p.N - n, lane);
        } else if constexpr (EPI == kEpiPlain) {
          if (p.e.residual) fetch_tile(tg[slot], p.e.residual + at, ld, rows, p.N - n, lane);
        }
      };
      if (!SPLIT && vec) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) fetch((warp >> 2) + i * kChunkStep, i);
      }
      const bool ready = mbar_wait(bar_accf + 8 * buf, (tile >> 1) & 1, &gone);
      if (!__all_sync(0xffffffffu, ready)) {
        gone = 1;
        if (lane == 0) atomicOr(&g_dense_status, 16);
        break;
      }
      tc_after();
      if constexpr (SPLIT) {
        // the sums into this CTA's shared memory (stages and slots are free: every MMA has completed,
        // and with them the last use of a slot)
        for (int q = warp >> 2; q < 2 * p.hb / 16; q += kChunkStep) {
          float d[16];
          tmem_ld16(acc + 16 * q, d);
          tmem_wait_ld();
          const uint32_t dst = sbase + (uint32_t)((quad * 32 + lane) * kSumPitch + 16 * q) * 4;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sts16(dst + 16 * i, make_uint4(__float_as_uint(d[4 * i]), __float_as_uint(d[4 * i + 1]),
                                           __float_as_uint(d[4 * i + 2]), __float_as_uint(d[4 * i + 3])));
        }
      } else {
#pragma unroll 1
        for (int q0 = warp >> 2; q0 < chunks; q0 += kAhead * kChunkStep) {
#pragma unroll
          for (int slot = 0; slot < kAhead; ++slot) {
            const int q = q0 + slot * kChunkStep;
            if (q >= chunks) break;
            const int n = n0 + 16 * q;
            float d[16], u[16];
            tmem_ld16(acc + 16 * q, d);
            if constexpr (EPI == kEpiGated) tmem_ld16(acc + p.hb + 16 * q, u);
            tmem_wait_ld();
            if (!vec) {  // rows of any length: element by element
              if (lane < rows) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  float(&d8)[8] = *reinterpret_cast<float(*)[8]>(d + 8 * i);
                  const float(&u8)[8] = *reinterpret_cast<float(*)[8]>((EPI == kEpiGated ? u : d) + 8 * i);
                  if (n + 8 * i < p.N) epilogue_n<EPI, TYPE, 8>(p.e, mrow + lane, n + 8 * i, p.N, false, d8, u8);
                }
              }
              continue;
            }
            const int64_t at = mrow * ld + n;
            const int cols = p.N - n;
            if constexpr (EPI == kEpiPlain) {
              if (p.e.residual) {
                turn_tile<TYPE>(stage, tg[slot], u, lane);
                fetch(q + kAhead * kChunkStep, slot);
#pragma unroll
                for (int i = 0; i < 16; ++i) d[i] += u[i];
              }
              store_tile<TYPE>(stage, d, p.e.out + at, ld, rows, cols, lane);
            } else if constexpr (EPI == kEpiGated) {
              // g and u stay in fp32 up to h, which is rounded once
              if (p.e.gate) {
                store_tile<TYPE>(stage, d, p.e.gate + at, ld, rows, cols, lane);
                store_tile<TYPE>(stage, u, p.e.up + at, ld, rows, cols, lane);
              }
#pragma unroll
              for (int i = 0; i < 16; ++i) d[i] = act_val(d[i], p.e.act) * u[i];
              store_tile<TYPE>(stage, d, p.e.out + at, ld, rows, cols, lane);
            } else {
              float g[16];
              turn_tile<TYPE>(stage, tg[slot], g, lane);
              turn_tile<TYPE>(stage, tu[slot], u, lane);
              fetch(q + kAhead * kChunkStep, slot);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                float val, grad;
                act_grad(g[i], p.e.act, val, grad);
                g[i] = d[i] * u[i] * grad;
                d[i] *= val;
              }
              store_tile<TYPE>(stage, g, p.e.dgate + at, ld, rows, cols, lane);
              store_tile<TYPE>(stage, d, p.e.dup + at, ld, rows, cols, lane);
            }
          }
        }
      }
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(CG == 2 ? map_rank(bar_acce + 8 * buf, leader) : bar_acce + 8 * buf);
    }
  }
  __syncwarp();
  if constexpr (SPLIT) {
    // ---- every CTA's sums lie in its shared memory: this one adds its slice of the rows
    cluster_sync();
    {
      const int slice = (kBM + p.splits - 1) / p.splits, r0 = split * slice;
      const int r1 = r0 + slice < kBM ? r0 + slice : kBM;
      const int nt = tile_n(first);
      const int n0 = EPI == kEpiGated ? nt * p.hb : nt * 2 * p.hb;
      // four columns per thread: a warp's reads from another CTA cover whole 128-byte lines
      // (eight columns in two reads with gaps took three times as long)
      const int groups = (EPI == kEpiGated ? p.hb : 2 * p.hb) / 4;
      const bool vec = ((p.N | p.e.ldo) & 7) == 0;
      for (int i = tid; i < (r1 - r0) * groups; i += C::kThreads) {
        const int r = r0 + i / groups, c = (i % groups) * 4;
        const int64_t m = (int64_t)(tile_m(first) * CG + rank) * kBM + r;
        if (m >= p.M || n0 + c >= p.N) continue;
        float d[4] = {}, u[4] = {};
        const uint32_t mine = sbase + (uint32_t)(r * kSumPitch + c) * 4;
        for (int sp = 0; sp < p.splits; sp += 4) {  // four splits' pieces in flight
          float4 v[4], w[4];
#pragma unroll
          for (int s = 0; s < 4; ++s)
            if (sp + s < p.splits) {
              const uint32_t src = map_rank(mine, (uint32_t)((sp + s) * CG + rank));
              v[s] = lds_cluster(src);
              if constexpr (EPI == kEpiGated) w[s] = lds_cluster(src + p.hb * 4);
            }
#pragma unroll
          for (int s = 0; s < 4; ++s)
            if (sp + s < p.splits) {
              d[0] += v[s].x, d[1] += v[s].y, d[2] += v[s].z, d[3] += v[s].w;
              if constexpr (EPI == kEpiGated) u[0] += w[s].x, u[1] += w[s].y, u[2] += w[s].z, u[3] += w[s].w;
            }
        }
        epilogue_n<EPI, TYPE, 4>(p.e, m, n0 + c, p.N, vec, d, u);
      }
    }
    __syncwarp();
  }
  tc_before();
  __syncthreads();
  // the peers' MMAs and sums read this CTA's shared memory and arrive on its barriers
  if constexpr (CG == 2 || SPLIT) cluster_sync();
  if (warp == kMmaWarp) {
    tc_after();
    if constexpr (CG == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
  }
}

__global__ void clear_status_kernel(int32_t reported) { atomicAnd(&g_dense_status, ~reported); }

__global__ void expire_wait_kernel(uint64_t limit_ns) {
  __shared__ __align__(8) uint64_t bar;
  int gone = 0;
  mbar_init(smem_u32(&bar), 1);
  if (!mbar_wait(smem_u32(&bar), 0, &gone, limit_ns)) atomicOr(&g_dense_status, kExpiredWait);
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return (PFN_cuTensorMapEncodeTiled_v12000) nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

cudaError_t encode(CUtensorMap* map, CUtensorMapDataType type, const void* ptr, int64_t rows, int64_t cols,
                   int64_t pitch_bytes, int box_cols, int box_rows, CUtensorMapSwizzle swizzle) {
  auto enc = encoder();
  if (!enc) return cudaErrorNotSupported;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)pitch_bytes};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  const cuuint32_t one[2] = {1, 1};
  const CUresult r = enc(map, type, 2, const_cast<void*>(ptr), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// Clusters of n CTAs of the kernel that the device holds at once: the SMs of a GPC beyond a
// multiple of n stay empty. Asked once per device and size.
int resident_clusters(int n) {
  if (n == 1) return kSms;
  static std::atomic<int> known[64][9];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return kSms / n;
  int got = known[dev][n].load(std::memory_order_relaxed);
  if (got) return got;
  auto kern = gemm_kernel<2, kEpiPlain, kBf16, false, true, true>;  // every form has the same shape
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n * kSms);
  cfg.blockDim = dim3(Cfg<true>::kThreads);
  cfg.dynamicSmemBytes = Cfg<true>::kSmem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = n;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<true>::kSmem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&got, kern, &cfg) != cudaSuccess || got < 1) {
    (void)cudaGetLastError();
    got = kSms / n;
  }
  known[dev][n].store(got, std::memory_order_relaxed);
  return got;
}

struct Plan {
  int cg, hb, tiles_m, tiles_n, splits, ks0, ks, spk;
};

// Tile width and K split of a product: the pair that takes the least time over the rounds of
// tiles, by a line fitted to every allowed pair of 16 products (64 to 800 tokens, 768 to 5632
// summed, both directions). With r weight rows per CTA a K step costs 0.11 + 0.21 r / 64 us, a
// round 4.5 us (its start and epilogue), the exchange of a split's sums 1 + 1.4 r / 64 us. The
// line was fitted before the last steps of the kernel; with it as it is the pair taken is 1.3 %
// (group 32) and 1.9 % (128) behind the fastest measured one in the mean of those 16, 11 % at
// worst (512 tokens, 5632 -> 2048, rows summed, group 128: 21.3 us, 19.1 with 128 x 3 splits), and
// 1.4 % and 10 % (group 32) for 16 others that had no part in the fit (40 to 1500 tokens). A new
// fit and a search over the five constants found none better. Over 16-bit weights a step takes
// 0.36 us at 128 rows and no less than 0.2.
Plan plan(int64_t M, int N, int K, int pairs, bool gated, bool rows_k, bool wide) {
  Plan best{};
  double least = 0;
  const int cg = M > kBM ? 2 : 1;
  const int tiles_m = (int)((M + cg * kBM - 1) / (cg * kBM));
  const int ks0 = (K + kBK - 1) / kBK, ks = ks0 * pairs;
  // a CTA holds at most 128 weight rows: a half over a pair, both halves alone
  for (int hb = cg == 2 ? 128 : 64; hb >= (cg == 2 || rows_k ? 64 : 32); hb -= rows_k ? 64 : 32) {
    const int tiles_n = gated ? (N + hb - 1) / hb : (N + 2 * hb - 1) / (2 * hb);
    for (int sp = 1; sp * cg <= (wide ? cg : 8); ++sp) {
      const int spk = (ks + sp - 1) / sp;
      if ((ks + spk - 1) / spk != sp) continue;  // no empty split
      const int64_t slots = resident_clusters(cg * sp);
      const double rounds = (double)(((int64_t)tiles_m * tiles_n + slots - 1) / slots);
      const double r = (cg == 2 ? hb : 2 * hb) / 64.0;
      const double t = wide ? rounds * (spk * std::max(0.2, 0.18 * r) + 2.0)
                            : rounds * (spk * (0.11 + 0.21 * r) + 4.5 + (sp > 1 ? 1.0 + 1.4 * r : 0.0));
      if (best.cg == 0 || t < least * 0.98) {
        least = t;
        best = Plan{cg, hb, tiles_m, tiles_n, sp, ks0, ks, spk};
      }
    }
  }
  return best;
}

template <int CG, int EPI, int TYPE, bool ROWS_K, bool SPLIT, bool PACKED>
cudaError_t launch_t(const GemmParams& p, cudaStream_t st) {
  using C = Cfg<PACKED>;
  auto kern = gemm_kernel<CG, EPI, TYPE, ROWS_K, SPLIT, PACKED>;
  static std::atomic<uint64_t> done{0};
  cudaError_t err = allow_smem(kern, C::kSmem, done);
  if (err != cudaSuccess) return err;
  const int ctas = SPLIT ? CG * p.splits : CG;
  const int most = SPLIT ? p.units : kSms / CG;  // a split tile has its cluster to itself
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.units < most ? p.units : most) * ctas));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (ctas > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = ctas;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <int CG, int EPI, int TYPE, bool ROWS_K>
cudaError_t launch_s(const GemmParams& p, cudaStream_t st) {
  if constexpr (CG == 2)
    if (p.wide) return launch_t<CG, EPI, TYPE, ROWS_K, false, false>(p, st);
  return p.splits > 1 ? launch_t<CG, EPI, TYPE, ROWS_K, true, true>(p, st)
                      : launch_t<CG, EPI, TYPE, ROWS_K, false, true>(p, st);
}
template <int CG, int TYPE>
cudaError_t launch_e(const GemmParams& p, int epi, bool rows_k, cudaStream_t st) {
  if (epi == kEpiGated) return launch_s<CG, kEpiGated, TYPE, false>(p, st);
  if (epi == kEpiGatedBackward) return launch_s<CG, kEpiGatedBackward, TYPE, true>(p, st);
  return rows_k ? launch_s<CG, kEpiPlain, TYPE, true>(p, st) : launch_s<CG, kEpiPlain, TYPE, false>(p, st);
}

}  // namespace

cudaError_t launch_dense_gemm(const DenseGemm& g, cudaStream_t st) {
  const bool gated = g.epilogue == kEpiGated, wide = g.wide[0] != nullptr;
  if (wide && g.M <= kBM) return cudaErrorInvalidValue;
  if (g.rows_k ? gated : g.epilogue == kEpiGatedBackward) return cudaErrorInvalidValue;
  const Plan q = plan(g.M, g.N, g.K, g.pairs, gated, g.rows_k, wide);
  GemmParams p;
  p.M = g.M;
  p.N = g.N;
  p.rows = g.rows_k ? g.K : g.N;
  const int cols = g.rows_k ? g.N : g.K;
  p.s_pitch = cols / g.group;
  p.lg = g.group == 32 ? 5 : g.group == 64 ? 6 : 7;
  p.gated = gated;
  p.hb = q.hb;
  p.ks0 = q.ks0;
  p.ks = q.ks;
  p.tiles_m = q.tiles_m;
  p.splits = q.splits;
  p.spk = q.spk;
  if ((int64_t)q.tiles_m * q.tiles_n * 8 > INT32_MAX / 2) return cudaErrorInvalidValue;
  p.units = q.tiles_m * q.tiles_n;
  // The rows of a short tile behind its box keep what the stage held: they only reach
  // accumulator rows that are not stored.
  p.a_rows = (int)std::min<int64_t>(kBM, (g.M + 7) / 8 * 8);
  p.wide = wide;
  p.early = g.early;
  p.e = g.e;
  const auto t16 = g.type == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  for (int i = 0; i < 2; ++i) {
    const int ai = g.pairs > 1 ? i : 0, wi = (g.pairs > 1 || gated) ? i : 0;
    cudaError_t err = cudaSuccess;
    if (i == 0 || ai) err = encode(&p.a[i], t16, g.a[ai], g.M, g.K, g.lda * 2, kBK, p.a_rows, CU_TENSOR_MAP_SWIZZLE_128B);
    if (err == cudaSuccess && (i == 0 || wi))
      err = wide ? encode(&p.w[i], t16, g.wide[wi], p.rows, cols, (int64_t)cols * 2, kBK, g.rows_k ? kBK : q.hb,
                          CU_TENSOR_MAP_SWIZZLE_128B)
                 : encode(&p.w[i], CU_TENSOR_MAP_DATA_TYPE_UINT32, g.w[wi].w, p.rows, cols / 8, (int64_t)cols / 2, 8,
                          g.rows_k ? kBK : q.hb, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (err != cudaSuccess) return err;
    if (i && !ai) p.a[1] = p.a[0];
    if (i && !wi) p.w[1] = p.w[0];
    p.q[i] = {g.w[wi].s, g.w[wi].b};
  }
  if (g.type == kF16) return q.cg == 2 ? launch_e<2, kF16>(p, g.epilogue, g.rows_k, st) : launch_e<1, kF16>(p, g.epilogue, g.rows_k, st);
  return q.cg == 2 ? launch_e<2, kBf16>(p, g.epilogue, g.rows_k, st) : launch_e<1, kBf16>(p, g.epilogue, g.rows_k, st);
}

cudaError_t dense_gemm_status(int32_t* status, cudaStream_t st) {
  cudaError_t err = cudaMemcpyFromSymbolAsync(status, g_dense_status, sizeof(int32_t), 0, cudaMemcpyDeviceToHost, st);
  if (err == cudaSuccess) err = cudaStreamSynchronize(st);
  if (err != cudaSuccess || *status == 0) return err;
  clear_status_kernel<<<1, 1, 0, st>>>(*status);
  err = cudaGetLastError();
  return err != cudaSuccess ? err : cudaStreamSynchronize(st);
}

cudaError_t launch_expire_wait(uint64_t limit_ns, cudaStream_t st) {
  expire_wait_kernel<<<1, 1, 0, st>>>(limit_ns);
  return cudaGetLastError();
}

}  // namespace moe
