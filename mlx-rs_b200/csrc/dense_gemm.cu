// dense_gemm.cu — 16-bit matrix products on tcgen05 with the feed-forward block's epilogues.
//
// D[m, n] = sum_p A_p[m, :] . B_p[n, :]^T with fp32 accumulators in tensor memory. Tokens are
// the MMA's rows (an epilogue thread owns one token and walks its columns), weight rows its
// columns. Persistent CTAs (CG = 1) or CTA pairs (CG = 2): 128 tokens per CTA x 256 weight
// rows per tile, K in steps of 64 elements (one 128-byte swizzled row per operand row).
//   warp 8    one lane streams both operands with TMA into a ring of mbarrier stages;
//   warp 9    allocates all 512 tensor-memory columns (two accumulators) and issues
//             tcgen05.mma from one lane: M = 128 (or 256 over the pair), N = 256, K = 16;
//   warps 0-7 read the finished accumulator back (warp w: TMEM lanes 32 (w % 4).., column
//             half w / 4) and apply the epilogue while the next tile accumulates in the
//             other buffer.
// In the pair form each CTA loads its own 128 tokens and half of the 256 weight rows, so a
// weight row crosses L2 -> SM once per 256 tokens; the leader (rank 0) owns the full and
// accumulator-empty barriers and issues the MMAs of both. In the gated form the first 128
// columns of a tile are gate rows and the second 128 the same rows of up, so that one thread
// holds g and u of the same element.
// K can be split over several CTAs when there are fewer tiles than SMs: fp32 partial sums,
// then one launch that adds them in split order and applies the epilogue (no atomics, the
// same bits on every run).
// B may lie with its N contiguous (BN_MAJOR: the weights' rows are the summed index, in the
// backward pass): boxes of 64 columns x 64 rows, read through the MN-major descriptor, so
// that both directions use the weights as they are stored.
// The epilogue moves global memory through a 2 KB buffer per warp: a thread owns a row of the
// accumulator, but a warp's accesses cover 64 contiguous bytes of eight rows each.
// Every wait is bounded (2 s): on expiry the CTA records a code in the device's status word,
// stops working and leaves through the same barriers as the rest of its pair.
#include <cudaTypedefs.h>

#include "dense.cuh"

namespace moe {

namespace {

constexpr int kBM = 128, kBN = 256, kBK = 64;
constexpr int kATile = kBM * kBK * 2;        // 16 KB
constexpr int kBHalf = 128 * kBK * 2;        // 16 KB: 128 weight rows
constexpr int kEpiWarps = 8;
constexpr int kTmaWarp = 8, kMmaWarp = 9;
constexpr int kThreads = 320;
constexpr int kStage2K = 2048;               // 32 rows x 32 columns of 16 bits
constexpr uint64_t kWaitLimitNs = 2000ull * 1000 * 1000;

__device__ int32_t g_dense_status;

template <int CG>
struct Cfg {
  static constexpr int kStages = CG == 2 ? 6 : 4;
  static constexpr int kStageBytes = kATile + (CG == 2 ? 1 : 2) * kBHalf;
  // full[S] empty[S] acc_full[2] acc_empty[2] | tmem base
  static constexpr int kStaging = kStages * kStageBytes;  // [epilogue warps][2 KB]
  static constexpr int kBars = kStaging + kEpiWarps * kStage2K;
  static constexpr int kSmem = kBars + 8 * (2 * kStages + 4) + 16 + 1024;
};

struct GemmParams {
  CUtensorMap a[2], b[2];
  int64_t M;
  int N;
  int gated;
  int ks0, ks;          // K steps of the first operand pair, of all
  int tiles_m, tiles_n, splits, spk;
  int64_t units;
  float* partial;       // [splits][M][tiles_n * kBN]
  DenseEpi e;
};

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
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(1000u)
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
MOE_DEV bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* gone) {
  if (mbar_try(bar, parity)) return true;
  const uint64_t t0 = now_ns();
  while (!mbar_try(bar, parity))
    if (*gone || now_ns() - t0 > kWaitLimitNs) return false;
  return true;
}
// The address of `a` in CTA `rank` of the cluster.
MOE_DEV uint32_t map_rank(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
MOE_DEV void mbar_arrive_cluster(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_bar) : "memory");
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
// Arrives on `bar` of every CTA of the group when the MMAs issued so far have completed.
template <int CG>
MOE_DEV void tc_commit(uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(
            bar),
        "h"((uint16_t)3)
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
MOE_DEV void tmem_ld32(uint32_t taddr, float (&r)[32]) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(taddr));
}
MOE_DEV void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }

// ---- eight consecutive elements of a 16-bit row, at column c of n (vec: rows are 16-byte
// aligned multiples of 8; otherwise element by element, columns beyond n left alone)
template <int TYPE>
MOE_DEV void load8(const uint16_t* row, int c, int n, bool vec, float (&v)[8]) {
  if (vec) {
    const uint4 q = *reinterpret_cast<const uint4*>(row + c);
    v[0] = Elem<TYPE>::lo(q.x), v[1] = Elem<TYPE>::hi(q.x), v[2] = Elem<TYPE>::lo(q.y), v[3] = Elem<TYPE>::hi(q.y);
    v[4] = Elem<TYPE>::lo(q.z), v[5] = Elem<TYPE>::hi(q.z), v[6] = Elem<TYPE>::lo(q.w), v[7] = Elem<TYPE>::hi(q.w);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < n ? Elem<TYPE>::to_f(row[c + i]) : 0.0f;
  }
}
template <int TYPE>
MOE_DEV void store8(uint16_t* row, int c, int n, bool vec, const float (&v)[8]) {
  uint32_t q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = Elem<TYPE>::pack(v[2 * i], v[2 * i + 1]);
  if (vec) {
    *reinterpret_cast<uint4*>(row + c) = make_uint4(q[0], q[1], q[2], q[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < n) row[c + i] = (uint16_t)(i & 1 ? q[i >> 1] >> 16 : q[i >> 1] & 0xffffu);
  }
}

// The epilogues on eight columns [c, c + 8) of token m (c < n). d: the sums; in the gated
// form the gate's, with u the up projection's.
template <int EPI, int TYPE>
MOE_DEV void epilogue8(const DenseEpi& e, int64_t m, int c, int n, bool vec, float (&d)[8], const float (&u)[8]) {
  const int64_t off = m * e.ldo;
  if constexpr (EPI == kEpiPlain) {
    if (e.residual) {
      float r[8];
      load8<TYPE>(e.residual + off, c, n, vec, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] += r[i];
    }
    store8<TYPE>(e.out + off, c, n, vec, d);
  } else if constexpr (EPI == kEpiGated) {
    // g and u stay in fp32 up to h, which is rounded once (the down projection's operand)
    if (e.gate) {
      store8<TYPE>(e.gate + off, c, n, vec, d);
      store8<TYPE>(e.up + off, c, n, vec, u);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = act_val(d[i], e.act) * u[i];
    store8<TYPE>(e.out + off, c, n, vec, d);
  } else {
    // d = dh: dup = dh act(g), dgate = dh u act'(g), each rounded once
    float g[8], up[8];
    load8<TYPE>(e.gate + off, c, n, vec, g);
    load8<TYPE>(e.up + off, c, n, vec, up);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float val, grad;
      act_grad(g[i], e.act, val, grad);
      const float dh = d[i];
      g[i] = dh * up[i] * grad;
      up[i] = dh * val;
    }
    store8<TYPE>(e.dgate + off, c, n, vec, g);
    store8<TYPE>(e.dup + off, c, n, vec, up);
  }
}

// ---- a warp's 32 rows x 32 columns through its staging buffer. 16-byte piece j of row r lies
// at piece j ^ ((r >> 1) & 3): conflict-free both by row (one lane each) and by four lanes
// of a row. cols: valid columns (a multiple of 8), rows: valid rows.
MOE_DEV uint32_t stage_off(int r, int j) { return (uint32_t)(r * 64 + ((j ^ ((r >> 1) & 3)) << 4)); }
MOE_DEV void sts16(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};\n" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
MOE_DEV uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
template <int TYPE>
MOE_DEV void store_tile(uint32_t stage, const float (&v)[32], uint16_t* base, int64_t ld, int rows, int cols, int lane) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    sts16(stage + stage_off(lane, j),
          make_uint4(Elem<TYPE>::pack(v[8 * j], v[8 * j + 1]), Elem<TYPE>::pack(v[8 * j + 2], v[8 * j + 3]),
                     Elem<TYPE>::pack(v[8 * j + 4], v[8 * j + 5]), Elem<TYPE>::pack(v[8 * j + 6], v[8 * j + 7])));
  __syncwarp();
  const int j = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 8 * i + (lane >> 2);
    const uint4 q = lds16(stage + stage_off(r, j));
    if (r < rows && 8 * j < cols) *reinterpret_cast<uint4*>(base + (int64_t)r * ld + 8 * j) = q;
  }
  __syncwarp();
}
struct Tile32 {
  uint4 q[4];
};
MOE_DEV void fetch_tile(Tile32& t, const uint16_t* base, int64_t ld, int rows, int cols, int lane) {
  const int j = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 8 * i + (lane >> 2);
    t.q[i] = r < rows && 8 * j < cols ? *reinterpret_cast<const uint4*>(base + (int64_t)r * ld + 8 * j)
                                      : make_uint4(0, 0, 0, 0);
  }
}
// The fetched tile, turned: this lane's row.
template <int TYPE>
MOE_DEV void turn_tile(uint32_t stage, const Tile32& t, float (&v)[32], int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i) sts16(stage + stage_off(8 * i + (lane >> 2), lane & 3), t.q[i]);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 q = lds16(stage + stage_off(lane, j));
    v[8 * j] = Elem<TYPE>::lo(q.x), v[8 * j + 1] = Elem<TYPE>::hi(q.x);
    v[8 * j + 2] = Elem<TYPE>::lo(q.y), v[8 * j + 3] = Elem<TYPE>::hi(q.y);
    v[8 * j + 4] = Elem<TYPE>::lo(q.z), v[8 * j + 5] = Elem<TYPE>::hi(q.z);
    v[8 * j + 6] = Elem<TYPE>::lo(q.w), v[8 * j + 7] = Elem<TYPE>::hi(q.w);
  }
  __syncwarp();
}

template <int CG, int EPI, int TYPE, bool BN_MAJOR>
__global__ void __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ GemmParams p) {
  using C = Cfg<CG>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar_full = sbase + C::kBars;
  const uint32_t bar_empty = bar_full + 8 * C::kStages;
  const uint32_t bar_accf = bar_empty + 8 * C::kStages;
  const uint32_t bar_acce = bar_accf + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kBars + 8 * (2 * C::kStages + 4));
  __shared__ int gone;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t rank = 0;
  if constexpr (CG == 2) asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(rank));
  const int64_t first = blockIdx.x / CG, stride = gridDim.x / CG;

  if (tid == 0) {
    gone = 0;
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(bar_full + 8 * s, 1);   // the leader's expect_tx
      mbar_init(bar_empty + 8 * s, 1);  // one commit
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_accf + 8 * i, 1);
      mbar_init(bar_acce + 8 * i, CG * kEpiWarps);
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
  if constexpr (CG == 2) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
  }
  tc_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  // unit -> (m tile, split, n tile), m fastest
  auto unit_of = [&](int64_t unit, int& mt, int& sp, int& nt) {
    mt = (int)(unit % p.tiles_m);
    const int64_t r = unit / p.tiles_m;
    sp = (int)(r % p.splits);
    nt = (int)(r / p.splits);
  };
  auto steps_of = [&](int sp, int& k0, int& k1) {
    k0 = sp * p.spk;
    k1 = k0 + p.spk < p.ks ? k0 + p.spk : p.ks;
  };

  if (warp == kTmaWarp) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int64_t unit = first; ok && unit < p.units; unit += stride) {
        int mt, sp, nt, k0, k1;
        unit_of(unit, mt, sp, nt);
        steps_of(sp, k0, k1);
        const int m0 = (mt * CG + (int)rank) * kBM;
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % C::kStages;
          if (!mbar_wait(bar_empty + 8 * s, ((it / C::kStages) & 1) ^ 1, &gone)) {
            gone = 1;
            atomicOr(&g_dense_status, 1);
            ok = false;
            break;
          }
          const uint32_t st = sbase + s * C::kStageBytes;
          uint32_t bar = bar_full + 8 * s;
          if (rank == 0) mbar_expect_tx(bar, CG * C::kStageBytes);
          if constexpr (CG == 2) bar = map_rank(bar, 0);
          const int pr = k >= p.ks0 ? 1 : 0;
          const int x = (k - (pr ? p.ks0 : 0)) * kBK;
          tma_2d<CG>(st, &p.a[pr], x, m0, bar);
#pragma unroll
          for (int h = 0; h < (CG == 2 ? 1 : 2); ++h) {
            const int half = CG == 2 ? (int)rank : h;
            if constexpr (BN_MAJOR) {
              const int n = nt * kBN + half * 128;
              tma_2d<CG>(st + kATile + h * kBHalf, &p.b[pr], n, x, bar);
              tma_2d<CG>(st + kATile + h * kBHalf + kBHalf / 2, &p.b[pr], n + 64, x, bar);
            } else {
              const CUtensorMap* bm = p.gated ? &p.b[half] : &p.b[pr];
              const int y = p.gated ? nt * 128 : nt * kBN + half * 128;
              tma_2d<CG>(st + kATile + h * kBHalf, bm, x, y, bar);
            }
          }
        }
      }
      // no copy may still be landing, and no MMA's arrival still be under way, when the CTA
      // leaves: the leader's full barriers count both CTAs' bytes, and the pair leaves together
      for (int i = it - C::kStages < 0 ? 0 : it - C::kStages; ok && i < it; ++i)
        if (!mbar_wait(bar_empty + 8 * (i % C::kStages), (i / C::kStages) & 1, &gone)) {
          gone = 1;
          atomicOr(&g_dense_status, 1);
          ok = false;
        }
      if (!ok && rank == 0)
        for (int i = it - C::kStages < 0 ? 0 : it - C::kStages; i < it; ++i) {
          int never = 0;
          if (!mbar_wait(bar_full + 8 * (i % C::kStages), (i / C::kStages) & 1, &never)) atomicOr(&g_dense_status, 2);
        }
    }
  } else if (warp == kMmaWarp) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = (1u << 4) | (TYPE == kBf16 ? (1u << 7) | (1u << 10) : 0u) | (BN_MAJOR ? 1u << 16 : 0u) |
                             ((uint32_t)(kBN >> 3) << 17) | ((uint32_t)(CG * kBM >> 4) << 24);
      int it = 0, tile = 0;
      bool ok = true;
      for (int64_t unit = first; ok && unit < p.units; unit += stride, ++tile) {
        int mt, sp, nt, k0, k1;
        unit_of(unit, mt, sp, nt);
        steps_of(sp, k0, k1);
        const int buf = tile & 1;
        if (!mbar_wait(bar_acce + 8 * buf, ((tile >> 1) & 1) ^ 1, &gone)) {
          gone = 1;
          atomicOr(&g_dense_status, 4);
          break;
        }
        tc_after();
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % C::kStages;
          if (!mbar_wait(bar_full + 8 * s, (it / C::kStages) & 1, &gone)) {
            gone = 1;
            atomicOr(&g_dense_status, 8);
            ok = false;
            break;
          }
          tc_after();
          const uint64_t ad = sw128_desc(sbase + s * C::kStageBytes);
          const uint32_t bs = sbase + s * C::kStageBytes + kATile;
          const uint64_t bd = BN_MAJOR ? sw128_mn_desc(bs) : sw128_desc(bs);
          constexpr int kBStep = BN_MAJOR ? (16 * 128) >> 4 : 32 >> 4;  // 16 rows, or 32 bytes of each row
#pragma unroll
          for (int j = 0; j < kBK / 16; ++j)
            tc_mma<CG>(tmem + buf * kBN, ad + 2 * j, bd + kBStep * j, idesc, (k > k0 || j > 0) ? 1u : 0u);
          tc_commit<CG>(bar_empty + 8 * s);
        }
        tc_commit<CG>(bar_accf + 8 * buf);
      }
    }
  } else {
    // ---- epilogue warps
    const int quad = warp & 3, half = warp >> 2;
    const bool vec = ((p.N | p.e.ldo) & 7) == 0;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t stage = sbase + C::kStaging + warp * kStage2K;
    int tile = 0;
    for (int64_t unit = first; unit < p.units; unit += stride, ++tile) {
      int mt, sp, nt;
      unit_of(unit, mt, sp, nt);
      const int buf = tile & 1;
      const bool ready = mbar_wait(bar_accf + 8 * buf, (tile >> 1) & 1, &gone);
      if (!__all_sync(0xffffffffu, ready)) {
        gone = 1;
        if (lane == 0) atomicOr(&g_dense_status, 16);
        break;
      }
      tc_after();
      const uint32_t acc = tmem + buf * kBN + lanes;
      const int64_t m = (int64_t)(mt * CG + (int)rank) * kBM + quad * 32 + lane;
      if (p.splits > 1) {
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          const int c = half * 128 + q * 32;
          float d[32];
          tmem_ld32(acc + c, d);
          tmem_wait_ld();
          if (m < p.M) {
            float4* dst = reinterpret_cast<float4*>(p.partial + (((int64_t)sp * p.M + m) * p.tiles_n + nt) * kBN + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) dst[i] = make_float4(d[4 * i], d[4 * i + 1], d[4 * i + 2], d[4 * i + 3]);
          }
        }
      } else {
        constexpr int kChunks = EPI == kEpiGated ? 2 : 4;  // of 32 output columns, this warp's half
        const int64_t mrow = m - lane;  // the warp's first row
        const int rows = p.M - mrow < 32 ? (int)(p.M - mrow) : 32;  // may be <= 0
        const int64_t ld = p.e.ldo;
        auto column = [&](int q) {
          return EPI == kEpiGated ? nt * 128 + half * 64 + q * 32 : nt * kBN + half * 128 + q * 32;
        };
        Tile32 tg, tu;
        auto fetch = [&](int q) {
          const int n = column(q);
          const int64_t at = mrow * ld + n;
          if constexpr (EPI == kEpiGatedBackward) {
            fetch_tile(tg, p.e.gate + at, ld, rows, p.N - n, lane);
            fetch_tile(tu, p.e.up + at, ld, rows, p.N - n, lane);
          } else if constexpr (EPI == kEpiPlain) {
            if (p.e.residual) fetch_tile(tg, p.e.residual + at, ld, rows, p.N - n, lane);
          }
        };
        if (vec) fetch(0);
#pragma unroll 1
        for (int q = 0; q < kChunks; ++q) {
          const int c = EPI == kEpiGated ? half * 64 + q * 32 : half * 128 + q * 32;
          const int n = column(q);
          float d[32], u[32];
          tmem_ld32(acc + c, d);
          if constexpr (EPI == kEpiGated) tmem_ld32(acc + 128 + c, u);
          tmem_wait_ld();
          if (!vec) {  // rows of any length: element by element
            if (m < p.M) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float(&d8)[8] = *reinterpret_cast<float(*)[8]>(d + 8 * i);
                const float(&u8)[8] = *reinterpret_cast<float(*)[8]>((EPI == kEpiGated ? u : d) + 8 * i);
                if (n + 8 * i < p.N) epilogue8<EPI, TYPE>(p.e, m, n + 8 * i, p.N, false, d8, u8);
              }
            }
            continue;
          }
          const int64_t at = mrow * ld + n;
          const int cols = p.N - n;
          if constexpr (EPI == kEpiPlain) {
            if (p.e.residual) {
              turn_tile<TYPE>(stage, tg, u, lane);
              if (q + 1 < kChunks) fetch(q + 1);
#pragma unroll
              for (int i = 0; i < 32; ++i) d[i] += u[i];
            }
            store_tile<TYPE>(stage, d, p.e.out + at, ld, rows, cols, lane);
          } else if constexpr (EPI == kEpiGated) {
            if (p.e.gate) {
              store_tile<TYPE>(stage, d, p.e.gate + at, ld, rows, cols, lane);
              store_tile<TYPE>(stage, u, p.e.up + at, ld, rows, cols, lane);
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) d[i] = act_val(d[i], p.e.act) * u[i];
            store_tile<TYPE>(stage, d, p.e.out + at, ld, rows, cols, lane);
          } else {
            float g[32];
            turn_tile<TYPE>(stage, tg, g, lane);
            turn_tile<TYPE>(stage, tu, u, lane);
            if (q + 1 < kChunks) fetch(q + 1);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
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
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(CG == 2 ? map_rank(bar_acce + 8 * buf, 0) : bar_acce + 8 * buf);
    }
  }
  __syncwarp();
  tc_before();
  __syncthreads();
  if constexpr (CG == 2) {
    // the peer's MMAs read this CTA's shared memory and arrive on its barriers
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
  }
  if (warp == kMmaWarp) {
    tc_after();
    if constexpr (CG == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
  }
}

// Adds the splits' partial sums in split order and applies the epilogue: a thread owns eight
// columns of one token.
template <int EPI, int TYPE>
__global__ void __launch_bounds__(256) reduce_kernel(const __grid_constant__ GemmParams p) {
  pdl_wait();
  const int groups = (p.N + 7) / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= p.M * groups) return;
  const int64_t m = i / groups;
  const int c = (int)(i - m * groups) * 8;
  const int64_t pitch = (int64_t)p.tiles_n * kBN;
  // gated: tile c / 128 holds 128 gate sums, then the 128 up sums
  const int64_t at = EPI == kEpiGated ? (int64_t)(c / 128) * kBN + c % 128 : c;
  float d[8] = {}, u[8] = {};
  for (int s = 0; s < p.splits; ++s) {
    const float* row = p.partial + ((int64_t)s * p.M + m) * pitch + at;
    const float4 a = *reinterpret_cast<const float4*>(row), b = *reinterpret_cast<const float4*>(row + 4);
    d[0] += a.x, d[1] += a.y, d[2] += a.z, d[3] += a.w, d[4] += b.x, d[5] += b.y, d[6] += b.z, d[7] += b.w;
    if constexpr (EPI == kEpiGated) {
      const float4 e = *reinterpret_cast<const float4*>(row + 128), f = *reinterpret_cast<const float4*>(row + 132);
      u[0] += e.x, u[1] += e.y, u[2] += e.z, u[3] += e.w, u[4] += f.x, u[5] += f.y, u[6] += f.z, u[7] += f.w;
    }
  }
  epilogue8<EPI, TYPE>(p.e, m, c, p.N, ((p.N | p.e.ldo) & 7) == 0, d, u);
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

// [rows][cols] 16-bit elements, rows ld apart, boxes of box_rows rows x 64 elements.
cudaError_t encode(CUtensorMap* map, const uint16_t* ptr, int64_t rows, int cols, int64_t ld, int box_rows, int type) {
  auto enc = encoder();
  if (!enc) return cudaErrorNotSupported;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {kBK, (cuuint32_t)box_rows};
  const cuuint32_t one[2] = {1, 1};
  const CUresult r =
      enc(map, type == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
          const_cast<uint16_t*>(ptr), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

struct Plan {
  int cg, tiles_m, tiles_n, splits, ks0, ks, spk;
};
constexpr int kSms = 148;

// Tiles and splits of a product. One CTA per 128 tokens when there is one such tile, pairs
// above. Splits: while the tiles leave at least half of the SMs idle and a split keeps eight
// K steps (a split's partial sums cost a write and a read of 4 bytes per output).
Plan plan(int64_t M, int N, int K, int pairs, bool gated) {
  Plan q{};
  q.cg = M > kBM ? 2 : 1;
  q.tiles_m = (int)((M + q.cg * kBM - 1) / (q.cg * kBM));
  q.tiles_n = gated ? (N + 127) / 128 : (N + kBN - 1) / kBN;
  q.ks0 = (K + kBK - 1) / kBK;
  q.ks = q.ks0 * pairs;
  const int64_t ctas = (int64_t)q.tiles_m * q.tiles_n * q.cg;
  q.splits = 1;
  while (ctas * q.splits * 2 <= kSms && q.ks / (q.splits * 2) >= 8) q.splits *= 2;
  q.spk = (q.ks + q.splits - 1) / q.splits;
  q.splits = (q.ks + q.spk - 1) / q.spk;  // no empty split
  return q;
}

template <int CG, int EPI, int TYPE, bool BN_MAJOR>
cudaError_t launch_t(const GemmParams& p, cudaStream_t st) {
  using C = Cfg<CG>;
  auto kern = gemm_kernel<CG, EPI, TYPE, BN_MAJOR>;
  cudaError_t err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (err != cudaSuccess) return err;
  const int64_t most = kSms / CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.units < most ? p.units : most) * CG));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (CG == 2) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = 2;
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
  err = cudaLaunchKernelEx(&cfg, kern, p);
  if (err != cudaSuccess || p.splits == 1) return err;
  const int64_t threads = p.M * ((p.N + 7) / 8);
  return launch_k(reduce_kernel<EPI, TYPE>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, p);
}

template <int CG, int TYPE>
cudaError_t launch_e(const GemmParams& p, int epi, bool n_major, cudaStream_t st) {
  if (epi == kEpiGated) return launch_t<CG, kEpiGated, TYPE, false>(p, st);
  if (epi == kEpiGatedBackward) return launch_t<CG, kEpiGatedBackward, TYPE, true>(p, st);
  return n_major ? launch_t<CG, kEpiPlain, TYPE, true>(p, st) : launch_t<CG, kEpiPlain, TYPE, false>(p, st);
}

}  // namespace

size_t dense_partial_bytes(int64_t M, int N, int K, int pairs, bool gated) {
  const Plan q = plan(M, N, K, pairs, gated);
  return q.splits == 1 ? 0 : (size_t)q.splits * M * q.tiles_n * kBN * sizeof(float);
}

cudaError_t launch_dense_gemm(const DenseGemm& g, cudaStream_t st) {
  const bool gated = g.epilogue == kEpiGated;
  if (g.b_rows_k ? gated : g.epilogue == kEpiGatedBackward) return cudaErrorInvalidValue;
  const Plan q = plan(g.M, g.N, g.K, g.pairs, gated);
  GemmParams p;
  p.M = g.M;
  p.N = g.N;
  p.gated = gated;
  p.ks0 = q.ks0;
  p.ks = q.ks;
  p.tiles_m = q.tiles_m;
  p.tiles_n = q.tiles_n;
  p.splits = q.splits;
  p.spk = q.spk;
  p.units = (int64_t)q.tiles_m * q.tiles_n * q.splits;
  p.partial = g.partial;
  p.e = g.e;
  if (q.splits > 1 && g.partial_bytes < (size_t)q.splits * g.M * q.tiles_n * kBN * sizeof(float))
    return cudaErrorInvalidValue;
  for (int i = 0; i < 2; ++i) {
    const int ai = g.pairs > 1 ? i : 0, bi = (g.pairs > 1 || gated) ? i : 0;
    cudaError_t err = encode(&p.a[i], g.a[ai], g.M, g.K, g.lda[ai], kBM, g.type);
    if (err == cudaSuccess)
      err = g.b_rows_k ? encode(&p.b[i], g.b[bi], g.K, g.N, g.ldb[bi], kBK, g.type)
                       : encode(&p.b[i], g.b[bi], g.N, g.K, g.ldb[bi], 128, g.type);
    if (err != cudaSuccess) return err;
  }
  if (g.type == kF16) return q.cg == 2 ? launch_e<2, kF16>(p, g.epilogue, g.b_rows_k, st) : launch_e<1, kF16>(p, g.epilogue, g.b_rows_k, st);
  return q.cg == 2 ? launch_e<2, kBf16>(p, g.epilogue, g.b_rows_k, st) : launch_e<1, kBf16>(p, g.epilogue, g.b_rows_k, st);
}

cudaError_t dense_status(int32_t* status, cudaStream_t st) {
  cudaError_t err = cudaMemcpyFromSymbolAsync(status, g_dense_status, sizeof(int32_t), 0, cudaMemcpyDeviceToHost, st);
  return err != cudaSuccess ? err : cudaStreamSynchronize(st);
}

}  // namespace moe
