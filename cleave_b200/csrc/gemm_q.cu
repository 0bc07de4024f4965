// Matrix product of two block-scaled 8-bit tensors (quant.cuh) on the 5th-generation tensor cores:
//
//   C[m, n] = act( sum over k-blocks kb of  sA(m, kb) * sB(n, kb) * sum over k in kb of qA(m, k) * qB(n, k)  + bias[n] )
//
// tcgen05.mma.kind::f8f6f4 multiplies the e4m3 bytes and adds up one 128-wide k-block in TMEM (four instructions of K = 32);
// the drain warps read that partial sum, multiply it by the two scales and add it to running sums in registers with
// round-to-nearest.  So scales may be any f32 values, and the tensor pipe's truncating adds never run over more than 128 terms.
//
// Operands are read where they lie, in either order: stored with k contiguous (K-major) or with the row / column index
// contiguous (MN-major); 8-bit operands take the 128-byte swizzle both ways, a 128 x 128 box is 16 KiB.  Out-of-range
// parts of a box read as zero, so sizes need not be multiples of anything.
//
// "P" is the operand on the MMA's M side (128 rows a tile), "Q" the one on its N side.  With few rows (a token, a small
// serving batch) P is the weight matrix and Q the tokens (`swap`): the weights stream through at 128 columns a tile and the
// MMA's N shrinks to 16, 32 or 64, which the weights' HBM time hides.
#include "quant.cuh"
#include "tc_common.cuh"

namespace cleave {

constexpr int kQStageP = 128 * 128;          // bytes of a P box: 128 rows (or columns) x one k-block
constexpr int kQMaxStages = 8;
constexpr int kQRingBudget = 96 * 1024;      // two CTAs fit an SM
constexpr int kQMaxSplit = 8;                // portable cluster size

// Where a side's scales are.
struct QScales {
  // scale of element i of a side in k-block kb: s[kb * s_k + i * s_i + (i / 128) * s_b]
  const float* s;
  int64_t s_k, s_b;
  int s_i, dim;
};

struct QGemmParams {
  float* c;
  const float* bias;
  int act;
  int m, n;
  int p_dim, q_dim;       // extents of the two sides
  int num_kb;             // k-blocks of 128
  int p_tiles;
  int p_mn, q_mn;         // stored with the contraction index as the row
  int swap;               // P is B (columns of C), Q is A (rows of C)
  QScales sp, sq;
  int stages;
  uint32_t stage_bytes;
  DeviceStatus* status;
};

// Bounded wait as mbar_wait, for a pipeline whose steps take a few hundred clocks: the timer, which takes as long to read as
// such a step, is first looked at after a thousand polls.
__device__ __forceinline__ bool q_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  unsigned long long t0 = 0;
  for (uint32_t polls = 1;; ++polls) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((polls & 0x3FFu) == 0) {
      if (*abort_flag) return false;
      const unsigned long long now = globaltimer_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > kWaitLimitNs) {
        *abort_flag = 1;
        return false;
      }
    }
  }
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float load_cluster_f32(uint32_t smem_addr, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_cta(smem_addr, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
// D[tmem] (+)= A[smem] * B[smem], e4m3 inputs, f32 accumulate, K = 32.
__device__ __forceinline__ void umma_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// f32 accumulator, both operands e4m3 (format 0), bit 15 / 16: MN-major A / B, N >> 3, M >> 4.
__host__ __device__ constexpr uint32_t instr_desc_e4m3(int a_mn, int b_mn, int m, int n) {
  return (1u << 4) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}
// Operand descriptor of k-step kk (32 of the k-block's 128) of a box at `base`.  Both orders use the 128-byte swizzle over
// 8 rows of 128 bytes.  K-major: a k-step is 32 bytes along the row.  MN-major: it is 32 rows of 128 bytes; 8-row groups
// follow at 1024 bytes (stride byte offset), the next 128 of M or N at 16 KiB (leading byte offset).
__device__ __forceinline__ uint64_t operand_desc(uint32_t base, int mn_major, int kk) {
  return make_smem_desc(base + (mn_major ? kk * 4096 : kk * 32), 1024u, 2u, mn_major ? 16384u : 16u);
}

// The next k-step in a descriptor's address field (units of 16 bytes).
__device__ __forceinline__ uint64_t k_step(int mn_major) { return mn_major ? 256u : 2u; }

__device__ __forceinline__ void tmem_ld_16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ float q_epilogue(float v, int act) {
  switch (act) {
    case CLEAVE_ACT_RELU: return act_apply(v, CLEAVE_ACT_RELU);
    case CLEAVE_ACT_SIGMOID: return __fdividef(1.0f, 1.0f + __expf(-v));   // as the f32 product's epilogue
    case CLEAVE_ACT_TANH: return tanhf(v);
    default: return v;
  }
}

// Arrival on a barrier of another CTA without the release of this thread's earlier writes: what it announces is that TMEM
// loads have completed (tcgen05.wait::ld), there is no memory to publish.  The releasing form waits for the warp's
// outstanding traffic, 1000 to 1300 clocks here, twice what a k-block's MMAs take (8192^3: 1.02 ms against 0.6).
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// Two f32 in one 64-bit register, added and multiplied lane by lane (round to nearest).
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// Waits for all TMEM loads of the warp; the registers pass through so that no use of them moves above the wait.
__device__ __forceinline__ void tmem_wait_16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}


// ---- scales ----------------------------------------------------------------------------------------------------------
// A k-block's scales come from global memory like its bytes do, a thousand clocks and more behind the request, so they are
// fetched as far ahead: the producer warp copies them (cp.async, 4 bytes a lane: rows of scales start at any multiple of 4)
// into a slot of their own ring, whose barrier the drain warps look at when the k-block is summed.  A slot more than the
// k-blocks that can be under way -- the byte ring, two accumulators, one being drained -- makes every slot free when it
// is filled again, so the ring needs no second barrier.
__device__ __forceinline__ const float* scale_at(const QScales& o, int i) {
  if (i >= o.dim) i = o.dim - 1;   // an element outside C: any scale will do
  return o.s + (int64_t)i * o.s_i + (int64_t)(i >> 7) * o.s_b;
}
__device__ __forceinline__ void copy_scale(uint32_t dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// This lane's copies so far count as one arrival on `bar` once they have landed.
__device__ __forceinline__ void arrive_after_copies(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(bar) : "memory");
}

// ---- drain ----------------------------------------------------------------------------------------------------------
// sum += scale_p * scale_q * (this lane's row of an accumulator, COLS columns from taddr on), two sums an instruction, the next
// 16 columns on their way from TMEM meanwhile.  scale_q: one value, or (QVEC) COLS of them, read as broadcasts.  release()
// runs when the last columns are in registers: the accumulator is free.
template <int COLS, bool QVEC, class Release>
__device__ __forceinline__ void drain_columns(uint64_t (&sum)[COLS / 2], uint32_t taddr, float scale_p, const float* scale_q,
                                              Release release) {
  const float both = QVEC ? scale_p : __fmul_rn(scale_p, *scale_q);
  const uint64_t both2 = pack2(__float_as_uint(both), __float_as_uint(both));
  uint32_t r[2][16];
  tmem_ld_16(taddr, r[0]);
#pragma unroll
  for (int g = 0; g < COLS / 16; ++g) {
    tmem_wait_16(r[g & 1]);
    if (g + 1 < COLS / 16) tmem_ld_16(taddr + (g + 1) * 16, r[(g + 1) & 1]);
    else release();
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const uint64_t v0 = pack2(r[g & 1][2 * j], r[g & 1][2 * j + 1]);
      const uint64_t v1 = pack2(r[g & 1][2 * j + 2], r[g & 1][2 * j + 3]);
      if constexpr (QVEC) {
        const ulonglong2 s = reinterpret_cast<const ulonglong2*>(scale_q)[g * 4 + j / 2];
        sum[g * 8 + j] = fma2(mul2(v0, both2), s.x, sum[g * 8 + j]);
        sum[g * 8 + j + 1] = fma2(mul2(v1, both2), s.y, sum[g * 8 + j + 1]);
      } else {
        sum[g * 8 + j] = fma2(v0, both2, sum[g * 8 + j]);
        sum[g * 8 + j + 1] = fma2(v1, both2, sum[g * 8 + j + 1]);
      }
    }
  }
}
__device__ __forceinline__ float low_half(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float high_half(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }

// Columns a drain warp reads: two warps share a TMEM lane quarter from N = 64 on.
template <int BNQ>
struct QTile {
  static constexpr int kHalves = BNQ >= 64 ? 2 : 1;
  static constexpr int kCols = BNQ / kHalves;
  static constexpr int kDrainWarps = 4 * kHalves;
  static constexpr int kThreads = 64 + 32 * kDrainWarps;
  static constexpr int kTmem = 2 * BNQ < 32 ? 32 : 2 * BNQ;
};

// One 128 x BNQ tile per cluster; the cluster's CTAs take equal runs of its k-blocks and add their sums through distributed
// shared memory, in rank order, each CTA for its own share of the rows.  Warp 0: TMA, warp 1: MMA, the others drain.
template <int BNQ, bool QVEC>
__global__ void __launch_bounds__(QTile<BNQ>::kThreads, 2)
gemm_q_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q, const QGemmParams p) {
  typedef QTile<BNQ> T;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kQMaxStages];
  __shared__ __align__(8) uint64_t bar_empty[kQMaxStages];
  __shared__ __align__(8) uint64_t bar_tmem_full[2];
  __shared__ __align__(8) uint64_t bar_tmem_empty[2];
  constexpr int kScaleQ = QVEC ? BNQ : 4;
  __shared__ __align__(8) uint64_t bar_scale[kQMaxStages + 3];
  __shared__ __align__(16) float scale_p[kQMaxStages + 3][128];
  __shared__ __align__(16) float scale_q[kQMaxStages + 3][kScaleQ];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank(), ranks = cluster_size();
  const int tile = blockIdx.x / ranks;
  const int pt = tile % p.p_tiles, qt = tile / p.p_tiles;
  const int kb0 = (int)((int64_t)p.num_kb * rank / ranks), kb1 = (int)((int64_t)p.num_kb * (rank + 1) / ranks);
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kQMaxStages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    for (int s = 0; s < kQMaxStages + 3; ++s) mbar_init(smem_u32(&bar_scale[s]), 32);
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&bar_tmem_full[a]), 1);
      mbar_init(smem_u32(&bar_tmem_empty[a]), T::kDrainWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"((uint32_t)T::kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = tmem_slot;
  float* red = reinterpret_cast<float*>(smem_raw + (ring - smem_u32(smem_raw)));   // the ring, once it is drained
  constexpr int kRedPitch = BNQ + 1;

  const int slots = p.stages + 3;
  if (warp == 0) {
    int stage = 0, slot = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    const float* src_p[4];
    constexpr int kPerQ = QVEC ? (BNQ + 31) / 32 : 1;
    const float* src_q[kPerQ];
#pragma unroll
    for (int i = 0; i < 4; ++i) src_p[i] = scale_at(p.sp, pt * 128 + lane + 32 * i) + (int64_t)kb0 * p.sp.s_k;
#pragma unroll
    for (int i = 0; i < kPerQ; ++i) src_q[i] = scale_at(p.sq, qt * BNQ + (QVEC ? lane + 32 * i : 0)) + (int64_t)kb0 * p.sq.s_k;
    for (int kb = kb0; kb < kb1; ++kb) {
      ok = __all_sync(0xffffffffu, q_wait(smem_u32(&bar_empty[stage]), phase ^ 1u, &abort_flag));
      if (!ok) {
        if (lane == 0) report(p.status, 1, 1100 + stage, kb);
        break;
      }
      if (lane == 0) {
        const uint32_t full = smem_u32(&bar_full[stage]);
        mbar_arrive_expect_tx(full, p.stage_bytes);
        const uint32_t sp = ring + stage * p.stage_bytes;
        tma_load_2d(sp, &map_p, full, p.p_mn ? pt * 128 : kb * 128, p.p_mn ? kb * 128 : pt * 128);
        tma_load_2d(sp + kQStageP, &map_q, full, p.q_mn ? qt * BNQ : kb * 128, p.q_mn ? kb * 128 : qt * BNQ);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        copy_scale(smem_u32(&scale_p[slot][lane + 32 * i]), src_p[i]);
        src_p[i] += p.sp.s_k;
      }
#pragma unroll
      for (int i = 0; i < kPerQ; ++i) {
        if (lane + 32 * i < kScaleQ) copy_scale(smem_u32(&scale_q[slot][lane + 32 * i]), src_q[i]);
        src_q[i] += p.sq.s_k;
      }
      arrive_after_copies(smem_u32(&bar_scale[slot]));
      ++issued;
      if (++slot == slots) slot = 0;
      if (++stage == p.stages) { stage = 0; phase ^= 1u; }
    }
    if (!ok) {
      // leaving early: give the copies in flight a bounded chance to land
      asm volatile("cp.async.wait_all;" ::: "memory");
      for (int s = 0; lane == 0 && s < p.stages; ++s) {
        const int fills = (issued + p.stages - 1 - s) / p.stages;   // how often stage s was filled
        if (fills == 0) continue;
        for (int spin = 0; spin < (1 << 20); ++spin)
          if (mbar_try_wait(smem_u32(&bar_full[s]), (uint32_t)(fills - 1) & 1u)) break;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = instr_desc_e4m3(p.p_mn, p.q_mn, 128, BNQ);
      const uint64_t desc_p = operand_desc(ring, p.p_mn, 0), desc_q = operand_desc(ring + kQStageP, p.q_mn, 0);
      const uint64_t step_p = k_step(p.p_mn), step_q = k_step(p.q_mn);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!q_wait(smem_u32(&bar_tmem_empty[acc]), acc_phase ^ 1u, &abort_flag)) {
          report(p.status, 2, 1200 + acc, kb);
          break;
        }
        if (!q_wait(smem_u32(&bar_full[stage]), phase, &abort_flag)) {
          report(p.status, 3, 1300 + stage, kb);
          break;
        }
        tcgen05_fence_after();
        const uint64_t at = (uint64_t)(stage * p.stage_bytes) >> 4;
        const uint32_t d = tmem_base + (uint32_t)(acc * BNQ);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_e4m3(d, desc_p + at + kk * step_p, desc_q + at + kk * step_q, idesc, kk ? 1u : 0u);
        tcgen05_commit(smem_u32(&bar_empty[stage]));
        tcgen05_commit(smem_u32(&bar_tmem_full[acc]));
        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
      }
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    uint64_t sum[T::kCols / 2];
#pragma unroll
    for (int j = 0; j < T::kCols / 2; ++j) sum[j] = 0;
    int acc = 0, slot = 0;
    uint32_t acc_phase = 0, slot_phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      bool ok = q_wait(smem_u32(&bar_scale[slot]), slot_phase, &abort_flag) &&
                q_wait(smem_u32(&bar_tmem_full[acc]), acc_phase, &abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        if (lane == 0) report(p.status, 4, 1400 + acc, kb);
        break;
      }
      tcgen05_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * BNQ + half * T::kCols);
      drain_columns<T::kCols, QVEC>(sum, taddr, scale_p[slot][quarter * 32 + lane], &scale_q[slot][QVEC ? half * T::kCols : 0], [&] {
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_tmem_empty[acc]));
      });
      if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
      if (++slot == slots) { slot = 0; slot_phase ^= 1u; }
    }
    // Every load has landed and every MMA has read it: the ring is free for the partial sums.
#pragma unroll
    for (int j = 0; j < T::kCols / 2; ++j) {
      float* at = red + (quarter * 32 + lane) * kRedPitch + half * T::kCols + 2 * j;
      at[0] = low_half(sum[j]);
      at[1] = high_half(sum[j]);
    }
  }

  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if (ranks > 1) cluster_sync_all();
  if (!abort_flag) {
    // This CTA's share of the tile's P rows, summed over the ranks in ascending order and stored along C's rows.
    const int share = 128 / (int)ranks, first = (int)rank * share;
    const int total = share * BNQ;
    for (int i = threadIdx.x; i < total; i += T::kThreads) {
      const int pr = first + (p.swap ? i % share : i / BNQ), qc = p.swap ? i / share : i % BNQ;
      const int gp = pt * 128 + pr, gq = qt * BNQ + qc;
      if (gp >= p.p_dim || gq >= p.q_dim) continue;
      float v;
      if (ranks == 1) {
        v = red[pr * kRedPitch + qc];
      } else {
        const uint32_t at = smem_u32(red + pr * kRedPitch + qc);
        v = load_cluster_f32(at, 0);
        for (uint32_t r = 1; r < ranks; ++r) v = __fadd_rn(v, load_cluster_f32(at, r));
      }
      const int row = p.swap ? gq : gp, col = p.swap ? gp : gq;
      if (p.bias != nullptr) v = __fadd_rn(v, __ldg(p.bias + col));
      p.c[(int64_t)row * p.n + col] = q_epilogue(v, p.act);
    }
  }
  if (ranks > 1) {
    __syncwarp();
    cluster_sync_all();   // the peers are done with this CTA's shared memory
  }
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)T::kTmem) : "memory");
  }
}

// ---- large products: CTA pairs ---------------------------------------------------------------------------------------
// The two CTAs of a cluster share a 256 x 256 tile (tcgen05 cta_group::2): each stages 128 rows of P and 128 of Q per
// k-block (32 KiB a stage, five stages), the MMA of CTA 0 reads Q from both, each CTA drains the sums of its own 128 rows.
// Persistent over the tiles; barriers as in gemm_tc_pair.cu.  At the tensor pipe's rate a k-block takes 512 clocks, in
// which the eight drain warps read 128 x 256 sums from TMEM and add them, scaled, to 128 running sums a thread.
constexpr int kQPairStages = 5;
constexpr int kQPairSlots = kQPairStages + 3;
constexpr int kQPairStageBytes = 2 * kQStageP;
constexpr int kQPairRing = kQPairStages * kQPairStageBytes;
constexpr int kQPairSmem = kQPairRing + kEpiWarps * 32 * 128 + 1024;

struct QPairParams {
  TcParams t;             // c, bias, act, m, n, num_kb, mblks, nblks, pair_group_m, c_tma, status
  int p_mn, q_mn;
  QScales sp, sq;
};

__device__ __forceinline__ void tma_pair_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar_cluster, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar_cluster), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void umma_e4m3_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Adds the bias, applies the activation and stores a drain warp's 32 x 32 block of C whose first element is (row0, col0);
// lane r holds row r.  The block passes through the warp's staging tile (16-byte word j of row r at slot j ^ (r & 7):
// conflict free, and TMA's 128-byte swizzle) and leaves as one bulk tensor store, which clips what lies outside C, or, where
// no tensor map describes C, as 128-byte rows.
__device__ __forceinline__ void store_q_block(float (&v)[32], const TcParams& p, const CUtensorMap* map_c, float4* stage,
                                              int row0, int col0, int lane) {
  if (row0 >= p.m || col0 >= p.n) return;   // uniform over the warp
  if (p.bias != nullptr) {
    if (col0 + 32 <= p.n && (reinterpret_cast<uintptr_t>(p.bias + col0) & 15u) == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float4 b = __ldg(reinterpret_cast<const float4*>(p.bias + col0) + j);
        v[4 * j] = __fadd_rn(v[4 * j], b.x);
        v[4 * j + 1] = __fadd_rn(v[4 * j + 1], b.y);
        v[4 * j + 2] = __fadd_rn(v[4 * j + 2], b.z);
        v[4 * j + 3] = __fadd_rn(v[4 * j + 3], b.w);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (col0 + j < p.n) v[j] = __fadd_rn(v[j], __ldg(p.bias + col0 + j));
    }
  }
  if (p.act == CLEAVE_ACT_TANH) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = q_epilogue(v[j], CLEAVE_ACT_TANH);
  } else if (p.act == CLEAVE_ACT_SIGMOID) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = q_epilogue(v[j], CLEAVE_ACT_SIGMOID);
  } else if (p.act == CLEAVE_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = q_epilogue(v[j], CLEAVE_ACT_RELU);
  }
  if (p.c_tma) {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // the tile's last store has been read
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j)
      stage[lane * 8 + (j ^ (lane & 7))] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // generic writes -> visible to the copy engine
    __syncwarp();
    if (lane == 0) {
      asm volatile(
          "cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
          ::"l"(map_c), "r"(smem_u32(stage)), "r"(col0), "r"(row0), "r"(0)
          : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    return;
  }
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j)
    stage[lane * 8 + (j ^ (lane & 7))] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  __syncwarp();
  const float* words = reinterpret_cast<const float*>(stage);
  const int rows = p.m - row0 < 32 ? p.m - row0 : 32;
  if (col0 + lane < p.n) {
    float* dst = p.c + (int64_t)row0 * p.n + col0 + lane;
    for (int r = 0; r < rows; ++r) dst[(int64_t)r * p.n] = words[r * 32 + (((lane >> 2) ^ (r & 7)) << 2) + (lane & 3)];
  }
}

__device__ __forceinline__ void decode_q_tile(int t, const TcParams& p, int& mb, int& nb) {
  const int span = p.pair_group_m * p.nblks;
  const int first = t / span * p.pair_group_m;
  const int rows_here = (p.mblks - first) < p.pair_group_m ? (p.mblks - first) : p.pair_group_m;
  const int r = t % span;
  mb = first + r % rows_here;
  nb = r / rows_here;
}

template <bool QVEC>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1)
gemm_q_pair_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                   const __grid_constant__ CUtensorMap map_c, const QPairParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kQPairStages];
  __shared__ __align__(8) uint64_t bar_empty[kQPairStages];
  __shared__ __align__(8) uint64_t bar_tmem_full[kAccStages];
  __shared__ __align__(8) uint64_t bar_tmem_empty[kAccStages];
  constexpr int kScaleQ = QVEC ? 256 : 4;   // one value for each 128 columns, or one for every column
  __shared__ __align__(8) uint64_t bar_scale[kQPairSlots];
  __shared__ __align__(16) float scale_p[kQPairSlots][128];
  __shared__ __align__(16) float scale_q[kQPairSlots][kScaleQ];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int tiles = p.t.mblks * p.t.nblks, n_clusters = gridDim.x >> 1, num_kb = p.t.num_kb;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < kQPairStages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    for (int s = 0; s < kQPairSlots; ++s) mbar_init(smem_u32(&bar_scale[s]), 32);
    for (int a = 0; a < kAccStages; ++a) {
      mbar_init(smem_u32(&bar_tmem_full[a]), 1);
      mbar_init(smem_u32(&bar_tmem_empty[a]), 2 * kEpiWarps);   // the drain warps of both CTAs
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                 "r"((uint32_t)kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();   // both CTAs' barriers and TMEM exist before anything crosses over
  tcgen05_fence_after();
  const uint32_t tmem_base = tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_p) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
    }
    int stage = 0, slot = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = blockIdx.x >> 1; ok && t < tiles; t += n_clusters) {
      int mb, nb;
      decode_q_tile(t, p.t, mb, nb);
      const int p0 = mb * 256 + (int)rank * 128, q0 = nb * 256 + (int)rank * 128;
      const float* src_p[4];
      constexpr int kPerQ = QVEC ? 8 : 1;
      const float* src_q[kPerQ];
#pragma unroll
      for (int i = 0; i < 4; ++i) src_p[i] = scale_at(p.sp, p0 + lane + 32 * i);
#pragma unroll
      for (int i = 0; i < kPerQ; ++i) src_q[i] = scale_at(p.sq, nb * 256 + (QVEC ? lane + 32 * i : (lane & 1) * 128));
      for (int kb = 0; kb < num_kb; ++kb) {
        ok = __all_sync(0xffffffffu, q_wait(smem_u32(&bar_empty[stage]), phase ^ 1u, &abort_flag));
        if (!ok) {
          if (lane == 0) report(p.t.status, 1, 1500 + stage, kb);
          break;
        }
        if (lane == 0) {
          const uint32_t full_own = smem_u32(&bar_full[stage]);
          const uint32_t full0 = map_to_cta(full_own, 0);
          if (rank == 0) mbar_arrive_expect_tx(full_own, 2 * kQPairStageBytes);   // both CTAs' boxes
          const uint32_t sp = ring + stage * kQPairStageBytes;
          tma_pair_load_2d(sp, &map_p, full0, p.p_mn ? p0 : kb * 128, p.p_mn ? kb * 128 : p0);
          tma_pair_load_2d(sp + kQStageP, &map_q, full0, p.q_mn ? q0 : kb * 128, p.q_mn ? kb * 128 : q0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          copy_scale(smem_u32(&scale_p[slot][lane + 32 * i]), src_p[i]);
          src_p[i] += p.sp.s_k;
        }
#pragma unroll
        for (int i = 0; i < kPerQ; ++i) {
          if (lane + 32 * i < kScaleQ) copy_scale(smem_u32(&scale_q[slot][lane + 32 * i]), src_q[i]);
          src_q[i] += p.sq.s_k;
        }
        arrive_after_copies(smem_u32(&bar_scale[slot]));
        ++issued;
        if (++slot == kQPairSlots) slot = 0;
        if (++stage == kQPairStages) { stage = 0; phase ^= 1u; }
      }
    }
    if (!ok) {
      // leaving early: give the copies in flight a bounded chance to land (CTA 0 sees their completion)
      asm volatile("cp.async.wait_all;" ::: "memory");
      for (int s = 0; rank == 0 && lane == 0 && s < kQPairStages; ++s) {
        const int fills = (issued + kQPairStages - 1 - s) / kQPairStages;
        if (fills == 0) continue;
        for (int spin = 0; spin < (1 << 20); ++spin)
          if (mbar_try_wait(smem_u32(&bar_full[s]), (uint32_t)(fills - 1) & 1u)) break;
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = instr_desc_e4m3(p.p_mn, p.q_mn, 256, 256);
      const uint64_t desc_p = operand_desc(ring, p.p_mn, 0), desc_q = operand_desc(ring + kQStageP, p.q_mn, 0);
      const uint64_t step_p = k_step(p.p_mn), step_q = k_step(p.q_mn);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = blockIdx.x >> 1; ok && t < tiles; t += n_clusters) {
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!q_wait(smem_u32(&bar_tmem_empty[acc]), acc_phase ^ 1u, &abort_flag)) {
            report(p.t.status, 2, 1600 + acc, kb);
            ok = false;
            break;
          }
          if (!q_wait(smem_u32(&bar_full[stage]), phase, &abort_flag)) {
            report(p.t.status, 3, 1700 + stage, kb);
            ok = false;
            break;
          }
          tcgen05_fence_after();
          const uint64_t at = (uint64_t)(stage * kQPairStageBytes) >> 4;
          const uint32_t d = tmem_base + (uint32_t)(acc * BN);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_e4m3_pair(d, desc_p + at + kk * step_p, desc_q + at + kk * step_q, idesc, kk ? 1u : 0u);
          tcgen05_commit_pair(smem_u32(&bar_empty[stage]));
          tcgen05_commit_pair(smem_u32(&bar_tmem_full[acc]));
          if (++stage == kQPairStages) { stage = 0; phase ^= 1u; }
          if (++acc == kAccStages) { acc = 0; acc_phase ^= 1u; }
        }
      }
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    int acc = 0, slot = 0;
    uint32_t acc_phase = 0, slot_phase = 0;
    float4* stage_tile = reinterpret_cast<float4*>(smem_raw + (ring - smem_u32(smem_raw)) + kQPairRing) + (warp - 2) * (32 * 8);
    bool ok = true;
    for (int t = blockIdx.x >> 1; ok && t < tiles; t += n_clusters) {
      int mb, nb;
      decode_q_tile(t, p.t, mb, nb);
      uint64_t sum[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) sum[j] = 0;
      for (int kb = 0; kb < num_kb; ++kb) {
        ok = q_wait(smem_u32(&bar_scale[slot]), slot_phase, &abort_flag) &&
             q_wait(smem_u32(&bar_tmem_full[acc]), acc_phase, &abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          if (lane == 0) report(p.t.status, 4, 1800 + acc, kb);
          break;
        }
        tcgen05_fence_after();
        const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * BN + half * 128);
        drain_columns<128, QVEC>(sum, taddr, scale_p[slot][quarter * 32 + lane], &scale_q[slot][QVEC ? half * 128 : half], [&] {
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(map_to_cta(smem_u32(&bar_tmem_empty[acc]), 0));
        });
        if (++acc == kAccStages) { acc = 0; acc_phase ^= 1u; }
        if (++slot == kQPairSlots) { slot = 0; slot_phase ^= 1u; }
      }
      if (!ok) break;
#pragma unroll
      for (int pass = 0; pass < 4; ++pass) {
        float v[32];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          v[2 * j] = low_half(sum[pass * 16 + j]);
          v[2 * j + 1] = high_half(sum[pass * 16 + j]);
        }
        store_q_block(v, p.t, &map_c, stage_tile, mb * 256 + (int)rank * 128 + quarter * 32, nb * 256 + half * 128 + 32 * pass,
                      lane);
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // stores have reached memory
  }

  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();   // the peer can no longer issue an MMA into this CTA's TMEM or signal its barriers
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)kTmemCols)
                 : "memory");
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------
struct QSide {
  const uint8_t* q;
  const float* s;
  int dim, k;        // extent of this side, contraction length
  int mn;            // stored [k, dim] instead of [dim, k]
  int blocks;
};

static bool side_map(CUtensorMap* map, const QSide& o, int box) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) {
    set_error(CLEAVE_CUDA_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    return false;
  }
  const int inner = o.mn ? o.dim : o.k, outer = o.mn ? o.k : o.dim;
  const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
  const cuuint64_t strides[1] = {(cuuint64_t)q_pitch(inner)};
  const cuuint32_t boxes[2] = {128u, o.mn ? 128u : (cuuint32_t)box};
  const cuuint32_t ones[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(o.q), dims, strides, boxes, ones,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error(CLEAVE_CUDA_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d (8-bit operand %d x %d)", (int)r, outer, inner);
    return false;
  }
  return true;
}

// Where a side's scales are.  Vector blocks run along k whichever way the operand is stored.
static QScales side_scales(const QSide& o) {
  if (o.blocks != CLEAVE_BLOCKS_TILES) return {o.s, o.dim, 0, 1, o.dim};
  if (o.mn) return {o.s, ceil_div(o.dim, kQBlock), 1, 0, o.dim};
  return {o.s, 1, ceil_div(o.k, kQBlock), 0, o.dim};
}

template <int BNQ, bool QVEC>
static bool launch_q(const CUtensorMap& map_p, const CUtensorMap& map_q, const QGemmParams& p, int tiles, int split) {
  const size_t smem = (size_t)p.stages * p.stage_bytes + 1024;
  static bool attr_set = false;
  if (!attr_set) {
    if (!cuda_ok(cudaFuncSetAttribute(gemm_q_kernel<BNQ, QVEC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      kQRingBudget + 1024),
                 "cudaFuncSetAttribute(8-bit gemm)"))
      return false;
    attr_set = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * split));
  cfg.blockDim = dim3(QTile<BNQ>::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = ctx().stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)split;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  profile_mark(true);
  const bool ok = cuda_ok(cudaLaunchKernelEx(&cfg, gemm_q_kernel<BNQ, QVEC>, map_p, map_q, p), "8-bit GEMM launch");
  profile_mark(false);
  if (ok) count_launch();
  return ok;
}

template <bool QVEC>
static bool launch_q_pair(const CUtensorMap* maps, const QPairParams& p) {
  static bool attr_set = false;
  if (!attr_set) {
    if (!cuda_ok(cudaFuncSetAttribute(gemm_q_pair_kernel<QVEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, kQPairSmem),
                 "cudaFuncSetAttribute(8-bit pair gemm)"))
      return false;
    attr_set = true;
  }
  const int tiles = p.t.mblks * p.t.nblks, pairs = ctx().sm_count / 2;
  profile_mark(true);
  gemm_q_pair_kernel<QVEC><<<2 * (tiles < pairs ? tiles : pairs), kGemmThreads, kQPairSmem, ctx().stream>>>(maps[0], maps[1],
                                                                                                         maps[2], p);
  count_launch();
  const bool ok = cuda_ok(cudaGetLastError(), "8-bit pair GEMM launch");
  profile_mark(false);
  return ok;
}

static bool gemm_q_pairs(const QSide& a, const QSide& b, float* c, const float* bias, int act) {
  QPairParams p = {};
  p.t.c = c;
  p.t.bias = bias;
  p.t.act = act;
  p.t.m = a.dim;
  p.t.n = b.dim;
  p.t.num_kb = ceil_div(a.k, kQBlock);
  p.t.mblks = ceil_div(a.dim, 256);
  p.t.nblks = ceil_div(b.dim, 256);
  p.t.pair_group_m = 8;
  p.t.status = ctx().status_dev;
  p.p_mn = a.mn;
  p.q_mn = b.mn;
  p.sp = side_scales(a);
  p.sq = side_scales(b);
  CUtensorMap maps[3];
  if (!side_map(&maps[0], a, 128) || !side_map(&maps[1], b, 128)) return false;
  maps[2] = maps[0];
  // whole 32 x 32 blocks of C leave as bulk tensor stores where a tensor map can describe C
  p.t.c_tma = aligned16(c) && b.dim % 4 == 0 && make_c_map(&maps[2], c, a.dim, b.dim, 1, 1) ? 1 : 0;
  return b.blocks == CLEAVE_BLOCKS_TILES ? launch_q_pair<false>(maps, p) : launch_q_pair<true>(maps, p);
}

static bool gemm_q(const QSide& a, const QSide& b, float* c, const float* bias, int act) {
  const int64_t pair_tiles = (int64_t)ceil_div(a.dim, 256) * ceil_div(b.dim, 256);
  if (pair_tiles >= ctx().sm_count / 4 && pair_tiles <= 0x3fffffff && a.dim > 128 && b.dim > 128)
    return gemm_q_pairs(a, b, c, bias, act);
  QGemmParams p = {};
  p.c = c;
  p.bias = bias;
  p.act = act;
  p.m = a.dim;
  p.n = b.dim;
  p.num_kb = ceil_div(a.k, kQBlock);
  // the shorter side goes to the MMA's N when it fits 64, where a narrower tile wastes less of it
  p.swap = a.dim <= 64 && a.dim < b.dim;
  const QSide& P = p.swap ? b : a;
  const QSide& Q = p.swap ? a : b;
  p.p_dim = P.dim;
  p.q_dim = Q.dim;
  p.p_mn = P.mn;
  p.q_mn = Q.mn;
  p.sp = side_scales(P);
  p.sq = side_scales(Q);
  p.status = ctx().status_dev;
  const int bn = Q.dim <= 16 ? 16 : Q.dim <= 32 ? 32 : Q.dim <= 64 ? 64 : 128;
  p.stage_bytes = kQStageP + (Q.mn ? kQStageP : bn * 128);
  p.stages = kQRingBudget / (int)p.stage_bytes;
  if (p.stages > kQMaxStages) p.stages = kQMaxStages;
  p.p_tiles = ceil_div(P.dim, 128);
  const int64_t tiles = (int64_t)p.p_tiles * ceil_div(Q.dim, bn);
  if (tiles > 0x7fffffffll / kQMaxSplit) {
    set_error(CLEAVE_CUDA_ERR_UNSUPPORTED, "gemm_e4m3: %d x %d has too many tiles", a.dim, b.dim);
    return false;
  }
  int split = 1;
  while (split < kQMaxSplit && tiles * split * 2 <= 2 * ctx().sm_count && split * 2 <= p.num_kb) split *= 2;
  CUtensorMap map_p, map_q;
  if (!side_map(&map_p, P, 128) || !side_map(&map_q, Q, bn)) return false;
  const bool vec = Q.blocks != CLEAVE_BLOCKS_TILES;
  switch (bn) {
    case 16: return vec ? launch_q<16, true>(map_p, map_q, p, (int)tiles, split) : launch_q<16, false>(map_p, map_q, p, (int)tiles, split);
    case 32: return vec ? launch_q<32, true>(map_p, map_q, p, (int)tiles, split) : launch_q<32, false>(map_p, map_q, p, (int)tiles, split);
    case 64: return vec ? launch_q<64, true>(map_p, map_q, p, (int)tiles, split) : launch_q<64, false>(map_p, map_q, p, (int)tiles, split);
    default: return vec ? launch_q<128, true>(map_p, map_q, p, (int)tiles, split) : launch_q<128, false>(map_p, map_q, p, (int)tiles, split);
  }
}

}  // namespace cleave

using namespace cleave;

extern "C" {

int32_t cleave_cuda_gemm_e4m3(cleave_buf c, cleave_buf a, cleave_buf a_scale, int32_t a_blocks, cleave_buf b, cleave_buf b_scale,
                              int32_t b_blocks, int32_t m, int32_t n, int32_t k, int32_t trans_a, int32_t trans_b,
                              cleave_buf bias, int32_t act) {
  ApiLock lock;
  if (!ensure_init()) return -cleave_cuda_last_error();   // also makes the library's device this thread's
  if (m <= 0 || n <= 0 || k <= 0)
    return -set_error(CLEAVE_CUDA_ERR_ARG, "gemm_e4m3: m, n, k must be positive (got %d, %d, %d)", m, n, k);
  const int ta = trans_a ? 1 : 0, tb = trans_b ? 1 : 0;
  QOperand A, B;
  if (!q_operand(a, a_scale, ta ? k : m, ta ? m : k, a_blocks, "gemm_e4m3", &A) ||
      !q_operand(b, b_scale, tb ? n : k, tb ? k : n, b_blocks, "gemm_e4m3", &B))
    return -cleave_cuda_last_error();
  // A scale has to be constant over a k-block: vector blocks must run along the contraction.
  if (a_blocks == (ta ? CLEAVE_BLOCKS_ROWS : CLEAVE_BLOCKS_COLS) || b_blocks == (tb ? CLEAVE_BLOCKS_COLS : CLEAVE_BLOCKS_ROWS))
    return -set_error(CLEAVE_CUDA_ERR_ARG,
                      "gemm_e4m3: the blocks of an operand must run along the contraction index (or be tiles): "
                      "a_blocks %d with trans_a %d, b_blocks %d with trans_b %d", a_blocks, ta, b_blocks, tb);
  Buf* C = as_buf(c, "gemm_e4m3");
  if (!C) return -cleave_cuda_last_error();
  if (C->len != (int64_t)m * n)
    return -set_error(CLEAVE_CUDA_ERR_SHAPE, "gemm_e4m3: output has %lld elements, not %d x %d", (long long)C->len, m, n);
  Buf* bi = nullptr;
  if (bias) {
    bi = as_buf(bias, "gemm_e4m3");
    if (!bi) return -cleave_cuda_last_error();
    if (bi->len != n)
      return -set_error(CLEAVE_CUDA_ERR_SHAPE, "gemm_e4m3: bias has %lld elements, n is %d", (long long)bi->len, n);
  }
  if (act < CLEAVE_ACT_IDENTITY || act > CLEAVE_ACT_TANH)
    return -set_error(CLEAVE_CUDA_ERR_ARG, "gemm_e4m3: unknown activation code %d", act);
  const MemRange out[1] = {{C->ptr, C->len * 4}};
  const MemRange in[5] = {{A.q, q_bytes(ta ? k : m, ta ? m : k)}, {A.s, q_scales(ta ? k : m, ta ? m : k, a_blocks) * 4},
                          {B.q, q_bytes(tb ? n : k, tb ? k : n)}, {B.s, q_scales(tb ? n : k, tb ? k : n, b_blocks) * 4},
                          {bi ? bi->ptr : nullptr, bi ? bi->len * 4 : 0}};
  if (!ranges_distinct(out, 1, in, 5, "gemm_e4m3")) return -cleave_cuda_last_error();
  Trace tr("gemm_e4m3", "m=%d n=%d k=%d ta=%d tb=%d act=%d", m, n, k, ta, tb, act);
  const QSide sa{A.q, A.s, m, k, ta, a_blocks}, sb{B.q, B.s, n, k, tb ? 0 : 1, b_blocks};
  return gemm_q(sa, sb, C->ptr, bi ? bi->ptr : nullptr, act) ? CLEAVE_CUDA_OK : -cleave_cuda_last_error();
}

}  // extern "C"
