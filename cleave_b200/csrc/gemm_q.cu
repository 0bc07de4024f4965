// Matrix product of two block-scaled 8-bit tensors (quant.cuh) on the 5th-generation tensor cores:
//
//   C[m, n] = act( sum over k-blocks kb of  sA(m, kb) * sB(n, kb) * sum over k in kb of qA(m, k) * qB(n, k)  + bias[n] )
//
// Two kernels.  gemm_q_kernel: tcgen05.mma.kind::f8f6f4 multiplies the e4m3 bytes and adds up one 128-wide k-block in TMEM
// (four instructions of K = 32); the drain warps read that partial sum, multiply it by the two scales and add it to running sums
// in registers with round-to-nearest.  So scales may be any f32 values.  gemm_q_pair_kernel, for large products whose scales
// are powers of two (the quantizer's are): the tensor pipe applies the scales itself.
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

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
// Bounded wait as mbar_wait, for pipelines whose steps take a few hundred clocks.  A waiting warp sleeps in the barrier (for up
// to kSleepNs at a time, woken when the phase completes) instead of polling: with 20 warps a CTA, polls took issue slots from
// the warps at work.  The timer, as slow to read as a step, is looked at every 16 sleeps.
constexpr uint32_t kSleepNs = 200000;
// CLUSTER: for a barrier through which another CTA released generic writes.
template <bool CLUSTER = false>
__device__ __forceinline__ bool q_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  unsigned long long t0 = 0;
  for (uint32_t sleeps = 1;; ++sleeps) {
    uint32_t ok;
    if constexpr (CLUSTER)
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(ok)
          : "r"(bar), "r"(parity), "r"(kSleepNs)
          : "memory");
    else
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(ok)
          : "r"(bar), "r"(parity), "r"(kSleepNs)
          : "memory");
    if (ok) return true;
    if ((sleeps & 15u) == 0) {
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
__device__ __forceinline__ float4 load_cluster_f32x4(uint32_t smem_addr, uint32_t rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(map_to_cta(smem_addr, rank)));
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

// Within 3 * 2^-23 of the sigmoid's value all the way down: e^v / (1 + e^v) on the negative side, where 1 / (1 + e^-v) runs out of range
// from v = -88 on, and expf, whose relative error does not grow with v as __expf's does (1e-6 of the value at v = -13).  The
// reciprocal of 1 to 2 by the approximation, off by one unit in the last place: rounded, the 4096 x 4096 x k1024 layer takes 47 us.
__device__ __forceinline__ float q_sigmoid(float v) {
  const float e = expf(-fabsf(v));
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__fadd_rn(1.0f, e)));
  return v < 0.0f ? __fmul_rn(e, r) : r;
}
__device__ __forceinline__ float q_epilogue(float v, int act) {
  switch (act) {
    case CLEAVE_ACT_RELU: return act_apply(v, CLEAVE_ACT_RELU);
    case CLEAVE_ACT_SIGMOID: return q_sigmoid(v);
    case CLEAVE_ACT_TANH: return tanhf(v);
    default: return v;
  }
}

// One choice for all of a thread's values: choosing for each of them spreads the code over more instruction lines, which a launch of
// one k-block fetches cold.
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int act) {
  if (act == CLEAVE_ACT_TANH) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = q_epilogue(v[j], CLEAVE_ACT_TANH);
  } else if (act == CLEAVE_ACT_SIGMOID) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = q_epilogue(v[j], CLEAVE_ACT_SIGMOID);
  } else if (act == CLEAVE_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = q_epilogue(v[j], CLEAVE_ACT_RELU);
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
__device__ __forceinline__ uint32_t scale_offset(const QScales& o, int i) {
  if (i >= o.dim) i = o.dim - 1;   // an element outside C: any scale will do
  return (uint32_t)(i * o.s_i) + (uint32_t)((i >> 7) * o.s_b);   // below 2^31: i, or the number of tiles
}
__device__ __forceinline__ void copy_scale(uint32_t dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// This lane's copies so far count as one arrival on `bar` once they have landed.
__device__ __forceinline__ void arrive_after_copies(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(bar) : "memory");
}

// ---- drain ----------------------------------------------------------------------------------------------------------
// sum += scale_p * scale_q * (this lane's row of an accumulator, COLS columns from taddr on), two sums an instruction.
// scale_q: one value, or (QVEC) COLS of them, read as broadcasts.  release() runs once the last columns are in registers:
// the accumulator is free.
template <int PIECE>
__device__ __forceinline__ void tmem_ld_wait_piece(uint32_t taddr, uint32_t (&r)[PIECE]) {
  if constexpr (PIECE == 32) {
    tmem_ld_32x32(taddr, r);
    tmem_ld_wait_for(r);
  } else {
    tmem_ld_16(taddr, r);
    tmem_wait_16(r);
  }
}
// Neither the scales' product nor one scale's with the block's sum may leave the range of f32 where the result does not (scales of 2^70
// and 2^60 for a sum of 2^-12).  A block's sum is 0 or from 2^-18 to 2^25, so its product with one scale is safe while that scale is
// within 2^-100 and 2^100, and the scales may be multiplied first while that product is a normal number.  Beyond that, the row's scale is
// brought back by a power of two that is multiplied on last: sum * scale_p' * scale_q, then sum += that * back.  A scale above 2^100
// is lowered by 2^32 only, so that the smallest scale of the other side does not lose bits; where a step overflows, the result does.
template <int COLS, int PIECE, bool QVEC, bool BEYOND, class Release>
__device__ __forceinline__ void drain_pieces(uint64_t (&sum)[COLS / 2], uint32_t taddr, float one, float back, const float* scale_q,
                                             Release release) {
  constexpr int kPiece = PIECE;
  const uint64_t one2 = pack2(__float_as_uint(one), __float_as_uint(one)), back2 = pack2(__float_as_uint(back), __float_as_uint(back));
#pragma unroll
  for (int g = 0; g < COLS / kPiece; ++g) {
    uint32_t r[kPiece];
    tmem_ld_wait_piece<kPiece>(taddr + g * kPiece, r);
    if (g == COLS / kPiece - 1) release();
#pragma unroll
    for (int j = 0; j < kPiece / 2; j += 2) {
      const uint64_t v0 = pack2(r[2 * j], r[2 * j + 1]), v1 = pack2(r[2 * j + 2], r[2 * j + 3]);
      uint64_t &s0 = sum[g * kPiece / 2 + j], &s1 = sum[g * kPiece / 2 + j + 1];
      ulonglong2 q;
      if constexpr (QVEC) q = reinterpret_cast<const ulonglong2*>(scale_q)[g * kPiece / 4 + j / 2];
      else if constexpr (BEYOND) q.x = q.y = pack2(__float_as_uint(*scale_q), __float_as_uint(*scale_q));
      if constexpr (BEYOND) {
        s0 = fma2(mul2(mul2(v0, one2), q.x), back2, s0);
        s1 = fma2(mul2(mul2(v1, one2), q.y), back2, s1);
      } else if constexpr (QVEC) {
        s0 = fma2(mul2(v0, one2), q.x, s0);
        s1 = fma2(mul2(v1, one2), q.y, s1);
      } else {
        s0 = fma2(v0, one2, s0);
        s1 = fma2(v1, one2, s1);
      }
    }
  }
}
template <int COLS, int PIECE, bool QVEC, class Release>
__device__ __forceinline__ void drain_columns(uint64_t (&sum)[COLS / 2], uint32_t taddr, float scale_p, const float* scale_q,
                                              Release release) {
  const float both = QVEC ? scale_p : __fmul_rn(scale_p, *scale_q);
  constexpr float kMost = QVEC ? 0x1p100f : 0x1.fffffep127f, kLeast = QVEC ? 0x1p-100f : 0x1p-126f;
  if (__all_sync(0xffffffffu, fabsf(both) >= kLeast && fabsf(both) <= kMost)) {
    drain_pieces<COLS, PIECE, QVEC, false>(sum, taddr, both, 1.0f, scale_q, release);
  } else {
    const float a = fabsf(scale_p), by = a > 0x1p100f ? 0x1p-32f : a < 0x1p-100f ? 0x1p64f : 1.0f;
    drain_pieces<COLS, PIECE, QVEC, true>(sum, taddr, __fmul_rn(scale_p, by), __frcp_rn(by), scale_q, release);
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
  __shared__ __align__(8) uint64_t bar_done[kQMaxStages];
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
      mbar_init(smem_u32(&bar_done[s]), 1);
    }
    for (int s = 0; s < kQMaxStages + 3; ++s) mbar_init(smem_u32(&bar_scale[s]), 32);
    for (int a = 0; a < 2; ++a) {
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
  // Laid out as C is: along P for swapped sides, along Q otherwise, so that whole 16-byte words are read (from the other CTAs too,
  // where 4-byte words at a stride cost 11 us of a 30 us product) and written; the pitches keep both free of bank conflicts.
  constexpr int kRedPitch = BNQ + 4, kRedPitchSwap = 132;

  const int slots = p.stages + 3;
  if (warp == 0) {
    int stage = 0, slot = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    uint32_t off_p[4];   // floats from the k-block's first scale
    constexpr int kPerQ = QVEC ? (BNQ + 31) / 32 : 1;
    uint32_t off_q[kPerQ];
#pragma unroll
    for (int i = 0; i < 4; ++i) off_p[i] = scale_offset(p.sp, pt * 128 + lane + 32 * i);
#pragma unroll
    for (int i = 0; i < kPerQ; ++i) off_q[i] = scale_offset(p.sq, qt * BNQ + (QVEC ? lane + 32 * i : 0));
    const float *src_p = p.sp.s + kb0 * p.sp.s_k, *src_q = p.sq.s + kb0 * p.sq.s_k;
    for (int kb = kb0; kb < kb1; ++kb) {
      ok = __all_sync(0xffffffffu, q_wait(smem_u32(&bar_done[stage]), phase ^ 1u, &abort_flag));
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
      for (int i = 0; i < 4; ++i) copy_scale(smem_u32(&scale_p[slot][lane + 32 * i]), src_p + off_p[i]);
#pragma unroll
      for (int i = 0; i < kPerQ; ++i)
        if (lane + 32 * i < kScaleQ) copy_scale(smem_u32(&scale_q[slot][lane + 32 * i]), src_q + off_q[i]);
      src_p += p.sp.s_k;
      src_q += p.sq.s_k;
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
        tcgen05_commit(smem_u32(&bar_done[stage]));
        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
      }
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    uint64_t sum[T::kCols / 2];
#pragma unroll
    for (int j = 0; j < T::kCols / 2; ++j) sum[j] = 0;
    int acc = 0, slot = 0, stage = 0;
    uint32_t phase = 0, slot_phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      bool ok = q_wait(smem_u32(&bar_scale[slot]), slot_phase, &abort_flag) &&
                q_wait(smem_u32(&bar_done[stage]), phase, &abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        if (lane == 0) report(p.status, 4, 1400 + acc, kb);
        break;
      }
      tcgen05_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * BNQ + half * T::kCols);
      // 64 columns a warp leave no registers for pieces of 32: they spill (4096 x 4096 x k1024 of any scales 94 us against 78)
      drain_columns<T::kCols, T::kCols == 32 ? 32 : 16, QVEC>(sum, taddr, scale_p[slot][quarter * 32 + lane],
                                                              &scale_q[slot][QVEC ? half * T::kCols : 0], [&] {
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_tmem_empty[acc]));
      });
      acc ^= 1;
      if (++stage == p.stages) { stage = 0; phase ^= 1u; }
      if (++slot == slots) { slot = 0; slot_phase ^= 1u; }
    }
    // Every load has landed and every MMA has read it: the ring is free for the partial sums.
    const int pr = quarter * 32 + lane;
    if (p.swap) {
#pragma unroll
      for (int j = 0; j < T::kCols / 2; ++j) {
        red[(half * T::kCols + 2 * j) * kRedPitchSwap + pr] = low_half(sum[j]);
        red[(half * T::kCols + 2 * j + 1) * kRedPitchSwap + pr] = high_half(sum[j]);
      }
    } else {
      float4* at = reinterpret_cast<float4*>(red + pr * kRedPitch + half * T::kCols);
#pragma unroll
      for (int j = 0; j < T::kCols / 4; ++j)
        at[j] = make_float4(low_half(sum[2 * j]), high_half(sum[2 * j]), low_half(sum[2 * j + 1]), high_half(sum[2 * j + 1]));
    }
  }

  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  // This CTA's share of the tile's P rows, four neighbours of C at a time, kBatch of those a thread: what does not depend on the
  // sums (places, bias) is fetched before the barrier, and the CTA tells its peers that it has read theirs before it stores.
  constexpr int kBatch = BNQ <= 64 ? 2 : 1;
  const int share = 128 / (int)ranks, first = (int)rank * share;
  const int inner4 = (p.swap ? share : BNQ) / 4, total = share * BNQ / 4;
  const bool vec_ok = p.n % 4 == 0 && (reinterpret_cast<uintptr_t>(p.c) & 15u) == 0;
  bool arrived = false;
  for (int base = 0; base < total; base += kBatch * T::kThreads) {   // the same trips for every thread
    const float* at[kBatch];
    int row[kBatch], col[kBatch];
    float bias[kBatch][4];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = base + u * T::kThreads + (int)threadIdx.x;
      const int outer = i / inner4, inner = (i - outer * inner4) * 4;
      const int pr = first + (p.swap ? inner : outer), qc = p.swap ? outer : inner;
      at[u] = p.swap ? red + qc * kRedPitchSwap + pr : red + pr * kRedPitch + qc;
      row[u] = p.swap ? qt * BNQ + qc : pt * 128 + pr;
      col[u] = p.swap ? pt * 128 + pr : qt * BNQ + qc;
      if (i >= total) row[u] = p.m;   // nothing to do
#pragma unroll
      for (int e = 0; e < 4; ++e) bias[u][e] = p.bias != nullptr && row[u] < p.m && col[u] + e < p.n ? __ldg(p.bias + col[u] + e) : 0.0f;
    }
    if (base == 0 && ranks > 1) {
      __syncwarp();   // the barrier's .aligned form needs the warp in one piece, and the lanes' loads above differ
      cluster_sync_all();
    }
    float4 part[kBatch][kQMaxSplit];
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
#pragma unroll
      for (int r = 0; r < kQMaxSplit; ++r)
        if (row[u] < p.m && r < (int)ranks)
          part[u][r] = ranks == 1 ? *reinterpret_cast<const float4*>(at[u]) : load_cluster_f32x4(smem_u32(at[u]), (uint32_t)r);
    if (ranks > 1 && base + kBatch * T::kThreads >= total) {
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // the loads above have been performed
      arrived = true;
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (row[u] >= p.m || col[u] >= p.n || abort_flag) continue;
      float v[4] = {part[u][0].x, part[u][0].y, part[u][0].z, part[u][0].w};
#pragma unroll
      for (int r = 1; r < kQMaxSplit; ++r)   // in rank order
        if (r < (int)ranks) {
          v[0] = __fadd_rn(v[0], part[u][r].x);
          v[1] = __fadd_rn(v[1], part[u][r].y);
          v[2] = __fadd_rn(v[2], part[u][r].z);
          v[3] = __fadd_rn(v[3], part[u][r].w);
        }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = p.bias != nullptr ? __fadd_rn(v[e], bias[u][e]) : v[e];
      activate(v, p.act);
      float* dst = p.c + (int64_t)row[u] * p.n + col[u];
      if (vec_ok) {   // n and col are multiples of 4
        *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col[u] + e < p.n) dst[e] = v[e];
      }
    }
  }
  __syncwarp();
  if (arrived) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // the peers have read this CTA's shared memory
  }
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)T::kTmem) : "memory");
  }
}

// ---- large products with power-of-two scales: CTA pairs, scales applied by the tensor pipe ---------------------------------
// The two CTAs of a cluster share a 256 x 256 tile (tcgen05 cta_group::2): each stages 128 rows of P and 128 of Q per
// k-block (32 KiB a stage), the MMA issued by CTA 0 reads Q from both, each CTA drains the sums of its own 128 rows.
//
// tcgen05.mma.kind::mxf8f6f4.block_scale multiplies every 32 products by a power of two per row of P and one per row of Q,
// given as exponent bytes in TMEM.  A scale that is a power of two is its f32 exponent field, so two warps fetch the
// scales, keep bits 23-30 of each, and pack four k-blocks' bytes of an element into one word (the instruction descriptor
// selects the byte); the issuer copies the words to TMEM once per four k-blocks.  The partial sums then need no work per k-block:
// the accumulator runs over eight (1024 terms) before the drain warps add it to 64 running sums a thread with
// round-to-nearest, which bounds what the tensor pipe's truncating adds can lose (32 adds of at most 2^-23).
//
// Layout of the words, in shared memory and TMEM: element r of 128 at row r % 32, word r / 32 of a row of four; TMEM holds it
// in four columns of 32 lanes, repeated in all four lane quarters (tcgen05.cp ... 32x128b.warpx4).  P: the CTA's own 128 rows;
// Q: all 256, in both CTAs.
//
// Measured, 8192^3, 256 MiB of C included: 440 to 453 us in bursts (2.43 PFLOP/s, 770 clocks a k-block at 1.53 GHz, the power limit; the
// pipe's own rate is 512) and 520 to 535 us over seconds, one scale per column or per 128 alike.  A drain that scales every k-block
// itself (as gemm_q_kernel does), same tile: 577 us with one scale for 128 columns, 1030 us with one per column, the pipe waiting for
// the drain's multiplies.  What it waits for now: the accumulator's drain at the end of a chunk (about 650 clocks in 4100), and power.
constexpr int kQPairDrainWarps = 16;
constexpr int kQPairCols = 64;                               // columns a drain warp sums: a quarter of the tile
constexpr int kQPairThreads = 128 + 32 * kQPairDrainWarps;   // warp 0 TMA, 1 MMA, 2 scales of P, 3 scales of Q
constexpr int kQPairStages = 4;                              // k-block kb of a tile is in stage kb % 4
constexpr int kQPairStageBytes = 2 * kQStageP;
constexpr int kQPairRing = kQPairStages * kQPairStageBytes;
constexpr int kQPairStaging = 32 * 128;                      // bytes of a drain warp's staging tile: 32 rows x 32 columns
constexpr int kQPairSmem = kQPairRing + kQPairDrainWarps * kQPairStaging + 1024;
constexpr int kQGroup = 4;                                   // k-blocks whose scales share a word: one turn of the ring
constexpr int kQChunk = 8;                                   // k-blocks summed in TMEM
constexpr int kQScaleSlots = 4;
constexpr int kQScaleSlotBytes = 3 * 512;                    // [P | Q 0..127 | Q 128..255]
constexpr int kQScaleCol = 256;                              // TMEM columns behind the accumulator: two sets of 4 + 8

struct QPairParams {
  TcParams t;             // c, bias, act, m, n, num_kb, mblks, nblks, pair_group_m, status
  QScales sp, sq;
};

__device__ __forceinline__ void tma_pair_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar_cluster, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar_cluster), "r"(c0), "r"(c1)
      : "memory");
}
// D[tmem] (+)= (A[smem] * scale) (B[smem] * scale), e4m3 inputs, one exponent byte per 32 along k, f32 accumulate, K = 32.
__device__ __forceinline__ void umma_e4m3_scaled_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                                      uint32_t a_scale_tmem, uint32_t b_scale_tmem, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scale_tmem), "r"(b_scale_tmem), "r"(accumulate)
      : "memory");
}
// Both operands e4m3 (format 0), scales as exponent bytes (bit 23), bits 15 / 16: MN-major A / B, N >> 3, M >> 4.  The byte of a
// scale word: bits 29-30 for A, 4-5 for B.
__host__ __device__ constexpr uint32_t instr_desc_e4m3_scaled(int a_mn, int b_mn, int m, int n) {
  return (1u << 23) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ uint32_t scale_byte_select(int i) { return ((uint32_t)i << 29) | ((uint32_t)i << 4); }
// 32 rows of 16 bytes of shared memory (unswizzled, 8-row groups 128 bytes apart) to 4 columns of TMEM, in both CTAs.
__device__ __forceinline__ void copy_scales_pair(uint32_t tmem, uint32_t smem) {
  const uint64_t desc = make_smem_desc(smem, 128u, 0u, 0u);
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// Adds the bias (shared memory, 32 values), applies the activation and stores a drain warp's 32 x 32 block of C whose first element is (row0, col0);
// lane r holds row r.  The block passes through the warp's staging tile (16-byte word j of row r at slot j ^ (r & 7):
// conflict free both ways), so that every store instruction writes whole 128-byte lines.  Plain stores: bulk tensor stores of the
// same tile queue in the copy engine before the next tile's loads, which then took 3000 to 4700 clocks to arrive.
__device__ __forceinline__ void store_q_block(float (&v)[32], const TcParams& p, const float* bias, float4* stage, int row0,
                                              int col0, int lane, bool vec_ok) {
  if (row0 >= p.m || col0 >= p.n) return;   // uniform over the warp
  if (p.bias != nullptr) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 b = reinterpret_cast<const float4*>(bias)[j];
      v[4 * j] = __fadd_rn(v[4 * j], b.x);
      v[4 * j + 1] = __fadd_rn(v[4 * j + 1], b.y);
      v[4 * j + 2] = __fadd_rn(v[4 * j + 2], b.z);
      v[4 * j + 3] = __fadd_rn(v[4 * j + 3], b.w);
    }
  }
  activate(v, p.act);
  __syncwarp();   // the tile's last block has been read
#pragma unroll
  for (int j = 0; j < 8; ++j)
    stage[lane * 8 + (j ^ (lane & 7))] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  __syncwarp();
  if (vec_ok) {   // C is 16-byte aligned and n a multiple of 4
    const int slot = lane & 7;
    if (col0 + 4 * slot < p.n) {
      float* dst = p.c + (int64_t)row0 * p.n + col0 + 4 * slot;
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const int r = it * 4 + (lane >> 3);
        if (row0 + r < p.m) *reinterpret_cast<float4*>(dst + (int64_t)r * p.n) = stage[r * 8 + (slot ^ (r & 7))];
      }
    }
    return;
  }
  const float* words = reinterpret_cast<const float*>(stage);
  if (col0 + lane < p.n) {
    float* dst = p.c + (int64_t)row0 * p.n + col0 + lane;
    for (int r = 0; r < 32 && row0 + r < p.m; ++r)
      dst[(int64_t)r * p.n] = words[r * 32 + (((lane >> 2) ^ (r & 7)) << 2) + (lane & 3)];
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

template <int P_MN, int Q_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kQPairThreads, 1)
gemm_q_pair_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                   const QPairParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(128) uint8_t scale_words[kQScaleSlots][kQScaleSlotBytes];
  __shared__ __align__(16) float bias_words[kQPairDrainWarps][kQPairCols];
  // full / done: a stage's bytes have landed (in CTA 0, for both) / its MMAs have read them; scale_full / scale_empty: the
  // same for a slot of scale words; acc_full / acc_empty: the accumulator is complete / has been read (in CTA 0)
  __shared__ __align__(8) uint64_t bar_full[kQPairStages];
  __shared__ __align__(8) uint64_t bar_done[kQPairStages];
  __shared__ __align__(8) uint64_t bar_scale_full[kQScaleSlots];
  __shared__ __align__(8) uint64_t bar_scale_empty[kQScaleSlots];
  __shared__ __align__(8) uint64_t bar_acc_full, bar_acc_empty;
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
      mbar_init(smem_u32(&bar_done[s]), 1);
    }
    for (int s = 0; s < kQScaleSlots; ++s) {
      mbar_init(smem_u32(&bar_scale_full[s]), rank == 0 ? 3 : 2);   // the CTA's two scale warps; in CTA 0 also CTA 1's word for its own
      mbar_init(smem_u32(&bar_scale_empty[s]), 1);
    }
    mbar_init(smem_u32(&bar_acc_full), 1);
    mbar_init(smem_u32(&bar_acc_empty), 2 * kQPairDrainWarps);
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
    // ---- bytes
    if (elect_one()) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_p) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
    }
    uint32_t phases = 0, used = 0;   // a bit a stage: the parity of its next fill; filled at all
    bool ok = true;
    for (int t = blockIdx.x >> 1; ok && t < tiles; t += n_clusters) {
      int mb, nb;
      decode_q_tile(t, p.t, mb, nb);
      const int p0 = mb * 256 + (int)rank * 128, q0 = nb * 256 + (int)rank * 128;
      for (int kb = 0; kb < num_kb; ++kb) {
        const int stage = kb % kQPairStages;
        ok = __all_sync(0xffffffffu, q_wait(smem_u32(&bar_done[stage]), ((phases >> stage) & 1u) ^ 1u, &abort_flag));
        if (!ok) {
          if (lane == 0) report(p.t.status, 1, 1500 + stage, kb);
          break;
        }
        if (elect_one()) {
          const uint32_t full_own = smem_u32(&bar_full[stage]);
          const uint32_t full0 = map_to_cta(full_own, 0);
          if (rank == 0) mbar_arrive_expect_tx(full_own, 2 * kQPairStageBytes);   // both CTAs' boxes
          const uint32_t sp = ring + stage * kQPairStageBytes;
          tma_pair_load_2d(sp, &map_p, full0, P_MN ? p0 : kb * 128, P_MN ? kb * 128 : p0);
          tma_pair_load_2d(sp + kQStageP, &map_q, full0, Q_MN ? q0 : kb * 128, Q_MN ? kb * 128 : q0);
        }
        __syncwarp();
        phases ^= 1u << stage;
        used |= 1u << stage;
      }
    }
    if (!ok && rank == 0 && lane == 0) {
      // leaving early: give the copies in flight a bounded chance to land (CTA 0 sees their completion)
      for (int s = 0; s < kQPairStages; ++s)
        for (int spin = 0; ((used >> s) & 1u) && spin < (1 << 20); ++spin)
          if (mbar_try_wait(smem_u32(&bar_full[s]), ((phases >> s) & 1u) ^ 1u)) break;
    }
  } else if (warp == 1) {
    // ---- MMAs, CTA 0 for both.  The whole warp runs the loop, so that its state stays in uniform registers; one lane issues.
    if (rank == 0) {
      constexpr uint32_t idesc = instr_desc_e4m3_scaled(P_MN, Q_MN, 256, 256);
      const uint64_t desc_p = operand_desc(ring, P_MN, 0), desc_q = operand_desc(ring + kQStageP, Q_MN, 0);
      const int my_tiles = (tiles - (int)(blockIdx.x >> 1) + n_clusters - 1) / n_clusters;
      const int groups = my_tiles * ((num_kb + kQGroup - 1) / kQGroup);
      uint32_t phases = 0, acc_phase = 0;
      bool ok = true;
      // The scale words of group g (counted over the tiles) go to TMEM while the group before it is being multiplied.
      auto fetch_scales = [&](int g) {
        const int slot = g % kQScaleSlots;
        ok = __all_sync(0xffffffffu, q_wait<true>(smem_u32(&bar_scale_full[slot]), (uint32_t)(g / kQScaleSlots) & 1u, &abort_flag));
        if (!ok) {
          if (lane == 0) report(p.t.status, 2, 1600 + slot, g);
          return;
        }
        tcgen05_fence_after();
        if (elect_one()) {   // ordered before the MMAs that follow from this thread
          const uint32_t scales = tmem_base + kQScaleCol + (uint32_t)(g & 1) * 16u;
          const uint32_t words = smem_u32(&scale_words[slot][0]);
          copy_scales_pair(scales, words);
          copy_scales_pair(scales + 4, words + 512);
          copy_scales_pair(scales + 8, words + 1024);
        }
        __syncwarp();
      };
      int g = 0;
      fetch_scales(0);
      for (int t = blockIdx.x >> 1; ok && t < tiles; t += n_clusters) {
        for (int kb0 = 0; ok && kb0 < num_kb; kb0 += kQGroup, ++g) {
          const bool chunk_start = kb0 % kQChunk == 0;
          if (chunk_start) {
            ok = __all_sync(0xffffffffu, q_wait(smem_u32(&bar_acc_empty), acc_phase ^ 1u, &abort_flag));
            if (!ok) {
              if (lane == 0) report(p.t.status, 5, 1650, kb0);
              break;
            }
          }
          const uint32_t scales = tmem_base + kQScaleCol + (uint32_t)(g & 1) * 16u;
#pragma unroll
          for (int s = 0; s < kQGroup; ++s) {
            if (kb0 + s >= num_kb) break;
            ok = __all_sync(0xffffffffu, q_wait(smem_u32(&bar_full[s]), (phases >> s) & 1u, &abort_flag));
            if (!ok) {
              if (lane == 0) report(p.t.status, 3, 1700 + s, kb0);
              break;
            }
            tcgen05_fence_after();
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                umma_e4m3_scaled_pair(tmem_base, desc_p + (uint32_t)((s * kQPairStageBytes + kk * (P_MN ? 4096 : 32)) >> 4),
                                      desc_q + (uint32_t)((s * kQPairStageBytes + kk * (Q_MN ? 4096 : 32)) >> 4),
                                      idesc | scale_byte_select(s), scales, scales + 4,
                                      s == 0 && kk == 0 && chunk_start ? 0u : 1u);
              tcgen05_commit_pair(smem_u32(&bar_done[s]));
            }
            __syncwarp();
            phases ^= 1u << s;
          }
          if (!ok) break;
          const bool chunk_end = kb0 + kQGroup >= num_kb || kb0 % kQChunk == kQChunk - kQGroup;
          if (elect_one()) {
            if (chunk_end) tcgen05_commit_pair(smem_u32(&bar_acc_full));
            tcgen05_commit_pair(smem_u32(&bar_scale_empty[g % kQScaleSlots]));
          }
          __syncwarp();
          if (chunk_end) acc_phase ^= 1u;
          if (g + 1 < groups) fetch_scales(g + 1);
        }
      }
    }
    else {
      // CTA 1 tells CTA 0 that its scale words are there.  The release that another CTA's copy to TMEM needs takes a thousand
      // clocks; here they delay nobody.
      const int my_tiles = (tiles - (int)(blockIdx.x >> 1) + n_clusters - 1) / n_clusters;
      const int groups = my_tiles * ((num_kb + kQGroup - 1) / kQGroup);
      for (int g = 0; g < groups; ++g) {
        const int slot = g % kQScaleSlots;
        if (!__all_sync(0xffffffffu, q_wait(smem_u32(&bar_scale_full[slot]), (uint32_t)(g / kQScaleSlots) & 1u, &abort_flag))) {
          if (lane == 0) report(p.t.status, 6, 1900 + slot, g);
          break;
        }
        if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&bar_scale_full[slot]), 0));
        __syncwarp();
      }
    }
  } else if (warp < 4) {
    // ---- scales: warp 2 the CTA's 128 rows of P, warp 3 the tile's 256 of Q
    const bool for_q = warp == 3;
    const QScales& o = for_q ? p.sq : p.sp;
    int slot = 0;
    uint32_t slot_phase = 0;
    bool ok = true;
    for (int t = blockIdx.x >> 1; ok && t < tiles; t += n_clusters) {
      int mb, nb;
      decode_q_tile(t, p.t, mb, nb);
      const int first = for_q ? nb * 256 : mb * 256 + (int)rank * 128;
      for (int kb0 = 0; kb0 < num_kb; kb0 += kQGroup) {
        // all loads of the group before the first use: one latency a group, and the slots let the warp run three groups ahead
        uint32_t bits[2][4][kQGroup], w[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float* src = o.s + scale_offset(o, first + h * 128 + i * 32 + lane) + (int64_t)kb0 * o.s_k;
#pragma unroll
            for (int j = 0; j < kQGroup; ++j)
              bits[h][i][j] = (h == 0 || for_q) && kb0 + j < num_kb ? __float_as_uint(__ldg(src + j * o.s_k)) : 0x3f800000u;
          }
        // The exponent is all that is used of a scale.  One with a sign, a mantissa, or an exponent field of 0 or 255 is no power of
        // two: the tensor lacks its mark, the product would be wrong, and the host hears of it.
        uint32_t odd = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < kQGroup; ++j)
              odd |= (bits[h][i][j] & 0x807fffffu) | ((bits[h][i][j] - 0x00800000u) & 0x80000000u) |
                     ((bits[h][i][j] + 0x00800000u) & 0x80000000u);
        if (__any_sync(0xffffffffu, odd != 0) && lane == 0) report(p.t.status, kStatusScales, for_q, kb0);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[h][i] = ((bits[h][i][0] >> 23) & 0xffu) | (((bits[h][i][1] >> 23) & 0xffu) << 8) |
                      (((bits[h][i][2] >> 23) & 0xffu) << 16) | (((bits[h][i][3] >> 23) & 0xffu) << 24);
        ok = __all_sync(0xffffffffu, q_wait(smem_u32(&bar_scale_empty[slot]), slot_phase ^ 1u, &abort_flag));
        if (!ok) {
          if (lane == 0) report(p.t.status, 3, 1700 + slot, kb0);
          break;
        }
        uint4* dst = reinterpret_cast<uint4*>(&scale_words[slot][for_q ? 512 : 0]) + lane;
        dst[0] = make_uint4(w[0][0], w[0][1], w[0][2], w[0][3]);
        if (for_q) dst[32] = make_uint4(w[1][0], w[1][1], w[1][2], w[1][3]);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // generic writes -> visible to the copy to TMEM
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_scale_full[slot]));
        if (++slot == kQScaleSlots) { slot = 0; slot_phase ^= 1u; }
      }
    }
  } else {
    // ---- drain and epilogue
    const int quarter = warp & 3, part = (warp - 4) >> 2;   // TMEM lanes 32 * quarter .., columns 64 * part ..
    uint32_t acc_phase = 0;
    float4* stage_tile = reinterpret_cast<float4*>(smem_raw + (ring - smem_u32(smem_raw)) + kQPairRing + (warp - 4) * kQPairStaging);
    const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(part * kQPairCols);
    float* bias_tile = bias_words[warp - 4];
    const bool vec_ok = p.t.n % 4 == 0 && (reinterpret_cast<uintptr_t>(p.t.c) & 15u) == 0;
    const uint32_t acc_empty0 = map_to_cta(smem_u32(&bar_acc_empty), 0);
    bool ok = true;
    for (int t = blockIdx.x >> 1; ok && t < tiles; t += n_clusters) {
      int mb, nb;
      decode_q_tile(t, p.t, mb, nb);
      float sum[kQPairCols], bias[2] = {0.0f, 0.0f};   // the warp's 64 columns of the bias, two a lane, fetched long before their use
      if (p.t.bias != nullptr) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int col = nb * 256 + part * kQPairCols + i * 32 + lane;
          if (col < p.t.n) bias[i] = __ldg(p.t.bias + col);
        }
      }
#pragma unroll
      for (int j = 0; j < kQPairCols; ++j) sum[j] = 0.0f;
      for (int kb = 0; kb < num_kb; kb += kQChunk) {
        ok = __all_sync(0xffffffffu, q_wait(smem_u32(&bar_acc_full), acc_phase, &abort_flag));
        if (!ok) {
          if (lane == 0) report(p.t.status, 4, 1800, kb);
          break;
        }
        tcgen05_fence_after();
#pragma unroll
        for (int g = 0; g < kQPairCols / 16; ++g) {
          uint32_t r[16];
          tmem_ld_16(taddr + g * 16, r);
          tmem_wait_16(r);
          if (g == kQPairCols / 16 - 1) {   // all columns are in registers: the accumulator is free
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(acc_empty0);
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) sum[g * 16 + j] = __fadd_rn(sum[g * 16 + j], __uint_as_float(r[j]));
        }
        acc_phase ^= 1u;
      }
      if (!ok) break;
      __syncwarp();   // the last tile's have been read
      bias_tile[lane] = bias[0];
      bias_tile[lane + 32] = bias[1];
      __syncwarp();
#pragma unroll
      for (int pass = 0; pass < kQPairCols / 32; ++pass) {
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = sum[pass * 32 + j];
        store_q_block(v, p.t, bias_tile + 32 * pass, stage_tile, mb * 256 + (int)rank * 128 + quarter * 32, nb * 256 + part * kQPairCols + 32 * pass, lane,
                      vec_ok);
      }
    }
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
  int blocks;        // CLEAVE_BLOCKS_*
  bool any_scales;   // not all of them powers of two
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

template <int P_MN, int Q_MN>
static bool launch_q_pair(const CUtensorMap* maps, const QPairParams& p) {
  static bool attr_set = false;
  if (!attr_set) {
    if (!cuda_ok(cudaFuncSetAttribute(gemm_q_pair_kernel<P_MN, Q_MN>, cudaFuncAttributeMaxDynamicSharedMemorySize, kQPairSmem),
                 "cudaFuncSetAttribute(8-bit pair gemm)"))
      return false;
    attr_set = true;
  }
  const int tiles = p.t.mblks * p.t.nblks, pairs = ctx().sm_count / 2;
  profile_mark(true);
  gemm_q_pair_kernel<P_MN, Q_MN><<<2 * (tiles < pairs ? tiles : pairs), kQPairThreads, kQPairSmem, ctx().stream>>>(
      maps[0], maps[1], p);
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
  p.sp = side_scales(a);
  p.sq = side_scales(b);
  CUtensorMap maps[2];
  if (!side_map(&maps[0], a, 128) || !side_map(&maps[1], b, 128)) return false;
  return a.mn ? (b.mn ? launch_q_pair<1, 1>(maps, p) : launch_q_pair<1, 0>(maps, p))
              : (b.mn ? launch_q_pair<0, 1>(maps, p) : launch_q_pair<0, 0>(maps, p));
}

static bool gemm_q(const QSide& a, const QSide& b, float* c, const float* bias, int act) {
  // CTA pairs from 19 tiles of 256 x 256 on (an eighth of the SMs), unless a side fits half a tile.  Measured, one CTA / pairs, us, B in
  // tiles: 16 tiles (1024 x 1024) k 512 13.8 / 12.4, k 4096 18.5 / 24.5; 24 tiles (1536 x 1024) 14.4 / 12.4, 26.7 / 24.5; 64 tiles
  // 18.5 / 14.2, 43.0 / 24.6; 136 x 8192 14.8 / 12.7, 26.7 / 24.6; but 128 x 8192, k 4096 20.4 / 24.6, k 8192 26.7 / 38.0.  A scale
  // per column of B: 16 tiles k 4096 26.7 / 24.5, 24 tiles 41.0 / 24.6, 128 x 8192, k 8192 41.1 / 39.0.
  const int64_t pair_tiles = (int64_t)ceil_div(a.dim, 256) * ceil_div(b.dim, 256);
  if (!a.any_scales && !b.any_scales && pair_tiles > ctx().sm_count / 8 && pair_tiles <= 0x3fffffff && a.dim > 128 && b.dim > 128)
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
  // few tiles: k is cut into as many runs as bring two CTAs to every SM (a token through 1024 x 4096: 256 CTAs of one k-block)
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
  const bool any_a = (a_blocks & CLEAVE_SCALES_ANY) != 0, any_b = (b_blocks & CLEAVE_SCALES_ANY) != 0;
  a_blocks &= ~CLEAVE_SCALES_ANY;
  b_blocks &= ~CLEAVE_SCALES_ANY;
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
  const QSide sa{A.q, A.s, m, k, ta, a_blocks, any_a}, sb{B.q, B.s, n, k, tb ? 0 : 1, b_blocks, any_b};
  return gemm_q(sa, sb, C->ptr, bi ? bi->ptr : nullptr, act) ? CLEAVE_CUDA_OK : -cleave_cuda_last_error();
}

}  // extern "C"
