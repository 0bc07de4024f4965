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
constexpr int kQRingBudget = 104 * 1024;     // two CTAs fit an SM
constexpr int kQMaxSplit = 8;                // portable cluster size

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
  // scale of element i of a side in k-block kb: s[kb * s_k + i * s_i + (i / 128) * s_b]
  const float *sp, *sq;
  int64_t sp_k, sq_k;
  int sp_i, sq_i;
  int64_t sp_b, sq_b;
  int stages;
  uint32_t stage_bytes;
  DeviceStatus* status;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float load_cluster_f32(uint32_t smem_addr, uint32_t rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
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
  __shared__ __align__(16) float s_scale[T::kDrainWarps][T::kCols];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
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

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(smem_u32(&bar_empty[stage]), phase ^ 1u, &abort_flag)) {
          report(p.status, 1, 1100 + stage, kb);
          ok = false;
          break;
        }
        const uint32_t full = smem_u32(&bar_full[stage]);
        mbar_arrive_expect_tx(full, p.stage_bytes);
        const uint32_t sp = ring + stage * p.stage_bytes;
        if (p.p_mn) tma_load_2d(sp, &map_p, full, pt * 128, kb * 128);
        else tma_load_2d(sp, &map_p, full, kb * 128, pt * 128);
        if (p.q_mn) tma_load_2d(sp + kQStageP, &map_q, full, qt * BNQ, kb * 128);
        else tma_load_2d(sp + kQStageP, &map_q, full, kb * 128, qt * BNQ);
        ++issued;
        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
      }
      if (!ok) {
        // leaving early: give the copies in flight a bounded chance to land
        for (int s = 0; s < p.stages; ++s) {
          const int fills = (issued + p.stages - 1 - s) / p.stages;   // how often stage s was filled
          if (fills == 0) continue;
          for (int spin = 0; spin < (1 << 20); ++spin)
            if (mbar_try_wait(smem_u32(&bar_full[s]), (uint32_t)(fills - 1) & 1u)) break;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = instr_desc_e4m3(p.p_mn, p.q_mn, 128, BNQ);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(smem_u32(&bar_tmem_empty[acc]), acc_phase ^ 1u, &abort_flag)) {
          report(p.status, 2, 1200 + acc, kb);
          break;
        }
        if (!mbar_wait(smem_u32(&bar_full[stage]), phase, &abort_flag)) {
          report(p.status, 3, 1300 + stage, kb);
          break;
        }
        tcgen05_fence_after();
        const uint32_t sp = ring + stage * p.stage_bytes;
        const uint32_t d = tmem_base + (uint32_t)(acc * BNQ);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_e4m3(d, operand_desc(sp, p.p_mn, kk), operand_desc(sp + kQStageP, p.q_mn, kk), idesc, kk ? 1u : 0u);
        tcgen05_commit(smem_u32(&bar_empty[stage]));
        tcgen05_commit(smem_u32(&bar_tmem_full[acc]));
        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
      }
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2, dw = warp - 2;
    int pi = pt * 128 + quarter * 32 + lane;
    if (pi >= p.p_dim) pi = p.p_dim - 1;   // a row outside C: any scale will do
    const float* sp = p.sp + (int64_t)pi * p.sp_i + (int64_t)(pi >> 7) * p.sp_b;
    const int q0 = qt * BNQ + half * T::kCols;
    constexpr int kPer = QVEC ? (T::kCols + 31) / 32 : 1;
    const float* sq[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      int qi = QVEC ? q0 + lane + 32 * i : q0;
      if (qi >= p.q_dim) qi = p.q_dim - 1;
      sq[i] = p.sq + (int64_t)qi * p.sq_i + (int64_t)(qi >> 7) * p.sq_b;
    }
    float acc_sum[T::kCols];
#pragma unroll
    for (int j = 0; j < T::kCols; ++j) acc_sum[j] = 0.0f;
    float next_p = __ldg(sp + (int64_t)kb0 * p.sp_k), next_q[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) next_q[i] = __ldg(sq[i] + (int64_t)kb0 * p.sq_k);
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      const float cur_p = next_p;
      float cur_q = next_q[0];
      if constexpr (QVEC) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (lane + 32 * i < T::kCols) s_scale[dw][lane + 32 * i] = next_q[i];
        __syncwarp();
      }
      if (kb + 1 < kb1) {   // the next block's scales travel while this one is drained
        next_p = __ldg(sp + (int64_t)(kb + 1) * p.sp_k);
#pragma unroll
        for (int i = 0; i < kPer; ++i) next_q[i] = __ldg(sq[i] + (int64_t)(kb + 1) * p.sq_k);
      }
      bool ok = mbar_wait(smem_u32(&bar_tmem_full[acc]), acc_phase, &abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        if (lane == 0) report(p.status, 4, 1400 + acc, kb);
        break;
      }
      tcgen05_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * BNQ + half * T::kCols);
      const float both = __fmul_rn(cur_p, cur_q);
#pragma unroll
      for (int g = 0; g < T::kCols / 16; ++g) {
        uint32_t r[16];
        tmem_ld_16(taddr + g * 16, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if constexpr (QVEC)
            acc_sum[g * 16 + j] = __fmaf_rn(__fmul_rn(__uint_as_float(r[j]), cur_p), s_scale[dw][g * 16 + j], acc_sum[g * 16 + j]);
          else
            acc_sum[g * 16 + j] = __fmaf_rn(__uint_as_float(r[j]), both, acc_sum[g * 16 + j]);
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_tmem_empty[acc]));
      if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
    }
    // Every load has landed and every MMA has read it: the ring is free for the partial sums.
#pragma unroll
    for (int j = 0; j < T::kCols; ++j)
      red[(quarter * 32 + lane) * kRedPitch + half * T::kCols + j] = acc_sum[j];
  }

  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if (ranks > 1) cluster_barrier();
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
    cluster_barrier();   // the peers are done with this CTA's shared memory
  }
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)T::kTmem) : "memory");
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

// Strides of a side's scales (QGemmParams).  Vector blocks run along k whichever way the operand is stored.
static void side_scales(const QSide& o, int64_t* s_k, int* s_i, int64_t* s_b) {
  if (o.blocks == CLEAVE_BLOCKS_TILES) {
    *s_i = 0;
    *s_k = o.mn ? ceil_div(o.dim, kQBlock) : 1;
    *s_b = o.mn ? 1 : ceil_div(o.k, kQBlock);
  } else {
    *s_i = 1;
    *s_k = o.dim;
    *s_b = 0;
  }
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

static bool gemm_q(const QSide& a, const QSide& b, float* c, const float* bias, int act) {
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
  p.sp = P.s;
  p.sq = Q.s;
  side_scales(P, &p.sp_k, &p.sp_i, &p.sp_b);
  side_scales(Q, &p.sq_k, &p.sq_i, &p.sq_b);
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
