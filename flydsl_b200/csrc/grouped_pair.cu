// Ragged grouped products on CTA pairs (tcgen05 cta_group::2): tiles of 256 x 256 for experts with many rows.
//
// Each CTA of a pair brings 128 rows of A and 128 rows (or columns) of B into shared memory, 32 KB per K block of 64, and the
// leader's MMAs read both halves.  The one-CTA kernel (grouped.cu) needs 48 KB for half the work: at the 64 bytes a cycle
// that an SM takes from L2 those are 768 cycles per K block against 512 of MMA, and that is what it measures.
//   warp 0      TMA producer; both CTAs' operands complete on the leader's barrier
//   warp 1      (leader) MMA issuer, two accumulators of 256 columns
//   warp 2      segment tables
//   warps 4-11  epilogue, two warpgroups with 128 columns each: 64 columns at a time to shared memory and out by one tiled
//               store (rows of another expert in the tile: by plain stores of the valid rows)
//
// Last K block of the weight gradient.  Its rows behind the expert's end have to be zero in both CTAs before the leader's
// MMAs read them.  The block is put together from boxes of 16, 8, 4, 2 and 1 rows that end with the expert, and the rest of
// the last 16-row step from boxes that lie behind the matrix, which the copy unit fills with zeros.  A warp that zeroes the
// rows in shared memory and reports to the leader across the cluster held the MMAs up instead: 32 experts of 1000 rows,
// 4096 x 7168, bf16 1479 us, with 1024 rows each 1358 us.
//
// Every wait is bounded as in the other kernels.  Epilogue warps keep step with one another on hardware barriers, so after a
// wait that ran out they walk on through their tiles without storing instead of leaving.
#include <cuda.h>

#include <algorithm>

#include "common.cuh"
#include "gemm_ptx.cuh"
#include "grouped.cuh"

namespace flymoe {

constexpr int kRpTile = 256;
constexpr int kRpHalf = 128 * kRagK * 2;                         // 16 KB: one operand of one CTA and K block
constexpr int kRpStageBytes = 2 * kRpHalf;
constexpr int kRpThreads = 384;
constexpr int kRpStaging = 128 * 128;                            // 128 rows x 64 columns of output per warpgroup
// Staging areas of a warpgroup, and operand stages.  AREAS == 2: the weight gradient of experts with few rows, whose tiles
// take more time to write than to sum up.  bf16, one area and five stages / two and four: 64 experts of 64 rows, 2048 x 2048,
// 145 / 131 us; 16 of 192, 2112 x 1088, 26.6 / 24.6; 8 of 500, 4096 x 4096, 150 / 146; 32 of 1024, 7168 x 4096, 1282 / 1370.
constexpr int rp_stages(int areas) { return areas == 2 ? 4 : 5; }

struct __align__(16) RagPairCtrl {
  unsigned long long full[5], empty[5];
  unsigned long long acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
  RaggedTables tab;
};
constexpr size_t rp_smem(int areas) {
  return size_t(rp_stages(areas)) * kRpStageBytes + 2 * areas * kRpStaging + sizeof(RagPairCtrl) + 1024;
}
static_assert(rp_smem(1) <= 232448 && rp_smem(2) <= 232448, "shared memory budget of one SM exceeded");

// Boxes of 64 columns and 16, 8, 4, 2, 1 rows of both operands: the weight gradient's last K blocks.
constexpr int kTailBoxes = 5;
struct TailMaps { CUtensorMap a[kTailBoxes], b[kTailBoxes]; };

// Rows [row, row + have) of a matrix of `rows` rows, and zeros up to the next multiple of 16, into a 64-column chunk.
__device__ __forceinline__ void load_tail(uint32_t dst, const CUtensorMap* maps, uint32_t bar, int col, int row, int have, int rows) {
  int at = 0;
  for (int part = 0; part < 2; ++part) {
    const int end = part == 0 ? have : (have + 15) / 16 * 16;
    const int shift = part == 0 ? row : rows;                    // second part: behind the last row, read as zeros
    for (int i = 0; i < kTailBoxes; ++i)
      for (; at + (16 >> i) <= end; at += 16 >> i) tma_load_2d_pair(dst + at * 128, maps + i, bar, col, shift + at);
  }
}

template <int FORM, int AREAS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kRpThreads, 1)
grouped_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                    const __grid_constant__ CUtensorMap tmap_out, const __grid_constant__ TailMaps tails, const RaggedArgs a) {
  extern __shared__ uint8_t smem_dyn[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  constexpr int kRpStages = rp_stages(AREAS);
  uint8_t* staging = smem + size_t(kRpStages) * kRpStageBytes;
  RagPairCtrl* ctrl = reinterpret_cast<RagPairCtrl*>(staging + 2 * AREAS * kRpStaging);
  volatile int* abort_flag = &ctrl->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = int(cluster_rank());
  constexpr bool kAMn = FORM == 2, kBMn = FORM != 0;

  if (warp == 2) {
    ragged_tables<FORM, kRpTile>(a, &ctrl->tab, lane);
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&ctrl->tmem_base)), "r"(uint32_t(kTmemCols)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else if (threadIdx.x == 0) {
    for (int i = 0; i < kRpStages; ++i) {
      mbar_init(smem_u32(&ctrl->full[i]), 1);
      mbar_init(smem_u32(&ctrl->empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctrl->acc_full[i]), 1);
      mbar_init(smem_u32(&ctrl->acc_empty[i]), 2 * kEpilogueWarps);
    }
    ctrl->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();                            // both CTAs' barriers and TMEM exist
  tcgen05_fence_after();
  const uint32_t tmem_base = ctrl->tmem_base;
  const RaggedTables* tab = &ctrl->tab;
  const int total = tab->tile0[a.experts];
  const int first = int(blockIdx.x) >> 1, step = int(gridDim.x) >> 1;
  const int k_blocks = (a.k_dim + kRagK - 1) / kRagK;
  auto rows_of = [&](int e) { return tab->start[e + 1] - tab->start[e]; };

  // Producer and issuer are one thread each, waits included (see grouped.cu).
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      RaggedTile tile;
      for (int t = first; t < total && ok; t += step) {
        tile.at(a, tab, t, FORM);
        const int seg = rows_of(tile.e), row0 = tab->start[tile.e], rest = seg & (kRagK - 1);
        const int KB = FORM == 2 ? (seg + kRagK - 1) / kRagK : k_blocks;
        for (int kb = 0; kb < KB; ++kb) {
          ok = mbar_wait(smem_u32(&ctrl->empty[stage]), phase ^ 1, abort_flag, a.status, 1, 32);
          if (!ok) break;
          const uint32_t sa = smem_u32(smem + size_t(stage) * kRpStageBytes), sb = sa + kRpHalf;
          const bool tail = FORM == 2 && kb + 1 == KB && rest != 0;
          // the leader announces the bytes of both CTAs; the other's may land before that
          const uint32_t bar = map_to_rank(smem_u32(&ctrl->full[stage]), 0);
          if (rank == 0)
            mbar_expect_tx(smem_u32(&ctrl->full[stage]), 2 * (tail ? (rest + 15) / 16 * 16 * 4 * 128 : kRpStageBytes));
          const int acol = (tile.m * kRpTile + rank * 128) * 2, bcol = (tile.n * kRpTile + rank * 128) * 2;
          if (tail) {
            for (int j = 0; j < 2; ++j) {
              load_tail(sa + j * kRagK * 128, tails.a, bar, acol + j * 128, row0 + kb * kRagK, rest, a.rows);
              load_tail(sb + j * kRagK * 128, tails.b, bar, bcol + j * 128, row0 + kb * kRagK, rest, a.rows);
            }
          } else if (FORM == 2) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              tma_load_2d_pair(sa + j * kRagK * 128, &tmap_a, bar, acol + j * 128, row0 + kb * kRagK);
              tma_load_2d_pair(sb + j * kRagK * 128, &tmap_b, bar, bcol + j * 128, row0 + kb * kRagK);
            }
          } else {
            tma_load_2d_pair(sa, &tmap_a, bar, kb * kRagK * 2, row0 + tile.m * kRpTile + rank * 128);
            if (FORM == 0) {
              tma_load_3d_pair(sb, &tmap_b, bar, kb * kRagK * 2, tile.n * kRpTile + rank * 128, tile.e);
            } else {
#pragma unroll
              for (int j = 0; j < 2; ++j) tma_load_3d_pair(sb + j * kRagK * 128, &tmap_b, bar, bcol + j * 128, kb * kRagK, tile.e);
            }
          }
          if (++stage == kRpStages) { stage = 0; phase ^= 1; }
        }
      }
      // the last releases of the ring are the leader's MMAs arriving in both CTAs: they have to land before this CTA's shared
      // memory goes away
      for (int i = 0; i < kRpStages && ok; ++i) {
        ok = mbar_wait(smem_u32(&ctrl->empty[stage]), phase ^ 1, abort_flag, a.status, 1, 32);
        if (++stage == kRpStages) { stage = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      const uint32_t idesc = ((a.bf16 ? kInstrDescBF16 : kInstrDescF16) - kInstrDescShape) | uint32_t(kRpTile >> 3) << 17 |
                             uint32_t(kRpTile >> 4) << 24 | (kAMn ? 1u << 15 : 0u) | (kBMn ? 1u << 16 : 0u);
      constexpr uint64_t a_step = kAMn ? (16 * 128) >> 4 : 2, b_step = kBMn ? (16 * 128) >> 4 : 2;
      const uint32_t base = smem_u32(smem);
      const uint64_t adesc0 = kAMn ? make_smem_desc_mn(base, kRagK * 128) : make_smem_desc(base);
      const uint64_t bdesc0 = kBMn ? make_smem_desc_mn(base + kRpHalf, kRagK * 128) : make_smem_desc(base + kRpHalf);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      RaggedTile tile;
      for (int t = first; t < total && ok; t += step) {
        int KB = k_blocks, rest = 0;
        if (FORM == 2) {
          tile.at(a, tab, t, FORM);
          const int seg = rows_of(tile.e);
          KB = (seg + kRagK - 1) / kRagK;
          rest = seg & (kRagK - 1);
          if (KB == 0) continue;                 // the epilogue writes zeros on its own
        }
        ok = mbar_wait(smem_u32(&ctrl->acc_empty[acc]), acc_phase ^ 1, abort_flag, a.status, 2);
        const uint32_t d_tmem = tmem_base + uint32_t(acc) * kRpTile;
        for (int kb = 0; kb < KB && ok; ++kb) {
          ok = mbar_wait_cluster(smem_u32(&ctrl->full[stage]), phase, abort_flag, a.status, 3);
          if (!ok) break;
          const uint64_t at = uint64_t(stage * (kRpStageBytes >> 4));
          const int steps = FORM == 2 && kb + 1 == KB && rest != 0 ? (rest + 15) / 16 : kRagK / 16;
          tcgen05_fence_after();
#pragma unroll
          for (int k = 0; k < kRagK / 16; ++k)
            if (FORM != 2 || k < steps)
              umma_pair<2>(d_tmem, adesc0 + at + a_step * k, bdesc0 + at + b_step * k, idesc, (k > 0 || kb > 0) ? 1u : 0u);
          umma_commit_pair(smem_u32(&ctrl->empty[stage]));
          if (kb + 1 == KB) umma_commit_pair(smem_u32(&ctrl->acc_full[acc]));
          if (++stage == kRpStages) { stage = 0; phase ^= 1; }
        }
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ epilogue
    const int wg = (warp - 4) >> 2, tid = threadIdx.x - 128 - wg * 128;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t tcol = tmem_base + (uint32_t((warp & 3) * 32) << 16) + uint32_t(wg * 128);
    const uint32_t empty_bar = map_to_rank(smem_u32(&ctrl->acc_empty[0]), 0);
    uint8_t* stg = staging + wg * AREAS * kRpStaging;
    int area = 0;
    const int sw = row & 7;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    RaggedTile tile;
    for (int t = first; t < total; t += step) {
      tile.at(a, tab, t, FORM);
      const int e = tile.e, seg = rows_of(e);
      const int m0 = tile.m * kRpTile + rank * 128;              // first row of this CTA inside the expert's output
      const int rows = max(0, min(128, (FORM == 2 ? a.m_dim : seg) - m0));
      const long long row0 = FORM == 2 ? (long long)e * a.m_dim + m0 : (long long)tab->start[e] + m0;
      const bool none = FORM == 2 && seg == 0;
      if (!none) {
        // a sum takes as long as its K blocks do, 0.29 us each (2^27 rows of 8 + 8 columns): the limit of a wait grows with them
        const unsigned long long limit = kWaitLimitNs + (FORM == 2 ? seg / kRagK * 4000ull : 0ull);
        ok = ok && warp_wait(smem_u32(&ctrl->acc_full[acc]), acc_phase, abort_flag, a.status, 4, 0, limit);
        tcgen05_fence_after();
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int col = tile.n * kRpTile + wg * 128 + q * 64;
        const bool wanted = rows > 0 && col < a.n_dim;           // the same in the whole warpgroup
        float v[64];
        if (wanted && !none) {
          tmem_ld_x32(tcol + uint32_t(acc) * kRpTile + q * 64, reinterpret_cast<uint32_t*>(v));
          tmem_ld_x32(tcol + uint32_t(acc) * kRpTile + q * 64 + 32, reinterpret_cast<uint32_t*>(v + 32));
          tmem_ld_wait();
        }
        if (q == 1 && !none) {
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_relaxed_cluster(empty_bar + uint32_t(acc) * 8u);
        }
        if (!wanted) continue;
        if (AREAS == 2) {
          area ^= kRpStaging;
          stg = staging + wg * AREAS * kRpStaging + area;
        }
        uint8_t* line = stg + row * 128;
        // the staging area's last store has been read out
        if (tid == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(AREAS - 1) : "memory");
        asm volatile("bar.sync %0, 128;" ::"r"(1 + wg) : "memory");
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint4*>(line + ((j ^ sw) * 16)) = none ? make_uint4(0, 0, 0, 0) : pack8(v + j * 8, a.bf16);
        const bool tiled = FORM == 2 || rows == 128;             // form 2: the map ends with the expert's matrix
        if (tiled) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("bar.sync %0, 128;" ::"r"(1 + wg) : "memory");
        if (tiled) {
          if (tid == 0 && ok) {
            if (FORM == 2) tma_store_3d(&tmap_out, smem_u32(stg), col * 2, m0, e);
            else tma_store_2d(&tmap_out, smem_u32(stg), col * 2, int(row0));
            bulk_commit();
          }
        } else if (ok) {
          for (int i = tid; i < rows * 8; i += 128) {
            const int r = i >> 3, c = i & 7;
            if (col + c * 8 < a.n_dim)
              *reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.out) + ((row0 + r) * a.n_dim + col + c * 8) * 2) =
                  *reinterpret_cast<const uint4*>(stg + r * 128 + ((c ^ (r & 7)) * 16));
          }
        }
      }
      if (!none && ++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
    if (tid == 0) bulk_wait_all();
    if (FORM != 2 && a.zero_uncovered) zero_uncovered_rows(a, tab, threadIdx.x - 128, 256);
  }

  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();                            // no remote arrival or MMA is outstanding when a CTA leaves
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(uint32_t(kTmemCols))
                 : "memory");
  }
}

// ------------------------------------------------------------------------------ host
template <int FORM, int AREAS>
static int launch_pair_form(const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mo, const TailMaps& tails,
                            const RaggedArgs& a, long long max_tiles, cudaStream_t stream) {
  auto* kernel = grouped_pair_kernel<FORM, AREAS>;
  static SmemLimitSeen seen;
  FLYMOE_CUDA_CHECK(allow_smem(reinterpret_cast<const void*>(kernel), int(rp_smem(AREAS)), seen));
  const unsigned pairs = unsigned(std::min<long long>(max_tiles, sm_count() / 2));
  kernel<<<2 * pairs, kRpThreads, rp_smem(AREAS), stream>>>(ma, mb, mo, tails, a);
  FLYMOE_CUDA_CHECK(cudaGetLastError());
  return FLYMOE_OK;
}

int launch_ragged_pair(int form, const void* p, const void* q, const RaggedArgs& args, int n, int k, cudaStream_t stream) {
  RaggedArgs a = args;
  a.n_tiles = ceil_div(a.n_dim, kRpTile);
  if (form == 2) a.m_tiles = ceil_div(a.m_dim, kRpTile);
  CUtensorMap ma, mb, mo;
  TailMaps tails = {};
  int rc;
  if (form == 2) {
    rc = matrix_map(&ma, p, n, a.rows, 0, kRagK);
    if (rc == FLYMOE_OK) rc = matrix_map(&mb, q, k, a.rows, 0, kRagK);
    if (rc == FLYMOE_OK) rc = matrix_map(&mo, a.out, a.n_dim, a.m_dim, a.experts, 128);
    for (int i = 0; i < kTailBoxes && rc == FLYMOE_OK; ++i) {
      rc = matrix_map(&tails.a[i], p, n, a.rows, 0, 16 >> i);
      if (rc == FLYMOE_OK) rc = matrix_map(&tails.b[i], q, k, a.rows, 0, 16 >> i);
    }
    const long long tiles = (long long)a.experts * a.m_tiles * a.n_tiles;
    if (rc != FLYMOE_OK) return rc;
    return a.rows / a.experts <= 512 ? launch_pair_form<2, 2>(ma, mb, mo, tails, a, tiles, stream)
                                     : launch_pair_form<2, 1>(ma, mb, mo, tails, a, tiles, stream);
  }
  rc = matrix_map(&ma, p, a.k_dim, a.rows, 0, 128);
  if (rc == FLYMOE_OK) rc = matrix_map(&mb, q, k, n, a.experts, form == 1 ? kRagK : 128);
  if (rc == FLYMOE_OK) rc = matrix_map(&mo, a.out, a.n_dim, a.rows, 0, 128);
  if (rc != FLYMOE_OK) return rc;
  const long long tiles = ((long long)a.rows / kRpTile + a.experts) * a.n_tiles;
  return form == 1 ? launch_pair_form<1, 1>(ma, mb, mo, tails, a, tiles, stream)
                   : launch_pair_form<0, 1>(ma, mb, mo, tails, a, tiles, stream);
}

}  // namespace flymoe
