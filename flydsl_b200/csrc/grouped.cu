// Matrix products grouped by expert over ragged rows (16-bit operands), and their two gradients.
//
// Rows are in expert order without padding: expert e owns rows offsets[e] .. offsets[e+1]-1.
//   form 0   y[r, n]     = sum_k x[r, k]  w[e, n, k]        forward
//   form 1   dx[r, k]    = sum_n dy[r, n] w[e, n, k]        input gradient
//   form 2   dw[e, n, k] = sum_{r in e} dy[r, n] x[r, k]    weight gradient (an expert without rows gets zeros)
// One kernel: 128 x 256 output tiles, K blocks of 64, fp32 accumulation in TMEM, one rounding at the end.  What changes is
// which axis of an operand is contiguous: form 0 reads both along the contraction (K-major tiles), form 1 the weights
// across it, form 2 both operands across it (MN-major tiles: 64-column chunks of 64 contraction rows, 128 bytes a row).
// No operand is transposed in memory.
//
// Ragged ends.  Forms 0 and 1: a tile may read rows of the next expert; they only reach accumulator rows that are not
// stored.  Form 2 contracts over the rows, so the last K block of an expert issues only the 16-row steps that hold rows of
// it, and of the last step the rows behind the end are overwritten with zeros in shared memory (both operands: what stands
// there may be infinite).
#include <cuda.h>
#include <stdio.h>
#include <stdlib.h>

#include "common.cuh"
#include "gemm_ptx.cuh"
#include "grouped.cuh"

namespace flymoe {

constexpr int kRagM = 128, kRagN = 256;
constexpr int kRagStages = 4;
constexpr int kRagStageBytes = (kRagM + kRagN) * kRagK * 2;      // 48 KB
constexpr int kRagThreads = 384;

struct __align__(16) RaggedCtrl {
  unsigned long long full[kRagStages];
  unsigned long long empty[kRagStages];
  unsigned long long acc_full[2];
  unsigned long long acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
  RaggedTables tab;
};
constexpr size_t kRagSmem = size_t(kRagStages) * kRagStageBytes + sizeof(RaggedCtrl) + 1024;
static_assert(kRagSmem <= 232448, "shared memory budget of one SM exceeded");

template <int FORM>
__global__ void __launch_bounds__(kRagThreads, 1)
grouped_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                    const RaggedArgs a) {
  extern __shared__ uint8_t smem_dyn[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  RaggedCtrl* ctrl = reinterpret_cast<RaggedCtrl*>(smem + size_t(kRagStages) * kRagStageBytes);
  volatile int* abort_flag = &ctrl->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr bool kAMn = FORM == 2, kBMn = FORM != 0;
  constexpr int kABytes = kRagM * kRagK * 2;

  if (warp == 2) {
    ragged_tables<FORM, kRagM>(a, &ctrl->tab, lane);
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&ctrl->tmem_base)), "r"(uint32_t(kTmemCols)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (threadIdx.x == 0) {
    for (int i = 0; i < kRagStages; ++i) {
      mbar_init(smem_u32(&ctrl->full[i]), 1);
      mbar_init(smem_u32(&ctrl->empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctrl->acc_full[i]), 1);
      mbar_init(smem_u32(&ctrl->acc_empty[i]), kEpilogueWarps);
    }
    ctrl->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = ctrl->tmem_base;
  const int total = ctrl->tab.tile0[a.experts];
  auto k_blocks = [&](int e) {
    return FORM == 2 ? (ctrl->tab.start[e + 1] - ctrl->tab.start[e] + kRagK - 1) / kRagK : (a.k_dim + kRagK - 1) / kRagK;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    RaggedTile tile;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      tile.at(a, &ctrl->tab, t, FORM);
      const int KB = k_blocks(tile.e), row0 = ctrl->tab.start[tile.e];
      for (int kb = 0; kb < KB; ++kb) {
        ok = warp_wait(smem_u32(&ctrl->empty[stage]), phase ^ 1, abort_flag, a.status, 1, 32);
        if (!ok) break;
        const uint32_t full = smem_u32(&ctrl->full[stage]);
        const uint32_t sa = smem_u32(smem + size_t(stage) * kRagStageBytes), sb = sa + kABytes;
        if (elect_one()) {
          mbar_expect_tx(full, kRagStageBytes);
          if (kAMn) {
#pragma unroll
            for (int j = 0; j < kRagM / 64; ++j)
              tma_load_2d(sa + j * kRagK * 128, &tmap_a, full, (tile.m * kRagM + j * 64) * 2, row0 + kb * kRagK);
          } else {
            tma_load_2d(sa, &tmap_a, full, kb * kRagK * 2, row0 + tile.m * kRagM);
          }
          if (FORM == 0) {
            tma_load_3d(sb, &tmap_b, full, kb * kRagK * 2, tile.n * kRagN, tile.e);
          } else {
#pragma unroll
            for (int j = 0; j < kRagN / 64; ++j) {
              const int col = (tile.n * kRagN + j * 64) * 2;
              if (FORM == 1) tma_load_3d(sb + j * kRagK * 128, &tmap_b, full, col, kb * kRagK, tile.e);
              else tma_load_2d(sb + j * kRagK * 128, &tmap_b, full, col, row0 + kb * kRagK);
            }
          }
        }
        __syncwarp();
        if (++stage == kRagStages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    const uint32_t idesc = (a.bf16 ? kInstrDescBF16 : kInstrDescF16) | (kAMn ? 1u << 15 : 0u) | (kBMn ? 1u << 16 : 0u);
    constexpr uint64_t a_step = kAMn ? (16 * 128) >> 4 : 2, b_step = kBMn ? (16 * 128) >> 4 : 2;
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    RaggedTile tile;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      int KB = (a.k_dim + kRagK - 1) / kRagK, seg = 0;
      if (FORM == 2) {
        tile.at(a, &ctrl->tab, t, FORM);
        KB = k_blocks(tile.e);
        seg = ctrl->tab.start[tile.e + 1] - ctrl->tab.start[tile.e];
        if (KB == 0) continue;                   // the epilogue writes zeros on its own
      }
      ok = warp_wait(smem_u32(&ctrl->acc_empty[acc]), acc_phase ^ 1, abort_flag, a.status, 2);
      const uint32_t d_tmem = tmem_base + uint32_t(acc) * kRagN;
      for (int kb = 0; kb < KB && ok; ++kb) {
        ok = warp_wait(smem_u32(&ctrl->full[stage]), phase, abort_flag, a.status, 3);
        if (!ok) break;
        uint8_t* sp = smem + size_t(stage) * kRagStageBytes;
        int steps = kRagK / 16;
        if (FORM == 2 && kb + 1 == KB && (seg & (kRagK - 1)) != 0) {
          const int have = seg & (kRagK - 1);    // rows of this expert in the block
          steps = (have + 15) / 16;
          zero_block_rows(sp, (kRagM + kRagN) / 64, have, steps * 16 - have, lane);
        }
        const uint32_t sa = smem_u32(sp);
        const uint64_t adesc = kAMn ? make_smem_desc_mn(sa, kRagK * 128) : make_smem_desc(sa);
        const uint64_t bdesc = kBMn ? make_smem_desc_mn(sa + kABytes, kRagK * 128) : make_smem_desc(sa + kABytes);
        tcgen05_fence_after();
        if (elect_one()) {
          for (int k = 0; k < steps; ++k)
            umma_f16(d_tmem, adesc + a_step * k, bdesc + b_step * k, idesc, (k > 0 || kb > 0) ? 1u : 0u);
          umma_commit(smem_u32(&ctrl->empty[stage]));
          if (kb + 1 == KB) umma_commit(smem_u32(&ctrl->acc_full[acc]));
        }
        __syncwarp();
        if (++stage == kRagStages) { stage = 0; phase ^= 1; }
      }
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ epilogue
    const int wg = (warp - 4) >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t tcol = tmem_base + (uint32_t((warp & 3) * 32) << 16) + uint32_t(wg * 128);
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    RaggedTile tile;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      tile.at(a, &ctrl->tab, t, FORM);
      const int e = tile.e, start = ctrl->tab.start[e], seg = ctrl->tab.start[e + 1] - start;
      const bool none = FORM == 2 && seg == 0;
      const int local = tile.m * kRagM + row;
      const bool valid = FORM == 2 ? local < a.m_dim : local < seg;
      const long long orow = FORM == 2 ? (long long)e * a.m_dim + local : (long long)start + local;
      const int col0 = tile.n * kRagN + wg * 128;
      uint8_t* op = static_cast<uint8_t*>(a.out) + (orow * a.n_dim + col0) * 2;
      const int cols = valid ? a.n_dim - col0 : 0;             // a multiple of 8
      if (none) {
        for (int j = 0; j < min(cols, 128); j += 8) *reinterpret_cast<uint4*>(op + j * 2) = make_uint4(0, 0, 0, 0);
        continue;
      }
      ok = warp_wait(smem_u32(&ctrl->acc_full[acc]), acc_phase, abort_flag, a.status, 4);
      if (!ok) break;
      tcgen05_fence_after();
      const uint32_t tc = tcol + uint32_t(acc) * kRagN;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float v[32];
        tmem_ld_x32(tc + q * 32, reinterpret_cast<uint32_t*>(v));
        tmem_ld_wait();
        if (q == 3) {
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&ctrl->acc_empty[acc]));
        }
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          if (q * 32 + j < cols) *reinterpret_cast<uint4*>(op + (q * 32 + j) * 2) = pack8(v + j, a.bf16);
        }
      }
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
    if (FORM != 2 && a.zero_uncovered) zero_uncovered_rows(a, &ctrl->tab, threadIdx.x - 128, 256);
  }

  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(uint32_t(kTmemCols))
                 : "memory");
  }
}

// ------------------------------------------------------------------------------ host
int ragged_map(CUtensorMap* map, const void* base, long long cols, long long rows, int mats, int box_rows) {
  cuuint64_t dims[3] = {cuuint64_t(cols) * 2, cuuint64_t(rows), cuuint64_t(mats)};
  cuuint64_t strides[2] = {cuuint64_t(cols) * 2, cuuint64_t(cols) * 2 * cuuint64_t(rows)};
  cuuint32_t box[3] = {128, cuuint32_t(box_rows), 1};
  return make_map(map, base, mats > 0 ? 3 : 2, dims, strides, box);
}

template <int FORM>
static int launch_ragged(const CUtensorMap& ma, const CUtensorMap& mb, const RaggedArgs& a, long long max_tiles,
                         cudaStream_t stream) {
  auto* kernel = grouped_gemm_kernel<FORM>;
  static SmemLimitSeen seen;
  FLYMOE_CUDA_CHECK(allow_smem(reinterpret_cast<const void*>(kernel), int(kRagSmem), seen));
  const long long sms = sm_count();
  kernel<<<unsigned(max_tiles < sms ? max_tiles : sms), kRagThreads, kRagSmem, stream>>>(ma, mb, a);
  FLYMOE_CUDA_CHECK(cudaGetLastError());
  return FLYMOE_OK;
}

static int envint(const char* n, int d) { const char* e = getenv(n); return e ? atoi(e) : d; }
static bool use_pairs(int rows, int experts) { return rows >= envint("PAIR", 128) * experts; }

static int ragged_common(RaggedArgs* a, const char* what, const void* out, const void* p, const void* q,
                         const int32_t* offsets, int rows, int experts, int n, int k, int dtype) {
  static thread_local char msg[160];
  auto fail = [&](const char* why) {
    snprintf(msg, sizeof(msg), "%s: %s", what, why);
    set_last_error_msg(msg);
    return FLYMOE_ERR_INVALID_ARGUMENT;
  };
  if (rows < 0) return fail("rows < 0");
  if (experts < 1 || experts > kRagMaxExperts) return fail("experts must be in [1, 1024]");
  if (n < 8 || n % 8 || k < 8 || k % 8) return fail("n and k must be positive multiples of 8");
  // the tensor maps count bytes and the kernels columns in 32 bits
  if (n > (1 << 29) || k > (1 << 29)) return fail("n and k must not exceed 2^29");
  if (dtype != FLYMOE_BF16 && dtype != FLYMOE_F16) return fail("dtype must be F16 or BF16");
  if (!offsets || (rows > 0 && (!out || !p || !q))) return fail("null pointer");
  if (!aligned16(out) || !aligned16(p) || !aligned16(q)) return fail("pointers must be 16-byte aligned");
  a->offsets = offsets;
  a->out = const_cast<void*>(out);
  a->rows = rows;
  a->experts = experts;
  a->bf16 = dtype == FLYMOE_BF16;
  a->status = device_status_ptr();
  if (a->status == nullptr) return fail("no CUDA device");
  return FLYMOE_OK;
}

}  // namespace flymoe

extern "C" int flymoe_grouped_gemm(void* out, const void* x, const void* w, const int32_t* offsets, int rows, int experts,
                                   int n, int k, int dtype, int input_grad, int zero_uncovered, void* stream) {
  using namespace flymoe;
  RaggedArgs a = {};
  int rc = ragged_common(&a, "grouped_gemm", out, x, w, offsets, rows, experts, n, k, dtype);
  if (rc != FLYMOE_OK || rows == 0) return rc;
  a.n_dim = input_grad ? k : n;
  a.k_dim = input_grad ? n : k;
  a.n_tiles = ceil_div(a.n_dim, kRagN);
  a.m_tiles = 0;
  a.zero_uncovered = zero_uncovered;
  a.group_m = 8;
  const long long max_tiles = ((long long)rows / kRagM + experts) * a.n_tiles;
  FLYMOE_REQUIRE(max_tiles < (1LL << 31), "grouped_gemm: too many tiles");
  if (use_pairs(rows, experts)) return launch_ragged_pair(input_grad ? 1 : 0, x, w, a, n, k, static_cast<cudaStream_t>(stream));
  CUtensorMap ma, mb;
  if ((rc = ragged_map(&ma, x, a.k_dim, rows, 0, kRagM)) != FLYMOE_OK) return rc;
  if ((rc = ragged_map(&mb, w, k, n, experts, input_grad ? kRagK : kRagN)) != FLYMOE_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return input_grad ? launch_ragged<1>(ma, mb, a, max_tiles, s) : launch_ragged<0>(ma, mb, a, max_tiles, s);
}

extern "C" int flymoe_grouped_gemm_wgrad(void* dw, const void* dy, const void* x, const int32_t* offsets, int rows,
                                         int experts, int n, int k, int dtype, void* stream) {
  using namespace flymoe;
  RaggedArgs a = {};
  int rc = ragged_common(&a, "grouped_gemm_wgrad", dw, dy, x, offsets, rows, experts, n, k, dtype);
  if (rc != FLYMOE_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    FLYMOE_REQUIRE(dw != nullptr, "grouped_gemm_wgrad: null pointer");
    FLYMOE_CUDA_CHECK(cudaMemsetAsync(dw, 0, size_t(experts) * n * k * 2, s));
    return FLYMOE_OK;
  }
  a.m_dim = n;
  a.n_dim = k;
  a.m_tiles = ceil_div(n, kRagM);
  a.n_tiles = ceil_div(k, kRagN);
  a.group_m = 8;
  const long long max_tiles = (long long)experts * a.m_tiles * a.n_tiles;
  FLYMOE_REQUIRE(max_tiles < (1LL << 31), "grouped_gemm_wgrad: too many tiles");
  if (use_pairs(rows, experts)) return launch_ragged_pair(2, dy, x, a, n, k, s);
  CUtensorMap ma, mb;
  if ((rc = ragged_map(&ma, dy, n, rows, 0, kRagK)) != FLYMOE_OK) return rc;
  if ((rc = ragged_map(&mb, x, k, rows, 0, kRagK)) != FLYMOE_OK) return rc;
  return launch_ragged<2>(ma, mb, a, max_tiles, s);
}
