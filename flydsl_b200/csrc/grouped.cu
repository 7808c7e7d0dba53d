// Matrix products grouped by expert over ragged rows (16-bit operands), and their two gradients.
//
// Rows are in expert order without padding: expert e owns rows offsets[e] .. offsets[e+1]-1.
//   form 0   y[r, n]     = sum_k x[r, k]  w[e, n, k]        forward
//   form 1   dx[r, k]    = sum_n dy[r, n] w[e, n, k]        input gradient
//   form 2   dw[e, n, k] = sum_{r in e} dy[r, n] x[r, k]    weight gradient (an expert without rows gets zeros)
// 16-bit operands through TMA, fp32 accumulation in TMEM, one rounding at the end.  What changes between the forms is which
// axis of an operand is contiguous: form 0 reads both along the contraction (K-major tiles), form 1 the weights across it,
// form 2 both operands across it (MN-major tiles: 64-column chunks of 64 contraction rows, 128 bytes a row).  No operand is
// transposed in memory.
//
// This file: forms 0 and 1 on one CTA per tile, of 128 rows x 256 or 128 columns or, where most experts have few rows, of 32
// rows x 128 or 32 (form 1: 64) columns; all of form 2 and experts with many rows run on CTA pairs (grouped_pair.cu).  A tile
// may read rows of the next expert; they only reach accumulator rows that are not stored.  A 32-row tile loads 32 rows per K block; the MMAs
// have 128 and read on into whatever follows in shared memory, which reaches no stored row either.  What small launches need
// is bytes in flight (a K block takes about 2 us from its request to its release when the weights come from HBM), so their
// tiles are narrow and the ring is deep: one expert of 4096 x 4096 with one row takes 14 us, on 128-row tiles 23 to 28.  64 rows on 32
// experts of 4096 x 7168: 1.63 GB of weights in 249 to 306 us by box, 5.3 to 6.5 TB/s.
#include <cuda.h>
#include <stdio.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "gemm_ptx.cuh"
#include "grouped.cuh"

namespace flymoe {

constexpr int kRagThreads = 384;
constexpr int kRagMaxStages = 24;
constexpr int kRagStaging = 8 * 32 * 64;         // epilogue: 32 rows x 32 columns a warp
// K blocks of 64 that share a stage: handing a stage over costs the issuing thread about as much as five MMAs.
template <int TM> constexpr int rag_sub() { return TM == 128 ? 1 : 2; }
template <int TM, int BN> constexpr int rag_stage_bytes() { return (TM + BN) * kRagK * 2 * rag_sub<TM>(); }
// As many K blocks as fit beside the tables; behind the last one, what a 128-row read of a 32-row block reaches.
template <int TM, int BN> constexpr int rag_stages() {
  const int n = (232448 - 1024 - 9216 - kRagStaging - (128 - TM) * kRagK * 2) / rag_stage_bytes<TM, BN>();
  return n > kRagMaxStages ? kRagMaxStages : n;
}

struct __align__(16) RaggedCtrl {
  unsigned long long full[kRagMaxStages], empty[kRagMaxStages];
  unsigned long long acc_full[2];
  unsigned long long acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
  RaggedTables tab;
};
template <int TM, int BN> constexpr size_t rag_ring() {
  return size_t(rag_stages<TM, BN>()) * rag_stage_bytes<TM, BN>() + (128 - TM) * kRagK * 2 + kRagStaging;
}
static_assert(sizeof(RaggedCtrl) <= 9216, "shared memory budget of one SM exceeded");

template <int FORM, int TM, int BN>
__global__ void __launch_bounds__(kRagThreads, 1)
grouped_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                    const RaggedArgs a) {
  constexpr int kStages = rag_stages<TM, BN>(), kStageBytes = rag_stage_bytes<TM, BN>();
  constexpr int kSub = rag_sub<TM>(), kStageK = kRagK * kSub, kABytes = TM * kStageK * 2;
  constexpr int kTmem = 2 * BN < 32 ? 32 : 2 * BN;             // two accumulators
  constexpr int kWgs = BN >= 64 ? 2 : 1;                         // warpgroups of the epilogue that have columns
  static_assert(FORM == 0 || BN % 64 == 0, "columns across the contraction come 64 at a time");
  extern __shared__ uint8_t smem_dyn[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  RaggedCtrl* ctrl = reinterpret_cast<RaggedCtrl*>(smem + rag_ring<TM, BN>());
  volatile int* abort_flag = &ctrl->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 2) {
    ragged_tables<FORM, TM>(a, &ctrl->tab, lane);
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&ctrl->tmem_base)), "r"(uint32_t(kTmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&ctrl->full[i]), 1);
      mbar_init(smem_u32(&ctrl->empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctrl->acc_full[i]), 1);
      mbar_init(smem_u32(&ctrl->acc_empty[i]), 4 * kWgs);
    }
    ctrl->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = ctrl->tmem_base;
  const RaggedTables* tab = &ctrl->tab;
  const int total = tab->tile0[a.experts];
  const int KB = (a.k_dim + kStageK - 1) / kStageK;

  // Producer and issuer are one thread each, waits included: with a warp that waits together and elects a thread for every K
  // block the issuer took 490 cycles a block, whatever the tile.
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      RaggedTile tile;
      for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
        tile.at(a, tab, t, FORM);
        const int row0 = tab->start[tile.e] + tile.m * TM;
        for (int kb = 0; kb < KB; ++kb) {
          ok = mbar_wait(smem_u32(&ctrl->empty[stage]), phase ^ 1, abort_flag, a.status, 1, 32);
          if (!ok) break;
          const uint32_t full = smem_u32(&ctrl->full[stage]);
          const uint32_t sa = smem_u32(smem + size_t(stage) * kStageBytes), sb = sa + kABytes;
          mbar_expect_tx(full, kStageBytes);
#pragma unroll
          for (int h = 0; h < kSub; ++h) {
            const int k = kb * kStageK + h * kRagK;
            tma_load_2d(sa + h * TM * 128, &tmap_a, full, k * 2, row0);
            if (FORM == 0) tma_load_3d(sb + h * BN * 128, &tmap_b, full, k * 2, tile.n * BN, tile.e);
          }
          if (FORM == 1) {
#pragma unroll
            for (int j = 0; j < BN / 64; ++j)
              tma_load_3d(sb + j * kStageK * 128, &tmap_b, full, (tile.n * BN + j * 64) * 2, kb * kStageK, tile.e);
          }
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      const uint32_t idesc = ((a.bf16 ? kInstrDescBF16 : kInstrDescF16) - kInstrDescShape) | uint32_t(BN >> 3) << 17 |
                             uint32_t(128 >> 4) << 24 | (FORM != 0 ? 1u << 16 : 0u);
      const uint32_t base = smem_u32(smem);
      const uint64_t adesc0 = make_smem_desc(base);
      const uint64_t bdesc0 = FORM != 0 ? make_smem_desc_mn(base + kABytes, kStageK * 128) : make_smem_desc(base + kABytes);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
        ok = mbar_wait(smem_u32(&ctrl->acc_empty[acc]), acc_phase ^ 1, abort_flag, a.status, 2);
        const uint32_t d_tmem = tmem_base + uint32_t(acc) * BN;
        for (int kb = 0; kb < KB && ok; ++kb) {
          ok = mbar_wait(smem_u32(&ctrl->full[stage]), phase, abort_flag, a.status, 3);
          if (!ok) break;
          const uint64_t at = uint64_t(stage * (kStageBytes >> 4));
          tcgen05_fence_after();
#pragma unroll
          for (int k = 0; k < kStageK / 16; ++k) {
            const uint64_t ak = (k / 4) * (TM * 128 >> 4) + (k % 4) * 2;
            const uint64_t bk = FORM != 0 ? k * (16 * 128 >> 4) : (k / 4) * (BN * 128 >> 4) + (k % 4) * 2;
            umma_f16(d_tmem, adesc0 + at + ak, bdesc0 + at + bk, idesc, (k > 0 || kb > 0) ? 1u : 0u);
          }
          umma_commit(smem_u32(&ctrl->empty[stage]));
          if (kb + 1 == KB) umma_commit(smem_u32(&ctrl->acc_full[acc]));
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp >= 4 && warp < 4 + 4 * kWgs) {
    // ------------------------------------------------------------------ epilogue
    // A thread has a row of the tile; 32 columns at a time go through the warp's staging area and leave four lanes a row, 64
    // contiguous bytes.  Stored straight from the registers (16 bytes a row) a full 128 x 256 tile took as long as 30 K blocks.
    constexpr int kCols = BN / kWgs;
    const int wg = (warp - 4) >> 2;
    const uint32_t tcol = tmem_base + (uint32_t((warp & 3) * 32) << 16) + uint32_t(wg * kCols);
    uint8_t* stg = smem + rag_ring<TM, BN>() - kRagStaging + (warp - 4) * 32 * 64;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    RaggedTile tile;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      tile.at(a, tab, t, FORM);
      const int row0 = tab->start[tile.e] + tile.m * TM + (warp & 3) * 32;
      const int rows = min(min(32, TM - (warp & 3) * 32), tab->start[tile.e + 1] - row0);      // this warp's, if positive
      ok = warp_wait(smem_u32(&ctrl->acc_full[acc]), acc_phase, abort_flag, a.status, 4);
      if (!ok) break;
      tcgen05_fence_after();
      const uint32_t tc = tcol + uint32_t(acc) * BN;
#pragma unroll
      for (int q = 0; q < kCols / 32; ++q) {
        const int col = tile.n * BN + wg * kCols + q * 32;
        const bool wanted = rows > 0 && col < a.n_dim;
        float v[32];
        if (wanted) {
          tmem_ld_x32(tc + q * 32, reinterpret_cast<uint32_t*>(v));
          tmem_ld_wait();
        }
        if (q + 1 == kCols / 32) {
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&ctrl->acc_empty[acc]));
        }
        if (!wanted) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<uint4*>(stg + lane * 64 + ((j ^ ((lane >> 1) & 3)) * 16)) = pack8(v + j * 8, a.bf16);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i * 8 + (lane >> 2), c = lane & 3;
          if (r < rows && col + c * 8 < a.n_dim)
            *reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.out) + ((long long)(row0 + r) * a.n_dim + col + c * 8) * 2) =
                *reinterpret_cast<const uint4*>(stg + r * 64 + ((c ^ ((r >> 1) & 3)) * 16));
        }
        __syncwarp();
      }
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
    if (a.zero_uncovered) zero_uncovered_rows(a, tab, threadIdx.x - 128, 128 * kWgs);
  }

  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(uint32_t(kTmem)) : "memory");
  }
}

// ------------------------------------------------------------------------------ host
template <int FORM, int TM, int BN>
static int launch_ragged(const void* x, const void* w, RaggedArgs a, int n, int k, cudaStream_t stream) {
  a.n_tiles = ceil_div(a.n_dim, BN);
  CUtensorMap ma, mb;
  int rc = matrix_map(&ma, x, a.k_dim, a.rows, 0, TM);
  if (rc == FLYMOE_OK) rc = matrix_map(&mb, w, k, n, a.experts, FORM == 1 ? kRagK * rag_sub<TM>() : BN);
  if (rc != FLYMOE_OK) return rc;
  auto* kernel = grouped_gemm_kernel<FORM, TM, BN>;
  constexpr size_t smem = rag_ring<TM, BN>() + sizeof(RaggedCtrl) + 1024;
  static SmemLimitSeen seen;
  FLYMOE_CUDA_CHECK(allow_smem(reinterpret_cast<const void*>(kernel), int(smem), seen));
  const long long tiles = ((long long)a.rows / TM + std::min(a.rows, a.experts)) * a.n_tiles, sms = sm_count();
  kernel<<<unsigned(std::min(tiles, sms)), kRagThreads, smem, stream>>>(ma, mb, a);
  FLYMOE_CUDA_CHECK(cudaGetLastError());
  return FLYMOE_OK;
}

enum RaggedTileKind { kPairTile, kTile256, kTile128, kFew128, kFewNarrow };
// Row tiles that an expert with `mean` rows on average can be expected to have: the sum over j of the chance of more than
// j * tm rows, spread as by even routing with experts that differ by a quarter of the mean besides.
static double expected_tiles(double mean, int tm) {
  const double sd = std::sqrt(mean + 0.0625 * mean * mean);
  double sum = 1.0 - std::exp(-mean);
  for (int j = 1; j < 64; ++j) {
    const double p = 0.5 * std::erfc((j * double(tm) + 0.5 - mean) / (sd * 1.4142135623730951));
    if (p < 1e-4) return sum;
    sum += p;
  }
  return mean / tm + 0.5;
}
// Tile of forms 0 and 1, by estimated cycles.  A K block costs what is longest of its MMAs (with the issuing thread's work)
// and its bytes at 70 to 77 a cycle; that and the time on HBM hide each other only in part (root of the sum of squares).
// Over 154 sizes (1 to 64 experts, 1 to 700 rows each, even and skewed) the two forms took 1.014 and 1.011 of the time of the
// best kind on geometric mean, 1.38 at worst (16 experts of 1048 x 2104, whose rows are not aligned to 128 bytes).  A fixed kind
// takes 1.12 to 2.12 on geometric mean: pairs for one row on one expert of 4096 x 4096 25 us against 14, 128 x 256 tiles for 8
// experts of 2048 x 2048 with 40 rows 20 against 16, 32 x 128 tiles for 32 experts of 4096 x 7168 with 160 rows 953 against 438.
static RaggedTileKind choose_tile(bool input_grad, int rows, int experts, int n_dim, int k_dim) {
  const int narrow = input_grad ? 64 : 32;       // columns across the contraction come 64 at a time
  struct Kind { int tm, tn, per_sm_x2, block, launch; double hbm; };
  const Kind kinds[5] = {{256, 256, 1, 540, 9700, 1.15}, {128, 256, 2, 720, 8100, 1.0}, {128, 128, 2, 425, 7400, 1.03},
                         {32, 128, 2, 310, 7400, 1.0}, {32, narrow, 2, 250, 6400, 1.1}};
  const double blocks = ceil_div(k_dim, kRagK), used = std::min(rows, experts);
  const double hbm_cycles = 2.0 * (used * n_dim * k_dim + double(rows) * (double(n_dim) + k_dim)) * 2.9e-4;
  int best = 0;
  double least = 0;
  for (int i = 0; i < 5; ++i) {
    const Kind& q = kinds[i];
    const double tiles = std::max(1.0, experts * expected_tiles(double(rows) / experts, q.tm)) * ceil_div(n_dim, q.tn);
    const double waves = std::ceil(tiles / (0.5 * sm_count() * q.per_sm_x2));
    const double work = waves * (blocks * q.block + 400), wire = hbm_cycles * q.hbm;
    const double cost = q.launch + std::sqrt(work * work + wire * wire);
    if (i == 0 || cost < least) { best = i; least = cost; }
  }
  return RaggedTileKind(best);
}

static int ragged_common(RaggedArgs* a, const char* what, const void* out, const void* p, const void* q,
                         const int32_t* offsets, int rows, int experts, int n, int k, int dtype) {
  static thread_local char msg[160];
  auto fail = [&](const char* why) {
    snprintf(msg, sizeof(msg), "%s: %s", what, why);
    set_last_error_msg(msg);
    return FLYMOE_ERR_INVALID_ARGUMENT;
  };
  if (rows < 0) return fail("rows < 0");
  if (rows > kMostRows) return fail("rows must not exceed 2^31 - 1025");
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
  a.zero_uncovered = zero_uncovered;
  a.group_m = 8;
  FLYMOE_REQUIRE(((long long)rows / 32 + experts) * ceil_div(a.n_dim, 32) < (1LL << 31), "grouped_gemm: too many tiles");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define FLYMOE_RAGGED_CASE(TM, BN) input_grad ? launch_ragged<1, TM, BN>(x, w, a, n, k, s) : launch_ragged<0, TM, BN>(x, w, a, n, k, s)
  switch (choose_tile(input_grad, rows, experts, a.n_dim, a.k_dim)) {
    case kTile256: return FLYMOE_RAGGED_CASE(128, 256);
    case kTile128: return FLYMOE_RAGGED_CASE(128, 128);
    case kFew128: return FLYMOE_RAGGED_CASE(32, 128);
    case kFewNarrow: return input_grad ? launch_ragged<1, 32, 64>(x, w, a, n, k, s) : launch_ragged<0, 32, 32>(x, w, a, n, k, s);
    default: return launch_ragged_pair(input_grad ? 1 : 0, x, w, a, n, k, s);
  }
#undef FLYMOE_RAGGED_CASE
}

extern "C" int flymoe_grouped_gemm_tile(int rows, int experts, int n, int k, int input_grad) {
  using namespace flymoe;
  if (rows < 1 || experts < 1 || n < 8 || k < 8) return -1;
  return choose_tile(input_grad != 0, rows, experts, input_grad ? k : n, input_grad ? n : k);
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
  a.group_m = 8;
  FLYMOE_REQUIRE((long long)experts * ceil_div(n, 128) * ceil_div(k, 128) < (1LL << 31), "grouped_gemm_wgrad: too many tiles");
  return launch_ragged_pair(2, dy, x, a, n, k, s);
}
