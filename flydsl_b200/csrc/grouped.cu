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

#include "common.cuh"
#include "gemm_ptx.cuh"

namespace flymoe {

constexpr int kRagM = 128, kRagN = 256, kRagK = 64;
constexpr int kRagStages = 4;
constexpr int kRagStageBytes = (kRagM + kRagN) * kRagK * 2;      // 48 KB
constexpr int kRagMaxExperts = 1024;
constexpr int kRagThreads = 384;

struct RaggedArgs {
  const int* offsets;          // [experts + 1]
  void* out;
  int rows, experts;
  int m_dim;                   // form 2: rows of an expert's output matrix
  int n_dim;                   // columns of the output
  int k_dim;                   // forms 0 and 1: length of the contraction
  int n_tiles, m_tiles;        // m_tiles: form 2 only
  int group_m;
  int bf16, zero_uncovered;
  int* status;
};

struct __align__(16) RaggedCtrl {
  unsigned long long full[kRagStages];
  unsigned long long empty[kRagStages];
  unsigned long long acc_full[2];
  unsigned long long acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
  int start[kRagMaxExperts + 1];                 // first row of an expert
  int tile0[kRagMaxExperts + 1];                 // first tile of an expert
};
constexpr size_t kRagSmem = size_t(kRagStages) * kRagStageBytes + sizeof(RaggedCtrl) + 1024;
static_assert(kRagSmem <= 232448, "shared memory budget of one SM exceeded");

// Segment bounds and tile counts.  Offsets come from the device, so they are taken into [0, rows] and made ascending
// here: whatever they hold, no access leaves the tensors.
template <int FORM>
__device__ __forceinline__ void ragged_tables(const RaggedArgs& a, RaggedCtrl* c, int lane) {
  int run = 0, tiles = 0;
  for (int e0 = 0; e0 <= a.experts; e0 += 32) {
    const int e = e0 + lane;
    int v = e <= a.experts ? min(max(__ldg(a.offsets + e), 0), a.rows) : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, v, off);
      if (lane >= off) v = max(v, o);
    }
    v = max(v, run);
    // tiles of expert e - 1 are known once its end is
    int before = __shfl_up_sync(0xffffffffu, v, 1);
    if (lane == 0) before = run;
    int t = 0;
    if (e >= 1 && e <= a.experts)
      t = FORM == 2 ? a.m_tiles * a.n_tiles : (v - before + kRagM - 1) / kRagM * a.n_tiles;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, t, off);
      if (lane >= off) t += o;
    }
    t += tiles;
    if (e <= a.experts) { c->start[e] = v; c->tile0[e] = t; }
    run = __shfl_sync(0xffffffffu, v, 31);
    tiles = __shfl_sync(0xffffffffu, t, 31);
  }
}

struct RaggedTile {
  int e = 0;                   // expert; only moves forward
  int m, n;                    // row and column tile inside the expert
  __device__ __forceinline__ void at(const RaggedArgs& a, const RaggedCtrl* c, int t, int form) {
    while (t >= c->tile0[e + 1]) ++e;
    const int local = t - c->tile0[e];
    const int mt = form == 2 ? a.m_tiles : (c->tile0[e + 1] - c->tile0[e]) / a.n_tiles;
    const int per_group = a.group_m * a.n_tiles;
    const int bg = local / per_group;
    const int rem = local - bg * per_group;
    const int gs = min(a.group_m, mt - bg * a.group_m);
    n = rem / gs;
    m = bg * a.group_m + (rem - n * gs);
  }
};

// MN-major, 128-byte-swizzled operand tile: chunks of 64 columns x 64 contraction rows (8 KB), 8-row groups 1024 B apart.
__device__ __forceinline__ uint64_t make_smem_desc_mn(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= uint64_t((smem_addr >> 4) & 0x3FFF);
  d |= uint64_t((kRagK * 128) >> 4) << 16;           // leading byte offset: next 64 columns
  d |= uint64_t(1024 >> 4) << 32;                    // stride byte offset: next 8 contraction rows
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;                            // SWIZZLE_128B
  return d;
}

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
    ragged_tables<FORM>(a, ctrl, lane);
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
  const int total = ctrl->tile0[a.experts];
  auto k_blocks = [&](int e) {
    return FORM == 2 ? (ctrl->start[e + 1] - ctrl->start[e] + kRagK - 1) / kRagK : (a.k_dim + kRagK - 1) / kRagK;
  };

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    RaggedTile tile;
    for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
      tile.at(a, ctrl, t, FORM);
      const int KB = k_blocks(tile.e), row0 = ctrl->start[tile.e];
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
        tile.at(a, ctrl, t, FORM);
        KB = k_blocks(tile.e);
        seg = ctrl->start[tile.e + 1] - ctrl->start[tile.e];
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
          const int zero = steps * 16 - have;
          // (64-column chunks of A and B) x zero rows x 8 vectors of 16 bytes; the swizzle stays inside a row
          for (int i = lane; i < zero * (kRagM + kRagN) / 8; i += 32) {
            const int chunk = i / (zero * 8), rem = i - chunk * zero * 8;
            *reinterpret_cast<uint4*>(sp + chunk * kRagK * 128 + (have + rem / 8) * 128 + (rem & 7) * 16) =
                make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        const uint32_t sa = smem_u32(sp);
        const uint64_t adesc = kAMn ? make_smem_desc_mn(sa) : make_smem_desc(sa);
        const uint64_t bdesc = kBMn ? make_smem_desc_mn(sa + kABytes) : make_smem_desc(sa + kABytes);
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
      tile.at(a, ctrl, t, FORM);
      const int e = tile.e, start = ctrl->start[e], seg = ctrl->start[e + 1] - start;
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
          uint4 pk;
          if (a.bf16) {
            pk.x = pack_bf16x2(v[j], v[j + 1]); pk.y = pack_bf16x2(v[j + 2], v[j + 3]);
            pk.z = pack_bf16x2(v[j + 4], v[j + 5]); pk.w = pack_bf16x2(v[j + 6], v[j + 7]);
          } else {
            pk.x = pack_f16x2(v[j], v[j + 1]); pk.y = pack_f16x2(v[j + 2], v[j + 3]);
            pk.z = pack_f16x2(v[j + 4], v[j + 5]); pk.w = pack_f16x2(v[j + 6], v[j + 7]);
          }
          if (q * 32 + j < cols) *reinterpret_cast<uint4*>(op + (q * 32 + j) * 2) = pk;
        }
      }
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
    if (FORM != 2 && a.zero_uncovered) {
      // rows that belong to no expert: in front of the first segment and behind the last
      const int lo = ctrl->start[0], hi = ctrl->start[a.experts];
      const long long vec = a.n_dim / 8, head = lo * vec, all = head + (a.rows - hi) * vec;
      uint4* out = static_cast<uint4*>(a.out);
      for (long long i = (long long)blockIdx.x * 256 + threadIdx.x - 128; i < all; i += (long long)gridDim.x * 256)
        out[i < head ? i : (long long)hi * vec + i - head] = make_uint4(0, 0, 0, 0);
    }
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
// Row-major 16-bit matrix [rows, cols] (or `mats` of them), boxes of 64 columns x box_rows rows.
static int ragged_map(CUtensorMap* map, const void* base, long long cols, long long rows, int mats, int box_rows) {
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
  CUtensorMap ma, mb;
  if ((rc = ragged_map(&ma, dy, n, rows, 0, kRagK)) != FLYMOE_OK) return rc;
  if ((rc = ragged_map(&mb, x, k, rows, 0, kRagK)) != FLYMOE_OK) return rc;
  return launch_ragged<2>(ma, mb, a, max_tiles, s);
}
