// Gradients of the adapters in bf16 on tcgen05: dA_l = s_l * sum over the rows of adapter l of dv^T x, dB_l likewise of
// dout^T v (see lora.cu for the operator, and for the fp16 form, whose running exponent needs the sums in registers).
//
// The contraction runs over the rows, so both operands lie across their rows in shared memory, as they come: a chunk is 32
// rows of an adapter, gathered by their ids (cp.async, rows of 512 bytes), and its v as high parts beside remainders
// (columns [0, RP) and [RP, 2 RP) of one operand, so that one MMA multiplies both; the two sums meet when they are read).
// A chunk's missing rows are zeros, other adapters' rows are never read into it: what they hold reaches nobody else.
//
// Bytes are what bounds it: x and dout once, 134 MB at 8192 rows of 4096 + 4096 columns.
#include <algorithm>

#include "common.cuh"
#include "gemm_ptx.cuh"
#include "lora_common.cuh"

namespace flymoe {

constexpr int kGradRows = 32;                    // of a chunk
// Chunks in shared memory, and of these the ones asked for before the oldest is handed over; two blocks have room on an SM.
template <int RP> constexpr int grad_stages() { return RP <= 32 ? 4 : 3; }
template <int RP> constexpr int grad_ahead() { return grad_stages<RP>() - 2; }
constexpr int kGradFill = 256, kGradThreads = kGradFill + 32 + 128;
constexpr int kGradXBytes = kGradRows * kWgCols * 2, kGradChunk = kGradRows * 128;      // 4 chunks of 64 columns
constexpr int kGradTmem = 256;
constexpr int kGradList = 1024;
constexpr int kGradLast = 1 << 16, kGradEnd = 1 << 17;     // of a chunk's note; the low bits are its adapter

struct __align__(16) GradCtrl {
  unsigned long long full[4], empty[4], sum_full[2], sum_empty[2];
  uint32_t tmem_base;
  int abort_flag, next_adapter, warp_n[kGradFill / 32], note[4], sum_adapter[2];
  int list[kGradList + kGradRows];
};
template <int RP> constexpr int grad_v_bytes() { return RP * 2 <= 64 ? kGradChunk : 2 * kGradChunk; }
template <int RP> constexpr size_t grad_smem() {
  return size_t(grad_stages<RP>()) * (kGradXBytes + grad_v_bytes<RP>() + kGradRows * RP * 4) + sizeof(GradCtrl) + 1024;
}
static_assert(2 * (grad_smem<64>() + 1024) <= 233472, "two blocks an SM");

__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(taddr));
}

// A block takes 256 columns (and up to RP ranks) of a gradient, one split of the rows and one group of adapters, and goes
// through those that have rows in it.  Warps 0..7 gather, warp 8 multiplies, warps 9..12 write the sums.  RP: its ranks, rounded up.
template <int RP>
__global__ void __launch_bounds__(kGradThreads, 2)
lora_wgrad_tc_kernel(const AdapterGradArgs p, int* status) {
  constexpr int N = 2 * RP, kSums = RP <= 32 ? 2 : 1, kVBytes = grad_v_bytes<RP>(), kStages = grad_stages<RP>(), kAhead = grad_ahead<RP>();
  static_assert(kSums * 2 * N <= kGradTmem, "sums of two halves of the columns");
  extern __shared__ uint8_t smem_dyn[];
  uint8_t* xs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  uint8_t* vs = xs + kStages * kGradXBytes;                  // high parts and remainders
  uint8_t* vf = vs + kStages * kVBytes;                      // v as it comes, [32][RP]
  GradCtrl* c = reinterpret_cast<GradCtrl*>(vf + kStages * kGradRows * RP * 4);
  volatile int* abort_flag = &c->abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const bool second = int(blockIdx.x) >= p.g[0].tiles;
  const AdapterGrad& q = second ? p.g[1] : p.g[0];
  const int col0 = (second ? int(blockIdx.x) - p.g[0].tiles : int(blockIdx.x)) * kWgCols;
  const int j0 = int(blockIdx.z) * kWgRank;      // first of this block's ranks
  const int ranks = min(kWgRank, p.rank - j0);
  const long long mat = (long long)q.cols * p.rank;
  const int split = int(blockIdx.y) / p.groups, group = int(blockIdx.y) - split * p.groups;

  if (warp == 8) {
    wait_for_previous_launch();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&c->tmem_base)), "r"(uint32_t(kGradTmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (tid == 0) {
    for (int i = 0; i < kStages; ++i) { mbar_init(smem_u32(&c->full[i]), kGradFill / 32); mbar_init(smem_u32(&c->empty[i]), 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(smem_u32(&c->sum_full[i]), 2); mbar_init(smem_u32(&c->sum_empty[i]), 4); }
    c->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  wait_for_previous_launch();
  let_next_launch_start();
  const uint32_t tmem = c->tmem_base;

  if (warp < kGradFill / 32) {
    // ------------------------------------------------------------------ gather
    const int begin = int((long long)p.rows * split / p.splits), end = int((long long)p.rows * (split + 1) / p.splits);
    const int others = p.groups - 1;             // an adapter's group is its number modulo `groups`, a power of two
    const uint8_t* X = static_cast<const uint8_t*>(q.x);
    const int* ids = written_before(p.ids);
    auto together = [] { asm volatile("bar.sync 1, %0;" ::"n"(kGradFill) : "memory"); };
    // The warps meet at a barrier without a limit, so a wait that gave up makes nobody leave: the walk through the rows goes on
    // and touches nothing any more.
    bool ok = true;
    int asked = 0, handed = 0;                   // chunks asked for, chunks handed over to the MMAs
    int older = 0, newer = 0;                    // adapters of up to two chunks between

    // the smallest adapter of the group above `l` with rows here, or p.adapters
    auto find_next = [&](int l) -> int {
      if (tid == 0) c->next_adapter = p.adapters;
      together();
      int best = p.adapters;
      for (int i = begin + tid; i < end; i += kGradFill) {
        const int id = fetch(ids + i);
        if (id > l && id < best && (id & others) == group) best = id;
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) best = min(best, __shfl_xor_sync(0xffffffffu, best, off));
      if (lane == 0) atomicMin(&c->next_adapter, best);
      together();
      return *const_cast<volatile int*>(&c->next_adapter);
    };
    // adapters without rows here: zeros, or (several splits) the finishing launch is told
    auto skip_adapters = [&](int from, int to) {
      if (p.splits > 1) {
        if (blockIdx.x == 0 && blockIdx.z == 0)
          for (int l = from + tid * p.groups; l < to; l += kGradFill * p.groups) p.present[(long long)split * p.adapters + l] = 0;
        return;
      }
      const int cn = min(kWgCols, q.cols - col0);
      for (int l = from; l < to; l += p.groups)
        for (int i = tid; i < ranks * cn; i += kGradFill) {
          const long long at = q.rank_major ? (long long)(j0 + i / cn) * q.cols + col0 + i % cn
                                            : (long long)(col0 + i / ranks) * p.rank + j0 + i % ranks;
          static_cast<__nv_bfloat16*>(q.out)[(long long)l * mat + at] = __nv_bfloat16(0.f);
        }
    };
    // v of the oldest chunk that is not handed over, from fp32 to its two parts; a thread converts what it has copied itself
    auto hand_over = [&](int flags) {
      const int stage = handed % kStages;
      if (ok) {
#pragma unroll
        for (int i = tid; i < kGradRows * (RP / 4); i += kGradFill) {
          const int r = i / (RP / 4), j = i - r * (RP / 4);
          const float4 x = *reinterpret_cast<const float4*>(vf + stage * kGradRows * RP * 4 + i * 16);
          uint2 h, w;
          split2<__nv_bfloat16>(x.x, x.y, h.x, w.x);
          split2<__nv_bfloat16>(x.z, x.w, h.y, w.y);
          auto place = [&](int n) {
            return vs + stage * kVBytes + (n >> 6) * kGradChunk + r * 128 + ((((n >> 3) & 7) ^ (r & 7)) * 16) + (n & 4) * 2;
          };
          *reinterpret_cast<uint2*>(place(j * 4)) = h;
          *reinterpret_cast<uint2*>(place(RP + j * 4)) = w;
        }
        if (tid == 0) c->note[stage] = flags;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(smem_u32(&c->full[stage]));
      ++handed;
    };

    const int piece = lane;                      // 16 bytes of a row; rows warp, warp + 8, ..
    const bool inside = col0 + piece * 8 < q.cols;
    const uint32_t xdst = smem_u32(xs) + (piece >> 3) * kGradChunk + warp * 128 + (((piece & 7) ^ (warp & 7)) * 16);
    const uint8_t* xsrc = X + (inside ? (long long)(col0 + piece * 8) * 2 : 0);
    const uint32_t row_bytes = uint32_t(q.cols) * 2;             // below 2^31

    int done = group;                             // adapters of the group below this one are dealt with
    for (int l = find_next(-1); l < p.adapters; l = find_next(l)) {
      skip_adapters(done, l);
      done = l + p.groups;
      if (p.splits > 1 && blockIdx.x == 0 && blockIdx.z == 0 && tid == 0) p.present[(long long)split * p.adapters + l] = 1;
      int next = begin, taken = 0, have = 0;     // ids scanned, entries of the list used and in it (same in all threads)
      while (true) {
        if (have - taken < kGradRows && next < end) {
          together();                            // nobody reads the part that moves
          const int rest = have - taken;
          const int keep = tid < rest ? c->list[taken + tid] : 0;
          together();
          if (tid < rest) c->list[tid] = keep;
          have = rest;
          taken = 0;
          while (have < kGradRows && next < end) {
            // 1024 ids, warp by warp 32 in a row
            uint32_t mine[4];
            int n = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int at = next + (warp * 4 + i) * 32 + lane;
              mine[i] = __ballot_sync(0xffffffffu, at < end && fetch(ids + at) == l);
              n += __popc(mine[i]);
            }
            if (lane == 0) c->warp_n[warp] = n;
            together();
            int pos = have, all = 0;
#pragma unroll
            for (int i = 0; i < kGradFill / 32; ++i) {
              const int w = c->warp_n[i];
              if (i < warp) pos += w;
              all += w;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if ((mine[i] >> lane) & 1) c->list[pos + __popc(mine[i] & ((1u << lane) - 1))] = next + (warp * 4 + i) * 32 + lane;
              pos += __popc(mine[i]);
            }
            have += all;
            next += kGradList;
            together();
          }
        }
        const int n = min(kGradRows, have - taken);
        if (n == 0) break;
        const int stage = asked % kStages;
        ok = ok && warp_wait(smem_u32(&c->empty[stage]), (asked / kStages & 1) ^ 1, abort_flag, status, 1);
        if (ok) {
#pragma unroll
          for (int k = 0; k < kGradRows / 8; ++k) {
            const int r = warp + k * 8;
            const bool here = r < n;
            const uint32_t row = here ? uint32_t(c->list[taken + r]) : 0u;
            cp_async16(xdst + stage * kGradXBytes + k * 1024, xsrc + uint64_t(row) * row_bytes, here && inside);
          }
#pragma unroll
          for (int i = tid; i < kGradRows * (RP / 4); i += kGradFill) {
            const int r = i / (RP / 4), j = i - r * (RP / 4);
            const bool here = r < n && j * 4 < ranks;
            const uint32_t row = here ? uint32_t(c->list[taken + r]) : 0u;
            cp_async16(smem_u32(vf + stage * kGradRows * RP * 4 + i * 16),
                       q.v + (uint64_t(row) * uint32_t(p.rank) + uint32_t(here ? j0 + j * 4 : 0)), here);
          }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        taken += n;
        if (asked - handed == kAhead) {
          asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
          hand_over(older | ((kAhead == 2 ? newer : l) != older ? kGradLast : 0));
        }
        older = kAhead == 1 || asked == handed ? l : newer;
        newer = l;
        ++asked;
      }
    }
    skip_adapters(done, p.adapters);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (asked - handed == 2) hand_over(older | (newer != older ? kGradLast : 0));
    if (asked > handed) hand_over(newer | kGradLast);
    const int stage = asked % kStages;
    ok = ok && warp_wait(smem_u32(&c->empty[stage]), (asked / kStages & 1) ^ 1, abort_flag, status, 1);
    if (ok && tid == 0) c->note[stage] = kGradEnd;
    __syncwarp();
    if (ok && lane == 0) mbar_arrive(smem_u32(&c->full[stage]));
  } else if (warp == 8) {
    // ------------------------------------------------------------------ MMAs: one thread
    if (elect_one()) {
      const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | (uint32_t(N >> 3) << 17) |
                             (uint32_t(128 >> 4) << 24);
      bool first = true;
      int sum = 0;
      uint32_t sp = 0;
      for (int i = 0;; ++i) {
        const int stage = i % kStages;
        if (!mbar_wait(smem_u32(&c->full[stage]), i / kStages & 1, abort_flag, status, 2)) break;
        const int note = *const_cast<volatile int*>(&c->note[stage]);
        if (first && !mbar_wait(smem_u32(&c->sum_empty[sum]), sp ^ 1, abort_flag, status, 3)) break;
        if (note & kGradEnd) {
          c->sum_adapter[sum] = -1;
          mbar_arrive(smem_u32(&c->sum_full[sum]));
          mbar_arrive(smem_u32(&c->sum_full[sum]));
          break;
        }
        tcgen05_fence_after();
        const uint64_t bd = make_smem_desc_mn(smem_u32(vs + stage * kVBytes), kGradChunk);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint64_t ad = make_smem_desc_mn(smem_u32(xs + stage * kGradXBytes + h * 2 * kGradChunk), kGradChunk);
#pragma unroll
          for (int k = 0; k < kGradRows / 16; ++k)
            umma_f16(tmem + sum * 2 * N + h * N, ad + uint64_t(k * (2048 >> 4)), bd + uint64_t(k * (2048 >> 4)), idesc,
                     (!first || k > 0) ? 1u : 0u);
        }
        umma_commit(smem_u32(&c->empty[stage]));
        first = (note & kGradLast) != 0;
        if (first) {
          c->sum_adapter[sum] = note & (kGradLast - 1);
          umma_commit(smem_u32(&c->sum_full[sum]));
          mbar_arrive(smem_u32(&c->sum_full[sum]));      // with the adapter's number
          if (++sum == kSums) { sum = 0; sp ^= 1; }
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ sums: a thread per column of each half
    int sum = 0;
    uint32_t sp = 0;
    while (warp_wait(smem_u32(&c->sum_full[sum]), sp, abort_flag, status, 4)) {
      const int l = *const_cast<volatile int*>(&c->sum_adapter[sum]);
      if (l < 0) break;
      tcgen05_fence_after();
      const float scale = p.splits == 1 ? fetch(p.scaling + l) : 1.f;
      float* partial = q.partial + ((long long)split * p.adapters + l) * mat;
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(q.out) + (long long)l * mat;
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        const int col = col0 + h * 128 + (warp & 3) * 32 + lane;
#pragma unroll 1
        for (int j = 0; j < RP; j += 16) {
          uint32_t hi[16], lo[16];
          const uint32_t at = tmem + (uint32_t((warp & 3) * 32) << 16) + sum * 2 * N + h * N + j;
          tmem_ld_x16(at, hi);
          tmem_ld_x16(at + RP, lo);
          tmem_ld_wait();
          float v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = of_two_parts(__uint_as_float(hi[i]), __uint_as_float(lo[i])) * scale;
          if (col >= q.cols) continue;
#pragma unroll
          for (int i = 0; i < 16; i += 8) {
            if (j + i >= ranks) break;
            if (q.rank_major) {
              const long long to = (long long)(j0 + j + i) * q.cols + col;
#pragma unroll
              for (int u = 0; u < 8; ++u) {
                if (p.splits > 1) partial[to + (long long)u * q.cols] = v[i + u];
                else out[to + (long long)u * q.cols] = __float2bfloat16_rn(v[i + u]);
              }
            } else {
              const long long to = (long long)col * p.rank + j0 + j + i;
              if (p.splits > 1) {
                *reinterpret_cast<float4*>(partial + to) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                *reinterpret_cast<float4*>(partial + to + 4) = make_float4(v[i + 4], v[i + 5], v[i + 6], v[i + 7]);
              } else {
                *reinterpret_cast<uint4*>(out + to) = make_uint4(pack_bf16x2(v[i], v[i + 1]), pack_bf16x2(v[i + 2], v[i + 3]),
                                                                 pack_bf16x2(v[i + 4], v[i + 5]), pack_bf16x2(v[i + 6], v[i + 7]));
              }
            }
          }
        }
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&c->sum_empty[sum]));
      if (++sum == kSums) { sum = 0; sp ^= 1; }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 8) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(uint32_t(kGradTmem)) : "memory");
  }
}

template <int RP>
static int launch(const AdapterGradArgs& p, cudaStream_t stream) {
  auto* kernel = lora_wgrad_tc_kernel<RP>;
  int* status = device_status_ptr();
  if (status == nullptr) return FLYMOE_ERR_CUDA;
  static SmemLimitSeen seen;
  FLYMOE_CUDA_CHECK(allow_smem(reinterpret_cast<const void*>(kernel), int(grad_smem<RP>()), seen));
  FLYMOE_CUDA_CHECK(launch_closely(kernel, dim3(p.g[0].tiles + p.g[1].tiles, p.splits * p.groups, ceil_div(p.rank, kWgRank)), kGradThreads,
                                   grad_smem<RP>(), stream, p, status));
  return FLYMOE_OK;
}
int launch_wgrad_sm100(const AdapterGradArgs& p, cudaStream_t stream) {
  return p.rank <= 16 ? launch<16>(p, stream) : p.rank <= 32 ? launch<32>(p, stream) : launch<64>(p, stream);
}

}  // namespace flymoe
