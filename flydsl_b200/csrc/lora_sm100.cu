// Adapters on tcgen05: shrink and expand for batches that fill tiles of 128 rows (see lora.cu for the operator).
//
// Both kernels stream their large operand through TMA and leave the thin products to the tensor cores, so what is left is
// the traffic: x once for the shrink, base and output once each for the expand (from 8192 to 32768 rows of 4096 columns
// each further 8192 rows cost 10 and 20 us, 6.7 TB/s, and an expand without a base, which only writes, 15.6 us, 4.3 TB/s;
// start and end of a launch cost 6 to 9 us more).  A tile goes through the distinct adapters among its rows; of each product
// only that adapter's rows are kept.
//
// Shrink: 128 rows x one split of K.  Every adapter of the tile has its own columns of TMEM (rank each); a K block of x is
// loaded once and multiplied with each adapter's block.  The splits' sums are folded by a launch of their own: a cluster over
// K would save it, but CTAs that wait for one another must not wait for TMEM as well, and the expand, whose blocks each
// read a row tile's v, took 15000 cycles to add up nine splits where one takes 2000.
//
// Expand: the base tile (128 x 128) is loaded into shared memory, gets the adapters' products added row by row where it
// lies, and is stored from there; rows without an adapter are simply not touched.  The rows' v stands in shared memory as high
// parts and remainders, [128, rank] each, for all column tiles of the row tile.  A warp of its own issues the stores: while an
// epilogue warp also waited for the store before to be read out, and the base was read after the MMAs, 8192 rows of 4096
// columns without a base took 24.8 us instead of 22.1.  Looking for NaNs costs about a microsecond of 27.
#include <cuda.h>

#include <algorithm>

#include "common.cuh"
#include "gemm_ptx.cuh"
#include "lora_common.cuh"

namespace flymoe {

constexpr int kTileRows = 128;
constexpr int kChunkBytes = kTileRows * 128;     // 128 rows x 64 16-bit columns, 128-byte swizzle

__device__ __forceinline__ uint32_t instr_desc(int bf16, int n) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (uint32_t(n >> 3) << 17) | (uint32_t(kTileRows >> 4) << 24);
}

// ---------------------------------------------------------------------------- shrink
constexpr int kShX = 4;                          // K blocks of x in flight
constexpr int kShABytes = 32768;                 // ring of adapter blocks, rank rows x 128 bytes each
struct __align__(16) ShrinkCtrl {
  unsigned long long x_full[kShX], x_empty[kShX], a_full[16], a_empty[16], acc_full;
  uint32_t tmem_base;
  int abort_flag, count, list[kTileAdapters];
};
constexpr size_t kShSmem = size_t(kShX) * kChunkBytes + kShABytes + sizeof(ShrinkCtrl) + 1024;

struct ShrinkTcArgs {
  ShrinkArgs p;
  int bf16, rank_pad, slots;
  int a_bytes;                 // an adapter's block in shared memory
  int* status;
};

__global__ void __launch_bounds__(256, 2)
lora_shrink_tc_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_a,
                      const ShrinkTcArgs q) {
  extern __shared__ uint8_t smem_dyn[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  uint8_t* aring = smem + kShX * kChunkBytes;
  ShrinkCtrl* c = reinterpret_cast<ShrinkCtrl*>(aring + kShABytes);
  volatile int* abort_flag = &c->abort_flag;
  const ShrinkArgs& p = q.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row0 = blockIdx.x * kTileRows;
  const int a_bytes = q.a_bytes;

  // Columns of TMEM for the adapters that are there: with room for as many as there may be, ranks from 33 on would leave one
  // block on an SM.  Sums are read 32 columns at a time, so also what the last read reaches past a rank of 16 modulo 32.
  uint32_t tmem_cols = 0;
  if (warp == 1) {
    wait_for_previous_launch();
    int id[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) id[i] = row_adapter(written_before(p.ids), row0 + i * 32 + lane, p.rows, p.adapters);
    int n = tile_adapters(id, lane, tile_limit(p.rank), c->list);
    if (blockIdx.y == 0 && lane == 0) p.counts[blockIdx.x] = n;
    if (n > tile_limit(p.rank)) n = 0;           // the other tiles are not this kernel's
    if (lane == 0) c->count = n;
    if (n > 0) {
      tmem_cols = 32;
      while (int(tmem_cols) < (n - 1) * q.rank_pad + (q.rank_pad + 31) / 32 * 32) tmem_cols *= 2;
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                   ::"r"(smem_u32(&c->tmem_base)), "r"(tmem_cols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  } else if (threadIdx.x == 0) {
    for (int i = 0; i < kShX; ++i) { mbar_init(smem_u32(&c->x_full[i]), 1); mbar_init(smem_u32(&c->x_empty[i]), 1); }
    for (int i = 0; i < 16; ++i) { mbar_init(smem_u32(&c->a_full[i]), 1); mbar_init(smem_u32(&c->a_empty[i]), 1); }
    mbar_init(smem_u32(&c->acc_full), 1);
    c->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  wait_for_previous_launch();
  let_next_launch_start();
  const uint32_t tmem = c->tmem_base;
  const int d = c->count;
  const int blocks = (p.k + 63) / 64;
  const int kb0 = int((long long)blocks * blockIdx.y / p.splits), kb1 = int((long long)blocks * (blockIdx.y + 1) / p.splits);

  // Producer and issuer are one thread each, waits included: a warp that waits together and elects a thread for every block
  // takes twice as long per block.
  if (warp == 0 && d > 0) {
    // ------------------------------------------------------------------ TMA producer
    if (elect_one()) {
      int xs = 0, as = 0;
      uint32_t xp = 0, ap = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        ok = mbar_wait(smem_u32(&c->x_empty[xs]), xp ^ 1, abort_flag, q.status, 1, 32);
        if (!ok) break;
        mbar_expect_tx(smem_u32(&c->x_full[xs]), kChunkBytes);
        tma_load_2d(smem_u32(smem + xs * kChunkBytes), &tmap_x, smem_u32(&c->x_full[xs]), kb * 128, row0);
        if (++xs == kShX) { xs = 0; xp ^= 1; }
        for (int i = 0; i < d; ++i) {
          ok = mbar_wait(smem_u32(&c->a_empty[as]), ap ^ 1, abort_flag, q.status, 1, 32);
          if (!ok) break;
          const uint32_t dst = smem_u32(aring + as * a_bytes), full = smem_u32(&c->a_full[as]);
          mbar_expect_tx(full, a_bytes);
          if (!p.transposed) tma_load_3d(dst, &tmap_a, full, kb * 128, 0, c->list[i]);
          else
            for (int j = 0; j < a_bytes; j += 8192) tma_load_3d(dst + j, &tmap_a, full, j / 64, kb * 64, c->list[i]);
          if (++as == q.slots) { as = 0; ap ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1 && d > 0) {
    // ------------------------------------------------------------------ MMA issuer
    if (elect_one()) {
      const uint32_t idesc = instr_desc(q.bf16, q.rank_pad) | (p.transposed ? 1u << 16 : 0u);
      const uint64_t b_step = p.transposed ? 16 * 128 / 16 : 2;
      int xs = 0, as = 0;
      uint32_t xp = 0, ap = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        ok = mbar_wait(smem_u32(&c->x_full[xs]), xp, abort_flag, q.status, 3);
        const uint64_t adesc = make_smem_desc(smem_u32(smem + xs * kChunkBytes));
        for (int i = 0; i < d && ok; ++i) {
          ok = mbar_wait(smem_u32(&c->a_full[as]), ap, abort_flag, q.status, 3);
          if (!ok) break;
          const uint32_t at = smem_u32(aring + as * a_bytes);
          const uint64_t bdesc = p.transposed ? make_smem_desc_mn(at, 8192) : make_smem_desc(at);
          tcgen05_fence_after();
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(tmem + i * q.rank_pad, adesc + k * 2, bdesc + k * b_step, idesc, (k > 0 || kb > kb0) ? 1u : 0u);
          umma_commit(smem_u32(&c->a_empty[as]));
          if (i + 1 == d) {
            umma_commit(smem_u32(&c->x_empty[xs]));
            if (kb + 1 == kb1) umma_commit(smem_u32(&c->acc_full));
          }
          if (++as == q.slots) { as = 0; ap ^= 1; }
        }
        if (++xs == kShX) { xs = 0; xp ^= 1; }
      }
    }
    __syncwarp();
  } else if (warp >= 4 && d > 0) {
    // ------------------------------------------------------------------ epilogue: a thread per row
    const int i = threadIdx.x - 128, mine = row_adapter(written_before(p.ids), row0 + i, p.rows, p.adapters);
    float* out = p.v + ((long long)blockIdx.y * p.rows + row0 + i) * p.rank;
    const bool summed = kb1 > kb0;               // more splits than K blocks: some have nothing to add
    if (!summed || warp_wait(smem_u32(&c->acc_full), 0, abort_flag, q.status, 4)) {
      tcgen05_fence_after();
      for (int a = 0; a < d; ++a) {
        const bool hit = mine == c->list[a];
        if (!__any_sync(0xffffffffu, hit)) continue;
        for (int j = 0; j < p.rank; j += 32) {
          float v[32];
          if (summed) {
            tmem_ld_x32(tmem + (uint32_t((warp & 3) * 32) << 16) + a * q.rank_pad + j, reinterpret_cast<uint32_t*>(v));
            tmem_ld_wait();
          }
          if (hit) {
#pragma unroll
            for (int u = 0; u < 32; u += 4)
              if (j + u < p.rank)
                *reinterpret_cast<float4*>(out + j + u) = summed ? make_float4(v[u], v[u + 1], v[u + 2], v[u + 3])
                                                                 : make_float4(0.f, 0.f, 0.f, 0.f);
          }
        }
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1 && tmem_cols > 0) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols) : "memory");
  }
}

// ---------------------------------------------------------------------------- expand
constexpr int kExCols = 128;                     // columns of a tile: two chunks of 64
constexpr int kExThreads = 384;
constexpr int kExEpi = 256;
struct __align__(16) ExpandCtrl {
  unsigned long long y_full[4], y_empty[4], b_full[3], b_empty[3], acc_full[4], acc_empty[4];
  unsigned long long row_ready;                  // a row tile's v is set up
  unsigned long long together;                   // barrier of the epilogue warps
  // Their part of the output tile is written.  One for each tile in shared memory: a warp without rows of an adapter is
  // through with a tile early, and may be with the next one before another warp is with this.
  unsigned long long tile_done[4];
  uint32_t tmem_base;
  int abort_flag, list[3][kTileAdapters];        // the adapter tiles' producer's, and the epilogue's for two row tiles
  int first[2];                                  // of this block's units, and of the next one's
  long long warp_cost[kExThreads / 32];
  float up[2][kTileRows];
};
constexpr int kExAcc = 4;                        // accumulators
template <int KC> constexpr int ex_b_stages() { return KC == 1 ? 3 : 2; }      // adapter tiles in flight
template <int KC> constexpr int ex_y_stages() { return KC == 1 ? 4 : 3; }      // base / output tiles in shared memory
template <int KC> constexpr size_t ex_smem() {
  return size_t(ex_y_stages<KC>()) * 2 * kChunkBytes + size_t(ex_b_stages<KC>()) * KC * kChunkBytes + 2 * KC * kChunkBytes + sizeof(ExpandCtrl) + 1024;
}
static_assert(ex_smem<1>() <= 232448 && ex_smem<2>() <= 232448, "shared memory budget of one SM exceeded");

struct ExpandTcArgs {
  ExpandArgs p;
  int col_tiles, units;
  int* status;
};

// Products that came out as NaN, once more from the definition: high part and remainder share an accumulator, where against an
// infinity the remainder turns infinite products into NaN (see lora.cu).  A warp goes through the rows of its lanes with `mine`,
// two of their 64 columns of output (in shared memory, from `tile` on) a lane; where a row's v has a NaN its outputs stay.
// A call and its synchronisation at 8192 rows, 4096 -> 4096, rank 128: 0.11 ms, with an infinity in one row 0.35, with NaNs
// everywhere 0.29 (16 with every lane on its own row alone).
template <typename T>
__device__ __noinline__ void expand_again(const ExpandArgs& p, bool mine, uint8_t* tile, int adapter, int row0, int col) {
  const int lane = threadIdx.x & 31, first = int(threadIdx.x & 96);          // of the warp's rows in the tile
  const T* base = static_cast<const T*>(p.base);
  __syncwarp();                                  // the rows are written
  for (uint32_t who = __ballot_sync(0xffffffffu, mine); who; who &= who - 1) {
    const int from = __ffs(who) - 1, l = __shfl_sync(0xffffffffu, adapter, from);
    const long long row = row0 + first + from;
    const T* b = static_cast<const T*>(p.b) + (long long)l * p.n * p.rank;
    const float* v = p.v + row * p.rank;
    bool nan = false;
    for (int j = lane; j < p.rank; j += 32) nan |= isnan(v[j]);
    if (__any_sync(0xffffffffu, nan)) continue;
    for (int i = lane; i < min(64, p.n - col); i += 32) {
      T* out = reinterpret_cast<T*>(tile + (first + from) * 128 + ((i >> 3) ^ (from & 7)) * 16) + (i & 7);
      if (!isnan(float(*out))) continue;
      float sum = 0.f;
      for (int j = 0; j < p.rank; ++j)
        sum = fmaf(v[j], float(b[p.transposed ? (long long)j * p.n + col + i : (long long)(col + i) * p.rank + j]), sum);
      const float y = base ? float(base[row * p.n + col + i]) : 0.f;         // the tile is not stored yet
      const uint32_t pk = pack2<T>(fmaf(p.scaling[l], sum, y), 0.f);
      *out = reinterpret_cast<const T*>(&pk)[0];
    }
  }
  __syncwarp();
}

// KC: chunks of 64 in the rank.
template <typename T, int KC>
__global__ void __launch_bounds__(kExThreads, 1)
lora_expand_tc_kernel(const __grid_constant__ CUtensorMap tmap_y, const __grid_constant__ CUtensorMap tmap_out,
                      const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ ExpandTcArgs q) {
  constexpr int kExY = ex_y_stages<KC>(), kExB = ex_b_stages<KC>();
  extern __shared__ uint8_t smem_dyn[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  uint8_t* bring = smem + kExY * 2 * kChunkBytes;
  uint8_t* vtile = bring + kExB * KC * kChunkBytes;              // [hi, lo][KC] chunks
  ExpandCtrl* c = reinterpret_cast<ExpandCtrl*>(vtile + 2 * KC * kChunkBytes);
  volatile int* abort_flag = &c->abort_flag;
  const ExpandArgs& p = q.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 1) {
    wait_for_previous_launch();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&c->tmem_base)), "r"(uint32_t(kExAcc * kExCols)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (threadIdx.x == 0) {
    for (int i = 0; i < kExY; ++i) { mbar_init(smem_u32(&c->y_full[i]), 1); mbar_init(smem_u32(&c->y_empty[i]), 1); mbar_init(smem_u32(&c->tile_done[i]), kExEpi / 32); }
    for (int i = 0; i < kExB; ++i) { mbar_init(smem_u32(&c->b_full[i]), 1); mbar_init(smem_u32(&c->b_empty[i]), 1); }
    for (int i = 0; i < kExAcc; ++i) { mbar_init(smem_u32(&c->acc_full[i]), 1); mbar_init(smem_u32(&c->acc_empty[i]), kExEpi / 32); }
    mbar_init(smem_u32(&c->row_ready), kExEpi);
    mbar_init(smem_u32(&c->together), kExEpi / 32);
    c->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  wait_for_previous_launch();
  let_next_launch_start();
  const uint32_t tmem = c->tmem_base;
  const int *ids = written_before(p.ids), *counts = written_before(p.counts);
  const int steps = (p.rank + 15) / 16;          // of the contraction
  // an adapter's tile: 128 columns along the rank, or (transposed) two chunks of 64 columns with a row per rank
  const uint32_t b_bytes = p.transposed ? steps * 16 * 256 : KC * kChunkBytes;
  const int most = tile_limit(p.rank);
  // adapters of a row tile; more than `most`: nothing to do here (the other kernel's, or no adapter and the base in place)
  auto adapters_of = [&](int rt) {
    const int d = fetch(counts + rt);
    return d == 0 && p.base == p.out ? most + 1 : d;
  };
  auto find_adapters = [&](int rt, int* list) {
    int id[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) id[i] = row_adapter(ids, rt * kTileRows + i * 32 + lane, p.rows, p.adapters);
    const int n = tile_adapters(id, lane, most, list);
    __syncwarp();
    return n;
  };
  // Blocks take consecutive column tiles of a row tile, so that the rows' v is set up once or twice per block, and as much
  // work each: a tile's time is that of its bytes up to two adapters, from there on each costs a third of that more.  In equal
  // numbers of tiles the blocks with the most adapters held the launch up (4096 rows, 16 runs of 8 adapters of rank 64, 7168
  // columns: 36 us against 33).
  auto cost_of = [&](int rt) {
    const int d = adapters_of(rt);
    return d > most ? 0 : max(35, 19 + 11 * d);
  };
  {
    const int tiles = (p.rows + kTileRows - 1) / kTileRows, per = (tiles + kExThreads - 1) / kExThreads;
    const int t0 = min(tiles, int(threadIdx.x) * per), t1 = min(tiles, t0 + per);
    long long mine = 0;
    for (int t = t0; t < t1; ++t) mine += (long long)cost_of(t) * q.col_tiles;
    long long upto = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += o;
    }
    if (lane == 31) c->warp_cost[warp] = upto;
    if (threadIdx.x < 2) c->first[threadIdx.x] = q.units;        // where nothing is left
    __syncthreads();
    long long all = 0;
#pragma unroll
    for (int i = 0; i < kExThreads / 32; ++i) {
      const long long w = c->warp_cost[i];
      if (i < warp) upto += w;
      all += w;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const long long want = all * (blockIdx.x + i) / gridDim.x;
      long long at = upto - mine;
      if (want < at || want >= upto) continue;
      int t = t0;
      for (; want >= at + (long long)cost_of(t) * q.col_tiles; ++t) at += (long long)cost_of(t) * q.col_tiles;
      const int cost = cost_of(t);
      c->first[i] = t * q.col_tiles + int((want - at + cost - 1) / cost);
    }
    __syncthreads();
  }
  const int u0 = c->first[0], u1 = c->first[1];

  // Producers and issuer: a warp looks at the ids, one thread (the same every time) does the rest, waits included.
  if (warp == 0) {
    // ------------------------------------------------------------------ base tiles
    int ys = 0;
    uint32_t yp = 0;
    bool ok = true;
    for (int u = u0; u < u1;) {
      const int rt = u / q.col_tiles, end = min(u1, (rt + 1) * q.col_tiles);
      const bool ours = adapters_of(rt) <= most;
      if (ours && elect_one()) {
        for (int t = u; t < end && ok; ++t) {
          const int col = (t - rt * q.col_tiles) * kExCols;
          ok = mbar_wait(smem_u32(&c->y_empty[ys]), yp ^ 1, abort_flag, q.status, 1, 32);
          if (!ok) break;
          const uint32_t full = smem_u32(&c->y_full[ys]), dst = smem_u32(smem + ys * 2 * kChunkBytes);
          if (p.base) {
            mbar_expect_tx(full, 2 * kChunkBytes);
            tma_load_2d(dst, &tmap_y, full, col * 2, rt * kTileRows);
            tma_load_2d(dst + kChunkBytes, &tmap_y, full, col * 2 + 128, rt * kTileRows);
          } else {
            mbar_arrive(full);
          }
          if (++ys == kExY) { ys = 0; yp ^= 1; }
        }
      }
      __syncwarp();
      u = end;
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ adapter tiles
    int bs = 0;
    int* list = c->list[0];
    uint32_t bp = 0;
    bool ok = true;
    for (int u = u0; u < u1;) {
      const int rt = u / q.col_tiles, end = min(u1, (rt + 1) * q.col_tiles);
      const int d = find_adapters(rt, list);
      if (d <= most && elect_one()) {
        for (int t = u; t < end && ok; ++t) {
          const int col = (t - rt * q.col_tiles) * kExCols;
          for (int i = 0; i < d && ok; ++i) {
            ok = mbar_wait(smem_u32(&c->b_empty[bs]), bp ^ 1, abort_flag, q.status, 1, 32);
            if (!ok) break;
            const uint32_t bfull = smem_u32(&c->b_full[bs]), bdst = smem_u32(bring + bs * KC * kChunkBytes);
            mbar_expect_tx(bfull, b_bytes);
            if (p.transposed) {
              tma_load_3d(bdst, &tmap_b, bfull, col * 2, 0, list[i]);
              tma_load_3d(bdst + b_bytes / 2, &tmap_b, bfull, col * 2 + 128, 0, list[i]);
            } else {
#pragma unroll
              for (int k = 0; k < KC; ++k) tma_load_3d(bdst + k * kChunkBytes, &tmap_b, bfull, k * 128, col, list[i]);
            }
            if (++bs == kExB) { bs = 0; bp ^= 1; }
          }
        }
      }
      __syncwarp();
      u = end;
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    const uint32_t idesc = instr_desc(std::is_same<T, __nv_bfloat16>::value, kExCols) | (p.transposed ? 1u << 16 : 0u);
    const uint32_t b_step = p.transposed ? 2048 >> 4 : 2, b_chunk = p.transposed ? 4 * (2048 >> 4) : kChunkBytes >> 4;
    int bs = 0, acc = 0;
    uint32_t bp = 0, rp = 0, accp = 0;
    bool ok = true;
    for (int u = u0; u < u1;) {
      const int rt = u / q.col_tiles, end = min(u1, (rt + 1) * q.col_tiles);
      const int d = adapters_of(rt);
      if (d >= 1 && d <= most && elect_one()) {         // otherwise nobody multiplies, and nobody signals
        ok = ok && mbar_wait(smem_u32(&c->row_ready), rp, abort_flag, q.status, 5);
        rp ^= 1;
        for (int t = (end - u) * d; t > 0 && ok; --t) {
          ok = mbar_wait(smem_u32(&c->acc_empty[acc]), accp ^ 1, abort_flag, q.status, 2) &&
               mbar_wait(smem_u32(&c->b_full[bs]), bp, abort_flag, q.status, 3);
          if (!ok) break;
          const uint32_t at = smem_u32(bring + bs * KC * kChunkBytes);
          const uint64_t bd = p.transposed ? make_smem_desc_mn(at, b_bytes / 2) : make_smem_desc(at);
          tcgen05_fence_after();
          for (int part = 0; part < 2; ++part) {
            const uint64_t ad = make_smem_desc(smem_u32(vtile + part * KC * kChunkBytes));
            for (int k = 0; k < steps; ++k)
              umma_f16(tmem + acc * kExCols, ad + uint64_t((k >> 2) * (kChunkBytes >> 4) + (k & 3) * 2),
                       bd + uint64_t((k >> 2) * b_chunk + (k & 3) * b_step), idesc, (part > 0 || k > 0) ? 1u : 0u);
          }
          umma_commit(smem_u32(&c->b_empty[bs]));
          umma_commit(smem_u32(&c->acc_full[acc]));
          if (++bs == kExB) { bs = 0; bp ^= 1; }
          if (++acc == kExAcc) { acc = 0; accp ^= 1; }
        }
      }
      __syncwarp();
      u = end;
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------------ output tiles
    int ys = 0, stored = 0;
    uint32_t yp = 0;
    bool ok = true;
    for (int u = u0; u < u1;) {
      const int rt = u / q.col_tiles, end = min(u1, (rt + 1) * q.col_tiles);
      const bool ours = adapters_of(rt) <= most;
      if (ours && lane == 0) {                   // the same thread every time: the groups of stores are its own
        for (int t = u; t < end && ok; ++t) {
          const int col = (t - rt * q.col_tiles) * kExCols;
          ok = mbar_wait(smem_u32(&c->tile_done[ys]), yp, abort_flag, q.status, 7);
          if (!ok) break;
          const uint32_t src = smem_u32(smem + ys * 2 * kChunkBytes);
          tma_store_2d(&tmap_out, src, col * 2, rt * kTileRows);
          if (col + 64 < p.n) tma_store_2d(&tmap_out, src + kChunkBytes, col * 2 + 128, rt * kTileRows);
          bulk_commit();
          // the store before this one has been read out of its tile: that tile is free
          asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
          if (stored++ > 0) mbar_arrive(smem_u32(&c->y_empty[ys == 0 ? kExY - 1 : ys - 1]));
          if (++ys == kExY) { ys = 0; yp ^= 1; }
        }
      }
      __syncwarp();
      u = end;
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ epilogue: a thread per row and half tile
    const int et = threadIdx.x - 128, wg = et >> 7, row = et & 127;
    const int sw = row & 7;
    int ys = 0, acc = 0, row_tile = -1, d = 0, mine = -1, turn = 0;
    uint32_t yp = 0, accp = 0;
    float scale = 0.f;
    bool ok = true;
    uint32_t together = 0;
    auto sync = [&]() -> bool {                  // bounded: a warp that gave up elsewhere does not leave the others waiting
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&c->together));
      const bool met = warp_wait(smem_u32(&c->together), together, abort_flag, q.status, 7);
      together ^= 1;
      return met;
    };
    for (int u = u0; u < u1 && ok; ++u) {
      const int rt = u / q.col_tiles, col = (u - rt * q.col_tiles) * kExCols;
      if (rt != row_tile) {
        // The MMAs of the previous row tile are done (their last sums have been read here): its v may go.  Eight threads to a
        // row; ids and v are asked for together.
        row_tile = rt;
        d = adapters_of(rt);
        if (d > most) continue;                  // its rows are the other kernel's
        turn ^= 1;
        const int r8 = et >> 3, l8 = et & 7, vecs = p.rank / 4;
        int id[4];
        float4 x[4][KC * 2];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const int r = rt * kTileRows + s * 32 + r8;
          id[s] = row_adapter(ids, r, p.rows, p.adapters);
#pragma unroll
          for (int h = 0; h < KC * 2; ++h) {
            x[s][h] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < p.rows && h * 8 + l8 < vecs) x[s][h] = fetch(reinterpret_cast<const float4*>(p.v) + (long long)r * vecs + h * 8 + l8);
          }
        }
        mine = row_adapter(ids, rt * kTileRows + row, p.rows, p.adapters);
        scale = mine >= 0 ? fetch(p.scaling + mine) : 0.f;
        if (et < 32) find_adapters(rt, c->list[1 + turn]);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const int r = s * 32 + r8;
          float down = 1.f;
          if (id[s] < 0) {                       // nothing has been summed up for it
#pragma unroll
            for (int h = 0; h < KC * 2; ++h) x[s][h] = make_float4(0.f, 0.f, 0.f, 0.f);
          }
          if constexpr (std::is_same<T, __half>::value) {
            float amax = 0.f;
#pragma unroll
            for (int h = 0; h < KC * 2; ++h)
              amax = fmaxf(amax, fmaxf(fmaxf(finite_abs(x[s][h].x), finite_abs(x[s][h].y)),
                                       fmaxf(finite_abs(x[s][h].z), finite_abs(x[s][h].w))));
#pragma unroll
            for (int off = 1; off < 8; off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
            const int e = scale_exponent(amax);
            down = exp2i(-e);
            if (l8 == 0) c->up[turn][r] = exp2i(e);
          }
#pragma unroll
          for (int h = 0; h < KC * 2; ++h) {
            const int k4 = h * 8 + l8;
            if (k4 >= (p.rank + 15) / 16 * 4) continue;
            uint2 hi, lo;
            split2<T>(x[s][h].x * down, x[s][h].y * down, hi.x, lo.x);
            split2<T>(x[s][h].z * down, x[s][h].w * down, hi.y, lo.y);
            uint8_t* at = vtile + (k4 >> 4) * kChunkBytes + r * 128 + ((((k4 >> 1) & 7) ^ (r & 7)) * 16) + (k4 & 1) * 8;
            *reinterpret_cast<uint2*>(at) = hi;
            *reinterpret_cast<uint2*>(at + KC * kChunkBytes) = lo;
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        ok = sync();                             // list and exponents, in this row tile's places, are written
        if (!ok) break;
        if constexpr (std::is_same<T, __half>::value) scale *= c->up[turn][row];
        if (d >= 1) mbar_arrive(smem_u32(&c->row_ready));
      }
      if (d > most) continue;
      ok = warp_wait(smem_u32(&c->y_full[ys]), yp, abort_flag, q.status, 6);
      if (!ok) break;
      uint8_t* line = smem + (ys * 2 + wg) * kChunkBytes + row * 128;
      uint4 y[8];                                // the base, on its way while the MMAs are waited for
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = make_uint4(0, 0, 0, 0);
      if (p.base == nullptr) {
        if (mine < 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(line + ((j ^ sw) * 16)) = y[j];
        }
      } else if (mine >= 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = *reinterpret_cast<const uint4*>(line + ((j ^ sw) * 16));
      }
      for (int i = 0; i < d && ok; ++i) {
        ok = warp_wait(smem_u32(&c->acc_full[acc]), accp, abort_flag, q.status, 4);
        if (!ok) break;
        tcgen05_fence_after();
        const bool hit = mine == c->list[1 + turn][i];
        if (__any_sync(0xffffffffu, hit)) {
          float v[64];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            tmem_ld_x32(tmem + (uint32_t((warp & 3) * 32) << 16) + acc * kExCols + wg * 64 + h * 32,
                        reinterpret_cast<uint32_t*>(v + h * 32));
          tmem_ld_wait();
          bool undefined = false;
          if (hit) {
            uint64_t sums = 0;                   // looks for NaNs
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              uint32_t* w = reinterpret_cast<uint32_t*>(&y[j]);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                add_pair(sums, v[j * 8 + k * 2], v[j * 8 + k * 2 + 1]);
                const float2 f = unpack2<T>(w[k]);
                w[k] = pack2<T>(fmaf(scale, v[j * 8 + k * 2], f.x), fmaf(scale, v[j * 8 + k * 2 + 1], f.y));
              }
              *reinterpret_cast<uint4*>(line + ((j ^ sw) * 16)) = y[j];
            }
            undefined = either_nan(sums);
          }
          if (__any_sync(0xffffffffu, undefined))
            expand_again<T>(p, undefined, smem + (ys * 2 + wg) * kChunkBytes, mine, rt * kTileRows, col + wg * 64);
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&c->acc_empty[acc]));
        if (++acc == kExAcc) { acc = 0; accp ^= 1; }
      }
      if (!ok) break;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&c->tile_done[ys]));
      if (++ys == kExY) { ys = 0; yp ^= 1; }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(uint32_t(kExAcc * kExCols)) : "memory");
  }
}

// ---------------------------------------------------------------------------- host
int launch_shrink_sm100(const ShrinkArgs& p, int bf16, cudaStream_t stream) {
  ShrinkTcArgs q = {p, bf16, (p.rank + 15) / 16 * 16, 0, 0, device_status_ptr()};
  if (q.status == nullptr) return FLYMOE_ERR_CUDA;
  q.a_bytes = p.transposed ? ceil_div(p.rank, 64) * 8192 : q.rank_pad * 128;
  q.slots = std::min(16, kShABytes / q.a_bytes);
  CUtensorMap mx, ma;
  int rc = matrix_map(&mx, p.x, p.k, p.rows, 0, kTileRows);
  if (rc == FLYMOE_OK)
    rc = p.transposed ? matrix_map(&ma, p.a, p.rank, p.k, p.adapters, 64) : matrix_map(&ma, p.a, p.k, p.rank, p.adapters, q.rank_pad);
  if (rc != FLYMOE_OK) return rc;
  static SmemLimitSeen seen;
  FLYMOE_CUDA_CHECK(allow_smem(reinterpret_cast<const void*>(lora_shrink_tc_kernel), int(kShSmem), seen));
  FLYMOE_CUDA_CHECK(launch_closely(lora_shrink_tc_kernel, dim3(ceil_div(p.rows, kTileRows), p.splits), 256, kShSmem, stream, mx, ma, q));
  return FLYMOE_OK;
}

template <typename T, int KC>
static int launch_expand_tc(const CUtensorMap& my, const CUtensorMap& mo, const CUtensorMap& mb, const ExpandTcArgs& q,
                            cudaStream_t stream) {
  auto* kernel = lora_expand_tc_kernel<T, KC>;
  static SmemLimitSeen seen;
  FLYMOE_CUDA_CHECK(allow_smem(reinterpret_cast<const void*>(kernel), int(ex_smem<KC>()), seen));
  FLYMOE_CUDA_CHECK(launch_closely(kernel, std::min(q.units, sm_count()), kExThreads, ex_smem<KC>(), stream, my, mo, mb, q));
  return FLYMOE_OK;
}

int launch_expand_sm100(const ExpandArgs& p, int bf16, cudaStream_t stream) {
  ExpandTcArgs q = {p, ceil_div(p.n, kExCols), 0, device_status_ptr()};
  if (q.status == nullptr) return FLYMOE_ERR_CUDA;
  const long long units = (long long)ceil_div(p.rows, kTileRows) * q.col_tiles;
  FLYMOE_REQUIRE(units < (1LL << 31), "lora_expand: too many tiles");
  q.units = int(units);
  CUtensorMap my, mo, mb;
  int rc = matrix_map(&my, p.base ? p.base : p.out, p.n, p.rows, 0, kTileRows);
  if (rc == FLYMOE_OK) rc = matrix_map(&mo, p.out, p.n, p.rows, 0, kTileRows);
  if (rc == FLYMOE_OK)
    rc = p.transposed ? matrix_map(&mb, p.b, p.n, p.rank, p.adapters, (p.rank + 15) / 16 * 16)
                      : matrix_map(&mb, p.b, p.rank, p.n, p.adapters, kExCols);
  if (rc != FLYMOE_OK) return rc;
  if (p.rank <= 64)
    return bf16 ? launch_expand_tc<__nv_bfloat16, 1>(my, mo, mb, q, stream) : launch_expand_tc<__half, 1>(my, mo, mb, q, stream);
  return bf16 ? launch_expand_tc<__nv_bfloat16, 2>(my, mo, mb, q, stream) : launch_expand_tc<__half, 2>(my, mo, mb, q, stream);
}

}  // namespace flymoe
