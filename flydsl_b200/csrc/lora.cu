// Low-rank adapters of many requests at once, beside a shared projection (16-bit operands).
//
//   out[m] = base[m] + s_l B_l (A_l x[m]),   l = ids[m];  a row whose id names no adapter passes through
//
// in two steps: shrink, v = x A_l^T (fp32 [rows, rank]), and expand, which adds s_l v B_l^T to the base.  The rank is the only
// small extent: both are bound by the bytes of x, the adapters in use, the base and the output, or by launches where rows
// are few.  Of every product only the adapter's own rows are kept, so nothing of one request, not even an infinity, reaches
// another.
//
// Two forms.  From 512 rows on, tiles of 128 rows with few adapters go through tcgen05 (lora_sm100.cu).  This file has the
// other: few rows, and tiles of many adapters.  Its blocks sort the rows of a window into groups of 16 that share an adapter
// and put each through mma.sync, whose smallest tile is 16 rows where tcgen05's is 128: with an adapter for every row or two the
// rows of a tile are what the work goes by.  Operand fragments are read from global memory 16 or 8 bytes a lane: the
// contraction index may be permuted as long as both operands agree, so a lane takes consecutive elements where the
// instruction's layout has pairs.
//
// v enters the second product as the sum of two 16-bit numbers (high part and remainder), which keeps 16 (bf16) or 22 (fp16)
// bits of it: one rounding of the output is all that shows.  fp16 has few exponent bits, so there a row of v is brought to
// the same power of two first.  A remainder that is zero or of the other sign makes no number of an infinity (0 * inf, inf - inf):
// where the product with the high part is not finite it is the result.  (In fp16 a number below 2^-38 of the largest beside
// it has no high part and counts as zero.)
//
// Gradients use the same kernels: dv = dout B_l is a shrink with B transposed, dx = s_l dv A_l an expand with A transposed
// (the tiles read them across, this file's kernels want copies).  dA_l = s_l sum dv^T x and dB_l = s_l sum dout^T v contract
// over an adapter's rows, found by scanning ids: bf16 on tcgen05 (lora_grad_sm100.cu), fp16 here, since a common power of two
// that may still grow needs the sums in registers (8192 rows, 4096 + 4096 columns, 4 adapters of rank 32: 45 us and 60).  No sum depends on the
// order of execution.
#include <algorithm>
#include <stdio.h>
#include <type_traits>

#include "common.cuh"
#include "gemm_ptx.cuh"
#include "lora_common.cuh"

namespace flymoe {

template <typename T>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load16(const void* p) { return fetch(static_cast<const uint4*>(p)); }

// ---------------------------------------------------------------------------- groups of rows
// The rows of a window (512) in groups of up to 16 that share an adapter, whatever order they come in.  Every block builds
// them for itself and all blocks alike: adapters in the order of their first rows, their rows in order.  A hash table finds
// the rows of an adapter; what is kept of it, the smallest row, does not depend on the order of its atomics.
constexpr int kWindow = 512, kTable = 1024;
constexpr int kGroupThreads = 256;
struct Groups {
  int id[kWindow];             // adapter of a row; -1: none
  uint16_t order[kWindow];     // rows of the window, an adapter's next to each other
  uint16_t start[kWindow + 2]; // first entry of `order` of a group; an adapter's groups follow each other
  uint16_t row_base[kWindow], group_base[kWindow];     // at an adapter's first row: entries and groups before it
  uint8_t in_chunk[kWindow / 32][kWindow];             // rows among 32 of the adapter with that first row
  int key[kTable], first[kTable];
  int warp_sum[2][8], count, skip[kWindow / 128];
};

// skip_tiles: rows of 128-row tiles with at most that many distinct adapters belong to the tcgen05 kernels; 0: none do.  keep_none:
// rows without an adapter form groups as well (adapter -1).
__device__ __forceinline__ void build_groups(Groups* s, const int* ids, int row0, int rows, int adapters, int skip_tiles,
                                             bool keep_none) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = min(kWindow, rows - row0), chunks = (n + 31) / 32;
  const int mask = (n > 128 ? kTable : 256) - 1;               // at least twice as many entries as rows
  for (int i = tid; i <= mask; i += kGroupThreads) { s->key[i] = -2; s->first[i] = kWindow; }
  for (int i = tid; i < chunks * kWindow / 4; i += kGroupThreads) reinterpret_cast<int*>(s->in_chunk)[i] = 0;
  if (skip_tiles > 0 && warp < kWindow / 128) {
    int q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = row_adapter(ids, row0 + warp * 128 + i * 32 + lane, rows, adapters);
    const int d = tile_adapters(q, lane, skip_tiles, nullptr);
    if (lane == 0) s->skip[warp] = d <= skip_tiles;
  }
  __syncthreads();
  if (skip_tiles > 0 && s->skip[0] && s->skip[1] && s->skip[2] && s->skip[3]) {      // nothing here (no rows: no adapters)
    if (tid == 0) s->count = 0;
    __syncthreads();
    return;
  }
  int slot[2], lead[2], rank[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = u * kGroupThreads + tid;
    slot[u] = -1;
    if (i >= n) continue;
    const int id = row_adapter(ids, row0 + i, rows, adapters);
    s->id[i] = id;
    if ((id < 0 && !keep_none) || (skip_tiles > 0 && s->skip[i / 128])) continue;
    int h = int((uint32_t(id) * 0x9E3779B1u) >> 22) & mask;
    for (;; h = (h + 1) & mask) {
      const int old = atomicCAS(&s->key[h], -2, id);
      if (old == -2 || old == id) break;
    }
    atomicMin(&s->first[h], i);
    slot[u] = h;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    lead[u] = slot[u] >= 0 ? s->first[slot[u]] : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, lead[u]);
    rank[u] = __popc(same & ((1u << lane) - 1));
    if (lead[u] >= 0 && rank[u] == 0) s->in_chunk[u * 8 + warp][lead[u]] = uint8_t(__popc(same));
  }
  __syncthreads();
  // totals at the first rows, two neighbouring rows a thread so that a scan over threads is one over rows
  int total[2] = {0, 0};
  for (int c = 0; c < chunks; ++c) {
    const int v = *reinterpret_cast<const uint16_t*>(&s->in_chunk[c][2 * tid]);
    total[0] += v & 0xff;
    total[1] += v >> 8;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (lead[u] >= 0)
      for (int c = 0; c < u * 8 + warp; ++c) rank[u] += s->in_chunk[c][lead[u]];
  const int rows_here = total[0] + total[1], groups_here = (total[0] + 15) / 16 + (total[1] + 15) / 16;
  int rs = rows_here, gs = groups_here;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, rs, off), b = __shfl_up_sync(0xffffffffu, gs, off);
    if (lane >= off) { rs += a; gs += b; }
  }
  if (lane == 31) { s->warp_sum[0][warp] = rs; s->warp_sum[1][warp] = gs; }
  __syncthreads();
  int rb = rs - rows_here, gb = gs - groups_here, all_groups = 0, all_rows = 0;
#pragma unroll
  for (int w = 0; w < kGroupThreads / 32; ++w) {
    if (w < warp) { rb += s->warp_sum[0][w]; gb += s->warp_sum[1][w]; }
    all_rows += s->warp_sum[0][w];
    all_groups += s->warp_sum[1][w];
  }
  s->row_base[2 * tid] = uint16_t(rb);
  s->row_base[2 * tid + 1] = uint16_t(rb + total[0]);
  s->group_base[2 * tid] = uint16_t(gb);
  s->group_base[2 * tid + 1] = uint16_t(gb + (total[0] + 15) / 16);
  if (tid == 0) { s->count = all_groups; s->start[all_groups] = uint16_t(all_rows); }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (lead[u] >= 0) {
      const int pos = s->row_base[lead[u]] + rank[u];
      s->order[pos] = uint16_t(u * kGroupThreads + tid);
      if ((rank[u] & 15) == 0) s->start[s->group_base[lead[u]] + rank[u] / 16] = uint16_t(pos);
    }
  __syncthreads();
}

// ---------------------------------------------------------------------------- shrink
constexpr int kShrinkWarps = kGroupThreads / 32;

// Blocks share out the groups of a window (`slots` of them) and the splits of K; within a split each of the eight warps takes
// a part of every group's product, and the parts meet in shared memory in a fixed order.
template <typename T, int NT>
__global__ void __launch_bounds__(kGroupThreads)
lora_shrink_kernel(const ShrinkArgs p, const int slots, const int skip_tiles) {
  constexpr int RP = NT * 8;
  extern __shared__ __align__(16) float part[];        // [warps][16][RP]
  __shared__ __align__(16) Groups s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = int(blockIdx.x) / slots * kWindow;
  after_previous_launch();
  build_groups(&s, written_before(p.ids), row0, p.rows, p.adapters, skip_tiles, false);
  const int steps = (p.k + 31) / 32;
  const int s0 = int((long long)steps * blockIdx.y / p.splits), s1 = int((long long)steps * (blockIdx.y + 1) / p.splits);
  const int from = s0 + (s1 - s0) * warp / kShrinkWarps, to = s0 + (s1 - s0) * (warp + 1) / kShrinkWarps;
  constexpr int U = NT <= 2 ? 4 : NT <= 4 ? 2 : 1;     // steps whose loads are in flight together
  for (int grp = int(blockIdx.x) % slots; grp < s.count; grp += slots) {
    const int at = s.start[grp];
    const int l = s.id[s.order[at]];
    // the group ends with the adapter's rows or after sixteen of them
    const int n = min(16, s.start[grp + 1] - at);
    const T* xr0 = static_cast<const T*>(p.x) + (long long)(row0 + s.order[at + min(g, n - 1)]) * p.k;
    const T* xr1 = static_cast<const T*>(p.x) + (long long)(row0 + s.order[at + min(g + 8, n - 1)]) * p.k;
    const T* al = static_cast<const T*>(p.a) + (long long)l * p.rank * p.k;
    float c[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) c[i][0] = c[i][1] = c[i][2] = c[i][3] = 0.f;
    for (int st = from; st < to; st += U) {
      uint4 x0[U], x1[U], b[U][NT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = (st + u) * 32 + t * 8;
        const bool ok = st + u < to && k < p.k;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        x0[u] = ok ? load16(xr0 + k) : zero;
        x1[u] = ok ? load16(xr1 + k) : zero;
#pragma unroll
        for (int i = 0; i < NT; ++i) b[u][i] = ok && i * 8 + g < p.rank ? load16(al + (long long)(i * 8 + g) * p.k + k) : zero;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t a0[4] = {x0[u].x, x1[u].x, x0[u].y, x1[u].y}, a1[4] = {x0[u].z, x1[u].z, x0[u].w, x1[u].w};
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          mma16816<T>(c[i], a0, b[u][i].x, b[u][i].y);
          mma16816<T>(c[i], a1, b[u][i].z, b[u][i].w);
        }
      }
    }
    float* slot = part + warp * 16 * RP;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      *reinterpret_cast<float2*>(slot + g * RP + i * 8 + t * 2) = make_float2(c[i][0], c[i][1]);
      *reinterpret_cast<float2*>(slot + (g + 8) * RP + i * 8 + t * 2) = make_float2(c[i][2], c[i][3]);
    }
    __syncthreads();
    float* out = p.v + (long long)blockIdx.y * p.rows * p.rank;
    for (int i = threadIdx.x; i < n * p.rank; i += kGroupThreads) {
      const int r = i / p.rank, j = i - r * p.rank;
      float sum = 0.f;
#pragma unroll
      for (int q = 0; q < kShrinkWarps; ++q) sum += part[(q * 16 + r) * RP + j];
      out[(long long)(row0 + s.order[at + r]) * p.rank + j] = sum;
    }
    __syncthreads();
  }
}

// The splits' sums added up, in their order.
__global__ void __launch_bounds__(256)
lora_fold_kernel(const float4* sums, float4* v, long long vecs, int splits) {
  after_previous_launch();
  const float4* planes = written_before(sums);
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < vecs; i += (long long)gridDim.x * 256) {
    float4 sum = fetch(planes + i);
    for (int s = 1; s < splits; ++s) {
      const float4 x = fetch(planes + s * vecs + i);
      sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
    }
    v[i] = sum;
  }
}

// ---------------------------------------------------------------------------- expand
// Blocks share out the groups of a window (`slots`) and the columns: a warp walks through `per_warp` groups of 32 columns
// with a row group's v in registers.  The columns are dealt to the four 8-wide MMAs so that a lane ends up with eight
// consecutive ones: base and output move 16 bytes a lane.
template <typename T, int KS>
__global__ void __launch_bounds__(kGroupThreads)
lora_expand_kernel(const ExpandArgs p, const int slots, const int per_warp, const int skip_tiles) {
  __shared__ __align__(16) Groups s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int row0 = int(blockIdx.x) / slots * kWindow;
  after_previous_launch();
  // rows without an adapter have to be written unless they are there already
  build_groups(&s, written_before(p.ids), row0, p.rows, p.adapters, skip_tiles, p.out != p.base);
  const int c0 = (int(blockIdx.y) * (kGroupThreads / 32) + warp) * per_warp * 32;
  if (c0 >= p.n) return;
  for (int grp = int(blockIdx.x) % slots; grp < s.count; grp += slots) {
    const int at = s.start[grp], n = min(16, s.start[grp + 1] - at);
    const int l = s.id[s.order[at]];
    const long long row[2] = {row0 + s.order[at + min(g, n - 1)], row0 + s.order[at + min(g + 8, n - 1)]};
    const bool live[2] = {g < n, g + 8 < n};
    float scale[2];
    uint32_t hi[KS][4], lo[KS][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      scale[h] = l >= 0 ? fetch(p.scaling + l) : 0.f;
      float4 x[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) x[ks] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (l >= 0 && live[h]) {
        const float* from = p.v + row[h] * p.rank + t * 4;
#pragma unroll 4
        for (int q = 0; q < p.splits; ++q, from += (long long)p.rows * p.rank) {
          float4 v[KS];                          // all in flight together
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
            v[ks] = ks * 16 + t * 4 < p.rank ? fetch(reinterpret_cast<const float4*>(from + ks * 16)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) { x[ks].x += v[ks].x; x[ks].y += v[ks].y; x[ks].z += v[ks].z; x[ks].w += v[ks].w; }
        }
      }
      if constexpr (std::is_same<T, __half>::value) {
        float amax = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          amax = fmaxf(amax, fmaxf(fmaxf(finite_abs(x[ks].x), finite_abs(x[ks].y)), fmaxf(finite_abs(x[ks].z), finite_abs(x[ks].w))));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int e = scale_exponent(amax);
        const float down = exp2i(-e);
        scale[h] *= exp2i(e);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) { x[ks].x *= down; x[ks].y *= down; x[ks].z *= down; x[ks].w *= down; }
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        split2<T>(x[ks].x, x[ks].y, hi[ks][h], lo[ks][h]);
        split2<T>(x[ks].z, x[ks].w, hi[ks][2 + h], lo[ks][2 + h]);
      }
    }
    const T* bl = static_cast<const T*>(p.b) + (long long)max(l, 0) * p.n * p.rank;
    for (int cg = 0; cg < per_warp && c0 + cg * 32 < p.n; ++cg) {
      const int col = c0 + cg * 32 + t * 8;      // this lane's eight columns
      uint4 y[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        y[h] = p.base && live[h] && col < p.n ? *reinterpret_cast<const uint4*>(static_cast<const T*>(p.base) + row[h] * p.n + col)
                                              : make_uint4(0, 0, 0, 0);
      float c[4][4], d[4][4];                    // products with the high parts, with the remainders
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[j][i] = d[j][i] = 0.f;
      if (l >= 0) {
        uint2 b[KS][4];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int k = ks * 16 + t * 4, bc = c0 + cg * 32 + 8 * (g >> 1) + 2 * j + (g & 1);
            b[ks][j] = bc < p.n && k < p.rank ? fetch(reinterpret_cast<const uint2*>(bl + (long long)bc * p.rank + k))
                                              : make_uint2(0, 0);
          }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mma16816<T>(c[j], hi[ks], b[ks][j].x, b[ks][j].y);
            mma16816<T>(d[j], lo[ks], b[ks][j].x, b[ks][j].y);
          }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) c[j][i] = of_two_parts(c[j][i], d[j][i]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!live[h] || col >= p.n) continue;
        uint4 o = y[h];
        if (l >= 0) {
          uint32_t* ow = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 q = unpack2<T>(ow[j]);
            ow[j] = pack2<T>(fmaf(scale[h], c[j][h * 2], q.x), fmaf(scale[h], c[j][h * 2 + 1], q.y));
          }
        }
        *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + row[h] * p.n + col) = o;
      }
    }
  }
}

// ---------------------------------------------------------------------------- gradients of the adapters
constexpr int kWgThreads = 256, kWgRows = 32, kWgList = 1024;
constexpr int kWgXStride = kWgCols * 2 + 16;     // 16 bytes of skew: a matrix's eight rows lie in different banks

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <int NT> constexpr int wg_stages() { return NT <= 4 ? 4 : 3; }     // two blocks an SM
template <int NT> constexpr int wg_v_stride() { return NT * 16 + 16; }
template <int NT> constexpr size_t wg_smem() {
  return size_t(wg_stages<NT>()) * kWgRows * (kWgXStride + NT * 32) + 2 * 2 * kWgRows * size_t(wg_v_stride<NT>());
}

// A block takes 256 columns (and up to 64 ranks) of a gradient and one split of the rows, and goes through the adapters with
// rows in it (of its group): it lists an adapter's rows by scanning the ids, gathers them 32 at a time (cp.async, three or two
// chunks in flight) and contracts over them; both operands are read across their rows with transposing ldmatrix.  Chunks of
// v share a running power of two; when a chunk needs a larger one the sums are brought to it.
template <int NT>
__global__ void __launch_bounds__(kWgThreads, 2)
lora_wgrad_kernel(const AdapterGradArgs p) {
  constexpr int RP = NT * 8, VS = wg_v_stride<NT>(), kStages = wg_stages<NT>();
  using T = __half;
  extern __shared__ __align__(16) uint8_t sm[];
  uint8_t* xs = sm;                                                     // [stages][32][kWgXStride]
  float* vf = reinterpret_cast<float*>(sm + kStages * kWgRows * kWgXStride);      // [stages][32][RP]
  uint8_t* vh = sm + kStages * kWgRows * (kWgXStride + RP * 4);       // [2][hi, lo][32][VS]
  __shared__ int list[kWgList + kWgRows], warp_n[8], next_adapter;
  __shared__ float warp_max[8];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const bool second = int(blockIdx.x) >= p.g[0].tiles;
  const AdapterGrad q = second ? p.g[1] : p.g[0];
  const int col0 = (second ? int(blockIdx.x) - p.g[0].tiles : int(blockIdx.x)) * kWgCols;
  const int j0 = int(blockIdx.z) * kWgRank;      // first of this block's ranks
  const int split = int(blockIdx.y) / p.groups, group = int(blockIdx.y) - split * p.groups;
  const int others = p.groups - 1;               // an adapter's group is its number modulo `groups`, a power of two
  const int begin = int((long long)p.rows * split / p.splits), end = int((long long)p.rows * (split + 1) / p.splits);
  const T* X = static_cast<const T*>(q.x);
  const long long mat = (long long)q.cols * p.rank;
  after_previous_launch();
  const int* ids = written_before(p.ids);

  // the smallest adapter of the group above `l` with rows here, or p.adapters
  auto find_next = [&](int l) -> int {
    if (tid == 0) next_adapter = p.adapters;
    __syncthreads();
    int best = p.adapters;
    for (int i = begin + tid; i < end; i += kWgThreads) {
      const int id = fetch(ids + i);
      if (id > l && id < best && (id & others) == group) best = id;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) best = min(best, __shfl_xor_sync(0xffffffffu, best, off));
    if (lane == 0) atomicMin(&next_adapter, best);
    __syncthreads();
    return next_adapter;
  };
  // adapters without rows here: zeros, or (several splits) the finishing launch is told
  auto skip_adapters = [&](int from, int to) {
    if (p.splits > 1) {
      if (blockIdx.x == 0 && blockIdx.z == 0)
        for (int l = from + tid * p.groups; l < to; l += kWgThreads * p.groups) p.present[(long long)split * p.adapters + l] = 0;
      return;
    }
    const int jn = min(kWgRank, p.rank - j0), cn = min(kWgCols, q.cols - col0);
    for (int l = from; l < to; l += p.groups)
      for (int i = tid; i < jn * cn; i += kWgThreads) {
        const long long at = q.rank_major ? (long long)(j0 + i / cn) * q.cols + col0 + i % cn
                                          : (long long)(col0 + i / jn) * p.rank + j0 + i % jn;
        static_cast<T*>(q.out)[(long long)l * mat + at] = T(0.f);
      }
  };

  // The sums of adapter l.  High parts and remainders share them; an adapter whose sums have a NaN is gone through once more
  // (`first` false) with the high parts alone, for the sums that are then not finite: against an infinity the remainder would
  // turn them into NaN.  Returns whether this thread has one.
  auto sum_up = [&](int l, auto first) -> bool {
    int next = begin, taken = 0, have = 0;       // ids scanned, entries of the list used and in it (same in all threads)
    // appends rows of this adapter until the list holds a chunk or the rows are through
    auto refill = [&]() {
      if (have - taken >= kWgRows || next >= end) return;
      __syncthreads();                           // nobody reads the part that moves
      const int rest = have - taken;
      const int keep = tid < rest ? list[taken + tid] : 0;
      __syncthreads();
      if (tid < rest) list[tid] = keep;
      have = rest;
      taken = 0;
      while (have < kWgRows && next < end) {
        // 1024 ids, warp by warp 32 in a row
        uint32_t mine[4];
        int n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = next + (warp * 4 + i) * 32 + lane;
          mine[i] = __ballot_sync(0xffffffffu, at < end && fetch(ids + at) == l);
          n += __popc(mine[i]);
        }
        if (lane == 0) warp_n[warp] = n;
        __syncthreads();
        int pos = have, all = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (i < warp) pos += warp_n[i];
          all += warp_n[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if ((mine[i] >> lane) & 1) list[pos + __popc(mine[i] & ((1u << lane) - 1))] = next + (warp * 4 + i) * 32 + lane;
          pos += __popc(mine[i]);
        }
        have += all;
        next += kWgList;
        __syncthreads();
      }
    };
    // one chunk of up to 32 rows into a stage; returns its rows
    auto load = [&](int stage) -> int {
      refill();
      const int n = min(kWgRows, have - taken);
      if (n > 0) {
#pragma unroll
        for (int i0 = 0; i0 < kWgRows * (kWgCols / 8); i0 += kWgThreads) {
          const int i = i0 + tid, r = i / (kWgCols / 8), c = i - r * (kWgCols / 8);
          const bool ok = r < n && col0 + c * 8 < q.cols;
          const T* src = X + (long long)list[taken + (r < n ? r : 0)] * q.cols + (ok ? col0 + c * 8 : 0);
          cp_async16(smem_u32(xs + (stage * kWgRows + r) * kWgXStride + c * 16), src, ok);
        }
#pragma unroll
        for (int i0 = 0; i0 < kWgRows * (RP / 4); i0 += kWgThreads) {
          const int i = i0 + tid, r = i / (RP / 4), c = i - r * (RP / 4);
          if (i >= kWgRows * (RP / 4)) break;
          const bool ok = r < n && j0 + c * 4 < p.rank;
          const float* src = q.v + (long long)list[taken + (r < n ? r : 0)] * p.rank + (ok ? j0 + c * 4 : 0);
          cp_async16(smem_u32(vf + (stage * kWgRows + r) * RP + c * 4), src, ok);
        }
        taken += n;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      return n;
    };

    float c[2][NT][4];
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int i = 0; i < NT; ++i) c[f][i][0] = c[f][i][1] = c[f][i][2] = c[f][i][3] = 0.f;
    int exponent = -200, next_exponent = -200;   // of the sums, of the chunk converted last
    uint32_t filled = 0;                         // stages that hold rows
    // a chunk's v as high parts and remainders, into one of two buffers
    auto convert = [&](int i) {
      uint8_t* vb = vh + (i & 1) * 2 * kWgRows * VS;
      const float* vc = vf + (i % kStages) * kWgRows * RP;
      float down = 1.f;
      {
        float amax = 0.f;
#pragma unroll
        for (int e = tid; e < kWgRows * RP / 4; e += kWgThreads) {
          const float4 x = reinterpret_cast<const float4*>(vc)[e];
          amax = fmaxf(amax, fmaxf(fmaxf(finite_abs(x.x), finite_abs(x.y)), fmaxf(finite_abs(x.z), finite_abs(x.w))));
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        if (lane == 0) warp_max[warp] = amax;
        __syncthreads();
        #pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, warp_max[i]);
        const int e = scale_exponent(amax);
        if (amax > 0.f && e > next_exponent) next_exponent = e;
        down = next_exponent < -110 ? 1.f : exp2i(-next_exponent);
      }
#pragma unroll
      for (int e = tid; e < kWgRows * RP / 4; e += kWgThreads) {
        const int r = e / (RP / 4), j = e - r * (RP / 4);
        const float4 x = reinterpret_cast<const float4*>(vc)[e];
        uint2 h, w;
        split2<T>(x.x * down, x.y * down, h.x, w.x);
        split2<T>(x.z * down, x.w * down, h.y, w.y);
        *reinterpret_cast<uint2*>(vb + r * VS + j * 8) = h;
        *reinterpret_cast<uint2*>(vb + (kWgRows + r) * VS + j * 8) = w;
      }
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) filled |= load(s) > 0 ? 1u << s : 0u;
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncthreads();
    convert(0);                                  // an adapter in the list has a row
    // one barrier a chunk: chunk i is multiplied while chunk i + 1 is converted and a later one asked for
    for (int i = 0; (filled >> (i % kStages)) & 1; ++i) {
      const int stage = i % kStages;
      {
        if (next_exponent > exponent) {          // the scale that chunk i was converted with
          if (exponent >= -110) {
            const float f = exp2i(max(-126, exponent - next_exponent));
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
              for (int b = 0; b < NT; ++b) { c[a][b][0] *= f; c[a][b][1] *= f; c[a][b][2] *= f; c[a][b][3] *= f; }
          }
          exponent = next_exponent;
        }
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 3) : "memory");
      __syncthreads();                           // chunk i + 1 is here, chunk i converted, chunk i - 1 multiplied
      const int into = (i + kStages - 1) % kStages;
      const bool got = load(into) > 0;
      filled = (filled & ~(1u << into)) | (got ? 1u << into : 0u);
      if ((filled >> ((i + 1) % kStages)) & 1) convert(i + 1);
      uint8_t* vb = vh + (i & 1) * 2 * kWgRows * VS;
      const uint32_t xa = smem_u32(xs + stage * kWgRows * kWgXStride) +
                          ((lane >> 4) * 8 + (lane & 7)) * kWgXStride + (warp * 32 + ((lane >> 3) & 1) * 8) * 2;
      const uint32_t va = smem_u32(vb) + (((lane >> 3) & 1) * 8 + (lane & 7)) * VS + (lane >> 4) * 16;
#pragma unroll
      for (int k = 0; k < kWgRows / 16; ++k) {
        uint32_t a[2][4];
        ldmatrix_x4_trans(a[0], xa + k * 16 * kWgXStride);
        ldmatrix_x4_trans(a[1], xa + k * 16 * kWgXStride + 32);
#pragma unroll
        for (int j = 0; j < NT / 2; ++j) {
          uint32_t h[4], w[4];
          ldmatrix_x4_trans(h, va + k * 16 * VS + j * 32);
          ldmatrix_x4_trans(w, va + (kWgRows + k * 16) * VS + j * 32);
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            mma16816<T>(c[f][2 * j], a[f], h[0], h[1]);
            mma16816<T>(c[f][2 * j + 1], a[f], h[2], h[3]);
          }
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            if (!first) break;
            mma16816<T>(c[f][2 * j], a[f], w[0], w[1]);
            mma16816<T>(c[f][2 * j + 1], a[f], w[2], w[3]);
          }
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    const float s = (p.splits == 1 ? fetch(p.scaling + l) : 1.f);
    const float up = exponent >= -110 ? exp2i(exponent) : 1.f;
    uint64_t sums = 0;                           // looks for NaNs
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int col = col0 + warp * 32 + f * 16 + h * 8 + g, j = j0 + i * 8 + t * 2;
          if (col >= q.cols || j >= p.rank) continue;
          const float v0 = c[f][i][h * 2] * up * s, v1 = c[f][i][h * 2 + 1] * up * s;
          add_pair(sums, c[f][i][h * 2], c[f][i][h * 2 + 1]);
          const bool put0 = first || !isfinite(c[f][i][h * 2]), put1 = first || !isfinite(c[f][i][h * 2 + 1]);
          const long long at = q.rank_major ? (long long)j * q.cols + col : (long long)col * p.rank + j;
          const long long step = q.rank_major ? q.cols : 1;
          if (p.splits > 1) {
            float* o = q.partial + ((long long)split * p.adapters + l) * mat + at;
            if (put0) o[0] = v0;
            if (put1) o[step] = v1;
          } else {
            const uint32_t pk = pack2<T>(v0, v1);
            T* o = static_cast<T*>(q.out) + (long long)l * mat + at;
            if (put0) o[0] = reinterpret_cast<const T*>(&pk)[0];
            if (put1) o[step] = reinterpret_cast<const T*>(&pk)[1];
          }
        }
    return either_nan(sums);
  };

  int done = group;                               // adapters of the group below this one are dealt with
  for (int l = find_next(-1); l < p.adapters; l = find_next(l)) {
    skip_adapters(done, l);
    done = l + p.groups;
    if (p.splits > 1 && blockIdx.x == 0 && blockIdx.z == 0 && tid == 0) p.present[(long long)split * p.adapters + l] = 1;
    const bool undefined = sum_up(l, std::true_type());
    // from here on the list and the stages are free for the next adapter
    if (__syncthreads_or(undefined)) {
      sum_up(l, std::false_type());
      __syncthreads();
    }
  }
  skip_adapters(done, p.adapters);
}

// out = s_l * sum of the splits' partials that hold rows of the adapter, in split order.
template <typename T>
__global__ void __launch_bounds__(256)
lora_wgrad_finish_kernel(const AdapterGradArgs p) {
  const AdapterGrad q = p.g[blockIdx.y];
  if (q.out == nullptr) return;
  const long long mat = (long long)q.cols * p.rank, all = mat * p.adapters;
  after_previous_launch();
  const float* partial = written_before(q.partial);
  const int* present = written_before(p.present);
  const float* scaling = written_before(p.scaling);
  for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; i < all; i += (long long)gridDim.x * 1024) {
    const int l = int(i / mat);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    bool any = false;
    for (int s = 0; s < p.splits; ++s) {
      if (fetch(present + (long long)s * p.adapters + l) == 0) continue;
      const float4 v = fetch(reinterpret_cast<const float4*>(partial + s * all + i));
      sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
      any = true;
    }
    const float f = any ? fetch(scaling + l) : 0.f;
    uint2 o;
    o.x = pack2<T>(sum.x * f, sum.y * f);
    o.y = pack2<T>(sum.z * f, sum.w * f);
    *reinterpret_cast<uint2*>(static_cast<T*>(q.out) + i) = o;
  }
}

// dst[m][c][r] = src[m][r][c] for two sets of matrices (blockIdx.y: of the first, then of the second), 64 x 64 tiles, 16 bytes
// in and out of global memory (both sizes are multiples of 8).
struct TransposeArgs {
  const uint16_t* src[2];
  uint16_t* dst[2];
  int rows[2], cols[2], mats;
};
__global__ void __launch_bounds__(256)
lora_transpose_kernel(const TransposeArgs p) {
  __shared__ uint16_t tile[64][66];
  const int which = int(blockIdx.y) >= p.mats;
  const int rows = p.rows[which], cols = p.cols[which], across = (cols + 63) / 64;
  const long long mat = (long long)(int(blockIdx.y) - which * p.mats) * rows * cols;
  const uint16_t* src = p.src[which] + mat;
  uint16_t* dst = p.dst[which] + mat;
  after_previous_launch();
  src = written_before(src);
  for (int t = blockIdx.x; t < across * ((rows + 63) / 64); t += gridDim.x) {
    const int c0 = t % across * 64, r0 = t / across * 64, x = (threadIdx.x & 7) * 8, y = threadIdx.x >> 3;
#pragma unroll
    for (int i = y; i < 64; i += 32)
      if (r0 + i < rows && c0 + x < cols) {
        const uint4 v = fetch(reinterpret_cast<const uint4*>(src + (long long)(r0 + i) * cols + c0 + x));
        uint32_t* to = reinterpret_cast<uint32_t*>(&tile[i][x]);
        to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
      }
    __syncthreads();
#pragma unroll
    for (int i = y; i < 64; i += 32)
      if (c0 + i < cols && r0 + x < rows) {
        uint32_t v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = uint32_t(tile[x + u * 2][i]) | uint32_t(tile[x + u * 2 + 1][i]) << 16;
        *reinterpret_cast<uint4*>(dst + (long long)(c0 + i) * rows + r0 + x) = make_uint4(v[0], v[1], v[2], v[3]);
      }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------- host
// Tiles of 128 rows from 512 rows on.  Both ways, whole calls, 4096 -> 4096, bf16, us on one B200 (tiles / groups of 16 rows):
// 4 adapters in runs: 256 rows, rank 16 14.4 / 13.3, rank 128 21.4 / 37.3; 512 rows 14.4 / 16.9 and 20.2 / 43.5; 8192 rows
// 48.1 / 86.3 and 66.1 / 284.  8 adapters in runs, 512 rows: 15.8 / 24.0 and 30.3 / 49.2.  16 adapters in any order (tiles then
// only add launches that find nothing to do): 256 rows 21.7 / 13.1 and 48.8 / 41.3; 512 rows 28.4 / 20.7 and 69.9 / 64.3;
// 8192 rows 132 / 87.6 and 411 / 323.
static bool on_tiles(int rows) { return rows >= 512; }

static int lora_check(const char* what, int rows, int k, int n, int rank, int adapters, int dtype) {
  char msg[160];
  const char* why = nullptr;
  if (rows < 0) why = "rows < 0";
  else if (rows > kMostRows) why = "rows must not exceed 2^31 - 1025";
  else if (k < 8 || k % 8 || n < 8 || n % 8) why = "k and n must be positive multiples of 8";
  else if (k > (1 << 29) || n > (1 << 29)) why = "k and n must not exceed 2^29";       // the tiles count bytes in 32 bits
  else if (rank < 8 || rank % 8 || rank > kLoraMaxRank) why = "rank must be a multiple of 8 in [8, 128]";
  else if (adapters < 1 || adapters > 32767) why = "adapters must be in [1, 32767]";
  else if (dtype != FLYMOE_BF16 && dtype != FLYMOE_F16) why = "dtype must be F16 or BF16";
  if (why == nullptr) return FLYMOE_OK;
  snprintf(msg, sizeof(msg), "%s: %s", what, why);
  set_last_error_msg(msg);
  return FLYMOE_ERR_INVALID_ARGUMENT;
}

// Pieces of k that a shrink's sums are cut into.
static int shrink_splits(int rows, int k) {
  if (rows < 1) return 1;
  if (on_tiles(rows)) {
    // A tile of 128 rows for every SM, at least four K blocks of 64 in a piece; two for every SM where a piece still has 16.
    // us of a call with 512 columns of output, pieces for one / for two tiles an SM: 4096 rows of 2304 17.5 / 19.3, 2048 of
    // 7168 17.2 / 18.0, 8192 of 4096 29.3 / 28.3, 16384 of 4096 46.5 / 43.6.
    const int tiles = ceil_div(rows, 128);
    return std::max({1, std::min({kLoraMaxSplits, sm_count() / tiles, k / 256}),
                     std::min({kLoraMaxSplits, 2 * sm_count() / tiles, k / 1024})});
  }
  // blocks of 16 rows for three on every SM, at least sixteen 32-wide steps (two a warp) in a piece
  return std::max(1, std::min({kLoraMaxSplits, 3 * sm_count() / ceil_div(rows, 16), ceil_div(k, 32) / 16}));
}
// Groups that a window of up to 512 rows can hold: one for every sixteen rows and one for every adapter's last.
static int window_groups(int rows, int adapters) {
  const int n = std::min(rows, kWindow);
  return std::min(n, n / 16 + std::min(adapters + 1, n));
}
template <typename T, int NT>
static int launch_shrink(const ShrinkArgs& p, int skip_tiles, cudaStream_t stream) {
  auto* kernel = lora_shrink_kernel<T, NT>;
  constexpr int smem = kShrinkWarps * 16 * NT * 8 * 4;
  static SmemLimitSeen seen;
  FLYMOE_CUDA_CHECK(allow_smem(reinterpret_cast<const void*>(kernel), smem, seen));
  // three blocks for every SM where there are that many groups
  const int windows = ceil_div(p.rows, kWindow);
  const int slots = std::max(1, std::min(window_groups(p.rows, p.adapters), 3 * sm_count() / (windows * p.splits)));
  FLYMOE_CUDA_CHECK(launch_closely(kernel, dim3(windows * slots, p.splits), kGroupThreads, smem, stream, p, slots, skip_tiles));
  return FLYMOE_OK;
}
template <typename T>
static int launch_shrink_rank(const ShrinkArgs& p, int skip, cudaStream_t s) {
  return p.rank <= 16 ? launch_shrink<T, 2>(p, skip, s) : p.rank <= 32 ? launch_shrink<T, 4>(p, skip, s)
       : p.rank <= 64 ? launch_shrink<T, 8>(p, skip, s) : launch_shrink<T, 16>(p, skip, s);
}
template <typename T, int KS>
static int launch_expand(const ExpandArgs& p, int skip_tiles, cudaStream_t stream) {
  const int windows = ceil_div(p.rows, kWindow), cols = ceil_div(p.n, 32), warps = kGroupThreads / 32;
  // Three blocks for every SM: row groups first, then columns.  A warp walks through up to eight column groups.
  const int want = 3 * sm_count();
  const int groups = window_groups(p.rows, p.adapters);
  const int spans = std::max(ceil_div(cols, 8 * warps),
                             std::min(ceil_div(cols, warps), want / int(std::min<long long>(want, (long long)windows * groups))));
  const int per_warp = ceil_div(cols, spans * warps);
  const int slots = int(std::max(1LL, std::min((long long)groups, want / ((long long)windows * spans))));
  FLYMOE_CUDA_CHECK(launch_closely(lora_expand_kernel<T, KS>, dim3(windows * slots, ceil_div(cols, per_warp * warps)), kGroupThreads,
                                   0, stream, p, slots, per_warp, skip_tiles));
  return FLYMOE_OK;
}
template <typename T>
static int launch_expand_rank(const ExpandArgs& p, int skip, cudaStream_t s) {
  return p.rank <= 16 ? launch_expand<T, 1>(p, skip, s) : p.rank <= 32 ? launch_expand<T, 2>(p, skip, s)
       : p.rank <= 64 ? launch_expand<T, 4>(p, skip, s) : launch_expand<T, 8>(p, skip, s);
}
template <int NT>
static int launch_wgrad_f16(const AdapterGradArgs& p, cudaStream_t stream) {
  auto* kernel = lora_wgrad_kernel<NT>;
  static SmemLimitSeen seen;
  FLYMOE_CUDA_CHECK(allow_smem(reinterpret_cast<const void*>(kernel), int(wg_smem<NT>()), seen));
  FLYMOE_CUDA_CHECK(launch_closely(kernel, dim3(p.g[0].tiles + p.g[1].tiles, p.splits * p.groups, ceil_div(p.rank, kWgRank)), kWgThreads,
                                   wg_smem<NT>(), stream, p));
  return FLYMOE_OK;
}
static int launch_wgrad(const AdapterGradArgs& p, bool bf, cudaStream_t s) {
  const int rc = bf ? launch_wgrad_sm100(p, s) : p.rank <= 16 ? launch_wgrad_f16<2>(p, s)
               : p.rank <= 32 ? launch_wgrad_f16<4>(p, s) : launch_wgrad_f16<8>(p, s);
  if (rc != FLYMOE_OK || p.splits == 1) return rc;
  const long long most = (long long)std::max(p.g[0].cols, p.g[1].cols) * p.rank * p.adapters / 4;
  FLYMOE_CUDA_CHECK(launch_closely(bf ? lora_wgrad_finish_kernel<__nv_bfloat16> : lora_wgrad_finish_kernel<__half>,
                                   dim3(unsigned(std::min<long long>((most + 255) / 256, 8LL * sm_count())), 2), 256, 0, s, p));
  return FLYMOE_OK;
}

// Floats of v: the sum, where there are several the splits behind it, and on tiles a number for each.
static long long v_planes(int rows, int splits, int rank) { return (splits > 1 ? splits + 1LL : 1LL) * rows * rank; }
static long long v_elems(int rows, int splits, int rank) {
  return v_planes(rows, splits, rank) + (on_tiles(rows) ? ceil_div(rows, 128) : 0);
}

// One product with the adapters and back: out = base + scaling * (x A^T) B^T, or with a_t / b_t (then `a` and `b` are only
// read where needs_transposed) for A and B given the other way round.  v: v_elems() floats; `kept`: null, or rows * rank
// floats (the first of v, or of their own) that hold x A^T afterwards.
struct Chain {
  const void *x, *a, *a_t, *base, *b, *b_t;
  void* out;                   // null: only x A^T
  float* v;
  const int* ids;
  const float* scaling;
  int rows, k, n, rank, adapters, dtype;
  float* kept;
};
static int run_chain(const Chain& c, cudaStream_t s) {
  const bool bf = c.dtype == FLYMOE_BF16, tiles = on_tiles(c.rows), others = !tiles || c.adapters > tile_limit(c.rank);
  const int skip = tiles ? tile_limit(c.rank) : 0;
  const int splits = shrink_splits(c.rows, c.k);
  float* sum = c.kept ? c.kept : c.v;
  float* planes = splits > 1 ? c.v + (long long)c.rows * c.rank : sum;
  int* counts = reinterpret_cast<int*>(c.v + v_planes(c.rows, splits, c.rank));
  ShrinkArgs sh = {c.x, c.a, c.ids, planes, counts, c.rows, c.k, c.rank, c.adapters, splits, 0};
  int rc = FLYMOE_OK;
  if (others) rc = bf ? launch_shrink_rank<__nv_bfloat16>(sh, skip, s) : launch_shrink_rank<__half>(sh, skip, s);
  if (rc == FLYMOE_OK && tiles) {
    if (c.a_t) { sh.a = c.a_t; sh.transposed = 1; }
    rc = launch_shrink_sm100(sh, bf, s);
  }
  if (rc != FLYMOE_OK) return rc;
  // tiles read a row's v once for every block that works on it, and the gradient wants it whole: one sum, not several
  const bool fold = splits > 1 && (tiles || c.kept);
  if (fold) {
    const long long vecs = (long long)c.rows * c.rank / 4;
    FLYMOE_CUDA_CHECK(launch_closely(lora_fold_kernel, unsigned(std::min<long long>((vecs + 255) / 256, 4LL * sm_count())), 256, 0, s,
                                     reinterpret_cast<const float4*>(planes), reinterpret_cast<float4*>(sum), vecs, splits));
  }
  if (!c.out) return FLYMOE_OK;
  ExpandArgs ex = {c.base, fold ? sum : planes, c.b, c.ids, c.scaling, c.out, counts, c.rows, c.n, c.rank, c.adapters,
                   fold ? 1 : splits, 0};
  if (others) rc = bf ? launch_expand_rank<__nv_bfloat16>(ex, skip, s) : launch_expand_rank<__half>(ex, skip, s);
  if (rc == FLYMOE_OK && tiles) {
    if (c.b_t) { ex.b = c.b_t; ex.transposed = 1; }
    rc = launch_expand_sm100(ex, bf, s);
  }
  return rc;
}
// Whether a backward pass reads A and B through the kernels of this file, which want the contraction along a row.
static bool needs_transposed(int rows, int rank, int adapters) { return !on_tiles(rows) || adapters > tile_limit(rank); }

// Blocks for every place on the device (two an SM) that the adapters' gradients are shared out to, besides their columns:
// pieces of the batch, whose blocks have like amounts of rows however the adapters share them, and groups of adapters, which
// need no partial sums but have like amounts only where the adapters have.  Pieces as long as their sums, written and read
// again, move at most the bytes of the rows where every piece has every adapter, with at least 256 rows in a piece;
// then groups.  Pieces only: 4096 rows in any order of 64 adapters of rank 64 took 404 us instead of 77.  Groups from half the
// bytes of the rows on: 8192 rows in runs of 4 adapters of rank 64 took 91 us instead of 52, in any order of 16 adapters of
// rank 16 66 instead of 87.
static int wgrad_places(int k, int n, int rank) {
  return 2 * sm_count() / ((ceil_div(k, kWgCols) + ceil_div(n, kWgCols)) * ceil_div(rank, kWgRank));
}
static int wgrad_splits(int rows, int k, int n, int rank, int adapters) {
  const long long fit = rows / (4LL * adapters * rank);
  return int(std::max(1LL, std::min({(long long)kLoraMaxSplits, (long long)wgrad_places(k, n, rank), fit, rows / 256LL})));
}
static int wgrad_groups(int splits, int k, int n, int rank, int adapters) {
  const int most = std::min(wgrad_places(k, n, rank) / splits, adapters);
  int groups = 1;
  while (groups * 2 <= most) groups *= 2;
  return groups;
}
// The backward pass's scratch, in floats: dv | A transposed | B transposed | partial sums, 16-byte aligned each.
struct BackwardScratch {
  long long dv, a_t, b_t, partial, total;
  int dv_splits, splits;
};
static BackwardScratch backward_scratch(int rows, int k, int n, int rank, int adapters) {
  BackwardScratch w;
  auto up4 = [](long long x) { return (x + 3) / 4 * 4; };
  w.dv_splits = shrink_splits(rows, n);
  w.splits = wgrad_splits(rows, k, n, rank, adapters);
  const bool both = needs_transposed(rows, rank, adapters);
  const long long weights = (long long)adapters * rank;
  w.dv = 0;
  w.a_t = up4(v_elems(rows, w.dv_splits, rank));
  w.b_t = w.a_t + (both ? up4(weights * k / 2) : 0);
  w.partial = w.b_t + (both ? up4(weights * n / 2) : 0);
  w.total = w.partial + (w.splits > 1 ? up4((long long)w.splits * adapters * ((long long)rank * ((long long)k + n) + 1)) : 0);
  return w;
}

}  // namespace flymoe

extern "C" int64_t flymoe_lora_v_elems(int rows, int k, int rank) {
  if (rows < 1 || k < 8 || rank < 8) return 0;
  return flymoe::v_elems(rows, flymoe::shrink_splits(rows, k), rank);
}

extern "C" int flymoe_lora_add(void* out, const void* base, const void* x, const void* a, const void* b, const int32_t* ids,
                               const float* scaling, float* v, int64_t v_floats, int rows, int k, int n, int rank, int adapters,
                               int keep_v, int dtype, void* stream) {
  return flymoe_lora_forward(out, base, x, a, b, ids, scaling, keep_v ? v : nullptr, v, v_floats, rows, k, n, rank, adapters, dtype,
                             stream);
}

extern "C" int flymoe_lora_forward(void* out, const void* base, const void* x, const void* a, const void* b, const int32_t* ids,
                                   const float* scaling, float* kept, float* v, int64_t v_floats, int rows, int k, int n,
                                   int rank, int adapters, int dtype, void* stream) {
  using namespace flymoe;
  int rc = lora_check("lora_add", rows, k, n, rank, adapters, dtype);
  if (rc != FLYMOE_OK || rows == 0) return rc;
  FLYMOE_REQUIRE(out && base && x && a && b && ids && scaling && v, "lora_add: null pointer");
  FLYMOE_REQUIRE(aligned16(out) && aligned16(base) && aligned16(x) && aligned16(a) && aligned16(b) && aligned16(v) &&
                     aligned16(kept),
                 "lora_add: pointers must be 16-byte aligned");
  if (v_floats < v_elems(rows, shrink_splits(rows, k), rank)) {
    set_last_error_msg("lora_add: v is smaller than flymoe_lora_v_elems()");
    return FLYMOE_ERR_WORKSPACE;
  }
  return run_chain({x, a, nullptr, base, b, nullptr, out, v, ids, scaling, rows, k, n, rank, adapters, dtype, kept},
                   static_cast<cudaStream_t>(stream));
}

extern "C" int64_t flymoe_lora_backward_workspace_elems(int rows, int k, int n, int rank, int adapters) {
  if (rows < 1 || k < 8 || n < 8 || rank < 8 || adapters < 1) return 4;
  return flymoe::backward_scratch(rows, k, n, rank, adapters).total;
}

extern "C" int flymoe_lora_backward(void* dx, void* da, void* db, const void* dout, const void* x, const void* a, const void* b,
                                    const int32_t* ids, const float* scaling, const float* v, float* workspace,
                                    int64_t workspace_elems, int rows, int k, int n, int rank, int adapters, int dtype,
                                    void* stream) {
  using namespace flymoe;
  int rc = lora_check("lora_backward", rows, k, n, rank, adapters, dtype);
  if (rc != FLYMOE_OK || (!dx && !da && !db)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t a_bytes = size_t(adapters) * rank * k * 2, b_bytes = size_t(adapters) * rank * n * 2;
  if (rows == 0) {
    if (da) FLYMOE_CUDA_CHECK(cudaMemsetAsync(da, 0, a_bytes, s));
    if (db) FLYMOE_CUDA_CHECK(cudaMemsetAsync(db, 0, b_bytes, s));
    return FLYMOE_OK;
  }
  FLYMOE_REQUIRE(dout && x && a && b && ids && scaling && (v || !db) && workspace, "lora_backward: null pointer");
  FLYMOE_REQUIRE(aligned16(dx) && aligned16(da) && aligned16(db) && aligned16(dout) && aligned16(x) && aligned16(a) &&
                     aligned16(b) && aligned16(v) && aligned16(workspace), "lora_backward: pointers must be 16-byte aligned");
  const BackwardScratch w = backward_scratch(rows, k, n, rank, adapters);
  if (workspace_elems < w.total) {
    set_last_error_msg("lora_backward: the workspace is smaller than flymoe_lora_backward_workspace_elems()");
    return FLYMOE_ERR_WORKSPACE;
  }
  float* dv = workspace + w.dv;
  if (dx || da) {
    const void *a_t = nullptr, *b_t = nullptr;   // dv contracts over B's columns, dx over A's rows: both the other way round
    if (needs_transposed(rows, rank, adapters)) {
      TransposeArgs t = {};
      uint16_t* at = reinterpret_cast<uint16_t*>(workspace + w.a_t);
      uint16_t* bt = reinterpret_cast<uint16_t*>(workspace + w.b_t);
      t.src[0] = static_cast<const uint16_t*>(b); t.dst[0] = bt; t.rows[0] = n; t.cols[0] = rank;
      t.src[1] = static_cast<const uint16_t*>(a); t.dst[1] = at; t.rows[1] = rank; t.cols[1] = k;
      t.mats = adapters;
      const int tiles = ceil_div(std::max(k, n), 64) * ceil_div(rank, 64);
      FLYMOE_CUDA_CHECK(launch_closely(lora_transpose_kernel,
                                       dim3(std::max(1, std::min(tiles, 16 * sm_count() / adapters)), dx ? 2 * adapters : adapters),
                                       256, 0, s, t));
      a_t = at;
      b_t = bt;
    }
    rc = run_chain({dout, b_t, b, nullptr, a_t, a, dx, dv, ids, scaling, rows, n, k, rank, adapters, dtype, da ? dv : nullptr}, s);
    if (rc != FLYMOE_OK) return rc;
  }
  if (!da && !db) return FLYMOE_OK;
  AdapterGradArgs p = {};
  const long long piece = (long long)w.splits * adapters * rank;
  float* partial = workspace + w.partial;
  if (da) p.g[0] = {x, dv, da, partial, k, ceil_div(k, kWgCols), 1};
  if (db) p.g[1] = {dout, v, db, partial + piece * k, n, ceil_div(n, kWgCols), 0};
  p.present = reinterpret_cast<int*>(partial + piece * ((long long)k + n));
  p.ids = ids;
  p.scaling = scaling;
  p.rows = rows;
  p.rank = rank;
  p.adapters = adapters;
  p.splits = w.splits;
  p.groups = wgrad_groups(w.splits, k, n, rank, adapters);
  return launch_wgrad(p, dtype == FLYMOE_BF16, s);
}
