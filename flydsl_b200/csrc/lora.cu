// Low-rank adapters of many requests at once, beside a shared projection (16-bit operands).
//
//   out[m] = base[m] + s_l B_l (A_l x[m]),   l = ids[m];  a row whose id names no adapter passes through
//
// in two launches: shrink, v = x A_l^T (fp32 [rows, rank], summed over K), and expand, which adds s_l v B_l^T to the base.
// Rows may come in any order of adapters: a warp works on a fragment of 16 or 32 rows and goes through the distinct
// adapters among them, and of each product only that adapter's rows are kept (so nothing of one request, not even an
// infinity, reaches another).  The rank is the only small extent; both launches are bound by the bytes of x, the adapters
// in use, the base and the output.
//
// v enters the second product as the sum of two 16-bit numbers (high part and remainder, two MMAs), which keeps 16 (bf16)
// or 22 (fp16) bits of it: one rounding of the output is all that shows.  fp16 has few exponent bits, so there a row of v
// is brought to the same power of two first.
//
// Gradients use the same kernels: dv = dout B_l is a shrink with B transposed, dx = s_l dv A_l an expand with A transposed
// (the adapters are small next to the rows); dA_l = s_l sum dv^T x and dB_l = s_l sum dout^T v contract over an adapter's
// rows, found by scanning ids.  No atomics anywhere: results do not depend on the order of execution.
//
// All products run on mma.sync: the shapes are thin (rank 8 to 128), the bound is memory.  Operand fragments are read from
// global memory 16 or 8 bytes a lane: the contraction index may be permuted as long as both operands agree, so a lane takes
// consecutive elements where the instruction's layout has pairs.
#include <algorithm>
#include <stdio.h>
#include <type_traits>

#include "common.cuh"
#include "gemm_ptx.cuh"

namespace flymoe {

constexpr int kLoraMaxRank = 128;
constexpr int kLoraMaxSplits = 16;

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
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) { return pack_bf16x2(a, b); }
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) { return pack_f16x2(a, b); }
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
// Two floats as high parts and remainders.  Where the high part is not finite there is no remainder.
template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack2<T>(a, b);
  const float2 h = unpack2<T>(hi);
  lo = pack2<T>(isfinite(h.x) ? a - h.x : 0.f, isfinite(h.y) ? b - h.y : 0.f);
}
// 2^e and 2^-e with the largest of `amax`'s numbers at 2^13 .. 2^14 afterwards (fp16 overflows at 2^16).
__device__ __forceinline__ int scale_exponent(float amax) {
  if (!(amax > 0.f)) return 0;
  const int e = int((__float_as_uint(amax) >> 23) & 0xff) - 127;     // 128: infinite, NaN
  return e >= 128 ? 0 : max(-110, min(110, e - 13));
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float(uint32_t(127 + e) << 23); }
__device__ __forceinline__ float finite_abs(float x) { return isfinite(x) ? fabsf(x) : 0.f; }
__device__ __forceinline__ uint4 ldg16(const void* p) { return __ldg(static_cast<const uint4*>(p)); }
__device__ __forceinline__ bool in_use(int id, int adapters) { return id >= 0 && id < adapters; }

// ---------------------------------------------------------------------------- shrink
struct ShrinkArgs {
  const void* x;               // [rows, k]
  const void* a;               // [adapters, rank, k]
  const int* ids;              // [rows]
  float* v;                    // [splits, rows, rank]
  int rows, k, rank, adapters, splits;
};
constexpr int kShrinkWarps = 8;

// A block takes 16 rows and one split of K.  Its warps share out (adapter, part of the split): one adapter gets all eight
// warps, eight or more one warp each; the parts meet in shared memory in a fixed order.
template <typename T, int NT>
__global__ void __launch_bounds__(kShrinkWarps * 32)
lora_shrink_kernel(const ShrinkArgs p) {
  constexpr int RP = NT * 8;
  extern __shared__ float part[];                      // [parts][16][RP]
  __shared__ int row_id[16], list[16], count;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.x * 16;
  if (warp == 0) {
    int id = -1;
    if (lane < 16 && row0 + lane < p.rows) {
      id = __ldg(p.ids + row0 + lane);
      if (!in_use(id, p.adapters)) id = -1;
    }
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    const bool first = id >= 0 && (same & ((1u << lane) - 1)) == 0;
    const uint32_t firsts = __ballot_sync(0xffffffffu, first);
    if (first) list[__popc(firsts & ((1u << lane) - 1))] = id;
    if (lane < 16) row_id[lane] = id;
    if (lane == 0) count = __popc(firsts);
  }
  __syncthreads();
  const int d = count;
  const int parts = d == 0 ? 1 : d >= kShrinkWarps ? 1 : kShrinkWarps / d;
  const int steps = (p.k + 31) / 32;
  const int s0 = int((long long)steps * blockIdx.y / p.splits), s1 = int((long long)steps * (blockIdx.y + 1) / p.splits);
  const T* xr0 = static_cast<const T*>(p.x) + (long long)min(row0 + g, p.rows - 1) * p.k;
  const T* xr1 = static_cast<const T*>(p.x) + (long long)min(row0 + g + 8, p.rows - 1) * p.k;
  const int id0 = row_id[g], id1 = row_id[g + 8];
  constexpr int U = NT <= 2 ? 4 : NT <= 4 ? 2 : 1;     // steps whose loads are in flight together
  for (int item = warp; item < d * parts; item += kShrinkWarps) {
    const int which = item / parts, part_i = item - which * parts;
    const int l = list[which];
    const int from = s0 + (s1 - s0) * part_i / parts, to = s0 + (s1 - s0) * (part_i + 1) / parts;
    const T* al = static_cast<const T*>(p.a) + (long long)l * p.rank * p.k;
    float c[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) c[i][0] = c[i][1] = c[i][2] = c[i][3] = 0.f;
    for (int s = from; s < to; s += U) {
      uint4 x0[U], x1[U], b[U][NT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = (s + u) * 32 + t * 8;
        const bool ok = s + u < to && k < p.k;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        x0[u] = ok ? ldg16(xr0 + k) : zero;
        x1[u] = ok ? ldg16(xr1 + k) : zero;
#pragma unroll
        for (int i = 0; i < NT; ++i) b[u][i] = ok && i * 8 + g < p.rank ? ldg16(al + (long long)(i * 8 + g) * p.k + k) : zero;
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
    float* slot = part + part_i * 16 * RP;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      if (id0 == l) *reinterpret_cast<float2*>(slot + g * RP + i * 8 + t * 2) = make_float2(c[i][0], c[i][1]);
      if (id1 == l) *reinterpret_cast<float2*>(slot + (g + 8) * RP + i * 8 + t * 2) = make_float2(c[i][2], c[i][3]);
    }
  }
  __syncthreads();
  float* out = p.v + ((long long)blockIdx.y * p.rows + row0) * p.rank;
  for (int i = threadIdx.x; i < 16 * p.rank; i += kShrinkWarps * 32) {
    const int r = i / p.rank, j = i - r * p.rank;
    if (row0 + r >= p.rows) break;
    float sum = 0.f;
    if (row_id[r] >= 0)
      for (int q = 0; q < parts; ++q) sum += part[(q * 16 + r) * RP + j];
    out[i] = sum;
  }
}

// The splits' sums added up into the first, in their order.
__global__ void __launch_bounds__(256)
lora_fold_kernel(float4* __restrict__ v, long long vecs, int splits) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < vecs; i += (long long)gridDim.x * 256) {
    float4 sum = v[i];
    for (int s = 1; s < splits; ++s) {
      const float4 x = v[s * vecs + i];
      sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
    }
    v[i] = sum;
  }
}

// ---------------------------------------------------------------------------- expand
struct ExpandArgs {
  const void* base;            // [rows, n] or null (zeros); may be `out`
  const float* v;              // [splits, rows, rank]
  const void* b;               // [adapters, n, rank]
  const int* ids;
  const float* scaling;        // [adapters]
  void* out;                   // [rows, n]
  int rows, n, rank, adapters, splits;
  int row_groups, groups_per_warp;
};

// A warp takes 16 * MF rows and `groups_per_warp` groups of 32 columns.  The columns of a group are dealt to the four
// 8-wide MMAs so that a lane ends up with eight consecutive ones: base and output move 16 bytes a lane.
template <typename T, int KS, int MF>
__global__ void __launch_bounds__(128)
lora_expand_kernel(const ExpandArgs p) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int rg = int(w % p.row_groups);
  const int c0 = int(w / p.row_groups) * p.groups_per_warp * 32;
  if (c0 >= p.n) return;
  const int row0 = rg * 16 * MF;
  int my_id = -1;
  if (lane < 16 * MF && row0 + lane < p.rows) {
    my_id = __ldg(p.ids + row0 + lane);
    if (!in_use(my_id, p.adapters)) my_id = -1;
  }
  const uint32_t used = __ballot_sync(0xffffffffu, my_id >= 0);
  // the rows of this lane: g, g + 8 of every 16-row fragment
  int id[2 * MF];
  float scale[2 * MF];
  uint32_t hi[MF][KS][4], lo[MF][KS][4];
#pragma unroll
  for (int f = 0; f < MF; ++f)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = f * 16 + h * 8 + g, row = row0 + r;
      id[f * 2 + h] = __shfl_sync(0xffffffffu, my_id, r);
      const bool live = id[f * 2 + h] >= 0;
      scale[f * 2 + h] = live ? __ldg(p.scaling + id[f * 2 + h]) : 0.f;
      float4 x[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        x[ks] = make_float4(0.f, 0.f, 0.f, 0.f);
        const int k = ks * 16 + t * 4;
        if (live && k < p.rank)
          for (int s = 0; s < p.splits; ++s) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(p.v + ((long long)s * p.rows + row) * p.rank + k));
            x[ks].x += q.x; x[ks].y += q.y; x[ks].z += q.z; x[ks].w += q.w;
          }
      }
      if constexpr (std::is_same<T, __half>::value) {
        float amax = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          amax = fmaxf(amax, fmaxf(fmaxf(fabsf(x[ks].x), fabsf(x[ks].y)), fmaxf(fabsf(x[ks].z), fabsf(x[ks].w))));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int e = scale_exponent(amax);
        const float down = exp2i(-e);
        scale[f * 2 + h] *= exp2i(e);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) { x[ks].x *= down; x[ks].y *= down; x[ks].z *= down; x[ks].w *= down; }
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        split2<T>(x[ks].x, x[ks].y, hi[f][ks][h], lo[f][ks][h]);
        split2<T>(x[ks].z, x[ks].w, hi[f][ks][2 + h], lo[f][ks][2 + h]);
      }
    }
  const bool copies = p.out != p.base;           // rows without an adapter have to be written too
  for (int grp = 0; grp < p.groups_per_warp; ++grp) {
    const int col = c0 + grp * 32 + t * 8;       // this lane's eight columns
    if (c0 + grp * 32 >= p.n) break;
    uint4 y[2 * MF];
#pragma unroll
    for (int i = 0; i < 2 * MF; ++i) {
      const int row = row0 + i * 8 + g;
      y[i] = p.base && row < p.rows && col < p.n
                 ? *reinterpret_cast<const uint4*>(static_cast<const T*>(p.base) + (long long)row * p.n + col)
                 : make_uint4(0, 0, 0, 0);
    }
    if (copies) {
#pragma unroll
      for (int i = 0; i < 2 * MF; ++i) {
        const int row = row0 + i * 8 + g;
        if (id[i] < 0 && row < p.rows && col < p.n)
          *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (long long)row * p.n + col) = y[i];
      }
    }
    for (uint32_t left = used; left;) {
      const int l = __shfl_sync(0xffffffffu, my_id, __ffs(left) - 1);
      left &= ~__ballot_sync(0xffffffffu, my_id == l);
      const T* bl = static_cast<const T*>(p.b) + (long long)l * p.n * p.rank;
      float c[MF][4][4];
#pragma unroll
      for (int f = 0; f < MF; ++f)
#pragma unroll
        for (int j = 0; j < 4; ++j) c[f][j][0] = c[f][j][1] = c[f][j][2] = c[f][j][3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint2 b[4];
        const int k = ks * 16 + t * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int bc = c0 + grp * 32 + 8 * (g >> 1) + 2 * j + (g & 1);
          b[j] = bc < p.n && k < p.rank ? __ldg(reinterpret_cast<const uint2*>(bl + (long long)bc * p.rank + k))
                                        : make_uint2(0, 0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int f = 0; f < MF; ++f) {
            mma16816<T>(c[f][j], hi[f][ks], b[j].x, b[j].y);
            mma16816<T>(c[f][j], lo[f][ks], b[j].x, b[j].y);
          }
      }
#pragma unroll
      for (int i = 0; i < 2 * MF; ++i) {
        const int row = row0 + i * 8 + g;
        if (id[i] != l || col >= p.n) continue;
        const float s = scale[i];
        uint4 o;
        uint32_t* ow = reinterpret_cast<uint32_t*>(&o);
        const uint32_t* yw = reinterpret_cast<const uint32_t*>(&y[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 q = unpack2<T>(yw[j]);
          ow[j] = pack2<T>(fmaf(s, c[i >> 1][j][(i & 1) * 2], q.x), fmaf(s, c[i >> 1][j][(i & 1) * 2 + 1], q.y));
        }
        *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (long long)row * p.n + col) = o;
      }
    }
  }
}

// ---------------------------------------------------------------------------- gradients of the adapters
struct AdapterGrad {
  const void* x;               // [rows, cols]: x for dA, dout for dB
  const float* v;              // [rows, rank]: dv for dA, v for dB
  void* out;                   // dA [adapters, rank, cols], dB [adapters, cols, rank]
  float* partial;              // [splits, adapters, cols, rank] in out's order, when splits > 1
  int cols, tiles;
  int rank_major;              // dA: columns are the inner axis
};
struct AdapterGradArgs {
  AdapterGrad g[2];
  const int* ids;
  const float* scaling;
  int rows, rank, adapters, splits;
};
constexpr int kWgCols = 128, kWgRows = 32, kWgStages = 4, kWgList = 1024;
constexpr int kWgXStride = kWgCols * 2 + 16;     // 16 bytes of skew: eight rows of a matrix in eight different banks groups

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <int NT> constexpr int wg_v_stride() { return NT * 16 + 16; }
template <int NT> constexpr size_t wg_smem() {
  return size_t(kWgStages) * kWgRows * (kWgXStride + NT * 32) + 2 * 2 * kWgRows * size_t(wg_v_stride<NT>());
}

// A block takes 128 columns of one adapter's gradient and one split of the rows: it scans the ids, gathers the adapter's
// rows 32 at a time (cp.async, four chunks in flight) and contracts over them; both operands are read across their rows
// with transposing ldmatrix.  fp16: chunks of v share a running power of two; when a chunk needs a larger one the sums are
// brought to it.
template <typename T, int NT>
__global__ void __launch_bounds__(128)
lora_wgrad_kernel(const AdapterGradArgs p) {
  constexpr int RP = NT * 8, VS = wg_v_stride<NT>();
  constexpr bool kHalf = std::is_same<T, __half>::value;
  extern __shared__ __align__(16) uint8_t sm[];
  uint8_t* xs = sm;                                                     // [stages][32][kWgXStride]
  float* vf = reinterpret_cast<float*>(sm + kWgStages * kWgRows * kWgXStride);      // [stages][32][RP]
  uint8_t* vh = sm + kWgStages * kWgRows * (kWgXStride + RP * 4);       // [2][hi, lo][32][VS]
  __shared__ int list[kWgList + kWgRows], warp_n[4], list_n;
  __shared__ float warp_max[4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const bool second = int(blockIdx.x) >= p.g[0].tiles;
  const AdapterGrad q = second ? p.g[1] : p.g[0];
  const int col0 = (second ? int(blockIdx.x) - p.g[0].tiles : int(blockIdx.x)) * kWgCols;
  const int l = blockIdx.y;
  int next = int((long long)p.rows * blockIdx.z / p.splits);
  const int end = int((long long)p.rows * (blockIdx.z + 1) / p.splits);
  const T* X = static_cast<const T*>(q.x);

  if (tid == 0) list_n = 0;
  int taken = 0, have = 0;                       // entries of the list already used, entries in it (same in all threads)
  __syncthreads();
  // appends rows of this adapter until the list holds a chunk or the rows are through
  auto refill = [&]() {
    if (have - taken >= kWgRows || next >= end) return;
    __syncthreads();                             // nobody reads the part that moves
    const int rest = have - taken;
    const int keep = tid < rest ? list[taken + tid] : 0;
    __syncthreads();
    if (tid < rest) list[tid] = keep;
    have = rest;
    taken = 0;
    while (have < kWgRows && next < end) {
      // 1024 ids: eight a thread, in order
      const int at = next + tid * 8;
      uint32_t mine = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (at + i < end && __ldg(p.ids + at + i) == l) mine |= 1u << i;
      int before = __popc(mine);
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, before, off);
        if (lane >= off) before += o;
      }
      if (lane == 31) warp_n[warp] = before;
      __syncthreads();
      int base = have, all = 0;
      for (int i = 0; i < 4; ++i) {
        if (i < warp) base += warp_n[i];
        all += warp_n[i];
      }
      int pos = base + before - __popc(mine);
      for (; mine; mine &= mine - 1) list[pos++] = at + __ffs(mine) - 1;
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
      for (int i = tid; i < kWgRows * (kWgCols / 8); i += 128) {
        const int r = i / (kWgCols / 8), c = i - r * (kWgCols / 8);
        const bool ok = r < n && col0 + c * 8 < q.cols;
        const T* src = X + (long long)(r < n ? list[taken + r] : 0) * q.cols + (ok ? col0 + c * 8 : 0);
        cp_async16(smem_u32(xs + (stage * kWgRows + r) * kWgXStride + c * 16), src, ok);
      }
      for (int i = tid; i < kWgRows * (RP / 4); i += 128) {
        const int r = i / (RP / 4), c = i - r * (RP / 4);
        const bool ok = r < n && c * 4 < p.rank;
        const float* src = q.v + (long long)(r < n ? list[taken + r] : 0) * p.rank + (ok ? c * 4 : 0);
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
  int exponent = -200;
  int chunk_n[kWgStages];
#pragma unroll
  for (int s = 0; s < kWgStages - 1; ++s) chunk_n[s] = load(s);
  for (int i = 0;; ++i) {
    const int stage = i % kWgStages;
    int n = 0;
#pragma unroll
    for (int s = 0; s < kWgStages; ++s)
      if (s == stage) n = chunk_n[s];
    if (n == 0) break;
    asm volatile("cp.async.wait_group %0;" ::"n"(kWgStages - 2) : "memory");
    __syncthreads();
    // the chunk's v as high parts and remainders
    uint8_t* vb = vh + (i & 1) * 2 * kWgRows * VS;
    const float* vc = vf + stage * kWgRows * RP;
    float down = 1.f;
    if constexpr (kHalf) {
      float amax = 0.f;
      for (int e = tid; e < kWgRows * RP / 4; e += 128) {
        const float4 x = reinterpret_cast<const float4*>(vc)[e];
        amax = fmaxf(amax, fmaxf(fmaxf(finite_abs(x.x), finite_abs(x.y)), fmaxf(finite_abs(x.z), finite_abs(x.w))));
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
      if (lane == 0) warp_max[warp] = amax;
      __syncthreads();
      amax = fmaxf(fmaxf(warp_max[0], warp_max[1]), fmaxf(warp_max[2], warp_max[3]));
      const int e = scale_exponent(amax);
      if (amax > 0.f && e > exponent) {
        const float f = exponent < -110 ? 0.f : exp2i(max(-126, exponent - e));
        if (exponent >= -110) {
#pragma unroll
          for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int b = 0; b < NT; ++b) { c[a][b][0] *= f; c[a][b][1] *= f; c[a][b][2] *= f; c[a][b][3] *= f; }
        }
        exponent = e;
      }
      down = exponent < -110 ? 1.f : exp2i(-exponent);
    }
    for (int e = tid; e < kWgRows * RP / 4; e += 128) {
      const int r = e / (RP / 4), j = e - r * (RP / 4);
      const float4 x = reinterpret_cast<const float4*>(vc)[e];
      uint2 h, w;
      split2<T>(x.x * down, x.y * down, h.x, w.x);
      split2<T>(x.z * down, x.w * down, h.y, w.y);
      *reinterpret_cast<uint2*>(vb + r * VS + j * 8) = h;
      *reinterpret_cast<uint2*>(vb + (kWgRows + r) * VS + j * 8) = w;
    }
    const int into = (i + kWgStages - 1) % kWgStages;
    const int got = load(into);                  // the stage that chunk i - 1 used: all have passed the barrier above
#pragma unroll
    for (int s = 0; s < kWgStages; ++s)
      if (s == into) chunk_n[s] = got;
    __syncthreads();
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
          mma16816<T>(c[f][2 * j], a[f], w[0], w[1]);
          mma16816<T>(c[f][2 * j + 1], a[f], h[2], h[3]);
          mma16816<T>(c[f][2 * j + 1], a[f], w[2], w[3]);
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  const float s = (p.splits == 1 ? __ldg(p.scaling + l) : 1.f);
  const float up = kHalf && exponent >= -110 ? exp2i(exponent) : 1.f;
  const long long mat = (long long)q.cols * p.rank;
#pragma unroll
  for (int f = 0; f < 2; ++f)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int col = col0 + warp * 32 + f * 16 + h * 8 + g, j = i * 8 + t * 2;
        if (col >= q.cols || j >= p.rank) continue;
        const float v0 = c[f][i][h * 2] * up * s, v1 = c[f][i][h * 2 + 1] * up * s;
        const long long at = q.rank_major ? (long long)j * q.cols + col : (long long)col * p.rank + j;
        const long long step = q.rank_major ? q.cols : 1;
        if (p.splits > 1) {
          float* o = q.partial + ((long long)blockIdx.z * p.adapters + l) * mat + at;
          o[0] = v0;
          o[step] = v1;
        } else {
          const uint32_t pk = pack2<T>(v0, v1);
          T* o = static_cast<T*>(q.out) + (long long)l * mat + at;
          o[0] = reinterpret_cast<const T*>(&pk)[0];
          o[step] = reinterpret_cast<const T*>(&pk)[1];
        }
      }
}

// out = s_l * sum of the splits' partials, in split order.
template <typename T>
__global__ void __launch_bounds__(256)
lora_wgrad_finish_kernel(const AdapterGradArgs p) {
  for (int which = 0; which < 2; ++which) {
    const AdapterGrad q = p.g[which];
    if (q.out == nullptr) continue;
    const long long mat = (long long)q.cols * p.rank, all = mat * p.adapters;
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; i < all; i += (long long)gridDim.x * 1024) {
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int s = 0; s < p.splits; ++s) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(q.partial + s * all + i));
        sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
      }
      const float f = __ldg(p.scaling + i / mat);
      uint2 o;
      o.x = pack2<T>(sum.x * f, sum.y * f);
      o.y = pack2<T>(sum.z * f, sum.w * f);
      *reinterpret_cast<uint2*>(static_cast<T*>(q.out) + i) = o;
    }
  }
}

// dst[m][c][r] = src[m][r][c], 32 x 32 tiles.
__global__ void __launch_bounds__(256)
lora_transpose_kernel(const uint16_t* __restrict__ src, uint16_t* __restrict__ dst, int rows, int cols) {
  __shared__ uint16_t tile[32][34];
  const long long mat = (long long)blockIdx.z * rows * cols;
  const int c0 = blockIdx.x * 32, r0 = blockIdx.y * 32, x = threadIdx.x & 31, y = threadIdx.x >> 5;
  for (int i = y; i < 32; i += 8)
    if (r0 + i < rows && c0 + x < cols) tile[i][x] = src[mat + (long long)(r0 + i) * cols + c0 + x];
  __syncthreads();
  for (int i = y; i < 32; i += 8)
    if (c0 + i < cols && r0 + x < rows) dst[mat + (long long)(c0 + i) * rows + r0 + x] = tile[x][i];
}

// ---------------------------------------------------------------------------- host
static int lora_check(const char* what, int rows, int width, int rank, int adapters, int splits, int dtype) {
  char msg[160];
  const char* why = nullptr;
  if (rows < 0) why = "rows < 0";
  else if (width < 8 || width % 8) why = "k and n must be positive multiples of 8";
  else if (rank < 8 || rank % 8 || rank > kLoraMaxRank) why = "rank must be a multiple of 8 in [8, 128]";
  else if (adapters < 1 || adapters > 65535) why = "adapters must be in [1, 65535]";
  else if (splits < 1 || splits > kLoraMaxSplits) why = "splits must be in [1, 16]";
  else if (dtype != FLYMOE_BF16 && dtype != FLYMOE_F16) why = "dtype must be F16 or BF16";
  if (why == nullptr) return FLYMOE_OK;
  snprintf(msg, sizeof(msg), "%s: %s", what, why);
  set_last_error_msg(msg);
  return FLYMOE_ERR_INVALID_ARGUMENT;
}

template <typename T, int NT>
static int launch_shrink(const ShrinkArgs& p, cudaStream_t stream) {
  auto* kernel = lora_shrink_kernel<T, NT>;
  constexpr int smem = kShrinkWarps * 16 * NT * 8 * 4;
  static SmemLimitSeen seen;
  FLYMOE_CUDA_CHECK(allow_smem(reinterpret_cast<const void*>(kernel), smem, seen));
  kernel<<<dim3(ceil_div(p.rows, 16), p.splits), kShrinkWarps * 32, smem, stream>>>(p);
  FLYMOE_CUDA_CHECK(cudaGetLastError());
  return FLYMOE_OK;
}
template <typename T>
static int launch_shrink_rank(const ShrinkArgs& p, cudaStream_t s) {
  return p.rank <= 16 ? launch_shrink<T, 2>(p, s) : p.rank <= 32 ? launch_shrink<T, 4>(p, s)
       : p.rank <= 64 ? launch_shrink<T, 8>(p, s) : launch_shrink<T, 16>(p, s);
}
template <typename T, int KS, int MF>
static int launch_expand(ExpandArgs p, cudaStream_t stream) {
  p.row_groups = ceil_div(p.rows, 16 * MF);
  const long long groups = ceil_div(p.n, 32);
  // columns a warp walks through with its rows' v in registers: as many as leave every SM 16 warps
  const long long per = groups * p.row_groups / (16LL * sm_count());
  p.groups_per_warp = int(per < 1 ? 1 : per > 8 ? 8 : per);
  const long long warps = (long long)p.row_groups * ceil_div(int(groups), p.groups_per_warp);
  lora_expand_kernel<T, KS, MF><<<unsigned((warps + 3) / 4), 128, 0, stream>>>(p);
  FLYMOE_CUDA_CHECK(cudaGetLastError());
  return FLYMOE_OK;
}
template <typename T>
static int launch_expand_rank(const ExpandArgs& p, cudaStream_t s) {
  return p.rank <= 16 ? launch_expand<T, 1, 2>(p, s) : p.rank <= 32 ? launch_expand<T, 2, 2>(p, s)
       : p.rank <= 64 ? launch_expand<T, 4, 2>(p, s) : launch_expand<T, 8, 1>(p, s);
}
template <typename T, int NT>
static int launch_wgrad(const AdapterGradArgs& p, cudaStream_t stream) {
  auto* kernel = lora_wgrad_kernel<T, NT>;
  static SmemLimitSeen seen;
  FLYMOE_CUDA_CHECK(allow_smem(reinterpret_cast<const void*>(kernel), int(wg_smem<NT>()), seen));
  kernel<<<dim3(p.g[0].tiles + p.g[1].tiles, p.adapters, p.splits), 128, wg_smem<NT>(), stream>>>(p);
  FLYMOE_CUDA_CHECK(cudaGetLastError());
  if (p.splits > 1) {
    lora_wgrad_finish_kernel<T><<<sm_count() * 2, 256, 0, stream>>>(p);
    FLYMOE_CUDA_CHECK(cudaGetLastError());
  }
  return FLYMOE_OK;
}
template <typename T>
static int launch_wgrad_rank(const AdapterGradArgs& p, cudaStream_t s) {
  return p.rank <= 16 ? launch_wgrad<T, 2>(p, s) : p.rank <= 32 ? launch_wgrad<T, 4>(p, s)
       : p.rank <= 64 ? launch_wgrad<T, 8>(p, s) : launch_wgrad<T, 16>(p, s);
}

}  // namespace flymoe

extern "C" int flymoe_lora_shrink_splits(int rows, int k) {
  if (rows < 1 || k < 8) return 1;
  // enough blocks of 16 rows for two on every SM, at least eight 32-wide steps (one a warp) in a split
  const int groups = flymoe::ceil_div(rows, 16), steps = flymoe::ceil_div(k, 32);
  return std::max(1, std::min({flymoe::kLoraMaxSplits, 2 * flymoe::sm_count() / groups, steps / 8}));
}

extern "C" int flymoe_lora_shrink(float* v, const void* x, const void* a, const int32_t* ids, int rows, int k, int rank,
                                  int adapters, int splits, int fold, int dtype, void* stream) {
  using namespace flymoe;
  int rc = lora_check("lora_shrink", rows, k, rank, adapters, splits, dtype);
  if (rc != FLYMOE_OK || rows == 0) return rc;
  FLYMOE_REQUIRE(v && x && a && ids, "lora_shrink: null pointer");
  FLYMOE_REQUIRE(aligned16(x) && aligned16(a) && aligned16(v), "lora_shrink: pointers must be 16-byte aligned");
  const ShrinkArgs p = {x, a, ids, v, rows, k, rank, adapters, splits};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  rc = dtype == FLYMOE_BF16 ? launch_shrink_rank<__nv_bfloat16>(p, s) : launch_shrink_rank<__half>(p, s);
  if (rc != FLYMOE_OK || !fold || splits == 1) return rc;
  const long long vecs = (long long)rows * rank / 4;
  lora_fold_kernel<<<unsigned(std::min<long long>((vecs + 255) / 256, 4LL * sm_count())), 256, 0, s>>>(
      reinterpret_cast<float4*>(v), vecs, splits);
  FLYMOE_CUDA_CHECK(cudaGetLastError());
  return FLYMOE_OK;
}

extern "C" int flymoe_lora_expand(void* out, const void* base, const float* v, const void* b, const int32_t* ids,
                                  const float* scaling, int rows, int n, int rank, int adapters, int splits, int dtype,
                                  void* stream) {
  using namespace flymoe;
  const int rc = lora_check("lora_expand", rows, n, rank, adapters, splits, dtype);
  if (rc != FLYMOE_OK || rows == 0) return rc;
  FLYMOE_REQUIRE(out && v && b && ids && scaling, "lora_expand: null pointer");
  FLYMOE_REQUIRE(aligned16(out) && aligned16(base) && aligned16(v) && aligned16(b), "lora_expand: pointers must be 16-byte aligned");
  const ExpandArgs p = {base, v, b, ids, scaling, out, rows, n, rank, adapters, splits, 0, 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == FLYMOE_BF16 ? launch_expand_rank<__nv_bfloat16>(p, s) : launch_expand_rank<__half>(p, s);
}

extern "C" int flymoe_lora_add(void* out, const void* base, const void* x, const void* a, const void* b, const int32_t* ids,
                               const float* scaling, float* v, int rows, int k, int n, int rank, int adapters, int splits,
                               int dtype, void* stream) {
  const int rc = flymoe_lora_shrink(v, x, a, ids, rows, k, rank, adapters, splits, 0, dtype, stream);
  return rc != FLYMOE_OK ? rc
                         : flymoe_lora_expand(out, base, v, b, ids, scaling, rows, n, rank, adapters, splits, dtype, stream);
}

extern "C" int flymoe_lora_wgrad_splits(int rows, int k, int n, int adapters) {
  if (rows < 1 || k < 8 || n < 8 || adapters < 1) return 1;
  // four blocks for every SM, at least 512 rows in a split (its partial sums cost as much as they save below that)
  const long long blocks = (long long)adapters * (flymoe::ceil_div(k, flymoe::kWgCols) + flymoe::ceil_div(n, flymoe::kWgCols));
  const long long want = 4LL * flymoe::sm_count() / blocks;
  return int(std::max(1LL, std::min({(long long)flymoe::kLoraMaxSplits, want, (long long)rows / 512})));
}

extern "C" int flymoe_lora_wgrad(void* da, void* db, const void* x, const void* dout, const float* v, const float* dv,
                                 const int32_t* ids, const float* scaling, float* partial, int rows, int k, int n, int rank,
                                 int adapters, int splits, int dtype, void* stream) {
  using namespace flymoe;
  int rc = lora_check("lora_wgrad", rows, k, rank, adapters, splits, dtype);
  if (rc == FLYMOE_OK) rc = lora_check("lora_wgrad", rows, n, rank, adapters, splits, dtype);
  if (rc != FLYMOE_OK || (!da && !db)) return rc;
  FLYMOE_REQUIRE(scaling && (rows == 0 || ids), "lora_wgrad: null pointer");
  FLYMOE_REQUIRE(rows == 0 || ((!da || (x && dv)) && (!db || (dout && v))), "lora_wgrad: null pointer");
  FLYMOE_REQUIRE(splits == 1 || partial, "lora_wgrad: partial is needed for more than one split");
  FLYMOE_REQUIRE(aligned16(da) && aligned16(db) && aligned16(x) && aligned16(dout) && aligned16(v) && aligned16(dv) &&
                     aligned16(partial), "lora_wgrad: pointers must be 16-byte aligned");
  AdapterGradArgs p = {};
  float* partial_b = da && partial ? partial + (long long)splits * adapters * k * rank : partial;
  if (da) p.g[0] = {x, dv, da, partial, k, ceil_div(k, kWgCols), 1};
  if (db) p.g[1] = {dout, v, db, partial_b, n, ceil_div(n, kWgCols), 0};
  p.ids = ids;
  p.scaling = scaling;
  p.rows = rows;
  p.rank = rank;
  p.adapters = adapters;
  p.splits = splits;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == FLYMOE_BF16 ? launch_wgrad_rank<__nv_bfloat16>(p, s) : launch_wgrad_rank<__half>(p, s);
}

extern "C" int flymoe_lora_transpose(const void* src, void* dst, int mats, int rows, int cols, void* stream) {
  using namespace flymoe;
  FLYMOE_REQUIRE(mats >= 0 && mats <= 65535 && rows >= 1 && cols >= 1, "lora_transpose: bad sizes");
  FLYMOE_REQUIRE(ceil_div(rows, 32) <= 65535, "lora_transpose: too many rows");
  if (mats == 0) return FLYMOE_OK;
  FLYMOE_REQUIRE(src && dst, "lora_transpose: null pointer");
  lora_transpose_kernel<<<dim3(ceil_div(cols, 32), ceil_div(rows, 32), mats), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint16_t*>(src), static_cast<uint16_t*>(dst), rows, cols);
  FLYMOE_CUDA_CHECK(cudaGetLastError());
  return FLYMOE_OK;
}
