// What the two kernels of the ragged grouped products share: arguments, segment tables, tile walk, epilogue arithmetic.
#pragma once
#include <cuda.h>

#include "common.cuh"
#include "gemm_ptx.cuh"

namespace flymoe {

constexpr int kRagK = 64;                        // K block
constexpr int kRagMaxExperts = 1024;

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

struct RaggedTables {
  int start[kRagMaxExperts + 1];                 // first row of an expert
  int tile0[kRagMaxExperts + 1];                 // first tile of an expert
};

// Segment bounds and tile counts.  Offsets come from the device, so they are taken into [0, rows] and made ascending
// here: whatever they hold, no access leaves the tensors.
template <int FORM, int TILE_M>
__device__ __forceinline__ void ragged_tables(const RaggedArgs& a, RaggedTables* c, int lane) {
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
      t = FORM == 2 ? a.m_tiles * a.n_tiles : (v - before + TILE_M - 1) / TILE_M * a.n_tiles;
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
  __device__ __forceinline__ void at(const RaggedArgs& a, const RaggedTables* c, int t, int form) {
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

// Eight sums as 16-bit values.
__device__ __forceinline__ uint4 pack8(const float* v, int bf16) {
  uint4 pk;
  if (bf16) {
    pk.x = pack_bf16x2(v[0], v[1]); pk.y = pack_bf16x2(v[2], v[3]);
    pk.z = pack_bf16x2(v[4], v[5]); pk.w = pack_bf16x2(v[6], v[7]);
  } else {
    pk.x = pack_f16x2(v[0], v[1]); pk.y = pack_f16x2(v[2], v[3]);
    pk.z = pack_f16x2(v[4], v[5]); pk.w = pack_f16x2(v[6], v[7]);
  }
  return pk;
}
// Rows that belong to no expert, in front of the first segment and behind the last, zeroed by `threads` threads of each CTA.
__device__ __forceinline__ void zero_uncovered_rows(const RaggedArgs& a, const RaggedTables* c, int thread, int threads) {
  const int lo = c->start[0], hi = c->start[a.experts];
  const long long vec = a.n_dim / 8, head = lo * vec, all = head + (a.rows - hi) * vec;
  uint4* out = static_cast<uint4*>(a.out);
  for (long long i = (long long)blockIdx.x * threads + thread; i < all; i += (long long)gridDim.x * threads)
    out[i < head ? i : (long long)hi * vec + i - head] = make_uint4(0, 0, 0, 0);
}

// CTA pairs (grouped_pair.cu).  form 0, 1: forward, input gradient; 2: weight gradient.
int launch_ragged_pair(int form, const void* p, const void* q, const RaggedArgs& a, int n, int k, cudaStream_t stream);

}  // namespace flymoe
