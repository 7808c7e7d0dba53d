// What the adapter kernels share: 16-bit packing, the two-part form of the middle factor, argument blocks.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace flymoe {

constexpr int kLoraMaxRank = 128;
constexpr int kLoraMaxSplits = 16;

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
// Sum of products with the high parts and with the remainders.
__device__ __forceinline__ float of_two_parts(float hi, float lo) { return isfinite(hi) ? hi + lo : hi; }
// Sums of many numbers, two at a time, that are NaN where one of the numbers is (or two infinities of either sign are there).
__device__ __forceinline__ void add_pair(uint64_t& sums, float a, float b) {
  asm("{\n\t.reg .b64 p;\n\tmov.b64 p, {%1, %2};\n\tadd.rn.f32x2 %0, %0, p;\n\t}" : "+l"(sums) : "f"(a), "f"(b));
}
__device__ __forceinline__ bool either_nan(uint64_t sums) {
  return isnan(__uint_as_float(uint32_t(sums))) || isnan(__uint_as_float(uint32_t(sums >> 32)));
}
// 2^e and 2^-e with the largest of `amax`'s numbers at 2^13 .. 2^14 afterwards (fp16 overflows at 2^16).
__device__ __forceinline__ int scale_exponent(float amax) {
  if (!(amax > 0.f)) return 0;
  const int e = int((__float_as_uint(amax) >> 23) & 0xff) - 127;     // 128: infinite, NaN
  return e >= 128 ? 0 : max(-110, min(110, e - 13));
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float(uint32_t(127 + e) << 23); }
__device__ __forceinline__ float finite_abs(float x) { return isfinite(x) ? fabsf(x) : 0.f; }
__device__ __forceinline__ bool in_use(int id, int adapters) { return id >= 0 && id < adapters; }

struct ShrinkArgs {
  const void* x;               // [rows, k]
  const void* a;               // [adapters, rank, k], or transposed [adapters, k, rank] (on tiles only)
  const int* ids;              // [rows]
  float* v;                    // [splits, rows, rank]
  int* counts;                 // on tiles: [tiles of 128 rows], distinct adapters of a tile, tile_limit() + 1 for more
  int rows, k, rank, adapters, splits, transposed;
};
struct ExpandArgs {
  const void* base;            // [rows, n] or null (zeros); may be `out`
  const float* v;              // [splits, rows, rank]; on tiles one split
  const void* b;               // [adapters, n, rank], or transposed [adapters, rank, n] (on tiles only)
  const int* ids;
  const float* scaling;        // [adapters]
  void* out;                   // [rows, n]
  const int* counts;           // on tiles: the shrink's
  int rows, n, rank, adapters, splits, transposed;
};

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
  int* present;                // [splits, adapters]: whether the split has rows of the adapter, when splits > 1
  int rows, rank, adapters, splits;
  int groups;                  // of adapters, a power of two: blockIdx.y = split * groups + group
};
constexpr int kWgCols = 256;                     // columns of a gradient a block sums up
constexpr int kWgRank = 64;                      // and its ranks; more are shared out

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}

// The launches of one operator follow each other closely (programmatic stream serialisation): the next one's blocks start,
// and set up what touches no global memory, while the last blocks of this one run.  Every kernel launched this way waits
// here before its first access to global memory; the wait ends when all launches before it are done.
//
// TMEM is taken between the two, never before the wait and never after the signal.  A block that held some while it waited
// could share an SM with a block of the launch that it waits for, which needs more than is left: neither
// tcgen05.alloc nor this wait has a limit.  The first thread of a block that signals does so for all of it.
//
// All that such a kernel reads may have been written while it already ran, inputs of a call among it (a call may read what the
// call before it wrote).  The read-only path (__ldg, const __restrict__) is for memory that nobody writes during the kernel,
// and a compiler may move it in front of the wait.  fetch() is an ordinary load that the compiler may move about, as long as
// its address is known: what it reads is written by no one after the wait, and addresses come from written_before(), which
// is defined behind the wait only, or from ids that were read through it.  (Loads in plain C++ stay under their conditions, one
// behind the other: shrink of 4096 rows, 64 adapters of rank 64, 125 us against 70.)
__device__ __forceinline__ void wait_for_previous_launch() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_launch_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void after_previous_launch() {        // for kernels without TMEM
  wait_for_previous_launch();
  let_next_launch_start();
}
template <typename T> __device__ __forceinline__ const T* written_before(const T* p) {
  asm volatile("" : "+l"(p)::"memory");
  return p;
}
__device__ __forceinline__ int fetch(const int* p) {
  int v;
  asm("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ float fetch(const float* p) {
  float v;
  asm("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ float4 fetch(const float4* p) {
  float4 v;
  asm("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 fetch(const uint2* p) {
  uint2 v;
  asm("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 fetch(const uint4* p) {
  uint4 v;
  asm("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
template <typename... Params, typename... Args>
inline cudaError_t launch_closely(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

// Tiles of 128 rows on tcgen05 (lora_sm100.cu), of which these launches take those with at most tile_limit(rank) distinct
// adapters among their rows; the kernels of lora.cu take the others, and batches of too few tiles.  As many as have room for
// their sums in TMEM.
constexpr int kTileAdapters = 8;
__host__ __device__ inline int tile_limit(int rank) { return rank <= 64 ? kTileAdapters : kTileAdapters / 2; }
int launch_shrink_sm100(const ShrinkArgs& p, int bf16, cudaStream_t stream);
int launch_expand_sm100(const ExpandArgs& p, int bf16, cudaStream_t stream);
int launch_wgrad_sm100(const AdapterGradArgs& p, cudaStream_t stream);           // bf16 (lora_grad_sm100.cu)

// Distinct adapters among the 128 ids that a warp holds, four a lane (negative: none): their number, most + 1 if there are
// more, and the first `most` of them in `list` (written by lane 0).
__device__ __forceinline__ int tile_adapters(const int* id, int lane, int most, int* list) {
  bool left[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) left[i] = id[i] >= 0;
  int count = 0;
  while (true) {
    const bool any = left[0] || left[1] || left[2] || left[3];
    const uint32_t who = __ballot_sync(0xffffffffu, any);
    if (who == 0 || count == most) return count + (who != 0);
    const int mine = left[0] ? id[0] : left[1] ? id[1] : left[2] ? id[2] : id[3];
    const int l = __shfl_sync(0xffffffffu, mine, __ffs(who) - 1);
    if (lane == 0 && list) list[count] = l;
    ++count;
#pragma unroll
    for (int i = 0; i < 4; ++i) left[i] = left[i] && id[i] != l;
  }
}
// A row's adapter, -1 for none and for rows behind the last.  ids: from written_before().
__device__ __forceinline__ int row_adapter(const int* ids, int row, int rows, int adapters) {
  if (row >= rows) return -1;
  const int id = fetch(ids + row);
  return in_use(id, adapters) ? id : -1;
}

}  // namespace flymoe
