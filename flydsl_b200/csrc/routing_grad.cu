// The router around ragged expert rows, differentiable: tables of a unit-1 sort, rows into expert order, their weighted sum
// back into tokens, and the gradients of the sum and of the top-k softmax gate.  All of it is bound by HBM traffic.
#include <math_constants.h>

#include <algorithm>

#include "common.cuh"
#include "vec8.cuh"

namespace flymoe {

constexpr int kMaxRouteExperts = 1024;

// ---------------------------------------------------------------------------- tables
// row_index[t*k+s] = sorted row of pair (t, s) (preset to -1); offsets[e] = first row of expert e, from the ascending
// expert list by binary search.
__global__ void __launch_bounds__(256)
route_tables_kernel(const int* __restrict__ sorted_ids, const int* __restrict__ row_expert,
                    const int* __restrict__ num_valid_ids, int* __restrict__ row_index, int* __restrict__ offsets,
                    int num_tokens, int topk, int experts, int max_rows) {
  const int valid = min(__ldg(num_valid_ids), max_rows);
  const int first = blockIdx.x * blockDim.x + threadIdx.x, step = gridDim.x * blockDim.x;
  for (int e = first; e <= experts; e += step) {
    int lo = 0, hi = valid;
    while (lo < hi) { const int mid = (lo + hi) >> 1; if (__ldg(row_expert + mid) < e) lo = mid + 1; else hi = mid; }
    offsets[e] = lo;
  }
  for (int r = first; r < valid; r += step) {
    const int id = __ldg(sorted_ids + r);
    const int t = id_token(id), s = id_slot(id);
    if (t < num_tokens && s < topk) row_index[(long long)t * topk + s] = r;
  }
}

// ---------------------------------------------------------------------------- rows <-> pairs
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

struct Routed {
  const int* sorted_ids;       // [rows] (slot << 24) | token
  const int* num_valid_ids;    // rows of them in use
  const int* row_index;        // [tokens * topk] or -1
  int tokens, topk, rows;
  // Sorted row of a pair, or -1.  A pair counts where both tables name it, so neither a pair without a row nor tables
  // that do not belong together can lead out of the tensors or to one row twice.
  __device__ __forceinline__ int row_of(int t, int s) const {
    const int r = __ldg(row_index + (long long)t * topk + s);
    if (r < 0 || r >= min(__ldg(num_valid_ids), rows)) return -1;
    return __ldg(sorted_ids + r) == ((s << 24) | t) ? r : -1;
  }
  // Pair of a sorted row (t * topk + s), or -1 under the same rule.
  __device__ __forceinline__ long long pair_of(int r) const {
    if (r >= min(__ldg(num_valid_ids), rows)) return -1;
    const int id = __ldg(sorted_ids + r), t = id_token(id), s = id_slot(id);
    if (t >= tokens || s >= topk) return -1;
    const long long p = (long long)t * topk + s;
    return __ldg(row_index + p) == r ? p : -1;
  }
};

// dst[r] = src[token of r], zeros for a row without a pair; one warp per row, 16 bytes per lane and step.
__global__ void __launch_bounds__(256)
permute_rows_kernel(const uint4* __restrict__ src, uint4* __restrict__ dst, const Routed p, int row_vec) {
  const int lane = threadIdx.x & 31;
  const int warps = gridDim.x * (blockDim.x >> 5);
  for (int r = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); r < p.rows; r += warps) {
    const long long pair = p.pair_of(r);
    uint4* d = dst + (long long)r * row_vec;
    if (pair >= 0) {
      const uint4* x = src + pair / p.topk * row_vec;
      for (int i = lane; i < row_vec; i += 128) {                // four loads in flight per lane
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + 32 * j < row_vec) v[j] = __ldg(x + i + 32 * j);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + 32 * j < row_vec) d[i + 32 * j] = v[j];
      }
    } else {
      for (int i = lane; i < row_vec; i += 32) d[i] = make_uint4(0, 0, 0, 0);
    }
  }
}

// out[t] = sum_s weights[t, s] * rows[row of (t, s)], fp32 in slot order, rounded once; weights null: ones.
// A block per token: its rows are looked up once, then every thread has eight of their 16-byte pieces in flight.  4096
// tokens x 8 rows of 7168, bf16 (one B200): 86 us, with the look-up in every thread 159.
constexpr int kCombineSlots = 256;
template <typename T>
__global__ void __launch_bounds__(256)
combine_rows_kernel(const T* __restrict__ rows, const float* __restrict__ weights, T* __restrict__ out, const Routed p,
                    int dim) {
  __shared__ int row[kCombineSlots];
  __shared__ float weight[kCombineSlots];
  constexpr int kVec = 16 / sizeof(T);           // elements of a 16-byte piece
  for (int t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    if (int(threadIdx.x) < p.topk) {
      const int r = p.row_of(t, threadIdx.x);
      row[threadIdx.x] = r;
      weight[threadIdx.x] = r >= 0 && weights ? __ldg(weights + (long long)t * p.topk + threadIdx.x) : 1.f;
    }
    __syncthreads();
    for (int col = threadIdx.x * kVec; col < dim; col += 256 * kVec) {
      float acc[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) acc[i] = 0.f;
      for (int s0 = 0; s0 < p.topk; s0 += 8) {
        uint4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (s0 + j < p.topk && row[s0 + j] >= 0)
            v[j] = __ldg(reinterpret_cast<const uint4*>(rows + (long long)row[s0 + j] * dim + col));
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (s0 + j < p.topk && row[s0 + j] >= 0) {
            const T* x = reinterpret_cast<const T*>(&v[j]);
#pragma unroll
            for (int i = 0; i < kVec; ++i) acc[i] = fmaf(float(x[i]), weight[s0 + j], acc[i]);
          }
      }
      uint4 o;
      T* y = reinterpret_cast<T*>(&o);
#pragma unroll
      for (int i = 0; i < kVec; ++i) y[i] = from_float<T>(acc[i]);
      *reinterpret_cast<uint4*>(out + (long long)t * dim + col) = o;
    }
    __syncthreads();
  }
}

// drows[row of (t, s)] = weights[t, s] * dout[t];  dweights[t, s] = <rows[row], dout[t]>; a pair without a row: 0.
// A warp per pair, the pairs of a token side by side (its dout row stays in the cache); rows without a pair are zeroed by
// the warps as they pass.  Either result may be null.
template <typename T>
__global__ void __launch_bounds__(256)
combine_backward_kernel(const T* __restrict__ dout, const T* __restrict__ rows, const float* __restrict__ weights,
                        T* __restrict__ drows, float* __restrict__ dweights, const Routed p, int dim) {
  constexpr int kVec = 16 / sizeof(T);           // elements of a 16-byte piece
  const int lane = threadIdx.x & 31;
  const long long warp = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), warps = (long long)gridDim.x * 8;
  const long long pairs = (long long)p.tokens * p.topk;
  for (long long i = warp; i < pairs; i += warps) {
    const int t = int(i / p.topk), r = p.row_of(t, int(i - (long long)t * p.topk));
    float dot = 0.f;
    if (r >= 0) {
      const float w = __ldg(weights + i);
      const T* g = dout + (long long)t * dim;
      const T* z = rows + (long long)r * dim;
      T* d = drows + (long long)r * dim;
      for (int c = lane * kVec; c < dim; c += 128 * kVec) {
        uint4 a[4], b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + 32 * kVec * j < dim) {
            a[j] = __ldg(reinterpret_cast<const uint4*>(g + c + 32 * kVec * j));
            if (dweights) b[j] = __ldg(reinterpret_cast<const uint4*>(z + c + 32 * kVec * j));
          }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + 32 * kVec * j < dim) {
            T* x = reinterpret_cast<T*>(&a[j]);
            const T* y = reinterpret_cast<const T*>(&b[j]);
#pragma unroll
            for (int q = 0; q < kVec; ++q) {
              const float f = float(x[q]);
              if (dweights) dot = fmaf(f, float(y[q]), dot);
              x[q] = from_float<T>(f * w);
            }
            if (drows) *reinterpret_cast<uint4*>(d + c + 32 * kVec * j) = a[j];
          }
      }
    }
    if (dweights) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
      if (lane == 0) dweights[i] = dot;
    }
  }
  if (drows == nullptr) return;
  for (long long r0 = warp * 32; r0 < p.rows; r0 += warps * 32) {
    const bool mine = r0 + lane < p.rows && p.pair_of(int(r0) + lane) < 0;
    uint32_t bare = __ballot_sync(0xffffffffu, mine);
    const float zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (; bare; bare &= bare - 1) {
      T* d = drows + (r0 + __ffs(bare) - 1) * dim;
      for (int c = lane * 8; c < dim; c += 256) Vec8<T>::store(d + c, zero);
    }
  }
}

// ---------------------------------------------------------------------------- gate
// One warp per token; expert e lives in lane e % 32, register e / 32; lane j holds pick j.
//   renormalised: w = softmax over the picks      dlogit_i = w_i (g_i - sum_j w_j g_j) on the picks, 0 elsewhere
//   else:         w = softmax over all, p         dlogit_e = [picked] p_e g_e - p_e sum_j p_j g_j
template <int VPL, typename T>
__global__ void __launch_bounds__(128)
topk_gating_backward_kernel(const T* __restrict__ logits, const float* __restrict__ weights, const int* __restrict__ ids,
                            const float* __restrict__ dweights, T* __restrict__ dlogits, int num_tokens, int num_experts,
                            int topk, int renormalize) {
  const int lane = threadIdx.x & 31;
  const int token = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (token >= num_tokens) return;
  const long long o = (long long)token * topk + lane;
  const bool pick = lane < topk;
  const float w = pick ? __ldg(weights + o) : 0.f, g = pick ? __ldg(dweights + o) : 0.f;
  const int id = pick ? __ldg(ids + o) : -1;
  float inner = pick ? w * g : 0.f;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) inner += __shfl_xor_sync(0xffffffffu, inner, off);
  float v[VPL];
  if (renormalize) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) v[i] = 0.f;
  } else {
    const T* row = logits + (long long)token * num_experts;
    float vmax = -CUDART_INF_F, sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      v[i] = i * 32 + lane < num_experts ? float(row[i * 32 + lane]) : -CUDART_INF_F;
      vmax = fmaxf(vmax, v[i]);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, off));
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      v[i] = i * 32 + lane < num_experts ? expf(v[i] - vmax) : 0.f;
      sum += v[i];
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
#pragma unroll
    for (int i = 0; i < VPL; ++i) v[i] = -(v[i] / sum) * inner;
  }
  const float d = renormalize ? w * (g - inner) : w * g;
  for (int j = 0; j < topk; ++j) {
    const float dj = __shfl_sync(0xffffffffu, d, j);
    const int at = __shfl_sync(0xffffffffu, id, j) - lane;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (at == i * 32) v[i] += dj;
  }
  T* out = dlogits + (long long)token * num_experts;
#pragma unroll
  for (int i = 0; i < VPL; ++i)
    if (i * 32 + lane < num_experts) out[i * 32 + lane] = from_float<T>(v[i]);
}

template <typename T>
static int launch_gating_backward(const void* logits, const float* w, const int* ids, const float* dw, void* dlogits, int tokens,
                                  int experts, int topk, int renorm, cudaStream_t stream) {
  const int vpl = ceil_div(experts, 32);
  const dim3 grid(ceil_div(tokens, 4)), block(128);
  const T* l = static_cast<const T*>(logits);
  T* d = static_cast<T*>(dlogits);
#define FLYMOE_GATE_CASE(V) \
  topk_gating_backward_kernel<V, T><<<grid, block, 0, stream>>>(l, w, ids, dw, d, tokens, experts, topk, renorm)
  if (vpl <= 1) FLYMOE_GATE_CASE(1);
  else if (vpl <= 2) FLYMOE_GATE_CASE(2);
  else if (vpl <= 4) FLYMOE_GATE_CASE(4);
  else if (vpl <= 8) FLYMOE_GATE_CASE(8);
  else if (vpl <= 16) FLYMOE_GATE_CASE(16);
  else FLYMOE_GATE_CASE(32);
#undef FLYMOE_GATE_CASE
  FLYMOE_CUDA_CHECK(cudaGetLastError());
  return FLYMOE_OK;
}

static int check_routed(const char* null_msg, const char* size_msg, const void* sorted_ids, const void* num_valid_ids,
                        const void* row_index, int tokens, int topk, int rows) {
  FLYMOE_REQUIRE(tokens >= 0 && tokens < (1 << 24) && topk >= 1 && topk <= 255 && rows >= 0 && rows <= kMostRows, size_msg);
  FLYMOE_REQUIRE(num_valid_ids && (rows == 0 || sorted_ids) && (tokens == 0 || row_index), null_msg);
  return FLYMOE_OK;
}

}  // namespace flymoe

extern "C" int flymoe_route_tables(const int32_t* sorted_ids, const int32_t* sorted_expert_ids,
                                   const int32_t* num_valid_ids, int32_t* row_index, int32_t* offsets, int num_tokens,
                                   int topk, int experts, int max_rows, void* stream) {
  using namespace flymoe;
  FLYMOE_REQUIRE(experts >= 1 && experts <= kMaxRouteExperts, "route_tables: experts must be in [1, 1024]");
  const int rc = check_routed("route_tables: null pointer", "route_tables: bad sizes", sorted_ids, num_valid_ids, row_index,
                              num_tokens, topk, max_rows);
  if (rc != FLYMOE_OK) return rc;
  FLYMOE_REQUIRE(offsets && (max_rows == 0 || sorted_expert_ids), "route_tables: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t pairs = size_t(num_tokens) * topk;
  if (pairs > 0) FLYMOE_CUDA_CHECK(cudaMemsetAsync(row_index, 0xFF, pairs * sizeof(int32_t), s));
  const int blocks = std::min(ceil_div(std::max(max_rows, experts + 1), 256), sm_count() * 8);
  route_tables_kernel<<<blocks, 256, 0, s>>>(sorted_ids, sorted_expert_ids, num_valid_ids, row_index, offsets, num_tokens,
                                             topk, experts, max_rows);
  FLYMOE_CUDA_CHECK(cudaGetLastError());
  return FLYMOE_OK;
}

extern "C" int flymoe_permute_rows(const void* x, void* rows_out, const int32_t* sorted_ids, const int32_t* num_valid_ids,
                                   const int32_t* row_index, int num_tokens, int topk, int rows, int row_bytes, void* stream) {
  using namespace flymoe;
  const int rc = check_routed("permute_rows: null pointer", "permute_rows: bad sizes", sorted_ids, num_valid_ids, row_index,
                              num_tokens, topk, rows);
  if (rc != FLYMOE_OK) return rc;
  FLYMOE_REQUIRE(row_bytes > 0 && row_bytes % 16 == 0, "permute_rows: row_bytes must be a multiple of 16");
  if (rows == 0) return FLYMOE_OK;
  FLYMOE_REQUIRE((x || num_tokens == 0) && rows_out, "permute_rows: null pointer");
  FLYMOE_REQUIRE(aligned16(x) && aligned16(rows_out), "permute_rows: pointers must be 16-byte aligned");
  const Routed p = {sorted_ids, num_valid_ids, row_index, num_tokens, topk, rows};
  permute_rows_kernel<<<std::min(ceil_div(rows, 8), sm_count() * 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint4*>(x), static_cast<uint4*>(rows_out), p, row_bytes / 16);
  FLYMOE_CUDA_CHECK(cudaGetLastError());
  return FLYMOE_OK;
}

extern "C" int flymoe_combine_rows(const void* rows_in, const float* weights, void* out, const int32_t* sorted_ids,
                                   const int32_t* num_valid_ids, const int32_t* row_index, int num_tokens, int topk, int rows,
                                   int dim, int dtype, void* stream) {
  using namespace flymoe;
  const int rc = check_routed("combine_rows: null pointer", "combine_rows: bad sizes", sorted_ids, num_valid_ids, row_index,
                              num_tokens, topk, rows);
  if (rc != FLYMOE_OK) return rc;
  FLYMOE_REQUIRE(dim >= 8 && dim % 8 == 0, "combine_rows: dim must be a positive multiple of 8");
  if (num_tokens == 0) return FLYMOE_OK;
  FLYMOE_REQUIRE((rows_in || rows == 0) && out, "combine_rows: null pointer");
  FLYMOE_REQUIRE(aligned16(rows_in) && aligned16(out), "combine_rows: pointers must be 16-byte aligned");
  const Routed p = {sorted_ids, num_valid_ids, row_index, num_tokens, topk, rows};
  const int grid = num_tokens;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == FLYMOE_BF16)
    combine_rows_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(rows_in), weights,
                                                            static_cast<__nv_bfloat16*>(out), p, dim);
  else if (dtype == FLYMOE_F16)
    combine_rows_kernel<__half><<<grid, 256, 0, s>>>(static_cast<const __half*>(rows_in), weights, static_cast<__half*>(out), p, dim);
  else if (dtype == FLYMOE_F32)
    combine_rows_kernel<float><<<grid, 256, 0, s>>>(static_cast<const float*>(rows_in), weights, static_cast<float*>(out), p, dim);
  else
    FLYMOE_REQUIRE(false, "combine_rows: dtype must be F16, BF16 or F32");
  FLYMOE_CUDA_CHECK(cudaGetLastError());
  return FLYMOE_OK;
}

extern "C" int flymoe_combine_rows_backward(const void* dout, const void* rows_in, const float* weights, void* drows,
                                            float* dweights, const int32_t* sorted_ids, const int32_t* num_valid_ids,
                                            const int32_t* row_index, int num_tokens, int topk, int rows, int dim, int dtype,
                                            void* stream) {
  using namespace flymoe;
  const int rc = check_routed("combine_rows_backward: null pointer", "combine_rows_backward: bad sizes", sorted_ids,
                              num_valid_ids, row_index, num_tokens, topk, rows);
  if (rc != FLYMOE_OK) return rc;
  FLYMOE_REQUIRE(dim >= 8 && dim % 8 == 0, "combine_rows_backward: dim must be a positive multiple of 8");
  const long long pairs = (long long)num_tokens * topk;
  if ((pairs == 0 && rows == 0) || (!drows && !dweights)) return FLYMOE_OK;
  FLYMOE_REQUIRE(pairs == 0 || (dout && weights), "combine_rows_backward: null pointer");
  FLYMOE_REQUIRE(!dweights || rows == 0 || rows_in, "combine_rows_backward: null pointer");
  FLYMOE_REQUIRE(aligned16(dout) && aligned16(rows_in) && aligned16(drows), "combine_rows_backward: pointers must be 16-byte aligned");
  const Routed p = {sorted_ids, num_valid_ids, row_index, num_tokens, topk, rows};
  const long long warps = std::max(pairs, ((long long)rows + 31) / 32);
  const int blocks = int(std::min<long long>((warps + 7) / 8, (long long)sm_count() * 16));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define FLYMOE_COMBINE_CASE(T)                                                                                     \
  combine_backward_kernel<T><<<blocks, 256, 0, s>>>(static_cast<const T*>(dout), static_cast<const T*>(rows_in), weights, \
                                                    static_cast<T*>(drows), dweights, p, dim)
  if (dtype == FLYMOE_BF16) FLYMOE_COMBINE_CASE(__nv_bfloat16);
  else if (dtype == FLYMOE_F16) FLYMOE_COMBINE_CASE(__half);
  else if (dtype == FLYMOE_F32) FLYMOE_COMBINE_CASE(float);
  else FLYMOE_REQUIRE(false, "combine_rows_backward: dtype must be F16, BF16 or F32");
#undef FLYMOE_COMBINE_CASE
  FLYMOE_CUDA_CHECK(cudaGetLastError());
  return FLYMOE_OK;
}

extern "C" int flymoe_topk_gating_softmax_backward(const void* gating, int gating_dtype, const float* topk_weights,
                                                   const int32_t* topk_indices, const float* dtopk_weights, void* dgating,
                                                   int num_tokens, int num_experts, int topk, int renormalize, void* stream) {
  using namespace flymoe;
  FLYMOE_REQUIRE(num_tokens >= 0, "gating_backward: num_tokens < 0");
  FLYMOE_REQUIRE(num_experts >= 1 && num_experts <= 1024, "gating_backward: num_experts must be in [1, 1024]");
  FLYMOE_REQUIRE(topk >= 1 && topk <= 32 && topk <= num_experts, "gating_backward: topk must be in [1, min(32, E)]");
  if (num_tokens == 0) return FLYMOE_OK;
  FLYMOE_REQUIRE((gating || renormalize) && topk_weights && topk_indices && dtopk_weights && dgating,
                 "gating_backward: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (gating_dtype) {
    case FLYMOE_F32:
      return launch_gating_backward<float>(gating, topk_weights, topk_indices, dtopk_weights, dgating, num_tokens, num_experts,
                                           topk, renormalize, s);
    case FLYMOE_F16:
      return launch_gating_backward<__half>(gating, topk_weights, topk_indices, dtopk_weights, dgating, num_tokens,
                                            num_experts, topk, renormalize, s);
    case FLYMOE_BF16:
      return launch_gating_backward<__nv_bfloat16>(gating, topk_weights, topk_indices, dtopk_weights, dgating, num_tokens,
                                                   num_experts, topk, renormalize, s);
    default:
      set_last_error_msg("gating_backward: dtype must be F32, F16 or BF16");
      return FLYMOE_ERR_INVALID_ARGUMENT;
  }
}
