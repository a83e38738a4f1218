// Norms of rows: y = (x - mean) * rstd * weight + bias (layer norm) and y = x * rstd * weight (RMSNorm), with
// rstd = 1 / sqrt(mean((x - mean)^2) + eps), and their gradients:
//   g = dy * weight, u = (x - mean) * rstd
//   dx = rstd * (g - mean(g) - u * mean(g * u))        (no mean(g) without centring)
//   dweight = sum over rows of dy * u, dbias = sum over rows of dy
// Every sum, mean and statistic is FP32; x, dy, y and dx are BF16, FP16 or FP32, parameters that type or FP32, and each
// output is rounded once. Bound by memory: forward 2, gradient 3 row lengths of traffic per row.
#include <cuda_fp16.h>

#include "common.cuh"

namespace hmc {
namespace {

template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
  T v[N];
};

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, VEC>*>(p);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, VEC>& v) {
  *reinterpret_cast<Pack<T, VEC>*>(p) = v;
}

// Sums over the threads of a row: the warp's, then one slot per warp read by everybody in warp order, so that the result
// does not depend on timing. Two calls in a row use different slots: a slot is written again only behind the next
// call's barrier, which no thread reaches before it has read this one's.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* slots, int warps) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if (warps == 1) return;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) slots[(threadIdx.x >> 5) * N + i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.0f;
  for (int w = 0; w < warps; ++w) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += slots[w * N + i];
  }
}

constexpr int MAX_WARPS = 32;

// One row per blockDim.x threads, NV packs of VEC values per thread, the row in registers between its two passes: the
// variance is that of the differences from the mean, so a common offset costs no digits. blockDim.y rows per block, one
// per warp, where a row is short.
template <typename T, typename W, int VEC, int NV, bool CENTER>
__global__ void __launch_bounds__(1024) row_norm_kernel(const T* __restrict__ x, long long x_stride, long long rows, int hidden,
                                                        const W* __restrict__ weight, const W* __restrict__ bias, float eps,
                                                        T* __restrict__ y, float* __restrict__ mean_out,
                                                        float* __restrict__ rstd_out) {
  __shared__ float slots[2][MAX_WARPS];
  const long long row = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= rows) return;  // only where a row is one warp, which meets no barrier
  const int warps = blockDim.x >> 5;
  const int packs = hidden / VEC;
  const float scale = 1.0f / static_cast<float>(hidden);
  const T* src = x + row * x_stride;
  Pack<T, VEC> in[NV];
  float sum[1] = {0.0f};
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * blockDim.x + threadIdx.x;
    if (at < packs) in[j] = load_pack<T, VEC>(src + static_cast<long long>(at) * VEC);
  }
  float mean = 0.0f;
  if (CENTER) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * blockDim.x + threadIdx.x < packs) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum[0] += widen(in[j].v[e]);
      }
    row_sum(sum, slots[0], warps);
    mean = sum[0] * scale;
  }
  float square[1] = {0.0f};
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (j * blockDim.x + threadIdx.x < packs) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = widen(in[j].v[e]) - mean;
        square[0] += d * d;
      }
    }
  row_sum(square, slots[1], warps);
  const float rstd = rsqrtf(square[0] * scale + eps);
  T* dst = y + row * hidden;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * blockDim.x + threadIdx.x;
    if (at < packs) {
      Pack<T, VEC> out;
      Pack<W, VEC> w, b;
      if (weight != nullptr) w = load_pack<W, VEC>(weight + static_cast<long long>(at) * VEC);
      if (CENTER && bias != nullptr) b = load_pack<W, VEC>(bias + static_cast<long long>(at) * VEC);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float v = (widen(in[j].v[e]) - mean) * rstd;
        if (weight != nullptr) v *= widen(w.v[e]);
        if (CENTER && bias != nullptr) v += widen(b.v[e]);
        out.v[e] = narrow<T>(v);
      }
      store_pack<T, VEC>(dst + static_cast<long long>(at) * VEC, out);
    }
  }
  if (threadIdx.x == 0 && rstd_out != nullptr) {
    if (CENTER) mean_out[row] = mean;
    rstd_out[row] = rstd;
  }
}

// Rows too long for the registers of a block: the same three passes, each reading the row again (from L2).
template <typename T, typename W, bool CENTER>
__global__ void __launch_bounds__(1024) long_row_norm_kernel(const T* __restrict__ x, long long x_stride, long long rows,
                                                             int hidden, const W* __restrict__ weight,
                                                             const W* __restrict__ bias, float eps, T* __restrict__ y,
                                                             float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  __shared__ float slots[2][MAX_WARPS];
  const long long row = blockIdx.x;
  const int warps = blockDim.x >> 5;
  const float scale = 1.0f / static_cast<float>(hidden);
  const T* src = x + row * x_stride;
  float mean = 0.0f;
  if (CENTER) {
    float sum[1] = {0.0f};
    for (int c = threadIdx.x; c < hidden; c += blockDim.x) sum[0] += widen(src[c]);
    row_sum(sum, slots[0], warps);
    mean = sum[0] * scale;
  }
  float square[1] = {0.0f};
  for (int c = threadIdx.x; c < hidden; c += blockDim.x) {
    const float d = widen(src[c]) - mean;
    square[0] += d * d;
  }
  row_sum(square, slots[1], warps);
  const float rstd = rsqrtf(square[0] * scale + eps);
  for (int c = threadIdx.x; c < hidden; c += blockDim.x) {
    float v = (widen(src[c]) - mean) * rstd;
    if (weight != nullptr) v *= widen(weight[c]);
    if (CENTER && bias != nullptr) v += widen(bias[c]);
    y[row * hidden + c] = narrow<T>(v);
  }
  if (threadIdx.x == 0 && rstd_out != nullptr) {
    if (CENTER) mean_out[row] = mean;
    rstd_out[row] = rstd;
  }
}

// Gradient: a block walks the rows blockIdx.x, + gridDim.x, ...; its threads own columns, so that the parameters'
// gradients stay in registers over all its rows and x and dy are read once. `partial_*` are [gridDim.x, hidden] in FP32.
template <typename T, typename W, int VEC, int NV, bool CENTER>
__global__ void __launch_bounds__(512) row_norm_grad_kernel(const T* __restrict__ x, long long x_stride,
                                                            const T* __restrict__ grad, long long grad_stride, long long rows,
                                                            int hidden, const W* __restrict__ weight,
                                                            const float* __restrict__ mean_in,
                                                            const float* __restrict__ rstd_in, T* __restrict__ grad_x,
                                                            float* __restrict__ partial_weight,
                                                            float* __restrict__ partial_bias) {
  __shared__ float slots[2][2 * MAX_WARPS];
  const int warps = blockDim.x >> 5;
  const int packs = hidden / VEC;
  const float scale = 1.0f / static_cast<float>(hidden);
  Pack<W, VEC> w[NV];
  float sum_weight[NV][VEC], sum_bias[CENTER ? NV : 1][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * blockDim.x + threadIdx.x;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[j].v[e] = narrow<W>(1.0f);
      sum_weight[j][e] = 0.0f;
      if (CENTER) sum_bias[j][e] = 0.0f;
    }
    if (at < packs && weight != nullptr) w[j] = load_pack<W, VEC>(weight + static_cast<long long>(at) * VEC);
  }
  int turn = 0;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
    Pack<T, VEC> in[NV], dy[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = j * blockDim.x + threadIdx.x;
      if (at < packs) {
        in[j] = load_pack<T, VEC>(x + row * x_stride + static_cast<long long>(at) * VEC);
        dy[j] = load_pack<T, VEC>(grad + row * grad_stride + static_cast<long long>(at) * VEC);
      }
    }
    const float mean = CENTER ? mean_in[row] : 0.0f;
    const float rstd = rstd_in[row];
    float sums[2] = {0.0f, 0.0f};  // of g * u and of g
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * blockDim.x + threadIdx.x < packs) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float d = widen(dy[j].v[e]), u = (widen(in[j].v[e]) - mean) * rstd, g = d * widen(w[j].v[e]);
          sums[0] += g * u;
          sum_weight[j][e] += d * u;
          if (CENTER) {
            sums[1] += g;
            sum_bias[j][e] += d;
          }
        }
      }
    row_sum(sums, slots[turn], warps);
    const float along = sums[0] * scale, offset = sums[1] * scale;
    if (grad_x != nullptr) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int at = j * blockDim.x + threadIdx.x;
        if (at < packs) {
          Pack<T, VEC> out;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float u = (widen(in[j].v[e]) - mean) * rstd, g = widen(dy[j].v[e]) * widen(w[j].v[e]);
            float v = g - u * along;
            if (CENTER) v -= offset;
            out.v[e] = narrow<T>(v * rstd);
          }
          store_pack<T, VEC>(grad_x + row * hidden + static_cast<long long>(at) * VEC, out);
        }
      }
    }
  }
  if (partial_weight == nullptr) return;
  const long long base = static_cast<long long>(blockIdx.x) * hidden;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * blockDim.x + threadIdx.x;
    if (at < packs) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        partial_weight[base + static_cast<long long>(at) * VEC + e] = sum_weight[j][e];
        if (CENTER) partial_bias[base + static_cast<long long>(at) * VEC + e] = sum_bias[j][e];
      }
    }
  }
}

// Rows too long for a block's registers: dx by one block per row, the parameters' partial sums by columns.
template <typename T, typename W, bool CENTER>
__global__ void __launch_bounds__(1024) long_row_norm_grad_kernel(const T* __restrict__ x, long long x_stride,
                                                                  const T* __restrict__ grad, long long grad_stride,
                                                                  int hidden, const W* __restrict__ weight,
                                                                  const float* __restrict__ mean_in,
                                                                  const float* __restrict__ rstd_in, T* __restrict__ grad_x) {
  __shared__ float slots[2 * MAX_WARPS];
  const long long row = blockIdx.x;
  const float scale = 1.0f / static_cast<float>(hidden);
  const float mean = CENTER ? mean_in[row] : 0.0f;
  const float rstd = rstd_in[row];
  float sums[2] = {0.0f, 0.0f};
  for (int c = threadIdx.x; c < hidden; c += blockDim.x) {
    const float g = widen(grad[row * grad_stride + c]) * (weight != nullptr ? widen(weight[c]) : 1.0f);
    sums[0] += g * ((widen(x[row * x_stride + c]) - mean) * rstd);
    sums[1] += g;
  }
  row_sum(sums, slots, blockDim.x >> 5);
  const float along = sums[0] * scale, offset = sums[1] * scale;
  for (int c = threadIdx.x; c < hidden; c += blockDim.x) {
    const float g = widen(grad[row * grad_stride + c]) * (weight != nullptr ? widen(weight[c]) : 1.0f);
    float v = g - (widen(x[row * x_stride + c]) - mean) * rstd * along;
    if (CENTER) v -= offset;
    grad_x[row * hidden + c] = narrow<T>(v * rstd);
  }
}

template <typename T, bool CENTER>
__global__ void __launch_bounds__(256) column_grad_kernel(const T* __restrict__ x, long long x_stride,
                                                          const T* __restrict__ grad, long long grad_stride, long long rows,
                                                          int hidden, const float* __restrict__ mean_in,
                                                          const float* __restrict__ rstd_in,
                                                          float* __restrict__ partial_weight,
                                                          float* __restrict__ partial_bias) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= hidden) return;
  float w = 0.0f, b = 0.0f;
  for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
    const float d = widen(grad[row * grad_stride + c]);
    w += d * ((widen(x[row * x_stride + c]) - (CENTER ? mean_in[row] : 0.0f)) * rstd_in[row]);
    b += d;
  }
  partial_weight[static_cast<long long>(blockIdx.y) * hidden + c] = w;
  if (CENTER) partial_bias[static_cast<long long>(blockIdx.y) * hidden + c] = b;
}

// Parameters' gradients: the partial sums of a column in the order of the blocks that made them.
constexpr int FINISH_SLICES = 8;
template <typename W>
__global__ void __launch_bounds__(32 * FINISH_SLICES) param_grad_kernel(const float* __restrict__ partial_weight,
                                                                        const float* __restrict__ partial_bias, int parts,
                                                                        int hidden, W* __restrict__ grad_weight,
                                                                        W* __restrict__ grad_bias) {
  __shared__ float sums[2][FINISH_SLICES][32];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float w = 0.0f, b = 0.0f;
  if (c < hidden) {
    for (int i = threadIdx.y; i < parts; i += FINISH_SLICES) {
      if (grad_weight != nullptr) w += partial_weight[static_cast<long long>(i) * hidden + c];
      if (grad_bias != nullptr) b += partial_bias[static_cast<long long>(i) * hidden + c];
    }
  }
  sums[0][threadIdx.y][threadIdx.x] = w;
  sums[1][threadIdx.y][threadIdx.x] = b;
  __syncthreads();
  if (threadIdx.y > 1 || c >= hidden) return;
  W* out = threadIdx.y == 0 ? grad_weight : grad_bias;
  if (out == nullptr) return;
  float v = 0.0f;
#pragma unroll
  for (int s = 0; s < FINISH_SLICES; ++s) v += sums[threadIdx.y][s][threadIdx.x];
  out[c] = narrow<W>(v);
}

bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int round_up(int v, int to) { return (v + to - 1) / to * to; }

constexpr int FORWARD_PACKS = 4;  // packs of 16 bytes per thread and row
constexpr int GRAD_PACKS = 2;
constexpr int SINGLES = 8;        // values per thread where rows start on no 16-byte boundary
constexpr int GRAD_THREADS = 512;

struct NormCall {
  const void *x, *grad, *weight, *bias;
  long long x_stride, grad_stride, rows;
  int hidden;
  float eps;
  const float *mean_in, *rstd_in;
  void *y, *grad_weight, *grad_bias;  // y: dx in the gradient
  float *mean, *rstd, *partial_weight, *partial_bias;
  int parts;
  cudaStream_t stream;
};

// Blocks of the gradient kernel: two per SM, each with partial sums of its own.
long long grad_parts(long long rows) {
  const long long most = 2ll * sm_count();
  return rows < most ? rows : most;
}

template <typename T, typename W, int VEC, int NV, bool CENTER>
int launch_forward(const NormCall& c) {
  const int need = (c.hidden / VEC + NV - 1) / NV;
  const int threads = round_up(need, 32);
  const int rows_per_block = threads == 32 ? 4 : 1;
  const long long blocks = (c.rows + rows_per_block - 1) / rows_per_block;
  row_norm_kernel<T, W, VEC, NV, CENTER><<<static_cast<unsigned>(blocks), dim3(threads, rows_per_block), 0, c.stream>>>(
      static_cast<const T*>(c.x), c.x_stride, c.rows, c.hidden, static_cast<const W*>(c.weight), static_cast<const W*>(c.bias),
      c.eps, static_cast<T*>(c.y), c.mean, c.rstd);
  HMC_LAUNCH_OK();
  return 0;
}

template <typename T, typename W, bool CENTER>
int forward(const NormCall& c) {
  constexpr int VEC = 16 / sizeof(T);
  const bool wide = c.hidden % VEC == 0 && c.x_stride % VEC == 0 && aligned_to(c.x, 16) && aligned_to(c.y, 16) &&
                    aligned_to(c.weight, 16) && aligned_to(c.bias, 16);
  if (wide && c.hidden <= 1024 * VEC * FORWARD_PACKS) return launch_forward<T, W, VEC, FORWARD_PACKS, CENTER>(c);
  if (c.hidden <= 1024 * SINGLES) return launch_forward<T, W, 1, SINGLES, CENTER>(c);
  long_row_norm_kernel<T, W, CENTER><<<static_cast<unsigned>(c.rows), 1024, 0, c.stream>>>(
      static_cast<const T*>(c.x), c.x_stride, c.rows, c.hidden, static_cast<const W*>(c.weight), static_cast<const W*>(c.bias),
      c.eps, static_cast<T*>(c.y), c.mean, c.rstd);
  HMC_LAUNCH_OK();
  return 0;
}

template <typename T, typename W, int VEC, int NV, bool CENTER>
int launch_grad(const NormCall& c) {
  const int threads = round_up((c.hidden / VEC + NV - 1) / NV, 32);
  row_norm_grad_kernel<T, W, VEC, NV, CENTER><<<static_cast<unsigned>(c.parts), threads, 0, c.stream>>>(
      static_cast<const T*>(c.x), c.x_stride, static_cast<const T*>(c.grad), c.grad_stride, c.rows, c.hidden,
      static_cast<const W*>(c.weight), c.mean_in, c.rstd_in, static_cast<T*>(c.y), c.partial_weight, c.partial_bias);
  HMC_LAUNCH_OK();
  return 0;
}

template <typename T, typename W, bool CENTER>
int gradient(const NormCall& c) {
  constexpr int VEC = 16 / sizeof(T);
  const bool wide = c.hidden % VEC == 0 && c.x_stride % VEC == 0 && c.grad_stride % VEC == 0 && aligned_to(c.x, 16) &&
                    aligned_to(c.grad, 16) && aligned_to(c.y, 16) && aligned_to(c.weight, 16);
  if (wide && c.hidden <= GRAD_THREADS * VEC * GRAD_PACKS) {
    if (int rc = launch_grad<T, W, VEC, GRAD_PACKS, CENTER>(c)) return rc;
  } else if (c.hidden <= GRAD_THREADS * SINGLES) {
    if (int rc = launch_grad<T, W, 1, SINGLES, CENTER>(c)) return rc;
  } else {
    if (c.y != nullptr) {
      long_row_norm_grad_kernel<T, W, CENTER><<<static_cast<unsigned>(c.rows), 1024, 0, c.stream>>>(
          static_cast<const T*>(c.x), c.x_stride, static_cast<const T*>(c.grad), c.grad_stride, c.hidden,
          static_cast<const W*>(c.weight), c.mean_in, c.rstd_in, static_cast<T*>(c.y));
      HMC_LAUNCH_OK();
    }
    if (c.partial_weight != nullptr) {
      const dim3 grid((c.hidden + 255) / 256, c.parts);
      column_grad_kernel<T, CENTER><<<grid, 256, 0, c.stream>>>(
          static_cast<const T*>(c.x), c.x_stride, static_cast<const T*>(c.grad), c.grad_stride, c.rows, c.hidden, c.mean_in,
          c.rstd_in, c.partial_weight, c.partial_bias);
      HMC_LAUNCH_OK();
    }
  }
  if (c.partial_weight != nullptr) {
    param_grad_kernel<W><<<(c.hidden + 31) / 32, dim3(32, FINISH_SLICES), 0, c.stream>>>(
        c.partial_weight, c.partial_bias, c.parts, c.hidden, static_cast<W*>(c.grad_weight), static_cast<W*>(c.grad_bias));
    HMC_LAUNCH_OK();
  }
  return 0;
}

template <typename T, typename W>
int run(const NormCall& c, bool center, bool backward) {
  if (backward) return center ? gradient<T, W, true>(c) : gradient<T, W, false>(c);
  return center ? forward<T, W, true>(c) : forward<T, W, false>(c);
}

int run(const NormCall& c, int dtype, int affine_dtype, bool center, bool backward) {
  if (dtype == HMC_DTYPE_F32) return run<float, float>(c, center, backward);
  if (dtype == HMC_DTYPE_BF16)
    return affine_dtype == HMC_DTYPE_F32 ? run<__nv_bfloat16, float>(c, center, backward)
                                         : run<__nv_bfloat16, __nv_bfloat16>(c, center, backward);
  return affine_dtype == HMC_DTYPE_F32 ? run<__half, float>(c, center, backward) : run<__half, __half>(c, center, backward);
}

int check(const char* name, int64_t rows, int64_t hidden, int64_t stride, int dtype, int affine_dtype) {
  HMC_REQUIRE(rows >= 0 && rows < (1ll << 31) && hidden > 0 && hidden <= HMC_NORM_MAX_HIDDEN, HMC_ERR_INVALID,
              "%s: rows (%lld) must be in [0, 2^31) and hidden (%lld) in [1, %d]", name, (long long)rows, (long long)hidden,
              HMC_NORM_MAX_HIDDEN);
  HMC_REQUIRE(stride >= 0, HMC_ERR_INVALID, "%s: row strides must not be negative", name);
  HMC_REQUIRE(dtype >= HMC_DTYPE_BF16 && dtype <= HMC_DTYPE_F32, HMC_ERR_INVALID, "%s: unknown dtype %d", name, dtype);
  HMC_REQUIRE(affine_dtype == dtype || affine_dtype == HMC_DTYPE_F32, HMC_ERR_INVALID,
              "%s: parameters must have the rows' dtype or FP32", name);
  return 0;
}

}  // namespace
}  // namespace hmc

extern "C" int hmc_row_norm(const void* x, int64_t x_stride, int64_t rows, int64_t hidden, int dtype, const void* weight,
                            const void* bias, int affine_dtype, int center, float eps, void* y, float* mean, float* rstd,
                            void* stream) {
  using namespace hmc;
  if (int rc = check("hmc_row_norm", rows, hidden, x_stride, dtype, affine_dtype)) return rc;
  if (rows == 0) return 0;
  HMC_REQUIRE(x != nullptr && y != nullptr, HMC_ERR_INVALID, "hmc_row_norm: null tensor pointer");
  HMC_REQUIRE(eps >= 0.0f, HMC_ERR_INVALID, "hmc_row_norm: eps must not be negative");
  HMC_REQUIRE(center || (bias == nullptr && mean == nullptr), HMC_ERR_INVALID,
              "hmc_row_norm: a norm without centring has neither bias nor mean");
  HMC_REQUIRE(!center || (mean == nullptr) == (rstd == nullptr), HMC_ERR_INVALID,
              "hmc_row_norm: mean and rstd are asked for together or not at all");
  NormCall c{};
  c.x = x, c.x_stride = x_stride, c.rows = rows, c.hidden = static_cast<int>(hidden);
  c.weight = weight, c.bias = bias, c.eps = eps, c.y = y, c.mean = mean, c.rstd = rstd;
  c.stream = static_cast<cudaStream_t>(stream);
  return run(c, dtype, affine_dtype, center != 0, false);
}

extern "C" int64_t hmc_row_norm_grad_workspace_bytes(int64_t rows, int64_t hidden) {
  if (rows <= 0 || hidden <= 0) return 0;
  return 2 * hmc::grad_parts(rows) * hidden * static_cast<int64_t>(sizeof(float));
}

extern "C" int hmc_row_norm_grad(const void* x, int64_t x_stride, const void* grad, int64_t grad_stride, int64_t rows,
                                 int64_t hidden, int dtype, const void* weight, int affine_dtype, int center, const float* mean,
                                 const float* rstd, void* grad_x, void* grad_weight, void* grad_bias, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  using namespace hmc;
  if (int rc = check("hmc_row_norm_grad", rows, hidden, x_stride < grad_stride ? x_stride : grad_stride, dtype, affine_dtype))
    return rc;
  HMC_REQUIRE(center || grad_bias == nullptr, HMC_ERR_INVALID, "hmc_row_norm_grad: a norm without centring has no bias");
  const bool params = grad_weight != nullptr || grad_bias != nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    const size_t bytes = hidden * (affine_dtype == HMC_DTYPE_F32 ? 4 : 2);
    if (grad_weight != nullptr) HMC_CUDA_OK(cudaMemsetAsync(grad_weight, 0, bytes, s));
    if (grad_bias != nullptr) HMC_CUDA_OK(cudaMemsetAsync(grad_bias, 0, bytes, s));
    return 0;
  }
  HMC_REQUIRE(x != nullptr && grad != nullptr && rstd != nullptr && (mean != nullptr || !center), HMC_ERR_INVALID,
              "hmc_row_norm_grad: null tensor pointer");
  HMC_REQUIRE(!params || (workspace != nullptr && aligned16(workspace) &&
                          workspace_bytes >= hmc_row_norm_grad_workspace_bytes(rows, hidden)),
              HMC_ERR_INVALID, "hmc_row_norm_grad: the workspace must hold %lld bytes on a 16-byte boundary",
              (long long)hmc_row_norm_grad_workspace_bytes(rows, hidden));
  if (grad_x == nullptr && !params) return 0;
  NormCall c{};
  c.x = x, c.x_stride = x_stride, c.grad = grad, c.grad_stride = grad_stride, c.rows = rows;
  c.hidden = static_cast<int>(hidden), c.weight = weight, c.mean_in = mean, c.rstd_in = rstd, c.y = grad_x;
  c.grad_weight = grad_weight, c.grad_bias = grad_bias, c.parts = static_cast<int>(grad_parts(rows)), c.stream = s;
  if (params) {
    c.partial_weight = static_cast<float*>(workspace);
    c.partial_bias = c.partial_weight + static_cast<long long>(c.parts) * hidden;
  }
  return run(c, dtype, affine_dtype, center != 0, true);
}
