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

// Short rows of any alignment, forward: a warp per row, NV packs of VEC values per lane in registers between the passes. The
// variance is that of the differences from the mean, here as below, so that a common offset costs no digits. (16384 rows of
// 300 BF16: 7.9 us.)
constexpr int SHORT_ROWS = 4;  // per block

template <typename T, typename W, int VEC, int NV, bool CENTER>
__global__ void __launch_bounds__(32 * SHORT_ROWS)
short_norm_kernel(const T* __restrict__ x, long long x_stride, long long rows, int hidden, const W* __restrict__ weight,
                  const W* __restrict__ bias, float eps, T* __restrict__ y, float* __restrict__ mean_out,
                  float* __restrict__ rstd_out) {
  chain_wait();
  chain_next();
  const int lane = threadIdx.x & 31, packs = hidden / VEC;
  const long long row = static_cast<long long>(blockIdx.x) * SHORT_ROWS + (threadIdx.x >> 5);
  if (row >= rows) return;
  const float scale = 1.0f / static_cast<float>(hidden);
  const T* src = x + row * x_stride;
  float v[NV][VEC];
  float mean = 0.0f, square = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * 32 + lane;
    Pack<T, VEC> in;
    if (at < packs) in = load_pack<T, VEC>(src + at * VEC);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      v[j][e] = at < packs ? widen(in.v[e]) : 0.0f;
      mean += v[j][e];
    }
  }
  mean = CENTER ? warp_sum(mean) * scale : 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (CENTER) v[j][e] = j * 32 + lane < packs ? v[j][e] - mean : 0.0f;
      square += v[j][e] * v[j][e];
    }
  const float rstd = rsqrtf(warp_sum(square) * scale + eps);
  T* dst = y + row * hidden;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * 32 + lane;
    if (at >= packs) continue;
    Pack<T, VEC> out;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float u = v[j][e] * rstd;
      if (weight != nullptr) u *= widen(weight[at * VEC + e]);
      if (CENTER && bias != nullptr) u += widen(bias[at * VEC + e]);
      out.v[e] = narrow<T>(u);
    }
    store_pack<T, VEC>(dst + at * VEC, out);
  }
  if (lane == 0 && rstd_out != nullptr) {
    if (CENTER) mean_out[row] = mean;
    rstd_out[row] = rstd;
  }
}

// Rows too long for the registers of a block, or longer than SHORT rows in a tensor that starts on no 16-byte boundary: the same
// three passes, each reading the row again (from L2).
template <typename T, typename W, bool CENTER>
__global__ void __launch_bounds__(1024) long_row_norm_kernel(const T* __restrict__ x, long long x_stride, long long rows,
                                                             int hidden, const W* __restrict__ weight,
                                                             const W* __restrict__ bias, float eps, T* __restrict__ y,
                                                             float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  chain_wait();
  chain_next();
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

// ------------------------------------------------------------------------------------------- many rows
// 16 bytes of T as FP32 pairs: the arithmetic of the kernels below takes two values per instruction, because counted in
// single ones it is longer than the memory's time (16384 rows of 7168 BF16, 72 us of traffic: 34 instructions per value and
// 123 us in single values, 10 and 76 us now).
template <typename T>
struct Quad;
template <>
struct Quad<float> {
  static constexpr int PAIRS = 2;
  static __device__ __forceinline__ void widen(const uint4& q, float2* v) {
    v[0] = make_float2(__uint_as_float(q.x), __uint_as_float(q.y));
    v[1] = make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
  }
  static __device__ __forceinline__ uint4 narrow(const float2* v) {
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
  }
};
template <>
struct Quad<__nv_bfloat16> {
  static constexpr int PAIRS = 4;
  static __device__ __forceinline__ float2 pair(uint32_t w) {  // a BF16 is the upper half of its FP32
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ void widen(const uint4& q, float2* v) {
    v[0] = pair(q.x), v[1] = pair(q.y), v[2] = pair(q.z), v[3] = pair(q.w);
  }
  static __device__ __forceinline__ uint4 narrow(const float2* v) {
    return make_uint4(pack_bf16x2(v[0].x, v[0].y), pack_bf16x2(v[1].x, v[1].y), pack_bf16x2(v[2].x, v[2].y),
                      pack_bf16x2(v[3].x, v[3].y));
  }
};
template <>
struct Quad<__half> {
  static constexpr int PAIRS = 4;
  static __device__ __forceinline__ float2 pair(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
  static __device__ __forceinline__ uint32_t word(float2 v) {
    const __half2 h = __floats2half2_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ void widen(const uint4& q, float2* v) {
    v[0] = pair(q.x), v[1] = pair(q.y), v[2] = pair(q.z), v[3] = pair(q.w);
  }
  static __device__ __forceinline__ uint4 narrow(const float2* v) {
    return make_uint4(word(v[0]), word(v[1]), word(v[2]), word(v[3]));
  }
};
// 2 * PAIRS parameters from p: one or two loads
template <typename W, int PAIRS>
__device__ __forceinline__ void widen_params(const W* p, float2* v) {
#pragma unroll
  for (int i = 0; i < PAIRS / Quad<W>::PAIRS; ++i)
    Quad<W>::widen(ld_16(p + i * 2 * Quad<W>::PAIRS), v + i * Quad<W>::PAIRS);
}

constexpr int STREAM_THREADS = 512;
constexpr int STREAM_WARPS = STREAM_THREADS / 32;

// Sums over a block of at most STREAM_WARPS warps, in an order of their own: the warp's by halving, one slot per warp (the unused
// ones are zero), and 16 lanes each over the slots. Two calls in a row use different slots, as in row_sum.
__device__ __forceinline__ float over_16_lanes(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float block_sum(float v, float* slots) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  return over_16_lanes(slots[threadIdx.x & 15]);
}
// Of two values at once: the lower 16 lanes take the first, the upper ones the second.
__device__ __forceinline__ float2 block_sum(float2 v, float* slots) {
  const bool upper = (threadIdx.x & 16) != 0;
  float mine = (upper ? v.y : v.x) + __shfl_xor_sync(0xffffffffu, upper ? v.x : v.y, 16);
  mine = over_16_lanes(mine);
  if ((threadIdx.x & 15) == 0) slots[(threadIdx.x & 16) + (threadIdx.x >> 5)] = mine;
  __syncthreads();
  mine = over_16_lanes(slots[threadIdx.x & 31]);
  return make_float2(__shfl_sync(0xffffffffu, mine, 0), __shfl_sync(0xffffffffu, mine, 16));
}

// Of the pairs (or first values) of ROWS rows behind one barrier.
template <int ROWS, bool BOTH>
__device__ __forceinline__ void block_sums(float2 (&v)[ROWS], float* slots) {
  const bool upper = (threadIdx.x & 16) != 0;
  float mine[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (BOTH) {
      mine[r] = over_16_lanes((upper ? v[r].y : v[r].x) + __shfl_xor_sync(0xffffffffu, upper ? v[r].x : v[r].y, 16));
      if ((threadIdx.x & 15) == 0) slots[r * 2 * STREAM_WARPS + (threadIdx.x & 16) + (threadIdx.x >> 5)] = mine[r];
    } else {
      mine[r] = warp_sum(v[r].x);
      if ((threadIdx.x & 31) == 0) slots[r * STREAM_WARPS + (threadIdx.x >> 5)] = mine[r];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (BOTH) {
      mine[r] = over_16_lanes(slots[r * 2 * STREAM_WARPS + (threadIdx.x & 31)]);
      v[r] = make_float2(__shfl_sync(0xffffffffu, mine[r], 0), __shfl_sync(0xffffffffu, mine[r], 16));
    } else {
      v[r].x = over_16_lanes(slots[r * STREAM_WARPS + (threadIdx.x & 15)]);
    }
  }
}

// A block walks the rows blockIdx.x, + gridDim.x, ... and copies the next ones asynchronously while it works on one: a ring
// of rows in shared memory in which a thread writes and reads its own packs only, so that the copies need no barrier.
// What is left per row is the reduction's, at which the blocks of an SM take turns: as many as their registers allow, with four
// rows in each ring. Bound by memory: RMSNorm of 8192 x 4096 BF16 20.4 us (134 MB, the copy rate), layer norm of 16384 x 7168
// 76 us (6.2 TB/s). One row alone takes 2.3 to 2.9 us; a block per row without a ring took 2.5 to 4.3.
// Two rows per turn, as below, take 13.1 us instead of 14.6 for 16384 x 1024 (BF16, layer norm), but 44 instead of 39 for 3584
// columns and 2.2 instead of 1.9 for one row.
constexpr int FORWARD_STAGES = 4;
constexpr int GRAD_STAGES = 3;

template <typename T, typename W, int NV, bool CENTER>
__global__ void __launch_bounds__(STREAM_THREADS)
stream_norm_kernel(const T* __restrict__ x, long long x_stride, long long rows, int hidden, const W* __restrict__ weight,
                   const W* __restrict__ bias, float eps, T* __restrict__ y, float* __restrict__ mean_out,
                   float* __restrict__ rstd_out) {
  chain_wait();
  chain_next();
  extern __shared__ uint4 ring_raw[];
  constexpr int stages = FORWARD_STAGES;
  __shared__ __align__(16) float slots[2][STREAM_WARPS];
  constexpr int PAIRS = Quad<T>::PAIRS, VEC = 2 * PAIRS;
  const int threads = blockDim.x, width = NV * threads;  // packs of a row in the ring
  const int packs = hidden / VEC;
  const float scale = 1.0f / static_cast<float>(hidden);
  uint4* ring = ring_raw + threadIdx.x;
  if (threadIdx.x < STREAM_WARPS) slots[0][threadIdx.x] = slots[1][threadIdx.x] = 0.0f;
  bool here[NV];
  float2 w[NV][PAIRS], b[CENTER ? NV : 1][PAIRS];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * threads + threadIdx.x;
    here[j] = at < packs;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      w[j][i] = both(1.0f);
      if (CENTER) b[j][i] = both(0.0f);
    }
    if (here[j] && weight != nullptr) widen_params<W, PAIRS>(weight + at * VEC, w[j]);
    if (CENTER && here[j] && bias != nullptr) widen_params<W, PAIRS>(bias + at * VEC, b[j]);
  }
  // rows are counted down in 32 bits and pointers moved on: 64-bit products per row cost more than the row's arithmetic
  const int step = gridDim.x;
  const T* src = x + blockIdx.x * x_stride + threadIdx.x * VEC;
  T* dst = y + static_cast<long long>(blockIdx.x) * hidden + threadIdx.x * VEC;
  const long long src_step = step * x_stride, dst_step = static_cast<long long>(step) * hidden;
  int ahead = blockIdx.x;  // the next row to copy
  const int end = static_cast<int>(rows);
  auto fetch = [&](int stage) {
    if (ahead < end) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (here[j]) copy_async_16(ring + stage * width + j * threads, src + j * threads * VEC);
      src += src_step;
      ahead += step;
    }
    copy_async_commit();
  };
  for (int s = 0; s < stages - 1; ++s) fetch(s);
  __syncthreads();  // the slots are zero
  int stage = 0, last = stages - 1, turn = 0;
  for (int row = blockIdx.x; row < end; row += step, dst += dst_step) {
    fetch(last);
    copy_async_wait<stages - 1>();  // the copies of a row are one group
    float2 v[NV][PAIRS];
    float2 part[2] = {both(0.0f), both(0.0f)};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      uint4 q = make_uint4(0, 0, 0, 0);
      if (here[j]) q = ring[stage * width + j * threads];
      Quad<T>::widen(q, v[j]);
      if (CENTER) {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) part[i & 1] = add2(part[i & 1], v[j][i]);
      }
    }
    float mean = 0.0f;
    if (CENTER) {
      const float2 all = add2(part[0], part[1]);
      mean = block_sum(all.x + all.y, slots[turn]) * scale;
      turn ^= 1;
      part[0] = part[1] = both(0.0f);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (here[j]) {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          if (CENTER) v[j][i] = add2(v[j][i], both(-mean));
          part[i & 1] = madd2(v[j][i], v[j][i], part[i & 1]);
        }
      }
    const float2 all = add2(part[0], part[1]);
    const float rstd = rsqrtf(block_sum(all.x + all.y, slots[turn]) * scale + eps);
    turn ^= 1;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (here[j]) {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          v[j][i] = times2(v[j][i], both(rstd));
          v[j][i] = CENTER ? madd2(v[j][i], w[j][i], b[j][i]) : times2(v[j][i], w[j][i]);
        }
        st_16(dst + j * threads * VEC, Quad<T>::narrow(v[j]));
      }
    if (threadIdx.x == 0 && rstd_out != nullptr) {
      if (CENTER) mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
    last = stage;
    if (++stage == stages) stage = 0;
  }
}

// The gradient over the same ring, x and dy per stage. Threads own columns: the parameters' gradients stay in registers over
// all rows of a block, so that x and dy are read once. Behind the reduction a row is widened again from the ring, since its g
// and u kept in registers would leave room for half the warps. Three 16-bit rows go through a turn and share its barrier and its
// loads of the weight, two turns fit the ring (16384 rows, layer norm, BF16, against two rows in three stages and one row in
// three: 1024 wide 19.7, 20.6 and 28 us, 2048 34, 36 and 46, 4096 66, 66 and 87, 7168 120, 127 and 140; the traffic alone takes
// 15.4, 31, 62 and 108). Two turns of two FP32 rows of 7168 do not fit; one row per turn is near the copy rate (8192 x 4096 67 us of 62,
// 8192 x 7168 116 of 108).
constexpr int WIDE_THREADS = 448;  // rows of 4097 to 7168 values
__host__ __device__ constexpr int wide_stages(int rows) { return rows > 1 ? 2 : GRAD_STAGES; }
template <typename T, typename W, int NV, int ROWS, int PITCH, bool CENTER>
__global__ void __launch_bounds__(PITCH, STREAM_THREADS / PITCH)
stream_wide_grad_kernel(const T* __restrict__ x, long long x_stride, const T* __restrict__ grad, long long grad_stride,
                        long long rows, int hidden, const W* __restrict__ weight, const float* __restrict__ mean_in,
                        const float* __restrict__ rstd_in, T* __restrict__ grad_x, float* __restrict__ partial_weight,
                        float* __restrict__ partial_bias) {
  chain_wait();
  extern __shared__ uint4 ring_raw[];
  constexpr int stages = wide_stages(ROWS), SUMS = (CENTER ? 2 : 1) * ROWS;
  __shared__ float slots[2][SUMS * STREAM_WARPS];
  constexpr int PAIRS = Quad<T>::PAIRS, VEC = 2 * PAIRS;
  constexpr int WIDTH = NV * PITCH;  // known at compile time: offsets in the ring cost no arithmetic
  const int threads = blockDim.x;
  const int packs = hidden / VEC;
  const float scale = 1.0f / static_cast<float>(hidden);
  uint4* ring = ring_raw + threadIdx.x;  // [stage][row][x, dy][NV][PITCH]; the weight in FP32 [NV][PAIRS / 2][PITCH]
  float4* gain = reinterpret_cast<float4*>(ring_raw + 2 * ROWS * stages * WIDTH) + threadIdx.x;
  for (int i = threadIdx.x; i < SUMS * STREAM_WARPS; i += threads) slots[0][i] = slots[1][i] = 0.0f;
  bool here[NV];
  float2 sum_weight[NV][PAIRS], sum_bias[CENTER ? NV : 1][PAIRS];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * threads + threadIdx.x;
    here[j] = at < packs;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      sum_weight[j][i] = both(0.0f);
      if (CENTER) sum_bias[j][i] = both(0.0f);
    }
    float2 w[PAIRS];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) w[i] = both(1.0f);
    if (here[j] && weight != nullptr) widen_params<W, PAIRS>(weight + at * VEC, w);
#pragma unroll
    for (int i = 0; i < PAIRS; i += 2)
      gain[(j * PAIRS + i) / 2 * PITCH] = make_float4(w[i].x, w[i].y, w[i + 1].x, w[i + 1].y);
  }
  const int first = ROWS * blockIdx.x, step = ROWS * gridDim.x, end = static_cast<int>(rows);
  const T *src_x = x + first * x_stride + threadIdx.x * VEC, *src_grad = grad + first * grad_stride + threadIdx.x * VEC;
  T* dst = grad_x + static_cast<long long>(first) * hidden + threadIdx.x * VEC;
  const long long x_step = step * x_stride, grad_step = step * grad_stride, dst_step = static_cast<long long>(step) * hidden;
  int ahead = first;  // the next rows to copy
  auto fetch = [&](int stage) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (ahead + r < end) {
        uint4* to = ring + (stage * ROWS + r) * 2 * WIDTH;
        const T *a = src_x + r * x_stride, *d = src_grad + r * grad_stride;
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (here[j]) {
            copy_async_16(to + j * PITCH, a + j * threads * VEC);
            copy_async_16(to + WIDTH + j * PITCH, d + j * threads * VEC);
          }
      }
    src_x += x_step, src_grad += grad_step;
    ahead = min(ahead + step, end);
    copy_async_commit();
  };
  for (int s = 0; s < stages - 1; ++s) fetch(s);
  __syncthreads();  // the slots are zero
  int stage = 0, last = stages - 1, turn = 0;
  float next_mean[ROWS], next_rstd[ROWS];
  auto stats = [&](int row) {  // a row that does not exist has scale 0
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      next_mean[r] = CENTER && row + r < end ? mean_in[row + r] : 0.0f;
      next_rstd[r] = row + r < end ? rstd_in[row + r] : 0.0f;
    }
  };
  stats(first);
  for (int row = first; row < end; row += step, turn ^= 1, dst += dst_step) {
    float mean[ROWS], rstd[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) mean[r] = next_mean[r], rstd[r] = next_rstd[r];
    stats(row + step);
    fetch(last);
    copy_async_wait<stages - 1>();
    const uint4* src = ring + stage * ROWS * 2 * WIDTH;
    auto gains = [&](int j, float2* w) {
#pragma unroll
      for (int i = 0; i < PAIRS; i += 2) {
        const float4 q = gain[(j * PAIRS + i) / 2 * PITCH];
        w[i] = make_float2(q.x, q.y), w[i + 1] = make_float2(q.z, q.w);
      }
    };
    auto widen = [&](int j, int r, float2* c, float2* d) {  // x - mean, dy
      uint4 a = make_uint4(0, 0, 0, 0), b = a;
      if (r == 0 || row + r < end) a = src[r * 2 * WIDTH + j * PITCH], b = src[(r * 2 + 1) * WIDTH + j * PITCH];
      Quad<T>::widen(a, c);
      Quad<T>::widen(b, d);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i)
        if (CENTER) c[i] = add2(c[i], both(-mean[r]));
    };
    float2 along[ROWS], total[ROWS];  // rstd times the sums of g (x - mean) and of g
#pragma unroll
    for (int r = 0; r < ROWS; ++r) along[r] = total[r] = both(0.0f);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (here[j]) {
        float2 w[PAIRS];
        gains(j, w);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          float2 c[PAIRS], d[PAIRS];
          widen(j, r, c, d);
#pragma unroll
          for (int i = 0; i < PAIRS; ++i) {
            if (CENTER) sum_bias[j][i] = add2(sum_bias[j][i], d[i]);
            d[i] = times2(d[i], both(rstd[r]));
            sum_weight[j][i] = madd2(d[i], c[i], sum_weight[j][i]);
            d[i] = times2(d[i], w[i]);
            along[r] = madd2(d[i], c[i], along[r]);
            if (CENTER) total[r] = add2(total[r], d[i]);
          }
        }
      }
    float2 sums[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) sums[r] = make_float2(along[r].x + along[r].y, total[r].x + total[r].y);
    block_sums<ROWS, CENTER>(sums, slots[turn]);
    if (grad_x != nullptr) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (r > 0 && row + r >= end) break;
        // dx = rstd (g - (x - mean) rstd mean(g u)) - rstd mean(g), u = (x - mean) rstd: rstd^2 alone may be out of range
        const float2 back = both(-sums[r].x * scale * rstd[r]), offset = both(CENTER ? -sums[r].y * scale : 0.0f);
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (here[j]) {
            float2 c[PAIRS], d[PAIRS], w[PAIRS];
            gains(j, w);
            widen(j, r, c, d);
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
              d[i] = madd2(c[i], back, times2(d[i], w[i]));
              d[i] = CENTER ? madd2(d[i], both(rstd[r]), offset) : times2(d[i], both(rstd[r]));
            }
            st_16(dst + r * hidden + j * threads * VEC, Quad<T>::narrow(d));
          }
      }
    }
    last = stage;
    if (++stage == stages) stage = 0;
  }
  if (partial_weight == nullptr) return;
  chain_next();
  const long long base = static_cast<long long>(blockIdx.x) * hidden + threadIdx.x * VEC;
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (here[j]) {
#pragma unroll
      for (int i = 0; i < PAIRS; i += 2) {
        const long long at = base + j * threads * VEC + 2 * i;
        *reinterpret_cast<float4*>(partial_weight + at) =
            make_float4(sum_weight[j][i].x, sum_weight[j][i].y, sum_weight[j][i + 1].x, sum_weight[j][i + 1].y);
        if (CENTER)
          *reinterpret_cast<float4*>(partial_bias + at) =
              make_float4(sum_bias[j][i].x, sum_bias[j][i].y, sum_bias[j][i + 1].x, sum_bias[j][i + 1].y);
      }
    }
}

// The gradient of the longest rows that stream (above 8192), 32 values per thread and one block per SM, whose ring fills shared
// memory: g and u stay in registers between the reduction and dx.
template <typename T, typename W, int NV, int PITCH, bool CENTER>
__global__ void __launch_bounds__(PITCH)
stream_longest_grad_kernel(const T* __restrict__ x, long long x_stride, const T* __restrict__ grad, long long grad_stride,
                        long long rows, int hidden, const W* __restrict__ weight, const float* __restrict__ mean_in,
                        const float* __restrict__ rstd_in, T* __restrict__ grad_x, float* __restrict__ partial_weight,
                        float* __restrict__ partial_bias) {
  chain_wait();
  extern __shared__ uint4 ring_raw[];
  constexpr int stages = GRAD_STAGES, SUMS = CENTER ? 2 : 1;
  __shared__ __align__(16) float slots[2][SUMS * STREAM_WARPS];
  constexpr int PAIRS = Quad<T>::PAIRS, VEC = 2 * PAIRS;
  constexpr int WIDTH = NV * PITCH;  // known at compile time: offsets in the ring cost no arithmetic
  const int threads = blockDim.x;
  const int packs = hidden / VEC;
  const float scale = 1.0f / static_cast<float>(hidden);
  uint4* ring = ring_raw + threadIdx.x;  // [stage][x, dy][NV][PITCH]
  for (int i = threadIdx.x; i < SUMS * STREAM_WARPS; i += threads) slots[0][i] = slots[1][i] = 0.0f;
  bool here[NV];
  constexpr int QUADS = PAIRS / Quad<W>::PAIRS;  // 16-byte pieces of a pack's parameters, kept as they are
  uint4 params[NV][QUADS];
  float2 sum_weight[NV][PAIRS], sum_bias[CENTER ? NV : 1][PAIRS];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * threads + threadIdx.x;
    here[j] = at < packs;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      sum_weight[j][i] = both(0.0f);
      if (CENTER) sum_bias[j][i] = both(0.0f);
    }
    float2 ones[Quad<W>::PAIRS];
#pragma unroll
    for (int i = 0; i < Quad<W>::PAIRS; ++i) ones[i] = both(1.0f);
#pragma unroll
    for (int i = 0; i < QUADS; ++i)
      params[j][i] = here[j] && weight != nullptr ? ld_16(weight + at * VEC + i * 2 * Quad<W>::PAIRS) : Quad<W>::narrow(ones);
  }
  const T *mine_x = x + threadIdx.x * VEC, *mine_grad = grad + threadIdx.x * VEC;
  auto fetch = [&](long long row, int stage) {
    if (row < rows) {
      const T *a = mine_x + row * x_stride, *d = mine_grad + row * grad_stride;
      uint4* dst = ring + stage * 2 * WIDTH;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (here[j]) {
          copy_async_16(dst + j * PITCH, a + j * threads * VEC);
          copy_async_16(dst + WIDTH + j * PITCH, d + j * threads * VEC);
        }
    }
    copy_async_commit();
  };
  for (int s = 0; s < stages - 1; ++s) fetch(blockIdx.x + static_cast<long long>(s) * gridDim.x, s);
  __syncthreads();  // the slots are zero
  int stage = 0, last = stages - 1, turn = 0;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
    const float mean = CENTER ? mean_in[row] : 0.0f, rstd = rstd_in[row];
    fetch(row + static_cast<long long>(stages - 1) * gridDim.x, last);
    copy_async_wait<stages - 1>();
    float2 u[NV][PAIRS], g[NV][PAIRS];
    float2 along = both(0.0f), total = both(0.0f);  // sums of g u and of g
    const uint4* src = ring + stage * 2 * WIDTH;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (here[j]) {
        float2 w[PAIRS];
#pragma unroll
        for (int i = 0; i < QUADS; ++i) Quad<W>::widen(params[j][i], w + i * Quad<W>::PAIRS);
        Quad<T>::widen(src[j * PITCH], u[j]);
        Quad<T>::widen(src[WIDTH + j * PITCH], g[j]);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          float2 &a = u[j][i], &d = g[j][i];
          if (CENTER) a = add2(a, both(-mean));
          a = times2(a, both(rstd));
          sum_weight[j][i] = madd2(d, a, sum_weight[j][i]);
          if (CENTER) sum_bias[j][i] = add2(sum_bias[j][i], d);
          d = times2(d, w[i]);
          along = madd2(d, a, along);
          if (CENTER) total = add2(total, d);
        }
      }
    float2 sums = make_float2(along.x + along.y, total.x + total.y);
    if (CENTER) sums = block_sum(sums, slots[turn]);
    else sums.x = block_sum(sums.x, slots[turn]);
    if (grad_x != nullptr) {
      T* dst = grad_x + row * hidden + threadIdx.x * VEC;
      const float2 back = both(-sums.x * scale * rstd), offset = both(CENTER ? -sums.y * scale * rstd : 0.0f);
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (here[j]) {
#pragma unroll
          for (int i = 0; i < PAIRS; ++i) {
            const float2 v = CENTER ? madd2(g[j][i], both(rstd), offset) : times2(g[j][i], both(rstd));
            g[j][i] = madd2(u[j][i], back, v);
          }
          st_16(dst + j * threads * VEC, Quad<T>::narrow(g[j]));
        }
    }
    last = stage;
    if (++stage == stages) stage = 0;
  }
  if (partial_weight == nullptr) return;
  chain_next();
  const long long base = static_cast<long long>(blockIdx.x) * hidden + threadIdx.x * VEC;
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (here[j]) {
#pragma unroll
      for (int i = 0; i < PAIRS; i += 2) {
        const long long at = base + j * threads * VEC + 2 * i;
        *reinterpret_cast<float4*>(partial_weight + at) =
            make_float4(sum_weight[j][i].x, sum_weight[j][i].y, sum_weight[j][i + 1].x, sum_weight[j][i + 1].y);
        if (CENTER)
          *reinterpret_cast<float4*>(partial_bias + at) =
              make_float4(sum_bias[j][i].x, sum_bias[j][i].y, sum_bias[j][i + 1].x, sum_bias[j][i + 1].y);
      }
    }
}

// Rows that start on no 16-byte boundary, or are no multiple of 16 bytes, of a tensor that starts on one. A ring again, but of
// windows: the 16-byte pieces that hold a row, copied by whichever thread, so that a barrier stands before their use. The
// first piece may begin with the end of the row before (the first row of all begins on its boundary), the last one ends
// with the row. VEC = 1 or 2 values per access behind that, which bounds these kernels: 16384 rows of 5003 BF16 take 183 us
// forward and 271 for the gradient (50 and 75 us of traffic), 4096 rows of 7161 FP32 57 and 95 us (36 and 54). Straight from
// memory, with too little under way, the BF16 rows took 237 and 497 us.
constexpr int WINDOW_WARPS = 16;
constexpr int WINDOW_MOST = 8192;  // values of a row
constexpr int WINDOW_STAGES = 6;

__device__ __forceinline__ void copy_async_part(void* smem_dst, const void* src, int bytes) {  // 16 bytes, zeros behind `bytes`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(smem_dst))),
               "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void window_fetch(uint8_t* dst, const void* row, int bytes) {
  const uintptr_t start = reinterpret_cast<uintptr_t>(row), end = start + bytes;
  for (uintptr_t at = (start & ~static_cast<uintptr_t>(15)) + threadIdx.x * 16; at < end; at += blockDim.x * 16) {
    const int valid = end - at < 16 ? static_cast<int>(end - at) : 16;
    copy_async_part(dst + (at - (start & ~static_cast<uintptr_t>(15))), reinterpret_cast<const void*>(at), valid);
  }
}
__device__ __forceinline__ int window_shift(const void* row) { return static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15); }
__device__ __forceinline__ void window_wait(int pending) {
  switch (pending) {
    case 1: copy_async_wait<1>(); break;
    case 2: copy_async_wait<2>(); break;
    case 3: copy_async_wait<3>(); break;
    case 4: copy_async_wait<4>(); break;
    default: copy_async_wait<5>(); break;
  }
}

template <typename T, typename W, int VEC, int NV, bool CENTER>
__global__ void __launch_bounds__(32 * WINDOW_WARPS)
window_norm_kernel(const T* __restrict__ x, long long x_stride, long long rows, int hidden, const W* __restrict__ weight,
                   const W* __restrict__ bias, float eps, T* __restrict__ y, float* __restrict__ mean_out,
                   float* __restrict__ rstd_out, int stages, int window) {
  chain_wait();
  chain_next();
  extern __shared__ uint4 ring_raw[];
  __shared__ float slots[2][WINDOW_WARPS];
  uint8_t* ring = reinterpret_cast<uint8_t*>(ring_raw);
  const int threads = blockDim.x, packs = hidden / VEC, bytes = hidden * static_cast<int>(sizeof(T));
  const float scale = 1.0f / static_cast<float>(hidden);
  if (threadIdx.x < WINDOW_WARPS) slots[0][threadIdx.x] = slots[1][threadIdx.x] = 0.0f;
  bool here[NV];
  float w[NV][VEC], b[CENTER ? NV : 1][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * threads + threadIdx.x;
    here[j] = at < packs;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[j][e] = here[j] && weight != nullptr ? widen(weight[at * VEC + e]) : 1.0f;
      if (CENTER) b[j][e] = here[j] && bias != nullptr ? widen(bias[at * VEC + e]) : 0.0f;
    }
  }
  auto fetch = [&](long long row, int stage) {
    if (row < rows) window_fetch(ring + stage * window, x + row * x_stride, bytes);
    copy_async_commit();
  };
  for (int s = 0; s < stages - 1; ++s) fetch(blockIdx.x + static_cast<long long>(s) * gridDim.x, s);
  int stage = 0, last = stages - 1, turn = 0;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    // the stage that is filled now was read before a barrier of the row before
    fetch(row + static_cast<long long>(stages - 1) * gridDim.x, last);
    window_wait(stages - 1);
    __syncthreads();
    const T* src = reinterpret_cast<const T*>(ring + stage * window + window_shift(x + row * x_stride)) + threadIdx.x * VEC;
    float v[NV][VEC];
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[j][e] = 0.0f;
      if (here[j]) {
        const Pack<T, VEC> in = load_pack<T, VEC>(src + j * threads * VEC);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          v[j][e] = widen(in.v[e]);
          sum += v[j][e];
        }
      }
    }
    float mean = 0.0f;
    if (CENTER) {
      mean = block_sum(sum, slots[turn]) * scale;
      turn ^= 1;
    }
    float square = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (CENTER) v[j][e] = here[j] ? v[j][e] - mean : 0.0f;
        square += v[j][e] * v[j][e];
      }
    const float rstd = rsqrtf(block_sum(square, slots[turn]) * scale + eps);
    turn ^= 1;
    T* dst = y + row * hidden + threadIdx.x * VEC;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (here[j]) {
        Pack<T, VEC> out;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float u = v[j][e] * rstd;
          out.v[e] = narrow<T>(CENTER ? u * w[j][e] + b[j][e] : u * w[j][e]);
        }
        store_pack<T, VEC>(dst + j * threads * VEC, out);
      }
    if (threadIdx.x == 0 && rstd_out != nullptr) {
      if (CENTER) mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
    last = stage;
    if (++stage == stages) stage = 0;
  }
}

template <typename T, typename W, int VEC, int NV, bool CENTER>
__global__ void __launch_bounds__(32 * WINDOW_WARPS)
window_norm_grad_kernel(const T* __restrict__ x, long long x_stride, const T* __restrict__ grad, long long grad_stride,
                        long long rows, int hidden, const W* __restrict__ weight, const float* __restrict__ mean_in,
                        const float* __restrict__ rstd_in, T* __restrict__ grad_x, float* __restrict__ partial_weight,
                        float* __restrict__ partial_bias, int stages, int window) {
  chain_wait();
  extern __shared__ uint4 ring_raw[];
  __shared__ __align__(16) float slots[2][2 * WINDOW_WARPS];
  uint8_t* ring = reinterpret_cast<uint8_t*>(ring_raw);  // [stage][x, dy]
  const int threads = blockDim.x, packs = hidden / VEC, bytes = hidden * static_cast<int>(sizeof(T));
  const float scale = 1.0f / static_cast<float>(hidden);
  for (int i = threadIdx.x; i < 2 * WINDOW_WARPS; i += threads) slots[0][i] = slots[1][i] = 0.0f;
  bool here[NV];
  float w[NV][VEC], sum_weight[NV][VEC], sum_bias[CENTER ? NV : 1][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * threads + threadIdx.x;
    here[j] = at < packs;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[j][e] = here[j] && weight != nullptr ? widen(weight[at * VEC + e]) : 1.0f;
      sum_weight[j][e] = 0.0f;
      if (CENTER) sum_bias[j][e] = 0.0f;
    }
  }
  auto fetch = [&](long long row, int stage) {
    if (row < rows) {
      window_fetch(ring + 2 * stage * window, x + row * x_stride, bytes);
      window_fetch(ring + (2 * stage + 1) * window, grad + row * grad_stride, bytes);
    }
    copy_async_commit();
  };
  for (int s = 0; s < stages - 1; ++s) fetch(blockIdx.x + static_cast<long long>(s) * gridDim.x, s);
  int stage = 0, last = stages - 1, turn = 0;
  float next_mean = CENTER && blockIdx.x < rows ? mean_in[blockIdx.x] : 0.0f;
  float next_rstd = blockIdx.x < rows ? rstd_in[blockIdx.x] : 0.0f;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
    const float mean = next_mean, rstd = next_rstd;
    const long long next = row + gridDim.x;
    if (next < rows) {
      if (CENTER) next_mean = mean_in[next];
      next_rstd = rstd_in[next];
    }
    fetch(row + static_cast<long long>(stages - 1) * gridDim.x, last);
    window_wait(stages - 1);
    __syncthreads();
    const uint8_t* at = ring + 2 * stage * window;
    const T* a = reinterpret_cast<const T*>(at + window_shift(x + row * x_stride)) + threadIdx.x * VEC;
    const T* d = reinterpret_cast<const T*>(at + window + window_shift(grad + row * grad_stride)) + threadIdx.x * VEC;
    float u[NV][VEC], g[NV][VEC];
    float2 sums = make_float2(0.0f, 0.0f);  // of g * u and of g
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (here[j]) {
        const Pack<T, VEC> in = load_pack<T, VEC>(a + j * threads * VEC), dy = load_pack<T, VEC>(d + j * threads * VEC);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float dv = widen(dy.v[e]);
          u[j][e] = (widen(in.v[e]) - mean) * rstd;
          sum_weight[j][e] += dv * u[j][e];
          if (CENTER) sum_bias[j][e] += dv;
          g[j][e] = dv * w[j][e];
          sums.x += g[j][e] * u[j][e];
          sums.y += g[j][e];
        }
      }
    sums = block_sum(sums, slots[turn]);
    last = stage;
    if (++stage == stages) stage = 0;
    if (grad_x == nullptr) continue;
    const float along = sums.x * scale, offset = CENTER ? sums.y * scale : 0.0f;
    T* dst = grad_x + row * hidden + threadIdx.x * VEC;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (here[j]) {
        Pack<T, VEC> out;
#pragma unroll
        for (int e = 0; e < VEC; ++e) out.v[e] = narrow<T>((g[j][e] - u[j][e] * along - offset) * rstd);
        store_pack<T, VEC>(dst + j * threads * VEC, out);
      }
  }
  if (partial_weight == nullptr) return;
  chain_next();
  const long long base = static_cast<long long>(blockIdx.x) * hidden;
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (here[j]) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const long long at = base + (j * threads + static_cast<int>(threadIdx.x)) * VEC + e;
        partial_weight[at] = sum_weight[j][e];
        if (CENTER) partial_bias[at] = sum_bias[j][e];
      }
    }
}

// Short rows, gradient: a warp per row, no barrier per row, the next row's loads under way. The warps of a block join their sums
// over rows one after the other in shared memory. Latency and the 32 accumulators per lane bound it: 16384 rows of 512 BF16
// 19.5 us (7.7 us of traffic); at 1024 the block kernel above is faster (70 against 25 us).
constexpr int SHORT_WARPS = 8;

template <typename T, typename W, int VEC, int NV, bool CENTER>
__global__ void __launch_bounds__(32 * SHORT_WARPS, 2)
short_norm_grad_kernel(const T* __restrict__ x, long long x_stride, const T* __restrict__ grad, long long grad_stride,
                       long long rows, int hidden, const W* __restrict__ weight, const float* __restrict__ mean_in,
                       const float* __restrict__ rstd_in, T* __restrict__ grad_x, float* __restrict__ partial_weight,
                       float* __restrict__ partial_bias) {
  chain_wait();
  __shared__ float joined[2][32 * VEC * NV];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, packs = hidden / VEC;
  const float scale = 1.0f / static_cast<float>(hidden);
  bool here[NV];
  float w[NV][VEC], sum_weight[NV][VEC], sum_bias[CENTER ? NV : 1][VEC];
  Pack<T, VEC> next_x[NV], next_grad[NV];
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto fetch = [&](long long row) {
    const T *a = x + row * x_stride + lane * VEC, *d = grad + row * grad_stride + lane * VEC;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (here[j]) {
        next_x[j] = load_pack<T, VEC>(a + j * 32 * VEC);
        next_grad[j] = load_pack<T, VEC>(d + j * 32 * VEC);
      }
    if (CENTER) next_mean = mean_in[row];
    next_rstd = rstd_in[row];
  };
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * 32 + lane;
    here[j] = at < packs;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      next_x[j].v[e] = next_grad[j].v[e] = narrow<T>(0.0f);
      w[j][e] = here[j] && weight != nullptr ? widen(weight[at * VEC + e]) : 1.0f;
      sum_weight[j][e] = 0.0f;
      if (CENTER) sum_bias[j][e] = 0.0f;
    }
  }
  const long long step = static_cast<long long>(gridDim.x) * SHORT_WARPS;
  const long long first = static_cast<long long>(blockIdx.x) * SHORT_WARPS + warp;
  if (first < rows) fetch(first);
  for (long long row = first; row < rows; row += step) {
    const float mean = next_mean, rstd = next_rstd;
    float u[NV][VEC], g[NV][VEC];
    float along = 0.0f, total = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = widen(next_grad[j].v[e]);
        u[j][e] = (widen(next_x[j].v[e]) - mean) * rstd;
        sum_weight[j][e] += d * u[j][e];
        if (CENTER) sum_bias[j][e] += d;
        g[j][e] = d * w[j][e];
        along += g[j][e] * u[j][e];
        if (CENTER) total += g[j][e];
      }
    if (row + step < rows) fetch(row + step);
    if (grad_x == nullptr) continue;
    along = warp_sum(along) * scale;
    total = CENTER ? warp_sum(total) * scale : 0.0f;
    T* dst = grad_x + row * hidden + lane * VEC;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (here[j]) {
        Pack<T, VEC> out;
#pragma unroll
        for (int e = 0; e < VEC; ++e) out.v[e] = narrow<T>((g[j][e] - u[j][e] * along - total) * rstd);
        store_pack<T, VEC>(dst + j * 32 * VEC, out);
      }
  }
  if (partial_weight == nullptr) return;
  chain_next();
  for (int turn = 0; turn < SHORT_WARPS; ++turn) {
    if (turn == warp) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int at = (j * 32 + lane) * VEC + e;
          joined[0][at] = (turn > 0 ? joined[0][at] : 0.0f) + sum_weight[j][e];
          if (CENTER) joined[1][at] = (turn > 0 ? joined[1][at] : 0.0f) + sum_bias[j][e];
        }
    }
    __syncthreads();
  }
  const long long base = static_cast<long long>(blockIdx.x) * hidden;
  for (int c = threadIdx.x; c < hidden; c += 32 * SHORT_WARPS) {
    partial_weight[base + c] = joined[0][c];
    if (CENTER) partial_bias[base + c] = joined[1][c];
  }
}

// Rows too long for a block's registers, or of a tensor that starts on no 16-byte boundary: dx by one block per row, the
// parameters' partial sums by columns, everything read twice or three times (mostly from L2).
template <typename T, typename W, bool CENTER>
__global__ void __launch_bounds__(1024) long_row_norm_grad_kernel(const T* __restrict__ x, long long x_stride,
                                                                  const T* __restrict__ grad, long long grad_stride,
                                                                  int hidden, const W* __restrict__ weight,
                                                                  const float* __restrict__ mean_in,
                                                                  const float* __restrict__ rstd_in, T* __restrict__ grad_x) {
  chain_wait();
  chain_next();
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
  chain_wait();
  chain_next();
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

// Parameters' gradients: the partial sums of a column in the order of the blocks that made them, 32 slices of them in
// parallel (8 slices took 12 us for 296 sums of 7168 columns, 32 take 5 to 6).
constexpr int FINISH_SLICES = 32;
template <typename W>
__global__ void __launch_bounds__(32 * FINISH_SLICES) param_grad_kernel(const float* __restrict__ partial_weight,
                                                                        const float* __restrict__ partial_bias, int parts,
                                                                        int hidden, W* __restrict__ grad_weight,
                                                                        W* __restrict__ grad_bias) {
  __shared__ float sums[2][FINISH_SLICES][32];
  chain_wait();
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
#pragma unroll 8
  for (int s = 0; s < FINISH_SLICES; ++s) v += sums[threadIdx.y][s][threadIdx.x];
  out[c] = narrow<W>(v);
}

bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int round_up(int v, int to) { return (v + to - 1) / to * to; }

constexpr int FORWARD_PACKS = 4;  // packs of 16 bytes per thread and row

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

// Blocks of the gradient kernels per SM at most, each with partial sums of its own: fewer of long rows.
int grad_blocks(long long hidden) { return hidden <= 1024 ? 8 : hidden <= 2048 ? 6 : hidden <= 4096 ? 3 : 2; }
long long grad_parts(long long rows, long long hidden) {
  const long long most = static_cast<long long>(grad_blocks(hidden)) * sm_count();
  return rows < most ? rows : most;
}

template <typename T, typename W, int VEC, int NV, bool CENTER>
int launch_short(const NormCall& c) {
  const long long blocks = (c.rows + SHORT_ROWS - 1) / SHORT_ROWS;
  return launch_chained(short_norm_kernel<T, W, VEC, NV, CENTER>, dim3(static_cast<unsigned>(blocks)), dim3(32 * SHORT_ROWS), 0,
                        c.stream, static_cast<const T*>(c.x), c.x_stride, c.rows, c.hidden, static_cast<const W*>(c.weight),
                        static_cast<const W*>(c.bias), c.eps, static_cast<T*>(c.y), c.mean, c.rstd);
}

constexpr int SM_SHARED = 227 * 1024;
constexpr int STREAM_SHARED = SM_SHARED - 2048;  // beside the reductions' slots

// Blocks of `threads` threads with `bytes` of shared memory that an SM holds of a kernel; asked once per block size.
struct Residency {
  int blocks[HMC_MAX_DEVICES][WINDOW_WARPS + 1];
};
template <typename Kernel>
int resident_blocks(Kernel kernel, int threads, int bytes, Residency& known, int* blocks) {
  int dev = 0;
  HMC_CUDA_OK(cudaGetDevice(&dev));
  int* slot = dev < HMC_MAX_DEVICES ? &known.blocks[dev][threads / 32] : nullptr;
  if (slot == nullptr || *slot == 0) {
    if (bytes > 0) HMC_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, STREAM_SHARED));
    int found = 0;
    HMC_CUDA_OK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&found, kernel, threads, bytes));
    if (found < 1) found = 1;
    if (slot == nullptr) {
      *blocks = found;
      return 0;
    }
    *slot = found;
  }
  *blocks = *slot;
  return 0;
}

template <typename T, typename W, int NV, bool CENTER>
int launch_stream(const NormCall& c) {
  constexpr int VEC = 16 / sizeof(T);
  const int threads = round_up((c.hidden / VEC + NV - 1) / NV, 32);
  const int bytes = FORWARD_STAGES * NV * threads * 16;
  static Residency known{};
  auto kernel = stream_norm_kernel<T, W, NV, CENTER>;
  int blocks = 0;
  if (int rc = resident_blocks(kernel, threads, bytes, known, &blocks)) return rc;
  const long long most = static_cast<long long>(blocks) * sm_count();
  return launch_chained(kernel, dim3(static_cast<unsigned>(c.rows < most ? c.rows : most)), dim3(threads), bytes, c.stream,
                        static_cast<const T*>(c.x), c.x_stride, c.rows, c.hidden, static_cast<const W*>(c.weight),
                        static_cast<const W*>(c.bias), c.eps, static_cast<T*>(c.y), c.mean, c.rstd);
}

// Packs per thread, so that a row has about 256 threads and no more than STREAM_THREADS.
template <typename T, typename W, bool CENTER>
int stream(const NormCall& c) {
  const int packs = c.hidden / (16 / static_cast<int>(sizeof(T)));
  if (packs <= 256) return launch_stream<T, W, 1, CENTER>(c);
  return packs <= 512 ? launch_stream<T, W, 2, CENTER>(c) : launch_stream<T, W, 4, CENTER>(c);
}

template <typename T, typename W, int NV, int PITCH, bool CENTER>
int launch_longest_grad(NormCall& c) {
  constexpr int VEC = 16 / sizeof(T);
  const int threads = round_up((c.hidden / VEC + NV - 1) / NV, 32);
  constexpr int bytes = GRAD_STAGES * 2 * NV * PITCH * 16;
  static PerDeviceFlag configured{};
  auto kernel = stream_longest_grad_kernel<T, W, NV, PITCH, CENTER>;
  if (int rc = allow_dynamic_smem(kernel, bytes, configured)) return rc;
  c.parts = static_cast<int>(c.rows < sm_count() ? c.rows : sm_count());
  return launch_chained(kernel, dim3(static_cast<unsigned>(c.parts)), dim3(threads), bytes, c.stream,
                        static_cast<const T*>(c.x), c.x_stride, static_cast<const T*>(c.grad), c.grad_stride, c.rows, c.hidden,
                        static_cast<const W*>(c.weight), c.mean_in, c.rstd_in, static_cast<T*>(c.y), c.partial_weight,
                        c.partial_bias);
}

template <typename T, typename W, int NV, int ROWS, int PITCH, bool CENTER>
int launch_wide_grad(NormCall& c) {
  constexpr int VEC = 16 / sizeof(T);
  const int threads = round_up((c.hidden / VEC + NV - 1) / NV, 32);
  const int bytes = NV * PITCH * (wide_stages(ROWS) * ROWS * 2 * 16 + VEC * 4);
  static Residency known{};
  auto kernel = stream_wide_grad_kernel<T, W, NV, ROWS, PITCH, CENTER>;
  int blocks = 0;
  if (int rc = resident_blocks(kernel, threads, bytes, known, &blocks)) return rc;
  if (blocks > grad_blocks(c.hidden)) blocks = grad_blocks(c.hidden);
  const long long most = static_cast<long long>(blocks) * sm_count(), pieces = (c.rows + ROWS - 1) / ROWS;
  c.parts = static_cast<int>(pieces < most ? pieces : most);
  return launch_chained(kernel, dim3(static_cast<unsigned>(c.parts)), dim3(threads), bytes, c.stream,
                        static_cast<const T*>(c.x), c.x_stride, static_cast<const T*>(c.grad), c.grad_stride, c.rows, c.hidden,
                        static_cast<const W*>(c.weight), c.mean_in, c.rstd_in, static_cast<T*>(c.y), c.partial_weight,
                        c.partial_bias);
}

// Threads of the gradient of the longest rows that stream, 32 values each: three stages of x and dy fill shared memory.
template <typename T>
constexpr int LONGEST = sizeof(T) == 4 ? 288 : STREAM_THREADS;

template <typename T, typename W, bool CENTER>
int stream_grad(NormCall& c) {
  constexpr int NV = sizeof(T) == 4 ? 4 : 2;    // 16 values per thread
  constexpr int ROWS = sizeof(T) == 4 ? 1 : 3;  // of a turn
  if (c.hidden <= 16 * 64) return launch_wide_grad<T, W, NV, ROWS, 64, CENTER>(c);
  if (c.hidden <= 16 * 128) return launch_wide_grad<T, W, NV, ROWS, 128, CENTER>(c);
  if (c.hidden <= 16 * 256) return launch_wide_grad<T, W, NV, ROWS, 256, CENTER>(c);
  if (c.hidden <= 16 * WIDE_THREADS) return launch_wide_grad<T, W, NV, ROWS, WIDE_THREADS, CENTER>(c);
  if (c.hidden <= 16 * STREAM_THREADS) return launch_wide_grad<T, W, NV, ROWS, STREAM_THREADS, CENTER>(c);
  return launch_longest_grad<T, W, 2 * NV, LONGEST<T>, CENTER>(c);
}

// Windows of a row in a ring of `each` of them per stage, of the longest row that the block's threads hold: the shared memory and
// with it the blocks per SM, from which the gradient's order of summation follows, depend on the block size alone.
struct WindowRing {
  int window, stages, bytes;
  WindowRing(long long row_bytes, int each) {
    window = static_cast<int>((row_bytes + 15 + 15) / 16 * 16);
    stages = STREAM_SHARED / (each * window);
    if (stages > WINDOW_STAGES) stages = WINDOW_STAGES;
    bytes = stages * each * window;
  }
};

template <typename T, typename W, int VEC, int NV, bool CENTER>
int launch_window(const NormCall& c) {
  const int threads = round_up((c.hidden / VEC + NV - 1) / NV, 32);
  const WindowRing ring(threads * NV * VEC * sizeof(T), 1);
  static Residency known{};
  auto kernel = window_norm_kernel<T, W, VEC, NV, CENTER>;
  int blocks = 0;
  if (int rc = resident_blocks(kernel, threads, ring.bytes, known, &blocks)) return rc;
  const long long most = static_cast<long long>(blocks) * sm_count();
  return launch_chained(kernel, dim3(static_cast<unsigned>(c.rows < most ? c.rows : most)), dim3(threads), ring.bytes, c.stream,
                        static_cast<const T*>(c.x), c.x_stride, c.rows, c.hidden, static_cast<const W*>(c.weight),
                        static_cast<const W*>(c.bias), c.eps, static_cast<T*>(c.y), c.mean, c.rstd, ring.stages, ring.window);
}

template <typename T, typename W, int VEC, bool CENTER>
int window(const NormCall& c) {
  if (c.hidden <= 2048) return launch_window<T, W, VEC, 8 / VEC, CENTER>(c);
  return launch_window<T, W, VEC, 16 / VEC, CENTER>(c);
}

template <typename T, typename W, bool CENTER>
int forward(const NormCall& c) {
  constexpr int VEC = 16 / sizeof(T);
  const bool wide = c.hidden % VEC == 0 && c.x_stride % VEC == 0 && aligned_to(c.x, 16) && aligned_to(c.y, 16) &&
                    aligned_to(c.weight, 16) && aligned_to(c.bias, 16);
  if (wide && c.hidden <= STREAM_THREADS * VEC * FORWARD_PACKS) return stream<T, W, CENTER>(c);
  const bool pairs = c.hidden % 2 == 0 && c.x_stride % 2 == 0 && aligned_to(c.x, 2 * sizeof(T)) && aligned_to(c.y, 2 * sizeof(T)) &&
                     aligned_to(c.weight, 2 * sizeof(W)) && aligned_to(c.bias, 2 * sizeof(W));
  if (c.hidden <= 32 * 16)
    return pairs ? launch_short<T, W, 2, 8, CENTER>(c) : launch_short<T, W, 1, 16, CENTER>(c);
  if (aligned_to(c.x, 16) && c.hidden <= WINDOW_MOST) return pairs ? window<T, W, 2, CENTER>(c) : window<T, W, 1, CENTER>(c);
  return launch_chained(long_row_norm_kernel<T, W, CENTER>, dim3(static_cast<unsigned>(c.rows)), dim3(1024), 0, c.stream,
                        static_cast<const T*>(c.x), c.x_stride, c.rows, c.hidden, static_cast<const W*>(c.weight),
                        static_cast<const W*>(c.bias), c.eps, static_cast<T*>(c.y), c.mean, c.rstd);
}

template <typename T, typename W, int VEC, int NV, bool CENTER>
int launch_window_grad(NormCall& c) {
  const int threads = round_up((c.hidden / VEC + NV - 1) / NV, 32);
  const WindowRing ring(threads * NV * VEC * sizeof(T), 2);
  static Residency known{};
  auto kernel = window_norm_grad_kernel<T, W, VEC, NV, CENTER>;
  int blocks = 0;
  if (int rc = resident_blocks(kernel, threads, ring.bytes, known, &blocks)) return rc;
  if (blocks > grad_blocks(c.hidden)) blocks = grad_blocks(c.hidden);
  const long long most = static_cast<long long>(blocks) * sm_count();
  c.parts = static_cast<int>(c.rows < most ? c.rows : most);
  return launch_chained(kernel, dim3(static_cast<unsigned>(c.parts)), dim3(threads), ring.bytes, c.stream,
                        static_cast<const T*>(c.x), c.x_stride, static_cast<const T*>(c.grad), c.grad_stride, c.rows, c.hidden,
                        static_cast<const W*>(c.weight), c.mean_in, c.rstd_in, static_cast<T*>(c.y), c.partial_weight,
                        c.partial_bias, ring.stages, ring.window);
}

template <typename T, typename W, int VEC, int NV, bool CENTER>
int launch_short_grad(NormCall& c) {
  static Residency known{};
  int blocks = 0;
  if (int rc = resident_blocks(short_norm_grad_kernel<T, W, VEC, NV, CENTER>, 32 * SHORT_WARPS, 0, known, &blocks)) return rc;
  if (blocks > 4) blocks = 4;  // 32 warps
  const long long most = static_cast<long long>(blocks) * sm_count();
  const long long pieces = (c.rows + SHORT_WARPS - 1) / SHORT_WARPS;
  c.parts = static_cast<int>(pieces < most ? pieces : most);
  return launch_chained(short_norm_grad_kernel<T, W, VEC, NV, CENTER>, dim3(static_cast<unsigned>(c.parts)),
                        dim3(32 * SHORT_WARPS), 0, c.stream, static_cast<const T*>(c.x), c.x_stride,
                        static_cast<const T*>(c.grad), c.grad_stride, c.rows, c.hidden, static_cast<const W*>(c.weight),
                        c.mean_in, c.rstd_in, static_cast<T*>(c.y), c.partial_weight, c.partial_bias);
}

template <typename T, typename W, int VEC, bool CENTER>
int window_grad(NormCall& c) {
  if (c.hidden <= 2048) return launch_window_grad<T, W, VEC, 8 / VEC, CENTER>(c);
  return launch_window_grad<T, W, VEC, 16 / VEC, CENTER>(c);
}

template <typename T, typename W, bool CENTER>
int gradient(NormCall& c) {
  constexpr int VEC = 16 / sizeof(T);
  const bool wide = c.hidden % VEC == 0 && c.x_stride % VEC == 0 && c.grad_stride % VEC == 0 && aligned_to(c.x, 16) &&
                    aligned_to(c.grad, 16) && aligned_to(c.y, 16) && aligned_to(c.weight, 16);
  const bool pairs = c.hidden % 2 == 0 && c.x_stride % 2 == 0 && c.grad_stride % 2 == 0 && aligned_to(c.x, 2 * sizeof(T)) &&
                     aligned_to(c.grad, 2 * sizeof(T)) && aligned_to(c.y, 2 * sizeof(T));
  int rc = 0;
  if (wide && c.hidden <= 32 * VEC) {
    rc = launch_short_grad<T, W, VEC, 1, CENTER>(c);
  } else if (wide && c.hidden <= 32 * VEC * 2) {
    rc = launch_short_grad<T, W, VEC, 2, CENTER>(c);
  } else if (wide && c.hidden <= 32 * LONGEST<T>) {
    rc = stream_grad<T, W, CENTER>(c);
  } else if (c.hidden <= 32 * 16) {
    rc = pairs ? launch_short_grad<T, W, 2, 8, CENTER>(c) : launch_short_grad<T, W, 1, 16, CENTER>(c);
  } else if (aligned_to(c.x, 16) && aligned_to(c.grad, 16) && c.hidden <= WINDOW_MOST) {
    rc = pairs ? window_grad<T, W, 2, CENTER>(c) : window_grad<T, W, 1, CENTER>(c);
  } else {
    if (c.y != nullptr) {
      if (int rc = launch_chained(long_row_norm_grad_kernel<T, W, CENTER>, dim3(static_cast<unsigned>(c.rows)), dim3(1024), 0,
                                  c.stream, static_cast<const T*>(c.x), c.x_stride, static_cast<const T*>(c.grad),
                                  c.grad_stride, c.hidden, static_cast<const W*>(c.weight), c.mean_in, c.rstd_in,
                                  static_cast<T*>(c.y))) return rc;
    }
    if (c.partial_weight != nullptr) {
      const dim3 grid((c.hidden + 255) / 256, c.parts);
      if (int rc = launch_chained(column_grad_kernel<T, CENTER>, grid, dim3(256), 0, c.stream, static_cast<const T*>(c.x),
                                  c.x_stride, static_cast<const T*>(c.grad), c.grad_stride, c.rows, c.hidden, c.mean_in,
                                  c.rstd_in, c.partial_weight, c.partial_bias)) return rc;
    }
  }
  if (rc != 0) return rc;
  if (c.partial_weight != nullptr) {
    return launch_chained(param_grad_kernel<W>, dim3((c.hidden + 31) / 32), dim3(32, FINISH_SLICES), 0, c.stream,
                          c.partial_weight,
                          c.partial_bias, c.parts, c.hidden, static_cast<W*>(c.grad_weight), static_cast<W*>(c.grad_bias));
  }
  return 0;
}

template <typename T, typename W>
int run(NormCall& c, bool center, bool backward) {
  if (backward) return center ? gradient<T, W, true>(c) : gradient<T, W, false>(c);
  return center ? forward<T, W, true>(c) : forward<T, W, false>(c);
}

int run(NormCall& c, int dtype, int affine_dtype, bool center, bool backward) {
  if (dtype == HMC_DTYPE_F32) return run<float, float>(c, center, backward);
  if (dtype == HMC_DTYPE_BF16)
    return affine_dtype == HMC_DTYPE_F32 ? run<__nv_bfloat16, float>(c, center, backward)
                                         : run<__nv_bfloat16, __nv_bfloat16>(c, center, backward);
  return affine_dtype == HMC_DTYPE_F32 ? run<__half, float>(c, center, backward) : run<__half, __half>(c, center, backward);
}

int check(const char* name, int64_t rows, int64_t hidden, int64_t stride, int dtype, int affine_dtype) {
  // blocks step through the rows in 32 bits, by less than 2^16
  HMC_REQUIRE(rows >= 0 && rows <= HMC_NORM_MAX_ROWS && hidden > 0 && hidden <= HMC_NORM_MAX_HIDDEN, HMC_ERR_INVALID,
              "%s: rows (%lld) must be in [0, %d] and hidden (%lld) in [1, %d]", name, (long long)rows, HMC_NORM_MAX_ROWS,
              (long long)hidden, HMC_NORM_MAX_HIDDEN);
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
  return 2 * hmc::grad_parts(rows, hidden) * hidden * static_cast<int64_t>(sizeof(float));
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
  c.grad_weight = grad_weight, c.grad_bias = grad_bias, c.parts = static_cast<int>(grad_parts(rows, hidden)), c.stream = s;
  if (params) {
    c.partial_weight = static_cast<float*>(workspace);
    c.partial_bias = c.partial_weight + static_cast<long long>(c.parts) * hidden;
  }
  return run(c, dtype, affine_dtype, center != 0, true);
}
