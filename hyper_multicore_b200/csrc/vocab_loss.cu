// Cross entropy of hidden states over a vocabulary, logits held in 16 bits for the gradient or not at all:
//   l_ij = x_i . w_j,  lse_i = log sum_j exp(l_ij),  loss_i = lse_i - l_i,t(i)
//   p_ij = exp(l_ij - lse_i)
//   dx_i = g_i (sum_{j != t(i)} p_ij w_j + (p_i,t(i) - 1) w_t(i))
//   dw_j = sum_{i: t(i) != j} g_i p_ij x_i + sum_{i: t(i) = j} g_i (p_ij - 1) x_i
// with g the gradient of the loss of a token. Tokens whose target is ignored are left out before anything is computed: the
// rows that count are packed, and every kernel takes their number from the device.
//
// Forward: one GEMM over 256 x 256 tiles whose epilogue keeps a row's maximum and sum of exponentials per 128 columns, and
// a kernel that joins those. Gradient: p in BF16 for a piece of the vocabulary, from what the forward kept of the logits or
// from the same GEMM again, and two GEMMs that take the piece to the two gradients. p without the target's entry only: that
// one is p - 1, which cancels for a token the model is sure of and carries the largest weight for one it is not, so it stays
// in FP32 (expm1 of -loss) and meets the products in FP32: for dx as the row w_t(i) in the epilogue, for dw as a sum over the
// tokens of a word made beforehand. The other entries are off by 2^-8 of their value at most (BF16) and, where their logits
// were kept, by 3.4e-4 before that. A row of dx is made of differences, p_ij (w_j - w_t(i)): what the words' rows have in common
// cancels only if the coefficients of a row add up to nothing. So the rounded entries of a row are added up in FP32, the
// target's row enters with minus that sum, and the whole is scaled by what the sum should be (1 - p_t(i)) over what it is. An error
// that all entries share, or that of one word which holds nearly all of the rest, then cancels too; left is
// 2 * 2^-8 sum_j p_ij |w_j - w_c| at most, c the likeliest wrong word. (Rows of 256 over 1000 words with a common component of ten times
// their own size: up to 1.8 % of a row's norm without this, its own rounding of 0.2 % with it. What the
// scaling puts right as a whole it may take from the lesser entries: one that is not the largest may be off by twice 2^-8.) A row of dw is not
// scaled: it is off by 2^-8 sum_i g_i p_ij |x_i| at most, each entry by its own rounding and no more; that does not average out where one
// token holds a word or all tokens rate it alike (0.66 % of a row's norm where what they have in common nearly cancels).
// A training step of 8192 x 4096 x 131072 takes 23.0 ms with all its logits kept (2 GiB of 16-bit codes) and 28.7 ms with none,
// 512 x 1024 x 32000 186 against 207 us (two inputs in turn). Gradients taken in the forward pass would hold the weight's gradient in FP32 until the
// backward one and only fit a loss that is reduced.
//
// The GEMM: CTA pairs (tcgen05.mma.cta_group::2, M = N = 256), one TMA producer, one issuer, eight epilogue warps, two
// accumulators; the layouts of the operands are those of the grouped GEMMs. Bound by the tensor cores: 4096 x 32768 x 4096 takes
// 750 to 785 us in its four forms (1400 to 1466 TFLOP/s, 0.86 to 0.90 of cuBLAS in a burst, tensor pipe 78 to 87 % busy); over seconds the
// power limit leaves 1250 to 1330 (cuBLAS: 1380). Short k (1024 and below) is bound by L2: 1 MB per 256 x 256 tile.
#include <cuda.h>

#include "common.cuh"
#include "gemm_shared.cuh"
#include "sm100.cuh"

namespace hmc {
namespace {

using namespace sm100;
using gemm::A_TILE_BYTES;
using gemm::ACC_STAGES;
using gemm::BK;
using gemm::CHUNK_BYTES;
using gemm::EPI_WARPS;
using gemm::NUM_THREADS;
using gemm::PIPE_BUDGET_NS;
using gemm::STORE_STAGE_BYTES;
using gemm::SWIZZLE_128B;
using gemm::TMEM_COLS;

constexpr int TILE = 256;       // rows and columns of a pair's tile
constexpr int HALF = TILE / 2;  // rows of A and columns of B that a CTA loads
constexpr int STAGE_BYTES = 2 * A_TILE_BYTES;
constexpr int STAGES = 6;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_WARPS * STORE_STAGE_BYTES + 1024 + 256;
constexpr int MAX_PARTS = 16;  // of a tile that is cut along k
constexpr int MIN_PART = 8;    // k-blocks of a part, at the least
// k-blocks that add up inside the tensor core before the sum goes to FP32 registers (STATS, few tokens). The loss of 8192 tokens
// of 4096 over 131072 words: 8 7.63 ms, 16 7.30, 32 7.22, 64 (all of it) 6.85. With 32 the loss is off by 1.5e-7 to 3e-7
// (FP32 throughout: 2.8e-7 to 9e-7).
constexpr int PROMOTE = 32;
// The same of the two gradient products: 1024 additions in the tensor core, which truncates, before a sum goes on in FP32 registers. (Over
// 131072 tokens at once the weight's gradient was off by 6.5e-4 of its terms, always towards zero, with this by 1e-4. The step of
// 8192 x 4096 x 131072, whose products over 32768 words take two chains, 23.3 instead of 23.1 ms.)
constexpr int PROMOTE_GRAD = 256;
// Tile rows that are walked together, so that a band's rows stay in L2 while the weight passes by once per band (8, 16, 32:
// 29987, 29527, 31442 us for a training step of 8192 x 4096 x 131072).
constexpr int BAND = 16;

enum Product { STATS, PROBS, GRAD_HIDDEN, GRAD_WEIGHT };

struct Params {
  int m, n, k;         // extents; the one that runs over tokens is the packed rows' number
  const int* count;    // packed rows
  const int* labels;   // [rows] target of a packed row, -1: none that exists
  const float* lse;    // [rows]
  const float* weights;  // [rows] gradient of a packed row's loss, up to `scale`
  const float* scale;
  const float* coef;   // [rows] weight * (p_target - 1)
  float2* partial;     // STATS: [2 * n_tiles][pitch] maximum and sum
  long long pitch;
  int kept;            // STATS: the words whose codes are stored, in whole tiles
  float* tops;         // STATS: [kept / HALF][pitch] what the codes count from
  int first_word;       // PROBS, GRAD_*: first word of the piece
  float* row_sums;      // PROBS: [2 * n_tiles][pitch] sums of what is stored
  const float* others;  // GRAD_HIDDEN: [rows] sum of a packed row's stored entries over all pieces
  const int* row_of;    // GRAD_HIDDEN: token of a packed row
  float* sums;          // GRAD_HIDDEN: [rows, n] FP32 sums over pieces, or NULL
  int add, last;        // GRAD_HIDDEN: sums holds earlier pieces; this piece is the last
  const __nv_bfloat16* head;  // GRAD_HIDDEN: the whole weight
  long long head_stride;
  __nv_bfloat16* out;         // GRAD_HIDDEN
  const int* slots;           // GRAD_WEIGHT: [vocab] row of word_sums, or -1
  const float* word_sums;     // GRAD_WEIGHT: [rows, n]
  float* part_sums;           // GRAD_HIDDEN: [parts][TILE][TILE] of the tiles that are cut
  int* failed;  // status words of this chain of launches
  int* status;  // the caller's, or NULL
};

// A wait that gave up is told to the chain, whose later launches answer with NaN, and to the caller.
__device__ __forceinline__ void give_up(int* failed, int* status, int role, int stage, int kb) {
  report_status(failed, HMC_STATUS_TIMEOUT_PIPELINE, role, stage, kb);
  report_status(status, HMC_STATUS_TIMEOUT_PIPELINE, role, stage, kb);
}
__device__ __forceinline__ bool has_failed(const int* failed, const int* status) {
  return __ldcg(failed) != 0 || (status != nullptr && __ldcg(status) != 0);
}
__device__ __forceinline__ float not_a_number() { return __int_as_float(0x7fffffff); }

// After a wait that gave up: the copies that are still on their way into shared memory, from this stage on. The leader's
// barriers count both CTAs' bytes, and the partner cannot leave before the leader. A stage that was never filled costs a tenth of a second.
__device__ __forceinline__ void await_copies(uint64_t* full_bar, int stages, int stage, uint32_t phase) {
  volatile int unused = 0;
  for (int s = 0; s < stages; ++s) {
    mbar_wait(&full_bar[stage], phase, &unused, 100ull * 1000 * 1000);
    unused = 0;
    if (++stage == stages) stage = 0, phase ^= 1u;
  }
}

// A unit of work: a tile and its range of k-blocks. Part -1 is the whole of it.
struct Unit {
  int mi, ni, part;
  int kb0, kb1;
};

// Tiles in bands of BAND tile rows, a band's columns one after the other. With `split`, the tiles that would leave pairs
// idle in the last wave are cut along k: into as many parts as shorten that wave most, counted with a hundredth of a tile's
// time per part for what they write, at most two parts per pair (512 x 1024 with k = 32000, 8 tiles for 74 pairs: 167 us whole, 35 +
// 8 us for joining them in 9 parts; 3687 x 4096 with k = 65536, 240 tiles: 1621 us whole, 1395 + 13).
struct Walker {
  int mt, nt, kiters, parts;
  long long whole, units;
  __device__ Walker(int m, int n, int k, int pairs, bool split)
      : mt((m + TILE - 1) / TILE), nt((n + TILE - 1) / TILE), kiters((k + BK - 1) / BK), parts(1) {
    const long long tiles = static_cast<long long>(mt) * nt;
    whole = tiles;
    if (split) {
      const int rest = static_cast<int>(tiles % pairs);
      float best = 1.0f;
      for (int s = 2; s <= MAX_PARTS && rest > 0 && rest * s <= 2 * pairs && s * MIN_PART <= kiters; ++s) {
        const float cost = static_cast<float>((rest * s + pairs - 1) / pairs) / static_cast<float>(s) + 0.01f * static_cast<float>(s);
        if (cost < best) best = cost, parts = s;
      }
      if (parts > 1) whole = tiles - rest;
    }
    units = whole + (tiles - whole) * parts;
  }
  __device__ void tile(long long idx, int& mi, int& ni) const {
    const long long per_band = static_cast<long long>(BAND) * nt;
    const int band = static_cast<int>(idx / per_band);
    const int local = static_cast<int>(idx - band * per_band);
    const int high = min(BAND, mt - band * BAND);
    mi = band * BAND + local % high;
    ni = local / high;
  }
  __device__ bool get(long long idx, Unit& u) const {
    if (idx >= units) return false;
    u.part = -1, u.kb0 = 0, u.kb1 = kiters;
    if (idx >= whole) {
      const int cut = static_cast<int>(idx - whole);
      u.part = cut % parts;
      u.kb0 = static_cast<int>(static_cast<long long>(kiters) * u.part / parts);
      u.kb1 = static_cast<int>(static_cast<long long>(kiters) * (u.part + 1) / parts);
      u.part = cut;  // where its sums go
      idx = whole + cut / parts;
    }
    tile(idx, u.mi, u.ni);
    return true;
  }
};

__device__ __forceinline__ float shifted_exp(float v, float top) { return __expf(v - top); }

// A kept logit: how far it is below the largest of its row's 128 columns, in steps of 2^-10 of a power of two. Rounding to
// a step is off by 2^-11 of one, 3.4e-4 of the probability, a twelfth of what BF16 adds afterwards. Codes end at 64 powers of two:
// what is further below, 5e-20 of the largest, is zero, as are the target's entry and the columns behind the vocabulary.
constexpr float CODE_STEPS = 1024.0f;
constexpr float LOG2_E = 1.44269504f;
constexpr float ROUND = 8388608.0f;  // 2^23: a sum with it is a whole number, in the low bits of the word
constexpr unsigned CODE_ZERO = 0xffff;

__device__ __forceinline__ uint32_t codes_of(float below0, float below1) {
  const float last = ROUND + static_cast<float>(CODE_ZERO);  // NaN too: its row's sum is NaN, which is enough
  const float a = fminf(__fmaf_rn(below0, -CODE_STEPS * LOG2_E, ROUND), last);
  const float b = fminf(__fmaf_rn(below1, -CODE_STEPS * LOG2_E, ROUND), last);
  return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x5410);
}

// 32 x 32 values of 16 bits leave as one box through shared memory; two boxes per warp in flight. A lane's row of values.
__device__ __forceinline__ void store_box(const CUtensorMap* tm, uint8_t* stage, unsigned& issued, const uint4 (&q)[4], int col,
                                          int row, int lane) {
  uint8_t* box = stage + (issued & 1) * (STORE_STAGE_BYTES / 2);
  if (issued > 1) {
    if (lane == 0) bulk_wait_read_but_one();
    __syncwarp();
  }
  uint8_t* base = box + lane * 64;  // 64-byte rows under the 64-byte swizzle
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(base + ((i ^ ((lane >> 1) & 3)) << 4)) = q[i];
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(tm, box, col, row);
    bulk_commit_group();
  }
  ++issued;
}
__device__ __forceinline__ void store_box(const CUtensorMap* tm, uint8_t* stage, unsigned& issued, const float* v, int col,
                                          int row, int lane) {
  uint4 q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    q[i] = make_uint4(pack_bf16x2(v[8 * i], v[8 * i + 1]), pack_bf16x2(v[8 * i + 2], v[8 * i + 3]),
                      pack_bf16x2(v[8 * i + 4], v[8 * i + 5]), pack_bf16x2(v[8 * i + 6], v[8 * i + 7]));
  store_box(tm, stage, issued, q, col, row, lane);
}

// Maximum and sum of exponentials of one row's 128 columns, without the target's; codes of the words that are kept.
// Two logits per instruction (f32x2) are slower here: 3687 x 65536 x 4096 1475 us against 1437.
__device__ __forceinline__ void epilogue_stats(const Params& p, const CUtensorMap* tm, uint8_t* stage, unsigned& issued,
                                               float (&v)[HALF], int first_row, int row, bool row_ok, int col, int half_tile,
                                               int lane) {
  const int label = row_ok ? p.labels[row] - col : -1;
  if (col + HALF > p.n) {
#pragma unroll
    for (int j = 0; j < HALF; ++j)
      if (col + j >= p.n) v[j] = -INFINITY;
  }
  if (label >= 0 && label < HALF) {
#pragma unroll
    for (int j = 0; j < HALF; ++j)
      if (j == label) v[j] = -INFINITY;
  }
  float high[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int j = 4; j < HALF; ++j) high[j & 3] = fmaxf(high[j & 3], v[j]);
  const float top = fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3]));
  const float shift = top == -INFINITY ? 0.0f : top;  // nothing but -inf: exp(-inf - 0), not exp(-inf + inf)
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < HALF; ++j) {
    v[j] -= shift;
    sum[j & 3] += __expf(v[j]);
  }
  if (row_ok) p.partial[half_tile * p.pitch + row] = make_float2(top, (sum[0] + sum[1]) + (sum[2] + sum[3]));
  if (col >= p.kept) return;
  if (row_ok) p.tops[half_tile * p.pitch + row] = top;
  __syncwarp();
#pragma unroll
  for (int c = 0; c < HALF; c += 32) {
    uint4 q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* b = v + c + 8 * i;
      q[i] = make_uint4(codes_of(b[0], b[1]), codes_of(b[2], b[3]),
                        codes_of(b[4], b[5]), codes_of(b[6], b[7]));
    }
    store_box(tm, stage, issued, q, col + c, first_row, lane);
  }
}

// What a chain of k-blocks left in the accumulator, added to the sums of those before it. A gradient has few such chains, long ones: the
// sums may live in local memory.
__device__ __forceinline__ void add_columns(uint32_t taddr, float* sums, bool first) {
#pragma unroll 1
  for (int c = 0; c < HALF; c += 32) {
    uint32_t raw[32];
    __syncwarp();
    tmem_ld_32x32(taddr + c, raw);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 32; ++j) sums[c + j] = (first ? 0.0f : sums[c + j]) + __uint_as_float(raw[j]);
  }
}

// 64 columns of the accumulator row of each lane: two loads under way at a time.
__device__ __forceinline__ void load_columns(uint32_t taddr, float (&v)[64]) {
  uint32_t lo[32], hi[32];
  __syncwarp();
  tmem_ld_32x32(taddr, lo);
  tmem_ld_32x32(taddr + 32, hi);
  tmem_ld_wait();
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(lo[j]), v[32 + j] = __uint_as_float(hi[j]);
}
// The same, or from sums of several chains.
__device__ __forceinline__ void load_columns(uint32_t taddr, const float* sums, int c, float (&v)[64]) {
  if (sums == nullptr) {
    load_columns(taddr + c, v);
    return;
  }
#pragma unroll
  for (int j = 0; j < 64; ++j) v[j] = sums[c + j];
}

// Eight values as BF16; their sum as rounded.
__device__ __forceinline__ uint4 pack_8(const float* v, float2& sum) {
  const uint4 q = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  sum = add2(sum, add2(add2(unpack_bf16x2(q.x), unpack_bf16x2(q.y)), add2(unpack_bf16x2(q.z), unpack_bf16x2(q.w))));
  return q;
}

// p of one row's 128 columns times the row's gradient, the target's entry left out, and the sum of what is stored.
__device__ __forceinline__ void epilogue_probs(const Params& p, const CUtensorMap* tm, uint32_t taddr, uint8_t* stage,
                                               unsigned& issued, int first_row, int row, bool row_ok, int col, int half_tile,
                                               int lane) {
  float2 sum = both(0.0f);
  const float lse = row_ok ? p.lse[row] : 0.0f;
  const float weight = row_ok ? p.weights[row] : 0.0f;
  const int label = row_ok ? p.labels[row] - p.first_word - col : -1;
#pragma unroll 1
  for (int c = 0; c < HALF; c += 64) {
    if (col + c >= p.n) break;
    float v[64];
    load_columns(taddr + c, v);
#pragma unroll
    for (int j = 0; j < 64; ++j) v[j] = row_ok ? shifted_exp(v[j], lse) * weight : 0.0f;
    const int own = label - c;
    if (own >= 0 && own < 64) {
#pragma unroll
      for (int j = 0; j < 64; ++j)
        if (j == own) v[j] = 0.0f;
    }
    if (col + c + 64 > p.n) {  // columns behind the piece are neither stored nor summed
#pragma unroll
      for (int j = 0; j < 64; ++j)
        if (col + c + j >= p.n) v[j] = 0.0f;
    }
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 64; h += 32) {
      if (col + c + h >= p.n) break;
      uint4 q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = pack_8(v + h + 8 * i, sum);
      store_box(tm, stage, issued, q, col + c + h, first_row, lane);
    }
  }
  if (row_ok) p.row_sums[half_tile * p.pitch + row] = sum.x + sum.y;
}

// With the last piece: what a row of dx takes the target's row times, and what the whole is scaled by.
__device__ __forceinline__ float2 row_coefficients(const Params& p, int row) {
  const float coef = p.coef[row], others = p.others[row], scale = has_failed(p.failed, p.status) ? not_a_number() : *p.scale;
  // nothing stored (a gradient of zero, no other word, a certain token): the true coefficient, which is as small
  return others != 0.0f ? make_float2(-others, scale * (-coef / others)) : make_float2(coef, scale);
}

// Eight columns of a row of dx from this piece's sums: added to those of earlier pieces, and with the last piece the target's
// row on top, scaled, rounded and stored at the token's place.
__device__ __forceinline__ void finish_grad_hidden(const Params& p, int row, int col, float* v, float2 by) {
  float* sums = p.sums + static_cast<long long>(row) * p.n + col;
  if (p.add) {
    const float4 a = *reinterpret_cast<const float4*>(sums), b = *reinterpret_cast<const float4*>(sums + 4);
    v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w, v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
  }
  if (!p.last) {
    *reinterpret_cast<float4*>(sums) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(sums + 4) = make_float4(v[4], v[5], v[6], v[7]);
    return;
  }
  const int label = p.labels[row];
  if (label >= 0) {
    const uint4 w = ld_16(p.head + label * p.head_stride + col);
    const uint32_t parts[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack_bf16x2(parts[e]);
      v[2 * e] += by.x * f.x;
      v[2 * e + 1] += by.x * f.y;
    }
  }
  const float scale = by.y;
  st_16(p.out + static_cast<long long>(p.row_of[row]) * p.n + col,
        make_uint4(pack_bf16x2(v[0] * scale, v[1] * scale), pack_bf16x2(v[2] * scale, v[3] * scale),
                   pack_bf16x2(v[4] * scale, v[5] * scale), pack_bf16x2(v[6] * scale, v[7] * scale)));
}

// lost: nothing is in the accumulator.
__device__ __forceinline__ void epilogue_grad_hidden(const Params& p, uint32_t taddr, const float* sums, int row, bool row_ok, int col,
                                                     bool lost) {
  const float2 by = row_ok && p.last ? row_coefficients(p, row) : both(0.0f);
#pragma unroll 1
  for (int c = 0; c < HALF; c += 64) {
    if (col + c >= p.n) break;
    float v[64];
    if (lost) {
#pragma unroll
      for (int j = 0; j < 64; ++j) v[j] = not_a_number();
    } else {
      load_columns(taddr, sums, c, v);
    }
    if (row_ok) {
#pragma unroll
      for (int j = 0; j < 64; j += 8)
        if (col + c + j < p.n) finish_grad_hidden(p, row, col + c + j, v + j, by);
    }
  }
}

// A part of a tile that is cut along k: its sums as they are.
__device__ __forceinline__ void epilogue_part(const Params& p, uint32_t taddr, const float* sums, int part, int row_in_tile, bool row_ok,
                                              int half) {
  float* dst = p.part_sums + (static_cast<long long>(part) * TILE + row_in_tile) * TILE + half * HALF;
#pragma unroll 1
  for (int c = 0; c < HALF; c += 64) {
    float v[64];
    load_columns(taddr, sums, c, v);
    if (row_ok) {
#pragma unroll
      for (int j = 0; j < 64; j += 4) *reinterpret_cast<float4*>(dst + c + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    }
  }
}

// The tiles that were cut: their parts in order, eight columns per thread, eight rows per block.
__global__ void __launch_bounds__(256) join_parts_kernel(Params p, int pairs) {
  chain_wait();
  chain_next();
  p.m = *p.count;
  const Walker walker(p.m, p.n, p.k, pairs, true);
  const long long tile = walker.whole + blockIdx.y;
  if (walker.parts == 1 || tile >= static_cast<long long>(walker.mt) * walker.nt) return;
  int mi, ni;
  walker.tile(tile, mi, ni);
  const int in_tile = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int row = mi * TILE + in_tile, col = ni * TILE + (threadIdx.x & 31) * 8;
  if (row >= p.m || col >= p.n) return;
  const float* src = p.part_sums + ((static_cast<long long>(blockIdx.y) * walker.parts * TILE + in_tile) * TILE) + (threadIdx.x & 31) * 8;
  float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int s = 0; s < walker.parts; ++s) {
    const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
    v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w, v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
    src += TILE * TILE;
  }
  finish_grad_hidden(p, row, col, v, p.last ? row_coefficients(p, row) : both(0.0f));
}

__device__ __forceinline__ void epilogue_grad_weight(const Params& p, const CUtensorMap* tm, uint32_t taddr, const float* sums,
                                                     uint8_t* stage, unsigned& issued, int first_row, int row, bool row_ok, int col, int lane,
                                                     bool empty, float filler) {
  const float scale = has_failed(p.failed, p.status) ? not_a_number() : *p.scale;
  const int slot = row_ok ? p.slots[p.first_word + row] : -1;
  const float* more = p.word_sums + static_cast<long long>(slot >= 0 ? slot : 0) * p.n + col;
#pragma unroll 1
  for (int c = 0; c < HALF; c += 64) {
    if (col + c >= p.n) break;
    float v[64];
    if (empty) {
#pragma unroll
      for (int j = 0; j < 64; ++j) v[j] = filler;
    } else {
      load_columns(taddr, sums, c, v);
      if (slot >= 0) {
#pragma unroll
        for (int j = 0; j < 64; j += 4)
          if (col + c + j < p.n) {
            const float4 a = *reinterpret_cast<const float4*>(more + c + j);
            v[j] += a.x, v[j + 1] += a.y, v[j + 2] += a.z, v[j + 3] += a.w;
          }
      }
#pragma unroll
      for (int j = 0; j < 64; ++j) v[j] *= scale;
    }
    __syncwarp();
#pragma unroll
    for (int h = 0; h < 64; h += 32)
      if (col + c + h < p.n) store_box(tm, stage, issued, v + h, col + c + h, first_row, lane);
  }
}

template <Product KIND>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NUM_THREADS, 1)
head_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                 const __grid_constant__ CUtensorMap tm_c, Params p) {
  constexpr int A_MAJOR = KIND == GRAD_WEIGHT ? HMC_MAJOR_MN : HMC_MAJOR_K;
  constexpr int B_MAJOR = KIND == GRAD_WEIGHT || KIND == GRAD_HIDDEN ? HMC_MAJOR_MN : HMC_MAJOR_K;
  constexpr int CHAIN = KIND == STATS ? PROMOTE : PROMOTE_GRAD;  // not PROBS
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* store_stage = smem + STAGES * STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(store_stage + EPI_WARPS * STORE_STAGE_BYTES);
  uint64_t* full_bar = bars;                               // leader only: the loads of both CTAs
  uint64_t* empty_bar = bars + STAGES;                     // one set per CTA
  uint64_t* acc_full_bar = bars + 2 * STAGES;              // one set per CTA
  uint64_t* acc_empty_bar = acc_full_bar + ACC_STAGES;     // leader only
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty_bar + ACC_STAGES);
  volatile int* abort_word = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();  // 0 = leader
  const long long pair = blockIdx.x >> 1;
  const long long pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int s = 0; s < ACC_STAGES; ++s) {
      mbar_init(&acc_full_bar[s], 1);
      mbar_init(&acc_empty_bar[s], 2 * EPI_WARPS);  // every epilogue warp of both CTAs
    }
    *abort_word = 0;
    mbar_fence_init();
    prefetch_tensormap(&tm_a);
    prefetch_tensormap(&tm_b);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before any cross-CTA signal
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  chain_wait();
  chain_next();

  const int count = *p.count;
  if (KIND == GRAD_WEIGHT) p.k = count;
  else p.m = count;
  const Walker walker(p.m, p.n, p.k, static_cast<int>(pairs), KIND == GRAD_HIDDEN);
  const int kiters = walker.kiters;
  Unit u;

  if (warp == 0) {
    // ======================================================================== TMA producer (both CTAs)
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (long long idx = pair; ok && walker.get(idx, u); idx += pairs) {
        const int m0 = u.mi * TILE + static_cast<int>(rank) * HALF;
        const int n0 = u.ni * TILE + static_cast<int>(rank) * HALF;
        for (int kb = u.kb0; kb < u.kb1; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1u, abort_word, PIPE_BUDGET_NS)) {
            give_up(p.failed, p.status, 0, stage, kb);
            ok = false;
            break;
          }
          uint8_t* a_dst = smem + stage * STAGE_BYTES;
          uint8_t* b_dst = a_dst + A_TILE_BYTES;
          // the leader's barrier counts the bytes of both CTAs
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * STAGE_BYTES);
          if (A_MAJOR == HMC_MAJOR_K) {
            tma_load_2d_pair(a_dst, &tm_a, &full_bar[stage], kb * BK, m0);
          } else {
            tma_load_2d_pair(a_dst, &tm_a, &full_bar[stage], m0, kb * BK);
            tma_load_2d_pair(a_dst + CHUNK_BYTES, &tm_a, &full_bar[stage], m0 + 64, kb * BK);
          }
          if (B_MAJOR == HMC_MAJOR_K) {
            tma_load_2d_pair(b_dst, &tm_b, &full_bar[stage], kb * BK, n0);
          } else {
            tma_load_2d_pair(b_dst, &tm_b, &full_bar[stage], n0, kb * BK);
            tma_load_2d_pair(b_dst + CHUNK_BYTES, &tm_b, &full_bar[stage], n0 + 64, kb * BK);
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ======================================================================== MMA issuer (leader only)
    if (rank == 0 && kiters > 0) {
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      constexpr uint32_t idesc = make_idesc_f32acc(1u, TILE, TILE, A_MAJOR, B_MAJOR);
      constexpr uint32_t A_LBO = A_MAJOR == HMC_MAJOR_MN ? CHUNK_BYTES : 16;
      constexpr uint32_t B_LBO = B_MAJOR == HMC_MAJOR_MN ? CHUNK_BYTES : 16;
      constexpr uint32_t A_KSTEP = A_MAJOR == HMC_MAJOR_MN ? (16 * 128) >> 4 : 32 >> 4;
      constexpr uint32_t B_KSTEP = B_MAJOR == HMC_MAJOR_MN ? (16 * 128) >> 4 : 32 >> 4;
      for (long long idx = pair; ok && walker.get(idx, u); idx += pairs) {
        // one accumulator per unit, or per CHAIN k-blocks of it
        for (int first = u.kb0; ok && first < u.kb1; first += KIND == PROBS ? u.kb1 - u.kb0 : CHAIN) {
          const int end = KIND == PROBS ? u.kb1 : min(u.kb1, first + CHAIN);
          if (!mbar_wait(&acc_empty_bar[acc], acc_phase ^ 1u, abort_word, PIPE_BUDGET_NS)) {
            if (lane == 0) give_up(p.failed, p.status, 1, acc, 0);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(acc * TILE);
          for (int kb = first; kb < end; ++kb) {
            if (!mbar_wait(&full_bar[stage], phase, abort_word, PIPE_BUDGET_NS)) {
              if (lane == 0) give_up(p.failed, p.status, 2, stage, kb);
              ok = false;
              break;
            }
            tc_fence_after_sync();
            if (lane == 0) {
              uint8_t* a_src = smem + stage * STAGE_BYTES;
              uint64_t da = make_smem_desc(smem_u32(a_src), A_LBO, 1024, SWIZZLE_128B);
              uint64_t db = make_smem_desc(smem_u32(a_src + A_TILE_BYTES), B_LBO, 1024, SWIZZLE_128B);
#pragma unroll
              for (int ks = 0; ks < BK / 16; ++ks) {
                umma_bf16_pair(tmem_d, da, db, idesc, (kb > first || ks > 0) ? 1u : 0u);
                da += A_KSTEP;
                db += B_KSTEP;
              }
              umma_commit_pair(&empty_bar[stage]);  // frees the slot in both CTAs
              if (kb == end - 1) umma_commit_pair(&acc_full_bar[acc]);
            }
            __syncwarp();
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (++acc == ACC_STAGES) {
            acc = 0;
            acc_phase ^= 1u;
          }
        }
      }
      if (!ok) await_copies(full_bar, STAGES, stage, phase);
    }
  } else {
    // ======================================================================== epilogue (both CTAs)
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    const int quarter = warp & 3;      // TMEM lane quarter this warp may read
    const int half = (warp - 2) >> 2;  // which half of the tile's columns this warp handles
    uint8_t* my_stage = store_stage + (warp - 2) * STORE_STAGE_BYTES;
    unsigned issued = 0;
    const uint32_t leader_acc_empty = map_to_cta(smem_u32(acc_empty_bar), 0);
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(half * HALF);
    auto filled = [&]() {  // the next accumulator, once its MMAs are done
      if (!mbar_wait(&acc_full_bar[acc], acc_phase, abort_word, PIPE_BUDGET_NS)) {
        if (lane == 0) give_up(p.failed, p.status, 3, acc, 0);
        ok = false;
      }
      tc_fence_after_sync();
      return ok;
    };
    auto release = [&]() {  // the issuer lives in the leader: its barrier from either CTA
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(leader_acc_empty + static_cast<uint32_t>(acc) * 8u);
      if (++acc == ACC_STAGES) {
        acc = 0;
        acc_phase ^= 1u;
      }
    };
    // a gradient's tiles that are lost to a wait that gave up are filled with NaN
    for (long long idx = pair; (ok || KIND == GRAD_HIDDEN || KIND == GRAD_WEIGHT) && walker.get(idx, u); idx += pairs) {
      const int in_tile = static_cast<int>(rank) * HALF + quarter * 32;
      const int first_row = u.mi * TILE + in_tile;
      const int row = first_row + lane;
      const bool row_ok = row < p.m;
      const int col = u.ni * TILE + half * HALF;
      if (kiters == 0) {  // no token counts: the weight's gradient is zero
        if (KIND == GRAD_WEIGHT) epilogue_grad_weight(p, &tm_c, 0, nullptr, my_stage, issued, first_row, row, row_ok, col, lane, true, 0.0f);
        continue;
      }
      if (KIND == STATS) {
        // The tensor core's sums lose about half a step per addition, always towards zero, so PROMOTE k-blocks at a time are
        // added up in FP32 registers. Reading an accumulator holds up the MMAs into the other one for about 250 cycles.
        float v[HALF];
#pragma unroll
        for (int j = 0; j < HALF; ++j) v[j] = 0.0f;
        for (int first = 0; first < kiters; first += CHAIN) {
          if (!filled()) break;
          const uint32_t taddr = lane_base + static_cast<uint32_t>(acc * TILE);
#pragma unroll
          for (int c = 0; c < HALF; c += 32) {
            uint32_t raw[32];
            tmem_ld_32x32(taddr + c, raw);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) v[c + j] += __uint_as_float(raw[j]);
          }
          release();
        }
        if (ok) epilogue_stats(p, &tm_c, my_stage, issued, v, first_row, row, row_ok, col, 2 * u.ni + half, lane);
        __syncwarp();
        continue;
      }
      float chains[HALF];
      const float* sums = nullptr;
      if (KIND != PROBS && u.kb1 - u.kb0 > CHAIN) {  // all chains but the last
        sums = chains;
        for (int first = u.kb0; ok && first + CHAIN < u.kb1; first += CHAIN) {
          if (!filled()) break;
          add_columns(lane_base + static_cast<uint32_t>(acc * TILE), chains, first == u.kb0);
          release();
        }
      }
      if (!ok || !filled()) {
        // of a tile that is cut, the launch that joins its parts writes NaN
        if (KIND == GRAD_HIDDEN && u.part < 0) epilogue_grad_hidden(p, 0, nullptr, row, row_ok, col, true);
        if (KIND == GRAD_WEIGHT)
          epilogue_grad_weight(p, &tm_c, 0, nullptr, my_stage, issued, first_row, row, row_ok, col, lane, true, not_a_number());
        continue;
      }
      const uint32_t taddr = lane_base + static_cast<uint32_t>(acc * TILE);
      if (sums != nullptr) add_columns(taddr, chains, false);
      if (KIND == PROBS) epilogue_probs(p, &tm_c, taddr, my_stage, issued, first_row, row, row_ok, col, 2 * u.ni + half, lane);
      if (KIND == GRAD_HIDDEN) {
        if (u.part >= 0) epilogue_part(p, taddr, sums, u.part, in_tile + lane, row_ok, half);
        else epilogue_grad_hidden(p, taddr, sums, row, row_ok, col, false);
      }
      if (KIND == GRAD_WEIGHT)
        epilogue_grad_weight(p, &tm_c, taddr, sums, my_stage, issued, first_row, row, row_ok, col, lane, false, 0.0f);
      release();
    }
    if (issued > 0 && lane == 0) bulk_wait_all();  // this thread's stores are in global memory
  }

  // Teardown: no CTA may leave while its partner can still reach into its shared memory or TMEM.
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------------------- few tokens
// Up to 128 tokens: the weight's rows take the M side of the tile and the tokens N = 32, 64 or 128 columns, so that the tensor
// cores do a fraction of a 256 x 256 tile's work beside the one pass over the weight, which is the bound: 16 tokens of 4096 over
// 131072 words 171 us (1.07 GB, 6.3 TB/s; on 256 x 256 tiles 182 to 198). Whole calls of 128 tokens take 206 us this way, of 129 the
// other way 236. An accumulator row is a word: the sums over words run across the lanes of a warp.
template <int N>
struct Few {
  static constexpr int B_BYTES = N / 2 * 128;                  // tokens' k-block that a CTA loads
  static constexpr int STAGE = A_TILE_BYTES + B_BYTES;
  static constexpr int STAGES = N == 32 ? 12 : N == 64 ? 10 : 8;
  static constexpr int SMEM = STAGES * STAGE + 1024 + 512;
  static constexpr int WARPS = N == 32 ? 4 : 8;                // epilogue: 32 columns at least per warp
  static constexpr int COLS = N * 4 / WARPS;                   // columns per warp
  static constexpr int THREADS = 64 + 32 * WARPS;
};

// The reduction over a warp's lanes of each of C columns (halving: a lane hands half of its columns to its partner and
// takes the partner's values of the other half); column lane * (C / 32) + i ends in out[i].
template <int C, bool MAX>
__device__ __forceinline__ void reduce_columns(const float (&v)[C], float (&out)[C / 32], int lane) {
  float w[C];
#pragma unroll
  for (int i = 0; i < C; ++i) w[i] = v[i];
#pragma unroll
  for (int s = 0; s < 5; ++s) {
    const int half = C >> (s + 1);
    const bool upper = (lane & (16 >> s)) != 0;
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float keep = upper ? w[i + half] : w[i], send = upper ? w[i] : w[i + half];
      const float other = __shfl_xor_sync(0xffffffffu, send, 16 >> s);
      w[i] = MAX ? fmaxf(keep, other) : keep + other;
    }
  }
#pragma unroll
  for (int i = 0; i < C / 32; ++i) out[i] = w[i];
}

template <int N>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Few<N>::THREADS, 1)
few_tokens_kernel(const __grid_constant__ CUtensorMap tm_words, const __grid_constant__ CUtensorMap tm_tokens, int vocab, int kiters,
                  const int* __restrict__ count, const int* __restrict__ labels, float2* __restrict__ partial, long long pitch,
                  int* failed, int* status) {
  using F = Few<N>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + F::STAGES * F::STAGE);
  uint64_t* full_bar = bars;                             // leader only: the loads of both CTAs
  uint64_t* empty_bar = bars + F::STAGES;                // one set per CTA
  uint64_t* acc_full_bar = bars + 2 * F::STAGES;         // one set per CTA
  uint64_t* acc_empty_bar = acc_full_bar + ACC_STAGES;   // leader only
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty_bar + ACC_STAGES);
  volatile int* abort_word = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = (vocab + TILE - 1) / TILE;
  if (threadIdx.x == 0) {
    for (int s = 0; s < F::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int s = 0; s < ACC_STAGES; ++s) {
      mbar_init(&acc_full_bar[s], 1);
      mbar_init(&acc_empty_bar[s], 2 * F::WARPS);  // every epilogue warp of both CTAs
    }
    *abort_word = 0;
    mbar_fence_init();
    prefetch_tensormap(&tm_words);
    prefetch_tensormap(&tm_tokens);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers exist before any cross-CTA signal
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  if (warp != 0) chain_wait();
  chain_next();

  if (warp == 0) {
    // ======================================================================== TMA producer (both CTAs)
    // The weight was there before the packing pass began (which starts this launch early only once it has waited for what
    // came before it): its first pieces are on their way before the tokens are packed.
    if (lane == 0) {
      const int first = pair * TILE + static_cast<int>(rank) * HALF, early = pair < tiles ? min(F::STAGES, kiters) : 0;
      for (int kb = 0; kb < early; ++kb) {
        if (rank == 0) mbar_arrive_expect_tx(&full_bar[kb], 2 * F::STAGE);
        tma_load_2d_pair(smem + kb * F::STAGE, &tm_words, &full_bar[kb], kb * BK, first);
      }
      chain_wait();
      for (int kb = 0; kb < early; ++kb)
        tma_load_2d_pair(smem + kb * F::STAGE + A_TILE_BYTES, &tm_tokens, &full_bar[kb], kb * BK, static_cast<int>(rank) * (N / 2));
      int stage = early % F::STAGES;
      uint32_t phase = early == F::STAGES ? 1 : 0;
      bool ok = true;
      for (int t = pair; ok && t < tiles; t += pairs) {
        const int word = t * TILE + static_cast<int>(rank) * HALF;
        for (int kb = t == pair ? early : 0; kb < kiters; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1u, abort_word, PIPE_BUDGET_NS)) {
            give_up(failed, status, 0, stage, kb);
            ok = false;
            break;
          }
          uint8_t* a_dst = smem + stage * F::STAGE;
          // the leader's barrier counts the bytes of both CTAs
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * F::STAGE);
          tma_load_2d_pair(a_dst, &tm_words, &full_bar[stage], kb * BK, word);
          tma_load_2d_pair(a_dst + A_TILE_BYTES, &tm_tokens, &full_bar[stage], kb * BK, static_cast<int>(rank) * (N / 2));
          if (++stage == F::STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ======================================================================== MMA issuer (leader only)
    if (rank == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      constexpr uint32_t idesc = make_idesc_f32acc(1u, TILE, N, HMC_MAJOR_K, HMC_MAJOR_K);
      for (int t = pair; ok && t < tiles; t += pairs) {
        for (int first = 0; ok && first < kiters; first += PROMOTE) {
          const int end = min(kiters, first + PROMOTE);
          if (!mbar_wait(&acc_empty_bar[acc], acc_phase ^ 1u, abort_word, PIPE_BUDGET_NS)) {
            if (lane == 0) give_up(failed, status, 1, acc, 0);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          for (int kb = first; kb < end; ++kb) {
            if (!mbar_wait(&full_bar[stage], phase, abort_word, PIPE_BUDGET_NS)) {
              if (lane == 0) give_up(failed, status, 2, stage, kb);
              ok = false;
              break;
            }
            tc_fence_after_sync();
            if (lane == 0) {
              uint8_t* a_src = smem + stage * F::STAGE;
              uint64_t da = make_smem_desc(smem_u32(a_src), 16, 1024, SWIZZLE_128B);
              uint64_t db = make_smem_desc(smem_u32(a_src + A_TILE_BYTES), 16, 1024, SWIZZLE_128B);
#pragma unroll
              for (int ks = 0; ks < BK / 16; ++ks) {
                umma_bf16_pair(tmem_base + static_cast<uint32_t>(acc * N), da, db, idesc, (kb > first || ks > 0) ? 1u : 0u);
                da += 32 >> 4;
                db += 32 >> 4;
              }
              umma_commit_pair(&empty_bar[stage]);  // frees the slot in both CTAs
              if (kb == end - 1) umma_commit_pair(&acc_full_bar[acc]);
            }
            __syncwarp();
            if (++stage == F::STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (++acc == ACC_STAGES) {
            acc = 0;
            acc_phase ^= 1u;
          }
        }
      }
      if (!ok) await_copies(full_bar, F::STAGES, stage, phase);
    }
  } else {
    // ======================================================================== epilogue (both CTAs)
    constexpr int C = F::COLS, OWN = C / 32;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    const int quarter = warp & 3;
    const int col = (warp - 2) / 4 * C;  // this warp's first token
    const uint32_t leader_acc_empty = map_to_cta(smem_u32(acc_empty_bar), 0);
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(col);
    const int rows = *count;
    float top[OWN], sum[OWN];  // of column lane * OWN + i over this warp's words so far
    int label[OWN];
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      top[i] = -INFINITY, sum[i] = 0.0f;
      const int token = col + lane * OWN + i;
      label[i] = token < rows ? labels[token] : -1;
    }
    for (int t = pair; ok && t < tiles; t += pairs) {
      float v[C];
#pragma unroll
      for (int j = 0; j < C; ++j) v[j] = 0.0f;
      for (int first = 0; first < kiters; first += PROMOTE) {
        if (!mbar_wait(&acc_full_bar[acc], acc_phase, abort_word, PIPE_BUDGET_NS)) {
          if (lane == 0) give_up(failed, status, 3, acc, 0);
          ok = false;
          break;
        }
        tc_fence_after_sync();
#pragma unroll
        for (int c = 0; c < C; c += 32) {
          uint32_t raw[32];
          tmem_ld_32x32(lane_base + static_cast<uint32_t>(acc * N + c), raw);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[c + j] += __uint_as_float(raw[j]);
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(leader_acc_empty + static_cast<uint32_t>(acc) * 8u);
        if (++acc == ACC_STAGES) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      if (!ok) break;
      const int word = t * TILE + static_cast<int>(rank) * HALF + quarter * 32 + lane;
#pragma unroll
      for (int j = 0; j < C; ++j) {
        if (word >= vocab) v[j] = -INFINITY;
        if (__shfl_sync(0xffffffffu, label[j % OWN], j / OWN) == word) v[j] = -INFINITY;  // the target is joined in FP32
      }
      float high[OWN], part[OWN];
      reduce_columns<C, true>(v, high, lane);
#pragma unroll
      for (int i = 0; i < OWN; ++i) high[i] = fmaxf(high[i], top[i]);
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const float most = __shfl_sync(0xffffffffu, high[j % OWN], j / OWN);
        v[j] = shifted_exp(v[j], most == -INFINITY ? 0.0f : most);
      }
      reduce_columns<C, false>(v, part, lane);
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        sum[i] = sum[i] * shifted_exp(top[i], high[i] == -INFINITY ? 0.0f : high[i]) + part[i];
        top[i] = high[i];
      }
    }
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int token = col + lane * OWN + i;
      if (token < rows) partial[(static_cast<long long>(blockIdx.x) * 4 + quarter) * pitch + token] = make_float2(top[i], sum[i]);
    }
  }

  // Teardown: no CTA may leave while its partner can still reach into its shared memory or TMEM.
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------------------- packing
constexpr int PACK_TOKENS = 8;  // tokens per block, one per warp
constexpr int PACK_THREADS = 256;

struct Targets {
  const void* data;
  int wide;  // INT64
  long long ignored, vocab;
  __device__ long long at(long long i) const {
    return wide ? static_cast<const long long*>(data)[i] : static_cast<const int*>(data)[i];
  }
};

__device__ __forceinline__ int block_count(int v) {  // sum over the block, in every thread
  __shared__ int slots[PACK_THREADS / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < PACK_THREADS / 32; ++w) v += slots[w];
  __syncthreads();
  return v;
}

// The tokens that count, in their order, as rows without gaps, and the logit of each one's target by FP32 multiply-adds: it
// enters the loss with its whole weight, where an error of the tensor core's sums would show. A block finds its place by
// counting the targets before its own; the last one writes the number of rows and clears the rows up to the next k-block of
// a contraction over them. Bound by latency (8192 x 4096: 50 us for 200 MB with the targets' rows; 5 us for 16 tokens).
__global__ void __launch_bounds__(PACK_THREADS) pack_rows_kernel(const __nv_bfloat16* __restrict__ x, long long x_stride,
                                                                 Targets targets, long long tokens, int hidden, int vector,
                                                                 int* __restrict__ count, int* __restrict__ done, int* __restrict__ failed,
                                                                 int* __restrict__ position,
                                                                 int* __restrict__ row_of, int* __restrict__ labels,
                                                                 __nv_bfloat16* __restrict__ packed,
                                                                 const __nv_bfloat16* __restrict__ head, long long head_stride,
                                                                 float* __restrict__ target_logit,
                                                                 float* __restrict__ token_loss) {
  __shared__ int place[PACK_TOKENS], known[PACK_TOKENS];  // packed row and target of a token, -1: none
  chain_wait();
  chain_next();
  const long long first = static_cast<long long>(blockIdx.x) * PACK_TOKENS;
  int before = 0;
  for (long long i = threadIdx.x; i < first; i += PACK_THREADS) before += targets.at(i) != targets.ignored;
  before = block_count(before);
  if (threadIdx.x < 32) {
    const long long i = threadIdx.x < PACK_TOKENS ? first + threadIdx.x : tokens;
    const long long target = i < tokens ? targets.at(i) : targets.ignored;
    const bool counts = i < tokens && target != targets.ignored;
    const unsigned mask = __ballot_sync(0xffffffffu, counts);
    const int at = before + __popc(mask & ((1u << threadIdx.x) - 1u));
    const int label = counts && target >= 0 && target < targets.vocab ? static_cast<int>(target) : -1;
    if (threadIdx.x < PACK_TOKENS) place[threadIdx.x] = counts ? at : -1, known[threadIdx.x] = label;
    if (i < tokens) position[i] = counts ? at : -1;
    if (counts) {
      row_of[at] = static_cast<int>(i);
      labels[at] = label;
    } else if (i < tokens && token_loss != nullptr) {
      token_loss[i] = 0.0f;
    }
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (place[warp] >= 0) {
    const __nv_bfloat16* src = x + (first + warp) * x_stride;
    __nv_bfloat16* dst = packed + static_cast<long long>(place[warp]) * hidden;
    const __nv_bfloat16* word = known[warp] >= 0 ? head + known[warp] * head_stride : nullptr;
    float2 dot = make_float2(0.0f, 0.0f);
#pragma unroll 4
    for (int c = lane * 8; c < hidden; c += 256) {
      uint4 q;
      if (vector) {
        q = ld_nc_16(src + c);
      } else {
        const uint16_t* bits = reinterpret_cast<const uint16_t*>(src + c);
        q.x = bits[0] | static_cast<uint32_t>(bits[1]) << 16, q.y = bits[2] | static_cast<uint32_t>(bits[3]) << 16;
        q.z = bits[4] | static_cast<uint32_t>(bits[5]) << 16, q.w = bits[6] | static_cast<uint32_t>(bits[7]) << 16;
      }
      st_16(dst + c, q);
      if (word != nullptr) {
        const uint4 w = ld_nc_16(word + c);
        dot = fma2(unpack_bf16x2(q.x), unpack_bf16x2(w.x), dot);
        dot = fma2(unpack_bf16x2(q.y), unpack_bf16x2(w.y), dot);
        dot = fma2(unpack_bf16x2(q.z), unpack_bf16x2(w.z), dot);
        dot = fma2(unpack_bf16x2(q.w), unpack_bf16x2(w.w), dot);
      }
    }
    const float logit = warp_sum(dot.x + dot.y);
    if (lane == 0) target_logit[place[warp]] = logit;
  }
  if (blockIdx.x != gridDim.x - 1) return;
  int rows = 0;
  for (int t = 0; t < PACK_TOKENS; ++t) rows += place[t] >= 0;
  rows += before;
  if (threadIdx.x == 0) *count = rows, *done = 0;
  if (threadIdx.x < HMC_STATUS_WORDS) failed[threadIdx.x] = 0;
  const long long end = min(tokens, static_cast<long long>((rows + BK - 1) / BK) * BK);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (long long c = rows * static_cast<long long>(hidden) + threadIdx.x * 8; c < end * hidden; c += PACK_THREADS * 8)
    st_16(packed + c, zero);
}

// ------------------------------------------------------------------------------------------- joining
constexpr int JOIN_SLICES = 32;

// Maximum and sum of a packed row from its parts, 32 rows per block: every slice its share of the parts in their order,
// then the slices in theirs. The block that finishes last adds up the losses, in an order of its own and in FP64, since a
// thread's share may be long; `done`, which the packing pass has cleared, tells it.
__global__ void __launch_bounds__(32 * JOIN_SLICES) join_kernel(const float2* __restrict__ partial, long long pitch, int parts,
                                                                const int* __restrict__ count,
                                                                const int* __restrict__ labels,
                                                                const int* __restrict__ row_of,
                                                                const float* __restrict__ target_logit,
                                                                float* __restrict__ lse, float* losses, int reduction,
                                                                int* __restrict__ done, int* failed, const int* status,
                                                                float* __restrict__ loss_out) {
  __shared__ float2 sums[JOIN_SLICES][33];
  chain_wait();
  chain_next();
  const bool lost = has_failed(failed, status);
  if (lost && blockIdx.x == 0 && threadIdx.x == 0 && threadIdx.y == 0) *failed = HMC_STATUS_TIMEOUT_PIPELINE;  // for the gradient
  const int row = blockIdx.x * 32 + threadIdx.x;
  const int rows = *count;
  const bool ok = row < rows;
  float top = -INFINITY, sum = 0.0f;
  if (ok) {
    constexpr int AHEAD = 4;  // parts loaded together
    for (int i = threadIdx.y; i < parts; i += AHEAD * JOIN_SLICES) {
      float2 part[AHEAD];
#pragma unroll
      for (int a = 0; a < AHEAD; ++a)
        part[a] = i + a * JOIN_SLICES < parts ? partial[(i + a * JOIN_SLICES) * pitch + row] : make_float2(-INFINITY, 0.0f);
      float high = top;
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) high = fmaxf(high, part[a].x);
      const float shift = high == -INFINITY ? 0.0f : high;
      sum *= shifted_exp(top, shift);
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) sum += part[a].y * shifted_exp(part[a].x, shift);
      top = high;
    }
  }
  sums[threadIdx.y][threadIdx.x] = make_float2(top, sum);
  __syncthreads();
  if (threadIdx.y == 0 && ok) {
    for (int s = 1; s < JOIN_SLICES; ++s) top = fmaxf(top, sums[s][threadIdx.x].x);
    // the target's logit joins the others here: loss = log(1 + sum over the others exp(l_j - l_target))
    const float own = target_logit[row], shift = fmaxf(top, own);
    sum = 0.0f;
    for (int s = 0; s < JOIN_SLICES; ++s) sum += sums[s][threadIdx.x].y * shifted_exp(sums[s][threadIdx.x].x, shift);
    const float log_sum = own >= top ? log1pf(sum) : logf(sum + shifted_exp(own, shift));
    float loss = log_sum + (shift - own);
    // a target outside the vocabulary has no loss, and neither has a row whose largest logit is infinite, or one whose sums were
    // not finished: NaN, which no later sum hides
    if (labels[row] < 0 || isinf(shift) || lost) loss = not_a_number();
    lse[row] = shift + log_sum;
    losses[row] = loss;
    if (reduction == HMC_REDUCE_NONE) loss_out[row_of[row]] = loss;
  }
  if (reduction == HMC_REDUCE_NONE) return;
  __shared__ int last;
  __shared__ double slots[JOIN_SLICES];
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0 && threadIdx.y == 0) last = atomicAdd(done, 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double v = 0.0;
  for (int i = threadIdx.y * 32 + threadIdx.x; i < rows; i += 32 * JOIN_SLICES) v += static_cast<double>(__ldcg(losses + i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threadIdx.x == 0) slots[threadIdx.y] = v;
  __syncthreads();
  if (threadIdx.y != 0) return;
  v = slots[threadIdx.x];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  // no row: the mean is NaN
  if (threadIdx.x == 0) *loss_out = static_cast<float>(reduction == HMC_REDUCE_MEAN ? v / rows : v);
}

// ------------------------------------------------------------------------------------------- gradient
// Per packed row the gradient of its loss (up to a common scale, which stays out of the BF16 products) and the weight of
// its target's row; per word the first row that has it as target and the number of them.
__global__ void __launch_bounds__(256) grad_rows_kernel(const float* __restrict__ grad, int reduction,
                                                        const int* __restrict__ count, const int* __restrict__ labels,
                                                        const int* __restrict__ row_of, const float* __restrict__ losses,
                                                        float* __restrict__ weights, float* __restrict__ coef,
                                                        float* __restrict__ scale, unsigned* __restrict__ slots,
                                                        int* __restrict__ members, const int* __restrict__ forward_failed,
                                                        const int* __restrict__ status, int* __restrict__ failed) {
  chain_next();  // the first of its chain
  const int rows = *count;
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i == 0) {
    float s = 1.0f;
    if (reduction == HMC_REDUCE_SUM) s = grad[0];
    if (reduction == HMC_REDUCE_MEAN) s = rows > 0 ? grad[0] / static_cast<float>(rows) : 0.0f;
    *scale = s;
  }
  const bool lost = has_failed(forward_failed, status);
  if (i < HMC_STATUS_WORDS) failed[i] = 0;
  if (i >= rows) return;
  const int label = labels[i];
  float w = reduction == HMC_REDUCE_NONE ? grad[row_of[i]] : 1.0f;
  if (label < 0 || lost) w = not_a_number();
  weights[i] = w;
  coef[i] = label >= 0 ? w * expm1f(-losses[i]) : 0.0f;  // w (p_target - 1)
  if (slots != nullptr && label >= 0) {
    atomicMin(&slots[label], static_cast<unsigned>(i));  // the smallest row, whatever the order of arrival
    atomicAdd(&members[label], 1);                       // from -1
  }
}

// Two to the power of `above` less a code, which is a half of `pair`: behind 2^23's upper bits it is a float that is exact.
__device__ __forceinline__ float power_of(uint32_t pair, uint32_t half, float above) {
  const float code = __uint_as_float(__byte_perm(pair, __float_as_uint(ROUND), half));
  const float x = code == ROUND + static_cast<float>(CODE_ZERO) ? above - INFINITY : __fmaf_rn(code - ROUND, -1.0f / CODE_STEPS, above);
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// p of a piece of the vocabulary out of its codes, times the row's gradient: what PROBS computes from the logits. A warp per row
// and 1024 words, eight rows per block, and the sum of what it stores; rows behind the last one that the products read with it are
// zero. Bound by memory, nearly by its instructions: 4096 x 65536 178 us (1.07 GB, 6.0 TB/s) where the product takes 1500; 2101 x 50257 78 us.
constexpr int SPREAD_WORDS = 1024;
__global__ void __launch_bounds__(256) spread_kernel(const uint16_t* __restrict__ codes, long long codes_pitch,
                                                     const float* __restrict__ tops, long long tops_pitch, int first_word, int width,
                                                     const int* __restrict__ count, const float* __restrict__ lse,
                                                     const float* __restrict__ weights, long long tokens,
                                                     __nv_bfloat16* __restrict__ probs, long long probs_pitch,
                                                     float* __restrict__ row_sums) {
  chain_wait();
  chain_next();
  const int rows = *count;
  const long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= (rows + TILE - 1) / TILE * TILE || row >= tokens) return;
  const int col = blockIdx.y * SPREAD_WORDS + (threadIdx.x & 31) * 8;
  const bool row_ok = row < rows;
  const float norm = row_ok ? lse[row] : 0.0f, weight = row_ok ? weights[row] : 0.0f;
  const uint16_t* src = codes + row * codes_pitch + first_word + col;
  __nv_bfloat16* dst = probs + row * probs_pitch + col;
  uint4 q[SPREAD_WORDS / 256];
  float from[SPREAD_WORDS / 256];
#pragma unroll
  for (int i = 0; i < SPREAD_WORDS / 256; ++i) {
    if (!row_ok || col + 256 * i >= width) continue;
    q[i] = ld_16(src + 256 * i);
    from[i] = tops[(first_word + col + 256 * i) / HALF * tops_pitch + row];
  }
  float2 sum = both(0.0f);
#pragma unroll
  for (int i = 0; i < SPREAD_WORDS / 256; ++i) {
    if (col + 256 * i >= width) break;
    uint4 out = make_uint4(0, 0, 0, 0);
    if (row_ok) {
      const float above = (from[i] - norm) * LOG2_E;
      auto two = [&](uint32_t pair) {
        const uint32_t word = pack_bf16x2(power_of(pair, 0x7610, above) * weight, power_of(pair, 0x7632, above) * weight);
        sum = add2(sum, unpack_bf16x2(word));
        return word;
      };
      out = make_uint4(two(q[i].x), two(q[i].y), two(q[i].z), two(q[i].w));
    }
    st_16(dst + 256 * i, out);
  }
  const float all = warp_sum(sum.x + sum.y);
  if (row_ok && (threadIdx.x & 31) == 0) row_sums[blockIdx.y * tops_pitch + row] = all;
}

// Sums of a packed row's stored entries: this piece's parts in their order, 32 slices of them in parallel, on top of those of
// earlier pieces. Bound by latency.
__global__ void __launch_bounds__(32 * JOIN_SLICES) row_sums_kernel(const float* __restrict__ row_sums, long long pitch, int parts,
                                                                    const int* __restrict__ count, int add,
                                                                    float* __restrict__ others) {
  __shared__ float sums[JOIN_SLICES][33];
  chain_wait();
  chain_next();
  const int row = blockIdx.x * 32 + threadIdx.x;
  const bool ok = row < *count;
  float sum = 0.0f;
  if (ok) {
#pragma unroll 8
    for (int i = threadIdx.y; i < parts; i += JOIN_SLICES) sum += row_sums[i * pitch + row];
  }
  sums[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y != 0 || !ok) return;
  sum = add ? others[row] : 0.0f;
#pragma unroll 8
  for (int s = 0; s < JOIN_SLICES; ++s) sum += sums[s][threadIdx.x];
  others[row] = sum;
}

// The sum of coef_i x_i over the rows that have a word as target, in their order, in slices of WORD_SLICE rows of a word:
// every row that is the first of a slice adds up its slice, into word_sums at its own row. (8192 tokens of 4096 by a power law, the
// commonest word with 480 of them: one block for all rows of a word 391 us, slices 74 us and their joining about 10.)
constexpr int WORD_THREADS = 256;
constexpr int WORD_SLICE = 32;

// Number of set `match`es in the block; place: those before this thread's.
__device__ __forceinline__ int matches(bool match, int& place) {
  __shared__ int found[WORD_THREADS / 32];
  const unsigned mask = __ballot_sync(0xffffffffu, match);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) found[warp] = __popc(mask);
  __syncthreads();
  int total = 0;
  place = __popc(mask & ((1u << lane) - 1u));
#pragma unroll
  for (int w = 0; w < WORD_THREADS / 32; ++w) {
    place += w < warp ? found[w] : 0;
    total += found[w];
  }
  __syncthreads();
  return total;
}

// Beside that, the rows of grad_hidden of the tokens that do not count (a block per token, too). Either may be absent.
__global__ void __launch_bounds__(WORD_THREADS) token_rows_kernel(const __nv_bfloat16* __restrict__ packed, int hidden,
                                                                  const int* __restrict__ count, const int* __restrict__ labels,
                                                                  const float* __restrict__ coef,
                                                                  const unsigned* __restrict__ slots,
                                                                  const int* __restrict__ members, float* __restrict__ word_sums,
                                                                  const int* __restrict__ position,
                                                                  __nv_bfloat16* __restrict__ grad_hidden) {
  __shared__ int slice[WORD_SLICE];
  chain_wait();
  chain_next();
  const int rows = *count;
  const int row = blockIdx.x;
  if (grad_hidden != nullptr && position[row] < 0) {
    for (int c = threadIdx.x * 8; c < hidden; c += WORD_THREADS * 8)
      st_16(grad_hidden + static_cast<long long>(row) * hidden + c, make_uint4(0, 0, 0, 0));
  }
  if (word_sums == nullptr || row >= rows) return;
  const int label = labels[row];
  if (label < 0) return;
  const int first = static_cast<int>(slots[label]);
  const int all = members[label] + 1;
  int place, before = 0;
  if (row != first) {
    if (all <= WORD_SLICE) return;
    for (int base = first; base < row; base += WORD_THREADS) {  // rows of this word before this one
      const int at = base + threadIdx.x;
      before += matches(at < row && labels[at] == label, place);
    }
    if (before % WORD_SLICE != 0) return;
  }
  const int want = min(WORD_SLICE, all - before);
  if (threadIdx.x == 0) slice[0] = row;
  int have = 1;
  for (int base = row + 1; have < want && base < rows; base += WORD_THREADS) {
    const int at = base + threadIdx.x;
    const bool match = at < rows && labels[at] == label;
    const int found = matches(match, place);
    if (match && have + place < want) slice[have + place] = at;
    have += found;
  }
  __syncthreads();
  const int n = min(have, want);
  for (int col = threadIdx.x * 8; col < hidden; col += WORD_THREADS * 8) {
    float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      const int from = slice[i];
      const float c = coef[from];
      const uint4 q = ld_16(packed + static_cast<long long>(from) * hidden + col);
      const uint32_t parts[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack_bf16x2(parts[e]);
        sum[2 * e] += c * f.x;
        sum[2 * e + 1] += c * f.y;
      }
    }
    float* dst = word_sums + static_cast<long long>(row) * hidden + col;
    *reinterpret_cast<float4*>(dst) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    *reinterpret_cast<float4*>(dst + 4) = make_float4(sum[4], sum[5], sum[6], sum[7]);
  }
}

// The slices of a word in their order, into the first one's place.
__global__ void __launch_bounds__(WORD_THREADS) word_slices_kernel(int hidden, const int* __restrict__ count,
                                                                   const int* __restrict__ labels,
                                                                   const unsigned* __restrict__ slots,
                                                                   const int* __restrict__ members,
                                                                   float* __restrict__ word_sums) {
  __shared__ int starts[WORD_THREADS / WORD_SLICE + 1];
  chain_wait();
  chain_next();
  const int rows = *count;
  const int row = blockIdx.x;
  if (row >= rows) return;
  const int label = labels[row];
  if (label < 0 || slots[label] != static_cast<unsigned>(row)) return;
  const int all = members[label] + 1;
  if (all <= WORD_SLICE) return;
  float* mine = word_sums + static_cast<long long>(row) * hidden;
  int seen = 1;
  for (int base = row + 1; seen < all && base < rows; base += WORD_THREADS) {
    const int at = base + threadIdx.x;
    const bool match = at < rows && labels[at] == label;
    int place;
    const int found = matches(match, place);
    // slices start at every WORD_SLICE-th row of the word
    const int from = (seen + WORD_SLICE - 1) / WORD_SLICE, to = (seen + found + WORD_SLICE - 1) / WORD_SLICE;
    seen += found;
    if (from == to) continue;
    if (match && (seen - found + place) % WORD_SLICE == 0) starts[(seen - found + place) / WORD_SLICE - from] = at;
    __syncthreads();
    for (int col = threadIdx.x * 4; col < hidden; col += WORD_THREADS * 4) {
      float4 sum = *reinterpret_cast<const float4*>(mine + col);
      for (int i = 0; i < to - from; ++i) {
        const float4 q = *reinterpret_cast<const float4*>(word_sums + static_cast<long long>(starts[i]) * hidden + col);
        sum.x += q.x, sum.y += q.y, sum.z += q.z, sum.w += q.w;
      }
      *reinterpret_cast<float4*>(mine + col) = sum;
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------- host
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                   const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = []() -> EncodeTiledFn {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &found) == cudaSuccess &&
        found == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeTiledFn>(sym);
    return nullptr;
  }();
  return fn;
}

// [rows, width] BF16 matrix with rows `pitch` elements apart, in boxes of box_width x box_rows.
int make_map(CUtensorMap* map, const void* base, long long width, long long rows, long long pitch, int box_width, int box_rows,
             CUtensorMapSwizzle swizzle) {
  EncodeTiledFn fn = encode_fn();
  HMC_REQUIRE(fn != nullptr, HMC_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch) * 2};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_width), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t step[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  HMC_REQUIRE(r == CUDA_SUCCESS, HMC_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
  return 0;
}
int map_k_major(CUtensorMap* map, const void* base, long long width, long long rows, long long pitch) {
  return make_map(map, base, width, rows, pitch, BK, HALF, CU_TENSOR_MAP_SWIZZLE_128B);
}
int map_mn_major(CUtensorMap* map, const void* base, long long width, long long rows, long long pitch) {
  return make_map(map, base, width, rows, pitch, 64, BK, CU_TENSOR_MAP_SWIZZLE_128B);
}
int map_store(CUtensorMap* map, const void* base, long long width, long long rows, long long pitch) {
  return make_map(map, base, width, rows, pitch, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B);
}

long long tiles_of(long long v) { return (v + TILE - 1) / TILE; }

// Tiles of a launch that may be cut along k, and the sums they leave: see Walker.
long long cut_tiles(long long tiles) {
  const long long pairs = sm_count() / 2;
  return tiles < pairs ? tiles : pairs - 1;
}

template <Product KIND>
int launch_product(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& c, const Params& p, long long tiles,
                   cudaStream_t stream) {
  static PerDeviceFlag configured{};
  if (int rc = allow_dynamic_smem(head_gemm_kernel<KIND>, SMEM_BYTES, configured)) return rc;
  const long long most = sm_count() / 2;
  // a product that is cut along k may have more units than tiles
  const int grid = static_cast<int>(2 * (KIND == GRAD_HIDDEN || tiles > most ? most : tiles));
  return launch_chained(head_gemm_kernel<KIND>, dim3(grid), dim3(NUM_THREADS), SMEM_BYTES, stream, a, b, c, p);
}

long long up256(long long bytes) { return (bytes + 255) / 256 * 256; }

constexpr long long FEW_TOKENS = 128;

// A piece of the vocabulary: what T rows of BF16 probabilities may take, in whole tiles, pieces of equal size. A training step of
// 8192 x 4096 x 131072 without kept logits, with pieces of 256 MiB 29.0 ms, 512 28.6, 1 GiB 28.8, 2 GiB (one piece) 30.1.
constexpr long long PIECE_BYTES = 512ll << 20;
long long piece_words(long long tokens, long long vocab) {
  long long most = PIECE_BYTES / (2 * tokens) / TILE * TILE;
  if (most < 4096) most = 4096;
  const long long pieces = (vocab + most - 1) / most;
  return tiles_of((vocab + pieces - 1) / pieces) * TILE;
}

// The words whose codes a forward leaves: as many pieces as KEEP_BYTES hold (a fortieth of the GPU's memory), in whole tiles.
// Kept against computed again: 4096 x 1024 x 32000 760 and 970 us, 16384 x 2048 x 131072 (all of it) 24.1 and 29.3 ms, twice the
// tokens (half of it) 56.0 and 61.6, 131072 x 512 x 65536 (a quarter of it) 46.9 and 47.9. The few-token kernel
// keeps none: with so few rows the logits cost one pass over the weight.
constexpr long long KEEP_BYTES = 4ll << 30;
long long kept_words(long long tokens, long long vocab) {
  if (tokens <= FEW_TOKENS) return 0;
  const long long piece = piece_words(tokens, vocab), most = KEEP_BYTES / (2 * tokens * piece) * piece, all = tiles_of(vocab) * TILE;
  return most < all ? most : all;
}

// What a forward leaves for its gradient, in one buffer of the caller.
struct State {
  int *count, *done, *failed, *position, *row_of, *labels;
  float *lse, *losses;
  __nv_bfloat16* packed;
  uint16_t* codes;  // [tokens][kept]
  float* tops;      // [kept / HALF][tokens]
  long long kept, bytes;
  State(void* base, long long tokens, long long hidden, long long vocab, bool keep) {
    kept = keep ? kept_words(tokens, vocab) : 0;
    char* p = static_cast<char*>(base);
    const long long words = up256(4 * tokens);
    count = reinterpret_cast<int*>(p);
    done = count + 1;
    failed = count + 4;  // status words
    position = reinterpret_cast<int*>(p + 256);
    row_of = reinterpret_cast<int*>(p + 256 + words);
    labels = reinterpret_cast<int*>(p + 256 + 2 * words);
    lse = reinterpret_cast<float*>(p + 256 + 3 * words);
    losses = reinterpret_cast<float*>(p + 256 + 4 * words);
    packed = reinterpret_cast<__nv_bfloat16*>(p + 256 + 5 * words);
    const long long at = 256 + 5 * words + up256(2 * tokens * hidden);
    codes = reinterpret_cast<uint16_t*>(p + at);
    tops = reinterpret_cast<float*>(p + at + 2 * tokens * kept);
    bytes = at + 2 * tokens * kept + 4 * tokens * (kept / HALF);
  }
};

// Parts that a launch over `vocab` words leaves per token: one per epilogue warp and column, or two per tile.
long long few_parts(long long vocab) {
  const long long pairs = sm_count() / 2, tiles = tiles_of(vocab);
  return 8 * (tiles < pairs ? tiles : pairs);
}

template <int N>
int launch_few(const CUtensorMap& words, const State& st, long long hidden, long long tokens, const Params& p, int* parts,
               cudaStream_t stream) {
  CUtensorMap rows;
  if (int rc = make_map(&rows, st.packed, hidden, tokens, hidden, BK, N / 2, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
  static PerDeviceFlag configured{};
  if (int rc = allow_dynamic_smem(few_tokens_kernel<N>, Few<N>::SMEM, configured)) return rc;
  *parts = static_cast<int>(few_parts(p.n));
  return launch_chained(few_tokens_kernel<N>, dim3(*parts / 4), dim3(Few<N>::THREADS), Few<N>::SMEM, stream, words, rows, p.n,
                        (p.k + BK - 1) / BK, p.count, p.labels, p.partial, p.pitch, p.failed, p.status);
}

struct GradSpace {
  float *scale, *weights, *coef, *word_sums, *sums, *part_sums, *row_sums, *others;
  unsigned* slots;
  int *members, *failed;
  __nv_bfloat16* probs;
  long long slot_bytes, bytes, piece;
  GradSpace(void* base, long long tokens, long long hidden, long long vocab) {
    piece = piece_words(tokens, vocab);
    long long at = 0;
    auto take = [&](long long size) {
      char* p = static_cast<char*>(base) + at;
      at += up256(size);
      return p;
    };
    scale = reinterpret_cast<float*>(take(4));
    failed = reinterpret_cast<int*>(take(4 * HMC_STATUS_WORDS));
    weights = reinterpret_cast<float*>(take(4 * tokens));
    coef = reinterpret_cast<float*>(take(4 * tokens));
    slots = reinterpret_cast<unsigned*>(take(4 * vocab));
    members = reinterpret_cast<int*>(take(4 * vocab));
    slot_bytes = reinterpret_cast<char*>(members) - reinterpret_cast<char*>(slots) + 4 * vocab;
    word_sums = reinterpret_cast<float*>(take(4 * tokens * hidden));
    sums = piece < vocab ? reinterpret_cast<float*>(take(4 * tokens * hidden)) : nullptr;
    part_sums = reinterpret_cast<float*>(take(2ll * (sm_count() / 2) * TILE * TILE * 4));
    row_sums = reinterpret_cast<float*>(take(4 * tokens * (piece / HALF)));
    others = reinterpret_cast<float*>(take(4 * tokens));
    probs = reinterpret_cast<__nv_bfloat16*>(take(2 * tokens * piece));
    bytes = at;
  }
};

int check_sizes(const char* name, int64_t tokens, int64_t hidden, int64_t vocab, int64_t weight_stride, const void* weight,
                int reduction) {
  HMC_REQUIRE(tokens > 0 && tokens < (1ll << 31) - TILE, HMC_ERR_INVALID, "%s: tokens (%lld) must be positive and below 2^31",
              name, (long long)tokens);
  HMC_REQUIRE(vocab > 0 && vocab < (1ll << 31) - TILE, HMC_ERR_INVALID, "%s: vocab (%lld) must be positive and below 2^31", name,
              (long long)vocab);
  HMC_REQUIRE(hidden > 0 && hidden % 8 == 0 && hidden < (1ll << 30), HMC_ERR_INVALID,
              "%s: hidden (%lld) must be a positive multiple of 8", name, (long long)hidden);
  HMC_REQUIRE(weight != nullptr && aligned16(weight) && weight_stride >= hidden && weight_stride % 8 == 0, HMC_ERR_INVALID,
              "%s: weight rows must start on 16-byte boundaries, at least hidden apart", name);
  HMC_REQUIRE(reduction >= HMC_REDUCE_NONE && reduction <= HMC_REDUCE_SUM, HMC_ERR_INVALID, "%s: unknown reduction %d", name,
              reduction);
  return 0;
}

}  // namespace
}  // namespace hmc

extern "C" int64_t hmc_vocab_loss_state_bytes(int64_t tokens, int64_t hidden, int64_t vocab, int keep) {
  return tokens > 0 && hidden > 0 && vocab > 0 ? hmc::State(nullptr, tokens, hidden, vocab, keep != 0).bytes : 0;
}

extern "C" int64_t hmc_vocab_loss_workspace_bytes(int64_t tokens, int64_t vocab) {
  using namespace hmc;
  if (tokens <= 0 || vocab <= 0) return 0;
  // of the most parts that any smaller call leaves too
  const long long parts = 2 * tiles_of(vocab) > few_parts(vocab) ? 2 * tiles_of(vocab) : few_parts(vocab);
  return up256(4 * tokens) + parts * tokens * 8;
}

extern "C" int64_t hmc_vocab_loss_grad_workspace_bytes(int64_t tokens, int64_t hidden, int64_t vocab) {
  return tokens > 0 && hidden > 0 && vocab > 0 ? hmc::GradSpace(nullptr, tokens, hidden, vocab).bytes : 0;
}

extern "C" int hmc_vocab_loss(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, const void* targets,
                              int targets_i64, int64_t tokens, int64_t hidden, int64_t vocab, int64_t ignore_index, int reduction,
                              int keep, void* state, float* loss, void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  using namespace hmc;
  if (int rc = check_sizes("hmc_vocab_loss", tokens, hidden, vocab, weight_stride, weight, reduction)) return rc;
  HMC_REQUIRE(x != nullptr && targets != nullptr && state != nullptr && loss != nullptr && x_stride >= 0, HMC_ERR_INVALID,
              "hmc_vocab_loss: null tensor pointer or negative row stride");
  HMC_REQUIRE(aligned16(state) && workspace != nullptr && aligned16(workspace) &&
                  workspace_bytes >= hmc_vocab_loss_workspace_bytes(tokens, vocab),
              HMC_ERR_INVALID, "hmc_vocab_loss: the workspace must hold %lld bytes, it and the state on 16-byte boundaries",
              (long long)hmc_vocab_loss_workspace_bytes(tokens, vocab));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const State st(state, tokens, hidden, vocab, keep != 0);
  float* target_logit = static_cast<float*>(workspace);
  float2* partial = reinterpret_cast<float2*>(static_cast<char*>(workspace) + up256(4 * tokens));
  float* token_loss = reduction == HMC_REDUCE_NONE ? loss : nullptr;
  const Targets given{targets, targets_i64, ignore_index, vocab};
  const int vector = aligned16(x) && x_stride % 8 == 0;
  if (int rc = launch_chained(pack_rows_kernel, dim3(static_cast<unsigned>((tokens + PACK_TOKENS - 1) / PACK_TOKENS)), dim3(PACK_THREADS),
                              0, s, static_cast<const __nv_bfloat16*>(x), x_stride, given, tokens, static_cast<int>(hidden), vector,
                              st.count, st.done, st.failed, st.position, st.row_of, st.labels, st.packed,
                              static_cast<const __nv_bfloat16*>(weight), weight_stride, target_logit, token_loss))
    return rc;

  Params p{};
  p.n = static_cast<int>(vocab), p.k = static_cast<int>(hidden);
  p.count = st.count, p.labels = st.labels, p.partial = partial, p.pitch = tokens, p.failed = st.failed, p.status = status;
  CUtensorMap a, b;
  if (int rc = map_k_major(&b, weight, hidden, vocab, weight_stride)) return rc;
  int parts = 0;
  if (tokens <= FEW_TOKENS) {
    const int rc = tokens <= 32   ? launch_few<32>(b, st, hidden, tokens, p, &parts, s)
                   : tokens <= 64 ? launch_few<64>(b, st, hidden, tokens, p, &parts, s)
                                  : launch_few<128>(b, st, hidden, tokens, p, &parts, s);
    if (rc != 0) return rc;
  } else {
    if (int rc = map_k_major(&a, st.packed, hidden, tokens, hidden)) return rc;
    CUtensorMap codes = a;
    if (st.kept > 0) {
      if (int rc = map_store(&codes, st.codes, st.kept, tokens, st.kept)) return rc;
      p.kept = static_cast<int>(st.kept), p.tops = st.tops;
    }
    if (int rc = launch_product<STATS>(a, b, codes, p, tiles_of(tokens) * tiles_of(vocab), s)) return rc;
    parts = static_cast<int>(2 * tiles_of(vocab));
  }
  return launch_chained(join_kernel, dim3(static_cast<unsigned>((tokens + 31) / 32)), dim3(32, JOIN_SLICES), 0, s, partial, tokens, parts,
                        st.count, st.labels, st.row_of, target_logit, st.lse, st.losses, reduction, st.done, st.failed, status, loss);
}

extern "C" int hmc_vocab_loss_grad(const void* state, const void* weight, int64_t weight_stride, int64_t tokens, int64_t hidden,
                                   int64_t vocab, int reduction, int keep, const float* grad_loss, void* grad_hidden, void* grad_weight,
                                   void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  using namespace hmc;
  if (int rc = check_sizes("hmc_vocab_loss_grad", tokens, hidden, vocab, weight_stride, weight, reduction)) return rc;
  HMC_REQUIRE(state != nullptr && grad_loss != nullptr && aligned16(state), HMC_ERR_INVALID,
              "hmc_vocab_loss_grad: null tensor pointer or a state off a 16-byte boundary");
  HMC_REQUIRE(aligned16(grad_hidden) && aligned16(grad_weight), HMC_ERR_INVALID,
              "hmc_vocab_loss_grad: gradients must be 16-byte aligned");
  if (grad_hidden == nullptr && grad_weight == nullptr) return 0;
  HMC_REQUIRE(workspace != nullptr && aligned16(workspace) &&
                  workspace_bytes >= hmc_vocab_loss_grad_workspace_bytes(tokens, hidden, vocab),
              HMC_ERR_INVALID, "hmc_vocab_loss_grad: the workspace must hold %lld bytes on a 16-byte boundary",
              (long long)hmc_vocab_loss_grad_workspace_bytes(tokens, hidden, vocab));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const State st(const_cast<void*>(state), tokens, hidden, vocab, keep != 0);
  const GradSpace w(workspace, tokens, hidden, vocab);
  const int width = static_cast<int>(hidden);
  if (grad_weight != nullptr) HMC_CUDA_OK(cudaMemsetAsync(w.slots, 0xff, w.slot_bytes, s));  // no first row, -1 members
  grad_rows_kernel<<<static_cast<unsigned>((tokens + 255) / 256), 256, 0, s>>>(
      grad_loss, reduction, st.count, st.labels, st.row_of, st.losses, w.weights, w.coef, w.scale,
      grad_weight != nullptr ? w.slots : nullptr, w.members, st.failed, status, w.failed);
  HMC_LAUNCH_OK();
  float* word_sums = grad_weight != nullptr ? w.word_sums : nullptr;
  if (int rc = launch_chained(token_rows_kernel, dim3(static_cast<unsigned>(tokens)), dim3(WORD_THREADS), 0, s, st.packed, width, st.count,
                              st.labels, w.coef, w.slots, w.members, word_sums, st.position,
                              static_cast<__nv_bfloat16*>(grad_hidden)))
    return rc;
  if (grad_weight != nullptr && tokens > WORD_SLICE) {
    if (int rc = launch_chained(word_slices_kernel, dim3(static_cast<unsigned>(tokens)), dim3(WORD_THREADS), 0, s, width, st.count,
                                st.labels, w.slots, w.members, w.word_sums))
      return rc;
  }

  Params base{};
  base.count = st.count, base.labels = st.labels, base.lse = st.lse, base.weights = w.weights, base.scale = w.scale;
  base.coef = w.coef, base.row_of = st.row_of, base.failed = w.failed, base.status = status;
  CUtensorMap rows_k, rows_mn;
  if (int rc = map_k_major(&rows_k, st.packed, hidden, tokens, hidden)) return rc;
  if (int rc = map_mn_major(&rows_mn, st.packed, hidden, tokens, hidden)) return rc;
  for (long long first = 0; first < vocab; first += w.piece) {
    const long long words = vocab - first < w.piece ? vocab - first : w.piece;
    const __nv_bfloat16* head = static_cast<const __nv_bfloat16*>(weight) + first * weight_stride;
    CUtensorMap head_k, head_mn, probs_store, probs_k, probs_mn;
    Params p = base;
    p.first_word = static_cast<int>(first);
    p.n = static_cast<int>(words), p.k = width;
    p.row_sums = w.row_sums, p.pitch = tokens;
    int parts;  // sums that the probabilities of a row leave
    if (first < st.kept) {
      const int whole = static_cast<int>(tiles_of(words) * TILE);
      parts = (whole + SPREAD_WORDS - 1) / SPREAD_WORDS;
      if (int rc = launch_chained(spread_kernel, dim3(static_cast<unsigned>((tokens + 7) / 8), parts), dim3(256), 0, s, st.codes,
                                  st.kept, st.tops, tokens, p.first_word, whole, st.count, st.lse, w.weights, tokens, w.probs, w.piece,
                                  w.row_sums))
        return rc;
    } else {
      parts = static_cast<int>(2 * tiles_of(words));
      if (int rc = map_k_major(&head_k, head, hidden, words, weight_stride)) return rc;
      if (int rc = map_store(&probs_store, w.probs, words, tokens, w.piece)) return rc;
      if (int rc = launch_product<PROBS>(rows_k, head_k, probs_store, p, tiles_of(tokens) * tiles_of(words), s)) return rc;
    }
    if (grad_hidden != nullptr) {
      if (int rc = launch_chained(row_sums_kernel, dim3(static_cast<unsigned>((tokens + 31) / 32)), dim3(32, JOIN_SLICES), 0, s, w.row_sums,
                                  tokens, parts, st.count, first > 0, w.others))
        return rc;
      if (int rc = map_k_major(&probs_k, w.probs, words, tokens, w.piece)) return rc;
      if (int rc = map_mn_major(&head_mn, head, hidden, words, weight_stride)) return rc;
      p.n = width, p.k = static_cast<int>(words);
      p.sums = w.sums, p.add = first > 0, p.last = first + words == vocab;
      p.head = static_cast<const __nv_bfloat16*>(weight), p.head_stride = weight_stride;
      p.out = static_cast<__nv_bfloat16*>(grad_hidden);
      p.part_sums = w.part_sums, p.others = w.others;
      const long long tiles = tiles_of(tokens) * tiles_of(width);
      if (int rc = launch_product<GRAD_HIDDEN>(probs_k, head_mn, probs_k, p, tiles, s)) return rc;
      if (int rc = launch_chained(join_parts_kernel, dim3(TILE / 8, static_cast<unsigned>(cut_tiles(tiles))), dim3(256), 0, s, p,
                                  sm_count() / 2))
        return rc;
    }
    if (grad_weight != nullptr) {
      CUtensorMap grad_store;
      __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(grad_weight) + first * hidden;
      if (int rc = map_mn_major(&probs_mn, w.probs, words, tokens, w.piece)) return rc;
      if (int rc = map_store(&grad_store, dst, hidden, words, hidden)) return rc;
      p.m = static_cast<int>(words), p.n = width;
      p.slots = reinterpret_cast<const int*>(w.slots), p.word_sums = w.word_sums;
      if (int rc = launch_product<GRAD_WEIGHT>(probs_mn, rows_mn, grad_store, p, tiles_of(words) * tiles_of(width), s)) return rc;
    }
  }
  return 0;
}
