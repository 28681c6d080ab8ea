// A paged cache held in 4 bits: rows quantised as they are written, read back, and attention over them.
//
// Format (block-scaled FP4, the MXFP4 element and scale types of the OCP microscaling formats).  A row is one
// token's K or V of one kv head; 32 consecutive elements are a block: 32 E2M1 codes (0, .5, 1, 1.5, 2, 3, 4, 6 and
// their negatives; element 2i in the low half of byte i) and one E8M0 scale byte s for 2^(s - 127), 255 for NaN.
// The pool is (num_pages, 2, h_kv, page_size, 17 D / 32) bytes; the bytes of one (page, K or V, head) are the codes
// of its tokens (D / 2 bytes each), then their scales (D / 32 bytes each).
//
// Quantisation of a block with largest magnitude a: scale 2^e with the smallest e in [-23, 13] for which
// a <= 7 2^e (7 is the last value nearer to the largest code, 6, than a further one would be), codes rounded to
// nearest, ties to the even code, magnitudes above 6 2^e saturate.  Every step is exact but that rounding, so the
// bits do not depend on how it is computed.  The range of e makes reading back exact in fp16: at e = -23 the codes
// are multiples of fp16's smallest subnormal, at e = 13 the largest is 49152.  A block with a value that is not
// finite is NaN as a whole.
//
// gfx950 converts two codes and their scale to two fp16 in one full-rate instruction (v_cvt_scalef32_pk_f16_fp4),
// and two fp16 to codes with exactly the rounding above (v_cvt_scalef32_pk_fp4_f16).  A scale byte moved to the
// exponent field of a float is the scale operand, 255 included (NaN).
#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "kernels_common.cuh"
#include "runtime_support.h"

namespace tvmkv {

constexpr int kRun = 16;            // tokens the attention kernels take from a page at a time
constexpr float kNoKey = -1e30f;    // running maximum of a row that has seen no key
constexpr float kEmptyLse = -5e4f;  // log-sum-exp of a row without keys (its output is 0)

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// eight codes -> eight fp16
__device__ __forceinline__ half8_t dequantise8(uint32_t codes, float scale) {
  const half2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0);
  const half2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1);
  const half2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2);
  const half2_t d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3);
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// ------------------------------------------------------------------------------------------
// append: k|v[i, h, :] -> slot position_map[i] (negative: none).  A lane quantises 8 elements, the four lanes of a
// block share its largest magnitude; as 16-bit integers magnitudes order like the values, infinities and NaN above
// all others.  Bound by its bytes: 2 D read and 17 D / 32 written per row.
// ------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void mxfp4_append_kernel(uint8_t* __restrict__ pages, const half_t* __restrict__ k_data,
                                                           const half_t* __restrict__ v_data,
                                                           const int32_t* __restrict__ position_map, int64_t rows,
                                                           int h_kv, int page_size, int d) {
  const int chunks = d / 8;
  const int64_t gid = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t row = gid / chunks;  // (token, K or V, head)
  if (row >= rows) return;           // whole blocks: chunks is a multiple of 4
  const int c = gid % chunks;
  const int h = row % h_kv;
  const int kv = row / h_kv & 1;
  const int64_t token = row / (2 * h_kv);
  const int32_t position = position_map[token];
  if (position < 0) return;
  Vec16 x = ld16((kv ? v_data : k_data) + (token * h_kv + h) * d + c * 8);
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) most = max(most, max(x.w[i] & 0x7fffu, x.w[i] >> 16 & 0x7fffu));
  most = max(most, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(most), kDppXor1, 0xf, 0xf, true)));
  most = max(most, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(most), kDppXor2, 0xf, 0xf, true)));
  const bool finite = most < 0x7c00u;
  // 1.f 2^k -> e = k - 2 up to f = .75, k - 1 above: the carry out of the mantissa
  const uint32_t bits = __float_as_uint(static_cast<float>(__builtin_bit_cast(half_t, static_cast<uint16_t>(most))));
  const int byte = min(max(static_cast<int>((bits + 0x1fffffu) >> 23) - 2, 127 - 23), 127 + 13);
  const float scale = scale_of(byte);
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, x.h2[0], scale, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, x.h2[1], scale, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, x.h2[2], scale, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, x.h2[3], scale, 3);
  const int64_t page = position / page_size;
  const int slot = position % page_size;
  uint8_t* slab = pages + ((page * 2 + kv) * h_kv + h) * (static_cast<int64_t>(page_size) * (17 * d / 32));
  *reinterpret_cast<uint32_t*>(slab + slot * (d / 2) + c * 4) = finite ? codes : 0;
  if ((c & 3) == 0) slab[page_size * (d / 2) + slot * (d / 32) + c / 4] = finite ? byte : 255;
}

// ------------------------------------------------------------------------------------------
// read: slot position_map[i] -> k|v[i, h, :] in fp16, exact; a negative position gives zeros.
// ------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void mxfp4_read_kernel(const uint8_t* __restrict__ pages, half_t* __restrict__ k_data,
                                                         half_t* __restrict__ v_data,
                                                         const int32_t* __restrict__ position_map, int64_t rows, int h_kv,
                                                         int page_size, int d) {
  const int chunks = d / 8;
  const int64_t gid = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t row = gid / chunks;
  if (row >= rows) return;
  const int c = gid % chunks;
  const int h = row % h_kv;
  const int kv = row / h_kv & 1;
  const int64_t token = row / (2 * h_kv);
  const int32_t position = position_map[token];
  Vec16 x = zero16();
  if (position >= 0) {
    const int64_t page = position / page_size;
    const int slot = position % page_size;
    const uint8_t* slab = pages + ((page * 2 + kv) * h_kv + h) * (static_cast<int64_t>(page_size) * (17 * d / 32));
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(slab + slot * (d / 2) + c * 4);
    x.h8 = dequantise8(codes, scale_of(slab[page_size * (d / 2) + slot * (d / 32) + c / 4]));
  }
  st16((kv ? v_data : k_data) + (token * h_kv + h) * d + c * 8, x);
}

// ------------------------------------------------------------------------------------------
// Attention.  With s = sm_scale log2(e) q.k the output of a row is sum 2^(s - m) v / sum 2^(s - m) and its
// log-sum-exp (base 2) m + log2(sum), m the running maximum; sums, statistics and outputs in float32, the weights
// rounded to fp16 for the second matrix product (11 bits, as the output itself).
//
// A row of a kv head is (query token, query head of its group), token-major.  A workgroup of four waves takes 16
// rows of a kv head and a range of the sequence's keys, a wave every fourth step of 32 keys (two runs of 16 tokens;
// page sizes are multiples of 16, so a run lies in one page):
//   S^T[token, row] = K Q^T    the lane (token, quarter of the row) loads its codes straight from memory, turns
//                              them into fp16 in registers and has the matrix instruction's A operand: the order of
//                              the contraction is free, q is loaded in the same one;
//   O^T[d, row]     = V^T P^T  V is turned into fp16 the same way and put into the wave's LDS tile, from where the
//                              transposing read takes it; P stays in registers.
// ------------------------------------------------------------------------------------------
struct Mxfp4Params {
  const half_t* q;
  const uint8_t* pages;
  const int32_t* q_indptr;  // NULL: one query token a sequence
  const int32_t* page_indptr;
  const int32_t* page_values;
  const int32_t* last_page_len;
  const int32_t* window_offset;  // (B) first stored token behind the evicted ones, or NULL
  const int32_t* sink_size;      // (B) first tokens that are never evicted, or NULL
  half_t* output;
  float* lse;
  float* part_o;   // (slots, h_q, D) outputs of the chunks, not normalised
  float* part_ml;  // (slots, h_q, 2) their maxima and sums
  int batch;
  int h_q;
  int h_kv;
  int group;
  int row_blocks;  // blocks of 16 rows of a sequence with one query token
  int causal;
  int page_size;
  uint32_t runs_per_page;
  uint32_t run_magic;  // 2^32 / runs_per_page, rounded up (0: 1)
  int chunk_runs;      // keys of a work item of a decode launch, in runs; even
  float scale_log2;
};

// The last of n sequences whose begin(i) is at most `slot` (begin increases, begin(0) <= slot): the lanes of the
// wave probe 64 of them at a time, one round trip to memory per factor of 64.
template <class Begin>
__device__ __forceinline__ int sequence_of(int n, int slot, int lane, Begin begin) {
  int lo = 0;
  while (n > 64) {
    const int stride = (n + 63) >> 6;
    const int at = lo + lane * stride;
    const bool hit = at < lo + n && begin(at) <= slot;
    const int first = lo + (__popcll(__ballot(hit)) - 1) * stride;
    n = min(stride, lo + n - first);
    lo = first;
  }
  const bool hit = lane < n && begin(lo + lane) <= slot;
  return __builtin_amdgcn_readfirstlane(lo + max(static_cast<int>(__popcll(__ballot(hit))), 1) - 1);
}

// First work item of a sequence: with it sequence i has chunks for all tokens that its pages could hold.
__device__ __forceinline__ int chunk_begin(const Mxfp4Params& p, int i) {
  return static_cast<int>(static_cast<int64_t>(p.page_indptr[i]) * p.runs_per_page / p.chunk_runs) + i;
}

// What a lane holds of a row: D / 4 elements in chunks of 8, and the scales of their blocks.  The lane group g4
// (0..3) has consecutive chunks, at head dim 256 four of either half of the row.
template <int D>
struct LaneRow {
  static constexpr int CH = D / 32;             // chunks
  static constexpr int NS = D == 96 || D == 256 ? 2 : 1;  // blocks they lie in
  uint32_t w[CH];
  uint32_t s[NS];

  static __device__ __forceinline__ int chunk(int g4, int c) { return D == 256 ? (c >> 2) * 16 + g4 * 4 + (c & 3) : g4 * CH + c; }
  static __device__ __forceinline__ int block(int g4, int i) {
    return D == 256 ? g4 + 4 * i : D == 128 ? g4 : D == 64 ? g4 >> 1 : (3 * g4 + 2 * i) >> 2;
  }
  static __device__ __forceinline__ int scale_index(int g4, int c) {
    return D == 256 ? c >> 2 : D == 96 ? ((3 * g4 + c) >> 2) - ((3 * g4) >> 2) : 0;
  }
  __device__ __forceinline__ void load(const uint8_t* slab, int page_size, int slot, int g4) {
    const uint8_t* row = slab + slot * (D / 2);
    if constexpr (D == 64) {
      const uint2 v = *reinterpret_cast<const uint2*>(row + g4 * 8);
      w[0] = v.x;
      w[1] = v.y;
    } else if constexpr (D == 96) {
#pragma unroll
      for (int c = 0; c < CH; ++c) w[c] = *reinterpret_cast<const uint32_t*>(row + g4 * 12 + c * 4);
    } else {
#pragma unroll
      for (int i = 0; i < D / 128; ++i) {
        const Vec16 v = ld16(row + i * 64 + g4 * 16);
#pragma unroll
        for (int c = 0; c < 4; ++c) w[i * 4 + c] = v.w[c];
      }
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) s[i] = slab[page_size * (D / 2) + slot * (D / 32) + block(g4, i)];
  }
  __device__ __forceinline__ half8_t values(int g4, int c) const {
    const int i = scale_index(g4, c);
    return dequantise8(w[c], scale_of(NS == 1 ? s[0] : (i ? s[NS - 1] : s[0])));
  }
};

template <int D, bool PREFILL>
__global__ __launch_bounds__(256) void mxfp4_attn_kernel(Mxfp4Params p) {
  constexpr int CH = LaneRow<D>::CH;
  constexpr int DB = D / 16;
  constexpr int VS = D + 16;  // halfs of a row of the V tile: 32 bytes on, so that rows meet other banks
  constexpr int OS = D + 4;   // floats of a row of the merge buffer
  static_assert(32 * VS * sizeof(half_t) >= 16 * OS * sizeof(float), "the merge buffer takes the V tile's place");
  __shared__ __attribute__((aligned(16))) half_t v_tiles[4][32 * VS];
  __shared__ float sm_m[4][16], sm_l[4][16];

  const int wave = threadIdx.x >> 6;
  const int lane = threadIdx.x & 63;
  const int c16 = lane & 15;
  const int g4 = lane >> 4;

  // ---- which rows, which keys ----------------------------------------------------------------
  const int kvh = blockIdx.x % p.h_kv;
  int slot, rb;
  if (PREFILL) {
    slot = blockIdx.x / p.h_kv;
    rb = 0;
  } else {
    slot = blockIdx.x / (p.h_kv * p.row_blocks);
    rb = blockIdx.x / p.h_kv % p.row_blocks;
  }
  const auto row_begin = [&](int i) { return static_cast<int>(static_cast<int64_t>(p.q_indptr[i]) * p.group / 16) + i; };
  const int b = PREFILL ? sequence_of(p.batch, slot, lane, row_begin)
                        : sequence_of(p.batch, slot, lane, [&](int i) { return chunk_begin(p, i); });
  const int page_begin = p.page_indptr[b];
  const int num_pages = p.page_indptr[b + 1] - page_begin;
  const int stored = num_pages > 0 ? (num_pages - 1) * p.page_size + p.last_page_len[b] : 0;
  const int sink = num_pages > 0 && p.sink_size != nullptr ? p.sink_size[b] : 0;
  const int window = num_pages > 0 && p.window_offset != nullptr ? p.window_offset[b] : 0;
  const int keys = stored - window + sink;
  const int q_begin = PREFILL ? p.q_indptr[b] : b;
  const int q_len = PREFILL ? p.q_indptr[b + 1] - q_begin : 1;
  const int rows = q_len * p.group;
  if (PREFILL) rb = slot - row_begin(b);
  const int row0 = rb * 16;
  if (row0 >= rows) return;  // a spare slot
  const int rows_here = min(16, rows - row0);
  // stored tokens [0, end) hold the first n keys; token t of them is one iff t < sink or t >= window
  const auto end_of = [&](int n) { return n <= sink ? n : n - sink + window; };
  const auto end_of_row = [&](int r) { return end_of(p.causal ? min(max(keys - q_len + 1 + r / p.group, 0), keys) : keys); };
  const int my_row = row0 + c16;
  const int my_end = c16 < rows_here ? end_of_row(my_row) : 0;
  const int first_end = end_of_row(row0);                  // every row sees the keys in front of it
  const int last_end = end_of_row(row0 + rows_here - 1);   // no row sees a key behind it
  int run_lo = 0, run_hi = (last_end + kRun - 1) / kRun;
  int chunks = 1;
  if (!PREFILL) {
    const int chunk = slot - chunk_begin(p, b);
    chunks = max(1, (run_hi + p.chunk_runs - 1) / p.chunk_runs);
    if (chunk >= chunks) return;
    run_lo = chunk * p.chunk_runs;
    run_hi = min(run_hi, run_lo + p.chunk_runs);
  }

  half8_t qf[CH];
  {
    const int token = q_begin + my_row / p.group;
    const half_t* q = p.q + (static_cast<int64_t>(token) * p.h_q + kvh * p.group + my_row % p.group) * D;
#pragma unroll
    for (int c = 0; c < CH; ++c) qf[c] = c16 < rows_here ? ld16(q + LaneRow<D>::chunk(g4, c) * 8).h8 : zero16().h8;
  }
  float4_t o[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i) o[i] = float4_t{0.f, 0.f, 0.f, 0.f};
  float m = kNoKey, l = 0.f;
  uint32_t poisoned = 0;  // 32-element parts of the output that are NaN, see below

  half_t* const vt = v_tiles[wave];
  const int64_t slab_bytes = static_cast<int64_t>(p.page_size) * (17 * D / 32);
  for (int run = run_lo + 2 * wave; run < run_hi; run += 8) {
    LaneRow<D> k[2], v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t at = min(run + h, run_hi - 1);
      const uint32_t nth = p.run_magic != 0 ? __umulhi(at, p.run_magic) : at;
      const int page = __builtin_amdgcn_readfirstlane(p.page_values[page_begin + nth]);
      const int in_page = static_cast<int>(at - nth * p.runs_per_page) * kRun + c16;
      const uint8_t* slab = p.pages + (static_cast<int64_t>(page) * 2 * p.h_kv + kvh) * slab_bytes;
      k[h].load(slab, p.page_size, in_page, g4);
      v[h].load(slab + p.h_kv * slab_bytes, p.page_size, in_page, g4);
    }
    const int t0 = run * kRun;
    const bool whole = t0 + 2 * kRun <= first_end && (t0 >= window || t0 + 2 * kRun <= sink);  // no key of the step is masked
    float s[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < CH; ++c) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[h].values(g4, c), qf[c], acc, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = t0 + h * kRun + 4 * g4 + i;
        s[h][i] = acc[i] * p.scale_log2;
        if (!whole) s[h][i] = t < my_end && (t < sink || t >= window) ? s[h][i] : -INFINITY;
      }
    }
    if (!whole) {
      // A weight of 0 times NaN is NaN: what no row of the item sees is read as 0, and blocks that are NaN reach
      // the rows that see them by a mark of their own.
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = t0 + h * kRun + c16;
        const bool seen = t < last_end && (t < sink || t >= window);
#pragma unroll
        for (int i = 0; i < LaneRow<D>::NS; ++i) {
          const bool nan = seen && v[h].s[i] == 255;
          for (uint64_t left = __ballot(nan); left != 0; left &= left - 1) {
            const int who = __ffsll(static_cast<long long>(left)) - 1;
            const int at = t0 + h * kRun + (who & 15);
            if (at < my_end) poisoned |= 1u << LaneRow<D>::block(who >> 4, i);
          }
          if (nan || !seen) v[h].s[i] = 0;
        }
      }
    }
    // softmax statistics: the lane has 8 of the step's 32 keys of row c16
    float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    top = fmaxf(m, max_xor32(max_xor16(top)));
    const float alpha = fast_exp2(m - top);
    m = top;
    l *= alpha;
#pragma unroll
    for (int i = 0; i < DB; ++i) o[i] *= alpha;
    half8_t pf;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = fast_exp2(s[h][i] - m);
        l += w;
        pf[h * 4 + i] = static_cast<half_t>(w);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        *reinterpret_cast<half8_t*>(vt + (h * kRun + c16) * VS + LaneRow<D>::chunk(g4, c) * 8) = v[h].values(g4, c);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < DB; ++i) {
      const half_t* src = vt + (4 * g4 + (c16 >> 2)) * VS + i * 16 + (c16 & 3) * 4;
      const half4_t lo = lds_read_tr16(src), hi = lds_read_tr16(src + kRun * VS);
      const half8_t a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pf, o[i], 0, 0, 0);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  // ---- the four waves' states become one ------------------------------------------------------
  l = sum_xor32(sum_xor16(l));
  if (__ballot(poisoned != 0) != 0) {
    poisoned |= __shfl_xor(poisoned, 16);
    poisoned |= __shfl_xor(poisoned, 32);
#pragma unroll
    for (int i = 0; i < DB; ++i) {
      if (poisoned >> (i / 2) & 1) o[i] = float4_t{NAN, NAN, NAN, NAN};
    }
  }
  if (g4 == 0) {
    sm_m[wave][c16] = m;
    sm_l[wave][c16] = l;
  }
  float* const mine = reinterpret_cast<float*>(vt);
#pragma unroll
  for (int i = 0; i < DB; ++i) *reinterpret_cast<float4_t*>(mine + c16 * OS + i * 16 + 4 * g4) = o[i];
  __syncthreads();
  for (int at = threadIdx.x; at < rows_here * (D / 4); at += 256) {
    const int r = at / (D / 4), f = at % (D / 4) * 4;
    const float most = fmaxf(fmaxf(sm_m[0][r], sm_m[1][r]), fmaxf(sm_m[2][r], sm_m[3][r]));
    float sum = 0.f;
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float part = fast_exp2(sm_m[w][r] - most);
      sum += sm_l[w][r] * part;
      acc += *reinterpret_cast<const float4_t*>(reinterpret_cast<const float*>(v_tiles[w]) + r * OS + f) * part;
    }
    const int hq = kvh * p.group + (row0 + r) % p.group;
    if (chunks == 1) {
      const int64_t out = static_cast<int64_t>(q_begin + (row0 + r) / p.group) * p.h_q + hq;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      half4_t h;
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = static_cast<half_t>(acc[i] * inv);
      *reinterpret_cast<half4_t*>(p.output + out * D + f) = h;
      if (f == 0) p.lse[out] = sum == 0.f ? kEmptyLse : most + fast_log2(sum);
    } else {
      const int64_t out = static_cast<int64_t>(slot) * p.h_q + hq;
      *reinterpret_cast<float4_t*>(p.part_o + out * D + f) = acc;
      if (f == 0) {
        p.part_ml[out * 2] = most;
        p.part_ml[out * 2 + 1] = sum;
      }
    }
  }
}

// Joins the chunks of a sequence's row: one wave per (sequence, query head).
template <int D>
__global__ __launch_bounds__(256) void mxfp4_merge_kernel(Mxfp4Params p) {
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.batch * p.h_q) return;
  const int b = row / p.h_q;
  const int hq = row % p.h_q;
  const int num_pages = p.page_indptr[b + 1] - p.page_indptr[b];
  const int stored = num_pages > 0 ? (num_pages - 1) * p.page_size + p.last_page_len[b] : 0;
  const int chunks = ((stored + kRun - 1) / kRun + p.chunk_runs - 1) / p.chunk_runs;
  if (chunks <= 1) return;  // the attention kernel wrote the row
  const int64_t first = static_cast<int64_t>(chunk_begin(p, b)) * p.h_q + hq;
  float most = kNoKey;
  for (int c = 0; c < chunks; ++c) most = fmaxf(most, p.part_ml[(first + static_cast<int64_t>(c) * p.h_q) * 2]);
  float sum = 0.f, acc[(D + 63) / 64] = {};
  for (int c = 0; c < chunks; ++c) {
    const int64_t at = first + static_cast<int64_t>(c) * p.h_q;
    const float part = fast_exp2(p.part_ml[at * 2] - most);
    sum += p.part_ml[at * 2 + 1] * part;
#pragma unroll
    for (int i = 0; i < (D + 63) / 64; ++i) {
      if (i * 64 + lane < D) acc[i] += p.part_o[at * D + i * 64 + lane] * part;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < (D + 63) / 64; ++i) {
    if (i * 64 + lane < D) p.output[static_cast<int64_t>(row) * D + i * 64 + lane] = static_cast<half_t>(acc[i] * inv);
  }
  if (lane == 0) p.lse[row] = sum == 0.f ? kEmptyLse : most + fast_log2(sum);
}

static void check_mxfp4(const char* what, int32_t h_kv, int32_t page_size, int32_t d) {
  KV_CHECK(h_kv > 0) << what << ": bad shape";
  KV_UNSUPPORTED(d != 64 && d != 96 && d != 128 && d != 256) << what << ": head_dim " << d << " is not built (64, 96, 128, 256)";
  KV_UNSUPPORTED(page_size <= 0 || page_size % kRun != 0) << what << ": page_size must be a multiple of 16, got " << page_size;
}

static void check_aligned(const char* what, std::initializer_list<const void*> data) {
  for (const void* p : data) KV_CHECK(reinterpret_cast<uintptr_t>(p) % 16 == 0) << what << ": data must be aligned to 16 bytes";
}

static dim3 blocks_for(const char* what, int64_t threads) {
  const int64_t blocks = (threads + 255) / 256;
  KV_CHECK(blocks < (int64_t{1} << 31)) << what << ": too many rows";
  return dim3(static_cast<unsigned>(blocks));
}

template <class Launch>
static void for_head_dim(int d, Launch&& launch) {
  switch (d) {
    case 64: launch(std::integral_constant<int, 64>{}); break;
    case 96: launch(std::integral_constant<int, 96>{}); break;
    case 128: launch(std::integral_constant<int, 128>{}); break;
    default: launch(std::integral_constant<int, 256>{}); break;
  }
}

static Mxfp4Params attn_params(const char* what, const void* q, const void* pages, const int32_t* page_indptr,
                               const int32_t* page_values, const int32_t* length_info, void* output, float* lse, double sm_scale,
                               int32_t batch, int64_t nnz_pages, int32_t h_q, int32_t h_kv, int32_t d, int32_t page_size,
                               int32_t sliding_window) {
  KV_CHECK(batch >= 0 && nnz_pages >= 0 && h_q > 0 && h_kv > 0 && h_q % h_kv == 0) << what << ": bad shape";
  check_mxfp4(what, h_kv, page_size, d);
  Mxfp4Params p = {};
  p.q = static_cast<const half_t*>(q);
  p.pages = static_cast<const uint8_t*>(pages);
  p.page_indptr = page_indptr;
  p.page_values = page_values;
  p.last_page_len = length_info;
  p.window_offset = sliding_window != 0 && length_info ? length_info + batch : nullptr;
  p.sink_size = sliding_window != 0 && length_info ? length_info + 2 * static_cast<int64_t>(batch) : nullptr;
  p.output = static_cast<half_t*>(output);
  p.lse = lse;
  p.batch = batch;
  p.h_q = h_q;
  p.h_kv = h_kv;
  p.group = h_q / h_kv;
  p.row_blocks = (p.group + 15) / 16;
  p.page_size = page_size;
  p.runs_per_page = page_size / kRun;
  p.run_magic = p.runs_per_page == 1 ? 0 : static_cast<uint32_t>(((uint64_t{1} << 32) + p.runs_per_page - 1) / p.runs_per_page);
  p.scale_log2 = static_cast<float>(sm_scale) * kLog2e;
  return p;
}

}  // namespace tvmkv

using namespace tvmkv;

extern "C" {

int tvmkv_mxfp4_append(void* pages, const void* k_data, const void* v_data, const int32_t* position_map, int64_t ntoken,
                       int64_t num_pages, int32_t num_kv_heads, int32_t page_size, int32_t head_dim, void* stream) {
  KV_API_BEGIN();
  check_mxfp4("mxfp4_append", num_kv_heads, page_size, head_dim);
  KV_CHECK(ntoken >= 0) << "mxfp4_append: bad shape";
  if (ntoken == 0) return TVMKV_OK;
  KV_CHECK(pages && k_data && v_data && position_map) << "mxfp4_append: NULL tensor";
  check_aligned("mxfp4_append", {pages, k_data, v_data});
  const int64_t rows = ntoken * 2 * num_kv_heads;
  hipLaunchKernelGGL(mxfp4_append_kernel, blocks_for("mxfp4_append", rows * (head_dim / 8)), dim3(256), 0, as_stream(stream),
                     static_cast<uint8_t*>(pages), static_cast<const half_t*>(k_data), static_cast<const half_t*>(v_data),
                     position_map, rows, num_kv_heads, page_size, head_dim);
  KV_LAUNCH_CHECK();
  KV_API_END();
}

int tvmkv_mxfp4_read_kv(const void* pages, const int32_t* position_map, void* k_data, void* v_data, int64_t ntoken,
                        int64_t num_pages, int32_t num_kv_heads, int32_t page_size, int32_t head_dim, void* stream) {
  KV_API_BEGIN();
  check_mxfp4("mxfp4_read_kv", num_kv_heads, page_size, head_dim);
  KV_CHECK(ntoken >= 0) << "mxfp4_read_kv: bad shape";
  if (ntoken == 0) return TVMKV_OK;
  KV_CHECK(pages && k_data && v_data && position_map) << "mxfp4_read_kv: NULL tensor";
  check_aligned("mxfp4_read_kv", {pages, k_data, v_data});
  const int64_t rows = ntoken * 2 * num_kv_heads;
  hipLaunchKernelGGL(mxfp4_read_kernel, blocks_for("mxfp4_read_kv", rows * (head_dim / 8)), dim3(256), 0, as_stream(stream),
                     static_cast<const uint8_t*>(pages), static_cast<half_t*>(k_data), static_cast<half_t*>(v_data), position_map,
                     rows, num_kv_heads, page_size, head_dim);
  KV_LAUNCH_CHECK();
  KV_API_END();
}

int tvmkv_mxfp4_batch_decode_paged_kv(const void* q, const void* pages, const int32_t* page_indptr, const int32_t* page_values,
                                      const int32_t* length_info, void* output, float* lse, double sm_scale, int32_t batch_size,
                                      int64_t nnz_pages, int64_t num_pages, int32_t h_q, int32_t h_kv, int32_t head_dim,
                                      int32_t page_size, int32_t sliding_window, void* stream) {
  KV_API_BEGIN();
  const char* const what = "mxfp4_batch_decode_paged_kv";
  Mxfp4Params p = attn_params(what, q, pages, page_indptr, page_values, length_info, output, lse, sm_scale, batch_size, nnz_pages,
                              h_q, h_kv, head_dim, page_size, sliding_window);
  if (batch_size == 0) return TVMKV_OK;
  KV_CHECK(q && pages && page_indptr && length_info && output && lse) << what << ": NULL tensor";
  KV_CHECK(nnz_pages == 0 || page_values) << what << ": NULL page table";
  check_aligned(what, {q, pages, output});
  // chunks: about six work items for every compute unit, at least one step of the four waves
  const int64_t runs = nnz_pages * p.runs_per_page;
  const int64_t wanted = std::max<int64_t>(1, 6 * compute_units() / (static_cast<int64_t>(h_kv) * p.row_blocks));
  p.chunk_runs = static_cast<int>(std::min<int64_t>(std::max<int64_t>((runs + wanted - 1) / wanted, 8) + 7, 1 << 20) / 8 * 8);
  const int64_t slots = runs / p.chunk_runs + batch_size;
  const int64_t items = slots * h_kv * p.row_blocks;
  KV_CHECK(items < (int64_t{1} << 31)) << what << ": too many work items";
  const hipStream_t s = as_stream(stream);
  const size_t o_bytes = static_cast<size_t>(slots) * h_q * head_dim * sizeof(float);
  const ScratchLease ws = lease_scratch(kScratchMxfp4, s, o_bytes + static_cast<size_t>(slots) * h_q * 2 * sizeof(float), 0);
  p.part_o = reinterpret_cast<float*>(ws.ptr);
  p.part_ml = reinterpret_cast<float*>(ws.ptr + o_bytes);
  for_head_dim(head_dim, [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    hipLaunchKernelGGL((mxfp4_attn_kernel<D, false>), dim3(static_cast<unsigned>(items)), dim3(256), 0, s, p);
    KV_LAUNCH_CHECK();
    hipLaunchKernelGGL(mxfp4_merge_kernel<D>, dim3((batch_size * h_q + 3) / 4), dim3(256), 0, s, p);
    KV_LAUNCH_CHECK();
  });
  KV_API_END();
}

int tvmkv_mxfp4_batch_prefill_paged_kv(const void* q, const int32_t* q_indptr, const void* pages, const int32_t* page_indptr,
                                       const int32_t* page_values, const int32_t* length_info, void* output, float* lse,
                                       int64_t causal, double sm_scale, int32_t batch_size, int64_t total_q, int64_t nnz_pages,
                                       int64_t num_pages, int32_t h_q, int32_t h_kv, int32_t head_dim, int32_t page_size,
                                       int32_t sliding_window, void* stream) {
  KV_API_BEGIN();
  const char* const what = "mxfp4_batch_prefill_paged_kv";
  Mxfp4Params p = attn_params(what, q, pages, page_indptr, page_values, length_info, output, lse, sm_scale, batch_size, nnz_pages,
                              h_q, h_kv, head_dim, page_size, sliding_window);
  KV_CHECK(total_q >= 0) << what << ": bad shape";
  if (batch_size == 0 || total_q == 0) return TVMKV_OK;
  KV_CHECK(q && q_indptr && pages && page_indptr && length_info && output && lse) << what << ": NULL tensor";
  KV_CHECK(nnz_pages == 0 || page_values) << what << ": NULL page table";
  check_aligned(what, {q, pages, output});
  p.q_indptr = q_indptr;
  p.causal = causal != 0;
  const int64_t items = (total_q * p.group / 16 + batch_size) * h_kv;
  KV_CHECK(items < (int64_t{1} << 31)) << what << ": too many work items";
  const hipStream_t s = as_stream(stream);
  for_head_dim(head_dim, [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    hipLaunchKernelGGL((mxfp4_attn_kernel<D, true>), dim3(static_cast<unsigned>(items)), dim3(256), 0, s, p);
    KV_LAUNCH_CHECK();
  });
  KV_API_END();
}

}  // extern "C"
