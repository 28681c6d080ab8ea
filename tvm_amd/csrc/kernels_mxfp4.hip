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
#include "exact_division.h"

namespace tvmkv {

constexpr int kRun = 16;            // tokens the attention kernels take from a page at a time
constexpr float kNoKey = -1e30f;    // running maximum of a row that has seen no key
constexpr float kEmptyLse = -5e4f;  // log-sum-exp of a row without keys (its output is 0)

typedef uint32_t uint32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint32x3_t __attribute__((ext_vector_type(3), aligned(4)));
typedef uint32_t uint32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// eight codes -> eight fp16
__device__ __forceinline__ half8_t dequantise8(uint32_t codes, float scale) {
  const half2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0);
  const half2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1);
  const half2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2);
  const half2_t d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3);
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Where a thread of the append and the read kernel is: it has 8 elements of K and of V of a (token, head), its neighbours
// the next 8, then come the other tokens of 16, then the heads: the tokens of a call mostly follow one another in their
// pages, where the codes of a head's tokens do, so that a workgroup's part of the cache is whole lines.  32 bits: the
// launchers cut calls of more than 2^30 threads into several.
struct RowPiece {
  bool there;
  uint32_t piece;    // of 8 elements
  uint64_t at;       // of its elements in the fp16 rows
  int32_t position;  // slot of the token
  uint8_t* k;        // slab of the page's K and of its V
  uint8_t* v;
  uint32_t codes, scale;  // offsets of the piece's codes and of its block's scale
};
template <int D>
__device__ __forceinline__ RowPiece row_piece(uint8_t* pages, const int32_t* position_map, uint32_t tokens, uint32_t h_kv, uint32_t page_size) {
  constexpr uint32_t kPieces = D / 8;
  const uint32_t gid = blockIdx.x * 256 + threadIdx.x;
  RowPiece x;
  const uint32_t row = gid / kPieces, sixteen = (row / 16) / h_kv, head = row / 16 - sixteen * h_kv;
  x.piece = gid % kPieces;
  x.there = sixteen * 16 + row % 16 < tokens;
  const uint32_t token = min(sixteen * 16 + row % 16, tokens - 1);
  x.at = (static_cast<uint64_t>(token) * h_kv + head) * D + x.piece * 8;
  x.position = position_map[token];
  const uint32_t at = max(x.position, 0), page = at / page_size, slot = at - page * page_size;
  const uint32_t slab = page_size * (17 * D / 32);
  x.k = pages + (static_cast<uint64_t>(page) * 2 * h_kv + head) * slab;
  x.v = x.k + static_cast<uint64_t>(h_kv) * slab;
  x.codes = slot * (D / 2) + x.piece * 4;
  x.scale = page_size * (D / 2) + slot * (D / 32) + x.piece / 4;
  return x;
}

// ------------------------------------------------------------------------------------------
// append: k|v[i, h, :] -> slot position_map[i] (negative: none).  The four lanes of a block share its largest
// magnitude; as 16-bit integers magnitudes order like the values, infinities and NaN above all others.  Bound by its
// bytes, 2 D read and 17 D / 32 written per row: 19 000 tokens with 8 heads of dim 128 in 21.5 us, 4.6 TB/s.  (The rows
// are read once, with the streaming hint: without it 24.9.)
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ void quantise8(const Vec16& x, uint32_t piece, uint32_t* codes_at, uint8_t* scale_at) {
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
  *codes_at = finite ? codes : 0;
  if ((piece & 3) == 0) *scale_at = finite ? byte : 255;
}

template <int D>
__global__ __launch_bounds__(256) void mxfp4_append_kernel(uint8_t* __restrict__ pages, const half_t* __restrict__ k_data,
                                                           const half_t* __restrict__ v_data,
                                                           const int32_t* __restrict__ position_map, uint32_t tokens, uint32_t h_kv,
                                                           uint32_t page_size) {
  const RowPiece x = row_piece<D>(pages, position_map, tokens, h_kv, page_size);
  const Vec16 k = ld16_nt(k_data + x.at), v = ld16_nt(v_data + x.at);
  if (!x.there || x.position < 0) return;  // whole blocks: four lanes have the same token
  quantise8(k, x.piece, reinterpret_cast<uint32_t*>(x.k + x.codes), x.k + x.scale);
  quantise8(v, x.piece, reinterpret_cast<uint32_t*>(x.v + x.codes), x.v + x.scale);
}

// ------------------------------------------------------------------------------------------
// read: slot position_map[i] -> k|v[i, h, :] in fp16, exact; a negative position gives zeros.  Bound by its bytes: the same
// tokens in 15.7 us, 6.3 TB/s (stores without the streaming hint 16.2, 64 sequences of 100-600 tokens 20.4 and 23.0).
// ------------------------------------------------------------------------------------------
template <int D>
__global__ __launch_bounds__(256) void mxfp4_read_kernel(const uint8_t* __restrict__ pages, half_t* __restrict__ k_data,
                                                         half_t* __restrict__ v_data,
                                                         const int32_t* __restrict__ position_map, uint32_t tokens, uint32_t h_kv,
                                                         uint32_t page_size) {
  const RowPiece x = row_piece<D>(const_cast<uint8_t*>(pages), position_map, tokens, h_kv, page_size);
  Vec16 k = zero16(), v = zero16();
  if (x.position >= 0) {
    const uint32_t k_codes = *reinterpret_cast<const uint32_t*>(x.k + x.codes), v_codes = *reinterpret_cast<const uint32_t*>(x.v + x.codes);
    const uint32_t k_scale = x.k[x.scale], v_scale = x.v[x.scale];
    k.h8 = dequantise8(k_codes, scale_of(k_scale));
    v.h8 = dequantise8(v_codes, scale_of(v_scale));
  }
  if (!x.there) return;
  __builtin_nontemporal_store(__builtin_bit_cast(uint32x4_t, k), reinterpret_cast<uint32x4_t*>(k_data + x.at));
  __builtin_nontemporal_store(__builtin_bit_cast(uint32x4_t, v), reinterpret_cast<uint32x4_t*>(v_data + x.at));
}

// ------------------------------------------------------------------------------------------
// Attention.  With s = sm_scale log2(e) q.k the output of a row is sum 2^(s - m) v / sum 2^(s - m) and its
// log-sum-exp (base 2) m + log2(sum), for any m; sums, statistics and outputs in float32, the weights rounded to fp16
// for the second matrix product (11 bits, as the output itself).  Their sum is of the weights before that rounding: outputs are
// off by 2.4e-4 to 3e-4 of their root mean square, 2.0e-4 of it the output's own rounding; the sum of the rounded weights gives
// 2.4e-4, and cost 5 % of prefill.
//
// A row of a kv head is (query token, query head of its group), token-major.  A workgroup of four waves takes up to
// 16 RB rows of a kv head and a range of the sequence's keys, a wave every fourth step of 32 keys (two runs of 16
// tokens; page sizes are multiples of 16, so a run lies in one page):
//   S^T[token, row] = K Q^T    the lane (token, quarter of the row) loads its codes straight from memory, turns
//                              them into fp16 in registers and has the matrix instruction's A operand: the order of
//                              the contraction is free, q is loaded in the same one;
//   O^T[d, row]     = V^T P^T  V is turned into fp16 the same way and put into the wave's LDS tile, from where the
//                              transposing read takes it; P stays in registers.  Decode loads it in the order of memory
//                              (sixteen lanes touch 256 bytes instead of 16 rows: 10 % of a launch at head dim 64);
//                              prefill, which waits for LDS rather than for memory, as K (at head dim 64 the other order
//                              writes with conflicts, 13 % slower).
// The codes of a wave's next step are on their way while it works on one.
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
  // states of work items that have only some of a row's keys: (slot, row block, kv head, row of the block)
  float* part_o;   // D each, not normalised
  float* part_ml;  // reference point, sum
  unsigned long long* arrivals;  // of the work items of some rows: epoch << 32 | those that have delivered their states
  int batch;
  int h_q;
  int h_kv;
  int group;
  int row_blocks;  // of a sequence with one query token
  int causal;
  int page_size;
  uint32_t runs_per_page;
  ExactDivision page_of_run;  // by runs_per_page
  float inv_group;
  uint32_t chunk_runs;  // decode: most keys of a work item, in runs; a multiple of 8
  int fit_items;        // decode: > 0: chunks as short as leave so many items a row block and kv head, chunk_runs at most
  uint32_t whole_runs;  // decode: where no sequence has more runs than these, sequences are left whole
  int shares;           // prefill: work items that share the keys of a row block
  uint32_t epoch;       // of the launch, if its work items share rows
  float scale_log2;     // > 0: |sm_scale| log2(e), never 0
  uint32_t q_sign;      // of sm_scale, at the sign bits of two fp16
};

// Sum of x over the lanes up to this one.
__device__ __forceinline__ int prefix_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // from 1, 2, 4 and 8 lanes below in the row of 16
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // the row below's last to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31's to rows 2 and 3
  return x;
}

// The sequence of a work item, and what the arrays hold for it.  Sequence i has items_of(entries of indptr i, i + 1) work
// items, one behind the other without gaps: the launch has more workgroups than items, since only the device knows the
// lengths, and spare ones between the others put the real ones on some of the compute units (64 sequences of 4096 tokens, 512
// items: 79 us with a spare one beside every real one, 50 without).  The wave adds the items up, a sequence a lane, or up
// to 8 neighbours a lane; with more sequences each has a fixed range of items instead, spare_begin(i, indptr[i] - indptr[0]) onwards, and
// the wave looks for the last that begins at or before the slot.
struct Sequence {
  int index, begin;  // begin: its first work item
  int page_begin, num_pages, last_page_len, sink, window;
  int q_begin, q_len;
};
template <bool PREFILL, class Items, class Begin>
__device__ __forceinline__ Sequence sequence_of(const Mxfp4Params& p, int slot, int lane, Items items_of, Begin spare_begin) {
  const int32_t* const indptr = PREFILL ? p.q_indptr : p.page_indptr;
  int at, begin, who;  // who: the lane that has the sequence's values
  bool found = true;
  if (p.batch > 64) {
    if (p.batch <= 512) {
      const int each = (p.batch + 63) >> 6;
      int x[9], count = 0;
#pragma unroll
      for (int j = 0; j <= 8; ++j) x[j] = indptr[min(lane * each + min(j, each), p.batch)];
#pragma unroll
      for (int j = 0; j < 8; ++j) count += j < each && lane * each + j < p.batch ? items_of(x[j], x[j + 1]) : 0;
      const int upto = prefix_sum(count);
      const int lanes = __popcll(__ballot(upto <= slot));
      found = lanes < 64;
      const int owner = min(lanes, 63);
      begin = __builtin_amdgcn_readlane(upto - count, owner);
      int n = owner * each;
      bool here = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int count_j = items_of(__builtin_amdgcn_readlane(x[j], owner), __builtin_amdgcn_readlane(x[j + 1], owner));
        here |= begin + count_j > slot || j + 1 >= each || n + 1 >= p.batch;
        begin += here ? 0 : count_j;
        n += here ? 0 : 1;
      }
      at = min(n, p.batch - 1);
    } else {
      int lo = 0, n = p.batch;
      const int base = indptr[0];  // (of a part of a larger table it need not be 0)
      while (n > 1) {
        const int stride = (n + 63) >> 6;
        const int i = lo + lane * stride;
        const bool hit = i < lo + n && spare_begin(i, indptr[i] - base) <= slot;
        const int first = lo + (max(static_cast<int>(__popcll(__ballot(hit))), 1) - 1) * stride;
        n = min(stride, lo + n - first);
        lo = first;
      }
      at = lo;
      begin = spare_begin(at, indptr[at] - base);
    }
    who = 0;
  } else {
    at = min(lane, p.batch - 1);
  }
  const int page = p.page_indptr[at], next_page = p.page_indptr[at + 1], last = p.last_page_len[at];
  const int sink = p.sink_size != nullptr ? p.sink_size[at] : 0, window = p.window_offset != nullptr ? p.window_offset[at] : 0;
  const int q = PREFILL ? p.q_indptr[at] : at, next_q = PREFILL ? p.q_indptr[at + 1] : at + 1;
  if (p.batch <= 64) {
    const int count = lane < p.batch ? (PREFILL ? items_of(q, next_q) : items_of(page, next_page)) : 0;
    int mine;  // the lane's first item
    if constexpr (PREFILL) {
      // the sequences with the most keys first, so that the last items to start are short ones (eight chunks on up to 4096
      // cached tokens 321 -> 307 us)
      const int key = min(next_page - page, (1 << 24) - 1) * 64 + 63 - lane;  // (unlike from lane to lane)
      mine = 0;
      for (int j = 0; j < p.batch; ++j) mine += __builtin_amdgcn_readlane(key, j) > key ? __builtin_amdgcn_readlane(count, j) : 0;
    } else {
      mine = prefix_sum(count) - count;
    }
    const uint64_t hit = __ballot(slot >= mine && slot < mine + count);
    found = hit != 0;
    who = found ? __ffsll(static_cast<long long>(hit)) - 1 : 0;
    begin = __builtin_amdgcn_readlane(mine, who);
  }
  const auto of = [&](int x) { return __builtin_amdgcn_readlane(x, who); };
  const int index = p.batch <= 64 ? who : __builtin_amdgcn_readfirstlane(at);
  Sequence s = {found ? index : -1, __builtin_amdgcn_readfirstlane(begin), of(page), of(next_page) - of(page), of(last), of(sink), of(window), of(q), of(next_q) - of(q)};
  if (s.num_pages == 0) s.sink = s.window = 0;
  return s;
}

// A global address that is the same in every lane.  (The address space is spelled out: behind the lane reads the compiler
// no longer knows it, and flat loads are waited for together with LDS reads.)
typedef __attribute__((address_space(1))) const uint8_t* global_bytes_t;
__device__ __forceinline__ global_bytes_t uniform_bytes(const uint8_t* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return reinterpret_cast<global_bytes_t>(static_cast<uint64_t>(hi) << 32 | lo);
}
// ONCE: the codes are read by one work item only and streamed through the caches (a plain read of a large array reaches
// 6.2 TB/s here, one with the streaming hint 6.9).  The scales are not, whose 64 bytes share a line with others' codes.
template <class T, bool ONCE = false>
__device__ __forceinline__ T load_global(global_bytes_t base, uint32_t offset) {
  const auto at = reinterpret_cast<__attribute__((address_space(1))) const T*>(base + offset);
  return ONCE ? __builtin_nontemporal_load(at) : *at;
}

// What a lane holds of a row: D / 4 elements in chunks of 8, and the scales of their blocks.  The lane group g4
// (0..3) has consecutive chunks, at head dim 256 four of either half of the row.
template <int D>
struct LaneRow {
  static constexpr int CH = D / 32;                       // chunks
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
  // codes, scales: of the run's first token
  template <bool ONCE>
  __device__ __forceinline__ void load(global_bytes_t codes, global_bytes_t scales, uint32_t token, uint32_t g4) {
    if constexpr (D == 64) {
      const auto x = load_global<uint32x2_t, ONCE>(codes, token * (D / 2) + g4 * 8);
      w[0] = x[0];
      w[1] = x[1];
    } else if constexpr (D == 96) {
      const auto x = load_global<uint32x3_t, ONCE>(codes, token * (D / 2) + g4 * 12);
#pragma unroll
      for (int c = 0; c < CH; ++c) w[c] = x[c];
    } else {
#pragma unroll
      for (int i = 0; i < D / 128; ++i) {
        const auto x = load_global<uint32x4_t, ONCE>(codes, token * (D / 2) + g4 * 16 + i * 64);
#pragma unroll
        for (int c = 0; c < 4; ++c) w[i * 4 + c] = x[c];
      }
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) s[i] = load_global<uint8_t>(scales, token * (D / 32) + block(g4, i));
  }
  __device__ __forceinline__ half8_t values(int g4, int c) const {
    const int i = scale_index(g4, c);
    return dequantise8(w[c], scale_of(NS == 1 ? s[0] : (i ? s[NS - 1] : s[0])));
  }
};

// Device-scope accesses: the states of a row's work items, which other XCDs may have written (each has its own L2).
constexpr int kDeviceScope = 16;  // the sc1 bit of a buffer access
struct SharedStates {
  __amdgpu_buffer_rsrc_t at;
  __device__ __forceinline__ SharedStates(float* base) : at(__builtin_amdgcn_make_buffer_rsrc(base, 0, -1, 0x00027000)) {}
  __device__ __forceinline__ void store4(uint32_t offset, float4_t v) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uint32x4_t, v), at, offset * 4, 0, kDeviceScope);
  }
  __device__ __forceinline__ void store2(uint32_t offset, float a, float b) {
    __builtin_amdgcn_raw_buffer_store_b64(uint32x2_t{__float_as_uint(a), __float_as_uint(b)}, at, offset * 4, 0, kDeviceScope);
  }
  __device__ __forceinline__ float4_t load4(uint32_t offset) const {
    return __builtin_bit_cast(float4_t, __builtin_amdgcn_raw_buffer_load_b128(at, offset * 4, 0, kDeviceScope));
  }
  __device__ __forceinline__ float2 load2(uint32_t offset) const {
    const uint32x2_t v = __builtin_amdgcn_raw_buffer_load_b64(at, offset * 4, 0, kDeviceScope);
    return make_float2(__uint_as_float(v[0]), __uint_as_float(v[1]));
  }
};

// Halfs of a row of a wave's V tile in LDS.  Sixteen lanes write the same 16 bytes of the 16 rows of a run, sixteen lanes
// of the transposing read take 32 bytes of four consecutive rows: at 12, 36 or 52 banks (of 64) from row to row neither
// meets a bank twice.  (At 8 banks the writes did, and a third of the tile's LDS cycles were conflicts.)
constexpr int v_row(int d) { return d == 64 || d == 96 ? d + 8 : d + 24; }

// Workgroups of a compute unit, four waves each, that a work item of rb blocks of 16 rows leaves registers for: the bound that the
// kernels are compiled for, and what the rules below count on.  At head dim 64 the compiler needs fewer (126 registers for two
// blocks, 163 to 167 for three), so that the hardware holds one more there; the rules' times were measured so.
constexpr int mxfp4_waves(int d, int rb) { return d == 256 ? 2 : rb == 1 ? 4 : d == 64 && rb == 2 ? 3 : 2; }

template <int D, int RB, bool PREFILL, bool ONCE>
__global__ __launch_bounds__(256, mxfp4_waves(D, RB)) void mxfp4_attn_kernel(Mxfp4Params p) {
  constexpr int CH = LaneRow<D>::CH;
  constexpr int DB = D / 16;
  constexpr int R = 16 * RB;
  constexpr int VH = D > 128 ? 2 : 1;  // V goes through the wave's tile in halves of 128 columns
  constexpr int VW = D / VH;
  constexpr int VS = v_row(VW);
  static_assert(32 * VS * sizeof(half_t) >= 16 * VW * sizeof(float), "the merge buffer takes the V tile's place");
  // Head dim 256 with two blocks of rows: two waves a SIMD, with q in LDS and one step's codes at a time in registers, the next
  // ones loaded as soon as they are used up (one wave a SIMD: 540 TFLOP/s instead of 729).  256 registers do not hold all of the
  // rest: prefill keeps 15 values in scratch memory, decode 22.
  constexpr bool LEAN = D == 256 && RB == 2;
  constexpr int kJoinBytes = (R * 64 + 4 * R) * sizeof(float) + 256 * sizeof(float4_t);  // the join of states, below
  constexpr int kTileHalfs = std::max<int>(32 * VS, kJoinBytes / 8);
  __shared__ __attribute__((aligned(16))) half_t v_tiles[4][kTileHalfs];
  __shared__ half8_t q_lds[LEAN ? RB * CH * 64 : 1];
  __shared__ float sm_m[4][16], sm_l[4][16];
  __shared__ int sm_last;

  // The arguments in one trip; read where they are used they are a dozen, one behind the other.
  asm volatile("" ::"s"(p.q), "s"(p.pages), "s"(p.page_indptr), "s"(p.page_values), "s"(p.last_page_len), "s"(p.batch), "s"(p.h_q),
               "s"(p.h_kv), "s"(p.group), "s"(p.page_size), "s"(p.runs_per_page), "s"(p.page_of_run.magic), "s"(p.page_of_run.shift),
               "s"(p.page_of_run.mask), "s"(p.scale_log2), "s"(p.q_sign));
  if constexpr (PREFILL) asm volatile("" ::"s"(p.q_indptr), "s"(p.causal), "s"(p.shares));
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int c16 = lane & 15;
  const int g4 = lane >> 4;
  const int v_token = PREFILL ? c16 : lane >> 2, v_quarter = PREFILL ? g4 : lane & 3;  // what the lane loads of V

  // ---- which rows, which keys ----------------------------------------------------------------
  const int kvh = blockIdx.x % p.h_kv;
  const int blocks = PREFILL ? 1 : p.row_blocks;
  const int slot = blockIdx.x / (p.h_kv * blocks);
  // Decode: items for a sequence's chunks, by what its pages could hold, and one for a sequence without pages (the launcher
  // makes sure that the runs of all pages are a 31-bit number).  Prefill: items for the blocks of its rows.
  // Two items a compute unit, started together, are what large launches run best with, and only the device has the lengths.
  uint32_t chunk_runs = p.chunk_runs;
  if (!PREFILL && (p.whole_runs > 0 || p.fit_items > 0)) {
    const int i = min(lane, p.batch - 1);
    const uint32_t runs = static_cast<uint32_t>(p.page_indptr[i + 1] - p.page_indptr[i]) * p.runs_per_page;
    if (p.whole_runs > 0) {
      const uint32_t longest = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(wave_max(static_cast<float>(runs))));
      if (longest <= p.whole_runs) chunk_runs = max(chunk_runs, (longest + 7) & ~7u);
    } else {
      // five halvings of what lies between one item for every sequence and an equal share of all keys, in steps
      const uint32_t own = lane < p.batch ? runs : 0;
      const uint32_t total = __builtin_amdgcn_readlane(prefix_sum(static_cast<int>(own)), 63);
      uint32_t lo = min(total / (8 * p.fit_items), chunk_runs / 8 - 1), hi = chunk_runs / 8;
      for (int k = 0; k < 5 && hi - lo > 1; ++k) {
        const uint32_t mid = (lo + hi) / 2;
        // (a rounded-up quotient more than an item holds is only one item too many)
        const int items = lane < p.batch ? max(static_cast<int>(ceilf(static_cast<float>(own) * (1.0000005f / static_cast<float>(8 * mid)))), 1) : 0;
        const bool fits = static_cast<int>(__builtin_amdgcn_readlane(prefix_sum(items), 63)) <= p.fit_items;
        hi = fits ? mid : hi;
        lo = fits ? lo : mid;
      }
      chunk_runs = hi * 8;
    }
  }
  const auto chunks_of = [&](int pages) {
    return max(static_cast<int>((static_cast<uint32_t>(pages) * p.runs_per_page + chunk_runs - 1) / chunk_runs), 1);
  };
  const Sequence seq = sequence_of<PREFILL>(
      p, slot, lane,
      [&](int first, int end) {
        if constexpr (PREFILL) return static_cast<int>((static_cast<int64_t>(end - first) * p.group + R - 1) / R);
        return chunks_of(end - first);
      },
      [&](int i, int first) {
        if constexpr (PREFILL) return static_cast<int>(static_cast<int64_t>(first) * p.group / R) + i;
        return static_cast<int>(static_cast<uint32_t>(first) * p.runs_per_page / chunk_runs) + i;
      });
  if (seq.index < 0) return;  // a spare slot
  const int b = seq.index, page_begin = seq.page_begin, window = seq.window;
  const int stored = seq.num_pages > 0 ? (seq.num_pages - 1) * p.page_size + seq.last_page_len : 0;
  const int sink = min(seq.sink, stored);  // (so that no key is looked for behind the stored ones)
  const int keys = stored - window + sink;
  const int q_begin = seq.q_begin, q_len = seq.q_len;
  const int rows = q_len * p.group;
  const int block = PREFILL ? slot - seq.begin : blockIdx.x / p.h_kv % blocks;
  const int row0 = block * R;
  if (row0 >= rows) return;  // a spare slot
  const int rows_here = min(R, rows - row0);
  // Rows: the token and head of row0, then small numbers, which a product with 1 / group divides exactly.
  const int token0 = row0 / p.group, head0 = row0 - token0 * p.group;
  const auto token_of = [&](int r) { return static_cast<int>((static_cast<float>(head0 + r) + 0.5f) * p.inv_group); };  // from token0 on
  // stored tokens [0, end) hold the first n keys; token t of them is one iff t < sink or t >= window
  const auto end_of = [&](int n) { return n <= sink ? n : n - sink + window; };
  const auto end_of_row = [&](int token) { return end_of(p.causal ? min(max(keys - q_len + 1 + token, 0), keys) : keys); };
  const int first_end = end_of_row(token0);                             // every row sees the keys in front of it
  const int last_end = end_of_row(token0 + token_of(rows_here - 1));  // no row sees a key behind it
  const int all_runs = (last_end + kRun - 1) / kRun;
  const int chunk = PREFILL ? static_cast<int>(blockIdx.z) : slot - seq.begin;
  // chunks of one length: whole ones and a rest end at different times (64 sequences of 1024-8192 tokens: 62 us, 57 so)
  const int most_chunks = PREFILL ? p.shares : chunks_of(seq.num_pages);
  const int per_chunk = ((all_runs + most_chunks - 1) / most_chunks + 7) & ~7;
  const int chunks = all_runs > per_chunk ? (all_runs + per_chunk - 1) / per_chunk : 1;
  if (chunk >= chunks) return;
  const int run_lo = chunk * per_chunk;
  const int run_hi = min(all_runs, run_lo + per_chunk);

  // Where the codes and the scales of the wave's next 64 steps are, a step a lane: of its two runs' K, in units of 16 bytes
  // (slabs are a multiple of that, and so are a run's codes and scales).
  const uint32_t slab16 = static_cast<uint32_t>(p.page_size) / kRun * (17 * D / 32);
  uint32_t codes16[2], scales16[2];
  const auto sign_q = [&](half8_t q) {
    Vec16 x;
    x.h8 = q;
#pragma unroll
    for (int i = 0; i < 4; ++i) x.w[i] ^= p.q_sign;
    return x.h8;
  };
  const auto load_ids = [&](int run) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t at = min(run + 8 * lane + h, run_hi - 1);
      const uint32_t nth = p.page_of_run(at);
      codes16[h] = p.page_values[page_begin + nth];
      scales16[h] = at - nth * p.runs_per_page;
    }
  };
  const auto place_ids = [&]() {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t slab = (codes16[h] * 2u * p.h_kv + kvh) * slab16, in_page = scales16[h];
      codes16[h] = slab + in_page * (D / 2);
      scales16[h] = slab + p.runs_per_page * (D / 2) + in_page * (D / 32);
    }
  };
  int run = run_lo + 2 * wave;
  const bool works = run < run_hi;
  int my_end[RB];
  half8_t qf[LEAN ? 1 : RB][LEAN ? 1 : CH];
  const auto load_q = [&]() {
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const int row = min(r * 16 + c16, rows_here - 1);  // (a row that isn't there computes as the last one and is not written)
      const int token = token_of(row);
      my_end[r] = PREFILL ? end_of_row(token0 + token) : last_end;
      const half_t* q = p.q + (static_cast<int64_t>(q_begin + token0 + token) * p.h_q + kvh * p.group + head0 + row - token * p.group) * D;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (LEAN && (r * CH + c) % 4 != wave) continue;
        const half8_t x = ld16(q + LaneRow<D>::chunk(g4, c) * 8).h8;
        if constexpr (LEAN) q_lds[(r * CH + c) * 64 + lane] = sign_q(x);
        else qf[r][c] = x;
      }
    }
  };
  float4_t o[RB][DB];
  float m[RB], l[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
#pragma unroll
    for (int i = 0; i < DB; ++i) o[r][i] = float4_t{0.f, 0.f, 0.f, 0.f};
    m[r] = kNoKey;
    l[r] = 0.f;
  }
  if constexpr (LEAN) {
    load_q();
    __syncthreads();
  }
  const auto q_at = [&](int r, int c) {
    if constexpr (LEAN) return q_lds[(r * CH + c) * 64 + lane];
    else return qf[r][c];
  };
  uint32_t poisoned[RB] = {};  // 32-element parts of the output that are NaN, see below

  half_t* const vt = v_tiles[wave];
  struct Step {
    LaneRow<D> k[2], v[2];
  };
  const global_bytes_t pool = uniform_bytes(p.pages);
  const uint32_t v_slab = slab16 * p.h_kv * 16;  // from K to V of a page
  const auto load = [&](int nth, Step& x, bool want_k, bool want_v) {  // of the nth step of the 64 whose pages are here
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      global_bytes_t k = pool + static_cast<uint64_t>(__builtin_amdgcn_readlane(codes16[h], nth)) * 16;
      global_bytes_t k_scales = pool + static_cast<uint64_t>(__builtin_amdgcn_readlane(scales16[h], nth)) * 16;
      global_bytes_t v = k + v_slab, v_scales = k_scales + v_slab;
      // kept in scalar registers: added up with the lanes' offsets first, they cost a 64-bit vector addition a load
      asm volatile("" : "+s"(k), "+s"(v), "+s"(k_scales), "+s"(v_scales));
      if (want_k) x.k[h].template load<ONCE>(k, k_scales, c16, g4);
      if (want_v) x.v[h].template load<ONCE>(v, v_scales, v_token, v_quarter);
    }
  };
  const auto work = [&](int t0, Step& x, int next) {  // next: the step that takes this one's place (LEAN)
    const bool whole = t0 + 2 * kRun <= first_end && (t0 >= window || t0 + 2 * kRun <= sink);  // no key of the step is masked
    float4_t s[RB][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int r = 0; r < RB; ++r) s[r][h] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const half8_t a = x.k[h].values(g4, c);
#pragma unroll
        for (int r = 0; r < RB; ++r) s[r][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q_at(r, c), s[r][h], 0, 0, 0);
      }
    }
    if (LEAN) load(next, x, true, false);
    if (!whole) {
#pragma unroll
      for (int r = 0; r < RB; ++r) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int t = t0 + h * kRun + 4 * g4 + i;
            const bool sees = (t < my_end[r]) & ((t < sink) | (t >= window));
            s[r][h][i] = sees ? s[r][h][i] : -INFINITY;
          }
        }
      }
      // A weight of 0 times NaN is NaN: what no row of the item sees is read as 0, and blocks that are NaN reach
      // the rows that see them by a mark of their own.
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = t0 + h * kRun + v_token;
        const bool seen = (t < last_end) & ((t < sink) | (t >= window));
#pragma unroll
        for (int i = 0; i < LaneRow<D>::NS; ++i) {
          const bool nan = seen && x.v[h].s[i] == 255;
          for (uint64_t left = __ballot(nan); left != 0; left &= left - 1) {
            const int who = __ffsll(static_cast<long long>(left)) - 1;
            const int at = t0 + h * kRun + (PREFILL ? who & 15 : who >> 2);
#pragma unroll
            for (int r = 0; r < RB; ++r) {
              if (at < my_end[r]) poisoned[r] |= 1u << LaneRow<D>::block(PREFILL ? who >> 4 : who & 3, i);
            }
          }
          if (nan || !seen) x.v[h].s[i] = 0;
        }
      }
    }
    const auto write_v = [&](int half) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int c = half * (CH / VH); c < (half + 1) * (CH / VH); ++c)
          *reinterpret_cast<half8_t*>(vt + (h * kRun + v_token) * VS + LaneRow<D>::chunk(v_quarter, c) * 8 - half * VW) = x.v[h].values(v_quarter, c);
      }
    };
    write_v(0);
    // Weights: the lane has 8 of the step's 32 keys of its row.  The reference point only has to keep them in fp16's
    // range: it moves when the row's maximum is 2^14 above it, to 2^-6 of that, and mostly stays after the first
    // steps, so that O is seldom rescaled; weights far below the maximum stay out of fp16's subnormal range.
    half8_t pf[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      float e[8], top = 0.f;
      const auto exponents = [&]() {
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = fmaf(s[r][i / 4][i % 4], p.scale_log2, -m[r]);
      };
      const auto highest = [&]() {
        top = s[r][0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, s[r][i / 4][i % 4]);
        top = max_xor32(max_xor16(top)) * p.scale_log2;
      };
      // Prefill, which the vector ALU holds up, takes the maximum of the exponents: one of what comes from a matrix instruction
      // costs another instruction a score (the compiler quiets it first; head dim 64 730 -> 773 TFLOP/s).  Decode has no register
      // for it.
      bool moves;
      if constexpr (PREFILL) {
        exponents();
        float over = e[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) over = fmaxf(over, e[i]);
        moves = max_xor32(max_xor16(over)) > 14.f;
      } else {
        highest();
        moves = top > m[r] + 14.f;
      }
      if (__ballot(moves) != 0) {
        if constexpr (PREFILL) highest();
        const float to = moves ? top - 6.f : m[r];
        const float alpha = fast_exp2(m[r] - to);
        m[r] = to;
        l[r] *= alpha;
#pragma unroll
        for (int i = 0; i < DB; ++i) o[r][i] *= alpha;
        if constexpr (PREFILL) exponents();
      }
      if constexpr (!PREFILL) exponents();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = fast_exp2(e[i]);
        l[r] += w;
        pf[r][i] = static_cast<half_t>(w);
      }
    }
#pragma unroll
    for (int half = 0; half < VH; ++half) {
      if (half > 0) write_v(half);
      if (LEAN && half == VH - 1) load(next, x, false, true);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = half * (DB / VH); i < (half + 1) * (DB / VH); ++i) {
        const half_t* src = vt + (4 * g4 + (c16 >> 2)) * VS + i * 16 - half * VW + (c16 & 3) * 4;
        const half4_t lo = lds_read_tr16(src), hi = lds_read_tr16(src + kRun * VS);
        const half8_t a = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
        for (int r = 0; r < RB; ++r) o[r][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pf[r], o[r][i], 0, 0, 0);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  };
  if (works) {
    // Page ids, q, then codes, each waited for when the next are on their way.
    load_ids(run);
    if constexpr (!LEAN) load_q();
    __builtin_amdgcn_sched_barrier(0);
    place_ids();
    // Two steps in flight, and every load is issued whether or not its step exists (past the end the last run is loaded
    // again): with a branch around them the compiler waits for the next step's loads in front of this one's work.
    int nth = 1;
    const auto next_ids = [&]() {
      if (nth == 64) {
        nth = 0;
        load_ids(run + 8);
        place_ids();
#pragma unroll
        for (int h = 0; h < 2; ++h) asm volatile("" : "+v"(codes16[h]), "+v"(scales16[h]));  // waited for in here
      }
    };
    Step x;
    load(0, x, true, true);
    if constexpr (LEAN) {
      do {
        next_ids();
        work(run * kRun, x, nth++);
      } while ((run += 8) < run_hi);
    } else {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int r = 0; r < RB; ++r) {
#pragma unroll
        for (int c = 0; c < CH; ++c) qf[r][c] = sign_q(qf[r][c]);
      }
      Step y;
      while (true) {
        next_ids();
        load(nth++, y, true, true);
        work(run * kRun, x, 0);
        if ((run += 8) >= run_hi) break;
        next_ids();
        load(nth++, x, true, true);
        work(run * kRun, y, 0);
        if ((run += 8) >= run_hi) break;
      }
    }
  }

  // ---- the four waves' states become one ------------------------------------------------------
  const uint32_t state = ((static_cast<uint32_t>(PREFILL ? slot * p.shares + chunk : slot) * blocks + (PREFILL ? 0 : block)) * p.h_kv + kvh) * R;
  SharedStates part_o(p.part_o), part_ml(p.part_ml);
  unsigned long long* const counter = p.arrivals + static_cast<int64_t>(PREFILL ? slot : b * blocks + block) * p.h_kv + kvh;
  // A word that an older launch left, also one that was abandoned half way, becomes (epoch, 0); on its way while the states merge.
  if (chunks > 1 && threadIdx.x == 0)
    __hip_atomic_fetch_max(counter, static_cast<unsigned long long>(p.epoch) << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const auto finish = [&](int r, int f, float most, float sum, float4_t acc) {  // elements f.. f + 3 of row r
    const int token = token_of(r);
    const int64_t out = static_cast<int64_t>(q_begin + token0 + token) * p.h_q + kvh * p.group + head0 + r - token * p.group;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    half4_t h;
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = static_cast<half_t>(acc[i] * inv);
    *reinterpret_cast<half4_t*>(p.output + out * D + f) = h;
    if (f == 0) p.lse[out] = sum == 0.f ? kEmptyLse : most + fast_log2(sum);
  };
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    if (r * 16 >= rows_here) break;
    if (r > 0) __syncthreads();
    l[r] = sum_xor32(sum_xor16(l[r]));
    if (__ballot(poisoned[r] != 0) != 0) {
      poisoned[r] |= __shfl_xor(poisoned[r], 16);
      poisoned[r] |= __shfl_xor(poisoned[r], 32);
#pragma unroll
      for (int i = 0; i < DB; ++i) {
        if (poisoned[r] >> (i / 2) & 1) o[r][i] = float4_t{NAN, NAN, NAN, NAN};
      }
    }
    if (g4 == 0) {
      sm_m[wave][c16] = m[r];
      sm_l[wave][c16] = l[r];
    }
    float* const mine = reinterpret_cast<float*>(vt);
#pragma unroll
    for (int half = 0; half < VH; ++half) {
      if (half > 0) __syncthreads();
      if (r * 16 + c16 < rows_here) {
#pragma unroll
        for (int i = 0; i < DB / VH; ++i)
          *reinterpret_cast<float4_t*>(mine + c16 * VW + ((i * 4 + g4) ^ (c16 & 7)) * 4) = o[r][half * (DB / VH) + i];
      }
      __syncthreads();
      for (int at = threadIdx.x; at < min(16, rows_here - r * 16) * (VW / 4); at += 256) {
        const int row = at / (VW / 4), f = at % (VW / 4) * 4;
        const float most = fmaxf(fmaxf(sm_m[0][row], sm_m[1][row]), fmaxf(sm_m[2][row], sm_m[3][row]));
        float sum = 0.f;
        float4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float part = fast_exp2(sm_m[w][row] - most);
          sum += sm_l[w][row] * part;
          acc += *reinterpret_cast<const float4_t*>(reinterpret_cast<const float*>(v_tiles[w]) + row * VW + (f / 4 ^ (row & 7)) * 4) * part;
        }
        const int column = half * VW + f;
        if (chunks == 1) {
          finish(r * 16 + row, column, most, sum, acc);
        } else {
          const uint32_t out = state + r * 16 + row;
          part_o.store4(out * D + column, acc);
          if (column == 0) part_ml.store2(out * 2, most, sum);
        }
      }
    }
  }
  if (chunks == 1) return;

  // ---- the work item that comes last joins the states of its rows' items ------------------------
  // Without device-scope fences, which write back and invalidate a whole L2: the states are stored at device scope,
  // every wave waits for its own stores, one thread counts the workgroup in.
  wait_vmcnt<0>();
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned long long before = __hip_atomic_fetch_add(counter, 1ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sm_last = static_cast<uint32_t>(before) == static_cast<uint32_t>(chunks - 1);
    // nobody of this launch touches the counter again: back to (epoch, 0), from which a replay of the launch counts
    if (sm_last) __hip_atomic_store(counter, static_cast<unsigned long long>(p.epoch) << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!sm_last) return;
  // 64 states at a time: a wave has a row's reference points and sums, a state a lane, and leaves their weights in LDS;
  // then every thread adds up four elements of a row, of all states or, where the rows leave threads over, of some.  What
  // this costs is round trips to memory (device-scope loads miss this XCD's L2), so that many loads are on their way
  // together, those of the outputs beside those of the statistics.
  constexpr int ITEMS = (R * (D / 4) + 255) / 256;
  constexpr int BATCH = 8;
  float* const weight = reinterpret_cast<float*>(v_tiles[0]);  // (R, 64)
  float* const row_most = weight + R * 64;                     // then the factor of what has been added up, then the sum
  float4_t* const partial = reinterpret_cast<float4_t*>(row_most + 4 * R);  // (256)
  static_assert(sizeof(v_tiles) >= kJoinBytes, "they take the V tiles' place");
  const uint32_t stride = static_cast<uint32_t>(blocks) * p.h_kv * R;  // states between neighbouring chunks
  const uint32_t first = state - chunk * stride;
  const int items = rows_here * (D / 4);
  const int span = items <= 32 ? 32 : items <= 64 ? 64 : items <= 128 ? 128 : 256;  // threads that share a state
  const int parts = 256 / span, part = threadIdx.x / span, item0 = threadIdx.x % span;
  float4_t acc[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) acc[i] = float4_t{0.f, 0.f, 0.f, 0.f};
  for (int c0 = 0; c0 < chunks; c0 += 64) {
    const int here = min(64, chunks - c0);
    const int per_part = (here + parts - 1) / parts;
    const int c_lo = part * per_part, c_hi = min(here, c_lo + per_part);
    float4_t v[BATCH];
    const auto load_batch = [&](int item, int c) {
      const int row = item / (D / 4), f = item % (D / 4) * 4;
      const uint32_t src = (first + c0 * stride + row) * D + f;
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        if (j % 4 == 0 && c + j >= c_hi) break;
        v[j] = part_o.load4(src + min(c + j, here - 1) * stride * D);
      }
    };
    if (item0 < items && c_lo < c_hi) load_batch(item0, c_lo);
    float2 ml[R / 4];
#pragma unroll
    for (int i = 0; i < R / 4; ++i) {
      const int row = wave + 4 * i;
      ml[i] = make_float2(kNoKey, 0.f);
      if (row < rows_here && lane < here) ml[i] = part_ml.load2((first + (c0 + lane) * stride + row) * 2);
    }
#pragma unroll
    for (int i = 0; i < R / 4; ++i) {
      const int row = wave + 4 * i;
      if (row >= rows_here) break;
      const float old = c0 == 0 ? kNoKey : row_most[row];
      const float most = fmaxf(wave_max(ml[i].x), old);
      const float w = fast_exp2(ml[i].x - most), rescale = fast_exp2(old - most);
      weight[row * 64 + lane] = w;
      const float sum = sum_xor32(sum_xor16(group_sum<16>(ml[i].y * w))) + (c0 == 0 ? 0.f : row_most[2 * R + row] * rescale);
      if (lane == 0) {
        row_most[row] = most;
        row_most[R + row] = rescale;
        row_most[2 * R + row] = sum;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int item = item0 + i * 256;
      if (item >= items) break;
      const int row = item / (D / 4);
      acc[i] *= row_most[R + row];
      for (int c = c_lo; c < c_hi; c += BATCH) {
        if (i > 0 || c > c_lo) load_batch(item, c);
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          if (c + j < c_hi) acc[i] += v[j] * weight[row * 64 + c + j];
        }
      }
    }
    __syncthreads();
  }
  if (parts > 1) {
    partial[threadIdx.x] = acc[0];
    __syncthreads();
    if (part > 0) return;
    for (int i = 1; i < parts; ++i) acc[0] += partial[threadIdx.x + i * span];
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int item = item0 + i * 256;
    if (item >= items) break;
    const int row = item / (D / 4);
    finish(row, item % (D / 4) * 4, row_most[row], row_most[2 * R + row], acc[i]);
  }
}

static double page_bytes(int32_t h_kv, int32_t page_size, int32_t d) { return 2.0 * h_kv * page_size * (17 * d / 32); }

static void check_mxfp4(const char* what, int32_t h_kv, int32_t page_size, int32_t d) {
  KV_CHECK(h_kv > 0) << what << ": bad shape";
  KV_UNSUPPORTED(d != 64 && d != 96 && d != 128 && d != 256) << what << ": head_dim " << d << " is not built (64, 96, 128, 256)";
  KV_UNSUPPORTED(page_size <= 0 || page_size % kRun != 0) << what << ": page_size must be a multiple of 16, got " << page_size;
  // offsets within K or V of a page are 32-bit numbers
  KV_UNSUPPORTED(page_bytes(h_kv, page_size, d) >= 8589934592.0) << what << ": a page of 8 GiB or more is not built";
}

static void check_aligned(const char* what, std::initializer_list<const void*> data) {
  for (const void* p : data) KV_CHECK(reinterpret_cast<uintptr_t>(p) % 16 == 0) << what << ": data must be aligned to 16 bytes";
}

// Launches over the (token, head) rows of a call: launch(head dim, first token, tokens, grid), of at most 2^30 threads each.
template <class Launch>
static void for_row_pieces(int d, int64_t ntoken, int64_t h_kv, Launch&& launch) {
  const int64_t sixteen = 16 * h_kv * (d / 8);  // threads of 16 tokens
  const int64_t most = std::max<int64_t>((int64_t{1} << 30) / sixteen, 1) * 16;
  for (int64_t first = 0; first < ntoken; first += most) {
    const int64_t tokens = std::min(most, ntoken - first);
    const dim3 grid(static_cast<unsigned>(((tokens + 15) / 16 * sixteen + 255) / 256));
    switch (d) {
      case 64: launch(std::integral_constant<int, 64>{}, first, static_cast<uint32_t>(tokens), grid); break;
      case 96: launch(std::integral_constant<int, 96>{}, first, static_cast<uint32_t>(tokens), grid); break;
      case 128: launch(std::integral_constant<int, 128>{}, first, static_cast<uint32_t>(tokens), grid); break;
      default: launch(std::integral_constant<int, 256>{}, first, static_cast<uint32_t>(tokens), grid); break;
    }
    KV_LAUNCH_CHECK();
  }
}

// Work items that the chip holds at once.
static int64_t resident_items(int cus, int d, int row_blocks) { return static_cast<int64_t>(mxfp4_waves(d, row_blocks)) * cus; }

template <bool PREFILL, int D>
static void launch_rows(const Mxfp4Params& p, int row_blocks, dim3 grid, hipStream_t s) {
  // (prefill: a sequence with more rows than an item has several of them for a key)
  const bool once = !PREFILL && p.row_blocks == 1;
  const auto launch = [&](auto blocks) {
    constexpr int RB = decltype(blocks)::value;
    if constexpr (!PREFILL) {
      if (once) {
        hipLaunchKernelGGL((mxfp4_attn_kernel<D, RB, PREFILL, true>), grid, dim3(256), 0, s, p);
        return;
      }
    }
    hipLaunchKernelGGL((mxfp4_attn_kernel<D, RB, PREFILL, false>), grid, dim3(256), 0, s, p);
  };
  if (row_blocks == 1) launch(std::integral_constant<int, 1>{});
  if (row_blocks == 2) launch(std::integral_constant<int, 2>{});
  if constexpr (D <= 128) {
    if (row_blocks == 3) launch(std::integral_constant<int, 3>{});
  }
  KV_LAUNCH_CHECK();
}

template <bool PREFILL>
static void launch_attention(const Mxfp4Params& p, int d, int row_blocks, dim3 grid, hipStream_t s) {
  switch (d) {
    case 64: return launch_rows<PREFILL, 64>(p, row_blocks, grid, s);
    case 96: return launch_rows<PREFILL, 96>(p, row_blocks, grid, s);
    case 128: return launch_rows<PREFILL, 128>(p, row_blocks, grid, s);
    default: return launch_rows<PREFILL, 256>(p, row_blocks, grid, s);
  }
}

// Scratch memory of a launch: arrival counters, which need no clearing between launches (runtime_support.h), then the states.
constexpr int64_t kMaxCounters = 1 << 18;
constexpr int64_t kMaxItems = (int64_t{1} << 24) - 1;  // a launch has fewer than 2^32 threads
static bool states_fit(int64_t states, int d) { return states * d < int64_t{1} << 30; }  // 32-bit addresses of bytes
static ScratchLease lease_states(const char* what, Mxfp4Params& p, hipStream_t s, int64_t states, int d) {
  if (states == 0) return {};  // no row's keys are shared
  KV_CHECK(states_fit(states, d)) << what << ": too many work items";
  constexpr size_t counter_bytes = kMaxCounters * sizeof(unsigned long long);
  const size_t o_bytes = static_cast<size_t>(states) * d * sizeof(float);
  // the first buffer holds the states of any launch whose items fill the chip once, so that a stream that has run one that
  // shares keys can capture the others
  const size_t at_least = counter_bytes + static_cast<size_t>(2048) * 16 * (d + 2) * sizeof(float);
  ScratchLease ws = lease_scratch(kScratchMxfp4, s, counter_bytes + o_bytes + static_cast<size_t>(states) * 2 * sizeof(float), counter_bytes, at_least);
  p.arrivals = reinterpret_cast<unsigned long long*>(ws.ptr);
  p.epoch = ws.epoch;
  p.part_o = reinterpret_cast<float*>(ws.ptr + counter_bytes);
  p.part_ml = reinterpret_cast<float*>(ws.ptr + counter_bytes + o_bytes);
  return ws;
}

// Blocks of 16 rows that a work item of a decode launch takes (three are what fits the registers at two waves a SIMD; head
// dim 256: two at one): for few keys one, which starts and ends sooner; where they fill the chip the fewest items for the
// group, of equal size.  32 sequences of U[1000,3000] tokens, 32 heads on one: 14.2 us with one block, 17.4 with two; 64 of
// U[20000,40000]: 102 and 74.
static int max_row_blocks(int d) { return d == 256 ? 2 : 3; }
static int forced_row_blocks(int d) {
  return static_cast<int>(std::min<int64_t>(std::max<int64_t>(option(kOptMxfp4RowBlocks), 0), max_row_blocks(d)));
}
static int decode_row_blocks(int cus, int64_t group, int64_t runs, int64_t h_kv, int d) {
  if (forced_row_blocks(d) > 0) return forced_row_blocks(d);
  const int64_t blocks = (group + 15) / 16, most = max_row_blocks(d);
  const int64_t items = (blocks + most - 1) / most;
  const int64_t fewest = (blocks + items - 1) / items;
  return runs * h_kv > 24 * resident_items(cus, d, static_cast<int>(fewest)) ? static_cast<int>(fewest) : 1;
}

static int64_t forced_chunk() {
  const int64_t forced = option(kOptDecodeChunkPages);
  return forced >= 8 && forced % 8 == 0 ? forced : 0;
}

// Keys of a work item in runs, a multiple of 8 (a step of its four waves), from shapes alone: `avg` runs a sequence, per_slot
// items for the same keys, `resident` items that the chip holds at once.
//  * Never under sqrt(2 avg): a step takes a work item 0.47 us on an idle chip, a further state its row 0.12 us.
//  * Sequences of up to five steps are left whole (nothing to join).
//  * Small launches, whose items can all start at once with half of the chip's room to themselves: that many.
//  * Few sequences, long: the shortest chunks with which there are two items a compute unit, as the device finds from the lengths
//    (fit_items).  Two read faster than the four that fit, and a few items more than two, all started together, give some units
//    three (32 x U[2048,16384]: 67, with chunks of 360 runs 87; 8 x 81920, 64 / 8: 125, with four a unit 135).
//  * More of them: sequences of unlike lengths leave workgroups over at the end, so that each has about two items, of 256 runs
//    at most (48 x U[20000,60000]: 355, with 900 runs 420; 64 x U[2048,16384]: 133, with 392 runs 141).  Where none is longer
//    than its share, sequences are left whole (whole_runs: 64 x 4096 57 -> 51, 64 x 8192 of dim 64 66 -> 62).
// Measured in us, 32 / 8 heads of dim 128 unless said, runs an item -> time, * = this rule:
//   1 x 500 tokens        8: 7.2   40*: 6.8                            24 x U[500,2500], 40 / 40 of dim 64   48: 37  96*: 32
//   1 x 2000              8: 8.7   16*: 8.4   32: 9.3   64: 12.0       1 x 32768    32: 19.1  64*: 16.2  128: 19.0
//   1 x 131072           64: 39.8  128*: 33.9  256: 33.4               8 x U[2000,6000]      24: 14.4  40*: 14.2  96: 15.5
//   16 x U[100,4000]     24: 14.6  48*: 15.1  96: 15.8  256: 25.5      64 x U[64,512]  16: 13.5  96*: 9.6  256: 9.7
//   64 x U[1024,8192]    64: 64.1  96: 61.2  160*: 57.3  256: 62.8     8 x U[32768,131072], 64 / 8   96: 144  found*: 123
//   32 x U[1000,3000], 32 / 1   8: 23.7  24*: 13.9  64: 14.6           20 x U[1500,2500], 16 / 2 of dim 256   8: 25.4  24*: 15.0
static int64_t pick_chunk_runs(int64_t runs, int64_t batch, int64_t per_slot, int64_t resident, int64_t two_each, int* fit_items) {
  if (forced_chunk() > 0) return forced_chunk();
  const auto steps = [](int64_t n) { return std::max<int64_t>((n + 7) / 8 * 8, 8); };
  const auto for_items = [&](int64_t items) {  // the shortest that leaves at most so many items
    const int64_t slots = items / per_slot - batch;
    return slots > 0 ? steps((runs + slots - 1) / slots) : runs + 8;
  };
  const int64_t avg = runs / batch;
  const int64_t least = steps(static_cast<int64_t>(std::sqrt(2.0 * static_cast<double>(avg))));
  const int64_t small = for_items(resident / 2), two = for_items(two_each);
  int64_t chunk = std::min<int64_t>(std::max<int64_t>(96, steps(avg * 5 / 8)), 256);
  if (avg <= 40) chunk = std::max<int64_t>(small, 40);
  else if (small <= 48) chunk = std::max(small, least);
  else if (batch <= 64 && 2 * batch * per_slot <= two_each && two <= 1 << 20) {
    chunk = two;
    *fit_items = static_cast<int>(two_each / per_slot);
  }
  return std::min<int64_t>(chunk, 1 << 20);
}

// How a prefill launch is cut, from shapes alone: blocks of 16 rows that a work item takes, and work items that share the keys
// of a row block.  An item turns a key's codes into fp16 once for all of its rows, so that more blocks are faster where the
// chip is full (8 chunks of 2048 tokens on 4096 + 2048 keys, 32 / 8 heads of dim 128, TFLOP/s at 1 / 2 / 3 blocks: 680 / 840 /
// 968; of dim 64: 526 / 716 / 773; 8 / 4 heads of dim 256: 470 / 729), and slower where it is not (40 tokens on 4000:
// 20.3 / 22.2 / 25.9 us).  Estimated in us: a compute unit takes its items `waves` at a time; an item's start and end cost 4
// and 2 a block, a step t_idle alone on its compute unit and t_full where that is full (measured); joining the shares of a
// row costs 1.5 and 0.12 a share and block.  (Two chunks of 216 tokens on 26000 keys, 16 / 2 heads of dim 256, 1 / 2 / 3 / 5 / 8
// shares: 387 / 350 / 396 / 319 / 316 us, estimated 385 / 313 / 346 / 343 / 309.)
struct Cut {
  int row_blocks;
  int shares;
};
static Cut cut_prefill(int cus, int64_t rows, int64_t batch, int64_t h_kv, int64_t runs, int d) {
  const double t_full[4][3] = {{1.05, 1.18, 1.10}, {1.35, 1.23, 1.40}, {1.63, 1.28, 1.70}, {2.28, 2.94, 0}};
  const int64_t forced = std::min<int64_t>(option(kOptPrefillKvSplits), 64);
  const int64_t sequence = (rows + batch - 1) / batch;  // rows of one
  Cut best = {1, 1};
  double least = 1e30;
  const int forced_blocks = forced_row_blocks(d);
  for (int blocks = std::max(forced_blocks, 1); blocks <= (forced_blocks > 0 ? forced_blocks : max_row_blocks(d)); ++blocks) {
    const int64_t items = (sequence + 16 * blocks - 1) / (16 * blocks) * batch * h_kv;
    const int waves = mxfp4_waves(d, blocks);
    const double idle = (0.35 + 0.15 * blocks) * (d == 256 ? 2.8 : 1.0), start = 4.0 + 2.0 * blocks;
    const double full = t_full[d == 64 ? 0 : d == 96 ? 1 : d == 128 ? 2 : 3][blocks - 1];
    const int64_t most = forced > 0 ? forced : items >= 2 * waves * cus ? 1 : std::min<int64_t>(std::max<int64_t>(runs / 8, 1), 64);
    for (int64_t n = forced > 0 ? forced : 1; n <= most; ++n) {
      const int64_t load = (items * n + cus - 1) / cus, rest = load % waves;  // items of a compute unit
      const double steps = static_cast<double>((runs + 8 * n - 1) / (8 * n));
      double us = static_cast<double>(load / waves) * (start + full * steps);
      if (rest > 0) us += start + (idle + (full - idle) * static_cast<double>(rest - 1) / (waves - 1)) * steps;
      if (n > 1) us += 1.5 + 0.12 * blocks * static_cast<double>(n);
      if (us < least) {
        least = us;
        best = {blocks, static_cast<int>(n)};
      }
    }
  }
  return best;
}

static Mxfp4Params attn_params(const char* what, const void* q, const void* pages, const int32_t* page_indptr,
                               const int32_t* page_values, const int32_t* length_info, void* output, float* lse, double sm_scale,
                               int32_t batch, int64_t nnz_pages, int64_t num_pages, int32_t h_q, int32_t h_kv, int32_t d,
                               int32_t page_size, int32_t sliding_window) {
  KV_CHECK(batch >= 0 && nnz_pages >= 0 && h_q > 0 && h_kv > 0 && h_q % h_kv == 0) << what << ": bad shape";
  check_mxfp4(what, h_kv, page_size, d);
  // 36-bit addresses within the pool
  KV_UNSUPPORTED(num_pages * page_bytes(h_kv, page_size, d) >= 68719476736.0) << what << ": a pool of 64 GiB or more is not built";
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
  p.page_size = page_size;
  p.runs_per_page = page_size / kRun;
  p.page_of_run = ExactDivision::by(p.runs_per_page);
  p.inv_group = 1.f / static_cast<float>(p.group);
  // The kernel takes maxima of scores that are not scaled yet and masks with -inf: a scale below 0 goes to q, and one of
  // 0 (all weights equal) becomes one that is as good as 0.
  p.scale_log2 = std::max(std::fabs(static_cast<float>(sm_scale)) * kLog2e, 1e-30f);
  p.q_sign = sm_scale < 0 ? 0x80008000u : 0;
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
  for_row_pieces(head_dim, ntoken, num_kv_heads, [&](auto dim, int64_t first, uint32_t tokens, dim3 grid) {
    constexpr int D = decltype(dim)::value;
    const int64_t at = first * num_kv_heads * D;
    hipLaunchKernelGGL(mxfp4_append_kernel<D>, grid, dim3(256), 0, as_stream(stream), static_cast<uint8_t*>(pages),
                       static_cast<const half_t*>(k_data) + at, static_cast<const half_t*>(v_data) + at, position_map + first, tokens,
                       static_cast<uint32_t>(num_kv_heads), static_cast<uint32_t>(page_size));
  });
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
  for_row_pieces(head_dim, ntoken, num_kv_heads, [&](auto dim, int64_t first, uint32_t tokens, dim3 grid) {
    constexpr int D = decltype(dim)::value;
    const int64_t at = first * num_kv_heads * D;
    hipLaunchKernelGGL(mxfp4_read_kernel<D>, grid, dim3(256), 0, as_stream(stream), static_cast<const uint8_t*>(pages),
                       static_cast<half_t*>(k_data) + at, static_cast<half_t*>(v_data) + at, position_map + first, tokens,
                       static_cast<uint32_t>(num_kv_heads), static_cast<uint32_t>(page_size));
  });
  KV_API_END();
}

int tvmkv_mxfp4_batch_decode_paged_kv(const void* q, const void* pages, const int32_t* page_indptr, const int32_t* page_values,
                                      const int32_t* length_info, void* output, float* lse, double sm_scale, int32_t batch_size,
                                      int64_t nnz_pages, int64_t num_pages, int32_t h_q, int32_t h_kv, int32_t head_dim,
                                      int32_t page_size, int32_t sliding_window, void* stream) {
  KV_API_BEGIN();
  const char* const what = "mxfp4_batch_decode_paged_kv";
  Mxfp4Params p = attn_params(what, q, pages, page_indptr, page_values, length_info, output, lse, sm_scale, batch_size, nnz_pages,
                              num_pages, h_q, h_kv, head_dim, page_size, sliding_window);
  if (batch_size == 0) return TVMKV_OK;
  KV_CHECK(q && pages && page_indptr && length_info && output && lse) << what << ": NULL tensor";
  KV_CHECK(nnz_pages == 0 || page_values) << what << ": NULL page table";
  check_aligned(what, {q, pages, output});
  const int cus = compute_units();
  const int64_t runs = nnz_pages * p.runs_per_page;
  const int row_blocks = decode_row_blocks(cus, p.group, runs, h_kv, head_dim), rows = 16 * row_blocks;
  p.row_blocks = (p.group + rows - 1) / rows;
  const int64_t per_slot = static_cast<int64_t>(h_kv) * p.row_blocks;
  KV_CHECK(runs < (int64_t{1} << 31)) << what << ": too many pages";
  p.chunk_runs = static_cast<uint32_t>(pick_chunk_runs(runs, batch_size, per_slot, resident_items(cus, head_dim, row_blocks), 2 * cus, &p.fit_items));
  if (batch_size * per_slot > kMaxCounters || !states_fit((runs / p.chunk_runs + batch_size) * per_slot * rows, head_dim)) {
    p.chunk_runs = 1 << 30;
    p.fit_items = 0;
  }
  if (batch_size <= 64 && forced_chunk() == 0 && p.fit_items == 0) {
    const int64_t whole = runs * per_slot * 11 / (20 * cus);  // an equal share of two items a compute unit, and a tenth
    if (whole > p.chunk_runs) p.whole_runs = static_cast<uint32_t>(std::min<int64_t>(whole, 1 << 20));
  }
  const int64_t slots = p.fit_items > 0 ? p.fit_items : runs / p.chunk_runs + batch_size;
  KV_CHECK(slots * per_slot <= kMaxItems) << what << ": too many work items";
  const hipStream_t s = as_stream(stream);
  const ScratchLease ws = lease_states(what, p, s, runs > p.chunk_runs || p.fit_items > 0 ? slots * per_slot * rows : 0, head_dim);
  launch_attention<false>(p, head_dim, row_blocks, dim3(static_cast<unsigned>(slots * per_slot)), s);
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
                              num_pages, h_q, h_kv, head_dim, page_size, sliding_window);
  KV_CHECK(total_q >= 0) << what << ": bad shape";
  if (batch_size == 0 || total_q == 0) return TVMKV_OK;
  KV_CHECK(q && q_indptr && pages && page_indptr && length_info && output && lse) << what << ": NULL tensor";
  KV_CHECK(nnz_pages == 0 || page_values) << what << ": NULL page table";
  check_aligned(what, {q, pages, output});
  // (total_q group / 16 + batch) h_kv, the most that any cut makes
  KV_CHECK(total_q <= (kMaxItems - static_cast<int64_t>(batch_size) * h_kv) / h_q * 16) << what << ": too many work items";
  p.q_indptr = q_indptr;
  p.causal = causal != 0;
  const hipStream_t s = as_stream(stream);
  const Cut cut = cut_prefill(compute_units(), total_q * p.group, batch_size, h_kv, nnz_pages * p.runs_per_page / batch_size, head_dim);
  const int row_blocks = cut.row_blocks, rows = 16 * row_blocks;
  const int64_t slots = total_q * p.group / rows + batch_size;
  p.shares = cut.shares;
  if (slots * h_kv > kMaxCounters || !states_fit(slots * p.shares * h_kv * rows, head_dim)) p.shares = 1;
  const ScratchLease ws = lease_states(what, p, s, p.shares > 1 ? slots * p.shares * h_kv * rows : 0, head_dim);
  launch_attention<true>(p, head_dim, row_blocks, dim3(static_cast<unsigned>(slots * h_kv), 1, p.shares), s);
  KV_API_END();
}

}  // extern "C"
