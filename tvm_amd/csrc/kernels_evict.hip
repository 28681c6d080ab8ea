// Eviction from the paged cache by the attention that tokens received: the sums of attention weights that go with an attention
// call, the choice of the tokens that stay and their move to the front of the sequence's pages.
//
// With s the scaled scores (base 2) of a query head and lse their log-sum-exp, a key's weight is 2^(s - lse).  The weights pool
// (weight pages, h_kv, page_size), float32, holds a sum for each stored token and kv head, over the query heads of the group
// and the queries that count.  Every entry is added to by one lane of one workgroup: the sums do not depend on the order in
// which workgroups run.
#include <algorithm>
#include <cstdint>
#include <functional>
#include <initializer_list>
#include <type_traits>

#include "kept_scores.cuh"
#include "kernels_common.cuh"
#include "prefill_merge.cuh"
#include "runtime_support.h"
#include "typed_kernels.h"
#include "exact_division.h"

namespace tvmkv {

typedef float float4_any_t __attribute__((ext_vector_type(4), aligned(4)));
typedef int int4_any_t __attribute__((ext_vector_type(4), aligned(4)));

// Where work items begin: sequence b of x_b = tokens that its pages hold owns the slots [X_b / per + b, ...), X_b the tokens of
// the pages in front of it; the grid, sized from shapes alone, has X_batch / per + batch slots.
struct SequenceOf {
  int index, slot_begin, page_begin, num_pages, last_page_len;
  __device__ __forceinline__ int stored(int page_shift) const {
    return num_pages > 0 ? ((num_pages - 1) << page_shift) + last_page_len : 0;
  }
};
__device__ __forceinline__ SequenceOf sequence_of_slot(const int32_t* page_indptr, const int32_t* last_page_len, int batch, int page_shift,
                                                       uint32_t per_shift, int slot, int lane) {
  const int base = page_indptr[0];
  const auto begin_of = [&](int page) {
    return static_cast<int>((static_cast<uint32_t>(page - base) << page_shift) >> per_shift);
  };
  int lo = 0, n = batch;
  while (n > 64) {  // the answer lies in [lo, lo + n)
    const int stride = (n + 63) >> 6, i = lo + lane * stride;
    const bool hit = i < lo + n && begin_of(page_indptr[min(i, batch)]) + i <= slot;
    const int first = lo + (max(static_cast<int>(__popcll(__ballot(hit))), 1) - 1) * stride;
    n = min(stride, lo + n - first);
    lo = first;
  }
  const int at = lo + min(lane, n - 1);
  const int page = page_indptr[at], next = page_indptr[at + 1], last = last_page_len[at];
  const int begin = begin_of(page) + at;
  const int who = max(static_cast<int>(__popcll(__ballot(lane < n && begin <= slot))), 1) - 1;
  const auto of = [&](int x) { return __builtin_amdgcn_readlane(x, who); };
  return {lo + who, of(begin), of(page), of(next) - of(page), of(last)};
}

// ------------------------------------------------------------------------------------------
// Weights from q, K and lse.  A wave keeps 32 TB tokens' K in registers as the A operand of the 32x32x16 matrix instruction and
// walks the rows (query token, query head of the group) that count, 32 at a time as the B operand: S^T[token, row] has a
// row a lane, so that a lane subtracts one lse, and its 16 sums a block are tokens'.  The lanes' sums are added at the end.
// The four waves share the rows, which asynchronous copies bring to shared memory kStages - 1 tiles ahead, with the rows' lse.
// A block's products run under the exponentials of the block before it.
//
// The product q K^T is done again, as attention writes no scores and a key's weight needs the row's lse first: 2 D operations, an exponential
// and two more vector instructions for each (row, key), K read once and q once for 128 or 256 tokens.  Bound by the issue of vector and
// matrix instructions: 8 chunks of 128-2048 queries on up to 4096 tokens, 32 / 8 heads of dim 128, 337 us (807 TFLOP/s of products;
// 0.64 of the issue slots and 0.35 of the matrix unit in use); two chunks of 100-300 on 20 000-32 768, 16 / 2 heads of dim 256, 108 us
// (521 TFLOP/s: 32 tokens a wave, as 64 tokens' K do not fit its registers, and so q read from shared memory twice as often).
// ------------------------------------------------------------------------------------------
struct KeyWeightsParams {
  const half_t* q;
  const half_t* pages;
  const int32_t* q_indptr;  // NULL: one query token a sequence
  const int32_t* page_indptr;
  const int32_t* page_values;
  const int32_t* weight_page_values;
  const int32_t* last_page_len;
  const float* lse;
  float* key_weights;
  float* shares;  // where the rows are shared, the sums of each share: (share, kv head, entry of the page table, token of the page)
  int nnz_pages;
  int batch;
  int h_q;
  int h_kv;
  int group;
  ExactDivision by_group;
  uint32_t inv_group;  // 2^16 / group, rounded up: divides numbers below 128 by groups below 64
  int causal;
  int observed;    // > 0: queries at a sequence's end that count
  int page_shift;  // pages hold 1 << page_shift tokens
  float scale_log2;
};

// The sequence of a slot where they are few: those with the most rows that count first, so that the last workgroups to start have the
// least to do, each with as many slots as it has tiles of T tokens.
__device__ __forceinline__ SequenceOf sequence_by_rows(const KeyWeightsParams& p, int T, int slot, int lane) {
  const int at = min(lane, p.batch - 1);
  const int page = p.page_indptr[at], num_pages = p.page_indptr[at + 1] - page, last = p.last_page_len[at];
  int rows = p.q_indptr != nullptr ? p.q_indptr[at + 1] - p.q_indptr[at] : 1;
  if (p.observed > 0) rows = min(rows, p.observed);
  const int stored = num_pages > 0 ? ((num_pages - 1) << p.page_shift) + last : 0;
  const int tiles = lane < p.batch && rows > 0 ? (stored + T - 1) / T : 0;
  const int key = min(rows, (1 << 24) - 1) * 64 + 63 - lane;  // unlike from lane to lane
  int begin = 0;
  for (int j = 0; j < p.batch; ++j) begin += __builtin_amdgcn_readlane(key, j) > key ? __builtin_amdgcn_readlane(tiles, j) : 0;
  const uint64_t hit = __ballot(slot >= begin && slot < begin + tiles);
  if (hit == 0) return {-1, 0, 0, 0, 0};
  const int who = __ffsll(static_cast<long long>(hit)) - 1;
  const auto of = [&](int x) { return __builtin_amdgcn_readlane(x, who); };
  return {who, of(begin), of(page), of(num_pages), of(last)};
}

// copy16_to_lds of 4 bytes a lane
__device__ __forceinline__ void copy4_to_lds(const void* src_base, uint32_t byte_off, uint32_t lds_addr) {
  lds_addr = __builtin_amdgcn_readfirstlane(lds_addr);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(byte_off), "s"(src_base), "s"(lds_addr) : "memory");
}

// A lane's part of token t's K as the A operand of 32 tokens' products: 8 of every 16 elements.
template <int D>
__device__ __forceinline__ void load_key(half8_t (&k)[D / 16], const KeyWeightsParams& p, const SequenceOf& s, int kvh, int t, int half) {
  const int page = p.page_values[s.page_begin + (t >> p.page_shift)];
  const half_t* row = p.pages + ((((static_cast<int64_t>(page) * 2 * p.h_kv + kvh) << p.page_shift) + (t & ((1 << p.page_shift) - 1))) * D) + half * 8;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) k[ks] = ld16(row + ks * 16).h8;
}
// Adds up a block's sums over the rows and to the pool's, or writes those of a share: lane i of 32 takes the sum of its half's i-th token.
__device__ __forceinline__ void add_block_sums(const float (&sum)[16], const KeyWeightsParams& p, const SequenceOf& s, int kvh, int share, int t0,
                                               int stored, int col, int half) {
  float mine = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float total = sum_xor16(group_sum<16>(sum[i]));
    mine = col == i ? total : mine;
  }
  const int t = t0 + (col & 3) + 8 * (col >> 2) + 4 * half;
  if (col < 16 && t < stored) {
    if (p.shares != nullptr) {
      p.shares[((static_cast<int64_t>(share * p.h_kv + kvh) * p.nnz_pages + s.page_begin) << p.page_shift) + t] = mine;
      return;
    }
    const int page = p.weight_page_values[s.page_begin + (t >> p.page_shift)];
    p.key_weights[((static_cast<int64_t>(page) * p.h_kv + kvh) << p.page_shift) + (t & ((1 << p.page_shift) - 1))] += mine;
  }
}

template <int D, int TB>
struct WeightTiles {
  static constexpr int kRow = D == 64 ? 64 : D <= 128 ? 128 : 256;  // halfs of a row in shared memory
  static constexpr int kPieces = kRow / 8;
  static constexpr int kRows = TB == 2 ? 64 : 32;        // of a tile
  static constexpr int kCopies = kRows * kPieces / 256;  // copy instructions of a wave for a tile
  static constexpr int kStages = TB == 2 ? 3 : 4;
  // Piece c of row r is at c ^ swizzle(r): 16 lanes read the same piece of 16 neighbouring rows, 256 bytes in all banks.
  static __device__ __forceinline__ int swizzle(int row) { return kRow == 64 ? row >> 1 & 7 : row & 15; }
};

template <int D, int TB>
__global__ __launch_bounds__(256, 2) void key_weights_kernel(KeyWeightsParams p) {
  using Tiles = WeightTiles<D, TB>;
  constexpr int KS = D / 16, PIECES = Tiles::kPieces, COPIES = Tiles::kCopies, STAGES = Tiles::kStages, R = Tiles::kRows;
  constexpr int T = 128 * TB;
  static_assert(TB == 1 || TB == 2, "the shift below");
  __shared__ __attribute__((aligned(16))) half_t rows_lds[STAGES][R * Tiles::kRow];
  __shared__ float lse_lds[STAGES][4][64];  // a copy for each wave
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int col = lane & 31;
  const int half = lane >> 5;
  const int kvh = blockIdx.x % p.h_kv, slot = blockIdx.x / p.h_kv;
  const SequenceOf s = p.batch <= 64 ? sequence_by_rows(p, T, slot, lane)
                                     : sequence_of_slot(p.page_indptr, p.last_page_len, p.batch, p.page_shift, TB == 1 ? 7 : 8, slot, lane);
  if (s.index < 0) return;  // a spare slot
  const int stored = s.stored(p.page_shift);
  const int tile_t0 = (slot - s.slot_begin) * T, t0 = tile_t0 + wave * 32 * TB;  // the workgroup's and the wave's first token
  if (tile_t0 >= stored) return;
  const int q_begin = p.q_indptr != nullptr ? p.q_indptr[s.index] : s.index;
  const int q_len = p.q_indptr != nullptr ? p.q_indptr[s.index + 1] - q_begin : 1;
  const int first_counted = p.observed > 0 ? max(q_len - p.observed, 0) : 0;
  const int in_front = stored - q_len;  // query i sees the keys up to in_front + i
  const int row_begin = first_counted * p.group, row_end = q_len * p.group;
  const auto end_of = [&](int token) { return p.causal ? min(in_front + token + 1, stored) : stored; };
  // no row in front of the first tile's sees a token of the workgroup's
  int first_tile = max(first_counted, p.causal ? tile_t0 - in_front : 0) * p.group / R, num_tiles = (row_end + R - 1) / R;
  if (p.shares != nullptr) {
    const int each = (max(num_tiles - first_tile, 0) + static_cast<int>(gridDim.y) - 1) / static_cast<int>(gridDim.y);
    first_tile += blockIdx.y * each;
    num_tiles = min(first_tile + each, num_tiles);
  } else if (first_tile >= num_tiles) {
    return;
  }

  half8_t k[TB][KS];
#pragma unroll
  for (int b = 0; b < TB; ++b) load_key<D>(k[b], p, s, kvh, min(t0 + b * 32 + col, stored - 1), half);
  float sum[TB][16];
#pragma unroll
  for (int b = 0; b < TB; ++b) {
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[b][i] = 0.f;
  }

  const int64_t head0 = static_cast<int64_t>(q_begin) * p.h_q + kvh * p.group;  // (query, head) of row 0
  // Tile by tile, tiles behind the last one as that one, so that a tile is always so many copies behind the next.
  // Offsets of a lane's copies, in heads, from the first head of the tile's first query, row `rest` of it: row r of the tile.
  const auto offset_of = [&](int r, int rest) {
    const uint32_t nth = rest + r;  // below 64 + group
    const uint32_t token = p.group >= 64 ? (nth >= static_cast<uint32_t>(p.group) ? 1 : 0) : __umul24(nth, p.inv_group) >> 16;
    return __umul24(token, p.h_q - p.group) + nth;
  };
  const auto row_of = [&](int i) { return ((wave * COPIES + i) * 64 + lane) / PIECES; };
  const auto piece_of = [&](int i) { return min((((wave * COPIES + i) * 64 + lane) % PIECES) ^ Tiles::swizzle(row_of(i)), D / 8 - 1) * 16; };
  // the same for every whole tile where tiles begin with a query's first head
  const bool regular = R % p.group == 0;
  uint32_t whole[COPIES], whole_lse = offset_of(lane & (R - 1), 0) * 4;
#pragma unroll
  for (int i = 0; i < COPIES; ++i) whole[i] = offset_of(row_of(i), 0) * (D * 2) + piece_of(i);
  const auto issue = [&](int tile, int stage) {
    const int r0 = min(tile, num_tiles - 1) * R, token0 = p.by_group(r0);
    const int64_t at0 = head0 + static_cast<int64_t>(token0) * p.h_q;
    const half_t* const q = p.q + at0 * D;
    const float* const lse = p.lse + at0;
    const uint32_t rows_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr_t)rows_lds[stage])) + wave * (COPIES * 1024);
    const uint32_t lse_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr_t)lse_lds[stage][wave]));
    if (regular && r0 + R <= row_end) {
#pragma unroll
      for (int i = 0; i < COPIES; ++i) copy16_to_lds(q, whole[i], rows_at + i * 1024);
      copy4_to_lds(lse, whole_lse, lse_at);
    } else {
      const int rest = r0 - token0 * p.group, last = row_end - 1 - r0;
#pragma unroll
      for (int i = 0; i < COPIES; ++i) copy16_to_lds(q, offset_of(min(row_of(i), last), rest) * (D * 2) + piece_of(i), rows_at + i * 1024);
      copy4_to_lds(lse, offset_of(min(lane & (R - 1), last), rest) * 4, lse_at);
    }
  };
  wait_vmcnt<0>();  // K is there: from here on only the copies count
  if (first_tile < num_tiles) {
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(first_tile + i, i);
  }
  int stage = 0, next_stage = STAGES - 1;
  for (int tile = first_tile; tile < num_tiles; ++tile, stage = stage + 1 < STAGES ? stage + 1 : 0) {
    // The wave's part of the tile has landed where no more than the later tiles' copies are outstanding; behind the barrier everyone's
    // has, and every wave is done with the stage that the next copies overwrite.
    wait_vmcnt<(STAGES - 2) * (COPIES + 1)>();
    __syncthreads();
    issue(tile + STAGES - 1, next_stage);
    next_stage = next_stage + 1 < STAGES ? next_stage + 1 : 0;
    const int r0 = tile * R;
    if (end_of(p.by_group(min(r0 + R - 1, row_end - 1))) <= t0) continue;  // no row of the tile sees a token of the wave's
    const half_t* const rows = rows_lds[stage];
    half8_t q[KS];
    float lse;
    const auto read = [&](int h) {
      lse = lse_lds[stage][wave][h * 32 + col];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        q[ks] = *reinterpret_cast<const half8_t*>(rows + (h * 32 + col) * Tiles::kRow + (((ks * 2 + half) ^ Tiles::swizzle(h * 32 + col)) * 8));
    };
    const auto product = [&](int b) {
      float16_t x = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[b][ks], q[ks], x, 0, 0, 0);
      return x;
    };
    // every row counts and sees all of the wave's tokens (those behind the last stored one are not written)
    if (r0 >= row_begin && r0 + R <= row_end && end_of(p.by_group(r0)) >= min(t0 + 32 * TB, stored)) {
      const auto add = [&](int b, const float16_t& x, float of) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[b][i] += fast_exp2(fmaf(x[i], p.scale_log2, -of));
      };
      float16_t x;
      float x_lse;
#pragma unroll
      for (int h = 0; h < R / 32; ++h) {
        read(h);
#pragma unroll
        for (int b = 0; b < TB; ++b) {
          __builtin_amdgcn_sched_barrier(0);
          const float16_t y = product(b);
          if (h > 0 || b > 0) {
            add((b + TB - 1) % TB, x, x_lse);
            interleave_mfma_valu<KS>();
          }
          x = y;
          x_lse = lse;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      add(TB - 1, x, x_lse);
    } else {
#pragma unroll
      for (int h = 0; h < R / 32; ++h) {
        if (r0 + h * 32 >= row_end) break;
        read(h);
        const int row = min(r0 + h * 32 + col, row_end - 1);
        const int end = r0 + h * 32 + col < row_end && row >= row_begin ? end_of(p.by_group(row)) : 0;
#pragma unroll
        for (int b = 0; b < TB; ++b) {
          const float16_t x = product(b);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int t = t0 + b * 32 + (i & 3) + 8 * (i >> 2) + 4 * half;
            const float w = fast_exp2(fmaf(x[i], p.scale_log2, -lse));
            sum[b][i] += t < end ? w : 0.f;
          }
        }
      }
    }
  }
  wait_vmcnt<0>();  // no copy is on its way into memory that is another workgroup's then
#pragma unroll
  for (int b = 0; b < TB; ++b) add_block_sums(sum[b], p, s, kvh, blockIdx.y, t0 + b * 32, stored, col, half);
}

// The shares' sums, in their order, to the pool's.  A wave has 256 tokens of a kv head, a lane four.
constexpr int kSharedTokensShift = 10;  // of a workgroup
__global__ __launch_bounds__(256) void shared_rows_kernel(KeyWeightsParams p, int shares) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int kvh = blockIdx.x % p.h_kv, slot = blockIdx.x / p.h_kv;
  const SequenceOf s = sequence_of_slot(p.page_indptr, p.last_page_len, p.batch, p.page_shift, kSharedTokensShift, slot, lane);
  const int stored = s.stored(p.page_shift), t = ((slot - s.slot_begin) << kSharedTokensShift) + (wave * 64 + lane) * 4;
  // (a sequence without queries may have had no workgroups)
  if (t >= stored || (p.q_indptr != nullptr && p.q_indptr[s.index + 1] <= p.q_indptr[s.index])) return;
  const int page = p.weight_page_values[s.page_begin + (t >> p.page_shift)];
  float* const at = p.key_weights + ((static_cast<int64_t>(page) * p.h_kv + kvh) << p.page_shift) + (t & ((1 << p.page_shift) - 1));
  const float* from = p.shares + ((static_cast<int64_t>(kvh) * p.nnz_pages + s.page_begin) << p.page_shift) + t;
  float4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int i = 0; i < shares; ++i, from += (static_cast<int64_t>(p.h_kv) * p.nnz_pages) << p.page_shift) sum += *reinterpret_cast<const float4_t*>(from);
  if (t + 4 <= stored) {
    float4_any_t* const sums = reinterpret_cast<float4_any_t*>(at);
    *sums = *sums + float4_any_t{sum[0], sum[1], sum[2], sum[3]};
  } else {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if (t + k < stored) at[k] += sum[k];
    }
  }
}

// Few rows in shares: the merge and the weights in one launch.  The first workgroups merge, the others weigh 128 tokens each, a wave 32;
// rows come straight from memory, and each workgroup finds its rows' lse from the shares'.  A chain of round trips: five queries on 700
// tokens (32 / 8 heads of dim 128) 5.5 us, apart 5.0 + 5.6.
template <int D>
__global__ __launch_bounds__(256) void merge_and_weigh_kernel(KeyWeightsParams p, PrefillShares shares, half_t* output, float* lse, int merging) {
  if (static_cast<int>(blockIdx.x) < merging) {
    merge_prefill_shares<float, D, true>(shares.output, shares.lse, output, lse, shares.rows, shares.splits, 0, p.q_indptr, p.batch, p.h_q, blockIdx.x);
    return;
  }
  constexpr int KS = D / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int item = blockIdx.x - merging, kvh = item % p.h_kv, slot = item / p.h_kv;
  const SequenceOf s = sequence_of_slot(p.page_indptr, p.last_page_len, p.batch, p.page_shift, 7, slot, lane);
  const int stored = s.stored(p.page_shift), t0 = (slot - s.slot_begin) * 128 + wave * 32;
  if (t0 >= stored) return;
  const int q_begin = p.q_indptr[s.index], q_len = p.q_indptr[s.index + 1] - q_begin;
  const int in_front = stored - q_len;
  const int row_begin = (p.observed > 0 ? max(q_len - p.observed, 0) : 0) * p.group, row_end = q_len * p.group;
  half8_t k[KS];
  load_key<D>(k, p, s, kvh, min(t0 + col, stored - 1), half);
  float sum[16] = {};
  for (int r0 = row_begin; r0 < row_end; r0 += 32) {
    const int row = min(r0 + col, row_end - 1), token = p.by_group(row);
    const int64_t at = static_cast<int64_t>(q_begin + token) * p.h_q + kvh * p.group + (row - token * p.group);
    half8_t q[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[ks] = ld16(p.q + at * D + half * 8 + ks * 16).h8;
    const float row_lse = merged_lse(shares.lse, shares.rows, shares.splits, at);
    float16_t x = {};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[ks], q[ks], x, 0, 0, 0);
    const int end = r0 + col >= row_end ? 0 : p.causal ? min(in_front + token + 1, stored) : stored;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float w = fast_exp2(fmaf(x[i], p.scale_log2, -row_lse));
      sum[i] += t0 + (i & 3) + 8 * (i >> 2) + 4 * half < end ? w : 0.f;
    }
  }
  add_block_sums(sum, p, s, kvh, 0, t0, stored, col, half);
}

// ------------------------------------------------------------------------------------------
// Weights from kept scores: decode's, which are few (4 bytes for each of the group's heads, where K has 2 D).  A wave has 256 tokens
// of a kv head, a lane the four of a run of 16 that a lane of the decode kernel had.  Each score is read once, in whole lines: 21 MB of 64
// sequences of 1024-4096 tokens in 10.6 us, 102 MB of 8 of 32 768-65 536 with 64 query heads in 23 (4.4 TB/s).  Whole calls with K read
// again, for all heads of a group at once, took 208 and 458 us, with kept scores 144 and 340.
// ------------------------------------------------------------------------------------------
struct KeptScoresParams {
  const float* scores;  // (kv head, 16-token run of the page table, head of the group, 16 tokens in the order of kept_score_token)
  const int32_t* page_indptr;
  const int32_t* weight_page_values;
  const int32_t* last_page_len;
  const float* lse;
  float* key_weights;
  int batch;
  int nnz_pages;
  int h_kv;
  int group;
  int page_shift;
};
constexpr int kKeptTokensShift = 10;  // of a workgroup
__global__ __launch_bounds__(256) void kept_scores_kernel(KeptScoresParams p) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int kvh = blockIdx.x % p.h_kv, slot = blockIdx.x / p.h_kv;
  const SequenceOf s = sequence_of_slot(p.page_indptr, p.last_page_len, p.batch, p.page_shift, kKeptTokensShift, slot, lane);
  const int stored = s.stored(p.page_shift);
  const int run = (((slot - s.slot_begin) << kKeptTokensShift) + wave * 256) / 16 + (lane >> 2);  // of the sequence
  if (run * 16 >= stored) return;
  const int part = lane & 3;
  const float* at = p.scores + (((kvh * static_cast<int64_t>(p.nnz_pages) + s.page_begin) << (p.page_shift - 4)) + run) * (p.group * 16) + 4 * part;
  const float* lse = p.lse + (static_cast<int64_t>(s.index) * p.h_kv + kvh) * p.group;
  const int page = p.weight_page_values[s.page_begin + (run >> (p.page_shift - 4))];
  const float4_t x = kept_weights(p.group, [&](int h) { return *reinterpret_cast<const float4_t*>(at + h * 16); }, [&](int h) { return lse[h]; });
  add_to_sums(p.key_weights + ((static_cast<int64_t>(page) * p.h_kv + kvh) << p.page_shift) + (run * 16 & ((1 << p.page_shift) - 1)), part, x,
              stored - run * 16);
}

// ------------------------------------------------------------------------------------------
// The choice.  As integers that order like them (NaN below everything, -0 as 0) the weights of a (sequence, kv head), a list from here
// on, go through passes over some of their bits that find the smallest one that stays, T, and how many of the weights equal to it
// do: counts, exact whatever their order.  Then a bit a token says which ones stay, and running counts of free places and of
// tokens without one pair them.  A wave takes blocks of 256 tokens, four neighbouring ones a lane; bit l of the block's four words of
// 64 is token 4 l + (0..3)'s, as a comparison leaves them.
//
// Lists of ordinary length are a workgroup's, in one launch: passes of 8 bits, the weights loaded once and kept in registers, up to
// HELD blocks a wave (longer lists are read again in every pass, their bits in scratch memory).  Where all are long they are cut into
// chunks of 4096 tokens, in six launches: the histograms of 11, 11 and 10 bits are added up in memory and the last of a list's
// workgroups goes on to find the digit; then the bits; then the places.  (One list of 131072 tokens by a single workgroup, which
// reads it with 25 GB/s, took 92 us, with T narrowed down by a sample first 60.)
//
// What bounds them is the chain of their steps, not the bytes (4 a token): 512 lists of 2112 tokens 11.7 us, 128 of 2000-16 384 14.9, 8 of 700 7.8;
// 2 of 131 072 in chunks 33 us, of which clearing 1-5, three passes 6.6 each, bits 4.8, places 9.0.  Where the choice is among equal
// weights, as of sums that are all 0, a chunk's workgroup reads those in front of its own, and the last one is the longest: 2 of 131 072
// equal ones 77 us, 2 of 2 000 000 1119 (unlike ones 106); 512 of 2112, in registers, 14.1.
// ------------------------------------------------------------------------------------------
struct SelectState {
  uint32_t least;  // of T, the bits that are known
  uint32_t need;   // how many of the weights that begin with them stay
  uint32_t cut;    // not all of them
  uint32_t unused;
};
struct SelectParams {
  const float* key_weights;
  const int32_t* page_indptr;
  const int32_t* weight_page_values;
  const int32_t* last_page_len;
  const int32_t* keep;
  int32_t* kept;
  // scratch memory
  uint64_t* words;  // four a block
  int32_t* counts;  // one a block
  SelectState* states;  // one a list
  uint32_t* histograms;  // (list, pass, kBins)
  uint32_t* arrivals;  // (list, pass): workgroups that have added their histogram
  int batch;
  int h_kv;
  int max_keep;
  int sinks;
  int recent;
  int page_shift;
};

constexpr uint32_t kOrderOfMinusInf = 0x007fffff, kOrderOfInf = 0xff800000;
__device__ __forceinline__ uint32_t weight_order(float w) {
  if (w != w) return 0;
  const uint32_t bits = __float_as_uint(w + 0.f);  // -0 + 0 = 0
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
// The smallest weight of this order or a larger one (but NaN): w >= weight_from(x) is weight_order(w) >= x for x > 0.
__device__ __forceinline__ float weight_from(uint32_t x) {
  x = min(max(x, kOrderOfMinusInf), kOrderOfInf);
  return __uint_as_float(x & 0x80000000u ? x ^ 0x80000000u : ~x);
}
__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~uint64_t{0} : (uint64_t{1} << n) - 1; }
// Sum of x over the lanes up to this one.
__device__ __forceinline__ int sum_of_lanes_up_to(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // from 1, 2, 4 and 8 lanes below in the row of 16
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // the row below's last to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31's to rows 2 and 3
  return x;
}
// Of a word that all lanes have: the lane's bit, the set bits of the lanes below it.
__device__ __forceinline__ bool bit_of_lane(uint64_t word) { return __builtin_amdgcn_inverse_ballot_w64(word); }
__device__ __forceinline__ int bits_below(uint64_t word, int and_these) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(word >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(word), and_these));
}
// The four words of a block, of 256 tokens.
struct BlockBits {
  uint64_t w[4];
  __device__ __forceinline__ int count() const { return __popcll(w[0]) + __popcll(w[1]) + __popcll(w[2]) + __popcll(w[3]); }
  // set bits of the tokens in front of the lane's, where all lanes have the block
  __device__ __forceinline__ int before() const { return bits_below(w[3], bits_below(w[2], bits_below(w[1], bits_below(w[0], 0)))); }
  // those of the tokens in front of the nth, or the others
  __device__ __forceinline__ BlockBits first(int n, bool others = false) const {
    BlockBits x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t mask = low_bits(max(n - i + 3, 0) >> 2);
      x.w[i] = w[i] & (others ? ~mask : mask);
    }
    return x;
  }
  __device__ __forceinline__ BlockBits inverse() const { return {{~w[0], ~w[1], ~w[2], ~w[3]}}; }
  // the token of the nth set bit
  __device__ __forceinline__ int nth(int n) const {
    int token = 0;
#pragma unroll
    for (int step = 128; step > 0; step >>= 1) token += first(token + step).count() <= n ? step : 0;
    return token;
  }
};
template <class Words>
__device__ __forceinline__ BlockBits load_block(Words words, int block) {
  BlockBits x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t word = words[block * 4 + i];
    x.w[i] = static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(word >> 32))) << 32 | static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(word)));
  }
  return x;
}

// What a list's lengths come to.
struct List {
  int page_begin, stored;
  int n, recent, sinks, places;  // tokens that stay: all, the last ones, the first ones; places in front of the recent ones' 
  int gone;
  int end;  // candidates: tokens [sinks, end), of which places - sinks stay and at least one does not
  __device__ __forceinline__ List(const SelectParams& p, int b, int page_begin, int stored) : page_begin(page_begin), stored(stored) {
    n = min(stored, max(min(p.keep[b], p.max_keep), 0));
    recent = min(p.recent, n);
    sinks = min(p.sinks, n - recent);
    places = n - recent;
    gone = stored - n;
    end = stored - recent;
  }
  __device__ __forceinline__ bool no_choice() const { return gone == 0 || places == sinks; }
  __device__ __forceinline__ int num_blocks() const { return (end + 255) >> 8; }
  // Four tokens' weights, by their group of four; a group behind the end is the last one (its tokens are none).
  __device__ __forceinline__ int page_of(const SelectParams& p, int group) const {
    return p.weight_page_values[page_begin + (min(group, (end - 1) >> 2) >> (p.page_shift - 2))];
  }
  __device__ __forceinline__ float4_any_t weights_of(const SelectParams& p, int kvh, int page, int group) const {
    const int in_page = min(group, (end - 1) >> 2) * 4 & ((1 << p.page_shift) - 1);
    return *reinterpret_cast<const float4_any_t*>(p.key_weights + ((static_cast<int64_t>(page) * p.h_kv + kvh) << p.page_shift) + in_page);
  }
  // a block's candidates for which `is` holds
  template <class Is>
  __device__ __forceinline__ BlockBits candidates(int block, float4_any_t w, Is is) const {
    BlockBits x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x.w[i] = __ballot(is(w[i]));
    if (block * 256 < sinks || block * 256 + 256 > end) x = x.first(end - block * 256).first(sinks - block * 256, true);
    return x;
  }
  template <class Add>
  __device__ __forceinline__ void add_candidates(int block, float4_any_t w, int lane, Add add) const {
    const int t = block * 256 + lane * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (t + i >= sinks && t + i < end) add(weight_order(w[i]));
    }
  }
  // Bits of the tokens in front of the recent ones that stay.  equal_before: weights equal to T in front of the block, where only the
  // first `need` of them stay.
  __device__ __forceinline__ BlockBits stay(int block, float4_any_t w, const SelectState& t, int equal_before) const {
    const float smallest = weight_from(t.least);
    BlockBits x = candidates(block, w, [&](float v) { return t.least == 0 || v >= smallest; });
    if (t.cut) {
      const BlockBits equal = equal_to(block, w, t);
      int rank = equal_before + equal.before();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool mine = bit_of_lane(equal.w[i]);
        x.w[i] &= ~__ballot(mine && rank >= static_cast<int>(t.need));
        rank += mine;
      }
    }
    if (block * 256 < sinks) {
      const BlockBits first = BlockBits{{~uint64_t{0}, ~uint64_t{0}, ~uint64_t{0}, ~uint64_t{0}}}.first(sinks - block * 256);
#pragma unroll
      for (int i = 0; i < 4; ++i) x.w[i] |= first.w[i];
    }
    return x;
  }
  __device__ __forceinline__ BlockBits equal_to(int block, float4_any_t w, const SelectState& t) const {
    const float smallest = weight_from(t.least);
    return candidates(block, w, [&](float v) { return t.least == 0 ? v != v : v == smallest; });
  }
  // Free places up to the block with the first token behind the places, tokens without a place from that block on.
  __device__ __forceinline__ int boundary() const { return places >> 8; }
  __device__ __forceinline__ BlockBits holes_in(const BlockBits& x, int block) const {
    return block < boundary() ? x.inverse() : x.inverse().first(block == boundary() ? places & 255 : 0);
  }
  __device__ __forceinline__ BlockBits homeless_in(const BlockBits& x, int block) const {
    return block > boundary() ? x : x.first(block == boundary() ? places & 255 : 256, true);
  }
};
template <class Words>
__device__ __forceinline__ BlockBits any_block(Words words, int block) {
  return {{words[block * 4], words[block * 4 + 1], words[block * 4 + 2], words[block * 4 + 3]}};
}
// The token without a place of a rank; counts: up to the boundary anything, behind it such tokens in front of the block.
template <class Words, class Counts>
__device__ __forceinline__ int homeless_of_rank(const List& l, Words words, Counts counts, int rank) {
  const BlockBits first = l.homeless_in(any_block(words, l.boundary()), l.boundary());
  if (rank < first.count()) return l.boundary() * 256 + first.nth(rank);
  int lo = l.boundary() + 1, hi = l.num_blocks() - 1;  // the last block that begins at or in front of the rank
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (counts[mid] <= rank) lo = mid; else hi = mid - 1;
  }
  return lo * 256 + any_block(words, lo).nth(rank - counts[lo]);
}
// Sums of two numbers over the threads in front of this one.
template <int WAVES>
__device__ __forceinline__ int2 sums_in_front(int (&shared)[2][WAVES], int a, int c, int wave, int lane) {
  const int a_to = sum_of_lanes_up_to(a), c_to = sum_of_lanes_up_to(c);
  __syncthreads();
  if (lane == 63) {
    shared[0][wave] = a_to;
    shared[1][wave] = c_to;
  }
  __syncthreads();
  int2 front = make_int2(a_to - a, c_to - c);
#pragma unroll
  for (int w = 0; w < WAVES - 1; ++w) {
    front.x += w < wave ? shared[0][w] : 0;
    front.y += w < wave ? shared[1][w] : 0;
  }
  return front;
}
// Where a list's blocks are in scratch memory: as many as the pages of the sequences in front could have.
__device__ __forceinline__ int64_t blocks_at(const SelectParams& p, const List& l, int b, int kvh) {
  return (((static_cast<int64_t>(l.page_begin - p.page_indptr[0]) << p.page_shift) >> 8) + b) * p.h_kv + static_cast<int64_t>(kvh) * l.num_blocks();
}
__device__ __forceinline__ void no_choice_made(const SelectParams& p, const List& l, int32_t* kept, int thread, int threads) {
  for (int i = l.places + thread; i < p.max_keep; i += threads) kept[i] = i < l.n ? i + l.gone : -1;
  if (l.no_choice()) {
    for (int i = thread; i < l.places; i += threads) kept[i] = i;
  }
}

template <int THREADS, int HELD, int BLOCKS, int LISTED, int COPIES>
__global__ __launch_bounds__(THREADS) void select_kept_kernel(SelectParams p) {
  constexpr int WAVES = THREADS / 64;
  __shared__ uint64_t lds_words[BLOCKS * 4];
  __shared__ int32_t lds_counts[BLOCKS];
  __shared__ int32_t homeless_lds[LISTED];
  __shared__ uint32_t histogram[256 * COPIES];  // lanes take turns: most weights fall into a few of the first pass's bins
  __shared__ uint32_t bins[256];
  __shared__ int per_wave[2][WAVES];
  __shared__ uint32_t found[3];
  __shared__ int num_homeless;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x, b = blockIdx.y;
  const int page_begin = p.page_indptr[b], num_pages = p.page_indptr[b + 1] - page_begin;
  const List l(p, b, page_begin, num_pages > 0 ? ((num_pages - 1) << p.page_shift) + p.last_page_len[b] : 0);
  int32_t* const kept = p.kept + (static_cast<int64_t>(b) * p.h_kv + kvh) * p.max_keep;
  no_choice_made(p, l, kept, tid, THREADS);
  if (l.no_choice()) return;
  const int num_blocks = l.num_blocks();
  float4_any_t held[HELD];  // of blocks wave, wave + WAVES, ..
  const auto hold = [&](int k0) {
    int page[HELD];
#pragma unroll
    for (int u = 0; u < HELD; ++u) page[u] = l.page_of(p, (k0 + u * WAVES) * 64 + lane);
#pragma unroll
    for (int u = 0; u < HELD; ++u) held[u] = l.weights_of(p, kvh, page[u], (k0 + u * WAVES) * 64 + lane);
  };
  const bool in_registers = num_blocks <= WAVES * HELD;
  hold(wave);
  // f(block, the lane's weights) for every block; all lanes of a wave take the same steps
  const auto every_block = [&](auto&& f) {
#pragma unroll 1
    for (int k0 = wave; k0 < num_blocks; k0 += HELD * WAVES) {
      if (!in_registers) hold(k0);
#pragma unroll
      for (int u = 0; u < HELD; ++u) {
        if (k0 + u * WAVES < num_blocks) f(k0 + u * WAVES, held[u]);
      }
    }
  };
  SelectState t = {0, static_cast<uint32_t>(l.places - l.sinks), 1, 0};
#pragma unroll 1
  for (int shift = 24; shift >= 0 && t.cut; shift -= 8) {
    for (int i = tid; i < 256 * COPIES; i += THREADS) histogram[i] = 0;
    __syncthreads();
    every_block([&](int block, float4_any_t w) {
      l.add_candidates(block, w, lane, [&](uint32_t x) {
        if (shift == 24 || ((x ^ t.least) >> shift) < 256) atomicAdd(&histogram[(x >> shift & 255) * COPIES + (lane & (COPIES - 1))], 1u);
      });
    });
    __syncthreads();
    constexpr int SHARE = THREADS / 256;  // threads that add a bin's copies up
    static_assert(SHARE == 1 || SHARE == 4, "a thread or four lanes");
    uint32_t copies = 0;
#pragma unroll
    for (int c = 0; c < COPIES / SHARE; ++c) copies += histogram[tid / SHARE * COPIES + ((tid % SHARE * (COPIES / SHARE) + c + tid / SHARE) & (COPIES - 1))];
    if (SHARE == 4) {
      copies += __builtin_amdgcn_update_dpp(0, copies, kDppXor1, 0xf, 0xf, true);
      copies += __builtin_amdgcn_update_dpp(0, copies, kDppXor2, 0xf, 0xf, true);
    }
    if (tid % SHARE == 0) bins[255 - tid / SHARE] = copies;  // the largest digit first
    __syncthreads();
    if (wave == 0) {
      uint32_t mine[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += mine[i] = bins[lane * 4 + i];
      uint32_t above = sum_of_lanes_up_to(sum) - sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (above < t.need && t.need <= above + mine[i]) {
          found[0] = 255 - (lane * 4 + i);
          found[1] = t.need - above;
          found[2] = mine[i];
        }
        above += mine[i];
      }
    }
    __syncthreads();
    t.least |= found[0] << shift;
    t.need = found[1];
    t.cut = found[1] != found[2];  // otherwise all weights with these bits stay
  }

  // A range of blocks a thread, for the running counts.
  const int per = (num_blocks + THREADS - 1) / THREADS, block_lo = min(tid * per, num_blocks), block_hi = min(block_lo + per, num_blocks);
  const auto finish = [&](auto* words, auto* counts) {
    if (t.cut) {  // weights equal to T in front of each block
      every_block([&](int block, float4_any_t w) {
        const BlockBits equal = l.equal_to(block, w, t);
        if (lane == 0) counts[block] = equal.count();
      });
      __syncthreads();
      int equal = 0;
      for (int k = block_lo; k < block_hi; ++k) equal += counts[k];
      int front = sums_in_front(per_wave, equal, 0, wave, lane).x;
      for (int k = block_lo; k < block_hi; ++k) {
        const int here = counts[k];
        counts[k] = front;
        front += here;
      }
      __syncthreads();
    }
    every_block([&](int block, float4_any_t w) {
      const BlockBits x = l.stay(block, w, t, t.cut ? counts[block] : 0);
      if (lane < 4) words[block * 4 + lane] = lane == 0 ? x.w[0] : lane == 1 ? x.w[1] : lane == 2 ? x.w[2] : x.w[3];
    });
    __syncthreads();
    int holes = 0, homeless = 0;
    for (int k = block_lo; k < block_hi; ++k) {
      const BlockBits x = any_block(words, k);
      holes += l.holes_in(x, k).count();
      homeless += l.homeless_in(x, k).count();
    }
    int2 front = sums_in_front(per_wave, holes, homeless, wave, lane);
    // counts of a block: up to the boundary the holes in front of it, behind it the tokens without a place in front of it
    for (int k = block_lo; k < block_hi; ++k) {
      const BlockBits x = any_block(words, k);
      counts[k] = k <= l.boundary() ? front.x : front.y;
      front.x += l.holes_in(x, k).count();
      front.y += l.homeless_in(x, k).count();
    }
    if (tid == THREADS - 1) num_homeless = front.y;
    __syncthreads();
    // Tokens without a place, in order, where they are few enough; else a place looks for its own.
    const bool listed = num_homeless <= LISTED;
    if (listed) {
      for (int k = l.boundary() + wave; k < num_blocks; k += WAVES) {
        const BlockBits x = l.homeless_in(load_block(words, k), k);
        int rank = (k == l.boundary() ? 0 : counts[k]) + x.before();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool mine = bit_of_lane(x.w[i]);
          if (mine) homeless_lds[rank] = k * 256 + lane * 4 + i;
          rank += mine;
        }
      }
      __syncthreads();
    }
    for (int k = wave; k * 256 < l.places; k += WAVES) {
      const BlockBits x = l.holes_in(load_block(words, k), k);
      const int at = k * 256 + lane * 4;
      int rank = counts[k] + x.before();
      int4_any_t from;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool hole = bit_of_lane(x.w[i]);
        from[i] = !hole ? at + i : listed ? homeless_lds[rank] : homeless_of_rank(l, words, counts, rank);
        rank += hole;
      }
      if (at + 4 <= l.places) {
        *reinterpret_cast<int4_any_t*>(kept + at) = from;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (at + i < l.places) kept[at + i] = from[i];
        }
      }
    }
  };
  if (num_blocks <= BLOCKS) {
    finish(lds_words, lds_counts);
  } else {
    const int64_t at = blocks_at(p, l, b, kvh);
    finish(p.words + at * 4, p.counts + at);
  }
}

// Long lists, in chunks of 16 blocks.
constexpr int kChunkShift = 12, kBins = 2048, kSelectPasses = 3;
constexpr int64_t kMostChunkedBlocks = 8192;  // whose counts a workgroup of the last launch keeps
__global__ __launch_bounds__(256) void select_clear_kernel(uint32_t* words, int64_t count) {
  for (int64_t i = blockIdx.x * int64_t{256} + threadIdx.x; i < count; i += gridDim.x * int64_t{256}) words[i] = 0;
}
// The list and the chunk of a workgroup of the other launches; a list without a choice has no chunks.
struct Chunk {
  int b, kvh, first_block;
  __device__ __forceinline__ Chunk(const SelectParams& p, int lane, SequenceOf& s) {
    kvh = blockIdx.x % p.h_kv;
    const int slot = blockIdx.x / p.h_kv;
    s = sequence_of_slot(p.page_indptr, p.last_page_len, p.batch, p.page_shift, kChunkShift, slot, lane);
    b = s.index;
    first_block = (slot - s.slot_begin) << (kChunkShift - 8);
  }
};

__global__ __launch_bounds__(256) void select_pass_kernel(SelectParams p, int nth) {
  __shared__ uint32_t histogram[kBins];
  __shared__ int per_wave[2][4];
  __shared__ int is_last;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  SequenceOf s;
  const Chunk c(p, lane, s);
  const List l(p, c.b, s.page_begin, s.stored(p.page_shift));
  if (l.no_choice() || c.first_block >= l.num_blocks()) return;
  const int64_t list = static_cast<int64_t>(c.b) * p.h_kv + c.kvh;
  SelectState t = {0, static_cast<uint32_t>(l.places - l.sinks), 1, 0};
  if (nth > 0) t = p.states[list];
  if (!t.cut) return;  // T is known well enough
  const int shift = nth == 0 ? 21 : nth == 1 ? 10 : 0, digits = nth == 2 ? 1023 : 2047;
  int page[4];
  float4_any_t w[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) page[u] = l.page_of(p, (c.first_block + wave + 4 * u) * 64 + lane);
#pragma unroll
  for (int u = 0; u < 4; ++u) w[u] = l.weights_of(p, c.kvh, page[u], (c.first_block + wave + 4 * u) * 64 + lane);
  for (int i = tid; i < kBins; i += 256) histogram[i] = 0;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    l.add_candidates(c.first_block + wave + 4 * u, w[u], lane, [&](uint32_t x) {
      if (nth == 0 || (x ^ t.least) >> shift <= static_cast<uint32_t>(digits)) atomicAdd(&histogram[x >> shift & digits], 1u);
    });
  }
  __syncthreads();
  uint32_t* const all = p.histograms + (list * kSelectPasses + nth) * kBins;
  for (int i = tid; i < kBins; i += 256) {
    if (histogram[i] != 0) __hip_atomic_fetch_add(all + i, histogram[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  wait_vmcnt<0>();
  __syncthreads();
  if (tid == 0) {
    const uint32_t chunks = (l.num_blocks() + 15) >> 4;
    is_last = __hip_atomic_fetch_add(p.arrivals + list * kSelectPasses + nth, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == chunks - 1;
  }
  __syncthreads();
  if (!is_last) return;
  constexpr int EACH = kBins / 256;
  uint32_t mine[EACH], sum = 0;  // the largest digit first
#pragma unroll
  for (int i = 0; i < EACH; ++i) mine[i] = __hip_atomic_load(all + kBins - 1 - (tid * EACH + i), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
  for (int i = 0; i < EACH; ++i) sum += mine[i];
  uint32_t above = sums_in_front(per_wave, static_cast<int>(sum), 0, wave, lane).x;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (above < t.need && t.need <= above + mine[i]) {
      const uint32_t left = t.need - above;
      p.states[list] = {t.least | static_cast<uint32_t>(kBins - 1 - (tid * EACH + i)) << shift, left, left != mine[i], 0};
    }
    above += mine[i];
  }
}

__global__ __launch_bounds__(256) void select_bits_kernel(SelectParams p) {
  __shared__ int per_wave[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  SequenceOf s;
  const Chunk c(p, lane, s);
  const List l(p, c.b, s.page_begin, s.stored(p.page_shift));
  if (l.no_choice() || c.first_block >= l.num_blocks()) return;
  const SelectState t = p.states[static_cast<int64_t>(c.b) * p.h_kv + c.kvh];
  // (a wave has neighbouring blocks here)
  const int block0 = c.first_block + 4 * wave;
  int page[4];
  float4_any_t w[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) page[u] = l.page_of(p, (block0 + u) * 64 + lane);
#pragma unroll
  for (int u = 0; u < 4; ++u) w[u] = l.weights_of(p, c.kvh, page[u], (block0 + u) * 64 + lane);
  int equal_before = 0;
  if (t.cut) {  // weights equal to T in front of the wave's: its workgroup counts them in the chunks in front of its own, a load a step
    int equal = 0;
    for (int k = wave; k < c.first_block; k += 4) {
      const int group = k * 64 + lane;
      equal += l.equal_to(k, l.weights_of(p, c.kvh, l.page_of(p, group), group), t).count();
    }
    int own = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) own += block0 + u < l.num_blocks() ? l.equal_to(block0 + u, w[u], t).count() : 0;
    if (lane == 0) per_wave[wave] = equal;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) equal_before += per_wave[i];
    __syncthreads();
    if (lane == 0) per_wave[wave] = own;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) equal_before += i < wave ? per_wave[i] : 0;
  }
  const int64_t at = blocks_at(p, l, c.b, c.kvh);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int block = block0 + u;
    if (block >= l.num_blocks()) break;
    const BlockBits x = l.stay(block, w[u], t, equal_before);
    if (t.cut) equal_before += l.equal_to(block, w[u], t).count();
    if (lane < 4) p.words[(at + block) * 4 + lane] = lane == 0 ? x.w[0] : lane == 1 ? x.w[1] : lane == 2 ? x.w[2] : x.w[3];
  }
}

// Places, a block of them a wave (each looks for its token: 23 us with four blocks a wave); lists without a choice, too.
__global__ __launch_bounds__(256) void select_places_kernel(SelectParams p) {
  __shared__ int32_t counts[kMostChunkedBlocks];
  __shared__ int per_wave[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int page_begin = p.page_indptr[b], num_pages = p.page_indptr[b + 1] - page_begin;
  const List l(p, b, page_begin, num_pages > 0 ? ((num_pages - 1) << p.page_shift) + p.last_page_len[b] : 0);
  int32_t* const kept = p.kept + (static_cast<int64_t>(b) * p.h_kv + kvh) * p.max_keep;
  no_choice_made(p, l, kept, blockIdx.x * 256 + tid, gridDim.x * 256);
  const int first_block = blockIdx.x * 4;
  if (l.no_choice() || first_block * 256 >= l.places) return;
  const uint64_t* const words = p.words + blocks_at(p, l, b, kvh) * 4;
  const int num_blocks = l.num_blocks();
  const int per = (num_blocks + 255) / 256, block_lo = min(tid * per, num_blocks), block_hi = min(block_lo + per, num_blocks);
  int holes = 0, homeless = 0;
  for (int k = block_lo; k < block_hi; ++k) {
    const BlockBits x = any_block(words, k);
    holes += l.holes_in(x, k).count();
    homeless += l.homeless_in(x, k).count();
  }
  int2 front = sums_in_front(per_wave, holes, homeless, wave, lane);
  for (int k = block_lo; k < block_hi; ++k) {
    const BlockBits x = any_block(words, k);
    counts[k] = k <= l.boundary() ? front.x : front.y;
    front.x += l.holes_in(x, k).count();
    front.y += l.homeless_in(x, k).count();
  }
  __syncthreads();
  const int k = first_block + wave;
  if (k * 256 < l.places) {
    const BlockBits x = l.holes_in(load_block(words, k), k);
    const int at = k * 256 + lane * 4;
    int rank = counts[k] + x.before();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool hole = bit_of_lane(x.w[i]);
      if (at + i < l.places) kept[at + i] = hole ? homeless_of_rank(l, words, counts, rank) : at + i;
      rank += hole;
    }
  }
}

// ------------------------------------------------------------------------------------------
// The move: row kept[i] to place i, in place; kept[i] is never in front of i, so that rows taken in order are still there when they
// are needed.  Where lists (sequence, kv head) are many or short, a workgroup fills all places of one, with a part of each row's bytes:
// it reads the rows of a few places, waits until all its waves have theirs, and writes.  Where they are few and long, a range of places is a
// workgroup's, in two launches: with n entries in the list and s the first place that is also a source (n if none is), the places in
// front of s can be filled in any order, none of the rows that they need is written meanwhile, and the first launch does it.  The
// second fills the others: in any order again if none of them is the source of one of them, else (recent tokens that move by fewer
// places than they are) in order as above.  Entries that name no token behind their place are passed over.
//
// Bytes alone, each moved row read and written once: 512 lists of 2112 tokens to 2048 (8 kv heads of dim 128) 40 us, 128 of 2000-16 384 to
// 2048 45, 4.4 and 4.5 TB/s where a large copy makes 5.2; rows of 256 bytes from all over the pool, a row's two parts in different pages.
// 2 lists of 131 072 to 16 384 (dim 256) by ranges 20 + 11 us, 3 TB/s in the first launch.
// ------------------------------------------------------------------------------------------
struct MoveParams {
  uint8_t* pages;
  float* key_weights;  // or NULL
  const int32_t* page_indptr;
  const int32_t* page_values;
  const int32_t* weight_page_values;
  const int32_t* kept;
  int h_kv;
  int max_keep;
  int page_shift;
  int pieces;            // of 16 bytes in the rows of K and V together
  int slices;            // parts of them that workgroups have which fill places in order
  ExactDivision by_row;  // pieces, pieces / slices
  ExactDivision by_slice;
};
constexpr int kMoveThreads = 256;
constexpr int kMoveWaves = kMoveThreads / 64;

// shared: words that no thread reads any more; they are free again afterwards.
__device__ __forceinline__ int smallest_of_workgroup(int x, int* shared, int wave, int lane) {
  x = min(x, __builtin_amdgcn_update_dpp(x, x, kDppXor1, 0xf, 0xf, false));
  x = min(x, __builtin_amdgcn_update_dpp(x, x, kDppXor2, 0xf, 0xf, false));
  x = min(x, __builtin_amdgcn_update_dpp(x, x, kDppRowHalfMirror, 0xf, 0xf, false));
  x = min(x, __builtin_amdgcn_update_dpp(x, x, kDppRowMirror, 0xf, 0xf, false));
  x = min(min(__builtin_amdgcn_readlane(x, 0), __builtin_amdgcn_readlane(x, 16)), min(__builtin_amdgcn_readlane(x, 32), __builtin_amdgcn_readlane(x, 48)));
  if (lane == 0) shared[wave] = x;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMoveWaves; ++w) x = min(x, shared[w]);
  __syncthreads();  // every wave has read them: the words are free again
  return x;
}

// Rows are read once and written once, and there are more of them than caches hold: both with the streaming hint (131072 tokens to
// 16384 95 -> 88 us).
__device__ __forceinline__ void st16_nt(void* p, const Vec16& v) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  __builtin_nontemporal_store(u32x4{v.w[0], v.w[1], v.w[2], v.w[3]}, reinterpret_cast<u32x4*>(p));
}
enum MoveLaunch { kMoveInOrder, kMoveFirst, kMoveSecond };
template <MoveLaunch LAUNCH>
__global__ __launch_bounds__(kMoveThreads) void move_kept_kernel(MoveParams p) {
  constexpr int EACH = 8;  // places a thread looks at before their rows are moved
  __shared__ uint2 list[kMoveThreads * EACH];  // K's rows in the pool: of a place, of its source
  __shared__ int per_wave[EACH][kMoveWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int part = blockIdx.x, parts = gridDim.x, kvh = blockIdx.y, b = blockIdx.z;
  const int page_begin = p.page_indptr[b], capacity = (p.page_indptr[b + 1] - page_begin) << p.page_shift;
  const int32_t* const kept = p.kept + (static_cast<int64_t>(b) * p.h_kv + kvh) * p.max_keep;
  const int in_page = (1 << p.page_shift) - 1;
  const auto moves = [&](int i, int from) { return from > i && from < capacity; };
  int lo = 0, hi = min(p.max_keep, capacity);
  bool in_order = LAUNCH == kMoveInOrder;
  if constexpr (LAUNCH != kMoveInOrder) {
    // what the list says: its smallest source, the place behind its last one that a row moves to
    int least = INT32_MAX, last = 0;
    const auto look = [&](int begin, int end) {
      for (int i0 = begin + tid * 4; i0 < end; i0 += EACH * kMoveThreads * 4) {
        int4_any_t from[EACH];
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
          const int i = i0 + u * kMoveThreads * 4;
          if (i + 4 <= end) {
            from[u] = *reinterpret_cast<const int4_any_t*>(kept + i);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) from[u][k] = i + k < end ? kept[i + k] : -1;
          }
        }
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int i = i0 + u * kMoveThreads * 4 + k;
            if (moves(i, from[u][k])) {
              least = min(least, from[u][k]);
              last = max(last, i + 1);
            }
          }
        }
      }
    };
    look(0, hi);
    const int n = -smallest_of_workgroup(-last, per_wave[0], wave, lane);
    hi = min(smallest_of_workgroup(least, per_wave[0], wave, lane), n);
    if constexpr (LAUNCH == kMoveSecond) {
      lo = hi;
      hi = n;
      if (lo >= hi) return;
      least = INT32_MAX;
      look(lo, hi);
      in_order = smallest_of_workgroup(least, per_wave[0], wave, lane) < n;
    }
  }
  int y0 = 0, width = p.pieces;
  const ExactDivision by_width = in_order ? p.by_slice : p.by_row;
  if (in_order) {
    if (part >= p.slices) return;
    width = p.pieces / p.slices;
    y0 = part * width;
  } else {
    const int each = (hi - lo + parts - 1) / parts;
    lo += part * each;
    hi = min(lo + each, hi);
  }
  const bool with_sums = p.key_weights != nullptr && y0 == 0;
  const auto sum_at = [&](int page, int t) { return p.key_weights + ((static_cast<int64_t>(page) * p.h_kv + kvh) << p.page_shift) + (t & in_page); };
  const auto row_at = [&](int page, int t) { return ((static_cast<uint32_t>(page) * 2 * p.h_kv + kvh) << p.page_shift) + (t & in_page); };
  const int half = p.pieces >> 1;  // a row's pieces of K, then those of V, which are so many rows behind
  const uint32_t to_v = static_cast<uint32_t>(p.h_kv) << p.page_shift;
  const auto piece_at = [&](uint32_t row, int y) {
    const bool v = y >= half;
    return p.pages + (static_cast<int64_t>(row + (v ? to_v : 0)) * half + (y - (v ? half : 0))) * 16;
  };
  // Loads are complete, not only issued, where a workgroup goes on to overwrite what they read.
  const auto all_have_read = [&] {
    if (in_order) {
      wait_vmcnt<0>();
      __syncthreads();
    }
  };
  for (int i0 = lo; i0 < hi; i0 += kMoveThreads * EACH) {
    int from[EACH], at[EACH];
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      const int i = i0 + u * kMoveThreads + tid;
      from[u] = i < hi ? kept[i] : -1;
    }
    // the pages of places and sources, of K / V and of the sums, where there is something to move
    int page[EACH], page_from[EACH];
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      const int i = i0 + u * kMoveThreads + tid;
      if (!moves(i, from[u])) from[u] = -1;
      if (from[u] >= 0) {
        page[u] = p.page_values[page_begin + (i >> p.page_shift)];
        page_from[u] = p.page_values[page_begin + (from[u] >> p.page_shift)];
      }
      const uint64_t who = __ballot(from[u] >= 0);
      at[u] = __popcll(who & ((uint64_t{1} << lane) - 1));
      if (lane == 0) per_wave[u][wave] = __popcll(who);
    }
    __syncthreads();
    int count = 0;
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
#pragma unroll
      for (int w = 0; w < kMoveWaves; ++w) {
        at[u] += w == wave ? count : 0;
        count += per_wave[u][w];
      }
      if (from[u] >= 0) list[at[u]] = make_uint2(row_at(page[u], i0 + u * kMoveThreads + tid), row_at(page_from[u], from[u]));
    }
    if (with_sums) {
      float* to[EACH];
      float sum[EACH];
#pragma unroll
      for (int u = 0; u < EACH; ++u) {
        if (from[u] >= 0) {
          const int i = i0 + u * kMoveThreads + tid;
          to[u] = sum_at(p.weight_page_values[page_begin + (i >> p.page_shift)], i);
          sum[u] = *sum_at(p.weight_page_values[page_begin + (from[u] >> p.page_shift)], from[u]);
        }
      }
      all_have_read();
#pragma unroll
      for (int u = 0; u < EACH; ++u) {
        if (from[u] >= 0) *to[u] = sum[u];
      }
    }
    __syncthreads();
    constexpr int U = 8;
    const int total = count * width;
    for (int x0 = 0; x0 < total; x0 += kMoveThreads * U) {
      Vec16 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int x = x0 + u * kMoveThreads + tid, row = by_width(x);
        if (x < total) v[u] = ld16_nt(piece_at(list[row].y, y0 + x - row * width));
      }
      all_have_read();
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int x = x0 + u * kMoveThreads + tid, row = by_width(x);
        if (x < total) st16_nt(piece_at(list[row].x, y0 + x - row * width), v[u]);
      }
    }
    __syncthreads();  // the list has been read
  }
}

// ------------------------------------------------------------------------------------------
// Launches
// ------------------------------------------------------------------------------------------
static int shift_of_page(const char* what, int32_t page_size) {
  KV_UNSUPPORTED(page_size < 16 || page_size > 128 || (page_size & (page_size - 1)) != 0)
      << what << ": page_size " << page_size << " is not built (16, 32, 64, 128)";
  int shift = 4;
  while ((1 << shift) < page_size) ++shift;
  return shift;
}
static void check_table(const char* what, int32_t batch, int64_t nnz_pages, int32_t h_kv, int32_t page_size) {
  KV_CHECK(batch >= 0 && nnz_pages >= 0 && h_kv > 0) << what << ": bad shape";
  KV_CHECK(nnz_pages <= (int64_t{1} << 30) / page_size) << what << ": too many pages";  // tokens are 30-bit numbers
}
static void check_aligned16(const char* what, std::initializer_list<const void*> tensors) {
  for (const void* t : tensors)
    KV_CHECK(reinterpret_cast<uintptr_t>(t) % 16 == 0) << what << ": q, pages and output must be aligned to 16 bytes";
}

// Bytes of a decode call's kept scores, a limit on memory: keeping them is faster wherever it was measured (102 MB 341 us, K read again 458).
constexpr size_t kMostKept = size_t{1} << 29;

static KeyWeightsParams weights_of_call(const void* q, const int32_t* q_indptr, const void* pages, const int32_t* page_indptr,
                                        const int32_t* page_values, const int32_t* length_info, const float* lse, float* key_weights,
                                        const int32_t* weight_page_values, bool causal, int64_t observed, double sm_scale, int32_t batch_size,
                                        int32_t h_q, int32_t h_kv, int page_shift) {
  KeyWeightsParams p{};
  p.q = static_cast<const half_t*>(q);
  p.pages = static_cast<const half_t*>(pages);
  p.q_indptr = q_indptr;
  p.page_indptr = page_indptr;
  p.page_values = page_values;
  p.weight_page_values = weight_page_values;
  p.last_page_len = length_info;
  p.lse = lse;
  p.key_weights = key_weights;
  p.batch = batch_size;
  p.h_q = h_q;
  p.h_kv = h_kv;
  p.group = h_q / h_kv;
  p.by_group = ExactDivision::by(p.group);
  p.inv_group = (65536 + p.group - 1) / p.group;
  p.causal = causal;
  p.observed = static_cast<int>(std::min<int64_t>(observed, INT32_MAX));
  p.page_shift = page_shift;
  p.scale_log2 = static_cast<float>(sm_scale) * kLog2e;
  return p;
}
// The sums from q, K and the lse that attention has written.
static void add_key_weights(const char* what, KeyWeightsParams p, int64_t total_q, int64_t nnz_pages, int32_t d, hipStream_t stream) {
  const int64_t batch_size = p.batch, h_kv = p.h_kv;
  const int page_shift = p.page_shift;
  if (batch_size == 0 || nnz_pages == 0) return;
  const int64_t rows = (p.observed > 0 ? std::min<int64_t>(total_q, p.observed * batch_size) : total_q) * p.group;  // that count, at most
  p.nnz_pages = static_cast<int>(nnz_pages);
  const auto launch = [&](auto dim, auto blocks) {
    constexpr int D = decltype(dim)::value, TB = decltype(blocks)::value;
    const int64_t tokens = nnz_pages << page_shift, items = (tokens / (128 * TB) + batch_size) * h_kv;
    KV_CHECK(items < (int64_t{1} << 31)) << what << ": too many work items";
    // Few workgroups of many rows share these: two workgroups a compute unit, or four where each has a long way to go, of two row tiles at
    // least, by the average sequence; two shares only where they save more than the second launch costs.  Whole calls alone / shared, us (query
    // heads / kv heads x dim):
    //   1 x 2048 tokens 32/8x128 216 / 96, on 8000 cached 567 / 522; 1 x 500 on 2000 88 / 65; 2 x 1000 64/8x128 305 / 235; 8 x 512 16/2x64 95 / 35;
    //   2 x 25-241 on 79-315 40/1x96 173 / 28; 27 x 14-973 40/1x96 913 / 264; not shared: 37 x 9/3x96, 18 tiles on 243 workgroups, 68 / 80,
    //   1 x 114 32/8x128, 7 tiles on 8, 16 / 18
    const int64_t tiles = rows / (batch_size * WeightTiles<D, TB>::kRows), per_unit = tiles >= 96 ? 4 : 2;
    int64_t shares = std::min<int64_t>({per_unit * compute_units() / items, tiles / 2, 32});
    if (tiles < 9 || shares < 2 || (shares == 2 && tiles < 28)) shares = 1;
    ScratchLease ws{};
    if (shares > 1) {
      ws = lease_scratch(kScratchKept, stream, static_cast<size_t>(shares) * tokens * h_kv * sizeof(float), 0);
      p.shares = reinterpret_cast<float*>(ws.ptr);
    }
    hipLaunchKernelGGL((key_weights_kernel<D, TB>), dim3(static_cast<unsigned>(items), static_cast<unsigned>(shares)), dim3(256), 0, stream, p);
    if (shares > 1) {
      const int64_t sums = ((tokens >> kSharedTokensShift) + batch_size) * h_kv;
      hipLaunchKernelGGL(shared_rows_kernel, dim3(static_cast<unsigned>(sums)), dim3(256), 0, stream, p, static_cast<int>(shares));
    }
  };
  // 64 tokens a wave instead of 32 where rows are many: half as much of q is read, by fewer waves.  32 / 64 tokens, whole calls in us:
  //   dim 128   1 x 64 queries on 2000 31.2 / 33.7 (256 rows), 64 x 64 on 1000 196.9 / 194.2, 8 x 1500 on 2000 944 / 925 (6000 rows)
  //   dim 96    28.5 / 29.7, 178.5 / 172.8, 875 / 853
  //   dim 64    24.5 / 26.1, 129.7 / 140.8, 621 / 601; 8 x 256 on 2000 103 / 108 (1024 rows), 1 x 2048 77.8 / 73.8 (8192)
  const bool many_rows = rows >= int64_t{d == 64 ? 4096 : 256} * batch_size;
  const auto launch_blocks = [&](auto dim) {
    if (many_rows) launch(dim, std::integral_constant<int, 2>{}); else launch(dim, std::integral_constant<int, 1>{});
  };
  if (d == 64) launch_blocks(std::integral_constant<int, 64>{});
  if (d == 80) launch_blocks(std::integral_constant<int, 80>{});
  if (d == 96) launch_blocks(std::integral_constant<int, 96>{});
  if (d == 112) launch_blocks(std::integral_constant<int, 112>{});
  if (d == 128) launch_blocks(std::integral_constant<int, 128>{});
  if (d == 256) launch(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
  KV_LAUNCH_CHECK();
}

static void check_attention(const char* what, const void* q, const void* pages, const int32_t* page_indptr, const int32_t* page_values,
                            const int32_t* length_info, const void* output, const float* lse, const float* key_weights,
                            const int32_t* weight_page_values, int32_t batch_size, int64_t nnz_pages, int32_t h_q, int32_t h_kv, int32_t d,
                            int32_t page_size) {
  KV_CHECK(h_q > 0 && h_kv > 0 && h_q % h_kv == 0) << what << ": bad shape";
  KV_UNSUPPORTED(!tuned_head_dim(d)) << what << ": head_dim " << d << " is not built (64, 80, 96, 112, 128, 256)";
  shift_of_page(what, page_size);
  check_table(what, batch_size, nnz_pages, h_kv, page_size);
  if (batch_size == 0) return;
  KV_CHECK(q && pages && page_indptr && length_info && output && lse && key_weights) << what << ": NULL tensor";
  KV_CHECK(nnz_pages == 0 || (page_values && weight_page_values)) << what << ": NULL page table";
  check_aligned16(what, {q, pages, output});
}
// A launcher that this one runs; its message is the call's.
static void run(int rc) {
  if (rc != TVMKV_OK) throw Error(rc, tvmkv_last_error());
}

}  // namespace tvmkv

using namespace tvmkv;

extern "C" {

int tvmkv_batch_decode_paged_kv_weights(const void* q, const void* pages, const int32_t* page_indptr, const int32_t* page_values,
                                        const int32_t* length_info, void* output, float* lse, float* key_weights,
                                        const int32_t* weight_page_values, double sm_scale, int32_t batch_size, int64_t nnz_pages,
                                        int64_t num_pages, int32_t h_q, int32_t h_kv, int32_t d, int32_t page_size, void* stream) {
  KV_API_BEGIN();
  const char* const what = "batch_decode_paged_kv_weights";
  check_attention(what, q, pages, page_indptr, page_values, length_info, output, lse, key_weights, weight_page_values, batch_size, nnz_pages,
                  h_q, h_kv, d, page_size);
  if (batch_size == 0) return TVMKV_OK;
  const size_t kept = static_cast<size_t>(nnz_pages) * page_size * h_q * sizeof(float);
  if (nnz_pages > 0 && h_q <= 16 * h_kv && kept <= kMostKept) {
    const hipStream_t s = as_stream(stream);
    const ScratchLease ws = lease_scratch(kScratchKept, s, kept, 0);
    KeptScoresParams p;
    p.scores = reinterpret_cast<const float*>(ws.ptr);
    p.page_indptr = page_indptr;
    p.weight_page_values = weight_page_values;
    p.last_page_len = length_info;
    p.lse = lse;
    p.key_weights = key_weights;
    p.batch = batch_size;
    p.nnz_pages = static_cast<int>(nnz_pages);
    p.h_kv = h_kv;
    p.group = h_q / h_kv;
    p.page_shift = shift_of_page(what, page_size);
    const int64_t items = (((nnz_pages << p.page_shift) >> kKeptTokensShift) + batch_size) * h_kv;
    KV_CHECK(items < (int64_t{1} << 31)) << what << ": too many work items";
    // A launch of a few short sequences adds the weights itself (one of 500 tokens 12.9 -> 10.3 us); a sequence's are added by one
    // workgroup, and longer ones take it longer than a second launch (41 of up to 2500 tokens 23.5 -> 26.4).  Lengths are on the device: the
    // rule goes by their average, and one long sequence among short ones is added by a workgroup a kv head, too (itself / a second launch: 2500 among
    // 15 of 20 tokens 18.4 / 17.3, 8000 35 / 28, 15 000 47 / 30).
    const int64_t tokens = nnz_pages * page_size;
    const bool itself = tokens <= 16384 && tokens <= int64_t{1024} * batch_size;
    bool added = false;
    run(decode_keeping_scores(q, pages, page_indptr, page_values, length_info, output, lse, reinterpret_cast<float*>(ws.ptr),
                              itself ? key_weights : nullptr, weight_page_values, &added, sm_scale, batch_size, nnz_pages, num_pages, h_q, h_kv, d,
                              page_size, stream));
    if (added) return TVMKV_OK;
    hipLaunchKernelGGL(kept_scores_kernel, dim3(static_cast<unsigned>(items)), dim3(256), 0, s, p);
    KV_LAUNCH_CHECK();
    return TVMKV_OK;
  }
  run(tvmkv_batch_decode_paged_kv(q, pages, page_indptr, page_values, length_info, nullptr, nullptr, output, lse, 0, 1.0, 1e4, sm_scale,
                                  batch_size, nnz_pages, num_pages, h_q, h_kv, d, page_size, 0, stream));
  add_key_weights(what, weights_of_call(q, nullptr, pages, page_indptr, page_values, length_info, lse, key_weights, weight_page_values, false, 0,
                                        sm_scale, batch_size, h_q, h_kv, shift_of_page(what, page_size)),
                  batch_size, nnz_pages, d, as_stream(stream));
  KV_API_END();
}

int tvmkv_batch_prefill_paged_kv_weights(const void* q, const int32_t* q_indptr, const void* pages, const int32_t* page_indptr,
                                         const int32_t* page_values, const int32_t* length_info, void* output, float* lse,
                                         float* key_weights, const int32_t* weight_page_values, int64_t causal, int64_t observed,
                                         double sm_scale, int32_t batch_size, int64_t total_q, int64_t nnz_pages, int64_t num_pages,
                                         int32_t h_q, int32_t h_kv, int32_t d, int32_t page_size, void* stream) {
  KV_API_BEGIN();
  const char* const what = "batch_prefill_paged_kv_weights";
  KV_CHECK(total_q >= 0 && total_q <= INT32_MAX / std::max(h_q, 1)) << what << ": bad shape";
  KV_CHECK(observed >= 0) << what << ": observed is " << observed << ", expected a number of queries, or 0 for all";
  if (batch_size == 0 || total_q == 0) batch_size = std::min(batch_size, 0);
  check_attention(what, q, pages, page_indptr, page_values, length_info, output, lse, key_weights, weight_page_values, batch_size, nnz_pages,
                  h_q, h_kv, d, page_size);
  if (batch_size == 0) return TVMKV_OK;
  KV_CHECK(q_indptr) << what << ": NULL tensor";
  const hipStream_t s = as_stream(stream);
  const KeyWeightsParams p = weights_of_call(q, q_indptr, pages, page_indptr, page_values, length_info, lse, key_weights, weight_page_values,
                                             causal != 0, observed, sm_scale, batch_size, h_q, h_kv, shift_of_page(what, page_size));
  // Where a launch is split: up to 16 rows of a kv head on average, or 64 on 16384 (token, kv head)s at most, merge and weights are one launch;
  // with more of them its workgroups, which all go over the lse of all shares of their rows, take longer than a launch.  Apart / in one, us:
  //   32 / 8 heads of dim 128    1 x 700 tokens   8 rows 17.1 / 14.1, 32 rows 16.6 / 13.7, 64 rows 17.0 / 15.8, 128 rows 20.1 / 19.8
  //                              1 x 2000         16 rows 17.7 / 13.9, 64 rows 19.8 / 18.4, 128 rows 24.5 / 26.1
  //                              1 x 8000         16 rows 26.0 / 22.1, 32 rows 25.8 / 25.6, 64 rows 28 / 34
  //                              8 x 2000         8 rows 29.3 / 28.5, 16 rows 30.0 / 29.9, 32 rows 30.8 / 32.9, 64 rows 36 / 42
  //   16 / 2 heads of dim 256    1 x 8000         16 rows 33.5 / 28.6, 64 rows 36.6 / 36.6, 128 rows 44 / 51
  //   32 / 1 heads of dim 64     4 x 4000         32 rows 18.6 / 14.1, 64 rows 19.8 / 17.4, 128 rows 23 / 26
  // Rows are counted on average, as they are on the device: of 16 sequences of 2000 tokens one with 64 queries and none in the others 31 / 32.5,
  // of 8000 and 15 of 200 63 / 71, of 64 of 2000 one with 256 81 / 75.
  bool added = false;
  const bool in_one = total_q * p.group <= int64_t{(nnz_pages << p.page_shift) * h_kv <= 16384 ? 64 : 16} * batch_size;
  const std::function<void(const PrefillShares&)> merge_and_weigh = [&](const PrefillShares& shares) {
    const auto launch = [&](auto dim) {
      constexpr int D = decltype(dim)::value, rows_of_block = 256 / (D / 8);
      const int64_t merging = (shares.rows + rows_of_block - 1) / rows_of_block;
      const int64_t items = merging + (((nnz_pages << p.page_shift) >> 7) + batch_size) * h_kv;
      KV_CHECK(items < (int64_t{1} << 31)) << what << ": too many work items";
      hipLaunchKernelGGL(merge_and_weigh_kernel<D>, dim3(static_cast<unsigned>(items)), dim3(256), 0, s, p, shares, static_cast<half_t*>(output), lse,
                         static_cast<int>(merging));
    };
    if (d == 64) launch(std::integral_constant<int, 64>{});
    if (d == 80) launch(std::integral_constant<int, 80>{});
    if (d == 96) launch(std::integral_constant<int, 96>{});
    if (d == 112) launch(std::integral_constant<int, 112>{});
    if (d == 128) launch(std::integral_constant<int, 128>{});
    if (d == 256) launch(std::integral_constant<int, 256>{});
    added = true;
  };
  run(prefill_paged_in_float(q, q_indptr, pages, page_indptr, page_values, length_info, output, lse, causal, sm_scale, batch_size, total_q,
                             nnz_pages, num_pages, h_q, h_kv, d, page_size, in_one ? &merge_and_weigh : nullptr, stream));
  if (!added) add_key_weights(what, p, total_q, nnz_pages, d, s);
  KV_API_END();
}

int tvmkv_select_kept_tokens(const float* key_weights, const int32_t* page_indptr, const int32_t* weight_page_values,
                             const int32_t* length_info, const int32_t* keep, int32_t* kept, int64_t num_sinks, int64_t num_recent,
                             int32_t batch_size, int64_t nnz_pages, int32_t h_kv, int32_t page_size, int32_t max_keep, void* stream) {
  KV_API_BEGIN();
  const char* const what = "select_kept_tokens";
  SelectParams p{};
  p.page_shift = shift_of_page(what, page_size);
  check_table(what, batch_size, nnz_pages, h_kv, page_size);
  KV_CHECK(num_sinks >= 0 && num_recent >= 0 && max_keep >= 0 && max_keep <= 1 << 30) << what << ": bad shape";
  KV_CHECK(batch_size < 65536) << what << ": too many sequences";  // a dimension of the grid
  if (batch_size == 0 || max_keep == 0) return TVMKV_OK;
  KV_CHECK(key_weights && page_indptr && length_info && keep && kept) << what << ": NULL tensor";
  KV_CHECK(nnz_pages == 0 || weight_page_values) << what << ": NULL page table";
  const hipStream_t s = as_stream(stream);
  p.key_weights = key_weights;
  p.page_indptr = page_indptr;
  p.weight_page_values = weight_page_values;
  p.last_page_len = length_info;
  p.keep = keep;
  p.kept = kept;
  p.h_kv = h_kv;
  p.max_keep = max_keep;
  p.sinks = static_cast<int>(std::min<int64_t>(num_sinks, INT32_MAX));
  p.recent = static_cast<int>(std::min<int64_t>(num_recent, INT32_MAX));
  p.batch = batch_size;
  // Scratch memory: what the launches leave for each other.  Of one workgroup a list it is the bits of lists that are longer than its shared
  // memory has room for: none where all tokens together are few enough.
  const int64_t tokens = nnz_pages << p.page_shift, lists = static_cast<int64_t>(batch_size) * h_kv;
  // Workgroups of 256 threads where several lists share a compute unit or are short, else of 1024.  256 / 1024 threads, us (lists of tokens):
  //   8 of 700 7.7 / 8.8, 128 of 2112 9.5 / 9.1, 128 of 4096 14.6 / 11.0, 512 of 4096 16.5 / 20.2, 512 of 6000 27 / 23, 1024 of 1100 10.9 / 30
  const bool small = tokens <= static_cast<int64_t>(batch_size) * (lists > compute_units() ? 4096 : 2048);
  // Long lists that are too few to fill the chip, a workgroup each / in chunks, us:
  //   8 of 24 000 tokens 23.4 / 30.1, 512 of 24 000 76 / 94, 4 of 40 000 31.7 / 30.9, 2 of 131 072 92 / 33
  const bool chunked = tokens > static_cast<int64_t>(batch_size) * 32768 && lists <= 4 * compute_units() && tokens <= kMostChunkedBlocks * 256;
  const int64_t blocks_in_lds = small ? 256 : 1024;
  ScratchLease ws{};
  if (chunked || tokens > blocks_in_lds * 256) {
    const size_t blocks = static_cast<size_t>((tokens >> 8) + batch_size) * h_kv, states = chunked ? static_cast<size_t>(lists) : 0;
    ws = lease_scratch(kScratchSelect, s,
                       blocks * (4 * sizeof(uint64_t) + sizeof(int32_t)) + states * (sizeof(SelectState) + kSelectPasses * (kBins + 1) * sizeof(uint32_t)), 0);
    p.words = reinterpret_cast<uint64_t*>(ws.ptr);
    p.states = reinterpret_cast<SelectState*>(p.words + blocks * 4);
    p.histograms = reinterpret_cast<uint32_t*>(p.states + states);
    p.arrivals = p.histograms + states * kSelectPasses * kBins;
    p.counts = reinterpret_cast<int32_t*>(p.arrivals + states * kSelectPasses);
  }
  if (chunked) {
    const int64_t to_clear = lists * kSelectPasses * (kBins + 1), items = ((tokens >> kChunkShift) + batch_size) * h_kv;
    const dim3 grid(static_cast<unsigned>(items));
    hipLaunchKernelGGL(select_clear_kernel, dim3(static_cast<unsigned>(std::min<int64_t>((to_clear + 255) / 256, 1024))), dim3(256), 0, s, p.histograms,
                       to_clear);
    for (int nth = 0; nth < kSelectPasses; ++nth) hipLaunchKernelGGL(select_pass_kernel, grid, dim3(256), 0, s, p, nth);
    hipLaunchKernelGGL(select_bits_kernel, grid, dim3(256), 0, s, p);
    hipLaunchKernelGGL(select_places_kernel, dim3((max_keep + 1023) / 1024, h_kv, batch_size), dim3(256), 0, s, p);
  } else if (small) {
    hipLaunchKernelGGL((select_kept_kernel<256, 4, 256, 2048, 8>), dim3(h_kv, batch_size), dim3(256), 0, s, p);
  } else {
    hipLaunchKernelGGL((select_kept_kernel<1024, 4, 1024, 16384, 32>), dim3(h_kv, batch_size), dim3(1024), 0, s, p);
  }
  KV_LAUNCH_CHECK();
  KV_API_END();
}

int tvmkv_move_kept_tokens(void* pages, float* key_weights, const int32_t* page_indptr, const int32_t* page_values,
                           const int32_t* weight_page_values, const int32_t* kept, int32_t batch_size, int64_t nnz_pages, int64_t num_pages,
                           int32_t h_kv, int32_t page_size, int32_t d, int32_t dtype_bits, int32_t max_keep, void* stream) {
  KV_API_BEGIN();
  const char* const what = "move_kept_tokens";
  MoveParams p;
  p.page_shift = shift_of_page(what, page_size);
  check_table(what, batch_size, nnz_pages, h_kv, page_size);
  KV_CHECK(max_keep >= 0 && max_keep <= 1 << 30) << what << ": bad shape";
  KV_UNSUPPORTED(dtype_bits != 16 && dtype_bits != 32) << what << ": rows of " << dtype_bits << " bits an element are not built (16, 32)";
  KV_UNSUPPORTED(d <= 0 || d > 256 || d * dtype_bits % 128 != 0) << what << ": head_dim " << d << " is not built";
  KV_CHECK(batch_size < 65536 && h_kv < 65536) << what << ": too many sequences or heads";  // dimensions of the grid
  KV_CHECK(num_pages >= 0) << what << ": bad shape";
  KV_UNSUPPORTED(num_pages >= (int64_t{1} << 32) / (2 * page_size) / h_kv) << what << ": a pool of 2^32 rows or more is not built";
  if (batch_size == 0 || max_keep == 0 || nnz_pages == 0) return TVMKV_OK;
  KV_CHECK(pages && page_indptr && kept) << what << ": NULL tensor";
  KV_CHECK(page_values && (key_weights == nullptr || weight_page_values)) << what << ": NULL page table";
  KV_CHECK(reinterpret_cast<uintptr_t>(pages) % 16 == 0) << what << ": pages must be aligned to 16 bytes";
  p.pages = static_cast<uint8_t*>(pages);
  p.key_weights = key_weights;
  p.page_indptr = page_indptr;
  p.page_values = page_values;
  p.weight_page_values = weight_page_values;
  p.kept = kept;
  p.h_kv = h_kv;
  p.max_keep = max_keep;
  p.pieces = 2 * (d * dtype_bits / 128);
  const int64_t lists = static_cast<int64_t>(batch_size) * h_kv;
  // In one launch and in order, in parts of 128 bytes at least, where that makes two workgroups a compute unit, or lists are short; else by
  // ranges of places.  In order / by ranges, us (lists, tokens, places; 8 kv heads of dim 128 but for the last):
  //   8 x 700 to 512 7.9 / 15.3, 16 x 2112 to 2048 9.0 / 18.4, 128 x 2112 to 2048 14.9 / 30, 512 x 4096 to 2048 120 / 126, 128 x 12 000 to 4000
  //   81 / 88; 32 x 24 000 to 4000 43 / 38, 8 x 12 000 to 4000 28.7 / 20.0, 4 x 40 000 to 8000 61 / 20.5
  // Few lists around the 2048 places, captured: to 2048 from 16 000 one 14.5 / 15.9, 8 17.0 / 16.8, 32 22 / 26, from 65 536 one 15.3 / 16.0, 8 18.4 / 17.0,
  // 32 26 / 27; to 1536 from 16 000 8 13.3 / 16.5; to 2500 from 16 000 one 17.8 / 15.8, 8 21.7 / 18.3, 32 27 / 29, from 65 536 8 23 / 19, 32 32 / 31.
  // Lists that lose few tokens are better in order up to 4000 places (8 x 5000 to 4000 13.8 / 16.6), which max_keep alone does not say.
  const auto cut_rows = [&](int64_t most, int least_pieces) {
    p.slices = 1;
    while (p.slices * 2 <= most && p.pieces % (p.slices * 2) == 0 && p.pieces / (p.slices * 2) >= least_pieces) p.slices *= 2;
    p.by_row = ExactDivision::by(p.pieces);
    p.by_slice = ExactDivision::by(p.pieces / p.slices);
  };
  const int wanted = 4 * compute_units();
  cut_rows(std::max<int64_t>(wanted / lists, 1), 8);
  if (lists * p.slices * 2 >= wanted || max_keep <= 2048) {
    hipLaunchKernelGGL(move_kept_kernel<kMoveInOrder>, dim3(p.slices, h_kv, batch_size), dim3(kMoveThreads), 0, as_stream(stream), p);
  } else {
    const int parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((max_keep + 63) / 64, wanted / lists)));
    cut_rows(parts, 4);
    hipLaunchKernelGGL(move_kept_kernel<kMoveFirst>, dim3(parts, h_kv, batch_size), dim3(kMoveThreads), 0, as_stream(stream), p);
    hipLaunchKernelGGL(move_kept_kernel<kMoveSecond>, dim3(parts, h_kv, batch_size), dim3(kMoveThreads), 0, as_stream(stream), p);
  }
  KV_LAUNCH_CHECK();
  KV_API_END();
}

}  // extern "C"
