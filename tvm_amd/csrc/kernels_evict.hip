// Eviction from the paged cache by the attention that tokens received: the sums of attention weights that go with an attention
// call, the choice of the tokens that stay and their move to the front of the sequence's pages.
//
// With s the scaled scores (base 2) of a query head and lse their log-sum-exp, a key's weight is 2^(s - lse).  The weights pool
// (weight pages, h_kv, page_size), float32, holds a sum for each stored token and kv head, over the query heads of the group
// and the queries that count.  Every entry is added to by one lane of one workgroup: the sums do not depend on the order in
// which workgroups run.
#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "kernels_common.cuh"
#include "runtime_support.h"
#include "typed_kernels.h"
#include "exact_division.h"

namespace tvmkv {

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
  int batch;
  int h_q;
  int h_kv;
  int group;
  ExactDivision by_group;
  int causal;
  int observed;    // > 0: queries at a sequence's end that count
  int page_shift;  // pages hold 1 << page_shift tokens
  float scale_log2;
};

template <int D, int TB>
__global__ __launch_bounds__(256) void key_weights_kernel(KeyWeightsParams p) {
  constexpr int KS = D / 16;
  constexpr int T = 128 * TB;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int col = lane & 31;
  const int half = lane >> 5;
  const int kvh = blockIdx.x % p.h_kv, slot = blockIdx.x / p.h_kv;
  const SequenceOf s = sequence_of_slot(p.page_indptr, p.last_page_len, p.batch, p.page_shift, TB == 1 ? 7 : 8, slot, lane);
  static_assert(TB == 1 || TB == 2, "the shift above");
  const int stored = s.stored(p.page_shift);
  const int t0 = (slot - s.slot_begin) * T + wave * 32 * TB;  // the wave's first token
  if (t0 >= stored) return;
  const int q_begin = p.q_indptr != nullptr ? p.q_indptr[s.index] : s.index;
  const int q_len = p.q_indptr != nullptr ? p.q_indptr[s.index + 1] - q_begin : 1;
  const int first_counted = p.observed > 0 ? max(q_len - p.observed, 0) : 0;
  const int in_front = stored - q_len;  // query i sees the keys up to in_front + i
  const int row_end = q_len * p.group;
  const int row_begin = first_counted * p.group;
  const int first_row = max(first_counted, p.causal ? t0 - in_front : 0) * p.group;  // no row in front of it sees the wave's tokens

  half8_t k[TB][KS];
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    const int t = min(t0 + b * 32 + col, stored - 1);
    const int page = p.page_values[s.page_begin + (t >> p.page_shift)];
    const half_t* row = p.pages + ((((static_cast<int64_t>(page) * 2 * p.h_kv + kvh) << p.page_shift) + (t & ((1 << p.page_shift) - 1))) * D) + half * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) k[b][ks] = ld16(row + ks * 16).h8;
  }
  float sum[TB][16];
#pragma unroll
  for (int b = 0; b < TB; ++b) {
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[b][i] = 0.f;
  }
  for (int r0 = first_row & ~31; r0 < row_end; r0 += 32) {
    const int row = min(r0 + col, row_end - 1);
    const int token = p.by_group(row);
    const int64_t at = static_cast<int64_t>(q_begin + token) * p.h_q + kvh * p.group + row - token * p.group;
    const bool counts = r0 + col < row_end && row >= row_begin;
    const int end = p.causal ? min(in_front + token + 1, stored) : stored;
    const float lse = p.lse[at];
    half8_t q[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[ks] = ld16(p.q + at * D + half * 8 + ks * 16).h8;
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      float16_t x = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[b][ks], q[ks], x, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int t = t0 + b * 32 + (i & 3) + 8 * (i >> 2) + 4 * half;
        const float w = fast_exp2(fmaf(x[i], p.scale_log2, -lse));
        sum[b][i] += counts && t < end ? w : 0.f;
      }
    }
  }
  // lane i of 32 takes the sum of its half's i-th token of a block
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    float mine = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float total = sum_xor16(group_sum<16>(sum[b][i]));
      mine = col == i ? total : mine;
    }
    const int t = t0 + b * 32 + (col & 3) + 8 * (col >> 2) + 4 * half;
    if (col < 16 && t < stored) {
      const int page = p.weight_page_values[s.page_begin + (t >> p.page_shift)];
      p.key_weights[((static_cast<int64_t>(page) * p.h_kv + kvh) << p.page_shift) + (t & ((1 << p.page_shift) - 1))] += mine;
    }
  }
}

// ------------------------------------------------------------------------------------------
// The choice.  A workgroup has the tokens of one (sequence, kv head); weights are compared as integers that order like them
// (NaN below everything, -0 as 0).  Four passes of 8 bits find the smallest weight that stays, T, and how many of the weights
// equal to it do: counts, exact whatever their order.  Then a bit a token says which ones stay, in shared memory or, for longer
// sequences, in scratch memory, and running counts of free places and of tokens without one pair them.
// ------------------------------------------------------------------------------------------
struct SelectParams {
  const float* key_weights;
  const int32_t* page_indptr;
  const int32_t* weight_page_values;
  const int32_t* last_page_len;
  const int32_t* keep;
  int32_t* kept;
  uint64_t* words;  // scratch memory: 64 tokens each, and as many counts; NULL where no sequence can be longer than kLdsWords
  int32_t* counts;
  int h_kv;
  int max_keep;
  int sinks;
  int recent;
  int page_shift;
};
constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / 64;
constexpr int kLdsWords = 4096;  // 262144 tokens

__device__ __forceinline__ uint32_t weight_order(float w) {
  if (w != w) return 0;
  const uint32_t bits = __float_as_uint(w + 0.f);  // -0 + 0 = 0
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
// The nth set bit of x, which has more than n.
__device__ __forceinline__ int nth_bit(uint64_t x, int n) {
  int at = 0;
#pragma unroll
  for (int width = 32; width > 0; width >>= 1) {
    const int below = __popcll(x >> at & ((uint64_t{1} << width) - 1));
    const bool up = n >= below;
    n -= up ? below : 0;
    at += up ? width : 0;
  }
  return at;
}
// Sum of what the waves in front of this one bring, and of all.
__device__ __forceinline__ int sum_before_wave(int* shared, int value, int wave, int lane, int* total) {
  __syncthreads();
  if (lane == 0) shared[wave] = value;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kSelectWaves; ++i) {
    before += i < wave ? shared[i] : 0;
    all += shared[i];
  }
  *total = all;
  return before;
}

__global__ __launch_bounds__(kSelectThreads) void select_kept_kernel(SelectParams p) {
  __shared__ uint64_t lds_words[kLdsWords];
  __shared__ int32_t lds_counts[kLdsWords];
  __shared__ uint32_t histogram[256];
  __shared__ int per_wave[kSelectWaves];
  __shared__ uint32_t chosen_digit, left_over, as_many;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x, b = blockIdx.y;
  const int page_begin = p.page_indptr[b], num_pages = p.page_indptr[b + 1] - page_begin;
  const int stored = num_pages > 0 ? ((num_pages - 1) << p.page_shift) + p.last_page_len[b] : 0;
  const int n = min(stored, max(min(p.keep[b], p.max_keep), 0));
  int32_t* const kept = p.kept + (static_cast<int64_t>(b) * p.h_kv + kvh) * p.max_keep;
  const int recent = min(p.recent, n), sinks = min(p.sinks, n - recent), places = n - recent;
  const int gone = stored - n;
  for (int i = places + tid; i < p.max_keep; i += kSelectThreads) kept[i] = i < n ? i + gone : -1;
  if (gone == 0 || places == sinks) {
    for (int i = tid; i < places; i += kSelectThreads) kept[i] = i;
    return;
  }
  const auto order_of = [&](int t) {
    const int page = p.weight_page_values[page_begin + (t >> p.page_shift)];
    return weight_order(p.key_weights[((static_cast<int64_t>(page) * p.h_kv + kvh) << p.page_shift) + (t & ((1 << p.page_shift) - 1))]);
  };
  const int end = stored - recent;  // candidates: tokens [sinks, end), of which `need` stay and at least one does not
  uint32_t least = 0, need = places - sinks;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelectThreads) histogram[i] = 0;
    __syncthreads();
    for (int t = sinks + tid; t < end; t += kSelectThreads) {
      const uint32_t x = order_of(t);
      if (shift == 24 || x >> (shift + 8) == least) atomicAdd(&histogram[x >> shift & 255], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t above = 0;
      int digit = 255;
      while (digit > 0 && above + histogram[digit] < need) above += histogram[digit--];
      chosen_digit = digit;
      left_over = need - above;
      as_many = histogram[digit];
    }
    __syncthreads();
    least = least << 8 | chosen_digit;
    need = left_over;
  }
  // Bits of the tokens in front of the recent ones, a range of words a wave.  Of the as_many weights equal to T the first
  // `need` stay.
  const int num_words = (end + 63) >> 6;
  uint64_t* const words = num_words <= kLdsWords ? lds_words : p.words + (((static_cast<int64_t>(page_begin - p.page_indptr[0]) << p.page_shift) >> 6) + b) * p.h_kv + static_cast<int64_t>(kvh) * num_words;
  int32_t* const counts = num_words <= kLdsWords ? lds_counts : p.counts + (words - p.words);
  const int per = (num_words + kSelectWaves - 1) / kSelectWaves, word_lo = min(wave * per, num_words), word_hi = min(word_lo + per, num_words);
  int equal_before = 0, total;
  if (need < as_many) {
    int equal = 0;
    for (int w = word_lo; w < word_hi; ++w) {
      const int t = w * 64 + lane;
      equal += __popcll(__ballot(t >= sinks && t < end && order_of(t) == least));
    }
    equal_before = sum_before_wave(per_wave, equal, wave, lane, &total);
  }
  const int boundary = places >> 6;  // the word with the first token behind the places; holes up to it, tokens without a place from it on
  const uint64_t in_places = (uint64_t{1} << (places & 63)) - 1;  // of its bits
  int holes = 0, homeless = 0;
  for (int w = word_lo; w < word_hi; ++w) {
    const int t = w * 64 + lane;
    bool stays = t < sinks;
    if (t >= sinks && t < end) {
      const uint32_t x = order_of(t);
      const uint64_t equal = __ballot(x == least);
      stays = x > least || (x == least && equal_before + static_cast<int>(__popcll(equal & ((uint64_t{1} << lane) - 1))) < static_cast<int>(need));
      equal_before += __popcll(equal);
    }
    const uint64_t word = __ballot(stays);
    if (lane == 0) words[w] = word;
    holes += __popcll(~word & (w < boundary ? ~uint64_t{0} : w == boundary ? in_places : 0));
    homeless += __popcll(word & (w > boundary ? ~uint64_t{0} : w == boundary ? ~in_places : 0));
  }
  int holes_before = sum_before_wave(per_wave, holes, wave, lane, &total);
  int homeless_before = sum_before_wave(per_wave, homeless, wave, lane, &total);
  // counts of a word: up to the boundary the holes in front of it, behind it the tokens without a place in front of it
  for (int w = word_lo; w < word_hi; ++w) {
    const uint64_t word = words[w];
    if (lane == 0) counts[w] = w <= boundary ? holes_before : homeless_before;
    holes_before += __popcll(~word & (w < boundary ? ~uint64_t{0} : 0));
    homeless_before += __popcll(word & (w > boundary ? ~uint64_t{0} : w == boundary ? ~in_places : 0));
  }
  __syncthreads();
  const uint64_t first_homeless = boundary < num_words ? words[boundary] & ~in_places : 0;
  for (int i = tid; i < places; i += kSelectThreads) {
    const uint64_t word = words[i >> 6];
    int from = i;
    if (!(word >> (i & 63) & 1)) {
      const int rank = counts[i >> 6] + __popcll(~word & ((uint64_t{1} << (i & 63)) - 1));
      if (rank < static_cast<int>(__popcll(first_homeless))) {
        from = boundary * 64 + nth_bit(first_homeless, rank);
      } else {
        int lo = boundary + 1, hi = num_words - 1;  // the last word that begins at or in front of the rank
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (counts[mid] <= rank) lo = mid; else hi = mid - 1;
        }
        from = lo * 64 + nth_bit(words[lo], rank - counts[lo]);
      }
    }
    kept[i] = from;
  }
}

// ------------------------------------------------------------------------------------------
// The move: row kept[i] to place i, in place.  kept[i] is never in front of i, so that places filled in order never overwrite a row
// that a later one needs: a workgroup has the rows of one of K, V or the sums of a (sequence, kv head), reads those of a few
// places, waits until all have, and writes.  Entries that name no token behind their place are passed over.
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
  int pieces;  // of 16 bytes in a row
  ExactDivision by_pieces;
};
constexpr int kMoveThreads = 256;
__global__ __launch_bounds__(kMoveThreads) void move_kept_kernel(MoveParams p) {
  __shared__ int places[kMoveThreads], sources[kMoveThreads];
  __shared__ int per_wave[kMoveThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int part = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int page_begin = p.page_indptr[b], capacity = (p.page_indptr[b + 1] - page_begin) << p.page_shift;
  const int32_t* const kept = p.kept + (static_cast<int64_t>(b) * p.h_kv + kvh) * p.max_keep;
  const int in_page = (1 << p.page_shift) - 1;
  const auto sum_at = [&](int t) {
    const int page = p.weight_page_values[page_begin + (t >> p.page_shift)];
    return p.key_weights + ((static_cast<int64_t>(page) * p.h_kv + kvh) << p.page_shift) + (t & in_page);
  };
  const auto row_at = [&](int t) {
    const int page = p.page_values[page_begin + (t >> p.page_shift)];
    return p.pages + ((((static_cast<int64_t>(page) * 2 + part) * p.h_kv + kvh) << p.page_shift) + (t & in_page)) * (p.pieces * 16);
  };
  const int limit = min(p.max_keep, capacity);
  for (int i0 = 0; i0 < limit; i0 += kMoveThreads) {
    const int i = i0 + tid;
    const int from = i < limit ? kept[i] : -1;
    const bool moves = from > i && from < capacity;
    if (part == 2) {
      float x = 0.f;
      if (moves) x = *sum_at(from);
      __syncthreads();
      if (moves) *sum_at(i) = x;
      continue;
    }
    const uint64_t who = __ballot(moves);
    if (lane == 0) per_wave[wave] = __popcll(who);
    __syncthreads();
    int at = __popcll(who & ((uint64_t{1} << lane) - 1)), count = 0;
#pragma unroll
    for (int w = 0; w < kMoveThreads / 64; ++w) {
      at += w < wave ? per_wave[w] : 0;
      count += per_wave[w];
    }
    if (moves) {
      places[at] = i;
      sources[at] = from;
    }
    __syncthreads();
    constexpr int U = 4;
    const int total = count * p.pieces;  // at most 256 rows of 64 pieces
    for (int x0 = 0; x0 < total; x0 += kMoveThreads * U) {
      Vec16 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int x = x0 + u * kMoveThreads + tid, row = p.by_pieces(x);
        if (x < total) v[u] = ld16(row_at(sources[row]) + (x - row * p.pieces) * 16);
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int x = x0 + u * kMoveThreads + tid, row = p.by_pieces(x);
        if (x < total) st16(row_at(places[row]) + (x - row * p.pieces) * 16, v[u]);
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
  KV_CHECK(nnz_pages < (int64_t{1} << 31) / page_size) << what << ": too many pages";  // tokens are 31-bit numbers
}
static void check_aligned16(const char* what, std::initializer_list<const void*> tensors) {
  for (const void* t : tensors)
    KV_CHECK(reinterpret_cast<uintptr_t>(t) % 16 == 0) << what << ": q, pages and output must be aligned to 16 bytes";
}

static void add_key_weights(const char* what, const void* q, const int32_t* q_indptr, const void* pages, const int32_t* page_indptr,
                            const int32_t* page_values, const int32_t* length_info, const float* lse, float* key_weights,
                            const int32_t* weight_page_values, bool causal, int64_t observed, double sm_scale, int32_t batch_size,
                            int64_t nnz_pages, int32_t h_q, int32_t h_kv, int32_t d, int page_shift, hipStream_t stream) {
  if (batch_size == 0 || nnz_pages == 0) return;
  KeyWeightsParams p;
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
  p.causal = causal;
  p.observed = static_cast<int>(std::min<int64_t>(observed, INT32_MAX));
  p.page_shift = page_shift;
  p.scale_log2 = static_cast<float>(sm_scale) * kLog2e;
  const int64_t items = (((nnz_pages << page_shift) >> 7) + batch_size) * h_kv;
  KV_CHECK(items < (int64_t{1} << 31)) << what << ": too many work items";
  const auto launch = [&](auto dim) {
    hipLaunchKernelGGL((key_weights_kernel<decltype(dim)::value, 1>), dim3(static_cast<unsigned>(items)), dim3(256), 0, stream, p);
  };
  if (d == 64) launch(std::integral_constant<int, 64>{});
  if (d == 80) launch(std::integral_constant<int, 80>{});
  if (d == 96) launch(std::integral_constant<int, 96>{});
  if (d == 112) launch(std::integral_constant<int, 112>{});
  if (d == 128) launch(std::integral_constant<int, 128>{});
  if (d == 256) launch(std::integral_constant<int, 256>{});
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
  run(tvmkv_batch_decode_paged_kv(q, pages, page_indptr, page_values, length_info, nullptr, nullptr, output, lse, 0, 1.0, 1e4, sm_scale,
                                  batch_size, nnz_pages, num_pages, h_q, h_kv, d, page_size, 0, stream));
  add_key_weights(what, q, nullptr, pages, page_indptr, page_values, length_info, lse, key_weights, weight_page_values, false, 0, sm_scale,
                  batch_size, nnz_pages, h_q, h_kv, d, shift_of_page(what, page_size), as_stream(stream));
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
  run(tvmkv_batch_prefill_paged_kv(q, q_indptr, pages, page_indptr, page_values, length_info, nullptr, nullptr, output, lse, causal, 0, 1.0, 1e4,
                                   sm_scale, batch_size, total_q, nnz_pages, num_pages, h_q, h_kv, d, page_size, 0, 0, stream));
  add_key_weights(what, q, q_indptr, pages, page_indptr, page_values, length_info, lse, key_weights, weight_page_values, causal != 0, observed,
                  sm_scale, batch_size, nnz_pages, h_q, h_kv, d, shift_of_page(what, page_size), as_stream(stream));
  KV_API_END();
}

int tvmkv_select_kept_tokens(const float* key_weights, const int32_t* page_indptr, const int32_t* weight_page_values,
                             const int32_t* length_info, const int32_t* keep, int32_t* kept, int64_t num_sinks, int64_t num_recent,
                             int32_t batch_size, int64_t nnz_pages, int32_t h_kv, int32_t page_size, int32_t max_keep, void* stream) {
  KV_API_BEGIN();
  const char* const what = "select_kept_tokens";
  SelectParams p;
  p.page_shift = shift_of_page(what, page_size);
  check_table(what, batch_size, nnz_pages, h_kv, page_size);
  KV_CHECK(num_sinks >= 0 && num_recent >= 0 && max_keep >= 0) << what << ": bad shape";
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
  p.words = nullptr;
  p.counts = nullptr;
  const int64_t tokens = nnz_pages << p.page_shift;
  ScratchLease ws{};
  if (tokens > kLdsWords * 64) {
    const size_t words = static_cast<size_t>((tokens >> 6) + batch_size) * h_kv;
    ws = lease_scratch(kScratchEvict, s, words * (sizeof(uint64_t) + sizeof(int32_t)), 0);
    p.words = reinterpret_cast<uint64_t*>(ws.ptr);
    p.counts = reinterpret_cast<int32_t*>(p.words + words);
  }
  hipLaunchKernelGGL(select_kept_kernel, dim3(h_kv, batch_size), dim3(kSelectThreads), 0, s, p);
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
  KV_CHECK(max_keep >= 0) << what << ": bad shape";
  KV_UNSUPPORTED(dtype_bits != 16 && dtype_bits != 32) << what << ": rows of " << dtype_bits << " bits an element are not built (16, 32)";
  KV_UNSUPPORTED(d <= 0 || d > 256 || d * dtype_bits % 128 != 0) << what << ": head_dim " << d << " is not built";
  KV_CHECK(batch_size < 65536 && h_kv < 65536) << what << ": too many sequences or heads";  // dimensions of the grid
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
  p.pieces = d * dtype_bits / 128;
  p.by_pieces = ExactDivision::by(p.pieces);
  hipLaunchKernelGGL(move_kept_kernel, dim3(key_weights != nullptr ? 3 : 2, h_kv, batch_size), dim3(kMoveThreads), 0, as_stream(stream), p);
  KV_LAUNCH_CHECK();
  KV_API_END();
}

}  // extern "C"
