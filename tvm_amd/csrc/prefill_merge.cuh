// The merge of a split prefill launch's shares (kernels_prefill.hip says what they are), and the log-sum-exp that it gives a row.
#ifndef TVMKV_CSRC_PREFILL_MERGE_CUH_
#define TVMKV_CSRC_PREFILL_MERGE_CUH_

#include "kernels_common.cuh"

namespace tvmkv {

// Shares in loops of as many as there are, unrolled by eight, or eight at once, the last one again in place of those that are not there:
// all that is needed is in flight together, and what is not needed costs loads and registers (merge_shares_at_once says when which).
constexpr int kSharesAtOnce = 8;
__device__ __forceinline__ void load_shares_lse(float (&l)[kSharesAtOnce], const float* part_lse, int64_t rows, int splits, int64_t row, int i0) {
#pragma unroll
  for (int u = 0; u < kSharesAtOnce; ++u) l[u] = part_lse[min(i0 + u, splits - 1) * rows + row];
}
__device__ __forceinline__ float largest_shares_lse(const float (&l)[kSharesAtOnce], const float* part_lse, int64_t rows, int splits, int64_t row) {
  float s_max = kNegInit;
#pragma unroll
  for (int u = 0; u < kSharesAtOnce; ++u) s_max = fmaxf(s_max, l[u]);
  for (int i0 = kSharesAtOnce; i0 < splits; i0 += kSharesAtOnce) {
    float more[kSharesAtOnce];
    load_shares_lse(more, part_lse, rows, splits, row, i0);
#pragma unroll
    for (int u = 0; u < kSharesAtOnce; ++u) s_max = fmaxf(s_max, more[u]);
  }
  return s_max;
}

// Rows of the block-th 256 threads, 256 / (DV / 8) of them.
template <typename T, int DV, bool AT_ONCE>
__device__ __forceinline__ void merge_prefill_shares(const T* __restrict__ part_o, const float* __restrict__ part_lse,
                                                     half_t* __restrict__ output, float* __restrict__ lse, int64_t rows, int splits,
                                                     int merge_into, const int32_t* __restrict__ q_indptr, int batch, int h_q, int block) {
  typedef T share_t __attribute__((ext_vector_type(8)));
  constexpr int TPR = DV / 8;  // threads per row, 8 features each
  const int64_t row = static_cast<int64_t>(block) * (256 / TPR) + threadIdx.x / TPR;
  const int piece = threadIdx.x % TPR;
  if (threadIdx.x >= 256 / TPR * TPR || row >= rows) return;
  const int64_t begin = static_cast<int64_t>(q_indptr[0]) * h_q, end = static_cast<int64_t>(q_indptr[batch]) * h_q;
  const auto load = [&](share_t(&v)[kSharesAtOnce], int i0) {
#pragma unroll
    for (int u = 0; u < kSharesAtOnce; ++u) v[u] = *reinterpret_cast<const share_t*>(part_o + (min(i0 + u, splits - 1) * rows + row) * DV + piece * 8);
  };
  float l[kSharesAtOnce];
  share_t v[kSharesAtOnce];
  float s_max = kNegInit;
  if constexpr (AT_ONCE) {
    load_shares_lse(l, part_lse, rows, splits, row, 0);
    load(v, 0);
  } else {
#pragma unroll 8
    for (int i = 0; i < splits; ++i) s_max = fmaxf(s_max, part_lse[i * rows + row]);
  }
  // (rows in front of the first sequence and behind the last one have no shares and stay as they are)
  if (row < begin || row >= end) return;
  if constexpr (AT_ONCE) s_max = largest_shares_lse(l, part_lse, rows, splits, row);
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  float w_sum = 0.f;
  const bool any_share = s_max > kNegInit;
  if (merge_into) {
    // output / lse already hold a state of the same rows (the launch was asked to merge into it): it is one more
    // state of the sum; shares that are all empty count as the one empty state (out 0, lse -5e4) an unsplit
    // launch would have merged
    const float s_prev = lse[row];
    s_max = fmaxf(s_max, s_prev);
    const float w = fast_exp2(s_prev - s_max);
    const Vec16 x = ld16(output + row * DV + piece * 8);
    w_sum = w + (any_share ? 0.f : fast_exp2(kNegInit - s_max));
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = w * static_cast<float>(x.h8[e]);
  }
  if (any_share && !AT_ONCE) {
#pragma unroll 8
    for (int i = 0; i < splits; ++i) {
      const float w = fast_exp2(part_lse[i * rows + row] - s_max);
      const share_t x = *reinterpret_cast<const share_t*>(part_o + (i * rows + row) * DV + piece * 8);
      w_sum += w;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += w * static_cast<float>(x[e]);
    }
  } else if (any_share) {
    for (int i0 = 0;;) {
#pragma unroll
      for (int u = 0; u < kSharesAtOnce; ++u) {
        if (i0 + u < splits) {
          const float w = fast_exp2(l[u] - s_max);
          w_sum += w;
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] += w * static_cast<float>(v[u][e]);
        }
      }
      i0 += kSharesAtOnce;
      if (i0 >= splits) break;
      load_shares_lse(l, part_lse, rows, splits, row, i0);
      load(v, i0);
    }
  }
  const float inv = w_sum > 0.f ? 1.0f / w_sum : 0.f;
  Vec16 out;
#pragma unroll
  for (int e = 0; e < 8; ++e) out.h8[e] = static_cast<half_t>(acc[e] * inv);
  *reinterpret_cast<Vec16*>(output + row * DV + piece * 8) = out;
  if (piece == 0) lse[row] = w_sum > 0.f ? s_max + fast_log2(w_sum) : kNegInit;
}

// The log-sum-exp that the merge gives a row, by itself.
__device__ __forceinline__ float merged_lse(const float* __restrict__ part_lse, int64_t rows, int splits, int64_t row) {
  float l[kSharesAtOnce];
  load_shares_lse(l, part_lse, rows, splits, row, 0);
  const float s_max = largest_shares_lse(l, part_lse, rows, splits, row);
  if (!(s_max > kNegInit)) return kNegInit;
  float w_sum = 0.f;
  for (int i0 = 0;;) {
#pragma unroll
    for (int u = 0; u < kSharesAtOnce; ++u) w_sum += i0 + u < splits ? fast_exp2(l[u] - s_max) : 0.f;
    i0 += kSharesAtOnce;
    if (i0 >= splits) break;
    load_shares_lse(l, part_lse, rows, splits, row, i0);
  }
  return s_max + fast_log2(w_sum);
}

}  // namespace tvmkv

#endif  // TVMKV_CSRC_PREFILL_MERGE_CUH_
