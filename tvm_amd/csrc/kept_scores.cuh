// Sums of attention weights from the scores that a decode launch kept (kernels_decode.hip writes them; it reads them in the same launch
// where they are few, kernels_evict.hip in one of its own).
#ifndef TVMKV_CSRC_KEPT_SCORES_CUH_
#define TVMKV_CSRC_KEPT_SCORES_CUH_

#include "kernels_common.cuh"
#include "typed_kernels.h"

namespace tvmkv {

typedef float float2_any_t __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t kept_uint4_t __attribute__((ext_vector_type(4)));

// Scores that other workgroups of the launch may have written: device-scope accesses (the sc1 bit), as each XCD has its own L2.
constexpr int kKeptDeviceScope = 16;
__device__ __forceinline__ void store_kept(float* scores, uint32_t at, float4_t x) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(kept_uint4_t, x), __builtin_amdgcn_make_buffer_rsrc(scores, 0, -1, 0x00027000), at * 4, 0,
                                         kKeptDeviceScope);
}
__device__ __forceinline__ float4_t load_kept(float* scores, uint32_t at) {
  return __builtin_bit_cast(float4_t, __builtin_amdgcn_raw_buffer_load_b128(__builtin_amdgcn_make_buffer_rsrc(scores, 0, -1, 0x00027000), at * 4, 0,
                                                                            kKeptDeviceScope));
}

// The weights of a lane's four tokens of a run, places 4 part .. of it, over the heads of a group: score_of(head), lse_of(head).
template <class Score, class Lse>
__device__ __forceinline__ float4_t kept_weights(int group, Score score_of, Lse lse_of) {
  float4_t sum = {0.f, 0.f, 0.f, 0.f};
  for (int g = 0; g < group; g += 4) {
    float4_t x[4];
    float of[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = score_of(min(g + i, group - 1));
      of[i] = lse_of(min(g + i, group - 1));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (g + i < group) {
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] += fast_exp2(x[i][k] - of[i]);
      }
    }
  }
  return sum;
}
// Adds them to the run's sums, of which `tokens` belong to tokens: what is there already rounds them once.  A lane's tokens are two
// pairs of neighbours.
__device__ __forceinline__ void add_to_sums(float* run, int part, float4_t x, int tokens) {
  static_assert(kept_score_token(1) == kept_score_token(0) + 1 && kept_score_token(2) == kept_score_token(0) + 8 && kept_score_token(4) == 2, "pairs");
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int token = 2 * part + 8 * k;
    float2_any_t* const at = reinterpret_cast<float2_any_t*>(run + token);
    if (token + 2 <= tokens) *at = *at + float2_any_t{x[2 * k], x[2 * k + 1]};
    if (token + 1 == tokens) run[token] += x[2 * k];
  }
}

}  // namespace tvmkv

#endif  // TVMKV_CSRC_KEPT_SCORES_CUH_
