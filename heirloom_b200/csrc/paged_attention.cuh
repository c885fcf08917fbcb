// The kernels behind hl_paged_attention and what they are given.
#pragma once
#include "paged.cuh"

namespace hl {

struct PagedAttention {
  PagedView p;
  DealShape z;
  const void* q;
  void* out;
  float* lse;            // [tokens][heads], may be null
  Joint* joints;         // [streams]
  float* pieces;         // [streams][2] pieces
  long long ld_q, ld_out;
  int heads;
  float scale_log2;      // softmax scale times log2(e)
};

// bf16 heads of 64 or 128 channels, blocks of 128 rows (paged_attention_tc.cu): how it is dealt out, and the launch.
DealShape paged_attention_tc_shape(int sms, int group);
int paged_attention_tc(hl_ctx* ctx, const PagedAttention& a);

// The same types with at most STEP_ROWS rows a key head (paged_attention_step.cu); `whole`: items are not shared out, nothing is to be joined.
constexpr int STEP_ROWS = 16;
DealShape paged_attention_step_shape(int sms, int group);
int paged_attention_step(hl_ctx* ctx, const PagedAttention& a, bool whole);

// 2^(a - b) where a may be minus infinity and b is its row's maximum or above it
__device__ __forceinline__ float piece_factor(float a, float b) { return a == -INFINITY ? 0.0f : exp2f(a - b); }

}  // namespace hl
