// The next tokens of many rows of logits at once, on the device, from given random numbers.
//
// With x the largest finite logit of a row and T its temperature, token i weighs w_i = exp((x_i - x) / T); infinities and NaN weigh nothing.
// By falling logit, equal ones by rising index, the tokens stand in ranks.  What stays are the first top_k ranks; of those the shortest
// prefix that weighs top_p of them or more; of those the tokens of min_p and more (the first one weighs 1).  The choice is the first token, by
// index, at which the running sum of what stays is above the drawn number times the whole sum.
//
// Which token that is depends on which side of a border a sum lies on, so weights are formed in 64 bits and kept as whole numbers in units
// of 2^-47 or so of the largest (as many bits as the sum of a row has room for): sums of them are exact, whatever their order, and a row's
// answer does not depend on how the work was shared out.  A rank is found by its key, the distance of a logit's bits from the largest one's in the
// order of the numbers: histograms of counts or weights over eleven bits of it at a time lead to the key at which a sum is reached, and
// among equal keys the index decides.
#include "common.cuh"
#include "paged.cuh"

namespace hl {
namespace {

constexpr int SR_THREADS = 1024, SR_WARPS = SR_THREADS / 32;
constexpr int SR_BINS = 2048;
constexpr uint32_t SR_NONE = 0xffffffffu;  // key of what weighs nothing

struct SampleParams {
  const void* logits;
  long long ld;
  int rows, vocab;
  const float *temperature, *top_p, *min_p;
  const int32_t* top_k;
  const double* draws;
  int64_t* tokens;
  float* probabilities;
  int weight_bits;  // a weight of one is 2^weight_bits
};

__device__ __forceinline__ uint32_t ordered_bits(float x) {  // rises with x; x is not -0
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

template <typename T>
struct SampleRow {
  const T* row;
  int vocab;
  float top;           // the largest finite logit
  uint32_t top_bits;
  double inverse;      // 1 / temperature
  double unit;         // 2^weight_bits
  __device__ __forceinline__ float logit(int i) const {
    float x;
    if constexpr (sizeof(T) == 2) x = from_bf16(row[i]);
    else x = row[i];
    return x + 0.0f;  // -0 counts as 0
  }
  __device__ __forceinline__ uint32_t key(float x) const {
    return fabsf(x) < INFINITY ? top_bits - ordered_bits(x) : SR_NONE;
  }
  __device__ __forceinline__ double weight(float x) const { return exp(((double)x - (double)top) * inverse); }
  __device__ __forceinline__ unsigned long long mass(float x) const { return (unsigned long long)rint(weight(x) * unit); }
};

struct SampleShared {
  unsigned count[SR_BINS], low[SR_BINS], high[SR_BINS];
  unsigned long long warp_sum[SR_WARPS];
  unsigned long long found_below, found_bin;
  int found;
  float warp_top[SR_WARPS];
  int warp_at[SR_WARPS];
};

// Sum over the block and, in *before, over the threads before this one.
__device__ __forceinline__ unsigned long long block_prefix(unsigned long long v, unsigned long long* before, SampleShared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long up = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long other = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += other;
  }
  __syncthreads();
  if (lane == 31) sh.warp_sum[warp] = up;
  __syncthreads();
  unsigned long long at = 0, total = 0;
#pragma unroll
  for (int w = 0; w < SR_WARPS; ++w) {
    const unsigned long long x = sh.warp_sum[w];
    if (w < warp) at += x;
    total += x;
  }
  *before = at + up - v;
  return total;
}

struct Cut {  // what stays: keys below `key`, and those equal to it up to index `index`
  uint32_t key;
  int index;
  __device__ __forceinline__ bool keeps(uint32_t k, int i) const { return k < key || (k == key && i <= index); }
};

// The shortest prefix, by rank, of what `cut` keeps whose counts (or weights, BY_WEIGHT) add up to `goal` or more; `goal` is at least 1.  With
// `share` > 0 the goal is that share of the whole sum.
template <bool BY_WEIGHT, typename T>
__device__ Cut select_prefix(const SampleRow<T>& r, const Cut cut, unsigned long long goal, double share, SampleShared& sh) {
  uint32_t base = 0;
  int shift = 18;  // 32 bins an octave, so that the first bins below the largest logit are a few tokens each
  unsigned long long below = 0;
  bool first = true;
  for (;;) {
    const int bins = first ? SR_BINS - 1 : SR_BINS;
    __syncthreads();
    for (int b = threadIdx.x; b < SR_BINS; b += SR_THREADS) sh.count[b] = sh.low[b] = sh.high[b] = 0;
    if (threadIdx.x == 0) sh.found = -1;
    __syncthreads();
    unsigned long long rest = 0;  // of what lies behind the bins
    for (int i = threadIdx.x; i < r.vocab; i += SR_THREADS) {
      const float x = r.logit(i);
      const uint32_t k = r.key(x);
      if (k == SR_NONE || !cut.keeps(k, i) || k < base) continue;
      const uint32_t b = (k - base) >> shift;
      unsigned long long w = 1;
      if constexpr (BY_WEIGHT) w = r.mass(x);
      if (b >= (uint32_t)bins) {
        rest += w;
        continue;
      }
      if constexpr (BY_WEIGHT) {  // a sum of 64 bits out of two of 32
        const unsigned lo = (unsigned)w, old = atomicAdd(&sh.low[b], lo);
        const unsigned up = (unsigned)(w >> 32) + (old + lo < lo ? 1u : 0u);
        if (up) atomicAdd(&sh.high[b], up);
      } else {
        atomicAdd(&sh.count[b], 1u);
      }
    }
    unsigned long long ignored;
    const unsigned long long behind = block_prefix(rest, &ignored, sh);  // and the histogram is complete
    const int b0 = threadIdx.x * (SR_BINS / SR_THREADS);
    unsigned long long bin[SR_BINS / SR_THREADS], mine = 0;
#pragma unroll
    for (int j = 0; j < SR_BINS / SR_THREADS; ++j) {
      if constexpr (BY_WEIGHT) bin[j] = (unsigned long long)sh.high[b0 + j] << 32 | sh.low[b0 + j];
      else bin[j] = sh.count[b0 + j];
      mine += bin[j];
    }
    unsigned long long at;
    const unsigned long long total = block_prefix(mine, &at, sh);
    if (first && share > 0.0) goal = max(1ull, (unsigned long long)ceil(share * (double)(total + behind)));
    if (first) goal = min(goal, total + behind);
    at += below;
#pragma unroll
    for (int j = 0; j < SR_BINS / SR_THREADS; ++j) {
      if (at < goal && at + bin[j] >= goal) {
        sh.found = b0 + j;
        sh.found_below = at;
        sh.found_bin = bin[j];
      }
      at += bin[j];
    }
    __syncthreads();
    const int found = sh.found;
    if (found < 0) {  // behind the fine bins
      if (!first) return cut;  // the row changed between two looks at it
      base = (uint32_t)(SR_BINS - 1) << 18;
      shift = 21;
      below += total;
      first = false;
      continue;
    }
    base += (uint32_t)found << shift;
    below = sh.found_below;
    first = false;
    if (shift == 0) break;
    shift = shift == 18 ? 7 : shift == 21 ? 10 : 0;
  }
  // Equal keys weigh the same; `need` of them stay, by index.
  const unsigned long long in_bin = sh.found_bin;
  Cut out{base, base == cut.key ? cut.index : 0x7fffffff};
  unsigned long long ties = 0;  // of this thread's stretch of the row
  const int stretch = (r.vocab + SR_THREADS - 1) / SR_THREADS, i0 = min(r.vocab, (int)threadIdx.x * stretch), i1 = min(r.vocab, i0 + stretch);
  for (int i = i0; i < i1; ++i) {
    const uint32_t k = r.key(r.logit(i));
    if (k == base && cut.keeps(k, i)) ++ties;
  }
  unsigned long long before;
  const unsigned long long all = block_prefix(ties, &before, sh);
  if (all == 0) return cut;
  const unsigned long long each = max(1ull, in_bin / all), need = (goal - below + each - 1) / each;
  if (need < all) {
    if (before < need && before + ties >= need) {
      unsigned long long seen = before;
      for (int i = i0; i < i1; ++i) {
        const uint32_t k = r.key(r.logit(i));
        if (k == base && cut.keeps(k, i) && ++seen == need) sh.found = i;
      }
    }
    __syncthreads();
    out.index = sh.found;
  }
  return out;
}

template <typename T>
__global__ void __launch_bounds__(SR_THREADS) sample_rows_kernel(const SampleParams p) {
  __shared__ SampleShared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x;
  pdl_begin();
  SampleRow<T> r;
  r.row = static_cast<const T*>(p.logits) + row * p.ld;
  r.vocab = p.vocab;
  float top = -INFINITY;
  int at = 0x7fffffff;
  for (int i = tid; i < p.vocab; i += SR_THREADS) {
    const float x = r.logit(i);
    if (fabsf(x) < INFINITY && x > top) {
      top = x;
      at = i;
    }
  }
  auto better = [&](float x, int i) {
    if (x > top || (x == top && i < at)) {
      top = x;
      at = i;
    }
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float x = __shfl_xor_sync(0xffffffffu, top, o);
    better(x, __shfl_xor_sync(0xffffffffu, at, o));
  }
  if (lane == 0) {
    sh.warp_top[warp] = top;
    sh.warp_at[warp] = at;
  }
  __syncthreads();
  for (int w = 0; w < SR_WARPS; ++w) better(sh.warp_top[w], sh.warp_at[w]);
  const float temperature = p.temperature ? p.temperature[row] : 1.0f;
  const bool none = top == -INFINITY;
  if (none || !(temperature > 0.0f)) {
    if (tid == 0) {
      p.tokens[row] = none ? -1 : at;
      if (p.probabilities) p.probabilities[row] = none ? 0.0f : 1.0f;
    }
    return;
  }
  r.top = top;
  r.top_bits = ordered_bits(top);
  r.inverse = 1.0 / (double)temperature;
  r.unit = (double)(1ull << p.weight_bits);
  Cut cut{SR_NONE, -1};
  const int k = p.top_k ? p.top_k[row] : 0;
  if (k > 0 && k < p.vocab) cut = select_prefix<false>(r, cut, (unsigned long long)k, 0.0, sh);
  const float share = p.top_p ? p.top_p[row] : 1.0f;
  if (share > 0.0f && share < 1.0f) cut = select_prefix<true>(r, cut, 1ull, (double)share, sh);
  const float asked = p.min_p ? p.min_p[row] : 0.0f, least = asked > 0.0f ? fminf(asked, 1.0f) : 0.0f;  // NaN: no filter
  auto mass = [&](int i) -> unsigned long long {
    const float x = r.logit(i);
    const uint32_t key = r.key(x);
    if (key == SR_NONE || !cut.keeps(key, i)) return 0;
    const double w = r.weight(x);
    return w >= (double)least ? (unsigned long long)rint(w * r.unit) : 0;
  };
  const int stretch = (p.vocab + SR_THREADS - 1) / SR_THREADS, i0 = min(p.vocab, tid * stretch), i1 = min(p.vocab, i0 + stretch);
  unsigned long long mine = 0;
  for (int i = i0; i < i1; ++i) mine += mass(i);
  unsigned long long before;
  const unsigned long long total = block_prefix(mine, &before, sh);
  // floor(draw * total), the draw as a fraction of 2^64
  const double u = p.draws[row], most = 1.0 - 1.1102230246251565e-16;
  const unsigned long long fraction = (unsigned long long)(fmin(fmax(u, 0.0), most) * 9007199254740992.0) << 11;
  const unsigned long long target = __umul64hi(total, fraction);
  if (before <= target && before + mine > target) {
    unsigned long long seen = before;
    int i = i0;
    for (; i < i1; ++i) {
      const unsigned long long w = mass(i);
      if (seen + w > target) break;
      seen += w;
    }
    p.tokens[row] = i;
    if (p.probabilities) p.probabilities[row] = (float)(r.weight(r.logit(i)) * r.unit / (double)total);
  }
}

}  // namespace
}  // namespace hl

extern "C" int hl_sample_rows(hl_ctx* ctx, const void* logits, int dtype, long long ld, int rows, int vocab, const float* temperature,
                              const int32_t* top_k, const float* top_p, const float* min_p, const double* draws, int64_t* tokens,
                              float* probabilities) {
  using namespace hl;
  HL_REQUIRE(ctx && logits && draws && tokens, "hl_sample_rows: null argument");
  HL_REQUIRE(dtype == HL_F32 || dtype == HL_BF16, "hl_sample_rows: logits must be f32 or bf16");
  HL_REQUIRE(rows > 0 && vocab > 0, "hl_sample_rows: requires rows and at least one logit");
  HL_REQUIRE(vocab <= (1 << 30), "hl_sample_rows: at most 2^30 logits a row");
  HL_REQUIRE(ld >= vocab, "hl_sample_rows: row stride smaller than the vocabulary");
  HL_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (dtype == HL_F32 ? 3 : 1)) == 0, "hl_sample_rows: misaligned logits");
  SampleParams p{};
  p.logits = logits; p.ld = ld; p.rows = rows; p.vocab = vocab;
  p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p;
  p.draws = draws; p.tokens = tokens; p.probabilities = probabilities;
  p.weight_bits = 62;
  while ((1ll << (62 - p.weight_bits)) < vocab) --p.weight_bits;  // a row's sum stays below 2^63
  OnDevice here(ctx->device);
  ProfileScope prof(ctx, HL_PROF_OTHER, (double)rows * vocab * (double)dtype_size(dtype));
  auto launch = dtype == HL_F32 ? pdl(sample_rows_kernel<float>, rows, SR_THREADS, 0, ctx->stream)
                                : pdl(sample_rows_kernel<__nv_bfloat16>, rows, SR_THREADS, 0, ctx->stream);
  launch(p);
  HL_LAUNCH_CHECK("sample_rows_kernel");
  count_launch(ctx);
  return HL_OK;
}
