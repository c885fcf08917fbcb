// What the kernels over a paged cache share: how the cache and a ragged batch of new tokens are described, where a CTA finds its share of
// an attention call, and what it leaves of items that it did not finish.
#pragma once
#include "common.cuh"
#include "paged_deal.h"

namespace hl {

// A cache and a batch as the kernels see them: checked on the host, strides in elements, those of dimensions of one set to something
// harmless.
struct PagedView {
  void *k, *v;
  long long page_stride, position_stride, head_stride;
  int pages, page_size, page_shift, kv_heads, head_dim;
  const int32_t *page_table, *lengths, *first;
  long long ld_table;
  int table_width, sequences, tokens, max_new, max_length;
  int* status;
};
// `name`: the entry point, for messages.
int paged_view(hl_ctx* ctx, const char* name, const hl_paged_cache* cache, const hl_paged_batch* batch, PagedView* out);

// The calling thread's device for the length of a call: a context's kernels go to its own device whatever the current one is.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    if (cudaGetDevice(&before_) != cudaSuccess) before_ = device;
    if (before_ != device) cudaSetDevice(device);
    else before_ = -1;
  }
  ~OnDevice() {
    if (before_ >= 0) cudaSetDevice(before_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;

 private:
  int before_ = -1;
};

#ifdef __CUDACC__
struct Deal {
  long long total, chunk;  // length of the line; of a stream's stretch
};

// All threads of the block; `shared`: 2 * 32 + 4 words of 64 bits, free again after the call.  Sets the deal, and the sequence that holds place
// `stream * chunk` of the line (s = sequences where that is behind the end).
template <int THREADS>
__device__ __forceinline__ void deal_start(const PagedView& p, const DealShape& z, int stream, long long* shared, Deal* deal, DealPlace* place) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int WARPS = THREADS / 32;
  long long mine = 0, here = 0;  // of this thread's sequences; of the one in the first round
#pragma unroll 1
  for (int s = tid; s < p.sequences; s += THREADS) {
    const long long w = deal_sequence(p, z, s);
    if (s == tid) here = w;
    mine += w;
  }
  const long long warp_total = warp_sum(mine);
  if (lane == 0) shared[warp] = warp_total;
  __syncthreads();
  long long total = 0;
#pragma unroll 1
  for (int w = 0; w < WARPS; ++w) total += shared[w];
  deal->total = total;
  deal->chunk = max(deal_divide(total + z.streams - 1, z.streams), (long long)z.least);
  const long long target = deal->chunk * stream;
  if (tid == 0) {
    shared[64] = p.sequences;
    shared[65] = total;
  }
  long long before = 0;  // sequences of earlier rounds
#pragma unroll 1
  for (int s0 = 0; s0 < p.sequences; s0 += THREADS) {
    const long long w = s0 == 0 ? here : (s0 + tid < p.sequences ? deal_sequence(p, z, s0 + tid) : 0);
    long long up = w;  // inclusive sum over the warp
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const long long other = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += other;
    }
    __syncthreads();
    if (lane == 31) shared[32 + warp] = up;
    __syncthreads();
    long long at = before, round = 0;
#pragma unroll 1
    for (int v = 0; v < WARPS; ++v) {
      if (v < warp) at += shared[32 + v];
      round += shared[32 + v];
    }
    at += up - w;
    if (w > 0 && target >= at && target < at + w) {
      shared[64] = s0 + tid;
      shared[65] = at;
    }
    before += round;
    if (target < before) break;  // the same for all threads
  }
  __syncthreads();
  place->s = (int)shared[64];
  place->before = shared[65];
  __syncthreads();
}

// ---- pieces -------------------------------------------------------------------------------------------------------------------------
// What a stream found out about an item that it did not work on from end to end: per row sum P V, the maximum against which P was
// formed (in units of log2) and sum P.  A stream has two such pieces at most: of the item it starts in (0) and of the one it ends in (1).
__device__ __forceinline__ bool deal_whole(const DealItem& it) { return it.tile0 == 0 && it.tile1 == it.tiles; }
__device__ __forceinline__ int deal_piece(const DealItem& it) { return it.tile0 > 0 ? 0 : 1; }
// Four channels of a row stand together, and rows side by side: channel c of row r.
__device__ __forceinline__ int piece_at(int rows, int r, int c) { return ((c >> 2) * rows + r) * 4 + (c & 3); }
__host__ __device__ inline size_t piece_floats(int rows, int head_dim) { return (size_t)rows * (head_dim + 2); }
// What joins the pieces of an item, by the stream that starts it: every stream says whether it leaves one that others go on with.
struct Joint {
  int row0, count;    // rows of the batch's sequence: its first; rows of the item
  int block_row, head;  // the item's first row within its sequence, and its key head
  int streams;        // 0: nothing to join
  int unused[3];      // pieces stand behind the joints, on 16 bytes
};
__device__ __forceinline__ Joint deal_joint(const DealShape& z, const Deal& deal, const DealItem& it, int stream) {
  Joint j{};
  j.row0 = it.q.row0;
  j.block_row = it.block << z.row_shift;
  j.count = min(z.rows(), it.q.n * z.group - j.block_row);
  j.head = it.head;
  j.streams = (int)deal_divide(it.at + z.extra + it.tiles - 1, deal.chunk) - stream + 1;
  return j;
}
__device__ __forceinline__ bool deal_goes_on(const DealItem& it) { return it.tile0 == 0 && it.tile1 < it.tiles; }
#endif

}  // namespace hl
