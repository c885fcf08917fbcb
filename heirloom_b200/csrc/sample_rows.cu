// The next tokens of many rows of logits at once, on the device, from given random numbers.
//
// With x the largest finite logit of a row and T its temperature, token i weighs w_i = exp((x_i - x) / T); infinities and NaN weigh nothing.
// By falling logit, equal ones by rising index, the tokens stand in ranks.  What stays are the first top_k ranks; of those the shortest
// prefix that weighs top_p of them or more; of those the tokens of min_p and more (the first one weighs 1).  The choice is the first token, by
// index, at which the running sum of what stays is above the drawn number times the whole sum.
//
// Which token that is depends on which side of a border a sum lies on, so weights are formed to 2^-28 of
// themselves and kept as whole numbers: sums of them are exact, whatever their order, and a row's
// answer does not depend on how the work was shared out.  A unit is as small as a sum of 2^62 at most allows: 2^-62 of the largest weight
// times the vocabulary as a power of two (2^-45 for 128001 logits, which hides 2^-28 of it at most), and for more than 2^18 logits, of which 2^-25 and more could be
// missed, 2^-61 times the row's sum, which takes one look more.
//
// A row goes to a cluster of one to eight CTAs, which read it once into shared memory, a slice each.  A cut by rank takes one histogram of
// counts or weights over the distance from the largest logit, 32 bins a unit of the temperature; the tokens of the bin in which the cut
// falls, some dozens, go to the cluster's first CTA, which puts them in order.  Where everything that can stay is that few, the first CTA ends the row by itself.
// Crowds of equal or nearly equal logits, more than such a list holds, are told apart by the bits of their keys, eleven at a time, and then by index.
// Few ranks (top_k up to some hundreds, the largest logit) take no histogram: the threads' own largest logits tell where to cut.
//
// Bound, for few rows, by latency; for many by the SM that has most to do: 256 rows are two CTAs on 108 SMs and one on 40, 48 rows of 128001 (clusters of four) two on 44
// SMs, rows that differ in their controls leave the long ones alone at the end (20 % of the chip's issue slots used).  An SM with work issues in 47 to 60 % of its cycles:
// a weight is some thirty instructions in a chain, and between looks there are barriers.  256 rows of 50304 f32 logits: the largest 20 us, top-k 50 with top-p 26, all
// tokens 41, top-p 0.9 alone 77, controls that differ by row 84; one row of 50 ranks 11; 48 bf16 rows of 128001, all tokens: 29.
#include <cooperative_groups.h>

#include <type_traits>

#include "common.cuh"
#include "paged.cuh"

namespace hl {
namespace {
namespace cg = cooperative_groups;

constexpr int SR_THREADS = 512, SR_WARPS = SR_THREADS / 32;
constexpr int SR_BINS = 2048;
constexpr int SR_LIST = SR_THREADS;          // tokens that one CTA puts in order, a thread a token
constexpr int SR_CANDIDATES = 2048;          // that all CTAs of a row may send to the first one
constexpr int SR_TILES = 2048;               // of a slice, at most
constexpr int SR_TABLE_BITS = 6, SR_TABLE = 1 << SR_TABLE_BITS;  // of powers of two
constexpr int SR_UNIT = 62;                  // a weight of one is 2^62 at most
constexpr int SR_LIST_BITS = 53;             // and 2^53 among those of one list
constexpr int SR_WIDE = 1 << 18;             // up to that many logits a row's units follow from their number; the look for the sum makes 205 us 260 for 48 whole rows of a million f32
constexpr int SR_CTAS = 8;                   // of a cluster at most
constexpr int SR_LEAST = 4096;               // logits of a CTA, where a row has more of them
constexpr size_t SR_MOST = 72 * 1024;        // of a slice in shared memory
constexpr int SR_KEPT = 8192;                // tokens of a CTA's short list, where the slice is not in shared memory

struct SampleParams {
  const void* logits;
  long long ld;
  int rows, vocab;
  int slice;        // logits of a CTA
  int stretch;      // of a thread, where it takes neighbouring logits
  int tile_pieces;  // pieces of 16 bytes of a tile, a multiple of 64
  const float *temperature, *top_p, *min_p;
  const int32_t* top_k;
  const double* draws;
  int64_t* tokens;
  float* probabilities;
  int weight_bits;  // a weight of one is 2^weight_bits, up to SR_WIDE logits
};

struct __align__(16) Power {  // 2^(-j / SR_TABLE)
  long long whole;  // times 2^SR_UNIT
  float value;      // times 2^38
};

struct Cut {  // what stays: keys below `key`, and those equal to it up to index `index`
  uint32_t key;
  int index;
  __device__ __forceinline__ bool keeps(uint32_t k, int i) const { return k < key || (k == key && i <= index); }
};
struct Found {  // the bin in which a sum is reached
  unsigned long long below, in_bin;  // the sum before it, and its own
  unsigned members, upto;            // tokens in it; in it and before it
  int bin;
};

struct SampleShared {
  union {
    struct {
      unsigned count[SR_BINS], low[SR_BINS], high[SR_BINS];
    } bins;
    struct {
      unsigned long long key[SR_LIST], mass[SR_LIST], swap[2][SR_LIST];
    } list;
    struct {  // sums of the tiles; the tokens of the bin in which a cut falls, of this CTA and, in the first one, of all
      unsigned long long tile_sum[SR_TILES], own[SR_LIST], key[SR_LIST], swap[2][SR_LIST];
    } last;
    struct {  // the tokens that may be among the first ranks: of this CTA, and in the first CTA those of all
      unsigned long long own[SR_LIST], all[SR_CANDIDATES], key[SR_LIST];
    } best;
  };
  Power table[SR_TABLE];
  unsigned long long warp_sum[SR_WARPS];
  unsigned warp_count[SR_WARPS];
  float warp_top[SR_WARPS];
  int at_tile;
  unsigned long long at_rest;
  // written by the cluster's CTAs
  float cta_top[SR_CTAS], cta_weight[SR_CTAS];
  unsigned long long cta_sum[2][SR_CTAS];
  unsigned cta_count[SR_CTAS], cta_best[SR_CTAS];
  Found found;
  Cut cut;
  unsigned list_size, own_size, best_size;
  unsigned warp_best[2][SR_WARPS];
};

__device__ __forceinline__ uint32_t ordered_bits(float x) {  // rises with x; x is not -0
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered_bits(uint32_t u) { return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u); }

// A token's place among the others as a number: those of larger logits come first, of equal ones those of lower index.
__device__ __forceinline__ unsigned long long rank_key(float x, int index) { return (unsigned long long)~ordered_bits(x) << 32 | (unsigned)index; }
__device__ __forceinline__ float logit_of(unsigned long long key) { return from_ordered_bits(~(uint32_t)(key >> 32)); }

// A CTA's slice of a row and what a logit of it is worth.  It is seen as pieces of 16 bytes from the boundary at or before its start; logits of
// the first and last piece that are not the slice's read as minus infinity, like everything that has no probability.
template <typename T, bool RESIDENT>
struct Slice {
  static constexpr int N = 16 / (int)sizeof(T);
  const T* data;       // of the first piece: in shared memory, where logits are clean, or in the row itself
  int begin, length;   // the slice's place in the row
  int off, pieces;     // logits of the first piece that are not the slice's; pieces
  uint2* list;         // (logit, place) of those that still matter, in shared memory,
  int listed;          // and how many; -1 before there is such a list
  float top;           // the row's largest finite logit
  uint32_t top_bits;
  float bins;          // a unit of distance
  float per_high, per_low;  // SR_TABLE-ths of a halving in a unit of distance, in two parts
  float most;          // of those, from where on a weight is 0
  int less;            // what the bits of `shifted` are more than the places to shift by
  const Power* table;
  // a weight of one is 2^bits from now on
  __device__ __forceinline__ void set_unit(int bits) {
    less = (0x4b400000 >> SR_TABLE_BITS) - (SR_UNIT - bits);
    most = (float)((63 - (SR_UNIT - bits)) * SR_TABLE - 1);
  }
  static __device__ __forceinline__ float clean(float x) { return fabsf(x) < INFINITY ? x + 0.0f : -INFINITY; }  // 0 for -0
  static __device__ __forceinline__ float plain(T x) {
    if constexpr (sizeof(T) == 2) return from_bf16(x);
    else return x;
  }
  static __device__ __forceinline__ void unpack(const uint4& u, float (&x)[N]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) {
        const float2 f = unpack_bf16x2(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      } else {
        x[i] = __uint_as_float(w[i]);
      }
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[N]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
      else w[i] = __float_as_uint(x[i]);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ bool inner(int v) const { return v * N >= off && (v + 1) * N <= off + length; }
  __device__ __forceinline__ uint4 raw(int v) const { return reinterpret_cast<const uint4*>(data)[v]; }
  // a piece as it stands in the row: u is raw(v) where inner(v)
  __device__ __forceinline__ void from_row(int v, const uint4& u, float (&x)[N]) const {
    if (inner(v)) {
      unpack(u, x);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = v * N + i >= off && v * N + i < off + length ? plain(data[v * N + i]) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = clean(x[i]);
  }
  __device__ __forceinline__ float logit(int e) const { return RESIDENT ? plain(data[off + e]) : clean(plain(data[off + e])); }
  __device__ __forceinline__ uint32_t key(float x) const { return top_bits - ordered_bits(x); }
  // Falls with x.  Rounded by adding 2^23, to the nearest: any order-keeping cut into bins will do.
  __device__ __forceinline__ int bin(float x) const {
    return (int)min(__float_as_uint(fmaf(top - x, bins, 8388608.0f)) - 0x4b000000u, (uint32_t)(SR_BINS - 1));
  }
  // f(x, e) for four logits at a time, e their places in the slice, in no order; minus infinity among them is no logit.  Where a short list of those that
  // still matter has been made, from there.
  template <typename F>
  __device__ __forceinline__ void for_each_four(F f) const {
    if (!RESIDENT && listed >= 0) {
      for (int i0 = threadIdx.x; i0 < listed; i0 += 4 * SR_THREADS) {
        float x[4];
        int e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint2 u = i0 + i * SR_THREADS < listed ? list[i0 + i * SR_THREADS] : make_uint2(0xff800000u, 0u);
          x[i] = __uint_as_float(u.x);
          e[i] = (int)u.y;
        }
        f(x, e);
      }
      return;
    }
    constexpr int AT_ONCE = RESIDENT ? 1 : 4;  // loads on their way
    for (int v0 = threadIdx.x; v0 < pieces; v0 += AT_ONCE * SR_THREADS) {
      uint4 u[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const int v = v0 + j * SR_THREADS;
        u[j] = v < pieces && (RESIDENT || inner(v)) ? raw(v) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const int v = v0 + j * SR_THREADS;
        if (v >= pieces) break;
        float x[N];
        if constexpr (RESIDENT) unpack(u[j], x);
        else from_row(v, u[j], x);
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          const float four[4] = {x[i], x[i + 1], x[i + 2], x[i + 3]};
          const int at = v * N + i - off, e[4] = {at, at + 1, at + 2, at + 3};
          f(four, e);
        }
      }
    }
  }
  // the same for the logits with a probability, one at a time
  template <typename F>
  __device__ __forceinline__ void for_each(F f) const {
    for_each_four([&](const float (&x)[4], const int (&e)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (x[i] > -INFINITY) f(x[i], e[i]);
    });
  }
  // exp((x - top) / T) in units of 2^-weight_bits, without 64-bit units and without branches: t, the halvings, as two f32 whose sums and
  // products are exact together (Knuth's and Dekker's), a table of 64ths of a halving as whole numbers, and the Taylor polynomial of degree 3
  // for what is left (Tang 1989, "Table-driven implementation of the exponential function"): below 2^-7.5, the next term is 2^-34.7.  What
  // is too small, minus infinity too, is shifted out.  Off by 2^-28.9 of itself at most (2^-30.5 by the polynomial's two roundings, 2^-31 by that of its product
  // with the table, 2^-31.5 by that of r, as much by the table's f32 half), 2^-29.7 was the most found, and by what is shifted out, less than a unit.  Logits of both types:
  // the difference of bf16 values is rounded too, where one is below 2^-16 of the other.
  __device__ __forceinline__ unsigned long long mass(float x) const {
    constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number in the low bits
    constexpr float kLn2 = 0.69314718f / SR_TABLE;
    const float d = top - x, t = d * per_high, back = d - top;
    float u = fmaf(d, per_low, fmaf(d, per_high, -t));
    u = fmaf((top - (d - back)) - (x + back), per_high, u);
    const float shifted = fminf(t, most) + kRound;
    const int n = __float_as_int(shifted);  // its low 22 bits
    const float r = (shifted - kRound) - t - u;
    const float q = r * fmaf(r, fmaf(r, kLn2 * kLn2 * kLn2 / 6.0f, kLn2 * kLn2 / 2.0f), kLn2);
    const Power f = table[n & (SR_TABLE - 1)];
    const long long m = f.whole + (long long)__float2int_rn(f.value * q) * (1 << (SR_UNIT - 38));
    return (unsigned long long)m >> ((n >> SR_TABLE_BITS) - less);
  }
};

// Sum over the block and, in *before, over the threads before this one.
template <typename V>
__device__ __forceinline__ V block_prefix(V v, V* before, V* warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V up = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V other = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += other;
  }
  __syncthreads();
  if (lane == 31) warps[warp] = up;
  __syncthreads();
  V at = 0, total = 0;
#pragma unroll
  for (int w = 0; w < SR_WARPS; ++w) {
    const V x = warps[w];
    if (w < warp) at += x;
    total += x;
  }
  *before = at + up - v;
  return total;
}

// The block's keys in rising order, a thread a key (Batcher's bitonic network; lanes swap by shuffles, warps through `swap`).
__device__ unsigned long long block_sort(unsigned long long key, unsigned long long (*swap)[SR_LIST]) {
  const int tid = threadIdx.x;
  int turn = 0;
#pragma unroll 1
  for (int k = 2; k <= SR_THREADS; k *= 2) {
#pragma unroll 1
    for (int j = k / 2; j > 0; j /= 2) {
      unsigned long long other;
      if (j >= 32) {
        swap[turn][tid] = key;
        __syncthreads();
        other = swap[turn][tid ^ j];
        turn ^= 1;
      } else {
        other = __shfl_xor_sync(0xffffffffu, key, j);
      }
      const bool smaller = ((tid & j) == 0) == ((tid & k) == 0);
      key = (key < other) == smaller ? key : other;
    }
  }
  return key;
}
static_assert(SR_LIST == SR_THREADS, "a thread a key");

// Adds w to a sum of 64 bits made of two of 32.
__device__ __forceinline__ void add_mass(unsigned* low, unsigned* high, unsigned long long w) {
  const unsigned lo = (unsigned)w, old = atomicAdd(low, lo);
  const unsigned up = (unsigned)(w >> 32) + (old + lo < lo ? 1u : 0u);
  if (up) atomicAdd(high, up);
}

// One histogram over the cluster: bin_of(x, index) is a token's bin, or -1.  Finds the bin in which the sum of counts (or weights,
// BY_WEIGHT) plus `below` reaches `goal`; with `share` > 0 the goal becomes that share of the whole sum.  Every CTA has the answer.
//
// Tokens whose weight is 0 are not counted by weight, but whoever gathers what a bin has counted need not look for them: they are in no bin with a cut by
// weight.  Bins are of falling logit and none that has a weight is wider than 1/32 of the temperature, so beside a weight of 0 (in units, rounded down) all
// weights of the bin are 1 at most and all behind it 0, while a share is 1 - 2^-24 or less, so that what the bin and those behind it weigh is 2^-24 of the sum
// or more, less one.  The sum is at least the largest token's 2^weight_bits, 2^44, for up to SR_WIDE logits, and 2^60 for more: that would be more tokens
// of weight 1 than there are.
template <bool BY_WEIGHT, typename S, typename F>
__device__ Found histogram(const cg::cluster_group& cluster, const S& s, SampleShared& sh, unsigned long long below,
                           unsigned long long& goal, double share, F bin_of) {
  const int tid = threadIdx.x, ctas = cluster.num_blocks(), rank = cluster.block_rank();
  for (int b = tid; b < SR_BINS; b += SR_THREADS) sh.bins.count[b] = sh.bins.low[b] = sh.bins.high[b] = 0;
  __syncthreads();
  s.for_each_four([&](const float (&x)[4], const int (&e)[4]) {
    int b[4];
    unsigned long long w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      b[i] = x[i] > -INFINITY ? bin_of(x[i], s.begin + e[i]) : -1;
      w[i] = BY_WEIGHT ? s.mass(x[i]) : 1ull;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (b[i] >= 0 && w[i] > 0) {
        atomicAdd(&sh.bins.count[b[i]], 1u);
        if constexpr (BY_WEIGHT) add_mass(&sh.bins.low[b[i]], &sh.bins.high[b[i]], w[i]);
      }
  });
  cluster.sync();
  // a CTA adds up a share of the bins, over all CTAs; a thread up to four neighbours
  const int share_bins = SR_BINS / ctas, each = max(1, share_bins / SR_THREADS);
  unsigned long long sum[SR_BINS / SR_THREADS] = {}, mine = 0;
  unsigned count[SR_BINS / SR_THREADS] = {}, my_count = 0;
#pragma unroll
  for (int j = 0; j < SR_BINS / SR_THREADS; ++j) {
    const int b = tid * each + j;
    if (j < each && b < share_bins) {
      const int at = rank * share_bins + b;
      for (int c = 0; c < ctas; ++c) {
        SampleShared* peer = cluster.map_shared_rank(&sh, c);
        count[j] += peer->bins.count[at];
        if constexpr (BY_WEIGHT) sum[j] += (unsigned long long)peer->bins.high[at] << 32 | peer->bins.low[at];
      }
      if constexpr (!BY_WEIGHT) sum[j] = count[j];
    }
    mine += sum[j];
    my_count += count[j];
  }
  unsigned long long at;
  unsigned count_at;
  const unsigned long long total = block_prefix(mine, &at, sh.warp_sum);
  const unsigned all = block_prefix(my_count, &count_at, sh.warp_count);
  if (tid < ctas) {
    SampleShared* peer = cluster.map_shared_rank(&sh, tid);
    peer->cta_sum[0][rank] = total;
    peer->cta_count[rank] = all;
  }
  if (rank == 0 && tid == 0) sh.list_size = 0;
  cluster.sync();
  unsigned long long everything = 0;
  at += below;
  for (int c = 0; c < ctas; ++c) {
    if (c < rank) {
      at += sh.cta_sum[0][c];
      count_at += sh.cta_count[c];
    }
    everything += sh.cta_sum[0][c];
  }
  if (share > 0.0) goal = max(1ull, (unsigned long long)ceil(share * (double)everything));
  goal = min(goal, below + everything);
#pragma unroll
  for (int j = 0; j < SR_BINS / SR_THREADS; ++j) {
    if (at < goal && at + sum[j] >= goal) {
      const Found f{at, sum[j], count[j], count_at + count[j], rank * share_bins + tid * each + j};
      for (int c = 0; c < ctas; ++c) cluster.map_shared_rank(&sh, c)->found = f;
    }
    at += sum[j];
    count_at += count[j];
  }
  cluster.sync();
  return sh.found;
}

// The keys (and indices) of the tokens that `takes(x, index)`, in the first CTA's list, as far as it has room; list_size counts them all.
template <typename S, typename F>
__device__ void gather(const cg::cluster_group& cluster, const S& s, SampleShared& sh, F takes) {
  SampleShared* first = cluster.map_shared_rank(&sh, 0);
  s.for_each([&](float x, int e) {
    if (!takes(x, s.begin + e)) return;
    const unsigned at = atomicAdd(&first->list_size, 1u);
    if (at < SR_LIST) first->list.key[at] = rank_key(x, s.begin + e);
  });
  cluster.sync();
}

// Among tokens with one key: the index of the one that stays last when `need` of those that `cut` keeps stay.
template <typename S>
__device__ int tie_index(const cg::cluster_group& cluster, const SampleParams& p, const S& s, SampleShared& sh, const Cut cut, uint32_t key,
                         unsigned long long need) {
  const int tid = threadIdx.x, ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const int e0 = min(tid * p.stretch, s.length), e1 = min(e0 + p.stretch, s.length);
  unsigned long long ties = 0, before;
  const float equal = from_ordered_bits(s.top_bits - key);
  for (int e = e0; e < e1; ++e) ties += s.logit(e) == equal && cut.keeps(key, s.begin + e);
  const unsigned long long total = block_prefix(ties, &before, sh.warp_sum);
  if (tid < ctas) cluster.map_shared_rank(&sh, tid)->cta_sum[1][rank] = total;
  cluster.sync();
  for (int c = 0; c < rank; ++c) before += sh.cta_sum[1][c];
  if (before < need && before + ties >= need) {
    for (int e = e0; e < e1; ++e)
      if (s.logit(e) == equal && cut.keeps(key, s.begin + e) && ++before == need)
        for (int c = 0; c < ctas; ++c) cluster.map_shared_rank(&sh, c)->cut = Cut{key, s.begin + e};
  }
  cluster.sync();
  return sh.cut.index;
}

// The shortest prefix, by rank, of what `cut` keeps whose counts (or weights) add up to `goal`, given the bin in which that happens.
template <bool BY_WEIGHT, typename S>
__device__ Cut cut_in_bin(const cg::cluster_group& cluster, const SampleParams& p, const S& s, SampleShared& sh, const Cut cut,
                          unsigned long long goal, const Found f) {
  const int tid = threadIdx.x, ctas = cluster.num_blocks(), bin = f.bin;
  if (f.members <= SR_LIST) {
    gather(cluster, s, sh, [&](float x, int i) { return s.bin(x) == bin && cut.keeps(s.key(x), i); });
    if (cluster.block_rank() == 0) {
      const int n = min(sh.list_size, (unsigned)SR_LIST);
      const unsigned long long key = block_sort(tid < n ? sh.list.key[tid] : ~0ull, sh.list.swap);
      const unsigned long long mass = tid < n ? (BY_WEIGHT ? s.mass(logit_of(key)) : 1ull) : 0ull;
      unsigned long long before;
      block_prefix(mass, &before, sh.warp_sum);
      before += f.below;
      if (before < goal && before + mass >= goal)
        for (int c = 0; c < ctas; ++c) cluster.map_shared_rank(&sh, c)->cut = Cut{s.key(logit_of(key)), (int)(uint32_t)key};
    }
    cluster.sync();
    return sh.cut;
  }
  // A crowd: by the bits of the keys.
  uint32_t prefix = 0;
  Found g = f;
#pragma unroll 1
  for (int shift = 21; shift >= 0; shift = shift == 21 ? 10 : shift == 10 ? 0 : -1) {
    const int above = shift == 21 ? 32 : shift == 10 ? 21 : 10;  // bits from there on are settled
    g = histogram<BY_WEIGHT>(cluster, s, sh, g.below, goal, 0.0, [&](float x, int i) {
      const uint32_t k = s.key(x);
      const bool takes = s.bin(x) == bin && cut.keeps(k, i) && (above == 32 || k >> above == prefix >> above);
      return takes ? (int)(k >> shift) & ((1 << (above - shift)) - 1) : -1;
    });
    prefix |= (uint32_t)g.bin << shift;
  }
  // equal keys weigh the same
  const unsigned long long each = max(1ull, g.in_bin / max(1u, g.members)), need = (goal - g.below + each - 1) / each;
  if (need >= g.members) return Cut{prefix, prefix == cut.key ? cut.index : 0x7fffffff};
  return Cut{prefix, tie_index(cluster, p, s, sh, cut, prefix, need)};
}

__device__ __forceinline__ void add_to_tile(SampleShared& sh, int tile, unsigned long long mass) {
  unsigned* words = reinterpret_cast<unsigned*>(&sh.last.tile_sum[tile]);  // low, high
  if (mass > 0) add_mass(words, words + 1, mass);
}

// The sum over the block of numbers up to a few; `turn` changes from call to call.
__device__ __forceinline__ unsigned block_total(unsigned v, int turn, SampleShared& sh) {
  v = __reduce_add_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) sh.warp_best[turn & 1][threadIdx.x >> 5] = v;
  __syncthreads();
  unsigned total = 0;
#pragma unroll
  for (int w = 0; w < SR_WARPS; ++w) total += sh.warp_best[turn & 1][w];
  return total;
}

// The choice among at most a block of tokens, a thread a token (`key`; ~0 for none), which are all that can stay.  n: how many there are; the keys
// stand in sh.list.key as well.  k, share: 0 for none; goal: 0, or the mass that top_p asks for.
template <typename S>
__device__ void choose_from_list(const SampleParams& p, const S& s, SampleShared& sh, int row, unsigned long long key, int n, int k, double share,
                                 unsigned long long goal, float lowest, unsigned long long fraction) {
  const int tid = threadIdx.x;
  const bool sorts = n > 64;  // below, each looks at each, which takes no barriers (n of 64: 1.6 us, as much as two sorts)
  if (sorts) key = block_sort(key, sh.list.swap);
  const bool mine = tid < n;
  const unsigned long long weight = mine ? s.mass(logit_of(key)) : 0ull;
  unsigned long long mass = weight, before = 0, ignored;
  int ranks = tid;
  if (sorts) {
    block_prefix(mass, &before, sh.warp_sum);
  } else {
    sh.list.mass[tid] = mass;
    __syncthreads();
    ranks = 0;
    if (mine) {
#pragma unroll 4
      for (int j = 0; j < n; ++j)
        if (sh.list.key[j] < key) {
          before += sh.list.mass[j];
          ++ranks;
        }
    }
  }
  if (k > 0 && share > 0.0) {
    const unsigned long long sum = block_prefix(ranks < k ? mass : 0ull, &ignored, sh.warp_sum);
    goal = max(1ull, (unsigned long long)ceil(share * (double)sum));
  }
  if ((k > 0 && ranks >= k) || (goal > 0 && before >= goal) || (mine && logit_of(key) < lowest)) mass = 0;
  __syncthreads();
  sh.list.mass[tid] = mass;
  const unsigned long long sum = block_prefix(mass, &before, sh.warp_sum), target = __umul64hi(sum, fraction);
  const unsigned index = (unsigned)key;
  if (sorts) {  // by index; the thread that a token had goes along
    const unsigned long long moved = block_sort(mass > 0 ? (unsigned long long)index << 32 | (unsigned)tid : ~0ull, sh.list.swap);
    const unsigned long long m = moved != ~0ull ? sh.list.mass[(unsigned)moved] : 0;
    block_prefix(m, &before, sh.warp_sum);
    if (before <= target && before + m > target) sh.at_tile = (int)(unsigned)moved;
    __syncthreads();
    if (tid != sh.at_tile) return;
  } else {
    if (mass == 0) return;
    unsigned long long at = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j)
      if ((unsigned)sh.list.key[j] < index) at += sh.list.mass[j];
    if (at > target || at + mass <= target) return;
  }
  p.tokens[row] = index;
  if (p.probabilities) p.probabilities[row] = (float)((double)weight / (double)sum);
}

// The key of rank k - 1, given the smallest and the largest key and how many keys lie below a number; or a number between that key and the next.
template <typename F>
__device__ __forceinline__ unsigned long long key_of_rank(int k, unsigned long long smallest, unsigned long long largest, F below) {
  const int bits = 64 - __clzll(smallest ^ largest);  // in which keys differ
  unsigned long long value = bits == 64 ? 0 : smallest >> bits << bits;
#pragma unroll 1
  for (int bit = bits - 1; bit >= 0; --bit) {
    const unsigned long long next = value | 1ull << bit;
    const unsigned c = below(next);
    if (c == (unsigned)k) return next - 1;
    if (c < (unsigned)k) value = next;
  }
  return value;
}

// The candidates of all CTAs, cut down to those of the first k ranks, in sh.list.key of the first CTA, ~0 behind them.  Returns their number.
__device__ int first_ranks(SampleShared& sh, int ctas, int room, int k) {
  constexpr int MOST = SR_CANDIDATES / SR_THREADS, LANE_MOST = SR_LIST / 32;
  const int tid = threadIdx.x, lane = tid & 31;
  unsigned total = 0;
  for (int c = 0; c < ctas; ++c) total += sh.cta_best[c];
  unsigned long long key[MOST], limit;  // keys up to the limit stay
  unsigned long long smallest = ~0ull, largest = 0;
  unsigned at = 0;                              // candidates of the CTAs before
#pragma unroll
  for (int u = 0; u < MOST; ++u) key[u] = ~0ull;
  for (int c = 0; c < ctas; ++c) {
    const unsigned n = sh.cta_best[c];
#pragma unroll
    for (int u = 0; u < MOST; ++u) {
      const unsigned i = tid + u * SR_THREADS - at;
      if (i < n) key[u] = sh.best.all[c * room + i];
    }
    at += n;
  }
#pragma unroll
  for (int u = 0; u < MOST; ++u) {
    smallest = min(smallest, key[u]);
    if (key[u] != ~0ull) largest = max(largest, key[u]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    smallest = min(smallest, __shfl_xor_sync(0xffffffffu, smallest, o));
    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));
  }
  __syncthreads();  // the lists share memory
  if (lane == 0) {
    sh.list.swap[0][tid >> 5] = smallest;
    sh.list.swap[1][tid >> 5] = largest;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SR_WARPS; ++w) {
    smallest = min(smallest, sh.list.swap[0][w]);
    largest = max(largest, sh.list.swap[1][w]);
  }
  if (k == 1) {
    if (tid == 0) sh.list.key[0] = smallest;
    __syncthreads();
    if (tid > 0) sh.list.key[tid] = ~0ull;
    __syncthreads();
    return total > 0 ? 1 : 0;
  }
  if (total <= SR_LIST) {  // a thread a candidate; one warp looks for the k-th, which takes no barriers
    sh.list.key[tid] = key[0];
    if (total <= (unsigned)k) {
      __syncthreads();
      return total;
    }
    __syncthreads();
    if (tid < 32) {
      unsigned long long mine[LANE_MOST];
#pragma unroll
      for (int u = 0; u < LANE_MOST; ++u) mine[u] = sh.list.key[lane + u * 32];
      const int turns = (total + 31) / 32;
      const unsigned long long value = key_of_rank(k, smallest, largest, [&](unsigned long long next) {
        unsigned c = 0;
#pragma unroll
        for (int u = 0; u < LANE_MOST; ++u)
          if (u < turns) c += mine[u] < next;
        return __reduce_add_sync(0xffffffffu, c);
      });
      unsigned n = 0;
#pragma unroll
      for (int u = 0; u < LANE_MOST; ++u) {
        if (u >= turns) break;
        const unsigned stays = __ballot_sync(0xffffffffu, mine[u] <= value);
        if (mine[u] <= value) sh.list.key[n + __popc(stays & ((1u << lane) - 1u))] = mine[u];
        n += __popc(stays);
      }
    }
    __syncthreads();
    if (tid >= k) sh.list.key[tid] = ~0ull;
    __syncthreads();
    return k;
  }
  int turn = 0;
  limit = key_of_rank(k, smallest, largest, [&](unsigned long long next) {
    unsigned c = 0;
#pragma unroll
    for (int u = 0; u < MOST; ++u) c += key[u] < next;
    return block_total(c, turn++, sh);
  });
  if (tid == 0) sh.best_size = 0;
  sh.list.key[tid] = ~0ull;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < MOST; ++u)
    if (key[u] <= limit) {
      const unsigned to = atomicAdd(&sh.best_size, 1u);
      if (to < SR_LIST) sh.list.key[to] = key[u];
    }
  __syncthreads();
  return k;
}

template <typename T, bool RESIDENT>
__global__ void __launch_bounds__(SR_THREADS, 2) sample_rows_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t sr_smem[];
  __shared__ SampleShared sh;
  const cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / ctas;
  if (tid < SR_TABLE) {
    const double f = exp2(-(double)tid / SR_TABLE);
    sh.table[tid] = Power{llrint(f * (double)(1ll << SR_UNIT)), (float)(f * (double)(1ll << 38))};
  }
  if (tid == 0) sh.own_size = 0;
  cluster.barrier_arrive();  // waited for before the first access to a neighbour, who has started then
  pdl_begin();
  Slice<T, RESIDENT> s;
  s.begin = min(rank * p.slice, p.vocab);
  s.length = min(p.slice, p.vocab - s.begin);
  s.table = sh.table;
  s.list = reinterpret_cast<uint2*>(sr_smem);
  s.listed = -1;
  const T* from = static_cast<const T*>(p.logits) + row * p.ld + s.begin;
  s.off = (int)((reinterpret_cast<uintptr_t>(from) & 15) / sizeof(T));
  s.pieces = s.length > 0 ? (s.off + s.length + s.N - 1) / s.N : 0;
  s.data = from - s.off;
  float top = -INFINITY;
  uint4* kept = reinterpret_cast<uint4*>(sr_smem);
  constexpr int AT_ONCE = 8;
  for (int v0 = tid; v0 < s.pieces; v0 += AT_ONCE * SR_THREADS) {
    uint4 u[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int v = v0 + j * SR_THREADS;
      u[j] = v < s.pieces && s.inner(v) ? s.raw(v) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int v = v0 + j * SR_THREADS;
      if (v >= s.pieces) break;
      float x[s.N];
      s.from_row(v, u[j], x);
#pragma unroll
      for (int i = 0; i < s.N; ++i) top = fmaxf(top, x[i]);
      if constexpr (RESIDENT) kept[v] = s.pack(x);
    }
  }
  if constexpr (RESIDENT) s.data = reinterpret_cast<const T*>(sr_smem);
  const float temperature = p.temperature ? p.temperature[row] : 1.0f;
  const int k = p.top_k ? p.top_k[row] : 0;
  const float share = p.top_p ? p.top_p[row] : 1.0f, asked = p.min_p ? p.min_p[row] : 0.0f;
  const bool greedy = !(temperature > 0.0f), by_k = k > 0 && k < p.vocab, by_p = share > 0.0f && share < 1.0f;
  // floor(draw * sum), the draw as a fraction of 2^64
  const unsigned long long fraction = (unsigned long long)(fmin(fmax(p.draws[row], 0.0), 1.0 - 1.1102230246251565e-16) * 9007199254740992.0) << 11;
  {
    const double per = fmin(1.4426950408889634074 * SR_TABLE / (double)temperature, 1e38);  // temperatures from 1e-36 on are told apart
    s.per_high = (float)per;
    s.per_low = (float)(per - (double)s.per_high);
    s.set_unit(SR_LIST_BITS);
  }

  // The smallest logit of which a token weighs min_p of the largest: w >= min_p where x >= top + T ln(min_p).  NaN: no filter.
  auto lowest_logit = [&](float largest) {
    return asked > 0.0f ? asked < 1.0f ? __double2float_ru((double)largest + (double)temperature * log((double)asked)) : largest : -INFINITY;
  };

  // Few ranks (one, at temperature 0): where that many threads have seen a logit of some size, that many logits of the CTA's slice are as large, so
  // the first ranks of the row are among those.  A sixteen-bit threshold on the threads' largest logits leaves little more than k
  // tokens a CTA, and one exchange.
  const int ranks = greedy ? 1 : by_k ? k : 0, room = min(SR_LIST, SR_CANDIDATES / ctas);
  const bool few_ranks = ranks > 0 && ranks <= room * 3 / 4;
  if (few_ranks) {
    const unsigned seen = top > -INFINITY ? ordered_bits(top) >> 16 : 0u;
    unsigned enough = 0;
#pragma unroll 1
    for (int bit = 15; bit >= 0; --bit)
      if (__syncthreads_count(seen >= (enough | 1u << bit)) >= ranks) enough |= 1u << bit;
    const float threshold = enough > 0 ? from_ordered_bits(enough << 16) : -3.402823466e38f;
    s.for_each([&](float x, int e) {
      if (x >= threshold) {
        const unsigned at = atomicAdd(&sh.own_size, 1u);
        if (at < SR_LIST) sh.best.own[at] = rank_key(x, s.begin + e);
      }
    });
    __syncthreads();
    const unsigned n = sh.own_size;
    cluster.barrier_wait();  // the first CTA has started
    if (tid < min((int)n, room)) cluster.map_shared_rank(&sh, 0)->best.all[rank * room + tid] = sh.best.own[tid];
    if (tid < ctas) cluster.map_shared_rank(&sh, tid)->cta_best[rank] = n;
    cluster.sync();
    bool fits = true;
    for (int c = 0; c < ctas; ++c) fits &= sh.cta_best[c] <= (unsigned)room;
    if (fits) {
      if (rank != 0) return;
      const int found = first_ranks(sh, ctas, room, ranks);
      const unsigned long long key = sh.list.key[tid];
      if (found == 0 || greedy) {
        if (tid == 0) {
          p.tokens[row] = found == 0 ? -1 : (long long)(unsigned)key;
          if (p.probabilities) p.probabilities[row] = found == 0 ? 0.0f : 1.0f;
        }
        return;
      }
      float most = tid < found ? logit_of(key) : -INFINITY;
      most = warp_max(most);
      if (lane == 0) sh.warp_top[warp] = most;
      __syncthreads();
      s.top = -INFINITY;
      for (int w = 0; w < SR_WARPS; ++w) s.top = fmaxf(s.top, sh.warp_top[w]);
      choose_from_list(p, s, sh, row, key, found, ranks, by_p ? (double)share : 0.0, 0, lowest_logit(s.top), fraction);
      return;
    }
    // too many equal ones
  } else {
    cluster.barrier_wait();
  }
  top = warp_max(top);
  if (lane == 0) sh.warp_top[warp] = top;
  __syncthreads();
  if (warp == 0) {
    top = warp_max(lane < SR_WARPS ? sh.warp_top[lane] : -INFINITY);
    if (lane < ctas) cluster.map_shared_rank(&sh, lane)->cta_top[rank] = top;
  }
  cluster.sync();
  s.top = -INFINITY;
  for (int c = 0; c < ctas; ++c) s.top = fmaxf(s.top, sh.cta_top[c]);
  const int e0 = min(tid * p.stretch, s.length), e1 = min(e0 + p.stretch, s.length);
  if (s.top == -INFINITY) {
    if (rank == 0 && tid == 0) {
      p.tokens[row] = -1;
      if (p.probabilities) p.probabilities[row] = 0.0f;
    }
    return;
  }
  s.top_bits = ordered_bits(s.top);
  if (greedy) {  // so many equal ones that no list holds them
    int best = 0x7fffffff;
    for (int e = e1 - 1; e >= e0; --e)
      if (s.logit(e) == s.top) best = s.begin + e;
    best = __reduce_min_sync(0xffffffffu, best);
    if (lane == 0) sh.warp_best[0][warp] = (unsigned)best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 0; w < SR_WARPS; ++w) best = min(best, (int)sh.warp_best[0][w]);
      cluster.map_shared_rank(&sh, 0)->cta_best[rank] = (unsigned)best;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
      for (int c = 0; c < ctas; ++c) best = min(best, (int)sh.cta_best[c]);
      p.tokens[row] = best;
      if (p.probabilities) p.probabilities[row] = 1.0f;
    }
    return;
  }
  if (p.vocab <= SR_WIDE) {
    s.set_unit(p.weight_bits);
  } else {
    const float per = s.per_high / SR_TABLE;
    float weight = 0.0f;  // of this thread's logits; up to 2^15 additions are off by 2^-9 of the sum
    s.for_each_four([&](const float (&x)[4], const int (&)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) weight += x[i] > -INFINITY ? ex2_fast(fmaxf(x[i] - s.top, -3.402823466e38f) * per) : 0.0f;
    });
    weight = warp_sum(weight);
    if (lane == 0) sh.warp_top[warp] = weight;
    __syncthreads();
    if (warp == 0) {
      weight = warp_sum(lane < SR_WARPS ? sh.warp_top[lane] : 0.0f);
      if (lane < ctas) cluster.map_shared_rank(&sh, lane)->cta_weight[rank] = weight;
    }
    cluster.sync();
    weight = 0.0f;
    for (int c = 0; c < ctas; ++c) weight += sh.cta_weight[c];
    s.set_unit(61 - ilogbf(weight * 1.01f));
  }
  s.bins = fminf(32.0f / temperature, 3.465e37f);  // where the weights stop telling temperatures apart as well
  Cut cut{0xffffffffu, -1};
  int pending = -1;  // the bin in which a cut by weight is still to be made
  unsigned long long pending_goal = 0, pending_below = 0;
  if (by_k || by_p) {
    unsigned long long goal = (unsigned long long)k;
    const auto all = [&](float x, int) { return s.bin(x); };
    const Found f = by_k ? histogram<false>(cluster, s, sh, 0, goal, 0.0, all) : histogram<true>(cluster, s, sh, 0, goal, (double)share, all);
    const int bin = f.bin;
    if (f.upto <= SR_LIST) {  // all that can stay
      gather(cluster, s, sh, [&](float x, int) { return s.bin(x) <= bin; });
      if (rank != 0) return;
      const int n = min(sh.list_size, (unsigned)SR_LIST);
      choose_from_list(p, s, sh, row, tid < n ? sh.list.key[tid] : ~0ull, n, by_k ? k : 0, by_p ? (double)share : 0.0, by_k ? 0ull : goal, lowest_logit(s.top), fraction);
      return;
    }
    if (!RESIDENT && f.upto <= SR_KEPT) {  // what lies behind does not stay: from here on the few are looked at
      if (tid == 0) sh.own_size = 0;
      __syncthreads();
      s.for_each([&](float x, int e) {
        if (s.bin(x) > bin) return;
        const unsigned at = atomicAdd(&sh.own_size, 1u);
        if (at < SR_KEPT) s.list[at] = make_uint2(__float_as_uint(x), (unsigned)e);
      });
      __syncthreads();
      s.listed = min(sh.own_size, (unsigned)SR_KEPT);
      __syncthreads();  // the count is used again
    }
    Found g = f;
    if (by_k) {
      cut = cut_in_bin<false>(cluster, p, s, sh, cut, goal, f);
      if (by_p) {
        const Cut ranked = cut;
        g = histogram<true>(cluster, s, sh, 0, goal, (double)share, [&](float x, int i) { return ranked.keeps(s.key(x), i) ? s.bin(x) : -1; });
      }
    }
    if (by_p) {
      if (g.members <= SR_LIST) {  // the last cut is made on the way through the last sums
        pending = g.bin;
        pending_goal = goal;
        pending_below = g.below;
      } else {
        cut = cut_in_bin<true>(cluster, p, s, sh, cut, goal, g);
      }
    }
  }

  // What stays, by index: sums over tiles of the slice, a warp a tile and N logits a lane, then the tile in which the sum is reached.  With a bin in which a
  // cut is still to be made, what lies before that bin is added up, and the bin's own tokens afterwards.
  float last = 0.0f;  // the last logit that stays, up to some index
  int last_index = 0;
  const float lowest = lowest_logit(s.top);
  auto stays_to = [&](const Cut& c) {
    last = c.key == 0xffffffffu ? -3.402823466e38f : from_ordered_bits(s.top_bits - c.key);
    last_index = c.key == 0xffffffffu ? 0x7fffffff : c.index;
  };
  stays_to(cut);
  auto stays = [&](float x, int e) { return x > last || (x == last && s.begin + e <= last_index); };
  if (pending >= 0) {
    if (tid == 0) sh.own_size = 0;
    __syncthreads();
  }
  auto weight = [&](auto cutting, float x, int e) -> unsigned long long {
    const unsigned long long w = s.mass(x);
    bool counts = stays(x, e);
    if constexpr (decltype(cutting)::value) {
      const int b = s.bin(x);
      if (counts && b == pending) {
        const unsigned at = atomicAdd(&sh.own_size, 1u);
        if (at < SR_LIST) sh.last.own[at] = rank_key(x, s.begin + e);
      }
      counts = counts && b < pending;
    }
    return counts && x >= lowest ? w : 0;
  };
  const int tile = p.tile_pieces, tiles = (s.pieces + tile - 1) / tile;  // at most SR_TILES
  auto add_up = [&](auto cutting) {
    const float from = decltype(cutting)::value ? last : fmaxf(last, lowest);  // nothing below it
    if (!RESIDENT && s.listed >= 0) {
      for (int t = tid; t < tiles; t += SR_THREADS) sh.last.tile_sum[t] = 0;
      __syncthreads();
      s.for_each([&](float x, int e) { add_to_tile(sh, (e + s.off) / (tile * s.N), weight(cutting, x, e)); });
    } else {
      for (int t = warp; t < tiles; t += SR_WARPS) {
        unsigned long long sum = 0;
        const int end = min((t + 1) * tile, s.pieces);
        constexpr int AT_ONCE = RESIDENT ? 1 : 2;  // loads on their way
        for (int v0 = t * tile + lane; v0 < end; v0 += AT_ONCE * 32) {
          uint4 u[AT_ONCE];
#pragma unroll
          for (int j = 0; j < AT_ONCE; ++j) u[j] = v0 + j * 32 < end && (RESIDENT || s.inner(v0 + j * 32)) ? s.raw(v0 + j * 32) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int j = 0; j < AT_ONCE; ++j) {
            const int v = v0 + j * 32;
            if (v >= end) break;
            float x[s.N];
            if constexpr (RESIDENT) s.unpack(u[j], x);
            else s.from_row(v, u[j], x);
#pragma unroll
            for (int i = 0; i < s.N; i += 4) {
              if (fmaxf(fmaxf(x[i], x[i + 1]), fmaxf(x[i + 2], x[i + 3])) >= from) {
                const int e = v * s.N + i - s.off;
                sum += (weight(cutting, x[i], e) + weight(cutting, x[i + 1], e + 1)) + (weight(cutting, x[i + 2], e + 2) + weight(cutting, x[i + 3], e + 3));
              }
            }
          }
        }
        sum = warp_sum(sum);
        if (lane == 0) sh.last.tile_sum[t] = sum;
      }
    }
  };
  if (pending >= 0) add_up(std::true_type{});
  else add_up(std::false_type{});
  __syncthreads();
  if (pending >= 0) {
    // The bin's tokens of all CTAs, in order, in the first one; then everybody adds its own that stay.
    const int own = min(sh.own_size, (unsigned)SR_LIST);
    if (tid < ctas) cluster.map_shared_rank(&sh, tid)->cta_best[rank] = own;
    cluster.sync();
    int n = 0, before = 0;
    for (int c = 0; c < ctas; ++c) {
      if (c < rank) before += sh.cta_best[c];
      n += sh.cta_best[c];
    }
    if (tid < own && before + tid < SR_LIST) cluster.map_shared_rank(&sh, 0)->last.key[before + tid] = sh.last.own[tid];
    cluster.sync();
    if (rank == 0) {
      const unsigned long long key = block_sort(tid < n ? sh.last.key[tid] : ~0ull, sh.last.swap);
      const unsigned long long mass = tid < n ? s.mass(logit_of(key)) : 0ull;
      unsigned long long at;
      block_prefix(mass, &at, sh.warp_sum);
      at += pending_below;
      if (at < pending_goal && at + mass >= pending_goal)
        for (int c = 0; c < ctas; ++c) cluster.map_shared_rank(&sh, c)->cut = Cut{s.key(logit_of(key)), (int)(uint32_t)key};
    }
    cluster.sync();
    stays_to(sh.cut);
    if (tid < own) {
      const unsigned long long key = sh.last.own[tid];
      const float x = logit_of(key);
      const int e = (int)(uint32_t)key - s.begin;
      if (stays(x, e) && x >= lowest) add_to_tile(sh, (e + s.off) / (tile * s.N), s.mass(x));
    }
    __syncthreads();
  }
  constexpr int EACH = SR_TILES / SR_THREADS;  // neighbouring tiles of a thread
  unsigned long long part[EACH], mine = 0, before;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    part[j] = tid * EACH + j < tiles ? sh.last.tile_sum[tid * EACH + j] : 0;
    mine += part[j];
  }
  const unsigned long long total = block_prefix(mine, &before, sh.warp_sum);
  if (tid < ctas) cluster.map_shared_rank(&sh, tid)->cta_sum[1][rank] = total;
  cluster.sync();
  unsigned long long sum = 0, here = 0;
  for (int c = 0; c < ctas; ++c) {
    if (c < rank) here += sh.cta_sum[1][c];
    sum += sh.cta_sum[1][c];
  }
  const unsigned long long target = __umul64hi(sum, fraction);
  if (target < here || target >= here + total) return;
  before += here;
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    if (before <= target && before + part[j] > target) {
      sh.at_tile = tid * EACH + j;
      sh.at_rest = target - before;
    }
    before += part[j];
  }
  __syncthreads();
  if (warp > 0) return;
  const int b0 = max(0, sh.at_tile * tile * s.N - s.off), b1 = min(s.length, (sh.at_tile + 1) * tile * s.N - s.off);
  unsigned long long rest = sh.at_rest;
  for (int b = b0; b < b1; b += 32) {
    const int e = b + lane;
    const unsigned long long m = e < b1 ? weight(std::false_type{}, s.logit(e), e) : 0;
    unsigned long long up = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long other = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += other;
    }
    if (up > rest && up - m <= rest) {
      p.tokens[row] = s.begin + e;
      if (p.probabilities) p.probabilities[row] = (float)((double)m / (double)sum);
    }
    const unsigned long long all = __shfl_sync(0xffffffffu, up, 31);
    if (all > rest) break;
    rest -= all;
  }
}

// CTAs a row: as many as are resident at once for all rows, and slices of some size (256 rows of top-k 50 with 1, 2, 4 CTAs a row: 25, 36, 46 us; 48 rows of 128001:
// 41, 32, 24; one row 17, 13, 11).
int row_ctas(const hl_ctx* ctx, int rows, int vocab) {
  int c = 1;
  while (c < SR_CTAS && 2ll * c * rows <= 2ll * ctx->sm_count && vocab >= 2 * c * SR_LEAST) c *= 2;
  return c;
}

template <typename T>
int sample(hl_ctx* ctx, SampleParams& p) {
  constexpr int N = 16 / (int)sizeof(T);
  const int ctas = row_ctas(ctx, p.rows, p.vocab);
  p.slice = ceil_div(p.vocab, ctas);
  p.stretch = ceil_div(p.slice, SR_THREADS);
  p.tile_pieces = 64 * ceil_div(ceil_div(p.slice, N) + 1, 64 * SR_TILES);
  const size_t shared = ((size_t)ceil_div(p.slice, N) + 1) * 16;
  const dim3 grid((unsigned)(p.rows * ctas));
  // Two CTAs an SM hide each other's waits; a slice that would leave room for one is read again from L2 instead.
  if (shared <= SR_MOST) {
    HL_ALLOW_SHARED(ctx, SR_MOST, sample_rows_kernel<T, true>);
    HL_CUDA(launch_pdl(sample_rows_kernel<T, true>, grid, SR_THREADS, shared, ctx->stream, ctas, p));
  } else {
    HL_ALLOW_SHARED(ctx, SR_KEPT * sizeof(uint2), sample_rows_kernel<T, false>);
    HL_CUDA(launch_pdl(sample_rows_kernel<T, false>, grid, SR_THREADS, SR_KEPT * sizeof(uint2), ctx->stream, ctas, p));
  }
  HL_LAUNCH_CHECK("sample_rows_kernel");
  count_launch(ctx);
  return HL_OK;
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
  HL_REQUIRE(vocab <= (1 << 24), "hl_sample_rows: at most 2^24 logits a row");
  HL_REQUIRE(rows <= (1 << 24), "hl_sample_rows: at most 2^24 rows");
  HL_REQUIRE(ld >= vocab, "hl_sample_rows: row stride smaller than the vocabulary");
  HL_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (dtype == HL_F32 ? 3 : 1)) == 0, "hl_sample_rows: misaligned logits");
  SampleParams p{};
  p.logits = logits; p.ld = ld; p.rows = rows; p.vocab = vocab;
  p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p;
  p.draws = draws; p.tokens = tokens; p.probabilities = probabilities;
  p.weight_bits = SR_UNIT;
  while ((1ll << (SR_UNIT - p.weight_bits)) < vocab) --p.weight_bits;  // a row's sum is 2^62 at most
  OnDevice here(ctx->device);
  ProfileScope prof(ctx, HL_PROF_OTHER, (double)rows * vocab * (double)dtype_size(dtype));
  return dtype == HL_F32 ? sample<float>(ctx, p) : sample<__nv_bfloat16>(ctx, p);
}
