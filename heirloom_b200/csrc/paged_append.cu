// New keys and values into a paged cache, turned by their positions on the way; the queries beside them.
//
// A channel pair (x, y) of a token at position t becomes (x cos a - y sin a, x sin a + y cos a) with a = t * frequency[pair]; channels
// behind the rotated ones, and values, are copied.  Angles are products of whole numbers and f32 frequencies formed in 64 bits (a position
// of 100000 in f32 would be off by a hundredth of a turn's radian), reduced to a fraction of a turn there, and only then given to f32 functions;
// what the fraction loses as it is rounded for them is put right to first order, so that sines are off by their own rounding.
//
// Bound by memory: every element is read once and written once.  A CTA takes a few tokens, forms their sines once in shared memory, and its
// threads walk over the 16-byte pieces of all heads (of 8 bytes where halves of the turned channels end within 16:
// the same prompts with 32 heads of 80 in bf16, 40 channels turned, 76 us, all 80 in pieces of 16 bytes 45).  13 prompts in chunks of 7 to 2048 tokens, 32 heads of 128 on 8 key heads: 62 us, 5.6 TB/s, 85 % of the copy
// rate; 64 one-token rows of 12 heads of 64: 3.0 us.
#include <type_traits>

#include "paged.cuh"

namespace hl {

int paged_view(hl_ctx* ctx, const char* name, const hl_paged_cache* c, const hl_paged_batch* b, PagedView* out) {
  const std::string at = std::string(name) + ": ";
  HL_REQUIRE(ctx && c && b, at + "null argument");
  HL_REQUIRE(c->k_pages && c->v_pages && b->page_table && b->lengths, at + "null argument");
  HL_REQUIRE(c->dtype == HL_BF16 || c->dtype == HL_F32, at + "the cache holds bf16 or f32");
  HL_REQUIRE(c->pages > 0 && c->kv_heads > 0, at + "the cache needs pages and heads");
  HL_REQUIRE(c->page_size >= 16 && c->page_size <= (1 << 20) && (c->page_size & (c->page_size - 1)) == 0,
             at + "page_size must be a power of two from 16 on");
  HL_REQUIRE(c->head_dim >= 8 && c->head_dim <= 256 && c->head_dim % 8 == 0, at + "head_dim must be a multiple of 8 up to 256");
  HL_REQUIRE(b->sequences > 0 && b->tokens > 0 && b->max_new > 0 && b->table_width > 0, at + "requires sequences, tokens and pages");
  HL_REQUIRE(b->ld_table >= b->table_width || b->sequences == 1, at + "page table rows overlap");
  HL_REQUIRE(b->first || (b->tokens == b->sequences && b->max_new == 1), at + "without `first` every sequence has one new token");
  const long long capacity = (long long)b->table_width * c->page_size;
  HL_REQUIRE(b->max_length >= 0 && b->max_length <= capacity, at + "max_length is more than the page table's rows hold");
  HL_REQUIRE(b->max_length > 0 || capacity <= 0x7fffffffll, at + "the page table's rows hold more than 2^31 positions: give max_length");
  PagedView v{};
  v.k = c->k_pages;
  v.v = c->v_pages;
  v.pages = c->pages;
  v.page_size = c->page_size;
  while ((1 << v.page_shift) < c->page_size) ++v.page_shift;
  v.kv_heads = c->kv_heads;
  v.head_dim = c->head_dim;
  v.page_stride = c->page_stride;
  v.position_stride = c->position_stride;
  v.head_stride = c->kv_heads == 1 ? c->head_dim : c->head_stride;
  if (c->pages == 1) v.page_stride = std::max(v.position_stride, v.head_stride);  // that of a single page says nothing
  const long long step = c->dtype == HL_BF16 ? 8 : 4;  // 16 bytes
  HL_REQUIRE(v.position_stride >= c->head_dim && v.head_stride >= c->head_dim && v.page_stride >= c->head_dim, at + "cache rows overlap");
  HL_REQUIRE(v.position_stride % step == 0 && v.head_stride % step == 0 && v.page_stride % step == 0,
             at + "cache strides must be multiples of 16 bytes");
  HL_REQUIRE(((reinterpret_cast<uintptr_t>(c->k_pages) | reinterpret_cast<uintptr_t>(c->v_pages)) & 15) == 0,
             at + "cache pointers must be 16-byte aligned");
  v.page_table = b->page_table;
  v.lengths = b->lengths;
  v.first = b->first;
  v.ld_table = b->ld_table;
  v.table_width = b->table_width;
  v.sequences = b->sequences;
  v.tokens = b->tokens;
  v.max_new = b->max_new;
  v.max_length = b->max_length > 0 ? b->max_length : (int)capacity;
  v.status = ctx->status_dev;
  *out = v;
  return HL_OK;
}

namespace {

constexpr int PA_THREADS = 256;
constexpr int PA_MAX_TOKENS = 8;    // of a CTA
constexpr int PA_LOOK = 1024;       // sequences that every block looks at
constexpr int PA_MAX_ANGLES = 512;  // PA_MAX_TOKENS tokens or fewer times pairs

struct AppendParams {
  PagedView p;
  const void *q, *k, *v;
  void* q_out;
  long long ld_q, ld_k, ld_v, ld_q_out;
  const float* frequencies;
  int pairs;          // channel pairs that are turned
  int interleaved;
  int heads;          // query heads, 0 without queries
  int tokens;         // of a CTA
  int units;          // pieces, or pairs of them, of a head
  int token_units;    // of all heads of a token
  int q_units, k_units;
  QuickDiv by_token_units, by_units;
};

template <typename T, int BYTES>
struct Piece {  // of 16 bytes, or 8
  static constexpr int N = BYTES / (int)sizeof(T), WORDS = BYTES / 4;
  using Raw = std::conditional_t<BYTES == 16, uint4, uint2>;
  float x[N];
  __device__ __forceinline__ void load(const T* from) {
    const Raw u = *reinterpret_cast<const Raw*>(from);
    uint32_t w[WORDS];
    w[0] = u.x;
    w[1] = u.y;
    if constexpr (BYTES == 16) {
      w[2] = u.z;
      w[3] = u.w;
    }
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if constexpr (sizeof(T) == 2) {
        const float2 f = unpack_bf16x2(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      } else {
        x[i] = __uint_as_float(w[i]);
      }
    }
  }
  __device__ __forceinline__ void store(T* to) const {
    uint32_t w[WORDS];
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      if constexpr (sizeof(T) == 2) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
      else w[i] = __float_as_uint(x[i]);
    }
    if constexpr (BYTES == 16) *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
  }
};

template <typename T, int BYTES>
__global__ void __launch_bounds__(PA_THREADS) paged_append_kernel(const AppendParams a) {
  __shared__ float2 turn[PA_MAX_ANGLES];  // (cos, sin) of [token][pair]
  __shared__ int sequence_of[PA_MAX_TOKENS], position[PA_MAX_TOKENS];
  __shared__ long long slot[PA_MAX_TOKENS];  // the token's place in the cache, head 0; -1: none
  const PagedView& p = a.p;
  const int tid = threadIdx.x, row0 = blockIdx.x * a.tokens, count = min(a.tokens, p.tokens - row0);
  pdl_begin();
  if (tid < PA_MAX_TOKENS) sequence_of[tid] = p.first || row0 + tid >= p.sequences ? -1 : row0 + tid;
  __syncthreads();
  // Which sequences do the rows belong to: all are looked at at once, or, where they are many, found by halving.  The first block looks at all for
  // what cannot be.
  auto holds = [&](const PagedSequence& q, int s) {
    for (int r = max(row0, q.row0); r < min(row0 + count, q.row0 + q.n); ++r) sequence_of[r - row0] = s;
  };
  const bool halving = p.sequences > PA_LOOK;
  if (!halving || blockIdx.x == 0)
    for (int s = tid; s < p.sequences; s += PA_THREADS) {
      PagedSequence q;
      if (!paged_sequence(p, s, &q)) atomicExch(p.status + ST_BAD_INDEX, 1);
      else if (p.first && !halving) holds(q, s);
    }
  if (p.first && halving) {
    bool found = true;
    if (tid < count) {
      int low = 0, high = p.sequences;  // the last sequence that starts at the row or before it
      while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (p.first[mid] <= row0 + tid) low = mid;
        else high = mid;
      }
      PagedSequence q;
      found = paged_sequence(p, low, &q) && row0 + tid >= q.row0 && row0 + tid < q.row0 + q.n;
      if (found) sequence_of[tid] = low;
    }
    // Entries that cannot be mislead the search for rows of other sequences too, so a block that did not find all of its rows looks at all sequences.
    // Blocks of rows behind the last sequence do so as well: 1500 sequences of two rows and 3000 rows behind them 8.7 us, without this look 7.5; 20000 and 40000 98
    // and 54.
    if (__syncthreads_or(!found)) {
      constexpr int AT_ONCE = 8;  // loads on their way
      for (int s0 = tid; s0 < p.sequences; s0 += AT_ONCE * PA_THREADS) {
        int start[AT_ONCE], end[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          const int s = min(s0 + i * PA_THREADS, p.sequences - 1);
          start[i] = p.first[s];
          end[i] = p.first[s + 1];
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          const int s = s0 + i * PA_THREADS;
          PagedSequence q;
          if (s < p.sequences && start[i] < row0 + count && end[i] > row0 && paged_sequence(p, s, &q)) holds(q, s);
        }
      }
    }
  }
  __syncthreads();
  if (tid < count) {
    const int s = sequence_of[tid];
    long long where = -1;
    int t = -1;
    if (s >= 0) {
      PagedSequence q;
      if (paged_sequence(p, s, &q)) t = q.length - q.n + (row0 + tid - q.row0);
      else sequence_of[tid] = -1;  // without `first`
      if (t >= 0) {
        const int page = p.page_table[s * p.ld_table + (t >> p.page_shift)];
        if (page >= 0 && page < p.pages) where = page * p.page_stride + (t & (p.page_size - 1)) * p.position_stride;
        else atomicExch(p.status + ST_BAD_INDEX, 1);
      }
    }
    position[tid] = t;
    slot[tid] = where;
  }
  __syncthreads();
  for (int i = tid; i < count * a.pairs; i += PA_THREADS) {
    const int token = i / a.pairs, pair = i - token * a.pairs;
    double turns = (double)max(position[token], 0) * (double)a.frequencies[pair] * 0.15915494309189533577;  // of the circle
    turns -= rint(turns);
    const float near = (float)turns, rest = (float)(turns - (double)near) * 6.2831853f;  // 2^-23.3 of a radian at most
    float s, c;
    sincospif(2.0f * near, &s, &c);
    turn[i] = make_float2(fmaf(-s, rest, c), fmaf(c, rest, s));
  }
  __syncthreads();
  using Part = Piece<T, BYTES>;
  constexpr int N = Part::N;
  const int half = a.pairs;  // distance of a pair's channels where they do not stand side by side
  const int paired = a.interleaved ? 0 : half / N;  // units of a head that are two pieces, one `half` behind the other
  for (int i = tid; i < count * a.token_units; i += PA_THREADS) {
    const int token = a.by_token_units(i);
    int u = i - token * a.token_units;
    const bool is_q = u < a.q_units, is_k = !is_q && u < a.q_units + a.k_units;
    const long long where = slot[token];
    if (sequence_of[token] < 0 || (!is_q && where < 0)) continue;  // rows of no sequence, and tokens of no place, are left alone
    if (!is_q) u -= a.q_units;
    if (!is_q && !is_k) {  // values: pieces of a head, one after the other
      u -= a.k_units;
      const int head = u / (p.head_dim / N), c = (u - head * (p.head_dim / N)) * N;
      const T* from = static_cast<const T*>(a.v) + (long long)(row0 + token) * a.ld_v + head * p.head_dim + c;
      using Raw = typename Part::Raw;
      *reinterpret_cast<Raw*>(static_cast<T*>(p.v) + where + head * p.head_stride + c) = *reinterpret_cast<const Raw*>(from);
      continue;
    }
    const int head = a.by_units(u);
    u -= head * a.units;
    const T* from = (is_q ? static_cast<const T*>(a.q) + (long long)(row0 + token) * a.ld_q : static_cast<const T*>(a.k) + (long long)(row0 + token) * a.ld_k) +
                    head * p.head_dim;
    T* to = is_q ? static_cast<T*>(a.q_out) + (long long)(row0 + token) * a.ld_q_out + head * p.head_dim
                 : static_cast<T*>(p.k) + where + head * p.head_stride;
    const float2* w = turn + token * a.pairs;
    if (u < paired) {
      Part x, y;
      x.load(from + u * N);
      y.load(from + half + u * N);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float2 cs = w[u * N + j];
        const float xr = x.x[j] * cs.x - y.x[j] * cs.y, yr = x.x[j] * cs.y + y.x[j] * cs.x;
        x.x[j] = xr;
        y.x[j] = yr;
      }
      x.store(to + u * N);
      y.store(to + half + u * N);
    } else {
      const int c = (u + paired) * N;
      Part x;
      x.load(from + c);
      if (a.interleaved) {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
          const int pair = (c + j) / 2;
          if (pair >= a.pairs) break;
          const float2 cs = w[pair];
          const float xr = x.x[j] * cs.x - x.x[j + 1] * cs.y, yr = x.x[j] * cs.y + x.x[j + 1] * cs.x;
          x.x[j] = xr;
          x.x[j + 1] = yr;
        }
      }
      x.store(to + c);
    }
  }
}

template <typename T, int BYTES>
int append(hl_ctx* ctx, AppendParams& a) {
  constexpr int N = Piece<T, BYTES>::N;
  const PagedView& p = a.p;
  a.units = p.head_dim / N - (a.interleaved ? 0 : a.pairs / N);
  a.q_units = a.heads * a.units;
  a.k_units = p.kv_heads * a.units;
  a.token_units = a.q_units + a.k_units + p.kv_heads * (p.head_dim / N);
  a.by_token_units = QuickDiv((uint32_t)a.token_units);
  a.by_units = QuickDiv((uint32_t)a.units);
  a.tokens = 1;
  while (a.tokens < PA_MAX_TOKENS && 2 * a.tokens * a.pairs <= PA_MAX_ANGLES && ceil_div(p.tokens, 2 * a.tokens) >= 8 * ctx->sm_count) a.tokens *= 2;
  pdl(paged_append_kernel<T, BYTES>, ceil_div(p.tokens, a.tokens), PA_THREADS, 0, ctx->stream)
      .streaming(2.0 * p.tokens * a.token_units * (double)BYTES)(a);
  HL_LAUNCH_CHECK("paged_append_kernel");
  count_launch(ctx);
  return HL_OK;
}

}  // namespace
}  // namespace hl

extern "C" int hl_paged_append(hl_ctx* ctx, const hl_paged_cache* cache, const hl_paged_batch* batch, const void* q, long long ld_q, void* q_out,
                               long long ld_q_out, int heads, const void* k, long long ld_k, const void* v, long long ld_v,
                               const float* frequencies, int rotary_dim, int interleaved) {
  using namespace hl;
  AppendParams a{};
  int rc = paged_view(ctx, "hl_paged_append", cache, batch, &a.p);
  if (rc != HL_OK) return rc;
  const long long step = cache->dtype == HL_BF16 ? 8 : 4, dim = cache->head_dim;
  HL_REQUIRE(k && v && (!q) == (!q_out), "hl_paged_append: null argument");
  HL_REQUIRE(q ? heads > 0 : heads == 0, "hl_paged_append: heads goes with q");
  HL_REQUIRE(rotary_dim >= 0 && rotary_dim <= dim && rotary_dim % 2 == 0, "hl_paged_append: rotary_dim must be even and at most head_dim");
  HL_REQUIRE(rotary_dim == 0 || frequencies, "hl_paged_append: rotary_dim without frequencies");
  HL_REQUIRE(interleaved || (rotary_dim / 2) % (step / 2) == 0, "hl_paged_append: halves of rotary_dim must be multiples of 8 bytes");
  HL_REQUIRE(ld_k >= cache->kv_heads * dim && ld_v >= cache->kv_heads * dim && (!q || (ld_q >= heads * dim && ld_q_out >= heads * dim)),
             "hl_paged_append: row strides must cover all heads");
  HL_REQUIRE(ld_k % step == 0 && ld_v % step == 0 && (!q || (ld_q % step == 0 && ld_q_out % step == 0)),
             "hl_paged_append: row strides must be multiples of 16 bytes");
  HL_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k) |
               reinterpret_cast<uintptr_t>(v)) & 15) == 0,
             "hl_paged_append: pointers must be 16-byte aligned");
  // a token's pieces are counted in 31 bits
  HL_REQUIRE(((long long)heads + 2ll * cache->kv_heads) * dim <= (1ll << 24), "hl_paged_append: too many heads");
  a.q = q; a.k = k; a.v = v; a.q_out = q_out;
  a.ld_q = ld_q; a.ld_k = ld_k; a.ld_v = ld_v; a.ld_q_out = ld_q_out;
  a.frequencies = frequencies;
  a.pairs = rotary_dim / 2;
  a.interleaved = interleaved ? 1 : 0;
  a.heads = heads;
  OnDevice here(ctx->device);
  ProfileScope prof(ctx, HL_PROF_OTHER, 2.0 * a.p.tokens * (heads + 2.0 * cache->kv_heads) * (double)dim * (double)dtype_size(cache->dtype));
  // Halves that end within 16 bytes are walked over in pieces of 8, so that a thread has both channels of its pairs.
  if (!interleaved && a.pairs % step != 0) return cache->dtype == HL_BF16 ? append<__nv_bfloat16, 8>(ctx, a) : append<float, 8>(ctx, a);
  return cache->dtype == HL_BF16 ? append<__nv_bfloat16, 16>(ctx, a) : append<float, 16>(ctx, a);
}
