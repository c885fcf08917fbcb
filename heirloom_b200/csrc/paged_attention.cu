// Attention of new tokens over a paged cache: the entry point, the kernel that takes every type and head size, and the one that joins
// pieces.
//
// Token i of the n new ones of a sequence of `length` positions sees the positions j <= length - n + i:
//   out = sum_j softmax_j(scale q . k_j) v_j,  lse = log sum_j exp(scale q . k_j)
// in one pass over the keys, with the running maximum and sum of each row in f32.  Rows that stand at no position (length < n) see
// nothing: zeros and an lse of minus infinity.
//
// Which kernel: bf16 heads of 64 and 128 channels take the tensor cores, with sixteen rows or fewer a key head (one-token steps) in a kernel of
// their own: 64 sequences of one token, 4 rows a key head, 152 us there and 189 in blocks of 128 rows.  Everything else takes the kernel here, which is not made for
// size: with 32 heads of 96 on 8 in bf16 64 steps over up to 8192 positions take 457 us (108 by bytes), a chunk of 2048 tokens over 4096 positions 4.2 ms (46 by products).
#include "paged_attention.cuh"

namespace hl {
namespace {

// ---- any type and head size: f32 arithmetic, 32 keys and 16 rows at a time --------------------------------------------------------
// Q as f32, keys and values as they are, in shared memory; two tiles, one of which is on its way while the other is worked on.  A warp has four
// rows: a lane a key for the scores, a lane four or eight channels for the values, so that warps meet only where a tile comes and goes.  Bound by shared
// memory (two reads of 16 bytes a lane for sixteen multiply-adds) and, for few tiles, by the first run through the code: it is kept short (nine
// sequences of up to 40 tokens and 700 positions, 6 heads of 80 in f32: 29 us; 73 with a thread a channel of all rows and tiles loaded when they were needed).
constexpr int PR_ROWS = 16, PR_KEYS = 32, PR_WARPS = 4, PR_THREADS = PR_WARPS * 32, PR_OWN = PR_ROWS / PR_WARPS;
constexpr int PR_MAX_DIM = 256;
// Up to that many positions a sequence is not shared out.  Its item then takes as long as 16 tiles of 64 keys, about what joining pieces costs.  One-token steps of 12
// heads of 64, whole and by the even deal: 1 or 8 sequences of up to 1024 positions 12 us and 14, 64 36 and 36 (all of 1024: 46 and 52), 200 91 and 85, 800 334 and 296; up
// to 256 positions 5 and 13, 13 and 18, 35 and 40, 137 and 140; up to 2048 positions 20 and 14 (1 or 8), 59 and 52 (64), 154 and 140 (200).
constexpr int STEP_WHOLE = 1024;
template <typename T>
__host__ __device__ constexpr int rows_pitch(int head_dim) { return head_dim * (int)sizeof(T) + 16; }  // bytes from key to key
template <typename T>
size_t rows_shared(int head_dim) { return sizeof(float) * (size_t)(PR_ROWS * head_dim) + 4 * (size_t)PR_KEYS * rows_pitch<T>(head_dim); }

template <typename T>
__device__ __forceinline__ float4 four(const void* at) {
  if constexpr (sizeof(T) == 2) {
    const uint2 u = *static_cast<const uint2*>(at);
    const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y);
    return make_float4(a.x, a.y, b.x, b.y);
  } else {
    return *static_cast<const float4*>(at);
  }
}
template <typename T>
__device__ __forceinline__ void store_four(T* to, float4 x) {
  if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w));
  else *reinterpret_cast<float4*>(to) = x;
}
__device__ __forceinline__ void add_scaled(float4& acc, float4 x, float f) {
  acc.x = fmaf(x.x, f, acc.x);
  acc.y = fmaf(x.y, f, acc.y);
  acc.z = fmaf(x.z, f, acc.z);
  acc.w = fmaf(x.w, f, acc.w);
}
__device__ __forceinline__ float4 scaled(float4 x, float f) { return make_float4(x.x * f, x.y * f, x.z * f, x.w * f); }

template <typename T>
__global__ void __launch_bounds__(PR_THREADS) paged_attention_rows_kernel(const PagedAttention a) {
  extern __shared__ __align__(16) uint8_t pr_smem[];
  __shared__ long long deal_shared[68];
  __shared__ __align__(16) float probability[PR_ROWS][PR_KEYS];
  const PagedView& p = a.p;
  const int D = p.head_dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = a.z.group;
  const int pitch = rows_pitch<T>(D), tile_bytes = PR_KEYS * pitch;
  float* sq = reinterpret_cast<float*>(pr_smem) + warp * PR_OWN * D;  // the warp's rows
  uint8_t* tiles = pr_smem + sizeof(float) * PR_ROWS * D;              // [2] keys, values
  constexpr int N = 16 / (int)sizeof(T);
  pdl_begin();
  if (blockIdx.x == 0)
    for (int s = tid; s < p.sequences; s += PR_THREADS) {
      PagedSequence q;
      if (!paged_sequence(p, s, &q)) atomicExch(p.status + ST_BAD_INDEX, 1);
    }
  Deal deal;
  DealPlace place;
  const int stream = blockIdx.x;
  deal_start<PR_THREADS>(p, a.z, stream, deal_shared, &deal, &place);
  const long long from = deal.chunk * stream, until = min(deal.total, from + deal.chunk);
  Joint joint{};
  for (DealItem it = deal_item(p, a.z, place, from, until); deal_valid(it); deal_next(p, a.z, it)) {
    if (deal_goes_on(it)) joint = deal_joint(a.z, deal, it, stream);
    const int row0 = it.block * PR_ROWS + warp * PR_OWN, rows = min(PR_OWN, it.q.n * group - row0);  // of this warp
    const int total_keys = deal_keys(a.z, it.blocks, it.block);
    // A tile on its way: a warp has eight keys, four lanes a key.  Behind the keys that are seen the cache may hold anything: zeros.
    auto fetch = [&](int tile) {
      const int j = tid >> 2, t = tile * PR_KEYS + j;
      long long where = -1;
      if (t < total_keys) {
        const int page = p.page_table[it.s * p.ld_table + (t >> p.page_shift)];
        if (page >= 0 && page < p.pages) where = page * p.page_stride + (t & (p.page_size - 1)) * p.position_stride + it.head * p.head_stride;
        else atomicExch(p.status + ST_BAD_INDEX, 1);
      }
      const int bytes = where >= 0 ? 16 : 0;
      const T *k = static_cast<const T*>(p.k) + max(where, 0ll), *v = static_cast<const T*>(p.v) + max(where, 0ll);
      const uint32_t to = (uint32_t)__cvta_generic_to_shared(tiles + (tile & 1) * 2 * tile_bytes + j * pitch);
      for (int c = lane & 3; c < D / N; c += 4) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + c * 16), "l"(k + c * N), "r"(bytes) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + c * 16 + (uint32_t)tile_bytes), "l"(v + c * N), "r"(bytes) : "memory");
      }
    };
    __syncthreads();  // the last item's tiles have been read
    fetch(it.tile0);
    asm volatile("cp.async.commit_group;" ::: "memory");
    // the rows' tokens, heads and keys, lane by lane
    const int row = row0 + lane, token = a.z.by_group(row), head = it.head * group + row - token * group;
    const int sees = lane < rows ? it.q.length - it.q.n + token + 1 : 0;
    for (int r = 0; r < rows; ++r) {
      const long long at = (it.q.row0 + __shfl_sync(0xffffffffu, token, r)) * a.ld_q + __shfl_sync(0xffffffffu, head, r) * D;
      for (int c = lane * 4; c < D; c += 128) *reinterpret_cast<float4*>(sq + r * D + c) = four<T>(static_cast<const T*>(a.q) + at + c);
    }
    __syncwarp();
    float4 acc[PR_OWN][2] = {};
    float m[PR_OWN], l[PR_OWN];
#pragma unroll
    for (int r = 0; r < PR_OWN; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.0f;
    }
#pragma unroll 1
    for (int tile = it.tile0; tile < it.tile1; ++tile) {
      if (tile + 1 < it.tile1) fetch(tile + 1);
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();  // everybody's copies of this tile
      if (rows > 0) {
        const uint8_t* sk = tiles + (tile & 1) * 2 * tile_bytes + lane * pitch;
        float s[PR_OWN] = {};
#pragma unroll 2
        for (int d = 0; d < D; d += 4) {
          const float4 k4 = four<T>(sk + d * sizeof(T));
#pragma unroll
          for (int r = 0; r < PR_OWN; ++r) {  // rows that there are not: what stands there reaches nobody
            const float4 q4 = *reinterpret_cast<const float4*>(sq + r * D + d);
            s[r] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[r]))));
          }
        }
#pragma unroll
        for (int r = 0; r < PR_OWN; ++r) {
          const float x = tile * PR_KEYS + lane < __shfl_sync(0xffffffffu, sees, r) ? s[r] * a.scale_log2 : -INFINITY;
          // what is not a number stays so: it reaches no maximum, but the sums
          const float top = fmaxf(m[r], warp_max(x)), f = piece_factor(m[r], top), pr = x == -INFINITY ? 0.0f : exp2f(x - top);
          m[r] = top;
          l[r] = l[r] * f + warp_sum(pr);
          acc[r][0] = scaled(acc[r][0], f);
          acc[r][1] = scaled(acc[r][1], f);
          probability[warp * PR_OWN + r][lane] = pr;
        }
        __syncwarp();
        const uint8_t* sv = tiles + (tile & 1) * 2 * tile_bytes + tile_bytes + lane * 4 * sizeof(T);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (lane * 4 + h * 128 < D) {
#pragma unroll 1
            for (int j = 0; j < PR_KEYS; j += 4) {
              float4 v[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) v[i] = four<T>(sv + (j + i) * pitch + h * 128 * sizeof(T));
#pragma unroll
              for (int r = 0; r < PR_OWN; ++r) {
                const float4 w = *reinterpret_cast<const float4*>(&probability[warp * PR_OWN + r][j]);
                add_scaled(acc[r][h], v[0], w.x);
                add_scaled(acc[r][h], v[1], w.y);
                add_scaled(acc[r][h], v[2], w.z);
                add_scaled(acc[r][h], v[3], w.w);
              }
            }
          }
        }
      }
      __syncthreads();  // the tile's place is filled again
    }
    const bool whole = deal_whole(it);
    float* piece = a.pieces + (size_t)(stream * 2 + deal_piece(it)) * piece_floats(PR_ROWS, D);
#pragma unroll
    for (int r = 0; r < PR_OWN; ++r) {
      const long long of = it.q.row0 + __shfl_sync(0xffffffffu, token, r);
      const int h = __shfl_sync(0xffffffffu, head, r), in_block = warp * PR_OWN + r;
      if (r >= rows) break;
      const float inv = l[r] > 0.0f || l[r] != l[r] ? 1.0f / l[r] : 0.0f;
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        const int c = lane * 4 + part * 128;
        if (c < D) {
          if (whole) store_four(static_cast<T*>(a.out) + of * a.ld_out + h * D + c, scaled(acc[r][part], inv));
          else *reinterpret_cast<float4*>(piece + piece_at(PR_ROWS, in_block, c)) = acc[r][part];
        }
      }
      if (lane == 0) {
        if (!whole) {
          piece[PR_ROWS * D + in_block] = m[r];
          piece[PR_ROWS * (D + 1) + in_block] = l[r];
        } else if (a.lse) {
          a.lse[of * a.heads + h] = (m[r] + log2f(l[r])) * 0.6931471805599453f;
        }
      }
    }
  }
  if (tid == 0) a.joints[stream] = joint;
}

// ---- pieces joined ----------------------------------------------------------------------------------------------------------------
// Block x looks after the item that stream x starts and others go on with, block y after some of its rows.  The pieces are added in an order of
// their own, not in that in which the streams finished.  Bound by latency: what a block reads it asks for in two round trips behind the joint's.
struct Pieces {  // of an item, stream by stream: the first stream's is the one of the item it ends in, the others' the one of the item they start in
  const float *first, *later;
  size_t step;
  __device__ __forceinline__ Pieces(const PagedAttention& a, int rows)
      : first(a.pieces + ((size_t)blockIdx.x * 2 + 1) * piece_floats(rows, a.p.head_dim)),
        later(a.pieces + ((size_t)blockIdx.x + 1) * 2 * piece_floats(rows, a.p.head_dim)),
        step(2 * piece_floats(rows, a.p.head_dim)) {}
  __device__ __forceinline__ const float* operator[](int i) const { return i == 0 ? first : later + (size_t)(i - 1) * step; }
};
struct RowPlace {
  long long token;
  int head;
  __device__ __forceinline__ RowPlace(const PagedAttention& a, const Joint& j, int r) {
    const int row = j.block_row + r, t = a.z.by_group(row);
    token = j.row0 + t;
    head = j.head * a.z.group + row - t * a.z.group;
  }
};
__device__ __forceinline__ float row_lse(float m, float sum) { return (m + log2f(sum)) * 0.6931471805599453f; }
__device__ __forceinline__ float row_inverse(float sum) { return sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f; }

// Blocks of 128 rows in bf16, of which a piece is long and pieces are few: a lane a row, a warp sixteen channels.
constexpr int JR_ROWS = 32, JR_CHANNELS = 16;
__global__ void paged_attention_join_rows_kernel(const PagedAttention a) {
  const int D = a.p.head_dim, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rows = a.z.rows(), r = blockIdx.y * JR_ROWS + lane;
  pdl_begin();
  const Joint j = a.joints[blockIdx.x];
  if (j.streams == 0 || r >= j.count) return;
  const Pieces piece(a, rows);
  float m = -INFINITY, sum = 0.0f;
  float4 acc[4] = {};
  for (int i = 0; i < j.streams; ++i) {
    const float* x = piece[i];
    const float pm = x[rows * D + r], pl = x[rows * (D + 1) + r];
    float4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const float4*>(x + piece_at(rows, r, warp * JR_CHANNELS + u * 4));
    const float top = fmaxf(m, pm), old = piece_factor(m, top), f = piece_factor(pm, top);
    m = top;
    sum = sum * old + pl * f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      acc[u] = scaled(acc[u], old);
      add_scaled(acc[u], v[u], f);
    }
  }
  const RowPlace at(a, j, r);
  const float inv = row_inverse(sum);
  __nv_bfloat16* to = static_cast<__nv_bfloat16*>(a.out) + at.token * a.ld_out + at.head * D + warp * JR_CHANNELS;
#pragma unroll
  for (int u = 0; u < 4; ++u) store_four(to + u * 4, scaled(acc[u], inv));
  if (a.lse && warp == 0) a.lse[at.token * a.heads + at.head] = row_lse(m, sum);
}

// Blocks of sixteen rows, of which there may be many pieces: four rows a block, a warp every eighth piece.
constexpr int JP_WARPS = 8, JP_ROWS = 4;
template <typename T>
__global__ void __launch_bounds__(JP_WARPS * 32) paged_attention_join_pieces_kernel(const PagedAttention a) {
  __shared__ __align__(16) float sums[JP_WARPS][JP_ROWS][PR_MAX_DIM];
  const int D = a.p.head_dim, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rows = a.z.rows(), r0 = blockIdx.y * JP_ROWS;
  pdl_begin();
  const Joint j = a.joints[blockIdx.x];
  if (j.streams == 0 || r0 >= j.count) return;
  const int count = min(JP_ROWS, j.count - r0);
  const Pieces piece(a, rows);
  // Lane by lane the pieces' statistics (rows that there are not hold anything, and reach nobody), every warp all of them.
  float m[JP_ROWS], sum[JP_ROWS];
  float4 acc[JP_ROWS][2] = {};
#pragma unroll
  for (int r = 0; r < JP_ROWS; ++r) {
    m[r] = -INFINITY;
    sum[r] = 0.0f;
  }
#pragma unroll 1
  for (int i0 = 0; i0 < j.streams; i0 += 32) {
    const int n = min(32, j.streams - i0);
    float4 pm = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY), pl = make_float4(0.f, 0.f, 0.f, 0.f);
    if (lane < n) {
      pm = *reinterpret_cast<const float4*>(piece[i0 + lane] + rows * D + r0);
      pl = *reinterpret_cast<const float4*>(piece[i0 + lane] + rows * (D + 1) + r0);
    }
    float f[JP_ROWS];
#pragma unroll
    for (int r = 0; r < JP_ROWS; ++r) {
      const float mine = r == 0 ? pm.x : r == 1 ? pm.y : r == 2 ? pm.z : pm.w, weight = r == 0 ? pl.x : r == 1 ? pl.y : r == 2 ? pl.z : pl.w;
      const float top = fmaxf(m[r], warp_max(mine)), old = piece_factor(m[r], top);
      f[r] = piece_factor(mine, top);
      sum[r] = sum[r] * old + warp_sum(weight * f[r]);
      m[r] = top;
      acc[r][0] = scaled(acc[r][0], old);
      acc[r][1] = scaled(acc[r][1], old);
    }
#pragma unroll 4
    for (int i = warp; i < n; i += JP_WARPS) {
#pragma unroll
      for (int r = 0; r < JP_ROWS; ++r) {
        const float w = __shfl_sync(0xffffffffu, f[r], i);
        if (r < count) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (lane * 4 + h * 128 < D) add_scaled(acc[r][h], *reinterpret_cast<const float4*>(piece[i0 + i] + piece_at(rows, r0 + r, lane * 4 + h * 128)), w);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < JP_ROWS; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (lane * 4 + h * 128 < D) *reinterpret_cast<float4*>(&sums[warp][r][lane * 4 + h * 128]) = acc[r][h];
  __syncthreads();
  if (warp >= count) return;  // a warp a row
  const RowPlace at(a, j, r0 + warp);
  float my_m = m[0], my_sum = sum[0];
#pragma unroll
  for (int r = 1; r < JP_ROWS; ++r)
    if (warp == r) {
      my_m = m[r];
      my_sum = sum[r];
    }
  const float inv = row_inverse(my_sum);
  for (int c = lane * 4; c < D; c += 128) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < JP_WARPS; ++w) add_scaled(x, *reinterpret_cast<const float4*>(&sums[w][warp][c]), 1.0f);
    store_four(static_cast<T*>(a.out) + at.token * a.ld_out + at.head * D + c, scaled(x, inv));
  }
  if (a.lse && lane == 0) a.lse[at.token * a.heads + at.head] = row_lse(my_m, my_sum);
}

// How a call is cut.  From what the host knows alone: a captured call has other lengths every time.
enum class Kernel { rows, tensor_cores, step, whole_step };
struct Route {
  DealShape z;
  Kernel kernel;
};
Route route(const hl_ctx* ctx, int dtype, int head_dim, int group, int max_new, int max_length) {
  Route r{};
  if (dtype == HL_BF16 && (head_dim == 64 || head_dim == 128)) {
    if ((long long)max_new * group <= STEP_ROWS) {
      r.kernel = max_length <= STEP_WHOLE ? Kernel::whole_step : Kernel::step;
      r.z = paged_attention_step_shape(ctx->sm_count, group);
    } else {
      r.kernel = Kernel::tensor_cores;
      r.z = paged_attention_tc_shape(ctx->sm_count, group);
    }
  } else {
    const int shared = (int)(dtype == HL_BF16 ? rows_shared<__nv_bfloat16>(head_dim) : rows_shared<float>(head_dim));
    const int streams = ctx->sm_count * std::max(1, std::min(8, 220 * 1024 / (shared + 4096)));
    r.kernel = Kernel::rows;
    r.z = deal_shape(4, 5, group, streams, 2, 1);
    static_assert(PR_ROWS == 1 << 4 && PR_KEYS == 1 << 5, "the shifts above");
  }
  return r;
}
template <typename T>
int rows_kernel(hl_ctx* ctx, const PagedAttention& a) {
  HL_ALLOW_SHARED(ctx, rows_shared<T>(PR_MAX_DIM), paged_attention_rows_kernel<T>);
  pdl(paged_attention_rows_kernel<T>, a.z.streams, PR_THREADS, rows_shared<T>(a.p.head_dim), ctx->stream)(a);
  HL_LAUNCH_CHECK("paged_attention_rows_kernel");
  return HL_OK;
}
size_t workspace_bytes(const Route& r, int head_dim) {
  return (size_t)r.z.streams * (sizeof(Joint) + 2 * piece_floats(r.z.rows(), head_dim) * sizeof(float));
}

}  // namespace
}  // namespace hl

extern "C" int hl_paged_attention_workspace(hl_ctx* ctx, int dtype, int heads, int kv_heads, int head_dim, size_t* bytes) {
  using namespace hl;
  HL_REQUIRE(ctx && bytes, "hl_paged_attention_workspace: null argument");
  HL_REQUIRE(dtype == HL_BF16 || dtype == HL_F32, "hl_paged_attention_workspace: the cache holds bf16 or f32");
  HL_REQUIRE(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, "hl_paged_attention_workspace: heads must be a multiple of kv_heads");
  HL_REQUIRE(head_dim >= 8 && head_dim <= 256 && head_dim % 8 == 0, "hl_paged_attention_workspace: head_dim must be a multiple of 8 up to 256");
  *bytes = 0;  // of any number of new tokens
  for (int max_new : {1, 1 << 20}) *bytes = std::max(*bytes, workspace_bytes(route(ctx, dtype, head_dim, heads / kv_heads, max_new, 1 << 30), head_dim));
  return HL_OK;
}

extern "C" int hl_paged_attention(hl_ctx* ctx, const hl_paged_cache* cache, const hl_paged_batch* batch, const void* q, long long ld_q, void* out,
                                  long long ld_out, float* lse, int heads, float scale, void* workspace, size_t workspace_size) {
  using namespace hl;
  PagedAttention a{};
  int rc = paged_view(ctx, "hl_paged_attention", cache, batch, &a.p);
  if (rc != HL_OK) return rc;
  const int dim = cache->head_dim, kv_heads = cache->kv_heads;
  HL_REQUIRE(q && out && workspace, "hl_paged_attention: null argument");
  HL_REQUIRE(heads > 0 && heads % kv_heads == 0, "hl_paged_attention: heads must be a multiple of kv_heads");
  HL_REQUIRE(scale > 0.0f && scale < INFINITY, "hl_paged_attention: scale must be positive");
  const long long step = cache->dtype == HL_BF16 ? 8 : 4, wide = (long long)heads * dim;
  HL_REQUIRE(ld_q >= wide && ld_out >= wide && ld_q % step == 0 && ld_out % step == 0,
             "hl_paged_attention: row strides must be multiples of 16 bytes and cover all heads");
  HL_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15) == 0,
             "hl_paged_attention: pointers must be 16-byte aligned");
  const int group = heads / kv_heads;
  // rows and keys of a sequence, times the query heads of a key head, are counted in 31 bits
  HL_REQUIRE((long long)group * (std::max(a.p.max_length, a.p.max_new) + 1024ll) < 0x7fffffffll, "hl_paged_attention: sequences are too long for so many heads");
  HL_REQUIRE((long long)a.p.sequences * kv_heads < 0x7fff0000ll, "hl_paged_attention: too many sequences");  // a walk steps once beyond the last
  HL_REQUIRE(wide < 0x7fffffffll, "hl_paged_attention: too many heads");                                     // a row's channels in 31 bits
  const Route r = route(ctx, cache->dtype, dim, group, a.p.max_new, a.p.max_length);
  size_t wanted = 0;
  if ((rc = hl_paged_attention_workspace(ctx, cache->dtype, heads, kv_heads, dim, &wanted)) != HL_OK) return rc;
  HL_REQUIRE(workspace_size >= wanted, "hl_paged_attention: the workspace is smaller than hl_paged_attention_workspace says");
  a.z = r.z;
  a.q = q; a.ld_q = ld_q;
  a.out = out; a.ld_out = ld_out;
  a.lse = lse;
  a.joints = static_cast<Joint*>(workspace);
  a.pieces = reinterpret_cast<float*>(a.joints + r.z.streams);
  a.heads = heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  OnDevice here(ctx->device);
  // bytes that the host knows of; how many keys there are stands on the device, so flops are not known
  ProfileScope prof(ctx, HL_PROF_OTHER, (double)a.p.tokens * heads * (2.0 * dim * (double)dtype_size(cache->dtype) + (lse ? 4.0 : 0.0)));
  switch (r.kernel) {
    case Kernel::rows: rc = cache->dtype == HL_BF16 ? rows_kernel<__nv_bfloat16>(ctx, a) : rows_kernel<float>(ctx, a); break;
    case Kernel::tensor_cores: rc = paged_attention_tc(ctx, a); break;
    case Kernel::step:
    case Kernel::whole_step: rc = paged_attention_step(ctx, a, r.kernel == Kernel::whole_step); break;
  }
  if (rc != HL_OK) return rc;
  count_launch(ctx);
  ctx->counters.attention_launches += 1;
  if (r.kernel == Kernel::whole_step) return HL_OK;
  if (r.kernel == Kernel::tensor_cores) {
    pdl(paged_attention_join_rows_kernel, dim3(r.z.streams, r.z.rows() / JR_ROWS), dim / JR_CHANNELS * 32, 0, ctx->stream)(a);
  } else {
    const dim3 joins(r.z.streams, r.z.rows() / JP_ROWS);
    if (cache->dtype == HL_BF16) pdl(paged_attention_join_pieces_kernel<__nv_bfloat16>, joins, JP_WARPS * 32, 0, ctx->stream)(a);
    else pdl(paged_attention_join_pieces_kernel<float>, joins, JP_WARPS * 32, 0, ctx->stream)(a);
  }
  HL_LAUNCH_CHECK("paged_attention_join_kernel");
  count_launch(ctx);
  return HL_OK;
}
