// Attention of new tokens over a paged cache: the entry point, the kernel that takes every type and head size, and the one that joins
// pieces.
//
// Token i of the n new ones of a sequence of `length` positions sees the positions j <= length - n + i:
//   out = sum_j softmax_j(scale q . k_j) v_j,  lse = log sum_j exp(scale q . k_j)
// in one pass over the keys, with the running maximum and sum of each row in f32.  Rows that stand at no position (length < n) see
// nothing: zeros and an lse of minus infinity.
#include "paged_attention.cuh"

namespace hl {
namespace {

// ---- any type and head size: f32 arithmetic, 32 keys and 16 rows at a time --------------------------------------------------------
// Q, K and V as f32 in shared memory (rows of K four words apart from a multiple of eight, so that 32 lanes that read 16 bytes of 32 rows
// touch all banks); a warp has four rows and a lane a key for the scores, a thread one or two channels of all rows for the values.
constexpr int PR_ROWS = 16, PR_KEYS = 32, PR_THREADS = 128;
constexpr int PR_MAX_DIM = 256;
constexpr int STEP_WHOLE = 1024;
size_t rows_shared(int head_dim) { return sizeof(float) * (size_t)(PR_ROWS * head_dim + PR_KEYS * (head_dim + 4) + PR_KEYS * head_dim); }

template <typename T>
__device__ __forceinline__ void load_piece(const T* from, float* to) {  // 16 bytes
  const uint4 u = *reinterpret_cast<const uint4*>(from);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      const float2 f = unpack_bf16x2(w[i]);
      to[2 * i] = f.x;
      to[2 * i + 1] = f.y;
    } else {
      to[i] = __uint_as_float(w[i]);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(PR_THREADS) paged_attention_rows_kernel(const PagedAttention a) {
  extern __shared__ __align__(16) float pr_smem[];
  __shared__ long long deal_shared[68];
  __shared__ __align__(16) float probability[PR_ROWS][PR_KEYS];
  __shared__ float factor[PR_ROWS], row_max[PR_ROWS], row_sum[PR_ROWS];
  __shared__ int row_keys[PR_ROWS];  // keys that the row sees
  const PagedView& p = a.p;
  const int D = p.head_dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float* sq = pr_smem;
  float* sk = sq + PR_ROWS * D;
  float* sv = sk + PR_KEYS * (D + 4);
  constexpr int N = 16 / (int)sizeof(T);
  const int vectors = D / N;
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
    const int group = a.z.group, row0 = it.block * PR_ROWS, rows = min(PR_ROWS, it.q.n * group - row0);
    const int total_keys = deal_keys(a.z, it.blocks, it.block);
    __syncthreads();  // the last item's shared memory has been read
    for (int i = tid; i < PR_ROWS * vectors; i += PR_THREADS) {
      const int r = i / vectors, c = (i - r * vectors) * N, row = row0 + r;
      float x[N] = {};
      if (r < rows)
        load_piece(static_cast<const T*>(a.q) + (long long)(it.q.row0 + a.z.by_group(row)) * a.ld_q + (it.head * group + (row - a.z.by_group(row) * group)) * D + c, x);
#pragma unroll
      for (int j = 0; j < N; ++j) sq[r * D + c + j] = x[j];
    }
    if (tid < PR_ROWS) {
      row_max[tid] = -INFINITY;
      row_sum[tid] = 0.0f;
      row_keys[tid] = tid < rows ? it.q.length - it.q.n + a.z.by_group(row0 + tid) + 1 : 0;
    }
    float acc[PR_ROWS][2] = {};
    for (int tile = it.tile0; tile < it.tile1; ++tile) {
      const int key0 = tile * PR_KEYS;
      __syncthreads();
      for (int i = tid; i < PR_KEYS * vectors; i += PR_THREADS) {
        const int j = i / vectors, c = (i - j * vectors) * N, t = key0 + j;
        float kx[N] = {}, vx[N] = {};
        if (t < total_keys) {  // behind them the cache may hold anything
          const int page = p.page_table[it.s * p.ld_table + (t >> p.page_shift)];
          if (page >= 0 && page < p.pages) {
            const long long where = page * p.page_stride + (t & (p.page_size - 1)) * p.position_stride + it.head * p.head_stride + c;
            load_piece(static_cast<const T*>(p.k) + where, kx);
            load_piece(static_cast<const T*>(p.v) + where, vx);
          } else {
            atomicExch(p.status + ST_BAD_INDEX, 1);
          }
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
          sk[j * (D + 4) + c + e] = kx[e];
          sv[j * D + c + e] = vx[e];
        }
      }
      __syncthreads();
      if (warp * 4 < rows) {
        float s[4] = {};
        for (int d = 0; d < D; d += 4) {
          const float4 k4 = *reinterpret_cast<const float4*>(sk + lane * (D + 4) + d);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float4 q4 = *reinterpret_cast<const float4*>(sq + (warp * 4 + r) * D + d);
            s[r] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[r]))));
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = warp * 4 + r;
          const float x = key0 + lane < row_keys[row] ? s[r] * a.scale_log2 : -INFINITY;
          const float before = row_max[row], m = fmaxf(before, warp_max(x));
          const float pr = m == -INFINITY ? 0.0f : exp2f(x - m);
          const float f = piece_factor(before, m), sum = warp_sum(pr);
          probability[row][lane] = pr;
          __syncwarp();  // all lanes have read the row's maximum
          if (lane == 0) {
            factor[row] = f;
            row_max[row] = m;
            row_sum[row] = row_sum[row] * f + sum;
          }
        }
      }
      __syncthreads();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = tid + h * PR_THREADS;
        if (c < D) {
#pragma unroll
          for (int r = 0; r < PR_ROWS; ++r)
            if (r < rows) acc[r][h] *= factor[r];
#pragma unroll 1
          for (int j = 0; j < PR_KEYS; j += 4) {
            const float v0 = sv[j * D + c], v1 = sv[(j + 1) * D + c], v2 = sv[(j + 2) * D + c], v3 = sv[(j + 3) * D + c];
#pragma unroll
            for (int r = 0; r < PR_ROWS; ++r)
              if (r < rows) {
                const float4 w = *reinterpret_cast<const float4*>(&probability[r][j]);
                acc[r][h] = fmaf(w.x, v0, fmaf(w.y, v1, fmaf(w.z, v2, fmaf(w.w, v3, acc[r][h]))));
              }
          }
        }
      }
    }
    if (deal_whole(it)) {
#pragma unroll
      for (int r = 0; r < PR_ROWS; ++r)
        if (r < rows) {
          const int row = row0 + r, head = it.head * group + (row - a.z.by_group(row) * group);
          const long long token = it.q.row0 + a.z.by_group(row);
          const float sum = row_sum[r], inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int c = tid + h * PR_THREADS;
            if (c < D) {
              T* to = static_cast<T*>(a.out) + token * a.ld_out + head * D + c;
              if constexpr (sizeof(T) == 2) *to = to_bf16(acc[r][h] * inv);
              else *to = acc[r][h] * inv;
            }
          }
          if (a.lse && tid == 0) a.lse[token * a.heads + head] = (row_max[r] + log2f(sum)) * 0.6931471805599453f;
        }
    } else {
      float* piece = a.pieces + (size_t)(stream * 2 + deal_piece(it)) * piece_floats(PR_ROWS, D);
#pragma unroll
      for (int r = 0; r < PR_ROWS; ++r)
        if (r < rows) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (tid + h * PR_THREADS < D) piece[piece_at(PR_ROWS, r, tid + h * PR_THREADS)] = acc[r][h];
        }
      if (tid < rows) {
        piece[PR_ROWS * D + tid] = row_max[tid];
        piece[PR_ROWS * (D + 1) + tid] = row_sum[tid];
      }
    }
  }
  if (tid == 0) a.joints[stream] = joint;
}

// ---- pieces joined ----------------------------------------------------------------------------------------------------------------
// Block x looks after the item that stream x starts and others go on with, block y after eight of its rows.  The pieces are added
// stream by stream, so that results do not depend on the order in which the streams finished.  A warp reads four channels of eight rows side by side.
constexpr int PJ_THREADS = 128, PJ_ROWS = 8, PJ_PARTS = PJ_THREADS / PJ_ROWS;

template <typename T>
__global__ void __launch_bounds__(PJ_THREADS) paged_attention_join_kernel(const PagedAttention a) {
  __shared__ float weight[PJ_PARTS][PJ_ROWS];  // of a piece's row
  __shared__ float2 row_stats[PJ_ROWS];        // maximum, 1 / sum
  const int D = a.p.head_dim, tid = threadIdx.x, all_rows = a.z.rows();
  pdl_begin();
  const Joint j = a.joints[blockIdx.x];
  const int r0 = blockIdx.y * PJ_ROWS;
  if (j.streams == 0 || r0 >= j.count) return;
  const size_t floats = piece_floats(all_rows, D);
  // the first stream's piece is the one of the item it ends in, the others' the one of the item they start in
  const float* first = a.pieces + ((size_t)blockIdx.x * 2 + 1) * floats;
  const float* later = a.pieces + ((size_t)blockIdx.x + 1) * 2 * floats;
  auto piece = [&](int i) { return i == 0 ? first : later + (size_t)(i - 1) * 2 * floats; };
  {  // sixteen lanes a row
    const int r = tid / PJ_PARTS, part = tid % PJ_PARTS, row = min(r0 + r, j.count - 1);
    float m = -INFINITY, sum = 0.0f;
    for (int i = part; i < j.streams; i += PJ_PARTS) m = fmaxf(m, piece(i)[all_rows * D + row]);
#pragma unroll
    for (int o = PJ_PARTS / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    for (int i = part; i < j.streams; i += PJ_PARTS) sum += piece(i)[all_rows * (D + 1) + row] * piece_factor(piece(i)[all_rows * D + row], m);
#pragma unroll
    for (int o = PJ_PARTS / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (part == 0) {
      row_stats[r] = make_float2(m, sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f);
      if (a.lse && r0 + r < j.count) {
        const int of = j.block_row + row, token = a.z.by_group(of);
        a.lse[(j.row0 + token) * (long long)a.heads + j.head * a.z.group + of - token * a.z.group] = (m + log2f(sum)) * 0.6931471805599453f;
      }
    }
  }
  __syncthreads();
  constexpr int TURNS = 256 / (PJ_PARTS * 4);  // four channels a thread and turn
  const int r = tid & (PJ_ROWS - 1), mine = min(r0 + r, j.count - 1);
  float4 acc[TURNS] = {};
#pragma unroll 1
  for (int i0 = 0; i0 < j.streams; i0 += PJ_PARTS) {
    const int n = min(PJ_PARTS, j.streams - i0);
    if (i0 > 0) __syncthreads();
    if (tid / PJ_ROWS < n) weight[tid / PJ_ROWS][r] = piece_factor(piece(i0 + tid / PJ_ROWS)[all_rows * D + mine], row_stats[r].x);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
      const int c = (tid / PJ_ROWS + t * PJ_PARTS) * 4, at = piece_at(all_rows, mine, c);
      if (c >= D) break;
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const float f = weight[i][r];
        const float4 x = *reinterpret_cast<const float4*>(piece(i0 + i) + at);
        acc[t].x = fmaf(x.x, f, acc[t].x);
        acc[t].y = fmaf(x.y, f, acc[t].y);
        acc[t].z = fmaf(x.z, f, acc[t].z);
        acc[t].w = fmaf(x.w, f, acc[t].w);
      }
    }
  }
  if (r0 + r >= j.count) return;
  const int row = j.block_row + mine, token = a.z.by_group(row), head = j.head * a.z.group + row - token * a.z.group;
  const float inv = row_stats[r].y;
#pragma unroll
  for (int t = 0; t < TURNS; ++t) {
    const int c = (tid / PJ_ROWS + t * PJ_PARTS) * 4;
    if (c >= D) break;
    T* to = static_cast<T*>(a.out) + (j.row0 + token) * a.ld_out + head * D + c;
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(acc[t].x * inv, acc[t].y * inv), pack_bf16x2(acc[t].z * inv, acc[t].w * inv));
    } else {
      *reinterpret_cast<float4*>(to) = make_float4(acc[t].x * inv, acc[t].y * inv, acc[t].z * inv, acc[t].w * inv);
    }
  }
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
    const int streams = ctx->sm_count * std::max(1, std::min(8, 220 * 1024 / ((int)rows_shared(head_dim) + 4096)));
    r.kernel = Kernel::rows;
    r.z = deal_shape(4, 5, group, streams, 8, 1);
    static_assert(PR_ROWS == 1 << 4 && PR_KEYS == 1 << 5, "the shifts above");
  }
  return r;
}
template <typename T>
int rows_kernel(hl_ctx* ctx, const PagedAttention& a) {
  HL_ALLOW_SHARED(ctx, rows_shared(PR_MAX_DIM), paged_attention_rows_kernel<T>);
  pdl(paged_attention_rows_kernel<T>, a.z.streams, PR_THREADS, rows_shared(a.p.head_dim), ctx->stream)(a);
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
  HL_REQUIRE((long long)a.p.sequences * kv_heads < 0x7fffffffll, "hl_paged_attention: too many sequences");
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
  ProfileScope prof(ctx, HL_PROF_ATTENTION_FWD, 4.0 * a.p.tokens * (double)heads * dim * a.p.max_length);
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
  const dim3 joins(r.z.streams, r.z.rows() / PJ_ROWS);
  if (cache->dtype == HL_BF16) pdl(paged_attention_join_kernel<__nv_bfloat16>, joins, PJ_THREADS, 0, ctx->stream)(a);
  else pdl(paged_attention_join_kernel<float>, joins, PJ_THREADS, 0, ctx->stream)(a);
  HL_LAUNCH_CHECK("paged_attention_join_kernel");
  count_launch(ctx);
  return HL_OK;
}
