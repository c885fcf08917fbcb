// Attention of few new tokens over a paged cache: bf16, heads of 64 or 128 channels, at most 16 rows (new tokens times the query heads that share
// a key head), as in one-token steps.
//
// Bound by the keys and values, each of which is read once: 512 bytes a position and key head of 128 channels, against 2 * 16 * 128 * 2
// multiply-adds of which one in sixteen counts where there is one row.  A CTA of four warps walks over its tiles of 64 keys; a warp has sixteen keys of each tile
// and a ring of copies of its own, so that nothing waits for another warp until an item ends.  S = Q Kᵀ and O += P V by the warp-wide
// matrix instruction of 16 rows: with so few rows the wide tensor-memory products would stand idle for fifteen sixteenths, and a hand-over a
// tile would cost more than the tile.  A row's P is formed against a reference maximum that is raised when the maximum has grown by more than 2^8, as
// in the kernel for many rows, and as there enters its product as bf16 (0.0023 of the results' norm, 0.0017 if it were f32).  What stands behind a sequence's last position is not read: such keys and values are zeros.
//
// Two deals.  Short sequences (1024 positions or fewer): a CTA takes whole items, known without the lengths, and nothing is joined.  Longer ones:
// the even deal of paged_deal.h.  Eight sequences of up to 1024 positions, 12 heads of 64: 11.6 us whole, 41 us as items of the tensor-core kernel; 64 ragged sequences
// of up to 8192, 32 heads of 128 on 8 key heads: 152 us, 6.2 TB/s, 95 % of the copy rate (there 189); two of 60001 and 131071 positions: 130 us, 92 %.
#include "paged_attention.cuh"

namespace hl {
namespace {

constexpr int PS_WARPS = 4, PS_THREADS = PS_WARPS * 32;
constexpr int PS_ROWS = 16, PS_KEYS = 64, PS_WARP_KEYS = PS_KEYS / PS_WARPS;

template <int HD>
struct PsShape {
  static constexpr int STAGES = HD == 128 ? 3 : 6;
  static constexpr int ROW = HD * 2;                                  // bytes
  static constexpr int TILE = PS_WARP_KEYS * ROW;                     // a warp's keys, or values
  static constexpr int RING = STAGES * 2 * TILE;                      // of a warp
  static constexpr int SUMS = PS_WARPS * (HD / 8) * 32 * 8;           // O of eight rows of all warps
  static constexpr int SMEM = PS_WARPS * RING + SUMS + PS_WARPS * PS_ROWS * 8;
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "shared memory per SM");
  static_assert(SUMS >= 68 * 8, "the deal's words stand there");
};

__device__ __forceinline__ void cp_async16(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Items a CTA takes whole: sequence by sequence, a key head each.
__device__ __forceinline__ void whole_item(const PagedView& p, const DealShape& z, int index, DealItem& it) {
  it.tile0 = it.tile1 = 0;
  const int items = p.sequences * p.kv_heads;
  for (; index < items; index += gridDim.x) {
    it.s = index / p.kv_heads;
    it.head = index - it.s * p.kv_heads;
    it.at = index;
    if (!paged_sequence(p, it.s, &it.q) && it.head == 0) atomicExch(p.status + ST_BAD_INDEX, 1);
    if (it.q.n == 0) continue;
    it.blocks = deal_blocks(z, it.q);
    it.tiles = it.tile1 = deal_tiles(z, it.blocks, 0);
    return;
  }
}

template <int HD, bool WHOLE>
__global__ void __launch_bounds__(PS_THREADS, 2) paged_attention_step_kernel(const PagedAttention a) {
  using Z = PsShape<HD>;
  extern __shared__ __align__(128) uint8_t ps_smem[];
  const PagedView& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, column = (lane & 3) * 2;
  uint8_t* sums = ps_smem + PS_WARPS * Z::RING;
  float2* row_stats = reinterpret_cast<float2*>(sums + Z::SUMS);  // [warp][row] maximum and sum
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(ps_smem) + warp * Z::RING;
  const int stream = blockIdx.x;
  pdl_begin();

  Deal deal{};
  DealItem load{}, it;
  if constexpr (WHOLE) {
    whole_item(p, a.z, stream, load);
  } else {
    if (stream == 0)
      for (int s = threadIdx.x; s < p.sequences; s += PS_THREADS) {
        PagedSequence q;
        if (!paged_sequence(p, s, &q)) atomicExch(p.status + ST_BAD_INDEX, 1);
      }
    DealPlace place;
    deal_start<PS_THREADS>(p, a.z, stream, reinterpret_cast<long long*>(sums), &deal, &place);
    const long long from = deal.chunk * stream;
    load = deal_item(p, a.z, place, from, min(deal.total, from + deal.chunk));
  }
  auto advance = [&](DealItem& i) {
    if constexpr (WHOLE) whole_item(p, a.z, (int)i.at + (int)gridDim.x, i);
    else deal_next(p, a.z, i);
  };
  it = load;

  // ---- copies: the tiles of all items one after the other, a group each
  constexpr int LANES = HD / 8, STEP = 32 / LANES, COPIES = PS_WARP_KEYS / STEP;  // lanes a row, rows a copy, copies a tile
  int load_tile = load.tile0, load_stage = 0;
  auto page_of = [&](const DealItem& i, int tile) {
    const int t = tile * PS_KEYS + warp * PS_WARP_KEYS;
    return deal_valid(i) && tile < i.tile1 && t < deal_keys(a.z, i.blocks, i.block) ? p.page_table[i.s * p.ld_table + (t >> p.page_shift)] : 0;
  };
  int next_page = page_of(load, load_tile);
  auto fetch = [&]() {
    if (deal_valid(load)) {
      const int page = next_page, keys = deal_keys(a.z, load.blocks, load.block), t0 = load_tile * PS_KEYS + warp * PS_WARP_KEYS;
      const bool known = page >= 0 && page < p.pages;
      if (!known && lane == 0) atomicExch(p.status + ST_BAD_INDEX, 1);
      const int row = lane / LANES, chunk = lane % LANES, left = known ? keys - t0 - row : 0;
      const long long where = (known ? page : 0) * p.page_stride + ((t0 & (p.page_size - 1)) + row) * p.position_stride + load.head * p.head_stride + chunk * 8;
      const __nv_bfloat16 *k = static_cast<const __nv_bfloat16*>(p.k) + where, *v = static_cast<const __nv_bfloat16*>(p.v) + where;
      const uint32_t to = ring + load_stage * 2 * Z::TILE + row * Z::ROW;
      const long long step = STEP * p.position_stride;
#pragma unroll
      for (int c = 0; c < COPIES; ++c) {
        const int r = row + c * STEP;
        const uint32_t at = to + c * STEP * Z::ROW + ((chunk ^ (r & 7)) << 4);
        const bool there = c * STEP < left;
        cp_async16(at, there ? k + c * step : p.k, there);
        cp_async16(at + Z::TILE, there ? v + c * step : p.v, there);
      }
      if (++load_tile == load.tile1) {
        advance(load);
        load_tile = load.tile0;
      }
      next_page = page_of(load, load_tile);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    load_stage = load_stage + 1 == Z::STAGES ? 0 : load_stage + 1;
  };
#pragma unroll 1
  for (int s = 0; s < Z::STAGES - 1; ++s) fetch();

  int stage = 0;
  Joint joint{};
  for (; deal_valid(it); advance(it)) {
    if constexpr (!WHOLE) {
      if (threadIdx.x == 0 && deal_goes_on(it)) joint = deal_joint(a.z, deal, it, stream);
    }
    const int group = a.z.group, row0 = it.block * PS_ROWS, count = min(PS_ROWS, it.q.n * group - row0);
    // Q: rows `quad` and `quad` + 8
    uint32_t q[HD / 16][4];
    int sees[2];  // keys that they see
    const __nv_bfloat16* q_row[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = row0 + quad + 8 * h, token = a.z.by_group(row);
      const bool mine = quad + 8 * h < count;
      sees[h] = mine ? it.q.length - it.q.n + token + 1 : 0;
      q_row[h] = mine ? static_cast<const __nv_bfloat16*>(a.q) + (it.q.row0 + token) * a.ld_q + (it.head * group + row - token * group) * (long long)HD + column : nullptr;
    }
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i) q[ks][i] = q_row[i & 1] ? *reinterpret_cast<const uint32_t*>(q_row[i & 1] + ks * 16 + (i >> 1) * 8) : 0u;
    const int all_see = it.q.length - it.q.n + a.z.by_group(row0) + 1;  // keys that every row sees
    float o[HD / 8][4] = {};
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // reference maxima in log2 units; sums of this lane's columns
#pragma unroll 1
    for (int tile = it.tile0; tile < it.tile1; ++tile) {
      asm volatile("cp.async.wait_group %0;" ::"n"(Z::STAGES - 2) : "memory");
      __syncwarp();
      fetch();  // into the stage that was read last
      const uint32_t sk = ring + stage * 2 * Z::TILE, sv = sk + Z::TILE;
      stage = stage + 1 == Z::STAGES ? 0 : stage + 1;
      const int key0 = tile * PS_KEYS + warp * PS_WARP_KEYS;
      float s[2][4] = {};
      {
        const int r = (lane & 7) + ((lane >> 4) << 3);  // keys 0-7, 0-7, 8-15, 8-15; channels 0-7, 8-15, 0-7, 8-15
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          uint32_t b[4];
          ldmatrix4(sk + r * Z::ROW + (((ks * 2 + ((lane >> 3) & 1)) ^ (r & 7)) << 4), b);
          mma16816(s[0], q[ks], b[0], b[1]);
          mma16816(s[1], q[ks], b[2], b[3]);
        }
      }
      if (key0 + PS_WARP_KEYS > all_see) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key0 + n * 8 + column + (i & 1) >= sees[i >> 1]) s[n][i] = -INFINITY;
      }
      float top[2];
      bool raise[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        top[h] = x * a.scale_log2;
        raise[h] = top[h] > m[h] + 8.0f;
      }
      if (__any_sync(0xffffffffu, raise[0] || raise[1])) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (raise[h]) {
            const float f = m[h] == -INFINITY ? 0.0f : ex2_fast(m[h] - top[h]);
            m[h] = top[h];
            l[h] *= f;
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) {
              o[n][2 * h] *= f;
              o[n][2 * h + 1] *= f;
            }
          }
      }
      uint32_t pa[4];  // P as the first operand: rows quad, quad + 8, then the same for keys 8-15
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float base = m[h] == -INFINITY ? 0.0f : m[h];  // a row that has seen nothing yet
          const float x = ex2_fast(fmaf(s[n][2 * h], a.scale_log2, -base)), y = ex2_fast(fmaf(s[n][2 * h + 1], a.scale_log2, -base));
          l[h] += x + y;
          pa[n * 2 + h] = pack_bf16x2(x, y);
        }
      {
        const int r = lane & 15;  // keys 0-15 twice; channels 0-7, then 8-15
#pragma unroll
        for (int ns = 0; ns < HD / 16; ++ns) {
          uint32_t b[4];
          ldmatrix4_trans(sv + r * Z::ROW + (((ns * 2 + (lane >> 4)) ^ (r & 7)) << 4), b);
          mma16816(o[2 * ns], pa, b[0], b[1]);
          mma16816(o[2 * ns + 1], pa, b[2], b[3]);
        }
      }
    }
    // ---- the warps' rows together
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if ((lane & 3) == 0) row_stats[warp * PS_ROWS + quad + 8 * h] = make_float2(m[h], l[h]);
    }
    __syncthreads();
    const bool whole = deal_whole(it);
    float* piece = WHOLE || whole ? nullptr : a.pieces + (size_t)(stream * 2 + deal_piece(it)) * piece_floats(PS_ROWS, HD);
    float2* mine = reinterpret_cast<float2*>(sums) + warp * (HD / 8) * 32 + lane;
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
      if (h * 8 >= count) break;
      float all_m = -INFINITY, all_l = 0.f;
#pragma unroll
      for (int w = 0; w < PS_WARPS; ++w) all_m = fmaxf(all_m, row_stats[w * PS_ROWS + quad + 8 * h].x);
#pragma unroll
      for (int w = 0; w < PS_WARPS; ++w) {
        const float2 x = row_stats[w * PS_ROWS + quad + 8 * h];
        all_l += x.y * piece_factor(x.x, all_m);
      }
      const float f = piece_factor(h ? m[1] : m[0], all_m);
      if (h) __syncthreads();  // the first eight rows' sums have been read
#pragma unroll
      for (int n = 0; n < HD / 8; ++n) mine[n * 32] = make_float2((h ? o[n][2] : o[n][0]) * f, (h ? o[n][3] : o[n][1]) * f);
      __syncthreads();
      const int row = row0 + quad + 8 * h, token = a.z.by_group(row);
      const long long at = it.q.row0 + token, head = it.head * group + row - token * group;
      const bool there = quad + 8 * h < count;
      const float inv = all_l > 0.0f || all_l != all_l ? 1.0f / all_l : 0.0f;
#pragma unroll
      for (int j = 0; j < HD / 8 / PS_WARPS; ++j) {
        const int n = warp * (HD / 8 / PS_WARPS) + j;
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < PS_WARPS; ++w) {
          const float2 x = reinterpret_cast<const float2*>(sums)[(w * (HD / 8) + n) * 32 + lane];
          sum.x += x.x;
          sum.y += x.y;
        }
        if (there) {
          if (piece) *reinterpret_cast<float2*>(piece + piece_at(PS_ROWS, quad + 8 * h, n * 8 + column)) = sum;
          else
            *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.out) + at * a.ld_out + head * HD + n * 8 + column) = pack_bf16x2(sum.x * inv, sum.y * inv);
        }
      }
      if (there && warp == 0 && (lane & 3) == 0) {
        if (piece) {
          piece[PS_ROWS * HD + quad + 8 * h] = all_m;
          piece[PS_ROWS * (HD + 1) + quad + 8 * h] = all_l;
        } else if (a.lse) {
          a.lse[at * a.heads + head] = (all_m + log2f(all_l)) * 0.6931471805599453f;
        }
      }
    }
    __syncthreads();  // sums and statistics have been read
  }
  if constexpr (!WHOLE) {
    if (threadIdx.x == 0) a.joints[stream] = joint;
  }
}

template <int HD>
int launch(hl_ctx* ctx, const PagedAttention& a, bool whole) {
  using Z = PsShape<HD>;
  if (whole) {
    HL_ALLOW_SHARED(ctx, Z::SMEM, paged_attention_step_kernel<HD, true>);
    const long long items = (long long)a.p.sequences * a.p.kv_heads;
    pdl(paged_attention_step_kernel<HD, true>, (unsigned)std::min<long long>(items, a.z.streams), PS_THREADS, Z::SMEM, ctx->stream)(a);
  } else {
    HL_ALLOW_SHARED(ctx, Z::SMEM, paged_attention_step_kernel<HD, false>);
    pdl(paged_attention_step_kernel<HD, false>, a.z.streams, PS_THREADS, Z::SMEM, ctx->stream)(a);
  }
  HL_LAUNCH_CHECK("paged_attention_step_kernel");
  return HL_OK;
}

}  // namespace

DealShape paged_attention_step_shape(int sms, int group) {
  static_assert(PS_ROWS == 1 << 4 && PS_KEYS == 1 << 6, "the shifts below");
  return deal_shape(4, 6, group, 2 * sms, 8, 1);
}

int paged_attention_step(hl_ctx* ctx, const PagedAttention& a, bool whole) {
  return a.p.head_dim == 64 ? launch<64>(ctx, a, whole) : launch<128>(ctx, a, whole);
}

}  // namespace hl
