// Attention of new tokens over a paged cache on the tensor cores: bf16, heads of 64 or 128 channels, blocks of 128 rows.
//
// The rows of a block are queries of one key head, token by token and the query heads that share the key head within a token, so that a block
// is full whatever their number is, and each key tile is read once for all of them.  S = Q Kᵀ and O += P V are tensor-memory accumulators, P
// goes from registers to tensor memory over the scores it came from; a row's P is formed against a reference maximum that the row raises only when its
// maximum has grown by more than 2^8, and O is rescaled in place then.  Two CTAs an SM, so that one's products lie under the other's
// exponentials; a CTA is one stream of the deal (paged_deal.h) and walks over its stretch of tiles: four softmax warps with a thread a
// row, a thread that fetches keys and values a page (or 64 positions of it) a copy, and a thread that issues the products.
//
// P enters its product as bf16, which the matrix unit wants of both operands, V being bf16; its sum is of the f32 values.  Results are then within 0.0023 of their norm where
// an f32 P leaves 0.0017 of rounding them to bf16.
//
// What stands behind a sequence's last position may be anything.  Its keys are masked after the product; its values would make NaN of a
// probability of zero, so the product with V stops at the last sixteen keys that are seen, and the softmax warps clear the values of
// those sixteen that are not before they hand over P.
//
// What bounds it is the chain of a tile (scores, maximum, exponentials, hand-over, product), 1.0 us for heads of 64 and 1.1 of 128 with two streams an
// SM, 1.2 PFLOP/s of products for 128; an item costs 2 to 4 us besides, of which the next item's Q is hidden under the last tile (4 us an item when it was
// loaded after it).  A chunk of 4096 tokens over 8192 positions, 32 heads of 128 on 8 key heads: 384 us, 1.07 PFLOP/s; 19 sequences of 1 to 511 tokens and up to 4000
// positions, 12 heads of 64: 93 us.  The thread that queues products, or copies, is elected: by a lane's number it took 613 us instead of 508 for the chunk.
// Rows of four lanes put together by shuffles before they are stored: 93 -> 99 us, taken back.
#include "paged_attention.cuh"
#include "tc05.cuh"

namespace hl {
namespace {

constexpr int PT_BM = 128, PT_BN = 64;
constexpr int PT_SOFTMAX_WARPS = 4;
constexpr int PT_THREADS = (PT_SOFTMAX_WARPS + 2) * 32;
constexpr int PT_TMEM_COLS = 256;  // S: 2 x 64 columns, O: head_dim columns
constexpr int PT_Q_BLOCK = PT_BM * 128, PT_KV_BLOCK = PT_BN * 128;  // 64 channels: rows of 128 bytes

template <int HD>
struct PtShape {
  static constexpr int BLOCKS = HD / 64, K_STAGES = HD == 64 ? 5 : 3, V_STAGES = HD == 64 ? 5 : 2;
  static constexpr int Q_BYTES = BLOCKS * PT_Q_BLOCK, KV_BYTES = BLOCKS * PT_KV_BLOCK;
  static constexpr int DATA = Q_BYTES + (K_STAGES + V_STAGES) * KV_BYTES;
  static constexpr int SMEM = DATA + 1024;  // barriers, and the deal's words
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "shared memory per SM");
};

struct PtShared {
  uint64_t q_full;
  uint64_t k_full[5], k_empty[5], v_full[5], v_empty[5];
  uint64_t s_full[2], p_full[2], o_full[2];  // by tile
  uint32_t tmem_base;
  int abort_flag;
  union {
    long long deal[68];               // while the deal is worked out
    DealItem walk[PT_SOFTMAX_WARPS];  // from then on: the item that each softmax warp is at, or has fetched Q for
  };
};
static_assert(sizeof(PtShared) <= 1024, "barriers outgrow their place");

template <int HD>
__global__ void __launch_bounds__(PT_THREADS, 2)
paged_attention_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PagedAttention a) {
  using Z = PtShape<HD>;
  extern __shared__ __align__(1024) uint8_t pt_smem[];  // swizzled tiles want 1024 bytes; checked below
  uint8_t* sq = pt_smem;
  uint8_t* sk = sq + Z::Q_BYTES;
  uint8_t* sv = sk + Z::K_STAGES * Z::KV_BYTES;
  PtShared* sh = reinterpret_cast<PtShared*>(pt_smem + Z::DATA);
  const bool layout_ok = (tc05::smem_u32(pt_smem) & 1023u) == 0;
  volatile int* abort_flag = &sh->abort_flag;
  const PagedView& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < Z::K_STAGES; ++s) {
      tc05::mbar_init(&sh->k_full[s], 1);
      tc05::mbar_init(&sh->k_empty[s], 1);
    }
    for (int s = 0; s < Z::V_STAGES; ++s) {
      tc05::mbar_init(&sh->v_full[s], 1);
      tc05::mbar_init(&sh->v_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc05::mbar_init(&sh->s_full[i], 1);
      tc05::mbar_init(&sh->p_full[i], PT_SOFTMAX_WARPS);
      tc05::mbar_init(&sh->o_full[i], 1);
    }
    tc05::mbar_init(&sh->q_full, PT_SOFTMAX_WARPS);
    sh->abort_flag = layout_ok ? 0 : 1;
    tc05::fence_barrier_init();
  }
  if (warp == PT_SOFTMAX_WARPS + 1) {
    tc05::tmem_alloc(&sh->tmem_base, PT_TMEM_COLS);
    tc05::tmem_relinquish();
  }
  tc05::tc_fence_before_sync();
  __syncthreads();
  tc05::tc_fence_after_sync();
  const uint32_t tmem_s0 = sh->tmem_base;        // S buffers at +0 and +64, P over the S it is formed from
  const uint32_t tmem_o0 = tmem_s0 + 2 * PT_BN;  // O at +128
  pdl_begin();  // everything above touches nothing a predecessor wrote

  if (blockIdx.x == 0)
    for (int s = threadIdx.x; s < p.sequences; s += PT_THREADS) {
      PagedSequence q;
      if (!paged_sequence(p, s, &q)) atomicExch(p.status + ST_BAD_INDEX, 1);
    }
  Deal deal;
  DealPlace place;
  const int stream = blockIdx.x;
  deal_start<PT_THREADS>(p, a.z, stream, sh->deal, &deal, &place);
  const long long from = deal.chunk * stream, until = min(deal.total, from + deal.chunk);

  if (warp == PT_SOFTMAX_WARPS) {
    // -------------------------------------------------------------------------- keys and values, by one thread
    if (tc05::elect_one() && !*abort_flag) {
      tc05::tma_prefetch_desc(&map_k);
      tc05::tma_prefetch_desc(&map_v);
      const int rows = min(p.page_size, PT_BN), copies = PT_BN / rows;  // positions a copy, copies a tile
      bool ok = true;
      int g = 0;  // tiles fetched so far
      for (DealItem it = deal_item(p, a.z, place, from, until); ok && deal_valid(it); deal_next(p, a.z, it)) {
        const int keys = deal_keys(a.z, it.blocks, it.block);
        const int32_t* table = p.page_table + it.s * p.ld_table;
        // the pages of a tile are looked up a tile ahead
        int next[4];
        auto look_up = [&](int tile) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int t = tile * PT_BN + c * rows;
            next[c] = c < copies && tile < it.tile1 && t < keys ? table[t >> p.page_shift] : 0;
          }
        };
        look_up(it.tile0);
        for (int j = it.tile0; j < it.tile1; ++j, ++g) {
          const int ks = g % Z::K_STAGES, vs = g % Z::V_STAGES, within = (j * PT_BN) & (p.page_size - 1);
          const int here = min(copies, max(1, (keys - j * PT_BN + rows - 1) / rows));  // copies with keys that are seen
          int page[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            page[c] = next[c];
            if (page[c] < 0 || page[c] >= p.pages) {  // outside the cache: the copy brings zeros
              page[c] = p.pages;
              atomicExch(p.status + ST_BAD_INDEX, 1);
            }
          }
          look_up(j + 1);
          ok = tc05::mbar_wait(&sh->k_empty[ks], ((uint32_t)(g / Z::K_STAGES) & 1u) ^ 1u, abort_flag);
          if (!ok) break;
          tc05::mbar_arrive_expect_tx(&sh->k_full[ks], (uint32_t)(here * rows * HD * 2));
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (c < here) {
#pragma unroll
              for (int blk = 0; blk < Z::BLOCKS; ++blk)
                tc05::tma_load_4d(sk + ks * Z::KV_BYTES + blk * PT_KV_BLOCK + c * rows * 128, &map_k, &sh->k_full[ks], blk * 64, within, it.head, page[c]);
            }
          ok = tc05::mbar_wait(&sh->v_empty[vs], ((uint32_t)(g / Z::V_STAGES) & 1u) ^ 1u, abort_flag);
          if (!ok) break;
          tc05::mbar_arrive_expect_tx(&sh->v_full[vs], (uint32_t)(here * rows * HD * 2));
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (c < here) {
#pragma unroll
              for (int blk = 0; blk < Z::BLOCKS; ++blk)
                tc05::tma_load_4d(sv + vs * Z::KV_BYTES + blk * PT_KV_BLOCK + c * rows * 128, &map_v, &sh->v_full[vs], blk * 64, within, it.head, page[c]);
            }
        }
      }
    }
  } else if (warp == PT_SOFTMAX_WARPS + 1) {
    // -------------------------------------------------------------------------- products, by one thread
    if (tc05::elect_one() && !*abort_flag) {
      constexpr uint32_t idesc_qk = tc05::instr_desc_bf16_f32(PT_BM, PT_BN, false, false);
      constexpr uint32_t idesc_pv = tc05::instr_desc_bf16_f32(PT_BM, HD, false, true);
      // Q·Kᵀ runs up to two tiles ahead of P·V within an item; the next item's waits for its Q, which takes the place of this one's.
      DealItem qi = deal_item(p, a.z, place, from, until), it = qi;
      int qj = qi.tile0, qg = 0, q_items = 0;  // the next scores: tile of the item, tile of the CTA
      auto issue_qk = [&]() -> bool {          // S[qg & 1] = Q · K(qj)ᵀ
        if (!deal_valid(qi)) return true;
        const int s = qg % Z::K_STAGES;
        if (qj == qi.tile0 && !tc05::mbar_wait(&sh->q_full, (uint32_t)q_items & 1u, abort_flag)) return false;
        if (!tc05::mbar_wait(&sh->k_full[s], (uint32_t)(qg / Z::K_STAGES) & 1u, abort_flag)) return false;
        // P·V of two tiles before reads the P that stands here: products of other sizes are not kept in order
        if (qg >= 2 && !tc05::mbar_wait(&sh->o_full[qg & 1], (uint32_t)((qg - 2) >> 1) & 1u, abort_flag)) return false;
        tc05::tc_fence_after_sync();
        const uint32_t aq = tc05::smem_u32(sq), ak = tc05::smem_u32(sk + s * Z::KV_BYTES);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)  // 16 channels a step; four steps per 64-channel block
          tc05::umma_ss(tmem_s0 + (uint32_t)((qg & 1) * PT_BN),
                        tc05::smem_desc_sw128(aq + (ks / 4) * PT_Q_BLOCK + (ks % 4) * 32, 16, 1024),
                        tc05::smem_desc_sw128(ak + (ks / 4) * PT_KV_BLOCK + (ks % 4) * 32, 16, 1024), idesc_qk, ks > 0 ? 1u : 0u);
        tc05::umma_commit(&sh->k_empty[s]);
        tc05::umma_commit(&sh->s_full[qg & 1]);
        ++qg;
        if (++qj == qi.tile1) {
          deal_next(p, a.z, qi);
          qj = qi.tile0;
          ++q_items;
        }
        return true;
      };
      bool ok = issue_qk();
      int ahead = 1;  // scores issued beyond the tile at hand
      int g = 0, items = 0;
      for (; ok && deal_valid(it); deal_next(p, a.z, it), ++items) {
        const int keys = deal_keys(a.z, it.blocks, it.block);
        for (int j = it.tile0; j < it.tile1; ++j, ++g) {
          while (ok && ahead < 2 && q_items == items && deal_valid(qi)) {
            ok = issue_qk();
            ++ahead;
          }
          if (!ok) break;
          // P(g) stands in S(g)'s columns and, in an item's first tile, the last item's O has been read
          const int s = g % Z::V_STAGES;
          ok = tc05::mbar_wait(&sh->p_full[g & 1], (uint32_t)(g >> 1) & 1u, abort_flag) &&
               tc05::mbar_wait(&sh->v_full[s], (uint32_t)(g / Z::V_STAGES) & 1u, abort_flag);
          if (!ok) break;
          tc05::tc_fence_after_sync();
          const int steps = (min(PT_BN, max(1, keys - j * PT_BN)) + 15) / 16;
          const uint32_t av = tc05::smem_u32(sv + s * Z::KV_BYTES);
#pragma unroll
          for (int ks = 0; ks < PT_BN / 16; ++ks)
            if (ks < steps) {
              // A = P, two keys a column; B = V: rows are keys (MN-major), 16 keys per step, channel blocks PT_KV_BLOCK apart
              const uint64_t db = tc05::smem_desc_sw128(av + ks * (16 * 128), PT_KV_BLOCK, 1024);
              tc05::umma_ts(tmem_o0, tmem_s0 + (uint32_t)((g & 1) * PT_BN + ks * 8), db, idesc_pv, (j > it.tile0 || ks > 0) ? 1u : 0u);
            }
          tc05::umma_commit(&sh->v_empty[s]);
          tc05::umma_commit(&sh->o_full[g & 1]);
          --ahead;
          if (ahead < 1 && deal_valid(qi)) {  // at the end of an item
            ok = issue_qk();
            ++ahead;
            if (!ok) break;
          }
        }
      }
    }
  } else {
    // -------------------------------------------------------------------------- softmax
    const uint32_t lane_sel = (uint32_t)(warp * 32) << 16;
    constexpr float kRaise = 8.0f;
    bool ok = !*abort_flag;
    int g = 0;  // key tiles done so far
    Joint joint{};
    DealItem& walk = sh->walk[warp];
    if (lane == 0) walk = deal_item(p, a.z, place, from, until);
    __syncwarp();
    const int group = a.z.group;
    // The warp's rows of an item's Q on their way into shared memory, HD / 8 lanes a row; zeros where there is no row.  The products that read the
    // item before are done by then.
    auto fetch_q = [&]() {
      constexpr int LANES = HD / 8, STEP = 32 / LANES;
      const int row = (walk.block << a.z.row_shift) + warp * 32 + lane, token = a.z.by_group(row);
      const long long at = row < walk.q.n * group ? (walk.q.row0 + token) * a.ld_q + (walk.head * group + row - token * group) * (long long)HD : -1;
      const int chunk = lane % LANES;
#pragma unroll 4
      for (int r0 = 0; r0 < 32; r0 += STEP) {
        const int from_row = r0 + lane / LANES, r = warp * 32 + from_row;
        const long long x = __shfl_sync(0xffffffffu, at, from_row);
        const uint32_t to = tc05::smem_u32(sq + (chunk / 8) * PT_Q_BLOCK + r * 128 + (((chunk & 7) ^ (r & 7)) << 4));
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(static_cast<const __nv_bfloat16*>(a.q) + (x >= 0 ? x : 0) + chunk * 8), "r"(x >= 0 ? 16 : 0) : "memory");
      }
    };
    if (deal_valid(walk)) fetch_q();
    while (ok && deal_valid(walk)) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      tc05::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc05::mbar_arrive(&sh->q_full);
      if (threadIdx.x == 0 && deal_goes_on(walk)) joint = deal_joint(a.z, deal, walk, stream);
      const int row0 = (walk.block << a.z.row_shift) + warp * 32, all_rows = walk.q.n * group, keys = deal_keys(a.z, walk.blocks, walk.block);
      const int row = row0 + lane, token = a.z.by_group(row);
      const bool mine = row < all_rows;
      const int before = walk.q.length - walk.q.n;                    // positions before the new tokens
      const int sees = mine ? before + token + 1 : 0;                 // keys that this row sees
      const int warp_sees = max(0, before + a.z.by_group(row0) + 1);  // those that all rows of the warp see
      const int count = min(32, all_rows - row0);                     // rows of this warp, none if less than one
      const int head = walk.head * group + row - token * group, out_row = walk.q.row0 + token;
      const int tile0 = walk.tile0, tile1 = walk.tile1, piece_of = deal_whole(walk) ? -1 : deal_piece(walk);
      float m_ref = 0.0f;  // reference maximum, in log2 units
      float l_run = 0.f;   // row sum, scaled to m_ref
      for (int j = tile0; j < tile1; ++j, ++g) {
        ok = tc05::mbar_wait(&sh->s_full[g & 1], (uint32_t)(g >> 1) & 1u, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc05::tc_fence_after_sync();
        if (j == tile1 - 1) {  // the item's last scores: the next one's Q comes in while they are worked on
          __syncwarp();
          if (lane == 0) deal_next(p, a.z, walk);
          __syncwarp();
          if (deal_valid(walk)) fetch_q();
        }
        const int key0 = j * PT_BN, seen = min(PT_BN, max(1, keys - key0));
        if (seen & 15) {  // values of the last sixteen keys that no row sees: cleared, a quarter of them a warp
          const int vs = g % Z::V_STAGES, first = seen * 8, last = (seen + 15) / 16 * 128;  // pieces of 16 bytes
          ok = tc05::mbar_wait(&sh->v_full[vs], (uint32_t)(g / Z::V_STAGES) & 1u, abort_flag);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          for (int i = first + warp * 32 + lane; i < last; i += PT_SOFTMAX_WARPS * 32) {
#pragma unroll
            for (int blk = 0; blk < Z::BLOCKS; ++blk)
              *reinterpret_cast<uint4*>(sv + vs * Z::KV_BYTES + blk * PT_KV_BLOCK + i * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          tc05::fence_proxy_async_smem();
        }
        if (count <= 0) {  // no rows: what stands in these lanes reaches nobody
          __syncwarp();
          if (lane == 0) tc05::mbar_arrive(&sh->p_full[g & 1]);
          continue;
        }
        uint32_t sb[PT_BN];
        tc05::tmem_ld_32x32b_x32(tmem_s0 + (uint32_t)((g & 1) * PT_BN) + lane_sel, *reinterpret_cast<uint32_t(*)[32]>(&sb[0]));
        tc05::tmem_ld_32x32b_x32(tmem_s0 + (uint32_t)((g & 1) * PT_BN) + lane_sel + 32, *reinterpret_cast<uint32_t(*)[32]>(&sb[32]));
        tc05::tmem_ld_wait();
        if (key0 + PT_BN > warp_sees) {
#pragma unroll
          for (int i = 0; i < PT_BN; ++i)
            if (key0 + i >= sees) sb[i] = 0xff800000u;
        }
        float m_tile;
        {  // eight independent running maxima, so that the 64 comparisons are not one dependent chain
          float mx[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) mx[u] = __uint_as_float(sb[u]);
#pragma unroll
          for (int i = 8; i < PT_BN; ++i) mx[i & 7] = fmaxf(mx[i & 7], __uint_as_float(sb[i]));
          m_tile = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
        }
        const float m_new = m_tile * a.scale_log2;
        const bool raise = m_new > m_ref + kRaise;
        if (j == tile0) {
          m_ref = m_new == -INFINITY ? 0.0f : m_new;  // a row that sees nothing of the first tile sees nothing of later ones
        } else if (__any_sync(0xffffffffu, raise)) {
          // rows of this warp rescale their O in place; P·V of tile j-1 must have landed, and P·V of tile j is not
          // issued before this warp has handed over P(j)
          ok = tc05::mbar_wait(&sh->o_full[(g - 1) & 1], (uint32_t)((g - 1) >> 1) & 1u, abort_flag);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          tc05::tc_fence_after_sync();
          const float f = raise ? ex2_fast(m_ref - m_new) : 1.0f;
          if (raise) m_ref = m_new;
          l_run *= f;
#pragma unroll 1
          for (int hb = 0; hb < HD / 32; ++hb) {
            uint32_t ob[32];
            tc05::tmem_ld_32x32b_x32(tmem_o0 + lane_sel + hb * 32, ob);
            tc05::tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 32; ++k) ob[k] = __float_as_uint(__uint_as_float(ob[k]) * f);
            tc05::tmem_st_32x32b_x32(tmem_o0 + lane_sel + hb * 32, ob);
          }
          tc05::tmem_st_wait();
        }
        const float neg_m = -m_ref;
        const uint32_t tp = tmem_s0 + (uint32_t)((g & 1) * PT_BN) + lane_sel;
        float2 l_tile = make_float2(0.f, 0.f);
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // sixteen keys
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 x = fma2(make_float2(__uint_as_float(sb[q * 16 + 2 * e]), __uint_as_float(sb[q * 16 + 2 * e + 1])),
                                  both(a.scale_log2), both(neg_m));
            const float2 pr = make_float2(ex2_fast(x.x), ex2_fast(x.y));
            l_tile = add2(l_tile, pr);
            w[e] = pack_bf16x2(pr.x, pr.y);
          }
          tc05::tmem_st_32x32b_x8(tp + q * 8, w);
        }
        l_run += l_tile.x + l_tile.y;
        tc05::tmem_st_wait();
        tc05::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) tc05::mbar_arrive(&sh->p_full[g & 1]);
      }
      if (!ok) break;
      ok = tc05::mbar_wait(&sh->o_full[(g - 1) & 1], (uint32_t)((g - 1) >> 1) & 1u, abort_flag);  // the last P·V
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc05::tc_fence_after_sync();
      if (count > 0) {
        // Straight from registers: the place of Q belongs to the next item already.
        const float inv = l_run > 0.0f || l_run != l_run ? 1.0f / l_run : 0.0f;
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + out_row * a.ld_out + head * HD;
        float* piece = a.pieces + (size_t)(stream * 2 + max(piece_of, 0)) * piece_floats(PT_BM, HD);
        const int r = warp * 32 + lane;
#pragma unroll 1
        for (int hb = 0; hb < HD; hb += 64) {
          uint32_t ob[64];
          tc05::tmem_ld_32x32b_x32(tmem_o0 + lane_sel + hb, *reinterpret_cast<uint32_t(*)[32]>(&ob[0]));
          tc05::tmem_ld_32x32b_x32(tmem_o0 + lane_sel + hb + 32, *reinterpret_cast<uint32_t(*)[32]>(&ob[32]));
          tc05::tmem_ld_wait();
          if (piece_of >= 0) {
#pragma unroll
            for (int i = 0; i < 64; i += 4)
              if (mine) *reinterpret_cast<uint4*>(piece + piece_at(PT_BM, r, hb + i)) = make_uint4(ob[i], ob[i + 1], ob[i + 2], ob[i + 3]);
          } else {
#pragma unroll
            for (int i = 0; i < 64; i += 8) {
              uint4 o;
              o.x = pack_bf16x2(__uint_as_float(ob[i]) * inv, __uint_as_float(ob[i + 1]) * inv);
              o.y = pack_bf16x2(__uint_as_float(ob[i + 2]) * inv, __uint_as_float(ob[i + 3]) * inv);
              o.z = pack_bf16x2(__uint_as_float(ob[i + 4]) * inv, __uint_as_float(ob[i + 5]) * inv);
              o.w = pack_bf16x2(__uint_as_float(ob[i + 6]) * inv, __uint_as_float(ob[i + 7]) * inv);
              if (l_run == 0.0f) o = make_uint4(0u, 0u, 0u, 0u);
              if (mine) *reinterpret_cast<uint4*>(out + hb + i) = o;
            }
          }
        }
        if (piece_of >= 0) {
          piece[PT_BM * HD + r] = l_run == 0.0f ? -INFINITY : m_ref;
          piece[PT_BM * (HD + 1) + r] = l_run;
        } else if (mine && a.lse) {
          a.lse[out_row * (long long)a.heads + head] = l_run == 0.0f ? -INFINITY : (m_ref + log2f(l_run)) * 0.6931471805599453f;
        }
      }
      tc05::tc_fence_before_sync();  // O has been read: the next item's first P is handed over behind this
    }
    if (threadIdx.x == 0) a.joints[stream] = joint;
  }

  tc05::tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    for (int i = 0; i < 2000; ++i) __nanosleep(100);
    if (threadIdx.x == 0) atomicExch(p.status + (layout_ok ? ST_WAIT_EXPIRED : ST_BAD_ARGUMENT), 1);
  }
  if (warp == PT_SOFTMAX_WARPS + 1) {
    tc05::tc_fence_after_sync();
    tc05::tmem_dealloc(tmem_s0, PT_TMEM_COLS);
  }
}

template <int HD>
int launch(hl_ctx* ctx, const PagedAttention& a) {
  const PagedView& p = a.p;
  CUtensorMap maps[2];
  const uint64_t dims[4] = {(uint64_t)HD, (uint64_t)p.page_size, (uint64_t)p.kv_heads, (uint64_t)p.pages};
  const uint64_t strides[3] = {(uint64_t)p.position_stride * 2, (uint64_t)p.head_stride * 2, (uint64_t)p.page_stride * 2};
  const uint32_t box[4] = {64, (uint32_t)std::min(p.page_size, PT_BN), 1, 1};
  for (int i = 0; i < 2; ++i) {
    const int rc = make_tensor_map(&maps[i], HL_BF16, 4, i ? p.v : p.k, dims, strides, box, 128);
    if (rc != HL_OK) return rc;
  }
  HL_ALLOW_SHARED(ctx, PtShape<HD>::SMEM, paged_attention_tc_kernel<HD>);
  pdl(paged_attention_tc_kernel<HD>, a.z.streams, PT_THREADS, PtShape<HD>::SMEM, ctx->stream)(maps[0], maps[1], a);
  HL_LAUNCH_CHECK("paged_attention_tc_kernel");
  return HL_OK;
}

}  // namespace

DealShape paged_attention_tc_shape(int sms, int group) { return deal_shape(7, 6, group, 2 * sms, 8, 3); }
static_assert(PT_BM == 1 << 7 && PT_BN == 1 << 6, "the shifts above");

int paged_attention_tc(hl_ctx* ctx, const PagedAttention& a) { return a.p.head_dim == 64 ? launch<64>(ctx, a) : launch<128>(ctx, a); }

}  // namespace hl
