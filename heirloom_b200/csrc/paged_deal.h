// How the work of an attention call over a paged cache is dealt out: arithmetic on lengths, the same on the host, where it is tested.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define HL_BOTH __host__ __device__ __forceinline__
// Called, not inlined: long code that every warp role of a kernel has need of, and that takes plain numbers.  What takes a kernel's parameters is inlined: to
// pass them by reference a thread copies all of them to its stack first (64 one-token steps 152 us, with called walks 215).
#define HL_CALLED inline __host__ __device__ __noinline__
#else
#define HL_BOTH inline
#define HL_CALLED inline
#endif

namespace hl {

// The new tokens of a sequence: rows row0 .. row0 + n - 1, of which the last stands at position length - 1.
struct PagedSequence {
  int n, length, row0;
};
// False where `first` or `lengths` hold what they cannot: such a sequence is left out and the status word set.
// View: PagedView, or what a test puts in its place.
template <typename View>
HL_BOTH bool paged_sequence(const View& p, int s, PagedSequence* out) {
  const int row0 = p.first ? p.first[s] : s, end = p.first ? p.first[s + 1] : s + 1;
  out->row0 = row0;
  out->n = end - row0;
  out->length = p.lengths[s];
  const bool ok = row0 >= 0 && end >= row0 && end <= p.tokens && out->n <= p.max_new && out->length >= 0 && out->length <= p.max_length;
  if (!ok) out->n = out->length = 0;
  return ok;
}

// ---- the deal -----------------------------------------------------------------------------------------------------------------------
// An item is a block of `rows` query rows of one sequence and key head (rows of a sequence: token by token, the query heads that share
// the key head within a token) with the tiles of `keys` keys that its last row sees; one tile where it sees none, so that somebody
// writes its zeros.  All tiles of a call, and before those of an item what the item costs besides, stand in one line, sequence by sequence, key head by key head, block by block, and every
// stream takes the same stretch of that line, whatever the lengths are: ragged batches and a lone long sequence keep all streams busy alike.
// The host knows none of the lengths (a captured call has others each time), so each CTA finds its stretch itself.
template <typename T>
HL_BOTH T deal_min(T a, T b) { return b < a ? b : a; }
template <typename T>
HL_BOTH T deal_max(T a, T b) { return a < b ? b : a; }

// A division of 64 bits is some hundred instructions.
HL_CALLED long long deal_divide(long long a, long long b) { return a / b; }

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery 1994); a division is some forty instructions.  QuickDiv, which is for device code alone, for both sides.
struct DealDivide {
  uint32_t mul, shift;
  DealDivide(uint32_t d = 1) : shift(0) {
    while ((1ull << shift) < d) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  HL_BOTH int operator()(int n) const { return (int)(((((uint64_t)(uint32_t)n * mul) >> 32) + (uint32_t)n) >> shift); }
};

struct DealShape {
  int row_shift, key_shift;  // rows and keys of a tile, as powers of two
  int group;                 // query heads a key head
  int streams;               // that take part at most
  int least;                 // tiles a stream takes at least: a joint costs more than a few tiles
  int extra;                 // what starting and ending an item costs, in tiles; less than `least`
  DealDivide by_group;
  HL_BOTH int rows() const { return 1 << row_shift; }
  HL_BOTH int keys() const { return 1 << key_shift; }
};
inline DealShape deal_shape(int row_shift, int key_shift, int group, int streams, int least, int extra) {
  return DealShape{row_shift, key_shift, group, streams, least, extra, DealDivide((uint32_t)group)};
}

// sum over i < n of floor((a i + b) / m), by Euclid's steps on (a, m); all below 2^31.  What is left below m on both counts is turned about by the reciprocity law of such
// sums (Graham, Knuth and Patashnik, "Concrete Mathematics", 3.5).
HL_CALLED long long floor_sum(unsigned n, unsigned m, unsigned a, unsigned b) {
  long long sum = 0;
  while (n > 0) {
    if (a >= m) {
      sum += (long long)n * (n - 1) / 2 * (a / m);
      a %= m;
    }
    if (b >= m) {
      sum += (long long)n * (b / m);
      b %= m;
    }
    const unsigned long long top = (unsigned long long)a * n + b;
    if (top < m) break;
    n = (unsigned)(top / m);
    b = (unsigned)(top % m);
    const unsigned t = m;
    m = a;
    a = t;
  }
  return sum;
}

struct DealBlocks {  // the row blocks of one key head of a sequence
  int n, length, blocks, dead;  // dead: leading blocks none of whose rows stands at a position
};
HL_BOTH DealBlocks deal_blocks(const DealShape& z, const PagedSequence& q) {
  DealBlocks d{q.n, q.length, 0, 0};
  d.blocks = (q.n * z.group + z.rows() - 1) >> z.row_shift;
  if (q.length < q.n) d.dead = deal_min((q.n - q.length) * z.group >> z.row_shift, d.blocks);
  return d;
}
// keys that the rows of block b see, and the tiles they make
HL_BOTH int deal_keys(const DealShape& z, const DealBlocks& d, int b) {
  const int last = z.by_group(deal_min(d.n * z.group, (b + 1) << z.row_shift) - 1);
  return deal_max(0, d.length - d.n + last + 1);
}
HL_BOTH int deal_tiles(const DealShape& z, const DealBlocks& d, int b) {
  return deal_max(1, (deal_keys(z, d, b) + z.keys() - 1) >> z.key_shift);
}
// cost of a block, and of the blocks before b, in tiles
HL_BOTH int deal_cost(const DealShape& z, const DealBlocks& d, int b) { return z.extra + deal_tiles(z, d, b); }
HL_BOTH long long deal_before(const DealShape& z, const DealBlocks& d, int b) {
  const int whole = deal_min(b, d.blocks - 1);  // the last block may be short of rows
  long long sum = deal_min(whole, d.dead);
  if (whole > d.dead)  // ceil((length - n + 1 + floor(last row / group)) / keys) as one division
    sum += floor_sum((unsigned)(whole - d.dead), (unsigned)(z.group << z.key_shift), (unsigned)z.rows(),
                     (unsigned)(z.group * (d.length - d.n + z.keys()) + ((d.dead + 1) << z.row_shift) - 1));
  if (b > whole) sum += deal_tiles(z, d, whole);
  return sum + (long long)b * z.extra;
}
template <typename View>
HL_BOTH long long deal_sequence(const View& p, const DealShape& z, int s) {
  PagedSequence q;
  paged_sequence(p, s, &q);
  if (q.n == 0) return 0;
  const DealBlocks d = deal_blocks(z, q);
  return p.kv_heads * (d.blocks == 1 ? (long long)deal_cost(z, d, 0) : deal_before(z, d, d.blocks));
}

struct DealPlace {  // of a place in the line: its sequence, the length of the line before that
  int s;
  long long before;
};

// A walk over a stretch of the line, item by item.
struct DealItem {
  PagedSequence q;
  DealBlocks blocks;
  int s, head, block;          // head: the key head
  int tiles, tile0, tile1;     // of the item; those of this stretch
  long long at;                // the item's place in the line: `extra`, then its tiles
  long long until;             // end of the stretch
};
HL_BOTH bool deal_valid(const DealItem& it) { return it.tile0 < it.tile1; }
HL_BOTH void deal_clip(const DealShape& z, DealItem& it, long long from) {
  const long long first = it.at + z.extra;
  it.tile0 = (int)deal_max(0ll, from - first);
  it.tile1 = (int)deal_max(0ll, deal_min((long long)it.tiles, it.until - first));
}
// The item that holds place `from` of the line, in sequence `place`, up to `until`.  Only the last item of a stretch can be without tiles, where the stretch
// ends in the item's `extra`; it is the next stream's then.
template <typename View>
HL_BOTH DealItem deal_item(const View& p, const DealShape& z, const DealPlace& place, long long from, long long until) {
  DealItem it{};
  it.until = until;
  if (place.s >= p.sequences || from >= until) return it;
  it.s = place.s;
  paged_sequence(p, it.s, &it.q);
  it.blocks = deal_blocks(z, it.q);
  long long rest = from - place.before;
  const long long a_head = it.blocks.blocks == 1 ? deal_cost(z, it.blocks, 0) : deal_before(z, it.blocks, it.blocks.blocks);
  it.head = (int)deal_divide(rest, a_head);
  rest -= it.head * a_head;
  int low = 0, high = it.blocks.blocks;  // the last block with no more than `rest` before it
  while (high - low > 1) {
    const int mid = (low + high) / 2;
    if (deal_before(z, it.blocks, mid) <= rest) low = mid;
    else high = mid;
  }
  it.block = low;
  it.at = from - rest + (low > 0 ? deal_before(z, it.blocks, low) : 0);
  it.tiles = deal_tiles(z, it.blocks, low);
  deal_clip(z, it, from);
  return it;
}
template <typename View>
HL_BOTH void deal_next(const View& p, const DealShape& z, DealItem& it) {
  it.at += it.tiles + z.extra;
  if (it.at >= it.until) {
    it.tile0 = it.tile1 = 0;
    return;
  }
  if (++it.block == it.blocks.blocks) {
    it.block = 0;
    if (++it.head == p.kv_heads) {
      it.head = 0;
      do {
        if (++it.s >= p.sequences) {  // the line goes on, so there is one, unless somebody changed the lengths meanwhile
          it.tile0 = it.tile1 = 0;
          return;
        }
        paged_sequence(p, it.s, &it.q);
      } while (it.q.n == 0);
      it.blocks = deal_blocks(z, it.q);
    }
  }
  it.tiles = deal_tiles(z, it.blocks, it.block);
  deal_clip(z, it, it.at);
}

}  // namespace hl
