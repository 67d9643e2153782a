// How an attention call is cut into work (attn_rows.cu, attn_tiles.cu), and what its sizes have to satisfy: plain arithmetic, the same on
// the host and in the kernels.
//
// An item is a block of consecutive new tokens of one sequence with the query heads of one kv head; its work is the key tiles that some row
// of it sees, and some units more for its beginning and end (its q, its results).  Items in order (sequence, block, kv head), each as
// `extra` units and then its tiles, form one line, which the CTAs of the launch share evenly: a CTA takes the tiles in its piece.  An item whose tiles cross a border is joined from its CTAs' partial results, in their order, by whichever
// finishes last.
#pragma once
#include <math.h>

#include <cstddef>
#include <cstdint>

#ifdef __CUDACC__
#define INFR_ATTN_HD __host__ __device__ __forceinline__
#else
#define INFR_ATTN_HD inline
#endif

namespace infr {

constexpr int ATTN_MAX_SEQ = 4096;     // sequences per call: what is known of them fits where the key tiles go later (16 bytes each)
constexpr int ATTN_MAX_CTAS = 1024;    // join counters of a context
constexpr int ATTN_ROWS_LIMIT = 16;    // rows (tokens x heads of a kv head) of an item of the few-rows kernel
constexpr int ATTN_TILE_ROWS = 128;    // and of the tensor-memory kernel

struct AttnSeq {
  int q0, q_len;  // rows of the call
  int past;       // tokens in the cache before them (negative: that many rows at the front see nothing)
};
struct AttnBlock {
  int t0, nt;        // its tokens
  int lo, hi;        // keys that some row sees
  int tile0, ntile;  // key tiles, at least one: a block without keys still has its zeros to write
};

// Sequence from cu_q[s], cu_q[s + 1] and the cache's length, forced into the call's rows and the page table; *bad where that changed them.
INFR_ATTN_HD AttnSeq attn_seq(int a, int b, int kv, bool packed, int rows, int cap, bool* bad) {
  const int q0 = a < 0 ? 0 : (a > rows ? rows : a);
  const int q1 = b < q0 ? q0 : (b > rows ? rows : b);
  int n = q1 - q0;
  bool off = q0 != a || q1 != b;
  if (!packed) {
    n = kv < 0 ? 0 : (kv > cap ? cap : kv);
    off = off || n != kv;
  }
  if (off) *bad = true;
  return {q0, q1 - q0, n - (q1 - q0)};
}

INFR_ATTN_HD int attn_blocks(int q_len, int tb) { return (q_len + tb - 1) / tb; }

// Blocks counted on by a sequence's.  Those of sequences that lie one after the other are at most the call's rows; cu_q out of order can make
// n_seq x rows of them, past 31 bits: counted as rows + 1, and such a call is served as one without rows.
INFR_ATTN_HD int attn_blocks_on(long long sum, int rows) { return sum > rows ? rows + 1 : (int)sum; }

// The window as the kernels get it: 0 where it leaves nothing out of `most` tokens, so that it always stays below them.
INFR_ATTN_HD int attn_window(uint32_t window, uint32_t most) { return window < most ? (int)window : 0; }
// The first key that a row at this position sees: by comparison ahead of any difference, since rows with negative positions (as far as -2^22) and
// windows near 2^31 have none in 32 bits.  (Rows that see nothing get 0.)
INFR_ATTN_HD int attn_first_key(int position, int window) { return window > 0 && position >= window ? position - window + 1 : 0; }

INFR_ATTN_HD AttnBlock attn_block(const AttnSeq& s, int b, int tb, int log2_tile, int window) {
  AttnBlock r;
  r.t0 = b * tb;
  r.nt = s.q_len - r.t0 < tb ? s.q_len - r.t0 : tb;
  const int last = s.past + r.t0 + r.nt;
  r.hi = last > 0 ? last : 0;
  r.lo = attn_first_key(s.past + r.t0, window);
  r.tile0 = r.lo >> log2_tile;
  const int end = (r.hi + (1 << log2_tile) - 1) >> log2_tile;
  r.ntile = end > r.tile0 ? end - r.tile0 : 1;
  return r;
}

// Keys from the first number and below the second are seen by every row of the block.
INFR_ATTN_HD int attn_full_lo(const AttnSeq& s, const AttnBlock& b, int window) { return attn_first_key(s.past + b.t0 + b.nt - 1, window); }
INFR_ATTN_HD int attn_full_hi(const AttnSeq& s, const AttnBlock& b) { return s.past + b.t0 + 1; }

// a / b for quotients below 2^20: an estimate in f32 is off by one at most (64-bit divisions are a hundred instructions each).
INFR_ATTN_HD int attn_small_div(long long a, long long b) {
  int q = (int)((float)a / (float)b);
  if ((long long)q * b > a) --q;
  if ((long long)(q + 1) * b <= a) ++q;
  return q;
}

// A line of u units over C CTAs: the first `more` have each + 1, the others `each`.
struct AttnLine {
  long long each;
  int more;
};
// Where CTA c begins, and which CTA has the tile at place i.
INFR_ATTN_HD long long attn_begin(const AttnLine& l, int c) { return c * l.each + (c < l.more ? c : l.more); }
INFR_ATTN_HD int attn_cta_of(const AttnLine& l, long long i) {
  const long long wide = l.more * (l.each + 1);
  return i < wide ? attn_small_div(i, l.each + 1) : l.more + attn_small_div(i - wide, l.each);
}

// How many CTAs share a line of `units` whose longest item has `most`: all, unless joining the parts would take longer than the shares do.
// A part costs its joiner `join` eighths of a unit, so shares of m units and most / m parts take m + most join / (8 m): least at m^2 = most join / 8.
INFR_ATTN_HD int attn_ctas(long long units, int grid, int most, int join) {
  const int m = (int)ceilf(sqrtf(0.125f * (float)join * (float)most));
  const long long n = m > 1 ? units / m : units;
  return (int)(units < 1 ? 0 : n < 1 ? 1 : n < grid ? n : grid);
}

// Whether the few-rows kernel serves a call of up to max_rows rows (tokens x g heads) to a (sequence, kv head), of which there are `pairs`.  Its
// time grows with the rows past eight, the tile kernel's does not; but that one's ends are longer, which counts while every pair has many CTAs.
// Measured (us, few-rows / tile kernel, heads of 128, 8000 keys): 32 rows, 4 pairs 26.8 / 35.0, 8 30.4 / 33.8, 16 42.7 / 36.3; 16 rows, 16 pairs 31.8 / 33.8,
// 64 74.9 / 66.0; 8 rows, 128 pairs of 4000 keys 56.8 / 65.3.  16 rows and 32 pairs are the border, and one number for all: there heads of 64 take 34.1 / 36.7, of
// 256 100.1 / 104.1, 1000 keys 21.1 / 22.5, but heads of 128 over 8000 keys 51.1 / 44.3 (8 sequences) and 44.7 / 41.8 (16): these lose up to a seventh.
inline bool attn_few_rows(uint64_t max_rows, uint32_t g, uint64_t pairs) {
  return g <= (uint32_t)ATTN_ROWS_LIMIT && max_rows <= (pairs <= 8 ? 32u : pairs <= 32 ? 16u : 8u);
}

// What a call gives, as numbers.
struct AttnSizes {
  uint32_t rows, n_seq, n_head, n_kv, head_dim;
  uint32_t n_pages, page_size, max_pages;  // 0 where the keys are packed rows
  bool paged;
};

// nullptr, or what is wrong with the sizes; *unsupported: right, but not covered.
inline const char* attn_sizes_error(const AttnSizes& s, bool* unsupported) {
  *unsupported = false;
  if (!s.n_seq || !s.n_head || !s.n_kv || !s.head_dim) return "zero dimension";
  if (s.n_head % s.n_kv) return "n_head must be a multiple of n_kv";
  if (s.paged && (!s.n_pages || !s.page_size || !s.max_pages)) return "a page table needs n_pages, page_size and max_pages";
  if (!s.paged && (s.n_pages || s.page_size || s.max_pages)) return "n_pages, page_size and max_pages need a page table";
  if (s.paged && (uint64_t)s.max_pages * s.page_size > 0x7FFF0000u) return "max_pages * page_size is past 31 bits";
  *unsupported = true;
  if (s.head_dim % 16 || s.head_dim > 256) return "head_dim must be a multiple of 16, at most 256";
  if (s.n_head / s.n_kv > (uint32_t)ATTN_TILE_ROWS) return "more than 128 query heads to a kv head";
  if (s.n_seq > (uint32_t)ATTN_MAX_SEQ) return "more than 4096 sequences per call";
  if (s.rows > (1u << 22) || s.n_head > 1024) return "more than 2^22 rows or 1024 heads";
  if (s.paged && s.page_size % 16) return "page_size must be a multiple of 16";
  if (s.paged && s.n_pages > (1u << 30)) return "more than 2^30 pages";
  *unsupported = false;
  return nullptr;
}

// Bytes of the cache that a call's pages or rows take; all ones where that is past 64 bits (accepted sizes go to 2^80).
inline uint64_t attn_cache_bytes(const AttnSizes& s) {
  const uint64_t tokens = s.paged ? (uint64_t)s.n_pages * s.page_size : s.rows, each = (uint64_t)s.n_kv * s.head_dim * 2;
  return tokens > ~0ull / each ? ~0ull : tokens * each;
}

// Values a buffer needs for `rows` rows of `wide` values that are `stride` apart.
inline uint64_t attn_span(uint64_t rows, uint64_t stride, uint64_t wide) { return rows ? (rows - 1) * stride + wide : 0; }

// Whether two sets of rows (addresses a and b; bytes of a row, bytes between rows) share a byte.  Of one stride they may lie between each
// other, as the parts of wide rows do; of two, spans that overlap count as shared.
inline bool attn_rows_meet(uint64_t a, uint64_t wide_a, uint64_t stride_a, uint64_t b, uint64_t wide_b, uint64_t stride_b, uint64_t rows) {
  if (!(a < b + attn_span(rows, stride_b, wide_b) && b < a + attn_span(rows, stride_a, wide_a))) return false;
  if (stride_a != stride_b) return true;
  const uint64_t d = b >= a ? (b - a) % stride_a : (stride_a - (a - b) % stride_a) % stride_a;  // from a row of a to the next row of b
  return d < wide_a || d + wide_b > stride_a;
}

}  // namespace infr
