// What the two attention kernels share: parameters, the line of units and a CTA's walk along it, joining of partial results.
#pragma once
#include <math_constants.h>

#include "attn_shape.h"
#include "kernels.cuh"
#include "tma.cuh"

namespace infr {

struct AttnParams {
  const float* q;
  float* out;
  const int *cu_q, *kv_len, *page_table;  // kv_len, page_table: null where the keys are packed rows
  const __half *k, *v;                    // for what the tiles' products of pieces get wrong (keys and values that are not finite)
  size_t page_pitch, head_pitch, row_pitch;  // of the cache, in values
  long long q_stride, out_stride;
  float* part;      // [2 CTAs][rows of an item][HD] sums, not yet divided
  float2* part_ml;  // [2 CTAs][rows of an item] reference and weight
  int* count;       // [CTAs] partial results in, per item by its first CTA; zero between launches
  DeviceStatus* status;
  float scale_log2;  // scale * log2(e)
  int rows, n_seq, n_kv, g, hd, page_size, max_pages, n_pages, window;
  int tb;            // tokens of an item
  uint32_t g_inv;    // ceil(2^16 / g): r / g = r * g_inv >> 16 for the rows r of an item
  int cap;           // max_pages * page_size
  int page_shift;    // log2(page_size), or -1
};

// Weights are 2^(x - reference + bias), two f16 pieces each: at most 2^15.9, and known to 2^-25.  The reference is a whole number (sums are
// brought to another one without error) that follows the keys' maximum up and, where that falls far enough, down again: what a weight is rounded by
// stays small against its neighbours' weights, not only against the row's largest, whose value may be next to nothing (a sink).
constexpr float ATTN_BIAS = 10.f;
constexpr float ATTN_SLACK = 5.9f;  // few-rows kernel: how far scores may pass the reference before it follows,
constexpr float ATTN_FALL = 14.f;   // and how far below it the largest of 16 keys may stay, looked at every fourth time: its weight is 2^-5 or more
// (64 streams, us: 84.7 without looking, 86 so, 88 with a slack of 1.9; rounds of shuffles for every 16 keys cost more than either)

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^(a - b) where a <= b, either possibly "no key yet" (-inf).
__device__ __forceinline__ float exp2_rel(float a, float b) { return a == -CUDART_INF_F ? 0.f : exp2_approx(a - b); }

// A part's sum x on its way into a join: where the part's weight has underflowed, what is not finite still arrives, so that a result does not
// depend on how its keys were cut into parts.
__device__ __forceinline__ float weighed(float w, float x) { return w != 0.f ? w * x : fabsf(x) < CUDART_INF_F ? 0.f : x; }

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* tm, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// mbar_wait_bounded in a tenth of the instructions (its loop is not unrolled): these kernels wait in many places, and their code has to stay
// in the instruction cache.
__device__ __forceinline__ bool attn_wait(uint64_t* bar, int phase) {
#pragma unroll 1
  for (uint32_t i = 0; i < (1u << 22); ++i) {
    if (mbar_try_wait(bar, (uint32_t)phase & 1)) return true;
    if (i > 4096) __nanosleep(64);
  }
  return false;
}
__device__ __forceinline__ bool wait_all(uint64_t* bar, int phase) { return __all_sync(0xFFFFFFFFu, attn_wait(bar, phase)); }

// Where a role has given up, copies and MMAs that nobody waits for any more are in flight: two milliseconds for what takes microseconds, by the clock
// (__nanosleep may return at once), before shared and tensor memory are somebody else's.
static __device__ __noinline__ void attn_let_land() {
  uint64_t begin, now;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(begin)::"memory");
#pragma unroll 1
  for (uint32_t i = 0; i < (1u << 24); ++i) {
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now)::"memory");
    if (now - begin > 2000000) return;
    __nanosleep(1000);
  }
}

__device__ __forceinline__ AttnSeq attn_load_seq(const AttnParams& p, int s) {
  bool bad = false;
  const AttnSeq r = attn_seq(__ldcg(p.cu_q + s), __ldcg(p.cu_q + s + 1), p.kv_len != nullptr ? __ldcg(p.kv_len + s) : 0, p.kv_len == nullptr, p.rows, p.cap, &bad);
  if (bad) p.status->bad_index = 2;
  return r;
}

// The page that a key is in (a division is a tenth of a slice's instructions).
__device__ __forceinline__ int attn_page_of(const AttnParams& p, int key) { return p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size; }
// A page's number as the table has it, and made sure of: apart, so that what lies between hides the load.
__device__ __forceinline__ int attn_page_entry(const AttnParams& p, int s, int page) { return __ldcg(p.page_table + (size_t)s * p.max_pages + page); }
__device__ __forceinline__ int attn_page_checked(const AttnParams& p, int id) {
  if ((unsigned)id < (unsigned)p.n_pages) return id;
  p.status->bad_index = 2;  // read as page 0, reported at the next sync
  return 0;
}
__device__ __forceinline__ int attn_page(const AttnParams& p, int s, int page) { return attn_page_checked(p, attn_page_entry(p, s, page)); }

// Token (of the item) and query head (of the kv head) of row r < 128: the error of g_inv adds less than 1 / 512.
__device__ __forceinline__ int attn_row_token(const AttnParams& p, int r) { return (int)((uint32_t)r * p.g_inv >> 16); }
__device__ __forceinline__ size_t attn_row_offset(const AttnParams& p, int token0, int head, int r, long long stride) {
  const int t = attn_row_token(p, r);
  return (size_t)(token0 + t) * stride + (size_t)(head * p.g + (r - t * p.g)) * p.hd;
}

// Where the values of a key and head begin in K or V; the keys behind it follow row_pitch apart up to its page's end.
__device__ __forceinline__ const __half* attn_value(const AttnParams& p, const __half* cache, int s, int q0, int head, int key) {
  if (p.page_table == nullptr) return cache + (size_t)(q0 + key) * p.row_pitch + (size_t)head * p.head_pitch;
  const int page = attn_page_of(p, key);
  return cache + (size_t)attn_page(p, s, page) * p.page_pitch + (size_t)(key - page * p.page_size) * p.row_pitch + (size_t)head * p.head_pitch;
}

// Powers of two that bring a row whose largest magnitude is `big` to [2^7, 2^8), and back; both normal numbers.
__device__ __forceinline__ void attn_row_scale(float big, float& down, float& up) {
  int e = (int)((__float_as_uint(big) >> 23) & 255u) - 134;
  e = big > 0.f && big < CUDART_INF_F ? max(-126, e) : 0;
  down = __uint_as_float((uint32_t)(127 - e) << 23);
  up = __uint_as_float((uint32_t)(127 + e) << 23);
}

// a and b as f16 pairs: the rounded values, and what the rounding left.
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// A pair of f16 bits with values that are not finite as zeros.
__device__ __forceinline__ uint32_t only_finite(uint32_t x) {
  if ((x & 0x7C00u) == 0x7C00u) x &= 0xFFFF0000u;
  if ((x & 0x7C000000u) == 0x7C000000u) x &= 0x0000FFFFu;
  return x;
}

// A CTA's share of the line: its tiles are those at the places [u0, u1).
struct AttnStart {
  AttnLine line;
  long long u0, u1, ub;     // ub: where the block's first head begins
  long long before, until;  // tiles ahead of u0 and of u1
  AttnSeq seq;
  int s, b, most;  // most: tiles of the line's longest item
};

// Inclusive sum over the block's threads; s_warp: one word per warp.
template <int THREADS>
__device__ __forceinline__ long long block_scan(long long v, long long* s_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += t;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
#pragma unroll 1
  for (int w = 0; w < warp; ++w) v += s_warp[w];
  return v;
}

// Every CTA works the whole line out for itself (a sequence and a few blocks per thread), which costs less than a launch for it.
// known: 16 bytes per sequence and one word of shared memory, free again after the call.  All threads take part.
// JOIN: see attn_ctas; 0 where joins cost little.
template <int THREADS, int LOG2_TILE, int EXTRA, int JOIN>
__device__ __forceinline__ void attn_plan(const AttnParams& p, int* known, long long* s_warp, AttnStart* st) {
  const int tid = threadIdx.x;
  AttnSeq* seqs = reinterpret_cast<AttnSeq*>(known);
  int* pre = known + 3 * p.n_seq;  // blocks ahead of each sequence
  if (tid == 0) pre[0] = st->most = 0;
  long long carry = 0;
#pragma unroll 1
  for (int s0 = 0; s0 < p.n_seq; s0 += THREADS) {
    const int s = s0 + tid;
    int n = 0;
    if (s < p.n_seq) {
      seqs[s] = attn_load_seq(p, s);
      n = attn_blocks(seqs[s].q_len, p.tb);
    }
    const long long sum = carry + block_scan<THREADS>(n, s_warp);
    if (s < p.n_seq) pre[s + 1] = attn_blocks_on(sum, p.rows);
    __syncthreads();
    carry = pre[min(s0 + THREADS, p.n_seq)];
  }
  const int F = carry > p.rows ? 0 : (int)carry;  // (reported: some sequence ends ahead of its beginning)
  const int per = (F + THREADS - 1) / THREADS, f0 = min(tid * per, F), f1 = min(f0 + per, F);
  int s = 0;
#pragma unroll 1
  for (int hi = p.n_seq; hi - s > 1;) {  // the last sequence that begins at or before block f0
    const int mid = (s + hi) / 2;
    if (pre[mid] <= f0) s = mid;
    else hi = mid;
  }
  // twice along this thread's blocks: their tiles, then the blocks that the CTA's borders fall into
  long long mine = 0, end = 0, u0 = 0, u1 = -1;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    long long tiles = end - mine;
    int at = s, most = 0;
#pragma unroll 1
    for (int f = f0; f < f1; ++f) {
      while (f >= pre[at + 1]) ++at;
      const int nt = attn_block(seqs[at], f - pre[at], p.tb, LOG2_TILE, p.window).ntile;
      if (pass == 1) {
        const long long ub = (tiles + (long long)EXTRA * f) * p.n_kv, n = (long long)(nt + EXTRA) * p.n_kv;
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
          const long long u = k == 0 ? u0 : u1;
          if (u < ub || u >= ub + n) continue;
          const int head = attn_small_div(u - ub, nt + EXTRA), in = (int)(u - ub - (long long)head * (nt + EXTRA)) - EXTRA;
          const long long ahead = tiles * p.n_kv + (long long)head * nt + (in > 0 ? in : 0);
          if (k == 0) st->s = at, st->seq = seqs[at], st->b = f - pre[at], st->ub = ub, st->before = ahead;
          else st->until = ahead;
        }
      }
      tiles += nt;
      if (JOIN > 0) most = max(most, nt);
    }
    if (pass == 0) {
      mine = tiles;
      if (JOIN > 0 && most > 0) atomicMax(&st->most, most);
      end = block_scan<THREADS>(mine, s_warp);
      if (tid == THREADS - 1) {
        const long long units = (end + (long long)EXTRA * F) * p.n_kv;
        const int ctas = attn_ctas(units, (int)gridDim.x, JOIN > 0 ? st->most + EXTRA : 0, JOIN);
        const bool idle = (int)blockIdx.x >= ctas;
        st->line.each = ctas > 0 ? units / ctas : 0;
        st->line.more = (int)(units - st->line.each * ctas);
        st->u0 = idle ? 0 : attn_begin(st->line, blockIdx.x);
        st->u1 = idle ? 0 : attn_begin(st->line, blockIdx.x + 1);
        st->before = 0;
        st->until = idle ? 0 : end * p.n_kv;  // (where u1 is the line's end)
      }
      __syncthreads();
      u0 = st->u0, u1 = st->u1;
      if (u0 >= u1) break;
    }
  }
  __syncthreads();
}

// One item after the other from the one that a CTA's share begins in.
template <int LOG2_TILE, int EXTRA>
struct AttnCursor {
  AttnSeq seq;
  AttnBlock blk;
  long long ub;  // the place of the item's first tile
  int s, b, head;

  __device__ __forceinline__ void start(const AttnParams& p, const AttnStart& st) {
    s = st.s, b = st.b, seq = st.seq;
    blk = attn_block(seq, b, p.tb, LOG2_TILE, p.window);
    head = attn_small_div(st.u0 - st.ub, blk.ntile + EXTRA);
    ub = st.ub + (long long)head * (blk.ntile + EXTRA) + EXTRA;
  }
  __device__ __forceinline__ void next(const AttnParams& p) {
    ub += blk.ntile + EXTRA;
    if (++head < p.n_kv) return;
    head = 0;
    ++b;
#pragma unroll 1
    while (b >= attn_blocks(seq.q_len, p.tb)) {
      if (s + 1 >= p.n_seq) return;  // past the line's end: nobody asks for more
      seq = attn_load_seq(p, ++s);
      b = 0;
    }
    blk = attn_block(seq, b, p.tb, LOG2_TILE, p.window);
  }
  // its tiles that the share has: first(), .. end() - 1; none where the share's border lies in the units ahead of them
  __device__ __forceinline__ int first(const AttnStart& st) const { return st.u0 > ub ? (int)(st.u0 - ub) : 0; }
  __device__ __forceinline__ int end(const AttnStart& st) const {
    const long long n = st.u1 - ub;
    return n >= blk.ntile ? blk.ntile : (n > 0 ? (int)n : 0);
  }
};

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN where one is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The score (times a positive number) of a visible key for which the products of q's pieces came out as NaN: the sum of q's products with the key's
// components that are not finite, which is all that decides it (inf times a piece of the other sign, or of zero, made the NaN).  NaN where the key is
// finite: then q is not.  (Not inlined: 11.1 -> 10.8 us for one token over 513 keys, which otherwise fetches its code too.)
static __device__ __noinline__ float attn_odd_score(const AttnParams& p, int s, int q0, int head, int key, const float* q) {
  const __half* k = attn_value(p, p.k, s, q0, head, key);
  float sum = 0.f;
  bool found = false;
#pragma unroll 2
  for (int i = 0; i < p.hd; i += 8) {
    const uint4 x = __ldcg(reinterpret_cast<const uint4*>(k + i));
    if (only_finite(x.x) == x.x && only_finite(x.y) == x.y && only_finite(x.z) == x.z && only_finite(x.w) == x.w) continue;
#pragma unroll 1
    for (int j = i; j < i + 8; ++j) {
      const float y = __half2float(__ldcg(k + j));
      if (!(fabsf(y) < CUDART_INF_F)) sum += y * __ldcg(q + j);
    }
    found = true;
  }
  return found ? sum * p.scale_log2 : CUDART_NAN_F;
}

// Which of an f16 pair's values are +inf or NaN (bits 0 and 1), and -inf or NaN (bits 16 and 17).
__device__ __forceinline__ uint32_t odd_pair(uint32_t x) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t h = x >> (16 * i), big = h & 0x7FFFu;
    if (big >= 0x7C00u) r |= (big > 0x7C00u ? 0x10001u : h & 0x8000u ? 0x10000u : 1u) << i;
  }
  return r;
}

// Some value that a row of this warp sees may not be finite: what the products of pieces made of it (inf times a piece of the other sign, or of
// zero, is NaN), or left out, in columns col0 .. of the result or part at dst, is put right: the sum of such values, whatever their weights.
// Columns that came out finite can only miss values of tiles with hidden keys, where they count as zeros.
// All lanes take part; those with a row are active: `to` its last key.  Keys by lane, 32 columns at a time, what is found noted in two words: other
// warps of the CTA wait meanwhile, and their waits have a limit.  (A row's lane by itself waits for memory at every key, and at every value found.)
// key0 .. key1: the keys of this part; full_lo .. full_hi: tiles inside have no hidden keys.
static __device__ __forceinline__ void attn_odd_values(const AttnParams& p, int s, int q0, int head, int key0, int key1, int tile, int full_lo, int full_hi, bool active,
                                                    int to, int col0, int cols, float* dst) {
  const int lane = threadIdx.x & 31, from = attn_first_key(to, p.window);
  const int lo = max(key0, __reduce_min_sync(0xFFFFFFFFu, active ? from : 0x7FFFFFFF)), hi = min(key1 - 1, __reduce_max_sync(0xFFFFFFFFu, active ? to : -1));
#pragma unroll 1
  for (int c = 0; c < cols && col0 + c < p.hd; c += 32) {
    const int n = min(32, p.hd - col0 - c);
    bool came_finite = true;
#pragma unroll 1
    for (int i = 0; i < n && active; ++i) came_finite &= fabsf(__ldcg(dst + c + i)) < CUDART_INF_F;
    const bool all = __any_sync(0xFFFFFFFFu, !came_finite);
    uint32_t plus = 0, minus = 0;  // columns: the row sees +inf or NaN there, -inf or NaN
#pragma unroll 1
    for (int ks = key0; ks < key1; ks += tile) {
      if (ks > hi || ks + tile <= lo || (!all && ks + tile <= full_hi && ks >= full_lo)) continue;
#pragma unroll 1
      for (int k0 = ks; k0 < ks + tile; k0 += 32) {
        const int key = k0 + lane;
        uint32_t mine_plus = 0, mine_minus = 0;
        if (key >= lo && key <= hi) {
          const uint4* v = reinterpret_cast<const uint4*>(attn_value(p, p.v, s, q0, head, key) + col0 + c);
#pragma unroll 1
          for (int j = 0; 8 * j < n; ++j) {
            const uint4 x = __ldcg(v + j);  // past L1, as all that an earlier kernel wrote: this one may have started beside it
            const uint32_t odd = odd_pair(x.x) | odd_pair(x.y) << 2 | odd_pair(x.z) << 4 | odd_pair(x.w) << 6;
            mine_plus |= (odd & 0xFFu) << (8 * j);
            mine_minus |= (odd >> 16) << (8 * j);
          }
        }
#pragma unroll 1
        for (uint32_t found = __ballot_sync(0xFFFFFFFFu, (mine_plus | mine_minus) != 0); found; found &= found - 1) {
          const int i = __ffs(found) - 1;
          const uint32_t a = __shfl_sync(0xFFFFFFFFu, mine_plus, i), b = __shfl_sync(0xFFFFFFFFu, mine_minus, i);
          if (active && k0 + i >= from && k0 + i <= to) plus |= a, minus |= b;
        }
      }
    }
#pragma unroll 1
    for (uint32_t found = plus | minus; found; found &= found - 1) {
      const int i = __ffs(found) - 1;
      __stcg(dst + c + i, !((plus >> i) & 1u) ? -CUDART_INF_F : (minus >> i) & 1u ? CUDART_NAN_F : CUDART_INF_F);
    }
    __syncwarp();
  }
}

// Whose partial results an item has: those of the CTAs first .. last, the first one's in its second slot, the others' in their first.
struct AttnShare {
  int first, last;
};
__device__ __forceinline__ AttnShare attn_share(long long ub, int ntile, const AttnStart& st) {
  return {attn_cta_of(st.line, ub), attn_cta_of(st.line, ub + ntile - 1)};
}
__device__ __forceinline__ int attn_slot(int cta, const AttnShare& sh) { return 2 * cta + (cta == sh.first ? 1 : 0); }

// After all threads have written their CTA's part: whether this CTA is the item's last and joins it.  Counting is by atomics, the join
// itself is in the order of the CTAs: the sums do not depend on who came last.
// (first, last are read behind the barrier.)
__device__ __forceinline__ bool attn_arrive(const AttnParams& p, const int& first, const int& last, int* s_last, bool leader, int threads_bar, int threads) {
  __threadfence();
  asm volatile("bar.sync %0, %1;" ::"r"(threads_bar), "r"(threads) : "memory");
  if (leader) {
    const int n = atomicAdd(p.count + first, 1);
    *s_last = n == last - first;
    if (n == last - first) p.count[first] = 0;
    __threadfence();
  }
  asm volatile("bar.sync %0, %1;" ::"r"(threads_bar), "r"(threads) : "memory");
  return *s_last != 0;
}

// Row r of the joined item, divided by its weight (zero where no key was seen), by a warp: the parts' weights by lane, their values eight
// parts in flight.  (A thread that walked the parts by itself took 24 us for 37 of them.)
template <int HD>
__device__ __forceinline__ void attn_join_row(const AttnParams& p, const AttnShare& sh, int item_rows, int r, float* dst) {
  constexpr int V = (HD + 127) / 128;
  const int lane = threadIdx.x & 31, parts = sh.last - sh.first + 1;
  float M = -CUDART_INF_F;
#pragma unroll 1
  for (int c = lane; c < parts; c += 32) M = fmaxf(M, __ldcg(&p.part_ml[(size_t)attn_slot(sh.first + c, sh) * item_rows + r]).x);
  M = warp_max(M);
  float L = 0.f;
  float4 o[V];
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int c0 = 0; c0 < parts; c0 += 32) {
    float w = 0.f;
    if (c0 + lane < parts) {
      const float2 ml = __ldcg(&p.part_ml[(size_t)attn_slot(sh.first + c0 + lane, sh) * item_rows + r]);
      w = exp2_rel(ml.x, M);
      L += w * ml.y;
    }
#pragma unroll 1
    for (int k0 = 0; k0 < min(32, parts - c0); k0 += 8) {
      float4 v[8][V];
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (c0 + k0 + k < parts && 4 * lane + 128 * j < HD)
            v[k][j] = __ldcg(reinterpret_cast<const float4*>(p.part + ((size_t)attn_slot(sh.first + c0 + k0 + k, sh) * item_rows + r) * HD + 4 * lane + 128 * j));
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float wk = __shfl_sync(0xFFFFFFFFu, w, k0 + k);
        if (c0 + k0 + k < parts) {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (4 * lane + 128 * j < HD)
              o[j].x += weighed(wk, v[k][j].x), o[j].y += weighed(wk, v[k][j].y), o[j].z += weighed(wk, v[k][j].z), o[j].w += weighed(wk, v[k][j].w);
        }
      }
    }
  }
  L = warp_sum(L);
  const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);  // NaN stays
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (4 * lane + 128 * j < p.hd) *reinterpret_cast<float4*>(dst + 4 * lane + 128 * j) = make_float4(o[j].x * inv, o[j].y * inv, o[j].z * inv, o[j].w * inv);
}

// Maps of a cache for boxes of 64 values x box_rows keys of one head: dimensions (values, keys of a page or packed rows, kv heads, pages).
bool attn_cache_map(CUtensorMap* tm, const __half* base, const AttnParams& p, int box_rows);

struct RopeParams {
  const float *q, *k, *v, *q_norm, *k_norm, *freq_factors;
  float* q_out;
  __half *k_cache, *v_cache;
  const int *cu_q, *kv_len, *page_table;
  DeviceStatus* status;
  size_t page_pitch, head_pitch, row_pitch;
  long long q_stride, k_stride, v_stride, qo_stride;
  double turns0, ratio;  // turns per token of pair 0, and of each pair relative to the one before
  float norm_eps;
  int rows, n_seq, n_head, n_kv, hd, page_size, max_pages, n_pages, cap, n_rot, interleaved;
};
int32_t launch_rope_kv(infr_cuda_ctx* ctx, const RopeParams& p);

int32_t launch_attn_rows(infr_cuda_ctx* ctx, AttnParams p, const __half* k, int max_rows);
int32_t launch_attn_tiles(infr_cuda_ctx* ctx, AttnParams p, const __half* k);

}  // namespace infr
