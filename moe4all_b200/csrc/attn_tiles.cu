// Attention of many rows per (sequence, kv head): prompts, and chunks of new tokens over a cache.  An item is 128 rows (whole tokens x the
// query heads of a kv head, so that these share the keys' tiles); its key tiles go through the tensor cores with accumulators in tensor
// memory, one pass with a running maximum.  What bounds it is the tensor cores: q and the weights are two f16 pieces each (f32 results), so
// a pair (row, key) costs 8 hd operations at the f16 rate.
//
// One CTA per SM, roles by warpgroup:
//   weights   a thread per row and 64 keys (two groups for tiles of 128): scores S from tensor memory -> maximum, reference -> weights P, back
//             over S as f16 pieces.  Both groups on one tile: what the MMAs wait for is a tile's weights, and with a tile to each
//             group these took twice as long (3.3 against 1.7 thousand cycles; the tensor cores' part of a tile is 2.1)
//   sums      a thread per row: the f32 sums in registers.  Each tile's P V starts from zero in tensor memory and is added here, brought
//             to a common maximum: an accumulation over thousands of steps in the tensor cores, which truncate, would lose an f32
//             result's last bits (measured: 1.3e-8 of the result per step)
//   control   a warp for the copies, a warp for the MMAs, two that look after tiles with hidden keys
// S and P of two tiles, and the sums of two (one for heads wider than 64), fill tensor memory: while a tile's weights are made the
// tensor cores work on the next tile's scores and the last one's sums.
//
// Measured (us; the tensor cores' floor at 2 x 4 hd operations a pair and the measured 1666 TFLOP/s): 8192 tokens of 32 / 4 heads of 128 1050 (660),
// four chunks of 512 tokens over up to 16000 keys 590 (366), 8192 tokens in 16 sequences of 64 / 8 heads of 64 234 (51); the same chunks with 16 / 2 heads
// of 192 343 (221), of 256 462 (219: one buffer each for K and V, 32 words a thread spilled).  What bounds it is
// the weights: 3.0 thousand cycles a tile of 128 keys (maxima 0.6, powers of two and pieces 1.7, the rest waits), against 2.1 - 2.3 of MMAs.  Short
// sequences of narrow heads pay per item: q into pieces 3 - 4 thousand cycles, results out 4 - 5, masked tiles on the diagonal.
// Loops are kept rolled, and waits short: the roles share one instruction cache, and with every tile's code straight-line it hit 60% of
// the time and the 8192 tokens took 4.6 ms.  (The weights' loop over 32 keys of 64 unrolled: 628 -> 685 us for the chunks as they were then.)
#include "attn.cuh"
#include "umma.cuh"

namespace infr {
namespace {

constexpr float TILE_BIAS = 15.f, TILE_FALL = 8.f;  // see ATTN_BIAS; the reference is no less than a tile's maximum, and no more than 9 above it
constexpr int JOIN_PARTS = 160;    // parts that an item can have: CTAs of a launch
constexpr int RING = 4;            // tiles' and items' words in shared memory: the roles are never further apart

template <int HD>
struct TilesShape {
  static constexpr int LOG2_TILE = HD <= 128 ? 7 : 6, BK = 1 << LOG2_TILE;
  // tiles' time that an item's beginning and end take (16 sequences of heads of 64: 2 257, 3 269, 4 281 us as they were then; wider heads' tiles are
  // 64 keys or twice the work, and their results twice the columns and more)
  static constexpr int EXTRA = HD == 64 ? 2 : 3;
  // what joining a part of an item takes, in eighths of a tile's time (us with 2, 4, 8 and 16: 9 tokens of 12 / 1 heads of 64
  // over 42730 keys 34.4, 33.0, 33.1, 37.1; 61 of 10 / 2 heads of 192 over 5855 keys 34.2, 34.2, 45.6, 46.7)
  static constexpr int JOIN = 4;
  static constexpr int W_GROUPS = BK / 64;
  static constexpr int S_GROUPS = 3 - W_GROUPS, COLS = HD / S_GROUPS;  // columns of a sums thread
  static constexpr int THREADS = 512;
  static constexpr int SLABS = HD / 64, TILE = BK * HD * 2, QPIECE = 128 * HD * 2;
  static constexpr int BUFS = HD == 64 ? 4 : HD <= 192 ? 2 : 1;  // tiles of K, and of V, in shared memory
  static constexpr int OBUFS = HD == 64 ? 2 : 1;
  // columns of tensor memory: scores of two tiles, sums, q's pieces (of heads wider than 192 the first)
  static constexpr uint32_t O_COL = 2 * BK, Q_COL = O_COL + OBUFS * HD;
  static constexpr int Q_TMEM = HD <= 192 ? 2 : 1;
  static_assert(Q_COL + Q_TMEM * HD / 2 <= 512, "more columns than tensor memory has");
  // items' words are read at their end, tiles' before: with two sums' buffers the weights may be that far ahead
  static constexpr int ENDS = OBUFS == 1 ? RING : 2 * RING;
  static constexpr int OUT_COLS = S_GROUPS == 1 ? 32 : 16, OUT = 4 * S_GROUPS * 32 * OUT_COLS * 4;  // results on their way out, by warp
  static constexpr int SMALL = (2 * RING + ENDS + 2 * W_GROUPS + ENDS * W_GROUPS) * 128 * 4;          // rows' words, see the kernel
  static constexpr int SMEM = 1024 + 2 * QPIECE + 2 * BUFS * TILE + OUT + SMALL;
  static_assert(SMEM + 2048 <= 232448, "more shared memory than a CTA has");
  // registers by role: together as many as the launch has
  static constexpr int REG_W = HD == 128 ? 104 : 112, REG_S = HD == 64 ? 168 : HD == 128 ? 208 : 160, REG_C = HD == 64 ? 120 : HD == 128 ? 96 : 80;
  static_assert(REG_W * W_GROUPS + REG_S * S_GROUPS + REG_C <= 512, "more registers than the launch has");
};

template <int N>
__device__ __forceinline__ void set_regs() {  // from the launch's 128
  if constexpr (N < 128) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
  if constexpr (N > 128) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// An item as the roles see it: its tiles here, n0 .. n1 - 1 of the CTA's.
struct __align__(16) TileItem {
  int n0, n1, row0, n_rows;          // first row of the call, rows (tokens x heads)
  int key0, lo, hi, pos0;            // first key of its first tile here; keys that some row sees; position of its first token
  int full_lo, full_hi, head, s;     // keys that every row sees
  int q0, whole, first_cta, last_cta;  // the sequence's first row; no other CTA has tiles of it; the CTAs that have
};
constexpr int ITEMS = 16;  // the copies are at most nine items ahead of the sums

struct TileBars {
  uint64_t i_full[ITEMS];
  uint64_t k_empty[4], v_full[4], v_empty[4];
  uint64_t s_full[2];
  uint64_t ready[4];    // all that step n of the MMAs needs: weights of tile n, its V there and looked after, its sums' columns free, K of tile n + 2
  uint64_t k_first[2];  // K of the first two tiles
  uint64_t o_full[2];
  uint64_t a_full[RING];       // a tile's references (and, at an item's end, weights)
  uint64_t f_full[RING];       // an item's score factors
  uint64_t q_full, q_empty[RING];
};

// Whether some row of the item does not see some key of [ks, ks + n).
__device__ __forceinline__ bool tile_masked(const TileItem& it, int ks, int n) { return ks + n > it.full_hi || ks < it.full_lo; }

// Bit i: whether the key k0 + i is one of from .. to.
__device__ __forceinline__ uint32_t seen_keys(int k0, int from, int to) {
  const int lo = max(0, from - k0), n = min(32, to + 1 - k0);  // bits lo .. n - 1
  return n <= lo ? 0u : (~0u >> (32 - (n - lo))) << lo;
}

__device__ __forceinline__ void hide(float (&s)[32], uint32_t seen) {
#pragma unroll
  for (int i = 0; i < 32; ++i) s[i] = (seen >> i) & 1u ? s[i] : -CUDART_INF_F;
}

// Scores of 64 keys at sa, some of which are NaN in this warp's rows: these are put right, and the row's maximum is given back.  (A column at a
// time: all lanes take part.)
static __device__ __noinline__ float tile_odd_scores(const AttnParams& p, const TileItem& it, int ks, int from, int to, int row, uint32_t sa, bool put_right, float top) {
  const float* q = p.q + attn_row_offset(p, it.row0, it.head, put_right ? row : 0, p.q_stride);
  if (put_right) top = -CUDART_INF_F;
#pragma unroll 1
  for (int i = 0; i < 64; ++i) {
    float x = umma::tmem_ld_32x1(sa + i);
    const bool seen = put_right && ks + i >= from && ks + i <= to;
    if (seen && x != x) x = attn_odd_score(p, it.s, it.q0, it.head, ks + i, q);
    if (seen) top = fmaxf(top, x);
    __syncwarp();
    umma::tmem_st_32x1(sa + i, x);
  }
  return top;
}

// 64 scores at sa become what they are above the reference.
static __device__ __noinline__ void tile_far_scores(uint32_t sa, float f, float ref) {
#pragma unroll 1
  for (int i = 0; i < 64; ++i) umma::tmem_st_32x1(sa + i, __fadd_rn(__fmul_rn(umma::tmem_ld_32x1(sa + i), f), -ref));
}

template <int HD>
__global__ void __launch_bounds__(TilesShape<HD>::THREADS, 1)
    k_attn_tiles(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ AttnParams p, const int granule) {
  using Sh = TilesShape<HD>;
  constexpr int BK = Sh::BK, SLABS = Sh::SLABS, BUFS = Sh::BUFS, OBUFS = Sh::OBUFS, TILE = Sh::TILE;
  extern __shared__ unsigned char smem_raw[];
  __shared__ TileBars bars;
  __shared__ TileItem s_item[ITEMS], s_parts[2];
  __shared__ long long s_scan[Sh::THREADS / 32];
  __shared__ AttnStart s_start;
  __shared__ uint32_t s_tmem;
  __shared__ int s_last, s_gave_up, s_odd[4 * RING];
  unsigned char* s_q = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char *s_k = s_q + 2 * Sh::QPIECE, *s_v = s_k + BUFS * TILE;
  unsigned char* s_out = s_v + BUFS * TILE;
  float* s_ref = reinterpret_cast<float*>(s_out + Sh::OUT);   // [RING][128] reference after a tile
  float* s_fac = s_ref + RING * 128;                          // [RING][128] score factors by item
  float* s_end = s_fac + RING * 128;                          // [ENDS][128] reference at an item's end
  float* s_l = s_end + Sh::ENDS * 128;                        // [ENDS][W_GROUPS][128] weights then
  float* s_max = s_l + Sh::ENDS * Sh::W_GROUPS * 128;         // [2][W_GROUPS][128] a tile's maxima by group
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wg = warp >> 2, role = wg == 3 ? 3 + (warp & 3) : wg < Sh::W_GROUPS ? 0 : 1;  // 0 weights, 1 sums, 3 copies, 4 MMAs, 5 and 6 hidden keys

  pdl_trigger();  // the next kernel may take the SMs that this one leaves free, and do what needs no input of its
  if (tid == 0) {
    for (int i = 0; i < ITEMS; ++i) mbar_init(bars.i_full + i, 1);
    for (int i = 0; i < 4; ++i) mbar_init(bars.k_empty + i, 1), mbar_init(bars.v_full + i, 1), mbar_init(bars.v_empty + i, 1), mbar_init(bars.ready + i, 4 * (Sh::W_GROUPS + Sh::S_GROUPS) + 3);
    for (int i = 0; i < 2; ++i) mbar_init(bars.s_full + i, 1), mbar_init(bars.o_full + i, 1), mbar_init(bars.k_first + i, 1);
    for (int i = 0; i < RING; ++i) mbar_init(bars.a_full + i, 4 * Sh::W_GROUPS), mbar_init(bars.f_full + i, 4 * Sh::W_GROUPS), mbar_init(bars.q_empty + i, 1);
    mbar_init(&bars.q_full, 4 * Sh::W_GROUPS);
    mbar_fence_init();
  }
  if (tid < 4 * RING) s_odd[tid] = 0;
  if (tid == 0) s_gave_up = 0;
  auto gave_up = [&]() {  // a bounded wait ran out
    atomicExch(&p.status->timeout, 11);
    s_gave_up = 1;
  };
  if (warp == 0) umma::tmem_alloc(&s_tmem);
  pdl_wait();
  attn_plan<Sh::THREADS, Sh::LOG2_TILE, Sh::EXTRA, Sh::JOIN>(p, reinterpret_cast<int*>(s_q), s_scan, &s_start);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the plan's words lay where tiles go
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const AttnStart st = s_start;
  const uint32_t tmem = s_tmem;
  const int N = (int)(st.until - st.before);  // tiles of this CTA
  bool ok = true;

  if (N > 0 && wg == 3) set_regs<Sh::REG_C>();
  if (N == 0) {
    // nothing to do
  } else if (role == 3) {
    // ---- copies, and the items' words
    AttnCursor<Sh::LOG2_TILE, Sh::EXTRA> c;
    c.start(p, st);
    int t = c.first(st), t_end = 0;  // the tile of its item that comes next, and where its tiles end here
    const int pieces = BK / granule;
    const bool packed = p.page_table == nullptr;
    int item = -1;
    struct Place {
      int y, w, head;  // of this lane's keys of a tile; y < 0: none
    };
    // Where tile n is.  Asked a step before its K is due, so that the page's number is there by then; V follows two steps later.
    auto place = [&](int n) {
      Place at = {-1, 0, 0};
      if (n >= N) return at;
      if (t >= t_end) {
        if (item >= 0) c.next(p), t = 0;
        t_end = c.end(st);
        ++item;
        if (lane == 0) {
          TileItem& it = s_item[item % ITEMS];
          const AttnShare sh = attn_share(c.ub, c.blk.ntile, st);
          it.n0 = n, it.n1 = n + t_end - t;
          it.row0 = c.seq.q0 + c.blk.t0, it.n_rows = c.blk.nt * p.g;
          it.key0 = (c.blk.tile0 + t) << Sh::LOG2_TILE, it.lo = c.blk.lo, it.hi = c.blk.hi, it.pos0 = c.seq.past + c.blk.t0;
          it.full_lo = attn_full_lo(c.seq, c.blk, p.window), it.full_hi = attn_full_hi(c.seq, c.blk), it.head = c.head, it.s = c.s;
          it.q0 = c.seq.q0, it.whole = sh.first == sh.last, it.first_cta = sh.first, it.last_cta = sh.last;
          mbar_arrive(bars.i_full + item % ITEMS);
        }
        // its q on the way to L2, a few tiles before it is turned into pieces
#pragma unroll 1
        for (int t = lane; t < c.blk.nt; t += 32)
          asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.q + (size_t)(c.seq.q0 + c.blk.t0 + t) * p.q_stride + (size_t)c.head * p.g * p.hd),
                       "r"(p.g * p.hd * 4) : "memory");
        __syncwarp();
      }
      at.head = c.head;
      const int key = ((c.blk.tile0 + t++) << Sh::LOG2_TILE) + lane * granule;
      if (lane < pieces && key < c.blk.hi && key + granule > c.blk.lo) {
        at.y = c.seq.q0 + key;
        if (!packed) {
          const int page = attn_page_of(p, key);
          at.w = attn_page_entry(p, c.s, page);
          at.y = key - page * p.page_size;
        }
      }
      return at;
    };
    auto load = [&](const Place& at, int n, const CUtensorMap* map, unsigned char* bufs, uint64_t* full, uint64_t* empty) {
      const int buf = n % BUFS;
      const int count = __popc(__ballot_sync(0xFFFFFFFFu, at.y >= 0));
      if (n >= BUFS) ok = wait_all(empty + buf, n / BUFS - 1);
      if (!ok) return;
      if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)(count * granule * 128 * SLABS));
      __syncwarp();
      if (at.y >= 0) {
        const int w = packed ? 0 : attn_page_checked(p, at.w);
        unsigned char* dst = bufs + buf * TILE + lane * granule * 128;
#pragma unroll
        for (int s = 0; s < SLABS; ++s) tma_load_4d(dst + s * (BK * 128), map, 64 * s, at.y, at.head, w, full);
      }
      __syncwarp();
    };
    // V of tile n, K of tile n + 2: the order in which they are used, and in which buffers come free
    Place v0 = {}, v1 = {}, k = place(0);
#pragma unroll 1
    for (int n = -2; n < N && ok; ++n) {
      if (n >= 0) load(v0, n, &vmap, s_v, bars.v_full + n % BUFS, bars.v_empty);
      v0 = v1, v1 = k;
      if (n + 2 < N && ok) {
        load(k, n + 2, &kmap, s_k, n < 0 ? bars.k_first + n + 2 : bars.ready + (n & 3), bars.k_empty);
        k = place(n + 3);
      } else if (ok && lane == 0) {
        mbar_arrive(bars.ready + (n & 3));
      }
    }
    if (!ok && lane == 0) gave_up();
  } else if (role == 4) {
    // ---- MMAs.  Scores run one tile ahead of the sums; their accumulators are free by then, since MMAs of one thread go in order
    const uint32_t idesc_s = umma::idesc_f16_f32(128, BK), idesc_o = umma::idesc_f16_f32(128, HD) | umma::IDESC_B_MN_MAJOR;
    const uint32_t tq = tmem + Sh::Q_COL;
    const uint64_t qdesc = umma::smem_desc_k_major_swz128(s_q, 0), kdesc = umma::smem_desc_k_major_swz128(s_k, 0);
    const uint64_t vdesc = umma::smem_desc_mn_major_swz128(smem_u32(s_v), 0, BK * 128);
    int s_it = 0, s_end = 0;  // items whose scores have begun, and the end of the last one's tiles
    // Both products take the smaller pieces first: the tensor cores truncate at every step, and then half of the steps only what is 2^-11
    // of the result (scores of size 10 in heads of 128: 16 steps' worth of 2^-24 of them would otherwise be on every weight).
    // Step n: the sums of tile n, then the scores of tile n + 2, whose accumulators are free by then: MMAs of one thread go in order.  What
    // is not there before a step is waited for behind the last step's MMAs.
#pragma unroll 1
    for (int n = -2; n < N && ok; ++n) {
      if (n >= 0) {
        const int buf = n % BUFS;
        ok = wait_all(bars.ready + (n & 3), n >> 2);
        if (!ok) break;
        umma::fence_after_sync();
        if (umma::elect_one()) {
          const uint32_t d = tmem + Sh::O_COL + (n % OBUFS) * HD, a = tmem + (n & 1) * BK;
          const uint64_t vd = vdesc + (uint64_t)((buf * TILE) >> 4);
#pragma unroll 1
          for (int piece = 1; piece >= 0; --piece)  // the small ones first: see above
#pragma unroll 2
            for (int k = 0; k < BK / 16; ++k)  // 32 keys: 16 columns of their weights, 16 of the rest
              umma::mma1_f16_ts(d, a + (k >> 1) * 32 + (k & 1) * 8 + 16 * piece, vd + (uint64_t)((k * 2048) >> 4), idesc_o, piece == 0 || k > 0 ? 1u : 0u);
          umma::commit1(bars.o_full + n % OBUFS);
          umma::commit1(bars.v_empty + buf);
        }
        __syncwarp();
      }
      const int next = n + 2;
      if (next < N) {
        if (next == s_end) {  // an item's q, into tensor memory behind the last item's scores
          ok = ok && wait_all(bars.i_full + s_it % ITEMS, s_it / ITEMS) && wait_all(&bars.q_full, s_it);
          if (!ok) break;
          s_end = s_item[s_it % ITEMS].n1;
          ++s_it;
          umma::fence_after_sync();
          if (umma::elect_one()) {
#pragma unroll 1
            for (int piece = 0; piece < Sh::Q_TMEM; ++piece)
#pragma unroll 2
              for (int k = 0; k < HD / 16; ++k)
                umma::copy1_128x256b(tq + piece * (HD / 2) + 8 * k, qdesc + (uint64_t)((piece * Sh::QPIECE + (k >> 2) * 16384 + (k & 3) * 32) >> 4));
            if (Sh::Q_TMEM == 2) umma::commit1(bars.q_empty + ((s_it - 1) & (RING - 1)));
          }
          __syncwarp();
        }
        const int buf = next % BUFS;
        if (n < 0) ok = ok && wait_all(bars.k_first + next, 0);
        if (!ok) break;
        umma::fence_after_sync();
        if (umma::elect_one()) {
          const uint32_t d = tmem + (next & 1) * BK;
          const uint64_t kd = kdesc + (uint64_t)((buf * TILE) >> 4);
#pragma unroll 1
          for (int piece = 1; piece >= 0; --piece)
#pragma unroll 4
            for (int k = 0; k < HD / 16; ++k) {
              const uint64_t b = kd + (uint64_t)(((k >> 2) * (BK * 128) + (k & 3) * 32) >> 4);
              if (piece < Sh::Q_TMEM) umma::mma1_f16_ts(d, tq + piece * (HD / 2) + 8 * k, b, idesc_s, piece == 0 || k > 0 ? 1u : 0u);
              else umma::mma1_f16_ss(d, qdesc + (uint64_t)((piece * Sh::QPIECE + (k >> 2) * 16384 + (k & 3) * 32) >> 4), b, idesc_s, k > 0 ? 1u : 0u);
            }
          umma::commit1(bars.s_full + (next & 1));
          umma::commit1(bars.k_empty + buf);
          if (Sh::Q_TMEM == 1 && next + 1 == s_end) umma::commit1(bars.q_empty + ((s_it - 1) & (RING - 1)));
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) gave_up();
  } else if (role > 4) {
    // ---- V tiles with hidden keys.  0 x value has to be 0 where a row does not see the key: keys that no row sees become zeros, and so do
    // values that are not finite; the item's end adds these to the rows that see them
    const int at = (warp & 1) * 32 + lane;
    int item = -1, end = 0;
    TileItem it;
#pragma unroll 1
    for (int n = 0; n < N && ok; ++n) {
      if (n == end) {
        ++item;
        ok = wait_all(bars.i_full + item % ITEMS, item / ITEMS);
        if (!ok) break;
        it = s_item[item % ITEMS];
        end = it.n1;
        if (at == 0) s_odd[(item + 2 * RING) % (4 * RING)] = 0;  // (eight items back: read)
      }
      const int ks = it.key0 + ((n - it.n0) << Sh::LOG2_TILE);
      ok = wait_all(bars.v_full + n % BUFS, n / BUFS);
      if (!ok) break;
      if (!tile_masked(it, ks, BK)) {
        if (lane == 0) mbar_arrive(bars.ready + (n & 3));
        continue;
      }
      bool odd = false;
      unsigned char* v = s_v + (n % BUFS) * TILE;
#pragma unroll 1
      for (int row = at; row < BK * SLABS; row += 64) {
        const int key = ks + (row & (BK - 1));
        const bool seen = key >= it.lo && key < it.hi;
        uint4* w = reinterpret_cast<uint4*>(v + row * 128);
        uint4 x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = w[(j + row) & 7];
        __half2 sum = __float2half2_rn(0.f);  // of 0 x value: NaN as soon as one is not finite
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const __half2* h = reinterpret_cast<const __half2*>(x + j);
#pragma unroll
          for (int i = 0; i < 4; ++i) sum = __hfma2(h[i], __float2half2_rn(0.f), sum);
        }
        if (!seen) {
#pragma unroll
          for (int j = 0; j < 8; ++j) w[(j + row) & 7] = make_uint4(0, 0, 0, 0);
        } else if (__hisnan(__low2half(sum)) || __hisnan(__high2half(sum))) {
          odd = true;
#pragma unroll 1
          for (int j = 0; j < 8; ++j) {
            const uint4 y = w[j];
            w[j] = make_uint4(only_finite(y.x), only_finite(y.y), only_finite(y.z), only_finite(y.w));
          }
        }
      }
      if (odd) s_odd[item % (4 * RING)] = 1;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(bars.ready + (n & 3));
    }
    if (!ok && lane == 0) gave_up();
  } else if (role == 0) {
    // ---- weights: thread = row, 64 keys of each tile
    set_regs<Sh::REG_W>();
    constexpr int GROUPS = Sh::W_GROUPS;
    const int row = tid & 127;
    const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16) + 64 * wg;
    // q of an item into two f16 pieces: eight lanes a row, the next rows on their way meanwhile.  What is left in the rows past the item's
    // reaches these rows' sums only.  (A short rolled loop: code that runs once an item comes from far away.)
    auto convert = [&](int item) {
      ok = wait_all(bars.i_full + item % ITEMS, item / ITEMS);
      if (!ok) return;
      const TileItem& it = s_item[item % ITEMS];
      const int n_rows = it.n_rows, l8 = lane & 7, r8 = tid >> 3;
      const float* q_item = p.q + (size_t)it.row0 * p.q_stride + (size_t)it.head * p.g * p.hd + 4 * l8;
      const int stride = (int)p.q_stride, head_pitch = p.hd, g = p.g;
      constexpr int STEP = 16 * GROUPS;
      float4 ahead[HD / 32];
      auto load = [&](int r) {
        const int t = attn_row_token(p, r);
        const float* src = q_item + (t * stride + (r - t * g) * head_pitch);
#pragma unroll
        for (int j = 0; j < HD / 32; ++j)
          ahead[j] = r < n_rows && 4 * (l8 + 8 * j) < p.hd ? __ldcg(reinterpret_cast<const float4*>(src + 32 * j)) : make_float4(0.f, 0.f, 0.f, 0.f);
      };
      load(r8);
      if (item > 0) ok = wait_all(bars.q_empty + ((item - 1) & (RING - 1)), (item - 1) / RING);
      if (!ok) return;
      float* fac = s_fac + (item & (RING - 1)) * 128;
#pragma unroll 1
      for (int r0 = 0; r0 < n_rows; r0 += STEP) {
        const int r = r0 + r8;
        float4 v[HD / 32];
        float big = 0.f;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) v[j] = ahead[j];
        if (r0 + STEP < n_rows) load(r + STEP);
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) big = fmaxf(big, fmaxf(fmaxf(fabsf(v[j].x), fabsf(v[j].y)), fmaxf(fabsf(v[j].z), fabsf(v[j].w))));
#pragma unroll
        for (int x = 1; x < 8; x <<= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, x));
        float down, up;
        attn_row_scale(big, down, up);
        if (p.scale_log2 < 0.f) down = -down;
        unsigned char* row_at = s_q + r * 128 + ((l8 & 1) << 3);
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
          uint2 hi, lo;
          split2(v[j].x * down, v[j].y * down, hi.x, lo.x);
          split2(v[j].z * down, v[j].w * down, hi.y, lo.y);
          unsigned char* dst = row_at + (j >> 1) * 16384 + ((((l8 >> 1) + 4 * (j & 1)) ^ (r & 7)) << 4);
          *reinterpret_cast<uint2*>(dst) = hi;
          *reinterpret_cast<uint2*>(dst + Sh::QPIECE) = lo;
        }
        // (not 0: hidden keys' -inf times it stays -inf)
        if (l8 == 0) fac[r] = fmaxf(up * fabsf(p.scale_log2), 1.2e-38f);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.q_full), mbar_arrive(bars.f_full + (item & (RING - 1)));
    };
    // an item's q is turned two tiles ahead of its first: its scores then follow the last item's without a break.  (Not earlier: the copies
    // know of an item three tiles ahead.)
    int turned = 0, n = 0;
#pragma unroll 1
    for (int item = 0; n < N && ok; ++item) {
      ok = wait_all(bars.i_full + item % ITEMS, item / ITEMS);
      if (!ok) break;
      const TileItem& it = s_item[item % ITEMS];
      const int n1 = it.n1, n_rows = it.n_rows;
      for (; turned <= item && ok; ++turned) convert(turned);
      ok = ok && wait_all(bars.f_full + (item & (RING - 1)), item / RING);
      if (!ok) break;
      const float f = s_fac[(item & (RING - 1)) * 128 + row];
      const int to = it.pos0 + (row < n_rows ? attn_row_token(p, row) : 0);  // the row sees the keys from .. to
      const int from = attn_first_key(to, p.window);
      const bool busy = (warp & 3) * 32 < n_rows;  // (other rows' weights are whatever is there: they reach those rows' sums only)
      float m = -CUDART_INF_F, l = 0.f;  // reference, weights
      // of the references that it fell from: where the weights go at the end (written behind a wait for the item's scores, not before: the sums have
      // read what an item ahead left there by then)
      float* highest = s_l + ((item % Sh::ENDS) * GROUPS + wg) * 128 + row;
      int ks = it.key0 + 64 * wg;
      int stop = n1 < N ? max(n, n1 - 2) : n1;  // where the next item's q is turned
#pragma unroll 1
      while (true) {
#pragma unroll 1
        for (; n < stop && ok; ++n, ks += BK) {
          ok = wait_all(bars.s_full + (n & 1), n >> 1);
          if (!ok) break;
          umma::fence_after_sync();
          const uint32_t sa = mine + (n & 1) * BK;
          float top = -CUDART_INF_F;
          const bool masked = ks + 64 > it.full_hi || ks < it.full_lo;
          if (busy) {
#pragma unroll 1
            for (int j = 0; j < 64; j += 32) {
              float s[32];
              umma::tmem_ld_32x32(sa + j, s);
              const uint32_t seen = masked ? seen_keys(ks + j, from, to) : ~0u;
              umma::tmem_ld_wait(s);
              if (masked) hide(s, seen);
              float t[2] = {top, -CUDART_INF_F};
#pragma unroll
              for (int i = 0; i < 32; i += 2) t[(i >> 1) & 1] = max_nan(t[(i >> 1) & 1], s[i], s[i + 1]);
              top = max_nan(t[0], t[1]);
            }
            const bool put_right = top != top && row < n_rows && l == l;  // (a row that is NaN already stays that)
            if (__any_sync(0xFFFFFFFFu, put_right)) top = tile_odd_scores(p, it, ks, from, to, row, sa, put_right, top);
          }
          if constexpr (GROUPS == 2) {
            float* at = s_max + (n & 1) * 256 + row;
            at[128 * wg] = top;
            asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp & 3)) : "memory");  // (the two warps of these rows)
            top = fmaxf(top, at[128 * (wg ^ 1)]);
          }
          if (m == -CUDART_INF_F) *highest = m;
          const float t = top * f;  // (a NaN leaves the reference where it is)
          float now = t > m ? ceilf(t) : m;
          if (t < m - TILE_FALL && t > -CUDART_INF_F) {  // down, but only as far as leaves the sums in range
            const float h = fmaxf(*highest, m);
            *highest = h;
            now = fmaxf(ceilf(t), h - 60.f);
          }
          l *= exp2_rel(m, now);
          m = now;
          if (busy) {
            // Scores past 2^22 lose the bias in one step (and weights past 2^16 f16's range): product, difference and bias one after the other for them
            const float ref = now == -CUDART_INF_F ? 0.f : now;
            const bool far = __any_sync(0xFFFFFFFFu, fabsf(ref) > 4194304.f && row < n_rows);
            const float ff = far ? 1.f : f, off = far ? TILE_BIAS : TILE_BIAS - ref;
            if (far) tile_far_scores(sa, f, ref);
            const float2 f2 = make_float2(ff, ff), off2 = make_float2(off, off), minus = make_float2(-1.f, -1.f);
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
            for (int j = 0; j < 64; j += 32) {
              float s[32];
              umma::tmem_ld_32x32(sa + j, s);
              const uint32_t seen = masked ? seen_keys(ks + j, from, to) : ~0u;
              umma::tmem_ld_wait(s);
              if (masked) hide(s, seen);
              uint32_t w[32];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float2 x = __ffma2_rn(make_float2(s[2 * i], s[2 * i + 1]), f2, off2);
                const float2 e = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                sum[i & 1] = __fadd2_rn(sum[i & 1], e);
                // the piece that f16 holds (below 2^-14, 2^-29 of the largest, rounded once more), and the rest
                const float2 h = make_float2(__uint_as_float(__float_as_uint(e.x) & 0xFFFFE000u), __uint_as_float(__float_as_uint(e.y) & 0xFFFFE000u));
                const float2 r = __ffma2_rn(h, minus, e);
                const __half2 hh = __floats2half2_rn(h.x, h.y), rr = __floats2half2_rn(r.x, r.y);
                w[i] = *reinterpret_cast<const uint32_t*>(&hh);
                w[16 + i] = *reinterpret_cast<const uint32_t*>(&rr);
              }
              umma::tmem_st_32x32_async(sa + j, w);
            }
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            umma::tmem_st_wait();
          }
          umma::fence_before_sync();
          if (wg == 0) s_ref[(n & (RING - 1)) * 128 + row] = m;
          if (n + 1 == n1) {
            *highest = l;
            if (wg == 0) s_end[(item % Sh::ENDS) * 128 + row] = m;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bars.ready + (n & 3)), mbar_arrive(bars.a_full + (n & (RING - 1)));
        }
        if (n >= n1 || !ok) break;
        convert(turned);
        ++turned;
        stop = n1;
      }
    }
    if (!ok && lane == 0) gave_up();
    if constexpr (GROUPS == 2)  // the other warp of these rows may give up later: it still waits for this one at the tiles until then
#pragma unroll 1
      for (; n < N; ++n) asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp & 3)) : "memory");
  } else {
    // ---- sums: thread = row, COLS of its columns
    set_regs<Sh::REG_S>();
    const int row = tid & 127, group = wg - Sh::W_GROUPS, col0 = group * Sh::COLS;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + Sh::O_COL + col0;
    float2 o[Sh::COLS / 2];
    float m = -CUDART_INF_F;
    int item = -1, first = 0, end = 0, n_rows = 0, parts = 0;
    for (int n = 0; n < OBUFS && n < N; ++n)
      if (lane == 0) mbar_arrive(bars.ready + n);
#pragma unroll 1
    for (int n = 0; n < N && ok; ++n) {
      if (n == end) {
        ++item;
        ok = wait_all(bars.i_full + item % ITEMS, item / ITEMS);
        if (!ok) break;
        first = n, end = s_item[item % ITEMS].n1, n_rows = s_item[item % ITEMS].n_rows;
        m = -CUDART_INF_F;
#pragma unroll
        for (int i = 0; i < Sh::COLS / 2; ++i) o[i] = make_float2(0.f, 0.f);
      }
      const bool mine = (warp & 3) * 32 < n_rows;
      ok = wait_all(bars.a_full + (n & (RING - 1)), n / RING);
      const float now = s_ref[(n & (RING - 1)) * 128 + row], a = exp2_rel(m, now);
      m = now;
      ok = ok && wait_all(bars.o_full + n % OBUFS, n / OBUFS);
      if (!ok) break;
      umma::fence_after_sync();
      if (mine) {
        const float2 a2 = make_float2(a, a);
#pragma unroll
        for (int j = 0; j < Sh::COLS; j += 16) {
          float t[16];
          umma::tmem_ld_32x16(lanes + (n % OBUFS) * HD + j, t);
          umma::tmem_ld_wait(t);
#pragma unroll
          for (int i = 0; i < 8; ++i) o[j / 2 + i] = __ffma2_rn(o[j / 2 + i], a2, make_float2(t[2 * i], t[2 * i + 1]));
        }
      }
      umma::fence_before_sync();
      __syncwarp();
      if (lane == 0 && n + OBUFS < N) mbar_arrive(bars.ready + ((n + OBUFS) & 3));
      if (n + 1 < end) continue;

      // ---- the item's end
      const TileItem& it = s_item[item % ITEMS];
      const bool whole = it.whole;
      const AttnShare share = {it.first_cta, it.last_cta};
      const bool odd_tiles = *reinterpret_cast<volatile int*>(s_odd + item % (4 * RING)) != 0;
      float L = 0.f;
#pragma unroll
      for (int w = 0; w < Sh::W_GROUPS; ++w) L += s_l[((item % Sh::ENDS) * Sh::W_GROUPS + w) * 128 + row];
      float at_end = s_end[(item % Sh::ENDS) * 128 + row];
      if (at_end == -CUDART_INF_F && L != 0.f) at_end = 0.f;  // nothing but NaN is a part that counts
      const float2 ml = make_float2(at_end, L);
      const size_t slot = (size_t)attn_slot(blockIdx.x, share) * 128 + row;
      const bool mine_row = row < n_rows;
      // (a part's rows lie side by side; the result's are found by the lane that stores them)
      const float inv = !whole ? 1.f : L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
      bool odd = odd_tiles;
      unsigned char* out = s_out + (warp & (4 * Sh::S_GROUPS - 1)) * 32 * Sh::OUT_COLS * 4;
      constexpr int WORDS = Sh::OUT_COLS / 4, ROWS = 32 / WORDS;  // 16-byte words of a row, rows that a warp stores at once
      const int first_row = (warp & 3) * 32;
      float* base = whole ? p.out + (size_t)it.row0 * p.out_stride + (size_t)it.head * p.g * p.hd : p.part + (slot - row) * HD;
      const int g = p.g, head_pitch = whole ? p.hd : HD, token_pitch = whole ? (int)p.out_stride : g * HD;
      if (mine) {
#pragma unroll
        for (int i0 = 0; i0 < Sh::COLS; i0 += Sh::OUT_COLS) {
#pragma unroll
          for (int i = 0; i < Sh::OUT_COLS; i += 4) {
            const float4 v = make_float4(o[(i0 + i) / 2].x, o[(i0 + i) / 2].y, o[(i0 + i) / 2 + 1].x, o[(i0 + i) / 2 + 1].y);
            odd |= !(fabsf(v.x) < CUDART_INF_F && fabsf(v.y) < CUDART_INF_F && fabsf(v.z) < CUDART_INF_F && fabsf(v.w) < CUDART_INF_F);
            *reinterpret_cast<float4*>(out + lane * Sh::OUT_COLS * 4 + ((i / 4 ^ (lane & (WORDS - 1))) << 4)) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
          }
          __syncwarp();
          const int word = lane & (WORDS - 1), col = col0 + i0 + 4 * word, stored = col < p.hd ? min(32, n_rows - first_row) : 0;
#pragma unroll 1
          for (int r = lane / WORDS; r < stored; r += ROWS) {
            const float4 v = *reinterpret_cast<const float4*>(out + r * Sh::OUT_COLS * 4 + ((word ^ (r & (WORDS - 1))) << 4));
            const int rr = first_row + r, t = attn_row_token(p, rr);
            __stcg(reinterpret_cast<float4*>(base + col + (t * token_pitch + (rr - t * g) * head_pitch)), v);
          }
          __syncwarp();
        }
        if (mine_row && !whole && group == 0) __stcg(p.part_ml + slot, ml);
        const bool put_right = mine_row && odd && L == L;
        if (__any_sync(0xFFFFFFFFu, put_right)) {  // (the rows' stores above are seen by the lanes that put them right)
          __threadfence();
          __syncwarp();
          attn_odd_values(p, it.s, it.q0, it.head, it.key0, it.key0 + ((end - first) << Sh::LOG2_TILE), BK, it.full_lo, it.full_hi, put_right,
                          it.pos0 + attn_row_token(p, row), col0, Sh::COLS,
                          whole ? p.out + attn_row_offset(p, it.row0, it.head, mine_row ? row : 0, p.out_stride) + col0 : p.part + slot * HD + col0);
        }
      }
      if (!whole) {  // the first and the last at most
        if (tid == 128 * Sh::W_GROUPS) s_parts[parts] = it;
        ++parts;
      }
    }
    // ---- items that other CTAs have tiles of: whoever comes last joins them.  All of these warps do or none does: one may have given up alone
    uint32_t all = ok;
    asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %0, 0;\n\tbar.red.and.pred b, 1, %1, a;\n\tselp.u32 %0, 1, 0, b;\n\t}" : "+r"(all) : "n"(128 * Sh::S_GROUPS) : "memory");
#pragma unroll 1
    for (int i = 0; i < parts && all; ++i) {
      if (attn_arrive(p, s_parts[i].first_cta, s_parts[i].last_cta, &s_last, tid == 128 * Sh::W_GROUPS, 1, 128 * Sh::S_GROUPS)) {
        const TileItem& it = s_parts[i];
        const AttnShare share = {it.first_cta, it.last_cta};
        const int n = share.last - share.first + 1, n_rows = it.n_rows, at = tid - 128 * Sh::W_GROUPS;
        float* base = p.out + (size_t)it.row0 * p.out_stride + (size_t)it.head * p.g * p.hd;
        // the parts' weights by row, then the sums by four columns, sixteen loads in flight (one after the other 11 parts of heads of 128 took 120 us)
        float* s_w = reinterpret_cast<float*>(s_k);  // (this CTA's products are done)
        static_assert(JOIN_PARTS * 128 * 4 <= 2 * BUFS * TILE + Sh::OUT, "the parts' weights lie where tiles and results were");
        if (at < n_rows) {
          float M = -CUDART_INF_F, L = 0.f;
#pragma unroll 8
          for (int c = 0; c < n; ++c) {
            const float2 ml = __ldcg(&p.part_ml[(size_t)attn_slot(share.first + c, share) * 128 + at]);
            s_w[c * 128 + at] = ml.x;
            M = fmaxf(M, ml.x);
          }
#pragma unroll 8
          for (int c = 0; c < n; ++c) {
            const float w = exp2_rel(s_w[c * 128 + at], M);
            L += w * __ldcg(&p.part_ml[(size_t)attn_slot(share.first + c, share) * 128 + at]).y;
            s_w[c * 128 + at] = w;
          }
          const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);  // NaN stays
#pragma unroll 1
          for (int c = 0; c < n; ++c) s_w[c * 128 + at] *= inv;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(128 * Sh::S_GROUPS) : "memory");
        const int words = p.hd / 4, stride = (int)p.out_stride, head_pitch = p.hd, g = p.g;
#pragma unroll 1
        for (int e0 = at; e0 < n_rows * words; e0 += 4 * 128 * Sh::S_GROUPS) {
          int row[4], col[4];
          float4 o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // (behind the last row: the last row again)
            const int e = min(e0 + i * 128 * Sh::S_GROUPS, n_rows * words - 1);
            row[i] = e / words, col[i] = 4 * (e - row[i] * words), o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll 1
          for (int c0 = 0; c0 < n; c0 += 4) {
            float4 v[4][4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float* part = p.part + (size_t)attn_slot(share.first + min(c0 + c, n - 1), share) * 128 * HD;
#pragma unroll
              for (int i = 0; i < 4; ++i) v[c][i] = __ldcg(reinterpret_cast<const float4*>(part + row[i] * HD + col[i]));
            }
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (c0 + c >= n) continue;
                const float w = s_w[(c0 + c) * 128 + row[i]];
                o[i].x += weighed(w, v[c][i].x), o[i].y += weighed(w, v[c][i].y), o[i].z += weighed(w, v[c][i].z), o[i].w += weighed(w, v[c][i].w);
              }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int t = attn_row_token(p, row[i]);
            if (e0 + i * 128 * Sh::S_GROUPS < n_rows * words) *reinterpret_cast<float4*>(base + col[i] + (t * stride + (row[i] - t * g) * head_pitch)) = o[i];
          }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(128 * Sh::S_GROUPS) : "memory");
      }
    }
    if (!ok && lane == 0) gave_up();
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  if (s_gave_up) attn_let_land();
  if (warp == 0) umma::tmem_dealloc(tmem);
}

template <int HD>
cudaError_t run_tiles(infr_cuda_ctx* ctx, const CUtensorMap& km, const CUtensorMap& vm, const AttnParams& p, int granule) {
  using Sh = TilesShape<HD>;
  const cudaError_t e = ensure_smem(reinterpret_cast<const void*>(&k_attn_tiles<HD>), Sh::SMEM);
  if (e != cudaSuccess) return e;
  return launch_ex(k_attn_tiles<HD>, dim3(ctx->sm_count < JOIN_PARTS ? ctx->sm_count : JOIN_PARTS), dim3(Sh::THREADS), Sh::SMEM, ctx->stream, true, km, vm, p, granule);
}

}  // namespace

int32_t launch_attn_tiles(infr_cuda_ctx* ctx, AttnParams p, const __half* k) {
  // a copy takes as many keys as lie side by side in every page
  int granule = p.hd <= 128 ? 128 : 64;
  while (p.page_table != nullptr && p.page_size % granule) granule >>= 1;
  p.k = k;
  CUtensorMap km, vm;
  if (!attn_cache_map(&km, k, p, granule) || !attn_cache_map(&vm, p.v, p, granule)) return fail(ctx, INFR_CUDA_ERR_CUDA, "attention: cuTensorMapEncodeTiled failed");
  p.tb = ATTN_TILE_ROWS / p.g;
  const cudaError_t e = p.hd <= 64 ? run_tiles<64>(ctx, km, vm, p, granule) : p.hd <= 128 ? run_tiles<128>(ctx, km, vm, p, granule)
                        : p.hd <= 192 ? run_tiles<192>(ctx, km, vm, p, granule) : run_tiles<256>(ctx, km, vm, p, granule);
  if (e != cudaSuccess) return check_cuda(ctx, e, "k_attn_tiles launch");
  ctx->launches += 1;
  return check_cuda(ctx, cudaGetLastError(), "k_attn_tiles launch");
}

}  // namespace infr
