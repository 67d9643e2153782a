// Attention of a few rows per (sequence, kv head) over pages of 8 bits (kv_q8.cuh): the form of attn_rows.cu - a warp to 16 keys of a tile, both products transposed, q
// and the weights as two f16 pieces each, results f32 - with the codes turned into f16 fragments in registers.
//
//   S^T[16 keys, 8 rows] = K[16, hd] q^T[hd, 8],    O^T[hd, 8 rows] += V^T[hd, 16 keys] P^T[16 keys, 8 rows]
//
// What a product sums over may go in any order that both operands have.  A lane takes for K 16 neighbouring values of a key at once: one 16-byte word and one
// scale are four steps of the product.  And the 16 keys stand in the order in which a transposing load of bytes gives V's, four neighbouring keys to a lane: row i
// of the scores is key 4 (i / 2) + i % 2, row 8 + i two behind it.  A block of 16 values of V is one product's 16 rows, so its scales are one number to each key.
//
// Half the bytes of f16 pages leave the instructions as the bound: a code costs one of them on its way to f16 (byte behind the exponent of 1024, times
// the scale and minus 1152 times it: exact; as 32nds, so that no product is past f16).  So there are sixteen warps where the registers hold that, in two groups that take tiles of 128 keys in turn; and one warp of a
// group asks for a whole tile, each in its turn (by every warp for itself the copies were a third of all instructions, and a warp more would take registers from all).
// Between items stands one barrier of the CTA, behind which all add up the warps' sums; an item's q and its other words are made ready two items ahead.
//
// Measured (heads of 128, 32 to 4 kv heads; f16 pages in turn): single tokens of 64 sequences of 700 to 8000 keys 76.3 us (83.2), one of 131072 keys 51.3 (59.5; 143 MB, 2.8
// TB/s), one of 513 13.0 (11.0), of which the plan and the first item take 8 to 10.  What bounds it is latency: four warps to a scheduler, 550 to 680 instructions to 16 keys,
// issue 0.43.  By stamps, of a warp's 133 thousand cycles in a CTA with five items the tiles' work takes 39 to 45, waits for them 11 to 26, asking for the next ones 8 to 11,
// the barrier and the warps' sums at items' ends 11 to 33, the plan and the first item 7 to 19; an operation less to every pair of codes was half a per cent.
#include "attn.cuh"
#include "kv_q8.cuh"

namespace infr {
namespace {

constexpr int ROWS_EXTRA = 3;  // tiles' time that an item's beginning and end take

__device__ __forceinline__ void mma16816_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {  // (no moves of zeros ahead of it)
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// (Through pointers that come from the aligned beginning the compiler reads generic addresses: 26 loads of 16 keys, and 64-bit sums for them.)
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

// Two 16 x 16 matrices of bytes transposed: r[0], r[1] are rows lane / 4 and 8 more of the first, columns 4 (lane % 4) .. + 3.
__device__ __forceinline__ void ldsm2_t8(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <int HD, int NT>
struct Q8Shape {
  static constexpr int WARPS = HD <= 128 && NT == 1 ? 16 : 8, GROUPS = WARPS / 8;  // that do the products
  static constexpr int THREADS = WARPS * 32, RB = 8 * NT;
  static constexpr int LOG2_TILE = 7, KEYS = 1 << LOG2_TILE;
  static constexpr int SIDE = KEYS * HD;                // bytes of a tile of K, or of V
  static constexpr int STAGE = 2 * SIDE, SCALES = 2 * KEYS * HD / 16;
  static constexpr int PITCH = HD + 4;                  // words: the fragments' columns fall on different banks
  static constexpr int SUMS = WARPS * RB * PITCH * 4, STATS = 2 * WARPS * RB * 4;
  static constexpr int Q = NT * HD / 16 * 512;          // an item's q, as fragments
  // Twice the groups: what asks for a group's tile n + STAGES - GROUPS then has waited for the tile that the group asked for ahead of it, tile n itself.
  static constexpr int STAGES = 2 * GROUPS;
  static constexpr int SMEM = 1024 + STAGES * (STAGE + SCALES) + SUMS + STATS + 2 * Q;
  static_assert(SMEM + 2048 <= 232448, "more shared memory than a CTA has");
  static_assert(SMEM - 1024 >= 16 * ATTN_MAX_SEQ + 4, "what is known of the sequences fits where keys and sums go later");
};

// Columns of rows of the item, the part of it that lies here, where 16 values of V that a row sees are not numbers, become NaN.  All of the warp's lanes take
// part, a row to each of the first ones; `active`: not NaN already.  Blocks of 16 from block0 on, every `step`-th.
static __device__ __noinline__ void attn_odd_blocks(const AttnParams& p, int s, int head, int key0, int key1, bool active, int to, int block0, int step, float* dst) {
  const int lane = threadIdx.x & 31, from = attn_first_key(to, p.window);
  const int lo = max(key0, __reduce_min_sync(0xFFFFFFFFu, active ? from : 0x7FFFFFFF)), hi = min(key1 - 1, __reduce_max_sync(0xFFFFFFFFu, active ? to : -1));
#pragma unroll 1
  for (int b = block0; b < p.hd / 16; b += step) {
    bool sees = false;
#pragma unroll 1
    for (int k0 = lo & ~31; k0 <= hi; k0 += 32) {
      const int key = k0 + lane;
      bool odd = false;
      if (key >= lo && key <= hi) {
        const int page = attn_page_of(p, key);
        odd = __ldcg(p.vs + ((size_t)attn_page(p, s, page) * p.page_pitch + (size_t)head * p.head_pitch + (size_t)(key - page * p.page_size) * p.row_pitch) / 16 + b) >= Q8_ODD;
      }
#pragma unroll 1
      for (uint32_t found = __ballot_sync(0xFFFFFFFFu, odd); found; found &= found - 1) {
        const int key = k0 + __ffs(found) - 1;
        sees |= active && key >= from && key <= to;
      }
    }
    if (sees)
      for (int i = 0; i < 16; i += 4) __stcg(reinterpret_cast<float4*>(dst + 16 * b + i), make_float4(CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F, CUDART_NAN_F));
  }
}

// The tile that a group asks for next.
template <class Cursor>
struct AskState {
  Cursor c;
  int t;           // which one of its item it is
  int2 place[8];   // by copy: its first key's place in the page (-1: no row sees any of its keys), and the page
};

// An item as the warps see it.
struct Q8Item {
  int tiles, key0;               // tiles of it here, and the first one's first key
  int lo, hi, full_lo, full_hi;  // keys that some row sees; that every row sees
  int row0, nt, n_rows, pos0;    // its first row of the call, tokens, rows (tokens x heads), position of its first token
  int head, s;
  int whole, first_cta, last_cta;  // no other CTA has tiles of it; the CTAs that have
};

// The item at the cursor, and its q as B fragments of q^T: rows scaled by a power of two, as two f16 pieces; of 64 values step k has 16 c + 4 k .. + 3 of lane c.
// By a warp.
template <int HD, int NT, class Cursor>
static __device__ __noinline__ void q8_item(const AttnParams& p, const AttnStart& st, const Cursor& c, Q8Item* item, uint4* q, float* factor) {
  const int lane = threadIdx.x & 31;
  const int row0 = c.seq.q0 + c.blk.t0, n_rows = c.blk.nt * p.g, head = c.head;
#pragma unroll 1
  for (int n = 0; n < NT; ++n) {
    const int r = 8 * n + (lane >> 2);
    const bool has = r < n_rows;
    const float* src = p.q + attn_row_offset(p, row0, head, has ? r : 0, p.q_stride);
    float4 v[HD / 16];
    float big = 0.f;
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) {
      const int i = 64 * (k >> 2) + 16 * (lane & 3) + 4 * (k & 3);
      v[k] = has && i < p.hd ? __ldcg(reinterpret_cast<const float4*>(src + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (n == 0 && lane == 0) {  // (while these are on their way)
      const int first = c.first(st), end = c.end(st);
      const AttnShare share = attn_share(c.ub, c.blk.ntile, st);
      item->tiles = end - first, item->key0 = (c.blk.tile0 + first) << Q8Shape<HD, NT>::LOG2_TILE;
      item->lo = c.blk.lo, item->hi = c.blk.hi, item->full_lo = attn_full_lo(c.seq, c.blk, p.window), item->full_hi = attn_full_hi(c.seq, c.blk);
      item->row0 = row0, item->nt = c.blk.nt, item->n_rows = n_rows, item->pos0 = c.seq.past + c.blk.t0;
      item->head = head, item->s = c.s;
      item->whole = first == 0 && end == c.blk.ntile, item->first_cta = share.first, item->last_cta = share.last;
    }
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) big = fmaxf(big, fmaxf(fmaxf(fabsf(v[k].x), fabsf(v[k].y)), fmaxf(fabsf(v[k].z), fabsf(v[k].w))));
    big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
    float down, up;
    attn_row_scale(big, down, up);
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) {
      uint4 w;
      split2(v[k].x * down * 32.f, v[k].y * down * 32.f, w.x, w.z);  // (keys come as 32nds; 32 down may be past f32)
      split2(v[k].z * down * 32.f, v[k].w * down * 32.f, w.y, w.w);
      q[(n * (HD / 16) + k) * 32 + lane] = w;
    }
    if ((lane & 3) == 0) factor[r] = up * p.scale_log2;
  }
}

// WHOLE: heads of HD values, not fewer: the places of scales are known then (an eighth fewer instructions to 16 keys of heads of 128).
template <int HD, int NT, bool WHOLE>
__global__ void __launch_bounds__(Q8Shape<HD, NT>::THREADS, 1)
    k_attn_rows_q8(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ AttnParams p, const int granule) {
  using Sh = Q8Shape<HD, NT>;
  constexpr int WARPS = Sh::WARPS, GROUPS = Sh::GROUPS, THREADS = Sh::THREADS, RB = Sh::RB, STAGES = Sh::STAGES, STAGE = Sh::STAGE, SIDE = Sh::SIDE, PITCH = Sh::PITCH;
  constexpr int SLABS = HD / 64, KST = HD / 16, SLAB = Sh::KEYS * 64;
  constexpr int AHEAD = WARPS == 16 ? 2 : 4;  // sums under way
  using Cursor = AttnCursor<Sh::LOG2_TILE, ROWS_EXTRA>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint64_t full[STAGES], empty[STAGES], item_ready[2], sums_read;
  __shared__ long long s_scan[WARPS];
  __shared__ AttnStart s_start;
  __shared__ AskState<Cursor> s_ask[GROUPS];
  __shared__ Cursor s_walk;    // the last item that has been made ready
  __shared__ Q8Item s_item[2], s_part[2];
  __shared__ int s_described, s_parts, s_last, s_gave_up[2];
  __shared__ float s_factor[2][RB], s_weight[RB];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* scales = ring + STAGES * STAGE;
  float* s_o = reinterpret_cast<float*>(scales + STAGES * Sh::SCALES);
  float* s_m = s_o + WARPS * RB * PITCH;
  float* s_l = s_m + WARPS * RB;
  uint4* s_q = reinterpret_cast<uint4*>(s_l + WARPS * RB);  // [2][NT][KST][32]

  pdl_trigger();  // the next kernel may take the SMs that this one leaves free, and do what needs no input of its
  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(full + i, 1), mbar_init(empty + i, 8);
    mbar_init(item_ready, 1), mbar_init(item_ready + 1, 1), mbar_init(&sums_read, WARPS);
    s_parts = s_gave_up[0] = s_gave_up[1] = 0;
  }
  mbar_fence_init();
  pdl_wait();
  attn_plan<THREADS, Sh::LOG2_TILE, ROWS_EXTRA, 0>(p, reinterpret_cast<int*>(ring), s_scan, &s_start);
  if (s_start.until == s_start.before) return;
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the plan's words lay where the copies go
  const int N = (int)(s_start.until - s_start.before);  // tiles of this CTA
  const int nb = WHOLE ? HD / 16 : p.hd / 16;  // scales of a key
  // A tile's copies take as many keys at once as lie side by side in every page, one to a lane.  The tile t of the cursor's item, or of those behind it:
  auto look = [&](Cursor& c, int& t) {
    while (t >= c.end(s_start)) {
      t -= c.end(s_start);
      c.next(p);
    }
    const int key = ((c.blk.tile0 + t) << Sh::LOG2_TILE) + lane * granule;
    int2 at = make_int2(-1, 0);
    if (lane * granule < Sh::KEYS && key < c.blk.hi && key + granule > c.blk.lo) {
      const int page = attn_page_of(p, key);
      at = make_int2(key - page * p.page_size, attn_page_entry(p, c.s, page));
    }
    return at;
  };
  auto copy = [&](int n, int2 at, int head) {
    const int stage = n % STAGES, count = __popc(__ballot_sync(0xFFFFFFFFu, at.x >= 0));
    if (lane == 0) mbar_arrive_expect_tx(full + stage, (uint32_t)(count * granule * (2 * HD + 2 * nb)));
    __syncwarp();
    if (at.x >= 0) {
      const int w = attn_page_checked(p, at.y);
      const size_t first = ((size_t)w * p.page_pitch + (size_t)head * p.head_pitch + (size_t)at.x * p.row_pitch) / 16;
      unsigned char *dst = ring + stage * STAGE + lane * granule * 64, *sc = scales + stage * Sh::SCALES + lane * granule * nb;
#pragma unroll
      for (int s = 0; s < SLABS; ++s) tma_load_4d(dst + s * SLAB, &kmap, 64 * s, at.x, head, w, full + stage);
      bulk_g2s(sc, p.ks + first, granule * nb, full + stage);
#pragma unroll
      for (int s = 0; s < SLABS; ++s) tma_load_4d(dst + SIDE + s * SLAB, &vmap, 64 * s, at.x, head, w, full + stage);
      bulk_g2s(sc + Sh::SCALES / 2, p.vs + first, granule * nb, full + stage);
    }
    __syncwarp();
  };
  // the first two items, the first tiles, and where the groups' next ones are: a warp to each
  static_assert(2 + STAGES + GROUPS <= WARPS, "a warp to each");
  if (warp < 2 + STAGES + GROUPS) {
    Cursor c;
    c.start(p, s_start);
    if (warp < 2) {
      int ahead = 0;
      if (warp == 1) ahead = c.end(s_start) - c.first(s_start);
      if (warp == 1 && ahead < N) c.next(p);
      if (warp == 0 || ahead < N) q8_item<HD, NT>(p, s_start, c, s_item + warp, s_q + warp * (Sh::Q / 16), s_factor[warp]);
      if (warp == 1 && lane == 0) {
        s_walk = c;
        s_described = ahead + (ahead < N ? c.end(s_start) - c.first(s_start) : 0);
      }
    } else {
      const int n = warp - 2;
      int t = c.first(s_start) + n;
      if (n < N) {
        const int2 at = look(c, t);
        if (n < STAGES) copy(n, at, c.head);
        else if (lane < 8) s_ask[n - STAGES].place[lane] = at;
      }
      if (n >= STAGES && lane == 0) s_ask[n - STAGES].c = c, s_ask[n - STAGES].t = t;
    }
  }
  __syncthreads();

  bool alive = true;
  const int c0 = 2 * (lane & 3);  // this thread's columns (rows of the item): c0, c0 + 1 of every eight
  const int key1 = 4 * (lane >> 3) + ((lane >> 2) & 1);  // and its keys of the warp's 16: this one, and two behind it
  const int key0 = 16 * (warp & 7), group = warp >> 3;   // the warp's keys of a tile, and its tiles: those of this parity
  const uint32_t ring_at = smem_u32(ring), scales_at = smem_u32(scales);
  int done = 0;  // tiles of the items ahead
#pragma unroll 1
  for (int item = 0; done < N; ++item) {
    const Q8Item& it = s_item[item & 1];
    if (item >= 2 && alive) alive = wait_all(item_ready + (item & 1), (item >> 1) - 1);
    const uint32_t q_at = smem_u32(s_q) + (item & 1) * Sh::Q + 16 * lane;
    float f[NT][2];  // of the thread's columns: score -> log2 units
    int lim[NT][2];  // and the last key their row sees
    const int tiles = it.tiles, lo = it.lo, hi = it.hi, full_lo = it.full_lo, full_hi = it.full_hi, first_key = it.key0 + key0;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int rr = 8 * n + c0 + j;
        f[n][j] = s_factor[item & 1][rr];
        lim[n][j] = it.pos0 + (rr < it.n_rows ? attn_row_token(p, rr) : it.nt - 1);
      }

    float o[KST][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int k = 0; k < KST; ++k)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[k][n][i] = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -CUDART_INF_F, l[n][0] = l[n][1] = 0.f;

    bool odd = false;  // values that are no numbers were left out
#pragma unroll 1
    for (int t = (done ^ group) & (GROUPS - 1); t < tiles; t += GROUPS) {
      const int n = done + t, stage = n % STAGES, ks = first_key + (t << Sh::LOG2_TILE);
      if (alive) alive = wait_all(full + stage, n / STAGES);
      // The place that the group's last tile has left, for the next one but: by one warp, each in its turn.  The wait for it is one for the group's last asker too, and
      // for what that left.  (In shared memory: in registers all warps would pay for it.)  Where the tile after that one is comes behind the scores.
      const bool asks = alive && (warp & 7) == ((n / GROUPS) & 7) && n >= GROUPS && n - GROUPS + STAGES < N;
      int2 next = make_int2(-1, 0);
      if (asks) {
        AskState<Cursor>& a = s_ask[group];
        alive = wait_all(empty + (n - GROUPS) % STAGES, (n - GROUPS) / STAGES);
        if (alive) copy(n - GROUPS + STAGES, lane < 8 ? a.place[lane] : next, a.c.head);
        if (n + STAGES < N) {
          if (lane == 0) {
            a.t += GROUPS;
            while (a.t >= a.c.end(s_start)) {
              a.t -= a.c.end(s_start);
              a.c.next(p);
            }
          }
          __syncwarp();
          int t = a.t;
          next = look(a.c, t);
        }
      }
      if (!alive || ks >= hi || ks + 16 <= lo) {
        if (asks && lane < 8) s_ask[group].place[lane] = next;
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + stage);
        continue;
      }
      const uint32_t kb = ring_at + stage * STAGE + key0 * 64, sc = scales_at + stage * Sh::SCALES + key0 * nb;
      const bool masked = ks + 16 > full_hi || ks < full_lo;
      // scales that are no numbers: in K's place one that is NaN in f16 too, in V's zeros that wait for the item's end.  Zeros too for keys that no row sees: 0 x value is 0
      // whatever the codes.  (Seldom: looked for a word to a lane, and written where they lie.)
      uint32_t bad = 0;
      for (int e = lane; e < 4 * nb; e += 32) {
        const uint32_t a = lds32(sc + 4 * e), b = lds32(sc + Sh::SCALES / 2 + 4 * e);
        bad |= (a & (a << 1)) | (b & (b << 1));
      }
      if (__any_sync(0xFFFFFFFFu, (bad & 0x80808080u) != 0) || masked) {
        unsigned char* w = scales + stage * Sh::SCALES + key0 * nb;
#pragma unroll 1
        for (int e = lane; e < 16 * nb; e += 32) {
          const int key = ks + e / nb;
          const bool seen = key >= lo && key < hi, k_odd = w[e] >= Q8_ODD, v_odd = w[Sh::SCALES / 2 + e] >= Q8_ODD;
          if (k_odd) w[e] = 0xFF;
          if (v_odd || !seen) w[Sh::SCALES / 2 + e] = 0;
          odd |= v_odd && seen;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (ahead of the next copy to here)
        __syncwarp();
      }
      // ---- scores, q's pieces apart
      float s[NT][4], part[NT][4];
#pragma unroll
      for (int b = 0; b < SLABS; ++b) {
        uint4 kw[2];     // this lane's 16 values of both keys
        uint32_t kd[2], ko[2];  // and their scales (behind the head's end q is 0 and the codes' values are finite)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int key = key1 + 2 * j, blk16 = 4 * b + (lane & 3);
          kw[j] = lds128(kb + b * SLAB + key * 64 + (((lane & 3) ^ ((key >> 1) & 3)) << 4));
          q8_32nds(WHOLE || blk16 < nb ? lds8(sc + key * nb + blk16) * 0x00800080u : 0u, kd[j], ko[j]);  // (both halves of a pair: << 7)
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t w0 = k == 0 ? kw[0].x : k == 1 ? kw[0].y : k == 2 ? kw[0].z : kw[0].w;
          const uint32_t w1 = k == 0 ? kw[1].x : k == 1 ? kw[1].y : k == 2 ? kw[1].z : kw[1].w;
          const uint32_t a[4] = {q8_lo32(w0, kd[0], ko[0]), q8_lo32(w1, kd[1], ko[1]), q8_hi32(w0, kd[0], ko[0]), q8_hi32(w1, kd[1], ko[1])};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 w = lds128(q_at + (n * KST + 4 * b + k) * 512);
            if (b == 0 && k == 0) {
              mma16816_zero(s[n], a, w.x, w.y);
              mma16816_zero(part[n], a, w.z, w.w);
            } else {
              mma16816(s[n], a, w.x, w.y);
              mma16816(part[n], a, w.z, w.w);
            }
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] += part[n][i];
      bool grows = false, falls = false;
      float top[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          s[n][j] *= f[n][j];
          s[n][2 + j] *= f[n][j];
          if (masked) {
            const int to = lim[n][j], from = attn_first_key(to, p.window), key = ks + key1;
            if (key > to || key < from) s[n][j] = -CUDART_INF_F;
            if (key + 2 > to || key + 2 < from) s[n][2 + j] = -CUDART_INF_F;
          }
          top[n][j] = max_nan(s[n][j], s[n][2 + j]);
          grows |= !(top[n][j] <= m[n][j] + ATTN_SLACK);  // (or there is none)
        }
      if ((t & 3) == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t high = __ballot_sync(0xFFFFFFFFu, !(top[n][j] < m[n][j] - ATTN_FALL));  // of each column's eight lanes
            high |= high >> 16, high |= high >> 8, high |= high >> 4;
            falls |= (high & 15u) != 15u;
          }
      }
      // (the maximum is looked for only where a score is past the slack, or all of a column's are far below: votes instead of rounds of shuffles)
      if (__any_sync(0xFFFFFFFFu, grows) || falls) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float mx = fmaxf(s[n][j], s[n][2 + j]), lx = l[n][j];  // (a NaN leaves the reference where it is)
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, x));
            if (falls) {
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) lx = fmaxf(lx, __shfl_xor_sync(0xFFFFFFFFu, lx, x));
            }
            float to = m[n][j];
            if (mx > to + ATTN_SLACK) to = ceilf(mx);
            // (down only as far as leaves the sums in range: weights so far below 2^60)
            else if (falls && mx < to - ATTN_FALL && mx > -CUDART_INF_F) to = fminf(to, fmaxf(ceilf(mx), to + (float)((int)(__float_as_uint(lx) >> 23) - 187)));
            const float w = to == m[n][j] ? 1.f : exp2_rel(m[n][j], to);
            m[n][j] = to;
            l[n][j] *= w;
#pragma unroll
            for (int k = 0; k < KST; ++k) o[k][n][j] *= w, o[k][n][2 + j] *= w;
          }
      }
      if (asks && lane < 8) s_ask[group].place[lane] = next;
      // ---- weights, transposed into B fragments
      uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float e[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float ref = m[n][j] == -CUDART_INF_F ? 0.f : m[n][j];
          e[j] = exp2_approx((s[n][j] - ref) + ATTN_BIAS);  // (in this order: scores of any size)
          e[2 + j] = exp2_approx((s[n][2 + j] - ref) + ATTN_BIAS);
          l[n][j] += e[j] + e[2 + j];
        }
        split2(e[0], e[1], ph[n][0], pl[n][0]);
        split2(e[2], e[3], ph[n][1], pl[n][1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) ph[n][i] = movm(ph[n][i]), pl[n][i] = movm(pl[n][i]);
      }
      // ---- sums, from zero for every slice and added here: the tensor cores truncate, and a running sum would lose 2^-23 of itself to every slice
      const uint32_t vb = kb + SIDE;
#pragma unroll
      for (int k0 = 0; k0 < KST; k0 += 4) {
        uint32_t ab[2][2];  // scales of blocks 0 and 1, and 2 and 3, of these four: of the lane's first two keys of every 16, and of the other two
        {
          uint32_t w[4];  // of the keys 4 c .. 4 c + 3, a byte to each of the four blocks
          const uint32_t vd = sc + Sh::SCALES / 2 + 2 * c0 * nb + k0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (WHOLE) {
              w[i] = lds32(vd + i * nb);
            } else {  // (one byte after the other: those behind the head's end are the next key's)
              w[i] = 0;
#pragma unroll
              for (int b = 0; b < 4; ++b)
                if (k0 + b < nb) w[i] |= lds8(vd + i * nb + b) << (8 * b);
            }
          }
          ab[0][0] = __byte_perm(w[0], w[1], 0x5140), ab[1][0] = __byte_perm(w[0], w[1], 0x7362);
          ab[0][1] = __byte_perm(w[2], w[3], 0x5140), ab[1][1] = __byte_perm(w[2], w[3], 0x7362);
        }
#pragma unroll
        for (int k1 = 0; k1 < 4; k1 += AHEAD) {
          float sum[AHEAD][NT][4];
#pragma unroll
          for (int k = 0; k < AHEAD; k += 2) {
            uint32_t r[4];
            const int c = k1 + k + (lane >> 4), kk = lane & 15;
            ldsm2_t8(r, vb + (k0 >> 2) * SLAB + kk * 64 + ((c ^ ((kk >> 1) & 3)) << 4));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t *two = ab[(k1 + k) >> 1], d01 = __byte_perm(two[0], 0, i ? 0x3424 : 0x1404) >> 1, d23 = __byte_perm(two[1], 0, i ? 0x3424 : 0x1404) >> 1;
              uint32_t a01, a23, o01, o23;
              q8_32nds(d01, a01, o01), q8_32nds(d23, a23, o23);
              const uint32_t a[4] = {q8_lo32(r[2 * i], a01, o01), q8_lo32(r[2 * i + 1], a01, o01), q8_hi32(r[2 * i], a23, o23), q8_hi32(r[2 * i + 1], a23, o23)};
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma16816_zero(sum[k + i][n], a, pl[n][0], pl[n][1]);
                mma16816(sum[k + i][n], a, ph[n][0], ph[n][1]);
              }
            }
          }
#pragma unroll
          for (int k = 0; k < AHEAD; ++k)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) o[k0 + k1 + k][n][i] += sum[k][n][i];
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + stage);
    }
    done += tiles;

    // ---- the warps' parts of the item
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[n][j] += __shfl_xor_sync(0xFFFFFFFFu, l[n][j], x);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (m[n][j] == -CUDART_INF_F && l[n][j] != 0.f) m[n][j] = 0.f;  // nothing but NaN: a part that counts, not one without keys
    if (item >= 1 && alive) alive = wait_all(&sums_read, item - 1);  // the last item's sums have been read
    bool keys = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) keys |= m[n][0] > -CUDART_INF_F || m[n][1] > -CUDART_INF_F;
    if (lane < 4) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) s_m[warp * RB + 8 * n + c0 + j] = m[n][j], s_l[warp * RB + 8 * n + c0 + j] = l[n][j];
    }
    if (__any_sync(0xFFFFFFFFu, keys)) {  // (without keys a part's weight is 0, and its sums are not read)
      float* mine = s_o + warp * RB * PITCH + (lane >> 2);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int k = 0; k < KST; ++k) {
            float* to = mine + (8 * n + c0 + j) * PITCH + 16 * k;
            to[0] = 32.f * o[k][n][j];  // (values come as 32nds)
            to[8] = 32.f * o[k][n][2 + j];
          }
    }
    if (!alive && lane == 0) s_gave_up[item & 1] = 1;
    const bool any_odd = __syncthreads_or(odd) != 0, whole = it.whole;
    if (s_gave_up[item & 1]) {  // (all leave at the same barrier)
      if (tid == 0) atomicExch(&p.status->timeout, 10);
      attn_let_land();  // copies are in flight: they land before this shared memory is somebody else's
      return;
    }
    const AttnShare share = {it.first_cta, it.last_cta};
#pragma unroll 1
    for (int e = tid; e < it.n_rows * (HD / 4); e += THREADS) {
      const int r = e / (HD / 4), i = 4 * (e % (HD / 4));
      float M = -CUDART_INF_F, L = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) M = fmaxf(M, s_m[w * RB + r]);
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int w = 0; w < WARPS; ++w) {
        const float wt = exp2_rel(s_m[w * RB + r], M);
        L += wt * s_l[w * RB + r];
        if (wt == 0.f) continue;
        const float4 v = *reinterpret_cast<const float4*>(s_o + (w * RB + r) * PITCH + i);
        sum.x += wt * v.x, sum.y += wt * v.y, sum.z += wt * v.z, sum.w += wt * v.w;
      }
      if (whole) {
        const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
        if (i < p.hd) *reinterpret_cast<float4*>(p.out + attn_row_offset(p, it.row0, it.head, r, p.out_stride) + i) = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
      } else {
        const size_t to = (size_t)attn_slot(blockIdx.x, share) * RB + r;
        __stcg(reinterpret_cast<float4*>(p.part + to * HD + i), sum);
        if (i == 0) __stcg(p.part_ml + to, make_float2(M, L));
      }
      if (i == 0) s_weight[r] = L;
    }
    if (any_odd) {  // some row may see values that are no numbers
      __threadfence();
      __syncthreads();
      const int r = lane < it.n_rows ? lane : 0;
      attn_odd_blocks(p, it.s, it.head, it.key0, it.key0 + (tiles << Sh::LOG2_TILE), lane < it.n_rows && s_weight[r] == s_weight[r], it.pos0 + attn_row_token(p, r), warp, WARPS,
                      whole ? p.out + attn_row_offset(p, it.row0, it.head, r, p.out_stride) : p.part + ((size_t)attn_slot(blockIdx.x, share) * RB + r) * HD);
    }
    if (tid == 0 && !whole && s_parts < 2) s_part[s_parts++] = it;
    __syncwarp();
    if (lane == 0) mbar_arrive(&sums_read);
    if (warp == WARPS - 1 && s_described < N) {  // the item after the next, in this one's place
      if (alive) alive = wait_all(&sums_read, item);
      if (lane == 0) s_walk.next(p);
      __syncwarp();
      q8_item<HD, NT>(p, s_start, s_walk, s_item + (item & 1), s_q + (item & 1) * (Sh::Q / 16), s_factor[item & 1]);
      __syncwarp();
      if (lane == 0) s_described += s_item[item & 1].tiles;
      __syncwarp();
      if (lane == 0) mbar_arrive(item_ready + (item & 1));
    }
  }
  if (__syncthreads_or(!alive)) {
    if (tid == 0) atomicExch(&p.status->timeout, 10);
    attn_let_land();
    return;
  }
  // ---- items that other CTAs have tiles of, the first and the last at most: whoever comes last joins them
#pragma unroll 1
  for (int i = 0; i < s_parts; ++i) {
    const Q8Item& it = s_part[i];
    if (attn_arrive(p, it.first_cta, it.last_cta, &s_last, tid == 0, 0, THREADS)) {
      const AttnShare share = {it.first_cta, it.last_cta};
#pragma unroll 1
      for (int r = warp; r < it.n_rows; r += WARPS) attn_join_row<HD>(p, share, RB, r, p.out + attn_row_offset(p, it.row0, it.head, r, p.out_stride));
    }
  }
}

// Codes of `box` keys of a head, 64 values wide.
bool attn_codes_map(CUtensorMap* tm, const uint8_t* base, const AttnParams& p, int box) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)p.hd, (cuuint64_t)p.page_size, (cuuint64_t)p.n_kv, (cuuint64_t)p.n_pages};
  const cuuint64_t strides[3] = {p.row_pitch, p.head_pitch, p.page_pitch};
  const cuuint32_t sizes[4] = {64, (cuuint32_t)box, 1, 1}, estr[4] = {1, 1, 1, 1};
  return enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<uint8_t*>(base), dims, strides, sizes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, int NT, bool WHOLE>
int32_t run_rows_q8(infr_cuda_ctx* ctx, const AttnParams& p) {
  using Sh = Q8Shape<HD, NT>;
  int granule = Sh::KEYS;
  while (p.page_size % granule) granule >>= 1;
  CUtensorMap km, vm;
  if (!attn_codes_map(&km, p.kq, p, granule) || !attn_codes_map(&vm, p.vq, p, granule)) return fail(ctx, INFR_CUDA_ERR_CUDA, "attention: cuTensorMapEncodeTiled failed");
  cudaError_t e = ensure_smem(reinterpret_cast<const void*>(&k_attn_rows_q8<HD, NT, WHOLE>), Sh::SMEM);
  if (e == cudaSuccess)
    e = launch_ex(k_attn_rows_q8<HD, NT, WHOLE>, dim3(ctx->sm_count < ATTN_MAX_CTAS ? ctx->sm_count : ATTN_MAX_CTAS), dim3(Sh::THREADS), Sh::SMEM, ctx->stream, true, km, vm, p, granule);
  if (e != cudaSuccess) return check_cuda(ctx, e, "k_attn_rows_q8 launch");
  ctx->launches += 1;
  return check_cuda(ctx, cudaGetLastError(), "k_attn_rows_q8 launch");
}

template <int HD>
int32_t run_rows_q8_of(infr_cuda_ctx* ctx, const AttnParams& p, int nt) {
  if constexpr (HD <= 128)
    if (nt == 2) return p.hd == HD ? run_rows_q8<HD, 2, true>(ctx, p) : run_rows_q8<HD, 2, false>(ctx, p);
  return p.hd == HD ? run_rows_q8<HD, 1, true>(ctx, p) : run_rows_q8<HD, 1, false>(ctx, p);
}

}  // namespace

// max_rows: see launch_attn_rows.  Heads wider than 128 have items of eight rows (attn_q8_rows_limit): of sixteen the sums do not fit beside the tiles.
int32_t launch_attn_rows_q8(infr_cuda_ctx* ctx, AttnParams p, int max_rows) {
  const int nt = p.hd > 128 || (p.g <= 8 && max_rows <= 8) ? 1 : 2;
  p.tb = 8 * nt / p.g;
  if (p.hd <= 64) return run_rows_q8_of<64>(ctx, p, nt);
  if (p.hd <= 128) return run_rows_q8_of<128>(ctx, p, nt);
  if (p.hd <= 192) return run_rows_q8_of<192>(ctx, p, nt);
  return run_rows_q8_of<256>(ctx, p, nt);
}

}  // namespace infr
