// Attention of a few rows per (sequence, kv head): single tokens and speculative windows, up to 16 rows (tokens x query heads of a kv head)
// to an item.  One pass over the keys: what bounds it is reading K and V once.
//
// A CTA takes key tiles of 16 keys per warp; each warp streams its own 16-key slices of K and V through a ring of its own (tiled copies, no
// barrier between warps) and keeps its own running maximum, weight and sums, joined at the item's end.  Both products are transposed so that
// the tensor cores' 16 rows are keys or head values, and the 8 columns the rows of the item:
//   S^T[16 keys, 8 rows] = K[16, hd] q^T[hd, 8],    O^T[hd, 8 rows] += V^T[hd, 16 keys] P^T[16 keys, 8 rows]
// The scores' fragments become P^T's through a transposition of 8 x 8 matrices in registers.  q and P go in as two f16 pieces each (22 bits;
// q scaled by a power of two per row so that f16's range holds it): f32 results stay f32 results.
//
// Measured (us; K and V at the measured 6538 GB/s): 64 tokens over 700 - 8000 keys each (32 / 4 heads of 128, 429 MB) 85 (66), one token over
// 131072 keys (268 MB) 60 (41), 16 tokens over up to 16000 keys (16 / 2 heads of 256, 257 MB) 59 (39), one token over 513 keys 10.8: what is
// left is the kernel's two ends, about 3 us until the plan of the call is known, 3 until the first tiles are there and 3 for the join of
// an item's parts; and, with heads of 256, a warp's own chain from tile to tile.  Nine to sixteen rows of heads of 192 and 256 do not fit the registers: 107 and 194
// words a thread are spilled.
#include "attn.cuh"
#include "kv_q8.cuh"

namespace infr {
namespace {

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// Two 16 x 16 matrices of bytes transposed: r[0], r[1] are rows lane / 4 and 8 more of the first, columns 4 (lane % 4) .. + 3.
__device__ __forceinline__ void ldsm2_t8(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movm(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
constexpr int ROWS_EXTRA = 3;  // tiles' time that an item's beginning and end take (64 streams: 1 93.7, 3 86.1, 6 87.0 us)

template <int HD, int NT, bool Q8>
struct RowsShape {
  static constexpr int WARPS = 8, THREADS = WARPS * 32, RB = 8 * NT;
  static constexpr int LOG2_TILE = 7;              // 16 keys a warp
  static constexpr int SIDE = 16 * HD * (Q8 ? 1 : 2);  // bytes of 16 keys of K, or of V
  static constexpr int SCALES = Q8 ? 2 * HD : 0;       // bytes of a unit's scales, which lie apart
  // A unit of the ring is both where eight warps' rings hold two of them or more, else (heads wider than 128) one of the two: K's place is
  // asked for again while V is used.  (Apart, heads of 128 lose: 93 -> 106 us for 64 streams.)
  static constexpr bool PAIRED = Q8 || HD <= 128;
  static constexpr int UNIT = PAIRED ? 2 * SIDE : SIDE;
  static constexpr int PITCH = HD + 4;             // words: the fragments' columns fall on different banks
  static constexpr int SLOTS = HD <= 128 ? WARPS : WARPS / 2;  // wide heads: half of the warps add theirs to the others' first
  static constexpr int MERGE = SLOTS * RB * PITCH * 4, STATS = 2 * WARPS * RB * 4;
  static constexpr int FIT = (232448 - 1024 - 1024 - MERGE - STATS) / (WARPS * (UNIT + SCALES));
  static constexpr int MOST = Q8 ? 8 : 6, UNITS = FIT > MOST ? MOST : FIT;
  static constexpr int SMEM = 1024 + WARPS * UNITS * (UNIT + SCALES) + MERGE + STATS + WARPS * UNITS * 8;
  static_assert(WARPS * UNITS * UNIT >= 16 * ATTN_MAX_SEQ + 4, "what is known of the sequences fits where the keys go later");
};

// Pages of 8 bits: columns of rows of the item, the part of it that lies here, where 16 values of V that a row sees are not numbers, become NaN.  All of
// the warp's lanes take part, a row to each of the first ones; `active`: not NaN already.  Blocks of 16 from block0 on, every `step`-th.
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

// Q8: pages of 8 bits.  The tensor cores' inner dimensions may go in any order that both operands have, so a lane takes for K 16 neighbouring values of a key
// at once (one scale, one 16-byte word: four steps of the product), and the 16 keys stand in the order in which a transposing load of bytes gives V's:
// row i of the scores is key 4 (i / 2) + i % 2 of the slice, row 8 + i two behind it.
template <int HD, int NT, bool Q8>
__global__ void __launch_bounds__(RowsShape<HD, NT, Q8>::THREADS, 1)
    k_attn_rows(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ AttnParams p) {
  using Sh = RowsShape<HD, NT, Q8>;
  constexpr int WARPS = Sh::WARPS, THREADS = Sh::THREADS, RB = Sh::RB, UNITS = Sh::UNITS, UNIT = Sh::UNIT, SIDE = Sh::SIDE, PITCH = Sh::PITCH, SLOTS = Sh::SLOTS;
  constexpr int SLABS = HD / 64, KST = HD / 16;
  constexpr int AHEAD = 4;  // sums under way (one or two at a time 60.5 us for 16 streams of heads of 256, so 58.8)
  static_assert(NT * KST * 512 <= Sh::MERGE, "q's pieces lie where the sums go");
  extern __shared__ unsigned char smem_raw[];
  __shared__ long long s_scan[WARPS];
  __shared__ AttnStart s_start;
  __shared__ int s_last;
  __shared__ float s_weight[RB], s_factor[RB];
  unsigned char* ring_all = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* scales = ring_all + WARPS * UNITS * UNIT + (threadIdx.x >> 5) * UNITS * Sh::SCALES;
  float* s_o = reinterpret_cast<float*>(ring_all + WARPS * UNITS * (UNIT + Sh::SCALES));
  uint4* s_q = reinterpret_cast<uint4*>(s_o);  // [NT][KST][32]
  float* s_m = s_o + SLOTS * RB * PITCH;
  float* s_l = s_m + WARPS * RB;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_l + WARPS * RB);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* ring = ring_all + warp * UNITS * UNIT;
  uint64_t* full = bars + warp * UNITS;

  pdl_trigger();  // the next kernel may take the SMs that this one leaves free, and do what needs no input of its
  if (lane == 0)
    for (int i = 0; i < UNITS; ++i) mbar_init(full + i, 1);
  mbar_fence_init();
  pdl_wait();
  attn_plan<THREADS, Sh::LOG2_TILE, ROWS_EXTRA, 0>(p, reinterpret_cast<int*>(ring_all), s_scan, &s_start);
  const AttnStart st = s_start;
  if (st.until == st.before) return;
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the plan's words lay where the copies go
  __syncthreads();

  const bool packed = p.page_table == nullptr;
  // ---- what the warp asks for: K and V of its slices of the CTA's tiles, one after the other, as many as its ring holds
  AttnCursor<Sh::LOG2_TILE, ROWS_EXTRA> ahead;
  ahead.start(p, st);
  AttnCursor<Sh::LOG2_TILE, ROWS_EXTRA> cur = ahead;  // what it works on
  int at = ahead.first(st);             // tile of its item to look at next
  int a_key = -1, a_page = 0, a_y = 0;  // first key of the slice to ask for (-1: none left), its page, its place there
  uint32_t asked = 0;
  auto find = [&]() {                   // the next tile of which this warp has keys
#pragma unroll 1
    while (ahead.ub < st.u1) {
      if (at >= ahead.end(st)) {
        ahead.next(p);
        at = 0;
        continue;
      }
      const int ks = ((ahead.blk.tile0 + at) << Sh::LOG2_TILE) + warp * 16;
      if (ks < ahead.blk.hi && ks + 16 > ahead.blk.lo) {
        a_key = ks;
        a_y = ahead.seq.q0 + ks;
        if (!packed) {
          const int page = attn_page_of(p, ks);
          a_page = attn_page_entry(p, ahead.s, page);
          a_y = ks - page * p.page_size;
        }
        return;
      }
      ++at;
    }
    a_key = -1;
  };
  auto ask_next = [&]() {  // K and V in turn, or both
    if (a_key < 0) return;
    if (lane == 0) {
      const int at = asked % UNITS;
      unsigned char* dst = ring + at * UNIT;
      mbar_arrive_expect_tx(full + at, Q8 ? UNIT + 2 * p.hd : UNIT);
      const int y = a_y, w = packed ? 0 : attn_page_checked(p, a_page);
      if constexpr (Q8) {
        const size_t first = ((size_t)w * p.page_pitch + (size_t)ahead.head * p.head_pitch + (size_t)y * p.row_pitch) / 16;
        bulk_g2s(scales + at * Sh::SCALES, p.ks + first, p.hd, full + at);  // (16 keys' hd / 16 bytes)
        bulk_g2s(scales + at * Sh::SCALES + HD, p.vs + first, p.hd, full + at);
      }
      const CUtensorMap* map = Sh::PAIRED || !(asked & 1) ? &kmap : &vmap;
#pragma unroll
      for (int s = 0; s < SLABS; ++s) {
        tma_load_4d(dst + s * (SIDE / SLABS), map, 64 * s, y, ahead.head, w, full + at);
        if (Sh::PAIRED) tma_load_4d(dst + SIDE + s * (SIDE / SLABS), &vmap, 64 * s, y, ahead.head, w, full + at);
      }
    }
    ++asked;
    if (Sh::PAIRED || !(asked & 1)) {
      ++at;
      find();
    }
  };
  find();
#pragma unroll 1
  for (int i = 0; i < UNITS; ++i) ask_next();

  uint32_t used = 0;
  bool alive = true;
  const int c0 = 2 * (lane & 3);  // this thread's columns (rows of the item): c0, c0 + 1 of every eight
  const int key1 = Q8 ? 4 * (lane >> 3) + ((lane >> 2) & 1) : lane >> 2;  // and its keys of a slice: this one and
  constexpr int NEXT = Q8 ? 2 : 8;                                        // the one so far behind it
  const int nb = p.hd / 16;       // Q8: scales of a key
  long long left = st.until - st.before;  // tiles
#pragma unroll 1
  for (;; cur.next(p)) {
    const AttnBlock& blk = cur.blk;
    const int first_tile = cur.first(st), end_tile = cur.end(st), n_rows = blk.nt * p.g;

    // ---- q: B fragments of q^T, rows scaled by a power of two, as two f16 pieces, put down by one warp per eight rows where the sums go
    // at the item's end (in every warp's registers they took the products' room: heads of 256 71 us instead of 60 for 16 streams, of 128
    // 93 instead of 90 for 64)
    float f[NT][2];  // of the thread's columns: score -> log2 units
    int lim[NT][2];  // and the last key their row sees
    __syncthreads();  // the last item's sums have been read
    if (warp < NT) {
      const int r = 8 * warp + (lane >> 2);
      const bool has = r < n_rows;
      const float* src = p.q + attn_row_offset(p, cur.seq.q0 + blk.t0, cur.head, has ? r : 0, p.q_stride);
      float2 v[KST][2];
      float big = 0.f;
#pragma unroll
      for (int k = 0; k < KST; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int i = Q8 ? 64 * (k >> 2) + 8 * c0 + 4 * (k & 3) + 2 * j : 16 * k + 8 * j + c0;
          v[k][j] = has && i < p.hd ? __ldcg(reinterpret_cast<const float2*>(src + i)) : make_float2(0.f, 0.f);
          big = fmaxf(big, fmaxf(fabsf(v[k][j].x), fabsf(v[k][j].y)));
        }
      big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, 2));
      float down, up;
      attn_row_scale(big, down, up);
#pragma unroll
      for (int k = 0; k < KST; ++k) {
        uint4 w;
        split2(v[k][0].x * down, v[k][0].y * down, w.x, w.z);
        split2(v[k][1].x * down, v[k][1].y * down, w.y, w.w);
        s_q[(warp * KST + k) * 32 + lane] = w;
      }
      if ((lane & 3) == 0) s_factor[r] = up * p.scale_log2;
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int rr = 8 * n + c0 + j;
        f[n][j] = s_factor[rr];
        lim[n][j] = cur.seq.past + blk.t0 + (rr < n_rows ? attn_row_token(p, rr) : blk.nt - 1);
      }
    const int full_hi = attn_full_hi(cur.seq, blk), full_lo = attn_full_lo(cur.seq, blk, p.window);

    float o[KST][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int k = 0; k < KST; ++k)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[k][n][i] = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -CUDART_INF_F, l[n][0] = l[n][1] = 0.f;

    bool odd = false;  // values that are not finite were left out
#pragma unroll 1
    for (int t = first_tile; t < end_tile; ++t) {
      const int ks = ((blk.tile0 + t) << Sh::LOG2_TILE) + warp * 16;
      if (ks >= blk.hi || ks + 16 <= blk.lo) continue;
      if (alive) {
        alive = wait_all(full + used % UNITS, used / UNITS);
        if (!alive && lane == 0) atomicExch(&p.status->timeout, 10);
      }
      if (alive) {
        const uint32_t kb = smem_u32(ring + (used % UNITS) * UNIT);
        const int i4 = lane >> 3, r8 = lane & 7;
        // ---- scores: pieces and even and odd steps apart, four chains of products instead of one
        float s[NT][4], part[NT][3][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][i] = part[n][0][i] = part[n][1][i] = part[n][2][i] = 0.f;
        uint4 kw[2];     // Q8: this lane's 16 values of both keys
        uint32_t kd[2];  // and their scales
#pragma unroll
        for (int k = 0; k < KST; ++k) {
          uint32_t a[4];
          if constexpr (Q8) {
            if ((k & 3) == 0) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int key = key1 + NEXT * h, b = k + (lane & 3);
                const unsigned char* row = ring + (used % UNITS) * UNIT + (k >> 2) * 1024 + key * 64;
                kw[h] = *reinterpret_cast<const uint4*>(row + (((lane & 3) ^ ((key >> 1) & 3)) << 4));
                // (behind the head's end q is 0 and the codes' values are finite)
                kd[h] = q8_scale_pair(HD % 64 == 0 && b >= nb ? 0u : scales[(used % UNITS) * Sh::SCALES + key * nb + b]);
              }
            }
            const uint32_t w0 = (k & 3) == 0 ? kw[0].x : (k & 3) == 1 ? kw[0].y : (k & 3) == 2 ? kw[0].z : kw[0].w;
            const uint32_t w1 = (k & 3) == 0 ? kw[1].x : (k & 3) == 1 ? kw[1].y : (k & 3) == 2 ? kw[1].z : kw[1].w;
            a[0] = q8_lo(w0, kd[0]), a[1] = q8_lo(w1, kd[1]), a[2] = q8_hi(w0, kd[0]), a[3] = q8_hi(w1, kd[1]);
          } else
          ldsm4(a, kb + (k >> 2) * 2048 + ((i4 & 1) * 8 + r8) * 128 + (((2 * (k & 3) + (i4 >> 1)) ^ r8) << 4));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 w = s_q[(n * KST + k) * 32 + lane];
            mma16816(k & 1 ? part[n][0] : s[n], a, w.x, w.y);
            mma16816(k & 1 ? part[n][2] : part[n][1], a, w.z, w.w);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][i] = (s[n][i] + part[n][0][i]) + (part[n][1][i] + part[n][2][i]);
        if (!Sh::PAIRED) {
          __syncwarp();
          ++used;
          ask_next();
        }
        const bool masked = ks + 16 > full_hi || ks < full_lo;
        const int key = ks + key1;
        bool grows = false, falls = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            s[n][j] *= f[n][j];
            s[n][2 + j] *= f[n][j];
            if (masked) {
              const int to = lim[n][j], from = attn_first_key(to, p.window);
              if (key > to || key < from) s[n][j] = -CUDART_INF_F;
              if (key + NEXT > to || key + NEXT < from) s[n][2 + j] = -CUDART_INF_F;
            }
            grows |= !(max_nan(s[n][j], s[n][2 + j]) <= m[n][j] + ATTN_SLACK);  // (or there is none)
          }
        if ((t & 3) == 0) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t high = __ballot_sync(0xFFFFFFFFu, fmaxf(s[n][j], s[n][2 + j]) >= m[n][j] - ATTN_FALL);  // of each column's eight lanes
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
              if (!Q8 && l[n][j] == l[n][j] && 8 * n + c0 + j < n_rows) {  // (a row that is NaN already stays that)
#pragma unroll
                for (int i = 0; i < 4; i += 2)
                  if (s[n][i + j] != s[n][i + j])
                    s[n][i + j] = attn_odd_score(p, cur.s, cur.seq.q0, cur.head, key + 4 * i,
                                                 p.q + attn_row_offset(p, cur.seq.q0 + blk.t0, cur.head, 8 * n + c0 + j, p.q_stride));
              }
              float mx = fmaxf(s[n][j], s[n][2 + j]), lx = l[n][j];
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
        // ---- sums, from zero for every slice and added here: the tensor cores truncate, and a running sum lost 2^-23 of itself to every slice (65536 keys
        // by eight warps: 5.7e-5 of a result of one sign, now 4e-7).  Where some row does not see some key, 0 x value must be 0 whatever the value: keys that no row sees become zeros, and
        // so do values that are not finite, which wait for the item's end.
        if (!Sh::PAIRED) {
          alive = wait_all(full + used % UNITS, used / UNITS);
          if (!alive) {
            if (lane == 0) atomicExch(&p.status->timeout, 10);
            continue;
          }
        }
        unsigned char* vs = ring + (used % UNITS) * UNIT + (Sh::PAIRED ? SIDE : 0);
        const uint32_t vb = smem_u32(vs);
        if (!Q8 && masked) {
#pragma unroll 1
          for (int e = lane; e < 16 * SLABS * 8; e += 32) {  // 16-byte words, 128 bytes of a key after the other
            const int kk = ks + ((e >> 3) & 15);
            uint4* w = reinterpret_cast<uint4*>(vs) + e;
            const uint4 x = *w;
            uint4 y = make_uint4(only_finite(x.x), only_finite(x.y), only_finite(x.z), only_finite(x.w));
            if (kk >= blk.hi || kk < blk.lo) y = make_uint4(0, 0, 0, 0);
            else odd |= x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w;
            *w = y;
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (ahead of the slot's next copy)
          __syncwarp();
        }
#pragma unroll
        for (int k0 = 0; k0 < KST; k0 += AHEAD) {
          uint32_t a[AHEAD][4];
          float sum[AHEAD][NT][4];
          if constexpr (Q8) {
            // scales of this lane's keys 4 c .. 4 c + 3 and the four blocks, a word to each key; those that are no numbers count as zeros and wait
            // for the item's end
            static_assert(AHEAD == 4, "a word of scales");
            const unsigned char* vd = scales + (used % UNITS) * Sh::SCALES + HD + 2 * c0 * nb + k0;
            uint32_t w[4], bad = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if ((nb & 3) == 0) {
                w[i] = k0 < nb ? *reinterpret_cast<const uint32_t*>(vd + i * nb) : 0u;
              } else {  // (one byte after the other: those behind the head's end are the next key's)
                w[i] = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b)
                  if (k0 + b < nb) w[i] |= (uint32_t)vd[i * nb + b] << (8 * b);
              }
              bad |= w[i] & (w[i] << 1);
            }
            if (bad & 0x80808080u) {
              odd = true;
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] &= ~(((w[i] & (w[i] << 1) & 0x80808080u) >> 7) * 0xFFu);
            }
            uint32_t ab[2][2];  // blocks 0 and 1, and 2 and 3: of the first two keys, of the other two
            ab[0][0] = __byte_perm(w[0], w[1], 0x5140), ab[1][0] = __byte_perm(w[0], w[1], 0x7362);
            ab[0][1] = __byte_perm(w[2], w[3], 0x5140), ab[1][1] = __byte_perm(w[2], w[3], 0x7362);
#pragma unroll
            for (int k = 0; k < AHEAD; k += 2) {
              uint32_t r[4];
              const int c = k + (lane >> 4), kk = lane & 15;
              ldsm2_t8(r, vb + (k0 >> 2) * 1024 + kk * 64 + ((c ^ ((kk >> 1) & 3)) << 4));
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t d01 = __byte_perm(ab[k >> 1][0], 0, i ? 0x3424 : 0x1404) >> 1, d23 = __byte_perm(ab[k >> 1][1], 0, i ? 0x3424 : 0x1404) >> 1;
                a[k + i][0] = q8_lo(r[2 * i], d01), a[k + i][1] = q8_lo(r[2 * i + 1], d01);
                a[k + i][2] = q8_hi(r[2 * i], d23), a[k + i][3] = q8_hi(r[2 * i + 1], d23);
              }
            }
          }
#pragma unroll
          for (int k = 0; k < AHEAD; ++k) {
            if constexpr (!Q8) ldsm4_t(a[k], vb + ((k0 + k) >> 2) * 2048 + ((i4 >> 1) * 8 + r8) * 128 + (((2 * ((k0 + k) & 3) + (i4 & 1)) ^ r8) << 4));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
              for (int i = 0; i < 4; ++i) sum[k][n][i] = 0.f;
              mma16816(sum[k][n], a[k], pl[n][0], pl[n][1]);
            }
          }
#pragma unroll
          for (int k = 0; k < AHEAD; ++k)
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816(sum[k][n], a[k], ph[n][0], ph[n][1]);
#pragma unroll
          for (int k = 0; k < AHEAD; ++k)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) o[k0 + k][n][i] += sum[k][n][i];
        }
        __syncwarp();
        ++used;
        ask_next();
      }
    }

    if constexpr (!Q8) {
#pragma unroll
      for (int k = 0; k < KST; ++k)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) odd |= !(fabsf(o[k][n][i]) < CUDART_INF_F);
    }

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
    __syncthreads();  // the last item's parts have been read
    // one half of the warps puts its sums down, the other adds its own to them, each brought to the higher maximum.  (No part is left out because its
    // weight has underflowed: what is not finite in it stays that, here as NaN, and is put right below)
    if (lane < 4) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) s_m[warp * RB + 8 * n + c0 + j] = m[n][j], s_l[warp * RB + 8 * n + c0 + j] = l[n][j];
    }
    float* mine = s_o + (warp & (SLOTS - 1)) * RB * PITCH + (lane >> 2);
    if (SLOTS == WARPS || warp >= SLOTS) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int k = 0; k < KST; ++k) {
            float* at = mine + (8 * n + c0 + j) * PITCH + 16 * k;
            at[0] = o[k][n][j];
            at[8] = o[k][n][2 + j];
          }
    }
    if constexpr (SLOTS < WARPS) __syncthreads();
    if (SLOTS < WARPS && warp < SLOTS) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float other = s_m[(warp + SLOTS) % WARPS * RB + 8 * n + c0 + j], to = fmaxf(m[n][j], other);
          const float a = exp2_rel(m[n][j], to), b = exp2_rel(other, to);
#pragma unroll
          for (int k = 0; k < KST; ++k) {
            float* at = mine + (8 * n + c0 + j) * PITCH + 16 * k;
            at[0] = a * o[k][n][j] + b * at[0];
            at[8] = a * o[k][n][2 + j] + b * at[8];
          }
        }
    }
    const bool any_odd = __syncthreads_or(odd) != 0;
    const bool whole = first_tile == 0 && end_tile == blk.ntile;
    AttnShare share = {0, 0};
    if (!whole) share = attn_share(cur.ub, blk.ntile, st);
    auto store = [&](int r, int i, float4 v) {
      *reinterpret_cast<float4*>(p.out + attn_row_offset(p, cur.seq.q0 + blk.t0, cur.head, r, p.out_stride) + i) = v;
    };
    for (int e = tid; e < RB * (HD / 4); e += THREADS) {
      const int r = e / (HD / 4), i = 4 * (e % (HD / 4));
      if (r >= n_rows) continue;
      float M = -CUDART_INF_F, L = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) M = fmaxf(M, s_m[w * RB + r]);
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < SLOTS; ++w) {
        constexpr bool two = SLOTS < WARPS;  // this slot holds two warps' sums
        const float m0 = s_m[w * RB + r], m1 = two ? s_m[(w + SLOTS) % WARPS * RB + r] : -CUDART_INF_F;
        const float wt = exp2_rel(fmaxf(m0, m1), M);
        const float4 v = *reinterpret_cast<const float4*>(s_o + (w * RB + r) * PITCH + i);
        L += exp2_rel(m0, M) * s_l[w * RB + r];
        if (two) L += exp2_rel(m1, M) * s_l[(w + SLOTS) % WARPS * RB + r];
        sum.x += wt * v.x, sum.y += wt * v.y, sum.z += wt * v.z, sum.w += wt * v.w;

      }
      if (whole) {
        const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
        if (i < p.hd) store(r, i, make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv));
      } else {
        const size_t at = (size_t)attn_slot(blockIdx.x, share) * RB + r;
        __stcg(reinterpret_cast<float4*>(p.part + at * HD + i), sum);
        if (i == 0) __stcg(p.part_ml + at, make_float2(M, L));
      }
      if (i == 0) s_weight[r] = L;
    }
    if (any_odd) {  // some value that a row sees may not be finite: put together by itself
      __threadfence();
      __syncthreads();
      const int r = lane < n_rows ? lane : 0;
      if constexpr (Q8) {
        attn_odd_blocks(p, cur.s, cur.head, (blk.tile0 + first_tile) << Sh::LOG2_TILE, (blk.tile0 + end_tile) << Sh::LOG2_TILE, lane < n_rows && s_weight[r] == s_weight[r],
                        cur.seq.past + blk.t0 + attn_row_token(p, r), warp, WARPS,
                        whole ? p.out + attn_row_offset(p, cur.seq.q0 + blk.t0, cur.head, r, p.out_stride) : p.part + ((size_t)attn_slot(blockIdx.x, share) * RB + r) * HD);
      } else
#pragma unroll 1
      for (int col0 = 32 * warp; col0 < p.hd; col0 += 32 * WARPS)
        attn_odd_values(p, cur.s, cur.seq.q0, cur.head, (blk.tile0 + first_tile) << Sh::LOG2_TILE, (blk.tile0 + end_tile) << Sh::LOG2_TILE, 1 << Sh::LOG2_TILE, full_lo,
                        full_hi, lane < n_rows && s_weight[r] == s_weight[r], cur.seq.past + blk.t0 + attn_row_token(p, r), col0, 32,
                        (whole ? p.out + attn_row_offset(p, cur.seq.q0 + blk.t0, cur.head, r, p.out_stride) : p.part + ((size_t)attn_slot(blockIdx.x, share) * RB + r) * HD) + col0);
    }
    if (!whole && attn_arrive(p, share.first, share.last, &s_last, tid == 0, 0, THREADS)) {
#pragma unroll 1
      for (int r = warp; r < n_rows; r += WARPS)
        attn_join_row<HD>(p, share, RB, r, p.out + attn_row_offset(p, cur.seq.q0 + blk.t0, cur.head, r, p.out_stride));
    }
    left -= end_tile - first_tile;
    if (left <= 0) break;
  }
  // a warp that gave up has copies in flight: they land before its shared memory is somebody else's
  if (!alive)
    for (; used < asked; ++used) attn_wait(full + used % UNITS, used / UNITS);
}

template <int HD, int NT, bool Q8>
cudaError_t run_rows(infr_cuda_ctx* ctx, const CUtensorMap& km, const CUtensorMap& vm, const AttnParams& p) {
  using Sh = RowsShape<HD, NT, Q8>;
  const cudaError_t e = ensure_smem(reinterpret_cast<const void*>(&k_attn_rows<HD, NT, Q8>), Sh::SMEM);
  if (e != cudaSuccess) return e;
  return launch_ex(k_attn_rows<HD, NT, Q8>, dim3(ctx->sm_count < ATTN_MAX_CTAS ? ctx->sm_count : ATTN_MAX_CTAS), dim3(Sh::THREADS), Sh::SMEM, ctx->stream, true, km, vm, p);
}

template <int HD>
cudaError_t run_rows_of(infr_cuda_ctx* ctx, const CUtensorMap& km, const CUtensorMap& vm, const AttnParams& p, int nt) {
  if (p.kq != nullptr) return nt == 1 ? run_rows<HD, 1, true>(ctx, km, vm, p) : run_rows<HD, 2, true>(ctx, km, vm, p);
  return nt == 1 ? run_rows<HD, 1, false>(ctx, km, vm, p) : run_rows<HD, 2, false>(ctx, km, vm, p);
}

// Codes of 16 keys of a head, 64 values wide.
bool attn_codes_map(CUtensorMap* tm, const uint8_t* base, const AttnParams& p) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)p.hd, (cuuint64_t)p.page_size, (cuuint64_t)p.n_kv, (cuuint64_t)p.n_pages};
  const cuuint64_t strides[3] = {p.row_pitch, p.head_pitch, p.page_pitch};
  const cuuint32_t box[4] = {64, 16, 1, 1}, estr[4] = {1, 1, 1, 1};
  return enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<uint8_t*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

bool attn_cache_map(CUtensorMap* tm, const __half* base, const AttnParams& p, int box_rows) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (!enc) return false;
  const bool packed = p.page_table == nullptr;
  const cuuint64_t dims[4] = {(cuuint64_t)p.hd, (cuuint64_t)(packed ? p.rows : p.page_size), (cuuint64_t)p.n_kv, (cuuint64_t)(packed ? 1 : p.n_pages)};
  const cuuint64_t strides[3] = {p.row_pitch * 2, p.head_pitch * 2, p.page_pitch * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, estr[4] = {1, 1, 1, 1};
  return enc(tm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<__half*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// max_rows: rows (tokens x heads of a kv head) that a sequence's new tokens make at most, as far as the caller knows; longer ones are
// cut into more items.
int32_t launch_attn_rows(infr_cuda_ctx* ctx, AttnParams p, const __half* k, int max_rows) {
  p.k = k;
  CUtensorMap km, vm;
  if (p.kq != nullptr ? !attn_codes_map(&km, p.kq, p) || !attn_codes_map(&vm, p.vq, p) : !attn_cache_map(&km, k, p, 16) || !attn_cache_map(&vm, p.v, p, 16)) return fail(ctx, INFR_CUDA_ERR_CUDA, "attention: cuTensorMapEncodeTiled failed");
  const int nt = p.g <= 8 && max_rows <= 8 ? 1 : 2;
  p.tb = 8 * nt / p.g;
  cudaError_t e;
  if (p.hd <= 64) e = run_rows_of<64>(ctx, km, vm, p, nt);
  else if (p.hd <= 128) e = run_rows_of<128>(ctx, km, vm, p, nt);
  else if (p.hd <= 192) e = run_rows_of<192>(ctx, km, vm, p, nt);
  else e = run_rows_of<256>(ctx, km, vm, p, nt);
  if (e != cudaSuccess) return check_cuda(ctx, e, "k_attn_rows launch");
  ctx->launches += 1;
  return check_cuda(ctx, cudaGetLastError(), "k_attn_rows launch");
}

}  // namespace infr
