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

namespace infr {
namespace {

constexpr int ROWS_EXTRA = 3;  // tiles' time that an item's beginning and end take (64 streams: 1 93.7, 3 86.1, 6 87.0 us)

template <int HD, int NT>
struct RowsShape {
  static constexpr int WARPS = 8, THREADS = WARPS * 32, RB = 8 * NT;
  static constexpr int LOG2_TILE = 7;              // 16 keys a warp
  static constexpr int SIDE = 16 * HD * 2;         // bytes of 16 keys of K, or of V
  // A unit of the ring is both where eight warps' rings hold two of them or more, else (heads wider than 128) one of the two: K's place is
  // asked for again while V is used.  (Apart, heads of 128 lose: 93 -> 106 us for 64 streams.)
  static constexpr bool PAIRED = HD <= 128;
  static constexpr int UNIT = PAIRED ? 2 * SIDE : SIDE;
  static constexpr int PITCH = HD + 4;             // words: the fragments' columns fall on different banks
  static constexpr int SLOTS = PAIRED ? WARPS : WARPS / 2;  // wide heads: half of the warps add theirs to the others' first
  static constexpr int MERGE = SLOTS * RB * PITCH * 4, STATS = 2 * WARPS * RB * 4;
  static constexpr int FIT = (232448 - 1024 - 1024 - MERGE - STATS) / (WARPS * UNIT);
  static constexpr int UNITS = FIT > 6 ? 6 : FIT;
  static constexpr int SMEM = 1024 + WARPS * UNITS * UNIT + MERGE + STATS + WARPS * UNITS * 8;
};

template <int HD, int NT>
__global__ void __launch_bounds__(RowsShape<HD, NT>::THREADS, 1)
    k_attn_rows(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ AttnParams p) {
  using Sh = RowsShape<HD, NT>;
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
  float* s_o = reinterpret_cast<float*>(ring_all + WARPS * UNITS * UNIT);
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
      mbar_arrive_expect_tx(full + at, UNIT);
      const int y = a_y, w = packed ? 0 : attn_page_checked(p, a_page);
      const CUtensorMap* map = Sh::PAIRED || !(asked & 1) ? &kmap : &vmap;
#pragma unroll
      for (int s = 0; s < SLABS; ++s) {
        tma_load_4d(dst + s * 2048, map, 64 * s, y, ahead.head, w, full + at);
        if (Sh::PAIRED) tma_load_4d(dst + SIDE + s * 2048, &vmap, 64 * s, y, ahead.head, w, full + at);
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
          const int i = 16 * k + 8 * j + c0;
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
#pragma unroll
        for (int k = 0; k < KST; ++k) {
          uint32_t a[4];
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
        const int key = ks + (lane >> 2);
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
              if (key + 8 > to || key + 8 < from) s[n][2 + j] = -CUDART_INF_F;
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
              if (l[n][j] == l[n][j] && 8 * n + c0 + j < n_rows) {  // (a row that is NaN already stays that)
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
        if (masked) {
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
#pragma unroll
          for (int k = 0; k < AHEAD; ++k) {
            ldsm4_t(a[k], vb + ((k0 + k) >> 2) * 2048 + ((i4 >> 1) * 8 + r8) * 128 + (((2 * ((k0 + k) & 3) + (i4 & 1)) ^ r8) << 4));
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

#pragma unroll
    for (int k = 0; k < KST; ++k)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) odd |= !(fabsf(o[k][n][i]) < CUDART_INF_F);

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

template <int HD, int NT>
cudaError_t run_rows(infr_cuda_ctx* ctx, const CUtensorMap& km, const CUtensorMap& vm, const AttnParams& p) {
  using Sh = RowsShape<HD, NT>;
  const cudaError_t e = ensure_smem(reinterpret_cast<const void*>(&k_attn_rows<HD, NT>), Sh::SMEM);
  if (e != cudaSuccess) return e;
  return launch_ex(k_attn_rows<HD, NT>, dim3(ctx->sm_count < ATTN_MAX_CTAS ? ctx->sm_count : ATTN_MAX_CTAS), dim3(Sh::THREADS), Sh::SMEM, ctx->stream, true, km, vm, p);
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
  if (p.kq != nullptr) return launch_attn_rows_q8(ctx, p, max_rows);
  p.k = k;
  CUtensorMap km, vm;
  if (!attn_cache_map(&km, k, p, 16) || !attn_cache_map(&vm, p.v, p, 16)) return fail(ctx, INFR_CUDA_ERR_CUDA, "attention: cuTensorMapEncodeTiled failed");
  const int nt = p.g <= 8 && max_rows <= 8 ? 1 : 2;
  p.tb = 8 * nt / p.g;
  cudaError_t e;
  if (p.hd <= 64) e = nt == 1 ? run_rows<64, 1>(ctx, km, vm, p) : run_rows<64, 2>(ctx, km, vm, p);
  else if (p.hd <= 128) e = nt == 1 ? run_rows<128, 1>(ctx, km, vm, p) : run_rows<128, 2>(ctx, km, vm, p);
  else if (p.hd <= 192) e = nt == 1 ? run_rows<192, 1>(ctx, km, vm, p) : run_rows<192, 2>(ctx, km, vm, p);
  else e = nt == 1 ? run_rows<256, 1>(ctx, km, vm, p) : run_rows<256, 2>(ctx, km, vm, p);
  if (e != cudaSuccess) return check_cuda(ctx, e, "k_attn_rows launch");
  ctx->launches += 1;
  return check_cuda(ctx, cudaGetLastError(), "k_attn_rows launch");
}

}  // namespace infr
