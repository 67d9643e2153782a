// Attention of many rows per (sequence, kv head): prompts, and chunks of new tokens over a cache.  An item is 128 rows (whole tokens x the
// query heads of a kv head, so that these share the keys' tiles); its key tiles go through the tensor cores with accumulators in tensor
// memory, one pass with a running maximum.  What bounds it is the tensor cores: q and the weights are two f16 pieces each (f32 results), so
// a pair (row, key) costs 8 hd operations at the f16 rate.
//
// One CTA per SM, roles by warpgroup:
//   weights   a thread per row: scores S from tensor memory -> running maximum -> weights P, back over S as f16 pieces
//   sums      a thread per row: the f32 sums in registers.  Each tile's P V starts from zero in tensor memory and is added here, times
//             the maximum's correction: an accumulation over thousands of steps in the tensor cores, which truncate, would lose
//             an f32 result's last bits (measured: 1.3e-8 of the result per step), and the correction is part of the same FMA
//   control   a warp for the copies, a warp for the MMAs, two that turn q into f16 pieces and look after tiles with hidden keys
// S and P of two tiles, and the sums of two (one for heads wider than 192), fill tensor memory: while a tile's weights are made the
// tensor cores work on the next tile's scores and the last one's sums.
#include "attn.cuh"
#include "umma.cuh"

namespace infr {
namespace {

constexpr float TILE_BIAS = 15.f;  // weights are 2^(x - maximum + 15): below f16's limit, 2^-40 of the largest still has a bit
constexpr int ALPHA_RING = 4, ITEM_RING = 16;

template <int HD>
struct TilesShape {
  static constexpr int LOG2_TILE = HD <= 128 ? 7 : 6, BK = 1 << LOG2_TILE;
  static constexpr int SUM_GROUPS = HD <= 128 ? 1 : 2, COLS = HD / SUM_GROUPS;  // columns of a sums thread
  static constexpr int THREADS = 128 * (2 + SUM_GROUPS);
  static constexpr int SLABS = HD / 64, TILE = BK * HD * 2, QPIECE = 128 * HD * 2;
  static constexpr int STAGES = HD == 64 ? 8 : HD == 128 ? 4 : HD == 192 ? 4 : 2;
  static constexpr int OBUFS = HD <= 192 ? 2 : 1;
  static constexpr uint32_t O_COL = 2 * BK;
  static constexpr int SMALL = ALPHA_RING * 128 * 4 + ITEM_RING * 128 * 8 + 4 * 128 * 4;  // corrections, (maximum, weight), score factors
  static constexpr int SMEM = 1024 + 2 * QPIECE + STAGES * TILE + SMALL;
  static_assert(SMEM + 1024 <= 232448, "more shared memory than a CTA has");
  // registers by role; together no more than the launch has
  static constexpr int REG_W = HD <= 128 ? 160 : 136, REG_S = HD <= 128 ? 208 : 152, REG_C = HD <= 128 ? 136 : 72;
};

template <int N>
__device__ __forceinline__ void regs_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

struct TileBars {
  uint64_t full[8], empty[8];   // tiles of K and V, in the order K0 K1 V0 K2 V1 ...
  uint64_t s_full[2], p_full[2];
  uint64_t o_full[2], o_empty[2];
  uint64_t a_full[ALPHA_RING];  // a tile's corrections (and, at an item's last, maximum and weight)
  uint64_t f_full[4];           // an item's score factors
  uint64_t q_full, q_empty;
  uint64_t v_ask, v_ok;         // a V tile with hidden keys: there, and looked after
};

// Whether some row of the item does not see some key of [ks, ks + n).
__device__ __forceinline__ bool tile_masked(const AttnParams& p, const AttnSeq& seq, const AttnBlock& blk, int ks, int n) {
  return ks + n > attn_full_hi(seq, blk) || ks < attn_full_lo(p, seq, blk);
}

template <int HD>
__global__ void __launch_bounds__(TilesShape<HD>::THREADS, 1)
    k_attn_tiles(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ AttnParams p, const int granule) {
  using Sh = TilesShape<HD>;
  constexpr int BK = Sh::BK, SLABS = Sh::SLABS, STAGES = Sh::STAGES, OBUFS = Sh::OBUFS, TILE = Sh::TILE;
  extern __shared__ unsigned char smem_raw[];
  __shared__ TileBars bars;
  __shared__ long long s_scan[Sh::THREADS / 32];
  __shared__ AttnStart s_start;
  __shared__ uint32_t s_tmem;
  __shared__ int s_last, s_odd[ITEM_RING];
  unsigned char* s_q = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* s_kv = s_q + 2 * Sh::QPIECE;
  float* s_alpha = reinterpret_cast<float*>(s_kv + STAGES * TILE);           // [ALPHA_RING][128]
  float2* s_ml = reinterpret_cast<float2*>(s_alpha + ALPHA_RING * 128);      // [ITEM_RING][128]
  float* s_fac = reinterpret_cast<float*>(s_ml + ITEM_RING * 128);           // [4][128]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wg = warp >> 2, control = 1 + Sh::SUM_GROUPS, role = wg == control ? 4 + (warp & 3) : wg;  // 4: copies, 5: MMAs

  if (tid == 0) {
    for (int i = 0; i < 8; ++i) mbar_init(bars.full + i, 1), mbar_init(bars.empty + i, 1);
    for (int i = 0; i < 2; ++i) mbar_init(bars.s_full + i, 1), mbar_init(bars.p_full + i, 4), mbar_init(bars.o_full + i, 1), mbar_init(bars.o_empty + i, 4 * Sh::SUM_GROUPS);
    for (int i = 0; i < ALPHA_RING; ++i) mbar_init(bars.a_full + i, 4);
    for (int i = 0; i < 4; ++i) mbar_init(bars.f_full + i, 2);
    mbar_init(&bars.q_full, 2), mbar_init(&bars.q_empty, 1), mbar_init(&bars.v_ask, 1), mbar_init(&bars.v_ok, 2);
    mbar_fence_init();
  }
  if (tid < ITEM_RING) s_odd[tid] = 0;
  if (warp == 0) umma::tmem_alloc(&s_tmem);
  pdl_wait();
  attn_plan<Sh::THREADS, Sh::LOG2_TILE>(p, reinterpret_cast<int*>(s_q), s_scan, &s_start);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the plan's words lay where tiles go
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const AttnStart st = s_start;
  const uint32_t tmem = s_tmem;
  const int N = (int)(st.u1 - st.u0);  // tiles of this CTA
  bool ok = true;

  if (N > 0 && wg == control) regs_less<Sh::REG_C>();
  if (N == 0) {
    // nothing to do
  } else if (role == 4) {
    // ---- copies
    AttnCursor<Sh::LOG2_TILE> kc, vc;
    kc.start(p, st);
    vc = kc;
    const int pieces = BK / granule;
    const bool packed = p.page_table == nullptr;
    int asked = 0;
    auto load = [&](AttnCursor<Sh::LOG2_TILE>& c, int n, const CUtensorMap* map) {
      const long long u = st.u0 + n;
      while (u >= c.ub + c.blk.ntile) c.next(p);
      const int ks = (c.blk.tile0 + (int)(u - c.ub)) << Sh::LOG2_TILE, key = ks + lane * granule;
      const bool has = lane < pieces && key < c.blk.hi && key + granule > c.blk.lo;
      int y = c.seq.q0 + key, w = 0;
      if (has && !packed) {
        w = attn_page(p, c.s, key / p.page_size);
        y = key % p.page_size;
      }
      const int stage = asked % STAGES;
      if (asked >= STAGES) ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(bars.empty + stage, (asked / STAGES - 1) & 1));
      if (!ok) return;
      const int count = __popc(__ballot_sync(0xFFFFFFFFu, has));
      if (lane == 0) mbar_arrive_expect_tx(bars.full + stage, (uint32_t)(count * granule * 128 * SLABS));
      __syncwarp();
      if (has) {
        unsigned char* dst = s_kv + stage * TILE + lane * granule * 128;
#pragma unroll
        for (int s = 0; s < SLABS; ++s) tma_load_4d(dst + s * (BK * 128), map, 64 * s, y, c.head, w, bars.full + stage);
      }
      __syncwarp();
      ++asked;
    };
    load(kc, 0, &kmap);
    for (int n = 0; n < N && ok; ++n) {
      if (n + 1 < N) load(kc, n + 1, &kmap);
      if (ok) load(vc, n, &vmap);
    }
    if (!ok) {
      if (lane == 0) atomicExch(&p.status->timeout, 11);
      // copies in flight land before the shared memory is somebody else's
      for (int i = max(0, asked - STAGES); i < asked; ++i) mbar_wait_bounded(bars.full + i % STAGES, (i / STAGES) & 1);
    }
  } else if (role == 5) {
    // ---- MMAs
    AttnCursor<Sh::LOG2_TILE> ic, cc;  // of the tile whose scores come next, and of the one whose sums do
    ic.start(p, st);
    cc = ic;
    const uint32_t idesc_s = umma::idesc_f16_f32(128, BK), idesc_o = umma::idesc_f16_f32(128, HD) | umma::IDESC_B_MN_MAJOR;
    const uint32_t kva = smem_u32(s_kv);
    int issued = 0, items = 0, asks = 0;
    bool starts = true;  // the next tile of scores is its item's first here
    for (int n = 0; n < N && ok; ++n) {
      // scores: one tile ahead, but not into the next item, whose q may still be on its way while this one's sums are due
      while (issued < N && issued <= n + 1 && (issued == n || !starts)) {
        if (starts) {
          ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&bars.q_full, items & 1));
          ++items;
        }
        const int i = issued == 0 ? 0 : 2 * issued - 1, stage = i % STAGES;
        ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait_bounded(bars.full + stage, (i / STAGES) & 1));
        if (!ok) break;
        umma::fence_after_sync();
        const long long u = st.u0 + issued;
        const bool last = u + 1 >= ic.ub + ic.blk.ntile || issued + 1 == N;
        if (umma::elect_one()) {
          const uint32_t d = tmem + (issued & 1) * BK;
#pragma unroll
          for (int piece = 0; piece < 2; ++piece)
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
              const uint64_t a = umma::smem_desc_k_major_swz128(s_q + piece * Sh::QPIECE + (k >> 2) * 16384, k & 3);
              const uint64_t b = umma::smem_desc_k_major_swz128(s_kv + stage * TILE + (k >> 2) * (BK * 128), k & 3);
              umma::mma1_f16_ss(d, a, b, idesc_s, piece + k > 0 ? 1u : 0u);
            }
          umma::commit1(bars.empty + stage);
          umma::commit1(bars.s_full + (issued & 1));
          if (last) umma::commit1(&bars.q_empty);
        }
        __syncwarp();
        ++issued;
        starts = last;
        if (u + 1 >= ic.ub + ic.blk.ntile && issued < N) ic.next(p);
      }
      if (!ok) break;
      const long long u = st.u0 + n;
      while (u >= cc.ub + cc.blk.ntile) cc.next(p);
      const int i = n + 1 < N ? 2 * n + 2 : 2 * N - 1, stage = i % STAGES;
      const bool masked = tile_masked(p, cc.seq, cc.blk, (cc.blk.tile0 + (int)(u - cc.ub)) << Sh::LOG2_TILE, BK);
      ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(bars.full + stage, (i / STAGES) & 1));
      if (ok && masked && lane == 0) mbar_arrive(&bars.v_ask);
      ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait_bounded(bars.p_full + (n & 1), (n >> 1) & 1));
      if (n >= OBUFS) ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait_bounded(bars.o_empty + n % OBUFS, (n / OBUFS - 1) & 1));
      if (masked) {
        ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&bars.v_ok, asks & 1));
        ++asks;
      }
      if (!ok) break;
      umma::fence_after_sync();
      if (umma::elect_one()) {
        const uint32_t d = tmem + Sh::O_COL + (n % OBUFS) * HD, a = tmem + (n & 1) * BK;
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) {
          const uint64_t b = umma::smem_desc_mn_major_swz128(kva + stage * TILE, k, BK * 128);
          const uint32_t ak = a + (k >> 1) * 32 + (k & 1) * 8;  // 32 keys: 16 columns of their weights, 16 of the rest
          umma::mma1_f16_ts(d, ak, b, idesc_o, k > 0 ? 1u : 0u);
          umma::mma1_f16_ts(d, ak + 16, b, idesc_o, 1u);
        }
        umma::commit1(bars.empty + stage);
        umma::commit1(bars.o_full + n % OBUFS);
      }
      __syncwarp();
    }
    if (!ok && lane == 0) atomicExch(&p.status->timeout, 11);
  } else if (role > 5) {
    // ---- q into two f16 pieces, and V tiles with hidden keys
    const int at = (warp & 1) * 32 + lane, l8 = lane & 7;
    AttnCursor<Sh::LOG2_TILE> c;
    c.start(p, st);
    int asks = 0, item = 0;
    for (int n = 0; n < N && ok; ++item) {
      const long long u = st.u0 + n;
      while (u >= c.ub + c.blk.ntile) c.next(p);
      const int end = (int)((c.ub + c.blk.ntile < st.u1 ? c.ub + c.blk.ntile : st.u1) - st.u0), n_rows = c.blk.nt * p.g;
      if (at == 0) s_odd[(item + 8) % ITEM_RING] = 0;
      if (item > 0) ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&bars.q_empty, (item - 1) & 1));
      if (!ok) break;
      // eight lanes a row, four rows a warp at once; rows past the item's are zeros
#pragma unroll(HD <= 128 ? 2 : 1)
      for (int r0 = 0; r0 < 128; r0 += 8) {
        const int r = r0 + (at >> 3);
        const bool has = r < n_rows;
        const float* src = p.q + (size_t)(c.seq.q0 + c.blk.t0 + (has ? r / p.g : 0)) * p.q_stride + (size_t)(c.head * p.g + (has ? r % p.g : 0)) * p.hd;
        float4 v[HD / 32];
        float big = 0.f;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
          const int i = 4 * (l8 + 8 * j);
          v[j] = has && i < p.hd ? __ldcg(reinterpret_cast<const float4*>(src + i)) : make_float4(0.f, 0.f, 0.f, 0.f);
          big = fmaxf(big, fmaxf(fmaxf(fabsf(v[j].x), fabsf(v[j].y)), fmaxf(fabsf(v[j].z), fabsf(v[j].w))));
        }
#pragma unroll
        for (int x = 1; x < 8; x <<= 1) big = fmaxf(big, __shfl_xor_sync(0xFFFFFFFFu, big, x));
        float down, up;
        attn_row_scale(big, down, up);
        if (p.scale_log2 < 0.f) down = -down;
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) {
          const int i = 4 * (l8 + 8 * j);
          uint2 hi, lo;
          split2(v[j].x * down, v[j].y * down, hi.x, lo.x);
          split2(v[j].z * down, v[j].w * down, hi.y, lo.y);
          unsigned char* dst = s_q + (i >> 6) * 16384 + r * 128 + ((((i >> 3) & 7) ^ (r & 7)) << 4) + ((i & 4) << 1);
          *reinterpret_cast<uint2*>(dst) = hi;
          *reinterpret_cast<uint2*>(dst + Sh::QPIECE) = lo;
        }
        // (not 0: hidden keys' -inf times it stays -inf)
        if (l8 == 0) s_fac[(item & 3) * 128 + r] = fmaxf(up * fabsf(p.scale_log2), 1.2e-38f);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.q_full), mbar_arrive(bars.f_full + (item & 3));
      for (; n < end && ok; ++n) {
        const int ks = (c.blk.tile0 + (int)(st.u0 + n - c.ub)) << Sh::LOG2_TILE;
        if (!tile_masked(p, c.seq, c.blk, ks, BK)) continue;
        // 0 x value has to be 0 where a row does not see the key: keys that no row sees become zeros, and so do values that are not
        // finite; the item's end adds these to the rows that see them
        ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&bars.v_ask, asks & 1));
        ++asks;
        if (!ok) break;
        const int i = n + 1 < N ? 2 * n + 2 : 2 * N - 1;
        bool odd = false;
        for (int row = at; row < BK; row += 64) {
          const bool seen = ks + row >= c.blk.lo && ks + row < c.blk.hi;
#pragma unroll
          for (int s = 0; s < SLABS; ++s) {
            unsigned char* base = s_kv + (i % STAGES) * TILE + s * (BK * 128) + row * 128;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              uint4* w = reinterpret_cast<uint4*>(base + (((j + row) & 7) << 4));
              if (!seen) {
                *w = make_uint4(0, 0, 0, 0);
                continue;
              }
              const uint4 x = *w;
              if (any_odd(x.x) || any_odd(x.y) || any_odd(x.z) || any_odd(x.w)) {
                *w = make_uint4(only_finite(x.x), only_finite(x.y), only_finite(x.z), only_finite(x.w));
                odd = true;
              }
            }
          }
        }
        if (odd) s_odd[item % ITEM_RING] = 1;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.v_ok);
      }
    }
    if (!ok && lane == 0) atomicExch(&p.status->timeout, 11);
  } else if (wg == 0) {
    // ---- weights: thread = row
    if (Sh::REG_W < 160) regs_more<Sh::REG_W>();
    else regs_less<Sh::REG_W>();
    AttnCursor<Sh::LOG2_TILE> c;
    c.start(p, st);
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    int item = -1;
    float m = -CUDART_INF_F, l = 0.f, f = 0.f;
    int to = 0, from = 0, n_rows = 0;  // the row sees the keys (from, to]
    for (int n = 0; n < N && ok; ++n) {
      const long long u = st.u0 + n;
      if (n == 0 || u >= c.ub + c.blk.ntile) {
        while (u >= c.ub + c.blk.ntile) c.next(p);
        ++item;
        n_rows = c.blk.nt * p.g;
        to = c.seq.past + c.blk.t0 + (tid < n_rows ? tid / p.g : c.blk.nt - 1);
        from = p.window > 0 ? to - p.window : -1;
        m = -CUDART_INF_F, l = 0.f;
        ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(bars.f_full + (item & 3), (item >> 2) & 1));
        f = s_fac[(item & 3) * 128 + tid];
      }
      const int ks = (c.blk.tile0 + (int)(u - c.ub)) << Sh::LOG2_TILE;
      const bool masked = tile_masked(p, c.seq, c.blk, ks, BK);
      ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait_bounded(bars.s_full + (n & 1), (n >> 1) & 1));
      if (!ok) break;
      umma::fence_after_sync();
      float alpha = 1.f;
      if (warp * 32 < n_rows) {  // (other rows' weights are whatever is there: they reach those rows' sums only)
        const uint32_t sa = lanes + (n & 1) * BK;
        float top = -CUDART_INF_F;
#pragma unroll
        for (int j = 0; j < BK / 32; ++j) {
          float s[32];
          umma::tmem_ld_32x32(sa + 32 * j, s);
          umma::tmem_ld_wait(s);
          if (masked) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (ks + 32 * j + i <= to && ks + 32 * j + i > from) top = fmaxf(top, s[i]);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) top = fmaxf(top, s[i]);
          }
        }
        const float now = fmaxf(m, top * f);
        alpha = exp2_rel(m, now);
        m = now;
        const float off = TILE_BIAS - (now == -CUDART_INF_F ? 0.f : now);
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (int j = 0; j < BK / 32; ++j) {
          float s[32];
          umma::tmem_ld_32x32(sa + 32 * j, s);
          umma::tmem_ld_wait(s);
          if (masked) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(ks + 32 * j + i <= to && ks + 32 * j + i > from)) s[i] = -CUDART_INF_F;
          }
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float a = exp2_approx(fmaf(s[2 * i], f, off)), b = exp2_approx(fmaf(s[2 * i + 1], f, off));
            sum0 += a, sum1 += b;
            split2(a, b, w[i], w[16 + i]);
          }
          umma::tmem_st_32x32_async(sa + 32 * j, w);
        }
        l = l * alpha + (sum0 + sum1);
        umma::tmem_st_wait();
      }
      umma::fence_before_sync();
      s_alpha[(n & (ALPHA_RING - 1)) * 128 + tid] = alpha;
      if (u + 1 >= c.ub + c.blk.ntile || n + 1 == N) {
        if (m == -CUDART_INF_F && l != 0.f) m = 0.f;  // nothing but NaN: a part that counts
        s_ml[(item % ITEM_RING) * 128 + tid] = make_float2(m, l);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bars.p_full + (n & 1)), mbar_arrive(bars.a_full + (n & (ALPHA_RING - 1)));
    }
    if (!ok && lane == 0) atomicExch(&p.status->timeout, 11);
  } else {
    // ---- sums: thread = row, COLS of its columns
    regs_more<Sh::REG_S>();
    AttnCursor<Sh::LOG2_TILE> c;
    c.start(p, st);
    const int row = tid & 127, col0 = (wg - 1) * Sh::COLS;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + Sh::O_COL + col0;
    float o[Sh::COLS];
    int item = 0, first = 0;
    for (int n = 0; n < N && ok; ++n) {
      const long long u = st.u0 + n;
      while (u >= c.ub + c.blk.ntile) c.next(p);
      if (n == first) {
#pragma unroll
        for (int i = 0; i < Sh::COLS; ++i) o[i] = 0.f;
      }
      const int n_rows = c.blk.nt * p.g;
      const bool mine = (warp & 3) * 32 < n_rows;
      ok = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(bars.a_full + (n & (ALPHA_RING - 1)), (n / ALPHA_RING) & 1));
      const float alpha = s_alpha[(n & (ALPHA_RING - 1)) * 128 + row];
      ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait_bounded(bars.o_full + n % OBUFS, (n / OBUFS) & 1));
      if (!ok) break;
      umma::fence_after_sync();
      if (mine) {
#pragma unroll
        for (int j = 0; j < Sh::COLS / 32; ++j) {
          float t[32];
          umma::tmem_ld_32x32(lanes + (n % OBUFS) * HD + 32 * j, t);
          umma::tmem_ld_wait(t);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[32 * j + i] = fmaf(o[32 * j + i], alpha, t[i]);
        }
      }
      umma::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bars.o_empty + n % OBUFS);
      if (!(u + 1 >= c.ub + c.blk.ntile || n + 1 == N)) continue;

      // ---- the item's end
      const bool whole = u + 1 >= c.ub + c.blk.ntile && st.u0 + first <= c.ub;
      const AttnShare share = attn_share(c.ub, c.blk.ntile, st);
      const bool odd_tiles = *reinterpret_cast<volatile int*>(s_odd + item % ITEM_RING) != 0;
      const float2 ml = s_ml[(item % ITEM_RING) * 128 + row];
      const size_t slot = (size_t)attn_slot(blockIdx.x, share) * 128 + row;
      const bool mine_row = row < n_rows;
      float* dst = whole ? p.out + (size_t)(c.seq.q0 + c.blk.t0 + (mine_row ? row / p.g : 0)) * p.out_stride + (size_t)(c.head * p.g + (mine_row ? row % p.g : 0)) * p.hd + col0
                         : p.part + slot * HD + col0;
      if (mine_row) {
        const float inv = !whole ? 1.f : ml.y > 0.f ? 1.f / ml.y : (ml.y == 0.f ? 0.f : ml.y);
        bool odd = odd_tiles;
#pragma unroll
        for (int i = 0; i < Sh::COLS; i += 4) {
          const float4 v = make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv);
          odd |= !(fabsf(o[i]) < CUDART_INF_F && fabsf(o[i + 1]) < CUDART_INF_F && fabsf(o[i + 2]) < CUDART_INF_F && fabsf(o[i + 3]) < CUDART_INF_F);
          if (col0 + i < p.hd) __stcg(reinterpret_cast<float4*>(dst + i), v);
        }
        if (!whole && wg == 1) __stcg(p.part_ml + slot, ml);
        if (odd && ml.y == ml.y) attn_odd_values(p, c.s, c.seq.q0, c.head, (c.blk.tile0 + (int)(max(st.u0 + first, c.ub) - c.ub)) << Sh::LOG2_TILE,
                                                      (c.blk.tile0 + (int)(u + 1 - c.ub)) << Sh::LOG2_TILE, BK, attn_full_lo(p, c.seq, c.blk), attn_full_hi(c.seq, c.blk),
                                                      c.seq.past + c.blk.t0 + row / p.g, col0, Sh::COLS, dst);
      }
      if (!whole && attn_arrive(p, share, &s_last, tid == 128, 1, 128 * Sh::SUM_GROUPS)) {
        for (int e = tid - 128; e < n_rows * (HD / 4); e += 128 * Sh::SUM_GROUPS) {
          const int r = e / (HD / 4), i = 4 * (e % (HD / 4));
          if (i < p.hd)
            *reinterpret_cast<float4*>(p.out + (size_t)(c.seq.q0 + c.blk.t0 + r / p.g) * p.out_stride + (size_t)(c.head * p.g + r % p.g) * p.hd + i) =
                attn_join4<HD>(p, share, 128, r, i);
        }
      }
      first = n + 1;
      ++item;
    }
    if (!ok && lane == 0) atomicExch(&p.status->timeout, 11);
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  if (warp == 0) umma::tmem_dealloc(tmem);
}

template <int HD>
cudaError_t run_tiles(infr_cuda_ctx* ctx, const CUtensorMap& km, const CUtensorMap& vm, const AttnParams& p, int granule) {
  using Sh = TilesShape<HD>;
  const cudaError_t e = ensure_smem(reinterpret_cast<const void*>(&k_attn_tiles<HD>), Sh::SMEM);
  if (e != cudaSuccess) return e;
  return launch_ex(k_attn_tiles<HD>, dim3(ctx->sm_count), dim3(Sh::THREADS), Sh::SMEM, ctx->stream, true, km, vm, p, granule);
}

}  // namespace

int32_t launch_attn_tiles(infr_cuda_ctx* ctx, AttnParams p, const __half* k) {
  // a copy takes as many keys as lie side by side in every page
  int granule = p.hd <= 128 ? 128 : 64;
  while (p.page_table != nullptr && p.page_size % granule) granule >>= 1;
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
