// A token of each row of logits:
//
//   w_i = exp((x_i - max x) / T)                                                 of the tokens above -inf
//   kept: the top_k largest (of equal ones the lowest), of these the shortest run from the largest that has top_p of their weight, of these
//         those with w_i >= min_p
//   token: the first in order whose weight and the kept ones' ahead of it are more than u times the kept ones' together
//
// What is kept is always a run from the largest, so it is one border: a value and an index.  Finding it needs no sort of the row: a histogram of the values says
// between which of them it lies, and the few that lie there are sorted.  Weights and their sums are f64: with f32 sums the token next to a border would
// go by the order of the additions, and there are 10^5 borders to a row.  Weights below 2^-64 of the largest count as none: all of them together are 2^-46,
// which an f32 u cannot tell from nothing.
//
// A cluster of eight CTAs has a row in its shared memory: the logits are read once.  Every decision is made from numbers that all eight have, in the same order,
// so that they take the same steps; what is shared goes through distributed shared memory, a cluster barrier behind it.
#include <cooperative_groups.h>
#include <math_constants.h>

#include "kernels.cuh"

namespace infr {
namespace {

namespace cg = cooperative_groups;

constexpr int SAMPLE_CTAS = 8, SAMPLE_THREADS = 512, SAMPLE_WARPS = SAMPLE_THREADS / 32;
constexpr int SAMPLE_BINS = 4 * SAMPLE_THREADS;  // a thread has four
constexpr int SAMPLE_LIST = 2048;                // candidates that are sorted
constexpr int SAMPLE_CAP = 40960;                // values of a row in a CTA's shared memory; what is behind them is read again from global memory
constexpr double SAMPLE_REACH = 45.0;            // weights down to e^-45 < 2^-64
typedef unsigned long long u64;

// Values in order: larger ones have smaller numbers; with the index behind them, the order in which tokens are taken.
__device__ __forceinline__ uint32_t rank_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? b : 0x7FFFFFFFu - b;
}
__device__ __forceinline__ float value_of(uint32_t r) { return __uint_as_float(r & 0x80000000u ? r : 0x7FFFFFFFu - r); }
__device__ __forceinline__ u64 place_of(float x, int i) { return (u64)rank_of(x) << 32 | (uint32_t)i; }

struct SampleShared {
  uint32_t hist[SAMPLE_BINS];
  u64 list[SAMPLE_LIST];
  double scan[2][SAMPLE_WARPS];
  int scan_n[SAMPLE_WARPS];
  // from every CTA, by rank
  u64 best[SAMPLE_CTAS];
  float low[SAMPLE_CTAS];
  int odd[SAMPLE_CTAS];
  double sum[SAMPLE_CTAS], above[SAMPLE_CTAS], kept[SAMPLE_CTAS];
  uint32_t first[SAMPLE_CTAS], last[SAMPLE_CTAS];
  int equal[SAMPLE_CTAS];
  // the first CTA's
  int n_list;
  u64 border;
  // of the bins
  int b1, b2, ahead, upto;
  int pick;
};

struct Sampler {
  SampleShared& sh;
  cg::cluster_group cluster;
  const float *xs, *gx;  // this CTA's values: in shared memory, and where they came from
  int n, base, me, tid;  // how many, index of the first
  float top;             // the row's largest value
  double inv_t;
  float floor_x;         // values from here on have a weight

  __device__ float x_at(int i) const { return i < SAMPLE_CAP ? xs[i] : __ldcg(gx + i) + 0.f; }
  __device__ double weight(float x) const { return x < floor_x ? 0.0 : x == top ? 1.0 : exp(((double)x - (double)top) * inv_t); }

  template <typename T>
  __device__ T warp_total(T v) const {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
  }
  // Sum over the block's threads before this one, and over all; `s`: a word per warp.
  template <typename T>
  __device__ T before(T v, T* s, T& all) const {
    const int lane = tid & 31, warp = tid >> 5;
    T x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T y = __shfl_up_sync(0xFFFFFFFFu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) s[warp] = x;
    __syncthreads();
    T ahead = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < SAMPLE_WARPS; ++w) {
      if (w == warp) ahead = all;
      all += s[w];
    }
    const T up = __shfl_up_sync(0xFFFFFFFFu, x, 1);
    return ahead + (lane ? up : T(0));
  }
  // This CTA's word into every CTA's array; read behind the next cluster barrier.
  template <typename T>
  __device__ void tell(T* array, T v) {
    if (tid < SAMPLE_CTAS) *cluster.map_shared_rank(array + me, tid) = v;
  }
  __device__ void clear_hist() {
    for (int b = tid; b < SAMPLE_BINS; b += SAMPLE_THREADS) sh.hist[b] = 0;
    if (tid == 0) sh.n_list = 0, sh.b1 = sh.b2 = SAMPLE_BINS;
    __syncthreads();
  }
  __device__ double total(const double* of_ctas) const {
    double t = 0;
    for (int r = 0; r < SAMPLE_CTAS; ++r) t += of_ctas[r];
    return t;
  }

  // The bins b1 .. b2 that the border lies in, how many values lie ahead of them and up to their end.  By count: the bin of the k-th value; by weight: those
  // that may have the value with which the sum passes `target`, by the weights `hi` and `lo` that a bin's values have at most and at least.
  // (`slack`: by how much of a weight a bin's edges are off)
  template <class Edge>
  __device__ void bracket(bool by_weight, int k, double target, double slack, Edge edge) {
    uint32_t c[4] = {0, 0, 0, 0};
#pragma unroll
    for (int r = 0; r < SAMPLE_CTAS; ++r) {
      const uint4 h = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh.hist, r) + 4 * tid);
      c[0] += h.x, c[1] += h.y, c[2] += h.z, c[3] += h.w;
    }
    int all = 0;
    int ahead = before<int>((int)(c[0] + c[1] + c[2] + c[3]), sh.scan_n, all);
    if (by_weight) {
      double hi[4], lo[4], w = edge(4 * tid);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double next = edge(4 * tid + j + 1);
        hi[j] = c[j] * w * (1.0 + slack), lo[j] = c[j] * next * (1.0 - slack);
        w = next;
      }
      double sum;
      double h = before<double>((hi[0] + hi[1]) + (hi[2] + hi[3]), sh.scan[0], sum), l = before<double>((lo[0] + lo[1]) + (lo[2] + lo[3]), sh.scan[1], sum);
      int b1 = SAMPLE_BINS, b2 = SAMPLE_BINS, end = -1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        h += hi[j], l += lo[j];
        if (!c[j]) continue;
        end = 4 * tid + j;
        // (what sums in another order may differ by)
        if (b1 == SAMPLE_BINS && h * (1.0 + 1e-12) >= target) b1 = end;
        if (b2 == SAMPLE_BINS && l * (1.0 - 1e-12) >= target) b2 = end;
      }
      if (b1 < SAMPLE_BINS) atomicMin(&sh.b1, b1);
      if (b2 < SAMPLE_BINS) atomicMin(&sh.b2, b2);
      if (tid == 0) sh.pick = -1;
      __syncthreads();
      if (end >= 0) atomicMax(&sh.pick, end);
      __syncthreads();
      if (tid == 0) {  // (no bin passes the target for certain, or at all: the last one with values)
        if (sh.b2 == SAMPLE_BINS) sh.b2 = sh.pick;
        if (sh.b1 == SAMPLE_BINS) sh.b1 = sh.pick;
      }
    } else {
      int at = ahead;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (at < k && k <= at + (int)c[j]) sh.b1 = sh.b2 = 4 * tid + j;
        at += (int)c[j];
      }
      if (tid == SAMPLE_THREADS - 1 && all < k) sh.b1 = sh.b2 = -1;  // all are kept
    }
    __syncthreads();
    const int b1 = sh.b1, b2 = sh.b2;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (4 * tid + j == b1) sh.ahead = ahead;
      ahead += (int)c[j];
      if (4 * tid + j == b2) sh.upto = ahead;
    }
    __syncthreads();
  }

  // The first CTA sorts the candidates: list[0 .. n - 1], padded to a power of two.
  __device__ void sort_list(int n) {
    int size = 32;
    while (size < n) size <<= 1;
    for (int i = n + tid; i < size; i += SAMPLE_THREADS) sh.list[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        for (int t = tid; t < size / 2; t += SAMPLE_THREADS) {
          const int a = 2 * t - (t & (j - 1)), b = a + j;
          const u64 x = sh.list[a], y = sh.list[b];
          if ((x > y) == ((a & k) == 0)) sh.list[a] = y, sh.list[b] = x;
        }
        __syncthreads();
      }
  }

  // The border among the values up to `within`: that of the k largest, or with p < 1 that of the run with p of the weight, or (k, then p) both where the
  // candidates hold all of the k; *both: whether they did.
  __device__ u64 find(u64 within, int k, double p, bool* both) {
    const bool by_weight = k <= 0;
    *both = false;
    // ---- bins of one width from the largest value down to the least that has a weight (a border of the k largest may lie behind: then nothing is left out)
    float low = CUDART_INF_F;
    for (int r = 0; r < SAMPLE_CTAS; ++r) low = fminf(low, sh.low[r]);
    low = fmaxf(low, floor_x);
    const float s = top > low ? (float)((double)(SAMPLE_BINS - 1) / (0.5 * ((double)top - (double)low))) : 0.f;
    const float half = 0.5f * top;  // (a difference of halves does not overflow)
    auto bin = [&](float x) { return min((int)((half - 0.5f * x) * s), SAMPLE_BINS - 1); };
    clear_hist();
    double mine = 0;
#pragma unroll 4
    for (int i = tid; i < n; i += SAMPLE_THREADS) {
      const float x = x_at(i);
      if (x < low || place_of(x, base + i) > within) continue;
      atomicAdd(&sh.hist[bin(x)], 1u);
      if (by_weight) mine += weight(x);
    }
    if (by_weight) {
      double all;
      before<double>(mine, sh.scan[0], all);
      tell(sh.sum, all);
    }
    cluster.sync();
    double target = by_weight ? p * total(sh.sum) : 0;
    const double width = s > 0.f ? 2.0 * inv_t / s : 0.0;
    // f32 moves a bin's edges by 2^-22 of their distance from the largest, which is 45 in the exponent at most
    bracket(by_weight, k, target, 2e-5, [&](int b) { return exp(-b * width); });
    int b1 = sh.b1, b2 = sh.b2, ahead = sh.ahead, upto = sh.upto;
    if (b1 < 0) return within;
    bool whole = !by_weight && upto <= SAMPLE_LIST;  // the list takes what lies ahead too
    uint32_t r1 = 0, r2 = 0;                          // the candidates as a range of ranks, once the bins are not enough
    bool by_rank = false;
    for (int level = 0;; ++level) {
      const int n_list = whole ? upto : upto - ahead;
      if (n_list <= SAMPLE_LIST) break;
      // ---- too many: bins of ranks, 2^11 to the candidates' range; after three of these a bin is one value
      uint32_t lo = 0xFFFFFFFFu, hi = 0;
      for (int i = tid; i < n; i += SAMPLE_THREADS) {
        const float x = x_at(i);
        if (x < low || place_of(x, base + i) > within) continue;
        const uint32_t r = rank_of(x);
        const int b = by_rank ? 0 : bin(x);
        if (by_rank ? r >= r1 && r <= r2 : b >= b1 && b <= b2) lo = min(lo, r), hi = max(hi, r);
      }
      lo = __reduce_min_sync(0xFFFFFFFFu, lo), hi = __reduce_max_sync(0xFFFFFFFFu, hi);
      if (tid == 0) sh.first[me] = 0xFFFFFFFFu, sh.last[me] = 0;
      __syncthreads();
      if ((tid & 31) == 0) atomicMin(&sh.first[me], lo), atomicMax(&sh.last[me], hi);
      __syncthreads();
      lo = sh.first[me], hi = sh.last[me];
      tell(sh.first, lo), tell(sh.last, hi);
      cluster.sync();  // (and the histograms have been read)
      for (int r = 0; r < SAMPLE_CTAS; ++r) lo = min(lo, sh.first[r]), hi = max(hi, sh.last[r]);
      r1 = lo, r2 = hi;
      by_rank = true;
      int shift = 0;
      while (((r2 - r1) >> shift) >= SAMPLE_BINS) ++shift;
      clear_hist();
      double over = 0;
      for (int i = tid; i < n; i += SAMPLE_THREADS) {
        const float x = x_at(i);
        const uint32_t r = rank_of(x);
        if (x < low || place_of(x, base + i) > within || r > r2) continue;
        if (r >= r1) atomicAdd(&sh.hist[(r - r1) >> shift], 1u);
        else if (by_weight) over += weight(x);
      }
      if (by_weight) {
        double all;
        before<double>(over, sh.scan[0], all);
        tell(sh.above, all);
      }
      cluster.sync();
      const double above = by_weight ? total(sh.above) : 0.0;
      const int was = ahead;
      bracket(by_weight, k - was, target - above, 0.0, [&](int b) {
        const u64 r = r1 + ((u64)b << shift);
        return r > r2 ? 0.0 : weight(value_of((uint32_t)r));
      });
      if (by_weight && (shift == 0 || level >= 8) && sh.b1 != sh.b2 && sh.upto - sh.ahead > SAMPLE_LIST) {
        // bins of one value each: the sums are what they are, the first that passes the target is the one.  (And so that this ends whatever the values are.)
        if (tid == 0) sh.b2 = sh.b1;
        __syncthreads();
        uint32_t c = 0;
        for (int r = 0; r < SAMPLE_CTAS; ++r) c += cluster.map_shared_rank(sh.hist, r)[sh.b1];
        if (tid == 0) sh.upto = sh.ahead + (int)c;
        __syncthreads();
      }
      b1 = sh.b1, b2 = sh.b2;
      ahead = was + sh.ahead, upto = was + sh.upto;
      r2 = (uint32_t)min((u64)r2, r1 + (((u64)b2 + 1) << shift) - 1);
      r1 = r1 + ((uint32_t)b1 << shift);
      whole = false;
      if (r1 == r2 && upto - ahead > SAMPLE_LIST) {
        // ---- one value very often: as many of it as are kept, from the lowest index on
        const float x0 = value_of(r1);
        double over1 = 0;
        int equal = 0;
        // (a thread's values side by side: in the order of their indices)
        const int each = (n + SAMPLE_THREADS - 1) / SAMPLE_THREADS | 1, i0 = min(tid * each, n), i1 = min(i0 + each, n);
        for (int i = i0; i < i1; ++i) {
          const float x = x_at(i);
          if (x < low || place_of(x, base + i) > within) continue;
          if (x == x0) ++equal;
          else if (by_weight && x > x0) over1 += weight(x);
        }
        double all = 0;
        int all_equal;
        if (by_weight) before<double>(over1, sh.scan[0], all);
        const int before_me = before<int>(equal, sh.scan_n, all_equal);
        cluster.sync();  // (the last words have been read)
        if (by_weight) tell(sh.above, all);
        tell(sh.equal, all_equal);
        cluster.sync();
        int keep = k - ahead;
        if (by_weight) {
          const double left = (target - total(sh.above)) / weight(x0);
          keep = left < 1.0 ? 1 : left > 2e9 ? 2000000000 : (int)ceil(left);
        }
        int there = 0, off = 0;
        for (int r = 0; r < SAMPLE_CTAS; ++r) {
          if (r < me) off += sh.equal[r];
          there += sh.equal[r];
        }
        keep = min(keep, there);
        off += before_me;
        if (off < keep && keep <= off + equal)
          for (int i = i0, at = off; i < i1; ++i) {
            const float x = x_at(i);
            if (x == x0 && place_of(x, base + i) <= within && ++at == keep)
              for (int r = 0; r < SAMPLE_CTAS; ++r) *cluster.map_shared_rank(&sh.border, r) = place_of(x, base + i);
          }
        cluster.sync();
        return sh.border;
      }
    }
    // ---- the candidates into the first CTA's list
    double over = 0;
    for (int i = tid; i < n; i += SAMPLE_THREADS) {
      const float x = x_at(i);
      const u64 at = place_of(x, base + i);
      if (x < low || at > within) continue;
      const uint32_t r = rank_of(x);
      const int b = by_rank ? 0 : bin(x);
      if (by_rank ? r > r2 : b > b2) continue;
      if (whole || (by_rank ? r >= r1 : b >= b1)) {
        const int to = atomicAdd(cluster.map_shared_rank(&sh.n_list, 0), 1);
        if (to < SAMPLE_LIST) *cluster.map_shared_rank(&sh.list[to], 0) = at;  // (always)
      } else if (by_weight) {
        over += weight(x);
      }
    }
    if (by_weight) {
      double all;
      before<double>(over, sh.scan[0], all);
      if (by_rank) cluster.sync();  // (the last level's words have been read)
      tell(sh.above, all);
    }
    cluster.sync();
    if (me == 0) {
      int count = min(sh.n_list, SAMPLE_LIST);
      sort_list(count);
      if (!by_weight) count = min(count, whole ? k : k - ahead);
      int last = count - 1;
      if (by_weight || (whole && p < 1.0)) {
        double w[4], sum = 0, all;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = 4 * tid + j;
          w[j] = e < count ? weight(value_of((uint32_t)(sh.list[e] >> 32))) : 0.0;
          sum += w[j];
        }
        double at = before<double>(sum, sh.scan[0], all);
        if (by_weight) at += total(sh.above);
        else target = p * all;
        if (tid == 0) sh.pick = count - 1;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          at += w[j];
          if (4 * tid + j < count && at >= target) {
            atomicMin(&sh.pick, 4 * tid + j);
            break;
          }
        }
        __syncthreads();
        last = sh.pick;
      }
      if (tid < SAMPLE_CTAS) *cluster.map_shared_rank(&sh.border, tid) = sh.list[last];
    }
    *both = whole;
    cluster.sync();
    return sh.border;
  }
};

struct SampleParams {
  const float *logits, *u, *temperature, *top_p, *min_p;
  const int* top_k;
  int* ids;
  float* prob;
  size_t stride;
  int n_vocab;
};

__global__ void __cluster_dims__(SAMPLE_CTAS, 1, 1) __launch_bounds__(SAMPLE_THREADS) k_sample(const __grid_constant__ SampleParams p) {
  extern __shared__ __align__(16) float s_x[];
  __shared__ SampleShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, me = (int)cluster.block_rank(), row = blockIdx.x / SAMPLE_CTAS;
  // shares of the row that begin at a multiple of four
  const int per = ((p.n_vocab + SAMPLE_CTAS - 1) / SAMPLE_CTAS + 3) & ~3, base = min(me * per, p.n_vocab), n = min(per, p.n_vocab - base);
  const float* gx = p.logits + (size_t)row * p.stride + base;
  pdl_trigger();
  pdl_wait();
  const float T = p.temperature != nullptr ? __ldcg(p.temperature + row) : 1.f;
  const int top_k = p.top_k != nullptr ? __ldcg(p.top_k + row) : 0;
  const float top_p = p.top_p != nullptr ? __ldcg(p.top_p + row) : 1.f, min_p = p.min_p != nullptr ? __ldcg(p.min_p + row) : 0.f;
  const float u = __ldcg(p.u + row);

  // ---- the row into shared memory; its largest value, the least above -inf, and whether all are numbers
  u64 best = ~0ull;
  float low = CUDART_INF_F;
  int odd = 0;
#pragma unroll 8
  for (int i = tid; i < n; i += SAMPLE_THREADS) {
    const float x = __ldcg(gx + i) + 0.f;  // (-0 is 0)
    if (i < SAMPLE_CAP) s_x[i] = x;
    odd |= x != x;
    if (x > -CUDART_INF_F) low = fminf(low, x);
    best = min(best, place_of(x, base + i));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    best = min(best, __shfl_xor_sync(0xFFFFFFFFu, best, o));
    low = fminf(low, __shfl_xor_sync(0xFFFFFFFFu, low, o));
  }
  if (tid == 0) sh.n_list = 0;
  if ((tid & 31) == 0) sh.list[tid >> 5] = best, sh.scan[0][tid >> 5] = low;
  odd = __syncthreads_or(odd);
  for (int w = 0; w < SAMPLE_WARPS; ++w) best = min(best, sh.list[w]), low = fminf(low, (float)sh.scan[0][w]);
  Sampler s = {sh, cluster, s_x, gx, n, base, me, tid, 0.f, 0.0, 0.f};
  cluster.sync();  // every CTA is there: its memory may be written
  s.tell(sh.best, best), s.tell(sh.low, low), s.tell(sh.odd, odd);
  cluster.sync();
  for (int r = 0; r < SAMPLE_CTAS; ++r) best = min(best, sh.best[r]), odd |= sh.odd[r];
  s.top = value_of((uint32_t)(best >> 32));
  const bool none = odd || s.top == -CUDART_INF_F, greedy = !(T > 0.f) || top_k == 1;
  if (none || greedy) {
    if (me == 0 && tid == 0) {
      p.ids[row] = none ? -1 : (int)(uint32_t)best;
      if (p.prob != nullptr) p.prob[row] = none ? 0.f : 1.f;
    }
    cluster.sync();
    return;
  }
  s.inv_t = 1.0 / (double)T;
  // (an infinite largest value leaves those like it; rounded down, never up)
  const double reach = (double)s.top - SAMPLE_REACH * (double)T;
  s.floor_x = s.top == CUDART_INF_F ? s.top : reach > -3.0e38 ? __double2float_rd(reach) : -3.402823466e38f;

  u64 border = ~0ull;
  bool both = false;
  if (top_k > 0 && top_k < p.n_vocab) border = s.find(border, top_k, (double)top_p, &both);
  if (top_p < 1.f && !both) {
    if (top_p > 0.f) {
      bool done;
      cluster.sync();
      border = s.find(border, 0, (double)top_p, &done);
    } else {
      border = best;
    }
  }

  // ---- the kept weights in the order of the tokens: a thread's side by side
  const double least = min_p > 0.f ? fmin((double)min_p, 1.0) : 0.0;
  const int each = (n + SAMPLE_THREADS - 1) / SAMPLE_THREADS | 1, i0 = min(tid * each, n), i1 = min(i0 + each, n);
  auto kept = [&](int i) {
    const float x = s.x_at(i);
    if (x < s.floor_x || place_of(x, base + i) > border) return 0.0;
    const double w = s.weight(x);
    return w >= least ? w : 0.0;
  };
  double sum = 0, all;
  for (int i = i0; i < i1; ++i) sum += kept(i);
  double at = s.before<double>(sum, sh.scan[0], all);
  if (tid == 0) sh.pick = -1;
  s.tell(sh.kept, all);
  cluster.sync();
  const double whole = s.total(sh.kept), want = (u > 0.f ? fmin((double)u, 1.0) : 0.0) * whole;
  int owner = 0;
  double off = 0, mine = 0;
  for (int r = 0; r < SAMPLE_CTAS; ++r) {  // the last CTA with weights that begins at or before it
    if (sh.kept[r] > 0 && off <= want) owner = r, mine = off;
    off += sh.kept[r];
  }
  if (owner == me) {
    at += mine;
    if (sum > 0 && at <= want) atomicMax(&sh.pick, tid);
    __syncthreads();
    if (tid == sh.pick) {
      int id = -1;
      double w = 0;
      for (int i = i0; i < i1; ++i) {
        const double x = kept(i);
        if (x <= 0) continue;
        id = i, w = x;
        at += x;
        if (at > want) break;
      }
      p.ids[row] = base + id;
      if (p.prob != nullptr) p.prob[row] = (float)(w / whole);
    }
  }
  cluster.sync();
}

}  // namespace

int32_t launch_sample(infr_cuda_ctx* ctx, const float* logits, const float* u, const float* temperature, const int* top_k, const float* top_p, const float* min_p, int* ids,
                      float* prob, size_t stride, int rows, int n_vocab) {
  const SampleParams p = {logits, u, temperature, top_p, min_p, top_k, ids, prob, stride, n_vocab};
  const int per = ((n_vocab + SAMPLE_CTAS - 1) / SAMPLE_CTAS + 3) & ~3;
  const size_t smem = (size_t)(per < SAMPLE_CAP ? per : SAMPLE_CAP) * 4;
  cudaError_t e = ensure_smem(reinterpret_cast<const void*>(&k_sample), (size_t)SAMPLE_CAP * 4);
  if (e == cudaSuccess) e = launch_ex(k_sample, dim3((unsigned)rows * SAMPLE_CTAS), dim3(SAMPLE_THREADS), smem, ctx->stream, true, p);
  if (e != cudaSuccess) return check_cuda(ctx, e, "k_sample launch");
  ctx->launches += 1;
  return check_cuda(ctx, cudaGetLastError(), "k_sample launch");
}

}  // namespace infr
