// A token of each row of logits:
//
//   w_i = exp((x_i - max x) / T)                                                 of the tokens above -inf
//   kept: the top_k largest (of equal ones the lowest), of these the shortest run from the largest that has top_p of their weight, of these
//         those with w_i >= min_p
//   token: the first in order whose weight and the kept ones' ahead of it are more than u times the kept ones' together
//
// What is kept is always a run from the largest, so it is one border: a value and an index.  Finding it needs no sort of the row: a histogram of the values says
// between which of them it lies, and the few that lie there are sorted.  Weights and their sums are f64: with f32 sums the token next to a border would
// go by the order of the additions, and there are 10^5 borders to a row.  Weights below e^-45 of the largest count as none (sample_shape.h): all of them together are
// 2^-47 of 150000 tokens, 2^-40 of the 2^24 that a row may have.  A u below that, 0 among them, would tell: it takes the first kept token with a weight.
//
// A cluster of eight CTAs has a row.  Every decision is made from numbers that all eight have got from one of them, added up in the same order, so that they
// take the same steps and meet at the same barriers whatever the row and its settings hold (and should somebody write them meanwhile).
//
// Measured, of 150000: one row of which the largest is taken 5.1 us, of the 20 largest 7.1, of all 12, of the 1000 largest those with 0.95 25.5, of all with 0.9, spread over
// thousands, 45; 64 rows 17, 25, 40, 65, 137, with settings of all kinds 74.  One pass over the row reads it (2.6 us of the 45); what bounds the rest is the f64 of a
// weight - thirteen operations to a value, in four passes - and the barriers of the cluster, a microsecond each.
#include <cooperative_groups.h>
#include <math_constants.h>

#include "kernels.cuh"
#include "sample_shape.h"

namespace infr {
namespace {

namespace cg = cooperative_groups;

constexpr int SAMPLE_CTAS = 8, SAMPLE_THREADS = 512;
constexpr int SAMPLE_BINS = 2048;
constexpr int SAMPLE_LIST = 2048;     // candidates that are sorted
constexpr int SAMPLE_FEW = 192;       // a run of p of a row's weight is looked for among so many largest ones first
constexpr int SAMPLE_MAXIMA = 1024;   // so many largest ones are looked for by the threads' largest,
constexpr int SAMPLE_FEW_BINS = 256;  // by bins of these,
constexpr int SAMPLE_SLOTS = SAMPLE_LIST / SAMPLE_CTAS;  // and so many candidates of a CTA looked at
constexpr int SAMPLE_CAP = 40960;     // values of a row in a CTA's shared memory at most
typedef unsigned long long u64;

__device__ __forceinline__ float max3_nan(float a, float b, float c) {  // NaN where one is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Values in order: larger ones have smaller numbers; with the index behind them, the order in which tokens are taken.
__device__ __forceinline__ uint32_t rank_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 is 0)
  return b & 0x80000000u ? b : 0x7FFFFFFFu - b;
}
__device__ __forceinline__ float value_of(uint32_t r) { return __uint_as_float(r & 0x80000000u ? r : 0x7FFFFFFFu - r); }
__device__ __forceinline__ u64 place_of(float x, int i) { return (u64)rank_of(x) << 32 | (uint32_t)i; }

struct __align__(16) SampleShared {
  union {
    uint32_t hist[SAMPLE_BINS];
    double few_weight[SAMPLE_THREADS];  // a candidate's to a thread
  };
  union {
    u64 list[SAMPLE_LIST];
    struct {
      uint32_t place[SAMPLE_BINS];   // 64ths of a bin that its values lie behind its beginning, together
      uint32_t places[SAMPLE_BINS];  // and those of all CTAs
    };
  };
  union {
    uint32_t sums[SAMPLE_BINS];  // of all CTAs' hist
    uint32_t few_hist[SAMPLE_CTAS][SAMPLE_FEW_BINS];
  };
  double power[32];            // 2^(j / 32)
  double scan[2][16];
  int scan_n[16];
  float scan_f[2][16];
  // from every CTA, by rank
  float top[SAMPLE_CTAS], least[SAMPLE_CTAS];
  float temperature, top_p, min_p, u;  // from the first CTA
  int top_k;
  int best[SAMPLE_CTAS], n_few[SAMPLE_CTAS];
  double sum[SAMPLE_CTAS], above[SAMPLE_CTAS], kept[SAMPLE_CTAS];
  uint32_t first[SAMPLE_CTAS], last[SAMPLE_CTAS];
  int equal[SAMPLE_CTAS];
  // the first CTA's
  int n_list, done;
  u64 border;
  // of the bins
  int b1, b2, ahead, upto;
  int pick;
};

struct Sampler {
  static constexpr int THREADS = SAMPLE_THREADS, WARPS = THREADS / 32, PER = SAMPLE_BINS / THREADS;  // bins (and candidates) of a thread
  SampleShared& sh;
  cg::cluster_group cluster;
  // This CTA's values, four to a word that lies on a 16-byte boundary: in shared memory, or (xs null) where they came from.  The row begins within its first
  // word as a rule; what is not of the row reads as -inf.
  const float *xs, *row;
  int words, base, n_vocab;  // index of the first value: may be negative
  int me, tid;
  float top;             // the row's largest value
  double steps;          // thirty-seconds of an octave to a unit of the logits: 32 log2(e) / T
  float floor_x;         // values from here on have a weight

  __device__ float4 from_row(int w) const {
    const int i = base + 4 * w;
    if (i >= 0 && i + 3 < n_vocab) return __ldcg(reinterpret_cast<const float4*>(row + i));
    float x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = i + j >= 0 && i + j < n_vocab ? __ldcg(row + i + j) : -CUDART_INF_F;
    return make_float4(x[0], x[1], x[2], x[3]);
  }
  __device__ float4 word(int w) const { return xs != nullptr ? *reinterpret_cast<const float4*>(xs + 4 * w) : from_row(w); }
  // f(value, index) for the values of the words from + k * step
  template <class F>
  __device__ __forceinline__ void each(int from, int to, int step, F f) const {
#pragma unroll 1
    for (int w0 = from; w0 < to; w0 += 2 * step) {
      const bool two = w0 + step < to;
      const float4 a = word(w0);
      float4 b = make_float4(-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F);
      if (two) b = word(w0 + step);
#pragma unroll 1
      for (int k = 0; k < 2; ++k) {
        const float4 v = k == 0 ? a : b;
        const int i = base + 4 * (w0 + k * step);
        f(v.x, i), f(v.y, i + 1), f(v.z, i + 2), f(v.w, i + 3);
      }
    }
  }
  template <class F>
  __device__ __forceinline__ void mine(F f) const { each(tid, words, THREADS, f); }
  // 2^(t / 32) of 64 bits, t <= 0: a table and the exponent for the whole part, five terms of e^r behind the first for the rest, |r| <= log(2) / 64: 2e-15.
  __device__ __forceinline__ double power32(double t) const {
    const double m = t + 6755399441055744.0;  // 1.5 2^52: the sum's low word is t rounded
    const int k = __double2loint(m);
    constexpr double c = 0.69314718055994531 / 32;
    const double f = t - (m - 6755399441055744.0), e = fma(f, fma(f, fma(f, fma(f, fma(f, c * c * c * c * c / 120, c * c * c * c / 24), c * c * c / 6), c * c / 2), c), 1.0) * sh.power[k & 31];
    return __hiloint2double(__double2hiint(e) + (k >> 5) * (1 << 20), __double2loint(e));
  }
  // exp((x - top) / T)
  __device__ __forceinline__ double weight(float x) const {  // (without branches: several at a time)
    const double w = power32(((double)x - (double)top) * steps);
    return x < floor_x ? 0.0 : x == top ? 1.0 : w;
  }
  // Whether a value is one of those up to a border.
  struct Upto {
    float x;
    int i;
    __device__ explicit Upto(u64 border) {
      const bool all = border == ~0ull;
      x = all ? -CUDART_INF_F : value_of((uint32_t)(border >> 32));
      i = all ? 0x7FFFFFFF : (int)(uint32_t)border;
    }
    __device__ __forceinline__ bool has(float y, int j) const { return y > x || (y == x && j <= i); }
  };
  // The weight of all values into every CTA's sum, and that of the threads' largest into `above`; there behind the next cluster barrier.
  __device__ void sum_up(u64 within, float my_top) {
    const Upto in(within);
    double sum = 0, all, largest;
    mine([&](float x, int i) {
      const double w = weight(x);
      sum += in.has(x, i) ? w : 0.0;
    });
    before<double>(sum, sh.scan[0], all);
    before<double>(weight(my_top), sh.scan[1], largest);
    tell(sh.sum, all), tell(sh.above, largest);
  }

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
    for (int w = 0; w < WARPS; ++w) {
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
  // The first CTA's word to all.
  __device__ void tell_one(int* word, int v) {
    if (tid < SAMPLE_CTAS) *cluster.map_shared_rank(word, tid) = v;
  }
  __device__ void clear_hist(bool places) {
    for (int b = tid; b < SAMPLE_BINS; b += THREADS) {
      sh.hist[b] = 0;
      if (places) sh.place[b] = 0;
    }
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
  // (`slack`: by how much of a weight a bin's edges are off.  `places`: how far in their bins the values lie is known: a weight is a convex function of that,
  // at most the chord between the edges, at least a `gap` of the first one's below it)
  template <class Edge>
  __device__ void bracket(bool by_weight, int k, double target, double slack, bool places, double gap, Edge edge) {
    // every CTA adds up an eighth of the bins, and tells the sums to all
    constexpr int EIGHTH = SAMPLE_BINS / SAMPLE_CTAS / 4;
    static_assert(EIGHTH * SAMPLE_CTAS % THREADS == 0, "every thread takes part in every round");
#pragma unroll 1
    for (int e = tid; e < EIGHTH * SAMPLE_CTAS; e += THREADS) {
      const int at = me * EIGHTH + e / SAMPLE_CTAS;  // four bins, by eight neighbouring threads
      uint4 h = reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh.hist, e % SAMPLE_CTAS))[at];
#pragma unroll
      for (int o = 1; o < SAMPLE_CTAS; o <<= 1) {
        h.x += __shfl_xor_sync(0xFFFFFFFFu, h.x, o), h.y += __shfl_xor_sync(0xFFFFFFFFu, h.y, o);
        h.z += __shfl_xor_sync(0xFFFFFFFFu, h.z, o), h.w += __shfl_xor_sync(0xFFFFFFFFu, h.w, o);
      }
      reinterpret_cast<uint4*>(cluster.map_shared_rank(sh.sums, e % SAMPLE_CTAS))[at] = h;
      if (places) {
        h = reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh.place, e % SAMPLE_CTAS))[at];
#pragma unroll
        for (int o = 1; o < SAMPLE_CTAS; o <<= 1) {
          h.x += __shfl_xor_sync(0xFFFFFFFFu, h.x, o), h.y += __shfl_xor_sync(0xFFFFFFFFu, h.y, o);
          h.z += __shfl_xor_sync(0xFFFFFFFFu, h.z, o), h.w += __shfl_xor_sync(0xFFFFFFFFu, h.w, o);
        }
        reinterpret_cast<uint4*>(cluster.map_shared_rank(sh.places, e % SAMPLE_CTAS))[at] = h;
      }
    }
    cluster.sync();
    uint32_t c[PER], sum_c = 0;
#pragma unroll
    for (int j = 0; j < PER; j += 4) {
      const uint4 h = *reinterpret_cast<const uint4*>(sh.sums + PER * tid + j);
      c[j] = h.x, c[j + 1] = h.y, c[j + 2] = h.z, c[j + 3] = h.w;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) sum_c += c[j];
    int all = 0;
    int ahead = before<int>((int)sum_c, sh.scan_n, all);
    if (by_weight) {
      double hi[PER], lo[PER], sum_hi = 0, sum_lo = 0, w = edge(PER * tid);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const double next = edge(PER * tid + j + 1);
        const double far = places ? (w - next) * (sh.places[PER * tid + j] * 0.015625) : 0.0;
        sum_hi += hi[j] = (c[j] * w - far) * (1.0 + slack);
        sum_lo += lo[j] = (places ? c[j] * (w - (w - next) * 0.015625 - w * gap) - far : c[j] * next) * (1.0 - slack);
        w = next;
      }
      double sum;
      double h = before<double>(sum_hi, sh.scan[0], sum), l = before<double>(sum_lo, sh.scan[1], sum);
      int b1 = SAMPLE_BINS, b2 = SAMPLE_BINS, end = -1;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        h += hi[j], l += lo[j];
        if (!c[j]) continue;
        end = PER * tid + j;
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
      for (int j = 0; j < PER; ++j) {
        if (at < k && k <= at + (int)c[j]) sh.b1 = sh.b2 = PER * tid + j;
        at += (int)c[j];
      }
      if (tid == THREADS - 1 && all < k) sh.b1 = sh.b2 = -1;  // all are kept
    }
    __syncthreads();
    const int b1 = sh.b1, b2 = sh.b2;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (PER * tid + j == b1) sh.ahead = ahead;
      ahead += (int)c[j];
      if (PER * tid + j == b2) sh.upto = ahead;
    }
    __syncthreads();
  }

  // The first CTA sorts the candidates, list[0 .. n - 1]: by counting into bins of one width, and within a bin (a few, unless values are equal) by counting
  // again.  (With a network of exchanges 1100 of them took 30 us.)
  __device__ void sort_list(int n) {
    u64 at[PER];
    float low = CUDART_INF_F;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int e = tid + j * THREADS;
      at[j] = e < n ? sh.list[e] : ~0ull;
      if (e < n) low = fminf(low, value_of((uint32_t)(at[j] >> 32)));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) low = fminf(low, __shfl_xor_sync(0xFFFFFFFFu, low, o));
    for (int b = tid; b < SAMPLE_BINS; b += THREADS) sh.hist[b] = 0;
    if ((tid & 31) == 0) sh.scan_f[0][tid >> 5] = low;
    __syncthreads();
    for (int w = 0; w < WARPS; ++w) low = fminf(low, sh.scan_f[0][w]);
    const float scale = top > low ? (float)((SAMPLE_BINS - 1) / (0.5 * ((double)top - (double)low))) : 0.f, half = 0.5f * top;
    int bin[PER], order[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      bin[j] = min((int)(fmaf(-0.5f, value_of((uint32_t)(at[j] >> 32)), half) * scale), SAMPLE_BINS - 1);
      if (tid + j * THREADS < n) order[j] = atomicAdd(&sh.hist[bin[j]], 1u);
    }
    __syncthreads();
    int sum = 0, all;
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += (int)sh.hist[PER * tid + j];
    int ahead = before<int>(sum, sh.scan_n, all);
#pragma unroll
    for (int j = 0; j < PER; ++j) sh.sums[PER * tid + j] = ahead, ahead += (int)sh.hist[PER * tid + j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (tid + j * THREADS < n) sh.list[sh.sums[bin[j]] + order[j]] = at[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (tid + j * THREADS < n) {
        const int first = sh.sums[bin[j]], count = sh.hist[bin[j]];
        order[j] = first;
#pragma unroll 1
        for (int i = first; i < first + count; ++i) order[j] += sh.list[i] < at[j];
      }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (tid + j * THREADS < n) sh.list[order[j]] = at[j];
    __syncthreads();
  }

  // The weights of the list's first `count` candidates, the thread's own in w, and the sum ahead of them.
  __device__ double list_weights(int count, double (&w)[PER], double& all) {
    double sum = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int e = PER * tid + j;
      w[j] = e < count ? weight(value_of((uint32_t)(sh.list[e] >> 32))) : 0.0;
      sum += w[j];
    }
    return before<double>(sum, sh.scan[0], all);
  }
  // The first of them with which the sum from `at` on reaches the target; the last one with a weight if none does.
  __device__ int list_find(int count, const double (&w)[PER], double at, double target) {
    if (tid == 0) sh.pick = SAMPLE_LIST, sh.b1 = -1;
    __syncthreads();
    int found = SAMPLE_LIST, last = -1;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      at += w[j];
      if (PER * tid + j >= count || w[j] <= 0) continue;
      last = PER * tid + j;
      if (found == SAMPLE_LIST && at >= target) found = last;
    }
    if (found < SAMPLE_LIST) atomicMin(&sh.pick, found);
    if (last >= 0) atomicMax(&sh.b1, last);
    __syncthreads();
    const int to = sh.pick == SAMPLE_LIST ? sh.b1 : sh.pick;
    __syncthreads();
    return to;
  }

  // Bins of one width from the largest value down to `low`, in 64 places each: the nearest place (a half of one behind, and f32's 2^-22 of the distance).
  // (A difference of halves does not overflow.)
  float place_scale, bin_half;
  __device__ void set_bins(float low) {
    place_scale = top > low ? (float)((double)(64 * (SAMPLE_BINS - 1)) / (0.5 * ((double)top - (double)low))) : 0.f;
    bin_half = 0.5f * top;
  }
  __device__ uint32_t place(float x) const {  // from half a bin ahead of the largest value on
    const float b = fminf(fmaf(fmaf(-0.5f, x, bin_half), place_scale, 8388608.f), 8388608.f + (64 * (SAMPLE_BINS - 1) + 31));
    return (__float_as_uint(b) & 0x7FFFFFu) + 32;
  }
  __device__ int bin(float x) const { return (int)(place(x) >> 6); }

  // The first rank from `first` on (up to the one of `low`, or one more) whose value is in bin b or one behind it: a warp's lanes at 32 places at a time.
  __device__ uint32_t rank_of_bin(int b, float low) const {
    u64 lo = rank_of(top), hi = (u64)rank_of(low) + 1;
#pragma unroll 1
    while (lo < hi) {
      const u64 step = (hi - lo + 31) / 32, at = lo + (tid & 31) * step;
      const bool ahead = at < hi && bin(value_of((uint32_t)at)) < b;
      const int n = __popc(__ballot_sync(0xFFFFFFFFu, ahead));  // (the lanes ahead are the first ones)
      if (n == 0) break;
      lo += (n - 1) * step + 1;
      hi = min(hi, lo + step - 1);
    }
    return (uint32_t)lo;
  }

  // The border of the first CTA's n candidates, to all: that of the k largest and (p < 1) of the run with p of their weight.
  __device__ void cut_list(int n, int k, double p) {
    sort_list(n);
    int last = max(0, min(n, k) - 1);
    if (p < 1.0) {
      double w[PER], all;
      const double at = list_weights(last + 1, w, all);
      last = max(0, list_find(last + 1, w, at, p * all));
    }
    if (tid < SAMPLE_CTAS) *cluster.map_shared_rank(&sh.border, tid) = sh.list[last];
  }

  // The token where no more than the k largest are needed: they are among the values that share a bin with the k-th largest of the threads' largest, or are
  // larger, and only the threads that have such a one look through their values again.  If these are few, the first CTA sorts them by counting (a thread to each)
  // and takes the token by itself; of more it finds the border.  of_all: the run has p of the whole row's weight (and may need more than these), else of the k
  // largest's.  NOTHING: too many candidates, or too few.
  enum Found { NOTHING, TOKEN, BORDER };
  __device__ Found few_largest(int k, bool of_all, double p, double least, double u, float my_top, float least_top, int* id, float* prob) {
    const double width = top > least_top ? (SAMPLE_FEW_BINS - 1) / (0.5 * ((double)top - (double)least_top)) : 0.0;
    const float scale = (float)width, half = 0.5f * top;
    auto few_bin = [&](float x) { return min((int)(fmaf(-0.5f, x, half) * scale), SAMPLE_FEW_BINS - 1); };
    if (tid < SAMPLE_FEW_BINS) sh.hist[tid] = 0;
    if (tid == 0) sh.n_list = 0, sh.done = 0;
    __syncthreads();
    const bool has = my_top > -CUDART_INF_F;
    const int my_bin = has ? few_bin(my_top) : SAMPLE_FEW_BINS;
    if (has) atomicAdd(&sh.hist[my_bin], 1u);
    __syncthreads();
    for (int e = tid; e < SAMPLE_FEW_BINS * SAMPLE_CTAS; e += THREADS)
      cluster.map_shared_rank(&sh.few_hist[me][0], e / SAMPLE_FEW_BINS)[e % SAMPLE_FEW_BINS] = sh.hist[e % SAMPLE_FEW_BINS];
    cluster.sync();
    int c = 0, all;
    if (tid < SAMPLE_FEW_BINS)
      for (int r = 0; r < SAMPLE_CTAS; ++r) c += (int)sh.few_hist[r][tid];
    const int ahead = before<int>(c, sh.scan_n, all);
    if (ahead < k && k <= ahead + c) sh.b2 = tid;
    __syncthreads();
    const int b2 = all >= k ? sh.b2 : -1;
    // a warp's lanes together for each of its threads that have candidates
#pragma unroll 1
    for (uint32_t ask = __ballot_sync(0xFFFFFFFFu, my_bin <= b2); ask; ask &= ask - 1) {
      const int from = (tid & ~31) + __ffs(ask) - 1;
#pragma unroll 1
      for (int w = from + (tid & 31) * THREADS; w < words; w += 32 * THREADS) {
        const float4 v = word(w);
        const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (x[j] > -CUDART_INF_F && few_bin(x[j]) <= b2) {
            const int to = atomicAdd(&sh.n_list, 1);
            if (to < SAMPLE_SLOTS) *cluster.map_shared_rank(&sh.list[me * SAMPLE_SLOTS + to], 0) = place_of(x[j], base + 4 * w + j);
          }
      }
    }
    __syncthreads();
    tell(sh.n_few, b2 < 0 ? SAMPLE_SLOTS + 1 : sh.n_list);
    cluster.sync();
    int n = 0;
    for (int r = 0; r < SAMPLE_CTAS; ++r) {
      if (sh.n_few[r] > SAMPLE_SLOTS) return NOTHING;
      n += sh.n_few[r];
    }
    if (n > THREADS) {
      if (of_all) return NOTHING;
      if (me == 0) {
        u64 at[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          int e = tid + j * THREADS;
          at[j] = ~0ull;
#pragma unroll 1
          for (int r = 0; r < SAMPLE_CTAS; ++r) {
            if (e >= 0 && e < sh.n_few[r]) at[j] = sh.list[r * SAMPLE_SLOTS + e];
            e -= sh.n_few[r];
          }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (tid + j * THREADS < n) sh.list[tid + j * THREADS] = at[j];
        __syncthreads();
        cut_list(n, k, p);
      }
      cluster.sync();
      return BORDER;
    }
    bool done = true;
    if (me == 0) {
      // thread e has candidate e
      u64 at = ~0ull;
      int e = tid;
      for (int r = 0; r < SAMPLE_CTAS; ++r) {
        if (e >= 0 && e < sh.n_few[r]) at = sh.list[r * SAMPLE_SLOTS + e];
        e -= sh.n_few[r];
      }
      double w = tid < n ? weight(value_of((uint32_t)(at >> 32))) : 0.0;
      __syncthreads();
      if (tid < n) sh.list[tid] = at;
      __syncthreads();
      int rank = 0;
#pragma unroll 4
      for (int i = 0; i < n; ++i) rank += sh.list[i] < at;
      __syncthreads();
      if (tid < n) sh.list[rank] = at, sh.few_weight[rank] = w;
      __syncthreads();
      // thread r has rank r
      at = tid < n ? sh.list[tid] : ~0ull;
      w = tid < n && (of_all || tid < k) ? sh.few_weight[tid] : 0.0;
      int count = of_all ? n : min(n, k);
      if (p < 1.0) {
        double sum;
        const double ahead_w = before<double>(w, sh.scan[0], sum), target = p * (of_all ? total(sh.sum) : sum);
        // (as they are added one by one, the first with which the sum reaches the target is the last)
        const int over = __syncthreads_count(tid < count && !(ahead_w + w >= target));
        done = over < count || !of_all;
        count = min(count, over + 1);
      }
      if (done) {  // (else the candidates are not enough)
        if (tid < count && (w <= 0 || w < least)) w = 0.0;
        if (tid < count) sh.few_weight[tid] = w;
        if (tid == 0) sh.pick = -1;
        __syncthreads();
        const int index = (int)(uint32_t)at;
        double lower = 0, kept = 0;
#pragma unroll 4
        for (int i = 0; i < count; ++i) {
          const double x = sh.few_weight[i];
          kept += x;
          if ((int)(uint32_t)sh.list[i] < index) lower += x;
        }
        if (tid < count && w > 0 && lower <= u * kept) atomicMax(&sh.pick, index);
        __syncthreads();
        if (done && tid < count && w > 0 && index == sh.pick) {
          *id = index;
          if (prob != nullptr) *prob = (float)(w / kept);
        }
      }
    }
    if (!of_all) return TOKEN;  // (nothing of another CTA is waited for)
    if (me == 0) tell_one(&sh.done, done ? 1 : 0);
    cluster.sync();
    return sh.done != 0 ? TOKEN : NOTHING;
  }

  // The border among the values up to `within`: that of the k largest, or with p < 1 that of the run with p of the weight, or (k, then p) both where the
  // candidates hold all of the k; *both: whether they did.
  __device__ u64 find(u64 within, int k, double p, bool* both) {
    const bool by_weight = k <= 0;
    const Upto in(within);
    *both = false;
    // ---- bins down to the least value that has a weight (a border of the k largest may lie behind: then nothing is left out)
    float low = floor_x;
    if (by_weight) {
      // (or could be the border: from it on lies more than 1 - p of the weight, in n_vocab values at most, none of them above it)
      const double least = (double)top + 32.0 * log2(0.999 * (1.0 - p) * total(sh.sum) / n_vocab) / steps;
      if (least > (double)low) low = __double2float_rd(least);
    }
    set_bins(low);
    clear_hist(by_weight);
    mine([&](float x, int i) {
      if (x >= low && in.has(x, i)) {
        const uint32_t at = place(x);
        atomicAdd(&sh.hist[at >> 6], 1u);
        if (by_weight) atomicAdd(&sh.place[at >> 6], at & 63);
      }
    });
    cluster.sync();
    const double target = by_weight ? p * total(sh.sum) : 0;
    const double width = place_scale > 0.f ? 128.0 * steps / place_scale : 0.0, gap = (width * (0.69314718055994531 / 32)) * (width * (0.69314718055994531 / 32)) / 8;
    // (f32 moves a bin's edges by 2^-22 of their distance from the largest, which is 45 in the exponent at most)
    bracket(by_weight, k, target, 3e-5, by_weight, gap, [&](int b) { return power32((0.5 + 1.0 / 128 - b) * width); });
    int b1 = sh.b1, b2 = sh.b2, ahead = sh.ahead, upto = sh.upto;
    if (b1 < 0) return within;
    bool whole = !by_weight && upto <= SAMPLE_LIST;  // the list takes what lies ahead too
    uint32_t r1 = 0, r2 = 0;                          // the candidates as a range of ranks, once the bins are not enough
    bool by_rank = false;
    double above = 0;          // by weight: of the values ahead of rank `from`, in all CTAs
    uint32_t from = 0;
    for (int level = 0;; ++level) {
      const int n_list = whole ? upto : upto - ahead;
      if (n_list <= SAMPLE_LIST) break;
      // ---- too many: bins of ranks, 2^11 to the candidates' range; after three of these a bin is one value
      uint32_t lo = 0xFFFFFFFFu, hi = 0;
      mine([&](float x, int i) {
        if (x < low || !in.has(x, i)) return;
        const uint32_t r = rank_of(x);
        const int b = by_rank ? 0 : bin(x);
        if (by_rank ? r >= r1 && r <= r2 : b >= b1 && b <= b2) lo = min(lo, r), hi = max(hi, r);
      });
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
      clear_hist(false);
      double over = 0;
      mine([&](float x, int i) {
        const uint32_t r = rank_of(x);
        if (x < low || r > r2 || !in.has(x, i)) return;
        if (r >= r1) atomicAdd(&sh.hist[(r - r1) >> shift], 1u);
        else if (by_weight) over += weight(x);
      });
      if (by_weight) {
        double all;
        before<double>(over, sh.scan[0], all);
        tell(sh.above, all);
      }
      cluster.sync();
      if (by_weight) above = total(sh.above);
      from = r1;
      const int was = ahead;
      bracket(by_weight, k - was, target - above, 0.0, false, 0.0, [&](int b) {
        const u64 r = r1 + ((u64)b << shift);
        return r > r2 ? 0.0 : weight(value_of((uint32_t)r));
      });
      b1 = sh.b1, b2 = sh.b2;
      if (b1 < 0 || level >= 16) return within;  // (not with values that stay as they are)
      int in_bins = sh.upto - sh.ahead;
      if (by_weight && (shift == 0 || level >= 8) && b1 != b2 && in_bins > SAMPLE_LIST) {
        // bins of one value each: the sums are what they are, the first that passes the target is the one.  (And so that the range becomes a bin's at last.)
        b2 = b1;
        in_bins = (int)sh.sums[b1];
      }
      ahead = was + sh.ahead, upto = ahead + in_bins;
      r2 = (uint32_t)min((u64)r2, r1 + (((u64)b2 + 1) << shift) - 1);
      r1 = r1 + ((uint32_t)b1 << shift);
      whole = false;
      if (r1 == r2 && upto - ahead > SAMPLE_LIST) {
        // ---- one value very often: as many of it as are kept, from the lowest index on
        const float x0 = value_of(r1);
        double over1 = 0;
        int equal = 0;
        // (a thread's words side by side: in the order of their indices)
        const int own = (words + THREADS - 1) / THREADS, w0 = min(tid * own, words), w1 = min(w0 + own, words);
        each(w0, w1, 1, [&](float x, int i) {
          if (x < low || !in.has(x, i)) return;
          if (x == x0) ++equal;
          else if (by_weight && x > x0) over1 += weight(x);
        });
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
        if (off < keep && keep <= off + equal) {
          int at = off;
          each(w0, w1, 1, [&](float x, int i) {
            if (x == x0 && in.has(x, i) && ++at == keep)
              for (int r = 0; r < SAMPLE_CTAS; ++r) *cluster.map_shared_rank(&sh.border, r) = place_of(x, i);
          });
        }
        cluster.sync();
        return sh.border;
      }
    }
    // ---- the candidates into a list of this CTA's, from which the first one fetches them (one by one into its list they waited a microsecond each)
    if (!by_rank) r1 = rank_of_bin(b1, low), r2 = rank_of_bin(b2 + 1, low) - 1;
    const float x1 = whole ? CUDART_INF_F : value_of(r1), x2 = value_of(r2), x0 = by_rank ? value_of(from) : CUDART_INF_F;
    double over = 0;
    mine([&](float x, int i) {
      const bool has = x >= x2 && in.has(x, i), listed = has && x <= x1;
      if (by_weight) {  // (a weight to all: several at a time, without branches)
        const double w = weight(x);
        over += has && !listed && x <= x0 ? w : 0.0;
      }
      if (listed) {
        const int to = atomicAdd(&sh.n_list, 1);
        if (to < SAMPLE_LIST) sh.list[to] = place_of(x, i);  // (always)
      }
    });
    if (by_weight) {
      double all;
      before<double>(over, sh.scan[0], all);
      if (by_rank) cluster.sync();  // (the last level's words have been read)
      tell(sh.above, all);
    }
    __syncthreads();
    tell(sh.n_few, sh.n_list);
    cluster.sync();
    if (me == 0) {
      int count = 0;
#pragma unroll 1
      for (int r = 0; r < SAMPLE_CTAS; ++r) {
        const int n = min(sh.n_few[r], SAMPLE_LIST - count);
        if (r > 0)
          for (int e = tid; e < n; e += THREADS) sh.list[count + e] = cluster.map_shared_rank(sh.list, r)[e];
        count += n;
      }
      __syncthreads();
      if (!by_weight) {
        cut_list(count, whole ? k : k - ahead, whole ? p : 1.0);
      } else {
        sort_list(count);
        double w[PER], all;
        const double at = list_weights(count, w, all);
        const int last = max(0, list_find(count, w, at + (above + total(sh.above)), target));
        if (tid < SAMPLE_CTAS) *cluster.map_shared_rank(&sh.border, tid) = sh.list[last];
      }
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
  int n_vocab, cached;
};

__global__ void __cluster_dims__(SAMPLE_CTAS, 1, 1) __launch_bounds__(SAMPLE_THREADS, 2) k_sample(const __grid_constant__ SampleParams p) {
  extern __shared__ __align__(16) float s_x[];
  __shared__ SampleShared sh;
  constexpr int THREADS = SAMPLE_THREADS, WARPS = THREADS / 32;
  cg::cluster_group cluster = cg::this_cluster();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // waited for ahead of the first word to another CTA: all are there then
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, me = (int)cluster.block_rank(), row = blockIdx.x / SAMPLE_CTAS;
  const float* x = p.logits + (size_t)row * p.stride;
  const int lead = (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3);  // values of the row's first word that are not the row's
  const int all_words = (p.n_vocab + lead + 3) / 4, per = (all_words + SAMPLE_CTAS - 1) / SAMPLE_CTAS, w0 = min(me * per, all_words);
  Sampler s = {sh, cluster, p.cached ? s_x : nullptr, x, min(per, all_words - w0), 4 * w0 - lead, p.n_vocab, me, tid, 0.f, 0.0, 0.f, 0.f, 0.f};
  if (tid < 32) sh.power[tid] = exp2(tid * 0.03125);
  pdl_trigger();
  pdl_wait();
  float T = 1.f, top_p = 1.f, min_p = 0.f, u = 0.f;
  int top_k = 0;
  if (me == 0 && tid < SAMPLE_CTAS) {
    if (p.temperature != nullptr) T = __ldcg(p.temperature + row);
    if (p.top_k != nullptr) top_k = __ldcg(p.top_k + row);
    if (p.top_p != nullptr) top_p = __ldcg(p.top_p + row);
    if (p.min_p != nullptr) min_p = __ldcg(p.min_p + row);
    u = __ldcg(p.u + row);
  }

  // ---- the row, once: its largest value (NaN where one is), and every thread's largest
  float top = -CUDART_INF_F;
#pragma unroll 1
  for (int v0 = tid; v0 < s.words; v0 += 6 * THREADS) {
    float4 v[6];
#pragma unroll
    for (int k = 0; k < 6; ++k)
      if (v0 + k * THREADS < s.words) v[k] = s.from_row(v0 + k * THREADS);
#pragma unroll
    for (int k = 0; k < 6; ++k) {
      if (v0 + k * THREADS >= s.words) break;
      if (p.cached) *reinterpret_cast<float4*>(s_x + 4 * (v0 + k * THREADS)) = v[k];
      top = max3_nan(max3_nan(top, v[k].x, v[k].y), v[k].z, v[k].w);
    }
  }
  const float my_top = top;
  float least_top = my_top > -CUDART_INF_F ? my_top : CUDART_INF_F;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top = max3_nan(top, top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    least_top = fminf(least_top, __shfl_xor_sync(0xFFFFFFFFu, least_top, o));
  }
  if (lane == 0) sh.scan_f[0][warp] = top, sh.scan_f[1][warp] = least_top;
  if (tid == 0) sh.n_list = 0, sh.pick = 0x7FFFFFFF;
  __syncthreads();
  for (int w = 0; w < WARPS; ++w) top = max3_nan(top, top, sh.scan_f[0][w]), least_top = fminf(least_top, sh.scan_f[1][w]);
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  s.tell(sh.top, top), s.tell(sh.least, least_top);
  if (me == 0 && tid < SAMPLE_CTAS) {
    SampleShared* to = cluster.map_shared_rank(&sh, tid);
    to->temperature = T, to->top_p = top_p, to->min_p = min_p, to->u = u, to->top_k = top_k;
  }
  cluster.sync();
  T = sh.temperature, top_p = sh.top_p, min_p = sh.min_p, u = sh.u, top_k = sh.top_k;
  for (int r = 0; r < SAMPLE_CTAS; ++r) top = max3_nan(top, top, sh.top[r]), least_top = fminf(least_top, sh.least[r]);
  s.top = top;
  const bool none = !(top > -CUDART_INF_F);
  if (none || !(T > 0.f) || top_k == 1 || top_p <= 0.f) {
    // ---- nothing to take, or the first of the largest
    if (my_top == top) s.mine([&](float y, int i) {
      if (y == top) atomicMin(&sh.pick, i);
    });
    __syncthreads();
    s.tell(sh.best, sh.pick);
    cluster.sync();
    if (me == 0 && tid == 0) {
      int id = sh.best[0];
      for (int r = 1; r < SAMPLE_CTAS; ++r) id = min(id, sh.best[r]);
      p.ids[row] = none ? -1 : id;
      if (p.prob != nullptr) p.prob[row] = none ? 0.f : 1.f;
    }
    return;
  }
  s.steps = 46.166241308446828 / (double)T;  // 32 log2(e)
  s.floor_x = sample_floor(top, T);
  const double least = min_p > 0.f ? fmin((double)min_p, 1.0) : 0.0, part = u > 0.f ? fmin((double)u, 1.0) : 0.0;

  u64 border = ~0ull;
  bool both = false;
  int* id_out = p.ids + row;
  float* prob_out = p.prob != nullptr ? p.prob + row : nullptr;
  const bool limited = top_k > 0 && top_k < p.n_vocab;
  if (limited && top_k <= SAMPLE_MAXIMA) {
    const auto found = s.few_largest(top_k, false, (double)top_p, least, part, my_top, least_top, id_out, prob_out);
    if (found == s.TOKEN) return;
    if (found == s.BORDER) border = sh.border, both = true;
  }
  if (!limited && top_p < 1.f) {  // (mostly a short run)
    s.sum_up(border, my_top);
    cluster.sync();
    // (where the threads' largest together are less than the run, as good as never)
    if (s.total(sh.above) >= (double)top_p * s.total(sh.sum) && s.few_largest(SAMPLE_FEW, true, (double)top_p, least, part, my_top, least_top, id_out, prob_out) == s.TOKEN) return;
  }
  if (limited && !both) border = s.find(border, top_k, (double)top_p, &both);
  if (top_p < 1.f && !both) {
    bool done;
    cluster.sync();
    if (limited) {
      s.sum_up(border, my_top);
      cluster.sync();
    }
    border = s.find(border, 0, (double)top_p, &done);
  }

  // ---- the kept weights in the order of the tokens: a warp's words side by side
  const Sampler::Upto in(border);
  const int own = (s.words + WARPS - 1) / WARPS, v0 = min(warp * own, s.words), v1 = min(v0 + own, s.words);
  const float cutoff = fmaxf(in.x, s.floor_x);
  auto kept = [&](float y, int i) {
    if (y < cutoff) return 0.0;
    const double w = s.weight(y);
    return w >= least && in.has(y, i) ? w : 0.0;
  };
  double sum = 0;
  if (border == ~0ull && least == 0.0) {
    s.each(v0 + lane, v1, 32, [&](float y, int) { sum += s.weight(y); });
  } else {
    s.each(v0 + lane, v1, 32, [&](float y, int i) { sum += kept(y, i); });
  }
  sum = s.warp_total(sum);
  __syncthreads();
  if (lane == 0) sh.scan[0][warp] = sum;
  __syncthreads();
  double all = 0;
  for (int w = 0; w < WARPS; ++w) all += sh.scan[0][w];
  s.tell(sh.kept, all);
  cluster.sync();
  const double whole = s.total(sh.kept), want = part * whole;
  int owner = 0;
  double off = 0, at = 0;
  for (int r = 0; r < SAMPLE_CTAS; ++r) {  // the last CTA with weights that begins at or before it
    if (sh.kept[r] > 0 && off <= want) owner = r, at = off;
    off += sh.kept[r];
  }
  if (owner != me) return;
  int from = 0;
  off = at;
  for (int w = 0; w < WARPS; ++w) {  // and its last such warp
    if (sh.scan[0][w] > 0 && off <= want) from = w, at = off;
    off += sh.scan[0][w];
  }
  if (from != warp) return;
  // its words again, 32 at a time: the first value that passes, or the last with a weight
  int id = -1;
  double w_id = 0;
#pragma unroll 1
  for (int v = v0; v < v1; v += 32) {
    double w[4] = {0, 0, 0, 0};
    const int i = s.base + 4 * (v + lane);
    if (v + lane < v1) {
      const float4 y = s.word(v + lane);
      w[0] = kept(y.x, i), w[1] = kept(y.y, i + 1), w[2] = kept(y.z, i + 2), w[3] = kept(y.w, i + 3);
    }
    double ahead = (w[0] + w[1]) + (w[2] + w[3]);
    const double four = ahead;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xFFFFFFFFu, ahead, o);
      if (lane >= o) ahead += y;
    }
    const double next = at + __shfl_sync(0xFFFFFFFFu, ahead, 31);
    double here = at + (ahead - four);
    int mine = -1, last = -1;
    double w_mine = 0, w_last = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      here += w[j];
      if (w[j] <= 0) continue;
      last = i + j, w_last = w[j];
      if (mine < 0 && here > want) mine = last, w_mine = w_last;
    }
    const uint32_t has = __ballot_sync(0xFFFFFFFFu, mine >= 0), any = __ballot_sync(0xFFFFFFFFu, last >= 0);
    const int lane_at = has ? __ffs(has) - 1 : any ? 31 - __clz(any) : 0;
    if (has || any) {
      id = __shfl_sync(0xFFFFFFFFu, has ? mine : last, lane_at);
      w_id = __shfl_sync(0xFFFFFFFFu, has ? w_mine : w_last, lane_at);
    }
    if (has) break;
    at = next;
  }
  if (lane == 0) {
    p.ids[row] = id;
    if (p.prob != nullptr) p.prob[row] = (float)(w_id / whole);
  }
}

}  // namespace

int32_t launch_sample(infr_cuda_ctx* ctx, const float* logits, const float* u, const float* temperature, const int* top_k, const float* top_p, const float* min_p, int* ids,
                      float* prob, size_t stride, int rows, int n_vocab) {
  SampleParams p = {logits, u, temperature, top_p, min_p, top_k, ids, prob, stride, n_vocab, 0};
  const int per = ((n_vocab + 3 + 3) / 4 + SAMPLE_CTAS - 1) / SAMPLE_CTAS * 4;
  // A row that fits is kept in shared memory, which leaves room for 37 rows at a time.  That was measured with 64 rows of 150000, settings of all kinds: kept 98 us, read
  // again from L2 108, with 256 threads to a CTA (all rows at once then, but each of them slower) 141, with four CTAs to a row 128.  Where all 64 take one of the 20 largest
  // the choice loses: 25 us, 26 from L2, but 17 with 256 threads.
  p.cached = per <= SAMPLE_CAP;
  const size_t smem = p.cached ? (size_t)per * 4 : 0;
  cudaError_t e = ensure_smem(reinterpret_cast<const void*>(&k_sample), (size_t)SAMPLE_CAP * 4);
  if (e == cudaSuccess) e = launch_ex(k_sample, dim3((unsigned)rows * SAMPLE_CTAS), dim3(SAMPLE_THREADS), smem, ctx->stream, true, p);
  if (e != cudaSuccess) return check_cuda(ctx, e, "k_sample launch");
  ctx->launches += 1;
  return check_cuda(ctx, cudaGetLastError(), "k_sample launch");
}

}  // namespace infr
