// What stands between a layer's q / k / v rows and its attention: per-head RMS norm and rotary embedding of q and k, k and v rounded to
// f16 into the cache.  Every value is read once and written once: memory bounds it.
//
// Sixteen lanes own a head; a lane takes eight values at a time as two 16-byte words that hold four whole pairs (halves style: the words
// are half the rotated range apart; interleaved: neighbours), so that a pair never leaves its lane.  The angles are products of a position
// and a frequency in 64 bits, reduced to a fraction of a turn before they are rounded to 32 (a position of 10^6 times a frequency near 1
// keeps 4 bits of f32 after the point); a row's sines are worked out once for all of its heads, by as many threads as there are pairs in a
// few rows.
//
// Measured: 8192 rows of 32 + 2 x 4 heads of 128 59.9 us, 5.3 TB/s of the rows and the cache (0.81 of the copy rate; 62.4 with heads divided
// out of an index instead of counted on, 64.5 with five CTAs to an SM in place of four); 777 rows 9.9 us, 32 rows 4.8 us: launch, plan, one row's chain.
#include "attn.cuh"

namespace infr {
namespace {

constexpr int ROPE_THREADS = 256, ROPE_TEAMS = ROPE_THREADS / 16, ROPE_MAX_PAIRS = 128, ROPE_ROWS = 4;

__device__ __forceinline__ float team_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float x = a * c - b * s;
  b = a * s + b * c;
  a = x;
}

__device__ __forceinline__ void store4_f16(__half* dst, const float4& v) {
  const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
  *reinterpret_cast<uint2*>(dst) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// JS: eight-value chunks of a lane: 1 for heads up to 128, else 2.
template <int JS>
__global__ void __launch_bounds__(ROPE_THREADS) k_rope_kv(const __grid_constant__ RopeParams p) {
  __shared__ __align__(16) float s_cos[ROPE_ROWS * ROPE_MAX_PAIRS], s_sin[ROPE_ROWS * ROPE_MAX_PAIRS];
  __shared__ int s_pos[ROPE_ROWS], s_first;
  __shared__ long long s_at[ROPE_ROWS];
  const int tid = threadIdx.x, team = tid >> 4, tl = tid & 15, lane = tid & 31;
  const int pairs = p.n_rot / 2, batch = pairs ? min(ROPE_ROWS, ROPE_THREADS / pairs) : ROPE_ROWS;
  const int my_row = pairs ? tid / pairs : 0, my_pair = pairs ? tid - my_row * pairs : 0;
  const bool turns_one = pairs && my_row < batch;
  pdl_trigger();
  double turns = p.turns0, x = p.ratio;  // of this thread's pair, per token: turns0 * ratio^pair by squares
#pragma unroll 1
  for (int b = my_pair; b; b >>= 1, x *= x)
    if (b & 1) turns *= x;
  const int n_vec = p.n_head + 2 * p.n_kv, chunks = p.hd / 8, rot = p.n_rot / 8;
  int oa[JS], ob[JS];
#pragma unroll
  for (int j = 0; j < JS; ++j) {
    const int c = tl + 16 * j;
    oa[j] = !p.interleaved && c < rot ? 4 * c : 8 * c;
    ob[j] = !p.interleaved && c < rot ? p.n_rot / 2 + 4 * c : 8 * c + 4;
  }
  const int r0 = (int)((long long)blockIdx.x * p.rows / gridDim.x), r1 = (int)((long long)(blockIdx.x + 1) * p.rows / gridDim.x);
  pdl_wait();
  if (turns_one && p.freq_factors != nullptr) turns /= (double)p.freq_factors[my_pair];
  if (tid < 32) {
    // the last sequence that begins at or before the first row (rows ahead of cu_q[0] belong to none): 32 places at a time
    int lo = 0, hi = p.n_seq;
#pragma unroll 1
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, i = lo + lane * step;
      const int n = __popc(__ballot_sync(0xFFFFFFFFu, i < hi && __ldcg(p.cu_q + i) <= r0));
      lo += max(n - 1, 0) * step;
      hi = min(hi, lo + step);
    }
    if (lane == 0) s_first = lo;
  }
  __syncthreads();
  bool bad = false;
  int s = s_first;
  AttnSeq seq = {0, 0, 0};
  auto load = [&](int i) {
    return attn_seq(__ldcg(p.cu_q + i), __ldcg(p.cu_q + i + 1), p.kv_len != nullptr ? __ldcg(p.kv_len + i) : 0, p.kv_len == nullptr, p.rows, p.cap, &bad);
  };
  if (tid < batch) seq = load(s);

  float4 a[JS], b[JS];  // of the head that comes next
  int fi = 0, fh = 0;   // its row of the batch and its number
  auto fetch = [&](int row0, int rows) {
    while (fh >= n_vec) fh -= n_vec, ++fi;
    const int i = fi, h = fh, r = row0 + i;
    const bool is_q = h < p.n_head, is_v = h >= p.n_head + p.n_kv;
    const float* src = is_q ? p.q + (size_t)r * p.q_stride + (size_t)h * p.hd
                            : (is_v ? p.v + (size_t)r * p.v_stride + (size_t)(h - p.n_head - p.n_kv) * p.hd : p.k + (size_t)r * p.k_stride + (size_t)(h - p.n_head) * p.hd);
#pragma unroll
    for (int j = 0; j < JS; ++j) {
      a[j] = b[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < rows && tl + 16 * j < chunks) {
        a[j] = __ldcg(reinterpret_cast<const float4*>(src + oa[j]));
        b[j] = __ldcg(reinterpret_cast<const float4*>(src + ob[j]));
      }
    }
  };

#pragma unroll 1
  for (int row0 = r0; row0 < r1; row0 += batch) {
    const int rows = min(batch, r1 - row0);
    fi = 0, fh = team;
    fetch(row0, rows);
    if (tid < rows) {  // positions, and places in the cache (-1: none)
      const int r = row0 + tid;
#pragma unroll 1
      while (s + 1 < p.n_seq && r >= seq.q0 + seq.q_len) seq = load(++s);
      const int pos = seq.past + r - seq.q0;
      const bool has = r >= seq.q0 && r < seq.q0 + seq.q_len && pos >= 0;
      long long at = (long long)r * p.row_pitch;
      if (has && p.page_table != nullptr) {
        const int page = pos / p.page_size, id = __ldcg(p.page_table + (size_t)s * p.max_pages + page);
        at = (unsigned)id < (unsigned)p.n_pages ? (long long)((size_t)id * p.page_pitch + (size_t)(pos - page * p.page_size) * p.row_pitch) : -1;
        if (at < 0) bad = true;  // a page that is not there is not written, and reported at the next sync
      }
      s_pos[tid] = has ? pos : -1;
      s_at[tid] = at;
    }
    __syncthreads();
    if (turns_one && my_row < rows) {
      const double t = (double)s_pos[my_row] * turns;
      sincospif(2.f * (float)(t - rint(t)), s_sin + my_row * ROPE_MAX_PAIRS + my_pair, s_cos + my_row * ROPE_MAX_PAIRS + my_pair);
    }
    __syncthreads();
#pragma unroll 1
    for (int e0 = 0; e0 < rows * n_vec; e0 += ROPE_TEAMS) {
      const int i = min(fi, rows - 1), h = fh, r = row0 + i;
      const bool is_q = h < p.n_head, is_v = h >= p.n_head + p.n_kv, has = fi < rows && s_pos[i] >= 0;
      const float* w = is_v ? nullptr : (is_q ? p.q_norm : p.k_norm);
      float4 x[JS], y[JS];
      float sq = 0.f;
#pragma unroll
      for (int j = 0; j < JS; ++j) {
        x[j] = a[j], y[j] = b[j];
        sq += x[j].x * x[j].x + x[j].y * x[j].y + x[j].z * x[j].z + x[j].w * x[j].w + y[j].x * y[j].x + y[j].y * y[j].y + y[j].z * y[j].z + y[j].w * y[j].w;
      }
      fh += ROPE_TEAMS;
      if (e0 + ROPE_TEAMS < rows * n_vec) fetch(row0, rows);
      if (p.q_norm != nullptr || p.k_norm != nullptr) sq = team_sum(sq);  // (every lane takes part)
      if (!has) continue;
      const float k = w != nullptr ? rsqrtf(sq / (float)p.hd + p.norm_eps) : 1.f;
      const long long at = s_at[i];
#pragma unroll
      for (int j = 0; j < JS; ++j) {
        const int c = tl + 16 * j;
        if (c >= chunks) continue;
        if (w != nullptr) {
          const float4 wa = *reinterpret_cast<const float4*>(w + oa[j]), wb = *reinterpret_cast<const float4*>(w + ob[j]);
          x[j].x *= k * wa.x, x[j].y *= k * wa.y, x[j].z *= k * wa.z, x[j].w *= k * wa.w;
          y[j].x *= k * wb.x, y[j].y *= k * wb.y, y[j].z *= k * wb.z, y[j].w *= k * wb.w;
        }
        if (!is_v && c < rot) {
          const float4 cs = *reinterpret_cast<const float4*>(s_cos + i * ROPE_MAX_PAIRS + 4 * c), sn = *reinterpret_cast<const float4*>(s_sin + i * ROPE_MAX_PAIRS + 4 * c);
          if (p.interleaved) {
            turn(x[j].x, x[j].y, cs.x, sn.x), turn(x[j].z, x[j].w, cs.y, sn.y);
            turn(y[j].x, y[j].y, cs.z, sn.z), turn(y[j].z, y[j].w, cs.w, sn.w);
          } else {
            turn(x[j].x, y[j].x, cs.x, sn.x), turn(x[j].y, y[j].y, cs.y, sn.y);
            turn(x[j].z, y[j].z, cs.z, sn.z), turn(x[j].w, y[j].w, cs.w, sn.w);
          }
        }
        if (is_q) {
          float* dst = p.q_out + (size_t)r * p.qo_stride + (size_t)h * p.hd;
          *reinterpret_cast<float4*>(dst + oa[j]) = x[j];
          *reinterpret_cast<float4*>(dst + ob[j]) = y[j];
        } else if (at >= 0) {
          __half* dst = (is_v ? p.v_cache + (size_t)(h - p.n_head - p.n_kv) * p.head_pitch : p.k_cache + (size_t)(h - p.n_head) * p.head_pitch) + at;
          store4_f16(dst + oa[j], x[j]);
          store4_f16(dst + ob[j], y[j]);
        }
      }
    }
    __syncthreads();  // the rows' words have been read
  }
  if (bad) p.status->bad_index = 2;
}

}  // namespace

int32_t launch_rope_kv(infr_cuda_ctx* ctx, const RopeParams& p) {
  // Eight to an SM: its threads' worth.  Of these four are there at once (64 registers; three of heads past 128, 80), the rest follow: 8192 rows in two
  // waves 59.9 us.  Fewer rows than that have a CTA each.
  const int most = ctx->sm_count * 8;
  const cudaError_t e = launch_ex(p.hd <= 128 ? k_rope_kv<1> : k_rope_kv<2>, dim3(p.rows < most ? p.rows : most), dim3(ROPE_THREADS), 0, ctx->stream, true, p);
  if (e != cudaSuccess) return check_cuda(ctx, e, "k_rope_kv launch");
  ctx->launches += 1;
  return check_cuda(ctx, cudaGetLastError(), "k_rope_kv launch");
}

}  // namespace infr
