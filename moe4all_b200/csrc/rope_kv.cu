// What stands between a layer's q / k / v rows and its attention: per-head RMS norm and rotary embedding of q and k, k and v rounded to
// f16 into the cache.  Every value is read once and written once: memory bounds it.
//
// Sixteen lanes own a head; a lane takes eight values at a time as two 16-byte words that hold four whole pairs (halves style: the words
// are half the rotated range apart; interleaved: neighbours), so that a pair never leaves its lane.  The angles are products of a position
// and a frequency in 64 bits, reduced to a fraction of a turn before they are rounded to 32 (a position of 10^6 times a frequency near 1
// keeps 4 bits of f32 after the point); a row's sines are worked out once for all of its heads.
#include "attn.cuh"

namespace infr {
namespace {

constexpr int ROPE_THREADS = 256, ROPE_TEAMS = ROPE_THREADS / 16, ROPE_MAX_PAIRS = 128;

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

__global__ void __launch_bounds__(ROPE_THREADS) k_rope_kv(const RopeParams p) {
  __shared__ __align__(16) float s_cos[2][ROPE_MAX_PAIRS], s_sin[2][ROPE_MAX_PAIRS];
  const int tid = threadIdx.x, team = tid >> 4, tl = tid & 15;
  pdl_wait();
  const int r0 = (int)((long long)blockIdx.x * p.rows / gridDim.x), r1 = (int)((long long)(blockIdx.x + 1) * p.rows / gridDim.x);
  // the last sequence that begins at or before the first row (rows ahead of cu_q[0] belong to none)
  int s = 0;
  for (int hi = p.n_seq; hi - s > 1;) {
    const int mid = (s + hi) / 2;
    if (__ldcg(p.cu_q + mid) <= r0) s = mid;
    else hi = mid;
  }
  bool bad = false;
  auto load = [&](int i) {
    return attn_seq(__ldcg(p.cu_q + i), __ldcg(p.cu_q + i + 1), p.kv_len != nullptr ? __ldcg(p.kv_len + i) : 0, p.kv_len == nullptr, p.rows, p.cap, &bad);
  };
  AttnSeq seq = load(s);
  const int pairs = p.n_rot / 2;
  double turns = 0.0;  // of this thread's pair, per token
  if (tid < pairs) {
    turns = p.turns0 * pow(p.ratio, (double)tid);
    if (p.freq_factors != nullptr) turns /= (double)p.freq_factors[tid];
  }
  const int n_vec = p.n_head + 2 * p.n_kv, chunks = p.hd / 8, rot = p.n_rot / 8;
  int buf = 0;
  for (int r = r0; r < r1; ++r) {
    while (s + 1 < p.n_seq && r >= seq.q0 + seq.q_len) seq = load(++s);
    const int pos = seq.past + r - seq.q0;
    if (r < seq.q0 || r >= seq.q0 + seq.q_len || pos < 0) continue;  // (the same for the whole CTA)
    float *co = s_cos[buf], *si = s_sin[buf];  // (two: the other's readers are past the next barrier)
    buf ^= 1;
    if (tid < pairs) {
      const double a = (double)pos * turns;
      sincospif(2.f * (float)(a - rint(a)), si + tid, co + tid);
    }
    size_t at = (size_t)r * p.row_pitch;
    bool writes = true;
    if (p.page_table != nullptr) {
      const int page = pos / p.page_size, id = __ldcg(p.page_table + (size_t)s * p.max_pages + page);
      writes = (unsigned)id < (unsigned)p.n_pages;  // a page that is not there is not written, and reported at the next sync
      if (!writes) bad = true;
      at = (size_t)id * p.page_pitch + (size_t)(pos - page * p.page_size) * p.row_pitch;
    }
    __syncthreads();
    for (int h0 = 0; h0 < n_vec; h0 += ROPE_TEAMS) {
      const int h = h0 + team;
      const bool has = h < n_vec, is_q = h < p.n_head, is_v = h >= p.n_head + p.n_kv;
      const int kvh = is_q ? 0 : (is_v ? h - p.n_head - p.n_kv : h - p.n_head);
      const float* src = is_q ? p.q + (size_t)r * p.q_stride + (size_t)h * p.hd
                              : (is_v ? p.v + (size_t)r * p.v_stride : p.k + (size_t)r * p.k_stride) + (size_t)kvh * p.hd;
      const float* w = is_v ? nullptr : (is_q ? p.q_norm : p.k_norm);
      float4 a[2], b[2];
      int oa[2], ob[2];
      float sq = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int c = tl + 16 * j;
        oa[j] = 8 * c, ob[j] = 8 * c + 4;
        if (!p.interleaved && c < rot) oa[j] = 4 * c, ob[j] = p.n_rot / 2 + 4 * c;
        a[j] = b[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (has && c < chunks) {
          a[j] = __ldcg(reinterpret_cast<const float4*>(src + oa[j]));
          b[j] = __ldcg(reinterpret_cast<const float4*>(src + ob[j]));
        }
        if (w != nullptr)
          sq += a[j].x * a[j].x + a[j].y * a[j].y + a[j].z * a[j].z + a[j].w * a[j].w + b[j].x * b[j].x + b[j].y * b[j].y + b[j].z * b[j].z + b[j].w * b[j].w;
      }
      // (every lane takes part: the warp's other team may have a norm to sum)
      const float total = team_sum(sq);
      if (!has) continue;
      const float k = w != nullptr ? rsqrtf(total / (float)p.hd + p.norm_eps) : 1.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int c = tl + 16 * j;
        if (c >= chunks) continue;
        if (w != nullptr) {
          const float4 wa = *reinterpret_cast<const float4*>(w + oa[j]), wb = *reinterpret_cast<const float4*>(w + ob[j]);
          a[j].x *= k * wa.x, a[j].y *= k * wa.y, a[j].z *= k * wa.z, a[j].w *= k * wa.w;
          b[j].x *= k * wb.x, b[j].y *= k * wb.y, b[j].z *= k * wb.z, b[j].w *= k * wb.w;
        }
        if (!is_v && c < rot) {
          const float4 cs = *reinterpret_cast<const float4*>(co + 4 * c), sn = *reinterpret_cast<const float4*>(si + 4 * c);
          if (p.interleaved) {
            turn(a[j].x, a[j].y, cs.x, sn.x), turn(a[j].z, a[j].w, cs.y, sn.y);
            turn(b[j].x, b[j].y, cs.z, sn.z), turn(b[j].z, b[j].w, cs.w, sn.w);
          } else {
            turn(a[j].x, b[j].x, cs.x, sn.x), turn(a[j].y, b[j].y, cs.y, sn.y);
            turn(a[j].z, b[j].z, cs.z, sn.z), turn(a[j].w, b[j].w, cs.w, sn.w);
          }
        }
        if (is_q) {
          float* dst = p.q_out + (size_t)r * p.qo_stride + (size_t)h * p.hd;
          *reinterpret_cast<float4*>(dst + oa[j]) = a[j];
          *reinterpret_cast<float4*>(dst + ob[j]) = b[j];
        } else if (writes) {
          __half* dst = (is_v ? p.v_cache : p.k_cache) + at + (size_t)kvh * p.head_pitch;
          store4_f16(dst + oa[j], a[j]);
          store4_f16(dst + ob[j], b[j]);
        }
      }
    }
  }
  if (bad) p.status->bad_index = 2;
}

}  // namespace

int32_t launch_rope_kv(infr_cuda_ctx* ctx, const RopeParams& p) {
  const int most = ctx->sm_count * 8;
  const cudaError_t e = launch_ex(k_rope_kv, dim3(p.rows < most ? p.rows : most), dim3(ROPE_THREADS), 0, ctx->stream, true, p);
  if (e != cudaSuccess) return check_cuda(ctx, e, "k_rope_kv launch");
  ctx->launches += 1;
  return check_cuda(ctx, cudaGetLastError(), "k_rope_kv launch");
}

}  // namespace infr
