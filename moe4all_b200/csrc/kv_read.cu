// Keys and values out of the cache's pages: as rows of a batch for whoever asked (k_kv_read), or, of pages in 8 bits, as f16 pages for the
// attention kernel that takes these (k_kv_unpack).  Every value is read once and written once: memory bounds both.
#include "attn.cuh"
#include "kv_q8.cuh"

namespace infr {
namespace {

constexpr int READ_THREADS = 256, READ_ROWS = 8;

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const unsigned char* from) {
  static_assert(N == 1 || N == 2 || N == 4, "a load's words");
  if constexpr (N == 4) {
    const uint4 x = __ldcg(reinterpret_cast<const uint4*>(from));
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  } else if constexpr (N == 2) {
    const uint2 x = __ldcg(reinterpret_cast<const uint2*>(from));
    w[0] = x.x, w[1] = x.y;
  } else {
    w[0] = __ldcg(reinterpret_cast<const uint32_t*>(from));
  }
}

// 16 bytes of the result to each thread, neighbours side by side (two of these to a thread were half a sector to each store: 332 MB 66 us); its place in a row
// worked out once, the rows behind each other.
template <bool Q8, bool F16, int ROWS>
__global__ void __launch_bounds__(READ_THREADS) k_kv_read(const __grid_constant__ KvReadParams p) {
  __shared__ long long s_at[ROWS];  // where a row's token lies (-1: a row that is no token; -2: of no sequence)
  __shared__ int s_first;
  const int tid = threadIdx.x, lane = tid & 31;
  const int r0 = (int)((long long)blockIdx.x * p.rows / gridDim.x), r1 = (int)((long long)(blockIdx.x + 1) * p.rows / gridDim.x);
  constexpr int VALUES = F16 ? 8 : 4, WORDS = VALUES * (Q8 ? 1 : 2) / 4;  // of a thread in a row
  const int chunks = p.hd / VALUES, side = p.n_kv * chunks;
  pdl_trigger();
  pdl_wait();
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
  auto load = [&](int i) { return attn_seq(__ldcg(p.cu_q + i), __ldcg(p.cu_q + i + 1), __ldcg(p.kv_len + i), false, p.rows, p.cap, &bad); };
  if (tid < ROWS) seq = load(s);
#pragma unroll 1
  for (int row0 = r0; row0 < r1; row0 += ROWS) {
    const int rows = min(ROWS, r1 - row0);
    if (tid < ROWS && tid >= rows) s_at[tid] = -2;
    if (tid < rows) {
      const int r = row0 + tid;
#pragma unroll 1
      while (s + 1 < p.n_seq && r >= seq.q0 + seq.q_len) seq = load(++s);
      const int pos = seq.past + r - seq.q0;
      long long at = -2;
      if (r >= seq.q0 && r < seq.q0 + seq.q_len) {
        at = -1;
        if (pos >= 0) {
          const int page = pos / p.page_size;
          int id = __ldcg(p.page_table + (size_t)s * p.max_pages + page);
          if ((unsigned)id >= (unsigned)p.n_pages) bad = true, id = 0;  // read as page 0, reported at the next sync
          at = (long long)((size_t)id * p.page_pitch + (size_t)(pos - page * p.page_size) * p.row_pitch);
        }
      }
      s_at[tid] = at;
    }
    __syncthreads();
#pragma unroll 1
    for (int u = tid; u < 2 * side; u += READ_THREADS) {
      const bool is_v = u >= side;
      const int c = is_v ? u - side : u, head = c / chunks;
      const size_t in = (size_t)head * p.head_pitch + (size_t)(c - head * chunks) * VALUES;
      const void* from = is_v ? p.v : p.k;
      const uint8_t* scales = is_v ? p.vs : p.ks;
      const size_t stride = is_v ? p.vo_stride : p.ko_stride;
      void* to = is_v ? p.v_out : p.k_out;
      // all rows' words first, none behind another's use
      uint32_t w[ROWS][WORDS], scale[ROWS];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const long long at = s_at[i];
        const size_t x = (size_t)at + in;
        scale[i] = 0;
#pragma unroll
        for (int j = 0; j < WORDS; ++j) w[i][j] = Q8 ? 0x80808080u : 0;
        if (at >= 0) {
          if constexpr (Q8) scale[i] = __ldcg(scales + x / 16);
          load_words(w[i], static_cast<const unsigned char*>(from) + (Q8 ? x : 2 * x));
        }
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const long long at = s_at[i];
        if (at == -2) continue;
        uint32_t f[VALUES / 2];  // f16 pairs
        if constexpr (Q8) {
          const uint32_t d2 = q8_scale_pair(scale[i]);
#pragma unroll
          for (int j = 0; j < WORDS; ++j) f[2 * j] = q8_lo(w[i][j], d2), f[2 * j + 1] = q8_hi(w[i][j], d2);
        } else {
#pragma unroll
          for (int j = 0; j < WORDS; ++j) f[j] = w[i][j];
        }
        const size_t y = (size_t)(row0 + i) * stride + (size_t)c * VALUES;
        if constexpr (F16) {
          *reinterpret_cast<uint4*>(static_cast<__half*>(to) + y) = make_uint4(f[0], f[1], f[2], f[3]);
        } else {
          const float2 a = __half22float2(*reinterpret_cast<const __half2*>(f)), b = __half22float2(*reinterpret_cast<const __half2*>(f + 1));
          *reinterpret_cast<float4*>(static_cast<float*>(to) + y) = make_float4(a.x, a.y, b.x, b.y);
        }
      }
    }
    __syncthreads();
  }
  if (bad) p.status->bad_index = 2;
}

// The pages that some row of the call sees: a warp to 128 blocks of 16 values, which are a part of a kv head of a page (a CTA to all of such a head were ten in a row for
// pages of 16 tokens, each with its own wait for the page's number).
constexpr int UNPACK_PIECE = 128;
__global__ void __launch_bounds__(READ_THREADS) k_kv_unpack(const __grid_constant__ AttnParams p, __half* __restrict__ k_out, __half* __restrict__ v, int* __restrict__ table) {
  extern __shared__ int s_pre[];  // pages ahead of each sequence, then the first page of each
  __shared__ long long s_scan[READ_THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31;
  int* s_page0 = s_pre + p.n_seq + 1;
  pdl_trigger();
  pdl_wait();
  if (tid == 0) s_pre[0] = 0;
  long long carry = 0;
#pragma unroll 1
  for (int s0 = 0; s0 < p.n_seq; s0 += READ_THREADS) {
    const int s = s0 + tid;
    int n = 0;
    if (s < p.n_seq) {
      const AttnSeq seq = attn_load_seq(p, s);
      const int hi = seq.past + seq.q_len, lo = attn_first_key(seq.past, p.window);
      const int first = lo / p.page_size;
      s_page0[s] = first;
      n = seq.q_len > 0 && hi > lo ? (hi - 1) / p.page_size + 1 - first : 0;
    }
    const long long sum = carry + block_scan<READ_THREADS>(n, s_scan);
    if (s < p.n_seq) s_pre[s + 1] = (int)min(sum, 0x7FFFFFFFll);  // (4096 sequences of 2^31 / 16 pages and more: not in 180 GB)
    __syncthreads();
    carry = s_pre[min(s0 + READ_THREADS, p.n_seq)];
  }
  const int blocks = p.hd / 16, per = p.page_size * blocks, pieces = (2 * per + UNPACK_PIECE - 1) / UNPACK_PIECE;  // 16 values to each of a unit's places
  const long long units = carry * p.n_kv * pieces, warps = (long long)gridDim.x * (READ_THREADS / 32), w = (long long)blockIdx.x * (READ_THREADS / 32) + (tid >> 5);
  const long long u0 = units * w / warps, u1 = units * (w + 1) / warps;
#pragma unroll 1
  for (long long u = u0; u < u1; ++u) {
    const long long side = u / pieces;
    const int piece = (int)(u - side * pieces), page = (int)(side / p.n_kv), head = (int)(side - (long long)page * p.n_kv);
    int s = 0;
#pragma unroll 1
    for (int hi = p.n_seq; hi - s > 1;) {  // the last sequence whose pages begin at or before this one
      const int mid = (s + hi) / 2;
      if (s_pre[mid] <= page) s = mid;
      else hi = mid;
    }
    while (s_pre[s + 1] <= page) ++s;  // (past sequences without pages)
    const int j = s_page0[s] + page - s_pre[s], id = attn_page(p, s, j);
    const int to_page = table != nullptr ? s * p.max_pages + j : id;
    if (table != nullptr && head == 0 && piece == 0 && lane == 0) table[(size_t)s * p.max_pages + j] = to_page;
    const size_t from = (size_t)id * p.page_pitch + (size_t)head * p.head_pitch, to = (size_t)to_page * p.page_pitch + (size_t)head * p.head_pitch;
    uint4 c[UNPACK_PIECE / 32];
    uint32_t d2[UNPACK_PIECE / 32];
#pragma unroll
    for (int k = 0; k < UNPACK_PIECE / 32; ++k) {
      const int e = piece * UNPACK_PIECE + 32 * k + lane;
      const size_t at = from + (size_t)(e >= per ? e - per : e) * 16;
      if (e < 2 * per) {
        c[k] = __ldcg(reinterpret_cast<const uint4*>((e >= per ? p.vq : p.kq) + at));
        d2[k] = q8_scale_pair(__ldcg((e >= per ? p.vs : p.ks) + at / 16));
      }
    }
#pragma unroll
    for (int k = 0; k < UNPACK_PIECE / 32; ++k) {
      const int e = piece * UNPACK_PIECE + 32 * k + lane;
      if (e >= 2 * per) continue;
      uint4* dst = reinterpret_cast<uint4*>((e >= per ? v : k_out) + to + (size_t)(e >= per ? e - per : e) * 16);
      dst[0] = make_uint4(q8_lo(c[k].x, d2[k]), q8_hi(c[k].x, d2[k]), q8_lo(c[k].y, d2[k]), q8_hi(c[k].y, d2[k]));
      dst[1] = make_uint4(q8_lo(c[k].z, d2[k]), q8_hi(c[k].z, d2[k]), q8_lo(c[k].w, d2[k]), q8_hi(c[k].w, d2[k]));
    }
  }
}

}  // namespace

template <bool Q8, bool F16>
static cudaError_t launch_read(infr_cuda_ctx* ctx, const KvReadParams& p) {
  // A row to each CTA while all of them are there at once, then eight: 777 rows of 8 x 128 values as f16 3.0 us for 4.3 with eight rows' instructions in the way, 32000
  // rows of 8 x 128 as f32 58.9 us for 64.9 with 27 rows in a loop, 65.0 with four.
  if (p.rows <= ctx->sm_count * 8) return launch_ex(k_kv_read<Q8, F16, 1>, dim3(p.rows), dim3(READ_THREADS), 0, ctx->stream, true, p);
  return launch_ex(k_kv_read<Q8, F16, READ_ROWS>, dim3((p.rows + READ_ROWS - 1) / READ_ROWS), dim3(READ_THREADS), 0, ctx->stream, true, p);
}

int32_t launch_kv_read(infr_cuda_ctx* ctx, const KvReadParams& p) {
  const cudaError_t e = p.ks != nullptr ? (p.f16 ? launch_read<true, true>(ctx, p) : launch_read<true, false>(ctx, p)) : (p.f16 ? launch_read<false, true>(ctx, p) : launch_read<false, false>(ctx, p));
  if (e != cudaSuccess) return check_cuda(ctx, e, "k_kv_read launch");
  ctx->launches += 1;
  return check_cuda(ctx, cudaGetLastError(), "k_kv_read launch");
}

int32_t launch_kv_unpack(infr_cuda_ctx* ctx, const AttnParams& p, __half* k, __half* v, int* table) {
  const size_t smem = (2 * (size_t)p.n_seq + 1) * 4;
  cudaError_t e = ensure_smem(reinterpret_cast<const void*>(&k_kv_unpack), smem);
  if (e == cudaSuccess) e = launch_ex(k_kv_unpack, dim3(ctx->sm_count * 8), dim3(READ_THREADS), smem, ctx->stream, true, p, k, v, table);
  if (e != cudaSuccess) return check_cuda(ctx, e, "k_kv_unpack launch");
  ctx->launches += 1;
  return check_cuda(ctx, cudaGetLastError(), "k_kv_unpack launch");
}

}  // namespace infr
