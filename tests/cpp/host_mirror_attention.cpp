// Drives rope_kv and attention through the C++ host mirror (include/infr_cuda.hpp): packed rows, two sequences.
//
//   host_mirror_attention <in.bin> <out.bin>
// in.bin: int32 {rows, n_seq, n_head, n_kv, head_dim, cu_q[n_seq + 1]}, then q, k, v f32.   out.bin: attention's rows f32.
#include <cstdio>
#include <vector>

#include "infr_cuda.hpp"

using namespace infr_cuda;

#define OK(status_expr)                                                                  \
  do {                                                                                   \
    Status s_ = (status_expr);                                                           \
    if (!s_.ok()) {                                                                      \
      std::fprintf(stderr, "%s: %s (%d)\n", #status_expr, s_.message.c_str(), s_.code);  \
      return 1;                                                                          \
    }                                                                                    \
  } while (0)

int main(int argc, char** argv) {
  if (argc != 3) return 2;
  FILE* f = std::fopen(argv[1], "rb");
  int32_t h[5];
  if (!f || std::fread(h, 4, 5, f) != 5) return 2;
  const size_t rows = h[0], n_seq = h[1], H = h[2], K = h[3], hd = h[4];
  std::vector<int32_t> cu(n_seq + 1);
  std::vector<float> q(rows * H * hd), k(rows * K * hd), v(rows * K * hd), out(rows * H * hd);
  if (std::fread(cu.data(), 4, cu.size(), f) != cu.size() || std::fread(q.data(), 4, q.size(), f) != q.size() ||
      std::fread(k.data(), 4, k.size(), f) != k.size() || std::fread(v.data(), 4, v.size(), f) != v.size())
    return 2;
  std::fclose(f);
  auto made = Backend::create(0);
  OK(made.status);
  Backend& be = made.value;
  std::vector<Buffer> b;
  for (size_t bytes : {cu.size() * 4, q.size() * 4, k.size() * 4, v.size() * 4, q.size() * 4, k.size() * 2, v.size() * 2, q.size() * 4}) {
    auto r = be.alloc(bytes);
    OK(r.status);
    b.push_back(std::move(r.value));
  }
  OK(be.upload(b[0], cu.data(), cu.size() * 4));
  OK(be.upload(b[1], q.data(), q.size() * 4));
  OK(be.upload(b[2], k.data(), k.size() * 4));
  OK(be.upload(b[3], v.data(), v.size() * 4));
  SeqBatch batch;
  batch.cu_q = &b[0];
  batch.rows = (uint32_t)rows, batch.n_seq = (uint32_t)n_seq, batch.n_head = (uint32_t)H, batch.n_kv = (uint32_t)K, batch.head_dim = (uint32_t)hd;
  RopeKv rope;
  rope.batch = batch;
  rope.q = &b[1], rope.k = &b[2], rope.v = &b[3], rope.q_out = &b[4], rope.k_cache = &b[5], rope.v_cache = &b[6];
  rope.n_rot = (uint32_t)hd;
  OK(be.rope_kv(rope));
  Attention at;
  at.batch = batch;
  at.q = &b[4], at.k = &b[5], at.v = &b[6], at.out = &b[7], at.scale = 0.125f;
  OK(be.attention(at));
  OK(be.sync());
  OK(be.download(b[7], out.data(), out.size() * 4));
  at.scale = 1.f / 0.f;  // a caller's mistake comes back as an error
  if (be.attention(at).kind != ErrorKind::Backend) return 1;
  f = std::fopen(argv[2], "wb");
  if (!f || std::fwrite(out.data(), 4, out.size(), f) != out.size()) return 2;
  std::fclose(f);
  std::puts("OK");
  return 0;
}
