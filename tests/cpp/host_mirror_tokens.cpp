// Drives a step from tokens to tokens through the C++ host mirror (include/infr_cuda.hpp): embed, rope_kv into pages of 8 bits, attention over them, kv_read, sample.
//
//   host_mirror_tokens <in.bin> <out.bin>
// in.bin: int32 {rows, n_vocab, head_dim, page_size}, ids i32 [rows], table bf16 [n_vocab, 3 head_dim], u f32 [rows].  One sequence, one head, its q, k and v side by
// side in a row of the table.   out.bin: embedded rows f32 [rows, 3 head_dim], attention's rows f32, the cache's k and v f32, ids i32 sampled from the attention's rows.
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
  int32_t h[4];
  if (!f || std::fread(h, 4, 4, f) != 4) return 2;
  const size_t rows = h[0], V = h[1], hd = h[2], page = h[3], pages = (rows + page - 1) / page;
  std::vector<int32_t> ids(rows), cu = {0, (int32_t)rows}, len = {(int32_t)rows}, table(pages);
  for (size_t i = 0; i < pages; ++i) table[i] = (int32_t)(pages - 1 - i);
  std::vector<uint16_t> weights(V * 3 * hd);
  std::vector<float> u(rows), x(rows * 3 * hd), out(rows * hd), k(rows * hd), v(rows * hd);
  if (std::fread(ids.data(), 4, rows, f) != rows || std::fread(weights.data(), 2, weights.size(), f) != weights.size() || std::fread(u.data(), 4, rows, f) != rows) return 2;
  std::fclose(f);
  auto made = Backend::create(0);
  OK(made.status);
  Backend& be = made.value;
  enum { IDS, TABLE, U, CU, LEN, PAGES, X, Q, KC, VC, KS, VS, OUT, K, VV, KIN, VIN };
  std::vector<Buffer> b;
  const size_t cache = pages * page * hd;
  for (size_t bytes : {rows * 4, weights.size() * 2, rows * 4, (size_t)8, (size_t)4, pages * 4, x.size() * 4, rows * hd * 4, cache, cache, cache / 16, cache / 16, rows * hd * 4, rows * hd * 4, rows * hd * 4,
                       rows * hd * 4, rows * hd * 4}) {
    auto r = be.alloc(bytes);
    OK(r.status);
    b.push_back(std::move(r.value));
  }
  OK(be.upload(b[IDS], ids.data(), rows * 4));
  OK(be.upload(b[TABLE], weights.data(), weights.size() * 2));
  OK(be.upload(b[U], u.data(), rows * 4));
  OK(be.upload(b[CU], cu.data(), 8));
  OK(be.upload(b[LEN], len.data(), 4));
  OK(be.upload(b[PAGES], table.data(), pages * 4));
  Embed embed;
  embed.table = &b[TABLE], embed.ids = &b[IDS], embed.dst = &b[X], embed.dtype = DType::BF16;
  embed.rows = (uint32_t)rows, embed.ne = (uint32_t)(3 * hd), embed.n_vocab = (uint32_t)V, embed.scale = 2.f;
  OK(be.embed(embed));
  OK(be.download(b[X], x.data(), x.size() * 4));
  std::vector<float> kin(rows * hd), vin(rows * hd);
  for (size_t r = 0; r < rows; ++r)
    for (size_t i = 0; i < hd; ++i) kin[r * hd + i] = x[(3 * r + 1) * hd + i], vin[r * hd + i] = x[(3 * r + 2) * hd + i];
  OK(be.upload(b[KIN], kin.data(), kin.size() * 4));
  OK(be.upload(b[VIN], vin.data(), vin.size() * 4));
  SeqBatch batch;
  batch.cu_q = &b[CU], batch.kv_len = &b[LEN], batch.page_table = &b[PAGES];
  batch.rows = (uint32_t)rows, batch.n_seq = 1, batch.n_head = 1, batch.n_kv = 1, batch.head_dim = (uint32_t)hd;
  batch.n_pages = batch.max_pages = (uint32_t)pages, batch.page_size = (uint32_t)page;
  RopeKv rope;
  rope.batch = batch;
  rope.q = &b[X], rope.q_stride = (uint32_t)(3 * hd), rope.k = &b[KIN], rope.v = &b[VIN], rope.q_out = &b[Q];
  rope.k_cache = &b[KC], rope.v_cache = &b[VC], rope.k_scale = &b[KS], rope.v_scale = &b[VS];
  OK(be.rope_kv(rope));
  Attention at;
  at.batch = batch;
  at.q = &b[Q], at.k = &b[KC], at.v = &b[VC], at.k_scale = &b[KS], at.v_scale = &b[VS], at.out = &b[OUT], at.scale = 0.125f;
  OK(be.attention(at));
  KvRead read;
  read.batch = batch;
  read.k_cache = &b[KC], read.v_cache = &b[VC], read.k_scale = &b[KS], read.v_scale = &b[VS], read.k = &b[K], read.v = &b[VV];
  OK(be.kv_read(read));
  Sample sample;
  sample.logits = &b[OUT], sample.u = &b[U], sample.ids = &b[IDS], sample.rows = (uint32_t)rows, sample.n_vocab = (uint32_t)hd;
  OK(be.sample(sample));
  OK(be.sync());
  OK(be.download(b[OUT], out.data(), out.size() * 4));
  OK(be.download(b[K], k.data(), k.size() * 4));
  OK(be.download(b[VV], v.data(), v.size() * 4));
  OK(be.download(b[IDS], ids.data(), rows * 4));
  at.v_scale = nullptr;  // a caller's mistake comes back as an error
  if (be.attention(at).kind != ErrorKind::Backend) return 1;
  f = std::fopen(argv[2], "wb");
  if (!f) return 2;
  for (const auto* a : {&x, &out, &k, &v})
    if (std::fwrite(a->data(), 4, a->size(), f) != a->size()) return 2;
  if (std::fwrite(ids.data(), 4, rows, f) != rows) return 2;
  std::fclose(f);
  std::puts("OK");
  return 0;
}
