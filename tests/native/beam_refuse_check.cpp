// The refusals of prefix attention, the rotation and the beam search (pz_refuse.h): one
// good call of each, then that call with one thing wrong.
#include <cstdio>

#include "pz_refuse.h"

static int bad = 0;
static void expect(const char* what, PzRefusal got, int code) {
  const bool ok = got.code == code && (code == PZ_OK) == (got.why == nullptr);
  if (!ok) bad++;
  std::printf("%s %s: %d %s\n", ok ? "ok " : "BAD", what, got.code, got.why ? got.why : "");
}

int main() {
  alignas(16) static float f[64];
  alignas(16) static uint16_t h[64];
  static int32_t i32[8], other[8];

  // a cache of 2 key heads of 64; 6 sequences of 2 prefixes
  pz_kv_cache cache = {PZ_BF16, 2, 64, h, h, 128, 10, 16, i32, 4, i32};
  struct Call {
    pz_kv_prefix p;
    int B, T, heads;
    const void* q;
  };
  auto prefix = [&](const char* what, int code, auto change) {
    pz_kv_cache c = cache;
    Call a = {{i32, 4, i32, 2, nullptr}, 6, 3, 4, h};
    change(c, a);
    expect(what,
           pz_refuse_prefix(&c, &a.p, h, h, 1024, a.B, a.T, a.heads, 0.125f, a.q, 1L << 23, h,
                            1L << 23),
           code);
  };
#define P [&](pz_kv_cache & c, Call & a)
#define N (void)c, (void)a
  prefix("prefix: good", PZ_OK, P { N; });
  prefix("prefix: ranges", PZ_OK, P { N; a.p.d_first = i32; a.B = 7; });
  prefix("prefix: more prefixes than sequences", PZ_OK, P { N; a.p.d_first = i32; a.p.n_prefixes = 100; });
  prefix("prefix: no sequences", PZ_OK, P { N; a.B = 0; });
  prefix("prefix: seven sequences of two", PZ_EINVAL, P { N; a.B = 7; });
  prefix("prefix: null tables", PZ_EINVAL, P { N; a.p.d_blocks = nullptr; });
  prefix("prefix: null lengths", PZ_EINVAL, P { N; a.p.d_len = nullptr; });
  prefix("prefix: empty tables", PZ_EINVAL, P { N; a.p.max_blocks = 0; });
  prefix("prefix: none", PZ_EINVAL, P { N; a.p.n_prefixes = 0; });
  prefix("prefix: too many", PZ_ERANGE, P { N; a.p.d_first = i32; a.p.n_prefixes = 4097; });
  prefix("prefix: as many without ranges", PZ_OK, P { N; a.B = 5000; a.p.n_prefixes = 5000; });
  prefix("prefix: positions past 32 bits", PZ_ERANGE, P { N; a.p.max_blocks = 1 << 27; });
  prefix("prefix: the most rows", PZ_OK, P { N; a.T = 64; a.heads = 512; });
  prefix("prefix: more rows", PZ_ERANGE, P { N; a.T = 64; a.heads = 514; });
  // (two parts of a sequence are in the workspace, whatever its heads)
  prefix("prefix: the most rows of 256", PZ_OK, P { N; c.head_dim = 256; c.ld = 512; a.T = 64; a.heads = 508; });
  prefix("prefix: more rows of 256", PZ_ERANGE, P { N; c.head_dim = 256; c.ld = 512; a.T = 64; a.heads = 510; });
  prefix("prefix: what the tree refuses", PZ_EINVAL, P { N; c.block_size = 4; });
  prefix("prefix: null q", PZ_EINVAL, P { N; a.q = nullptr; });
  expect("prefix: null prefix",
         pz_refuse_prefix(&cache, nullptr, h, h, 128, 6, 3, 4, 0.125f, h, 256, h, 256), PZ_EINVAL);

  // rotation of 2 + 1 heads of 64
  struct Rows {
    const void *q, *k, *qo, *ko;
    long lq, lk, lqo, lko;
    int n;
    const int32_t* pos;
  };
  auto rope = [&](const char* what, int code, auto change) {
    pz_qk_rope r = {PZ_BF16, 2, 1, 64, f, f, 1e-6f, 64, PZ_ROPE_HALVES, f, 1.0f};
    Rows a = {h, h, h, h, 192, 192, 192, 192, 5, i32};
    change(r, a);
    expect(what, pz_refuse_rope(&r, a.q, a.lq, a.k, a.lk, a.qo, a.lqo, a.ko, a.lko, a.n, a.pos),
           code);
  };
#define R [&](pz_qk_rope & r, Rows & a)
#define M (void)r, (void)a
  rope("rope: good", PZ_OK, R { M; });
  rope("rope: no tokens", PZ_OK, R { M; a.n = 0; });
  rope("rope: no norms, any eps", PZ_OK, R { M; r.d_q_norm = r.d_k_norm = nullptr; r.eps = -1.0f; });
  rope("rope: no rotation", PZ_OK, R { M; r.rot_dim = 0; r.d_freq = nullptr; a.pos = nullptr; });
  rope("rope: queries alone", PZ_OK, R { M; r.n_kv_heads = 0; a.k = a.ko = nullptr; });
  rope("rope: keys alone", PZ_OK, R { M; r.n_heads = 0; a.q = a.qo = nullptr; });
  rope("rope: neither", PZ_EINVAL, R { M; r.n_heads = r.n_kv_heads = 0; });
  rope("rope: negative heads", PZ_EINVAL, R { M; r.n_heads = -1; });
  rope("rope: negative tokens", PZ_EINVAL, R { M; a.n = -1; });
  rope("rope: type", PZ_EINVAL, R { M; r.type = 3; });
  rope("rope: no elements", PZ_EINVAL, R { M; r.head_dim = 0; });
  rope("rope: heads of 1024", PZ_OK, R { M; r.head_dim = 1024; a.lq = a.lk = a.lqo = a.lko = 4096; });
  rope("rope: heads of 1025", PZ_ENOTSUP, R { M; r.head_dim = 1025; });
  rope("rope: more heads", PZ_ERANGE, R { M; r.n_heads = (1 << 16) + 1; });
  rope("rope: odd rotation", PZ_EINVAL, R { M; r.rot_dim = 63; });
  rope("rope: a longer rotation", PZ_EINVAL, R { M; r.rot_dim = 66; });
  rope("rope: layout", PZ_EINVAL, R { M; r.layout = 2; });
  rope("rope: no frequencies", PZ_EINVAL, R { M; r.d_freq = nullptr; });
  rope("rope: no positions", PZ_EINVAL, R { M; a.pos = nullptr; });
  rope("rope: negative eps", PZ_EINVAL, R { M; r.eps = -1e-6f; });
  rope("rope: eps NaN", PZ_EINVAL, R { M; r.eps = __builtin_nanf(""); });
  rope("rope: null q", PZ_EINVAL, R { M; a.q = nullptr; });
  rope("rope: null k out", PZ_EINVAL, R { M; a.ko = nullptr; });
  rope("rope: short rows", PZ_EINVAL, R { M; a.lq = 127; });
  rope("rope: short rows out", PZ_EINVAL, R { M; a.lko = 63; });
  rope("rope: in place at another stride", PZ_EINVAL, R { M; a.lqo = 200; });
  rope("rope: elsewhere at another stride", PZ_OK, R { M; a.qo = h + 8; a.lqo = 200; });
  rope("rope: off 2 bytes", PZ_EINVAL, R { M; a.q = reinterpret_cast<const char*>(h) + 1; });
  rope("rope: fp32 off 4 bytes", PZ_EINVAL, R { M; r.type = PZ_F32; a.k = h + 1; });
  rope("rope: weights off 4 bytes", PZ_EINVAL, R { M; r.d_q_norm = reinterpret_cast<const float*>(h + 1); });
  rope("rope: more than a launch", PZ_ERANGE, R { M; a.n = 1 << 25; });
  expect("rope: null", pz_refuse_rope(nullptr, h, 192, h, 192, h, 192, h, 192, 5, i32), PZ_EINVAL);

  // selection of 2 groups of 4 beams
  struct Sel {
    const float* x;
    long ld;
    int G, W, V, K;
    const float* score;
    const int32_t *parent, *ids;
    const float* out;
  };
  auto select = [&](const char* what, int code, auto change) {
    Sel a = {f, 100, 2, 4, 100, 8, f, i32, i32, f};
    change(a);
    expect(what, pz_refuse_select(a.x, a.ld, a.G, a.W, a.V, a.score, a.K, a.parent, a.ids, a.out),
           code);
  };
  select("select: good", PZ_OK, [](Sel&) {});
  select("select: no groups", PZ_OK, [](Sel& a) { a.G = 0; });
  select("select: the widest", PZ_OK, [](Sel& a) { a.W = 64; a.K = 128; });
  select("select: wider", PZ_ERANGE, [](Sel& a) { a.W = 65; });
  select("select: more than are kept", PZ_ERANGE, [](Sel& a) { a.K = 129; });
  select("select: no beams", PZ_EINVAL, [](Sel& a) { a.W = 0; });
  select("select: none", PZ_EINVAL, [](Sel& a) { a.K = 0; });
  select("select: negative groups", PZ_EINVAL, [](Sel& a) { a.G = -1; });
  select("select: too many groups", PZ_ERANGE, [](Sel& a) { a.G = (1 << 20) + 1; });
  select("select: no vocabulary", PZ_EINVAL, [](Sel& a) { a.V = 0; });
  select("select: short rows", PZ_EINVAL, [](Sel& a) { a.ld = 99; });
  select("select: the largest vocabulary", PZ_OK, [](Sel& a) { a.ld = a.V = 1 << 22; });
  select("select: a larger one", PZ_ERANGE, [](Sel& a) { a.ld = a.V = (1 << 22) + 1; });
  select("select: null logits", PZ_EINVAL, [](Sel& a) { a.x = nullptr; });
  select("select: null scores", PZ_EINVAL, [](Sel& a) { a.score = nullptr; });
  select("select: null parents", PZ_EINVAL, [](Sel& a) { a.parent = nullptr; });
  select("select: null ids", PZ_EINVAL, [](Sel& a) { a.ids = nullptr; });
  select("select: null scores out", PZ_EINVAL, [](Sel& a) { a.out = nullptr; });

  // reordering of 2 groups of 4 beams in 3 layers
  struct Reo {
    pz_kv_cache c[3];
    int layers, G, W, n_pool, ahead;
    const int32_t *parent, *pool, *blocks, *len;
  };
  auto reorder = [&](const char* what, int code, auto change) {
    Reo a = {{cache, cache, cache}, 3, 2, 4, 8, 1, i32, i32, other, other};
    change(a);
    expect(what, pz_refuse_reorder(a.layers ? a.c : nullptr, a.layers, a.G, a.W, a.parent, a.pool,
                                   a.n_pool, a.ahead, a.blocks, a.len),
           code);
  };
  reorder("reorder: good", PZ_OK, [](Reo&) {});
  reorder("reorder: other buffers", PZ_OK, [](Reo& a) { a.c[1].d_k = f; a.c[2].d_v = f; });
  reorder("reorder: no groups", PZ_OK, [](Reo& a) { a.G = 0; });
  reorder("reorder: no pool", PZ_OK, [](Reo& a) { a.n_pool = 0; a.pool = nullptr; });
  reorder("reorder: nothing ahead", PZ_OK, [](Reo& a) { a.ahead = 0; });
  reorder("reorder: no layers", PZ_EINVAL, [](Reo& a) { a.layers = 0; });
  reorder("reorder: negative groups", PZ_EINVAL, [](Reo& a) { a.G = -1; });
  reorder("reorder: no beams", PZ_EINVAL, [](Reo& a) { a.W = 0; });
  reorder("reorder: wider", PZ_ERANGE, [](Reo& a) { a.W = 65; });
  reorder("reorder: null parents", PZ_EINVAL, [](Reo& a) { a.parent = nullptr; });
  reorder("reorder: null pool", PZ_EINVAL, [](Reo& a) { a.pool = nullptr; });
  reorder("reorder: a larger pool", PZ_ERANGE, [](Reo& a) { a.n_pool = PZ_BEAM_MAX_POOL + 1; });
  reorder("reorder: negative pool", PZ_EINVAL, [](Reo& a) { a.n_pool = -1; });
  reorder("reorder: negative ahead", PZ_EINVAL, [](Reo& a) { a.ahead = -1; });
  reorder("reorder: too many beams", PZ_ERANGE, [](Reo& a) { a.G = 1 << 18; a.W = 5; });
  reorder("reorder: tables past 2^30", PZ_ERANGE, [](Reo& a) { a.W = 64; for (auto& c : a.c) { c.max_blocks = (1 << 24) + 1; c.block_size = 8; } });
  reorder("reorder: null tables out", PZ_EINVAL, [](Reo& a) { a.blocks = nullptr; });
  reorder("reorder: null lengths out", PZ_EINVAL, [](Reo& a) { a.len = nullptr; });
  reorder("reorder: tables in place", PZ_EINVAL, [](Reo& a) { a.blocks = a.c[0].d_blocks; });
  reorder("reorder: lengths in place", PZ_EINVAL, [](Reo& a) { a.len = a.c[0].d_len; });
  reorder("reorder: layers of another shape", PZ_EINVAL, [](Reo& a) { a.c[2].n_kv_heads = 1; });
  reorder("reorder: layers of other tables", PZ_EINVAL, [](Reo& a) { a.c[1].d_blocks = other; });
  reorder("reorder: a bad layer", PZ_EINVAL, [](Reo& a) { a.c[2].d_v = nullptr; });
  reorder("reorder: a layer of another type", PZ_EINVAL, [](Reo& a) { a.c[1].type = PZ_F16; });
  return bad != 0;
}
