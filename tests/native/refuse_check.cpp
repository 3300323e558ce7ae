// The refusals of the logit rules, the 8-bit LM head and the tree attention
// (pz_refuse.h): one good call of each, then that call with one thing wrong.
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
  alignas(16) static int8_t i8[64];
  alignas(16) static uint16_t h[64];
  static int32_t i32[8];
  static uint32_t u32[8];

  // rules: 2 rows of 100 logits
  pz_logit_rules good = {};
  good.rep_penalty = 1.0f;
  auto rules = [&](const char* what, int code, auto change) {
    pz_logit_rules r = good;
    const float *in = f, *out = f;
    long ld_in = 100, ld_out = 100;
    int B = 2, V = 100;
    change(r, in, out, ld_in, ld_out, B, V);
    expect(what, pz_refuse_rules(in, ld_in, out, ld_out, B, V, &r), code);
  };
#define R [&](pz_logit_rules & r, const float*& in, const float*& out, long& ld_in, long& ld_out, int& B, int& V)
#define U (void)r, (void)in, (void)out, (void)ld_in, (void)ld_out, (void)B, (void)V
  rules("rules: none", PZ_OK, R { U; });
  rules("rules: no rows", PZ_OK, R { U; B = 0; });
  rules("rules: null in", PZ_EINVAL, R { U; in = nullptr; });
  rules("rules: null out", PZ_EINVAL, R { U; out = nullptr; });
  rules("rules: negative B", PZ_EINVAL, R { U; B = -1; });
  rules("rules: no vocabulary", PZ_EINVAL, R { U; V = 0; });
  rules("rules: short input rows", PZ_EINVAL, R { U; ld_in = 99; });
  rules("rules: short output rows", PZ_EINVAL, R { U; ld_out = 99; });
  rules("rules: in place at another stride", PZ_EINVAL, R { U; ld_out = 101; });
  rules("rules: another buffer at another stride", PZ_OK, R { U; out = f + 1; ld_out = 101; });
  rules("rules: negative H", PZ_EINVAL, R { U; r.H = -1; });
  rules("rules: H without a history", PZ_EINVAL, R { U; r.H = 1; });
  rules("rules: H with one", PZ_OK, R { U; r.H = 1; r.d_hist = i32; });
  rules("rules: negative n_bias", PZ_EINVAL, R { U; r.n_bias = -1; });
  rules("rules: biases without ids", PZ_EINVAL, R { U; r.n_bias = 1; r.d_bias = f; });
  rules("rules: ids without biases", PZ_EINVAL, R { U; r.n_bias = 1; r.d_bias_ids = i32; });
  rules("rules: negative n_masks", PZ_EINVAL, R { U; r.n_masks = -1; });
  rules("rules: masks without words", PZ_EINVAL, R { U; r.n_masks = 2; r.ld_mask = 4; });
  rules("rules: short masks", PZ_EINVAL, R { U; r.n_masks = 2; r.d_mask = u32; r.ld_mask = 3; });
  rules("rules: a mask a row", PZ_OK, R { U; r.n_masks = 2; r.d_mask = u32; r.ld_mask = 4; });
  rules("rules: fewer masks than rows", PZ_EINVAL, R { U; r.n_masks = 1; r.d_mask = u32; r.ld_mask = 4; });
  rules("rules: fewer masks with their rows", PZ_OK, R { U; r.n_masks = 1; r.d_mask = u32; r.ld_mask = 4; r.d_mask_row = i32; });
  rules("rules: V past 2^30", PZ_ERANGE, R { U; V = (1 << 30) + 1; ld_in = ld_out = V; });
  rules("rules: H past 2^30", PZ_ERANGE, R { U; r.d_hist = i32; r.H = (1 << 30) + 1; });
  expect("rules: null rules", pz_refuse_rules(f, 100, f, 100, 2, 100, nullptr), PZ_EINVAL);

  // quantisation
  expect("quant: good", pz_refuse_quant(f, PZ_F32, 8, 2, 8, i8, 8, f), PZ_OK);
  expect("quant: no rows", pz_refuse_quant(f, PZ_F32, 8, 0, 8, i8, 8, f), PZ_OK);
  expect("quant: null x", pz_refuse_quant(nullptr, PZ_F32, 8, 2, 8, i8, 8, f), PZ_EINVAL);
  expect("quant: null q", pz_refuse_quant(f, PZ_F32, 8, 2, 8, nullptr, 8, f), PZ_EINVAL);
  expect("quant: more rows than a launch", pz_refuse_quant(f, PZ_F32, 8, 1 << 24, 8, i8, 8, f),
         PZ_ERANGE);
  expect("quant: null scale", pz_refuse_quant(f, PZ_F32, 8, 2, 8, i8, 8, nullptr), PZ_EINVAL);
  expect("quant: negative rows", pz_refuse_quant(f, PZ_F32, 8, -2, 8, i8, 8, f), PZ_EINVAL);
  expect("quant: empty rows", pz_refuse_quant(f, PZ_F32, 8, 2, 0, i8, 8, f), PZ_EINVAL);
  expect("quant: short rows", pz_refuse_quant(f, PZ_F32, 7, 2, 8, i8, 8, f), PZ_EINVAL);
  expect("quant: short q rows", pz_refuse_quant(f, PZ_F32, 8, 2, 8, i8, 7, f), PZ_EINVAL);
  expect("quant: type", pz_refuse_quant(f, 3, 8, 2, 8, i8, 8, f), PZ_EINVAL);
  expect("quant: fp32 off 4 bytes", pz_refuse_quant(h + 1, PZ_F32, 8, 2, 8, i8, 8, f), PZ_EINVAL);
  expect("quant: bf16 on 2 bytes", pz_refuse_quant(h + 1, PZ_BF16, 8, 2, 8, i8, 8, f), PZ_OK);

  // product
  auto i8c = [&](const char* what, int code, const int8_t* w, const float* sw, int V, int n,
                 const int8_t* x, const float* sx, int B, long ldx) {
    expect(what, pz_refuse_i8(w, sw, V, n, x, sx, B, ldx, 4), code);
  };
  i8c("i8: good", PZ_OK, i8, f, 8, 16, i8, f, 4, 16);
  i8c("i8: any alignment", PZ_OK, i8 + 1, f, 8, 3, i8 + 1, f, 4, 5);
  i8c("i8: null w", PZ_EINVAL, nullptr, f, 8, 16, i8, f, 4, 16);
  i8c("i8: null sw", PZ_EINVAL, i8, nullptr, 8, 16, i8, f, 4, 16);
  i8c("i8: null x", PZ_EINVAL, i8, f, 8, 16, nullptr, f, 4, 16);
  i8c("i8: null sx", PZ_EINVAL, i8, f, 8, 16, i8, nullptr, 4, 16);
  i8c("i8: V", PZ_EINVAL, i8, f, 0, 16, i8, f, 4, 16);
  i8c("i8: n", PZ_EINVAL, i8, f, 8, 0, i8, f, 4, 16);
  i8c("i8: B", PZ_EINVAL, i8, f, 8, 16, i8, f, -1, 16);
  i8c("i8: short rows", PZ_EINVAL, i8, f, 8, 16, i8, f, 4, 15);
  i8c("i8: the longest rows", PZ_OK, i8, f, 8, PZ_I8_MAX_N, i8, f, 4, PZ_I8_MAX_N);
  i8c("i8: longer ones", PZ_ERANGE, i8, f, 8, PZ_I8_MAX_N + 1, i8, f, 4, PZ_I8_MAX_N + 1);
  i8c("i8: more rows than the sampler's", PZ_ERANGE, i8, f, 8, 16, i8, f, 5, 16);

  // cache and tree: 2 sequences of 3 nodes, 4 heads over 2 key heads of 64
  pz_kv_cache c0 = {};
  c0.type = PZ_BF16;
  c0.n_kv_heads = 2;
  c0.head_dim = 64;
  c0.d_k = h;
  c0.d_v = h;
  c0.ld = 128;
  c0.n_blocks = 5;
  c0.block_size = 16;
  c0.d_blocks = i32;
  c0.max_blocks = 4;
  c0.d_len = i32;
  struct Call {
    const void *kn, *vn;
    long ld_n;
    int B, T, heads;
    float scale;
    const void* q;
    long ld_q;
    const void* out;
    long ld_out;
  };
  auto tree = [&](const char* what, int code, auto change) {
    pz_kv_cache c = c0;
    Call a = {h, h, 128, 2, 3, 4, 0.125f, h, 256, h, 256};
    change(c, a);
    expect(what,
           pz_refuse_tree(&c, a.kn, a.vn, a.ld_n, a.B, a.T, a.heads, a.scale, a.q, a.ld_q, a.out,
                          a.ld_out),
           code);
  };
#define C [&](pz_kv_cache & c, Call & a)
#define N (void)c, (void)a
  tree("tree: good", PZ_OK, C { N; });
  tree("tree: fp16", PZ_OK, C { N; c.type = PZ_F16; });
  tree("tree: no sequences", PZ_OK, C { N; a.B = 0; });
  tree("tree: fp32", PZ_ENOTSUP, C { N; c.type = PZ_F32; });
  tree("tree: head_dim 96", PZ_ENOTSUP, C { N; c.head_dim = 96; c.ld = a.ld_n = 192; });
  tree("tree: negative B", PZ_EINVAL, C { N; a.B = -1; });
  tree("tree: no nodes", PZ_EINVAL, C { N; a.T = 0; });
  tree("tree: the widest", PZ_OK, C { N; a.T = 64; });
  tree("tree: wider", PZ_ERANGE, C { N; a.T = 65; });
  tree("tree: null k", PZ_EINVAL, C { N; c.d_k = nullptr; });
  tree("tree: null v", PZ_EINVAL, C { N; c.d_v = nullptr; });
  tree("tree: null blocks", PZ_EINVAL, C { N; c.d_blocks = nullptr; });
  tree("tree: null lengths", PZ_EINVAL, C { N; c.d_len = nullptr; });
  tree("tree: no key heads", PZ_EINVAL, C { N; c.n_kv_heads = 0; });
  tree("tree: no pages", PZ_EINVAL, C { N; c.n_blocks = 0; });
  tree("tree: no table", PZ_EINVAL, C { N; c.max_blocks = 0; });
  tree("tree: pages of 8", PZ_OK, C { N; c.block_size = 8; });
  tree("tree: pages of 4", PZ_EINVAL, C { N; c.block_size = 4; });
  tree("tree: pages of 24", PZ_EINVAL, C { N; c.block_size = 24; });
  tree("tree: positions past 32 bits", PZ_ERANGE, C { N; c.block_size = 1 << 16; c.max_blocks = 1 << 15; });
  tree("tree: short slots", PZ_EINVAL, C { N; c.ld = 120; });
  tree("tree: slots off 16 bytes", PZ_EINVAL, C { N; c.ld = 132; });
  tree("tree: short nodes", PZ_EINVAL, C { N; a.ld_n = 120; });
  tree("tree: nodes off 16 bytes", PZ_EINVAL, C { N; a.ld_n = 129; });
  tree("tree: null kn", PZ_EINVAL, C { N; a.kn = nullptr; });
  tree("tree: null vn", PZ_EINVAL, C { N; a.vn = nullptr; });
  tree("tree: kn off 16 bytes", PZ_EINVAL, C { N; a.kn = h + 1; });
  tree("tree: v off 16 bytes", PZ_EINVAL, C { N; c.d_v = h + 4; });
  tree("tree: no heads", PZ_EINVAL, C { N; a.heads = 0; });
  tree("tree: three heads over two", PZ_EINVAL, C { N; a.heads = 3; });
  tree("tree: more heads", PZ_ERANGE, C { N; a.heads = (1 << 16) + 2; a.ld_q = a.ld_out = 1L << 23; });
  tree("tree: more key heads", PZ_ERANGE,
       C { N; c.n_kv_heads = (1 << 16) + 2; a.heads = c.n_kv_heads; c.ld = a.ld_n = a.ld_q = a.ld_out = 1L << 23; });
  tree("tree: more sequences than a launch", PZ_ERANGE, C { N; a.B = 1 << 23; });
  tree("tree: scale 0", PZ_EINVAL, C { N; a.scale = 0.0f; });
  tree("tree: scale NaN", PZ_EINVAL, C { N; a.scale = __builtin_nanf(""); });
  tree("tree: scale times log2(e) infinite", PZ_EINVAL, C { N; a.scale = 2.9e38f; });
  tree("tree: scale infinite", PZ_EINVAL, C { N; a.scale = __builtin_inff(); });
  tree("tree: null q", PZ_EINVAL, C { N; a.q = nullptr; });
  tree("tree: null out", PZ_EINVAL, C { N; a.out = nullptr; });
  tree("tree: short q rows", PZ_EINVAL, C { N; a.ld_q = 248; });
  tree("tree: out rows off 16 bytes", PZ_EINVAL, C { N; a.ld_out = 260; });
  tree("tree: q off 16 bytes", PZ_EINVAL, C { N; a.q = h + 2; });
  expect("tree: null cache", pz_refuse_cache(nullptr, h, h, 128, 2, 3), PZ_EINVAL);
  expect("append: as many as a launch", pz_refuse_cache(&c0, h, h, 128, (1 << 18) - 1, 64), PZ_OK);
  expect("append: more", pz_refuse_cache(&c0, h, h, 128, 1 << 18, 64), PZ_ERANGE);
  expect("launch: all its threads", pz_launch_fits((1 << 24) - 1, 256) ? PZ_TAKEN : PzRefusal{PZ_ERANGE, ""}, PZ_OK);
  expect("launch: one too many",
         pz_launch_fits(1 << 24, 256) ? PZ_TAKEN : PzRefusal{PZ_ERANGE, ""}, PZ_ERANGE);
  expect("append: good", pz_refuse_cache(&c0, h, h, 128, 2, 3), PZ_OK);
  return bad != 0;
}
