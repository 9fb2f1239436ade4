// kv_case.cpp -- one call of a beam, attention or cache entry point on the CPU
// simulation of the kernels (TEST INFRASTRUCTURE ONLY).
//   kv_case <op> <dir>   reads <dir>/meta.txt (name value pairs) and the raw
//                        arrays <dir>/<name>.bin, each loaded into an
//                        allocation of exactly its size; writes the outputs
//                        (and the pools) next to them and prints the status.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <string>

#include <unistd.h>

#include "tgs_ctx.h"

static std::string dir;
static std::map<std::string, double> meta;
static std::map<std::string, std::pair<char*, size_t>> arrays;

static void* in(const std::string& name) {
  if (arrays.count(name)) return arrays[name].first;
  FILE* f = std::fopen((dir + "/" + name + ".bin").c_str(), "rb");
  if (!f) return nullptr;
  std::fseek(f, 0, SEEK_END);
  const size_t n = std::ftell(f);
  std::fseek(f, 0, SEEK_SET);
  char* p = (char*)std::aligned_alloc(16, (n + 15) / 16 * 16);
  if (n % 16) {  // (exactly n bytes: reads past them are found)
    std::free(p);
    p = (char*)std::malloc(n);
  }
  if (n && std::fread(p, 1, n, f) != n) std::abort();
  std::fclose(f);
  arrays[name] = {p, n};
  return p;
}
static int I(const char* name) { return (int)meta[name]; }
static int64_t L(const char* name) { return (int64_t)meta[name]; }

int main(int argc, char** argv) {
  if (argc < 3) return 2;
  alarm(900);
  const std::string op = argv[1];
  dir = argv[2];
  FILE* m = std::fopen((dir + "/meta.txt").c_str(), "r");
  if (!m) return 3;
  char key[64];
  double val;
  while (std::fscanf(m, "%63s %lf", key, &val) == 2) meta[key] = val;
  std::fclose(m);
  tgs_ctx h;
  h.max_batch = 4096;
  h.max_vocab = 152064;
  h.num_cu = I("num_cu");
  h.lds_limit = 163840;
  h.ws_words = (size_t)L("ws_words");
  h.ws = (unsigned long long*)std::malloc(h.ws_words * 8);
  tgs_kv_cache c = {in("k"), in("v"), L("k_layer"), L("k_page"), L("v_layer"), L("v_page"), I("layers"), I("pages"),
                    I("page"), I("kv_heads"), I("D"), I("dtype")};
  tgs_kv_rows r = {in("k_new"), in("v_new"), L("kl"), L("ks"), L("kt"), L("kh"), L("vl"), L("vs"), L("vt"), L("vh")};
  tgs_kv_seqs s = {(const int32_t*)in("tables"), (const int32_t*)in("lens"), I("B"), I("P")};
  int rc = -100;
  auto i32 = [&](const char* n) { return (int32_t*)in(n); };
  auto f32 = [&](const char* n) { return (float*)in(n); };
  if (op == "beam")
    rc = tgs_beam_select(&h, in("logits"), (tgs_dtype)I("dtype"), I("G"), I("W"), I("V"), L("stride"), f32("scores"), I("n"),
                         i32("hist"), i32("hist_len"), I("H"), f32("o_scores"), i32("o_parents"), i32("o_tokens"),
                         i32("o_hist"), i32("o_hist_len"), nullptr);
  else if (op == "attn") {
    tgs_attn a = {in("q"), L("qs"), L("qt"), L("qh"), i32("parents"), in("o_out"), f32("o_lse"), I("T"), I("Hq"),
                  I("max_len"), (float)meta["scale"]};
    rc = tgs_tree_attention(&h, &c, &r, &s, &a, nullptr);
  } else if (op == "append")
    rc = tgs_kv_append(&h, &c, &r, &s, I("T"), i32("counts"), i32("o_lens"), nullptr);
  else if (op == "commit")
    rc = tgs_tree_commit(&h, &c, &r, &s, I("T"), i32("parents"), i32("draft"), i32("sampled"), i32("o_n_acc"),
                         i32("o_tokens"), i32("o_path"), i32("o_lens"), nullptr);
  else if (op == "fork")
    rc = tgs_kv_fork(&h, &c, &s, i32("parents"), I("room"), i32("o_tables"), i32("o_lens"), nullptr);
  std::printf("rc %d %s\n", rc, h.err.c_str());
  for (auto& [name, a] : arrays)
    if (name.rfind("o_", 0) == 0 || name == "k" || name == "v") {
      FILE* f = std::fopen((dir + "/" + name + ".out").c_str(), "wb");
      std::fwrite(a.first, 1, a.second, f);
      std::fclose(f);
    }
  return 0;
}

// (the shim poisons the section that plain __shared__ variables lie in; these
// kernels have none)
static __attribute__((section("tgs_lds"), used)) unsigned char kv_case_lds[16];
