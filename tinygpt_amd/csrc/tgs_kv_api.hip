// tgs_kv_api.hip -- host side of the beam, tree-attention and paged-cache
// entry points of include/tgs_sampler.h: argument checks, the split of the
// work and the launches.  Nothing here allocates or synchronises.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <mutex>

#include "tgs_ctx.h"
#include "tgs_kv.h"

namespace {

using tgs::DeviceGuard;
using tgs::fail;
using tgs::hip_fail;

int shift_of(int page) {
  int s = 0;
  while ((1 << s) < page) s++;
  return s;
}

bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

int check_cache(tgs_ctx* h, const tgs_kv_cache* c) {
  if (!c || !c->k || !c->v) return fail(h, TGS_EINVAL, "cache: null buffer");
  if (c->dtype != TGS_BF16 && c->dtype != TGS_F16) return fail(h, TGS_EINVAL, "cache: dtype (bf16 or fp16)");
  if (c->page < 8 || c->page > 1024 || (c->page & (c->page - 1)))
    return fail(h, TGS_EINVAL, "cache: a page holds a power of two of tokens, 8 to 1024");
  if (c->layers < 1 || c->n_pages < 1 || c->kv_heads < 1 || c->head_dim < 8 || c->head_dim % 8 ||
      (int64_t)c->kv_heads * c->head_dim > 65535)
    return fail(h, TGS_EINVAL, "cache: shape");
  const int64_t whole = (int64_t)c->kv_heads * c->page * c->head_dim;
  if (c->k_page < whole || c->v_page < whole || c->k_page % 8 || c->v_page % 8 || c->k_layer % 8 || c->v_layer % 8 ||
      c->k_layer < 0 || c->v_layer < 0 || !aligned16(c->k) || !aligned16(c->v))
    return fail(h, TGS_EINVAL, "cache: strides and alignment");
  return TGS_OK;
}

int check_seqs(tgs_ctx* h, const tgs_kv_cache* c, const tgs_kv_seqs* s) {
  if (!s || s->B < 0 || s->width < 1 || (int64_t)s->width * c->page > INT32_MAX)
    return fail(h, TGS_EINVAL, "sequences: shape");
  if (s->B > 0 && (!s->tables || !s->lens)) return fail(h, TGS_EINVAL, "sequences: null buffer");
  return TGS_OK;
}

// The kernels whose dynamic LDS passes the default limit, once per device.
int raise_lds(tgs_ctx* h) {
  static std::mutex mu;
  static uint64_t ready = 0;
  const uint64_t bit = 1ull << (h->device & 63);
  std::lock_guard<std::mutex> lock(mu);
  if (h->device < 64 && (ready & bit)) return TGS_OK;
  hipError_t e = tgs::set_kv_fork_lds_limit(h->lds_limit);
  if (e == hipSuccess) e = tgs::set_attn_lds();
  if (e != hipSuccess) return hip_fail(h, e, "LDS limit");
  if (h->device < 64) ready |= bit;
  return TGS_OK;
}

int write_args(tgs_ctx* h, const tgs_kv_cache* c, const tgs_kv_rows* r, const tgs_kv_seqs* s, int T, int32_t* lens_out,
               tgs::KvWriteArgs& a) {
  if (int rc = check_cache(h, c)) return rc;
  if (int rc = check_seqs(h, c, s)) return rc;
  if (T < 1) return fail(h, TGS_EINVAL, "rows: at least one per sequence");
  std::memset(&a, 0, sizeof(a));
  if (s->B == 0) return TGS_OK;
  if (!r || !r->k || !r->v || !lens_out) return fail(h, TGS_EINVAL, "null buffer");
  if (lens_out == s->lens) return fail(h, TGS_EINVAL, "lens_out must not be lens");
  a.c = *c;
  a.r = *r;
  a.tables = s->tables;
  a.P = s->width;
  a.B = s->B;
  a.T = T;
  a.page_shift = shift_of(c->page);
  a.lens = s->lens;
  a.lens_out = lens_out;
  a.half_d = tgs::fast_div(c->head_dim / 2);
  a.chunks = tgs::fast_div(c->head_dim / 8);
  a.heads = tgs::fast_div(c->kv_heads);
  return TGS_OK;
}

}  // namespace

extern "C" {

int tgs_beam_select(tgs_handle h, const void* d_logits, tgs_dtype dt, int G, int W, int V, int64_t row_stride,
                    const float* d_scores, int n_out, const int32_t* d_hist, const int32_t* d_hist_len, int hist_cap,
                    float* d_out_scores, int32_t* d_out_parents, int32_t* d_out_tokens, int32_t* d_out_hist,
                    int32_t* d_out_hist_len, tgs_stream stream) {
  if (!h) return TGS_EINVAL;
  if (dt != TGS_F32 && dt != TGS_BF16) return fail(h, TGS_EINVAL, "dtype");
  if (G < 0 || W < 1 || W > tgs::BEAM_MAX || V < 1 || row_stride < V || n_out < 1 || n_out > tgs::BEAM_MAX ||
      (int64_t)n_out > (int64_t)W * V || hist_cap < 0)
    return fail(h, TGS_EINVAL, "shape");
  if (G == 0) return TGS_OK;
  if (!d_logits || !d_scores || !d_out_scores || !d_out_parents || !d_out_tokens ||
      (hist_cap > 0 && (!d_hist || !d_hist_len || !d_out_hist || !d_out_hist_len)))
    return fail(h, TGS_EINVAL, "null buffer");
  if (V > h->max_vocab) return fail(h, TGS_ETOOBIG, "vocab beyond the handle's limit");
  if ((int64_t)G * W > h->max_batch) return fail(h, TGS_ETOOBIG, "rows beyond the handle's limit");
  // chunks per row: about four workgroups per CU, chunks of at least 2048 ids,
  // never more ids than a workgroup's registers hold
  const int rows = G * W, epv = dt == TGS_BF16 ? 8 : 4, most = tgs::beam_chunk_ids(dt);
  int S = std::min(std::max(4 * h->num_cu / rows, 1), 32);
  S = std::max(std::min(S, V / 2048), 1);
  S = std::max(S, (V + most - 1) / most);
  const int L = ((V + S - 1) / S + epv - 1) / epv * epv;
  S = (V + L - 1) / L;
  // [rows * S][n_out] composites, then [rows * S][2] doubles
  if ((size_t)rows * S * (n_out + 2) > h->ws_words) return fail(h, TGS_ETOOBIG, "rows beyond the handle's workspace");
  DeviceGuard g(h->device);
  if (!g.ok) return fail(h, TGS_EHIP, "hipSetDevice");
  tgs::BeamArgs a;
  std::memset(&a, 0, sizeof(a));
  a.logits = d_logits;
  a.row_stride = row_stride;
  a.G = G;
  a.W = W;
  a.V = V;
  a.n = n_out;
  a.scores = d_scores;
  a.hist = d_hist;
  a.hist_len = d_hist_len;
  a.H = hist_cap;
  a.out_scores = d_out_scores;
  a.out_parents = d_out_parents;
  a.out_tokens = d_out_tokens;
  a.out_hist = d_out_hist;
  a.out_hist_len = d_out_hist_len;
  a.S = S;
  a.L = L;
  a.lists = h->ws;
  a.sums = (double*)(h->ws + (size_t)rows * S * n_out);
  hipError_t e = tgs::launch_beam(a, dt, (hipStream_t)stream);
  if (e != hipSuccess) return hip_fail(h, e, "beam kernel launch");
  return TGS_OK;
}

int tgs_tree_attention(tgs_handle h, const tgs_kv_cache* cache, const tgs_kv_rows* rows, const tgs_kv_seqs* seqs,
                       const tgs_attn* attn, tgs_stream stream) {
  if (!h) return TGS_EINVAL;
  if (int rc = check_cache(h, cache)) return rc;
  if (int rc = check_seqs(h, cache, seqs)) return rc;
  if (!attn || !rows) return fail(h, TGS_EINVAL, "null argument");
  const int D = cache->head_dim, T = attn->T, B = seqs->B;
  if (cache->layers != 1) return fail(h, TGS_EINVAL, "attention: one layer of the cache");
  if (D != 64 && D != 96 && D != 128 && D != 256) return fail(h, TGS_EINVAL, "attention: head_dim 64, 96, 128 or 256");
  if (T < 1 || T > tgs::KV_MAX_NODES) return fail(h, TGS_EINVAL, "attention: 1 to 64 nodes");
  if (attn->q_heads < 1 || attn->q_heads % cache->kv_heads)
    return fail(h, TGS_EINVAL, "attention: query heads a multiple of key heads");
  if (!(attn->scale > 0.0f) || !(attn->scale < 1e30f) || attn->max_len < 0)
    return fail(h, TGS_EINVAL, "attention: scale and max_len");
  if (B == 0) return TGS_OK;
  if (!attn->q || !attn->out || !rows->k || !rows->v) return fail(h, TGS_EINVAL, "null buffer");
  if (!aligned16(attn->out)) return fail(h, TGS_EINVAL, "attention: out must be 16-byte aligned");
  if ((int64_t)B * cache->kv_heads * T * (attn->q_heads / cache->kv_heads) > INT32_MAX)
    return fail(h, TGS_ETOOBIG, "attention: rows");
  DeviceGuard g(h->device);
  if (!g.ok) return fail(h, TGS_EHIP, "hipSetDevice");
  if (int rc = raise_lds(h)) return rc;
  tgs::AttnArgs a;
  std::memset(&a, 0, sizeof(a));
  a.q = attn->q;
  a.k_new = rows->k;
  a.v_new = rows->v;
  a.q_b = attn->q_seq, a.q_t = attn->q_tok, a.q_h = attn->q_head;
  a.kn_b = rows->k_seq, a.kn_t = rows->k_tok, a.kn_h = rows->k_head;
  a.vn_b = rows->v_seq, a.vn_t = rows->v_tok, a.vn_h = rows->v_head;
  a.k = cache->k;
  a.v = cache->v;
  a.k_page = cache->k_page;
  a.v_page = cache->v_page;
  a.tables = seqs->tables;
  a.lens = seqs->lens;
  a.parents = attn->parents;
  a.out = attn->out;
  a.lse = attn->lse;
  a.B = B;
  a.T = T;
  a.Hq = attn->q_heads;
  a.Hkv = cache->kv_heads;
  a.G = a.Hq / a.Hkv;
  a.D = D;
  a.P = seqs->width;
  a.n_pages = cache->n_pages;
  a.page_shift = shift_of(cache->page);
  a.scale_log2 = attn->scale * 1.4426950408889634f;
  a.M = T * a.G;
  const tgs::AttnPlan p = tgs::attn_plan(a.M, D);
  a.QB = p.QB;
  a.nqb = p.nqb;
  // Workers: as many as the chip holds at once, of at least p.least tiles, as
  // far as the workspace has room for their parts.  Where every (sequence,
  // key head) is short, one workgroup each and no join.
  const int64_t len = std::min<int64_t>(attn->max_len, (int64_t)a.P * cache->page);
  const int64_t per = (len + p.tile - 1) / p.tile + (T + p.tile - 1) / p.tile;
  int64_t n = 0;
  if (per > 2 * p.least) {
    n = std::min<int64_t>((int64_t)h->num_cu * p.per_cu / p.nqb, (per * B * a.Hkv + p.least - 1) / p.least);
    const int64_t part = (int64_t)2 * p.QB * (D + 2) * p.nqb;  // floats
    n = std::min(n, (int64_t)h->ws_words * 2 / part);
    if (p.nqb > 1 && n >= 8) n = n / 8 * 8;  // (row groups of a worker on one XCD)
  }
  a.nwg = (int)n;
  a.part_o = (float*)h->ws;
  a.part_ml = a.part_o + n * p.nqb * 2 * p.QB * D;
  hipError_t e = tgs::launch_attn(a, p, cache->dtype, (hipStream_t)stream);
  if (e != hipSuccess) return hip_fail(h, e, "attention kernel launch");
  return TGS_OK;
}

int tgs_kv_append(tgs_handle h, const tgs_kv_cache* cache, const tgs_kv_rows* rows, const tgs_kv_seqs* seqs, int T,
                  const int32_t* d_counts, int32_t* d_lens_out, tgs_stream stream) {
  if (!h) return TGS_EINVAL;
  tgs::KvWriteArgs a;
  if (int rc = write_args(h, cache, rows, seqs, T, d_lens_out, a)) return rc;
  if (a.B == 0) return TGS_OK;
  a.counts = d_counts;
  // blocks that T rows, or as many as a table holds, lie in at most
  a.nblk = T == 1 ? 1 : (int)((std::min<int64_t>(T, (int64_t)a.P * cache->page) + 7) / 8 + 1);
  if ((int64_t)a.nblk * a.B * cache->layers > INT32_MAX) return fail(h, TGS_ETOOBIG, "rows");
  DeviceGuard g(h->device);
  if (!g.ok) return fail(h, TGS_EHIP, "hipSetDevice");
  hipError_t e = tgs::launch_kv_append(a, (hipStream_t)stream);
  if (e != hipSuccess) return hip_fail(h, e, "append kernel launch");
  return TGS_OK;
}

int tgs_tree_commit(tgs_handle h, const tgs_kv_cache* cache, const tgs_kv_rows* rows, const tgs_kv_seqs* seqs, int T,
                    const int32_t* d_parents, const int32_t* d_draft, const int32_t* d_sampled, int32_t* d_n_acc,
                    int32_t* d_tokens, int32_t* d_path, int32_t* d_lens_out, tgs_stream stream) {
  if (!h) return TGS_EINVAL;
  if (T > tgs::KV_MAX_NODES) return fail(h, TGS_EINVAL, "commit: at most 64 nodes");
  tgs::KvWriteArgs a;
  if (int rc = write_args(h, cache, rows, seqs, T, d_lens_out, a)) return rc;
  if (a.B == 0) return TGS_OK;
  if (!d_parents || !d_draft || !d_sampled || !d_n_acc || !d_tokens || !d_path)
    return fail(h, TGS_EINVAL, "null buffer");
  a.parents = d_parents;
  a.draft = d_draft;
  a.sampled = d_sampled;
  a.n_acc = d_n_acc;
  a.tokens = d_tokens;
  a.path = d_path;
  a.nblk = T < 3 ? 1 : 2;  // (a path is seldom longer than two blocks)
  if ((int64_t)a.nblk * a.B * cache->layers > INT32_MAX) return fail(h, TGS_ETOOBIG, "rows");
  DeviceGuard g(h->device);
  if (!g.ok) return fail(h, TGS_EHIP, "hipSetDevice");
  hipError_t e = tgs::launch_tree_commit(a, (hipStream_t)stream);
  if (e != hipSuccess) return hip_fail(h, e, "commit kernel launch");
  return TGS_OK;
}

int tgs_kv_fork(tgs_handle h, const tgs_kv_cache* cache, const tgs_kv_seqs* seqs, const int32_t* d_parents, int room,
                int32_t* d_tables_out, int32_t* d_lens_out, tgs_stream stream) {
  if (!h) return TGS_EINVAL;
  if (int rc = check_cache(h, cache)) return rc;
  if (int rc = check_seqs(h, cache, seqs)) return rc;
  if (room < 0) return fail(h, TGS_EINVAL, "fork: room");
  const int R = seqs->B, P = seqs->width;
  if (R == 0) return TGS_OK;
  if (!d_parents || !d_tables_out || !d_lens_out) return fail(h, TGS_EINVAL, "null buffer");
  if (d_tables_out == seqs->tables || d_lens_out == seqs->lens)
    return fail(h, TGS_EINVAL, "fork: outputs must not be inputs");
  if ((int64_t)R * P >= INT32_MAX || cache->layers > 32767) return fail(h, TGS_ETOOBIG, "fork: rows");
  // workspace: copies, and for pools beyond the planning kernel's LDS owners and free pages
  const size_t pages = tgs::kv_fork_lds(cache->n_pages, R) ? 0 : (size_t)cache->n_pages;
  if ((size_t)R * 2 + pages > h->ws_words)
    return fail(h, TGS_ETOOBIG, "fork: pages beyond the handle's workspace");
  DeviceGuard g(h->device);
  if (!g.ok) return fail(h, TGS_EHIP, "hipSetDevice");
  if (int rc = raise_lds(h)) return rc;
  tgs::KvForkArgs a;
  std::memset(&a, 0, sizeof(a));
  a.c = *cache;
  a.tables = seqs->tables;
  a.lens = seqs->lens;
  a.parents = d_parents;
  a.tables_out = d_tables_out;
  a.lens_out = d_lens_out;
  a.R = R;
  a.P = P;
  a.room = room;
  a.page_shift = shift_of(cache->page);
  a.copies = (int4*)h->ws;
  a.owner = (int*)(a.copies + R);
  a.fresh = a.owner + pages;
  hipError_t e = tgs::launch_kv_fork(a, h->num_cu, (hipStream_t)stream);
  if (e != hipSuccess) return hip_fail(h, e, "fork kernel launch");
  return TGS_OK;
}

}  // extern "C"
