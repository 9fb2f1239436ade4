// tgs_kv.h -- argument blocks of the paged-cache, beam and tree-attention
// kernels (host entry points in tgs_kv_api.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/tgs_sampler.h"

namespace tgs {

// x / d for x < 2^16 and 1 <= d < 2^16 by a multiplication: with
// m = floor(2^32 / d) + 1 the product's error is below x / 2^32 < 1 / d.
struct FastDiv {
  unsigned m, d;
};
inline FastDiv fast_div(unsigned d) { return {d == 1 ? 0u : (unsigned)((1ull << 32) / d) + 1u, d}; }

constexpr int KV_MAX_NODES = 64;   // nodes of a drafted tree
constexpr int KV_NT = 256;         // threads of the write and copy kernels
constexpr int KV_PLAN_NT = 1024;   // threads of the fork's planning kernel

// New rows written to the cache (append: the first counts[b] of sequence b;
// commit: the accepted path of its tree).
struct KvWriteArgs {
  tgs_kv_cache c;
  tgs_kv_rows r;
  const int* tables;  // [B][P]
  int P, B, T, page_shift;
  int nblk;           // workgroups per (sequence, layer)
  const int* lens;    // [B]
  const int* counts;  // [B] or nullptr (T for every sequence); append only
  const int* parents;  // [B][T] from here on commit only
  const int* draft;
  const int* sampled;
  int* n_acc;   // [B]
  int* tokens;  // [B][T]
  int* path;    // [B][T]
  int* lens_out;  // [B]
  FastDiv half_d, chunks, heads;  // head_dim / 2, head_dim / 8, kv_heads
};
hipError_t launch_kv_append(const KvWriteArgs& a, hipStream_t st);
hipError_t launch_tree_commit(const KvWriteArgs& a, hipStream_t st);

struct KvForkArgs {
  tgs_kv_cache c;
  const int* tables;   // [R][P]
  const int* lens;     // [R]
  const int* parents;  // [R]
  int* tables_out;     // [R][P]
  int* lens_out;       // [R]
  int R, P, room, page_shift;
  int* owner;          // [n_pages] workspace, for pools beyond the planning kernel's LDS
  int* fresh;          // [n_pages] workspace, likewise: the free pages, in order
  int4* copies;        // [R] workspace: source page, new page, 8-token blocks, -
};
size_t kv_fork_lds(int n_pages, int rows);  // dynamic LDS of the planning kernel (0: its lists lie in the workspace)
hipError_t launch_kv_fork(const KvForkArgs& a, int num_cu, hipStream_t st);
hipError_t set_kv_fork_lds_limit(size_t bytes);

// Selection over beams and vocabulary.
constexpr int BEAM_NT = 256;
constexpr int BEAM_MAX = 64;  // beams of a request, and entries selected from it, at most
constexpr int BEAM_NVT = 8;   // 16-byte vectors a thread holds of its chunk
constexpr int BEAM_CAP = 1024;
struct BeamArgs {
  const void* logits;  // [G * W] rows of V
  long long row_stride;
  int G, W, V, n;
  const float* scores;  // [G * W]
  const int* hist;      // [G * W][H] or nullptr
  const int* hist_len;
  int H;
  float* out_scores;  // [G * n]
  int* out_parents;
  int* out_tokens;
  int* out_hist;
  int* out_hist_len;
  int S, L;                   // chunks per row, ids per chunk (whole vectors)
  unsigned long long* lists;  // [G * W * S][n] largest composites of each chunk, 0 padded
  double* sums;               // [G * W * S][2] e and the sum of 2^(x log2 e - e), or m and minus the sum of e^(x - m)
};
int beam_chunk_ids(int dtype);
hipError_t launch_beam(const BeamArgs& a, int dtype, hipStream_t st);

// Attention of drafted nodes over a paged cache and their own ancestors.
struct AttnArgs {
  const void* q;
  const void* k_new;
  const void* v_new;
  long long q_b, q_t, q_h, kn_b, kn_t, kn_h, vn_b, vn_t, vn_h;  // strides, elements
  const void* k;
  const void* v;
  long long k_page, v_page;
  const int* tables;
  const int* lens;
  const int* parents;  // nullptr: a chain
  void* out;           // [B][T][Hq][D]
  float* lse;          // [B][T][Hq] or nullptr
  int B, T, Hq, Hkv, G, D, P, n_pages, page_shift;
  float scale_log2;    // scale * log2(e)
  int M;               // query rows of a key head: T * G
  int QB, nqb;         // rows of a workgroup, groups of them per key head
  int nwg;             // workers per row group: each takes an even share of the tiles; 0: one workgroup per (sequence, head)
  float* part_o;       // [nqb * nwg][2][QB][D]
  float* part_ml;      // [nqb * nwg][2][QB][2]
};
struct AttnPlan {
  int wide;   // 0: a wave owns its tiles; 1: tiles shared through LDS
  int tile;   // tokens of a unit of work
  int QB, nqb;
  int per_cu;  // workgroups that a CU holds
  int least;   // tiles worth a worker of their own
};
AttnPlan attn_plan(int M, int D);
hipError_t launch_attn(const AttnArgs& a, const AttnPlan& p, int dtype, hipStream_t st);
hipError_t set_attn_lds();  // dynamic LDS of the attention kernels

}  // namespace tgs
