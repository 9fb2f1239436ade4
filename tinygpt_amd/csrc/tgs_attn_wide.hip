// tgs_attn_wide.hip -- tree attention where a key head has more than 32 query
// rows: a tile's keys and values go through LDS, where every wave of the
// workgroup, each with 32 rows of its own, reads them.
//
// Tiles of 64 tokens.  The next tile is on its way to registers while this
// one is worked on.  Keys lie in LDS row by row with the 16-byte chunks of a
// row permuted by the row's number, so that the 16 lanes served together take
// 16 different chunks; values lie as in the cache, where a lane's operands
// are neighbours already.
#include "tgs_attn.h"

namespace tgs {
namespace attn {



template <typename DT, int D, int QW>
struct Wide {
  static constexpr int NTHR = QW * 64, KK = D / 16, DT32 = D / 32, C = D / 8;
  static constexpr int NCH = (WTILE * C + NTHR - 1) / NTHR;  // chunks a thread moves, of keys and of values
  static constexpr bool EVEN = WTILE * C % NTHR == 0;
  struct Shared {
    uint4 k[WTILE * C];
    uint4 v[WTILE * C];
  };

  const AttnArgs& a;
  const int tid, lane, wave, col, half;
  int b, h, qb, len, nc;
  const int* table;
  bool bad;

  __device__ __forceinline__ Wide(const AttnArgs& a_)
      : a(a_), tid((int)threadIdx.x), lane(lane_id()), wave(tid >> 6), col(lane & 31), half(lane >> 5), b(0), h(0), qb(0),
        len(0), nc(0), table(nullptr), bad(false) {}

  // Where chunk ch of row tok lies.
  static __device__ __forceinline__ int at_key(int tok, int ch) {
    if constexpr (C % 16 == 0) return tok * C + (ch ^ (tok & 15));
    else if constexpr (C == 8) return tok * C + (ch ^ ((tok >> 1) & 7));
    else {  // 12 chunks: rows 4 apart start at the same banks; turned by 0 .. 3 they differ
      const int x = ch + ((tok >> 2) & 3);
      return tok * C + (x < C ? x : x - C);
    }
  }

  // Page of each of the tile's eight 8-token blocks, block lane % 8 in a lane.
  __device__ __forceinline__ int entries(int i) const {
    if (i >= nc) return 0;
    const int blk = i * WTILE + (lane & 7) * 8, last = len - 1;
    return table[(blk < last ? blk : last) >> a.page_shift];
  }

  __device__ __forceinline__ void load(int i, int entry, uint4 (&k)[NCH], uint4 (&v)[NCH]) {
    if (i < nc) {  // (the drafted nodes' tile goes to LDS directly)
      if ((unsigned)entry >= (unsigned)a.n_pages) {
        bad = true;  // (its sequence's rows become NaN)
        entry = 0;
      }
      const long long head = ((long long)h * D) << a.page_shift;
      const int mask = (1 << a.page_shift) - 1;
      const bool tail = (i + 1) * WTILE > len;
#pragma unroll
      for (int n = 0; n < NCH; n++) {
        const int c = EVEN || n * NTHR + tid < WTILE * C ? n * NTHR + tid : 0;
        const int tok = c / C, ch = c - tok * C;
        int p = i * WTILE + tok;
        p = p < len ? p : len - 1;
        const long long pg = __shfl(entry, tok >> 3, 64);
        k[n] = *(const uint4*)((const uint16_t*)a.k + pg * a.k_page + head + (long long)(p & mask) * D + ch * 8);
      }
#pragma unroll
      for (int n = 0; n < NCH; n++) {
        const int c = EVEN || n * NTHR + tid < WTILE * C ? n * NTHR + tid : 0;
        const int blk = c / D, d = c - blk * D;
        int p = i * WTILE + blk * 8;
        const int last = (len - 1) & ~7;
        const int first = p;
        p = p < last ? p : last;
        const long long pg = __shfl(entry, blk, 64);
        v[n] = *(const uint4*)((const uint16_t*)a.v + pg * a.v_page + head + (long long)(p & mask) * D + d * 8);
        // what lies past the end is not 0 (it may be anything, NaN too)
        if (tail) v[n] = keep_first(v[n], len - first);
      }
    }
  }

  __device__ __forceinline__ void store(Shared& s, const uint4 (&k)[NCH], const uint4 (&v)[NCH]) {
#pragma unroll
    for (int n = 0; n < NCH; n++) {
      const int c = n * NTHR + tid;
      if (EVEN || c < WTILE * C) {
        const int tok = c / C;
        s.k[at_key(tok, c - tok * C)] = k[n];
        s.v[c] = v[n];
      }
    }
  }

  // The drafted nodes' tile, from their own rows.
  __device__ __forceinline__ void store_tree(Shared& s, int t0) {
    const uint16_t* kb = (const uint16_t*)a.k_new + b * a.kn_b + h * a.kn_h;
    const uint16_t* vb = (const uint16_t*)a.v_new + b * a.vn_b + h * a.vn_h;
#pragma unroll 1
    for (int c = tid; c < WTILE * C; c += NTHR) {
      const int tok = c / C, ch = c - tok * C, p = t0 + tok < a.T ? t0 + tok : a.T - 1;
      s.k[at_key(tok, ch)] = load_row16<false>(kb + p * a.kn_t + ch * 8);
      const int blk = c / D, d = c - blk * D;
      s.v[c] = tree_values(vb + d, a.vn_t, t0 + blk * 8, a.T);
    }
  }

  __device__ __forceinline__ void segment(Shared& s, int t0, int t1, bool full, long long part) {
    len = seq_len(a, b);
    nc = (len + WTILE - 1) / WTILE;
    table = a.tables + (long long)b * a.P;
    bad = false;
    const int row0 = qb * a.QB + wave * 32;  // of the M
    const bool work = row0 < a.M;
    const int i = row0 + col;
    const int node = i < a.M ? i / a.G : 0, hg = i < a.M ? i - node * a.G : 0;
    u64 sees = t1 > nc ? ancestors(a, b) : 0ull;
    sees = ((u64)(uint32_t)__shfl((int)(sees >> 32), node, 64) << 32) | (uint32_t)__shfl((int)(uint32_t)sees, node, 64);
    uint4 q[KK];
    {
      const uint16_t* p = (const uint16_t*)a.q + b * a.q_b + node * a.q_t + (long long)(h * a.G + hg) * a.q_h + half * 8;
#pragma unroll
      for (int kk = 0; kk < KK; kk++) q[kk] = load_row16<false>(p + kk * 16);
    }
    // product row r = 8 x + 4 y + j (j < 4, y < 2) of a half tile is its token 16 (x / 2) + 8 y + 4 (x % 2) + j
    const int tok = (col >> 4) * 16 + ((col >> 2) & 1) * 8 + ((col >> 3) & 1) * 4 + (col & 3);
    f32x16 o[DT32];
    float m = NEG, l = 0.0f;
#pragma unroll
    for (int d = 0; d < DT32; d++)
#pragma unroll
      for (int x = 0; x < 16; x++) o[d][x] = 0.0f;
    uint4 k[NCH], v[NCH];
    int e = entries(t0);
    load(t0, e, k, v);
    e = t0 + 1 < t1 ? entries(t0 + 1) : e;
    for (int t = t0; t < t1; t++) {
      __syncthreads();
      if (t < nc)
        store(s, k, v);
      else
        store_tree(s, (t - nc) * WTILE);
      __syncthreads();
      if (t + 1 < t1) {
        load(t + 1, e, k, v);
        e = t + 2 < t1 ? entries(t + 2) : e;
      }
      if (!work) continue;
      f32x16 sc[2];
#pragma unroll
      for (int x = 0; x < 2; x++) {
#pragma unroll
        for (int j = 0; j < 16; j++) sc[x][j] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < KK; kk++)
          sc[x] = mfma32<DT>(s.k[at_key(x * 32 + tok, kk * 2 + half)], q[kk], sc[x]);
      }
      // element j of half tile x is token 32 x + 16 (j / 8) + 8 half + j % 8
      if (t >= nc) {
        const u64 in = sees >> (8 * half);
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
          for (int j = 0; j < 16; j++)
            if (!((in >> (32 * x + 16 * (j >> 3) + (j & 7))) & 1)) sc[x][j] = NEG;
      } else if ((t + 1) * WTILE > len) {
        const int left = len - t * WTILE - 8 * half;
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
          for (int j = 0; j < 16; j++)
            if (32 * x + 16 * (j >> 3) + (j & 7) >= left) sc[x][j] = NEG;
      }
      float top = sc[0][0];
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int j = 0; j < 16; j++) top = fmaxf(top, sc[x][j]);
      top *= a.scale_log2;
      if (__ballot(top > m + SLACK)) {
        top = fmaxf(top, xor_lane<32>(top));
        const float now = fmaxf(m, top);
        const float f = m == NEG ? 0.0f : exp2_hw(m - now);
        m = now;
        l *= f;
#pragma unroll
        for (int d = 0; d < DT32; d++) o[d] *= f;
      }
      const float base = m == NEG ? 0.0f : m;
      uint4 p[4];
#pragma unroll
      for (int y = 0; y < 4; y++) {  // the 16 tokens 16 y .. of the tile
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
          w[j] = exp2_hw(__builtin_fmaf(sc[y >> 1][(y & 1) * 8 + j], a.scale_log2, -base));
          l += w[j];
        }
        p[y] = make_uint4(pack2<DT>(w[0], w[1]), pack2<DT>(w[2], w[3]), pack2<DT>(w[4], w[5]), pack2<DT>(w[6], w[7]));
      }
#pragma unroll
      for (int y = 0; y < 4; y++)
#pragma unroll
        for (int d = 0; d < DT32; d++) o[d] = mfma32<DT>(s.v[(y * 2 + half) * D + d * 32 + col], p[y], o[d]);
    }
    l += xor_lane<32>(l);
    if (__ballot(bad)) l = __builtin_nanf("");  // (every wave read every entry)
    if (i >= a.M) return;
    if (full) {
      const long long row = ((long long)b * a.T + node) * a.Hq + h * a.G + hg;
      const float r = 1.0f / l;
#pragma unroll
      for (int d = 0; d < DT32; d++)
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const f32x4 y = {o[d][4 * x], o[d][4 * x + 1], o[d][4 * x + 2], o[d][4 * x + 3]};
          store4<DT>((uint16_t*)a.out + row * D + d * 32 + x * 8 + half * 4, y * r);
        }
      if (a.lse && half == 0) a.lse[row] = row_lse(m, l);
    } else {
      const long long row = part + wave * 32 + col;
#pragma unroll
      for (int d = 0; d < DT32; d++)
#pragma unroll
        for (int x = 0; x < 4; x++)
          *(f32x4*)(a.part_o + row * D + d * 32 + x * 8 + half * 4) =
              f32x4{o[d][4 * x], o[d][4 * x + 1], o[d][4 * x + 2], o[d][4 * x + 3]};
      if (half == 0) {
        a.part_ml[row * 2] = m;
        a.part_ml[row * 2 + 1] = l;
      }
    }
  }
};

template <typename DT, int D, int QW>
__global__ __launch_bounds__(QW * 64, D == 256 ? 1 : 2) void wide_kernel(AttnArgs a) {
  typedef Wide<DT, D, QW> K;
  TGS_DYN_SMEM(dyn);
  typename K::Shared& s = *(typename K::Shared*)dyn;
  K n(a);
  const int tree = (a.T + WTILE - 1) / WTILE;
  if (a.nwg == 0) {
    const int seg = blockIdx.x / a.nqb;
    n.qb = blockIdx.x % a.nqb;
    n.b = seg / a.Hkv;
    n.h = seg % a.Hkv;
    n.segment(s, 0, cache_tiles<WTILE>(a, n.b) + tree, true, 0);
    return;
  }
  // the row groups that read the same tiles run at the same time on one XCD
  // (workgroups are dealt out to the 8 XCDs in turn)
  const int x = blockIdx.x;
  const int w = a.nwg % 8 == 0 ? x / (8 * a.nqb) * 8 + x % 8 : x / a.nqb;
  n.qb = a.nwg % 8 == 0 ? x / 8 % a.nqb : x % a.nqb;
  int before, all, b;
  tiles_before<WTILE>(a, 0, before, all);
  const long long U = (long long)all * a.Hkv;
  const long long u0 = share_start(U, a.nwg, w), u1 = share_start(U, a.nwg, w + 1);
  if (u0 == u1) return;
  long long skip;
  find_tile<WTILE>(a, u0, a.Hkv, b, skip);
  int nt = cache_tiles<WTILE>(a, b) + tree;
  int h = (int)((u0 - skip) / nt), at = (int)((u0 - skip) - (long long)h * nt);
  for (long long u = u0; u < u1;) {
    const int end = nt - at < u1 - u ? nt : at + (int)(u1 - u);
    n.b = b;
    n.h = h;
    n.segment(s, at, end, at == 0 && end == nt, ((long long)(n.qb * a.nwg + w) * 2 + (u != u0)) * a.QB);
    u += end - at;
    at = 0;
    if (++h == a.Hkv) {
      h = 0;
      if (++b < a.B) nt = cache_tiles<WTILE>(a, b) + tree;
    }
  }
}

template <typename DT, int D, int QW>
hipError_t wide_run(const AttnArgs& a, hipStream_t st) {
  typedef Wide<DT, D, QW> K;
  const int grid = (a.nwg ? a.nwg : a.B * a.Hkv) * a.nqb;
  hipLaunchKernelGGL((wide_kernel<DT, D, QW>), dim3(grid), dim3(QW * 64), sizeof(typename K::Shared), st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.nwg == 0) return e;
  const long long rows = (long long)a.B * a.Hkv * a.M;
  hipLaunchKernelGGL((join_kernel<DT, WTILE>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
  return hipGetLastError();
}

template <typename DT, int D>
hipError_t wide_dim(const AttnArgs& a, int qw, hipStream_t st) {
  if (qw == 2) return wide_run<DT, D, 2>(a, st);
  if (qw == 4) return wide_run<DT, D, 4>(a, st);
  if constexpr (D <= 128)
    if (qw == 8) return wide_run<DT, D, 8>(a, st);
  return hipErrorInvalidValue;
}
template <typename DT>
hipError_t wide_type(const AttnArgs& a, int qw, hipStream_t st) {
  switch (a.D) {
    case 64: return wide_dim<DT, 64>(a, qw, st);
    case 96: return wide_dim<DT, 96>(a, qw, st);
    case 128: return wide_dim<DT, 128>(a, qw, st);
    case 256: return wide_dim<DT, 256>(a, qw, st);
  }
  return hipErrorInvalidValue;
}

}  // namespace attn

hipError_t launch_attn_wide(const AttnArgs& a, const AttnPlan& p, int dtype, hipStream_t st) {
  return dtype == TGS_BF16 ? attn::wide_type<attn::BF16>(a, p.qw, st) : attn::wide_type<attn::F16>(a, p.qw, st);
}

AttnPlan attn_plan(int M, int D) {
  AttnPlan p;
  if (M <= 32) {
    p.wide = 0;
    p.qw = M <= 16 ? 1 : 2;
    p.tile = attn::NTILE;
    p.QB = 16 * p.qw;
    p.per_cu = 1;
    p.least = 8;  // one per wave
  } else {
    p.wide = 1;
    p.qw = M <= 64 ? 2 : M <= 128 || D == 256 ? 4 : 8;
    p.tile = attn::WTILE;
    p.QB = 32 * p.qw;
    p.per_cu = D == 256 ? 1 : 8 / p.qw;
    p.least = 4;
  }
  p.nqb = (M + p.QB - 1) / p.QB;
  return p;
}

hipError_t launch_attn(const AttnArgs& a, const AttnPlan& p, int dtype, hipStream_t st) {
  return p.wide ? launch_attn_wide(a, p, dtype, st) : launch_attn_narrow(a, p, dtype, st);
}

hipError_t set_attn_lds_limit(size_t bytes) { return set_attn_narrow_lds(bytes); }

}  // namespace tgs
