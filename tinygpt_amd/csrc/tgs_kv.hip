// tgs_kv.hip -- the paged key/value cache's writes and forks.
//
// Layout of a layer: keys [page][kv_head][token][D], values
// [page][kv_head][token / 8][D][8]: the eight tokens of a block lie next to
// each other for each d, which is the operand order of the attention's second
// product.  No arithmetic: every kernel here moves 16-bit values and is bound
// by bytes, or by latency for single tokens; appended keys may turn by their
// positions on the way, in floats.  Measured: prompts of 300 to 2048 tokens, 16
// layers, 175 us (923 MB, 5.3 TB/s read and written); pages of 128 forked beams 83 us
// (403 MB, 4.9 TB/s), of an 8-bit cache 51 us (220 MB, 4.3 TB/s).
#include "tgs_device.h"
#include "tgs_e8.h"
#include "tgs_kv.h"
#include "tgs_kv_write.h"
#include "tgs_row.h"

namespace tgs {
namespace kv {

// ROT: void, or the type of the keys that are turned.
template <class ROT>
struct WriteShared {
  alignas(16) e8::Turn cs[8][ROTARY_MAX / 2];
  WriteHead head;
};
template <>
struct WriteShared<void> {
  WriteHead head;
};

// Workgroup (x, sequence b, layer l) over the 8-token blocks x, x + nblk, ...
// of the positions that b's new rows take.  Keys move as 16-byte vectors.  A
// whole block of values is transposed in registers: a thread takes two
// neighbouring d of the eight tokens (a wave reads 256 contiguous bytes per
// token) and stores 32 contiguous bytes.
// A block that the rows cover in part is read, filled in and written whole: 16
// bytes a d instead of 2-byte stores 16 bytes apart, of which every one costs
// the cache a line (64 trees of 63 nodes, 32 layers: 45 us, was 59).
// Keys that turn (ROT) go by units of two chunks, with the cosines and sines of the
// block's positions in LDS.
template <bool COMMIT, class ROT>
__global__ __launch_bounds__(KV_NT) void write_kernel(KvWriteArgs a) {
  TGS_STATIC_SMEM(WriteShared<ROT>, sh);
  WriteHead& s = sh.head;
  const int x = blockIdx.x % a.nblk, bl = blockIdx.x / a.nblk, b = bl % a.B, l = bl / a.B;
  const int tid = threadIdx.x;
  const int len = a.lens[b], n = rows_of<COMMIT>(a, s, b);
  const int* table = a.tables + (long long)b * a.P;
  int bad = past_table(a, len, n);
  if (!bad) bad = outside_pool(a, table, len, n);
  bad = __syncthreads_or(bad);
  if (l == 0 && x == 0) report<COMMIT>(a, s, b, len, n, bad);
  if (bad || n == 0) return;
  const int D = a.c.head_dim, H = a.c.kv_heads, page = 1 << a.page_shift;
  const uint16_t* kn = (const uint16_t*)a.r.k + l * a.r.k_layer + b * a.r.k_seq;
  const uint16_t* vn = (const uint16_t*)a.r.v + l * a.r.v_layer + b * a.r.v_seq;
  const int last = (len + n - 1) >> 3;
  for (int blk = (len >> 3) + x; blk <= last; blk += a.nblk) {
    const int pos0 = blk << 3;
    const int t0 = pos0 > len ? pos0 : len, t1 = pos0 + 8 < len + n ? pos0 + 8 : len + n;  // positions written
    const int nt = t1 - t0;
    const long long pg = table[pos0 >> a.page_shift];
    uint16_t* kp = (uint16_t*)a.c.k + l * a.c.k_layer + pg * a.c.k_page + (long long)(t0 & (page - 1)) * D;
    uint16_t* vp = (uint16_t*)a.c.v + l * a.c.v_layer + pg * a.c.v_page + (long long)(pos0 & (page - 1)) * D;
    const int C = D >> 3;
    if constexpr (!__is_same(ROT, void)) {
      const int half = a.rot.dims >> 1, U = e8::units(D);
      __syncthreads();  // (the block before is done with the table)
      for (int e = tid; e < nt * half; e += KV_NT) {
        const int i = div_by((unsigned)e, a.turns), j = e - i * half;
        sh.cs[i][j] = e8::turn((uint32_t)(t0 + i), a.rot.freq[j]);
      }
      __syncthreads();
      for (int e = tid; e < nt * H * U; e += KV_NT) {  // (token, head, unit)
        const unsigned row = div_by((unsigned)e, a.units), u = (unsigned)e - row * U;
        const int i = div_by(row, a.heads), h = row - i * H;
        const uint16_t* from = kn + (t0 - len + i) * a.r.k_tok + h * a.r.k_head;
        uint16_t* to = kp + ((long long)h * page + i) * D;
        const e8::Unit w = e8::unit_of((int)u, D, a.rot.dims, a.rot.pairs);
        const uint4 lo = load_row16<false>(from + w.a), hi = w.b >= 0 ? load_row16<false>(from + w.b) : lo;
        uint32_t y[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        if (w.angle >= 0) e8::turn_words<ROT>(y, sh.cs[i] + w.angle, a.rot.pairs);
        *(uint4*)(to + w.a) = make_uint4(y[0], y[1], y[2], y[3]);
        if (w.b >= 0) *(uint4*)(to + w.b) = make_uint4(y[4], y[5], y[6], y[7]);
      }
    } else
    for (int e = tid; e < nt * H * C; e += KV_NT) {  // 16-byte vectors of keys: (token, head, chunk)
      const unsigned row = div_by((unsigned)e, a.chunks), ch = (unsigned)e - row * C;
      const int i = div_by(row, a.heads), h = row - i * H;
      const int node = COMMIT ? s.path[t0 - len + i] : t0 - len + i;
      const uint4 x = load_row16<false>(kn + node * a.r.k_tok + h * a.r.k_head + ch * 8);
      *(uint4*)(kp + ((long long)h * page + i) * D + ch * 8) = x;
    }
    const int D2 = D >> 1;
    for (int e = tid; e < H * D2; e += KV_NT) {  // pairs of d: (head, d / 2)
      const unsigned h = div_by((unsigned)e, a.half_d), d = 2 * ((unsigned)e - h * D2);
      uint16_t* to = vp + (long long)h * page * D + d * 8;
      uint32_t x[8];
      auto take = [&](int i) {  // token pos0 + i
        const int j = pos0 + i - len;
        const uint16_t* p = vn + (COMMIT ? s.path[j] : j) * a.r.v_tok + h * a.r.v_head + d;
        __builtin_memcpy(&x[i], p, 4);
      };
      uint4 lo, hi;
      if (nt == 8) {
#pragma unroll
        for (int i = 0; i < 8; i++) take(i);
        auto word = [&](int i, uint32_t& l0, uint32_t& h0) {
          l0 = (x[i] & 0xFFFFu) | (x[i + 1] << 16);
          h0 = (x[i] >> 16) | (x[i + 1] & 0xFFFF0000u);
        };
        word(0, lo.x, hi.x);
        word(2, lo.y, hi.y);
        word(4, lo.z, hi.z);
        word(6, lo.w, hi.w);
      } else {
        lo = *(const uint4*)to;
        hi = *(const uint4*)(to + 8);
        const int at = t0 & 7;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          x[i] = 0;
          if (i >= at && i < at + nt) take(i);
        }
        auto word = [&](int i, uint32_t& l0, uint32_t& h0) {
          const uint32_t m = (i >= at && i < at + nt ? 0xFFFFu : 0u) | (i + 1 >= at && i + 1 < at + nt ? 0xFFFF0000u : 0u);
          l0 = (l0 & ~m) | (((x[i] & 0xFFFFu) | (x[i + 1] << 16)) & m);
          h0 = (h0 & ~m) | (((x[i] >> 16) | (x[i + 1] & 0xFFFF0000u)) & m);
        };
        word(0, lo.x, hi.x);
        word(2, lo.y, hi.y);
        word(4, lo.z, hi.z);
        word(6, lo.w, hi.w);
      }
      *(uint4*)to = lo;
      *(uint4*)(to + 8) = hi;
    }
  }
}

// ------------------------------------------------------------------ fork
//
// Row r of the new tables continues row parents[r]: it shares the pages that
// are full; from the page that its next token goes to on, every page has one
// writer.  A page that no row holds in full stays with the first row (in row,
// then slot order) that names it there; the others get free pages, handed out
// in ascending order to rows and slots in order, and copy what their parent's
// page holds.  A page is free when no new row names it.  Where they are too few,
// a row gets all that it needs or none, and the rows behind it what is left.  A
// row with tokens in a slot that names no page of the pool is given none.

constexpr int OWNER_FREE = 0x7FFFFFFF;  // else the first row * P + slot that writes to the page, or -1: shared

template <bool LDS>
__device__ __forceinline__ int owner_get(const int* o, int p) {
  if constexpr (LDS) return o[p];
  return __hip_atomic_load(o + p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct PlanShared {
  int wave[KV_PLAN_NT / 64];
  int at[KV_PLAN_NT];  // whether rows are bad (LDS), their needs, the first free page of each (-1: too few left)
  int given;
  int4 copy;
};

// Exclusive sum of x over the workgroup, and the total.
__device__ __forceinline__ int block_excl(int x, PlanShared& s, int& total) {
  const int w = threadIdx.x >> 6;
  const int incl = wave_incl_scan(x);
  __syncthreads();
  if (lane_id() == 63) s.wave[w] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < KV_PLAN_NT / 64; i++) {
    if (i < w) before += s.wave[i];
    total += s.wave[i];
  }
  return before + incl - x;
}

// A new row: its parent, length and slots: shared [0, full), its own [full, end).
// Without a parent (par -1) or of one whose length is none it has no slots, and
// the length 0 or -1.
struct ForkRow {
  int par, len, full, end;
};
__device__ __forceinline__ ForkRow fork_row(const KvForkArgs& a, int par, int len) {
  const long long cap = (long long)a.P << a.page_shift;
  if ((unsigned)par >= (unsigned)a.R) return ForkRow{-1, 0, 0, 0};
  if (len < 0 || len > cap) return ForkRow{-1, -1, 0, 0};
  const long long end = ((long long)len + a.room + (1 << a.page_shift) - 1) >> a.page_shift;
  return ForkRow{par, len, len >> a.page_shift, end < a.P ? (int)end : a.P};
}

// One workgroup plans the fork: owners of the pages, the free list, the new
// tables and the copies (with `out`; else only row `want`'s copy, to s.copy).
// LDS: the rows (at most one a thread), owners and free list lie there.
template <bool LDS>
__device__ __forceinline__ void plan(const KvForkArgs& a, PlanShared& s, unsigned char* dyn, bool out, int want) {
  const int tid = threadIdx.x, N = a.c.n_pages, P = a.P;
  int* owner = LDS ? (int*)dyn : a.owner;
  int* fresh = LDS ? owner + N : a.fresh;
  int2* rows = (int2*)(owner + 2 * (LDS ? N : 0));
  auto load_row = [&](int r) {
    const int par = a.parents[r];
    return make_int2(par, (unsigned)par < (unsigned)a.R ? a.lens[par] : -1);
  };
  auto row_of = [&](int r) {
    const int2 x = LDS ? rows[r] : load_row(r);
    return fork_row(a, x.x, x.y);
  };
  // whether rows are bad: few are, so that only those mark themselves
  auto bad_row = [&](int r) -> int& {
    if constexpr (LDS) return s.at[r];
    else return a.copies[r].w;
  };
  if (LDS && tid < a.R) rows[tid] = load_row(tid);
  for (int r = tid; r < a.R; r += KV_PLAN_NT) bad_row(r) = 0;
  for (int i = tid; i < N; i += KV_PLAN_NT) owner[i] = OWNER_FREE;
  if (!LDS) __threadfence();
  __syncthreads();
  for (int r = tid >> 6; r < a.R; r += KV_PLAN_NT / 64) {
    const ForkRow w = row_of(r);
    const int* t = a.tables + (long long)(w.par < 0 ? 0 : w.par) * P;
    for (int i = lane_id(); i < w.end; i += 64) {
      const int p = t[i];
      if ((unsigned)p < (unsigned)N)
        atomicMin(&owner[p], i < w.full ? -1 : r * P + i);
      else if ((long long)i << a.page_shift < w.len)
        bad_row(r) = 1;
      if (out && i < w.full) a.tables_out[(long long)r * P + i] = p;
    }
  }
  if (!LDS) __threadfence();
  __syncthreads();
  // the free pages in ascending order
  const int per = (N + KV_PLAN_NT - 1) / KV_PLAN_NT;
  const int n0 = tid * per < N ? tid * per : N, n1 = n0 + per < N ? n0 + per : N;
  int mine = 0;
  for (int i = n0; i < n1; i++) mine += owner_get<LDS>(owner, i) == OWNER_FREE;
  int n_free;
  int at = block_excl(mine, s, n_free);
  for (int i = n0; i < n1; i++)
    if (owner_get<LDS>(owner, i) == OWNER_FREE) fresh[at++] = i;
  if (!LDS) __threadfence();
  __syncthreads();
  int base = 0;
  for (int r0 = 0; r0 < a.R; r0 += KV_PLAN_NT) {
    const int r = r0 + tid;
    const ForkRow w = r < a.R ? row_of(r) : ForkRow{-1, 0, 0, 0};
    const int* t = a.tables + (long long)(w.par < 0 ? 0 : w.par) * P;
    const bool bad = r < a.R && bad_row(r);
    int need = 0;
    for (int i = w.full; i < w.end && !bad; i++) {
      const int p = t[i];
      need += !((unsigned)p < (unsigned)N && owner_get<LDS>(owner, p) == r * P + i);
    }
    int total;
    int next = base + block_excl(need, s, total);
    if (total <= n_free - base) {
      base += total;
    } else {
      s.at[tid] = need;
      __syncthreads();
      if (tid == 0) {
        for (int i = 0; i < KV_PLAN_NT; i++) {
          const int x = s.at[i];
          s.at[i] = x <= n_free - base ? base : -1;
          if (x <= n_free - base) base += x;
        }
        s.given = base;
      }
      __syncthreads();
      next = s.at[tid];
      base = s.given;
    }
    if (r >= a.R) continue;
    const bool fits = next >= 0 && !bad;
    int* to_row = a.tables_out + (long long)r * P;
    int4 copy = make_int4(-1, -1, 0, 0);
    for (int i = w.full; i < w.end; i++) {
      const int p = t[i];
      int to = p;
      if (!((unsigned)p < (unsigned)N && owner_get<LDS>(owner, p) == r * P + i)) {
        to = fits ? fresh[next++] : -1;
        const int held = w.len - (i << a.page_shift);
        if (held > 0 && fits) copy = make_int4(p, to, a.scales ? (held + e8::BLOCK - 1) / e8::BLOCK : (held + 7) >> 3, 0);
      }
      if (out) to_row[i] = to;
    }
    if (r == want) s.copy = copy;
    if (!out) continue;
    if (want < 0) a.copies[r] = copy;
    // -1: the pool ran out of pages, or the row is bad
    a.lens_out[r] = w.par < 0 ? w.len : fits && (long long)w.len + a.room <= ((long long)P << a.page_shift) ? w.len : -1;
  }
  if (!out) return;
  for (int r = tid >> 6; r < a.R; r += KV_PLAN_NT / 64) {
    const ForkRow w = row_of(r);
    for (int i = w.end + lane_id(); i < P; i += 64) a.tables_out[(long long)r * P + i] = -1;
  }
}

// The blocks of row r's page that are in use lie contiguous per head: copies
// those of layer y / 2, keys or values (and with them their scales).  A block's
// vectors of 16 bytes are as many as a head has dimensions, of 8 tokens in 16
// bits or of 16 in 8 (E8).
template <bool E8>
__device__ __forceinline__ void copy_page(const KvForkArgs& a, const int4& c, int y) {
  if (c.z == 0) return;
  const int l = y >> 1, D = a.c.head_dim, H = a.c.kv_heads;
  const bool val = y & 1;
  constexpr int BYTES = E8 ? 1 : 2, PER = E8 ? e8::BLOCK : 8;
  unsigned char* pool = (unsigned char*)(val ? a.c.v : a.c.k) + l * (val ? a.c.v_layer : a.c.k_layer) * BYTES;
  const long long ps = (val ? a.c.v_page : a.c.k_page) * BYTES;
  const uint4* from = (const uint4*)(pool + c.x * ps);
  uint4* to = (uint4*)(pool + c.y * ps);
  const int n = c.z * D;  // vectors of a head's blocks
  const int hs = (D << a.page_shift) / PER;  // and of its page
  // A wave a head, so that every thread has work where a head's blocks are few.
  // (Non-temporal stores leave the memory-side cache to the pages that are copied, where
  // it still has them: 83 us where plain ones take 100, an 8-bit cache's 51 : 60, and
  // where it does not 60 : 61.  One vector at a time 66, loads that are non-temporal too
  // 65.)
  for (int h = threadIdx.x >> 6; h < H; h += blockDim.x >> 6) {
    for (int i0 = 0; i0 < n; i0 += 256) {  // (four on their way)
      const int i = i0 + lane_id();
      uint4 x[4];
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (i + 64 * j < n) x[j] = from[(long long)h * hs + i + 64 * j];
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (i + 64 * j < n) tg_store_nt(to + (long long)h * hs + i + 64 * j, x[j]);
    }
    if constexpr (E8) {
      uint8_t* scales = a.scales + l * a.s_layer + ((h << a.page_shift) / PER) * 2 + val;
      for (int i = lane_id(); i < c.z; i += 64) scales[c.y * a.s_page + 2 * i] = scales[c.x * a.s_page + 2 * i];
    }
  }
}

template <bool LDS>
__global__ __launch_bounds__(KV_PLAN_NT) void plan_kernel(KvForkArgs a) {
  TGS_STATIC_SMEM(PlanShared, s);
  TGS_DYN_SMEM(dyn);
  plan<LDS>(a, s, dyn, true, -1);
}

// Workgroup (row, layer and pool).
template <bool E8>
__global__ __launch_bounds__(KV_NT) void copy_kernel(KvForkArgs a) {
  copy_page<E8>(a, a.copies[blockIdx.x], blockIdx.y);
}

// Both in one launch, every workgroup planning for itself: where no more than
// a workgroup a CU copies, planning 256 times at once costs less than a second
// launch (4 beams of 530 tokens, 16 layers: kernels of 12 us in two, 5.8 in one).
template <bool E8>
__global__ __launch_bounds__(KV_PLAN_NT) void fork_kernel(KvForkArgs a) {
  TGS_STATIC_SMEM(PlanShared, s);
  TGS_DYN_SMEM(dyn);
  plan<true>(a, s, dyn, blockIdx.x == 0 && blockIdx.y == 0, blockIdx.x);
  __syncthreads();
  copy_page<E8>(a, s.copy, blockIdx.y);
}

}  // namespace kv

hipError_t launch_kv_append(const KvWriteArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((kv::write_kernel<false, void>), dim3(a.nblk * a.B * a.c.layers), dim3(KV_NT), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_kv_append_rotated(const KvWriteArgs& a, hipStream_t st) {
  const dim3 grid(a.nblk * a.B * a.c.layers);
  if (a.c.dtype == TGS_BF16)
    hipLaunchKernelGGL((kv::write_kernel<false, e8::BF16>), grid, dim3(KV_NT), 0, st, a);
  else
    hipLaunchKernelGGL((kv::write_kernel<false, e8::F16>), grid, dim3(KV_NT), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_tree_commit(const KvWriteArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((kv::write_kernel<true, void>), dim3(a.nblk * a.B * a.c.layers), dim3(KV_NT), 0, st, a);
  return hipGetLastError();
}

constexpr size_t FORK_LDS = 128 * 1024;  // of the planning workgroup at most
size_t kv_fork_lds(int n_pages, int rows) {
  const size_t n = (size_t)n_pages * 8 + 16 + (size_t)rows * 8;
  return rows <= KV_PLAN_NT && n <= FORK_LDS ? n : 0;
}

hipError_t launch_kv_fork(const KvForkArgs& a, int num_cu, hipStream_t st) {
  const size_t lds = kv_fork_lds(a.c.n_pages, a.R);
  if (lds && (long long)a.R * 2 * a.c.layers <= num_cu) {
    const dim3 grid(a.R, 2 * a.c.layers);
    if (a.scales)
      hipLaunchKernelGGL(kv::fork_kernel<true>, grid, dim3(KV_PLAN_NT), lds, st, a);
    else
      hipLaunchKernelGGL(kv::fork_kernel<false>, grid, dim3(KV_PLAN_NT), lds, st, a);
    return hipGetLastError();
  }
  if (lds)
    hipLaunchKernelGGL(kv::plan_kernel<true>, dim3(1), dim3(KV_PLAN_NT), lds, st, a);
  else
    hipLaunchKernelGGL(kv::plan_kernel<false>, dim3(1), dim3(KV_PLAN_NT), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (a.scales)
    hipLaunchKernelGGL(kv::copy_kernel<true>, dim3(a.R, 2 * a.c.layers), dim3(KV_NT), 0, st, a);
  else
    hipLaunchKernelGGL(kv::copy_kernel<false>, dim3(a.R, 2 * a.c.layers), dim3(KV_NT), 0, st, a);
  return hipGetLastError();
}

hipError_t set_kv_fork_lds_limit(size_t bytes) {
  const int n = (int)(bytes < FORK_LDS ? bytes : FORK_LDS);
  for (const void* f : {(const void*)kv::plan_kernel<true>, (const void*)kv::fork_kernel<false>, (const void*)kv::fork_kernel<true>}) {
    const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, n);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace tgs
