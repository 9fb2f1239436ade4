// tgs_beam.hip -- beam search's selection: of a request's W beams over V ids
// each, the n largest of score[w] + x[w][v] - logsumexp(x[w]), and the
// histories that go with them.
//
// One read of the logits bounds it, and the operations on every element next
// to that.  chunk_kernel holds a chunk of a row in registers: thread maxima give
// a bound that a few more than n ids pass (the n-th largest of the maxima),
// vectors whose maximum passes it are searched, and what is found is sorted.
// The sum of exponentials comes from the same registers, each thread's terms
// relative to a power of two of its own, so that no thread waits for the
// chunk's maximum and scaling the sums to a common power is exact.  The terms and
// the sum of a vector's are 32-bit (the logsumexp is right to 2^-21), what is
// summed from them is 64-bit.  Inside a row the order is the logits' own, so it
// needs no arithmetic; join_kernel orders the candidates of different beams by
// totals in 64 bits, so that no further rounding to 32 decides between them.
//
// 32 requests of 8 beams over 128,256 ids, bf16 (66 MB): chunks 28 us, 2.4 TB/s,
// in two rounds of four workgroups a CU that each load, sort and collect in
// turn; join 10 us.  4 beams over 32,000 ids, fp32: 5.4 and 5.8 us, the latency
// of dependent steps.  Joining in the last workgroup to finish, in one launch,
// took 0.5 and 7 us more: it has to wait for its stores to drain first.
#include "tgs_device.h"
#include "tgs_kv.h"
#include "tgs_row.h"

namespace tgs {
namespace beam {

// 2^x by the hardware instruction; results below 2^-126 are 0, next to a sum
// that holds its maximum's own term, 2^-0.5 or more.
__device__ __forceinline__ float exp2_hw(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_exp2f(x);
#else
  return exp2f(x);
#endif
}

struct ChunkShared {
  BlockScratch bs;
  uint32_t top[BEAM_NT / 64][64];
  u64 cand[BEAM_CAP];
  double sum[BEAM_NT / 64];
  float base[BEAM_NT / 64];
  unsigned n;
};

// The vector as a new value to the compiler, in program order: a pass over the
// chunk unpacks it again instead of keeping every id's 32 bits from the pass
// before (which spilled hundreds of registers).
__device__ __forceinline__ uint4 again(uint4 x) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(x.x), "+v"(x.y), "+v"(x.z), "+v"(x.w));
#endif
  return x;
}

constexpr float NEG = -__builtin_inff();
constexpr float NO_BASE = -1e30f;  // (the exponent of a sum of nothing)
constexpr double LN2 = 0.69314718055994530942;

// Logits of a magnitude beyond this (masks by large finite numbers) are far: a
// whole number of 32 bits cannot stand for x log2 e there, or not closely.  A
// wave that holds a far maximum takes its terms as e^(x - maximum) instead, and
// its sum is handed on negative, with the maximum in the exponent's place.
constexpr float FAR = 4194304.0f;

// x 2^e for a whole e <= 0; 0 far below.
__device__ __forceinline__ double scaled(double x, float e) { return __builtin_ldexp(x, (int)fmaxf(e, -4000.0f)); }

// The natural logarithm of a sum and its base as they are handed on.
__device__ __forceinline__ double log_sum(double base, double sum) {
  return (sum < 0.0 ? base : base * LN2) + log(__builtin_fabs(sum));
}

// Workgroup (row, chunk): ids [c L, min(V, (c + 1) L)), NVT vectors a thread.
template <typename Tin, int NVT>
__global__ __launch_bounds__(BEAM_NT, 4) void chunk_kernel(BeamArgs a) {
  constexpr int EPV = Elem<Tin>::EPV;
  TGS_STATIC_SMEM(ChunkShared, s);
  const int row = blockIdx.x / a.S, c = blockIdx.x % a.S, tid = threadIdx.x, w = tid >> 6;
  const Tin* rowp = (const Tin*)a.logits + (long long)row * a.row_stride;
  const int v0 = c * a.L, v1 = v0 + a.L < a.V ? v0 + a.L : a.V;
  const int nvec = (v1 - v0) / EPV, tail0 = v0 + nvec * EPV;
  constexpr uint32_t NB = sizeof(Tin) == 2 ? 0xFF80FF80u : 0xFF800000u;  // -inf
  uint4 raw[NVT];
#pragma unroll
  for (int j = 0; j < NVT; j++) {
    const int i = j * BEAM_NT + tid;
    raw[j] = make_uint4(NB, NB, NB, NB);
    if (i < nvec) raw[j] = load_row16<true>(rowp + v0 + i * EPV);
  }
  // the last ids of a row that is not whole vectors, one a thread
  const float xt = tid < v1 - tail0 ? Elem<Tin>::scalar(rowp, tail0 + tid) : NEG;
  if (tid == 0) s.n = 0;
  float tm = fmaxf(xt, NEG), vm[NVT];  // (of a NaN and a number the number)
#pragma unroll
  for (int j = 0; j < NVT; j++) {
    vm[j] = NEG;
#pragma unroll
    for (int e = 0; e < EPV; e++) vm[j] = fmaxf(vm[j], Elem<Tin>::get(raw[j], e));
    tm = fmaxf(tm, vm[j]);
  }
  const uint32_t mine = wave_sort_desc(tg_key(tm));
  s.top[w][lane_id()] = mine;
  // Terms 2^(x log2 e - base), the constant in two parts, base the whole
  // number at the thread's maximum.
  constexpr float L2H = 0x1.715476p+0f, L2L = 0x1.4ae0cp-26f;
  const bool some = tm > NEG && tm < -NEG;
  float base = some ? __builtin_rintf(tm * L2H) : 0.0f;
  auto term = [&](float x) { return exp2_hw(__builtin_fmaf(x, L2L, __builtin_fmaf(x, L2H, -base))); };
  double sum = (double)term(xt);
#pragma unroll
  for (int j = 0; j < NVT; j++) {
    raw[j] = again(raw[j]);
    float part = 0.0f;  // (of one vector's terms)
#pragma unroll
    for (int e = 0; e < EPV; e++) part += term(Elem<Tin>::get(raw[j], e));
    sum += (double)part;
  }
  auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < NVT; j++) {
      raw[j] = again(raw[j]);
#pragma unroll
      for (int e = 0; e < EPV; e++) f(Elem<Tin>::get(raw[j], e), v0 + (j * BEAM_NT + tid) * EPV + e);
    }
    f(xt, tail0 + tid);
  };
  if (sum != sum) {  // NaN logits count as -inf (+inf ones leave an infinite sum)
    sum = 0.0;
    each([&](float x, int) { sum += x > NEG ? (double)term(x) : 0.0; });
  }
  if (sum == 0.0) base = NO_BASE;
  float wbase = wave_maxf(base);
  bool far = false;
  if (__ballot(some && fabsf(tm) > FAR)) {
    wbase = wave_maxf(tm);
    far = fabsf(wbase) > FAR && wbase < -NEG;
    base = far ? wbase : __builtin_rintf(wbase * L2H);
    sum = 0.0;
    each([&](float x, int) {
      if (x > NEG) sum += (double)(far ? exp2_hw((x - base) * L2H) : term(x));
    });
    wbase = base;
  }
  sum = scaled(sum, base - wbase);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (lane_id() == 0) {
    s.base[w] = wbase;
    s.sum[w] = far ? -sum : sum;
  }
  __syncthreads();
  uint32_t top = s.top[0][lane_id()];
#pragma unroll
  for (int i = 1; i < BEAM_NT / 64; i++) top = wave_merge_top64(top, s.top[i][lane_id()]);
  const float bound = tg_unkey(readlane_u32(top, a.n - 1));
  auto keep = [&](float x, int v) {
    if (x >= bound && x > NEG) {
      const unsigned at = atomicAdd(&s.n, 1u);
      if (at < (unsigned)BEAM_CAP) s.cand[at] = comp_key(tg_key(x), v);
    }
  };
  if (tm >= bound) {
#pragma unroll
    for (int j = 0; j < NVT; j++)
      if (vm[j] >= bound) {
        raw[j] = again(raw[j]);
#pragma unroll
        for (int e = 0; e < EPV; e++) keep(Elem<Tin>::get(raw[j], e), v0 + (j * BEAM_NT + tid) * EPV + e);
      }
    keep(xt, tail0 + tid);
  }
  __syncthreads();
  unsigned n = s.n;
  if (n > (unsigned)BEAM_CAP) {  // many equal logits: the exact n-th by its composite
    const u64 least = block_select_kth<u64, 64, BEAM_NT>(
        [&](auto f) {
          each([&](float x, int v) {
            if (x > NEG) f(comp_key(tg_key(x), v));
          });
        },
        (unsigned)a.n, s.bs);
    __syncthreads();
    if (tid == 0) s.n = 0;
    __syncthreads();
    each([&](float x, int v) {
      if (x > NEG && comp_key(tg_key(x), v) >= least) {
        const unsigned at = atomicAdd(&s.n, 1u);
        if (at < (unsigned)BEAM_CAP) s.cand[at] = comp_key(tg_key(x), v);
      }
    });
    __syncthreads();
    n = s.n;
  }
  if (w == 0) {
    const int lane = lane_id();
    u64 best = wave_sort_desc((unsigned)lane < n ? s.cand[lane] : 0ull);
    for (unsigned i = 64; i < n; i += 64)
      best = wave_merge_top64(best, wave_sort_desc(i + lane < n ? s.cand[i + lane] : 0ull));
    if (lane < a.n) a.lists[(long long)blockIdx.x * a.n + lane] = best;
    if (lane == 0) {
      float b = s.base[0];
      bool far = s.sum[0] < 0.0;
#pragma unroll
      for (int i = 1; i < BEAM_NT / 64; i++) {
        b = fmaxf(b, s.base[i]);
        far |= s.sum[i] < 0.0;
      }
      double at = (double)b, t = 0.0;
      if (far) {
        at = -__builtin_inf();
#pragma nounroll
        for (int i = 0; i < BEAM_NT / 64; i++) {
          s.sum[i] = log_sum((double)s.base[i], s.sum[i]);
          at = fmax(at, s.sum[i]);
        }
#pragma nounroll
        for (int i = 0; i < BEAM_NT / 64; i++) t -= exp(s.sum[i] - at);
      } else {
#pragma unroll
        for (int i = 0; i < BEAM_NT / 64; i++) t += scaled(s.sum[i], s.base[i] - b);
      }
      a.sums[2 * (long long)blockIdx.x] = at;
      a.sums[2 * (long long)blockIdx.x + 1] = t;
    }
  }
}

struct JoinShared {
  double total[BEAM_MAX][BEAM_MAX];  // -inf past a beam's candidates
  int id[BEAM_MAX][BEAM_MAX];
  double best[BEAM_MAX];
  int parent[BEAM_MAX], token[BEAM_MAX];
};

// Workgroup per request.  A wave per beam joins its chunks; a candidate's
// place among all is its place in its own sorted list plus, by bisection, the
// number of candidates ahead of it in every other.
constexpr int JOIN_NT = 512;
__global__ __launch_bounds__(JOIN_NT) void join_kernel(BeamArgs a) {
  TGS_STATIC_SMEM(JoinShared, s);
  const int g = blockIdx.x, tid = threadIdx.x, lane = lane_id();
  const int W = a.W, n = a.n;
  const double NINF = -__builtin_inf();
  for (int w = tid >> 6; w < W; w += JOIN_NT / 64) {
    const long long row = (long long)g * W + w;
    const u64* lists = a.lists + row * a.S * n;
    const double* sums = a.sums + row * a.S * 2;
    const float score = a.scores[row];
    const double base = lane < a.S ? sums[2 * lane] : (double)NO_BASE;
    double t = lane < a.S ? sums[2 * lane + 1] : 0.0;
    const int per = 64 / n, li = lane / n;  // lists a batch; the lane's list and entry
    u64 best = 0ull;
    for (int i = 0; i < a.S; i += per) {
      u64 x = li < per && i + li < a.S ? lists[(i + li) * n + lane - li * n] : 0ull;
      if (per > 1) x = wave_sort_desc(x);
      best = i == 0 ? x : wave_merge_top64(best, x);
    }
    double top;
    const bool far = __ballot(t < 0.0) != 0;
    if (far) {
      const double x = log_sum(base, t);
      top = x;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) top = fmax(top, __shfl_xor(top, o, 64));
      t = exp(x - top);
    } else {
      const float m = (float)base, mt = wave_maxf(m);
      t = scaled(t, m - mt);
      top = (double)mt * LN2;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
    const double lse = top + log(t);
    // a beam that has ended (its score not a number above -inf), or whose row
    // holds +inf or nothing, has no candidates
    const bool live = __builtin_isfinite(score) && __builtin_isfinite(lse);
    if (lane < n) {
      const bool has = live && best != 0ull;
      s.total[w][lane] = has ? (double)score + ((double)comp_y(best) - lse) : NINF;
      s.id[w][lane] = has ? comp_id(best) : -1;
    }
  }
  for (int i = tid; i < n; i += JOIN_NT) {
    s.best[i] = NINF;
    s.parent[i] = -1;
    s.token[i] = -1;
  }
  __syncthreads();
  for (int i = tid; i < W * n; i += JOIN_NT) {
    const int w = i / n, j = i - w * n;
    const double x = s.total[w][j];
    if (x == NINF) continue;
    int rank = j;
    for (int o = 0; o < W && rank < n; o++) {
      if (o == w) continue;
      int lo = 0, hi = n;  // entries of o ahead of x; of equal ones the lower beam's
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        const double y = s.total[o][mid];
        if (y > x || (y == x && o < w))
          lo = mid + 1;
        else
          hi = mid;
      }
      rank += lo;
    }
    if (rank < n) {
      s.best[rank] = x;
      s.parent[rank] = g * W + w;
      s.token[rank] = s.id[w][j];
    }
  }
  __syncthreads();
  const long long out = (long long)g * n;
  for (int i = tid; i < n; i += JOIN_NT) {
    a.out_scores[out + i] = (float)s.best[i];
    a.out_parents[out + i] = s.parent[i];
    a.out_tokens[out + i] = s.token[i];
  }
  if (a.H == 0) return;
  for (int r = tid >> 6; r < n; r += JOIN_NT / 64) {
    const int p = s.parent[r], H = a.H;
    int have = p < 0 ? 0 : a.hist_len[p];
    have = have < 0 ? 0 : have > H ? H : have;
    const int drop = have == H, kept = p < 0 ? -1 : have - drop;
    const int* from = a.hist + (long long)(p < 0 ? 0 : p) * H + drop;
    int* to = a.out_hist + (out + r) * H;
    for (int j = lane; j < H; j += 64) to[j] = j < kept ? from[j] : j == kept ? s.token[r] : -1;
    if (lane == 0) a.out_hist_len[out + r] = kept + 1;
  }
}

template <typename Tin>
hipError_t launch_t(const BeamArgs& a, hipStream_t st) {
  const int per = BEAM_NT * Elem<Tin>::EPV;
  const dim3 grid(a.G * a.W * a.S);
  if (a.L <= 4 * per)
    hipLaunchKernelGGL((chunk_kernel<Tin, 4>), grid, dim3(BEAM_NT), 0, st, a);
  else
    hipLaunchKernelGGL((chunk_kernel<Tin, BEAM_NVT>), grid, dim3(BEAM_NT), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(join_kernel, dim3(a.G), dim3(JOIN_NT), 0, st, a);
  return hipGetLastError();
}

}  // namespace beam

int beam_chunk_ids(int dtype) { return BEAM_NT * BEAM_NVT * (dtype == TGS_BF16 ? 8 : 4); }

hipError_t launch_beam(const BeamArgs& a, int dtype, hipStream_t st) {
  return dtype == TGS_BF16 ? beam::launch_t<uint16_t>(a, st) : beam::launch_t<float>(a, st);
}

}  // namespace tgs
