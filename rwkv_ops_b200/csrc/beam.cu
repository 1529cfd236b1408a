// Beam search: the W best continuations of W beams over the vocabulary, in one launch and one pass over the logits.
//
// Per group of W beams with running scores s_i (log-probabilities) and logits x_i[V]:
//   candidate (i, t) has the score s_i + x_i[t] - log sum_u e^{x_i[u]};   the W best, ties to the lowest i V + t.
//
// What bounds it is reading the logits once.  The W best of a row come from its own logits in their own order, so a warp streams
// a slice of a row and keeps, besides the running maximum and sum, the W best of what it has seen, sorted, one to a lane.  After the first
// tiles hardly any element passes the W-th best (W ln(n / W) of n), so that list costs a comparison per element and a shuffle of a few
// instructions now and then.  One cluster of CTAs works on a group; its warps' lists and sums meet in the shared memory of the first CTA, where
// the normalisers are put together and candidates compared in float64: a sum of two float32 would tie where the scores do not.
//
// A beam that has finished goes on with `eos` alone, at the score it has; its logits are not read.  NaN and +inf logits count as -inf (never
// generated), a NaN score as -inf.  Where fewer than W candidates are possible the rest are impossible ones, score -inf, lowest
// indices first.
#include <algorithm>
#include <cfloat>
#include <climits>

#include "common.cuh"
#include "tc.cuh"

namespace rwkvb200 {
namespace {

constexpr int NWARP = 16;      // of a CTA
constexpr int MAXC = 8;        // CTAs of a cluster
constexpr int MAXW = 32;
constexpr float NEG = -INFINITY;

// A list of the best (value, index) of a warp, sorted, entry l in lane l; entries beyond the first `n` lanes do not matter.
template <typename F, typename I>
struct Best {
  static constexpr I NONE = sizeof(I) == 8 ? (I)LLONG_MAX : (I)INT_MAX;
  F v = (F)NEG;
  I i = NONE;
};
typedef Best<float, int> RowBest;              // of a row: its tokens
typedef Best<double, long long> GroupBest;     // of a group: i V + t
template <typename F, typename I>
__device__ __forceinline__ bool before(F v, I i, F v2, I i2) { return v > v2 || (v == v2 && i < i2); }
// (x, j), the same in every lane, into the list
template <typename F, typename I>
__device__ __forceinline__ void insert(Best<F, I>& b, F x, I j, int lane) {
  const int pos = __popc(__ballot_sync(0xffffffffu, before(b.v, b.i, x, j)));
  const F uv = __shfl_up_sync(0xffffffffu, b.v, 1);
  const I ui = __shfl_up_sync(0xffffffffu, b.i, 1);
  if (lane > pos) { b.v = uv; b.i = ui; }
  else if (lane == pos) { b.v = x; b.i = j; }
}
// every lane's (x, j), those that are among the W best, into the list; (wv, wi) is the W-th best
template <typename F, typename I>
__device__ __forceinline__ void offer(Best<F, I>& b, F& wv, I& wi, F x, I j, int W, int lane) {
  uint32_t some = __ballot_sync(0xffffffffu, before(x, j, wv, wi));
  while (some) {
    const int src = __ffs(some) - 1;
    insert(b, __shfl_sync(0xffffffffu, x, src), __shfl_sync(0xffffffffu, j, src), lane);
    wv = __shfl_sync(0xffffffffu, b.v, W - 1);
    wi = __shfl_sync(0xffffffffu, b.i, W - 1);
    some &= some - 1;
    some &= __ballot_sync(0xffffffffu, before(x, j, wv, wi));
  }
}

template <typename F, typename I>
__device__ __forceinline__ void offer(Best<F, I>& b, F x, I j, int W, int lane) {
  F wv = __shfl_sync(0xffffffffu, b.v, W - 1);
  I wi = __shfl_sync(0xffffffffu, b.i, W - 1);
  offer(b, wv, wi, x, j, W, lane);
}

template <typename T> struct Vec { static constexpr int N = 16 / (int)sizeof(T); };
// 16 bytes of logits as floats, those that are NaN or +inf as -inf
__device__ __forceinline__ float clean(float x) { return x <= FLT_MAX ? x : NEG; }
__device__ __forceinline__ void unpack(const uint4& u, float* x, const float*) {
  x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(const uint4& u, float* x, const __nv_bfloat16*) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void unpack(const uint4& u, float* x, const __half*) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x; x[2 * i + 1] = f.y;
  }
}

// Piece p of a row, its elements p N .. p N + N - 1, whatever the row's alignment: every piece is the same elements in every row, so that
// equal rows have equal sums to the last bit.  A row that does not start on 16 bytes (`shift` bytes behind it) has its pieces cut out of two
// aligned ones, the second of which the next lane reads as well (it comes from L1); where these reach over the ends of the row, or the row ends in the
// piece, elements are read one by one.  Elements behind the end are -inf.
template <typename T>
__device__ __forceinline__ void fetch(const T* x, int p, int V, int shift, uint4 (&u)[2]) {
  constexpr int N = Vec<T>::N;
  const int e = p * N - shift / (int)sizeof(T);      // the first element of the aligned piece
  if (shift == 0 ? e + N <= V : e >= 0 && e + 2 * N <= V) {
    u[0] = __ldg(reinterpret_cast<const uint4*>(x + e));
    if (shift) u[1] = __ldg(reinterpret_cast<const uint4*>(x + e) + 1);
  } else {      // (put where align() finds it)
    __align__(16) T t[2 * N];
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) t[i] = e + i >= p * N && e + i < min(V, p * N + N) ? x[e + i] : from_f32<T>(NEG);
    u[0] = *reinterpret_cast<const uint4*>(t);
    u[1] = *reinterpret_cast<const uint4*>(t + N);
  }
}
__device__ __forceinline__ void align(uint4 (&u)[2], int shift) {      // (a warp has one row: no lane takes another way)
  const uint32_t w[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
  auto cut = [&](int i) {
    if (shift & 2) u[0] = make_uint4(__funnelshift_r(w[i], w[i + 1], 16), __funnelshift_r(w[i + 1], w[i + 2], 16),
                                     __funnelshift_r(w[i + 2], w[i + 3], 16), __funnelshift_r(w[i + 3], w[i + 4], 16));
    else u[0] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  };
  switch (shift >> 2) {
    case 1: cut(1); break;
    case 2: cut(2); break;
    case 3: cut(3); break;
    default: cut(0);
  }
}

// Running maximum and sum of a lane, in float32: a lane adds a few hundred terms that are at most one.
struct Sum {
  float m = NEG, s = 0.f;
  template <int N> __device__ __forceinline__ void add(const float (&x)[N], float top) {
    if (top > m) {
      s *= tc::ex2((m - top) * tc::LOG2E);      // (m = -inf: the factor is zero)
      m = top;
    }
    const float base = m == NEG ? 0.f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) s += tc::ex2((x[i] - base) * tc::LOG2E);
  }
};

struct Smem {
  float m[MAXC * NWARP], s[MAXC * NWARP];          // in the first CTA: of every warp of the cluster
  float val[MAXC * NWARP][MAXW];
  int tok[MAXC * NWARP][MAXW];
  double top[MAXW], shift[MAXW];                   // of a row: the maximum; s_i - log (sum relative to it)
  GroupBest best[NWARP][MAXW];
};

template <typename T>
__global__ void __launch_bounds__(NWARP * 32, 2)
beam_select_kernel(const T* __restrict__ logits, long long stride_g, long long stride_w, const float* __restrict__ scores,
                   const uint8_t* __restrict__ finished, long long eos, float* __restrict__ scores_out, long long* __restrict__ parents,
                   long long* __restrict__ tokens, uint8_t* __restrict__ finished_out, int W, int V) {
  extern __shared__ __align__(16) unsigned char raw[];
  Smem& sm = *reinterpret_cast<Smem*>(raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = blockIdx.x, rank = blockIdx.y, n_cta = gridDim.y;
  const int n_warp = n_cta * NWARP, per_row = n_warp / W;      // warps to a row (W <= 32 <= 2 NWARP; one CTA: see the launch)
  const int all = rank * NWARP + warp, row = all / per_row, part = all % per_row;
  earlier_kernels_done();
  later_kernels_may_start();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // (the first CTA has to be there before it is written to)
  RowBest best;      // of this warp's slice
  Sum sum;
  const bool works = row < W;
  const bool done = works && finished && finished[(long long)g * W + row];
  if (works && !done) {
    constexpr int N = Vec<T>::N, U = 16 / N;      // 16 elements of a lane at a time, in pieces of 16 bytes
    const T* x = logits + g * stride_g + row * stride_w;
    const int shift = (int)(reinterpret_cast<uintptr_t>(x) & 15);
    const int n_piece = (V + N - 1) / N;
    const int lo = (int)((long long)n_piece * part / per_row), hi = (int)((long long)n_piece * (part + 1) / per_row);
    float wv = NEG;      // the W-th best
    int wi = RowBest::NONE;
    for (int p = lo + lane; p - lane < hi; p += 32 * U) {
      uint4 u4[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u) fetch(x, p + 32 * u < hi ? p + 32 * u : n_piece, V, shift, u4[u]);
      float f[16];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        align(u4[u], shift);
        unpack(u4[u][0], f + u * N, (const T*)nullptr);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] = clean(f[i]);
      float top = f[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, f[i]);
      sum.add(f, top);
      if (__any_sync(0xffffffffu, before(top, p * N, wv, wi))) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int q = p + 32 * (i / N), j = q * N + i % N;
          offer(best, wv, wi, f[i], q < hi && j < V ? j : RowBest::NONE, W, lane);
        }
      }
    }
  }
  // the warp's sum, relative to its maximum
  float m = sum.m;
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  float s = sum.m == NEG ? 0.f : sum.s * tc::ex2((sum.m - m) * tc::LOG2E);
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  const uint32_t home = tc::cluster_addr(tc::smem_u32(&sm), 0);
  auto put = [&](const void* p, int bits) { tc::store_cluster(home + (tc::smem_u32(p) - tc::smem_u32(&sm)), bits); };
  if (lane == 0) { put(&sm.m[all], __float_as_int(m)); put(&sm.s[all], __float_as_int(s)); }
  if (lane < W) { put(&sm.val[all][lane], __float_as_int(best.v)); put(&sm.tok[all][lane], best.i == RowBest::NONE ? -1 : best.i); }
  tc::cluster_sync();
  if (rank) return;

  for (int i = warp; i < W; i += NWARP) {
    const float score = scores[(long long)g * W + i];
    double mm = NEG, ss = 0.0;
    for (int q = lane; q < per_row; q += 32) mm = fmax(mm, (double)sm.m[i * per_row + q]);
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) mm = fmax(mm, __shfl_xor_sync(0xffffffffu, mm, d));
    for (int q = lane; q < per_row; q += 32) {
      const float mq = sm.m[i * per_row + q];
      if (mq != NEG) ss += (double)sm.s[i * per_row + q] * exp((double)mq - mm);
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
    // (a row without a possible token: every candidate is -inf)
    if (lane == 0) {      // (the maximum apart: only differences of logits count, however large these are)
      sm.top[i] = mm;
      sm.shift[i] = score != score ? (double)NEG : ss > 0.0 ? (double)score - log(ss) : (double)NEG;
    }
  }
  __syncthreads();
  GroupBest b;
  auto offer_row = [&](int i, float x, long long t) {      // t < 0: nothing
    const double sc = x == NEG ? (double)NEG : sm.shift[i] + ((double)x - sm.top[i]);
    offer(b, t < 0 ? (double)NEG : sc, t < 0 ? GroupBest::NONE : (long long)i * V + t, W, lane);
  };
  for (int q = warp; q < W * per_row; q += NWARP) {
    const int i = q / per_row;
    if (finished && finished[(long long)g * W + i]) {
      if (q % per_row == 0) {      // eos at the beam's score, and (impossible) tokens from the first one on
        const float score = scores[(long long)g * W + i];
        long long t = lane == 0 ? eos : lane - 1 < eos ? lane - 1 : lane;
        if (t >= V) t = -1;
        offer(b, lane == 0 && score == score ? (double)score : (double)NEG, t < 0 ? GroupBest::NONE : (long long)i * V + t, W, lane);
        if (W == 32) offer(b, (double)NEG, lane == 0 && eos >= 32 && 31 < V ? (long long)i * V + 31 : GroupBest::NONE, W, lane);
      }
      continue;
    }
    offer_row(i, lane < W ? sm.val[q][lane] : NEG, lane < W ? sm.tok[q][lane] : -1);
  }
  sm.best[warp][lane] = b;
  __syncthreads();
  if (warp) return;
  for (int q = 1; q < NWARP; ++q) {
    const GroupBest c = sm.best[q][lane];
    offer(b, lane < W ? c.v : (double)NEG, lane < W ? c.i : GroupBest::NONE, W, lane);
  }
  if (lane < W) {
    const long long at = (long long)g * W + lane, parent = b.i / V, t = b.i - parent * V;
    scores_out[at] = (float)b.v;
    parents[at] = parent;
    tokens[at] = t;
    if (finished_out) finished_out[at] = (finished && finished[(long long)g * W + parent]) || t == eos;
  }
}

template <typename T>
int select(const void* logits, long long sg, long long sw, const float* scores, const uint8_t* finished, long long eos, float* scores_out,
           long long* parents, long long* tokens, uint8_t* finished_out, int G, int W, int V, cudaStream_t st) {
  DeviceFacts f;
  if (int e = device_facts(&f)) return e;
  constexpr int smem = (int)sizeof(Smem);
  if (int e = allow_smem<beam_select_kernel<T>>(f, smem)) return e;
  // CTAs to a group: eight while they all find room beside each other (two to an SM), fewer as the groups are more; enough warps for the
  // beams, and no more CTAs than there are pieces of a few tiles to work on
  int c = MAXC;
  while (c > 1 && (long long)G * c > 2 * f.sms) c >>= 1;
  while (c > 1 && (long long)W * V < (long long)c * NWARP * 256) c >>= 1;
  while (c * NWARP < W) c <<= 1;
  return launch(beam_select_kernel<T>, dim3(G, c), NWARP * 32, smem, st, c == 1 ? 1 : c, (const T*)logits, sg, sw, scores, finished, eos, scores_out,
                parents, tokens, finished_out, W, V);
}

}  // namespace

int launch_beam_select(const void* logits, int dtype, long long sg, long long sw, const float* scores, const uint8_t* finished, long long eos,
                       float* scores_out, long long* parents, long long* tokens, uint8_t* finished_out, int G, int W, int V, cudaStream_t st) {
  ProfScope prof("beam_select_kernel", st);
  RWKVB200_DISPATCH_DTYPE(dtype, return select<T>(logits, sg, sw, scores, finished, eos, scores_out, parents, tokens, finished_out, G, W, V, st));
  return RWKVB200_OK;
}

}  // namespace rwkvb200
