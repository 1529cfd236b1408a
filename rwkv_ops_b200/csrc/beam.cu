// Beam search: the W best continuations of W beams over the vocabulary, in one launch and one pass over the logits.
//
// Per group of W beams with running scores s_i (log-probabilities) and logits x_i[V]:
//   candidate (i, t) has the score s_i + x_i[t] - log sum_u e^{x_i[u]};   the W best, ties to the lowest i, then to the larger logit, then to the lowest t.
//
// What bounds it is reading the logits once.  The W best of a row come from its own logits in their own order.  A warp streams a slice of a row and
// keeps, for each lane, the running maximum, the tile it is in, the largest of the other tiles and the running sum: some 250 instructions for 512 tokens, where
// sorted lists kept on the way took three times that in time.  The W-th largest of the lanes' maxima is at most the W-th best of the row, so only the lanes that
// reach it have any of the W best: a few of the row's lanes, of which 16 tokens each (all, where another tile reaches it, too) are read once more, from L2, and
// offered to a list.  One cluster of CTAs works on a group; its warps' lists and sums meet in the shared memory of the first CTA, where the normalisers are put
// together and candidates compared in float64: a sum of two float32 would tie where the scores do not.
// What runs once is kept short in code: it is fetched while everyone waits for it.
// Measured: 64 groups of 8 beams over 50277 float32 logits 35 us, 2.9 TB/s: the stream near memory's rate, then second look, lists and merging, one after the other,
// each a wait on shared memory or L2 (issue slots 64 %, most stalls at barriers).  With 95 % of the tokens at -inf 33 us; where fewer tokens than beams are possible, or all
// logits are equal, every lane reaches the bound and all tokens are read once more, a lane's at a time: 141 us.  One group of 4 beams over 65536 bfloat16 logits 12.9 us with the call.
//
// A beam that has finished goes on with `eos` alone, at the score it has; its logits are not read.  NaN and +inf logits count as -inf (never
// generated), a NaN score as -inf.  Where fewer than W candidates are possible the rest are impossible ones, score -inf, lowest
// indices first.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "tc.cuh"

namespace rwkvb200 {
namespace {

constexpr int NWARP = 16;      // of a CTA
constexpr int MAXC = 8;        // CTAs of a cluster
constexpr int MAXW = 32;
constexpr float NEG = -INFINITY;
constexpr float LN2 = 0.6931471805599453f, LOG2E_LO = (float)(1.4426950408889634 - (double)tc::LOG2E);

// A list of the best (value, index) of a warp, sorted, entry l in lane l; entries beyond the first `n` lanes do not matter.
template <typename F, typename I>
struct Best {
  static constexpr I NONE = (I)INT_MAX;
  F v = (F)NEG;
  I i = NONE;
};
typedef Best<float, int> RowBest;              // of a row: its tokens
constexpr int NO_ORDER = INT_MAX;              // of a group's candidates
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

// Logits as floats, those that are NaN or +inf as -inf.
__device__ __forceinline__ float clean(float x) { return x <= FLT_MAX ? x : NEG; }

// A tile: 512 tokens of a row, 16 to a lane, in words of 4 bytes that lie next to each other across the lanes: nothing but the element's own alignment is asked
// of a row (and not even a word's of 16-bit rows of odd length), and every tile is the same tokens of the same lanes in every row, so that equal rows have
// equal sums to the last bit.
constexpr int TILE = 512;
template <typename T>
struct Tile {
  static constexpr int PER = 4 / (int)sizeof(T), N = 16 / PER;      // elements of a word, words of a lane
  uint32_t w[N];
  // the token of element i of a lane
  static __device__ __forceinline__ int token(int base, int lane, int i) { return base + (i / PER) * (32 * PER) + PER * lane + i % PER; }
  __device__ __forceinline__ void load(const T* x, int base, int V, int lane, bool words) {
    const bool whole = base + TILE <= V;
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const int t = token(base, lane, q * PER);
      if constexpr (PER == 1) {
        w[q] = whole || t < V ? __ldg(reinterpret_cast<const uint32_t*>(x) + t) : 0xff800000u;
      } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(x);
        constexpr uint32_t none = std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;      // -inf
        if (words && (whole || t + 1 < V)) {
          w[q] = __ldg(reinterpret_cast<const uint32_t*>(h + t));
        } else {
          const uint32_t lo = t < V ? __ldg(h + t) : none, hi = t + 1 < V ? __ldg(h + t + 1) : none;
          w[q] = lo | hi << 16;
        }
      }
    }
  }
  __device__ __forceinline__ void values(float (&f)[16]) const {
#pragma unroll
    for (int q = 0; q < N; ++q) {
      if constexpr (PER == 1) {
        f[q] = clean(__uint_as_float(w[q]));
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[q]));
        f[2 * q] = clean(v.x); f[2 * q + 1] = clean(v.y);
      } else {
        f[2 * q] = clean(__uint_as_float(w[q] << 16)); f[2 * q + 1] = clean(__uint_as_float(w[q] & 0xffff0000u));
      }
    }
  }
};

// Running maximum of a lane, and the sum of e^{x - ref} over its tokens.  A row that has few warps gives a lane thousands of terms (V / 32 with one warp), so the sum
// is two floats, s + c: a tile's 16 terms are added pair by pair and go in with what rounding loses kept in c; one float32 dropped every faint term behind a large one
// (2e-4 of the logarithm at 131072 tokens).  `ref` follows the maximum only when that is 8 above it: each move multiplies the sum by a rounded factor, and a sum
// that matters sees two of them at most.  A term is 2^y (1 + ln 2 r), y = d log2 e as rounded and r what the rounding left out, some 2^-24 |d|: without r, a million
// equal faint tokens are off by the same amount each.
struct Sum {
  float m = NEG, ref = NEG, s = 0.f, c = 0.f;
  __device__ __forceinline__ void add(const float (&x)[16], float top) {
    if (top > m) m = top;
    if (top > ref + 8.f) {
      const float f = expf(ref - top);      // (ref = -inf: zero)
      s *= f;
      c *= f;
      ref = top;
    }
    const float base = ref == NEG ? 0.f : ref;
    float four[4], r = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float d = fmaxf(x[4 * q + i] - base, -200.f), y = d * tc::LOG2E;      // (2^-288: zero)
        e[i] = tc::ex2(y);
        r = fmaf(e[i], fmaf(d, LOG2E_LO, fmaf(d, tc::LOG2E, -y)), r);
      }
      four[q] = (e[0] + e[1]) + (e[2] + e[3]);
    }
    const float p = (four[0] + four[1]) + (four[2] + four[3]), t = s + p, b = t - s;
    c += fmaf(LN2, r, (s - (t - b)) + (p - b));
    s = t;
  }
};

// A token and its logit as one number, larger is better: the logit's bits in the order of the numbers, then the complement of the token.  0: none.
typedef unsigned long long Key;
__device__ __forceinline__ uint32_t key_hi(float v) { const uint32_t u = __float_as_uint(v); return u >> 31 ? ~u : u | 0x80000000u; }
__device__ __forceinline__ float key_logit(Key k) { const uint32_t u = (uint32_t)(k >> 32); return __uint_as_float(u >> 31 ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ int key_token(Key k) { return (int)~(uint32_t)k; }

struct Smem {
  union {
    Key key[MAXC * NWARP * MAXW];                  // in the first CTA: of every warp of the cluster, the W best of its slice [warp][W]
    struct { double score[MAXW * MAXW + MAXW]; int order[MAXW * MAXW + MAXW], token[MAXW * MAXW + MAXW]; } last;      // then the group's candidates
  };
  Key best[MAXW][MAXW];                            // of a row: its W best
  double s[MAXC * NWARP];                          // of every warp of the cluster: the sum relative to its maximum
  float m[MAXC * NWARP];                           // and that
  double top[MAXW], shift[MAXW];                   // of a row: the maximum; s_i - log (sum relative to it)
  float top_lanes[NWARP][MAXW];                    // of this CTA's warps, the W largest of the lanes' maxima
};
static_assert(sizeof(Smem) <= 48 * 1024, "");
// The cluster's barrier, for threads that may come to it apart: what goes before it here are loops and choices of single lanes.
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  __syncwarp();
}
// the lanes' x in descending order
__device__ __forceinline__ float sort_lanes(float x, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, x, j);
      const bool larger = ((lane & j) == 0) == ((lane & k) == 0);      // (descending as a whole: lane & 32 is 0)
      x = larger ? fmaxf(x, y) : fminf(x, y);
    }
  return x;
}
// the n-th largest of the lanes' x, in every lane
__device__ __forceinline__ float nth_largest(float x, int n, int lane) { return __shfl_sync(0xffffffffu, sort_lanes(x, lane), n - 1); }

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
  cluster_arrive();      // (the first CTA has to be there before it is written to)
  RowBest best;      // of this warp's slice
  Sum sum;
  const bool works = row < W && !(finished && finished[(long long)g * W + row]);
  const T* x = logits + g * stride_g + row * stride_w;
  const int n_tile = (V + TILE - 1) / TILE;
  const int lo = works ? (int)((long long)n_tile * part / per_row) : 0, hi = works ? (int)((long long)n_tile * (part + 1) / per_row) : 0;
  float other = NEG;      // the largest of a lane's tokens outside the tile with its maximum
  int at = lo;            // that tile
  if (lo < hi) {
    const bool words = (reinterpret_cast<uintptr_t>(x) & 3) == 0;
    Tile<T> next;      // the next tile is on its way while one is looked at (two of them cost spilled registers: 64 groups of 8 float32 rows 47.6 us, so 35.0)
    next.load(x, lo * TILE, V, lane, words);
#pragma unroll 1
    for (int t = lo; t < hi; ++t) {
      const Tile<T> tile = next;
      if (t + 1 < hi) next.load(x, (t + 1) * TILE, V, lane, words);
      float f[16];
      tile.values(f);
      float top = f[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, f[i]);
      other = fmaxf(other, fminf(top, sum.m));
      if (top > sum.m) at = t;
      sum.add(f, top);
    }
  }
  const float sorted = sort_lanes(sum.m, lane);
  if (lane < W) sm.top_lanes[warp][lane] = sorted;
  __syncthreads();
  if (lo < hi) {
    // what the row's W best are at least, as far as this CTA's warps know: of the warps' W largest, folded onto 32 lanes, the W-th largest
    const int w0 = max(0, warp - part), w1 = min(NWARP, warp - part + per_row);      // (a row's warps that lie in this CTA)
    float most = NEG;
    for (int e = lane; e < (w1 - w0) * W; e += 32) most = fmaxf(most, sm.top_lanes[w0 + e / W][e % W]);
    const float least = nth_largest(most, W, lane);      // (-inf where few tokens are possible: then the impossible ones count, too)
    float wv = NEG;
    int wi = RowBest::NONE;
    const uint32_t lanes = __ballot_sync(0xffffffffu, sum.m >= least), whole = lanes & __ballot_sync(0xffffffffu, other >= least);
    // (all that is going to be looked at next is asked for before the first of it is: the way to L2 is what this takes)
    constexpr int AHEAD = 4;
    float f[AHEAD];
    int token[AHEAD];
    const auto ask = [&](int q, int j, bool have) {
      token[q] = have && j < V ? j : RowBest::NONE;
      f[q] = token[q] != RowBest::NONE ? clean(to_f32(x[j])) : NEG;
    };
    const auto look = [&]() {
#pragma unroll
      for (int q = 0; q < AHEAD; ++q)
        if (__any_sync(0xffffffffu, f[q] >= least)) offer(best, wv, wi, f[q], f[q] >= least ? token[q] : RowBest::NONE, W, lane);
    };
    for (uint32_t left = lanes & ~whole; left;) {      // one tile of each lane's tokens, two lanes at a time
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        const int l0 = __ffs(left) - 1;
        const bool one = left != 0;
        left &= left - 1;
        const int l1 = __ffs(left) - 1;
        const bool two = left != 0;
        left &= left - 1;
        const int l = max(0, lane < 16 ? l0 : l1), t0 = __shfl_sync(0xffffffffu, at, l);
        ask(q, Tile<T>::token(t0 * TILE, l, lane & 15), lane < 16 ? one : two);
      }
      look();
    }
    for (uint32_t left = whole; left; left &= left - 1) {      // all tiles of a lane's
      const int l = __ffs(left) - 1, n = (hi - lo) * 16;
      for (int e = lane; e - lane < n; e += 32 * AHEAD) {
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) ask(q, Tile<T>::token((lo + ((e + 32 * q) >> 4)) * TILE, l, e & 15), e + 32 * q < n);
        look();
      }
    }
  }
  // the warp's sum, relative to its maximum
  float m = sum.m;
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  double s = sum.m == NEG ? 0.0 : ((double)sum.s + (double)sum.c) * (double)expf(sum.ref - m);
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  cluster_wait();
  const uint32_t home = tc::cluster_addr(tc::smem_u32(&sm), 0);
  auto put = [&](const void* p, int bits) {      // a word to the first CTA
    tc::store_cluster(home + (tc::smem_u32(p) - tc::smem_u32(&sm)), bits); };
  if (lane == 0) { put(&sm.m[all], __float_as_int(m)); put(&sm.s[all], __double2loint(s)); put(reinterpret_cast<const int*>(&sm.s[all]) + 1, __double2hiint(s)); }
  if (lane < W) {
    const uint32_t* k = reinterpret_cast<const uint32_t*>(&sm.key[all * W + lane]);
    const bool any = best.i != RowBest::NONE;
    put(k, any ? (int)~(uint32_t)best.i : 0);
    put(k + 1, any ? (int)key_hi(best.v + 0.f) : 0);      // (zeros of either sign are equal)
  }
  cluster_arrive();
  cluster_wait();
  if (rank) return;

  // The rows' normalisers, a warp to a row, and their W best: the place of a candidate is the number of those before it, counted by a thread.
  for (int i = threadIdx.x; i < W * MAXW; i += NWARP * 32) sm.best[i / MAXW][i % MAXW] = 0;
  for (int i = warp; i < W; i += NWARP) {
    const float score = scores[(long long)g * W + i];
    float mm = NEG;
    for (int q = lane; q < per_row; q += 32) mm = fmaxf(mm, sm.m[i * per_row + q]);
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
    double ss = 0.0;
    for (int q = lane; q < per_row; q += 32) {
      const float mq = sm.m[i * per_row + q];
      if (mq != NEG) ss += sm.s[i * per_row + q] * (double)expf(mq - mm);
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
  const int n_key = per_row * W;      // of a row
  for (int e = threadIdx.x; e < W * n_key; e += NWARP * 32) {
    const Key mine = sm.key[e];
    if (!mine) continue;
    const Key* k = sm.key + e / n_key * n_key;
    int place = 0;
#pragma unroll 8
    for (int q = 0; q < n_key; ++q) place += k[q] > mine;
    if (place < W) sm.best[e / n_key][place] = mine;
  }
  __syncthreads();
  // The group's candidates: the rows' W best and, behind them, the finished beams' eos.  Of equal scores the lower beam's comes first, and of one beam's the one
  // that its own order puts first: by logits, which may differ where the sums do not, then by tokens (for impossible candidates and a finished beam by tokens).
  const int n_last = W * W + W;
  for (int e = threadIdx.x; e < n_last; e += NWARP * 32) {
    const int i = e < W * W ? e / W : e - W * W, at = e - i * W;
    const bool over = finished && finished[(long long)g * W + i];
    double score = NEG;
    int t = -1;      // (none)
    if (e >= W * W) {
      if (over) {
        const float s = scores[(long long)g * W + i];
        if (s == s) score = s;
        t = (int)eos;
      }
    } else if (over) {                            // impossible tokens from the first one on, but eos
      t = at < (int)eos ? at : at + 1;
    } else if (sm.shift[i] == (double)NEG) {      // a beam that is impossible: all its tokens are, the first ones first
      t = at;
    } else if (const Key k = sm.best[i][at]) {
      t = key_token(k);
      if (key_logit(k) != NEG) score = sm.shift[i] + ((double)key_logit(k) - sm.top[i]);
    }
    sm.last.score[e] = score;
    sm.last.token[e] = t;
    // (a finished beam's tokens: eos before the W-th or behind all of the others)
    const int place = e < W * W ? over && at >= (int)eos ? at + 1 : at : (int)(eos < W ? eos : W);
    sm.last.order[e] = t < 0 || t >= V ? NO_ORDER : i * (W + 1) + place;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n_last; e += NWARP * 32) {
    const double score = sm.last.score[e];
    const int j = sm.last.order[e];
    if (j == NO_ORDER) continue;
    int place = 0;
#pragma unroll 4
    for (int q = 0; q < n_last; ++q) place += before(sm.last.score[q], sm.last.order[q], score, j);
    if (place < W) {
      const long long at = (long long)g * W + place, parent = e < W * W ? e / W : e - W * W, t = sm.last.token[e];
      scores_out[at] = (float)score;
      parents[at] = parent;
      tokens[at] = t;
      if (finished_out) finished_out[at] = (finished && finished[(long long)g * W + parent]) || t == eos;
    }
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
  while (c > 1 && (long long)W * V <= (long long)(c >> 1) * NWARP * TILE) c >>= 1;
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
