// Linear attention with a decay for each head in float32 arithmetic on the CUDA cores: float32 and float16 tokens, and head
// size 128.  The equations are in linattn.cuh.
//
// The state between chunks of 64 tokens is a linear recurrence whose decay is a number, so it is split off: every chunk's
// addition to the state (one kernel, all chunks at once), a scan over the chunks (elementwise), and then outputs or gradients of
// all chunks at once from the state before each.  A chunk is one CTA's work whatever the number of sequences.
//
// What bounds it: float32 multiply-adds at the latency of shared memory that feeds them (issue slots 46 - 54 % used, the multiply-add pipe 33 - 40 %, no other
// unit above 55 %).  B2 T1024 H16 of 64 in float32, forward and backward, 512 chunks: adding 19 us and scanning 7.5 us in either direction, outputs 37 us,
// gradients 109 us in 3.5 waves of blocks; the bytes of the tensors alone would take 11.
#include "linattn.cuh"

namespace rwkvb200 {
namespace la {
namespace {

constexpr int C = 64;         // tokens of a chunk
constexpr int PAD = 4;        // rows of shared tiles are 4 floats longer: 16-byte reads of 16 rows do not conflict
constexpr int LD = 64 + PAD;
constexpr int NTHR = 256;

// acc[a][b] += sum over kk < n of A(RA ig + a, kk) B(kk, j).  AM / BM: the contraction index is the row of the array (A[kk][i], B[kk][j]) instead of its
// column (A[i][kk], B[j][kk]).  Columns j: 4 jg + b with BM, so that they are one read, else jg + 16 b, so that 16 rows' reads do not conflict.  A warp's
// two ig and 16 jg take 12 shared-memory cycles for 64 multiply-adds in every form, below the 16 that these take.
template <bool AM, bool BM, int RA>
__device__ __forceinline__ void mm(float (&acc)[RA][4], const float* A, int lda, const float* B, int ldb, int n, int ig, int jg) {
#pragma unroll 4
  for (int kk = 0; kk < n; kk += 4) {
    float a[RA][4], b[4][4];
#pragma unroll
    for (int x = 0; x < (AM ? 4 : RA); ++x) {
      if constexpr (!AM) {
        const float4 f = *reinterpret_cast<const float4*>(A + (RA * ig + x) * lda + kk);
        a[x][0] = f.x; a[x][1] = f.y; a[x][2] = f.z; a[x][3] = f.w;
      } else if constexpr (RA == 4) {
        const float4 f = *reinterpret_cast<const float4*>(A + (kk + x) * lda + 4 * ig);
        a[0][x] = f.x; a[1][x] = f.y; a[2][x] = f.z; a[3][x] = f.w;
      } else {
        const float2 f = *reinterpret_cast<const float2*>(A + (kk + x) * lda + 2 * ig);
        a[0][x] = f.x; a[1][x] = f.y;
      }
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if constexpr (BM) {
        const float4 f = *reinterpret_cast<const float4*>(B + (kk + x) * ldb + 4 * jg);
        b[0][x] = f.x; b[1][x] = f.y; b[2][x] = f.z; b[3][x] = f.w;
      } else {
        const float4 f = *reinterpret_cast<const float4*>(B + (jg + 16 * x) * ldb + kk);
        b[x][0] = f.x; b[x][1] = f.y; b[x][2] = f.z; b[x][3] = f.w;
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int x = 0; x < RA; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = fmaf(a[x][c], b[y][c], acc[x][y]);
  }
}
template <int RA>
__device__ __forceinline__ void clear(float (&acc)[RA][4]) {
#pragma unroll
  for (int x = 0; x < RA; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y) acc[x][y] = 0.f;
}

// Rows 0 .. 63 (the first n of them from p with `stride` elements between rows, zeros behind) of W columns, as float32.
template <typename T, int W>
__device__ __forceinline__ void load_rows(float* dst, int ld, const T* p, long long stride, int n) {
  for (int i = threadIdx.x; i < 64 * (W / 4); i += blockDim.x) {
    const int row = i / (W / 4), c = i % (W / 4) * 4;
    const float4 f = row < n ? load4(p + row * stride + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    *reinterpret_cast<float4*>(dst + row * ld + c) = f;
  }
}

// 64 rows of 64 columns of a state, transposed.
__device__ __forceinline__ void load_transposed(float* dst, const float* p, int stride) {
  for (int i = threadIdx.x; i < 64 * 16; i += blockDim.x) {
    const int row = i & 63, c = i >> 6 << 2;      // (a warp's 32 rows: writes next to each other)
    const float4 f = load4(p + row * stride + c);
    dst[c * LD + row] = f.x; dst[(c + 1) * LD + row] = f.y; dst[(c + 2) * LD + row] = f.z; dst[(c + 3) * LD + row] = f.w;
  }
}

// Inclusive prefix sums of g over a chunk, each as two floats: sums and differences of them are exact to far below float32's last bit, and the many
// differences that are taken cost no float64 arithmetic, of which an SM does little (the gradient kernel of B2 T1024 H16: 110 us with it, 108 without).
struct Sums { float hi[C], lo[C]; };
__device__ __forceinline__ float between(const Sums& L, int i, int j) { return (L.hi[i] - L.hi[j]) + (L.lo[i] - L.lo[j]); }
// by the first warp, of n tokens (those behind do not decay); L[63] is the sum over the chunk
__device__ __forceinline__ void prefix(Sums& L, float* g, const Tokens& t, const float* w, long long wb, int t0, int n) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x, i = 2 * lane;
    const float g0 = i < n ? g_of(w[wb + (t0 + i) * t.wst]) : 0.f;
    const float g1 = i + 1 < n ? g_of(w[wb + (t0 + i + 1) * t.wst]) : 0.f;
    double s = (double)g0 + (double)g1;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += up;
    }
    const double s0 = s - (double)g1;
    L.hi[i] = (float)s0; L.lo[i] = (float)(s0 - (double)L.hi[i]);
    L.hi[i + 1] = (float)s; L.lo[i + 1] = (float)(s - (double)L.hi[i + 1]);
    if (g) { g[i] = g0; g[i + 1] = g1; }
  }
}

// The sequence of a packed batch that slot s belongs to: the last one whose slots start at s or before, found by a warp, 32 of them at a time (one look for 32
// sequences, two for 1024); -1: s is before the first.
__device__ __forceinline__ int sequence_of(const Tokens& t, int s) {
  const int lane = threadIdx.x & 31;
  int lo = -1, end = t.n_seq;
  while (end - lo > 1) {      // it is lo or one of lo + 1 .. end - 1
    const int step = (end - lo - 1 + 31) / 32, at = lo + 1 + lane * step;
    const int n = __popc(__ballot_sync(0xffffffffu, at < end && t.place(at, 0) <= s));
    const int from = lo;
    if (n) lo = from + 1 + (n - 1) * step;
    end = min(end, from + 1 + n * step);
    if (!n) end = from + 1;
  }
  return lo;
}
// Which chunk a block works on: chunk c of (sequence n, head h), none where rows < 1.  `slot`: of the head's, over all sequences.
struct Where { int n, h, c, slot, t0, rows; };
__device__ __forceinline__ Where where(const Tokens& t) {
  Where x;
  const int b = blockIdx.x;
  if (t.compact) {
    x.h = b / t.slots; x.slot = b % t.slots;
    x.n = sequence_of(t, x.slot);
    x.c = x.n < 0 ? 0 : x.slot - t.place(x.n, 0);
  } else {
    const int unit = b / t.NT;
    x.c = b % t.NT;
    x.n = unit / t.H; x.h = unit % t.H;
    x.slot = x.n * t.NT + x.c;
  }
  x.t0 = x.c * C;
  x.rows = x.n < 0 ? 0 : min(C, t.length(x.n) - x.t0);
  return x;
}

// What a chunk adds to the state (REV: to its gradient, walking backwards), a 64 x 64 block of it, into the slot after (before) the chunk, and the
// chunk's decay.
template <typename T, int D, bool REV>
__global__ void __launch_bounds__(NTHR, 4) la_add_kernel(const T* __restrict__ val, const T* __restrict__ key, const float* __restrict__ w,
                                                      float* __restrict__ states, float* __restrict__ decay, Tokens tok) {
  __shared__ __align__(16) float av[64 * LD], bk[64 * LD];
  __shared__ Sums L;
  earlier_kernels_done();
  later_kernels_may_start();
  const int pv = blockIdx.y / (D / 64), pk = blockIdx.y % (D / 64);
  const Where x = where(tok);
  if (x.rows < 1) return;
  prefix(L, nullptr, tok, w, tok.wbase(x.n, x.h), x.t0, x.rows);
  const long long base = tok.base(x.n, x.h) + x.t0 * tok.st;
  load_rows<T, 64>(av, LD, val + base + 64 * pv, tok.st, x.rows);
  load_rows<T, 64>(bk, LD, key + base + 64 * pk, tok.st, x.rows);
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * 64; i += NTHR) {
    const int j = i >> 6;
    bk[j * LD + (i & 63)] *= expf(REV ? L.hi[j] : between(L, C - 1, j));
  }
  __syncthreads();
  const int ig = threadIdx.x >> 4, jg = threadIdx.x & 15;
  float acc[4][4];
  clear(acc);
  mm<true, true>(acc, av, LD, bk, LD, 64, ig, jg);
  float* out = states + (tok.first(x.n, x.h, 1) + (REV ? x.c : x.c + 1)) * (D * D) + (64 * pv) * D + 64 * pk;
#pragma unroll
  for (int a = 0; a < 4; ++a) store4(out + (4 * ig + a) * D + 4 * jg, make_float4(acc[a][0], acc[a][1], acc[a][2], acc[a][3]));
  if (blockIdx.y == 0 && threadIdx.x == 0) decay[tok.first(x.n, x.h, 0) + x.c] = expf(L.hi[C - 1]);
}

// The scan over the chunks, four elements of a unit's state to a thread.  Forward: slot 0 is the initial state (or zero), slot c + 1 =
// decay[c] slot c + what it holds; the last one goes to `last` as well.  REV: slot NT is the gradient of the final state (or zero), slot c =
// decay[c] slot c + 1 + what it holds; slot 0 goes to `last`.
template <int D, bool REV>
__global__ void __launch_bounds__(256) la_scan_kernel(float* __restrict__ states, const float* __restrict__ decay, const float* __restrict__ first,
                                                      int n_first, float* __restrict__ last, Tokens tok) {
  earlier_kernels_done();
  later_kernels_may_start();
  constexpr int PER = D * D / 4;
  const int unit = blockIdx.x / (PER / 256), e = 4 * ((blockIdx.x % (PER / 256)) * 256 + threadIdx.x);
  const int n = unit / tok.H, h = unit % tok.H, NT = (tok.length(n) + C - 1) / C;
  float4 S = make_float4(0.f, 0.f, 0.f, 0.f);
  if (first && n_first > 0) S = *reinterpret_cast<const float4*>(first + ((long long)(n_first == 1 ? 0 : n) * tok.H + h) * (D * D) + e);
  float* slot = states + tok.first(n, h, 1) * (D * D) + e;
  const float* dec = decay + tok.first(n, h, 0);
  *reinterpret_cast<float4*>(slot + (long long)(REV ? NT : 0) * (D * D)) = S;
  constexpr int AHEAD = 8;
  for (int c0 = 0; c0 < NT; c0 += AHEAD) {
    float4 add[AHEAD];
    float f[AHEAD];
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      if (c0 + q < NT) {
        const int c = REV ? NT - 1 - c0 - q : c0 + q;
        add[q] = *reinterpret_cast<const float4*>(slot + (long long)(REV ? c : c + 1) * (D * D));
        f[q] = dec[c];
      }
    }
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      if (c0 + q < NT) {
        const int c = REV ? NT - 1 - c0 - q : c0 + q;
        S.x = fmaf(f[q], S.x, add[q].x); S.y = fmaf(f[q], S.y, add[q].y);
        S.z = fmaf(f[q], S.z, add[q].z); S.w = fmaf(f[q], S.w, add[q].w);
        *reinterpret_cast<float4*>(slot + (long long)(REV ? c : c + 1) * (D * D)) = S;
      }
    }
  }
  if (last) *reinterpret_cast<float4*>(last + (long long)unit * (D * D) + e) = S;
}

template <int D> struct OutSmem {
  float r[64 * (D + PAD)], k[64 * (D + PAD)], S[D * LD], v[64 * LD], A[64 * LD];      // S: [k][v]
  Sums L;
};
// 64 columns of the outputs of a chunk.
template <typename T, int D>
__global__ void __launch_bounds__(NTHR) la_out_kernel(const T* __restrict__ r, const T* __restrict__ k, const T* __restrict__ v,
                                                      const float* __restrict__ w, const float* __restrict__ states, T* __restrict__ o, Tokens tok) {
  extern __shared__ __align__(16) unsigned char raw[];
  OutSmem<D>& sm = *reinterpret_cast<OutSmem<D>*>(raw);
  constexpr int LDD = D + PAD;
  earlier_kernels_done();
  later_kernels_may_start();
  const int pv = blockIdx.y;
  const Where x = where(tok);
  if (x.rows < 1) return;
  prefix(sm.L, nullptr, tok, w, tok.wbase(x.n, x.h), x.t0, x.rows);
  const long long base = tok.base(x.n, x.h) + x.t0 * tok.st;
  load_rows<T, D>(sm.r, LDD, r + base, tok.st, x.rows);
  load_rows<T, D>(sm.k, LDD, k + base, tok.st, x.rows);
  load_rows<T, 64>(sm.v, LD, v + base + 64 * pv, tok.st, x.rows);
#pragma unroll
  for (int p = 0; p < D / 64; ++p)
    load_transposed(sm.S + 64 * p * LD, states + (tok.first(x.n, x.h, 1) + x.c) * (D * D) + 64 * pv * D + 64 * p, D);
  __syncthreads();
  const int ig = threadIdx.x >> 4, jg = threadIdx.x & 15;
  float acc[4][4];
  clear(acc);
  mm<false, false>(acc, sm.r, LDD, sm.k, LDD, D, ig, jg);
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int i = 4 * ig + a, j = jg + 16 * b;
      sm.A[i * LD + j] = j <= i ? acc[a][b] * expf(between(sm.L, i, j)) : 0.f;
    }
  clear(acc);
  mm<false, true>(acc, sm.r, LDD, sm.S, LD, D, ig, jg);
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const float f = expf(sm.L.hi[4 * ig + a]);
#pragma unroll
    for (int b = 0; b < 4; ++b) acc[a][b] *= f;
  }
  __syncthreads();
  mm<false, true>(acc, sm.A, LD, sm.v, LD, 64, ig, jg);
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const int i = 4 * ig + a;
    if (i < x.rows) store4(o + base + i * tok.st + 64 * pv + 4 * jg, make_float4(acc[a][0], acc[a][1], acc[a][2], acc[a][3]));
  }
}

constexpr int G_THR = 2 * NTHR;      // of the gradient kernel
template <int D> struct GradSmem {
  float r[64 * (D + PAD)], k[64 * (D + PAD)], v[64 * (D + PAD)], d_o[64 * (D + PAD)], A[64 * LD], E[64 * LD], S[2][64 * LD];
  Sums L;
  float g[C];
  float pairs[G_THR / 32][C], t1[C], t2[C], t3[G_THR / 32];
};
// The sum of x over the 16 threads that hold a row's columns.
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int m = 8; m >= 1; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  return x;
}

// The gradients of a chunk.  dstates: slot c + 1 is the gradient of the state after chunk c.  Two halves of the block work on a product each: one on r k^T and
// dr, the other on d_o v^T and dk, and on dv half its rows each (float32,
// B2 T1024 H16: 121 us with 8 warps to a block, 108 with 16).
template <typename T, int D>
__global__ void __launch_bounds__(G_THR) la_grad_kernel(const T* __restrict__ r, const T* __restrict__ k, const T* __restrict__ v,
                                                        const float* __restrict__ w, const T* __restrict__ d_o,
                                                        const float* __restrict__ states, const float* __restrict__ dstates,
                                                        T* __restrict__ dr, T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ dw,
                                                        int dw_parts, Tokens tok) {
  extern __shared__ __align__(16) unsigned char raw[];
  GradSmem<D>& sm = *reinterpret_cast<GradSmem<D>*>(raw);
  constexpr int LDD = D + PAD, P = D / 64, NW = G_THR / 32;
  earlier_kernels_done();
  later_kernels_may_start();
  const int tid = threadIdx.x;
  const Where x = where(tok);
  const long long part = (long long)x.slot * tok.H + x.h;      // of a w per head: what this chunk adds to its gradient
  if (x.rows < 1) {
    if (dw_parts && tid == 0) dw[part] = 0.f;
    return;
  }
  prefix(sm.L, sm.g, tok, w, tok.wbase(x.n, x.h), x.t0, x.rows);
  const long long base = tok.base(x.n, x.h) + x.t0 * tok.st;
  load_rows<T, D>(sm.r, LDD, r + base, tok.st, x.rows);
  load_rows<T, D>(sm.k, LDD, k + base, tok.st, x.rows);
  load_rows<T, D>(sm.v, LDD, v + base, tok.st, x.rows);
  load_rows<T, D>(sm.d_o, LDD, d_o + base, tok.st, x.rows);
  const float* S0 = states + (tok.first(x.n, x.h, 1) + x.c) * (D * D);
  const float* dS = dstates + (tok.first(x.n, x.h, 1) + x.c + 1) * (D * D);
  const bool first = tid < NTHR;      // which half
  const int ig = (tid & (NTHR - 1)) >> 4, jg = tid & 15, warp = tid >> 5, lane = tid & 31;
  // <dS, S0>
  {
    float s = 0.f;
    for (int i = 4 * tid; i < D * D; i += 4 * G_THR) {
      const float4 a = load4(S0 + i), b = load4(dS + i);
      s += a.x * b.x + a.y * b.y + a.z * b.z + a.w * b.w;
    }
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    if (lane == 0) sm.t3[warp] = s;
  }
  __syncthreads();
  float acc[4][4];
  clear(acc);
  mm<false, false>(acc, first ? sm.r : sm.d_o, LDD, first ? sm.k : sm.v, LDD, D, ig, jg);
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int i = 4 * ig + a, j = jg + 16 * b;
      (first ? sm.A : sm.E)[i * LD + j] = j <= i ? acc[a][b] * expf(between(sm.L, i, j)) : 0.f;      // (a choice, so that infinities above the diagonal stay there)
    }
  __syncthreads();
  if (!first) {
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int i = 4 * ig + a, j = jg + 16 * b;
        sm.S[0][i * LD + j] = j < i ? sm.A[i * LD + j] * acc[a][b] : 0.f;      // (the diagonal does not depend on the decay)
      }
  }
  if (tid < C) { sm.t1[tid] = 0.f; sm.t2[tid] = 0.f; }
  __syncthreads();
  {
    // What the pairs on both sides of t add to dg_t: prefix sums along the rows, then their columns from the diagonal down.  Every term of such a
    // sum carries the decay of t, so a token whose decay is strong gets a gradient that is as exact as any.
    float y[2] = {0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 64 / NW; ++q) {
      const int i = warp + NW * q;
      const float2 m = *reinterpret_cast<const float2*>(&sm.S[0][i * LD + 2 * lane]);
      float s = m.x + m.y;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const float up = __shfl_up_sync(0xffffffffu, s, d);
        if (lane >= d) s += up;
      }
      const float left = __shfl_up_sync(0xffffffffu, s, 1);
      const float p0 = lane ? left : 0.f;      // sum of the columns before 2 lane
      if (2 * lane <= i) y[0] += p0;
      if (2 * lane + 1 <= i) y[1] += p0 + m.x;
    }
    sm.pairs[warp][2 * lane] = y[0];
    sm.pairs[warp][2 * lane + 1] = y[1];
  }
  float f[4];      // the decay between a row's token and the state: before the chunk, behind it
#pragma unroll
  for (int a = 0; a < 4; ++a) f[a] = expf(first ? sm.L.hi[4 * ig + a] : between(sm.L, C - 1, 4 * ig + a));
  const int row0 = first ? 0 : 32;      // of dv
  float fv[2];
#pragma unroll
  for (int a = 0; a < 2; ++a) fv[a] = expf(between(sm.L, C - 1, row0 + 2 * ig + a));
  for (int p = 0; p < P; ++p) {      // 64 columns of each gradient
    clear(acc);
    for (int pv = 0; pv < P; ++pv) {
      __syncthreads();
      load_rows<float, 64>(sm.S[0], LD, S0 + 64 * pv * D + 64 * p, D, 64);
      load_rows<float, 64>(sm.S[1], LD, dS + 64 * pv * D + 64 * p, D, 64);
      __syncthreads();
      mm<false, true>(acc, (first ? sm.d_o : sm.v) + 64 * pv, LDD, sm.S[first ? 0 : 1], LD, 64, ig, jg);
    }
    const float* q = (first ? sm.r : sm.k) + 64 * p;      // (what it is multiplied with in dg)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const float4 q4 = *reinterpret_cast<const float4*>(q + (4 * ig + a) * LDD + 4 * jg);
#pragma unroll
      for (int b = 0; b < 4; ++b) acc[a][b] *= f[a];
      const float s = row_sum(acc[a][0] * q4.x + acc[a][1] * q4.y + acc[a][2] * q4.z + acc[a][3] * q4.w);
      if (jg == 0) (first ? sm.t1 : sm.t2)[4 * ig + a] += s;
    }
    if (first) mm<false, true>(acc, sm.E, LD, sm.k + 64 * p, LDD, 64, ig, jg);
    else       mm<true, true>(acc, sm.E, LD, sm.r + 64 * p, LDD, 64, ig, jg);
    T* out = first ? dr : dk;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int i = 4 * ig + a;
      if (i < x.rows) store4(out + base + i * tok.st + 64 * p + 4 * jg, make_float4(acc[a][0], acc[a][1], acc[a][2], acc[a][3]));
    }
    float av[2][4];
    clear(av);
    for (int pk = 0; pk < P; ++pk) {
      __syncthreads();
      load_transposed(sm.S[0], dS + 64 * p * D + 64 * pk, D);
      __syncthreads();
      mm<false, true>(av, sm.k + row0 * LDD + 64 * pk, LDD, sm.S[0], LD, 64, ig, jg);
    }
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b) av[a][b] *= fv[a];
    mm<true, true>(av, sm.A + row0, LD, sm.d_o + 64 * p, LDD, 64, ig, jg);
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const int i = row0 + 2 * ig + a;
      if (i < x.rows) store4(dv + base + i * tok.st + 64 * p + 4 * jg, make_float4(av[a][0], av[a][1], av[a][2], av[a][3]));
    }
  }
  __syncthreads();
  if (warp == 0) {      // dg_t, two tokens to a lane
    double after[2], before[2], pairs[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int i = 2 * lane + q;
      pairs[q] = 0.0;
#pragma unroll
      for (int u = 0; u < NW; ++u) pairs[q] += sm.pairs[u][i];
      after[q] = sm.t1[i];
      before[q] = sm.t2[i];
    }
    double sa = after[0] + after[1], sb = before[0] + before[1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double dn = __shfl_down_sync(0xffffffffu, sa, d), up = __shfl_up_sync(0xffffffffu, sb, d);
      if (lane + d < 32) sa += dn;
      if (lane >= d) sb += up;
    }
    double t3 = 0.0;
#pragma unroll
    for (int u = 0; u < NW; ++u) t3 += sm.t3[u];
    t3 *= (double)expf(sm.L.hi[C - 1]);
    double sum = 0.0;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int i = 2 * lane + q;
      const double dg = pairs[q] + (q ? sa - after[0] : sa) + (q ? sb - before[1] : sb - before[1] - before[0]) + t3;
      if (i < x.rows) {
        const double y = dg * (double)sm.g[i];
        if (dw_parts) sum += y;
        else dw[tok.wbase(x.n, x.h) + (x.t0 + i) * tok.wst] = (float)y;
      }
    }
    if (dw_parts) {
#pragma unroll
      for (int m = 16; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
      if (lane == 0) dw[part] = (float)sum;
    }
  }
}

// Partial sums over a stretch of rows of a [rows][H] array, and the sums over the stretches.
__global__ void __launch_bounds__(256) la_dw_part_kernel(const float* __restrict__ dw, long long rows, int H, double* __restrict__ part) {
  __shared__ double s[8][32];
  earlier_kernels_done();
  later_kernels_may_start();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long per = (rows + gridDim.x - 1) / gridDim.x, lo = blockIdx.x * per, hi = min(rows, lo + per);
  const int h = blockIdx.y * 32 + lane;
  double x = 0.0;
  if (h < H)
    for (long long i = lo + warp; i < hi; i += 8) x += dw[i * H + h];
  s[warp][lane] = x;
  __syncthreads();
  if (warp == 0 && h < H) {
#pragma unroll
    for (int u = 1; u < 8; ++u) x += s[u][lane];
    part[(long long)blockIdx.x * H + h] = x;
  }
}
__global__ void __launch_bounds__(256) la_dw_sum_kernel(const double* __restrict__ part, int parts, int H, float* __restrict__ dw) {
  earlier_kernels_done();
  later_kernels_may_start();
  const int h = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;      // a warp to a head
  if (h >= H) return;
  double x = 0.0;
  for (int i = lane; i < parts; i += 32) x += part[(long long)i * H + h];
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  if (lane == 0) dw[h] = (float)x;
}

inline size_t a256(size_t x) { return (x + 255) & ~size_t(255); }

struct Scratch { float *dstates, *decay, *dw; double* part; };
Scratch scratch_of(void* p, const Tokens& t, int D, bool w_per_head, bool backward) {
  Scratch s = {};
  unsigned char* q = static_cast<unsigned char*>(p);
  const size_t slots = (size_t)t.slots * t.H, more = (size_t)t.n_seq * t.H;
  s.decay = reinterpret_cast<float*>(q); q += a256(slots * 4);
  if (backward) {
    s.dstates = reinterpret_cast<float*>(q); q += a256((slots + more) * D * D * 4);
    if (w_per_head) {
      s.dw = reinterpret_cast<float*>(q); q += a256(slots * 4);      // [slots][H]
      s.part = reinterpret_cast<double*>(q);
    }
  }
  return s;
}

template <typename T, int D>
int fwd(const Args& a, cudaStream_t st) {
  const Tokens& t = a.tok;
  const int units = t.n_seq * t.H;
  const Scratch s = scratch_of(a.scratch, t, D, a.w_per_head, false);
  DeviceFacts f;
  if (int e = device_facts(&f)) return e;
  {
    ProfScope prof("linattn_add_kernel", st);
    if (int e = launch(la_add_kernel<T, D, false>, dim3(t.slots * t.H, D * D / 4096), NTHR, 0, st, 1, (const T*)a.v, (const T*)a.k, a.w, a.states,
                       s.decay, t)) return e;
  }
  {
    ProfScope prof("linattn_scan_kernel", st);
    if (int e = launch(la_scan_kernel<D, false>, units * (D * D / 1024), 256, 0, st, 1, a.states, (const float*)s.decay, a.h0, a.n_state, a.ht, t)) return e;
  }
  if (!a.o) return RWKVB200_OK;
  ProfScope prof("linattn_out_kernel", st);
  constexpr int smem = (int)sizeof(OutSmem<D>);
  if (int e = allow_smem<la_out_kernel<T, D>>(f, smem)) return e;
  return launch(la_out_kernel<T, D>, dim3(t.slots * t.H, D / 64), NTHR, smem, st, 1, (const T*)a.r, (const T*)a.k, (const T*)a.v, a.w,
                (const float*)a.states, (T*)a.o, t);
}

template <typename T, int D>
int bwd(const Args& a, cudaStream_t st) {
  const Tokens& t = a.tok;
  const int units = t.n_seq * t.H;
  const Scratch s = scratch_of(a.scratch, t, D, a.w_per_head, true);
  DeviceFacts f;
  if (int e = device_facts(&f)) return e;
  {
    ProfScope prof("linattn_add_kernel", st);
    if (int e = launch(la_add_kernel<T, D, true>, dim3(t.slots * t.H, D * D / 4096), NTHR, 0, st, 1, (const T*)a.d_o, (const T*)a.r, a.w, s.dstates,
                       s.decay, t)) return e;
  }
  {
    ProfScope prof("linattn_scan_kernel", st);
    if (int e = launch(la_scan_kernel<D, true>, units * (D * D / 1024), 256, 0, st, 1, s.dstates, (const float*)s.decay, a.d_ht, t.n_seq, a.dh0, t)) return e;
  }
  {
    ProfScope prof("linattn_grad_kernel", st);
    constexpr int smem = (int)sizeof(GradSmem<D>);
    if (int e = allow_smem<la_grad_kernel<T, D>>(f, smem)) return e;
    if (int e = launch(la_grad_kernel<T, D>, t.slots * t.H, G_THR, smem, st, 1, (const T*)a.r, (const T*)a.k, (const T*)a.v, a.w, (const T*)a.d_o,
                       (const float*)a.states, (const float*)s.dstates, (T*)a.dr, (T*)a.dk, (T*)a.dv, a.w_per_head ? s.dw : a.dw, a.w_per_head, t)) return e;
  }
  return a.w_per_head ? launch_sum_dw(s.dw, t.slots, t.H, s.part, a.dw, st) : RWKVB200_OK;
}

}  // namespace

int launch_sum_dw(const float* dw_rows, long long rows, int H, double* partial, float* dw, cudaStream_t st) {
  ProfScope prof("linattn_dw_kernel", st);
  const int parts = (int)(rows < DW_PARTS * 8 ? (rows + 7) / 8 : DW_PARTS);
  if (int e = launch(la_dw_part_kernel, dim3(parts, (H + 31) / 32), 256, 0, st, 1, dw_rows, rows, H, partial)) return e;
  return launch(la_dw_sum_kernel, (H + 7) / 8, 256, 0, st, 1, (const double*)partial, parts, H, dw);
}

size_t simt_states_bytes(int n_seq, int max_len, int total, int H, int D) {
  return (size_t)(chunk_slots(n_seq, max_len, total, C) + n_seq) * H * D * D * 4;
}
size_t simt_scratch_bytes(int n_seq, int max_len, int total, int H, int D, bool w_per_head, bool backward) {
  const size_t slots = (size_t)chunk_slots(n_seq, max_len, total, C) * H;
  size_t n = a256(slots * 4);
  if (backward) {
    n += a256((slots + (size_t)n_seq * H) * D * D * 4);
    if (w_per_head) n += a256(slots * 4) + a256((size_t)DW_PARTS * H * 8);
  }
  return n;
}

int launch_simt_fwd(const Args& args, cudaStream_t st) {
  Args a = args;
  set_chunks(a, C);
  RWKVB200_DISPATCH_DTYPE(a.dtype, return a.D == 64 ? fwd<T, 64>(a, st) : fwd<T, 128>(a, st));
  return RWKVB200_OK;
}
int launch_simt_bwd(const Args& args, cudaStream_t st) {
  Args a = args;
  set_chunks(a, C);
  RWKVB200_DISPATCH_DTYPE(a.dtype, return a.D == 64 ? bwd<T, 64>(a, st) : bwd<T, 128>(a, st));
  return RWKVB200_OK;
}

}  // namespace la
}  // namespace rwkvb200
