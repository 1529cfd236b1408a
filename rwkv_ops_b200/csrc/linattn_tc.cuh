// Linear attention with a decay for each head on tcgen05 (bfloat16 tokens, head size 64): what the forward and backward kernels share.  The
// equations are in linattn.cuh; a chunk is 128 tokens, so that products over tokens fill the 128 lanes of TMEM and a thread owns a
// token's row.
//
// Precision.  r, k, v, d_o are bfloat16 and enter products as they are.  The keys (queries) that are added to the state (its gradient) carry a decay and are split
// into three bfloat16 parts (three products, exact to float32's last bits: states go from chunk to chunk and are float32).  The states that meet v and d_o in the
// backward are in three parts, too, as from these products comes the part of dw that reaches beyond its chunk (with two, 2^-17 of an element, dw was
// off by 1.2e-6 instead of 3e-7); the one that meets k, for dv alone, is in two.  The smallest part goes first: an accumulator in TMEM cuts off what a product adds below its own last bit, and 24 steps of a chunk at
// full size leave states 5e-7 too small, 8 of them 1.3e-7.  A and E are rounded once to bfloat16, as is the state that meets r in the forward: those results are
// rounded to bfloat16 anyway.
//
// Work is cut into items, a stretch of consecutive chunks of one (sequence, head).  With as many units as the device holds CTAs, an item is a unit.  With
// fewer, a unit is several parts: a first kernel finds what each adds to the state, keys and values only, and then all parts are walked at once from the state
// each starts with.  That reads half of the tokens twice and pays as soon as the chain of chunks is more than a few.
#pragma once

#include "linattn.cuh"
#include "tc.cuh"

namespace rwkvb200 {
namespace la {

using namespace tc;
typedef __nv_bfloat16 bf16;

constexpr int CT = 128;                        // tokens of a chunk
constexpr int TOK_BYTES = 2 * TILE_BYTES;      // a chunk of a token tensor: two tiles of 64 tokens x 64 channels

// Decay factors of a chunk.  L is the inclusive prefix sum, Lb(I) its value before the I-th block of 32 tokens; every exponent is a sum over tokens, so
// every factor is at most one.  A block of 32 x 32 pairs below the diagonal takes its factor e^{L_i - L_j} as row * col, a diagonal one from `in`.
struct Decays {
  float start[CT];        // e^{L_i}
  float end[CT];          // e^{Lc - L_i}
  float row[CT];          // e^{L_i - Lb(i / 32)}
  float in[CT], in_lo[CT];      // (L_i - Lb(i / 32)) log2 e, in two floats: under fast decays neighbours differ by little of what has summed up
  float col[3][CT];       // [I - 1][j]: e^{Lb(I) - L_j}, j < 32 I
  float all;              // e^{Lc}
  float pad[3];
};

// w of a chunk, four consecutive tokens to a lane of one warp.
struct RawW { float w[4]; };
__device__ __forceinline__ RawW load_w(const Tokens& t, const float* w, long long wb, int t0, int n) {
  RawW x;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int i = 4 * (threadIdx.x & 31) + q;
    x.w[q] = i < n ? __ldg(w + wb + (long long)(t0 + i) * t.wst) : 0.f;
  }
  return x;
}
// by one warp; tokens from n on do not decay.  g (may be NULL): the tokens' g
// (with exponentials in float64 this took 5000 cycles of its warp, for which the others waited)
__device__ __forceinline__ void make_decays(Decays& d, const RawW& x, int n, float* g) {
  const int lane = threadIdx.x & 31;
  float y[4];
  double L[4], s = 0.0;
#pragma unroll
  for (int q = 0; q < 4; ++q) y[q] = 4 * lane + q < n ? g_of(x.w[q]) : 0.f;
  if (g) *reinterpret_cast<float4*>(g + 4 * lane) = make_float4(y[0], y[1], y[2], y[3]);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    s += (double)y[q];
    L[q] = s;
  }
  double up = s;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const double z = __shfl_up_sync(0xffffffffu, up, m);
    if (lane >= m) up += z;
  }
  const double before = up - s;      // sums of the lanes before
  constexpr double LOG2E64 = 1.4426950408889634;
#pragma unroll
  for (int q = 0; q < 4; ++q) L[q] = (L[q] + before) * LOG2E64;      // in units of log 2 from here on
  // Prefix sums up to the ends of the blocks of 32 tokens; a token's distances to the start and to the end of its own block are all the exponentials it
  // takes, the others are these times the blocks' own.
  const double e0 = __shfl_sync(0xffffffffu, L[3], 7), e1 = __shfl_sync(0xffffffffu, L[3], 15), e2 = __shfl_sync(0xffffffffu, L[3], 23),
               e3 = __shfl_sync(0xffffffffu, L[3], 31);
  const int I = lane >> 3;
  const double from = I == 0 ? 0.0 : I == 1 ? e0 : I == 2 ? e1 : e2, to = I == 0 ? e0 : I == 1 ? e1 : I == 2 ? e2 : e3;
  float in[4], low[4], row[4], tail[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const double z = L[q] - from;
    in[q] = (float)z;
    low[q] = (float)(z - (double)in[q]);
    row[q] = ex2(in[q]);
    tail[q] = ex2((float)(to - L[q]));
  }
  const float head = ex2((float)from), rest = ex2((float)(e3 - to));      // of the tokens before, behind this block
  const float gap1 = ex2((float)(e1 - e0)), gap2 = ex2((float)(e2 - e1));
  // from the end of this block to the start of block 1, 2, 3 (those behind it)
  const float c1 = 1.f, c2 = I == 0 ? gap1 : 1.f, c3 = I == 0 ? gap1 * gap2 : I == 1 ? gap2 : 1.f;
  const auto put = [&](float* p, const float (&v)[4], float f) {
    *reinterpret_cast<float4*>(p + 4 * lane) = make_float4(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
  };
  put(d.start, row, head);
  put(d.end, tail, rest);
  put(d.row, row, 1.f);
  put(d.in, in, 1.f);
  put(d.in_lo, low, 1.f);
  put(d.col[0], tail, c1);
  put(d.col[1], tail, c2);
  put(d.col[2], tail, c3);
  if (lane == 0) d.all = ex2((float)e3);
}

// 16 factors of a row of a diagonal block, columns first .. first + 15: e^{L_i - L_j} (those above the diagonal mean nothing).
__device__ __forceinline__ void diagonal_factors(const Decays& d, int row, int first, float (&f)[16]) {
  const float hi = d.in[row], lo = d.in_lo[row];
#pragma unroll
  for (int j = 0; j < 16; j += 4) {
    const float4 h = *reinterpret_cast<const float4*>(d.in + first + j), l = *reinterpret_cast<const float4*>(d.in_lo + first + j);
    f[j] = ex2((hi - h.x) + (lo - l.x)); f[j + 1] = ex2((hi - h.y) + (lo - l.y));
    f[j + 2] = ex2((hi - h.z) + (lo - l.z)); f[j + 3] = ex2((hi - h.w) + (lo - l.w));
  }
}
// and of a block I below the diagonal
__device__ __forceinline__ void block_factors(const Decays& d, int row, int I, int first, float (&f)[16]) {
  const float fr = d.row[row];
#pragma unroll
  for (int j = 0; j < 16; j += 4) {
    const float4 g = *reinterpret_cast<const float4*>(d.col[I - 1] + first + j);
    f[j] = fr * g.x; f[j + 1] = fr * g.y; f[j + 2] = fr * g.z; f[j + 3] = fr * g.w;
  }
}

// The kept states are [unit][chunk][4096] in an order of their own: what the 16 lanes that hold 16 rows read or write at once lies together.  Offset of
// columns 4 c .. 4 c + 3 of row 16 wq + l.
__device__ __forceinline__ int kept_at(int c, int wq, int l) { return ((c * 4 + wq) * 16 + l) * 4; }

// 16 results of a row to memory as bfloat16: the last rows of a sequence of a packed batch, behind which the next one's lie.  Whole chunks are staged in
// shared memory and leave by TMA: an SM gets rid of some 16 bytes a cycle, and the threads do not wait for that.
__device__ __forceinline__ void store_row16(bf16* p, const float (&y)[16]) {
#pragma unroll
  for (int j = 0; j < 16; j += 8)
    *reinterpret_cast<uint4*>(p + j) = make_uint4(pack_bf16(y[j], y[j + 1]), pack_bf16(y[j + 2], y[j + 3]), pack_bf16(y[j + 4], y[j + 5]),
                                                  pack_bf16(y[j + 6], y[j + 7]));
}

// Stretches of the units of a call: parts of `per` chunks.  What a part starts from is put together from what the parts before it (backward: behind it) add to
// the state; that is found by a pass of its own over those, each in `sub` pieces of `per_sub` chunks, as there are more SMs than parts.
struct Cut {
  int n_units, parts, per, sub, per_sub;
  __host__ __device__ int adds() const { return (parts - 1) * sub; }      // of a unit
  bool chained() const { return adds() > 12; }      // put together by a kernel of its own; otherwise by each part, at its start
};
struct Stretch { int unit, part, n, h, len, NT, lo, hi; };
// PACKED: the units of up to RANKED sequences in the order of their lengths, the longest first: a unit that starts last then is a short one.  Every CTA finds
// the order by itself, a thread to a sequence that compares it with all others, and pays for that before its first chunk.  Forward and backward, lengths
// of 1 to 4000 with a median of 30, in the order of lengths and as they come: 16 sequences of 32 heads 97 and 120 us, 48 of 8 heads 75 and 87, of 32 heads 214
// and 207, 96 of 32 heads 429 and 392, 256 of 32 heads 1273 and 940.  All threads call it; `slot` is shared memory.
constexpr int RANKED = 64;
template <bool PACKED>
__device__ __forceinline__ Stretch unit_of(const Tokens& t, const Cut& cut, int* slot) {
  Stretch x;
  x.unit = blockIdx.x % cut.n_units; x.part = blockIdx.x / cut.n_units;
  x.n = x.unit / t.H; x.h = x.unit % t.H;
  if (PACKED && t.n_seq <= RANKED) {
    const int me = threadIdx.x;
    if (me < t.n_seq) {
      const int len = __ldg(t.len + me);
      int place = 0;
      for (int q = 0; q < t.n_seq; ++q) {
        const int other = __ldg(t.len + q);
        place += other > len || (other == len && q < me);
      }
      if (place == x.n) *slot = me;
    }
    __syncthreads();
    x.n = *slot;
    x.unit = x.n * t.H + x.h;
  }
  x.len = t.length(x.n);
  x.NT = (x.len + CT - 1) / CT;
  return x;
}
template <bool PACKED>
__device__ __forceinline__ Stretch stretch_of(const Tokens& t, const Cut& cut, int* slot) {
  Stretch x = unit_of<PACKED>(t, cut, slot);
  x.lo = min(x.part * cut.per, x.NT);
  x.hi = min(x.lo + cut.per, x.NT);
  return x;
}
// a piece of the pass that adds: `part` counts the pieces of a unit, in the order of the chunks
template <bool PACKED>
__device__ __forceinline__ Stretch piece_of(const Tokens& t, const Cut& cut, bool reverse, int* slot) {
  Stretch x = unit_of<PACKED>(t, cut, slot);
  const int p = x.part / cut.sub + reverse, s = x.part % cut.sub;
  x.lo = min(p * cut.per + s * cut.per_sub, x.NT);
  x.hi = min(min(x.lo + cut.per_sub, (p + 1) * cut.per), x.NT);
  return x;
}

// Memory of a call that has parts: what the pieces add [unit][adds] and their decays, and (chained) what the parts start from [unit][parts].  All states in the order of
// kept_at().
struct Pieces { float *add, *start, *decay; };
inline size_t pieces_bytes(const Cut& c) {
  if (c.parts == 1) return 0;
  return ((size_t)c.n_units * (c.adds() + (c.chained() ? c.parts : 0)) * 4096 + (size_t)c.n_units * c.adds()) * 4;
}
inline Pieces pieces_at(void* p, const Cut& c) {
  Pieces x;
  x.add = static_cast<float*>(p);
  x.start = x.add + (size_t)c.n_units * c.adds() * 4096;
  x.decay = x.start + (size_t)c.n_units * (c.chained() ? c.parts : 0) * 4096;
  return x;
}
// The state that a part of a unit starts from (reverse: its gradient behind the part): N / 4 pieces of four columns of a row from c0 on.
template <int N>
__device__ __forceinline__ void start_of(float (&S)[N], const Stretch& x, const Cut& cut, bool reverse, bool chained, const float* add, const float* start,
                                         const float* decay, const float* first, int c0, int wq, int lane) {
  const bool have = lane < 16;      // (the lanes that hold a row)
  if (x.part == (reverse ? cut.parts - 1 : 0) || !chained) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const float4 f = have && first ? __ldcg(reinterpret_cast<const float4*>(first + (16 * wq + lane) * 64 + 4 * c0 + j)) : make_float4(0.f, 0.f, 0.f, 0.f);
      S[j] = f.x; S[j + 1] = f.y; S[j + 2] = f.z; S[j + 3] = f.w;
    }
    const int n = reverse ? (cut.parts - 1 - x.part) * cut.sub : x.part * cut.sub;
    for (int i = 0; i < n; ++i) {
      const int a = x.unit * cut.adds() + (reverse ? cut.adds() - 1 - i : i);
      const float d = __ldcg(decay + a);
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        const float4 f = have ? __ldcg(reinterpret_cast<const float4*>(add + (long long)a * 4096 + kept_at(c0 + j / 4, wq, lane))) : make_float4(0.f, 0.f, 0.f, 0.f);
        S[j] = fmaf(d, S[j], f.x); S[j + 1] = fmaf(d, S[j + 1], f.y); S[j + 2] = fmaf(d, S[j + 2], f.z); S[j + 3] = fmaf(d, S[j + 3], f.w);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const float4 f = have ? __ldcg(reinterpret_cast<const float4*>(start + (long long)(x.unit * cut.parts + x.part) * 4096 + kept_at(c0 + j / 4, wq, lane)))
                            : make_float4(0.f, 0.f, 0.f, 0.f);
      S[j] = f.x; S[j + 1] = f.y; S[j + 2] = f.z; S[j + 3] = f.w;
    }
  }
}

// rows n .. 127 of a chunk's token tile (they belong to the next sequence of a packed batch) as zeros
__device__ __forceinline__ void zero_rows(unsigned char* tile, int n) {
  for (int i = n * 8 + threadIdx.x; i < CT * 8; i += blockDim.x) *reinterpret_cast<uint4*>(tile + 16 * i) = make_uint4(0, 0, 0, 0);
}

Cut cut_units(int n_seq, int max_len, int H, bool backward);
// what the pieces add, and (chained) what the parts start from; values v and keys k, or backwards d_o and r
int launch_pieces(const Args& a, const Cut& cut, const CUtensorMap& map_val, const CUtensorMap& map_key, const Pieces& p, bool reverse, int* status,
                  cudaStream_t st);

}  // namespace la
}  // namespace rwkvb200
