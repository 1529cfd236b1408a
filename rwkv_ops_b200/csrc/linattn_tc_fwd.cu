// Linear attention with a decay for each head, forward on tcgen05: bfloat16 tokens, head size 64 (linattn_tc.cuh).
#include <algorithm>
#include <type_traits>

#include "linattn_tc.cuh"

namespace rwkvb200 {
namespace la {
namespace {

constexpr int NTHR = 256;
// The two warps that have no block of A on or below the diagonal issue products and copies, and make the next chunk's decays.
constexpr int ISSUE = 5, DECAYS = 4;

struct FwdSmem {
  unsigned char r[TOK_BYTES], k[TOK_BYTES], v[TOK_BYTES];      // k and r become the first and the third part of e^{Lc - L_j} k_j
  unsigned char klo[TOK_BYTES];       // the second
  unsigned char A[2][TOK_BYTES];      // A [token i][token j], two times 64 columns; the first half stages o afterwards
  unsigned char S[TILE_BYTES];        // the state before the chunk, [v][k], rounded
  Decays dec[2];
  uint64_t bar_in, bar_1, bar_2;
  uint32_t tmem_base;
  int sequence;
};
struct AddSmem {      // keys and values alone: three CTAs to an SM
  unsigned char k[TOK_BYTES], v[TOK_BYTES], klo[TOK_BYTES], r[TOK_BYTES];      // (r: the third part alone)
  Decays dec[2];
  uint64_t bar_in, bar_1, bar_2;
  uint32_t tmem_base;
  int sequence;
};
constexpr uint32_t TM_S = 0, TM_O2 = 0, TM_O1 = 128;

// One item: the chunks of a stretch in order, the state in registers (a row to the lower half lanes of a warp, 32 columns).  Per chunk two batches of
// products with the threads' work between them:
//   r k^T, r S^T            meanwhile the keys are scaled and split
//   A v, v^T (scaled keys)  after A = (r k^T) * decays has been rounded and stored; then o and the next state
// ADD: keys and values alone, from a zero state; what the piece adds and its decay go to `add` and `decay`.  REV: the same for the
// gradient of the state, from the last chunk to the first, with r for keys and d_o for values.
// Two CTAs share an SM (113 KB each, 256 TMEM columns each), so that one's products and loads run under the other's arithmetic.
//
// What bounds it: the steps of a chunk in turn, products, TMEM reads, the threads' rounding and storing, 4.5 us with two CTAs to an SM, 5 with states kept (tensor pipe 22 % of the
// cycles, issue slots 30 %); memory a third below a copy's rate.  Measured, H 32: training of B 8 x T 4096, states kept, 160 us for 671 MB (4.2 TB/s); inference of
// B 4 x T 16384 386 us, 95 of them in the pass over keys and values, for 1086 MB without that pass.
template <bool PACKED, bool ADD, bool REV = false>
__global__ void __launch_bounds__(NTHR, ADD ? 3 : 2)
la_tc_fwd_kernel(const float* __restrict__ w, const float* __restrict__ h0, int n_state, bf16* __restrict__ o, float* __restrict__ ht,
                 float* __restrict__ states, float* __restrict__ add, const float* __restrict__ start, float* __restrict__ decay, int chained,
                 const __grid_constant__ CUtensorMap map_r, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                 const __grid_constant__ CUtensorMap map_o, Tokens tok, Cut cut, int* status) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  typedef std::conditional_t<ADD, AddSmem, FwdSmem> Smem;
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  constexpr uint32_t TM_U = ADD ? 0 : 64, TM_COLS = ADD ? 64 : 256;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wq = warp & 3, half = warp >> 2, row = 32 * wq + lane;      // the token whose row this thread reads, and which half of the columns
  if (tid == 0) {
    mbar_init(&sm.bar_in, 1); mbar_init(&sm.bar_1, 1); mbar_init(&sm.bar_2, 1);
    fence_mbar_init();
  }
  if (tid == 32) tma_prefetch_maps(map_r, map_k, map_v, map_o);
  if (warp == 0) tmem_alloc(&sm.tmem_base, TM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  earlier_kernels_done();
  later_kernels_may_start();
  const uint32_t tm = sm.tmem_base;
  const Stretch x = ADD ? piece_of<PACKED>(tok, cut, REV, &sm.sequence) : stretch_of<PACKED>(tok, cut, &sm.sequence);
  const int seq0 = PACKED ? __ldg(tok.start + x.n) : 0, brow = PACKED ? 0 : x.n;
  const long long wb = tok.wbase(x.n, x.h), at = tok.base(x.n, x.h) + (long long)row * tok.st + 32 * half;      // of w; of this thread's part of a row
  auto rows_of = [&](int c) { return min(CT, x.len - c * CT); };
  auto load_in = [&](int c) {      // one thread
    const int t0 = seq0 + c * CT;
    mbar_expect_tx(&sm.bar_in, (ADD ? 2 : 3) * TOK_BYTES);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      tma_load_4d(sm.k + q * TILE_BYTES, &map_k, &sm.bar_in, 0, t0 + 64 * q, x.h, brow);
      if constexpr (!ADD) tma_load_4d(sm.r + q * TILE_BYTES, &map_r, &sm.bar_in, 0, t0 + 64 * q, x.h, brow);
      tma_load_4d(sm.v + q * TILE_BYTES, &map_v, &sm.bar_in, 0, t0 + 64 * q, x.h, brow);
    }
  };
  auto prefetch_in = [&](int c) {
    const int t0 = seq0 + c * CT;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      tma_prefetch_4d(&map_k, 0, t0 + 64 * q, x.h, brow);
      if constexpr (!ADD) tma_prefetch_4d(&map_r, 0, t0 + 64 * q, x.h, brow);
      tma_prefetch_4d(&map_v, 0, t0 + 64 * q, x.h, brow);
    }
  };
  // the state: lanes 0 .. 15 hold row v = 16 wq + lane, columns 32 half .. + 31
  const bool st_lane = lane < 16;
  const int srow = 16 * wq + (lane & 15);
  const long long sat = (long long)srow * 64 + 32 * half;
  float S[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) S[j] = 0.f;
  auto put_state = [&](float* to) {
#pragma unroll
    for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(to + sat + j) = make_float4(S[j], S[j + 1], S[j + 2], S[j + 3]);
  };
  auto put_kept = [&](float* to) {
#pragma unroll
    for (int j = 0; j < 8; ++j) *reinterpret_cast<float4*>(to + kept_at(8 * half + j, wq, lane)) = make_float4(S[4 * j], S[4 * j + 1], S[4 * j + 2], S[4 * j + 3]);
  };
  auto keep_state = [&](int c) { put_kept(states + (PACKED ? tok.first(x.n, x.h, 0) + c : (long long)x.unit * tok.NT + c) * 4096); };
  bool ok = true;
  float product = 1.f;
  const int n_chunks = x.hi - x.lo;
  auto chunk = [&](int i) { return REV ? x.hi - 1 - i : x.lo + i; };      // the i-th
  if (n_chunks > 0) {
    if (warp == ISSUE && elect_one()) load_in(chunk(0));
    if (warp == DECAYS) make_decays(sm.dec[0], load_w(tok, w, wb, chunk(0) * CT, rows_of(chunk(0))), rows_of(chunk(0)), nullptr);
    if constexpr (!ADD) {
      start_of(S, x, cut, false, chained, add, start, decay, h0 ? h0 + ((long long)(n_state == 1 ? 0 : x.n) * tok.H + x.h) * 4096 : nullptr, 8 * half, wq, lane);
      if (st_lane) {
        if (states) keep_state(x.lo);
        tile_store_row32(sm.S, srow, 32 * half, S);
      }
      // A above the diagonal of blocks: never written to again
      for (int e = tid; e < 2 * CT * 8; e += NTHR) *reinterpret_cast<uint4*>(sm.A[0] + 16 * e) = make_uint4(0, 0, 0, 0);
    }
    fence_async_smem();
    __syncthreads();
    for (int i = 0; i < n_chunks; ++i) {
      const int c = chunk(i);
      const uint32_t ph = i & 1;
      RawW raw;      // w of the next chunk
      if (warp == DECAYS && i + 1 < n_chunks) raw = load_w(tok, w, wb, chunk(i + 1) * CT, rows_of(chunk(i + 1)));
      const Decays& d = sm.dec[ph];
      const int n = rows_of(c);
      ok = mbar_wait(&sm.bar_in, ph, status, 501) && ok;
      if (PACKED && n < CT) {
        zero_rows(sm.k, n);
        zero_rows(sm.v, n);
        fence_async_smem();
        __syncthreads();
      }
      if constexpr (!ADD) {
        if (warp == ISSUE && elect_one()) {
          tc_fence_after();
          umma_tile<128, 128, 0, 0>(tmem_addr(tm, 0, TM_S), smem_u32(sm.r), smem_u32(sm.k), false);
          bulk_wait_read();            // o of the chunk before has left its place in A, which is written to after these products
          umma_tile<128, 64, 0, 0>(tmem_addr(tm, 0, TM_O1), smem_u32(sm.r), smem_u32(sm.S), false);
          umma_commit(&sm.bar_1);
        }
      }
      if (i + 1 < n_chunks && warp == ISSUE && elect_one()) prefetch_in(chunk(i + 1));
      // scaled keys, 32 columns of a token, in three parts; two wait until the products have read the keys and queries as they are
      uint4 hi[4], rest[4];
      {
        const float f = REV ? d.start[row] : d.end[row];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t off = (row >> 6) * TILE_BYTES + tile_chunk_off(row & 63, 4 * half + q);
          const uint4 u = *reinterpret_cast<const uint4*>(sm.k + off);
          const uint32_t in[4] = {u.x, u.y, u.z, u.w};
          uint32_t h[4], l[4], m[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float a = bf16_lo(in[e]) * f, b = bf16_hi(in[e]) * f;
            h[e] = pack_bf16(a, b);
            a -= bf16_lo(h[e]); b -= bf16_hi(h[e]);
            l[e] = pack_bf16(a, b);
            m[e] = pack_bf16(a - bf16_lo(l[e]), b - bf16_hi(l[e]));
          }
          hi[q] = make_uint4(h[0], h[1], h[2], h[3]);
          *reinterpret_cast<uint4*>(sm.klo + off) = make_uint4(l[0], l[1], l[2], l[3]);
          rest[q] = make_uint4(m[0], m[1], m[2], m[3]);
          if constexpr (ADD) {      // (no product reads them, and no other thread)
            *reinterpret_cast<uint4*>(sm.k + off) = hi[q];
            *reinterpret_cast<uint4*>(sm.r + off) = rest[q];
          }
        }
      }
      if constexpr (!ADD) {
        ok = mbar_wait(&sm.bar_1, ph, status, 502) && ok;
        tc_fence_after();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t off = (row >> 6) * TILE_BYTES + tile_chunk_off(row & 63, 4 * half + q);
          *reinterpret_cast<uint4*>(sm.k + off) = hi[q];
          *reinterpret_cast<uint4*>(sm.r + off) = rest[q];
        }
      }
      if constexpr (!ADD) {
        // A: blocks of 32 x 32 on and below the diagonal (warp: rows 32 wq .., columns 64 half ..)
        unsigned char* At = sm.A[half] + (row >> 6) * TILE_BYTES;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int J = 2 * half + b;
          if (J <= wq) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {      // 16 columns at a time: registers (a spilled one goes to L2, there is no L1 left)
              uint32_t s[16];
              float p[16];
              tmem_ld16(tmem_addr(tm, 32 * wq, TM_S + 32 * J + 16 * h), s);
              if (J < wq) {
                block_factors(d, row, wq, 32 * J + 16 * h, p);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) p[j] *= __uint_as_float(s[j]);
              } else {
                diagonal_factors(d, row, 32 * J + 16 * h, p);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) p[j] = 16 * h + j <= lane ? __uint_as_float(s[j]) * p[j] : 0.f;
              }
              tile_store_row<16>(At, row & 63, 32 * b + 16 * h, p);
            }
          } else if (J == 1) {      // (wq == 0: the staged o was here)
#pragma unroll
            for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(At + tile_chunk_off(row & 63, 4 * b + q)) = make_uint4(0, 0, 0, 0);
          }
        }
      }
      if (warp == DECAYS && i + 1 < n_chunks) make_decays(sm.dec[ph ^ 1], raw, rows_of(chunk(i + 1)), nullptr);
      fence_async_smem();
      tc_fence_before();
      __syncthreads();
      if (warp == ISSUE && elect_one()) {
        tc_fence_after();
        if constexpr (!ADD) {
          umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_O2), smem_u32(sm.A[0]), smem_u32(sm.v), false);
          umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_O2), smem_u32(sm.A[1]), smem_u32(sm.v) + TILE_BYTES, true);
        }
        umma_tile<64, 64, 1, 1, 8>(tmem_addr(tm, 0, TM_U), smem_u32(sm.v), smem_u32(sm.r), false);
        umma_tile<64, 64, 1, 1, 8>(tmem_addr(tm, 0, TM_U), smem_u32(sm.v), smem_u32(sm.klo), true);
        umma_tile<64, 64, 1, 1, 8>(tmem_addr(tm, 0, TM_U), smem_u32(sm.v), smem_u32(sm.k), true);
        umma_commit(&sm.bar_2);
      }
      ok = mbar_wait(&sm.bar_2, ph, status, 503) && ok;
      tc_fence_after();
      if (i + 1 < n_chunks && warp == ISSUE && elect_one()) load_in(chunk(i + 1));
      const float all = d.all;
      {
        uint32_t u[32];
        tmem_ld32(tmem_addr(tm, 32 * wq, TM_U + 32 * half), u);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) S[j] = fmaf(all, S[j], __uint_as_float(u[j]));
      }
      if constexpr (ADD) {
        product *= all;
      } else {
        if (st_lane) {
          tile_store_row32(sm.S, srow, 32 * half, S);
          if (states && c + 1 < x.hi) keep_state(c + 1);
        }
        const float f = d.start[row];
        bf16* to = o + at + (long long)(c * CT) * tok.st;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t a[16], b[16];
          tmem_ld16(tmem_addr(tm, 32 * wq, TM_O1 + 32 * half + 16 * h), a);
          tmem_ld16(tmem_addr(tm, 32 * wq, TM_O2 + 32 * half + 16 * h), b);
          tmem_ld_wait();
          float y[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) y[j] = fmaf(f, __uint_as_float(a[j]), __uint_as_float(b[j]));
          if (!o) continue;      // (the states alone)
          if (PACKED && n < CT) {
            if (row < n) store_row16(to + 16 * h, y);
          } else {
            tile_store_row<16>(sm.A[0] + (row >> 6) * TILE_BYTES, row & 63, 32 * half + 16 * h, y);
          }
        }
      }
      fence_async_smem();
      tc_fence_before();
      if (!__syncthreads_and(ok)) break;
      if constexpr (!ADD) {
        if (o && !(PACKED && n < CT) && warp == ISSUE && elect_one()) {
#pragma unroll
          for (int q = 0; q < 2; ++q)      // (rows past the end of the batch are clipped)
            if (64 * q < n) tma_store_4d(&map_o, sm.A[0] + q * TILE_BYTES, 0, seq0 + c * CT + 64 * q, x.h, brow);
          bulk_commit();
        }
      }
    }
  } else if (!ADD && st_lane) {      // no chunk: a sequence without tokens hands its state on
    if (x.part == 0 && h0) {
#pragma unroll
      for (int j = 0; j < 32; ++j) S[j] = h0[((long long)(n_state == 1 ? 0 : x.n) * tok.H + x.h) * 4096 + sat + j];
    }
  }
  if constexpr (ADD) {
    if (st_lane) put_kept(add + ((long long)x.unit * cut.adds() + x.part) * 4096);
    if (tid == 0) decay[x.unit * cut.adds() + x.part] = product;
  } else {
    if (st_lane && ht && (x.NT == 0 ? x.part == 0 : x.lo < x.hi && x.hi == x.NT)) put_state(ht + (long long)x.unit * 4096);
  }
  if (warp == ISSUE && elect_one()) bulk_wait_all();
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tm, TM_COLS);
}

// What the parts of a unit start from (reverse: the gradient behind them), from what the pieces add; four elements of a state to a thread.
__global__ void __launch_bounds__(256) la_chain_kernel(const float* __restrict__ add, const float* __restrict__ decay, float* __restrict__ start,
                                                       const float* __restrict__ first, int n_first, int H, Cut cut, int reverse) {
  earlier_kernels_done();
  later_kernels_may_start();
  const int i = blockIdx.x * 256 + threadIdx.x, unit = i >> 10, e = i & 1023;
  float4 S = make_float4(0.f, 0.f, 0.f, 0.f);
  if (first) {
    const int c = e >> 6, v = e & 63;      // columns 4 c .. of row v (kept_at)
    S = *reinterpret_cast<const float4*>(first + (n_first == 1 ? (long long)(unit % H) : (long long)unit) * 4096 + v * 64 + 4 * c);
  }
  const int n = cut.adds();
  const float* a0 = add + (long long)unit * n * 4096 + 4 * e;
  float* s0 = start + (long long)unit * cut.parts * 4096 + 4 * e;
  constexpr int AHEAD = 8;
  for (int q0 = 0; q0 < n; q0 += AHEAD) {
    float4 f[AHEAD];
    float d[AHEAD];
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      if (q0 + q < n) {
        const int a = reverse ? n - 1 - q0 - q : q0 + q;
        f[q] = *reinterpret_cast<const float4*>(a0 + (long long)a * 4096);
        d[q] = decay[unit * n + a];
      }
    }
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      if (q0 + q < n) {
        S.x = fmaf(d[q], S.x, f[q].x); S.y = fmaf(d[q], S.y, f[q].y);
        S.z = fmaf(d[q], S.z, f[q].z); S.w = fmaf(d[q], S.w, f[q].w);
        const int done = q0 + q + 1;
        if (done % cut.sub == 0) {
          const int p = done / cut.sub;      // parts behind the first (before the last) that this is the start of
          *reinterpret_cast<float4*>(s0 + (long long)(reverse ? cut.parts - 1 - p : p) * 4096) = S;
        }
      }
    }
  }
}

template <bool PACKED>
int fwd(const Args& a, cudaStream_t st) {
  const Tokens& t = a.tok;
  DeviceFacts f;
  if (int e = device_facts(&f)) return e;
  constexpr int smem = (int)sizeof(FwdSmem);
  static_assert(smem <= 115712, "two CTAs of 113 KB each share an SM");
  if (int e = need_aligned_smem<la_tc_fwd_kernel<PACKED, false>>(f)) return e;
  if (int e = allow_smem<la_tc_fwd_kernel<PACKED, false>>(f, smem)) return e;
  const int B = t.start ? 1 : t.n_seq, T = t.start ? (int)a.tokens : t.T, head_first = t.st == 64 && t.H > 1;
  CUtensorMap mr, mk, mv, mo;
  const void* r = a.r ? a.r : a.k;      // (the states alone: whatever r k^T is, it goes nowhere)
  if (int e = make_token_tensor_map(&mr, r, B, T, t.H, head_first)) return e;
  if (int e = make_token_tensor_map(&mk, a.k, B, T, t.H, head_first)) return e;
  if (int e = make_token_tensor_map(&mv, a.v, B, T, t.H, head_first)) return e;
  if (int e = make_token_tensor_map(&mo, a.o ? a.o : a.k, B, T, t.H, head_first)) return e;
  const Cut cut = cut_units(t.n_seq, t.T, t.H, false);
  const Pieces p = pieces_at(a.scratch, cut);
  if (cut.parts > 1) {
    if (int e = launch_pieces(a, cut, mv, mk, p, false, f.status, st)) return e;
  }
  ProfScope prof("linattn_tc_fwd_kernel", st);
  return launch(la_tc_fwd_kernel<PACKED, false>, cut.n_units * cut.parts, NTHR, smem, st, 1, a.w, a.h0, a.n_state, (bf16*)a.o, a.ht, a.states, p.add,
                (const float*)p.start, p.decay, (int)cut.chained(), mr, mk, mv, mo, t, cut, f.status);
}

}  // namespace

int launch_pieces(const Args& a, const Cut& cut, const CUtensorMap& map_val, const CUtensorMap& map_key, const Pieces& p, bool reverse, int* status,
                  cudaStream_t st) {
  DeviceFacts f;
  if (int e = device_facts(&f)) return e;
  constexpr int smem = (int)sizeof(AddSmem);
  const auto go = [&](auto packed, auto rev) {
    constexpr bool PACKED = decltype(packed)::value, REV = decltype(rev)::value;
    if (int e = need_aligned_smem<la_tc_fwd_kernel<PACKED, true, REV>>(f)) return e;
    if (int e = allow_smem<la_tc_fwd_kernel<PACKED, true, REV>>(f, smem)) return e;
    ProfScope prof("linattn_tc_add_kernel", st);
    return launch(la_tc_fwd_kernel<PACKED, true, REV>, cut.n_units * cut.adds(), NTHR, smem, st, 1, a.w, (const float*)nullptr, 0, (bf16*)nullptr,
                  (float*)nullptr, (float*)nullptr, p.add, (const float*)nullptr, p.decay, 0, map_key, map_key, map_val, map_key, a.tok, cut, status);
  };
  const std::true_type yes;
  const std::false_type no;
  if (int e = a.tok.start ? (reverse ? go(yes, yes) : go(yes, no)) : (reverse ? go(no, yes) : go(no, no))) return e;
  if (!cut.chained()) return RWKVB200_OK;
  ProfScope prof("linattn_chain_kernel", st);
  return launch(la_chain_kernel, cut.n_units * 4, 256, 0, st, 1, (const float*)p.add, (const float*)p.decay, p.start, reverse ? a.d_ht : a.h0,
                reverse ? a.tok.n_seq : a.n_state, a.tok.H, cut, (int)reverse);
}

// How many parts and pieces: the least time by an estimate of 4.2 us for a chunk where two CTAs share an SM, 2.8 alone (backward 5.4, one to an SM), 2.6 for a
// chunk of the pass over keys and values, and 4 for its launch and what the parts start from.  Measured are 4.5, 3.2 and (backward) 5.4 to 6, 4 where three CTAs of that
// pass share an SM, and about one for each piece before a part's start: the estimate is low, more so for several parts.  What it is for holds: with the number of parts
// forced, 8 to 256 units of 1000 to 16384 tokens, its choice was the fastest, or 4 % from it (128 units of 4096 tokens: 113 us in two parts, 109 in one; of
// 16384 tokens 385 in two, 416 in one; 32 units of 16384 tokens 141 in nine, 406 in one).
Cut cut_units(int n_seq, int max_len, int H, bool backward) {
  constexpr int SMS = 148;      // of a B200
  const int NT = (max_len + CT - 1) / CT, units = n_seq * H, slots = backward ? SMS : 2 * SMS;
  Cut best = {units, 1, NT, 1, NT};
  double least = 1e30;
  for (int parts = 1; parts <= NT && (parts == 1 || (long long)units * parts <= slots); ++parts) {
    Cut c = {units, parts, (NT + parts - 1) / parts, 1, 0};
    if ((NT + c.per - 1) / c.per != parts) continue;      // (the same stretches as with fewer)
    c.sub = parts == 1 ? 1 : std::max(1, std::min(c.per, 3 * SMS / (units * (parts - 1))));
    c.per_sub = (c.per + c.sub - 1) / c.sub;
    c.sub = (c.per + c.per_sub - 1) / c.per_sub;
    const long long items = (long long)units * parts;
    const double waves = (double)((items + slots - 1) / slots);
    const double t = waves * c.per * (backward ? 5.4 : items > SMS ? 4.2 : 2.8) + (parts > 1 ? 4 + 2.6 * c.per_sub : 0);
    if (t < least) { least = t; best = c; }
  }
  return best;
}

size_t tc_states_bytes(int n_seq, int max_len, int total, int H, bool keep) {
  return keep ? (size_t)chunk_slots(n_seq, max_len, total, CT) * H * 4096 * 4 : 0;
}

size_t tc_scratch_bytes(int n_seq, int max_len, int H, bool w_per_head, bool backward) {
  const Cut c = cut_units(n_seq, max_len, H, backward);
  size_t n = pieces_bytes(c);
  if (backward && w_per_head) n = (n + 255) / 256 * 256 + ((size_t)n_seq * c.parts * H * 4 + 255) / 256 * 256 + (size_t)DW_PARTS * H * 8;
  return n;
}

int launch_tc_fwd(const Args& a, cudaStream_t st) {
  Args b = a;
  set_chunks(b, CT);
  return a.tok.start ? fwd<true>(b, st) : fwd<false>(b, st);
}

}  // namespace la
}  // namespace rwkvb200
