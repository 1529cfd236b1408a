// Linear attention with a decay for each head, backward on tcgen05: bfloat16 tokens, head size 64 (linattn_tc.cuh).
#include <algorithm>

#include "linattn_tc.cuh"

namespace rwkvb200 {
namespace la {
namespace {

constexpr int NTHR = 512, NWARP = NTHR / 32;

struct BwdSmem {
  unsigned char r[TOK_BYTES], k[TOK_BYTES], v[TOK_BYTES], d_o[TOK_BYTES];
  unsigned char rhi[TOK_BYTES], rlo[TOK_BYTES];      // e^{L_i} r_i, of which the third part takes the place of v; dr and dk are staged here afterwards
  unsigned char A[2][TOK_BYTES], E[2][TOK_BYTES];    // [token i][token j], two times 64 columns; dv is staged in the halves that are zero, see stage_v
  unsigned char S[3][TILE_BYTES], dS[2][TILE_BYTES]; // the state before the chunk and the gradient of the one after it in three parts, [v][k] (the last: see dS3)
  Decays dec[2];
  float g[3][CT], decay[3];      // g and e^{Lc} of this chunk, the next one (being made) and the one before (whose dw is)
  double dw_sum[32];
  // What the pairs of a 32 x 32 block (I, J) of tokens add to dg_t (M = A_ij (d_o_i . v_j)): near[I][J]: for t in J, the sum over j < t (I > J: all rows i; I == J:
  // rows i >= t); far[I][J]: for t in I, the sum over rows i >= t; and all of it for t between.
  float near[2][4][4][32], far[2][4][4][32], all[2][4][4];
  float t1[2][4][CT], t2[2][4][CT], t3[2][NWARP];
  uint64_t bar_in, bar_1, bar_x, bar_2;      // rows are here; products are done
  uint64_t bar_ae, bar_r, bar_read;          // of all warps: A and E are stored; the scaled r is; r and k have been read
  uint64_t bar_free;                         // the staged gradients have left
  uint32_t tmem_base;
  int sequence;
};
// The warps whose block of pairs lies above the diagonal (4, 8, 9, 12, 13, 14) do the other jobs: ISSUE the products (a thread that issues is held up by those
// under way, some 50 cycles each), STORE the copies of the gradients, DECAYS the next chunk's decays, DW the dw of the chunk before and (LOAD) the loads.
constexpr int ISSUE = 14, STORE = 4, DECAYS = 8, LOAD = 12, DW = 12, ISSUE_W = 9;
constexpr uint32_t TM_S = 0, TM_P = 128, TM_YR = 0, TM_YK = 64, TM_YV = 128, TM_XR = 256, TM_XK = 320, TM_XV = 384, TM_W = 448, TM_COLS = 512;

// the sum over a warp's lanes of x[c], in lanes c and c + 16
__device__ __forceinline__ float column_sum(float (&x)[16], int lane) {
#pragma unroll
  for (int m = 8; m >= 1; m >>= 1) {
    const bool up = lane & m;
#pragma unroll
    for (int c = 0; c < m; ++c) {
      const float send = up ? x[c] : x[c + m], keep = up ? x[c + m] : x[c];
      x[c] = keep + __shfl_xor_sync(0xffffffffu, send, m);
    }
  }
  return x[0] + __shfl_xor_sync(0xffffffffu, x[0], 16);
}
// 16 values of a row, columns col0 .. (a multiple of 8), as the tiles of their three bfloat16 parts
__device__ __forceinline__ void store_split16(unsigned char (*hi_lo)[TILE_BYTES], unsigned char* third, int row, int col0, const float* x) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t h[4], l[4], m[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float a = x[8 * c + 2 * e], b = x[8 * c + 2 * e + 1];
      h[e] = pack_bf16(a, b);
      a -= bf16_lo(h[e]); b -= bf16_hi(h[e]);
      l[e] = pack_bf16(a, b);
      m[e] = pack_bf16(a - bf16_lo(l[e]), b - bf16_hi(l[e]));
    }
    const uint32_t off = tile_chunk_off(row, (col0 >> 3) + c);
    *reinterpret_cast<uint4*>(hi_lo[0] + off) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(hi_lo[1] + off) = make_uint4(l[0], l[1], l[2], l[3]);
    *reinterpret_cast<uint4*>(third + off) = make_uint4(m[0], m[1], m[2], m[3]);
  }
}

// One item: the chunks of a stretch from the last to the first, the gradient of the state in registers.  Per chunk two batches of products:
//   r k^T, d_o v^T; d_o S, v dS, k dS^T     the first two are waited for, the others run on while A and E are made of them (all but where the third part of dS is)
//   E k, E^T r, A^T d_o; d_o^T (scaled r)   after A and E have been stored; meanwhile the states' part of dw
// then the three gradients are put together and staged, and leave while the next chunk is worked on.
// Sixteen warps, one CTA to an SM (all of TMEM, 226 KB): warp w reads token rows 32 (w % 4) .. and a quarter of the columns; the six warps whose block of pairs lies
// above the diagonal clear it and do the single-thread jobs, the next chunk's decays and the dw of the chunk before.  Within a chunk warps wait for products
// and rows only, and the issuing threads for the warps; all warps meet once, at its end.
//
// What bounds it: the chain of a chunk's steps, products, TMEM reads, rounding and storing, products, with one CTA to wait in.  No unit is near its limit (tensor pipe
// 27 % of the cycles, issue slots 43 %; shared memory moves some 800 KB a chunk, 6k of 11k cycles at 128 bytes each), and leaving out the
// column sums, the stores of A and E, or the copies of the gradients changes a chunk by less than 6 %.  Measured: B 8 x T 4096, H 32, 390 us for 1.07 GB
// (2.7 TB/s; 365 with the states in two parts: products 10, splitting and storing 6 in a chunk's last step, waiting 9); 256 items on 148 SMs are two waves.
template <bool PACKED>
__global__ void __launch_bounds__(NTHR, 1)
la_tc_bwd_kernel(const float* __restrict__ w, const float* __restrict__ d_ht, const float* __restrict__ states, bf16* __restrict__ dr,
                 bf16* __restrict__ dk, bf16* __restrict__ dv, float* __restrict__ dw, int dw_parts, float* __restrict__ dh0,
                 const float* __restrict__ add, const float* __restrict__ start, const float* __restrict__ decay, int chained,
                 const __grid_constant__ CUtensorMap map_r, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                 const __grid_constant__ CUtensorMap map_dr, const __grid_constant__ CUtensorMap map_dk, const __grid_constant__ CUtensorMap map_dv,
                 Tokens tok, Cut cut, int* status) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  BwdSmem& sm = *reinterpret_cast<BwdSmem*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wq = warp & 3, qt = warp >> 2, row = 32 * wq + lane;
  if (tid == 0) {
    mbar_init(&sm.bar_in, 1); mbar_init(&sm.bar_1, 1); mbar_init(&sm.bar_x, 1); mbar_init(&sm.bar_2, 2);
    mbar_init(&sm.bar_ae, NWARP); mbar_init(&sm.bar_read, NWARP); mbar_init(&sm.bar_free, 1); mbar_init(&sm.bar_r, NWARP);
    fence_mbar_init();
  }
  if (tid == 32) tma_prefetch_maps(map_r, map_k, map_v, map_do, map_dr, map_dk, map_dv);
  if (warp == 0) tmem_alloc(&sm.tmem_base, TM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  earlier_kernels_done();
  later_kernels_may_start();
  const uint32_t tm = sm.tmem_base;
  const Stretch x = stretch_of<PACKED>(tok, cut, &sm.sequence);
  const int seq0 = PACKED ? __ldg(tok.start + x.n) : 0, brow = PACKED ? 0 : x.n;
  const long long wb = tok.wbase(x.n, x.h), at = tok.base(x.n, x.h) + (long long)row * tok.st + 16 * qt;      // of w; of this thread's part of a row
  auto rows_of = [&](int c) { return min(CT, x.len - c * CT); };
  auto load_in = [&](int c) {      // one thread
    const int t0 = seq0 + c * CT;
    mbar_expect_tx(&sm.bar_in, 4 * TOK_BYTES);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      tma_load_4d(sm.r + q * TILE_BYTES, &map_r, &sm.bar_in, 0, t0 + 64 * q, x.h, brow);
      tma_load_4d(sm.k + q * TILE_BYTES, &map_k, &sm.bar_in, 0, t0 + 64 * q, x.h, brow);
      tma_load_4d(sm.d_o + q * TILE_BYTES, &map_do, &sm.bar_in, 0, t0 + 64 * q, x.h, brow);
      tma_load_4d(sm.v + q * TILE_BYTES, &map_v, &sm.bar_in, 0, t0 + 64 * q, x.h, brow);
    }
  };
  auto kept_slot = [&](int c) { return PACKED ? tok.first(x.n, x.h, 0) + c : (long long)x.unit * tok.NT + c; };
  auto prefetch_in = [&](int c) {
    const int t0 = seq0 + c * CT;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      tma_prefetch_4d(&map_r, 0, t0 + 64 * q, x.h, brow);
      tma_prefetch_4d(&map_k, 0, t0 + 64 * q, x.h, brow);
      tma_prefetch_4d(&map_do, 0, t0 + 64 * q, x.h, brow);
      tma_prefetch_4d(&map_v, 0, t0 + 64 * q, x.h, brow);
    }
    bulk_prefetch_l2(states + kept_slot(c) * 4096, 4096 * 4);
  };
  auto stage_v = [&](int tile) { return tile ? sm.E[1] : sm.A[1]; };      // 64 rows of dv: rows 0 .. 63 of the right halves, all above the diagonal
  auto store_out = [&](int c) {      // the staged gradients of a chunk
    const int n = rows_of(c), t0 = seq0 + c * CT;
    if (PACKED && n < CT) return;      // (they were not staged)
#pragma unroll
    for (int q = 0; q < 2; ++q) {      // (rows past the end of the batch are clipped)
      if (64 * q < n) {
        tma_store_4d(&map_dv, stage_v(q), 0, t0 + 64 * q, x.h, brow);
        tma_store_4d(&map_dr, sm.rhi + q * TILE_BYTES, 0, t0 + 64 * q, x.h, brow);
        tma_store_4d(&map_dk, sm.rlo + q * TILE_BYTES, 0, t0 + 64 * q, x.h, brow);
      }
    }
    bulk_commit();
  };
  // a warp's part of a step is done: what it wrote may be read by products and copies, what it read overwritten
  auto arrive = [&](uint64_t& bar) {
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar);
  };
  // states: lanes 0 .. 15 hold row v = 16 wq + lane, columns 16 qt .. + 15
  const bool st_lane = lane < 16;
  const int srow = 16 * wq + (lane & 15);
  const long long sat = (long long)srow * 64 + 16 * qt;
  float dS[16], S0[16];
  auto get_kept = [&](int c) {
    const float* from = states + kept_slot(c) * 4096;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 f = st_lane ? __ldcg(reinterpret_cast<const float4*>(from + kept_at(4 * qt + j, wq, lane))) : make_float4(0.f, 0.f, 0.f, 0.f);
      S0[4 * j] = f.x; S0[4 * j + 1] = f.y; S0[4 * j + 2] = f.z; S0[4 * j + 3] = f.w;
    }
  };
  // The third part of the gradient lies where the last rows' left half of E comes later: that of the chunk before has been read, that of this one is stored after the
  // products with the states.
  unsigned char* dS3 = sm.E[0] + TILE_BYTES;
  // the gradient of a chunk's state into its tiles, and its product with the state
  auto put_tiles = [&](int ph) {
    float s = 0.f;
    if (st_lane) {
      store_split16(sm.dS, dS3, srow, 16 * qt, dS);
#pragma unroll
      for (int j = 0; j < 16; ++j) s = fmaf(S0[j], dS[j], s);
    }
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    if (lane == 0) sm.t3[ph][warp] = s;
  };
  start_of(dS, x, cut, true, chained, add, start, decay, d_ht ? d_ht + (long long)x.unit * 4096 : nullptr, 4 * qt, wq, lane);
  bool ok = true;
  if (warp == DW) sm.dw_sum[lane] = 0.0;
  // dw of chunk c, the i-th of the stretch, by one warp: four tokens to a lane
  auto write_dw = [&](int c, int i) {
    const int I = lane >> 3, at = 4 * (lane & 7), n = rows_of(c), ph = i & 1;
    float t3 = lane < NWARP ? sm.t3[ph][lane] : 0.f;
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) t3 += __shfl_xor_sync(0xffffffffu, t3, m);
    t3 = sm.decay[i % 3] * __shfl_sync(0xffffffffu, t3, 0);
    const auto add4 = [](float (&to)[4], const float* p) {
      const float4 f = *reinterpret_cast<const float4*>(p);
      to[0] += f.x; to[1] += f.y; to[2] += f.z; to[3] += f.w;
    };
    float dg[4] = {t3, t3, t3, t3}, after[4] = {0.f, 0.f, 0.f, 0.f}, before[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      if (a >= I) add4(dg, &sm.near[ph][a][I][at]);
      else add4(dg, &sm.far[ph][I][a][at]);
      add4(after, &sm.t1[ph][a][4 * lane]);
      add4(before, &sm.t2[ph][a][4 * lane]);
    }
    float over = 0.f;      // blocks of pairs on both sides of this one
#pragma unroll
    for (int a = 2; a < 4; ++a)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (e < I && I < a) over += sm.all[ph][a][e];
    const float sa = (after[0] + after[1]) + (after[2] + after[3]), sb = (before[0] + before[1]) + (before[2] + before[3]);
    float down = sa, up = sb;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const float a = __shfl_down_sync(0xffffffffu, down, m), e = __shfl_up_sync(0xffffffffu, up, m);
      if (lane + m < 32) down += a;
      if (lane >= m) up += e;
    }
    const float later = __shfl_down_sync(0xffffffffu, down, 1), earlier = __shfl_up_sync(0xffffffffu, up, 1);      // of the lanes behind, before
    float behind = (lane < 31 ? later : 0.f) + over, ahead = lane ? earlier : 0.f;
#pragma unroll
    for (int q = 3; q >= 0; --q) { behind += after[q]; dg[q] += behind; }
    const float4 g4 = *reinterpret_cast<const float4*>(&sm.g[i % 3][4 * lane]);
    const float g[4] = {g4.x, g4.y, g4.z, g4.w};
    float part = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float y = (dg[q] + ahead) * g[q];
      ahead += before[q];
      if (4 * lane + q < n) {
        if (dw_parts) part += y;
        else dw[wb + (long long)(c * CT + 4 * lane + q) * tok.wst] = y;
      }
    }
    if (dw_parts) sm.dw_sum[lane] += (double)part;
  };
  if (x.lo < x.hi) {
    if (warp == LOAD && elect_one()) load_in(x.hi - 1);
    if (warp == DECAYS) {
      make_decays(sm.dec[0], load_w(tok, w, wb, (x.hi - 1) * CT, rows_of(x.hi - 1)), rows_of(x.hi - 1), sm.g[0]);
      if (lane == 0) sm.decay[0] = sm.dec[0].all;
    }
    get_kept(x.hi - 1);
    if (st_lane) store_split16(sm.S, sm.S[2], srow, 16 * qt, S0);
    put_tiles(0);
    fence_async_smem();
    __syncthreads();
    for (int c = x.hi - 1; c >= x.lo; --c) {
      const int i = x.hi - 1 - c;
      const uint32_t ph = i & 1;
      RawW raw;      // w of the next chunk
      if (warp == DECAYS && c > x.lo) raw = load_w(tok, w, wb, (c - 1) * CT, CT);
      const Decays& d = sm.dec[ph];
      const int n = rows_of(c);
      ok = mbar_wait(&sm.bar_in, ph, status, 511) && ok;
      if (PACKED && n < CT) {
        zero_rows(sm.r, n);
        zero_rows(sm.k, n);
        zero_rows(sm.v, n);
        zero_rows(sm.d_o, n);
        fence_async_smem();
        __syncthreads();
      }
      if (warp == ISSUE && elect_one()) {
        tc_fence_after();
        umma_tile<128, 128, 0, 0>(tmem_addr(tm, 0, TM_S), smem_u32(sm.r), smem_u32(sm.k), false);
        umma_tile<128, 128, 0, 0>(tmem_addr(tm, 0, TM_P), smem_u32(sm.d_o), smem_u32(sm.v), false);
        umma_commit(&sm.bar_1);
        umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_XR), smem_u32(sm.d_o), smem_u32(sm.S[2]), false);
        umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_XR), smem_u32(sm.d_o), smem_u32(sm.S[1]), true);
        umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_XR), smem_u32(sm.d_o), smem_u32(sm.S[0]), true);
        umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_XK), smem_u32(sm.v), smem_u32(dS3), false);
        umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_XK), smem_u32(sm.v), smem_u32(sm.dS[1]), true);
        umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_XK), smem_u32(sm.v), smem_u32(sm.dS[0]), true);
        umma_commit(&sm.bar_x);
        umma_tile<128, 64, 0, 0>(tmem_addr(tm, 0, TM_XV), smem_u32(sm.k), smem_u32(sm.dS[1]), false);      // (bar_2 waits for these, too)
        umma_tile<128, 64, 0, 0>(tmem_addr(tm, 0, TM_XV), smem_u32(sm.k), smem_u32(sm.dS[0]), true);
      }
      if (warp == STORE && elect_one()) {
        if (i) {
          store_out(c + 1);
          bulk_wait_read();
        }
        mbar_arrive(&sm.bar_free);
        if (c > x.lo) prefetch_in(c - 1);
      }
      ok = mbar_wait(&sm.bar_1, ph, status, 512) && ok;
      tc_fence_after();
      unsigned char* At = sm.A[qt >> 1] + (row >> 6) * TILE_BYTES;
      unsigned char* Et = sm.E[qt >> 1] + (row >> 6) * TILE_BYTES;
      if (wq >= 2 && qt < 2) ok = mbar_wait(&sm.bar_x, ph, status, 514) && ok;      // (the third part has been read)
      if (qt <= wq) {
        const bool diag = qt == wq;
        float run = 0.f, cs[2];      // of the pairs' part of dg: the sum of a row so far, and of its columns
#pragma unroll
        for (int h = 0; h < 2; ++h) {      // 16 columns at a time: registers (a spilled one goes to L2, there is no L1 left)
          uint32_t s[16], p[16];
          tmem_ld16(tmem_addr(tm, 32 * wq, TM_S + 32 * qt + 16 * h), s);
          tmem_ld16(tmem_addr(tm, 32 * wq, TM_P + 32 * qt + 16 * h), p);
          float a[16], e[16];
          if (!diag) {
            block_factors(d, row, wq, 32 * qt + 16 * h, e);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              a[j] = __uint_as_float(s[j]) * e[j];
              e[j] *= __uint_as_float(p[j]);
            }
          } else {
            diagonal_factors(d, row, 32 * qt + 16 * h, e);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) {      // (choices, so that infinities above the diagonal stay there)
              a[j] = 16 * h + j <= lane ? __uint_as_float(s[j]) * e[j] : 0.f;
              e[j] = 16 * h + j <= lane ? __uint_as_float(p[j]) * e[j] : 0.f;
            }
          }
          tile_store_row<16>(At, row & 63, 32 * (qt & 1) + 16 * h, a);
          tile_store_row<16>(Et, row & 63, 32 * (qt & 1) + 16 * h, e);
          if (!diag) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              a[j] *= __uint_as_float(p[j]);
              run += a[j];
            }
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {      // to t: the columns before it, of rows from it on
              const int t = 16 * h + j;
              const float m = t < lane ? a[j] * __uint_as_float(p[j]) : 0.f;
              a[j] = t <= lane ? run : 0.f;
              run += m;
            }
          }
          cs[h] = column_sum(a, lane);
        }
        const float mine = lane < 16 ? cs[0] : cs[1];
        if (!diag) {
          float up = mine, down = run;
#pragma unroll
          for (int e = 1; e < 32; e <<= 1) {
            const float u = __shfl_up_sync(0xffffffffu, up, e), v = __shfl_down_sync(0xffffffffu, down, e);
            if (lane >= e) up += u;
            if (lane + e < 32) down += v;
          }
          const float ex = __shfl_up_sync(0xffffffffu, up, 1);
          sm.near[ph][wq][qt][lane] = lane ? ex : 0.f;
          sm.far[ph][wq][qt][lane] = down;
          if (lane == 31) sm.all[ph][wq][qt] = up;
        } else {
          sm.near[ph][wq][qt][lane] = mine;
        }
      } else {
        if (warp == DECAYS && c > x.lo) {
          make_decays(sm.dec[ph ^ 1], raw, CT, sm.g[(i + 1) % 3]);
          if (lane == 0) sm.decay[(i + 1) % 3] = sm.dec[ph ^ 1].all;
        }
        if (warp == DW && i) write_dw(c + 1, i - 1);
        ok = mbar_wait(&sm.bar_free, ph, status, 518) && ok;      // (the gradients of the chunk before were staged in what follows)
        const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t off = tile_chunk_off(row & 63, 4 * (qt & 1) + j);
          *reinterpret_cast<uint4*>(At + off) = z;
          *reinterpret_cast<uint4*>(Et + off) = z;
        }
      }
      tc_fence_before();
      arrive(sm.bar_ae);
      // the scaled r in three parts, 8 tokens to a warp (B 8 x T 4096, H 32, with states in two parts: 361 us; by the three warps that have the least else to do 385)
      ok = mbar_wait(&sm.bar_free, ph, status, 518) && ok;
      ok = mbar_wait(&sm.bar_x, ph, status, 514) && ok;
      tc_fence_after();
      {
        uint4 u[2];
        float f[2];
        uint32_t off[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int t = 8 * warp + 4 * q + (lane >> 3);
          off[q] = (t >> 6) * TILE_BYTES + tile_chunk_off(t & 63, lane & 7);
          u[q] = *reinterpret_cast<const uint4*>(sm.r + off[q]);
          f[q] = d.start[t];
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t in[4] = {u[q].x, u[q].y, u[q].z, u[q].w};
          uint32_t hi[4], lo[4], rest[4];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float a = bf16_lo(in[g]) * f[q], b = bf16_hi(in[g]) * f[q];
            hi[g] = pack_bf16(a, b);
            a -= bf16_lo(hi[g]); b -= bf16_hi(hi[g]);
            lo[g] = pack_bf16(a, b);
            rest[g] = pack_bf16(a - bf16_lo(lo[g]), b - bf16_hi(lo[g]));
          }
          *reinterpret_cast<uint4*>(sm.rhi + off[q]) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(sm.rlo + off[q]) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          *reinterpret_cast<uint4*>(sm.v + off[q]) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
        }
      }
      arrive(sm.bar_r);
      if (c > x.lo) get_kept(c - 1);
      // the states' parts of dr and dk, and of dw
      const auto state_part = [&](uint32_t col, float f, const unsigned char* tile, float* to) {
        uint32_t a[16];
        float y[16], s = 0.f;
        tmem_ld16(tmem_addr(tm, 32 * wq, col + 16 * qt), a);
        tile_load_row<16>(tile + (row >> 6) * TILE_BYTES, row & 63, 16 * qt, y);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) s = fmaf(__uint_as_float(a[j]), y[j], s);
        to[row] = s * f;
      };
      state_part(TM_XR, d.start[row], sm.r, sm.t1[ph][qt]);
      state_part(TM_XK, d.end[row], sm.k, sm.t2[ph][qt]);
      if (c > x.lo && st_lane) store_split16(sm.S, sm.S[2], srow, 16 * qt, S0);      // (the products with this chunk's are done)
      arrive(sm.bar_read);
      if (warp == ISSUE_W) {
        ok = mbar_wait(&sm.bar_r, ph, status, 515) && ok;
        tc_fence_after();
        if (elect_one()) {
          umma_tile<64, 64, 1, 1, 8>(tmem_addr(tm, 0, TM_W), smem_u32(sm.d_o), smem_u32(sm.v), false);
          umma_tile<64, 64, 1, 1, 8>(tmem_addr(tm, 0, TM_W), smem_u32(sm.d_o), smem_u32(sm.rlo), true);
          umma_tile<64, 64, 1, 1, 8>(tmem_addr(tm, 0, TM_W), smem_u32(sm.d_o), smem_u32(sm.rhi), true);
          umma_commit(&sm.bar_2);
        }
      }
      if (warp == ISSUE) {
        ok = mbar_wait(&sm.bar_ae, ph, status, 516) && ok;
        tc_fence_after();
      }
      if (warp == ISSUE && elect_one()) {
        umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_YR), smem_u32(sm.E[0]), smem_u32(sm.k), false);
        umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_YR), smem_u32(sm.E[1]), smem_u32(sm.k) + TILE_BYTES, true);
        umma_tile<128, 64, 1, 1, 8>(tmem_addr(tm, 0, TM_YK), smem_u32(sm.E[0]), smem_u32(sm.r), false, TOK_BYTES);
        umma_tile<128, 64, 1, 1, 8>(tmem_addr(tm, 0, TM_YV), smem_u32(sm.A[0]), smem_u32(sm.d_o), false, TOK_BYTES);
        umma_commit(&sm.bar_2);
      }
      ok = mbar_wait(&sm.bar_2, ph, status, 513) && ok;
      tc_fence_after();
      if (c > x.lo && warp == LOAD) {
        ok = mbar_wait(&sm.bar_read, ph, status, 517) && ok;
        if (elect_one()) load_in(c - 1);
      }
      {
        const float fe = d.end[row];
        uint32_t a[16], b[16];
        float y[16];
        const long long to = at + (long long)(c * CT) * tok.st;
        const auto gradient = [&](uint32_t state_col, uint32_t col, float f, unsigned char* stage, bf16* out) {
          tmem_ld16(tmem_addr(tm, 32 * wq, state_col + 16 * qt), a);
          tmem_ld16(tmem_addr(tm, 32 * wq, col + 16 * qt), b);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) y[j] = fmaf(f, __uint_as_float(a[j]), __uint_as_float(b[j]));
          if (PACKED && n < CT) {
            if (row < n) store_row16(out + to, y);
          } else {
            tile_store_row<16>(stage, row & 63, 16 * qt, y);
          }
        };
        gradient(TM_XR, TM_YR, d.start[row], sm.rhi + (row >> 6) * TILE_BYTES, dr);
        gradient(TM_XK, TM_YK, fe, sm.rlo + (row >> 6) * TILE_BYTES, dk);
        gradient(TM_XV, TM_YV, fe, stage_v(row >> 6), dv);
        tmem_ld16(tmem_addr(tm, 32 * wq, TM_W + 16 * qt), a);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) dS[j] = fmaf(d.all, dS[j], __uint_as_float(a[j]));
      }
      if (c > x.lo) put_tiles(ph ^ 1);
      fence_async_smem();
      tc_fence_before();
      if (!__syncthreads_and(ok)) break;
    }
    if (warp == STORE && elect_one()) {
      store_out(x.lo);
      bulk_wait_all();
    }
    if (warp == DW) write_dw(x.lo, x.hi - 1 - x.lo);
  }
  if (dh0 && st_lane && x.part == 0 && (x.lo < x.hi || x.NT == 0)) {
#pragma unroll
    for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4*>(dh0 + (long long)x.unit * 4096 + sat + j) = make_float4(dS[j], dS[j + 1], dS[j + 2], dS[j + 3]);
  }
  if (dw_parts && warp == DW) {      // (of the whole stretch: summed over sequences and stretches by another kernel)
    double sum = sm.dw_sum[lane];
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    if (lane == 0) dw[((long long)x.n * cut.parts + x.part) * tok.H + x.h] = (float)sum;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tm, TM_COLS);
}

template <bool PACKED>
int bwd(const Args& a, cudaStream_t st) {
  const Tokens& t = a.tok;
  DeviceFacts f;
  if (int e = device_facts(&f)) return e;
  constexpr int smem = (int)sizeof(BwdSmem);
  static_assert(smem <= 227 * 1024, "one CTA to an SM");
  if (int e = need_aligned_smem<la_tc_bwd_kernel<PACKED>>(f)) return e;
  if (int e = allow_smem<la_tc_bwd_kernel<PACKED>>(f, smem)) return e;
  const int B = t.start ? 1 : t.n_seq, T = t.start ? (int)a.tokens : t.T, head_first = t.st == 64 && t.H > 1;
  const void* in[] = {a.r, a.k, a.v, a.d_o, a.dr, a.dk, a.dv};
  CUtensorMap m[7];
  for (int i = 0; i < 7; ++i)
    if (int e = make_token_tensor_map(&m[i], in[i], B, T, t.H, head_first)) return e;
  const Cut cut = cut_units(t.n_seq, t.T, t.H, true);
  const Pieces p = pieces_at(a.scratch, cut);
  const size_t chain = pieces_bytes(cut);
  float* dw_rows = reinterpret_cast<float*>(static_cast<unsigned char*>(a.scratch) + (chain + 255) / 256 * 256);      // [n_seq][parts][H]
  const size_t n_rows = (size_t)t.n_seq * cut.parts;
  double* dw_part = reinterpret_cast<double*>(reinterpret_cast<unsigned char*>(dw_rows) + (n_rows * t.H * 4 + 255) / 256 * 256);
  if (cut.parts > 1) {
    if (int e = launch_pieces(a, cut, m[3], m[0], p, true, f.status, st)) return e;
  }
  {
    ProfScope prof("linattn_tc_bwd_kernel", st);
    if (int e = launch(la_tc_bwd_kernel<PACKED>, cut.n_units * cut.parts, NTHR, smem, st, 1, a.w, a.d_ht, (const float*)a.states, (bf16*)a.dr, (bf16*)a.dk,
                       (bf16*)a.dv, a.w_per_head ? dw_rows : a.dw, a.w_per_head, a.dh0, (const float*)p.add,
                       (const float*)p.start, (const float*)p.decay, (int)cut.chained(), m[0], m[1], m[2], m[3], m[4], m[5],
                       m[6], t, cut, f.status)) return e;
  }
  return a.w_per_head ? launch_sum_dw(dw_rows, (long long)n_rows, t.H, dw_part, a.dw, st) : RWKVB200_OK;
}

}  // namespace

int launch_tc_bwd(const Args& a, cudaStream_t st) {
  Args b = a;
  set_chunks(b, CT);
  return a.tok.start ? bwd<true>(b, st) : bwd<false>(b, st);
}

}  // namespace la
}  // namespace rwkvb200
