// Linear attention with a decay for each head, backward on tcgen05: bfloat16 tokens, head size 64 (linattn_tc.cuh).
#include <algorithm>

#include "linattn_tc.cuh"

namespace rwkvb200 {
namespace la {
namespace {

constexpr int NTHR = 512, NWARP = NTHR / 32;

struct BwdSmem {
  unsigned char r[TOK_BYTES], k[TOK_BYTES], v[TOK_BYTES], d_o[TOK_BYTES];
  unsigned char rhi[TOK_BYTES], rlo[TOK_BYTES];      // e^{L_i} r_i
  unsigned char A[2][TOK_BYTES], E[2][TOK_BYTES];    // [token i][token j], two times 64 columns; dr, dk, dv are staged in the first three afterwards
  unsigned char S[2][TILE_BYTES], dS[2][TILE_BYTES]; // the state before the chunk and the gradient of the one after it, hi and lo, [v][k]
  Decays dec[2];
  float g[2][CT];
  // What the pairs of a 32 x 32 block (I, J) of tokens add to dg_t (M = A_ij (d_o_i . v_j)): near[I][J]: for t in J, the sum over j < t (I > J: all rows i; I == J:
  // rows i >= t); far[I][J]: for t in I, the sum over rows i >= t; and all of it for t between.
  float near[2][4][4][32], far[2][4][4][32], all[2][4][4];
  float t1[4][CT], t2[4][CT], t3[2][NWARP];
  uint64_t bar_in, bar_1, bar_2;
  uint32_t tmem_base;
};
constexpr uint32_t TM_S = 0, TM_P = 128, TM_YR = 0, TM_YK = 64, TM_YV = 128, TM_XR = 256, TM_XK = 320, TM_XV = 384, TM_W = 448, TM_COLS = 512;

// the sum over a warp's lanes of x[c], in lane c
__device__ __forceinline__ float column_sum(float (&x)[32], int lane) {
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) {
    const bool up = lane & m;
#pragma unroll
    for (int c = 0; c < m; ++c) {
      const float send = up ? x[c] : x[c + m], keep = up ? x[c + m] : x[c];
      x[c] = keep + __shfl_xor_sync(0xffffffffu, send, m);
    }
  }
  return x[0];
}
// 16 values of a row, columns col0 .. (a multiple of 8), as hi and lo tiles
__device__ __forceinline__ void store_split16(unsigned char* hi_t, unsigned char* lo_t, int row, int col0, const float* x) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = x[8 * c + 2 * e], b = x[8 * c + 2 * e + 1];
      h[e] = pack_bf16(a, b);
      l[e] = pack_bf16(a - bf16_lo(h[e]), b - bf16_hi(h[e]));
    }
    const uint32_t off = tile_chunk_off(row, (col0 >> 3) + c);
    *reinterpret_cast<uint4*>(hi_t + off) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(lo_t + off) = make_uint4(l[0], l[1], l[2], l[3]);
  }
}

// One item: the chunks of a stretch from the last to the first, the gradient of the state in registers.  Per chunk two batches of products:
//   r k^T, d_o v^T, d_o S, v dS, k dS^T          meanwhile e^{L_i} r_i is split
//   E k, E^T r, A^T d_o, d_o^T (scaled r)        after A and E have been stored; meanwhile the states' part of dw
// then the three gradients are put together, staged in the space of A and E and stored, while the next chunk's rows arrive.
// Sixteen warps, one CTA to an SM (all of TMEM, 210 KB): warp w reads token rows 32 (w % 4) .. and a quarter of the columns; the six warps whose block of pairs lies
// above the diagonal clear it, and one of them makes the next chunk's decays, another the chunk before's dw.
template <bool PACKED>
__global__ void __launch_bounds__(NTHR, 1)
la_tc_bwd_kernel(const float* __restrict__ w, const float* __restrict__ d_ht, const float* __restrict__ states, bf16* __restrict__ dr,
                 bf16* __restrict__ dk, bf16* __restrict__ dv, float* __restrict__ dw, int dw_parts, float* __restrict__ dh0,
                 const float* __restrict__ part_states, const __grid_constant__ CUtensorMap map_r, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do, const __grid_constant__ CUtensorMap map_dr,
                 const __grid_constant__ CUtensorMap map_dk, const __grid_constant__ CUtensorMap map_dv, Tokens tok, Cut cut, int* status) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  BwdSmem& sm = *reinterpret_cast<BwdSmem*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wq = warp & 3, qt = warp >> 2, row = 32 * wq + lane;
  if (tid == 0) {
    mbar_init(&sm.bar_in, 1); mbar_init(&sm.bar_1, 1); mbar_init(&sm.bar_2, 1);
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
  const Stretch x = stretch_of(tok, cut);
  const int seq0 = PACKED ? __ldg(tok.start + x.n) : 0, brow = PACKED ? 0 : x.n;
  const long long wb = tok.wbase(x.n, x.h);
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
  // states: lanes 0 .. 15 hold row v = 16 wq + lane, columns 16 qt .. + 15
  const bool st_lane = lane < 16;
  const int srow = 16 * wq + (lane & 15);
  const long long sat = (long long)srow * 64 + 16 * qt;
  float dS[16], S0[16];
  auto get_state = [&](float (&s)[16], const float* from) {
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      const float4 f = st_lane && from ? __ldcg(reinterpret_cast<const float4*>(from + sat + j)) : make_float4(0.f, 0.f, 0.f, 0.f);
      s[j] = f.x; s[j + 1] = f.y; s[j + 2] = f.z; s[j + 3] = f.w;
    }
  };
  auto state_before = [&](int c) { return states + ((long long)x.unit * tok.NT + c) * 4096; };
  // both states of a chunk into their tiles, and their product
  auto put_tiles = [&](int ph) {
    float s = 0.f;
    if (st_lane) {
      store_split16(sm.S[0], sm.S[1], srow, 16 * qt, S0);
      store_split16(sm.dS[0], sm.dS[1], srow, 16 * qt, dS);
#pragma unroll
      for (int j = 0; j < 16; ++j) s = fmaf(S0[j], dS[j], s);
    }
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    if (lane == 0) sm.t3[ph][warp] = s;
  };
  get_state(dS, x.part + 1 < cut.parts ? part_states + ((long long)x.unit * cut.parts + x.part) * 4096 : d_ht ? d_ht + (long long)x.unit * 4096 : nullptr);
  bool ok = true;
  double dw_sum = 0.0;
  // dw of chunk c (its sums are in buffers `ph`), four tokens to a lane
  auto write_dw = [&](int c, uint32_t ph) {
    const Decays& d = sm.dec[ph];
    const int I = lane >> 3, n = rows_of(c);
    float t3 = 0.f;
#pragma unroll
    for (int u = 0; u < NWARP; ++u) t3 += sm.t3[ph][u];
    t3 *= d.all;
    float pairs[4], after[4], before[4], sa = 0.f, sb = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int t = 4 * lane + q;
      after[q] = sm.t1[0][t] + sm.t1[1][t] + sm.t1[2][t] + sm.t1[3][t];
      before[q] = sm.t2[0][t] + sm.t2[1][t] + sm.t2[2][t] + sm.t2[3][t];
      sa += after[q]; sb += before[q];
      float p = 0.f;
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        if (a >= I) p += sm.near[ph][a][I][t & 31];
        if (a < I) p += sm.far[ph][I][a][t & 31];
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (b < I && I < a) p += sm.all[ph][a][b];
      }
      pairs[q] = p;
    }
    float down = sa, up = sb;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const float a = __shfl_down_sync(0xffffffffu, down, m), b = __shfl_up_sync(0xffffffffu, up, m);
      if (lane + m < 32) down += a;
      if (lane >= m) up += b;
    }
    const float later = __shfl_down_sync(0xffffffffu, down, 1), earlier = __shfl_up_sync(0xffffffffu, up, 1);      // of the lanes behind, before
    float behind = lane < 31 ? later : 0.f, ahead = lane ? earlier : 0.f;
    float dg[4];
#pragma unroll
    for (int q = 3; q >= 0; --q) { behind += after[q]; dg[q] = pairs[q] + behind + t3; }
#pragma unroll
    for (int q = 0; q < 4; ++q) { dg[q] += ahead; ahead += before[q]; }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int t = 4 * lane + q;
      const float y = dg[q] * sm.g[ph][t];
      if (t < n) {
        if (dw_parts) dw_sum += y;
        else dw[wb + (long long)(c * CT + t) * tok.wst] = y;
      }
    }
  };
  if (x.lo < x.hi) {
    if (warp == 0 && elect_one()) load_in(x.hi - 1);
    RawW raw;
    if (warp == 8) {      // the decays are this warp's job: its block of pairs is above the diagonal
      raw = load_w(tok, w, wb, (x.hi - 1) * CT, rows_of(x.hi - 1));
      make_decays(sm.dec[0], raw, rows_of(x.hi - 1), sm.g[0]);
      if (x.hi - 2 >= x.lo) raw = load_w(tok, w, wb, (x.hi - 2) * CT, CT);
    }
    get_state(S0, state_before(x.hi - 1));
    put_tiles(0);
    fence_async_smem();
    __syncthreads();
    for (int c = x.hi - 1; c >= x.lo; --c) {
      const uint32_t ph = (x.hi - 1 - c) & 1;
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
      if (warp == 0 && elect_one()) {
        tc_fence_after();
        umma_tile<128, 128, 0, 0>(tmem_addr(tm, 0, TM_S), smem_u32(sm.r), smem_u32(sm.k), false);
        umma_tile<128, 128, 0, 0>(tmem_addr(tm, 0, TM_P), smem_u32(sm.d_o), smem_u32(sm.v), false);
        umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_XR), smem_u32(sm.d_o), smem_u32(sm.S[0]), false);
        umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_XR), smem_u32(sm.d_o), smem_u32(sm.S[1]), true);
        umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_XK), smem_u32(sm.v), smem_u32(sm.dS[0]), false);
        umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_XK), smem_u32(sm.v), smem_u32(sm.dS[1]), true);
        umma_tile<128, 64, 0, 0>(tmem_addr(tm, 0, TM_XV), smem_u32(sm.k), smem_u32(sm.dS[0]), false);
        umma_commit(&sm.bar_1);
        bulk_wait_read();      // the gradients of the chunk before have left their place in A and E
      }
      if (c > x.lo) get_state(S0, state_before(c - 1));
      {
        const unsigned char* rt = sm.r + (row >> 6) * TILE_BYTES;
        float y[16];
        tile_load_row<16>(rt, row & 63, 16 * qt, y);
        const float f = d.start[row];
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] *= f;
        store_split16(sm.rhi + (row >> 6) * TILE_BYTES, sm.rlo + (row >> 6) * TILE_BYTES, row & 63, 16 * qt, y);
      }
      if (warp == 12 && c + 1 < x.hi) write_dw(c + 1, ph ^ 1);
      __syncthreads();      // (the staged gradients have been read, dw of the chunk before is done with its buffers)
      ok = mbar_wait(&sm.bar_1, ph, status, 512) && ok;
      tc_fence_after();
      unsigned char* At = sm.A[qt >> 1] + (row >> 6) * TILE_BYTES;
      unsigned char* Et = sm.E[qt >> 1] + (row >> 6) * TILE_BYTES;
      if (qt <= wq) {
        uint32_t s[32], p[32];
        tmem_ld32(tmem_addr(tm, 32 * wq, TM_S + 32 * qt), s);
        tmem_ld32(tmem_addr(tm, 32 * wq, TM_P + 32 * qt), p);
        float f[32], m[32];
        if (qt < wq) {
          const float fr = d.row[row];
          const float* col = d.col[wq - 1] + 32 * qt;
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 g = *reinterpret_cast<const float4*>(col + j);
            f[j] = fr * g.x; f[j + 1] = fr * g.y; f[j + 2] = fr * g.z; f[j + 3] = fr * g.w;
          }
        } else {
          diagonal_factors(d, row, 32 * qt, f);
        }
        tmem_ld_wait();
        const bool diag = qt == wq;
        float a[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float pj = __uint_as_float(p[j]);
          a[j] = __uint_as_float(s[j]) * f[j];
          if (diag && j > lane) a[j] = 0.f;      // (infinities above the diagonal stay there)
          m[j] = diag && j >= lane ? 0.f : a[j] * pj;
        }
        tile_store_row32(At, row & 63, 32 * (qt & 1), a);
#pragma unroll
        for (int j = 0; j < 32; ++j) a[j] = diag && j > lane ? 0.f : __uint_as_float(p[j]) * f[j];
        tile_store_row32(Et, row & 63, 32 * (qt & 1), a);
        if (diag) {
          float run = 0.f;
#pragma unroll
          for (int j = 0; j < 32; ++j) {      // to t = j: the columns before it, of rows from it on
            const float mj = m[j];
            m[j] = j <= lane ? run : 0.f;
            run += mj;
          }
          sm.near[ph][wq][qt][lane] = column_sum(m, lane);
        } else {
          float rs = 0.f;
#pragma unroll
          for (int j = 0; j < 32; ++j) rs += m[j];
          const float cs = column_sum(m, lane);
          float up = cs, down = rs;
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
        }
      } else {
        float z[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) z[j] = 0.f;
        tile_store_row32(At, row & 63, 32 * (qt & 1), z);
        tile_store_row32(Et, row & 63, 32 * (qt & 1), z);
        if (warp == 8 && c > x.lo) {
          make_decays(sm.dec[ph ^ 1], raw, CT, sm.g[ph ^ 1]);
          if (c - 1 > x.lo) raw = load_w(tok, w, wb, (c - 2) * CT, CT);
        }
      }
      fence_async_smem();
      tc_fence_before();
      __syncthreads();
      if (warp == 0 && elect_one()) {
        tc_fence_after();
        umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_YR), smem_u32(sm.E[0]), smem_u32(sm.k), false);
        umma_tile<128, 64, 0, 1>(tmem_addr(tm, 0, TM_YR), smem_u32(sm.E[1]), smem_u32(sm.k) + TILE_BYTES, true);
        umma_tile<128, 64, 1, 1, 8>(tmem_addr(tm, 0, TM_YK), smem_u32(sm.E[0]), smem_u32(sm.r), false, TOK_BYTES);
        umma_tile<128, 64, 1, 1, 8>(tmem_addr(tm, 0, TM_YV), smem_u32(sm.A[0]), smem_u32(sm.d_o), false, TOK_BYTES);
        umma_tile<64, 64, 1, 1, 8>(tmem_addr(tm, 0, TM_W), smem_u32(sm.d_o), smem_u32(sm.rhi), false);
        umma_tile<64, 64, 1, 1, 8>(tmem_addr(tm, 0, TM_W), smem_u32(sm.d_o), smem_u32(sm.rlo), true);
        umma_commit(&sm.bar_2);
      }
      // the states' parts of dr and dk, and of dw
      float xr[16], xk[16];
      {
        uint32_t a[16], b[16];
        tmem_ld16(tmem_addr(tm, 32 * wq, TM_XR + 16 * qt), a);
        tmem_ld16(tmem_addr(tm, 32 * wq, TM_XK + 16 * qt), b);
        float rr[16], kk[16];
        tile_load_row<16>(sm.r + (row >> 6) * TILE_BYTES, row & 63, 16 * qt, rr);
        tile_load_row<16>(sm.k + (row >> 6) * TILE_BYTES, row & 63, 16 * qt, kk);
        const float fs = d.start[row], fe = d.end[row];
        tmem_ld_wait();
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          xr[j] = __uint_as_float(a[j]) * fs;
          xk[j] = __uint_as_float(b[j]) * fe;
          s1 = fmaf(xr[j], rr[j], s1);
          s2 = fmaf(xk[j], kk[j], s2);
        }
        sm.t1[qt][row] = s1;
        sm.t2[qt][row] = s2;
      }
      fence_async_smem();      // (r and k have been read; the next rows are copied over them)
      ok = mbar_wait(&sm.bar_2, ph, status, 513) && ok;
      tc_fence_after();
      __syncthreads();
      if (c > x.lo && warp == 0 && elect_one()) load_in(c - 1);
      {
        const float fe = d.end[row];
        uint32_t a[16], b[16];
        float y[16];
        auto put = [&](unsigned char* stage, bf16* out) {
          if (PACKED && n < CT) {      // the rows behind belong to the next sequence
            if (row < n) {
              bf16* to = out + tok.base(x.n, x.h) + (long long)(c * CT + row) * tok.st + 16 * qt;
#pragma unroll
              for (int j = 0; j < 16; j += 8)
                *reinterpret_cast<uint4*>(to + j) = make_uint4(pack_bf16(y[j], y[j + 1]), pack_bf16(y[j + 2], y[j + 3]),
                                                               pack_bf16(y[j + 4], y[j + 5]), pack_bf16(y[j + 6], y[j + 7]));
            }
          } else {
            tile_store_row<16>(stage + (row >> 6) * TILE_BYTES, row & 63, 16 * qt, y);
          }
        };
        tmem_ld16(tmem_addr(tm, 32 * wq, TM_YR + 16 * qt), a);
        tmem_ld16(tmem_addr(tm, 32 * wq, TM_YK + 16 * qt), b);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = xr[j] + __uint_as_float(a[j]);
        put(sm.A[0], dr);
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = xk[j] + __uint_as_float(b[j]);
        put(sm.A[1], dk);
        tmem_ld16(tmem_addr(tm, 32 * wq, TM_XV + 16 * qt), a);
        tmem_ld16(tmem_addr(tm, 32 * wq, TM_YV + 16 * qt), b);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) y[j] = fmaf(fe, __uint_as_float(a[j]), __uint_as_float(b[j]));
        put(sm.E[0], dv);
        tmem_ld16(tmem_addr(tm, 32 * wq, TM_W + 16 * qt), a);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) dS[j] = fmaf(d.all, dS[j], __uint_as_float(a[j]));
      }
      if (c > x.lo) put_tiles(ph ^ 1);
      fence_async_smem();
      tc_fence_before();
      if (!__syncthreads_and(ok)) break;
      if (!(PACKED && n < CT) && warp == 0 && elect_one()) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {      // (rows past the end of the batch are clipped)
          if (64 * q < n) {
            tma_store_4d(&map_dr, sm.A[0] + q * TILE_BYTES, 0, seq0 + c * CT + 64 * q, x.h, brow);
            tma_store_4d(&map_dk, sm.A[1] + q * TILE_BYTES, 0, seq0 + c * CT + 64 * q, x.h, brow);
            tma_store_4d(&map_dv, sm.E[0] + q * TILE_BYTES, 0, seq0 + c * CT + 64 * q, x.h, brow);
          }
        }
        bulk_commit();
      }
    }
    if (warp == 12) write_dw(x.lo, (x.hi - 1 - x.lo) & 1);
  }
  if (dh0 && st_lane && x.part == 0 && (x.lo < x.hi || x.NT == 0)) {
#pragma unroll
    for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4*>(dh0 + (long long)x.unit * 4096 + sat + j) = make_float4(dS[j], dS[j + 1], dS[j + 2], dS[j + 3]);
  }
  if (dw_parts && warp == 12) {      // (of the whole stretch: summed over sequences and stretches by another kernel)
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) dw_sum += __shfl_xor_sync(0xffffffffu, dw_sum, m);
    if (lane == 0) dw[((long long)x.n * cut.parts + x.part) * tok.H + x.h] = (float)dw_sum;
  }
  if (warp == 0 && elect_one()) bulk_wait_all();
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
  const int B = t.start ? 1 : t.n_seq, T = t.start ? (int)a.w_rows : t.T, head_first = t.st == 64 && t.H > 1;
  const void* in[] = {a.r, a.k, a.v, a.d_o, a.dr, a.dk, a.dv};
  CUtensorMap m[7];
  for (int i = 0; i < 7; ++i)
    if (int e = make_token_tensor_map(&m[i], in[i], B, T, t.H, head_first)) return e;
  const Cut cut = cut_units(t.n_seq, t.T, t.H, true);
  float* part_states = static_cast<float*>(a.scratch);
  float* part_decay = part_states + (size_t)cut.n_units * cut.parts * 4096;
  const size_t chain = cut.parts > 1 ? (size_t)cut.n_units * cut.parts * (4096 + 1) * 4 : 0;
  float* dw_rows = reinterpret_cast<float*>(static_cast<unsigned char*>(a.scratch) + (chain + 255) / 256 * 256);      // [n_seq][parts][H]
  const size_t n_rows = (size_t)t.n_seq * cut.parts;
  double* dw_part = reinterpret_cast<double*>(reinterpret_cast<unsigned char*>(dw_rows) + (n_rows * t.H * 4 + 255) / 256 * 256);
  if (cut.parts > 1) {
    if (int e = launch_tc_add(a, cut, m[3], m[0], part_states, part_decay, f.status, st)) return e;
    if (int e = launch_chain(part_states, part_decay, a.d_ht, t.n_seq, t, cut, true, st)) return e;
  }
  {
    ProfScope prof("linattn_tc_bwd_kernel", st);
    if (int e = launch(la_tc_bwd_kernel<PACKED>, cut.n_units * cut.parts, NTHR, smem, st, 1, a.w, a.d_ht, (const float*)a.states, (bf16*)a.dr, (bf16*)a.dk,
                       (bf16*)a.dv, a.w_per_head ? dw_rows : a.dw, a.w_per_head, a.dh0, (const float*)part_states, m[0], m[1], m[2], m[3], m[4], m[5],
                       m[6], t, cut, f.status)) return e;
  }
  return a.w_per_head ? launch_sum_dw(dw_rows, (long long)n_rows, t.H, dw_part, a.dw, st) : RWKVB200_OK;
}

}  // namespace

int launch_tc_bwd(const Args& a, cudaStream_t st) {
  Args b = a;
  b.tok.NT = (a.tok.T + CT - 1) / CT;
  return a.tok.start ? bwd<true>(b, st) : bwd<false>(b, st);
}

}  // namespace la
}  // namespace rwkvb200
