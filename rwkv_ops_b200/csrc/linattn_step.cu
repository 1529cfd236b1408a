// Linear attention, one token on a resident state, and the reordering of resident states by beam.
//
// Per (sequence, head): S = e^{g} S + v k^T, o = S r, with S [V][K] read and written once: 2 D^2 elements of the state and 4 D of
// the tokens, so memory is all there is to it: 16,384 states of 64 x 64 floats in 84 us, 6.5 TB/s, the rate of a copy.  Few states are a launch (32 of them 6.5 us with the call).
//
// In a beam search every beam goes on from the state of the beam it was selected from.  A thread owns the same 16 bytes of the
// states of all beams of a group: it reads them from where the parents are, and writes only after that, so the states are
// reordered in place, without a second buffer, a barrier or any traffic of its own (a parent of several beams comes from memory
// once, its other readings from L1).
#include <algorithm>
#include <type_traits>

#include "linattn.cuh"

namespace rwkvb200 {
namespace la {
namespace {

// 16 bytes of a state as floats and back
__device__ __forceinline__ void unpack(const uint4& u, float (&x)[4]) {
  x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ uint4 pack(const float (&x)[4]) {
  return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
}
__device__ __forceinline__ void unpack(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ uint4 pack(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&t);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ int parent_of(const long long* parents, long long at, int W) {      // (clamped: a bad index stays inside the group)
  const long long p = __ldg(parents + at);
  return p < 0 ? 0 : p >= W ? W - 1 : (int)p;
}

constexpr int STEP_THR = 256;
// W: beams held in registers (at least the beams of a group); ROWS: rows of the state to a thread; ST: element type of the state.
// A CTA: STEP_THR / (lanes of a row) * ROWS rows of one head of one group.
template <typename T, typename ST, int D, int W, int ROWS>
__global__ void __launch_bounds__(STEP_THR) la_step_kernel(const T* __restrict__ r, const T* __restrict__ k, const T* __restrict__ v,
                                                           const float* __restrict__ w, int w_stride, ST* state, T* __restrict__ o,
                                                           const long long* __restrict__ parents, int beams, int H) {
  constexpr int KQ = 16 / (int)sizeof(ST), LR = D / KQ, RG = STEP_THR / LR;      // lanes to a row, rows side by side
  const int tid = threadIdx.x, q = tid % LR, row0 = blockIdx.y * (RG * ROWS) + tid / LR;
  const int g = blockIdx.x / H, h = blockIdx.x % H;
  earlier_kernels_done();
  later_kernels_may_start();
  // a beam's parent and decay to a lane: found once by a warp, not by every thread
  const int lane = tid & 31;
  const long long seq0 = (long long)g * beams;
  const int from = lane < beams ? parents ? parent_of(parents, seq0 + lane, beams) : lane : 0;
  const float decay = lane < beams ? decay_of(__ldg(w + (seq0 + lane) * w_stride + h)) : 0.f;
  uint4 X[W][ROWS];
#pragma unroll
  for (int j = 0; j < W; ++j) {
    if (j < beams) {
      const long long seq = seq0;
      const int p = W == 1 ? 0 : __shfl_sync(0xffffffffu, from, j);
      const ST* S = state + ((seq + p) * H + h) * (D * D) + KQ * q;
#pragma unroll
      for (int x = 0; x < ROWS; ++x) X[j][x] = *reinterpret_cast<const uint4*>(S + (row0 + RG * x) * D);
    }
  }
#pragma unroll
  for (int j = 0; j < W; ++j) {
    if (j < beams) {
      const long long seq = seq0 + j, at = (seq * H + h) * D;
      const float d = __shfl_sync(0xffffffffu, decay, j);
      float rr[KQ], kk[KQ];
      if constexpr (KQ == 8 && std::is_same<T, __nv_bfloat16>::value) {
        unpack(__ldg(reinterpret_cast<const uint4*>(r + at + KQ * q)), rr);
        unpack(__ldg(reinterpret_cast<const uint4*>(k + at + KQ * q)), kk);
      } else {
#pragma unroll
        for (int c = 0; c < KQ; c += 4) {
          const float4 r4 = load4(r + at + KQ * q + c), k4 = load4(k + at + KQ * q + c);
          rr[c] = r4.x; rr[c + 1] = r4.y; rr[c + 2] = r4.z; rr[c + 3] = r4.w;
          kk[c] = k4.x; kk[c + 1] = k4.y; kk[c + 2] = k4.z; kk[c + 3] = k4.w;
        }
      }
      ST* S = state + (seq * H + h) * (D * D) + KQ * q;
      float sum[ROWS];
#pragma unroll
      for (int x = 0; x < ROWS; ++x) {
        const float vv = to_f32(v[at + row0 + RG * x]);
        float s[KQ];
        unpack(X[j][x], s);
        sum[x] = 0.f;
#pragma unroll
        for (int c = 0; c < KQ; ++c) {
          // a state that is rounded to bfloat16: the two products and the sum as written, so that it is bit for bit what this arithmetic gives anywhere (a
          // difference in float32's last place can become one in bfloat16's, which the states after it keep; 21 x 5 beams, 40 heads, with fma 17.3 us, so 18.1)
          if constexpr (KQ == 8) s[c] = __fadd_rn(__fmul_rn(s[c], d), __fmul_rn(vv, kk[c]));
          else s[c] = fmaf(s[c], d, vv * kk[c]);
          sum[x] = fmaf(s[c], rr[c], sum[x]);      // (from the float32 value of the new state, whatever it is stored as)
        }
        *reinterpret_cast<uint4*>(S + (row0 + RG * x) * D) = pack(s);
      }
#pragma unroll
      for (int m = LR / 2; m >= 1; m >>= 1)
#pragma unroll
        for (int x = 0; x < ROWS; ++x) sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], m);
      if (q == 0) {
#pragma unroll
        for (int x = 0; x < ROWS; ++x) o[at + row0 + RG * x] = from_f32<T>(sum[x]);
      }
    }
  }
}

template <typename T, typename ST, int D, int W, int ROWS>
int step(const void* r, const float* w, int w_stride, const void* k, const void* v, void* state, void* o, const long long* parents, int groups,
         int beams, int H, cudaStream_t st) {
  constexpr int RG = STEP_THR / (D * (int)sizeof(ST) / 16);
  return launch(la_step_kernel<T, ST, D, W, ROWS>, dim3(groups * H, D / (RG * ROWS)), STEP_THR, 0, st, 1, (const T*)r, (const T*)k, (const T*)v, w,
                w_stride, (ST*)state, (T*)o, parents, beams, H);
}
// Rows to a thread: four 16-byte loads in flight with one beam, as the beams are more the beams themselves; a CTA of a bfloat16 state has
// twice the rows side by side, and 64 of them are all there are of head size 64.
template <typename T, typename ST, int D>
int step_beams(const void* r, const float* w, int w_stride, const void* k, const void* v, void* state, void* o, const long long* parents, int groups,
               int beams, int H, cudaStream_t st) {
  constexpr int RG = STEP_THR / (D * (int)sizeof(ST) / 16), R4 = std::min(4, D / RG), R2 = std::min(2, D / RG);
  if (beams == 1) return step<T, ST, D, 1, R4>(r, w, w_stride, k, v, state, o, parents, groups, beams, H, st);
  if (beams == 2) return step<T, ST, D, 2, R2>(r, w, w_stride, k, v, state, o, parents, groups, beams, H, st);
  if (beams <= 4) return step<T, ST, D, 4, 1>(r, w, w_stride, k, v, state, o, parents, groups, beams, H, st);
  if (beams <= 8) return step<T, ST, D, 8, 1>(r, w, w_stride, k, v, state, o, parents, groups, beams, H, st);
  if (beams <= 16) return step<T, ST, D, 16, 1>(r, w, w_stride, k, v, state, o, parents, groups, beams, H, st);
  return step<T, ST, D, 32, 1>(r, w, w_stride, k, v, state, o, parents, groups, beams, H, st);
}

// Rows of `pieces` times 16 bytes, [groups][beams] of them; row j of a group becomes what row parents[j] was.  A thread: COLS pieces of the rows of
// a group.  Rows that stay are neither read nor written.
template <int W, int COLS>
__global__ void __launch_bounds__(256) reorder_kernel(uint4* state, const long long* __restrict__ parents, int beams, long long pieces) {
  earlier_kernels_done();
  later_kernels_may_start();
  const long long row0 = (long long)blockIdx.y * beams, c0 = (long long)blockIdx.x * (256 * COLS) + threadIdx.x;
  uint4 X[W][COLS];
  uint32_t moved = 0;
#pragma unroll
  for (int j = 0; j < W; ++j) {
    if (j < beams) {
      const int p = parent_of(parents, row0 + j, beams);
      if (p != j) {
        moved |= 1u << j;
#pragma unroll
        for (int c = 0; c < COLS; ++c)
          if (c0 + 256 * c < pieces) X[j][c] = state[(row0 + p) * pieces + c0 + 256 * c];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < W; ++j) {
    if (moved >> j & 1) {
#pragma unroll
      for (int c = 0; c < COLS; ++c)
        if (c0 + 256 * c < pieces) state[(row0 + j) * pieces + c0 + 256 * c] = X[j][c];
    }
  }
}
template <int W, int COLS>
int reorder(void* state, const long long* parents, int groups, int beams, long long pieces, cudaStream_t st) {
  // groups beyond what a grid's second dimension holds: several launches
  for (int g = 0; g < groups; g += 65535) {
    const int n = std::min(65535, groups - g);
    if (int e = launch(reorder_kernel<W, COLS>, dim3((unsigned)((pieces + 256 * COLS - 1) / (256 * COLS)), n), 256, 0, st, 1,
                       static_cast<uint4*>(state) + (long long)g * beams * pieces, parents + (long long)g * beams, beams, pieces)) return e;
  }
  return RWKVB200_OK;
}

}  // namespace

int launch_step(const void* r, const float* w, int w_stride, const void* k, const void* v, void* state, int state_dtype, void* o,
                const long long* parents, int groups, int beams, int H, int D, int dtype, cudaStream_t st) {
  ProfScope prof("linattn_step_kernel", st);
  RWKVB200_DISPATCH_DTYPE(dtype, {
    if (state_dtype == RWKVB200_BF16)
      return D == 64 ? step_beams<T, __nv_bfloat16, 64>(r, w, w_stride, k, v, state, o, parents, groups, beams, H, st)
                     : step_beams<T, __nv_bfloat16, 128>(r, w, w_stride, k, v, state, o, parents, groups, beams, H, st);
    return D == 64 ? step_beams<T, float, 64>(r, w, w_stride, k, v, state, o, parents, groups, beams, H, st)
                   : step_beams<T, float, 128>(r, w, w_stride, k, v, state, o, parents, groups, beams, H, st);
  });
  return RWKVB200_OK;
}

int launch_reorder(void* state, const long long* parents, int groups, int beams, long long row_bytes, cudaStream_t st) {
  ProfScope prof("reorder_kernel", st);
  const long long pieces = row_bytes / 16;
  if (beams <= 2) return reorder<2, 4>(state, parents, groups, beams, pieces, st);
  if (beams <= 4) return reorder<4, 2>(state, parents, groups, beams, pieces, st);
  if (beams <= 8) return reorder<8, 1>(state, parents, groups, beams, pieces, st);
  if (beams <= 16) return reorder<16, 1>(state, parents, groups, beams, pieces, st);
  return reorder<32, 1>(state, parents, groups, beams, pieces, st);
}

}  // namespace la
}  // namespace rwkvb200
