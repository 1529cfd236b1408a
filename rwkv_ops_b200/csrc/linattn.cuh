// Linear attention with a decay for each head: shared definitions.
//
// One (batch, head), g_t = -exp(w_t) (a number per head, or per token and head), S the [V][K] state:
//   S_t = e^{g_t} S_{t-1} + v_t k_t^T        o_t = S_t r_t
// In a chunk with inclusive prefix sums L_i of g, S0 the state before it, Lc the sum over the whole chunk:
//   A_ij = (r_i . k_j) e^{L_i - L_j}  (j <= i, else 0)
//   o_i  = e^{L_i} S0 r_i + sum_j A_ij v_j
//   S_c  = e^{Lc} S0 + sum_j e^{Lc - L_j} v_j k_j^T
// Backward (do_i and dS_c given):
//   E_ij = (do_i . v_j) e^{L_i - L_j}  (j <= i)
//   dr_i = e^{L_i} S0^T do_i + sum_j E_ij k_j
//   dk_j = e^{Lc - L_j} dS_c^T v_j + sum_i E_ij r_i
//   dv_j = e^{Lc - L_j} dS_c k_j + sum_i A_ij do_i
//   dS0  = e^{Lc} dS_c + sum_i e^{L_i} do_i r_i^T
//   dg_t = sum_{i >= t > j} A_ij (do_i . v_j) + sum_{i >= t} e^{L_i} r_i . S0^T do_i
//          + sum_{j < t} e^{Lc - L_j} k_j . dS_c^T v_j + e^{Lc} <dS_c, S0>          dw_t = dg_t g_t
// Every exponent is a sum of g over some tokens, so no factor exceeds one whatever the decay, and no range has to be
// watched, and every term of dg_t carries the factor e^{g_t}: summed as they stand (the pairs by prefix sums along the rows of
// A * E's products), never as differences of longer sums, they keep their digits where the decay is strong.
//
// Prefix sums are taken in float64 and rounded as differences: a sum of 128 large g would leave float32 too few digits for the
// neighbours whose difference is small.  g below -200 counts as -200: e^{-200} is zero in float32 times anything, and the sums
// stay finite.
#pragma once

#include <algorithm>

#include "common.cuh"

namespace rwkvb200 {
namespace la {

// g is a float32 exponential and only its sums are float64: an error of 2^-23 of L, times e^L, is never more than 2^-24.
constexpr float G_FLOOR = -200.f;
__device__ __forceinline__ float g_of(float w) {
  const float g = -expf(w);
  return g < G_FLOOR ? G_FLOOR : g;      // (a NaN stays one)
}

// Where the tokens lie.  Token tensors have strides sb / st / sh (elements) over batch, token and head, w its own (zero over
// batch and token where it is a number per head).  Dense: sequence n is batch row n with T tokens; packed (start != nullptr): all
// sequences lie in one row, sequence n at tokens start[n] .. start[n] + len[n] - 1, and T is the longest length.
struct Tokens {
  long long sb, st, sh, wsb, wst, wsh;
  const int* start;
  const int* len;
  int n_seq, T, H;
  // What is kept of every chunk of C = 2^shift tokens lies in slots.  Dense: NT of them to a (sequence, head), as many as the longest sequence has chunks.  Packed and compact:
  // `slots` of them to a head, sequence n's from start[n] / C + n on; sequences in the order of their places, none overlapping another, never meet there (a
  // sequence has at most len / C + 1 chunks), and one long sequence among many short ones takes what its tokens take and not their number times its length.
  int shift, NT, slots, compact;
  __device__ __forceinline__ int length(int n) const { return len ? __ldg(len + n) : T; }
  __device__ __forceinline__ long long base(int n, int h) const { return (start ? __ldg(start + n) * st : n * sb) + h * sh; }
  __device__ __forceinline__ long long wbase(int n, int h) const { return (start ? __ldg(start + n) * wst : n * wsb) + h * wsh; }
  // the first slot of a (sequence, head); with one slot more than chunks to a sequence where `more` is 1
  __device__ __forceinline__ int place(int n, int more) const { return (__ldg(start + n) >> shift) + n * (1 + more); }
  __device__ __forceinline__ long long first(int n, int h, int more) const {
    return compact ? (long long)h * (slots + more * n_seq) + place(n, more) : (long long)(n * H + h) * (NT + more);
  }
};

// Chunk slots of a head (dense and padded: of all its sequences), and whether they are compact: where that is fewer.
inline long long padded_slots(int n_seq, int max_len, int C) { return (long long)n_seq * ((max_len + (long long)C - 1) / C); }
inline long long compact_slots(int n_seq, int total, int C) { return total / C + (long long)n_seq; }
inline long long chunk_slots(int n_seq, int max_len, int total, int C) {      // total 0: not compact
  const long long p = padded_slots(n_seq, max_len, C);
  return total > 0 ? std::min(p, compact_slots(n_seq, total, C)) : p;
}

// What a call works on; pointers that do not apply are NULL.
struct Args {
  const void *r, *k, *v, *d_o;
  const float *w, *h0, *d_ht;
  void *o, *dr, *dk, *dv;
  float *ht, *dh0;
  float* dw;              // gradient of w: like w
  float* states;          // [slots][D][D]: the state before every chunk (linattn_simt.cu: and the last one)
  void* scratch;
  int n_state, w_per_head, dtype, D, compact;
  long long tokens;       // in all
  Tokens tok;
};

// The chunks of a call's tokens, C (64 or 128) of them to a chunk.
inline void set_chunks(Args& a, int C) {
  Tokens& t = a.tok;
  t.shift = C == 128 ? 7 : 6; t.NT = (int)((t.T + (long long)C - 1) / C); t.compact = a.compact;
  t.slots = (int)chunk_slots(t.n_seq, t.T, a.compact ? (int)a.tokens : 0, C);
}

// The gradient of a w per head, from what stretches of sequences add to it [rows][H]: partial sums [parts][H] in float64, added up in a fixed order.
int launch_sum_dw(const float* dw_rows, long long rows, int H, double* partial, float* dw, cudaStream_t st);
constexpr int DW_PARTS = 128;

// float32 arithmetic on the CUDA cores: every dtype, head sizes 64 and 128, chunks of 64 tokens (linattn_simt.cu)
int launch_simt_fwd(const Args& a, cudaStream_t st);
int launch_simt_bwd(const Args& a, cudaStream_t st);
size_t simt_states_bytes(int n_seq, int max_len, int total, int H, int D);      // total 0: dense or padded
size_t simt_scratch_bytes(int n_seq, int max_len, int total, int H, int D, bool w_per_head, bool backward);

// tensor cores: bfloat16 tokens, head size 64, chunks of 128 tokens (linattn_tc_fwd.cu, linattn_tc_bwd.cu)
inline bool tc_applies(int D, int dtype) { return D == 64 && dtype == RWKVB200_BF16; }
int launch_tc_fwd(const Args& a, cudaStream_t st);
int launch_tc_bwd(const Args& a, cudaStream_t st);
size_t tc_states_bytes(int n_seq, int max_len, int total, int H, bool keep);
size_t tc_scratch_bytes(int n_seq, int max_len, int H, bool w_per_head, bool backward);

// one token in place on states [groups * beams][H][D][D], float32 or bfloat16 (linattn_step.cu); w_stride: H, or 0 for a w per head
int launch_step(const void* r, const float* w, int w_stride, const void* k, const void* v, void* state, int state_dtype, void* o,
                const long long* parents, int groups, int beams, int H, int D, int dtype, cudaStream_t st);
int launch_reorder(void* state, const long long* parents, int groups, int beams, long long row_bytes, cudaStream_t st);
constexpr int MAX_BEAMS = 32;

}  // namespace la
}  // namespace rwkvb200
