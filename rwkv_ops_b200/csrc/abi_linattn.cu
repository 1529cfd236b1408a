// extern "C" entry points of linear attention, its decode step, the reordering of states and the beam selection: argument
// checks and dispatch.
#include "linattn.cuh"

namespace rwkvb200 {
int launch_beam_select(const void* logits, int dtype, long long sg, long long sw, const float* scores, const uint8_t* finished, long long eos,
                       float* scores_out, long long* parents, long long* tokens, uint8_t* finished_out, int G, int W, int V, cudaStream_t st);

namespace {

int check_dims(long long n_seq, long long T, long long H, int D, int dtype) {
  if (n_seq <= 0 || T <= 0 || H <= 0) return RWKVB200_E_SHAPE;
  if (D != 64 && D != 128) return RWKVB200_E_UNSUPPORTED;
  if (dtype != RWKVB200_F32 && dtype != RWKVB200_BF16 && dtype != RWKVB200_F16) return RWKVB200_E_DTYPE;
  // a grid has up to 16 blocks for a state
  return n_seq * H > (1 << 26) ? RWKVB200_E_TOO_LARGE : RWKVB200_OK;
}
// total 0: dense, or packed with as many slots to each sequence as the longest one has chunks.  A grid has a block for every slot of every head.
int check_sizes(int n_seq, int T, int total, int H, int D, int dtype) {
  if (int e = check_dims(n_seq, T, H, D, dtype)) return e;
  return la::chunk_slots(n_seq, T, total, 64) * H > 0x7fffffffLL ? RWKVB200_E_TOO_LARGE : RWKVB200_OK;
}
size_t states_bytes_of(int n_seq, int T, int total, int H, int D, int dtype, int keep) {
  if (check_sizes(n_seq, T, total, H, D, dtype)) return 0;
  return la::tc_applies(D, dtype) ? la::tc_states_bytes(n_seq, T, total, H, keep) : la::simt_states_bytes(n_seq, T, total, H, D);
}
size_t workspace_bytes_of(int n_seq, int T, int total, int H, int D, int dtype, int w_per_head, int backward) {
  if (check_sizes(n_seq, T, total, H, D, dtype)) return 0;
  return la::tc_applies(D, dtype) ? la::tc_scratch_bytes(n_seq, T, H, w_per_head, backward)
                                  : la::simt_scratch_bytes(n_seq, T, total, H, D, w_per_head, backward);
}
// Whether the states of a packed batch lie compactly: where a caller has brought no memory for the padded form, or that has too many blocks.
bool compact_of(bool packed, const void* states, size_t states_bytes, int n_seq, int T, int total, int H, int D, int dtype) {
  if (!packed || !states) return false;
  const size_t padded = states_bytes_of(n_seq, T, 0, H, D, dtype, 1), compact = states_bytes_of(n_seq, T, total, H, D, dtype, 1);
  return compact && (!padded || (compact < padded && states_bytes < padded));
}
template <typename... P> bool any_null(const P*... p) { return (... || !p); }
template <typename... P> bool misaligned(const P*... p) { return (... || !aligned16(p)); }

la::Tokens tokens_of(const int* start, const int* len, int n_seq, int T, int total, int H, int D, int head_first, int w_per_head) {
  la::Tokens t;
  const long long rows = start ? total : T;      // of a batch row
  t.sb = rows * H * D;
  t.st = head_first ? D : (long long)H * D;
  t.sh = head_first ? rows * D : D;
  t.wsb = w_per_head ? 0 : rows * H;
  t.wst = w_per_head ? 0 : head_first ? 1 : H;
  t.wsh = w_per_head ? 1 : head_first ? rows : 1;
  t.start = start; t.len = len;
  t.n_seq = n_seq; t.T = T; t.H = H;
  return t;
}

}  // namespace
}  // namespace rwkvb200

using namespace rwkvb200;

extern "C" {

size_t rwkvb200_linattn_states_bytes(int n_seq, int max_len, int H, int head_size, int dtype, int keep) {
  return states_bytes_of(n_seq, max_len, 0, H, head_size, dtype, keep);
}

size_t rwkvb200_linattn_packed_states_bytes(int n_seq, int max_len, int total, int H, int head_size, int dtype, int keep) {
  return total > 0 ? states_bytes_of(n_seq, max_len, total, H, head_size, dtype, keep) : 0;
}

size_t rwkvb200_linattn_workspace_bytes(int n_seq, int max_len, int total, int H, int head_size, int dtype, int w_per_head, int backward) {
  return workspace_bytes_of(n_seq, max_len, 0, H, head_size, dtype, w_per_head, backward);
}

size_t rwkvb200_linattn_packed_workspace_bytes(int n_seq, int max_len, int total, int H, int head_size, int dtype, int w_per_head, int backward) {
  return total > 0 ? workspace_bytes_of(n_seq, max_len, total, H, head_size, dtype, w_per_head, backward) : 0;
}

int rwkvb200_linattn_fwd(const void* r, const float* w, int w_per_head, const void* k, const void* v, const float* h0, int n_state, void* o,
                         float* ht, float* states, size_t states_bytes, void* workspace, size_t workspace_bytes, const int32_t* seq_start,
                         const int32_t* seq_len, int n_seq, int max_len, int total, int H, int head_size, int dtype, int head_first, void* stream) {
  if (int e = check_dims(n_seq, max_len, H, head_size, dtype)) return e;
  if (any_null(w, k, v) || (o && !r) || (!o && !states) || (seq_start && !seq_len) || (!seq_start && seq_len)) return RWKVB200_E_NULL;
  if (seq_start && (total <= 0 || head_first)) return RWKVB200_E_SHAPE;
  if (n_state != 0 && n_state != 1 && n_state != n_seq) return RWKVB200_E_SHAPE;
  if (n_state != 0 && !h0) return RWKVB200_E_NULL;
  if (misaligned(r, k, v, h0, o, ht, states, (const char*)workspace)) return RWKVB200_E_ALIGN;
  const bool compact = compact_of(seq_start, states, states_bytes, n_seq, max_len, total, H, head_size, dtype);
  const int slots_of = seq_start && (compact || !states) ? total : 0;
  if (int e = check_sizes(n_seq, max_len, slots_of, H, head_size, dtype)) return e;
  const size_t ns = states_bytes_of(n_seq, max_len, slots_of, H, head_size, dtype, states != nullptr);
  const size_t nw = workspace_bytes_of(n_seq, max_len, slots_of, H, head_size, dtype, w_per_head, 0);
  if ((ns && (!states || states_bytes < ns)) || (nw && (!workspace || workspace_bytes < nw))) return RWKVB200_E_WORKSPACE;
  la::Args a = {};
  a.r = r; a.k = k; a.v = v; a.w = w; a.h0 = n_state ? h0 : nullptr; a.n_state = n_state;
  a.o = o; a.ht = ht; a.states = states; a.scratch = workspace;
  a.w_per_head = w_per_head != 0; a.dtype = dtype; a.D = head_size; a.compact = compact;
  a.tokens = seq_start ? total : (long long)n_seq * max_len;
  a.tok = tokens_of(seq_start, seq_len, n_seq, max_len, total, H, head_size, head_first, w_per_head);
  return la::tc_applies(head_size, dtype) ? la::launch_tc_fwd(a, (cudaStream_t)stream) : la::launch_simt_fwd(a, (cudaStream_t)stream);
}

int rwkvb200_linattn_bwd(const void* r, const float* w, int w_per_head, const void* k, const void* v, const void* d_o, const float* d_ht,
                         const float* states, size_t states_bytes, void* dr, float* dw, void* dk, void* dv, float* dh0, void* workspace,
                         size_t workspace_bytes, const int32_t* seq_start, const int32_t* seq_len, int n_seq, int max_len, int total, int H,
                         int head_size, int dtype, int head_first, void* stream) {
  if (int e = check_dims(n_seq, max_len, H, head_size, dtype)) return e;
  if (any_null(r, w, k, v, d_o, states, dr, dw, dk, dv) || (seq_start && !seq_len) || (!seq_start && seq_len)) return RWKVB200_E_NULL;
  if (seq_start && (total <= 0 || head_first)) return RWKVB200_E_SHAPE;
  if (misaligned(r, k, v, d_o, d_ht, states, dr, dk, dv, dh0, (const char*)workspace)) return RWKVB200_E_ALIGN;
  const bool compact = compact_of(seq_start, states, states_bytes, n_seq, max_len, total, H, head_size, dtype);
  const int slots_of = compact ? total : 0;
  if (int e = check_sizes(n_seq, max_len, slots_of, H, head_size, dtype)) return e;
  const size_t ns = states_bytes_of(n_seq, max_len, slots_of, H, head_size, dtype, 1);
  const size_t nw = workspace_bytes_of(n_seq, max_len, slots_of, H, head_size, dtype, w_per_head, 1);
  if (states_bytes < ns || (nw && (!workspace || workspace_bytes < nw))) return RWKVB200_E_WORKSPACE;
  la::Args a = {};
  a.r = r; a.k = k; a.v = v; a.w = w; a.d_o = d_o; a.d_ht = d_ht;
  a.dr = dr; a.dw = dw; a.dk = dk; a.dv = dv; a.dh0 = dh0; a.states = const_cast<float*>(states); a.scratch = workspace;
  a.w_per_head = w_per_head != 0; a.dtype = dtype; a.D = head_size; a.compact = compact;
  a.tokens = seq_start ? total : (long long)n_seq * max_len;
  a.tok = tokens_of(seq_start, seq_len, n_seq, max_len, total, H, head_size, head_first, w_per_head);
  return la::tc_applies(head_size, dtype) ? la::launch_tc_bwd(a, (cudaStream_t)stream) : la::launch_simt_bwd(a, (cudaStream_t)stream);
}

int rwkvb200_linattn_step(const void* r, const float* w, int w_per_head, const void* k, const void* v, void* state, int state_dtype, void* o,
                          const int64_t* parents, int groups, int beams, int H, int head_size, int dtype, void* stream) {
  if (groups <= 0 || beams <= 0) return RWKVB200_E_SHAPE;
  if (int e = check_dims((long long)groups * beams, 1, H, head_size, dtype)) return e;
  if (state_dtype != RWKVB200_F32 && state_dtype != RWKVB200_BF16) return RWKVB200_E_DTYPE;
  if (any_null(r, w, k, v, state, o)) return RWKVB200_E_NULL;
  if (misaligned(r, k, v, state, o)) return RWKVB200_E_ALIGN;
  if (parents && beams > la::MAX_BEAMS) return RWKVB200_E_TOO_LARGE;
  if (!parents) { groups *= beams; beams = 1; }
  return la::launch_step(r, w, w_per_head ? 0 : H, k, v, state, state_dtype, o, (const long long*)parents, groups, beams, H, head_size, dtype,
                         (cudaStream_t)stream);
}

int rwkvb200_reorder_states(void* state, const int64_t* parents, int groups, int beams, size_t row_bytes, void* stream) {
  if (groups <= 0 || beams <= 0 || row_bytes == 0 || row_bytes % 16) return RWKVB200_E_SHAPE;
  if (any_null((const char*)state, parents)) return RWKVB200_E_NULL;
  if (!aligned16(state)) return RWKVB200_E_ALIGN;
  if (beams > la::MAX_BEAMS || row_bytes > (size_t(1) << 38)) return RWKVB200_E_TOO_LARGE;
  if (beams == 1) return RWKVB200_OK;      // a beam alone is its own parent
  return la::launch_reorder(state, (const long long*)parents, groups, beams, (long long)row_bytes, (cudaStream_t)stream);
}

int rwkvb200_beam_select(const void* logits, int dtype, int64_t group_stride, int64_t beam_stride, const float* scores, const uint8_t* finished,
                         int64_t eos, float* scores_out, int64_t* parents, int64_t* tokens, uint8_t* finished_out, int groups, int beams, int vocab,
                         void* stream) {
  if (groups <= 0 || beams <= 0 || vocab <= 0 || group_stride < 0 || beam_stride < 0) return RWKVB200_E_SHAPE;
  if (eos >= vocab || (eos < 0 && (finished || finished_out))) return RWKVB200_E_SHAPE;
  if (dtype != RWKVB200_F32 && dtype != RWKVB200_BF16 && dtype != RWKVB200_F16) return RWKVB200_E_DTYPE;
  if (any_null((const char*)logits, scores, scores_out, parents, tokens)) return RWKVB200_E_NULL;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == RWKVB200_F32 ? 4 : 2)) return RWKVB200_E_ALIGN;
  if (beams > la::MAX_BEAMS || vocab > (1 << 30)) return RWKVB200_E_TOO_LARGE;
  return launch_beam_select(logits, dtype, group_stride, beam_stride, scores, finished, eos < 0 ? -1 : eos, scores_out, (long long*)parents,
                            (long long*)tokens, finished_out, groups, beams, vocab, (cudaStream_t)stream);
}

}  // extern "C"
