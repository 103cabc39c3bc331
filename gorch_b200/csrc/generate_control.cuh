// generate_control_kernel: the bookkeeping of the reference's generate loops for a batch of
// sequences, on the device, so that a decode step needs no host round trip: after the sampling
// kernels have written one token id per row, this kernel applies the loop's rules to every row
// that is still live and leaves what the model's next forward needs in device memory.
//
// Rules (one iteration of the loops of model/generate.go:60-88 (uncached), :107-129 (cached) and
// model/qwen/generate.go:47-61), in the reference's order:
//   1. the iteration limit `i < MaxNewTokens` is tested before anything else;
//   2. a stop token ends the sequence and is NOT appended (generate.go:82-84; qwen isStop :54-56);
//   3. the token is appended to the result;
//   4. cached loops: if the cache already holds MaxSeq positions the sequence ends (the token
//      stays appended, no forward follows; generate.go:121-123, qwen :58-60); otherwise the token
//      is the next forward's input and the cache grows by one;
//      uncached loop: the next forward's input is the last MaxSeq tokens of the result
//      (generate.go:62-65): its start is written to window_start.
// A row that appends its MaxNewTokens-th token is marked finished at once (the reference runs one
// more forward whose logits it never reads).
//
// One CTA walks all rows (a few words of traffic per row), counts the live ones and writes the
// count for a host that wants to poll it now and then instead of every step.
#pragma once

#include <cstdint>

#include "small_set.cuh"   // pdl_wait, pdl_launch

namespace gs {

constexpr int GC_NT = 256;
constexpr int GC_MAX_STOPS = 16;

// done[] codes
constexpr int GC_LIVE = 0;
constexpr int GC_STOP = 1;       // a stop token was sampled
constexpr int GC_MAX_NEW = 2;    // MaxNewTokens tokens appended
constexpr int GC_MAX_SEQ = 3;    // cached loops: the cache reached MaxSeq
constexpr int GC_ERROR = 4;      // the sampler reported an unusable id, the row's mask leaves nothing to sample, or the token buffer is full

struct GenControlArgs {
  const int32_t* ids;        // [B] this step's sampled ids
  const uint32_t* flags;     // [B] the sampler's row flags, or null
  int32_t* tokens;           // [B, capacity] prompt + appended tokens
  long long capacity;
  int32_t* lengths;          // [B] tokens held per row
  int32_t* n_new;            // [B] tokens appended so far
  int32_t* cache_len;        // [B] positions in the KV cache (cached loops)
  int32_t* done;             // [B] GC_* code
  int32_t* next_input;       // [B] token of the next forward (cached), last token (uncached)
  int32_t* window_start;     // [B] uncached loop: start of the next input window; may be null
  int32_t* live_count;       // [1]
  int32_t stops[GC_MAX_STOPS];
  int n_stop;
  int max_new;
  int max_seq;
  int cached;
  uint32_t bad_flags;        // sampler flags that make an id unusable
  const uint32_t* mask;      // [n_masks, mask_stride] words of allowed tokens, or null
  long long mask_stride;
  int n_masks;
  const int32_t* mask_rows;  // [B] or null: row b has mask b
  // with a mask: the logits that the ids were sampled from (the mask's -Inf in them), and the ids again, to be replaced
  const void* logits;        // [B, row_stride]
  long long row_stride;
  int V, bf16;
  int32_t* out_ids;
  int B;
};

// The index of a row's largest logit, the lowest of equal ones; -1 when that is not finite or the row holds a NaN. All of the CTA's threads.
template <typename T>
__device__ __noinline__ int gc_row_argmax(const GenControlArgs& A, int b, bu::Scratch& sc, int tid) {
  RowView<T> rv;
  rv.init(static_cast<const T*>(A.logits) + b * A.row_stride, A.V);
  unsigned long long best = 0ull;
  bool odd = false;
  constexpr int U = 8;                                        // vectors of a thread on their way together
  for (int v0 = tid; v0 < rv.nvec; v0 += U * GC_NT) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; u++) raw[u] = *(rv.vbase + min(v0 + u * GC_NT, rv.nvec - 1));
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (v0 + u * GC_NT >= rv.nvec) break;
      rv.visit_raw(raw[u], v0 + u * GC_NT, [&](float x, int i, int) {
        odd |= !(x < INFINITY);
        const unsigned long long p = (static_cast<unsigned long long>(okey(x)) << 32) | static_cast<uint32_t>(~i);
        best = p > best ? p : best;
      });
    }
  }
  best = bu::max_u64<GC_NT / 32>(best, sc, tid);
  if (__syncthreads_or(odd) || !(okey_to_float(static_cast<uint32_t>(best >> 32)) > -INFINITY)) return -1;
  return static_cast<int>(~static_cast<uint32_t>(best));
}

// Bound: latency, a launch and two trips to L2: a row's words are read at once, before any decision. The kernel
// starts beside the sampling kernel's last CTAs and waits for them here.
__global__ void __launch_bounds__(GC_NT) generate_control_kernel(const __grid_constant__ GenControlArgs A) {
  __shared__ bu::Scratch sc;
  __shared__ int s_look[GC_NT], s_nlook;
  const int tid = threadIdx.x;
  int live = 0;
  pdl_launch();
  pdl_wait();
  // a usable id: whether the row is still live after it
  auto take = [&](int b, int id, int len, int cl, int n) -> bool {
    bool stop = false;
    for (int s = 0; s < A.n_stop; s++) stop |= (id == A.stops[s]);
    if (stop) { A.done[b] = GC_STOP; return false; }
    if (len >= A.capacity) { A.done[b] = GC_ERROR; return false; }
    A.tokens[static_cast<long long>(b) * A.capacity + len] = id;
    A.lengths[b] = len + 1;
    A.n_new[b] = ++n;
    if (A.cached) {
      if (cl >= A.max_seq) { A.done[b] = GC_MAX_SEQ; return false; }
      A.cache_len[b] = cl + 1;
    } else if (A.window_start != nullptr) {
      A.window_start[b] = (len + 1 > A.max_seq) ? len + 1 - A.max_seq : 0;
    }
    A.next_input[b] = id;
    if (n >= A.max_new) { A.done[b] = GC_MAX_NEW; return false; }
    return true;
  };
  if (tid == 0) s_nlook = 0;
  if (A.mask != nullptr) __syncthreads();
  for (int b0 = 0; b0 < A.B; b0 += GC_NT) {
    const int b = b0 + tid;
    bool look = false;
    if (b < A.B) {
      const int done = A.done[b], id = A.ids[b], len = A.lengths[b], cl = A.cached ? A.cache_len[b] : 0, n = A.n_new[b];
      const uint32_t fl = (A.flags != nullptr) ? A.flags[b] : 0u;
      if (done == GC_LIVE) {
        if (n >= A.max_new) {
          A.done[b] = GC_MAX_NEW;
        } else if (id < 0 || (fl & A.bad_flags) != 0u) {
          A.done[b] = GC_ERROR;
        } else {
          bool allowed = true;
          if (A.mask != nullptr) {
            const int m = A.mask_rows ? A.mask_rows[b] : b;
            allowed = m < 0 || m >= A.n_masks || ((A.mask[m * A.mask_stride + (id >> 5)] >> (id & 31)) & 1u) != 0u;
          }
          look = !allowed;
          if (allowed) live += take(b, id, len, cl, n) ? 1 : 0;
        }
      }
    }
    // An id that the mask does not allow: it leaves nothing, or the row cannot be sampled from (NaN, +Inf), or the draw ran past the last
    // kept token, which gives V - 1 whatever the mask (rounding, with a uniform next to 1; mode A's top_p, which may
    // remove every token). In the last case the row's largest logit, which the mask allows, takes its place. All of them are rare, and end
    // the row or happen once in a long while: a row's scan by this one CTA (30 us for 151,936 columns) is no cost to speak of.
    if (A.mask == nullptr || !__syncthreads_or(look)) continue;
    if (look) s_look[atomicAdd(&s_nlook, 1)] = b;
    __syncthreads();
    const int nlook = s_nlook;
    for (int i = 0; i < nlook; i++) {
      const int row = s_look[i];
      const int id = A.bf16 ? gc_row_argmax<uint16_t>(A, row, sc, tid) : gc_row_argmax<float>(A, row, sc, tid);
      if (tid == 0) {
        if (id < 0) {
          A.done[row] = GC_ERROR;
        } else {
          A.out_ids[row] = id;
          live += take(row, id, A.lengths[row], A.cached ? A.cache_len[row] : 0, A.n_new[row]) ? 1 : 0;
        }
      }
    }
    __syncthreads();
    if (tid == 0) s_nlook = 0;
    __syncthreads();
  }
  live = bu::sum_i<GC_NT / 32>(live, sc, tid);
  if (tid == 0) *A.live_count = live;
}

}  // namespace gs
