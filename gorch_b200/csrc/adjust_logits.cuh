// The rules of a request on its logits, between the LM head and the sampling step: penalties for tokens that the
// request already holds, biases, and the mask of a grammar. (The reference samples from the bare logits,
// model/generate.go:75-79; these are what a serving program puts in front of that line.) For a row b and a token v
//   c = how often v occurs among the row's generated tokens, held = v occurs in its prompt or among them
//   y = held ? (x > 0 ? x / repetition : x * repetition) : x
//   y = c > 0 ? (y - frequency * c) - presence : y
//   y = y + bias                (of the last entry listed for v)
//   y = -Inf                    where the row's mask has a 0 for v, whatever x held
// in f32, each operation rounded once, and one rounding to bf16 at the end for bf16 logits. A logit that no rule
// touches keeps its bits.
//
// Without penalties and biases, adjust_rows_kernel: a stream over every column (in place it writes what the mask takes away, and
// reads the vectors of which the mask keeps some).
// With them, a CTA takes ranges of a row's columns and counts the tokens that fall into a range in shared memory, a word of 16 or 32
// bits per column (integer atomics: the order does not matter). Meanwhile the range's logits are on their way to shared
// memory; the touched ones are changed there, and the range leaves for the output with the mask applied on the way. In place only
// the touched logits are read, and written where they lie; behind a barrier the mask goes over the range. Two kernels: adjust_stream_kernel for short histories,
// adjust_touched_kernel, whose CTAs each walk the row's whole history, for long ones.
// Bound: memory out of place, one read and one write of the row (512 x 151,936 with 1,000 tokens each: bf16 61 us, 5.1 TB/s; f32 106 us, 5.9
// TB/s; with 16 biases and a mask for half of the rows besides, bf16 68 us; the copy alone 47 and 92); in place, where little is moved, the latency of three trips to L2 one after the other
// (lengths, tokens, logits): 64 rows with 2,048 tokens each 12 us, 512 with 1,000 each 22 us.
// Other splits that were measured for those 512 bf16 rows: the rules in a kernel of their own behind the copy, 66 us (it reads and
// writes single sectors that have left L2 by then); a hash table of the tokens in place of the words, 75 us; a look at
// the words for every logit that passes, 191 us.
#pragma once

#include <cstdint>

#include "row_softmax.cuh"   // bf16_bits_rne

namespace gs {

constexpr int AL_NT = 256;
constexpr int AL_NW = AL_NT / 32;
constexpr int AL_T_NT = 512;                  // adjust_touched_kernel
constexpr int AL_T_NW = AL_T_NT / 32;
constexpr int AL_T_BATCH = 8;                 // its loads of tokens
constexpr int AL_MASK_CHUNK = 8 * AL_NT;      // adjust_rows_kernel in place: vectors of a CTA
constexpr int AL_REG_TOKENS = 16 * AL_NT;     // of a row that adjust_stream_kernel takes
constexpr int AL_U = 4;                       // adjust_rows_kernel: 16-byte vectors per thread
constexpr int AL_BATCH = 4;                   // touched columns that a lane works on together
constexpr int AL_LIST = 32 * AL_BATCH + 64;   // touched columns that a warp collects before it works on them
constexpr int AL_MAX_COLS = 16384;            // of a range
constexpr int AL_STAGE_BYTES = 16384;         // adjust_stream_kernel out of place: logits of a range

struct AdjustArgs {
  const void* x;                  // [B, row_stride]
  int64_t row_stride;
  void* out;                      // [B, out_stride]; x itself in place
  int64_t out_stride;
  int32_t V;
  int32_t chunk, nchunk;          // 16-byte vectors of a row that a CTA takes (a multiple of 8), CTAs per row
  const float* penalties;         // [B][4]: repetition, presence, frequency, unused; or null
  const int32_t* history;         // [B, history_stride] token ids
  int64_t history_stride;
  const int32_t* lengths;         // [B]
  const int32_t* prompt_lengths;  // [B] or null: 0
  const int32_t* n_new;           // [B] or null: the generated tokens are the last n_new (instead of prompt_lengths)
  const int32_t* bias_offsets;    // [B + 1] or null
  const int32_t* bias_ids;
  const float* bias_values;
  int32_t n_bias;
  const uint32_t* mask;           // [n_masks, mask_stride] words, or null
  int64_t mask_stride;
  int32_t n_masks;
  const int32_t* mask_rows;       // [B] or null: row b has mask b
  const int32_t* row_done;        // [B] or null: rows that are not 0 here are left alone
  int32_t wide;                   // counts of 32 bits: histories of 2^15 tokens and more
  int32_t shared_out;             // both kernels run: rows of more than AL_REG_TOKENS tokens are adjust_touched_kernel's, the others the other's
};

__device__ __forceinline__ const uint32_t* al_mask_row(const AdjustArgs& A, int64_t row) {
  if (A.mask == nullptr) return nullptr;
  const int64_t m = A.mask_rows ? A.mask_rows[row] : row;
  return (m >= 0 && m < A.n_masks) ? A.mask + m * A.mask_stride : nullptr;
}

// A vector of which the mask's bits keep some elements: -Inf for the others. Four bits go to the top of four bytes (bit i of b times
// 2^(7 j + 7) lands on bit 8 i + 7 for j = i alone, and no two products on one place), and prmt repeats a byte's top bit.
__device__ __forceinline__ uint32_t al_spread(uint32_t four_bits) { return four_bits * 0x10204080u; }
template <uint32_t SEL>
__device__ __forceinline__ uint32_t al_keep(uint32_t r, uint32_t spread, uint32_t neg_inf) {
  uint32_t m;
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(m) : "r"(spread), "n"(SEL));
  return (r & m) | (neg_inf & ~m);
}
template <typename T>
__device__ __forceinline__ uint4 al_masked(const uint4& r, uint32_t bits) {
  uint4 o;
  const uint32_t lo = al_spread(bits & 15u);
  if (sizeof(T) == 4) {
    o.x = al_keep<0x8888>(r.x, lo, 0xff800000u); o.y = al_keep<0x9999>(r.y, lo, 0xff800000u);
    o.z = al_keep<0xaaaa>(r.z, lo, 0xff800000u); o.w = al_keep<0xbbbb>(r.w, lo, 0xff800000u);
  } else {
    const uint32_t hi = al_spread(bits >> 4);
    o.x = al_keep<0x9988>(r.x, lo, 0xff80ff80u); o.y = al_keep<0xbbaa>(r.y, lo, 0xff80ff80u);
    o.z = al_keep<0x9988>(r.z, hi, 0xff80ff80u); o.w = al_keep<0xbbaa>(r.w, hi, 0xff80ff80u);
  }
  return o;
}

// The mask's bits for the VEC columns from i0 on, which may begin below 0 (columns outside the row: any). aligned: i0 is a multiple of VEC
// (a row that starts on 16 bytes): the bits lie in one byte.
template <int VEC>
__device__ __forceinline__ uint32_t al_mask_bits(const uint32_t* mrow, int i0, int last_word, bool aligned) {
  constexpr uint32_t ALL = (1u << VEC) - 1u;
  if (mrow == nullptr) return ALL;
  if (aligned) return (static_cast<uint32_t>(__ldg(reinterpret_cast<const unsigned char*>(mrow) + (i0 >> 3))) >> (i0 & 7)) & ALL;
  if (i0 < 0) return (__ldg(mrow) << -i0) & ALL;
  return __funnelshift_r(__ldg(mrow + (i0 >> 5)), __ldg(mrow + min((i0 >> 5) + 1, last_word)), i0 & 31) & ALL;
}

// A vector (columns i0 ..) to the output row with the masked elements at -Inf. A row's first and last vector hold elements of others:
// element by element; in place those that the mask keeps are not written there.
template <typename T, bool IN_PLACE>
__device__ __forceinline__ void al_store(T* orow, bool vec_ok, int V, int i0, const uint4& raw, uint32_t bits) {
  constexpr int VEC = Elem<T>::VEC;
  const uint4 o = al_masked<T>(raw, bits);
  if (vec_ok && i0 >= 0 && i0 + VEC <= V) {
    *reinterpret_cast<uint4*>(orow + i0) = o;
    return;
  }
  const uint32_t ow[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
  for (int c = 0; c < VEC; c++) {
    const int i = i0 + c;
    if (i < 0 || i >= V || (IN_PLACE && ((bits >> c) & 1u))) continue;
    if (sizeof(T) == 4) reinterpret_cast<uint32_t*>(orow)[i] = ow[c & 3];
    else reinterpret_cast<uint16_t*>(orow)[i] = static_cast<uint16_t>(ow[c >> 1] >> (16 * (c & 1)));
  }
}

// The mask in place, over the vectors v0 .. v1 - 1 by NT threads: what it takes away is written, a vector of which it keeps some read first.
// Rows that start on 16 bytes go by two vectors and the mask's one or two bytes for them: where little is kept the instructions
// count (256 x 151,936 f32, 0.2 % kept, us: by vectors 41, so 34).
template <typename T, int NT>
__device__ __forceinline__ void al_mask_in_place(T* orow, const RowView<T>& rv, const uint32_t* mrow, int v0, int v1, int tid) {
  constexpr int VEC = Elem<T>::VEC, U = 4, P = 2;
  constexpr uint32_t ALL = (1u << VEC) - 1u, NEG = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
  constexpr uint32_t PAIR = VEC == 4 ? 0xffu : 0xffffu;
  const uint4 neg = make_uint4(NEG, NEG, NEG, NEG);
  int v = v0;                                                          // the first vector that the pairs leave
  if (rv.shift == 0) {
    const int pairs = (min(v1, rv.V / VEC) - v0) >> 1;
    uint4* at = reinterpret_cast<uint4*>(orow) + v0;                   // (v0 is even: a pair's bits begin a byte)
    for (int q0 = tid; q0 < pairs; q0 += P * NT) {
      uint32_t bits[P];
      uint4 raw[2 * P];
#pragma unroll
      for (int u = 0; u < P; u++) {
        const int q = q0 + u * NT;
        bits[u] = q >= pairs ? PAIR : VEC == 4 ? __ldg(reinterpret_cast<const unsigned char*>(mrow) + (v0 >> 1) + q)
                                               : __ldg(reinterpret_cast<const unsigned short*>(mrow) + (v0 >> 1) + q);
      }
#pragma unroll
      for (int u = 0; u < P; u++) {
        const uint4* from = at + 2 * (q0 + u * NT);
        raw[2 * u] = raw[2 * u + 1] = neg;
        if (bits[u] != 0u && bits[u] != PAIR) { raw[2 * u] = al_masked<T>(from[0], bits[u] & ALL); raw[2 * u + 1] = al_masked<T>(from[1], bits[u] >> VEC); }
      }
#pragma unroll
      for (int u = 0; u < P; u++) {
        uint4* to = at + 2 * (q0 + u * NT);
        if (bits[u] != PAIR) { to[0] = raw[2 * u]; to[1] = raw[2 * u + 1]; }
      }
    }
    v = v0 + 2 * max(pairs, 0);
  }
  const int last_word = (rv.V - 1) >> 5;
  for (v += tid; v < v1; v += U * NT) {
    uint32_t bits[U];
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int w = v + u * NT;
      bits[u] = w < v1 ? al_mask_bits<VEC>(mrow, w * VEC - rv.shift, last_word, rv.shift == 0) : ALL;
    }
#pragma unroll
    for (int u = 0; u < U; u++) raw[u] = (bits[u] != ALL && bits[u] != 0u) ? *(rv.vbase + v + u * NT) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int i0 = (v + u * NT) * VEC - rv.shift;
      if (bits[u] != ALL) al_store<T, true>(orow, true, rv.V, i0, raw[u], bits[u]);
    }
  }
}

template <typename T, bool IN_PLACE>
__global__ void __launch_bounds__(AL_NT) adjust_rows_kernel(const __grid_constant__ AdjustArgs A) {
  constexpr int VEC = Elem<T>::VEC, U = AL_U;
  constexpr uint32_t ALL = (1u << VEC) - 1u;
  const int64_t row = blockIdx.x / static_cast<unsigned>(A.nchunk);
  const int part = static_cast<int>(blockIdx.x - static_cast<unsigned>(row) * static_cast<unsigned>(A.nchunk));
  pdl_launch();
  pdl_wait();                                                        // whatever fills the inputs, or still reads the output
  if (A.row_done != nullptr && A.row_done[row] != 0) return;
  RowView<T> rv;
  rv.init(static_cast<const T*>(A.x) + row * A.row_stride, A.V);
  const int v0 = part * (AL_NT * U) + threadIdx.x;
  const uint32_t* mrow = al_mask_row(A, row);
  T* orow = static_cast<T*>(A.out) + row * A.out_stride;
  if constexpr (IN_PLACE) {
    if (mrow != nullptr) al_mask_in_place<T, AL_NT>(orow, rv, mrow, part * A.chunk, min((part + 1) * A.chunk, rv.nvec), threadIdx.x);
  } else {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int v = v0 + u * AL_NT;
      raw[u] = v < rv.nvec ? __ldg(rv.vbase + v) : make_uint4(0u, 0u, 0u, 0u);
    }
    const int last_word = (A.V - 1) >> 5;
    uint32_t bits[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int v = v0 + u * AL_NT;
      bits[u] = v < rv.nvec ? al_mask_bits<VEC>(mrow, v * VEC - rv.shift, last_word, rv.shift == 0) : ALL;
    }
    const bool vec_ok = ((reinterpret_cast<uintptr_t>(orow) - static_cast<uintptr_t>(rv.shift) * sizeof(T)) & 15u) == 0;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int v = v0 + u * AL_NT;
      if (v < rv.nvec) al_store<T, false>(orow, vec_ok, A.V, v * VEC - rv.shift, raw[u], bits[u]);
    }
  }
}

// Shared memory of adjust_touched_kernel for a range of `cols` columns: counts, and out of place the logits.
__host__ __device__ inline int al_count_bytes(int cols, bool wide) { return wide ? 4 * cols : 2 * cols; }
inline int al_dyn_bytes(int cols, bool wide, int elem, bool in_place) { return al_count_bytes(cols, wide) + (in_place ? 0 : cols * elem); }

template <typename T, bool IN_PLACE>
__global__ void __launch_bounds__(AL_T_NT) adjust_touched_kernel(const __grid_constant__ AdjustArgs A) {
  constexpr int VEC = Elem<T>::VEC;
    extern __shared__ __align__(16) unsigned char al_dyn[];
  __shared__ uint16_t s_list[AL_T_NW][AL_LIST];
  __shared__ int s_ids[AL_T_NT];
  __shared__ uint32_t s_done[AL_MAX_COLS / 32];                      // columns whose bias has been served
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / static_cast<unsigned>(A.nchunk);
  const int part = static_cast<int>(blockIdx.x - static_cast<unsigned>(row) * static_cast<unsigned>(A.nchunk));
  const int cols = A.chunk * VEC;
  const bool wide = A.wide != 0;
  uint32_t* words = reinterpret_cast<uint32_t*>(al_dyn);
  T* data = reinterpret_cast<T*>(al_dyn + al_count_bytes(cols, wide));
  pdl_launch();
  pdl_wait();                                                        // whatever fills the inputs, or still reads the output
  if (A.row_done != nullptr && A.row_done[row] != 0) return;
  if (A.shared_out && min(static_cast<int64_t>(A.lengths[row]), A.history_stride) <= AL_REG_TOKENS) return;
  const T* xrow = static_cast<const T*>(A.x) + row * A.row_stride;
  T* orow = static_cast<T*>(A.out) + row * A.out_stride;
  RowView<T> rv;
  rv.init(xrow, A.V);
  const int v0 = part * A.chunk, v1 = min(v0 + A.chunk, rv.nvec);
  if (v0 >= v1) return;                                              // (rows differ by a vector, depending on where they start)
  if (!IN_PLACE) {
    const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(data));
    for (int v = v0 + tid; v < v1; v += AL_T_NT)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(at + static_cast<uint32_t>(v - v0) * 16u), "l"(rv.vbase + v) : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  const int c0 = v0 * VEC - rv.shift;                                // column of the range's first element: below 0 in a row's first vector
  const int lo = max(c0, 0), hi = min(v1 * VEC - rv.shift, A.V);
  const uint32_t* mrow = al_mask_row(A, row);
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  int len = 0, prompt = 0, off0 = 0, off1 = 0;
  if (A.penalties != nullptr) {
    rep = A.penalties[4 * row]; pres = A.penalties[4 * row + 1]; freq = A.penalties[4 * row + 2];
    len = static_cast<int>(min(static_cast<int64_t>(max(A.lengths[row], 0)), A.history_stride));
    if (A.n_new != nullptr) prompt = len - A.n_new[row];
    else if (A.prompt_lengths != nullptr) prompt = A.prompt_lengths[row];
    if (rep == 1.0f && pres == 0.0f && freq == 0.0f) len = 0;        // a row without penalties does not read its history
  }
  if (A.bias_offsets != nullptr) {
    off0 = min(max(A.bias_offsets[row], 0), A.n_bias);
    off1 = min(max(A.bias_offsets[row + 1], off0), A.n_bias);
  }
  if (len > 0 || off1 > off0) {
    uint4* w4 = reinterpret_cast<uint4*>(words);
    for (int i = tid; i < al_count_bytes(cols, wide) / 16; i += AL_T_NT) w4[i] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
  }

  // ---- the history: the tokens in batches, so that a thread has several loads on their way before it looks at the first
  auto add = [&](int t, int i) {
    if (t < lo || t >= hi) return;
    const int e = t - c0;
    if (wide) {
      if (i < prompt) atomicOr(&words[e], 0x80000000u); else atomicAdd(&words[e], 1u);
    } else {
      const int sh = (e & 1) * 16;                                   // (fewer than 2^15 tokens: a count does not reach the next bit)
      if (i < prompt) atomicOr(&words[e >> 1], 0x8000u << sh); else atomicAdd(&words[e >> 1], 1u << sh);
    }
  };
  if (len > 0) {
    const int32_t* hist = A.history + row * A.history_stride;
    if ((reinterpret_cast<uintptr_t>(hist) & 15u) == 0) {
      const int4* h4 = reinterpret_cast<const int4*>(hist);
      const int nq = len >> 2;
      for (int q0 = tid; q0 < nq; q0 += AL_T_BATCH * AL_T_NT) {
        int4 t[AL_T_BATCH];
#pragma unroll
        for (int j = 0; j < AL_T_BATCH; j++) t[j] = (q0 + j * AL_T_NT < nq) ? __ldg(h4 + q0 + j * AL_T_NT) : make_int4(-1, -1, -1, -1);
#pragma unroll
        for (int j = 0; j < AL_T_BATCH; j++) {
          const int i = 4 * (q0 + j * AL_T_NT);
          add(t[j].x, i); add(t[j].y, i + 1); add(t[j].z, i + 2); add(t[j].w, i + 3);
        }
      }
      const int i = 4 * nq + tid;
      if (i < len) add(__ldg(hist + i), i);
    } else {
      for (int i0 = tid; i0 < len; i0 += AL_T_BATCH * AL_T_NT) {
        int t[AL_T_BATCH];
#pragma unroll
        for (int j = 0; j < AL_T_BATCH; j++) t[j] = (i0 + j * AL_T_NT < len) ? __ldg(hist + i0 + j * AL_T_NT) : -1;
#pragma unroll
        for (int j = 0; j < AL_T_BATCH; j++) add(t[j], i0 + j * AL_T_NT);
      }
    }
  }
  if (!IN_PLACE) asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();

  auto word_of = [&](int e) -> uint32_t {                            // the column's count, "held" in the top bit
    if (wide) return words[e];
    const uint32_t h = (words[e >> 1] >> ((e & 1) * 16)) & 0xffffu;
    return (h & 0x7fffu) | ((h & 0x8000u) << 16);
  };
  auto penalised = [&](float x, uint32_t w) -> float {
    float y = (x > 0.0f) ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
    const uint32_t n = w & 0x7fffffffu;
    if (n != 0u) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, static_cast<float>(n))), pres);
    return y;
  };
  auto put = [&](T* at, float y) {
    if (sizeof(T) == 4) *reinterpret_cast<float*>(at) = y;
    else *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(bf16_bits_rne(y));
  };
  auto allowed = [&](int t) -> bool { return mrow == nullptr || ((__ldg(mrow + (t >> 5)) >> (t & 31)) & 1u) != 0u; };

  // ---- the biases, from the last entry to the first, AL_T_NT at a time: the last one for a column counts. A biased column is
  // finished here, its penalties included, and its count taken away.
  if (off1 > off0) {
    for (int i = tid; i < (cols + 31) / 32; i += AL_T_NT) s_done[i] = 0u;
    for (int top = off1; top > off0; top -= AL_T_NT) {
      const int i = top - 1 - tid;
      const int t = (i >= off0) ? __ldg(A.bias_ids + i) : -1;
      const bool mine = t >= lo && t < hi;
      const float value = mine ? __ldg(A.bias_values + i) : 0.0f;
      s_ids[tid] = mine ? t : -1;
      if (!__syncthreads_or(mine)) continue;
      bool last = mine && ((s_done[(t - c0) >> 5] >> ((t - c0) & 31)) & 1u) == 0u;
      if (last) for (int j = 0; j < tid; j++) if (s_ids[j] == t) { last = false; break; }
      __syncthreads();
      if (last) {
        const int e = t - c0;
        atomicOr(&s_done[e >> 5], 1u << (e & 31));
        const uint32_t w = word_of(e);
        if (wide) words[e] = 0u;
        else if (w != 0u) atomicAnd(&words[e >> 1], (e & 1) ? 0x0000ffffu : 0xffff0000u);
        if (!IN_PLACE || allowed(t)) {
          const float x = Elem<T>::to_float(IN_PLACE ? xrow[t] : data[e]);
          put(IN_PLACE ? orow + t : data + e, __fadd_rn(w != 0u ? penalised(x, w) : x, value));
        }
      }
      __syncthreads();
    }
  }

  // ---- the penalties: every warp walks its share of the counts, collects the touched columns and works on them
  // AL_BATCH per lane at a time
  if (len > 0) {
    int held = 0;
    auto flush = [&](int n) {                                        // the last n of the list
      __syncwarp();
      int e[AL_BATCH];
      T x[AL_BATCH];
      bool go[AL_BATCH];
#pragma unroll
      for (int j = 0; j < AL_BATCH; j++) {
        const bool on = j * 32 + lane < n;
        e[j] = on ? s_list[warp][held - n + j * 32 + lane] : 0;
        go[j] = on && (!IN_PLACE || allowed(c0 + e[j]));
        if (go[j]) x[j] = IN_PLACE ? xrow[c0 + e[j]] : data[e[j]];
      }
#pragma unroll
      for (int j = 0; j < AL_BATCH; j++)
        if (go[j]) put(IN_PLACE ? orow + c0 + e[j] : data + e[j], penalised(Elem<T>::to_float(x[j]), word_of(e[j])));
      held -= n;
      __syncwarp();
    };
    const int nw = al_count_bytes(cols, wide) / 4;
    for (int i0 = warp * 32; i0 < nw; i0 += AL_T_NT) {
      const int i = i0 + lane;
      const uint32_t w = (i < nw) ? words[i] : 0u;
      const uint32_t first = __ballot_sync(FULL, wide ? w != 0u : (w & 0xffffu) != 0u), second = __ballot_sync(FULL, !wide && (w >> 16) != 0u);
      if ((first | second) == 0u) continue;
      const uint32_t below = (1u << lane) - 1u;
      if ((first >> lane) & 1u) s_list[warp][held + __popc(first & below)] = static_cast<uint16_t>(wide ? i : 2 * i);
      held += __popc(first);
      if ((second >> lane) & 1u) s_list[warp][held + __popc(second & below)] = static_cast<uint16_t>(2 * i + 1);
      held += __popc(second);
      if (held >= 32 * AL_BATCH) flush(32 * AL_BATCH);
    }
    if (held > 0) flush(held);
  }

  // ---- the range, out of place; in place what the mask takes away
  __syncthreads();
  if (IN_PLACE) {
    if (mrow != nullptr) al_mask_in_place<T, AL_T_NT>(orow, rv, mrow, v0, v1, tid);
    return;
  }
  const int last_word = (A.V - 1) >> 5;
  const bool vec_ok = ((reinterpret_cast<uintptr_t>(orow) - static_cast<uintptr_t>(rv.shift) * sizeof(T)) & 15u) == 0;
#pragma unroll 4
  for (int v = v0 + tid; v < v1; v += AL_T_NT) {
    const int i0 = v * VEC - rv.shift;
    al_store<T, false>(orow, vec_ok, A.V, i0, reinterpret_cast<const uint4*>(data)[v - v0], al_mask_bits<VEC>(mrow, i0, last_word, rv.shift == 0));
  }
}

// ---- histories of up to AL_REG_TOKENS tokens. The grid is the GPU's, and a CTA goes over a run of ranges, most of them of one row. At
// a row's first range it reads the tokens into registers and sorts them by range into a list (every warp counts its own tokens per
// range, so that few stand in line for an address). Counting a range is then a pass over its part of the list, and so is
// finding the touched columns again: the first thread that takes a column's count away works on it, which also leaves the
// counts at zero for the next range. The next ranges' logits are on their way meanwhile.
// (With a pass over all the row's tokens for every range, 512 x 151,936 bf16 with 1,000 tokens each took 74 us: 630 instructions a
// warp and range, most of them with a lane or two at work.)
constexpr int AL_STREAM_PER_SM = 4;           // CTAs of 64 registers a thread
constexpr int AL_BINS = 64;                   // ranges of a row that are sorted for at a time
constexpr int AL_BUFS = 2;                    // ranges in shared memory: the one worked on, and one on its way
constexpr int AL_STREAM_STATIC = AL_REG_TOKENS * 2 + AL_NT * 4 + AL_BINS * AL_NW * 4 + AL_MAX_COLS / 8 + 512;   // at most; of its static shared memory
inline int al_stream_bytes(int cols, int elem, bool in_place) { return 2 * cols + (in_place ? 0 : AL_BUFS * cols * elem); }

template <typename T, bool IN_PLACE>
__global__ void __launch_bounds__(AL_NT, 4) adjust_stream_kernel(const __grid_constant__ AdjustArgs A, const int64_t total) {
  constexpr int VEC = Elem<T>::VEC;
  constexpr uint32_t ALL = (1u << VEC) - 1u;
  extern __shared__ __align__(16) unsigned char al_dyn[];
  __shared__ __align__(16) int s_ids[AL_NT];
  __shared__ uint16_t s_tok[AL_REG_TOKENS];                          // column within its range, 0x8000: a generated token
  __shared__ int s_bin[AL_BINS][AL_NW], s_start[AL_BINS + 1];
  __shared__ uint32_t s_done[AL_MAX_COLS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cols = A.chunk * VEC;
  uint32_t* words = reinterpret_cast<uint32_t*>(al_dyn);
  T* data = nullptr;
  for (int i = tid; i < cols / 8; i += AL_NT) reinterpret_cast<uint4*>(words)[i] = make_uint4(0u, 0u, 0u, 0u);
  const int64_t u1 = total * (blockIdx.x + 1) / gridDim.x;
  int64_t u = total * blockIdx.x / gridDim.x;
  pdl_launch();
  pdl_wait();                                                        // whatever fills the inputs, or still reads the output
  // the range that comes next on its way: ahead of the one worked on
  int64_t f_row = u / A.nchunk;
  int f_part = static_cast<int>(u - f_row * A.nchunk), f_left = static_cast<int>(u1 - u), f_buf = 0;
  auto fetch = [&]() {
    if (IN_PLACE) return;
    if (f_left > 0) {
      RowView<T> rv;
      rv.init(static_cast<const T*>(A.x) + f_row * A.row_stride, A.V);
      const int a0 = f_part * A.chunk, n = min(A.chunk, rv.nvec - a0);
      const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(al_dyn)) + 2u * cols + static_cast<uint32_t>(f_buf * cols * static_cast<int>(sizeof(T)));
      for (int v = tid; v < n; v += AL_NT)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(at + static_cast<uint32_t>(v) * 16u), "l"(rv.vbase + a0 + v) : "memory");
      if (++f_part == A.nchunk) { f_part = 0; f_row++; }
      if (++f_buf == AL_BUFS) f_buf = 0;
      f_left--;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int i = 0; i < AL_BUFS - 1; i++) fetch();
  __syncthreads();                                                   // the counts are at zero
  int64_t row = u / A.nchunk;
  int part = static_cast<int>(u - row * A.nchunk), left = static_cast<int>(u1 - u), buf = 0;
  int bin = AL_BINS;                                                 // the range's place among those sorted for; AL_BINS: not yet
  bool any = false;                                                  // the row has penalties
  int b_id = -1;                                                     // of a row with at most AL_NT biases: this thread's, if no later one is for its token
  float b_value = 0.0f;
  bool live = true;
  const uint32_t* mrow = nullptr;
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  int off0 = 0, off1 = 0;
  auto penalised = [&](float x, uint32_t h) -> float {
    float y = (x > 0.0f) ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
    const uint32_t n = h & 0x7fffu;
    if (n != 0u) y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, static_cast<float>(n))), pres);
    return y;
  };
  auto put = [&](T* at, float y) {
    if (sizeof(T) == 4) *reinterpret_cast<float*>(at) = y;
    else *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(bf16_bits_rne(y));
  };
  for (; left > 0; left--) {
    if (bin == AL_BINS) {                                            // a row's first range, or one beyond those sorted for
      bin = 0;
      // what says how many tokens and biases the row has; then those, all on their way at once
      live = A.row_done == nullptr || A.row_done[row] == 0;
      mrow = al_mask_row(A, row);
      off0 = off1 = 0;
      any = false;
      int len = 0, prompt = 0;
      if (A.bias_offsets != nullptr && live) {
        off0 = min(max(A.bias_offsets[row], 0), A.n_bias);
        off1 = min(max(A.bias_offsets[row + 1], off0), A.n_bias);
      }
      if (A.penalties != nullptr && live) {
        rep = A.penalties[4 * row]; pres = A.penalties[4 * row + 1]; freq = A.penalties[4 * row + 2];
        len = static_cast<int>(min(static_cast<int64_t>(max(A.lengths[row], 0)), A.history_stride));
        if (A.n_new != nullptr) prompt = len - A.n_new[row];
        else if (A.prompt_lengths != nullptr) prompt = A.prompt_lengths[row];
        if (A.shared_out && len > AL_REG_TOKENS) { live = false; len = off0 = off1 = 0; }
        any = len > 0 && (rep != 1.0f || pres != 0.0f || freq != 0.0f);   // (a row without penalties does not read its history)
      }
      const int n_own = off1 - off0 <= AL_NT ? off1 - off0 : 0;
      if (any || n_own > 0) {
        const int mine = off1 - 1 - tid;                             // a thread's bias: the last one's is thread 0
        b_id = tid < n_own ? __ldg(A.bias_ids + mine) : -1;
        b_value = tid < n_own ? __ldg(A.bias_values + mine) : 0.0f;
        {
          const int32_t* hist = A.history + (any ? row * A.history_stride : 0);
          const bool quads = (reinterpret_cast<uintptr_t>(hist) & 15u) == 0;
          const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(static_cast<const T*>(A.x) + row * A.row_stride) & 15u) / sizeof(T));
          int tok[16], at[16];
          if (!any) len = 0;
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int i = 4 * (j * AL_NT + tid);
            if (quads && i + 4 <= len) {
              const int4 t = __ldg(reinterpret_cast<const int4*>(hist + i));
              tok[4 * j] = t.x; tok[4 * j + 1] = t.y; tok[4 * j + 2] = t.z; tok[4 * j + 3] = t.w;
            } else {
#pragma unroll
              for (int c = 0; c < 4; c++) tok[4 * j + c] = (i + c < len) ? __ldg(hist + i + c) : -1;
            }
          }
          s_ids[tid] = b_id;
          for (int i = tid; i < AL_BINS * AL_NW; i += AL_NT) s_bin[i / AL_NW][i % AL_NW] = 0;
          __syncthreads();
          bool later = false;                                        // a later entry names the same token
#pragma unroll 4
          for (int j = 0; j < n_own; j += 4) {
            const int4 o = *reinterpret_cast<const int4*>(&s_ids[j]);
            later |= (o.x == b_id && j < tid) || (o.y == b_id && j + 1 < tid) || (o.z == b_id && j + 2 < tid) || (o.w == b_id && j + 3 < tid);
          }
          if (later) b_id = -1;
          const int njs = (len + 4 * AL_NT - 1) / (4 * AL_NT);       // groups of four tokens that hold any
#pragma unroll
          for (int j = 0; j < 4; j++) {
            if (j >= njs) break;
#pragma unroll
            for (int c = 0; c < 4; c++) {
              const int t = tok[4 * j + c];
              int b = -1;
              if (t >= 0 && t < A.V) {
                const unsigned col = static_cast<unsigned>(t) + static_cast<unsigned>(shift);
                const unsigned p = col / static_cast<unsigned>(cols) - static_cast<unsigned>(part);
                if (p < static_cast<unsigned>(AL_BINS)) {
                  b = static_cast<int>(p);
                  at[4 * j + c] = atomicAdd(&s_bin[b][warp], 1);
                  tok[4 * j + c] = static_cast<int>(col % static_cast<unsigned>(cols)) | ((4 * (j * AL_NT + tid) + c >= prompt) ? 0x8000 : 0) | (b << 16);
                }
              }
              if (b < 0) tok[4 * j + c] = -1;
            }
          }
          __syncthreads();
          if (warp == 0) {                                           // where each range's tokens begin, and each warp's among them
            static_assert(AL_BINS == 64, "two ranges per lane");
            int n0 = 0, n1 = 0;
            for (int w = 0; w < AL_NW; w++) { n0 += s_bin[2 * lane][w]; n1 += s_bin[2 * lane + 1][w]; }
            int incl = n0 + n1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const int up = __shfl_up_sync(FULL, incl, o); if (lane >= o) incl += up; }
            int begin = incl - n0 - n1;
            s_start[2 * lane] = begin;
            for (int w = 0; w < AL_NW; w++) { const int n = s_bin[2 * lane][w]; s_bin[2 * lane][w] = begin; begin += n; }
            s_start[2 * lane + 1] = begin;
            for (int w = 0; w < AL_NW; w++) { const int n = s_bin[2 * lane + 1][w]; s_bin[2 * lane + 1][w] = begin; begin += n; }
            if (lane == 31) s_start[AL_BINS] = begin;
          }
          __syncthreads();
#pragma unroll
          for (int j = 0; j < 4; j++) {
            if (j >= njs) break;
#pragma unroll
            for (int c = 0; c < 4; c++) {
              const int t = tok[4 * j + c];
              if (t >= 0) s_tok[s_bin[t >> 16][warp] + at[4 * j + c]] = static_cast<uint16_t>(t);
            }
          }
          __syncthreads();
        }
      }
    }
    const int l0 = any ? s_start[bin] : 0, l1 = any ? s_start[bin + 1] : 0;   // the range's tokens on the list
    const T* xrow = static_cast<const T*>(A.x) + row * A.row_stride;
    T* orow = static_cast<T*>(A.out) + row * A.out_stride;
    RowView<T> rv;
    rv.init(xrow, A.V);
    const int v0 = part * A.chunk, v1 = min(v0 + A.chunk, rv.nvec);  // (v1 <= v0: a row that starts on a vector has one less)
    const int c0 = v0 * VEC - rv.shift, lo = max(c0, 0), hi = min(v1 * VEC - rv.shift, A.V);
    data = reinterpret_cast<T*>(al_dyn + 2 * cols) + (IN_PLACE ? 0 : buf * cols);
    auto allowed = [&](int t) -> bool { return mrow == nullptr || ((__ldg(mrow + (t >> 5)) >> (t & 31)) & 1u) != 0u; };
    for (int i = l0 + tid; i < l1; i += AL_NT) {
      const uint32_t t = s_tok[i], e = t & 0x7fffu, sh = (e & 1u) * 16u; // (fewer than 2^15 tokens: a count does not reach the next bit)
      if (t & 0x8000u) atomicAdd(&words[e >> 1], 1u << sh); else atomicOr(&words[e >> 1], 0x8000u << sh);
    }
    if (!IN_PLACE) asm volatile("cp.async.wait_group %0;" :: "n"(AL_BUFS - 2) : "memory");
    __syncthreads();                                                 // the counts, the logits; and the buffer before this one is free
    fetch();
    if (++buf == AL_BUFS) buf = 0;
    const int last_word = (A.V - 1) >> 5;
    const bool bytes = mrow != nullptr && rv.shift == 0;             // the mask's bytes: on their way while the touched columns are worked on
    uint32_t mbyte[AL_STAGE_BYTES / 16 / AL_NT];
    if (!IN_PLACE) {
#pragma unroll
      for (int j = 0; j < AL_STAGE_BYTES / 16 / AL_NT; j++) {
        const int v = v0 + j * AL_NT + tid;
        mbyte[j] = (bytes && v < v1) ? __ldg(reinterpret_cast<const unsigned char*>(mrow) + (v * VEC >> 3)) : 0u;
      }
    }
    // ---- the biases: the last one for a column counts. A biased column is finished here, its penalties included, and its count
    // taken away.
    auto biased = [&](int t, float value) {
      const int e = t - c0, sh = (e & 1) * 16;
      const uint32_t h = l1 > l0 ? (atomicAnd(&words[e >> 1], ~(0xffffu << sh)) >> sh) & 0xffffu : 0u;
      if (IN_PLACE && !allowed(t)) return;
      const float x = Elem<T>::to_float(IN_PLACE ? xrow[t] : data[e]);
      put(IN_PLACE ? orow + t : data + e, __fadd_rn(h != 0u ? penalised(x, h) : x, value));
    };
    if (off1 - off0 > AL_NT) {                                       // from the last entry to the first, AL_NT at a time
      for (int i = tid; i < (cols + 31) / 32; i += AL_NT) s_done[i] = 0u;
      for (int top = off1; top > off0; top -= AL_NT) {
        const int i = top - 1 - tid;
        const int t = (i >= off0) ? __ldg(A.bias_ids + i) : -1;
        const bool mine = t >= lo && t < hi;
        s_ids[tid] = mine ? t : -1;
        if (!__syncthreads_or(mine)) continue;
        bool last = mine && ((s_done[(t - c0) >> 5] >> ((t - c0) & 31)) & 1u) == 0u;
        if (last) for (int j = 0; j < tid; j++) if (s_ids[j] == t) { last = false; break; }
        __syncthreads();
        if (last) {
          atomicOr(&s_done[(t - c0) >> 5], 1u << ((t - c0) & 31));
          biased(t, __ldg(A.bias_values + i));
        }
        __syncthreads();
      }
    } else if (off1 > off0) {
      if (b_id >= lo && b_id < hi) biased(b_id, b_value);
      __syncthreads();                                               // ahead of whoever looks for counts
    }
    // ---- the penalties
    for (int i = l0 + tid; i < l1; i += AL_NT) {
      const uint32_t e = s_tok[i] & 0x7fffu, sh = (e & 1u) * 16u;
      const uint32_t h = (atomicAnd(&words[e >> 1], ~(0xffffu << sh)) >> sh) & 0xffffu;
      const int t = c0 + static_cast<int>(e);
      if (h == 0u || (IN_PLACE && !allowed(t))) continue;
      put(IN_PLACE ? orow + t : data + e, penalised(Elem<T>::to_float(IN_PLACE ? xrow[t] : data[e]), h));
    }
    __syncthreads();                                                 // the range's logits, and the counts at zero again
    // ---- the range, out of place; in place what the mask takes away
    bin++;
    if (++part == A.nchunk) { part = 0; row++; bin = AL_BINS; }      // (the next round's)
    if (!live || (IN_PLACE && mrow == nullptr)) continue;
    const bool vec_ok = IN_PLACE || ((reinterpret_cast<uintptr_t>(orow) - static_cast<uintptr_t>(rv.shift) * sizeof(T)) & 15u) == 0;
    if (IN_PLACE) {
      al_mask_in_place<T, AL_NT>(orow, rv, mrow, v0, v1, tid);
    } else {
#pragma unroll
      for (int j = 0; j < AL_STAGE_BYTES / 16 / AL_NT; j++) {
        const int v = v0 + j * AL_NT + tid, i0 = v * VEC - rv.shift;
        if (v >= v1) break;
        const uint32_t bits = bytes ? (mbyte[j] >> (i0 & 7)) & ALL : al_mask_bits<VEC>(mrow, i0, last_word, false);
        al_store<T, false>(orow, vec_ok, A.V, i0, reinterpret_cast<const uint4*>(data)[v - v0], bits);
      }
    }
  }
}

}  // namespace gs
