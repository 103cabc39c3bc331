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
// Bound: memory. Out of place a row is read and written once, in place only the vectors that change are
// touched, and a vector of which the mask leaves nothing is written without being read.
// A CTA takes a chunk of a row (AL_NT threads x U vectors of 16 bytes). The touched tokens are few and anywhere, so the
// CTA keeps one word per column of its chunk in shared memory: how often the column's token was generated, a
// bit for "held", a bit for "biased". All threads walk the row's history and count what falls into the chunk
// with shared-memory atomics (integers: the order does not matter), while the chunk's logits are on their way to registers.
// The entries of the bias map that fall into the chunk are collected beside them; a biased column, which is rare,
// looks its entry up there.
#pragma once

#include <cstdint>

#include "row_softmax.cuh"   // bf16_bits_rne

namespace gs {

constexpr int AL_NT = 256;
constexpr int AL_BIAS_CAP = 512;              // entries of the bias map in one chunk that are kept in shared memory
constexpr uint32_t AL_HELD = 0x80000000u, AL_BIASED = 0x40000000u, AL_COUNT = 0x3fffffffu;
constexpr int AL_U = 8;                       // 16-byte vectors per thread

struct AdjustArgs {
  const void* x;                  // [B, row_stride]
  int64_t row_stride;
  void* out;                      // [B, out_stride]; x itself in place
  int64_t out_stride;
  int32_t V, nchunk;
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
};

// Shared memory for a chunk's words.
inline int adjust_words_bytes(bool f32) { return AL_NT * AL_U * (f32 ? 4 : 8) * 4; }

struct AlBias { int32_t at, id; float value; };     // entry number in the map, token, bias

// A vector of which the mask's bits keep some elements: -Inf for the others.
template <typename T>
__device__ __forceinline__ uint4 al_masked(const uint4& r, uint32_t bits) {
  uint4 o;
  if (sizeof(T) == 4) {
    o.x = (bits & 1u) ? r.x : 0xff800000u;
    o.y = (bits & 2u) ? r.y : 0xff800000u;
    o.z = (bits & 4u) ? r.z : 0xff800000u;
    o.w = (bits & 8u) ? r.w : 0xff800000u;
  } else {
    auto two = [](uint32_t w, uint32_t b) {
      const uint32_t lo = (b & 1u) ? (w & 0xffffu) : 0xff80u, hi = (b & 2u) ? (w & 0xffff0000u) : 0xff800000u;
      return lo | hi;
    };
    o.x = two(r.x, bits); o.y = two(r.y, bits >> 2); o.z = two(r.z, bits >> 4); o.w = two(r.w, bits >> 6);
  }
  return o;
}

// What a row's rules make of a logit that they touch; w is the column's word. (Rare, and called from every place of an
// unrolled loop: not inlined.)
struct AlRow { float rep, pres, freq; int off0, off1, nbias; };
__device__ __noinline__ float al_touched(float x, uint32_t w, int col, const AlRow& r, const AdjustArgs& A, const AlBias* s_bias) {
  float y = x;
  if (w & ~AL_BIASED) {
    y = (y > 0.0f) ? __fdiv_rn(y, r.rep) : __fmul_rn(y, r.rep);
    const uint32_t c = w & AL_COUNT;
    if (c != 0u) y = __fsub_rn(__fsub_rn(y, __fmul_rn(r.freq, static_cast<float>(c))), r.pres);
  }
  if (w & AL_BIASED) {                                               // the last entry that names the column
    int at = -1;
    float value = 0.0f;
    if (r.nbias <= AL_BIAS_CAP) {
      for (int i = 0; i < r.nbias; i++) if (s_bias[i].id == col && s_bias[i].at > at) { at = s_bias[i].at; value = s_bias[i].value; }
    } else {
      for (int i = r.off1 - 1; i >= r.off0; i--) if (A.bias_ids[i] == col) { value = A.bias_values[i]; break; }
    }
    y = __fadd_rn(y, value);
  }
  return y;
}

// WORDS: the call has penalties or biases.
template <typename T, bool IN_PLACE, bool WORDS>
__global__ void __launch_bounds__(AL_NT) adjust_logits_kernel(const __grid_constant__ AdjustArgs A) {
  constexpr int VEC = Elem<T>::VEC, U = AL_U, COLS = AL_NT * U * VEC;
  constexpr uint32_t ALL = (1u << VEC) - 1u;
  extern __shared__ __align__(16) uint32_t al_words[];               // [COLS] when WORDS
  __shared__ AlBias s_bias[WORDS ? AL_BIAS_CAP : 1];
  __shared__ int s_nbias;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / static_cast<unsigned>(A.nchunk);
  const int chunk = static_cast<int>(blockIdx.x - static_cast<unsigned>(row) * static_cast<unsigned>(A.nchunk));
  if (WORDS) {
    uint4* w4 = reinterpret_cast<uint4*>(al_words);
    for (int i = tid; i < COLS / 4; i += AL_NT) w4[i] = make_uint4(0u, 0u, 0u, 0u);
    if (tid == 0) s_nbias = 0;
  }
  pdl_launch();
  pdl_wait();                                                        // whatever fills the inputs, or still reads the output
  if (A.row_done != nullptr && A.row_done[row] != 0) return;
  RowView<T> rv;
  rv.init(static_cast<const T*>(A.x) + row * A.row_stride, A.V);
  const int v0 = chunk * (AL_NT * U);
  if (v0 >= rv.nvec) return;                                         // (rows differ by a vector, depending on where they start)
  const int c0 = v0 * VEC - rv.shift;                                // column of the chunk's first element (below 0 in the first vector)
  uint4 raw[U];
  if (!IN_PLACE) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int v = v0 + u * AL_NT + tid;
      raw[u] = (v < rv.nvec) ? __ldg(rv.vbase + v) : make_uint4(0u, 0u, 0u, 0u);
    }
  }
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  int off0 = 0, off1 = 0;
  if (WORDS) {
    __syncthreads();
    if (A.penalties != nullptr) {
      rep = A.penalties[4 * row]; pres = A.penalties[4 * row + 1]; freq = A.penalties[4 * row + 2];
      if (rep != 1.0f || pres != 0.0f || freq != 0.0f) {             // (a row without penalties does not read its history)
        const int len = static_cast<int>(min(static_cast<int64_t>(max(A.lengths[row], 0)), A.history_stride));
        int prompt = 0;
        if (A.n_new != nullptr) prompt = len - A.n_new[row];
        else if (A.prompt_lengths != nullptr) prompt = A.prompt_lengths[row];
        const int32_t* h = A.history + row * A.history_stride;
#pragma unroll 4
        for (int i = tid; i < len; i += AL_NT) {
          const int t = h[i], at = t - c0;
          if (t >= 0 && t < A.V && at >= 0 && at < COLS) {
            if (i < prompt) atomicOr(&al_words[at], AL_HELD);
            else atomicAdd(&al_words[at], 1u);
          }
        }
      }
    }
    if (A.bias_offsets != nullptr) {
      off0 = min(max(A.bias_offsets[row], 0), A.n_bias);
      off1 = min(max(A.bias_offsets[row + 1], off0), A.n_bias);
      for (int i = off0 + tid; i < off1; i += AL_NT) {
        const int t = A.bias_ids[i], at = t - c0;
        if (t >= 0 && t < A.V && at >= 0 && at < COLS) {
          atomicOr(&al_words[at], AL_BIASED);
          const int slot = atomicAdd(&s_nbias, 1);
          if (slot < AL_BIAS_CAP) s_bias[slot] = AlBias{i, t, A.bias_values[i]};
        }
      }
    }
    __syncthreads();
  }
  const uint32_t* mrow = nullptr;
  if (A.mask != nullptr) {
    const int64_t m = A.mask_rows ? A.mask_rows[row] : row;
    if (m >= 0 && m < A.n_masks) mrow = A.mask + m * A.mask_stride;
  }
  const int last_word = (A.V - 1) >> 5;
  // the mask's bits for the VEC columns from i0 on (i0 may begin below 0; columns outside the row: any)
  auto mask_bits = [&](int i0) -> uint32_t {
    if (i0 < 0) return (__ldg(mrow) << -i0) & ALL;
    const int w = i0 >> 5;
    return __funnelshift_r(__ldg(mrow + w), __ldg(mrow + min(w + 1, last_word)), i0 & 31) & ALL;
  };
  const AlRow rr{rep, pres, freq, off0, off1, WORDS ? s_nbias : 0};
  T* orow = static_cast<T*>(A.out) + row * A.out_stride;
  const bool vec_ok = IN_PLACE || ((reinterpret_cast<uintptr_t>(orow) - static_cast<uintptr_t>(rv.shift) * sizeof(T)) & 15u) == 0;
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int v = v0 + u * AL_NT + tid;
    if (v >= rv.nvec) break;
    const int i0 = v * VEC - rv.shift;
    const uint32_t bits = mrow ? mask_bits(i0) : ALL;
    uint4 w[VEC / 4];
    uint32_t any = 0u;
    if (WORDS) {
#pragma unroll
      for (int q = 0; q < VEC / 4; q++) {
        w[q] = reinterpret_cast<const uint4*>(al_words)[(u * AL_NT + tid) * (VEC / 4) + q];
        any |= w[q].x | w[q].y | w[q].z | w[q].w;
      }
    }
    if (IN_PLACE) {
      if (any == 0u && bits == ALL) continue;
      if (bits == 0u) raw[u] = make_uint4(0u, 0u, 0u, 0u);
      else raw[u] = rv.vbase[v];
    }
    uint4 o = al_masked<T>(raw[u], bits);
    if (WORDS && any != 0u) {
      const uint32_t ws[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[VEC / 4 - 1].x, w[VEC / 4 - 1].y, w[VEC / 4 - 1].z, w[VEC / 4 - 1].w};
      float x[VEC];
      Elem<T>::unpack(raw[u], x);
      uint32_t* ow = &o.x;
#pragma unroll
      for (int c = 0; c < VEC; c++) {
        if (ws[c] == 0u || !((bits >> c) & 1u)) continue;
        const float y = al_touched(x[c], ws[c], i0 + c, rr, A, s_bias);
        if (sizeof(T) == 4) ow[c] = __float_as_uint(y);
        else if (c & 1) ow[c >> 1] = (ow[c >> 1] & 0xffffu) | (bf16_bits_rne(y) << 16);
        else ow[c >> 1] = (ow[c >> 1] & 0xffff0000u) | bf16_bits_rne(y);
      }
    }
    if (vec_ok && i0 >= 0 && i0 + VEC <= A.V) {
      *reinterpret_cast<uint4*>(orow + i0) = o;
    } else {
      const uint32_t* ow = &o.x;
#pragma unroll
      for (int c = 0; c < VEC; c++) {
        const int i = i0 + c;
        if (i < 0 || i >= A.V) continue;
        if (sizeof(T) == 4) reinterpret_cast<uint32_t*>(orow)[i] = ow[c];
        else reinterpret_cast<uint16_t*>(orow)[i] = static_cast<uint16_t>(ow[c >> 1] >> (16 * (c & 1)));
      }
    }
  }
}

}  // namespace gs
