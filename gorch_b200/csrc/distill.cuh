// Distillation from a teacher's top logits over [B, V] rows of a student's logits x (the reference trains on hard targets alone,
// loss.go:55-141; this stands beside its cross-entropy, and TopK, index_ops.go:153-190, makes the teacher's part).
// A row's teacher is k entries (token i, logit t_i); those with a token outside [0, V) or a logit of -Inf are none.
//   p = softmax(t / T) over the entries, q = softmax(x / T) over the vocabulary
//   loss = T^2 sum_i p_i (log p_i - log q_i)
//        = T sum_i p_i ((t_i - tM) - (x_i - M)) - T^2 log tS + T^2 log S,   M = max x, S = sum_j exp((x_j - M) / T), tM and tS the same of t
//   d loss / d x_j = T (q_j - sum of the p_i with i's token = j)
// A row without entries has loss 0 and gradient 0, and its logits are not read. A token listed twice counts twice.
// The forward pass leaves (M, S, tM, tS) for the backward pass, and not log S: exp((x - M) / T) / S is as exact as its f32 parts,
// where a rounded M / T + log S would put 1e-6 of relative error on every q.
//
// Bound: memory. Forward reads x once, backward reads x and writes the f32 gradient once.
#pragma once

#include <cooperative_groups.h>

#include <cstdint>

#include "row_softmax.cuh"

namespace gs {

constexpr int DF_NT = 512;
constexpr int DF_U = 8;                       // 16-byte loads of a thread that are on their way together
constexpr int DF_MAX_C = 8;                   // CTAs per row
constexpr int DB_NT = 256;
constexpr int DB_U = 4;                       // vectors of a thread, all of them on their way at once
constexpr int DB_LIST = 256;                  // a CTA's entries that are kept in shared memory
constexpr float DS_MIN_T = 1e-6f, DS_MAX_T = 1e6f;

// exp(x / T) = 2^(x log2(e) / T): log2(e) / T to f32 and what that leaves out, and where exp(x / T) is 0 in f32.
struct DsScale { float hi, lo, floor; };
inline DsScale ds_scale(float T) {
  const double c = 1.4426950408889634 / static_cast<double>(T);
  DsScale s;
  s.hi = static_cast<float>(c);
  s.lo = static_cast<float>(c - static_cast<double>(s.hi));
  s.floor = -200.0f * T;
  return s;
}

struct DistillArgs {
  const void* x;              // [B, row_stride] f32 or bf16
  int64_t row_stride;
  int32_t V, k;
  int64_t B;
  const int32_t* ids;         // [B, t_stride]
  const float* teacher;       // [B, t_stride]
  int64_t t_stride;
  float T;
  DsScale sc;
  float* row_loss;            // forward: [B]
  float* stats;               // [B][4] (M, S, tM, tS): forward writes, backward reads; tS 0: a row without entries
  const float* row_grads;     // backward: [B] or null: 1
  float scale;
  int32_t accumulate;
  float* dx;                  // [B, dx_stride]
  int64_t dx_stride;
  int32_t nchunk;             // backward: CTAs per row
};

// exp(d / T) of two d <= 0: as rs_exp2, with the temperature in the constants. (Below the floor the result is 0 all the same, and an
// Inf would turn into Inf - Inf.)
__device__ __forceinline__ rs_f2 ds_exp2(float d0, float d1, const DsScale& s) {
  constexpr float LN2 = 0.693147182464599609375f;
  const rs_f2 D = rs_pk(rs_maxnan(d0, s.floor), rs_maxnan(d1, s.floor));
  const rs_f2 NT = rs_mul2(D, rs_pk(-s.hi, -s.hi));
  rs_f2 R = rs_fma2(D, rs_pk(s.hi, s.hi), NT);
  R = rs_fma2(D, rs_pk(s.lo, s.lo), R);
  float n0, n1;
  rs_upk(NT, n0, n1);
  const rs_f2 P = rs_pk(rs_ex2(-n0), rs_ex2(-n1));
  return rs_fma2(P, rs_mul2(R, rs_pk(LN2, LN2)), P);
}

__device__ __forceinline__ bool ds_entry(int id, float t, int V) { return id >= 0 && id < V && !(t == -INFINITY); }

// A cluster of C CTAs takes a row, each a slice of it. Every thread keeps a running maximum m and the sum of exp((x - m) / T) over its
// own elements, rescaled when m grows; the terms' precision is that of rs_max_sum (row_softmax.cuh). The first CTA adds up
// the teacher's side while its first logits are on their way.
template <typename T>
__global__ void __launch_bounds__(DF_NT, 2) distill_fwd_kernel(const __grid_constant__ DistillArgs A) {
  namespace cg = cooperative_groups;
  constexpr int VEC = Elem<T>::VEC, NW = DF_NT / 32, U = DF_U;
  __shared__ bu::Scratch sc;
  __shared__ RsHalf xch[DF_MAX_C];
  const int tid = threadIdx.x;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int64_t row = blockIdx.x / C;
  pdl_launch();                                                // the mean's kernel, which waits for the losses
  pdl_wait();
  RowView<T> rv;
  const T* xrow = static_cast<const T*>(A.x) + row * A.row_stride;
  rv.init(xrow, A.V);
  const int per = static_cast<int>(rr_per(rv.nvec, C));
  const int v0 = min(rank * per, rv.nvec), v1 = min(v0 + per, rv.nvec);
  const int32_t* ids = A.ids + row * A.t_stride;
  const float* tea = A.teacher + row * A.t_stride;
  float tm = -INFINITY;
  bool tnan = false, some = false;
  for (int i = tid; i < A.k; i += DF_NT) {
    const float t = __ldg(tea + i);
    if (!ds_entry(__ldg(ids + i), t, A.V)) continue;
    some = true;
    tnan |= t != t;
    tm = fmaxf(tm, t);
  }
  if (!__syncthreads_or(some)) {                               // (every CTA of the cluster comes to the same)
    if (rank == 0 && tid == 0) {
      A.row_loss[row] = 0.0f;
      for (int i = 0; i < 4; i++) A.stats[4 * row + i] = 0.0f;
    }
    return;
  }
  uint4 raw[U];
  auto load = [&](int v) {
#pragma unroll
    for (int u = 0; u < U; u++) if (v + u * DF_NT < v1) raw[u] = __ldg(rv.vbase + v + u * DF_NT);
  };
  load(v0 + tid);
  if (C > 1) cluster.barrier_arrive();
  double ts = 0.0, at = 0.0, ax = 0.0;                         // sums of exp((t - tM) / T), and of it times t - tM and x
  if (rank == 0) {
    tm = okey_to_float(static_cast<uint32_t>(bu::max_u64<NW>(static_cast<unsigned long long>(okey(tm)), sc, tid)));
    if (tnan) ts = __longlong_as_double(0x7ff8000000000000ll);
    for (int i = tid; i < A.k; i += DF_NT) {
      const float t = __ldg(tea + i);
      const int id = __ldg(ids + i);
      if (!ds_entry(id, t, A.V)) continue;
      const float d = t - tm;                                  // (t = tM = Inf: NaN, and so is the row)
      const double e = static_cast<double>(expf(__fdiv_rn(d, A.T)));
      ts += e;
      if (e != 0.0) { at += e * static_cast<double>(d); ax += e * static_cast<double>(Elem<T>::to_float(xrow[id])); }
    }
    bu::sum_d3<NW>(ts, at, ax, sc, tid);
  }
  float m = -INFINITY;
  rs_f2 s2 = rs_pk(0.0f, 0.0f);
  const float c = A.sc.hi;
  for (int va = v0 + tid; va < v1; va += U * DF_NT) {
    float bm = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int v = va + u * DF_NT;
      if (v >= v1) { raw[u] = make_uint4(0u, 0u, 0u, 0u); continue; }
      if (v == 0 || v >= rv.nvec - 1) raw[u] = mask_edges(rv, v, raw[u]);
      bm = fmaxf(bm, vec_max<T>(raw[u]));
    }
    if (bm > m) {
      const float f = expf(__fdiv_rn(m - bm, A.T));            // (m = -Inf: 0)
      s2 = rs_mul2(s2, rs_pk(f, f));
      m = bm;
    }
    const float mm = (m > -INFINITY) ? m : 0.0f;               // (only -Inf and NaN so far: exp(-Inf) = 0, and a NaN shows in the sum)
    const rs_f2 NM = rs_pk(-mm, -mm), L = rs_pk(c, c);
#pragma unroll
    for (int u = 0; u < U; u++) {
      if (va + u * DF_NT >= v1) break;
      float x[VEC];
      Elem<T>::unpack(raw[u], x);
#pragma unroll
      for (int q = 0; q < VEC; q += 2) {
        float t0, t1;
        rs_upk(rs_mul2(rs_add2(rs_pk(x[q], x[q + 1]), NM), L), t0, t1);
        s2 = rs_add2(s2, rs_pk(rs_ex2(t0), rs_ex2(t1)));
      }
    }
    load(va + U * DF_NT);
  }
  float M = okey_to_float(static_cast<uint32_t>(bu::max_u64<NW>(static_cast<unsigned long long>(okey(m)), sc, tid)));
  float sa, sb;
  rs_upk(s2, sa, sb);
  const float s = sa + sb;
  double S = bu::sum_d<NW>((m > -INFINITY || s != s) ? static_cast<double>(s) * static_cast<double>(expf(__fdiv_rn((m > -INFINITY ? m : M) - M, A.T))) : 0.0, sc, tid);
  if (C > 1) {
    cluster.barrier_wait();
    if (tid == 0) { RsHalf* p = cluster.map_shared_rank(&xch[rank], 0); p->m = M; p->s = S; }
    cluster.sync();                                            // the last remote access
    if (rank != 0) return;
    float Mt = -INFINITY;
    for (int r = 0; r < C; r++) Mt = fmaxf(Mt, xch[r].m);
    double St = 0.0;
    for (int r = 0; r < C; r++) {
      const double sr = xch[r].s;
      if (xch[r].m > -INFINITY || sr != sr) St += sr * static_cast<double>(expf(__fdiv_rn((xch[r].m > -INFINITY ? xch[r].m : Mt) - Mt, A.T)));
    }
    M = Mt;
    S = St;
  }
  if (rank == 0 && tid == 0) {
    if (!(M > -INFINITY)) S = __longlong_as_double(0x7ff8000000000000ll);   // a row of -Inf only
    const double Td = static_cast<double>(A.T);
    A.row_loss[row] = static_cast<float>(Td * (at / ts - (ax / ts - static_cast<double>(M))) + Td * Td * (log(S) - log(ts)));
    A.stats[4 * row] = M;
    A.stats[4 * row + 1] = static_cast<float>(S);
    A.stats[4 * row + 2] = tm;
    A.stats[4 * row + 3] = static_cast<float>(ts);
  }
}

// A CTA takes DB_NT x DB_U vectors of a row. The teacher's entries that fall among them are few: a bit per column says
// whether a column has one, and such a column looks through the list of the CTA's entries.
template <typename T>
__global__ void __launch_bounds__(DB_NT) distill_bwd_kernel(const __grid_constant__ DistillArgs A) {
  constexpr int VEC = Elem<T>::VEC, U = DB_U, COLS = DB_NT * U * VEC;
  __shared__ uint32_t s_bits[COLS / 32];
  __shared__ int s_at[DB_LIST], s_id[DB_LIST];                 // number of the entry, its token
  __shared__ int s_n;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / static_cast<unsigned>(A.nchunk);
  const int part = static_cast<int>(blockIdx.x - static_cast<unsigned>(row) * static_cast<unsigned>(A.nchunk));
  for (int i = tid; i < COLS / 32; i += DB_NT) s_bits[i] = 0u;
  if (tid == 0) s_n = 0;
  pdl_launch();
  pdl_wait();                                                  // the forward pass
  const T* xrow = static_cast<const T*>(A.x) + row * A.row_stride;
  float* drow = A.dx + row * A.dx_stride;
  RowView<T> rv;
  rv.init(xrow, A.V);
  const int v0 = part * (DB_NT * U);
  if (v0 >= rv.nvec) return;
  const float M = A.stats[4 * row], S = A.stats[4 * row + 1], tM = A.stats[4 * row + 2], tS = A.stats[4 * row + 3];
  const float g = A.row_grads ? A.row_grads[row] : 1.0f;
  const bool none = tS == 0.0f;
  if (none && A.accumulate) return;
  uint4 raw[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int v = v0 + u * DB_NT + tid;
    raw[u] = (!none && v < rv.nvec) ? *(rv.vbase + v) : make_uint4(0u, 0u, 0u, 0u);   // (dx may lie where x lies)
  }
  const int c0 = v0 * VEC - rv.shift;                          // column of the first element: below 0 in a row's first vector
  const int lo = max(c0, 0), hi = min(c0 + COLS, A.V);
  const int32_t* ids = A.ids + row * A.t_stride;
  const float* tea = A.teacher + row * A.t_stride;
  __syncthreads();
  if (!none) {
    for (int i = tid; i < A.k; i += DB_NT) {
      const int id = __ldg(ids + i);
      if (id < lo || id >= hi || __ldg(tea + i) == -INFINITY) continue;
      atomicOr(&s_bits[(id - c0) >> 5], 1u << ((id - c0) & 31));
      const int at = atomicAdd(&s_n, 1);
      if (at < DB_LIST) { s_at[at] = i; s_id[at] = id; }
    }
  }
  __syncthreads();
  const int n = s_n;
  const float coef = none ? 0.0f : static_cast<float>(static_cast<double>(A.scale) * static_cast<double>(g) * static_cast<double>(A.T));
  const float inv = none ? 0.0f : 1.0f / S;
  // the teacher's probability of a column: its entries' in the order of the list they came in
  auto teacher = [&](int col) -> float {
    float p = 0.0f;
    if (n <= DB_LIST) {
      for (int after = -1;;) {
        int next = A.k;
        for (int j = 0; j < n; j++) if (s_id[j] == col && s_at[j] > after) next = min(next, s_at[j]);
        if (next == A.k) return p;
        p += expf(__fdiv_rn(__ldg(tea + next) - tM, A.T)) / tS;
        after = next;
      }
    }
    for (int i = 0; i < A.k; i++) if (__ldg(ids + i) == col && !(__ldg(tea + i) == -INFINITY)) p += expf(__fdiv_rn(__ldg(tea + i) - tM, A.T)) / tS;
    return p;
  };
  const bool vec_ok = ((reinterpret_cast<uintptr_t>(drow) - static_cast<uintptr_t>(rv.shift) * 4u) & 15u) == 0;
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int v = v0 + u * DB_NT + tid, i0 = v * VEC - rv.shift, e0 = (u * DB_NT + tid) * VEC;
    if (v >= rv.nvec) break;
    float x[VEC], y[VEC];
    Elem<T>::unpack(raw[u], x);
#pragma unroll
    for (int c = 0; c < VEC; c += 2) rs_upk(rs_mul2(ds_exp2(x[c] - M, x[c + 1] - M, A.sc), rs_pk(inv, inv)), y[c], y[c + 1]);
    uint32_t bits = (n > 0) ? (s_bits[e0 >> 5] >> (e0 & 31)) & ((1u << VEC) - 1u) : 0u;
    while (bits) {
      const int c = __ffs(bits) - 1;
      bits &= bits - 1u;
      const float p = teacher(i0 + c);
#pragma unroll
      for (int j = 0; j < VEC; j++) if (j == c) y[j] -= p;
    }
#pragma unroll
    for (int c = 0; c < VEC; c++) y[c] = none ? 0.0f : y[c] * coef;
    if (A.accumulate) {
#pragma unroll
      for (int c = 0; c < VEC; c++) if (i0 + c >= 0 && i0 + c < A.V) y[c] += drow[i0 + c];
    }
    rs_store<float, VEC>(drow, vec_ok, A.V, i0, y);
  }
}

}  // namespace gs
