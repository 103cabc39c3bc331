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
// Bound: memory. Forward reads x once (1,500 x 168,320 f32, a twentieth of the rows without entries: 192 us, 5.0 TB/s), backward reads x
// and writes the f32 gradient once (329 us, 6.0 TB/s).
#pragma once

#include <cooperative_groups.h>

#include <cstdint>

#include "row_softmax.cuh"

namespace gs {

constexpr int DF_NT = 256;
constexpr int DF_PER_SM = 4;                  // CTAs of 64 registers a thread
constexpr int DF_U = 8;                       // 16-byte loads of a thread that are on their way together (us, loads x CTAs per SM: 4 x 6: 220, 6 x 5: 193,
                                              // 8 x 4: 192, 8 x 3: 245)
constexpr int DF_MAX_C = 8;                   // CTAs per row
constexpr int DB_NT = 256;
constexpr int DB_U = 4;                       // 16-byte vectors of a thread that are on their way together
constexpr int DB_MAX_P = 8;                   // batches of them that a CTA takes at most
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
  int32_t nchunk, batches;    // backward: CTAs per row, batches of vectors each
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
// own elements, rescaled when m grows (the terms' precision is that of rs_max_sum, row_softmax.cuh). In the first CTA the
// threads do the same with the teacher's entries, and for the sums of p times t and x. So a row costs one reduction at its end,
// and its first logits are asked for before anything is known of it but that its first entry is one.
template <typename T>
__global__ void __launch_bounds__(DF_NT, DF_PER_SM) distill_fwd_kernel(const __grid_constant__ DistillArgs A) {
  namespace cg = cooperative_groups;
  constexpr int VEC = Elem<T>::VEC, NW = DF_NT / 32, U = DF_U;
  __shared__ bu::Scratch sc;
  __shared__ double s_sum[4][NW];
  __shared__ RsHalf xch[DF_MAX_C];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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
  if (!ds_entry(__ldg(ids), __ldg(tea), A.V)) {                // perhaps a row without entries
    bool some = false;
    for (int i = tid; i < A.k; i += DF_NT) some |= ds_entry(__ldg(ids + i), __ldg(tea + i), A.V);
    if (!__syncthreads_or(some)) {                             // (every CTA of the cluster comes to the same)
      if (rank == 0 && tid == 0) {
        A.row_loss[row] = 0.0f;
        for (int i = 0; i < 4; i++) A.stats[4 * row + i] = 0.0f;
      }
      return;
    }
  }
  uint4 raw[U];
  auto load = [&](int v) {
#pragma unroll
    for (int u = 0; u < U; u++) if (v + u * DF_NT < v1) raw[u] = __ldg(rv.vbase + v + u * DF_NT);
  };
  load(v0 + tid);
  if (C > 1) cluster.barrier_arrive();
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
  // the teacher's side: sums of e = exp((t - own maximum) / T), of e (t - own maximum) and of e x
  float tm = -INFINITY;
  double ts = 0.0, at = 0.0, ax = 0.0;
  if (rank == 0) {
    for (int i = tid; i < A.k; i += DF_NT) {
      const float t = __ldg(tea + i);
      const int id = __ldg(ids + i);
      if (!ds_entry(id, t, A.V)) continue;
      const double x = static_cast<double>(Elem<T>::to_float(__ldg(xrow + id)));
      if (t > tm) {
        const double d = static_cast<double>(tm) - static_cast<double>(t), f = static_cast<double>(expf(static_cast<float>(d / static_cast<double>(A.T))));
        if (f > 0.0) { at = f * (at + ts * d); ax *= f; } else { at = 0.0; ax = 0.0; }   // (what is 0 in f32 is no term: not 0 times Inf)
        ts = ts * f + 1.0;
        ax += x;
        tm = t;
      } else {
        const float d = t - tm;                                // (NaN or Inf: the row becomes NaN)
        const double e = static_cast<double>(expf(__fdiv_rn(d, A.T)));
        ts += e;
        if (e != 0.0) { at += e * static_cast<double>(d); ax += e * x; }
      }
    }
  }
  // the row's maxima, then its sums
  uint32_t km = okey(m), kt = okey(tm), unused = 0u;
  bu::max_u3<NW>(km, kt, unused, sc, tid);
  float M = okey_to_float(km);
  const float tM = okey_to_float(kt);
  float sa, sb;
  rs_upk(s2, sa, sb);
  const float s = sa + sb;
  double sum = (m > -INFINITY || s != s) ? static_cast<double>(s) * static_cast<double>(expf(__fdiv_rn((m > -INFINITY ? m : M) - M, A.T))) : 0.0;
  sum = warp_sum_d(sum);
  const bool warp_teaches = rank == 0 && warp * 32 < A.k;
  if (warp_teaches) {
    const double d = static_cast<double>(tm) - static_cast<double>(tM);
    const double f = ts == 0.0 ? 0.0 : static_cast<double>(expf(static_cast<float>(d / static_cast<double>(A.T))));
    if (ts == ts) {                                            // (a NaN stays: with nothing else among the thread's entries there is no maximum, and f = 0)
      if (f == 0.0) { ts = 0.0; at = 0.0; ax = 0.0; } else { at = f * (at + ts * d); ax *= f; ts *= f; }
    }
    ts = warp_sum_d(ts); at = warp_sum_d(at); ax = warp_sum_d(ax);
  }
  if (lane == 0) { s_sum[0][warp] = sum; s_sum[1][warp] = warp_teaches ? ts : 0.0; s_sum[2][warp] = warp_teaches ? at : 0.0; s_sum[3][warp] = warp_teaches ? ax : 0.0; }
  __syncthreads();
  double S = 0.0;
  for (int w = 0; w < NW; w++) S += s_sum[0][w];
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
  if (tid == 0) {
    if (!(M > -INFINITY)) S = __longlong_as_double(0x7ff8000000000000ll);   // a row of -Inf only
    ts = at = ax = 0.0;
    for (int w = 0; w < NW; w++) { ts += s_sum[1][w]; at += s_sum[2][w]; ax += s_sum[3][w]; }
    const double Td = static_cast<double>(A.T);
    A.row_loss[row] = static_cast<float>(Td * (at / ts - (ax / ts - static_cast<double>(M))) + Td * Td * (log(S) - log(ts)));
    A.stats[4 * row] = M;
    A.stats[4 * row + 1] = static_cast<float>(S);
    A.stats[4 * row + 2] = tM;
    A.stats[4 * row + 3] = static_cast<float>(ts);
  }
}

// A CTA takes A.batches x DB_NT x DB_U vectors of a row. The teacher's entries that fall among them are few: a bit per column says
// whether a column has one; such columns are left out of the stream and finished behind it, an entry per thread. A column
// whose token is listed more than once (which a bit that is already there shows) is finished by its first entry, with the
// others' probabilities added in the list's order. (With the lookup inside the stream, a call there: 401 us for 1,500 x 168,320 f32.)
template <typename T>
__global__ void __launch_bounds__(DB_NT, 4) distill_bwd_kernel(const __grid_constant__ DistillArgs A) {
  constexpr int VEC = Elem<T>::VEC, U = DB_U, COLS = DB_NT * U * VEC;
  __shared__ uint32_t s_bits[DB_MAX_P * COLS / 32];
  __shared__ int s_any, s_twice;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / static_cast<unsigned>(A.nchunk);
  const int part = static_cast<int>(blockIdx.x - static_cast<unsigned>(row) * static_cast<unsigned>(A.nchunk));
  for (int i = tid; i < A.batches * (COLS / 32); i += DB_NT) s_bits[i] = 0u;
  if (tid == 0) { s_any = 0; s_twice = 0; }
  pdl_launch();
  pdl_wait();                                                  // the forward pass
  const T* xrow = static_cast<const T*>(A.x) + row * A.row_stride;
  float* drow = A.dx + row * A.dx_stride;
  RowView<T> rv;
  rv.init(xrow, A.V);
  const int v0 = part * A.batches * (DB_NT * U), v1 = min(v0 + A.batches * (DB_NT * U), rv.nvec);
  if (v0 >= v1) return;
  const float M = A.stats[4 * row], S = A.stats[4 * row + 1], tM = A.stats[4 * row + 2], tS = A.stats[4 * row + 3];
  const float g = A.row_grads ? A.row_grads[row] : 1.0f;
  const bool none = tS == 0.0f;
  if (none && A.accumulate) return;
  uint4 raw[U];
  auto load = [&](int v) {
#pragma unroll
    for (int u = 0; u < U; u++) raw[u] = (!none && v + u * DB_NT < v1) ? *(rv.vbase + v + u * DB_NT) : make_uint4(0u, 0u, 0u, 0u);   // (dx may lie where x lies)
  };
  load(v0 + tid);
  const int c0 = v0 * VEC - rv.shift;                          // column of the first element: below 0 in a row's first vector
  const int lo = max(c0, 0), hi = min(v1 * VEC - rv.shift, A.V);
  const int32_t* ids = A.ids + row * A.t_stride;
  const float* tea = A.teacher + row * A.t_stride;
  __syncthreads();
  if (!none) {
    for (int i = tid; i < A.k; i += DB_NT) {
      const int id = __ldg(ids + i);
      if (id < lo || id >= hi || __ldg(tea + i) == -INFINITY) continue;
      const uint32_t bit = 1u << ((id - c0) & 31);
      if (atomicOr(&s_bits[(id - c0) >> 5], bit) & bit) s_twice = 1;
      s_any = 1;
    }
  }
  __syncthreads();
  const bool any = s_any != 0, twice = s_twice != 0;
  const float coef = none ? 0.0f : static_cast<float>(static_cast<double>(A.scale) * static_cast<double>(g) * static_cast<double>(A.T));
  const float inv = none ? 0.0f : 1.0f / S;
  const bool vec_ok = ((reinterpret_cast<uintptr_t>(drow) - static_cast<uintptr_t>(rv.shift) * 4u) & 15u) == 0;
  for (int va = v0 + tid; va < v1; va += U * DB_NT) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int v = va + u * DB_NT, i0 = v * VEC - rv.shift, e0 = (v - v0) * VEC;
      if (v >= v1) break;
      float x[VEC], y[VEC];
      Elem<T>::unpack(raw[u], x);
#pragma unroll
      for (int c = 0; c < VEC; c += 2) {
        const rs_f2 q = rs_mul2(ds_exp2(x[c] - M, x[c + 1] - M, A.sc), rs_pk(inv, inv));
        rs_upk(rs_mul2(q, rs_pk(coef, coef)), y[c], y[c + 1]);
      }
      if (none) {
#pragma unroll
        for (int c = 0; c < VEC; c++) y[c] = 0.0f;
      }
      if (A.accumulate) {
        if (vec_ok && i0 >= 0 && i0 + VEC <= A.V) {
#pragma unroll
          for (int c = 0; c < VEC; c += 4) {
            const float4 o = *reinterpret_cast<const float4*>(drow + i0 + c);
            y[c] += o.x; y[c + 1] += o.y; y[c + 2] += o.z; y[c + 3] += o.w;
          }
        } else {
#pragma unroll
          for (int c = 0; c < VEC; c++) if (i0 + c >= 0 && i0 + c < A.V) y[c] += drow[i0 + c];
        }
      }
      const uint32_t bits = any ? (s_bits[e0 >> 5] >> (e0 & 31)) & ((1u << VEC) - 1u) : 0u;
      if (bits == 0u) {
        rs_store<float, VEC>(drow, vec_ok, A.V, i0, y);
      } else {
#pragma unroll
        for (int c = 0; c < VEC; c++) if (!((bits >> c) & 1u) && i0 + c >= 0 && i0 + c < A.V) drow[i0 + c] = y[c];
      }
    }
    load(va + U * DB_NT);
  }
  if (!any) return;
  for (int i = tid; i < A.k; i += DB_NT) {
    const int id = __ldg(ids + i);
    if (id < lo || id >= hi) continue;
    const float t = __ldg(tea + i);
    if (t == -INFINITY) continue;
    float p = expf(__fdiv_rn(t - tM, A.T)) / tS;
    if (twice) {
      bool first = true;
      for (int j = 0; j < A.k && first; j++) {
        if (j == i || __ldg(ids + j) != id || __ldg(tea + j) == -INFINITY) continue;
        if (j < i) first = false;
        else p += expf(__fdiv_rn(__ldg(tea + j) - tM, A.T)) / tS;
      }
      if (!first) continue;
    }
    float q, unused;
    const float d = Elem<T>::to_float(xrow[id]) - M;           // (left alone by the stream, where dx lies over x)
    rs_upk(rs_mul2(ds_exp2(d, d, A.sc), rs_pk(inv, inv)), q, unused);
    const float y = (q - p) * coef;
    drow[id] = A.accumulate ? y + drow[id] : y;
  }
}

}  // namespace gs
