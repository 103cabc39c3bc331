// LM-head projection with the sampling step's first pass in its epilogue.
//
// logits[b, v] = sum_k x[b, k] * w[v, k]: the last matmul of a decode step, MatMulTransB(last, Embed.Weight)
// in model/qwen/qwen.go:80-85 (nn/gpt.go:119-120 for GPT-2; nn/extembed.go:152-195 is its CPU loop), with
// x [B, K] and w [V, K] in bf16 and f32 accumulation. It is the one dense contraction next to the
// sampling path, and it produces the [B, V] logits that the sampling kernels otherwise read back from
// HBM: here the rows of a batch tile stay in tensor memory until the epilogue has taken what sampling
// needs from them.
//
// A pair of CTAs (a cluster of two, tcgen05 cta_group::2) works on one tile of 256 vocabulary rows x up
// to 256 batch rows; the vocabulary is the M side, so that a TMEM lane is a vocabulary column of the
// output and a warp writes 32 neighbouring logits of a batch row at a time. CTA r of the pair holds
// vocabulary rows 128 r .. of the tile, half of the batch rows, and the accumulator of its own vocabulary
// rows. Per item K is walked in chunks of 128:
//   warp 0      producer (both CTAs): TMA loads (w: 128 x 64, x: N / 2 x 64, 128-byte swizzle; two of each per
//               chunk, so that 256 neighbouring bytes of a row are asked for together: 32 x 1,024 x 151,936 in 51 us,
//               6.1 TB/s of weights; 61 us and 5.1 with one) into a ring of shared-memory stages; the bytes of
//               both CTAs complete on the leader's mbarrier
//   warp 1      issuer (leader): one elected thread issues tcgen05.mma (M = 256, N, K = 16) into one of two
//               accumulators of 256 TMEM columns; tcgen05.commit frees the stage / publishes the
//               accumulator in both CTAs
//   warps 2-9   epilogue (both CTAs): thread = vocabulary row (a TMEM lane), the batch rows' logits by
//               tcgen05.ld; either stores them, or (fused sampling) appends those at or above their batch
//               row's threshold to that row's candidate list
//
// Bound: at 512 rows the L2-to-SM traffic, the tensor pipe and HBM ask for about the same time each. A
// tile of 128 x 128 per CTA moves 2.5 GB from L2 for 512 x 1024 x 151,936 (4.1 ms of it per PFLOP; 10 TB/s
// measured: 250 us); a pair's 256 x 256 moves 1.25 GB. At 64 rows it is HBM, the weights' one read.
// Items are dealt out round by round over the pairs; what the last round would leave to a few pairs is cut
// into 32-row items for all of them.
// Every CTA fetches its own tiles (plain TMA loads), and every tensor map covers this GPU's own memory.
//
// Every wait on an mbarrier is bounded: a wait that runs out sets an abort flag that the CTA's other roles
// see in their own waits (the other CTA's run out by themselves), the kernel reports LMH_ERR_TIMEOUT in its
// status word, frees its tensor memory and returns.
#pragma once

#include <cuda.h>

#include "row_softmax.cuh"     // bf16_bits_rne
#include "sample_batch.cuh"

namespace gs {

constexpr int LMH_TILE_V = 256;          // vocabulary rows of a tile (UMMA M over the pair); 128 per CTA
constexpr int LMH_CTA_V = 128;
constexpr int LMH_MAX_N = 256;           // batch rows of an item (UMMA N)
constexpr int LMH_BK = 64;               // K of one TMA box: 64 bf16 = one 128-byte swizzle row
constexpr int LMH_SUB = 2;               // boxes of either operand per stage
constexpr int LMH_EPI = 8;               // epilogue warps: two for each quarter of the TMEM lanes
constexpr int LMH_NT = 64 + 32 * LMH_EPI;   // warp 0 producer, warp 1 issuer, then the epilogue
constexpr int LMH_MAX_STAGES = 12;
constexpr int LMH_RING_BYTES = 208 * 1024;
constexpr int LMH_W_BYTES = LMH_CTA_V * LMH_BK * 2;                 // a box of w: 16 KB
constexpr int LMH_DYN_BYTES = LMH_RING_BYTES + 1024;                // + room to align the swizzled tiles to 1024 bytes
constexpr int LMH_TMEM_COLS = 512;       // two accumulators of 256 f32 columns
constexpr uint32_t LMH_WAIT_LIMIT = 4000000u;

constexpr uint32_t LMH_ERR_TIMEOUT = 1u;

// tcgen05 instruction descriptor (kind::f16): D = F32 (bits 4-5 = 1), A = B = BF16 (bits 7-9, 10-12 = 1),
// both K-major (bits 15, 16 = 0), N / 8 at bits 17-22, M / 16 at bits 24-28.
__host__ __device__ constexpr uint32_t lmh_idesc(int n) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(LMH_TILE_V >> 4) << 24);
}

constexpr int LMH_CAND_CAP = 2048;       // candidates per row (entries of 8 bytes)
struct LmhRow {
  int32_t cnt;             // candidates so far (those beyond LMH_CAND_CAP are not stored)
  int32_t nan;             // 1: a NaN in the row; 2: at index 0
};

struct LmHeadArgs {
  CUtensorMap map_x;       // x [B, K] bf16, box 64 x box_n, 128-byte swizzle
  CUtensorMap map_w;       // w [V, K] bf16, box 64 x cta_v, 128-byte swizzle
  int32_t B, V, K;
  int32_t box_n;           // batch rows that one TMA load of x brings: half of the largest item
  int32_t item_n;          // batch rows of a full item, a multiple of 32
  int32_t stages;          // of the ring
  int32_t cta_v;           // vocabulary rows of a tile that each CTA takes, at most LMH_CTA_V
  int32_t tile0, tile_step, ntile;   // vocabulary tiles (of 2 cta_v rows) tile0 + i * tile_step, i < ntile
  float* out_logits;       // [B, ld_out] f32, or null
  int64_t ld_out;
  int32_t compact;         // 1: tile i goes to columns [i * 2 cta_v, ...) of out_logits (the sample of tiles)
  // fused sampling (all null when unused)
  const float* thr;        // [B] candidate threshold per row (raw logit units)
  uint2* cand;             // [B][LMH_CAND_CAP] (logit bits, index)
  LmhRow* rows;            // [B]
  uint32_t* status;        // [1] LMH_ERR_* bits, in host memory
  int32_t clear_status;    // 1: this launch clears it first
  int32_t chained;         // 1: launched as a dependent of the kernel that fills thr, with x and w there before; 0: of any kernel
};

// ---- low-rank adapters beside the projection -----------------------------------------------------------
// logits[b, v] += h[b] . b[a][v], h[b] = scale[a] * (a[a] x[b]), for the adapter a that row b has (none: no term). For the tensor pipe
// these are further columns of K. The batch rows are taken in the order of their adapters (x is copied in that order, and the
// epilogue writes to the rows' own places), so that in a group of item_n of them an adapter's rows are a run. After K the
// products of an item go on over its runs, in units of LMA_UNIT columns of the rank: the adapter's b [V, rank] on the w side, h
// on the x side, over the multiple of 32 batch rows that holds the run, with zeros in the rows around it. LMA_STAGE units share a
// stage of the ring (32-byte rows, 32-byte swizzle; what a rank leaves of a unit is filled with zeros by the copy). Four warps of
// their own ask for a stage's units, one each, once the producer has found the stage free and announced its bytes (256 rows with 32
// adapters of rank 32 over 1,024 x 151,936: 225 us so, 355 with one thread asking for all, 401 with cp.async in place of TMA,
// all with two parts of h and one sum (see below); now 235 to 245, and the projection alone 95). What bounds it: W and the b's are 121 us at
// the copy rate; a stage's way round the ring, with three
// stages of 64 KB for 256 rows, is about 50 us of the rest, the MMAs 34 (with two parts of h), the loads 32 (six or eight units to a stage did not make it
// faster: 276, 237 for 225). 64 rows with eight adapters of rank 16: 93 us (70 alone); one row: 70 (53 alone).
// So an adapter's b passes once per group, its products cost what its rows cost, rounded up to 32 (with every unit over all
// rows of the item, 256 x 1,024 x 151,936 with 32 adapters of rank 32 took 290 us, though 64 rows with eight of rank 16 took 83),
// and the epilogue's results are complete.
// h goes in as three bf16, eight bits of the f32 value after eight, each multiplied with the same tile of b: nothing of h is lost.
// The tensor pipe cuts its sums off where f32 would round them, which over K = 1,024 puts 1.0e-6 of the logits' size on them, and in
// proportion to K. So they are cut into runs of LMA_SEG products, each with an accumulator of its own (the last goes on over
// the adapters), and the epilogue adds those in registers, rounding to nearest. Errors as a share of the logits' size, root mean squares
// against 64 bits, 64 rows, rank 16: K = 1,024: 4.9e-7 (one sum: 1.0e-6; an f32 product: 2.5e-7), K = 4,096: 4.7e-7 (4.4e-6; 5.9e-7); rank 256:
// 8.0e-7. Runs of 256 halve it and cost more: one row 70 -> 76 us, 256 rows with 32 adapters of rank 32 236 -> 277.
// 0 times an Inf or NaN in an adapter's b is NaN, in the rows around its run too (and so is a part of h that is 0 times an Inf of the row's
// own): where a group has adapters, the epilogue's warps work the NaNs out again at their end, from the row's own operands, unless x holds one.
constexpr int LMA_UNIT = 16;             // columns of the rank in a unit: K of one MMA, 32 bytes
constexpr int LMA_PARTS = 3;             // bf16 that make up a value of h
constexpr int LMA_SEG = 512;             // products of a sum on the tensor pipe
// Of an item's nkc chunks of K, the first of the sum behind the one that begins with chunk kc. The last sum, which goes on over the
// adapters, has fewer chunks where their rank is high, and the sums ahead of it what is left.
__device__ __forceinline__ int lma_next_sum(int kc, int nkc, int units) {
  constexpr int SEG = LMA_SEG / (LMH_SUB * LMH_BK), STEPS = LMH_SUB * LMH_BK / 16;   // chunks of a sum, steps of a chunk
  const int last = nkc - max(1, min(SEG, SEG + (2 * STEPS - LMA_PARTS * units) / STEPS));
  return kc >= last ? nkc : min(kc + SEG, last);
}
constexpr int LMA_STAGE = 4;             // units in a stage, and warps of a CTA that ask for them: one for each of a stage's units
// Four warpgroups: producer and issuer (and two warps without work), two of the epilogue, those who ask for units. An epilogue thread holds the
// sums of 128 logits, so the other warpgroups hand registers over to it, out of the 128 a thread that the block is launched with.
constexpr int LMA_EPI0 = 4;              // the epilogue's first warp
constexpr int LMA_RUN_NT = 512;
constexpr int LMA_REGS_EPI = 176, LMA_REGS = 72, LMA_REGS_LAUNCH = 128;
static_assert(LMA_EPI0 + LMH_EPI + LMA_STAGE == LMA_RUN_NT / 32 && 256 * LMA_REGS_EPI + 256 * LMA_REGS <= LMA_RUN_NT * LMA_REGS_LAUNCH, "what is handed over is there");
constexpr int LMA_RING_BYTES = 200 * 1024, LMA_DYN_BYTES = LMA_RING_BYTES + 1024;
constexpr int LMA_MAX_RANK = 256;
constexpr int LMA_NT = 256;              // of the kernels ahead of the projection
constexpr int LMA_BOX = 16;              // batch rows of h that one TMA load brings
// a stage's units: b in the first of w's boxes, two parts of h on the x side, the third in the second of w's boxes
static_assert(LMA_PARTS == 3 && LMH_SUB == 2 && LMA_STAGE * 2 * 32 <= LMH_SUB * LMH_BK * 2 && LMA_STAGE * LMH_CTA_V * 32 <= LMH_W_BYTES &&
              LMA_STAGE * (LMH_MAX_N / 2) * 32 <= LMH_W_BYTES, "a stage holds its units");
static_assert(LMA_NT >= LMH_MAX_N && LMA_SEG % (LMH_SUB * LMH_BK) == 0, "a thread per batch row of a group, whole chunks in a sum");

struct LmaRun { int32_t adapter, n0, n1, pad; };   // of a group: its rows n0 .. n1 - 1, multiples of 32, hold the adapter's
struct LmAdaptArgs {
  CUtensorMap map_b;       // b [n, V, rank] bf16, box 16 x cta_v, 32-byte swizzle
  CUtensorMap map_h;       // h [group][unit][LMA_PARTS][item_n] rows of 16 bf16, box 16 x LMA_BOX, 32-byte swizzle
  const uint16_t *x, *w, *a, *b;
  int64_t ldx, ldw, a_pitch, a_stride, b_pitch, b_stride;   // in elements
  const float* scales;     // [n] or null: 1
  const int32_t* row_adapter;   // [B]; outside [0, n): none
  int32_t n, rank, units;  // adapters, their rank, units of one
  int32_t max_runs;        // of a group
  int32_t B, K, item_n;
  // the workspace
  int32_t* nruns;          // [group]
  LmaRun* runs;            // [group][max_runs]
  int32_t* order;          // [B] the row at each place of the order
  int32_t* sorted;         // [B] its adapter, -1: none
  int32_t* row_nan;        // [B] whether its x holds a NaN
  uint16_t* xs;            // [B, K] x in that order
  uint16_t* h;
};
__device__ __forceinline__ int64_t lma_h_row(const LmAdaptArgs& D, int group, int unit, int piece, int row) {
  return ((static_cast<int64_t>(group) * D.max_runs * D.units + unit) * LMA_PARTS + piece) * D.item_n + row;
}

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// The place of row b in the order of (adapter, row), rows without one last. All of the CTA's threads; keys: 4 * LMA_NT words.
__device__ __forceinline__ int lma_place(const LmAdaptArgs& D, int b, int key, int* keys, int tid) {
  int place = 0;
  for (int j0 = 0; j0 < D.B; j0 += 4 * LMA_NT) {
    __syncthreads();
    for (int j = tid; j < 4 * LMA_NT; j += LMA_NT) {
      const int a = j0 + j < D.B ? D.row_adapter[j0 + j] : 0;
      keys[j] = j0 + j < D.B ? ((a < 0 || a >= D.n) ? D.n : a) : 0x7fffffff;
    }
    __syncthreads();
    const int lim = min(4 * LMA_NT, D.B - j0);
#pragma unroll 4
    for (int j = 0; j < lim; j += 4) {
      const int4 o = *reinterpret_cast<const int4*>(&keys[j]);
      const int at = j0 + j;
      place += (o.x < key || (o.x == key && at < b)) + (o.y < key || (o.y == key && at + 1 < b)) + (o.z < key || (o.z == key && at + 2 < b)) +
               (o.w < key || (o.w == key && at + 3 < b));
    }
  }
  return place;
}
__global__ void __launch_bounds__(LMA_NT) lm_adapters_order_kernel(const __grid_constant__ LmAdaptArgs D) {
  __shared__ __align__(16) int keys[4 * LMA_NT];
  const int tid = threadIdx.x, b = blockIdx.x * LMA_NT + tid;
  int a = b < D.B ? D.row_adapter[b] : -1;
  if (a < 0 || a >= D.n) a = -1;
  const int place = lma_place(D, b, a < 0 ? D.n : a, keys, tid);
  if (b < D.B) { D.order[place] = b; D.sorted[place] = a; }
  pdl_launch();
}

// The next eight bits of v as a bf16, taken off v. Cut off, not rounded: a value next to f32's largest stays finite, and
// 8 + 8 + 8 bits are all that f32 has. An infinity or a NaN is in the first part alone.
__device__ __forceinline__ uint32_t lma_part(float& v) {
  if (!(fabsf(v) < INFINITY)) {
    const uint32_t bits = bf16_bits_rne(v);
    v = 0.0f;
    return bits;
  }
  const uint32_t top = __float_as_uint(v) & 0xffff0000u;
  v -= __uint_as_float(top);                                         // (exact)
  return top >> 16;
}

// A CTA per place of the order: the runs of its group, its row of x, its h. Up to LMA_NT rows are put in order here (ordered == 0).
__global__ void __launch_bounds__(LMA_NT) lm_adapters_kernel(const __grid_constant__ LmAdaptArgs D, const int32_t ordered) {
  __shared__ __align__(16) int keys[4 * LMA_NT];
  __shared__ int s_ad[LMA_NT + 1], s_start[LMA_NT + 1], s_first[LMA_NT / 32], s_row, s_mine;
  __shared__ float s_h[LMA_MAX_RANK];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int p = blockIdx.x, g = p / D.item_n, g0 = g * D.item_n, rows = min(D.item_n, D.B - g0);
  pdl_launch();
  if (ordered) {
    pdl_wait();
    s_ad[tid] = tid < rows ? D.sorted[g0 + tid] : -1;
    if (tid == 0) s_row = D.order[p];
  } else {
    int a = tid < D.B ? D.row_adapter[tid] : -1;
    if (a < 0 || a >= D.n) a = -1;
    s_ad[tid] = -1;
    const int place = lma_place(D, tid, a < 0 ? D.n : a, keys, tid);   // (its barriers come before the next line)
    if (tid < D.B) {
      if (place >= g0 && place < g0 + rows) s_ad[place - g0] = a;
      if (place == p) s_row = tid;
      if (p == 0) { D.order[place] = tid; D.sorted[place] = a; }
    }
  }
  if (tid == 0) s_mine = -1;
  __syncthreads();
  const int a = s_ad[tid];
  const bool first = a >= 0 && (tid == 0 || s_ad[tid - 1] != a);
  const uint32_t votes = __ballot_sync(FULL, first);
  if (lane == 0) s_first[warp] = __popc(votes);
  const int taught = __syncthreads_count(a >= 0);                    // rows with an adapter: the first ones
  int run = __popc(votes & ((1u << lane) - 1u)), nruns = 0;
  for (int w = 0; w < LMA_NT / 32; w++) { run += w < warp ? s_first[w] : 0; nruns += s_first[w]; }
  if (first) s_start[run] = tid;
  if (tid == 0) s_start[nruns] = taught;
  __syncthreads();
  const int mine = s_ad[p - g0], row = s_row;
  if (tid < nruns) {
    LmaRun r;
    r.adapter = s_ad[s_start[tid]];
    r.n0 = s_start[tid] & ~31;
    r.n1 = (s_start[tid + 1] + 31) & ~31;
    r.pad = 0;
    if (p == g0) D.runs[static_cast<int64_t>(g) * D.max_runs + tid] = r;
    if (r.adapter == mine) s_mine = tid;
  }
  if (p == g0 && tid == 0) D.nruns[g] = nruns;
  // x in its place, and h = scale * a x, a rank's row per warp
  const uint4* x4 = reinterpret_cast<const uint4*>(D.x + row * D.ldx);
  uint4* xs4 = reinterpret_cast<uint4*>(D.xs + static_cast<int64_t>(p) * D.K);
  const int nk = D.K / 8;
  bool nan = false;
  for (int k = tid; k < nk; k += LMA_NT) {
    const uint4 q = __ldg(x4 + k);
    xs4[k] = q;
    const uint32_t ws[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int c = 0; c < 4; c++) nan |= (ws[c] & 0x7fffu) > 0x7f80u || (ws[c] & 0x7fff0000u) > 0x7f800000u;
  }
  if (mine >= 0) {
    const float scale = D.scales ? D.scales[mine] : 1.0f;
    for (int r = warp; r < D.rank; r += LMA_NT / 32) {
      const uint4* a4 = reinterpret_cast<const uint4*>(D.a + mine * D.a_stride + r * D.a_pitch);
      float acc = 0.0f;
#pragma unroll 4
      for (int k = lane; k < nk; k += 32) {
        const uint4 q = __ldg(x4 + k), t = __ldg(a4 + k);
        acc = fmaf(bf16_lo(q.x), bf16_lo(t.x), acc); acc = fmaf(bf16_hi(q.x), bf16_hi(t.x), acc);
        acc = fmaf(bf16_lo(q.y), bf16_lo(t.y), acc); acc = fmaf(bf16_hi(q.y), bf16_hi(t.y), acc);
        acc = fmaf(bf16_lo(q.z), bf16_lo(t.z), acc); acc = fmaf(bf16_hi(q.z), bf16_hi(t.z), acc);
        acc = fmaf(bf16_lo(q.w), bf16_lo(t.w), acc); acc = fmaf(bf16_hi(q.w), bf16_hi(t.w), acc);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(FULL, acc, o);
      if (lane == 0) s_h[r] = acc * scale;
    }
  }
  const int any = __syncthreads_or(nan);                             // (and s_h and s_mine are there)
  if (tid == 0) D.row_nan[p] = any;
  // this row of the runs whose 32s hold it: half of a unit's row at a time, 16 bytes of each part
  const int at = p - g0;
  for (int i = tid; i < nruns * D.units * 2; i += LMA_NT) {
    const int unit = i >> 1, half = i & 1, q = unit / D.units;
    if (at < (s_start[q] & ~31) || at >= ((s_start[q + 1] + 31) & ~31)) continue;
    uint32_t o[LMA_PARTS][4] = {};
    if (q == s_mine) {
      const int r0 = (unit - q * D.units) * LMA_UNIT + half * 8;
#pragma unroll
      for (int c = 0; c < 8; c++) {
        float v = (r0 + c < D.rank) ? s_h[r0 + c] : 0.0f;
#pragma unroll
        for (int piece = 0; piece < LMA_PARTS; piece++) o[piece][c >> 1] |= lma_part(v) << (16 * (c & 1));
      }
    }
#pragma unroll
    for (int piece = 0; piece < LMA_PARTS; piece++)
      *(reinterpret_cast<uint4*>(D.h + lma_h_row(D, g, unit, piece, at) * LMA_UNIT) + half) = make_uint4(o[piece][0], o[piece][1], o[piece][2], o[piece][3]);
  }
}

// One logit from its row's own operands, in f32. p: the row's place in the order; a: its adapter (below 0: none), run: that one's in its
// group. The adapter's part first: a NaN there settles it at little cost.
__device__ __forceinline__ float lma_logit(const LmAdaptArgs& D, int p, int v, int a, int run) {
  float own = 0.0f;
  if (a >= 0) {
    const int g = p / D.item_n;
    const uint16_t* brow = D.b + a * D.b_stride + v * D.b_pitch;
    for (int r = 0; r < D.rank && own == own; r++) {
      float h = 0.0f;                                                    // (the parts' sum is exact)
#pragma unroll
      for (int piece = 0; piece < LMA_PARTS; piece++)
        h += __uint_as_float(static_cast<uint32_t>(D.h[lma_h_row(D, g, run * D.units + r / LMA_UNIT, piece, p - g * D.item_n) * LMA_UNIT + r % LMA_UNIT]) << 16);
      own = fmaf(h, __uint_as_float(static_cast<uint32_t>(__ldg(brow + r)) << 16), own);
    }
  }
  const uint4 *x4 = reinterpret_cast<const uint4*>(D.xs + static_cast<int64_t>(p) * D.K), *w4 = reinterpret_cast<const uint4*>(D.w + v * D.ldw);
  float acc = 0.0f;
  for (int k0 = 0; k0 < D.K / 8 && own == own && acc == acc; k0 += LMH_BK / 8) {
    uint4 q[LMH_BK / 8], t[LMH_BK / 8];
#pragma unroll
    for (int k = 0; k < LMH_BK / 8; k++) { q[k] = x4[k0 + k]; t[k] = __ldg(w4 + k0 + k); }
#pragma unroll
    for (int k = 0; k < LMH_BK / 8; k++) {
      const uint32_t qs[4] = {q[k].x, q[k].y, q[k].z, q[k].w}, ts[4] = {t[k].x, t[k].y, t[k].z, t[k].w};
#pragma unroll
      for (int c = 0; c < 4; c++) { acc = fmaf(bf16_lo(qs[c]), bf16_lo(ts[c]), acc); acc = fmaf(bf16_hi(qs[c]), bf16_hi(ts[c]), acc); }
    }
  }
  return acc + own;
}

// A group's runs in shared memory, one table for each of the threads that walk them: a trip to L2 for every run of every
// item was much of the time (64 rows with eight adapters: 106 us with, 92 without).
struct LmaTable { int32_t adapter[LMA_NT]; uint16_t n0[LMA_NT], n1[LMA_NT]; int32_t group, nruns; };
__device__ __forceinline__ void lma_fetch_runs(LmaTable& t, const LmAdaptArgs& D, int g) {
  if (t.group == g) return;
  t.group = g;
  t.nruns = D.nruns[g];
  const LmaRun* runs = D.runs + static_cast<int64_t>(g) * D.max_runs;
#pragma unroll 8
  for (int i = 0; i < t.nruns; i++) {
    const int4 r = *reinterpret_cast<const int4*>(runs + i);
    t.adapter[i] = r.x;
    t.n0[i] = static_cast<uint16_t>(r.y);
    t.n1[i] = static_cast<uint16_t>(r.z);
  }
}
// The units of an item, in order: every run that has rows among the item's, and its share of them. The producers and the issuer
// walk them alike.
struct LmaUnits {
  const LmaTable& t;
  int units, g, i0, i1, run, nruns, ru, n0, n1, adapter;
  __device__ __forceinline__ LmaUnits(LmaTable& table, const LmAdaptArgs& D, int b0, int n) : t(table) {
    g = b0 / D.item_n; i0 = b0 - g * D.item_n; i1 = i0 + n;
    lma_fetch_runs(table, D, g);
    nruns = t.nruns;
    units = D.units;
    run = -1;
    ru = units - 1;
  }
  __device__ __forceinline__ bool next() {
    if (++ru < units) return run < nruns;
    ru = 0;
    while (++run < nruns) {
      adapter = t.adapter[run];
      n0 = max(static_cast<int>(t.n0[run]), i0);
      n1 = min(static_cast<int>(t.n1[run]), i1);
      if (n0 < n1) return true;
    }
    return false;
  }
};

// Work items in the order in which pair p takes them: p, p + npairs, ...: first the whole rounds of full
// items (all batch rows of `full` vocabulary tiles, item_n at a time), then the remaining tiles in items
// of small_n batch rows, at most one round of them.
struct LmhItem { int vt, b0, n; };
struct LmhPlan {
  int nb, full, nfull, nsmall, total, item_n, small_n, B;
  __host__ __device__ LmhPlan(int B_, int ntile, int item_n_, int npairs) {
    B = B_; item_n = item_n_;
    nb = (B + item_n - 1) / item_n;
    full = (ntile * nb / npairs) * npairs / nb;
    nfull = full * nb;
    const int rest = (ntile - full) * nb;
    int s = 1;
    while (rest > 0 && 2 * s * rest <= npairs && item_n / (2 * s) >= 32) s *= 2;
    small_n = (item_n / s + 31) & ~31;
    nsmall = (B + small_n - 1) / small_n;
    total = nfull + (ntile - full) * nsmall;
  }
  __device__ __forceinline__ LmhItem at(int i) const {
    LmhItem it;
    const bool f = i < nfull;
    const int q = f ? i : i - nfull, per = f ? nb : nsmall, n = f ? item_n : small_n;
    it.vt = (f ? 0 : full) + q / per;
    it.b0 = (q % per) * n;
    it.n = min(n, ((B - it.b0) + 31) & ~31);
    return it;
  }
};

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}
// Bounded wait for the phase with parity `parity` to complete; false when it ran out or another role gave up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  for (uint32_t it = 0; it < LMH_WAIT_LIMIT; it++) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
    if ((it & 63u) == 63u && *abort_flag) return false;
  }
  *abort_flag = 1;
  return false;
}
// The address of this CTA's shared variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(cluster_addr) : "memory");
}
// A tile into this CTA's shared memory; its bytes complete on a barrier that may be the pair's other CTA's.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, unsigned long long pol) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
               :: "r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "l"(pol) : "memory");
}
// Shared-memory matrix descriptor of a K-major tile of 128-byte rows with the 128-byte swizzle: start
// address / 16, leading byte offset 1 (unused for swizzled K-major), stride byte offset 1024 / 16 (eight
// rows), descriptor version 1 at bit 46, layout type 2 (128-byte swizzle) at bits 61-63.
__device__ __forceinline__ uint64_t umma_desc(uint32_t smem_addr_bytes) {
  return static_cast<uint64_t>((smem_addr_bytes & 0x3ffffu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// The same for 32-byte rows with the 32-byte swizzle: eight rows are 256 bytes, layout type 6.
__device__ __forceinline__ uint64_t umma_desc_32b(uint32_t smem_addr_bytes) {
  return static_cast<uint64_t>((smem_addr_bytes & 0x3ffffu) >> 4) | (1ull << 16) | (16ull << 32) | (1ull << 46) | (6ull << 61);
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, unsigned long long pol) {
  asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5}], [%2], %6;"
               :: "r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "l"(pol) : "memory");
}
__device__ __forceinline__ void umma_f16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      :: "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// Arrives on the barrier at this offset in both CTAs of the pair when the MMAs issued so far are done.
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               :: "r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr) : "memory");
}

// The items of an epilogue warp again, behind all its others: a lane reads back what it wrote. (Behind them, so that no wait is held up
// by it, and where the sums' registers are free.)
__device__ __noinline__ void lma_second_look(const LmHeadArgs& A, const LmAdaptArgs& D) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = warp & 3, half = (warp - LMA_EPI0) >> 2;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1, rank = blockIdx.x & 1;
  const LmhPlan plan(A.B, A.ntile, A.item_n, npairs);
  for (int i = pair; i < plan.total; i += npairs) {
    const LmhItem it = plan.at(i);
    const int nruns = D.nruns[it.b0 / A.item_n];
    if (nruns == 0) continue;
    const LmaRun* runs = D.runs + static_cast<int64_t>(it.b0 / A.item_n) * D.max_runs;
    const int in_tile = rank * A.cta_v + q * 32 + lane, v = (A.tile0 + it.vt * A.tile_step) * 2 * A.cta_v + in_tile;
    const bool live = q * 32 + lane < A.cta_v && v < A.V;
    for (int c = half * 32; c < it.n; c += 64) {
      const int b0 = it.b0 + c, nb = min(32, A.B - b0);
      for (int j = 0; j < nb; j++) {
        if (D.row_nan[b0 + j]) continue;
        float* at = A.out_logits + D.order[b0 + j] * A.ld_out + v;
        const bool odd = live && *at != *at;
        if (!__any_sync(FULL, odd)) continue;
        const int a = D.sorted[b0 + j];
        int run = -1;
        for (int r0 = 0; a >= 0 && run < 0; r0 += 32) {                  // (it is there)
          const uint32_t hit = __ballot_sync(FULL, r0 + lane < nruns && runs[r0 + lane].adapter == a);
          if (hit != 0u || r0 + 32 >= nruns) run = r0 + max(__ffs(hit) - 1, 0);
        }
        if (odd) *at = lma_logit(D, b0 + j, v, a, run);
      }
    }
  }
}

// s += 16 columns of an accumulator, rounded to nearest. (One statement, so that 16 registers and no more hold what is loaded.)
__device__ __forceinline__ void tmem_add16(uint32_t taddr, float* s) {
  asm volatile(
      "{\n\t.reg .b32 t<16>;\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {t0, t1, t2, t3, t4, t5, t6, t7, t8, t9, t10, t11, t12, t13, t14, t15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;\n\t"
      "add.rn.f32 %0, %0, t0;\n\tadd.rn.f32 %1, %1, t1;\n\tadd.rn.f32 %2, %2, t2;\n\tadd.rn.f32 %3, %3, t3;\n\t"
      "add.rn.f32 %4, %4, t4;\n\tadd.rn.f32 %5, %5, t5;\n\tadd.rn.f32 %6, %6, t6;\n\tadd.rn.f32 %7, %7, t7;\n\t"
      "add.rn.f32 %8, %8, t8;\n\tadd.rn.f32 %9, %9, t9;\n\tadd.rn.f32 %10, %10, t10;\n\tadd.rn.f32 %11, %11, t11;\n\t"
      "add.rn.f32 %12, %12, t12;\n\tadd.rn.f32 %13, %13, t13;\n\tadd.rn.f32 %14, %14, t14;\n\tadd.rn.f32 %15, %15, t15;\n\t}"
      : "+f"(s[0]), "+f"(s[1]), "+f"(s[2]), "+f"(s[3]), "+f"(s[4]), "+f"(s[5]), "+f"(s[6]), "+f"(s[7]),
        "+f"(s[8]), "+f"(s[9]), "+f"(s[10]), "+f"(s[11]), "+f"(s[12]), "+f"(s[13]), "+f"(s[14]), "+f"(s[15])
      : "r"(taddr) : "memory");
}

// ADAPT: with D's adapters (D is null otherwise). It is then launched as a dependent of the kernel that puts the rows in order, with w
// there before.
template <bool ADAPT>
__device__ __forceinline__ void lm_head_run(const LmHeadArgs& A, const LmAdaptArgs* D) {
  // accumulators in tensor memory
  constexpr int MAX_ACC = LMH_TMEM_COLS / (ADAPT ? LMH_MAX_N / 2 : LMH_MAX_N);
  const int acc_cols = ADAPT && A.item_n <= LMH_MAX_N / 2 ? LMH_MAX_N / 2 : LMH_MAX_N;
  const uint32_t nacc = static_cast<uint32_t>(LMH_TMEM_COLS / acc_cols);
  extern __shared__ __align__(16) unsigned char lmh_dyn[];
  __shared__ __align__(8) unsigned long long full_bar[LMH_MAX_STAGES], empty_bar[LMH_MAX_STAGES], acc_full[MAX_ACC], acc_empty[MAX_ACC];
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_s;
  __shared__ __align__(16) float stash_thr[LMH_EPI][32];
  __shared__ uint2 stash[LMH_EPI][64];
  __shared__ int stash_row[LMH_EPI][64];
  __shared__ __align__(16) unsigned char lma_space[ADAPT ? (2 + LMA_STAGE) * sizeof(LmaTable) : 16];
  __shared__ int lma_places[ADAPT ? LMH_EPI : 1][ADAPT ? LMH_MAX_N / 2 : 1];   // of an epilogue warp's batch rows: the rows' own places
  __shared__ uint32_t lma_given;                                        // stages of units that the producer has found free and announced
  LmaTable* lma_tables = reinterpret_cast<LmaTable*>(lma_space);     // warp 0's, warp 1's, and of those that ask for units
  constexpr int EPI0 = ADAPT ? LMA_EPI0 : 2;                            // the epilogue's first warp
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = blockIdx.x & 1u;                                // in the pair; 0 leads
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const uint32_t ring = (smem_addr(lmh_dyn) + 1023u) & ~1023u;          // the swizzled tiles need 1024-byte alignment
  volatile int* abort_flag = &abort_s;
  const int nk64 = A.K / LMH_BK, nkc = (nk64 + LMH_SUB - 1) / LMH_SUB;  // K boxes and chunks per item
  const int nst = A.stages;
  const uint32_t x_bytes = static_cast<uint32_t>(A.box_n) * LMH_BK * 2, stage_bytes = LMH_SUB * (LMH_W_BYTES + x_bytes);
  const LmhPlan plan(A.B, A.ntile, A.item_n, npairs);
  pdl_launch();
  // What fills x and w, or uses the output. Ahead of the tensor memory, which a kernel that still runs may want, and of the
  // bounded waits. The launch overlaps that kernel's end (us a call, back to back, without | so: 4 x 512 x 1,000: 10.1 | 7.5,
  // 16 x 512 x 4,096: 10.2 | 7.0, 300 x 1,024 x 8,192: 14.5 | 12.4, 512 x 1,024 x 151,936: 180.1 | 178.1).
  if (!A.chained) pdl_wait();

  if (tid == 0) {
    for (int s = 0; s < nst; s++) { mbar_init(smem_addr(&full_bar[s]), 1); mbar_init(smem_addr(&empty_bar[s]), 1); }
    for (int b = 0; b < MAX_ACC; b++) { mbar_init(smem_addr(&acc_full[b]), 1); mbar_init(smem_addr(&acc_empty[b]), 2 * LMH_EPI); }
    abort_s = 0;
    if constexpr (ADAPT) {
      for (int t = 0; t < 2 + LMA_STAGE; t++) lma_tables[t].group = -1;
      lma_given = 0;
    }
    if (A.clear_status && blockIdx.x == 0) *A.status = 0u;              // (a wait runs out seconds later, if ever)
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {                                                      // one warp of each CTA takes the tensor memory
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_addr(&tmem_base_s)), "r"(LMH_TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");   // both CTAs' barriers exist
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_base_s;

  if constexpr (ADAPT) {
    if (warp < EPI0 || warp >= EPI0 + LMH_EPI) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(LMA_REGS));
  }
  if (warp == 0) {
    // ---- producer: this CTA's share of every stage; its bytes complete on the leader's barrier
    if (lane == 0) {
      unsigned long long pol_w, pol_x;                                  // the weights pass once per batch tile, x stays
      asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(pol_w));
      asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(pol_x));
      if (plan.nb > 1) asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(pol_w));
      uint32_t stage = 0, phase = 0;
      [[maybe_unused]] uint32_t given = 0;                              // stages of units handed on
      bool ok = true;
      for (int i = pair; i < plan.total && ok; i += npairs) {
        const LmhItem it = plan.at(i);
        const int v0 = ((A.tile0 + it.vt * A.tile_step) * 2 + static_cast<int>(rank)) * A.cta_v;
        const int xb = it.b0 + static_cast<int>(rank) * (it.n >> 1);
        int asked = 0;
        if constexpr (ADAPT) {
          if (i == pair) {                                              // the first stages' weights ahead of the wait for x in its order
            asked = min(nst, nkc);
            for (int kc = 0; kc < asked; kc++) {
              const uint32_t own = smem_addr(&full_bar[kc]), bar = map_rank(own, 0);
              const int subs = min(LMH_SUB, nk64 - kc * LMH_SUB);
              if (rank == 0) mbar_expect_tx(own, 2 * subs * (static_cast<uint32_t>(A.cta_v) * LMH_BK * 2 + x_bytes));
              for (int u = 0; u < subs; u++) tma_load_2d_pair(ring + kc * stage_bytes + u * LMH_W_BYTES, &A.map_w, bar, (kc * LMH_SUB + u) * LMH_BK, v0, pol_w);
            }
            pdl_wait();
          }
        }
        for (int kc = 0; kc < nkc; kc++) {
          if (!ADAPT || kc >= asked) if (!mbar_wait(smem_addr(&empty_bar[stage]), phase ^ 1u, abort_flag)) { ok = false; break; }
          const uint32_t own = smem_addr(&full_bar[stage]), bar = map_rank(own, 0);
          const uint32_t sw = ring + stage * stage_bytes, sx = sw + LMH_SUB * LMH_W_BYTES;
          const int subs = min(LMH_SUB, nk64 - kc * LMH_SUB);
          if (!ADAPT || kc >= asked) {
            if (rank == 0) mbar_expect_tx(own, 2 * subs * (static_cast<uint32_t>(A.cta_v) * LMH_BK * 2 + x_bytes));
            for (int u = 0; u < subs; u++) tma_load_2d_pair(sw + u * LMH_W_BYTES, &A.map_w, bar, (kc * LMH_SUB + u) * LMH_BK, v0, pol_w);
          }
          for (int u = 0; u < subs; u++) tma_load_2d_pair(sx + u * x_bytes, &A.map_x, bar, (kc * LMH_SUB + u) * LMH_BK, xb, pol_x);
          if (++stage == static_cast<uint32_t>(nst)) { stage = 0; phase ^= 1u; }
        }
        if constexpr (ADAPT) {
          LmaUnits un(lma_tables[0], *D, it.b0, it.n);
          bool more = ok && un.next();
          while (more) {
            uint32_t bytes = 0;
            for (int u = 0; u < LMA_STAGE && more; u++, more = un.next()) bytes += static_cast<uint32_t>(A.cta_v) * 32 + static_cast<uint32_t>(un.n1 - un.n0) * (LMA_PARTS * 16);
            if (!mbar_wait(smem_addr(&empty_bar[stage]), phase ^ 1u, abort_flag)) { ok = false; break; }
            // (the pair's other CTA may have its copies there before this says how many there are: the phase waits for this arrival)
            if (rank == 0) mbar_expect_tx(smem_addr(&full_bar[stage]), 2 * bytes);
            given++;
            asm volatile("st.release.cta.shared.u32 [%0], %1;" :: "r"(smem_addr(&lma_given)), "r"(given) : "memory");
            if (++stage == static_cast<uint32_t>(nst)) { stage = 0; phase ^= 1u; }
          }
        }
      }
    }
  } else if (ADAPT && warp >= EPI0 + LMH_EPI) {
    // ---- who asks for the units: warp j for the j-th of every stage. (Which stages are free is the producer's word: one of these
    // could be rounds ahead of a barrier, and its parity would not say so.)
    if (lane == 0) {
      const int j = warp - (EPI0 + LMH_EPI);
      unsigned long long pol_w, pol_x;
      asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(pol_w));
      asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(pol_x));
      if (plan.nb > 1) asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(pol_w));
      uint32_t stage = 0, seen = 0;                                     // seen: stages of units so far
      bool ok = true;
      const uint32_t hb = static_cast<uint32_t>(A.box_n) * 32;
      pdl_wait();
      for (int i = pair; i < plan.total && ok; i += npairs) {
        const LmhItem it = plan.at(i);
        const int v0 = ((A.tile0 + it.vt * A.tile_step) * 2 + static_cast<int>(rank)) * A.cta_v;
        stage = (stage + static_cast<uint32_t>(nkc)) % nst;
        LmaUnits un(lma_tables[2 + j], *D, it.b0, it.n);
        bool more = un.next();
        while (more && ok) {
          const uint32_t sw = ring + stage * stage_bytes, sx = sw + LMH_SUB * LMH_W_BYTES, bar = map_rank(smem_addr(&full_bar[stage]), 0);
          for (int u = 0; u < LMA_STAGE && more; u++, more = un.next()) {
            if (u != j) continue;
            const int half = (un.n1 - un.n0) >> 1, r0 = un.n0 + static_cast<int>(rank) * half;   // this CTA's batch rows of the unit
            const int hrow = static_cast<int>(lma_h_row(*D, un.g, un.run * D->units + un.ru, 0, r0));
            for (uint32_t have = 0, polls = 0; have <= seen; polls++) {
              asm volatile("ld.acquire.cta.shared.u32 %0, [%1];" : "=r"(have) : "r"(smem_addr(&lma_given)) : "memory");
              if ((polls & 63u) == 63u) {                               // (a stage comes within a tile's time; after a thousand looks, with pauses)
                if (polls > 1024u) __nanosleep(200);
                if (have <= seen && (polls == LMH_WAIT_LIMIT + 63u || *abort_flag)) { *abort_flag = 1; ok = false; break; }
              }
            }
            if (!ok) break;
            tma_load_3d_pair(sw + u * (LMH_CTA_V * 32), &D->map_b, bar, un.ru * LMA_UNIT, v0, un.adapter, pol_w);
            for (int q = 0; q < half; q += LMA_BOX) {
              tma_load_2d_pair(sx + 2 * u * hb + q * 32, &D->map_h, bar, 0, hrow + q, pol_x);
              tma_load_2d_pair(sx + (2 * u + 1) * hb + q * 32, &D->map_h, bar, 0, hrow + A.item_n + q, pol_x);
              tma_load_2d_pair(sw + LMH_W_BYTES + u * hb + q * 32, &D->map_h, bar, 0, hrow + 2 * A.item_n + q, pol_x);
            }
          }
          seen++;
          if (++stage == static_cast<uint32_t>(nst)) stage = 0;
        }
      }
    }
  } else if (warp == 1) {
    // ---- issuer
    if (rank == 0 && lane == 0) {
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      bool ok = true;
      for (int i = pair; i < plan.total && ok; i += npairs) {
        const uint32_t idesc = lmh_idesc(plan.at(i).n);
        if (!mbar_wait(smem_addr(&acc_empty[acc]), acc_phase ^ 1u, abort_flag)) { ok = false; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t d_tmem = tmem_base + acc * acc_cols;
        int fresh = 0;                                                  // the chunk that begins a sum, and the one that begins the next
        [[maybe_unused]] int next_sum = nkc;
        if constexpr (ADAPT) next_sum = lma_next_sum(0, nkc, D->units);
        for (int kc = 0; kc < nkc; kc++) {
          if (ADAPT && kc == next_sum) {                                // on to the next accumulator
            umma_commit_pair(smem_addr(&acc_full[acc]));
            if (++acc == nacc) { acc = 0; acc_phase ^= 1u; }
            if (!mbar_wait(smem_addr(&acc_empty[acc]), acc_phase ^ 1u, abort_flag)) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            d_tmem = tmem_base + acc * acc_cols;
            fresh = kc;
            if constexpr (ADAPT) next_sum = lma_next_sum(kc, nkc, D->units);
          }
          if (!mbar_wait(smem_addr(&full_bar[stage]), phase, abort_flag)) { ok = false; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t sw = ring + stage * stage_bytes, sx = sw + LMH_SUB * LMH_W_BYTES;
          const int subs = min(LMH_SUB, nk64 - kc * LMH_SUB);
          for (int u = 0; u < subs; u++) {
#pragma unroll
            for (int k = 0; k < LMH_BK / 16; k++)
              umma_f16_pair(d_tmem, umma_desc(sw + u * LMH_W_BYTES + k * 32), umma_desc(sx + u * x_bytes + k * 32), idesc, (kc > fresh || u > 0 || k > 0) ? 1u : 0u);
          }
          umma_commit_pair(smem_addr(&empty_bar[stage]));               // the stage is free once these MMAs have read it
          if (++stage == static_cast<uint32_t>(nst)) { stage = 0; phase ^= 1u; }
        }
        if constexpr (ADAPT) {
          pdl_wait();
          const LmhItem it = plan.at(i);
          LmaUnits un(lma_tables[1], *D, it.b0, it.n);
          bool more = ok && un.next();
          while (more) {
            if (!mbar_wait(smem_addr(&full_bar[stage]), phase, abort_flag)) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t sw = ring + stage * stage_bytes, sx = sw + LMH_SUB * LMH_W_BYTES, hb = static_cast<uint32_t>(A.box_n) * 32;
            for (int u = 0; u < LMA_STAGE && more; u++, more = un.next()) {
              for (int piece = 0; piece < LMA_PARTS; piece++)
                umma_f16_pair(d_tmem + static_cast<uint32_t>(un.n0 - un.i0), umma_desc_32b(sw + u * (LMH_CTA_V * 32)),
                              umma_desc_32b(piece < 2 ? sx + (2 * u + piece) * hb : sw + LMH_W_BYTES + u * hb), lmh_idesc(un.n1 - un.n0), 1u);
            }
            umma_commit_pair(smem_addr(&empty_bar[stage]));
            if (++stage == static_cast<uint32_t>(nst)) { stage = 0; phase ^= 1u; }
          }
        }
        if (ok) umma_commit_pair(smem_addr(&acc_full[acc]));            // the accumulator is complete
        if (++acc == nacc) { acc = 0; acc_phase ^= 1u; }
      }
    }
  } else if (warp >= EPI0) {
    if constexpr (ADAPT) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(LMA_REGS_EPI));
    // ---- epilogue: warp w reads TMEM lanes 32 * (w % 4) .. + 31; thread = vocabulary row
    const int q = warp & 3, half = (warp - EPI0) >> 2;                     // this warp's lanes, and its share of the columns
    uint32_t acc = 0, acc_phase = 0;
    bool ok = true;
    int nstash = 0;
    auto flush = [&](int count) {                                       // the stash's first `count` entries to their rows' lists
      __syncwarp();
      if (lane < count) {
        const uint2 e = stash[warp - EPI0][lane];
        const int b = stash_row[warp - EPI0][lane];
        const float x = __uint_as_float(e.x);
        if (x != x) {
          atomicOr(&A.rows[b].nan, (e.y == 0u) ? 3 : 1);
        } else {
          const int slot = atomicAdd(&A.rows[b].cnt, 1);
          if (slot < LMH_CAND_CAP) A.cand[static_cast<int64_t>(b) * LMH_CAND_CAP + slot] = e;
        }
      }
      __syncwarp();
    };
    [[maybe_unused]] int places_of = -1, places_n = 0;
    [[maybe_unused]] bool adapted = false, saw_nan = false;
    if (A.chained) pdl_wait();                                          // the thresholds; tiles and MMAs are under way meanwhile
    for (int i = pair; i < plan.total && ok; i += npairs) {
      const LmhItem it = plan.at(i);
      const int in_tile = static_cast<int>(rank) * A.cta_v + q * 32 + lane;
      const int v = (A.tile0 + it.vt * A.tile_step) * 2 * A.cta_v + in_tile;
      const bool live = q * 32 + lane < A.cta_v && v < A.V;
      const int ocol = A.compact ? it.vt * 2 * A.cta_v + in_tile : v;
      const uint32_t lanes = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
      // the accumulator is free again: one arrival per epilogue warp of either CTA at the leader's barrier
      auto give_back = [&]() {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_rank(smem_addr(&acc_empty[acc]), 0));
        if (++acc == nacc) { acc = 0; acc_phase ^= 1u; }
      };
      if constexpr (ADAPT) {
        if (it.b0 != places_of || it.n != places_n) {                  // other batch rows than the last item's: a trip to L2
          places_of = it.b0;
          places_n = it.n;
          adapted = D->nruns[it.b0 / A.item_n] > 0;
          __syncwarp();
          for (int c = half * 32; c < it.n; c += 64) lma_places[warp - EPI0][c / 64 * 32 + lane] = it.b0 + c + lane < A.B ? D->order[it.b0 + c + lane] : 0;
          __syncwarp();
        }
        auto finish = [&](float (&sum)[32], int c) {                   // the logits of 32 batch rows to their rows' places
          const int b0 = it.b0 + c, nb = min(32, A.B - b0);            // (uniform)
          if (adapted && live) {
#pragma unroll
            for (int j = 0; j < 32; j++) saw_nan |= sum[j] != sum[j] && j < nb;
          }
#pragma unroll
          for (int j = 0; j < 32; j++) {
            const int64_t to = lma_places[warp - EPI0][c / 64 * 32 + j];
            if (j < nb && live) __stcs(A.out_logits + to * A.ld_out + ocol, sum[j]);
            if (j % 8 == 7) asm volatile("" ::: "memory");             // (else 32 addresses at a time, and no registers left)
          }
        };
        constexpr int CHUNKS = LMH_MAX_N / 64;                         // of 32 batch rows that a warp has
        float sum[CHUNKS][32] = {};
        for (int kc = 0; kc < nkc && ok; kc = lma_next_sum(kc, nkc, D->units)) {                  // an item's sums, added up as they come
          if (!mbar_wait(smem_addr(&acc_full[acc]), acc_phase, abort_flag)) { ok = false; break; }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
          for (int ch = 0; ch < CHUNKS; ch++) {
            const int c = half * 32 + ch * 64;
            if (c >= it.n) break;                                      // (uniform)
            tmem_add16(lanes + acc * acc_cols + c, sum[ch]);
            tmem_add16(lanes + acc * acc_cols + c + 16, sum[ch] + 16);
          }
          give_back();
        }
        if (!ok) break;
#pragma unroll
        for (int ch = 0; ch < CHUNKS; ch++) {
          const int c = half * 32 + ch * 64;
          if (c < it.n) finish(sum[ch], c);
        }
        continue;
      }
      if (!mbar_wait(smem_addr(&acc_full[acc]), acc_phase, abort_flag)) { ok = false; break; }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
      for (int c = half * 32; c < it.n; c += 64) {
        uint32_t r[32];
        tmem_ld32(lanes + acc * acc_cols + c, r);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        const int b0 = it.b0 + c, nb = min(32, A.B - b0);              // batch rows of these columns (uniform)
        if (A.out_logits && live) {
          float* dst = A.out_logits + static_cast<int64_t>(b0) * A.ld_out + ocol;
          if (nb == 32) {
#pragma unroll
            for (int j = 0; j < 32; j++) __stcs(dst + j * A.ld_out, __uint_as_float(r[j]));
          } else {
#pragma unroll
            for (int j = 0; j < 32; j++) if (j < nb) __stcs(dst + j * A.ld_out, __uint_as_float(r[j]));
          }
        }
        if (A.thr) {
          // a batch row's threshold is the same for all lanes, and few lanes hold a logit that reaches it: those go to
          // the warp's stash, and from there, 32 at a time, to their rows' lists (an atomic on a row's count per
          // logit where it is found made every warp wait in nearly every chunk)
          stash_thr[warp - EPI0][lane] = (lane < nb) ? A.thr[b0 + lane] : INFINITY;
          __syncwarp();
          const float4* t4 = reinterpret_cast<const float4*>(stash_thr[warp - EPI0]);
          uint32_t m = 0u;                                             // columns of this lane that reach their threshold
#pragma unroll
          for (int j = 0; j < 32; j++) {
            const float4 t = t4[j >> 2];
            const float tj = (j & 3) == 0 ? t.x : (j & 3) == 1 ? t.y : (j & 3) == 2 ? t.z : t.w;
            m |= !(__uint_as_float(r[j]) < tj) ? (1u << j) : 0u;       // (true for a NaN)
          }
          if (!live) m = 0u;
          for (uint32_t votes; (votes = __ballot_sync(FULL, m != 0u)) != 0u;) {   // one hit of every lane that has any
            if (m) {
              const int j = __ffs(m) - 1;
              m &= m - 1;
              uint32_t x = r[0];
#pragma unroll
              for (int jj = 1; jj < 32; jj++) x = (j == jj) ? r[jj] : x;
              const int at = nstash + __popc(votes & ((1u << lane) - 1u));
              stash[warp - EPI0][at] = make_uint2(x, static_cast<uint32_t>(v));
              stash_row[warp - EPI0][at] = b0 + j;
            }
            nstash += __popc(votes);
            if (nstash >= 32) {                                        // uniform
              flush(32);
              nstash -= 32;
              const uint2 e = stash[warp - EPI0][32 + lane];
              const int er = stash_row[warp - EPI0][32 + lane];
              __syncwarp();
              if (lane < nstash) { stash[warp - EPI0][lane] = e; stash_row[warp - EPI0][lane] = er; }
            }
          }
          __syncwarp();
        }
      }
      give_back();
    }
    if (nstash > 0) flush(nstash);
    if constexpr (ADAPT) {                                              // the NaNs among what this warp wrote, once more
      if (__any_sync(FULL, saw_nan)) lma_second_look(A, *D);
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(LMA_REGS));   // (as the warps have that it meets again)
    }
  }
  // ---- teardown
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  if (abort_s) {
    // a wait ran out: give the copies and MMAs still in flight time to land before the shared and
    // tensor memory they target is given back (bounded: about a millisecond)
    for (int it = 0; it < 1000; it++) __nanosleep(1000);
    if (tid == 0) atomicOr_system(A.status, LMH_ERR_TIMEOUT);
  }
  // neither CTA leaves while the other may still arrive on its barriers or read its tiles
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(tmem_base), "r"(LMH_TMEM_COLS) : "memory");
  }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(LMH_NT, 1) lm_head_kernel(const __grid_constant__ LmHeadArgs A) {
  lm_head_run<false>(A, nullptr);
}
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(LMA_RUN_NT, 1) lm_head_adapters_kernel(const __grid_constant__ LmHeadArgs A, const __grid_constant__ LmAdaptArgs D) {
  lm_head_run<true>(A, &D);
}

// ---- fused sampling on top of the projection (greedy and top-k rows) --------------------------------
//
//   1. the projection over a sample of vocabulary tiles (1/32 of the vocabulary, spread over it)
//      gives each row 1024 to 4096 of its logits;
//   2. lmh_threshold_kernel: the r-th largest of that sample, r chosen so that eight times top_k
//      logits of the whole row (at least 256, at most a third of the list) are expected above it: an
//      estimate, not a bound;
//   3. the projection over all tiles: the epilogue appends every logit at or above the row's
//      threshold to the row's candidate list (no [B, V] logits are written);
//   4. lmh_finish_kernel: the exact top_k-th largest of the candidates with ties kept
//      (model/generate.go:157-164), then softmax / top-p / draw on the kept set exactly as the
//      one-GPU narrow kernel does. A row whose estimate failed (fewer than top_k candidates, or more
//      than the list holds) or whose config the fused path does not serve is counted in nfail; the
//      host then recomputes the batch through the unfused path.
constexpr int LMH_SAMPLE_MIN = 1024, LMH_SAMPLE_MAX = 4096;   // logits of a row's sample
constexpr int LMH_F_NT = 256;
constexpr int LMH_F_DYN_BYTES = LMH_CAND_CAP * 8 + 16384 + KEEP_MAX * 8;

struct LmhSampleArgs {
  KernelArgs k;             // V, cfgs, uniforms, out_ids, out_flags, exp_table (logits unused)
  const float* sample;      // [B, nsample] logits of the sampled tiles
  int32_t nsample;
  int32_t fuse_top_k;       // rows with 0 < top_k <= fuse_top_k (or temperature 0) are served
  float* thr;               // [B]
  const uint2* cand;        // [B, LMH_CAND_CAP]
  LmhRow* rows;             // [B]
  int32_t* nfail;           // [1], in host memory
  int64_t B;
};

__device__ __forceinline__ bool lmh_row_served(const RowCfg& c, int V, int fuse_top_k) {
  const float T = c.temperature;
  if (T == 0.0f) return true;
  if (!(T > 0.0f) || !(T < INFINITY)) return true;            // reported as a bad config by the finish kernel
  const int topk = (c.top_k > 0 && c.top_k < V) ? c.top_k : 0;
  return topk > 0 && topk <= fuse_top_k;
}

__global__ void __launch_bounds__(LMH_F_NT) lmh_threshold_kernel(const __grid_constant__ LmhSampleArgs M) {
  constexpr int PER = LMH_SAMPLE_MAX / LMH_F_NT;              // sample logits per thread
  __shared__ bu::Scratch sc;
  __shared__ uint32_t cnts[1024];
  __shared__ int bc[4];
  const int tid = threadIdx.x;
  pdl_launch();
  const int64_t row = blockIdx.x;
  const RowCfg cfg = M.k.cfgs[row];
  const bool served = lmh_row_served(cfg, M.k.V, M.fuse_top_k);
  pdl_wait();                                                 // the sample's logits
  float thr = served ? -INFINITY : INFINITY;                  // -Inf: a sample too small to say, everything is a candidate
  if (served) {
    const int keff = (cfg.temperature == 0.0f || !(cfg.temperature > 0.0f) || !(cfg.temperature < INFINITY)) ? 1 : cfg.top_k;
    const int n = M.nsample;
    uint32_t key[PER], tmin = 0xffffffffu, tmax = 0u;
#pragma unroll
    for (int j = 0; j < PER; j++) {
      const int i = j * LMH_F_NT + tid;
      key[j] = (i < n) ? okey(M.sample[row * n + i]) : 0u;    // (0, a NaN's key, is below every other)
      tmin = min(tmin, key[j]);
      tmax = max(tmax, key[j]);
    }
    // expected logits of the whole row above the threshold: eight times top_k, at least 256, at most a
    // third of the list; the r-th largest of the sample stands for the (r V / n)-th largest of the row
    const long long want = min(max(8ll * keff, 256ll), static_cast<long long>(LMH_CAND_CAP / 3));
    const int r = max(2, static_cast<int>((want * n + M.k.V / 2) / M.k.V));
    if (r < n) {
      const uint32_t lo = sample_threshold<LMH_F_NT, 1024>([&](auto&& g) {
#pragma unroll
        for (int j = 0; j < PER; j++) g(key[j]);
      }, r, tmin, tmax, cnts, bc, sc, tid);
      if (lo > 0x007fffffu) thr = okey_to_float(lo);          // NaNs order lowest: a NaN threshold would collect nothing
    }
  }
  if (tid == 0) { M.thr[row] = thr; M.rows[row].cnt = 0; M.rows[row].nan = 0; }
}

__global__ void __launch_bounds__(LMH_F_NT, 4) lmh_finish_kernel(const __grid_constant__ LmhSampleArgs M) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ bu::Scratch sc;
  __shared__ uint32_t s_sel[256];
  __shared__ int s_bc[4];
  __shared__ int s_cnt;
  uint2* list = reinterpret_cast<uint2*>(dyn);                                       // the row's candidates
  unsigned char* work = dyn + LMH_CAND_CAP * 8;                                       // for finish_small_set
  uint2* kept = reinterpret_cast<uint2*>(dyn + LMH_CAND_CAP * 8 + 16384);            // KEEP_MAX entries
  const KernelArgs& A = M.k;
  const int tid = threadIdx.x;
  constexpr int NW = LMH_F_NT / 32;
  pdl_wait();                                                 // the candidates
  for (int64_t row = blockIdx.x; row < M.B; row += gridDim.x) {
    __syncthreads();
    const RowCfg cfg = A.cfgs[row];
    const float Tm = cfg.temperature;
    auto write_row = [&](int id, uint32_t fl) {
      if (tid == 0) {
        A.out_ids[row] = id;
        if (A.out_flags) A.out_flags[row] = fl;
      }
    };
    auto give_up = [&]() { if (tid == 0) atomicAdd_system(M.nfail, 1); write_row(-1, FLAG_INTERNAL); };
    if (!lmh_row_served(cfg, A.V, M.fuse_top_k)) { give_up(); continue; }
    if (Tm != 0.0f && (!(Tm > 0.0f) || !(Tm < INFINITY))) { write_row(-1, FLAG_BAD_CFG); continue; }
    const int cnt = M.rows[row].cnt, nanb = M.rows[row].nan;
    uint32_t kmax = 0x007fffffu;                                // -Inf
    for (int j = tid; j < min(cnt, LMH_CAND_CAP); j += LMH_F_NT) {
      const uint2 e = M.cand[row * LMH_CAND_CAP + j];
      list[j] = e;
      kmax = max(kmax, okey(__uint_as_float(e.x)));
    }
    kmax = static_cast<uint32_t>(bu::max_u64<NW>(kmax, sc, tid));   // (its barriers publish the list)
    const int keff = (Tm == 0.0f) ? 1 : cfg.top_k;
    if (cnt > LMH_CAND_CAP || (cnt < keff && !(nanb & 1))) { give_up(); continue; }   // the estimate failed for this row
    // ---- greedy (generate.go:134-144): largest logit, lowest index; a NaN at index 0 is never beaten
    if (Tm == 0.0f) {
      unsigned long long best = 0ull;
      for (int j = tid; j < cnt; j += LMH_F_NT) {
        const unsigned long long p = (static_cast<unsigned long long>(okey(__uint_as_float(list[j].x))) << 32) |
                                     static_cast<uint32_t>(~list[j].y);
        best = p > best ? p : best;
      }
      best = bu::max_u64<NW>(best, sc, tid);
      int id = static_cast<int>(~static_cast<uint32_t>(best & 0xffffffffull));
      if ((nanb & 2) || cnt == 0) id = 0;
      write_row(id, 0u);
      continue;
    }
    const float m = scale_t(okey_to_float(kmax), Tm);
    // A NaN anywhere, or an infinite maximum: the walk of generate.go:231-239 falls through
    if ((nanb & 1) || !(fabsf(m) < INFINITY)) { write_row(A.V - 1, FLAG_NONFINITE | FLAG_FALLBACK); continue; }
    // ---- top_k-th largest with ties (generate.go:157-164), then the kept set
    const int topk = cfg.top_k;
    const int nk = narrow_list<LMH_F_NT>(list, cnt, topk, Tm, 0u, kmax, kept, s_sel, s_bc, &s_cnt, tid);
    if (nk > KEEP_MAX || cnt <= topk) { give_up(); continue; }
    const bool topp_on = (cfg.top_p > 0.0f && cfg.top_p < 1.0f);
    const int mode = cfg.topp_mode;
    const double plim = (mode == 0) ? static_cast<double>(cfg.top_p) * 1.5 : static_cast<double>(cfg.top_p);
    // Everything at or above the exact threshold must be on the list: that holds when the exact
    // threshold (the floor of the k-th value's class of equal quotients) is not below the list's own.
    if (!finish_small_set<LMH_F_NT, false>(A, row, kept, nk, topk, m, Tm, topp_on, mode, plim, A.uniforms[row], M.thr[row], work, nullptr, 0u))
      give_up();
  }
}

}  // namespace gs
