// rel_attention.hip -- attention with a learned relative position bias, forward and backward, for gfx950.
//
//   s_ij = scale q_i.k_j + table[bucket(j - p_i)][head],  p_i = i + query_offset,  o_i = softmax(s_i) V
// over the keys that query i sees; scores, probabilities and the bias matrix never leave the chip.  The reference
// (modeling_t5.py's attention) materialises the (b, h, nq, nk) bias, scores and probabilities.
//
// What a query sees is always ONE interval [lo, hi) of keys -- key lengths, causal and prefix masks and packed documents are
// all intervals -- so masks cost two integers a row, and whole tiles are classified by four: outside (skipped), inside
// (no mask code), or cut.
//
// The bias is a function of the distance alone and constant from `reach` on: a workgroup keeps log2(e) * bias for the
// 2 reach + 1 distances in LDS; tiles wholly beyond `reach` add one constant, the few along the diagonal gather.
//
// Statistics, accumulators, the running maximum and sum are f32.  P and dS are rounded to the operand type where they become
// an operand of the next product (bf16 / f16 matrix instructions take nothing else; f32 stays f32).  f16 has no exponents to
// spare for that -- P is 1 / nk on average, gradients are small -- so its backward pass holds 2^8 P and dS times the power of
// two that brings the largest |dO| (of the query for dQ, of the queries that see a key for dK) to [4, 8), and takes both back out
// of the f32 sums.  |dS| may be as large as 2 |dO|_1 max |V|: where that power is too much for f16 (65504) it is lowered.  For dQ
// when a block's dS reaches DS_MOST -- like the running maximum, a branch seldom taken (16 heads of 128 on 4, 2 x 4096 packed
// tokens: 156 us without it, 158 with it); for dK beforehand, by the largest |dS| that the dQ kernel has met (a branch there as
// well: 245 us instead of 200).  (It is not raised for small V: below 2^-10 or so, dS of many keys comes near f16's subnormals, where
// its error is 2^-27 of the largest |dO| whatever its own size.)
#include "lang_core.h"

#include <limits.h>

#include <algorithm>

namespace {
using namespace lang;

struct Params {
  const void *q, *k, *v, *table, *grad;
  const int *key_lengths, *prefix_lengths, *key_ranges;
  void *out, *dq, *dk, *dv, *dtable;
  float *out32, *lse, *hist;
  float2 *stat;                               // backward: lse, delta of a query and head
  int2 *rows;                                 // backward: first key and number of keys that a query sees
  float *part;                                // backward: dK, dV of every split, (2, splits, b, nk, hkv, d), or NULL: one split
  float *piece, *piece_ml;                    // one output, maximum and sum (forward), one dQ for every key split, or NULL
  int4 *blocks;                               // backward: interval summary of every 32 queries
  int *tops;                                  // backward, f16: by how much a head's 32 queries let dS be raised for dK (see dQ)
  long q_b, q_n, q_h, k_b, k_n, k_h, v_b, v_n, v_h, grad_b, grad_n, grad_h;
  int b, nq, nk, h, hkv, group, causal, offset, table_rows, qtiles, ktiles, head_splits, query_splits, key_splits;
  float scale;
  Buckets bk;
};

// The keys [lo, hi) that query i of sequence b sees; lo = hi = 0 for none.
__device__ __forceinline__ void interval(const Params &p, int b, int i, int &lo, int &hi) {
  lo = 0;
  hi = p.nk;
  if (p.key_lengths) hi = min(hi, p.key_lengths[b]);
  if (p.causal) {
    long seen = (long)i + p.offset + 1;
    if (p.prefix_lengths) seen = max(seen, (long)p.prefix_lengths[b]);
    hi = (int)min((long)hi, seen);
  }
  if (p.key_ranges) {
    const int2 r = reinterpret_cast<const int2 *>(p.key_ranges)[(long)b * p.nq + i];
    lo = max(lo, r.x);
    hi = min(hi, r.y);
  }
  if (lo >= hi) lo = hi = 0;
}

// What 32 queries see together: any = the union's ends, all = the interval that every one of them sees whole.
struct Span { int any_lo, any_hi, all_lo, all_hi; };
__device__ __forceinline__ Span span_of(int lo, int hi, bool valid) {
  Span s;
  s.any_lo = wave_min_i32(valid && lo < hi ? lo : INT_MAX);
  s.any_hi = wave_max_i32(valid && lo < hi ? hi : 0);
  s.all_lo = wave_max_i32(valid ? lo : 0);
  s.all_hi = wave_min_i32(valid ? hi : INT_MAX);
  return s;
}

// [lo, hi) -> its part `split` of `splits`, in whole tiles
template <int KT> __device__ __forceinline__ void cut_piece(int &lo, int &hi, int split, int splits) {
  if (lo >= hi) return;
  const int first = lo / KT, tiles = (hi + KT - 1) / KT - first, share = (tiles + splits - 1) / splits;
  lo = max(lo, (first + split * share) * KT);
  hi = min(hi, (first + (split + 1) * share) * KT);
  if (lo >= hi) hi = 0;                        // nothing left: the loop over [lo, hi) starts at 0
}

// Consecutive workgroups go to the 8 XCDs in turn; give each XCD a contiguous share of the work instead, so that the
// workgroups that read the same keys share an L2.
__device__ __forceinline__ int xcd_contiguous(int id, int total) {
  const int each = total >> 3;
  return id < each * 8 ? (id & 7) * each + (id >> 3) : id;
}

// Rows [row0, row0 + ROWS) of a token-major operand through registers into an LDS tile; rows outside [lo, hi) become zero.  Their
// loads repeat the nearest row inside (no branch: a load under a condition is waited for at once, and the next tile's loads
// are to be in flight while this one is used); `store` clears them, which only tiles at an end pay for.
template <typename T, int D, int ROWS, int NT> struct Stage {
  typedef Tile<T, D> TL;
  static constexpr int N = (ROWS * TL::CH + NT - 1) / NT;
  u32x4 r[N];
  __device__ __forceinline__ void load(const T *base, long stride, int row0, int lo, int hi, int tid) {
    const char *tile = reinterpret_cast<const char *>(base + (long)row0 * stride);      // one scalar address, 32-bit offsets
    const int first = max(lo - row0, 0), last = min(hi - 1 - row0, ROWS - 1);
    const unsigned pitch = (unsigned)stride * (unsigned)sizeof(T);                       // below 2^24: the host looks
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = tid + i * NT, row = c / TL::CH, ch = c - row * TL::CH;
      r[i] = *reinterpret_cast<const u32x4 *>(tile + (__umul24((unsigned)min(max(row, first), last), pitch) + (unsigned)ch * 16u));
    }
  }
  __device__ __forceinline__ void store(char *tile, int row0, int lo, int hi, int tid) {
    const bool whole = row0 >= lo && row0 + ROWS <= hi;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = tid + i * NT, row = c / TL::CH, ch = c - row * TL::CH;
      if (!whole && (row0 + row < lo || row0 + row >= hi)) r[i] = u32x4{0, 0, 0, 0};
      if (ROWS * TL::CH % NT == 0 || row < ROWS) *reinterpret_cast<u32x4 *>(tile + TL::at(row, ch)) = r[i];
    }
  }
};

// fragment f of a stationary row: elements 16 f + 8 half .. + 7  (rows that do not exist repeat the last one: a lane that has
// one takes part in nothing but its own column)
template <typename T, int D>
__device__ __forceinline__ void load_row(frag_t<T> (&f)[D / 16], const T *row, int half) {
#pragma unroll
  for (int s = 0; s < D / 16; ++s) f[s] = *reinterpret_cast<const frag_t<T> *>(row + 16 * s + 8 * half);
}

// A (D x 32) accumulator whose columns are rows of a dense tensor: registers 4 g .. 4 g + 3 are four consecutive elements.
template <typename T, int D>
__device__ __forceinline__ void store_row(T *row, const f32x16 (&acc)[D / 32], float factor, int half) {
#pragma unroll
  for (int blk = 0; blk < D / 32; ++blk)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = acc[blk][4 * g + e] * factor;
      *reinterpret_cast<vec4_t<T> *>(row + 32 * blk + 8 * g + 4 * half) = to_vec4<T>(x);
    }
}

template <typename T> constexpr bool narrow() { return std::is_same<T, _Float16>::value; }
constexpr float SLACK = 8.f;                  // of the forward pass's reference value (see there)
constexpr int P_UP = 8, DS_UP = 3;            // f16: exponents that P and dS are raised by (see the top)
// f16: from DS_MOST on, a query's dS is brought back to [2^(DS_KEEP - 1), 2^DS_KEEP): half a subnormal step is then at most 2^-36
// of its largest.  For dK the largest of all is below 2^DS_TOP (dP and delta are summed in another order there: an error of 2^9 at
// most where |dO| < 8, |V| <= 65504 and d = 128, which 65504 still holds).
constexpr float DS_MOST = 32768.f;
constexpr int DS_KEEP = 12, DS_TOP = 14;
// exponents by which dS of a query whose largest one is `top` has to go down (an infinite one stays where it is)
__device__ __forceinline__ int too_much(float top) {
  return top >= DS_MOST && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - DS_KEEP : 0;
}

template <typename T> constexpr int key_tile() { return sizeof(T) == 2 ? 64 : 32; }
// keys of a tile of the dQ kernel: 32 leave LDS and registers for two workgroups a CU where a row is long
template <typename T> constexpr int dq_tile(int d) { return sizeof(T) == 2 && d == 64 ? 64 : 32; }
// queries of a tile of the dK / dV kernel, likewise (at 128 wide K, V and both sums fill a SIMD with one wave anyway)
template <typename T> constexpr int dkv_tile(int d) { return sizeof(T) == 2 && d != 96 ? 64 : 32; }
// At 96 wide that kernel's K rows stay in LDS: with V and both sums they are more than two waves' registers (2 x 4096 packed bf16
// tokens, 16 heads on 4: 160 us instead of 170; at 128 wide they would be 37 registers over even so, and 250 us instead of 197).
template <typename T> constexpr bool dkv_keys_in_lds(int d) { return sizeof(T) == 2 && d == 96; }

// s (scaled scores of a 32 x 32 block, in log2 units) += bias.  first = position of register 0's row minus that of the lane's
// column, i.e. register r stands at relative position first + sign * (16 (r >> 3) + (r & 7)).
template <int SIGN>
__device__ __forceinline__ void add_bias(f32x16 &s, const float *by_distance, int reach, int first) {
  const float *b = by_distance + first + reach + EDGE;
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] += b[SIGN * (16 * (r >> 3) + (r & 7))];
}

// Where a block of keys [k0, k0 + n) stands for queries at positions [p0, p0 + 32): wholly behind or ahead of `reach`, or near.
enum Where { NEAR, BEHIND, AHEAD };
__device__ __forceinline__ Where where(int k0, int n, int p0, int reach) {
  return k0 + n - 1 - p0 <= -reach ? BEHIND : k0 - (p0 + 31) >= reach ? AHEAD : NEAR;
}

// ---- forward -------------------------------------------------------------------------------------------------------------
// A wave owns 32 queries (columns), a workgroup NW waves that share the streamed key tiles in a double-buffered LDS pair:
// the next tile's loads are in flight while the current one is used, one barrier a tile.
// S^T = K Q^T, then O^T = V^T P^T: a query is one lane (and lane ^ 32), its softmax is in-lane work.
// TWO: 16-bit P goes into its product as the sum of two parts, rounded and rest.  Where a backward pass follows: the unrounded
// output's use is delta, and a row of dS sums to 0 only as far as delta agrees with the P of the backward pass, which is not
// rounded (with one part the table's gradient of 4 x 432 bf16 tokens, 32 heads, was off by 0.0027 of its size, most of it in the
// buckets that hold most of a row; the rounding of the result itself is 0.0017).  And where the launch is small enough for latency
// to decide (see launch_fwd).
template <typename T, int D, int NW, bool TWO>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 4 ? (D == 128 ? 1 : 2) : D == 64 ? 3 : 2) void rel_fwd_kernel(const Params p) {
  typedef Tile<T, D> TL;
  constexpr int KT = key_tile<T>(), NT = NW * 64, SUB = KT / 32, TB = KT * TL::ROW;
  extern __shared__ __align__(16) char lds[];
  float *bias = reinterpret_cast<float *>(lds + 4 * TB);
  __shared__ int ends[2][NW];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
  const int id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int split = id % p.key_splits, item = id / p.key_splits;
  const int bh = item / p.qtiles, qt = p.qtiles - 1 - item % p.qtiles;      // causal: the long rows first
  const int b = bh / p.h, head = bh - b * p.h;
  BiasFill<T> fill;
  fill.start(p.bk, p.table, p.h, head, tid);
  const int qi = (qt * NW + wave) * 32 + col;
  const bool valid = qi < p.nq;
  int lo = 0, hi = 0;
  if (valid) interval(p, b, qi, lo, hi);
  const Span sp = span_of(lo, hi, valid);
  if (lane == 0) {
    ends[0][wave] = sp.any_lo;
    ends[1][wave] = sp.any_hi;
  }
  __syncthreads();
  int wlo = INT_MAX, whi = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    wlo = min(wlo, ends[0][w]);
    whi = max(whi, ends[1][w]);
  }
  if (p.key_splits > 1) cut_piece<KT>(wlo, whi, split, p.key_splits);
  const int kvh = head / p.group;
  const T *kb = reinterpret_cast<const T *>(p.k) + b * p.k_b + kvh * p.k_h;
  const T *vb = reinterpret_cast<const T *>(p.v) + b * p.v_b + kvh * p.v_h;
  const float scale2 = p.scale * LOG2E;
  const int reach = p.bk.reach, qpos = qi + p.offset, q0pos = (qt * NW + wave) * 32 + p.offset;
  const int first = wlo < whi ? wlo / KT * KT : 0;
  Stage<T, D, KT, NT> ks, vs;
  if (wlo < whi) {
    ks.load(kb, p.k_n, first, wlo, whi, tid);
    vs.load(vb, p.v_n, first, wlo, whi, tid);
  }
  frag_t<T> qf[D / 16];
  load_row<T, D>(qf, reinterpret_cast<const T *>(p.q) + b * p.q_b + (long)min(qi, p.nq - 1) * p.q_n + head * p.q_h, half);
  fill.finish(bias, p.bk, p.table, p.h, head, tid, NT);
  if (wlo < whi) {
    ks.store(lds, first, wlo, whi, tid);
    vs.store(lds + TB, first, wlo, whi, tid);
  }
  f32x16 o[D / 32] = {};
  float m = -INFINITY, l = 0.f;
  __syncthreads();
  const bool biased = p.bk.n > 0;
  const float bias_behind = biased ? bias[0] : 0.f, bias_ahead = biased ? bias[2 * (reach + EDGE)] : 0.f;
  loads_done();
  int buf = 0;
  for (int t = first; t < whi; t += KT, buf ^= 1) {
    const bool more = t + KT < whi;
    if (more) {
      ks.load(kb, p.k_n, t + KT, wlo, whi, tid);
      vs.load(vb, p.v_n, t + KT, wlo, whi, tid);
    }
    if (t < sp.any_hi && t + KT > sp.any_lo) {
      const char *kt = lds + buf * 2 * TB, *vt = kt + TB;
      f32x16 s[SUB];
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        s[u] = f32x16{};
#pragma unroll
        for (int f = 0; f < D / 16; ++f)
          s[u] = mma32(TL::row_frag(kt, u * 32 + kappa(col), 2 * f + half), qf[f], s[u]);
      }
      float add = 0.f;
      bool plain = scale2 >= 0.f && t >= sp.all_lo && t + KT <= sp.all_hi;      // no mask, no bias but one: nothing per element
      if (biased) {
        const Where w = where(t, KT, q0pos, reach);
        if (w == NEAR) plain = false;
        else add = w == BEHIND ? bias_behind : bias_ahead;
        if (!plain) {
#pragma unroll
          for (int u = 0; u < SUB; ++u) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[u][r] = __builtin_fmaf(s[u][r], scale2, add);
            if (w == NEAR) add_bias<1>(s[u], bias, reach, t + u * 32 + 8 * half - qpos);
          }
        }
      } else if (!plain) {
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[u][r] *= scale2;
      }
      if (t < sp.all_lo || t + KT > sp.all_hi) {
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if ((unsigned)(t + u * 32 + reg_row(r, half) - lo) >= (unsigned)(hi - lo)) s[u][r] = -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
      if (plain) top = __builtin_fmaf(top, scale2, add);
      // The reference value m follows the running maximum only when a score passes it by 2^SLACK: exponentials up to that are as
      // good as up to 1 (f32 sums; a rounding is relative), and rescaling the output costs as much as a third of a tile.
      if (__any(top > m + SLACK)) {
        const float now = fmaxf(m, max_halves(top));
        const float keep = now == -INFINITY ? 1.f : exp2_(m - now);
        m = now;
        l *= keep;
#pragma unroll
        for (int blk = 0; blk < D / 32; ++blk)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[blk][r] *= keep;
      }
      const float base = m == -INFINITY ? 0.f : m;
      const float factor = plain ? scale2 : 1.f, offset = plain ? add - base : -base;
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[u][r] = exp2_(__builtin_fmaf(s[u][r], factor, offset));
          l += s[u][r];
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          f32x8 x;
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = s[u][8 * g + j];
          const frag_t<T> pf = to_frag<T>(x);
          frag_t<T> rest;
          if constexpr (TWO) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] -= (float)pf[j];
            rest = to_frag<T>(x);
          }
#pragma unroll
          for (int blk = 0; blk < D / 32; ++blk) {
            const frag_t<T> vf = TL::col_frag(vt, u * 32 + 16 * g + 8 * half, 32 * blk + (lane & 16), lane);
            o[blk] = mma32(vf, pf, o[blk]);
            if constexpr (TWO) o[blk] = mma32(vf, rest, o[blk]);
          }
        }
      }
    }
    if (more) {
      ks.store(lds + (buf ^ 1) * 2 * TB, t + KT, wlo, whi, tid);
      vs.store(lds + (buf ^ 1) * 2 * TB + TB, t + KT, wlo, whi, tid);
    }
    __syncthreads();
  }
  if (!valid) return;
  l = sum_halves(l);
  const bool empty = lo >= hi || (m == -INFINITY && l == 0.f);              // nothing seen, or every bias -inf
  const float inv = empty ? 0.f : 1.f / l;
  const long row = (((long)b * p.nq + qi) * p.h + head) * D;
  if (p.piece) {
    store_row<float, D>(p.piece + split * ((long)p.b * p.nq * p.h * D) + row, o, 1.f, half);
    if (half == 0)
      reinterpret_cast<float2 *>(p.piece_ml)[(split * (long)p.b * p.h + bh) * p.nq + qi] = make_float2(m, l);
    return;
  }
  store_row<T, D>(reinterpret_cast<T *>(p.out) + row, o, inv, half);
  if (p.out32) {
    store_row<float, D>(p.out32 + row, o, inv, half);
    if (half == 0) p.lse[((long)b * p.h + head) * p.nq + qi] = empty ? INFINITY : m + __builtin_amdgcn_logf(l);
  }
}

// Joins the key splits of a row in their order: D / 4 lanes a row (query, head).
template <typename T, int D>
__global__ __launch_bounds__(256) void rel_join_kernel(const Params p) {
  constexpr int PER = D / 4, ROWS = 256 / PER;
  const int e = threadIdx.x % PER;
  const long row = (long)blockIdx.x * ROWS + threadIdx.x / PER, rows = (long)p.b * p.nq * p.h;      // (b, nq, h)
  if (threadIdx.x / PER >= ROWS || row >= rows) return;
  const int head = (int)(row % p.h);
  const long at = row / p.h, stat = (at / p.nq * p.h + head) * p.nq + at % p.nq;                    // (b, h, nq)
  const float2 *ml = reinterpret_cast<const float2 *>(p.piece_ml) + stat;
  float top = -INFINITY, sum = 0.f;
  for (int s = 0; s < p.key_splits; ++s) top = fmaxf(top, ml[s * rows].x);
  const float base = top == -INFINITY ? 0.f : top;
  f32x4 x = {};
#pragma unroll 4
  for (int s = 0; s < p.key_splits; ++s) {
    const float2 v = ml[s * rows];
    const float keep = exp2_(v.x - base);
    const f32x4 y = *reinterpret_cast<const f32x4 *>(p.piece + (s * rows + row) * D + 4 * e);
    sum = __builtin_fmaf(v.y, keep, sum);
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = __builtin_fmaf(y[q], keep, x[q]);
  }
  const bool empty = top == -INFINITY && sum == 0.f;
  const float inv = empty ? 0.f : 1.f / sum;
#pragma unroll
  for (int q = 0; q < 4; ++q) x[q] *= inv;
  reinterpret_cast<vec4_t<T> *>(p.out)[row * PER + e] = to_vec4<T>(x);
  if (p.out32) {
    reinterpret_cast<f32x4 *>(p.out32)[row * PER + e] = x;
    if (e == 0) p.lse[stat] = empty ? INFINITY : top + __builtin_amdgcn_logf(sum);
  }
}

// ---- backward: dQ, delta, the table's gradient ------------------------------------------------------------------------------
// Same tiling as the forward pass (a query is a lane): P = exp2(s - lse), dP^T = V dO^T, dS = P (dP - delta) with
// delta = dO.O from the unrounded O, dQ^T = K^T dS^T.
// Table: dS summed by distance.  Beyond `reach` everything falls into the end buckets: two registers.  A 32 x 32 block along
// the diagonal goes through wave-private LDS, one row of 36 floats a distance, element (query i, key j) at [j - i + 31][i]: the
// addresses are a lane's base plus constants, and lane l then adds row l and puts the sum to its distance -- 64 distances, 64
// lanes, no two meet and the order of the sums is fixed.  (Adding every element to its distance by an LDS atomic cost 200
// address and mask instructions and twice the LDS time: 88 us instead of 32 for 4 x 32 heads of 432 tokens.)
constexpr int DIAG_ROW = 36, DIAG = 64 * DIAG_ROW;        // floats; 36: 16-byte rows whose columns spread over the banks
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 4 ? 1 : 2) void rel_bwd_dq_kernel(const Params p) {
  typedef Tile<T, D> TL;
  constexpr int KT = dq_tile<T>(D), NT = NW * 64, SUB = KT / 32, TB = KT * TL::ROW;
  extern __shared__ __align__(16) char lds[];
  float *bias = reinterpret_cast<float *>(lds + 4 * TB);
  const int reach = p.bk.reach, span = bias_floats(reach);
  float *sums = bias + (span + 3) / 4 * 4;                // [NW][span]
  __shared__ int ends[2][NW];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
  const int id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int split = id % p.key_splits, item = id / p.key_splits;
  const int bh = item / p.qtiles, qt = p.qtiles - 1 - item % p.qtiles;
  const int b = bh / p.h, head = bh - b * p.h;
  BiasFill<T> fill;
  fill.start(p.bk, p.table, p.h, head, tid);
  const int qi = (qt * NW + wave) * 32 + col;
  const bool valid = qi < p.nq;
  int lo = 0, hi = 0;
  if (valid) interval(p, b, qi, lo, hi);
  const Span sp = span_of(lo, hi, valid);
  if (lane == 0) {
    ends[0][wave] = sp.any_lo;
    ends[1][wave] = sp.any_hi;
    if (head == 0 && split == 0) p.blocks[((long)b * p.qtiles + qt) * NW + wave] = make_int4(sp.any_lo, sp.any_hi, sp.all_lo, sp.all_hi);
  }
  __syncthreads();
  int wlo = INT_MAX, whi = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    wlo = min(wlo, ends[0][w]);
    whi = max(whi, ends[1][w]);
  }
  if (p.key_splits > 1) cut_piece<KT>(wlo, whi, split, p.key_splits);
  const int kvh = head / p.group;
  const T *kb = reinterpret_cast<const T *>(p.k) + b * p.k_b + kvh * p.k_h;
  const T *vb = reinterpret_cast<const T *>(p.v) + b * p.v_b + kvh * p.v_h;
  const int first = wlo < whi ? wlo / KT * KT : 0;
  Stage<T, D, KT, NT> ks, vs;
  if (wlo < whi) {
    ks.load(kb, p.k_n, first, wlo, whi, tid);
    vs.load(vb, p.v_n, first, wlo, whi, tid);
  }
  frag_t<T> qf[D / 16], gf[D / 16];
  const int qrow = min(qi, p.nq - 1);
  load_row<T, D>(qf, reinterpret_cast<const T *>(p.q) + b * p.q_b + (long)qrow * p.q_n + head * p.q_h, half);
  load_row<T, D>(gf, reinterpret_cast<const T *>(p.grad) + b * p.grad_b + (long)qrow * p.grad_n + head * p.grad_h, half);
  const long row = (((long)b * p.nq + qrow) * p.h + head) * D, stat = ((long)b * p.h + head) * p.nq + qrow;
  float delta = 0.f, lse = p.lse[stat];
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    const f32x8 x = *reinterpret_cast<const f32x8 *>(p.out32 + row + 16 * s + 8 * half);
#pragma unroll
    for (int j = 0; j < 8; ++j) delta = __builtin_fmaf((float)gf[s][j], x[j], delta);
  }
  delta = sum_halves(delta);
  if (valid && half == 0 && split == 0) {
    p.stat[stat] = make_float2(lse, delta);
    if (head == 0) p.rows[(long)b * p.nq + qi] = make_int2(lo, hi - lo);
  }
  if (!valid) lse = INFINITY;
  float undo = 1.f;                                       // dS is held times 1 / undo
  float peak = 0.f;                                       // f16: the largest |dS|, as held
  int grads = -64;                                        // f16: exponent of the largest |dO|; -64: none
  if constexpr (narrow<T>()) {
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf((float)gf[s][j]));
    top = max_halves(top);
    const bool plain = !(top > 0.f && top < INFINITY);
    const int e = plain ? DS_UP : __builtin_amdgcn_frexp_expf(top);      // top in [2^(e-1), 2^e)
    undo = __builtin_ldexpf(1.f, e - DS_UP);
    if (!plain && lse < INFINITY) grads = e;              // (a query that sees nothing has no gradient, whatever its dO is)
    lse += (float)(e - DS_UP);
  }
  const bool biased = p.bk.n > 0;
  if (biased) {
    fill.finish(bias, p.bk, p.table, p.h, head, tid, NT);
    for (int i = tid; i < NW * ((span + 3) / 4 + DIAG / 4); i += NT) reinterpret_cast<f32x4 *>(sums)[i] = f32x4{};
  }
  if (wlo < whi) {
    ks.store(lds, first, wlo, whi, tid);
    vs.store(lds + TB, first, wlo, whi, tid);
  }
  const float scale2 = p.scale * LOG2E;
  const int qpos = qi + p.offset, q0pos = (qt * NW + wave) * 32 + p.offset;
  float *mine = sums + wave * ((span + 3) / 4 * 4), *diag = sums + NW * ((span + 3) / 4 * 4) + wave * DIAG;
  // element of register 0: key 8 half, query col; lane l reads distance l - 31
  float *const diag_put = diag + (8 * half - col + 31) * DIAG_ROW + col, *const diag_get = diag + lane * DIAG_ROW;
  f32x16 dq[D / 32] = {};
  float behind = 0.f, ahead = 0.f;
  __syncthreads();
  const float bias_behind = biased ? bias[0] : 0.f, bias_ahead = biased ? bias[2 * (reach + EDGE)] : 0.f;
  loads_done();
  int buf = 0;
  for (int t = first; t < whi; t += KT, buf ^= 1) {
    const bool more = t + KT < whi;
    if (more) {
      ks.load(kb, p.k_n, t + KT, wlo, whi, tid);
      vs.load(vb, p.v_n, t + KT, wlo, whi, tid);
    }
    if (t < sp.any_hi && t + KT > sp.any_lo) {
      const char *kt = lds + buf * 2 * TB, *vt = kt + TB;
      const bool cut = t < sp.all_lo || t + KT > sp.all_hi;
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        f32x16 s{}, dp{};
#pragma unroll
        for (int f = 0; f < D / 16; ++f) {
          s = mma32(TL::row_frag(kt, u * 32 + kappa(col), 2 * f + half), qf[f], s);
          dp = mma32(TL::row_frag(vt, u * 32 + kappa(col), 2 * f + half), gf[f], dp);
        }
        const Where w = biased ? where(t + u * 32, 32, q0pos, reach) : BEHIND;
        const int rel0 = t + u * 32 + 8 * half - qpos;
        if (w == NEAR) {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], scale2, -lse);
          add_bias<1>(s, bias, reach, rel0);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = exp2_(s[r]) * (dp[r] - delta);
        } else {
          const float add = (w == BEHIND ? bias_behind : bias_ahead) - lse;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = exp2_(__builtin_fmaf(s[r], scale2, add)) * (dp[r] - delta);
        }
        if (cut) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if ((unsigned)(t + u * 32 + reg_row(r, half) - lo) >= (unsigned)(hi - lo)) s[r] = 0.f;
        }
        if constexpr (narrow<T>()) {
          float top = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(s[r]));
          peak = fmaxf(peak, top);
          if (__any(top >= DS_MOST)) {
            const int down = too_much(max_halves(top));
            const float keep = __builtin_ldexpf(1.f, -down);
            peak *= keep;
            undo = __builtin_ldexpf(undo, down);
            lse += (float)down;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= keep;
#pragma unroll
            for (int blk = 0; blk < D / 32; ++blk)
#pragma unroll
              for (int r = 0; r < 16; ++r) dq[blk][r] *= keep;
          }
        }
        if (biased) {
          if (w == NEAR) {
#pragma unroll
            for (int r = 0; r < 16; ++r) diag_put[(16 * (r >> 3) + (r & 7)) * DIAG_ROW] = narrow<T>() ? s[r] * undo : s[r];
            __builtin_amdgcn_wave_barrier();
            f32x4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const f32x4 *>(diag_get + 4 * i);
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += (x[i][0] + x[i][1]) + (x[i][2] + x[i][3]);
            mine[t + u * 32 - q0pos - 31 + lane + reach + EDGE] += sum;
            __builtin_amdgcn_wave_barrier();
          } else {
            float x = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) x += s[r];
            if (narrow<T>()) x *= undo;
            if (w == BEHIND) behind += x;
            else ahead += x;
          }
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          f32x8 x;
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = s[8 * g + j];
          const frag_t<T> df = to_frag<T>(x);
#pragma unroll
          for (int blk = 0; blk < D / 32; ++blk)
            dq[blk] = mma32(TL::col_frag(kt, u * 32 + 16 * g + 8 * half, 32 * blk + (lane & 16), lane), df, dq[blk]);
        }
      }
    }
    if (more) {
      ks.store(lds + (buf ^ 1) * 2 * TB, t + KT, wlo, whi, tid);
      vs.store(lds + (buf ^ 1) * 2 * TB + TB, t + KT, wlo, whi, tid);
    }
    __syncthreads();
  }
  if constexpr (narrow<T>()) {
    peak *= undo;
    if (peak > 0.f && peak < INFINITY && grads > -64) grads = max(grads, __builtin_amdgcn_frexp_expf(peak) - (DS_TOP - DS_UP));
    const int most = wave_max_i32(grads);
    if (lane == 0) p.tops[(((long)bh * p.qtiles + qt) * NW + wave) * p.key_splits + split] = most;
  }
  if (valid) {
    if (p.piece) store_row<float, D>(p.piece + split * ((long)p.b * p.nq * p.h * D) + row, dq, p.scale * undo, half);
    else store_row<T, D>(reinterpret_cast<T *>(p.dq) + row, dq, p.scale * undo, half);
  }
  if (!biased) return;
  const float far_behind = wave_allreduce_sum_f32(behind), far_ahead = wave_allreduce_sum_f32(ahead);
  if (lane == 0) {
    mine[0] += far_behind;
    mine[2 * (reach + EDGE)] += far_ahead;
  }
  __syncthreads();
  // distances -> buckets (keys ahead share bucket 0 unless they have their own), one row of partial sums a workgroup: the
  // waves' rows are added first, then a wave takes every fourth bucket, its lanes the distances
  float *part = p.hist + (((long)bh * p.qtiles + qt) * p.key_splits + split) * p.table_rows;
  const int pitch = (span + 3) / 4 * 4, most = reach + EDGE;
  for (int i = tid; i < span; i += NT) {
    float x = sums[i];
#pragma unroll
    for (int w = 1; w < NW; ++w) x += sums[w * pitch + i];
    sums[i] = x;
  }
  __syncthreads();
  for (int bucket = wave; bucket < p.table_rows; bucket += NW) {
    float x = 0.f;
    const auto add = [&](int from, int to) {               // relative positions [from, to]
      for (int a = from + lane; a <= to; a += 64) x += sums[a + most];
    };
    const bool second = p.bk.both && bucket >= p.bk.n && bucket < 2 * p.bk.n;
    const int i = second ? bucket - p.bk.n : bucket;
    if (bucket < p.bk.n || second) {
      const int from = p.bk.border[i], to = i + 1 < p.bk.n ? p.bk.border[i + 1] - 1 : most;
      if (second) add(max(from, 1), to);
      else add(-to, -from);
      if (i == 0 && !p.bk.both) add(1, most);
    }
    x = wave_allreduce_sum_f32(x);
    if (lane == 0) part[bucket] = x;
  }
}

// table gradient: partial rows (b, head, query tile) -> (rows, h), summed in f32 in a fixed order
template <typename T>
__global__ __launch_bounds__(256) void rel_bwd_table_kernel(const float *hist, int b, int h, int qtiles, int rows, T *dtable) {
  const int head = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int bucket = blockIdx.y * 4 + wave; bucket < rows; bucket += 4 * gridDim.y) {
    float x = 0.f;
    const int n = b * qtiles;
    for (int i = lane; i < n; i += 64) {
      const int bi = i / qtiles, qt = i - bi * qtiles;
      x += hist[(((long)bi * h + head) * qtiles + qt) * rows + bucket];
    }
    x = wave_allreduce_sum_f32(x);
    if (lane == 0) dtable[(long)bucket * h + head] = (T)x;
  }
}

// ---- backward: dK, dV --------------------------------------------------------------------------------------------------------
// A wave owns 32 keys (columns; K and V rows in registers), a workgroup NW waves that share the streamed query tiles (Q, dO,
// lse, delta, intervals; the last three made ready by the dQ kernel: computed here, behind loads of their own, they had every
// tile wait for memory -- 245 us instead of 197 for packed documents of 128 wide heads, 35 instead of 31 for the encoder's).  S = Q K^T, dP = dO V^T with queries along the registers: P and dS are at once the B operands of
// dV^T += dO^T P and dK^T += Q^T dS.  The heads that share the keys are a loop: their sums stay in the accumulators -- unless
// there are too few workgroups for the chip (see splits_of): then heads and runs of queries become workgroups of their own,
// which leave f32 sums that a small kernel adds in order.
// Two waves a SIMD where the registers allow it (f32 of 64 wide spills 10 for it: 140 us instead of 150 for 7 x 547 tokens, 8 heads).
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, (sizeof(T) == 2 ? D < 128 : D == 64) ? 2 : 1) void rel_bwd_dkv_kernel(const Params p) {
  typedef Tile<T, D> TL;
  constexpr int QT = dkv_tile<T>(D), NT = NW * 64, SUB = QT / 32, TB = QT * TL::ROW;
  extern __shared__ __align__(16) char lds[];
  __shared__ float stats[2][2][QT];            // [buffer][lse, delta]
  __shared__ int rows[2][2][QT];               // [buffer][lo, hi]
  __shared__ int todo[256], ntodo;
  constexpr bool KL = dkv_keys_in_lds<T>(D);
  float *bias = reinterpret_cast<float *>(lds + 4 * TB + (KL ? NW * 32 * TL::ROW : 0));
  const int reach = p.bk.reach;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
  const int id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int splits = p.head_splits * p.query_splits, split = id % splits, tile_id = id / splits;
  const int bh = tile_id / p.ktiles, kt0 = tile_id % p.ktiles;
  const int b = bh / p.hkv, kvh = bh - b * p.hkv;
  const int heads = p.group / p.head_splits, head0 = kvh * p.group + split / p.query_splits * heads;
  const int k0 = kt0 * NW * 32, kw = k0 + wave * 32, key = kw + col;
  const bool valid = key < p.nk;
  frag_t<T> kf[D / 16], vf[D / 16];
  const int krow = min(key, p.nk - 1);
  load_row<T, D>(kf, reinterpret_cast<const T *>(p.k) + b * p.k_b + (long)krow * p.k_n + kvh * p.k_h, half);
  load_row<T, D>(vf, reinterpret_cast<const T *>(p.v) + b * p.v_b + (long)krow * p.v_n + kvh * p.v_h, half);
  char *const ktile = lds + 4 * TB + wave * 32 * TL::ROW;      // this wave's, a lane's row at kappa(col): conflict-free as ever
  if constexpr (KL) {
#pragma unroll
    for (int f = 0; f < D / 16; ++f) *reinterpret_cast<frag_t<T> *>(ktile + TL::at(kappa(col), 2 * f + half)) = kf[f];
  }
  const bool biased = p.bk.n > 0;
  const float scale2 = p.scale * LOG2E;
  const int nblocks = (p.nq + 31) / 32, ntiles = (p.nq + QT - 1) / QT;
  const int4 *blocks = p.blocks + (long)b * p.qtiles * NW;

  int up = 0;                                  // f16: dS is held times 2^up, P times 2^P_UP
  if constexpr (narrow<T>()) {
    int most = -64;
    const int each = nblocks * p.key_splits;
    for (int i = tid; i < p.group * each; i += NT) {
      const int hh = i / each;
      most = max(most, p.tops[((long)b * p.h + kvh * p.group + hh) * p.qtiles * NW * p.key_splits + (i - hh * each)]);
    }
    most = wave_max_i32(most);
    if (lane == 0) todo[wave] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) most = max(most, todo[w]);
    up = most == -64 ? 0 : DS_UP - most;
  }
  const float ds_factor = __builtin_ldexpf(1.f, up - (narrow<T>() ? P_UP : 0));

  f32x16 dk[D / 32] = {}, dv[D / 32] = {};
  const int run = (ntiles + p.query_splits - 1) / p.query_splits;
  const int tile0 = split % p.query_splits * run, tile1 = min(tile0 + run, ntiles);
  for (int head = head0; head < head0 + heads; ++head) {
    BiasFill<T> fill;
    fill.start(p.bk, p.table, p.h, head, tid);
    __syncthreads();
    fill.finish(bias, p.bk, p.table, p.h, head, tid, NT);
    const T *qb = reinterpret_cast<const T *>(p.q) + b * p.q_b + head * p.q_h;
    const T *gb = reinterpret_cast<const T *>(p.grad) + b * p.grad_b + head * p.grad_h;
    const float2 *stats_of = p.stat + ((long)b * p.h + head) * p.nq;
    const int2 *rows_of = p.rows + (long)b * p.nq;
    for (int chunk = tile0; chunk < tile1; chunk += 256) {
      // query tiles that see any of these keys, in order; bit 30: some query does not see all of them
      __syncthreads();
      if (wave == 0) {
        int n = 0;
        for (int c = chunk; c < min(chunk + 256, tile1); c += 64) {
          const int tile = c + lane;
          bool any = false, cut = false;
          if (tile < tile1) {
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
              const int blk = tile * SUB + u;
              if (blk >= nblocks) continue;
              const int4 s = blocks[blk];
              any |= s.x < k0 + NW * 32 && s.y > k0;
              cut |= s.z > k0 || s.w < min(k0 + NW * 32, p.nk);
            }
          }
          const unsigned long long mask = __ballot(any);
          if (any) todo[n + __popcll(mask & ((1ull << lane) - 1))] = tile | (cut ? 1 << 30 : 0);
          n += __popcll(mask);
        }
        if (lane == 0) ntodo = n;
      }
      __syncthreads();
      const int n = ntodo;
      Stage<T, D, QT, NT> qs, gs;
      float2 st;
      int2 row;
      auto fetch = [&](int tile) {
        const int q0 = tile * QT;
        qs.load(qb, p.q_n, q0, 0, p.nq, tid);
        gs.load(gb, p.grad_n, q0, 0, p.nq, tid);
        const int qi = min(q0 + tid % QT, p.nq - 1);       // (nothing is done to what is loaded: that would wait for the tile)
        st = stats_of[qi];
        row = rows_of[qi];
      };
      auto put = [&](int buf, int tile) {
        qs.store(lds + buf * 2 * TB, tile * QT, 0, p.nq, tid);
        gs.store(lds + buf * 2 * TB + TB, tile * QT, 0, p.nq, tid);
        if (tid < QT) {
          const bool some = tile * QT + tid < p.nq;
          stats[buf][0][tid] = some ? st.x - (narrow<T>() ? P_UP : 0) : INFINITY;
          stats[buf][1][tid] = some ? st.y * ds_factor : 0.f;
          rows[buf][0][tid] = row.x;
          rows[buf][1][tid] = some ? row.y : 0;
        }
      };
      if (n > 0) {
        fetch(todo[0] & ~(1 << 30));
        put(0, todo[0] & ~(1 << 30));
      }
      __syncthreads();
      loads_done();
      for (int i = 0; i < n; ++i) {
        const int buf = i & 1, entry = todo[i], q0 = (entry & ~(1 << 30)) * QT;
        const bool cut = entry >> 30;
        if (i + 1 < n) fetch(todo[i + 1] & ~(1 << 30));
        const char *qt = lds + buf * 2 * TB, *gt = qt + TB;
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          f32x16 s{}, dp{};
#pragma unroll
          for (int f = 0; f < D / 16; ++f) {
            s = mma32(TL::row_frag(qt, u * 32 + kappa(col), 2 * f + half), KL ? TL::row_frag(ktile, kappa(col), 2 * f + half) : kf[f], s);
            dp = mma32(TL::row_frag(gt, u * 32 + kappa(col), 2 * f + half), vf[f], dp);
          }
          const int p0 = q0 + u * 32 + p.offset;
          const Where w = biased ? where(kw, 32, p0, reach) : BEHIND;
          if (w == NEAR) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= scale2;
            add_bias<-1>(s, bias, reach, key - (p0 + 8 * half));
          } else {
            const float add = biased ? bias[w == BEHIND ? 0 : 2 * (reach + EDGE)] : 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], scale2, add);
          }
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int at = u * 32 + 16 * g + 8 * half;
            const f32x4 l0 = *reinterpret_cast<const f32x4 *>(&stats[buf][0][at]);
            const f32x4 l1 = *reinterpret_cast<const f32x4 *>(&stats[buf][0][at + 4]);
            const f32x4 d0 = *reinterpret_cast<const f32x4 *>(&stats[buf][1][at]);
            const f32x4 d1 = *reinterpret_cast<const f32x4 *>(&stats[buf][1][at + 4]);
            f32x8 x, y;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              x[j] = exp2_(s[8 * g + j] - (j < 4 ? l0[j & 3] : l1[j & 3]));
              y[j] = x[j] * __builtin_fmaf(dp[8 * g + j], ds_factor, -(j < 4 ? d0[j & 3] : d1[j & 3]));
            }
            if (cut) {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if ((unsigned)(key - rows[buf][0][at + j]) >= (unsigned)rows[buf][1][at + j]) x[j] = y[j] = 0.f;
            }
            const frag_t<T> pf = to_frag<T>(x), df = to_frag<T>(y);
#pragma unroll
            for (int blk = 0; blk < D / 32; ++blk) {
              dv[blk] = mma32(TL::col_frag(gt, at, 32 * blk + (lane & 16), lane), pf, dv[blk]);
              dk[blk] = mma32(TL::col_frag(qt, at, 32 * blk + (lane & 16), lane), df, dk[blk]);
            }
          }
        }
        if (i + 1 < n) put(buf ^ 1, todo[i + 1] & ~(1 << 30));
        __syncthreads();
      }
    }
  }
  if (!valid) return;
  const long row = (((long)b * p.nk + key) * p.hkv + kvh) * D;
  if (p.part) {
    const long all = (long)p.b * p.nk * p.hkv * D;
    store_row<float, D>(p.part + split * all + row, dk, p.scale * __builtin_ldexpf(1.f, -up), half);
    store_row<float, D>(p.part + (splits + split) * all + row, dv, narrow<T>() ? 1.f / (1 << P_UP) : 1.f, half);
    return;
  }
  store_row<T, D>(reinterpret_cast<T *>(p.dk) + row, dk, p.scale * __builtin_ldexpf(1.f, -up), half);
  store_row<T, D>(reinterpret_cast<T *>(p.dv) + row, dv, narrow<T>() ? 1.f / (1 << P_UP) : 1.f, half);
}

// dK, dV = the sums of their splits, in order
template <typename T>
__global__ __launch_bounds__(256) void rel_bwd_fold_kernel(const float *part, int splits, long quads, T *dk, T *dv) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= quads) return;
  const f32x4 *from = reinterpret_cast<const f32x4 *>(part) + (long)blockIdx.y * splits * quads + i;
  f32x4 x = from[0];
#pragma unroll 4
  for (int s = 1; s < splits; ++s) {
    const f32x4 y = from[s * quads];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += y[e];
  }
  reinterpret_cast<vec4_t<T> *>(blockIdx.y ? dv : dk)[i] = to_vec4<T>(x);
}

// ---- host side -----------------------------------------------------------------------------------------------------------------
constexpr int NW = 4;                          // waves of a workgroup: 128 queries (forward, dQ) or keys (dK, dV)

int check(const char *where, const sig3d_rel_attention_args *a) {
  LANG_NEED(where, a != nullptr, "no arguments");
  LANG_NEED(where, a->dtype >= 0 && a->dtype <= 2, "dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
  LANG_NEED(where, a->b >= 1 && a->nq >= 1 && a->nk >= 1 && a->h >= 1 && a->hkv >= 1, "sizes must be positive");
  LANG_NEED(where, a->d == 64 || a->d == 96 || a->d == 128, "head size must be 64, 96 or 128");
  LANG_NEED(where, a->h % a->hkv == 0, "heads must be a multiple of key heads");
  LANG_NEED(where, a->nq <= (1 << 29) && a->nk <= (1 << 29), "at most 2^29 tokens");
  LANG_NEED(where, a->query_offset > -(1 << 29) && a->query_offset < (1 << 29), "query_offset out of range");
  const int e = a->dtype == 0 ? 4 : 2;
  const long strides[9] = {a->q_b, a->q_n, a->q_h, a->k_b, a->k_n, a->k_h, a->v_b, a->v_n, a->v_h};
  for (long s : strides) LANG_NEED(where, s >= 0 && s * e % 16 == 0, "strides must be non-negative multiples of 16 bytes");
  const long rows[3] = {a->q_n, a->k_n, a->v_n};
  for (long s : rows) LANG_NEED(where, s * e < (1l << 24), "token strides must be below 16 MB");
  LANG_NEED(where, a->q && a->k && a->v && a->out && aligned16(a->q) && aligned16(a->k) && aligned16(a->v) && aligned16(a->out),
       "q, k, v, out must be 16-byte aligned addresses");
  LANG_NEED(where, (a->out32 == nullptr) == (a->lse == nullptr) && aligned16(a->out32), "out32 and lse come together");
  if (int e = check_buckets(where, a->buckets, a->table, a->table_rows)) return e;
  LANG_NEED(where, (long)a->b * a->h * ((a->nq + 31) / 32) < INT_MAX / 16 && (long)a->b * a->h * ((a->nk + 31) / 32) < INT_MAX / 16, "grid too large");
  return 0;
}

Params params(const sig3d_rel_attention_args *a) {
  Params p = {};
  p.q = a->q; p.k = a->k; p.v = a->v; p.table = a->table; p.grad = a->grad;
  p.key_lengths = a->key_lengths; p.prefix_lengths = a->prefix_lengths; p.key_ranges = a->key_ranges;
  p.out = a->out; p.dq = a->dq; p.dk = a->dk; p.dv = a->dv; p.dtable = a->dtable;
  p.out32 = a->out32; p.lse = a->lse;
  p.q_b = a->q_b; p.q_n = a->q_n; p.q_h = a->q_h; p.k_b = a->k_b; p.k_n = a->k_n; p.k_h = a->k_h;
  p.v_b = a->v_b; p.v_n = a->v_n; p.v_h = a->v_h; p.grad_b = a->grad_b; p.grad_n = a->grad_n; p.grad_h = a->grad_h;
  p.b = a->b; p.nq = a->nq; p.nk = a->nk; p.h = a->h; p.hkv = a->hkv; p.group = a->h / a->hkv;
  p.causal = a->causal; p.offset = a->query_offset; p.table_rows = a->table_rows;
  p.qtiles = sig3d_ceil_div(a->nq, NW * 32);
  p.ktiles = sig3d_ceil_div(a->nk, NW * 32);
  p.scale = a->scale;
  p.bk = device_buckets(a->buckets);
  return p;
}

int key_splits(const sig3d_rel_attention_args *a);

// workspace of the backward pass: lse and delta (b h nq), intervals (b nq), their summaries (b, 4 per 128 queries) int4, exponents
// (f16), partial table gradients
long work_stat(const sig3d_rel_attention_args *a) { return ((long)a->b * a->h * a->nq * 2 + 3) / 4 * 4; }
long work_rows(const sig3d_rel_attention_args *a) { return ((long)a->b * a->nq * 2 + 3) / 4 * 4; }
long work_blocks(const sig3d_rel_attention_args *a) { return (long)a->b * sig3d_ceil_div(a->nq, NW * 32) * NW * 4; }
long work_tops(const sig3d_rel_attention_args *a) {
  return a->dtype == 2 ? ((long)a->b * a->h * sig3d_ceil_div(a->nq, NW * 32) * NW * key_splits(a) + 3) / 4 * 4 : 0;
}
long work_hist(const sig3d_rel_attention_args *a) {
  return a->buckets.n > 0 ? (long)a->b * a->h * sig3d_ceil_div(a->nq, NW * 32) * key_splits(a) * a->table_rows : 0;
}

// Key splits of the forward and the dQ kernel: where batch, heads and tiles of 128 queries are fewer workgroups than two for each
// of 256 CUs, down to 8 tiles of keys (f32: 4; a tile there is 6000 cycles of the matrix cores).  (2 x 1021 tokens, 8 heads of 96
// floats: 126 us forward and 176 us dQ as 128 workgroups.)
int key_splits(const sig3d_rel_attention_args *a) {
  const long items = (long)a->b * a->h * sig3d_ceil_div(a->nq, NW * 32);
  const int tiles = sig3d_ceil_div(a->nk, a->dtype == 0 ? 32 : 64), least = a->dtype == 0 ? 4 : 8;
  return (int)std::max<long>(1, std::min<long>(std::min<long>(16, (512 + items - 1) / items), tiles / least));
}
long work_piece(const sig3d_rel_attention_args *a) {
  const int n = key_splits(a);
  return n > 1 ? (long)n * a->b * a->nq * a->h * a->d : 0;
}
long work_ml(const sig3d_rel_attention_args *a) {
  const int n = key_splits(a);
  return n > 1 ? ((long)n * a->b * a->nq * a->h * 2 + 3) / 4 * 4 : 0;
}

// Splits of the dK / dV kernel.  Causal and packed rows make workgroups very unequal -- the first keys of a document are seen by
// all of it -- so there should be several for every CU (4 for each of 256); a run of queries is worth a workgroup from 8 tiles
// on.  A split costs a write and a read of 8 bytes an element of dK and dV.  (2 x 4096 packed tokens, 16 heads on 4, 128 wide:
// 524 us as 256 workgroups, at the time 245 so.)
struct Splits { int heads, queries; };
Splits splits_of(const sig3d_rel_attention_args *a) {
  const long base = (long)a->b * a->hkv * sig3d_ceil_div(a->nk, NW * 32);
  const int want = (int)std::min<long>(16, (1024 + base - 1) / base), group = a->h / a->hkv;
  Splits s = {1, 1};
  for (int n = 2; n <= want; ++n)
    if (group % n == 0) s.heads = n;
  const int tiles = sig3d_ceil_div(a->nq, a->dtype == 0 || a->d == 96 ? 32 : 64);
  s.queries = std::max(1, std::min(want / s.heads, tiles / 8));
  return s;
}
long work_part(const sig3d_rel_attention_args *a) {
  const Splits s = splits_of(a);
  const long n = (long)s.heads * s.queries;
  return n > 1 ? 2 * n * a->b * a->nk * a->hkv * a->d : 0;
}

template <typename T, int D, bool TWO> int launch_fwd(const Params &p, hipStream_t stream) {
  static sig3d_once_per_device once;
  const size_t lds = 4 * key_tile<T>() * Tile<T, D>::ROW + bias_floats(p.bk.reach) * sizeof(float);
  if (int e = allow_lds(rel_fwd_kernel<T, D, NW, TWO>, once)) return e;
  rel_fwd_kernel<T, D, NW, TWO><<<p.b * p.h * p.qtiles * p.key_splits, NW * 64, lds, stream>>>(p);
  SIG3D_LAUNCH_CHECK("rel_fwd_kernel");
  if (p.piece) {
    rel_join_kernel<T, D><<<sig3d_ceil_div((long)p.b * p.nq * p.h, 256 / (D / 4)), 256, 0, stream>>>(p);
    SIG3D_LAUNCH_CHECK("rel_join_kernel");
  }
  return 0;
}

template <typename T, int D> int launch_bwd(const Params &p, hipStream_t stream) {
  static sig3d_once_per_device once_q, once_kv;
  const int span = (bias_floats(p.bk.reach) + 3) / 4 * 4;
  const size_t tiles = (4 * dkv_tile<T>(D) + (dkv_keys_in_lds<T>(D) ? NW * 32 : 0)) * Tile<T, D>::ROW;
  const size_t dq_tiles = 4 * dq_tile<T>(D) * Tile<T, D>::ROW;
  if (int e = allow_lds(rel_bwd_dq_kernel<T, D, NW>, once_q)) return e;
  if (int e = allow_lds(rel_bwd_dkv_kernel<T, D, NW>, once_kv)) return e;
  rel_bwd_dq_kernel<T, D, NW><<<p.b * p.h * p.qtiles * p.key_splits, NW * 64, dq_tiles + ((NW + 1) * span + NW * DIAG) * sizeof(float), stream>>>(p);
  SIG3D_LAUNCH_CHECK("rel_bwd_dq_kernel");
  if (p.piece) {
    const long quads = (long)p.b * p.nq * p.h * D / 4;
    rel_bwd_fold_kernel<T><<<dim3(sig3d_ceil_div(quads, 256), 1), 256, 0, stream>>>(p.piece, p.key_splits, quads,
                                                                                   reinterpret_cast<T *>(p.dq), nullptr);
    SIG3D_LAUNCH_CHECK("rel_bwd_fold_kernel");
  }
  rel_bwd_dkv_kernel<T, D, NW><<<p.b * p.hkv * p.ktiles * p.head_splits * p.query_splits, NW * 64, tiles + span * sizeof(float), stream>>>(p);
  SIG3D_LAUNCH_CHECK("rel_bwd_dkv_kernel");
  if (p.part) {
    const long quads = (long)p.b * p.nk * p.hkv * D / 4;
    rel_bwd_fold_kernel<T><<<dim3(sig3d_ceil_div(quads, 256), 2), 256, 0, stream>>>(
        p.part, p.head_splits * p.query_splits, quads, reinterpret_cast<T *>(p.dk), reinterpret_cast<T *>(p.dv));
    SIG3D_LAUNCH_CHECK("rel_bwd_fold_kernel");
  }
  if (p.bk.n > 0) {
    rel_bwd_table_kernel<T><<<dim3(p.h, sig3d_ceil_div(p.table_rows, 4)), 256, 0, stream>>>(
        p.hist, p.b, p.h, p.qtiles * p.key_splits, p.table_rows, reinterpret_cast<T *>(p.dtable));
    SIG3D_LAUNCH_CHECK("rel_bwd_table_kernel");
  }
  return 0;
}

}  // namespace

extern "C" int sig3d_rel_attention_fwd(const sig3d_rel_attention_args *a, void *stream) {
  if (int e = check("sig3d_rel_attention_fwd", a)) return e;
  Params p = params(a);
  p.key_splits = key_splits(a);
  if (p.key_splits > 1) {
    SIG3D_REQUIRE(a->work && aligned16(a->work), "missing workspace");
    p.piece = a->work;
    p.piece_ml = a->work + work_piece(a);
  }
  return by_type(a->dtype, a->d, [&](auto t, auto d) {
    typedef decltype(t) T;
    constexpr int D = decltype(d)::value;
    // P in two parts (see the kernel) without a backward pass: up to one workgroup for each of 256 CUs.  (12 heads of 52 bf16
    // tokens: 8.2 us instead of 7.8; 16 heads of 200: 12.3 instead of 11.6; 512 workgroups, 128 heads of 432: 25.7 instead of 22.1.)
    if constexpr (sizeof(T) == 2) {
      if (p.out32 || (long)p.b * p.h * p.qtiles * p.key_splits <= 256) return launch_fwd<T, D, true>(p, (hipStream_t)stream);
    }
    return launch_fwd<T, D, false>(p, (hipStream_t)stream);
  });
}

extern "C" long sig3d_rel_attention_fwd_work_floats(const sig3d_rel_attention_args *a) {
  if (check("sig3d_rel_attention_fwd_work_floats", a)) return -1;
  return work_piece(a) + work_ml(a);
}

extern "C" long sig3d_rel_attention_bwd_work_floats(const sig3d_rel_attention_args *a) {
  if (check("sig3d_rel_attention_bwd_work_floats", a)) return -1;
  return work_stat(a) + work_rows(a) + work_blocks(a) + work_tops(a) + (work_hist(a) + 3) / 4 * 4 + work_part(a) + work_piece(a);
}

extern "C" int sig3d_rel_attention_bwd(const sig3d_rel_attention_args *a, void *stream) {
  if (int e = check("sig3d_rel_attention_bwd", a)) return e;
  const int e = a->dtype == 0 ? 4 : 2;
  SIG3D_REQUIRE(a->out32 && a->lse && a->grad && a->dq && a->dk && a->dv && a->work, "missing array");
  SIG3D_REQUIRE(aligned16(a->grad) && aligned16(a->dq) && aligned16(a->dk) && aligned16(a->dv) && aligned16(a->work),
                "addresses must be 16-byte aligned");
  SIG3D_REQUIRE(a->grad_b >= 0 && a->grad_n >= 0 && a->grad_h >= 0 && a->grad_b * e % 16 == 0 && a->grad_n * e % 16 == 0 &&
                    a->grad_h * e % 16 == 0 && a->grad_n * e < (1l << 24),
                "strides must be non-negative multiples of 16 bytes, that of a token below 16 MB");
  SIG3D_REQUIRE(a->buckets.n == 0 || a->dtable, "a bias needs dtable");
  Params p = params(a);
  p.stat = reinterpret_cast<float2 *>(a->work);
  p.rows = reinterpret_cast<int2 *>(a->work + work_stat(a));
  p.blocks = reinterpret_cast<int4 *>(a->work + work_stat(a) + work_rows(a));
  p.tops = reinterpret_cast<int *>(a->work + work_stat(a) + work_rows(a) + work_blocks(a));
  p.hist = a->work + work_stat(a) + work_rows(a) + work_blocks(a) + work_tops(a);
  const Splits s = splits_of(a);
  p.head_splits = s.heads;
  p.query_splits = s.queries;
  if (s.heads * s.queries > 1) p.part = p.hist + (work_hist(a) + 3) / 4 * 4;
  p.key_splits = key_splits(a);
  if (p.key_splits > 1) p.piece = p.hist + (work_hist(a) + 3) / 4 * 4 + work_part(a);
  return by_type(a->dtype, a->d, [&](auto t, auto d) {
    return launch_bwd<decltype(t), decltype(d)::value>(p, (hipStream_t)stream);
  });
}
