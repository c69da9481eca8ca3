// decode_attention.hip -- attention of new tokens over the key / value cache, with prefixes that many sequences share, for gfx950.
//
// Sequence i sees [the rows of shared sequence i / (b / groups) | its own rows up to the query].  Decoding is bound by reading
// keys and values, so each part is read as few times as its users allow: the queries of ALL sequences of a group that share a
// key head are rows of one product over the shared keys (up to 32 rows a workgroup), and only the own rows are read per
// sequence.  Both parts are cut along the keys until the chip is full; a piece leaves (max, sum, unnormalised output), and a
// second kernel joins the pieces of a row in their order.  Small calls -- one piece, nothing worth sharing -- are one launch:
// a workgroup walks shared and own rows of one sequence and writes the result itself.
//
// A wave owns every fourth 32-key tile of its workgroup's piece and NB blocks of 16 query rows; no barrier until the waves join.
// S^T = K Q^T on 16x16x32: the K fragment is loaded straight from memory (a lane's 16 bytes are a fragment), in the row order
// that makes two S tiles' registers the P fragment (key 8 g + 4 t + r for tile t, lane group g, register r).  V is staged in
// wave-private LDS for the transposing read.  The next tile's loads are in flight while one is used.
// In 16 bits a wave with one block of rows puts P into its product as two parts, rounded and rest: it waits for memory anyway (64
// questions on a scene of 5000 rows, 30 000-token contexts: within 2 %), and the result is left with its own rounding.  Two blocks
// would pay for it (2 scenes, 48 questions: 57 us instead of 54), for a factor of 1.4 in the error of the shared rows' part.
// An e4m3 cache is widened to the query's type on the way in -- exact, the scale being a power of two.
#include "lang_core.h"

#include <limits.h>

#include <algorithm>

namespace {
using namespace lang;

constexpr int WAVES = 4, KT = 32;
constexpr float SLACK = 8.f;

struct Side { const void *k, *v; const float *k_scale, *v_scale; int capacity; };
struct DecodeParams {
  const void *q, *table;
  Side own, shared;
  const int *lengths, *shared_lengths, *counts;
  void *out;
  float *part;               // pieces: D + 4 floats a row and piece (output, max, sum, two unused)
  long q_b, q_n, q_h;
  int b, t, h, hkv, group, each;       // each: sequences of a shared prefix (0: nothing is shared)
  int own_splits, shared_splits;       // most pieces of a row's own and shared keys (see piece_rows)
  int own_tiles, shared_tiles, own_items, shared_items, own_bias_heads, shared_bias_heads;
  int joined;                // own items walk the shared rows too, no shared items
  int direct;                // one piece a row: the result is written here
  float scale;
  Buckets bk;
};

// One 32-key tile of one side on its way from memory.
template <typename T, int D, bool Q> struct Flight {
  static constexpr int KS = D / 32;                         // reduction steps of a score
  static constexpr int VE = Q ? 16 : 8;                     // elements of a piece of V: 16 bytes in 8 or 16 bits
  static constexpr int VN = KT * D / VE / 64;               // pieces of V a lane carries
  frag_t<T> k[2][Q ? 1 : KS];
  uint2 kq[2][Q ? KS : 1];
  float ks[2];
  frag_t<T> v[Q ? 1 : VN];
  uint4 vq[Q ? VN : 1];
  float vs[Q ? VN : 1];

  // k, v, k_scale, v_scale: the tile's first row (uniform over the wave, so that a load is one scalar base and a 32-bit offset);
  // n: rows of the tile that exist.  Loads of rows beyond them repeat the last one: scores are masked, put_v zeroes.
  __device__ __forceinline__ void load(const char *kp, const char *vp, const float *k_scale, const float *v_scale, int n, int lane) {
    constexpr int ROW = D * (Q ? 1 : (int)sizeof(T));
    const int m = lane & 15, g = lane >> 4, last = n - 1;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const unsigned row = min(8 * (m >> 2) + 4 * t + (m & 3), last);
      if constexpr (Q) {
        ks[t] = k_scale[row];
#pragma unroll
        for (int f = 0; f < KS; ++f)       // lane group g holds D / 4 consecutive values: 16 bytes a load, and Q likewise
          kq[t][f] = *reinterpret_cast<const uint2 *>(kp + (row * ROW + g * (D / 4) + 8 * f));
      } else {
#pragma unroll
        for (int f = 0; f < KS; ++f)
          k[t][f] = *reinterpret_cast<const frag_t<T> *>(kp + (row * ROW + (32 * f + 8 * g) * (unsigned)sizeof(T)));
      }
    }
#pragma unroll
    for (int i = 0; i < VN; ++i) {
      const unsigned c = lane + 64 * i, r = c / (D / VE), o = c - r * (D / VE), row = min((int)r, last);
      if constexpr (Q) {
        vq[i] = *reinterpret_cast<const uint4 *>(vp + (row * ROW + VE * o));
        vs[i] = v_scale[row];
      } else {
        v[i] = *reinterpret_cast<const frag_t<T> *>(vp + (row * ROW + VE * o * (unsigned)sizeof(T)));
      }
    }
  }
  __device__ __forceinline__ frag_t<T> key(int t, int f) const {
    if constexpr (Q) return from_e4m3<T>(kq[t][f], ks[t]);
    else return k[t][f];
  }
  __device__ __forceinline__ void put_v(char *tile, int n, int lane) const {
#pragma unroll
    for (int i = 0; i < VN; ++i) {
      const int c = lane + 64 * i, r = c / (D / VE), o = c - r * (D / VE);
      const bool none = n < KT && r >= n;
      if constexpr (Q) {
        put_piece(tile, r, 2 * o, none ? frag_t<T>{} : from_e4m3<T>(make_uint2(vq[i].x, vq[i].y), vs[i]));
        put_piece(tile, r, 2 * o + 1, none ? frag_t<T>{} : from_e4m3<T>(make_uint2(vq[i].z, vq[i].w), vs[i]));
      } else {
        put_piece(tile, r, o, none ? frag_t<T>{} : v[i]);
      }
    }
  }
  static __device__ __forceinline__ void put_piece(char *tile, int r, int o, frag_t<T> x) {
    typedef Tile<T, D, true> TL;
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<frag_t<T> *>(tile + TL::at(r, o)) = x;
    } else {
      *reinterpret_cast<f32x4 *>(tile + TL::at(r, 2 * o)) = __builtin_shufflevector(x, x, 0, 1, 2, 3);
      *reinterpret_cast<f32x4 *>(tile + TL::at(r, 2 * o + 1)) = __builtin_shufflevector(x, x, 4, 5, 6, 7);
    }
  }
};

// which element of a head fragment f of lane group g starts at (see Flight::load)
template <int D, bool Q> __device__ __forceinline__ int element(int f, int g) { return Q ? g * (D / 4) + 8 * f : 32 * f + 8 * g; }

// over the four 16-lane groups
__device__ __forceinline__ void both_groups(float x, float &lo, float &hi) {
  const auto s = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  const unsigned a = s[0], b = s[1];
  lo = __builtin_bit_cast(float, a);
  hi = __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float max_groups(float x) {
  float lo, hi;
  both_groups(x, lo, hi);
  return max_halves(fmaxf(lo, hi));
}
__device__ __forceinline__ float sum_groups(float x) {
  float lo, hi;
  both_groups(x, lo, hi);
  return sum_halves(lo + hi);
}

// The tiles of a sequence are cut into at most `most` pieces of equal length, of at least LEAST tiles (four a wave: below that a
// workgroup is all start and join).  Short sequences of a ragged batch have few pieces, and the workgroups of the others leave
// at once; long ones do not get longer pieces than they must.
constexpr int LEAST = 4 * WAVES;
__device__ __forceinline__ int piece_tiles(int tiles, int most) { return max(LEAST, (tiles + most - 1) / most); }
__device__ __forceinline__ int clamp_rows(int n, int capacity) { return min(max(n, 0), capacity); }
__device__ __forceinline__ int tiles_of(int rows) { return (rows + KT - 1) / KT; }

// LDS tiles of V a wave has
template <typename T, int D> constexpr int TILES = D == 64 && sizeof(T) == 2 ? 2 : 1;

// One item: 16 NB query rows over one piece of their keys, by WV = 4 waves of a workgroup (a wave every fourth tile, joined
// through LDS) or by one wave alone.
template <typename T, int D, bool Q, int NB, int WV>
__device__ __forceinline__ void walk(const DecodeParams &p, int item, bool shared, char *lds) {
  typedef Tile<T, D, true> TL;
  typedef Flight<T, D, Q> FL;
  constexpr int KS = FL::KS, TB = KT * TL::ROW, DT = D / 16;
  constexpr bool TWO = sizeof(T) == 2 && NB == 1;           // parts of P (see the top)
  // tiles a step: a lone wave has nobody to hide its latencies behind but its own second tile
  constexpr int NT = WV == 1 ? TILES<T, D> : 1;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int wave = WV == 1 ? 0 : wv, tid = WV == 1 ? lane : threadIdx.x;   // among those that share the item
  char *vt = lds + wv * TILES<T, D> * TB;
  const int heads = shared ? p.shared_bias_heads : p.own_bias_heads, reach = p.bk.reach;
  float *bias = reinterpret_cast<float *>(lds + WAVES * TILES<T, D> * TB) + (WV == 1 ? wv * heads * (reach + 1) : 0);

  // item -> (sequence or group, key head, block of rows, piece)
  const int splits = shared ? p.shared_splits : p.own_splits, tiles = shared ? p.shared_tiles : p.own_tiles;
  const int piece = item % splits;
  item /= splits;
  const int rt = item % tiles;
  item /= tiles;
  const int kvh = item % p.hkv, unit = item / p.hkv;                       // unit: sequence, or group
  const int per = p.group * p.t, rows = shared ? p.each * per : per;
  const int r0 = rt * 16 * NB;

  // log2(e) * bias of the heads of these rows by distance behind the query.  These loads go out before those of keys and
  // queries: loads return in order, and these are two in a row (bucket, entry).
  const bool biased = p.bk.n > 0;
  const int in0 = shared ? r0 % per : r0, gi0 = p.t == 1 ? in0 : in0 / p.t, biases = biased ? heads * (reach + 1) : 0;
  const T *table = reinterpret_cast<const T *>(p.table);
  auto bias_at = [&](int i) {
    int hh = heads == 1 ? 0 : i / (reach + 1);
    const int a = i - hh * (reach + 1);
    hh += gi0;
    return (float)table[(long)bucket_of(p.bk, -a) * p.h + kvh * p.group + (hh >= p.group ? hh - p.group : hh)] * LOG2E;
  };
  float first_bias = 0.f;
  if (tid < biases) first_bias = bias_at(tid);

  const int shared_len = p.each && (shared || p.joined)
                             ? clamp_rows(p.shared_lengths[shared ? unit : unit / p.each], p.shared.capacity) : 0;
  const int own_len = shared ? 0 : clamp_rows(p.lengths[unit], p.own.capacity);
  // the piece, in tiles: those of the shared rows, then those of the own rows
  const int far_tiles = tiles_of(shared_len), all_tiles = far_tiles + tiles_of(own_len);
  const int share = piece_tiles(all_tiles, splits), from = piece * share, to = min(from + share, all_tiles);
  if (piece > 0 && from >= all_tiles) return;

  const long far_row = ((long)(shared ? unit : (p.each ? unit / p.each : 0)) * p.hkv + kvh) * p.shared.capacity;
  const long own_row = ((long)unit * p.hkv + kvh) * p.own.capacity;
  FL fl[NT];
  auto fetch = [&](FL &f, int tile) {
    const bool far = tile < far_tiles;
    const int k0 = (far ? tile : tile - far_tiles) * KT;
    const long row = (far ? far_row : own_row) + k0;
    constexpr int ROW = D * (Q ? 1 : (int)sizeof(T));
    const void *kp = far ? p.shared.k : p.own.k, *vp = far ? p.shared.v : p.own.v;
    const float *ksp = far ? p.shared.k_scale : p.own.k_scale, *vsp = far ? p.shared.v_scale : p.own.v_scale;
    f.load(reinterpret_cast<const char *>(kp) + row * ROW, reinterpret_cast<const char *>(vp) + row * ROW, ksp + row, vsp + row,
           min((far ? shared_len : own_len) - k0, KT), lane);
  };
#pragma unroll
  for (int u = 0; u < NT; ++u)
    if (from + wave + u * WV < to) fetch(fl[u], from + wave + u * WV);

  int pos[NB], qhead[NB];                    // own row of the query (below 0: no query); its head in the group
  frag_t<T> qf[NB][KS];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int r = r0 + 16 * n + col, row = min(r, rows - 1);
    const int sub = shared ? row / per : 0, in = row - sub * per, seq = shared ? unit * p.each + sub : unit;
    qhead[n] = p.t == 1 ? in : in / p.t;
    const int j = in - qhead[n] * p.t;
    pos[n] = -1;
    if (r < rows) {
      const int len = shared ? clamp_rows(p.lengths[seq], p.own.capacity) : own_len;
      const int count = p.counts ? clamp_rows(p.counts[seq], p.t) : p.t;
      if (j < count) pos[n] = max(len - count + j, -1);
    }
#pragma unroll
    for (int f = 0; f < KS; ++f)             // whatever stands where no query is stays in that lane's column, which `live` clears
      qf[n][f] = *reinterpret_cast<const frag_t<T> *>(reinterpret_cast<const T *>(p.q) + seq * p.q_b + (long)j * p.q_n +
                                                     (kvh * p.group + qhead[n]) * p.q_h + element<D, Q>(f, g));
  }
  if (biased) {
    if (tid < biases) bias[tid] = first_bias;
    for (int i = tid + WV * 64; i < biases; i += WV * 64) bias[i] = bias_at(i);
    if constexpr (WV == 1) __builtin_amdgcn_wave_barrier();
    else __syncthreads();
  }
  int mine[NB];                              // where the head's biases start
  float farthest[NB];
  int lowest = 1 << 30;                      // position of the first query here (none: beyond every row)
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    int hh = qhead[n] - gi0;
    if (hh < 0) hh += p.group;
    mine[n] = min(hh, max(heads - 1, 0)) * (reach + 1);
    farthest[n] = biased ? bias[mine[n] + reach] : 0.f;
    if (pos[n] >= 0) lowest = min(lowest, pos[n]);
  }
  lowest = wave_min_i32(lowest);

  f32x4 o[NB][DT] = {};
  float m[NB], l[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) { m[n] = -INFINITY; l[n] = 0.f; }
  const float scale2 = p.scale * LOG2E;

  for (int tile = from + wave; tile < to; tile += NT * WV) {
    f32x4 s[NB][2 * NT] = {};
    int k0[NT], end[NT], ahead[NT];
    bool far[NT], near = false, cut = false;
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const int at = tile + u * WV;
      far[u] = at < far_tiles;
      k0[u] = (far[u] ? at : at - far_tiles) * KT;
      end[u] = at < to ? (far[u] ? shared_len : own_len) : 0;
      // distance of a query at own row pos from key 0 of the tile: shared rows stand before the own ones
      ahead[u] = far[u] ? shared_len - k0[u] : -k0[u];
      near |= biased && lowest + ahead[u] - (KT - 1) < reach;
      cut |= k0[u] + KT > end[u] || (!far[u] && k0[u] + KT > lowest + 1);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          const frag_t<T> kf = fl[u].key(t, i);
#pragma unroll
          for (int n = 0; n < NB; ++n) s[n][2 * u + t] = mma16(kf, qf[n][i], s[n][2 * u + t]);
        }
      fl[u].put_v(vt + u * TB, min(end[u] - k0[u], KT), lane);
    }
#pragma unroll
    for (int u = 0; u < NT; ++u)
      if (tile + (NT + u) * WV < to) fetch(fl[u], tile + (NT + u) * WV);
    frag_t<T> pf[NB][NT], rest[NB][TWO ? NT : 1];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float x[8 * NT];
#pragma unroll
      for (int j = 0; j < 8 * NT; ++j) x[j] = __builtin_fmaf(s[n][j >> 2][j & 3], scale2, near ? 0.f : farthest[n]);
      if (near) {
#pragma unroll
        for (int j = 0; j < 8 * NT; ++j) x[j] += bias[mine[n] + min(max(pos[n] + ahead[j >> 3] - 8 * g - (j & 7), 0), reach)];
      }
      if (cut) {
#pragma unroll
        for (int j = 0; j < 8 * NT; ++j)
          if (k0[j >> 3] + 8 * g + (j & 7) >= (far[j >> 3] ? end[j >> 3] : min(end[j >> 3], pos[n] + 1))) x[j] = -INFINITY;
      }
      float top = x[0];
#pragma unroll
      for (int j = 1; j < 8 * NT; ++j) top = fmaxf(top, x[j]);
      if (__any(top > m[n] + SLACK)) {       // exponentials up to 2^SLACK are as good as up to 1: the maximum seldom moves
        const float now = fmaxf(m[n], max_groups(top));
        const float keep = now == -INFINITY ? 1.f : exp2_(m[n] - now);
        m[n] = now;
        l[n] *= keep;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[n][d][r] *= keep;
      }
      const float base = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        f32x8 e;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          e[j] = exp2_(x[8 * u + j] - base);
          l[n] += e[j];
        }
        pf[n][u] = to_frag<T>(e);
        if constexpr (TWO) {
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] -= (float)pf[n][u][j];
          rest[n][u] = to_frag<T>(e);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const frag_t<T> vf = TL::col_frag(vt + u * TB, 8 * g, 16 * d, lane);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          o[n][d] = mma16(vf, pf[n][u], o[n][d]);
          if constexpr (TWO) o[n][d] = mma16(vf, rest[n][u], o[n][d]);
        }
      }
    __builtin_amdgcn_wave_barrier();
  }

  // Results: of this piece, [shared rows' | own rows'] [row][piece][D + 4] = unnormalised output, maximum, sum; or the outputs.
  auto put = [&](int r, int e, f32x4 x, float top, float sum) {
    if (p.direct) {
      const int sub = shared ? r / per : 0, in = r - sub * per, gi = p.t == 1 ? in : in / p.t;
      const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] *= inv;
      const long at = (((long)(shared ? unit * p.each + sub : unit) * p.t + in - gi * p.t) * p.h + kvh * p.group + gi) * D + 4 * e;
      *reinterpret_cast<vec4_t<T> *>(reinterpret_cast<T *>(p.out) + at) = to_vec4<T>(x);
    } else {
      const long base_row = shared ? 0 : (long)p.shared_splits * p.b * p.hkv * per;
      float *to_ = p.part + (base_row + (((long)unit * p.hkv + kvh) * rows + r) * splits + piece) * (D + 4);
      *reinterpret_cast<f32x4 *>(to_ + 4 * e) = x;
      if (e == 0) { to_[D] = top; to_[D + 1] = sum; }
    }
  };
  if constexpr (WV == 1) {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const float sum = sum_groups(l[n]);
      const bool live = pos[n] >= 0;                                        // what is no query has seen the shared rows for nothing
      if (r0 + 16 * n + col < rows)
#pragma unroll
        for (int d = 0; d < DT; ++d) put(r0 + 16 * n + col, 4 * d + g, live ? o[n][d] : f32x4{}, live ? m[n] : -INFINITY, live ? sum : 0.f);
    }
    return;
  }
  // join the four waves, one block of 16 rows at a time: a wave leaves its output, scaled to the common maximum, in LDS
  float *mine_o = reinterpret_cast<float *>(lds);                           // [WAVES][16][D]; the V tiles are done with
  float *stat = bias + biases;                                              // [2][WAVES][16]
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const bool live = pos[n] >= 0;
    const float sum = live ? sum_groups(l[n]) : 0.f;
    if (!live) m[n] = -INFINITY;
    __syncthreads();
    if (g == 0) {
      stat[wave * 16 + col] = m[n];
      stat[(WAVES + wave) * 16 + col] = sum;
    }
    __syncthreads();
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, stat[w * 16 + col]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) total += stat[(WAVES + w) * 16 + col] * exp2_(stat[w * 16 + col] - base);
    const float keep = exp2_(m[n] - base);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      f32x4 x;
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = live ? o[n][d][r] * keep : 0.f;
      // 16-byte slots of a row rotate with the row: the 16 rows of a store instruction spread over the banks
      *reinterpret_cast<f32x4 *>(mine_o + (wave * 16 + col) * D + ((4 * d + g + col) % (D / 4)) * 4) = x;
    }
    __syncthreads();
    constexpr int PER = D / 4;                                              // 16-byte slots of a row
    if (g == 0 && wave == 0) { stat[col] = top; stat[WAVES * 16 + col] = total; }
    __syncthreads();
    for (int i = tid; i < 16 * PER; i += WAVES * 64) {
      const int c = i / PER, e = i - c * PER, r = r0 + 16 * n + c;
      if (r >= rows) continue;
      f32x4 x = {};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const f32x4 y = *reinterpret_cast<const f32x4 *>(mine_o + (w * 16 + c) * D + ((e + c) % PER) * 4);
#pragma unroll
        for (int q = 0; q < 4; ++q) x[q] += y[q];
      }
      put(r, e, x, stat[c], stat[WAVES * 16 + c]);
    }
  }
}

// Waves a SIMD: a wave's loads hide behind another one's arithmetic (f32 keeps its registers: 512 a lane).
template <typename T> constexpr int resident(int d) { return sizeof(T) == 4 ? 1 : d == 64 ? 3 : 2; }

template <typename T, int D, bool Q, int NB, int WV>
__global__ __launch_bounds__(WAVES * 64, resident<T>(D)) void decode_kernel(const DecodeParams p) {
  extern __shared__ __align__(16) char lds[];
  if ((int)blockIdx.x < p.shared_items) {
    walk<T, D, Q, NB, WAVES>(p, blockIdx.x, true, lds);
  } else {
    const int item = (blockIdx.x - p.shared_items) * (WAVES / WV) + (WV == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
    if (item < p.own_items) walk<T, D, Q, 1, WV>(p, item, false, lds);
  }
}

// Joins the pieces of a row, shared ones first.  A wave owns a row: lane i weighs piece i (64 at a time), then groups of D / 4
// lanes add every (64 / (D / 4))-th piece and the groups are added in their order.
template <typename T, int D>
__global__ __launch_bounds__(256) void decode_join_kernel(const DecodeParams p) {
  constexpr int PER = D / 4, GROUPS = 64 / PER, STEP = D + 4;
  __shared__ float weight[4][64];
  __shared__ __align__(16) float partial[4][GROUPS][D];
  const int per = p.group * p.t, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = blockIdx.x * 4 + wave;                                     // (sequence, key head, head of the group, token)
  if (row >= p.b * p.hkv * per) return;
  const int in = row % per, kvh = row / per % p.hkv, seq = row / per / p.hkv;
  const int far_tiles = p.each ? tiles_of(clamp_rows(p.shared_lengths[seq / p.each], p.shared.capacity)) : 0;
  const int own_tiles = tiles_of(clamp_rows(p.lengths[seq], p.own.capacity)) + (p.joined ? far_tiles : 0);
  const int own_piece = piece_tiles(own_tiles, p.own_splits), own_n = max(1, (own_tiles + own_piece - 1) / own_piece);
  const float *own = p.part + ((long)p.shared_splits * p.b * p.hkv * per + (long)row * p.own_splits) * STEP;
  int far_n = 0;
  const float *far = nullptr;
  if (p.shared_splits) {
    const int piece = piece_tiles(far_tiles, p.shared_splits);
    far_n = max(1, (far_tiles + piece - 1) / piece);
    far = p.part + ((((long)(seq / p.each) * p.hkv + kvh) * p.each + seq % p.each) * per + in) * p.shared_splits * STEP;
  }
  const int n = far_n + own_n, grp = lane / PER, e = lane % PER;
  float top = -INFINITY, sum = 0.f;
  f32x4 x = {};
  for (int first = 0; first < n; first += 64) {
    const int i = first + lane, last = min(n - first, 64);
    float m = -INFINITY, l = 0.f;
    if (i < n) {
      const float *piece = i < far_n ? far + (long)i * STEP : own + (long)(i - far_n) * STEP;
      m = piece[D];
      l = piece[D + 1];
    }
    float now = m;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) now = fmaxf(now, __shfl_xor(now, s));
    now = fmaxf(now, top);
    const float base = now == -INFINITY ? 0.f : now, keep = exp2_(top - base), w = exp2_(m - base);
    weight[wave][lane] = w;
    sum = sum * keep + wave_allreduce_sum_f32(l * w);
    top = now;
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] *= keep;
    __builtin_amdgcn_wave_barrier();
    if (grp < GROUPS) {
#pragma unroll 4
      for (int j = grp; j < last; j += GROUPS) {
        const int k = first + j;
        const float *piece = k < far_n ? far + (long)k * STEP : own + (long)(k - far_n) * STEP;
        const f32x4 y = *reinterpret_cast<const f32x4 *>(piece + 4 * e);
        const float wj = weight[wave][j];
#pragma unroll
        for (int q = 0; q < 4; ++q) x[q] = __builtin_fmaf(y[q], wj, x[q]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (grp < GROUPS) *reinterpret_cast<f32x4 *>(&partial[wave][grp][4 * e]) = x;
  __builtin_amdgcn_wave_barrier();
  if (lane < PER) {
#pragma unroll
    for (int s = 1; s < GROUPS; ++s) {
      const f32x4 y = *reinterpret_cast<const f32x4 *>(&partial[wave][s][4 * lane]);
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] += y[q];
    }
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] *= inv;
    const long at = (((long)seq * p.t + in % p.t) * p.h + kvh * p.group + in / p.t) * D + 4 * lane;
    *reinterpret_cast<vec4_t<T> *>(reinterpret_cast<T *>(p.out) + at) = to_vec4<T>(x);
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------------
struct Plan {
  int nb, wv, own_splits, shared_splits, own_tiles, shared_tiles, shared_items, own_items, own_heads, shared_heads, joined, direct;
  size_t lds;
};

int check(const char *where, const sig3d_decode_attention_args *a) {
  LANG_NEED(where, a != nullptr, "no arguments");
  LANG_NEED(where, a->dtype >= 0 && a->dtype <= 2, "dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
  LANG_NEED(where, a->d == 64 || a->d == 96 || a->d == 128, "head size must be 64, 96 or 128");
  LANG_NEED(where, a->b >= 1 && a->t >= 1 && a->h >= 1 && a->hkv >= 1 && a->capacity >= 1, "sizes must be positive");
  LANG_NEED(where, a->h % a->hkv == 0, "heads must be a multiple of key heads");
  LANG_NEED(where, a->capacity <= (1 << 29) && a->shared_capacity <= (1 << 29), "at most 2^29 rows");
  LANG_NEED(where, a->groups >= 0 && (a->groups == 0 || a->b % a->groups == 0), "groups must divide the batch");
  LANG_NEED(where, a->groups == 0 || a->shared_capacity >= 1, "shared sequences without rows");
  LANG_NEED(where, (long)a->b * a->t * a->h < (1l << 24), "too many query rows");
  return check_buckets(where, a->buckets, a->table, a->table_rows);
}

// Blocks of 16 query rows a workgroup takes over shared keys: what leaves registers for two waves a SIMD and more (four blocks:
// 64 questions over 5000 shared rows, 64 wide, took 39 us instead of 36).
constexpr int BLOCKS = 2;

Plan plan(const sig3d_decode_attention_args *a) {
  Plan s = {};
  const int group = a->h / a->hkv, per = group * a->t, each = a->groups ? a->b / a->groups : 0;
  const int reach = a->buckets.n ? std::max(1, a->buckets.border[a->buckets.n - 1]) : 0;
  const int e = a->dtype == 0 ? 4 : 2, row = a->d * e + 32;
  // V tiles (they also hold the four waves' outputs while these join: 16 rows of d floats each, less), statistics of the join
  const size_t tiles_bytes = WAVES * KT * row * (a->d == 64 && e == 2 ? 2 : 1) + 2 * WAVES * 16 * 4;
  s.own_tiles = sig3d_ceil_div(per, 16);
  const long base = (long)a->b * a->hkv * s.own_tiles;
  // Walking the shared rows once a sequence costs nothing where no other sequence shares them, and one launch instead of two
  // where they are short.
  s.joined = each > 0 && (each == 1 || a->shared_capacity <= 256);
  s.nb = 1;
  const int own_rows = a->capacity + (s.joined ? a->shared_capacity : 0);
  // About four workgroups of own rows for every CU (more pieces: more starts and joins; 8 ragged contexts of up to 30 000 rows took
  // 79 us with 4096 workgroups, 72 with 1024), and one of shared rows: they are the long ones, and what a workgroup costs before
  // and after its tiles is spread over more of them (2 scenes, 48 questions: 75 us with 768, 60 with 256).
  s.own_splits = (int)std::min<long>(std::max<long>(1, 1024 / base), sig3d_ceil_div(own_rows, LEAST * KT));
  if (each > 0 && !s.joined) {
    const long rows = (long)each * per;
    // (one block of rows where the biases of two would not fit: many heads and a far reach)
    const size_t biases = a->buckets.n ? (size_t)std::min(group, (16 * BLOCKS + a->t - 2) / a->t + 1) * (reach + 1) * 4 : 0;
    s.nb = rows > 16 && tiles_bytes + biases <= MOST_LDS ? BLOCKS : 1;
    s.shared_tiles = sig3d_ceil_div(rows, 16 * s.nb);
    const long far = (long)a->groups * a->hkv * s.shared_tiles;
    s.shared_splits = (int)std::min<long>(std::max<long>(1, 256 / far), sig3d_ceil_div(a->shared_capacity, LEAST * KT));
    s.shared_items = (int)(far * s.shared_splits);
  }
  s.own_items = (int)(base * s.own_splits);
  s.direct = s.own_splits == 1 && !s.shared_splits;
  if (a->buckets.n) {
    s.own_heads = std::min(group, (16 + a->t - 2) / a->t + 1);
    s.shared_heads = s.shared_splits ? std::min(group, (16 * s.nb + a->t - 2) / a->t + 1) : 0;
  }
  // One wave an item where a sequence is short: four would start and join for a tile or two each.
  const size_t one = (size_t)WAVES * s.own_heads * (reach + 1) * 4;
  s.wv = one <= 32 * 1024 && (own_rows <= 2 * KT || (base >= 1024 && own_rows <= 16 * KT)) ? 1 : WAVES;
  s.lds = tiles_bytes + std::max(s.wv == 1 ? one : s.own_heads * (reach + 1) * 4ul, s.shared_heads * (reach + 1) * 4ul);
  return s;
}

template <typename T, int D, bool Q, int NB, int WV> int launch(const DecodeParams &p, const Plan &s, hipStream_t stream) {
  static sig3d_once_per_device once;
  if (int e = allow_lds(decode_kernel<T, D, Q, NB, WV>, once)) return e;
  decode_kernel<T, D, Q, NB, WV><<<s.shared_items + sig3d_ceil_div(s.own_items, WAVES / WV), WAVES * 64, s.lds, stream>>>(p);
  SIG3D_LAUNCH_CHECK("decode_kernel");
  if (!p.direct) {
    decode_join_kernel<T, D><<<sig3d_ceil_div((long)p.b * p.h * p.t, 4), 256, 0, stream>>>(p);
    SIG3D_LAUNCH_CHECK("decode_join_kernel");
  }
  return 0;
}

}  // namespace

extern "C" long sig3d_decode_attention_work_floats(const sig3d_decode_attention_args *a) {
  if (check("sig3d_decode_attention_work_floats", a)) return -1;
  const Plan s = plan(a);
  return s.direct ? 0 : (long)a->b * a->t * a->h * (s.own_splits + s.shared_splits) * (a->d + 4);
}

extern "C" int sig3d_decode_attention(const sig3d_decode_attention_args *a, void *stream) {
  if (int e = check("sig3d_decode_attention", a)) return e;
  const Plan s = plan(a);
  SIG3D_REQUIRE(a->q && a->out && a->k_cache && a->v_cache && a->lengths && (s.direct || a->work), "missing array");
  SIG3D_REQUIRE(a->groups == 0 || (a->shared_k && a->shared_v && a->shared_lengths), "missing shared array");
  const bool quantized = a->k_scale != nullptr;
  SIG3D_REQUIRE((a->v_scale != nullptr) == quantized && (a->groups == 0 || ((a->shared_k_scale != nullptr) == quantized &&
                (a->shared_v_scale != nullptr) == quantized)), "own and shared rows must be held alike");
  SIG3D_REQUIRE(aligned16(a->q) && aligned16(a->out) && aligned16(a->k_cache) && aligned16(a->v_cache) && aligned16(a->shared_k) &&
                aligned16(a->shared_v) && aligned16(a->work), "addresses must be 16-byte aligned");
  const int e = a->dtype == 0 ? 4 : 2;
  SIG3D_REQUIRE(a->q_b >= 0 && a->q_n >= 0 && a->q_h >= 0 && a->q_b * e % 16 == 0 && a->q_n * e % 16 == 0 && a->q_h * e % 16 == 0,
                "strides must be non-negative multiples of 16 bytes");
  SIG3D_REQUIRE((long)a->b * a->hkv * s.own_tiles * s.own_splits + s.shared_items < INT_MAX, "grid too large");
  SIG3D_REQUIRE(s.lds <= MOST_LDS, "biases too large for LDS");      // (no call: 16 heads, the longest rows and the farthest reach take 136 KB)
  DecodeParams p = {};
  p.q = a->q; p.table = a->table;
  p.own = {a->k_cache, a->v_cache, a->k_scale, a->v_scale, a->capacity};
  p.shared = {a->shared_k, a->shared_v, a->shared_k_scale, a->shared_v_scale, a->shared_capacity};
  p.lengths = a->lengths; p.shared_lengths = a->shared_lengths; p.counts = a->counts;
  p.out = a->out; p.part = a->work;
  p.q_b = a->q_b; p.q_n = a->q_n; p.q_h = a->q_h;
  p.b = a->b; p.t = a->t; p.h = a->h; p.hkv = a->hkv; p.group = a->h / a->hkv;
  p.each = a->groups ? a->b / a->groups : 0;
  p.own_splits = s.own_splits; p.shared_splits = s.shared_splits; p.own_tiles = s.own_tiles; p.shared_tiles = s.shared_tiles;
  p.own_items = s.own_items; p.shared_items = s.shared_items; p.own_bias_heads = s.own_heads; p.shared_bias_heads = s.shared_heads;
  p.joined = s.joined; p.direct = s.direct;
  p.scale = a->scale;
  p.bk = device_buckets(a->buckets);
  return by_type(a->dtype, a->d, [&](auto t, auto d) {
    typedef decltype(t) T;
    constexpr int D = decltype(d)::value;
    const auto go = [&](auto q, auto nb, auto wv) {
      return launch<T, D, decltype(q)::value, decltype(nb)::value, decltype(wv)::value>(p, s, (hipStream_t)stream);
    };
    const auto by_rows = [&](auto q) {
      const std::integral_constant<int, 1> one;
      const std::integral_constant<int, BLOCKS> some;
      const std::integral_constant<int, WAVES> all;
      if (s.nb == 1) return s.wv == 1 ? go(q, one, one) : go(q, one, all);
      return s.wv == 1 ? go(q, some, one) : go(q, some, all);
    };
    return quantized ? by_rows(std::true_type()) : by_rows(std::false_type());
  });
}
