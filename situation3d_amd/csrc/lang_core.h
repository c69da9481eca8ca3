// lang_core.h -- what the language-side attention kernels (rel_attention.hip, decode_attention.hip, kv_cache.hip) share:
// element types, matrix-core steps over one register layout, LDS tiles, relative-position buckets, visible key intervals.
//
// One register layout serves bf16, f16 and f32.  A fragment is 8 consecutive reduction indices of one row: for the 32-wide
// products lane (row = lane & 31, half = lane >> 5) holds indices 8 half .. 8 half + 7 of a 16-index step.  bf16 / f16 feed
// it to one 32x32x16 instruction; f32 feeds element j to the j-th of eight 32x32x2 instructions, whose two reduction
// indices are then {j, 8 + j}: the same sixteen products, exact f32.
//
// Accumulators (C map: col = lane & 31, row = (r & 3) + 8 (r >> 2) + 4 half) become the next product's B operand without any
// lane exchange: the A rows of the first product are read in the order kappa(m) = m with bits 2 and 3 swapped, so register r
// of a lane stands for row 16 (r >> 3) + 8 half + (r & 7), and registers 0..7 / 8..15 ARE two fragments.
#pragma once
#include "sig3d_common.h"

#include <type_traits>

namespace lang {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f;

template <typename T> struct Num;
template <> struct Num<__bf16> { typedef bf16x8 frag; typedef bf16x4 quad; };
template <> struct Num<_Float16> { typedef f16x8 frag; typedef f16x4 quad; };
template <> struct Num<float> { typedef f32x8 frag; typedef f32x4 quad; };
template <typename T> using frag_t = typename Num<T>::frag;
template <typename T> using vec4_t = typename Num<T>::quad;

__device__ __forceinline__ f32x16 mma32(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma32(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}
// 16-wide form: lane (row = lane & 15, g = lane >> 4) holds reduction indices 8 g .. 8 g + 7 of a 32-index step; C map:
// col = lane & 15, row = 4 g + r.
__device__ __forceinline__ f32x4 mma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// f32 -> T, round to nearest even
template <typename T> __device__ __forceinline__ frag_t<T> to_frag(f32x8 x) { return __builtin_convertvector(x, frag_t<T>); }
template <typename T> __device__ __forceinline__ vec4_t<T> to_vec4(f32x4 x) { return __builtin_convertvector(x, vec4_t<T>); }
template <> __device__ __forceinline__ f32x8 to_frag<float>(f32x8 x) { return x; }
template <> __device__ __forceinline__ f32x4 to_vec4<float>(f32x4 x) { return x; }

// x of lane & 31 and of (lane & 31) + 32 (elements of the builtin's vector have to be copied out before a bit_cast)
__device__ __forceinline__ void both_halves(float x, float &lo, float &hi) {
  const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  const unsigned a = s[0], b = s[1];
  lo = __builtin_bit_cast(float, a);
  hi = __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float max_halves(float x) {
  float lo, hi;
  both_halves(x, lo, hi);
  return fmaxf(lo, hi);
}
__device__ __forceinline__ float sum_halves(float x) {
  float lo, hi;
  both_halves(x, lo, hi);
  return lo + hi;
}
// Waits for every load so far.  Before a loop: what was loaded ahead of it would else be waited for inside, by counts that also
// cover the loads which that iteration has just sent out.
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }      // vmcnt 0, the others free
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ int wave_min_i32(int v) { return -wave_allreduce_max_i32(-v); }
__device__ __forceinline__ int wave_max_i32(int v) { return wave_allreduce_max_i32(v); }

__device__ __forceinline__ int kappa(int m) { return (m & 0x13) | ((m & 4) << 1) | ((m & 8) >> 1); }
__device__ __forceinline__ int reg_row(int r, int half) { return 16 * (r >> 3) + 8 * half + (r & 7); }

// eight e4m3 values times a power of two
template <typename T> __device__ __forceinline__ frag_t<T> from_e4m3(uint2 w, float scale);
template <> __device__ __forceinline__ f32x8 from_e4m3<float>(uint2 w, float scale) {
  f32x8 f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const unsigned x = i ? w.y : w.x;
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x, scale, false);
    const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x, scale, true);
    f[4 * i] = lo[0]; f[4 * i + 1] = lo[1]; f[4 * i + 2] = hi[0]; f[4 * i + 3] = hi[1];
  }
  return f;
}
template <> __device__ __forceinline__ bf16x8 from_e4m3<__bf16>(uint2 w, float scale) {
  bf16x8 f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const unsigned x = i ? w.y : w.x;
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, false);
    const auto hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, true);
    f[4 * i] = lo[0]; f[4 * i + 1] = lo[1]; f[4 * i + 2] = hi[0]; f[4 * i + 3] = hi[1];
  }
  return f;
}
template <> __device__ __forceinline__ f16x8 from_e4m3<_Float16>(uint2 w, float scale) {
  f16x8 f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const unsigned x = i ? w.y : w.x;
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, scale, false);
    const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, scale, true);
    f[4 * i] = lo[0]; f[4 * i + 1] = lo[1]; f[4 * i + 2] = hi[0]; f[4 * i + 3] = hi[1];
  }
  return f;
}

// ---- LDS tiles ------------------------------------------------------------------------------------------------------
// [rows][D] of T in 16-byte chunks; chunk c of a row sits at c ^ swz(row).  swz separates, inside a 128-byte bank window,
// the eight rows that eight consecutive lanes of a fragment read touch (kappa order: 0-3, 8-11), and the four rows of a
// 16-lane group of a transposing read (32 bytes each).  Rows of 12 chunks (96 x 2 bytes) are padded to 16.
// PAD: a tile that is only read transposed has its rows 32 bytes further apart instead: the four rows of a group are as far
// apart, and every address is a lane's base plus a constant.
template <typename T, int D, bool PAD = false> struct Tile {
  static constexpr int CH = D * (int)sizeof(T) / 16;        // chunks of data in a row
  static constexpr int CHP = PAD ? CH + 2 : (CH + 7) / 8 * 8;       // chunks stored
  static constexpr int ROW = CHP * 16;                      // bytes
  static __device__ __forceinline__ int swz(int row) { return PAD ? 0 : ((row & 3) << 1) | ((row >> 3) & 1); }
  // (the upper bits of a chunk stay out of the exclusive or: they are constants of an unrolled loop, and of the instruction)
  static __device__ __forceinline__ int at(int row, int chunk) {
    return row * ROW + (((chunk & 7) ^ swz(row)) << 4) + ((chunk & ~7) << 4);
  }

  // elements 8 o .. 8 o + 7 of a row
  static __device__ __forceinline__ frag_t<T> row_frag(const char *t, int row, int o) {
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const frag_t<T> *>(t + at(row, o));
    } else {
      const f32x4 lo = *reinterpret_cast<const f32x4 *>(t + at(row, 2 * o));
      const f32x4 hi = *reinterpret_cast<const f32x4 *>(t + at(row, 2 * o + 1));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // lane of a 16-lane group: rows row0 .. row0 + 7 of column col0 + (lane & 15)   (row0 a multiple of 8, col0 of 16)
  static __device__ __forceinline__ frag_t<T> col_frag(const char *t, int row0, int col0, int lane) {
    if constexpr (sizeof(T) == 2) {
      // the transposing read hands lane i of a 16-lane group column i of a [4 rows][16 columns] block, lane i itself
      // addressing row i >> 2, columns 4 (i & 3) .. + 3
      const int li = lane & 15, row = row0 + (li >> 2), chunk = (col0 >> 3) + ((li & 3) >> 1), in = (li & 1) * 8;
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(t + at(row, chunk) + in));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(t + at(row + 4, chunk) + in));
      return __builtin_bit_cast(frag_t<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const int col = col0 + (lane & 15);
      f32x8 f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        f[j] = *reinterpret_cast<const float *>(t + at(row0 + j, col >> 2) + (col & 3) * 4);
      return f;
    }
  }
};

// ---- relative position buckets -----------------------------------------------------------------------------------------
// One direction has n buckets; border[i] is the smallest distance of bucket i (host-made from whole numbers), and from
// distance `reach` = border of the last bucket on nothing changes any more.  of[a]: the bucket of distance a <= reach, so that
// a kernel finds it with one load (counting borders costs 3 instructions each, for every wave of every workgroup).
struct Buckets {
  int n, reach, both;      // both: keys ahead of the query have buckets n .. 2 n - 1 of their own; else they share bucket 0
  short border[SIG3D_REL_MAX_BUCKETS];
  unsigned char of[SIG3D_REL_MAX_REACH + 4];
};
__device__ __forceinline__ int bucket_of(const Buckets &bk, int relative) {      // |relative| <= reach
  const int a = relative < 0 ? -relative : (bk.both ? relative : 0);
  return bk.of[a] + (bk.both && relative > 0 ? bk.n : 0);
}
// by_distance[r + reach + EDGE] = log2(e) * table[bucket(r)][head], for r in [-reach - EDGE, reach + EDGE]: a tile that any
// distance below `reach` touches stays inside, so that nobody clamps an index
constexpr int EDGE = 96;
__host__ __device__ constexpr int bias_floats(int reach) { return 2 * (reach + EDGE) + 1; }
// `start` sends a thread's first load out (two in a row: bucket, entry), `finish` puts the values where they belong: between
// the two there is time for everything else that a workgroup loads before it begins.
template <typename T> struct BiasFill {
  float first = 0.f;
  static __device__ __forceinline__ float value(const Buckets &bk, const T *table, int heads, int head, int i) {
    const int r = min(max(i - bk.reach - EDGE, -bk.reach), bk.reach);
    return (float)table[(long)bucket_of(bk, r) * heads + head] * LOG2E;
  }
  __device__ __forceinline__ void start(const Buckets &bk, const void *table, int heads, int head, int tid) {
    if (bk.n > 0) first = value(bk, reinterpret_cast<const T *>(table), heads, head, min(tid, bias_floats(bk.reach) - 1));
  }
  __device__ __forceinline__ void finish(float *by_distance, const Buckets &bk, const void *table, int heads, int head, int tid,
                                         int threads) const {
    if (bk.n <= 0) return;
    const int n = bias_floats(bk.reach);
    if (tid < n) by_distance[tid] = first;
    for (int i = tid + threads; i < n; i += threads)
      by_distance[i] = value(bk, reinterpret_cast<const T *>(table), heads, head, i);
  }
};

// ---- host side ---------------------------------------------------------------------------------------------------------
#define LANG_NEED(where, cond, msg)               \
  do {                                            \
    if (!(cond)) {                                \
      sig3d_set_error_msg(where, msg);            \
      return (int)hipErrorInvalidValue;           \
    }                                             \
  } while (0)

constexpr size_t MOST_LDS = 152 * 1024;       // of a workgroup, beside its static arrays

inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

inline int check_buckets(const char *where, const sig3d_rel_buckets &k, const void *table, int table_rows) {
  LANG_NEED(where, k.n >= 0 && k.n <= SIG3D_REL_MAX_BUCKETS, "too many buckets");
  if (k.n == 0) return 0;
  LANG_NEED(where, table != nullptr, "buckets without a table");
  LANG_NEED(where, table_rows >= k.n * (k.both ? 2 : 1), "table has too few rows");
  LANG_NEED(where, k.border[0] == 0, "border[0] must be 0");
  for (int i = 1; i < k.n; ++i) LANG_NEED(where, k.border[i] >= k.border[i - 1], "borders must not decrease");
  LANG_NEED(where, k.border[k.n - 1] <= SIG3D_REL_MAX_REACH, "borders beyond SIG3D_REL_MAX_REACH");
  return 0;
}

inline Buckets device_buckets(const sig3d_rel_buckets &k) {
  Buckets d = {};
  d.n = k.n;
  d.both = k.both;
  if (k.n > 0) d.reach = k.border[k.n - 1] > 0 ? k.border[k.n - 1] : 1;
  for (int i = 0; i < k.n; ++i) d.border[i] = (short)k.border[i];
  if (k.n > 0)
    for (int a = 0, i = 0; a <= d.reach; ++a) {
      while (i + 1 < k.n && k.border[i + 1] <= a) ++i;
      d.of[a] = (unsigned char)i;
    }
  return d;
}

// dynamic LDS up to what a CU has beside the kernels' static arrays
template <typename K> int allow_lds(K kernel, sig3d_once_per_device &once) {
  if (once.pending()) {
    SIG3D_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)MOST_LDS));
    once.done();
  }
  return 0;
}

template <typename F> int by_type(int dtype, int d, F f) {
  switch (dtype * 3 + (d - 64) / 32) {
    case 0: return f(float(), std::integral_constant<int, 64>());
    case 1: return f(float(), std::integral_constant<int, 96>());
    case 2: return f(float(), std::integral_constant<int, 128>());
    case 3: return f(__bf16(), std::integral_constant<int, 64>());
    case 4: return f(__bf16(), std::integral_constant<int, 96>());
    case 5: return f(__bf16(), std::integral_constant<int, 128>());
    case 6: return f(_Float16(), std::integral_constant<int, 64>());
    case 7: return f(_Float16(), std::integral_constant<int, 96>());
    default: return f(_Float16(), std::integral_constant<int, 128>());
  }
}

}  // namespace lang
