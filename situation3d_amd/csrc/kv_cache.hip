// kv_cache.hip -- writing the key / value cache, quantised on the way, and reading it back, for gfx950.
//
// A row is one (sequence, key head, token): d values.  Held as e4m3 it costs d bytes and one f32 scale, a power of two:
//   scale = 2^e, e smallest with max |x| <= 448 * 2^e;   held = e4m3(x / scale), to nearest even.
// With a power of two the quotient and the value read back are exact, so writing a value that came out of the cache gives it
// again, and the 4 significant bits are the only rounding (half a step: 2^-4 of the value).
//
// Both directions move bytes and do next to no arithmetic: HBM bound.  The cache is head-major, (b, hkv, capacity, d), so
// that a decoding workgroup streams one contiguous run; tokens arrive and leave token-major.  Work is ordered (sequence,
// head, token): cache traffic is contiguous, and the token-major side moves whole rows of d elements (128 bytes and more).
#include "lang_core.h"

namespace {
using namespace lang;

struct AppendParams {
  const void *k, *v;
  void *k_cache, *v_cache;
  float *k_scale, *v_scale;
  const int *start, *counts;
  int *lengths;
  long k_b, k_n, k_h, v_b, v_n, v_h;
  int t, capacity, hkv;
};

// LANES neighbouring lanes hold a row, one 16-byte piece each (of 96 elements: 12 of 16 lanes, 24 of 32): a load instruction
// moves whole rows.  (Four lanes with every fourth piece: 64 bytes of a row at a time, 72 us for 8192 x 4 x 8 rows of 128
// floats instead of 70, and as much for the read: 72 instead of 46.)
template <typename T, int D> struct Piece {
  static constexpr int PER = 16 / (int)sizeof(T), USED = D / PER, LANES = USED <= 8 ? 8 : USED <= 16 ? 16 : 32;
  typedef T piece __attribute__((ext_vector_type(PER)));
  static __device__ __forceinline__ float over_lanes(float top) {
    top = fmaxf(top, __builtin_bit_cast(float, dpp_i32<0xB1>(__builtin_bit_cast(int, top))));
    top = fmaxf(top, __builtin_bit_cast(float, dpp_i32<0x4E>(__builtin_bit_cast(int, top))));
    top = fmaxf(top, __builtin_bit_cast(float, dpp_i32<0x141>(__builtin_bit_cast(int, top))));
    if constexpr (LANES >= 16) top = fmaxf(top, __builtin_bit_cast(float, dpp_i32<0x140>(__builtin_bit_cast(int, top))));
    if constexpr (LANES == 32) top = fmaxf(top, __shfl_xor(top, 16));
    return top;
  }
  // The largest value of 4 significant bits that T holds.  Beyond it the nearest such value may be 2^16 (f16) or 2^128, which
  // would come back as an infinity: values up to T's largest are brought down to it, by less than 2^-4 of theirs.
  static constexpr float LIMIT = std::is_same<T, _Float16>::value ? 61440.f : 0x1.ep127f;
  // A row's e4m3 values, and its scale by its first lane.  Infinities and NaN do not count in the scale; infinities become the
  // largest value that the scale and T allow.  Only a wave with values beyond LIMIT looks.
  static __device__ __forceinline__ void quantize(unsigned char *to, float *scale, piece x, bool mine, bool first) {
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) top = fmaxf(top, fabsf((float)x[e]));        // fmaxf drops NaN
    top = over_lanes(top);
    const bool beyond = __any(top > LIMIT);
    if (beyond) {
      top = 0.f;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const float a = fabsf((float)x[e]);
        top = a < INFINITY ? fmaxf(top, a) : top;
      }
      top = fminf(over_lanes(top), LIMIT);
    }
    // top = m 2^x with m in [0.5, 1), 448 = 0.875 2^9; scales stay normal numbers
    const int ex = __builtin_amdgcn_frexp_expf(top) - 9 + (__builtin_amdgcn_frexp_mantf(top) > 0.875f ? 1 : 0);
    const int exponent = top > 0.f ? max(ex, -126) : 0;
    const float inv = __builtin_ldexpf(1.f, -exponent);
    float y[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) y[e] = (float)x[e] * inv;
    if (beyond) {
      const float most = fminf(448.f, LIMIT * inv);
#pragma unroll
      for (int e = 0; e < PER; ++e) y[e] = fabsf(y[e]) > most ? copysignf(most, y[e]) : y[e];
    }
    unsigned w[PER / 4];
#pragma unroll
    for (int g = 0; g < PER / 4; ++g) {
      const int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * g], y[4 * g + 1], 0, false);
      w[g] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * g + 2], y[4 * g + 3], p, true);
    }
    if (mine) {
      if constexpr (PER == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[PER / 4 - 1]);
      else *reinterpret_cast<unsigned *>(to) = w[0];
    }
    if (first) *scale = __builtin_ldexpf(1.f, exponent);
  }
};

// Rows a thread has in flight.  Reads wait on memory (3000 cycles a request at 3.5 TB/s in total); 1, 2 and 4 rows, tokens before
// heads and heads before tokens all measured within 10 %.
constexpr int UNROLL = 2;

// grid (blocks of rows, b).  One block a sequence, or `start` given: lengths is updated here, after everyone has read it.
template <typename T, int D, bool Q>
__global__ __launch_bounds__(256) void cache_append_kernel(const AppendParams p) {
  typedef Piece<T, D> P;
  constexpr int ROWS = 256 / P::LANES;
  const int b = blockIdx.y, l = threadIdx.x % P::LANES, rows = p.hkv * p.t;
  const int first = p.start ? p.start[b] : p.lengths[b];
  const int count = p.counts ? min(max(p.counts[b], 0), p.t) : p.t;
  const bool mine = P::USED == P::LANES || l < P::USED;
  for (int r0 = blockIdx.x * ROWS * UNROLL + threadIdx.x / P::LANES; r0 < rows; r0 += gridDim.x * ROWS * UNROLL) {
    typename P::piece k[UNROLL], v[UNROLL];
    long row[UNROLL];                                              // of the cache; negative: nothing to do (a row's lanes agree)
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int r = min(r0 + u * ROWS, rows - 1), head = r / p.t, i = r - head * p.t;
      const long to = (long)first + i;
      row[u] = r0 + u * ROWS < rows && i < count && to >= 0 && to < p.capacity ? ((long)b * p.hkv + head) * p.capacity + to : -1;
      // no condition on a load (it would be waited for inside): what is not to be moved repeats the last token that is
      const int from = min(i, max(count - 1, 0)), e = min(l, P::USED - 1) * P::PER;
      k[u] = *reinterpret_cast<const typename P::piece *>(reinterpret_cast<const T *>(p.k) + b * p.k_b + from * p.k_n + head * p.k_h + e);
      v[u] = *reinterpret_cast<const typename P::piece *>(reinterpret_cast<const T *>(p.v) + b * p.v_b + from * p.v_n + head * p.v_h + e);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (row[u] < 0) continue;
      const long at = row[u] * D + l * P::PER;
      if constexpr (Q) {
        P::quantize(reinterpret_cast<unsigned char *>(p.k_cache) + at, p.k_scale + row[u], k[u], mine, l == 0);
        P::quantize(reinterpret_cast<unsigned char *>(p.v_cache) + at, p.v_scale + row[u], v[u], mine, l == 0);
      } else if (mine) {
        *reinterpret_cast<typename P::piece *>(reinterpret_cast<T *>(p.k_cache) + at) = k[u];
        *reinterpret_cast<typename P::piece *>(reinterpret_cast<T *>(p.v_cache) + at) = v[u];
      }
    }
  }
  if (gridDim.x == 1 || p.start) {
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x == 0) p.lengths[b] = (int)min(max((long)first + count, 0l), (long)p.capacity);
  }
}

__global__ __launch_bounds__(256) void cache_advance_kernel(int b, int t, int capacity, const int *counts, int *lengths) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= b) return;
  const int count = counts ? min(max(counts[i], 0), t) : t;
  lengths[i] = (int)min(max((long)lengths[i] + count, 0l), (long)capacity);
}

struct ReadParams {
  const void *k, *v;
  const float *k_scale, *v_scale;
  const int *lengths;
  void *k_out, *v_out;
  int n, capacity, hkv;
};

// a thread: 16 bytes of a K row of the result and of the V row beside it.  grid (pieces / 256, hkv, b)
template <typename T, int D, bool Q>
__global__ __launch_bounds__(256) void cache_read_kernel(const ReadParams p) {
  typedef Piece<T, D> P;
  typedef typename P::piece piece;
  const unsigned c = blockIdx.x * 256 + threadIdx.x;              // below 2^31 + 256: the host looks
  const int i = c / P::USED, o = c - i * P::USED;
  if (i >= p.n) return;
  const int b = blockIdx.z, head = blockIdx.y;
  piece k{}, v{};
  if (i < p.lengths[b]) {
    const long row = ((long)b * p.hkv + head) * p.capacity + i, at = row * D + o * P::PER;
    if constexpr (Q) {
      const unsigned *kp = reinterpret_cast<const unsigned *>(reinterpret_cast<const unsigned char *>(p.k) + at);
      const unsigned *vp = reinterpret_cast<const unsigned *>(reinterpret_cast<const unsigned char *>(p.v) + at);
      const float ks = p.k_scale[row], vs = p.v_scale[row];
      if constexpr (P::PER == 8) {
        k = from_e4m3<T>(*reinterpret_cast<const uint2 *>(kp), ks);
        v = from_e4m3<T>(*reinterpret_cast<const uint2 *>(vp), vs);
      } else {
        k = __builtin_shufflevector(from_e4m3<T>(make_uint2(*kp, 0), ks), f32x8{}, 0, 1, 2, 3);
        v = __builtin_shufflevector(from_e4m3<T>(make_uint2(*vp, 0), vs), f32x8{}, 0, 1, 2, 3);
      }
    } else {
      k = *reinterpret_cast<const piece *>(reinterpret_cast<const T *>(p.k) + at);
      v = *reinterpret_cast<const piece *>(reinterpret_cast<const T *>(p.v) + at);
    }
  }
  const long to = (((long)b * p.n + i) * p.hkv + head) * D + o * P::PER;
  *reinterpret_cast<piece *>(reinterpret_cast<T *>(p.k_out) + to) = k;
  *reinterpret_cast<piece *>(reinterpret_cast<T *>(p.v_out) + to) = v;
}

int check_cache(const char *where, int dtype, int b, int capacity, int hkv, int d) {
  LANG_NEED(where, dtype >= 0 && dtype <= 2, "dtype must be 0 (f32), 1 (bf16) or 2 (f16)");
  LANG_NEED(where, d == 64 || d == 96 || d == 128, "head size must be 64, 96 or 128");
  LANG_NEED(where, b >= 1 && b <= 65535 && hkv >= 1 && hkv <= 65535 && capacity >= 1, "sizes out of range");
  return 0;
}

}  // namespace

extern "C" int sig3d_cache_append(const sig3d_cache_append_args *a, void *stream) {
  SIG3D_REQUIRE(a != nullptr, "no arguments");
  if (int e = check_cache("sig3d_cache_append", a->dtype, a->b, a->capacity, a->hkv, a->d)) return e;
  SIG3D_REQUIRE(a->t >= 1 && (long)a->t * a->hkv < (1l << 30), "token count out of range");
  SIG3D_REQUIRE(a->k && a->v && a->k_cache && a->v_cache && a->lengths, "missing array");
  SIG3D_REQUIRE((a->k_scale == nullptr) == (a->v_scale == nullptr), "k_scale and v_scale come together");
  SIG3D_REQUIRE(aligned16(a->k) && aligned16(a->v) && aligned16(a->k_cache) && aligned16(a->v_cache),
                "addresses must be 16-byte aligned");
  const auto apart = [&](const int *x) { return !x || x + a->b <= a->lengths || x >= a->lengths + a->b; };
  SIG3D_REQUIRE(apart(a->start) && apart(a->counts), "start and counts must not lie in lengths, which the call writes");
  const int e = a->dtype == 0 ? 4 : 2;
  const long strides[6] = {a->k_b, a->k_n, a->k_h, a->v_b, a->v_n, a->v_h};
  for (long s : strides) SIG3D_REQUIRE(s >= 0 && s * e % 16 == 0, "strides must be non-negative multiples of 16 bytes");
  const AppendParams p = {a->k, a->v, a->k_cache, a->v_cache, a->k_scale, a->v_scale, a->start, a->counts, a->lengths,
                          a->k_b, a->k_n, a->k_h, a->v_b, a->v_n, a->v_h, a->t, a->capacity, a->hkv};
  const int rows = a->hkv * a->t;
  // without `start` every workgroup of a sequence reads the length that the call moves: one workgroup up to 512 rows (a
  // decoding step: 32 heads are half a pass), else a launch of its own moves it
  const bool one = !a->start && rows <= 512;
  const int piece = a->dtype == 0 ? 4 : 8, lanes = a->d / piece <= 8 ? 8 : a->d / piece <= 16 ? 16 : 32;
  const dim3 grid(one ? 1 : sig3d_ceil_div(rows, 256 / lanes * UNROLL), a->b);
  const int err = by_type(a->dtype, a->d, [&](auto t, auto d) {
    typedef decltype(t) T;
    constexpr int D = decltype(d)::value;
    if (a->k_scale) cache_append_kernel<T, D, true><<<grid, 256, 0, (hipStream_t)stream>>>(p);
    else cache_append_kernel<T, D, false><<<grid, 256, 0, (hipStream_t)stream>>>(p);
    SIG3D_LAUNCH_CHECK("cache_append_kernel");
    return 0;
  });
  if (err || grid.x == 1 || a->start) return err;
  cache_advance_kernel<<<sig3d_ceil_div(a->b, 256), 256, 0, (hipStream_t)stream>>>(a->b, a->t, a->capacity, a->counts, a->lengths);
  SIG3D_LAUNCH_CHECK("cache_advance_kernel");
  return 0;
}

extern "C" int sig3d_cache_read(const sig3d_cache_read_args *a, void *stream) {
  SIG3D_REQUIRE(a != nullptr, "no arguments");
  if (int e = check_cache("sig3d_cache_read", a->dtype, a->b, a->capacity, a->hkv, a->d)) return e;
  SIG3D_REQUIRE(a->n >= 1 && a->n <= a->capacity && (long)a->n * a->d < (1l << 33), "row count out of range");
  SIG3D_REQUIRE(a->k_cache && a->v_cache && a->lengths && a->k_out && a->v_out, "missing array");
  SIG3D_REQUIRE((a->k_scale == nullptr) == (a->v_scale == nullptr), "k_scale and v_scale come together");
  SIG3D_REQUIRE(aligned16(a->k_cache) && aligned16(a->v_cache) && aligned16(a->k_out) && aligned16(a->v_out),
                "addresses must be 16-byte aligned");
  const ReadParams p = {a->k_cache, a->v_cache, a->k_scale, a->v_scale, a->lengths, a->k_out, a->v_out, a->n, a->capacity, a->hkv};
  const dim3 grid(sig3d_ceil_div((long)a->n * (a->d / (a->dtype == 0 ? 4 : 8)), 256), a->hkv, a->b);
  return by_type(a->dtype, a->d, [&](auto t, auto dd) {
    typedef decltype(t) T;
    constexpr int D = decltype(dd)::value;
    if (a->k_scale) cache_read_kernel<T, D, true><<<grid, 256, 0, (hipStream_t)stream>>>(p);
    else cache_read_kernel<T, D, false><<<grid, 256, 0, (hipStream_t)stream>>>(p);
    SIG3D_LAUNCH_CHECK("cache_read_kernel");
    return 0;
  });
}
