// Attention of a batch's new tokens over KV caches, split along the keys.
//
// A call has up to two key segments: a prefix that the sequences of a group
// share (segment 0) and every sequence's own cache (segment 1).  For a key /
// value head the rows of segment 0 are all query rows of all sequences of the
// group (group heads x new tokens x sequences), so a prefix key is read once
// for all of them; those of segment 1 are one sequence's.  The key axis of
// each segment is cut into `nsplit` ranges of `chunk` keys, a work item
// computes one range for one tile of rows, and cache_combine_kernel joins the
// ranges and the segments of a row:
//   o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i,   M = max_i m_i
// with o_i, l_i the sums of 2^(x - m_i) v and 2^(x - m_i) over range i and
// x = q.k * scale * log2(e).
#pragma once
#include "common.cuh"

namespace mib200 {

// Division of 0 <= n < 2^31 by a divisor known on the host: one multiplication
// and a shift.  With 2^(s-1) < d <= 2^s and m = floor(2^(31+s) / d) + 1, the
// product n m exceeds 2^(31+s) n / d by at most n 2^s / d < 2^(31+s) / d, too
// little to reach the next quotient.
struct FastDiv {
  uint32_t d, m;
  int shift;
  FastDiv() = default;
  __host__ explicit FastDiv(int64_t v) {
    d = (uint32_t)(v < 1 ? 1 : v);
    int s = 0;
    while ((1ull << s) < d) ++s;
    shift = 31 + s;
    m = (uint32_t)((1ull << shift) / d + 1);
  }
  __device__ __forceinline__ int div(int n) const {
    return (int)(((uint64_t)(uint32_t)n * m) >> shift);
  }
  // n / d and n % d
  __device__ __forceinline__ int divmod(int n, int& rem) const {
    const int q = div(n);
    rem = n - q * (int)d;
    return q;
  }
  __device__ __forceinline__ int mod(int n) const { return n - div(n) * (int)d; }
};

struct CacheSeg {
  const uint16_t* k;
  const uint16_t* v;
  long long ks_b, ks_h, ks_s, vs_b, vs_h, vs_s;  // element strides
  const int32_t* len;  // valid keys per batch entry of the segment, or null: cap
  int cap;
  int nb;      // batch entries (prefixes, or sequences)
  int seqs;    // sequences per batch entry
  int rows;    // query rows per (entry, kv head): seqs * group * Sq
  FastDiv rtiles, nsplit;  // row tiles; key ranges
  int chunk;               // keys per range
  int slot0;   // first partial slot
  int causal;  // rows see keys < len - (Sq - 1 - s); otherwise every valid key
};

struct CacheParams {
  const uint16_t* q;
  long long qs_b, qs_h, qs_s;
  uint16_t* out;
  long long os_b, os_h, os_s;
  float* lse;  // [B, Hq, Sq] natural logarithm, or null
  int Hq, Hkv, group, Sq, D;
  FastDiv div_hkv, div_sq, div_rows;  // by Hkv, Sq and group * Sq
  float scale_log2;
  CacheSeg seg[2];
  int items0;        // work items of segment 0
  int NS;            // partial slots per row (both segments); 1: items write out / lse themselves
  float* opart;      // [rows][NS][D] unnormalised
  float2* ml;        // [rows][NS] (m, l), log2 units
  // weights of the own caches' keys (cache_rows_kernel, kWeights)
  const float* z;    // lse of the rows [B, Hq, Sq], times z_mul in log2 units
  float z_mul;
  const float* win;  // or null: 0
  long long wi_b, wi_h;
  float* wout;
  long long wo_b, wo_h;
};

// (sequence, query head, token) of row r of (entry e, kv head h).
__device__ __forceinline__ void cache_row(const CacheParams& p, const CacheSeg& s, int e, int h,
                                          int r, int& b, int& head, int& tok) {
  int rem;
  const int i = p.div_rows.divmod(r, rem);
  const int g = p.div_sq.divmod(rem, tok);
  b = e * s.seqs + i;
  head = h * p.group + g;
}

__device__ __forceinline__ int cache_len(const CacheSeg& s, int e) {
  return s.len ? min(max(s.len[e], 0), s.cap) : s.cap;
}

// Two fp32 operations in one instruction (sm_100).
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)),
        "l"(reinterpret_cast<uint64_t&>(c)));
  return r;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return r;
}

// The larger / smaller of two values, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A block that gave up a wait may have asked for copies or products just before.
// They take microseconds; a millisecond goes by before it gives up the memory
// that they write to.
__device__ __noinline__ void let_land() {
  for (int i = 0; i < 64; ++i) __nanosleep(20000);
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// |scale|, but not 0: a hidden score of -inf has to stay -inf when it is scaled.
// A scale that is NaN stays one.
__device__ __forceinline__ float score_scale(float scale) {
  const float a = fabsf(scale);
  return a < 1e-30f ? 1e-30f : a;
}

// A row's reference m after scores whose maximum is t.  A NaN among them
// (t is NaN) leaves it finite: the row's sums carry the NaN, and -inf keeps
// meaning that nothing has been seen.
__device__ __forceinline__ float next_ref(float m, float t) {
  if (t != t) return m == -INFINITY ? 0.f : m;
  return fmaxf(m, t);
}

// 2^x of two values on the FMA pipe, for x up to 128 (0 below -126.5, infinity
// from 127.5, NaN for NaN).  x = n + f with n the nearest integer (adding
// 1.5 * 2^23 leaves it in the low bits), 2^f by a polynomial of degree 5, the
// minimax one for the relative error over [-1/2, 1/2] found by Remez exchange
// (7.5e-8; 1.5e-7 with its coefficients in fp32, 2.1e-7 computed in fp32), times
// 2^n put together from its bits: n = -127 gives 0 and n = 128 infinity.
__device__ __forceinline__ float2 poly_exp2(float2 x) {
  x.x = max_nan(x.x, -127.f);
  x.y = max_nan(x.y, -127.f);
  const float2 t = add2(x, make_float2(12582912.f, 12582912.f));
  const float2 n = add2(t, make_float2(-12582912.f, -12582912.f));
  const float2 f = fma2(n, make_float2(-1.f, -1.f), x);
  float2 r = make_float2(1.3276472e-3f, 1.3276472e-3f);
  r = fma2(r, f, make_float2(9.6755413e-3f, 9.6755413e-3f));
  r = fma2(r, f, make_float2(5.5507133e-2f, 5.5507133e-2f));
  r = fma2(r, f, make_float2(2.4022120e-1f, 2.4022120e-1f));
  r = fma2(r, f, make_float2(6.9314697e-1f, 6.9314697e-1f));
  r = fma2(r, f, make_float2(1.0000001f, 1.0000001f));
  return mul2(r, make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000),
                             __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000)));
}

}  // namespace mib200
