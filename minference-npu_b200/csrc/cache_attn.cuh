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

struct CacheSeg {
  const uint16_t* k;
  const uint16_t* v;
  long long ks_b, ks_h, ks_s, vs_b, vs_h, vs_s;  // element strides
  const int32_t* len;  // valid keys per batch entry of the segment, or null: cap
  int cap;
  int nb;      // batch entries (prefixes, or sequences)
  int seqs;    // sequences per batch entry
  int rows;    // query rows per (entry, kv head): seqs * group * Sq
  int rtiles;  // row tiles
  int nsplit, chunk;
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
  float scale_log2;
  CacheSeg seg[2];
  long long items0;  // work items of segment 0
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
  const int per = p.group * p.Sq;
  const int i = r / per, rem = r - i * per;
  const int g = rem / p.Sq;
  b = e * s.seqs + i;
  head = h * p.group + g;
  tok = rem - g * p.Sq;
}

__device__ __forceinline__ int cache_len(const CacheSeg& s, int e) {
  return s.len ? min(max(s.len[e], 0), s.cap) : s.cap;
}

}  // namespace mib200
