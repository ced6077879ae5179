// Attention weight per cached key:
//   w_out[b, h, j] = w_in[b, h, j] + sum over the group's query heads and the
//                    new tokens r that see key j of exp(s_rj - lse_r)
// with s = scale * q.k.  lse comes with the call (from the attention of the
// same rows) or is computed first from the keys.
#include "cache_attn.cuh"
#include "host_util.h"
#include "mma_sync.cuh"

namespace mib200 {

struct WeightParams {
  const uint16_t* q;
  long long qs_b, qs_h, qs_s;
  const uint16_t* k;
  long long ks_b, ks_h, ks_s;
  const int32_t* len;
  const float* lse;  // [B, Hq, Sq]
  float lse_mul;     // to log2 units
  const float* win;  // or null: zero
  long long wi_b, wi_h;
  float* wout;
  long long wo_b, wo_h;
  int B, Hq, Hkv, group, Sq, C, D, causal;
  float scale_log2;
};

// log-sum-exp (log2 units) of every row from its ranges' (m, l).
__global__ void weight_lse_kernel(const float2* ml, int NS, float* lse, long long nrows) {
  const long long row = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (row >= nrows) return;
  float M = -INFINITY, l = 0.f;
  for (int i = 0; i < NS; ++i) M = fmaxf(M, ml[row * NS + i].x);
  if (M != -INFINITY)
    for (int i = 0; i < NS; ++i) {
      const float2 x = ml[row * NS + i];
      l += x.y * fast_exp2(x.x - M);
    }
  lse[row] = M == -INFINITY ? M : M + log2f(l);
}

// ---------------------------------------------------------------------------
// Many rows (more than 8 per key/value head): two tcgen05 passes over
// Q K^T that keep nothing of it, row statistics and key sums.  Both are bound
// by the exponentials, one per (row, key) and pass: 16 per clock and SM on the
// MUFU unit.  Every fourth pair is computed on the FMA pipe instead
// (poly_exp2), and eight epilogue warps (two per TMEM lane quadrant, taking
// turns at the steps) on each of two blocks per SM hide the latencies of either.
// Warp 8 issues TMA, warp 9 the products.  Measured, all queries of a 16384
// prompt of 32 heads of 96: 2.50 ms with the MUFU alone, 2.39 with every eighth
// pair on the FMA pipe, 2.37 with every fourth, 2.78 with every second; four
// epilogue warps 3.66.
// ---------------------------------------------------------------------------
constexpr int kPolyEvery = 4;
constexpr int kScanThreads = 320;

// acc += sum over 32 columns of 2^(s * sc + z[c]); z per column in shared memory.
// The exponents are at most about 0 (z is minus a log-sum-exp; -inf adds 0); an
// lse that is no row's could bring one past 128, the polynomial's range.
__device__ __forceinline__ void exp_sum_cols(const float (&s)[32], float sc, const float* z,
                                             float2& a0, float2& a1) {
  const float2 sc2 = make_float2(sc, sc);
#pragma unroll
  for (int c = 0; c < 32; c += 4) {
    const float4 zz = *reinterpret_cast<const float4*>(z + c);
    const float2 x0 = fma2(make_float2(s[c], s[c + 1]), sc2, make_float2(zz.x, zz.y));
    const float2 x1 = fma2(make_float2(s[c + 2], s[c + 3]), sc2, make_float2(zz.z, zz.w));
    a0 = add2(a0, (c / 2) % kPolyEvery == 0
                      ? poly_exp2(make_float2(min_nan(x0.x, 128.f), min_nan(x0.y, 128.f)))
                      : make_float2(fast_exp2(x0.x), fast_exp2(x0.y)));
    a1 = add2(a1, make_float2(fast_exp2(x1.x), fast_exp2(x1.y)));
  }
}
// The same with one addend for all columns.  top: the largest exponent of those
// that the polynomial took (it must stay below 128).
__device__ __forceinline__ void exp_sum_row(const float (&s)[32], float sc, float z, float2& a0,
                                            float2& a1, float& top) {
  const float2 sc2 = make_float2(sc, sc), z2 = make_float2(z, z);
  top = -INFINITY;
#pragma unroll
  for (int c = 0; c < 32; c += 4) {
    const float2 x0 = fma2(make_float2(s[c], s[c + 1]), sc2, z2);
    const float2 x1 = fma2(make_float2(s[c + 2], s[c + 3]), sc2, z2);
    if ((c / 2) % kPolyEvery == 0) {
      top = fmax3(top, x0.x, x0.y);
      a0 = add2(a0, poly_exp2(x0));
    } else {
      a0 = add2(a0, make_float2(fast_exp2(x0.x), fast_exp2(x0.y)));
    }
    a1 = add2(a1, make_float2(fast_exp2(x1.x), fast_exp2(x1.y)));
  }
}

// Gathers query rows [r0, r0 + 16) of a tile into 64-byte swizzled chunks of 32
// dims (`chunk` bytes apart), by one warp.  Row r of the key/value head is token
// r % Sq of its query head r / Sq; rows from `rows` on are zero.
template <int DK>
__device__ __forceinline__ void gather_rows16(const WeightParams& p, const FastDiv& div_sq, int b,
                                              int h, int row0, int r0, int rows, uint32_t flip,
                                              uint8_t* dst, int chunk) {
  constexpr int U = DK / 8, kIter = U / 2;
  const int lane = threadIdx.x & 31;
  int tok;
  const int g = div_sq.divmod(min(row0 + r0 + (lane & 15), rows - 1), tok);
  const unsigned long long mine = reinterpret_cast<unsigned long long>(
      p.q + b * p.qs_b + (long long)(h * p.group + g) * p.qs_h + (long long)tok * p.qs_s);
  uint4 x[kIter];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int r = (i * 32 + lane) / U, u = (i * 32 + lane) % U;
    const unsigned long long a = __shfl_sync(0xffffffffu, mine, r);
    x[i] = make_uint4(0, 0, 0, 0);
    if (row0 + r0 + r < rows && u * 8 < p.D)
      x[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a) + u * 8);
  }
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int r = r0 + (i * 32 + lane) / U, u = (i * 32 + lane) % U;
    x[i].x ^= flip, x[i].y ^= flip, x[i].z ^= flip, x[i].w ^= flip;
    *reinterpret_cast<uint4*>(dst + (u >> 2) * chunk + r * 64 + (((u & 3) ^ ((r >> 1) & 3)) << 4)) =
        x[i];
  }
}

// ---------------------------------------------------------------------------
// Row statistics: an item is a tile of 128 query rows of a key/value head (the
// M rows) against a range of 128-key blocks.  A row's exponentials are taken
// against its maximum so far without looking for a larger one: only a sum that
// passes 2^40 (or none so far) makes the warp look, so the maximum costs
// nothing in between.  Leaves (maximum, sum), or the log-sum-exp where the item
// has the whole row.  Measured: 64 rows of 32 heads of 96 over 65536 keys 65 us
// (6.2 TB/s of K); all queries of a 16384 prompt 1.11 ms (0.98 at the MUFU's
// rate alone).
// ---------------------------------------------------------------------------
template <int DK>
struct StatSmem {
  static constexpr int NC = DK / 32;
  static constexpr int KS = DK == 128 ? 2 : (DK == 96 ? 3 : 5);
  static constexpr int kQTile = NC * 128 * 64, kKBlock = NC * 128 * 64;
  static constexpr int kKOff = kQTile;
  static constexpr int kJoinOff = kKOff + KS * kKBlock;
  static constexpr int kBarOff = kJoinOff + 128 * 8;
  // k_full[KS] k_empty[KS] s_full[2] s_empty[2] q_full
  static constexpr int kSlotOff = kBarOff + (2 * KS + 5) * 8;
  static constexpr int kAlloc = kSlotOff + 8 + 512;
  static_assert(kAlloc <= 113 * 1024, "two blocks per SM");
};

struct StatParams {
  WeightParams w;
  FastDiv rtiles, nsplit, div_hkv, div_sq;
  int blocks;  // 128-key blocks per range
  float2* ml;  // [rows][nsplit], or null
  float* lse;  // [rows], log2 units, where nsplit is 1
};

template <typename DT, int DK>
__global__ void __launch_bounds__(kScanThreads, 2)
    row_stats_kernel(const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ StatParams sp) {
  using L = StatSmem<DK>;
  constexpr int NC = L::NC, KS = L::KS;
  const WeightParams& p = sp.w;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 511) & ~static_cast<uintptr_t>(511));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* k_empty = k_full + KS;
  uint64_t* s_full = k_empty + KS;
  uint64_t* s_empty = s_full + 2;
  uint64_t* q_full = s_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kSlotOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kSlotOff + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto all = [](bool x) { return __all_sync(0xffffffffu, x) != 0; };
  pdl_launch();

  int rt, split, h;
  // late row tiles first: a causal prompt's last rows see the most keys
  const int b = sp.div_hkv.divmod(
      sp.rtiles.divmod(sp.nsplit.divmod(blockIdx.x, split), rt), h);
  const int r0 = ((int)sp.rtiles.d - 1 - rt) * 128;
  const int rows = p.group * p.Sq;
  const int nrows = min(128, rows - r0);
  const int len = p.len ? min(max(p.len[b], 0), p.C) : p.C;
  int end = len;  // keys that the tile's last token sees
  if (p.causal) {
    const int last = r0 + nrows - 1;
    int smax;
    if (sp.div_sq.divmod(last, smax) != sp.div_sq.div(r0)) smax = p.Sq - 1;
    end = max(0, len - (p.Sq - 1 - smax));
  }
  const int nblk = (end + 127) >> 7;
  const int j0 = (int)min((long long)split * sp.blocks, (long long)nblk);
  const int nent = min(nblk - j0, sp.blocks);

  if (threadIdx.x == 0) {
    for (int i = 0; i < KS; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1), mbar_init(&s_empty[i], 128);
    mbar_init(q_full, 256);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 8) {
    if (lane == 0) {
      for (int j = 0; j < nent; ++j) {
        if (*abort_flag) break;
        const int st = j % KS, use = j / KS;
        if (use > 0 && !mbar_wait(&k_empty[st], (use - 1) & 1, 151)) {
          *abort_flag = 1;
          break;
        }
        mbar_arrive_expect_tx(&k_full[st], L::kKBlock);
        for (int c = 0; c < NC; ++c)
          tma_load_4d(smem + L::kKOff + st * L::kKBlock + c * (128 * 64), &tm_k, &k_full[st],
                      c * 32, (j0 + j) * 128, h, b);
      }
    }
  } else if (warp == 9) {
    constexpr uint32_t idesc = make_idesc_f16(DType<DT>::kBF16, 128, 128, false, false);
    const uint64_t qd = make_desc_sw64(smem_u32(smem), 16, 512);
    const uint64_t kd0 = make_desc_sw64(smem_u32(smem + L::kKOff), 16, 512);
    bool ok = all(nent == 0 || mbar_wait(q_full, 0, 152));
    for (int j = 0; ok && j < nent; ++j) {
      const int st = j % KS;
      if (*abort_flag) break;
      ok = all(mbar_wait(&k_full[st], (j / KS) & 1, 153));
      if (ok && j >= 2) ok = all(mbar_wait(&s_empty[j & 1], ((j >> 1) - 1) & 1, 154));
      if (!ok) break;
      tc_fence_after();
      if (elect_one_sync()) {
        const uint64_t kd = kd0 + (uint64_t)((st * L::kKBlock) >> 4);
#pragma unroll
        for (int ks = 0; ks < DK / 16; ++ks) {
          const uint64_t off = ((ks >> 1) * (128 * 64) + (ks & 1) * 32) >> 4;
          umma_f16_ss(tmem_base + (j & 1) * 128, qd + off, kd + off, idesc, ks > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[j & 1]);
        umma_commit(&k_empty[st]);
      }
      __syncwarp();
    }
    if (!ok && lane == 0) *abort_flag = 1;
  } else {
    // thread = row (warp & 3) * 32 + lane; warps 0-3 take the even blocks, 4-7
    // the odd ones, each group with its own S buffer
    const int row = (warp & 3) * 32 + lane, half = warp >> 2;
    const bool live = row < nrows;
    int tok;
    const int g = sp.div_sq.divmod(r0 + min(row, nrows - 1), tok);
    if (nent > 0) {
      gather_rows16<DK>(p, sp.div_sq, b, h, r0, warp * 16, rows,
                        p.scale_log2 < 0.f ? 0x80008000u : 0u, smem, 128 * 64);
      fence_proxy_async_smem();
      mbar_arrive(q_full);
    }
    const int lim = p.causal ? len - (p.Sq - 1 - tok) : len;  // keys that the row sees
    const int wlo = __reduce_min_sync(0xffffffffu, live ? lim : 0x7fffffff);
    const int whi = __reduce_max_sync(0xffffffffu, live ? lim : 0);
    const float sc = score_scale(p.scale_log2);
    const uint32_t tcol = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + half * 128;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = half; j < nent; j += 2) {
      if (!all(mbar_wait(&s_full[half], (j >> 1) & 1, 155))) { ok = false; break; }
      tc_fence_after();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int key0 = (j0 + j) * 128 + q * 32;
        float s[32];
        tmem_ld32(tcol + q * 32, s);
        tmem_wait_ld();
        if (q == 3) {  // the buffer may be filled again
          tc_fence_before();
          mbar_arrive(&s_empty[half]);
        }
        if (key0 >= whi) continue;
        if (key0 + 32 > wlo) {
          const uint64_t vis = bits_below((long long)lim - key0);
#pragma unroll
          for (int c = 0; c < 32; ++c) s[c] = ((vis >> c) & 1ull) ? s[c] : -INFINITY;
        }
        float2 a0 = make_float2(0.f, 0.f), a1 = a0;
        float top;
        exp_sum_row(s, sc, m == -INFINITY ? -INFINITY : -m, a0, a1, top);
        a0 = add2(a0, a1);
        float sum = a0.x + a0.y;
        const bool bad = m == -INFINITY || !(sum < 1.1e12f) || top > 40.f;
        if (__any_sync(0xffffffffu, bad)) {
          float t = s[0];
#pragma unroll
          for (int c = 1; c < 31; c += 2) t = max3_nan(t, s[c], s[c + 1]);
          t = max_nan(t, s[31]) * sc;
          if (bad) {
            const float mn = next_ref(m, t);
            if (m != -INFINITY) l *= fast_exp2(m - mn);
            m = mn;
          }
          a0 = a1 = make_float2(0.f, 0.f);
          exp_sum_row(s, sc, m == -INFINITY ? -INFINITY : -m, a0, a1, top);
          a0 = add2(a0, a1);
          sum = m == -INFINITY ? 0.f : a0.x + a0.y;
        }
        l += sum;
      }
    }
    if (!all(ok)) *abort_flag = 1;
    float2* join = reinterpret_cast<float2*>(smem + L::kJoinOff);
    if (half) join[row] = make_float2(m, l);
    named_barrier(1, 256);
    if (!half && live) {
      const float2 o = join[row];
      const float mn = fmaxf(m, o.x);
      const float lt = mn == -INFINITY ? 0.f : l * fast_exp2(m - mn) + o.y * fast_exp2(o.x - mn);
      const long long at = ((long long)b * p.Hq + h * p.group + g) * p.Sq + tok;
      if (sp.lse) sp.lse[at] = mn == -INFINITY ? mn : mn + log2f(lt);
      else sp.ml[at * sp.nsplit.d + split] = make_float2(mn, lt);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) let_land();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 256);
  }
}

// ---------------------------------------------------------------------------
// Key sums: S^T = K Q^T, a tile of 128 keys (the M rows, one per thread)
// against blocks of NB query rows.  A key's weight is a sum along its own TMEM
// lane, so nothing crosses threads (but the sums of the two groups of epilogue
// warps, once per tile) and nothing is written back.  A step is one block
// against one tile; warps 0-3 take the even steps, 4-7 the odd ones.  What a cache holds past its length
// stays in its own lanes, whose sums are dropped.
//
// RES: the rows of the key/value head are one block (NB = 64 or 128, packed
// over its query heads), which stays in shared memory while key tiles stream;
// otherwise a key tile stays while the blocks of each head's rows that see it
// stream.  Measured on the same: 69 us (RES; 5.8 TB/s) and 1.38 ms.
// ---------------------------------------------------------------------------
template <int DK, int NB, bool RES>
struct ColsSmem {
  static constexpr int NC = DK / 32;
  static constexpr int kKTile = NC * 128 * 64, kQBlock = NC * NB * 64;
  static constexpr int QS = RES ? 1 : (DK == 64 ? 4 : 2);
  static constexpr int KS = RES ? (104 * 1024 - kQBlock) / kKTile : (DK == 128 ? 1 : 2);
  static constexpr int SB = 256 / NB;  // S buffers
  static constexpr int kQOff = KS * kKTile;
  static constexpr int kRowOff = kQOff + QS * kQBlock;  // per warp: NB x -lse, NB x token
  static constexpr int kJoinOff = kRowOff + 8 * 2 * NB * 4;
  static constexpr int kBarOff = kJoinOff + 2 * 128 * 4;
  // k_full[KS] k_empty[KS] q_full[QS] q_empty[QS] s_full[SB] s_empty[SB]
  static constexpr int kSlotOff = kBarOff + (2 * KS + 2 * QS + 2 * SB) * 8;
  static constexpr int kAlloc = kSlotOff + 8 + 512;
  static_assert(kAlloc <= 113 * 1024, "two blocks per SM");
};

struct ColsParams {
  WeightParams w;
  int tiles, per;  // key tiles of a (b, h); tiles per item
  FastDiv ranges;  // items per (b, h)
  FastDiv div_hkv, div_sq;
};

template <typename DT, int DK, int NB, bool RES>
__global__ void __launch_bounds__(kScanThreads, 2)
    weight_tiles_kernel(const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_q,
                        const __grid_constant__ ColsParams cp) {
  using L = ColsSmem<DK, NB, RES>;
  constexpr int NC = L::NC, KS = L::KS, QS = L::QS, SB = L::SB;
  const WeightParams& p = cp.w;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 511) & ~static_cast<uintptr_t>(511));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* k_empty = k_full + KS;
  uint64_t* q_full = k_empty + KS;
  uint64_t* q_empty = q_full + QS;
  uint64_t* s_full = q_empty + QS;
  uint64_t* s_empty = s_full + SB;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kSlotOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kSlotOff + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto all = [](bool x) { return __all_sync(0xffffffffu, x) != 0; };

  int range, h;
  const int b = cp.div_hkv.divmod(cp.ranges.divmod(blockIdx.x, range), h);
  const int len = p.len ? min(max(p.len[b], 0), p.C) : p.C;
  const int t0 = range * cp.per, t1 = min(cp.tiles, t0 + cp.per);
  const int tv = min(t1, (len + 127) >> 7);  // tiles from tv on hold no valid key
  const int rows = p.group * p.Sq;
  const int nsb = RES ? 1 : (p.Sq + NB - 1) / NB;
  const int heads = RES ? 1 : p.group;
  // First block of a head's rows that sees key tile t.
  auto first_block = [&](int t) {
    return !RES && p.causal ? max(0, t * 128 - len + p.Sq) / NB : 0;
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < KS; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < QS; ++i) mbar_init(&q_full[i], RES ? 256 : 1), mbar_init(&q_empty[i], 1);
    for (int i = 0; i < SB; ++i) mbar_init(&s_full[i], 1), mbar_init(&s_empty[i], 128);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 8) {
    if (lane == 0) {
      bool ok = true;
      int nq = 0;
      for (int t = t0; ok && t < tv; ++t) {
        if (*abort_flag) break;
        const int st = (t - t0) % KS, use = (t - t0) / KS;
        if (use > 0 && !mbar_wait(&k_empty[st], (use - 1) & 1, 141)) { ok = false; break; }
        mbar_arrive_expect_tx(&k_full[st], L::kKTile);
        for (int c = 0; c < NC; ++c)
          tma_load_4d(smem + st * L::kKTile + c * (128 * 64), &tm_k, &k_full[st], c * 32, t * 128,
                      h, b);
        if constexpr (!RES) {
          for (int g = 0; ok && g < heads; ++g)
            for (int sb = first_block(t); sb < nsb; ++sb, ++nq) {
              const int qs = nq % QS, qu = nq / QS;
              if (qu > 0 && !mbar_wait(&q_empty[qs], (qu - 1) & 1, 142)) { ok = false; break; }
              mbar_arrive_expect_tx(&q_full[qs], L::kQBlock);
              for (int c = 0; c < NC; ++c)
                tma_load_4d(smem + L::kQOff + qs * L::kQBlock + c * (NB * 64), &tm_q, &q_full[qs],
                            c * 32, sb * NB, h * p.group + g, b);
            }
        }
      }
      if (!ok) *abort_flag = 1;
    }
  } else if (warp == 9) {
    constexpr uint32_t idesc = make_idesc_f16(DType<DT>::kBF16, 128, NB, false, false);
    const uint64_t kd0 = make_desc_sw64(smem_u32(smem), 16, 512);
    const uint64_t qd0 = make_desc_sw64(smem_u32(smem + L::kQOff), 16, 512);
    bool ok = all(!RES || tv <= t0 || mbar_wait(&q_full[0], 0, 144));
    int n = 0;
    for (int t = t0; ok && t < tv; ++t) {
      const int st = (t - t0) % KS;
      if (*abort_flag) { ok = false; break; }
      if (!all(mbar_wait(&k_full[st], ((t - t0) / KS) & 1, 143))) { ok = false; break; }
      const int f = first_block(t);
      for (int g = 0; ok && g < heads; ++g)
        for (int sb = f; sb < nsb; ++sb, ++n) {
          const int qs = n % QS, buf = n % SB;
          if (!RES && !all(mbar_wait(&q_full[qs], (n / QS) & 1, 144))) { ok = false; break; }
          if (n >= SB && !all(mbar_wait(&s_empty[buf], (n / SB - 1) & 1, 145))) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one_sync()) {
            const uint64_t kd = kd0 + (uint64_t)((st * L::kKTile) >> 4);
            const uint64_t qd = qd0 + (uint64_t)((RES ? 0 : qs * L::kQBlock) >> 4);
#pragma unroll
            for (int ks = 0; ks < DK / 16; ++ks) {
              const uint32_t off = (ks & 1) * 32;
              umma_f16_ss(tmem_base + buf * NB, kd + (((ks >> 1) * (128 * 64) + off) >> 4),
                          qd + (((ks >> 1) * (NB * 64) + off) >> 4), idesc, ks > 0 ? 1u : 0u);
            }
            umma_commit(&s_full[buf]);
            if constexpr (!RES) umma_commit(&q_empty[qs]);
            if (g == heads - 1 && sb == nsb - 1) umma_commit(&k_empty[st]);
          }
          __syncwarp();
        }
    }
    if (!ok && lane == 0) *abort_flag = 1;
  } else {
    // thread = key (warp & 3) * 32 + lane of the tile
    const int key = (warp & 3) * 32 + lane, grp = warp >> 2;
    if constexpr (RES) {
      if (tv > t0) {
        if (warp * 16 < NB)
          gather_rows16<DK>(p, cp.div_sq, b, h, 0, warp * 16, rows, 0u, smem + L::kQOff, NB * 64);
        fence_proxy_async_smem();
        mbar_arrive(&q_full[0]);
      }
    }
    pdl_wait();  // lse may come from the kernel before
    const uint32_t tcol = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    float* nz = reinterpret_cast<float*>(smem + L::kRowOff) + warp * (2 * NB);
    int* tok = reinterpret_cast<int*>(nz) + NB;
    float* join = reinterpret_cast<float*>(smem + L::kJoinOff);
    const float* win = p.win ? p.win + b * p.wi_b + h * p.wi_h : nullptr;
    float* wout = p.wout + b * p.wo_b + h * p.wo_h;
    const float* lse = p.lse + ((long long)b * p.Hq + h * p.group) * p.Sq;
    // a block's rows: -lse (log2 units; -inf: adds nothing) and tokens, in
    // shared memory of the warp; fetched a step of the group ahead
    float zn[NB / 32];
    auto fetch = [&](int g, int sb) {
#pragma unroll
      for (int x = 0; x < NB / 32; ++x) {
        const int r = sb * NB + x * 32 + lane;
        zn[x] = g < heads && r < (RES ? rows : p.Sq) ? lse[(long long)g * p.Sq + r] : -INFINITY;
      }
    };
    auto lay = [&](int sb) {
      __syncwarp();
#pragma unroll
      for (int x = 0; x < NB / 32; ++x) {
        const int r = sb * NB + x * 32 + lane;
        nz[x * 32 + lane] = zn[x] == -INFINITY ? zn[x] : -zn[x] * p.lse_mul;
        tok[x * 32 + lane] = RES ? cp.div_sq.mod(r) : r;
      }
      __syncwarp();
    };
    bool ok = true;
    // Sum over the rows of step n's block; whole: all of them see all of the
    // warp's keys, otherwise those of tokens from smin on see this thread's.
    auto step = [&](int n, bool whole, int smin) -> float {
      const int buf = n % SB;
      ok = all(mbar_wait(&s_full[buf], (n / SB) & 1, 146));
      if (!ok) return 0.f;
      tc_fence_after();
      float2 a0 = make_float2(0.f, 0.f), a1 = a0;
#pragma unroll
      for (int q = 0; q < NB / 32; ++q) {
        float s[32];
        tmem_ld32(tcol + buf * NB + q * 32, s);
        tmem_wait_ld();
        if (q == NB / 32 - 1) {  // the buffer may be filled again
          tc_fence_before();
          mbar_arrive(&s_empty[buf]);
        }
        if (whole) {
          exp_sum_cols(s, p.scale_log2, nz + q * 32, a0, a1);
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (tok[q * 32 + c] >= smin)
              a0.x += fast_exp2(fmaf(s[c], p.scale_log2, nz[q * 32 + c]));
        }
      }
      a0 = add2(a0, a1);
      return a0.x + a0.y;  // a block's sum; the blocks add up outside
    };
    if constexpr (RES) {
      // a step per tile: each group has its own tiles
      if (tv > t0) {
        fetch(0, 0);
        lay(0);
      }
      for (int t = t0 + grp; t < t1; t += 2) {
        const int j = t * 128 + key;
        const float w0 = win && j < p.C ? win[j] : 0.f;
        const int smin = p.causal ? j - len + p.Sq : 0;  // token from which a row sees the key
        float tot = 0.f;
        if (ok && t < tv) tot = step(t - t0, __shfl_sync(0xffffffffu, smin, 31) <= 0, smin);
        if (j < len ? ok : (j < p.C && win != wout)) wout[j] = j < len ? w0 + tot : w0;
      }
    } else {
      int n = 0;
      for (int t = t0; t < t1; ++t) {
        const int j = t * 128 + key;
        const float w0 = !grp && win && j < p.C ? win[j] : 0.f;
        const int smin = p.causal ? j - len + p.Sq : 0;
        const int wmin = __shfl_sync(0xffffffffu, smin, 31);
        float tot = 0.f;
        if (t < tv) {
          const int f = first_block(t), per = nsb - f, steps = heads * per;
          // this group's steps of the tile: i, i + 2, ... as (head, block)
          int i = (n ^ grp) & 1, g = 0, sb = f;
          auto advance = [&](int by) {
            sb += by;
            while (sb >= nsb) sb -= per, ++g;
          };
          advance(i);
          if (i < steps) fetch(g, sb);
          for (; ok && i < steps; i += 2) {
            const int cur = sb;
            lay(cur);
            advance(2);
            if (i + 2 < steps) fetch(g, sb);
            tot += step(n + i, wmin <= cur * NB, smin);
          }
          n += steps;
        }
        // the groups' sums meet once per tile; a buffer is written again two
        // barriers after it was read
        if (grp) join[(t & 1) * 128 + key] = tot;
        named_barrier(1, 256);
        if (!grp && (j < len ? ok : (j < p.C && win != wout)))
          wout[j] = j < len ? w0 + (tot + join[(t & 1) * 128 + key]) : w0;
      }
    }
    if (!all(ok)) *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) let_land();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 256);
  }
}

// Ranges per row tile of the statistics (two items per SM run at a time; see
// tile_blocks), in 128-key blocks.
static int stat_ranges(int64_t B, int64_t Hkv, int64_t rows, int64_t C) {
  const int64_t blocks = (C + 127) / 128;
  const int64_t per = tile_blocks({0, B * Hkv * ((rows + 127) / 128)}, {0, blocks});
  return (int)((blocks + per - 1) / per);
}

template <typename DT, int DK>
static int launch_stats(const WeightParams& w, const mi_rows& k, float2* ml, float* lse,
                        cudaStream_t st) {
  using L = StatSmem<DK>;
  StatParams sp{};
  const int64_t rows = (int64_t)w.group * w.Sq, rtiles = (rows + 127) / 128;
  const int64_t blocks = (w.C + 127) / 128;
  const int ns = stat_ranges(w.B, w.Hkv, rows, w.C);
  const long long items = (long long)w.B * w.Hkv * rtiles * ns;
  if (items > 0x7fffffffll) return MI_ERR_SHAPE;
  sp.w = w;
  sp.rtiles = FastDiv(rtiles);
  sp.nsplit = FastDiv(ns);
  sp.div_hkv = FastDiv(w.Hkv);
  sp.div_sq = FastDiv(w.Sq);
  sp.blocks = (int)((blocks + ns - 1) / ns);
  sp.ml = ml;
  sp.lse = ns == 1 ? lse : nullptr;
  CUtensorMap tk;
  const int rc = make_rows4_map(&tk, k, w.B, w.Hkv, w.C, w.D, 32, 128);
  if (rc != MI_OK) return rc;
  cudaError_t err = allow_smem<row_stats_kernel<DT, DK>>(L::kAlloc);
  if (err == cudaSuccess) {
    row_stats_kernel<DT, DK><<<(unsigned)items, kScanThreads, L::kAlloc, st>>>(tk, sp);
    err = cudaGetLastError();
  }
  if (err == cudaSuccess && ns > 1) {
    const long long n = (long long)w.B * w.Hq * w.Sq;
    weight_lse_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(ml, ns, lse, n);
    err = cudaGetLastError();
  }
  return err == cudaSuccess ? MI_OK : MI_ERR_LAUNCH;
}

template <typename DT, int DK, int NB, bool RES>
static int launch_cols_t(const WeightParams& w, const mi_rows& q, const mi_rows& k, bool after,
                         cudaStream_t st) {
  using L = ColsSmem<DK, NB, RES>;
  ColsParams cp{};
  cp.w = w;
  cp.tiles = (w.C + 127) / 128;
  const long long all = (long long)w.B * w.Hkv * cp.tiles;
  // tiles per item: with resident rows three rounds of two items per SM
  // (one: 162 us for 64 rows of 32 x 65536 keys, two and three: 138);
  // otherwise enough that an item has 16 blocks
  const long long steps = (long long)w.group * ((w.Sq + NB - 1) / NB);
  const long long slots = 148 * 2 * 3;
  const long long per = RES ? (all + slots - 1) / slots : (16 + steps - 1) / steps;
  cp.per = (int)(per < 1 ? 1 : (per > cp.tiles ? cp.tiles : per));
  const int ranges = (cp.tiles + cp.per - 1) / cp.per;
  cp.ranges = FastDiv(ranges);
  cp.div_hkv = FastDiv(w.Hkv);
  cp.div_sq = FastDiv(w.Sq);
  const long long items = (long long)w.B * w.Hkv * ranges;
  if (items > 0x7fffffffll) return MI_ERR_SHAPE;
  CUtensorMap tk, tq;
  memset(&tq, 0, sizeof(tq));
  int rc = make_rows4_map(&tk, k, w.B, w.Hkv, w.C, w.D, 32, 128);
  if (rc == MI_OK && !RES) rc = make_rows4_map(&tq, q, w.B, w.Hq, w.Sq, w.D, 32, NB);
  if (rc != MI_OK) return rc;
  constexpr auto kern = weight_tiles_kernel<DT, DK, NB, RES>;
  cudaError_t err = allow_smem<weight_tiles_kernel<DT, DK, NB, RES>>(L::kAlloc);
  if (err == cudaSuccess) {
    // beside the end of the statistics of the same call, whose own launch has
    // waited for whatever wrote the keys
    if (after) {
      err = launch_after(kern, dim3((unsigned)items), kScanThreads, L::kAlloc, st, tk, tq, cp);
    } else {
      kern<<<(unsigned)items, kScanThreads, L::kAlloc, st>>>(tk, tq, cp);
      err = cudaGetLastError();
    }
  }
  if (err != cudaSuccess) {
    debug_launch_failure("weight_tiles_kernel", reinterpret_cast<const void*>(kern), err,
                         kScanThreads, L::kAlloc);
    return MI_ERR_LAUNCH;
  }
  return MI_OK;
}

// One resident block where the key/value head's rows fit it, else streamed
// blocks of 128 rows of a head (64 where a head has no more).
template <typename DT, int DK>
static int launch_weights_many(const WeightParams& w, const mi_rows& q, const mi_rows& k,
                               float2* ml, float* lse, cudaStream_t st) {
  WeightParams p = w;
  if (!p.lse) {
    const int rc = launch_stats<DT, DK>(p, k, ml, lse, st);
    if (rc != MI_OK) return rc;
    p.lse = lse;
    p.lse_mul = 1.f;
  }
  const long long rows = (long long)p.group * p.Sq;
  if (rows <= 64) return launch_cols_t<DT, DK, 64, true>(p, q, k, !w.lse, st);
  if (rows <= 128) return launch_cols_t<DT, DK, 128, true>(p, q, k, !w.lse, st);
  if (p.Sq <= 64) return launch_cols_t<DT, DK, 64, false>(p, q, k, !w.lse, st);
  return launch_cols_t<DT, DK, 128, false>(p, q, k, !w.lse, st);
}

}  // namespace mib200

using namespace mib200;

// Partial statistics per row of the call's split.
static int64_t weights_slots(int64_t B, int64_t Hkv, int64_t group, int64_t Sq, int64_t C,
                             int64_t D) {
  return group * Sq > kRowsMost ? stat_ranges(B, Hkv, group * Sq, C)
                                : cache_plan(B, Hkv, group, Sq, 1, 0, C, D).NS;
}

extern "C" size_t mi_attn_weights_workspace_size(const mi_attn_weights_args* a) {
  if (!a || !cache_sizes_ok(a->B, a->Hq, a->Hkv, a->S_q, 1, 0, a->C, a->D)) return SIZE_MAX;
  if (a->B == 0 || a->Hq == 0 || a->S_q == 0 || a->C == 0 || a->lse) return 0;
  const int64_t ns = weights_slots(a->B, a->Hkv, a->Hq / a->Hkv, a->S_q, a->C, a->D);
  const size_t rows = (size_t)(a->B * a->Hq * a->S_q);
  if ((double)rows * ns > 1e13) return SIZE_MAX;
  return align_up(rows * ns * 8) + align_up(rows * 4);
}

extern "C" int mi_attn_weights(const mi_attn_weights_args* args, void* workspace,
                               size_t workspace_bytes, void* stream) {
  if (!args) return MI_ERR_SHAPE;
  const mi_attn_weights_args& a = *args;
  const int64_t B = a.B, Hq = a.Hq, Hkv = a.Hkv, S_q = a.S_q, C = a.C, D = a.D;
  const int dtype = a.dtype;
  const float* lse = a.lse;
  const int32_t* lengths = a.lengths;
  const mi_rows &q = a.q, &k = a.k;
  if (dtype != MI_F16 && dtype != MI_BF16) return MI_ERR_DTYPE;
  if (!cache_sizes_ok(B, Hq, Hkv, S_q, 1, 0, C, D)) return MI_ERR_SHAPE;
  if (B == 0 || C == 0) return MI_OK;
  if (Hq == 0 || S_q == 0) return MI_ERR_SHAPE;  // no rows: nothing to add
  if (!a.w_out) return MI_ERR_SHAPE;
  if (!rows_ok(q, B, Hq, S_q) || !rows_ok(k, B, Hkv, C)) return MI_ERR_ALIGN;
  const int64_t group = Hq / Hkv;
  const size_t need = mi_attn_weights_workspace_size(args);
  if (need == SIZE_MAX) return MI_ERR_SHAPE;
  if (need && (!workspace || workspace_bytes < need ||
               (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return MI_ERR_WORKSPACE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int rc;

  WeightParams w{};
  w.q = static_cast<const uint16_t*>(q.ptr);
  w.qs_b = q.stride_b;
  w.qs_h = q.stride_h;
  w.qs_s = q.stride_s;
  w.k = static_cast<const uint16_t*>(k.ptr);
  w.ks_b = k.stride_b;
  w.ks_h = k.stride_h;
  w.ks_s = k.stride_s;
  w.len = lengths;
  w.lse = lse;
  w.lse_mul = 1.4426950408889634f;
  w.win = a.w_in;
  w.wi_b = a.w_in_stride_b;
  w.wi_h = a.w_in_stride_h;
  w.wout = a.w_out;
  w.wo_b = a.w_out_stride_b;
  w.wo_h = a.w_out_stride_h;
  w.B = (int)B;
  w.Hq = (int)Hq;
  w.Hkv = (int)Hkv;
  w.group = (int)group;
  w.Sq = (int)S_q;
  w.C = (int)C;
  w.D = (int)D;
  w.causal = a.causal ? 1 : 0;
  w.scale_log2 = a.softmax_scale * 1.4426950408889634f;

  const size_t rows = (size_t)(B * Hq * S_q);
  float2* ml = static_cast<float2*>(workspace);
  float* lse2 = nullptr;
  if (!lse)
    lse2 = reinterpret_cast<float*>(
        static_cast<uint8_t*>(workspace) +
        align_up(rows * weights_slots(B, Hkv, group, S_q, C, D) * 8));
  if (group * S_q > kRowsMost) {  // the few-row form needs all rows in one tile
#define MI_MANY(DK)                                                                      \
  if (D <= DK)                                                                           \
    return dtype == MI_BF16 ? launch_weights_many<__nv_bfloat16, DK>(w, q, k, ml, lse2, st) \
                            : launch_weights_many<__half, DK>(w, q, k, ml, lse2, st);
    MI_MANY(64)
    MI_MANY(96)
    MI_MANY(128)
#undef MI_MANY
  }
  const CachePlan pl = cache_plan(B, Hkv, group, S_q, 1, 0, C, D);
  CacheParams p{};
  p.q = w.q;
  p.qs_b = w.qs_b;
  p.qs_h = w.qs_h;
  p.qs_s = w.qs_s;
  set_heads(p, Hq, Hkv, S_q, D);
  p.scale_log2 = w.scale_log2;
  p.seg[0].seqs = 1;
  set_seg(p.seg[1], k, k, lengths, C, B, 1, group * S_q, w.causal);
  p.seg[1].rtiles = FastDiv(pl.rtiles[1]);
  p.seg[1].nsplit = FastDiv(pl.nsplit[1]);
  p.seg[1].chunk = pl.chunk[1];
  p.NS = pl.NS;
  const long long items = (long long)B * Hkv * pl.rtiles[1] * pl.nsplit[1];
  if (items > 0x7fffffffll) return MI_ERR_SHAPE;
  if (!lse) {
    p.ml = ml;
    rc = launch_rows_dk<kStats>(p, dtype, items, st);
    if (rc != MI_OK) return rc;
    weight_lse_kernel<<<(unsigned)((rows + 255) / 256), 256, 0, st>>>(ml, pl.NS, lse2,
                                                                      (long long)rows);
    if (cudaGetLastError() != cudaSuccess) return MI_ERR_LAUNCH;
    w.lse = lse2;
    w.lse_mul = 1.f;
  }
  p.z = w.lse;
  p.z_mul = w.lse_mul;
  p.win = w.win;
  p.wi_b = w.wi_b;
  p.wi_h = w.wi_h;
  p.wout = w.wout;
  p.wo_b = w.wo_b;
  p.wo_h = w.wo_h;
  return launch_rows_dk<kWeights>(p, dtype, items, st);
}
