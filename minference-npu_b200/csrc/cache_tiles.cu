// Attention over caches for many query rows per key/value head (tcgen05).
//
// A work item is one 128-row tile of query rows -- the rows of all sequences
// that share a prefix, or of one sequence -- against a range of the 64-key
// blocks that the tile walks: prefix blocks, then (if the tile's rows belong
// to one sequence) the blocks of its own cache.  Warp roles and the TMEM
// hand-over are those of attn_fwd_kernel: warps 0-3 softmax (one row per
// thread), warp 4 TMA, warp 5 MMA issue, two items per SM so that one item's
// softmax overlaps the other's products.  Differences, each for this shape of
// work: the tile's rows come from several heads and sequences, so Q is
// gathered with plain loads; row sums are kept in registers, because at
// D = 128 O fills what the two S buffers leave of half the TMEM; the row's
// reference moves only when a block's sum of P says so; O leaves unnormalised
// (or finished, when the item has the whole row).
//
// P is rounded to the inputs' type, which V has (both operands of a product
// have one type); the row sums are taken before.  Against 64 bits a bf16 output
// is 2.2e-3 off (2-norm), where its own rounding alone makes 1.7e-3.
//
// Bound by the keys' bytes at few rows and by the latency of the softmax's chain
// (1 us a 64-key block and item; tensor and MUFU pipes both at 58 %) at many.
// Measured: 128 rows of 8 heads of 128 over 65536 keys 50 us (5.4 TB/s); 4096
// rows over 16384 keys and 384 own 264 us for a call alone on the GPU (1.06
// PFLOP/s), 289 among others; with a running maximum in every block 285 alone.
// Eight softmax warps on alternate blocks were slower (D = 64 235 -> 274 us), and
// so were exponentials on the FMA pipe (every eighth pair 267, every fourth 290).
#include <cstring>

#include "cache_attn.cuh"
#include "host_util.h"
#include "mma_sync.cuh"

namespace mib200 {

// Items of one kind: rows of segment `rows_of`, keys of segment 0 and / or 1.
struct TileGroup {
  int rows_of;
  int use0, use1;
  FastDiv rtiles, nsplit;
  int blocks;  // key blocks per range
  int slot0;
  int items;
};

struct TileParams {
  CacheParams c;
  TileGroup grp[2];
};

template <int DK>
struct TileSmem {
  static constexpr int NC = DK / 32;
  static constexpr int kQBytes = NC * 128 * 64;
  static constexpr int kBlock = NC * 64 * 64;  // 64 keys of K or V
  // two blocks per SM: 113 KB each at most
  static constexpr int KS = DK == 128 ? 2 : (DK == 96 ? 3 : 5);
  static constexpr int VS = DK == 128 ? 3 : (DK == 96 ? 4 : 5);
  static constexpr int kKOff = kQBytes;
  static constexpr int kVOff = kKOff + KS * kBlock;
  static constexpr int kBarOff = kVOff + VS * kBlock;
  // k_full[KS] k_empty[KS] v_full[VS] v_empty[VS] s_full[2] p_full[2] pv_done[2] q_full
  static constexpr int kNumBars = 2 * KS + 2 * VS + 7;
  static constexpr int kSlotOff = kBarOff + kNumBars * 8;
  static constexpr int kBytes = kSlotOff + 8;
  static constexpr int kAlloc = kBytes + 512;  // the base is aligned to a swizzle atom
  static constexpr uint32_t kTmemCols = 256;
  static_assert(kAlloc <= 113 * 1024, "two blocks per SM");
  static_assert(128 + DK <= 256, "TMEM");
  // The epilogue stages O in the ring, a padded row per thread.
  static constexpr int kOPitch = DK * 4 + 16;
  static_assert(128 * kOPitch <= (KS + VS) * kBlock, "O rows fit the ring");
};

// Untiled bulk copy shared -> global: both 16-byte aligned, a multiple of 16 bytes.
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst),
               "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bulk_wait0() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

constexpr int kTileThreads = 192;
// Sum of a block's P from which its row's reference moves; its logarithm, for
// a block's maximum over the reference.
constexpr float kTileSum = 32768.0f, kTileRise = 15.0f;

template <typename DT, int DK>
__global__ void __launch_bounds__(kTileThreads, 2)
    cache_tiles_kernel(const __grid_constant__ CUtensorMap tm_kp,
                       const __grid_constant__ CUtensorMap tm_vp,
                       const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v,
                       const __grid_constant__ TileParams tp) {
  using L = TileSmem<DK>;
  constexpr int NC = L::NC, KS = L::KS, VS = L::VS;
  constexpr bool kBF16 = DType<DT>::kBF16;
  const CacheParams& p = tp.c;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 511) & ~static_cast<uintptr_t>(511));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* k_empty = k_full + KS;
  uint64_t* v_full = k_empty + KS;
  uint64_t* v_empty = v_full + VS;
  uint64_t* s_full = v_empty + VS;
  uint64_t* p_full = s_full + 2;
  uint64_t* pv_done = p_full + 2;
  uint64_t* q_full = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kSlotOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kSlotOff + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch();

  // ---- the item ---------------------------------------------------------------
  int it = blockIdx.x, rt, sp, h;
  const bool second = it >= tp.grp[0].items;
  if (second) it -= tp.grp[0].items;
  const TileGroup& gr = tp.grp[second ? 1 : 0];
  const CacheSeg& rs = p.seg[gr.rows_of];
  it = gr.rtiles.divmod(it, rt);
  it = gr.nsplit.divmod(it, sp);
  const int e = p.div_hkv.divmod(it, h);                         // entry of the row segment
  const int e0 = gr.rows_of == 0 ? e : e / p.seg[0].seqs;  // prefix
  const int r0 = rt * 128;
  const int nrows = min(128, rs.rows - r0);
  const int len0 = gr.use0 ? cache_len(p.seg[0], e0) : 0;
  const int len1 = gr.use1 ? cache_len(p.seg[1], e) : 0;
  const bool causal = p.seg[1].causal != 0;
  int end1 = len1;  // own keys that the tile's last token sees
  if (gr.use1 && causal) {
    const int last = r0 + nrows - 1;
    int smax;
    if (p.div_sq.divmod(last, smax) != p.div_sq.div(r0)) smax = p.Sq - 1;
    end1 = max(0, len1 - (p.Sq - 1 - smax));
  }
  const int n0 = (len0 + 63) >> 6, n1 = (end1 + 63) >> 6;
  const int j0 = min(n0 + n1, (int)min((long long)sp * gr.blocks, (long long)(n0 + n1)));
  const int nent = min(n0 + n1 - j0, gr.blocks);

  // ---- Q: each softmax warp asks for its 32 rows (a lane per 16 bytes, addresses
  // passed around by shuffle) before the first keys are asked for, whose burst
  // it would otherwise wait behind (5 us) ------------------------------------------
  constexpr int U = DK / 8;
  const int row = threadIdx.x;
  const bool live = row < nrows;
  int b = 0, hd = 0, tk = 0;
  uint4 qx[U];
  if (live) cache_row(p, rs, e, h, r0 + row, b, hd, tk);
  if (warp < 4 && nent > 0) {
    const unsigned long long mine = reinterpret_cast<unsigned long long>(
        p.q + (live ? b * p.qs_b + hd * p.qs_h + tk * p.qs_s : 0));
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int idx = i * 32 + lane, r = idx / U, u = idx % U;
      const unsigned long long a = __shfl_sync(0xffffffffu, mine, r);
      qx[i] = make_uint4(0, 0, 0, 0);
      if (warp * 32 + r < nrows && u * 8 < p.D)
        qx[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a) + u * 8);
    }
  }

  // ---- set-up: barriers, TMEM --------------------------------------------------
  if (threadIdx.x == 0) {
    for (int s = 0; s < KS; ++s) mbar_init(&k_full[s], 1), mbar_init(&k_empty[s], 1);
    for (int s = 0; s < VS; ++s) mbar_init(&v_full[s], 1), mbar_init(&v_empty[s], 1);
    for (int i = 0; i < 2; ++i)
      mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 128), mbar_init(&pv_done[i], 1);
    mbar_init(q_full, 128);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 4) {
    // ---- TMA: K0, K1, V0, K2, V1, ... ---------------------------------------
    if (lane == 0) {
      auto load = [&](uint8_t* dst, uint64_t* full, int j, bool val) {
        const int J = j0 + j;
        const bool own = J >= n0;
        const CUtensorMap* map = own ? (val ? &tm_v : &tm_k) : (val ? &tm_vp : &tm_kp);
        const int key = (own ? J - n0 : J) * 64, ent = own ? e : e0;
        mbar_arrive_expect_tx(full, L::kBlock);
        for (int c = 0; c < NC; ++c) tma_load_4d(dst + c * (64 * 64), map, full, c * 32, key, h, ent);
      };
      bool ok = true;
      for (int j = 0; ok && j < nent + 1; ++j) {
        if (*abort_flag) break;
        if (j < nent) {
          const int st = j % KS, use = j / KS;
          if (use > 0 && !mbar_wait(&k_empty[st], (use - 1) & 1, 131)) { ok = false; break; }
          load(smem + L::kKOff + st * L::kBlock, &k_full[st], j, false);
        }
        if (j >= 1) {
          const int st = (j - 1) % VS, use = (j - 1) / VS;
          if (use > 0 && !mbar_wait(&v_empty[st], (use - 1) & 1, 132)) { ok = false; break; }
          load(smem + L::kVOff + st * L::kBlock, &v_full[st], j - 1, true);
        }
      }
      if (!ok) *abort_flag = 1;
    }
  } else if (warp == 5) {
    // ---- MMA issue (converged warp, one elected lane) ------------------------
    constexpr uint32_t idesc_qk = make_idesc_f16(kBF16, 128, 64, false, false);
    constexpr uint32_t idesc_pv = make_idesc_f16(kBF16, 128, DK, false, true);
    const uint64_t qd0 = make_desc_sw64(smem_u32(smem), 16, 512);
    const uint64_t kd0 = make_desc_sw64(smem_u32(smem + L::kKOff), 16, 512);
    const uint64_t vd0 = make_desc_sw64(smem_u32(smem + L::kVOff), 64 * 64, 512);
    auto issue_qk = [&](int j) -> bool {
      const int st = j % KS;
      if (!__all_sync(0xffffffffu, mbar_wait(&k_full[st], (j / KS) & 1, 133))) return false;
      tc_fence_after();
      if (elect_one_sync()) {
        const uint64_t kd = kd0 + (uint64_t)((st * L::kBlock) >> 4);
#pragma unroll
        for (int ks = 0; ks < DK / 16; ++ks) {
          const uint32_t off = (ks & 1) * 32;
          umma_f16_ss(tmem_base + (j & 1) * 64, qd0 + (((ks >> 1) * (128 * 64) + off) >> 4),
                      kd + (((ks >> 1) * (64 * 64) + off) >> 4), idesc_qk, ks > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[j & 1]);
        umma_commit(&k_empty[st]);
      }
      __syncwarp();
      return true;
    };
    bool ok = __all_sync(0xffffffffu, nent == 0 || mbar_wait(q_full, 0, 130));
    if (ok && nent > 0) ok = issue_qk(0);
    for (int j = 0; ok && j < nent; ++j) {
      if (*abort_flag) { ok = false; break; }
      // S buffer (j+1)&1 last held P(j-1), which PV(j-1) has read: products of
      // one thread run in issue order.
      if (j + 1 < nent && !issue_qk(j + 1)) { ok = false; break; }
      if (!__all_sync(0xffffffffu, mbar_wait(&p_full[j & 1], (j >> 1) & 1, 134))) {
        ok = false;
        break;
      }
      const int st = j % VS;
      if (!__all_sync(0xffffffffu, mbar_wait(&v_full[st], (j / VS) & 1, 135))) {
        ok = false;
        break;
      }
      tc_fence_after();
      if (elect_one_sync()) {
        const uint64_t vd = vd0 + (uint64_t)((st * L::kBlock) >> 4);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          umma_f16_ts(tmem_base + 128, tmem_base + (j & 1) * 64 + ks * 8,
                      vd + (uint64_t)((ks * 1024) >> 4), idesc_pv, (j > 0 || ks > 0) ? 1u : 0u);
        umma_commit(&pv_done[j & 1]);
        umma_commit(&v_empty[st]);
      }
      __syncwarp();
    }
    if (!ok && lane == 0) *abort_flag = 1;
  } else {
    // ---- softmax: thread = row ---------------------------------------------------
    // Q into chunks of 32 dims with the 64-byte swizzle.  A negative scale is
    // taken into Q (its sign bits), so that the largest score is the largest
    // product.
    if (nent > 0) {
      const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int idx = i * 32 + lane, r = warp * 32 + idx / U, u = idx % U;
        uint4 x = qx[i];
        x.x ^= flip, x.y ^= flip, x.z ^= flip, x.w ^= flip;
        *reinterpret_cast<uint4*>(smem + (u >> 2) * (128 * 64) + r * 64 +
                                  (((u & 3) ^ ((r >> 1) & 3)) << 4)) = x;
      }
      fence_proxy_async_smem();
      mbar_arrive(q_full);
    }
    const uint32_t lane_base = tmem_base + ((uint32_t)(warp * 32) << 16);
    int lim0 = len0, lim1 = len1;  // keys that the row sees
    if (live && causal) lim1 = len1 - (p.Sq - 1 - p.div_sq.mod(r0 + row));
    // Blocks below `full` are whole for every row of the warp, blocks from
    // `none` on empty.  Rows past the tile's last (Q = 0) take what the others
    // see; a warp of such rows only sees nothing.
    const int full0 = __reduce_min_sync(0xffffffffu, live ? lim0 : 0x7fffffff);
    const int full1 = __reduce_min_sync(0xffffffffu, live ? lim1 : 0x7fffffff);
    const int none0 = __reduce_max_sync(0xffffffffu, live ? lim0 : 0);
    const int none1 = __reduce_max_sync(0xffffffffu, live ? lim1 : 0);
    if (!live) lim0 = none0, lim1 = none1;
    const float sc = score_scale(p.scale_log2);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    auto all = [](bool x) { return __all_sync(0xffffffffu, x) != 0; };
    for (int j = 0; j < nent; ++j) {
      const int J = j0 + j;
      const bool own = J >= n0;
      const int key0 = (own ? J - n0 : J) * 64;
      if (!all(mbar_wait(&s_full[j & 1], (j >> 1) & 1, 136))) { ok = false; break; }
      tc_fence_after();
      const uint32_t tmem_s = lane_base + (j & 1) * 64;
      const bool empty = key0 >= (own ? none1 : none0);
      const bool whole = key0 + 64 <= (own ? full1 : full0);
      // a cache's stale rows: 0 * V must not let them through
      const int held = own ? len1 : len0;
      if (key0 + 64 > held) {
        if (!all(mbar_wait(&v_full[j % VS], (j / VS) & 1, 137))) { ok = false; break; }
        uint8_t* vb = smem + L::kVOff + (j % VS) * L::kBlock;
        for (int i = threadIdx.x; i < NC * 64 * 4; i += 128)
          if (((i >> 2) & 63) >= held - key0)
            *reinterpret_cast<uint4*>(vb + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
      }
      float s[64];
      uint32_t pk[32];
      if (!empty) {
        tmem_ld32(tmem_s, *reinterpret_cast<float(*)[32]>(&s[0]));
        tmem_ld32(tmem_s + 32, *reinterpret_cast<float(*)[32]>(&s[32]));
        tmem_wait_ld();
        if (!whole) {
          const uint64_t vis = bits_below((long long)(own ? lim1 : lim0) - key0);
#pragma unroll
          for (int c = 0; c < 64; ++c) s[c] = ((vis >> c) & 1ull) ? s[c] : -INFINITY;
        }
      }
      auto row_max = [&]() -> float {
        float a = max3_nan(s[0], s[1], s[2]), b = max3_nan(s[3], s[4], s[5]);
        float c = max3_nan(s[6], s[7], s[8]), d = max3_nan(s[9], s[10], s[11]);
#pragma unroll
        for (int x = 12; x < 60; x += 8) {
          a = max3_nan(a, s[x], s[x + 1]);
          b = max3_nan(b, s[x + 2], s[x + 3]);
          c = max3_nan(c, s[x + 4], s[x + 5]);
          d = max3_nan(d, s[x + 6], s[x + 7]);
        }
        return max_nan(max3_nan(a, b, max3_nan(s[60], s[61], s[62])), max3_nan(c, d, s[63]));
      };
      auto exp_block = [&](float nm) -> float {
        float2 t0 = make_float2(0.f, 0.f), t1 = t0;
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const float2 x = fma2(make_float2(s[2 * c], s[2 * c + 1]), make_float2(sc, sc),
                                make_float2(nm, nm));
          const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
          if (c & 1) t1 = add2(t1, e);
          else t0 = add2(t0, e);
          pk[c] = DType<DT>::pack2(e.x, e.y);
        }
        t0 = add2(t0, t1);
        return t0.x + t0.y;
      };
      // P against the row's reference straight away, without looking for its
      // maximum: a sum below 2^15 says that every P is (fp16 holds it).  Only
      // if some row passes that does the warp look, move the references,
      // rescale O and compute P again.  While some row of the warp has no
      // reference (it has seen nothing yet, or never will), there are no sums
      // to go by: the warp looks, and every row's maximum is held to 2^15.
      const bool spec = !empty && all(m != -INFINITY);
      float sum = INFINITY, mn = m;
      if (spec) sum = exp_block(-m);
      bool need = !empty && !(sum < kTileSum);
      if (__any_sync(0xffffffffu, need)) {
        mn = next_ref(m, row_max() * sc);
        need = mn > m && (spec ? need : m == -INFINITY || mn - m >= kTileRise);
      }
      bool again = !spec;
      if (__any_sync(0xffffffffu, need)) {
        if (j > 0) {
          if (!all(mbar_wait(&pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1, 138))) {
            ok = false;
            break;
          }
          tc_fence_after();
        }
        const float f = need ? (m == -INFINITY ? 0.f : fast_exp2(m - mn)) : 1.f;
        l *= f;
        if (j > 0) {
#pragma unroll
          for (int c = 0; c < DK / 16; ++c) {
            float o[16];
            tmem_ld16(lane_base + 128 + c * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int x = 0; x < 16; ++x) o[x] *= f;
            tmem_st16(lane_base + 128 + c * 16, o);
          }
          tmem_wait_st();
        }
        if (need) m = mn;
        again = true;
      }
      if (again) {
        if (empty || m == -INFINITY) {  // nothing seen yet
          sum = 0.f;
#pragma unroll
          for (int c = 0; c < 32; ++c) pk[c] = 0u;
        } else {
          sum = exp_block(-m);
        }
      }
      l += sum;
      tmem_st32u(tmem_s, pk);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[j & 1]);
    }

    // ---- epilogue ------------------------------------------------------------
    if (ok && nent > 0) {
      ok = all(mbar_wait(&pv_done[(nent - 1) & 1], ((nent - 1) >> 1) & 1, 139));
      tc_fence_after();
    }
    if (!ok) *abort_flag = 1;
    const long long grow = ((long long)b * p.Hq + hd) * p.Sq + tk;
    const bool direct = p.NS == 1;
    const bool seen = m != -INFINITY && ok;
    const long long at = grow * p.NS + gr.slot0 + sp;
    // Every product has run, so the ring is free: each thread lays its row
    // there (padded, so that 16-byte stores of a warp do not collide) and
    // sends it off with one bulk copy.
    const float inv = seen && l > 0.f ? 1.f / l : 0.f;
    uint8_t* orow = smem + L::kKOff + row * L::kOPitch;
    if (nent > 0 || direct) {
#pragma unroll
      for (int c = 0; c < DK / 32; ++c) {
        float o[32];
        __syncwarp();
        if (nent > 0 && ok) {
          tmem_ld32(lane_base + 128 + c * 32, o);
          tmem_wait_ld();
        }
        if (direct) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (seen) {
              x.x = DType<DT>::pack2(o[u * 8] * inv, o[u * 8 + 1] * inv);
              x.y = DType<DT>::pack2(o[u * 8 + 2] * inv, o[u * 8 + 3] * inv);
              x.z = DType<DT>::pack2(o[u * 8 + 4] * inv, o[u * 8 + 5] * inv);
              x.w = DType<DT>::pack2(o[u * 8 + 6] * inv, o[u * 8 + 7] * inv);
            }
            *reinterpret_cast<uint4*>(orow + c * 64 + u * 16) = x;
          }
        } else {
#pragma unroll
          for (int u = 0; u < 8; ++u)
            *reinterpret_cast<float4*>(orow + c * 128 + u * 16) =
                make_float4(o[u * 4], o[u * 4 + 1], o[u * 4 + 2], o[u * 4 + 3]);
        }
      }
      fence_proxy_async_smem();
      if (live && ok && (direct || seen)) {
        if (direct)
          bulk_store(p.out + b * p.os_b + hd * p.os_h + tk * p.os_s, orow, p.D * 2);
        else
          bulk_store(p.opart + at * p.D, orow, p.D * 4);
        bulk_commit();
        bulk_wait0();
      }
    }
    if (live) {
      if (!direct) p.ml[at] = make_float2(m, l);
      else if (p.lse) p.lse[grow] = seen ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) let_land();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
  // The own caches' kernel of the same call may still run: end after it, so that
  // what waits for this kernel waits for both.
  pdl_wait();
}

template <typename DT, int DK>
static int launch_tiles_t(const TileParams& tp, const mi_rows& kp, const mi_rows& vp,
                          const mi_rows& k, const mi_rows& v, bool after,
                          cudaStream_t st) {
  using L = TileSmem<DK>;
  const CacheParams& p = tp.c;
  CUtensorMap m[4];
  memset(m, 0, sizeof(m));
  const mi_rows* t[4] = {&kp, &vp, &k, &v};
  const bool use0 = (tp.grp[0].items && tp.grp[0].use0) || (tp.grp[1].items && tp.grp[1].use0);
  const bool use1 = (tp.grp[0].items && tp.grp[0].use1) || (tp.grp[1].items && tp.grp[1].use1);
  for (int i = 0; i < 4; ++i) {
    if (!(i < 2 ? use0 : use1)) continue;
    const CacheSeg& s = p.seg[i / 2];
    const int rc = make_rows4_map(&m[i], *t[i], s.nb, p.Hkv, s.cap, p.D, 32, 64);
    if (rc != MI_OK) return rc;
  }
  constexpr auto kern = cache_tiles_kernel<DT, DK>;
  cudaError_t err = allow_smem<cache_tiles_kernel<DT, DK>>(L::kAlloc);
  if (err == cudaSuccess) {
    const dim3 grid((unsigned)(tp.grp[0].items + tp.grp[1].items));
    if (after) {
      err = launch_after(kern, grid, kTileThreads, L::kAlloc, st, m[0], m[1], m[2], m[3], tp);
    } else {
      kern<<<grid, kTileThreads, L::kAlloc, st>>>(m[0], m[1], m[2], m[3], tp);
      err = cudaGetLastError();
    }
  }
  if (err != cudaSuccess) {
    debug_launch_failure("cache_tiles_kernel", reinterpret_cast<const void*>(kern), err,
                         kTileThreads, L::kAlloc);
    return MI_ERR_LAUNCH;
  }
  return MI_OK;
}

static int launch_tiles(const TileParams& tp, int dtype, const mi_rows& kp, const mi_rows& vp,
                        const mi_rows& k, const mi_rows& v, bool after,
                        cudaStream_t st) {
  const bool bf = dtype == MI_BF16;
  const int D = tp.c.D;
  if (D <= 64)
    return bf ? launch_tiles_t<__nv_bfloat16, 64>(tp, kp, vp, k, v, after, st)
              : launch_tiles_t<__half, 64>(tp, kp, vp, k, v, after, st);
  if (D <= 96)
    return bf ? launch_tiles_t<__nv_bfloat16, 96>(tp, kp, vp, k, v, after, st)
              : launch_tiles_t<__half, 96>(tp, kp, vp, k, v, after, st);
  return bf ? launch_tiles_t<__nv_bfloat16, 128>(tp, kp, vp, k, v, after, st)
            : launch_tiles_t<__half, 128>(tp, kp, vp, k, v, after, st);
}

}  // namespace mib200
