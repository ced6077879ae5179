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
// Many rows: S^T = K Q^T on tcgen05, a tile of 128 keys (the M rows, one per
// thread) against blocks of 64 query rows.  A key's weight is then a sum along
// its own TMEM lane: 64 exponentials and adds per block and thread, no exchange
// between threads, nothing written back.  Bound by the exponentials (16 per
// clock and SM).  What a cache holds past its length stays in its own lanes,
// whose sums are dropped.
//
// RESQ: all rows of the key/value head (at most QS blocks, packed over its
// query heads) stay in shared memory while key tiles stream; otherwise a key
// tile stays while the blocks of each head's rows that see it stream.
// ---------------------------------------------------------------------------
template <int DK>
struct ColsSmem {
  static constexpr int NC = DK / 32;
  static constexpr int KS = 2, QS = DK == 128 ? 2 : (DK == 96 ? 4 : 6), SB = 4;
  static constexpr int kKTile = NC * 128 * 64, kQBlock = NC * 64 * 64;
  static constexpr int kQOff = KS * kKTile;
  static constexpr int kRowOff = kQOff + QS * kQBlock;  // per warp: 64 x (-lse), 64 x token
  static constexpr int kBarOff = kRowOff + 4 * 2 * 512;
  // k_full[KS] k_empty[KS] q_full[QS] q_empty[QS] s_full[SB] s_empty[SB]
  static constexpr int kSlotOff = kBarOff + (2 * KS + 2 * QS + 2 * SB) * 8;
  static constexpr int kAlloc = kSlotOff + 8 + 512;
  static constexpr uint32_t kTmemCols = SB * 64;
  static_assert(kAlloc <= 113 * 1024, "two blocks per SM");
};

struct ColsParams {
  WeightParams w;
  int tiles, per;    // key tiles of a (b, h); tiles per item
  int ranges;        // items per (b, h)
};

template <typename DT, int DK, bool RESQ>
__global__ void __launch_bounds__(192, 2)
    weight_tiles_kernel(const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_q,
                        const __grid_constant__ ColsParams cp) {
  using L = ColsSmem<DK>;
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

  long long it = blockIdx.x;
  const int range = (int)(it % cp.ranges);
  it /= cp.ranges;
  const int h = (int)(it % p.Hkv), b = (int)(it / p.Hkv);
  const int len = p.len ? min(max(p.len[b], 0), p.C) : p.C;
  const int t0 = range * cp.per, t1 = min(cp.tiles, t0 + cp.per);
  const int tv = min(t1, (len + 127) >> 7);  // tiles from tv on hold no valid key
  const int rows = p.group * p.Sq;
  const int nsb = RESQ ? (rows + 63) >> 6 : (p.Sq + 63) >> 6;
  // First 64-row block of a head that sees key tile t.
  auto first_block = [&](int t) {
    return !RESQ && p.causal ? max(0, t * 128 - len + p.Sq) >> 6 : 0;
  };
  const int heads = RESQ ? 1 : p.group;

  if (threadIdx.x == 0) {
    for (int i = 0; i < KS; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < QS; ++i) mbar_init(&q_full[i], 1), mbar_init(&q_empty[i], 1);
    for (int i = 0; i < SB; ++i) mbar_init(&s_full[i], 1), mbar_init(&s_empty[i], 128);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, L::kTmemCols);
    tmem_relinquish();
  }
  if constexpr (RESQ) {
    if (tv > t0) {
      for (int i = threadIdx.x; i < nsb * 64 * (DK / 8); i += 192) {
        const int r = i / (DK / 8), u = i - r * (DK / 8);
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < rows && u * 8 < p.D)
          x = *reinterpret_cast<const uint4*>(p.q + b * p.qs_b +
                                              (long long)(h * p.group + r / p.Sq) * p.qs_h +
                                              (long long)(r % p.Sq) * p.qs_s + u * 8);
        *reinterpret_cast<uint4*>(smem + L::kQOff + (r >> 6) * L::kQBlock + (u >> 2) * (64 * 64) +
                                  (r & 63) * 64 + (((u & 3) ^ ((r >> 1) & 3)) << 4)) = x;
      }
    }
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 4) {
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
        if constexpr (!RESQ) {
          for (int g = 0; ok && g < heads; ++g)
            for (int sb = first_block(t); sb < nsb; ++sb, ++nq) {
              const int qs = nq % QS, qu = nq / QS;
              if (qu > 0 && !mbar_wait(&q_empty[qs], (qu - 1) & 1, 142)) { ok = false; break; }
              mbar_arrive_expect_tx(&q_full[qs], L::kQBlock);
              for (int c = 0; c < NC; ++c)
                tma_load_4d(smem + L::kQOff + qs * L::kQBlock + c * (64 * 64), &tm_q, &q_full[qs],
                            c * 32, sb * 64, h * p.group + g, b);
            }
        }
      }
      if (!ok) *abort_flag = 1;
    }
  } else if (warp == 5) {
    constexpr uint32_t idesc = make_idesc_f16(DType<DT>::kBF16, 128, 64, false, false);
    const uint64_t kd0 = make_desc_sw64(smem_u32(smem), 16, 512);
    const uint64_t qd0 = make_desc_sw64(smem_u32(smem + L::kQOff), 16, 512);
    auto all = [](bool x) { return __all_sync(0xffffffffu, x) != 0; };
    bool ok = true;
    int n = 0;
    for (int t = t0; ok && t < tv; ++t) {
      const int st = (t - t0) % KS;
      if (*abort_flag) { ok = false; break; }
      if (!all(mbar_wait(&k_full[st], ((t - t0) / KS) & 1, 143))) { ok = false; break; }
      const int f = first_block(t);
      for (int g = 0; ok && g < heads; ++g)
        for (int sb = f; sb < nsb; ++sb, ++n) {
          const int qs = RESQ ? sb : n % QS, buf = n % SB;
          if (!RESQ && !all(mbar_wait(&q_full[qs], (n / QS) & 1, 144))) { ok = false; break; }
          if (n >= SB && !all(mbar_wait(&s_empty[buf], (n / SB - 1) & 1, 145))) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one_sync()) {
            const uint64_t kd = kd0 + (uint64_t)((st * L::kKTile) >> 4);
            const uint64_t qd = qd0 + (uint64_t)((qs * L::kQBlock) >> 4);
#pragma unroll
            for (int ks = 0; ks < DK / 16; ++ks) {
              const uint32_t off = (ks & 1) * 32;
              umma_f16_ss(tmem_base + buf * 64, kd + (((ks >> 1) * (128 * 64) + off) >> 4),
                          qd + (((ks >> 1) * (64 * 64) + off) >> 4), idesc, ks > 0 ? 1u : 0u);
            }
            umma_commit(&s_full[buf]);
            if constexpr (!RESQ) umma_commit(&q_empty[qs]);
            if (g == heads - 1 && sb == nsb - 1) umma_commit(&k_empty[st]);
          }
          __syncwarp();
        }
    }
    if (!ok && lane == 0) *abort_flag = 1;
  } else {
    const uint32_t lane_base = tmem_base + ((uint32_t)(warp * 32) << 16);
    float* srow = reinterpret_cast<float*>(smem + L::kRowOff) + warp * 256;
    const float* win = p.win ? p.win + b * p.wi_b + h * p.wi_h : nullptr;
    float* wout = p.wout + b * p.wo_b + h * p.wo_h;
    bool ok = true;
    auto all = [](bool x) { return __all_sync(0xffffffffu, x) != 0; };
    int n = 0;
    for (int t = t0; t < t1; ++t) {
      const int j = t * 128 + threadIdx.x;
      float tot = 0.f;
      // token from which a row sees the key; whole: every row of the block does
      const int smin = p.causal ? j - len + p.Sq : 0;
      const int wmin = __shfl_sync(0xffffffffu, smin, 31);
      if (ok && t < tv) {
        const int f = first_block(t);
        for (int g = 0; ok && g < heads; ++g)
          for (int sb = f; sb < nsb; ++sb, ++n) {
            // this block's rows: -lse (log2 units; -inf: adds nothing) and tokens
            float* nz = srow + (n & 1) * 128;
            int* tok = reinterpret_cast<int*>(nz) + 64;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int r = sb * 64 + lane + 32 * x;
              const int hd = RESQ ? r / p.Sq : g, s = RESQ ? r - hd * p.Sq : r;
              float z = -INFINITY;
              if (RESQ ? r < rows : s < p.Sq)
                z = p.lse[((long long)b * p.Hq + h * p.group + hd) * p.Sq + s];
              nz[lane + 32 * x] = z == -INFINITY ? z : -z * p.lse_mul;
              tok[lane + 32 * x] = s;
            }
            __syncwarp();
            const int buf = n % SB;
            if (!all(mbar_wait(&s_full[buf], (n / SB) & 1, 146))) { ok = false; break; }
            tc_fence_after();
            float s[64];
            tmem_ld32(lane_base + buf * 64, *reinterpret_cast<float(*)[32]>(&s[0]));
            tmem_ld32(lane_base + buf * 64 + 32, *reinterpret_cast<float(*)[32]>(&s[32]));
            tmem_wait_ld();
            tc_fence_before();
            mbar_arrive(&s_empty[buf]);
            const bool whole = RESQ ? wmin <= 0 : wmin <= sb * 64;
            float2 a0 = make_float2(0.f, 0.f), a1 = a0;
            if (whole) {
#pragma unroll
              for (int c = 0; c < 64; c += 4) {
                const float4 z = *reinterpret_cast<const float4*>(nz + c);
                a0 = add2(a0, make_float2(fast_exp2(fmaf(s[c], p.scale_log2, z.x)),
                                          fast_exp2(fmaf(s[c + 1], p.scale_log2, z.y))));
                a1 = add2(a1, make_float2(fast_exp2(fmaf(s[c + 2], p.scale_log2, z.z)),
                                          fast_exp2(fmaf(s[c + 3], p.scale_log2, z.w))));
              }
            } else {
#pragma unroll
              for (int c = 0; c < 64; ++c)
                if (tok[c] >= smin) a0.x += fast_exp2(fmaf(s[c], p.scale_log2, nz[c]));
            }
            a0 = add2(a0, a1);
            tot += a0.x + a0.y;  // two-level sum: a block, then the blocks
          }
      }
      if (j < len) {
        if (ok) wout[j] = (win ? win[j] : 0.f) + tot;
      } else if (j < p.C && win != wout) {
        wout[j] = win ? win[j] : 0.f;
      }
    }
    if (!ok) *abort_flag = 1;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

template <typename DT, int DK>
static int launch_weight_tiles(const WeightParams& w, const mi_rows& q, const mi_rows& k,
                               cudaStream_t st) {
  using L = ColsSmem<DK>;
  ColsParams cp{};
  cp.w = w;
  cp.tiles = (w.C + 127) / 128;
  const long long rows = (long long)w.group * w.Sq;
  const bool resq = rows <= 64 * L::QS;
  const long long all = (long long)w.B * w.Hkv * cp.tiles;
  // tiles per item: with resident rows, three rounds of two items per SM;
  // otherwise enough that an item has 16 blocks
  const long long steps = (long long)w.group * ((w.Sq + 63) / 64);
  long long per = resq ? (all + 148 * 6 - 1) / (148 * 6) : (16 + steps - 1) / steps;
  cp.per = (int)(per < 1 ? 1 : (per > cp.tiles ? cp.tiles : per));
  cp.ranges = (cp.tiles + cp.per - 1) / cp.per;
  const long long items = (long long)w.B * w.Hkv * cp.ranges;
  if (items > 0x7fffffffll) return MI_ERR_SHAPE;
  CUtensorMap tk, tq;
  memset(&tq, 0, sizeof(tq));
  int rc = make_rows4_map(&tk, k, w.B, w.Hkv, w.C, w.D, 32, 128);
  if (rc == MI_OK && !resq) rc = make_rows4_map(&tq, q, w.B, w.Hq, w.Sq, w.D, 32, 64);
  if (rc != MI_OK) return rc;
  auto kern = resq ? weight_tiles_kernel<DT, DK, true> : weight_tiles_kernel<DT, DK, false>;
  cudaError_t err = resq ? allow_smem<weight_tiles_kernel<DT, DK, true>>(L::kAlloc)
                         : allow_smem<weight_tiles_kernel<DT, DK, false>>(L::kAlloc);
  if (err == cudaSuccess) {
    kern<<<(unsigned)items, 192, L::kAlloc, st>>>(tk, tq, cp);
    err = cudaGetLastError();
  }
  if (err != cudaSuccess) {
    debug_launch_failure("weight_tiles_kernel", reinterpret_cast<const void*>(kern), err, 192,
                         L::kAlloc);
    return MI_ERR_LAUNCH;
  }
  return MI_OK;
}

static int launch_weights_many(const WeightParams& p, int dtype, const mi_rows& q,
                               const mi_rows& k, cudaStream_t st) {
  const bool bf = dtype == MI_BF16;
  if (p.D <= 64)
    return bf ? launch_weight_tiles<__nv_bfloat16, 64>(p, q, k, st)
              : launch_weight_tiles<__half, 64>(p, q, k, st);
  if (p.D <= 96)
    return bf ? launch_weight_tiles<__nv_bfloat16, 96>(p, q, k, st)
              : launch_weight_tiles<__half, 96>(p, q, k, st);
  return bf ? launch_weight_tiles<__nv_bfloat16, 128>(p, q, k, st)
            : launch_weight_tiles<__half, 128>(p, q, k, st);
}

}  // namespace mib200

using namespace mib200;

extern "C" size_t mi_attn_weights_workspace_size(const mi_attn_weights_args* a) {
  if (!a || !cache_sizes_ok(a->B, a->Hq, a->Hkv, a->S_q, 1, 0, a->C, a->D)) return SIZE_MAX;
  if (a->B == 0 || a->Hq == 0 || a->S_q == 0 || a->C == 0 || a->lse) return 0;
  const CachePlan pl = cache_plan(a->B, a->Hkv, a->Hq / a->Hkv, a->S_q, 1, 0, a->C);
  const size_t rows = (size_t)(a->B * a->Hq * a->S_q);
  if ((double)rows * pl.NS > 1e13) return SIZE_MAX;
  return align_up(rows * pl.NS * 8) + align_up(rows * 4);
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

  // the rows' split, for their statistics and for the few-row form of the weights
  const CachePlan pl = cache_plan(B, Hkv, group, S_q, 1, 0, C);
  const size_t rows = (size_t)(B * Hq * S_q);
  CacheParams p{};
  p.q = w.q;
  p.qs_b = w.qs_b;
  p.qs_h = w.qs_h;
  p.qs_s = w.qs_s;
  p.Hq = w.Hq;
  p.Hkv = w.Hkv;
  p.group = w.group;
  p.Sq = w.Sq;
  p.D = w.D;
  p.scale_log2 = w.scale_log2;
  p.seg[0].seqs = 1;
  set_seg(p.seg[1], k, k, lengths, C, B, 1, group * S_q, w.causal);
  p.seg[1].rtiles = pl.rtiles[1];
  p.seg[1].nsplit = pl.nsplit[1];
  p.seg[1].chunk = pl.chunk[1];
  p.NS = pl.NS;
  const long long items = (long long)B * Hkv * pl.rtiles[1] * pl.nsplit[1];
  if (items > 0x7fffffffll) return MI_ERR_SHAPE;
  if (!lse) {
    p.ml = static_cast<float2*>(workspace);
    float* lse2 = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                           align_up(rows * pl.NS * 8));
    if (pl.tile[1]) {
      TileParams tp{};
      tp.c = p;
      tp.grp[1] = {1, 0, 1, pl.rtiles[1], pl.nsplit[1], pl.chunk[1] / 64, 0, items};
      rc = launch_tiles<true>(tp, dtype, k, k, k, k, st);
    } else {
      rc = launch_rows_dk<kStats>(p, dtype, pl.nt, items, false, st);
    }
    if (rc != MI_OK) return rc;
    weight_lse_kernel<<<(unsigned)((rows + 255) / 256), 256, 0, st>>>(p.ml, pl.NS, lse2,
                                                                      (long long)rows);
    if (cudaGetLastError() != cudaSuccess) return MI_ERR_LAUNCH;
    w.lse = lse2;
    w.lse_mul = 1.f;
  }
  if (pl.tile[1]) return launch_weights_many(w, dtype, q, k, st);
  p.z = w.lse;
  p.z_mul = w.lse_mul;
  p.win = w.win;
  p.wi_b = w.wi_b;
  p.wi_h = w.wi_h;
  p.wout = w.wout;
  p.wo_b = w.wo_b;
  p.wo_h = w.wo_h;
  return launch_rows_dk<kWeights>(p, dtype, pl.nt, items, false, st);
}
