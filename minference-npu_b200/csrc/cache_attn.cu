// Attention over a shared prefix and per-sequence caches: the kernel for few
// query rows, the kernel that joins partial results, and the C entry point.
// The split of the work is described at the top of cache_attn.cuh.
#include "cache_attn.cuh"
#include "cache_tiles.cu"
#include "host_util.h"
#include "mma_sync.cuh"

namespace mib200 {

// ---------------------------------------------------------------------------
// Few rows: a work item is a tile of up to 8 rows against `chunk` keys.  Its
// warps take groups of 16 keys in turn; each warp streams its own groups
// through its own shared-memory ring (cp.async) and keeps its own running
// maximum, sum and O, so there is no barrier in the loop.  Their states are
// joined at the end.  Bound by the cache's bytes.  Keys are the M side of both
// products, so that a single row costs an 8-wide tile, not a 16-wide one:
//   S^T (16 keys x 8 rows) = K Q^T     Q fragments stay in registers
//   O^T (D x 8 rows) += V^T P^T        P^T is S^T's registers rounded to the
//                                      inputs' type and transposed in place
// Rows of a ring stage are padded by 16 bytes, which makes the ldmatrix rows
// of 128, 192 and 256 bytes fall into distinct banks.  P is rounded because both
// operands of a product have one type; the row sums are taken before.  Keys past
// the end of the range are filled with zeros instead of being read, so whatever a
// cache holds past its length cannot reach O through 0 * V.
// Measured: two caches of 65536 and 49152 keys, 32 heads of 96, 219 us
// (6.4 TB/s); 201 MB of 1024-key caches 39 us.  With the rows as the M side and
// two blocks of 100 KB an SM the first took 257 us.
//
// kStats: the rows' (maximum, sum) only; no V.
// kWeights: given the lse of all the head's rows (one tile), a key's weight is
// summed over them and added to win; no V.  16 caches of 8192 keys, 8 heads of
// 128: 40 us (5.1 TB/s).
// ---------------------------------------------------------------------------
enum RowsMode { kAttention, kStats, kWeights };

template <int DK, RowsMode MODE>
struct RowsSmem {
  // A warp waits on its own instruction latencies more than on memory, so four
  // warps share a block's bytes in flight.
  static constexpr int W = 4;
  static constexpr int kPitch = DK * 2 + 16;
  static constexpr int kTile = 16 * kPitch;  // 16 keys of K or V
  // one warp's stage; kWeights: and 16 of win
  static constexpr int kStage = MODE == kAttention ? 2 * kTile
                                                   : kTile + (MODE == kWeights ? 64 : 0);
  // four blocks per SM (three for the attention's 70 KB at D = 128)
  static constexpr int kFit =
      (MODE == kAttention && DK == 128 ? 70 * 1024 : 55 * 1024) / (W * kStage);
  static constexpr int ST = kFit > 8 ? 8 : kFit;
  static_assert(ST >= 2, "a stage to load beside the one in use");
  static constexpr int kWarpRing = ST * kStage;
  static constexpr int kRing = W * kWarpRing;
};

template <typename DT, int DK, RowsMode MODE>
__global__ void __launch_bounds__(32 * RowsSmem<DK, MODE>::W,
                                  MODE == kAttention && DK == 128 ? 3 : 4)
    cache_rows_kernel(const __grid_constant__ CacheParams p) {
  using L = RowsSmem<DK, MODE>;
  constexpr int kRowsWarps = L::W;
  constexpr int KS = DK / 16, R = 8, CPR = DK / 8;
  constexpr bool kO = MODE == kAttention;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float sm_m[kRowsWarps][R], sm_l[kRowsWarps][R];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch();

  int it = blockIdx.x, rt, sp, h;
  const bool own = it >= p.items0;
  if (own) it -= p.items0;
  const CacheSeg& sg = p.seg[own ? 1 : 0];
  it = sg.rtiles.divmod(it, rt);
  it = sg.nsplit.divmod(it, sp);
  const int e = p.div_hkv.divmod(it, h);
  const int r0 = rt * R;
  const int nrows = min(R, sg.rows - r0);
  const int len = cache_len(sg, e);
  // Keys that the tile's last token sees (its rows cover tokens in order
  // unless they wrap into another head).
  int end = len;
  if (sg.causal) {
    const int last = r0 + nrows - 1;
    int smax;
    if (p.div_sq.divmod(last, smax) != p.div_sq.div(r0)) smax = p.Sq - 1;
    end = max(0, len - (p.Sq - 1 - smax));
  }
  const int kb = sp * sg.chunk;
  const int ke = (int)min((long long)kb + sg.chunk, (long long)end);
  const int ngroups = ke > kb ? (ke - kb + 15) >> 4 : 0;

  const float* win = nullptr;
  float* wout = nullptr;
  if constexpr (MODE == kWeights) {
    win = p.win ? p.win + e * p.wi_b + h * p.wi_h : nullptr;
    wout = p.wout + e * p.wo_b + h * p.wo_h;
  }

  // ---- loader: lane l brings 16-byte pieces (l&3) + 4v of rows l/4 and l/4+8 -
  const uint32_t ring = smem_u32(smem) + warp * L::kWarpRing;
  const int lrow = lane >> 2, lcol = lane & 3;
  const uint32_t ldst = ring + lrow * L::kPitch + lcol * 16;
  const uint16_t* kbase = sg.k + e * sg.ks_b + h * sg.ks_h + lcol * 8;
  const uint16_t* vbase = kO ? sg.v + e * sg.vs_b + h * sg.vs_h + lcol * 8 : nullptr;
  auto load = [&](int g) {
    if (g < ngroups) {
      const uint32_t off = ((g / kRowsWarps) % L::ST) * L::kStage;
      const uint32_t st = ldst + off;
      const int key = kb + g * 16 + lrow;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bool in = key + 8 * u < ke;
        const long long kk = in ? key + 8 * u : 0;
        const uint16_t* kr = kbase + kk * sg.ks_s;
        const uint16_t* vr = kO ? vbase + kk * sg.vs_s : nullptr;
#pragma unroll
        for (int v = 0; v < CPR / 4; ++v) {
          const bool ok = in && (lcol + 4 * v) * 8 < p.D;
          cp16(st + u * 8 * L::kPitch + v * 64, ok ? kr + v * 32 : kbase, ok);
          if constexpr (kO)
            cp16(st + L::kTile + u * 8 * L::kPitch + v * 64, ok ? vr + v * 32 : vbase, ok);
        }
      }
      if constexpr (MODE == kWeights) {
        const int j = kb + g * 16 + lane;
        if (lane < 16 && win) cp4(ring + off + L::kTile + lane * 4, j < ke ? win + j : win, j < ke);
      }
    }
    cp_commit();
  };

  // ---- Q: every warp fetches the rows for itself, ahead of its first keys (whose
  // loads would otherwise queue before them), through the ring stage that is
  // loaded last, into fragments ---------------------------------------------------
  uint8_t* qs = smem + warp * L::kWarpRing + (L::ST - 1) * L::kStage;
  constexpr int kQIter = R * CPR / 32;
  uint4 qx[kQIter];
  {
    const uint16_t* qp = p.q;  // lanes 0-7 work the rows' addresses out
    if (lane < nrows) {
      int b, hd, tk;
      cache_row(p, sg, e, h, r0 + lane, b, hd, tk);
      qp += b * p.qs_b + hd * p.qs_h + tk * p.qs_s;
    }
#pragma unroll
    for (int i = 0; i < kQIter; ++i) {
      const int r = (i * 32 + lane) / CPR, c = (i * 32 + lane) % CPR;
      const unsigned long long a =
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(qp), r);
      qx[i] = make_uint4(0, 0, 0, 0);
      if (r < nrows && c * 8 < p.D)
        qx[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a) + c * 8);
    }
  }
#pragma unroll
  for (int s = 0; s < L::ST - 1; ++s) load(warp + s * kRowsWarps);
#pragma unroll
  for (int i = 0; i < kQIter; ++i) {
    const int r = (i * 32 + lane) / CPR, c = (i * 32 + lane) % CPR;
    *reinterpret_cast<uint4*>(qs + r * L::kPitch + c * 16) = qx[i];
  }
  __syncwarp();
  uint32_t qf[KS][2];
#pragma unroll
  for (int ks = 0; ks < KS; ks += 2) {
    uint32_t b[4];
    ldsm4(b, smem_u32(qs) + (lane & 7) * L::kPitch + ks * 32 + (lane >> 3) * 16);
    qf[ks][0] = b[0], qf[ks][1] = b[1], qf[ks + 1][0] = b[2], qf[ks + 1][1] = b[3];
  }
  __syncwarp();
  int lim[2];  // keys that row (lane & 3) * 2 + x sees
  int minlim = 0x7fffffff;
  float nz[2];  // kWeights: -lse (log2 units; -inf: the row adds nothing)
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int r = (lane & 3) * 2 + x;
    lim[x] = 0;
    nz[x] = -INFINITY;
    if (r < nrows) {
      int tok;
      const int g = p.div_sq.divmod(r0 + r, tok);
      lim[x] = sg.causal ? len - (p.Sq - 1 - tok) : len;
      minlim = min(minlim, lim[x]);
      if constexpr (MODE == kWeights) {
        const float z = p.z[((long long)e * p.Hq + h * p.group + g) * p.Sq + tok];
        if (z != -INFINITY) nz[x] = -z * p.z_mul;
      }
    }
  }
  minlim = __reduce_min_sync(0xffffffffu, minlim);

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[kO ? DK / 16 : 1][4];
  if constexpr (kO)
#pragma unroll
    for (int d = 0; d < DK / 16; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;

  for (int g = warp; g < ngroups; g += kRowsWarps) {
    load(g + (L::ST - 1) * kRowsWarps);
    cp_wait<L::ST - 1>();
    __syncwarp();
    const uint32_t st = ring + ((g / kRowsWarps) % L::ST) * L::kStage;
    // two accumulators: the products of one wait for each other
    float s[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
    const uint32_t ka = st + (lane & 15) * L::kPitch + (lane >> 4) * 16;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t a[4];
      ldsm4(a, ka + ks * 32);
      mma16816<DT>((ks & 1) ? s2 : s, a, qf[ks][0], qf[ks][1]);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) s[c] += s2[c];
    const int key0 = kb + g * 16;
    const bool full = key0 + 16 <= min(minlim, ke);
    if constexpr (MODE == kWeights) {
      float t0 = 0.f, t1 = 0.f;  // keys lane/4 and lane/4 + 8
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int key = key0 + (lane >> 2), lm = min(lim[x], ke);
        const float p0 = fast_exp2(fmaf(s[x], p.scale_log2, nz[x]));
        const float p1 = fast_exp2(fmaf(s[2 + x], p.scale_log2, nz[x]));
        t0 += full || key < lm ? p0 : 0.f;
        t1 += full || key + 8 < lm ? p1 : 0.f;
      }
      t0 += __shfl_xor_sync(0xffffffffu, t0, 1);
      t1 += __shfl_xor_sync(0xffffffffu, t1, 1);
      t0 += __shfl_xor_sync(0xffffffffu, t0, 2);
      t1 += __shfl_xor_sync(0xffffffffu, t1, 2);
      // lanes 4i and 4i+1 write keys i and i + 8
      if ((lane & 3) < 2) {
        const int i = (lane >> 2) + 8 * (lane & 1);
        float w = (lane & 1) ? t1 : t0;
        if (win)
          w += *reinterpret_cast<const float*>(smem + (st - smem_u32(smem)) + L::kTile + i * 4);
        if (key0 + i < ke) wout[key0 + i] = w;
      }
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) s[c] *= p.scale_log2;
      if (!full) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (key0 + (lane >> 2) + 8 * (c >> 1) >= min(lim[c & 1], ke)) s[c] = -INFINITY;
      }
      float pr[4], f[2];
      bool grew = false;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float t = fmaxf(s[x], s[2 + x]);
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
        const float mn = fmaxf(m[x], t);
        const float base = mn == -INFINITY ? 0.f : mn;
        f[x] = fast_exp2(m[x] - base);
        grew |= mn != m[x];
        m[x] = mn;
        pr[x] = fast_exp2(s[x] - base);
        pr[2 + x] = fast_exp2(s[2 + x] - base);
        l[x] = l[x] * f[x] + (pr[x] + pr[2 + x]);
      }
      if constexpr (kO) {
        const uint32_t pb0 = movm_t(DType<DT>::pack2(pr[0], pr[1]));
        const uint32_t pb1 = movm_t(DType<DT>::pack2(pr[2], pr[3]));
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int d = 0; d < DK / 16; ++d)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[d][c] *= f[c & 1];
        }
        const uint32_t va = st + L::kTile + ((lane & 7) + ((lane >> 4) << 3)) * L::kPitch +
                            ((lane >> 3) & 1) * 16;
#pragma unroll
        for (int d = 0; d < DK / 16; ++d) {
          uint32_t a[4];
          ldsm4_t(a, va + d * 32);
          mma16816<DT>(o[d], a, pb0, pb1);
        }
      }
    }
    __syncwarp();  // the stage is free for the load of the next step
  }
  cp_wait<0>();

  if constexpr (MODE == kWeights) {
    // keys of the range past the length: their weights pass through
    const int last = (int)min((long long)kb + sg.chunk, (long long)sg.cap);
    if (win != wout)
      for (int j = max(kb, max(ke, 0)) + tid; j < last; j += 32 * kRowsWarps)
        wout[j] = win ? win[j] : 0.f;
    return;
  }

  // ---- join the warps ---------------------------------------------------------
  constexpr int kOP = DK + 4;  // floats per row of O in shared memory
  __syncthreads();
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 4);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 8);
    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 16);
    const int r = (lane & 3) * 2 + x;
    if (lane < 4) {
      sm_m[warp][r] = m[x];
      sm_l[warp][r] = l[x];
    }
    if constexpr (kO) {
      float* row = reinterpret_cast<float*>(smem) + (warp * R + r) * kOP + (lane >> 2);
#pragma unroll
      for (int d = 0; d < DK / 16; ++d) {
        row[d * 16] = o[d][x];
        row[d * 16 + 8] = o[d][2 + x];
      }
    }
  }
  __syncthreads();
  const int D4 = kO ? p.D >> 2 : 1;
  const bool direct = kO && p.NS == 1;
  for (int i = tid; i < nrows * D4; i += 32 * kRowsWarps) {
    const int r = i / D4, c = i - r * D4;
    float M = sm_m[0][r];
#pragma unroll
    for (int w = 1; w < kRowsWarps; ++w) M = fmaxf(M, sm_m[w][r]);
    const float base = M == -INFINITY ? 0.f : M;
    float lt = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) {
      const float f = fast_exp2(sm_m[w][r] - base);
      lt += f * sm_l[w][r];
      if constexpr (kO) {
        const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<float*>(smem) +
                                                          (w * R + r) * kOP + c * 4);
        acc.x += f * x.x;
        acc.y += f * x.y;
        acc.z += f * x.z;
        acc.w += f * x.w;
      }
    }
    if (lt != lt) M = 0.f;  // NaN scores, perhaps none else: -inf means nothing seen
    int b, hd, tk;
    cache_row(p, sg, e, h, r0 + r, b, hd, tk);
    const long long row = ((long long)b * p.Hq + hd) * p.Sq + tk;
    if (direct) {
      const float inv = lt > 0.f ? 1.f / lt : 0.f;
      const uint2 x = make_uint2(DType<DT>::pack2(acc.x * inv, acc.y * inv),
                                 DType<DT>::pack2(acc.z * inv, acc.w * inv));
      *reinterpret_cast<uint2*>(p.out + b * p.os_b + hd * p.os_h + tk * p.os_s + c * 4) =
          M == -INFINITY ? make_uint2(0, 0) : x;
      if (c == 0 && p.lse)
        p.lse[row] = M == -INFINITY ? M : (M + log2f(lt)) * 0.69314718055994531f;
    } else {
      const long long at = row * p.NS + sg.slot0 + sp;
      if (kO && M != -INFINITY) *reinterpret_cast<float4*>(p.opart + at * p.D + c * 4) = acc;
      if (c == 0) p.ml[at] = make_float2(M, lt);
    }
  }
}

// ---------------------------------------------------------------------------
// Joins the partial results of a row: WPR warps per row, each with every
// WPR-th slot, a lane per 4 dims.  Bound by latency, so a warp asks for its
// first eight slots before it knows their weights.  Slots without a visible
// key have m = -inf; what lies there is not used.
// ---------------------------------------------------------------------------
template <typename DT, int WPR>
__global__ void __launch_bounds__(WPR > 4 ? 32 * WPR : 128)
    cache_combine_kernel(const __grid_constant__ CacheParams p, long long nrows) {
  constexpr int kWarps = WPR > 4 ? WPR : 4, kBatch = 8;
  __shared__ float4 part[kWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = warp % WPR;
  const long long row = (long long)blockIdx.x * (kWarps / WPR) + warp / WPR;
  pdl_wait();
  const bool live = row < nrows;
  const bool act = lane * 4 < p.D;
  float M = -INFINITY, lt = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
    const float2* ml = p.ml + row * p.NS;
    const float* op = p.opart + row * p.NS * p.D + lane * 4;
    float4 v[kBatch];
    float2 x[kBatch];
    auto fetch = [&](int s0) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int s = s0 + i * WPR;
        x[i] = s < p.NS ? ml[s] : make_float2(-INFINITY, 0.f);
        if (s < p.NS && act) v[i] = *reinterpret_cast<const float4*>(op + (long long)s * p.D);
      }
    };
    fetch(sub);
    for (int i = lane; i < p.NS; i += 32) {
      const float2 y = ml[i];
      const float mn = fmaxf(M, y.x);
      if (mn != -INFINITY) lt = lt * fast_exp2(M - mn) + y.y * fast_exp2(y.x - mn);
      M = mn;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, M, o);
      const float l2 = __shfl_xor_sync(0xffffffffu, lt, o);
      const float mn = fmaxf(M, m2);
      if (mn != -INFINITY) lt = lt * fast_exp2(M - mn) + l2 * fast_exp2(m2 - mn);
      M = mn;
    }
    for (int s0 = sub; s0 < p.NS; s0 += kBatch * WPR) {
      if (s0 != sub) fetch(s0);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (x[i].x != -INFINITY) {
          const float f = fast_exp2(x[i].x - M);
          acc.x += f * v[i].x;
          acc.y += f * v[i].y;
          acc.z += f * v[i].z;
          acc.w += f * v[i].w;
        }
      }
    }
  }
  if constexpr (WPR > 1) {
    part[warp][lane] = acc;
    __syncthreads();
    if (sub) return;
#pragma unroll
    for (int w = 1; w < WPR; ++w) {
      const float4 y = part[warp + w][lane];
      acc.x += y.x;
      acc.y += y.y;
      acc.z += y.z;
      acc.w += y.w;
    }
  }
  if (!live) return;
  const float inv = lt > 0.f ? 1.f / lt : 0.f;
  const int tk = (int)(row % p.Sq);
  const long long bh = row / p.Sq;
  const int hd = (int)(bh % p.Hq);
  const long long b = bh / p.Hq;
  if (act)
    *reinterpret_cast<uint2*>(p.out + b * p.os_b + hd * p.os_h + tk * p.os_s + lane * 4) =
        M == -INFINITY ? make_uint2(0, 0)
                       : make_uint2(DType<DT>::pack2(acc.x * inv, acc.y * inv),
                                    DType<DT>::pack2(acc.z * inv, acc.w * inv));
  if (lane == 0 && p.lse)
    p.lse[row] = M == -INFINITY ? M : (M + log2f(lt)) * 0.69314718055994531f;
}

// ---------------------------------------------------------------------------
// Host: the split, checks and launches
// ---------------------------------------------------------------------------
struct CachePlan {
  // rows of a sequence walk prefix and own cache in one tile (segment 1's
  // fields below; ranges cover both)
  bool joint;
  bool tile[2];            // segment by cache_tiles_kernel, otherwise by cache_rows_kernel
  int rtiles[2], nsplit[2];
  int chunk[2];            // keys per range
  int NS;
};

// cache_rows_kernel: keys per range.  Four items run on each of the 148 SMs.
// An item costs its keys plus `extra` keys (set-up, first loads, the partial
// result: about 1 us at 27 keys a microsecond and block).  Items of several
// rounds start as others end, so they fill the device but for a third of an
// item at the end; those of a single round all wait for the slowest (15 %
// behind).  The join costs 4 us.  Measured: two 65536-key caches of 32 heads
// 218 us at 1024 keys a range, 215 at 512, 216 at 256, 255 in one round.
constexpr int64_t kRowsSlots = 4 * 148, kRowsUnit = 32;
static int64_t rows_chunk(const int64_t (&tiles)[2], const int64_t (&cap)[2], double* out_cost) {
  constexpr int64_t extra = 32;
  const double total = (double)tiles[0] * cap[0] + (double)tiles[1] * cap[1];
  int64_t best = kRowsUnit;
  double best_cost = 1e300;
  for (int64_t rounds = 1; rounds <= 16; rounds += rounds < 4 ? 1 : 4) {
    // the shortest ranges that fit this many rounds
    const int64_t slots = rounds * kRowsSlots;
    int64_t ch = ((int64_t)(total / slots) / kRowsUnit + 1) * kRowsUnit, items = 0;
    for (;; ch += (ch / 16 / kRowsUnit + 1) * kRowsUnit) {
      items = tiles[0] * ((cap[0] + ch - 1) / ch) + tiles[1] * ((cap[1] + ch - 1) / ch);
      if (items <= slots || (ch >= cap[0] && ch >= cap[1])) break;
    }
    const double fill = (double)items / kRowsSlots;
    double cost = (fill <= 1 ? 1.15 : fill + 0.3) * (ch + extra);
    if (ch < cap[0] || ch < cap[1]) cost += 110;
    if (cost < best_cost) best_cost = cost, best = ch;
  }
  *out_cost = best_cost;
  return best;
}

// Up to kRowsMost rows go past warp-level tiles, more than kRowsPast to 128-row
// tcgen05 tiles; between, one or several 8-row tiles win while there are few
// keys (they need no second kernel and little set-up), the tcgen05 tile
// otherwise, and the costs of both plans decide.  Measured (us, 8-row tiles
// against tcgen05): 16 rows of 8 heads over a prefix of 256, 1024 and 4096 keys 7.4,
// 11.6, 14.6 against 13.8, 14.9, 16.9; four own caches of 4096 keys 23.4 against 18.9;
// 16384 keys of 32 heads 63 against 44.
constexpr int64_t kRowsMost = 8, kRowsPast = 32;
constexpr double kRowsKeysPerUs = 27.0 * 96;  // times the head dim; a block of cache_rows_kernel
constexpr double kSecondKernelUs = 3;

// cache_tiles_kernel: key blocks per range, for tiles of up to two kinds.  Two
// items run on each of the 148 SMs; an item costs its blocks plus kItemCost
// (set-up, first loads, epilogue), and a partial result to be joined kJoinCost
// more, in units of a 64-key block (1 us).
static int64_t tile_blocks(const int64_t (&tiles)[2], const int64_t (&blocks)[2],
                           double* out_cost = nullptr) {
  constexpr double kItemCost = 5, kJoinCost = 4;
  const int64_t slots = 2 * 148;
  const int64_t most = blocks[0] > blocks[1] ? blocks[0] : blocks[1];
  const double total = (double)tiles[0] * blocks[0] + (double)tiles[1] * blocks[1];
  int64_t best = most;
  double best_cost = 1e300;
  for (int64_t rounds = 0; rounds <= 6; ++rounds) {
    int64_t per = most, items = 0;
    if (rounds) per = (int64_t)(total / (rounds * slots)) + 1;
    for (;; per += per / 32 + 1) {  // about the shortest ranges that fit these rounds
      items = tiles[0] * ((blocks[0] + per - 1) / per) + tiles[1] * ((blocks[1] + per - 1) / per);
      if (!rounds || items <= rounds * slots || per >= most) break;
    }
    const int64_t waves = (items + slots - 1) / slots;
    const double cost = (double)waves * (per + kItemCost + (per < most ? kJoinCost : 0));
    if (cost < best_cost) best_cost = cost, best = per < most ? per : most;
  }
  if (out_cost) *out_cost = best_cost;
  return best < 1 ? 1 : best;
}

// The plan with each segment by the kernel that `tile` names, and its cost in us.
static CachePlan cache_plan_of(const bool (&tile)[2], const bool (&use)[2],
                               const int64_t (&rows)[2], const int64_t (&cap)[2],
                               const int64_t (&nb)[2], int64_t Hkv, int64_t D, double* cost) {
  CachePlan pl{};
  int64_t few[2] = {0, 0}, few_cap[2] = {0, 0};   // tiles and keys by cache_rows_kernel
  int64_t many[2] = {0, 0}, blocks[2] = {0, 0};   // tiles and key blocks by cache_tiles_kernel
  for (int s = 0; s < 2; ++s) {
    if (!use[s]) continue;
    pl.tile[s] = tile[s];
    const int per = tile[s] ? 128 : 8;
    pl.rtiles[s] = (int)((rows[s] + per - 1) / per);
    if (tile[s]) many[s] = nb[s] * Hkv * pl.rtiles[s], blocks[s] = (cap[s] + 63) / 64;
    else few[s] = nb[s] * Hkv * pl.rtiles[s], few_cap[s] = cap[s];
  }
  double few_cost = 0, many_cost = 0;
  const bool any_few = few[0] || few[1], any_many = many[0] || many[1];
  const int64_t chunk = any_few ? rows_chunk(few, few_cap, &few_cost) : 0;
  const int64_t tile_chunk = any_many ? tile_blocks(many, blocks, &many_cost) * 64 : 0;
  for (int s = 0; s < 2; ++s) {
    if (!use[s]) continue;
    const int64_t ch = tile[s] ? tile_chunk : chunk;
    pl.chunk[s] = (int)ch;
    // at least one range: with no key at all it writes the zeros
    pl.nsplit[s] = cap[s] ? (int)((cap[s] + ch - 1) / ch) : 1;
  }
  pl.NS = pl.nsplit[0] + pl.nsplit[1];
  *cost = few_cost * D / kRowsKeysPerUs + many_cost + (any_few && any_many ? kSecondKernelUs : 0);
  return pl;
}

static CachePlan cache_plan(int64_t B, int64_t Hkv, int64_t group, int64_t Sq, int64_t G,
                            int64_t P, int64_t C, int64_t D) {
  const bool use[2] = {P > 0, C > 0 || P == 0};
  const int64_t rows[2] = {use[0] ? B / G * group * Sq : 0, use[1] ? group * Sq : 0};
  const int64_t cap[2] = {P, C}, nb[2] = {G, B};
  bool tile[2];
  for (int s = 0; s < 2; ++s) tile[s] = cap[s] > 0 && rows[s] > kRowsMost;
  // One walk over prefix and own keys where a sequence's rows fill tiles about
  // as well as all sequences' rows together do.
  const int64_t own_tiles = B * ((rows[1] + 127) / 128);
  const int64_t all_tiles = G * ((rows[0] + 127) / 128);
  if (tile[0] && tile[1] && rows[1] > kRowsPast && own_tiles * 4 <= all_tiles * 5) {
    CachePlan pl{};
    pl.joint = pl.tile[1] = true;
    pl.rtiles[1] = (int)((rows[1] + 127) / 128);
    const int64_t blocks = (P + 63) / 64 + (C + 63) / 64;
    pl.chunk[1] = (int)tile_blocks({0, B * Hkv * pl.rtiles[1]}, {0, blocks}) * 64;
    pl.nsplit[1] = (int)((blocks * 64 + pl.chunk[1] - 1) / pl.chunk[1]);
    pl.NS = pl.nsplit[1];
    return pl;
  }
  double best_cost, cost;
  CachePlan best = cache_plan_of(tile, use, rows, cap, nb, Hkv, D, &best_cost);
  const bool open[2] = {tile[0] && rows[0] <= kRowsPast, tile[1] && rows[1] <= kRowsPast};
  for (int c = 1; c < 4; ++c) {  // with the segments of few rows that are open the other way
    if (((c & 1) && !open[0]) || ((c & 2) && !open[1])) continue;
    const bool other[2] = {tile[0] && !(c & 1), tile[1] && !(c & 2)};
    const CachePlan pl = cache_plan_of(other, use, rows, cap, nb, Hkv, D, &cost);
    if (cost < best_cost) best_cost = cost, best = pl;
  }
  return best;
}

static bool cache_sizes_ok(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t G, int64_t P,
                           int64_t C, int64_t D) {
  if (B < 0 || Hq < 0 || Hkv < 1 || Sq < 0 || G < 1 || P < 0 || C < 0) return false;
  if (D < 32 || D > 128 || D % 8) return false;
  if (P > (1 << 30) || C > (1 << 30) || P + C > (1 << 30)) return false;
  if (Hq % Hkv || B % G) return false;
  // rows are counted in 32 bits
  const int64_t lim = 1ll << 30;
  return B <= lim && Hq <= lim && Sq <= lim && B * Hq <= lim && B * Hq * Sq <= lim;
}

// Rows that 16-byte loads and tensor maps can read; the strides of dimensions
// of one entry are not looked at.
static bool rows_ok(const mi_rows& t, int64_t n0, int64_t n1, int64_t n2) {
  if (!t.ptr || (reinterpret_cast<uintptr_t>(t.ptr) & 15)) return false;
  const int64_t n[3] = {n0, n1, n2}, s[3] = {t.stride_b, t.stride_h, t.stride_s};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (s[i] <= 0 || s[i] % 8)) return false;
  return true;
}

template <typename DT, int DK, RowsMode MODE>
static int launch_rows(const CacheParams& p, long long items, cudaStream_t stream) {
  using L = RowsSmem<DK, MODE>;
  constexpr int kRowsWarps = L::W;
  constexpr auto kern = cache_rows_kernel<DT, DK, MODE>;
  constexpr int kJoin = MODE == kAttention ? kRowsWarps * 8 * (DK + 4) * 4 : 0;
  constexpr int bytes = L::kRing > kJoin ? L::kRing : kJoin;
  cudaError_t err = allow_smem<cache_rows_kernel<DT, DK, MODE>>(bytes);
  if (err == cudaSuccess) {
    kern<<<(unsigned)items, 32 * kRowsWarps, bytes, stream>>>(p);
    err = cudaGetLastError();
  }
  if (err != cudaSuccess) {
    debug_launch_failure("cache_rows_kernel", reinterpret_cast<const void*>(kern), err,
                         32 * kRowsWarps, bytes);
    return MI_ERR_LAUNCH;
  }
  return MI_OK;
}

template <RowsMode MODE>
static int launch_rows_dk(const CacheParams& p, int dtype, long long items, cudaStream_t st) {
  const bool bf = dtype == MI_BF16;
  if (p.D <= 64)
    return bf ? launch_rows<__nv_bfloat16, 64, MODE>(p, items, st)
              : launch_rows<__half, 64, MODE>(p, items, st);
  if (p.D <= 96)
    return bf ? launch_rows<__nv_bfloat16, 96, MODE>(p, items, st)
              : launch_rows<__half, 96, MODE>(p, items, st);
  return bf ? launch_rows<__nv_bfloat16, 128, MODE>(p, items, st)
            : launch_rows<__half, 128, MODE>(p, items, st);
}

static void set_seg(CacheSeg& s, const mi_rows& k, const mi_rows& v, const int32_t* len,
                    int64_t cap, int64_t nb, int64_t seqs, int64_t rows, int causal) {
  s.k = static_cast<const uint16_t*>(k.ptr);
  s.v = static_cast<const uint16_t*>(v.ptr);
  s.ks_b = nb > 1 ? k.stride_b : 0;
  s.ks_h = k.stride_h;
  s.ks_s = k.stride_s;
  s.vs_b = nb > 1 ? v.stride_b : 0;
  s.vs_h = v.stride_h;
  s.vs_s = v.stride_s;
  s.len = len;
  s.cap = (int)cap;
  s.nb = (int)nb;
  s.seqs = (int)seqs;
  s.rows = (int)rows;
  s.causal = causal;
}

static void set_heads(CacheParams& p, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t D) {
  p.Hq = (int)Hq;
  p.Hkv = (int)Hkv;
  p.group = (int)(Hq / Hkv);
  p.Sq = (int)Sq;
  p.D = (int)D;
  p.div_hkv = FastDiv(Hkv);
  p.div_sq = FastDiv(Sq);
  p.div_rows = FastDiv(Hq / Hkv * Sq);
}

}  // namespace mib200

using namespace mib200;

namespace mib200 {
// Workspace of a call with plan `pl`; SIZE_MAX past any memory.
static size_t shared_prefix_need(const mi_shared_prefix_args& a, const CachePlan& pl) {
  if (pl.NS == 1) return 0;
  if ((double)a.B * a.Hq * a.S_q * pl.NS * (a.D * 4 + 8) > 1e15) return SIZE_MAX;
  const size_t slots = (size_t)(a.B * a.Hq * a.S_q) * pl.NS;
  return align_up(slots * a.D * 4) + align_up(slots * 8);
}
}  // namespace mib200

extern "C" size_t mi_shared_prefix_fwd_workspace_size(const mi_shared_prefix_args* a) {
  if (!a || !cache_sizes_ok(a->B, a->Hq, a->Hkv, a->S_q, a->G, a->P, a->C, a->D)) return SIZE_MAX;
  if (a->B == 0 || a->Hq == 0 || a->S_q == 0) return 0;
  return shared_prefix_need(
      *a, cache_plan(a->B, a->Hkv, a->Hq / a->Hkv, a->S_q, a->G, a->P, a->C, a->D));
}

extern "C" int mi_shared_prefix_fwd(const mi_shared_prefix_args* args, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  if (!args) return MI_ERR_SHAPE;
  const mi_shared_prefix_args& a = *args;
  const int64_t B = a.B, Hq = a.Hq, Hkv = a.Hkv, S_q = a.S_q, G = a.G, P = a.P, C = a.C, D = a.D;
  if (a.dtype != MI_F16 && a.dtype != MI_BF16) return MI_ERR_DTYPE;
  if (!cache_sizes_ok(B, Hq, Hkv, S_q, G, P, C, D)) return MI_ERR_SHAPE;
  if (B == 0 || Hq == 0 || S_q == 0) return MI_OK;
  if (!rows_ok(a.q, B, Hq, S_q) || !rows_ok(a.out, B, Hq, S_q)) return MI_ERR_ALIGN;
  if (P && (!rows_ok(a.k_prefix, G, Hkv, P) || !rows_ok(a.v_prefix, G, Hkv, P)))
    return MI_ERR_ALIGN;
  if (C && (!rows_ok(a.k, B, Hkv, C) || !rows_ok(a.v, B, Hkv, C))) return MI_ERR_ALIGN;
  const int64_t group = Hq / Hkv;
  const CachePlan pl = cache_plan(B, Hkv, group, S_q, G, P, C, D);
  const size_t need = shared_prefix_need(a, pl);
  if (need == SIZE_MAX) return MI_ERR_SHAPE;
  if (need && (!workspace || workspace_bytes < need ||
               (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return MI_ERR_WORKSPACE;

  CacheParams p{};
  p.q = static_cast<const uint16_t*>(a.q.ptr);
  p.qs_b = a.q.stride_b;
  p.qs_h = a.q.stride_h;
  p.qs_s = a.q.stride_s;
  p.out = static_cast<uint16_t*>(a.out.ptr);
  p.os_b = a.out.stride_b;
  p.os_h = a.out.stride_h;
  p.os_s = a.out.stride_s;
  p.lse = a.lse;
  set_heads(p, Hq, Hkv, S_q, D);
  p.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  set_seg(p.seg[0], a.k_prefix, a.v_prefix, a.prefix_lengths, P, G, B / G, B / G * group * S_q, 0);
  set_seg(p.seg[1], a.k, a.v, a.lengths, C, B, 1, group * S_q, a.causal ? 1 : 0);
  for (int s = 0; s < 2; ++s) {
    p.seg[s].rtiles = FastDiv(pl.rtiles[s]);
    p.seg[s].nsplit = FastDiv(pl.nsplit[s]);
    p.seg[s].chunk = pl.chunk[s];
  }
  p.seg[1].slot0 = pl.nsplit[0];
  p.NS = pl.NS;
  const int64_t slots = B * Hq * S_q * pl.NS;
  p.opart = static_cast<float*>(workspace);
  if (need)
    p.ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) +
                                     align_up((size_t)slots * D * 4));
  const long long items[2] = {(long long)G * Hkv * pl.rtiles[0] * pl.nsplit[0],
                              (long long)B * Hkv * pl.rtiles[1] * pl.nsplit[1]};
  if (items[0] + items[1] > 0x7fffffffll) return MI_ERR_SHAPE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = a.dtype == MI_BF16;
  TileParams tp{};
  for (int s = 0; s < 2; ++s) {
    if (!pl.tile[s]) continue;
    TileGroup& g = tp.grp[s];
    g.rows_of = s;
    g.use0 = s == 0 || pl.joint;
    g.use1 = s == 1;
    g.rtiles = FastDiv(pl.rtiles[s]);
    g.nsplit = FastDiv(pl.nsplit[s]);
    g.blocks = pl.chunk[s] / 64;
    g.slot0 = p.seg[s].slot0;
    g.items = (int)items[s];
  }
  // The own caches' kernel first: the prefix's tiles start as its blocks end
  // (the other way round the last tiles end alone: 35 us against 32 for 32
  // sequences of 512 keys over 8192).
  const long long few = (pl.tile[0] ? 0 : items[0]) + (pl.tile[1] ? 0 : items[1]);
  if (few) {
    p.items0 = pl.tile[0] ? 0 : (int)items[0];
    const int rc = launch_rows_dk<kAttention>(p, a.dtype, few, st);
    if (rc != MI_OK) return rc;
  }
  if (pl.tile[0] || pl.tile[1]) {
    tp.c = p;
    const int rc =
        launch_tiles(tp, a.dtype, a.k_prefix, a.v_prefix, a.k, a.v, few > 0, st);
    if (rc != MI_OK) return rc;
  }
  if (p.NS == 1) return MI_OK;
  const long long nrows = B * Hq * S_q;
  // a warp joins up to eight slots at once; many rows need fewer warps each
  const int wpr = p.NS <= 8 || nrows >= 16384 ? 1 : (p.NS <= 32 || nrows >= 4096 ? 4 : 8);
  const dim3 grid((unsigned)(wpr == 1 ? (nrows + 3) / 4 : nrows));
#define MI_JOIN(W)                                                                            \
  (bf ? launch_after(cache_combine_kernel<__nv_bfloat16, W>, grid, W > 4 ? 32 * W : 128, 0,   \
                     st, p, nrows)                                                            \
      : launch_after(cache_combine_kernel<__half, W>, grid, W > 4 ? 32 * W : 128, 0, st, p, nrows))
  const cudaError_t err = wpr == 1 ? MI_JOIN(1) : (wpr == 4 ? MI_JOIN(4) : MI_JOIN(8));
#undef MI_JOIN
  return err == cudaSuccess ? MI_OK : MI_ERR_LAUNCH;
}
