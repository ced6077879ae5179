// Eviction from a KV cache by accumulated weight: per (sequence, head) the
// rows to keep are chosen (forced first and last rows, then the greatest
// weights, ties to the lower index) and moved, in order, to new buffers.
#include <cooperative_groups.h>

#include "cache_attn.cuh"
#include "host_util.h"

namespace mib200 {

struct EvictParams {
  const float* w;
  long long w_b, w_h;
  const int32_t* len;
  int H, C, D, keep, sink, recent;
  FastDiv div_h, div_row;  // by H; by the pieces of a row
  int32_t* index;          // [B, H, keep]
  int32_t* new_len;        // [B]
  const uint16_t *k, *v;
  long long ks_b, ks_h, ks_s, vs_b, vs_h, vs_s;
  uint16_t *ko, *vo;
  long long ko_b, ko_h, ko_s, vo_b, vo_h, vo_s;
  float* wo;
  long long wo_b, wo_h;
};

// Selection key: forced rows above everything, NaN below everything, -0 = +0.
__device__ __forceinline__ uint32_t evict_key(float w, int j, int n, int sink, int recent) {
  if (j < sink || j >= n - recent) return 0xffffffffu;
  return w != w ? 0u : float_to_ordered(w + 0.0f);
}

// One cluster of CL blocks per (b, h) selects and moves.
//
// Selection: the k-th largest key by a radix search over 11, 11 and 10 bits.
// A warp owns a contiguous segment of the keys, in rounds of 32; with KPT > 0
// they stay in its registers (KPT rounds), so the weights are read once,
// otherwise (more keys than the cluster's registers hold) they are read again
// in every pass.  A pass counts digits in shared memory; through distributed
// shared memory one warp of each block then adds up the cluster's sums of 32
// digits, finds the group, adds up that group's digits, and all blocks find the
// same digit (3 KB read a block and pass; adding up all 2048 counts took 3 us a
// pass).  With T the k-th key and e of the keys equal to it to be kept, a kept
// key's place is the number of keys above T before it plus the smaller of e and
// the number of keys equal to T before it.  Bound by the barriers' latency.
//
// Move: the kept rows are shared out evenly over the cluster, whichever block
// found them, in 16-byte pieces (V; single elements for rows without that
// alignment); bound by their bytes.
//
// Measured: 32 heads of 65536 rows of 96 to 8192: 52 us, of which the search 19;
// 256 heads of up to 4097 rows of 128 to 2048: 93 us (5.7 TB/s).  As a search
// kernel over a cluster and a move kernel they took 81 and 107.
constexpr int kEvictThreads = 512;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kMoveRows = 512;
constexpr int kEvictCopies = 4;
// Four copies of a pass's counts, by lane: weights share exponents, and equal
// digits within a warp add one after the other.  A pass leaves its sums in one
// of two buffers: a block writes a buffer again only after the barrier of the
// pass between, by which every block has read it.
struct EvictSmem {
  int copies[kEvictCopies * 2048];
  int fine[2][2048];
  int coarse[2][64];  // sums of 32 places
};

template <int CL, int KPT, typename V>
__global__ void __launch_bounds__(kEvictThreads, 2)
    evict_kernel(const __grid_constant__ EvictParams p) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint8_t evict_smem[];
  EvictSmem& sm = *reinterpret_cast<EvictSmem*>(evict_smem);
  __shared__ int cnt_gt[kEvictWarps], cnt_eq[kEvictWarps];
  __shared__ int cta_gt, cta_eq, sel_digit, sel_left;
  __shared__ int src[kMoveRows];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned lt = (1u << lane) - 1u;
  int rank = 0;
  if constexpr (CL > 1) rank = (int)cg::this_cluster().block_rank();
  auto cluster_sync = [&]() {
    if constexpr (CL > 1) cg::this_cluster().sync();
    else __syncthreads();
  };
  // the same shared variable of block r of the cluster
  auto peer = [&](auto* x, int r) {
    if constexpr (CL > 1) return cg::this_cluster().map_shared_rank(x, r);
    else return x;
  };
  const int bh = blockIdx.x / CL;
  int h;
  const int b = p.div_h.divmod(bh, h);
  const int n = p.len ? min(max(p.len[b], 0), p.C) : p.C;
  const int keep = min(n, p.keep);
  const float* w = p.w + b * p.w_b + h * p.w_h;
  int32_t* index = p.index + (long long)bh * p.keep;
  if (h == 0 && rank == 0 && tid == 0) p.new_len[b] = keep;

  if (n > p.keep) {
    // ---- select (uniform over the cluster) ------------------------------------
    const int cseg = (((n + CL - 1) / CL) + 31) & ~31;
    const int cbeg = min(n, rank * cseg), cend = min(n, cbeg + cseg);
    const int seg = (((cend - cbeg + kEvictWarps - 1) / kEvictWarps) + 31) & ~31;
    const int wbeg = min(cend, cbeg + warp * seg), wend = min(cend, wbeg + seg);
    constexpr int kRegs = KPT > 0 ? KPT : 1;
    uint32_t key[kRegs];
    if constexpr (KPT > 0) {
      float x[KPT];
#pragma unroll
      for (int u = 0; u < KPT; ++u) {
        const int i = wbeg + u * 32 + lane;
        x[u] = i < wend ? w[i] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < KPT; ++u)
        key[u] = evict_key(x[u], wbeg + u * 32 + lane, n, p.sink, p.recent);
    }
    // f(i, key, valid) for every round of 32 keys of the warp, in order
    auto walk = [&](auto&& f) {
      if constexpr (KPT > 0) {
#pragma unroll
        for (int u = 0; u < KPT; ++u) {
          const int i = wbeg + u * 32 + lane;
          if (wbeg + u * 32 < wend) f(i, key[u], i < wend);
        }
      } else {
        for (int base = wbeg; base < wend; base += 32) {
          const int i = base + lane;
          f(i, i < wend ? evict_key(w[i], i, n, p.sink, p.recent) : 0u, i < wend);
        }
      }
    };
    for (int i = tid; i < kEvictCopies * 2048; i += kEvictThreads) sm.copies[i] = 0;
    __syncthreads();
    uint32_t prefix = 0, pmask = 0;
    int left = keep;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
      const int bins = pass == 2 ? 1024 : 2048;
      // digits run from the top down: digit bins-1 counts in place 0
      walk([&](int, uint32_t kk, bool valid) {
        if (valid && (kk & pmask) == prefix)
          atomicAdd(&sm.copies[(lane % kEvictCopies) * 2048 + bins - 1 -
                               ((kk >> shift) & (bins - 1))], 1);
      });
      __syncthreads();
      // four places per thread, then groups of 32 places; clear for the next pass
      int* fine = sm.fine[pass & 1];
      int* coarse = sm.coarse[pass & 1];
      if (4 * tid < bins) {
        int4 x = make_int4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < kEvictCopies; ++c) {
          int4* cp = reinterpret_cast<int4*>(&sm.copies[c * 2048 + 4 * tid]);
          const int4 y = *cp;
          x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
          *cp = make_int4(0, 0, 0, 0);
        }
        *reinterpret_cast<int4*>(&fine[4 * tid]) = x;
        int sum = x.x + x.y + x.z + x.w;
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        if ((tid & 7) == 0) coarse[tid >> 3] = sum;
      }
      cluster_sync();
      if (warp == 0) {
        // the group (two per lane), then the place in it, of the left-th key
        const int groups = bins / 32;
        int c0 = 0, c1 = 0;
        if (2 * lane < groups) {
          int2 x[CL];  // asked for together: each is a round trip to another SM
#pragma unroll
          for (int r = 0; r < CL; ++r)
            x[r] = *reinterpret_cast<const int2*>(peer(&coarse[2 * lane], r));
#pragma unroll
          for (int r = 0; r < CL; ++r) c0 += x[r].x, c1 += x[r].y;
        }
        int incl = c0 + c1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        int first = __ffs(__ballot_sync(0xffffffffu, incl >= left)) - 1;
        const int g0 = __shfl_sync(0xffffffffu, c0, first);
        int before = __shfl_sync(0xffffffffu, incl - c0 - c1, first);
        int group = 2 * first;
        if (before + g0 < left) before += g0, ++group;
        int x[CL], c = 0;
#pragma unroll
        for (int r = 0; r < CL; ++r) x[r] = *peer(&fine[group * 32 + lane], r);
#pragma unroll
        for (int r = 0; r < CL; ++r) c += x[r];
        incl = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        first = __ffs(__ballot_sync(0xffffffffu, before + incl >= left)) - 1;
        if (lane == first) {
          sel_digit = bins - 1 - (group * 32 + lane);
          sel_left = left - (before + incl - c);
        }
      }
      __syncthreads();
      prefix |= (uint32_t)sel_digit << shift;
      pmask |= (uint32_t)(bins - 1) << shift;
      left = sel_left;
    }
    int gt = 0, eq = 0;
    walk([&](int, uint32_t kk, bool valid) {
      gt += valid && kk > prefix;
      eq += valid && kk == prefix;
    });
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) cnt_gt[warp] = gt, cnt_eq[warp] = eq;
    __syncthreads();
    gt = eq = 0;
    int bgt = 0, beq = 0;
    for (int x = 0; x < kEvictWarps; ++x) {
      if (x == warp) gt = bgt, eq = beq;
      bgt += cnt_gt[x], beq += cnt_eq[x];
    }
    if (tid == 0) cta_gt = bgt, cta_eq = beq;
    if constexpr (CL > 1) {
      cluster_sync();
#pragma unroll
      for (int r = 0; r < CL - 1; ++r) {
        const int g = *peer(&cta_gt, r);
        const int q = *peer(&cta_eq, r);
        if (r < rank) gt += g, eq += q;
      }
    }
    walk([&](int i, uint32_t kk, bool valid) {
      const bool g = valid && kk > prefix, q = valid && kk == prefix;
      const unsigned gb = __ballot_sync(0xffffffffu, g), qb = __ballot_sync(0xffffffffu, q);
      const int ng = gt + __popc(gb & lt), nq = eq + __popc(qb & lt);
      if (g || (q && nq < left)) index[ng + min(nq, left)] = i;
      gt += __popc(gb);
      eq += __popc(qb);
    });
    cluster_sync();  // the index is written; no block reads another's counts any more
  }

  // ---- move ---------------------------------------------------------------------
  constexpr int E = sizeof(V) / 2;
  const int per_cta = (p.keep + CL - 1) / CL;
  const int m0 = min(p.keep, rank * per_cta), m1 = min(p.keep, m0 + per_cta);
  const int pieces = p.D / E;
  const uint16_t* kb = p.k + b * p.ks_b + h * p.ks_h;
  const uint16_t* vb = p.v + b * p.vs_b + h * p.vs_h;
  uint16_t* ko = p.ko + b * p.ko_b + h * p.ko_h;
  uint16_t* vo = p.vo + b * p.vo_b + h * p.vo_h;
  float* wo = p.wo + b * p.wo_b + h * p.wo_h;
  for (int i0 = m0; i0 < m1; i0 += kMoveRows) {
    const int rows = min(kMoveRows, m1 - i0);
    __syncthreads();
    if (tid < rows) {
      const int i = i0 + tid;
      int j = -1;
      if (i < keep) j = n > p.keep ? __ldcg(index + i) : i;  // another block wrote it
      src[tid] = j;
      wo[i] = j >= 0 ? w[j] : 0.f;
      if (i >= keep || n <= p.keep) index[i] = j;
    }
    __syncthreads();
    constexpr int kBatch = 4;
    for (int t0 = tid; t0 < rows * pieces; t0 += kBatch * kEvictThreads) {
      V x[kBatch], y[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int t = t0 + u * kEvictThreads;
        x[u] = y[u] = V{};
        if (t < rows * pieces) {
          int c;
          const long long j = src[p.div_row.divmod(t, c)];
          if (j >= 0) {
            x[u] = *reinterpret_cast<const V*>(kb + j * p.ks_s + c * E);
            y[u] = *reinterpret_cast<const V*>(vb + j * p.vs_s + c * E);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int t = t0 + u * kEvictThreads;
        if (t < rows * pieces) {
          int c;
          const long long d = i0 + p.div_row.divmod(t, c);
          *reinterpret_cast<V*>(ko + d * p.ko_s + c * E) = x[u];
          *reinterpret_cast<V*>(vo + d * p.vo_s + c * E) = y[u];
        }
      }
    }
  }
}

static bool evict_sizes_ok(int64_t B, int64_t H, int64_t C, int64_t D, int64_t keep) {
  return B >= 0 && H >= 0 && C >= 0 && D >= 1 && D <= 1024 && keep >= 1 && C <= (1 << 30) &&
         keep <= (1 << 30) && B <= (1 << 27) && H <= (1 << 27) && B * H <= (1 << 27);
}

// Blocks per (b, h): enough to fill the device twice, but no segment under 1024
// keys, below which the cluster's barriers cost more than the keys (32 heads of
// 1025 keys: 10.4 us with one block, 10.7 with four; 64 of 3000: 22 us with
// one, 16.4 with two, 17.7 with four).
constexpr int64_t kEvictMin = 1024;
static int evict_cluster(int64_t BH, int64_t C) {
  int cl = 1;
  while (cl < 8 && BH * cl * 2 <= 2 * 148 && C >= cl * 2 * kEvictMin) cl *= 2;
  return cl;
}

template <int CL, int KPT, typename V>
static int launch_evict(const EvictParams& p, int64_t BH, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(BH * CL));
  cfg.blockDim = dim3(kEvictThreads);
  cfg.dynamicSmemBytes = sizeof(EvictSmem);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CL;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CL > 1 ? 1 : 0;
  constexpr auto kern = evict_kernel<CL, KPT, V>;
  cudaError_t err = allow_smem<evict_kernel<CL, KPT, V>>(sizeof(EvictSmem));
  if (err == cudaSuccess) err = cudaLaunchKernelEx(&cfg, kern, p);
  if (err != cudaSuccess) {
    cudaGetLastError();  // reported by the status alone
    debug_launch_failure("evict_kernel", reinterpret_cast<const void*>(kern), err, kEvictThreads,
                         0);
    return MI_ERR_LAUNCH;
  }
  return MI_OK;
}

template <int CL, typename V>
static int launch_evict_keys(const EvictParams& p, int64_t BH, cudaStream_t st) {
  // rounds of 32 keys per warp (each level of the split rounds up to 32)
  const int64_t cseg = ((p.C + CL - 1) / CL + 31) & ~31ll;
  const int64_t rounds = ((cseg + kEvictWarps - 1) / kEvictWarps + 31) / 32;
  if (rounds <= 4) return launch_evict<CL, 4, V>(p, BH, st);
  if (rounds <= 16) return launch_evict<CL, 16, V>(p, BH, st);
  return launch_evict<CL, 0, V>(p, BH, st);
}

template <typename V>
static int launch_evict_cl(const EvictParams& p, int64_t BH, cudaStream_t st) {
  switch (evict_cluster(BH, p.C)) {
    case 1: return launch_evict_keys<1, V>(p, BH, st);
    case 2: return launch_evict_keys<2, V>(p, BH, st);
    case 4: return launch_evict_keys<4, V>(p, BH, st);
    default: return launch_evict_keys<8, V>(p, BH, st);
  }
}

// 16-byte rows: base and the strides of dimensions with more than one entry.
static bool wide_rows(const mi_rows& t, int64_t n0, int64_t n1, int64_t n2) {
  return !(reinterpret_cast<uintptr_t>(t.ptr) & 15) && (n0 <= 1 || t.stride_b % 8 == 0) &&
         (n1 <= 1 || t.stride_h % 8 == 0) && (n2 <= 1 || t.stride_s % 8 == 0);
}

}  // namespace mib200

using namespace mib200;

extern "C" int mi_evict_cache(const mi_evict_args* args, void* stream) {
  if (!args) return MI_ERR_SHAPE;
  const mi_evict_args& a = *args;
  const int64_t B = a.B, H = a.H, C = a.C, D = a.D, keep = a.keep;
  if (!evict_sizes_ok(B, H, C, D, keep)) return MI_ERR_SHAPE;
  if (a.sink < 0 || a.recent < 0 || a.sink > keep || a.recent > keep || a.sink + a.recent > keep)
    return MI_ERR_SHAPE;
  if (B == 0 || H == 0) return MI_OK;
  if (!a.index || !a.new_lengths || !a.weights_out || !a.k_out.ptr || !a.v_out.ptr ||
      (C && (!a.weights || !a.k.ptr || !a.v.ptr)))
    return MI_ERR_SHAPE;
  const bool wide = D % 8 == 0 && wide_rows(a.k, B, H, C) && wide_rows(a.v, B, H, C) &&
                    wide_rows(a.k_out, B, H, keep) && wide_rows(a.v_out, B, H, keep);
  EvictParams p{};
  p.w = a.weights;
  p.w_b = a.weights_stride_b;
  p.w_h = a.weights_stride_h;
  p.len = a.lengths;
  p.H = (int)H;
  p.C = (int)C;
  p.D = (int)D;
  p.keep = (int)keep;
  p.sink = (int)a.sink;
  p.recent = (int)a.recent;
  p.div_h = FastDiv(H);
  p.div_row = FastDiv(wide ? D / 8 : D);
  p.index = a.index;
  p.new_len = a.new_lengths;
  p.k = static_cast<const uint16_t*>(a.k.ptr);
  p.v = static_cast<const uint16_t*>(a.v.ptr);
  p.ks_b = a.k.stride_b, p.ks_h = a.k.stride_h, p.ks_s = a.k.stride_s;
  p.vs_b = a.v.stride_b, p.vs_h = a.v.stride_h, p.vs_s = a.v.stride_s;
  p.ko = static_cast<uint16_t*>(a.k_out.ptr);
  p.vo = static_cast<uint16_t*>(a.v_out.ptr);
  p.ko_b = a.k_out.stride_b, p.ko_h = a.k_out.stride_h, p.ko_s = a.k_out.stride_s;
  p.vo_b = a.v_out.stride_b, p.vo_h = a.v_out.stride_h, p.vo_s = a.v_out.stride_s;
  p.wo = a.weights_out;
  p.wo_b = a.weights_out_stride_b;
  p.wo_h = a.weights_out_stride_h;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return wide ? launch_evict_cl<uint4>(p, B * H, st) : launch_evict_cl<uint16_t>(p, B * H, st);
}
