// Eviction from a KV cache by accumulated weight: per (sequence, head) the
// rows to keep are chosen (forced first and last rows, then the greatest
// weights, ties to the lower index) and moved, in order, to new buffers.
#include <cooperative_groups.h>

#include "host_util.h"
#include "topk.cuh"

namespace mib200 {

struct EvictParams {
  const float* w;
  long long w_b, w_h;
  const int32_t* len;
  int H, C, keep, sink, recent;
  int32_t* index;    // [B, H, keep]
  int32_t* new_len;  // [B]
  uint32_t* keys;    // [B*H][C] when a segment does not fit shared memory, else null
};

// Selection key: forced rows above everything, NaN below everything, -0 = +0.
__device__ __forceinline__ uint32_t evict_key(float w, int j, int n, int sink, int recent) {
  if (j < sink || j >= n - recent) return 0xffffffffu;
  return w != w ? 0u : float_to_ordered(w + 0.0f);
}

constexpr int kEvictThreads = 512;
constexpr int kEvictSegKeys = 40960;  // keys one CTA holds in shared memory (160 KB)

// A cluster of CL CTAs selects for one (b, h); every CTA holds its segment of
// the keys in shared memory, so the weights are read once.
template <int CL>
__global__ void __launch_bounds__(kEvictThreads) evict_select_kernel(EvictParams p) {
  extern __shared__ __align__(16) uint32_t seg[];
  __shared__ TopkSmem<kEvictThreads> sm;
  int rank = 0;
  if constexpr (CL > 1) rank = (int)cooperative_groups::this_cluster().block_rank();
  const long long bh = blockIdx.x / CL;
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  const int n = p.len ? min(max(p.len[b], 0), p.C) : p.C;
  const int keep = min(n, p.keep);
  const float* w = p.w + b * p.w_b + h * p.w_h;
  int32_t* index = p.index + bh * p.keep;
  if (h == 0 && rank == 0 && threadIdx.x == 0) p.new_len[b] = keep;
  for (int i = keep + rank * kEvictThreads + threadIdx.x; i < p.keep; i += CL * kEvictThreads)
    index[i] = -1;
  if (n <= p.keep) {  // everything stays (uniform over the cluster)
    for (int i = rank * kEvictThreads + threadIdx.x; i < n; i += CL * kEvictThreads) index[i] = i;
    return;
  }
  // the segment that cluster_topk gives this CTA
  const int cseg = (((n + CL - 1) / CL) + 31) & ~31;
  const int cbeg = min(n, rank * cseg), cend = min(n, cbeg + cseg);
  uint32_t* keys = p.keys ? p.keys + bh * p.C : seg - cbeg;
  for (int i = cbeg + threadIdx.x; i < cend; i += kEvictThreads)
    keys[i] = evict_key(w[i], i, n, p.sink, p.recent);
  __syncthreads();
  cluster_topk<kEvictThreads, CL>(keys, n, keep, sm, [&](int pos, int i) { index[pos] = i; });
}

struct MoveParams {
  const uint16_t *k, *v;
  long long ks_b, ks_h, ks_s, vs_b, vs_h, vs_s;
  const float* w;
  long long w_b, w_h;
  uint16_t *ko, *vo;
  long long ko_b, ko_h, ko_s, vo_b, vo_h, vo_s;
  float* wo;
  long long wo_b, wo_h;
  const int32_t* index;
  int H, D, keep, tiles;
};

constexpr int kMoveRows = 64;

template <typename V>
__global__ void __launch_bounds__(256) evict_move_kernel(const __grid_constant__ MoveParams p) {
  constexpr int E = sizeof(V) / 2;
  __shared__ int src[kMoveRows];
  const long long bh = blockIdx.x / p.tiles;
  const int i0 = (int)(blockIdx.x % p.tiles) * kMoveRows;
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  const int rows = min(kMoveRows, p.keep - i0);
  if (threadIdx.x < rows) {
    const int j = p.index[bh * p.keep + i0 + threadIdx.x];
    src[threadIdx.x] = j;
    p.wo[b * p.wo_b + h * p.wo_h + i0 + threadIdx.x] =
        j >= 0 ? p.w[b * p.w_b + h * p.w_h + j] : 0.f;
  }
  __syncthreads();
  const int per = p.D / E;
  const uint16_t* kb = p.k + b * p.ks_b + h * p.ks_h;
  const uint16_t* vb = p.v + b * p.vs_b + h * p.vs_h;
  uint16_t* ko = p.ko + b * p.ko_b + h * p.ko_h;
  uint16_t* vo = p.vo + b * p.vo_b + h * p.vo_h;
#pragma unroll 4
  for (int i = threadIdx.x; i < rows * per; i += 256) {
    const int r = i / per, c = (i - r * per) * E;
    const long long j = src[r], d = i0 + r;
    V x{}, y{};
    if (j >= 0) {
      x = *reinterpret_cast<const V*>(kb + j * p.ks_s + c);
      y = *reinterpret_cast<const V*>(vb + j * p.vs_s + c);
    }
    *reinterpret_cast<V*>(ko + d * p.ko_s + c) = x;
    *reinterpret_cast<V*>(vo + d * p.vo_s + c) = y;
  }
}

static bool evict_sizes_ok(int64_t B, int64_t H, int64_t C, int64_t D, int64_t keep) {
  return B >= 0 && H >= 0 && C >= 0 && D >= 1 && D <= 1024 && keep >= 1 && C <= (1 << 30) &&
         keep <= (1 << 30) && B <= (1 << 30) && H <= (1 << 30) && B * H <= (1 << 24);
}

// CTAs per (b, h): enough to fill the device, but no segment under 2048 keys
// (below that the cluster's barriers cost more than the keys), and at least
// what holds the keys in shared memory.
static int evict_cluster(int64_t BH, int64_t C) {
  int cl = 1;
  while (cl < 8 && ((BH * cl * 2 <= 592 && C >= cl * 2 * 2048) || C > (int64_t)cl * kEvictSegKeys))
    cl *= 2;
  return cl;
}

template <int CL>
static int launch_select(const EvictParams& p, int64_t BH, cudaStream_t st) {
  auto kern = evict_select_kernel<CL>;
  const int64_t seg = ((p.C + CL - 1) / CL + 31) & ~31ll;
  const int bytes = p.keys ? 0 : (int)(seg * 4);
  cudaError_t err = allow_smem<evict_select_kernel<CL>>(kEvictSegKeys * 4);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(BH * CL));
  cfg.blockDim = dim3(kEvictThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CL;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (err == cudaSuccess) err = cudaLaunchKernelEx(&cfg, kern, p);
  if (err != cudaSuccess) {
    debug_launch_failure("evict_select_kernel", reinterpret_cast<const void*>(kern), err,
                         kEvictThreads, bytes);
    return MI_ERR_LAUNCH;
  }
  return MI_OK;
}

// 16-byte rows: base and the strides of dimensions with more than one entry.
static bool wide_rows(const mi_rows& t, int64_t n0, int64_t n1, int64_t n2) {
  return !(reinterpret_cast<uintptr_t>(t.ptr) & 15) && (n0 <= 1 || t.stride_b % 8 == 0) &&
         (n1 <= 1 || t.stride_h % 8 == 0) && (n2 <= 1 || t.stride_s % 8 == 0);
}

}  // namespace mib200

using namespace mib200;

extern "C" size_t mi_evict_cache_workspace_size(const mi_evict_args* a) {
  if (!a || !evict_sizes_ok(a->B, a->H, a->C, a->D, a->keep)) return SIZE_MAX;
  return a->C > 8ll * kEvictSegKeys ? align_up((size_t)(a->B * a->H) * a->C * 4) : 0;
}

extern "C" int mi_evict_cache(const mi_evict_args* args, void* workspace, size_t workspace_bytes,
                              void* stream) {
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
  const size_t need = mi_evict_cache_workspace_size(args);
  if (need && (!workspace || workspace_bytes < need ||
               (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return MI_ERR_WORKSPACE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  EvictParams p{};
  p.w = a.weights;
  p.w_b = a.weights_stride_b;
  p.w_h = a.weights_stride_h;
  p.len = a.lengths;
  p.H = (int)H;
  p.C = (int)C;
  p.keep = (int)keep;
  p.sink = (int)a.sink;
  p.recent = (int)a.recent;
  p.index = a.index;
  p.new_len = a.new_lengths;
  p.keys = need ? static_cast<uint32_t*>(workspace) : nullptr;
  const int cl = evict_cluster(B * H, C);
  int rc = cl == 1   ? launch_select<1>(p, B * H, st)
           : cl == 2 ? launch_select<2>(p, B * H, st)
           : cl == 4 ? launch_select<4>(p, B * H, st)
                     : launch_select<8>(p, B * H, st);
  if (rc != MI_OK) return rc;

  MoveParams m{};
  m.k = static_cast<const uint16_t*>(a.k.ptr);
  m.v = static_cast<const uint16_t*>(a.v.ptr);
  m.ks_b = a.k.stride_b, m.ks_h = a.k.stride_h, m.ks_s = a.k.stride_s;
  m.vs_b = a.v.stride_b, m.vs_h = a.v.stride_h, m.vs_s = a.v.stride_s;
  m.w = a.weights;
  m.w_b = a.weights_stride_b, m.w_h = a.weights_stride_h;
  m.ko = static_cast<uint16_t*>(a.k_out.ptr);
  m.vo = static_cast<uint16_t*>(a.v_out.ptr);
  m.ko_b = a.k_out.stride_b, m.ko_h = a.k_out.stride_h, m.ko_s = a.k_out.stride_s;
  m.vo_b = a.v_out.stride_b, m.vo_h = a.v_out.stride_h, m.vo_s = a.v_out.stride_s;
  m.wo = a.weights_out;
  m.wo_b = a.weights_out_stride_b, m.wo_h = a.weights_out_stride_h;
  m.index = a.index;
  m.H = (int)H;
  m.D = (int)D;
  m.keep = (int)keep;
  m.tiles = (int)((keep + kMoveRows - 1) / kMoveRows);
  const long long blocks = (long long)B * H * m.tiles;
  if (blocks > 0x7fffffffll) return MI_ERR_SHAPE;
  const bool wide = D % 8 == 0 && wide_rows(a.k, B, H, C) && wide_rows(a.v, B, H, C) &&
                    wide_rows(a.k_out, B, H, keep) && wide_rows(a.v_out, B, H, keep);
  if (wide) evict_move_kernel<uint4><<<(unsigned)blocks, 256, 0, st>>>(m);
  else evict_move_kernel<uint16_t><<<(unsigned)blocks, 256, 0, st>>>(m);
  return cudaGetLastError() == cudaSuccess ? MI_OK : MI_ERR_LAUNCH;
}
