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
  int tiles;  // key tiles per (b, h)
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

// Few rows: a warp keeps 16 keys (the A operand, so a thread's results belong
// to two keys and the sum over rows stays in its registers) and walks the
// query rows eight at a time.  Bound by the bytes of K.
constexpr int kColsKeys = 64;

template <typename DT, int DK>
__global__ void __launch_bounds__(128) weight_cols_kernel(const __grid_constant__ WeightParams p) {
  constexpr int kPitch = DK * 2 + 16, KS = DK / 16, CPR = DK / 8;
  __shared__ __align__(16) uint8_t sk[kColsKeys * kPitch];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  long long it = blockIdx.x;
  const int tile = (int)(it % p.tiles);
  it /= p.tiles;
  const int h = (int)(it % p.Hkv), b = (int)(it / p.Hkv);
  const int len = p.len ? min(max(p.len[b], 0), p.C) : p.C;
  const int k0 = tile * kColsKeys + warp * 16;
  const float* win = p.win ? p.win + b * p.wi_b + h * p.wi_h : nullptr;
  float* wout = p.wout + b * p.wo_b + h * p.wo_h;
  if (k0 >= p.C) return;
  if (k0 >= len) {  // stale keys: their weights pass through
    const int j = k0 + lane;
    if (lane < 16 && j < p.C && (win != wout)) wout[j] = win ? win[j] : 0.f;
    return;
  }
  const uint16_t* kb = p.k + b * p.ks_b + h * p.ks_h;
  const uint32_t sw = smem_u32(sk) + warp * 16 * kPitch;
  for (int i = lane; i < 16 * CPR; i += 32) {
    const int r = i / CPR, c = i - r * CPR;
    const bool ok = k0 + r < len && c * 8 < p.D;
    cp16(sw + r * kPitch + c * 16, ok ? kb + (long long)(k0 + r) * p.ks_s + c * 8 : kb, ok);
  }
  cp_commit();
  cp_wait<0>();
  __syncwarp();
  uint32_t a[KS][4];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
    ldsm4(a[ks], sw + (lane & 15) * kPitch + ks * 32 + (lane >> 4) * 16);

  const int rows = p.group * p.Sq;
  // First token that sees this warp's first key, and the row limit of a key.
  const int slo = p.causal ? max(0, k0 - len + p.Sq) : 0;
  float tot[2] = {0.f, 0.f};
  for (int rb = 0; rb < rows; rb += 256) {
    float part[2] = {0.f, 0.f};  // two-level sums: 32 steps, then the total
    for (int r0 = rb; r0 < min(rows, rb + 256); r0 += 8) {
      if (r0 / p.Sq == (r0 + 7) / p.Sq && (r0 + 7) % p.Sq < slo) continue;
      const int rq = r0 + (lane >> 2);
      float c[4] = {0.f, 0.f, 0.f, 0.f};
      const int rr = min(rq, rows - 1);
      const uint16_t* qp = p.q + b * p.qs_b + (long long)(h * p.group + rr / p.Sq) * p.qs_h +
                           (long long)(rr % p.Sq) * p.qs_s + (lane & 3) * 2;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint32_t b0 = ks * 16 < p.D ? *reinterpret_cast<const uint32_t*>(qp + ks * 16) : 0u;
        const uint32_t b1 =
            ks * 16 + 8 < p.D ? *reinterpret_cast<const uint32_t*>(qp + ks * 16 + 8) : 0u;
        mma16816<DT>(c, a[ks], b0, b1);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = r0 + (lane & 3) * 2 + x;
        if (r >= rows) continue;
        const int s = r % p.Sq;
        const float z = p.lse[((long long)b * p.Hq + h * p.group + r / p.Sq) * p.Sq + s];
        const float nz = z == -INFINITY ? -INFINITY : -z * p.lse_mul;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int j = k0 + (lane >> 2) + 8 * y;
          const bool vis = j < len && (!p.causal || j < len - (p.Sq - 1 - s));
          if (vis) part[y] += fast_exp2(fmaf(c[2 * y + x], p.scale_log2, nz));
        }
      }
    }
    tot[0] += part[0];
    tot[1] += part[1];
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    tot[y] += __shfl_xor_sync(0xffffffffu, tot[y], 1);
    tot[y] += __shfl_xor_sync(0xffffffffu, tot[y], 2);
    const int j = k0 + (lane >> 2) + 8 * y;
    if ((lane & 3) == 0 && j < p.C) {
      if (j < len) wout[j] = (win ? win[j] : 0.f) + tot[y];
      else if (win != wout) wout[j] = win ? win[j] : 0.f;
    }
  }
}

template <typename DT>
static int launch_cols(const WeightParams& p, cudaStream_t st) {
  const long long items = (long long)p.tiles * p.Hkv * p.B;
  if (items > 0x7fffffffll) return MI_ERR_SHAPE;
  if (p.D <= 64) weight_cols_kernel<DT, 64><<<(unsigned)items, 128, 0, st>>>(p);
  else if (p.D <= 96) weight_cols_kernel<DT, 96><<<(unsigned)items, 128, 0, st>>>(p);
  else weight_cols_kernel<DT, 128><<<(unsigned)items, 128, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? MI_OK : MI_ERR_LAUNCH;
}

}  // namespace mib200

using namespace mib200;

extern "C" size_t mi_attn_weights_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t S_q,
                                                 int64_t C, int64_t D, int have_lse) {
  if (!cache_sizes_ok(B, Hq, Hkv, S_q, 1, 0, C, D)) return SIZE_MAX;
  if (B == 0 || Hq == 0 || S_q == 0 || C == 0 || have_lse) return 0;
  const CachePlan pl = cache_plan(B, Hkv, Hq / Hkv, S_q, 1, 0, C);
  const size_t rows = (size_t)(B * Hq * S_q);
  if ((double)rows * pl.NS > 1e13) return SIZE_MAX;
  return align_up(rows * pl.NS * 8) + align_up(rows * 4);
}

extern "C" int mi_attn_weights(mi_tensor4 q, mi_tensor4 k, const float* lse,
                               const int32_t* lengths, const float* w_in, int64_t w_in_stride_b,
                               int64_t w_in_stride_h, float* w_out, int64_t w_out_stride_b,
                               int64_t w_out_stride_h, int64_t B, int64_t Hq, int64_t Hkv,
                               int64_t S_q, int64_t C, int64_t D, int dtype, int causal,
                               float softmax_scale, void* workspace, size_t workspace_bytes,
                               void* stream) {
  if (dtype != MI_F16 && dtype != MI_BF16) return MI_ERR_DTYPE;
  if (!cache_sizes_ok(B, Hq, Hkv, S_q, 1, 0, C, D)) return MI_ERR_SHAPE;
  if (B == 0 || C == 0) return MI_OK;
  if (Hq == 0 || S_q == 0) return MI_ERR_SHAPE;  // no rows: nothing to add
  if (!w_out) return MI_ERR_SHAPE;
  int rc;
  if ((rc = cache_view_ok(q, B, Hq, S_q)) != MI_OK) return rc;
  if ((rc = cache_view_ok(k, B, Hkv, C)) != MI_OK) return rc;
  const int64_t group = Hq / Hkv;
  const size_t need = mi_attn_weights_workspace_size(B, Hq, Hkv, S_q, C, D, lse != nullptr);
  if (need == SIZE_MAX) return MI_ERR_SHAPE;
  if (need && (!workspace || workspace_bytes < need ||
               (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return MI_ERR_WORKSPACE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool bf = dtype == MI_BF16;

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
  w.win = w_in;
  w.wi_b = w_in_stride_b;
  w.wi_h = w_in_stride_h;
  w.wout = w_out;
  w.wo_b = w_out_stride_b;
  w.wo_h = w_out_stride_h;
  w.B = (int)B;
  w.Hq = (int)Hq;
  w.Hkv = (int)Hkv;
  w.group = (int)group;
  w.Sq = (int)S_q;
  w.C = (int)C;
  w.D = (int)D;
  w.causal = causal ? 1 : 0;
  w.scale_log2 = softmax_scale * 1.4426950408889634f;
  w.tiles = (int)((C + kColsKeys - 1) / kColsKeys);

  if (!lse) {
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
    set_seg(p.seg[1], k, k, lengths, C, B, 1, group * S_q, w.causal);
    p.seg[1].rtiles = pl.rtiles[1];
    p.seg[1].nsplit = pl.nsplit[1];
    p.seg[1].chunk = pl.chunk[1];
    p.NS = pl.NS;
    p.ml = static_cast<float2*>(workspace);
    float* lse2 = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                           align_up(rows * pl.NS * 8));
    const long long items = (long long)B * Hkv * pl.rtiles[1] * pl.nsplit[1];
    if (items > 0x7fffffffll) return MI_ERR_SHAPE;
    rc = bf ? launch_rows_dk<__nv_bfloat16, true>(p, pl.mt, items, st)
            : launch_rows_dk<__half, true>(p, pl.mt, items, st);
    if (rc != MI_OK) return rc;
    weight_lse_kernel<<<(unsigned)((rows + 255) / 256), 256, 0, st>>>(p.ml, pl.NS, lse2,
                                                                      (long long)rows);
    if (cudaGetLastError() != cudaSuccess) return MI_ERR_LAUNCH;
    w.lse = lse2;
    w.lse_mul = 1.f;
  }
  return bf ? launch_cols<__nv_bfloat16>(w, st) : launch_cols<__half>(w, st);
}
