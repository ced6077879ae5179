// Host-side helpers: TMA tensor-map construction for BNSD views.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <atomic>
#include <cstdio>
#include <cstdlib>

#include "../../include/minference_b200.h"

namespace mib200 {

inline size_t align_up(size_t x) { return (x + 255) & ~(size_t)255; }

// A query-row window [row_begin, row_end) of an S-row sequence that the
// attention launch can restrict itself to: whole 128-row tiles, except that
// the window may end at S.
inline bool row_window_ok(int64_t row_begin, int64_t row_end, int64_t S) {
  if (row_begin < 0 || row_end < row_begin || row_end > S) return false;
  return row_begin % 128 == 0 && (row_end % 128 == 0 || row_end == S);
}

// cuTensorMapEncodeTiled is fetched through the runtime's driver entry point
// so the library does not link libcuda directly.
inline PFN_cuTensorMapEncodeTiled_v12000 get_encode_tiled() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) ==
            cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }
  return fn;
}

// 4-D map over a [B, H, S, D] view of 16-bit elements with a box of
// box_d x box_s elements (box_d * 2 == 64 bytes, 64-byte swizzle).
// Rows beyond S read as zeros.
inline int make_bnsd_map(CUtensorMap* map, const mi_tensor4& t, int64_t B, int64_t H, int64_t S,
                         int64_t D, int box_d, int box_s) {
  auto enc = get_encode_tiled();
  if (!enc) return MI_ERR_LAUNCH;
  if (t.stride_d != 1) return MI_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(t.ptr) & 15) return MI_ERR_ALIGN;
  const int64_t es = 2;
  if (t.head_index) {  // the map spans every head of the view; the kernel picks them
    if (t.head_extent < 1) return MI_ERR_SHAPE;
    H = t.head_extent;
  }
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)S, (cuuint64_t)H, (cuuint64_t)B};
  int64_t st[3] = {t.stride_s * es, t.stride_h * es, t.stride_b * es};
  cuuint64_t strides[3];
  int64_t span = D * es;  // bytes covered by the inner dimensions so far
  for (int i = 0; i < 3; ++i) {
    if (dims[i + 1] == 1) st[i] = ((span + 15) / 16) * 16;  // stride of a size-1 dim is unused
    if (st[i] <= 0 || st[i] % 16) return MI_ERR_ALIGN;
    strides[i] = (cuuint64_t)st[i];
    const int64_t ext = st[i] * (int64_t)dims[i + 1];
    if (ext > span) span = ext;
  }
  cuuint32_t box[4] = {(cuuint32_t)box_d, (cuuint32_t)box_s, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, t.ptr, dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MI_OK : MI_ERR_ALIGN;
}

// 2-D map over `rows` rows of D 16-bit elements, `row_stride` elements apart,
// with a box of box_d x 1 (the shape tile::gather4 loads take); 64-byte
// swizzle like the 4-D maps.
inline int make_rows_map(CUtensorMap* map, void* ptr, int64_t rows, int64_t row_stride,
                         int64_t D, int box_d) {
  auto enc = get_encode_tiled();
  if (!enc) return MI_ERR_LAUNCH;
  if ((reinterpret_cast<uintptr_t>(ptr) & 15) || (row_stride * 2) % 16 || rows <= 0 ||
      rows >= (1ll << 31))
    return MI_ERR_ALIGN;
  cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(row_stride * 2)};
  cuuint32_t box[2] = {(cuuint32_t)box_d, 1};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, ptr, dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MI_OK : MI_ERR_ALIGN;
}

// With MI_DEBUG=1 in the environment, a failed kernel launch prints the CUDA
// error and the kernel's resource attributes to stderr (the C ABI itself only
// returns MI_ERR_LAUNCH).
inline void debug_launch_failure(const char* name, const void* func, cudaError_t err,
                                 int threads, int smem_bytes) {
  const char* dbg = getenv("MI_DEBUG");
  if (!dbg || dbg[0] != '1') return;
  cudaFuncAttributes fa{};
  cudaFuncGetAttributes(&fa, func);
  fprintf(stderr,
          "[minference_b200] %s launch failed: %s (threads %d, dynamic smem %d; kernel: %d regs, "
          "max threads %d, static smem %zu, local %zu)\n",
          name, cudaGetErrorString(err), threads, smem_bytes, fa.numRegs, fa.maxThreadsPerBlock,
          fa.sharedSizeBytes, fa.localSizeBytes);
}

// Raises a kernel's shared-memory limit once per device (the call costs about
// as much as a launch's arguments).
template <auto Kern>
inline cudaError_t allow_smem(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (err != cudaSuccess || (done.load(std::memory_order_acquire) & bit)) return err;
  err = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return err;
}

// Programmatic launch: the kernel may be set up and start while the one before
// it drains; it waits (griddepcontrol.wait) before it reads that one's results.
// Only behind a kernel of the same call, whose own launch has waited for
// whatever wrote the inputs.
template <typename K, typename... A>
inline cudaError_t launch_after(K kern, dim3 grid, int threads, size_t smem, cudaStream_t stream,
                                A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kern, args...);
  if (err != cudaSuccess) cudaGetLastError();  // reported by the status alone
  return err;
}

// 4-D map of a [B, H, S, D] tensor given by its rows (see make_bnsd_map).
inline int make_rows4_map(CUtensorMap* map, const mi_rows& r, int64_t B, int64_t H, int64_t S,
                          int64_t D, int box_d, int box_s) {
  mi_tensor4 t{};
  t.ptr = r.ptr;
  t.stride_b = r.stride_b;
  t.stride_h = r.stride_h;
  t.stride_s = r.stride_s;
  t.stride_d = 1;
  return make_bnsd_map(map, t, B, H, S, D, box_d, box_s);
}

}  // namespace mib200
