// Host-side launch of one native kernel variant.  The variant templates are
// instantiated per element type in mgb_tc_{f16,bf16,f32}.cu so the three
// families compile in parallel.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include "mgb_common.cuh"

namespace mgb {

// A native tensor-core tile: orientation and token / weight tile extents.
// `pair` selects the CTA-pair kernel (tm = tn = 256 per cluster of two CTAs).
struct TcVariant {
  bool swap;
  int tm;
  int tn;
  bool pair = false;
  bool promote = false;  // fp32 only: accumulator chunks summed in registers (tc_grouped_kernel PROMOTE)
};

// Compile-time facts of a variant the host needs (box sizes, ring depth, slots),
// plus, for the CTA-pair kernel, how many clusters the device runs at once.
struct TcVariantInfo {
  int bk;
  int stages;
  int smem_bytes;
  int max_clusters = 0;
  int box_rows = 0;  // token rows one CTA loads per stage (the activation box height)
  int box_cols = 0;  // weight columns one CTA loads per stage
};

// Returns false for a variant that is not instantiated.
template <typename T>
bool tc_variant_info(const TcVariant& v, TcVariantInfo* info);

// Launches tc_grouped_kernel<T, v.swap, v.tm, v.tn> (or the pair kernel);
// returns a cudaError_t value.  `out` is the output map (template for groups).
template <typename T>
int tc_launch(const TcVariant& v, const CUtensorMap& act, const CUtensorMap& wgt, const CUtensorMap& out,
              const GroupedParams& p, int grid, cudaStream_t stream);

// Launches build_maps_kernel<T>: the A / B / C tensor maps of every problem
// of a grouped launch into p.desc_slots; returns a cudaError_t value.
template <typename T>
int maps_launch(const CUtensorMap& act, const CUtensorMap& wgt, const CUtensorMap& out, const GroupedParams& p,
                cudaStream_t stream);

// FP8 block-scaled variants (mgb_fp8.cu): tiles swap-AB {16, 32, 64} x 256
// and 128 x 128; returns false / cudaErrorInvalidValue for others.
bool fp8_variant_info(const TcVariant& v, TcVariantInfo* info);
int fp8_launch(const TcVariant& v, const CUtensorMap& act, const CUtensorMap& wgt, const CUtensorMap& out,
               const GroupedParams& p, int grid, cudaStream_t stream);
int fp8_maps_launch(const CUtensorMap& act, const CUtensorMap& wgt, const CUtensorMap& out, const GroupedParams& p,
                    cudaStream_t stream);

// The current device's error word (device pointer), or nullptr when the CUDA
// runtime cannot resolve it; kernels outside the GEMM families OR their
// kErr* bits into it.
uint32_t* current_error_word();

// The current device's SM count and the wait budget of bounded barrier waits
// (mgb_set_debug); false when the CUDA runtime cannot resolve them.
bool current_launch_limits(int* sm_count, long long* wait_budget);

// Clusters of `size` (2, 4 or 8) CTAs that the current device holds at once,
// for kernels of one CTA per SM like `kernel` (clusters do not cross a GPC,
// whose SMs hold whole clusters only).
int resident_clusters(const void* kernel, int threads, int smem_bytes, int size);

// 2-D row-major tensor map with the 128- or 64-byte swizzle: `inner` contiguous
// elements per row, `outer` rows, `pitch` bytes between rows, boxes of
// box_inner x box_outer.  `dtype` is an mgb_dtype, or kMapBytes8 for bytes.
// current_launch_limits must have succeeded before.
constexpr int kMapBytes8 = 100;
bool encode_map_2d(CUtensorMap* map, int dtype, const void* base, uint64_t inner, uint64_t outer, uint64_t pitch,
                   uint32_t box_inner, uint32_t box_outer, int swizzle_bytes = 128);

// 3-D map of `outer` such matrices `stride` bytes apart (a whole number of
// pitches), one of them per box, with the 128-byte swizzle.
bool encode_map_3d(CUtensorMap* map, int dtype, const void* base, uint64_t inner, uint64_t rows, uint64_t outer,
                   uint64_t pitch, uint64_t stride, uint32_t box_inner, uint32_t box_rows);

// Launches `kernel` with programmatic stream serialization: its blocks may be
// set up while the kernel before it on the stream still runs, so it must call
// grid_dependency_wait before it touches global memory.
template <typename... Params, typename... Args>
inline cudaError_t launch_overlapped(void (*kernel)(Params...), unsigned grid, unsigned block, size_t smem,
                                     cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1] = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(block, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

// Launches simt_grouped_kernel<T>; returns a cudaError_t value.
template <typename T>
int simt_launch(const GroupedParams& p, int grid, cudaStream_t stream);

}  // namespace mgb
