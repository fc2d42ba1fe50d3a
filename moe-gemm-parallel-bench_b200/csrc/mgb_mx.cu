// Host side of the e8m0 block-scaled products and quantisation
// (mgb_mx_kernel.cuh): argument checks, the choice of kernel, launches.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstdint>
#include <cstring>

#include "../../include/moe_gemm_b200.h"
#include "mgb_dispatch.cuh"
#include "mgb_mx_kernel.cuh"

namespace {

using namespace mgb;

int64_t cdiv(int64_t a, int64_t b) { return a / b + (a % b != 0 ? 1 : 0); }

// a * b, or -1 from 2^31 on: the quantisation kernels count blocks in 32 bits
// (FastDiv) and a thread block each.
int64_t block_count(int64_t a, int64_t b) {
  constexpr int64_t limit = 1ll << 31;
  return a < limit && b < limit && a * b < limit ? a * b : -1;
}
bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <int G, int ROWS>
int launch_mx(const MxParams& p, int64_t tiles, int sm_count, cudaStream_t stream, mgb_launch_info* info) {
  using Cfg = MxCfg<G, ROWS>;
  static bool configured[128] = {};
  static int clusters[128] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 128) return MGB_ERR_CUDA;
  cudaLaunchAttribute attr[2] = {};
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kMxThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg::kSmemBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = G * p.split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(mx_kernel<G, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes) !=
        cudaSuccess) {
      return MGB_ERR_CUDA;
    }
    clusters[dev] = sm_count / G;
    if (G == 2) {
      cfg.gridDim = dim3(static_cast<unsigned>(sm_count & ~1), 1, 1);
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, mx_kernel<G, ROWS>, &cfg) == cudaSuccess && n > 0) {
        clusters[dev] = n;
      } else {
        cudaGetLastError();
      }
    }
    configured[dev] = true;
  }
  // A split launch has one cluster per tile (never more CTAs than SMs).
  const int64_t grid = p.split > 1 ? tiles : std::max<int64_t>(1, std::min<int64_t>(tiles, clusters[dev]));
  cfg.gridDim = dim3(static_cast<unsigned>(grid * G * p.split), 1, 1);
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  if (info != nullptr) info->grid = static_cast<int32_t>(cfg.gridDim.x);
  return cudaLaunchKernelEx(&cfg, mx_kernel<G, ROWS>, p) == cudaSuccess ? MGB_OK : MGB_ERR_CUDA;
}

FastDiv fast_div(int64_t d) {
  uint32_t log = 0;
  while ((1ll << log) < d) ++log;
  const uint32_t s = 31 + log;
  return FastDiv{static_cast<uint32_t>(d), static_cast<uint32_t>(((1ull << s) + d - 1) / d), s};
}

// The widest access that the bases, pitches (elements) and row length allow.
template <typename T>
int access_of(const void* x, int64_t pitch, int64_t stride, const void* q, int64_t q_pitch, int64_t q_stride, int64_t cols) {
  const int size = static_cast<int>(sizeof(T));
  const auto whole = [&](int bytes, int out) {
    return aligned(x, bytes) && (pitch * size) % bytes == 0 && (stride * size) % bytes == 0 && cols % out == 0 &&
           aligned(q, out) && q_pitch % out == 0 && q_stride % out == 0;
  };
  return whole(32, 16) ? k32Bytes : whole(16, 8) ? k16Bytes : kScalar;
}

template <typename T>
int rows_typed(const void* x, int64_t rows, int64_t cols, int64_t pitch, void* q, int64_t q_pitch, void* scale,
               cudaStream_t s) {
  const int64_t blocks = block_count(rows, cdiv(cols, 128));
  if (blocks < 0) return MGB_ERR_INVALID;
  const int access = access_of<T>(x, pitch, 0, q, q_pitch, 0, cols);
  const bool dense = pitch == cols && q_pitch == cols && cols % 128 == 0;
  const auto kernel = access == k32Bytes   ? quantize_rows_kernel<T, k32Bytes>
                      : access == k16Bytes ? quantize_rows_kernel<T, k16Bytes>
                                           : quantize_rows_kernel<T, kScalar>;
  return launch_overlapped(kernel, static_cast<unsigned>(cdiv(blocks, 32)), 256, 0, s, static_cast<const T*>(x),
                           static_cast<uint32_t>(blocks), fast_div(cdiv(cols, 128)), cols, pitch,
                           static_cast<uint8_t*>(q), q_pitch, static_cast<uint8_t*>(scale), dense) == cudaSuccess
             ? MGB_OK
             : MGB_ERR_CUDA;
}

template <typename T>
int blocks_typed(const void* x, int64_t matrices, int64_t rows, int64_t cols, int64_t pitch, int64_t stride, void* q,
                 void* scale, cudaStream_t s) {
  const int64_t kb = cdiv(cols, 128), per = block_count(cdiv(rows, 128), kb);
  if (per < 0 || block_count(matrices, per) < 0) return MGB_ERR_INVALID;
  const int access = access_of<T>(x, pitch, stride, q, cols, rows * cols, cols);
  const auto kernel = access == k32Bytes   ? quantize_blocks_kernel<T, k32Bytes>
                      : access == k16Bytes ? quantize_blocks_kernel<T, k16Bytes>
                                           : quantize_blocks_kernel<T, kScalar>;
  return launch_overlapped(kernel, static_cast<unsigned>(matrices * per), 256, 0, s, static_cast<const T*>(x), rows,
                           cols, pitch, stride, static_cast<uint8_t*>(q), cols, rows * cols,
                           static_cast<uint8_t*>(scale), fast_div(kb), fast_div(per)) == cudaSuccess
             ? MGB_OK
             : MGB_ERR_CUDA;
}

int launch_few(const MxParams& p, unsigned grid, cudaStream_t s) {
  static bool configured[128] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 128) return MGB_ERR_CUDA;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(mx_few_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmemBytes) != cudaSuccess) {
      return MGB_ERR_CUDA;
    }
    configured[dev] = true;
  }
  return launch_overlapped(mx_few_kernel, grid, kFewWarps * 32, kFewSmemBytes, s, p) == cudaSuccess ? MGB_OK
                                                                                                          : MGB_ERR_CUDA;
}

// Whether the weight-streaming kernel runs: at most 8 rows an expert on
// average (one pass over its weight rows) and two waves of its CTAs (two per
// SM), each of which starts anew.  4 rows, against the tiles: n 1024, k 1024
// 3.0 and 7.5 us; n 4096, k 7168 9.2 and 13.3; two such experts 16.1 and 18.7;
// 8 of 1024 x 2048 7.5 and 10.8; 16 of them 12.5 and 11.6; 32 of 1024 x 1024
// 16.9 and 12.1; 8 of 4096 x 7168 67 and 50.
bool few_rows(int64_t rows, int64_t experts, int64_t n, int sms) {
  return rows <= 8 * experts && experts * cdiv(n, 16) <= 4 * static_cast<int64_t>(sms);
}

}  // namespace

extern "C" {

size_t block_scaled_mm_scratch_bytes(int32_t experts) {
  // The tile list, where it does not fit shared memory.
  return experts > 0 && 2 * static_cast<int64_t>(experts) + 1 > kMxListWords
             ? (static_cast<size_t>(experts) + 1 + 31) / 32 * 32 * sizeof(int32_t)
             : 0;
}

int block_scaled_mm_launch(const void* a, int64_t a_pitch, const void* sa, const void* b, int64_t b_pitch,
                           int64_t b_stride, const void* sb, void* c, int64_t c_pitch, const int32_t* offs,
                           int32_t experts, int64_t rows, int64_t n, int64_t k, void* scratch, size_t scratch_bytes,
                           void* stream, mgb_launch_info* info) {
  if (experts <= 0 || experts > (1 << 20) || rows < 0 || rows > (1ll << 31) - 1024 || n <= 0 || n >= (1ll << 31) || k <= 0 ||
      k >= (1ll << 30) || k % 16 != 0 || n % 8 != 0 || (offs == nullptr && experts != 1)) {
    return MGB_ERR_INVALID;
  }
  if ((rows > 0 && (a == nullptr || sa == nullptr || c == nullptr)) || b == nullptr || sb == nullptr ||
      !aligned(a, 16) || !aligned(b, 16) || !aligned(c, 16) || a_pitch < k || a_pitch % 16 != 0 || b_pitch < k ||
      b_pitch % 16 != 0 || (experts > 1 && (b_stride % b_pitch != 0 || b_stride < n * b_pitch)) || c_pitch < n ||
      c_pitch % 8 != 0) {
    return MGB_ERR_INVALID;
  }
  const size_t need = block_scaled_mm_scratch_bytes(experts);
  if (need > 0 && (scratch == nullptr || !aligned(scratch, 128) || scratch_bytes < need)) return MGB_ERR_SCRATCH;
  int sms = 0;
  MxParams p;
  std::memset(&p, 0, sizeof(p));
  p.error_word = current_error_word();
  if (p.error_word == nullptr || !current_launch_limits(&sms, &p.wait_budget)) return MGB_ERR_CUDA;
  if (info != nullptr) std::memset(info, 0, sizeof(*info));
  if (rows == 0) return MGB_OK;
  p.a = static_cast<const uint8_t*>(a);
  p.sa = static_cast<const uint8_t*>(sa);
  p.b = static_cast<const uint8_t*>(b);
  p.sb = static_cast<const uint8_t*>(sb);
  p.c = static_cast<__nv_bfloat16*>(c);
  p.a_pitch = a_pitch;
  p.b_pitch = b_pitch;
  p.b_stride = b_stride;
  p.c_pitch = c_pitch;
  p.offs = offs;
  p.experts = experts;
  p.rows = rows;
  p.n = n;
  p.k = k;
  p.kb = cdiv(k, 128);
  p.nb = cdiv(n, 128);
  p.scale_words = p.kb % 4 == 0 && aligned(sa, 4) && aligned(sb, 4);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t each = cdiv(rows, experts);
  if (few_rows(rows, experts, n, sms)) {
    const unsigned grid = static_cast<unsigned>(cdiv(n, 16) * experts);
    if (info != nullptr) {
      info->path = 3;
      info->swap_ab = 1;
      info->tile_m = 8;
      info->tile_n = 16;
      info->tile_k = 128;
      info->grid = static_cast<int32_t>(grid);
    }
    return launch_few(p, grid, s);
  }
  // Pairs' tiles of up to 224 rows x 256 outputs from 112 rows an expert where
  // they cover the device's pairs once (32 experts, n 4096, k 7168: 214 against
  // 289 us at 128 rows, 208 against 205 at 112, 204 against 187 at 104); else
  // one CTA's 128 x 128, or 64 x 128 up to 20 rows an expert (171 against
  // 175 us at 16; at 32 172 against 178, but 191 against 177 under uneven
  // routing, which gives some experts a second tile).
  const int64_t segments = std::min<int64_t>(experts, rows);
  const int64_t pair_tiles = (cdiv(rows, MxCfg<2>::kTokens) + segments - 1) * cdiv(n, MxCfg<2>::kOut);
  bool pair = each >= 112 && pair_tiles >= sms / 2;
  // One segment's tiles are counted exactly: pairs where they take fewer waves
  // (640 x 4096 x 7168: 28 against 40 us), or more than two; else the smaller
  // tiles end sooner (512 x 7168 x 7168: 45 against 50 us).
  if (experts == 1) {
    const int64_t waves = cdiv(pair_tiles, sms / 2);
    pair = each >= 112 && (waves > 2 || waves < cdiv(cdiv(rows, 128) * cdiv(n, 128), sms));
  }
  const bool half = !pair && each <= 20;
  const int tile_rows = pair ? MxCfg<2>::kTokens : half ? 64 : 128;
  const int tile_cols = pair ? MxCfg<2>::kOut : MxCfg<1>::kOut;
  const int64_t tiles = (cdiv(rows, tile_rows) + segments - 1) * cdiv(n, tile_cols);
  if (tiles >= (1ll << 31)) return MGB_ERR_INVALID;  // the list's 32-bit tile numbers
  // Split K: as many CTAs a tile (2, 4 or 8) as the SMs hold at once, each
  // with at least four K blocks.
  p.split = 1;
  const auto fits = [&](int size) {
    return tiles <= resident_clusters(reinterpret_cast<const void*>(mx_kernel<1, 128>), kMxThreads, MxCfg<1>::kSmemBytes, size);
  };
  while (!pair && p.split < 8 && tiles * p.split * 2 <= sms && p.kb >= 8 * p.split && fits(p.split * 2)) p.split *= 2;
  p.split_blocks = static_cast<int32_t>(cdiv(cdiv(p.kb, p.split), 4) * 4);
  const uint64_t stride = static_cast<uint64_t>(experts > 1 ? b_stride : b_pitch * n);
  if (!encode_map_2d(&p.map[0], kMapBytes8, a, k, rows, a_pitch, 128, pair ? MxCfg<2>::kRowsB : half ? 64 : 128) ||
      !encode_map_3d(&p.map[1], kMapBytes8, b, k, n, experts, b_pitch, stride, 128, 128) ||
      (!pair && !encode_map_2d(&p.map[2], MGB_BF16, c, n, rows, c_pitch * 2, 32, 32, 64))) {
    return MGB_ERR_CUDA;
  }
  if (need > 0) {
    int32_t* list = static_cast<int32_t*>(scratch);
    if (launch_overlapped(mx_list_kernel, 1, 32, 0, s, p, list, tile_rows, tile_cols) != cudaSuccess) return MGB_ERR_CUDA;
    p.tile_start = list;
  }
  if (info != nullptr) {
    info->path = pair ? 2 : 0;
    info->tile_m = tile_rows;
    info->tile_n = tile_cols;
    info->tile_k = 128;
    info->stages = pair ? MxCfg<2>::kStages : half ? MxCfg<1, 64>::kStages : MxCfg<1>::kStages;
  }
  return pair   ? launch_mx<2, 128>(p, tiles, sms, s, info)
         : half ? launch_mx<1, 64>(p, tiles, sms, s, info)
                : launch_mx<1, 128>(p, tiles, sms, s, info);
}

int quantize_rows_launch(const void* x, int64_t rows, int64_t cols, int64_t pitch, int32_t dtype, void* q,
                         int64_t q_pitch, void* scale, void* stream) {
  if (rows < 0 || cols <= 0 || pitch < cols || q_pitch < cols || (rows > 0 && (x == nullptr || q == nullptr || scale == nullptr))) {
    return MGB_ERR_INVALID;
  }
  if (dtype != MGB_FP16 && dtype != MGB_BF16 && dtype != MGB_FP32) return MGB_ERR_INVALID;
  if (!aligned(x, dtype == MGB_FP32 ? 4 : 2)) return MGB_ERR_INVALID;
  if (rows == 0) return MGB_OK;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case MGB_FP16: return rows_typed<__half>(x, rows, cols, pitch, q, q_pitch, scale, s);
    case MGB_BF16: return rows_typed<__nv_bfloat16>(x, rows, cols, pitch, q, q_pitch, scale, s);
    default: return rows_typed<float>(x, rows, cols, pitch, q, q_pitch, scale, s);
  }
}

int quantize_blocks_launch(const void* x, int64_t matrices, int64_t rows, int64_t cols, int64_t pitch, int64_t stride,
                           int32_t dtype, void* q, void* scale, void* stream) {
  if (matrices < 0 || rows <= 0 || cols <= 0 || pitch < cols || (matrices > 0 && (x == nullptr || q == nullptr || scale == nullptr))) {
    return MGB_ERR_INVALID;
  }
  if (dtype != MGB_FP16 && dtype != MGB_BF16 && dtype != MGB_FP32) return MGB_ERR_INVALID;
  if (!aligned(x, dtype == MGB_FP32 ? 4 : 2)) return MGB_ERR_INVALID;
  if (matrices == 0) return MGB_OK;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case MGB_FP16: return blocks_typed<__half>(x, matrices, rows, cols, pitch, stride, q, scale, s);
    case MGB_BF16: return blocks_typed<__nv_bfloat16>(x, matrices, rows, cols, pitch, stride, q, scale, s);
    default: return blocks_typed<float>(x, matrices, rows, cols, pitch, stride, q, scale, s);
  }
}

}  // extern "C"
