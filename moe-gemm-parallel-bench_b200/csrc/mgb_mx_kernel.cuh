// e4m3 products with power-of-two block scales, and the quantisation to them.
//
//   C[m, n] = sum_kb 2^(sa[m, kb] - 127) 2^(sb[n / 128, kb] - 127) sum_{k in kb} A[m, k] B[n, k]
//
// over 128-deep K blocks kb; scales are e8m0 bytes (byte 255 is NaN).  The
// sm_100 block-scaled MMA (tcgen05.mma kind::mxf8f6f4.block_scale) applies one
// such byte per row and 32 K inside the tensor core, so a 128-deep block is
// four MMAs that name the same byte and the accumulator stays in TMEM for all
// of K: no partial is read back and scaled in registers, which is what bounds
// the fp32-scaled path (mgb_fp8_kernel.cuh).
//
// Kernels here may be resident while the kernel before them still writes what
// they read (grid_dependency_wait orders the two), so none of that memory is
// read-only for a kernel's whole life: it is read by ordinary loads, not by
// non-coherent ones, and no pointer is declared unaliased.
#pragma once

#include <cuda_fp8.h>

#include "mgb_tc_kernel.cuh"

namespace mgb {

// ------------------------------------------------------------ quantisation
// Exponent byte of the smallest power of two s with amax <= 448 s (clamped to
// the format; 1 for a block of zeros).  amax = 1.f 2^(E - 127): 448 = 1.75 2^8,
// so s = 2^(E - 127 - 8), doubled when 1.f > 1.75.
__device__ __forceinline__ int scale_byte(uint32_t amax_bits) {
  if (amax_bits == 0) return 127;
  const int e = static_cast<int>(amax_bits >> 23) - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return e < 0 ? 0 : e > 254 ? 254 : e;
}

// 2^(127 - byte): what an element is multiplied by (exact: a power of two).
__device__ __forceinline__ float inverse_scale(int byte) {
  const int b = 254 - byte;
  return __uint_as_float(b > 0 ? static_cast<uint32_t>(b) << 23 : 0x00400000u);
}

// 2^(byte - 127); byte 255 is NaN.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
}

// Two e4m3 values of a * inv, b * inv, round to nearest even.
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b, float inv) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3);
}

// Sixteen consecutive elements of a row as loaded (16-bit types stay packed):
// eight lanes hold a 1 x 128 block.
template <typename T>
struct Sixteen {
  static constexpr int kWords = 4 * static_cast<int>(sizeof(T));
  uint32_t w[kWords];
};

// How rows may be addressed: element by element; in 16-byte pieces (rows and
// their length in whole pieces of eight 16-bit elements); in 32-byte pieces.
enum Access : int { kScalar = 0, k16Bytes = 1, k32Bytes = 2 };

// From column `col`; columns past `cols` are 0.
template <typename T, int ACCESS>
__device__ __forceinline__ Sixteen<T> load16(const T* row, int64_t col, int64_t cols) {
  Sixteen<T> v;
  if constexpr (ACCESS == k32Bytes) {
    const bool in = col < cols;
    if (!in) {
#pragma unroll
      for (int i = 0; i < Sixteen<T>::kWords; ++i) v.w[i] = 0u;
    } else {
#pragma unroll
      for (int i = 0; i < Sixteen<T>::kWords / 8; ++i) {
        uint32_t* w = v.w + 8 * i;
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                     : "l"(reinterpret_cast<const uint32_t*>(row + col) + 8 * i));
      }
    }
  } else if constexpr (ACCESS == k16Bytes) {
    constexpr int kPiece = 16 / static_cast<int>(sizeof(T));  // elements per piece
#pragma unroll
    for (int i = 0; i < Sixteen<T>::kWords / 4; ++i) {
      const uint4 x = col + i * kPiece < cols ? __ldcs(reinterpret_cast<const uint4*>(row + col) + i)
                                              : make_uint4(0u, 0u, 0u, 0u);
      v.w[4 * i] = x.x;
      v.w[4 * i + 1] = x.y;
      v.w[4 * i + 2] = x.z;
      v.w[4 * i + 3] = x.w;
    }
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v.w[i] = col + i < cols ? __float_as_uint(row[col + i]) : 0u;
  } else {
    const uint16_t* r = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t lo = col + 2 * i < cols ? r[col + 2 * i] : 0u, hi = col + 2 * i + 1 < cols ? r[col + 2 * i + 1] : 0u;
      v.w[i] = lo | (hi << 16);
    }
  }
  return v;
}

// Elements 2 i and 2 i + 1.
template <typename T>
__device__ __forceinline__ float2 two_floats(const Sixteen<T>& v, int i) {
  if constexpr (sizeof(T) == 4) {
    return make_float2(__uint_as_float(v.w[2 * i]), __uint_as_float(v.w[2 * i + 1]));
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return make_float2(__uint_as_float(v.w[i] << 16), __uint_as_float(v.w[i] & 0xFFFF0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&v.w[i]));
  }
}

// Largest |element| as the type's bits: sign cleared, a floating value's bits
// order as an unsigned integer, so 16-bit pairs take one packed maximum.
// Infinities and NaNs come out on top (>= non_finite).
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const Sixteen<T>& v, uint32_t top) {
#pragma unroll
  for (int i = 0; i < Sixteen<T>::kWords; ++i) {
    if constexpr (sizeof(T) == 4) {
      top = max(top, v.w[i] & 0x7FFFFFFFu);
    } else {
      top = __vmaxu2(top, v.w[i] & 0x7FFF7FFFu);
    }
  }
  return top;
}
template <typename T>
__device__ __forceinline__ uint32_t fold_top(uint32_t top) {
  return sizeof(T) == 4 ? top : max(top & 0xFFFFu, top >> 16);
}
template <typename T>
constexpr uint32_t non_finite() {
  return sizeof(T) == 4 ? 0x7F800000u : std::is_same<T, __nv_bfloat16>::value ? 0x7F80u : 0x7C00u;
}
// The fp32 bits of a value given by the type's bits.
template <typename T>
__device__ __forceinline__ uint32_t float_bits(uint32_t bits) {
  if constexpr (sizeof(T) == 4) {
    return bits;
  } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return bits << 16;
  } else {
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(bits))));
  }
}
// Rare: the maximum over the finite elements of a block that holds others.
template <typename T>
__device__ __forceinline__ uint32_t finite_top_bits(const Sixteen<T>& v, uint32_t top) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t b = sizeof(T) == 4 ? v.w[i % Sixteen<T>::kWords] & 0x7FFFFFFFu : (v.w[i / 2] >> (16 * (i & 1))) & 0x7FFFu;
    if (b < non_finite<T>()) top = max(top, b);
  }
  return top;
}

// Sixteen e4m3 values; `odd`: the block holds infinities or NaNs, which become NaN.
template <typename T, int ACCESS>
__device__ __forceinline__ void store16(uint8_t* row, int64_t col, int64_t cols, const Sixteen<T>& v, float inv, bool odd) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 a = two_floats(v, 2 * i), b = two_floats(v, 2 * i + 1);
    if (odd) {
      const float nan = __uint_as_float(0x7FC00000u);
      a = make_float2(isinf(a.x) ? nan : a.x, isinf(a.y) ? nan : a.y);
      b = make_float2(isinf(b.x) ? nan : b.x, isinf(b.y) ? nan : b.y);
    }
    w[i] = e4m3_pair(a.x, a.y, inv) | (e4m3_pair(b.x, b.y, inv) << 16);
  }
  if constexpr (ACCESS == k32Bytes) {
    if (col < cols) *reinterpret_cast<uint4*>(row + col) = make_uint4(w[0], w[1], w[2], w[3]);
  } else if constexpr (ACCESS == k16Bytes) {
    if (col < cols) *reinterpret_cast<uint2*>(row + col) = make_uint2(w[0], w[1]);
    if (col + 8 < cols) *reinterpret_cast<uint2*>(row + col + 8) = make_uint2(w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (col + i < cols) row[col + i] = static_cast<uint8_t>(w[i / 4] >> (8 * (i % 4)));
    }
  }
}

// n / d for n < 2^31 as a multiply and a shift: with 2^(s-1) < d <= 2^s and
// m = ceil(2^(31+s) / d), n m / 2^(31+s) exceeds n / d by less than 1 / d.
struct FastDiv {
  uint32_t d, m, s;
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * m) >> s);
  }
};

// Rows: a thread per sixteen elements, eight threads per 1 x 128 block, one
// block of 32 blocks per CTA step: 32-byte loads, 16-byte stores, no loop.
// One read and one write of every element, bound by memory.  `dense`: rows of
// whole blocks without padding, whose b-th block starts at element 128 b.
// (bf16 8191 x 7168, 176 MB: 30.0 to 32.1 us; 8 elements a thread, four blocks in
// flight 2 us more; a copy of as many bytes 27 us.)
template <typename T, int ACCESS>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* x, uint32_t blocks, FastDiv kb, int64_t cols,
                                                            int64_t pitch, uint8_t* q, int64_t q_pitch, uint8_t* scale,
                                                            bool dense) {
  grid_launch_dependents();
  grid_dependency_wait();
  const uint32_t b = blockIdx.x * 32u + (threadIdx.x >> 3);
  const int l = threadIdx.x & 7;
  const uint32_t eight = 0xFFu << (threadIdx.x & 24);  // the threads of a block
  if (b >= blocks) return;
  uint32_t row = 0;
  int64_t col = b * 128ll + l * 16;
  if (!dense) {
    row = kb.div(b);
    col = (b - row * kb.d) * 128ll + l * 16;
  } else {
    cols = static_cast<int64_t>(blocks) * 128;
  }
  const Sixteen<T> v = load16<T, ACCESS>(x + row * pitch, col, cols);
  uint32_t top = fold_top<T>(top_bits<T>(v, 0u));
#pragma unroll
  for (int d = 4; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(eight, top, d));
  const bool odd = top >= non_finite<T>();
  if (odd) {
    top = finite_top_bits<T>(v, 0u);
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(eight, top, d));
  }
  const int byte = scale_byte(float_bits<T>(top));
  store16<T, ACCESS>(q + row * q_pitch, col, cols, v, inverse_scale(byte), odd);
  if (l == 0) scale[b] = static_cast<uint8_t>(byte);
}

// Blocks: one CTA per 128 x 128 block, its 16384 elements in registers (8
// threads by 16 elements across, 32 rows per step), one pass over memory.
template <typename T, int ACCESS>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const T* x, int64_t rows, int64_t cols, int64_t pitch,
                                                              int64_t matrix, uint8_t* q, int64_t q_pitch,
                                                              int64_t q_matrix, uint8_t* scale, FastDiv kb,
                                                              FastDiv per) {
  __shared__ uint32_t tops[8];
  const uint32_t e = per.div(blockIdx.x), in = blockIdx.x - e * per.d;
  const uint32_t rb = kb.div(in);
  const int64_t r0 = rb * 128ll + (threadIdx.x >> 3), c = (in - rb * kb.d) * 128ll + (threadIdx.x & 7) * 16;
  const T* base = x + e * matrix;
  Sixteen<T> v[4];
  grid_launch_dependents();
  grid_dependency_wait();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t r = r0 + i * 32;
    v[i] = load16<T, ACCESS>(base + r * pitch, r < rows ? c : cols, cols);
  }
  const auto reduce = [&](uint32_t top) {
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, tops[i]);
    return top;
  };
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = top_bits<T>(v[i], top);
  top = reduce(fold_top<T>(top));
  const bool odd = top >= non_finite<T>();  // the same in every thread
  if (odd) {
    top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = finite_top_bits<T>(v[i], top);
    top = reduce(top);
  }
  const int byte = scale_byte(float_bits<T>(top));
  const float inv = inverse_scale(byte);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t r = r0 + i * 32;
    if (r < rows) store16<T, ACCESS>(q + e * q_matrix + r * q_pitch, c, cols, v[i], inv, odd);
  }
  if (threadIdx.x == 0) scale[blockIdx.x] = static_cast<uint8_t>(byte);
}

// ------------------------------------------------------------------ product
struct MxParams {
  const uint8_t* a;   // [rows, k]
  const uint8_t* sa;  // [rows, kb]
  const uint8_t* b;   // [experts, n, k]
  const uint8_t* sb;  // [experts, nb, kb]
  __nv_bfloat16* c;   // [rows, n]
  int64_t a_pitch, b_pitch, b_stride, c_pitch;  // elements
  const int32_t* offs;
  int32_t experts;
  int64_t rows, n, k;
  int64_t kb, nb;       // scale columns and rows: ceil(k / 128), ceil(n / 128)
  int32_t scale_words;  // scale rows are whole, aligned 32-bit words
  const int32_t* tile_start;  // [experts + 1] first tile of every expert; nullptr: built in shared memory
  int32_t split;        // CTAs of a cluster that share a tile's K (one CTA tiles; 1: none)
  int32_t split_blocks; // K blocks of each, a multiple of 4
  long long wait_budget;
  uint32_t* error_word;
  // A and C whole (a segment's rows are addressed absolutely; rows loaded past
  // its end only reach accumulator rows that are not stored), B 3-D by expert.
  // A pair needs no map of C.
  CUtensorMap map[3];
};

// Rows [start, start + len) of expert e, clamped into the tensor whatever offs holds.
__device__ __forceinline__ int64_t mx_segment(const int32_t* offs, int64_t rows, int e, int64_t& start,
                                              bool* bad = nullptr) {
  if (offs == nullptr) {
    start = 0;
    return rows;
  }
  const int64_t lo = e > 0 ? offs[e - 1] : 0, hi = offs[e];
  if (bad != nullptr) *bad = lo < 0 || hi < lo || hi > rows;
  start = lo < 0 ? 0 : lo > rows ? rows : lo;
  const int64_t end = hi < start ? start : hi > rows ? rows : hi;
  return end - start;
}

// Tiles of an expert's segment.
__device__ __forceinline__ int64_t mx_tiles(const int32_t* offs, const MxParams& p, int e, int tile_rows, int tile_cols,
                                            bool* bad) {
  int64_t start;
  return ceil_div64(mx_segment(offs, p.rows, e, start, bad), tile_rows) * ceil_div64(p.n, tile_cols);
}

// The tile list of a launch with too many experts for shared memory (one warp).
__global__ void __launch_bounds__(32)
    mx_list_kernel(const __grid_constant__ MxParams p, int32_t* list, int tile_rows, int tile_cols) {
  const int lane = threadIdx.x;
  const int per = (p.experts + 31) / 32;
  const int lo = lane * per, hi = lo + per < p.experts ? lo + per : p.experts;
  grid_launch_dependents();
  grid_dependency_wait();  // offs and this scratch may be in use until here
  int64_t sum = 0;
  bool bad = false;
  for (int e = lo; e < hi; ++e) {
    sum += mx_tiles(p.offs, p, e, tile_rows, tile_cols, &bad);
    if (bad) atomicOr(p.error_word, kErrBadDims);
  }
  const int64_t incl = warp_scan(sum, lane);
  int64_t run = incl - sum;
  for (int e = lo; e < hi; ++e) {
    list[e] = static_cast<int32_t>(run);
    run += mx_tiles(p.offs, p, e, tile_rows, tile_cols, &bad);
  }
  if (lane == 31) list[p.experts] = list_end(incl);
}

// Words of shared memory for the tile list and row ends, if they fit.
constexpr int kMxListWords = 400;

// A role's position in the tile list (`ts` and `offs` in shared or global memory).
// Blocks of ROWS token rows; EVEN: of equal numbers of token rows instead,
// ROWS or a multiple of 64 below it.
template <int ROWS, bool EVEN>
struct MxWalk {
  const MxParams& p;
  const int32_t* ts;
  const int32_t* offs;
  int e = -1;
  int32_t first = 0, end = 0, m_blocks = 1, each = ROWS;
  int64_t len = 0, start = 0;

  __device__ __forceinline__ MxWalk(const MxParams& params, const int32_t* list, const int32_t* ends)
      : p(params), ts(list), offs(ends) {}

  __device__ __forceinline__ bool seek(int64_t tile) {
    if (tile >= ts[p.experts]) return false;
    const int32_t t = static_cast<int32_t>(tile);
    if (t >= end || e < 0) {
      int lo = e < 0 ? 0 : e, hi = p.experts - 1;
      while (lo < hi) {  // empty experts share their successor's first tile
        const int mid = (lo + hi + 1) >> 1;
        if (ts[mid] <= t) {
          lo = mid;
        } else {
          hi = mid - 1;
        }
      }
      e = lo;
      first = ts[lo];
      end = ts[lo + 1];
      len = mx_segment(offs, p.rows, lo, start);
      m_blocks = static_cast<int32_t>(ceil_div64(len, ROWS));
      if (EVEN) each = whole(static_cast<int32_t>(ceil_div64(len, m_blocks)));
    }
    return true;
  }
  // Bands of 8 row blocks, row block fastest inside a band.
  __device__ __forceinline__ void blocks(int64_t tile, int64_t& mb, int64_t& nb) const {
    const uint32_t local = static_cast<uint32_t>(tile) - first;
    const uint32_t band_tiles = 8u * (static_cast<uint32_t>(end - first) / m_blocks);
    const uint32_t band = local / band_tiles;
    const uint32_t in = local - band * band_tiles;
    const uint32_t rows_in = m_blocks - band * 8 < 8 ? m_blocks - band * 8 : 8;
    const uint32_t column = in / rows_in;
    mb = band * 8 + (in - column * rows_in);
    nb = column;
  }
  static __host__ __device__ constexpr int32_t whole(int32_t rows) {
    rows = (rows + 63) / 64 * 64;
    return rows < ROWS ? rows : ROWS;
  }
  // Token rows of row block mb.
  __device__ __forceinline__ int32_t count(int64_t mb) const {
    const int64_t left = len - mb * each;
    return static_cast<int32_t>(left < each ? left : each);
  }
};

// D[tmem] (+)= (A 2^sa) (B 2^sb), e4m3 operands, one e8m0 scale per row and 32 K.
template <int G>
__device__ __forceinline__ void mma_mx(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                       uint32_t sfb, uint32_t accumulate) {
  if constexpr (G == 2) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  }
}

// 32 rows x 16 bytes of shared memory into 4 TMEM columns, repeated for the
// four lane quarters (the layout in which the MMA reads scales).
template <int G>
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t desc) {
  if constexpr (G == 2) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  } else {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  }
}

// Instruction descriptor of the block-scaled MMA: e4m3 operands (format 0),
// both K-major, e8m0 scales (bit 23); `byte` names the scale byte of a
// 32-bit TMEM word for both operands.
__host__ __device__ constexpr uint32_t instr_desc_mx(uint32_t m, uint32_t n, uint32_t byte) {
  return (byte << 4) | ((n >> 3) << 17) | (1u << 23) | ((m >> 7) << 27) | (byte << 29);
}

__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity, long long budget,
                                                  volatile int* abort) {
  if (mbar_try_wait_cluster(bar, parity)) return true;
  const long long start = clock64();
  while (true) {
    if (mbar_try_wait_cluster(bar, parity)) return true;
    if (*abort || clock64() - start > budget) return false;
  }
}

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// Whether every block of 1 to ROWS token rows gives a pair's MMA an N that is a
// multiple of 32 and covers the block.
template <int ROWS>
constexpr bool pair_sizes_hold() {
  for (int rows = 1; rows <= ROWS; ++rows) {
    const int n = MxWalk<ROWS, true>::whole(rows);
    if (n % 32 != 0 || n < rows || n > ROWS) return false;
  }
  return true;
}

// Tiles.  One CTA: ROWS token rows (M = 128) x 128 outputs, ROWS = 128 or 64.
// A 64-row tile still runs M = 128 MMAs: the operand's upper rows are whatever
// lies behind it in shared memory and only reach accumulator rows that are
// never stored.  It halves the token half of a stage, so eight stages (128 KB
// of weights per SM) are in flight instead of six (96 KB) while the weights'
// bytes bound the launch.
// A pair: 256 weight rows (M) x up to 224 token rows (N: 64, 128, 192 or 224,
// named by the instruction): an expert's rows are cut into equal blocks, so
// MMAs are spent on its rows rounded up to such a block instead of whole
// 256-row tiles.  N stays a multiple of 32 (pair_sizes_hold): a build whose
// blocks were rounded to 16 rows, N = 16 modulo 32, stopped twice in
// back-to-back launches.  The cause is not known; the form is not used.
// The accumulator is transposed: lanes are outputs, columns token rows.
// Two accumulators and the scale words share the 512 TMEM columns: 2 x 224 +
// 2 x 12 for a pair (N = 256 would leave none for the scales), 2 x 128 + 2 x 8
// for one CTA.
template <int G, int ROWS = 128>
struct MxCfg {
  static_assert(ROWS == 128 || (G == 1 && ROWS == 64), "token rows a CTA loads");
  static constexpr int kBK = 128;
  // K blocks that are loaded back to back: 512 consecutive bytes of a row while
  // its DRAM page is open (32 experts of 128 rows 233 -> 225 us, of 256 rows
  // 326 -> 315; one CTA's launches lose 2% by the deeper wait).
  static constexpr int kBurst = G == 2 ? 4 : 1;
  static constexpr int kRowsB = G == 2 ? 112 : 128;  // rows of the N-side operand a CTA loads
  static constexpr int kMmaM = 128 * G;
  static constexpr int kTileN = kRowsB * G;                    // accumulator columns
  static constexpr int kTokens = G == 2 ? kTileN : ROWS;       // token rows of a tile, at most
  static constexpr int kOut = G == 2 ? kMmaM : kTileN;         // output columns of a tile
  using Walk = MxWalk<kTokens, G == 2>;
  static constexpr int kABytes = ROWS * 128, kBBytes = kRowsB * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kScaleAtoms = 1 + G;           // 128 rows x 4 bytes each: A, then B's 128-row groups
  static constexpr int kScaleBytes = kScaleAtoms * 512;  // one slot: four K blocks
  static constexpr int kScaleCols = 4 * kScaleAtoms;
  static constexpr int kTmemCols = 512;
  static constexpr int kScaleTmem = 2 * kTileN;  // first scale column
  // One CTA: a staging block of 32 rows x 64 bytes per epilogue warp: the epilogue
  // runs under the next tile's MMAs, and the shared memory makes a stage.
  static constexpr int kBlockBytes = 32 * 64;
  static constexpr int kEpiBytes = 4 * kBlockBytes;
  static constexpr int kStages = (kTcSmemBudget - kEpiBytes - 2 * kScaleBytes) / kStageBytes;
  static constexpr int kSmemBytes = kStages * kStageBytes + kEpiBytes + 2 * kScaleBytes + 2048 + 1024;
  static_assert(kStageBytes % 1024 == 0 && kABytes % 1024 == 0, "swizzle atoms");
  static_assert(kScaleTmem + 2 * kScaleCols <= kTmemCols, "TMEM columns");
  static_assert(kSmemBytes <= 232448 && kStages >= 4, "shared memory");
  static_assert((2 * kStages + 9) * 8 + 12 + kMxListWords * 4 <= 2048, "barriers and the tile list");
  static_assert(G == 1 || pair_sizes_hold<kTokens>(), "N of a pair's MMA");
  // Split K (one CTA): a row of partial sums, padded against bank conflicts.
  static constexpr int kSumRow = kTileN * 4 + 16;
  static_assert(G == 2 || ROWS * kSumRow <= kStages * kStageBytes, "partial sums fit the ring");
};

static_assert(MxCfg<1, 64>::kStages == 8 && MxCfg<1, 128>::kStages == 6, "as the text above has it");

constexpr int kMxThreads = 256;

// Warps: 0 TMA producer, 1 MMA issuer, 2 scales, 3 idle, 4-7 epilogue.
// Scales: warp 2 gathers the bytes of four K blocks (one 32-bit word per row)
// into the slot's 512-byte atoms, row j 32 + l at byte 16 l + 4 j; the issuer
// copies them to TMEM and names byte kb % 4 in the MMAs of K block kb.  A
// slot (its shared memory and its TMEM columns) is free again when the MMAs
// of its four K blocks are done.
// Split K (p.split > 1, at most one tile per cluster): the CTAs of a cluster
// compute one tile over consecutive K ranges and leave fp32 sums in their own
// (then idle) operand rings; CTA r adds rows [r ROWS / split, ...) of all of
// them over distributed shared memory, in rank order, and stores them.  For
// launches whose tiles would leave at least half of the SMs idle.
// 32 experts, n 4096, k 7168 (940 MB, 144 us to read), launches in a row: 189 us
// at 16 rows each, 213 at 128.  8191 x 4096 x 7168: 210 to 230 us in a row (2.1 to
// 2.3 PFLOP/s) at 1.5 GHz under the power limit, where the tensor pipe could do
// 3.6.  In a launch alone the pipe is 65% busy, DRAM 11%, and operands leave L2 at
// 13.5 TB/s (2.6 GB; a 224 x 256 tile loads 60 KB a K block): the operand traffic
// is the likeliest bound.
template <int G, int ROWS>
__global__ void __launch_bounds__(kMxThreads, 1) mx_kernel(const __grid_constant__ MxParams p) {
  using Cfg = MxCfg<G, ROWS>;
  constexpr int S = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem;
  uint8_t* epi_stage = smem + S * Cfg::kStageBytes;
  uint8_t* scales = epi_stage + Cfg::kEpiBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + 2 * Cfg::kScaleBytes);
  uint64_t* empty = full + S;
  uint64_t* sf_full = empty + S;
  uint64_t* sf_empty = sf_full + 2;
  uint64_t* acc_full = sf_empty + 2;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain_bar = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* never = abort + 1;
  int32_t* list = reinterpret_cast<int32_t*>(tmem_slot + 3);  // kMxListWords

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = G == 2 ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const int split = G == 2 ? 1 : p.split;
  const int64_t first_item = blockIdx.x / (G * split);
  const int64_t items_step = split > 1 ? 1ll << 60 : gridDim.x / G;  // one tile where K is split
  // The next kernel may set up as SMs come free; it waits for this one's end.
  grid_launch_dependents();
  if (threadIdx.x < (G == 2 ? 2 : 3)) prefetch_tmap(&p.map[threadIdx.x]);
  // This CTA's K blocks of every tile.
  const int32_t share = split > 1 ? static_cast<int32_t>(cluster_ctarank()) : 0;
  const int32_t kb_from = share * p.split_blocks;
  const int32_t kb_to = static_cast<int32_t>(split > 1 && kb_from + p.split_blocks < p.kb ? kb_from + p.split_blocks : p.kb);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sf_full[b], G);
      mbar_init(&sf_empty[b], 1);
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4 * G);
    }
    mbar_init(drain_bar, 1);
    *abort = 0;
    *never = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (G == 2) {
      tmem_alloc_pair(tmem_slot, Cfg::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, Cfg::kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (G == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const long long budget = p.wait_budget;
  grid_dependency_wait();  // global memory is read only from here on
  const int32_t* ts = p.tile_start;
  const int32_t* offs = p.offs;
  if (ts == nullptr) {
    // The tile list: first tiles of every expert, then the row ends.
    int32_t* ends = list + p.experts + 1;
    for (int i = threadIdx.x; i < p.experts; i += kMxThreads) {
      ends[i] = p.offs != nullptr ? p.offs[i] : static_cast<int32_t>(p.rows);
    }
    __syncthreads();
    if (warp == 0) {
      int64_t before = 0;
      for (int base = 0; base < p.experts; base += 32) {
        const int e = base + lane;
        bool bad = false;
        const int64_t tiles = e < p.experts ? mx_tiles(ends, p, e, Cfg::kTokens, Cfg::kOut, &bad) : 0;
        if (bad && blockIdx.x == 0) atomicOr(p.error_word, kErrBadDims);
        const int64_t incl = warp_scan(tiles, lane);
        if (e < p.experts) list[e] = static_cast<int32_t>(before + incl - tiles);
        before += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) list[p.experts] = list_end(before);
    }
    __syncthreads();
    ts = list;
    offs = ends;
  }

  auto fail = [&](uint32_t bits) {
    atomicOr(p.error_word, bits);
    *abort = 1;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    // One thread; stage and phase step along instead of dividing a counter.
    if (lane == 0) {
      const uint64_t pol_keep = policy_evict_last(), pol_shared = policy_evict_normal();
      const uint64_t pol_stream = policy_evict_first();
      const uint32_t ring0 = smem_u32(ring), full0 = smem_u32(full), empty0 = smem_u32(empty);
      const uint32_t lead0 = G == 2 ? mapa_shared(full0, 0) : full0;  // the leader's barriers
      typename Cfg::Walk walk(p, ts, offs);
      int s = 0;
      uint32_t phase = 0, loaded = 0;
      bool ok = true;
      const int32_t begin = kb_from * Cfg::kBK, end = kb_to * Cfg::kBK;
      for (int64_t t = first_item; ok && walk.seek(t); t += items_step) {
        int64_t mb, nb;
        walk.blocks(t, mb, nb);
        // Absolute token row: a pair's CTAs hold half of the N rows each.
        const int32_t half = G == 2 ? static_cast<int32_t>(rank) * (Cfg::Walk::whole(walk.count(mb)) / 2) : 0;
        const int32_t m0 = static_cast<int32_t>(walk.start + mb * walk.each) + half;
        const int32_t n0 = static_cast<int32_t>(nb * Cfg::kOut + rank * 128);
        const uint64_t pol_b = walk.m_blocks == 1 ? pol_stream : pol_shared;
        int ready = 0;
        for (int32_t kx = begin; kx < end; kx += Cfg::kBK) {
          if (ready == 0) {
            int w = s;
            uint32_t wp = phase;
            for (; ready < Cfg::kBurst && kx + ready * Cfg::kBK < end; ++ready) {
              if (!bar_wait(empty0 + w * 8, wp ^ 1u, budget, abort)) {
                ok = false;
                break;
              }
              if (++w == S) {
                w = 0;
                wp ^= 1u;
              }
            }
            if (!ok) {
              fail(kErrWaitEmpty);
              break;
            }
          }
          --ready;
          const uint32_t st = ring0 + s * Cfg::kStageBytes;
          if (leader) mbar_arrive_expect_tx(&full[s], G * Cfg::kStageBytes);
          tile_load<G>(&p.map[0], lead0 + s * 8, st + (G == 2 ? Cfg::kABytes : 0), kx, m0, pol_keep);
          tile_load_3d<G>(&p.map[1], lead0 + s * 8, st + (G == 2 ? 0 : Cfg::kABytes), kx, n0, walk.e, pol_b);
          ++loaded;
          if (++s == S) {
            s = 0;
            phase ^= 1u;
          }
        }
      }
      if (*abort && leader) {
        for (uint32_t i = loaded > static_cast<uint32_t>(S) ? loaded - S : 0u; i < loaded; ++i) {
          if (!bar_wait(full0 + (i % S) * 8, (i / S) & 1u, budget, never)) {
            atomicOr(p.error_word, kErrWaitTeardown);
            break;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer (leader only)
    if (lane == 0 && leader) {
      const uint32_t full0 = smem_u32(full), empty0 = smem_u32(empty);
      typename Cfg::Walk walk(p, ts, offs);
      int s = 0;
      uint32_t phase = 0, acc_it = 0, sf_it = 0;
      bool ok = true;
      const uint64_t a_desc = smem_desc(smem_u32(ring), 16, 1024, kLayoutSw128);
      const uint64_t b_desc = smem_desc(smem_u32(ring) + Cfg::kABytes, 16, 1024, kLayoutSw128);
      // Scale atoms: no swizzle, 8-row groups of 16-byte rows 128 bytes apart.
      const uint64_t s_desc = smem_desc(smem_u32(scales), 0, 128, 0);
      for (int64_t t = first_item; ok && walk.seek(t); t += items_step) {
        const int buf = static_cast<int>(acc_it & 1);
        if (!mbar_wait(&acc_empty[buf], ((acc_it >> 1) & 1u) ^ 1u, budget, abort)) {
          fail(kErrWaitAccEmpty);
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + buf * Cfg::kTileN;
        uint32_t cols = Cfg::kTileN;
        if constexpr (G == 2) {
          int64_t mb, nb;
          walk.blocks(t, mb, nb);
          cols = Cfg::Walk::whole(walk.count(mb));
        }
        uint32_t acc = 0;
        for (int32_t kb4 = kb_from; ok && kb4 < kb_to; kb4 += 4) {
          const int slot = static_cast<int>(sf_it & 1);
          const uint32_t sf = tmem_base + Cfg::kScaleTmem + slot * Cfg::kScaleCols;
          if (!mbar_wait_cluster(&sf_full[slot], (sf_it >> 1) & 1u, budget, abort)) {
            fail(kErrWaitFull);
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int i = 0; i < Cfg::kScaleAtoms; ++i) {
            tmem_copy_scales<G>(sf + 4 * i, s_desc + ((slot * Cfg::kScaleBytes + i * 512) >> 4));
          }
#pragma unroll
          for (int b = 0; b < 4; ++b) {  // K block kb4 + b names byte b of its scale words
            if (kb4 + b >= kb_to) break;
            if (!bar_wait(full0 + s * 8, phase, budget, abort)) {
              fail(kErrWaitFull);
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t stage = static_cast<uint32_t>(s) * (Cfg::kStageBytes >> 4);
            const uint64_t ad = a_desc + stage, bd = b_desc + stage;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
              mma_mx<G>(d, ad + ks * 2, bd + ks * 2, instr_desc_mx(Cfg::kMmaM, G == 2 ? cols : Cfg::kTileN, b), sf, sf + 4, acc);
              acc = 1;
            }
            tile_commit<G>(empty0 + s * 8);
            if (++s == S) {
              s = 0;
              phase ^= 1u;
            }
          }
          if (!ok) break;
          tile_commit<G>(smem_u32(&sf_empty[slot]));
          ++sf_it;
        }
        if (!ok) break;
        tile_commit<G>(smem_u32(&acc_full[buf]));
        ++acc_it;
      }
      if (*abort) {
        tile_commit<G>(smem_u32(drain_bar));
        if (!mbar_wait(drain_bar, 0, budget, never)) atomicOr(p.error_word, kErrWaitTeardown);
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // -------------------------------------------------------------- scales
    typename Cfg::Walk walk(p, ts, offs);
    uint32_t sf_it = 0;
    bool ok = true;
    // Four consecutive bytes of a scale row from K block kb on; blocks past the end are 1.
    const bool words = p.scale_words;
    auto word = [&](const uint8_t* row, int64_t kb) -> uint32_t {
      if (words) return *reinterpret_cast<const uint32_t*>(row + kb);
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) w |= (kb + i < p.kb ? static_cast<uint32_t>(row[kb + i]) : 127u) << (8 * i);
      return w;
    };
    for (int64_t t = first_item; ok && walk.seek(t); t += items_step) {
      int64_t mb, nb;
      walk.blocks(t, mb, nb);
      // Rows past the segment read its last row's scales: never stored.
      const auto token = [&](int i) {
        const int64_t m = mb * walk.each + i;
        return p.sa + (walk.start + (m < walk.len ? m : walk.len - 1)) * p.kb;
      };
      const auto weight = [&](int64_t n) { return p.sb + (walk.e * p.nb + (n < p.n ? n : p.n - 1) / 128) * p.kb; };
      const int64_t n0 = nb * Cfg::kOut + rank * 128;
      const uint8_t* row[4 * Cfg::kScaleAtoms];
#pragma unroll
      for (int j = 0; j < 4 * Cfg::kScaleAtoms; ++j) {
        if constexpr (G == 2) {
          row[j] = j < 4 ? weight(n0) : token((j - 4) * 32 + lane);
        } else {
          row[j] = j < 4 ? token(j * 32 + lane) : weight(n0);
        }
      }
      for (int64_t kb = kb_from; kb < kb_to; kb += 4) {
        const int slot = static_cast<int>(sf_it & 1);
        uint32_t w[4 * Cfg::kScaleAtoms];
#pragma unroll
        for (int j = 0; j < 4 * Cfg::kScaleAtoms; ++j) w[j] = word(row[j], kb);  // in flight during the wait
        if (!mbar_wait_warp(&sf_empty[slot], ((sf_it >> 1) & 1u) ^ 1u, budget, abort)) {
          if (lane == 0) fail(kErrWaitEmpty);
          ok = false;
          break;
        }
#pragma unroll
        for (int i = 0; i < Cfg::kScaleAtoms; ++i) {
          *reinterpret_cast<uint4*>(scales + slot * Cfg::kScaleBytes + i * 512 + lane * 16) =
              make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
        fence_proxy_async_smem();  // generic writes -> visible to the copy into TMEM
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(G == 2 ? mapa_shared(smem_u32(&sf_full[slot]), 0) : smem_u32(&sf_full[slot]));
        ++sf_it;
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3;
    uint8_t* block = epi_stage + quarter * Cfg::kBlockBytes;
    const uint64_t pol_out = policy_evict_normal();
    typename Cfg::Walk walk(p, ts, offs);
    uint32_t acc_it = 0;
    for (int64_t t = first_item; walk.seek(t); t += items_step) {
      int64_t mb, nb;
      walk.blocks(t, mb, nb);
      const int buf = static_cast<int>(acc_it & 1);
      if (!mbar_wait_warp(&acc_full[buf], (acc_it >> 1) & 1u, budget, abort)) {
        if (lane == 0) fail(kErrWaitAccFull);
        break;
      }
      tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * Cfg::kTileN;
      if constexpr (G == 2) {
        // Lane pairs trade values: the even lane has two outputs of an even
        // token row, the odd lane of the next; 16 lanes store 64 bytes of a row.
        const int64_t n = nb * Cfg::kOut + rank * 128 + quarter * 32 + (lane & ~1);
        const int odd = lane & 1, count = walk.count(mb);
        __nv_bfloat16* to = p.c + (walk.start + mb * walk.each + odd) * p.c_pitch + n;
        if (n - (lane & ~1) < p.n) {
#pragma unroll 1
          for (int c = 0; c < count; c += 32, to += 32 * p.c_pitch) {
            uint32_t v[32];
            __syncwarp();
            tmem_ld32(taddr + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? v[j] : v[j + 1], 1);
              const uint32_t two = odd ? pack_pair<__nv_bfloat16>(other, v[j + 1]) : pack_pair<__nv_bfloat16>(v[j], other);
              if (c + j + odd < count && n < p.n) *reinterpret_cast<uint32_t*>(to + j * p.c_pitch) = two;
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(&acc_empty[buf]), 0));
        ++acc_it;
        continue;
      }
      const int32_t row0 = static_cast<int32_t>(mb * ROWS + quarter * 32);
      const int32_t c0 = static_cast<int32_t>(nb * Cfg::kTileN);
      if (split > 1) {
        // The last MMAs are done and nothing more is loaded: the ring holds the sums.
        if (quarter * 32 < ROWS) {
          float* sums = reinterpret_cast<float*>(ring + (quarter * 32 + lane) * Cfg::kSumRow);
#pragma unroll 1
          for (int c = 0; c < Cfg::kTileN; c += 32) {
            uint32_t v[32];
            tmem_ld32(taddr + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              *reinterpret_cast<uint4*>(sums + c + 4 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            }
          }
        }
        break;  // one tile per cluster
      }
      if (quarter * 32 < ROWS && row0 < walk.len) {
        // Chunks of 32 columns; the map clips C's edges.
        const int64_t cols = p.n - c0 < Cfg::kTileN ? p.n - c0 : Cfg::kTileN;
        // Where the segment ends inside these 32 rows, each lane stores its
        // own row straight from registers.
        const bool ragged = row0 + 32 > walk.len;
#pragma unroll 1
        for (int c = 0; c * 32 < cols; ++c) {
          uint32_t v[32];
          tmem_ld32(taddr + c * 32, v);
          if (ragged) {
            tmem_ld_wait();
            if (row0 + lane < walk.len) {
              uint4* to = reinterpret_cast<uint4*>(p.c + (walk.start + row0 + lane) * p.c_pitch + c0 + c * 32);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                if (c * 32 + 8 * j < cols) {  // n is a multiple of 8
                  to[j] = make_uint4(
                      pack_pair<__nv_bfloat16>(v[8 * j], v[8 * j + 1]), pack_pair<__nv_bfloat16>(v[8 * j + 2], v[8 * j + 3]),
                      pack_pair<__nv_bfloat16>(v[8 * j + 4], v[8 * j + 5]),
                      pack_pair<__nv_bfloat16>(v[8 * j + 6], v[8 * j + 7]));
                }
              }
            }
            continue;
          }
          if (lane == 0) bulk_wait_group_read<0>();  // the previous chunk's store has read the block
          __syncwarp();
          tmem_ld_wait();
          // 32 rows x 64 bytes, 64-byte swizzle: 16-byte unit j of row r at j ^ ((r / 2) % 4).
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            *reinterpret_cast<uint4*>(block + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
                make_uint4(pack_pair<__nv_bfloat16>(v[8 * j], v[8 * j + 1]), pack_pair<__nv_bfloat16>(v[8 * j + 2], v[8 * j + 3]),
                           pack_pair<__nv_bfloat16>(v[8 * j + 4], v[8 * j + 5]),
                           pack_pair<__nv_bfloat16>(v[8 * j + 6], v[8 * j + 7]));
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&p.map[2], block, c0 + c * 32, static_cast<int32_t>(walk.start) + row0, pol_out);
            bulk_commit_group();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_relaxed(&acc_empty[buf]);
      ++acc_it;
    }
    if (lane == 0) bulk_wait_group_read<0>();  // tensor stores have read the CTA's shared memory before it goes away
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (G == 2 || split > 1) cluster_sync();
  if (G == 1 && split > 1) {
    typename Cfg::Walk walk(p, ts, offs);
    if (walk.seek(first_item) && !*abort) {
      int64_t mb, nb;
      walk.blocks(first_item, mb, nb);
      const int per = ROWS / split;
      const int col = (threadIdx.x & 31) * 4;
      const int64_t c = nb * Cfg::kTileN + col;
      // CTAs without K blocks (a short last share) left no sums.
      const int parts = static_cast<int>((p.kb + p.split_blocks - 1) / p.split_blocks);
      for (int r = share * per + warp; r < (share + 1) * per; r += kMxThreads / 32) {
        const int64_t m = mb * ROWS + r;
        if (m >= walk.len) break;
        const float4 sum = join_parts(smem_u32(ring + r * Cfg::kSumRow + col * 4), parts);
        if (c < p.n) {  // n is a multiple of 8: four columns are inside or past the end
          uint2 out;
          out.x = pack_pair<__nv_bfloat16>(__float_as_uint(sum.x), __float_as_uint(sum.y));
          out.y = pack_pair<__nv_bfloat16>(__float_as_uint(sum.z), __float_as_uint(sum.w));
          *reinterpret_cast<uint2*>(p.c + (walk.start + m) * p.c_pitch + c) = out;
        }
      }
    }
    cluster_sync();  // the others' sums are read until here
  }
  if (warp == 1) {
    tc_fence_after();
    if constexpr (G == 2) {
      tmem_dealloc_pair(tmem_base, Cfg::kTmemCols);
    } else {
      tmem_dealloc(tmem_base, Cfg::kTmemCols);
    }
  }
}

// -------------------------------------------------------------- few tokens
// Decoding: at most a few tokens per expert, so the weights' bytes bound the
// product and the tensor pipe idles whatever drives it.  The 128-row tiles
// above would run on n / 128 SMs and stream the weights through too few of
// them; here a CTA takes 16 weight rows and its 8 warps split K (interleaved
// 128-deep blocks), so n / 16 CTAs stream.  Every thread copies the weight
// bytes that it will use itself into its own shared-memory slots (cp.async,
// no barrier), kFewDepth K blocks ahead: two CTAs keep 192 KB of weights per
// SM in flight without holding registers for them.  The warps' sums are
// joined in shared memory in warp order (the result does not depend on
// timing).
// Weights are the 16-row operand of the warp-level m16n8k32 MMA, 8 tokens its
// columns (more tokens take further passes).  A thread loads 16 consecutive
// bytes of a row and uses them as the fragments of two MMAs; weights and tokens are permuted along K alike, so
// the sum is over the same products.  Each 128-deep block starts from zero and
// is added to the fp32 sums times its two scales.  1 x 4096 x 7168 (29 MB,
// 4.5 us to read), launches in a row on weights that L2 does not hold: 10.3 us.
__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes global -> shared, zeros unless `in` (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}

constexpr int kFewWarps = 8;
constexpr int kFewDepth = 6;            // K blocks of 2 KB per warp in flight
constexpr int kFewBlock = 16 * 128;     // 16 weight rows x 128
constexpr int kFewSums = kFewWarps * 8 * 17 * 4;  // [warp][token][row], padded against bank conflicts
constexpr int kFewSmemBytes = kFewWarps * kFewDepth * kFewBlock + kFewSums;
static_assert(2 * (kFewSmemBytes + 1024) <= 233472, "two CTAs per SM");

__global__ void __launch_bounds__(kFewWarps * 32, 2) mx_few_kernel(const __grid_constant__ MxParams p) {
  extern __shared__ uint8_t few_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  float(*sums)[8][17] = reinterpret_cast<float(*)[8][17]>(few_smem + kFewWarps * kFewDepth * kFewBlock);
  const uint32_t slots = smem_u32(few_smem) + warp * kFewDepth * kFewBlock + lane * 16;
  const int64_t n_groups = ceil_div64(p.n, 16);
  const int e = static_cast<int>(blockIdx.x / n_groups);
  const int64_t r0 = (blockIdx.x - e * n_groups) * 16;
  const int depth = static_cast<int>(p.k), kblocks = static_cast<int>(p.kb);
  bool live[2];
  const uint8_t* wrow[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t r = r0 + g + 8 * h;
    live[h] = r < p.n;
    wrow[h] = p.b + e * p.b_stride + (live[h] ? r : 0) * p.b_pitch + t * 16;
  }
  grid_launch_dependents();
  grid_dependency_wait();  // global memory is read only from here on
  int64_t start;
  bool bad = false;
  const int64_t len = mx_segment(p.offs, p.rows, e, start, &bad);
  if (bad && r0 == 0 && threadIdx.x == 0) atomicOr(p.error_word, kErrBadDims);
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  const uint8_t* wscale = p.sb + (e * p.nb + r0 / 128) * p.kb;  // 16 rows lie inside one 128-row block
  // Copies of this warp's i-th K block (warp + 8 i) into slot i % depth, as one group.
  const auto fetch = [&](int i) {
    const int kb = warp + i * kFewWarps;
    if (kb < kblocks) {
      const uint32_t slot = slots + (i % kFewDepth) * kFewBlock;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        // K is a multiple of 16: a 16-byte piece is inside the row or past its end.
        const int k = kb * 128 + c * 64;
        const bool in = k + t * 16 < depth;
#pragma unroll
        for (int h = 0; h < 2; ++h) copy16(slot + (2 * h + c) * 512, wrow[h] + (in ? k : 0), in && live[h]);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int64_t m0 = 0; m0 < len; m0 += 8) {
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint8_t* xrow = p.a + (start + m0 + g) * p.a_pitch + t * 16;  // token m0 + g
    const uint8_t* xscale = p.sa + (start + m0 + 2 * t) * p.kb;         // tokens m0 + 2t, 2t + 1
    const int left = static_cast<int>(len - m0 < 8 ? len - m0 : 8);
#pragma unroll
    for (int i = 0; i < kFewDepth; ++i) fetch(i);
#pragma unroll 1
    for (int b = 0; warp + b * kFewWarps < kblocks; ++b) {
      const int kb = warp + b * kFewWarps;
      // Tokens and scales first: they arrive while the weights are waited for.
      uint4 x[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int k = kb * 128 + c * 64;
        x[c] = g < left && k + t * 16 < depth ? *reinterpret_cast<const uint4*>(xrow + k) : zero;
      }
      const int sw = wscale[kb];
      int sx[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) sx[j] = 2 * t + j < left ? xscale[j * p.kb + kb] : 127;
      asm volatile("cp.async.wait_group %0;" ::"n"(kFewDepth - 1) : "memory");
      uint4 w[2][2];
      const uint32_t slot = slots + (b % kFewDepth) * kFewBlock;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4& v = w[i / 2][i % 2];
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(slot + i * 512)
                     : "memory");
      }
      float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        mma_e4m3(part, w[0][c].x, w[1][c].x, w[0][c].y, w[1][c].y, x[c].x, x[c].y);
        mma_e4m3(part, w[0][c].z, w[1][c].z, w[0][c].w, w[1][c].w, x[c].z, x[c].w);
      }
      // Columns 2t, 2t + 1 of the accumulator are tokens m0 + 2t, m0 + 2t + 1.
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // The scales' product in two equal steps: one alone may leave fp32's range.
        const int half = (sw + sx[j]) >> 1;  // 2^(sw - 127) 2^(sx - 127) = 2^(half - 127) 2^(sw + sx - half - 127)
        const float s1 = scale_value(sw == 255 || sx[j] == 255 ? 255 : half), s2 = scale_value(sw + sx[j] - half);
        acc[j] += part[j] * s1 * s2;
        acc[2 + j] += part[2 + j] * s1 * s2;
      }
      fetch(b + kFewDepth);  // into the slot just read
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      sums[warp][2 * t + j][g] = acc[j];
      sums[warp][2 * t + j][g + 8] = acc[2 + j];
    }
    __syncthreads();
    if (threadIdx.x < 128) {
      const int row = threadIdx.x & 15, tok = threadIdx.x >> 4;
      float s = 0.0f;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) s += sums[w][tok][row];
      const int64_t m = m0 + tok;
      if (m < len && r0 + row < p.n) p.c[(start + m) * p.c_pitch + r0 + row] = __float2bfloat16_rn(s);
    }
    __syncthreads();  // the sums are rewritten by the next tokens
  }
}

}  // namespace mgb
