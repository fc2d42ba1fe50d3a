// Grouped products of the gated feed-forward block and its backward pass,
// fp16 / bf16, tokens sorted by expert.
//
// A launch runs up to kFfnMaxJobs jobs of one epilogue kind over the same
// expert segments.  Segment e holds the rows [offs[e-1], offs[e]) of every
// token tensor.  A job is, per expert e,
//   rows  C[rows of e, N] = A[rows of e, K] op(B_e)     M = rows of e
//   wgrad C_e[M, N] = A[rows of e, M]^T B[rows of e, N]  contraction over rows of e
// with either operand K-major (contraction contiguous) or MN-major, chosen at
// run time: TMA loads it in the box its layout needs (K-major: 64 contraction
// x 128 outer; MN-major: 64 outer x 64 contraction, two boxes) and the MMA
// descriptors name the layout, so no operand is ever transposed in memory:
//   x W13, h W2          A K-major,  B MN-major
//   dy W2^T, dgu W13^T   A K-major,  B K-major
//   x^T dgu, h^T dy      A MN-major, B MN-major
// The last contraction block of a weight gradient's segment must not see the
// next expert's rows (a zero times their NaN would be NaN): its operands have a
// tensor map per expert whose rows end with the segment, so the tail reads
// zeros.  They are cut from the row ends on the device: in a backward pass by
// the launch before (a kernel less: 51 rows 30.9 -> 28.4 us a call), else by
// ffn_plan_kernel.  A rows job may load rows past its segment (they only reach accumulator rows that
// are not stored), so one map of the whole tensor serves, addressed by
// absolute rows, and one 3-D map of all experts' weights; groups of 32 rows
// that cross a segment's end are written by ordinary stores.
//
// Epilogues (fp32 accumulators, one rounding per stored value):
// h and the gradient of gate_up are operands of the next product, so 16-bit:
// y, dx and dW13 carry that rounding beside their own (bf16: 2.3e-3 from the
// formula in the Frobenius norm where one rounding alone is 1.7e-3).
//   plain            C
//   swiglu           gate | up tiles side by side in one accumulator; stores
//                    h = silu(g) u, g and u (the backward pass reads g, u)
//   swiglu backward  accumulator = dh; g, u arrive by TMA while the MMAs run;
//                    stores dg = dh u s (1 + g (1 - s)), du = dh g s, s = sigmoid(g)
//
// One CTA per SM, roles by warp: 0 TMA producer, 1 MMA issuer, 2-5 epilogue.
// G = 2: CTA pairs, 256 x 256 tiles (tcgen05 cta_group::2, M = 256, N = 256),
// or 256 x 512 (two of those MMAs on the same rows);
// G = 1: one CTA, 128 x 128 tiles, four times as many, where 256 x 256 tiles
// would leave too many SMs idle (the host estimates both).  Both load 128 rows of A and
// 128 columns of B per CTA and 64-deep contraction block (32 KB a stage).
// Split contraction (G = 1, p.split > 1; for launches whose row tiles would
// leave at least half of the SMs idle through a long contraction): the CTAs of
// a cluster first take the other jobs' tiles one by one, then share one tile
// of job 0: each sums a range of its contraction, leaves fp32 sums in its own
// (then idle) operand ring, and CTA r adds rows [128 r / split, ...) of all of
// them over distributed shared memory, in rank order, and applies the
// epilogue.
// Large launches: bf16 8192^3 runs at 1590 (wgrad) and 1600 TFLOP/s (dgrad)
// where the measured library product has 1618; 32 experts of 512 uneven rows,
// hidden 7168, ffn 2048: forward 1.42 to 1.53 ms, backward 2.95 to 3.09 ms, at
// 1.2 to 1.3 GHz under the 1 kW limit.  In launches alone (16 experts of 512
// rows, 4096 x 1536, 1.6 GHz) no unit is full: tensor pipe 50 to 66% busy, DRAM 37
// to 44%, and operands leave L2 at 11 to 13.5 TB/s, the gate and up launch's
// 256 x 256 tiles most.  Few rows are bound by the weights' bytes and by about
// 7 us per launch (setup 0.6, tile list 0.8, first operands 1.4, the join, the gap
// to the next): 16 rows, hidden 1024, ffn 704: 17.1 us for both products.
// Every wait is bounded; loads carry no multicast.
#pragma once

#include "mgb_tc_kernel.cuh"

namespace mgb {

constexpr int kFfnMaxJobs = 3;
constexpr int kFfnLaunches = 2;  // of one call
constexpr int kFfnWgrads = 2;    // weight gradient jobs of one call
static_assert(1 + kFfnWgrads <= kFfnMaxJobs, "templates of cut maps behind a one-job launch");
constexpr int kFfnMaps = 6;  // per job and expert: A, B, then the epilogue's
enum FfnEpilogue : int { kFfnPlain = 0, kFfnSwiglu = 1, kFfnSwigluBwd = 2 };

// One tensor of a job: rows follow the segments (token tensors) or the
// expert (weights, `expert_stride` elements apart).
struct FfnTensor {
  char* data;
  int64_t pitch;          // elements between rows
  int64_t expert_stride;  // weights: elements between experts
  int32_t token;          // 1: rows are token rows
};

struct FfnJob {
  FfnTensor t[kFfnMaps];
  int32_t wgrad;  // contraction over the segment's rows
  int32_t b_mn;   // rows: B is MN-major (wgrad: both operands are)
  int64_t m;      // wgrad: output rows
  int64_t n;      // output columns
  int64_t k;      // rows: contraction depth
  int64_t up;     // swiglu: column of B where the up half starts
  CUtensorMap* operands;  // wgrad: [experts][2] maps of A and B, cut on the device
};

struct FfnParams {
  FfnJob job[kFfnMaxJobs];
  int32_t jobs;
  int32_t experts;
  const int32_t* offs;  // [experts] row ends; nullptr: one segment of `rows`
  int64_t rows;
  const int32_t* tile_start;  // [jobs * experts + 1] first tile of every (job, expert); nullptr: built in shared memory
  int32_t split;        // CTAs of a cluster that share the contraction of job 0's tiles (one CTA tiles; 1: none)
  int32_t cuts;         // swiglu backward: weight gradients of the next launch whose operand maps this one cuts
  long long wait_budget;
  uint32_t* error_word;
  // 2-D of a token tensor, 3-D of weights; not of a wgrad job's operands.
  // Behind the scalars, which then share few lines of the constant cache.
  CUtensorMap map[kFfnMaxJobs][kFfnMaps];
};

// What the plan kernel prepares from the row ends: the operand maps of weight
// gradients, and the tile lists of launches with too many experts for shared
// memory.
struct FfnPlan {
  CUtensorMap map[kFfnWgrads][2];  // templates of one row
  FfnTensor t[kFfnWgrads][2];
  CUtensorMap* operands[kFfnWgrads];
  struct List {
    int32_t jobs, tile_rows, tile_cols;
    int32_t wgrad[kFfnMaxJobs];
    int64_t m[kFfnMaxJobs], n[kFfnMaxJobs];
    int32_t* tile_start;
  } list[kFfnLaunches];
  int32_t wgrads, lists, experts;
  const int32_t* offs;
  int64_t rows;
  uint32_t* error_word;
};

// Rows [start, start + len) of expert e, clamped into the tensor whatever offs holds.
__device__ __forceinline__ int64_t ffn_segment(const int32_t* offs, int64_t rows, int e, int64_t& start,
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

// A weight gradient's operand map for expert e: the template that the warp has
// copied to `staging` with its base moved to the segment and its rows ending
// there, published at `to`.
__device__ __forceinline__ void ffn_cut_map(CUtensorMap* staging, const FfnTensor& t, const int32_t* offs, int64_t rows,
                                            int e, CUtensorMap* to, int lane) {
  if (lane == 0) {
    int64_t start = 0;
    const int64_t len = ffn_segment(offs, rows, e, start);
    if (len > 0) {  // an empty segment's maps are never used
      tmap_replace_address(staging, t.data + start * t.pitch * 2);
      tmap_replace_dim(staging, 1, static_cast<uint32_t>(len));
    }
  }
  __syncwarp();
  tmap_publish(to, staging);
}

// A block per weight gradient and expert, a warp per operand (the parameters'
// constant-cache misses then overlap), then a block per tile list.
__global__ void __launch_bounds__(64) ffn_plan_kernel(const __grid_constant__ FfnPlan p) {
  __shared__ alignas(128) CUtensorMap staging[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_launch_dependents();
  if (static_cast<int>(blockIdx.x) >= p.wgrads * p.experts) {
    if (warp > 0) return;
    const FfnPlan::List& l = p.list[blockIdx.x - p.wgrads * p.experts];
    const int pairs = l.jobs * p.experts;
    const int per = (pairs + 31) / 32;
    const int lo = lane * per, hi = lo + per < pairs ? lo + per : pairs;
    grid_dependency_wait();  // offs and this scratch may be in use until here
    auto tiles_of = [&](int i) -> int64_t {
      const int job = i / p.experts;
      int64_t start;
      bool bad = false;
      const int64_t len = ffn_segment(p.offs, p.rows, i % p.experts, start, &bad);
      if (bad) atomicOr(p.error_word, kErrBadDims);
      return ceil_div64(l.wgrad[job] ? l.m[job] : len, l.tile_rows) * ceil_div64(l.n[job], l.tile_cols);
    };
    int64_t sum = 0;
    for (int i = lo; i < hi; ++i) sum += tiles_of(i);
    const int64_t incl = warp_scan(sum, lane);
    int64_t run = incl - sum;
    for (int i = lo; i < hi; ++i) {
      l.tile_start[i] = static_cast<int32_t>(run);
      run += tiles_of(i);
    }
    if (lane == 31) l.tile_start[pairs] = list_end(incl);
    return;
  }
  const int job = blockIdx.x / p.experts, e = blockIdx.x % p.experts;
  const FfnTensor t = p.t[job][warp];
  if (lane < 8) {
    reinterpret_cast<uint4*>(&staging[warp])[lane] = reinterpret_cast<const uint4*>(&p.map[job][warp])[lane];
  }
  __syncwarp();
  grid_dependency_wait();
  ffn_cut_map(&staging[warp], t, p.offs, p.rows, e, p.operands[job] + 2 * e + warp, lane);
}

// Words of shared memory for the launch's tile list and row ends, if they fit:
// a role then finds a tile without a chain of global loads.
constexpr int kListWords = 400;

// Clock cycles that a 64-deep contraction block adds to the bounded wait for
// its accumulator (it takes about 600).
constexpr long long kBlockCycles = 4096;

// A role's position in the tile list (`ts` and `offs` in shared or global
// memory) of ROWS x COLS output tiles.
template <int ROWS, int COLS>
struct FfnWalk {
  const FfnParams& p;
  const int32_t* ts;
  const int32_t* offs;
  int pair = -1;  // job * experts + e
  int32_t first = 0, end = 0;
  int64_t start = 0, len = 0;  // rows of the expert's segment
  int64_t rows = 0;    // output rows
  int32_t m_blocks = 1, n_blocks = 1;
  int64_t kblocks = 0;
  const FfnJob* job = nullptr;
  const CUtensorMap* maps = nullptr;  // the job's
  int expert = 0;

  __device__ __forceinline__ FfnWalk(const FfnParams& params, const int32_t* list, const int32_t* ends)
      : p(params), ts(list), offs(ends) {}

  // Moves to the (job, expert) of tile t.
  __device__ __forceinline__ void seek(int32_t t) {
    if (pair >= 0 && t >= first && t < end) return;
    // The last pair whose first tile is <= t owns it (empty pairs share their successor's).
    int lo = pair >= 0 && t >= end ? pair : 0, hi = p.jobs * p.experts - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (ts[mid] <= t) {
        lo = mid;
      } else {
        hi = mid - 1;
      }
    }
    pair = lo;
    first = ts[lo];
    end = ts[lo + 1];
    job = &p.job[lo / p.experts];
    maps = p.map[lo / p.experts];
    expert = lo % p.experts;
    len = ffn_segment(offs, p.rows, expert, start);
    rows = job->wgrad ? job->m : len;
    m_blocks = static_cast<int32_t>(ceil_div64(rows, ROWS));
    n_blocks = static_cast<int32_t>(ceil_div64(job->n, COLS));
    kblocks = ceil_div64(job->wgrad ? len : job->k, 64);
  }
  // Bands of 8 row blocks, row block fastest inside a band (as TileWalk).
  __device__ __forceinline__ void blocks(int32_t t, int64_t& mb, int64_t& nb) const {
    const uint32_t local = t - first;
    const uint32_t band_tiles = 8u * n_blocks;
    const uint32_t band = local / band_tiles;
    const uint32_t in = local - band * band_tiles;
    const uint32_t rows_in = m_blocks - band * 8 < 8 ? m_blocks - band * 8 : 8;
    const uint32_t column = in / rows_in;
    mb = band * 8 + (in - column * rows_in);
    nb = column;
  }
};

// The tiles a CTA (or pair) works on, in order: `first`, `first + step`, ...
// below `end`, then with a split the cluster's tile of job 0 (`shared`, -1:
// none), of which it takes contraction blocks [kb_from, kb_to).
struct FfnItems {
  int32_t next, step, end, shared;
  int share, split;
  bool last = false;  // the current item is the shared one
  int32_t kb_from = 0, kb_to = 0;

  template <class Walk>
  __device__ __forceinline__ FfnItems(const Walk& walk, int group) {
    const FfnParams& p = walk.p;
    split = p.split;
    end = walk.ts[p.jobs * p.experts];
    next = blockIdx.x / group;
    step = gridDim.x / group;
    shared = -1;
    share = 0;
    if (split > 1) {
      const int32_t mine = walk.ts[p.experts];  // tiles of job 0
      next += mine;
      share = static_cast<int>(cluster_ctarank());
      const int32_t c = blockIdx.x / split;
      if (c < mine && end > 0) shared = c;
    }
  }
  template <class Walk>
  __device__ __forceinline__ bool advance(Walk& walk, int32_t& t) {
    if (next < end) {
      t = next;
      next += step;
      walk.seek(t);
      kb_from = 0;
      kb_to = static_cast<int32_t>(walk.kblocks);
      return true;
    }
    if (last || shared < 0) return false;
    last = true;
    t = shared;
    walk.seek(t);
    const int32_t per = blocks_each(walk);
    kb_from = share * per;
    const int32_t all = static_cast<int32_t>(walk.kblocks);
    kb_to = kb_from + per < all ? kb_from + per : all;
    return true;
  }
  template <class Walk>
  __device__ __forceinline__ int32_t blocks_each(const Walk& walk) const {
    return static_cast<int32_t>((walk.kblocks + split - 1) / split);
  }
};

// NH = 256-column halves of a pair's tile: 2 is the 256 x 512 tile of the
// plain epilogue.  It moves 48 KB into a CTA per 128 x 512 x 64 products
// where the 256 x 256 tile moves 32 KB per 128 x 256 x 64, a quarter less per
// product; its one 512-column accumulator fills TMEM and is freed by halves.
template <typename T, int EPI, int G, int NH = 1>
struct FfnCfg {
  static_assert(sizeof(T) == 2 && (G == 1 || G == 2), "16-bit types, one CTA or a pair");
  static_assert(NH == 1 || (NH == 2 && G == 2 && EPI == kFfnPlain), "wide tiles: pairs, plain epilogue");
  static constexpr int kBK = 64;
  static constexpr int kOperand = 128 * 128;  // 128 rows (or columns) x 64 contraction
  static constexpr int kStageBytes = (1 + NH) * kOperand;
  static constexpr int kTileM = 128 * G;
  static constexpr int kMmaN = 128 * G;
  static constexpr int kAccCols = NH * kMmaN;
  static constexpr int kTileOut = EPI == kFfnSwiglu ? kAccCols / 2 : kAccCols;  // output columns per tile
  static constexpr int kTmemCols = NH == 2 ? 512 : 2 * kAccCols;                // two accumulators, or two halves
  // Staging blocks (32 rows x 128 bytes) per epilogue warp: plain two, in
  // turn; swiglu h, g and u of one chunk; backward two pairs (g, u), each
  // overwritten in place by (dg, du).
  static constexpr int kEpiBlocks = EPI == kFfnPlain ? 2 : EPI == kFfnSwiglu ? 3 : 4;
  static constexpr int kEpiBytes = 4 * kEpiBlocks * kEpiWarpBytes;
  static constexpr int kStages = (kTcSmemBudget - kEpiBytes) / kStageBytes;
  static constexpr int kSmemBytes = kStages * kStageBytes + kEpiBytes + 2048 + 1024;
  static_assert((2 * kStages + 13) * 8 + 12 + kListWords * 4 <= 2048, "barriers and the tile list");
  static constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  static_assert(kStages >= 4 && kSmemBytes <= 232448, "shared memory");
  // Split contraction: a row of partial sums, padded against bank conflicts.
  static constexpr int kSumRow = kAccCols * 4 + 16;
  static_assert(G == 2 || kTileM * kSumRow <= kStages * kStageBytes, "partial sums fit the ring");
  using Walk = FfnWalk<kTileM, kTileOut>;
};

// 32 rows of a tile as one warp stores them: staged in shared memory and by
// tensor stores at absolute coordinates; or, where the segment ends inside
// (`ragged`), each lane its own row straight from registers (no staging: the
// fence between the staging writes and the tensor store also waits for
// ordinary stores in flight, a microsecond a chunk).
struct RowGroup {
  const CUtensorMap* maps;
  int64_t start, len;  // the segment
  int32_t row0;        // first row, inside the segment
  int32_t z;           // weights: expert
  bool ragged, weights;

  template <class Walk>
  __device__ __forceinline__ RowGroup(const Walk& walk, int32_t row) {
    maps = walk.maps;
    weights = walk.job->wgrad != 0;
    start = weights ? 0 : walk.start;
    len = walk.rows;
    row0 = row;
    z = walk.expert;
    ragged = !weights && row + 32 > len;
  }
  __device__ __forceinline__ bool empty() const { return row0 >= len; }
  // Lane 0: the staged block of columns from x to tensor i.
  __device__ __forceinline__ void put(int i, const uint8_t* block, int32_t x, uint64_t policy) const {
    if (weights) {
      tma_store_3d(&maps[i], block, x, row0, z, policy);
    } else {
      tma_store_2d(&maps[i], block, x, static_cast<int32_t>(start + row0), policy);
    }
  }
  // Every lane: 32 columns from x of its row of tensor t (ragged groups).
  template <typename T>
  __device__ __forceinline__ void put_row(const FfnTensor& t, const uint32_t (&v)[32], int64_t x, int64_t cols,
                                          int lane) const {
    if (row0 + lane >= len) return;
    uint4* to = reinterpret_cast<uint4*>(t.data + ((start + row0 + lane) * t.pitch + x) * 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (x + 8 * i < cols) {  // columns are multiples of 8
        to[i] = make_uint4(pack_pair<T>(v[8 * i], v[8 * i + 1]), pack_pair<T>(v[8 * i + 2], v[8 * i + 3]),
                           pack_pair<T>(v[8 * i + 4], v[8 * i + 5]), pack_pair<T>(v[8 * i + 6], v[8 * i + 7]));
      }
    }
  }
};

// Plain epilogue of one warp: TN columns from TMEM in 32-column units, the
// next unit's load in flight while one is converted and staged; 64-column
// chunks leave through two staging blocks in turn.
template <typename T, int TN>
__device__ __forceinline__ void ffn_store_plain(const FfnJob& j, const RowGroup& rows, uint32_t taddr, int32_t n0,
                                                uint8_t* blocks, int lane, uint32_t& seq, uint64_t policy) {
  // No TMEM load may be issued for nothing: only the loop below waits for one.
  if (rows.empty() || n0 >= j.n) return;
  const int64_t left = j.n - n0;
  const int units = 2 * (left >= TN ? TN / 64 : static_cast<int>((left + 63) / 64));
  if (rows.ragged) {
#pragma unroll 1
    for (int g = 0; g < units; ++g) {
      uint32_t v[32];
      tmem_ld32(taddr + g * 32, v);
      tmem_ld_wait();
      rows.put_row<T>(j.t[2], v, n0 + g * 32, j.n, lane);
    }
    return;
  }
  uint32_t v[2][32];
  tmem_ld32(taddr, v[0]);
#pragma unroll
  for (int g = 0; g < TN / 32; ++g) {
    if (g >= units) break;
    uint8_t* block = blocks + (seq & 1) * kEpiWarpBytes;
    if (g % 2 == 0) {
      if (lane == 0) bulk_wait_group_read<1>();  // the store last issued from this block has read it
      __syncwarp();
    }
    tmem_ld_wait();
    if (g + 1 < units) tmem_ld32(taddr + (g + 1) * 32, v[(g + 1) & 1]);
    write_unit_smem<T>(v[g & 1], block, lane, g % 2);
    if (g % 2 == 1) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        rows.put(2, block, n0 + (g / 2) * 64, policy);
        bulk_commit_group();
      }
      ++seq;
    }
  }
}

// sigmoid(g) and 1 - sigmoid(g) from e = exp(-|g|), which never overflows: with
// exp(-g) the divisor passes 2^126 from g = -87.3 on, where the fast divide
// returns 0, although sigmoid(g) times a large u or dh is still a number.  Fast
// exponential and divide: a few ulp in fp32, far below the 16-bit rounding of
// what is stored.
__device__ __forceinline__ float2 sigmoids(float g) {
  const float e = __expf(-fabsf(g));
  const float near = __fdividef(1.0f, 1.0f + e), far = e * near;
  return g < 0.0f ? make_float2(far, near) : make_float2(near, far);
}

__device__ __forceinline__ float swiglu(float g, float u) { return g * sigmoids(g).x * u; }

// Gradients of h = silu(g) u.  u and g meet the sigmoid first and dh then, so
// that no step leaves fp32's range where the result does not: dh g alone may at a
// gate of the type's lowest value (and infinity times its sigmoid 0 is NaN), u
// times silu'(g), which reaches 1.1, at the largest u.
__device__ __forceinline__ void swiglu_grad(float dh, float g, float u, float& dg, float& du) {
  const float2 s = sigmoids(g);
  du = dh * (g * s.x);
  dg = dh * (u * s.x) * (1.0f + g * s.y);
}

// Swiglu epilogue of one warp: gate columns [0, TO), up columns [TO, 2 TO) of
// the accumulator; h from the fp32 values, g and u rounded once as stored.
template <typename T, int TO>
__device__ __forceinline__ void ffn_store_swiglu(const FfnJob& j, const RowGroup& rows, uint32_t taddr, int32_t o0,
                                                 uint8_t* blocks, int lane, uint64_t policy) {
  if (rows.empty() || o0 >= j.n) return;
  const int64_t left = j.n - o0;
  const int chunks = left >= TO ? TO / 64 : static_cast<int>((left + 63) / 64);
#pragma unroll 1
  for (int c = 0; c < chunks; ++c) {
    if (!rows.ragged) {
      if (lane == 0) bulk_wait_group_read<0>();  // the previous chunk's stores have read the blocks
      __syncwarp();
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t gate[32], up[32];
      tmem_ld32(taddr + c * 64 + u * 32, gate);
      tmem_ld32(taddr + TO + c * 64 + u * 32, up);
      tmem_ld_wait();
      const int64_t x = o0 + c * 64 + u * 32;
      if (rows.ragged) {
        rows.put_row<T>(j.t[3], gate, x, j.n, lane);
        rows.put_row<T>(j.t[4], up, x, j.n, lane);
      } else {
        write_unit_smem<T>(gate, blocks + kEpiWarpBytes, lane, u);
        write_unit_smem<T>(up, blocks + 2 * kEpiWarpBytes, lane, u);
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        gate[i] = __float_as_uint(swiglu(__uint_as_float(gate[i]), __uint_as_float(up[i])));
      }
      if (rows.ragged) {
        rows.put_row<T>(j.t[2], gate, x, j.n, lane);
      } else {
        write_unit_smem<T>(gate, blocks, lane, u);
      }
    }
    if (!rows.ragged) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
#pragma unroll
        for (int i = 0; i < 3; ++i) rows.put(2 + i, blocks + i * kEpiWarpBytes, o0 + c * 64, policy);
        bulk_commit_group();
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ float2 unpack_pair(uint32_t v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
}

// One warp's state of the swiglu backward epilogue: two pairs of blocks, each
// with an mbarrier its loads land on.
struct FfnGateLoads {
  uint8_t* blocks;
  uint64_t* bars;  // two
  uint32_t issued = 0, used = 0;

  // Lane 0: loads the (g, u) chunk at (x, y) into the next pair, once the
  // stores issued from it have read it.
  __device__ __forceinline__ void issue(const CUtensorMap* maps, int32_t x, int32_t y) {
    const int set = issued & 1;
    bulk_wait_group_read<0>();
    mbar_arrive_expect_tx(&bars[set], 2 * kEpiWarpBytes);
    const uint64_t pol = policy_evict_first();
    tma_load_2d(&maps[4], &bars[set], blocks + set * 2 * kEpiWarpBytes, x, y, pol);
    tma_load_2d(&maps[5], &bars[set], blocks + set * 2 * kEpiWarpBytes + kEpiWarpBytes, x, y, pol);
  }
};

// Calls f(a_mn, b_mn) with the job's operand layouts as compile-time
// constants, so that the loops per contraction block hold no layout branch.
template <int EPI, class F>
__device__ __forceinline__ void by_layout(const FfnJob& j, F&& f) {
  using No = std::integral_constant<bool, false>;
  using Yes = std::integral_constant<bool, true>;
  if constexpr (EPI == kFfnSwiglu) {
    f(No{}, Yes{});
  } else if constexpr (EPI == kFfnSwigluBwd) {
    f(No{}, No{});
  } else if (j.wgrad) {
    f(Yes{}, Yes{});
  } else if (j.b_mn) {
    f(No{}, Yes{});
  } else {
    f(No{}, No{});
  }
}

// Four consecutive 16-bit values (columns are multiples of 8: all inside a row or past it).
template <typename T>
__device__ __forceinline__ void store4(const FfnTensor& t, int64_t row, int64_t col, float a, float b, float c, float d) {
  uint2 v;
  v.x = pack_pair<T>(__float_as_uint(a), __float_as_uint(b));
  v.y = pack_pair<T>(__float_as_uint(c), __float_as_uint(d));
  *reinterpret_cast<uint2*>(t.data + (row * t.pitch + col) * 2) = v;
}
template <typename T>
__device__ __forceinline__ float4 load4(const FfnTensor& t, int64_t row, int64_t col) {
  const uint2 v = *reinterpret_cast<const uint2*>(t.data + (row * t.pitch + col) * 2);
  const float2 a = unpack_pair<T>(v.x), b = unpack_pair<T>(v.y);
  return make_float4(a.x, a.y, b.x, b.y);
}

// This CTA's rows of a split tile: the `parts` partial sums in rank order,
// then the epilogue; a warp per row, a lane per four accumulator columns.
template <typename T, int EPI, class Cfg>
__device__ __forceinline__ void ffn_join(const FfnParams& p, const typename Cfg::Walk& walk, const FfnItems& items, int parts,
                                         uint32_t ring, int warp, int lane) {
  const FfnJob& j = *walk.job;
  int64_t mb, nb;
  walk.blocks(items.shared, mb, nb);
  const int rows = Cfg::kTileM / items.split;
  for (int r = items.share * rows + warp; r < (items.share + 1) * rows; r += kTcThreads / 32) {
    const int64_t m = mb * Cfg::kTileM + r;
    if (m >= walk.rows) break;
    const float4 s = join_parts(ring + r * Cfg::kSumRow + lane * 16, parts);
    const int64_t row = walk.start + m;
    if constexpr (EPI == kFfnSwiglu) {
      // Lanes 0-15 hold gate columns, lane l + 16 the up columns of lane l's.
      const float4 u = make_float4(__shfl_down_sync(0xffffffffu, s.x, 16), __shfl_down_sync(0xffffffffu, s.y, 16),
                                   __shfl_down_sync(0xffffffffu, s.z, 16), __shfl_down_sync(0xffffffffu, s.w, 16));
      const int64_t col = nb * Cfg::kTileOut + (lane & 15) * 4;
      if (col < j.n) {
        store4<T>(j.t[lane < 16 ? 3 : 4], row, col, s.x, s.y, s.z, s.w);
        if (lane < 16) {
          store4<T>(j.t[2], row, col, swiglu(s.x, u.x), swiglu(s.y, u.y), swiglu(s.z, u.z), swiglu(s.w, u.w));
        }
      }
    } else {
      const int64_t col = nb * Cfg::kTileOut + lane * 4;
      if (col < j.n) {
        if constexpr (EPI == kFfnPlain) {
          store4<T>(j.t[2], row, col, s.x, s.y, s.z, s.w);
        } else {
          const float4 g = load4<T>(j.t[4], row, col), u = load4<T>(j.t[5], row, col);
          float4 dg, du;
          swiglu_grad(s.x, g.x, u.x, dg.x, du.x);
          swiglu_grad(s.y, g.y, u.y, dg.y, du.y);
          swiglu_grad(s.z, g.z, u.z, dg.z, du.z);
          swiglu_grad(s.w, g.w, u.w, dg.w, du.w);
          store4<T>(j.t[2], row, col, dg.x, dg.y, dg.z, dg.w);
          store4<T>(j.t[3], row, col, du.x, du.y, du.z, du.w);
        }
      }
    }
  }
}

template <typename T, int EPI, int G, int NH>
__global__ void __launch_bounds__(kTcThreads, 1) ffn_kernel(const __grid_constant__ FfnParams p) {
  using Cfg = FfnCfg<T, EPI, G, NH>;
  constexpr int S = Cfg::kStages;
  constexpr int BK = Cfg::kBK;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem;
  uint8_t* epi_stage = smem + S * Cfg::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(epi_stage + Cfg::kEpiBytes);
  uint64_t* empty = full + S;
  uint64_t* acc_full = empty + S;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* drain_bar = acc_empty + 2;
  uint64_t* gate_bars = drain_bar + 1;  // two per epilogue warp
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gate_bars + 8);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* never = abort + 1;
  int32_t* list = reinterpret_cast<int32_t*>(tmem_slot + 3);  // kListWords

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = G == 2 ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  // The next kernel may set up as SMs come free; it waits for this one's end.
  grid_launch_dependents();
  if (warp == 2) {  // the parameters' maps, while the kernel before may still run
    const int job = lane / kFfnMaps, i = lane % kFfnMaps;
    if (job < p.jobs && (i >= 2 || !p.job[job].wgrad) && p.job[job].t[i].data != nullptr) prefetch_tmap(&p.map[job][i]);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4 * G);
    }
    mbar_init(drain_bar, 1);
    for (int i = 0; i < 8; ++i) mbar_init(&gate_bars[i], 1);
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
  if constexpr (G == 2) cluster_sync();  // the peer's barriers exist before anything lands on them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const long long budget = p.wait_budget;
  grid_dependency_wait();  // global memory is read only from here on
  const int32_t* ts = p.tile_start;
  const int32_t* offs = p.offs;
  if (ts == nullptr) {
    // The tile list: first tiles of every (job, expert), then the row ends.
    const int pairs = p.jobs * p.experts;
    int32_t* ends = list + pairs + 1;
    for (int i = threadIdx.x; i < p.experts; i += kTcThreads) {
      ends[i] = p.offs != nullptr ? p.offs[i] : static_cast<int32_t>(p.rows);
    }
    __syncthreads();
    if (warp == 0) {
      int64_t before = 0;
      for (int base = 0; base < pairs; base += 32) {
        const int i = base + lane;
        int64_t tiles = 0;
        if (i < pairs) {
          const FfnJob& j = p.job[i / p.experts];
          int64_t start;
          bool bad = false;
          const int64_t len = ffn_segment(ends, p.rows, i % p.experts, start, &bad);
          if (bad && blockIdx.x == 0) atomicOr(p.error_word, kErrBadDims);
          tiles = ceil_div64(j.wgrad ? j.m : len, Cfg::kTileM) * ceil_div64(j.n, Cfg::kTileOut);
        }
        const int64_t incl = warp_scan(tiles, lane);
        if (i < pairs) list[i] = static_cast<int32_t>(before + incl - tiles);
        before += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) list[pairs] = list_end(before);
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
      const uint64_t pol_keep = policy_evict_last();
      const uint64_t pol_shared = policy_evict_normal();
      const uint64_t pol_stream = policy_evict_first();
      const uint32_t ring0 = smem_u32(ring), full0 = smem_u32(full), empty0 = smem_u32(empty);
      const uint32_t lead0 = G == 2 ? mapa_shared(full0, 0) : full0;  // the leader's barriers
      typename Cfg::Walk walk(p, ts, offs);
      FfnItems items(walk, G);
      int s = 0;
      uint32_t phase = 0, loaded = 0;
      int built = -1;
      bool ok = true;
      for (int32_t t; ok && items.advance(walk, t);) {
        const FfnJob& j = *walk.job;
        int64_t mb, nb;
        walk.blocks(t, mb, nb);
        const CUtensorMap* own = nullptr;  // wgrad: the expert's operand maps
        if (EPI == kFfnPlain && j.wgrad) {
          own = j.operands + 2 * walk.expert;
          if (walk.pair != built && walk.kblocks > 0) {
            tmap_acquire(&own[0]);
            tmap_acquire(&own[1]);
            built = walk.pair;
          }
        }
        const int32_t m0 = static_cast<int32_t>(mb * Cfg::kTileM + rank * 128);
        // Rows job: absolute row.  A pair's upper half that lies past the segment
        // reads zeros from past the tensor (no traffic, and quieter MMAs).
        const int32_t y0 = static_cast<int32_t>(m0 < walk.rows ? walk.start + m0 : p.rows);
        // First B column of this CTA's two 64-column boxes (swiglu: gate and up
        // columns of the same outputs; a pair's CTA 0 holds gate, CTA 1 up).
        int32_t b0, b1;
        if constexpr (EPI == kFfnSwiglu) {
          const int32_t o = static_cast<int32_t>(nb * Cfg::kTileOut);
          if constexpr (G == 2) {
            b0 = o + (rank ? static_cast<int32_t>(j.up) : 0);
            b1 = b0 + 64;
          } else {
            b0 = o;
            b1 = o + static_cast<int32_t>(j.up);
          }
        } else {
          b0 = static_cast<int32_t>(nb * Cfg::kAccCols + rank * 128);
          b1 = b0 + 64;
        }
        // Weights that one row block reads are streamed; shared operands keep
        // normal priority; activations of a rows job are kept for the other
        // column blocks.
        const uint64_t pol_a = j.wgrad ? pol_shared : pol_keep;
        const uint64_t pol_b = !j.wgrad && walk.m_blocks == 1 ? pol_stream : pol_shared;
        const int32_t begin = items.kb_from * BK, end = items.kb_to * BK;
        const auto load = [&](const CUtensorMap* map, uint32_t dst, int32_t x, int32_t y, uint64_t pol) {
          tile_load<G>(map, lead0 + s * 8, dst, x, y, pol);
        };
        const auto load_weight = [&](uint32_t dst, int32_t x, int32_t y) {
          tile_load_3d<G>(&walk.maps[1], lead0 + s * 8, dst, x, y, walk.expert, pol_b);
        };
        const auto run = [&](auto a_mn, auto b_mn) {
          for (int32_t kx = begin; kx < end; kx += BK) {
            if (!bar_wait(empty0 + s * 8, phase ^ 1u, budget, abort)) {
              fail(kErrWaitEmpty);
              ok = false;
              break;
            }
            const uint32_t st_a = ring0 + s * Cfg::kStageBytes, st_b = st_a + Cfg::kOperand;
            if (leader) mbar_arrive_expect_tx(&full[s], G * Cfg::kStageBytes);
            if constexpr (a_mn.value) {
              load(&own[0], st_a, m0, kx, pol_a);
              load(&own[0], st_a + Cfg::kOperand / 2, m0 + 64, kx, pol_a);
            } else {
              load(&walk.maps[0], st_a, kx, y0, pol_a);
            }
#pragma unroll
            for (int h = 0; h < NH; ++h) {
              const uint32_t dst = st_b + h * Cfg::kOperand;
              if constexpr (a_mn.value) {
                load(&own[1], dst, b0 + 256 * h, kx, pol_b);
                load(&own[1], dst + Cfg::kOperand / 2, b1 + 256 * h, kx, pol_b);
              } else if constexpr (b_mn.value) {
                load_weight(dst, b0 + 256 * h, kx);
                load_weight(dst + Cfg::kOperand / 2, b1 + 256 * h, kx);
              } else {
                load_weight(dst, kx, b0 + 256 * h);
              }
            }
            ++loaded;
            if (++s == S) {
              s = 0;
              phase ^= 1u;
            }
          }
        };
        by_layout<EPI>(j, run);
      }
      if (*abort && leader) {  // loads in flight land before the CTA's memory goes away
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
      FfnItems items(walk, G);
      int s = 0;
      uint32_t phase = 0, acc_it = 0;
      bool ok = true;
      for (int32_t t; ok && items.advance(walk, t);) {
        if (items.kb_to <= items.kb_from) continue;
        // Two accumulators in turn, or (wide) the halves of one.
        const int buf = NH == 2 ? 0 : static_cast<int>(acc_it & 1);
        const uint32_t acc_phase = ((NH == 2 ? acc_it : acc_it >> 1) & 1u) ^ 1u;
        if (!mbar_wait(&acc_empty[buf], acc_phase, budget, abort)) {
          fail(kErrWaitAccEmpty);
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem_base + buf * Cfg::kAccCols;
        const int32_t kblocks = items.kb_to - items.kb_from;
        const auto run = [&](auto a_mn, auto b_mn) {
          // K-major: a k-step of 16 is 32 bytes along the swizzled row.
          // MN-major: 16 contraction rows of 128 bytes; the second 64 columns
          // one box (8 KB) on.
          constexpr uint32_t kStepA = a_mn.value ? 16 * 128 / 16 : 32 / 16, kStepB = b_mn.value ? 16 * 128 / 16 : 32 / 16;
          constexpr uint32_t kIdesc = instr_desc(Cfg::kFmt, a_mn.value, b_mn.value, Cfg::kTileM, Cfg::kMmaN);
          const uint64_t a_desc = smem_desc(smem_u32(ring), a_mn.value ? Cfg::kOperand / 2 : 16, 1024, kLayoutSw128);
          const uint64_t b_desc =
              smem_desc(smem_u32(ring) + Cfg::kOperand, b_mn.value ? Cfg::kOperand / 2 : 16, 1024, kLayoutSw128);
          // The four MMAs of half h on stage `at`.
          const auto issue = [&](int at, int h, bool first) {
            const uint32_t stage = static_cast<uint32_t>(at) * (Cfg::kStageBytes >> 4);
            const uint64_t ad = a_desc + stage, bd = b_desc + stage + h * (Cfg::kOperand >> 4);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
              const uint32_t acc = ks > 0 || !first ? 1u : 0u;
              if constexpr (G == 2) {
                mma_f16_pair(d + h * Cfg::kMmaN, ad + ks * kStepA, bd + ks * kStepB, kIdesc, acc);
              } else {
                mma_f16(d + h * Cfg::kMmaN, ad + ks * kStepA, bd + ks * kStepB, kIdesc, acc);
              }
            }
          };
          int32_t kb = 0;
          if constexpr (NH == 2) {
            // Half 0 is free: its MMAs of the first k-blocks (up to a ring of
            // them, their stages kept) run while the epilogue drains half 1.
            const int32_t held = kblocks < S ? kblocks : S;
            int at = s;
            uint32_t at_phase = phase;
            for (; kb < held; ++kb) {
              if (!bar_wait(full0 + at * 8, at_phase, budget, abort)) {
                fail(kErrWaitFull);
                ok = false;
                return;
              }
              tc_fence_after();
              issue(at, 0, kb == 0);
              if (++at == S) {
                at = 0;
                at_phase ^= 1u;
              }
            }
            if (!mbar_wait(&acc_empty[1], acc_phase, budget, abort)) {
              fail(kErrWaitAccEmpty);
              ok = false;
              return;
            }
            tc_fence_after();
            for (kb = 0; kb < held; ++kb) {
              issue(s, 1, kb == 0);
              tile_commit<G>(empty0 + s * 8);
              if (++s == S) {
                s = 0;
                phase ^= 1u;
              }
            }
          }
          for (; kb < kblocks; ++kb) {
            if (!bar_wait(full0 + s * 8, phase, budget, abort)) {
              fail(kErrWaitFull);
              ok = false;
              return;
            }
            tc_fence_after();
#pragma unroll
            for (int h = 0; h < NH; ++h) issue(s, h, kb == 0);
            tile_commit<G>(empty0 + s * 8);
            if (++s == S) {
              s = 0;
              phase ^= 1u;
            }
          }
        };
        by_layout<EPI>(*walk.job, run);
        if (!ok) break;
        tile_commit<G>(smem_u32(&acc_full[buf]));
        ++acc_it;
      }
      if (*abort) {
        if constexpr (G == 2) {
          mma_commit_pair(drain_bar, 0x1);
        } else {
          mma_commit(drain_bar);
        }
        if (!mbar_wait(drain_bar, 0, budget, never)) atomicOr(p.error_word, kErrWaitTeardown);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3;
    uint8_t* blocks = epi_stage + quarter * Cfg::kEpiBlocks * kEpiWarpBytes;
    const uint64_t pol_out = policy_evict_normal();
    FfnGateLoads gates{blocks, gate_bars + 2 * quarter};
    if constexpr (EPI == kFfnSwigluBwd) {
      if (p.cuts > 0) {
        // The next launch's operand maps, under this one's first MMAs: a warp
        // per map, templates and tensors in the job slots behind its own.
        CUtensorMap* staging = reinterpret_cast<CUtensorMap*>(blocks);
        for (int i = blockIdx.x * 4 + quarter; i < p.cuts * 2 * p.experts; i += gridDim.x * 4) {
          const int slot = 1 + i / (2 * p.experts), e = i / 2 % p.experts, o = i & 1;
          if (lane < 8) {
            reinterpret_cast<uint4*>(staging)[lane] = reinterpret_cast<const uint4*>(&p.map[slot][o])[lane];
          }
          __syncwarp();
          ffn_cut_map(staging, p.job[slot].t[o], offs, p.rows, e, p.job[slot].operands + 2 * e + o, lane);
          __syncwarp();  // the staged map has been copied before the next one
        }
        fence_proxy_async_smem();  // the staging is written by tensor loads next
        __syncwarp();
      }
    }
    typename Cfg::Walk walk(p, ts, offs);
    FfnItems items(walk, G);
    uint32_t acc_it = 0, chunk_seq = 0;
    // An accumulator is waited for through its whole contraction, every block of
    // which the other roles may wait for: 2^31 rows are seconds.
    const auto whole_budget = [&] { return budget + (items.kb_to - items.kb_from) * kBlockCycles; };
    for (int32_t t; items.advance(walk, t);) {
      const FfnJob& j = *walk.job;
      int64_t mb, nb;
      walk.blocks(t, mb, nb);
      const int32_t row0 = static_cast<int32_t>(mb * Cfg::kTileM + rank * 128 + quarter * 32);
      const int32_t n0 = static_cast<int32_t>(nb * Cfg::kTileOut);
      if (items.last) {
        if (items.kb_to <= items.kb_from) break;  // a short last share has no blocks and leaves no sums
        if (!mbar_wait_warp(&acc_full[acc_it & 1], (acc_it >> 1) & 1u, whole_budget(), abort)) {
          if (lane == 0) fail(kErrWaitAccFull);
          break;
        }
        tc_fence_after();
        // The last MMAs are done and nothing more is loaded: the ring holds the sums.
        const uint32_t from = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + (acc_it & 1) * Cfg::kAccCols;
        uint8_t* sums = ring + (quarter * 32 + lane) * Cfg::kSumRow;
#pragma unroll 1
        for (int c = 0; c < Cfg::kAccCols; c += 32) {
          uint32_t v[32];
          tmem_ld32(from + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            reinterpret_cast<uint4*>(sums + c * 4)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          }
        }
        break;  // the last item
      }
      if (walk.kblocks <= 0) {
        // An expert without rows: its weight gradient is zero.
        const FfnTensor& c = j.t[2];
        T* out = reinterpret_cast<T*>(c.data) + walk.expert * c.expert_stride;
        for (int r = 0; r < 32 && row0 + r < walk.rows; ++r) {
          for (int64_t col = n0 + lane * 8; col < j.n && col < n0 + Cfg::kTileOut; col += 256) {
            T* dst = out + (row0 + r) * c.pitch + col;  // n is a multiple of 8: whole 16-byte pieces
            *reinterpret_cast<uint4*>(dst) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        continue;
      }
      const RowGroup rows(walk, row0);
      const int32_t y0 = static_cast<int32_t>(rows.start) + row0;
      int chunks = 0;
      if constexpr (EPI == kFfnSwigluBwd) {
        if (!rows.empty()) {
          const int64_t left = j.n - n0;
          chunks = left >= Cfg::kTileOut ? Cfg::kTileOut / 64 : static_cast<int>((left + 63) / 64);
          if (lane == 0) gates.issue(walk.maps, n0, y0);  // the first chunk arrives while the MMAs run
          ++gates.issued;
        }
      }
      const int buf = NH == 2 ? 0 : static_cast<int>(acc_it & 1);
      if (!mbar_wait_warp(&acc_full[buf], (NH == 2 ? acc_it : acc_it >> 1) & 1u, whole_budget(), abort)) {
        if (lane == 0) fail(kErrWaitAccFull);
        break;
      }
      tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * Cfg::kAccCols;
      if constexpr (NH == 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // each half is released as soon as it is drained
          ffn_store_plain<T, 256>(j, rows, taddr + h * 256, n0 + h * 256, blocks, lane, chunk_seq, pol_out);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(&acc_empty[h]), 0));
        }
        ++acc_it;
        continue;
      } else if constexpr (EPI == kFfnPlain) {
        ffn_store_plain<T, Cfg::kTileOut>(j, rows, taddr, n0, blocks, lane, chunk_seq, pol_out);
      } else if constexpr (EPI == kFfnSwiglu) {
        ffn_store_swiglu<T, Cfg::kTileOut>(j, rows, taddr, n0, blocks, lane, pol_out);
      } else {
        bool lost = false;
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          const int set = gates.used & 1;
          if (c + 1 < chunks) {
            if (lane == 0) gates.issue(walk.maps, n0 + (c + 1) * 64, y0);
            ++gates.issued;
          }
          if (!mbar_wait_warp(&gates.bars[set], (gates.used >> 1) & 1u, budget, abort)) {
            lost = true;
            break;
          }
          ++gates.used;
          uint8_t* gb = blocks + set * 2 * kEpiWarpBytes + lane * 128;
          uint8_t* ub = gb + kEpiWarpBytes;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t dh[32];
            tmem_ld32(taddr + c * 64 + u * 32, dh);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int at = ((4 * u + i) ^ (lane & 7)) << 4;
              uint4 gv = *reinterpret_cast<const uint4*>(gb + at), uv = *reinterpret_cast<const uint4*>(ub + at);
              uint32_t* gw = &gv.x;
              uint32_t* uw = &uv.x;
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                const float2 gf = unpack_pair<T>(gw[w]), uf = unpack_pair<T>(uw[w]);
                float dg0, dg1, du0, du1;
                swiglu_grad(__uint_as_float(dh[8 * i + 2 * w]), gf.x, uf.x, dg0, du0);
                swiglu_grad(__uint_as_float(dh[8 * i + 2 * w + 1]), gf.y, uf.y, dg1, du1);
                gw[w] = pack_pair<T>(__float_as_uint(dg0), __float_as_uint(dg1));
                uw[w] = pack_pair<T>(__float_as_uint(du0), __float_as_uint(du1));
              }
              if (!rows.ragged) {
                *reinterpret_cast<uint4*>(gb + at) = gv;
                *reinterpret_cast<uint4*>(ub + at) = uv;
              } else if (row0 + lane < rows.len) {
                const int64_t x = n0 + c * 64 + u * 32 + i * 8;
                if (x < j.n) {
                  const int64_t row = rows.start + row0 + lane;
                  *reinterpret_cast<uint4*>(j.t[2].data + (row * j.t[2].pitch + x) * 2) = gv;
                  *reinterpret_cast<uint4*>(j.t[3].data + (row * j.t[3].pitch + x) * 2) = uv;
                }
              }
            }
          }
          if (!rows.ragged) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              const uint8_t* from = blocks + set * 2 * kEpiWarpBytes;
              rows.put(2, from, n0 + c * 64, pol_out);
              rows.put(3, from + kEpiWarpBytes, n0 + c * 64, pol_out);
              bulk_commit_group();
            }
          } else {
            __syncwarp();  // read by every lane before the next loads land there
          }
        }
        if (lost) {
          if (lane == 0) fail(kErrWaitAccFull);
          break;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (G == 2) {
          mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(&acc_empty[buf]), 0));
        } else {
          mbar_arrive_relaxed(&acc_empty[buf]);
        }
      }
      ++acc_it;
    }
    if (EPI == kFfnSwigluBwd && *abort) {  // (g, u) loads in flight land first
      for (; gates.used != gates.issued; ++gates.used) {
        if (!mbar_wait_warp(&gates.bars[gates.used & 1], (gates.used >> 1) & 1u, budget, never)) {
          if (lane == 0) atomicOr(p.error_word, kErrWaitTeardown);
          break;
        }
      }
    }
    if (lane == 0) bulk_wait_group_read<0>();  // tensor stores have read the CTA's shared memory before it goes away
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (G == 2 || p.split > 1) cluster_sync();
  if constexpr (G == 1) {
    if (p.split > 1) {
      typename Cfg::Walk walk(p, ts, offs);
      FfnItems items(walk, 1);
      if (items.shared >= 0 && !*abort) {
        walk.seek(items.shared);
        const int32_t per = items.blocks_each(walk);
        ffn_join<T, EPI, Cfg>(p, walk, items, static_cast<int>((walk.kblocks + per - 1) / per), smem_u32(ring), warp, lane);
      }
      cluster_sync();  // the others' sums are read until here
    }
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

}  // namespace mgb
