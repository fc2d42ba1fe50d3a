// Host side of the gated feed-forward block's launches (mgb_ffn_kernel.cuh):
// argument checks, tensor-map templates, tile choice and the C entry points.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>

#include "../../include/moe_gemm_b200.h"
#include "mgb_dispatch.cuh"
#include "mgb_ffn_kernel.cuh"

namespace {

using namespace mgb;

constexpr int64_t kMaxExtent = 1ll << 31;
constexpr int64_t kMaxRows = kMaxExtent - 1024;  // a row block past the last row still has a 32-bit coordinate
constexpr size_t kMapBytes = sizeof(CUtensorMap);

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// What the thread's last call launched (ffn_last_launches).
thread_local mgb_ffn_launch_info last_launch[kFfnLaunches];
thread_local int last_launches = 0;

// The box of an operand or staged block, in rows of 64 columns.
enum Box : uint32_t { kKMajor = 128, kMnMajor = 64, kStage = 32 };

template <typename T, int EPI, int G, int NH>
int launch_kernel(const FfnParams& p, int64_t tiles, int sm_count, cudaStream_t stream) {
  using Cfg = FfnCfg<T, EPI, G, NH>;
  auto kernel = ffn_kernel<T, EPI, G, NH>;
  static bool configured[128] = {};
  static int clusters[128] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 128) return MGB_ERR_CUDA;
  cudaLaunchAttribute attr[2] = {};
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kTcThreads, 1, 1);
  cfg.dynamicSmemBytes = Cfg::kSmemBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = G * p.split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes) != cudaSuccess) {
      return MGB_ERR_CUDA;
    }
    clusters[dev] = sm_count / G;
    if (G == 2) {  // clusters of two that the device keeps resident at once
      cfg.gridDim = dim3(static_cast<unsigned>(sm_count & ~1), 1, 1);
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess && n > 0) {
        clusters[dev] = n;
      } else {
        cudaGetLastError();
      }
    }
    configured[dev] = true;
  }
  // `tiles` of a split launch are its clusters (never more CTAs than SMs).
  const int64_t grid = p.split > 1 ? tiles : std::max<int64_t>(1, std::min<int64_t>(tiles, clusters[dev]));
  cfg.gridDim = dim3(static_cast<unsigned>(grid * G * p.split), 1, 1);
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) return MGB_ERR_CUDA;
  last_launch[last_launches++] = {EPI, G == 2 ? 1 : 0, Cfg::kTileM, Cfg::kTileOut, p.split,
                                  static_cast<int32_t>(cfg.gridDim.x)};
  return MGB_OK;
}

// Output tile of a launch.
struct Tile {
  int g;     // CTAs
  bool wide; // 512 columns
};

template <typename T, int EPI>
int launch_typed(Tile tile, const FfnParams& p, int64_t tiles, int sms, cudaStream_t s) {
  if constexpr (EPI == kFfnPlain) {
    if (tile.wide) return launch_kernel<T, EPI, 2, 2>(p, tiles, sms, s);
  }
  return tile.g == 2 ? launch_kernel<T, EPI, 2, 1>(p, tiles, sms, s) : launch_kernel<T, EPI, 1, 1>(p, tiles, sms, s);
}

template <int EPI>
int launch_epilogue(int dtype, Tile tile, const FfnParams& p, int64_t tiles, int sms, cudaStream_t s) {
  return dtype == MGB_BF16 ? launch_typed<__nv_bfloat16, EPI>(tile, p, tiles, sms, s)
                           : launch_typed<__half, EPI>(tile, p, tiles, sms, s);
}

FfnTensor tensor(const void* data, int64_t pitch, int64_t expert_stride, bool token) {
  return FfnTensor{static_cast<char*>(const_cast<void*>(data)), pitch, expert_stride, token ? 1 : 0};
}

// Scratch of a call: the operand maps of weight gradients, and a tile list for
// each launch whose list does not fit shared memory.
size_t maps_bytes(int64_t experts, int wgrads) { return static_cast<size_t>(experts) * wgrads * 2 * kMapBytes; }
bool global_list(int64_t experts, int jobs) { return (jobs + 1) * experts + 1 > kListWords; }
size_t list_bytes(int64_t experts, int jobs) {
  return global_list(experts, jobs) ? (static_cast<size_t>(experts) * jobs + 1 + 31) / 32 * 32 * sizeof(int32_t) : 0;
}

// The launches of one call: jobs are added launch by launch, then run()
// issues the plan kernel where one is needed and the product kernels.
struct Launcher {
  FfnPlan plan;
  FfnParams params[kFfnLaunches];
  Tile tile[kFfnLaunches];
  int epilogue[kFfnLaunches];
  int launches = 0;
  int dtype;
  int64_t rows, experts;
  uint8_t* scratch;
  cudaStream_t stream;
  int sms;
  long long budget;
  bool ok = true;

  FfnParams& now() { return params[launches - 1]; }
  void begin_launch(int epi) {
    FfnParams& p = params[launches];
    std::memset(static_cast<void*>(&p), 0, sizeof(p));
    p.experts = static_cast<int32_t>(experts);
    p.offs = plan.offs;
    p.rows = rows;
    p.wait_budget = budget;
    p.error_word = plan.error_word;
    p.split = 1;
    epilogue[launches++] = epi;
  }
  FfnJob& job() { return now().job[now().jobs - 1]; }
  // The last job's tensor i, [t_rows, cols] in boxes of `box`.
  void set(int i, const FfnTensor& t, int64_t t_rows, int64_t cols, Box box) {
    job().t[i] = t;
    CUtensorMap* map = &now().map[now().jobs - 1][i];
    const uint64_t pitch = static_cast<uint64_t>(t.pitch) * 2;
    if (t.token) {
      ok = ok && encode_map_2d(map, dtype, t.data, cols, t_rows, pitch, 64, box);
    } else {
      const uint64_t stride = experts > 1 ? static_cast<uint64_t>(t.expert_stride) * 2 : pitch * t_rows;
      ok = ok && encode_map_3d(map, dtype, t.data, cols, t_rows, experts, pitch, stride, 64, box);
    }
  }
  // Rows job: C[rows, n] = A[rows, k] op(B_e); its epilogue's tensors follow.
  void rows_job(const FfnTensor& a, const FfnTensor& b, bool b_mn, int64_t n, int64_t k, int64_t b_cols) {
    ++now().jobs;
    FfnJob& j = job();
    j.b_mn = b_mn;
    j.n = n;
    j.k = k;
    if (rows > 0) set(0, a, rows, k, kKMajor);
    if (b_mn) {
      set(1, b, k, b_cols, kMnMajor);
    } else {
      set(1, b, n, k, kKMajor);
    }
  }
  // Without rows the tensor stays unset: the kernel prefetches the map of every
  // tensor that is there, and there is none to encode.
  void output(int i, const FfnTensor& t, int64_t cols) {
    if (rows > 0) set(i, t, rows, cols, kStage);
  }
  // Weight gradient job: C_e[m, n] = A[rows, m]^T B[rows, n].
  void wgrad_job(const FfnTensor& a, const FfnTensor& b, const FfnTensor& c, int64_t m, int64_t n) {
    ++now().jobs;
    FfnJob& j = job();
    j.wgrad = 1;
    j.b_mn = 1;
    j.m = m;
    j.n = n;
    set(2, c, m, n, kStage);
    const int w = plan.wgrads++;
    const FfnTensor operand[2] = {a, b};
    const int64_t cols[2] = {m, n};
    for (int i = 0; i < 2; ++i) {
      plan.t[w][i] = operand[i];
      // Without rows the maps are never used; the template still needs a legal base.
      const void* base = operand[i].data != nullptr ? operand[i].data : static_cast<const void*>(scratch);
      ok = ok && encode_map_2d(&plan.map[w][i], dtype, base, cols[i], 1, static_cast<uint64_t>(operand[i].pitch) * 2, 64,
                               kMnMajor);
    }
  }

  // Output tile of a launch: the least estimated time among one CTA's
  // 128 x 128 tiles (whose long contractions may be split), pairs' 256 x 256
  // and, for the plain epilogue, 256 x 512 ones.  The unit is a 64-deep block
  // of a CTA or pair (0.3 us; a 512-column one 1.9 of them); a tile adds its
  // start and epilogue (4, 5 and 9 units by size, measured on contractions of
  // a few blocks).  bf16 4096^3: 512 columns 98 us, 256 104; 8192^3: 690
  // against 760.  Rows of ragged segments are estimated as evenly spread.
  Tile tile_of(const FfnParams& p, int epi) const {
    const Tile tiles[3] = {{2, true}, {2, false}, {1, false}};
    const double block[3] = {1.9, 1.0, 1.0}, fixed[3] = {9.0, 5.0, 4.0};
    Tile best = tiles[1];
    double least = 1e300;
    for (int c = epi == kFfnPlain ? 0 : 1; c < 3; ++c) {
      const Tile t = tiles[c];
      const int64_t segments = std::max<int64_t>(1, std::min(experts, rows));
      const double each = static_cast<double>(std::max<int64_t>(rows, 1)) / segments;
      FfnParams q;
      q.split = 1;
      if (t.g == 1) {
        q.job[0] = p.job[0];
        split_of(q, t, epi, 0);
      }
      double work = 0, longest = 0;
      for (int i = 0; i < p.jobs; ++i) {
        const FfnJob& j = p.job[i];
        const double m = j.wgrad ? experts * cdiv(j.m, tile_rows(t)) : segments * std::ceil(each / tile_rows(t));
        const double depth = j.wgrad ? std::ceil(each / 64) : cdiv(j.k, 64);
        const int split = i == 0 ? q.split : 1;
        const double one = depth / split * block[c] + fixed[c];
        work += m * cdiv(j.n, tile_cols(t, epi)) * one * split;
        longest = std::max(longest, one);
      }
      const double time = std::max(work / (sms / t.g), longest);
      if (time < least * 0.999) {
        least = time;
        best = t;
      }
    }
    return best;
  }
  static int tile_rows(Tile t) { return 128 * t.g; }
  static int tile_cols(Tile t, int epi) { return (epi == kFfnSwiglu ? 64 : t.wide ? 256 : 128) * t.g; }

  // Tiles of a job, at most (a segment boundary adds one row block).
  int64_t tiles_of(const FfnJob& j, Tile t, int epi) const {
    const int64_t m = j.wgrad ? experts * cdiv(j.m, tile_rows(t))
                              : cdiv(rows, tile_rows(t)) + std::max<int64_t>(std::min(experts, rows) - 1, 0);
    return m * cdiv(j.n, tile_cols(t, epi));
  }

  // Splits the contraction of job 0's tiles: as many CTAs a tile (2, 4 or 8)
  // as the SMs hold at once, each with at least four blocks.  Returns the
  // launch's clusters (its tiles, unsplit).
  int64_t split_of(FfnParams& p, Tile t, int epi, int64_t tiles) const {
    if (rows == 0 || t.g != 1 || p.job[0].wgrad) return tiles;
    const int64_t own = tiles_of(p.job[0], t, epi);
    const int64_t blocks = cdiv(p.job[0].k, 64);
    while (p.split < 8 && own * p.split * 2 <= sms && blocks >= 8 * p.split && own <= clusters(p.split * 2)) p.split *= 2;
    if (p.split == 1) return tiles;
    // Other jobs' tiles go to every CTA one by one.
    return std::max(own, std::min<int64_t>(clusters(p.split), cdiv(tiles - own, p.split)));
  }
  static int clusters(int size) {
    using Cfg = FfnCfg<__nv_bfloat16, kFfnPlain, 1>;
    return resident_clusters(reinterpret_cast<const void*>(ffn_kernel<__nv_bfloat16, kFfnPlain, 1, 1>), kTcThreads,
                             Cfg::kSmemBytes, size);
  }

  int run() {
    if (!ok) return MGB_ERR_CUDA;
    CUtensorMap* maps = reinterpret_cast<CUtensorMap*>(scratch);
    uint8_t* list = scratch + maps_bytes(experts, plan.wgrads);
    int64_t tiles[kFfnLaunches];
    int wgrad = 0;
    for (int i = 0; i < launches; ++i) {
      FfnParams& p = params[i];
      tile[i] = tile_of(p, epilogue[i]);
      tiles[i] = 0;
      for (int k = 0; k < p.jobs; ++k) {
        tiles[i] += tiles_of(p.job[k], tile[i], epilogue[i]);
        if (p.job[k].wgrad) {
          plan.operands[wgrad] = maps;
          p.job[k].operands = maps;
          maps += 2 * experts;
          ++wgrad;
        }
      }
      if (tiles[i] >= (1ll << 31)) return MGB_ERR_INVALID;  // the list's 32-bit tile numbers
      if (global_list(experts, p.jobs)) {
        FfnPlan::List& l = plan.list[plan.lists++];
        l.jobs = p.jobs;
        l.tile_rows = tile_rows(tile[i]);
        l.tile_cols = tile_cols(tile[i], epilogue[i]);
        for (int k = 0; k < p.jobs; ++k) {
          l.wgrad[k] = p.job[k].wgrad;
          l.m[k] = p.job[k].m;
          l.n[k] = p.job[k].n;
        }
        l.tile_start = reinterpret_cast<int32_t*>(list);
        p.tile_start = l.tile_start;
        list += list_bytes(experts, p.jobs);
      }
    }
    if (plan.lists == 0 && launches == 2 && epilogue[0] == kFfnSwigluBwd) {
      // The first launch cuts the second one's maps.
      FfnParams& p = params[0];
      p.cuts = plan.wgrads;
      for (int w = 0; w < plan.wgrads; ++w) {
        p.job[1 + w].operands = plan.operands[w];
        for (int i = 0; i < 2; ++i) {
          p.map[1 + w][i] = plan.map[w][i];
          p.job[1 + w].t[i] = plan.t[w][i];
        }
      }
    } else if (const int64_t blocks = plan.wgrads * experts + plan.lists; blocks > 0) {
      const unsigned grid = static_cast<unsigned>(blocks);
      if (launch_overlapped(ffn_plan_kernel, grid, 64, 0, stream, plan) != cudaSuccess) return MGB_ERR_CUDA;
    }
    for (int i = 0; i < launches; ++i) {
      FfnParams& p = params[i];
      const int64_t grid = split_of(p, tile[i], epilogue[i], tiles[i]);
      const int st = epilogue[i] == kFfnPlain    ? launch_epilogue<kFfnPlain>(dtype, tile[i], p, grid, sms, stream)
                     : epilogue[i] == kFfnSwiglu ? launch_epilogue<kFfnSwiglu>(dtype, tile[i], p, grid, sms, stream)
                                                 : launch_epilogue<kFfnSwigluBwd>(dtype, tile[i], p, grid, sms, stream);
      if (st) return st;
    }
    return MGB_OK;
  }
};

// Every extent is positive and fits a tensor map, columns are whole 16-byte
// pieces, experts are few enough for one block each.
int check_shape(int32_t dtype, int32_t experts, int64_t rows, int64_t a, int64_t b, const int32_t* offs) {
  if (dtype != MGB_FP16 && dtype != MGB_BF16) return MGB_ERR_INVALID;
  if (experts <= 0 || experts > (1 << 20) || rows < 0 || a <= 0 || b <= 0 || a % 8 != 0 || b % 8 != 0) {
    return MGB_ERR_INVALID;
  }
  if (rows > kMaxRows || a >= kMaxExtent / 2 || b >= kMaxExtent / 2) return MGB_ERR_INVALID;
  if (offs == nullptr && experts != 1) return MGB_ERR_INVALID;
  return MGB_OK;
}

bool token_ok(const void* data, int64_t pitch, int64_t rows, int64_t cols) {
  return (rows == 0 || data != nullptr) && aligned16(data) && pitch >= cols && pitch % 8 == 0;
}

bool weight_ok(const void* data, int64_t pitch, int64_t stride, int64_t experts, int64_t rows, int64_t cols) {
  // A 3-D tensor map's strides are whole multiples of one another.
  return data != nullptr && aligned16(data) && pitch >= cols && pitch % 8 == 0 &&
         (experts == 1 || (stride % pitch == 0 && stride >= rows * pitch));
}

int start(Launcher& l, int32_t dtype, int64_t rows, int32_t experts, const int32_t* offs, int call, void* scratch,
          size_t scratch_bytes, void* stream) {
  const size_t need = ffn_scratch_bytes(experts, call);
  if (need > 0 && (scratch == nullptr || reinterpret_cast<uintptr_t>(scratch) % 128 != 0 || scratch_bytes < need)) {
    return MGB_ERR_SCRATCH;
  }
  last_launches = 0;
  std::memset(static_cast<void*>(&l.plan), 0, sizeof(l.plan));
  l.plan.error_word = current_error_word();
  if (l.plan.error_word == nullptr || !current_launch_limits(&l.sms, &l.budget)) return MGB_ERR_CUDA;
  l.plan.experts = experts;
  l.plan.offs = offs;
  l.plan.rows = rows;
  l.rows = rows;
  l.experts = experts;
  l.dtype = dtype;
  l.scratch = static_cast<uint8_t*>(scratch);
  l.stream = static_cast<cudaStream_t>(stream);
  return MGB_OK;
}

// A launch of dgate_up = swiglu backward of dc b^T, or da = dc b^T.
void dgrad(Launcher& l, const FfnTensor& dc, const FfnTensor& b, const FfnTensor& out, const void* gate_up,
           int64_t gate_up_pitch, int64_t n, int64_t k) {
  l.begin_launch(gate_up != nullptr ? kFfnSwigluBwd : kFfnPlain);
  l.rows_job(dc, b, false, k, n, 0);
  const auto half = [](const void* base, int64_t pitch, int64_t at) {
    return tensor(base != nullptr ? static_cast<const char*>(base) + at * 2 : nullptr, pitch, 0, true);
  };
  l.output(2, half(out.data, out.pitch, 0), k);
  if (gate_up != nullptr) {
    l.output(3, half(out.data, out.pitch, k), k);
    l.output(4, half(gate_up, gate_up_pitch, 0), k);
    l.output(5, half(gate_up, gate_up_pitch, k), k);
  }
}

}  // namespace

extern "C" {

size_t ffn_scratch_bytes(int32_t experts, int32_t call) {
  if (experts <= 0) return 0;
  switch (call) {
    case MGB_FFN_FORWARD: return 2 * list_bytes(experts, 1);
    case MGB_FFN_BACKWARD: return maps_bytes(experts, 2) + list_bytes(experts, 1) + list_bytes(experts, 3);
    case MGB_FFN_DGRAD: return list_bytes(experts, 1);
    case MGB_FFN_WGRAD: return maps_bytes(experts, 1) + list_bytes(experts, 1);
    default: return 0;
  }
}

int gated_ffn_forward_launch(const mgb_ffn_args* f) {
  if (f == nullptr) return MGB_ERR_INVALID;
  const int64_t rows = f->rows, hid = f->hidden, ffn = f->ffn;
  if (int st = check_shape(f->dtype, f->experts, rows, hid, ffn, f->offs)) return st;
  if (!token_ok(f->x, f->x_pitch, rows, hid) || !token_ok(f->h, f->h_pitch, rows, ffn) ||
      !token_ok(f->gate_up, f->gate_up_pitch, rows, 2 * ffn) ||
      !weight_ok(f->w13, f->w13_pitch, f->w13_stride, f->experts, hid, 2 * ffn)) {
    return MGB_ERR_INVALID;
  }
  const bool down = f->w2 != nullptr;
  if (down && (!weight_ok(f->w2, f->w2_pitch, f->w2_stride, f->experts, ffn, hid) ||
               !token_ok(f->y, f->y_pitch, rows, hid))) {
    return MGB_ERR_INVALID;
  }
  Launcher l;
  if (int st = start(l, f->dtype, rows, f->experts, f->offs, MGB_FFN_FORWARD, f->scratch, f->scratch_bytes, f->stream)) {
    return st;
  }
  if (rows == 0) return MGB_OK;
  const auto half = [&](int64_t at) {
    return tensor(static_cast<const char*>(f->gate_up) + at * 2, f->gate_up_pitch, 0, true);
  };
  const FfnTensor h = tensor(f->h, f->h_pitch, 0, true);
  l.begin_launch(kFfnSwiglu);
  l.rows_job(tensor(f->x, f->x_pitch, 0, true), tensor(f->w13, f->w13_pitch, f->w13_stride, false), true, ffn, hid,
             2 * ffn);
  l.job().up = ffn;
  l.output(2, h, ffn);
  l.output(3, half(0), ffn);
  l.output(4, half(ffn), ffn);
  if (down) {
    l.begin_launch(kFfnPlain);
    l.rows_job(h, tensor(f->w2, f->w2_pitch, f->w2_stride, false), true, hid, ffn, hid);
    l.output(2, tensor(f->y, f->y_pitch, 0, true), hid);
  }
  return l.run();
}

int gated_ffn_backward_launch(const mgb_ffn_args* f) {
  if (f == nullptr) return MGB_ERR_INVALID;
  const int64_t rows = f->rows, hid = f->hidden, ffn = f->ffn;
  if (int st = check_shape(f->dtype, f->experts, rows, hid, ffn, f->offs)) return st;
  if (!token_ok(f->y, f->y_pitch, rows, hid) || !token_ok(f->x, f->x_pitch, rows, hid) ||
      !token_ok(f->h, f->h_pitch, rows, ffn) || !token_ok(f->gate_up, f->gate_up_pitch, rows, 2 * ffn) ||
      !token_ok(f->dgate_up, f->dgate_up_pitch, rows, 2 * ffn) || !token_ok(f->dx, f->dx_pitch, rows, hid) ||
      !weight_ok(f->w13, f->w13_pitch, f->w13_stride, f->experts, hid, 2 * ffn) ||
      !weight_ok(f->w2, f->w2_pitch, f->w2_stride, f->experts, ffn, hid) ||
      !weight_ok(f->dw13, f->dw13_pitch, f->dw13_stride, f->experts, hid, 2 * ffn) ||
      !weight_ok(f->dw2, f->dw2_pitch, f->dw2_stride, f->experts, ffn, hid)) {
    return MGB_ERR_INVALID;
  }
  Launcher l;
  if (int st = start(l, f->dtype, rows, f->experts, f->offs, MGB_FFN_BACKWARD, f->scratch, f->scratch_bytes, f->stream)) return st;
  const FfnTensor dy = tensor(f->y, f->y_pitch, 0, true), x = tensor(f->x, f->x_pitch, 0, true);
  const FfnTensor h = tensor(f->h, f->h_pitch, 0, true), dgu = tensor(f->dgate_up, f->dgate_up_pitch, 0, true);
  if (rows > 0) {
    dgrad(l, dy, tensor(f->w2, f->w2_pitch, f->w2_stride, false), dgu, f->gate_up, f->gate_up_pitch, hid, ffn);
  }
  // dx, dW13 and dW2 depend on nothing but dgate_up: one launch.
  l.begin_launch(kFfnPlain);
  l.rows_job(dgu, tensor(f->w13, f->w13_pitch, f->w13_stride, false), false, hid, 2 * ffn, 0);
  l.output(2, tensor(f->dx, f->dx_pitch, 0, true), hid);
  l.wgrad_job(x, dgu, tensor(f->dw13, f->dw13_pitch, f->dw13_stride, false), hid, 2 * ffn);
  l.wgrad_job(h, dy, tensor(f->dw2, f->dw2_pitch, f->dw2_stride, false), ffn, hid);
  return l.run();
}

int grouped_gemm_dgrad_launch(const void* dc, int64_t dc_pitch, const void* b, int64_t b_pitch, int64_t b_stride,
                              const int32_t* offs, int32_t experts, int64_t rows, int64_t n, int64_t k,
                              const void* gate_up, int64_t gate_up_pitch, void* out, int64_t out_pitch, int32_t dtype,
                              void* scratch, size_t scratch_bytes, void* stream) {
  if (int st = check_shape(dtype, experts, rows, n, k, offs)) return st;
  const int64_t out_cols = gate_up != nullptr ? 2 * k : k;
  if (!token_ok(dc, dc_pitch, rows, n) || !weight_ok(b, b_pitch, b_stride, experts, k, n) ||
      !token_ok(out, out_pitch, rows, out_cols) ||
      (gate_up != nullptr && !token_ok(gate_up, gate_up_pitch, rows, out_cols))) {
    return MGB_ERR_INVALID;
  }
  Launcher l;
  if (int st = start(l, dtype, rows, experts, offs, MGB_FFN_DGRAD, scratch, scratch_bytes, stream)) return st;
  if (rows == 0) return MGB_OK;
  dgrad(l, tensor(dc, dc_pitch, 0, true), tensor(b, b_pitch, b_stride, false), tensor(out, out_pitch, 0, true), gate_up,
        gate_up_pitch, n, k);
  return l.run();
}

int grouped_gemm_wgrad_launch(const void* a, int64_t a_pitch, const void* dc, int64_t dc_pitch, const int32_t* offs,
                              int32_t experts, int64_t rows, int64_t n, int64_t k, void* db, int64_t db_pitch,
                              int64_t db_stride, int32_t dtype, void* scratch, size_t scratch_bytes, void* stream) {
  if (int st = check_shape(dtype, experts, rows, n, k, offs)) return st;
  if (!token_ok(a, a_pitch, rows, k) || !token_ok(dc, dc_pitch, rows, n) ||
      !weight_ok(db, db_pitch, db_stride, experts, k, n)) {
    return MGB_ERR_INVALID;
  }
  Launcher l;
  if (int st = start(l, dtype, rows, experts, offs, MGB_FFN_WGRAD, scratch, scratch_bytes, stream)) return st;
  l.begin_launch(kFfnPlain);
  l.wgrad_job(tensor(a, a_pitch, 0, true), tensor(dc, dc_pitch, 0, true), tensor(db, db_pitch, db_stride, false), k, n);
  return l.run();
}

int32_t ffn_last_launches(mgb_ffn_launch_info* info, int32_t capacity) {
  for (int i = 0; info != nullptr && i < last_launches && i < capacity; ++i) info[i] = last_launch[i];
  return last_launches;
}

}  // extern "C"
