// Host side of the gated feed-forward block's launches (mgb_ffn_kernel.cuh):
// argument checks, tensor-map templates, tile choice and the C entry points.
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
#include "mgb_ffn_kernel.cuh"

namespace {

using namespace mgb;

constexpr int64_t kMaxExtent = 1ll << 31;
constexpr size_t kMapBytes = sizeof(CUtensorMap);

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// The box of an operand or staged block.
enum Box { kKMajor, kMnMajor, kStage };

bool encode(CUtensorMap* map, int dtype, const FfnTensor& t, int64_t rows, int64_t cols, Box box, const void* dummy) {
  // A tensor without rows is never read; its template still needs a legal base and extent.
  const void* base = t.data != nullptr ? t.data : dummy;
  return encode_map_2d(map, dtype, base, static_cast<uint64_t>(cols), static_cast<uint64_t>(std::max<int64_t>(rows, 1)),
                       static_cast<uint64_t>(t.pitch) * 2, 64, box == kKMajor ? 128 : box == kMnMajor ? 64 : 32);
}

template <typename T, int EPI, int G>
int launch_kernel(const FfnParams& p, int64_t tiles, int sm_count, cudaStream_t stream) {
  using Cfg = FfnCfg<T, EPI, G>;
  auto kernel = ffn_kernel<T, EPI, G>;
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
  attr[0].val.clusterDim.x = G;
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
  const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(tiles, clusters[dev]));
  cfg.gridDim = dim3(static_cast<unsigned>(grid * G), 1, 1);
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  return e == cudaSuccess ? MGB_OK : MGB_ERR_CUDA;
}

template <int EPI>
int launch_epilogue(int dtype, int g, const FfnParams& p, int64_t tiles, int sms, cudaStream_t s) {
  if (dtype == MGB_BF16) {
    return g == 2 ? launch_kernel<__nv_bfloat16, EPI, 2>(p, tiles, sms, s)
                  : launch_kernel<__nv_bfloat16, EPI, 1>(p, tiles, sms, s);
  }
  return g == 2 ? launch_kernel<__half, EPI, 2>(p, tiles, sms, s) : launch_kernel<__half, EPI, 1>(p, tiles, sms, s);
}

// Tile edge of a launch over `p`'s jobs: pairs' 256 x 256 tiles when they
// cover the device's pairs once, else one CTA's 128 x 128 tiles (four times
// as many).  Rows of ragged segments are estimated as evenly spread.
int tile_group(const FfnParams& p, int epi, int sms) {
  int64_t tiles = 0;
  for (int i = 0; i < p.jobs; ++i) {
    const FfnJob& j = p.job[i];
    const int64_t n = cdiv(j.n, epi == kFfnSwiglu ? 128 : 256);
    const int64_t m = j.wgrad ? p.experts * cdiv(j.m, 256)
                              : std::max<int64_t>(cdiv(p.rows, 256), std::min<int64_t>(p.experts, p.rows));
    tiles += m * n;
  }
  return tiles >= sms / 2 ? 2 : 1;
}

struct Plan {
  FfnParams p;
  FfnTemplates tmpl;
};

FfnTensor tensor(const void* data, int64_t pitch, int64_t expert_stride, bool token) {
  return FfnTensor{static_cast<char*>(const_cast<void*>(data)), pitch, expert_stride, token ? 1 : 0};
}

size_t job_bytes(int64_t experts, int jobs) {
  const size_t pairs = static_cast<size_t>(experts) * jobs;
  return pairs * kFfnMaps * kMapBytes + (pairs + 1 + 15) / 16 * 16 * sizeof(int64_t);
}

// One launch: the plan kernel (maps and tile list) and the product kernel.
// `at` moves past the scratch it takes, so that launches of one call that
// may overlap (programmatic launch) never share any.
struct Launcher {
  int dtype;
  int64_t rows;
  int32_t experts;
  const int32_t* offs;
  uint8_t* at;
  cudaStream_t stream;
  int sms;
  uint32_t* error_word;
  long long budget;

  void init(Plan& plan, int jobs) {
    std::memset(static_cast<void*>(&plan), 0, sizeof(plan));
    plan.p.jobs = jobs;
    plan.p.experts = experts;
    plan.p.offs = offs;
    plan.p.rows = rows;
    plan.p.wait_budget = budget;
    plan.p.error_word = error_word;
  }

  // Rows job i: C[rows, n] = A[rows, k] op(B_e).
  bool rows_job(Plan& plan, int i, FfnTensor a, FfnTensor b, bool b_mn, int64_t n, int64_t k, int64_t b_cols) {
    FfnJob& j = plan.p.job[i];
    j.t[0] = a;
    j.t[1] = b;
    j.maps = 2;
    j.b_mn = b_mn;
    j.n = n;
    j.k = k;
    return encode(&plan.tmpl.map[i][0], dtype, a, rows, k, kKMajor, at) &&
           (b_mn ? encode(&plan.tmpl.map[i][1], dtype, b, k, b_cols, kMnMajor, at)
                 : encode(&plan.tmpl.map[i][1], dtype, b, n, k, kKMajor, at));
  }
  // Weight gradient job i: C_e[m, n] = A[rows, m]^T B[rows, n].
  bool wgrad_job(Plan& plan, int i, FfnTensor a, FfnTensor b, FfnTensor c, int64_t m, int64_t n) {
    FfnJob& j = plan.p.job[i];
    j.t[0] = a;
    j.t[1] = b;
    j.maps = 2;
    j.wgrad = 1;
    j.a_mn = j.b_mn = 1;
    j.m = m;
    j.n = n;
    return encode(&plan.tmpl.map[i][0], dtype, a, rows, m, kMnMajor, at) &&
           encode(&plan.tmpl.map[i][1], dtype, b, rows, n, kMnMajor, at) && add(plan, i, c, m, n);
  }
  // The next tensor of job i's epilogue.
  bool add(Plan& plan, int i, FfnTensor t, int64_t t_rows, int64_t cols) {
    FfnJob& j = plan.p.job[i];
    j.t[j.maps] = t;
    return encode(&plan.tmpl.map[i][j.maps++], dtype, t, t_rows, cols, kStage, at);
  }

  template <int EPI>
  int run(Plan& plan) {
    FfnParams& p = plan.p;
    const int g = tile_group(p, EPI, sms);
    p.tile_rows = 128 * g;
    p.tile_cols = EPI == kFfnSwiglu ? 64 * g : 128 * g;
    const size_t pairs = static_cast<size_t>(experts) * p.jobs;
    p.maps = at;
    p.tile_start = reinterpret_cast<int64_t*>(at + pairs * kFfnMaps * kMapBytes);
    at += job_bytes(experts, p.jobs);
    int64_t tiles = 0;  // at most: a segment boundary adds one row block
    for (int i = 0; i < p.jobs; ++i) {
      const FfnJob& j = p.job[i];
      const int64_t m = j.wgrad ? experts * cdiv(j.m, p.tile_rows) : cdiv(rows, p.tile_rows) + experts - 1;
      tiles += m * cdiv(j.n, p.tile_cols);
    }
    ffn_plan_kernel<<<static_cast<unsigned>(pairs + 1), 32, 0, stream>>>(plan.tmpl, p);
    if (cudaGetLastError() != cudaSuccess) return MGB_ERR_CUDA;
    return launch_epilogue<EPI>(dtype, g, p, tiles, sms, stream);
  }
};

// Every extent is positive and fits a tensor map, columns are whole 16-byte
// pieces, experts are few enough for one block each.
int check_shape(int32_t dtype, int32_t experts, int64_t rows, int64_t a, int64_t b, const int32_t* offs) {
  if (dtype != MGB_FP16 && dtype != MGB_BF16) return MGB_ERR_INVALID;
  if (experts <= 0 || experts > (1 << 20) || rows < 0 || a <= 0 || b <= 0 || a % 8 != 0 || b % 8 != 0) {
    return MGB_ERR_INVALID;
  }
  if (rows >= kMaxExtent || a >= kMaxExtent / 2 || b >= kMaxExtent / 2) return MGB_ERR_INVALID;
  if (offs == nullptr && experts != 1) return MGB_ERR_INVALID;
  return MGB_OK;
}

bool token_ok(const void* data, int64_t pitch, int64_t rows, int64_t cols) {
  return (rows == 0 || data != nullptr) && aligned16(data) && pitch >= cols && pitch % 8 == 0;
}

bool weight_ok(const void* data, int64_t pitch, int64_t stride, int64_t experts, int64_t rows, int64_t cols) {
  return data != nullptr && aligned16(data) && pitch >= cols && pitch % 8 == 0 && stride % 8 == 0 &&
         (experts == 1 || stride >= (rows - 1) * pitch + cols);
}

int start(Launcher& l, int32_t dtype, int64_t rows, int32_t experts, const int32_t* offs, int jobs, void* scratch,
          size_t scratch_bytes, void* stream) {
  if (scratch == nullptr || reinterpret_cast<uintptr_t>(scratch) % 128 != 0 ||
      scratch_bytes < ffn_scratch_bytes(experts, jobs)) {
    return MGB_ERR_SCRATCH;
  }
  int sms = 0;
  uint32_t* word = current_error_word();
  if (word == nullptr || !current_launch_limits(&sms, &l.budget)) return MGB_ERR_CUDA;
  l.dtype = dtype;
  l.rows = rows;
  l.experts = experts;
  l.offs = offs;
  l.at = static_cast<uint8_t*>(scratch);
  l.stream = static_cast<cudaStream_t>(stream);
  l.sms = sms;
  l.error_word = word;
  return MGB_OK;
}

// dgate_up = swiglu backward of dc b^T, or da = dc b^T.
int dgrad(Launcher& l, FfnTensor dc, FfnTensor b, FfnTensor out, const void* gate_up, int64_t gate_up_pitch, int64_t n,
          int64_t k) {
  Plan plan;
  l.init(plan, 1);
  bool ok = l.rows_job(plan, 0, dc, b, false, k, n, 0);
  if (gate_up == nullptr) {
    return ok && l.add(plan, 0, out, l.rows, k) ? l.run<kFfnPlain>(plan) : MGB_ERR_CUDA;
  }
  const auto half = [&](const void* base, int64_t pitch, int64_t at) {
    return tensor(base != nullptr ? static_cast<const char*>(base) + at * 2 : nullptr, pitch, 0, true);
  };
  ok = ok && l.add(plan, 0, half(out.data, out.pitch, 0), l.rows, k) &&
       l.add(plan, 0, half(out.data, out.pitch, k), l.rows, k) &&
       l.add(plan, 0, half(gate_up, gate_up_pitch, 0), l.rows, k) &&
       l.add(plan, 0, half(gate_up, gate_up_pitch, k), l.rows, k);
  return ok ? l.run<kFfnSwigluBwd>(plan) : MGB_ERR_CUDA;
}

}  // namespace

extern "C" {

size_t ffn_scratch_bytes(int32_t experts, int32_t jobs) {
  if (experts <= 0 || jobs <= 0) return 0;
  // One plan per job at most (the jobs of a call share plans or take turns).
  size_t bytes = 0;
  for (int32_t i = 0; i < jobs; ++i) bytes += job_bytes(experts, 1) + 128;
  return bytes;
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
  if (int st = start(l, f->dtype, rows, f->experts, f->offs, down ? 2 : 1, f->scratch, f->scratch_bytes, f->stream)) {
    return st;
  }
  if (rows == 0) return MGB_OK;
  Plan plan;
  l.init(plan, 1);
  const auto half = [&](int64_t at) {
    return tensor(static_cast<const char*>(f->gate_up) + at * 2, f->gate_up_pitch, 0, true);
  };
  plan.p.job[0].up = ffn;
  const FfnTensor h = tensor(f->h, f->h_pitch, 0, true);
  if (!l.rows_job(plan, 0, tensor(f->x, f->x_pitch, 0, true), tensor(f->w13, f->w13_pitch, f->w13_stride, false), true,
                  ffn, hid, 2 * ffn) ||
      !l.add(plan, 0, h, rows, ffn) || !l.add(plan, 0, half(0), rows, ffn) || !l.add(plan, 0, half(ffn), rows, ffn)) {
    return MGB_ERR_CUDA;
  }
  if (int st = l.run<kFfnSwiglu>(plan)) return st;
  if (!down) return MGB_OK;
  l.init(plan, 1);
  if (!l.rows_job(plan, 0, h, tensor(f->w2, f->w2_pitch, f->w2_stride, false), true, hid, ffn, hid) ||
      !l.add(plan, 0, tensor(f->y, f->y_pitch, 0, true), rows, hid)) {
    return MGB_ERR_CUDA;
  }
  return l.run<kFfnPlain>(plan);
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
  if (int st = start(l, f->dtype, rows, f->experts, f->offs, 4, f->scratch, f->scratch_bytes, f->stream)) return st;
  const FfnTensor dy = tensor(f->y, f->y_pitch, 0, true), x = tensor(f->x, f->x_pitch, 0, true);
  const FfnTensor h = tensor(f->h, f->h_pitch, 0, true), dgu = tensor(f->dgate_up, f->dgate_up_pitch, 0, true);
  if (rows > 0) {
    if (int st = dgrad(l, dy, tensor(f->w2, f->w2_pitch, f->w2_stride, false), dgu, f->gate_up, f->gate_up_pitch, hid,
                       ffn)) {
      return st;
    }
  }
  // dx, dW13 and dW2 depend on nothing but dgate_up: one launch.
  Plan plan;
  l.init(plan, 3);
  if (!l.rows_job(plan, 0, dgu, tensor(f->w13, f->w13_pitch, f->w13_stride, false), false, hid, 2 * ffn, 0) ||
      !l.add(plan, 0, tensor(f->dx, f->dx_pitch, 0, true), rows, hid) ||
      !l.wgrad_job(plan, 1, x, dgu, tensor(f->dw13, f->dw13_pitch, f->dw13_stride, false), hid, 2 * ffn) ||
      !l.wgrad_job(plan, 2, h, dy, tensor(f->dw2, f->dw2_pitch, f->dw2_stride, false), ffn, hid)) {
    return MGB_ERR_CUDA;
  }
  return l.run<kFfnPlain>(plan);
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
  if (int st = start(l, dtype, rows, experts, offs, 1, scratch, scratch_bytes, stream)) return st;
  if (rows == 0) return MGB_OK;
  return dgrad(l, tensor(dc, dc_pitch, 0, true), tensor(b, b_pitch, b_stride, false), tensor(out, out_pitch, 0, true),
               gate_up, gate_up_pitch, n, k);
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
  if (int st = start(l, dtype, rows, experts, offs, 1, scratch, scratch_bytes, stream)) return st;
  Plan plan;
  l.init(plan, 1);
  if (!l.wgrad_job(plan, 0, tensor(a, a_pitch, 0, true), tensor(dc, dc_pitch, 0, true),
                   tensor(db, db_pitch, db_stride, false), k, n)) {
    return MGB_ERR_CUDA;
  }
  return l.run<kFfnPlain>(plan);
}

}  // extern "C"
