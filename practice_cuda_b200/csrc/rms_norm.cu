// C entry points of the root-mean-square norm.
#include <algorithm>

#include "host.cuh"
#include "rms_norm.cuh"

using namespace pcb;

namespace {

bool fits_units(const void* p, int64_t row_stride, int es) {
  return aligned(p, 16) && (row_stride * es) % 16 == 0;
}

template <int XT, int YT, int LANES, int NV, int MAX_THREADS>
int launch_norm_fwd(const norm::FwdArgs& p, int threads, cudaStream_t s) {
  const int64_t rows = LANES ? MAX_THREADS / (LANES ? LANES : 1) : 1;  // per CTA
  const unsigned grid = (unsigned)((p.rows + rows - 1) / rows);
  const int block = LANES ? MAX_THREADS : threads;
  if (p.res) norm::rms_norm_fwd_kernel<XT, YT, LANES, NV, MAX_THREADS, true><<<grid, block, 0, s>>>(p);
  else norm::rms_norm_fwd_kernel<XT, YT, LANES, NV, MAX_THREADS, false><<<grid, block, 0, s>>>(p);
  return check_launch("rms_norm_fwd_kernel");
}

int threads_of(int items, int per_thread, int step) {
  const int t = (items + per_thread - 1) / per_thread;
  return (t + step - 1) / step * step;
}

// False: the generic kernel takes the rows.  Columns that a thread has beyond the
// width cost as much as the others, so a CTA has eight a thread up to 8192 columns
// (16384 x 1021 bf16 with a residual and y on a B200: 68 us, 115 with sixteen; 16384 x
// 3001: 193 and 250 us; 8192 x 8191: 330 and 369 us), but for 16-bit rows of 4097
// to 6144, whose eight columns leave an SM one CTA where sixteen leave it two
// (12000 x 5001: 344 and 293 us; in fp32, with more registers, 342 and 444 us).
// Without a residual, whose sum it would read back, the generic kernel is faster
// beyond 2048 columns (16384 x 4095: 149 us, 211 with eight columns a thread; 16384
// x 1901: 96 us with eight).
template <int XT, int YT, int WT>
bool launch_norm_fwd_elems(const norm::FwdArgs& p, cudaStream_t s) {
  constexpr int NE = norm::kElems;
  const int threads = threads_of(p.dim, 8, 128), wide = threads_of(p.dim, NE, 128);
  if (p.dim <= 32 * NE)
    norm::rms_norm_fwd_elems_kernel<XT, YT, WT, true, NE, 256><<<(unsigned)((p.rows + 7) / 8), 256, 0, s>>>(p);
  else if (!p.res && p.dim > 2048)
    return false;
  else if (threads <= 512)
    norm::rms_norm_fwd_elems_kernel<XT, YT, WT, false, 8, 512><<<(unsigned)p.rows, threads, 0, s>>>(p);
  else if (XT != PCB_DTYPE_F32 && threads <= 768)
    norm::rms_norm_fwd_elems_kernel<XT, YT, WT, false, XT == PCB_DTYPE_F32 ? 8 : NE, 512>
        <<<(unsigned)p.rows, wide, 0, s>>>(p);
  else if (threads <= 1024)
    norm::rms_norm_fwd_elems_kernel<XT, YT, WT, false, 8, 1024><<<(unsigned)p.rows, threads, 0, s>>>(p);
  else if (wide <= 1024)
    norm::rms_norm_fwd_elems_kernel<XT, YT, WT, false, NE, 1024><<<(unsigned)p.rows, wide, 0, s>>>(p);
  else
    return false;
  return true;
}

// Four units of eight elements a lane keep a row in registers at 32 values a
// thread.  Rows up to 1024 wide are a warp's (up to 128 wide, half a warp's)
// and need no barrier; wider ones get a CTA of as many warps as they need
// (128 threads at 4096: 97 us for 16384 rows of bf16 on a B200, 101 us with two
// units a lane).
template <int XT, int YT>
int dispatch_norm_fwd(const norm::FwdArgs& p, bool vec, cudaStream_t s) {
  const int units = p.dim / norm::kUnit;
  if (vec && units <= 4096) {
    if (units <= 16) return launch_norm_fwd<XT, YT, 16, 1, 256>(p, 0, s);
    if (units <= 32) return launch_norm_fwd<XT, YT, 32, 1, 256>(p, 0, s);
    if (units <= 64) return launch_norm_fwd<XT, YT, 32, 2, 256>(p, 0, s);
    if (units <= 128) return launch_norm_fwd<XT, YT, 32, 4, 256>(p, 0, s);
    if (units <= 2048) return launch_norm_fwd<XT, YT, 0, 4, 512>(p, threads_of(units, 4, 32), s);
    return launch_norm_fwd<XT, YT, 0, 4, 1024>(p, threads_of(units, 4, 32), s);
  }
  const bool same = p.w_dtype == XT, f32 = p.w_dtype == PCB_DTYPE_F32;
  if ((same && launch_norm_fwd_elems<XT, YT, XT>(p, s)) ||
      (!same && f32 && launch_norm_fwd_elems<XT, YT, PCB_DTYPE_F32>(p, s)))
    return check_launch("rms_norm_fwd_elems_kernel");
  // Wide rows, or a weight of the other 16-bit type.
  const int64_t grid = std::min<int64_t>(p.rows, (int64_t)device_info().sm_count * 8);
  norm::rms_norm_fwd_generic_kernel<XT, YT><<<(unsigned)grid, norm::kGenericThreads, 0, s>>>(p);
  return check_launch("rms_norm_fwd_generic_kernel");
}

// CTAs of the backward pass: those that are resident at once, each of which
// leaves one row of dw shares.
constexpr int kNormBwdMost = 4;  // per SM, in any variant
int norm_bwd_ctas(int64_t rows, int rows_per_cta, int per_sm) {
  const int64_t ctas = (rows + rows_per_cta - 1) / rows_per_cta;
  return (int)std::min<int64_t>(ctas, (int64_t)device_info().sm_count * per_sm);
}

constexpr int kNormDwSmem = 160 * 1024;  // dw shares of one CTA of the generic backward

template <int XT, int LANES, int NV>
int launch_norm_bwd(const norm::BwdArgs& p, int& parts, cudaStream_t s) {
  constexpr int threads = LANES > 256 ? LANES : 256, rows = threads / LANES;
  parts = norm_bwd_ctas(p.rows, rows, LANES > 256 ? 1 : 2);
  const int smem = rows > 1 ? p.dim * 4 : 0;  // at most 2048 columns of fp32 (128 lanes of two units)
  norm::rms_norm_bwd_kernel<XT, LANES, NV><<<parts, threads, smem, s>>>(p);
  return check_launch("rms_norm_bwd_kernel");
}

// 16-bit rows of at most 512 NV units.
template <int XT, int NV>
int launch_norm_bwd_staged(const norm::BwdArgs& p, int& parts, cudaStream_t s) {
  auto kernel = norm::rms_norm_bwd_staged_kernel<XT, NV>;
  const int smem = p.dim / norm::kUnit * norm::kStagedBytes;
  ensure_smem_attr(kernel, smem);
  parts = norm_bwd_ctas(p.rows, 1, 1);
  kernel<<<parts, norm::kStagedThreads, smem, s>>>(p);
  return check_launch("rms_norm_bwd_staged_kernel");
}

// False: the rows are too wide for these kernels.  Eight columns a thread keep
// clear of register spills and let more of a row's loads be on their way (8192 x
// 7001 bf16 on a B200: 218 us, 253 with sixteen; fp32 241 either way); sixteen take
// the widths beyond (4096 x 16383 bf16: 292 us with a few registers spilled, 1197 us
// in the generic kernel, which reads the row again from memory).
template <int XT, int WT>
bool launch_norm_bwd_elems(const norm::BwdArgs& p, int& parts, cudaStream_t s) {
  if (p.dim <= 32 * norm::kElems) {
    parts = norm_bwd_ctas(p.rows, 8, 2);
    norm::rms_norm_bwd_elems_kernel<XT, WT, true, norm::kElems, 256><<<parts, 256, 0, s>>>(p);
  } else if (p.dim <= 512 * 8) {
    const int threads = threads_of(p.dim, 8, 32);
    parts = norm_bwd_ctas(p.rows, 1, std::min(kNormBwdMost, 1024 / threads));
    norm::rms_norm_bwd_elems_kernel<XT, WT, false, 8, 512><<<parts, threads, 0, s>>>(p);
  } else if (p.dim <= 1024 * 8) {
    parts = norm_bwd_ctas(p.rows, 1, 1);
    norm::rms_norm_bwd_elems_kernel<XT, WT, false, 8, 1024><<<parts, threads_of(p.dim, 8, 32), 0, s>>>(p);
  } else if (p.dim <= 1024 * 16) {
    parts = norm_bwd_ctas(p.rows, 1, 1);
    norm::rms_norm_bwd_elems_kernel<XT, WT, false, 16, 1024><<<parts, threads_of(p.dim, 16, 32), 0, s>>>(p);
  } else {
    return false;
  }
  return true;
}

template <int XT>
int dispatch_norm_bwd(const norm::BwdArgs& p, bool vec, int& parts, cudaStream_t s) {
  const int units = p.dim / norm::kUnit;
  if (vec && units <= 2048) {
    // Two units a lane, or one of fp32, whose rows take twice the registers.
    constexpr int NV = XT == PCB_DTYPE_F32 ? 1 : 2;
    if (units <= 32) return launch_norm_bwd<XT, 32, 1>(p, parts, s);
    if (units <= 64) return launch_norm_bwd<XT, 64 / NV, NV>(p, parts, s);
    if (units <= 128) return launch_norm_bwd<XT, 128 / NV, NV>(p, parts, s);
    if (units <= 256) return launch_norm_bwd<XT, 256 / NV, NV>(p, parts, s);
    if (units <= 512) return launch_norm_bwd<XT, 512 / NV, NV>(p, parts, s);
    if constexpr (XT == PCB_DTYPE_F32) {
      if (units <= 1024) return launch_norm_bwd<XT, 1024, 1>(p, parts, s);
      return launch_norm_bwd<XT, 1024, 2>(p, parts, s);
    } else {
      if (units <= 1024) return launch_norm_bwd<XT, 512, 2>(p, parts, s);
      return launch_norm_bwd_staged<XT, 4>(p, parts, s);
    }
  }
  const bool same = p.w_dtype == XT, f32 = p.w_dtype == PCB_DTYPE_F32;
  if ((same && launch_norm_bwd_elems<XT, XT>(p, parts, s)) ||
      (!same && f32 && launch_norm_bwd_elems<XT, PCB_DTYPE_F32>(p, parts, s)))
    return check_launch("rms_norm_bwd_elems_kernel");
  parts = norm_bwd_ctas(p.rows, 1, kNormBwdMost);
  const bool in_smem = (int64_t)p.dim * 4 <= kNormDwSmem;
  const int smem = in_smem ? p.dim * 4 : 0;
  auto kernel = norm::rms_norm_bwd_generic_kernel<XT>;
  if (smem > 48 * 1024) ensure_smem_attr(kernel, smem);
  kernel<<<parts, norm::kGenericThreads, smem, s>>>(p, in_smem ? 1 : 0);
  return check_launch("rms_norm_bwd_generic_kernel");
}

int norm_bad_sizes(int64_t rows, int64_t dim) {
  if (rows < 0 || dim <= 0) return fail(PCB_ERR_INVALID, "rms norm needs rows >= 0 and dim > 0");
  if (rows > INT32_MAX || dim > (1 << 26)) return fail(PCB_ERR_UNSUPPORTED, "rms norm: dimension too large");
  return PCB_OK;
}

}  // namespace

extern "C" {

int pcb_rms_norm_fwd(const void* x, int x_dtype, int64_t rows, int64_t dim, int64_t sx, const void* residual,
                     int64_t sr, const void* weight, int w_dtype, float eps, void* h, int64_t sh, void* y, int64_t sy,
                     void* q, int q_dtype, int64_t sq, float* scale, int64_t ssr, int64_t ssb, int quant_mode,
                     int pow2_scales, float quant_eps, float* rstd, void* stream) {
  if (int st = norm_bad_sizes(rows, dim)) return st;
  if (!is_float_in(x_dtype) || !is_float_in(w_dtype)) return fail(PCB_ERR_INVALID, "rms norm: bad dtype");
  if (quant_mode < norm::kQuantNone || quant_mode > norm::kQuantRow)
    return fail(PCB_ERR_INVALID, "rms norm: quant_mode must be 0 (none), 1 (1x128 blocks) or 2 (rows)");
  if (quant_mode != norm::kQuantNone && !is_fp8(q_dtype)) return fail(PCB_ERR_INVALID, "rms norm: q must be E4M3 or E5M2");
  if (pow2_scales && quant_mode != norm::kQuantBlock)
    return fail(PCB_ERR_UNSUPPORTED, "rms norm: power-of-two scales go with 1x128 blocks");
  if (quant_mode == norm::kQuantNone && !y) return fail(PCB_ERR_INVALID, "rms norm: neither y nor q is wanted");
  if (rows == 0) return PCB_OK;
  if (!x || !weight || !rstd || (residual && !h) || (quant_mode != norm::kQuantNone && (!q || !scale)))
    return fail(PCB_ERR_INVALID, "null pointer");
  const norm::FwdArgs p{x, sx, residual, sr, weight, w_dtype, residual ? h : nullptr, sh, y, sy,
                        quant_mode == norm::kQuantNone ? nullptr : q, sq, scale, ssr, ssb, rstd, rows, (int)dim, eps,
                        quant_eps, quant_mode, pow2_scales ? 1 : 0};
  const int es = elem_size(x_dtype);
  const bool vec = dim % norm::kUnit == 0 && fits_units(x, sx, es) && (!residual || (fits_units(residual, sr, es) && fits_units(h, sh, es))) &&
                   aligned(weight, 16) && (!y || fits_units(y, sy, es)) &&
                   (quant_mode == norm::kQuantNone || (aligned(q, 8) && sq % 8 == 0));
  return dispatch_xy(x_dtype, quant_mode == norm::kQuantNone ? PCB_DTYPE_E4M3 : q_dtype, [&](auto xc, auto yc) -> int {
    return dispatch_norm_fwd<decltype(xc)::value, decltype(yc)::value>(p, vec, (cudaStream_t)stream);
  });
}

int64_t pcb_rms_norm_bwd_workspace_bytes(int64_t rows, int64_t dim) {
  if (rows <= 0 || dim <= 0) return 0;
  return (int64_t)norm_bwd_ctas(rows, 1, kNormBwdMost) * dim * 4;
}

int pcb_rms_norm_bwd(const void* dy, int64_t sdy, const void* h, int64_t sh, int x_dtype, int64_t rows, int64_t dim,
                     const void* dh, int64_t sdh, const void* weight, int w_dtype, const float* rstd, void* dx,
                     int64_t sdx, void* dw, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int st = norm_bad_sizes(rows, dim)) return st;
  if (!is_float_in(x_dtype) || !is_float_in(w_dtype)) return fail(PCB_ERR_INVALID, "rms norm: bad dtype");
  if (!dw) return fail(PCB_ERR_INVALID, "null pointer");
  cudaStream_t s = (cudaStream_t)stream;
  if (rows == 0) {
    if (cudaMemsetAsync(dw, 0, (size_t)dim * elem_size(w_dtype), s) != cudaSuccess) return check_launch("rms norm dw");
    return PCB_OK;
  }
  if (!dy || !h || !weight || !rstd || !dx) return fail(PCB_ERR_INVALID, "null pointer");
  if (!workspace || !aligned(workspace, 16) || workspace_bytes < pcb_rms_norm_bwd_workspace_bytes(rows, dim))
    return fail(PCB_ERR_INVALID, "rms norm workspace too small or misaligned");
  const norm::BwdArgs p{dy, sdy, h, sh, dh, sdh, weight, w_dtype, rstd, dx, sdx, static_cast<float*>(workspace), rows,
                        (int)dim};
  const int es = elem_size(x_dtype);
  const bool vec = dim % norm::kUnit == 0 && fits_units(dy, sdy, es) && fits_units(h, sh, es) &&
                   (!dh || fits_units(dh, sdh, es)) && fits_units(dx, sdx, es) && aligned(weight, 16);
  int parts = 0;
  int st = x_dtype == PCB_DTYPE_F32   ? dispatch_norm_bwd<PCB_DTYPE_F32>(p, vec, parts, s)
           : x_dtype == PCB_DTYPE_F16 ? dispatch_norm_bwd<PCB_DTYPE_F16>(p, vec, parts, s)
                                      : dispatch_norm_bwd<PCB_DTYPE_BF16>(p, vec, parts, s);
  if (st) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((dim + 31) / 32), 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const float* partial = p.partial;
  if (w_dtype == PCB_DTYPE_F32) cudaLaunchKernelEx(&cfg, norm::rms_norm_dw_kernel<PCB_DTYPE_F32>, partial, parts, (int)dim, dw);
  else if (w_dtype == PCB_DTYPE_F16) cudaLaunchKernelEx(&cfg, norm::rms_norm_dw_kernel<PCB_DTYPE_F16>, partial, parts, (int)dim, dw);
  else cudaLaunchKernelEx(&cfg, norm::rms_norm_dw_kernel<PCB_DTYPE_BF16>, partial, parts, (int)dim, dw);
  return check_launch("rms_norm_dw_kernel");
}

}  // extern "C"
