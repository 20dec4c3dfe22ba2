// Root-mean-square norm with the residual's addition and an FP8 output, and
// its backward pass.
//
//   h = T(x + r)  (T: the input type; h is the residual that later layers read,
//                  and the norm is that of h as it is held)
//   s = 1 / sqrt(mean_j h_j^2 + eps),   y_j = h_j s w_j
//   q = sat(y f), f = fp8_max / max(amax, quant_eps) per 1x128 block or per row
//   backward, n = h s:  dx_j = s (w_j dy_j - n_j mean_k(n_k w_k dy_k)) + dh_j,
//                       dw_j = sum_rows dy_j n_j
//
// Everything between the loads and the one rounding of each output is fp32.
#pragma once

#include "common.cuh"

namespace pcb {
namespace norm {

enum QuantMode : int { kQuantNone = 0, kQuantBlock = 1, kQuantRow = 2 };
constexpr int kQuantCols = 128;  // columns of a quantization block
constexpr int kUnit = 8;         // elements of one row that a lane handles at a time
constexpr int kGenericThreads = 256;

struct FwdArgs {
  const void* x;
  long long sx;
  const void* res;  // null: no residual, h is x
  long long sr;
  const void* w;
  int w_dtype;
  void* h;  // null without a residual
  long long sh;
  void* y;  // null: not wanted
  long long sy;
  void* q;  // null with kQuantNone
  long long sq;
  float* scale;
  long long ssr, ssb;
  float* rstd;
  long long rows;
  int dim;
  float eps, quant_eps;
  int quant_mode, pow2;
};

struct BwdArgs {
  const void* dy;
  long long sdy;
  const void* h;
  long long sh;
  const void* dh;  // gradient of the residual output, or null
  long long sdh;
  const void* w;
  int w_dtype;
  const float* rstd;
  void* dx;
  long long sdx;
  float* partial;  // [gridDim.x][dim]: each CTA's share of dw
  long long rows;
  int dim;
};

// Eight consecutive elements as fp32.  off is in elements and 16-byte aligned.
template <typename T>
struct Raw8;
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void unpack(float (&f)[8]) const {
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
  __device__ __forceinline__ void pack(const float (&f)[8]) {
    a = make_float4(f[0], f[1], f[2], f[3]);
    b = make_float4(f[4], f[5], f[6], f[7]);
  }
  __device__ __forceinline__ void store(float* p) const {
    *reinterpret_cast<float4*>(p) = a;
    *reinterpret_cast<float4*>(p + 4) = b;
  }
};
template <typename T, typename T2, T2 (*FROM2)(float, float), float2 (*TO2)(T2)>
struct Raw8Half {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void unpack(float (&f)[8]) const {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = TO2(*reinterpret_cast<const T2*>(&u[i]));
      f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
  }
  __device__ __forceinline__ void pack(const float (&f)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T2 t = FROM2(f[2 * i], f[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
    v = make_uint4(u[0], u[1], u[2], u[3]);
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = v; }
};
__device__ __forceinline__ __nv_bfloat162 from2_bf16(float a, float b) { return __floats2bfloat162_rn(a, b); }
__device__ __forceinline__ float2 to2_bf16(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ __half2 from2_f16(float a, float b) { return __floats2half2_rn(a, b); }
__device__ __forceinline__ float2 to2_f16(__half2 v) { return __half22float2(v); }
template <>
struct Raw8<__nv_bfloat16> : Raw8Half<__nv_bfloat16, __nv_bfloat162, from2_bf16, to2_bf16> {};
template <>
struct Raw8<__half> : Raw8Half<__half, __half2, from2_f16, to2_f16> {};

__device__ __forceinline__ float load1(const void* p, int dt, long long i) {
  if (dt == PCB_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dt == PCB_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The weight of columns [8u, 8u + 8); its type may differ from x's.
__device__ __forceinline__ void load_weight(const void* w, int dt, int u, float (&f)[8]) {
  if (dt == PCB_DTYPE_F32) {
    Raw8<float> r;
    r.load(static_cast<const float*>(w) + u * kUnit);
    r.unpack(f);
  } else if (dt == PCB_DTYPE_BF16) {
    Raw8<__nv_bfloat16> r;
    r.load(static_cast<const __nv_bfloat16*>(w) + u * kUnit);
    r.unpack(f);
  } else {
    Raw8<__half> r;
    r.load(static_cast<const __half*>(w) + u * kUnit);
    r.unpack(f);
  }
}

// Sum and unsigned maximum over a warp's groups of LANES lanes; every lane
// gets the result, formed in the same order.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int LANES>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  if constexpr (LANES == 32) {
    return __reduce_max_sync(0xffffffffu, v);
  } else {
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }
}
// The same over the CTA, in one barrier; `red` is not used again.
struct CtaRed {
  float sum[32];
  uint32_t top[32];
};
__device__ __forceinline__ void cta_sum_max(float& v, uint32_t& top, CtaRed& red) {
  v = lanes_sum<32>(v);
  top = lanes_max<32>(top);
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) red.sum[warp] = v, red.top[warp] = top;
  __syncthreads();
  v = 0.f, top = 0;
  for (int i = 0; i < warps; ++i) v += red.sum[i], top = max(top, red.top[i]);
}
// For loops over rows: two barriers, `red` can be used again.
template <int THREADS>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = lanes_sum<32>(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) v += red[i];
  __syncthreads();
  return v;
}
template <int THREADS>
__device__ __forceinline__ uint32_t row_max(uint32_t v, float* red) {
  uint32_t* r = reinterpret_cast<uint32_t*>(red);
  v = lanes_max<32>(v);
  if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) v = max(v, r[i]);
  __syncthreads();
  return v;
}

// max(|m|, |a|, |b|), NaN if any of them is.
__device__ __forceinline__ float max3_abs(float m, float a, float b) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(a), "f"(b));
  return r;
}
// f s w of eight elements.
__device__ __forceinline__ void scale8(float (&f)[8], float s, const float (&w)[8]) {
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    const float2 t = __fmul2_rn(__fmul2_rn(make_float2(f[k], f[k + 1]), make_float2(s, s)), make_float2(w[k], w[k + 1]));
    f[k] = t.x, f[k + 1] = t.y;
  }
}
__device__ __forceinline__ float max8_abs(float m, const float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 8; k += 2) m = max3_abs(m, f[k], f[k + 1]);
  return m;
}

// 1 / sqrt(mean + eps), correctly rounded: an error here would move a whole
// row across the FP8 grid's ties.
__device__ __forceinline__ float rstd_of(float sum, int dim, float eps) {
  return __frsqrt_rn(__fdiv_rn(sum, (float)dim) + eps);
}

// The factor that takes y to the FP8 grid and the scale that takes it back:
// the arithmetic of the per-block and the per-row quantizers.
template <int YT>
__device__ __forceinline__ float quant_factor(uint32_t amax_bits, const FwdArgs& p, float& scale) {
  const float safe = clamp_min_eps(__uint_as_float(amax_bits), p.quant_eps);
  const float f = p.pow2 ? pow2_quant_scale(safe, Fp8Max<YT>::value) : quant_scale_from_amax(safe, Fp8Max<YT>::value);
  scale = p.quant_mode == kQuantRow ? __fdiv_rn(safe, Fp8Max<YT>::value) : __frcp_rn(f);
  return f;
}

// Forward, the whole row in registers (NV units of eight elements a lane): one
// reading of x and r, one writing of each output.  A row is LANES (16 or 32)
// lanes of a warp, or with LANES == 0 a CTA of as many threads as the width needs.
// Sixteen lanes hold one 128-column block, so its amax is a shuffle.  A row's
// scale needs max |h s w|, taken as s max |h w| so that the one barrier of the sum
// serves it too.  A CTA ends with its row: many rows at once hide a row's way
// through its loads, sum and stores better than resident CTAs that load the next
// row ahead (16384 x 4096 bf16 on a B200, every output: 98 us against 116; weights
// loaded with the row instead of where they are used, which costs registers: 122).
// Bound by HBM traffic where all outputs are wanted (606 MB in 98 us, 6.2 TB/s), by
// instruction issue where one FP8 byte is written for two bytes read.
template <int XT, int YT, int LANES, int NV, int MAX_THREADS, bool RES>
__global__ void __launch_bounds__(MAX_THREADS) rms_norm_fwd_kernel(const FwdArgs p) {
  using T = typename InType<XT>::T;
  constexpr int ROWS = LANES ? MAX_THREADS / (LANES ? LANES : 1) : 1;  // per CTA
  const int lanes = LANES ? LANES : (int)blockDim.x;
  const int lane = LANES ? (int)threadIdx.x % (LANES ? LANES : 1) : (int)threadIdx.x;
  const long long row = (long long)blockIdx.x * ROWS + (LANES ? threadIdx.x / (LANES ? LANES : 1) : 0);
  const bool live = row < p.rows;  // the lanes of a warp stay together for its shuffles
  const int units = live ? p.dim / kUnit : 0;
  Raw8<T> hv[NV], rv[RES ? NV : 1];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = lane + i * lanes;
    hv[i].zero();
    if (RES) rv[RES ? i : 0].zero();
    if (u < units) {
      hv[i].load(static_cast<const T*>(p.x) + row * p.sx + u * kUnit);
      if (RES && p.res) rv[RES ? i : 0].load(static_cast<const T*>(p.res) + row * p.sr + u * kUnit);
    }
  }
  float2 ss2 = make_float2(0.f, 0.f);
  float top_hw = 0.f;  // max |h w|, for a row's scale
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = lane + i * lanes;
    float f[8];
    hv[i].unpack(f);
    if (RES && p.res) {  // tested although it always holds: without it ptxas gives the loads more registers (133 us, not 97)
      float g[8];
      rv[RES ? i : 0].unpack(g);
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        const float2 t = __fadd2_rn(make_float2(f[k], f[k + 1]), make_float2(g[k], g[k + 1]));
        f[k] = t.x, f[k + 1] = t.y;
      }
      hv[i].pack(f);  // rounded to T: the residual that later layers read
      hv[i].unpack(f);
      if (u < units) hv[i].store(static_cast<T*>(p.h) + row * p.sh + u * kUnit);
    }
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      const float2 t = make_float2(f[k], f[k + 1]);
      ss2 = __ffma2_rn(t, t, ss2);
    }
    if (p.quant_mode == kQuantRow && u < units) {
      float w[8];
      load_weight(p.w, p.w_dtype, u, w);
      #pragma unroll
      for (int k = 0; k < 8; ++k) f[k] *= w[k];
      top_hw = max8_abs(top_hw, f);
    }
  }
  float ss = ss2.x + ss2.y;
  uint32_t top = abs_bits(top_hw);
  if constexpr (LANES == 0) {
    __shared__ CtaRed red;
    cta_sum_max(ss, top, red);
  } else {
    ss = lanes_sum<LANES ? LANES : 32>(ss);
    if (p.quant_mode == kQuantRow) top = lanes_max<LANES ? LANES : 32>(top);
  }
  const float rstd = rstd_of(ss, p.dim, p.eps);
  if (live && lane == 0) p.rstd[row] = rstd;

  float factor = 0.f;
  if (p.quant_mode == kQuantRow) {
    float scale;
    factor = quant_factor<YT>(abs_bits(__uint_as_float(top) * rstd), p, scale);
    if (live && lane == 0) p.scale[row * p.ssr] = scale;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = lane + i * lanes;
    const bool in = u < units;
    float f[8];
    float m = 0.f;
    if (in) {
      float w[8];
      hv[i].unpack(f);
      load_weight(p.w, p.w_dtype, u, w);
      scale8(f, rstd, w);
      m = max8_abs(0.f, f);
      if (p.y) {
        Raw8<T> o;
        o.pack(f);
        o.store(static_cast<T*>(p.y) + row * p.sy + u * kUnit);
      }
    }
    if (p.quant_mode == kQuantNone) continue;
    if (p.quant_mode == kQuantBlock) {
      float scale;
      factor = quant_factor<YT>(lanes_max<16>(abs_bits(m)), p, scale);
      if (in && (lane & 15) == 0) p.scale[row * p.ssr + (long long)(u >> 4) * p.ssb] = scale;
    }
    if (in) {
      uint32_t q[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 t = __fmul2_rn(make_float2(f[2 * k], f[2 * k + 1]), make_float2(factor, factor));
        q[k] = cvt2_fp8<YT>(t.x, t.y);
      }
      const uint2 o = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.q) + row * p.sq + u * kUnit) = o;
    }
  }
}

// The same element by element, for rows that do not suit 16-byte loads (odd
// widths, strides or alignments): a thread holds the columns t, t + threads, ...
// (NE of them at most), so every access of a warp is contiguous and all of a row's loads
// are in flight together.  A row is a warp's (widths up to 32 NE) or a CTA's,
// whose threads are a multiple of 128: four warps hold a 128-column block.
constexpr int kElems = 16;
// WT is the weight's type: x's or fp32.
template <int XT, int YT, int WT, bool WARP, int NE, int MAX_THREADS>
__global__ void __launch_bounds__(MAX_THREADS) rms_norm_fwd_elems_kernel(const FwdArgs p) {
  using T = typename InType<XT>::T;
  using W = typename InType<WT>::T;
  const int threads = WARP ? 32 : (int)blockDim.x;
  const int t = WARP ? (int)threadIdx.x & 31 : (int)threadIdx.x;
  const long long row = WARP ? (long long)blockIdx.x * (MAX_THREADS / 32) + (threadIdx.x >> 5) : (long long)blockIdx.x;
  if (row >= p.rows) return;  // a whole warp, or nobody
  const T* x = static_cast<const T*>(p.x) + row * p.sx;
  T raw[NE], res[NE];
  W w[NE];
#pragma unroll
  for (int k = 0; k < NE; ++k) {
    const int c = t + k * threads;
    raw[k] = res[k] = from_f32<T>(0.f);
    w[k] = from_f32<W>(0.f);
    if (c < p.dim) {
      raw[k] = x[c];
      w[k] = static_cast<const W*>(p.w)[c];
      if (p.res) res[k] = static_cast<const T*>(p.res)[row * p.sr + c];
    }
  }
  float f[NE];
  float ss = 0.f;
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < NE; ++k) {
    const int c = t + k * threads;
    f[k] = InType<XT>::to_f32(raw[k]);
    if (p.res) {
      const T h = from_f32<T>(f[k] + InType<XT>::to_f32(res[k]));
      f[k] = InType<XT>::to_f32(h);
      if (c < p.dim) static_cast<T*>(p.h)[row * p.sh + c] = h;
    }
    ss = fmaf(f[k], f[k], ss);
    if (p.quant_mode == kQuantRow) top = max(top, abs_bits(f[k] * InType<WT>::to_f32(w[k])));
  }
  if constexpr (WARP) {
    ss = lanes_sum<32>(ss);
    top = lanes_max<32>(top);
  } else {
    __shared__ CtaRed red;
    cta_sum_max(ss, top, red);
  }
  const float rstd = rstd_of(ss, p.dim, p.eps);
  if (t == 0) p.rstd[row] = rstd;
#pragma unroll
  for (int k = 0; k < NE; ++k) {
    const int c = t + k * threads;
    f[k] = f[k] * rstd * InType<WT>::to_f32(w[k]);
    if (p.y && c < p.dim) static_cast<T*>(p.y)[row * p.sy + c] = from_f32<T>(f[k]);
  }
  if (p.quant_mode == kQuantNone) return;
  uint8_t* q = static_cast<uint8_t*>(p.q) + row * p.sq;
  if (p.quant_mode == kQuantRow) {
    float scale;
    const float factor = quant_factor<YT>(abs_bits(__uint_as_float(top) * rstd), p, scale);
    if (t == 0) p.scale[row * p.ssr] = scale;
#pragma unroll
    for (int k = 0; k < NE; ++k)
      if (t + k * threads < p.dim) q[t + k * threads] = cvt1_fp8<YT>(__fmul_rn(f[k], factor));
    return;
  }
  if constexpr (WARP) {
#pragma unroll
    for (int b = 0; b < NE / 4; ++b) {  // a warp's four columns a lane
      uint32_t amax = 0;
#pragma unroll
      for (int k = 4 * b; k < 4 * b + 4; ++k)
        if (t + k * 32 < p.dim) amax = max(amax, abs_bits(f[k]));
      if (b * kQuantCols >= p.dim) break;
      float scale;
      const float factor = quant_factor<YT>(lanes_max<32>(amax), p, scale);
      if (t == 0) p.scale[row * p.ssr + (long long)b * p.ssb] = scale;
#pragma unroll
      for (int k = 4 * b; k < 4 * b + 4; ++k)
        if (t + k * 32 < p.dim) q[t + k * 32] = cvt1_fp8<YT>(__fmul_rn(f[k], factor));
    }
  } else {
    // Block b of the row: the four warps 4 (b % groups) .. + 3 in pass b / groups.
    __shared__ uint32_t tops[NE][MAX_THREADS / 32];
    __shared__ float factors[NE * MAX_THREADS / 128];
    const int warp = t >> 5, groups = threads / 128;
#pragma unroll
    for (int k = 0; k < NE; ++k) {
      const uint32_t m = lanes_max<32>(t + k * threads < p.dim ? abs_bits(f[k]) : 0u);
      if ((t & 31) == 0) tops[k][warp] = m;
    }
    __syncthreads();
    for (int b = t; b * kQuantCols < p.dim; b += threads) {
      const uint32_t* m = tops[b / groups] + 4 * (b % groups);
      float scale;
      factors[b] = quant_factor<YT>(max(max(m[0], m[1]), max(m[2], m[3])), p, scale);
      p.scale[row * p.ssr + (long long)b * p.ssb] = scale;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NE; ++k) {
      const int c = t + k * threads;
      if (c < p.dim) q[c] = cvt1_fp8<YT>(__fmul_rn(f[k], factors[k * groups + (warp >> 2)]));
    }
  }
}

// Forward for rows too wide for registers: one CTA per row, element by
// element, h read again (from L1 / L2) for each pass over the row.
template <int XT, int YT>
__global__ void __launch_bounds__(kGenericThreads) rms_norm_fwd_generic_kernel(const FwdArgs p) {
  using T = typename InType<XT>::T;
  __shared__ float red[kGenericThreads / 32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.sx;
    const T* h = x;
    float ss = 0.f;
    if (p.res) {
      const T* r = static_cast<const T*>(p.res) + row * p.sr;
      T* ho = static_cast<T*>(p.h) + row * p.sh;
      for (int c = t; c < p.dim; c += kGenericThreads) {
        const T v = from_f32<T>(InType<XT>::to_f32(x[c]) + InType<XT>::to_f32(r[c]));
        ho[c] = v;
        const float f = InType<XT>::to_f32(v);
        ss = fmaf(f, f, ss);
      }
      h = ho;  // other threads read it after the barriers of row_sum
    } else {
      for (int c = t; c < p.dim; c += kGenericThreads) {
        const float f = InType<XT>::to_f32(x[c]);
        ss = fmaf(f, f, ss);
      }
    }
    const float rstd = rstd_of(row_sum<kGenericThreads>(ss, red), p.dim, p.eps);
    if (t == 0) p.rstd[row] = rstd;
    auto value = [&](int c) { return InType<XT>::to_f32(h[c]) * rstd * load1(p.w, p.w_dtype, c); };
    auto store_q = [&](int c, float v, float factor) {
      static_cast<uint8_t*>(p.q)[row * p.sq + c] = cvt1_fp8<YT>(__fmul_rn(v, factor));
    };
    T* y = p.y ? static_cast<T*>(p.y) + row * p.sy : nullptr;
    if (p.quant_mode == kQuantBlock) {
      // A warp per 128-column block, four columns a lane.
      for (int b = warp; b * kQuantCols < p.dim; b += kGenericThreads / 32) {
        float f[4];
        uint32_t amax = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = b * kQuantCols + k * 32 + lane;
          f[k] = c < p.dim ? value(c) : 0.f;
          amax = max(amax, abs_bits(f[k]));
        }
        amax = __reduce_max_sync(0xffffffffu, amax);
        float scale;
        const float factor = quant_factor<YT>(amax, p, scale);
        if (lane == 0) p.scale[row * p.ssr + (long long)b * p.ssb] = scale;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = b * kQuantCols + k * 32 + lane;
          if (c < p.dim) {
            store_q(c, f[k], factor);
            if (y) y[c] = from_f32<T>(f[k]);
          }
        }
      }
    } else {
      float factor = 0.f;
      if (p.quant_mode == kQuantRow) {
        uint32_t amax = 0;
        for (int c = t; c < p.dim; c += kGenericThreads) amax = max(amax, abs_bits(value(c)));
        float scale;
        factor = quant_factor<YT>(row_max<kGenericThreads>(amax, red), p, scale);
        if (t == 0) p.scale[row * p.ssr] = scale;
      }
      for (int c = t; c < p.dim; c += kGenericThreads) {
        const float v = value(c);
        if (y) y[c] = from_f32<T>(v);
        if (p.quant_mode == kQuantRow) store_q(c, v, factor);
      }
    }
    __syncthreads();  // red is reused by the next row
  }
}

// Backward, one row per LANES threads at a time, rows handed out in strides of
// the grid.  A lane keeps its columns' weights and its share of dw in
// registers over all rows; the CTA's shares are joined in shared memory and
// written to partial[blockIdx.x], which rms_norm_dw_kernel sums in a fixed
// order.  Bound by HBM traffic (dy, h, dh read once, dx written once); the next
// row's values are loaded before this row's are used, so that a row's sum, which
// all of its threads wait for, does not leave the memory idle.
template <int XT, int LANES, int NV>
__global__ void __launch_bounds__(LANES > 256 ? LANES : 256, LANES > 256 ? 1 : 2) rms_norm_bwd_kernel(const BwdArgs p) {
  using T = typename InType<XT>::T;
  constexpr int THREADS = LANES > 256 ? LANES : 256;
  constexpr int ROWS = THREADS / LANES;  // rows in flight per CTA
  constexpr int WARPS = LANES / 32;      // warps per row
  constexpr bool ROOMY = LANES < 1024;   // 1024 threads have 64 registers each: the weight is read again, no row ahead
  extern __shared__ float dw_shared[];   // [dim] when ROWS > 1
  __shared__ float red[2][THREADS / 32];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int units = p.dim / kUnit;
  float w_reg[ROOMY ? NV : 1][8], dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = lane + i * LANES;
#pragma unroll
    for (int k = 0; k < 8; ++k) dw[i][k] = 0.f;
    if constexpr (ROOMY) {
#pragma unroll
      for (int k = 0; k < 8; ++k) w_reg[i][k] = 0.f;
      if (u < units) load_weight(p.w, p.w_dtype, u, w_reg[i]);
    }
  }
  auto weight = [&](int i, float (&w)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = ROOMY ? w_reg[ROOMY ? i : 0][k] : 0.f;
    if (!ROOMY && lane + i * LANES < units) load_weight(p.w, p.w_dtype, lane + i * LANES, w);
  };
  const float inv_dim = 1.f / (float)p.dim;
  int turn = 0;
  Raw8<T> dyv[NV], hv[NV], dhv[NV];
  float rstd = 0.f;
  auto load_row = [&](long long row, Raw8<T>(&a)[NV], Raw8<T>(&b)[NV], Raw8<T>(&c)[NV], float& s) {
    const bool live = row < p.rows;
    s = live ? __ldg(p.rstd + row) : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = lane + i * LANES;
      a[i].zero(), b[i].zero(), c[i].zero();
      if (live && u < units) {
        a[i].load(static_cast<const T*>(p.dy) + row * p.sdy + u * kUnit);
        b[i].load(static_cast<const T*>(p.h) + row * p.sh + u * kUnit);
        if (p.dh) c[i].load(static_cast<const T*>(p.dh) + row * p.sdh + u * kUnit);
      }
    }
  };
  const long long step = (long long)gridDim.x * ROWS;
  if (ROOMY) load_row((long long)blockIdx.x * ROWS + group, dyv, hv, dhv, rstd);
  // Every group of the CTA takes the same number of turns, since the sums of
  // rows wider than a warp meet at a CTA barrier.
  for (long long row0 = (long long)blockIdx.x * ROWS; row0 < p.rows; row0 += step, turn ^= 1) {
    const long long row = row0 + group;
    const bool live = row < p.rows;
    Raw8<T> dy_next[NV], h_next[NV], dh_next[NV];
    float rstd_next = 0.f;
    if (ROOMY) load_row(row + step, dy_next, h_next, dh_next, rstd_next);
    else load_row(row, dyv, hv, dhv, rstd);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float a[8], b[8], w[8];
      dyv[i].unpack(a);
      hv[i].unpack(b);
      weight(i, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float n = b[k] * rstd;
        dot = fmaf(n, a[k] * w[k], dot);
        dw[i][k] = fmaf(a[k], n, dw[i][k]);
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if constexpr (LANES > 32) {
      // Two buffers in turn: one barrier a row is enough.
      float* r = red[turn];
      if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = dot;
      __syncthreads();
      dot = 0.f;
#pragma unroll
      for (int i = 0; i < WARPS; ++i) dot += r[group * WARPS + i];
    }
    const float mean = dot * inv_dim;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = lane + i * LANES;
      if (!live || u >= units) continue;
      float a[8], b[8], d[8], w[8];
      dyv[i].unpack(a);
      hv[i].unpack(b);
      dhv[i].unpack(d);
      weight(i, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float v = rstd * (a[k] * w[k] - b[k] * rstd * mean);
        d[k] = p.dh ? v + d[k] : v;
      }
      Raw8<T> o;
      o.pack(d);
      o.store(static_cast<T*>(p.dx) + row * p.sdx + u * kUnit);
    }
    if (ROOMY) {
#pragma unroll
      for (int i = 0; i < NV; ++i) dyv[i] = dy_next[i], hv[i] = h_next[i], dhv[i] = dh_next[i];
      rstd = rstd_next;
    }
  }
  float* out = p.partial + (long long)blockIdx.x * p.dim;
  if constexpr (ROWS == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = lane + i * LANES;
      if (u < units) {
        Raw8<float> o;
        o.pack(dw[i]);
        o.store(out + u * kUnit);
      }
    }
  } else {
    // The groups add their shares one after the other: a fixed order.
    for (int gi = 0; gi < ROWS; ++gi) {
      __syncthreads();
      if (group == gi) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int u = lane + i * LANES;
          if (u >= units) continue;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            dw_shared[u * kUnit + k] = gi == 0 ? dw[i][k] : dw_shared[u * kUnit + k] + dw[i][k];
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.dim; c += THREADS) out[c] = dw_shared[c];
  }
}

// Backward for 16-bit rows whose values, with a row ahead, are too many for
// registers: one row per CTA at a time, two rows in shared memory, each thread
// copying (cp.async) and reading its own units of them, so that a row needs no
// barrier but that of its sum and the next one is on its way meanwhile.  4096 x
// 16384 bf16 on a B200: 110 us (4.9 TB/s), against 183 us with 1024 threads that
// read each row when they come to it, and 110 us with 1024 threads here.  Rows up to
// 8192 wide stay in registers (8192 x 8192: 97 us, 130 us here), and fp32 ones
// up to that width are faster read by 1024 threads (4096 x 8192: 112 and 151 us).
constexpr int kStagedThreads = 512;
constexpr int kStagedBytes = 2 * 3 * 16;  // of shared memory, per unit of the row
template <int XT, int NV>
__global__ void __launch_bounds__(kStagedThreads, 1) rms_norm_bwd_staged_kernel(const BwdArgs p) {
  using T = typename InType<XT>::T;
  static_assert(sizeof(T) == 2, "a unit is one 16-byte copy");
  extern __shared__ uint4 stage[];  // [2][dy, h, dh][units]
  __shared__ float red[2][kStagedThreads / 32];
  const int t = threadIdx.x, units = p.dim / kUnit;
  float w[NV][8], dw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = t + i * kStagedThreads;
#pragma unroll
    for (int k = 0; k < 8; ++k) w[i][k] = dw[i][k] = 0.f;
    if (u < units) load_weight(p.w, p.w_dtype, u, w[i]);
  }
  auto fetch = [&](long long row, int s) {
    if (row < p.rows) {
      const T* src[3] = {static_cast<const T*>(p.dy) + row * p.sdy, static_cast<const T*>(p.h) + row * p.sh,
                         p.dh ? static_cast<const T*>(p.dh) + row * p.sdh : nullptr};
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int u = t + i * kStagedThreads;
        if (u >= units) continue;
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          if (j == 2 && !p.dh) continue;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(stage + (s * 3 + j) * units + u)),
                       "l"(src[j] + u * kUnit)
                       : "memory");
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto value = [&](int s, int j, int u, float (&f)[8]) {
    Raw8<T> r;
    r.v = stage[(s * 3 + j) * units + u];
    r.unpack(f);
  };
  const float inv_dim = 1.f / (float)p.dim;
  int s = 0;
  fetch(blockIdx.x, 0);
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, s ^= 1) {
    fetch(row + gridDim.x, s ^ 1);
    const float rstd = __ldg(p.rstd + row);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = t + i * kStagedThreads;
      if (u >= units) continue;
      float a[8], b[8];
      value(s, 0, u, a);
      value(s, 1, u, b);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float n = b[k] * rstd;
        dot = fmaf(n, a[k] * w[i][k], dot);
        dw[i][k] = fmaf(a[k], n, dw[i][k]);
      }
    }
    dot = lanes_sum<32>(dot);
    // Two buffers in turn: one barrier a row is enough.
    if ((t & 31) == 0) red[s][t >> 5] = dot;
    __syncthreads();
    dot = 0.f;
#pragma unroll
    for (int i = 0; i < kStagedThreads / 32; ++i) dot += red[s][i];
    const float mean = dot * inv_dim;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = t + i * kStagedThreads;
      if (u >= units) continue;
      float a[8], b[8], d[8];
      value(s, 0, u, a);
      value(s, 1, u, b);
      if (p.dh) value(s, 2, u, d);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float v = rstd * (a[k] * w[i][k] - b[k] * rstd * mean);
        d[k] = p.dh ? v + d[k] : v;
      }
      Raw8<T> o;
      o.pack(d);
      o.store(static_cast<T*>(p.dx) + row * p.sdx + u * kUnit);
    }
  }
  float* out = p.partial + (long long)blockIdx.x * p.dim;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = t + i * kStagedThreads;
    if (u >= units) continue;
    Raw8<float> o;
    o.pack(dw[i]);
    o.store(out + u * kUnit);
  }
}

// Backward element by element, for rows that do not suit 16-byte loads: as in
// the forward, a thread holds the columns t, t + threads, ... with their share of
// dw, over all rows of its warp (widths up to 32 NE) or CTA.
template <int XT, int WT, bool WARP, int NE, int MAX_THREADS>
__global__ void __launch_bounds__(MAX_THREADS) rms_norm_bwd_elems_kernel(const BwdArgs p) {
  using T = typename InType<XT>::T;
  using W = typename InType<WT>::T;
  constexpr int ROWS = WARP ? MAX_THREADS / 32 : 1;
  __shared__ float red[2][MAX_THREADS / 32];
  __shared__ float dw_shared[WARP ? 32 * NE : 1];
  const int threads = WARP ? 32 : (int)blockDim.x;
  const int t = WARP ? (int)threadIdx.x & 31 : (int)threadIdx.x;
  const int group = WARP ? (int)threadIdx.x >> 5 : 0;
  const float inv_dim = 1.f / (float)p.dim;
  float dw[NE];
  W w[NE];
#pragma unroll
  for (int k = 0; k < NE; ++k) {
    dw[k] = 0.f;
    w[k] = t + k * threads < p.dim ? static_cast<const W*>(p.w)[t + k * threads] : from_f32<W>(0.f);
  }
  int turn = 0;
  for (long long row = (long long)blockIdx.x * ROWS + group; row < p.rows; row += (long long)gridDim.x * ROWS, turn ^= 1) {
    T a[NE], h[NE], d[NE];
#pragma unroll
    for (int k = 0; k < NE; ++k) {
      const int c = t + k * threads;
      a[k] = h[k] = d[k] = from_f32<T>(0.f);
      if (c < p.dim) {
        a[k] = static_cast<const T*>(p.dy)[row * p.sdy + c];
        h[k] = static_cast<const T*>(p.h)[row * p.sh + c];
        if (p.dh) d[k] = static_cast<const T*>(p.dh)[row * p.sdh + c];
      }
    }
    const float rstd = __ldg(p.rstd + row);
    float dot = 0.f;
#pragma unroll
    for (int k = 0; k < NE; ++k) {
      const float n = InType<XT>::to_f32(h[k]) * rstd, g = InType<XT>::to_f32(a[k]);  // zeros beyond the width
      dot = fmaf(n, g * InType<WT>::to_f32(w[k]), dot);
      dw[k] = fmaf(g, n, dw[k]);
    }
    dot = lanes_sum<32>(dot);
    if constexpr (!WARP) {
      // Two buffers in turn: one barrier a row is enough.
      float* r = red[turn];
      if ((t & 31) == 0) r[t >> 5] = dot;
      __syncthreads();
      dot = 0.f;
      for (int i = 0; i < threads / 32; ++i) dot += r[i];
    }
    const float mean = dot * inv_dim;
#pragma unroll
    for (int k = 0; k < NE; ++k) {
      const int c = t + k * threads;
      if (c < p.dim) {
        const float v = rstd * (InType<XT>::to_f32(a[k]) * InType<WT>::to_f32(w[k]) -
                                InType<XT>::to_f32(h[k]) * rstd * mean);
        static_cast<T*>(p.dx)[row * p.sdx + c] = from_f32<T>(p.dh ? v + InType<XT>::to_f32(d[k]) : v);
      }
    }
  }
  float* out = p.partial + (long long)blockIdx.x * p.dim;
  if constexpr (WARP) {
    // The warps add their shares one after the other: a fixed order.
    for (int g = 0; g < ROWS; ++g) {
      __syncthreads();
      if (group == g) {
#pragma unroll
        for (int k = 0; k < NE; ++k) {
          const int c = t + k * 32;
          if (c < p.dim) dw_shared[c] = g == 0 ? dw[k] : dw_shared[c] + dw[k];
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.dim; c += MAX_THREADS) out[c] = dw_shared[c];
  } else {
#pragma unroll
    for (int k = 0; k < NE; ++k)
      if (t + k * threads < p.dim) out[t + k * threads] = dw[k];
  }
}

// Backward for rows too wide for registers: a CTA per row, element by
// element.  A thread owns the columns t, t + 256, ... over all of its rows and
// keeps their share of dw in shared memory, or in its row of `partial` where
// that does not fit (the launch then asks for no shared memory).
template <int XT>
__global__ void __launch_bounds__(kGenericThreads) rms_norm_bwd_generic_kernel(const BwdArgs p, int dw_in_smem) {
  using T = typename InType<XT>::T;
  extern __shared__ float dw_shared[];
  __shared__ float red[kGenericThreads / 32];
  const int t = threadIdx.x;
  float* out = p.partial + (long long)blockIdx.x * p.dim;
  float* dw = dw_in_smem ? dw_shared : out;
  for (int c = t; c < p.dim; c += kGenericThreads) dw[c] = 0.f;
  const float inv_dim = 1.f / (float)p.dim;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* dy = static_cast<const T*>(p.dy) + row * p.sdy;
    const T* h = static_cast<const T*>(p.h) + row * p.sh;
    const T* dh = p.dh ? static_cast<const T*>(p.dh) + row * p.sdh : nullptr;
    T* dx = static_cast<T*>(p.dx) + row * p.sdx;
    const float rstd = __ldg(p.rstd + row);
    float dot = 0.f;
    for (int c = t; c < p.dim; c += kGenericThreads) {
      const float a = InType<XT>::to_f32(dy[c]), n = InType<XT>::to_f32(h[c]) * rstd;
      dot = fmaf(n, a * load1(p.w, p.w_dtype, c), dot);
      dw[c] = fmaf(a, n, dw[c]);
    }
    const float mean = row_sum<kGenericThreads>(dot, red) * inv_dim;
    for (int c = t; c < p.dim; c += kGenericThreads) {
      const float a = InType<XT>::to_f32(dy[c]), n = InType<XT>::to_f32(h[c]) * rstd;
      const float v = rstd * (a * load1(p.w, p.w_dtype, c) - n * mean);
      dx[c] = from_f32<T>(dh ? v + InType<XT>::to_f32(dh[c]) : v);
    }
  }
  if (dw_in_smem)
    for (int c = t; c < p.dim; c += kGenericThreads) out[c] = dw_shared[c];
}

// dw[c] = sum over the CTAs' shares, in a fixed order: 32 columns per CTA,
// each of the 8 warps a strided part of the rows of `partial`.
template <int WT>
__global__ void __launch_bounds__(256) rms_norm_dw_kernel(const float* partial, int parts, int dim, void* dw) {
  __shared__ float sums[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float v = 0.f;
  if (c < dim)
#pragma unroll 8
    for (int i = warp; i < parts; i += 8) v += partial[(long long)i * dim + c];
  sums[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < dim) {
#pragma unroll
    for (int i = 1; i < 8; ++i) v += sums[i][lane];
    static_cast<typename InType<WT>::T*>(dw)[c] = from_f32<typename InType<WT>::T>(v);
  }
}

}  // namespace norm
}  // namespace pcb
