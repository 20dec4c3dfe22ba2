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

// Sum / unsigned max over the LANES threads that share a row (a warp, or the
// whole CTA through `red`, one word per warp).  Every thread gets the result,
// formed in the same order.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (LANES > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < LANES / 32; ++i) v += red[i];
    __syncthreads();
  }
  return v;
}
template <int LANES>
__device__ __forceinline__ uint32_t row_max(uint32_t v, float* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (LANES > 32) {
    uint32_t* r = reinterpret_cast<uint32_t*>(red);
    if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < LANES / 32; ++i) v = max(v, r[i]);
    __syncthreads();
  }
  return v;
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

// Forward, one row per LANES threads, the whole row in registers (NV units of
// eight elements a lane): one reading of x and r, one writing of each output.
// Units 16 lanes wide are one 128-column block, so its amax is a 16-lane
// shuffle.  Bound by HBM traffic.
template <int XT, int YT, int LANES, int NV>
__global__ void __launch_bounds__(LANES > 32 ? LANES : 256) rms_norm_fwd_kernel(const FwdArgs p) {
  using T = typename InType<XT>::T;
  constexpr int ROWS = LANES > 32 ? 1 : 256 / LANES;  // rows per CTA
  __shared__ float red[32];
  const int lane = threadIdx.x % LANES;
  const long long row = (long long)blockIdx.x * ROWS + threadIdx.x / LANES;
  if (row >= p.rows) return;  // a whole warp at a time
  const int units = p.dim / kUnit;
  const T* x = static_cast<const T*>(p.x) + row * p.sx;
  const T* r = p.res ? static_cast<const T*>(p.res) + row * p.sr : nullptr;
  Raw8<T> hv[NV], rv[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = lane + i * LANES;
    if (u < units) {
      hv[i].load(x + u * kUnit);
      if (r) rv[i].load(r + u * kUnit);
    } else {
      hv[i].zero();
      rv[i].zero();
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float f[8];
    hv[i].unpack(f);
    if (r) {
      float g[8];
      rv[i].unpack(g);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] += g[k];
      hv[i].pack(f);  // rounded to T: the residual that later layers read
      hv[i].unpack(f);
      const int u = lane + i * LANES;
      if (u < units) hv[i].store(static_cast<T*>(p.h) + row * p.sh + u * kUnit);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) ss = fmaf(f[k], f[k], ss);
  }
  const float rstd = rstd_of(row_sum<LANES>(ss, red), p.dim, p.eps);
  if (lane == 0) p.rstd[row] = rstd;

  float factor = 0.f;
  if (p.quant_mode == kQuantRow) {
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = lane + i * LANES;
      if (u < units) {
        float f[8], w[8];
        hv[i].unpack(f);
        load_weight(p.w, p.w_dtype, u, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) amax = max(amax, abs_bits(f[k] * rstd * w[k]));
      }
    }
    float scale;
    factor = quant_factor<YT>(row_max<LANES>(amax, red), p, scale);
    if (lane == 0) p.scale[row * p.ssr] = scale;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = lane + i * LANES;
    const bool in = u < units;
    float f[8];
    uint32_t amax = 0;
    if (in) {
      float w[8];
      hv[i].unpack(f);
      load_weight(p.w, p.w_dtype, u, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        f[k] = f[k] * rstd * w[k];
        amax = max(amax, abs_bits(f[k]));
      }
      if (p.y) {
        Raw8<T> o;
        o.pack(f);
        o.store(static_cast<T*>(p.y) + row * p.sy + u * kUnit);
      }
    }
    if (p.quant_mode == kQuantNone) continue;
    if (p.quant_mode == kQuantBlock) {
#pragma unroll
      for (int o = 8; o; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      float scale;
      factor = quant_factor<YT>(amax, p, scale);
      if (in && (lane & 15) == 0) p.scale[row * p.ssr + (long long)(u >> 4) * p.ssb] = scale;
    }
    if (in) {
      uint2 o;
      o.x = cvt2_fp8<YT>(__fmul_rn(f[0], factor), __fmul_rn(f[1], factor)) |
            (uint32_t)cvt2_fp8<YT>(__fmul_rn(f[2], factor), __fmul_rn(f[3], factor)) << 16;
      o.y = cvt2_fp8<YT>(__fmul_rn(f[4], factor), __fmul_rn(f[5], factor)) |
            (uint32_t)cvt2_fp8<YT>(__fmul_rn(f[6], factor), __fmul_rn(f[7], factor)) << 16;
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.q) + row * p.sq + u * kUnit) = o;
    }
  }
}

// Forward for any width, stride and alignment: one CTA per row, element by
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

// Backward for any width, stride and alignment: a CTA per row, element by
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
