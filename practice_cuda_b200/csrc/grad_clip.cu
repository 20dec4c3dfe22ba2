// The global norm of many gradient tensors, and their clipping.
//
//   norm = sqrt(sum_t sum_i g_ti^2)  (or max |g_ti|),
//   out_ti = g_ti * min(1, max_norm / (norm + eps))
//
// Two launches for any number of tensors up to a table's capacity: every
// tensor is cut into chunks, the first kernel leaves one partial per CTA, and
// the second sums the partials in a fixed order in every CTA (so no CTA waits
// for another and nothing depends on the order of atomics) before it scales.
// The second kernel walks the chunks from the last to the first: the end of
// what the first one read is still in L2 (47 million bf16 values on a B200: 51.7 us,
// from the first to the last 53.4 us).  Bound by HBM traffic, each gradient being
// read twice, less what L2 holds, and written once: 2.2 billion bf16 values in
// 2064 us (6.4 TB/s of 13.25 GB), 93 million in 100 us (5.6 TB/s), and by the call
// itself below a few million values.
//
// Squares are summed in fp32 over the 16 or 32 elements that a thread loads
// at a time and in fp64 from there on; a group whose fp32 sum is not finite
// (elements above 1.8e19), or so small that its squares are subnormal or nothing
// in fp32, is summed again in fp64.  So the norm is as exact for any gradients, and
// overflows only where the result does.
#include <algorithm>
#include <new>
#include <vector>

#include "host.cuh"

using namespace pcb;

namespace pcb {
namespace clip {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;   // elements of one tensor that a CTA takes at a time
constexpr int kLoads = 4;      // 16-byte loads in flight per thread
constexpr int kCtasPerSm = 8;  // resident CTAs: 64 KB per SM in flight

// The tensors of one launch, passed by value (a launch holds at most 32,764
// bytes of parameters), so nothing outlives the call on the host.
template <int N>
struct Table {
  const void* in[N];
  void* out[N];
  long long numel[N];
  int first_chunk[N + 1];  // running count of chunks
  unsigned char dtype[N];
  int count;
};
constexpr int kSmall = 64, kLarge = 1000;
static_assert(sizeof(Table<kLarge>) <= 32000, "a launch's parameters");

__host__ __device__ inline int head_of(const void* p, int es) {  // elements before the first 16-byte boundary
  return (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / es);
}
__host__ __device__ inline long long chunks_of(const void* p, int es, long long numel) {
  const long long body = numel - head_of(p, es);
  return body <= 0 ? 1 : (body + kChunk - 1) / kChunk;
}

template <typename T>
struct Vec;  // 16 bytes of T
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(uint4 v, float* f) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(uint4 v, float* f) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(u[i] << 16);
      f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(uint4 v, float* f) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* f) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 t = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};

// The elements of chunk `k` of a tensor: [begin, end), of which the loads of
// 16 bytes start at `body` (later than `begin` in the first chunk only).
struct Range {
  long long begin, body, end;
};
__device__ __forceinline__ Range range_of(const void* p, int es, long long numel, long long k) {
  const long long head = min((long long)head_of(p, es), numel);
  const long long body = head + k * kChunk;
  return Range{k == 0 ? 0 : body, body, min(numel, body + kChunk)};
}

// NaN stays NaN (fmax would drop it): unsigned bits of |v|.
struct MaxAcc {
  uint32_t v = 0;
  __device__ __forceinline__ void add(const float* f, int n) {
    for (int i = 0; i < n; ++i) v = max(v, abs_bits(f[i]));
  }
  __device__ __forceinline__ double value() const { return (double)__uint_as_float(v); }
  static __device__ __forceinline__ double join(double a, double b) { return (a != a || a > b) ? a : b; }
};
struct SquareAcc {
  double v = 0.0;
  __device__ __forceinline__ void add(const float* f, int n) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < n; ++i) s = fmaf(f[i], f[i], s);
    // Squares below 2^-126 are off by up to 2^-150 each: 32 of them by 2^-29 of 1e-35.
    if (s >= 1e-35f && s <= 3.4e38f) {
      v += (double)s;
      return;
    }
    uint32_t any = 0;  // zeros are common, and are not summed again
#pragma unroll
    for (int i = 0; i < n; ++i) any |= abs_bits(f[i]);
    if (any == 0) return;
#pragma unroll
    for (int i = 0; i < n; ++i) v += (double)f[i] * (double)f[i];
  }
  __device__ __forceinline__ double value() const { return v; }
  static __device__ __forceinline__ double join(double a, double b) { return a + b; }
};

template <typename ACC>
__device__ double block_join(double v) {
  __shared__ double part[kThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v = ACC::join(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) v = ACC::join(v, part[i]);
  return v;
}

template <typename T, typename ACC>
__device__ __forceinline__ void chunk_norm(const void* base, long long numel, long long k, ACC& acc) {
  constexpr int N = Vec<T>::N;
  const T* g = static_cast<const T*>(base);
  const Range r = range_of(base, sizeof(T), numel, k);
  const int vecs = (int)(max(r.end - r.body, 0ll) / N);
  const uint4* v = reinterpret_cast<const uint4*>(g + r.body);
  for (int i0 = threadIdx.x; i0 < vecs; i0 += kThreads * kLoads) {
    uint4 u[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) u[j] = i0 + j * kThreads < vecs ? __ldg(v + i0 + j * kThreads) : make_uint4(0, 0, 0, 0);
    float f[N * kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) Vec<T>::unpack(u[j], f + j * N);
    acc.add(f, N * kLoads);
  }
  const long long tail = r.body + (long long)vecs * N;
  const int loose = (int)(r.body - r.begin) + (int)max(r.end - tail, 0ll);  // fewer than 16 elements
  if (threadIdx.x < loose) {
    const int before = (int)(r.body - r.begin);
    const float f = Vec<T>::get(g[threadIdx.x < before ? r.begin + threadIdx.x : tail + (threadIdx.x - before)]);
    acc.add(&f, 1);
  }
}

template <int N, typename ACC>
__global__ void __launch_bounds__(kThreads) grad_norm_kernel(const __grid_constant__ Table<N> t, double* partial) {
  ACC acc;
  int at = 0;
  for (int c = blockIdx.x; c < t.first_chunk[t.count]; c += gridDim.x) {
    while (c >= t.first_chunk[at + 1]) ++at;  // at most one walk through the table per CTA
    const long long k = c - t.first_chunk[at];
    if (t.dtype[at] == PCB_DTYPE_F32) chunk_norm<float>(t.in[at], t.numel[at], k, acc);
    else if (t.dtype[at] == PCB_DTYPE_BF16) chunk_norm<__nv_bfloat16>(t.in[at], t.numel[at], k, acc);
    else chunk_norm<__half>(t.in[at], t.numel[at], k, acc);
  }
  const double v = block_join<ACC>(acc.value());
  if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

// The norm from the partials, in the same order in every CTA.
template <typename ACC>
__device__ float norm_of(const double* partial, int parts, bool squares) {
  double v = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) v = ACC::join(v, partial[i]);
  v = block_join<ACC>(v);
  return (float)(squares ? sqrt(v) : v);
}

template <typename ACC>
__global__ void __launch_bounds__(kThreads) grad_norm_final_kernel(const double* partial, int parts, bool squares,
                                                                   float* norm) {
  const float v = norm_of<ACC>(partial, parts, squares);
  if (threadIdx.x == 0) *norm = v;
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const void* base, void* out, long long numel, long long k, float factor) {
  constexpr int N = Vec<T>::N;
  const T* g = static_cast<const T*>(base);
  T* o = static_cast<T*>(out);
  const Range r = range_of(base, sizeof(T), numel, k);
  const int vecs = (int)(max(r.end - r.body, 0ll) / N);
  const uint4* v = reinterpret_cast<const uint4*>(g + r.body);
  const bool aligned_out = ((reinterpret_cast<uintptr_t>(o + r.body)) & 15) == 0;
  for (int i0 = threadIdx.x; i0 < vecs; i0 += kThreads * kLoads) {
    uint4 u[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      if (i0 + j * kThreads < vecs) u[j] = v[i0 + j * kThreads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int i = i0 + j * kThreads;
      if (i >= vecs) break;
      float f[N];
      Vec<T>::unpack(u[j], f);
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] *= factor;
      T* dst = o + r.body + (long long)i * N;
      if (aligned_out) {
        *reinterpret_cast<uint4*>(dst) = Vec<T>::pack(f);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) dst[e] = Vec<T>::put(f[e]);
      }
    }
  }
  const long long tail = r.body + (long long)vecs * N;
  const int before = (int)(r.body - r.begin), loose = before + (int)max(r.end - tail, 0ll);
  if (threadIdx.x < loose) {
    const long long i = threadIdx.x < before ? r.begin + threadIdx.x : tail + (threadIdx.x - before);
    o[i] = Vec<T>::put(Vec<T>::get(g[i]) * factor);
  }
}

// partial: the partials of the whole call (norm is then written), or null
// where *norm is given.
template <int N, typename ACC>
__global__ void __launch_bounds__(kThreads) grad_scale_kernel(const __grid_constant__ Table<N> t, const double* partial,
                                                              int parts, bool squares, float* norm, float max_norm,
                                                              float eps, bool in_place) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float total;
  if (partial) {
    total = norm_of<ACC>(partial, parts, squares);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  } else {
    total = *norm;
  }
  // A NaN norm gives a NaN factor; an infinite one gives 0 (and NaN at the infinities).
  float factor = __fdiv_rn(max_norm, total + eps);
  if (factor > 1.f || total == 0.f) factor = 1.f;
  if (in_place && factor == 1.f) return;  // every value is multiplied by one where it stands
  const int chunks = t.first_chunk[t.count];
  int at = t.count - 1;
  // From the last chunk to the first.
  for (int i = blockIdx.x; i < chunks; i += gridDim.x) {
    const int c = chunks - 1 - i;
    while (c < t.first_chunk[at]) --at;
    const long long k = c - t.first_chunk[at];
    if (t.dtype[at] == PCB_DTYPE_F32) chunk_scale<float>(t.in[at], t.out[at], t.numel[at], k, factor);
    else if (t.dtype[at] == PCB_DTYPE_BF16) chunk_scale<__nv_bfloat16>(t.in[at], t.out[at], t.numel[at], k, factor);
    else chunk_scale<__half>(t.in[at], t.out[at], t.numel[at], k, factor);
  }
}

}  // namespace clip
}  // namespace pcb

namespace {

struct List {
  const void* const* in;
  void* const* out;
  const int64_t* numel;
  const int* dtype;
  int64_t count;
};

int check_list(const List& l, bool scaled) {
  if (l.count < 0) return fail(PCB_ERR_INVALID, "negative count");
  if (l.count && (!l.in || !l.numel || !l.dtype || (scaled && !l.out))) return fail(PCB_ERR_INVALID, "null pointer");
  int64_t chunks = 0;
  for (int64_t i = 0; i < l.count; ++i) {
    if (!is_float_in(l.dtype[i])) return fail(PCB_ERR_INVALID, "gradient dtype must be F32, F16 or BF16");
    if (l.numel[i] < 0) return fail(PCB_ERR_INVALID, "negative size");
    if (l.numel[i] && (!l.in[i] || (scaled && !l.out[i]))) return fail(PCB_ERR_INVALID, "null pointer");
    const int es = elem_size(l.dtype[i]);
    if (!aligned(l.in[i], es) || (scaled && !aligned(l.out[i], es)))
      return fail(PCB_ERR_INVALID, "gradient pointer is not a multiple of its element size");
    chunks += clip::chunks_of(l.in[i], es, l.numel[i]);
  }
  if (chunks > INT32_MAX) return fail(PCB_ERR_UNSUPPORTED, "too many gradient elements");
  return PCB_OK;
}

// CTAs scale chunks side by side, so what is written for one tensor must be no
// other tensor's, neither read nor written; out[i] may be in[i] itself.
int check_overlap(const List& l) {
  struct Span {
    uintptr_t begin, end;
  };
  auto span = [&](const void* p, int64_t i) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    return Span{at, at + (uintptr_t)l.numel[i] * elem_size(l.dtype[i])};
  };
  auto before = [](const Span& a, const Span& b) { return a.begin < b.begin; };
  std::vector<Span> out;
  try {
    out.reserve((size_t)l.count);
  } catch (const std::bad_alloc&) {
    return fail(PCB_ERR_UNSUPPORTED, "too many gradients");
  }
  for (int64_t i = 0; i < l.count; ++i)
    if (l.numel[i]) out.push_back(span(l.out[i], i));
  if (!std::is_sorted(out.begin(), out.end(), before)) std::sort(out.begin(), out.end(), before);
  bool apart = true;
  for (size_t k = 1; k < out.size(); ++k) apart &= out[k - 1].end <= out[k].begin;
  for (int64_t i = 0; apart && i < l.count; ++i) {
    if (!l.numel[i] || l.in[i] == l.out[i]) continue;
    const Span in = span(l.in[i], i);
    // The first written span that ends behind in.begin: they are apart, so their ends are in order too.
    const auto at = std::partition_point(out.begin(), out.end(), [&](const Span& o) { return o.end <= in.begin; });
    apart = at == out.end() || at->begin >= in.end;
  }
  return apart ? PCB_OK : fail(PCB_ERR_INVALID, "gradients or outputs overlap: each element may be scaled once only");
}

// Calls f(table, grid) for each table of at most N tensors; empty tensors are left out.
template <int N, typename F>
int for_tables(const List& l, F&& f) {
  const int most = device_info().sm_count * clip::kCtasPerSm;
  clip::Table<N> t;
  int64_t i = 0;
  while (i < l.count) {
    int n = 0;
    t.first_chunk[0] = 0;
    for (; i < l.count && n < N; ++i) {
      if (l.numel[i] == 0) continue;
      t.in[n] = l.in[i];
      t.out[n] = l.out ? l.out[i] : nullptr;
      t.numel[n] = l.numel[i];
      t.dtype[n] = (unsigned char)l.dtype[i];
      t.first_chunk[n + 1] = t.first_chunk[n] + (int)clip::chunks_of(l.in[i], elem_size(l.dtype[i]), l.numel[i]);
      ++n;
    }
    if (n == 0) break;
    t.count = n;
    if (int st = f(t, std::min(t.first_chunk[n], most))) return st;
  }
  return PCB_OK;
}

template <int N, typename ACC>
int run_norm(const List& l, double* partial, int& parts, cudaStream_t s) {
  parts = 0;
  return for_tables<N>(l, [&](const clip::Table<N>& t, int grid) -> int {
    clip::grad_norm_kernel<N, ACC><<<grid, clip::kThreads, 0, s>>>(t, partial + parts);
    parts += grid;
    return check_launch("grad_norm_kernel");
  });
}

template <int N, typename ACC>
int run_scale(const List& l, const double* partial, int parts, bool squares, float* norm, float max_norm, float eps,
              bool in_place, cudaStream_t s) {
  return for_tables<N>(l, [&](const clip::Table<N>& t, int grid) -> int {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid, 1, 1);
    cfg.blockDim = dim3(clip::kThreads, 1, 1);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, clip::grad_scale_kernel<N, ACC>, t, partial, parts, squares, norm, max_norm, eps, in_place);
    return check_launch("grad_scale_kernel");
  });
}

bool any_moves(const List& l) {
  for (int64_t i = 0; i < l.count; ++i)
    if (l.numel[i] && l.in[i] != l.out[i]) return true;
  return false;
}

// norm (and scale, where `scale` is set) for one table size and accumulator.
template <int N, typename ACC>
int run(const List& l, bool squares, bool scale, float* norm, float max_norm, float eps, double* partial,
        cudaStream_t s) {
  int parts = 0;
  if (int st = run_norm<N, ACC>(l, partial, parts, s)) return st;
  if (!scale || parts == 0) {
    clip::grad_norm_final_kernel<ACC><<<1, clip::kThreads, 0, s>>>(partial, parts, squares, norm);
    return check_launch("grad_norm_final_kernel");
  }
  return run_scale<N, ACC>(l, partial, parts, squares, norm, max_norm, eps, !any_moves(l), s);
}

int entry(const List& l, int norm_type, bool scale, float* norm, float max_norm, float eps, void* workspace,
          int64_t workspace_bytes, void* stream) {
  if (norm_type != PCB_GRAD_NORM_L2 && norm_type != PCB_GRAD_NORM_MAX) return fail(PCB_ERR_INVALID, "bad norm type");
  if (int st = check_list(l, scale)) return st;
  if (scale)
    if (int st = check_overlap(l)) return st;
  if (!norm || !workspace || !aligned(workspace, 8) || workspace_bytes < pcb_grad_norm_workspace_bytes(l.count))
    return fail(PCB_ERR_INVALID, "gradient norm workspace too small or misaligned");
  double* partial = static_cast<double*>(workspace);
  cudaStream_t s = (cudaStream_t)stream;
  const bool small = l.count <= clip::kSmall;
  if (norm_type == PCB_GRAD_NORM_L2)
    return small ? run<clip::kSmall, clip::SquareAcc>(l, true, scale, norm, max_norm, eps, partial, s)
                 : run<clip::kLarge, clip::SquareAcc>(l, true, scale, norm, max_norm, eps, partial, s);
  return small ? run<clip::kSmall, clip::MaxAcc>(l, false, scale, norm, max_norm, eps, partial, s)
               : run<clip::kLarge, clip::MaxAcc>(l, false, scale, norm, max_norm, eps, partial, s);
}

}  // namespace

extern "C" {

int64_t pcb_grad_norm_workspace_bytes(int64_t count) {
  if (count < 0) return 0;
  const int64_t launches = count <= clip::kSmall ? 1 : (count + clip::kLarge - 1) / clip::kLarge;
  return 8 * std::max<int64_t>(1, launches * device_info().sm_count * clip::kCtasPerSm);
}

int pcb_grad_norm(const void* const* grads, const int64_t* numel, const int* dtypes, int64_t count, int norm_type,
                  float* norm, void* workspace, int64_t workspace_bytes, void* stream) {
  return entry(List{grads, nullptr, numel, dtypes, count}, norm_type, false, norm, 0.f, 0.f, workspace,
               workspace_bytes, stream);
}

int pcb_grad_clip(const void* const* grads, void* const* out, const int64_t* numel, const int* dtypes, int64_t count,
                  int norm_type, float max_norm, float eps, float* norm, void* workspace, int64_t workspace_bytes,
                  void* stream) {
  if (!(max_norm >= 0.f)) return fail(PCB_ERR_INVALID, "max_norm must not be negative");
  return entry(List{grads, out, numel, dtypes, count}, norm_type, true, norm, max_norm, eps, workspace,
               workspace_bytes, stream);
}

int pcb_grad_scale(const void* const* grads, void* const* out, const int64_t* numel, const int* dtypes, int64_t count,
                   const float* norm, float max_norm, float eps, void* stream) {
  if (!(max_norm >= 0.f)) return fail(PCB_ERR_INVALID, "max_norm must not be negative");
  const List l{grads, out, numel, dtypes, count};
  if (int st = check_list(l, true)) return st;
  if (int st = check_overlap(l)) return st;
  if (!norm) return fail(PCB_ERR_INVALID, "null pointer");
  float* n = const_cast<float*>(norm);  // read only where no partials are given
  cudaStream_t s = (cudaStream_t)stream;
  if (count <= clip::kSmall)
    return run_scale<clip::kSmall, clip::SquareAcc>(l, nullptr, 0, true, n, max_norm, eps, !any_moves(l), s);
  return run_scale<clip::kLarge, clip::SquareAcc>(l, nullptr, 0, true, n, max_norm, eps, !any_moves(l), s);
}

}  // extern "C"
