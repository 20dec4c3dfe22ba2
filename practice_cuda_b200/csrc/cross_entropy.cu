// C entry points of the output projection's cross entropy.
#include <algorithm>

#include "cross_entropy.cuh"
#include "host.cuh"

using namespace pcb;

namespace {

// 3-D map (inner, outer, 1) of 16-bit elements with 64-element rows in the
// 128-byte swizzle.
bool make_map(CUtensorMap* map, const void* base, int dt, int64_t inner, int64_t outer, int64_t stride, int box_outer,
              CUtensorMapL2promotion promotion) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t row = (cuuint64_t)stride * 2;
  const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, 1};
  const cuuint64_t strides[2] = {row, std::max<cuuint64_t>(16, (cuuint64_t)outer * row)};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_outer, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, dt == PCB_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
            const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool load_map(CUtensorMap* map, const void* base, int dt, int64_t inner, int64_t outer, int64_t stride, int box_outer) {
  return make_map(map, base, dt, inner, outer, stride, box_outer, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}
// An MN-major operand as (64 elements, K rows, slabs of 64 elements): one load
// brings both slabs of a 128-wide tile side by side.  Whole slabs only: the
// last one must lie within the row's stride.
bool slab_map(CUtensorMap* map, const void* base, int dt, int64_t slabs, int64_t rows, int64_t stride) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {64, (cuuint64_t)rows, (cuuint64_t)slabs};
  const cuuint64_t strides[2] = {(cuuint64_t)stride * 2, 128};
  const cuuint32_t box[3] = {64, loss::BK, 2};
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, dt == PCB_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
            const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// B of a product of G: [rows, dim], dim contiguous.
bool load_b(CUtensorMap* map, loss::Problem& q, const void* base, int dt, int64_t dim, int64_t rows, int64_t stride) {
  q.b_slabs = dim % 64 == 0 ? 1 : 0;
  if (q.b_slabs) return slab_map(map, base, dt, dim / 64, rows, stride);
  return load_map(map, base, dt, dim, rows, stride, loss::BK);
}
bool store_map(CUtensorMap* map, void* base, int dt, int64_t inner, int64_t outer, int64_t stride) {
  return make_map(map, base, dt, inner, outer, stride, 32, CU_TENSOR_MAP_L2_PROMOTION_NONE);
}

constexpr int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Launch of one of the tcgen05 kernels over `workers` CTAs or pairs.  They
// re-split their registers with setmaxnreg, which is only valid when the launch
// holds exactly kLaunchRegs per thread (otherwise setmaxnreg.inc could never be
// satisfied).
template <bool PAIR>
int launch_tiles(void (*kernel)(loss::Params), int num_regs, int smem, const loss::Params& p, cudaStream_t s,
                 const char* what) {
  if (num_regs != loss::kLaunchRegs)
    return fail(PCB_ERR_UNSUPPORTED, "cross entropy kernel register count differs from its setmaxnreg split");
  ensure_smem_attr(kernel, smem);
  const int sms = device_info().sm_count;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(PAIR ? 2 * std::min(p.num_tiles, sms / 2) : std::min(p.num_tiles, sms)), 1, 1);
  cfg.blockDim = dim3(loss::kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  // griddepcontrol.wait precedes every global access of the kernels.
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, p);
  return check_launch(what);
}

int regs_of(const void* kernel) {
  cudaFuncAttributes fa{};
  return cudaFuncGetAttributes(&fa, kernel) == cudaSuccess ? fa.numRegs : -1;
}

template <int MODE, bool PAIR>
int launch_logits_as(const loss::Params& p, cudaStream_t s) {
  static const int regs = regs_of((const void*)loss::logits_kernel<MODE, PAIR>);
  return launch_tiles<PAIR>(loss::logits_kernel<MODE, PAIR>, regs, loss::Smem<PAIR>::ALLOC, p, s, "logits_kernel");
}

template <int MODE>
int launch_logits(const loss::Params& p, bool pair, cudaStream_t s) {
  return pair ? launch_logits_as<MODE, true>(p, s) : launch_logits_as<MODE, false>(p, s);
}

int launch_grad_products(const loss::Params& p, cudaStream_t s) {
  static const int regs = regs_of((const void*)loss::grad_products_kernel);
  return launch_tiles<true>(loss::grad_products_kernel, regs, loss::ProductSmem::ALLOC, p, s, "grad_products_kernel");
}

// Up to 128 tokens a CTA has a tile to itself.
bool on_pairs(int64_t tokens) { return tokens > loss::BM; }

// Columns of a logit tile.  On single CTAs: the vocabulary in as few rounds
// over the SMs as 256-column tiles need, and evenly so (a multiple of 16, the
// step of the instruction's N).
int logit_tile(int64_t tokens, int64_t vocab) {
  if (on_pairs(tokens)) return loss::TILE;
  const int64_t sms = std::max(1, device_info().sm_count);
  const int64_t rounds = up(vocab, sms * loss::TILE);
  return (int)std::max<int64_t>(32, up(up(vocab, sms * rounds), 16) * 16);
}

template <typename K, typename... A>
int launch_after(K kernel, const char* what, int64_t grid, int threads, cudaStream_t s, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, args...);
  return check_launch(what);
}

// tile counts and K split of a problem
void shape(loss::Problem& q, int64_t m, int64_t n, int64_t k, int splits, bool pair = true, int tile_n = loss::TILE) {
  q.m = (int)m;
  q.n = (int)n;
  q.m_blocks = (int)up(m, pair ? loss::TILE : loss::BM);
  q.n_blocks = (int)up(n, tile_n);
  q.k_stages = (int)up(k, loss::BK);
  const int target = pair ? loss::kChunkStages : loss::kChunkStagesSingle;
  const int chunks = (int)up(q.k_stages, target);
  q.chunk_stages = (int)up(q.k_stages, chunks);  // even chunks: a last one of a stage or two would stall the others
  q.a_rows = (int)std::min<int64_t>(loss::BM, up(m, 8) * 8);
  q.split_stages = (int)up(q.k_stages, splits);
  q.splits = (int)up(q.k_stages, q.split_stages);  // none of them empty
  q.tiles = q.m_blocks * q.n_blocks * q.splits;
}

bool too_large(int64_t tokens, int64_t vocab, int64_t dim) {
  return tokens > (1 << 26) || vocab > (1 << 26) || dim > (1 << 26) ||
         up(tokens, loss::TILE) * up(vocab, loss::TILE) > (1 << 30) ||
         up(std::max(tokens, vocab), loss::TILE) * up(dim, loss::WIDE) > (1 << 24);  // (times at most 64 splits)
}
// Sizes that need a workspace: no tokens need none, and what the passes refuse is not computed with.
bool has_workspace(int64_t tokens, int64_t vocab, int64_t dim) {
  return tokens > 0 && vocab > 0 && dim > 0 && !too_large(tokens, vocab, dim);
}

int check_shapes(int dtype, int64_t tokens, int64_t vocab, int64_t dim, int reduction) {
  if (dtype != PCB_DTYPE_F16 && dtype != PCB_DTYPE_BF16)
    return fail(PCB_ERR_INVALID, "linear cross entropy: x and weight must be F16 or BF16");
  if (tokens < 0 || vocab <= 0 || dim <= 0)
    return fail(PCB_ERR_INVALID, "linear cross entropy needs tokens >= 0, vocab > 0 and dim > 0");
  if (reduction < loss::kNone || reduction > loss::kMean)
    return fail(PCB_ERR_INVALID, "linear cross entropy: reduction must be 0 (none), 1 (sum) or 2 (mean)");
  if (too_large(tokens, vocab, dim))
    return fail(PCB_ERR_UNSUPPORTED, "linear cross entropy: dimension too large, or too many tiles");
  return PCB_OK;
}

int check_operands(const void* x, int64_t sx, const void* w, int64_t sw) {
  if (!x || !w) return fail(PCB_ERR_INVALID, "null pointer");
  if (!aligned(x, 16) || !aligned(w, 16) || sx % 8 != 0 || sw % 8 != 0)
    return fail(PCB_ERR_LAYOUT, "linear cross entropy: rows of x and weight must start on 16-byte boundaries");
  if (device_info().major != 10) return fail(PCB_ERR_DEVICE, "linear cross entropy needs an sm_100 device");
  return PCB_OK;
}

// A workspace cut into 256-byte aligned parts.
struct Cut {
  int64_t at = 0;
  int64_t take(int64_t bytes) {
    const int64_t a = at;
    at += up(bytes, 256) * 256;
    return a;
  }
};

// Where the logits take about 90 us or more, tokens that are left out are packed
// away.  Packed and as they are, on a B200, loss / loss and gradients in us: 1021
// tokens of 50001 x 2056 fp16 with 30 % left out 126 / 627 and 179 / 729, with 60 %
// 101 / 465 and 179 / 710, with none 183 / 741 and 177 / 735; 4096 tokens of 32000 x
// 4096 with 30 % 549 / 2286 and 679 / 2885; 2048 tokens of 8192 x 4096 with 30 % 96 /
// 381 and 106 / 457.  It costs three launches, about 6 us, where no token is left
// out, and below this size that is more than most masks save.  The gain comes
// in whole tiles of 256 tokens: 768 tokens of which 534 are left still fill three (131
// / 564 and 146 / 590), hence no fewer than two of them.
bool packs(int64_t tokens, int64_t vocab, int64_t dim) {
  return tokens >= 512 && (double)tokens * vocab * dim >= (double)(1ll << 36);
}

// What the forward pass leaves for the backward pass of packed tokens.  G takes
// their order too, so dX leaves the products' kernel row by row to its own places
// (16 bytes a lane); the copy of x is what dW's product reads.
struct Order {
  int64_t live, order, target, x, stride, bytes;
  Order(int64_t tokens, int64_t vocab, int64_t dim) {
    Cut c;
    stride = up(dim, 64) * 64;  // elements
    live = c.take(4);
    order = c.take(tokens * 4);
    target = c.take(tokens * 8);
    x = c.take(tokens * stride * 2);
    bytes = packs(tokens, vocab, dim) ? c.at : 0;
  }
  void use(loss::Params& p, const void* state) const {
    const char* s = static_cast<const char*>(state);
    p.live = reinterpret_cast<const int*>(s + live);
    p.order = reinterpret_cast<const int*>(s + order);
    p.target_packed = reinterpret_cast<const long long*>(s + target);
  }
};

struct FwdPlan {
  int64_t partial, target_logit, sums, ticket, bytes;
  FwdPlan(int64_t tokens, int64_t vocab) {
    Cut c;
    partial = c.take(up(vocab, logit_tile(tokens, vocab)) * 2 * tokens * 8);
    target_logit = c.take(tokens * 4);
    sums = c.take(up(tokens, 32) * 16);
    ticket = c.take(4);
    bytes = c.at;
  }
};

// Parts that dX's K (the vocabulary) is cut into.  Its tiles are few and long
// where tokens are few; more parts even out the pairs' shares and cost the
// writing and reading of their fp32 accumulators.  The shares are counted in
// stages (0.27 us of the tensor cores) as the kernel hands them out: a tile's
// epilogue is worth about six stages, a stage's time about 1.7 MB of traffic, and
// the joining kernel about ten stages of its own.  Loss and gradients on a B200, in one
// part, as this chooses and in the best of the ten numbers below: 8 tokens of 32000 x
// 4096 441, 271 and 253 us, 256 tokens 451, 296 and 296, 512 tokens 534, 466 and 466; 64
// tokens of 32000 x 1024 364, 122 and 118, 1024 tokens 431, 239 and 239; 8 tokens of 8192
// x 4096 192, 152 and 138.  At fifteen sizes it is never more than 10 % off the best.
int split_of(int64_t tokens, int64_t vocab, int64_t dim, bool want_dw) {
  const int workers = std::max(1, device_info().sm_count / 2);
  const int64_t cols = up(dim, loss::WIDE), stages = up(vocab, loss::BK), halves = dim > loss::TILE ? 2 : 1;
  const int64_t dx_tiles = up(tokens, loss::TILE) * cols, dw_tiles = want_dw ? up(vocab, loss::TILE) * cols : 0;
  const int64_t dw_stages = up(tokens, loss::BK);
  if (dx_tiles >= 8 * workers) return 1;  // long rounds already come out nearly even
  int best = 1;
  double least = 0;
  for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
    if (stages / s < 4 && s > 1) break;
    const int part = (int)up(stages, s), t0 = (int)(dx_tiles * up(stages, part));
    const int extra = loss::extra_of(t0, part, (int)dw_tiles, (int)dw_stages, workers);
    int64_t longest = 0;
    for (int w = 0; w < workers; ++w) {
      int64_t longs = (t0 - w + workers - 1) / workers;
      const int r = t0 % workers;
      int64_t left = dw_tiles - (r > 0 ? (int64_t)extra * (workers - r) : 0), shorts = r > 0 && w >= r ? extra : 0;
      shorts += std::max<int64_t>(0, (left - (w >= r ? w - r : w - r + workers) + workers - 1) / workers);
      longest = std::max(longest, longs * (part * halves + 6) + shorts * (dw_stages * halves + 6));
    }
    const double cost = (double)longest + (s > 1 ? 10 + (double)s * tokens * dim * 8 / 1.7e6 : 0);
    if (s == 1 || cost < least) best = s, least = cost;
  }
  return best;
}

struct BwdPlan {
  int64_t cols, pieces, pitch;  // of G
  int splits;                   // parts of K of dX
  int64_t g, acc, weight, alpha, x, pitch_x, residue, first, next, bytes;
  bool copies;  // dW reads a copy of X without the rows of tokens that are left out
  BwdPlan(int64_t tokens, int64_t vocab, int64_t dim, int64_t piece, bool want_dx, bool want_dw, bool packed) {
    pitch_x = up(dim, 64) * 64;
    copies = want_dw && !packed;
    const int64_t copy = copies ? tokens * pitch_x * 2 : 0;
    // G of one piece takes 128 MiB at most (and is no narrower than 2048
    // columns): pieces of even width, whole tiles each.  The copy of X is within
    // that where it is large.
    const int64_t budget = ((int64_t)128 << 20) - (packs(tokens, vocab, dim) ? copy : 0);
    if (piece <= 0) piece = std::max<int64_t>(2048, budget / 2 / tokens);
    piece = std::min(piece, up(vocab, loss::TILE) * loss::TILE);  // whatever a caller names: sums with it stay in range
    piece = std::max<int64_t>(loss::TILE, piece / loss::TILE * loss::TILE);
    pieces = up(vocab, piece);
    cols = up(up(vocab, pieces), loss::TILE) * loss::TILE;
    pieces = up(vocab, cols);
    pitch = std::min(cols, up(vocab, 64) * 64);
    const int64_t dx_tiles = up(tokens, loss::TILE) * up(dim, loss::WIDE);
    splits = want_dx && pieces == 1 ? split_of(tokens, vocab, dim, want_dw) : 1;
    Cut c;
    g = c.take(tokens * pitch * 2);
    acc = c.take(want_dx && (pieces > 1 || splits > 1) ? dx_tiles * splits * loss::TILE * loss::WIDE * 4 : 0);
    weight = c.take(tokens * 4);
    alpha = c.take(4);
    x = c.take(copy);
    residue = c.take(tokens * 4);
    first = c.take(want_dw ? vocab * 4 : 0);
    next = c.take(want_dw ? tokens * 4 : 0);
    bytes = c.at;
  }
};

loss::Params base_params(int dtype, int64_t tokens, int64_t vocab, const int64_t* target, int64_t ignore_index) {
  loss::Params p;
  std::memset(&p, 0, sizeof(p));
  p.fmt = dtype == PCB_DTYPE_BF16 ? 1 : 0;
  p.tokens = (int)tokens;
  p.target = reinterpret_cast<const long long*>(target);
  p.ignore_index = ignore_index;
  p.vocab = vocab;
  return p;
}

// The entry points' own argument of packed tokens.
int check_packed(int dtype, int64_t tokens, int64_t vocab, int64_t dim, int reduction, const void* packed,
                 int64_t packed_bytes) {
  if (int st = check_shapes(dtype, tokens, vocab, dim, reduction)) return st;
  const int64_t need = tokens > 0 ? Order(tokens, vocab, dim).bytes : 0;
  if (need ? !packed || !aligned(packed, 256) || packed_bytes < need : packed != nullptr)
    return fail(PCB_ERR_INVALID, "linear cross entropy: packed state missing, too small, misaligned or not needed");
  return PCB_OK;
}

// `order` (null: every token is multiplied, in its own place) is the state that
// the forward pass leaves for the backward pass of packed tokens.
int forward(const void* x, int64_t sx, const void* weight, int64_t sw, int dtype, int64_t tokens,
                      int64_t vocab, int64_t dim, const int64_t* target, int64_t ignore_index, int reduction,
                      float* loss_out, float* stats, float* count, void* order, void* workspace,
                      int64_t workspace_bytes, void* stream) {
  if (int st = check_shapes(dtype, tokens, vocab, dim, reduction)) return st;
  if (tokens == 0) return PCB_OK;
  if (!target || !loss_out || !stats || !count) return fail(PCB_ERR_INVALID, "null pointer");
  const FwdPlan plan(tokens, vocab);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < plan.bytes)
    return fail(PCB_ERR_INVALID, "linear cross entropy workspace too small or misaligned");
  if (int st = check_operands(x, sx, weight, sw)) return st;
  cudaStream_t s = (cudaStream_t)stream;
  char* ws = static_cast<char*>(workspace);
  loss::Params p = base_params(dtype, tokens, vocab, target, ignore_index);
  loss::Problem& q = p.prob[0];
  const Order packed(tokens, vocab, dim);
  if (order) {
    char* at = static_cast<char*>(order);
    int* places = reinterpret_cast<int*>(at + packed.order);
    int* live = reinterpret_cast<int*>(at + packed.live);
    if (int st = launch_after(loss::loss_order_kernel, "loss_order_kernel", 1, 1024, s, p.target,
                              (long long)ignore_index, (int)tokens, places, live))
      return st;
    if (int st = launch_after(loss::loss_pack_kernel, "loss_pack_kernel",
                              std::min<int64_t>(tokens, (int64_t)device_info().sm_count * 8), 256, s,
                              static_cast<const uint16_t*>(x), (long long)sx, p.target, (const int*)places,
                              (const int*)live, (int)tokens, (int)dim, reinterpret_cast<uint16_t*>(at + packed.x),
                              (long long)packed.stride, reinterpret_cast<long long*>(at + packed.target)))
      return st;
    packed.use(p, order);
  }
  const bool pair = on_pairs(tokens);
  p.tile_n = logit_tile(tokens, vocab);
  shape(q, tokens, vocab, dim, 1, pair, p.tile_n);
  q.m_live = 1;
  if (order && !load_map(&q.packed, static_cast<char*>(order) + packed.x, dtype, dim, tokens, packed.stride, q.a_rows))
    return fail(PCB_ERR_LAYOUT, "cuTensorMapEncodeTiled rejected the operand layout");
  if (!load_map(&q.a, x, dtype, dim, tokens, sx, q.a_rows) ||
      !load_map(&q.b, weight, dtype, dim, vocab, sw, pair ? loss::TILE / 2 : p.tile_n))
    return fail(PCB_ERR_LAYOUT, "cuTensorMapEncodeTiled rejected the operand layout");
  p.num_tiles = q.tiles;
  p.partial = reinterpret_cast<float2*>(ws + plan.partial);
  p.target_logit = reinterpret_cast<float*>(ws + plan.target_logit);
  p.ticket = reinterpret_cast<unsigned*>(ws + plan.ticket);
  if (int st = launch_logits<loss::kStats>(p, pair, s)) return st;
  loss::RowArgs r{p.live, p.order, p.partial, p.target_logit, p.target, ignore_index, vocab, (int)tokens,
                  2 * q.n_blocks, reduction, stats, loss_out, count, reinterpret_cast<double*>(ws + plan.sums), p.ticket};
  return launch_after(loss::loss_rows_kernel, "loss_rows_kernel", up(tokens, 32), loss::kRowWarps * 32, s, r);
}

int backward(const void* x, int64_t sx, const void* weight, int64_t sw, int dtype, int64_t tokens,
                      int64_t vocab, int64_t dim, const int64_t* target, int64_t ignore_index, int reduction,
                      const float* stats, const float* count, const void* order,
                      const float* dloss, void* dx, int64_t sdx, void* dw, int64_t sdw, int64_t piece, void* workspace,
                      int64_t workspace_bytes, void* stream) {
  if (int st = check_shapes(dtype, tokens, vocab, dim, reduction)) return st;
  cudaStream_t s = (cudaStream_t)stream;
  if (tokens == 0) {
    if (dw && cudaMemset2DAsync(dw, (size_t)sdw * 2, 0, (size_t)dim * 2, (size_t)vocab, s) != cudaSuccess)
      return check_launch("linear cross entropy dw");
    return PCB_OK;
  }
  if (!dx && !dw) return PCB_OK;
  if (!target || !stats || !count || !dloss) return fail(PCB_ERR_INVALID, "null pointer");
  const BwdPlan plan(tokens, vocab, dim, piece, dx != nullptr, dw != nullptr, order != nullptr);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < plan.bytes)
    return fail(PCB_ERR_INVALID, "linear cross entropy workspace too small or misaligned");
  if (int st = check_operands(x, sx, weight, sw)) return st;
  char* ws = static_cast<char*>(workspace);
  void* g = ws + plan.g;
  float4* acc = reinterpret_cast<float4*>(ws + plan.acc);
  loss::Params base = base_params(dtype, tokens, vocab, target, ignore_index);
  base.stats = stats;
  const Order packed(tokens, vocab, dim);
  const void* packed_x = nullptr;
  if (order) {
    packed.use(base, order);
    packed_x = static_cast<const char*>(order) + packed.x;
    if (dx)
      if (int st = launch_after(loss::loss_zero_rows_kernel, "loss_zero_rows_kernel",
                                std::min<int64_t>(tokens, (int64_t)device_info().sm_count * 8), 256, s, base.order,
                                base.live, (int)tokens, (int)dim, static_cast<uint16_t*>(dx), (long long)sdx,
                                aligned(dx, 16) && sdx % 8 == 0 ? 1 : 0))
        return st;
  }
  if (reduction == loss::kNone) {
    float* row_weight = reinterpret_cast<float*>(ws + plan.weight);
    float* alpha = reinterpret_cast<float*>(ws + plan.alpha);
    if (int st = launch_after(loss::loss_weights_kernel, "loss_weights_kernel", 1, 1024, s, dloss, base.target,
                              (long long)ignore_index, (int)tokens, base.live, base.order, row_weight, alpha))
      return st;
    base.row_weight = row_weight;
    base.alpha = alpha;
  } else {
    base.dloss = dloss;
    base.count = reduction == loss::kMean ? count : nullptr;
  }
  if (plan.copies)
    if (int st = launch_after(loss::loss_kept_rows_kernel, "loss_kept_rows_kernel",
                              std::min<int64_t>(tokens, (int64_t)device_info().sm_count * 8), 256, s,
                              static_cast<const uint16_t*>(x), (long long)sx, base.target, (long long)ignore_index,
                              count, (int)tokens, (int)dim, reinterpret_cast<uint16_t*>(ws + plan.x),
                              (long long)plan.pitch_x))
      return st;
  base.residue = reinterpret_cast<float*>(ws + plan.residue);
  base.x = static_cast<const uint16_t*>(x);
  base.w = static_cast<const uint16_t*>(weight);
  base.sx = sx;
  base.sw = sw;
  if (dw) {
    int* first = reinterpret_cast<int*>(ws + plan.first);
    int* next = reinterpret_cast<int*>(ws + plan.next);
    if (int st = launch_after(loss::loss_tokens_of_targets_kernel, "loss_tokens_of_targets_kernel",
                              up(tokens, loss::kListTokens), loss::kListThreads, s, base, first, next))
      return st;
    base.first = first;
    base.next = next;
  }
  for (int64_t i = 0; i < plan.pieces; ++i) {
    const int64_t col0 = i * plan.cols, cols = std::min(plan.cols, vocab - col0);
    const char* w = static_cast<const char*>(weight) + col0 * sw * 2;
    bool ok = true;
    loss::Params p = base;
    p.col0 = (int)col0;
    const bool pair = on_pairs(tokens);
    p.tile_n = logit_tile(tokens, cols);
    loss::Problem& q = p.prob[0];
    shape(q, tokens, cols, dim, 1, pair, p.tile_n);
    q.m_live = 1;
    ok &= load_map(&q.a, x, dtype, dim, tokens, sx, q.a_rows);
    if (packed_x) ok &= load_map(&q.packed, packed_x, dtype, dim, tokens, packed.stride, q.a_rows);
    ok &= load_map(&q.b, w, dtype, dim, cols, sw, pair ? loss::TILE / 2 : p.tile_n);
    ok &= store_map(&q.c_box, g, dtype, cols, tokens, plan.pitch);
    q.c_tma = pair;  // a single CTA's column halves need not be whole 64-column boxes
    q.c = g;
    q.scm = plan.pitch;
    p.num_tiles = q.tiles;
    if (!ok) return fail(PCB_ERR_LAYOUT, "cuTensorMapEncodeTiled rejected the operand layout");
    if (int st = launch_logits<loss::kGradient>(p, pair, s)) return st;

    p = base;
    p.col0 = (int)col0;
    int n = 0;
    if (dx) {
      loss::Problem& d = p.prob[n++];
      shape(d, tokens, dim, cols, plan.splits, true, loss::WIDE);
      ok &= load_map(&d.a, g, dtype, cols, tokens, plan.pitch, d.a_rows);
      ok &= load_b(&d.b, d, w, dtype, dim, cols, sw);
      d.acc = acc;
      if (plan.splits > 1) d.acc_mode = loss::kAccSlab;
      else if (plan.pieces > 1) d.acc_mode = i == 0 ? loss::kAccWrite : i + 1 < plan.pieces ? loss::kAccAdd : loss::kAccLast;
      d.c = dx;
      d.scm = sdx;
      d.c_tma = aligned(dx, 16) && sdx % 8 == 0;
      if (d.c_tma) ok &= store_map(&d.c_box, dx, dtype, dim, tokens, sdx);
      d.m_live = 1;
    }
    if (dw) {
      loss::Problem& d = p.prob[n++];
      ok &= slab_map(&d.a, g, dtype, plan.pitch / 64, tokens, plan.pitch);  // rows of dW beyond cols are not stored
      ok &= load_b(&d.b, d, x, dtype, dim, tokens, sx);
      if (packed_x) ok &= load_b(&d.packed, d, packed_x, dtype, dim, tokens, packed.stride);
      if (plan.copies) {
        ok &= load_b(&d.packed, d, ws + plan.x, dtype, dim, tokens, plan.pitch_x);
        p.kept = count;
      }
      shape(d, cols, dim, tokens, 1, true, loss::WIDE);
      d.k_live = 1;
      d.a_mn = 1;
      char* out = static_cast<char*>(dw) + col0 * sdw * 2;
      d.c = out;
      d.scm = sdw;
      d.c_tma = aligned(out, 16) && sdw % 8 == 0;
      if (d.c_tma) ok &= store_map(&d.c_box, out, dtype, dim, cols, sdw);
    }
    if (!ok) return fail(PCB_ERR_LAYOUT, "cuTensorMapEncodeTiled rejected the operand layout");
    p.num_tiles = p.prob[0].tiles;
    if (n > 1) p.num_tiles += p.prob[1].tiles;
    if (int st = launch_grad_products(p, s)) return st;
    if (dx && plan.splits > 1) {
      const loss::Problem& d = p.prob[0];
      const loss::JoinArgs j{acc, d.n, d.n_blocks, d.splits, p.fmt, static_cast<uint16_t*>(dx), sdx,
                             d.c_tma};
      if (int st = launch_after(loss::loss_join_kernel, "loss_join_kernel",
                                (int64_t)d.m_blocks * d.n_blocks * 4 * loss::kJoinParts, 256, s, j, p))
        return st;
    }
  }
  return PCB_OK;
}

}  // namespace

namespace pcb {
// This translation unit's device error word, read and cleared (the device is idle).
cudaError_t take_loss_device_error(unsigned int (&h)[3]) {
  cudaError_t e = cudaMemcpyFromSymbol(h, g_device_error, sizeof(h));
  const unsigned int zero[3] = {0, 0, 0};
  return e != cudaSuccess ? e : cudaMemcpyToSymbol(g_device_error, zero, sizeof(zero));
}
}  // namespace pcb

extern "C" {

int pcb_repack_u16(const void* src, int64_t rows, int64_t cols, int64_t src_stride, void* dst, int64_t dst_stride,
                   void* stream) {
  if (rows < 0 || cols < 0 || dst_stride < cols) return fail(PCB_ERR_INVALID, "bad repack sizes");
  if (cols > (1 << 26)) return fail(PCB_ERR_UNSUPPORTED, "repack: dimension too large");
  if (rows == 0 || cols == 0) return PCB_OK;
  if (!src || !dst) return fail(PCB_ERR_INVALID, "null pointer");
  if (!aligned(src, 2) || !aligned(dst, 4) || dst_stride % 2 != 0)
    return fail(PCB_ERR_LAYOUT, "repack: dst needs 4-byte aligned rows");
  const int64_t grid = std::min<int64_t>(rows, (int64_t)device_info().sm_count * 8);
  loss::repack_rows_kernel<<<(unsigned)grid, 256, 0, (cudaStream_t)stream>>>(
      static_cast<const uint16_t*>(src), rows, (int)cols, src_stride, static_cast<uint32_t*>(dst), dst_stride / 2);
  return check_launch("repack_rows_kernel");
}

int64_t pcb_linear_ce_packed_bytes(int64_t tokens, int64_t vocab, int64_t dim) {
  if (!has_workspace(tokens, vocab, dim)) return 0;
  return Order(tokens, vocab, dim).bytes;
}

int64_t pcb_linear_ce_fwd_workspace_bytes(int64_t tokens, int64_t vocab) {
  if (!has_workspace(tokens, vocab, 1)) return 0;
  return FwdPlan(tokens, vocab).bytes;
}

int pcb_linear_ce_fwd(const void* x, int64_t sx, const void* weight, int64_t sw, int dtype, int64_t tokens,
                      int64_t vocab, int64_t dim, const int64_t* target, int64_t ignore_index, int reduction,
                      float* loss_out, float* stats, float* count, void* workspace, int64_t workspace_bytes,
                      void* stream) {
  return forward(x, sx, weight, sw, dtype, tokens, vocab, dim, target, ignore_index, reduction, loss_out, stats, count,
                 nullptr, workspace, workspace_bytes, stream);
}

int pcb_linear_ce_packed_fwd(const void* x, int64_t sx, const void* weight, int64_t sw, int dtype, int64_t tokens,
                             int64_t vocab, int64_t dim, const int64_t* target, int64_t ignore_index, int reduction,
                             float* loss_out, float* stats, float* count, void* packed, int64_t packed_bytes,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  if (int st = check_packed(dtype, tokens, vocab, dim, reduction, packed, packed_bytes)) return st;
  return forward(x, sx, weight, sw, dtype, tokens, vocab, dim, target, ignore_index, reduction, loss_out, stats, count,
                 packed, workspace, workspace_bytes, stream);
}

int64_t pcb_linear_ce_bwd_workspace_bytes(int64_t tokens, int64_t vocab, int64_t dim, int64_t piece, int want_dx,
                                          int want_dw) {
  if (!has_workspace(tokens, vocab, dim)) return 0;
  const int64_t plain = BwdPlan(tokens, vocab, dim, piece, want_dx != 0, want_dw != 0, false).bytes;
  return std::max(plain, pcb_linear_ce_packed_bwd_workspace_bytes(tokens, vocab, dim, piece, want_dx, want_dw));
}

int64_t pcb_linear_ce_packed_bwd_workspace_bytes(int64_t tokens, int64_t vocab, int64_t dim, int64_t piece,
                                                 int want_dx, int want_dw) {
  if (!has_workspace(tokens, vocab, dim)) return 0;
  return BwdPlan(tokens, vocab, dim, piece, want_dx != 0, want_dw != 0, packs(tokens, vocab, dim)).bytes;
}

int pcb_linear_ce_bwd(const void* x, int64_t sx, const void* weight, int64_t sw, int dtype, int64_t tokens,
                      int64_t vocab, int64_t dim, const int64_t* target, int64_t ignore_index, int reduction,
                      const float* stats, const float* count, const float* dloss, void* dx, int64_t sdx, void* dw,
                      int64_t sdw, int64_t piece, void* workspace, int64_t workspace_bytes, void* stream) {
  return backward(x, sx, weight, sw, dtype, tokens, vocab, dim, target, ignore_index, reduction, stats, count, nullptr,
                  dloss, dx, sdx, dw, sdw, piece, workspace, workspace_bytes, stream);
}

int pcb_linear_ce_packed_bwd(const void* x, int64_t sx, const void* weight, int64_t sw, int dtype, int64_t tokens,
                             int64_t vocab, int64_t dim, const int64_t* target, int64_t ignore_index, int reduction,
                             const float* stats, const float* count, const void* packed, int64_t packed_bytes,
                             const float* dloss, void* dx, int64_t sdx, void* dw, int64_t sdw, int64_t piece,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  if (int st = check_packed(dtype, tokens, vocab, dim, reduction, packed, packed_bytes)) return st;
  return backward(x, sx, weight, sw, dtype, tokens, vocab, dim, target, ignore_index, reduction, stats, count, packed,
                  dloss, dx, sdx, dw, sdw, piece, workspace, workspace_bytes, stream);
}

}  // extern "C"
