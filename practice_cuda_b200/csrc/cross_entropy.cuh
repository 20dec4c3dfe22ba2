// Softmax cross entropy of an output projection without its logits.
//
//   l = X W^T (X [tokens, dim], W [vocab, dim]),
//   m_i = max_j l_ij, s_i = sum_j exp(l_ij - m_i), nll_i = (m_i - l_i,target) + log s_i
//   G_ij = (exp(l_ij - m_i) / s_i - [j = target_i]) w_i,  dX = a G W,  dW = a G^T X
//
// Two tcgen05 kernels, the first of them in two forms:
//   logits_kernel<kStats>     a tile of logits leaves the tensor memory as the
//              maximum and the sum of exponentials of each row's 128 columns, and
//              the target's logit; the logits are never written.
//   logits_kernel<kGradient>  the logits of one piece of the vocabulary again,
//              leaving as G in the operands' 16-bit type (the one rounding that a
//              tensor-core product of G asks for; w_i and a are split so that it
//              is of the order of 1 and the loss's scale stays in fp32); what that
//              takes from each token's own entry is kept in fp32 (see fetch_rows).
//   grad_products_kernel      dX += G W and dW = G^T X of that piece in one launch:
//              the tiles of both share the grid, so neither leaves SMs idle at its
//              end; its epilogue adds what the own entries lost.
// Logits, softmax statistics and every sum are fp32.  m and log2 s are kept apart:
// their sum would lose the small part of a sure token's probability beside a large
// logit.  The tensor cores truncate as they accumulate, which moves a logit of 4096
// products by about 3e-6 of its size towards zero, and a mean loss with it; so
// the logits' accumulators are added up in registers every 512 products (see
// kChunkStages; 2.9e-6 without).  The products of G stay in the tensor cores: what
// they lose is small beside the rounding of the gradients to 16 bits.  On 4096
// tokens of 32000 x 4096 bf16, dX and dW are 1.7e-3 and 1.6e-3 of their norm off, as
// rounding exact ones is.  Where a column is the target of many more tokens than
// are corrected (kMostCorrected), what rounding G takes shows: dW of 512 x 256 is 1.7e-3
// off with 4096 tokens, 2.1e-3 with 16384, 2.7e-3 with 262144.
//
// Tiles are 256 x 256 on a CTA pair (cta_group::2), fed by 64-deep stages of
// 128-byte swizzled operands by TMA, with two accumulators of 256 fp32 columns in
// tensor memory, so that an epilogue runs under the next products.  Up to 128
// tokens, where reading W is what takes the time, a tile is one CTA's: 128 rows
// and as many columns as spread the vocabulary evenly over the SMs.
#pragma once

#include "gemm_sm100.cuh"
#include "repack.cuh"

namespace pcb {
namespace loss {

enum Mode : int { kStats = 0, kGradient = 1 };
enum Acc : int { kAccNone = 0, kAccWrite = 1, kAccAdd = 2, kAccLast = 3, kAccSlab = 4 };

constexpr int BM = 128;            // rows of the tile per CTA
constexpr int TILE = 256;          // tile rows of the pair, and tile columns
constexpr int BK = 64;             // K elements of a stage: one 128-byte swizzle atom of 16-bit values
constexpr int UMMA_K = 16;
// Stages between two promotions of a logit's accumulator, at most.  On a B200 the
// mean loss of 4096 tokens (dim 4096) is 3.1e-7 off with 8 and takes 657 us, 2.2e-7
// and 671 us with 6, 1.4e-7 and 694 us with 4.  (Longer first chunks, which run
// while the epilogue finishes the tile before, take kGradient from 361 to 342 us at
// 4096 x 16384 x 4096 in a burst, and nothing off it under the power cap.)  On single
// CTAs, which wait for W, promotions are free.
constexpr int kChunkStages = 8, kChunkStagesSingle = 2;
constexpr int A_BYTES = BM * BK * 2;
constexpr int SLAB = 64 * BK * 2;  // 64 MN elements x 64 K rows of an MN-major operand
constexpr uint32_t K_STEP = UMMA_K * 2 >> 4;     // an instruction's K: 32 bytes along a K-major row,
constexpr uint32_t MN_STEP = UMMA_K * 128 >> 4;  // or 16 K rows of an MN-major slab
constexpr int WIDE = 2 * TILE;  // tile columns of the products of G
constexpr int NACC = 2;
constexpr int kThreads = 384;
constexpr int kEpiWarp0 = 4;
constexpr int EPI_COLS = TILE / 2;  // columns of an epilogue thread, at most
// Register split of the logit kernels (setmaxnreg), whose epilogue threads
// hold 128 fp32 accumulators: what the launch holds is checked on the host.
constexpr int kLaunchRegs = 168;
constexpr int kLowRegs = 56, kHighRegs = 224;
static_assert(128 * kLowRegs + 256 * kHighRegs == kThreads * kLaunchRegs, "register split must match the launch");
constexpr int kGroupM = 16;         // tile rows that share the columns of W in L2
constexpr int kAccVec = EPI_COLS / 4;  // float4s of an epilogue thread's share of a tile
constexpr float kLog2e = 1.4426950408889634f;
// G carries 2^kGradShift (taken out of `alpha`): its small entries (1 / vocab,
// and a column that no token is likely to take has nothing larger) stay off
// the subnormals of the 16-bit types and of the exponential, and the largest,
// 2^14, is within fp16.  The shift is a term of the exponent, so it costs nothing.
constexpr int kGradShift = 14;
constexpr float kGradScale = 16384.f;

template <bool PAIR>
struct Smem {
  static constexpr int STAGES = PAIR ? 6 : 4;
  static constexpr int B_BYTES = (PAIR ? TILE / 2 : TILE) * BK * 2;  // a pair's CTA stages half of the columns
  static constexpr int OFF_B = STAGES * A_BYTES;
  static constexpr int OFF_CSTG = OFF_B + STAGES * B_BYTES;  // 4 KB per epilogue warp
  static constexpr int OFF_BAR = OFF_CSTG + 8 * 4096;
  static constexpr int OFF_MISC = OFF_BAR + (2 * STAGES + 2 * NACC) * 8;
  static constexpr int ALLOC = OFF_MISC + 16 + 1024;  // slack for the 1 KB alignment
  static_assert(ALLOC <= 232448, "shared memory per CTA");
};

// The products of G: 48 KB stages of A and of two 128-column parts of B per CTA.
struct ProductSmem {
  static constexpr int STAGES = 4;
  static constexpr int B_BYTES = 2 * 2 * SLAB;
  static constexpr int OFF_B = STAGES * A_BYTES;
  static constexpr int OFF_CSTG = OFF_B + STAGES * B_BYTES;  // 4 KB per epilogue warp
  static constexpr int OFF_BAR = OFF_CSTG + 8 * 4096;
  static constexpr int OFF_MISC = OFF_BAR + (2 * STAGES + 4) * 8;
  static constexpr int ALLOC = OFF_MISC + 16 + 1024;
  static_assert(ALLOC <= 232448, "shared memory per CTA");
};

enum Site : int { SITE_LOSS_PRODUCER = 16, SITE_LOSS_MMA = 17, SITE_LOSS_EPILOGUE = 18, SITE_LOSS_TARGET = 19 };

// One matrix product C [m, n] = A B of a launch.
struct Problem {
  CUtensorMap a, b, c_box;
  CUtensorMap packed;  // takes the place of a (logits) or b (dW) where tokens are left out
  int m, n;
  int m_blocks, n_blocks, splits;  // splits: parts of K, each a tile of its own
  int tiles;                       // m_blocks * n_blocks * splits
  int k_stages, split_stages;
  int chunk_stages;  // of the logits: stages between two promotions
  int a_rows;        // rows of A that a load brings (K-major A)
  int m_live, k_live;  // m or k is the tokens: only those in Live count
  // products of G, where B is N-major:
  int a_mn;     // A is M-major
  int b_slabs;  // B's map takes both 64-column slabs of a 128-column part in one load
  int c_tma;  // C leaves through TMA stores
  void* c;
  long long scm;
  float4* acc;  // fp32 accumulators in tile order, for the Acc modes
  int acc_mode;
};

struct Params {
  Problem prob[2];
  int num_tiles;
  int tile_n;  // tile columns (TILE on a CTA pair)
  int fmt;  // 0 fp16, 1 bf16
  // Tokens that are left out: `order` puts the others first, `*live` says how
  // many they are, and target_packed holds the targets in that order (null: every
  // token is taken, in its own place).
  int tokens;
  const int* live;
  const int* order;
  const long long* target_packed;
  // Where nothing is packed: how many tokens count, if dW's product reads a copy
  // of X without the others' rows (null: X as it is).
  const float* kept;
  // rows
  const long long* target;
  long long ignore_index;
  long long vocab;
  const float* stats;       // [2][m]: m_i and log2 s_i
  const float* row_weight;  // null: 1
  int col0;                 // first vocabulary column of the piece
  // What rounding G took from each token's target entry, and where it goes (see
  // add_row): the operands themselves, and each target's tokens in G's order.
  float* residue;     // [tokens]
  const int* first;   // [vocab]: the first token, where there is one (else anything)
  const int* next;    // [tokens]: the next one, or kNoToken
  const uint16_t* x;
  const uint16_t* w;
  long long sx, sw;
  float2* partial;          // [n_blocks * 2][m]: maximum and sum of exponentials
  float* target_logit;      // [m]
  unsigned* ticket;         // zeroed here for the kernel that follows
  // alpha = *dloss / *count (or *dloss, or *alpha)
  const float* dloss;
  const float* count;
  const float* alpha;
};

__device__ __forceinline__ float alpha_of(const Params& p) {
  if (p.alpha) return *p.alpha;
  float a = *p.dloss;
  if (p.count) a = *p.count > 0.f ? __fdiv_rn(a, *p.count) : 0.f;
  return a * (1.f / kGradScale);
}

template <bool PAIR>
__device__ __forceinline__ void umma_f16_elect(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo,
                                               uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  if constexpr (PAIR) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t.reg .b64 ad, bd;\n\t"
        "mov.b64 ad, {%1, %2};\n\t"
        "mov.b64 bd, {%3, %4};\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %5, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t.reg .b64 ad, bd;\n\t"
        "mov.b64 ad, {%1, %2};\n\t"
        "mov.b64 bd, {%3, %4};\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], ad, bd, %5, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}

// Results below 2^-126 are zero.
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, int fmt) {
  if (fmt) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float2 unpack2(uint32_t v, int fmt) {
  if (fmt) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// 32 consecutive columns of this thread's tensor-memory lane, written.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A gradient of one token is mostly one entry of G times a row: -(1 - p) w_t in
// dX, x_i in dW's row of the target.  Rounding that entry to 16 bits moves all of
// the row by up to 2^-8 of it (bf16) together, as much as the rounding of its elements
// does: gradients up to twice as far off as their type asks for.  So the entry's
// remainder, which the logits' kernel keeps, is multiplied in the products' epilogue,
// in fp32.  A warp fetches the rows of up to 16 lanes together into its staging buffer,
// before it waits for its tile, and adds them to the accumulators in the tensor
// memory, 32 columns at a time, so that the registers of the epilogue, which holds 128
// accumulators a thread, stay as they are without.  Of 160 drawn sizes (1 to 4096 tokens,
// bf16 and fp16) the gradients' error is then 1.00 to 1.01 times that of fp32 products,
// 0.9 to 2.1 times without.  Loss and gradients of 8 tokens of 32000 x 4096 take 269 us
// so and 248 us without, of 256 tokens 297 and 273 us, of 1024 tokens 765 and 726 us, of
// 4096 tokens 3286 and 3297 us; of 512 tokens of 8192 x 4096, where nearly every tile of
// dW has rows with two tokens, 200 and 148 us, of 2048 tokens 450 and 390 us.  (Added to
// the registers after the tensor memory is given back: 355 us with 256 tokens of 32000 x
// 4096, since they spill; loaded by each lane for itself: 373 us; up to three tokens of
// a row fetched at once: 310 us, and 173 us with 512 of 8192 x 4096.)
constexpr int kFetched = 16;  // rows of 256 bytes: 4 KB
// `row` (16-byte aligned) of the lanes in `lanes`, `cols` elements of it at most.
__device__ __forceinline__ void fetch_rows(const uint16_t* row, uint32_t lanes, int cols, uint32_t stg, int lane) {
  const int u = lane & 15;  // 16 bytes of a row, two rows at a time
  const uint32_t bytes = (uint32_t)max(0, min(8, cols - u * 8)) * 2u;
  for (int r = 0; r < kFetched && lanes; r += 2) {
    const int even = __ffs(lanes) - 1;
    lanes &= lanes - 1;
    const int odd = __ffs(lanes) - 1;  // -1: no more of them
    lanes &= lanes - 1;
    const int from = lane < 16 ? even : odd, slot = r + (lane >> 4);
    const uint64_t at = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(row), max(from, 0));
    if (from >= 0 && bytes)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(stg + slot * 256u + ((uint32_t)(u ^ slot) << 4)),
                   "l"(at + u * 16u), "r"(bytes)
                   : "memory");
  }
}
// Adds f times the row in `slot` (none: -1) to the lane's 128 accumulators at taddr.
__device__ __forceinline__ void add_row(uint32_t taddr, uint32_t stg, int slot, float f, int cols, int fmt) {
#pragma unroll 1
  for (int g = 0; g < EPI_COLS / 32; ++g) {
    if (g * 32 >= cols) break;
    uint32_t v[32];
    gemm::tmem_ld32_nowait(taddr + g * 32, v);
    gemm::tmem_wait_ld();
    gemm::tmem_regs_ready(v);
    if (slot >= 0) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        uint32_t w[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(stg + slot * 256u + ((uint32_t)((g * 4 + u) ^ slot) << 4))
                     : "memory");
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 x = unpack2(w[k], fmt);
          v[u * 8 + 2 * k] = __float_as_uint(fmaf(f, x.x, __uint_as_float(v[u * 8 + 2 * k])));
          v[u * 8 + 2 * k + 1] = __float_as_uint(fmaf(f, x.y, __uint_as_float(v[u * 8 + 2 * k + 1])));
        }
      }
    }
    __syncwarp();
    tmem_st32(taddr + g * 32, v);
  }
  tmem_wait_st();
}
// Tokens of one target that are corrected so in its row of dW, one after the other:
// a column that thousands of tokens share must not hold its tile up for as many
// fetches, and beyond a few tokens their roundings cancel for the most part.
constexpr int kMostCorrected = 8;
constexpr int kNoToken = 0x7fffffff;

// The tile that worker `w` of `workers` (CTAs or pairs) takes in turn `i`, or -1:
// of t0 long tiles and then total - t0 short ones.  Workers take turns.  Where the
// long tiles do not come out even, the workers with one less of them take `extra`
// short ones in its place, and the turns go on, beginning with them.
__host__ __device__ __forceinline__ int tile_of(int t0, int total, int extra, int w, int workers, int i) {
  const int own = (t0 - w + workers - 1) / workers;
  if (i < own) return i * workers + w;
  i -= own;
  const int r = t0 % workers;
  int at = t0;
  if (r > 0) {
    if (w >= r) {
      if (i < extra) return t0 + i * (workers - r) + (w - r);
      i -= extra;
    }
    at += extra * (workers - r);
  }
  const int tile = at + i * workers + (w >= r ? w - r : w - r + workers);
  return tile < total ? tile : -1;
}
// Short tiles that workers with one long tile less take in its place.
__host__ __device__ __forceinline__ int extra_of(int long_tiles, int long_stages, int short_tiles, int short_stages,
                                                 int workers) {
  const int left = long_tiles % workers;
  if (left == 0 || short_tiles == 0 || long_tiles + short_tiles < workers) return 0;
  const int most = short_tiles / (workers - left), fit = long_stages / short_stages;
  return most < fit ? most : fit;
}

// Whether all tokens count, of which *kept do (beyond 2^24 a float cannot say).
__device__ __forceinline__ bool all_kept(const float* kept, int tokens) {
  return tokens < (1 << 24) && *kept == (float)tokens;
}

// What a launch has to do once it is known how many tokens count.
struct Live {
  int rows;       // those tokens
  bool dense;     // all of them: nothing is packed
  bool copied;    // dW reads the copy of X
  int m_blocks;   // of prob[0]
  int tiles;      // of prob[0]
  int total, extra;
  int token_stages;  // of a product over the tokens
};
__device__ __forceinline__ Live live_of(const Params& p, int tile_m, int workers) {
  Live l;
  const Problem& q = p.prob[0];
  l.rows = p.live ? *p.live : p.tokens;
  l.dense = l.rows == p.tokens;
  l.copied = !l.dense || (p.kept && !all_kept(p.kept, p.tokens));
  const int rows = max(l.rows, 1);  // without any, one row of zeros in G
  l.m_blocks = q.m_live ? (rows + tile_m - 1) / tile_m : q.m_blocks;
  l.tiles = l.m_blocks * q.n_blocks * q.splits;
  l.total = l.tiles + p.num_tiles - q.tiles;
  l.token_stages = (rows + BK - 1) / BK;
  l.extra = l.total > l.tiles ? extra_of(l.tiles, q.split_stages, l.total - l.tiles, l.token_stages, workers) : 0;
  return l;
}
__device__ __forceinline__ int tile_of(const Live& l, int w, int workers, int i) {
  return tile_of(l.tiles, l.total, l.extra, w, workers, i);
}

struct TileAt {
  int prob, mb, nb, split, index;  // index: within its problem
};
// Tiles in groups of kGroupM tile rows, rows fastest: the tiles in flight share
// few columns of B, and a group's rows of A stay in L2.
__device__ __forceinline__ TileAt locate(const Params& p, const Live& l, int tile) {
  TileAt t;
  t.prob = tile >= l.tiles ? 1 : 0;
  const Problem& q = p.prob[t.prob];
  int i = tile - (t.prob ? l.tiles : 0);
  t.index = i;
  const int m_blocks = t.prob ? q.m_blocks : l.m_blocks;
  const int area = m_blocks * q.n_blocks;
  t.split = i / area;
  i -= t.split * area;
  const int group = i / (kGroupM * q.n_blocks);
  const int rows = min(kGroupM, m_blocks - group * kGroupM);
  i -= group * kGroupM * q.n_blocks;
  t.nb = i / rows;
  t.mb = group * kGroupM + i - t.nb * rows;
  return t;
}

// 64 columns of a warp's 32 rows of the first m: every lane packs its row's 128
// bytes into the warp's staging buffer (128-byte swizzle), from where one TMA store
// takes the box.  Where C's rows do not suit TMA, or go to the places in `order`
// (not null), the warp writes row by row (columns below `limit`).
__device__ __forceinline__ void store_box(const Problem& q, const int* order, int m, const uint32_t (&w)[32],
                                          uint32_t stg, int lane, int row0, int col, int limit) {
  if (lane == 0) gemm::bulk_wait_read<0>();
  __syncwarp();
  const uint32_t swz = (uint32_t)(lane & 7);
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const uint32_t dst = stg + (uint32_t)lane * 128u + (((uint32_t)c ^ swz) << 4);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w[4 * c]), "r"(w[4 * c + 1]),
                 "r"(w[4 * c + 2]), "r"(w[4 * c + 3])
                 : "memory");
  }
  if (!order && q.c_tma) {
    gemm::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0 && row0 < m && col < q.n) gemm::tma_store_3d(&q.c_box, stg, col, row0, 0);
    return;
  }
  __syncwarp();
  uint16_t* c = static_cast<uint16_t*>(q.c);
  const int rows = min(32, m - row0);
  const int place = order && lane < rows ? order[row0 + lane] : row0 + lane;  // C's row
  if (q.c_tma && limit % 8 == 0) {  // 16 bytes a lane, four rows at a time
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + (lane >> 3), u = lane & 7;
      const long long at = __shfl_sync(0xffffffffu, place, r);
      uint4 v;
      const uint32_t src = stg + (uint32_t)r * 128u + (((uint32_t)u ^ ((uint32_t)r & 7u)) << 4);
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                   : "r"(src)
                   : "memory");
      if (r < rows && col + u * 8 < limit) *reinterpret_cast<uint4*>(c + at * q.scm + col + u * 8) = v;
    }
    __syncwarp();
    return;
  }
  for (int r = 0; r < rows; ++r) {
    const long long at = __shfl_sync(0xffffffffu, place, r);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = h * 32 + lane;  // column within the box
      uint16_t v;
      const uint32_t src = stg + (uint32_t)r * 128u + ((((uint32_t)e >> 3) ^ ((uint32_t)r & 7u)) << 4) + ((uint32_t)e & 7u) * 2u;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(src) : "memory");
      if (col + e < limit) c[at * q.scm + col + e] = v;
    }
  }
  __syncwarp();
}

// The logits of a tile and what the epilogue makes of them (MODE).  On pairs
// bound by the tensor cores' operand stream: at 4096 tokens, 16384 columns and dim
// 4096 on a B200, kStats takes 334 us (1.64 PFLOP/s, tensor pipe 92 % busy),
// kGradient, which writes 134 MB of G beside it, 364 us (83 %).  On single CTAs
// bound by reading W: 8 tokens of 32000 x 4096 in 51 us with loss_rows_kernel
// behind it (5.1 TB/s).
template <int MODE, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) logits_kernel(const __grid_constant__ Params p) {
  using S = Smem<PAIR>;
  constexpr int STAGES = S::STAGES;
  constexpr int TILE_M = PAIR ? TILE : BM;
  // Bytes of a stage on the (leader's) full barrier.
  // The rows of A below a_rows are loaded; those of the tile beyond it hold
  // whatever was there and reach no row that is stored.
  const uint32_t b_bytes = PAIR ? 2 * S::B_BYTES : (uint32_t)p.tile_n * BK * 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t s_base = smem_u32(smem);
  const uint32_t bar_full = s_base + S::OFF_BAR;      // [STAGES]
  const uint32_t bar_empty = bar_full + 8 * STAGES;   // [STAGES]
  const uint32_t bar_tfull = bar_empty + 8 * STAGES;  // [NACC]
  const uint32_t bar_tempty = bar_tfull + 8 * NACC;   // [NACC]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::OFF_MISC + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? gemm::cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const int worker = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
  const int workers = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int i = 0; i < NACC; ++i) {
      mbar_init(bar_tfull + 8 * i, 1);
      mbar_init(bar_tempty + 8 * i, PAIR ? 16 : 8);  // one arrive per epilogue warp (of both CTAs)
    }
    *abort_flag = 0;
    fence_barrier_init();
    gemm::prefetch_tmap(&p.prob[0].a);
    gemm::prefetch_tmap(&p.prob[0].b);
  }
  if constexpr (PAIR) {
    if (warp == 1) gemm::tmem_alloc_pair(smem_u32(tmem_slot), NACC * TILE);
    gemm::tc_fence_before();
    gemm::cluster_sync_all();  // both CTAs' barriers exist before any remote arrive / TMA
  } else {
    if (warp == 1) gemm::tmem_alloc(smem_u32(tmem_slot), NACC * TILE);
    gemm::tc_fence_before();
    __syncthreads();
  }
  gemm::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // Launched ahead of the previous kernel's end, which hides the launch (the kernels
  // of this file let it start only once their CTAs have left); nothing global is
  // read or written before that kernel has completed.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (MODE == kStats && blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0;
  const Live live = live_of(p, TILE_M, workers);

  if (warp < kEpiWarp0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLowRegs));
    if (warp == 0) {
      // ------------------------------ TMA producer ------------------------------
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int i = 0, tile; ok && (tile = tile_of(live, worker, workers, i)) >= 0; ++i) {
          const TileAt t = locate(p, live, tile);
          const Problem& q = p.prob[t.prob];
          const int a_row = t.mb * TILE_M + (int)rank * BM;
          const int b_col = PAIR ? t.nb * TILE + (int)rank * (TILE / 2) : t.nb * p.tile_n;
          const CUtensorMap* a_map = live.dense ? &q.a : &q.packed;
          for (int ks = 0; ks < q.k_stages; ++ks) {
            if (!mbar_spin_bounded(bar_empty + 8 * stage, phase ^ 1, abort_flag, SITE_LOSS_PRODUCER)) {
              ok = false;
              break;
            }
            const uint32_t fb = bar_full + 8 * stage;
            const uint32_t a_dst = s_base + stage * A_BYTES;
            const uint32_t b_dst = s_base + S::OFF_B + stage * S::B_BYTES;
            if (leader) mbar_arrive_expect_tx(fb, (uint32_t)(PAIR ? 2 : 1) * q.a_rows * BK * 2 + b_bytes);
            if constexpr (PAIR) {
              const uint32_t fbl = gemm::mapa_shared(fb, 0);
              gemm::tma_load_3d_pair(a_dst, a_map, fbl, ks * BK, a_row, 0);
              gemm::tma_load_3d_pair(b_dst, &q.b, fbl, ks * BK, b_col, 0);
            } else {
              gemm::tma_load_3d(a_dst, a_map, fb, ks * BK, a_row, 0);
              gemm::tma_load_3d(b_dst, &q.b, fb, ks * BK, b_col, 0);
            }
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1;
            }
          }
        }
        if (!ok) {
          // Let the copies already issued land before the CTA can exit.
          for (int s = 0; s < STAGES; ++s) mbar_wait_bounded(bar_full + 8 * s, 0, abort_flag, SITE_LOSS_PRODUCER);
        }
      }
    } else if (warp == 1) {
      // ------------------------------- MMA issuer -------------------------------
      if (leader) {
        int stage = 0;
        uint32_t phase = 0, acc_cnt = 0;
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
          return mbar_spin_bounded_warp(bar, parity, abort_flag, SITE_LOSS_MMA);
        };
        const uint64_t desc = gemm::make_sw128_desc(s_base, 16u);
        const uint32_t idesc = gemm::make_idesc(p.tile_n, p.fmt, p.fmt, 0, 0, TILE_M);
        for (int i = 0, tile; ok && (tile = tile_of(live, worker, workers, i)) >= 0; ++i) {
          const Problem& q = p.prob[0];
          int ks = 0;
          while (ks < q.k_stages && ok) {
            const uint32_t abuf = acc_cnt % NACC, d_tmem = tmem_base + abuf * TILE;
            if (!wait(bar_tempty + 8 * abuf, ((acc_cnt / NACC) & 1) ^ 1)) {
              ok = false;
              break;
            }
            const int stop = min(q.k_stages, ks + q.chunk_stages);
            for (bool fresh = true; ks < stop; ++ks, fresh = false) {
              if (!wait(bar_full + 8 * stage, phase)) {
                ok = false;
                break;
              }
              gemm::tc_fence_after();
              const uint32_t a_lo = (uint32_t)desc + (uint32_t)(stage * A_BYTES >> 4);
              const uint32_t b_lo = (uint32_t)desc + (uint32_t)((S::OFF_B + stage * S::B_BYTES) >> 4);
#pragma unroll
              for (int kk = 0; kk < BK / UMMA_K; ++kk)
                umma_f16_elect<PAIR>(d_tmem, a_lo + kk * K_STEP, (uint32_t)(desc >> 32), b_lo + kk * K_STEP,
                                     (uint32_t)(desc >> 32), idesc, (kk > 0 || !fresh) ? 1u : 0u);
              gemm::umma_commit_elect<PAIR>(bar_empty + 8 * stage);  // stage (of both CTAs) free once these retire
              if (++stage == STAGES) {
                stage = 0;
                phase ^= 1;
              }
            }
            if (!ok) break;
            gemm::umma_commit_elect<PAIR>(bar_tfull + 8 * abuf);  // accumulator ready (both CTAs)
            ++acc_cnt;
          }
        }
      }
    }
  } else {
    // -------------------------------- epilogue --------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kHighRegs));
    const int ew = warp - kEpiWarp0;  // 0..7
    const int quarter = warp & 3;     // tensor-memory lanes 32 * quarter .. + 31
    const int half = ew >> 2;         // column half
    const int half_cols = PAIR ? EPI_COLS : p.tile_n / 2;
    const uint32_t stg = s_base + S::OFF_CSTG + (uint32_t)ew * 4096u;
    const uint32_t bar_tempty_l = PAIR ? gemm::mapa_shared(bar_tempty, 0) : bar_tempty;
    uint32_t acc_cnt = 0;
    bool ok = true;
    for (int i = 0, tile; ok && (tile = tile_of(live, worker, workers, i)) >= 0; ++i) {
      const TileAt t = locate(p, live, tile);
      const Problem& q = p.prob[t.prob];
      const int row0 = t.mb * TILE_M + (int)rank * BM + quarter * 32;  // of the warp
      const int row = row0 + lane;
      const int col0 = t.nb * (PAIR ? TILE : p.tile_n) + half * half_cols;
      const int limit = min(q.n, col0 + half_cols);  // columns of this half
      const bool in = row < live.rows;
      auto wait_full = [&](uint32_t abuf) -> bool {
        if (!mbar_spin_bounded_warp(bar_tfull + 8 * abuf, (acc_cnt / NACC) & 1, abort_flag, SITE_LOSS_EPILOGUE))
          return false;
        gemm::tc_fence_after();
        return true;
      };
      auto release = [&](uint32_t abuf) {  // this warp has read its part of the accumulator
        gemm::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR) gemm::mbar_arrive_cluster(bar_tempty_l + 8 * abuf);
          else mbar_arrive(bar_tempty + 8 * abuf);
        }
      };
      auto address = [&](uint32_t abuf) {
        return tmem_base + ((uint32_t)(quarter * 32) << 16) + abuf * TILE + half * half_cols;
      };

      // Row values are read before the wait, so their latency is hidden.
      int target = -1;  // within the piece
      float top = 0.f, shift = 0.f, weight = 0.f, sure = 0.f;
      if (in) {
        const long long tv = live.dense ? p.target[row] : p.target_packed[row];
        const bool valid = tv != p.ignore_index;
        if (MODE == kGradient && valid) {
          top = p.stats[row];
          shift = (float)kGradShift - p.stats[q.m + row];
          weight = p.row_weight ? p.row_weight[row] : 1.f;
          if (tv < 0 || tv >= p.vocab) weight = NAN;  // no such column
        }
        if (valid && tv >= p.col0 + col0 && tv < p.col0 + limit) {
          target = (int)(tv - p.col0);
          if (MODE == kGradient) sure = kGradScale * expm1f(-p.stats[q.m + row] / kLog2e);
        }
      }
      // The logits: the accumulators of all chunks, summed.
      float acc[EPI_COLS];
      const int chunks = (q.k_stages + q.chunk_stages - 1) / q.chunk_stages;
      for (int ch = 0; ch < chunks; ++ch, ++acc_cnt) {
        const uint32_t abuf = acc_cnt % NACC;
        if (!wait_full(abuf)) {
          ok = false;
          break;
        }
        const uint32_t taddr = address(abuf);
        uint32_t v[2][32];
        gemm::tmem_ld32_nowait(taddr, v[0]);
        gemm::tmem_wait_ld();
        gemm::tmem_regs_ready(v[0]);
#pragma unroll
        for (int c = 0; c < EPI_COLS / 32; ++c) {
          if (c + 1 < EPI_COLS / 32) gemm::tmem_ld32_nowait(taddr + (c + 1) * 32, v[(c + 1) & 1]);
          else release(abuf);
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float x = __uint_as_float(v[c & 1][j]);
            acc[c * 32 + j] = ch == 0 ? x : acc[c * 32 + j] + x;
          }
          if (c + 1 < EPI_COLS / 32) {
            gemm::tmem_wait_ld();
            gemm::tmem_regs_ready(v[(c + 1) & 1]);
          }
        }
      }
      if (!ok) break;

      if constexpr (MODE == kStats) {
        float tl = 0.f;
        if (target >= 0) {
#pragma unroll
          for (int j = 0; j < EPI_COLS; ++j)
            if (target == col0 + j) tl = acc[j];
        }
        if (col0 + EPI_COLS > limit) {  // columns beyond this half, or the vocabulary
#pragma unroll
          for (int j = 0; j < EPI_COLS; ++j)
            if (col0 + j >= limit) acc[j] = -INFINITY;
        }
        float mc[4] = {acc[0], acc[1], acc[2], acc[3]};
#pragma unroll
        for (int j = 4; j < EPI_COLS; ++j) mc[j & 3] = fmaxf(mc[j & 3], acc[j]);
        const float m = fmaxf(fmaxf(mc[0], mc[1]), fmaxf(mc[2], mc[3]));
        const float base = m == -INFINITY ? 0.f : m;  // nothing but -inf: exp(-inf - 0) = 0
        float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < EPI_COLS; ++j) sc[j & 3] += exp2_approx((acc[j] - base) * kLog2e);
        if (in) {
          p.partial[(long long)(t.nb * 2 + half) * q.m + row] = make_float2(m, (sc[0] + sc[1]) + (sc[2] + sc[3]));
          if (target >= 0) p.target_logit[row] = tl;
        }
      } else {
#pragma unroll
        for (int b = 0; b < EPI_COLS / 64; ++b) {  // boxes of 64 columns
          uint32_t w[32];
#pragma unroll
          for (int j = 0; j < 64; ++j)
            acc[b * 64 + j] = exp2_approx(fmaf(acc[b * 64 + j] - top, kLog2e, shift));
          if (target >= col0 + b * 64 && target < col0 + b * 64 + 64) {
            float own = 0.f;
#pragma unroll
            for (int j = 0; j < 64; ++j)
              if (target == col0 + b * 64 + j) {
                // A target with more than half of the probability is the largest logit,
                // so p - 1 = 1 / s - 1: from log s itself, since in p - 1 little is left of the digits.
                const float e = acc[b * 64 + j];
                acc[b * 64 + j] = e > 0.5f * kGradScale ? sure : e - kGradScale;
                own = acc[b * 64 + j] * weight;
              }
            p.residue[row] = weight == 0.f ? 0.f : own - unpack2(pack2(own, 0.f, p.fmt), p.fmt).x;
          }
          // Tokens left out get zeros, whatever their logits are.
#pragma unroll
          for (int j = 0; j < 32; ++j)
            w[j] = weight == 0.f
                       ? 0u
                       : pack2(acc[b * 64 + 2 * j] * weight, acc[b * 64 + 2 * j + 1] * weight, p.fmt);
          if (b * 64 < half_cols) store_box(q, nullptr, q.m, w, stg, lane, row0, col0 + b * 64, limit);
        }
      }
    }
    // The staging buffers stay valid until every issued store has completed.
    if (MODE != kStats && lane == 0) gemm::bulk_wait_all();
  }

  __syncwarp();
  gemm::tc_fence_before();
  if constexpr (PAIR) {
    gemm::cluster_sync_all();  // no CTA leaves while its peer may still touch its smem / barriers
    gemm::tc_fence_after();
    if (warp == 1) gemm::tmem_dealloc_pair(tmem_base, NACC * TILE);
  } else {
    __syncthreads();
    gemm::tc_fence_after();
    if (warp == 1) gemm::tmem_dealloc(tmem_base, NACC * TILE);
  }
}

// dX = G W and dW = G^T X, or what is wanted of them, in one launch.  A CTA
// pair's tile is 256 x 512: two instructions of N = 256 share the stage of A, so
// that an SM takes in 48 bytes of operands a clock at the tensor cores' full rate
// instead of 64, and its TMA stream gives 54 to 60 at best.  That stream is what
// bounds these products, more so for operands that are not K-major: on a B200
// (4096 tokens, 16384 columns, dim 4096) dX takes 366 us and dW 345 us with the
// tensor pipe 80 % (92 % of what 128 tiles on 74 pairs allow) and 88 % busy; in
// 256 x 256 tiles 430 and 398 us.  The accumulators fill the tensor memory, so the epilogue takes a half
// into registers at once (128 fp32 a thread) and gives it back before it stores
// it, and the next tile's first stages are issued for the first half alone while
// the second is still being read.  A tile at the right edge with no more than 256
// columns has one half.
__global__ void __launch_bounds__(kThreads, 1) grad_products_kernel(const __grid_constant__ Params p) {
  using S = ProductSmem;
  constexpr int STAGES = S::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t s_base = smem_u32(smem);
  const uint32_t bar_full = s_base + S::OFF_BAR;      // [STAGES]
  const uint32_t bar_empty = bar_full + 8 * STAGES;   // [STAGES]
  const uint32_t bar_tfull = bar_empty + 8 * STAGES;  // [2] halves
  const uint32_t bar_tempty = bar_tfull + 16;         // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + S::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::OFF_MISC + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = gemm::cluster_ctarank();
  const bool leader = rank == 0;
  const int worker = (int)(blockIdx.x >> 1), workers = (int)(gridDim.x >> 1);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(bar_tfull + 8 * h, 1);
      mbar_init(bar_tempty + 8 * h, 16);  // one arrive per epilogue warp of both CTAs
    }
    *abort_flag = 0;
    fence_barrier_init();
    gemm::prefetch_tmap(&p.prob[0].a);
    gemm::prefetch_tmap(&p.prob[0].b);
  }
  if (warp == 1) gemm::tmem_alloc_pair(smem_u32(tmem_slot), WIDE);
  gemm::tc_fence_before();
  gemm::cluster_sync_all();  // both CTAs' barriers exist before any remote arrive / TMA
  gemm::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // Nothing global is read or written before the previous kernel has completed.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Live live = live_of(p, TILE, workers);

  if (warp < kEpiWarp0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLowRegs));
    if (warp == 0) {
      // ------------------------------ TMA producer ------------------------------
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int i = 0, tile; ok && (tile = tile_of(live, worker, workers, i)) >= 0; ++i) {
          const TileAt t = locate(p, live, tile);
          const Problem& q = p.prob[t.prob];
          const CUtensorMap* b_map = q.k_live && live.copied ? &q.packed : &q.b;
          const int a_row = t.mb * TILE + (int)rank * BM;
          const int b_col = t.nb * WIDE + (int)rank * (TILE / 2);
          const int halves = t.nb * WIDE + TILE < q.n ? 2 : 1;
          const uint32_t bytes = 2u * ((q.a_mn ? A_BYTES : q.a_rows * BK * 2) + halves * 2 * SLAB);
          const int ks0 = t.split * q.split_stages;
          const int ks1 = q.k_live ? live.token_stages : min(q.k_stages, ks0 + q.split_stages);
          for (int ks = ks0; ks < ks1; ++ks) {
            if (!mbar_spin_bounded(bar_empty + 8 * stage, phase ^ 1, abort_flag, SITE_LOSS_PRODUCER)) {
              ok = false;
              break;
            }
            const uint32_t fb = bar_full + 8 * stage, fbl = gemm::mapa_shared(fb, 0);
            const uint32_t a_dst = s_base + stage * A_BYTES;
            const uint32_t b_dst = s_base + S::OFF_B + stage * S::B_BYTES;
            if (leader) mbar_arrive_expect_tx(fb, bytes);
            if (q.a_mn) gemm::tma_load_3d_pair(a_dst, &q.a, fbl, 0, ks * BK, a_row / 64);
            else gemm::tma_load_3d_pair(a_dst, &q.a, fbl, ks * BK, a_row, 0);
            for (int h = 0; h < halves; ++h) {
              const uint32_t dst = b_dst + h * 2 * SLAB;
              const int col = b_col + h * TILE;
              if (q.b_slabs) {
                gemm::tma_load_3d_pair(dst, b_map, fbl, 0, ks * BK, col / 64);
              } else {
                gemm::tma_load_3d_pair(dst, b_map, fbl, col, ks * BK, 0);
                gemm::tma_load_3d_pair(dst + SLAB, b_map, fbl, col + 64, ks * BK, 0);
              }
            }
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1;
            }
          }
        }
        if (!ok) {
          // Let the copies already issued land before the CTA can exit.
          for (int s = 0; s < STAGES; ++s) mbar_wait_bounded(bar_full + 8 * s, 0, abort_flag, SITE_LOSS_PRODUCER);
        }
      }
    } else if (warp == 1 && leader) {
      // ------------------------------- MMA issuer -------------------------------
      int stage = 0;
      uint32_t phase = 0, used[2] = {0, 0};  // tiles that have filled each half
      auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
        return mbar_spin_bounded_warp(bar, parity, abort_flag, SITE_LOSS_MMA);
      };
      const uint64_t k_desc = gemm::make_sw128_desc(s_base, 16u), mn_desc = gemm::make_sw128_desc(s_base, SLAB);
      for (int i = 0, tile; (tile = tile_of(live, worker, workers, i)) >= 0; ++i) {
        const TileAt t = locate(p, live, tile);
        const Problem& q = p.prob[t.prob];
        const uint64_t a_desc = q.a_mn ? mn_desc : k_desc;
        const uint32_t a_step = q.a_mn ? MN_STEP : K_STEP;
        const uint32_t idesc = gemm::make_idesc(TILE, p.fmt, p.fmt, q.a_mn, 1, 2 * BM);
        const int ks0 = t.split * q.split_stages;
        const int stages = q.k_live ? live.token_stages : min(q.k_stages, ks0 + q.split_stages) - ks0;
        const bool wide = t.nb * WIDE + TILE < q.n;
        auto issue = [&](int st, int h, bool fresh) {
          const uint32_t a_lo = (uint32_t)a_desc + (uint32_t)(st * A_BYTES >> 4);
          const uint32_t b_lo = (uint32_t)mn_desc + (uint32_t)((S::OFF_B + st * S::B_BYTES + h * 2 * SLAB) >> 4);
#pragma unroll
          for (int kk = 0; kk < BK / UMMA_K; ++kk)
            umma_f16_elect<true>(tmem_base + h * TILE, a_lo + kk * a_step, (uint32_t)(a_desc >> 32),
                                 b_lo + kk * MN_STEP, (uint32_t)(mn_desc >> 32), idesc, (kk > 0 || !fresh) ? 1u : 0u);
        };
        auto advance = [&] {
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        };
        if (!wait(bar_tempty, (used[0] & 1) ^ 1)) break;
        bool ok = true;
        int done = 0;
        if (wide) {
          // The first stages for the first half, then for the second.
          const int head = min(stages, STAGES), stage0 = stage;
          const uint32_t phase0 = phase;
          for (int s = 0; s < head && ok; ++s) {
            ok = wait(bar_full + 8 * stage, phase);
            if (!ok) break;
            gemm::tc_fence_after();
            issue(stage, 0, s == 0);
            advance();
          }
          if (!ok) break;
          if (head == stages) gemm::umma_commit_elect<true>(bar_tfull);
          if (!wait(bar_tempty + 8, (used[1] & 1) ^ 1)) break;
          gemm::tc_fence_after();
          stage = stage0;
          phase = phase0;
          for (int s = 0; s < head; ++s) {
            issue(stage, 1, s == 0);
            gemm::umma_commit_elect<true>(bar_empty + 8 * stage);  // stage (of both CTAs) free once these retire
            advance();
          }
          done = head;
        }
        for (; done < stages; ++done) {
          ok = wait(bar_full + 8 * stage, phase);
          if (!ok) break;
          gemm::tc_fence_after();
          issue(stage, 0, done == 0);
          if (done + 1 == stages) gemm::umma_commit_elect<true>(bar_tfull);
          if (wide) issue(stage, 1, false);
          gemm::umma_commit_elect<true>(bar_empty + 8 * stage);
          advance();
        }
        if (!ok) break;
        ++used[0];
        if (wide) {
          gemm::umma_commit_elect<true>(bar_tfull + 8);
          ++used[1];
        }
      }
    }
  } else {
    // -------------------------------- epilogue --------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kHighRegs));
    const int ew = warp - kEpiWarp0;  // 0..7
    const int quarter = warp & 3;     // tensor-memory lanes 32 * quarter .. + 31
    const int part = ew >> 2;         // 128 of a half's 256 columns
    const uint32_t stg = s_base + S::OFF_CSTG + (uint32_t)ew * 4096u;
    const uint32_t bar_tempty_l = gemm::mapa_shared(bar_tempty, 0);
    const float alpha = alpha_of(p);
    uint32_t used[2] = {0, 0};
    bool ok = true;
    for (int i = 0, tile; ok && (tile = tile_of(live, worker, workers, i)) >= 0; ++i) {
      const TileAt t = locate(p, live, tile);
      const Problem& q = p.prob[t.prob];
      const int row0 = t.mb * TILE + (int)rank * BM + quarter * 32;  // of the warp
      const int halves = t.nb * WIDE + TILE < q.n ? 2 : 1;
      const bool add = q.acc_mode == kAccAdd || q.acc_mode == kAccLast;
      const bool stored = q.acc_mode == kAccNone || q.acc_mode == kAccLast;
      const int m = q.m_live ? live.rows : q.m;
      const int* order = q.m_live && !live.dense ? p.order : nullptr;
      // The token whose remainder of G the lane's row takes (see fetch_rows), or the first of
      // them: in dX the row's own, in the part of K that holds its target; in dW what `first`
      // holds for the row, if that is a token with this target.
      int head = kNoToken;
      if (row0 + lane < m) head = q.m_live ? row0 + lane : p.first[p.col0 + row0 + lane];
      int token = kNoToken;
      if ((unsigned)head < (unsigned)live.rows) {
        const long long tv = live.dense ? p.target[head] : p.target_packed[head];
        const long long k = tv - p.col0 - (long long)t.split * q.split_stages * BK;  // in dX's part of K
        const bool takes = q.m_live ? tv < p.vocab && k >= 0 && k < (long long)q.split_stages * BK
                                    : tv == p.col0 + row0 + lane;
        if (takes && tv != p.ignore_index) token = head;
      }
      for (int h = 0; h < halves; ++h) {
        const int col0 = t.nb * WIDE + h * TILE + part * EPI_COLS;
        int at = col0 < q.n ? token : kNoToken;
        uint32_t lanes = __ballot_sync(0xffffffffu, at != kNoToken);
        const uint16_t* row = nullptr;
        float rest = 0.f;
        int after = kNoToken;
        auto look_up = [&] {
          rest = p.residue[at];
          if (q.m_live) {
            row = p.w + (live.dense ? p.target[at] : p.target_packed[at]) * p.sw + col0;
          } else {
            row = p.x + (live.dense ? at : p.order[at]) * p.sx + col0;
            after = p.next[at];
          }
        };
        auto fetch = [&] {
          if (lane == 0) gemm::bulk_wait_read<0>();  // the staging buffer's last store
          __syncwarp();
          fetch_rows(row, lanes, q.n - col0, stg, lane);
        };
        if (lanes) {  // on its way while the products are
          if (at != kNoToken) look_up();
          fetch();
        }
        if (!mbar_spin_bounded_warp(bar_tfull + 8 * h, used[h] & 1, abort_flag, SITE_LOSS_EPILOGUE)) {
          ok = false;
          break;
        }
        ++used[h];
        gemm::tc_fence_after();
        const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + h * TILE + part * EPI_COLS;
        for (int taken = 1; lanes;) {
          asm volatile("cp.async.wait_all;" ::: "memory");
          __syncwarp();
          const int slot = __popc(lanes & ((1u << lane) - 1u));
          const bool mine = (lanes >> lane & 1) && slot < kFetched;
          add_row(taddr, stg, mine ? slot : -1, rest, q.n - col0, p.fmt);
          lanes &= ~__ballot_sync(0xffffffffu, mine);
          if (lanes == 0) {  // the next of each, where there are any
            at = taken++ == kMostCorrected ? kNoToken : after;
            after = kNoToken;
            lanes = __ballot_sync(0xffffffffu, at != kNoToken);
            if (at != kNoToken) look_up();
          }
          if (lanes) fetch();
        }
        uint32_t v[EPI_COLS / 32][32];
#pragma unroll
        for (int c = 0; c < EPI_COLS / 32; ++c) gemm::tmem_ld32_nowait(taddr + c * 32, v[c]);
        gemm::tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < EPI_COLS / 32; ++c) gemm::tmem_regs_ready(v[c]);
        gemm::tc_fence_before();
        __syncwarp();
        if (lane == 0) gemm::mbar_arrive_cluster(bar_tempty_l + 8 * h);

        float4* acc = nullptr;
        if (q.acc_mode != kAccNone)
          acc = q.acc + (((long long)t.index * 2 + rank) * 2 + h) * kAccVec * 256 + ew * 32 + lane;
        const bool in = row0 + lane < m;
        if (add && in) {
#pragma unroll
          for (int c = 0; c < EPI_COLS / 32; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 o = acc[(long long)(c * 8 + j) * 256];
              v[c][4 * j] = __float_as_uint(__uint_as_float(v[c][4 * j]) + o.x);
              v[c][4 * j + 1] = __float_as_uint(__uint_as_float(v[c][4 * j + 1]) + o.y);
              v[c][4 * j + 2] = __float_as_uint(__uint_as_float(v[c][4 * j + 2]) + o.z);
              v[c][4 * j + 3] = __float_as_uint(__uint_as_float(v[c][4 * j + 3]) + o.w);
            }
        }
        if (stored) {
#pragma unroll
          for (int b = 0; b < EPI_COLS / 64; ++b) {
            uint32_t w[32];
#pragma unroll
            for (int j = 0; j < 32; ++j)
              w[j] = pack2(__uint_as_float(v[2 * b + j / 16][2 * j % 32]) * alpha,
                           __uint_as_float(v[2 * b + j / 16][2 * j % 32 + 1]) * alpha, p.fmt);
            store_box(q, order, m, w, stg, lane, row0, col0 + b * 64, q.n);
          }
        } else if (in) {
#pragma unroll
          for (int c = 0; c < EPI_COLS / 32; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j)
              acc[(long long)(c * 8 + j) * 256] =
                  make_float4(__uint_as_float(v[c][4 * j]), __uint_as_float(v[c][4 * j + 1]),
                              __uint_as_float(v[c][4 * j + 2]), __uint_as_float(v[c][4 * j + 3]));
        }
      }
    }
    // The staging buffers stay valid until every issued copy and store has completed.
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (lane == 0) gemm::bulk_wait_all();
  }

  __syncwarp();
  gemm::tc_fence_before();
  gemm::cluster_sync_all();  // no CTA leaves while its peer may still touch its smem / barriers
  gemm::tc_fence_after();
  if (warp == 1) gemm::tmem_dealloc_pair(tmem_base, WIDE);
}

// ---------------------------------------------------------------------------
// The rows' statistics joined, the losses and their reduction.  A CTA
// takes 32 tokens, each of its 32 warps a strided part of the partials, read
// eight at a time.
// ---------------------------------------------------------------------------
enum Reduction : int { kNone = 0, kSum = 1, kMean = 2 };

struct RowArgs {
  const int* live;  // tokens that count, and the order that puts them first; null: every token in its place
  const int* order;
  const float2* partial;
  const float* target_logit;
  const long long* target;
  long long ignore_index, vocab;
  int tokens, parts, reduction;
  float* stats;     // [2][tokens]
  float* loss;      // [tokens] or [1]
  float* count;     // [1], tokens that are not left out
  double* sums;     // [gridDim.x][2]
  unsigned* ticket;
};

constexpr int kRowWarps = 32, kRowLoads = 8;
__global__ void __launch_bounds__(kRowWarps * 32) loss_rows_kernel(const RowArgs p) {
  // Sums of exponentials in fp64: one that is hardly above 1 holds what a sure token's loss
  // and gradients are made of.
  __shared__ float ms[kRowWarps][32];
  __shared__ double ss[kRowWarps][32];
  __shared__ double total[2][kRowWarps];
  __shared__ bool last;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x * 32 + lane;
  const int live = p.live ? *p.live : p.tokens;
  float m = -INFINITY;
  double s = 0.0;
  if (row < live) {
    for (int i = warp; i < p.parts; i += kRowWarps * kRowLoads) {
      float2 o[kRowLoads];
#pragma unroll
      for (int j = 0; j < kRowLoads; ++j) {
        const int part = i + j * kRowWarps;
        o[j] = part < p.parts ? p.partial[(long long)part * p.tokens + row] : make_float2(-INFINITY, 0.f);
      }
      float mn = m;
#pragma unroll
      for (int j = 0; j < kRowLoads; ++j) mn = fmaxf(mn, o[j].x);
      const float base = mn == -INFINITY ? 0.f : mn;
      s *= (double)exp2f((m - base) * kLog2e);
#pragma unroll
      for (int j = 0; j < kRowLoads; ++j) s += (double)(o[j].y * exp2f((o[j].x - base) * kLog2e));
      m = mn;
    }
  }
  ms[warp][lane] = m;
  ss[warp][lane] = s;
  __syncthreads();
  double nll = 0.0, valid = 0.0;
  if (warp == 0 && row < p.tokens) {
    float top = ms[0][lane];
#pragma unroll
    for (int i = 1; i < kRowWarps; ++i) top = fmaxf(top, ms[i][lane]);
    const float base = top == -INFINITY ? 0.f : top;
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kRowWarps; ++i) sum += ss[i][lane] * (double)exp2f((ms[i][lane] - base) * kLog2e);
    const float log_sum = log1pf((float)(sum - 1.0));
    p.stats[row] = base;
    p.stats[p.tokens + row] = sum < 1.5 ? log_sum * kLog2e : log2f((float)sum);
    const int at = live < p.tokens ? p.order[row] : row;  // the token's own place
    const long long t = p.target[at];
    float v = 0.f;
    if (t != p.ignore_index) {
      valid = 1.0;
      if (t < 0 || t >= p.vocab) {
        v = NAN;  // no such column
        report_error(PCB_ERR_INVALID, SITE_LOSS_TARGET);
      } else {
        v = (base - p.target_logit[row]) + log_sum;  // the maxima cancel before the small part is added
      }
      nll = (double)v;
    }
    if (p.reduction == kNone) p.loss[at] = v;
  }
  if (warp == 0) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      nll += __shfl_xor_sync(0xffffffffu, nll, o);
      valid += __shfl_xor_sync(0xffffffffu, valid, o);
    }
    if (lane == 0) {
      p.sums[2 * blockIdx.x] = nll;
      p.sums[2 * blockIdx.x + 1] = valid;
      __threadfence();
      last = atomicAdd(p.ticket, 1u) == gridDim.x - 1;
    }
  }
  __syncthreads();
  if (!last) return;
  // The CTA that comes last adds all CTAs' sums, always in the same order.
  __threadfence();
  double a = 0.0, b = 0.0;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += kRowWarps * 32) {
    a += __ldcg(p.sums + 2 * i);
    b += __ldcg(p.sums + 2 * i + 1);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (lane == 0) total[0][warp] = a, total[1][warp] = b;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kRowWarps; ++i) a += total[0][i], b += total[1][i];
    p.count[0] = (float)b;
    if (p.reduction != kNone) p.loss[0] = (float)(p.reduction == kMean ? a / b : a);  // 0 / 0: every token is left out
  }
}

// Tokens that are left out cost nothing where there are many: the others are
// packed in front, in their order, and only they are multiplied.  order[i] is the
// token in place i, those left out behind the others; *live how many others there
// are.  One CTA: a count and a position for 1024 tokens at a time.
__global__ void __launch_bounds__(1024) loss_order_kernel(const long long* target, long long ignore_index, int tokens,
                                                          int* order, int* live) {
  __shared__ int sums[33];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // First the number of tokens that count, then the places.
  int mine = 0;
  for (int i = threadIdx.x; i < tokens; i += 1024) mine += target[i] != ignore_index;
  mine = __reduce_add_sync(0xffffffffu, mine);
  if (lane == 0) sums[warp] = mine;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) total += sums[i];
  if (threadIdx.x == 0) *live = total;
  int taken = 0, left_out = total;  // next place of either kind
  for (int i0 = 0; i0 < tokens; i0 += 1024) {
    const int i = i0 + threadIdx.x;
    const bool takes = i < tokens && target[i] != ignore_index;
    const unsigned votes = __ballot_sync(0xffffffffu, takes);
    __syncthreads();
    if (lane == 0) sums[warp] = __popc(votes);
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 32; ++w) {
      before += w < warp ? sums[w] : 0;
      all += sums[w];
    }
    before += __popc(votes & ((1u << lane) - 1u));
    if (takes) order[taken + before] = i;
    else if (i < tokens) order[left_out + (int)threadIdx.x - before] = i;
    taken += all;
    left_out += min(1024, tokens - i0) - all;
  }
}

__device__ __forceinline__ void copy_row(const uint16_t* src, uint16_t* dst, int units, int dim, bool zero) {
  for (int u = threadIdx.x; u < units; u += 256) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (!zero && u * 8 + 8 <= dim) {
      v = reinterpret_cast<const uint4*>(src)[u];
    } else if (!zero && u * 8 < dim) {  // the row's last elements
      alignas(16) uint16_t e[8] = {};
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (u * 8 + k < dim) e[k] = src[u * 8 + k];
      v = *reinterpret_cast<const uint4*>(e);
    }
    reinterpret_cast<uint4*>(dst)[u] = v;
  }
}

// The rows of x and the targets in that order; zeros for the rows that a
// tile or a stage reads beyond them.  Nothing where every token counts.
__global__ void __launch_bounds__(256) loss_pack_kernel(const uint16_t* x, long long sx, const long long* target,
                                                        const int* order, const int* live, int tokens, int dim,
                                                        uint16_t* packed, long long stride, long long* target_packed) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int rows = *live;
  if (rows == tokens) return;
  const int end = min(tokens, (max(rows, 1) + TILE - 1) / TILE * TILE), units = (int)(stride / 8);
  for (int row = blockIdx.x; row < tokens; row += gridDim.x) {
    const int at = order[row];
    if (threadIdx.x == 0) target_packed[row] = target[at];
    if (row >= end) continue;
    copy_row(x + (long long)at * sx, packed + row * stride, units, dim, row >= rows);
  }
}

// Where nothing is packed, the X of dW's product, with zeros for the tokens
// that are left out: their rows of G are zeros, but what they hold may be NaN or
// infinite.  Nothing where every token counts.
__global__ void __launch_bounds__(256) loss_kept_rows_kernel(const uint16_t* x, long long sx, const long long* target,
                                                             long long ignore_index, const float* kept, int tokens,
                                                             int dim, uint16_t* out, long long stride) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (all_kept(kept, tokens)) return;
  for (int row = blockIdx.x; row < tokens; row += gridDim.x)
    copy_row(x + (long long)row * sx, out + row * stride, (int)(stride / 8), dim, target[row] == ignore_index);
}

// Each target's tokens, in G's order: first[target] is the first of them, next[i]
// the one behind token i (kNoToken: none).  Eight threads compare a token with all
// others, 4096 of them at a time, until they have found one before it and one
// behind it: as many comparisons as G has entries at most, beside 6 to 8 products of
// each of those with a row.  Which entry of `first` belongs to no token is seen by
// its token's target, so nothing has to be cleared.
constexpr int kListTokens = 32, kListThreads = 8 * kListTokens, kListTile = 4096;
__global__ void __launch_bounds__(kListThreads) loss_tokens_of_targets_kernel(const Params p, int* first, int* next) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ int4 tile[kListTile / 4];
  const int rows = p.live ? *p.live : p.tokens;
  const long long* targets = rows == p.tokens ? p.target : p.target_packed;
  auto target_of = [&](int i) -> int {  // -1: it has no column
    if (i >= rows) return -1;
    const long long t = targets[i];
    return t == p.ignore_index || t < 0 || t >= p.vocab ? -1 : (int)t;
  };
  const long long i0 = (long long)blockIdx.x * kListTokens;
  if (i0 >= rows) return;
  const int i = (int)i0 + (int)(threadIdx.x >> 3), sub = threadIdx.x & 7;
  const int own = target_of(i);
  int behind = kNoToken;
  int lead = own >= 0;
  // From the tile that holds the token to the last, then from the first to it.
  const int tiles = (int)(((long long)rows + kListTile - 1) / kListTile), mid = (int)(i0 / kListTile);
  for (int turn = 0; turn < tiles; ++turn) {
    const bool after = turn < tiles - mid;
    const int base = (after ? mid + turn : turn - (tiles - mid)) * kListTile;
    const bool open = own >= 0 && (after ? behind == kNoToken : lead != 0);
    if (!__syncthreads_or(open)) {
      if (!after) break;
      turn = tiles - mid - 1;  // on with the first tile
      continue;
    }
    const int count = min(kListTile, rows - base), quads = (count + 3) / 4;
    for (int k = threadIdx.x; k < quads; k += kListThreads)
      tile[k] = make_int4(target_of(base + 4 * k), target_of(base + 4 * k + 1), target_of(base + 4 * k + 2),
                          target_of(base + 4 * k + 3));
    __syncthreads();
    if (open) {
      for (int k = sub; k < quads; k += 8) {
        const int4 t = tile[k];
        if (t.x != own && t.y != own && t.z != own && t.w != own) continue;
        const int same[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = base + 4 * k + e;
          if (same[e] != own) continue;
          if (j < i) lead = 0;
          else if (j > i) behind = min(behind, j);
        }
        if (after ? behind != kNoToken : lead == 0) break;  // this thread's next ones are further off
      }
    }
#pragma unroll
    for (int o = 4; o; o >>= 1) {
      behind = min(behind, __shfl_xor_sync(0xffffffffu, behind, o));
      lead &= __shfl_xor_sync(0xffffffffu, lead, o);
    }
  }
  if (sub == 0 && i < rows) next[i] = behind;
  if (sub == 0 && lead) first[own] = i;
}

// Zeros for the rows of dX of tokens that are left out.
__global__ void __launch_bounds__(256) loss_zero_rows_kernel(const int* order, const int* live, int tokens, int dim,
                                                             uint16_t* dx, long long sdx, int vec) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int row = *live + blockIdx.x; row < tokens; row += gridDim.x) {
    uint16_t* dst = dx + (long long)order[row] * sdx;
    const int units = vec ? dim / 8 : 0;
    for (int u = threadIdx.x; u < units; u += 256) reinterpret_cast<uint4*>(dst)[u] = make_uint4(0, 0, 0, 0);
    for (int c = units * 8 + threadIdx.x; c < dim; c += 256) dst[c] = 0;
  }
}

// Losses that are not reduced: their gradients g_i as weights w_i = g_i / A of
// at most 1 in magnitude and the factor A (a power of two), so that G is
// rounded at the same place whatever the scale.  One CTA.
__global__ void __launch_bounds__(1024) loss_weights_kernel(const float* dloss, const long long* target,
                                                            long long ignore_index, int tokens, const int* live,
                                                            const int* order, float* weight, float* alpha) {
  __shared__ uint32_t top[32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  uint32_t m = 0;
  for (int i = threadIdx.x; i < tokens; i += 1024)
    if (target[i] != ignore_index) m = max(m, abs_bits(dloss[i]));
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32; ++i) m = max(m, top[i]);
  // Exponent of the largest magnitude; 1 where it is zero, subnormal or not finite.
  const int e = (int)(m >> 23);
  const bool usable = e >= 2 && e < 253;
  const float up = usable ? __uint_as_float((uint32_t)(e + 1) << 23) : 1.f;     // 2^(e + 1) > max
  const float down = usable ? __uint_as_float((uint32_t)(253 - e) << 23) : 1.f; // 1 / up
  const bool packed = live && *live < tokens;
  for (int i = threadIdx.x; i < tokens; i += 1024) weight[i] = dloss[packed ? order[i] : i] * down;
  if (threadIdx.x == 0) *alpha = up * (1.f / kGradScale);
}

// Rows copied to another stride, two elements (a word of dst) a thread at a
// time: a row that starts on an odd element is read as the aligned words around its
// pairs and shifted, so loads and stores stay whole and contiguous across the warp.
constexpr int kRepackLoads = 8;
struct RowIn {
  const uint16_t* e;
  __device__ __forceinline__ uint32_t pair(int i) const { return __ldg(reinterpret_cast<const uint32_t*>(e + i)); }
  __device__ __forceinline__ uint16_t half(int i) const { return __ldg(e + i); }
};
__global__ void __launch_bounds__(256) repack_rows_kernel(const uint16_t* src, long long rows, int cols,
                                                          long long src_stride, uint32_t* dst, long long dst_words) {
  const int words = (cols + 1) / 2;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const RowIn in{src + row * src_stride};
    const bool odd = reinterpret_cast<uintptr_t>(in.e) & 2;
    uint32_t* out = dst + row * dst_words;
    for (int j0 = threadIdx.x; j0 < words; j0 += 256 * kRepackLoads) {
      WordParts w[kRepackLoads];
#pragma unroll
      for (int k = 0; k < kRepackLoads; ++k) {
        const int j = j0 + k * 256;
        w[k] = j < words ? load_word_parts(in, odd, j, cols) : WordParts{0, 0};
      }
#pragma unroll
      for (int k = 0; k < kRepackLoads; ++k) {
        const int j = j0 + k * 256;
        if (j >= words) break;
        const uint32_t v = join_word_parts(w[k], odd);
        if (2 * j + 1 < cols) out[j] = v;
        else *reinterpret_cast<uint16_t*>(out + j) = (uint16_t)v;
      }
    }
  }
}

// dX from the parts of K: the fp32 accumulators of all parts summed in order.
// A thread has 32 columns of a row, 64 bytes of what it writes.
struct JoinArgs {
  const float4* acc;
  int n, n_blocks, splits, fmt;
  uint16_t* out;
  long long stride;
  int vec;  // rows of out start on 16 bytes
};
constexpr int kJoinVecs = 8;                       // float4s of a thread
constexpr int kJoinParts = kAccVec / kJoinVecs;    // of an epilogue thread's share of a half
__global__ void __launch_bounds__(256) loss_join_kernel(const JoinArgs p, const __grid_constant__ Params pp) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float alpha = alpha_of(pp);
  const Live live = live_of(pp, TILE, 1);
  // blockIdx.x: (tile of the first part, CTA of the pair, half, 32 of a thread's 128 columns)
  const int g = blockIdx.x % kJoinParts, h = blockIdx.x / kJoinParts % 2, rank = blockIdx.x / kJoinParts / 2 % 2;
  const int index = blockIdx.x / kJoinParts / 4;
  const int ew = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (index >= live.m_blocks * p.n_blocks) return;
  const TileAt t = locate(pp, live, index);
  const int row = t.mb * TILE + rank * BM + (ew & 3) * 32 + lane;
  const int col = t.nb * WIDE + h * TILE + (ew >> 2) * EPI_COLS + g * kJoinVecs * 4;
  if (row >= live.rows || col >= p.n) return;
  float4 v[kJoinVecs];
#pragma unroll
  for (int j = 0; j < kJoinVecs; ++j) v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  const long long part = (long long)live.m_blocks * p.n_blocks * 4 * kAccVec * 256;
  const float4* a = p.acc + ((((long long)index * 2 + rank) * 2 + h) * kAccVec + g * kJoinVecs) * 256 + threadIdx.x;
  for (int s = 0; s < p.splits; ++s, a += part) {
#pragma unroll
    for (int j = 0; j < kJoinVecs; ++j) {
      const float4 o = a[j * 256];
      v[j].x += o.x, v[j].y += o.y, v[j].z += o.z, v[j].w += o.w;
    }
  }
  uint16_t* out = p.out + (long long)(live.dense ? row : pp.order[row]) * p.stride + col;
#pragma unroll
  for (int j = 0; j < kJoinVecs; j += 2) {
    const float4 x = v[j], y = v[j + 1];
    const uint4 w = make_uint4(pack2(x.x * alpha, x.y * alpha, p.fmt), pack2(x.z * alpha, x.w * alpha, p.fmt),
                               pack2(y.x * alpha, y.y * alpha, p.fmt), pack2(y.z * alpha, y.w * alpha, p.fmt));
    const int c = 4 * j;
    if (p.vec && col + c + 8 <= p.n) {
      *reinterpret_cast<uint4*>(out + c) = w;
    } else {
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (col + c + k < p.n) out[c + k] = (uint16_t)(u[k / 2] >> (16 * (k & 1)));
    }
  }
}

}  // namespace loss
}  // namespace pcb
