// Backward pass of exact attention: dQ, dK and dV from q, k, v, out, dout and
// the forward pass's log-sum-exp, on tcgen05 with TMA-staged tiles.
//
//   P  = exp(scale q.k - lse)         recomputed, never stored
//   delta = rowsum(dout * out)
//   dV = P^T dout        dP = dout V^T        dS = P * (dP - delta)
//   dQ = scale dS K      dK = scale dS^T Q
//
// Two kinds of work item share one launch of persistent CTAs, one per SM,
// which take items from a counter (the longer dK/dV items first):
//   dK/dV: 128 keys of one key/value head against the query tiles of every
//     query head of its group: S^T = K Q^T, dP^T = V dO^T (keys are the rows,
//     so P^T and dS^T are written back to tensor memory as they come and are
//     the A operands of dV += P^T dO and dK += dS^T Q);
//   dQ: 128 queries of one head against the key tiles: S = Q K^T,
//     dP = dO V^T, dQ += dS K.
// S and dP are so computed twice: seven products instead of the formula's
// five.  In return no partial dQ leaves the CTA that owns it: no FP32 scratch
// of dQ's size, no atomics on results, and results that do not depend on the
// order items run in.  A single pass would add 64 KB of FP32 reductions to L2
// and a dS tile in shared memory for each pair of tiles, and is bound by
// shared-memory bandwidth (about 3750 cycles a pair at 128 B a cycle, against
// 7 * 512 for the products here).
//
// What bounds it: the products, for D > 64 and long walks (70 % of the cycles,
// at the power limit in a run of calls: 2 x 16 x 9216^2 x 128 takes 3.48 ms in a
// burst, 1399 TFLOP/s of the seven, 4.0 sustained); for D <= 64 the chain of a
// tile (product, exponentials, product, dS; 16 x 4096^2 x 64: 271 us); for few
// keys what an item costs beside its tiles, about 5000 cycles of first loads,
// results and cold code (64 heads of 9216 queries and 512 keys: 550 us).
//
// The walked tiles are 128 rows for head dimensions above 64 and 64 rows up to
// 64, where the elementwise work is what takes time: then two CTAs share an
// SM (256 TMEM columns each), and one's exponentials run beside the other's
// loads, stores and waits.
//
// Warp roles: warp 0 TMA producer and item scheduler, warp 1 MMA issuer and
// TMEM owner, the other 16 (8) warps elementwise (warp % 4 is the TMEM lane
// quadrant, and each group of four warps takes 32 columns of a tile).
// Rings, barriers and tensor memory live across items: an item's first tiles
// load and its first S and dP run while the one before stores its results.
// 18 warps put five on one scheduler, which caps registers at 96: for D > 64
// the elementwise warps spill 116 to 140 bytes (8 to 24 up to 64).
//
// Precision: products of 16-bit operands accumulated in FP32; P and dS are
// rounded once, as operands: P to the type of v, dS to that of q and k.  FP16
// has too small a range for them.  With FP16 v, P is held times 2^8; FP16 dS
// is held times a power of two chosen from the largest norms of dO and V rows
// (|dP - delta| <= 2 |dO||V|), which cannot overflow; both are taken out again
// in FP32 at the end.  So held, a dS below 2^-29 of that bound (rows of dO far
// smaller than the head's largest) loses bits to FP16's subnormals, and one
// below 2^-40 is 0.  QK16: q and k are FP16 copies (times a power of two each)
// of what v's BF16 could hold less exactly, and dQ, dK leave in FP32.
#include <cudaTypedefs.h>

#include <type_traits>

#include "kernels.h"
#include "umma.cuh"

namespace b2 {

namespace {

using namespace umma;

constexpr int kTile = 128;  // rows that an item owns
constexpr uint32_t kHalfBytes = kTile * 128;  // 128 rows x 64 16-bit columns
// Rings of the walked tiles.  K (or Q) is read by the first and the last
// product of its tile pair, so with two stages each pair waits for its load.
constexpr int kStagesA = 3, kStagesB = 2;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kShiftP16 = 8;  // FP16 v: P is held times 2^8
constexpr int kStatRows = 64;  // rows of a block of the statistics kernel

// HALVES: 64-column halves of the head dimension that the products cover.
template <int HALVES>
struct Cfg {
  static constexpr int kWalk = HALVES == 1 ? 64 : 128;  // rows of a walked tile
  static constexpr int kGroups = kWalk / 32;            // column groups of 32
  static constexpr int kElemWarps = 4 * kGroups;        // times the TMEM lane quadrants
  static constexpr int kThreads = 64 + 32 * kElemWarps;
  static constexpr int kCtas = HALVES == 1 ? 2 : 1;     // per SM
  static constexpr uint32_t kStatBytes = 2 * kWalk * 4;
  // dK/dV: P and dS take the columns of S and dP that they come from.  With
  // one CTA per SM the waits of the issuing thread that this needs are not
  // hidden (3.56 against 3.48 ms for 32 heads of 9216^2 x 128); with two they
  // are, and it saves the other warps two waits a tile (274 against 292 us
  // for 16 of 4096^2 x 64).
  static constexpr bool kInPlace = HALVES == 1;
  static constexpr bool kDpEarly = HALVES == 2;         // dQ: dP(i+1) is issued before dQ(i)
  // TMEM columns.
  //   dK/dV: S and dP take turns in kX (each is free again as soon as the
  //     elementwise warps have loaded it), P, dS, dV, dK; in place (below):
  //     S, dP, dV, dK.
  //   dQ: S, dP, dQ, dS, and Q: as the A operand of S it costs no
  //     shared-memory reads there, whose 128 bytes a cycle A and B of a
  //     128 x 128 product take all of (1.53 ms against 1.69 for all of dQ).
  //     The same for V in the dK/dV items needs P and dS to share columns, and
  //     their products to wait for one another: 2.20 ms against 2.06.
  static constexpr uint32_t kX = 0, kP = kWalk, kDS = kP + kWalk / 2, kDV = 2 * kWalk, kDK = kDV + 64 * HALVES;
  static constexpr uint32_t kS = 0, kDP = kWalk, kDQ = 2 * kWalk, kDSq = kDQ + 64 * HALVES, kQ = kDSq + kWalk / 2;
  static constexpr uint32_t kTmem = kDK + 64 * HALVES;  // 512 or 256
  static_assert(kQ + 32 * HALVES == kTmem, "both kinds of item fill the columns");
};

struct GradArgs {
  Rows dq, dk, dv;
  const float* stat;       // [B*H][query tiles][2][128]: -lse*log2e (+ shift), -delta
  const float* do_norm;    // [B*H][2 * query tiles] largest squared norms of dO rows, by 64 rows
  const float* v_norm;     // [B*Hk][v_blocks] the same of the valid V rows
  const float* qk_scale;   // QK16: the powers of two q and k are held times, or NULL
  int* counter;            // the next item
  const int32_t* key_lengths;
  int heads, kv_heads, group;
  int tq, tk, dim;
  int q_tiles, k_tiles, q_walk, v_blocks;  // own tiles, walked query tiles
  int n_dkv, n_items;  // items of the dK/dV kind (they come first), and all
  int causal;
  float scale, scale_log2;
  int* status;
};

// ------------------------------------------------------------ items
// Decoded by the producer and read by the others from shared memory: their
// code between two items runs once an item, instruction fetches and all, and
// took half of an item of four tile pairs.
struct __align__(16) Work {
  int n;         // tile pairs; -1: no item is left
  int dkv;
  int b, h, hk;  // batch, query head (dQ), key/value head
  int r0;        // the first of its own 128 rows
  int len;       // keys of the batch
  int first, per_head;  // dK/dV: the first query tile, and how many of each head
  int rows;             // own rows that exist
  char *out0, *out1;    // row r0 of dQ, or of dV and dK
  const float* stat;    // dQ: statistics of row r0
};

struct __align__(16) Misc {
  uint64_t item_full[2], item_empty[2];
  uint64_t own_full[2], own_empty[2];  // the item's own two tiles in shared memory
  uint64_t own_tmem;             // dQ: Q in tensor memory
  uint64_t a_full[kStagesA], a_empty[kStagesA];  // walked tiles: Q or K
  uint64_t b_full[kStagesB], b_empty[kStagesB];  // dO or V
  uint64_t stat_full[2], stat_empty[2];          // -lse and -delta of a query tile
  uint64_t s_full, s_read, p_full, dp_full, dp_read, ds_full, dv_done, dk_done;
  uint64_t acc_full, acc_free;  // the item's results are complete; are stored
  uint64_t exit_done;
  Work item[2];
  uint32_t tmem;
  int abort_flag;
};

template <int HALVES>
struct Smem {
  static constexpr uint32_t own_tile = HALVES * kHalfBytes, tile = HALVES * Cfg<HALVES>::kWalk * 128;
  static constexpr uint32_t own = 0;  // dK/dV: K and V; dQ: dO and Q
  static constexpr uint32_t a = own + 2 * own_tile;
  static constexpr uint32_t b = a + kStagesA * tile;
  static constexpr uint32_t stat = b + kStagesB * tile;  // [2]
  static constexpr uint32_t misc = stat + 2 * Cfg<HALVES>::kStatBytes;
  // no more CTAs to an SM than its TMEM columns serve
  static constexpr uint32_t used = misc + sizeof(Misc);
  static constexpr uint32_t least = (HALVES == 1 ? 80 : 120) * 1024;
  static constexpr uint32_t total = used < least ? least : used;
};
static_assert(Smem<2>::total <= 232448, "shared memory budget");
static_assert(2 * (Smem<1>::total + 1024) <= 233472, "two CTAs per SM");

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// A walked tile of one head: HALVES boxes of 64 columns.
template <int HALVES>
__device__ __forceinline__ void load_tile(void* dst, const CUtensorMap* map, uint64_t* bar, int row, int h, int b) {
#pragma unroll
  for (int dh = 0; dh < HALVES; ++dh)
    tma_load_4d(static_cast<char*>(dst) + dh * kHalfBytes, map, bar, dh * 64, row, h, b);
}
// An own tile: 128 rows, by boxes of as many rows as a walked tile has.
template <int HALVES>
__device__ __forceinline__ void load_own(char* dst, const CUtensorMap* map, uint64_t* bar, int row, int h, int b) {
  constexpr int kWalk = Cfg<HALVES>::kWalk;
#pragma unroll
  for (int r = 0; r < kTile; r += kWalk) load_tile<HALVES>(dst + r * 128, map, bar, row + r, h, b);
}

// Descriptors of a tile at shared-memory address `addr`, as rows of a product
// (K-major) or as its contraction (MN-major, 64-column halves kHalfBytes
// apart).  Steps inside a tile are added to the address field (16-byte
// units), one 64-bit add per MMA: building each descriptor from its address
// kept the issuing thread busy for 300 to 400 cycles a product.
__device__ __forceinline__ uint64_t rows_desc(uint32_t addr) { return smem_desc_sw128(addr, 16, 1024); }
__device__ __forceinline__ uint64_t cols_desc(uint32_t addr) { return smem_desc_sw128(addr, kHalfBytes, 1024); }

// Products cover STEPS 16-column steps of the head dimension: all that it has
// (what pads it to 64 or 128 columns is zeros).
// D[128 x walk] = A B^T over the head dimension, both tiles K-major in shared memory.
template <bool BF16, int HALVES, int STEPS>
__device__ __forceinline__ void product_rows(uint32_t d, uint64_t a_desc, uint64_t b_desc) {
  constexpr uint32_t idesc = idesc_f16(128, Cfg<HALVES>::kWalk, BF16, false, false);
#pragma unroll
  for (int kk = 0; kk < STEPS; ++kk) {
    const uint32_t off = ((kk >> 2) * kHalfBytes + (kk & 3) * 32) >> 4;
    mma_ss(d, a_desc + off, b_desc + off, idesc, kk > 0 ? 1u : 0u);
  }
}

// The same with A (16-bit pairs: 32 * HALVES columns) in tensor memory at `a`.
template <bool BF16, int HALVES, int STEPS>
__device__ __forceinline__ void product_rows_ts(uint32_t d, uint32_t a, uint64_t b_desc) {
  constexpr uint32_t idesc = idesc_f16(128, Cfg<HALVES>::kWalk, BF16, false, false);
#pragma unroll
  for (int kk = 0; kk < STEPS; ++kk)
    mma_ts(d, a + kk * 8, b_desc + (((kk >> 2) * kHalfBytes + (kk & 3) * 32) >> 4), idesc, kk > 0 ? 1u : 0u);
}

// D[128 x D] (+)= A B with A (128 x walk, 16-bit pairs) in tensor memory at
// `a`, B's rows as contraction.
template <bool BF16, int HALVES, int STEPS, bool IN_PLACE = false>
__device__ __forceinline__ void product_cols(uint32_t d, uint32_t a, uint64_t b_desc, bool accumulate) {
  constexpr uint32_t idesc = idesc_f16(128, 16 * STEPS, BF16, false, true);
#pragma unroll
  for (int kk = 0; kk < Cfg<HALVES>::kWalk / 16; ++kk)
    mma_ts(d, a + (IN_PLACE ? (kk >> 1) * 32 + (kk & 1) * 8 : kk * 8), b_desc + kk * (2048 >> 4), idesc, kk > 0 ? 1u : accumulate ? 1u : 0u);
}

__device__ __forceinline__ uint64_t pack_f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack_f2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul_f2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Powers of two of a pair of columns.  (Computing half of them with a
// polynomial on the FMA pipes instead changed nothing: 2.04 against 2.06 ms
// for dK/dV, 1.74 against 1.69 ms for dQ at 9216^2 x 32 heads.)
__device__ __forceinline__ void exp2_pair(uint64_t x2, uint32_t& p0, uint32_t& p1) {
  float a, b;
  unpack_f2(x2, a, b);
  p0 = __float_as_uint(ex2(a));
  p1 = __float_as_uint(ex2(b));
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Columns cg*32 .. +31 of row `row` of a tile in shared memory (as TMA wrote
// it: 128-byte rows, 16-byte chunks swizzled by the row) to tensor memory.
template <int HALVES>
__device__ __forceinline__ void row_to_tmem(uint32_t taddr, const char* tile, int row, int cg) {
  const char* src = tile + (cg >> 1) * kHalfBytes + row * 128;
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 x = *reinterpret_cast<const uint4*>(src + ((((cg & 1) * 4 + i) ^ (row & 7)) << 4));
    w[4 * i] = x.x, w[4 * i + 1] = x.y, w[4 * i + 2] = x.z, w[4 * i + 3] = x.w;
  }
  tmem_st16(taddr + cg * 16, w);
  tmem_wait_st();
}

// Zero the 16-bit elements of 32 packed columns whose bit is set.
__device__ __forceinline__ void clear_pairs(uint32_t (&w)[16], uint32_t bad) {
#pragma unroll
  for (int c = 0; c < 32; c += 2) {
    const uint32_t two = bad >> c;
    w[c / 2] &= (two & 1u ? 0u : 0xFFFFu) | (two & 2u ? 0u : 0xFFFF0000u);
  }
}

// The first n of 32 columns.
__device__ __forceinline__ uint32_t bad_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

__device__ __forceinline__ int key_count(const GradArgs& a, int b) {
  return a.key_lengths != nullptr ? min(max(a.key_lengths[b], 0), a.tk) : a.tk;
}

// A warp's largest of n non-negative values.
__device__ __forceinline__ float warp_most(const float* x, int64_t n, int lane) {
  float most = 0.f;
  for (int64_t i = lane; i < n; i += 32) most = fmaxf(most, x[i]);
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, w));
  return most;
}

// The least n with x < 2^n for a square x; of one that is 0 in FP32, of its least value.
__device__ __forceinline__ int square_log2(float x) { return x > 0.f ? ilogbf(x) + 1 : -148; }

// FP16 dS: the power of two it is held times (the shift of P aside), so that
// 2^shift * 2 max|dO| max|V| times it stays below 2^15.
__device__ __forceinline__ float ds_gain(const GradArgs& a, int b, int hk, int shift, int lane) {
  const int64_t bh = int64_t(b) * a.heads + int64_t(hk) * a.group, bhk = int64_t(b) * a.kv_heads + hk;
  const float do2 = warp_most(a.do_norm + bh * 2 * a.q_tiles, int64_t(a.group) * 2 * a.q_tiles, lane);
  const float v2 = warp_most(a.v_norm + bhk * a.v_blocks, a.v_blocks, lane);
  const float bound2 = do2 * v2;
  // the product where FP32 holds it: its exponent may be one less than the factors' together
  const int twice = bound2 > 1e-36f && bound2 < 3e38f ? square_log2(bound2) : square_log2(do2) + square_log2(v2);
  const int e = 15 - shift - 1 - ((twice + 1) >> 1);  // bound < 2^ceil(twice / 2)
  return ldexpf(1.f, min(max(e, -100), 100));
}

// Rows of a result tile in global memory.
struct OutTile {
  char* base;  // row 0
  int64_t step;
  int rows, dim;  // that exist; columns
};

// Columns [from, to) of a warp's 32 accumulator rows at `taddr` to global
// memory, scaled; `zero` rows (that see nothing, or lie past the keys) as
// zeros.  Four lanes store 64 bytes of a row together: stored by its own lane
// alone, each row's 16 bytes touch a line of their own, and a tile took 4500
// cycles.
template <typename TO>
__device__ __forceinline__ void store_rows(uint32_t taddr, const OutTile& o, int row, int lane, int from, int to, float mul,
                                           bool zero) {
  constexpr int kCols = 64 / sizeof(TO);  // columns of 64 bytes
  const int q = lane & 3;
#pragma unroll 1
  for (int c0 = from; c0 < to; c0 += 32) {
    uint32_t r[32];
    tmem_ld32(taddr + c0, r);
    tmem_wait_ld();
#pragma unroll
    for (int part = 0; part < 32; part += kCols) {
      uint32_t w[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if constexpr (sizeof(TO) == 4) w[e] = __float_as_uint(__uint_as_float(r[part + e]) * mul);
        else w[e] = Cvt<TO>::pack2(__uint_as_float(r[part + 2 * e]) * mul, __uint_as_float(r[part + 2 * e + 1]) * mul);
        if (zero) w[e] = 0u;
      }
      transpose_quads(w, lane);
      const int col = c0 + part + q * (kCols / 4);
      char* dst = o.base + int64_t(row - q) * o.step + col * int(sizeof(TO));
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (row - q + j < o.rows && col < o.dim)
          *reinterpret_cast<uint4*>(dst + j * o.step) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    }
  }
}

template <typename TO>
__device__ __forceinline__ void store_zero_row(char* row, int dim) {
  for (int c = 0; c < dim * int(sizeof(TO)); c += 16) *reinterpret_cast<uint4*>(row + c) = make_uint4(0u, 0u, 0u, 0u);
}

template <int HALVES>
__device__ __forceinline__ Work decode(const GradArgs& a, int id) {
  constexpr int kWalk = Cfg<HALVES>::kWalk;
  Work w;
  const int off = a.tk - a.tq;  // causal: query i sees keys up to i + off
  w.dkv = id < a.n_dkv;
  if (w.dkv) {
    const int bhk = id / a.k_tiles;
    w.r0 = (id - bhk * a.k_tiles) * kTile;
    w.b = bhk / a.kv_heads;
    w.h = 0;
    w.hk = bhk - w.b * a.kv_heads;
    w.len = key_count(a, w.b);
    w.first = a.causal ? max(0, w.r0 - off) / kWalk : 0;
    w.per_head = w.r0 < w.len ? a.q_walk - w.first : 0;
    w.n = w.per_head * a.group;
    w.rows = a.tk - w.r0;
    w.out0 = a.dv.row(bhk, w.r0);
    w.out1 = a.dk.row(bhk, w.r0);
    w.stat = nullptr;
  } else {
    id -= a.n_dkv;
    const int bh = id / a.q_tiles;
    const int qt = a.q_tiles - 1 - (id - bh * a.q_tiles);  // causal: the longest first
    w.r0 = qt * kTile;
    w.b = bh / a.heads;
    w.h = bh - w.b * a.heads;
    w.hk = w.h / a.group;
    w.len = key_count(a, w.b);
    const int keys = a.causal ? min(w.len, min(w.r0 + kTile, a.tq) + off) : w.len;  // that any of the rows sees
    w.first = w.per_head = 0;
    w.n = keys > 0 ? (keys + kWalk - 1) / kWalk : 0;
    w.rows = a.tq - w.r0;
    w.out0 = a.dq.row(bh, w.r0);
    w.out1 = nullptr;
    w.stat = a.stat + (int64_t(bh) * a.q_tiles + qt) * (2 * kTile);
  }
  return w;
}

// A place in a ring of barriers: stage and the parity of its current phase.
template <int STAGES>
struct Place {
  int s = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next() {
    if (++s == STAGES) s = 0, ph ^= 1u;
  }
};

// The next item, once the producer has published it; false if none is left
// (or on abort).
__device__ __forceinline__ bool next_item(Misc& m, const Place<2>& at, volatile int* abort_flag, int* status, Work& w) {
  if (!mbar_wait(&m.item_full[at.s], at.ph, abort_flag, status, 20)) return false;
  w = m.item[at.s];
  return w.n >= 0;
}

// ------------------------------------------------------------ TMA producer
template <int HALVES>
__device__ void produce(const CUtensorMap* q_map, const CUtensorMap* k_map, const CUtensorMap* v_map,
                        const CUtensorMap* do_map, const GradArgs& a, char* smem, Misc& m) {
  using L = Smem<HALVES>;
  constexpr int kWalk = Cfg<HALVES>::kWalk;
  volatile int* abort_flag = &m.abort_flag;
  Place<2> at, st;
  Place<kStagesA> pa;
  Place<kStagesB> pb;
  int na = 0, nb = 0, ns = 0, owns = 0, own_loads[2] = {};
  bool ok = !*abort_flag;
  auto own_tile = [&](int which, const CUtensorMap* map, const Work& w) {
    if (!mbar_wait(&m.own_empty[which], (owns & 1) ^ 1, abort_flag, a.status, 22)) return false;
    mbar_expect_tx(&m.own_full[which], L::own_tile);
    load_own<HALVES>(smem + L::own + which * L::own_tile, map, &m.own_full[which], w.r0, w.dkv ? w.hk : w.h, w.b);
    ++own_loads[which];
    return true;
  };
  while (ok) {
    const int id = atomicAdd(a.counter, 1);
    if (!(ok = mbar_wait(&m.item_empty[at.s], at.ph ^ 1, abort_flag, a.status, 21))) break;
    Work w;
    if (id < a.n_items) w = decode<HALVES>(a, id);
    else w.n = -1;
    m.item[at.s] = w;
    mbar_arrive(&m.item_full[at.s]);
    at.next();
    if (w.n < 0) break;
    // Q of a dQ item first: its tile is free once the item before has Q in tensor memory
    if (!w.dkv && w.n > 0 && !(ok = own_tile(1, q_map, w))) break;
    int g = 0, qt = w.first;  // dK/dV: head of the group and query tile
    for (int i = 0; ok && i < w.n; ++i) {
      const int h = w.hk * a.group + g;
      const int row = (w.dkv ? qt : i) * kWalk, head = w.dkv ? h : w.hk;
      if (!(ok = mbar_wait(&m.a_empty[pa.s], pa.ph ^ 1, abort_flag, a.status, 1))) break;
      mbar_expect_tx(&m.a_full[pa.s], L::tile);
      load_tile<HALVES>(smem + L::a + pa.s * L::tile, w.dkv ? q_map : k_map, &m.a_full[pa.s], row, head, w.b);
      pa.next(), ++na;
      if (w.dkv) {
        if (!(ok = mbar_wait(&m.stat_empty[st.s], st.ph ^ 1, abort_flag, a.status, 17))) break;
        mbar_expect_tx(&m.stat_full[st.s], Cfg<HALVES>::kStatBytes);
        char* dst = smem + L::stat + st.s * Cfg<HALVES>::kStatBytes;
        const float* src = a.stat + ((int64_t(w.b) * a.heads + h) * a.q_tiles + row / kTile) * (2 * kTile) + row % kTile;
        bulk_load(dst, src, kWalk * 4, &m.stat_full[st.s]);
        bulk_load(dst + kWalk * 4, src + kTile, kWalk * 4, &m.stat_full[st.s]);
        st.next(), ++ns;
      }
      if (!(ok = mbar_wait(&m.b_empty[pb.s], pb.ph ^ 1, abort_flag, a.status, 2))) break;
      mbar_expect_tx(&m.b_full[pb.s], L::tile);
      load_tile<HALVES>(smem + L::b + pb.s * L::tile, w.dkv ? do_map : v_map, &m.b_full[pb.s], row, head, w.b);
      pb.next(), ++nb;
      if (i == 0) {  // the other own tiles, once the item before has read its own
        if (!(ok = own_tile(0, w.dkv ? k_map : do_map, w))) break;
        if (w.dkv && !(ok = own_tile(1, v_map, w))) break;
        ++owns;
      }
      if (++qt == w.first + w.per_head) qt = w.first, ++g;
    }
  }
  if (*abort_flag) {
    int no_abort = 0;
    drain_loads(m.a_full, kStagesA, na, nullptr, a.status);
    drain_loads(m.b_full, kStagesB, nb, nullptr, a.status);
    drain_loads(m.stat_full, 2, ns, nullptr, a.status);
    for (int t = 0; t < 2; ++t)
      if (own_loads[t] > 0) mbar_wait(&m.own_full[t], (own_loads[t] - 1) & 1, &no_abort, a.status, 31);
  }
}

// ------------------------------------------------------------ MMA issuer
template <bool VBF16, bool QBF16, int HALVES, int STEPS>
__device__ void issue(const GradArgs& a, char* smem, Misc& m, uint32_t tmem) {
  using L = Smem<HALVES>;
  using C = Cfg<HALVES>;
  volatile int* abort_flag = &m.abort_flag;
  const uint32_t base = smem_u32(smem);
  constexpr bool kDpEarly = C::kDpEarly;
  constexpr uint32_t step = L::tile >> 4;  // stages are L::tile apart
  const uint64_t own0 = rows_desc(base + L::own), own1 = rows_desc(base + L::own + L::own_tile);
  const uint64_t a_rows = rows_desc(base + L::a), a_cols = cols_desc(base + L::a);
  const uint64_t b_rows = rows_desc(base + L::b), b_cols = cols_desc(base + L::b);
  Place<2> at;
  Place<kStagesA> ca, ta;  // stages of tile i and of tile i + 1
  Place<kStagesB> cb, tb;
  uint32_t it = 0;   // tile pairs so far: every barrier of a pair completes once a pair
  int owns = 0, dqs = 0;
  bool ok = true;
  while (ok) {
    Work w;
    if (!next_item(m, at, abort_flag, a.status, w)) break;
    mbar_arrive(&m.item_empty[at.s]);
    at.next();
    if (w.n == 0) continue;
    // the last item's products are complete: nothing is read any more from
    // the columns and tiles that this one fills
    ok = (owns == 0 || mbar_wait(&m.acc_full, (owns - 1) & 1, abort_flag, a.status, 24)) &&
         (w.dkv ? mbar_wait(&m.own_full[0], owns & 1, abort_flag, a.status, 3) &&
                      mbar_wait(&m.own_full[1], owns & 1, abort_flag, a.status, 3)
                : mbar_wait(&m.own_tmem, dqs & 1, abort_flag, a.status, 4));
    if (!ok) break;
    if (!w.dkv) mbar_arrive(&m.own_empty[1]);
    tc_fence_after();
    auto own_read = [&](int i) {  // after dP(i): the last reads of the own tiles have been issued
      if (i + 1 < w.n) return;
      mma_commit(&m.own_empty[0]);
      if (w.dkv) mma_commit(&m.own_empty[1]);
    };
    for (int i = -1; i < w.n; ++i) {
      const uint32_t ph = (it + i) & 1, next = ph ^ 1;
      const bool more = i + 1 < w.n;
      if (C::kInPlace && w.dkv) {
        // Order dV(i), S(i+1), dK(i), dP(i+1): P and dS are written over the
        // columns of the S and dP they come from, and S(i+1) and dP(i+1) wait
        // for the product that reads them.
        if (i >= 0) {
          ok = mbar_wait(&m.p_full, ph, abort_flag, a.status, 6) &&
               (i > 0 || owns == 0 || mbar_wait(&m.acc_free, (owns - 1) & 1, abort_flag, a.status, 25));
          if (!ok) break;
          tc_fence_after();
          product_cols<VBF16, HALVES, STEPS, true>(tmem + C::kDV, tmem + C::kS, b_cols + cb.s * step, i > 0);
          mma_commit(&m.b_empty[cb.s]);
          mma_commit(&m.dv_done);
          cb.next();
        }
        if (more) {
          ok = mbar_wait(&m.a_full[ta.s], ta.ph, abort_flag, a.status, 7) &&
               (i < 0 || mbar_wait(&m.dv_done, ph, abort_flag, a.status, 8));
          if (!ok) break;
          tc_fence_after();
          product_rows<QBF16, HALVES, STEPS>(tmem + C::kS, own0, a_rows + ta.s * step);
          mma_commit(&m.s_full);
          ta.next();
        }
        if (i >= 0) {
          if (!(ok = mbar_wait(&m.ds_full, ph, abort_flag, a.status, 9))) break;
          tc_fence_after();
          product_cols<QBF16, HALVES, STEPS, true>(tmem + C::kDK, tmem + C::kDP, a_cols + ca.s * step, i > 0);
          mma_commit(&m.dk_done);
          mma_commit(&m.a_empty[ca.s]);
          ca.next();
        }
        if (more) {
          ok = mbar_wait(&m.b_full[tb.s], tb.ph, abort_flag, a.status, 10) &&
               (i < 0 || mbar_wait(&m.dk_done, ph, abort_flag, a.status, 11));
          if (!ok) break;
          tc_fence_after();
          product_rows<VBF16, HALVES, STEPS>(tmem + C::kDP, own1, b_rows + tb.s * step);
          mma_commit(&m.dp_full);
          own_read(i + 1);
          tb.next();
        }
      } else if (w.dkv) {
        // Order S(i+1), dV(i), dP(i+1), dK(i): S and dP wait for the
        // elementwise warps to have loaded the other out of their common
        // columns, and dV or dK runs while they do.
        if (more) {
          ok = mbar_wait(&m.a_full[ta.s], ta.ph, abort_flag, a.status, 7) &&
               (i < 0 || mbar_wait(&m.dp_read, ph, abort_flag, a.status, 8));
          if (!ok) break;
          tc_fence_after();
          product_rows<QBF16, HALVES, STEPS>(tmem + C::kX, own0, a_rows + ta.s * step);
          mma_commit(&m.s_full);
          ta.next();
        }
        if (i >= 0) {
          ok = mbar_wait(&m.p_full, ph, abort_flag, a.status, 6) &&
               (i > 0 || owns == 0 || mbar_wait(&m.acc_free, (owns - 1) & 1, abort_flag, a.status, 25));
          if (!ok) break;
          tc_fence_after();
          product_cols<VBF16, HALVES, STEPS>(tmem + C::kDV, tmem + C::kP, b_cols + cb.s * step, i > 0);
          mma_commit(&m.b_empty[cb.s]);
          cb.next();
        }
        if (more) {
          ok = mbar_wait(&m.b_full[tb.s], tb.ph, abort_flag, a.status, 10) &&
               mbar_wait(&m.s_read, next, abort_flag, a.status, 11);
          if (!ok) break;
          tc_fence_after();
          product_rows<VBF16, HALVES, STEPS>(tmem + C::kX, own1, b_rows + tb.s * step);
          mma_commit(&m.dp_full);
          own_read(i + 1);
          tb.next();
        }
        if (i >= 0) {
          if (!(ok = mbar_wait(&m.ds_full, ph, abort_flag, a.status, 9))) break;
          tc_fence_after();
          product_cols<QBF16, HALVES, STEPS>(tmem + C::kDK, tmem + C::kDS, a_cols + ca.s * step, i > 0);
          mma_commit(&m.dk_done);
          mma_commit(&m.a_empty[ca.s]);
          ca.next();
        }
      } else {
        // Order S(i+1), dP(i+1), dQ(i): each goes out as soon as the
        // elementwise warps have read the one before, and runs under their
        // arithmetic of tile i.  With two CTAs per SM the other's products
        // do that, and the wait it saves counts: dP(i+1) last (288 us
        // against 300 for 16 x 4096 x 64).
        auto dp = [&] {
          ok = mbar_wait(&m.b_full[tb.s], tb.ph, abort_flag, a.status, 10) &&
               (i >= 0 || mbar_wait(&m.own_full[0], owns & 1, abort_flag, a.status, 3));
          if (!ok) return;
          if constexpr (kDpEarly) {
            if (i >= 0 && !(ok = mbar_wait(&m.dp_read, ph, abort_flag, a.status, 11))) return;
          }
          tc_fence_after();
          product_rows<VBF16, HALVES, STEPS>(tmem + C::kDP, own0, b_rows + tb.s * step);
          mma_commit(&m.dp_full);
          mma_commit(&m.b_empty[tb.s]);
          own_read(i + 1);
          tb.next(), cb.next();
        };
        if (more) {  // the elementwise warps hold S(i)
          ok = mbar_wait(&m.a_full[ta.s], ta.ph, abort_flag, a.status, 7) &&
               (i < 0 || mbar_wait(&m.s_read, ph, abort_flag, a.status, 8));
          if (!ok) break;
          tc_fence_after();
          product_rows_ts<QBF16, HALVES, STEPS>(tmem + C::kS, tmem + C::kQ, a_rows + ta.s * step);
          mma_commit(&m.s_full);
          ta.next();
        }
        if (kDpEarly && more) {
          dp();
          if (!ok) break;
        }
        if (i >= 0) {
          ok = mbar_wait(&m.ds_full, ph, abort_flag, a.status, 9) &&
               (i > 0 || owns == 0 || mbar_wait(&m.acc_free, (owns - 1) & 1, abort_flag, a.status, 25));
          if (!ok) break;
          tc_fence_after();
          product_cols<QBF16, HALVES, STEPS>(tmem + C::kDQ, tmem + C::kDSq, a_cols + ca.s * step, i > 0);
          if constexpr (kDpEarly) mma_commit(&m.dk_done);
          mma_commit(&m.a_empty[ca.s]);
          ca.next();
        }
        if (!kDpEarly && more) {
          dp();
          if (!ok) break;
        }
      }
    }
    if (!ok) break;
    mma_commit(&m.acc_full);
    it += w.n;
    ++owns;
    dqs += w.dkv ? 0 : 1;
  }
  // every product completes before TMEM is released (bounded by time only,
  // even after an abort)
  mma_commit(&m.exit_done);
  int no_abort = 0;
  mbar_wait(&m.exit_done, 0, &no_abort, a.status, 12);
}

// ------------------------------------------------------------ elementwise
template <bool VBF16, bool QBF16, bool OUT32, int HALVES>
__device__ void elementwise(const GradArgs& a, char* smem, Misc& m, uint32_t tmem) {
  using T = typename std::conditional<VBF16, __nv_bfloat16, __half>::type;   // v, dO, P
  using TS = typename std::conditional<QBF16, __nv_bfloat16, __half>::type;  // q, k, dS
  using TO = typename std::conditional<OUT32, float, TS>::type;              // dQ, dK
  using L = Smem<HALVES>;
  using C = Cfg<HALVES>;
  constexpr int kWalk = C::kWalk;
  constexpr int kShift = VBF16 ? 0 : kShiftP16;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int cg = (warp - 2) >> 2;  // column group: columns cg*32 .. +31 of a tile
  const int sub = warp & 3;
  const int row = sub * 32 + lane;
  const uint32_t lanes = static_cast<uint32_t>(sub * 32) << 16;
  const int off = a.tk - a.tq;
  volatile int* abort_flag = &m.abort_flag;
  float q_scale = 1.f, k_scale = 1.f;
  if (a.qk_scale != nullptr) q_scale = a.qk_scale[0], k_scale = a.qk_scale[1];
  const float mul_s = a.scale_log2 / (q_scale * k_scale);
  const uint64_t scale2 = pack_f2(mul_s, mul_s);
  constexpr float p_mul = 1.f / static_cast<float>(1 << kShift);
  const float mul_dk = a.scale * p_mul / q_scale, mul_dq = a.scale * p_mul / k_scale;
  const int64_t step_dv = a.dv.st * int64_t(sizeof(T)), step_dk = a.dk.st * int64_t(sizeof(TO)),
                step_dq = a.dq.st * int64_t(sizeof(TO));
  Place<2> at, st;
  uint32_t it = 0;
  int owns = 0;
  bool ok = true;
  bool q_ready = false;  // dQ: the item's Q is in tensor memory already
  // Items stay in shared memory while they are worked on (copies of their
  // fields would not fit the registers beside two tiles' columns).
  auto have = [&](const Place<2>& p) {
    return mbar_wait(&m.item_full[p.s], p.ph, abort_flag, a.status, 20) && m.item[p.s].n >= 0;
  };
  // Q of a dQ item (owns: the item's number among those with products)
  auto take_q = [&](int number) {
    if (!mbar_wait(&m.own_full[1], number & 1, abort_flag, a.status, 27)) return false;
    row_to_tmem<HALVES>(tmem + lanes + C::kQ, smem + L::own + L::own_tile, row, cg);
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&m.own_tmem);
    return true;
  };
  bool any = have(at);
  while (any) {
    const Work& w = m.item[at.s];
    const int own = w.r0 + row;  // key or query
    if (w.n == 0) {  // column groups 0 and 1: zeros for dV and dK, or dQ
      if (row < w.rows && cg == 0) {
        if (w.dkv) store_zero_row<T>(w.out0 + row * step_dv, a.dim);
        else store_zero_row<TO>(w.out0 + row * step_dq, a.dim);
      }
      if (row < w.rows && cg == 1 && w.dkv) store_zero_row<TO>(w.out1 + row * step_dk, a.dim);
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.item_empty[at.s]);
      at.next();
      any = have(at);
      continue;
    }
    const int n = w.n, len = w.len;
    float gain = 1.f;
    if constexpr (!QBF16) gain = ds_gain(a, w.b, w.hk, kShift, lane);
    const uint64_t gain2 = pack_f2(gain, gain);
    if (w.dkv) {
      const uint32_t s_addr = tmem + lanes + C::kX + cg * 32;  // kX is kS
      const uint32_t dp_addr = C::kInPlace ? tmem + lanes + C::kDP + cg * 32 : s_addr;
      const uint32_t p_addr = C::kInPlace ? s_addr : tmem + lanes + C::kP + cg * 16;
      const uint32_t ds_addr = C::kInPlace ? dp_addr : tmem + lanes + C::kDS + cg * 16;
      int lim = own - off - w.first * kWalk - cg * 32;  // causal: columns below it are queries before the key
      int qt = 0;
      for (int i = 0; i < n; ++i) {
        const uint32_t ph = (it + i) & 1;
        const float* stat = reinterpret_cast<const float*>(smem + L::stat + st.s * C::kStatBytes) + cg * 32;
        const int before = lim;
        if (a.causal) {
          lim -= kWalk;
          if (++qt == w.per_head) lim += w.per_head * kWalk, qt = 0;
        }
        const bool masked = a.causal && before > 0;
        if (!(ok = mbar_wait(&m.stat_full[st.s], st.ph, abort_flag, a.status, 13))) break;
        if (!(ok = mbar_wait(&m.s_full, ph, abort_flag, a.status, 14))) break;
        tc_fence_after();
        uint32_t v[32], p[16];
        tmem_ld32(s_addr, v);
        tmem_wait_ld();
        if constexpr (!C::kInPlace) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&m.s_read);
        }
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const float4 nl = *reinterpret_cast<const float4*>(stat + c);
          exp2_pair(fma_f2(pack_f2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), scale2, pack_f2(nl.x, nl.y)), v[c],
                    v[c + 1]);
          exp2_pair(fma_f2(pack_f2(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3])), scale2, pack_f2(nl.z, nl.w)),
                    v[c + 2], v[c + 3]);
          p[c / 2] = Cvt<T>::pack2(__uint_as_float(v[c]), __uint_as_float(v[c + 1]));
          p[c / 2 + 1] = Cvt<T>::pack2(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3]));
        }
        if (masked) clear_pairs(p, bad_below(before));
        if constexpr (C::kInPlace) {
          tmem_st16(p_addr, p);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&m.p_full);
            mbar_arrive(&m.s_read);  // for the parity of dQ items' waits
          }
        }
        // dP(i) was issued after dV(i-1), so with it done P's columns are free
        if (!(ok = mbar_wait(&m.dp_full, ph, abort_flag, a.status, 15))) break;
        tc_fence_after();
        uint32_t d[32];
        if constexpr (!C::kInPlace) tmem_st16(p_addr, p);
        tmem_ld32(dp_addr, d);
        if constexpr (!C::kInPlace) tmem_wait_st();
        tmem_wait_ld();
        if constexpr (!C::kInPlace) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&m.dp_read);
            mbar_arrive(&m.p_full);
          }
        }
        // dS = P (dP - delta)
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const float4 nd = *reinterpret_cast<const float4*>(stat + kWalk + c);
#pragma unroll
          for (int e = c; e < c + 4; e += 2) {
            uint64_t pe = pack_f2(__uint_as_float(v[e]), __uint_as_float(v[e + 1]));
            if constexpr (!QBF16) pe = mul_f2(pe, gain2);
            const uint64_t x = mul_f2(pe, add_f2(pack_f2(__uint_as_float(d[e]), __uint_as_float(d[e + 1])),
                                                 e == c ? pack_f2(nd.x, nd.y) : pack_f2(nd.z, nd.w)));
            float x0, x1;
            unpack_f2(x, x0, x1);
            p[e / 2] = Cvt<TS>::pack2(x0, x1);
          }
        }
        if (masked) clear_pairs(p, bad_below(before));  // 0 * inf
        if constexpr (!C::kInPlace) {
          if (i > 0 && !(ok = mbar_wait(&m.dk_done, ph ^ 1, abort_flag, a.status, 19))) break;  // the last dS is read
          tc_fence_after();
        }
        tmem_st16(ds_addr, p);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&m.stat_empty[st.s]);
          mbar_arrive(&m.ds_full);
        }
        st.next();
      }
    } else {
      const uint32_t s_addr = tmem + lanes + C::kS + cg * 32;
      const uint32_t dp_addr = tmem + lanes + C::kDP + cg * 32;
      const uint32_t ds_addr = tmem + lanes + C::kDSq + cg * 16;
      if (!q_ready) {
        // Q takes columns that a dK/dV item's results may still be read from
        ok = (owns == 0 || mbar_wait(&m.acc_free, (owns - 1) & 1, abort_flag, a.status, 26)) && take_q(owns);
        if (!ok) break;
      }
      const float nl = w.stat[row], nd = w.stat[kTile + row];
      const uint64_t nl2 = pack_f2(nl, nl), nd2 = pack_f2(nd, nd);
      const int seen = a.causal ? min(len, own + off + 1) : len;  // keys this row sees
      for (int i = 0; i < n; ++i) {
        const uint32_t ph = (it + i) & 1;
        const int lim = seen - i * kWalk - cg * 32;  // columns from `lim` on are masked
        if (!(ok = mbar_wait(&m.s_full, ph, abort_flag, a.status, 14))) break;
        tc_fence_after();
        uint32_t v[32];
        tmem_ld32(s_addr, v);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.s_read);
#pragma unroll
        for (int c = 0; c < 32; c += 2)
          exp2_pair(fma_f2(pack_f2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), scale2, nl2), v[c], v[c + 1]);
        // a partly valid last key tile: rows past the keys may hold anything,
        // and dS's zeros times inf or NaN would reach dQ
        const int k0 = i * kWalk;
        if (len < min(k0 + kWalk, a.tk)) {
          const int tid = threadIdx.x - 64;
          const int from = len - k0, rows = min(kWalk, a.tk - k0) - from;
          char* tile = smem + L::a + ((it + i) % kStagesA) * L::tile;
          for (int x = tid; x < rows * 8 * HALVES; x += 32 * C::kElemWarps) {
            const int r = from + x / (8 * HALVES), ch = x % (8 * HALVES);
            *reinterpret_cast<uint4*>(tile + (ch >> 3) * kHalfBytes + r * 128 + (ch & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
        }
        if (!(ok = mbar_wait(&m.dp_full, ph, abort_flag, a.status, 15))) break;
        tc_fence_after();
        uint32_t d[32], ds[16];
        tmem_ld32(dp_addr, d);
        tmem_wait_ld();
        if constexpr (C::kDpEarly) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&m.dp_read);
        }
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          uint64_t p = pack_f2(__uint_as_float(v[c]), __uint_as_float(v[c + 1]));
          if constexpr (!QBF16) p = mul_f2(p, gain2);
          float x0, x1;
          unpack_f2(mul_f2(p, add_f2(pack_f2(__uint_as_float(d[c]), __uint_as_float(d[c + 1])), nd2)), x0, x1);
          ds[c / 2] = Cvt<TS>::pack2(x0, x1);
        }
        if (lim < 32) clear_pairs(ds, ~bad_below(lim));
        if constexpr (C::kDpEarly) {
          if (i > 0 && !(ok = mbar_wait(&m.dk_done, ph ^ 1, abort_flag, a.status, 19))) break;  // the last dS is read
          tc_fence_after();
        }  // otherwise dP(i) was issued after dQ(i-1)
        tmem_st16(ds_addr, ds);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.ds_full);
      }
    }
    ok = ok && mbar_wait(&m.acc_full, owns & 1, abort_flag, a.status, 16);
    if (!ok || *abort_flag) break;
    tc_fence_after();
    // between dQ items the next Q goes in first, so that the next S and dP run
    // while this item's results are stored
    Place<2> then = at;
    then.next();
    any = have(then);
    q_ready = any && !w.dkv && !m.item[then.s].dkv && m.item[then.s].n > 0;
    if (q_ready && !take_q(owns + 1)) break;
    float inv_gain = 1.f;
    if constexpr (!QBF16) inv_gain = 1.f / gain;
    if (w.dkv) {  // the first half of the column groups stores dV, the second dK, 64 columns each
      const int from = cg % (C::kGroups / 2) * 64, to = from + 64;
      if (cg >= C::kGroups / 2)
        store_rows<TO>(tmem + lanes + C::kDK, OutTile{w.out1, step_dk, w.rows, a.dim}, row, lane, from, to,
                       mul_dk * inv_gain, own >= len);
      else
        store_rows<T>(tmem + lanes + C::kDV, OutTile{w.out0, step_dv, w.rows, a.dim}, row, lane, from, to, p_mul,
                      own >= len);
    } else {
      const bool none = (a.causal ? min(len, own + off + 1) : len) <= 0;
      store_rows<TO>(tmem + lanes + C::kDQ, OutTile{w.out0, step_dq, w.rows, a.dim}, row, lane, cg * 32, cg * 32 + 32,
                     mul_dq * inv_gain, none);
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) {
      mbar_arrive(&m.acc_free);
      mbar_arrive(&m.item_empty[at.s]);
    }
    it += n;
    ++owns;
    at = then;
  }
}

template <bool VBF16, bool QBF16, bool OUT32, int HALVES>
__global__ void __launch_bounds__(Cfg<HALVES>::kThreads, Cfg<HALVES>::kCtas)
attn_grad_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                 const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap do_map,
                 const __grid_constant__ GradArgs a) {
  extern __shared__ __align__(1024) char smem[];
  constexpr int kElemWarps = Cfg<HALVES>::kElemWarps;
  Misc& m = *reinterpret_cast<Misc*>(smem + Smem<HALVES>::misc);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    m.abort_flag = 0;
    if ((smem_u32(smem) & 1023u) != 0) {
      m.abort_flag = 1;
      atomicCAS(a.status, 0, 0x300);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&m.item_full[s], 1);
      mbar_init(&m.item_empty[s], 1 + kElemWarps);
      mbar_init(&m.stat_full[s], 1);
      mbar_init(&m.stat_empty[s], kElemWarps);
    }
    for (int s = 0; s < kStagesA; ++s) {
      mbar_init(&m.a_full[s], 1);
      mbar_init(&m.a_empty[s], 1);
    }
    for (int s = 0; s < kStagesB; ++s) {
      mbar_init(&m.b_full[s], 1);
      mbar_init(&m.b_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&m.own_full[t], 1);
      mbar_init(&m.own_empty[t], 1);
    }
    mbar_init(&m.own_tmem, kElemWarps);
    mbar_init(&m.s_full, 1);
    mbar_init(&m.s_read, kElemWarps);
    mbar_init(&m.p_full, kElemWarps);
    mbar_init(&m.dp_full, 1);
    mbar_init(&m.dp_read, kElemWarps);
    mbar_init(&m.ds_full, kElemWarps);
    mbar_init(&m.dv_done, 1);
    mbar_init(&m.dk_done, 1);
    mbar_init(&m.acc_full, 1);
    mbar_init(&m.acc_free, kElemWarps);
    mbar_init(&m.exit_done, 1);
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  grid_dep_wait();  // the statistics and the counter come from the kernel before
  if (warp == 1) tmem_alloc<Cfg<HALVES>::kTmem>(&m.tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = m.tmem;
  if (warp == 0) {
    if ((threadIdx.x & 31) == 0) produce<HALVES>(&q_map, &k_map, &v_map, &do_map, a, smem, m);
  } else if (warp == 1) {
    if (elect_one())
      with_steps<HALVES>(a.dim, [&](auto steps) { issue<VBF16, QBF16, HALVES, decltype(steps)::value>(a, smem, m, tmem); });
  } else {
    elementwise<VBF16, QBF16, OUT32, HALVES>(a, smem, m, tmem);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<Cfg<HALVES>::kTmem>(tmem);
  }
}

// ------------------------------------------------------------ row statistics
struct StatArgs {
  Rows out, out_low, dout, v;  // out_low: what out's type could not hold of the output, or no base
  const float* lse;
  float* stat;
  float* do_norm;
  float* v_norm;
  int* counter;
  const int32_t* key_lengths;
  int heads, kv_heads;
  int tq, tk, dim;
  int causal;
  int q_tiles, v_blocks;
  int q_blocks;  // blocks of the query part; the rest walks V (NORMS)
};

// A group of 16 lanes sums x[u] for each u: lane l returns that of u = l >> 2
// (the exchanges halve the values still held: 5 shuffles for the 4 sums).
__device__ __forceinline__ float sum_rows(const float (&x)[4], int l) {
  const bool h8 = l & 8, h4 = l & 4;
  const float y0 = (h8 ? x[2] : x[0]) + __shfl_xor_sync(0xffffffffu, h8 ? x[0] : x[2], 8);
  const float y1 = (h8 ? x[3] : x[1]) + __shfl_xor_sync(0xffffffffu, h8 ? x[1] : x[3], 8);
  float z = (h4 ? y1 : y0) + __shfl_xor_sync(0xffffffffu, h4 ? y0 : y1, 4);
  z += __shfl_xor_sync(0xffffffffu, z, 2);
  return z + __shfl_xor_sync(0xffffffffu, z, 1);
}

// (a + low) . b of eight elements; LOW: whether there is a low part.
template <typename T, bool LOW>
__device__ __forceinline__ float dot8(const uint4& a, const uint4& low, const uint4& b) {
  const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, lw[4] = {low.x, low.y, low.z, low.w}, bw[4] = {b.x, b.y, b.z, b.w};
  uint64_t sum = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a0, a1, b0, b1;
    Cvt<T>::unpack2(aw[i], a0, a1);
    Cvt<T>::unpack2(bw[i], b0, b1);
    uint64_t a2 = pack_f2(a0, a1);
    if constexpr (LOW) {
      Cvt<T>::unpack2(lw[i], a0, a1);
      a2 = add_f2(a2, pack_f2(a0, a1));
    }
    sum = fma_f2(a2, pack_f2(b0, b1), sum);
  }
  float s0, s1;
  unpack_f2(sum, s0, s1);
  return s0 + s1;
}

// -lse*log2e and -delta of every query row, padded to whole tiles with rows
// that give P = 0.  NORMS: also the largest finite squared norms of 64 dO rows
// and of 64 valid V rows (rows that are not finite say nothing of the others).  Block 0 resets the item counter of the kernel after.
// A block takes 64 rows of one head, 16 lanes a row and four rows of each
// lane at a time.  What counts is instructions: with a row address and
// separate shuffles for each row it took 80 us for 64 heads of 9216 x 128 (16
// of them without keys, so not read), and takes 56.
template <typename T, bool NORMS>
__global__ void __launch_bounds__(256) attn_grad_stat_kernel(const __grid_constant__ StatArgs a) {
  constexpr int kShift = std::is_same<T, __half>::value ? kShiftP16 : 0;
  __shared__ float part[8];
  const int g = threadIdx.x >> 4;
  const int l = threadIdx.x & 15;
  const bool active = 8 * l < a.dim;
  const bool queries = static_cast<int>(blockIdx.x) < a.q_blocks;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.counter = 0;
  const int id = queries ? blockIdx.x : blockIdx.x - a.q_blocks;
  const int per_head = queries ? a.q_tiles * (kTile / kStatRows) : a.v_blocks;
  const int head = id / per_head;
  const int r0 = (id - head * per_head) * kStatRows;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  float most = 0.f;
  if (queries) {
    const int len = a.key_lengths != nullptr ? min(max(a.key_lengths[head / a.heads], 0), a.tk) : a.tk;
    const int mine = r0 + (l >> 2) * 16 + g;  // the row this lane writes
    const float lse = (l & 3) == 0 && mine < a.tq ? a.lse[int64_t(head) * a.tq + mine] : -INFINITY;
    const int rows = active && len > 0 ? a.tq - r0 - g : 0;  // rows without a key have no gradient
    float sum[4] = {}, norm[4] = {};
    const int64_t o_step = a.out.st * int64_t(16 * sizeof(T)), d_step = a.dout.st * int64_t(16 * sizeof(T));
    const char* op = a.out.row(head, r0 + g) + l * 16;
    const char* dp = a.dout.row(head, r0 + g) + l * 16;
    uint4 o[4], d[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool in = u * 16 < rows;
      o[u] = in ? *reinterpret_cast<const uint4*>(op + u * o_step) : zero;
      d[u] = in ? *reinterpret_cast<const uint4*>(dp + u * d_step) : zero;
    }
    const int low_end = a.out_low.base != nullptr ? low_rows(len, a.tq, a.causal, a.tk - a.tq) : 0;
    if (r0 < low_end) {
      const char* lp = a.out_low.row(head, r0 + g) + l * 16;
      const int64_t l_step = a.out_low.st * int64_t(16 * sizeof(T));
      uint4 low[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) low[u] = u * 16 < min(rows, low_end - r0 - g) ? *reinterpret_cast<const uint4*>(lp + u * l_step) : zero;
#pragma unroll
      for (int u = 0; u < 4; ++u) sum[u] = dot8<T, true>(o[u], low[u], d[u]);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) sum[u] = dot8<T, false>(o[u], zero, d[u]);
    }
    const float delta = sum_rows(sum, l);
    if constexpr (NORMS) {
#pragma unroll
      for (int u = 0; u < 4; ++u) norm[u] = dot8<T, false>(d[u], zero, d[u]);
      most = sum_rows(norm, l);
    }
    if ((l & 3) == 0) {
      float* dst = a.stat + (int64_t(head) * a.q_tiles + mine / kTile) * (2 * kTile) + mine % kTile;
      dst[0] = lse == -INFINITY ? -INFINITY : -lse * kLog2e + static_cast<float>(kShift);
      dst[kTile] = -delta;
    }
  } else if constexpr (NORMS) {
    const int b = head / a.kv_heads;
    const int len = a.key_lengths != nullptr ? min(a.key_lengths[b], a.tk) : a.tk;
    const int rows = active ? len - r0 - g : 0;
    const char* vp = a.v.row(head, r0 + g) + l * 16;
    const int64_t v_step = a.v.st * int64_t(16 * sizeof(T));
    uint4 x[4];
    float norm[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = u * 16 < rows ? *reinterpret_cast<const uint4*>(vp + u * v_step) : zero;
#pragma unroll
    for (int u = 0; u < 4; ++u) norm[u] = dot8<T, false>(x[u], zero, x[u]);
    most = sum_rows(norm, l);
  }
  if constexpr (NORMS) {
    if (!(most < INFINITY)) most = 0.f;
#pragma unroll
    for (int w = 16; w >= 4; w >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, w));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 8; ++w) most = fmaxf(most, part[w]);
      (queries ? a.do_norm : a.v_norm)[int64_t(head) * per_head + r0 / kStatRows] = most;
    }
  }
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Byte offsets in the workspace.
struct Layout {
  size_t stat, do_norm, v_norm, counter, total;
};
Layout layout_of(int64_t bh, int64_t bhk, int64_t q_tiles, int64_t v_blocks) {
  Layout l;
  l.stat = 0;
  l.do_norm = align256(size_t(bh) * q_tiles * 2 * kTile * 4);
  l.v_norm = l.do_norm + align256(size_t(bh) * q_tiles * 2 * 4);
  l.counter = l.v_norm + align256(size_t(bhk) * v_blocks * 4);
  l.total = l.counter + 256;
  return l;
}

template <bool VBF16, bool QBF16, bool OUT32, int HALVES>
cudaError_t launch_grad(const CUtensorMap* maps, const GradArgs& a, cudaStream_t st) {
  const auto kernel = attn_grad_kernel<VBF16, QBF16, OUT32, HALVES>;
  const int smem = static_cast<int>(Smem<HALVES>::total);
  const cudaError_t err = ensure_smem(reinterpret_cast<const void*>(kernel), smem);
  if (err != cudaSuccess) return err;
  const int most = sm_count() * Cfg<HALVES>::kCtas;
  return launch_pdl(kernel, dim3(a.n_items < most ? a.n_items : most), dim3(Cfg<HALVES>::kThreads), size_t(smem), st, maps[0], maps[1],
                    maps[2], maps[3], a);
}

template <int HALVES>
cudaError_t launch_halves(bool v_bf16, bool qk16, const CUtensorMap* maps, const GradArgs& a, cudaStream_t st) {
  if (qk16)
    return v_bf16 ? launch_grad<true, false, true, HALVES>(maps, a, st) : launch_grad<false, false, true, HALVES>(maps, a, st);
  return v_bf16 ? launch_grad<true, true, false, HALVES>(maps, a, st) : launch_grad<false, false, false, HALVES>(maps, a, st);
}

}  // namespace

int64_t attn_grad_workspace_bytes(int batch, int heads, int kv_heads, int tq, int tk) {
  return static_cast<int64_t>(layout_of(int64_t(batch) * heads, int64_t(batch) * kv_heads, (int64_t(tq) + kTile - 1) / kTile,
                                        (int64_t(tk) + kStatRows - 1) / kStatRows)
                                  .total);
}

cudaError_t launch_attn_grad(const AttnGradCall& c, int* status, cudaStream_t st) {
  const b2_view &q = *c.q, &k = *c.k;
  CUtensorMap maps[4];
  const b2_view* views[4] = {c.q, c.k, c.v, c.dout};
  for (int i = 0; i < 4; ++i)
    if (!linear_rows_map(&maps[i], *views[i], q.head_dim <= 64 ? Cfg<1>::kWalk : Cfg<2>::kWalk)) return cudaErrorInvalidValue;
  const bool v_bf16 = c.v->dtype == B2_BF16, qk16 = c.qk_scale != nullptr;
  const int64_t bh = int64_t(q.batch) * q.heads, bhk = int64_t(q.batch) * k.heads;
  StatArgs s{};
  s.out = make_rows(*c.out), s.dout = make_rows(*c.dout), s.v = make_rows(*c.v);
  if (c.out_low != nullptr) s.out_low = make_rows(*c.out_low);
  s.lse = c.lse;
  s.key_lengths = c.key_lengths;
  s.heads = q.heads, s.kv_heads = k.heads;
  s.tq = q.tokens, s.tk = k.tokens, s.dim = q.head_dim;
  s.causal = c.causal;
  s.q_tiles = (q.tokens + kTile - 1) / kTile;
  s.v_blocks = (k.tokens + kStatRows - 1) / kStatRows;
  const Layout l = layout_of(bh, bhk, s.q_tiles, s.v_blocks);
  char* ws = static_cast<char*>(c.workspace);
  s.stat = reinterpret_cast<float*>(ws + l.stat);
  s.do_norm = reinterpret_cast<float*>(ws + l.do_norm);
  s.v_norm = reinterpret_cast<float*>(ws + l.v_norm);
  s.counter = reinterpret_cast<int*>(ws + l.counter);
  s.q_blocks = static_cast<int>(bh * s.q_tiles * (kTile / kStatRows));
  const bool norms = !v_bf16 || qk16;  // dS in FP16
  const int blocks = s.q_blocks + (norms ? static_cast<int>(bhk * s.v_blocks) : 0);
  if (!v_bf16) attn_grad_stat_kernel<__half, true><<<blocks, 256, 0, st>>>(s);
  else if (norms) attn_grad_stat_kernel<__nv_bfloat16, true><<<blocks, 256, 0, st>>>(s);
  else attn_grad_stat_kernel<__nv_bfloat16, false><<<blocks, 256, 0, st>>>(s);
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  GradArgs a{};
  a.dq = make_rows(*c.dq), a.dk = make_rows(*c.dk), a.dv = make_rows(*c.dv);
  a.stat = s.stat, a.do_norm = s.do_norm, a.v_norm = s.v_norm;
  a.qk_scale = c.qk_scale;
  a.counter = s.counter;
  a.key_lengths = c.key_lengths;
  a.heads = s.heads, a.kv_heads = s.kv_heads, a.group = q.heads / k.heads;
  a.tq = s.tq, a.tk = s.tk, a.dim = s.dim;
  a.q_tiles = s.q_tiles, a.v_blocks = s.v_blocks;
  const int walk = q.head_dim <= 64 ? Cfg<1>::kWalk : Cfg<2>::kWalk;
  a.q_walk = (q.tokens + walk - 1) / walk;
  a.k_tiles = (k.tokens + kTile - 1) / kTile;
  a.n_dkv = static_cast<int>(bhk * a.k_tiles);
  a.n_items = static_cast<int>(a.n_dkv + bh * a.q_tiles);
  a.causal = c.causal;
  a.scale = c.scale;
  a.scale_log2 = c.scale * kLog2e;
  a.status = status;
  return q.head_dim <= 64 ? launch_halves<1>(v_bf16, qk16, maps, a, st) : launch_halves<2>(v_bf16, qk16, maps, a, st);
}

}  // namespace b2
