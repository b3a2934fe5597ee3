// Backward pass of exact attention: dQ, dK and dV from q, k, v, out, dout and
// the forward pass's log-sum-exp, on tcgen05 with TMA-staged tiles.
//
//   P  = exp(scale q.k - lse)         recomputed, never stored
//   delta = rowsum(dout * out)
//   dV = P^T dout        dP = dout V^T        dS = P * (dP - delta)
//   dQ = scale dS K      dK = scale dS^T Q
//
// Two kinds of CTA share one launch:
//   dK/dV: owns 128 keys of one key/value head and walks the query tiles of
//     every query head of its group: S^T = K Q^T, dP^T = V dO^T (keys are the
//     rows, so P^T and dS^T are written back to tensor memory as they come and
//     are the A operands of dV += P^T dO and dK += dS^T Q);
//   dQ: owns 128 queries of one head and walks the key tiles: S = Q K^T,
//     dP = dO V^T, dQ += dS K.
// S and dP are so computed twice: seven products instead of the formula's
// five.  In return no partial dQ leaves the CTA that owns it: no FP32 scratch
// of dQ's size, no atomics, and results that do not depend on the order CTAs
// run in.  A single pass would add 64 KB of FP32 reductions to L2 and a dS
// tile in shared memory for each pair of tiles, and is bound by shared-memory
// bandwidth (about 3750 cycles a pair at 128 B a cycle, against 7 * 512 for
// the products here).
//
// Warp roles (576 threads, one CTA per SM): warp 0 TMA producer, warp 1 MMA
// issuer and TMEM owner, warps 2..17 elementwise (warp % 4 is the TMEM lane
// quadrant, and each group of four warps takes 32 columns of a tile).
//
// Precision: products of 16-bit operands accumulated in FP32; P and dS are
// rounded to the inputs' type once, as operands.  FP16 has too small a range
// for them, so there P is held times 2^8 and dS times a power of two chosen
// from the largest norms of dO and V rows (|dP - delta| <= 2 |dO||V|), which
// cannot overflow; both are taken out again in FP32 at the end.
#include <cudaTypedefs.h>

#include <type_traits>

#include "kernels.h"
#include "umma.cuh"

namespace b2 {

namespace {

using namespace umma;

constexpr int kTile = 128;
constexpr int kElemWarps = 16;  // 4 TMEM lane quadrants x 4 column groups of 32
constexpr int kThreads = 64 + 32 * kElemWarps;
constexpr uint32_t kHalfBytes = kTile * 128;  // 128 rows x 64 16-bit columns
constexpr uint32_t kStatBytes = 2 * kTile * 4;
// Rings of the walked tiles.  K (or Q) is read by the first and the last
// product of its tile pair, so with two stages each pair waits for its load.
// The second ring gets what the CTA's own tiles leave.
constexpr int kStagesA = 3, kStagesDkv = 2, kStagesDq = 3, kMaxB = 3;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kShiftP16 = 8;  // FP16: P is held times 2^8

// TMEM columns.
//   dK/dV: S and dP take turns in kColX (each is free again as soon as the
//     elementwise warps have loaded it), P, dS, dV, dK.
//   dQ: S, dP, dQ, dS, and Q: as the A operand of S it costs no shared-memory
//     reads there, whose 128 bytes a cycle A and B of a 128 x 128 product
//     take all of (1.53 ms against 1.69 for all of dQ).  The same for V in the
//     dK/dV CTAs needs P and dS to share columns, and their products to wait
//     for one another: 2.20 ms against 2.06.
constexpr uint32_t kColX = 0, kColP = 128, kColDS = 192, kColDV = 256, kColDK = 384;
constexpr uint32_t kColS = 0, kColDP = 128, kColDQ = 256, kColDSq = 384, kColQ = 448;

struct GradArgs {
  Rows q, dq, dk, dv;
  const float* stat;       // [B*H][query tiles][2][128]: -lse*log2e (+ shift), -delta
  const uint32_t* maxima;  // FP16: [B*Hk][2] bits of the largest squared norms of dO and V rows
  const int32_t* key_lengths;
  int heads, kv_heads, group;
  int tq, tk, dim;
  int q_tiles, k_tiles;
  int n_dkv;  // CTAs of the dK/dV kind (they come first)
  int causal;
  float scale, scale_log2;
  int* status;
};

struct __align__(8) Misc {
  uint64_t own_full;      // the CTA's own tile (two for dK/dV) in shared memory
  uint64_t own_tmem;      // dQ: Q in tensor memory
  uint64_t a_full[kStagesA], a_empty[kStagesA];  // walked tiles: Q or K
  uint64_t b_full[kMaxB], b_empty[kMaxB];  // dO or V
  uint64_t stat_full[2], stat_empty[2];          // -lse and -delta of a query tile
  uint64_t s_full, s_read, p_full, dp_full, dp_read, ds_full;
  uint64_t dk_done, all_done;
  uint32_t tmem;
  int abort_flag;
};

template <int HALVES>
struct Smem {
  static constexpr uint32_t tile = HALVES * kHalfBytes;
  static constexpr uint32_t a = 0;
  static constexpr uint32_t own = a + kStagesA * tile;  // dK/dV: K and V; dQ: dO
  static constexpr uint32_t b_dkv = own + 2 * tile, b_dq = own + tile;
  static constexpr uint32_t stat = own + 4 * tile;  // [2]
  static constexpr uint32_t misc = stat + 2 * kStatBytes;
  // one CTA per SM (each owns all 512 TMEM columns)
  static constexpr uint32_t used = misc + sizeof(Misc);
  static constexpr uint32_t total = used < 120 * 1024 ? 120 * 1024 : used;
};
static_assert(Smem<2>::total <= 232448, "shared memory budget");

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// 128 rows of one head as HALVES boxes of 64 columns.
template <int HALVES>
__device__ __forceinline__ void load_tile(void* dst, const CUtensorMap* map, uint64_t* bar, int row, int h, int b) {
#pragma unroll
  for (int dh = 0; dh < HALVES; ++dh)
    tma_load_4d(static_cast<char*>(dst) + dh * kHalfBytes, map, bar, dh * 64, row, h, b);
}

// Descriptors of a tile at shared-memory address `addr`, as rows of a product
// (K-major) or as its contraction (MN-major, 64-column halves kHalfBytes
// apart).  Steps inside a tile are added to the address field (16-byte
// units), one 64-bit add per MMA: building each descriptor from its address
// kept the issuing thread busy for 300 to 400 cycles a product.
__device__ __forceinline__ uint64_t rows_desc(uint32_t addr) { return smem_desc_sw128(addr, 16, 1024); }
__device__ __forceinline__ uint64_t cols_desc(uint32_t addr) { return smem_desc_sw128(addr, kHalfBytes, 1024); }

// D[128 x 128] = A B^T over the head dimension, both tiles K-major in shared memory.
template <bool BF16, int HALVES>
__device__ __forceinline__ void product_rows(uint32_t d, uint64_t a_desc, uint64_t b_desc) {
  constexpr uint32_t idesc = idesc_f16(128, 128, BF16, false, false);
#pragma unroll
  for (int kk = 0; kk < 4 * HALVES; ++kk) {
    const uint32_t off = ((kk >> 2) * kHalfBytes + (kk & 3) * 32) >> 4;
    mma_ss(d, a_desc + off, b_desc + off, idesc, kk > 0 ? 1u : 0u);
  }
}

// The same with A (16-bit pairs: 32 * HALVES columns) in tensor memory at `a`.
template <bool BF16, int HALVES>
__device__ __forceinline__ void product_rows_ts(uint32_t d, uint32_t a, uint64_t b_desc) {
  constexpr uint32_t idesc = idesc_f16(128, 128, BF16, false, false);
#pragma unroll
  for (int kk = 0; kk < 4 * HALVES; ++kk)
    mma_ts(d, a + kk * 8, b_desc + (((kk >> 2) * kHalfBytes + (kk & 3) * 32) >> 4), idesc, kk > 0 ? 1u : 0u);
}

// D[128 x D] (+)= A B with A (128 x 128, 16-bit pairs: 64 columns) in tensor
// memory at `a`, B's rows as contraction.
template <bool BF16, int HALVES>
__device__ __forceinline__ void product_cols(uint32_t d, uint32_t a, uint64_t b_desc, bool accumulate) {
  constexpr uint32_t idesc = idesc_f16(128, 64 * HALVES, BF16, false, true);
#pragma unroll
  for (int kk = 0; kk < 8; ++kk)
    mma_ts(d, a + kk * 8, b_desc + kk * (2048 >> 4), idesc, kk > 0 ? 1u : accumulate ? 1u : 0u);
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

// One row of the CTA's own operand to tensor memory: columns cg*32 .. +31 of
// the head dimension (zeros past it, and for no row) by column group cg.
template <int HALVES>
__device__ __forceinline__ void row_to_tmem(uint32_t taddr, const char* row, int cg, int dim) {
  if (cg >= 2 * HALVES) return;
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (row != nullptr && cg * 32 + 8 * i < dim) x = *reinterpret_cast<const uint4*>(row + cg * 64 + 16 * i);
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

__device__ __forceinline__ int key_count(const GradArgs& a, int b) {
  return a.key_lengths != nullptr ? min(max(a.key_lengths[b], 0), a.tk) : a.tk;
}

// FP16: the power of two dS is held times (P's 2^8 aside), so that
// 2^8 * 2 max|dO| max|V| times it stays below 2^15.
__device__ __forceinline__ float ds_gain(const GradArgs& a, int bhk) {
  const float bound2 = __uint_as_float(a.maxima[2 * bhk]) * __uint_as_float(a.maxima[2 * bhk + 1]);
  if (!(bound2 > 0.f) || !(bound2 < 3e38f)) return 1.f;
  const int e = 15 - kShiftP16 - 1 - 1 - (ilogbf(bound2) >> 1);  // bound < 2^(ilogb(bound2)/2 + 1)
  return ldexpf(1.f, min(max(e, -60), 60));
}

// Store 32 FP32 accumulator columns of one row, scaled, as 16-bit.
template <typename T>
__device__ __forceinline__ void store_cols(char* row, int c0, int dim, const uint32_t* r, float mul) {
  uint32_t w[16];
#pragma unroll
  for (int c = 0; c < 32; c += 2) w[c / 2] = Cvt<T>::pack2(__uint_as_float(r[c]) * mul, __uint_as_float(r[c + 1]) * mul);
  uint4* dst = reinterpret_cast<uint4*>(row + c0 * 2);
#pragma unroll
  for (int q4 = 0; q4 < 4; ++q4)
    if (c0 + 8 * q4 < dim) dst[q4] = make_uint4(w[4 * q4], w[4 * q4 + 1], w[4 * q4 + 2], w[4 * q4 + 3]);
}

// Columns [from, to) of one accumulator row at `taddr` to global memory; a row
// that sees nothing (or lies past the keys) is written as zeros.  The loads
// are a warp's: every lane calls this, row NULL stores nothing.
template <typename T>
__device__ __forceinline__ void store_row(uint32_t taddr, char* row, int from, int to, int dim, float mul, bool zero) {
#pragma unroll 1
  for (int c0 = from; c0 < to; c0 += 32) {
    uint32_t r[32];
    tmem_ld32(taddr + c0, r);
    tmem_wait_ld();
    if (row == nullptr) continue;
    if (zero) {
#pragma unroll
      for (int c = 0; c < 32; ++c) r[c] = 0u;
    }
    store_cols<T>(row, c0, dim, r, mul);
  }
}

template <typename T>
__device__ __forceinline__ void store_zero_row(char* row, int dim) {
  for (int c = 0; c < dim; c += 8) *reinterpret_cast<uint4*>(row + c * 2) = make_uint4(0u, 0u, 0u, 0u);
}

// ------------------------------------------------------------ dK and dV
template <bool BF16, int HALVES>
__device__ __forceinline__ void dkv_cta(const CUtensorMap* q_map, const CUtensorMap* k_map, const CUtensorMap* v_map,
                                        const CUtensorMap* do_map, const GradArgs& a, char* smem, Misc& m,
                                        uint32_t tmem) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  using L = Smem<HALVES>;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int kt = blockIdx.x % a.k_tiles;
  const int bhk = blockIdx.x / a.k_tiles;
  const int b = bhk / a.kv_heads;
  const int hk = bhk - b * a.kv_heads;
  const int k0 = kt * kTile;
  const int len = key_count(a, b);
  const int off = a.tk - a.tq;  // causal: query i sees keys up to i + off
  const int first = a.causal ? max(0, k0 - off) / kTile : 0;
  const int per_head = k0 < len ? a.q_tiles - first : 0;
  const int n = per_head * a.group;
  volatile int* abort_flag = &m.abort_flag;

  if (warp == 0) {
    if (lane == 0 && n > 0 && !*abort_flag) {
      mbar_expect_tx(&m.own_full, 2 * L::tile);
      load_tile<HALVES>(smem + L::own, k_map, &m.own_full, k0, hk, b);
      load_tile<HALVES>(smem + L::own + L::tile, v_map, &m.own_full, k0, hk, b);
      int na = 0, nb = 0, ns = 0;
      for (int i = 0; i < n; ++i) {
        const int sa = i % kStagesA, sb = i % kStagesDkv, ss = i & 1;
        const int g = i / per_head;
        const int qt = first + i - g * per_head;
        const int h = hk * a.group + g;
        if (!mbar_wait(&m.a_empty[sa], ((i / kStagesA) & 1) ^ 1, abort_flag, a.status, 1)) break;
        mbar_expect_tx(&m.a_full[sa], L::tile);
        load_tile<HALVES>(smem + L::a + sa * L::tile, q_map, &m.a_full[sa], qt * kTile, h, b);
        na = i + 1;
        if (!mbar_wait(&m.stat_empty[ss], ((i >> 1) & 1) ^ 1, abort_flag, a.status, 17)) break;
        mbar_expect_tx(&m.stat_full[ss], kStatBytes);
        bulk_load(smem + L::stat + ss * kStatBytes, a.stat + ((int64_t(b) * a.heads + h) * a.q_tiles + qt) * (2 * kTile),
                  kStatBytes, &m.stat_full[ss]);
        ns = i + 1;
        if (!mbar_wait(&m.b_empty[sb], ((i / kStagesDkv) & 1) ^ 1, abort_flag, a.status, 2)) break;
        mbar_expect_tx(&m.b_full[sb], L::tile);
        load_tile<HALVES>(smem + L::b_dkv + sb * L::tile, do_map, &m.b_full[sb], qt * kTile, h, b);
        nb = i + 1;
      }
      if (*abort_flag) {
        drain_loads(m.a_full, kStagesA, na, &m.own_full, a.status);
        drain_loads(m.b_full, kStagesDkv, nb, nullptr, a.status);
        drain_loads(m.stat_full, 2, ns, nullptr, a.status);
      }
    }
  } else if (warp == 1) {
    if (n > 0 && elect_one()) {
      const uint32_t base = smem_u32(smem);
      const uint64_t k_rows = rows_desc(base + L::own), v_rows = rows_desc(base + L::own + L::tile);
      const uint64_t q_rows = rows_desc(base + L::a), q_cols = cols_desc(base + L::a);  // stage 0; stages L::tile apart
      const uint64_t do_rows = rows_desc(base + L::b_dkv), do_cols = cols_desc(base + L::b_dkv);
      constexpr uint32_t step = L::tile >> 4;
      bool ok = mbar_wait(&m.own_full, 0, abort_flag, a.status, 3);
      // Order S(i+1), dV(i), dP(i+1), dK(i): S and dP wait for the elementwise
      // warps to have loaded the other out of their common columns, and dV or
      // dK runs while they do.
      for (int i = -1; ok && i < n; ++i) {
        const int sa = i < 0 ? 0 : i % kStagesA, sb = i < 0 ? 0 : i % kStagesDkv;
        const int ta = (i + 1) % kStagesA, tb = (i + 1) % kStagesDkv;  // the next tiles' stages and phases
        const uint32_t ph = i & 1, next = ph ^ 1, ta_ph = ((i + 1) / kStagesA) & 1, tb_ph = ((i + 1) / kStagesDkv) & 1;
        const bool more = i + 1 < n;
        if (more) {
          ok = mbar_wait(&m.a_full[ta], ta_ph, abort_flag, a.status, 7) &&
               (i < 0 || mbar_wait(&m.dp_read, ph, abort_flag, a.status, 8));
          if (!ok) break;
          tc_fence_after();
          product_rows<BF16, HALVES>(tmem + kColX, k_rows, q_rows + ta * step);
          mma_commit(&m.s_full);
        }
        if (i >= 0) {
          if (!(ok = mbar_wait(&m.p_full, ph, abort_flag, a.status, 6))) break;
          tc_fence_after();
          product_cols<BF16, HALVES>(tmem + kColDV, tmem + kColP, do_cols + sb * step, i > 0);
          mma_commit(&m.b_empty[sb]);
        }
        if (more) {
          ok = mbar_wait(&m.b_full[tb], tb_ph, abort_flag, a.status, 10) &&
               mbar_wait(&m.s_read, next, abort_flag, a.status, 11);
          if (!ok) break;
          tc_fence_after();
          product_rows<BF16, HALVES>(tmem + kColX, v_rows, do_rows + tb * step);
          mma_commit(&m.dp_full);
        }
        if (i >= 0) {
          if (!(ok = mbar_wait(&m.ds_full, ph, abort_flag, a.status, 9))) break;
          tc_fence_after();
          product_cols<BF16, HALVES>(tmem + kColDK, tmem + kColDS, q_cols + sa * step, i > 0);
          mma_commit(&m.dk_done);
          mma_commit(&m.a_empty[sa]);
        }
      }
      // every product completes before TMEM is read and released (bounded by
      // time only, even after an abort)
      mma_commit(&m.all_done);
      int no_abort = 0;
      mbar_wait(&m.all_done, 0, &no_abort, a.status, 12);
    }
  } else {
    const int cg = (warp - 2) >> 2;  // column group: queries cg*32 .. +31 of a tile
    const int sub = warp & 3;
    const int row = sub * 32 + lane;
    const int key = k0 + row;
    const uint32_t lanes = static_cast<uint32_t>(sub * 32) << 16;
    const uint32_t s_addr = tmem + lanes + kColX + cg * 32;
    const uint32_t p_addr = tmem + lanes + kColP + cg * 16, ds_addr = tmem + lanes + kColDS + cg * 16;
    float gain = 1.f;
    if constexpr (!BF16) gain = ds_gain(a, bhk);
    const uint64_t gain2 = pack_f2(gain, gain);
    const uint64_t scale2 = pack_f2(a.scale_log2, a.scale_log2);
    bool ok = true;
    int qt = 0;  // query tile after the first
    for (int i = 0; i < n; ++i) {
      const int s = i & 1;
      const uint32_t ph = i & 1;
      const float* stat = reinterpret_cast<const float*>(smem + L::stat + s * kStatBytes) + cg * 32;
      uint32_t bad = 0u;  // causal: columns below `lim` are queries before the key
      if (a.causal) {
        const int lim = key - off - (first + qt) * kTile - cg * 32;
        bad = lim <= 0 ? 0u : lim >= 32 ? ~0u : (1u << lim) - 1u;
        qt = qt + 1 < per_head ? qt + 1 : 0;
      }
      if (!(ok = mbar_wait(&m.stat_full[s], (i >> 1) & 1, abort_flag, a.status, 13))) break;
      if (!(ok = mbar_wait(&m.s_full, ph, abort_flag, a.status, 14))) break;
      tc_fence_after();
      uint32_t v[32], w[16];
      tmem_ld32(s_addr, v);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.s_read);
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        const float4 nl = *reinterpret_cast<const float4*>(stat + c);
        exp2_pair(fma_f2(pack_f2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), scale2, pack_f2(nl.x, nl.y)),
                  v[c], v[c + 1]);
        exp2_pair(fma_f2(pack_f2(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3])), scale2, pack_f2(nl.z, nl.w)),
                  v[c + 2], v[c + 3]);
        w[c / 2] = Cvt<T>::pack2(__uint_as_float(v[c]), __uint_as_float(v[c + 1]));
        w[c / 2 + 1] = Cvt<T>::pack2(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3]));
      }
      if (bad != 0u) clear_pairs(w, bad);
      // dP(i) was issued after dV(i-1), so with it done P's columns are free
      if (!(ok = mbar_wait(&m.dp_full, ph, abort_flag, a.status, 15))) break;
      tc_fence_after();
      uint32_t d[32];
      tmem_st16(p_addr, w);
      tmem_ld32(s_addr, d);
      tmem_wait_st();
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&m.dp_read);
        mbar_arrive(&m.p_full);
      }
      // dS = P (dP - delta)
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        const float4 nd = *reinterpret_cast<const float4*>(stat + kTile + c);
#pragma unroll
        for (int e = c; e < c + 4; e += 2) {
          uint64_t p = pack_f2(__uint_as_float(v[e]), __uint_as_float(v[e + 1]));
          if constexpr (!BF16) p = mul_f2(p, gain2);
          const uint64_t x = mul_f2(p, add_f2(pack_f2(__uint_as_float(d[e]), __uint_as_float(d[e + 1])),
                                              e == c ? pack_f2(nd.x, nd.y) : pack_f2(nd.z, nd.w)));
          float x0, x1;
          unpack_f2(x, x0, x1);
          w[e / 2] = Cvt<T>::pack2(x0, x1);
        }
      }
      if (bad != 0u) clear_pairs(w, bad);  // 0 * inf
      if (i > 0 && !(ok = mbar_wait(&m.dk_done, ph ^ 1, abort_flag, a.status, 19))) break;  // the last dS is read
      tc_fence_after();
      tmem_st16(ds_addr, w);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&m.stat_empty[s]);
        mbar_arrive(&m.ds_full);
      }
    }
    // column groups 0 and 1 store the halves of dV, 2 and 3 those of dK
    const bool is_dk = cg >= 2;
    const Rows& out = is_dk ? a.dk : a.dv;
    char* orow = key < a.tk ? out.row(bhk, key) : nullptr;
    if (n == 0) {
      if (orow != nullptr && (cg & 1) == 0) store_zero_row<T>(orow, a.dim);
    } else {
      ok = ok && mbar_wait(&m.all_done, 0, abort_flag, a.status, 16);
      tc_fence_after();
      if (ok && !*abort_flag) {
        const float p_mul = BF16 ? 1.f : 1.f / (1 << kShiftP16);
        const float mul = is_dk ? a.scale * p_mul / gain : p_mul;
        const int from = (cg & 1) * 32 * HALVES;
        store_row<T>(tmem + lanes + (is_dk ? kColDK : kColDV), orow, from, from + 32 * HALVES, a.dim, mul, key >= len);
      }
    }
  }
}

// ------------------------------------------------------------ dQ
template <bool BF16, int HALVES>
__device__ __forceinline__ void dq_cta(const CUtensorMap* q_map, const CUtensorMap* k_map, const CUtensorMap* v_map,
                                       const CUtensorMap* do_map, const GradArgs& a, char* smem, Misc& m,
                                       uint32_t tmem) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  using L = Smem<HALVES>;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int id = blockIdx.x - a.n_dkv;
  const int bh = id / a.q_tiles;
  const int qt = a.q_tiles - 1 - (id - bh * a.q_tiles);  // causal: the longest first
  const int b = bh / a.heads;
  const int h = bh - b * a.heads;
  const int hk = h / a.group;
  const int q0 = qt * kTile;
  const int len = key_count(a, b);
  const int off = a.tk - a.tq;
  const int keys = a.causal ? min(len, min(q0 + kTile, a.tq) + off) : len;  // keys any of the rows sees
  const int n = keys > 0 ? (keys + kTile - 1) / kTile : 0;
  volatile int* abort_flag = &m.abort_flag;

  if (warp == 0) {
    if (lane == 0 && n > 0 && !*abort_flag) {
      mbar_expect_tx(&m.own_full, L::tile);
      load_tile<HALVES>(smem + L::own, do_map, &m.own_full, q0, h, b);
      int na = 0, nb = 0;
      for (int i = 0; i < n; ++i) {
        const int sa = i % kStagesA, sb = i % kStagesDq;
        if (!mbar_wait(&m.a_empty[sa], ((i / kStagesA) & 1) ^ 1, abort_flag, a.status, 1)) break;
        mbar_expect_tx(&m.a_full[sa], L::tile);
        load_tile<HALVES>(smem + L::a + sa * L::tile, k_map, &m.a_full[sa], i * kTile, hk, b);
        na = i + 1;
        if (!mbar_wait(&m.b_empty[sb], ((i / kStagesDq) & 1) ^ 1, abort_flag, a.status, 2)) break;
        mbar_expect_tx(&m.b_full[sb], L::tile);
        load_tile<HALVES>(smem + L::b_dq + sb * L::tile, v_map, &m.b_full[sb], i * kTile, hk, b);
        nb = i + 1;
      }
      if (*abort_flag) {
        drain_loads(m.a_full, kStagesA, na, &m.own_full, a.status);
        drain_loads(m.b_full, kStagesDq, nb, nullptr, a.status);
      }
    }
  } else if (warp == 1) {
    if (n > 0 && elect_one()) {
      const uint32_t base = smem_u32(smem);
      const uint64_t do_rows = rows_desc(base + L::own);
      const uint64_t k_rows = rows_desc(base + L::a), k_cols = cols_desc(base + L::a);
      const uint64_t v_rows = rows_desc(base + L::b_dq);
      constexpr uint32_t step = L::tile >> 4;
      bool ok = mbar_wait(&m.own_full, 0, abort_flag, a.status, 3) && mbar_wait(&m.own_tmem, 0, abort_flag, a.status, 4);
      tc_fence_after();
      // Order S(i+1), dQ(i), dP(i+1): S runs ahead of the exponentials of the
      // tile before, dP under those of its own.
      for (int i = -1; ok && i < n; ++i) {
        const int sa = i < 0 ? 0 : i % kStagesA;
        const int ta = (i + 1) % kStagesA, tb = (i + 1) % kStagesDq;
        const uint32_t ph = i & 1, ta_ph = ((i + 1) / kStagesA) & 1, tb_ph = ((i + 1) / kStagesDq) & 1;
        const bool more = i + 1 < n;
        if (more) {  // the elementwise warps hold S(i)
          ok = mbar_wait(&m.a_full[ta], ta_ph, abort_flag, a.status, 7) &&
               (i < 0 || mbar_wait(&m.s_read, ph, abort_flag, a.status, 8));
          if (!ok) break;
          tc_fence_after();
          product_rows_ts<BF16, HALVES>(tmem + kColS, tmem + kColQ, k_rows + ta * step);
          mma_commit(&m.s_full);
        }
        if (i >= 0) {
          if (!(ok = mbar_wait(&m.ds_full, ph, abort_flag, a.status, 9))) break;
          tc_fence_after();
          product_cols<BF16, HALVES>(tmem + kColDQ, tmem + kColDSq, k_cols + sa * step, i > 0);
          mma_commit(&m.a_empty[sa]);
        }
        if (more) {  // and dP(i) (ds_full says so)
          if (!(ok = mbar_wait(&m.b_full[tb], tb_ph, abort_flag, a.status, 10))) break;
          tc_fence_after();
          product_rows<BF16, HALVES>(tmem + kColDP, do_rows, v_rows + tb * step);
          mma_commit(&m.dp_full);
          mma_commit(&m.b_empty[tb]);
        }
      }
      mma_commit(&m.all_done);
      int no_abort = 0;
      mbar_wait(&m.all_done, 0, &no_abort, a.status, 12);
    }
  } else {
    const int cg = (warp - 2) >> 2;  // column group: keys cg*32 .. +31 of a tile
    const int sub = warp & 3;
    const int row = sub * 32 + lane;
    const int query = q0 + row;
    const uint32_t lanes = static_cast<uint32_t>(sub * 32) << 16;
    const uint32_t s_addr = tmem + lanes + kColS + cg * 32;
    const uint32_t dp_addr = tmem + lanes + kColDP + cg * 32;
    const uint32_t ds_addr = tmem + lanes + kColDSq + cg * 16;
    if (n > 0) {
      row_to_tmem<HALVES>(tmem + lanes + kColQ, query < a.tq ? a.q.row(bh, query) : nullptr, cg, a.dim);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.own_tmem);
    }
    const float* stat = a.stat + (int64_t(bh) * a.q_tiles + qt) * (2 * kTile) + row;
    const float nl = stat[0], nd = stat[kTile];
    float gain = 1.f;
    if constexpr (!BF16) gain = ds_gain(a, b * a.kv_heads + hk);
    const uint64_t scale2 = pack_f2(a.scale_log2, a.scale_log2);
    const uint64_t nl2 = pack_f2(nl, nl), nd2 = pack_f2(nd, nd), gain2 = pack_f2(gain, gain);
    const int seen = a.causal ? min(len, query + off + 1) : len;  // keys this row sees
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const uint32_t ph = i & 1;
      const int lim = seen - i * kTile - cg * 32;  // columns from `lim` on are masked
      const uint32_t bad = lim >= 32 ? 0u : lim <= 0 ? ~0u : ~0u << lim;
      if (!(ok = mbar_wait(&m.s_full, ph, abort_flag, a.status, 14))) break;
      tc_fence_after();
      uint32_t v[32], w[16];
      tmem_ld32(s_addr, v);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.s_read);
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        exp2_pair(fma_f2(pack_f2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), scale2, nl2), v[c], v[c + 1]);
      }
      // a partly valid last key tile: rows past the keys may hold anything,
      // and dS's zeros times inf or NaN would reach dQ
      const int k0 = i * kTile;
      if (len < min(k0 + kTile, a.tk)) {
        const int tid = threadIdx.x - 64;
        const int from = len - k0, rows = min(kTile, a.tk - k0) - from;
        char* tile = smem + L::a + (i % kStagesA) * L::tile;
        for (int x = tid; x < rows * 8 * HALVES; x += 32 * kElemWarps) {
          const int r = from + x / (8 * HALVES), ch = x % (8 * HALVES);
          *reinterpret_cast<uint4*>(tile + (ch >> 3) * kHalfBytes + r * 128 + (ch & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
      }
      if (!(ok = mbar_wait(&m.dp_full, ph, abort_flag, a.status, 15))) break;
      tc_fence_after();
      uint32_t d[32];
      tmem_ld32(dp_addr, d);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        uint64_t p = pack_f2(__uint_as_float(v[c]), __uint_as_float(v[c + 1]));
        if constexpr (!BF16) p = mul_f2(p, gain2);
        float x0, x1;
        unpack_f2(mul_f2(p, add_f2(pack_f2(__uint_as_float(d[c]), __uint_as_float(d[c + 1])), nd2)), x0, x1);
        w[c / 2] = Cvt<T>::pack2(x0, x1);
      }
      if (bad != 0u) clear_pairs(w, bad);
      // dP(i) was issued after dQ(i-1), so dS's columns are free
      tmem_st16(ds_addr, w);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.ds_full);
    }
    char* orow = query < a.tq ? a.dq.row(bh, query) : nullptr;
    if (n == 0) {
      if (cg == 0 && orow != nullptr) store_zero_row<T>(orow, a.dim);
    } else if (cg < 2) {
      ok = ok && mbar_wait(&m.all_done, 0, abort_flag, a.status, 16);
      tc_fence_after();
      if (ok && !*abort_flag) {
        const float mul = BF16 ? a.scale : a.scale / (gain * (1 << kShiftP16));
        store_row<T>(tmem + lanes + kColDQ, orow, cg * 32 * HALVES, (cg + 1) * 32 * HALVES, a.dim, mul, seen <= 0);
      }
    }
  }
}

template <bool BF16, int HALVES>
__global__ void __launch_bounds__(kThreads, 1)
attn_grad_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                 const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap do_map,
                 const __grid_constant__ GradArgs a) {
  extern __shared__ __align__(1024) char smem[];
  Misc& m = *reinterpret_cast<Misc*>(smem + Smem<HALVES>::misc);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    m.abort_flag = 0;
    if ((smem_u32(smem) & 1023u) != 0) {
      m.abort_flag = 1;
      atomicCAS(a.status, 0, 0x300);
    }
    mbar_init(&m.own_full, 1);
    for (int s = 0; s < kStagesA; ++s) {
      mbar_init(&m.a_full[s], 1);
      mbar_init(&m.a_empty[s], 1);
    }
    for (int s = 0; s < kMaxB; ++s) {
      mbar_init(&m.b_full[s], 1);
      mbar_init(&m.b_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&m.stat_full[s], 1);
      mbar_init(&m.stat_empty[s], kElemWarps);
    }
    mbar_init(&m.s_full, 1);
    mbar_init(&m.s_read, kElemWarps);
    mbar_init(&m.p_full, kElemWarps);
    mbar_init(&m.dp_full, 1);
    mbar_init(&m.ds_full, kElemWarps);
    mbar_init(&m.dp_read, kElemWarps);
    mbar_init(&m.dk_done, 1);
    mbar_init(&m.own_tmem, kElemWarps);
    mbar_init(&m.all_done, 1);
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  grid_dep_wait();  // the statistics come from the kernel before
  if (warp == 1) tmem_alloc<512>(&m.tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = m.tmem;
  if (static_cast<int>(blockIdx.x) < a.n_dkv)
    dkv_cta<BF16, HALVES>(&q_map, &k_map, &v_map, &do_map, a, smem, m, tmem);
  else
    dq_cta<BF16, HALVES>(&q_map, &k_map, &v_map, &do_map, a, smem, m, tmem);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<512>(tmem);
  }
}

// ------------------------------------------------------------ row statistics
struct StatArgs {
  Rows out, dout, v;
  const float* lse;
  float* stat;
  uint32_t* maxima;
  const int32_t* key_lengths;
  int heads, kv_heads, group;
  int tq, tk, dim;
  int q_tiles;
  int q_blocks;  // blocks of the query part; the rest walks V (FP16)
};

constexpr int kStatRows = 64;  // rows of a block: 16 groups of 16 lanes, 4 rows each

// -lse*log2e and -delta of every query row, padded to whole tiles with rows
// that give P = 0.  FP16: also the largest squared norms of dO rows and valid
// V rows per key/value head (atomicMax of non-negative float bits: the order
// does not matter).
template <typename T>
__global__ void __launch_bounds__(256) attn_grad_stat_kernel(const __grid_constant__ StatArgs a) {
  constexpr bool kF16 = std::is_same<T, __half>::value;
  const int g = threadIdx.x >> 4;
  const int l = threadIdx.x & 15;
  const bool active = 8 * l < a.dim;
  if (static_cast<int>(blockIdx.x) < a.q_blocks) {
    const int blocks_per_head = a.q_tiles * (kTile / kStatRows);
    const int bh = blockIdx.x / blocks_per_head;
    const int r0 = (blockIdx.x - bh * blocks_per_head) * kStatRows;
    float most = 0.f;
    uint4 o[4], d[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = r0 + u * 16 + g;
      o[u] = d[u] = make_uint4(0u, 0u, 0u, 0u);
      if (active && r < a.tq) {
        o[u] = reinterpret_cast<const uint4*>(a.out.row(bh, r))[l];
        d[u] = reinterpret_cast<const uint4*>(a.dout.row(bh, r))[l];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = r0 + u * 16 + g;
      const uint32_t ow[4] = {o[u].x, o[u].y, o[u].z, o[u].w}, dw[4] = {d[u].x, d[u].y, d[u].z, d[u].w};
      float sum = 0.f, norm = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float o0, o1, d0, d1;
        Cvt<T>::unpack2(ow[i], o0, o1);
        Cvt<T>::unpack2(dw[i], d0, d1);
        sum = fmaf(o0, d0, sum);
        sum = fmaf(o1, d1, sum);
        if constexpr (kF16) norm = fmaf(d0, d0, fmaf(d1, d1, norm));
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, w);
        if constexpr (kF16) norm += __shfl_xor_sync(0xffffffffu, norm, w);
      }
      most = fmaxf(most, norm);
      if (l == 0) {
        const float lse = r < a.tq ? a.lse[int64_t(bh) * a.tq + r] : -INFINITY;
        float* dst = a.stat + (int64_t(bh) * a.q_tiles + r / kTile) * (2 * kTile) + r % kTile;
        dst[0] = lse == -INFINITY ? -INFINITY : -lse * kLog2e + (kF16 ? static_cast<float>(kShiftP16) : 0.f);
        dst[kTile] = -sum;
      }
    }
    if constexpr (kF16) {
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
      if ((threadIdx.x & 31) == 0) {
        const int b = bh / a.heads;
        atomicMax(a.maxima + 2 * (b * a.kv_heads + (bh - b * a.heads) / a.group), __float_as_uint(most));
      }
    }
  } else if constexpr (kF16) {
    const int id = blockIdx.x - a.q_blocks;
    const int blocks_per_head = (a.tk + kStatRows - 1) / kStatRows;
    const int bhk = id / blocks_per_head;
    const int r0 = (id - bhk * blocks_per_head) * kStatRows;
    const int b = bhk / a.kv_heads;
    const int len = a.key_lengths != nullptr ? min(a.key_lengths[b], a.tk) : a.tk;
    float most = 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = r0 + u * 16 + g;
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (active && r < len) x = reinterpret_cast<const uint4*>(a.v.row(bhk, r))[l];
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      float norm = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v0, v1;
        Cvt<T>::unpack2(w[i], v0, v1);
        norm = fmaf(v0, v0, fmaf(v1, v1, norm));
      }
#pragma unroll
      for (int s = 8; s > 0; s >>= 1) norm += __shfl_xor_sync(0xffffffffu, norm, s);
      most = fmaxf(most, norm);
    }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
    if ((threadIdx.x & 31) == 0) atomicMax(a.maxima + 2 * bhk + 1, __float_as_uint(most));
  }
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

template <bool BF16, int HALVES>
cudaError_t launch_grad(unsigned blocks, const CUtensorMap* maps, const GradArgs& a, cudaStream_t st) {
  const auto kernel = attn_grad_kernel<BF16, HALVES>;
  const int smem = static_cast<int>(Smem<HALVES>::total);
  const cudaError_t err = ensure_smem(reinterpret_cast<const void*>(kernel), smem);
  if (err != cudaSuccess) return err;
  return launch_pdl(kernel, dim3(blocks), dim3(kThreads), size_t(smem), st, maps[0], maps[1], maps[2], maps[3], a);
}

}  // namespace

int64_t attn_grad_workspace_bytes(int batch, int heads, int kv_heads, int tq) {
  const int64_t q_tiles = (int64_t(tq) + kTile - 1) / kTile;
  return static_cast<int64_t>(align256(size_t(batch) * heads * q_tiles * 2 * kTile * 4) +
                              align256(size_t(batch) * kv_heads * 2 * 4));
}

cudaError_t launch_attn_grad(const AttnGradCall& c, int* status, cudaStream_t st) {
  const b2_view &q = *c.q, &k = *c.k;
  CUtensorMap maps[4];
  const b2_view* views[4] = {c.q, c.k, c.v, c.dout};
  for (int i = 0; i < 4; ++i)
    if (!linear_rows_map(&maps[i], *views[i], kTile)) return cudaErrorInvalidValue;
  const bool bf16 = q.dtype == B2_BF16;
  StatArgs s{};
  s.out = make_rows(*c.out), s.dout = make_rows(*c.dout), s.v = make_rows(*c.v);
  s.lse = c.lse;
  s.key_lengths = c.key_lengths;
  s.heads = q.heads, s.kv_heads = k.heads, s.group = q.heads / k.heads;
  s.tq = q.tokens, s.tk = k.tokens, s.dim = q.head_dim;
  s.q_tiles = (q.tokens + kTile - 1) / kTile;
  s.stat = static_cast<float*>(c.workspace);
  const int64_t bh = int64_t(q.batch) * q.heads, bhk = int64_t(q.batch) * k.heads;
  s.maxima = reinterpret_cast<uint32_t*>(static_cast<char*>(c.workspace) +
                                         align256(size_t(bh) * s.q_tiles * 2 * kTile * 4));
  s.q_blocks = static_cast<int>(bh * s.q_tiles * (kTile / kStatRows));
  const int v_blocks = bf16 ? 0 : static_cast<int>(bhk * ((k.tokens + kStatRows - 1) / kStatRows));
  cudaError_t err;
  if (!bf16 && (err = cudaMemsetAsync(s.maxima, 0, size_t(bhk) * 8, st)) != cudaSuccess) return err;
  if (bf16) attn_grad_stat_kernel<__nv_bfloat16><<<s.q_blocks, 256, 0, st>>>(s);
  else attn_grad_stat_kernel<__half><<<s.q_blocks + v_blocks, 256, 0, st>>>(s);
  if ((err = cudaGetLastError()) != cudaSuccess) return err;
  GradArgs a{};
  a.q = make_rows(q), a.dq = make_rows(*c.dq), a.dk = make_rows(*c.dk), a.dv = make_rows(*c.dv);
  a.stat = s.stat;
  a.maxima = s.maxima;
  a.key_lengths = c.key_lengths;
  a.heads = s.heads, a.kv_heads = s.kv_heads, a.group = s.group;
  a.tq = s.tq, a.tk = s.tk, a.dim = s.dim;
  a.q_tiles = s.q_tiles;
  a.k_tiles = (k.tokens + kTile - 1) / kTile;
  a.n_dkv = static_cast<int>(bhk * a.k_tiles);
  a.causal = c.causal;
  a.scale = c.scale;
  a.scale_log2 = c.scale * kLog2e;
  a.status = status;
  const unsigned blocks = static_cast<unsigned>(a.n_dkv + bh * a.q_tiles);
  if (q.head_dim <= 64) return bf16 ? launch_grad<true, 1>(blocks, maps, a, st) : launch_grad<false, 1>(blocks, maps, a, st);
  return bf16 ? launch_grad<true, 2>(blocks, maps, a, st) : launch_grad<false, 2>(blocks, maps, a, st);
}

}  // namespace b2
