// Exact attention, forward, with shared key/value heads, per-batch key counts
// and a causal mask: out = softmax(scale q k^T) v and lse, one pass over the
// keys with the running maximum and sum, on tcgen05 with TMA-staged tiles.
//
// An item is 128 query rows of one head and walks its 64-key tiles:
//   S = Q K^T in tensor memory (two buffers), P = exp(scale S - max) rounded to
//   the type of v and written back over S, O += P V, O /= sum at the end.
// O is rescaled only when a row's maximum has grown by 2^8 (P stays below
// that).  The sum is of P before its rounding.  FP16 P is held times 2^8, as in
// the backward pass: without, keys below 2^-25 of the largest would leave P V
// and stay in the sum (65535 at 2^-25.5: 1.4e-3 of the row, all of it lost).  O
// is then rescaled from 2^7 on, and P stays below 2^15.
//
// Persistent CTAs, two per SM (112 KB of shared memory, 256 TMEM columns
// each), step through the items by the grid's size: barriers, rings and tensor
// memory are set up once, and the next item's Q and first tiles load and its
// first S runs while this one's last tiles and results are under way.  With a
// CTA for each item, set-up, first loads and cold code took 6.3 us of it,
// against 1.2 us for each tile.  Causal items run longest first; the
// others head by head, so that the heads in flight share K and V in L2.
//
// What bounds it: the softmax chain of a tile (load S, maximum, exponentials,
// store P), which two CTAs overlap; tensor and exponential pipes are each half
// used.  2 x 16 x 9216^2 x 128: 1.18 ms, 1177 TFLOP/s (a CTA an item: 1.455;
// FP16 1.22); 64 heads of 9216 queries and 512 keys: 192 us (249).  Three CTAs per SM with
// one S buffer and half a row's logits in registers, for D <= 64: 211 us
// against 133 (16 x 4096^2 x 64).
#include <cudaTypedefs.h>

#include <type_traits>

#include "kernels.h"
#include "umma.cuh"

namespace b2 {

namespace {

using namespace umma;

constexpr int kRows = 128;  // query rows of an item
constexpr int kKeys = 64;   // keys of a tile
constexpr int kStagesK = 2, kStagesV = 3;  // P V of a tile needs V one tile later than S needs K
constexpr int kVWarp = 6;   // warp 0: Q and K, warp 1: MMA and TMEM, warps 2-5: softmax, warp 6: V
constexpr int kThreads = 32 * (kVWarp + 1);
constexpr uint32_t kTmem = 256, kO = 0, kS = 128;  // columns: O, and S by kKeys
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kShiftP16 = 8.f;  // FP16 v: P is held times 2^8

struct ForwardArgs {
  Rows o, o_low;  // o_low: what o's type cannot hold, or no base
  float* lse;
  const float* qk_scale;  // FP16 q, k held times these, whatever the type of v; or NULL
  const int32_t* key_lengths;
  int heads, group, bh;  // query heads, of each key/value head, batches * heads
  int tq, tk, off;       // causal: query i sees keys up to i + off
  int q_tiles, n_items;
  int causal;
  float scale_log2;
  int* status;
};

struct __align__(8) Misc {
  uint64_t q_full, q_empty;
  uint64_t k_full[kStagesK], k_empty[kStagesK];
  uint64_t v_full[kStagesV], v_empty[kStagesV];
  uint64_t s_full[2], p_full[2], pv_done[2];  // by S buffer
  uint64_t acc_free;                          // an item's O has been read
  uint64_t exit_done;
  uint32_t tmem;
  int abort_flag;
};

template <int HALVES>
struct Smem {
  static constexpr uint32_t tile = HALVES * kKeys * 128;
  static constexpr uint32_t q = 0;  // [halves][128 rows][128 B]
  static constexpr uint32_t k = q + HALVES * kRows * 128;
  static constexpr uint32_t v = k + kStagesK * tile;
  static constexpr uint32_t misc = v + kStagesV * tile;
  static constexpr uint32_t used = misc + sizeof(Misc);
  static constexpr uint32_t least = 80 * 1024;  // no more CTAs to an SM than its TMEM columns serve
  static constexpr uint32_t total = used < least ? least : used;
};
static_assert(2 * (Smem<2>::total + 1024) <= 233472, "two CTAs per SM");

struct Item {
  int bh, b, r0;
  int len;  // keys of the batch
  int n;    // key tiles that any of the rows sees
};

__device__ __forceinline__ Item decode(const ForwardArgs& a, int id) {
  Item w;
  int qt;
  if (a.causal) {
    const int t = id / a.bh;
    w.bh = id - t * a.bh;
    qt = a.q_tiles - 1 - t;
  } else {
    w.bh = id / a.q_tiles;
    qt = id - w.bh * a.q_tiles;
  }
  w.r0 = qt * kRows;
  w.b = w.bh / a.heads;
  w.len = a.key_lengths != nullptr ? min(max(__ldg(a.key_lengths + w.b), 0), a.tk) : a.tk;
  const int keys = a.causal ? min(w.len, min(w.r0 + kRows, a.tq) + a.off) : w.len;
  w.n = keys > 0 ? (keys + kKeys - 1) / kKeys : 0;
  return w;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// (lo, hi) = (x0, x1) * (s, s) + (t, t) with one packed FMA
__device__ __forceinline__ void fma2(float& lo, float& hi, float x0, float x1, float s, float t) {
  uint64_t x, sv, tv, d;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(x) : "f"(x0), "f"(x1));
  asm("mov.b64 %0, {%1, %1};\n" : "=l"(sv) : "f"(s));
  asm("mov.b64 %0, {%1, %1};\n" : "=l"(tv) : "f"(t));
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(x), "l"(sv), "l"(tv));
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(lo), "=f"(hi) : "l"(d));
}

// (a0, a1) += (b0, b1) with one packed add
__device__ __forceinline__ void add2(float& a0, float& a1, float b0, float b1) {
  uint64_t x, y, d;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(x) : "f"(a0), "f"(a1));
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(y) : "f"(b0), "f"(b1));
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(x), "l"(y));
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a0), "=f"(a1) : "l"(d));
}

// ------------------------------------------------------------ TMA producers
template <int HALVES>
__device__ void produce_qk(const CUtensorMap* q_map, const CUtensorMap* k_map, const ForwardArgs& a, char* smem, Misc& m) {
  using L = Smem<HALVES>;
  volatile int* abort_flag = &m.abort_flag;
  int owns = 0, t = 0;
  bool ok = !*abort_flag;
  for (int id = blockIdx.x; ok && id < a.n_items; id += gridDim.x) {
    const Item w = decode(a, id);
    if (w.n == 0) continue;
    const int h = w.bh - w.b * a.heads;
    if (!(ok = mbar_wait(&m.q_empty, (owns & 1) ^ 1, abort_flag, a.status, 1))) break;
    mbar_expect_tx(&m.q_full, HALVES * kRows * 128);
    for (int dh = 0; dh < HALVES; ++dh)
      tma_load_4d(smem + L::q + dh * kRows * 128, q_map, &m.q_full, dh * 64, w.r0, h, w.b);
    ++owns;
    for (int j = 0; j < w.n; ++j, ++t) {
      const int s = t % kStagesK;
      if (!(ok = mbar_wait(&m.k_empty[s], ((t / kStagesK) & 1) ^ 1, abort_flag, a.status, 2))) break;
      mbar_expect_tx(&m.k_full[s], L::tile);
      for (int dh = 0; dh < HALVES; ++dh)
        tma_load_4d(smem + L::k + s * L::tile + dh * kKeys * 128, k_map, &m.k_full[s], dh * 64, j * kKeys, h / a.group, w.b);
    }
  }
  if (*abort_flag) {
    int no_abort = 0;
    drain_loads(m.k_full, kStagesK, t, nullptr, a.status);
    if (owns > 0) mbar_wait(&m.q_full, (owns - 1) & 1, &no_abort, a.status, 31);
  }
}

template <int HALVES>
__device__ void produce_v(const CUtensorMap* v_map, const ForwardArgs& a, char* smem, Misc& m) {
  using L = Smem<HALVES>;
  volatile int* abort_flag = &m.abort_flag;
  int t = 0;
  bool ok = !*abort_flag;
  for (int id = blockIdx.x; ok && id < a.n_items; id += gridDim.x) {
    const Item w = decode(a, id);
    const int hk = (w.bh - w.b * a.heads) / a.group;
    for (int j = 0; j < w.n; ++j, ++t) {
      const int s = t % kStagesV;
      if (!(ok = mbar_wait(&m.v_empty[s], ((t / kStagesV) & 1) ^ 1, abort_flag, a.status, 3))) break;
      mbar_expect_tx(&m.v_full[s], L::tile);
      for (int dh = 0; dh < HALVES; ++dh)
        tma_load_4d(smem + L::v + s * L::tile + dh * kKeys * 128, v_map, &m.v_full[s], dh * 64, j * kKeys, hk, w.b);
    }
  }
  if (*abort_flag) drain_loads(m.v_full, kStagesV, t, nullptr, a.status);
}

// ------------------------------------------------------------ MMA issuer
// A place in the sequence of all tiles of the CTA's items.
struct Cursor {
  int id, n, j;  // the item, its tiles and the tile in it
  int own;       // items with tiles before it
  uint32_t g;    // tiles before it
  __device__ __forceinline__ void seek(const ForwardArgs& a) {
    while (id < a.n_items && (n = decode(a, id).n) == 0) id += gridDim.x;
  }
  __device__ __forceinline__ void next(const ForwardArgs& a) {
    ++g;
    if (++j < n) return;
    j = 0;
    ++own;
    id += gridDim.x;
    seek(a);
  }
};

// S runs up to two tiles, and into the next item, ahead of P V; whichever can
// go out does, S first.  STEPS: the 16-column steps of the head dimension that
// products cover, all that it has (what pads it is zeros).
template <bool BF16, bool QBF16, int HALVES, int STEPS>
__device__ void issue(const ForwardArgs& a, char* smem, Misc& m, uint32_t tmem) {
  using L = Smem<HALVES>;
  constexpr uint32_t idesc_s = idesc_f16(128, kKeys, QBF16, false, false);
  constexpr uint32_t idesc_o = idesc_f16(128, 16 * STEPS, BF16, false, true);
  volatile int* abort_flag = &m.abort_flag;
  const uint64_t q_desc = smem_desc_sw128(smem_u32(smem + L::q), 16, 1024);
  const uint64_t k_desc = smem_desc_sw128(smem_u32(smem + L::k), 16, 1024);
  const uint64_t v_desc = smem_desc_sw128(smem_u32(smem + L::v), kKeys * 128, 1024);
  Cursor s{static_cast<int>(blockIdx.x), 0, 0, 0, 0u};
  s.seek(a);
  Cursor p = s;
  long long idle = 0;
  while (p.id < a.n_items && !*abort_flag) {
    const int sk = s.g % kStagesK, pv = p.g % kStagesV;
    // S(g) takes the buffer of P(g - 2)
    if (s.id < a.n_items &&
        (s.g < 2 || (s.g - 2 < p.g && mbar_test_wait(&m.pv_done[s.g & 1], ((s.g - 2) >> 1) & 1))) &&
        (s.j > 0 || mbar_test_wait(&m.q_full, s.own & 1)) && mbar_test_wait(&m.k_full[sk], (s.g / kStagesK) & 1)) {
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < STEPS; ++kk)
        mma_ss(tmem + kS + kKeys * (s.g & 1), q_desc + (((kk >> 2) * kRows * 128 + (kk & 3) * 32) >> 4),
               k_desc + ((sk * L::tile + (kk >> 2) * kKeys * 128 + (kk & 3) * 32) >> 4), idesc_s, kk > 0 ? 1u : 0u);
      mma_commit(&m.s_full[s.g & 1]);
      mma_commit(&m.k_empty[sk]);
      if (s.j == s.n - 1) mma_commit(&m.q_empty);
      s.next(a);
      idle = 0;
    } else if (p.g < s.g && mbar_test_wait(&m.p_full[p.g & 1], (p.g >> 1) & 1) &&
               mbar_test_wait(&m.v_full[pv], (p.g / kStagesV) & 1) &&
               (p.j > 0 || p.own == 0 || mbar_test_wait(&m.acc_free, (p.own - 1) & 1))) {
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        mma_ts(tmem + kO, tmem + kS + kKeys * (p.g & 1) + kk * 8, v_desc + ((pv * L::tile + kk * 2048) >> 4), idesc_o,
               p.j > 0 || kk > 0 ? 1u : 0u);
      mma_commit(&m.pv_done[p.g & 1]);
      mma_commit(&m.v_empty[pv]);
      p.next(a);
      idle = 0;
    } else {
      const long long now = clock64();
      if (idle == 0) idle = now;
      if (now - idle > (1ll << 32)) {
        *abort_flag = 1;
        atomicCAS(a.status, kStatusOk, (kStatusTimeout << 8) | 23);
      }
    }
  }
  // every product completes before TMEM is released (bounded by time only,
  // even after an abort)
  mma_commit(&m.exit_done);
  int no_abort = 0;
  mbar_wait(&m.exit_done, 0, &no_abort, a.status, 7);
}

// ------------------------------------------------------------ softmax
// Rows r0.. of a warp's 32, whose batch has no keys or that see none.
__device__ __forceinline__ void store_zeros(const Rows& o, int bh, int r0, int tq, int lane) {
  const int chunks = o.dim >> 3;
  char* base = o.row(bh, r0);
  for (int x = lane; x < 32 * chunks; x += 32) {
    const int r = x / chunks, c = x - r * chunks;
    if (r0 + r < tq) *reinterpret_cast<uint4*>(base + r * o.st * 2 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
}

template <bool BF16, bool QK16, int HALVES>
__device__ void softmax(const ForwardArgs& a, char* smem, Misc& m, uint32_t tmem) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  using L = Smem<HALVES>;
  constexpr float kGrowth = BF16 ? 8.f : 7.f;
  volatile int* abort_flag = &m.abort_flag;
  const int lane = threadIdx.x & 31;
  const int sub = (threadIdx.x >> 5) & 3;  // TMEM sub-partition of this warp
  const int row = sub * 32 + lane;
  const uint32_t base = tmem + (static_cast<uint32_t>(sub * 32) << 16);
  float scale_log2 = a.scale_log2;
  if constexpr (QK16) scale_log2 /= a.qk_scale[0] * a.qk_scale[1];
  uint32_t g = 0;
  for (int id = blockIdx.x; id < a.n_items; id += gridDim.x) {
    const Item w = decode(a, id);
    const int r = w.r0 + row;
    const bool low = a.o_low.base != nullptr && r < low_rows(w.len, a.tq, a.causal, a.off);
    if (w.n == 0) {  // no row sees a key, so all of them have a low part
      store_zeros(a.o, w.bh, w.r0 + sub * 32, a.tq, lane);
      if (a.o_low.base != nullptr) store_zeros(a.o_low, w.bh, w.r0 + sub * 32, a.tq, lane);
      if (r < a.tq && a.lse != nullptr) a.lse[int64_t(w.bh) * a.tq + r] = -INFINITY;
      continue;
    }
    const int last = r + a.off;  // causal: the last key the row sees
    float mrun = -INFINITY, lrun = 0.f;  // mrun: the maximum less P's shift
    for (int j = 0; j < w.n; ++j, ++g) {
      const uint32_t sb = g & 1;
      if (!mbar_wait(&m.s_full[sb], (g >> 1) & 1, abort_flag, a.status, 8)) return;
      tc_fence_after();
      const uint32_t s_addr = base + kS + kKeys * sb;
      uint32_t v[kKeys];
      tmem_ld32(s_addr, v);
      tmem_ld32(s_addr + 32, v + 32);
      tmem_wait_ld();
      // logits in the log2 domain, masked ones -inf; unmasked tiles keep raw S
      // and fold the scale into the argument of the exponential
      const int k0 = j * kKeys, klen = min(kKeys, w.len - k0);
      const bool plain = klen == kKeys && (!a.causal || last - k0 >= kKeys - 1);
      if (!plain) {
        uint64_t bad = klen < kKeys ? ~0ull << klen : 0ull;
        if (a.causal && last - k0 < kKeys - 1) bad |= last < k0 ? ~0ull : ~0ull << (last - k0 + 1);
#pragma unroll
        for (int c = 0; c < kKeys; ++c) {
          const uint32_t word = static_cast<uint32_t>(c < 32 ? bad : bad >> 32);
          const float x = __uint_as_float(v[c]) * scale_log2;
          v[c] = (word >> (c & 31)) & 1u ? __float_as_uint(-INFINITY) : __float_as_uint(x);
        }
      }
      const float mul = plain ? scale_log2 : 1.f;
      float m0 = fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1]));
      float m1 = fmaxf(__uint_as_float(v[2]), __uint_as_float(v[3]));
#pragma unroll
      for (int c = 4; c < kKeys; c += 4) {
        m0 = max3(m0, __uint_as_float(v[c]), __uint_as_float(v[c + 1]));
        m1 = max3(m1, __uint_as_float(v[c + 2]), __uint_as_float(v[c + 3]));
      }
      const float mx = BF16 ? fmaxf(m0, m1) * mul : fmaf(fmaxf(m0, m1), mul, -kShiftP16);
      float alpha = 1.f;
      bool rescale = false;
      const float mnew = fmaxf(mrun, mx);
      if (mrun == -INFINITY) {
        mrun = mnew;
      } else if (mnew > mrun + kGrowth) {
        alpha = ex2(mrun - mnew);
        mrun = mnew;
        rescale = true;
      }
      if (__any_sync(0xffffffffu, rescale)) {
        // once the P V before is done (the one before that was, ahead of S)
        if (j >= 1 && !mbar_wait(&m.pv_done[sb ^ 1], ((g - 1) >> 1) & 1, abort_flag, a.status, 9)) return;
        tc_fence_after();
#pragma unroll 1
        for (int c0 = 0; c0 < 64 * HALVES; c0 += 32) {
          uint32_t o[32];
          tmem_ld32(base + kO + c0, o);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
          tmem_st32(base + kO + c0, o);
        }
        tmem_wait_st();
      }
      // no maximum yet: masked keys (-inf) give 0, and NaN, which no maximum shows, stays
      const float neg = mrun == -INFINITY ? 0.f : -mrun;
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int c = 0; c < kKeys; c += 2) {
        float x0, x1;
        fma2(x0, x1, __uint_as_float(v[c]), __uint_as_float(v[c + 1]), mul, neg);
        const float p0 = ex2(x0);
        const float p1 = ex2(x1);
        add2(s0, s1, p0, p1);
        v[c / 2] = Cvt<T>::pack2(p0, p1);
      }
      lrun = lrun * alpha + (s0 + s1);
      tmem_st32(s_addr, v);
      tmem_wait_st();
      // V rows past the batch's keys may hold anything: P is 0 there, but
      // 0 * inf is not, so they are cleared in the tile first
      if (klen < min(kKeys, a.tk - k0)) {
        if (!mbar_wait(&m.v_full[g % kStagesV], (g / kStagesV) & 1, abort_flag, a.status, 25)) return;
        char* tile = smem + L::v + (g % kStagesV) * L::tile;
        const int rows = min(kKeys, a.tk - k0) - klen;
        for (int x = threadIdx.x - 64; x < rows * 8 * HALVES; x += 128) {
          const int rr = klen + x / (8 * HALVES), ch = x % (8 * HALVES);
          *reinterpret_cast<uint4*>(tile + (ch >> 3) * kKeys * 128 + rr * 128 + (ch & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&m.p_full[sb]);
    }
    if (!mbar_wait(&m.pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, abort_flag, a.status, 10)) return;
    tc_fence_after();
    const float inv = lrun > 0.f ? 1.f / lrun : 0.f;
    const float empty = a.causal && last < 0 ? 0.f : NAN;  // without a sum: no key seen, or -inf from all (0 / 0)
    const int q = lane & 3;
    char* quad_row = a.o.row(w.bh, r - q);
    char* low_row = low ? a.o_low.row(w.bh, r) : nullptr;
#pragma unroll 1
    for (int c0 = 0; c0 < 64 * HALVES; c0 += 32) {
      uint32_t o[32], x[16];
      tmem_ld32(base + kO + c0, o);
      tmem_wait_ld();
      // Four lanes store 64 bytes of a row together: by its own lane alone,
      // each row's 16 bytes touch a line of their own.
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        const float f0 = lrun == 0.f ? empty : __uint_as_float(o[c]) * inv;
        const float f1 = lrun == 0.f ? empty : __uint_as_float(o[c + 1]) * inv;
        x[c / 2] = Cvt<T>::pack2(f0, f1);
        if (low) {  // what the output's type cannot hold
          float h0, h1;
          Cvt<T>::unpack2(x[c / 2], h0, h1);
          o[c / 2] = Cvt<T>::pack2(f0 - h0, f1 - h1);
        }
      }
      if (low && r < a.tq) {
        uint4* dst = reinterpret_cast<uint4*>(low_row + c0 * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c0 + 8 * i < a.o.dim) dst[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      }
      transpose_quads(x, lane);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r - q + i < a.tq && c0 + 8 * q < a.o.dim)
          *reinterpret_cast<uint4*>(quad_row + i * a.o.st * 2 + (c0 + 8 * q) * 2) =
              make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&m.acc_free);
    if (r < a.tq && a.lse != nullptr) {
      const float none = lrun != 0.f ? lrun : -INFINITY;  // NaN rows stay NaN
      a.lse[int64_t(w.bh) * a.tq + r] = lrun > 0.f ? (mrun + __log2f(lrun)) * kLn2 : none;
    }
  }
}

template <bool BF16, bool QK16, int HALVES>
__global__ void __launch_bounds__(kThreads, 2)
attn_forward_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                    const __grid_constant__ CUtensorMap v_map, const __grid_constant__ ForwardArgs a) {
  extern __shared__ __align__(1024) char smem[];
  Misc& m = *reinterpret_cast<Misc*>(smem + Smem<HALVES>::misc);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    m.abort_flag = 0;
    if ((smem_u32(smem) & 1023u) != 0) {
      m.abort_flag = 1;
      atomicCAS(a.status, 0, 0x300);
    }
    mbar_init(&m.q_full, 1);
    mbar_init(&m.q_empty, 1);
    for (int s = 0; s < kStagesK; ++s) {
      mbar_init(&m.k_full[s], 1);
      mbar_init(&m.k_empty[s], 1);
    }
    for (int s = 0; s < kStagesV; ++s) {
      mbar_init(&m.v_full[s], 1);
      mbar_init(&m.v_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&m.s_full[b], 1);
      mbar_init(&m.p_full[b], 4);
      mbar_init(&m.pv_done[b], 1);
    }
    mbar_init(&m.acc_free, 4);
    mbar_init(&m.exit_done, 1);
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  grid_dep_wait();  // q, k and v may come from the kernel before
  if (warp == 1) tmem_alloc<kTmem>(&m.tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = m.tmem;
  if (warp == 0) {
    if ((threadIdx.x & 31) == 0) produce_qk<HALVES>(&q_map, &k_map, a, smem, m);
  } else if (warp == 1) {
    if (elect_one())
      with_steps<HALVES>(a.o.dim, [&](auto steps) { issue<BF16, BF16 && !QK16, HALVES, decltype(steps)::value>(a, smem, m, tmem); });
  } else if (warp == kVWarp) {
    if ((threadIdx.x & 31) == 0) produce_v<HALVES>(&v_map, a, smem, m);
  } else {
    softmax<BF16, QK16, HALVES>(a, smem, m, tmem);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<kTmem>(tmem);
  }
}

template <bool BF16, bool QK16, int HALVES>
cudaError_t launch(const CUtensorMap* maps, const ForwardArgs& a, cudaStream_t st) {
  const auto kernel = attn_forward_kernel<BF16, QK16, HALVES>;
  const int smem = static_cast<int>(Smem<HALVES>::total);
  const cudaError_t err = ensure_smem(reinterpret_cast<const void*>(kernel), smem);
  if (err != cudaSuccess) return err;
  const int most = 2 * sm_count();
  return launch_pdl(kernel, dim3(a.n_items < most ? a.n_items : most), dim3(kThreads), size_t(smem), st, maps[0], maps[1],
                    maps[2], a);
}

template <bool BF16, bool QK16>
cudaError_t launch_halves(int dim, const CUtensorMap* maps, const ForwardArgs& a, cudaStream_t st) {
  return dim <= 64 ? launch<BF16, QK16, 1>(maps, a, st) : launch<BF16, QK16, 2>(maps, a, st);
}

}  // namespace

cudaError_t launch_attn_forward(const AttnForwardCall& c, int* status, cudaStream_t st) {
  const b2_view &q = *c.q, &k = *c.k;
  CUtensorMap maps[3];
  if (!linear_rows_map(&maps[0], q, kRows) || !linear_rows_map(&maps[1], k, kKeys) || !linear_rows_map(&maps[2], *c.v, kKeys))
    return cudaErrorInvalidValue;
  ForwardArgs a{};
  a.o = make_rows(*c.out);
  if (c.out_low != nullptr) a.o_low = make_rows(*c.out_low);
  a.lse = c.lse;
  a.qk_scale = c.qk_scale;
  a.key_lengths = c.key_lengths;
  a.heads = q.heads;
  a.group = q.heads / k.heads;
  a.bh = q.batch * q.heads;
  a.tq = q.tokens;
  a.tk = k.tokens;
  a.off = k.tokens - q.tokens;
  a.q_tiles = (q.tokens + kRows - 1) / kRows;
  a.n_items = a.bh * a.q_tiles;
  a.causal = c.causal;
  a.scale_log2 = c.scale * kLog2e;
  a.status = status;
  if (c.v->dtype == B2_BF16)
    return c.qk_scale != nullptr ? launch_halves<true, true>(q.head_dim, maps, a, st)
                                 : launch_halves<true, false>(q.head_dim, maps, a, st);
  return c.qk_scale != nullptr ? launch_halves<false, true>(q.head_dim, maps, a, st)
                               : launch_halves<false, false>(q.head_dim, maps, a, st);
}

}  // namespace b2
