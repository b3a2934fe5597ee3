// Per-head RMS norm of queries and keys and rotary positions with several
// axes, in one pass over the rows, and the gradients of both.
//
//   z = x * rsqrt(mean(x^2) + eps) * w           (norm; z = x without it)
//   (y_a, y_b) = (z_a c - z_b s, z_a s + z_b c)  for every rotated pair (a, b)
//   c + i s = exp(2 pi i * pos[axis(p)] * turn[p])
//
// A pair's rate turn = theta^(-2j/d) / (2 pi) and its position are multiplied
// in FP64 and reduced to a fraction of a turn there, so positions of millions
// keep full FP32 accuracy of the angle (in FP32 the product would already be
// off by pos * 2^-24 rad); only the fraction goes to sincospif.
//
// Gradients (r = rsqrt(mean(x^2) + eps), xh = x r, g = dz w):
//   dz = rotation by the negative angle of dy
//   dx = r (g - xh mean(g xh)),  dw = sum over rows of dz xh
//
// What bounds it: HBM.  Forward reads and writes every row once; backward
// reads x and dy and writes dx.  r is recomputed from x, which is read anyway,
// so nothing but x is kept between the passes.
//
// Layout: a group of G lanes owns a row, each lane four pairs (G = 16 for
// D = 128), so a 16-bit row moves with one 16-byte access a lane (interleaved
// pairs) or two of 8 bytes (halves).  A block takes `tt` tokens; its 256
// threads compute the tokens' cos / sin once into shared memory (one
// sincospif per thread for 16 + 16 heads, D = 128) while the first rows are on
// their way; every group then walks heads of one token, query heads first,
// four rows in flight.  The backward pass, with two rows to read for one it
// writes, fetches them by asynchronous copies into slots that only their own
// thread reads: 142 us against 204 (9170 tokens of 56 + 56 heads x 128) for
// loads into registers.
// 9216 x (16 + 16) x 128, norm and rotation forward: 34 us (HBM alone: 23);
// 32760 x 40 x 128, rotation: 114 us (102.6).
#include <math.h>
#include <string.h>

#include <type_traits>

#include "kernels.h"

namespace b2 {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;     // D <= 256
constexpr int kMaxTokens = 16;     // tokens of a block
// Blocks of the forward pass: four on an SM, which stride over the tiles.
constexpr int kBlocks = 148 * 4;
// Blocks of one side in the backward pass (two sides fill the SMs with three
// blocks each), and so partial weight gradients.
constexpr int kGradBlocks = 222;

enum Layout { kInterleaved = 0, kHalves = 1, kScalar = 2 };

// Rows are read once: leave L1 alone.
__device__ __forceinline__ uint4 load16(const char* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 load8(const char* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

struct RowSet {
  char* base;
  int64_t sb, sh, st;  // strides in elements
};

struct Side {
  RowSet x, dy, y;  // y: output (forward) or dx (backward)
  const void* w;
  void* dw;
  int heads;
};

struct RotaryArgs {
  Side side[2];
  const void* pos;
  int64_t pb, pt, pa;
  int pos_dtype;
  int sides;
  int batch, tokens, dim;
  int rot_pairs;    // rotated pairs; pairs past them pass through
  int interleaved;  // used by the scalar layout
  int inverse;
  int w_dtype;
  float eps;
  int group_log2;   // lanes of a row
  int tt_log2;      // tokens of a block
  float* partial;   // [side][kGradBlocks][dim] weight-gradient partials
  const int32_t* lengths;  // backward: tokens of each batch that side 1 has, or NULL
  float* scale;     // FP16 output of other inputs: the powers of two the sides are held times
  double turn[kMaxPairs];
  uint8_t axis[kMaxPairs];
};

__device__ __forceinline__ double position(const RotaryArgs& a, int b, int t, int axis) {
  const int64_t i = int64_t(b) * a.pb + int64_t(t) * a.pt + int64_t(axis) * a.pa;
  switch (a.pos_dtype) {
    case B2_POS_I32: return static_cast<double>(static_cast<const int32_t*>(a.pos)[i]);
    case B2_POS_I64: return static_cast<double>(static_cast<const int64_t*>(a.pos)[i]);
    case B2_POS_F32: return static_cast<double>(static_cast<const float*>(a.pos)[i]);
    default: return static_cast<const double*>(a.pos)[i];
  }
}

// Column of member m (0: first, 1: second) of pair p.  Pairs past the rotated
// ones cover the remaining columns: two by two, or (halves) four first and
// four second members of four pairs, as the lane's two chunks hold them.
template <int LAYOUT>
__device__ __forceinline__ int element(int p, int m, int rot_pairs, bool interleaved) {
  if (LAYOUT == kInterleaved || (LAYOUT == kScalar && interleaved)) return 2 * p + m;
  if (p < rot_pairs) return p + m * rot_pairs;
  return LAYOUT == kHalves ? 2 * (p & ~3) + 4 * m + (p & 3) : 2 * p + m;
}

// Pair i (0..3) of lane l.
template <int LAYOUT>
__device__ __forceinline__ int pair_of(int l, int i) {
  return LAYOUT == kScalar ? l + 32 * i : 4 * l + i;
}

// Columns of the two four-element chunks of lane l (vector layouts).
template <int LAYOUT>
__device__ __forceinline__ void chunks(int l, int rot_pairs, int& c0, int& c1) {
  if (LAYOUT == kInterleaved || 4 * l >= rot_pairs) {
    c0 = 8 * l;
    c1 = 8 * l + 4;
  } else {
    c0 = 4 * l;
    c1 = rot_pairs + 4 * l;
  }
}

// A lane's eight elements of one row as they lie in memory.
template <typename T, int LAYOUT>
struct Raw {
  static constexpr int kWords = sizeof(T) * 2;  // 32-bit words of eight elements
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const char* row, int l, int c0, int c1, int rot_pairs, bool interleaved, int pairs) {
    if constexpr (LAYOUT == kScalar) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = pair_of<LAYOUT>(l, i);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const T v = p < pairs ? reinterpret_cast<const T*>(row)[element<LAYOUT>(p, m, rot_pairs, interleaved)] : T(0.f);
          set(i, m, v);
        }
      }
    } else if constexpr (sizeof(T) == 4) {
      const uint4 a = load16(row + c0 * 4);
      const uint4 b = load16(row + c1 * 4);
      w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    } else if constexpr (LAYOUT == kInterleaved) {
      const uint4 a = load16(row + c0 * 2);
      w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    } else {
      const uint2 a = load8(row + c0 * 2);
      const uint2 b = load8(row + c1 * 2);
      w[0] = a.x, w[1] = a.y, w[2] = b.x, w[3] = b.y;
    }
  }
  __device__ __forceinline__ void store(char* row, int l, int c0, int c1, int rot_pairs, bool interleaved, int pairs) const {
    if constexpr (LAYOUT == kScalar) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = pair_of<LAYOUT>(l, i);
        if (p >= pairs) continue;
#pragma unroll
        for (int m = 0; m < 2; ++m) reinterpret_cast<T*>(row)[element<LAYOUT>(p, m, rot_pairs, interleaved)] = get(i, m);
      }
    } else if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<uint4*>(row + c0 * 4) = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(row + c1 * 4) = make_uint4(w[4], w[5], w[6], w[7]);
    } else if constexpr (LAYOUT == kInterleaved) {
      *reinterpret_cast<uint4*>(row + c0 * 2) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      *reinterpret_cast<uint2*>(row + c0 * 2) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(row + c1 * 2) = make_uint2(w[2], w[3]);
    }
  }
  // The same through shared memory: fetch() starts copies into a slot of the
  // lane's own, take() reads it once they have landed.  No other thread
  // touches the slot, so waiting for the thread's own copies is enough.
  static constexpr int kSlot = sizeof(T) * 8;
  __device__ __forceinline__ static void fetch(char* slot, const char* row, int c0, int c1) {
    const uint32_t to = smem_u32(slot);
    if constexpr (sizeof(T) == 4) {
      cp_async16(to, row + c0 * 4, 16);
      cp_async16(to + 16, row + c1 * 4, 16);
    } else if constexpr (LAYOUT == kInterleaved) {
      cp_async16(to, row + c0 * 2, 16);
    } else {
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(to), "l"(row + c0 * 2) : "memory");
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n" ::"r"(to + 8), "l"(row + c1 * 2) : "memory");
    }
  }
  __device__ __forceinline__ void take(const char* slot) {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(slot + i * 4);
      w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
    }
  }
  // member m of pair i sits at eight-element slot: interleaved 2i+m, halves
  // (and the scalar layout) 4m+i
  static __device__ __forceinline__ constexpr int slot(int i, int m) { return LAYOUT == kInterleaved ? 2 * i + m : 4 * m + i; }
  __device__ __forceinline__ T get(int i, int m) const { return reinterpret_cast<const T*>(w)[slot(i, m)]; }
  __device__ __forceinline__ void set(int i, int m, T v) { reinterpret_cast<T*>(w)[slot(i, m)] = v; }
  __device__ __forceinline__ void widen(float (&v)[8]) const {  // v[2i+m]
    float e[8];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) Cvt<T>::unpack2(w[i], e[2 * i], e[2 * i + 1]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = e[slot(i, 0)];
      v[2 * i + 1] = e[slot(i, 1)];
    }
  }
  __device__ __forceinline__ void narrow(const float (&v)[8]) {
    float e[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[slot(i, 0)] = v[2 * i];
      e[slot(i, 1)] = v[2 * i + 1];
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(e[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = Cvt<T>::pack2(e[2 * i], e[2 * i + 1]);
    }
  }
};

__device__ __forceinline__ float weight_at(const void* w, int dtype, int i) {
  if (dtype == B2_F32) return static_cast<const float*>(w)[i];
  if (dtype == B2_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
  return __half2float(static_cast<const __half*>(w)[i]);
}

// The pairs' rates in shared memory: lanes index them differently, which the
// constant bank of the parameters answers one address at a time (10 us of a
// 9216-token call).
struct RateTable {
  double turn[kMaxPairs];
  uint8_t axis[kMaxPairs];
};
__device__ __forceinline__ void fill_rates(const RotaryArgs& a, RateTable& r) {
  for (int p = threadIdx.x; p < a.rot_pairs; p += kThreads) r.turn[p] = a.turn[p], r.axis[p] = a.axis[p];
}

// cos / sin of a tile's tokens: cs[token][pair].
__device__ __forceinline__ void fill_angles(const RotaryArgs& a, const RateTable& r, float2* cs, int n0, int n_tokens) {
  const int b0 = n0 / a.tokens, t0 = n0 - b0 * a.tokens;
  const int count = min(1 << a.tt_log2, n_tokens - n0) * a.rot_pairs;
  for (int i = threadIdx.x; i < count; i += kThreads) {
    const int tok = static_cast<int>(static_cast<unsigned>(i) / static_cast<unsigned>(a.rot_pairs));
    const int p = i - tok * a.rot_pairs;
    int b = b0, at = t0 + tok;
    while (at >= a.tokens) at -= a.tokens, ++b;  // a tile may span batches
    double turns = position(a, b, at, r.axis[p]) * r.turn[p];
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * static_cast<float>(turns), &s, &c);
    cs[tok * kMaxPairs + p] = make_float2(c, a.inverse ? -s : s);
  }
}

struct Lane {
  int l, tok, gi, gpt, gpt_log2;  // lane in its group, token of the block, group among the token's, groups per token
  int c0, c1;
  bool active;          // the lane's pairs exist
  bool rotates;         // and are rotated (vector layouts)
};

template <int LAYOUT>
__device__ __forceinline__ Lane lane_of(const RotaryArgs& a) {
  Lane t;
  const int g = threadIdx.x >> a.group_log2;
  t.l = threadIdx.x & ((1 << a.group_log2) - 1);
  t.gpt_log2 = 8 - a.group_log2 - a.tt_log2;
  t.gpt = 1 << t.gpt_log2;
  t.gi = g & (t.gpt - 1);
  t.tok = g >> t.gpt_log2;
  t.active = LAYOUT == kScalar ? true : 8 * t.l < a.dim;
  t.rotates = 4 * t.l < a.rot_pairs;
  chunks<LAYOUT>(t.l, a.rot_pairs, t.c0, t.c1);
  return t;
}

// cos and sin of a lane's pairs, (1, 0) for those that pass through.
template <int LAYOUT>
__device__ __forceinline__ void load_angles(const RotaryArgs& a, const float2* cs, const Lane& t, float2 (&ang)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = pair_of<LAYOUT>(t.l, i);
    ang[i] = p < a.rot_pairs ? cs[t.tok * kMaxPairs + p] : make_float2(1.f, 0.f);
  }
}

// The sides' weights in the order of the lanes' pairs: ws[side][8 l + 2 i + m].
template <int LAYOUT>
__device__ __forceinline__ void fill_weights(const RotaryArgs& a, int side, float* ws) {
  const int l = threadIdx.x >> 3, i = (threadIdx.x >> 1) & 3, m = threadIdx.x & 1;
  const int p = pair_of<LAYOUT>(l, i);
  const void* w = a.side[side].w;
  ws[side * kThreads + threadIdx.x] =
      w != nullptr && p < (a.dim >> 1) ? weight_at(w, a.w_dtype, element<LAYOUT>(p, m, a.rot_pairs, a.interleaved != 0)) : 1.f;
}
__device__ __forceinline__ void load_weights(const float* ws, int side, int l, float (&w)[8]) {
  const float4 lo = *reinterpret_cast<const float4*>(ws + side * kThreads + 8 * l);
  const float4 hi = *reinterpret_cast<const float4*>(ws + side * kThreads + 8 * l + 4);
  w[0] = lo.x, w[1] = lo.y, w[2] = lo.z, w[3] = lo.w, w[4] = hi.x, w[5] = hi.y, w[6] = hi.z, w[7] = hi.w;
}

// Sums over the lanes of a row's group; every lane of the warp takes part.
template <int N>
__device__ __forceinline__ void group_sums(float (&v)[N], int group_log2) {
#pragma unroll
  for (int k = 5; k > 0; --k)
    if (group_log2 >= k) {
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], 1 << (k - 1));
    }
}

__device__ __forceinline__ float group_sum(float v, int group_log2) {
  float one[1] = {v};
  group_sums<1>(one, group_log2);
  return one[0];
}

// (v_a, v_b) = (v_a k.x - v_b k.y, v_a k.z + v_b k.w) for the rotated pairs,
// (v_a k.x, v_b k.w) for the others: a rotation by nothing would turn
// x + 0 * inf into NaN.  All pairs of a lane rotate or none does, but in the
// scalar layout.
template <int LAYOUT>
__device__ __forceinline__ void turn(const float4 (&k)[4], float (&v)[8], const Lane& t, int rot_pairs) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = v[2 * i], y = v[2 * i + 1];
    if (LAYOUT == kScalar ? pair_of<LAYOUT>(t.l, i) < rot_pairs : t.rotates) {
      v[2 * i] = x * k[i].x - y * k[i].y;
      v[2 * i + 1] = x * k[i].z + y * k[i].w;
    } else {
      v[2 * i] = x * k[i].x;
      v[2 * i + 1] = y * k[i].w;
    }
  }
}

// Rows of x and of dy in flight for a thread of the backward pass.  Forward
// keeps its four rows in registers instead: computing four at a time hides
// the group sums, and measured 114 us against 126 (32760 x 40 x 128) for the
// same ring of slots.
constexpr int kAheadGrad = 4;

// A group's rows of one token and side: heads gi, gi + gpt, ...
struct Walk {
  char* p;
  int64_t step;  // bytes between the rows
  __device__ __forceinline__ Walk(const RowSet& r, int b, int tok, const Lane& t, int es)
      : p(r.base + (int64_t(b) * r.sb + int64_t(tok) * r.st + t.gi * r.sh) * es), step(t.gpt * r.sh * es) {}
  __device__ __forceinline__ char* at(int u) const { return p + u * step; }
  __device__ __forceinline__ void next(int u = 1) { p += u * step; }
};

// The power of two a normed side is held times in FP16, from its largest
// weight: |y| <= sqrt(2 D) max|w|, which becomes 2^13 .. 2^14.
__device__ __forceinline__ float side_scale(const RotaryArgs& a, int side, float* shared) {
  float most = 0.f;
  for (int d = threadIdx.x; d < a.dim; d += kThreads)
    most = fmaxf(most, a.side[side].w != nullptr ? fabsf(weight_at(a.side[side].w, a.w_dtype, d)) : 1.f);
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, w));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = most;
  __syncthreads();
  most = shared[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) most = fmaxf(most, shared[w]);
  const float bound = most * sqrtf(2.f * a.dim);
  if (!(bound > 0.f) || !(bound < 3e38f)) return 1.f;
  return ldexpf(1.f, min(max(13 - ilogbf(bound), -60), 60));
}

// TO: the output's type, T but for the FP16 copies that attention's products
// read (the scale above then multiplies the weights).
template <typename T, typename TO, int LAYOUT, bool NORM>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 && LAYOUT != kScalar ? 4 : 2)
rotary_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int U = 4;  // rows of a group in flight
  __shared__ float2 cs[kMaxTokens * kMaxPairs];
  __shared__ RateTable rates;
  __shared__ __align__(16) float ws[NORM ? 2 * kThreads : 4];
  const int n_tokens = a.batch * a.tokens;
  const Lane t = lane_of<LAYOUT>(a);
  const int pairs = a.dim >> 1;
  const bool inter = a.interleaved != 0;
  const float inv_dim = 1.f / static_cast<float>(a.dim);
  fill_rates(a, rates);
  if constexpr (NORM) {
    fill_weights<LAYOUT>(a, 0, ws);
    fill_weights<LAYOUT>(a, 1, ws);
    if (a.scale != nullptr) {
      __shared__ float shared[kThreads / 32];
      for (int side = 0; side < a.sides; ++side) {
        const float scale = side_scale(a, side, shared);
        ws[side * kThreads + threadIdx.x] *= scale;
        if (blockIdx.x == 0 && threadIdx.x == 0) a.scale[side] = scale;
      }
    }
  }
  for (int n0 = blockIdx.x << a.tt_log2; n0 < n_tokens; n0 += gridDim.x << a.tt_log2) {
    const int n = n0 + t.tok;
    const int b = n / a.tokens;
    const int tok = n - b * a.tokens;
    float2 ang[4];
    for (int side = 0; side < a.sides; ++side) {
      const Side& s = a.side[side];
      Walk x(s.x, b, tok, t, sizeof(T)), y(s.y, b, tok, t, sizeof(TO));
      int left = n < n_tokens && t.active ? (s.heads - t.gi + t.gpt - 1) >> t.gpt_log2 : 0;  // rows of this group
      // every thread of the block runs the same number of steps: the group
      // sums are full-warp shuffles
      const int steps = (s.heads + t.gpt - 1) >> t.gpt_log2;
      float4 k[4];  // rotation times weights
      for (int step = 0; step < steps; step += U, left -= U) {
        Raw<T, LAYOUT> raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (u < left) raw[u].load(x.at(u), t.l, t.c0, t.c1, a.rot_pairs, inter, pairs);
          else
            for (int i = 0; i < Raw<T, LAYOUT>::kWords; ++i) raw[u].w[i] = 0u;
        }
        x.next(U);
        if (step == 0) {
          if (side == 0) {  // with the first rows on their way
            __syncthreads();  // the last tile's angles are read
            fill_angles(a, rates, cs, n0, n_tokens);
            __syncthreads();
            load_angles<LAYOUT>(a, cs, t, ang);
          }
          float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
          if constexpr (NORM) load_weights(ws, side, t.l, w);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            k[i] = make_float4(w[2 * i] * ang[i].x, w[2 * i + 1] * ang[i].y, w[2 * i] * ang[i].y, w[2 * i + 1] * ang[i].x);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (step + u >= steps) break;
          float v[8];
          raw[u].widen(v);
          if constexpr (NORM) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(v[i], v[i], sum);
            const float rstd = rsqrtf(group_sum(sum, a.group_log2) * inv_dim + a.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= rstd;
          }
          turn<LAYOUT>(k, v, t, a.rot_pairs);
          if (u < left) {
            Raw<TO, LAYOUT> to;
            to.narrow(v);
            to.store(y.at(u), t.l, t.c0, t.c1, a.rot_pairs, inter, pairs);
          }
        }
        y.next(U);
      }
    }
  }
}

// Gradients of norm + rotation.  Blocks stride over the token tiles of one
// side, so a lane's weight gradients stay in registers until the end and the
// partials are few; their order, and so the result, is fixed.
template <typename T, typename TD, int LAYOUT>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 && LAYOUT != kScalar ? 3 : 2)
rotary_grad_kernel(const __grid_constant__ RotaryArgs a) {
  using R = Raw<T, LAYOUT>;
  using RD = Raw<TD, LAYOUT>;  // dy
  extern __shared__ __align__(16) char slots[];
  __shared__ float2 cs[kMaxTokens * kMaxPairs];
  __shared__ RateTable rates;
  __shared__ __align__(16) float ws[2 * kThreads];
  const Side& s = a.side[blockIdx.y];
  const int n_tokens = a.batch * a.tokens;
  const Lane t = lane_of<LAYOUT>(a);
  const int pairs = a.dim >> 1;
  const bool inter = a.interleaved != 0;
  const float inv_dim = 1.f / static_cast<float>(a.dim);
  const int steps = (s.heads + t.gpt - 1) >> t.gpt_log2;
  constexpr int kStage = kThreads * (R::kSlot + RD::kSlot);  // x, then dy
  char* const own_x = slots + threadIdx.x * R::kSlot;
  char* const own_dy = slots + kThreads * R::kSlot + threadIdx.x * RD::kSlot;
  float w[8], dw[8] = {};
  fill_rates(a, rates);
  fill_weights<LAYOUT>(a, blockIdx.y, ws);
  __syncthreads();
  load_weights(ws, blockIdx.y, t.l, w);
  for (int n0 = blockIdx.x << a.tt_log2; n0 < n_tokens; n0 += gridDim.x << a.tt_log2) {
    const int n = n0 + t.tok;
    const int b = n / a.tokens;
    const int tok = n - b * a.tokens;
    Walk wx(s.x, b, tok, t, sizeof(T)), wdy(s.dy, b, tok, t, sizeof(TD)), wy(s.y, b, tok, t, sizeof(T));
    const int rows = n < n_tokens && t.active ? (s.heads - t.gi + t.gpt - 1) >> t.gpt_log2 : 0;
    // keys past a batch's count: whatever they hold, their gradient is 0
    const bool dead = a.lengths != nullptr && blockIdx.y == 1 && n < n_tokens && tok >= a.lengths[b];
    auto fetch = [&](int j) {
      if constexpr (LAYOUT != kScalar) {
        if (j < rows) {
          R::fetch(own_x + (j % kAheadGrad) * kStage, wx.p, t.c0, t.c1);
          RD::fetch(own_dy + (j % kAheadGrad) * kStage, wdy.p, t.c0, t.c1);
        }
        wx.next(), wdy.next();
        cp_async_commit();
      }
    };
#pragma unroll 1
    for (int j = 0; j < kAheadGrad; ++j) fetch(j);
    __syncthreads();  // the last tile's angles are read
    fill_angles(a, rates, cs, n0, n_tokens);
    __syncthreads();
    float4 k[4];  // the rotation back
    {
      float2 ang[4];
      load_angles<LAYOUT>(a, cs, t, ang);
#pragma unroll
      for (int i = 0; i < 4; ++i) k[i] = make_float4(ang[i].x, -ang[i].y, -ang[i].y, ang[i].x);
    }
#pragma unroll 1
    for (int j = 0; j < steps; ++j) {
      R rx;
      RD rdy;
      if constexpr (LAYOUT == kScalar) {
        if (j < rows) {
          rx.load(wx.p, t.l, t.c0, t.c1, a.rot_pairs, inter, pairs);
          rdy.load(wdy.p, t.l, t.c0, t.c1, a.rot_pairs, inter, pairs);
        } else {
          rx = R{};
          rdy = RD{};
        }
        wx.next(), wdy.next();
      } else {
        cp_async_wait<kAheadGrad - 1>();
        rx.take(own_x + (j % kAheadGrad) * kStage);
        rdy.take(own_dy + (j % kAheadGrad) * kStage);
      }
      float x[8], g[8];
      rx.widen(x);
      rdy.widen(g);
      fetch(j + kAheadGrad);
      turn<LAYOUT>(k, g, t, a.rot_pairs);  // dz
      const bool counts = j < rows && !dead;
      if (!counts) {  // what a slot held before may be NaN, and so may the angles of a token past the last
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = g[i] = 0.f;
      }
      float sum = 0.f, dot = 0.f, gw[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum = fmaf(x[i], x[i], sum);
        gw[i] = g[i] * w[i];
        dot = fmaf(gw[i], x[i], dot);
      }
      float sums[2] = {sum, dot};
      group_sums<2>(sums, a.group_log2);
      const float r = counts ? rsqrtf(sums[0] * inv_dim + a.eps) : 0.f;  // eps may be 0
      const float back = -sums[1] * inv_dim * r;  // -mean(g w xh)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] *= r;  // xh
        dw[i] = fmaf(g[i], x[i], dw[i]);
        g[i] = fmaf(back, x[i], gw[i]) * r;
      }
      if (j < rows) {
        rx.narrow(g);
        rx.store(wy.p, t.l, t.c0, t.c1, a.rot_pairs, inter, pairs);
      }
      wy.next();
    }
  }
  if (s.dw == nullptr) return;
  // sum the groups of the block in a fixed order: [group][column] over cs
  __syncthreads();
  float* part = reinterpret_cast<float*>(cs);
  const int g = threadIdx.x >> a.group_log2;
  const int groups = kThreads >> a.group_log2;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int p = pair_of<LAYOUT>(t.l, i);
      if (p < pairs) part[g * a.dim + element<LAYOUT>(p, m, a.rot_pairs, inter)] = dw[2 * i + m];
    }
  __syncthreads();
  for (int d = threadIdx.x; d < a.dim; d += kThreads) {
    float sum = 0.f;
    for (int k = 0; k < groups; ++k) sum += part[k * a.dim + d];
    a.partial[(int64_t(blockIdx.y) * kGradBlocks + blockIdx.x) * a.dim + d] = sum;
  }
}

// dw[d] = sum of the blocks' partials, in a fixed order.
__global__ void __launch_bounds__(1024) rotary_dw_kernel(const __grid_constant__ RotaryArgs a, int blocks) {
  __shared__ float part[32][33];
  const Side& s = a.side[blockIdx.y];
  grid_dep_wait();
  if (s.dw == nullptr) return;
  const int d = blockIdx.x * 32 + threadIdx.x;
  const float* src = a.partial + int64_t(blockIdx.y) * kGradBlocks * a.dim;
  float sum = 0.f;
  if (d < a.dim) {
#pragma unroll 4
    for (int k = threadIdx.y; k < blocks; k += 32) sum += src[int64_t(k) * a.dim + d];
  }
  part[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  sum = part[threadIdx.x][threadIdx.y];  // thread (x, y): partial x of column y
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  const int col = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && col < a.dim) {
    if (a.w_dtype == B2_F32) static_cast<float*>(s.dw)[col] = sum;
    else if (a.w_dtype == B2_BF16) static_cast<__nv_bfloat16*>(s.dw)[col] = __float2bfloat16_rn(sum);
    else static_cast<__half*>(s.dw)[col] = __float2half_rn(sum);
  }
}

RowSet rows_of(const b2_view* v) {
  if (v == nullptr) return RowSet{};
  return RowSet{static_cast<char*>(v->base), v->stride_b, v->stride_h, v->stride_t};
}

// Turns per position and axis of every pair.  The last rotation's are kept
// per thread (64 calls of pow are 2.5 us of host time for D = 128).
struct Rates {
  int n_axes = 0;
  int32_t dims[B2_MAX_AXES];
  double theta[B2_MAX_AXES];
  int pairs;
  double turn[kMaxPairs];
  uint8_t axis[kMaxPairs];
};

const Rates& rates_of(const b2_rotary& r) {
  static thread_local Rates k;
  bool same = k.n_axes == r.n_axes;
  for (int i = 0; same && i < r.n_axes; ++i) same = k.dims[i] == r.axes_dims[i] && k.theta[i] == r.theta[i];
  if (same) return k;
  k.n_axes = r.n_axes;
  k.pairs = 0;
  for (int x = 0; x < r.n_axes; ++x) {
    k.dims[x] = r.axes_dims[x];
    k.theta[x] = r.theta[x];
    for (int j = 0; j < r.axes_dims[x] / 2; ++j, ++k.pairs) {
      k.turn[k.pairs] = pow(r.theta[x], -2.0 * j / r.axes_dims[x]) / 6.283185307179586476925286766559;
      k.axis[k.pairs] = static_cast<uint8_t>(x);
    }
  }
  return k;
}

// T: inputs; TX: the other type of the call (forward: the output's, backward: dy's).
template <typename T, typename TX, int LAYOUT>
cudaError_t launch_layout(const RotaryArgs& a, bool norm, bool grad, int64_t tiles, cudaStream_t st) {
  using Kernel = void (*)(const RotaryArgs);
  Kernel kernel;
  int smem = 0;
  if (grad) {
    kernel = rotary_grad_kernel<T, TX, LAYOUT>;
    if (LAYOUT != kScalar) smem = kAheadGrad * kThreads * (Raw<T, LAYOUT>::kSlot + Raw<TX, LAYOUT>::kSlot);
  } else if constexpr (std::is_same<T, TX>::value) {
    kernel = norm ? Kernel(rotary_kernel<T, TX, LAYOUT, true>) : Kernel(rotary_kernel<T, TX, LAYOUT, false>);
  } else {
    return cudaErrorInvalidValue;
  }
  cudaError_t err = ensure_smem(reinterpret_cast<const void*>(kernel), smem);
  if (err != cudaSuccess) return err;
  const int most = grad ? kGradBlocks : kBlocks;
  const dim3 grid(static_cast<unsigned>(tiles < most ? tiles : most), grad ? a.sides : 1);
  kernel<<<grid, kThreads, smem, st>>>(a);
  if ((err = cudaGetLastError()) != cudaSuccess || (a.side[0].dw == nullptr && a.side[1].dw == nullptr)) return err;
  return launch_pdl(rotary_dw_kernel, dim3((a.dim + 31) / 32, a.sides), dim3(32, 32), size_t(0), st, a,
                    static_cast<int>(grid.x));
}

template <typename T, typename TX>
cudaError_t launch_typed(const RotaryArgs& a, int layout, bool norm, bool grad, int64_t tiles, cudaStream_t st) {
  if (layout == kInterleaved) return launch_layout<T, TX, kInterleaved>(a, norm, grad, tiles, st);
  if (layout == kHalves) return launch_layout<T, TX, kHalves>(a, norm, grad, tiles, st);
  return launch_layout<T, TX, kScalar>(a, norm, grad, tiles, st);
}

// The FP16 copies of BF16 queries and keys.
template <int LAYOUT>
cudaError_t launch_copies(const RotaryArgs& a, int64_t tiles, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(tiles < kBlocks ? tiles : kBlocks));
  rotary_kernel<__nv_bfloat16, __half, LAYOUT, true><<<grid, kThreads, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

int64_t rotary_workspace_bytes(int head_dim) { return int64_t(2) * kGradBlocks * head_dim * 4; }

cudaError_t launch_rotary(const RotaryCall& c, cudaStream_t st) {
  RotaryArgs a{};
  const b2_view& v = *c.x[0];
  const int sides = c.x[1] != nullptr ? 2 : 1;
  const bool grad = c.dy[0] != nullptr;
  int rows = 0;  // of a token that a block walks
  for (int i = 0; i < sides; ++i) {
    Side& s = a.side[i];
    s.x = rows_of(c.x[i]);
    s.dy = rows_of(c.dy[i]);
    s.y = rows_of(c.y[i]);
    s.w = c.w[i];
    s.dw = c.dw[i];
    s.heads = c.x[i]->heads;
    rows = grad ? (s.heads > rows ? s.heads : rows) : rows + s.heads;
  }
  a.pos = c.rot->positions;
  a.pb = c.rot->stride_b, a.pt = c.rot->stride_t, a.pa = c.rot->stride_axis;
  a.pos_dtype = c.rot->pos_dtype;
  a.sides = sides;
  a.batch = v.batch, a.tokens = v.tokens, a.dim = v.head_dim;
  a.interleaved = c.rot->interleaved;
  a.inverse = c.rot->inverse;
  a.w_dtype = c.w_dtype;
  a.eps = c.eps;
  a.partial = c.partial;
  const Rates& rates = rates_of(*c.rot);
  const int p = rates.pairs;
  memcpy(a.turn, rates.turn, sizeof(double) * p);
  memcpy(a.axis, rates.axis, p);
  a.rot_pairs = p;
  // rotations that end inside a lane's four pairs (R % 8 != 0) go pair by pair
  const int layout = p % 4 ? kScalar : a.interleaved ? kInterleaved : kHalves;
  a.group_log2 = 5;
  if (layout != kScalar)
    while (a.group_log2 > 0 && (8 << (a.group_log2 - 1)) >= a.dim) --a.group_log2;
  // Tokens of a tile: the number that takes the fewest row steps of the
  // busiest block, counting a tile's set-up (angles, two barriers) as four.
  const int groups_log2 = 8 - a.group_log2;
  const int64_t n_tokens = int64_t(a.batch) * a.tokens;
  const int blocks = grad ? kGradBlocks : kBlocks;
  int tt_log2 = 0;
  int64_t best = 0;
  for (int x = 0; x <= groups_log2 && x <= 4; ++x) {
    const int64_t rounds = (((n_tokens + (1 << x) - 1) >> x) + blocks - 1) / blocks;
    const int64_t cost = rounds * ((((int64_t(rows) << x) + (1 << groups_log2) - 1) >> groups_log2) + 4);
    if (x == 0 || cost < best) best = cost, tt_log2 = x;
  }
  a.tt_log2 = tt_log2;
  const int64_t tiles = (n_tokens + (1 << tt_log2) - 1) >> tt_log2;
  a.scale = c.scale;
  a.lengths = c.lengths;
  if (c.scale != nullptr && v.dtype == B2_BF16)
    return layout == kInterleaved ? launch_copies<kInterleaved>(a, tiles, st)
                                  : layout == kHalves ? launch_copies<kHalves>(a, tiles, st) : launch_copies<kScalar>(a, tiles, st);
  const bool dy32 = grad && c.dy[0]->dtype == B2_F32;
  switch (v.dtype) {
    case B2_BF16:
      return dy32 ? launch_typed<__nv_bfloat16, float>(a, layout, c.norm, grad, tiles, st)
                  : launch_typed<__nv_bfloat16, __nv_bfloat16>(a, layout, c.norm, grad, tiles, st);
    case B2_F16:
      return dy32 ? launch_typed<__half, float>(a, layout, c.norm, grad, tiles, st)
                  : launch_typed<__half, __half>(a, layout, c.norm, grad, tiles, st);
    default: return launch_typed<float, float>(a, layout, c.norm, grad, tiles, st);
  }
}

}  // namespace b2
