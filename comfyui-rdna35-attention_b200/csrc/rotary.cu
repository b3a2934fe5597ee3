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
// pairs) or two of 8 bytes (halves).  A block takes `tt` tokens of one side
// (queries or keys); its 256 threads compute the tokens' cos / sin once into
// shared memory (one sincospif per thread for H = 16, D = 128) and every group
// then walks heads of one token, four rows in flight.
#include <math.h>
#include <string.h>

#include "kernels.h"

namespace b2 {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;     // D <= 256
constexpr int kMaxTokens = 16;     // tokens of a block
constexpr int kGradBlocks = 148 * 4;  // blocks of one side in the backward pass: partial weight gradients

enum Layout { kInterleaved = 0, kHalves = 1, kScalar = 2 };

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
  int batch, tokens, dim;
  int rot_pairs;    // rotated pairs; pairs past them pass through
  int interleaved;  // used by the scalar layout
  int inverse;
  int w_dtype;
  float eps;
  int group_log2;   // lanes of a row
  int tt_log2;      // tokens of a block
  float* partial;   // [side][kGradBlocks][dim] weight-gradient partials
  double turn[kMaxPairs];
  uint8_t axis[kMaxPairs];
};

__device__ __forceinline__ char* row_ptr(const RowSet& r, int64_t b, int h, int64_t t, int es) {
  return r.base + (b * r.sb + int64_t(h) * r.sh + t * r.st) * es;
}

__device__ __forceinline__ double position(const RotaryArgs& a, int64_t b, int64_t t, int axis) {
  const int64_t i = b * a.pb + t * a.pt + int64_t(axis) * a.pa;
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
      const uint4 a = *reinterpret_cast<const uint4*>(row + c0 * 4);
      const uint4 b = *reinterpret_cast<const uint4*>(row + c1 * 4);
      w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    } else if constexpr (LAYOUT == kInterleaved) {
      const uint4 a = *reinterpret_cast<const uint4*>(row + c0 * 2);
      w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    } else {
      const uint2 a = *reinterpret_cast<const uint2*>(row + c0 * 2);
      const uint2 b = *reinterpret_cast<const uint2*>(row + c1 * 2);
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

// cos / sin of the block's tokens: cs[token][pair].
__device__ __forceinline__ void fill_angles(const RotaryArgs& a, float2* cs, int64_t n0, int tt, int64_t n_tokens) {
  for (int i = threadIdx.x; i < tt * a.rot_pairs; i += kThreads) {
    const int tok = i / a.rot_pairs;
    const int p = i - tok * a.rot_pairs;
    const int64_t n = n0 + tok;
    if (n >= n_tokens) break;
    const int64_t b = n / a.tokens;
    double turns = position(a, b, n - b * a.tokens, a.axis[p]) * a.turn[p];
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * static_cast<float>(turns), &s, &c);
    cs[tok * kMaxPairs + p] = make_float2(c, a.inverse ? -s : s);
  }
}

struct Lane {
  int l, tok, gi, gpt;  // lane in its group, token of the block, group among the token's, groups per token
  int c0, c1;
  bool active;          // the lane's pairs exist
};

template <int LAYOUT>
__device__ __forceinline__ Lane lane_of(const RotaryArgs& a) {
  Lane t;
  const int g = threadIdx.x >> a.group_log2;
  t.l = threadIdx.x & ((1 << a.group_log2) - 1);
  const int gpt_log2 = 8 - a.group_log2 - a.tt_log2;
  t.gpt = 1 << gpt_log2;
  t.gi = g & (t.gpt - 1);
  t.tok = g >> gpt_log2;
  t.active = LAYOUT == kScalar ? true : 8 * t.l < a.dim;
  chunks<LAYOUT>(t.l, a.rot_pairs, t.c0, t.c1);
  return t;
}

template <int LAYOUT>
__device__ __forceinline__ void load_angles(const RotaryArgs& a, const float2* cs, const Lane& t, float2 (&ang)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = pair_of<LAYOUT>(t.l, i);
    ang[i] = p < a.rot_pairs ? cs[t.tok * kMaxPairs + p] : make_float2(1.f, 0.f);
  }
}

template <int LAYOUT>
__device__ __forceinline__ void load_weights(const RotaryArgs& a, const Side& s, const Lane& t, float (&w)[8]) {
  const int pairs = a.dim >> 1;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const int p = pair_of<LAYOUT>(t.l, i);
      w[2 * i + m] =
          s.w != nullptr && p < pairs
              ? weight_at(s.w, a.w_dtype, element<LAYOUT>(p, m, a.rot_pairs, a.interleaved != 0))
              : 1.f;
    }
}

// Sum over the lanes of a row's group; every lane of the warp takes part.
__device__ __forceinline__ float group_sum(float v, int group_log2) {
  for (int off = 1 << group_log2 >> 1; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// Pairs past the rotated ones keep their bits (an identity rotation would
// turn x + 0 * inf into NaN).
template <int LAYOUT>
__device__ __forceinline__ void rotate(const float2 (&ang)[4], float (&v)[8], int l, int rot_pairs, bool back) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (pair_of<LAYOUT>(l, i) < rot_pairs) {
      const float c = ang[i].x, s = back ? -ang[i].y : ang[i].y;
      const float x = v[2 * i], y = v[2 * i + 1];
      v[2 * i] = x * c - y * s;
      v[2 * i + 1] = x * s + y * c;
    }
  }
}

template <typename T, int LAYOUT, bool NORM>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int U = 4;  // rows in flight per group
  __shared__ float2 cs[kMaxTokens * kMaxPairs];
  const Side& s = a.side[blockIdx.y];
  const int tt = 1 << a.tt_log2;
  const int64_t n_tokens = int64_t(a.batch) * a.tokens;
  const int64_t n0 = int64_t(blockIdx.x) * tt;
  const Lane t = lane_of<LAYOUT>(a);
  const int pairs = a.dim >> 1;
  const bool inter = a.interleaved != 0;
  const int64_t n = n0 + t.tok;
  const int64_t b = n / a.tokens;
  const int64_t tok = n - b * a.tokens;
  const bool here = n < n_tokens && t.active;
  const float inv_dim = 1.f / static_cast<float>(a.dim);
  float w[8];
  if constexpr (NORM) load_weights<LAYOUT>(a, s, t, w);
  fill_angles(a, cs, n0, tt, n_tokens);
  __syncthreads();
  float2 ang[4];
  load_angles<LAYOUT>(a, cs, t, ang);
  // every thread of the block runs the same number of steps: the group sums
  // are full-warp shuffles
  for (int h0 = 0; h0 < s.heads; h0 += U * t.gpt) {
    Raw<T, LAYOUT> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * t.gpt + t.gi;
      if (here && h < s.heads)
        raw[u].load(row_ptr(s.x, b, h, tok, sizeof(T)), t.l, t.c0, t.c1, a.rot_pairs, inter, pairs);
      else
        for (int i = 0; i < Raw<T, LAYOUT>::kWords; ++i) raw[u].w[i] = 0u;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (h0 + u * t.gpt >= s.heads) break;
      const int h = h0 + u * t.gpt + t.gi;
      float v[8];
      raw[u].widen(v);
      if constexpr (NORM) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(v[i], v[i], sum);
        const float r = rsqrtf(group_sum(sum, a.group_log2) * inv_dim + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= r * w[i];
      }
      rotate<LAYOUT>(ang, v, t.l, a.rot_pairs, false);
      if (here && h < s.heads) {
        raw[u].narrow(v);
        raw[u].store(row_ptr(s.y, b, h, tok, sizeof(T)), t.l, t.c0, t.c1, a.rot_pairs, inter, pairs);
      }
    }
  }
}

// Gradients of norm + rotation.  Blocks stride over the token tiles, so a
// lane's weight gradients stay in registers until the end and the partials
// are few; their order, and so the result, is fixed.
template <typename T, int LAYOUT>
__global__ void __launch_bounds__(kThreads) rotary_grad_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int U = 2;
  __shared__ float2 cs[kMaxTokens * kMaxPairs];
  const Side& s = a.side[blockIdx.y];
  const int tt = 1 << a.tt_log2;
  const int64_t n_tokens = int64_t(a.batch) * a.tokens;
  const Lane t = lane_of<LAYOUT>(a);
  const int pairs = a.dim >> 1;
  const bool inter = a.interleaved != 0;
  const float inv_dim = 1.f / static_cast<float>(a.dim);
  float w[8], dw[8] = {};
  load_weights<LAYOUT>(a, s, t, w);
  for (int64_t n0 = int64_t(blockIdx.x) * tt; n0 < n_tokens; n0 += int64_t(gridDim.x) * tt) {
    const int64_t n = n0 + t.tok;
    const int64_t b = n / a.tokens;
    const int64_t tok = n - b * a.tokens;
    const bool here = n < n_tokens && t.active;
    __syncthreads();
    fill_angles(a, cs, n0, tt, n_tokens);
    __syncthreads();
    float2 ang[4];
    load_angles<LAYOUT>(a, cs, t, ang);
    for (int h0 = 0; h0 < s.heads; h0 += U * t.gpt) {
      Raw<T, LAYOUT> rx[U], rdy[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int h = h0 + u * t.gpt + t.gi;
        if (here && h < s.heads) {
          rx[u].load(row_ptr(s.x, b, h, tok, sizeof(T)), t.l, t.c0, t.c1, a.rot_pairs, inter, pairs);
          rdy[u].load(row_ptr(s.dy, b, h, tok, sizeof(T)), t.l, t.c0, t.c1, a.rot_pairs, inter, pairs);
        } else {
          for (int i = 0; i < Raw<T, LAYOUT>::kWords; ++i) rx[u].w[i] = rdy[u].w[i] = 0u;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (h0 + u * t.gpt >= s.heads) break;
        const int h = h0 + u * t.gpt + t.gi;
        float x[8], g[8];
        rx[u].widen(x);
        rdy[u].widen(g);
        rotate<LAYOUT>(ang, g, t.l, a.rot_pairs, true);  // dz
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
        const float r = rsqrtf(group_sum(sum, a.group_log2) * inv_dim + a.eps);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] *= r;                          // xh
          dw[i] = fmaf(g[i], x[i], dw[i]);
          g[i] *= w[i];
          dot = fmaf(g[i], x[i], dot);
        }
        dot = group_sum(dot, a.group_log2) * inv_dim;
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = r * fmaf(-x[i], dot, g[i]);
        if (here && h < s.heads) {
          rx[u].narrow(g);
          rx[u].store(row_ptr(s.y, b, h, tok, sizeof(T)), t.l, t.c0, t.c1, a.rot_pairs, inter, pairs);
        }
      }
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

template <typename T>
cudaError_t launch_typed(const RotaryArgs& a, int layout, bool norm, bool grad, int sides, int64_t tiles,
                         cudaStream_t st) {
  if (grad) {
    const dim3 grid(static_cast<unsigned>(tiles < kGradBlocks ? tiles : kGradBlocks), sides);
    if (layout == kInterleaved) rotary_grad_kernel<T, kInterleaved><<<grid, kThreads, 0, st>>>(a);
    else if (layout == kHalves) rotary_grad_kernel<T, kHalves><<<grid, kThreads, 0, st>>>(a);
    else rotary_grad_kernel<T, kScalar><<<grid, kThreads, 0, st>>>(a);
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess || (a.side[0].dw == nullptr && a.side[1].dw == nullptr)) return err;
    return launch_pdl(rotary_dw_kernel, dim3((a.dim + 31) / 32, sides), dim3(32, 32), size_t(0), st, a,
                      static_cast<int>(grid.x));
  }
  const dim3 grid(static_cast<unsigned>(tiles), sides);
  if (norm) {
    if (layout == kInterleaved) rotary_kernel<T, kInterleaved, true><<<grid, kThreads, 0, st>>>(a);
    else if (layout == kHalves) rotary_kernel<T, kHalves, true><<<grid, kThreads, 0, st>>>(a);
    else rotary_kernel<T, kScalar, true><<<grid, kThreads, 0, st>>>(a);
  } else {
    if (layout == kInterleaved) rotary_kernel<T, kInterleaved, false><<<grid, kThreads, 0, st>>>(a);
    else if (layout == kHalves) rotary_kernel<T, kHalves, false><<<grid, kThreads, 0, st>>>(a);
    else rotary_kernel<T, kScalar, false><<<grid, kThreads, 0, st>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace

int64_t rotary_workspace_bytes(int head_dim) { return int64_t(2) * kGradBlocks * head_dim * 4; }

cudaError_t launch_rotary(const RotaryCall& c, cudaStream_t st) {
  RotaryArgs a{};
  const b2_view& v = *c.x[0];
  const int sides = c.x[1] != nullptr ? 2 : 1;
  int most_heads = 0;
  for (int i = 0; i < sides; ++i) {
    Side& s = a.side[i];
    s.x = rows_of(c.x[i]);
    s.dy = rows_of(c.dy[i]);
    s.y = rows_of(c.y[i]);
    s.w = c.w[i];
    s.dw = c.dw[i];
    s.heads = c.x[i]->heads;
    most_heads = s.heads > most_heads ? s.heads : most_heads;
  }
  a.pos = c.rot->positions;
  a.pb = c.rot->stride_b, a.pt = c.rot->stride_t, a.pa = c.rot->stride_axis;
  a.pos_dtype = c.rot->pos_dtype;
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
  // halves of fewer than four aligned pairs a lane (R % 8 != 0) go pair by pair
  const int layout = a.interleaved ? kInterleaved : (p % 4 == 0 ? kHalves : kScalar);
  a.group_log2 = 5;
  if (layout != kScalar)
    while (a.group_log2 > 0 && (8 << (a.group_log2 - 1)) >= a.dim) --a.group_log2;
  // tokens of a block: about eight rows a group, so that a block's cos / sin
  // and set-up are spread over many rows; fewer while the grid would leave
  // SMs without a block
  const int groups_log2 = 8 - a.group_log2;
  const int64_t n_tokens = int64_t(a.batch) * a.tokens;
  int tt_log2 = groups_log2 < 4 ? groups_log2 : 4;
  while (tt_log2 > 0 && ((most_heads << tt_log2) > (8 << groups_log2) || (n_tokens >> tt_log2) * sides < 148 * 2)) --tt_log2;
  a.tt_log2 = tt_log2;
  const int64_t tiles = (n_tokens + (1 << tt_log2) - 1) >> tt_log2;
  const bool grad = c.dy[0] != nullptr;
  switch (v.dtype) {
    case B2_BF16: return launch_typed<__nv_bfloat16>(a, layout, c.norm, grad, sides, tiles, st);
    case B2_F16: return launch_typed<__half>(a, layout, c.norm, grad, sides, tiles, st);
    default: return launch_typed<float>(a, layout, c.norm, grad, sides, tiles, st);
  }
}

}  // namespace b2
