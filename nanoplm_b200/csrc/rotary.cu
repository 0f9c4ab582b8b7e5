// Rotary positions of queries and keys in one launch: half (i, i + R/2) or interleaved (2i, 2i + 1) pairs, the first R of a
// head's D channels, any number of query and key heads, any token, head and batch strides.
//
// For pair i of a token at position p, with a = p w_i, and the factor f of the frequency scaling:
//   y1 = f (x1 cos a - x2 sin a),  y2 = f (x2 cos a + x1 sin a);  the gradient is the transpose, sin negated.
//
// Bound by memory: a pair costs 4 multiplications, and its cos and sin serve all heads of the token. So a block takes a few
// tokens, forms their cos and sin once in shared memory and then streams the heads. No table: a table in fp32 ends at a
// largest position, and fp32 angles are off by p 2^-24 radians. Here p w_i is formed in fp64 as a number of turns, whose
// whole part is dropped before the rest becomes a fp32 argument in [-1, 1] half turns of sincospi. That cast is off by at most
// 2 pi 2^-26 = 9.4e-8 radians (1.6 units of 2^-24), whatever the position; the three roundings of fp64 before it show
// beyond position 2^26 and come to 5e-7 radians at 2^31 (replayed with 60 digits).
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"

namespace nplm {

constexpr int ROT_THREADS = 256;
constexpr int ROT_STAGED = 32 * 1024;   // shared memory of a block that turns pairs there
constexpr int ROT_PAIRS = 2048;     // cos and sin of a block's tokens: 16 KB
// Items that a thread has in flight.
__host__ __device__ constexpr int rot_unroll(int bytes) { return bytes >= 16 ? 2 : 4; }

// Division of numbers below 2^32 / d by d: a product with 2^32 / d, rounded up, whose excess stays below a 1 / d.
struct RotDiv {
  uint32_t m, one;
  RotDiv() = default;
  explicit RotDiv(uint32_t d) : m(d > 1 ? static_cast<uint32_t>((0x100000000ull + d - 1) / d) : 0u), one(d == 1) {}
  __device__ __forceinline__ int of(int j) const {
    return static_cast<int>(__umulhi(static_cast<uint32_t>(j), m) + static_cast<uint32_t>(j) * one);
  }
};

struct RotaryArgs {
  const void* x[2];                 // queries, keys (keys may have no heads)
  void* y[2];
  long long xb[2], xt[2], xh[2], yb[2], yt[2], yh[2];   // strides in elements: batch, token, head
  int heads[2];
  const void* pos;
  long long pb, pt;                 // strides of the positions
  int pos64;
  const double* freq;               // [R / 2] radians a position
  float factor, sign;
  long long tokens;                 // batch * seq
  long long seq;
  int D, R, tile;                   // tile: tokens a block
  int in_place;                     // the channels from R on are there already
  int near;                         // batches follow one another, and tokens and strides are numbers of 31 bits
  int xt32[2], xh32[2], yt32[2], yh32[2];
  RotDiv by_half, by_heads, by_run; // by_run: pieces of a token
  RotDiv by_items;                  // (items of a head; the heads that a block takes at a time, and whole tokens in them)
  int across, step_t;
  int run;                          // bytes of a piece of a run; 0: heads are no runs
};

// An access as it is moved, and its VE values.
template <int BYTES>
struct RotRaw;
template <>
struct RotRaw<16> { using type = uint4; };
template <>
struct RotRaw<8> { using type = uint2; };
template <>
struct RotRaw<4> { using type = uint32_t; };
template <>
struct RotRaw<2> { using type = unsigned short; };

__device__ __forceinline__ float2 rot_pair(uint32_t w, __nv_bfloat16) { return unpack_bf16x2(w); }
__device__ __forceinline__ float2 rot_pair(uint32_t w, __half) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
__device__ __forceinline__ uint32_t rot_word(float2 v, __nv_bfloat16) { return pack_bf16x2(v.x, v.y); }
__device__ __forceinline__ uint32_t rot_word(float2 v, __half) {
  const __half2 h = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, int VE>
struct RotVec {
  using Raw = typename RotRaw<sizeof(T) * VE>::type;
  Raw raw;
  __device__ __forceinline__ void get(float (&v)[VE]) const {
    if constexpr (sizeof(T) == 4) {
      const float* w = reinterpret_cast<const float*>(&raw);
#pragma unroll
      for (int e = 0; e < VE; ++e) v[e] = w[e];
    } else if constexpr (VE == 1) {
      v[0] = rot_pair(raw, T()).x;
    } else {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
      for (int e = 0; e < VE; e += 2) {
        const float2 p = rot_pair(w[e / 2], T());
        v[e] = p.x;
        v[e + 1] = p.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&v)[VE]) {
    if constexpr (sizeof(T) == 4) {
      float* w = reinterpret_cast<float*>(&raw);
#pragma unroll
      for (int e = 0; e < VE; ++e) w[e] = v[e];
    } else if constexpr (VE == 1) {
      raw = static_cast<unsigned short>(rot_word(make_float2(v[0], 0.f), T()));
    } else {
      uint32_t* w = reinterpret_cast<uint32_t*>(&raw);
#pragma unroll
      for (int e = 0; e < VE; e += 2) w[e / 2] = rot_word(make_float2(v[e], v[e + 1]), T());
    }
  }
};

__device__ __forceinline__ void rot_split(const RotaryArgs& a, long long t, long long& b, long long& s) {
  b = 0;
  s = t;
  if (a.seq != a.tokens) {
    b = a.tokens >> 32 ? t / a.seq : static_cast<uint32_t>(t) / static_cast<uint32_t>(a.seq);
    s = t - b * a.seq;
  }
}

// Where head h of token t is read and written. NEAR: by products of 32 bits where they reach: 55 424 tokens of 12 + 12 heads of 64,
// bf16, both ways 124 -> 122 us, 32 768 of 16 + 4 heads of 128, fp16 119 -> 115; narrow accesses lose by it (100 000 of 10 heads of 37,
// 2 turn: 181 -> 202).
template <typename T, bool NEAR>
__device__ __forceinline__ void rot_head(const RotaryArgs& a, long long t, int h, const T*& from, T*& to) {
  const int k = h >= a.heads[0], hh = h - (k ? a.heads[0] : 0);
  if (NEAR && a.near) {
    const int at = static_cast<int>(t);
    from = static_cast<const T*>(k ? a.x[1] : a.x[0]) + (static_cast<long long>(at) * (k ? a.xt32[1] : a.xt32[0]) +
                                                         static_cast<long long>(hh) * (k ? a.xh32[1] : a.xh32[0]));
    to = static_cast<T*>(k ? a.y[1] : a.y[0]) + (static_cast<long long>(at) * (k ? a.yt32[1] : a.yt32[0]) +
                                                 static_cast<long long>(hh) * (k ? a.yh32[1] : a.yh32[0]));
    return;
  }
  long long b, s;
  rot_split(a, t, b, s);
  from = static_cast<const T*>(a.x[k]) + b * a.xb[k] + s * a.xt[k] + hh * a.xh[k];
  to = static_cast<T*>(a.y[k]) + b * a.yb[k] + s * a.yt[k] + hh * a.yh[k];
}

// The same for a kernel that has registers for the places of a block's first token: `tok` tokens on.
template <typename T>
struct RotPlace {
  const T *x0, *x1;
  T *y0, *y1;
  __device__ __forceinline__ RotPlace(const RotaryArgs& a, long long t0) {
    x0 = static_cast<const T*>(a.x[0]) + t0 * a.xt[0];
    x1 = static_cast<const T*>(a.x[1]) + t0 * a.xt[1];
    y0 = static_cast<T*>(a.y[0]) + t0 * a.yt[0];
    y1 = static_cast<T*>(a.y[1]) + t0 * a.yt[1];
  }
  __device__ __forceinline__ const T* from(const RotaryArgs& a, long long t0, int tok, int h) const {
    const bool k = h >= a.heads[0];
    const int hh = h - (k ? a.heads[0] : 0);
    if (a.near) return (k ? x1 : x0) + (tok * (k ? a.xt32[1] : a.xt32[0]) + hh * (k ? a.xh32[1] : a.xh32[0]));
    const T* from;
    T* to;
    rot_head<T, false>(a, t0 + tok, h, from, to);
    return from;
  }
  __device__ __forceinline__ T* to(const RotaryArgs& a, long long t0, int tok, int h) const {
    const bool k = h >= a.heads[0];
    const int hh = h - (k ? a.heads[0] : 0);
    if (a.near) return (k ? y1 : y0) + (tok * (k ? a.yt32[1] : a.yt32[0]) + hh * (k ? a.yh32[1] : a.yh32[0]));
    const T* from;
    T* to;
    rot_head<T, false>(a, t0 + tok, h, from, to);
    return to;
  }
};

// cos and sin (times factor and sign) of the block's tokens: [tokens][half].
__device__ __forceinline__ void rotary_angles(const RotaryArgs& a, long long t0, int tokens, int half, float* sm_cos, float* sm_sin) {
  for (int j = threadIdx.x; j < tokens * half; j += ROT_THREADS) {
    const int tk = a.by_half.of(j), p2 = j - tk * half;
    long long b, s;
    rot_split(a, t0 + tk, b, s);
    const long long from = b * a.pb + s * a.pt;
    const double p = a.pos64 ? static_cast<double>(static_cast<const long long*>(a.pos)[from])
                             : static_cast<double>(static_cast<const int*>(a.pos)[from]);
    const double turns = p * (a.freq[p2] * 0.15915494309189535);   // 1 / (2 pi)
    const float rest = static_cast<float>(turns - rint(turns));
    float sn, cs;
    sincospif(2.f * rest, &sn, &cs);
    sm_cos[j] = a.factor * cs;
    sm_sin[j] = a.factor * a.sign * sn;
  }
}

// Two accesses' worth of a head, VE pairs, turned by their cos and sin.
template <typename T, int VE, bool INTER>
__device__ __forceinline__ void rot_turn(RotVec<T, VE>& v0, RotVec<T, VE>& v1, const float* cos, const float* sin) {
  float cs[VE], sn[VE];
  if constexpr (VE >= 4) {
#pragma unroll
    for (int e = 0; e < VE; e += 4) {
      const float4 cc = *reinterpret_cast<const float4*>(cos + e);
      const float4 ss = *reinterpret_cast<const float4*>(sin + e);
      cs[e] = cc.x; cs[e + 1] = cc.y; cs[e + 2] = cc.z; cs[e + 3] = cc.w;
      sn[e] = ss.x; sn[e + 1] = ss.y; sn[e + 2] = ss.z; sn[e + 3] = ss.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      cs[e] = cos[e];
      sn[e] = sin[e];
    }
  }
  float x[2 * VE], lo[VE], hi[VE];
  v0.get(lo);
  v1.get(hi);
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    x[e] = lo[e];
    x[VE + e] = hi[e];
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) {      // the two members of pair e of this item
    const int j0 = INTER ? 2 * e : e, j1 = INTER ? 2 * e + 1 : VE + e;
    const float x1 = x[j0], x2 = x[j1];
    x[j0] = x1 * cs[e] - x2 * sn[e];
    x[j1] = x2 * cs[e] + x1 * sn[e];
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    lo[e] = x[e];
    hi[e] = x[VE + e];
  }
  v0.set(lo);
  v1.set(hi);
}

// VE: elements an access, a divisor of R / 2, of D - R and of all strides, with the addresses on its multiples. A thread's
// item is VE pairs of a head (two accesses) or up to 2 VE channels behind the rotated ones. Its place in the head stays the
// same, so that only token and head advance from item to item. Two items of 16 bytes in flight and four blocks a
// multiprocessor, fetched before the cos and sin are formed: 55 424 tokens, 12 + 12 heads of 64, bf16, forward and backward 122 us (5.6
// TB/s, 0.86 of the copy rate; loads behind the cos and sin 255); 32 768 tokens, 16 + 4 heads of 128 of which 32 turn, fp16, 115 us.
template <typename T, int VE, bool INTER>
__global__ void __launch_bounds__(ROT_THREADS, 4)
rotary_kernel(const __grid_constant__ RotaryArgs a) {
  using Vec = RotVec<T, VE>;
  using Raw = typename Vec::Raw;
  constexpr int ROT_UNROLL = rot_unroll(sizeof(T) * VE);
  __shared__ __align__(16) float sm_cos[ROT_PAIRS], sm_sin[ROT_PAIRS];
  grid_chain();
  const int half = a.R >> 1;
  const long long t0 = static_cast<long long>(blockIdx.x) * a.tile;
  const int tokens = static_cast<int>(min(static_cast<long long>(a.tile), a.tokens - t0));
  const int rot = half / VE;                                          // items a head: pairs,
  const int behind = a.in_place ? 0 : (a.D - a.R + 2 * VE - 1) / (2 * VE);   // and what is copied
  const int per_head = rot + behind;
  const int stride = a.across;                                        // heads that the block takes at a time
  const int first = a.by_items.of(threadIdx.x), c = threadIdx.x - first * per_head;
  const int heads = a.heads[0] + a.heads[1];
  const int rows = first < stride ? tokens * heads : 0;
  const int step_t = a.step_t, step_h = stride - step_t * heads;
  int tok = a.by_heads.of(first), h = first - tok * heads, row = first;
  const bool pairs = c < rot;
  // offsets of the two accesses in a head
  const int i = c * VE;
  const int o0 = pairs ? (INTER ? 2 * i : i) : a.R + (c - rot) * 2 * VE;
  const int o1 = pairs ? (INTER ? 2 * i + VE : i + half) : o0 + VE;
  const bool second = o1 < a.D;

  Vec v0[ROT_UNROLL], v1[ROT_UNROLL];
  T* to[ROT_UNROLL];
  int at[ROT_UNROLL];
  auto load = [&]() {
#pragma unroll
    for (int u = 0; u < ROT_UNROLL; ++u) {
      to[u] = nullptr;
      if (row < rows) {
        constexpr bool NEAR = sizeof(T) * VE >= 16;
        const T* from;
        rot_head<T, NEAR>(a, t0 + tok, h, from, to[u]);
        at[u] = tok * half + i;
        v0[u].raw = *reinterpret_cast<const Raw*>(from + o0);
        if (second) v1[u].raw = *reinterpret_cast<const Raw*>(from + o1);
        tok += step_t;
        h += step_h;
        if (h >= heads) {
          h -= heads;
          ++tok;
        }
      }
      row += stride;
    }
  };
  load();     // on its way while cos and sin are formed
  rotary_angles(a, t0, tokens, half, sm_cos, sm_sin);
  __syncthreads();
  while (true) {
#pragma unroll
    for (int u = 0; u < ROT_UNROLL; ++u) {
      if (to[u] != nullptr) {
        if (pairs) {
          rot_turn<T, VE, INTER>(v0[u], v1[u], sm_cos + at[u], sm_sin + at[u]);
        }
        *reinterpret_cast<Raw*>(to[u] + o0) = v0[u].raw;
        if (second) *reinterpret_cast<Raw*>(to[u] + o1) = v1[u].raw;
      }
    }
    if (row >= rows) break;
    load();
  }
}

// The same for pairs that lie on no 16 bytes: values move through shared memory in pieces as wide as they can be, and the pairs are
// turned there. Narrow accesses to global memory leave too little in flight and cost addresses (32 bits here where they reach).
// Heads on 16 bytes are taken one by one (100 000 tokens x 8 of 64, 50 turn: 106 us, as runs 112); others where they lie side by
// side, as one run of a token. Forward and backward in us, narrow accesses / staged (floor):
//   bf16, 100 000 tokens x 8 heads of 64, 50 turn            264 / 107 (64)      30 000 x 16 of 80, 40 turn (8 bytes)   141 / 107 (95)
//   bf16, 30 000 x 16 of 128, 30 turn, interleaved           289 / 84 (76)       fp32, 30 000 x 16 of 96, 36 turn       178 / 119 (114)
//   bf16, 100 000 x 8 of 75, 50 turn, runs in 8 bytes        338 / 150 (74)      fp32, 50 000 x 16 of 33, 20 turn       160 / 86 (65)
// With 16 bytes it does not pay: bf16, 60 000 x 16 of 96, all turn 142 / 153.
// Shared memory: [tokens][heads][D] values, then cos and sin.
template <int BYTES>
__device__ __forceinline__ void rot_piece_in(void* to, const char* from) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(to)), "l"(from), "n"(BYTES) : "memory");
}

// The runs of the block's tokens between memory and shared memory, in pieces of BYTES.
template <typename T, int BYTES, bool OUT>
__device__ __forceinline__ void rot_runs(const RotaryArgs& a, const RotPlace<T>& place, long long t0, int tokens, int heads, char* values) {
  const int pieces = heads * a.D * static_cast<int>(sizeof(T)) / BYTES, of_q = a.heads[0] * a.D * static_cast<int>(sizeof(T)) / BYTES;
#pragma unroll 4
  for (int j = threadIdx.x; j < tokens * pieces; j += ROT_THREADS) {
    const int tok = a.by_run.of(j), piece = j - tok * pieces;
    const bool k = piece >= of_q;
    const int h = k ? a.heads[0] : 0, at = (piece - (k ? of_q : 0)) * BYTES;
    if constexpr (OUT) {
      using Raw = typename RotRaw<BYTES>::type;
      *reinterpret_cast<Raw*>(reinterpret_cast<char*>(place.to(a, t0, tok, h)) + at) = *reinterpret_cast<const Raw*>(values + j * BYTES);
    } else {
      rot_piece_in<BYTES>(values + j * BYTES, reinterpret_cast<const char*>(place.from(a, t0, tok, h)) + at);
    }
  }
}
template <typename T, bool OUT>
__device__ __forceinline__ void rot_runs(const RotaryArgs& a, const RotPlace<T>& place, long long t0, int tokens, int heads, void* values) {
  char* v = static_cast<char*>(values);
  if (a.run == 16) rot_runs<T, 16, OUT>(a, place, t0, tokens, heads, v);
  else if (a.run == 8) rot_runs<T, 8, OUT>(a, place, t0, tokens, heads, v);
  else rot_runs<T, 4, OUT>(a, place, t0, tokens, heads, v);
}

template <typename T, int VE, bool INTER, bool RUNS>
__global__ void __launch_bounds__(ROT_THREADS, 4)
rotary_staged_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ __align__(16) uint8_t rot_smem[];
  grid_chain();
  const int half = a.R >> 1, heads = a.heads[0] + a.heads[1];
  const long long t0 = static_cast<long long>(blockIdx.x) * a.tile;
  const int tokens = static_cast<int>(min(static_cast<long long>(a.tile), a.tokens - t0));
  const int rows = tokens * heads, pieces = RUNS ? 1 : a.D * static_cast<int>(sizeof(T)) / 16;
  T* values = reinterpret_cast<T*>(rot_smem);
  float* sm_cos = reinterpret_cast<float*>(rot_smem + ((static_cast<size_t>(a.tile) * heads * a.D * sizeof(T) + 15) & ~size_t(15)));
  float* sm_sin = sm_cos + a.tile * half;
  const int stride = ROT_THREADS / pieces, first = threadIdx.x / pieces, piece = threadIdx.x - first * pieces;
  const RotPlace<T> place(a, t0);
  if constexpr (RUNS) {
    rot_runs<T, false>(a, place, t0, tokens, heads, values);
  } else if (first < stride) {
    for (int row = first; row < rows; row += stride) {
      const int tok = a.by_heads.of(row);
      const T* from = place.from(a, t0, tok, row - tok * heads);
      rot_piece_in<16>(reinterpret_cast<char*>(values + row * a.D) + piece * 16, reinterpret_cast<const char*>(from) + piece * 16);
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  rotary_angles(a, t0, tokens, half, sm_cos, sm_sin);
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  // a thread turns the same VE pairs of every so many-th head
  const int items = half / VE, across = ROT_THREADS / items, from = threadIdx.x / items, i = (threadIdx.x - from * items) * VE;
  if (from < across) {
    for (int row = from; row < rows; row += across) {
      const int at = a.by_heads.of(row) * half + i;
      T* p0 = values + row * a.D + (INTER ? 2 * i : i);
      T* p1 = p0 + (INTER ? VE : half);
      RotVec<T, VE> v0, v1;
      v0.raw = *reinterpret_cast<const typename RotVec<T, VE>::Raw*>(p0);
      v1.raw = *reinterpret_cast<const typename RotVec<T, VE>::Raw*>(p1);
      rot_turn<T, VE, INTER>(v0, v1, sm_cos + at, sm_sin + at);
      *reinterpret_cast<typename RotVec<T, VE>::Raw*>(p0) = v0.raw;
      *reinterpret_cast<typename RotVec<T, VE>::Raw*>(p1) = v1.raw;
    }
  }
  __syncthreads();
  if constexpr (RUNS) {
    rot_runs<T, true>(a, place, t0, tokens, heads, values);
  } else if (first < stride) {
    for (int row = first; row < rows; row += stride) {
      const int tok = a.by_heads.of(row);
      T* to = place.to(a, t0, tok, row - tok * heads);
      *reinterpret_cast<uint4*>(reinterpret_cast<char*>(to) + piece * 16) =
          *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(values + row * a.D) + piece * 16);
    }
  }
}

template <typename T, int VE, bool INTER>
static cudaError_t launch_staged(const RotaryArgs& a, unsigned blocks, size_t smem, cudaStream_t st) {
  const bool chained = a.tokens * (a.heads[0] + a.heads[1]) * a.D <= CHAIN_ELEMENTS;
  return a.run ? launch_when(chained, rotary_staged_kernel<T, VE, INTER, true>, blocks, ROT_THREADS, smem, st, a)
               : launch_when(chained, rotary_staged_kernel<T, VE, INTER, false>, blocks, ROT_THREADS, smem, st, a);
}

template <typename T, int VE>
static cudaError_t launch_staged(const RotaryArgs& a, int interleaved, unsigned blocks, size_t smem, cudaStream_t st) {
  return interleaved ? launch_staged<T, VE, true>(a, blocks, smem, st) : launch_staged<T, VE, false>(a, blocks, smem, st);
}

// (in accesses of 4 or 2 where pairs and heads are multiples of that)
template <typename T>
static cudaError_t launch_staged(const RotaryArgs& a, int interleaved, unsigned blocks, size_t smem, cudaStream_t st) {
  const int half = a.R / 2;
  if (half % 4 == 0 && a.D % 4 == 0) return launch_staged<T, 4>(a, interleaved, blocks, smem, st);
  if (half % 2 == 0 && a.D % 2 == 0) return launch_staged<T, 2>(a, interleaved, blocks, smem, st);
  return launch_staged<T, 1>(a, interleaved, blocks, smem, st);
}

template <typename T, int VE>
static cudaError_t launch_rotary(const RotaryArgs& a, int interleaved, unsigned blocks, cudaStream_t st) {
  const long long n = a.tokens * (a.heads[0] + a.heads[1]) * a.D;
  return interleaved ? launch_when(n <= CHAIN_ELEMENTS, rotary_kernel<T, VE, true>, blocks, ROT_THREADS, 0, st, a)
                     : launch_when(n <= CHAIN_ELEMENTS, rotary_kernel<T, VE, false>, blocks, ROT_THREADS, 0, st, a);
}

template <typename T>
static cudaError_t launch_rotary(const RotaryArgs& a, int ve, int interleaved, unsigned blocks, cudaStream_t st) {
  if (ve * sizeof(T) >= 16) return launch_rotary<T, 16 / sizeof(T)>(a, interleaved, blocks, st);
  if (ve >= 4) return launch_rotary<T, 4>(a, interleaved, blocks, st);
  if (ve >= 2) return launch_rotary<T, 2>(a, interleaved, blocks, st);
  return launch_rotary<T, 1>(a, interleaved, blocks, st);
}

}  // namespace nplm

using namespace nplm;

// The arguments of a call, packed by the caller (ops/kernels.py has the same layout): one conversion on its side, not 20.
// strides: batch, token and head of q, then of its output, then the same of k. k may be null (k_heads 0). pos: int32 or int64
// (pos64), strides pb, pt. D at most 512. dtype: 0 bf16, 1 fp16, 2 fp32.
struct RotaryCall {
  const void* q;
  void* q_out;
  const void* k;
  void* k_out;
  long long strides[12];
  const void* pos;
  long long pb, pt;
  const double* freq;
  long long batch, seq;
  int q_heads, k_heads, pos64, transposed, D, R, dtype, interleaved;
  float factor;
};

extern "C" int nplm_rotary_qk(const RotaryCall* call, cudaStream_t st) {
  const RotaryCall& c = *call;
  const int q_heads = c.q_heads, k_heads = c.k_heads, D = c.D, R = c.R, dtype = c.dtype;
  const long long batch = c.batch, seq = c.seq;
  if (batch < 0 || seq < 0 || q_heads < 1 || k_heads < 0 || q_heads > 65536 || k_heads > 65536 || D < 2 || D > 512 || R < 2 ||
      R > D || R % 2 || dtype < 0 || dtype > 2)
    return -1;
  if (batch == 0 || seq == 0) return 0;
  RotaryArgs a;
  a.x[0] = c.q; a.x[1] = c.k; a.y[0] = c.q_out; a.y[1] = c.k_out;
  a.heads[0] = q_heads; a.heads[1] = k_heads;
  for (int j = 0; j < 2; ++j) {
    const long long* strides = c.strides + 6 * j;
    a.xb[j] = strides[0]; a.xt[j] = strides[1]; a.xh[j] = strides[2];
    a.yb[j] = strides[3]; a.yt[j] = strides[4]; a.yh[j] = strides[5];
  }
  a.pos = c.pos; a.pos64 = c.pos64; a.pb = c.pb; a.pt = c.pt; a.freq = c.freq; a.factor = c.factor;
  a.sign = c.transposed ? -1.f : 1.f;
  a.tokens = batch * seq; a.seq = seq; a.D = D; a.R = R;
  a.in_place = 1;
  for (int j = 0; j < (k_heads ? 2 : 1); ++j)
    a.in_place &= a.x[j] == a.y[j] && a.xb[j] == a.yb[j] && a.xt[j] == a.yt[j] && a.xh[j] == a.yh[j];
  // the widest access, up to 16 bytes, that sizes, strides and addresses allow
  const int size = dtype == 2 ? 4 : 2;
  int ve = 16 / size;
  auto fits = [&](int v) {
    if ((R / 2) % v || (D - R) % v) return false;
    for (int j = 0; j < (k_heads ? 2 : 1); ++j) {
      const long long all = a.xb[j] | a.xt[j] | a.xh[j] | a.yb[j] | a.yt[j] | a.yh[j];
      if (all % v || reinterpret_cast<uintptr_t>(a.x[j]) % (v * size) || reinterpret_cast<uintptr_t>(a.y[j]) % (v * size))
        return false;
    }
    return true;
  };
  while (ve > 1 && !fits(ve)) ve /= 2;
  const int half = R / 2, heads = q_heads + k_heads;
  // for narrow pairs: heads on 16 bytes, or heads side by side in pieces of 16, 8 or 4 bytes (of 2: bf16, 100 000 tokens x 10 heads of
  // 37, 2 turn 340 us, by narrow accesses 181)
  bool whole = D * size % 16 == 0;
  int run = 16;
  for (int j = 0; j < (k_heads ? 2 : 1); ++j) {
    const long long tokens_at = a.xb[j] | a.xt[j] | a.yb[j] | a.yt[j], all = tokens_at | a.xh[j] | a.yh[j];
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.x[j]) | reinterpret_cast<uintptr_t>(a.y[j]);
    whole &= all * size % 16 == 0 && at % 16 == 0;
    if (a.heads[j] > 1 && (a.xh[j] != D || a.yh[j] != D)) run = 0;
    while (run && (tokens_at * size % run || at % run || static_cast<long long>(a.heads[j]) * D * size % run)) run /= 2;
  }
  if (whole || run < 4) run = 0;
  a.by_half = RotDiv(half);
  a.by_heads = RotDiv(heads);
  a.near = a.tokens <= 0x7fffffffLL;
  for (int j = 0; j < (k_heads ? 2 : 1); ++j) {
    const long long reach = a.xt[j] | a.yt[j] | a.xh[j] | a.yh[j];
    a.near &= reach <= 0x7fffffffLL && (batch == 1 || (a.xb[j] == seq * a.xt[j] && a.yb[j] == seq * a.yt[j]));
    a.xt32[j] = static_cast<int>(a.xt[j]); a.xh32[j] = static_cast<int>(a.xh[j]);
    a.yt32[j] = static_cast<int>(a.yt[j]); a.yh32[j] = static_cast<int>(a.yh[j]);
  }
  const long long token_bytes = static_cast<long long>(heads) * D * size + 2 * half * 4;       // values, cos and sin
  if (ve * size <= 8 && (whole || run) && token_bytes <= ROT_STAGED) {
    a.run = run;
    if (run) a.by_run = RotDiv(static_cast<uint32_t>(heads * D * size / run));
    // (few tokens: four blocks a multiprocessor; 4 301 x 8 heads of 70, 34 turn, fp32 19 us with one, 14 with four)
    const long long even = (a.tokens + 591) / 592;
    a.tile = static_cast<int>(ROT_STAGED / token_bytes);
    if (a.tile > even) a.tile = static_cast<int>(even);
    for (int j = 0; j < (k_heads ? 2 : 1); ++j)      // (a tile's offsets are of 31 bits)
      a.near &= std::max(a.xt[j], a.yt[j]) * a.tile + std::max(a.xh[j], a.yh[j]) * a.heads[j] <= 0x7fffffffLL;
    const long long blocks = (a.tokens + a.tile - 1) / a.tile;
    if (blocks > 0x7fffffffLL) return -2;
    const size_t smem = static_cast<size_t>(a.tile) * token_bytes + 16;      // (cos and sin start on 16 bytes)
    const unsigned n = static_cast<unsigned>(blocks);
    const cudaError_t e = dtype == 0   ? launch_staged<__nv_bfloat16>(a, c.interleaved, n, smem, st)
                          : dtype == 1 ? launch_staged<__half>(a, c.interleaved, n, smem, st)
                                       : launch_staged<float>(a, c.interleaved, n, smem, st);
    return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
  }
  const int per_token = heads * (half / ve + (a.in_place ? 0 : (D - R + 2 * ve - 1) / (2 * ve)));
  // as many tokens as the unrolled items of all threads, at least one, as long as their cos and sin fit
  const int per_head = per_token / heads;
  int tile = ROT_THREADS / per_head * rot_unroll(ve * size) / heads;
  if (tile > ROT_PAIRS / half) tile = ROT_PAIRS / half;
  if (tile < 1) tile = 1;
  a.tile = tile;
  a.by_items = RotDiv(per_head);
  a.across = ROT_THREADS / per_head;
  a.step_t = a.across / heads;
  const long long blocks = (a.tokens + tile - 1) / tile;
  if (blocks > 0x7fffffffLL) return -2;
  const unsigned n = static_cast<unsigned>(blocks);
  cudaError_t e;
  if (dtype == 0) e = launch_rotary<__nv_bfloat16>(a, ve, c.interleaved, n, st);
  else if (dtype == 1) e = launch_rotary<__half>(a, ve, c.interleaved, n, st);
  else e = launch_rotary<float>(a, ve, c.interleaved, n, st);
  if (e != cudaSuccess) return static_cast<int>(e);
  return static_cast<int>(cudaGetLastError());
}
