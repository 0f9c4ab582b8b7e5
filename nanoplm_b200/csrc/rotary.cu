// Rotary positions of queries and keys in one launch: half (i, i + R/2) or interleaved (2i, 2i + 1) pairs, the first R of a
// head's D channels, any number of query and key heads, any token, head and batch strides.
//
// For pair i of a token at position p, with a = p w_i, and the factor f of the frequency scaling:
//   y1 = f (x1 cos a - x2 sin a),  y2 = f (x2 cos a + x1 sin a);  the gradient is the transpose, sin negated.
//
// Bound by memory: a pair costs 4 multiplications, and its cos and sin serve all heads of the token. So a block takes a few
// tokens, forms their cos and sin once in shared memory and then streams the heads. No table: a table in fp32 ends at a
// largest position, and fp32 angles are off by p 2^-24 radians. Here p w_i is formed in fp64 as a number of turns, whose
// whole part is dropped before the rest becomes a fp32 argument in [-1, 1] half turns of sincospi, good to fp32's last
// bits for every position that a 32-bit integer holds.
#include <cuda_fp16.h>

#include "common.cuh"

namespace nplm {

constexpr int ROT_THREADS = 256;
constexpr int ROT_STAGED = 32 * 1024;   // shared memory of a block that turns pairs there
constexpr int ROT_PAIRS = 2048;     // cos and sin of a block's tokens: 16 KB
// Items that a thread has in flight.
__host__ __device__ constexpr int rot_unroll(int bytes) { return bytes >= 16 ? 2 : 4; }

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

// cos and sin (times factor and sign) of the block's tokens: [tokens][half].
__device__ __forceinline__ void rotary_angles(const RotaryArgs& a, long long t0, int tokens, int half, float* sm_cos, float* sm_sin) {
  for (int j = threadIdx.x; j < tokens * half; j += ROT_THREADS) {
    const int tk = j / half, p2 = j - tk * half;
    const long long t = t0 + tk;
    long long b = 0, s = t;
    if (a.seq != a.tokens) {
      b = t / a.seq;
      s = t - b * a.seq;
    }
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

// VE: elements an access, a divisor of R / 2, of D - R and of all strides, with the addresses on its multiples. A thread's
// item is VE pairs of a head (two accesses) or up to 2 VE channels behind the rotated ones. Its place in the head stays the
// same, so that only token and head advance from item to item. Two items of 16 bytes in flight and four blocks a
// multiprocessor, fetched before the cos and sin are formed: 55 424 tokens, 12 + 12 heads of 64, bf16, forward and backward 124 us (5.5
// TB/s, 0.85 of the copy rate; loads behind the cos and sin 255); 32 768 tokens, 16 + 4 heads of 128 of which 32 turn, fp16, 119 us.
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
  const int stride = ROT_THREADS / per_head;                          // heads that the block takes at a time
  const int first = threadIdx.x / per_head, c = threadIdx.x - first * per_head;
  const int heads = a.heads[0] + a.heads[1];
  const int rows = first < stride ? tokens * heads : 0;
  const int step_t = stride / heads, step_h = stride - step_t * heads;
  int tok = first / heads, h = first - tok * heads, row = first;
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
        const int k = h >= a.heads[0];
        const int hh = h - (k ? a.heads[0] : 0);
        const long long t = t0 + tok;
        long long b = 0, s = t;
        if (a.seq != a.tokens) {
          b = t / a.seq;
          s = t - b * a.seq;
        }
        const T* from = static_cast<const T*>(a.x[k]) + b * a.xb[k] + s * a.xt[k] + hh * a.xh[k];
        to[u] = static_cast<T*>(a.y[k]) + b * a.yb[k] + s * a.yt[k] + hh * a.yh[k];
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
          float cs[VE], sn[VE];
          if constexpr (VE >= 4) {
#pragma unroll
            for (int e = 0; e < VE; e += 4) {
              const float4 cc = *reinterpret_cast<const float4*>(sm_cos + at[u] + e);
              const float4 ss = *reinterpret_cast<const float4*>(sm_sin + at[u] + e);
              cs[e] = cc.x; cs[e + 1] = cc.y; cs[e + 2] = cc.z; cs[e + 3] = cc.w;
              sn[e] = ss.x; sn[e + 1] = ss.y; sn[e + 2] = ss.z; sn[e + 3] = ss.w;
            }
          } else {
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              cs[e] = sm_cos[at[u] + e];
              sn[e] = sm_sin[at[u] + e];
            }
          }
          float x[2 * VE], lo[VE], hi[VE];
          v0[u].get(lo);
          v1[u].get(hi);
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
          v0[u].set(lo);
          v1[u].set(hi);
        }
        *reinterpret_cast<Raw*>(to[u] + o0) = v0[u].raw;
        if (second) *reinterpret_cast<Raw*>(to[u] + o1) = v1[u].raw;
      }
    }
    if (row >= rows) break;
    load();
  }
}

// The same for pairs that lie on no 16 bytes while whole heads do: a head moves in pieces of 16 bytes through shared memory, and
// the pairs are turned there. Accesses of 2 or 4 bytes to global memory leave too little in flight. Forward and backward in us, so /
// staged: bf16, 100 000 tokens x 8 heads of 64, 50 turn 264 / 171 (floor 64); 30 000 x 16 of 128, 30 turn, interleaved 289 / 125 (76);
// fp32, 30 000 x 16 of 80, 42 turn 247 / 153 (95). With accesses of 8 bytes it does not pay: bf16, 60 000 x 16 of 80, 40 turn 147 / 199.
// Shared memory: [rows][D] values, then cos and sin.
template <typename T, bool INTER>
__global__ void __launch_bounds__(ROT_THREADS, 4)
rotary_staged_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ __align__(16) uint8_t rot_smem[];
  grid_chain();
  const int half = a.R >> 1, heads = a.heads[0] + a.heads[1];
  const long long t0 = static_cast<long long>(blockIdx.x) * a.tile;
  const int tokens = static_cast<int>(min(static_cast<long long>(a.tile), a.tokens - t0));
  const int rows = tokens * heads, pieces = a.D * static_cast<int>(sizeof(T)) / 16;
  T* values = reinterpret_cast<T*>(rot_smem);
  float* sm_cos = reinterpret_cast<float*>(rot_smem + static_cast<size_t>(a.tile) * heads * a.D * sizeof(T));
  float* sm_sin = sm_cos + a.tile * half;
  const int stride = ROT_THREADS / pieces, first = threadIdx.x / pieces, piece = threadIdx.x - first * pieces;
  auto place = [&](int row, const long long (&sb)[2], const long long (&st)[2], const long long (&sh)[2], const void* const* base) {
    const int tok = row / heads, h = row - tok * heads, k = h >= a.heads[0];
    const long long t = t0 + tok;
    long long b = 0, s = t;
    if (a.seq != a.tokens) {
      b = t / a.seq;
      s = t - b * a.seq;
    }
    return static_cast<const T*>(base[k]) + b * sb[k] + s * st[k] + (h - (k ? a.heads[0] : 0)) * sh[k];
  };
  if (first < stride) {
    for (int row = first; row < rows; row += stride) {
      const T* from = place(row, a.xb, a.xt, a.xh, a.x);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(values + row * a.D) + piece * 16),
                   "l"(reinterpret_cast<const char*>(from) + piece * 16)
                   : "memory");
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  rotary_angles(a, t0, tokens, half, sm_cos, sm_sin);
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  // all pairs of all rows: pair after pair of a row, row after row
  for (int j = threadIdx.x; j < rows * half; j += ROT_THREADS) {
    const int row = j / half, i = j - row * half, at = row / heads * half + i;
    T* x = values + row * a.D;
    const int j0 = INTER ? 2 * i : i, j1 = INTER ? 2 * i + 1 : i + half;
    const float x1 = static_cast<float>(x[j0]), x2 = static_cast<float>(x[j1]), co = sm_cos[at], sn = sm_sin[at];
    x[j0] = static_cast<T>(x1 * co - x2 * sn);      // (to the nearest)
    x[j1] = static_cast<T>(x2 * co + x1 * sn);
  }
  __syncthreads();
  if (first < stride) {
    for (int row = first; row < rows; row += stride) {
      T* to = const_cast<T*>(place(row, a.yb, a.yt, a.yh, a.y));
      *reinterpret_cast<uint4*>(reinterpret_cast<char*>(to) + piece * 16) =
          *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(values + row * a.D) + piece * 16);
    }
  }
}

template <typename T>
static cudaError_t launch_staged(const RotaryArgs& a, int interleaved, unsigned blocks, size_t smem, cudaStream_t st) {
  const bool chained = a.tokens * (a.heads[0] + a.heads[1]) * a.D <= CHAIN_ELEMENTS;
  return interleaved ? launch_when(chained, rotary_staged_kernel<T, true>, blocks, ROT_THREADS, smem, st, a)
                     : launch_when(chained, rotary_staged_kernel<T, false>, blocks, ROT_THREADS, smem, st, a);
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
  if (batch < 0 || seq < 0 || q_heads < 1 || k_heads < 0 || q_heads > 65536 || k_heads > 65536 || D < 2 || D > 512 || R < 2 || R > D || R % 2 || dtype < 0 ||
      dtype > 2)
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
  bool whole = D * size % 16 == 0;       // heads on 16 bytes
  for (int j = 0; j < (k_heads ? 2 : 1); ++j) {
    const long long all = a.xb[j] | a.xt[j] | a.xh[j] | a.yb[j] | a.yt[j] | a.yh[j];
    whole &= all * size % 16 == 0 && reinterpret_cast<uintptr_t>(a.x[j]) % 16 == 0 && reinterpret_cast<uintptr_t>(a.y[j]) % 16 == 0;
  }
  const long long token_bytes = static_cast<long long>(heads) * D * size + 2 * half * 4;       // values, cos and sin
  if (ve * size <= 4 && whole && token_bytes <= ROT_STAGED) {
    const long long even = (a.tokens + 147) / 148;      // (few tokens: over all multiprocessors)
    a.tile = static_cast<int>(ROT_STAGED / token_bytes);
    if (a.tile > even) a.tile = static_cast<int>(even);
    const long long blocks = (a.tokens + a.tile - 1) / a.tile;
    if (blocks > 0x7fffffffLL) return -2;
    const size_t smem = static_cast<size_t>(a.tile) * token_bytes;
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
