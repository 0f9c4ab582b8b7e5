// The end of a residual block in one operator: norm of the block's output, gate, residual scale, sum, and the norm with which
// the next block starts. For a row (token) with block input x and block output f, channels c:
//   n = w_post u(f),   y = r x + g n,   h = w_next u(y),    u(v) = (v - mean v) / sqrt(var v + eps)   (RMSNorm: mean 0)
// with the gate g = 1, a weight per channel, or a value per token and channel, as it is or through a sigmoid.
// Backward, from dy and dh (B_v d = (d - mean d - u(v) mean(d u(v))) / sqrt(var v + eps), the gradient of u):
//   t = dy + B_y(w_next dh),   dx = r t,   df = B_f(w_post g t),   dg = t n,
//   dw_next = sum u(y) dh,   dw_post = sum u(f) g t,   dr = sum t x,   and dg summed where the gate is a weight.
//
// Bound by memory: forward reads x, f (and g) and writes y, h; backward reads dy, dh, x, f (g) and writes dx, df (dg). Op by
// op the row travels three times as often. A row belongs to a group of threads, eight channels a thread, so that the channels
// of a thread never change: the four column sums of the backward pass stay in its registers (in a warp-a-row layout they are
// 4 C / 32 registers a lane, which ends at 512 channels) and leave once a block, as partial sums that a second small kernel
// adds in a fixed order: the same bits every run. Statistics, sums and the residual sum are fp32; y and h are rounded
// once, and h is formed from the unrounded y, which the backward pass forms again from x and f.
#include <cuda_fp16.h>

#include "common.cuh"

namespace nplm {

constexpr int SW_STAGES = 2;        // rows that a group has on their way
constexpr int SW_MAX_C = 4096;

enum : int { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_TOKEN = 2, GATE_SIGMOID = 3 };

struct SandwichArgs {
  const void *x, *f, *gate, *dy, *dh;                 // rows of C, `*s` elements apart
  long long xs, fs, gs, dys, dhs;
  const void *post, *next, *scale;                    // [C] each; post, next null: 1; scale null: 1
  void *y, *h;                                        // forward outputs, contiguous rows; h may be null
  void *dx, *df, *dg;                                 // backward outputs, contiguous rows; dg only for gates of tokens
  float* stats;                                       // [4][T]: mean f, 1 / std f, mean y, 1 / std y; null: not kept
  float* partial;                                     // [4][blocks][C]: dw_next, dw_post, dr, dg
  long long T;
  int C, tpr, groups;                                 // threads a row, rows that a block works on at a time
  float eps;
  int rms, gate_mode, param32;                        // param32: the [C] weights are fp32, else of the rows' type
  int want;                                           // bit k: column sum k is wanted
};

template <typename T>
struct Io;
template <>
struct Io<float> {
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Io<__nv_bfloat16> {
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Io<__half> {
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};

__device__ __forceinline__ void sw_cp_async_16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void sw_cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void sw_cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Eight values of a type, as they lie in memory.
template <typename T>
struct alignas(16) Eight {
  T v[8];
};

// What a thread knows of its place: its group's row slots, its eight channels.
template <typename T, bool ALIGNED>
struct Place {
  int lane, group, tpr, C;
  __device__ __forceinline__ int channel(int e) const { return ALIGNED ? lane * 8 + e : e * tpr + lane; }
  __device__ __forceinline__ bool on(int e) const { return channel(ALIGNED ? 0 : e) < C; }
  // the slot of a [C] table in shared memory: two halves of four channels a thread, so that a warp's 16-byte reads are
  // consecutive
  __device__ __forceinline__ int slot(int e) const { return (e >> 2) * tpr * 4 + lane * 4 + (e & 3); }
  __device__ __forceinline__ void load(const T* row, float (&v)[8]) const {
    if (ALIGNED) {
      if (on(0)) {
        const Eight<T> p = *reinterpret_cast<const Eight<T>*>(row + lane * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = Io<T>::get(p.v[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = on(e) ? Io<T>::get(row[e * tpr + lane]) : 0.f;
    }
  }
  __device__ __forceinline__ void store(T* row, const float (&v)[8]) const {
    if (ALIGNED) {
      if (on(0)) {
        Eight<T> p;
#pragma unroll
        for (int e = 0; e < 8; ++e) p.v[e] = Io<T>::put(v[e]);
        *reinterpret_cast<Eight<T>*>(row + lane * 8) = p;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (on(e)) row[e * tpr + lane] = Io<T>::put(v[e]);
    }
  }
  __device__ __forceinline__ void table(const float* t, float (&v)[8]) const {
    const float4 a = *reinterpret_cast<const float4*>(t + lane * 4);
    const float4 b = *reinterpret_cast<const float4*>(t + tpr * 4 + lane * 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
};

// Sums over the threads of a group, in every one of them and in the same order. slots: [2][16] pairs of the group; the barrier
// of one sum keeps the slots of the one before it from being overwritten too early, so two sets are enough.
struct GroupSum {
  float2* slots;
  int warps, warp, bar, threads, phase;
  __device__ __forceinline__ void two(float& a, float& b) {
    a = warp_sum(a);
    b = warp_sum(b);
    if (warps == 1) return;
    float2* s = slots + phase * 16;
    phase ^= 1;
    if ((threadIdx.x & 31) == 0) s[warp] = make_float2(a, b);
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(threads) : "memory");
    a = b = 0.f;
    for (int w = 0; w < warps; ++w) {
      const float2 v = s[w];
      a += v.x;
      b += v.y;
    }
  }
  __device__ __forceinline__ float one(float a) {
    float b = 0.f;
    a = warp_sum(a);
    if (warps == 1) return a;
    float2* s = slots + phase * 16;
    phase ^= 1;
    if ((threadIdx.x & 31) == 0) s[warp] = make_float2(a, 0.f);
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(threads) : "memory");
    for (int w = 0; w < warps; ++w) b += s[w].x;
    return b;
  }
};

template <typename T>
__device__ __forceinline__ float sw_param(const void* p, int c, int param32) {
  if (p == nullptr) return 1.f;
  return param32 ? static_cast<const float*>(p)[c] : Io<T>::get(static_cast<const T*>(p)[c]);
}

// Shared memory: tables post, next, scale, gate [4][tpr * 8] fp32 | sums [groups][2][16] float2 | ring [groups][stages][parts][C]
template <typename T, bool ALIGNED>
__device__ __forceinline__ void sw_tables(const SandwichArgs& a, const Place<T, ALIGNED>& at, float* tables) {
  if (at.group == 0) {
    const int wide = a.tpr * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = at.channel(e);
      const bool on = c < a.C;
      const int s = at.slot(e);
      tables[s] = on ? sw_param<T>(a.post, c, a.param32) : 0.f;
      tables[wide + s] = on ? sw_param<T>(a.next, c, a.param32) : 0.f;
      tables[2 * wide + s] = on ? sw_param<T>(a.scale, c, a.param32) : 0.f;
      tables[3 * wide + s] = !on ? 0.f : a.gate_mode == GATE_CHANNEL ? sw_param<T>(a.gate, c, a.param32) : 1.f;
    }
  }
  __syncthreads();
}

__device__ __forceinline__ float sw_sigmoid(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(512, 2)
sandwich_fwd_kernel(const __grid_constant__ SandwichArgs a) {
  extern __shared__ __align__(128) uint8_t sw_smem[];
  const int group = threadIdx.x / a.tpr;
  const Place<T, ALIGNED> at{static_cast<int>(threadIdx.x) - group * a.tpr, group, a.tpr, a.C};
  float* tables = reinterpret_cast<float*>(sw_smem);
  const int wide = a.tpr * 8;
  float2* sums = reinterpret_cast<float2*>(tables + 4 * wide);
  uint8_t* ring = reinterpret_cast<uint8_t*>(sums + a.groups * 32);
  GroupSum sum{sums + group * 32, a.tpr >> 5, at.lane >> 5, 1 + group, a.tpr, 0};
  const bool token_gate = a.gate_mode >= GATE_TOKEN;
  const int parts = token_gate ? 3 : 2;
  const size_t row_bytes = static_cast<size_t>(a.C) * sizeof(T);
  ring += static_cast<size_t>(group) * SW_STAGES * parts * row_bytes;
  grid_chain();
  const long long row0 = static_cast<long long>(blockIdx.x) * a.groups + group;
  const long long stride = static_cast<long long>(gridDim.x) * a.groups;
  const T *x = static_cast<const T*>(a.x), *f = static_cast<const T*>(a.f), *gate = static_cast<const T*>(a.gate);
  auto fetch = [&](long long row, int stage) {
    if (ALIGNED) {
      if (row < a.T && at.on(0)) {
        uint8_t* d = ring + static_cast<size_t>(stage) * parts * row_bytes + at.lane * sizeof(Eight<T>);
#pragma unroll
        for (int j = 0; j < static_cast<int>(sizeof(Eight<T>)); j += 16) {
          sw_cp_async_16(d + j, reinterpret_cast<const uint8_t*>(x + row * a.xs + at.lane * 8) + j);
          sw_cp_async_16(d + row_bytes + j, reinterpret_cast<const uint8_t*>(f + row * a.fs + at.lane * 8) + j);
          if (token_gate)
            sw_cp_async_16(d + 2 * row_bytes + j, reinterpret_cast<const uint8_t*>(gate + row * a.gs + at.lane * 8) + j);
        }
      }
      sw_cp_commit();
    }
  };
#pragma unroll
  for (int i = 0; i < SW_STAGES; ++i) fetch(row0 + i * stride, i);
  sw_tables<T, ALIGNED>(a, at, tables);
  const float inv_c = 1.f / a.C;
  int stage = 0;
  for (long long row = row0; row < a.T; row += stride) {
    float v[8], xv[8], w[8];
    const T *px, *pf, *pg;
    if (ALIGNED) {
      sw_cp_wait<SW_STAGES - 1>();
      const uint8_t* s = ring + static_cast<size_t>(stage) * parts * row_bytes;
      px = reinterpret_cast<const T*>(s);
      pf = reinterpret_cast<const T*>(s + row_bytes);
      pg = reinterpret_cast<const T*>(s + 2 * row_bytes);
    } else {
      px = x + row * a.xs;
      pf = f + row * a.fs;
      pg = gate + row * a.gs;
    }
    at.load(pf, v);
    at.load(px, xv);
    // norm of the block's output
    float mean_f = 0.f, s = 0.f;
    if (!a.rms) {
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[e];
      mean_f = sum.one(s) * inv_c;
    }
    s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = at.on(e) ? v[e] - mean_f : 0.f;
      s += v[e] * v[e];
    }
    const float rstd_f = rsqrtf(sum.one(s) * inv_c + a.eps);
    at.table(tables, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] * rstd_f * w[e];
    // gate, residual scale, sum
    if (token_gate) {
      at.load(pg, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= a.gate_mode == GATE_SIGMOID ? sw_sigmoid(w[e]) : w[e];
    } else if (a.gate_mode == GATE_CHANNEL) {
      at.table(tables + 3 * wide, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= w[e];
    }
    if (a.scale != nullptr) {
      at.table(tables + 2 * wide, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += w[e] * xv[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += xv[e];
    }
    at.store(static_cast<T*>(a.y) + row * a.C, v);
    fetch(row + SW_STAGES * stride, stage);
    if (++stage == SW_STAGES) stage = 0;
    float mean_y = 0.f, rstd_y = 0.f;
    if (a.h != nullptr) {       // the next block's norm
      s = 0.f;
      if (!a.rms) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s += v[e];
        mean_y = sum.one(s) * inv_c;
      }
      s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = at.on(e) ? v[e] - mean_y : 0.f;
        s += v[e] * v[e];
      }
      rstd_y = rsqrtf(sum.one(s) * inv_c + a.eps);
      at.table(tables + wide, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * rstd_y * w[e];
      at.store(static_cast<T*>(a.h) + row * a.C, v);
    }
    if (a.stats != nullptr && at.lane == 0) {
      a.stats[row] = mean_f;
      a.stats[a.T + row] = rstd_f;
      a.stats[2 * a.T + row] = mean_y;
      a.stats[3 * a.T + row] = rstd_y;
    }
  }
}

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(512)
sandwich_bwd_kernel(const __grid_constant__ SandwichArgs a) {
  extern __shared__ __align__(128) uint8_t sw_smem[];
  const int group = threadIdx.x / a.tpr;
  const Place<T, ALIGNED> at{static_cast<int>(threadIdx.x) - group * a.tpr, group, a.tpr, a.C};
  float* tables = reinterpret_cast<float*>(sw_smem);
  const int wide = a.tpr * 8;
  float2* sums = reinterpret_cast<float2*>(tables + 4 * wide);
  uint8_t* ring = reinterpret_cast<uint8_t*>(sums + a.groups * 32);
  GroupSum sum{sums + group * 32, a.tpr >> 5, at.lane >> 5, 1 + group, a.tpr, 0};
  const bool token_gate = a.gate_mode >= GATE_TOKEN, has_dy = a.dy != nullptr, has_dh = a.dh != nullptr;
  const int parts = 2 + token_gate + has_dy + has_dh;
  const size_t row_bytes = static_cast<size_t>(a.C) * sizeof(T);
  uint8_t* mine = ring + static_cast<size_t>(group) * SW_STAGES * parts * row_bytes;
  grid_chain();
  const long long row0 = static_cast<long long>(blockIdx.x) * a.groups + group;
  const long long stride = static_cast<long long>(gridDim.x) * a.groups;
  const T *x = static_cast<const T*>(a.x), *f = static_cast<const T*>(a.f), *gate = static_cast<const T*>(a.gate);
  const T *dy = static_cast<const T*>(a.dy), *dh = static_cast<const T*>(a.dh);
  const size_t o_dy = 2 * row_bytes, o_dh = o_dy + has_dy * row_bytes, o_g = o_dh + has_dh * row_bytes;
  auto fetch = [&](long long row, int stage) {
    if (ALIGNED) {
      if (row < a.T && at.on(0)) {
        uint8_t* d = mine + static_cast<size_t>(stage) * parts * row_bytes + at.lane * sizeof(Eight<T>);
        const int c = at.lane * 8;
#pragma unroll
        for (int j = 0; j < static_cast<int>(sizeof(Eight<T>)); j += 16) {
          sw_cp_async_16(d + j, reinterpret_cast<const uint8_t*>(x + row * a.xs + c) + j);
          sw_cp_async_16(d + row_bytes + j, reinterpret_cast<const uint8_t*>(f + row * a.fs + c) + j);
          if (has_dy) sw_cp_async_16(d + o_dy + j, reinterpret_cast<const uint8_t*>(dy + row * a.dys + c) + j);
          if (has_dh) sw_cp_async_16(d + o_dh + j, reinterpret_cast<const uint8_t*>(dh + row * a.dhs + c) + j);
          if (token_gate) sw_cp_async_16(d + o_g + j, reinterpret_cast<const uint8_t*>(gate + row * a.gs + c) + j);
        }
      }
      sw_cp_commit();
    }
  };
#pragma unroll
  for (int i = 0; i < SW_STAGES; ++i) fetch(row0 + i * stride, i);
  sw_tables<T, ALIGNED>(a, at, tables);
  const float inv_c = 1.f / a.C;
  float acc[4][8];
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[k][e] = 0.f;
  int stage = 0;
  for (long long row = row0; row < a.T; row += stride) {
    const float mean_f = a.stats[row], rstd_f = a.stats[a.T + row];
    const float mean_y = a.stats[2 * a.T + row], rstd_y = a.stats[3 * a.T + row];
    const T *px, *pf, *pdy, *pdh, *pg;
    if (ALIGNED) {
      sw_cp_wait<SW_STAGES - 1>();
      const uint8_t* s = mine + static_cast<size_t>(stage) * parts * row_bytes;
      px = reinterpret_cast<const T*>(s);
      pf = reinterpret_cast<const T*>(s + row_bytes);
      pdy = reinterpret_cast<const T*>(s + o_dy);
      pdh = reinterpret_cast<const T*>(s + o_dh);
      pg = reinterpret_cast<const T*>(s + o_g);
    } else {
      px = x + row * a.xs;
      pf = f + row * a.fs;
      pdy = dy + row * a.dys;
      pdh = dh + row * a.dhs;
      pg = gate + row * a.gs;
    }
    float uf[8], g[8], t[8], w[8];      // u(f), the gate, t
    at.load(pf, uf);
#pragma unroll
    for (int e = 0; e < 8; ++e) uf[e] = at.on(e) ? (uf[e] - mean_f) * rstd_f : 0.f;
    if (token_gate) {
      at.load(pg, g);
      if (a.gate_mode == GATE_SIGMOID) {
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = sw_sigmoid(g[e]);
      }
    } else {
      at.table(tables + 3 * wide, g);
    }
    if (has_dh) {
      float uy[8], v[8];
      at.table(tables, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) uy[e] = g[e] * (uf[e] * w[e]);
      at.load(px, v);
      at.table(tables + 2 * wide, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) uy[e] = at.on(e) ? (uy[e] + w[e] * v[e] - mean_y) * rstd_y : 0.f;
      at.load(pdh, v);
      at.table(tables + wide, w);
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        acc[0][e] += v[e] * uy[e];
        t[e] = v[e] * w[e];
        s1 += t[e];
        s2 += t[e] * uy[e];
      }
      sum.two(s1, s2);
      s1 = a.rms ? 0.f : s1 * inv_c;
      s2 *= inv_c;
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = rstd_y * (t[e] - s1 - uy[e] * s2);
      if (has_dy) {
        at.load(pdy, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] += v[e];
      }
    } else {
      at.load(pdy, t);
    }
    {   // dx, and the sum for the residual scale
      float v[8], o[8];
      at.load(px, v);
      at.table(tables + 2 * wide, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (at.on(e)) acc[2][e] += t[e] * v[e];
        o[e] = w[e] * t[e];
      }
      at.store(static_cast<T*>(a.dx) + row * a.C, o);
    }
    at.table(tables, w);
    float s1 = 0.f, s2 = 0.f;
    if (token_gate) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        o[e] = t[e] * (uf[e] * w[e]);
        if (a.gate_mode == GATE_SIGMOID) o[e] *= g[e] * (1.f - g[e]);
      }
      at.store(static_cast<T*>(a.dg) + row * a.C, o);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at.on(e)) acc[3][e] += t[e] * (uf[e] * w[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      t[e] = at.on(e) ? t[e] * g[e] : 0.f;
      acc[1][e] += t[e] * uf[e];
      t[e] *= w[e];
      s1 += t[e];
      s2 += t[e] * uf[e];
    }
    sum.two(s1, s2);
    s1 = a.rms ? 0.f : s1 * inv_c;
    s2 *= inv_c;
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = rstd_f * (t[e] - s1 - uf[e] * s2);
    at.store(static_cast<T*>(a.df) + row * a.C, t);
    fetch(row + SW_STAGES * stride, stage);
    if (++stage == SW_STAGES) stage = 0;
  }
  if (a.want == 0) return;
  // the groups' column sums meet in the tables' memory, one kind at a time, and leave as this block's partial sums
  if (ALIGNED) sw_cp_wait<0>();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (!(a.want >> k & 1)) continue;
    float* out = a.partial + (static_cast<size_t>(k) * gridDim.x + blockIdx.x) * a.C;
    for (int j = 0; j < a.groups; ++j) {
      __syncthreads();
      if (group == j) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int s = at.slot(e);
          tables[s] = j ? tables[s] + acc[k][e] : acc[k][e];
        }
      }
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at.channel(e) < a.C) out[at.channel(e)] = tables[at.slot(e)];
    }
  }
}

// out[k][c] (= or +=) the sum over the blocks' partial sums, in their order. kind: 0 none, 1 bf16, 2 fp16, 3 fp32, 4 add to fp32.
struct ColumnSums {
  void* out[4];
  int kind[4];
};

__global__ void __launch_bounds__(512)
sandwich_columns_kernel(const float* __restrict__ partial, const __grid_constant__ ColumnSums to, int blocks, int C) {
  grid_chain();
  __shared__ float part[16][33];
  const int k = blockIdx.y, c = blockIdx.x * 32 + threadIdx.x;
  if (to.kind[k] == 0) return;
  float s = 0.f;
  if (c < C)
    for (int b = threadIdx.y; b < blocks; b += 16) s += partial[(static_cast<size_t>(k) * blocks + b) * C + c];
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < C) {
    s = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) s += part[j][threadIdx.x];
    if (to.kind[k] == 1) static_cast<__nv_bfloat16*>(to.out[k])[c] = __float2bfloat16_rn(s);
    else if (to.kind[k] == 2) static_cast<__half*>(to.out[k])[c] = __float2half_rn(s);
    else if (to.kind[k] == 3) static_cast<float*>(to.out[k])[c] = s;
    else static_cast<float*>(to.out[k])[c] += s;
  }
}

static int sw_shape(int C, int* tpr, int* groups) {
  if (C < 1 || C > SW_MAX_C) return -3;
  *tpr = ((C + 7) / 8 + 31) / 32 * 32;
  *groups = *tpr >= 256 ? 1 : 256 / *tpr;
  return 0;
}

static size_t sw_smem_bytes(const SandwichArgs& a, int parts, int size, bool aligned) {
  return static_cast<size_t>(a.tpr) * 8 * 4 * 4 + static_cast<size_t>(a.groups) * 32 * 8 +
         (aligned ? static_cast<size_t>(a.groups) * SW_STAGES * parts * a.C * size : 0);
}

template <typename T, bool ALIGNED>
static int sw_launch(const SandwichArgs& a, bool backward, unsigned blocks, size_t smem, cudaStream_t st) {
  auto kern = backward ? sandwich_bwd_kernel<T, ALIGNED> : sandwich_fwd_kernel<T, ALIGNED>;
  static bool configured_on[2][MAX_DEVICES];
  const int dev = current_device_slot();
  if (dev < 0) return -4;
  if (!configured_on[backward][dev]) {
    NPLM_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    configured_on[backward][dev] = true;
  }
  const cudaError_t e = launch_when(a.T * a.C <= CHAIN_ELEMENTS, kern, blocks, a.tpr * a.groups, smem, st, a);
  if (e != cudaSuccess) return static_cast<int>(e);
  return static_cast<int>(cudaGetLastError());
}

static int sw_run(const SandwichArgs& a, bool backward, int dtype, unsigned blocks, cudaStream_t st) {
  const int size = dtype == 2 ? 4 : 2;
  const void* rows[] = {a.x, a.f, a.gate_mode >= GATE_TOKEN ? a.gate : nullptr, a.dy, a.dh, a.y, a.h, a.dx, a.df, a.dg};
  const long long strides[] = {a.xs, a.fs, a.gate_mode >= GATE_TOKEN ? a.gs : 0, a.dys, a.dhs};
  bool aligned = a.C % 8 == 0;
  for (const void* p : rows) aligned &= reinterpret_cast<uintptr_t>(p) % 16 == 0;
  for (long long s : strides) aligned &= s * size % 16 == 0;
  const int parts = 2 + (a.gate_mode >= GATE_TOKEN) + (a.dy != nullptr) + (a.dh != nullptr);
  const size_t smem = sw_smem_bytes(a, parts, size, aligned);
  if (dtype == 0) return aligned ? sw_launch<__nv_bfloat16, true>(a, backward, blocks, smem, st)
                                 : sw_launch<__nv_bfloat16, false>(a, backward, blocks, smem, st);
  if (dtype == 1) return aligned ? sw_launch<__half, true>(a, backward, blocks, smem, st)
                                 : sw_launch<__half, false>(a, backward, blocks, smem, st);
  return aligned ? sw_launch<float, true>(a, backward, blocks, smem, st) : sw_launch<float, false>(a, backward, blocks, smem, st);
}

// Blocks of a pass: all rows at once where they fit, else as many blocks as the multiprocessors hold.
static unsigned sw_blocks(const SandwichArgs& a, int threads_an_sm) {
  const long long all = (a.T + a.groups - 1) / a.groups;
  int per_sm = threads_an_sm / (a.tpr * a.groups);
  if (per_sm < 1) per_sm = 1;
  const long long most = 148LL * per_sm;
  return static_cast<unsigned>(all < most ? all : most);
}

}  // namespace nplm

using namespace nplm;

// Blocks of nplm_sandwich_bwd, which its partial sums are counted in; negative: no such width.
extern "C" int nplm_sandwich_bwd_blocks(long long T, int C) {
  SandwichArgs a = {};
  a.T = T;
  a.C = C;
  const int rc = sw_shape(C, &a.tpr, &a.groups);
  return rc ? rc : static_cast<int>(sw_blocks(a, 512));
}

// dtype: 0 bf16, 1 fp16, 2 fp32. gate_mode: 0 none, 1 [C], 2 rows, 3 rows through a sigmoid. strides: rows of x, f, gate.
// stats: fp32 [4][T] for the backward pass, or null. h null: no norm follows.
extern "C" int nplm_sandwich_fwd(const void* x, const void* f, const void* gate, const void* post, const void* next,
                                 const void* scale, const long long* strides, void* y, void* h, float* stats, long long T,
                                 int C, float eps, int rms, int gate_mode, int dtype, int param32, cudaStream_t st) {
  if (T < 0 || dtype < 0 || dtype > 2 || gate_mode < 0 || gate_mode > 3 || (gate_mode != 0) != (gate != nullptr)) return -1;
  if (T == 0) return 0;
  SandwichArgs a = {};
  a.x = x; a.f = f; a.gate = gate; a.post = post; a.next = next; a.scale = scale;
  a.xs = strides[0]; a.fs = strides[1]; a.gs = strides[2];
  a.y = y; a.h = h; a.stats = stats; a.T = T; a.C = C; a.eps = eps; a.rms = rms; a.gate_mode = gate_mode; a.param32 = param32;
  const int rc = sw_shape(C, &a.tpr, &a.groups);
  return rc ? rc : sw_run(a, false, dtype, sw_blocks(a, 1024), st);
}

// dy or dh may be null. strides: rows of x, f, gate, dy, dh. partial: fp32 [4][blocks][C] scratch. sums / kinds: where the column
// sums of w_next, w_post, the scale and a [C] gate go, and as what (see ColumnSums).
extern "C" int nplm_sandwich_bwd(const void* dy, const void* dh, const void* x, const void* f, const void* gate,
                                 const void* post, const void* next, const void* scale, const float* stats,
                                 const long long* strides, void* dx, void* df, void* dg, float* partial, void* const* sums,
                                 const int* kinds, long long T, int C, int rms, int gate_mode, int dtype, int param32,
                                 cudaStream_t st) {
  if (T < 0 || dtype < 0 || dtype > 2 || gate_mode < 0 || gate_mode > 3 ||
      (T > 0 && ((gate_mode != 0) != (gate != nullptr) || (dy == nullptr && dh == nullptr))))
    return -1;
  SandwichArgs a = {};
  ColumnSums to;
  for (int k = 0; k < 4; ++k) {
    to.out[k] = sums[k];
    to.kind[k] = kinds[k];
    if (kinds[k]) a.want |= 1 << k;
  }
  a.x = x; a.f = f; a.gate = gate; a.post = post; a.next = next; a.scale = scale; a.dy = dy; a.dh = dh;
  a.xs = strides[0]; a.fs = strides[1]; a.gs = strides[2]; a.dys = strides[3]; a.dhs = strides[4];
  a.stats = const_cast<float*>(stats); a.dx = dx; a.df = df; a.dg = dg; a.partial = partial;
  a.T = T; a.C = C; a.rms = rms; a.gate_mode = gate_mode; a.param32 = param32;
  int rc = sw_shape(C, &a.tpr, &a.groups);
  if (rc) return rc;
  unsigned blocks = 0;      // (no rows: the column sums are zero)
  if (T > 0) {
    blocks = sw_blocks(a, 512);
    rc = sw_run(a, true, dtype, blocks, st);
    if (rc) return rc;
  }
  if (a.want) {
    const cudaError_t e = launch_chained(sandwich_columns_kernel, dim3((C + 31) / 32, 4), dim3(32, 16), 0, st,
                                         static_cast<const float*>(partial), to, static_cast<int>(blocks), C);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return static_cast<int>(cudaGetLastError());
}
