// The end of a residual block in one operator: norm of the block's output, gate, residual scale, sum, and the norm with which
// the next block starts. For a row (token) with block input x and block output f, channels c:
//   n = w_post u(f),   y = r x + g n,   h = w_next u(y),    u(v) = (v - mean v) / sqrt(var v + eps)   (RMSNorm: mean 0)
// with the gate g = 1, a weight per channel, or a value per token and channel, as it is or through a sigmoid.
// Backward, from dy and dh (B_v d = (d - mean d - u(v) mean(d u(v))) / sqrt(var v + eps), the gradient of u):
//   t = dy + B_y(w_next dh),   dx = r t,   df = B_f(w_post g t),   dg = t n,
//   dw_next = sum u(y) dh,   dw_post = sum u(f) g t,   dr = sum t x,   and dg summed where the gate is a weight: then
//   S = sum u(f) t gives both, dw_post = g S and dg = w_post S.
//
// Bound by memory: forward reads x, f (and g) and writes y, h; backward reads dy, dh, x, f (g) and writes dx, df (dg). Op by
// op the row travels three times as often. A row belongs to a group of threads, eight channels a thread, so that the channels
// of a thread never change: the column sums of the backward pass stay in its registers (in a warp-a-row layout they are
// 4 C / 32 registers a lane, which ends at 512 channels) and leave once a block, as partial sums that a second small kernel
// adds in a fixed order: the same bits every run. Statistics, sums and the residual sum are fp32; y and h are rounded
// once, and h is formed from the unrounded y, which the backward pass forms again from x and f. Reciprocal roots are rsqrtf, off by at
// most 2 units in the last place; a row's own sums are off by more.
//
// Measured, forward and backward with a gate of tokens, bf16: 55 424 x 1024 250 us (5.9 TB/s, 0.91 of the copy rate); 13 000 x
// 4096 361 us (0.59: a block holds one row, and its threads wait together for each sum); 55 000 x 1002 419 us (0.53) and x 1001
// 462 us (0.48), bound by instructions: words of two channels to load, mask and store. 1001 channel by channel 780 us, 1002 with
// a thread copying its own words 424 us (without a gate 339 against 327).
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace nplm {

constexpr int SW_STAGES = 2;        // steps ahead of which a group's rows are fetched (WORDS: 3); fewer where shared memory holds no more
constexpr int SW_MAX_C = 4096;
constexpr size_t SW_MAX_SMEM = 227 * 1024;

enum : int { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_TOKEN = 2, GATE_SIGMOID = 3 };

struct SandwichArgs {
  const void *x, *f, *gate, *dy, *dh;                 // rows of C, `*s` elements apart
  long long xs, fs, gs, dys, dhs;
  long long nx, nf, ng, ndy, ndh, nout;               // WORDS: elements from a group's row to its next one
  const void *post, *next, *scale;                    // [C] each; post, next null: 1; scale null: 1
  void *y, *h;                                        // forward outputs, contiguous rows; h may be null
  void *dx, *df, *dg;                                 // backward outputs, contiguous rows; dg only for gates of tokens
  float4* stats;                                      // [T]: mean f, 1 / std f, mean y, 1 / std y; null: not kept
  float* partial;                                     // [4][blocks][C]: dw_next, dw_post, dr, dg
  long long T;
  int C, tpr, groups;                                 // threads a row, rows that a block works on at a time
  uint32_t stages;
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
__device__ __forceinline__ void sw_cp_async_4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// (bytes of the word are copied, the others are zero)
__device__ __forceinline__ void sw_cp_async_4(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void sw_cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void sw_cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A thread's eight channels as four pairs, for the packed fp32 instructions.
struct Eight {
  float2 p[4];
};
__device__ __forceinline__ float2 sw_both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float sw_total(const Eight& v) {
  const float2 s = add2(add2(v.p[0], v.p[1]), add2(v.p[2], v.p[3]));
  return s.x + s.y;
}
__device__ __forceinline__ float sw_dot(const Eight& a, const Eight& b) {
  float2 s = mul2(a.p[0], b.p[0]);
#pragma unroll
  for (int k = 1; k < 4; ++k) s = fma2(a.p[k], b.p[k], s);
  return s.x + s.y;
}
__device__ __forceinline__ float2 sw_unpack(uint32_t w, __nv_bfloat16) { return unpack_bf16x2(w); }
__device__ __forceinline__ float2 sw_unpack(uint32_t w, __half) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
__device__ __forceinline__ uint32_t sw_pack(float2 v, __nv_bfloat16) { return pack_bf16x2(v.x, v.y); }
__device__ __forceinline__ uint32_t sw_pack(float2 v, __half) {
  const __half2 h = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// How a row lies in a group's threads, eight channels a thread. STRIDED: any width, addresses and strides, single channels tpr apart.
// ALIGNED: widths and addresses on 16 bytes, eight neighbours, or none. FULL: the same, and no thread has none. WORDS: tensors on 4
// bytes; the group fetches the 16-byte pieces that a row touches, and a thread takes words tpr apart from them: single fp32 channels,
// or pairs of 16 bits. Where width and strides are odd numbers of 16 bits, rows of odd numbers start in the middle of a word,
// in all tensors alike: there the pairs start one channel before the row (`shift`). A group's rows are a whole number of grids
// apart, an even number of rows, so they have one shift.
enum : int { STRIDED = 0, ALIGNED = 1, FULL = 2, WORDS = 3 };

template <typename T, int MODE>
struct Place {
  static constexpr bool PAIRS = MODE == WORDS && sizeof(T) == 2, SINGLES = MODE == STRIDED || (MODE == WORDS && sizeof(T) == 4);
  int lane, group, tpr, C, shift;
  bool any, edge;                  // PAIRS: one of the words holds one channel
  uint32_t keep[PAIRS ? 4 : 1];    // PAIRS: the bits of the words that are channels of the row
  __device__ __forceinline__ Place(int tpr_, int C_, int groups) : tpr(tpr_), C(C_) {
    group = threadIdx.x / tpr;
    lane = threadIdx.x - group * tpr;
    shift = PAIRS && C % 2 ? (blockIdx.x * groups + group) & 1 : 0;
    any = MODE == FULL || MODE == WORDS || channel(0) < C;
    edge = false;
    if constexpr (PAIRS) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool low = on(2 * k), high = on(2 * k + 1);
        keep[k] = (low ? 0xffffu : 0u) | (high ? 0xffff0000u : 0u);
        edge |= low != high;
      }
    }
  }
  __device__ __forceinline__ int channel(int e, int by) const {
    return SINGLES ? e * tpr + lane : PAIRS ? 2 * ((e >> 1) * tpr + lane) + (e & 1) - by : lane * 8 + e;
  }
  __device__ __forceinline__ int channel(int e) const { return channel(e, shift); }
  __device__ __forceinline__ bool on(int e) const {
    return MODE == FULL ? true : MODE == ALIGNED ? any : static_cast<unsigned>(channel(e)) < static_cast<unsigned>(C);
  }
  // the slot of a [C] table in shared memory: two halves of four channels a thread, so that a warp's 16-byte reads are
  // consecutive
  __device__ __forceinline__ int slot(int e) const { return (e >> 2) * tpr * 4 + lane * 4 + (e & 3); }
  // What `load` takes, out of the ring where it is about to be filled again.
  struct Words {
    uint32_t w[4];
  };
  __device__ __forceinline__ auto grab(const T* mine) const {
    if constexpr (PAIRS) {
      Words r;
#pragma unroll
      for (int k = 0; k < 4; ++k) r.w[k] = reinterpret_cast<const uint32_t*>(mine)[k * tpr];
      return r;
    } else if constexpr (MODE == WORDS) {
      return load(mine);
    } else {
      return mine;
    }
  }
  __device__ __forceinline__ Eight load(const Words& r) const {
    Eight v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v.p[k] = sw_unpack(r.w[k] & keep[PAIRS ? k : 0], T());
    return v;
  }
  __device__ __forceinline__ Eight load(const Eight& v) const { return v; }
  // The thread's channels of a row; `mine` is where its first one lies.
  __device__ __forceinline__ Eight load(const T* mine) const {
    Eight v;
    if constexpr (SINGLES) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v.p[k].x = on(2 * k) ? Io<T>::get(mine[2 * k * tpr]) : 0.f;
        v.p[k].y = on(2 * k + 1) ? Io<T>::get(mine[(2 * k + 1) * tpr]) : 0.f;
      }
    } else if constexpr (PAIRS) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v.p[k] = sw_unpack(reinterpret_cast<const uint32_t*>(mine)[k * tpr] & keep[k], T());
    } else if (MODE == FULL || any) {
      if constexpr (sizeof(T) == 2) {
        const uint4 u = *reinterpret_cast<const uint4*>(mine);
        v.p[0] = sw_unpack(u.x, T());
        v.p[1] = sw_unpack(u.y, T());
        v.p[2] = sw_unpack(u.z, T());
        v.p[3] = sw_unpack(u.w, T());
      } else {
        const float4 a = *reinterpret_cast<const float4*>(mine), b = *reinterpret_cast<const float4*>(mine + 4);
        v.p[0] = make_float2(a.x, a.y);
        v.p[1] = make_float2(a.z, a.w);
        v.p[2] = make_float2(b.x, b.y);
        v.p[3] = make_float2(b.z, b.w);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) v.p[k] = sw_both(0.f);
    }
    return v;
  }
  __device__ __forceinline__ void store(T* mine, const Eight& v) const {
    if constexpr (SINGLES) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (on(2 * k)) mine[2 * k * tpr] = Io<T>::put(v.p[k].x);
        if (on(2 * k + 1)) mine[(2 * k + 1) * tpr] = Io<T>::put(v.p[k].y);
      }
    } else if constexpr (PAIRS) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (keep[k] == 0xffffffffu) reinterpret_cast<uint32_t*>(mine)[k * tpr] = sw_pack(v.p[k], T());
      if (edge) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (keep[k] == 0xffffu) mine[2 * k * tpr] = Io<T>::put(v.p[k].x);
          if (keep[k] == 0xffff0000u) mine[2 * k * tpr + 1] = Io<T>::put(v.p[k].y);
        }
      }
    } else if (MODE == FULL || any) {
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(mine) =
            make_uint4(sw_pack(v.p[0], T()), sw_pack(v.p[1], T()), sw_pack(v.p[2], T()), sw_pack(v.p[3], T()));
      } else {
        *reinterpret_cast<float4*>(mine) = make_float4(v.p[0].x, v.p[0].y, v.p[1].x, v.p[1].y);
        *reinterpret_cast<float4*>(mine + 4) = make_float4(v.p[2].x, v.p[2].y, v.p[3].x, v.p[3].y);
      }
    }
  }
  __device__ __forceinline__ Eight table(const float* t) const {
    const float4 a = *reinterpret_cast<const float4*>(t + lane * 4), b = *reinterpret_cast<const float4*>(t + tpr * 4 + lane * 4);
    return Eight{{make_float2(a.x, a.y), make_float2(a.z, a.w), make_float2(b.x, b.y), make_float2(b.z, b.w)}};
  }
  // (v - mean) with zeros behind the row
  __device__ __forceinline__ Eight centred(const Eight& v, float mean) const {
    Eight r;
    const float2 m = sw_both(MODE == ALIGNED && !any ? 0.f : -mean);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (PAIRS) {      // (v is zero behind the row; a product with one or zero is exact)
        r.p[k] = fma2(sw_unpack(keep[k] & (std::is_same<T, __half>::value ? 0x3c003c00u : 0x3f803f80u), T()), m, v.p[k]);
      } else {
        r.p[k] = add2(v.p[k], m);
        if (SINGLES && !on(2 * k)) r.p[k].x = 0.f;
        if (SINGLES && !on(2 * k + 1)) r.p[k].y = 0.f;
      }
    }
    return r;
  }
};

// Whether rows are fetched to shared memory ahead of their use: each thread its own channels, but for WORDS.
template <typename T, int MODE>
constexpr bool SW_RING = MODE != STRIDED || sizeof(T) == 4;

template <typename T, int MODE>
__device__ __forceinline__ void sw_fetch(const Place<T, MODE>& at, uint8_t* to, const T* from) {
  if constexpr (MODE == STRIDED) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (at.on(e)) sw_cp_async_4(to + e * at.tpr * sizeof(T), from + e * at.tpr);
  } else {
#pragma unroll
    for (int j = 0; j < static_cast<int>(8 * sizeof(T)); j += 16) sw_cp_async_16(to + j, reinterpret_cast<const uint8_t*>(from) + j);
  }
}

// WORDS: the row from `from` on (its first channel less the shift) to a slot that begins where 16 bytes of memory do. The first and
// the last row of a tensor go word by word, so that nothing outside the tensor is read.
template <typename T, int MODE>
__device__ __forceinline__ void sw_fetch_row(const Place<T, MODE>& at, uint8_t* slot, const T* from, bool inner) {
  const uint32_t before = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(from)) & 15u;
  const int bytes = (at.C + at.shift) * static_cast<int>(sizeof(T));
  const uint8_t* src = reinterpret_cast<const uint8_t*>(from) - before;
  if (inner) {
    const int end = static_cast<int>(before) + bytes;
#pragma unroll
    for (int j = 0; j <= static_cast<int>(sizeof(T)) / 2; ++j) {      // (8 channels a thread, and the piece that a misplaced row has more)
      const int b = 16 * (at.lane + j * at.tpr);
      if (b < end) sw_cp_async_16(slot + b, src + b);
    }
  } else {
    for (int b = 4 * at.lane; b < bytes; b += 4 * at.tpr)
      sw_cp_async_4(slot + before + b, src + before + b, bytes - b < 4 ? bytes - b : 4);
  }
}
// All but the last `stages` - 2 (+ MORE) steps of this thread's copies have arrived.
template <int MORE>
__device__ __forceinline__ void sw_arrived(uint32_t stages) {
  if (stages == 3) sw_cp_wait<1 + MORE>();
  else sw_cp_wait<MORE>();
}
// Before the group's threads meet in a sum: the next step's copies have arrived. A group within a warp meets here.
template <bool SUB>
__device__ __forceinline__ void sw_ready(uint32_t stages, int warps) {
  sw_arrived<0>(stages);
  if (SUB || warps == 1) __syncwarp();
}
// `p` of a slot, where the row starts in it: the row `steps` steps of `step` elements before `ahead`. (A row that is not there, behind
// the last one, may start between words; its slot is read all the same.)
template <typename T>
__device__ __forceinline__ const T* sw_within(const T* p, const T* ahead, long long step, uint32_t steps) {
  const uint32_t row = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ahead)) -
                       steps * static_cast<uint32_t>(step) * static_cast<uint32_t>(sizeof(T));
  return reinterpret_cast<const T*>(reinterpret_cast<const uint8_t*>(p) + (row & 12u));
}

// Sums of two numbers over the threads of a group, in every one of them and in the same order. Within a warp one exchange gives
// either number to half of the lanes, which then add it up in four; the warps' sums meet in slots: [2][2][16] of the group,
// the ones behind the last warp zero. The barrier of one sum keeps the slots of the one before it from being
// overwritten too early, so two sets are enough.
//
// SUB: several groups a warp, threads (a power of two) lanes each; all of the warp's lanes take part.
template <bool SUB>
struct GroupSum {
  float* slots;
  int warps, warp, bar, threads, phase;
  __device__ __forceinline__ void two(float& a, float& b) {
    if (SUB) {
      for (int o = threads >> 1; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
      }
      return;
    }
    const int lane = threadIdx.x & 31;
    const bool high = lane & 16;
    const float keep = high ? b : a, give = high ? a : b;
    float v = keep + __shfl_xor_sync(0xffffffffu, give, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (warps == 1) {
      a = __shfl_sync(0xffffffffu, v, 0);
      b = __shfl_sync(0xffffffffu, v, 16);
      return;
    }
    float* s = slots + phase * 32;
    phase ^= 1;
    if ((lane & 15) == 0) s[lane + warp] = v;     // lane 0: the first sixteen, lane 16: the others
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(threads) : "memory");
    const float4 x = *reinterpret_cast<const float4*>(s), y = *reinterpret_cast<const float4*>(s + 16);
    a = (x.x + x.y) + (x.z + x.w);
    b = (y.x + y.y) + (y.z + y.w);
    for (int w = 4; w < warps; w += 4) {
      const float4 x2 = *reinterpret_cast<const float4*>(s + w), y2 = *reinterpret_cast<const float4*>(s + 16 + w);
      a += (x2.x + x2.y) + (x2.z + x2.w);
      b += (y2.x + y2.y) + (y2.z + y2.w);
    }
  }
};

template <typename T>
__device__ __forceinline__ float sw_param(const void* p, int c, int param32) {
  if (p == nullptr) return 1.f;
  return param32 ? static_cast<const float*>(p)[c] : Io<T>::get(static_cast<const T*>(p)[c]);
}

// Shared memory: tables post, next, scale, gate [4][tpr * 8] fp32 (where shifts differ: of even and of odd groups) | sums
// [groups][2][2][16] where a row has several warps | ring [groups][stages][rows][parts][C]
__host__ __device__ constexpr int sw_sums(int tpr, int groups) { return tpr > 32 ? groups * 64 : 0; }
__host__ __device__ constexpr int sw_sets(int mode, int C, int size, int groups) {
  return mode == WORDS && size == 2 && C % 2 && groups > 1 ? 2 : 1;
}
// (WORDS: room for what a row's first and last 16 bytes hold of its neighbours)
__host__ __device__ constexpr uint32_t sw_row_bytes(int mode, int C, int size) {
  return mode == WORDS ? (C * size + 32) & ~15 : C * size;
}

template <typename T, int MODE>
__device__ __forceinline__ void sw_tables(const SandwichArgs& a, const Place<T, MODE>& at, float* tables, float* sums) {
  const int wide = a.tpr * 8;
  const void* of[4] = {a.post, a.next, a.scale, a.gate_mode == GATE_CHANNEL ? a.gate : nullptr};
  const int sets = sw_sets(MODE, a.C, sizeof(T), a.groups);
#pragma unroll
  for (int k = 0; k < (MODE == WORDS ? 8 : 4); ++k) {
    if (k % a.groups != at.group || k >= 4 * sets) continue;
    const int shift = sets > 1 ? (at.shift + at.group + (k >> 2)) & 1 : at.shift;      // of the groups of the set
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = at.channel(e, shift);
      tables[k * wide + at.slot(e)] = c >= 0 && c < a.C ? sw_param<T>(of[k & 3], c, a.param32) : 0.f;
    }
  }
  for (int i = threadIdx.x; i < sw_sums(a.tpr, a.groups); i += blockDim.x) sums[i] = 0.f;
  __syncthreads();
}

// Gates through a sigmoid g = 1 / (1 + e^-v). 16-bit rows hold g, by the approximate exponential and reciprocal: off by 2^-21 of itself
// for |v| up to 8 and by |v| 2^-24 beyond, far below the rows' own rounding; 0 where e^-v overflows. fp32 rows hold the smaller of g and
// 1 - g with the sign of v, good to fp32's last bits wherever v is: g and the slope g (1 - g) lose none of them next to 0 and 1
// (27 000 x 1024, both ways: 302 us, approximate 293).
__device__ __forceinline__ float sw_smaller(float v) {
  const float e = expf(-fabsf(v)), d = 1.f + e;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));      // (of a number between 1 and 2)
  const float q = e * r;
  return copysignf(fmaf(fmaf(-q, d, e), r, q), v);           // the quotient, corrected by what it leaves of e (Newton)
}
__device__ __forceinline__ float sw_from_smaller(float s) { return signbit(s) ? -s : 1.f - s; }
template <typename T>
__device__ __forceinline__ Eight sw_sigmoid(const Eight& v) {
  Eight r;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) {
      r.p[k] = make_float2(sw_smaller(v.p[k].x), sw_smaller(v.p[k].y));
    } else {
      float2 t = mul2(v.p[k], sw_both(-1.4426950408889634f));
      asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t.x));
      asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(t.y));
      t = add2(t, sw_both(1.f));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.p[k].x) : "f"(t.x));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.p[k].y) : "f"(t.y));
    }
  }
  return r;
}
// g, and g (1 - g), of what sw_sigmoid gave
template <typename T>
__device__ __forceinline__ Eight sw_gate(const Eight& held) {
  if constexpr (sizeof(T) != 4) {
    return held;
  } else {
    Eight r;
#pragma unroll
    for (int k = 0; k < 4; ++k) r.p[k] = make_float2(sw_from_smaller(held.p[k].x), sw_from_smaller(held.p[k].y));
    return r;
  }
}
template <typename T>
__device__ __forceinline__ float2 sw_slope(float2 held) {
  const float2 g = sizeof(T) == 4 ? make_float2(fabsf(held.x), fabsf(held.y)) : held;
  return fma2(make_float2(-g.x, -g.y), g, g);
}
__device__ __forceinline__ Eight sw_mul(const Eight& a, const Eight& b) {
  Eight r;
#pragma unroll
  for (int k = 0; k < 4; ++k) r.p[k] = mul2(a.p[k], b.p[k]);
  return r;
}
__device__ __forceinline__ Eight sw_scaled(const Eight& a, float s) {
  Eight r;
#pragma unroll
  for (int k = 0; k < 4; ++k) r.p[k] = mul2(a.p[k], sw_both(s));
  return r;
}
__device__ __forceinline__ Eight sw_fma(const Eight& a, const Eight& b, const Eight& c) {
  Eight r;
#pragma unroll
  for (int k = 0; k < 4; ++k) r.p[k] = fma2(a.p[k], b.p[k], c.p[k]);
  return r;
}
__device__ __forceinline__ Eight sw_add(const Eight& a, const Eight& b) {
  Eight r;
#pragma unroll
  for (int k = 0; k < 4; ++k) r.p[k] = add2(a.p[k], b.p[k]);
  return r;
}

// GATE: the gate's form, or -1 where it is looked up. (The full mode has a kernel for each form that reads different rows.)
constexpr int GATE_ANY = -1;

// Two rows at a time: their sums share the exchanges and barriers, and the tables are read once for both.
template <typename T, int MODE, int GATE, bool SUB>
__global__ void __maxnreg__(MODE == STRIDED || MODE == WORDS ? 128 : 80)
sandwich_fwd_kernel(const __grid_constant__ SandwichArgs a) {
  extern __shared__ __align__(128) uint8_t sw_smem[];
  const Place<T, MODE> at(a.tpr, a.C, a.groups);
  float* tables = reinterpret_cast<float*>(sw_smem);
  const int wide = a.tpr * 8, sets = sw_sets(MODE, a.C, sizeof(T), a.groups);
  float* sums = tables + sets * 4 * wide;
  GroupSum<SUB> sum{sums + (SUB ? 0 : at.group * 64), a.tpr >> 5, at.lane >> 5, 1 + at.group, a.tpr, 0};
  const int gate_mode = GATE == GATE_ANY ? a.gate_mode : GATE == GATE_NONE ? (a.gate_mode ? GATE_CHANNEL : GATE_NONE) : GATE;
  const bool token_gate = GATE == GATE_ANY ? gate_mode >= GATE_TOKEN : GATE >= GATE_TOKEN;
  const uint32_t row_bytes = sw_row_bytes(MODE, a.C, sizeof(T)), parts = token_gate ? 3 : 2;
  const uint32_t step_bytes = 2 * parts * row_bytes;      // two rows of all parts
  uint8_t* ring = reinterpret_cast<uint8_t*>(sums + sw_sums(a.tpr, a.groups)) + at.group * a.stages * step_bytes +
                  (MODE == WORDS ? 4 * at.lane : at.channel(0) * static_cast<int>(sizeof(T)));
  grid_chain();
  const long long row0 = static_cast<long long>(blockIdx.x) * a.groups + at.group;
  const long long stride = static_cast<long long>(gridDim.x) * a.groups;
  // where the thread's channels of the row to fetch next lie, and how far the next row is
  const int c0 = MODE == WORDS ? -at.shift : at.channel(0);
  const T *x = static_cast<const T*>(a.x) + row0 * a.xs + c0, *f = static_cast<const T*>(a.f) + row0 * a.fs + c0;
  const T* gate = token_gate ? static_cast<const T*>(a.gate) + row0 * a.gs + c0 : nullptr;
  const long long dx = stride * a.xs, df = stride * a.fs, dg = stride * a.gs, dy = stride * a.C;
  T *y = static_cast<T*>(a.y) + row0 * a.C + at.channel(0), *h = static_cast<T*>(a.h) + row0 * a.C + at.channel(0);
  const bool with_next = a.h != nullptr;
  long long ahead = row0;     // the row that `x` and the others are at
  auto fetch = [&](uint32_t stage) {
    if (SW_RING<T, MODE>) {
      uint8_t* d = ring + stage * step_bytes;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if constexpr (MODE == WORDS) {
          if (ahead < a.T) {
            const bool inner = ahead > 0 && ahead < a.T - 1;
            sw_fetch_row(at, d - 4 * at.lane, x, inner);
            sw_fetch_row(at, d - 4 * at.lane + row_bytes, f, inner);
            if (token_gate) sw_fetch_row(at, d - 4 * at.lane + 2 * row_bytes, gate, inner);
          }
        } else if (ahead < a.T && at.any) {
          sw_fetch(at, d, x);
          sw_fetch(at, d + row_bytes, f);
          if (token_gate) sw_fetch(at, d + 2 * row_bytes, gate);
        }
        d += parts * row_bytes;
        x += dx;
        f += df;
        if (token_gate) gate += dg;
        ahead += stride;
      }
      sw_cp_commit();
    }
  };
  for (int i = 0; i < a.stages; ++i) fetch(i);
  if (MODE == WORDS) sw_arrived<1>(a.stages);      // (the first step is there for all after the barrier in sw_tables)
  sw_tables<T, MODE>(a, at, tables, sums);
  if (sets > 1) tables += (at.group & 1) * 4 * wide;
  const float inv_c = 1.f / a.C;
  uint32_t stage = 0;
  const int behind = SUB ? (threadIdx.x & 31) / a.tpr : 0;      // groups of the warp before this one, whose rows come first
  for (long long row = row0; row - behind < a.T; row += 2 * stride) {
    // (a row that is not there holds what the memory did, and is not stored)
    const bool live = !SUB || row < a.T, two = row + stride < a.T;
    const T *px[2], *pf[2], *pg[2];
    if (SW_RING<T, MODE>) {
      const uint8_t* s = ring + stage * step_bytes;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        px[k] = reinterpret_cast<const T*>(s + k * parts * row_bytes);
        pf[k] = reinterpret_cast<const T*>(s + k * parts * row_bytes + row_bytes);
        pg[k] = reinterpret_cast<const T*>(s + k * parts * row_bytes + 2 * row_bytes);
        if (MODE == WORDS) {
          px[k] = sw_within(px[k], x, dx, 2 * a.stages - k);
          pf[k] = sw_within(pf[k], f, df, 2 * a.stages - k);
          pg[k] = sw_within(pg[k], gate, dg, 2 * a.stages - k);
        }
      }
      if (MODE == WORDS) {
      } else if (a.stages > 1) {
        sw_cp_wait<1>();
      } else {
        sw_cp_wait<0>();
      }
    } else {
      px[0] = live ? x : static_cast<const T*>(a.x) + at.channel(0);
      pf[0] = live ? f : static_cast<const T*>(a.f) + at.channel(0);
      pg[0] = live || !token_gate ? gate : static_cast<const T*>(a.gate) + at.channel(0);
      px[1] = two ? x + dx : px[0];
      pf[1] = two ? f + df : pf[0];
      pg[1] = two ? gate + dg : pg[0];
    }
    // norm of the block's output
    Eight v[2];
    v[0] = at.load(pf[0]);
    v[1] = at.load(pf[1]);
    float mean_f[2] = {0.f, 0.f}, rstd_f[2];
    if (!a.rms) {
      mean_f[0] = sw_total(v[0]);
      mean_f[1] = sw_total(v[1]);
      sum.two(mean_f[0], mean_f[1]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        mean_f[k] *= inv_c;
        v[k] = at.centred(v[k], mean_f[k]);
      }
    }
    rstd_f[0] = sw_dot(v[0], v[0]);
    rstd_f[1] = sw_dot(v[1], v[1]);
    const auto x0 = at.grab(px[0]), x1 = at.grab(px[1]);
    auto g0 = x0, g1 = x1;
    if (token_gate) {
      g0 = at.grab(pg[0]);
      g1 = at.grab(pg[1]);
    }
    if (MODE == WORDS) sw_ready<SUB>(a.stages, sum.warps);
    sum.two(rstd_f[0], rstd_f[1]);
    if (MODE == WORDS) {      // all have taken this step's rows, and the next one's are there
      fetch(stage);
      if (++stage == a.stages) stage = 0;
    }
    {
      const Eight w = at.table(tables);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        rstd_f[k] = rsqrtf(fmaf(rstd_f[k], inv_c, a.eps));
        v[k] = sw_mul(sw_scaled(v[k], rstd_f[k]), w);
      }
    }
    // gate, residual scale, sum
    if (token_gate) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const Eight g = at.load(k ? g1 : g0);
        v[k] = sw_mul(v[k], gate_mode == GATE_SIGMOID ? sw_gate<T>(sw_sigmoid<T>(g)) : g);
      }
    } else if (gate_mode == GATE_CHANNEL) {
      const Eight g = at.table(tables + 3 * wide);
      v[0] = sw_mul(v[0], g);
      v[1] = sw_mul(v[1], g);
    }
    if (a.scale != nullptr) {
      const Eight r = at.table(tables + 2 * wide);
      v[0] = sw_fma(r, at.load(x0), v[0]);
      v[1] = sw_fma(r, at.load(x1), v[1]);
    } else {
      v[0] = sw_add(at.load(x0), v[0]);
      v[1] = sw_add(at.load(x1), v[1]);
    }
    if (live) at.store(y, v[0]);
    if (two) at.store(y + dy, v[1]);
    y += 2 * dy;
    if (MODE == WORDS) {
    } else if (SW_RING<T, MODE>) {
      fetch(stage);
      if (++stage == a.stages) stage = 0;
    } else {
      x += 2 * dx;
      f += 2 * df;
      if (token_gate) gate += 2 * dg;
    }
    float mean_y[2] = {0.f, 0.f}, rstd_y[2] = {0.f, 0.f};
    if (with_next) {       // the next block's norm
      if (!a.rms) {
        mean_y[0] = sw_total(v[0]);
        mean_y[1] = sw_total(v[1]);
        sum.two(mean_y[0], mean_y[1]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          mean_y[k] *= inv_c;
          v[k] = at.centred(v[k], mean_y[k]);
        }
      }
      rstd_y[0] = sw_dot(v[0], v[0]);
      rstd_y[1] = sw_dot(v[1], v[1]);
      sum.two(rstd_y[0], rstd_y[1]);
      const Eight w = at.table(tables + wide);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        rstd_y[k] = rsqrtf(fmaf(rstd_y[k], inv_c, a.eps));
        v[k] = sw_mul(sw_scaled(v[k], rstd_y[k]), w);
      }
      if (live) at.store(h, v[0]);
      if (two) at.store(h + dy, v[1]);
      h += 2 * dy;
    }
    if (a.stats != nullptr && at.lane == 0 && live) {
      a.stats[row] = make_float4(mean_f[0], rstd_f[0], mean_y[0], rstd_y[0]);
      if (two) a.stats[row + stride] = make_float4(mean_f[1], rstd_f[1], mean_y[1], rstd_y[1]);
    }
  }
}

template <typename T, int MODE, int GATE, bool SUB>
__global__ void __launch_bounds__(512)
sandwich_bwd_kernel(const __grid_constant__ SandwichArgs a) {
  extern __shared__ __align__(128) uint8_t sw_smem[];
  const Place<T, MODE> at(a.tpr, a.C, a.groups);
  float* tables = reinterpret_cast<float*>(sw_smem);
  const int wide = a.tpr * 8, sets = sw_sets(MODE, a.C, sizeof(T), a.groups);
  float* sums = tables + sets * 4 * wide;
  GroupSum<SUB> sum{sums + (SUB ? 0 : at.group * 64), a.tpr >> 5, at.lane >> 5, 1 + at.group, a.tpr, 0};
  const int gate_mode = GATE == GATE_ANY ? a.gate_mode : GATE;      // (none and a weight are the same: the table has the ones)
  const bool token_gate = gate_mode >= GATE_TOKEN;
  const bool has_dy = a.dy != nullptr, has_dh = a.dh != nullptr;
  const uint32_t row_bytes = sw_row_bytes(MODE, a.C, sizeof(T));
  const uint32_t o_dy = 2 * row_bytes, o_dh = o_dy + has_dy * row_bytes, o_g = o_dh + has_dh * row_bytes;
  const uint32_t step_bytes = o_g + token_gate * row_bytes;
  uint8_t* ring = reinterpret_cast<uint8_t*>(sums + sw_sums(a.tpr, a.groups)) + at.group * a.stages * step_bytes +
                  (MODE == WORDS ? 4 * at.lane : at.channel(0) * static_cast<int>(sizeof(T)));
  grid_chain();
  const long long row0 = static_cast<long long>(blockIdx.x) * a.groups + at.group;
  const long long stride = static_cast<long long>(gridDim.x) * a.groups;
  const int c0 = MODE == WORDS ? -at.shift : at.channel(0);
  const T *x = static_cast<const T*>(a.x) + row0 * a.xs + c0, *f = static_cast<const T*>(a.f) + row0 * a.fs + c0;
  const T* gate = token_gate ? static_cast<const T*>(a.gate) + row0 * a.gs + c0 : nullptr;
  const T* dy = has_dy ? static_cast<const T*>(a.dy) + row0 * a.dys + c0 : nullptr;
  const T* dh = has_dh ? static_cast<const T*>(a.dh) + row0 * a.dhs + c0 : nullptr;
  // (WORDS, short of registers, takes them from the arguments: 55 000 x 1001 470 -> 462 us, without a gate 364 -> 351; FULL loses by it)
  const long long nx = MODE == WORDS ? a.nx : stride * a.xs, nf = MODE == WORDS ? a.nf : stride * a.fs;
  const long long ng = MODE == WORDS ? a.ng : stride * a.gs, ndy = MODE == WORDS ? a.ndy : stride * a.dys;
  const long long ndh = MODE == WORDS ? a.ndh : stride * a.dhs, nout = MODE == WORDS ? a.nout : stride * a.C;
  long long out = row0 * a.C + at.channel(0);
  long long ahead = row0;
  auto advance = [&]() {
    x += nx;
    f += nf;
    if (has_dy) dy += ndy;
    if (has_dh) dh += ndh;
    if (token_gate) gate += ng;
  };
  auto fetch = [&](uint32_t stage) {
    if (SW_RING<T, MODE>) {
      if constexpr (MODE == WORDS) {
        if (ahead < a.T) {
          const bool inner = ahead > 0 && ahead < a.T - 1;
          uint8_t* d = ring - 4 * at.lane + stage * step_bytes;
          sw_fetch_row(at, d, x, inner);
          sw_fetch_row(at, d + row_bytes, f, inner);
          if (has_dy) sw_fetch_row(at, d + o_dy, dy, inner);
          if (has_dh) sw_fetch_row(at, d + o_dh, dh, inner);
          if (token_gate) sw_fetch_row(at, d + o_g, gate, inner);
        }
      } else if (ahead < a.T && at.any) {
        uint8_t* d = ring + stage * step_bytes;
        sw_fetch(at, d, x);
        sw_fetch(at, d + row_bytes, f);
        if (has_dy) sw_fetch(at, d + o_dy, dy);
        if (has_dh) sw_fetch(at, d + o_dh, dh);
        if (token_gate) sw_fetch(at, d + o_g, gate);
      }
      advance();
      ahead += stride;
      sw_cp_commit();
    }
  };
  for (int i = 0; i < a.stages; ++i) fetch(i);
  if (MODE == WORDS) sw_arrived<1>(a.stages);      // (the first step is there for all after the barrier in sw_tables)
  sw_tables<T, MODE>(a, at, tables, sums);
  if (sets > 1) tables += (at.group & 1) * 4 * wide;
  const float inv_c = 1.f / a.C;
  // column sums u(y) dh, u(f) g t (where the gate is a weight u(f) t, which gives both w_post's and the gate's) and t x
  Eight acc[4];
#pragma unroll
  for (int k = 0; k < 3; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[k].p[e] = sw_both(0.f);
  uint32_t stage = 0;
  float4 st = make_float4(0.f, 0.f, 0.f, 0.f);      // statistics of the next row
  if (row0 < a.T) st = a.stats[row0];
  const int behind = SUB ? (threadIdx.x & 31) / a.tpr : 0;
  for (long long row = row0; row - behind < a.T; row += stride) {
    const bool live = !SUB || row < a.T;
    const float mean_f = st.x, rstd_f = st.y, mean_y = st.z, rstd_y = st.w;
    if (row + stride < a.T) st = a.stats[row + stride];
    const T *px, *pf, *pdy, *pdh, *pg;
    if (SW_RING<T, MODE>) {
      const uint8_t* s = ring + stage * step_bytes;
      px = reinterpret_cast<const T*>(s);
      pf = reinterpret_cast<const T*>(s + row_bytes);
      pdy = reinterpret_cast<const T*>(s + o_dy);
      pdh = reinterpret_cast<const T*>(s + o_dh);
      pg = reinterpret_cast<const T*>(s + o_g);
      if (MODE == WORDS) {
        px = sw_within(px, x, nx, a.stages);
        pf = sw_within(pf, f, nf, a.stages);
        pdy = sw_within(pdy, dy, ndy, a.stages);
        pdh = sw_within(pdh, dh, ndh, a.stages);
        pg = sw_within(pg, gate, ng, a.stages);
      } else if (a.stages > 1) {
        sw_cp_wait<1>();
      } else {
        sw_cp_wait<0>();
      }
    } else {
      px = live ? x : static_cast<const T*>(a.x) + c0;
      pf = live ? f : static_cast<const T*>(a.f) + c0;
      pdy = live || !has_dy ? dy : static_cast<const T*>(a.dy) + c0;
      pdh = live || !has_dh ? dh : static_cast<const T*>(a.dh) + c0;
      pg = live || !token_gate ? gate : static_cast<const T*>(a.gate) + c0;
    }
    const Eight uf = sw_scaled(at.centred(at.load(pf), mean_f), rstd_f);       // u(f)
    Eight g, t;
    if (token_gate) {
      g = at.load(pg);
      if (gate_mode == GATE_SIGMOID) g = sw_sigmoid<T>(g);
    } else {
      g = at.table(tables + 3 * wide);
    }
    constexpr bool held = sizeof(T) == 4;      // g as sw_sigmoid holds it, where that has run
    if (has_dh) {
      Eight uy = sw_mul(held && gate_mode == GATE_SIGMOID ? sw_gate<T>(g) : g, sw_mul(uf, at.table(tables)));
      uy = sw_fma(at.table(tables + 2 * wide), at.load(px), uy);
      uy = sw_scaled(at.centred(uy, mean_y), rstd_y);
      const Eight d = at.load(pdh);
      if (live) acc[0] = sw_fma(d, uy, acc[0]);
      t = sw_mul(d, at.table(tables + wide));
      float s1 = sw_total(t), s2 = sw_dot(t, uy);
      sum.two(s1, s2);
      s1 = a.rms ? 0.f : -s1 * inv_c * rstd_y;
      s2 *= -inv_c * rstd_y;
#pragma unroll
      for (int k = 0; k < 4; ++k) t.p[k] = fma2(uy.p[k], sw_both(s2), fma2(t.p[k], sw_both(rstd_y), sw_both(s1)));
      if (has_dy) t = sw_add(t, at.load(pdy));
    } else {
      t = at.load(pdy);
    }
    {   // dx, and the sum for the residual scale
      if (live) acc[2] = sw_fma(t, at.load(px), acc[2]);
      if (live) at.store(static_cast<T*>(a.dx) + out, sw_mul(t, at.table(tables + 2 * wide)));
    }
    const Eight w = at.table(tables);
    if (token_gate) {
      const Eight tn = sw_mul(t, sw_mul(uf, w));      // t n
      if (gate_mode == GATE_SIGMOID) {
        Eight o;
#pragma unroll
        for (int k = 0; k < 4; ++k) o.p[k] = mul2(tn.p[k], sw_slope<T>(g.p[k]));
        if (live) at.store(static_cast<T*>(a.dg) + out, o);
      } else {
        if (live) at.store(static_cast<T*>(a.dg) + out, tn);
      }
      t = sw_mul(t, held && gate_mode == GATE_SIGMOID ? sw_gate<T>(g) : g);
    }
    if (live) acc[1] = sw_fma(t, uf, acc[1]);
    t = sw_mul(t, token_gate ? w : sw_mul(g, w));
    float s1 = sw_total(t), s2 = sw_dot(t, uf);
    if (MODE == WORDS) sw_ready<SUB>(a.stages, sum.warps);
    sum.two(s1, s2);
    if (MODE == WORDS) {      // all have taken this step's rows, and the next one's are there
      fetch(stage);
      if (++stage == a.stages) stage = 0;
    }
    s1 = a.rms ? 0.f : -s1 * inv_c * rstd_f;
    s2 *= -inv_c * rstd_f;
#pragma unroll
    for (int k = 0; k < 4; ++k) t.p[k] = fma2(uf.p[k], sw_both(s2), fma2(t.p[k], sw_both(rstd_f), sw_both(s1)));
    if (live) at.store(static_cast<T*>(a.df) + out, t);
    out += nout;
    if (MODE == WORDS) {
    } else if (SW_RING<T, MODE>) {
      fetch(stage);
      if (++stage == a.stages) stage = 0;
    } else {
      advance();
    }
  }
  if (a.want == 0) return;
  // the groups' column sums meet in the tables' memory, one kind at a time, and leave as this block's partial sums
  if (SW_RING<T, MODE>) sw_cp_wait<0>();
  if (!token_gate) {
    acc[3] = sw_mul(acc[1], at.table(tables));
    acc[1] = sw_mul(acc[1], at.table(tables + 3 * wide));
  }
  tables = reinterpret_cast<float*>(sw_smem);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (!(a.want >> k & 1)) continue;
    float* out = a.partial + (static_cast<size_t>(k) * gridDim.x + blockIdx.x) * a.C;
    if (SUB) {        // a warp's groups first
      for (int o = a.tpr; o < 32; o <<= 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[k].p[e].x += __shfl_xor_sync(0xffffffffu, acc[k].p[e].x, o);
          acc[k].p[e].y += __shfl_xor_sync(0xffffffffu, acc[k].p[e].y, o);
        }
      }
    }
    const int members = SUB ? static_cast<int>(blockDim.x) >> 5 : a.groups;
    const int me = SUB ? (behind == 0 ? static_cast<int>(threadIdx.x) >> 5 : -1) : at.group;
    for (int j = 0; j < members; ++j) {
      __syncthreads();
      if (me == j) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (sets > 1 && !at.on(e)) continue;
          const int q = sets > 1 ? at.channel(e) : at.slot(e);
          const float v = e & 1 ? acc[k].p[e / 2].y : acc[k].p[e / 2].x;
          tables[q] = j ? tables[q] + v : v;
        }
      }
    }
    __syncthreads();
    if (at.group == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at.on(e)) out[at.channel(e)] = tables[sets > 1 ? at.channel(e) : at.slot(e)];
    }
  }
}

// out[k][c] (= or +=) the sum over the blocks' partial sums, in their order. kind: 0 none, 1 bf16, 2 fp16, 3 fp32, 4 add to fp32.
// A kind is a block's, so no two outputs may share memory.
struct ColumnSums {
  void* out[4];
  int kind[4];
};

__global__ void __launch_bounds__(1024)
sandwich_columns_kernel(const float* __restrict__ partial, const __grid_constant__ ColumnSums to, int blocks, int C) {
  grid_chain();
  __shared__ float part[32][33];
  const int k = blockIdx.y, c = blockIdx.x * 32 + threadIdx.x;
  if (to.kind[k] == 0) return;
  float s = 0.f;
  if (c < C) {
    const float* p = partial + (static_cast<size_t>(k) * blocks + threadIdx.y) * C + c;
    const size_t step = static_cast<size_t>(32) * C;
    int b = threadIdx.y;
    for (; b + 96 < blocks; b += 128, p += 4 * step) s += (p[0] + p[step]) + (p[2 * step] + p[3 * step]);
    for (; b < blocks; b += 32, p += step) s += *p;
  }
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  // warp y adds up column y
  s = part[threadIdx.x][threadIdx.y];
  s = warp_sum(s);
  const int mine = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && mine < C) {
    if (to.kind[k] == 1) static_cast<__nv_bfloat16*>(to.out[k])[mine] = __float2bfloat16_rn(s);
    else if (to.kind[k] == 2) static_cast<__half*>(to.out[k])[mine] = __float2half_rn(s);
    else if (to.kind[k] == 3) static_cast<float*>(to.out[k])[mine] = s;
    else static_cast<float*>(to.out[k])[mine] += s;
  }
}

// Threads a row, rows a block and blocks of a pass. An SM holds 512 threads of 128 registers (backward, and rows that are read
// channel by channel or word by word), in one block where that can be: fewer partial sums, tables and prologues. Forward 768
// of 80: two blocks of 384
// (55 424 x 1024 with a gate of tokens, forward and backward: 282 us with 512 a multiprocessor forward, 263 with 768). Few rows
// are spread over all multiprocessors.
static int sw_shape(SandwichArgs& a, bool backward, int mode, unsigned* blocks) {
  if (a.C < 1 || a.C > SW_MAX_C) return -3;
  const int threads = (a.C + 7) / 8;
  a.tpr = (threads + 31) / 32 * 32;
  while (a.tpr / 2 >= threads && a.tpr <= 32 && a.tpr > 1) a.tpr /= 2;      // up to 128 channels: several rows a warp
  const bool wide = !backward && mode != STRIDED && mode != WORDS;
  const int most = wide ? 384 : 512;
  a.groups = a.tpr > most ? 1 : most / a.tpr;
  const long long spread = (a.T + 147) / 148;
  if (a.groups > spread) a.groups = static_cast<int>(spread < 1 ? 1 : spread);
  if (a.tpr < 32) a.groups = (a.groups + 32 / a.tpr - 1) / (32 / a.tpr) * (32 / a.tpr);      // whole warps
  int per_sm = (wide ? 768 : 512) / (a.tpr * a.groups);
  if (per_sm < 1) per_sm = 1;
  const long long all = (a.T + a.groups - 1) / a.groups, room = 148LL * per_sm;
  *blocks = static_cast<unsigned>(all < room ? all : room);
  return 0;
}

// (WORDS: threads without channels read their words of a slot all the same, behind the last slot as well)
static size_t sw_smem_bytes(const SandwichArgs& a, int mode, int rows, int parts, int size) {
  const bool ring = mode != STRIDED || size == 4;
  return static_cast<size_t>(sw_sets(mode, a.C, size, a.groups)) * a.tpr * 8 * 4 * 4 +
         static_cast<size_t>(sw_sums(a.tpr, a.groups)) * 4 +
         (ring ? static_cast<size_t>(a.groups) * a.stages * rows * parts * sw_row_bytes(mode, a.C, size) : 0) +
         (mode == WORDS && size == 2 ? a.tpr * 16 + 16 - std::min<size_t>(a.tpr * 16 + 16, sw_row_bytes(mode, a.C, size)) : 0);
}

template <typename T, int MODE, int GATE, bool SUB>
static int sw_launch(const SandwichArgs& a, bool backward, unsigned blocks, size_t smem, cudaStream_t st) {
  auto kern = backward ? sandwich_bwd_kernel<T, MODE, GATE, SUB> : sandwich_fwd_kernel<T, MODE, GATE, SUB>;
  static bool configured_on[2][MAX_DEVICES];
  const int dev = current_device_slot();
  if (dev < 0) return -4;
  if (!configured_on[backward][dev]) {
    NPLM_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(SW_MAX_SMEM)));
    configured_on[backward][dev] = true;
  }
  const cudaError_t e = launch_when(a.T * a.C <= CHAIN_ELEMENTS, kern, blocks, a.tpr * a.groups, smem, st, a);
  if (e != cudaSuccess) return static_cast<int>(e);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int MODE>
static int sw_launch(const SandwichArgs& a, bool backward, unsigned blocks, size_t smem, cudaStream_t st) {
  if constexpr (MODE != FULL) {      // (which has whole warps)
    if (a.tpr < 32) return sw_launch<T, MODE, GATE_ANY, true>(a, backward, blocks, smem, st);
  }
  if constexpr (MODE == FULL || MODE == WORDS) {
    if (a.gate_mode == GATE_SIGMOID) return sw_launch<T, MODE, GATE_SIGMOID, false>(a, backward, blocks, smem, st);
    if (a.gate_mode == GATE_TOKEN) return sw_launch<T, MODE, GATE_TOKEN, false>(a, backward, blocks, smem, st);
    return sw_launch<T, MODE, GATE_NONE, false>(a, backward, blocks, smem, st);
  } else {
    return sw_launch<T, MODE, GATE_ANY, false>(a, backward, blocks, smem, st);
  }
}

template <typename T>
static int sw_launch(const SandwichArgs& a, bool backward, int mode, unsigned blocks, size_t smem, cudaStream_t st) {
  if (mode == STRIDED) return sw_launch<T, STRIDED>(a, backward, blocks, smem, st);
  if (mode == ALIGNED) return sw_launch<T, ALIGNED>(a, backward, blocks, smem, st);
  if (mode == WORDS) return sw_launch<T, WORDS>(a, backward, blocks, smem, st);
  return sw_launch<T, FULL>(a, backward, blocks, smem, st);
}

static int sw_run(SandwichArgs& a, bool backward, int dtype, unsigned* blocks, cudaStream_t st) {
  const int size = dtype == 2 ? 4 : 2;
  const void* rows[] = {a.x, a.f, a.gate_mode >= GATE_TOKEN ? a.gate : nullptr, a.dy, a.dh, a.y, a.h, a.dx, a.df, a.dg};
  const long long strides[] = {a.xs, a.fs, a.gs, a.dys, a.dhs};
  bool aligned = a.C % 8 == 0, words = true, even = a.C % 2 == 0, odd = !even;
  for (const void* p : rows) {
    aligned &= reinterpret_cast<uintptr_t>(p) % 16 == 0;
    words &= reinterpret_cast<uintptr_t>(p) % 4 == 0;
  }
  for (int k = 0; k < 5; ++k) {      // (the rows that are read)
    if (rows[k] == nullptr) continue;
    aligned &= strides[k] * size % 16 == 0;
    even &= strides[k] % 2 == 0;
    odd &= strides[k] % 2 != 0;
    words &= strides[k] * size >= 16;      // the 16 bytes around an inner row's ends are of the tensor's span
  }
  // (several groups of a warp add up their column sums channel by channel, so they would need one shift)
  words &= size == 4 || even || (odd && a.C > 128);
  const int rows_a_step = backward ? 1 : 2, parts = 2 + (a.gate_mode >= GATE_TOKEN) + (a.dy != nullptr) + (a.dh != nullptr);
  int mode = aligned ? (a.C % 256 == 0 ? FULL : ALIGNED) : words ? WORDS : STRIDED, rc = sw_shape(a, backward, mode, blocks);
  if (rc) return rc;
  a.stages = mode == WORDS ? 3 : SW_STAGES;
  size_t smem = sw_smem_bytes(a, mode, rows_a_step, parts, size);
  if (smem > SW_MAX_SMEM) {
    a.stages -= 1;
    smem = sw_smem_bytes(a, mode, rows_a_step, parts, size);
  }
  if (smem > SW_MAX_SMEM && mode == WORDS) {      // (wide fp32 rows)
    mode = STRIDED;
    rc = sw_shape(a, backward, mode, blocks);
    if (rc) return rc;
    smem = sw_smem_bytes(a, mode, rows_a_step, parts, size);
    if (smem > SW_MAX_SMEM) {
      a.stages = 1;
      smem = sw_smem_bytes(a, mode, rows_a_step, parts, size);
    }
  }
  if (smem > SW_MAX_SMEM) return -3;
  if (!backward) {      // (no more blocks than shared memory holds at a time; 1 KB of it is the system's)
    const unsigned room = 148 * static_cast<unsigned>((SW_MAX_SMEM + 1024) / (smem + 1024));
    if (*blocks > room) *blocks = room;
  }
  const long long next = static_cast<long long>(*blocks) * a.groups;
  a.nx = next * a.xs; a.nf = next * a.fs; a.ng = next * a.gs; a.ndy = next * a.dys; a.ndh = next * a.dhs; a.nout = next * a.C;
  if (dtype == 0) return sw_launch<__nv_bfloat16>(a, backward, mode, *blocks, smem, st);
  if (dtype == 1) return sw_launch<__half>(a, backward, mode, *blocks, smem, st);
  return sw_launch<float>(a, backward, mode, *blocks, smem, st);
}

}  // namespace nplm

using namespace nplm;

// Blocks of nplm_sandwich_bwd, which its partial sums are counted in; negative: no such width.
extern "C" int nplm_sandwich_bwd_blocks(long long T, int C) {
  SandwichArgs a = {};
  a.T = T;
  a.C = C;
  unsigned blocks = 0;
  const int rc = sw_shape(a, true, FULL, &blocks);
  return rc ? rc : static_cast<int>(blocks);
}

// The arguments of a call, packed by the caller (ops/kernels.py has the same layout): one conversion on its side, not 30.
// dtype: 0 bf16, 1 fp16, 2 fp32. gate_mode: 0 none, 1 [C], 2 rows, 3 rows through a sigmoid. strides: rows of x, f, gate, dy, dh.
// stats: fp32 [T][4] for the backward pass, or null. Forward: y, h (null: no norm follows). Backward: dy or dh may be
// null; dx, df, dg; partial: fp32 [4][blocks][C] scratch; sums, kinds: where the column sums of w_next, w_post, the scale and a [C]
// gate go, and as what (see ColumnSums).
struct SandwichCall {
  const void *x, *f, *gate, *post, *next, *scale, *dy, *dh;
  void *y, *h, *dx, *df, *dg;
  float *stats, *partial;
  void* sums[4];
  long long strides[5], T;
  int kinds[4], C, rms, gate_mode, dtype, param32;
  float eps;
};

static int sw_args(const SandwichCall& c, SandwichArgs* out) {
  if (c.T < 0 || c.dtype < 0 || c.dtype > 2 || c.gate_mode < 0 || c.gate_mode > 3 ||
      (c.T > 0 && (c.gate_mode != 0) != (c.gate != nullptr)))
    return -1;
  SandwichArgs a = {};
  a.x = c.x; a.f = c.f; a.gate = c.gate; a.post = c.post; a.next = c.next; a.scale = c.scale; a.dy = c.dy; a.dh = c.dh;
  a.xs = c.strides[0]; a.fs = c.strides[1]; a.gs = c.strides[2]; a.dys = c.strides[3]; a.dhs = c.strides[4];
  a.y = c.y; a.h = c.h; a.dx = c.dx; a.df = c.df; a.dg = c.dg;
  a.stats = reinterpret_cast<float4*>(c.stats); a.partial = c.partial;
  a.T = c.T; a.C = c.C; a.eps = c.eps; a.rms = c.rms; a.gate_mode = c.gate_mode; a.param32 = c.param32;
  *out = a;
  return 0;
}

extern "C" int nplm_sandwich_fwd(const SandwichCall* call, cudaStream_t st) {
  SandwichArgs a;
  const int rc = sw_args(*call, &a);
  if (rc || a.T == 0) return rc;
  unsigned blocks;
  return sw_run(a, false, call->dtype, &blocks, st);
}

extern "C" int nplm_sandwich_bwd(const SandwichCall* call, cudaStream_t st) {
  SandwichArgs a;
  const int rc = sw_args(*call, &a);
  if (rc) return rc;
  if (a.T > 0 && a.dy == nullptr && a.dh == nullptr) return -1;
  ColumnSums to;
  for (int k = 0; k < 4; ++k) {
    to.out[k] = call->sums[k];
    to.kind[k] = call->kinds[k];
    if (to.kind[k]) a.want |= 1 << k;
  }
  unsigned blocks = 0;      // (no rows: the column sums are zero)
  if (a.T > 0) {
    const int rc2 = sw_run(a, true, call->dtype, &blocks, st);
    if (rc2) return rc2;
  }
  if (a.want) {
    const cudaError_t e = launch_chained(sandwich_columns_kernel, dim3((a.C + 31) / 32, 4), dim3(32, 32), 0, st,
                                         static_cast<const float*>(a.partial), to, static_cast<int>(blocks), a.C);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return static_cast<int>(cudaGetLastError());
}
