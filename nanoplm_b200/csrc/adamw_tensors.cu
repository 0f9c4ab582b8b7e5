// One AdamW step over all tensors of a model in one launch (128 tensors a launch), moments in fp32 or in 8 bits.
//
//   g' = s g,  m <- b1 m + (1 - b1) g',  v <- b2 v + (1 - b2) g'^2,
//   p <- (1 - lr wd) p - (lr / bc1) m / (sqrt(v) / sqrt(bc2) + eps),   s = gradient scale and clipping by the global norm
//
// 8-bit moments. 256 consecutive elements of a tensor are a block, and a tensor starts a block. A moment's code is the top of
// its fp32 pattern (exponent and 3 bits of mantissa) less an offset that the block shares: with E the exponent field of
// (pattern of the block's largest magnitude + 2^20 - 1), which no rounding of the block exceeds,
//   second moment: ((pattern + r) >> 20) - 8 max(E - 31, 0), 8 bits: 32 octaves below the block's largest; 0 is zero
//   first moment:  ((pattern + r) >> 20) - 8 max(E - 15, 0), 7 bits below the sign: 16 octaves
// r is a random number of 20 bits: the rounding is stochastic and the kept value the true one on average. Neighbouring codes are 6
// to 12 % apart while an average with b2 = 0.999 moves by 0.1 % a step, so rounding to the nearest code would never move it.
// A second moment below code 1 is kept as code 1 (a zero would let its element step by m / eps), a first moment there as code 1
// or zero, with the probability that keeps its mean. Codes are shifted patterns, so reading back and coding again gives the
// same values whatever r. All of m, v and their codes is computed with separately rounded operations in the order of
// the formulas, and gives the bits of the restatement in ops/moments.py; the quotient of p is not.
//
// Bound by memory: fp32 weights and gradients with a bf16 copy move 18 bytes an element with 8-bit moments (p 4 + 4, g 4, copy 2,
// codes 4, and 4 bytes a block) and 30 with fp32 ones. A warp takes a block: the block's largest pattern is then one
// integer reduction a moment, and a lane has twice 4 consecutive elements, so that every access of a warp is contiguous. The
// table of tensors travels in the launch's parameters: nothing is kept between calls, and a captured launch has its own.
#include "common.cuh"

namespace nplm {

constexpr int AT_BLOCK = 256;        // elements that share an offset
constexpr int AT_TENSORS = 128;      // tensors a launch
constexpr int AT_CHUNK = 32;         // blocks of one tensor that a thread block takes
constexpr int AT_WARPS = 8;

struct AdamTensors {
  void* p[AT_TENSORS];
  const void* g[AT_TENSORS];
  void* copy[AT_TENSORS];
  long long numel[AT_TENSORS];
  long long block[AT_TENSORS];         // first block of the tensor in the moments
  int chunk[AT_TENSORS + 1];           // first chunk of the tensor in this launch
  unsigned char flags[AT_TENSORS];     // 1: weight decay, 2: all addresses on 16 bytes
  int n;
};

// A 32-bit mix with two multiplications and three shifts (Wellons, "Prospecting for hash functions", 2018).
__device__ __forceinline__ uint32_t at_mix(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x7feb352du;
  x = (x ^ (x >> 15)) * 0x846ca68bu;
  return x ^ (x >> 16);
}

template <bool SIGNED>
__device__ __forceinline__ uint32_t at_base(uint32_t e) {      // offset of the block's codes
  constexpr uint32_t below = SIGNED ? 15 : 31;
  return (e > below ? e - below : 0u) << 3;
}
template <bool SIGNED>
__device__ __forceinline__ float at_decode(uint32_t code, uint32_t base) {
  const uint32_t low = SIGNED ? code & 127u : code;
  const uint32_t bits = low ? (low + base) << 20 : 0u;
  return __uint_as_float(SIGNED ? bits | (code & 128u) << 24 : bits);
}
template <bool SIGNED>
__device__ __forceinline__ uint32_t at_encode(float x, uint32_t base, uint32_t r) {
  const uint32_t bits = __float_as_uint(x) & 0x7fffffffu;
  if (bits == 0u) return 0u;
  const uint32_t least = (base + 1u) << 20;       // the pattern of code 1
  uint32_t code = ((bits + r) >> 20) - base;
  if (bits < least) {
    if (!SIGNED) return 1u;
    code = __fmul_rn(static_cast<float>(r), __fmul_rn(__uint_as_float(least), 9.5367431640625e-7f)) < fabsf(x) ? 1u : 0u;
  }
  return SIGNED && code ? code | (__float_as_uint(x) >> 24 & 128u) : code;
}
__device__ __forceinline__ uint32_t at_exponent(uint32_t largest) { return (largest + 0xfffffu) >> 23; }

template <typename T>
__device__ __forceinline__ float at_get(T v);
template <>
__device__ __forceinline__ float at_get<float>(float v) { return v; }
template <>
__device__ __forceinline__ float at_get<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T at_put(float v);
template <>
__device__ __forceinline__ float at_put<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 at_put<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int N>
struct alignas(sizeof(T) * N) AtVec {
  T v[N];
};

// The eight elements of a lane in a block. VEC: two runs of four, the block whole and every address on its multiples;
// else every 32nd, as far as the tensor goes.
template <bool VEC>
__device__ __forceinline__ int at_place(int lane, int e) { return VEC ? (e >> 2) * 128 + lane * 4 + (e & 3) : e * 32 + lane; }
template <bool VEC, typename T>
__device__ __forceinline__ void at_load(const T* p, int lane, int n, T (&v)[8]) {
  if (VEC) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const AtVec<T, 4> t = *reinterpret_cast<const AtVec<T, 4>*>(p + j * 128 + lane * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j * 4 + e] = t.v[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e * 32 + lane < n ? p[e * 32 + lane] : T(0.f);
  }
}
template <bool VEC, typename T>
__device__ __forceinline__ void at_store(T* p, int lane, int n, const T (&v)[8]) {
  if (VEC) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      AtVec<T, 4> t;
#pragma unroll
      for (int e = 0; e < 4; ++e) t.v[e] = v[j * 4 + e];
      *reinterpret_cast<AtVec<T, 4>*>(p + j * 128 + lane * 4) = t;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e * 32 + lane < n) p[e * 32 + lane] = v[e];
  }
}

struct AdamScalars {
  float b1, b2, c1, c2, eps, decay, step, inv_bc2, scale;
  uint32_t key;
};

// One block of a tensor: elements [0, n), their place `at` in the moments' buffers.
template <typename P, typename G, int BITS, bool VEC>
__device__ __forceinline__ void at_block(P* p, const G* g, __nv_bfloat16* copy, int n, void* m_all, void* v_all,
                                         uint8_t* scales, long long blocks, long long block, const AdamScalars& s, bool decays,
                                         int lane) {
  const long long at = block * AT_BLOCK;
  P pv[8];
  G gv[8];
  float m[8], v[8];
  at_load<VEC>(p, lane, n, pv);
  at_load<VEC>(g, lane, n, gv);
  if (BITS == 8) {
    uint8_t *mc = static_cast<uint8_t*>(m_all) + at, *vc = static_cast<uint8_t*>(v_all) + at;
    const uint32_t bm = at_base<true>(scales[block]), bv = at_base<false>(scales[blocks + block]);
    uint8_t cm[8], cv[8];   // (the codes' own buffers are whole blocks on multiples of 16)
    if (VEC) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t a = *reinterpret_cast<const uint32_t*>(mc + j * 128 + lane * 4);
        const uint32_t b = *reinterpret_cast<const uint32_t*>(vc + j * 128 + lane * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          cm[j * 4 + e] = a >> 8 * e & 255u;
          cv[j * 4 + e] = b >> 8 * e & 255u;
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        cm[e] = mc[e * 32 + lane];
        cv[e] = vc[e * 32 + lane];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      m[e] = at_decode<true>(cm[e], bm);
      v[e] = at_decode<false>(cv[e], bv);
    }
  } else {
    at_load<VEC>(static_cast<const float*>(m_all) + at, lane, n, m);
    at_load<VEC>(static_cast<const float*>(v_all) + at, lane, n, v);
  }
  __nv_bfloat16 half[8];
  uint32_t top_m = 0, top_v = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float gr = __fmul_rn(at_get<G>(gv[e]), s.scale);
    m[e] = __fadd_rn(__fmul_rn(m[e], s.b1), __fmul_rn(gr, s.c1));
    v[e] = __fadd_rn(__fmul_rn(v[e], s.b2), __fmul_rn(__fmul_rn(gr, gr), s.c2));
    if (!VEC && at_place<VEC>(lane, e) >= n) m[e] = v[e] = 0.f;     // behind the tensor: stays zero
    float root;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v[e]));
    const float step = __fdividef(m[e], fmaf(root, s.inv_bc2, s.eps));
    const float pn = fmaf(-s.step, step, __fmul_rn(at_get<P>(pv[e]), decays ? s.decay : 1.f));
    pv[e] = at_put<P>(pn);
    half[e] = at_put<__nv_bfloat16>(pn);
    if (BITS == 8) {
      top_m = max(top_m, __float_as_uint(m[e]) & 0x7fffffffu);
      top_v = max(top_v, __float_as_uint(v[e]) & 0x7fffffffu);
    }
  }
  at_store<VEC>(p, lane, n, pv);
  if (copy != nullptr) at_store<VEC>(copy, lane, n, half);
  if (BITS == 8) {
    uint8_t *mc = static_cast<uint8_t*>(m_all) + at, *vc = static_cast<uint8_t*>(v_all) + at;
    const uint32_t em = at_exponent(__reduce_max_sync(0xffffffffu, top_m)), ev = at_exponent(__reduce_max_sync(0xffffffffu, top_v));
    const uint32_t bm = at_base<true>(em), bv = at_base<false>(ev);
    const uint32_t key = at_mix(s.key + static_cast<uint32_t>(at >> 32)), low = static_cast<uint32_t>(at);
    uint32_t cm[8], cv[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t r = at_mix((low + at_place<VEC>(lane, e)) ^ key);
      cm[e] = at_encode<true>(m[e], bm, r & 0xfffffu);
      cv[e] = at_encode<false>(v[e], bv, r >> 12);
    }
    if (VEC) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        *reinterpret_cast<uint32_t*>(mc + j * 128 + lane * 4) =
            cm[j * 4] | cm[j * 4 + 1] << 8 | cm[j * 4 + 2] << 16 | cm[j * 4 + 3] << 24;
        *reinterpret_cast<uint32_t*>(vc + j * 128 + lane * 4) =
            cv[j * 4] | cv[j * 4 + 1] << 8 | cv[j * 4 + 2] << 16 | cv[j * 4 + 3] << 24;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        mc[e * 32 + lane] = static_cast<uint8_t>(cm[e]);
        vc[e * 32 + lane] = static_cast<uint8_t>(cv[e]);
      }
    }
    if (lane == 0) {
      scales[block] = static_cast<uint8_t>(em);
      scales[blocks + block] = static_cast<uint8_t>(ev);
    }
  } else {
    at_store<VEC>(static_cast<float*>(m_all) + at, lane, n, m);
    at_store<VEC>(static_cast<float*>(v_all) + at, lane, n, v);
  }
}

// hyper: [lr, beta1, beta2, eps, weight_decay, bias_corr1, bias_corr2, grad_scale, max_norm]; rng: one 64-bit number, another one
// each step. Both in device memory, so that a captured step sees their values at its replay.
template <typename P, typename G, int BITS>
__global__ void __launch_bounds__(AT_WARPS * 32)
adamw_tensors_kernel(const __grid_constant__ AdamTensors t, void* m_all, void* v_all, uint8_t* scales, long long blocks,
                     const float* __restrict__ hyper, const float* __restrict__ sumsq, const long long* __restrict__ rng) {
  grid_chain();
  const int chunk = blockIdx.x, lane = threadIdx.x & 31;
  int lo = 0, hi = t.n;                 // the last tensor that starts at or before this chunk
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.chunk[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  AdamScalars s;
  const float lr = hyper[0], gs = hyper[7], most = hyper[8];
  s.b1 = hyper[1];
  s.b2 = hyper[2];
  s.c1 = 1.f - s.b1;
  s.c2 = 1.f - s.b2;
  s.eps = hyper[3];
  s.decay = __fsub_rn(1.f, __fmul_rn(lr, hyper[4]));
  s.step = lr / hyper[5];
  s.inv_bc2 = 1.f / sqrtf(hyper[6]);
  s.scale = gs;
  if (sumsq != nullptr && most > 0.f) {
    const float norm = __fmul_rn(sqrtf(*sumsq), gs);
    s.scale = __fmul_rn(gs, fminf(most / __fadd_rn(norm, 1e-6f), 1.f));
  }
  s.key = 0;
  if (BITS == 8) {
    const unsigned long long seed = static_cast<unsigned long long>(*rng);
    s.key = at_mix(static_cast<uint32_t>(seed) ^ at_mix(static_cast<uint32_t>(seed >> 32)));
  }
  const long long numel = t.numel[lo];
  const bool decays = t.flags[lo] & 1, aligned = t.flags[lo] & 2;
  const long long first = static_cast<long long>(chunk - t.chunk[lo]) * AT_CHUNK;
  P* p = static_cast<P*>(t.p[lo]);
  const G* g = static_cast<const G*>(t.g[lo]);
  __nv_bfloat16* copy = static_cast<__nv_bfloat16*>(t.copy[lo]);
  for (int j = threadIdx.x >> 5; j < AT_CHUNK; j += AT_WARPS) {
    const long long at = (first + j) * AT_BLOCK, left = numel - at;
    if (left <= 0) return;
    const int n = static_cast<int>(left < AT_BLOCK ? left : AT_BLOCK);
    __nv_bfloat16* c = copy == nullptr ? nullptr : copy + at;
    if (aligned && n == AT_BLOCK)
      at_block<P, G, BITS, true>(p + at, g + at, c, n, m_all, v_all, scales, blocks, t.block[lo] + first + j, s, decays, lane);
    else
      at_block<P, G, BITS, false>(p + at, g + at, c, n, m_all, v_all, scales, blocks, t.block[lo] + first + j, s, decays, lane);
  }
}

// The values of all codes, both moments in one launch: four codes a thread.
template <typename O>
__global__ void __launch_bounds__(256)
moment_values_kernel(const uint32_t* __restrict__ mc, const uint32_t* __restrict__ vc, const uint8_t* __restrict__ scales,
                     long long blocks, O* __restrict__ m, O* __restrict__ v) {
  grid_chain();
  const long long n = blocks * (AT_BLOCK / 4);
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += gridDim.x * 256LL) {
    const long long block = i / (AT_BLOCK / 4);
    const uint32_t a = mc[i], b = vc[i];
    const uint32_t bm = at_base<true>(scales[block]), bv = at_base<false>(scales[blocks + block]);
    AtVec<O, 4> x, y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x.v[e] = at_put<O>(at_decode<true>(a >> 8 * e & 255u, bm));
      y.v[e] = at_put<O>(at_decode<false>(b >> 8 * e & 255u, bv));
    }
    *reinterpret_cast<AtVec<O, 4>*>(m + i * 4) = x;
    *reinterpret_cast<AtVec<O, 4>*>(v + i * 4) = y;
  }
}

// The codes of fp32 moments, rounded to the nearest (r = half a step): a warp a block.
__global__ void __launch_bounds__(256)
moment_codes_kernel(const float* __restrict__ m, const float* __restrict__ v, uint8_t* __restrict__ mc, uint8_t* __restrict__ vc,
                    uint8_t* __restrict__ scales, long long blocks) {
  grid_chain();
  const int lane = threadIdx.x & 31;
  for (long long block = blockIdx.x * 8LL + (threadIdx.x >> 5); block < blocks; block += gridDim.x * 8LL) {
    const long long at = block * AT_BLOCK;
    float x[8], y[8];
    at_load<true>(m + at, lane, AT_BLOCK, x);
    at_load<true>(v + at, lane, AT_BLOCK, y);
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top_m = max(top_m, __float_as_uint(x[e]) & 0x7fffffffu);
      top_v = max(top_v, __float_as_uint(y[e]) & 0x7fffffffu);
    }
    const uint32_t em = at_exponent(__reduce_max_sync(0xffffffffu, top_m)), ev = at_exponent(__reduce_max_sync(0xffffffffu, top_v));
    const uint32_t bm = at_base<true>(em), bv = at_base<false>(ev);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t a = 0, b = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a |= at_encode<true>(x[j * 4 + e], bm, 0x80000u) << 8 * e;
        b |= at_encode<false>(y[j * 4 + e], bv, 0x80000u) << 8 * e;
      }
      *reinterpret_cast<uint32_t*>(mc + at + j * 128 + lane * 4) = a;
      *reinterpret_cast<uint32_t*>(vc + at + j * 128 + lane * 4) = b;
    }
    if (lane == 0) {
      scales[block] = static_cast<uint8_t>(em);
      scales[blocks + block] = static_cast<uint8_t>(ev);
    }
  }
}

template <typename P, typename G>
static cudaError_t at_launch(const AdamTensors& t, int bits, long long elements, void* m, void* v, uint8_t* scales,
                             long long blocks, const float* hyper, const float* sumsq, const long long* rng, cudaStream_t st) {
  const int grid = t.chunk[t.n];
  const bool chained = elements <= CHAIN_ELEMENTS;
  if (bits == 8)
    return launch_when(chained, adamw_tensors_kernel<P, G, 8>, grid, AT_WARPS * 32, 0, st, t, m, v, scales, blocks, hyper, sumsq, rng);
  return launch_when(chained, adamw_tensors_kernel<P, G, 32>, grid, AT_WARPS * 32, 0, st, t, m, v, scales, blocks, hyper, sumsq, rng);
}

}  // namespace nplm

using namespace nplm;

// n tensors: p, g, copy (a null entry, or copy itself null: none), numel, first block in the moments, decay. p_type, g_type: 0
// bf16, 2 fp32; copies are bf16. bits 8: m, v uint8 [blocks][256], scales uint8 [2][blocks]; 32: m, v fp32 [blocks][256].
extern "C" int nplm_adamw_tensors(void* const* p, const void* const* g, void* const* copy, const long long* numel,
                                  const long long* block, const unsigned char* decay, int n, int p_type, int g_type, int bits,
                                  void* m, void* v, void* scales, long long blocks, const float* hyper, const float* sumsq,
                                  const long long* rng, cudaStream_t st) {
  if (n < 0 || (p_type != 0 && p_type != 2) || (g_type != 0 && g_type != 2) || (bits != 8 && bits != 32)) return -1;
  if (bits == 8 && (scales == nullptr || rng == nullptr)) return -1;
  AdamTensors t;
  int i = 0;
  while (i < n) {
    t.n = 0;
    t.chunk[0] = 0;
    long long chunks = 0, elements = 0;
    for (; i < n && t.n < AT_TENSORS; ++i) {
      if (numel[i] == 0) continue;
      const long long has = (numel[i] + AT_BLOCK - 1) / AT_BLOCK;
      if (numel[i] < 0 || block[i] < 0 || block[i] + has > blocks) return -2;
      const long long more = (has + AT_CHUNK - 1) / AT_CHUNK;
      if (more > 0x7fffffffLL) return -2;
      if (chunks + more > 0x7fffffffLL) break;    // the rest in another launch
      const int k = t.n++;
      t.p[k] = p[i];
      t.g[k] = g[i];
      t.copy[k] = copy == nullptr ? nullptr : copy[i];
      t.numel[k] = numel[i];
      t.block[k] = block[i];
      chunks += more;
      elements += numel[i];
      t.chunk[t.n] = static_cast<int>(chunks);
      const uintptr_t all = reinterpret_cast<uintptr_t>(t.p[k]) | reinterpret_cast<uintptr_t>(t.g[k]) |
                            reinterpret_cast<uintptr_t>(t.copy[k]);
      t.flags[k] = (decay[i] ? 1 : 0) | (all % 16 == 0 ? 2 : 0);
    }
    if (t.n == 0) break;
    uint8_t* sc = static_cast<uint8_t*>(scales);
    cudaError_t e;
    if (p_type == 2 && g_type == 2) e = at_launch<float, float>(t, bits, elements, m, v, sc, blocks, hyper, sumsq, rng, st);
    else if (p_type == 2) e = at_launch<float, __nv_bfloat16>(t, bits, elements, m, v, sc, blocks, hyper, sumsq, rng, st);
    else if (g_type == 2) e = at_launch<__nv_bfloat16, float>(t, bits, elements, m, v, sc, blocks, hyper, sumsq, rng, st);
    else e = at_launch<__nv_bfloat16, __nv_bfloat16>(t, bits, elements, m, v, sc, blocks, hyper, sumsq, rng, st);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return static_cast<int>(cudaGetLastError());
}

static int at_grid(long long blocks, int of) {
  const long long b = (blocks + of - 1) / of;
  return static_cast<int>(b < 148LL * 32 ? b : 148LL * 32);
}

// out_type: 0 bf16, 2 fp32.
extern "C" int nplm_moment_values(const void* mc, const void* vc, const void* scales, long long blocks, void* m, void* v,
                                  int out_type, cudaStream_t st) {
  if (blocks < 0 || (out_type != 0 && out_type != 2)) return -1;
  if (blocks == 0) return 0;
  const uint32_t *a = static_cast<const uint32_t*>(mc), *b = static_cast<const uint32_t*>(vc);
  const uint8_t* s = static_cast<const uint8_t*>(scales);
  const bool chained = blocks * AT_BLOCK <= CHAIN_ELEMENTS;
  const cudaError_t e =
      out_type == 2 ? launch_when(chained, moment_values_kernel<float>, at_grid(blocks, 4), 256, 0, st, a, b, s, blocks,
                                  static_cast<float*>(m), static_cast<float*>(v))
                    : launch_when(chained, moment_values_kernel<__nv_bfloat16>, at_grid(blocks, 4), 256, 0, st, a, b, s, blocks,
                                  static_cast<__nv_bfloat16*>(m), static_cast<__nv_bfloat16*>(v));
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

extern "C" int nplm_moment_codes(const float* m, const float* v, void* mc, void* vc, void* scales, long long blocks,
                                 cudaStream_t st) {
  if (blocks < 0) return -1;
  if (blocks == 0) return 0;
  const cudaError_t e = launch_when(blocks * AT_BLOCK <= CHAIN_ELEMENTS, moment_codes_kernel, at_grid(blocks, 8), 256, 0, st, m, v,
                                    static_cast<uint8_t*>(mc), static_cast<uint8_t*>(vc), static_cast<uint8_t*>(scales), blocks);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}
