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
// the formulas, and gives the bits of the restatement in ops/moments.py; the quotient of p is not (see at_weights).
//
// Bound by memory: fp32 weights and gradients with a bf16 copy move 18 bytes an element with 8-bit moments (p 4 + 4, g 4, copy 2,
// codes 4, and 4 bytes a block) and 30 with fp32 ones. A warp takes a block: the block's largest pattern is then one
// integer reduction a moment, and a lane has twice 4 consecutive elements, so that every access of a warp is contiguous. The
// table of tensors travels in the launch's parameters: nothing is kept between calls, and a captured launch has its own.
//
// Measured: 114 M elements, fp32 gradients and a bf16 copy: 8-bit moments 307 us (6.7 TB/s, the copy rate, with an instruction issued
// in 83 % of the cycles), with their values read back 420 us, and 436 where one step with one set of random numbers has been
// repeated until most first moments are below code 1; fp32 moments 510 us (6.7 TB/s). 32 M bf16 weights and gradients at
// addresses off 16 bytes, 8-bit moments and their values: 132 us, 3.4 TB/s, bound by instructions (one issued in 89 % of the
// cycles): as many an element as fp32 weights take, beside 14 instead of 22 bytes. (By single elements from and to memory 139.)
#include "common.cuh"

namespace nplm {

constexpr int AT_BLOCK = 256;        // elements that share an offset
constexpr int AT_TENSORS = 128;      // tensors a launch
constexpr int AT_WARPS = 8;
constexpr int AT_CHUNK = 4 * AT_WARPS;    // most blocks of one tensor that a thread block takes, its warps side by side
constexpr int AT_STAGES = 2;         // blocks of a warp in shared memory: the one it works on and the next

static_assert(AT_CHUNK <= 32, "a lane an exponent");

struct AdamTensors {
  void* p[AT_TENSORS];
  const void* g[AT_TENSORS];
  void* copy[AT_TENSORS];
  long long numel[AT_TENSORS];
  long long block[AT_TENSORS];         // first block of the tensor in the moments
  int chunk[AT_TENSORS + 1];           // first chunk of the tensor in this launch
  unsigned char flags[AT_TENSORS];     // 1: weight decay, 2: all addresses on 16 bytes
  int n, per_chunk;
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
__device__ __forceinline__ uint32_t at_exponent(uint32_t largest) { return (min(largest, 0x7f800000u) + 0xfffffu) >> 23; }

// Bytes of a (0 - 3) and b (4 - 7).
template <uint32_t SELECT>
__device__ __forceinline__ uint32_t at_bytes(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "n"(SELECT));
  return d;
}

// Four codes as values. bottom: the block's offset << 20. A code's byte moves to bits 20 - 27 (with one byte selection and one
// multiplication, which leaves the integer pipe, the busiest one here, to the rest) and the offset is added; zeros are few and set apart.
template <bool SIGNED>
__device__ __forceinline__ void at_decode(uint32_t four, uint32_t bottom, float* x) {
  const uint32_t low = SIGNED ? four & 0x7f7f7f7fu : four;
  uint32_t bits[4] = {at_bytes<0x4044>(low, 0u) * 16u + bottom, at_bytes<0x4144>(low, 0u) * 16u + bottom,
                      at_bytes<0x4244>(low, 0u) * 16u + bottom, at_bytes<0x4344>(low, 0u) * 16u + bottom};
  if (SIGNED) {
    bits[0] |= four << 24 & 0x80000000u;
    bits[1] |= four << 16 & 0x80000000u;
    bits[2] |= four << 8 & 0x80000000u;
    bits[3] |= four & 0x80000000u;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(bits[e]);
  const bool zeros = SIGNED ? ((low + 0x7f7f7f7fu) & 0x80808080u) != 0x80808080u : ((low - 0x01010101u) & ~low & 0x80808080u) != 0u;
  if (zeros) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if ((low >> 8 * e & 255u) == 0u) x[e] = 0.f;
  }
}

// The codes of four values, whatever they are: zero is 0, a second moment below code 1 is 1, a first moment there 1 or 0 with its
// mean kept. r: random numbers of 20 bits.
template <bool SIGNED>
__device__ __forceinline__ uint32_t at_codes(const float* x, const uint32_t* r, uint32_t bottom) {
  const uint32_t least = bottom + 0x100000u;      // the pattern of code 1
  const float step = __fmul_rn(__uint_as_float(least), 9.5367431640625e-7f);    // 2^-20 of it
  uint32_t four = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t bits = __float_as_uint(x[e]) & 0x7fffffffu;
    uint32_t code = (bits + r[e] - bottom) >> 20;
    if (bits < least) code = bits == 0u ? 0u : !SIGNED ? 1u : __fmul_rn(static_cast<float>(r[e]), step) < __uint_as_float(bits);
    if (SIGNED && code) code |= __float_as_uint(x[e]) >> 24 & 128u;
    four |= code << 8 * e;
  }
  return four;
}

// The same for values of at least code 1 in a block with an exponent E that at_plain admits. Times 2^(96 - the block's lowest
// exponent), an exact product, a value's pattern is 96 x 8 + code on bits 20 and up, and 96 x 8 = 0 modulo 256: no offset is
// left to subtract, nor a sign to cut off, where the pattern is moved up by 4 bits and its top byte taken.
constexpr int AT_OCTAVE = 96;
template <bool SIGNED>
__device__ __forceinline__ bool at_plain(uint32_t e) {
  // 2^(96 - lowest) is a number, and the lowest codes are of the normal range (with E at `below` they are patterns of subnormal numbers,
  // which a product does not move by octaves)
  constexpr uint32_t below = SIGNED ? 15 : 31;
  return e - below - 1u < AT_OCTAVE + 125u;
}
template <bool SIGNED>
__device__ __forceinline__ float at_lift(uint32_t e) {
  return __uint_as_float((AT_OCTAVE + 127u + (SIGNED ? 15 : 31) - e) << 23);
}
constexpr float AT_LEAST = 5.2386894822120667e-10f;           // 1.125 x 2^-31: code 1, lifted
__device__ __forceinline__ uint32_t at_top_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return at_bytes<0x5410>(at_bytes<0x0073>(a, b), at_bytes<0x0073>(c, d));
}

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

// A lane has two runs of four elements of a block, 128 apart. vec: the block is whole and every address on its multiples; else
// element by element, as far as the tensor goes.
__device__ __forceinline__ int at_place(int lane, int e) { return (e >> 2) * 128 + lane * 4 + (e & 3); }
template <typename T>
__device__ __forceinline__ void at_load(const T* p, int lane, int n, bool vec, T (&v)[8]) {
  if (vec) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const AtVec<T, 4> t = *reinterpret_cast<const AtVec<T, 4>*>(p + j * 128 + lane * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j * 4 + e] = t.v[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = at_place(lane, e) < n ? p[at_place(lane, e)] : T(0.f);
  }
}
template <typename T>
__device__ __forceinline__ void at_store(T* p, int lane, int n, bool vec, const T (&v)[8]) {
  if (vec) {
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
      if (at_place(lane, e) < n) p[at_place(lane, e)] = v[e];
  }
}

struct AdamScalars {
  float b1, b2, c1, c2, eps, decay, step, inv_bc2, scale;
  uint32_t key;
};

__device__ __forceinline__ float2 at_both(float v) { return make_float2(v, v); }

__device__ __forceinline__ void at_copy_16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
template <typename T>
__device__ __forceinline__ void at_fetch(T* to, const T* from, int lane) {      // a whole block, on 16 bytes
#pragma unroll
  for (int j = 0; j < static_cast<int>(sizeof(T) * AT_BLOCK); j += 512)
    if (j + lane * 16 < static_cast<int>(sizeof(T) * AT_BLOCK))
      at_copy_16(reinterpret_cast<char*>(to) + j + lane * 16, reinterpret_cast<const char*>(from) + j + lane * 16);
}

// Whether a 16-bit tensor starts in the middle of a word: shared memory then holds its blocks one element on, so that words of either
// side are words of the other.
template <typename T>
__device__ __forceinline__ int at_shift(const T* p) {
  return sizeof(T) == 2 ? static_cast<int>(reinterpret_cast<uintptr_t>(p) >> 1) & 1 : 0;
}
// A whole block in words; with a shift the first one holds the element before the block, too, and the last one is read by half.
template <typename T>
__device__ __forceinline__ void at_fetch_words(T* to, const T* from, int shift, int lane) {
  constexpr int words = AT_BLOCK * static_cast<int>(sizeof(T)) / 4;
  const char* src = reinterpret_cast<const char*>(from - shift);
  char* dst = reinterpret_cast<char*>(to);
#pragma unroll
  for (int i = 0; i < words; i += 32)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst + 4 * (i + lane))), "l"(src + 4 * (i + lane)) : "memory");
  if (shift && lane == 0)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, 2;" ::"r"(smem_u32(dst + 4 * words)), "l"(src + 4 * words) : "memory");
}
// n elements of a block from shared memory (`from`, with the shift of `to`) to where they belong, lane beside lane.
template <typename T>
__device__ __forceinline__ void at_spread(T* to, const T* from, int shift, int n, int lane) {
  if (sizeof(T) == 2 && n == AT_BLOCK) {
    uint32_t* w = reinterpret_cast<uint32_t*>(to - shift);
    const uint32_t* r = reinterpret_cast<const uint32_t*>(from);
#pragma unroll
    for (int i = 0; i < AT_BLOCK / 2; i += 32)
      if (i + lane >= shift) w[i + lane] = r[i + lane];
    if (shift && lane < 2) to[lane * (AT_BLOCK - 1)] = from[shift + lane * (AT_BLOCK - 1)];
  } else {
#pragma unroll
    for (int i = 0; i < AT_BLOCK; i += 32)
      if (i + lane < n) to[i + lane] = from[shift + i + lane];
  }
}

// A block of a tensor with 8-bit moments in shared memory, with room for a shift.
template <typename P, typename G>
struct alignas(16) AtStage {
  P p[AT_BLOCK + 8];
  G g[AT_BLOCK + 8];
  uint8_t m[AT_BLOCK], v[AT_BLOCK];
};

// A block of a tensor.
template <typename P, typename G>
struct AtPlace {
  P* p;
  const G* g;
  __nv_bfloat16* copy;        // or null
  int rest;                   // elements from here to the end of the thread block's chunk, or of the tensor where that comes first
  int block;                  // in the moments
  bool aligned, decays, begins;      // begins: the tensor's first block
  __device__ __forceinline__ int n() const { return rest < AT_BLOCK ? rest : AT_BLOCK; }
  __device__ __forceinline__ bool vec() const { return aligned && rest >= AT_BLOCK; }
  __device__ __forceinline__ void find(const AdamTensors& t, int chunk, int warp) {
    int lo = 0, hi = t.n;     // the last tensor that starts at or before this chunk
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (t.chunk[mid] <= chunk) lo = mid;
      else hi = mid;
    }
    const int off = (chunk - t.chunk[lo]) * t.per_chunk + warp;
    const long long at = static_cast<long long>(off) * AT_BLOCK, left = t.numel[lo] - at;
    const int most = (t.per_chunk - warp) * AT_BLOCK;
    rest = left < most ? static_cast<int>(left) : most;
    block = static_cast<int>(t.block[lo]) + off;
    p = static_cast<P*>(t.p[lo]) + at;
    g = static_cast<const G*>(t.g[lo]) + at;
    copy = static_cast<__nv_bfloat16*>(t.copy[lo]);
    if (copy != nullptr) copy += at;
    decays = t.flags[lo] & 1;
    aligned = t.flags[lo] & 2;
    begins = off == 0;
  }
  // The warp's next block of the chunk; false behind the last.
  __device__ __forceinline__ bool next() {
    constexpr int step = AT_WARPS * AT_BLOCK;
    rest -= step;
    p += step;
    g += step;
    if (copy != nullptr) copy += step;
    block += AT_WARPS;
    return rest > 0;
  }
};

// The moments and the weights of a lane's eight elements.
__device__ __forceinline__ void at_moments(const float (&g)[8], float (&m)[8], float (&v)[8], const AdamScalars& s) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {      // products in pairs; a packed sum of them would become one rounding
    const float2 gr = mul2(make_float2(g[e], g[e + 1]), at_both(s.scale));
    const float2 m0 = mul2(make_float2(m[e], m[e + 1]), at_both(s.b1)), m1 = mul2(gr, at_both(s.c1));
    const float2 v0 = mul2(make_float2(v[e], v[e + 1]), at_both(s.b2)), v1 = mul2(mul2(gr, gr), at_both(s.c2));
    m[e] = __fadd_rn(m0.x, m1.x);
    m[e + 1] = __fadd_rn(m0.y, m1.y);
    v[e] = __fadd_rn(v0.x, v1.x);
    v[e + 1] = __fadd_rn(v0.y, v1.y);
  }
}
// pv: the weights, old and then new; half: their copies. s.decay: the tensor's. Root and reciprocal are the approximate ones (2^-23 of
// the value each): the update is good to 2^-20 of itself, and its sum with the weight is rounded to the weight's type.
template <typename P>
__device__ __forceinline__ void at_weights(P (&pv)[8], const float (&m)[8], const float (&v)[8], __nv_bfloat16 (&half)[8], const AdamScalars& s) {
  float root[8];
  // (The root of a second moment below fp32's normal range, 2^-63, is under 2^-25 of such an eps where bias correction 2 is 2e-5 or more,
  // under 2^-21 where it is the smallest that 1 - beta2 can be. A bound on eps / inv_bc2 instead: 422 -> 444 us, by what the compiler
  // makes of the rest.)
  if (s.eps >= 1e-9f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root[e]) : "f"(v[e]));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) asm("sqrt.approx.f32 %0, %1;" : "=f"(root[e]) : "f"(v[e]));
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(fmaf(root[e], s.inv_bc2, s.eps)));
    const float pn = fmaf(-s.step, m[e] * inv, __fmul_rn(at_get<P>(pv[e]), s.decay));
    pv[e] = at_put<P>(pn);
    half[e] = at_put<__nv_bfloat16>(pn);
  }
}

// A block with fp32 moments.
template <typename P, typename G>
__device__ __forceinline__ void at_block(const AtPlace<P, G>& at, float* m_all, float* v_all, const AdamScalars& s, int lane) {
  float *mp = m_all + static_cast<long long>(at.block) * AT_BLOCK, *vp = v_all + static_cast<long long>(at.block) * AT_BLOCK;
  P pv[8];
  G gv[8];
  float g[8], m[8], v[8];
  at_load(at.p, lane, at.n(), at.vec(), pv);
  at_load(at.g, lane, at.n(), at.vec(), gv);
  at_load(mp, lane, AT_BLOCK, true, m);
  at_load(vp, lane, AT_BLOCK, true, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) g[e] = at_get<G>(gv[e]);
  at_moments(g, m, v, s);       // (behind the tensor m, v and g are zero, and stay so)
  __nv_bfloat16 half[8];
  at_weights(pv, m, v, half, s);
  at_store(at.p, lane, at.n(), at.vec(), pv);
  if (at.copy != nullptr) at_store(at.copy, lane, at.n(), at.vec(), half);
  at_store(mp, lane, AT_BLOCK, true, m);
  at_store(vp, lane, AT_BLOCK, true, v);
}

// Codes of a lane's eight moments in a block of exponent e; x: their 32 random bits, of which the first moment takes the lowest 20
// and the second the highest. low: the smallest magnitude.
template <bool SIGNED>
__device__ __forceinline__ void at_pack(const float (&v)[8], float low, uint32_t e, const uint32_t (&x)[8], uint32_t (&code)[2]) {
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = SIGNED ? x[i] & 0xfffffu : x[i] >> 12;
  if (!at_plain<SIGNED>(e)) {
    const uint32_t bottom = at_base<SIGNED>(e) << 20;
    code[0] = at_codes<SIGNED>(v, r, bottom);
    code[1] = at_codes<SIGNED>(v + 4, r + 4, bottom);
    return;
  }
  const float lift = at_lift<SIGNED>(e);
  float a[8];
  uint32_t u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[i] = v[i] * lift;
    u[i] = __float_as_uint(a[i]) + r[i];
  }
  if (!(low * lift >= AT_LEAST)) {
    // Some are below code 1: they become code 1 or 0 by the rule of at_codes, without a rounding.
    const float step = __fmul_rn(__uint_as_float((at_base<SIGNED>(e) + 1u) << 20), 9.5367431640625e-7f), far = step * -8388608.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // (r step with r as a number: its bits behind 2^23, less that, in one operation that rounds once)
      const bool up = SIGNED ? __fmaf_rn(__uint_as_float(0x4b000000u | r[i]), step, far) < fabsf(v[i]) : v[i] != 0.f;
      const uint32_t one = __float_as_uint(AT_LEAST) | (__float_as_uint(v[i]) & 0x80000000u);
      const uint32_t to = up ? one : __float_as_uint(AT_LEAST / 1.125f);
      u[i] = fabsf(a[i]) < AT_LEAST ? to : u[i];
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t t[4];
#pragma unroll
    // (the sum moved up, in this form: it is the one that the tests of the codes' bits have passed)
    for (int i = 0; i < 4; ++i) t[i] = u[4 * j + i] << 4;
    code[j] = at_top_bytes(t[0], t[1], t[2], t[3]);
    if (SIGNED) code[j] |= 0x80808080u & at_top_bytes(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
  }
}

// A block with 8-bit moments, its inputs in shared memory. em, ev: its exponents, and then the new ones. p, copy: its first element.
// ps, gs: shifts of weights and gradients there. mc, vc: the lane's codes. first, key: the place of its first element modulo 2^32, and what it is mixed with.
template <typename P, typename G>
__device__ __forceinline__ void at_block(AtStage<P, G>& in, int ps, int gs, P* p, __nv_bfloat16* copy, int n, bool vec, uint32_t* mc,
                                         uint32_t* vc, uint32_t first, uint32_t key, uint32_t& em, uint32_t& ev,
                                         const AdamScalars& s, int lane) {
  float m[8], v[8];
  {
    G gv[8];
    float g[8];
    at_load(in.g + gs, lane, AT_BLOCK, gs == 0, gv);
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = at_get<G>(gv[e]);
    const uint32_t *sm = reinterpret_cast<const uint32_t*>(in.m) + lane, *sv = reinterpret_cast<const uint32_t*>(in.v) + lane;
    const uint32_t bm = at_base<true>(em) << 20, bv = at_base<false>(ev) << 20;
    at_decode<true>(sm[0], bm, m);
    at_decode<true>(sm[32], bm, m + 4);
    at_decode<false>(sv[0], bv, v);
    at_decode<false>(sv[32], bv, v + 4);
    at_moments(g, m, v, s);
  }
  {
    P pv[8];
    __nv_bfloat16 half[8];
    at_load(in.p + ps, lane, AT_BLOCK, ps == 0, pv);
    at_weights(pv, m, v, half, s);
    if (vec) {
      at_store(p, lane, n, true, pv);
      if (copy != nullptr) at_store(copy, lane, n, true, half);
    } else {      // through shared memory, the copies in the place of the gradients, and from there lane beside lane
      const int cs = copy != nullptr ? at_shift(copy) : 0;
      __nv_bfloat16* copies = reinterpret_cast<__nv_bfloat16*>(in.g);
      __syncwarp();      // all have their gradients
      at_store(in.p + ps, lane, AT_BLOCK, ps == 0, pv);
      if (copy != nullptr) at_store(copies + cs, lane, AT_BLOCK, cs == 0, half);
      __syncwarp();
      at_spread(p, in.p, ps, n, lane);
      if (copy != nullptr) at_spread(copy, copies, cs, n, lane);
    }
  }
  float top_m = fabsf(m[0]), top_v = v[0], low_m = fabsf(m[0]), low_v = v[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    top_m = fmaxf(top_m, fabsf(m[e]));
    low_m = fminf(low_m, fabsf(m[e]));
    top_v = fmaxf(top_v, v[e]);
    low_v = fminf(low_v, v[e]);
  }
  em = at_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(top_m)));
  ev = at_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(top_v)));
  // The random bits are at_mix(place ^ key) of the element's place. Places of a block differ in their lowest 8 bits, so the
  // mix's first shift gives all of them the same.
  uint32_t mine = (first + lane * 4) ^ key;
  mine ^= mine >> 16;
  uint32_t x[8], code[2];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    uint32_t h = (mine ^ ((e >> 2) * 128 + (e & 3))) * 0x7feb352du;
    h = (h ^ (h >> 15)) * 0x846ca68bu;
    x[e] = h ^ (h >> 16);
  }
  at_pack<true>(m, low_m, em, x, code);
  mc[0] = code[0];
  mc[32] = code[1];
  at_pack<false>(v, low_v, ev, x, code);
  vc[0] = code[0];
  vc[32] = code[1];
}

// hyper: [lr, beta1, beta2, eps, weight_decay, bias_corr1, bias_corr2, grad_scale, max_norm]; rng: one 64-bit number, another one
// each step. Both in device memory, so that a captured step sees their values at its replay.
__device__ __forceinline__ AdamScalars at_scalars(const float* hyper, const float* sumsq, const long long* rng) {
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
  if (rng != nullptr) {
    const unsigned long long seed = static_cast<unsigned long long>(*rng);
    s.key = at_mix(static_cast<uint32_t>(seed) ^ at_mix(static_cast<uint32_t>(seed >> 32)));
  }
  return s;
}

template <typename P, typename G>
__global__ void __launch_bounds__(AT_WARPS * 32, 4)
adamw_tensors_kernel(const __grid_constant__ AdamTensors t, float* m, float* v, const float* __restrict__ hyper,
                     const float* __restrict__ sumsq) {
  grid_chain();
  const int lane = threadIdx.x & 31;
  AtPlace<P, G> at;
  at.find(t, blockIdx.x, warp_index());
  if (at.rest <= 0) return;
  AdamScalars s = at_scalars(hyper, sumsq, nullptr);
  if (!at.decays) s.decay = 1.f;
  do at_block(at, m, v, s, lane);
  while (at.next());
}

// The blocks of a chunk that are a warp's. WHOLE: all of them are, on 16 bytes; their addresses are then steps from lane to lane
// and block to block, and nothing is asked of them.
template <typename P, typename G, bool WHOLE>
__device__ __forceinline__ void at_chunk(AtPlace<P, G> at, AtStage<P, G>* ring, uint8_t* m_all, uint8_t* v_all,
                                         uint8_t (*exponents)[AT_CHUNK], int held, const float* hyper, const float* sumsq,
                                         const long long* rng, int warp, int lane) {
  constexpr int step = AT_WARPS * AT_BLOCK;
  const long long first = static_cast<long long>(at.block) * AT_BLOCK;
  const P* p_next = at.p;
  const G* g_next = at.g;
  const uint8_t* codes = (lane < 16 ? m_all : v_all) + first + (lane & 15) * 16;
  int left = at.rest;         // elements from the block to fetch next on
  const int ps = WHOLE || at.aligned ? 0 : at_shift(at.p), gs = WHOLE || at.aligned ? 0 : at_shift(at.g);
  bool begins = at.begins;
  auto fetch = [&](AtStage<P, G>& to) {
    if (WHOLE || (at.aligned && left >= AT_BLOCK)) {
      at_fetch(to.p, p_next, lane);
      at_fetch(to.g, g_next, lane);
    } else if (left >= AT_BLOCK && !(begins && ps + gs)) {
      at_fetch_words(to.p, p_next, ps, lane);
      at_fetch_words(to.g, g_next, gs, lane);
    } else {      // a tensor's ends (there for the warp after its next __syncwarp)
      P pv[8];
      G gv[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pv[e] = e * 32 + lane < left ? p_next[e * 32 + lane] : P(0.f);
        gv[e] = e * 32 + lane < left ? g_next[e * 32 + lane] : G(0.f);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        to.p[ps + e * 32 + lane] = pv[e];
        to.g[gs + e * 32 + lane] = gv[e];
      }
    }
    at_copy_16((lane < 16 ? to.m : to.v) + (lane & 15) * 16, codes);
    p_next += step;
    g_next += step;
    codes += step;
    left -= step;
    begins = false;
  };
  if (warp < held) fetch(ring[0]);
  asm volatile("cp.async.commit_group;" ::: "memory");
  AdamScalars s = at_scalars(hyper, sumsq, rng);
  if (!at.decays) s.decay = 1.f;
  __syncthreads();            // the exponents are there
  uint32_t high = static_cast<uint32_t>(first >> 32), low = static_cast<uint32_t>(first);
  uint32_t key = at_mix(s.key + high);
  uint32_t *mc = reinterpret_cast<uint32_t*>(m_all + first) + lane, *vc = reinterpret_cast<uint32_t*>(v_all + first) + lane;
  P* p = at.p;
  __nv_bfloat16* copy = at.copy;
  int rest = at.rest, stage = 0;
  for (int j = warp; j < held; j += AT_WARPS) {
    __syncwarp();     // every lane has read the stage that is filled now
    if (j + AT_WARPS < held) fetch(ring[stage ^ 1]);
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    uint32_t em = exponents[0][j], ev = exponents[1][j];
    const int n = WHOLE || rest >= AT_BLOCK ? AT_BLOCK : rest;
    at_block(ring[stage], ps, gs, p, copy, n, WHOLE || (at.aligned && n == AT_BLOCK), mc, vc, low, key, em, ev, s, lane);
    if (lane == 0) {
      exponents[0][j] = static_cast<uint8_t>(em);
      exponents[1][j] = static_cast<uint8_t>(ev);
    }
    p += step;
    if (copy != nullptr) copy += step;
    mc += step / 4;
    vc += step / 4;
    rest -= step;
    low += step;
    if (low < step) key = at_mix(s.key + ++high);
    stage ^= 1;
  }
}

// With 8-bit moments a warp's next block is on its way to shared memory while it works on one: there is about as much to
// compute as to move, and registers for only half the warps. The exponents of the chunk are read before and written after all
// else, in one access each: single bytes, written by one warp into sectors that others were about to read, took as long again
// as the whole rest (113 M elements: 655 us, without them 300).
template <typename P, typename G>
__global__ void __launch_bounds__(AT_WARPS * 32, 4)
adamw_tensors_8bit_kernel(const __grid_constant__ AdamTensors t, uint8_t* m, uint8_t* v, uint8_t* scales, long long blocks,
                          const float* __restrict__ hyper, const float* __restrict__ sumsq, const long long* __restrict__ rng) {
  extern __shared__ __align__(128) uint8_t at_smem[];
  __shared__ uint8_t exponents[2][AT_CHUNK];
  grid_chain();
  const int lane = threadIdx.x & 31, warp = warp_index();
  AtStage<P, G>* ring = reinterpret_cast<AtStage<P, G>*>(at_smem) + warp * AT_STAGES;
  AtPlace<P, G> at;
  at.find(t, blockIdx.x, warp);
  const int of_chunk = at.block - warp, elements = at.rest + warp * AT_BLOCK;       // the chunk's first block, and its elements
  const int held = (elements + AT_BLOCK - 1) / AT_BLOCK;
  if (warp < 2 && lane < held) exponents[warp][lane] = scales[warp * blocks + of_chunk + lane];
  if (at.aligned && elements % AT_BLOCK == 0)
    at_chunk<P, G, true>(at, ring, m, v, exponents, held, hyper, sumsq, rng, warp, lane);
  else
    at_chunk<P, G, false>(at, ring, m, v, exponents, held, hyper, sumsq, rng, warp, lane);
  __syncthreads();
  if (warp < 2 && lane < held) scales[warp * blocks + of_chunk + lane] = exponents[warp][lane];
}

// The values of all codes, both moments in one launch: eight codes a thread.
template <typename O>
__global__ void __launch_bounds__(256)
moment_values_kernel(const uint2* __restrict__ mc, const uint2* __restrict__ vc, const uint8_t* __restrict__ scales,
                     long long blocks, O* __restrict__ m, O* __restrict__ v) {
  grid_chain();
  const long long n = blocks * (AT_BLOCK / 8);
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += gridDim.x * 256LL) {
    const long long block = i / (AT_BLOCK / 8);
    const uint2 a = mc[i], b = vc[i];
    const uint32_t bm = at_base<true>(scales[block]) << 20, bv = at_base<false>(scales[blocks + block]) << 20;
    float f[8], g[8];
    at_decode<true>(a.x, bm, f);
    at_decode<true>(a.y, bm, f + 4);
    at_decode<false>(b.x, bv, g);
    at_decode<false>(b.y, bv, g + 4);
    AtVec<O, 8> x, y;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x.v[e] = at_put<O>(f[e]);
      y.v[e] = at_put<O>(g[e]);
    }
    *reinterpret_cast<AtVec<O, 8>*>(m + i * 8) = x;
    *reinterpret_cast<AtVec<O, 8>*>(v + i * 8) = y;
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
    at_load(m + at, lane, AT_BLOCK, true, x);
    at_load(v + at, lane, AT_BLOCK, true, y);
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top_m = max(top_m, __float_as_uint(x[e]) & 0x7fffffffu);
      top_v = max(top_v, __float_as_uint(y[e]) & 0x7fffffffu);
    }
    const uint32_t em = at_exponent(__reduce_max_sync(0xffffffffu, top_m)), ev = at_exponent(__reduce_max_sync(0xffffffffu, top_v));
    const uint32_t bm = at_base<true>(em) << 20, bv = at_base<false>(ev) << 20;
    const uint32_t half[4] = {0x80000u, 0x80000u, 0x80000u, 0x80000u};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      *reinterpret_cast<uint32_t*>(mc + at + j * 128 + lane * 4) = at_codes<true>(x + j * 4, half, bm);
      *reinterpret_cast<uint32_t*>(vc + at + j * 128 + lane * 4) = at_codes<false>(y + j * 4, half, bv);
    }
    if (lane == 0) {
      scales[block] = static_cast<uint8_t>(em);
      scales[blocks + block] = static_cast<uint8_t>(ev);
    }
  }
}

template <typename P, typename G>
static int at_launch(const AdamTensors& t, int bits, long long elements, void* m, void* v, uint8_t* scales, long long blocks,
                     const float* hyper, const float* sumsq, const long long* rng, cudaStream_t st) {
  const bool chained = elements <= CHAIN_ELEMENTS;
  const int grid = t.chunk[t.n];
  if (bits == 32)
    return static_cast<int>(launch_when(chained, adamw_tensors_kernel<P, G>, grid, AT_WARPS * 32, 0, st, t, static_cast<float*>(m),
                                        static_cast<float*>(v), hyper, sumsq));
  auto kern = adamw_tensors_8bit_kernel<P, G>;
  constexpr int smem = AT_WARPS * AT_STAGES * sizeof(AtStage<P, G>);
  static bool configured_on[MAX_DEVICES];
  const int dev = current_device_slot();
  if (dev < 0) return -4;
  if (!configured_on[dev]) {
    NPLM_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    configured_on[dev] = true;
  }
  return static_cast<int>(launch_when(chained, kern, grid, AT_WARPS * 32, smem, st, t, static_cast<uint8_t*>(m),
                                      static_cast<uint8_t*>(v), scales, blocks, hyper, sumsq, rng));
}

}  // namespace nplm

using namespace nplm;

// n tensors: p, g, copy (null: none), numel, first block in the moments, decay. p_type, g_type: 0
// bf16, 2 fp32; copies are bf16. bits 8: m, v uint8 [blocks][256], scales uint8 [2][blocks]; 32: m, v fp32 [blocks][256].
extern "C" int nplm_adamw_tensors(void* const* p, const void* const* g, void* const* copy, const long long* numel,
                                  const long long* block, const unsigned char* decay, int n, int p_type, int g_type, int bits,
                                  void* m, void* v, void* scales, long long blocks, const float* hyper, const float* sumsq,
                                  const long long* rng, cudaStream_t st) {
  if (n < 0 || (p_type != 0 && p_type != 2) || (g_type != 0 && g_type != 2) || (bits != 8 && bits != 32)) return -1;
  if (bits == 8 && (scales == nullptr || rng == nullptr)) return -1;
  AdamTensors t;
  // A thread block takes 32 blocks in a row, so that looking up their tensor counts little; 8 while that leaves multiprocessors
  // without work.
  long long all = 0;
  for (int k = 0; k < n; ++k) all += (numel[k] + AT_BLOCK - 1) / AT_BLOCK;
  t.per_chunk = all >= 148LL * 4 * AT_CHUNK ? AT_CHUNK : AT_WARPS;
  int i = 0;
  while (i < n) {
    t.n = 0;
    t.chunk[0] = 0;
    long long chunks = 0, elements = 0;
    for (; i < n && t.n < AT_TENSORS; ++i) {
      if (numel[i] == 0) continue;
      const long long has = (numel[i] + AT_BLOCK - 1) / AT_BLOCK;
      if (numel[i] < 0 || block[i] < 0 || block[i] + has > blocks || blocks > 0x7fffffffLL) return -2;
      const long long more = (has + t.per_chunk - 1) / t.per_chunk;
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
    int e;
    if (p_type == 2 && g_type == 2) e = at_launch<float, float>(t, bits, elements, m, v, sc, blocks, hyper, sumsq, rng, st);
    else if (p_type == 2) e = at_launch<float, __nv_bfloat16>(t, bits, elements, m, v, sc, blocks, hyper, sumsq, rng, st);
    else if (g_type == 2) e = at_launch<__nv_bfloat16, float>(t, bits, elements, m, v, sc, blocks, hyper, sumsq, rng, st);
    else e = at_launch<__nv_bfloat16, __nv_bfloat16>(t, bits, elements, m, v, sc, blocks, hyper, sumsq, rng, st);
    if (e) return e;
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
  const uint2 *a = static_cast<const uint2*>(mc), *b = static_cast<const uint2*>(vc);
  const uint8_t* s = static_cast<const uint8_t*>(scales);
  const bool chained = blocks * AT_BLOCK <= CHAIN_ELEMENTS;
  const cudaError_t e =
      out_type == 2 ? launch_when(chained, moment_values_kernel<float>, at_grid(blocks, 8), 256, 0, st, a, b, s, blocks,
                                  static_cast<float*>(m), static_cast<float*>(v))
                    : launch_when(chained, moment_values_kernel<__nv_bfloat16>, at_grid(blocks, 8), 256, 0, st, a, b, s, blocks,
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
