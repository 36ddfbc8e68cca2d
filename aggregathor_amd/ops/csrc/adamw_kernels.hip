// gfx950 kernels of the optimizer step: the L2 norm over many tensors, and the
// AdamW step over many tensors with states in 32 or in 8 bits.
//
// With g the gradient, scaled by s = min(1, max_norm / norm) where it is
// clipped, and t the tensor's number of steps:
//
//   m = beta1 m + (1 - beta1) s g
//   v = beta2 v + (1 - beta2) (s g)^2
//   p = p (1 - lr wd) - lr / (1 - beta1^t) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// 8-bit states. Groups of 32 consecutive elements of a tensor share a power of
// two (one byte, the exponent with its bias of 127), and each element of m and
// of r = sqrt(v) is an e4m3 code times it. The root is kept rather than v since
// its range in binades is half as wide. The power puts the group's largest
// value into [128, 256], so that rounding up never leaves the format; 17
// binades below it the format ends. A root that is not zero is never stored as
// zero: it would make the next step divide by eps.
// To nearest, an average that moves by 1 - beta2 = 0.1 % a step would stand
// still in a format whose half step is 6 %. So codes are rounded up or down by
// chance, without bias: floor(y / quantum + u), u from 16 bits of a hash of
// (seed, tensor, step, element). The hash makes a step's result a function of
// its inputs, the same on every rank and in every replay.
// The step itself uses the new m and v before they are rounded.
//
// m, v, scales and codes are those of plain IEEE fp32, one rounding an operation
// (no contraction into fused multiply-adds), so that states can be compared with
// another implementation's bit by bit. The quotient takes the hardware's
// reciprocal, and with 32-bit states the root its square root, which are off by
// a unit in the last place at most (seen over all normal numbers): with 8-bit
// states the vector units are as busy as the memory, at 83 instructions an
// element for 16 bytes (114 with the full sequences for quotient, root and
// rounding took 411 us for VGG-16 where this takes 357).

#include <hip/hip_runtime.h>

#include "adamw_kernels.h"

#pragma clang fp contract(off)

namespace adamw {

namespace {

constexpr int kBlock = 256;

// Four elements of T. Tensors start anywhere (a gradient is a view into the
// flat gradient), so a quad is only aligned like its element: gfx950 loads and
// stores it in one instruction all the same.
typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t codes4 __attribute__((aligned(1)));

// Pointers that come out of memory could be to anything for all the compiler
// knows; these are to global memory, which has loads and stores of its own.
template <typename T>
using Global = __attribute__((address_space(1))) T*;

struct F32 {
  typedef float Elem;
  typedef f32x4 Quad;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};

struct BF16 {
  typedef uint16_t Elem;
  typedef u16x4 Quad;
  static __device__ __forceinline__ float get(uint16_t v) {
    return __uint_as_float((uint32_t)v << 16);
  }
  static __device__ __forceinline__ uint16_t put(float v) {
    return __builtin_bit_cast(uint16_t, (__bf16)v);
  }
};

struct F16 {
  typedef uint16_t Elem;
  typedef u16x4 Quad;
  static __device__ __forceinline__ float get(uint16_t v) {
    return (float)__builtin_bit_cast(_Float16, v);
  }
  static __device__ __forceinline__ uint16_t put(float v) {
    return __builtin_bit_cast(uint16_t, (_Float16)v);
  }
};

// Elements [i, i + 4) below n; those behind it are zero.
template <bool Full, typename T>
__device__ __forceinline__ typename T::Quad load4(
    Global<const typename T::Elem> base, int i, int n) {
  typename T::Quad q;
  if (Full || i + 4 <= n) {
    q = __builtin_nontemporal_load(
        (Global<const typename T::Quad>)(base + i));
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c) q[c] = i + c < n ? base[i + c] : 0;
  }
  return q;
}

template <bool Full, typename T>
__device__ __forceinline__ void store4(Global<typename T::Elem> base, int i, int n,
                                       const float (&x)[4]) {
  typename T::Quad q;
#pragma unroll
  for (int c = 0; c < 4; ++c) q[c] = T::put(x[c]);
  if (Full || i + 4 <= n) {
    __builtin_nontemporal_store(
        q, (Global<typename T::Quad>)(base + i));
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (i + c < n) base[i + c] = q[c];
  }
}

template <typename T>
__device__ __forceinline__ void widen(typename T::Quad q, float (&out)[4]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) out[c] = T::get(q[c]);
}

// Four codes as one word.
template <bool Full>
__device__ __forceinline__ uint32_t load_codes(Global<const uint8_t> base, int i,
                                               int n) {
  if (Full || i + 4 <= n)
    return __builtin_nontemporal_load(
        (Global<const codes4>)(base + i));
  uint32_t w = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (i + c < n) w |= (uint32_t)base[i + c] << (8 * c);
  return w;
}

template <bool Full>
__device__ __forceinline__ void store_codes(Global<uint8_t> base, int i, int n,
                                            uint32_t w) {
  if (Full || i + 4 <= n) {
    __builtin_nontemporal_store(w, (Global<codes4>)(base + i));
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (i + c < n) base[i + c] = (uint8_t)(w >> (8 * c));
  }
}

// What all elements of a workgroup share.
struct Common {
  float clip, beta1, rest1, beta2, rest2, eps, keep, rate, unbias;
  uint32_t key;
};

// ---------------------------------------------------------------------------
// 8-bit states

__device__ __forceinline__ uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x9E3779B1u;
  x ^= x >> 15;
  x *= 0x85EBCA77u;
  return x ^ (x >> 16);
}

__device__ __forceinline__ void decode(uint32_t w, float scale,
                                       float (&out)[4]) {
  auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  out[0] = lo[0] * scale;
  out[1] = lo[1] * scale;
  out[2] = hi[0] * scale;
  out[3] = hi[1] * scale;
}

__device__ __forceinline__ uint32_t encode(const float (&z)[4]) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], w, true);
}

// Power of two with this biased exponent.
__device__ __forceinline__ float pow2(uint32_t biased) {
  return __uint_as_float(biased << 23);
}

// y >= 0 rounded to a value that e4m3 has, up with a probability of chance / 2^16:
// floor(y / quantum + chance / 2^16) quanta. Above 2^-6 the quantum is the value
// of the lowest of the three leading bits of the mantissa, so adding the chance
// right below that bit and cutting off there does it. Below, the quantum stays
// 2^-9, as if y had 2^-6 to it.
__device__ __forceinline__ float round_by_chance(float y, uint32_t chance) {
  const float low = y < 0x1p-6f ? 0x1p-6f : 0.f;
  const uint32_t bits = __float_as_uint(y + low) + (chance << 4);
  return __uint_as_float(bits & 0xFFF00000u) - low;
}

// Largest of a value over the eight lanes that share a group.
__device__ __forceinline__ uint32_t max8(uint32_t v) {
  // xor 1, xor 2 within four lanes, then each four against the other.
  uint32_t o = __builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true);
  v = v > o ? v : o;
  o = __builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true);
  v = v > o ? v : o;
  o = __builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true);
  return v > o ? v : o;
}

// Bits of the largest |x|; as whole numbers they order alike, with infinity and
// NaN above all others.
constexpr uint32_t kInf = 0x7F800000u;

template <bool Finite>
__device__ __forceinline__ uint32_t top_bits(const float (&x)[4]) {
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t b = __float_as_uint(x[c]) & 0x7FFFFFFFu;
    if (Finite) b = b < kInf ? b : 0u;
    top = top > b ? top : b;
  }
  return top;
}

// One quad's new 8-bit states.
struct Codes {
  uint32_t m, r, m_scale, r_scale;
};

// From m and v; gives the denominators too. `tm` and `tv` are top_bits of the
// group. Plain: everything in the wave is finite.
template <bool Plain>
__device__ __forceinline__ Codes encode_states(const Common& k, long at,
                                               uint32_t tm, uint32_t tv,
                                               const float (&m)[4],
                                               const float (&v)[4],
                                               float (&denominator)[4]) {
  Codes out;
  const uint32_t em = tm >> 23;
  out.m_scale = em < 14 ? 7 : em - 7;
  const int half = ((int)(tv >> 23) - 127) >> 1;
  out.r_scale = (uint32_t)(half + 120);
  const float im = pow2(254 - out.m_scale);
  const float root_unit = pow2(out.r_scale) * k.unbias;
  const uint32_t key = k.key + 0x9E3779B9u * (uint32_t)(at >> 32);
  float zm[4], zr[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t h = mix((uint32_t)(at + c) ^ key);
    zm[c] = copysignf(round_by_chance(fabsf(m[c]) * im, h & 0xFFFFu), m[c]);
    // v / scale^2, its root and the root's last bit, which is right for all that
    // is above 2^-100 (tried for every such number). What is below 2^-126, whose
    // root is 2^71 below the group's largest, is raised to that: the hardware
    // takes denormals for zero.
    const float x = fmaxf(ldexpf(v[c], 2 * (7 - half)), 0x1p-126f);
    const float over = __builtin_amdgcn_rsqf(x), near = x * over;
    const float y = __builtin_fmaf(__builtin_fmaf(-near, near, x), 0.5f * over,
                                   near);
    denominator[c] = __builtin_fmaf(y, root_unit, k.eps);
    zr[c] = fmaxf(round_by_chance(y, h >> 16), v[c] > 0.f ? 0x1p-9f : 0.f);
    if (!Plain) {
      // NaN where there is none to store (the format has no infinity), and the
      // formula's own values in the denominator.
      const bool fine_m = fabsf(m[c]) < INFINITY, fine_v = v[c] < INFINITY;
      zm[c] = fine_m ? zm[c] : NAN;
      zr[c] = fine_v ? zr[c] : NAN;
      denominator[c] = fine_v ? denominator[c] : v[c];
    }
  }
  out.m = encode(zm);
  out.r = encode(zr);
  return out;
}

// ---------------------------------------------------------------------------
// The update

__device__ __forceinline__ void moments(const Common& k, const float (&g)[4],
                                        float (&m)[4], float (&v)[4]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const float s = g[c] * k.clip;
    m[c] = m[c] * k.beta1 + s * k.rest1;
    v[c] = v[c] * k.beta2 + s * s * k.rest2;
  }
}

__device__ __forceinline__ void move(const Common& k, const float (&m)[4],
                                     const float (&denominator)[4],
                                     float (&p)[4]) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    p[c] = p[c] * k.keep -
           k.rate * (m[c] * __builtin_amdgcn_rcpf(denominator[c]));
}

// The hardware's root, which takes denormals for zero, of a number that may be
// one.
__device__ __forceinline__ float root_of(float v) {
  const bool low = v < 0x1p-96f;
  return __builtin_amdgcn_sqrtf(v * (low ? 0x1p64f : 1.f)) *
         (low ? 0x1p-32f : 1.f);
}

struct Scalars {
  double beta1, beta2;
  float lr, rest1, rest2, eps, keep, max_norm;
  const float* norm;
};

// rate = lr / (1 - beta1^t) and unbias = 1 / sqrt(1 - beta2^t), the powers by
// squaring in 64 bits (1 - beta^t loses what 32 hold while it is near zero):
// beta1's in even lanes, beta2's in odd ones. Every wave does it for itself:
// with 8-bit states VGG-16 took 367 us so, and 401 us where three waves waited
// for one.
__device__ __forceinline__ Common common(const Scalars& s, uint32_t key,
                                         uint32_t t) {
  Common k;
  k.clip = 1.f;
  if (s.norm != nullptr) {
    const float norm = *s.norm;
    k.clip = norm <= s.max_norm ? 1.f : s.max_norm / norm;
  }
  k.beta1 = (float)s.beta1;
  k.rest1 = s.rest1;
  k.beta2 = (float)s.beta2;
  k.rest2 = s.rest2;
  k.eps = s.eps;
  k.keep = s.keep;
  k.key = mix(key + t);
  const bool odd = threadIdx.x & 1;
  double x = odd ? s.beta2 : s.beta1, power = 1.0;
  for (; t != 0; t >>= 1) {
    if (t & 1) power *= x;
    x *= x;
  }
  const float rest = (float)(1.0 - power);
  const float out = odd ? 1.f / sqrtf(rest) : s.lr / rest;
  k.rate = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(out), 0));
  k.unbias =
      __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(out), 1));
  return k;
}

// Step counts are read by all workgroups and written once, by the first wave of
// the last workgroup that has read them. (A launch of its own for that took 3 to
// 4 us a step.) One address takes an arrival in 12 ns, so they arrive at 32, and
// the last of each of these at one. Counters wrap by themselves to the zero that
// the next launch needs.
// Up to 64 of them arrive at one at once: a second arrival would take longer
// than they wait for each other. Measured, one address / 32 and one: the step of
// 64, 96, 128, 192, 512 workgroups 3.88 / 4.00, 3.96 / 3.96, 4.3 / 4.2, 5.2 / 4.2,
// 9.7 / 5.6 us, the norm 5.1 / 5.2, 5.3 / 5.1, 5.6 / 5.2, 6.2 / 5.2, 10.2 / 5.8.
__device__ __forceinline__ unsigned lines() {
  return gridDim.x <= 64 ? 1 : kTicketLines;
}

__device__ __forceinline__ unsigned on_line() {  // workgroups that share one
  return (gridDim.x - blockIdx.x % lines() + lines() - 1) / lines();
}

__device__ __forceinline__ unsigned arrive(unsigned* tickets) {
  return atomicInc(tickets + 32 * (1 + blockIdx.x % lines()), on_line() - 1);
}

// Whether this workgroup, given what arrive() returned, was the last.
__device__ __forceinline__ bool last(unsigned* tickets, unsigned arrived) {
  if (arrived != on_line() - 1) return false;
  return lines() == 1 || atomicInc(tickets, lines() - 1) == lines() - 1;
}

template <int Bits, int Quads, typename P, typename G, bool Full>
__device__ __forceinline__ void update_chunk(const Work& w, const void* grad,
                                             const int* steps,
                                             unsigned* tickets,
                                             unsigned& arrived,
                                             const Scalars& s) {
  typedef typename P::Elem PElem;
  typedef typename G::Elem GElem;
  const Global<PElem> param = (Global<PElem>)w.p;
  const Global<const GElem> g_at = (Global<const GElem>)grad + w.start;
  const Global<float> m32 = (Global<float>)w.m, v32 = (Global<float>)w.r;
  const Global<uint8_t> m8 = (Global<uint8_t>)w.m, r8 = (Global<uint8_t>)w.r;
  const Global<uint8_t> m8s = (Global<uint8_t>)w.ms;
  const Global<uint8_t> r8s = (Global<uint8_t>)w.rs;
  const int n = w.left;

  // The count first, then all loads of data: loads come back in order, so the
  // wait for the count leaves the others on their way. (With the count last
  // VGG-16, clipped, took 705 us instead of 700, ResNet-50 116.2 instead of
  // 115.5.)
  int count = __hip_atomic_load(steps + w.tensor, __ATOMIC_RELAXED,
                                __HIP_MEMORY_SCOPE_AGENT);
  typename P::Quad pq[Quads];
  typename G::Quad gq[Quads];
  f32x4 mq[Quads], vq[Quads];
  uint32_t mw[Quads], rw[Quads], ms[Quads], rs[Quads];
#pragma unroll
  for (int q = 0; q < Quads; ++q) {
    const int i = 4 * (q * kBlock + (int)threadIdx.x);
    if constexpr (Bits == 32) {
      mq[q] = load4<Full, F32>(m32, i, n);
      vq[q] = load4<Full, F32>(v32, i, n);
    } else {
      mw[q] = load_codes<Full>(m8, i, n);
      rw[q] = load_codes<Full>(r8, i, n);
      ms[q] = Full || i < n ? m8s[i / kGroup] : 0;
      rs[q] = Full || i < n ? r8s[i / kGroup] : 0;
    }
    gq[q] = load4<Full, G>(g_at, i, n);
    pq[q] = load4<Full, P>(param, i, n);
  }
  // A barrier waits for no load, and the one behind the arrival that says "read"
  // would write the count under a wave whose load is still on its way. So each
  // wave has it in a register before the barrier: this use is where it waits.
  asm volatile("" : "+v"(count) : : "memory");
  __syncthreads();  // all four waves have read it
  if (threadIdx.x == 0) arrived = arrive(tickets);
  const int step = __builtin_amdgcn_readfirstlane(count + 1);
  const Common k = common(s, w.key, (uint32_t)step);

#pragma unroll
  for (int q = 0; q < Quads; ++q) {
    const int i = 4 * (q * kBlock + (int)threadIdx.x);
    float p[4], g[4], m[4], v[4], denominator[4];
    widen<P>(pq[q], p);
    widen<G>(gq[q], g);
    if constexpr (Bits == 32) {
      widen<F32>(mq[q], m);
      widen<F32>(vq[q], v);
      moments(k, g, m, v);
      store4<Full, F32>(m32, i, n, m);
      store4<Full, F32>(v32, i, n, v);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        denominator[c] = root_of(v[c]) * k.unbias + k.eps;
    } else {
      decode(mw[q], pow2(ms[q]), m);
      decode(rw[q], pow2(rs[q]), v);
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = v[c] * v[c];
      moments(k, g, m, v);
      // All eight lanes of a group come here, also those behind the end.
      uint32_t tm = max8(top_bits<false>(m)), tv = max8(top_bits<false>(v));
      Codes codes;
      if (__builtin_expect(__any(tm >= kInf || tv >= kInf), 0)) {
        tm = max8(top_bits<true>(m));
        tv = max8(top_bits<true>(v));
        codes = encode_states<false>(k, w.start + i, tm, tv, m, v, denominator);
      } else {
        codes = encode_states<true>(k, w.start + i, tm, tv, m, v, denominator);
      }
      store_codes<Full>(m8, i, n, codes.m);
      store_codes<Full>(r8, i, n, codes.r);
      if ((Full || i < n) && threadIdx.x % (kGroup / 4) == 0) {
        m8s[i / kGroup] = (uint8_t)codes.m_scale;
        r8s[i / kGroup] = (uint8_t)codes.r_scale;
      }
    }
    move(k, m, denominator, p);
    store4<Full, P>(param, i, n, p);
  }
}

template <int Bits, int Quads, typename P, typename G>
__device__ __forceinline__ void update_tensor(const Work& w, const void* grad,
                                              const int* steps,
                                              unsigned* tickets,
                                              unsigned& arrived,
                                              const Scalars& s) {
  if (w.left == Quads * 4 * kBlock)
    update_chunk<Bits, Quads, P, G, true>(w, grad, steps, tickets, arrived, s);
  else
    update_chunk<Bits, Quads, P, G, false>(w, grad, steps, tickets, arrived,
                                           s);
}

template <int Bits, int Quads>
__global__ __launch_bounds__(kBlock) void update_kernel(
    const Work* __restrict__ work, long nwork, int first, int count, int* steps,
    unsigned* tickets, const Grads grads, const Scalars s) {
  unsigned arrived = 0;
  const void* grad = nullptr;
  Work w;
  if (blockIdx.x < nwork) {  // without work, one workgroup counts
    w = work[blockIdx.x];
    grad = grads.g[w.tensor - first];
  }
  if (grad == nullptr) {
    if (threadIdx.x == 0) arrived = arrive(tickets);
  } else {
    const int at = w.tensor - first;
    const uint32_t type = (grads.types[at / 16] >> (2 * (at % 16))) & 3;
    switch (w.type * 4 + type) {
      case kF32 * 4 + kF32:
        update_tensor<Bits, Quads, F32, F32>(w, grad, steps, tickets, arrived,
                                           s);
        break;
      case kF32 * 4 + kBF16:
        update_tensor<Bits, Quads, F32, BF16>(w, grad, steps, tickets, arrived,
                                           s);
        break;
      case kF32 * 4 + kF16:
        update_tensor<Bits, Quads, F32, F16>(w, grad, steps, tickets, arrived,
                                           s);
        break;
      case kBF16 * 4 + kBF16:
        update_tensor<Bits, Quads, BF16, BF16>(w, grad, steps, tickets, arrived,
                                           s);
        break;
      case kF16 * 4 + kF16:
        update_tensor<Bits, Quads, F16, F16>(w, grad, steps, tickets, arrived,
                                           s);
        break;
    }
  }
  if (threadIdx.x >= 64) return;
  if (__builtin_amdgcn_readfirstlane(threadIdx.x == 0 &&
                                     last(tickets, arrived)))
    for (int i = threadIdx.x; i < count; i += 64)
      if (grads.g[i] != nullptr) steps[first + i] += 1;
}

// ---------------------------------------------------------------------------
// The norm. Squares are summed in 64 bits: no sum of them is too long, none of
// fp32 overflows or vanishes, and the vector units have the rate for it at
// four bytes an element. Which workgroup adds which elements is fixed by the
// spans alone, so the result is the same every time.
// Loads are not nontemporal here: a step reads the same gradients next. (Clipped
// VGG-16 697 us instead of 722, ResNet-50 with 8-bit states 88 instead of 91; the
// norms by themselves 46.7 and 19.9 us instead of 43.6 and 18.9.)

template <typename T>
__device__ __forceinline__ double chunk_squares(const void* ptr, int chunk,
                                                long n) {
  constexpr int kElems = kNormChunkBytes / sizeof(typename T::Elem);
  const Global<const typename T::Elem> base =
      (Global<const typename T::Elem>)ptr + (long)chunk * kElems;
  n -= (long)chunk * kElems;
  double sum[4] = {0, 0, 0, 0};
  if (n >= kElems) {
#pragma unroll
    for (int q = 0; q < kElems / (4 * kBlock); ++q) {
      float x[4];
      widen<T>(*(Global<const typename T::Quad>)(
                   base + 4 * (q * kBlock + (int)threadIdx.x)),
               x);
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[c] = fma((double)x[c], (double)x[c], sum[c]);
    }
  } else {
    for (int i = 4 * threadIdx.x; i < (int)n; i += 4 * kBlock) {
      float x[4];
      widen<T>(load4<false, T>(base, i, (int)n), x);
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[c] = fma((double)x[c], (double)x[c], sum[c]);
    }
  }
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

// Sum over the workgroup, in thread 0.
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kBlock / 64];
  __syncthreads();  // the last call's are read
#pragma unroll
  for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d, 64);
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
  __syncthreads();
  v = 0;
  if (threadIdx.x == 0)
    for (int w = 0; w < kBlock / 64; ++w) v += part[w];
  return v;
}

// With tickets the last workgroup to arrive adds the partial sums up, always in
// the same order. The sums are written and read past the caches of the compute
// dies (agent scope), and one has arrived in memory before its workgroup does at
// the tickets: s_waitcnt is what the workgroup fence is here. (A release at agent
// scope would write back what the dies' caches hold of others' data too, once a
// workgroup: 45 us for ResNet-50's gradient instead of 18.)
__global__ __launch_bounds__(kBlock) void norm_kernel(const Spans spans,
                                                      double* partials,
                                                      unsigned* tickets,
                                                      float* out) {
  double sum = 0;
  int span = 0;
  for (int c = blockIdx.x; c < spans.start[spans.count]; c += gridDim.x) {
    while (c >= spans.start[span + 1]) ++span;
    const int chunk = c - spans.start[span];
    const long n = spans.n4t[span] >> 2;
    switch (spans.n4t[span] & 3) {
      case kF32:
        sum += chunk_squares<F32>(spans.ptr[span], chunk, n);
        break;
      case kBF16:
        sum += chunk_squares<BF16>(spans.ptr[span], chunk, n);
        break;
      case kF16:
        sum += chunk_squares<F16>(spans.ptr[span], chunk, n);
        break;
    }
  }
  sum = block_sum(sum);
  if (tickets == nullptr) {
    if (threadIdx.x == 0) partials[blockIdx.x] = sum;
    return;
  }
  __shared__ bool finish;
  if (threadIdx.x == 0) {
    __hip_atomic_store(partials + blockIdx.x, sum, __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);
    finish = last(tickets, arrive(tickets));
  }
  __syncthreads();
  if (!finish) return;
  sum = 0;
  for (int i = threadIdx.x; i < (int)gridDim.x; i += kBlock)
    sum += __hip_atomic_load(partials + i, __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
  sum = block_sum(sum);
  if (threadIdx.x == 0) *out = (float)sqrt(sum);
}

__global__ __launch_bounds__(kBlock) void norm_finish_kernel(
    const double* __restrict__ partials, int count, float* out) {
  double sum = 0;
  for (int i = threadIdx.x; i < count; i += kBlock) sum += partials[i];
  sum = block_sum(sum);
  if (threadIdx.x == 0) *out = (float)sqrt(sum);
}

}  // namespace

bool supported(int p, int g) { return p == g || p == kF32; }

void update(int bits, long chunk, const Work* work, long nwork, int first,
            int count, int* steps, unsigned* tickets, const Grads& grads,
            const Hyper& h, hipStream_t stream) {
  const Scalars s = {h.beta1,
                     h.beta2,
                     (float)h.lr,
                     (float)(1.0 - h.beta1),
                     (float)(1.0 - h.beta2),
                     (float)h.eps,
                     (float)(1.0 - h.lr * h.weight_decay),
                     (float)h.max_norm,
                     h.norm};
  const dim3 grid((unsigned)(nwork > 0 ? nwork : 1));
  auto* const kernel = bits == 32             ? update_kernel<32, 1>
                       : chunk == kChunkSmall ? update_kernel<8, 1>
                                              : update_kernel<8, 2>;
  static_assert(kChunkSmall == 4 * kBlock && kChunkLarge == 8 * kBlock);
  kernel<<<grid, kBlock, 0, stream>>>(work, nwork, first, count, steps, tickets,
                                      grads, s);
}

int norm_blocks(const Spans& spans) {
  const int chunks = spans.start[spans.count];
  return chunks < kNormBlocks ? chunks : kNormBlocks;
}

void norm_partials(const Spans& spans, double* partials, unsigned* tickets,
                   float* out, hipStream_t stream) {
  static_assert(sizeof(Spans) + 3 * sizeof(void*) <= 4096);  // the arguments
  norm_kernel<<<norm_blocks(spans), kBlock, 0, stream>>>(spans, partials,
                                                         tickets, out);
}

void norm_finish(const double* partials, int count, float* out,
                 hipStream_t stream) {
  norm_finish_kernel<<<1, kBlock, 0, stream>>>(partials, count, out);
}

}  // namespace adamw
