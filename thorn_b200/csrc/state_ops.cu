// Optimizer state in 8 bits and in 32: (R)Adam(-atan2)W with 8-bit moments or with
// fp32 moments and fp32 master weights, the orthogonalized group's momentum in 8 bits
// with its Newton-Schulz input, and the apply onto fp32 master weights.
//
// 8-bit state: e4m3 codes in blocks of 128 consecutive elements with one power of two
// per block (an e8m0 byte): value = code * 2^(byte - 127).  A power of two makes the
// division by the scale exact, and a float code's relative precision does not depend on
// where in its binade the block's maximum lies.  Codes are rounded stochastically, so a
// change smaller than half a step (a second moment with beta2 near 1) is kept on average
// instead of being lost at every step.
//
// Every kernel runs over flat chunks of 4096 elements with 8 consecutive elements per
// thread, so 16 lanes hold one block of 128 and its maximum takes four shuffles.  Blocks of
// 128 threads: with 256 (chunks of 8192) two 128256 x 4096 tensors took 1729 us instead of
// 1711 and a stack of 4096 matrices of 64 x 64 took 45 us instead of 26.
#include <math.h>

#include "common.cuh"

namespace thorn {

constexpr int kStThreads = 128;
constexpr int kStStep = kStThreads * 8;   // elements per block and iteration
constexpr int kStChunk = 4 * kStStep;     // elements per thread block
constexpr int kQBlock = 128;              // elements per 8-bit scale
constexpr int64_t kStMaxGrid = 1ll << 30;
constexpr int64_t kStMaxElems = kStMaxGrid * kStChunk;  // one launch covers the largest tensor

static inline int64_t st_cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tensors of one launch: a by-value kernel parameter.  Blocks find their tensor by
// bisection of the block prefix.
template <class E, int CAP>
struct StTable {
  E t[CAP];
  uint32_t start[CAP + 1];
  int n;
};

template <class E, int CAP>
__device__ __forceinline__ int st_find(const StTable<E, CAP>& tb, uint32_t bid) {
  int lo = 0, hi = tb.n;  // start[lo] <= bid < start[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tb.start[mid] <= bid) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Fills tables with the tensors that `take` accepts and calls launch(table, blocks) for each.
template <class E, int CAP, class Src, class Take, class Launch>
static int st_launch(const Src* ts, int n, Take take, Launch launch) {
  StTable<E, CAP> tb;
  tb.n = 0;
  int64_t total = 0;
  auto flush = [&]() -> int {
    if (tb.n == 0) return THORN_OK;
    launch(tb, (unsigned)total);
    count_launch();
    tb.n = 0;
    total = 0;
    return check_launch();
  };
  for (int i = 0; i < n; ++i) {
    E e;
    int64_t nb = take(ts[i], e);
    if (nb <= 0) continue;
    if (tb.n == CAP || total + nb > kStMaxGrid) {
      const int st = flush();
      if (st) return st;
    }
    tb.t[tb.n] = e;
    tb.start[tb.n] = (uint32_t)total;
    total += nb;
    tb.start[++tb.n] = (uint32_t)total;
  }
  return flush();
}

// ---------------------------------------------------------------------------
// stochastic rounding
// ---------------------------------------------------------------------------
// Key of a tensor from the caller's seed: two multiply-xorshift rounds (constants: the
// fractional bits of the golden ratio, sqrt 2 and sqrt 3), so that consecutive seeds give
// unrelated keys.
static uint64_t rounding_key(uint64_t seed) {
  uint64_t z = seed + 0x9E3779B97F4A7C15ull;
  z = (z ^ (z >> 32)) * 0x6A09E667F3BCC909ull;
  z = (z ^ (z >> 29)) * 0xBB67AE8584CAA73Bull;
  return z ^ (z >> 32);
}

__device__ __forceinline__ uint32_t mul_fold(uint32_t a, uint32_t b) {
  const uint64_t t = (uint64_t)a * b;
  return (uint32_t)(t >> 32) ^ (uint32_t)t;
}

// 32 random bits for elements 4q .. 4q+3 of a run: a Weyl sequence through two
// multiply-and-fold rounds.  q's upper half and the run enter the second word of the key,
// which a chunk's elements share.
struct Rounding {
  uint32_t a, k;
  __device__ __forceinline__ Rounding(int64_t i0, uint64_t key, uint32_t run) {
    const uint64_t q = (uint64_t)i0 >> 2;
    a = (uint32_t)q * 0x9E3779B9u + (uint32_t)key;
    k = (uint32_t)(key >> 32) ^ ((uint32_t)(q >> 32) + run);
  }
  // for the four elements that follow `step` times four others
  __device__ __forceinline__ uint32_t bits(uint32_t step) const {
    const uint32_t w = a + step * 0x9E3779B9u;
    const uint32_t x = mul_fold(w, w ^ k);
    return mul_fold(x, x ^ 0xBB67AE85u);
  }
};

// Four values -> four e4m3 codes (element 0 in the low byte), each rounded up in magnitude
// with the probability of its distance to the lower neighbour.  The instruction takes 16
// bits per pair of elements: the second of a pair reads them in reversed order.
__device__ __forceinline__ uint32_t encode4(float y0, float y1, float y2, float y3, uint32_t bits) {
  uint32_t d;
  asm("cvt.rs.satfinite.e4m3x4.f32 %0, {%1, %2, %3, %4}, %5;" : "=r"(d) : "f"(y3), "f"(y2), "f"(y1), "f"(y0), "r"(bits));
  return d;
}

// Two fp32 values in one 64-bit register pair: Blackwell's packed multiply and fma round
// each half like the scalar instruction and take one issue slot for both.  The 8-bit
// kernels are bound by instruction issue, not by the fp32 pipes.
using f2 = unsigned long long;
__device__ __forceinline__ f2 pack_f2(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack_f2(f2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ f2 dup(float a) { return pack_f2(a, a); }
__device__ __forceinline__ f2 mul(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 add(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// A packed product and a packed sum may come out as one fma.  Where the product is to be
// rounded for itself, as the definition of the state has it, the sum is written as an fma
// by a one that the compiler does not see (an argument of the kernel).
__device__ __forceinline__ f2 fma(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// 8 codes -> the 8 fp32 values of the codes as pairs (the block's scale is not applied)
__device__ __forceinline__ void decode8(uint2 c, f2* v) {
  const uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t h0, h1;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(h0), "=r"(h1)
        : "r"(w[i]));
    float a, b;
    unpack2(h0, a, b, (__half*)nullptr);
    v[2 * i] = pack_f2(a, b);
    unpack2(h1, a, b, (__half*)nullptr);
    v[2 * i + 1] = pack_f2(a, b);
  }
}
__device__ __forceinline__ uint2 encode8(const f2* y, uint32_t r0, uint32_t r1) {
  float a, b, c, d;
  uint2 o;
  unpack_f2(y[0], a, b);
  unpack_f2(y[1], c, d);
  o.x = encode4(a, b, c, d, r0);
  unpack_f2(y[2], a, b);
  unpack_f2(y[3], c, d);
  o.y = encode4(a, b, c, d, r1);
  return o;
}

// 2^(b - 127); infinity for b = 255, whose codes are NaN
__device__ __forceinline__ float scale_value(uint32_t b) { return __uint_as_float(max(b << 23, 0x00400000u)); }

// The upper 16 bits of max|v| of 8 values, rounded up: enough for the block's scale (the
// only mantissa it is compared with is 1.75), and two of them fit one shuffle.  A NaN
// stays one.  Magnitudes from 2^128 - 2^120 up round to infinity.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t top_up(const f2* v) {
  float x[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) unpack_f2(v[k], x[2 * k], x[2 * k + 1]);
  const float t = max3_abs(max3_abs(x[0], x[1], x[2]), max3_abs(x[3], x[4], x[5]), max3_abs(x[6], x[7], x[7]));
  return __float_as_uint(t) + 0xffffu;
}
__device__ __forceinline__ uint32_t top16(const f2* v) { return top_up(v) >> 16; }

// Scale byte b of a block from its top16, the smallest power of two with max <= 448 * 2^k
// (448 = 1.75 * 2^8 is the largest e4m3 value), and 2^(127 - b).  A block that is not finite
// gets 255 and NaN, which makes all its codes NaN.
__device__ __forceinline__ uint32_t block_scale(uint32_t top, float& inverse) {
  const uint32_t b = (uint32_t)max((int)((top + 0x1fu) >> 7) - 8, 0);
  const bool finite = top < 0x7f80u;
  inverse = __uint_as_float(finite ? (254u - b) << 23 : 0x7fc00000u);
  return finite ? b : 255u;
}

// block_scale of two blocks whose top16 lie in the halves of `top`, in 16-bit pairs.
__device__ __forceinline__ void block_scales(uint32_t top, uint32_t& b0, uint32_t& b1, float& i0, float& i1) {
  const uint32_t q = __vmaxu2(((top + 0x001f001fu) >> 7) & 0x01ff01ffu, 0x00080008u) - 0x00080008u;
  b0 = q & 0xffffu;
  b1 = q >> 16;
  i0 = __uint_as_float((254u - b0) << 23);
  i1 = __uint_as_float((254u - b1) << 23);
  if ((top + 0x00800080u) & 0x80008000u) {  // one of them is not finite
    if ((top & 0xffffu) >= 0x7f80u) b0 = 255u, i0 = __uint_as_float(0x7fc00000u);
    if (top >= 0x7f800000u) b1 = 255u, i1 = __uint_as_float(0x7fc00000u);
  }
}

// ---------------------------------------------------------------------------
// 8 consecutive elements as they lie in memory.  FULL: all 8 are inside the tensor and
// aligned for vector accesses; otherwise `n` says how many are inside, plus kVec where the
// tensor is aligned, and what is not a whole aligned 8 is read one by one, zeros behind.
// ---------------------------------------------------------------------------
constexpr int kVec = 16;
template <class T>
struct Raw8 {
  uint4 x[sizeof(T) / 2];
};
template <bool FULL, class T>
__device__ __forceinline__ void load_raw(const T* p, int n, Raw8<T>& r) {
  if (FULL || n == 8 + kVec) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.x[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    T e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = k < (n & 15) ? p[k] : from_f<T>(0.f);
    memcpy(&r, e, sizeof(r));
  }
}
template <class T>
__device__ __forceinline__ void values(const Raw8<T>& r, f2* v) {
  if constexpr (std::is_same<T, float>::value) {
    memcpy(v, &r, sizeof(r));
  } else {
    const uint32_t w[4] = {r.x[0].x, r.x[0].y, r.x[0].z, r.x[0].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float a, b;
      unpack2(w[k], a, b, (T*)nullptr);
      v[k] = pack_f2(a, b);
    }
  }
}
template <bool FULL, class T>
__device__ __forceinline__ void store8(T* p, const f2* v, int n) {
  if constexpr (FULL && std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < 2; ++i) reinterpret_cast<ulonglong2*>(p)[i] = make_ulonglong2(v[2 * i], v[2 * i + 1]);
  } else {
    float x[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) unpack_f2(v[k], x[2 * k], x[2 * k + 1]);
    store_n(p, x, FULL ? 8 : n & 15, FULL || (n & kVec));
  }
}
template <bool FULL>
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, int n) {
  if (FULL || n == 8 + kVec) return *reinterpret_cast<const uint2*>(p);
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < (n & 15)) w[k >> 2] |= (uint32_t)p[k] << (8 * (k & 3));
  return make_uint2(w[0], w[1]);
}
template <bool FULL>
__device__ __forceinline__ void store_codes(uint8_t* p, uint2 c, int n) {
  if (FULL || n == 8 + kVec) {
    *reinterpret_cast<uint2*>(p) = c;
  } else {
    const uint32_t w[2] = {c.x, c.y};
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < (n & 15)) p[k] = (uint8_t)(w[k >> 2] >> (8 * (k & 3)));
  }
}

// i / cols, by the short division where it does
__device__ __forceinline__ int64_t row_of(int64_t i, int64_t cols) {
  return ((uint64_t)i | (uint64_t)cols) >> 32 ? i / cols : (int64_t)((uint32_t)i / (uint32_t)cols);
}

__device__ __forceinline__ int elems8(int64_t i, int64_t end, int vec) {
  return (int)max64(0, min64(8, end - i)) + (vec ? kVec : 0);
}

// A warp's segment of a chunk is kStSeg consecutive elements, taken 256 at a time: 8 blocks
// of 128, whose 8 scale bytes it reads and writes as one word each.  Bytes written block by
// block and read a moment later from the same 32-byte sector stalled the momentum pass on
// 16384 x 4096 at 145 us.  Iteration `it` of the lanes' half `half` uses byte 2 it + half.
constexpr int kStSeg = kStChunk / (kStThreads / 32);
constexpr int kStIter = kStSeg / 256;
static_assert(kStIter == 4 && kStSeg == 8 * kQBlock, "a segment's scale bytes are one 8-byte word");

// This lane's half's bytes of iterations 0..3, the first in the low byte.  A matrix of a
// stack may start its scales at any byte.
__device__ __forceinline__ uint32_t load_seg_bytes(const uint8_t* p) {
  const int half = (threadIdx.x >> 4) & 1;
  if ((reinterpret_cast<uintptr_t>(p) & 7u) == 0) {
    const uint2 s = *reinterpret_cast<const uint2*>(p);
    return __byte_perm(s.x, s.y, half ? 0x7531 : 0x6420);
  }
  return p[half] | (uint32_t)p[2 + half] << 8 | (uint32_t)p[4 + half] << 16 | (uint32_t)p[6 + half] << 24;
}
__device__ __forceinline__ uint32_t seg_byte(uint32_t b, int it) { return (b >> (8 * it)) & 0xffu; }
__device__ __forceinline__ uint32_t put_byte(uint32_t w, uint32_t b, int it) {
  return __byte_perm(w, b, it == 0 ? 0x3214 : (it == 1 ? 0x3240 : (it == 2 ? 0x3410 : 0x4210)));
}
__device__ __forceinline__ void store_seg_bytes(uint8_t* p, uint32_t b) {
  const uint32_t o = __shfl_xor_sync(0xffffffffu, b, 16);
  if ((threadIdx.x & 31) == 0) {
    const uint2 s = make_uint2(__byte_perm(b, o, 0x5140), __byte_perm(b, o, 0x7362));
    if ((reinterpret_cast<uintptr_t>(p) & 7u) == 0) {
      *reinterpret_cast<uint2*>(p) = s;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) p[k] = (uint8_t)((k < 4 ? s.x : s.y) >> (8 * (k & 3)));
    }
  }
}

// ---------------------------------------------------------------------------
// the update's arithmetic
// ---------------------------------------------------------------------------
__device__ __forceinline__ float rsqrt_approx(float x) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float sqrt_approx(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Second moments under 2^-94 (gradients near 1e-14 and smaller) are out of reach of the short
// arithmetic below: zero over zero, and subnormal numbers, which the approximate instructions
// flush.  A thread that finds one among its eight takes the scaled form for all of them.
constexpr float kLowX2 = 5.0487097934144756e-29f;  // 2^-94
__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ bool any_low(const f2* v) {
  float x[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) unpack_f2(v[k], x[2 * k], x[2 * k + 1]);
  return min3(min3(x[0], x[1], x[2]), min3(x[3], x[4], x[5]), fminf(x[6], x[7])) < kLowX2;
}

// The angle of y over the root of x2 is that of 2^110 y over the root of 2^220 x2: the smallest
// x2 becomes 2^71 and the largest taken here 2^126.  A zero is taken as 2^-126: then zero over
// zero is zero, and the smallest other y, 2^-39 after scaling, is 2^24 times its root.
__device__ __forceinline__ void scale_low(float& y, float& x2) {
  if (x2 < kLowX2) {
    constexpr float s = 1.2980742146337069e33f;  // 2^110
    y *= s;
    x2 = fmaxf(x2 * s * s, 1.17549435e-38f);
  }
}
__device__ __forceinline__ void scale_low2(f2& y, f2& x2) {
  float y0, y1, q0, q1;
  unpack_f2(y, y0, y1);
  unpack_f2(x2, q0, q1);
  scale_low(y0, q0);
  scale_low(y1, q1);
  y = pack_f2(y0, y1);
  x2 = pack_f2(q0, q1);
}

// Square roots of two second moments; LOW: one of them may be below the normal numbers.
template <bool LOW>
__device__ __forceinline__ f2 root2(f2 x2) {
  float a, b;
  unpack_f2(x2, a, b);
  if (!LOW) return pack_f2(sqrt_approx(a), sqrt_approx(b));
  constexpr float up = 1.8446744073709552e19f, down = 2.3283064365386963e-10f;  // 2^64, 2^-32
  return pack_f2(a < kLowX2 ? sqrt_approx(a * up) * down : sqrt_approx(a),
                 b < kLowX2 ? sqrt_approx(b * up) * down : sqrt_approx(b));
}

// Infinity over infinity is one over one.
__device__ __forceinline__ void scale_infinite(float& y, float& x2) {
  if (isinf(y) && isinf(x2)) {
    y = copysignf(1.f, y);
    x2 = 1.f;
  }
}
__device__ __forceinline__ void scale_infinite2(f2& y, f2& x2) {
  float y0, y1, q0, q1;
  unpack_f2(y, y0, y1);
  unpack_f2(x2, q0, q1);
  scale_infinite(y0, q0);
  scale_infinite(y1, q1);
  y = pack_f2(y0, y1);
  x2 = pack_f2(q0, q1);
}

// atan2(y, sqrt(x2)) of two elements, x2 a normal number, or infinite with y finite: with
// t = y / sqrt(x2), atan(s) for s = t where |t| <= 1, else +-pi/2 + atan(s) for s = -1/t.  The
// polynomial in s^2 is the minimax fit of atan(s)/s on [0, 1] with eight coefficients (Remez
// exchange: 9.9e-8 relative, 2.1e-7 with the roundings of its fp32 evaluation).  The general function, with an exact
// square root and divisions, made the first 8-bit step of two 128256 x 4096 tensors 4108 us
// where this made it 3103.
__device__ __forceinline__ f2 angle2(f2 y, f2 x2) {
  float t0, t1, q0, q1;
  unpack_f2(x2, q0, q1);
  unpack_f2(mul(y, pack_f2(rsqrt_approx(q0), rsqrt_approx(q1))), t0, t1);
  float r0 = 0.f, r1 = 0.f;
  if (fabsf(t0) > 1.f) {
    r0 = copysignf(1.57079632679f, t0);
    t0 = rcp_approx(-t0);
  }
  if (fabsf(t1) > 1.f) {
    r1 = copysignf(1.57079632679f, t1);
    t1 = rcp_approx(-t1);
  }
  const f2 s = pack_f2(t0, t1), r = pack_f2(r0, r1);
  const f2 z = mul(s, s);
  f2 p = dup(-0.0046932776f);
  p = fma(p, z, dup(0.02425241f));
  p = fma(p, z, dup(-0.0594864f));
  p = fma(p, z, dup(0.09914293f));
  p = fma(p, z, dup(-0.14019482f));
  p = fma(p, z, dup(0.19969724f));
  p = fma(p, z, dup(-0.3333199f));
  p = fma(p, z, dup(0.9999999f));
  return fma(s, p, r);
}

// ===========================================================================
// (R)Adam(-atan2)W with 8-bit moments, or fp32 moments and fp32 master weights
// ===========================================================================
struct StAdam {
  void* p;
  const void* g;
  float* w;
  void* m;
  void* v;
  uint8_t* ms;
  uint8_t* vs;
  int64_t numel;
  uint64_t key;
  float lr;
  float c, eps;  // bc1 / sqrt(bc2), eps / sqrt(bc2): u = c m / (sqrt(v) + eps)
  int degenerate;
  int vec;
};
struct StAdamScalars {
  float w1, beta2, w2, wd, one;  // w1 = 1 - beta1, w2 = 1 - beta2, formed in double
};
template <int CAP>
struct StAdamArgs {
  StTable<StAdam, CAP> tb;
  StAdamScalars s;
};

// What a thread reads for 8 elements.
template <class P, bool S8, bool MASTER>
struct AdamIn {
  using W = std::conditional_t<MASTER, float, P>;
  using S = std::conditional_t<S8, uint2, Raw8<float>>;
  Raw8<P> g;
  Raw8<W> w;
  S m, v;
};
template <bool FULL, class P, bool S8, bool MASTER>
__device__ __forceinline__ void adam_load(const StAdam& e, int64_t i0, int n, AdamIn<P, S8, MASTER>& in) {
  using W = typename AdamIn<P, S8, MASTER>::W;
  load_raw<FULL>((const P*)e.g + i0, n, in.g);
  if constexpr (S8) {
    in.m = load_codes<FULL>((const uint8_t*)e.m + i0, n);
    in.v = load_codes<FULL>((const uint8_t*)e.v + i0, n);
  } else {
    load_raw<FULL>((const float*)e.m + i0, n, in.m);
    load_raw<FULL>((const float*)e.v + i0, n, in.v);
  }
  if (e.p != nullptr) load_raw<FULL>((const W*)(MASTER ? (void*)e.w : e.p) + i0, n, in.w);
}

// One thread's 8 elements at i0; mb, vb: the scale bytes of their block, read and written.
// The moments are formed with the roundings of separate fp32 operations (the products with
// the power-of-two scales inside the fmas are exact).
template <bool EPS, bool FULL, class P, bool S8, bool MASTER>
__device__ __forceinline__ void adam_step8(const StAdam& e, const StAdamScalars& sc, int64_t i0, int n,
                                           const AdamIn<P, S8, MASTER>& in, const Rounding& rnd, uint32_t step,
                                           uint32_t& mb, uint32_t& vb) {
  f2 g[4], m[4], v[4];
  const f2 w1 = dup(sc.w1), w2 = dup(sc.w2), one = dup(sc.one);
  values(in.g, g);
  if constexpr (S8) {
    decode8(in.m, m);
    decode8(in.v, v);
    const float ms1 = scale_value(mb);
    const f2 ms = dup(ms1), neg = dup(-ms1), vs = dup(scale_value(vb) * sc.beta2);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      m[k] = fma(m[k], ms, mul(fma(m[k], neg, g[k]), w1));
      v[k] = fma(mul(v[k], vs), one, mul(mul(g[k], g[k]), w2));
    }
    uint32_t top = __byte_perm(top_up(m), top_up(v), 0x7632);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
    float mi1, vi1;
    block_scales(top, mb, vb, mi1, vi1);
    const f2 mi = dup(mi1), vi = dup(vi1);
    const uint32_t r0 = rnd.bits(step), r1 = rnd.bits(step + 1);
    f2 y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = mul(m[k], mi);
    store_codes<FULL>((uint8_t*)e.m + i0, encode8(y, r0, r1), n);
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = mul(v[k], vi);
    uint2 c = encode8(y, r0, r1);
    // a second moment beside one that is not zero is held at no less than the smallest code:
    // a byte c + 0x7f has its top bit clear only for c = 0
    if (top >= 0x10000u) {
      c.x |= (~(c.x + 0x7f7f7f7fu) & 0x80808080u) >> 7;
      c.y |= (~(c.y + 0x7f7f7f7fu) & 0x80808080u) >> 7;
    }
    store_codes<FULL>((uint8_t*)e.v + i0, c, n);
  } else {
    values(in.m, m);
    values(in.v, v);
    const f2 b2 = dup(sc.beta2), neg = dup(-1.f);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      m[k] = fma(m[k], one, mul(fma(m[k], neg, g[k]), w1));
      v[k] = fma(mul(v[k], b2), one, mul(mul(g[k], g[k]), w2));
    }
    store8<FULL>((float*)e.m + i0, m, n);
    store8<FULL>((float*)e.v + i0, v, n);
  }
  if (e.p == nullptr) return;
  if (!e.degenerate) {
    const f2 c = dup(e.c);
#pragma unroll
    for (int k = 0; k < 4; ++k) m[k] = mul(m[k], c);
    if constexpr (!EPS) {
      // an 8-bit block with an infinite second moment has the scale byte 255
      const bool infinite = S8 ? vb == 255u : top_up(v) >= 0x7f80ffffu;
      if (any_low(v) || infinite) {
#pragma unroll
        for (int k = 0; k < 4; ++k) scale_low2(m[k], v[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k) scale_infinite2(m[k], v[k]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) m[k] = angle2(m[k], v[k]);
    } else {
      if (any_low(v)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = root2<true>(v[k]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = root2<false>(v[k]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float a, b;
        unpack_f2(v[k], a, b);
        m[k] = mul(m[k], pack_f2(rcp_approx(a + e.eps), rcp_approx(b + e.eps)));
      }
    }
  }
  f2 w[4];
  values(in.w, w);
  if (sc.wd > 0.f) {
    const f2 wd = dup(sc.wd);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float s0, s1, u0, u1, d0, d1;
      unpack_f2(mul(m[k], w[k]), s0, s1);
      unpack_f2(m[k], u0, u1);
      unpack_f2(fma(wd, w[k], m[k]), d0, d1);
      m[k] = pack_f2(s0 >= 0.f ? d0 : u0, s1 >= 0.f ? d1 : u1);
    }
  }
  const f2 lr = dup(-e.lr);
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = fma(lr, m[k], w[k]);
  if constexpr (MASTER) store8<FULL>(e.w + i0, w, n);
  store8<FULL>((P*)e.p + i0, w, n);
}

// S8: moments in 8 bits, else fp32.  MASTER: the update is applied to fp32 master weights
// and p receives their rounding.  EPS: the quotient, else the arc tangent (kernels of their own:
// one with a branch on eps took 2.8 % longer for the two 128256 x 4096 tensors below).
//
// The 8-bit form of 16-bit parameters without masters: 44 instructions per element.  Two
// 128256 x 4096 tensors take 1690 us in a burst of 20 (0.97 of the copy rate) and 1955 where a
// second of it has brought the clock down to 1.62 GHz at 1000 W: there instruction issue binds.
// GPUs differ: 1890 to 2030 in other such runs.  On 16384 x 4096 (115 us) issue slots are 77 %
// busy, DRAM 66 %, at 51 % of the warps.  Nine blocks per SM (56 registers): 1845 us against 1869
// at eight, sustained, in one run of an earlier build; without reading one turn ahead 1909 at
// eight and 1936 at twelve.
// The others are bound by DRAM.  Those that move more bytes per element take six blocks (80
// registers): 377 us for 151936 x 1024 with masters, 450 at the 86 registers that they once took by
// themselves; the fp32 form moves 28 bytes per element at the copy rate (656 us for that size).
template <class P, bool S8, bool MASTER, bool EPS, int CAP>
__global__ void __launch_bounds__(kStThreads, S8 && !MASTER && sizeof(P) == 2 ? 9 : 6)
    adamw_state_kernel(const __grid_constant__ StAdamArgs<CAP> a) {
  const int ti = st_find(a.tb, blockIdx.x);
  const StAdam& e = a.tb.t[ti];
  const int64_t base = int64_t(blockIdx.x - a.tb.start[ti]) * kStChunk;
  const int64_t seg = base + (threadIdx.x >> 5) * kStSeg, i0 = seg + (threadIdx.x & 31) * 8, blk = seg >> 7;
  using In = AdamIn<P, S8, MASTER>;
  const Rounding rnd(i0, e.key, 0u);
  if (e.vec && base + kStChunk <= e.numel) {
    uint32_t ms = 0u, vs = 0u;
    if constexpr (S8) {
      ms = load_seg_bytes(e.ms + blk);
      vs = load_seg_bytes(e.vs + blk);
    }
    uint32_t mout = 0u, vout = 0u;
    In in;
    adam_load<true>(e, i0, 8, in);
#pragma unroll
    for (int it = 0; it < kStIter; ++it) {
      In next;
      if (it + 1 < kStIter) adam_load<true>(e, i0 + (it + 1) * 256, 8, next);
      uint32_t mb = seg_byte(ms, it), vb = seg_byte(vs, it);
      adam_step8<EPS, true>(e, a.s, i0 + it * 256, 8, in, rnd, it * 64, mb, vb);
      mout = put_byte(mout, mb, it);
      vout = put_byte(vout, vb, it);
      in = next;
    }
    if constexpr (S8) {
      store_seg_bytes(e.ms + blk, mout);
      store_seg_bytes(e.vs + blk, vout);
    }
  } else {
#pragma unroll 1
    for (int it = 0; it < kStIter && seg + it * 256 < e.numel; ++it) {
      const int64_t i = i0 + it * 256;
      const int n = elems8(i, e.numel, e.vec);
      const bool some = i < e.numel;
      In in;
      adam_load<false>(e, i, n, in);
      uint32_t mb = 0u, vb = 0u;
      if (S8 && some) {
        mb = e.ms[i >> 7];
        vb = e.vs[i >> 7];
      }
      adam_step8<EPS, false>(e, a.s, i, n, in, rnd, it * 64, mb, vb);
      if (S8 && some && (threadIdx.x & 15) == 0) {
        e.ms[i >> 7] = (uint8_t)mb;
        e.vs[i >> 7] = (uint8_t)vb;
      }
    }
  }
}

// ===========================================================================
// momentum in 8 bits and the Newton-Schulz input
// ===========================================================================
// Matrices of one tensor, as one launch sees them.  Two forms by the matrix's length: up to
// kStChunk elements a group of lanes holds a whole matrix and writes the input from registers.
// Longer matrices take two readings: the momentum leaves one partial sum of squares per chunk,
// and the input reads g and the new codes again.
struct StMomentum {
  const void* g;
  uint8_t* m;
  uint8_t* ms;
  void* x;
  float* part;   // [matrices][chunks] partial sums of squares
  float* norm;   // [matrices] their sums, where a launch of its own forms them
  int64_t run;   // elements of one matrix
  int64_t cols, ldx;
  int64_t batch;
  int64_t chunks;        // of one matrix
  uint64_t key;
  int vec;
};
template <int CAP>
struct StMomentumArgs {
  StTable<StMomentum, CAP> tb;
  float beta1, one;
};

// One matrix of a tensor.
template <class P>
struct StMatrix {
  const P* g;
  uint8_t* m;
  uint8_t* ms;
};
template <class P>
__device__ __forceinline__ StMatrix<P> matrix_of(const StMomentum& e, int64_t b) {
  return StMatrix<P>{(const P*)e.g + b * e.run, e.m + b * e.run, e.ms + b * ((e.run + kQBlock - 1) / kQBlock)};
}

// Momentum of one thread's 8 elements, mb as above; u = g + beta1 m from the rounded m.
template <bool FULL, class P>
__device__ __forceinline__ void momentum_step8(const StMatrix<P>& t, int64_t i0, int n, const Raw8<P>& graw, uint2 c,
                                               uint32_t& mb, float beta1, float onef, const Rounding& rnd,
                                               uint32_t step, f2* u) {
  f2 g[4], m[4];
  values(graw, g);
  decode8(c, m);
  const f2 s = dup(scale_value(mb) * beta1), one = dup(onef);
#pragma unroll
  for (int k = 0; k < 4; ++k) m[k] = fma(mul(m[k], s), one, g[k]);
  uint32_t top = top16(m);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  float inv1;
  mb = block_scale(top, inv1);
  const f2 inv = dup(inv1);
#pragma unroll
  for (int k = 0; k < 4; ++k) m[k] = mul(m[k], inv);
  c = encode8(m, rnd.bits(step), rnd.bits(step + 1));
  store_codes<FULL>(t.m + i0, c, n);
  decode8(c, m);
  const f2 s2 = dup(scale_value(mb) * beta1);
#pragma unroll
  for (int k = 0; k < 4; ++k) u[k] = add(g[k], mul(m[k], s2));
}

// x = u * inv of 8 elements of a matrix
template <bool FULL, class X>
__device__ __forceinline__ void store_input8(const StMomentum& e, X* xb, int64_t i0, int n, f2* u, float inv1) {
  const f2 inv = dup(inv1);
#pragma unroll
  for (int k = 0; k < 4; ++k) u[k] = mul(u[k], inv);
  if (FULL || e.ldx == e.cols) {
    store8<FULL>(xb + i0, u, n);
  } else {  // rows padded to a longer leading dimension
    float v[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) unpack_f2(u[k], v[2 * k], v[2 * k + 1]);
    int64_t r = row_of(i0, e.cols), col = i0 - r * e.cols;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k < (n & 15)) xb[r * e.ldx + col] = from_f<X>(v[k]);
      if (++col == e.cols) {
        col = 0;
        ++r;
      }
    }
  }
}
__device__ __forceinline__ float inverse_norm(float sumsq) { return 1.f / (sqrtf(sumsq) + 1e-8f); }

// Momentum of one chunk by the block; returns this thread's sum of squares of u.
template <class P>
__device__ __forceinline__ float momentum_chunk(const StMomentum& e, float beta1, float onef, int64_t b, int64_t chunk) {
  const int64_t base = chunk * kStChunk;
  const int64_t seg = base + (threadIdx.x >> 5) * kStSeg, i0 = seg + (threadIdx.x & 31) * 8, blk = seg >> 7;
  const StMatrix<P> t = matrix_of<P>(e, b);
  const Rounding rnd(i0, e.key, (uint32_t)b);
  f2 sq = dup(0.f), u[4];
  if (e.vec && base + kStChunk <= e.run) {
    Raw8<P> g[kStIter];
    uint2 c[kStIter];
#pragma unroll
    for (int it = 0; it < kStIter; ++it) {
      load_raw<true>(t.g + i0 + it * 256, 8, g[it]);
      c[it] = load_codes<true>(t.m + i0 + it * 256, 8);
    }
    const uint32_t ms = load_seg_bytes(t.ms + blk);
    uint32_t out = 0u;
#pragma unroll
    for (int it = 0; it < kStIter; ++it) {
      uint32_t mb = seg_byte(ms, it);
      momentum_step8<true>(t, i0 + it * 256, 8, g[it], c[it], mb, beta1, onef, rnd, it * 64, u);
#pragma unroll
      for (int k = 0; k < 4; ++k) sq = fma(u[k], u[k], sq);
      out = put_byte(out, mb, it);
    }
    store_seg_bytes(t.ms + blk, out);
  } else {
#pragma unroll 1
    for (int it = 0; it < kStIter && seg + it * 256 < e.run; ++it) {
      const int64_t i = i0 + it * 256;
      const int n = elems8(i, e.run, e.vec);
      Raw8<P> g;
      load_raw<false>(t.g + i, n, g);
      uint32_t mb = i < e.run ? t.ms[i >> 7] : 0u;
      momentum_step8<false>(t, i, n, g, load_codes<false>(t.m + i, n), mb, beta1, onef, rnd, it * 64, u);
#pragma unroll
      for (int k = 0; k < 4; ++k) sq = fma(u[k], u[k], sq);
      if (i < e.run && (threadIdx.x & 15) == 0) t.ms[i >> 7] = (uint8_t)mb;
    }
  }
  float s0, s1;
  unpack_f2(sq, s0, s1);
  return s0 + s1;
}

// The momentum pass: 4 bytes per element with 16-bit gradients, 19 instructions, which keep
// the issue slots 81 % busy (49 us for 16384 x 4096, its DRAM 61 %; both passes 312 us for the
// 218 M elements of a decoder layer).  Twelve blocks per SM (40 registers): more loads in flight
// than at the registers that it takes by itself (322 us against 339 in an earlier build).  The
// bound is that of 16-bit gradients, which spill 8 bytes; fp32 ones spill 88 (14336 x 4096, both
// passes: 136 us, 90 with bf16 gradients).
template <class P, int CAP>
__global__ void __launch_bounds__(kStThreads, 12) momentum8_kernel(const __grid_constant__ StMomentumArgs<CAP> a) {
  __shared__ float red[32];
  const int ti = st_find(a.tb, blockIdx.x);
  const StMomentum& e = a.tb.t[ti];
  const int64_t local = blockIdx.x - a.tb.start[ti];
  const int64_t b = local / e.chunks;
  const float sq = momentum_chunk<P>(e, a.beta1, a.one, b, local - b * e.chunks);
  if (e.x != nullptr) {
    const float tot = block_sum(sq, red);
    if (threadIdx.x == 0) e.part[local] = tot;
  }
}

// Matrices that LANES lanes hold in IT times 8 elements each: half a warp, a warp or a block
// of them.  Momentum, norm and input at once; the lanes take 8 elements in turn, so that all
// of them have work, and every load is issued before the first is used.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float x, float* red) {
  if constexpr (LANES == kStThreads) {
    return block_sum(x, red);
  } else {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
  }
}
template <class P, class X, int LANES, int IT>
__device__ __forceinline__ void momentum_small(const StMomentum& e, int64_t block, float beta1, float one, float* red) {
  const int64_t first = block * (kStThreads / LANES) + threadIdx.x / LANES;
  const bool live = first < e.batch;  // lanes without a matrix stay for the shuffles
  const int64_t b = live ? first : 0, run = live ? e.run : 0;
  const int64_t i0 = (threadIdx.x % LANES) * 8;
  const StMatrix<P> t = matrix_of<P>(e, b);
  Raw8<P> g[IT];
  uint2 c[IT];
  uint32_t mb[IT];
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int64_t i = i0 + it * (LANES * 8);
    const int n = elems8(i, run, e.vec);
    load_raw<false>(t.g + i, n, g[it]);
    c[it] = load_codes<false>(t.m + i, n);
    mb[it] = i < run ? t.ms[i >> 7] : 0u;
  }
  const Rounding rnd(i0, e.key, (uint32_t)b);
  f2 sq = dup(0.f), u[IT][4];
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int64_t i = i0 + it * (LANES * 8);
    momentum_step8<false>(t, i, elems8(i, run, e.vec), g[it], c[it], mb[it], beta1, one, rnd, it * (LANES * 2), u[it]);
#pragma unroll
    for (int k = 0; k < 4; ++k) sq = fma(u[it][k], u[it][k], sq);
    if (i < run && (threadIdx.x & 15) == 0) t.ms[i >> 7] = (uint8_t)mb[it];
  }
  float s0, s1;
  unpack_f2(sq, s0, s1);
  const float inv = inverse_norm(lanes_sum<LANES>(s0 + s1, red));
  X* xb = (X*)e.x + b * (e.run / e.cols) * e.ldx;
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int64_t i = i0 + it * (LANES * 8);
    if (i < run) store_input8<false>(e, xb, i, elems8(i, run, e.vec), u[it], inv);
  }
}

// Lanes that hold a matrix of up to kStChunk elements.
__host__ __device__ inline int small_lanes(int64_t run) { return run <= 128 ? 16 : (run <= 1024 ? 32 : kStThreads); }

// One launch for all lengths: the 30 tensors of a small convolutional model took 15.2 us,
// 19.5 with the lengths that need one turn in a launch of their own (five blocks per SM) and
// 23.5 with a launch per form; 60000 matrices of 8 x 8 took 18.7 us against 16.5 (floor 4.8: half
// of the 16 lanes have nothing), and 4096 of 64 x 64 take 26.5 (floor 15.7).  The widest form's 80
// registers, with 32 to 48 bytes of spills, are those of all three.
template <class P, class X, int CAP>
__global__ void __launch_bounds__(kStThreads, 6) momentum8_small_kernel(const __grid_constant__ StMomentumArgs<CAP> a) {
  __shared__ float red[32];
  const int ti = st_find(a.tb, blockIdx.x);
  const StMomentum& e = a.tb.t[ti];
  const int64_t block = blockIdx.x - a.tb.start[ti];
  const int lanes = small_lanes(e.run);
  if (lanes == 16) momentum_small<P, X, 16, 1>(e, block, a.beta1, a.one, red);
  else if (lanes == 32) momentum_small<P, X, 32, 4>(e, block, a.beta1, a.one, red);
  else momentum_small<P, X, kStThreads, 4>(e, block, a.beta1, a.one, red);
}

// Partials that an input block sums by itself; the norm of a longer matrix is formed once,
// by a launch between the passes.
constexpr int kOwnSum = 4 * kStThreads;

template <int CAP>
__global__ void __launch_bounds__(1024) momentum8_norm_kernel(const __grid_constant__ StMomentumArgs<CAP> a) {
  __shared__ float red[32];
  const int ti = st_find(a.tb, blockIdx.x);
  const StMomentum& e = a.tb.t[ti];
  const int64_t b = blockIdx.x - a.tb.start[ti];
  const float* part = e.part + b * e.chunks;
  float s = 0.f;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < e.chunks; i += 1024) s += part[i];
  s = block_sum(s, red);
  if (threadIdx.x == 0) e.norm[b] = s;
}

// The input pass: 5 bytes per element, bound by DRAM (47 us for 16384 x 4096, DRAM 75 %).  From
// the last chunk to the first: what the momentum pass read and wrote last is then still in L2.
// Rows padded to a longer leading dimension take the element-wise stores: 4096 x 4097 into rows
// of 4104 takes 74 us with its momentum pass, 31 in its own layout.
template <class P, class X, int CAP>
__global__ void __launch_bounds__(kStThreads) momentum8_input_kernel(const __grid_constant__ StMomentumArgs<CAP> a) {
  __shared__ float red[32];
  const uint32_t bid = gridDim.x - 1 - blockIdx.x;
  const int ti = st_find(a.tb, bid);
  const StMomentum& e = a.tb.t[ti];
  const int64_t local = bid - a.tb.start[ti];
  const int64_t b = local / e.chunks, base = (local - b * e.chunks) * kStChunk;
  const int64_t seg = base + (threadIdx.x >> 5) * kStSeg, i0 = seg + (threadIdx.x & 31) * 8, blk = seg >> 7;
  const StMatrix<P> t = matrix_of<P>(e, b);
  X* xb = (X*)e.x + b * (e.run / e.cols) * e.ldx;
  const bool full = e.vec && e.ldx == e.cols && base + kStChunk <= e.run;
  Raw8<P> g[kStIter];
  uint2 c[kStIter];
  uint32_t ms = 0u;
  if (full) {
#pragma unroll
    for (int it = 0; it < kStIter; ++it) {
      load_raw<true>(t.g + i0 + it * 256, 8, g[it]);
      c[it] = load_codes<true>(t.m + i0 + it * 256, 8);
    }
    ms = load_seg_bytes(t.ms + blk);
  }
  float sumsq;
  if (e.chunks <= kOwnSum) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < kOwnSum / kStThreads; ++k) {
      const int i = k * kStThreads + threadIdx.x;
      if (i < e.chunks) s += e.part[b * e.chunks + i];
    }
    sumsq = block_sum(s, red);
  } else {
    sumsq = e.norm[b];
  }
  const float inv = inverse_norm(sumsq);
  f2 u[4], q[4];
  if (full) {
#pragma unroll
    for (int it = 0; it < kStIter; ++it) {
      values(g[it], q);
      decode8(c[it], u);
      const f2 s = dup(scale_value(seg_byte(ms, it)) * a.beta1);
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = add(q[k], mul(u[k], s));
      store_input8<true>(e, xb, i0 + it * 256, 8, u, inv);
    }
  } else {
#pragma unroll 1
    for (int it = 0; it < kStIter; ++it) {
      const int64_t i = i0 + it * 256;
      if (i >= e.run) break;
      const int n = elems8(i, e.run, e.vec);
      Raw8<P> r;
      load_raw<false>(t.g + i, n, r);
      values(r, q);
      decode8(load_codes<false>(t.m + i, n), u);
      const f2 s = dup(scale_value(t.ms[i >> 7]) * a.beta1);
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = add(q[k], mul(u[k], s));
      store_input8<false>(e, xb, i, n, u, inv);
    }
  }
}

// ===========================================================================
// apply onto fp32 master weights
// ===========================================================================
// 12 bytes per element, bound by DRAM: 391 us for 218 M elements (6.7 TB/s).  The factors are
// formed for every 8 elements and again at each row that they cross: 14336 x 4096 takes 109 us
// without, 111 with row factors and 116 with the matrix's as well; 4096 matrices of 40 x 39 take
// 12.8, 16.8 and 32.4.
struct StApply {
  const void* U;
  void* p;
  float* w;
  const float* row_scale;
  const float* mat_stats;
  int64_t numel, rows, cols;
  float lr;
  int vec;
};
template <int CAP>
struct StApplyArgs {
  StTable<StApply, CAP> tb;
  float wd;
};

constexpr float kF32Eps = 1.1920928955078125e-07f;  // the master weights' type

template <class U, class P, bool FULL>
__device__ __forceinline__ void apply_step8(const StApply& e, float wd, int64_t i0, int n) {
  f2 u[4], w[4];
  Raw8<U> ur;
  Raw8<float> wr;
  load_raw<FULL>((const U*)e.U + i0, n, ur);
  load_raw<FULL>((const float*)e.w + i0, n, wr);
  values(ur, u);
  values(wr, w);
  float uv[8], wv[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    unpack_f2(u[k], uv[2 * k], uv[2 * k + 1]);
    unpack_f2(w[k], wv[2 * k], wv[2 * k + 1]);
  }
  if (e.row_scale != nullptr) {
    int64_t r = row_of(i0, e.cols), c = i0 - r * e.cols;
    auto factor = [&](int64_t row) {
      float s = e.row_scale[row];
      if (e.mat_stats != nullptr) {
        const float* st = e.mat_stats + 2 * row_of(row, e.rows);
        s *= sqrtf(st[0]) / fmaxf(sqrtf(st[1]), kF32Eps);
      }
      return s;
    };
    float s = factor(r);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uv[k] *= s;  // past the end: zeros that are not stored
      if (++c == e.cols) {
        c = 0;
        ++r;
        if (k < 7 && i0 + k + 1 < e.numel) s = factor(r);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (wd > 0.f && uv[k] * wv[k] >= 0.f) uv[k] = fmaf(wd, wv[k], uv[k]);
    wv[k] = fmaf(-e.lr, uv[k], wv[k]);
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = pack_f2(wv[2 * k], wv[2 * k + 1]);
  store8<FULL>(e.w + i0, w, n);
  store8<FULL>((P*)e.p + i0, w, n);
}

template <class U, class P, int CAP>
__global__ void __launch_bounds__(kStThreads) apply_master_kernel(const __grid_constant__ StApplyArgs<CAP> a) {
  const int ti = st_find(a.tb, blockIdx.x);
  const StApply& e = a.tb.t[ti];
  const int64_t base = int64_t(blockIdx.x - a.tb.start[ti]) * kStChunk;
  if (e.vec && base + kStChunk <= e.numel) {
#pragma unroll 1
    for (int it = 0; it < kStChunk / kStStep; ++it)
      apply_step8<U, P, true>(e, a.wd, base + it * kStStep + threadIdx.x * 8, 8);
  } else {
#pragma unroll 1
    for (int it = 0; it < kStChunk / kStStep; ++it) {
      const int64_t i0 = base + it * kStStep + threadIdx.x * 8;
      if (i0 >= e.numel) break;
      const int n = elems8(i0, e.numel, e.vec);
      apply_step8<U, P, false>(e, a.wd, i0, n);
    }
  }
}

// ---------------------------------------------------------------------------
// dispatch
// ---------------------------------------------------------------------------
// Tensors per launch.  A launch costs more with a longer parameter: 4.8 us for one tensor at
// a table of 32 (3 KB), 5.5 at 256.  The AdamW step, which meets many small tensors, takes a
// table of 128 where it gets more than 32: 65 norm weights of 4096 took 21.2 us in three
// launches of 32, 7.4 in one of 128, 11.3 in one of 256.  Momentum and apply keep 32: 64 matrices
// of 128 x 128 take 16.5 us, 32 of them 8.3.
constexpr int kStCap = 32;
constexpr int kStCapMany = 128;


static bool st_half(int d) { return d == THORN_BF16 || d == THORN_F16; }
static bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

// elements of a batch of matrices; -1: negative sizes or more than kStMaxElems
static int64_t st_elems(int64_t b, int64_t r, int64_t c) {
  if (b < 0 || r < 0 || c < 0) return -1;
  if (b == 0 || r == 0 || c == 0) return 0;
  if (b > kStMaxElems / r || b * r > kStMaxElems / c) return -1;
  return b * r * c;
}

template <class P, bool S8, bool MASTER, bool EPS, int CAP>
static int adam_launch(const thorn_adamw_state_tensor* ts, int n, const StAdamScalars& sc, float eps, cudaStream_t st) {
  return st_launch<StAdam, CAP>(
      ts, n,
      [eps](const thorn_adamw_state_tensor& t, StAdam& e) -> int64_t {
        if ((t.w != nullptr) != MASTER) return 0;
        const double root = sqrt((double)t.bc2);
        // an eps stays a normal number: the kernel's reciprocal flushes subnormal arguments
        const float eps_root = fmaxf((float)(eps / root), 1.17549435e-38f);
        e = StAdam{t.p, t.g, (float*)t.w, t.m, t.v, (uint8_t*)t.m_scale, (uint8_t*)t.v_scale, t.numel,
                   rounding_key(t.seed), t.lr, (float)(t.bc1 / root), eps_root, t.degenerate, 0};
        const bool mv = S8 ? aligned8(t.m) && aligned8(t.v) : aligned16(t.m) && aligned16(t.v);
        e.vec = mv && aligned16(t.g) && aligned16(t.p) && aligned16(t.w);
        return st_cdiv(t.numel, kStChunk);
      },
      [&](const StTable<StAdam, CAP>& tb, unsigned nb) {
        StAdamArgs<CAP> a;
        a.tb = tb;
        a.s = sc;
        adamw_state_kernel<P, S8, MASTER, EPS, CAP><<<nb, kStThreads, 0, st>>>(a);
      });
}
template <class P, bool S8, bool MASTER>
static int adam_launch(const thorn_adamw_state_tensor* ts, int n, const StAdamScalars& sc, float eps, cudaStream_t st) {
  const bool many = n > kStCap;
  if (eps > 0.f)
    return many ? adam_launch<P, S8, MASTER, true, kStCapMany>(ts, n, sc, eps, st)
                : adam_launch<P, S8, MASTER, true, kStCap>(ts, n, sc, eps, st);
  return many ? adam_launch<P, S8, MASTER, false, kStCapMany>(ts, n, sc, eps, st)
              : adam_launch<P, S8, MASTER, false, kStCap>(ts, n, sc, eps, st);
}

}  // namespace thorn

using namespace thorn;

static StAdamScalars adam_scalars(double beta1, double beta2, float wd) {
  return StAdamScalars{(float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), wd, 1.f};
}

extern "C" int thorn_adamw8_multi(const thorn_adamw_state_tensor* ts, int n, int p_dtype, double beta1, double beta2,
                                  float weight_decay, float eps, void* stream) {
  if (n < 0 || (n > 0 && ts == nullptr) || (p_dtype != THORN_F32 && !st_half(p_dtype))) return THORN_ERR_ARG;
  for (int i = 0; i < n; ++i) {
    const auto& t = ts[i];
    if (t.numel < 0 || t.numel > kStMaxElems) return THORN_ERR_ARG;
    if (t.numel > 0 && (!t.g || !t.m || !t.v || !t.m_scale || !t.v_scale)) return THORN_ERR_ARG;
    if (t.w && p_dtype == THORN_F32) return THORN_ERR_ARG;
  }
  const StAdamScalars sc = adam_scalars(beta1, beta2, weight_decay);
  cudaStream_t st = (cudaStream_t)stream;
  if (p_dtype == THORN_F32) return adam_launch<float, true, false>(ts, n, sc, eps, st);
  int rc;
  if (p_dtype == THORN_BF16) {
    rc = adam_launch<__nv_bfloat16, true, false>(ts, n, sc, eps, st);
    return rc ? rc : adam_launch<__nv_bfloat16, true, true>(ts, n, sc, eps, st);
  }
  rc = adam_launch<__half, true, false>(ts, n, sc, eps, st);
  return rc ? rc : adam_launch<__half, true, true>(ts, n, sc, eps, st);
}

extern "C" int thorn_adamw_master_multi(const thorn_adamw_state_tensor* ts, int n, int p_dtype, double beta1,
                                        double beta2, float weight_decay, float eps, void* stream) {
  if (n < 0 || (n > 0 && ts == nullptr) || !st_half(p_dtype)) return THORN_ERR_ARG;
  for (int i = 0; i < n; ++i) {
    const auto& t = ts[i];
    if (t.numel < 0 || t.numel > kStMaxElems) return THORN_ERR_ARG;
    if (t.numel > 0 && (!t.g || !t.m || !t.v || !t.w)) return THORN_ERR_ARG;
  }
  const StAdamScalars sc = adam_scalars(beta1, beta2, weight_decay);
  cudaStream_t st = (cudaStream_t)stream;
  if (p_dtype == THORN_BF16) return adam_launch<__nv_bfloat16, false, true>(ts, n, sc, eps, st);
  return adam_launch<__half, false, true>(ts, n, sc, eps, st);
}

extern "C" int64_t thorn_momentum8_scratch_bytes(int64_t batch, int64_t rows, int64_t cols) {
  if (st_elems(batch, rows, cols) <= 0 || rows * cols <= kStChunk) return 0;
  return st_cdiv(batch * (st_cdiv(rows * cols, kStChunk) + 1), 4) * 16;
}

template <class P, class X>
static int momentum_launch(const thorn_momentum8_tensor* ts, int n, float beta1, cudaStream_t st) {
  using Table = StTable<StMomentum, kStCap>;
  auto args = [&](const Table& tb) {
    StMomentumArgs<kStCap> a;
    a.tb = tb;
    a.beta1 = beta1;
    a.one = 1.f;
    return a;
  };
  auto entry = [](const thorn_momentum8_tensor& t) {
    const int64_t run = t.rows * t.cols;
    StMomentum e{};
    e.g = t.g;
    e.m = (uint8_t*)t.m;
    e.ms = (uint8_t*)t.m_scale;
    e.x = t.x;
    e.run = run;
    e.cols = t.cols;
    e.ldx = t.ldx;
    e.batch = t.batch;
    e.chunks = st_cdiv(run, kStChunk);
    e.key = rounding_key(t.seed);
    e.vec = (t.batch == 1 || run % 8 == 0) && aligned16(t.g) && aligned8(t.m) && aligned16(t.x);
    if (t.x && run > kStChunk) {
      e.norm = (float*)t.scratch;
      e.part = e.norm + t.batch;
    }
    return e;
  };
  auto live = [](const thorn_momentum8_tensor& t) { return st_elems(t.batch, t.rows, t.cols) > 0; };
  // matrices that half a warp, a warp or a block holds
  int rc = st_launch<StMomentum, kStCap>(
      ts, n,
      [&](const thorn_momentum8_tensor& t, StMomentum& e) -> int64_t {
        const int64_t run = t.rows * t.cols;
        if (!live(t) || !t.x || run > kStChunk) return 0;
        e = entry(t);
        return st_cdiv(t.batch, kStThreads / small_lanes(run));
      },
      [&](const Table& tb, unsigned nb) { momentum8_small_kernel<P, X, kStCap><<<nb, kStThreads, 0, st>>>(args(tb)); });
  if (rc) return rc;
  // momentum only, or longer than a block holds
  auto is_long = [&](const thorn_momentum8_tensor& t) { return live(t) && (!t.x || t.rows * t.cols > kStChunk); };
  rc = st_launch<StMomentum, kStCap>(
      ts, n,
      [&](const thorn_momentum8_tensor& t, StMomentum& e) -> int64_t {
        if (!is_long(t)) return 0;
        e = entry(t);
        return t.batch * e.chunks;
      },
      [&](const Table& tb, unsigned nb) { momentum8_kernel<P, kStCap><<<nb, kStThreads, 0, st>>>(args(tb)); });
  if (rc) return rc;
  rc = st_launch<StMomentum, kStCap>(
      ts, n,
      [&](const thorn_momentum8_tensor& t, StMomentum& e) -> int64_t {
        if (!is_long(t) || !t.x) return 0;
        e = entry(t);
        return e.chunks > kOwnSum ? t.batch : 0;
      },
      [&](const Table& tb, unsigned nb) { momentum8_norm_kernel<kStCap><<<nb, 1024, 0, st>>>(args(tb)); });
  if (rc) return rc;
  return st_launch<StMomentum, kStCap>(
      ts, n,
      [&](const thorn_momentum8_tensor& t, StMomentum& e) -> int64_t {
        if (!is_long(t) || !t.x) return 0;
        e = entry(t);
        return t.batch * e.chunks;
      },
      [&](const Table& tb, unsigned nb) { momentum8_input_kernel<P, X, kStCap><<<nb, kStThreads, 0, st>>>(args(tb)); });
}

extern "C" int thorn_momentum8_multi(const thorn_momentum8_tensor* ts, int n, int p_dtype, int x_dtype, float beta1,
                                     void* stream) {
  if (n < 0 || (n > 0 && ts == nullptr) || (p_dtype != THORN_F32 && !st_half(p_dtype)) || !st_half(x_dtype))
    return THORN_ERR_ARG;
  for (int i = 0; i < n; ++i) {
    const auto& t = ts[i];
    const int64_t k = st_elems(t.batch, t.rows, t.cols);
    if (k < 0) return THORN_ERR_ARG;
    if (k == 0) continue;
    if (!t.g || !t.m || !t.m_scale) return THORN_ERR_ARG;
    if (t.x && (t.ldx < t.cols || t.ldx > kStMaxElems / (t.batch * t.rows))) return THORN_ERR_ARG;
    if (t.x && t.rows * t.cols > kStChunk && (!t.scratch || !aligned16(t.scratch))) return THORN_ERR_ARG;
    if (t.batch > kStMaxGrid / st_cdiv(t.rows * t.cols, kStChunk)) return THORN_ERR_ARG;
  }
  cudaStream_t st = (cudaStream_t)stream;
  auto with_p = [&](auto* pp) -> int {
    using P = std::remove_pointer_t<decltype(pp)>;
    if (x_dtype == THORN_F16) return momentum_launch<P, __half>(ts, n, beta1, st);
    return momentum_launch<P, __nv_bfloat16>(ts, n, beta1, st);
  };
  if (p_dtype == THORN_F32) return with_p((float*)nullptr);
  if (p_dtype == THORN_BF16) return with_p((__nv_bfloat16*)nullptr);
  return with_p((__half*)nullptr);
}

extern "C" int thorn_apply_master_multi(const thorn_apply_master_tensor* ts, int n, int u_dtype, int p_dtype,
                                        float weight_decay, void* stream) {
  if (n < 0 || (n > 0 && ts == nullptr) || !st_half(u_dtype) || !st_half(p_dtype)) return THORN_ERR_ARG;
  for (int i = 0; i < n; ++i) {
    const int64_t k = st_elems(ts[i].batch, ts[i].rows, ts[i].cols);
    if (k < 0 || (k > 0 && (!ts[i].U || !ts[i].p || !ts[i].w || (ts[i].mat_stats && !ts[i].row_scale))))
      return THORN_ERR_ARG;
  }
  cudaStream_t st = (cudaStream_t)stream;
  auto run = [&](auto* pu, auto* pp) -> int {
    using U = std::remove_pointer_t<decltype(pu)>;
    using P = std::remove_pointer_t<decltype(pp)>;
    return st_launch<StApply, kStCap>(
        ts, n,
        [](const thorn_apply_master_tensor& t, StApply& e) -> int64_t {
          const int64_t k = st_elems(t.batch, t.rows, t.cols);
          if (k <= 0) return 0;
          e = StApply{t.U, t.p, t.w, t.row_scale, t.mat_stats, k, t.rows, t.cols, t.lr, 0};
          e.vec = aligned16(t.U) && aligned16(t.p) && aligned16(t.w);
          return st_cdiv(k, kStChunk);
        },
        [&](const StTable<StApply, kStCap>& tb, unsigned nb) {
          StApplyArgs<kStCap> a;
          a.tb = tb;
          a.wd = weight_decay;
          apply_master_kernel<U, P, kStCap><<<nb, kStThreads, 0, st>>>(a);
        });
  };
  auto with_u = [&](auto* pu) -> int {
    return p_dtype == THORN_BF16 ? run(pu, (__nv_bfloat16*)nullptr) : run(pu, (__half*)nullptr);
  };
  return u_dtype == THORN_BF16 ? with_u((__nv_bfloat16*)nullptr) : with_u((__half*)nullptr);
}
