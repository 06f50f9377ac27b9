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
// Every kernel runs over flat chunks of 8192 elements with 8 consecutive elements per
// thread, so 16 lanes hold one block of 128 and its maximum takes four shuffles.
#include <cuda_fp8.h>
#include <math.h>

#include "common.cuh"

namespace thorn {

constexpr int kStThreads = 256;
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

// 32 random bits for elements 4q .. 4q+3 of run `run`: a Weyl sequence through two
// multiply-and-fold rounds (7 integer instructions for four elements).
__device__ __forceinline__ uint32_t round_bits(int64_t q, uint64_t key, uint32_t run) {
  const uint32_t a = (uint32_t)q * 0x9E3779B9u + (uint32_t)key;
  const uint32_t x = mul_fold(a, a ^ ((uint32_t)(key >> 32) ^ ((uint32_t)(q >> 32) + run)));
  return mul_fold(x, x ^ 0xBB67AE85u);
}

// Four values -> four e4m3 codes (element 0 in the low byte), each rounded up in magnitude
// with the probability of its distance to the lower neighbour.  The instruction takes 16
// bits per pair of elements: the second of a pair reads them in reversed order.
__device__ __forceinline__ uint32_t encode4(float y0, float y1, float y2, float y3, uint32_t bits) {
  uint32_t d;
  asm("cvt.rs.satfinite.e4m3x4.f32 %0, {%1, %2, %3, %4}, %5;" : "=r"(d) : "f"(y3), "f"(y2), "f"(y1), "f"(y0), "r"(bits));
  return d;
}

// 8 codes -> 8 fp32 values of the codes (the block's scale is not applied)
__device__ __forceinline__ void decode8(uint2 c, float* v) {
  const uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t h0, h1;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
        : "=r"(h0), "=r"(h1)
        : "r"(w[i]));
    unpack2(h0, v[4 * i], v[4 * i + 1], (__half*)nullptr);
    unpack2(h1, v[4 * i + 2], v[4 * i + 3], (__half*)nullptr);
  }
}

// 2^(b - 127), NaN for b = 255
__device__ __forceinline__ float scale_value(uint32_t b) {
  return __uint_as_float(b == 255u ? 0x7fc00000u : (b == 0u ? 0x00400000u : b << 23));
}
// 2^(127 - b), NaN for b = 255
__device__ __forceinline__ float scale_inverse(uint32_t b) {
  return __uint_as_float(b == 255u ? 0x7fc00000u : (254u - b) << 23);
}

// The upper 16 bits of max|v| of 8 values, rounded up: enough for the block's scale (the
// only mantissa it is compared with is 1.75), and two of them fit one shuffle.  Integer
// maxima keep a NaN (its bits are above infinity's).  Magnitudes from 2^128 - 2^120 up
// round to infinity.
__device__ __forceinline__ uint32_t top16(const float* v) {
  uint32_t t = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) t = max(t, __float_as_uint(v[k]) & 0x7fffffffu);
  return (t + 0xffffu) >> 16;
}

// Scale byte of a block from its top16: the smallest power of two with max <= 448 * 2^k
// (448 = 1.75 * 2^8 is the largest e4m3 value); 255 for a block that is not finite.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top >= 0x7f80u) return 255u;
  const int b = (int)((top + 0x1fu) >> 7) - 8;
  return b < 0 ? 0u : (uint32_t)b;
}

// ---------------------------------------------------------------------------
// 8 consecutive elements as they lie in memory
// ---------------------------------------------------------------------------
template <class T>
struct Raw8 {
  uint4 x[sizeof(T) / 2];
};
template <class T>
__device__ __forceinline__ Raw8<T> load_raw(const T* p, int n, bool full) {
  Raw8<T> r;
  if (full) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.x[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    T e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = k < n ? p[k] : from_f<T>(0.f);
    memcpy(&r, e, sizeof(r));
  }
  return r;
}
template <class T>
__device__ __forceinline__ void unpack_raw(const Raw8<T>& r, float* v) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[4 * i] = __uint_as_float(r.x[i].x);
      v[4 * i + 1] = __uint_as_float(r.x[i].y);
      v[4 * i + 2] = __uint_as_float(r.x[i].z);
      v[4 * i + 3] = __uint_as_float(r.x[i].w);
    }
  } else {
    unpack2(r.x[0].x, v[0], v[1], (T*)nullptr);
    unpack2(r.x[0].y, v[2], v[3], (T*)nullptr);
    unpack2(r.x[0].z, v[4], v[5], (T*)nullptr);
    unpack2(r.x[0].w, v[6], v[7], (T*)nullptr);
  }
}
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, int n, bool full) {
  if (full) return *reinterpret_cast<const uint2*>(p);
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < n) w[k >> 2] |= (uint32_t)p[k] << (8 * (k & 3));
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void store_codes(uint8_t* p, uint2 c, int n, bool full) {
  if (full) {
    *reinterpret_cast<uint2*>(p) = c;
    return;
  }
  const uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < n) p[k] = (uint8_t)(w[k >> 2] >> (8 * (k & 3)));
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
  float lr, bc1, bc2;
  int degenerate;
  int vec;
};
struct StAdamScalars {
  float w1, beta2, w2, wd, eps;  // w1 = 1 - beta1, w2 = 1 - beta2, formed in double
};
template <int CAP>
struct StAdamArgs {
  StTable<StAdam, CAP> tb;
  StAdamScalars s;
};

// S8: moments in 8 bits, else fp32.  MASTER: the update is applied to fp32 master weights
// and p receives their rounding.
template <class P, bool S8, bool MASTER, int CAP>
__global__ void __launch_bounds__(kStThreads) adamw_state_kernel(const __grid_constant__ StAdamArgs<CAP> a) {
  using W = std::conditional_t<MASTER, float, P>;
  const int ti = st_find(a.tb, blockIdx.x);
  const StAdam& e = a.tb.t[ti];
  const int64_t base = int64_t(blockIdx.x - a.tb.start[ti]) * kStChunk;
  const P* G = (const P*)e.g;
  W* Wp = MASTER ? (W*)e.w : (W*)e.p;
  const bool apply = e.p != nullptr;
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int it = 0; it < kStChunk / kStStep; ++it) {
    const int64_t i0 = base + it * kStStep + threadIdx.x * 8;
    if (base + it * kStStep >= e.numel) break;
    const int n = (int)max64(0, min64(8, e.numel - i0));
    const bool full = e.vec && n == 8;
    float gv[8], mv[8], vv[8], wv[8];
    unpack_raw(load_raw(G + i0, n, full), gv);
    if constexpr (S8) {
      const uint8_t* M = (const uint8_t*)e.m;
      const uint8_t* V = (const uint8_t*)e.v;
      const uint2 mc = load_codes(M + i0, n, full), vc = load_codes(V + i0, n, full);
      const float ms = scale_value(n > 0 ? e.ms[i0 / kQBlock] : 0u), vs = scale_value(n > 0 ? e.vs[i0 / kQBlock] : 0u);
      decode8(mc, mv);
      decode8(vc, vv);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        mv[k] = k < n ? mv[k] * ms : 0.f;
        vv[k] = k < n ? vv[k] * vs : 0.f;
      }
    } else {
      unpack_raw(load_raw((const float*)e.m + i0, n, full), mv);
      unpack_raw(load_raw((const float*)e.v + i0, n, full), vv);
    }
    if (apply) unpack_raw(load_raw(Wp + i0, n, full), wv);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      mv[k] = __fadd_rn(mv[k], __fmul_rn(__fsub_rn(gv[k], mv[k]), a.s.w1));
      vv[k] = __fadd_rn(__fmul_rn(vv[k], a.s.beta2), __fmul_rn(__fmul_rn(gv[k], gv[k]), a.s.w2));
    }
    if constexpr (S8) {
      uint32_t top = top16(mv) | (top16(vv) << 16);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
      const uint32_t mb = scale_byte(top & 0xffffu), vb = scale_byte(top >> 16);
      const float mi = scale_inverse(mb), vi = scale_inverse(vb);
      const float low = (top >> 16) != 0u ? 0.001953125f : 0.f;  // the smallest code, 2^-9
      uint32_t mc[2], vc[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t r = round_bits(i0 / 4 + h, e.key, 0u);
        float y[4], z[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          y[k] = mv[4 * h + k] * mi;
          z[k] = fmaxf(vv[4 * h + k] * vi, low);
        }
        mc[h] = encode4(y[0], y[1], y[2], y[3], r);
        vc[h] = encode4(z[0], z[1], z[2], z[3], r);
      }
      store_codes((uint8_t*)e.m + i0, make_uint2(mc[0], mc[1]), n, full);
      store_codes((uint8_t*)e.v + i0, make_uint2(vc[0], vc[1]), n, full);
      if ((lane & 15) == 0 && n > 0) {
        e.ms[i0 / kQBlock] = (uint8_t)mb;
        e.vs[i0 / kQBlock] = (uint8_t)vb;
      }
    } else {
      store_n((float*)e.m + i0, mv, n, e.vec);
      store_n((float*)e.v + i0, vv, n, e.vec);
    }
    if (apply) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float u;
        if (e.degenerate) u = mv[k];
        else if (a.s.eps == 0.f) u = atan2f(mv[k] * e.bc1, sqrtf(vv[k] * e.bc2));
        else u = (mv[k] * e.bc1) / (sqrtf(vv[k] * e.bc2) + a.s.eps);
        if (a.s.wd > 0.f && u * wv[k] >= 0.f) u = u + a.s.wd * wv[k];
        wv[k] = wv[k] - e.lr * u;
      }
      if (MASTER) store_n(e.w + i0, wv, n, e.vec);
      store_n((P*)e.p + i0, wv, n, e.vec);
    }
  }
}

// ===========================================================================
// momentum in 8 bits and the Newton-Schulz input
// ===========================================================================
struct StMomentum {
  const void* g;
  uint8_t* m;
  uint8_t* ms;
  void* x;
  float* norm;   // [batch], then [batch][chunks] partial sums of squares
  int64_t batch, cols, ldx;
  int64_t run;   // elements of one matrix
  int64_t chunks;
  uint64_t key;
  int vec;
};
template <int CAP>
struct StMomentumArgs {
  StTable<StMomentum, CAP> tb;
  float beta1;
};

__device__ __forceinline__ void momentum_u8(const float* g, const float* m, float b1, float* u) {
#pragma unroll
  for (int k = 0; k < 8; ++k) u[k] = __fadd_rn(g[k], __fmul_rn(m[k], b1));
}

template <class P, int CAP>
__global__ void __launch_bounds__(kStThreads) momentum8_kernel(const __grid_constant__ StMomentumArgs<CAP> a) {
  __shared__ float red[32];
  const int ti = st_find(a.tb, blockIdx.x);
  const StMomentum& e = a.tb.t[ti];
  const int64_t local = blockIdx.x - a.tb.start[ti];
  const int64_t b = local / e.chunks, base = (local - b * e.chunks) * kStChunk;
  const P* G = (const P*)e.g + b * e.run;
  uint8_t* M = e.m + b * e.run;
  uint8_t* MS = e.ms + b * ((e.run + kQBlock - 1) / kQBlock);
  const int lane = threadIdx.x & 31;
  float sq = 0.f;
#pragma unroll 1
  for (int it = 0; it < kStChunk / kStStep; ++it) {
    const int64_t i0 = base + it * kStStep + threadIdx.x * 8;
    if (base + it * kStStep >= e.run) break;
    const int n = (int)max64(0, min64(8, e.run - i0));
    const bool full = e.vec && n == 8;
    float gv[8], mv[8], u[8];
    unpack_raw(load_raw(G + i0, n, full), gv);
    const uint2 mc = load_codes(M + i0, n, full);
    const float ms = scale_value(n > 0 ? MS[i0 / kQBlock] : 0u);
    decode8(mc, mv);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      mv[k] = k < n ? __fadd_rn(__fmul_rn(mv[k] * ms, a.beta1), gv[k]) : 0.f;
    uint32_t top = top16(mv);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const uint32_t mb = scale_byte(top);
    const float mi = scale_inverse(mb);
    uint2 c;
    c.x = encode4(mv[0] * mi, mv[1] * mi, mv[2] * mi, mv[3] * mi, round_bits(i0 / 4, e.key, (uint32_t)b));
    c.y = encode4(mv[4] * mi, mv[5] * mi, mv[6] * mi, mv[7] * mi, round_bits(i0 / 4 + 1, e.key, (uint32_t)b));
    store_codes(M + i0, c, n, full);
    if ((lane & 15) == 0 && n > 0) MS[i0 / kQBlock] = (uint8_t)mb;
    decode8(c, mv);
    const float mn = scale_value(mb);
#pragma unroll
    for (int k = 0; k < 8; ++k) mv[k] *= mn;
    momentum_u8(gv, mv, a.beta1, u);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) sq = __fmaf_rn(u[k], u[k], sq);
  }
  if (e.x != nullptr) {
    const float tot = block_sum(sq, red);
    if (threadIdx.x == 0) e.norm[e.batch + local] = tot;
  }
}

// One block per matrix: the fixed-order sum of its chunks' partials, and its root.
template <int CAP>
__global__ void __launch_bounds__(kStThreads) momentum8_norm_kernel(const __grid_constant__ StMomentumArgs<CAP> a) {
  __shared__ double red[32];
  const int ti = st_find(a.tb, blockIdx.x);
  const StMomentum& e = a.tb.t[ti];
  const int64_t b = blockIdx.x - a.tb.start[ti];
  const float* part = e.norm + e.batch + b * e.chunks;
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < e.chunks; i += kStThreads) s += (double)part[i];
  s = block_sum_d(s, red);
  if (threadIdx.x == 0) e.norm[b] = sqrtf((float)s);
}

template <class P, class X, int CAP>
__global__ void __launch_bounds__(kStThreads) momentum8_input_kernel(const __grid_constant__ StMomentumArgs<CAP> a) {
  const int ti = st_find(a.tb, blockIdx.x);
  const StMomentum& e = a.tb.t[ti];
  const int64_t local = blockIdx.x - a.tb.start[ti];
  const int64_t b = local / e.chunks, base = (local - b * e.chunks) * kStChunk;
  const P* G = (const P*)e.g + b * e.run;
  const uint8_t* M = e.m + b * e.run;
  const uint8_t* MS = e.ms + b * ((e.run + kQBlock - 1) / kQBlock);
  const int64_t rows = e.run / e.cols;
  X* xb = (X*)e.x + b * rows * e.ldx;
  const float inv = 1.f / (e.norm[b] + 1e-8f);
#pragma unroll 1
  for (int it = 0; it < kStChunk / kStStep; ++it) {
    const int64_t i0 = base + it * kStStep + threadIdx.x * 8;
    const int n = (int)max64(0, min64(8, e.run - i0));
    if (n == 0) break;
    const bool full = e.vec && n == 8;
    float gv[8], mv[8], u[8];
    unpack_raw(load_raw(G + i0, n, full), gv);
    decode8(load_codes(M + i0, n, full), mv);
    const float ms = scale_value(MS[i0 / kQBlock]);
#pragma unroll
    for (int k = 0; k < 8; ++k) mv[k] *= ms;
    momentum_u8(gv, mv, a.beta1, u);
#pragma unroll
    for (int k = 0; k < 8; ++k) u[k] *= inv;
    if (e.ldx == e.cols) {
      store_n(xb + i0, u, n, e.vec);
    } else {  // rows padded to a longer leading dimension
      int64_t r = i0 / e.cols, c = i0 - r * e.cols;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (k < n) xb[r * e.ldx + c] = from_f<X>(u[k]);
        if (++c == e.cols) {
          c = 0;
          ++r;
        }
      }
    }
  }
}

// ===========================================================================
// apply onto fp32 master weights
// ===========================================================================
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

template <class U, class P, int CAP>
__global__ void __launch_bounds__(kStThreads) apply_master_kernel(const __grid_constant__ StApplyArgs<CAP> a) {
  const int ti = st_find(a.tb, blockIdx.x);
  const StApply& e = a.tb.t[ti];
  const int64_t base = int64_t(blockIdx.x - a.tb.start[ti]) * kStChunk;
#pragma unroll 1
  for (int it = 0; it < kStChunk / kStStep; ++it) {
    const int64_t i0 = base + it * kStStep + threadIdx.x * 8;
    const int n = (int)max64(0, min64(8, e.numel - i0));
    if (n == 0) break;
    const bool full = e.vec && n == 8;
    float uv[8], wv[8];
    unpack_raw(load_raw((const U*)e.U + i0, n, full), uv);
    unpack_raw(load_raw((const float*)e.w + i0, n, full), wv);
    if (e.row_scale != nullptr) {
      int64_t r = i0 / e.cols, c = i0 - r * e.cols;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (k < n) {
          float s = e.row_scale[r];
          if (e.mat_stats != nullptr) {
            const int64_t b = r / e.rows;
            s *= sqrtf(e.mat_stats[2 * b]) / fmaxf(sqrtf(e.mat_stats[2 * b + 1]), kF32Eps);
          }
          uv[k] *= s;
        }
        if (++c == e.cols) {
          c = 0;
          ++r;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float u = uv[k];
      if (a.wd > 0.f && u * wv[k] >= 0.f) u = u + a.wd * wv[k];
      wv[k] = wv[k] - e.lr * u;
    }
    store_n(e.w + i0, wv, n, e.vec);
    store_n((P*)e.p + i0, wv, n, e.vec);
  }
}

// ---------------------------------------------------------------------------
// dispatch
// ---------------------------------------------------------------------------
constexpr int kStCap = 32;  // tensors per launch

static bool st_half(int d) { return d == THORN_BF16 || d == THORN_F16; }
static bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

// elements of a batch of matrices; -1: negative sizes or more than kStMaxElems
static int64_t st_elems(int64_t b, int64_t r, int64_t c) {
  if (b < 0 || r < 0 || c < 0) return -1;
  if (b == 0 || r == 0 || c == 0) return 0;
  if (b > kStMaxElems / r || b * r > kStMaxElems / c) return -1;
  return b * r * c;
}

template <class P, bool S8, bool MASTER>
static int adam_launch(const thorn_adamw_state_tensor* ts, int n, const StAdamScalars& sc, cudaStream_t st) {
  return st_launch<StAdam, kStCap>(
      ts, n,
      [](const thorn_adamw_state_tensor& t, StAdam& e) -> int64_t {
        if ((t.w != nullptr) != MASTER) return 0;
        e = StAdam{t.p, t.g, (float*)t.w, t.m, t.v, (uint8_t*)t.m_scale, (uint8_t*)t.v_scale, t.numel,
                   rounding_key(t.seed), t.lr, t.bc1, t.bc2, t.degenerate, 0};
        const bool mv = S8 ? aligned8(t.m) && aligned8(t.v) : aligned16(t.m) && aligned16(t.v);
        e.vec = mv && aligned16(t.g) && aligned16(t.p) && aligned16(t.w);
        return st_cdiv(t.numel, kStChunk);
      },
      [&](const StTable<StAdam, kStCap>& tb, unsigned nb) {
        StAdamArgs<kStCap> a;
        a.tb = tb;
        a.s = sc;
        adamw_state_kernel<P, S8, MASTER, kStCap><<<nb, kStThreads, 0, st>>>(a);
      });
}

}  // namespace thorn

using namespace thorn;

static StAdamScalars adam_scalars(double beta1, double beta2, float wd, float eps) {
  return StAdamScalars{(float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), wd, eps};
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
  const StAdamScalars sc = adam_scalars(beta1, beta2, weight_decay, eps);
  cudaStream_t st = (cudaStream_t)stream;
  if (p_dtype == THORN_F32) return adam_launch<float, true, false>(ts, n, sc, st);
  int rc;
  if (p_dtype == THORN_BF16) {
    rc = adam_launch<__nv_bfloat16, true, false>(ts, n, sc, st);
    return rc ? rc : adam_launch<__nv_bfloat16, true, true>(ts, n, sc, st);
  }
  rc = adam_launch<__half, true, false>(ts, n, sc, st);
  return rc ? rc : adam_launch<__half, true, true>(ts, n, sc, st);
}

extern "C" int thorn_adamw_master_multi(const thorn_adamw_state_tensor* ts, int n, int p_dtype, double beta1,
                                        double beta2, float weight_decay, float eps, void* stream) {
  if (n < 0 || (n > 0 && ts == nullptr) || !st_half(p_dtype)) return THORN_ERR_ARG;
  for (int i = 0; i < n; ++i) {
    const auto& t = ts[i];
    if (t.numel < 0 || t.numel > kStMaxElems) return THORN_ERR_ARG;
    if (t.numel > 0 && (!t.g || !t.m || !t.v || !t.w)) return THORN_ERR_ARG;
  }
  const StAdamScalars sc = adam_scalars(beta1, beta2, weight_decay, eps);
  cudaStream_t st = (cudaStream_t)stream;
  if (p_dtype == THORN_BF16) return adam_launch<__nv_bfloat16, false, true>(ts, n, sc, st);
  return adam_launch<__half, false, true>(ts, n, sc, st);
}

extern "C" int64_t thorn_momentum8_scratch_bytes(int64_t batch, int64_t rows, int64_t cols) {
  if (st_elems(batch, rows, cols) <= 0) return 0;
  return (batch + batch * st_cdiv(rows * cols, kStChunk)) * (int64_t)sizeof(float);
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
    if (!t.g || !t.m || !t.m_scale || (t.x && (!t.scratch || t.ldx < t.cols || t.ldx > kStMaxElems / (t.batch * t.rows))))
      return THORN_ERR_ARG;
    if (t.batch > kStMaxGrid || t.batch > kStMaxGrid / st_cdiv(t.rows * t.cols, kStChunk)) return THORN_ERR_ARG;
  }
  cudaStream_t st = (cudaStream_t)stream;
  auto entry = [](const thorn_momentum8_tensor& t, StMomentum& e) -> int64_t {
    if (st_elems(t.batch, t.rows, t.cols) <= 0) return 0;
    const int64_t run = t.rows * t.cols;
    e = StMomentum{t.g, (uint8_t*)t.m, (uint8_t*)t.m_scale, t.x, (float*)t.scratch, t.batch, t.cols, t.ldx, run,
                   st_cdiv(run, kStChunk), rounding_key(t.seed), 0};
    e.vec = (t.batch == 1 || run % 8 == 0) && aligned16(t.g) && aligned8(t.m) && aligned16(t.x);
    return t.batch * e.chunks;
  };
  auto with_x = [&](const thorn_momentum8_tensor& t, StMomentum& e) -> int64_t { return t.x ? entry(t, e) : 0; };
  auto each_p = [&](auto f) -> int {
    if (p_dtype == THORN_F32) return f((float*)nullptr);
    if (p_dtype == THORN_BF16) return f((__nv_bfloat16*)nullptr);
    return f((__half*)nullptr);
  };
  auto args = [&](const StTable<StMomentum, kStCap>& tb) {
    StMomentumArgs<kStCap> a;
    a.tb = tb;
    a.beta1 = beta1;
    return a;
  };
  return each_p([&](auto* pp) -> int {
    using P = std::remove_pointer_t<decltype(pp)>;
    int rc = st_launch<StMomentum, kStCap>(ts, n, entry, [&](const StTable<StMomentum, kStCap>& tb, unsigned nb) {
      momentum8_kernel<P, kStCap><<<nb, kStThreads, 0, st>>>(args(tb));
    });
    if (rc) return rc;
    rc = st_launch<StMomentum, kStCap>(
        ts, n, [&](const thorn_momentum8_tensor& t, StMomentum& e) -> int64_t { return with_x(t, e) > 0 ? t.batch : 0; },
        [&](const StTable<StMomentum, kStCap>& tb, unsigned nb) {
          momentum8_norm_kernel<kStCap><<<nb, kStThreads, 0, st>>>(args(tb));
        });
    if (rc) return rc;
    return st_launch<StMomentum, kStCap>(ts, n, with_x, [&](const StTable<StMomentum, kStCap>& tb, unsigned nb) {
      if (x_dtype == THORN_F16) momentum8_input_kernel<P, __half, kStCap><<<nb, kStThreads, 0, st>>>(args(tb));
      else momentum8_input_kernel<P, __nv_bfloat16, kStCap><<<nb, kStThreads, 0, st>>>(args(tb));
    });
  });
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
