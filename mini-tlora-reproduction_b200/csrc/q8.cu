// Row quantizer of the 8-bit matrices, its inverse, and the CUDA-core form of
// the 8-bit products.
//
//   s[i] = fl32(max_k |x[i, k]| / 127),   q[i, k] = round_half_even(x[i, k] / s[i])
//
// with x optionally multiplied by a float per column first (one fp32
// rounding).  The quotient is rounded exactly, as if x / s had infinite
// precision, so the integers do not depend on how a kernel forms it.  A row
// of zeros has s = 0 and q = 0; a row that holds an infinity or a NaN has
// s = NaN and q = 0, so that whatever is computed from the row is NaN, as it
// would be from the row itself, and no other row is touched.
#include <algorithm>
#include <type_traits>

#include "q8.cuh"

namespace mlora {
namespace {

// round_half_even(x / s) of finite x and s > 0, decided exactly: the
// remainder r = x - q0 s of the rounded fp32 quotient q0 is one fma without
// rounding wherever it decides (x and s have 24 bits and |r| is about s / 2
// there, so r is a multiple of half an ulp of s that fits 24 bits; a larger
// |r| may round, but not past s / 2).
__device__ __noinline__ int q8_exact(float x, float s) {
  const float q0 = rintf(__fdiv_rn(x, s));
  const float r = fmaf(-q0, s, x), r2 = r + r;
  int q = int(fminf(fmaxf(q0, -128.f), 128.f));
  if (r2 > s || (r2 == s && (q & 1))) ++q;
  else if (r2 < -s || (r2 == -s && (q & 1))) --q;
  return max(-127, min(127, q));  // s may have been rounded down where it is subnormal
}

// Two fp32 operations in one instruction (each rounded as the single one is).
struct F2 {
  uint64_t v;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Eight elements of a row as loaded, their values and the magnitudes' maximum.
template <class T> struct Vec8;
template <> struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
};
template <> struct Vec8<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <> struct Vec8<__half> {
  uint4 a;
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = h.x;
      f[2 * i + 1] = h.y;
    }
  }
};

// Running maximum of magnitudes, as float bits; a NaN stays (it is larger than
// an infinity as bits).  16-bit elements two at a time.
template <class T> struct Pair;
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct Pair<__half> { using type = __half2; };
template <class T> struct Top {
  using P = typename Pair<T>::type;
  uint32_t v = 0;
  __device__ __forceinline__ void see(const Vec8<T>& x) {
    const uint32_t w[4] = {x.a.x & 0x7fff7fffu, x.a.y & 0x7fff7fffu, x.a.z & 0x7fff7fffu, x.a.w & 0x7fff7fffu};
    auto larger = [](uint32_t a, uint32_t b) {
      const P m = __hmax2_nan(*reinterpret_cast<const P*>(&a), *reinterpret_cast<const P*>(&b));
      return *reinterpret_cast<const uint32_t*>(&m);
    };
    v = larger(v, larger(larger(w[0], w[1]), larger(w[2], w[3])));
  }
  __device__ __forceinline__ uint32_t bits() const {
    const float lo = to_f(*reinterpret_cast<const T*>(&v)), hi = to_f(*(reinterpret_cast<const T*>(&v) + 1));
    return max(__float_as_uint(lo) & 0x7fffffffu, __float_as_uint(hi) & 0x7fffffffu);
  }
};
template <> struct Top<float> {
  float v = 0.f;
  __device__ __forceinline__ void see(const Vec8<float>& x) {
    float f[8];
    x.get(f);
#pragma unroll
    for (int i = 0; i < 8; ++i) v = max_nan(v, fabsf(f[i]));
  }
  __device__ __forceinline__ uint32_t bits() const { return __float_as_uint(v); }
};

// eight elements from column c of a row; past `cols` they are zero
template <class T, bool VEC>
__device__ __forceinline__ Vec8<T> load8(const T* row, int64_t c, int64_t cols) {
  Vec8<T> v;
  if constexpr (VEC) {
    memset(&v, 0, sizeof(v));
    if (c < cols) v = *reinterpret_cast<const Vec8<T>*>(row + c);
  } else {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = c + i < cols ? row[c + i] : from_f<T>(0.f);
    memcpy(&v, e, sizeof(v));
  }
  return v;
}

// f *= col_scale[c ..] (fp32, one rounding)
template <bool VEC>
__device__ __forceinline__ void scale8(float (&f)[8], const float* col_scale, int64_t c, int64_t cols) {
  if constexpr (VEC) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (c < cols) {
      a = __ldg(reinterpret_cast<const float4*>(col_scale + c));
      b = __ldg(reinterpret_cast<const float4*>(col_scale + c) + 1);
    }
    mul2(F2(f[0], f[1]), F2(a.x, a.y)).get(f[0], f[1]);
    mul2(F2(f[2], f[3]), F2(a.z, a.w)).get(f[2], f[3]);
    mul2(F2(f[4], f[5]), F2(b.x, b.y)).get(f[4], f[5]);
    mul2(F2(f[6], f[7]), F2(b.z, b.w)).get(f[6], f[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) f[i] *= __ldg(col_scale + c + i);
  }
}

// How the quotients of a row are rounded.  The low bits of x r + 1.5 2^23 (one
// fma) hold the integer nearest x r.
//
// kOne: r = `above` is a reciprocal of s moved by 2^-21, and that one product
// decides.  For 16-bit x and a scale that is their maximum over 127: with
// 11-bit (or 8-bit) significands m1 of x and m2 of the maximum, 127 x / max =
// 127 m1 2^-e / m2 is either a border k + 1/2 or at least a relative
// 1 / (254 m1) > 2^-19 away from it, more than the move and the roundings of s
// and r (2^-21 + 2^-23) bridge.  It is a border only at |x| = max / 2, unless
// 127 divides m2, which makes s exact (such rows are kTwo); there the
// rounding of s decides, and r is moved the way that s was rounded.
//
// kTwo: reciprocals moved by 2^-20 down and up enclose the quotient; where both
// give one integer it is the quotient's, else the sign of x - (n + 1/2) s, which
// one fma has exactly, decides between n and n + 1.
//
// kSlow: s is so small that its reciprocal is not accurate, or 0 or NaN.
enum Rounding { kOne, kTwo, kSlow };
struct RowScale {
  float s, below, above;
  Rounding how;
};

__device__ __forceinline__ uint2 round8(const float (&f)[8], const RowScale& r) {
  constexpr float kMagic = 12582912.f;
  const F2 magic(kMagic, kMagic);
  // the integers of f times a reciprocal, as float bits
  auto round = [&](float by, uint32_t (&o)[8]) {
    const F2 by2(by, by);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      fma2(F2(f[2 * i], f[2 * i + 1]), by2, magic).get(a, b);
      o[2 * i] = __float_as_uint(a);
      o[2 * i + 1] = __float_as_uint(b);
    }
  };
  uint32_t q[8];
  round(r.above, q);
  if (r.how != kOne) {
    uint32_t lo[8], differ = 0;
    round(r.below, lo);
#pragma unroll
    for (int i = 0; i < 8; ++i) differ |= q[i] ^ lo[i];
    if (r.how == kSlow) {
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = r.s > 0.f ? uint32_t(q8_exact(f[i], r.s)) : 0u;
    } else if (differ) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = fminf(__uint_as_float(q[i]), __uint_as_float(lo[i])) - kMagic;
        const float d = fmaf(-(n + 0.5f), r.s, f[i]);
        const uint32_t u = __float_as_uint(n + kMagic);
        if (q[i] != lo[i]) q[i] = u + (d > 0.f || (d == 0.f && (u & 1u)) ? 1u : 0u);
      }
    }
  }
  uint2 w;
  w.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  w.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
  return w;
}

// Scale of a row from its largest magnitude (as float bits); SHORT: the row's
// values have 16-bit significands' precision (see kOne).
template <bool SHORT>
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
  RowScale r;
  if (top >= 0x7f800000u) {  // an infinity or a NaN in the row
    r.s = __int_as_float(0x7fc00000);
    r.below = r.above = 0.f;
    r.how = kSlow;
    return r;
  }
  r.s = __fdiv_rn(__uint_as_float(top), 127.f);
  const float inv = 1.f / r.s;
  r.how = r.s > 1e-30f ? kTwo : kSlow;
  r.below = inv * (1.f - 0x1p-20f);
  r.above = inv * (1.f + 0x1p-20f);
  if (SHORT && r.how == kTwo) {
    const float left = fmaf(-127.f, r.s, __uint_as_float(top));  // > 0: s was rounded down
    if (left != 0.f) {
      r.above = inv * (left > 0.f ? 1.f + 0x1p-21f : 1.f - 0x1p-21f);
      r.how = kOne;
    }
  }
  return r;
}

// Largest block of the kernel that holds NV groups a thread, and the blocks that
// an SM should hold of it (a cap on the registers; 0 = none): with 24 to 32
// warps an SM enough rows are in flight while others are rounded.
template <int NV> constexpr int kQuantThreads = NV == 6 ? 256 : NV == 8 || NV == 12 ? 128 : 512;
template <int NV> constexpr int kQuantBlocks = NV == 6 ? 3 : NV == 8 ? 8 : NV == 12 ? 6 : 0;

// 2^sh threads (32..512) per row, several rows per block; thread t of a row
// takes the 8-column groups t, t + 2^sh, ...  NV > 0: the row (CS: its products
// with the column scales) is held in registers between the maximum and the
// rounding, so it is read once; NV = 0: twice.  Bound by HBM, 2 bytes in and 1
// out per 16-bit element, if the work around each row is spread over enough
// elements of a thread and enough rows are in flight (kQuantBlocks).  65,536 x
// 4096 bf16: 122 us (its bytes: 123; 148 with twice the registers and half the
// warps); float32 200 us (205).  With column scales bf16 4096 columns 148 us, 11,008
// columns 499 (331), float32 4096 columns 232 (205): two more loads and a product
// an element, and values held in float32.
template <class T, bool VEC, bool CS, int NV>
__global__ void __launch_bounds__(kQuantThreads<NV>, kQuantBlocks<NV>)
    k_quantize(const T* __restrict__ src, int64_t rows, int cols, int64_t ld,
                                                   const float* __restrict__ col_scale, int8_t* __restrict__ q,
                                                   float* __restrict__ scale, int sh) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the product after it may start
  using Held = typename std::conditional<CS, Vec8<float>, Vec8<T>>::type;
  using HeldT = typename std::conditional<CS, float, T>::type;
  __shared__ uint32_t part[16];
  const int tpr = 1 << sh, t = threadIdx.x & (tpr - 1);
  const int64_t row = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) >> sh;
  const bool live = row < rows;
  const T* x = src + (live ? row : 0) * ld;
  const int ldq = int(q8_ld(cols)), step = tpr * 8;
  const int end = live ? cols : 0;
  auto product = [&](const Vec8<T>& u, int c) -> Held {
    if constexpr (CS) {
      float f[8];
      u.get(f);
      scale8<VEC>(f, col_scale, c, end);
      Held h;
      h.a = make_float4(f[0], f[1], f[2], f[3]);
      h.b = make_float4(f[4], f[5], f[6], f[7]);
      return h;
    } else {
      return u;
    }
  };
  Held v[NV > 0 ? NV : 1];
  Top<HeldT> most;
  if (NV > 0) {
    Vec8<T> u[NV > 0 ? NV : 1];  // all loads first: they are in flight together
#pragma unroll
    for (int i = 0; i < NV; ++i) u[i] = load8<T, VEC>(x, t * 8 + i * step, end);
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = product(u[i], t * 8 + i * step);
#pragma unroll
    for (int i = 0; i < NV; ++i) most.see(v[i]);
  } else {
    for (int c = t * 8; c < end; c += step) most.see(product(load8<T, VEC>(x, c, end), c));
  }
  uint32_t top = __reduce_max_sync(0xffffffffu, most.bits());
  if (sh > 5) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) part[warp] = top;
    __syncthreads();
    // the warps of this row: 2^(sh - 5) aligned entries
    const int nw = 1 << (sh - 5);
    top = __reduce_max_sync(0xffffffffu, part[(warp & ~(nw - 1)) + (lane & (nw - 1))]);
  }
  if (!live) return;
  const RowScale r = row_scale<!CS && sizeof(T) == 2>(top);
  if (t == 0) scale[row] = r.s;
  int8_t* out = q + row * ldq;
  auto emit = [&](const Held& u, int c) {
    float f[8];
    u.get(f);
    *reinterpret_cast<uint2*>(out + c) = round8(f, r);
  };
  if (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t * 8 + i * step < ldq) emit(v[i], t * 8 + i * step);
  } else {
    for (int c = t * 8; c < ldq; c += step) emit(product(load8<T, VEC>(x, c, end), c), c);
  }
}

// One row by a block of 256 threads, read twice (it is small and stays in L1):
// 16-byte aligned, cols a multiple of 8.
template <class T>
__device__ void quantize_row(const T* x, int cols, int8_t* out, float* scale) {
  __shared__ uint32_t part[8];
  const int ldq = int(q8_ld(cols)), t = threadIdx.x;
  Top<T> most;
  for (int c = t * 8; c < cols; c += 2048) most.see(load8<T, true>(x, c, cols));
  const uint32_t w = __reduce_max_sync(0xffffffffu, most.bits());
  if (t % 32 == 0) part[t / 32] = w;
  __syncthreads();
  const RowScale r = row_scale<true>(__reduce_max_sync(0xffffffffu, part[t & 7]));
  if (t == 0) *scale = r.s;
  for (int c = t * 8; c < ldq; c += 2048) {
    float f[8];
    load8<T, true>(x, c, cols).get(f);
    *reinterpret_cast<uint2*>(out + c) = round8(f, r);
  }
}

// Launch shape of a row kernel over `groups` column groups: the fewest threads
// per row (2^sh) that leave a thread at most `most` groups, and, where the rows
// alone do not fill the SMs, as many as shorten a row's time.
struct RowGrid {
  int sh, block, nv;
  unsigned grid;
};
RowGrid row_grid(int64_t rows, int64_t groups, int most) {
  RowGrid g;
  g.sh = 5;
  while (g.sh < 9 && groups > (int64_t(most) << g.sh)) ++g.sh;
  while (g.sh < 9 && groups > (int64_t(1) << g.sh) && (rows << g.sh) < 148 * 1024) ++g.sh;
  g.block = std::max(1 << g.sh, 128);
  g.nv = int((groups + (int64_t(1) << g.sh) - 1) >> g.sh);
  g.grid = unsigned(((rows << g.sh) + g.block - 1) / g.block);
  return g;
}

template <class T, bool VEC, bool CS>
int launch_quantize(const T* src, int64_t rows, int64_t cols, int64_t ld, const float* cs, int8_t* q, float* scale,
                    cudaStream_t st) {
  const int64_t groups = q8_ld(cols) / 8;  // the zero bytes past `cols` included
  constexpr bool kWide = CS || sizeof(T) == 4;  // held as float32
  const RowGrid g = row_grid(rows, groups, !kWide ? 12 : CS && sizeof(T) == 4 ? 4 : 6);
#define MLORA_QUANT(NV) \
  k_quantize<T, VEC, CS, NV><<<g.grid, g.block, 0, st>>>(src, rows, int(cols), ld, cs, q, scale, g.sh)
  if (g.nv <= 1) MLORA_QUANT(1);
  else if (g.nv <= 2) MLORA_QUANT(2);
  else if (g.nv <= 3) MLORA_QUANT(3);
  else if (g.nv <= 4) MLORA_QUANT(4);
  else if (g.nv <= 6 && g.block <= kQuantThreads<6>) MLORA_QUANT(6);
  else if (g.nv <= 8 && g.block <= kQuantThreads<8>) MLORA_QUANT(8);
  else if (!kWide && g.nv <= 12 && g.block <= kQuantThreads<12>) MLORA_QUANT((kWide ? 0 : 12));
  else if (!kWide && g.nv <= 16) MLORA_QUANT((kWide ? 0 : 16));  // rows over larger blocks
  else if (kWide && g.nv <= 10) MLORA_QUANT((kWide ? 10 : 0));
  else MLORA_QUANT(0);
#undef MLORA_QUANT
  count_launch();
  return cudaGetLastError() == cudaSuccess ? MLORA_OK : MLORA_ERR_CUDA;
}

template <class T>
int quantize_t(const void* src, int64_t rows, int64_t cols, int64_t ld, const float* cs, int8_t* q, float* scale,
               cudaStream_t st) {
  const T* x = static_cast<const T*>(src);
  // 16-byte loads: aligned rows of whole 8-element groups
  const bool vec = aligned(src, 16) && cols % 8 == 0 && (ld * int64_t(sizeof(T))) % 16 == 0 && aligned(cs, 16);
  if (cs)
    return vec ? launch_quantize<T, true, true>(x, rows, cols, ld, cs, q, scale, st)
               : launch_quantize<T, false, true>(x, rows, cols, ld, cs, q, scale, st);
  return vec ? launch_quantize<T, true, false>(x, rows, cols, ld, cs, q, scale, st)
             : launch_quantize<T, false, false>(x, rows, cols, ld, cs, q, scale, st);
}

// dst[i, k] = T(s[i] q[i, k]): one fp32 product, rounded once.  127 s of a row
// whose largest magnitude is that of float32 can round past it: a finite scale
// gives finite float32 values.  Thread t of a row takes the groups t, t + 2^sh,
// ... of 16 bytes of the output (4 or 8 columns); rows of any width (VEC
// false) go element by element, neighbouring threads on neighbouring columns.
// Bound by HBM: 65,536 x 4096 to bf16 123 us, its bytes' time.
template <class T>
__device__ __forceinline__ T q8_value(int q, float s) {
  float v = float(q) * s;
  if (std::is_same<T, float>::value && isinf(v) && isfinite(s)) v = copysignf(3.402823466e38f, v);
  return from_f<T>(v);
}
template <class T, bool VEC>
__global__ void __launch_bounds__(512) k_dequantize(const int8_t* __restrict__ q, const float* __restrict__ scale,
                                                     int64_t rows, int cols, T* __restrict__ dst, int sh) {
  constexpr int PER = VEC ? 16 / int(sizeof(T)) : 1;
  const int tpr = 1 << sh, t = threadIdx.x & (tpr - 1);
  const int64_t row = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) >> sh;
  if (row >= rows) return;
  const float s = __ldg(scale + row);
  const int8_t* in = q + row * q8_ld(cols);
  T* out = dst + row * cols;
#pragma unroll 4
  for (int c = t * PER; c < cols; c += tpr * PER) {
    if constexpr (VEC) {
      alignas(16) T o[PER];
      uint32_t w[2];
      if constexpr (PER == 8) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(in + c));
        w[0] = u.x; w[1] = u.y;
      } else {
        w[0] = __ldg(reinterpret_cast<const uint32_t*>(in + c));
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) o[i] = q8_value<T>(int8_t((w[i / 4] >> (8 * (i % 4))) & 0xff), s);
      *reinterpret_cast<uint4*>(out + c) = *reinterpret_cast<const uint4*>(o);
    } else {
      out[c] = q8_value<T>(in[c], s);
    }
  }
}

template <class T>
int dequantize_t(const int8_t* q, const float* scale, int64_t rows, int64_t cols, void* dst, cudaStream_t st) {
  const bool vec = aligned(dst, 16) && cols % 8 == 0;
  const RowGrid g = row_grid(rows, vec ? cols * int64_t(sizeof(T)) / 16 : cols, 4);
  if (vec)
    k_dequantize<T, true><<<g.grid, g.block, 0, st>>>(q, scale, rows, int(cols), static_cast<T*>(dst), g.sh);
  else
    k_dequantize<T, false><<<g.grid, g.block, 0, st>>>(q, scale, rows, int(cols), static_cast<T*>(dst), g.sh);
  count_launch();
  return cudaGetLastError() == cudaSuccess ? MLORA_OK : MLORA_ERR_CUDA;
}

// ---------------------------------------------------------------- CUDA-core product
// 64 x 64 tile, 4 x 4 outputs per thread, 64 bytes of K per step as 16 words
// of four 8-bit values (dp4a).  Serves what the tensor-core kernel cannot
// describe; the LoRA expand reuses the fp32 tile product of the CUDA-core
// family on the scaled accumulator.
constexpr int QK = 16;  // words of K per step

template <class T, bool BWD>
__global__ void __launch_bounds__(NT) k_q8_main(Q8Main a, int nb0) {
  __shared__ int Aw[QK][LD], Bw[QK][LD];
  __shared__ float As[BK][LD], Bs[BK][LD];
  const int n0 = (nb0 + int(blockIdx.y)) * BN;
  const int64_t m0 = int64_t(blockIdx.x) * BM;
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  const int N = BWD ? a.d_in : a.d_out, K = BWD ? a.d_out : a.d_in;
  const int64_t lda = q8_ld(K), ldw = q8_ld(a.d_in);
  int acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += 4 * QK) {
#pragma unroll
    for (int p = 0; p < (BM * QK) / NT; ++p) {
      const int e = tid + p * NT, r = e / QK, kk = e % QK, k = k0 + 4 * kk;
      const int64_t row = m0 + r;
      // whole words: the bytes from K to the leading dimension are zero
      Aw[kk][r] = row < a.M && k < K ? *reinterpret_cast<const int*>(a.Aq + row * lda + k) : 0;
      if (!BWD) {
        Bw[kk][r] = n0 + r < N && k < K ? *reinterpret_cast<const int*>(a.Wq + int64_t(n0 + r) * ldw + k) : 0;
      } else {
        const int j = e % BN, kb = e / BN, kr = k0 + 4 * kb;  // consecutive threads: consecutive columns
        uint32_t w = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (n0 + j < N && kr + b < K)
            w |= uint32_t(uint8_t(a.Wq[int64_t(kr + b) * ldw + n0 + j])) << (8 * b);
        Bw[kb][j] = int(w);
      }
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < QK; ++kk) {
      int av[4], bv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { av[i] = Aw[kk][ty * 4 + i]; bv[i] = Bw[kk][tx * 4 + i]; }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(av[i], bv[j], acc[i][j]);
    }
    __syncthreads();
  }
  float f[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = m0 + ty * 4 + i;
    const float sa = row < a.M ? a.a_scale[row] : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx * 4 + j;
      f[i][j] = float(acc[i][j]) * sa * (!BWD && n < N ? a.w_scale[n] : 1.f);
    }
  }
  if (a.expand) {
    const int t = int(m0 / kTileRows), rt = int(m0 % kTileRows);
    const T* zt = static_cast<const T*>(a.zt);
    const T* pack = static_cast<const T*>(a.pack);
    for (int c = a.plan.tile_chunk_begin[t]; c < a.plan.tile_chunk_begin[t + 1]; ++c) {
      const Chunk ch = a.plan.chunks[c];
      if (!(ch.lo < rt + BM && ch.hi > rt)) continue;
      const T* zc = zt + int64_t(c) * kTileRows * kChunk + int64_t(rt) * kChunk;
      auto fa = [&](int r, int k) -> float { return to_f(zc[r * kChunk + k]); };
      if (!BWD) {
        auto fb = [&](int j, int k) -> float {
          return n0 + j < N ? to_f(pack[int64_t(n0 + j) * a.R + ch.pcol + k]) : 0.f;
        };
        accum<true, true>(f, fa, fb, kChunk, As, Bs);
      } else {
        auto fb = [&](int j, int k) -> float {
          return n0 + j < N ? to_f(pack[int64_t(ch.pcol + k) * a.d_in + n0 + j]) : 0.f;
        };
        accum<true, false>(f, fa, fb, kChunk, As, Bs);
      }
    }
  }
  const T* bias = static_cast<const T*>(a.bias);
  T* out = static_cast<T*>(a.out);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = m0 + ty * 4 + i;
    if (row >= a.M) continue;
    const int64_t orow = a.out_rows ? int64_t(a.out_rows[row]) : row;
    if (orow < 0 || orow >= a.M) {
      flag_error(a.err, kErrBounds);
      continue;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx * 4 + j;
      if (n >= N) continue;
      float v = f[i][j];
      if (!BWD && bias) v += to_f(bias[n]);
      out[orow * N + n] = from_f<T>(v);
    }
  }
}

// ---------------------------------------------------------------- float32 layers
// The low-rank terms of float32 layers stay on the CUDA cores, next to the
// 8-bit product on the tensor cores.
//
// k_low32: Zt[c] = mask(s_a src A_chunk^T) (forward; K = d_in, a pack row is
// contiguous in k) or dZt[c] = mask(s_a src B_chunk) (backward; K = d_out, a
// pack row holds the ranks of one k).  A block takes kLowRows rows of one
// chunk and its eight warps share out K; lane l sums ranks l and l + 32, the
// warps' sums are added in their order.  Ranks past the adapter's are zero
// without being computed.  640 rows, K = 1024, four jobs: 17 us forward, 12 us
// backward in a running step (the 64 x 64 tile product of the CUDA-core family:
// 105 and 74, with 24 blocks; the bytes and operations: under 1).  Latency of the operands' loads bounds it.
constexpr int kLowRows = 8, kLowWarps = 8, kLowStep = 32;

template <bool BWD>
__global__ void __launch_bounds__(kLowWarps * 32) k_low32(PlanDev plan, const float* __restrict__ src,
                                                          const float* __restrict__ pack, float* __restrict__ zt,
                                                          int64_t M, int K, int64_t ldp) {
  __shared__ float xs[kLowWarps][kLowRows][kLowStep];
  // forward: 32 k x 32 ranks of A per warp; then the warps' sums
  __shared__ float work[kLowWarps * 32 * 33];
  static_assert(sizeof(work) >= sizeof(float) * kLowWarps * kLowRows * kChunk, "the sums fit the pack's space");
  const int c = blockIdx.x, r0 = blockIdx.y * kLowRows;
  const Chunk ch = plan.chunks[c];
  float* out = zt + int64_t(c) * kTileRows * kChunk;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t row0 = int64_t(ch.tile) * kTileRows + r0;
  float (*as)[33] = reinterpret_cast<float (*)[33]>(work + warp * 32 * 33);
  float acc[2][kLowRows] = {};
  if (ch.lo < r0 + kLowRows && ch.hi > r0) {
    for (int k0 = warp * kLowStep; k0 < K; k0 += kLowWarps * kLowStep) {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kLowRows; ++i)
        xs[warp][i][lane] = row0 + i < M && k0 + lane < K ? src[(row0 + i) * K + k0 + lane] : 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int n = ch.nr - 32 * h;  // ranks of this half
        if (n <= 0) continue;
        float b[kLowStep];  // backward: this lane's rank of B, all k of the step
        if (!BWD) {
          __syncwarp();
#pragma unroll 8
          for (int j = 0; j < 32; ++j)
            as[lane][j] = j < n && k0 + lane < K ? __ldg(pack + (ch.pcol + 32 * h + j) * ldp + k0 + lane) : 0.f;
        } else {
#pragma unroll
          for (int kk = 0; kk < kLowStep; ++kk)
            b[kk] = lane < n && k0 + kk < K ? __ldg(pack + int64_t(k0 + kk) * ldp + ch.pcol + 32 * h + lane) : 0.f;
        }
        __syncwarp();
#pragma unroll
        for (int kk = 0; kk < kLowStep; ++kk) {
          const float a = BWD ? b[kk] : as[kk][lane];
#pragma unroll
          for (int i = 0; i < kLowRows; ++i) acc[h][i] = fmaf(xs[warp][i][kk], a, acc[h][i]);
        }
      }
    }
  }
  __syncthreads();
  float (*sums)[kLowRows][kChunk] = reinterpret_cast<float (*)[kLowRows][kChunk]>(work);
#pragma unroll
  for (int i = 0; i < kLowRows; ++i) {
    sums[warp][i][lane] = acc[0][i];
    sums[warp][i][lane + 32] = acc[1][i];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < kLowRows * kChunk; e += kLowWarps * 32) {
    const int i = e / kChunk, j = e % kChunk, r = r0 + i;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kLowWarps; ++w) s += sums[w][i][j];
    out[r * kChunk + j] = r >= ch.lo && r < ch.hi ? ch.scale * s : 0.f;
  }
}

// k_sum32: one 64-column block of d_in of dA (KIND 0; SRC8: from the saved 8-bit
// rows) or of d_out of dB (KIND 1) for one adapter and 16 of its ranks:
//   dA[r, col] = sum_i dZt[i, r] x[i, col],   dB[col, r] = sum_i Zt[i, r] dY[i, col].
// The eight warps share out the rows of each tile, lane l holds columns 2 l and
// 2 l + 1; their sums are added in order.  Only rows of the adapter's segments
// are read.  640 rows x 1024, four jobs: 11 us for dA, 14 us for dB in a running
// step (the CUDA-core family's reduction: 98, over whole tiles with index tables
// in the inner loop; the bytes and operations: under 1).  zt is 16-byte aligned.
constexpr int kSumRanks = 16, kSumCols = 64;
template <int KIND, bool SRC8>
__global__ void __launch_bounds__(256) k_sum32(PlanDev plan, const int8_t* __restrict__ Xq,
                                               const float* __restrict__ x_scale, const float* __restrict__ src,
                                               const float* __restrict__ zt, float* __restrict__ out, int64_t M,
                                               int D, int64_t ldo, float* upd, float lr) {
  __shared__ float sums[8][kSumRanks][kSumCols];
  const ReduceItem it = plan.reduce[blockIdx.x];
  if (it.kind != KIND) return;
  const int j = it.j0 + int(blockIdx.y) / 4, jr = (int(blockIdx.y) % 4) * kSumRanks;  // chunk, first rank in it
  if (int(blockIdx.y) / 4 >= it.nc || j * kChunk + jr >= it.rank) return;
  const int c0 = it.block * 128 + int(blockIdx.z) * kSumCols;
  if (c0 >= D) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, col = c0 + 2 * lane;
  const int64_t ldq = q8_ld(D);
  float acc[kSumRanks][2] = {};
  for (int e = it.lb; e < it.le; ++e) {
    const int c = plan.list[e] + j;
    const Chunk ch = plan.chunks[c];
    const float* z = zt + int64_t(c) * kTileRows * kChunk + jr;
    const int64_t row0 = int64_t(ch.tile) * kTileRows;
#pragma unroll 4
    for (int r = ch.lo + warp; r < ch.hi; r += 8) {
      const int64_t row = row0 + r;
      float x0, x1;
      if (SRC8) {
        const char2 q = col < ldq ? *reinterpret_cast<const char2*>(Xq + row * ldq + col) : make_char2(0, 0);
        const float s = __ldg(x_scale + row);
        x0 = float(q.x) * s;
        x1 = float(q.y) * s;
      } else {
        x0 = col < D ? src[row * D + col] : 0.f;
        x1 = col + 1 < D ? src[row * D + col + 1] : 0.f;
      }
      const float4* z4 = reinterpret_cast<const float4*>(z + r * kChunk);
#pragma unroll
      for (int g = 0; g < kSumRanks / 4; ++g) {
        const float4 w = __ldg(z4 + g);
        const float v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          acc[4 * g + k][0] = fmaf(v[k], x0, acc[4 * g + k][0]);
          acc[4 * g + k][1] = fmaf(v[k], x1, acc[4 * g + k][1]);
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kSumRanks; ++k) {
    sums[warp][k][2 * lane] = acc[k][0];
    sums[warp][k][2 * lane + 1] = acc[k][1];
  }
  __syncthreads();
  const int pcol = plan.chunks[plan.list[it.lb] + j].pcol + jr;
  const int live = it.rank - j * kChunk - jr;
  for (int e = threadIdx.x; e < kSumRanks * kSumCols; e += 256) {
    // consecutive threads: consecutive elements of the output
    const int k = KIND == 0 ? e / kSumCols : e % kSumRanks, x = KIND == 0 ? e % kSumCols : e / kSumRanks;
    if (k >= live || c0 + x >= D) continue;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += sums[w][k][x];
    const int64_t o = KIND == 0 ? int64_t(pcol + k) * ldo + c0 + x : int64_t(c0 + x) * ldo + pcol + k;
    out[o] = s;
    if (upd) sgd_apply(upd + o, s, lr);  // fused SGD step
  }
}

template <class T>
int launch_q8_main(const Q8Main& a, cudaStream_t st) {
  const int N = a.bwd ? a.d_in : a.d_out;
  // the column blocks are the grid's second dimension, which holds 65,535
  const int blocks = (N + BN - 1) / BN;
  for (int nb0 = 0; nb0 < blocks; nb0 += 65535) {
    const dim3 grid(unsigned((a.M + BM - 1) / BM), unsigned(std::min(blocks - nb0, 65535)));
    if (a.bwd) k_q8_main<T, true><<<grid, NT, 0, st>>>(a, nb0);
    else k_q8_main<T, false><<<grid, NT, 0, st>>>(a, nb0);
    count_launch();
  }
  return cudaGetLastError() == cudaSuccess ? MLORA_OK : MLORA_ERR_CUDA;
}

}  // namespace

int q8_quantize(const void* src, int64_t rows, int64_t cols, int64_t ld, int dtype, const float* cs, int8_t* q,
                float* scale, cudaStream_t st) {
  if (rows == 0) return MLORA_OK;
  if (dtype == MLORA_BF16) return quantize_t<__nv_bfloat16>(src, rows, cols, ld, cs, q, scale, st);
  if (dtype == MLORA_F16) return quantize_t<__half>(src, rows, cols, ld, cs, q, scale, st);
  return quantize_t<float>(src, rows, cols, ld, cs, q, scale, st);
}

int q8_dequantize(const int8_t* q, const float* scale, int64_t rows, int64_t cols, int dtype, void* dst,
                  cudaStream_t st) {
  if (rows == 0) return MLORA_OK;
  if (dtype == MLORA_BF16) return dequantize_t<__nv_bfloat16>(q, scale, rows, cols, dst, st);
  if (dtype == MLORA_F16) return dequantize_t<__half>(q, scale, rows, cols, dst, st);
  return dequantize_t<float>(q, scale, rows, cols, dst, st);
}

int q8_low32(bool bwd, const PlanDev& plan, const float* src, const float* pack, float* zt, int64_t M, int d_in,
             int d_out, int R, cudaStream_t st) {
  if (plan.n_chunks == 0) return MLORA_OK;
  const dim3 grid(plan.n_chunks, kTileRows / kLowRows);
  if (bwd) k_low32<true><<<grid, kLowWarps * 32, 0, st>>>(plan, src, pack, zt, M, d_out, R);
  else k_low32<false><<<grid, kLowWarps * 32, 0, st>>>(plan, src, pack, zt, M, d_in, d_in);
  count_launch();
  return cudaGetLastError() == cudaSuccess ? MLORA_OK : MLORA_ERR_CUDA;
}

int q8_sum32(int kind, const PlanDev& plan, const int8_t* Xq, const float* x_scale, const float* src, const float* zt,
             float* out, int64_t M, int D, int64_t ldo, float* upd, float lr, cudaStream_t st) {
  if (plan.n_reduce == 0) return MLORA_OK;
  const dim3 grid(plan.n_reduce, 4 * kMaxChunksPerItem, 128 / kSumCols);
  if (kind == 1) k_sum32<1, false><<<grid, 256, 0, st>>>(plan, nullptr, nullptr, src, zt, out, M, D, ldo, upd, lr);
  else if (Xq) k_sum32<0, true><<<grid, 256, 0, st>>>(plan, Xq, x_scale, nullptr, zt, out, M, D, ldo, upd, lr);
  else k_sum32<0, false><<<grid, 256, 0, st>>>(plan, nullptr, nullptr, src, zt, out, M, D, ldo, upd, lr);
  count_launch();
  return cudaGetLastError() == cudaSuccess ? MLORA_OK : MLORA_ERR_CUDA;
}

int q8_main_simt(const Q8Main& a, cudaStream_t st) {
  if (a.M == 0) return MLORA_OK;
  if (a.dtype == MLORA_BF16) return launch_q8_main<__nv_bfloat16>(a, st);
  if (a.dtype == MLORA_F16) return launch_q8_main<__half>(a, st);
  return launch_q8_main<float>(a, st);
}

}  // namespace mlora
