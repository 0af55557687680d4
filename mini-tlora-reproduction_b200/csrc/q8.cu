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
#include "q8.cuh"

namespace mlora {
namespace {

// round_half_even(x / s) of finite x and s > 0, decided exactly: the
// remainder r = x - q0 s of the rounded fp32 quotient q0 is one fma without
// rounding wherever it decides (x and s have 24 bits and |r| is about s / 2
// there, so r is a multiple of half an ulp of s that fits 24 bits; a larger
// |r| may round, but not past s / 2).
__device__ __forceinline__ int q8_exact(float x, float s) {
  const float q0 = rintf(__fdiv_rn(x, s));
  const float r = fmaf(-q0, s, x), r2 = r + r;
  int q = int(fminf(fmaxf(q0, -128.f), 128.f));
  if (r2 > s || (r2 == s && (q & 1))) ++q;
  else if (r2 < -s || (r2 == -s && (q & 1))) --q;
  return max(-127, min(127, q));  // s may have been rounded down where it is subnormal
}

template <class T> struct Vec8;  // eight elements as loaded
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

// eight elements from column c of a row; past `cols` they are zero
template <class T, bool VEC>
__device__ __forceinline__ Vec8<T> load8(const T* row, int64_t c, int64_t cols) {
  Vec8<T> v;
  if constexpr (VEC) {
    if (c < cols) return *reinterpret_cast<const Vec8<T>*>(row + c);
    memset(&v, 0, sizeof(v));
  } else {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = c + i < cols ? row[c + i] : from_f<T>(0.f);
    memcpy(&v, e, sizeof(v));
  }
  return v;
}

template <class T, bool VEC>
__device__ __forceinline__ void values8(const Vec8<T>& v, const float* col_scale, int64_t c, int64_t cols,
                                        float (&f)[8]) {
  v.get(f);
  if (!col_scale) return;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c + i < cols) f[i] *= __ldg(col_scale + c + i);
}

// The 8-bit row of eight values: bits of t + 1.5 2^23 hold the integer
// nearest t = x (1 / s), whose error is below 127 2^-22; a t within 1e-4 of a
// border is decided exactly (one value in ten thousand).
__device__ __forceinline__ uint2 round8(const float (&f)[8], float s, float inv, bool plain) {
  constexpr float kMagic = 12582912.f;
  int q[8];
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = f[i] * inv, m = t + kMagic;
    q[i] = __float_as_int(m);
    far = fmaxf(far, fabsf(t - (m - kMagic)));
  }
  if (!plain || far > 0.4999f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = s > 0.f ? q8_exact(f[i], s) : 0;
  }
  uint2 w;
  w.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  w.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
  return w;
}

constexpr int kQT = 256;  // threads of a quantizer block

// Scale of a row from its largest magnitude (as float bits); `plain`: the
// reciprocal route of round8 holds (1 / s is finite and accurate).
__device__ __forceinline__ float row_scale(uint32_t top, bool* plain) {
  if (top >= 0x7f800000u) {  // an infinity or a NaN in the row
    *plain = false;
    return __int_as_float(0x7fc00000);
  }
  const float s = __fdiv_rn(__uint_as_float(top), 127.f);
  *plain = s > 1e-30f;
  return s;
}

// `tpr` threads (a power of two, 32..256) per row, kQT / tpr rows per block,
// thread t of a row takes columns 8 t + 8 tpr v.  NV > 0: the row is held in
// registers between the maximum and the rounding; NV = 0: it is read twice.
template <class T, bool VEC, int NV>
__global__ void __launch_bounds__(kQT) k_quantize(const T* __restrict__ src, int64_t rows, int64_t cols, int64_t ld,
                                                   const float* __restrict__ col_scale, int8_t* __restrict__ q,
                                                   float* __restrict__ scale, int tpr) {
  __shared__ uint32_t part[kQT / 32];
  const int t = threadIdx.x % tpr, rb = threadIdx.x / tpr;
  const int64_t row = int64_t(blockIdx.x) * (kQT / tpr) + rb;
  const bool live = row < rows;
  const T* x = src + (live ? row : 0) * ld;
  const int64_t ldq = q8_ld(cols), step = int64_t(tpr) * 8;
  Vec8<T> v[NV > 0 ? NV : 1];
  uint32_t top = 0;
  auto widen = [&](const Vec8<T>& u, int64_t c) {
    float f[8];
    values8<T, VEC>(u, col_scale, c, cols, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
  };
  if (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = load8<T, VEC>(x, live ? t * 8 + i * step : cols, cols);
#pragma unroll
    for (int i = 0; i < NV; ++i) widen(v[i], t * 8 + i * step);
  } else if (live) {
    for (int64_t c = t * 8; c < cols; c += step) widen(load8<T, VEC>(x, c, cols), c);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (tpr > 32) {
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = top;
    __syncthreads();
    const int w0 = rb * (tpr / 32);
    for (int w = 0; w < tpr / 32; ++w) top = max(top, part[w0 + w]);
  }
  if (!live) return;
  bool plain;
  const float s = row_scale(top, &plain);
  const float inv = 1.f / s;
  if (t == 0) scale[row] = s;
  int8_t* out = q + row * ldq;
  auto emit = [&](const Vec8<T>& u, int64_t c) {
    float f[8];
    values8<T, VEC>(u, col_scale, c, cols, f);
    *reinterpret_cast<uint2*>(out + c) = round8(f, s, inv, plain);
  };
  if (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t * 8 + i * step < ldq) emit(v[i], t * 8 + i * step);
  } else {
    for (int64_t c = t * 8; c < ldq; c += step) emit(load8<T, VEC>(x, c, cols), c);
  }
}

template <class T, bool VEC>
int launch_quantize(const T* src, int64_t rows, int64_t cols, int64_t ld, const float* cs, int8_t* q, float* scale,
                    cudaStream_t st) {
  // about four 8-element groups per thread: enough 16-byte loads in flight,
  // few enough registers for full occupancy
  const int64_t groups = q8_ld(cols) / 8;  // the zero bytes past `cols` included
  int tpr = 32;
  while (tpr < kQT && groups > 4 * tpr) tpr *= 2;
  const int64_t per = kQT / tpr, nv = (groups + tpr - 1) / tpr;
  const unsigned grid = unsigned((rows + per - 1) / per);
#define MLORA_QUANT(NV) k_quantize<T, VEC, NV><<<grid, kQT, 0, st>>>(src, rows, cols, ld, cs, q, scale, tpr)
  if (nv <= 1) MLORA_QUANT(1);
  else if (nv <= 2) MLORA_QUANT(2);
  else if (nv <= 4) MLORA_QUANT(4);
  else if (nv <= 8) MLORA_QUANT(8);
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
  const bool vec = aligned(src, 16) && cols % 8 == 0 && (ld * int64_t(sizeof(T))) % 16 == 0;
  return vec ? launch_quantize<T, true>(x, rows, cols, ld, cs, q, scale, st)
             : launch_quantize<T, false>(x, rows, cols, ld, cs, q, scale, st);
}

// dst[i, k] = T(s[i] q[i, k]): one fp32 product, rounded once.  127 s of a row
// whose largest magnitude is that of float32 can round past it: a finite scale
// gives finite values.  A block takes 8-column groups of consecutive rows.
template <class T, bool VEC>
__global__ void __launch_bounds__(256) k_dequantize(const int8_t* __restrict__ q, const float* __restrict__ scale,
                                                     int64_t rows, int64_t cols, T* __restrict__ dst) {
  const int64_t groups = (cols + 7) / 8, ldq = q8_ld(cols), n = rows * groups;
  const int64_t stride = int64_t(gridDim.x) * blockDim.x;
  for (int64_t e = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; e < n; e += stride) {
    const int64_t row = e / groups, c = (e - row * groups) * 8;
    const uint2 w = *reinterpret_cast<const uint2*>(q + row * ldq + c);
    const float s = __ldg(scale + row);
    const float lim = isfinite(s) ? 3.402823466e38f : __int_as_float(0x7fc00000);  // NaN: no limit
    T o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t u = (i < 4 ? w.x : w.y) >> (8 * (i % 4));
      const float v = float(int8_t(u & 0xff)) * s;
      o[i] = from_f<T>(isinf(v) ? copysignf(lim, v) : v);
    }
    T* d = dst + row * cols + c;
    if (VEC) {
      memcpy(__builtin_assume_aligned(d, 16), o, sizeof(o));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < cols) d[i] = o[i];
    }
  }
}

template <class T>
int dequantize_t(const int8_t* q, const float* scale, int64_t rows, int64_t cols, void* dst, cudaStream_t st) {
  const int64_t n = rows * ((cols + 7) / 8);
  const int64_t blocks = (n + 255) / 256;
  const unsigned grid = unsigned(blocks < 65536 * 8 ? blocks : 65536 * 8);
  if (aligned(dst, 16) && cols % 8 == 0)
    k_dequantize<T, true><<<grid, 256, 0, st>>>(q, scale, rows, cols, static_cast<T*>(dst));
  else
    k_dequantize<T, false><<<grid, 256, 0, st>>>(q, scale, rows, cols, static_cast<T*>(dst));
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
__global__ void __launch_bounds__(NT) k_q8_main(Q8Main a) {
  __shared__ int Aw[QK][LD], Bw[QK][LD];
  __shared__ float As[BK][LD], Bs[BK][LD];
  const int n0 = blockIdx.y * BN;
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

template <class T>
int launch_q8_main(const Q8Main& a, cudaStream_t st) {
  const int N = a.bwd ? a.d_in : a.d_out;
  const dim3 grid(unsigned((a.M + BM - 1) / BM), unsigned((N + BN - 1) / BN));
  if (a.bwd) k_q8_main<T, true><<<grid, NT, 0, st>>>(a);
  else k_q8_main<T, false><<<grid, NT, 0, st>>>(a);
  count_launch();
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

int q8_main_simt(const Q8Main& a, cudaStream_t st) {
  if (a.M == 0) return MLORA_OK;
  if (a.dtype == MLORA_BF16) return launch_q8_main<__nv_bfloat16>(a, st);
  if (a.dtype == MLORA_F16) return launch_q8_main<__half>(a, st);
  return launch_q8_main<float>(a, st);
}

}  // namespace mlora
