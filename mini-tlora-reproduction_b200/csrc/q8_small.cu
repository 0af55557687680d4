// 8-bit products of a few rows (tokens being generated, small batches): the
// weight is the traffic, one byte per element, read once.
//
//   Y[i, j] = s_x[i] s_w[j] sum_k Xq[i, k] Wq[j, k] + bias[j] + sum_c Zt[c][i, :] B_pack[j, chunk c]
//
// k_q8_few: a block owns 16 output channels and its eight warps share out K in
// 128-byte pieces.  A lane's 16-byte loads go straight to registers, two
// pieces (32 KB a block, four blocks an SM) in flight at once, and are the A
// operand of mma.m16n8k32 as they come: the sum over k does not depend on the order of k,
// so the eight tokens of a B operand are read at the same offsets and no data
// is rearranged.  (A 128-row tensor-memory tile would spend 15/16 of its rows
// on nothing, and the tensor pipe is idle either way: HBM feeds a block less
// than one such instruction in 20 cycles.)  The warps' integer sums meet in
// shared memory, one thread finishes one output.
//
// One row 4096 -> 4096 6.4 us (weight bytes: 2.6), 4096 -> 11008 11.6 (6.9), 8192 ->
// 8192 13.7 (10.3), with the launch before it; sixteen rows 8.7, 17.5 and 19.7,
// where reading the rows from L2 for every block costs as much as the weight.
// (32 channels a block halve that but leave SMs idle: 11.5, 15.4 and 23.)
//
// k_few_prep, the launch before it, quantizes the rows and computes the
// low-rank intermediate; k_q8_few starts reading the weight while it runs
// (programmatic dependent launch) and waits for it before it reads a row.
#include "q8.cuh"

namespace mlora {
namespace {

constexpr int kFewThreads = 256, kFewWarps = 8;
constexpr int kFewCh = 16;     // output channels (k_q8_few) or ranks (k_few_prep) of a block
constexpr int kFewPieces = 2;  // pieces of K a warp has in flight

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <class T>
__device__ __forceinline__ void mma_16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  if (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct FewParams {
  int rows, d_in, d_out, R;
  const int8_t* Xq;
  const float* x_scale;
  const int8_t* Wq;
  const float* w_scale;
  const void* bias;
  void* out;
  const int32_t* out_rows;
  int expand;
  PlanDev plan;
  const void* zt;
  const void* pack;
  int pdl;  // launched to overlap the kernel before it
  int* err;
};

__device__ __forceinline__ uint4 ldg_stream(const void* p) {  // read once: leave L1 alone
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// NT = 8-token groups (rows <= 8 NT)
template <class T, int NT>
__global__ void __launch_bounds__(kFewThreads, 4) k_q8_few(const __grid_constant__ FewParams p) {
  __shared__ int sums[kFewWarps][kFewCh][8 * NT + 1];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, q = lane % 4;
  const int n0 = blockIdx.x * kFewCh;
  const int ld = int(q8_ld(p.d_in));
  const int pieces = (ld + 127) / 128;
  // rows g and g + 8 of the block's channels; past d_out: row 0 again, its sums are dropped
  const int8_t* w0 = p.Wq + int64_t(n0 + g < p.d_out ? n0 + g : n0) * ld;
  const int8_t* w1 = p.Wq + int64_t(n0 + g + 8 < p.d_out ? n0 + g + 8 : n0) * ld;
  int acc[NT][4] = {};
  bool waited = false;
  for (int c0 = warp; c0 < pieces; c0 += kFewWarps * kFewPieces) {
    uint4 a[kFewPieces][2][2];  // [piece][16-byte half][row]
#pragma unroll
    for (int i = 0; i < kFewPieces; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = (c0 + i * kFewWarps) * 128 + h * 64 + q * 16;
        a[i][h][0] = k < ld ? ldg_stream(w0 + k) : make_uint4(0, 0, 0, 0);
        a[i][h][1] = k < ld ? ldg_stream(w1 + k) : make_uint4(0, 0, 0, 0);
      }
    if (!waited) {
      if (p.pdl) asm volatile("griddepcontrol.wait;" ::: "memory");
      waited = true;
    }
#pragma unroll
    for (int i = 0; i < kFewPieces; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = (c0 + i * kFewWarps) * 128 + h * 64 + q * 16;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int row = 8 * t + g;
          uint4 b = make_uint4(0, 0, 0, 0);
          if (row < p.rows && k < ld) b = *reinterpret_cast<const uint4*>(p.Xq + int64_t(row) * ld + k);
          const uint4 u = a[i][h][0], v = a[i][h][1];
          mma_s8(acc[t], u.x, v.x, u.y, v.y, b.x, b.y);
          mma_s8(acc[t], u.z, v.z, u.w, v.w, b.z, b.w);
        }
      }
  }
  if (!waited && p.pdl) asm volatile("griddepcontrol.wait;" ::: "memory");
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    sums[warp][g][8 * t + 2 * q] = acc[t][0];
    sums[warp][g][8 * t + 2 * q + 1] = acc[t][1];
    sums[warp][g + 8][8 * t + 2 * q] = acc[t][2];
    sums[warp][g + 8][8 * t + 2 * q + 1] = acc[t][3];
  }
  __syncthreads();
  // 16 consecutive threads: the 16 channels of one row
  const int ch = threadIdx.x % kFewCh, n = n0 + ch;
  const T* bias = static_cast<const T*>(p.bias);
  const T* zt = static_cast<const T*>(p.zt);
  const T* pack = static_cast<const T*>(p.pack);
  T* out = static_cast<T*>(p.out);
  for (int row = threadIdx.x / kFewCh; row < 8 * NT; row += kFewThreads / kFewCh) {
    if (row >= p.rows || n >= p.d_out) continue;
    int s = 0;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) s += sums[w][ch][row];
    float f = float(s) * p.x_scale[row] * __ldg(p.w_scale + n);
    if (p.expand) {
      const int c1 = p.plan.n_chunks;  // all in the one plan tile
      for (int c = 0; c < c1; ++c) {
        const Chunk ck = p.plan.chunks[c];
        if (row < ck.lo || row >= ck.hi) continue;
        constexpr int PER = 16 / int(sizeof(T));
        const uint4* z4 = reinterpret_cast<const uint4*>(zt + (int64_t(c) * kTileRows + row) * kChunk);
        const uint4* b4 = reinterpret_cast<const uint4*>(pack + int64_t(n) * p.R + ck.pcol);
        float e = 0.f;
#pragma unroll
        for (int v = 0; v < kChunk / PER; ++v) {
          const uint4 zv = z4[v], bv = __ldg(b4 + v);
          const T* ze = reinterpret_cast<const T*>(&zv);
          const T* be = reinterpret_cast<const T*>(&bv);
#pragma unroll
          for (int i = 0; i < PER; ++i) e = fmaf(to_f(ze[i]), to_f(be[i]), e);
        }
        f += e;
      }
    }
    if (bias) f += to_f(bias[n]);
    const int64_t orow = p.out_rows ? int64_t(p.out_rows[row]) : row;
    if (orow < 0 || orow >= p.rows) {  // out_rows is not a permutation
      flag_error(p.err, kErrBounds);
      continue;
    }
    out[orow * p.d_out + n] = from_f<T>(f);
  }
}

struct PrepParams {
  int rows, d_in;
  const void* X;
  int8_t* Xq;
  float* x_scale;
  PlanDev plan;
  const void* A_pack;
  void* zt;
};

// Blocks [0, rows): the 8-bit form of a row.  Blocks rows + 4 c + r: ranks 16 r
// .. of chunk c, Zt[c][i, j] = s_a sum_k X[i, k] A_pack[pcol + j, k] on the rows
// of the chunk and zero on the others of the tile.  d_in is a multiple of 8
// and the pointers are 16-byte aligned (16-bit types).
template <class T>
__global__ void __launch_bounds__(kFewThreads) k_few_prep(const __grid_constant__ PrepParams p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ float sums[kFewWarps][kFewCh][17];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const T* X = static_cast<const T*>(p.X);
  if (int(blockIdx.x) < p.rows) {
    quantize_row<T>(X + int64_t(blockIdx.x) * p.d_in, p.d_in, p.Xq + blockIdx.x * q8_ld(p.d_in),
                    p.x_scale + blockIdx.x);
    return;
  }
  const int b = blockIdx.x - p.rows, c = b / 4, j0 = (b % 4) * kFewCh;
  const Chunk ck = p.plan.chunks[c];
  const int g = lane / 4, q = lane % 4;
  const T* a0 = static_cast<const T*>(p.A_pack) + int64_t(ck.pcol + j0 + g) * p.d_in;
  const T* a1 = a0 + int64_t(8) * p.d_in;
  T* zt = static_cast<T*>(p.zt) + int64_t(c) * kTileRows * kChunk + j0;
  const int lo = max(ck.lo, 0), hi = min(ck.hi, p.rows);
  // rows of the tile that are not the chunk's: zero, two 16-byte groups each
  for (int e = threadIdx.x; e < 2 * kTileRows; e += kFewThreads) {
    const int row = e / 2;
    if (row < lo || row >= hi) reinterpret_cast<uint4*>(zt + int64_t(row) * kChunk)[e % 2] = make_uint4(0, 0, 0, 0);
  }
  // 64-element pieces of K: 16-byte loads, as in k_q8_few
  const int pieces = (p.d_in + 63) / 64;
  for (int r0 = lo; r0 < hi; r0 += 16) {
    float acc[2][4] = {};
    for (int c0 = warp; c0 < pieces; c0 += kFewWarps * kFewPieces) {
      uint4 a[kFewPieces][2][2];
#pragma unroll
      for (int i = 0; i < kFewPieces; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = (c0 + i * kFewWarps) * 64 + h * 32 + q * 8;
          a[i][h][0] = k < p.d_in ? ldg_stream(a0 + k) : make_uint4(0, 0, 0, 0);
          a[i][h][1] = k < p.d_in ? ldg_stream(a1 + k) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
      for (int i = 0; i < kFewPieces; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = (c0 + i * kFewWarps) * 64 + h * 32 + q * 8;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int row = r0 + 8 * t + g;
            if (8 * t >= hi - r0) continue;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (row < hi && k < p.d_in) v = __ldg(reinterpret_cast<const uint4*>(X + int64_t(row) * p.d_in + k));
            const uint4 u = a[i][h][0], w = a[i][h][1];
            mma_16<T>(acc[t], u.x, w.x, u.y, w.y, v.x, v.y);
            mma_16<T>(acc[t], u.z, w.z, u.w, w.w, v.z, v.w);
          }
        }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sums[warp][g][8 * t + 2 * q] = acc[t][0];
      sums[warp][g][8 * t + 2 * q + 1] = acc[t][1];
      sums[warp][g + 8][8 * t + 2 * q] = acc[t][2];
      sums[warp][g + 8][8 * t + 2 * q + 1] = acc[t][3];
    }
    __syncthreads();
    const int j = threadIdx.x % kFewCh, row = r0 + threadIdx.x / kFewCh;
    if (row < hi) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) s += sums[w][j][threadIdx.x / kFewCh];
      // rounded to the layer's type, as the tensor-core shrink leaves it: the same
      // block serves the expand here and dB in the backward
      zt[int64_t(row) * kChunk + j] = from_f<T>(ck.scale * s);
    }
  }
}

template <class K, class P>
cudaError_t launch_few(K kern, unsigned grid, cudaStream_t st, bool pdl, const P& prm) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kFewThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, prm);
}

template <class T>
int launch_q8_few(const Q8Main& a, Q8After after, cudaStream_t st) {
  FewParams p;
  memset(&p, 0, sizeof(p));
  p.rows = int(a.M); p.d_in = a.d_in; p.d_out = a.d_out; p.R = a.R;
  p.Xq = a.Aq; p.x_scale = a.a_scale; p.Wq = a.Wq; p.w_scale = a.w_scale;
  p.bias = a.bias; p.out = a.out; p.out_rows = a.out_rows;
  p.expand = a.expand ? 1 : 0;
  if (a.expand) p.plan = a.plan;
  p.zt = a.zt; p.pack = a.pack; p.err = a.err;
  p.pdl = after != kAfterOther && pdl_enabled() ? 1 : 0;
  const unsigned grid = unsigned((a.d_out + kFewCh - 1) / kFewCh);
  if (a.M <= 8) MLORA_CUDA_TRY(launch_few(k_q8_few<T, 1>, grid, st, p.pdl != 0, p));
  else MLORA_CUDA_TRY(launch_few(k_q8_few<T, 2>, grid, st, p.pdl != 0, p));
  count_launch();
  return MLORA_OK;
}

}  // namespace

// The weight-streaming kernel takes up to 16 rows of the forward.  Measured at 16
// rows against the tensor-memory tiles (17 rows): 4096 -> 4096 8.7 and 17.3 us,
// 4096 -> 11008 17.5 and 18.3, 8192 -> 8192 19.7 and 27.5.  With four groups of
// eight rows it took 13 to 16, 32 to 34 and 38 to 42 us for 17 to 31 rows: the
// tiles are faster there on all but the smallest layers.
bool q8_few_ok(const Q8Main& a) {
  return !a.bwd && a.M <= kQ8Few &&
         (!a.expand || (aligned(a.zt, 16) && aligned(a.pack, 16)));  // 16-byte loads of the expand
}

int q8_main_few(const Q8Main& a, Q8After after, cudaStream_t st) {
  if (a.M == 0) return MLORA_OK;
  if (a.dtype == MLORA_BF16) return launch_q8_few<__nv_bfloat16>(a, after, st);
  if (a.dtype == MLORA_F16) return launch_q8_few<__half>(a, after, st);
  return launch_q8_few<float>(a, after, st);
}

// Rows in 8 bits and the low-rank intermediate of a few rows in one launch
// (16-bit types, d_in a multiple of 8, 16-byte aligned tensors).
int q8_few_prep(const void* X, int64_t rows, int d_in, int dtype, int8_t* Xq, float* x_scale, const PlanDev& plan,
                const void* A_pack, void* zt, cudaStream_t st) {
  PrepParams p;
  memset(&p, 0, sizeof(p));
  p.rows = int(rows); p.d_in = d_in; p.X = X; p.Xq = Xq; p.x_scale = x_scale;
  p.plan = plan; p.A_pack = A_pack; p.zt = zt;
  const unsigned grid = unsigned(rows + 4 * plan.n_chunks);
  if (dtype == MLORA_F16) k_few_prep<__half><<<grid, kFewThreads, 0, st>>>(p);
  else k_few_prep<__nv_bfloat16><<<grid, kFewThreads, 0, st>>>(p);
  count_launch();
  return cudaGetLastError() == cudaSuccess ? MLORA_OK : MLORA_ERR_CUDA;
}

}  // namespace mlora
