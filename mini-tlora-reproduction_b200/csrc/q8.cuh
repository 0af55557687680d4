// 8-bit integer matrices: rows of int8 with one float scale per row, the
// quantizer that makes them and the matrix products that read them.
#pragma once

#include "common.cuh"

namespace mlora {

// Leading dimension (bytes) of an 8-bit matrix of `cols` columns: rows start
// on 16-byte boundaries, which TMA and 16-byte loads need; the bytes past
// `cols` are zero.
inline __host__ __device__ int64_t q8_ld(int64_t cols) { return (cols + 15) / 16 * 16; }

// Longest contraction of one product: |q| <= 127, so 127^2 * 131072 is still
// below 2^31 and a 32-bit accumulator cannot overflow.
constexpr int kQ8MaxK = 131072;

int q8_quantize(const void* src, int64_t rows, int64_t cols, int64_t ld_src, int dtype, const float* col_scale,
                int8_t* q, float* scale, cudaStream_t st);
int q8_dequantize(const int8_t* q, const float* scale, int64_t rows, int64_t cols, int dtype, void* dst,
                  cudaStream_t st);

// One 8-bit product with its epilogue.
//   forward   out = s_a[i] s_w[j] sum_k Aq[i, k] Wq[j, k] + bias[j] + sum_c Zt[c] B_pack[j, chunk c]   (N = d_out)
//   backward  out = s_a[i] sum_k Aq[i, k] Wq[k, j] + sum_c dZt[c] A_pack[chunk c, j]                    (N = d_in)
struct Q8Main {
  bool bwd = false;
  int64_t M = 0;
  int d_in = 0, d_out = 0, R = 0, dtype = MLORA_F32;
  const int8_t* Aq = nullptr;      // Xq [M, q8_ld(d_in)] or Gq [M, q8_ld(d_out)]
  const float* a_scale = nullptr;  // [M]
  const int8_t* Wq = nullptr;      // [d_out, q8_ld(d_in)]
  const float* w_scale = nullptr;  // [d_out], forward only (the backward's Gq already holds it)
  const void* bias = nullptr;      // forward only
  void* out = nullptr;
  const int32_t* out_rows = nullptr;
  // LoRA expand: the routing plan and its low-rank blocks (none without chunks)
  bool expand = false;
  PlanDev plan = {};
  const void* zt = nullptr;
  const void* pack = nullptr;  // B_pack or A_pack
  int max_ctas = 0;
  int* err = nullptr;
};

// dA from inputs saved in 8 bits (tensor-core family):
//   dA chunk = sum_i (x_scale[i] dZ[i, :])^T Xq[i, :]
// `scratch`: x_scale dZ as bf16 high and low parts, [2][n_chunks][256][64],
// left by the backward shrink, then the parts of split items.
struct Q8Saved {
  int64_t M = 0;
  int d_in = 0, dtype = MLORA_BF16;
  const int8_t* Xq = nullptr;
  PlanDev plan = {};
  void* scratch = nullptr;
  void* dA = nullptr;
  void* A_upd = nullptr;  // fused SGD step on A_pack
  float lr = 0.f;
  int max_ctas = 0;
};
constexpr int kSavedCols = 256;  // d_in columns of an item

inline size_t q8_dz8_bytes(size_t n_chunks) { return 2 * n_chunks * kTileRows * kChunk * 2; }
inline size_t q8_scratch_bytes(const Plan& p) {
  return q8_dz8_bytes(p.chunks.size()) + size_t(p.saved_parts) * kChunk * kSavedCols * 4;
}
int q8_da_tc(const Q8Saved& a, cudaStream_t st);

// What the launch before an 8-bit product on its stream was: the one that made
// the 8-bit rows, or the shrink that made the low-rank blocks (then the rows
// are older), which both allow the product to start early; or another.
enum Q8After { kAfterOther, kAfterRows, kAfterShrink };

// The forward of at most kQ8Few rows.
constexpr int kQ8Few = 16;
bool q8_few_ok(const Q8Main& a);
int q8_main_few(const Q8Main& a, Q8After after, cudaStream_t st);
int q8_few_prep(const void* X, int64_t rows, int d_in, int dtype, int8_t* Xq, float* x_scale, const PlanDev& plan,
                const void* A_pack, void* zt, cudaStream_t st);

// float32 layers: the low-rank intermediate of all tiles (forward or backward),
// and dA (kind 0, from the saved 8-bit rows Xq or from src = X) or dB (kind 1,
// src = dY).
int q8_low32(bool bwd, const PlanDev& plan, const float* src, const float* pack, float* zt, int64_t M, int d_in,
             int d_out, int R, cudaStream_t st);
int q8_sum32(int kind, const PlanDev& plan, const int8_t* Xq, const float* x_scale, const float* src, const float* zt,
             float* out, int64_t M, int D, int64_t ldo, float* upd, float lr, cudaStream_t st);

int q8_main_simt(const Q8Main& a, cudaStream_t st);
bool q8_tc_ok(const Q8Main& a);
int q8_main_tc(const Q8Main& a, Q8After after, cudaStream_t st);

}  // namespace mlora
