// Tensor-core form of the 8-bit products (tcgen05 kind::i8, s32 accumulators
// in TMEM, operands staged by TMA).
//
//   forward   Y[i, j]  = s_x[i] s_w[j] acc + bias[j] + sum_c Zt[c] Bpack[:, chunk c]^T
//   backward  dX[i, k] = s_g[i] acc + sum_c dZt[c] Apack[chunk c, :]
//
// k_q8: a cluster of two CTAs per 256 x 256 output tile, one
// tcgen05.mma.cta_group::2 (M = 256, N = 256, K = 32) per 32 bytes of K.  A
// k-block is 128 bytes of K per row (128-byte swizzle): 16 KB of A and 16 KB
// of B per CTA, as many bytes as 64 16-bit columns, for twice the products.
// The weight is stored once, [d_out, d_in]: K-major for the forward, MN-major
// for dX.
//
// The LoRA terms are 16-bit products with fp32 sums and the backbone's sums
// are integers, so they cannot share an accumulator from the start.  The
// epilogue warps rewrite a tile's integers in TMEM as the scaled fp32 values
// (tcgen05.ld, multiply, tcgen05.st), the MMA issuer then adds the tile's
// expand k-blocks onto them (kind::f16), and the epilogue drains the sum.
// All of that happens while the next tile's integer mainloop fills the other
// accumulator: its expand k-blocks sit in the ring after the first kDefer
// k-blocks of the next tile, by which time the rewrite has finished.
//
// Bound by power on large shapes: the tensor pipe is active 70 to 82 % at 1.6 to
// 1.65 GHz under the cap (65,536 x 4096 -> 11008: 1.96 ms, 3.0 P op/s; the
// library's integer product 1.81 ms; 8192 rows 297 and 240 us).  At the full rate a 256 x 256 tile also
// takes 64 bytes a cycle into each SM, of which 57 are reached; tiles of 256 x
// 512, which need 48, were built and timed in turn with these: 1 to 3 % faster
// from K = 8192 on, none at K = 4096, slower with few tiles, and not kept.
// The tile order keeps a group of weight blocks in L2 while the rows stream, as
// in the 16-bit mainloops (groups of 4, 8 or 32 blocks instead of 16: 2 to 15 %
// slower, within noise, 1 % faster).  Tiles are dealt round-robin to the
// resident pairs: all tiles of a launch are equal up to a few expand k-blocks.
#include "q8.cuh"

namespace mlora {
namespace {

constexpr int kDefer = 8;       // k-blocks of the next tile before a tile's expand
constexpr int kQ8K = 128;       // bytes of K per k-block
constexpr int kQ8Stages = 6;    // 32 KB per CTA each
constexpr int kQ8StageBytes = 32 * 1024;
// Warps: 0 and 6 issue TMA loads, 1 the MMAs, 2..5 drain columns 0..127 of a
// tile and 8..11 columns 128..255 (a warp reaches the quarter of the TMEM lanes
// that its number modulo four names), 7 has no part.
constexpr int kQ8Threads = 32 * 12;
constexpr int kQ8EpiWarps = 8, kQ8EpiCols = 128;
constexpr int kQ8OutBytes = kQ8EpiWarps * 2048;               // a 32 x 32 slice of 16-bit values per warp
constexpr int kQ8ColBytes = kQ8EpiWarps * 2 * kQ8EpiCols * 4;  // column scales and biases, per warp
constexpr int kQ8Smem = kQ8Stages * kQ8StageBytes + kQ8OutBytes + kQ8ColBytes + 1024 + 512;
static_assert(kQ8Smem <= 232448, "dynamic shared memory above 227 KB");

struct Q8Params {
  CUtensorMap mA, mB;  // 8-bit operands, 128 x 128 byte boxes
  CUtensorMap mZ, mP;  // 16-bit low-rank blocks and pack of the expand
  CUtensorMap mY;      // output store map (tma_out)
  PlanDev plan;
  int64_t M;
  int N;
  int n_tiles, n_nblk, group, n_items;
  int nk;              // 128-byte k-blocks of the integer product
  int a_rows;          // at most 128 rows in all: they are the A box, and the odd CTA loads no A (0: 128-row
                       // boxes in both); the tile's other rows are whatever the ring held, and are not stored
  int expand;
  int dtype;
  int pdl_rows, pdl_z;  // launched to overlap the kernel before it, which makes the 8-bit rows / the
                        // low-rank blocks: wait for it before reading them
  int tma_out;         // 16-bit output rows that TMA can describe, in place
  const float* a_scale;
  const float* w_scale;  // forward
  const void* bias;
  void* out;
  const int32_t* out_rows;
  int* err;
};

__device__ __forceinline__ void tc_mma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
// Instruction descriptor of kind::i8: signed 8-bit A and B, s32 accumulator
__device__ __forceinline__ uint32_t idesc_i8(int m, int n, bool b_mn) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(b_mn) << 16) | (uint32_t(n >> 3) << 17) |
         (uint32_t(m >> 4) << 24);
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const float (&f)[32]) {
  uint32_t r[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(f[i]);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Bounded wait of a whole warp: true only if every lane's wait succeeded, so
// that the lanes go on, or give up, together.
__device__ __forceinline__ bool warp_wait(uint64_t* b, uint32_t parity, volatile int* abort_flag, int* err) {
  return __all_sync(0xffffffffu, mbar_wait(b, parity, abort_flag, err));
}

struct Q8Item {
  int t, nb;   // plan tile, 256-wide N block
  int c0, nc;  // its expand chunks
};

// Item `i` of the launch: groups of `group` N blocks sweep all tiles.
__device__ __forceinline__ Q8Item q8_item(const Q8Params& p, int i) {
  Q8Item it;
  const int per = p.group * p.n_tiles, g = i / per, r = i % per;
  const int n0 = g * p.group, gs = min(p.group, p.n_nblk - n0);
  it.t = r / gs;
  it.nb = n0 + r % gs;
  it.c0 = it.nc = 0;
  if (p.expand) {
    it.c0 = p.plan.tile_chunk_begin[it.t];
    it.nc = p.plan.tile_chunk_begin[it.t + 1] - it.c0;
    if (it.c0 < 0 || it.nc < 0 || it.c0 + it.nc > p.plan.n_chunks) {  // a corrupted plan
      flag_error(p.err, kErrBounds);
      it.c0 = it.nc = 0;
    }
  }
  return it;
}

// bias[n] of an output of type `dtype`
__device__ __forceinline__ float q8_bias(const Q8Params& p, int n) {
  if (p.dtype == MLORA_BF16) return to_f(static_cast<const __nv_bfloat16*>(p.bias)[n]);
  if (p.dtype == MLORA_F16) return to_f(static_cast<const __half*>(p.bias)[n]);
  return static_cast<const float*>(p.bias)[n];
}
__device__ __forceinline__ float4 lds_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

// One 32 x 32 slice of finished values (lane = row row_w0 + lane, columns n..)
// to the output.  Warp-collective.
__device__ __forceinline__ void q8_store_slice(const Q8Params& p, const float (&f)[32], int64_t row_w0, int n,
                                               uint32_t buf, int lane) {
  const bool f16 = p.dtype == MLORA_F16;
  if (p.tma_out) {
    if (lane == 0) bulk_wait_read_0();  // the store issued from this buffer one slice ago
    __syncwarp();
    const uint32_t rowb = buf + uint32_t(lane) * 64u, sw = uint32_t(lane >> 1) & 3u;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      sts128(rowb + ((uint32_t(q) ^ sw) << 4), pack2(f[8 * q], f[8 * q + 1], f16),
             pack2(f[8 * q + 2], f[8 * q + 3], f16), pack2(f[8 * q + 4], f[8 * q + 5], f16),
             pack2(f[8 * q + 6], f[8 * q + 7], f16));
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
      if (row_w0 < p.M) tma_store(&p.mY, buf, n, int(row_w0));
      bulk_commit();
    }
    return;
  }
  const int64_t row = row_w0 + lane;
  int64_t orow = row < p.M ? (p.out_rows ? int64_t(p.out_rows[row]) : row) : -1;
  if (row < p.M && (orow < 0 || orow >= p.M)) {  // out_rows is not a permutation
    flag_error(p.err, kErrBounds);
    orow = -1;
  }
  // Any other output goes through shared memory, so that a warp writes
  // neighbouring elements of a row, at any alignment: 64 bytes a row and pass,
  // one row of 32 16-bit values or two half rows of 16 float32 values at a time.
  if (p.dtype == MLORA_F32) {
    float* out = static_cast<float*>(p.out);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      __syncwarp();
#pragma unroll
      for (int q = 0; q < 4; ++q)
        sts128(buf + uint32_t(lane) * 64u + ((uint32_t(q) ^ (uint32_t(lane >> 1) & 3u)) << 4),
               __float_as_uint(f[16 * h + 4 * q]), __float_as_uint(f[16 * h + 4 * q + 1]),
               __float_as_uint(f[16 * h + 4 * q + 2]), __float_as_uint(f[16 * h + 4 * q + 3]));
      __syncwarp();
      const int c = lane & 15, col = n + 16 * h + c;
      float v[16];  // all reads first: their latency is paid once
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t r = 2u * uint32_t(i) + (uint32_t(lane) >> 4);
        const uint32_t a = buf + r * 64u + (((uint32_t(c) >> 2) ^ ((r >> 1) & 3u)) << 4) + (uint32_t(c) & 3u) * 4u;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[i]) : "r"(a));
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int64_t o = __shfl_sync(0xffffffffu, orow, 2 * i + (lane >> 4));
        if (o >= 0 && col < p.N) out[o * p.N + col] = v[i];
      }
    }
    return;
  }
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
  if (n + 32 <= p.N && (p.N & 7) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
    if (orow >= 0) store32(out + orow * p.N + n, f, f16);
    return;
  }
  __syncwarp();
  const uint32_t rowb = buf + uint32_t(lane) * 64u, sw = uint32_t(lane >> 1) & 3u;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    sts128(rowb + ((uint32_t(q) ^ sw) << 4), pack2(f[8 * q], f[8 * q + 1], f16),
           pack2(f[8 * q + 2], f[8 * q + 3], f16), pack2(f[8 * q + 4], f[8 * q + 5], f16),
           pack2(f[8 * q + 6], f[8 * q + 7], f16));
  __syncwarp();
  uint16_t v[32];
#pragma unroll
  for (int r = 0; r < 32; ++r) {
    const uint32_t a = buf + uint32_t(r) * 64u + (((uint32_t(lane) >> 3) ^ ((uint32_t(r) >> 1) & 3u)) << 4) +
                       (uint32_t(lane) & 7u) * 2u;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v[r]) : "r"(a));
  }
#pragma unroll
  for (int r = 0; r < 32; ++r) {
    const int64_t o = __shfl_sync(0xffffffffu, orow, r);
    if (o >= 0 && n + lane < p.N) reinterpret_cast<uint16_t*>(out)[o * p.N + n + lane] = v[r];
  }
}

template <bool BWD>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kQ8Threads, 1) k_q8(const __grid_constant__ Q8Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* stage_out = smem + kQ8Stages * kQ8StageBytes;
  float* cols = reinterpret_cast<float*>(stage_out + kQ8OutBytes);  // [8][scales 128, biases 128]
  uint64_t* full = reinterpret_cast<uint64_t*>(stage_out + kQ8OutBytes + kQ8ColBytes);
  uint64_t* empty = full + kQ8Stages;
  uint64_t* ifull = empty + kQ8Stages;  // [2] integer sums of the accumulator complete
  uint64_t* conv = ifull + 2;           // [2] rewritten as fp32 in both CTAs (used in the even CTA)
  uint64_t* xfull = conv + 2;           // [2] expand added
  uint64_t* tempty = xfull + 2;         // [2] drained in both CTAs (used in the even CTA)
  uint64_t* drain = tempty + 2;         // [1]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t crank = cluster_rank();
  const bool leader = crank == 0;
  const int pair = blockIdx.x / 2, n_pairs = gridDim.x / 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kQ8Stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&ifull[a], 1);
      mbar_init(&conv[a], 2 * kQ8EpiWarps);  // one arrival per epilogue warp of both CTAs
      mbar_init(&xfull[a], 1);
      mbar_init(&tempty[a], 2 * kQ8EpiWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_slot)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if ((warp == 0 || warp == 6) && lane == 0) {
    // ---------------------------------------------------------------- TMA producers (both CTAs)
    const uint32_t pid = warp == 0 ? 0u : 1u;
    uint32_t gk = 0;
    int stage = 0;
    uint32_t phase = 0;
    uint32_t issued = 0, issued_par = 0;
    bool ok = true;
    const uint64_t pol_keep = policy_evict_last(), pol_norm = policy_evict_normal();
    // the ring slot of the next k-block, when it is this warp's
    auto claim = [&](uint32_t bytes) -> int {
      const int s = (gk++ % 2u) == pid ? stage : -1;
      if (s >= 0) {
        if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, p.err)) {
          ok = false;
          return -1;
        }
        if (leader) mbar_expect_tx(&full[stage], bytes);
        issued |= 1u << stage;
        issued_par = (issued_par & ~(1u << stage)) | (phase << stage);
      }
      if (++stage == kQ8Stages) { stage = 0; phase ^= 1; }
      return s;
    };
    bool rows_ready = !p.pdl_rows, z_ready = !p.pdl_z;
    const uint32_t main_bytes = p.a_rows ? uint32_t(p.a_rows) * kQ8K + kQ8StageBytes : 2 * kQ8StageBytes;
    auto expand = [&](const Q8Item& it) {
      if (it.nc > 0 && !z_ready) {
        grid_dep_wait();
        z_ready = true;
      }
      for (int i = 0; i < it.nc && ok; ++i) {
        const int s = claim(2 * kQ8StageBytes);
        if (s < 0) continue;
        uint8_t* sA = smem + s * kQ8StageBytes;
        uint8_t* sB = sA + kA2Bytes;
        const uint32_t bar = mapa(su32(&full[s]), 0);
        const int c = it.c0 + i, pcol = p.plan.chunks[c].pcol, nh = it.nb * 256 + int(crank) * 128;
        tma_load_pair(sA, &p.mZ, bar, 0, c * kTileRows + int(crank) * kHalfRows, pol_norm);
        if (!BWD) {
          tma_load_pair(sB, &p.mP, bar, pcol, nh, pol_keep);
        } else {
          for (int h = 0; h < 2; ++h) tma_load_pair(sB + h * kBox64, &p.mP, bar, nh + 64 * h, pcol, pol_keep);
        }
      }
    };
    Q8Item last;
    last.nc = 0;
    for (int item = pair; item < p.n_items && ok; item += n_pairs) {
      const Q8Item it = q8_item(p, item);
      const int row0 = it.t * kTileRows + int(crank) * kHalfRows;
      const int nh = it.nb * 256 + int(crank) * 128;
      const int defer = min(kDefer, p.nk);
      for (int kb = 0; kb < p.nk && ok; ++kb) {
        if (kb == defer) expand(last);
        if (!ok) break;
        const int s = claim(main_bytes);
        if (s < 0) continue;
        uint8_t* sA = smem + s * kQ8StageBytes;
        uint8_t* sB = sA + kA2Bytes;
        const uint32_t bar = mapa(su32(&full[s]), 0);
        if (!BWD) tma_load_pair(sB, &p.mB, bar, kb * kQ8K, nh, pol_keep);
        else tma_load_pair(sB, &p.mB, bar, nh, kb * kQ8K, pol_keep);
        if (!rows_ready) {
          grid_dep_wait();
          rows_ready = true;
        }
        if (p.a_rows == 0 || leader) tma_load_pair(sA, &p.mA, bar, kb * kQ8K, row0, pol_norm);
      }
      if (ok && defer == p.nk) expand(last);
      last = it;
    }
    if (ok) expand(last);
    if (!rows_ready || !z_ready) grid_dep_wait();  // never finish before the kernel this launch overlaps
    if (!ok && leader) {
      // let copies already in flight land before the CTAs exit
      const unsigned long long t0 = now_ns();
      for (int s = 0; s < kQ8Stages; ++s) {
        if (!((issued >> s) & 1u)) continue;
        while (!mbar_try(su32(&full[s]), (issued_par >> s) & 1u)) {
          if (now_ns() - t0 > kTimeoutNs) break;
        }
      }
    }
  } else if (warp == 1 && lane == 0 && leader) {
    // ---------------------------------------------------------------- MMA issuer (even CTA)
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint32_t id_i8 = idesc_i8(256, 256, BWD), id_16 = idesc_16(256, 256, false, BWD, p.dtype == MLORA_F16);
    const uint32_t i8_step = BWD ? (32 * 128) >> 4 : 32 >> 4;   // 32 rows, or 32 bytes, of K
    const uint32_t x_step = BWD ? (16 * 128) >> 4 : 32 >> 4;    // 16 rows, or 16 columns, of K
    const uint32_t x_lbo = BWD ? uint32_t(kBox64) : 16u;
    int acc = 0;
    uint32_t acc_phase = 0;
    uint32_t conv_phase[2] = {0, 0};
    int last_nc = 0;
    // next filled stage -> its A address
    auto take = [&](uint32_t& sA) {
      if (!mbar_wait(&full[stage], phase, abort_flag, p.err)) return ok = false;
      tc_fence_after();
      sA = su32(smem + stage * kQ8StageBytes);
      return true;
    };
    auto release = [&]() {
      tc_commit_pair_both(&empty[stage]);
      if (++stage == kQ8Stages) { stage = 0; phase ^= 1; }
    };
    // expand of the previous item, on accumulator b
    auto expand = [&](int b) {
      if (last_nc == 0) return;
      if (!mbar_wait_cluster(&conv[b], conv_phase[b], abort_flag, p.err)) { ok = false; return; }
      conv_phase[b] ^= 1;
      tc_fence_after();
      const uint32_t d = tmem + uint32_t(b * kAccCols);
      for (int i = 0; i < last_nc; ++i) {
        uint32_t sA;
        if (!take(sA)) return;
        const uint64_t ad = sdesc(sA, 16u, 1024), bd = sdesc(sA + kA2Bytes, x_lbo, 1024);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc_mma_pair(d, ad + uint64_t(k * 2), bd + uint64_t(k * x_step), id_16, 1);
        release();
      }
      tc_commit_pair_both(&xfull[b]);
    };
    for (int item = pair; item < p.n_items && ok; item += n_pairs) {
      const Q8Item it = q8_item(p, item);
      if (!mbar_wait_cluster(&tempty[acc], acc_phase ^ 1, abort_flag, p.err)) { ok = false; break; }
      tc_fence_after();
      const uint32_t d = tmem + uint32_t(acc * kAccCols);
      const int defer = min(kDefer, p.nk);
      for (int kb = 0; kb < p.nk && ok; ++kb) {
        if (kb == defer) expand(acc ^ 1);
        uint32_t sA;
        if (!ok || !take(sA)) break;
        const uint64_t ad = sdesc(sA, 16u, 1024), bd = sdesc(sA + kA2Bytes, 16u, 1024);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tc_mma_i8_pair(d, ad + uint64_t(k * 2), bd + uint64_t(k * i8_step), id_i8, (kb | k) != 0);
        release();
      }
      if (ok && defer == p.nk) expand(acc ^ 1);
      if (!ok) break;
      tc_commit_pair_both(&ifull[acc]);
      last_nc = it.nc;
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if (ok) expand(acc ^ 1);
    tc_commit_pair_local(drain);
    const unsigned long long t0 = now_ns();
    while (!mbar_try(su32(drain), 0)) {
      if (now_ns() - t0 > kTimeoutNs) { flag_error(p.err, kErrTimeout); break; }
    }
  } else if ((warp >= 2 && warp < 6) || warp >= 8) {
    // ---------------------------------------------------------------- epilogue (both CTAs)
    const int quad = warp % 4;
    const uint32_t tempty0 = mapa(su32(&tempty[0]), 0), conv0 = mapa(su32(&conv[0]), 0);
    const int ew = warp < 6 ? warp - 2 : warp - 4;        // 0..7
    const int first = ew < 4 ? 0 : kQ8EpiCols, end = first + kQ8EpiCols;  // this warp's columns of a tile
    const uint32_t obuf = su32(stage_out) + uint32_t(ew) * 2048u;
    float* cs = cols + ew * 2 * kQ8EpiCols;
    const uint32_t cs32 = su32(cs) - uint32_t(first) * 4u;
    int acc = 0;
    uint32_t acc_phase = 0;
    uint32_t x_phase[2] = {0, 0};
    if (p.pdl_rows) grid_dep_wait();  // the row scales are that kernel's
    for (int item = pair; item < p.n_items; item += n_pairs) {
      const Q8Item it = q8_item(p, item);
      // the tile's column scales and biases, fetched while its sums are formed
      // (a copy per warp: no warp waits for another)
      if (!BWD) {
        __syncwarp();
#pragma unroll
        for (int c = lane; c < kQ8EpiCols; c += 32) {
          const int n = it.nb * 256 + first + c;
          cs[c] = n < p.N ? __ldg(p.w_scale + n) : 0.f;
          cs[kQ8EpiCols + c] = n < p.N && p.bias ? q8_bias(p, n) : 0.f;
        }
        __syncwarp();
      }
      const int64_t row_w0 = int64_t(it.t) * kTileRows + int(crank) * kHalfRows + quad * 32;
      const int n0 = it.nb * 256;
      const float sa = row_w0 + lane < p.M ? __ldg(p.a_scale + row_w0 + lane) : 0.f;
      const uint32_t tbase = tmem + (uint32_t(quad * 32) << 16) + uint32_t(acc * kAccCols);
      if (!warp_wait(&ifull[acc], acc_phase, abort_flag, p.err)) break;
      tc_fence_after();
      auto scaled = [&](int col, float (&f)[32]) {
        uint32_t v[32];
        tc_ld32(tbase + col, v);
#pragma unroll
        for (int q = 0; q < 32; ++q) f[q] = __int2float_rn(int(v[q])) * sa;
        if (!BWD) {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const float4 s = lds_f4(cs32 + uint32_t(col + 4 * q) * 4u);
            f[4 * q] *= s.x; f[4 * q + 1] *= s.y; f[4 * q + 2] *= s.z; f[4 * q + 3] *= s.w;
          }
        }
      };
      const bool expanded = it.nc > 0;
      if (expanded) {
        for (int col = first; col < end && n0 + col < p.N; col += 32) {
          float f[32];
          scaled(col, f);
          tc_st32(tbase + col, f);
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(conv0 + 8u * uint32_t(acc));
        if (!warp_wait(&xfull[acc], x_phase[acc], abort_flag, p.err)) break;
        x_phase[acc] ^= 1;
        tc_fence_after();
      }
      for (int col = first; col < end && n0 + col < p.N; col += 32) {
        float f[32];
        if (expanded) {
          uint32_t v[32];
          tc_ld32(tbase + col, v);
#pragma unroll
          for (int q = 0; q < 32; ++q) f[q] = __uint_as_float(v[q]);
        } else {
          scaled(col, f);
        }
        if (!BWD && p.bias) {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const float4 s = lds_f4(cs32 + uint32_t(kQ8EpiCols + col + 4 * q) * 4u);
            f[4 * q] += s.x; f[4 * q + 1] += s.y; f[4 * q + 2] += s.z; f[4 * q + 3] += s.w;
          }
        }
        q8_store_slice(p, f, row_w0, n0 + col, obuf, lane);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty0 + 8u * uint32_t(acc));
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if (lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

// 2-D map over an 8-bit matrix [rows, cols] with rows ld bytes apart; boxes of
// box_rows x 128 bytes, 128-byte swizzle.  The extent is q8_ld(cols): its last
// bytes are zero.
bool make_map8(CUtensorMap* m, const int8_t* base, int64_t rows, int64_t ld, int box_rows = 128) {
  EncodeFn enc = get_encode();
  if (!enc || rows < 1 || ld < 16 || ld % 16 || reinterpret_cast<uintptr_t>(base) % 16) return false;
  cuuint64_t dims[2] = {cuuint64_t(ld), cuuint64_t(rows)};
  cuuint64_t strides[1] = {cuuint64_t(ld)};
  cuuint32_t box[2] = {128u, cuuint32_t(box_rows)}, estr[2] = {1u, 1u};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

// Any sizes, alignments and types, except that the expand reads 16-bit
// operands by TMA (a LoRA call of the tensor-core family), and that a tile
// takes two CTAs.
bool q8_tc_ok(const Q8Main& a) {
  if (a.expand && (a.dtype == MLORA_F32 || (a.bwd && a.d_in % 8) || !aligned(a.pack, 16) || !aligned(a.zt, 16)))
    return false;
  return tc_available() && cta_budget(a.max_ctas) >= 2;
}

int q8_main_tc(const Q8Main& a, Q8After after, cudaStream_t st) {
  Q8Params prm;
  memset(&prm, 0, sizeof(prm));
  const int K = a.bwd ? a.d_out : a.d_in, N = a.bwd ? a.d_in : a.d_out;
  // up to 128 rows: a box of just these (17 rows of 4096 -> 11008 took 41 us with
  // 128-row boxes, whose reads past a tensor of fewer than 32 rows are slow)
  prm.a_rows = a.M <= 128 ? int(a.M) : 0;
  if (!make_map8(&prm.mA, a.Aq, a.M, q8_ld(K), prm.a_rows ? prm.a_rows : 128) || !make_map8(&prm.mB, a.Wq, a.d_out, q8_ld(a.d_in)))
    return MLORA_ERR_UNSUPPORTED;
  if (a.expand) {
    const int64_t zrows = int64_t(a.plan.n_chunks) * kTileRows;
    if (!make_map(&prm.mZ, a.zt, zrows, 64, 128) ||
        !(a.bwd ? make_map(&prm.mP, a.pack, a.R, a.d_in, 64) : make_map(&prm.mP, a.pack, a.d_out, a.R, 128)))
      return MLORA_ERR_UNSUPPORTED;
    prm.expand = 1;
    prm.plan = a.plan;
  }
  prm.M = a.M;
  prm.N = N;
  prm.dtype = a.dtype;
  prm.tma_out = a.dtype != MLORA_F32 && !a.out_rows && N % 8 == 0 && aligned(a.out, 16);
  if (prm.tma_out && !make_out_map(&prm.mY, a.out, a.M, N)) return MLORA_ERR_UNSUPPORTED;
  prm.n_tiles = mlora_num_tiles(a.M);
  prm.n_nblk = (N + 255) / 256;
  // as for the 16-bit mainloops: about 48 MB of weight blocks stay in L2
  const double block = 256.0 * K;
  prm.group = std::max(1, std::min(std::max(4, std::min(16, int(48.0 * (1 << 20) / block + 0.5))), prm.n_nblk));
  prm.n_items = prm.n_tiles * prm.n_nblk;
  prm.nk = (K + kQ8K - 1) / kQ8K;
  prm.a_scale = a.a_scale;
  prm.w_scale = a.w_scale;
  prm.bias = a.bias;
  prm.out = a.out;
  prm.out_rows = a.out_rows;
  prm.err = a.err;
  const void* fn = a.bwd ? reinterpret_cast<const void*>(&k_q8<true>) : reinterpret_cast<const void*>(&k_q8<false>);
  MLORA_CUDA_TRY(set_smem_once(fn, kQ8Smem));
  const unsigned grid = 2u * unsigned(std::min(prm.n_items, cta_budget(a.max_ctas) / 2));
  const bool pdl = after != kAfterOther && pdl_enabled();
  prm.pdl_rows = pdl && after == kAfterRows ? 1 : 0;
  prm.pdl_z = pdl ? 1 : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kQ8Threads);
  cfg.dynamicSmemBytes = kQ8Smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  MLORA_CUDA_TRY(cudaLaunchKernelEx(&cfg, a.bwd ? &k_q8<true> : &k_q8<false>, prm));
  count_launch();
  return cudaGetLastError() == cudaSuccess ? MLORA_OK : MLORA_ERR_CUDA;
}

}  // namespace mlora

// ------------------------------------------------------------------ dA from saved 8-bit inputs
//   dA chunk [64 ranks, 256 columns] = sum_i w[i, :]^T Xq[i, :],   w = x_scale dZ
//
// k_q8_da reads every saved byte once per rank chunk and is meant to be bound
// by that.  The scales went into w (fp32, then two bf16 numbers: 16 bits), so
// the integers enter the product as they are: eight warps turn each 64 x 256
// block of bytes into bf16 (exact up to 256) in the layout of an MN-major
// operand, and one M = 128, N = 256 MMA per 16 rows multiplies the stacked
// high and low parts of w (ranks 0..63 twice) with it.  The high and the low
// sums are added in the epilogue.
//
// Per 64 rows of a block the shared memory moves 32 KB in by TMA, 48 KB
// through the conversion and 48 KB into the MMAs, about 1000 cycles, against
// 700 cycles of the SM's share of HBM for the 16 KB of new bytes.  Measured:
// 65,536 x 4096, 8 jobs 111 us (the saved bytes: 41; loads alone 61, without
// the conversion 80), 18,432 rows of 16 jobs 35 us (12).
//
// Long sums are split over several items (SavedItem): each stores its fp32
// block, and the last to finish adds the blocks in their order, so the result
// does not depend on which one that is.
namespace mlora {
namespace {

constexpr int kDaStages = 4, kDaStageBytes = 32 * 1024;  // 64 x 256 bytes of X, 2 x 64 x 64 of w
constexpr int kDaConv = 2, kDaConvBytes = 32 * 1024;     // 64 x 256 bf16
constexpr int kDaConvWarps = 8, kDaProducers = 2;
constexpr int kDaConvGroup = kDaConvWarps / kDaConv;     // warps that convert one k-block
constexpr int kDaThreads = 32 * (4 + kDaConvWarps + 1 + kDaProducers);
constexpr int kDaSumBytes = 4 * 32 * 32 * 4;             // sums that the epilogue warps hand over
constexpr int kDaSmem = kDaStages * kDaStageBytes + kDaConv * kDaConvBytes + kDaSumBytes + 1024 + 512;
static_assert(kDaSmem <= 232448, "dynamic shared memory above 227 KB");

struct DaParams {
  CUtensorMap mX;  // saved rows, 128-byte x 64-row boxes
  CUtensorMap mW;  // [2 n_chunks 256, 64] high parts, then low parts
  PlanDev plan;
  int d_in, f16, zrows;
  float* parts;  // stored parts, [.][64][256]
  __nv_bfloat16* dA;
  __nv_bfloat16* A_upd;
  float lr;
};

// Item `i`; false (and flagged) if the plan is corrupted.
__device__ __forceinline__ bool da_item(const DaParams& p, int i, SavedItem& it) {
  it = p.plan.saved[i];
  const bool ok = it.lb >= 0 && it.le <= p.plan.n_list && it.e0 >= it.lb && it.e0 < it.le && it.j >= 0 &&
                  it.block >= 0 && it.nks > 0 && it.nks <= 4 * (it.le - it.lb) && it.part >= 0 &&
                  it.part < it.nparts;
  if (!ok) flag_error(p.plan.err, kErrBounds);
  return ok;
}

// Item of this block's round k, or -1: the items are sorted by length, and every
// other round deals them out backwards, so that a block with a long item of
// one round has a short one in the next.
__device__ __forceinline__ int da_deal(int k, int n_items) {
  const int i = k * int(gridDim.x) + int((k & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
  return i < n_items ? i : -1;
}

// {chunk, tile, first slice, end slice} of list entry e (clamped and flagged
// if the plan is corrupted)
__device__ __forceinline__ int4 da_entry(const DaParams& p, int e) {
  int4 d = p.plan.list_desc[e];
  if (d.x < 0 || d.x >= p.plan.n_chunks || d.y < 0 || d.y >= p.plan.n_tiles || d.z < 0 || d.w > kTileRows ||
      d.z >= d.w) {
    flag_error(p.plan.err, kErrBounds);
    d = make_int4(0, 0, 0, 1);
  }
  return make_int4(d.x, d.y, first_slice(d), end_slice(d));
}

// two bytes of `w` (selected into the low bytes of the halves) as bf16: a
// byte with bits s vvvvvvv stands for vvvvvvv - 128 s, and (128 + vvvvvvv) -
// (128 + 128 s) is exact
__device__ __forceinline__ uint32_t bytes_to_bf16x2(uint32_t w, uint32_t sel) {
  const uint32_t b = __byte_perm(w, 0, sel);
  const uint32_t m = (b & 0x007f007fu) | 0x43004300u, c = (b & 0x00800080u) | 0x43004300u;
  const __nv_bfloat162 r =
      __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&m), *reinterpret_cast<const __nv_bfloat162*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ void pair_barrier(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

__global__ void __launch_bounds__(kDaThreads, 1) k_q8_da(const __grid_constant__ DaParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* conv = smem + kDaStages * kDaStageBytes;
  float* sums = reinterpret_cast<float*>(conv + kDaConv * kDaConvBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(sums) + kDaSumBytes);
  uint64_t* empty = full + kDaStages;   // the converting warps and the MMAs
  uint64_t* cfull = empty + kDaStages;  // [kDaConv] converted
  uint64_t* cempty = cfull + kDaConv;   // [kDaConv] read by the MMAs
  uint64_t* tfull = cempty + kDaConv;   // [2]
  uint64_t* tempty = tfull + 2;         // [2]
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* going = abort_flag + 1;  // [4] per epilogue warp

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  constexpr int kMma = 4 + kDaConvWarps;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kDaStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kDaConvGroup + 1);
    }
    for (int s = 0; s < kDaConv; ++s) {
      mbar_init(&cfull[s], kDaConvGroup);
      mbar_init(&cempty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 4);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == kMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_slot)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int n_items = p.plan.n_saved;

  if (warp > kMma && lane == 0) {
    // ---------------------------------------------------------------- TMA producers (alternate k-blocks)
    const uint32_t pid = uint32_t(warp - kMma - 1);
    uint32_t gk = 0, phase = 0, issued = 0, issued_par = 0;
    int stage = 0;
    bool ok = true;
    const uint64_t pol_stream = policy_evict_first(), pol_norm = policy_evict_normal();
    for (int round = 0; round * int(gridDim.x) < n_items && ok; ++round) {
      const int item = da_deal(round, n_items);
      if (item < 0) break;
      SavedItem it;
      if (!da_item(p, item, it)) continue;
      int e = it.e0, q = it.q0;
      int4 d = da_entry(p, e);
      for (int kb = 0; kb < it.nks; ++kb) {
        if ((gk++ % kDaProducers) == pid) {
          if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, p.plan.err)) { ok = false; break; }
          uint8_t* sX = smem + stage * kDaStageBytes;
          uint8_t* sW = sX + 16 * 1024;
          mbar_expect_tx(&full[stage], kDaStageBytes);
          for (int h = 0; h < 2; ++h)
            tma_load(sX + h * 8192, &p.mX, &full[stage], it.block * kSavedCols + 128 * h, d.y * kTileRows + 64 * q,
                     pol_stream);
          const int wrow = (d.x + it.j) * kTileRows + 64 * q;
          for (int h = 0; h < 2; ++h)
            tma_load(sW + h * kBox64, &p.mW, &full[stage], 0, wrow + h * p.zrows, pol_norm);
          issued |= 1u << stage;
          issued_par = (issued_par & ~(1u << stage)) | (phase << stage);
        }
        if (++stage == kDaStages) { stage = 0; phase ^= 1; }
        if (++q >= d.w && ++e < it.le) {
          d = da_entry(p, e);
          q = d.z;
        }
      }
    }
    if (!ok) {
      const unsigned long long t0 = now_ns();
      for (int s = 0; s < kDaStages; ++s) {
        if (!((issued >> s) & 1u)) continue;
        while (!mbar_try(su32(&full[s]), (issued_par >> s) & 1u)) {
          if (now_ns() - t0 > kTimeoutNs) break;
        }
      }
    }
  } else if (warp == kMma && lane == 0) {
    // ---------------------------------------------------------------- MMA issuer
    int stage = 0, cs = 0, acc = 0;
    uint32_t phase = 0, cphase = 0, acc_phase = 0;
    bool ok = true;
    const uint32_t idesc = idesc_16(128, 256, true, true, false);  // bf16 for either type of the layer
    for (int round = 0; round * int(gridDim.x) < n_items && ok; ++round) {
      const int item = da_deal(round, n_items);
      if (item < 0) break;
      SavedItem it;
      if (!da_item(p, item, it)) continue;
      if (!mbar_wait(&tempty[acc], acc_phase ^ 1, abort_flag, p.plan.err)) { ok = false; break; }
      tc_fence_after();
      const uint32_t d = tmem + uint32_t(acc * kAccCols);
      for (int kb = 0; kb < it.nks; ++kb) {
        if (!mbar_wait(&full[stage], phase, abort_flag, p.plan.err) ||
            !mbar_wait(&cfull[cs], cphase, abort_flag, p.plan.err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t ad = sdesc(su32(smem + stage * kDaStageBytes) + 16u * 1024u, uint32_t(kBox64), 1024);
        const uint64_t bd = sdesc(su32(conv + cs * kDaConvBytes), uint32_t(kBox64), 1024);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tc_mma(d, ad + uint64_t(k * 128), bd + uint64_t(k * 128), idesc, (kb | k) != 0);
        tc_commit(&empty[stage]);
        tc_commit(&cempty[cs]);
        if (++stage == kDaStages) { stage = 0; phase ^= 1; }
        if (++cs == kDaConv) { cs = 0; cphase ^= 1; }
      }
      if (!ok) break;
      tc_commit(&tfull[acc]);
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    tc_commit(drain);
    const unsigned long long t0 = now_ns();
    while (!mbar_try(su32(drain), 0)) {
      if (now_ns() - t0 > kTimeoutNs) { flag_error(p.plan.err, kErrTimeout); break; }
    }
  } else if (warp >= 4 && warp < kMma) {
    // ---------------------------------------------------------------- conversion
    // Two groups of four warps convert alternate k-blocks, each into its own
    // buffer, so that one group's waits and stores overlap the other's.
    // A thread turns a 16-byte piece (columns 16 cl .. of a 64-column box, one
    // row) into two 16-byte groups of bf16.  A quarter warp covers the four
    // pieces of a box in rows r and r ^ 5: with the 128-byte swizzle its loads
    // (bit 2 of the row differs) and its stores (bit 0) both touch all banks.
    const int cs = (warp - 4) / kDaConvGroup;
    const int t = ((warp - 4) % kDaConvGroup) * 32 + lane;  // 0..127
    const uint32_t dst = su32(conv + cs * kDaConvBytes);
    const uint32_t cl = uint32_t(t & 3), flip = (t & 4) ? 5u : 0u, r0 = 2u * uint32_t(t >> 3);
    int stage = 0, turn = 0;
    uint32_t phase = 0, cphase = 0;
    bool ok = true;
    for (int round = 0; round * int(gridDim.x) < n_items && ok; ++round) {
      const int item = da_deal(round, n_items);
      if (item < 0) break;
      SavedItem it;
      if (!da_item(p, item, it)) continue;
      for (int kb = 0; kb < it.nks; ++kb) {
        if (turn == cs) {
          if (!warp_wait(&full[stage], phase, abort_flag, p.plan.err) ||
              !warp_wait(&cempty[cs], cphase ^ 1, abort_flag, p.plan.err)) {
            ok = false;
            break;
          }
          const uint32_t src = su32(smem + stage * kDaStageBytes);
          // rows (r0 + 32 i) ^ flip, the four boxes of each
          uint4 v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t k = (r0 + 32u * (uint32_t(i) >> 2)) ^ flip, box = uint32_t(i) & 3u;
            v[i] = lds128(src + (box >> 1) * 8192u + k * 128u + ((((box & 1u) * 4u + cl) ^ (k & 7u)) << 4));
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t k = (r0 + 32u * (uint32_t(i) >> 2)) ^ flip, box = uint32_t(i) & 3u;
            const uint32_t row = dst + box * uint32_t(kBox64) + k * 128u, g = (2u * cl) ^ (k & 7u);
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
            uint32_t o[8];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              o[2 * q] = bytes_to_bf16x2(w[q], 0x4140);
              o[2 * q + 1] = bytes_to_bf16x2(w[q], 0x4342);
            }
            sts128(row + (g << 4), o[0], o[1], o[2], o[3]);
            sts128(row + ((g ^ 1u) << 4), o[4], o[5], o[6], o[7]);
          }
          fence_async_smem();  // the MMAs read what was written here
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&cfull[cs]);
            mbar_arrive(&empty[stage]);
          }
          cphase ^= 1;
        }
        turn = turn + 1 == kDaConv ? 0 : turn + 1;
        if (++stage == kDaStages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp < 4) {
    // ---------------------------------------------------------------- epilogue
    // Lanes 0..63 of the accumulator hold the high sums of ranks 0..63 (warps
    // 0 and 1), lanes 64..127 the low sums (warps 2 and 3).  Warps i and i + 2
    // trade 32-column slices through shared memory: of every two, the one
    // finishes the even and the other the odd slice.
    const int half = warp & 1;  // ranks 32 half ..
    const bool low = warp >= 2;
    const uint32_t give = su32(sums) + uint32_t(warp) * 4096u, take = su32(sums) + uint32_t(warp ^ 2) * 4096u;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int round = 0; round * int(gridDim.x) < n_items; ++round) {
      const int item = da_deal(round, n_items);
      if (item < 0) break;
      SavedItem it;
      if (!da_item(p, item, it)) continue;
      // both warps of a pair must agree to go on before they meet at a barrier
      const bool ok = warp_wait(&tfull[acc], acc_phase, abort_flag, p.plan.err);
      if (lane == 0) going[warp] = ok ? 1 : 0;
      pair_barrier(1 + half);
      const bool both = going[half] != 0 && going[half + 2] != 0;
      pair_barrier(1 + half);
      if (!both) break;
      tc_fence_after();
      const uint32_t tbase = tmem + (uint32_t(warp * 32) << 16) + uint32_t(acc * kAccCols);
      const int c0 = it.block * kSavedCols;
      const int r = 32 * half + lane;  // rank row inside the chunk
      const bool live = r < it.rank - it.j * 64;
      const int64_t row0 = int64_t(p.plan.chunks[p.plan.list[it.lb] + it.j].pcol + r) * p.d_in + c0;
      auto finish = [&](int col, const float (&f)[32]) {
        // 32 columns of one rank row of dA: 64 contiguous bytes (d_in is a multiple of 8)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          if (!live || c0 + col + 8 * g >= p.d_in) break;
          uint32_t w[4];
#pragma unroll
          for (int h = 0; h < 4; ++h) w[h] = pack2(f[8 * g + 2 * h], f[8 * g + 2 * h + 1], p.f16 != 0);
          reinterpret_cast<uint4*>(p.dA + row0 + col)[g] = make_uint4(w[0], w[1], w[2], w[3]);
          if (p.A_upd) {  // fused SGD step, from the gradient as stored
            uint4* P = reinterpret_cast<uint4*>(p.A_upd + row0 + col) + g;
            const uint4 old = *P;
            uint32_t o[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const float2 g2 = unpack2(w[h], p.f16 != 0), o2 = unpack2(o[h], p.f16 != 0);
              o[h] = pack2(sgd_new(o2.x, g2.x, p.lr, p.f16 != 0), sgd_new(o2.y, g2.y, p.lr, p.f16 != 0), p.f16 != 0);
            }
            *P = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
      };
      // a part is [64 column groups][64 ranks][4 columns]: a warp's stores are contiguous
      auto part_of = [&](int k, int col) {
        return reinterpret_cast<float4*>(p.parts) + (int64_t(it.part0 + k) * 64 + col / 4) * 64 + r;
      };
      for (int col2 = 0; col2 < kSavedCols && c0 + col2 < p.d_in; col2 += 64) {
        const int col = col2 + (low ? 32 : 0);  // the slice this warp finishes
        uint32_t v[32];
        tc_ld32(tbase + (col ^ 32), v);
#pragma unroll
        for (int q = 0; q < 8; ++q)
          sts128(give + uint32_t(lane) * 128u + ((uint32_t(q) ^ (uint32_t(lane) & 7u)) << 4), v[4 * q], v[4 * q + 1],
                 v[4 * q + 2], v[4 * q + 3]);
        tc_ld32(tbase + col, v);
        pair_barrier(1 + half);
        float f[32];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const float4 o = lds_f4(take + uint32_t(lane) * 128u + ((uint32_t(q) ^ (uint32_t(lane) & 7u)) << 4));
          f[4 * q] = __uint_as_float(v[4 * q]) + o.x;
          f[4 * q + 1] = __uint_as_float(v[4 * q + 1]) + o.y;
          f[4 * q + 2] = __uint_as_float(v[4 * q + 2]) + o.z;
          f[4 * q + 3] = __uint_as_float(v[4 * q + 3]) + o.w;
        }
        pair_barrier(1 + half);
        if (it.nparts > 1) {
          float4* dst = part_of(it.part, col);
#pragma unroll
          for (int q = 0; q < 8; ++q)
            __stcg(dst + q * 64, make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]));
        } else if (c0 + col < p.d_in) {
          finish(col, f);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
      if (it.nparts > 1) {
        // this warp's slices of the part are stored: the warp that stores the
        // last part's adds them all up, in the parts' order
        int last = 0;
        __threadfence();
        __syncwarp();
        if (lane == 0) last = atomicAdd(p.plan.saved_done + 4 * it.group + warp, 1) == it.nparts - 1;
        last = __shfl_sync(0xffffffffu, last, 0);
        __threadfence();
        if (!last) continue;
        for (int col = low ? 32 : 0; col < kSavedCols && c0 + col < p.d_in; col += 64) {
          float f[32];
#pragma unroll
          for (int q = 0; q < 32; ++q) f[q] = 0.f;
#pragma unroll 2
          for (int k = 0; k < it.nparts; ++k) {
            const float4* src = part_of(k, col);
            float4 u[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) u[q] = __ldcg(src + q * 64);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              f[4 * q] += u[q].x; f[4 * q + 1] += u[q].y; f[4 * q + 2] += u[q].z; f[4 * q + 3] += u[q].w;
            }
          }
          finish(col, f);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

}  // namespace

int q8_da_tc(const Q8Saved& a, cudaStream_t st) {
  if (a.plan.n_saved == 0) return MLORA_OK;
  DaParams prm;
  memset(&prm, 0, sizeof(prm));
  const int64_t zrows = int64_t(a.plan.n_chunks) * kTileRows;
  if (2 * zrows > INT32_MAX) return MLORA_ERR_UNSUPPORTED;
  if (!make_map8(&prm.mX, a.Xq, a.M, q8_ld(a.d_in), 64) || !make_map(&prm.mW, a.scratch, 2 * zrows, 64, 64))
    return MLORA_ERR_UNSUPPORTED;
  prm.plan = a.plan;
  prm.d_in = a.d_in;
  prm.f16 = a.dtype == MLORA_F16 ? 1 : 0;
  prm.zrows = int(zrows);
  prm.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(a.scratch) + q8_dz8_bytes(a.plan.n_chunks));
  prm.dA = static_cast<__nv_bfloat16*>(a.dA);
  prm.A_upd = static_cast<__nv_bfloat16*>(a.A_upd);
  prm.lr = a.lr;
  const int sms = cta_budget(a.max_ctas);
  if (sms <= 0) return MLORA_ERR_CUDA;
  MLORA_CUDA_TRY(set_smem_once(reinterpret_cast<const void*>(&k_q8_da), kDaSmem));
  k_q8_da<<<std::min(a.plan.n_saved, sms), kDaThreads, kDaSmem, st>>>(prm);
  count_launch();
  return cudaGetLastError() == cudaSuccess ? MLORA_OK : MLORA_ERR_CUDA;
}

}  // namespace mlora
