// C-ABI entry points (include/mlora.h): argument checks, plan upload and
// dispatch between the tcgen05 tensor-core family and the SIMT family.
#include <algorithm>
#include <cstring>
#include <initializer_list>
#include <memory>
#include <new>

#include "common.cuh"
#include "q8.cuh"
#include "simt.cuh"
#include "tc.cuh"

namespace mlora {

namespace {

size_t zt_bytes(const Plan& p, int dtype) {
  return size_t(p.chunks.size()) * kTileRows * kChunk * elem_bytes(dtype);
}

// Plan of a routing description.  A step calls with the same description
// several times, and so do the steps of a fixed job mix: the last few plans of
// the thread are kept and found again by their description's content.  The
// reference stays valid until the thread's next call.
const Plan* plan_of(const mlora_problem* prob, const mlora_routing* route, int* status) {
  struct Kept {
    int64_t rows;
    int32_t d_in, d_out, r_pack;
    std::vector<int32_t> seg_start, seg_adapter, rank, pack_off;
    std::vector<float> scaling;
    Plan plan;
  };
  constexpr size_t kKept = 8;
  thread_local std::vector<std::unique_ptr<Kept>> kept;  // most recently used first
  *status = validate(prob, route);
  if (*status != MLORA_OK) return nullptr;
  auto same = [](const auto& v, const auto* a, size_t n) {
    return v.size() == n && (n == 0 || std::memcmp(v.data(), a, n * sizeof(*a)) == 0);
  };
  const size_t ns = size_t(route->n_seg), na = size_t(route->n_adapters), nb = ns ? ns + 1 : 0;
  for (size_t i = 0; i < kept.size(); ++i) {
    const Kept& k = *kept[i];
    if (k.rows == prob->rows && k.d_in == prob->d_in && k.d_out == prob->d_out && k.r_pack == route->r_pack &&
        same(k.seg_start, route->seg_start, nb) && same(k.seg_adapter, route->seg_adapter, ns) &&
        same(k.rank, route->rank, na) && same(k.pack_off, route->pack_off, na) &&
        same(k.scaling, route->scaling, na)) {
      std::rotate(kept.begin(), kept.begin() + i, kept.begin() + i + 1);
      return &kept[0]->plan;
    }
  }
  // no exception may leave a C entry point: without host memory for the plan
  // the call is refused
  try {
    auto k = std::make_unique<Kept>();
    *status = build_plan(prob, route, &k->plan);
    if (*status != MLORA_OK) return nullptr;
    k->rows = prob->rows; k->d_in = prob->d_in; k->d_out = prob->d_out; k->r_pack = route->r_pack;
    k->seg_start.assign(route->seg_start, route->seg_start + nb);
    k->seg_adapter.assign(route->seg_adapter, route->seg_adapter + ns);
    k->rank.assign(route->rank, route->rank + na);
    k->pack_off.assign(route->pack_off, route->pack_off + na);
    k->scaling.assign(route->scaling, route->scaling + na);
    kept.insert(kept.begin(), std::move(k));
    if (kept.size() > kKept) kept.pop_back();
    return &kept[0]->plan;
  } catch (const std::bad_alloc&) {
    *status = MLORA_ERR_WORKSPACE;
    return nullptr;
  }
}

// layout of the caller's workspace: [plan tables | dZt scratch]
size_t ws_bytes(const Plan& p, int dtype) { return align_up(p.bytes, 1024) + zt_bytes(p, dtype); }

// Copy the plan tables into the workspace (one async H2D from pageable memory,
// staged before return) and return the device view.
int upload_plan(const Plan& p, void* ws, cudaStream_t st, PlanDev* dev) {
  thread_local std::vector<uint8_t> host;
  try {
    host.assign(p.bytes, 0);
  } catch (const std::bad_alloc&) {
    return MLORA_ERR_WORKSPACE;
  }
  auto put = [&](size_t off, const void* src, size_t n) {
    if (n) std::memcpy(host.data() + off, src, n);
  };
  put(p.off_tcb, p.tile_chunk_begin.data(), sizeof(int32_t) * p.tile_chunk_begin.size());
  put(p.off_chunks, p.chunks.data(), sizeof(Chunk) * p.chunks.size());
  put(p.off_shrink, p.shrink.data(), sizeof(ShrinkItem) * p.shrink.size());
  put(p.off_reduce, p.reduce.data(), sizeof(ReduceItem) * p.reduce.size());
  put(p.off_list, p.list.data(), sizeof(int32_t) * p.list.size());
  put(p.off_list_desc, p.list_desc.data(), sizeof(int4) * p.list_desc.size());
  put(p.off_saved, p.saved.data(), sizeof(SavedItem) * p.saved.size());
  MLORA_CUDA_TRY(cudaMemcpyAsync(ws, host.data(), p.bytes, cudaMemcpyHostToDevice, st));
  uint8_t* b = (uint8_t*)ws;
  std::memset(dev, 0, sizeof(*dev));
  dev->n_tiles = p.n_tiles;
  dev->n_chunks = int32_t(p.chunks.size());
  dev->n_shrink = int32_t(p.shrink.size());
  dev->n_reduce = int32_t(p.reduce.size());
  dev->n_list = int32_t(p.list.size());
  dev->tile_chunk_begin = (const int32_t*)(b + p.off_tcb);
  dev->chunks = (const Chunk*)(b + p.off_chunks);
  dev->shrink = (const ShrinkItem*)(b + p.off_shrink);
  dev->reduce = (const ReduceItem*)(b + p.off_reduce);
  dev->list = (const int32_t*)(b + p.off_list);
  dev->list_desc = (const int4*)(b + p.off_list_desc);
  dev->counters = (int32_t*)(b + p.off_counters);
  dev->n_saved = int32_t(p.saved.size());
  dev->saved = (const SavedItem*)(b + p.off_saved);
  dev->saved_done = dev->counters + 16;
  return MLORA_OK;
}

// Device view of a plan already in the workspace (MLORA_PLAN_RESIDENT): no
// copy; the per-launch work counters are reset on the stream, if the call has
// kernels that use them.
int view_plan(const Plan& p, void* ws, bool counters, cudaStream_t st, PlanDev* dev) {
  uint8_t* b = (uint8_t*)ws;
  std::memset(dev, 0, sizeof(*dev));
  dev->n_tiles = p.n_tiles;
  dev->n_chunks = int32_t(p.chunks.size());
  dev->n_shrink = int32_t(p.shrink.size());
  dev->n_reduce = int32_t(p.reduce.size());
  dev->n_list = int32_t(p.list.size());
  dev->tile_chunk_begin = (const int32_t*)(b + p.off_tcb);
  dev->chunks = (const Chunk*)(b + p.off_chunks);
  dev->shrink = (const ShrinkItem*)(b + p.off_shrink);
  dev->reduce = (const ReduceItem*)(b + p.off_reduce);
  dev->list = (const int32_t*)(b + p.off_list);
  dev->list_desc = (const int4*)(b + p.off_list_desc);
  dev->counters = (int32_t*)(b + p.off_counters);
  dev->n_saved = int32_t(p.saved.size());
  dev->saved = (const SavedItem*)(b + p.off_saved);
  dev->saved_done = dev->counters + 16;
  if (counters) MLORA_CUDA_TRY(cudaMemsetAsync(dev->counters, 0, p.bytes - p.off_counters, st));
  return MLORA_OK;
}

// Plan of a call: uploaded now, or already resident in the workspace; the
// kernels report their device-side checks into the call's status word.
int stage_plan(const mlora_problem* prob, const Plan& p, void* ws, cudaStream_t st, PlanDev* dev,
               bool counters = true) {
  const int s =
      (prob->flags & MLORA_PLAN_RESIDENT) ? view_plan(p, ws, counters, st, dev) : upload_plan(p, ws, st, dev);
  dev->err = prob->err_word;
  return s;
}

// Every tensor pointer of a call meets the alignment of the kernel family:
// 16 bytes for the tensor-core kernels (TMA boxes, 16-byte vector loads of
// the bias and stores of dB / the intermediates), the element size for the
// CUDA-core kernels.
bool pointers_aligned(std::initializer_list<const void*> ptrs, size_t a) {
  for (const void* q : ptrs)
    if (!aligned(q, a)) return false;
  return true;
}

bool tc_shape_ok(const mlora_problem* prob) {
  // TMA: global strides must be multiples of 16 bytes (bf16: 8 elements)
  return (prob->dtype == MLORA_BF16 || prob->dtype == MLORA_F16) && prob->d_in % 8 == 0 && prob->d_out % 8 == 0;
}

// Kernel family of a call whose tensor pointers are `ptrs`; -1 = unsupported
// (an explicit tensor-core request with a shape or pointer the tensor-core
// kernels cannot take, or pointers not aligned to their element size).
int choose_impl(const mlora_problem* prob, std::initializer_list<const void*> ptrs) {
  if (!pointers_aligned(ptrs, size_t(elem_bytes(prob->dtype)))) return -1;
  const bool tc_ok = tc_shape_ok(prob) && pointers_aligned(ptrs, 16);
  if (prob->impl == MLORA_IMPL_SIMT) return MLORA_IMPL_SIMT;
  if (prob->impl == MLORA_IMPL_TC || prob->impl == MLORA_IMPL_TC_1SM || prob->impl == MLORA_IMPL_TC_2SM ||
      prob->impl == MLORA_IMPL_TC_WIDE)
    return tc_ok ? MLORA_IMPL_TC : -1;
  if (prob->impl != MLORA_IMPL_AUTO) return -1;
  return (tc_ok && tc_available()) ? MLORA_IMPL_TC : MLORA_IMPL_SIMT;
}

// Checks of the 8-bit operands of a call (alignment: rows of an 8-bit matrix
// start on 16-byte boundaries, which its leading dimension keeps).
int check_q8(std::initializer_list<const void*> mats, std::initializer_list<const void*> scales) {
  for (const void* q : mats)
    if (!aligned(q, 16)) return MLORA_ERR_UNSUPPORTED;
  for (const void* s : scales)
    if (!aligned(s, 4)) return MLORA_ERR_UNSUPPORTED;
  return MLORA_OK;
}

// One 8-bit product: a few rows by streaming the weight, more on the tensor
// cores, whatever their size, unless the call asks for the CUDA cores.
int q8_main(const Q8Main& a, int impl, Q8After after, cudaStream_t st) {
  if (impl != MLORA_IMPL_SIMT && q8_few_ok(a)) return q8_main_few(a, after, st);
  if (impl != MLORA_IMPL_SIMT && a.expand && a.dtype == MLORA_F32) {
    // float32: the expand is not a tensor-core operand; it is added after
    Q8Main product = a;
    product.expand = false;
    if (q8_tc_ok(product)) {
      const int s = q8_main_tc(product, after, st);
      return s != MLORA_OK ? s : simt_expand_add32(a.bwd, a.plan, (const float*)a.pack, (const float*)a.zt,
                                                   (float*)a.out, a.out_rows, a.M, a.d_in, a.d_out, a.R, st);
    }
  }
  const bool tc = impl != MLORA_IMPL_SIMT && q8_tc_ok(a);
  return tc ? q8_main_tc(a, after, st) : q8_main_simt(a, st);
}

}  // namespace
}  // namespace mlora

using namespace mlora;

extern "C" int mlora_zsave_bytes(const mlora_problem* prob, const mlora_routing* route, size_t* bytes) {
  if (!bytes) return MLORA_ERR_INVALID_ARG;
  int st;
  const Plan* p = plan_of(prob, route, &st);
  if (!p) return st;
  *bytes = zt_bytes(*p, prob->dtype);
  return MLORA_OK;
}

extern "C" int mlora_workspace_bytes(const mlora_problem* prob, const mlora_routing* route, size_t* bytes) {
  if (!bytes) return MLORA_ERR_INVALID_ARG;
  int st;
  const Plan* p = plan_of(prob, route, &st);
  if (!p) return st;
  *bytes = ws_bytes(*p, prob->dtype);
  return MLORA_OK;
}

extern "C" int mlora_plan_upload(const mlora_problem* prob, const mlora_routing* route, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  int st;
  const Plan* plan = plan_of(prob, route, &st);
  if (!plan) return st;
  const Plan& p = *plan;
  if (!workspace) return MLORA_ERR_INVALID_ARG;
  if (!aligned(workspace, 16)) return MLORA_ERR_UNSUPPORTED;
  if (workspace_bytes < ws_bytes(p, prob->dtype)) return MLORA_ERR_WORKSPACE;
  PlanDev dev;
  return upload_plan(p, workspace, (cudaStream_t)stream, &dev);
}

extern "C" int32_t mlora_num_tiles(int64_t rows) {
  return rows <= 0 ? 0 : int32_t((rows + kTileRows - 1) / kTileRows);
}

namespace {

// Kernel family of the 8-bit product of a layer call whose other kernels run as
// `impl`: left open by MLORA_IMPL_AUTO, since the 8-bit operands are always
// aligned, whatever the 16-bit ones are.
int q8_impl(const mlora_problem* prob, int impl) {
  return prob->impl == MLORA_IMPL_AUTO ? MLORA_IMPL_AUTO : impl;
}

// The 8-bit backbone product of mlora_forward_q8, with the LoRA expand of the
// intermediate that the shrink before it left in zsave.
int q8_forward_main(const mlora_problem* prob, const mlora_routing* route, const mlora_q8* q8, const PlanDev& dev,
                    int impl, Q8After after, const void* bias, const void* B_pack, void* Y, const void* zsave,
                    cudaStream_t s) {
  Q8Main m;
  m.M = prob->rows; m.d_in = prob->d_in; m.d_out = prob->d_out; m.R = route->r_pack; m.dtype = prob->dtype;
  m.Aq = q8->Xq; m.a_scale = q8->x_scale;
  m.Wq = q8->Wq; m.w_scale = q8->w_scale;
  m.bias = bias; m.out = Y; m.out_rows = route->out_rows;
  m.expand = dev.n_chunks > 0;
  m.plan = dev; m.zt = zsave; m.pack = B_pack;
  m.max_ctas = prob->max_ctas;
  m.err = prob->err_word;
  return q8_main(m, impl, after, s);
}

// mlora_forward_staged, or with `ar` mlora_forward_push (MAIN pushes the
// partial tiles to their owner ranks instead of writing Y), or with `q8`
// mlora_forward_q8 over all tiles.
int forward_staged(const mlora_problem* prob, const mlora_routing* route, const void* X, const void* W,
                   const void* bias, const void* A_pack, const void* B_pack, void* Y, void* zsave,
                   void* workspace, size_t workspace_bytes, int32_t stages, int32_t tile_begin,
                   int32_t tile_end, const mlora_peer_ar* ar, const mlora_q8* q8, void* stream) {
  int st;
  const Plan* plan = plan_of(prob, route, &st);
  if (!plan) return st;
  const Plan& p = *plan;
  if (stages & ~(MLORA_STAGE_SHRINK | MLORA_STAGE_MAIN | MLORA_STAGE_NO_EXPAND)) return MLORA_ERR_INVALID_ARG;
  if (tile_begin < 0 || tile_end < tile_begin || tile_end > p.n_tiles) return MLORA_ERR_INVALID_ARG;
  if (prob->rows == 0 || tile_end == tile_begin) return MLORA_OK;
  const bool need_z = !p.chunks.empty() &&
                      ((stages & MLORA_STAGE_SHRINK) || ((stages & MLORA_STAGE_MAIN) && !(stages & MLORA_STAGE_NO_EXPAND)));
  if (!X || !workspace) return MLORA_ERR_INVALID_ARG;
  if ((stages & MLORA_STAGE_MAIN) && !Y && !ar) return MLORA_ERR_INVALID_ARG;
  if (need_z && !zsave) return MLORA_ERR_INVALID_ARG;
  if (!p.chunks.empty() && (stages & MLORA_STAGE_SHRINK) && !A_pack) return MLORA_ERR_INVALID_ARG;
  if (need_z && (stages & MLORA_STAGE_MAIN) && !(stages & MLORA_STAGE_NO_EXPAND) && !B_pack)
    return MLORA_ERR_INVALID_ARG;
  if (workspace_bytes < ws_bytes(p, prob->dtype)) return MLORA_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return MLORA_ERR_UNSUPPORTED;  // plan tables hold 16-byte entries
  const int impl = choose_impl(prob, {X, W, bias, A_pack, B_pack, Y, zsave});
  if (impl < 0) return MLORA_ERR_UNSUPPORTED;
  if (ar && (impl != MLORA_IMPL_TC || route->out_rows)) return MLORA_ERR_UNSUPPORTED;
  const bool q8_base = q8 && q8->Wq;
  // a few rows in 16 bits: rows and shrink in one launch
  const bool few = q8_base && impl == MLORA_IMPL_TC && prob->rows <= kQ8Few && !p.chunks.empty();
  cudaStream_t s = (cudaStream_t)stream;
  PlanDev dev;
  st = stage_plan(prob, p, workspace, s, &dev, !few);
  if (st != MLORA_OK) return st;
  // the launch that the 8-bit product follows
  const Q8After after = few || dev.n_chunks == 0 ? kAfterRows : impl == MLORA_IMPL_TC ? kAfterShrink : kAfterOther;
  if (few) {
    st = q8_few_prep(X, prob->rows, prob->d_in, prob->dtype, q8->Xq, q8->x_scale, dev, A_pack, zsave, s);
    if (st != MLORA_OK) return st;
    return q8_forward_main(prob, route, q8, dev, q8_impl(prob, impl), after, bias, B_pack, Y, zsave, s);
  }
  if (q8 && q8->Xq) {  // operand of the 8-bit product, the saved form of X, or both
    st = q8_quantize(X, prob->rows, prob->d_in, prob->d_in, prob->dtype, nullptr, (int8_t*)q8->Xq,
                     q8->x_scale, s);
    if (st != MLORA_OK) return st;
  }
  if (q8_base) stages &= ~MLORA_STAGE_MAIN;  // the kernels below run the shrink only
  if (impl == MLORA_IMPL_TC) {
    TcCall a;
    a.ar = ar;
    a.plan = dev;
    a.host = &p;
    a.M = prob->rows; a.d_in = prob->d_in; a.d_out = prob->d_out; a.R = route->r_pack;
    a.dtype = prob->dtype;
    a.X = X; a.W = W; a.bias = bias; a.A_pack = A_pack; a.B_pack = B_pack;
    a.Y = Y; a.zsave = zsave; a.out_rows = route->out_rows;
    a.stages = stages; a.t0 = tile_begin; a.t1 = tile_end;
    a.max_ctas = prob->max_ctas;
    // the forward on 2-SM pairs from K = 2048 on; below it the 1-SM mainloop
    // (measured: pairs 2-9 % faster at K 2048-8192, 15 % slower at K 1024)
    a.pair_fwd = prob->impl == MLORA_IMPL_TC_2SM || prob->impl == MLORA_IMPL_TC_WIDE ||
                 (prob->impl != MLORA_IMPL_TC_1SM && prob->d_in >= 2048);
    a.wide = prob->impl == MLORA_IMPL_TC_WIDE;
    st = tc_forward(a, s);
    if (st != MLORA_OK || !q8_base) return st;
    return q8_forward_main(prob, route, q8, dev, q8_impl(prob, impl), after, bias, B_pack, Y, zsave, s);
  }
  if (q8_base && prob->dtype == MLORA_F32) {
    st = q8_low32(false, dev, (const float*)X, (const float*)A_pack, (float*)zsave, prob->rows, prob->d_in,
                  prob->d_out, route->r_pack, s);
    if (st != MLORA_OK) return st;
    return q8_forward_main(prob, route, q8, dev, q8_impl(prob, impl), after, bias, B_pack, Y, zsave, s);
  }
  SimtCall a;
  a.plan = dev;
  a.n_chunks = dev.n_chunks;
  a.n_reduce = dev.n_reduce;
  a.M = prob->rows; a.d_in = prob->d_in; a.d_out = prob->d_out; a.R = route->r_pack;
  a.dtype = prob->dtype;
  a.X = X; a.W = W; a.bias = bias; a.A_pack = A_pack; a.B_pack = B_pack;
  a.Y = Y; a.zsave = zsave; a.out_rows = route->out_rows;
  a.stages = stages; a.t0 = tile_begin; a.t1 = tile_end;
  a.c_begin = p.tile_chunk_begin[tile_begin];
  a.c_end = p.tile_chunk_begin[tile_end];
  st = simt_forward(a, s);
  if (st != MLORA_OK || !q8_base) return st;
  return q8_forward_main(prob, route, q8, dev, q8_impl(prob, impl), after, bias, B_pack, Y, zsave, s);
}

}  // namespace

extern "C" int mlora_forward_staged(const mlora_problem* prob, const mlora_routing* route,
                                    const void* X, const void* W, const void* bias,
                                    const void* A_pack, const void* B_pack, void* Y, void* zsave,
                                    void* workspace, size_t workspace_bytes, int32_t stages,
                                    int32_t tile_begin, int32_t tile_end, void* stream) {
  return forward_staged(prob, route, X, W, bias, A_pack, B_pack, Y, zsave, workspace, workspace_bytes, stages,
                        tile_begin, tile_end, nullptr, nullptr, stream);
}

extern "C" int mlora_forward_push(const mlora_problem* prob, const mlora_routing* route,
                                  const void* X, const void* W, const void* bias,
                                  const void* A_pack, const void* B_pack, void* zsave,
                                  void* workspace, size_t workspace_bytes, int32_t stages,
                                  int32_t tile_begin, int32_t tile_end, const mlora_peer_ar* ar, void* stream) {
  if (!prob || !route || !ar) return MLORA_ERR_INVALID_ARG;
  if (ar->world < 1 || ar->world > MLORA_AR_MAX_RANKS || ar->rank < 0 || ar->rank >= ar->world)
    return MLORA_ERR_INVALID_ARG;
  if (ar->d_out != prob->d_out || ar->d_out % 8 != 0 || ar->n_tiles != mlora_num_tiles(prob->rows))
    return MLORA_ERR_INVALID_ARG;
  for (int r = 0; r < ar->world; ++r)
    if (!ar->recv[r] || !ar->arrive[r]) return MLORA_ERR_INVALID_ARG;
  if (prob->dtype != MLORA_BF16 && prob->dtype != MLORA_F16) return MLORA_ERR_UNSUPPORTED;
  return forward_staged(prob, route, X, W, bias, A_pack, B_pack, nullptr, zsave, workspace, workspace_bytes,
                        stages, tile_begin, tile_end, ar, nullptr, stream);
}

extern "C" int mlora_forward(const mlora_problem* prob, const mlora_routing* route, const void* X,
                             const void* W, const void* bias, const void* A_pack,
                             const void* B_pack, void* Y, void* zsave, void* workspace,
                             size_t workspace_bytes, void* stream) {
  if (!prob) return MLORA_ERR_INVALID_ARG;
  return mlora_forward_staged(prob, route, X, W, bias, A_pack, B_pack, Y, zsave, workspace,
                              workspace_bytes, MLORA_STAGE_SHRINK | MLORA_STAGE_MAIN, 0,
                              mlora_num_tiles(prob->rows), stream);
}

namespace {

// The kernels of a backward call on a staged plan; with `q8`, dA reads the
// saved 8-bit rows of X.  `isolate`: the reductions keep what is not finite in a
// row out of other segments' gradients (8-bit calls).
int backward_kernels(const mlora_problem* prob, const mlora_routing* route, const Plan& p, const PlanDev& dev,
                     int impl, const void* dY, const void* X, const void* W, const void* A_pack, const void* B_pack,
                     const void* zsave, void* dzsave, void* dX, void* dA_pack, void* dB_pack, int32_t stages,
                     int32_t tile_begin, int32_t tile_end, int32_t db_begin, int32_t db_end, bool isolate,
                     const mlora_q8* q8, cudaStream_t s) {
  if (impl == MLORA_IMPL_TC) {
    TcCall a;
    a.plan = dev;
    a.host = &p;
    a.M = prob->rows; a.d_in = prob->d_in; a.d_out = prob->d_out; a.R = route->r_pack;
    a.dtype = prob->dtype;
    a.X = X; a.W = W; a.A_pack = A_pack; a.B_pack = B_pack; a.dY = dY;
    a.zsave = (void*)zsave; a.dzt = dzsave; a.dX = dX; a.dA = dA_pack; a.dB = dB_pack;
    a.out_rows = route->out_rows;
    a.max_ctas = prob->max_ctas;
    a.pair_dx = prob->impl != MLORA_IMPL_TC_1SM;
    a.wide = prob->impl == MLORA_IMPL_TC_WIDE;
    a.bwd_stages = stages; a.t0 = tile_begin; a.t1 = tile_end; a.db0 = db_begin; a.db1 = db_end;
    a.lr = prob->lr;
    a.isolate = isolate;
    if (q8) { a.x_scale = q8->x_scale; a.dz8 = q8->scratch; }
    return tc_backward(a, s);
  }
  SimtCall a;
  a.plan = dev;
  a.n_chunks = dev.n_chunks;
  a.n_reduce = dev.n_reduce;
  a.M = prob->rows; a.d_in = prob->d_in; a.d_out = prob->d_out; a.R = route->r_pack;
  a.dtype = prob->dtype;
  a.X = X; a.W = W; a.A_pack = A_pack; a.B_pack = B_pack; a.dY = dY;
  a.zsave = (void*)zsave; a.dzt = dzsave; a.dX = dX; a.dA = dA_pack; a.dB = dB_pack;
  a.out_rows = route->out_rows;
  a.bwd_stages = stages; a.db0 = db_begin; a.db1 = db_end;
  a.lr = prob->lr;
  a.isolate = isolate;
  if (q8) { a.Xq = q8->Xq; a.x_scale = q8->x_scale; }
  a.c_begin = p.tile_chunk_begin[tile_begin];
  a.c_end = p.tile_chunk_begin[tile_end];
  return simt_backward(a, s);
}

Q8Saved saved_call(const mlora_problem* prob, const mlora_routing* route, const Plan& p, const PlanDev& dev,
                   const void* A_pack, void* dA_pack, int32_t stages, const mlora_q8* q8) {
  Q8Saved c;
  c.M = prob->rows; c.d_in = prob->d_in; c.dtype = prob->dtype;
  c.Xq = q8->Xq;
  c.plan = dev;
  c.scratch = q8->scratch;
  c.dA = dA_pack;
  c.A_upd = (stages & MLORA_BWD_SGD_A) ? const_cast<void*>(A_pack) : nullptr;
  c.lr = prob->lr;
  c.max_ctas = prob->max_ctas;
  return c;
}

// mlora_backward_q8 on a staged plan: the 8-bit product takes the place of
// the dX mainloop, the saved 8-bit rows that of X in dA.
int q8_backward(const mlora_problem* prob, const mlora_routing* route, const Plan& p, const PlanDev& dev, int impl,
                const void* dY, const void* X, const void* W, const void* A_pack, const void* B_pack,
                const void* zsave, void* dzsave, void* dX, void* dA_pack, void* dB_pack, int32_t stages,
                const mlora_q8* q8, cudaStream_t s) {
  const int nb_out = (prob->d_out + 127) / 128;
  const bool q8_dx = dX && q8->Wq && (stages & MLORA_BWD_DX);
  const bool saved8 = q8->Xq != nullptr;
  const int32_t reduce = MLORA_BWD_DA | MLORA_BWD_DB | MLORA_BWD_SGD_A | MLORA_BWD_SGD_B;
  if (!q8_dx && !saved8 && prob->dtype != MLORA_F32)
    return backward_kernels(prob, route, p, dev, impl, dY, X, W, A_pack, B_pack, zsave, dzsave, dX, dA_pack,
                            dB_pack, stages, 0, p.n_tiles, 0, nb_out, true, nullptr, s);
  // dZ (and the 16-bit dX), then the 8-bit dX, then the reductions
  const bool f32 = prob->dtype == MLORA_F32;
  int32_t first = stages & ~reduce;
  int st = MLORA_OK;
  if (f32 && (first & MLORA_BWD_DZ)) {
    st = q8_low32(true, dev, (const float*)dY, (const float*)B_pack, (float*)dzsave, prob->rows, prob->d_in,
                  prob->d_out, route->r_pack, s);
    if (st != MLORA_OK) return st;
    first &= ~MLORA_BWD_DZ;
  }
  st = backward_kernels(prob, route, p, dev, impl, dY, X, W, A_pack, B_pack, zsave, dzsave, q8_dx ? nullptr : dX,
                        dA_pack, dB_pack, first, 0, p.n_tiles, 0, nb_out, true,
                        saved8 && dA_pack ? q8 : nullptr, s);
  if (st != MLORA_OK) return st;
  if (q8_dx) {
    st = q8_quantize(dY, prob->rows, prob->d_out, prob->d_out, prob->dtype, q8->w_scale, q8->Gq, q8->g_scale, s);
    if (st != MLORA_OK) return st;
    Q8Main m;
    m.bwd = true;
    m.M = prob->rows; m.d_in = prob->d_in; m.d_out = prob->d_out; m.R = route->r_pack; m.dtype = prob->dtype;
    m.Aq = q8->Gq; m.a_scale = q8->g_scale;
    m.Wq = q8->Wq;
    m.out = dX; m.out_rows = route->out_rows;
    m.expand = dev.n_chunks > 0;
    m.plan = dev; m.zt = dzsave; m.pack = A_pack;
    m.max_ctas = prob->max_ctas;
    m.err = prob->err_word;
    st = q8_main(m, q8_impl(prob, impl), kAfterRows, s);
    if (st != MLORA_OK) return st;
  }
  if (f32) {
    if (dA_pack && (stages & MLORA_BWD_DA)) {
      float* upd = (stages & MLORA_BWD_SGD_A) ? (float*)const_cast<void*>(A_pack) : nullptr;
      st = q8_sum32(0, dev, q8->Xq, q8->x_scale, (const float*)X, (const float*)dzsave, (float*)dA_pack, prob->rows,
                    prob->d_in, prob->d_in, upd, prob->lr, s);
      if (st != MLORA_OK) return st;
    }
    if (!dB_pack || !(stages & MLORA_BWD_DB)) return MLORA_OK;
    // q8_sum32 reads the low-rank blocks 16 bytes at a time.  dZ lies in the
    // workspace, zsave where the caller has it: off such a boundary the
    // reduction that reads single elements takes its place
    if (!aligned(zsave, 16))
      return backward_kernels(prob, route, p, dev, MLORA_IMPL_SIMT, dY, nullptr, W, A_pack, B_pack, zsave, dzsave,
                              nullptr, nullptr, dB_pack, stages & (MLORA_BWD_DB | MLORA_BWD_SGD_B), 0, p.n_tiles, 0,
                              nb_out, true, nullptr, s);
    float* upd = (stages & MLORA_BWD_SGD_B) ? (float*)const_cast<void*>(B_pack) : nullptr;
    return q8_sum32(1, dev, nullptr, nullptr, (const float*)dY, (const float*)zsave, (float*)dB_pack, prob->rows,
                    prob->d_out, route->r_pack, upd, prob->lr, s);
  }
  if (!saved8)
    return backward_kernels(prob, route, p, dev, impl, dY, X, W, A_pack, B_pack, zsave, dzsave, nullptr, dA_pack,
                            dB_pack, stages & reduce, 0, p.n_tiles, 0, nb_out, true, nullptr, s);
  // dA from the saved 8-bit rows, dB as ever
  const int32_t of_a = MLORA_BWD_DA | MLORA_BWD_SGD_A, of_b = MLORA_BWD_DB | MLORA_BWD_SGD_B;
  if (dA_pack && (stages & MLORA_BWD_DA) && impl == MLORA_IMPL_TC) {
    st = q8_da_tc(saved_call(prob, route, p, dev, A_pack, dA_pack, stages, q8), s);
    if (st != MLORA_OK) return st;
  } else if (dA_pack && (stages & MLORA_BWD_DA)) {
    st = backward_kernels(prob, route, p, dev, MLORA_IMPL_SIMT, dY, nullptr, W, A_pack, B_pack, zsave, dzsave,
                          nullptr, dA_pack, nullptr, stages & of_a, 0, p.n_tiles, 0, nb_out, true, q8, s);
    if (st != MLORA_OK) return st;
  }
  if (!dB_pack || !(stages & MLORA_BWD_DB)) return MLORA_OK;
  return backward_kernels(prob, route, p, dev, impl, dY, nullptr, W, A_pack, B_pack, zsave, dzsave, nullptr, nullptr,
                          dB_pack, stages & of_b, 0, p.n_tiles, 0, nb_out, true, nullptr, s);
}

// mlora_backward_staged, or with `q8` mlora_backward_q8 over all ranges.
int backward_staged(const mlora_problem* prob, const mlora_routing* route, const void* dY, const void* X,
                    const void* W, const void* A_pack, const void* B_pack, const void* zsave, void* dzsave, void* dX,
                    void* dA_pack, void* dB_pack, void* workspace, size_t workspace_bytes, int32_t stages,
                    int32_t tile_begin, int32_t tile_end, int32_t db_begin, int32_t db_end, const mlora_q8* q8,
                    void* stream) {
  int st;
  const Plan* plan = plan_of(prob, route, &st);
  if (!plan) return st;
  const Plan& p = *plan;
  if (stages & ~(MLORA_BWD_DZ | MLORA_BWD_DX | MLORA_BWD_DA | MLORA_BWD_DB | MLORA_BWD_SGD_A | MLORA_BWD_SGD_B))
    return MLORA_ERR_INVALID_ARG;
  // the fused SGD step updates the weights whose gradients the call writes
  if ((stages & MLORA_BWD_SGD_A) && (!(stages & MLORA_BWD_DA) || !dA_pack || !A_pack)) return MLORA_ERR_INVALID_ARG;
  if ((stages & MLORA_BWD_SGD_B) && (!(stages & MLORA_BWD_DB) || !dB_pack || !B_pack)) return MLORA_ERR_INVALID_ARG;
  const int nb_out = (prob->d_out + 127) / 128;
  if (tile_begin < 0 || tile_end < tile_begin || tile_end > p.n_tiles) return MLORA_ERR_INVALID_ARG;
  if (db_begin < 0 || db_end < db_begin || db_end > nb_out) return MLORA_ERR_INVALID_ARG;
  if (prob->rows == 0) return MLORA_OK;
  if (!dY || !workspace) return MLORA_ERR_INVALID_ARG;
  const bool lora = !p.chunks.empty();
  const bool need_dz = lora && ((stages & MLORA_BWD_DZ) || (dX && (stages & MLORA_BWD_DX)) ||
                                (dA_pack && (stages & MLORA_BWD_DA)));
  if (need_dz && (!dzsave || !B_pack)) return MLORA_ERR_INVALID_ARG;
  if (lora && dX && (stages & MLORA_BWD_DX) && !A_pack) return MLORA_ERR_INVALID_ARG;
  if (lora && dB_pack && (stages & MLORA_BWD_DB) && !zsave) return MLORA_ERR_INVALID_ARG;
  const bool saved8 = q8 && q8->Xq;
  // (the 8-bit call reads X for dA only, and not where its 8-bit rows are given)
  if (q8 ? lora && dA_pack && (stages & MLORA_BWD_DA) && !X && !saved8
         : ((dA_pack && (stages & MLORA_BWD_DA)) || (dB_pack && (stages & MLORA_BWD_DB))) && !X)
    return MLORA_ERR_INVALID_ARG;
  if (workspace_bytes < ws_bytes(p, prob->dtype)) return MLORA_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return MLORA_ERR_UNSUPPORTED;  // plan tables hold 16-byte entries
  const int impl = choose_impl(prob, {dY, X, W, A_pack, B_pack, zsave, dzsave, dX, dA_pack, dB_pack});
  if (impl < 0) return MLORA_ERR_UNSUPPORTED;
  if (saved8 && lora && dA_pack && (stages & MLORA_BWD_DA) && impl == MLORA_IMPL_TC) {
    if (!q8->scratch) return MLORA_ERR_INVALID_ARG;
    if (!aligned(q8->scratch, 16)) return MLORA_ERR_UNSUPPORTED;
    if (q8->scratch_bytes < q8_scratch_bytes(p)) return MLORA_ERR_WORKSPACE;
  }
  cudaStream_t s = (cudaStream_t)stream;
  PlanDev dev;
  st = stage_plan(prob, p, workspace, s, &dev);
  if (st != MLORA_OK) return st;
  if (q8) return q8_backward(prob, route, p, dev, impl, dY, X, W, A_pack, B_pack, zsave, dzsave, dX, dA_pack,
                             dB_pack, stages, q8, s);
  return backward_kernels(prob, route, p, dev, impl, dY, X, W, A_pack, B_pack, zsave, dzsave, dX, dA_pack, dB_pack,
                          stages, tile_begin, tile_end, db_begin, db_end, false, nullptr, s);
}

}  // namespace

extern "C" int mlora_backward_staged(const mlora_problem* prob, const mlora_routing* route,
                                     const void* dY, const void* X, const void* W, const void* A_pack,
                                     const void* B_pack, const void* zsave, void* dzsave, void* dX,
                                     void* dA_pack, void* dB_pack, void* workspace, size_t workspace_bytes,
                                     int32_t stages, int32_t tile_begin, int32_t tile_end, int32_t db_begin,
                                     int32_t db_end, void* stream) {
  return backward_staged(prob, route, dY, X, W, A_pack, B_pack, zsave, dzsave, dX, dA_pack, dB_pack, workspace,
                         workspace_bytes, stages, tile_begin, tile_end, db_begin, db_end, nullptr, stream);
}

namespace {

int backward_all(const mlora_problem* prob, const mlora_routing* route, const void* dY, const void* X, const void* W,
                 const void* A_pack, const void* B_pack, const void* zsave, void* dX, void* dA_pack, void* dB_pack,
                 void* workspace, size_t workspace_bytes, const mlora_q8* q8, void* stream) {
  if (!prob || !route) return MLORA_ERR_INVALID_ARG;
  size_t plan_bytes = 0;
  {
    int st;
    const Plan* p = plan_of(prob, route, &st);
    if (!p) return st;
    plan_bytes = p->bytes;
  }
  // dZ scratch lives in the workspace after the plan tables
  void* dzt = workspace ? (uint8_t*)workspace + align_up(plan_bytes, 1024) : nullptr;
  int32_t stages = ((dX || dA_pack) ? MLORA_BWD_DZ : 0) | MLORA_BWD_DX | MLORA_BWD_DA | MLORA_BWD_DB;
  if (prob->flags & MLORA_FUSED_SGD)
    stages |= (dA_pack ? MLORA_BWD_SGD_A : 0) | (dB_pack ? MLORA_BWD_SGD_B : 0);
  return backward_staged(prob, route, dY, X, W, A_pack, B_pack, zsave, dzt, dX, dA_pack, dB_pack, workspace,
                         workspace_bytes, stages, 0, mlora_num_tiles(prob->rows), 0, (prob->d_out + 127) / 128, q8,
                         stream);
}

}  // namespace

extern "C" int mlora_backward(const mlora_problem* prob, const mlora_routing* route, const void* dY,
                              const void* X, const void* W, const void* A_pack, const void* B_pack,
                              const void* zsave, void* dX, void* dA_pack, void* dB_pack,
                              void* workspace, size_t workspace_bytes, void* stream) {
  return backward_all(prob, route, dY, X, W, A_pack, B_pack, zsave, dX, dA_pack, dB_pack, workspace,
                      workspace_bytes, nullptr, stream);
}

// ---------------------------------------------------------------- 8-bit entry points

extern "C" int64_t mlora_q8_ld(int64_t cols) { return cols <= 0 ? 0 : q8_ld(cols); }

namespace {

int check_rows_cols(int64_t rows, int64_t cols, int32_t dtype) {
  if (rows < 0 || rows > (int64_t(1) << 31) - kTileRows || cols < 1) return MLORA_ERR_INVALID_ARG;
  if (cols > (int64_t(1) << 30)) return MLORA_ERR_UNSUPPORTED;  // column indices and their steps are 32-bit
  if (dtype != MLORA_F32 && dtype != MLORA_BF16 && dtype != MLORA_F16) return MLORA_ERR_UNSUPPORTED;
  return MLORA_OK;
}

// shape of an 8-bit product whose sums run over d_in (the forward) or d_out (dX)
int check_q8_problem(const mlora_problem* prob, bool over_d_out) {
  if (!prob) return MLORA_ERR_INVALID_ARG;
  int st = check_rows_cols(prob->rows, prob->d_in, prob->dtype);
  if (st == MLORA_OK) st = check_rows_cols(prob->rows, prob->d_out, prob->dtype);
  if (st != MLORA_OK) return st;
  if (prob->max_ctas < 0) return MLORA_ERR_INVALID_ARG;
  return (over_d_out ? prob->d_out : prob->d_in) > kQ8MaxK ? MLORA_ERR_UNSUPPORTED : MLORA_OK;
}

}  // namespace

extern "C" int mlora_q8_scratch_bytes(const mlora_problem* prob, const mlora_routing* route, size_t* bytes) {
  if (!bytes) return MLORA_ERR_INVALID_ARG;
  int st;
  const Plan* p = plan_of(prob, route, &st);
  if (!p) return st;
  *bytes = prob->dtype == MLORA_F32 ? 0 : q8_scratch_bytes(*p);
  return MLORA_OK;
}

extern "C" int mlora_q8_quantize(const void* src, int64_t rows, int64_t cols, int64_t ld_src, int32_t dtype,
                                 const float* col_scale, int8_t* q, float* scale, void* stream) {
  int st = check_rows_cols(rows, cols, dtype);
  if (st != MLORA_OK) return st;
  if (ld_src < cols) return MLORA_ERR_INVALID_ARG;
  if (rows == 0) return MLORA_OK;
  if (!src || !q || !scale) return MLORA_ERR_INVALID_ARG;
  if (!aligned(src, size_t(elem_bytes(dtype)))) return MLORA_ERR_UNSUPPORTED;
  if ((st = check_q8({q}, {scale, col_scale})) != MLORA_OK) return st;
  return q8_quantize(src, rows, cols, ld_src, dtype, col_scale, q, scale, (cudaStream_t)stream);
}

extern "C" int mlora_q8_dequantize(const int8_t* q, const float* scale, int64_t rows, int64_t cols, int32_t dtype,
                                   void* dst, void* stream) {
  int st = check_rows_cols(rows, cols, dtype);
  if (st != MLORA_OK) return st;
  if (rows == 0) return MLORA_OK;
  if (!q || !scale || !dst) return MLORA_ERR_INVALID_ARG;
  if (!aligned(dst, size_t(elem_bytes(dtype)))) return MLORA_ERR_UNSUPPORTED;
  if ((st = check_q8({q}, {scale})) != MLORA_OK) return st;
  return q8_dequantize(q, scale, rows, cols, dtype, dst, (cudaStream_t)stream);
}

extern "C" int mlora_q8_linear(const mlora_problem* prob, const void* X, int64_t ld_x, int8_t* Xq, float* x_scale,
                               const int8_t* Wq, const float* w_scale, const void* bias, void* Y, void* stream) {
  int st = check_q8_problem(prob, false);
  if (st != MLORA_OK) return st;
  if (X && ld_x < prob->d_in) return MLORA_ERR_INVALID_ARG;
  if (prob->rows == 0) return MLORA_OK;
  if (!Xq || !x_scale || !Wq || !w_scale || !Y) return MLORA_ERR_INVALID_ARG;
  if (!pointers_aligned({X, bias, Y}, size_t(elem_bytes(prob->dtype)))) return MLORA_ERR_UNSUPPORTED;
  if ((st = check_q8({Xq, Wq}, {x_scale, w_scale})) != MLORA_OK) return st;
  cudaStream_t s = (cudaStream_t)stream;
  if (X && (st = q8_quantize(X, prob->rows, prob->d_in, ld_x, prob->dtype, nullptr, Xq, x_scale, s)) != MLORA_OK)
    return st;
  Q8Main m;
  m.M = prob->rows; m.d_in = prob->d_in; m.d_out = prob->d_out; m.dtype = prob->dtype;
  m.Aq = Xq; m.a_scale = x_scale; m.Wq = Wq; m.w_scale = w_scale; m.bias = bias; m.out = Y;
  m.max_ctas = prob->max_ctas; m.err = prob->err_word;
  return q8_main(m, prob->impl, X ? kAfterRows : kAfterOther, s);
}

extern "C" int mlora_q8_linear_dx(const mlora_problem* prob, const void* dY, int8_t* Gq, float* g_scale,
                                  const int8_t* Wq, const float* w_scale, void* dX, void* stream) {
  int st = check_q8_problem(prob, true);
  if (st != MLORA_OK) return st;
  if (prob->rows == 0) return MLORA_OK;
  if (!dY || !Gq || !g_scale || !Wq || !w_scale || !dX) return MLORA_ERR_INVALID_ARG;
  if (!pointers_aligned({dY, dX}, size_t(elem_bytes(prob->dtype)))) return MLORA_ERR_UNSUPPORTED;
  if ((st = check_q8({Gq, Wq}, {g_scale, w_scale})) != MLORA_OK) return st;
  cudaStream_t s = (cudaStream_t)stream;
  st = q8_quantize(dY, prob->rows, prob->d_out, prob->d_out, prob->dtype, w_scale, Gq, g_scale, s);
  if (st != MLORA_OK) return st;
  Q8Main m;
  m.bwd = true;
  m.M = prob->rows; m.d_in = prob->d_in; m.d_out = prob->d_out; m.dtype = prob->dtype;
  m.Aq = Gq; m.a_scale = g_scale; m.Wq = Wq; m.out = dX;
  m.max_ctas = prob->max_ctas; m.err = prob->err_word;
  return q8_main(m, prob->impl, kAfterRows, s);
}

extern "C" int mlora_forward_q8(const mlora_problem* prob, const mlora_routing* route, const mlora_q8* q8,
                                const void* X, const void* W, const void* bias, const void* A_pack,
                                const void* B_pack, void* Y, void* zsave, void* workspace, size_t workspace_bytes,
                                void* stream) {
  if (!prob || !route || !q8) return MLORA_ERR_INVALID_ARG;
  if (prob->rows != 0 && ((q8->Wq && (W || !q8->w_scale || !q8->Xq)) || (q8->Xq && !q8->x_scale)))
    return MLORA_ERR_INVALID_ARG;
  if (q8->Wq && check_q8_problem(prob, false) == MLORA_ERR_UNSUPPORTED) return MLORA_ERR_UNSUPPORTED;
  int st = check_q8({q8->Wq, q8->Xq}, {q8->w_scale, q8->x_scale});
  if (st != MLORA_OK) return st;
  return forward_staged(prob, route, X, W, bias, A_pack, B_pack, Y, zsave, workspace, workspace_bytes,
                        MLORA_STAGE_SHRINK | MLORA_STAGE_MAIN, 0, mlora_num_tiles(prob->rows), nullptr, q8, stream);
}

extern "C" int mlora_backward_q8(const mlora_problem* prob, const mlora_routing* route, const mlora_q8* q8,
                                 const void* dY, const void* X, const void* W, const void* A_pack,
                                 const void* B_pack, const void* zsave, void* dX, void* dA_pack, void* dB_pack,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  if (!prob || !route || !q8) return MLORA_ERR_INVALID_ARG;
  if (prob->rows != 0 &&
      ((q8->Wq && (W || !q8->w_scale || (dX && (!q8->Gq || !q8->g_scale)))) || (q8->Xq && !q8->x_scale)))
    return MLORA_ERR_INVALID_ARG;
  if (q8->Wq && dX && check_q8_problem(prob, true) == MLORA_ERR_UNSUPPORTED) return MLORA_ERR_UNSUPPORTED;
  int st = check_q8({q8->Wq, q8->Xq, q8->Gq}, {q8->w_scale, q8->x_scale, q8->g_scale});
  if (st != MLORA_OK) return st;
  return backward_all(prob, route, dY, X, W, A_pack, B_pack, zsave, dX, dA_pack, dB_pack, workspace,
                      workspace_bytes, q8, stream);
}

extern "C" int mlora_sgd(const mlora_sgd_item* items, int32_t n_items, float lr, int32_t dtype,
                         void* stream) {
  if (n_items < 0 || (n_items > 0 && !items)) return MLORA_ERR_INVALID_ARG;
  if (dtype != MLORA_F32 && dtype != MLORA_BF16 && dtype != MLORA_F16) return MLORA_ERR_UNSUPPORTED;
  for (int i = 0; i < n_items; ++i) {
    const mlora_sgd_item& it = items[i];
    if (it.rows < 0 || it.cols < 0) return MLORA_ERR_INVALID_ARG;
    if (it.rows * it.cols == 0) continue;
    if (!it.param || !it.grad || it.ld_param < it.cols || it.ld_grad < it.cols) return MLORA_ERR_INVALID_ARG;
  }
  return sgd_items(dtype, items, n_items, lr, (cudaStream_t)stream);
}

extern "C" int mlora_get_error(int32_t* flags) {
  if (!flags) return MLORA_ERR_INVALID_ARG;
  int v = 0;
  MLORA_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_err_word, sizeof(int)));
  *flags = v;
  return MLORA_OK;
}

extern "C" int mlora_clear_error(void) {
  int z = 0;
  MLORA_CUDA_TRY(cudaMemcpyToSymbol(g_err_word, &z, sizeof(int)));
  return MLORA_OK;
}

extern "C" int64_t mlora_launch_count(void) { return g_launches.load(); }

extern "C" const char* mlora_status_string(int status) {
  switch (status) {
    case MLORA_OK: return "ok";
    case MLORA_ERR_INVALID_ARG: return "invalid argument (shape, pointer or routing)";
    case MLORA_ERR_UNSUPPORTED: return "unsupported dtype, shape or kernel family";
    case MLORA_ERR_WORKSPACE: return "workspace or save buffer too small";
    case MLORA_ERR_CUDA: return "CUDA runtime error";
    case MLORA_ERR_DEVICE_FLAG: return "device bounds check fired";
    case MLORA_ERR_TIMEOUT: return "bounded device wait timed out";
    default: return "unknown status";
  }
}
