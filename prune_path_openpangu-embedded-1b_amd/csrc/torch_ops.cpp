// torch.library registration of the PrunePath ops (namespace `prunepath`) over the C ABI
// of libprunepath_moe.so (include/prunepath_moe.h). Host code only: the kernels live
// in the HIP library; this file checks arguments, allocates outputs with the caching
// allocator, passes the current HIP stream and turns a failed call into a RuntimeError
// (TORCH_CHECK). Each op also has a Meta implementation (shapes only) for fake-tensor
// tracing. There is no CPU implementation: CPU tensors are refused.
//
// Ops and the reference interfaces they stand for (paths relative to the reference
// repository root):
//   route, route_logits   softmax_thresholding (src/MoEBlock_origin.py:50-97); the
//                         prefill router / sort / select / scatter
//                         (src/tl_kernel_optimized_Ultimate_PanGU.py:40-124, 550-564)
//   bucket                moe_local_scan / moe_global_scan / moe_dispatch (:133-266)
//   pack_experts,
//   pack_router           physical_reorder_for_inference (src/openpangu_moe.py:212-256)
//   moe_decode(_into)     TauSparseMoE.forward_decode (:494-530)
//   moe_decode_batch(_into)  TauSparseMoE.forward_prefill (:532-604) for 1 <= N <= 64
//                         tokens (the reference takes it for every N > 1, :606-615)
//   moe_prefill(_into)    TauSparseMoE.forward_prefill (:532-604)
//   masked_gate(_bwd)     MoELayer.forward's expert gating and its backward
//                         (src/MoEBlock_origin.py:205-212)
//   rotary, qk_norm_rotary(_bwd), kv_append(_q), kv_read(_into), paged_attention(_into)
//                         no counterpart in the reference's own code: the attention side of a
//                         decoder that serves several sequences
#include <ATen/ATen.h>
#include <algorithm>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/core/stack.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include "../../include/prunepath_moe.h"

namespace {

using at::Tensor;
using c10::optional;

void* stream_of(const Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == PP_OK, "prunepath.", what, " failed (code ", rc, "): ", pp_last_error());
}

void need_gpu(const char* name, const Tensor& ref, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts) {
    if (t == nullptr || !t->defined()) continue;
    TORCH_CHECK(t->is_cuda(), "prunepath.", name, ": tensors must be on the GPU (got ", t->device(),
                "); there is no CPU implementation");
    TORCH_CHECK(t->is_contiguous(), "prunepath.", name, ": tensors must be contiguous");
    TORCH_CHECK(t->device() == ref.device(), "prunepath.", name, ": tensors on different devices (",
                ref.device(), ", ", t->device(), ")");
  }
}

const void* ptr(const optional<Tensor>& t) { return (t.has_value() && t->defined()) ? t->data_ptr() : nullptr; }

int x_code(const Tensor& x, const char* name) {
  if (x.scalar_type() == at::kBFloat16) return PP_DTYPE_BF16;
  TORCH_CHECK(x.scalar_type() == at::kFloat, "prunepath.", name, ": x must be float32 or bfloat16 (got ",
              x.scalar_type(), ")");
  return PP_DTYPE_F32;
}

int w_code(const Tensor& w, const char* name) {
  if (w.scalar_type() == at::kBFloat16) return PP_DTYPE_BF16;
  TORCH_CHECK(w.scalar_type() == at::kFloat, "prunepath.", name, ": weights must be float32 or bfloat16 (got ",
              w.scalar_type(), ")");
  return PP_DTYPE_F32;
}

void check_bias(const optional<Tensor>& bias, int64_t E, const char* name) {
  if (!bias.has_value()) return;
  TORCH_CHECK(bias->scalar_type() == at::kFloat && bias->numel() == E, "prunepath.", name,
              ": bias must be float32 [E]");
}

// ------------------------------------------------------------------ routing
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> route_gpu(const Tensor& x, const Tensor& router_packed,
                                                             const optional<Tensor>& bias, int64_t E,
                                                             double tau) {
  TORCH_CHECK(x.dim() == 2, "prunepath.route: x must be [N, H]");
  check_bias(bias, E, "route");
  need_gpu("route", x, {&x, &router_packed, bias.has_value() ? &*bias : nullptr});
  const c10::DeviceGuard g(x.device());
  const int64_t N = x.size(0), H = x.size(1);
  auto f = x.options().dtype(at::kFloat);
  Tensor logits = at::empty({N, E}, f), probs = at::empty({N, E}, f), gates = at::empty({N, E}, f);
  Tensor mask = at::empty({N, E}, x.options().dtype(at::kByte));
  Tensor count = at::empty({N}, x.options().dtype(at::kInt));
  check_rc(pp_route(x.data_ptr(), x_code(x, "route"), N, (int)H, router_packed.data_ptr<float>(),
                    (const float*)ptr(bias), (int)E, (float)tau, logits.data_ptr<float>(), probs.data_ptr<float>(),
                    gates.data_ptr<float>(), mask.data_ptr<uint8_t>(), count.data_ptr<int32_t>(), stream_of(x)),
           "route");
  return {logits, probs, gates, mask, count};
}

// Meta implementations use symbolic sizes (c10::SymInt), so the ops trace with dynamic shapes.
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> route_meta(const Tensor& x, const Tensor&,
                                                              const optional<Tensor>&, int64_t E, double) {
  const c10::SymInt N = x.sym_size(0);
  auto f = x.options().dtype(at::kFloat);
  return {at::empty_symint({N, E}, f), at::empty_symint({N, E}, f), at::empty_symint({N, E}, f),
          at::empty_symint({N, E}, x.options().dtype(at::kByte)), at::empty_symint({N}, x.options().dtype(at::kInt))};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> route_logits_gpu(const Tensor& logits, double tau) {
  TORCH_CHECK(logits.scalar_type() == at::kFloat && logits.dim() == 2,
              "prunepath.route_logits: logits must be float32 [N, E]");
  need_gpu("route_logits", logits, {&logits});
  const c10::DeviceGuard g(logits.device());
  const int64_t N = logits.size(0), E = logits.size(1);
  Tensor probs = at::empty_like(logits), gates = at::empty_like(logits);
  Tensor mask = at::empty({N, E}, logits.options().dtype(at::kByte));
  Tensor count = at::empty({N}, logits.options().dtype(at::kInt));
  check_rc(pp_route_logits(logits.data_ptr<float>(), N, (int)E, (float)tau, probs.data_ptr<float>(),
                           gates.data_ptr<float>(), mask.data_ptr<uint8_t>(), count.data_ptr<int32_t>(),
                           stream_of(logits)),
           "route_logits");
  return {probs, gates, mask, count};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> route_logits_meta(const Tensor& logits, double) {
  const c10::SymInt N = logits.sym_size(0), E = logits.sym_size(1);
  return {at::empty_like(logits), at::empty_like(logits), at::empty_symint({N, E}, logits.options().dtype(at::kByte)),
          at::empty_symint({N}, logits.options().dtype(at::kInt))};
}

// ------------------------------------------------------------------ bucketing
// Output shapes of bucket: token_ids / pair_gates hold N*E + 1 entries (never empty),
// tiles the pp_max_tiles bound (N*E) / tile_m + E rows.
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> bucket_shapes(const Tensor& mask, int64_t tile_m) {
  const c10::SymInt N = mask.sym_size(0), E = mask.sym_size(1);
  const int64_t tm = tile_m > 0 ? tile_m : pp_gemm_tile_m();
  const c10::SymInt cap = N * E + 1, mt = (N * E) / tm + E;
  auto i32 = mask.options().dtype(at::kInt);
  return {at::empty_symint({E + 1}, i32),
          at::empty_symint({cap}, i32),
          at::empty_symint({cap}, mask.options().dtype(at::kFloat)),
          at::empty_symint({N, E}, i32),
          at::empty_symint({mt, 4}, i32),
          at::empty({4}, i32)};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> bucket_gpu(const Tensor& mask, const Tensor& gates,
                                                                      int64_t tile_m) {
  TORCH_CHECK(mask.scalar_type() == at::kByte && gates.scalar_type() == at::kFloat && mask.dim() == 2 &&
                  mask.sizes() == gates.sizes(),
              "prunepath.bucket: mask uint8 [N, E] and gates float32 [N, E] required");
  need_gpu("bucket", mask, {&mask, &gates});
  const c10::DeviceGuard g(mask.device());
  const int64_t N = mask.size(0), E = mask.size(1);
  const int tm = tile_m > 0 ? (int)tile_m : pp_gemm_tile_m();
  auto r = bucket_shapes(mask, tm);
  TORCH_CHECK(std::get<4>(r).size(0) == pp_max_tiles(N, (int)E, tm), "prunepath.bucket: tile bound mismatch");
  // capacity tails (token_ids / pair_gates past offsets[E], tiles past meta[0]) are zero,
  // so every output element is defined and the op's results are the same on every call
  std::get<1>(r).zero_();
  std::get<2>(r).zero_();
  std::get<4>(r).zero_();
  Tensor ws = at::empty({(int64_t)pp_bucket_workspace_bytes(N, (int)E)}, mask.options().dtype(at::kByte));
  check_rc(pp_bucket(mask.data_ptr<uint8_t>(), gates.data_ptr<float>(), N, (int)E, tm,
                     std::get<0>(r).data_ptr<int32_t>(), std::get<1>(r).data_ptr<int32_t>(),
                     std::get<2>(r).data_ptr<float>(), std::get<3>(r).data_ptr<int32_t>(),
                     std::get<4>(r).data_ptr<int32_t>(), std::get<5>(r).data_ptr<int32_t>(), ws.data_ptr(),
                     stream_of(mask)),
           "bucket");
  return r;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> bucket_meta(const Tensor& mask, const Tensor&,
                                                                       int64_t tile_m) {
  return bucket_shapes(mask, tile_m);
}

// ------------------------------------------------------------------ rearrangement
struct PackLayout {
  int64_t H, I, s_n, s_h, d_n, d_h;
};

PackLayout pack_layout(const Tensor& w_gate, const Tensor& w_down, c10::string_view layout) {
  TORCH_CHECK(w_gate.dim() == 2 && w_down.dim() == 2, "prunepath.pack_experts: 2-D weights required");
  if (layout == "linear") {  // gate/up [I, H], down [H, I]
    const int64_t I = w_gate.size(0), H = w_gate.size(1);
    TORCH_CHECK(w_down.size(0) == H && w_down.size(1) == I, "prunepath.pack_experts: down must be [H, I]");
    return {H, I, H, 1, 1, I};
  }
  TORCH_CHECK(layout == "tau", "prunepath.pack_experts: layout must be 'linear' or 'tau'");
  const int64_t H = w_gate.size(0), I = w_gate.size(1);  // W_gate/W_up [H, I], W_down [I, H]
  TORCH_CHECK(w_down.size(0) == I && w_down.size(1) == H, "prunepath.pack_experts: W_down must be [I, H]");
  return {H, I, 1, I, H, 1};
}

Tensor pack_experts_gpu(const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down, int64_t E, int64_t G,
                        const optional<Tensor>& perm, c10::string_view layout) {
  const PackLayout L = pack_layout(w_gate, w_down, layout);
  TORCH_CHECK(w_up.sizes() == w_gate.sizes() && w_up.scalar_type() == w_gate.scalar_type() &&
                  w_down.scalar_type() == w_gate.scalar_type(),
              "prunepath.pack_experts: gate/up/down shapes or dtypes disagree");
  TORCH_CHECK(L.I == E * G, "prunepath.pack_experts: I=", L.I, " != E*G=", E * G);
  if (perm.has_value())
    TORCH_CHECK(perm->scalar_type() == at::kInt && perm->numel() == L.I, "prunepath.pack_experts: perm must be int32 [I]");
  need_gpu("pack_experts", w_gate, {&w_gate, &w_up, &w_down, perm.has_value() ? &*perm : nullptr});
  const c10::DeviceGuard g(w_gate.device());
  Tensor out = at::empty({(int64_t)(pp_packed_expert_bytes((int)L.H, (int)E, (int)G) / 2)},
                         w_gate.options().dtype(at::kBFloat16));
  check_rc(pp_pack_experts(w_gate.data_ptr(), w_up.data_ptr(), L.s_n, L.s_h, w_down.data_ptr(), L.d_n, L.d_h,
                           w_code(w_gate, "pack_experts"), (const int32_t*)ptr(perm), (int)L.H, (int)E, (int)G,
                           out.data_ptr(), stream_of(w_gate)),
           "pack_experts");
  return out;
}

Tensor pack_experts_meta(const Tensor& w_gate, const Tensor&, const Tensor&, int64_t E, int64_t G,
                         const optional<Tensor>&, c10::string_view layout) {
  // packed = rows [E*G][3][H] + down_t [E][H][G]: 4*E*G*H bf16 (pp_packed_expert_bytes / 2)
  const c10::SymInt H = layout == "linear" ? w_gate.sym_size(1) : w_gate.sym_size(0);
  return at::empty_symint({H * (4 * E * G)}, w_gate.options().dtype(at::kBFloat16));
}

std::pair<int64_t, int64_t> router_dims(const Tensor& w, c10::string_view layout, int64_t* s_e, int64_t* s_h) {
  TORCH_CHECK(w.dim() == 2, "prunepath.pack_router: 2-D router weights required");
  if (layout == "linear") {  // [E, H]
    *s_e = w.size(1);
    *s_h = 1;
    return {w.size(0), w.size(1)};
  }
  TORCH_CHECK(layout == "tau", "prunepath.pack_router: layout must be 'linear' or 'tau'");
  *s_e = 1;  // [H, E]
  *s_h = w.size(1);
  return {w.size(1), w.size(0)};
}

Tensor pack_router_gpu(const Tensor& w, c10::string_view layout) {
  int64_t s_e, s_h;
  const auto [E, H] = router_dims(w, layout, &s_e, &s_h);
  need_gpu("pack_router", w, {&w});
  const c10::DeviceGuard g(w.device());
  Tensor out = at::empty({(E + 15) / 16 * 16, H}, w.options().dtype(at::kFloat));
  check_rc(pp_pack_router(w.data_ptr(), s_e, s_h, w_code(w, "pack_router"), (int)H, (int)E, out.data_ptr<float>(),
                          stream_of(w)),
           "pack_router");
  return out;
}

Tensor pack_router_meta(const Tensor& w, c10::string_view layout) {
  const c10::SymInt E = layout == "linear" ? w.sym_size(0) : w.sym_size(1);
  const c10::SymInt H = layout == "linear" ? w.sym_size(1) : w.sym_size(0);
  return at::empty_symint({(E + 15) / 16 * 16, H}, w.options().dtype(at::kFloat));
}

// ------------------------------------------------------------------ decode
void decode_workspace_init_gpu(const Tensor& ws, int64_t H, int64_t E) {
  TORCH_CHECK(ws.scalar_type() == at::kByte && ws.numel() >= (int64_t)pp_decode_workspace_bytes((int)H, (int)E),
              "prunepath.decode_workspace_init: uint8 workspace of pp_decode_workspace_bytes(H, E) required");
  need_gpu("decode_workspace_init", ws, {&ws});
  const c10::DeviceGuard g(ws.device());
  check_rc(pp_decode_workspace_init(ws.data_ptr(), (int)H, (int)E, stream_of(ws)), "decode_workspace_init");
}

void decode_workspace_init_meta(const Tensor&, int64_t, int64_t) {}

void decode_into(const Tensor& x, const Tensor& router_packed, const optional<Tensor>& bias, int64_t E, int64_t G,
                 double tau, const Tensor& packed, const Tensor& workspace, const Tensor& out, int64_t grid) {
  const int64_t H = x.numel();
  check_bias(bias, E, "moe_decode");
  TORCH_CHECK(workspace.scalar_type() == at::kByte &&
                  workspace.numel() >= (int64_t)pp_decode_workspace_bytes((int)H, (int)E),
              "prunepath.moe_decode: uint8 workspace of pp_decode_workspace_bytes(H, E) required");
  TORCH_CHECK(out.scalar_type() == at::kBFloat16 && out.numel() == H, "prunepath.moe_decode: out must be bf16 [1, H]");
  need_gpu("moe_decode", x, {&x, &router_packed, bias.has_value() ? &*bias : nullptr, &packed, &workspace, &out});
  const c10::DeviceGuard g(x.device());
  check_rc(pp_moe_decode(x.data_ptr(), x_code(x, "moe_decode"), (int)H, router_packed.data_ptr<float>(),
                         (const float*)ptr(bias), (int)E, (int)G, (float)tau, packed.data_ptr(), out.data_ptr(),
                         workspace.data_ptr(), (int)grid, stream_of(x)),
           "moe_decode");
}

Tensor moe_decode_gpu(const Tensor& x, const Tensor& router_packed, const optional<Tensor>& bias, int64_t E,
                      int64_t G, double tau, const Tensor& packed, const Tensor& workspace, int64_t grid) {
  Tensor out = at::empty({1, x.numel()}, x.options().dtype(at::kBFloat16));
  decode_into(x, router_packed, bias, E, G, tau, packed, workspace, out, grid);
  return out;
}

void moe_decode_into_meta(const Tensor&, const Tensor&, const optional<Tensor>&, int64_t, int64_t, double,
                          const Tensor&, const Tensor&, const Tensor&, int64_t) {}

Tensor moe_decode_meta(const Tensor& x, const Tensor&, const optional<Tensor>&, int64_t, int64_t, double,
                       const Tensor&, const Tensor&, int64_t) {
  return at::empty_symint({c10::SymInt(1), x.sym_numel()}, x.options().dtype(at::kBFloat16));
}

// ------------------------------------------------------------------ small-batch decode
void decode_batch_into(const Tensor& x, const Tensor& router_packed, const optional<Tensor>& bias, int64_t E,
                       int64_t G, double tau, const Tensor& packed, const Tensor& workspace,
                       const Tensor& batch_workspace, const Tensor& out, const optional<Tensor>& logits_out,
                       const optional<Tensor>& mask_out, int64_t grid) {
  TORCH_CHECK(x.dim() == 2, "prunepath.moe_decode_batch: x must be [N, H]");
  const int64_t N = x.size(0), H = x.size(1);
  check_bias(bias, E, "moe_decode_batch");
  TORCH_CHECK(workspace.scalar_type() == at::kByte &&
                  workspace.numel() >= (int64_t)pp_decode_workspace_bytes((int)H, (int)E),
              "prunepath.moe_decode_batch: uint8 workspace of pp_decode_workspace_bytes(H, E) required");
  TORCH_CHECK(batch_workspace.scalar_type() == at::kByte &&
                  batch_workspace.numel() >= (int64_t)pp_decode_batch_workspace_bytes((int)H, (int)E, (int)G),
              "prunepath.moe_decode_batch: uint8 batch_workspace of pp_decode_batch_workspace_bytes(H, E, G) required");
  TORCH_CHECK(out.scalar_type() == at::kBFloat16 && out.numel() == N * H && out.is_contiguous(),
              "prunepath.moe_decode_batch: out must be contiguous bf16 [N, H]");
  if (logits_out.has_value())
    TORCH_CHECK(logits_out->scalar_type() == at::kFloat && logits_out->numel() == N * E && logits_out->is_contiguous(),
                "prunepath.moe_decode_batch: logits_out must be contiguous fp32 [N, E]");
  if (mask_out.has_value())
    TORCH_CHECK(mask_out->scalar_type() == at::kByte && mask_out->numel() == N * E && mask_out->is_contiguous(),
                "prunepath.moe_decode_batch: mask_out must be contiguous uint8 [N, E]");
  need_gpu("moe_decode_batch", x,
           {&x, &router_packed, bias.has_value() ? &*bias : nullptr, &packed, &workspace, &batch_workspace, &out,
            logits_out.has_value() ? &*logits_out : nullptr, mask_out.has_value() ? &*mask_out : nullptr});
  const c10::DeviceGuard g(x.device());
  check_rc(pp_moe_decode_batch(x.data_ptr(), x_code(x, "moe_decode_batch"), N, (int)H,
                               router_packed.data_ptr<float>(), (const float*)ptr(bias), (int)E, (int)G, (float)tau,
                               packed.data_ptr(), out.data_ptr(),
                               logits_out.has_value() ? logits_out->data_ptr<float>() : nullptr,
                               mask_out.has_value() ? mask_out->data_ptr<uint8_t>() : nullptr, workspace.data_ptr(),
                               batch_workspace.data_ptr(), (int)grid, stream_of(x)),
           "moe_decode_batch");
}

Tensor moe_decode_batch_gpu(const Tensor& x, const Tensor& router_packed, const optional<Tensor>& bias, int64_t E,
                            int64_t G, double tau, const Tensor& packed, const Tensor& workspace,
                            const Tensor& batch_workspace, int64_t grid) {
  TORCH_CHECK(x.dim() == 2, "prunepath.moe_decode_batch: x must be [N, H]");
  Tensor out = at::empty({x.size(0), x.size(1)}, x.options().dtype(at::kBFloat16));
  decode_batch_into(x, router_packed, bias, E, G, tau, packed, workspace, batch_workspace, out, c10::nullopt,
                    c10::nullopt, grid);
  return out;
}

Tensor moe_decode_batch_meta(const Tensor& x, const Tensor&, const optional<Tensor>&, int64_t, int64_t, double,
                             const Tensor&, const Tensor&, const Tensor&, int64_t) {
  return at::empty_symint(x.sym_sizes(), x.options().dtype(at::kBFloat16));
}

void moe_decode_batch_into_meta(const Tensor&, const Tensor&, const optional<Tensor>&, int64_t, int64_t, double,
                                const Tensor&, const Tensor&, const Tensor&, const Tensor&, const optional<Tensor>&,
                                const optional<Tensor>&, int64_t) {}

// ------------------------------------------------------------------ prefill
// One implementation behind both boundaries: pp_moe_prefill_routed (the grouped pipeline,
// or for G % 64 != 0 the dense form of csrc/dense.hip), hand-written kernels only.
void prefill_into(const Tensor& x, const Tensor& router_packed, const optional<Tensor>& bias, int64_t E, int64_t G,
                  double tau, const Tensor& packed, const Tensor& workspace, const Tensor& out,
                  const optional<Tensor>& logits_out, const optional<Tensor>& mask_out) {
  TORCH_CHECK(x.dim() == 2, "prunepath.moe_prefill: x must be [N, H]");
  const int64_t N = x.size(0), H = x.size(1);
  check_bias(bias, E, "moe_prefill");
  TORCH_CHECK(x.is_contiguous() && packed.is_contiguous(), "prunepath.moe_prefill: x and packed must be contiguous");
  TORCH_CHECK(workspace.scalar_type() == at::kByte &&
                  workspace.numel() >= (int64_t)pp_prefill_workspace_bytes(N, (int)H, (int)E, (int)G),
              "prunepath.moe_prefill: uint8 workspace of pp_prefill_workspace_bytes(N, H, E, G) required");
  TORCH_CHECK(out.scalar_type() == at::kBFloat16 && out.numel() == N * H && out.is_contiguous(),
              "prunepath.moe_prefill: out must be contiguous bf16 [N, H]");
  if (logits_out.has_value())
    TORCH_CHECK(logits_out->scalar_type() == at::kFloat && logits_out->numel() == N * E && logits_out->is_contiguous(),
                "prunepath.moe_prefill: logits_out must be contiguous fp32 [N, E]");
  if (mask_out.has_value())
    TORCH_CHECK(mask_out->scalar_type() == at::kByte && mask_out->numel() == N * E && mask_out->is_contiguous(),
                "prunepath.moe_prefill: mask_out must be contiguous uint8 [N, E]");
  need_gpu("moe_prefill", x,
           {&x, &router_packed, bias.has_value() ? &*bias : nullptr, &packed, &workspace, &out,
            logits_out.has_value() ? &*logits_out : nullptr, mask_out.has_value() ? &*mask_out : nullptr});
  const c10::DeviceGuard g(x.device());
  check_rc(pp_moe_prefill_routed(x.data_ptr(), x_code(x, "moe_prefill"), N, (int)H, router_packed.data_ptr<float>(),
                                 (const float*)ptr(bias), (int)E, (int)G, (float)tau, packed.data_ptr(),
                                 out.data_ptr(), workspace.data_ptr(),
                                 logits_out.has_value() ? logits_out->data_ptr<float>() : nullptr,
                                 mask_out.has_value() ? mask_out->data_ptr<uint8_t>() : nullptr, stream_of(x)),
           "moe_prefill");
}

Tensor moe_prefill_gpu(const Tensor& x, const Tensor& router_packed, const optional<Tensor>& bias, int64_t E,
                       int64_t G, double tau, const Tensor& packed) {
  TORCH_CHECK(x.dim() == 2, "prunepath.moe_prefill: x must be [N, H]");
  const int64_t N = x.size(0), H = x.size(1);
  Tensor out = at::empty({N, H}, x.options().dtype(at::kBFloat16));
  Tensor ws = at::empty({(int64_t)pp_prefill_workspace_bytes(N, (int)H, (int)E, (int)G)},
                        x.options().dtype(at::kByte));
  prefill_into(x, router_packed, bias, E, G, tau, packed, ws, out, c10::nullopt, c10::nullopt);
  return out;
}

Tensor moe_prefill_meta(const Tensor& x, const Tensor&, const optional<Tensor>&, int64_t, int64_t, double,
                        const Tensor&) {
  return at::empty_symint(x.sym_sizes(), x.options().dtype(at::kBFloat16));
}

void moe_prefill_into_meta(const Tensor&, const Tensor&, const optional<Tensor>&, int64_t, int64_t, double,
                           const Tensor&, const Tensor&, const Tensor&, const optional<Tensor>&,
                           const optional<Tensor>&) {}

// CPU tensors: refused with the op's name (there is no host implementation, on purpose).
// ------------------------------------------------------------------ masked gating (training)
// masked_gate / masked_gate_bwd: MoELayer.forward's mask matmul and multiply
// (src/MoEBlock_origin.py:205-212), out = inter * gates[:, expert_ids], and its backward
// (autograd of masked_gate is registered from Python: ops.py). inter / d_out [..., I]
// (fp32 or bf16, the rows flattened), gates [..., E] fp32, expert_ids / perm int32 [I],
// seg int32 [E + 1] (masked_gate_layout in ops.py); perm and seg are the backward's
// expert segments, carried by the forward for autograd.
void masked_gate_check(const char* name, const Tensor& inter, const Tensor& gates, const Tensor& eid) {
  TORCH_CHECK(inter.dim() >= 1 && gates.dim() >= 1, "prunepath.", name, ": inter [..., I] and gates [..., E]");
  TORCH_CHECK(gates.scalar_type() == at::kFloat, "prunepath.", name, ": gates must be float32");
  TORCH_CHECK(eid.scalar_type() == at::kInt && eid.numel() == inter.size(-1), "prunepath.", name,
              ": expert_ids must be int32 [I]");
  TORCH_CHECK(gates.numel() / std::max<int64_t>(1, gates.size(-1)) == inter.numel() / std::max<int64_t>(1, inter.size(-1)),
              "prunepath.", name, ": inter and gates have different row counts");
}

Tensor masked_gate_gpu(const Tensor& inter, const Tensor& gates, const Tensor& eid, const Tensor& perm,
                       const Tensor& seg) {
  masked_gate_check("masked_gate", inter, gates, eid);
  need_gpu("masked_gate", inter, {&inter, &gates, &eid, &perm, &seg});
  const c10::DeviceGuard g(inter.device());
  const int64_t I = inter.size(-1), E = gates.size(-1), n = inter.numel() / std::max<int64_t>(1, I);
  Tensor out = at::empty_like(inter);
  if (n == 0) return out;
  check_rc(pp_masked_gate_fwd(inter.data_ptr(), x_code(inter, "masked_gate"), gates.data_ptr<float>(),
                              eid.data_ptr<int32_t>(), n, (int)I, (int)E, out.data_ptr(), stream_of(inter)),
           "masked_gate");
  return out;
}

Tensor masked_gate_meta(const Tensor& inter, const Tensor&, const Tensor&, const Tensor&, const Tensor&) {
  return at::empty_like(inter);
}

std::tuple<Tensor, Tensor> masked_gate_bwd_gpu(const Tensor& d_out, const Tensor& inter, const Tensor& gates,
                                               const Tensor& eid, const Tensor& perm, const Tensor& seg,
                                               bool need_d_inter) {
  masked_gate_check("masked_gate_bwd", inter, gates, eid);
  TORCH_CHECK(d_out.sizes() == inter.sizes() && d_out.scalar_type() == inter.scalar_type(),
              "prunepath.masked_gate_bwd: d_out must match inter's shape and dtype");
  TORCH_CHECK(perm.scalar_type() == at::kInt && perm.numel() == inter.size(-1) && seg.scalar_type() == at::kInt &&
                  seg.numel() == gates.size(-1) + 1,
              "prunepath.masked_gate_bwd: perm int32 [I] and seg int32 [E + 1] required");
  need_gpu("masked_gate_bwd", inter, {&d_out, &inter, &gates, &eid, &perm, &seg});
  const c10::DeviceGuard g(inter.device());
  const int64_t I = inter.size(-1), E = gates.size(-1), n = inter.numel() / std::max<int64_t>(1, I);
  Tensor d_inter = need_d_inter ? at::empty_like(inter) : at::empty({0}, inter.options());
  Tensor d_gates = at::empty_like(gates);
  if (n == 0) return {d_inter, d_gates};
  check_rc(pp_masked_gate_bwd(d_out.data_ptr(), inter.data_ptr(), x_code(inter, "masked_gate_bwd"),
                              gates.data_ptr<float>(), eid.data_ptr<int32_t>(), perm.data_ptr<int32_t>(),
                              seg.data_ptr<int32_t>(), n, (int)I, (int)E, need_d_inter ? d_inter.data_ptr() : nullptr,
                              d_gates.data_ptr<float>(), stream_of(inter)),
           "masked_gate_bwd");
  return {d_inter, d_gates};
}

std::tuple<Tensor, Tensor> masked_gate_bwd_meta(const Tensor&, const Tensor& inter, const Tensor& gates,
                                                const Tensor&, const Tensor&, const Tensor&, bool need_d_inter) {
  return {need_d_inter ? at::empty_like(inter) : at::empty({0}, inter.options()), at::empty_like(gates)};
}

// ------------------------------------------------------------------ rotary positions
int rotary_layout(c10::string_view layout, const char* name) {
  if (layout == "half") return PP_ROTARY_HALF;
  TORCH_CHECK(layout == "interleaved", "prunepath.", name, ": layout must be 'half' or 'interleaved'");
  return PP_ROTARY_INTERLEAVED;
}

void same_device(const char* name, const Tensor& ref, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts) {
    TORCH_CHECK(t->is_cuda(), "prunepath.", name, ": tensors must be on the GPU (got ", t->device(),
                "); there is no CPU implementation");
    TORCH_CHECK(t->device() == ref.device(), "prunepath.", name, ": tensors on different devices (", ref.device(), ", ",
                t->device(), ")");
  }
}

// The stride of a dimension as the kernels take it: that of one of a single element says nothing, and must
// not fail the checks of alignment.
int64_t step(const Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

// The bytes from a tensor's first element to its last.
struct Span {
  uintptr_t first, end;
  explicit Span(const Tensor& t) : first((uintptr_t)t.data_ptr()), end(first) {
    int64_t n = 1;
    const auto sizes = t.sizes(), strides = t.strides();
    for (size_t i = 0; i < sizes.size(); ++i) {
      if (sizes[i] == 0) return;
      n += (sizes[i] - 1) * strides[i];
    }
    end += (uintptr_t)(n * (int64_t)t.element_size());
  }
};

// What a call writes lies apart from what it reads, but for an output that is the input itself.
void apart(const char* name, const Span& out, const Span& in) {
  TORCH_CHECK(out.end <= in.first || in.end <= out.first, "prunepath.", name, ": an output overlaps another argument");
}
bool same_rows(const Tensor& out, const Tensor& in) {
  return out.data_ptr() == in.data_ptr() && out.scalar_type() == in.scalar_type() && in.is_contiguous();
}

// x with channels next to each other, and an empty result of its shape that has them so: the strides are the
// same for real and for fake tensors.
Tensor rotary_input(const Tensor& x) {
  return x.sym_size(-1) > 1 && x.sym_stride(-1) != 1 ? x.contiguous() : x;
}
Tensor rotary_output(const Tensor& in) {
  Tensor out = at::empty_like(in);
  return out.sym_size(-1) > 1 && out.sym_stride(-1) != 1 ? at::empty_symint(in.sym_sizes(), in.options()) : out;
}

// The checks of shapes and types are the same for real and for fake tensors: sizes may be symbolic.
bool same_sizes(const Tensor& a, const Tensor& b, int64_t dims) {
  for (int64_t i = 0; i < dims; ++i)
    if (!a.sym_size(i).sym_eq(b.sym_size(i)).expect_true(__FILE__, __LINE__)) return false;
  return true;
}

void rotary_check(const Tensor& x, const Tensor& positions, const Tensor& inv_freq) {
  TORCH_CHECK(x.dim() == 3 || x.dim() == 4, "prunepath.rotary: x must be [N, heads, D] or [B, L, heads, D]");
  x_code(x, "rotary");
  TORCH_CHECK(positions.dim() == x.dim() - 2 && same_sizes(x, positions, x.dim() - 2),
              "prunepath.rotary: positions must have x's leading shape");
  TORCH_CHECK(positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt,
              "prunepath.rotary: positions must be int32 or int64");
  TORCH_CHECK(inv_freq.scalar_type() == at::kDouble && inv_freq.dim() == 1 && inv_freq.is_contiguous(),
              "prunepath.rotary: inv_freq must be contiguous float64 [rotary_dim / 2]");
  const c10::SymInt pairs = inv_freq.sym_size(0);
  TORCH_SYM_CHECK(pairs.sym_ge(1).sym_and((pairs * 2).sym_le(x.sym_size(-1))), "prunepath.rotary: ", pairs,
                  " pairs for heads of ", x.sym_size(-1), " channels");
}

// x [N, heads, D] or [B, L, heads, D] with positions of the leading shape. Strides go to the kernel;
// only channels that are not next to each other are copied first.
Tensor rotary_gpu(const Tensor& x, const Tensor& positions, const Tensor& inv_freq, c10::string_view layout,
                  double mscale, bool inverse) {
  const int lay = rotary_layout(layout, "rotary");
  rotary_check(x, positions, inv_freq);
  same_device("rotary", x, {&x, &positions, &inv_freq});
  const c10::DeviceGuard g(x.device());
  const Tensor in = rotary_input(x);
  Tensor out = rotary_output(in);
  const int64_t d = in.dim();
  const bool four = d == 4;
  const int64_t xs[3] = {four ? step(in, 0) : 0, step(in, d - 3), step(in, d - 2)};
  const int64_t ys[3] = {four ? step(out, 0) : 0, step(out, d - 3), step(out, d - 2)};
  const int64_t ps[2] = {four ? step(positions, 0) : 0, step(positions, d - 3)};
  check_rc(pp_rotary(in.data_ptr(), x_code(in, "rotary"), xs, positions.data_ptr(),
                     positions.scalar_type() == at::kLong, ps, four ? in.size(0) : 1, in.size(d - 3),
                     (int)in.size(d - 2), (int)in.size(d - 1), inv_freq.data_ptr<double>(), (int)(2 * inv_freq.numel()),
                     lay, (float)mscale, inverse, out.data_ptr(), ys, stream_of(in)),
           "rotary");
  return out;
}

Tensor rotary_meta(const Tensor& x, const Tensor& positions, const Tensor& inv_freq, c10::string_view layout, double, bool) {
  rotary_layout(layout, "rotary");
  rotary_check(x, positions, inv_freq);
  return rotary_output(rotary_input(x));
}

// The op's gradient in x is the op with the opposite angles, which has a gradient in its turn.
Tensor rotary_call(const Tensor& x, const Tensor& positions, const Tensor& inv_freq, c10::string_view layout,
                   double mscale, bool inverse) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("prunepath::rotary", "")
                       .typed<Tensor(const Tensor&, const Tensor&, const Tensor&, c10::string_view, double, bool)>();
  return op.call(x, positions, inv_freq, layout, mscale, inverse);
}

// A node of its own rather than an autograd::Function, whose context and outputs cost 3 us more a step.
struct RotaryBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable positions, inv_freq;
  std::string layout;
  double mscale = 1.0;
  bool inverse = false;
  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    if (!grads[0].defined()) return {Tensor()};
    Tensor p, f;
    {
      std::lock_guard<std::mutex> lock(mutex_);  // another thread's backward of the same graph may release them
      p = positions.unpack(), f = inv_freq.unpack();
    }
    return {rotary_call(grads[0], p, f, layout, mscale, !inverse)};
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    positions.reset_data();
    inv_freq.reset_data();
  }
  std::string name() const override { return "RotaryBackward"; }
};

Tensor rotary_autograd(const Tensor& x, const Tensor& positions, const Tensor& inv_freq, c10::string_view layout,
                       double mscale, bool inverse) {
  TORCH_CHECK(!c10::GradMode::is_enabled() || !inv_freq.requires_grad(),
              "prunepath.rotary: no gradient in inv_freq");
  TORCH_CHECK(!x._fw_grad(0).defined() && !inv_freq._fw_grad(0).defined(), "prunepath.rotary: no forward-mode gradient");
  std::shared_ptr<RotaryBackward> node;
  if (c10::GradMode::is_enabled() && x.requires_grad()) {
    node = std::shared_ptr<RotaryBackward>(new RotaryBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    node->positions = torch::autograd::SavedVariable(positions, false);
    node->inv_freq = torch::autograd::SavedVariable(inv_freq, false);
    node->layout = std::string(layout), node->mscale = mscale, node->inverse = inverse;
  }
  Tensor y;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    y = rotary_call(x, positions, inv_freq, layout, mscale, inverse);
  }
  if (node) torch::autograd::set_history(y, node);
  return y;
}

// ------------------------------------------------------------------ norms of queries and keys
// Query and key heads of the same tokens, [N, heads, D] or [B, L, heads, D].
void norm_check(const char* name, const Tensor& q, const Tensor& k, const Tensor& q_weight, const Tensor& k_weight,
                const Tensor& positions, const Tensor& inv_freq) {
  TORCH_CHECK((q.dim() == 3 || q.dim() == 4) && q.dim() == k.dim() && q.scalar_type() == k.scalar_type(), "prunepath.", name,
              ": q and k must be [N, heads, D] or [B, L, heads, D] of one dtype");
  x_code(q, name);
  TORCH_CHECK(same_sizes(q, k, q.dim() - 2), "prunepath.", name, ": q and k of different tokens");
  const c10::SymInt D = q.sym_size(-1);
  TORCH_SYM_CHECK(k.sym_size(-1).sym_eq(D), "prunepath.", name, ": query heads of ", D, " channels and key heads of ", k.sym_size(-1));
  TORCH_SYM_CHECK(D.sym_ge(2).sym_and(D.sym_le(256)), "prunepath.", name, ": head size ", D, " unsupported (2 to 256)");
  for (const Tensor* w : {&q_weight, &k_weight}) {
    TORCH_CHECK(w->dim() == 1 && (w->scalar_type() == at::kFloat || w->scalar_type() == q.scalar_type()) &&
                    w->scalar_type() == q_weight.scalar_type() && w->is_contiguous(),
                "prunepath.", name, ": weights must be contiguous [D], both float32 or both like q");
    TORCH_SYM_CHECK(w->sym_size(0).sym_eq(D), "prunepath.", name, ": ", w->sym_size(0), " weights for heads of ", D, " channels");
  }
  TORCH_CHECK(positions.dim() == q.dim() - 2 && same_sizes(q, positions, q.dim() - 2), "prunepath.", name,
              ": positions must have q's leading shape");
  TORCH_CHECK(positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt, "prunepath.", name,
              ": positions must be int32 or int64");
  TORCH_CHECK(inv_freq.scalar_type() == at::kDouble && inv_freq.dim() == 1 && inv_freq.is_contiguous(), "prunepath.", name,
              ": inv_freq must be contiguous float64 [rotary_dim / 2]");
  const c10::SymInt pairs = inv_freq.sym_size(0);
  TORCH_SYM_CHECK(pairs.sym_ge(1).sym_and((pairs * 2).sym_le(D)), "prunepath.", name, ": ", pairs, " pairs for heads of ", D, " channels");
}

// Strides of batch, token and head.
struct NormStrides {
  int64_t s[3];
  explicit NormStrides(const Tensor& t) : s{t.dim() == 4 ? step(t, 0) : 0, step(t, t.dim() - 3), step(t, t.dim() - 2)} {}
};

std::tuple<Tensor, Tensor> qk_norm_rotary_gpu(const Tensor& q, const Tensor& k, const Tensor& q_weight, const Tensor& k_weight,
                                              const Tensor& positions, const Tensor& inv_freq, c10::string_view layout,
                                              double mscale, double eps) {
  const char* const name = "qk_norm_rotary";
  const int lay = rotary_layout(layout, name);
  norm_check(name, q, k, q_weight, k_weight, positions, inv_freq);
  same_device(name, q, {&q, &k, &q_weight, &k_weight, &positions, &inv_freq});
  const c10::DeviceGuard g(q.device());
  const Tensor qi = rotary_input(q), ki = rotary_input(k);
  Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
  const int64_t d = q.dim();
  const NormStrides qs(qi), ks(ki);
  const int64_t ps[2] = {d == 4 ? step(positions, 0) : 0, step(positions, d - 3)};
  check_rc(pp_qk_norm_rotary(qi.data_ptr(), qs.s, ki.data_ptr(), ks.s, x_code(q, name), q_weight.data_ptr(), k_weight.data_ptr(),
                             w_code(q_weight, name), positions.data_ptr(), positions.scalar_type() == at::kLong, ps,
                             d == 4 ? q.size(0) : 1, q.size(d - 3), (int)q.size(d - 2), (int)k.size(d - 2), (int)q.size(d - 1),
                             inv_freq.data_ptr<double>(), (int)(2 * inv_freq.numel()), lay, (float)mscale, (float)eps,
                             qo.data_ptr(), ko.data_ptr(), stream_of(q)),
           name);
  return {qo, ko};
}

std::tuple<Tensor, Tensor> qk_norm_rotary_meta(const Tensor& q, const Tensor& k, const Tensor& q_weight, const Tensor& k_weight,
                                               const Tensor& positions, const Tensor& inv_freq, c10::string_view layout, double,
                                               double) {
  rotary_layout(layout, "qk_norm_rotary");
  norm_check("qk_norm_rotary", q, k, q_weight, k_weight, positions, inv_freq);
  return {at::empty_symint(q.sym_sizes(), q.options()), at::empty_symint(k.sym_sizes(), k.options())};
}

void norm_bwd_check(const Tensor& dq, const Tensor& dk, const Tensor& q, const Tensor& k, const Tensor& q_weight,
                    const Tensor& k_weight, const Tensor& positions, const Tensor& inv_freq) {
  const char* const name = "qk_norm_rotary_bwd";
  norm_check(name, q, k, q_weight, k_weight, positions, inv_freq);
  TORCH_CHECK(dq.dim() == q.dim() && dk.dim() == k.dim() && dq.scalar_type() == q.scalar_type() && dk.scalar_type() == k.scalar_type() &&
                  same_sizes(dq, q, q.dim()) && same_sizes(dk, k, k.dim()),
              "prunepath.qk_norm_rotary_bwd: dq and dk must be like q and k");
}

std::tuple<Tensor, Tensor, Tensor, Tensor> qk_norm_rotary_bwd_gpu(const Tensor& dq, const Tensor& dk, const Tensor& q,
                                                                  const Tensor& k, const Tensor& q_weight, const Tensor& k_weight,
                                                                  const Tensor& positions, const Tensor& inv_freq,
                                                                  c10::string_view layout, double mscale, double eps,
                                                                  bool weights) {
  const char* const name = "qk_norm_rotary_bwd";
  const int lay = rotary_layout(layout, name);
  norm_bwd_check(dq, dk, q, k, q_weight, k_weight, positions, inv_freq);
  same_device(name, q, {&dq, &dk, &q, &k, &q_weight, &k_weight, &positions, &inv_freq});
  const c10::DeviceGuard g(q.device());
  const Tensor qi = rotary_input(q), ki = rotary_input(k), dqi = rotary_input(dq), dki = rotary_input(dk);
  Tensor qg = at::empty(q.sizes(), q.options()), kg = at::empty(k.sizes(), k.options());
  Tensor wq = at::empty({weights ? q.size(-1) : 0}, q_weight.options()), wk = at::empty({weights ? q.size(-1) : 0}, k_weight.options());
  const int64_t d = q.dim(), B = d == 4 ? q.size(0) : 1, L = q.size(d - 3);
  const NormStrides qs(qi), ks(ki), dqs(dqi), dks(dki);
  const int64_t ps[2] = {d == 4 ? step(positions, 0) : 0, step(positions, d - 3)};
  const int rd = (int)(2 * inv_freq.numel());
  const size_t need = weights ? pp_qk_norm_rotary_workspace_bytes(x_code(q, name), B, L, (int)q.size(d - 2), (int)k.size(d - 2),
                                                                  (int)q.size(d - 1), rd)
                              : 0;
  Tensor ws;
  if (need) ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
  check_rc(pp_qk_norm_rotary_bwd(dqi.data_ptr(), dqs.s, dki.data_ptr(), dks.s, qi.data_ptr(), qs.s, ki.data_ptr(), ks.s,
                                 x_code(q, name), q_weight.data_ptr(), k_weight.data_ptr(), w_code(q_weight, name),
                                 positions.data_ptr(), positions.scalar_type() == at::kLong, ps, B, L, (int)q.size(d - 2),
                                 (int)k.size(d - 2), (int)q.size(d - 1), inv_freq.data_ptr<double>(), rd, lay, (float)mscale,
                                 (float)eps, qg.data_ptr(), kg.data_ptr(), weights ? wq.data_ptr() : nullptr,
                                 weights ? wk.data_ptr() : nullptr, need ? ws.data_ptr() : nullptr, need, stream_of(q)),
           name);
  return {qg, kg, wq, wk};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> qk_norm_rotary_bwd_meta(const Tensor& dq, const Tensor& dk, const Tensor& q,
                                                                   const Tensor& k, const Tensor& q_weight, const Tensor& k_weight,
                                                                   const Tensor& positions, const Tensor& inv_freq,
                                                                   c10::string_view layout, double, double, bool weights) {
  rotary_layout(layout, "qk_norm_rotary_bwd");
  norm_bwd_check(dq, dk, q, k, q_weight, k_weight, positions, inv_freq);
  const c10::SymInt n = weights ? q.sym_size(-1) : c10::SymInt(0);
  return {at::empty_symint(q.sym_sizes(), q.options()), at::empty_symint(k.sym_sizes(), k.options()),
          at::empty_symint({n}, q_weight.options()), at::empty_symint({n}, k_weight.options())};
}

std::tuple<Tensor, Tensor> qk_norm_rotary_call(const Tensor& q, const Tensor& k, const Tensor& q_weight, const Tensor& k_weight,
                                               const Tensor& positions, const Tensor& inv_freq, c10::string_view layout,
                                               double mscale, double eps) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("prunepath::qk_norm_rotary", "")
                       .typed<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                         const Tensor&, c10::string_view, double, double)>();
  return op.call(q, k, q_weight, k_weight, positions, inv_freq, layout, mscale, eps);
}
std::tuple<Tensor, Tensor, Tensor, Tensor> qk_norm_rotary_bwd_call(const Tensor& dq, const Tensor& dk, const Tensor& q,
                                                                   const Tensor& k, const Tensor& q_weight, const Tensor& k_weight,
                                                                   const Tensor& positions, const Tensor& inv_freq,
                                                                   c10::string_view layout, double mscale, double eps,
                                                                   bool weights) {
  static auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("prunepath::qk_norm_rotary_bwd", "")
          .typed<std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                            const Tensor&, const Tensor&, const Tensor&, c10::string_view, double,
                                                            double, bool)>();
  return op.call(dq, dk, q, k, q_weight, k_weight, positions, inv_freq, layout, mscale, eps, weights);
}

struct QkNormBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable saved[6];  // q, k, their weights, positions, inv_freq
  std::string layout;
  double mscale = 1.0, eps = 0.0;
  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    const bool has_q = grads[0].defined(), has_k = grads[1].defined();
    if (!has_q && !has_k) return {Tensor(), Tensor(), Tensor(), Tensor()};
    Tensor t[6];
    {
      std::lock_guard<std::mutex> lock(mutex_);  // another thread's backward of the same graph may release them
      for (int i = 0; i < 6; ++i) t[i] = saved[i].unpack();
    }
    // what has no gradient takes part with no heads
    for (int i = 0; i < 2; ++i)
      if (!grads[i].defined()) {
        t[i] = t[i].narrow(-2, 0, 0);
        grads[i] = at::empty_symint(t[i].sym_sizes(), t[i].options());
      }
    const bool weights = task_should_compute_output(2) || task_should_compute_output(3);
    auto [dq, dk, wq, wk] = qk_norm_rotary_bwd_call(grads[0], grads[1], t[0], t[1], t[2], t[3], t[4], t[5], layout, mscale, eps, weights);
    auto asked = [&](int i, bool has, const Tensor& x) { return has && task_should_compute_output(i) ? x : Tensor(); };
    return {asked(0, has_q, dq), asked(1, has_k, dk), asked(2, has_q, wq), asked(3, has_k, wk)};
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto& s : saved) s.reset_data();
  }
  std::string name() const override { return "QkNormRotaryBackward"; }
};

std::tuple<Tensor, Tensor> qk_norm_rotary_autograd(const Tensor& q, const Tensor& k, const Tensor& q_weight, const Tensor& k_weight,
                                                   const Tensor& positions, const Tensor& inv_freq, c10::string_view layout,
                                                   double mscale, double eps) {
  const Tensor* const in[6] = {&q, &k, &q_weight, &k_weight, &positions, &inv_freq};
  const bool grad = c10::GradMode::is_enabled();
  TORCH_CHECK(!grad || !inv_freq.requires_grad(), "prunepath.qk_norm_rotary: no gradient in inv_freq");
  for (const Tensor* t : in) TORCH_CHECK(!t->_fw_grad(0).defined(), "prunepath.qk_norm_rotary: no forward-mode gradient");
  std::shared_ptr<QkNormBackward> node;
  if (grad && (q.requires_grad() || k.requires_grad() || q_weight.requires_grad() || k_weight.requires_grad())) {
    node = std::shared_ptr<QkNormBackward>(new QkNormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(q, k, q_weight, k_weight));
    for (int i = 0; i < 6; ++i) node->saved[i] = torch::autograd::SavedVariable(*in[i], false);
    node->layout = std::string(layout), node->mscale = mscale, node->eps = eps;
  }
  std::tuple<Tensor, Tensor> y;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    y = qk_norm_rotary_call(q, k, q_weight, k_weight, positions, inv_freq, layout, mscale, eps);
  }
  if (node) {
    torch::autograd::set_history(std::get<0>(y), node);
    torch::autograd::set_history(std::get<1>(y), node);
  }
  return y;
}

// ------------------------------------------------------------------ paged cache
// Heads, D and the cache of a call: shapes, types and what the kernels take of them.
void paged_check(const char* name, const Tensor& k_pages, const Tensor& v_pages, const optional<Tensor>& k_scales,
                 const optional<Tensor>& v_scales, const Tensor& block_table, const Tensor& kv_lens, const Tensor& cu_q,
                 const c10::SymInt& Hq, const c10::SymInt& D) {
  TORCH_CHECK(k_scales.has_value() == v_scales.has_value(), "prunepath.", name, ": scales of keys and of values belong together");
  if (k_scales) {
    TORCH_CHECK(k_pages.dim() == 4 && v_pages.dim() == 5 && k_pages.scalar_type() == at::kFloat8_e4m3fn &&
                    v_pages.scalar_type() == at::kFloat8_e4m3fn,
                "prunepath.", name, ": with scales k_pages [pages, kv_heads, page, D] and v_pages [pages, kv_heads, page / 16, D, 16] "
                "float8_e4m3fn required");
    TORCH_CHECK(k_scales->dim() == 3 && v_scales->dim() == 3 && k_scales->scalar_type() == at::kFloat8_e8m0fnu &&
                    v_scales->scalar_type() == at::kFloat8_e8m0fnu,
                "prunepath.", name, ": scales must be float8_e8m0fnu [pages, kv_heads, page / 16]");
    const c10::SymInt blocks = v_pages.sym_size(2);
    TORCH_SYM_CHECK(k_pages.sym_size(3).sym_eq(D).sym_and(v_pages.sym_size(3).sym_eq(D)).sym_and(v_pages.sym_size(4).sym_eq(16))
                        .sym_and(k_pages.sym_size(2).sym_eq(blocks * 16)).sym_and(v_pages.sym_size(0).sym_eq(k_pages.sym_size(0)))
                        .sym_and(v_pages.sym_size(1).sym_eq(k_pages.sym_size(1))),
                    "prunepath.", name, ": shapes of k_pages ", k_pages.sym_sizes(), ", v_pages ", v_pages.sym_sizes(),
                    " and head size ", D, " disagree");
    for (const Tensor* s : {&*k_scales, &*v_scales})
      TORCH_SYM_CHECK(s->sym_size(0).sym_eq(k_pages.sym_size(0)).sym_and(s->sym_size(1).sym_eq(k_pages.sym_size(1)))
                          .sym_and(s->sym_size(2).sym_eq(blocks)),
                      "prunepath.", name, ": scales ", s->sym_sizes(), " for pages ", k_pages.sym_sizes());
  } else {
    TORCH_CHECK(k_pages.dim() == 4 && v_pages.dim() == 4 && k_pages.scalar_type() == at::kBFloat16 &&
                    v_pages.scalar_type() == at::kBFloat16,
                "prunepath.", name, ": k_pages [pages, kv_heads, page, D] and v_pages [pages, kv_heads, D, page] bfloat16 required");
  }
  if (!k_scales) TORCH_SYM_CHECK(k_pages.sym_size(3).sym_eq(D).sym_and(v_pages.sym_size(2).sym_eq(D))
                      .sym_and(v_pages.sym_size(0).sym_eq(k_pages.sym_size(0)))
                      .sym_and(v_pages.sym_size(1).sym_eq(k_pages.sym_size(1)))
                      .sym_and(v_pages.sym_size(3).sym_eq(k_pages.sym_size(2))),
                  "prunepath.", name, ": shapes of k_pages ", k_pages.sym_sizes(), ", v_pages ", v_pages.sym_sizes(),
                  " and head size ", D, " disagree");
  TORCH_CHECK(block_table.dim() == 2 && block_table.scalar_type() == at::kInt && kv_lens.dim() == 1 &&
                  kv_lens.scalar_type() == at::kInt && cu_q.dim() == 1 && cu_q.scalar_type() == at::kInt,
              "prunepath.", name, ": block_table [seqs, max_pages], kv_lens [seqs] and cu_q [seqs + 1] must be int32");
  for (const Tensor* t : {&k_pages, &v_pages, &block_table, &kv_lens, &cu_q, k_scales ? &*k_scales : &k_pages, v_scales ? &*v_scales : &v_pages})
    TORCH_CHECK(t->is_contiguous(), "prunepath.", name, ": the cache, its scales, block_table, kv_lens and cu_q must be contiguous");
  const c10::SymInt seqs = kv_lens.sym_size(0), Hkv = k_pages.sym_size(1);
  TORCH_SYM_CHECK(block_table.sym_size(0).sym_eq(seqs).sym_and(cu_q.sym_size(0).sym_eq(seqs + 1)), "prunepath.", name,
                  ": block_table ", block_table.sym_sizes(), ", kv_lens ", kv_lens.sym_sizes(), " and cu_q ",
                  cu_q.sym_sizes(), " disagree");
  TORCH_SYM_CHECK(Hkv.sym_ge(1), "prunepath.", name, ": a cache of no heads");
  TORCH_SYM_CHECK((Hq % Hkv).sym_eq(0), "prunepath.", name, ": ", Hq, " query heads on ", Hkv,
                  " key heads (need a multiple)");
  TORCH_SYM_CHECK(D.sym_eq(64).sym_or(D.sym_eq(128)), "prunepath.", name, ": head size ", D, " unsupported (64 or 128)");
}

struct Paged {
  int64_t n, seqs, Hq, Hkv, D, pages, max_pages, page;
};

Paged paged_sizes(const char* name, const Tensor& k_pages, const Tensor& block_table, int64_t n, int64_t Hq) {
  Paged p;
  p.n = n, p.Hq = Hq, p.D = k_pages.size(3);
  p.pages = k_pages.size(0), p.Hkv = k_pages.size(1), p.page = k_pages.size(2);
  p.seqs = block_table.size(0), p.max_pages = block_table.size(1);
  TORCH_CHECK(p.pages <= 0x7fffffff && p.max_pages <= 0x7fffffff && p.page <= 0x7fffffff && p.Hkv <= 0x7fffffff &&
                  p.seqs <= 0x7fffffff && Hq <= 0x7fffffff,
              "prunepath.", name, ": a size beyond 2^31");
  return p;
}

// q and q_out: a tensor or nullptr
void kv_append_check(const Tensor* q, const Tensor* q_out, const Tensor& k, const Tensor& v, const Tensor& k_pages,
                     const Tensor& v_pages, const Tensor& block_table, const Tensor& kv_lens, const Tensor& cu_q,
                     const optional<Tensor>& inv_freq, const optional<Tensor>& q_weight, const optional<Tensor>& k_weight,
                     const optional<Tensor>& k_scales, const optional<Tensor>& v_scales) {
  const char* const name = "kv_append";
  x_code(k, name);
  TORCH_CHECK(k.dim() == 3 && v.dim() == 3 && k.scalar_type() == v.scalar_type() && same_sizes(k, v, 3),
              "prunepath.kv_append: k and v must be [N, kv_heads, D] of one dtype");
  if (q)
    TORCH_CHECK(q->dim() == 3 && q->scalar_type() == k.scalar_type() &&
                    q->sym_size(0).sym_eq(k.sym_size(0)).sym_and(q->sym_size(2).sym_eq(k.sym_size(2)))
                        .sym_and(q->sym_stride(2).sym_eq(1)).expect_true(__FILE__, __LINE__),
                "prunepath.kv_append: q must be [N, heads, D] of k's dtype, channels contiguous");
  paged_check(name, k_pages, v_pages, k_scales, v_scales, block_table, kv_lens, cu_q, q ? q->sym_size(1) : c10::SymInt(0), k.sym_size(2));
  TORCH_CHECK(q ? q_weight.has_value() == k_weight.has_value() : !q_weight.has_value(),
              "prunepath.kv_append: norms of queries and of keys belong together");
  for (const optional<Tensor>* w : {&q_weight, &k_weight})
    if (*w) {
      TORCH_CHECK((*w)->dim() == 1 && ((*w)->scalar_type() == at::kFloat || (*w)->scalar_type() == k.scalar_type()) &&
                      (*w)->scalar_type() == (*k_weight).scalar_type() && (*w)->is_contiguous(),
                  "prunepath.kv_append: weights must be contiguous [D], both float32 or both like k");
      TORCH_SYM_CHECK((*w)->sym_size(0).sym_eq(k.sym_size(2)), "prunepath.kv_append: ", (*w)->sym_size(0), " weights for heads of ",
                      k.sym_size(2), " channels");
    }
  TORCH_SYM_CHECK(k.sym_size(1).sym_eq(k_pages.sym_size(1)), "prunepath.kv_append: ", k.sym_size(1),
                  " heads for a cache of ", k_pages.sym_size(1));
  TORCH_SYM_CHECK(k.sym_stride(2).sym_eq(1).sym_and(v.sym_stride(2).sym_eq(1)),
                  "prunepath.kv_append: channels must be contiguous");
  if (inv_freq) {
    TORCH_CHECK(inv_freq->scalar_type() == at::kDouble && inv_freq->dim() == 1 && inv_freq->is_contiguous(),
                "prunepath.kv_append: inv_freq must be contiguous float64 [rotary_dim / 2]");
    const c10::SymInt rd = inv_freq->sym_size(0) * 2;
    TORCH_SYM_CHECK(rd.sym_le(k.sym_size(2)).sym_and((rd % 16).sym_eq(0)), "prunepath.kv_append: rotary_dim ", rd,
                    " unsupported (a multiple of 16 up to the head size ", k.sym_size(2), ")");
  }
  if (q_out)
    TORCH_CHECK(q_out->scalar_type() == at::kBFloat16 && q_out->dim() == 3 && same_sizes(*q_out, *q, 3) &&
                    q_out->is_contiguous(),
                "prunepath.kv_append: q_out must be contiguous bfloat16 of q's shape");
}

void kv_append_into(const optional<Tensor>& q, const optional<Tensor>& q_out, bool zero_tail, const Tensor& k,
                    const Tensor& v, const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table,
                    const Tensor& kv_lens, const Tensor& cu_q, const optional<Tensor>& inv_freq,
                    c10::string_view layout, double mscale, const optional<Tensor>& q_weight,
                    const optional<Tensor>& k_weight, double eps, const optional<Tensor>& k_scales,
                    const optional<Tensor>& v_scales) {
  const char* const name = "kv_append";
  const int lay = rotary_layout(layout, name);
  kv_append_check(q ? &*q : nullptr, q ? &*q_out : nullptr, k, v, k_pages, v_pages, block_table, kv_lens, cu_q, inv_freq, q_weight,
                  k_weight, k_scales, v_scales);
  auto given = [](const optional<Tensor>& t) { return t ? &*t : nullptr; };
  // (a row of weights inside another tensor may start anywhere)
  auto row = [](const optional<Tensor>& t) { return t && ((uintptr_t)t->data_ptr() & 15) ? optional<Tensor>(t->clone()) : t; };
  const Paged p = paged_sizes(name, k_pages, block_table, k.size(0), q ? q->size(1) : 0);
  need_gpu(name, k, {&k_pages, &v_pages, &block_table, &kv_lens, &cu_q, given(inv_freq), given(q_weight), given(k_weight),
                     given(k_scales), given(v_scales)});
  same_device(name, k, {&k, &v});
  const Span sk(k), sv(v), kp(k_pages), vp(v_pages), st(block_table), sl(kv_lens), sc(cu_q);
  auto span = [&](const optional<Tensor>& t) { return t ? Span(*t) : st; };
  const Span sf = span(inv_freq), sqw = span(q_weight), skw = span(k_weight);
  const Span* const reads[] = {&sk, &sv, &st, &sl, &sc, &sf, &sqw, &skw};
  for (const Span* in : reads) {
    apart(name, kp, *in);
    apart(name, vp, *in);
  }
  apart(name, kp, vp);
  const Span ks8 = k_scales ? Span(*k_scales) : kp, vs8 = v_scales ? Span(*v_scales) : vp;
  if (k_scales) {
    for (const Span* in : reads) {
      apart(name, ks8, *in);
      apart(name, vs8, *in);
    }
    for (const Span* pages : {&kp, &vp}) {
      apart(name, ks8, *pages);
      apart(name, vs8, *pages);
    }
    apart(name, ks8, vs8);
  }
  int64_t qs[2] = {0, 0};
  if (q) {
    same_device(name, k, {&*q, &*q_out});
    const Span sq(*q);
    for (const Span* out : {&kp, &vp, &ks8, &vs8}) apart(name, *out, sq);
    if (!zero_tail) {  // a given q_out
      const Span so(*q_out);
      for (const Span* out : {&kp, &vp, &ks8, &vs8}) apart(name, so, *out);
      for (const Span* in : reads) apart(name, so, *in);
      if (!same_rows(*q_out, *q)) apart(name, so, sq);
    }
    qs[0] = step(*q, 0), qs[1] = step(*q, 1);
  }
  const c10::DeviceGuard g(k.device());
  const int64_t ks[2] = {step(k, 0), step(k, 1)}, vs[2] = {step(v, 0), step(v, 1)};
  const optional<Tensor> qw = row(q_weight), kw = row(k_weight);
  check_rc(pp_kv_append_with(q ? q->data_ptr() : nullptr, qs, k.data_ptr(), ks, v.data_ptr(), vs, x_code(k, name), p.n,
                             (int)p.seqs, cu_q.data_ptr<int32_t>(), kv_lens.data_ptr<int32_t>(),
                             block_table.data_ptr<int32_t>(), (int)p.max_pages, (int)p.pages, (int)p.page, (int)p.Hq,
                             (int)p.Hkv, (int)p.D, (const double*)ptr(inv_freq), inv_freq ? (int)(2 * inv_freq->numel()) : 0,
                             lay, (float)mscale, ptr(qw), ptr(kw), kw ? w_code(*kw, name) : 0, (float)eps,
                             k_pages.data_ptr(), v_pages.data_ptr(), (void*)ptr(k_scales), (void*)ptr(v_scales),
                             q ? q_out->data_ptr() : nullptr, zero_tail, stream_of(k)),
           name);
}

void kv_append_gpu(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages,
                   const Tensor& block_table, const Tensor& kv_lens, const Tensor& cu_q,
                   const optional<Tensor>& inv_freq, c10::string_view layout, double mscale, const optional<Tensor>& k_weight, double eps,
                   const optional<Tensor>& k_scales, const optional<Tensor>& v_scales) {
  kv_append_into(c10::nullopt, c10::nullopt, false, k, v, k_pages, v_pages, block_table, kv_lens, cu_q, inv_freq,
                 layout, mscale, c10::nullopt, k_weight, eps, k_scales, v_scales);
}

Tensor kv_append_q_gpu(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages,
                       const Tensor& block_table, const Tensor& kv_lens, const Tensor& cu_q,
                       const optional<Tensor>& inv_freq, c10::string_view layout, double mscale, const optional<Tensor>& q_weight,
                       const optional<Tensor>& k_weight, double eps, const optional<Tensor>& k_scales, const optional<Tensor>& v_scales) {
  Tensor out = at::empty(q.sizes(), q.options().dtype(at::kBFloat16));
  kv_append_into(q, out, true, k, v, k_pages, v_pages, block_table, kv_lens, cu_q, inv_freq, layout, mscale, q_weight, k_weight, eps,
                 k_scales, v_scales);
  return out;
}

void kv_append_q_into_gpu(const Tensor& q, const Tensor& q_out, const Tensor& k, const Tensor& v, const Tensor& k_pages,
                          const Tensor& v_pages, const Tensor& block_table, const Tensor& kv_lens, const Tensor& cu_q,
                          const optional<Tensor>& inv_freq, c10::string_view layout, double mscale, const optional<Tensor>& q_weight,
                          const optional<Tensor>& k_weight, double eps, const optional<Tensor>& k_scales, const optional<Tensor>& v_scales) {
  kv_append_into(q, q_out, false, k, v, k_pages, v_pages, block_table, kv_lens, cu_q, inv_freq, layout, mscale, q_weight, k_weight,
                 eps, k_scales, v_scales);
}

void kv_append_meta(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages,
                    const Tensor& block_table, const Tensor& kv_lens, const Tensor& cu_q,
                    const optional<Tensor>& inv_freq, c10::string_view layout, double, const optional<Tensor>& k_weight, double,
                    const optional<Tensor>& k_scales, const optional<Tensor>& v_scales) {
  rotary_layout(layout, "kv_append");
  kv_append_check(nullptr, nullptr, k, v, k_pages, v_pages, block_table, kv_lens, cu_q, inv_freq, c10::nullopt, k_weight, k_scales,
                  v_scales);
}
Tensor kv_append_q_meta(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages,
                        const Tensor& block_table, const Tensor& kv_lens, const Tensor& cu_q,
                        const optional<Tensor>& inv_freq, c10::string_view layout, double, const optional<Tensor>& q_weight,
                        const optional<Tensor>& k_weight, double, const optional<Tensor>& k_scales, const optional<Tensor>& v_scales) {
  rotary_layout(layout, "kv_append");
  kv_append_check(&q, nullptr, k, v, k_pages, v_pages, block_table, kv_lens, cu_q, inv_freq, q_weight, k_weight, k_scales, v_scales);
  return at::empty_symint(q.sym_sizes(), q.options().dtype(at::kBFloat16));
}
void kv_append_q_into_meta(const Tensor& q, const Tensor& q_out, const Tensor& k, const Tensor& v, const Tensor& k_pages,
                           const Tensor& v_pages, const Tensor& block_table, const Tensor& kv_lens, const Tensor& cu_q,
                           const optional<Tensor>& inv_freq, c10::string_view layout, double, const optional<Tensor>& q_weight,
                           const optional<Tensor>& k_weight, double, const optional<Tensor>& k_scales, const optional<Tensor>& v_scales) {
  rotary_layout(layout, "kv_append");
  kv_append_check(&q, &q_out, k, v, k_pages, v_pages, block_table, kv_lens, cu_q, inv_freq, q_weight, k_weight, k_scales, v_scales);
}

// ------------------------------------------------------------------ read
void read_check(const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table, const Tensor& kv_lens, const Tensor& cu_q,
                const c10::SymInt& rows, const optional<Tensor>& k_scales, const optional<Tensor>& v_scales) {
  TORCH_CHECK(k_pages.dim() == 4, "prunepath.kv_read: k_pages must be [pages, kv_heads, page, D]");
  paged_check("kv_read", k_pages, v_pages, k_scales, v_scales, block_table, kv_lens, cu_q, c10::SymInt(0), k_pages.sym_size(3));
  TORCH_SYM_CHECK(rows.sym_ge(0), "prunepath.kv_read: ", rows, " rows");
}
void read_check_out(const Tensor& k_pages, const Tensor& k_out, const Tensor& v_out) {
  for (const Tensor* t : {&k_out, &v_out}) {
    TORCH_CHECK(t->dim() == 3 && t->scalar_type() == at::kBFloat16 && t->is_contiguous(),
                "prunepath.kv_read: results must be contiguous bfloat16 [rows, kv_heads, D]");
    TORCH_SYM_CHECK(t->sym_size(0).sym_eq(k_out.sym_size(0)).sym_and(t->sym_size(1).sym_eq(k_pages.sym_size(1)))
                        .sym_and(t->sym_size(2).sym_eq(k_pages.sym_size(3))),
                    "prunepath.kv_read: results ", t->sym_sizes(), " for pages ", k_pages.sym_sizes());
  }
}

void read_into(const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table, const Tensor& kv_lens, const Tensor& cu_q,
               const Tensor& k_out, const Tensor& v_out, const optional<Tensor>& k_scales, const optional<Tensor>& v_scales,
               bool zero_tail) {
  const char* const name = "kv_read";
  const Paged p = paged_sizes(name, k_pages, block_table, k_out.size(0), 0);
  need_gpu(name, k_pages, {&k_pages, &v_pages, &block_table, &kv_lens, &cu_q, &k_out, &v_out, k_scales ? &*k_scales : nullptr,
                           v_scales ? &*v_scales : nullptr});
  if (!zero_tail) {  // given results
    const Span ko(k_out), vo(v_out);
    apart(name, ko, vo);
    for (const Tensor* in : {&k_pages, &v_pages, &block_table, &kv_lens, &cu_q, k_scales ? &*k_scales : &k_pages,
                             v_scales ? &*v_scales : &v_pages}) {
      apart(name, ko, Span(*in));
      apart(name, vo, Span(*in));
    }
  }
  const c10::DeviceGuard g(k_pages.device());
  check_rc(pp_kv_read(k_pages.data_ptr(), v_pages.data_ptr(), ptr(k_scales), ptr(v_scales), p.n, (int)p.seqs,
                      cu_q.data_ptr<int32_t>(), kv_lens.data_ptr<int32_t>(), block_table.data_ptr<int32_t>(), (int)p.max_pages,
                      (int)p.pages, (int)p.page, (int)p.Hkv, (int)p.D, k_out.data_ptr(), v_out.data_ptr(), zero_tail,
                      stream_of(k_pages)),
           name);
}

std::tuple<Tensor, Tensor> kv_read_gpu(const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table,
                                       const Tensor& kv_lens, const Tensor& cu_q, c10::SymInt rows,
                                       const optional<Tensor>& k_scales, const optional<Tensor>& v_scales) {
  read_check(k_pages, v_pages, block_table, kv_lens, cu_q, rows, k_scales, v_scales);
  const int64_t n = rows.guard_int(__FILE__, __LINE__);
  auto bf = k_pages.options().dtype(at::kBFloat16);
  Tensor k = at::empty({n, k_pages.size(1), k_pages.size(3)}, bf), v = at::empty_like(k);
  read_into(k_pages, v_pages, block_table, kv_lens, cu_q, k, v, k_scales, v_scales, true);
  return {k, v};
}
void kv_read_into_gpu(const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table, const Tensor& kv_lens,
                      const Tensor& cu_q, const Tensor& k_out, const Tensor& v_out, const optional<Tensor>& k_scales,
                      const optional<Tensor>& v_scales) {
  read_check(k_pages, v_pages, block_table, kv_lens, cu_q, 0, k_scales, v_scales);
  read_check_out(k_pages, k_out, v_out);
  read_into(k_pages, v_pages, block_table, kv_lens, cu_q, k_out, v_out, k_scales, v_scales, false);
}
std::tuple<Tensor, Tensor> kv_read_meta(const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table,
                                        const Tensor& kv_lens, const Tensor& cu_q, c10::SymInt rows,
                                        const optional<Tensor>& k_scales, const optional<Tensor>& v_scales) {
  read_check(k_pages, v_pages, block_table, kv_lens, cu_q, rows, k_scales, v_scales);
  auto bf = k_pages.options().dtype(at::kBFloat16);
  const std::vector<c10::SymInt> shape = {rows, k_pages.sym_size(1), k_pages.sym_size(3)};
  return {at::empty_symint(shape, bf), at::empty_symint(shape, bf)};
}
void kv_read_into_meta(const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table, const Tensor& kv_lens,
                       const Tensor& cu_q, const Tensor& k_out, const Tensor& v_out, const optional<Tensor>& k_scales,
                       const optional<Tensor>& v_scales) {
  read_check(k_pages, v_pages, block_table, kv_lens, cu_q, 0, k_scales, v_scales);
  read_check_out(k_pages, k_out, v_out);
}

// out: a tensor or nullptr
void attention_check(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table,
                     const Tensor& kv_lens, const Tensor& cu_q, const optional<Tensor>& k_scales, const optional<Tensor>& v_scales,
                     int64_t window, int64_t sinks, const Tensor* out) {
  TORCH_CHECK(q.dim() == 3 && q.scalar_type() == at::kBFloat16 && q.sym_stride(2).sym_eq(1).expect_true(__FILE__, __LINE__),
              "prunepath.paged_attention: q must be bfloat16 [N, heads, D], channels contiguous");
  if (out)
    TORCH_CHECK(out->scalar_type() == at::kBFloat16 && out->dim() == 3 && same_sizes(*out, q, 3) && out->is_contiguous(),
                "prunepath.paged_attention: out must be contiguous bfloat16 of q's shape");
  TORCH_CHECK(window >= 0 && sinks >= 0 && (window > 0 || sinks == 0), "prunepath.paged_attention: a window of ", window, " tokens and ",
              sinks, " first ones (a window of at least 1, and first tokens only beside one; 0 and 0: none)");
  paged_check("paged_attention", k_pages, v_pages, k_scales, v_scales, block_table, kv_lens, cu_q, q.sym_size(1), q.sym_size(2));
}

void attention_into(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table,
                    const Tensor& kv_lens, const Tensor& cu_q, double scale, const Tensor& out, bool zero_tail,
                    const optional<Tensor>& k_scales, const optional<Tensor>& v_scales, int64_t window, int64_t sinks) {
  const char* const name = "paged_attention";
  attention_check(q, k_pages, v_pages, block_table, kv_lens, cu_q, k_scales, v_scales, window, sinks, &out);
  const Paged p = paged_sizes(name, k_pages, block_table, q.size(0), q.size(1));
  need_gpu(name, q, {&k_pages, &v_pages, &block_table, &kv_lens, &cu_q, &out, k_scales ? &*k_scales : nullptr,
                     v_scales ? &*v_scales : nullptr});
  same_device(name, q, {&q});
  if (!zero_tail) {  // a given out
    const Span so(out);
    for (const Tensor* in : {&k_pages, &v_pages, &block_table, &kv_lens, &cu_q, k_scales ? &*k_scales : &k_pages,
                             v_scales ? &*v_scales : &v_pages})
      apart(name, so, Span(*in));
    if (!same_rows(out, q)) apart(name, so, Span(q));
  }
  const c10::DeviceGuard g(q.device());
  const size_t need = pp_paged_attention_with_workspace_bytes(p.n, (int)p.seqs, (int)p.max_pages, (int)p.page, (int)p.Hq,
                                                              (int)p.Hkv, (int)p.D, k_scales.has_value(), window, sinks);
  Tensor ws;
  if (need) ws = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
  const int64_t qs[2] = {step(q, 0), step(q, 1)};
  check_rc(pp_paged_attention_with(q.data_ptr(), qs, p.n, (int)p.seqs, cu_q.data_ptr<int32_t>(), kv_lens.data_ptr<int32_t>(),
                                   block_table.data_ptr<int32_t>(), (int)p.max_pages, k_pages.data_ptr(), v_pages.data_ptr(),
                                   ptr(k_scales), ptr(v_scales), (int)p.pages, (int)p.page, (int)p.Hq, (int)p.Hkv, (int)p.D,
                                   (float)scale, window, sinks, out.data_ptr(), zero_tail, need ? ws.data_ptr() : nullptr, need,
                                   stream_of(q)),
           name);
}

void paged_attention_into_gpu(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table,
                              const Tensor& kv_lens, const Tensor& cu_q, double scale, const Tensor& out, const optional<Tensor>& k_scales,
                              const optional<Tensor>& v_scales, int64_t window, int64_t sinks) {
  attention_into(q, k_pages, v_pages, block_table, kv_lens, cu_q, scale, out, false, k_scales, v_scales, window, sinks);
}

Tensor paged_attention_gpu(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table,
                           const Tensor& kv_lens, const Tensor& cu_q, double scale, const optional<Tensor>& k_scales,
                           const optional<Tensor>& v_scales, int64_t window, int64_t sinks) {
  Tensor out = at::empty(q.sizes(), q.options());
  attention_into(q, k_pages, v_pages, block_table, kv_lens, cu_q, scale, out, true, k_scales, v_scales, window, sinks);
  return out;
}

Tensor paged_attention_meta(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table,
                            const Tensor& kv_lens, const Tensor& cu_q, double, const optional<Tensor>& k_scales,
                            const optional<Tensor>& v_scales, int64_t window, int64_t sinks) {
  attention_check(q, k_pages, v_pages, block_table, kv_lens, cu_q, k_scales, v_scales, window, sinks, nullptr);
  return at::empty_symint(q.sym_sizes(), q.options());
}
void paged_attention_into_meta(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& block_table,
                               const Tensor& kv_lens, const Tensor& cu_q, double, const Tensor& out, const optional<Tensor>& k_scales,
                               const optional<Tensor>& v_scales, int64_t window, int64_t sinks) {
  attention_check(q, k_pages, v_pages, block_table, kv_lens, cu_q, k_scales, v_scales, window, sinks, &out);
}

// ------------------------------------------------------------------ ops for inference
void refuse_gradient(const char* op, const Tensor& t) {
  TORCH_CHECK(!t._fw_grad(0).defined(), "prunepath.", op, ": no forward-mode gradient");
  TORCH_CHECK(!c10::GradMode::is_enabled() || !t.requires_grad(), "prunepath.", op,
              ": inference only, but an argument requires a gradient (call it under torch.no_grad())");
}
void refuse_gradient(const char* op, const optional<Tensor>& t) {
  if (t && t->defined()) refuse_gradient(op, *t);
}
template <typename T>
void refuse_gradient(const char*, const T&) {}

// The kernel of an op's Autograd key: a call that would need a gradient, or has a tangent, is refused, any
// other goes on to the key below. It stands there, not in the GPU's kernel, so that traced calls meet it too:
// under the tracer the GPU's kernel only ever runs with gradients off.
template <typename Op, typename R, typename... A>
struct Inference {
  static R call(c10::DispatchKeySet keys, A... args) {
    (refuse_gradient(Op::name(), args), ...);
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow((std::string("prunepath::") + Op::name()).c_str(), "")
                         .template typed<R(A...)>();
    return op.redispatch(keys & c10::after_autograd_keyset, args...);
  }
};
template <typename Op, typename R, typename... A>
constexpr auto inference(R (*)(A...)) {
  return &Inference<Op, R, A...>::call;
}
// The kernel of an op's ADInplaceOrView key: what the op has written (its arguments of the given numbers)
// counts as changed, so that a backward that saved it before raises, as after torch's own operations in place.
void changed(const Tensor& t) {
  if (t.defined() && !t.is_inference()) torch::autograd::impl::bump_version(t);
}
void changed(const optional<Tensor>& t) {
  if (t) changed(*t);
}
template <typename T>
void changed(const T&) {}

template <typename Op, unsigned numbers, typename R, typename... A>
struct Written {
  static R call(c10::DispatchKeySet keys, A... args) {
    static auto op = c10::Dispatcher::singleton()
                         .findSchemaOrThrow((std::string("prunepath::") + Op::name()).c_str(), "")
                         .template typed<R(A...)>();
    const auto count = [&] {
      unsigned i = 0;
      ((numbers >> i++ & 1 ? changed(args) : void()), ...);
    };
    if constexpr (std::is_void_v<R>) {
      op.redispatch(keys & c10::after_ADInplaceOrView_keyset, args...);
      count();
    } else {
      R out = op.redispatch(keys & c10::after_ADInplaceOrView_keyset, args...);
      count();
      return out;
    }
  }
};
template <typename Op, unsigned numbers, typename R, typename... A>
constexpr auto written(R (*)(A...)) {
  return &Written<Op, numbers, R, A...>::call;
}

// The gradient of qk_norm_rotary has none of its own.
std::tuple<Tensor, Tensor, Tensor, Tensor> qk_norm_rotary_bwd_autograd(const Tensor& dq, const Tensor& dk,
                                                                       const Tensor& q, const Tensor& k, const Tensor& q_weight,
                                                                       const Tensor& k_weight, const Tensor& positions,
                                                                       const Tensor& inv_freq, c10::string_view layout,
                                                                       double mscale, double eps, bool weights) {
  for (const Tensor* t : {&dq, &dk, &q, &k, &q_weight, &k_weight, &inv_freq}) {
    TORCH_CHECK(!t->_fw_grad(0).defined(), "prunepath.qk_norm_rotary_bwd: no forward-mode gradient");
    TORCH_CHECK(!c10::GradMode::is_enabled() || !t->requires_grad(), "prunepath.qk_norm_rotary: no second derivative");
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return qk_norm_rotary_bwd_call(dq, dk, q, k, q_weight, k_weight, positions, inv_freq, layout, mscale, eps, weights);
}

#define INFERENCE(m, op)                        \
  do {                                          \
    struct Op {                                 \
      static const char* name() { return #op; } \
    };                                          \
    m.impl(#op, inference<Op>(&op##_gpu));      \
  } while (0)
#define WRITES(m, op, fn, numbers)              \
  do {                                          \
    struct Op {                                 \
      static const char* name() { return #op; } \
    };                                          \
    m.impl(#op, written<Op, numbers>(&fn));     \
  } while (0)

void refuse_cpu(const c10::OperatorHandle& op, torch::jit::Stack*) {
  TORCH_CHECK(false, op.schema().name(), ": tensors must be on the GPU (got cpu); there is no CPU implementation");
}

}  // namespace

TORCH_LIBRARY(prunepath, m) {
  m.def("route(Tensor x, Tensor router_packed, Tensor? bias, int E, float tau) -> "
        "(Tensor logits, Tensor probs, Tensor gates, Tensor mask, Tensor count)");
  m.def("route_logits(Tensor logits, float tau) -> (Tensor probs, Tensor gates, Tensor mask, Tensor count)");
  m.def("bucket(Tensor mask, Tensor gates, int tile_m=0) -> (Tensor offsets, Tensor token_ids, Tensor pair_gates, "
        "Tensor token_pairs, Tensor tiles, Tensor meta)");
  m.def("pack_experts(Tensor w_gate, Tensor w_up, Tensor w_down, int E, int G, Tensor? perm=None, "
        "str layout='linear') -> Tensor");
  m.def("pack_router(Tensor w_router, str layout='linear') -> Tensor");
  m.def("decode_workspace_init(Tensor(a!) workspace, int H, int E) -> ()");
  m.def("moe_decode(Tensor x, Tensor router_packed, Tensor? bias, int E, int G, float tau, Tensor packed, "
        "Tensor(a!) workspace, int grid=0) -> Tensor");
  m.def("moe_decode_into(Tensor x, Tensor router_packed, Tensor? bias, int E, int G, float tau, Tensor packed, "
        "Tensor(a!) workspace, Tensor(b!) out, int grid=0) -> ()");
  m.def("moe_decode_batch(Tensor x, Tensor router_packed, Tensor? bias, int E, int G, float tau, Tensor packed, "
        "Tensor(a!) workspace, Tensor(b!) batch_workspace, int grid=0) -> Tensor");
  m.def("moe_decode_batch_into(Tensor x, Tensor router_packed, Tensor? bias, int E, int G, float tau, Tensor packed, "
        "Tensor(a!) workspace, Tensor(b!) batch_workspace, Tensor(c!) out, Tensor(d!)? logits_out=None, "
        "Tensor(e!)? mask_out=None, int grid=0) -> ()");
  m.def("moe_prefill(Tensor x, Tensor router_packed, Tensor? bias, int E, int G, float tau, Tensor packed) -> Tensor");
  m.def("moe_prefill_into(Tensor x, Tensor router_packed, Tensor? bias, int E, int G, float tau, Tensor packed, "
        "Tensor(a!) workspace, Tensor(b!) out, Tensor(c!)? logits_out=None, Tensor(d!)? mask_out=None) -> ()");
  m.def("masked_gate(Tensor inter, Tensor gates, Tensor expert_ids, Tensor perm, Tensor seg) -> Tensor");
  m.def("masked_gate_bwd(Tensor d_out, Tensor inter, Tensor gates, Tensor expert_ids, Tensor perm, Tensor seg, "
        "bool need_d_inter=True) -> (Tensor d_inter, Tensor d_gates)");
  m.def("rotary(Tensor x, Tensor positions, Tensor inv_freq, str layout='half', float mscale=1.0, bool inverse=False) "
        "-> Tensor");
  m.def("qk_norm_rotary(Tensor q, Tensor k, Tensor q_weight, Tensor k_weight, Tensor positions, Tensor inv_freq, "
        "str layout='half', float mscale=1.0, float eps=1e-06) -> (Tensor q, Tensor k)");
  m.def("qk_norm_rotary_bwd(Tensor dq, Tensor dk, Tensor q, Tensor k, Tensor q_weight, Tensor k_weight, Tensor positions, "
        "Tensor inv_freq, str layout='half', float mscale=1.0, float eps=1e-06, bool weights=True) -> "
        "(Tensor q, Tensor k, Tensor q_weight, Tensor k_weight)");
  m.def("kv_append(Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor block_table, Tensor kv_lens, "
        "Tensor cu_q, Tensor? inv_freq=None, str layout='half', float mscale=1.0, Tensor? k_weight=None, float eps=1e-06, "
        "Tensor(d!)? k_scales=None, Tensor(e!)? v_scales=None) -> ()");
  m.def("kv_append_q(Tensor q, Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor block_table, "
        "Tensor kv_lens, Tensor cu_q, Tensor? inv_freq=None, str layout='half', float mscale=1.0, Tensor? q_weight=None, "
        "Tensor? k_weight=None, float eps=1e-06, Tensor(d!)? k_scales=None, Tensor(e!)? v_scales=None) -> Tensor");
  m.def("kv_append_q_into(Tensor q, Tensor(c!) q_out, Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, "
        "Tensor block_table, Tensor kv_lens, Tensor cu_q, Tensor? inv_freq=None, str layout='half', "
        "float mscale=1.0, Tensor? q_weight=None, Tensor? k_weight=None, float eps=1e-06, Tensor(d!)? k_scales=None, "
        "Tensor(e!)? v_scales=None) -> ()");
  m.def("kv_read(Tensor k_pages, Tensor v_pages, Tensor block_table, Tensor kv_lens, Tensor cu_q, SymInt rows, "
        "Tensor? k_scales=None, Tensor? v_scales=None) -> (Tensor k, Tensor v)");
  m.def("kv_read_into(Tensor k_pages, Tensor v_pages, Tensor block_table, Tensor kv_lens, Tensor cu_q, Tensor(a!) k_out, "
        "Tensor(b!) v_out, Tensor? k_scales=None, Tensor? v_scales=None) -> ()");
  m.def("paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor block_table, Tensor kv_lens, Tensor cu_q, "
        "float scale, Tensor? k_scales=None, Tensor? v_scales=None, int window=0, int sinks=0) -> Tensor");
  m.def("paged_attention_into(Tensor q, Tensor k_pages, Tensor v_pages, Tensor block_table, Tensor kv_lens, "
        "Tensor cu_q, float scale, Tensor(a!) out, Tensor? k_scales=None, Tensor? v_scales=None, int window=0, "
        "int sinks=0) -> ()");
}

TORCH_LIBRARY_IMPL(prunepath, CUDA, m) {
  m.impl("route", &route_gpu);
  m.impl("route_logits", &route_logits_gpu);
  m.impl("bucket", &bucket_gpu);
  m.impl("pack_experts", &pack_experts_gpu);
  m.impl("pack_router", &pack_router_gpu);
  m.impl("decode_workspace_init", &decode_workspace_init_gpu);
  m.impl("moe_decode", &moe_decode_gpu);
  m.impl("moe_decode_into", &decode_into);
  m.impl("moe_decode_batch", &moe_decode_batch_gpu);
  m.impl("moe_decode_batch_into", &decode_batch_into);
  m.impl("moe_prefill", &moe_prefill_gpu);
  m.impl("moe_prefill_into", &prefill_into);
  m.impl("masked_gate", &masked_gate_gpu);
  m.impl("masked_gate_bwd", &masked_gate_bwd_gpu);
  m.impl("rotary", &rotary_gpu);
  m.impl("qk_norm_rotary", &qk_norm_rotary_gpu);
  m.impl("qk_norm_rotary_bwd", &qk_norm_rotary_bwd_gpu);
  m.impl("kv_append", &kv_append_gpu);
  m.impl("kv_append_q", &kv_append_q_gpu);
  m.impl("kv_append_q_into", &kv_append_q_into_gpu);
  m.impl("kv_read", &kv_read_gpu);
  m.impl("kv_read_into", &kv_read_into_gpu);
  m.impl("paged_attention", &paged_attention_gpu);
  m.impl("paged_attention_into", &paged_attention_into_gpu);
}

TORCH_LIBRARY_IMPL(prunepath, Meta, m) {
  m.impl("route", &route_meta);
  m.impl("route_logits", &route_logits_meta);
  m.impl("bucket", &bucket_meta);
  m.impl("pack_experts", &pack_experts_meta);
  m.impl("pack_router", &pack_router_meta);
  m.impl("decode_workspace_init", &decode_workspace_init_meta);
  m.impl("moe_decode", &moe_decode_meta);
  m.impl("moe_decode_into", &moe_decode_into_meta);
  m.impl("moe_decode_batch", &moe_decode_batch_meta);
  m.impl("moe_decode_batch_into", &moe_decode_batch_into_meta);
  m.impl("moe_prefill", &moe_prefill_meta);
  m.impl("moe_prefill_into", &moe_prefill_into_meta);
  m.impl("masked_gate", &masked_gate_meta);
  m.impl("masked_gate_bwd", &masked_gate_bwd_meta);
  m.impl("rotary", &rotary_meta);
  m.impl("qk_norm_rotary", &qk_norm_rotary_meta);
  m.impl("qk_norm_rotary_bwd", &qk_norm_rotary_bwd_meta);
  m.impl("kv_append", &kv_append_meta);
  m.impl("kv_append_q", &kv_append_q_meta);
  m.impl("kv_append_q_into", &kv_append_q_into_meta);
  m.impl("kv_read", &kv_read_meta);
  m.impl("kv_read_into", &kv_read_into_meta);
  m.impl("paged_attention", &paged_attention_meta);
  m.impl("paged_attention_into", &paged_attention_into_meta);
}

TORCH_LIBRARY_IMPL(prunepath, Autograd, m) {
  m.impl("rotary", &rotary_autograd);
  m.impl("qk_norm_rotary", &qk_norm_rotary_autograd);
  m.impl("qk_norm_rotary_bwd", &qk_norm_rotary_bwd_autograd);
  INFERENCE(m, kv_append);
  INFERENCE(m, kv_append_q);
  INFERENCE(m, kv_append_q_into);
  INFERENCE(m, kv_read);
  INFERENCE(m, kv_read_into);
  INFERENCE(m, paged_attention);
  INFERENCE(m, paged_attention_into);
}

TORCH_LIBRARY_IMPL(prunepath, ADInplaceOrView, m) {
  WRITES(m, decode_workspace_init, decode_workspace_init_gpu, 1 << 0);
  WRITES(m, moe_decode, moe_decode_gpu, 1 << 7);
  WRITES(m, moe_decode_into, decode_into, 1 << 7 | 1 << 8);
  WRITES(m, moe_decode_batch, moe_decode_batch_gpu, 1 << 7 | 1 << 8);
  WRITES(m, moe_decode_batch_into, decode_batch_into, 1 << 7 | 1 << 8 | 1 << 9 | 1 << 10 | 1 << 11);
  WRITES(m, moe_prefill_into, prefill_into, 1 << 7 | 1 << 8 | 1 << 9 | 1 << 10);
  WRITES(m, kv_append, kv_append_gpu, 1 << 2 | 1 << 3 | 1 << 12 | 1 << 13);
  WRITES(m, kv_append_q, kv_append_q_gpu, 1 << 3 | 1 << 4 | 1 << 14 | 1 << 15);
  WRITES(m, kv_append_q_into, kv_append_q_into_gpu, 1 << 1 | 1 << 4 | 1 << 5 | 1 << 15 | 1 << 16);
  WRITES(m, kv_read_into, kv_read_into_gpu, 1 << 5 | 1 << 6);
  WRITES(m, paged_attention_into, paged_attention_into_gpu, 1 << 7);
}

TORCH_LIBRARY_IMPL(prunepath, CPU, m) {
  for (const char* name : {"route", "route_logits", "bucket", "pack_experts", "pack_router", "decode_workspace_init",
                           "moe_decode", "moe_decode_into", "moe_decode_batch", "moe_decode_batch_into",
                           "moe_prefill", "moe_prefill_into", "masked_gate", "masked_gate_bwd", "rotary",
                           "qk_norm_rotary", "qk_norm_rotary_bwd", "kv_append", "kv_append_q", "kv_append_q_into", "kv_read",
                           "kv_read_into", "paged_attention", "paged_attention_into"})
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&refuse_cpu>());
}
