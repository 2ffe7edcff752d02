// torch <-> gfx950 kernel bindings.  Host-only TU: validates tensors, allocates
// outputs through the torch caching allocator, and launches on the CURRENT HIP
// stream of the tensor's device (so kernels order correctly with hipBLASLt GEMMs
// and RCCL, and are capturable into HIP graphs).
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/extension.h>

#include "hx_launch.h"

namespace {

using torch::Tensor;
using OptT = c10::optional<Tensor>;

inline hipStream_t cur_stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

inline void check_cuda(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}
// Per-update dropout key: a 1-element int64 tensor on the kernel's device, read by the
// kernels themselves (ops/rng.py keeps it; graph-captured steps replay with new keys).
inline const uint64_t* seed_ptr(const Tensor& seed) {
  TORCH_CHECK(seed.is_cuda() && seed.scalar_type() == torch::kInt64 && seed.numel() >= 1,
              "dropout seed must be a 1-element int64 GPU tensor");
  return reinterpret_cast<const uint64_t*>(seed.data_ptr<int64_t>());
}
inline int act_bf16(const Tensor& t) {
  TORCH_CHECK(t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16, "activations must be fp32 or bf16");
  return t.scalar_type() == torch::kBFloat16 ? 1 : 0;
}
inline void check_f32(const Tensor& t, const char* name) {
  check_cuda(t, name);
  TORCH_CHECK(t.scalar_type() == torch::kFloat32, name, " must be fp32");
}
template <typename T>
inline T* ptr_or_null(const OptT& t) {
  return (t.has_value() && t->defined()) ? reinterpret_cast<T*>(t->data_ptr()) : nullptr;
}
inline bool has(const OptT& t) { return t.has_value() && t->defined(); }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ------------------------------------------------------------------ debug mode
// ``--debug-kernels``: host-side validation that needs device reads
// (range checks on indices, finite checks on every fused op's output).  Each check
// synchronises, so it is off by default; combined with AMD_SERIALIZE_KERNEL=3 the
// first kernel producing a bad value is the one that raises.
bool g_debug = false;
void set_debug(bool on) { g_debug = on; }
bool get_debug() { return g_debug; }
inline void dbg_range(const Tensor& t, int64_t lo, int64_t hi, const char* what) {
  if (!g_debug || t.numel() == 0) return;
  const int64_t mn = t.min().item<int64_t>(), mx = t.max().item<int64_t>();
  TORCH_CHECK(mn >= lo && mx < hi, what, " out of range: [", mn, ", ", mx, "] not within [", lo, ", ", hi, ")");
}
inline void dbg_finite(const Tensor& t, const char* what) {
  if (!g_debug || !t.defined() || t.numel() == 0) return;
  TORCH_CHECK(torch::isfinite(t).all().item<bool>(), "non-finite values produced by ", what);
}

// ------------------------------------------------------------------ optimizer
void grad_norm_clip(Tensor g, Tensor gscale, Tensor out_norm, Tensor clipped, double max_norm) {
  check_f32(g, "grad");
  check_f32(gscale, "gscale");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(g.device());
  TORCH_CHECK(aligned16(g.data_ptr()), "flat grad must be 16-byte aligned");
  auto ws = torch::empty({hx_grad_norm_partials()}, g.options().dtype(torch::kFloat64));
  hx_grad_norm_clip(g.data_ptr<float>(), g.numel(), ws.data_ptr<double>(), gscale.data_ptr<float>(),
                    out_norm.data_ptr<float>(), clipped.data_ptr<float>(), (float)max_norm, cur_stream(g));
}

// hp (optional, device fp32 [2]): step size and wd * lr read by the kernel instead of the
// host values -- a captured training step (utils/train_graph.py) refreshes them per replay
inline const float* hp_ptr(const OptT& hp, int64_t need) {
  if (!has(hp)) return nullptr;
  TORCH_CHECK(hp->is_cuda() && hp->scalar_type() == torch::kFloat32 && hp->numel() >= need && hp->is_contiguous(),
              "optimizer hyper-parameters must be a contiguous fp32 GPU tensor");
  return hp->data_ptr<float>();
}

void adam(Tensor p, Tensor g, Tensor m, Tensor v, OptT shadow, Tensor gscale, int64_t start, int64_t end, double b1,
          double b2, double eps, double step_size, double wd_lr, OptT hp) {
  check_f32(p, "param");
  check_f32(g, "grad");
  check_f32(m, "exp_avg");
  check_f32(v, "exp_avg_sq");
  TORCH_CHECK(start >= 0 && end <= p.numel() && start <= end && start % 4 == 0, "bad param range");
  TORCH_CHECK(g.numel() == p.numel() && m.numel() == p.numel() && v.numel() == p.numel(), "flat size mismatch");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(p.device());
  uint16_t* sh = nullptr;
  if (has(shadow)) {
    TORCH_CHECK(shadow->scalar_type() == torch::kBFloat16 && shadow->numel() == p.numel(), "bad bf16 shadow");
    sh = reinterpret_cast<uint16_t*>(shadow->data_ptr()) + start;
  }
  hx_adam(p.data_ptr<float>() + start, g.data_ptr<float>() + start, m.data_ptr<float>() + start,
          v.data_ptr<float>() + start, sh, gscale.data_ptr<float>(), end - start, (float)b1, (float)b2, (float)eps,
          (float)step_size, (float)wd_lr, hp_ptr(hp, 2), cur_stream(p));
}

void adam_masked(Tensor p, Tensor g, Tensor m, Tensor v, OptT shadow, Tensor gscale, Tensor table, Tensor used,
                 Tensor steps, Tensor hp, double lr, double b1, double b2, double eps, double wd, OptT lr_dev) {
  check_f32(p, "param");
  check_f32(g, "grad");
  check_f32(m, "exp_avg");
  check_f32(v, "exp_avg_sq");
  TORCH_CHECK(g.numel() == p.numel() && m.numel() == p.numel() && v.numel() == p.numel(), "flat size mismatch");
  const int64_t nparam = steps.numel();
  TORCH_CHECK(steps.is_cuda() && steps.scalar_type() == torch::kInt32 && steps.is_contiguous(), "steps: int32 GPU");
  TORCH_CHECK(used.is_cuda() && used.scalar_type() == torch::kFloat64 && used.is_contiguous() &&
                  used.numel() == nparam, "used flags: contiguous f64 GPU tensor, one per parameter");
  TORCH_CHECK(hp.is_cuda() && hp.scalar_type() == torch::kFloat32 && hp.numel() >= 2 * nparam, "hp: f32 [2*nparam]");
  TORCH_CHECK(table.is_cuda() && table.scalar_type() == torch::kInt64 && table.dim() == 2 && table.size(1) == 3 &&
                  table.is_contiguous(), "table: int64 [nblocks, 3]");
  uint16_t* sh = nullptr;
  if (has(shadow)) {
    TORCH_CHECK(shadow->scalar_type() == torch::kBFloat16 && shadow->numel() == p.numel(), "bad bf16 shadow");
    sh = reinterpret_cast<uint16_t*>(shadow->data_ptr());
  }
  if (has(lr_dev))
    TORCH_CHECK(lr_dev->is_cuda() && lr_dev->scalar_type() == torch::kFloat64 && lr_dev->numel() == 1, "lr_dev: f64 [1]");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(p.device());
  hx_adam_masked(p.data_ptr<float>(), g.data_ptr<float>(), m.data_ptr<float>(), v.data_ptr<float>(), sh,
                 gscale.data_ptr<float>(), table.data_ptr<int64_t>(), (int)table.size(0), used.data_ptr<double>(),
                 steps.data_ptr<int>(), hp.data_ptr<float>(), (int)nparam, lr, b1, b2, (float)eps, wd,
                 has(lr_dev) ? lr_dev->data_ptr<double>() : nullptr, cur_stream(p));
}

void adadelta(Tensor p, Tensor g, Tensor sq, Tensor acc, Tensor gscale, int64_t start, int64_t end, double lr,
              double rho, double eps, double wd, OptT hp) {
  check_f32(p, "param");
  TORCH_CHECK(start >= 0 && end <= p.numel() && start <= end, "bad param range");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(p.device());
  hx_adadelta(p.data_ptr<float>() + start, g.data_ptr<float>() + start, sq.data_ptr<float>() + start,
              acc.data_ptr<float>() + start, gscale.data_ptr<float>(), end - start, (float)lr, (float)rho,
              (float)eps, (float)wd, hp_ptr(hp, 1), cur_stream(p));
}

// ------------------------------------------------------------------ layernorm
// amax_out (fp32 runs only): receives max |out| of every row, [rows] (the fp16x3 GEMMs' per-row
// operand scale, ops/gemm16.py)
inline float* amax_ptr(const OptT& a, int64_t need, const char* what) {
  if (!has(a)) return nullptr;
  check_f32(*a, what);
  TORCH_CHECK(a->is_contiguous() && a->numel() >= need, what, ": needs ", need, " fp32 partials");
  return a->data_ptr<float>();
}
// pieces_out (fp32 runs, with amax_out): fp16 P2 pieces [rows, 2H] of the output at its row scales,
// the consumer GEMM's A operand already split (gemm_f16 with fp16 A)
inline uint16_t* pieces_ptr(const OptT& p, int64_t rows, int H, const OptT& amax, const char* what) {
  if (!has(p)) return nullptr;
  TORCH_CHECK(has(amax), what, ": pieces need the row maxima output too");
  TORCH_CHECK(p->is_cuda() && p->scalar_type() == torch::kHalf && p->is_contiguous() && p->numel() == rows * 2 * H &&
                  H % 16 == 0 && aligned16(p->data_ptr()), what, ": fp16 [rows, 2H] (H % 16 == 0)");
  return reinterpret_cast<uint16_t*>(p->data_ptr());
}
std::vector<Tensor> ln_fwd(Tensor y, OptT bias, OptT res, Tensor gamma, Tensor beta, double eps, double keep_prob,
                           const Tensor& seed, int64_t stream, bool drop_after, bool save_z, OptT amax_out,
                           OptT pieces_out) {
  check_cuda(y, "input");
  const int H = (int)y.size(-1);
  const int64_t rows = y.numel() / H;
  TORCH_CHECK(H % 4 == 0 && H <= 2048, "LayerNorm hidden size must be a multiple of 4 and <= 2048");
  check_f32(gamma, "gamma");
  check_f32(beta, "beta");
  if (has(res)) {
    check_cuda(*res, "residual");
    TORCH_CHECK(res->scalar_type() == y.scalar_type() && res->numel() == y.numel(), "residual mismatch");
  }
  if (has(bias)) check_f32(*bias, "bias");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(y.device());
  auto out = torch::empty_like(y);
  Tensor z = save_z ? torch::empty_like(y) : Tensor();
  auto st = y.options().dtype(torch::kFloat32);
  auto mean = torch::empty({rows}, st), rstd = torch::empty({rows}, st);
  hx_ln_fwd(act_bf16(y), y.data_ptr(), ptr_or_null<float>(bias), has(res) ? res->data_ptr() : nullptr,
            gamma.data_ptr<float>(), beta.data_ptr<float>(), out.data_ptr(), save_z ? z.data_ptr() : nullptr,
            mean.data_ptr<float>(), rstd.data_ptr<float>(), rows, H, (float)eps, (float)keep_prob, seed_ptr(seed),
            (uint64_t)stream, drop_after ? 1 : 0, cur_stream(y),
            act_bf16(y) ? nullptr : amax_ptr(amax_out, rows, "ln_fwd amax"),
            act_bf16(y) ? nullptr : pieces_ptr(pieces_out, rows, H, amax_out, "ln_fwd pieces"));
  dbg_finite(out, "ln_fwd");
  return {out, z, mean, rstd};
}

std::vector<Tensor> ln_bwd(Tensor dout, Tensor z, Tensor mean, Tensor rstd, Tensor gamma, double keep_prob,
                           const Tensor& seed, int64_t stream, bool drop_after, bool want_dy, bool want_dbias,
                           OptT dgamma_out, OptT dbeta_out, OptT dbias_out, OptT amax_out, OptT colmax_out,
                           OptT pieces_out) {
  check_cuda(dout, "grad_output");
  check_cuda(z, "saved input");
  const int H = (int)z.size(-1);
  const int64_t rows = z.numel() / H;
  c10::hip::HIPGuardMasqueradingAsCUDA guard(z.device());
  auto dz = torch::empty_like(z);
  Tensor dy = want_dy ? torch::empty_like(z) : Tensor();
  auto f32 = z.options().dtype(torch::kFloat32);
  auto dgamma = has(dgamma_out) ? *dgamma_out : torch::empty({H}, f32);
  auto dbeta = has(dbeta_out) ? *dbeta_out : torch::empty({H}, f32);
  Tensor dbias = want_dbias ? (has(dbias_out) ? *dbias_out : torch::empty({H}, f32)) : Tensor();
  TORCH_CHECK(dgamma.numel() == H && dbeta.numel() == H && dgamma.is_contiguous() && dbeta.is_contiguous(),
              "bad dgamma/dbeta outputs");
  const int nblk = hx_ln_bwd_blocks(rows);
  auto partial = torch::empty({(int64_t)nblk * 4 * H}, f32);
  hx_ln_bwd(act_bf16(z), dout.data_ptr(), z.data_ptr(), mean.data_ptr<float>(), rstd.data_ptr<float>(),
            gamma.data_ptr<float>(), dz.data_ptr(), want_dy ? dy.data_ptr() : nullptr, partial.data_ptr<float>(), nblk,
            rows, H, (float)keep_prob, seed_ptr(seed), (uint64_t)stream, drop_after ? 1 : 0,
            (want_dy && want_dbias) ? 1 : 0, dgamma.data_ptr<float>(), dbeta.data_ptr<float>(),
            want_dbias ? dbias.data_ptr<float>() : nullptr, 0, cur_stream(z),
            act_bf16(z) ? nullptr : amax_ptr(amax_out, rows, "ln_bwd amax"),
            act_bf16(z) ? nullptr : amax_ptr(colmax_out, H, "ln_bwd colmax"),
            act_bf16(z) ? nullptr : pieces_ptr(pieces_out, rows, H, amax_out, "ln_bwd pieces"));
  dbg_finite(dz, "ln_bwd (dz)");
  return {dz, dy, dgamma, dbeta, dbias};
}

std::vector<Tensor> embed_ln_fwd(Tensor ids, OptT tt, Tensor wte, Tensor wpe, Tensor wtt, Tensor gamma, Tensor beta,
                                 double eps, double keep_prob, const Tensor& seed, int64_t stream, bool bf16_out,
                                 OptT amax_out, OptT pieces_out) {
  dbg_range(ids, 0, wte.size(0), "token ids");
  if (has(tt)) dbg_range(*tt, 0, wtt.size(0), "token type ids");
  check_cuda(ids, "input_ids");
  TORCH_CHECK(ids.scalar_type() == torch::kInt64 && ids.dim() == 2, "input_ids must be int64 [B, S]");
  check_f32(wte, "word_embeddings");
  check_f32(wpe, "position_embeddings");
  check_f32(wtt, "token_type_embeddings");
  const int64_t B = ids.size(0), S = ids.size(1);
  const int H = (int)wte.size(1);
  TORCH_CHECK(H % 4 == 0 && H <= 2048, "hidden size must be a multiple of 4 and <= 2048");
  TORCH_CHECK(S <= wpe.size(0), "sequence longer than max_position_embeddings");
  if (has(tt)) TORCH_CHECK(tt->scalar_type() == torch::kInt64 && tt->numel() == ids.numel(), "token_type_ids mismatch");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(ids.device());
  auto opt = wte.options().dtype(bf16_out ? torch::kBFloat16 : torch::kFloat32);
  auto out = torch::empty({B, S, H}, opt), z = torch::empty({B, S, H}, opt);
  auto f32 = wte.options();
  auto mean = torch::empty({B * S}, f32), rstd = torch::empty({B * S}, f32);
  hx_embed_ln_fwd(bf16_out ? 1 : 0, ids.data_ptr<int64_t>(), has(tt) ? tt->data_ptr<int64_t>() : nullptr,
                  wte.data_ptr<float>(), wpe.data_ptr<float>(), wtt.data_ptr<float>(), gamma.data_ptr<float>(),
                  beta.data_ptr<float>(), out.data_ptr(), z.data_ptr(), mean.data_ptr<float>(), rstd.data_ptr<float>(),
                  B * S, (int)S, H, (float)eps, (float)keep_prob, seed_ptr(seed), (uint64_t)stream, cur_stream(ids),
                  bf16_out ? nullptr : amax_ptr(amax_out, B * S, "embed_ln_fwd amax"),
                  bf16_out ? nullptr : pieces_ptr(pieces_out, B * S, H, amax_out, "embed_ln_fwd pieces"));
  dbg_finite(out, "embed_ln_fwd");
  return {out, z, mean, rstd};
}

// Scatter-ACCUMULATES the embedding gradients into dwte / dwpe / dwtt (caller zeroes them
// when they are fresh).
// word-embedding gradient, accumulated into dwte: rows visited in id-sorted order
void embed_word_grad(Tensor dz, Tensor ids, Tensor order, Tensor dwte) {
  check_cuda(dz, "grad");
  check_cuda(ids, "ids");
  check_cuda(order, "order");
  check_f32(dwte, "dwte");
  TORCH_CHECK(ids.scalar_type() == torch::kLong && order.scalar_type() == torch::kLong, "ids/order must be int64");
  const int H = (int)dz.size(-1);
  const int64_t rows = dz.numel() / H;
  TORCH_CHECK(ids.numel() == rows && order.numel() == rows, "ids/order/grad row mismatch");
  TORCH_CHECK(dwte.size(-1) == H && H % 4 == 0 && H <= 2048, "bad embedding width");
  dbg_range(ids, 0, dwte.size(0), "token ids");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dz.device());
  hx_embed_word_grad_sorted(act_bf16(dz), dz.data_ptr(), ids.data_ptr<int64_t>(), order.data_ptr<int64_t>(),
                            dwte.data_ptr<float>(), rows, H, cur_stream(dz));
}

// token-type embedding gradient (ntypes <= 3) into dwtt [ntypes, H] (overwritten)
void embed_type_grad(Tensor dz, Tensor tt, Tensor dwtt) {
  check_cuda(dz, "grad");
  check_f32(dwtt, "dwtt");
  TORCH_CHECK(tt.scalar_type() == torch::kLong && tt.is_contiguous() && tt.device() == dz.device(), "tt: int64");
  const int H = (int)dz.size(-1);
  const int64_t rows = dz.numel() / H;
  const int ntypes = (int)dwtt.size(0);
  TORCH_CHECK(dz.is_contiguous() && tt.numel() == rows && dwtt.dim() == 2 && dwtt.size(1) == H &&
                  dwtt.is_contiguous() && ntypes >= 1 && ntypes <= 3 && H % 4 == 0 && H <= 2048,
              "embed_type_grad: contiguous dz [rows, H], tt [rows], dwtt [ntypes <= 3, H]");
  dbg_range(tt, 0, ntypes, "token type ids");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dz.device());
  Tensor part = torch::empty({(int64_t)hx_type_grad_blocks(rows) * ntypes * H}, dz.options().dtype(torch::kFloat32));
  hx_type_grad(act_bf16(dz), dz.data_ptr(), tt.data_ptr<int64_t>(), part.data_ptr<float>(), dwtt.data_ptr<float>(),
               rows, H, ntypes, cur_stream(dz));
}

// ------------------------------------------------------------------ elementwise
Tensor bias_act_fwd(Tensor y, OptT b, int64_t act) {
  check_cuda(y, "input");
  const int N = (int)y.size(-1);
  TORCH_CHECK(N % 4 == 0, "bias_act: last dim must be a multiple of 4");
  if (has(b)) check_f32(*b, "bias");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(y.device());
  auto out = torch::empty_like(y);
  hx_bias_act_fwd(act_bf16(y), (int)act, y.data_ptr(), ptr_or_null<float>(b), out.data_ptr(), y.numel() / N, N,
                  cur_stream(y));
  dbg_finite(out, "bias_act_fwd");
  return out;
}

std::vector<Tensor> bias_act_bwd(Tensor dout, OptT y, OptT b, OptT saved_out, int64_t act, bool want_dbias,
                                 OptT dbias_out) {
  check_cuda(dout, "grad_output");
  const int N = (int)dout.size(-1);
  const int64_t rows = dout.numel() / N;
  TORCH_CHECK(N % 4 == 0, "bias_act: last dim must be a multiple of 4");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dout.device());
  auto dy = torch::empty_like(dout);
  auto f32 = dout.options().dtype(torch::kFloat32);
  Tensor dbias, ws;
  if (want_dbias) {
    dbias = has(dbias_out) ? *dbias_out : torch::empty({N}, f32);
    ws = torch::empty({(int64_t)hx_colsum_ws_floats(rows, N)}, f32);
  }
  hx_bias_act_bwd(act_bf16(dout), (int)act, dout.data_ptr(), has(y) ? y->data_ptr() : nullptr, ptr_or_null<float>(b),
                  has(saved_out) ? saved_out->data_ptr() : nullptr, dy.data_ptr(),
                  want_dbias ? ws.data_ptr<float>() : nullptr, want_dbias ? dbias.data_ptr<float>() : nullptr, rows, N,
                  0, cur_stream(dout));
  dbg_finite(dy, "bias_act_bwd");
  return {dy, dbias};
}

Tensor colsum(Tensor x, OptT scale, OptT out_) {
  TORCH_CHECK(x.is_cuda(), "input must be a GPU tensor");
  const int N = (int)x.size(-1);
  // 2-D with unit column stride: any row stride (e.g. the valid columns of a padded buffer)
  const bool strided2d = x.dim() == 2 && x.stride(1) == 1;
  TORCH_CHECK(strided2d || x.is_contiguous(), "colsum: contiguous input or 2-D rows with unit column stride");
  const int64_t rows = strided2d ? x.size(0) : x.numel() / N;
  const int64_t ld = strided2d ? x.stride(0) : N;
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  auto f32 = x.options().dtype(torch::kFloat32);
  auto out = has(out_) ? *out_ : torch::empty({N}, f32);
  TORCH_CHECK(out.numel() == N && out.is_contiguous(), "bad colsum output");
  auto ws = torch::empty({(int64_t)hx_colsum_ws_floats(rows, N)}, f32);
  hx_colsum(act_bf16(x), x.data_ptr(), ptr_or_null<float>(scale), ws.data_ptr<float>(), out.data_ptr<float>(), rows,
            N, 0, cur_stream(x), ld);
  return out;
}

Tensor dropout(Tensor x, double keep_prob, const Tensor& seed, int64_t stream) {
  check_cuda(x, "input");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  auto out = torch::empty_like(x);
  hx_dropout(act_bf16(x), x.data_ptr(), out.data_ptr(), x.numel(), (float)keep_prob, seed_ptr(seed),
             (uint64_t)stream, cur_stream(x));
  return out;
}

Tensor softmax_xent_(Tensor logits, OptT bias, Tensor labels, int64_t ignore_index) {
  dbg_range(labels, std::min<int64_t>(ignore_index, 0), logits.size(-1), "MLM labels");
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.stride(1) == 1, "logits must be a 2-D row-major GPU tensor");
  check_cuda(labels, "labels");
  TORCH_CHECK(labels.scalar_type() == torch::kInt64 && labels.numel() == logits.size(0), "labels must be int64 [rows]");
  if (has(bias)) {
    check_f32(*bias, "bias");
    TORCH_CHECK(bias->numel() >= logits.size(1), "bias too small");
  }
  c10::hip::HIPGuardMasqueradingAsCUDA guard(logits.device());
  auto loss = torch::empty({logits.size(0)}, logits.options().dtype(torch::kFloat32));
  hx_softmax_xent(act_bf16(logits), logits.data_ptr(), ptr_or_null<float>(bias), labels.data_ptr<int64_t>(),
                  loss.data_ptr<float>(), logits.size(0), (int)logits.size(1), logits.stride(0), ignore_index,
                  cur_stream(logits));
  dbg_finite(loss, "softmax_xent");
  return loss;
}

// ------------------------------------------------------------------ attention
std::vector<Tensor> attn_fwd(Tensor qkv, Tensor mask_bias, int64_t nh, double keep, const Tensor& seed, int64_t stream,
                             OptT bias, int split = 0, OptT amax_out = OptT(), OptT colmax_out = OptT()) {
  // split: 0 none (fp32 / bf16 MFMA), 2 fp16x3 (attention_f16.hip)
  check_cuda(qkv, "qkv");
  const int bf = act_bf16(qkv);
  check_f32(mask_bias, "mask_bias");
  TORCH_CHECK(qkv.dim() == 3, "qkv must be [B, S, 3H]");
  const int64_t B = qkv.size(0), S = qkv.size(1), H = qkv.size(2) / 3;
  TORCH_CHECK(H == nh * 64, "fused attention needs head_dim == 64");
  TORCH_CHECK(mask_bias.numel() == B * S, "mask_bias must be [B, S]");
  if (has(bias)) {
    check_f32(*bias, "qkv bias");
    TORCH_CHECK(bias->numel() == 3 * H, "qkv bias must have 3H elements");
  }
  c10::hip::HIPGuardMasqueradingAsCUDA guard(qkv.device());
  auto out = torch::empty({B, S, H}, qkv.options());
  auto lse = torch::empty({B, nh, S}, qkv.options().dtype(torch::kFloat32));
  Tensor dmask;
  // 1 bit per (key, query), stored [key][query word] with both padded to 128
  const int64_t Sp = (S + 127) / 128 * 128;
  if (keep < 1.0) dmask = torch::empty({B, nh, Sp, Sp / 32}, qkv.options().dtype(torch::kInt32));
  else dmask = torch::empty({0}, qkv.options().dtype(torch::kInt32));
  uint32_t* dm = keep < 1.0 ? reinterpret_cast<uint32_t*>(dmask.data_ptr<int32_t>()) : nullptr;
  if (split) {
    TORCH_CHECK(!bf, "attn_fwd_f16: fp32 activations only");
    float* am = amax_ptr(amax_out, B * S * nh, "attn_fwd amax");   // [B * S rows][nh heads]
    float* cm = amax_ptr(colmax_out, B * ((S + 127) / 128) * H, "attn_fwd colmax");   // [B * qblocks][H]
    hx_attn_fwd_f16(qkv.data_ptr<float>(), ptr_or_null<float>(bias), mask_bias.data_ptr<float>(),
                    out.data_ptr<float>(), lse.data_ptr<float>(), dm, (int)B, (int)S, (int)nh, (float)keep,
                    seed_ptr(seed), (uint64_t)stream, cur_stream(qkv), am, cm);
  } else {
    hx_attn_fwd(bf, qkv.data_ptr(), ptr_or_null<float>(bias), mask_bias.data_ptr<float>(), out.data_ptr(),
                lse.data_ptr<float>(), dm, (int)B, (int)S, (int)nh, (float)keep, seed_ptr(seed), (uint64_t)stream,
                cur_stream(qkv));
  }
  dbg_finite(out, "attn_fwd");
  return {out, lse, dmask};
}
// fp32 attention forward on the fp16 matrix cores (fp16x3, attention_f16.hip): {out, lse, dmask}
std::vector<Tensor> attn_fwd_f16(Tensor qkv, Tensor mask_bias, int64_t nh, double keep, const Tensor& seed,
                                 int64_t stream, OptT bias, OptT amax_out, OptT colmax_out) {
  return attn_fwd(qkv, mask_bias, nh, keep, seed, stream, bias, 2, amax_out, colmax_out);
}

// returns {dqkv, dbias} (dbias: [3H] fp32 when bias is given or want_dbias -- written into
// dbq/dbk/dbv when those slots are given -- else an empty tensor)
std::vector<Tensor> attn_bwd(Tensor dout, Tensor qkv, Tensor mask_bias, Tensor out, Tensor lse, Tensor dmask,
                             int64_t nh, double keep, OptT bias, OptT dbq, OptT dbk, OptT dbv, int split = 0,
                             OptT amax_out = OptT(), OptT colmax_out = OptT(), bool want_dbias = false) {
  // split: 0 none (fp32 / bf16 MFMA), 2 fp16x3 (attention_f16.hip)
  check_cuda(dout, "grad_output");
  check_cuda(qkv, "qkv");
  const int bf = act_bf16(qkv);
  TORCH_CHECK(!(split && bf), "attn_bwd_f16: fp32 activations only");
  TORCH_CHECK(dout.scalar_type() == qkv.scalar_type() && out.scalar_type() == qkv.scalar_type(),
              "attention activations must share one dtype");
  const int64_t B = qkv.size(0), S = qkv.size(1), H = qkv.size(2) / 3;
  c10::hip::HIPGuardMasqueradingAsCUDA guard(qkv.device());
  // one key block per head (S <= 128): every dQKV element is written exactly once (no
  // memset).  Otherwise dQ partials from the S/128 key blocks are added atomically in
  // fp32: into dqkv itself (fp32, its dQ third zero-filled) or a [B, S, H] fp32 scratch (bf16).
  const bool multi = S > 128;
  Tensor dqkv = torch::empty_like(qkv);
  if (multi && !bf) dqkv.narrow(-1, 0, H).zero_();   // only the dQ third is accumulated into
  Tensor dq32;
  float* dq_acc = nullptr;
  int dq_ld = 0;
  if (multi && bf) {
    dq32 = torch::zeros({B, S, H}, qkv.options().dtype(torch::kFloat32));
    dq_acc = dq32.data_ptr<float>();
    dq_ld = (int)H;
  } else if (multi) {
    dq_acc = dqkv.data_ptr<float>();
    dq_ld = (int)(3 * H);
  }
  Tensor dbias, part;
  float *pq = nullptr, *pk = nullptr, *pv = nullptr;
  // the QKV-bias gradient: when the bias is added here, or (want_dbias) when the projection
  // already added it and only its gradient -- the column sums of dQKV -- is wanted
  if (has(bias) || want_dbias) {
    const bool slots = has(dbq) && has(dbk) && has(dbv);
    if (slots) {
      for (const auto* t : {&dbq, &dbk, &dbv}) {
        check_f32(**t, "qkv bias grad");
        TORCH_CHECK((*t)->numel() == H, "qkv bias grad must have H elements");
      }
      pq = dbq->data_ptr<float>(); pk = dbk->data_ptr<float>(); pv = dbv->data_ptr<float>();
    } else {
      dbias = torch::empty({3 * H}, qkv.options().dtype(torch::kFloat32));
      pq = dbias.data_ptr<float>(); pk = pq + H; pv = pq + 2 * H;
    }
    part = torch::empty({B * ((S + 127) / 128), 3 * H}, qkv.options().dtype(torch::kFloat32));
  }
  hx_attn_bwd(split ? 3 : bf, qkv.data_ptr(), ptr_or_null<float>(bias), pq, pk, pv, part.defined() ? part.data_ptr<float>() : nullptr,
              mask_bias.data_ptr<float>(), dout.data_ptr(), out.data_ptr(), lse.data_ptr<float>(),
              keep < 1.0 ? reinterpret_cast<const uint32_t*>(dmask.data_ptr<int32_t>()) : nullptr,
              dqkv.data_ptr(), dq_acc, dq_ld, (int)B, (int)S, (int)nh, (float)keep, cur_stream(qkv),
              split ? amax_ptr(amax_out, B * S * nh, "attn_bwd amax") : nullptr,   // [B * S][nh]
              split ? amax_ptr(colmax_out, B * ((S + 127) / 128) * 3 * H, "attn_bwd colmax") : nullptr);   // [B * kb][3H]
  if (multi && bf) dqkv.narrow(-1, 0, H).copy_(dq32);
  dbg_finite(dqkv, "attn_bwd");
  return {dqkv, dbias};
}

// ------------------------------------------------------------------ bf16 weight gradient
// out[M, N] (fp32, overwritten) = dy[T, M]^T . x[T, N] (bf16, unit column stride, 16-B rows)
bool wgrad_bf16_ok(const Tensor& dy, const Tensor& x) {
  if (!dy.is_cuda() || dy.scalar_type() != torch::kBFloat16 || x.scalar_type() != torch::kBFloat16) return false;
  if (dy.dim() != 2 || x.dim() != 2 || dy.size(0) != x.size(0) || dy.size(0) < 1) return false;
  if (dy.stride(1) != 1 || x.stride(1) != 1 || dy.stride(0) % 8 || x.stride(0) % 8) return false;
  if (!aligned16(dy.data_ptr()) || !aligned16(x.data_ptr())) return false;
  return dy.size(1) % 128 == 0 && x.size(1) % 128 == 0 && dy.size(0) < (1LL << 31);
}
Tensor wgrad_bf16(Tensor dy, Tensor x, Tensor out) {
  TORCH_CHECK(wgrad_bf16_ok(dy, x), "wgrad_bf16: unsupported operands (need bf16 [T, M] / [T, N] row-major "
              "with M, N multiples of 128 and 16-byte rows)");
  check_f32(out, "wgrad out");
  const int64_t T = dy.size(0), M = dy.size(1), N = x.size(1);
  // out may hold fewer rows than the (tile-padded) M: rows past out.size(0) are not stored
  TORCH_CHECK(out.size(0) <= M && out.size(0) > 0 && out.size(1) == N && out.is_contiguous(),
              "wgrad out must be [<= M, N]");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dy.device());
  int cfg = 0, nsplit = 1;
  hx_wgrad_bf16_plan((int)M, (int)N, (int)T, &cfg, &nsplit);
  Tensor ws;
  if (nsplit > 1) ws = torch::empty({nsplit * M * N}, out.options());
  hx_wgrad_bf16(dy.data_ptr(), (int)dy.stride(0), x.data_ptr(), (int)x.stride(0), out.data_ptr<float>(),
                nsplit > 1 ? ws.data_ptr<float>() : nullptr, (int)M, (int)N, (int)T, cfg, nsplit, (int)out.size(0),
                cur_stream(dy));
  dbg_finite(out, "wgrad_bf16");
  return out;
}

// ------------------------------------------------------------------ fp16x3 GEMMs (gemm_f16.hip)
// fp32 operands travel with max |x| partials (any 1-D fp32 tensor whose max is max |x|): the
// kernels turn them into the power-of-two scale of the fp16 split
inline void check_af32(const Tensor& a, const char* what) {
  check_f32(a, what);
  TORCH_CHECK(a.dim() == 2 && a.stride(1) == 1 && a.stride(0) % 4 == 0 && aligned16(a.data_ptr()) &&
                  a.size(1) % 16 == 0 && a.size(0) < (1LL << 31),
              what, ": fp32 [rows, K] with unit column stride, 16-B aligned rows and K % 16 == 0");
}
// max |x| partials of an fp32 operand: 1-D = partials of the whole tensor (any number; their max
// is a per-tensor bound), 2-D [rows, P] = P partials per operand row (the row's own scale)
struct ScaleSrc {
  const float* p;
  int np, rs;
};
inline ScaleSrc scale_src(const Tensor& t, const Tensor& ref, int64_t rows, const char* what) {
  check_f32(t, what);
  TORCH_CHECK(t.is_contiguous() && t.numel() >= 1 && t.numel() < (1LL << 31) && t.device() == ref.device(), what,
              ": max |x| partials on the operand's device");
  if (t.dim() == 1) return {t.data_ptr<float>(), (int)t.numel(), 0};
  TORCH_CHECK(t.dim() == 2 && t.size(0) == rows && t.size(1) >= 1 && t.size(1) <= 64, what,
              ": per-row max |x| partials must be [rows, P <= 64] (rows = ", rows, ")");
  return {t.data_ptr<float>(), (int)t.size(1), (int)t.size(1)};
}
inline void check_amax(const Tensor& t, const Tensor& ref, const char* what) {
  check_f32(t, what);
  TORCH_CHECK(t.is_contiguous() && t.numel() >= 1 && t.numel() < (1LL << 31) && t.device() == ref.device(), what,
              ": max |x| partials on the operand's device");
}
inline void check_p2(const Tensor& b, int64_t K, const char* what) {
  TORCH_CHECK(b.is_cuda() && b.scalar_type() == torch::kHalf && b.dim() == 2 && b.is_contiguous() &&
                  b.size(1) == 2 * K && aligned16(b.data_ptr()), what, ": fp16 P2 pieces [N, 2K]");
}

// max |x| of every row: [rows, 1]
Tensor amax_rows(Tensor x) {
  check_f32(x, "amax_rows");
  TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1 && x.stride(0) % 4 == 0 && x.size(1) % 4 == 0 &&
                  aligned16(x.data_ptr()), "amax_rows: fp32 [rows, cols] with 16-B rows, cols % 4 == 0");
  Tensor out = torch::empty({x.size(0), 1}, x.options());
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  hx_amax_rows(x.data_ptr<float>(), x.size(0), (int)x.size(1), x.stride(0), out.data_ptr<float>(), cur_stream(x));
  return out;
}

// fp32 rows [rows, K] -> fp16 P2 pieces [rows, 2K] at each row's scale (the max of its partials
// amax [rows, P]): the pre-split A operand of gemm_f16*
Tensor split_rows_f16(Tensor x, Tensor amax) {
  check_af32(x, "split_rows_f16");
  const ScaleSrc sa = scale_src(amax, x, x.size(0), "split_rows_f16");
  TORCH_CHECK(sa.rs == sa.np, "split_rows_f16: per-row partials [rows, P]");
  Tensor out = torch::empty({x.size(0), 2 * x.size(1)}, x.options().dtype(torch::kHalf));
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  hx_split_rows_f16(x.data_ptr<float>(), x.stride(0), sa.p, sa.np, x.size(0), (int)x.size(1),
                    reinterpret_cast<uint16_t*>(out.data_ptr()), cur_stream(x));
  return out;
}

// [(wf, wt, rmax, cmax)] per weight W [N, K]: P2 fp16 pieces of W (rows scaled by their own
// maxima) and of W^T (rows = columns of W, scaled by the column maxima); rmax [N, 1] / cmax [K, 1]
// are the per-row scale sources of the forward / data-gradient products
// rows: optional padded row count per weight (>= its rows, a multiple of 64): the pieces cover the
// padded rows, read as zero past W's own (the MLM decoder's vocabulary, without a padded copy)
std::vector<std::vector<Tensor>> split_weight_f16(std::vector<Tensor> Ws, std::vector<int64_t> rows) {
  TORCH_CHECK(!Ws.empty() && Ws.size() <= HX_WBATCH, "split_weight_f16: 1..64 weights");
  TORCH_CHECK(rows.empty() || rows.size() == Ws.size(), "split_weight_f16: one padded row count per weight");
  HxWeightBatch d{};
  d.n = (int)Ws.size();
  int64_t rc_floats = 0;
  for (size_t i = 0; i < Ws.size(); ++i) rc_floats += (rows.empty() ? Ws[i].size(0) : rows[i]) + Ws[i].size(1);
  Tensor rc = torch::empty({rc_floats}, Ws[0].options());
  std::vector<std::vector<Tensor>> out;
  int tiles = 0;
  int64_t off = 0;
  for (int i = 0; i < d.n; ++i) {
    const Tensor& W = Ws[i];
    check_f32(W, "split_weight_f16 input");
    const int64_t N = rows.empty() ? W.size(0) : rows[i], K = W.size(1);
    TORCH_CHECK(W.dim() == 2 && W.is_contiguous() && N % 64 == 0 && N >= W.size(0) && W.size(0) >= 1 &&
                    K % 64 == 0 && aligned16(W.data_ptr()) && W.device() == Ws[0].device(),
                "split_weight_f16: every W contiguous [N, K] (N padded to a multiple of 64 >= its rows), K a "
                "multiple of 64, one device");
    auto hf = W.options().dtype(torch::kHalf);
    Tensor wf = torch::empty({N, 2 * K}, hf), wt = torch::empty({K, 2 * N}, hf);
    d.W[i] = W.data_ptr<float>();
    d.wf[i] = reinterpret_cast<uint16_t*>(wf.data_ptr());
    d.wt[i] = reinterpret_cast<uint16_t*>(wt.data_ptr());
    d.N[i] = (int)N;
    d.K[i] = (int)K;
    d.nv[i] = N > W.size(0) ? (int)W.size(0) : 0;
    d.start[i] = tiles;
    d.roff[i] = off;
    tiles += (int)((N / 64) * (K / 64));
    out.push_back({wf, wt, rc.narrow(0, off, N).view({N, 1}), rc.narrow(0, off + N, K).view({K, 1})});
    off += N + K;
  }
  d.start[d.n] = tiles;
  c10::hip::HIPGuardMasqueradingAsCUDA guard(Ws[0].device());
  hx_split_weight_f16(d, rc.data_ptr<float>(), rc_floats, cur_stream(Ws[0]));
  return out;
}

// A is fp32 [M, K], or its fp16 P2 pieces [M, 2K] split at the row scales of aa (split_rows_f16,
// or a fused producer): then the kernel reads them as they are (no split in the k loop)
static HxGemmF16 f16_args(const Tensor& a, const Tensor& aa, const Tensor& b, const Tensor& ba, const char* what) {
  const bool pieces = a.scalar_type() == torch::kHalf;
  if (pieces) {
    TORCH_CHECK(a.is_cuda() && a.dim() == 2 && a.stride(1) == 1 && a.size(1) % 32 == 0 && a.stride(0) % 8 == 0 &&
                    aligned16(a.data_ptr()) && a.size(0) < (1LL << 31) && aa.dim() == 2,
                what, ": fp16 A pieces [M, 2K] (K % 16 == 0, 16-B rows) with per-row max |x| partials");
  } else {
    check_af32(a, what);
  }
  const int64_t K = pieces ? a.size(1) / 2 : a.size(1);
  check_p2(b, K, what);
  TORCH_CHECK(b.device() == a.device() && b.size(0) < (1LL << 31), what, ": operands on one device");
  const ScaleSrc sa = scale_src(aa, b, a.size(0), what), sb = scale_src(ba, b, b.size(0), what);
  HxGemmF16 p{};
  p.A = a.data_ptr();
  p.lda = pieces ? a.stride(0) / 2 : a.stride(0);
  p.apieces = pieces ? 1 : 0;
  p.a_amax = sa.p;
  p.na = sa.np;
  p.a_rs = sa.rs;
  p.B = reinterpret_cast<const uint16_t*>(b.data_ptr());
  p.ldb = b.size(1);
  p.b_amax = sb.p;
  p.nb = sb.np;
  p.b_rs = sb.rs;
  p.M = (int)a.size(0);
  p.N = (int)b.size(0);
  p.K = (int)K;
  p.ks = 1;
  return p;
}
inline void check_vec(const OptT& v, int64_t n, const char* what) {
  if (!has(v)) return;
  check_f32(*v, what);
  TORCH_CHECK(v->numel() == n && v->is_contiguous() && aligned16(v->data_ptr()), what, ": fp32 [N], 16-B aligned");
}

// C (+)= a . b^T (+ bias); ks split-K slabs (0 = plan: deep reductions with few output tiles),
// combined (with the beta / bias epilogue) by one pass over the slabs
Tensor gemm_f16(Tensor a, Tensor a_amax, Tensor b, Tensor b_amax, OptT out_, bool beta, OptT bias, int64_t ks) {
  HxGemmF16 p = f16_args(a, a_amax, b, b_amax, "gemm_f16");
  check_vec(bias, p.N, "gemm_f16 bias");
  const int cfg = hx_gemm_f16_plan(p.M, p.N, p.K);
  TORCH_CHECK(cfg >= 0, "gemm_f16: no tile for N = ", p.N);
  TORCH_CHECK(!beta || has(out_), "gemm_f16: beta needs an output to accumulate into");
  if (ks <= 0) ks = hx_gemm_f16_ks(p.M, p.N, p.K, cfg);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(a.device());
  auto f32 = a.options().dtype(torch::kFloat32);
  Tensor out = has(out_) ? *out_ : torch::empty({p.M, p.N}, f32);
  TORCH_CHECK(out.scalar_type() == torch::kFloat32 && out.dim() == 2 && out.size(0) == p.M && out.size(1) == p.N &&
                  out.stride(1) == 1 && out.stride(0) % 4 == 0 && aligned16(out.data_ptr()),
              "gemm_f16: out must be fp32 [M, N] with unit column stride and 16-B rows");
  if (ks > 1) {
    Tensor part = torch::empty({ks, p.M, p.N}, f32);
    p.C = part.data_ptr<float>();
    p.ldc = p.N;
    p.ks = (int)ks;
    p.c_zs = (int64_t)p.M * p.N;
    TORCH_CHECK(hx_gemm_f16(p, cfg, cur_stream(a)) == 0, "gemm_f16: split-K launch failed (ks must divide K / 16)");
    hx_gemm_f16_slab_combine(part.data_ptr<float>(), out.data_ptr<float>(), out.stride(0), p.M, p.N, (int)ks,
                             beta ? 1 : 0, ptr_or_null<float>(bias), cur_stream(a));
    dbg_finite(out, "gemm_f16");
    return out;
  }
  p.C = out.data_ptr<float>();
  p.ldc = out.stride(0);
  p.beta = beta ? 1 : 0;
  p.bias = ptr_or_null<float>(bias);
  TORCH_CHECK(hx_gemm_f16(p, cfg, cur_stream(a)) == 0, "gemm_f16: launch failed");
  dbg_finite(out, "gemm_f16");
  return out;
}

// FFN up: u = a . b^T + bias -> (gelu'(u) if dmode else u, h = gelu(u) fp32, max |h| per (row, N
// tile) [M, TN] -- h's per-row scale source for the FFN-down GEMM --, max |h| per (M tile, column)
// [TM, N] -- h's column maxima for the FFN-down weight gradient)
std::vector<Tensor> gemm_f16_gelu(Tensor a, Tensor a_amax, Tensor b, Tensor b_amax, OptT bias, int64_t dmode) {
  HxGemmF16 p = f16_args(a, a_amax, b, b_amax, "gemm_f16_gelu");
  check_vec(bias, p.N, "gemm_f16_gelu bias");
  const int cfg = hx_gemm_f16_plan(p.M, p.N, p.K);
  TORCH_CHECK(cfg >= 0, "gemm_f16_gelu: no tile for N = ", p.N);
  auto f32 = a.options().dtype(torch::kFloat32);
  Tensor c = torch::empty({p.M, p.N}, f32), h = torch::empty({p.M, p.N}, f32);
  Tensor rm = torch::empty({p.M, hx_gemm_f16_tn(p.N, cfg)}, f32), cm = torch::empty({hx_gemm_f16_tm(p.M, cfg), p.N}, f32);
  p.kind = 1;
  p.C = c.data_ptr<float>();
  p.ldc = p.N;
  p.bias = ptr_or_null<float>(bias);
  p.P = h.data_ptr<float>();
  p.ldp = p.N;
  p.rowmax = rm.data_ptr<float>();
  p.colmax = cm.data_ptr<float>();
  p.dmode = dmode ? 1 : 0;
  c10::hip::HIPGuardMasqueradingAsCUDA guard(a.device());
  TORCH_CHECK(hx_gemm_f16(p, cfg, cur_stream(a)) == 0, "gemm_f16_gelu: launch failed");
  dbg_finite(h, "gemm_f16_gelu");
  return {c, h, rm, cm};
}

// FFN down data gradient + GELU backward: t = (a . b^T) * (dmode ? u : gelu'(u + bias)) ->
// (t fp32, max |t| per (row, N tile) [M, TN], max |t| per (M tile, column) [TM, N], dbias =
// column sums of t (into dbias_out when given))
std::vector<Tensor> gemm_f16_dgelu(Tensor a, Tensor a_amax, Tensor b, Tensor b_amax, Tensor u, OptT bias,
                                   OptT dbias_out, int64_t dmode) {
  TORCH_CHECK(!dmode || !has(bias), "gemm_f16_dgelu: dmode 1 takes gelu'(u), which has the bias in it");
  HxGemmF16 p = f16_args(a, a_amax, b, b_amax, "gemm_f16_dgelu");
  check_vec(bias, p.N, "gemm_f16_dgelu bias");
  check_f32(u, "gemm_f16_dgelu u");
  TORCH_CHECK(u.dim() == 2 && u.size(0) == p.M && u.size(1) == p.N && u.is_contiguous() && aligned16(u.data_ptr()),
              "gemm_f16_dgelu: u must be fp32 [M, N]");
  const int cfg = hx_gemm_f16_plan(p.M, p.N, p.K);
  TORCH_CHECK(cfg >= 0, "gemm_f16_dgelu: no tile for N = ", p.N);
  const int prow = hx_gemm_f16_colpart_rows(p.M, cfg);
  auto f32 = a.options().dtype(torch::kFloat32);
  Tensor t = torch::empty({p.M, p.N}, f32);
  Tensor rm = torch::empty({p.M, hx_gemm_f16_tn(p.N, cfg)}, f32), cm = torch::empty({hx_gemm_f16_tm(p.M, cfg), p.N}, f32);
  Tensor part = torch::empty({prow, p.N}, f32);
  Tensor db = has(dbias_out) ? *dbias_out : torch::empty({p.N}, f32);
  TORCH_CHECK(db.numel() == p.N && db.scalar_type() == torch::kFloat32 && db.is_contiguous(), "gemm_f16_dgelu: dbias");
  p.kind = 2;
  p.bias = ptr_or_null<float>(bias);
  p.aux = u.data_ptr<float>();
  p.ldaux = p.N;
  p.P = t.data_ptr<float>();
  p.ldp = p.N;
  p.colpart = part.data_ptr<float>();
  p.rowmax = rm.data_ptr<float>();
  p.colmax = cm.data_ptr<float>();
  p.dmode = dmode ? 1 : 0;
  c10::hip::HIPGuardMasqueradingAsCUDA guard(a.device());
  TORCH_CHECK(hx_gemm_f16(p, cfg, cur_stream(a)) == 0, "gemm_f16_dgelu: launch failed");
  hx_fold_cols(part.data_ptr<float>(), prow, p.N, db.data_ptr<float>(), 0, cur_stream(a));
  dbg_finite(t, "gemm_f16_dgelu");
  return {t, rm, cm, db};
}

// ------------------------------------------------------------------ 8-bit blocks (quant8.hip, gemm_fp8.hip)
inline int64_t blocks128(int64_t n) { return (n + 127) / 128; }
inline void check_bias8(const OptT& b, int64_t N, const Tensor& like, const char* what) {
  if (!has(b)) return;
  check_f32(*b, what);
  TORCH_CHECK(b->numel() == N && b->device() == like.device(), what, ": fp32 [N] on the tensor's device");
}
// a bias of any stride, one after the other
inline OptT bias8(const OptT& b, int64_t N, const Tensor& like, const char* what) {
  const OptT d = has(b) && !b->is_contiguous() ? OptT(b->contiguous()) : b;
  check_bias8(d, N, like, what);
  return d;
}
inline void check_rows8(const Tensor& x, const char* what) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && (x.stride(1) == 1 || x.size(1) == 1) && (x.stride(0) >= x.size(1) || x.size(0) <= 1),
              what, ": a 2-D GPU tensor with unit column stride");
  act_bf16(x);
  // (a launch has fewer than 2^32 threads, 512 of them to a tile of 128 x 128)
  TORCH_CHECK(x.size(0) < (1LL << 31) - 128 && x.size(1) >= 1 && x.size(1) <= (1LL << 22) &&
                  blocks128(x.size(0)) * blocks128(x.size(1)) < (1LL << 22),
              what, ": fewer than 2^31 rows of 1 .. 2^22 columns, and fewer than 2^22 blocks of 128 x 128");
}
inline Tensor scale_words(int64_t rows, int64_t cols, const Tensor& like) {
  // one byte per row and block of 128; four blocks of a row to a word, rows rounded up to 4
  return torch::empty({(blocks128(cols) + 3) / 4, (rows + 3) / 4 * 4, 4}, like.options().dtype(torch::kUInt8));
}

static HxSplit8 split8_job(const Tensor& x, uint8_t* q, uint8_t* s, uint8_t* qt, uint8_t* st, float* colpart) {
  HxSplit8 j{};
  j.bf16 = act_bf16(x);
  j.x = x.data_ptr();
  j.R = (int)x.size(0);
  j.C = (int)x.size(1);
  j.ld = x.size(0) > 1 ? x.stride(0) : x.size(1);
  j.q = q;
  j.s = s;
  j.qt = qt;
  j.st = st;
  j.colpart = colpart;
  return j;
}

// x [R, C] -> (q, s, qt, st, sum): its e4m3 codes blocked along the columns (by_rows) and transposed,
// blocked along the rows (by_cols), and its fp32 column sums (sum_out / want_sum); undefined where
// not wanted
std::vector<OptT> split8(Tensor x, bool by_rows, bool by_cols, bool want_sum, OptT sum_out) {
  check_rows8(x, "split8");
  const int64_t R = x.size(0), C = x.size(1);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  auto u8 = x.options().dtype(torch::kUInt8);
  auto f32 = x.options().dtype(torch::kFloat32);
  OptT q, s, qt, st, sum;
  if (by_rows) {
    q = torch::empty({R, blocks128(C) * 128}, u8);
    s = scale_words(R, C, x);
  }
  if (by_cols) {
    TORCH_CHECK(R <= (1LL << 22), "split8: at most 2^22 rows blocked along the rows");
    qt = torch::empty({C, blocks128(R) * 128}, u8);
    st = scale_words(C, R, x);
  }
  Tensor part;
  if (want_sum) {
    sum = has(sum_out) ? *sum_out : torch::empty({C}, f32);
    check_f32(*sum, "split8 column sums");
    TORCH_CHECK(sum->numel() == C && sum->device() == x.device(), "split8: column sums [C]");
    if (R == 0) sum->zero_();
    else part = hx_split8_row_tiles(R) == 1 ? *sum : torch::empty({hx_split8_row_tiles(R), C}, f32);   // one tile's sums are the sums
  }
  if (R > 0 && (by_rows || by_cols || want_sum)) {
    const HxSplit8 job = split8_job(x, ptr_or_null<uint8_t>(q), ptr_or_null<uint8_t>(s), ptr_or_null<uint8_t>(qt),
                                    ptr_or_null<uint8_t>(st), want_sum ? part.data_ptr<float>() : nullptr);
    hx_split8(&job, 1, cur_stream(x));
    if (want_sum && hx_split8_row_tiles(R) > 1)
      hx_fold_cols(part.data_ptr<float>(), hx_split8_row_tiles(R), (int)C, sum->data_ptr<float>(), 0, cur_stream(x));
  }
  return {q, s, qt, st, sum};
}

// every weight's codes, one launch: [(q, s, qt, st)] as split8 makes them (by_cols: qt and st, else undefined)
std::vector<std::vector<OptT>> split8_weights(std::vector<Tensor> Ws, bool by_cols) {
  TORCH_CHECK(!Ws.empty() && Ws.size() <= HX_WBATCH, "split8_weights: 1..64 weights");
  HxSplit8Batch d{};
  d.n = (int)Ws.size();
  std::vector<std::vector<OptT>> out;
  c10::hip::HIPGuardMasqueradingAsCUDA guard(Ws[0].device());
  auto u8 = Ws[0].options().dtype(torch::kUInt8);
  int64_t tiles = 0;
  for (int i = 0; i < d.n; ++i) {
    const Tensor& W = Ws[i];
    check_rows8(W, "split8_weights");
    check_f32(W, "split8_weights");
    TORCH_CHECK(W.size(0) >= 1 && W.size(0) <= (1LL << 22) && aligned16(W.data_ptr()) && W.device() == Ws[0].device(),
                "split8_weights: contiguous fp32 [1 .. 2^22, K] weights with 16-B aligned storage on one device");
    const int64_t N = W.size(0), K = W.size(1);
    std::vector<OptT> w{torch::empty({N, blocks128(K) * 128}, u8), scale_words(N, K, W), c10::nullopt, c10::nullopt};
    if (by_cols) {
      w[2] = torch::empty({K, blocks128(N) * 128}, u8);
      w[3] = scale_words(K, N, W);
    }
    d.W[i] = W.data_ptr<float>();
    d.q[i] = ptr_or_null<uint8_t>(w[0]);
    d.s[i] = ptr_or_null<uint8_t>(w[1]);
    d.qt[i] = ptr_or_null<uint8_t>(w[2]);
    d.st[i] = ptr_or_null<uint8_t>(w[3]);
    out.push_back(std::move(w));
    d.R[i] = (int)N;
    d.C[i] = (int)K;
    d.start[i] = (int)tiles;
    tiles += blocks128(N) * blocks128(K);
    TORCH_CHECK(tiles < (1LL << 23), "split8_weights: too many tiles");
  }
  d.start[d.n] = (int)tiles;
  hx_split8_many(d, cur_stream(Ws[0]));
  return out;
}

// memory for the call alone, without a tensor around it (0.5 us instead of 1.3): returned to the stream's
// allocator when it goes out of scope, as a tensor's would be
struct Scratch8 {
  c10::DataPtr p;
  explicit Scratch8(int64_t bytes) { if (bytes) p = c10::hip::HIPCachingAllocator::get()->allocate((size_t)bytes); }
  uint8_t* get() const { return static_cast<uint8_t*>(p.get()); }
};
inline int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

// the tile, the split and the bytes of slabs of a product [M, N] over K
struct Plan8 {
  int cfg = 0, ks = 1;
  int64_t bytes = 0;
  Plan8() = default;
  Plan8(int64_t M, int64_t N, int64_t K, bool out_bf16) {
    // a tile's rows of codes and an operand's scale words lie within one buffer descriptor each
    const int64_t groups = (blocks128(K) + 3) / 4, most = 1LL << 31;
    TORCH_CHECK(K <= (1LL << 22) && std::max(M, N) < most - 256 && (std::max(M, N) + 3) / 4 * groups * 16 < most,
                "gemm_fp8: at most 2^22 deep, fewer than 2^31 rows and bytes of scale words (rows / 4 x depth / 512 x 16)");
    hx_gemm_fp8_plan((int)M, (int)N, (int)blocks128(K), out_bf16 ? 0 : 1, &cfg, &ks);
    bytes = ks > 1 ? up256(ks * M * N * 4) : 0;
  }
};
// out [M, N] (fp32 or bf16, unit column stride) (+)= A . B^T (+ bias) from split8's codes and scale words;
// slabs: the plan's bytes; with `fin`, the sum over a split reduction's slabs is left to it
static void gemm8_run(const Plan8& plan, uint8_t* slabs, const uint8_t* a, const uint8_t* as, int64_t M, const uint8_t* b, const uint8_t* bs,
                      int64_t N, int64_t K, const Tensor& out, bool beta, const float* bias, HxFinish* fin = nullptr) {
  const bool out_bf16 = out.scalar_type() == torch::kBFloat16;
  const int es = out_bf16 ? 2 : 4;
  HxGemm8 g{};
  g.A = a;
  g.sa = reinterpret_cast<const uint32_t*>(as);
  g.B = b;
  g.sb = reinterpret_cast<const uint32_t*>(bs);
  g.lda = g.ldb = blocks128(K) * 128;
  g.C = out.data_ptr();
  g.ldc = M > 1 ? out.stride(0) : N;
  g.bias = bias;
  g.M = (int)M;
  g.N = (int)N;
  g.nkb = (int)blocks128(K);
  g.beta = beta ? 1 : 0;
  g.ks = plan.ks;
  const int cfg = plan.cfg;
  // 16-B stores, and a tile's 256 rows within one buffer descriptor
  g.vec = aligned16(g.C) && g.ldc * es % 16 == 0 && N * es % 16 == 0 && 256 * g.ldc * es < (1LL << 31);
  const hipStream_t stream = cur_stream(out);
  if (g.ks > 1) {
    float* part = reinterpret_cast<float*>(slabs);
    HxGemm8 p = g;
    p.C = part;
    p.ldc = N;
    p.c_zs = M * N;
    p.bias = nullptr;
    p.beta = 0;
    p.vec = N % 4 == 0 && 1024 * N < (1LL << 31);
    TORCH_CHECK(hx_gemm_fp8(p, cfg, out_bf16 ? 0 : 1, 0, stream) == 0, "gemm_fp8: split-K launch failed");
    HxFinish own{};
    HxFinish& f = fin ? *fin : own;
    f.slabs[f.n++] = HxSlabs{part, g.C, g.ldc, g.bias, g.M, g.N, g.ks, g.beta, N % 4 == 0 && aligned16(g.C) && g.ldc % 4 == 0, out_bf16};
    if (!fin) hx_fp8_finish(f, stream);
  } else {
    TORCH_CHECK(hx_gemm_fp8(g, cfg, out_bf16 ? 0 : 1, out_bf16 ? 1 : 0, stream) == 0, "gemm_fp8: launch failed");
  }
}

// C [M, N] (+)= A . B^T (+ bias) on split8's codes: A (q, s) of an [M, K] operand, B of an [N, K] one.
// bf16 results on the scaled e4m3 instructions, fp32 results on decoded bf16 ones (gemm_fp8.hip).
Tensor gemm_fp8(Tensor a, Tensor as, Tensor b, Tensor bs, int64_t K, bool out_bf16, OptT out_, bool beta, OptT bias) {
  const int64_t M = a.size(0), N = b.size(0), nkb = blocks128(K);
  auto operand = [&](const Tensor& q, const Tensor& s, const char* what) {
    TORCH_CHECK(q.is_cuda() && q.scalar_type() == torch::kUInt8 && q.dim() == 2 && q.is_contiguous() && aligned16(q.data_ptr()) &&
                    q.size(1) == nkb * 128 && q.size(0) < (1LL << 31) - 256 && q.size(1) <= (1LL << 22) && q.device() == a.device(), what,
                ": codes [rows, K rounded up to 128] on one device");
    TORCH_CHECK(s.is_cuda() && s.scalar_type() == torch::kUInt8 && s.is_contiguous() && aligned16(s.data_ptr()) && s.device() == a.device() &&
                    s.numel() == (nkb + 3) / 4 * ((q.size(0) + 3) / 4 * 4) * 4 && s.numel() < (1LL << 31), what, ": scale words");
  };
  TORCH_CHECK(K >= 1, "gemm_fp8: an empty reduction");
  operand(a, as, "gemm_fp8 a");
  operand(b, bs, "gemm_fp8 b");
  bias = bias8(bias, N, a, "gemm_fp8 bias");
  TORCH_CHECK(!beta || has(out_), "gemm_fp8: beta needs an output to accumulate into");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(a.device());
  const auto dt = out_bf16 ? torch::kBFloat16 : torch::kFloat32;
  Tensor out = has(out_) ? *out_ : torch::empty({M, N}, a.options().dtype(dt));
  TORCH_CHECK(out.scalar_type() == dt && out.device() == a.device() && out.dim() == 2 && out.size(0) == M && out.size(1) == N &&
                  (out.stride(1) == 1 || N == 1) && (M <= 1 || out.stride(0) >= N),
              "gemm_fp8: out must be [M, N] of the result type with unit column stride");
  if (M == 0 || N == 0) return out;
  const Plan8 plan(M, N, K, out_bf16);
  const Scratch8 slabs(plan.bytes);
  gemm8_run(plan, slabs.get(), a.data_ptr<uint8_t>(), as.data_ptr<uint8_t>(), M, b.data_ptr<uint8_t>(), bs.data_ptr<uint8_t>(), N, K, out, beta,
            ptr_or_null<float>(bias));
  dbg_finite(out, "gemm_fp8");
  return out;
}

// codes and scale words of an operand [rows, n] inside a workspace
struct Codes8 {
  int64_t rows, n, qb, sb;   // bytes of the codes and of the scale words, 256-B steps
  Codes8(int64_t rows_, int64_t n_, bool on = true)
      : rows(rows_), n(n_), qb(on ? up256(rows_ * blocks128(n_) * 128) : 0), sb(on ? up256((blocks128(n_) + 3) / 4 * ((rows_ + 3) / 4) * 16) : 0) {}
  int64_t bytes() const { return qb + sb; }
  uint8_t* q(uint8_t* base) const { return bytes() ? base : nullptr; }
  uint8_t* s(uint8_t* base) const { return bytes() ? base + qb : nullptr; }
};

// x [M, K] W^T (+ bias) from W's codes; with `keep`, also x's codes blocked along the rows (the weight
// gradient's operand).  Small products that need no such copy go through one launch (fp8_rows_k).
static Tensor linear_fp8_y(const Tensor& x2, const Tensor& wq, const Tensor& ws, const OptT& b, bool keep, OptT* qt, OptT* st) {
  const int64_t M = x2.size(0), K = x2.size(1), N = wq.size(0);
  if (!keep && M > 0) {
    check_rows8(x2, "linear_fp8");
    TORCH_CHECK(wq.is_cuda() && wq.device() == x2.device() && wq.size(1) == blocks128(K) * 128 && wq.is_contiguous() && aligned16(wq.data_ptr()) &&
                    ws.numel() == (blocks128(K) + 3) / 4 * ((N + 3) / 4 * 4) * 4, "linear_fp8: the weight's codes do not fit x");
    const OptT bias = bias8(b, N, x2, "linear_fp8 bias");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(x2.device());
    const int bf16 = act_bf16(x2);
    Tensor y = torch::empty({M, N}, x2.options());
    if (hx_fp8_rows_fit(M, N, blocks128(K), bf16)) {
      HxRows8 g{};
      g.x = x2.data_ptr();
      g.ldx = M > 1 ? x2.stride(0) : K;
      g.B = wq.data_ptr<uint8_t>();
      g.ldb = wq.size(1);
      g.sb = reinterpret_cast<const uint32_t*>(ws.data_ptr());
      g.y = y.data_ptr();
      g.bias = ptr_or_null<float>(bias);
      g.M = (int)M;
      g.N = (int)N;
      g.K = (int)K;
      g.nkb = (int)blocks128(K);
      TORCH_CHECK(hx_fp8_rows(g, bf16, cur_stream(x2)) == 0, "linear_fp8: launch failed");
    } else {
      const Plan8 plan(M, N, K, bf16);
      const Codes8 cx(M, K);
      const Scratch8 tmp(cx.bytes() + plan.bytes);
      uint8_t* px = tmp.get();
      const HxSplit8 job = split8_job(x2, cx.q(px), cx.s(px), nullptr, nullptr, nullptr);
      hx_split8(&job, 1, cur_stream(x2));
      gemm8_run(plan, px + cx.bytes(), cx.q(px), cx.s(px), M, wq.data_ptr<uint8_t>(), ws.data_ptr<uint8_t>(), N, K, y, false, ptr_or_null<float>(bias));
    }
    dbg_finite(y, "linear_fp8");
    return y;
  }
  std::vector<OptT> c = split8(x2, true, keep, false, c10::nullopt);
  if (keep) {
    *qt = c[2];
    *st = c[3];
  }
  return gemm_fp8(*c[0], *c[1], wq, ws, K, x2.scalar_type() == torch::kBFloat16, c10::nullopt, false, b);
}
// [.., K] -> [rows, K] with unit column stride (a contiguous copy if it has none)
static Tensor as_rows8(const Tensor& x) {
  Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  const bool ok = (x2.stride(1) == 1 || x2.size(1) == 1) && (x2.stride(0) >= x2.size(1) || x2.size(0) <= 1);
  return ok ? x2 : x2.contiguous();
}

// forward alone, for the autograd functions of the Python layer: (y, x's kept codes, their scales)
std::vector<OptT> linear_fp8_fwd(Tensor x2, Tensor wq, Tensor ws, OptT bias, bool keep) {
  OptT qt, st;
  Tensor y = linear_fp8_y(x2, wq, ws, bias, keep, &qt, &st);
  return {y, qt, st};
}

// A gradient that is captured into a graph for a leaf whose accumulator was made on another stream (an
// eager graph of the same leaf is alive): autograd would make that stream wait for the capturing one,
// which a capture cannot hold and which ends the process.  Refused before it comes to that.
static void refuse_stale_leaves(const Tensor& like, const std::string& what) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(cur_stream(like), &st) != hipSuccess || st == hipStreamCaptureStatusNone) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  for (const auto& e : node->next_edges()) {
    if (!e.function || !dynamic_cast<torch::autograd::AccumulateGrad*>(e.function.get())) continue;
    const auto s = e.function->stream();
    TORCH_CHECK(!s || s->id() == c10::hip::getCurrentHIPStream(like.get_device()).id(), what,
                ": a captured backward needs its leaves' eager graphs released first (one of them lives on another stream)");
  }
}
static void refuse_tangent(const OptT& t, const char* what) {
  TORCH_CHECK(!has(t) || !t->_fw_grad(/*level=*/0).defined(), what, ": no forward-mode derivatives (an argument is a dual tensor)");
}
static void refuse_second_derivative(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": first derivatives only (create_graph=True is not supported)");
}

// The whole layer as one autograd node for parameters that autograd accumulates itself (no flat gradient
// slots, no residual mailbox).  A small layer's step is bound by the host: a node in C++ runs its
// backward without the interpreter lock, all of a direction's codes share one workspace, and x and W
// are split in one launch (training step of 41 x 1024 x 1024: 164 us of host through Python and single
// calls).
struct LinearFp8 : public torch::autograd::Function<LinearFp8> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, Tensor x, OptT W, OptT b, OptT wq, OptT ws, OptT wqt, OptT wst,
                        bool grad) {
    const bool own = !has(wq);   // W's codes are made here
    const int64_t K = x.size(-1), N = own ? W->size(0) : wq->size(0);
    Tensor x2 = as_rows8(x);
    const int64_t M = x2.size(0);
    const bool keep = grad && has(W) && W->requires_grad(), wt = grad && x.requires_grad();
    const OptT bias = bias8(b, N, x2, "linear_fp8 bias");   // (no gradient is recorded here: apply() turns it off)
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = N;
    Tensor y, kept, wtq, wts;   // what the backward needs: x's codes; the codes of W^T and their scales
    if (wt && !own) {
      wtq = wqt.value_or(Tensor());
      wts = wst.value_or(Tensor());
    }
    if (!own && !keep) {
      y = linear_fp8_y(x2, *wq, *ws, bias, false, nullptr, nullptr);
    } else {
      check_rows8(x2, "linear_fp8");
      Tensor W2 = own ? as_rows8(*W) : Tensor();
      if (own) check_rows8(W2, "linear_fp8 weight");
      TORCH_CHECK(!keep || M <= (1LL << 22), "linear_fp8: at most 2^22 rows in a training step");
      TORCH_CHECK(!own || N <= (1LL << 22), "linear_fp8: at most 2^22 output features");
      c10::hip::HIPGuardMasqueradingAsCUDA guard(x2.device());
      const auto u8 = x2.options().dtype(torch::kUInt8);
      const Codes8 cx(M, K), cxt(K, M, keep), cw(N, K, own);
      const Plan8 plan = M > 0 ? Plan8(M, N, K, x2.scalar_type() == torch::kBFloat16) : Plan8();
      const Scratch8 tmp(cx.bytes() + cw.bytes() + plan.bytes);
      if (keep && M > 0) kept = torch::empty({cxt.bytes()}, u8);
      if (own && wt) {
        // of the shapes that an Fp8Weight has: a checkpointed segment may run with one and be recomputed
        // without it, and what is saved has to match
        wtq = torch::empty({K, blocks128(N) * 128}, u8);
        wts = scale_words(K, N, x2);
      }
      uint8_t *px = tmp.get(), *pw = px + cx.bytes(), *slabs = pw + cw.bytes();
      uint8_t* pk = kept.defined() ? kept.data_ptr<uint8_t>() : nullptr;
      uint8_t* pt = own && wt ? wtq.data_ptr<uint8_t>() : nullptr;
      HxSplit8 jobs[2];
      int n = 0;
      if (M > 0) jobs[n++] = split8_job(x2, cx.q(px), cx.s(px), cxt.q(pk), pk ? cxt.s(pk) : nullptr, nullptr);
      if (own) jobs[n++] = split8_job(W2, cw.q(pw), cw.s(pw), pt, pt ? wts.data_ptr<uint8_t>() : nullptr, nullptr);
      if (n) hx_split8(jobs, n, cur_stream(x2));
      y = torch::empty({M, N}, x2.options());
      if (M > 0) {
        if (!own)
          TORCH_CHECK(wq->is_cuda() && wq->device() == x2.device() && wq->size(1) == blocks128(K) * 128 && wq->is_contiguous(),
                      "linear_fp8: the weight's codes do not fit x");
        gemm8_run(plan, slabs, cx.q(px), cx.s(px), M, own ? cw.q(pw) : wq->data_ptr<uint8_t>(), own ? cw.s(pw) : ws->data_ptr<uint8_t>(), N, K, y,
                  false, ptr_or_null<float>(bias));
        dbg_finite(y, "linear_fp8");
      }
    }
    ctx->save_for_backward({kept, wtq, wts});
    // in one list: N, whether W is bf16, the edges of W and b (the inputs that are there have the first
    // edges, in order), then x's shape
    std::vector<int64_t> kept_ints{N, has(W) && W->scalar_type() == torch::kBFloat16, has(W) ? 1 : 0, has(b) ? (has(W) ? 2 : 1) : 0};
    kept_ints.insert(kept_ints.end(), x.sizes().begin(), x.sizes().end());
    ctx->saved_data["ints"] = std::move(kept_ints);
    if (x.dim() == 2) return y;
    return y.view(shape);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    refuse_second_derivative("linear_fp8");
    refuse_stale_leaves(g[0], "linear_fp8");
    const auto saved = ctx->get_saved_variables();
    const auto ints = ctx->saved_data["ints"].toIntVector();
    const int64_t N = ints[0], K = ints.back(), ew = ints[2], eb = ints[3];
    const c10::IntArrayRef xshape = c10::IntArrayRef(ints).slice(4);
    const bool need_x = ctx->needs_input_grad(0), need_w = ew && ctx->needs_input_grad(ew), need_b = eb && ctx->needs_input_grad(eb);
    Tensor dy = as_rows8(g[0]);
    check_rows8(dy, "linear_fp8 output gradient");
    const int64_t M = dy.size(0);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(dy.device());
    const auto f32 = dy.options().dtype(torch::kFloat32);
    Tensor dx, dW, db;
    if (need_x) dx = torch::empty({M, K}, dy.options());
    if (need_w) dW = M > 0 ? torch::empty({N, K}, f32) : torch::zeros({N, K}, f32);
    if (need_b) db = M > 0 ? torch::empty({N}, f32) : torch::zeros({N}, f32);
    if (M > 0) {
      const Codes8 cd(M, N, need_x), cdt(N, M, need_w), cxt(K, M, need_w);
      const bool fold = need_b && hx_split8_row_tiles(M) > 1;   // (one tile's column sums are the sums)
      const int64_t part = fold ? up256(hx_split8_row_tiles(M) * N * 4) : 0;
      const Plan8 px = need_x ? Plan8(M, K, N, dy.scalar_type() == torch::kBFloat16) : Plan8();
      const Plan8 pw = need_w ? Plan8(N, K, M, false) : Plan8();
      const Scratch8 tmp(cd.bytes() + cdt.bytes() + part + pw.bytes + px.bytes);
      uint8_t *pd = tmp.get(), *pt = pd + cd.bytes(), *pp = pt + cdt.bytes(), *slabs = pp + part;
      const HxSplit8 job = split8_job(dy, cd.q(pd), cd.s(pd), cdt.q(pt), cdt.s(pt),
                                      fold ? reinterpret_cast<float*>(pp) : need_b ? db.data_ptr<float>() : nullptr);
      hx_split8(&job, 1, cur_stream(dy));
      HxFinish fin{};
      if (fold) {
        fin.part = reinterpret_cast<float*>(pp);
        fin.sum = db.data_ptr<float>();
        fin.rows = hx_split8_row_tiles(M);
        fin.cols = (int)N;
      }
      if (need_w) {
        uint8_t* pk = saved[0].data_ptr<uint8_t>();
        gemm8_run(pw, slabs, cdt.q(pt), cdt.s(pt), N, cxt.q(pk), cxt.s(pk), K, M, dW, false, nullptr, &fin);
      }
      if (need_x) {
        TORCH_CHECK(saved[1].defined(), "linear_fp8: the weight's codes were made without those of its transpose");
        gemm8_run(px, slabs + pw.bytes, cd.q(pd), cd.s(pd), M, saved[1].data_ptr<uint8_t>(), saved[2].data_ptr<uint8_t>(), K, N, dx, false, nullptr, &fin);
      }
      hx_fp8_finish(fin, cur_stream(dy));
      if (need_w) dbg_finite(dW, "linear_fp8 weight gradient");
      if (need_x) dbg_finite(dx, "linear_fp8 input gradient");
    }
    if (need_x && xshape.size() != 2) dx = dx.view(xshape);
    if (need_w && ints[1]) dW = dW.to(torch::kBFloat16);
    return {dx, dW, db, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
// Inference with a kept weight's codes (of K input features), arguments checked here: a single token's call
// is bound by the host
Tensor linear_fp8_infer(Tensor x, Tensor wq, Tensor ws, int64_t K, OptT b) {
  TORCH_CHECK_TYPE(x.scalar_type() == torch::kFloat32 || x.scalar_type() == torch::kBFloat16, "linear_fp8: an fp32 or bf16 tensor, got ",
                   x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == K, "linear_fp8: x of shape ", x.sizes(), ", the weight takes ", K, " features");
  TORCH_CHECK_VALUE(x.device() == wq.device(), "linear_fp8: x on ", x.device(), ", the weight on ", wq.device());
  if (has(b))
    TORCH_CHECK_VALUE(b->scalar_type() == torch::kFloat32 && b->dim() == 1 && b->size(0) == wq.size(0) && b->device() == x.device(),
                      "linear_fp8: the bias must be fp32 [", wq.size(0), "] on ", x.device(), ", got ", b->scalar_type(), " ", b->sizes(),
                      " on ", b->device());
  refuse_tangent(x, "linear_fp8");
  refuse_tangent(b, "linear_fp8");
  at::NoGradGuard no_grad;
  if (x.dim() == 2 && x.is_contiguous()) return linear_fp8_y(x, wq, ws, b, false, nullptr, nullptr);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = wq.size(0);
  return linear_fp8_y(as_rows8(x), wq, ws, b, false, nullptr, nullptr).view(shape);
}

// W: the parameter whose gradient is wanted (or none); w8: its codes and scales (wq, ws, wqt, wst -- the
// last two may be absent), or empty: they are made from W
Tensor linear_fp8(Tensor x, OptT W, OptT b, std::vector<OptT> w8, bool grad) {
  TORCH_CHECK(w8.empty() ? has(W) : w8.size() == 4 && has(w8[0]) && has(w8[1]), "linear_fp8: a weight or its codes and scales");
  if (w8.empty()) return LinearFp8::apply(x, W, b, OptT(), OptT(), OptT(), OptT(), grad);
  const bool wanted = grad && (x.requires_grad() || (has(W) && W->requires_grad()) || (has(b) && b->requires_grad()));
  if (!wanted) return linear_fp8_infer(x, *w8[0], *w8[1], x.size(-1), b);   // no node
  return LinearFp8::apply(x, W, b, w8[0], w8[1], w8[2], w8[3], grad);
}

// ---- int8 blocks along the last dimension (contiguous rows): codes [rows, nb, 128], scale bytes [rows, nb]
inline void check_kept(const Tensor& q, const Tensor& s, const Tensor& like, int64_t rows, int64_t N, const char* what) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == torch::kUInt8 && q.is_contiguous() && aligned16(q.data_ptr()) &&
                  q.numel() == rows * blocks128(N) * 128 && s.is_cuda() && s.scalar_type() == torch::kUInt8 && s.is_contiguous() &&
                  s.numel() == rows * blocks128(N) && q.device() == like.device() && s.device() == like.device(),
              what, ": int8 codes [rows, blocks, 128] and scale bytes [rows, blocks] on the tensor's device");
}
inline std::pair<int64_t, int64_t> rows_cols8(const Tensor& x, const char* what) {
  check_cuda(x, what);
  act_bf16(x);
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) < (1LL << 30), what, ": a last dimension of 1 .. 2^30");
  const int64_t rows = x.numel() / x.size(-1);
  TORCH_CHECK(blocks128(x.size(-1)) * ((rows + 63) / 64) < (1LL << 31), what, ": too many rows");
  return {rows, x.size(-1)};
}

// what the backward launches: 256 threads to 128 columns of a chunk of rows
inline void check_gelu8_grid(int64_t rows, int64_t N) {
  TORCH_CHECK(blocks128(N) * hx_gelu8_chunks(rows) < (1LL << 24), "bias_act(bits=8): ", rows, " rows of ", N, " are too many");
}
// (gelu(y + b), y's int8 codes and scale bytes: undefined without `keep`)
std::vector<OptT> gelu8_fwd(Tensor y, OptT b, bool keep) {
  const auto [rows, N] = rows_cols8(y, "gelu8_fwd y");
  b = bias8(b, N, y, "gelu8_fwd bias");
  if (keep) check_gelu8_grid(rows, N);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(y.device());
  Tensor out = torch::empty_like(y);
  OptT q, s;
  if (keep) {
    q = torch::empty({rows, blocks128(N), 128}, y.options().dtype(torch::kUInt8));
    s = torch::empty({rows, blocks128(N)}, y.options().dtype(torch::kUInt8));
  }
  if (rows > 0)
    hx_gelu8_fwd(act_bf16(y), y.data_ptr(), ptr_or_null<float>(b), out.data_ptr(), ptr_or_null<uint8_t>(q), ptr_or_null<uint8_t>(s), rows, (int)N,
                 cur_stream(y));
  dbg_finite(out, "gelu8_fwd");
  return {out, q, s};
}

std::vector<OptT> gelu8_bwd(Tensor dout, Tensor q, Tensor s, OptT b, bool want_db, OptT db_out) {
  const auto [rows, N] = rows_cols8(dout, "gelu8_bwd dout");
  check_kept(q, s, dout, rows, N, "gelu8_bwd");
  b = bias8(b, N, dout, "gelu8_bwd bias");
  check_gelu8_grid(rows, N);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dout.device());
  auto f32 = dout.options().dtype(torch::kFloat32);
  Tensor dy = torch::empty_like(dout);
  const int chunks = want_db ? hx_gelu8_chunks(rows) : 0;
  const Scratch8 part(chunks > 1 ? chunks * N * 4 : 0);   // (one chunk's sums are the sums)
  OptT db;
  if (want_db) {
    db = has(db_out) ? *db_out : torch::empty({N}, f32);
    check_bias8(db, N, dout, "gelu8_bwd bias gradient");
    if (rows == 0) db->zero_();
  }
  if (rows > 0)
    hx_gelu8_bwd(act_bf16(dout), dout.data_ptr(), q.data_ptr<uint8_t>(), s.data_ptr<uint8_t>(), ptr_or_null<float>(b),
                 dy.data_ptr(), chunks > 1 ? reinterpret_cast<float*>(part.get()) : ptr_or_null<float>(db), ptr_or_null<float>(db), rows, (int)N,
                 cur_stream(dout));
  dbg_finite(dy, "gelu8_bwd");
  return {dy, db};
}

// gelu(y + b) of a feed-forward layer straight to the second product's operand: (q, s, qt, st) as split8 (qt, st
// for by_cols), and y's int8 blocks (kept: codes, scale bytes)
std::vector<OptT> gelu8_split_fwd(Tensor y, OptT b, bool by_cols, bool keep) {
  check_rows8(y, "gelu8_split_fwd");
  const int64_t R = y.size(0), C = y.size(1);
  b = bias8(b, C, y, "gelu8_split_fwd bias");
  TORCH_CHECK(!by_cols || R <= (1LL << 22), "gelu8_split_fwd: at most 2^22 rows blocked along the rows");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(y.device());
  auto u8 = y.options().dtype(torch::kUInt8);
  Tensor q = torch::empty({R, blocks128(C) * 128}, u8), s = scale_words(R, C, y);
  OptT qt, st, kq, ks;
  if (by_cols) {
    qt = torch::empty({C, blocks128(R) * 128}, u8);
    st = scale_words(C, R, y);
  }
  if (keep) {
    kq = torch::empty({R, blocks128(C), 128}, u8);
    ks = torch::empty({R, blocks128(C)}, u8);
  }
  if (R > 0)
    hx_gelu8_split_fwd(split8_job(y, q.data_ptr<uint8_t>(), s.data_ptr<uint8_t>(), ptr_or_null<uint8_t>(qt), ptr_or_null<uint8_t>(st), nullptr),
                       ptr_or_null<float>(b), ptr_or_null<uint8_t>(kq), ptr_or_null<uint8_t>(ks), cur_stream(y));
  return {q, s, qt, st, kq, ks};
}

// dout gelu'(y + b) straight to the operands of the first product's gradients: (q, s) by_rows, (qt, st) by_cols, and
// the bias gradient
std::vector<OptT> gelu8_split_bwd(Tensor dout, Tensor kq, Tensor ks, OptT b, bool by_rows, bool by_cols, bool want_db, OptT db_out) {
  check_rows8(dout, "gelu8_split_bwd");
  const int64_t R = dout.size(0), C = dout.size(1);
  check_kept(kq, ks, dout, R, C, "gelu8_split_bwd");
  b = bias8(b, C, dout, "gelu8_split_bwd bias");
  TORCH_CHECK(!by_cols || R <= (1LL << 22), "gelu8_split_bwd: at most 2^22 rows blocked along the rows");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dout.device());
  auto u8 = dout.options().dtype(torch::kUInt8);
  OptT q, s, qt, st, db;
  if (by_rows) {
    q = torch::empty({R, blocks128(C) * 128}, u8);
    s = scale_words(R, C, dout);
  }
  if (by_cols) {
    qt = torch::empty({C, blocks128(R) * 128}, u8);
    st = scale_words(C, R, dout);
  }
  const int tiles = want_db ? hx_split8_row_tiles(R) : 0;
  const Scratch8 part(tiles > 1 ? tiles * C * 4 : 0);
  if (want_db) {
    db = has(db_out) ? *db_out : torch::empty({C}, dout.options().dtype(torch::kFloat32));
    check_bias8(db, C, dout, "gelu8_split_bwd bias gradient");
    if (R == 0) db->zero_();
  }
  if (R > 0 && (by_rows || by_cols || want_db)) {
    float* sums = tiles > 1 ? reinterpret_cast<float*>(part.get()) : ptr_or_null<float>(db);
    hx_gelu8_split_bwd(split8_job(dout, ptr_or_null<uint8_t>(q), ptr_or_null<uint8_t>(s), ptr_or_null<uint8_t>(qt), ptr_or_null<uint8_t>(st), sums),
                       ptr_or_null<float>(b), kq.data_ptr<uint8_t>(), ks.data_ptr<uint8_t>(), cur_stream(dout));
    if (tiles > 1) hx_fold_cols(sums, tiles, (int)C, db->data_ptr<float>(), 0, cur_stream(dout));
  }
  return {q, s, qt, st, db};
}

// bias + GELU as one autograd node (see LinearFp8)
struct BiasGelu8 : public torch::autograd::Function<BiasGelu8> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, Tensor y, OptT b) {
    std::vector<OptT> r = gelu8_fwd(y, b, true);
    ctx->save_for_backward({*r[1], *r[2], has(b) ? *b : Tensor()});
    return *r[0];
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
    refuse_second_derivative("bias_act(bits=8)");
    refuse_stale_leaves(g[0], "bias_act(bits=8)");
    const auto saved = ctx->get_saved_variables();
    const bool need_b = saved[2].defined() && ctx->needs_input_grad(1);
    std::vector<OptT> r = gelu8_bwd(g[0].contiguous(), saved[0], saved[1], saved[2].defined() ? OptT(saved[2]) : OptT(), need_b, c10::nullopt);
    return {*r[0], need_b ? *r[1] : Tensor()};
  }
};
Tensor bias_gelu8(Tensor y, OptT b) {
  const bool wanted = at::GradMode::is_enabled() && (y.requires_grad() || (has(b) && b->requires_grad()));
  return wanted ? BiasGelu8::apply(y.contiguous(), b) : *gelu8_fwd(y.contiguous(), b, false)[0];   // (no node, nothing kept)
}

std::vector<Tensor> pack8(Tensor x) {
  at::NoGradGuard no_grad;
  if (!x.is_contiguous()) x = x.contiguous();
  const auto [rows, N] = rows_cols8(x, "pack8 x");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  Tensor q = torch::empty({rows, blocks128(N), 128}, x.options().dtype(torch::kUInt8));
  Tensor s = torch::empty({rows, blocks128(N)}, x.options().dtype(torch::kUInt8));
  if (rows > 0)
    hx_pack8(act_bf16(x), x.data_ptr(), q.data_ptr<uint8_t>(), s.data_ptr<uint8_t>(), rows, (int)N, cur_stream(x));
  return {q, s};
}

// codes [rows, nb, 128] and scale bytes -> their values, a tensor of `shape`
Tensor unpack8(Tensor q, Tensor s, std::vector<int64_t> shape, bool bf16) {
  TORCH_CHECK(!shape.empty(), "unpack8: a shape of at least one dimension");
  const int64_t N = shape.back();
  TORCH_CHECK(q.dim() == 3 && N >= 1 && N < (1LL << 30) && q.size(1) == blocks128(N) && q.size(2) == 128,
              "unpack8: codes [rows, ceil(N / 128), 128]");
  const int64_t rows = q.size(0);
  check_kept(q, s, q, rows, N, "unpack8");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  Tensor x = torch::empty(shape, q.options().dtype(bf16 ? torch::kBFloat16 : torch::kFloat32));
  TORCH_CHECK(x.numel() == rows * N, "unpack8: codes of ", rows, " rows for another shape");
  if (rows > 0)
    hx_unpack8(bf16, q.data_ptr<uint8_t>(), s.data_ptr<uint8_t>(), x.data_ptr(), rows, (int)N, cur_stream(q));
  return x;
}

// the per-column scale source of a weight-gradient operand: 1-D = partials of the whole tensor (a
// per-tensor bound), 2-D [P, cols] = P partials per column; with aff = (gamma, beta) the
// LayerNorm-output bound (|gamma| z + |beta|) mul instead (t unused)
inline HxColScale col_scale_src(const Tensor& t, const Tensor& ref, int64_t cols, const char* what, const OptT& g,
                                const OptT& b, double z, double mul) {
  HxColScale c{};
  if (has(g)) {
    TORCH_CHECK(has(b), what, ": the affine bound needs gamma and beta");
    check_f32(*g, what);
    check_f32(*b, what);
    TORCH_CHECK(g->numel() == cols && b->numel() == cols && g->is_contiguous() && b->is_contiguous() &&
                    g->device() == ref.device() && b->device() == ref.device(), what, ": gamma / beta [cols]");
    c.g = g->data_ptr<float>();
    c.b = b->data_ptr<float>();
    c.z = (float)z;
    c.mul = (float)mul;
    return c;
  }
  check_f32(t, what);
  TORCH_CHECK(t.is_contiguous() && t.numel() >= 1 && t.numel() < (1LL << 31) && t.device() == ref.device(), what,
              ": max |x| partials on the operand's device");
  c.p = t.data_ptr<float>();
  if (t.dim() == 1) {
    c.np = (int)t.numel();
    return c;
  }
  TORCH_CHECK(t.dim() == 2 && t.size(1) == cols && t.size(0) >= 1 && t.size(0) <= 256, what,
              ": per-column max |x| partials must be [P <= 256, cols] (cols = ", cols, ")");
  c.np = (int)t.size(0);
  c.cs = (int)cols;
  return c;
}

// max |x| of every row and every column in one read: ([rows, 1], [1, cols]); cols <= 4096
std::vector<Tensor> amax_rows_cols(Tensor x) {
  // rows may be strided (the dQ third of a [rows, 3H] gradient)
  TORCH_CHECK(x.is_cuda() && x.scalar_type() == torch::kFloat32, "amax_rows_cols: fp32 GPU tensor");
  TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1 && x.stride(0) % 4 == 0 && x.size(1) % 4 == 0 &&
                  x.size(1) <= 4096 && aligned16(x.data_ptr()),
              "amax_rows_cols: fp32 [rows, cols <= 4096] with 16-B rows, cols % 4 == 0");
  Tensor r = torch::empty({x.size(0), 1}, x.options());
  Tensor c = torch::empty({1, x.size(1)}, x.options());
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  TORCH_CHECK(hx_amax_rows_cols(x.data_ptr<float>(), x.size(0), (int)x.size(1), x.stride(0), r.data_ptr<float>(),
                                c.data_ptr<float>(), cur_stream(x)) == 0, "amax_rows_cols: launch");
  return {r, c};
}

// max |x| of every column: [1, cols]
Tensor amax_cols(Tensor x) {
  check_f32(x, "amax_cols");
  TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1 && x.stride(0) % 4 == 0 && x.size(1) % 4 == 0 &&
                  aligned16(x.data_ptr()), "amax_cols: fp32 [rows, cols] with 16-B rows, cols % 4 == 0");
  Tensor out = torch::empty({1, x.size(1)}, x.options());
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  hx_amax_cols(x.data_ptr<float>(), x.size(0), (int)x.size(1), x.stride(0), out.data_ptr<float>(), cur_stream(x));
  return out;
}

// dW = dy^T x over the token rows: dy [T, M], x [T, N] fp32 (M, N multiples of 128); out [<= M, N]
// (rows of dy's padding columns past out.size(0) are not stored); dy_amax / x_amax: per-column
// max |x| partials of each operand ([P, M] / [P, N]) or per-tensor partials (1-D)
Tensor wgrad_f16(Tensor dy, Tensor dy_amax, Tensor x, Tensor x_amax, Tensor out, OptT x_gamma, OptT x_beta, double x_z,
                 double x_mul) {
  check_f32(dy, "wgrad_f16 dy");
  check_f32(x, "wgrad_f16 x");
  TORCH_CHECK(dy.dim() == 2 && x.dim() == 2 && dy.size(0) == x.size(0) && dy.stride(1) == 1 && x.stride(1) == 1 &&
                  dy.stride(0) % 4 == 0 && x.stride(0) % 4 == 0 && aligned16(dy.data_ptr()) &&
                  aligned16(x.data_ptr()) && dy.size(1) % 128 == 0 && x.size(1) % 128 == 0 &&
                  dy.size(0) < (1 << 30) && x.device() == dy.device(),
              "wgrad_f16: dy [T, M], x [T, N] fp32 with 16-B rows, M and N multiples of 128");
  const int64_t T = dy.size(0), M = dy.size(1), N = x.size(1);
  const HxColScale sa = col_scale_src(dy_amax, dy, M, "wgrad_f16 dy partials", OptT(), OptT(), 0, 0);
  const HxColScale sb = col_scale_src(x_amax, dy, N, "wgrad_f16 x partials", x_gamma, x_beta, x_z, x_mul);
  check_f32(out, "wgrad_f16 out");
  TORCH_CHECK(out.dim() == 2 && out.size(0) <= M && out.size(1) == N && out.is_contiguous(),
              "wgrad_f16: out must be contiguous fp32 [<= M, N]");
  int cfg = 0, nsplit = 1;
  hx_wgrad_f16_plan((int)M, (int)N, (int)T, &cfg, &nsplit);
  Tensor ws;
  if (nsplit > 1) ws = torch::empty({nsplit, M, N}, dy.options());
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dy.device());
  TORCH_CHECK(hx_wgrad_f16(dy.data_ptr<float>(), (int)dy.stride(0), sa, x.data_ptr<float>(), (int)x.stride(0), sb,
                           out.data_ptr<float>(), nsplit > 1 ? ws.data_ptr<float>() : nullptr, (int)M, (int)N, (int)T,
                           cfg, nsplit, (int)out.size(0), cur_stream(dy)) == 0,
              "wgrad_f16: launch failed");
  dbg_finite(out, "wgrad_f16");
  return out;
}

// --precision bf16 on the same kernel: out (+)= a . b^T (+ bias), a bf16 [M, K], b bf16 [N, K]
// (contiguous); the output is bf16 (out_bf16) or fp32
Tensor gemm_bf16(Tensor a, Tensor b, OptT out_, bool beta, OptT bias, bool out_bf16) {
  TORCH_CHECK(a.is_cuda() && a.scalar_type() == torch::kBFloat16 && b.scalar_type() == torch::kBFloat16 &&
                  a.dim() == 2 && b.dim() == 2 && a.stride(1) == 1 && a.stride(0) % 8 == 0 &&
                  aligned16(a.data_ptr()) && b.is_contiguous() && aligned16(b.data_ptr()) && a.size(1) == b.size(1) &&
                  a.size(1) % 32 == 0 && a.device() == b.device(),
              "gemm_bf16: a [M, K] / b [N, K] bf16 with 16-B rows, K % 32 == 0");
  HxGemmF16 p{};
  p.A = a.data_ptr();
  p.lda = a.stride(0);
  p.B = reinterpret_cast<const uint16_t*>(b.data_ptr());
  p.ldb = b.size(1);
  p.M = (int)a.size(0);
  p.N = (int)b.size(0);
  p.K = (int)a.size(1);
  p.ks = 1;
  p.abf16 = 1;
  p.obf16 = out_bf16 ? 1 : 0;
  check_vec(bias, p.N, "gemm_bf16 bias");
  const int cfg = hx_gemm_bf16_plan(p.M, p.N, p.K);
  TORCH_CHECK(cfg >= 0, "gemm_bf16: no tile for N = ", p.N);
  TORCH_CHECK(!beta || has(out_), "gemm_bf16: beta needs an output to accumulate into");
  Tensor out = has(out_) ? *out_ : torch::empty({p.M, p.N}, a.options().dtype(out_bf16 ? torch::kBFloat16
                                                                                       : torch::kFloat32));
  TORCH_CHECK(out.scalar_type() == (out_bf16 ? torch::kBFloat16 : torch::kFloat32) && out.dim() == 2 &&
                  out.size(0) == p.M && out.size(1) == p.N && out.stride(1) == 1 && out.stride(0) % 8 == 0 &&
                  aligned16(out.data_ptr()),
              "gemm_bf16: out [M, N] of the output dtype with 16-B rows");
  p.C = reinterpret_cast<float*>(out.data_ptr());
  p.ldc = out.stride(0);
  p.beta = beta ? 1 : 0;
  p.bias = ptr_or_null<float>(bias);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(a.device());
  TORCH_CHECK(hx_gemm_f16(p, cfg, cur_stream(a)) == 0, "gemm_bf16: launch failed");
  dbg_finite(out, "gemm_bf16");
  return out;
}

static HxGemmF16 bf16_args(const Tensor& a, const Tensor& b, const char* what) {
  TORCH_CHECK(a.is_cuda() && a.scalar_type() == torch::kBFloat16 && b.scalar_type() == torch::kBFloat16 &&
                  a.dim() == 2 && b.dim() == 2 && a.stride(1) == 1 && a.stride(0) % 8 == 0 &&
                  aligned16(a.data_ptr()) && b.is_contiguous() && aligned16(b.data_ptr()) && a.size(1) == b.size(1) &&
                  a.size(1) % 32 == 0 && a.device() == b.device(),
              what, ": a [M, K] / b [N, K] bf16 with 16-B rows, K % 32 == 0");
  HxGemmF16 p{};
  p.A = a.data_ptr();
  p.lda = a.stride(0);
  p.B = reinterpret_cast<const uint16_t*>(b.data_ptr());
  p.ldb = b.size(1);
  p.M = (int)a.size(0);
  p.N = (int)b.size(0);
  p.K = (int)a.size(1);
  p.ks = 1;
  p.abf16 = 1;
  p.obf16 = 1;
  return p;
}

// --precision bf16 FFN up: u = a . b^T + bias -> (gelu'(u), gelu(u)), both bf16 [M, N]
std::vector<Tensor> gemm_bf16_gelu(Tensor a, Tensor b, Tensor bias) {
  HxGemmF16 p = bf16_args(a, b, "gemm_bf16_gelu");
  check_vec(bias, p.N, "gemm_bf16_gelu bias");
  const int cfg = hx_gemm_bf16_plan(p.M, p.N, p.K);
  TORCH_CHECK(cfg >= 0, "gemm_bf16_gelu: no tile for N = ", p.N);
  Tensor d = torch::empty({p.M, p.N}, a.options()), h = torch::empty({p.M, p.N}, a.options());
  p.kind = 1;
  p.C = reinterpret_cast<float*>(d.data_ptr());
  p.ldc = p.N;
  p.bias = bias.data_ptr<float>();
  p.P = reinterpret_cast<float*>(h.data_ptr());
  p.ldp = p.N;
  p.dmode = 1;
  c10::hip::HIPGuardMasqueradingAsCUDA guard(a.device());
  TORCH_CHECK(hx_gemm_f16(p, cfg, cur_stream(a)) == 0, "gemm_bf16_gelu: launch failed");
  dbg_finite(h, "gemm_bf16_gelu");
  return {d, h};
}

// --precision bf16 FFN-down data gradient + GELU backward: t = (a . b^T) * (dmode ? d : gelu'(d + bias))
// (d: bf16 gelu'(u) from gemm_bf16_gelu, or the pre-bias u) -> (t bf16, dbias = column sums of t
// into dbias_out when given)
std::vector<Tensor> gemm_bf16_dgelu(Tensor a, Tensor b, Tensor d, OptT dbias_out, OptT bias, int64_t dmode) {
  TORCH_CHECK(!dmode || !has(bias), "gemm_bf16_dgelu: dmode 1 takes gelu'(u), which has the bias in it");
  HxGemmF16 p = bf16_args(a, b, "gemm_bf16_dgelu");
  check_vec(bias, p.N, "gemm_bf16_dgelu bias");
  TORCH_CHECK(d.scalar_type() == torch::kBFloat16 && d.dim() == 2 && d.size(0) == p.M && d.size(1) == p.N &&
                  d.is_contiguous() && aligned16(d.data_ptr()) && d.device() == a.device(),
              "gemm_bf16_dgelu: d must be bf16 [M, N]");
  const int cfg = hx_gemm_bf16_plan(p.M, p.N, p.K);
  TORCH_CHECK(cfg >= 0, "gemm_bf16_dgelu: no tile for N = ", p.N);
  const int prow = hx_gemm_f16_colpart_rows(p.M, cfg);
  auto f32 = a.options().dtype(torch::kFloat32);
  Tensor t = torch::empty({p.M, p.N}, a.options());
  Tensor part = torch::empty({prow, p.N}, f32);
  Tensor db = has(dbias_out) ? *dbias_out : torch::empty({p.N}, f32);
  TORCH_CHECK(db.numel() == p.N && db.scalar_type() == torch::kFloat32 && db.is_contiguous() && db.device() == a.device(),
              "gemm_bf16_dgelu: dbias");
  p.kind = 2;
  p.bias = ptr_or_null<float>(bias);
  p.aux = reinterpret_cast<const float*>(d.data_ptr());
  p.ldaux = p.N;
  p.P = reinterpret_cast<float*>(t.data_ptr());
  p.ldp = p.N;
  p.colpart = part.data_ptr<float>();
  p.dmode = dmode ? 1 : 0;
  c10::hip::HIPGuardMasqueradingAsCUDA guard(a.device());
  TORCH_CHECK(hx_gemm_f16(p, cfg, cur_stream(a)) == 0, "gemm_bf16_dgelu: launch failed");
  hx_fold_cols(part.data_ptr<float>(), prow, p.N, db.data_ptr<float>(), 0, cur_stream(a));
  dbg_finite(t, "gemm_bf16_dgelu");
  return {t, db};
}

// W^T in bf16 ([K, N]) of every fp32 weight W [N, K] in the list, one launch
std::vector<Tensor> weight_bf16_t(std::vector<Tensor> Ws) {
  TORCH_CHECK(!Ws.empty() && Ws.size() <= HX_WBATCH, "weight_bf16_t: 1..64 weights");
  HxWeightBatch d{};
  d.n = (int)Ws.size();
  std::vector<Tensor> out;
  int tiles = 0;
  for (int i = 0; i < d.n; ++i) {
    const Tensor& W = Ws[i];
    check_f32(W, "weight_bf16_t input");
    TORCH_CHECK(W.dim() == 2 && W.is_contiguous() && W.size(0) % 64 == 0 && W.size(1) % 64 == 0 &&
                    aligned16(W.data_ptr()) && W.device() == Ws[0].device(),
                "weight_bf16_t: every W contiguous [N, K], N and K multiples of 64, one device");
    Tensor wt = torch::empty({W.size(1), W.size(0)}, W.options().dtype(torch::kBFloat16));
    d.W[i] = W.data_ptr<float>();
    d.wt[i] = reinterpret_cast<uint16_t*>(wt.data_ptr());
    d.wf[i] = nullptr;
    d.N[i] = (int)W.size(0);
    d.K[i] = (int)W.size(1);
    d.start[i] = tiles;
    tiles += (int)((W.size(0) / 64) * (W.size(1) / 64));
    out.push_back(wt);
  }
  d.start[d.n] = tiles;
  c10::hip::HIPGuardMasqueradingAsCUDA guard(Ws[0].device());
  hx_weight_bf16_t(d, cur_stream(Ws[0]));
  return out;
}

// ------------------------------------------------------------------ xGMI all-reduce
// Contexts travel to Python as integers (owned by parallel/xgmi.py).
inline void xar_check(int rc) { TORCH_CHECK(rc == 0, hx_xar_last_error()); }
inline void* as_ctx(int64_t h) { return reinterpret_cast<void*>(static_cast<uintptr_t>(h)); }
int64_t xar_create(int64_t rank, int64_t world, int64_t nblocks, double timeout_s, int64_t oneshot_max_bytes) {
  void* c = nullptr;
  xar_check(hx_xar_create((int)rank, (int)world, (int)nblocks, timeout_s, oneshot_max_bytes, &c));
  return static_cast<int64_t>(reinterpret_cast<uintptr_t>(c));
}
void xar_register(int64_t h, Tensor buf) {
  check_f32(buf, "xGMI registered buffer");
  TORCH_CHECK(buf.is_contiguous() && aligned16(buf.data_ptr()), "xGMI registered buffer: contiguous, 16-B aligned");
  xar_check(hx_xar_register(as_ctx(h), buf.data_ptr<float>(), buf.numel()));
}
py::bytes xar_export(int64_t h) {
  char buf[kXarRecord];
  xar_check(hx_xar_export(as_ctx(h), buf));
  return py::bytes(buf, kXarRecord);
}
void xar_open(int64_t h, py::bytes recs) {
  const std::string s = recs;
  xar_check(hx_xar_open(as_ctx(h), s.data()));
}
void xar_allreduce(int64_t h, Tensor buf) {
  check_f32(buf, "all-reduce bucket");
  TORCH_CHECK(aligned16(buf.data_ptr()), "all-reduce bucket must be 16-byte aligned");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(buf.device());
  xar_check(hx_xar_allreduce(as_ctx(h), buf.data_ptr<float>(), buf.numel(), cur_stream(buf)));
}
void xar_allreduce_sim(std::vector<int64_t> hs, std::vector<Tensor> bufs, int64_t mute) {
  TORCH_CHECK(hs.size() == bufs.size() && hs.size() >= 2 && hs.size() <= 8, "1 context per simulated rank (2..8)");
  std::vector<void*> cs;
  std::vector<float*> ps;
  for (size_t i = 0; i < hs.size(); ++i) {
    check_f32(bufs[i], "bucket");
    TORCH_CHECK(bufs[i].numel() == bufs[0].numel() && aligned16(bufs[i].data_ptr()), "equal, aligned buckets");
    cs.push_back(as_ctx(hs[i]));
    ps.push_back(bufs[i].data_ptr<float>());
  }
  c10::hip::HIPGuardMasqueradingAsCUDA guard(bufs[0].device());
  TORCH_CHECK(mute >= -1 && mute < (int64_t)hs.size(), "mute must be -1 or a simulated rank");
  xar_check(hx_xar_allreduce_sim(cs.data(), ps.data(), (int)hs.size(), bufs[0].numel(), (int)mute,
                                 cur_stream(bufs[0])));
}
int64_t xar_error(int64_t h) { return hx_xar_error(as_ctx(h)); }
void xar_error_async(int64_t h, Tensor out) {
  TORCH_CHECK(out.is_cuda() && out.scalar_type() == at::kInt && out.numel() >= 1 && out.is_contiguous(),
              "error word target: contiguous int32 GPU tensor");
  c10::hip::HIPGuardMasqueradingAsCUDA guard(out.device());
  xar_check(hx_xar_error_async(as_ctx(h), out.data_ptr<int32_t>(), cur_stream(out)));
}
// PCI bus id ("dddd:bb:dd.f") of a device visible to this process: the process-independent
// identity of a GPU (local ordinals differ between processes with different visible sets)
std::string device_pci_bus_id(int64_t dev) {
  char id[64] = {0};
  TORCH_CHECK(hipDeviceGetPCIBusId(id, (int)sizeof(id), (int)dev) == hipSuccess, "hipDeviceGetPCIBusId failed");
  return std::string(id);
}
int64_t xar_oneshot_max(int64_t h) { return hx_xar_oneshot_max(as_ctx(h)); }
void xar_destroy(int64_t h) { hx_xar_destroy(as_ctx(h)); }

}  // namespace

namespace hx {
void register_reducer(py::module& m);   // csrc/native/reducer.cpp
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  hx::register_reducer(m);
  m.doc() = "hetseq_9cme_amd gfx950 (MI355X) kernels";
  m.def("grad_norm_clip", &grad_norm_clip);
  m.def("adam", &adam);
  m.def("adam_masked", &adam_masked, py::arg("p"), py::arg("g"), py::arg("m"), py::arg("v"), py::arg("shadow"),
        py::arg("gscale"), py::arg("table"), py::arg("used"), py::arg("steps"), py::arg("hp"), py::arg("lr"),
        py::arg("b1"), py::arg("b2"), py::arg("eps"), py::arg("wd"), py::arg("lr_dev") = py::none());
  m.def("adam_mask_chunk", &hx_adam_mask_chunk);
  m.def("adadelta", &adadelta);
  m.def("ln_fwd", &ln_fwd, py::arg("y"), py::arg("bias"), py::arg("res"), py::arg("gamma"), py::arg("beta"),
        py::arg("eps"), py::arg("keep_prob"), py::arg("seed"), py::arg("stream"), py::arg("drop_after"),
        py::arg("save_z"), py::arg("amax_out") = py::none(), py::arg("pieces_out") = py::none());
  m.def("ln_bwd", &ln_bwd, py::arg("dout"), py::arg("z"), py::arg("mean"), py::arg("rstd"), py::arg("gamma"),
        py::arg("keep_prob"), py::arg("seed"), py::arg("stream"), py::arg("drop_after"), py::arg("want_dy"),
        py::arg("want_dbias"), py::arg("dgamma_out"), py::arg("dbeta_out"), py::arg("dbias_out"),
        py::arg("amax_out") = py::none(), py::arg("colmax_out") = py::none(), py::arg("pieces_out") = py::none());
  m.def("ln_fwd_blocks", &hx_ln_fwd_blocks);
  m.def("ln_bwd_blocks", &hx_ln_bwd_blocks);
  m.def("embed_ln_fwd", &embed_ln_fwd, py::arg("ids"), py::arg("tt"), py::arg("wte"), py::arg("wpe"), py::arg("wtt"),
        py::arg("gamma"), py::arg("beta"), py::arg("eps"), py::arg("keep_prob"), py::arg("seed"), py::arg("stream"),
        py::arg("bf16_out"), py::arg("amax_out") = py::none(), py::arg("pieces_out") = py::none());
  m.def("embed_word_grad", &embed_word_grad);
  m.def("embed_type_grad", &embed_type_grad);
  m.def("bias_act_fwd", &bias_act_fwd);
  m.def("bias_act_bwd", &bias_act_bwd);
  m.def("colsum", &colsum);
  m.def("dropout", &dropout);
  m.def("softmax_xent_", &softmax_xent_);
  m.def("attn_fwd", [](Tensor qkv, Tensor mask_bias, int64_t nh, double keep, const Tensor& seed, int64_t stream,
                        OptT bias) { return attn_fwd(qkv, mask_bias, nh, keep, seed, stream, bias, false); });
  m.def("attn_fwd_f16", &attn_fwd_f16, py::arg("qkv"), py::arg("mask_bias"), py::arg("nh"), py::arg("keep"),
        py::arg("seed"), py::arg("stream"), py::arg("bias"), py::arg("amax_out") = py::none(),
        py::arg("colmax_out") = py::none());
  m.def("attn_bwd", [](Tensor dout, Tensor qkv, Tensor mask_bias, Tensor out, Tensor lse, Tensor dmask, int64_t nh,
                       double keep, OptT bias, OptT dbq, OptT dbk, OptT dbv, bool want_dbias) {
    return attn_bwd(dout, qkv, mask_bias, out, lse, dmask, nh, keep, bias, dbq, dbk, dbv, 0, OptT(), OptT(), want_dbias);
  }, py::arg("dout"), py::arg("qkv"), py::arg("mask_bias"), py::arg("out"), py::arg("lse"), py::arg("dmask"),
     py::arg("nh"), py::arg("keep"), py::arg("bias"), py::arg("dbq"), py::arg("dbk"), py::arg("dbv"),
     py::arg("want_dbias") = false);
  // fp32 attention backward on the fp16 matrix cores (fp16x3, attention_f16.hip)
  m.def("attn_bwd_f16", [](Tensor dout, Tensor qkv, Tensor mask_bias, Tensor out, Tensor lse, Tensor dmask, int64_t nh,
                           double keep, OptT bias, OptT dbq, OptT dbk, OptT dbv, OptT amax_out, OptT colmax_out,
                           bool want_dbias) {
    return attn_bwd(dout, qkv, mask_bias, out, lse, dmask, nh, keep, bias, dbq, dbk, dbv, 2, amax_out, colmax_out,
                    want_dbias);
  }, py::arg("dout"), py::arg("qkv"), py::arg("mask_bias"), py::arg("out"), py::arg("lse"), py::arg("dmask"),
     py::arg("nh"), py::arg("keep"), py::arg("bias"), py::arg("dbq"), py::arg("dbk"), py::arg("dbv"),
     py::arg("amax_out") = py::none(), py::arg("colmax_out") = py::none(), py::arg("want_dbias") = false);
  m.def("wgrad_bf16", &wgrad_bf16);
  m.def("wgrad_bf16_ok", &wgrad_bf16_ok);
  m.def("amax_rows", &amax_rows);
  m.def("split_rows_f16", &split_rows_f16);
  m.def("amax_cols", &amax_cols);
  m.def("amax_rows_cols", &amax_rows_cols);
  m.def("split_weight_f16", &split_weight_f16, py::arg("Ws"), py::arg("rows") = std::vector<int64_t>());
  m.def("gemm_f16", &gemm_f16, py::arg("a"), py::arg("a_amax"), py::arg("b"), py::arg("b_amax"),
        py::arg("out") = py::none(), py::arg("beta") = false, py::arg("bias") = py::none(), py::arg("ks") = 0);
  m.def("gemm_f16_gelu", &gemm_f16_gelu, py::arg("a"), py::arg("a_amax"), py::arg("b"), py::arg("b_amax"),
        py::arg("bias"), py::arg("dmode") = 1);
  m.def("gemm_f16_dgelu", &gemm_f16_dgelu, py::arg("a"), py::arg("a_amax"), py::arg("b"), py::arg("b_amax"),
        py::arg("u"), py::arg("bias") = py::none(), py::arg("dbias_out") = py::none(), py::arg("dmode") = 1);
  m.def("wgrad_f16", &wgrad_f16, py::arg("dy"), py::arg("dy_amax"), py::arg("x"), py::arg("x_amax"), py::arg("out"),
        py::arg("x_gamma") = py::none(), py::arg("x_beta") = py::none(), py::arg("x_z") = 0.0,
        py::arg("x_mul") = 1.0);
  m.def("gemm_bf16_gelu", &gemm_bf16_gelu, py::arg("a"), py::arg("b"), py::arg("bias"));
  m.def("gemm_bf16_dgelu", &gemm_bf16_dgelu, py::arg("a"), py::arg("b"), py::arg("d"),
        py::arg("dbias_out") = py::none(), py::arg("bias") = py::none(), py::arg("dmode") = 1);
  m.def("gemm_bf16", &gemm_bf16, py::arg("a"), py::arg("b"), py::arg("out") = py::none(), py::arg("beta") = false,
        py::arg("bias") = py::none(), py::arg("out_bf16") = true);
  m.def("split8", &split8, py::arg("x"), py::arg("by_rows"), py::arg("by_cols"), py::arg("want_sum") = false,
        py::arg("sum_out") = py::none());
  m.def("split8_weights", &split8_weights, py::arg("Ws"), py::arg("by_cols") = true);
  m.def("gemm_fp8", &gemm_fp8, py::arg("a"), py::arg("as"), py::arg("b"), py::arg("bs"), py::arg("K"), py::arg("out_bf16"),
        py::arg("out") = py::none(), py::arg("beta") = false, py::arg("bias") = py::none());
  m.def("linear_fp8_fwd", &linear_fp8_fwd, py::arg("x"), py::arg("wq"), py::arg("ws"), py::arg("bias"), py::arg("keep"));
  m.def("linear_fp8", &linear_fp8, py::arg("x"), py::arg("W"), py::arg("bias"), py::arg("w8"), py::arg("grad"));
  m.def("linear_fp8_infer", &linear_fp8_infer, py::arg("x"), py::arg("wq"), py::arg("ws"), py::arg("K"), py::arg("bias"));
  m.def("refuse_stale_leaves", &refuse_stale_leaves);
  m.def("bias_gelu8", &bias_gelu8, py::arg("y"), py::arg("bias"));
  m.def("gelu8_fwd", &gelu8_fwd);
  m.def("gelu8_bwd", &gelu8_bwd, py::arg("dout"), py::arg("q"), py::arg("s"), py::arg("bias"), py::arg("want_db"),
        py::arg("db_out") = py::none());
  m.def("gelu8_split_fwd", &gelu8_split_fwd, py::arg("y"), py::arg("bias"), py::arg("by_cols"), py::arg("keep"));
  m.def("gelu8_split_bwd", &gelu8_split_bwd, py::arg("dout"), py::arg("kept"), py::arg("scales"), py::arg("bias"), py::arg("by_rows"),
        py::arg("by_cols"), py::arg("want_db"), py::arg("db_out") = py::none());
  m.def("pack8", &pack8);
  m.def("unpack8", &unpack8);
  m.def("weight_bf16_t", &weight_bf16_t);

  m.def("gemm_f16_plan", &hx_gemm_f16_plan);
  m.def("gemm_f16_ks", &hx_gemm_f16_ks);
  m.def("gemm_f16_tiles", &hx_gemm_f16_tiles);
  m.def("wgrad_f16_plan", [](int64_t M, int64_t N, int64_t T) {
    int c = 0, s = 1;
    hx_wgrad_f16_plan((int)M, (int)N, (int)T, &c, &s);
    return std::make_tuple(c, s);
  });

  m.def("xar_create", &xar_create);
  m.def("xar_register", &xar_register);
  m.def("device_pci_bus_id", &device_pci_bus_id);
  m.def("xar_export", &xar_export);
  m.def("xar_open", &xar_open);
  m.def("xar_allreduce", &xar_allreduce);
  m.def("xar_allreduce_sim", &xar_allreduce_sim);
  m.def("xar_error", &xar_error);
  m.def("xar_error_async", &xar_error_async);
  m.def("xar_oneshot_max", &xar_oneshot_max);
  m.def("xar_destroy", &xar_destroy);
  m.def("set_debug", &set_debug);
  m.def("get_debug", &get_debug);
  // CUs reserved for a concurrent comm kernel (cu_reserve.hip)
  m.def("num_cus", &hx_num_cus);
  m.def("set_reserved_cus", &hx_set_reserved_cus);
  m.def("reserved_cus", &hx_reserved_cus);
  m.def("cu_slots", &hx_cu_slots);
  m.def("cu_masked_stream", [](int64_t first_cu, int64_t count) {
    hipStream_t st = hx_cu_masked_stream((int)first_cu, (int)count);
    TORCH_CHECK(st != nullptr, "hipExtStreamCreateWithCUMask failed");
    return (int64_t)(uintptr_t)st;
  });
  m.def("priority_stream", [](int64_t prio) {
    hipStream_t st = hx_priority_stream((int)prio);
    TORCH_CHECK(st != nullptr, "hipStreamCreateWithPriority failed");
    return (int64_t)(uintptr_t)st;
  });
  m.def("stream_priority_range", []() {
    int least = 0, greatest = 0;
    hx_stream_priority_range(&least, &greatest);
    return std::vector<int64_t>{least, greatest};
  });
  m.def("destroy_stream", [](int64_t h) { hx_destroy_stream(reinterpret_cast<hipStream_t>((uintptr_t)h)); });
  m.def("spin", [](int64_t blocks, double us, int64_t lds_bytes, Tensor sink, int64_t stream) {
    TORCH_CHECK(sink.is_cuda() && sink.scalar_type() == torch::kInt32 && sink.numel() >= 256, "spin: int32 sink[256]");
    TORCH_CHECK(lds_bytes >= 0 && lds_bytes <= 160 * 1024 && us >= 0 && us < 1e7, "spin: bad arguments");
    hipStream_t st = stream ? reinterpret_cast<hipStream_t>((uintptr_t)stream) : cur_stream(sink);
    hx_spin((int)blocks, us, (int)lds_bytes, reinterpret_cast<uint32_t*>(sink.data_ptr<int>()), st);
  });
}
