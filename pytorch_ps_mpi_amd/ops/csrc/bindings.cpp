// bindings.cpp — torch extension surface for the CDNA4 PS kernels.
// Pure HIP-side code (no CUDA compat paths): streams come from c10::hip.

#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cstdint>
#include <iterator>
#include <vector>

extern "C" {
int ps_fused_sgd(void* stream, float* p, float* buf, const float* g, void* p_out,
                 int p_out_is_bf16, int64_t n, float lr, float momentum,
                 float dampening, float wd, int nesterov, int mom_init, float gscale);
int ps_fused_adam(void* stream, float* p, float* m1, float* m2, float* vmax,
                  const float* g, void* p_out, int p_out_is_bf16, int64_t n,
                  float lr, float beta1, float beta2, float eps, float wd,
                  float bc1, float bc2_sqrt, int amsgrad, float gscale);
int ps_fused_adamw(void* stream, float* p, void* out, int out_kind,
                   const float* g, void* m, void* v, float* ms, float* vs,
                   const float* decay, int64_t n, int64_t offset,
                   float step_size, float lr_wd, double beta1, double beta2,
                   float inv_bc2_sqrt, float eps, float gscale, uint32_t key);
int ps_state8_values(void* stream, const uint8_t* codes, const float* scales,
                     void* out, int out_is_bf16, int is_signed, int64_t n);
int ps_rope(void* stream, const void* q, const void* k, void* yq, void* yk,
            const void* pos, int pos64, int dtype, const int64_t* strides,
            int64_t B, int64_t N, int H, int KV, int D, int P,
            const int* start, const double* rev, int inter, int backward);
int64_t ps_join_blocks(int64_t groups, int64_t rows, int64_t D, int post,
                       int bf16);
int ps_join_fwd(void* stream, void* const* t, float* const* stats, int bf16,
                int64_t groups, int64_t rows, int64_t D, int layer,
                int gate_kind, int64_t gate_step, float scale, float eps);
int ps_join_bwd(void* stream, void* const* t, float* const* stats,
                void* const* sums, float* part, int bf16, int64_t groups,
                int64_t rows, int64_t D, int layer, int gate_kind,
                int64_t gate_step, float scale);
int64_t ps_wa_part_floats(int64_t B, int64_t H, int64_t KV, int64_t N, int64_t D,
                          int64_t window, int64_t sinks);
int ps_wa_fwd(void* stream, const void* q, const void* k, const void* v,
              void* o, void* low, float* lse, const int32_t* lengths,
              const int64_t* st, int64_t B, int64_t H, int64_t KV, int64_t N, int64_t D,
              int64_t window, int64_t sinks, float scale);
int ps_wa_bwd(void* stream, const void* q, const void* k, const void* v,
              const void* o, const void* low, const void* go, float* lse,
              float* delta, void* dq, void* dk, void* dv, float* part,
              const int32_t* lengths, const int64_t* st, int64_t B, int64_t H,
              int64_t KV, int64_t N, int64_t D, int64_t window, int64_t sinks,
              float scale);
int ps_reduce_accum(void* stream, float* dst, const void** srcs, int nsrc,
                    int src_is_bf16, int64_t n, float scale, float beta);
int ps_f32_to_bf16(void* stream, const float* src, void* dst, int64_t n);
int ps_bf16_to_f32(void* stream, const void* src, float* dst, int64_t n);
int ps_quant8_encode(void* stream, const void* src, int src_is_bf16,
                     float* scales, int8_t* q, int64_t n);
int ps_quant8_reduce(void* stream, float* dst, const void** scales,
                     const void** qs, int nsrc, int64_t n, float gscale, float beta);
int ps_topk_workspace_words(void);
int ps_topk_encode(void* stream, const void* src, int src_is_bf16, int64_t n,
                   int64_t k, uint32_t* ws, int32_t* out_idx, void* out_val);
int ps_topk_scatter(void* stream, float* dst, const int32_t* idx,
                    const void* val, int val_is_bf16, int64_t k, float gscale);
int ps_topk_encode_thresh(void* stream, const void* src, int src_is_bf16,
                          int64_t n, int off_keys, int64_t kmax, uint32_t* ws,
                          int32_t* hdr, int32_t* out_idx, void* out_val);
int ps_topk_scatter_var(void* stream, float* dst, const int32_t* hdr,
                        const int32_t* idx, const void* val, int val_is_bf16,
                        int64_t kmax, float gscale);
int ps_bn_fwd_stats(void* stream, const void* x, float* psum, float* psumsq,
                    int64_t rows, int64_t C);
int ps_bn_finalize(void* stream, const float* psum, const float* psumsq,
                   const void* gamma, const void* beta, void* rmean,
                   void* rvar, float* mean, float* invstd, float* scale,
                   float* shift, int64_t C, double count, float eps,
                   float momentum, int t_is_bf16);
int ps_bn_eval_coef(void* stream, const void* gamma, const void* beta,
                    const void* rmean, const void* rvar, float* scale,
                    float* shift, int64_t C, float eps, int t_is_bf16);
int ps_bn_normalize(void* stream, const void* x, const void* z, void* y,
                    const float* scale, const float* shift, int64_t rows,
                    int64_t C, int relu);
int ps_bn_bwd_stats(void* stream, const void* x, const void* dy,
                    const void* z, const float* scale, const float* shift,
                    float* dsum, float* dxsum, int64_t rows, int64_t C,
                    int relu);
int ps_bn_bwd_coef(void* stream, const float* dsum, const float* dxsum,
                   const float* mean, const float* invstd, const void* gamma,
                   void* dgamma, void* dbeta, float* ca, float* cbx,
                   float* cc, int64_t C, double count, int train,
                   int t_is_bf16);
int ps_bn_bwd_dx(void* stream, const void* x, const void* dy, const void* z,
                 void* dx, void* dz, const float* ca, const float* cbx,
                 const float* cc, const float* scale, const float* shift,
                 int64_t rows, int64_t C, int relu);
int ps_ln_fwd(void* stream, const void* x, void* y, const void* gamma,
              const void* beta, float* mean, float* rstd, int64_t rows,
              int64_t D, float eps);
int ps_ln_bwd_dx(void* stream, const void* x, const void* dy, void* dx,
                 const void* gamma, const float* mean, const float* rstd,
                 int64_t rows, int64_t D);
int ps_ln_bwd_dgb(void* stream, const void* x, const void* dy,
                  const float* mean, const float* rstd, float* dgamma,
                  float* dbeta, int64_t rows, int64_t D);
int ps_colsum(void* stream, const void* dy, float* out, int64_t rows,
              int64_t D);
int ps_ce_fwd(void* stream, const void* logits, const int64_t* targets,
              float* losses, float* lse, int64_t T, int64_t V);
int ps_ce_bwd(void* stream, const void* logits, const int64_t* targets,
              const float* lse, void* dlogits, int64_t T, int64_t V,
              float gscale, const float* gout_dev);
int ps_attn_fwd(void* stream, const void* q, const void* k, const void* v,
                void* o, float* lse, int64_t rows, int64_t N, float scale,
                int causal);
int ps_attn_bwd(void* stream, const void* q, const void* k, const void* v,
                const void* o, const void* dout, const float* lse,
                float* delta, void* dq, void* dk, void* dv, int64_t rows,
                int64_t N, float scale, int causal);
int ps_fa_fwd(void* stream, const void* q, const void* k, const void* v,
              void* o, float* lse, int64_t BH, int64_t N, float scale,
              int causal, int64_t H, int64_t sB, int64_t sH, int64_t sN);
int ps_fa_bwd(void* stream, const void* q, const void* k, const void* v,
              const void* o, const void* dout, const float* lse, float* delta,
              void* dq, void* dk, void* dv, int64_t BH, int64_t N,
              float scale, int causal, int64_t H, int64_t sB, int64_t sH,
              int64_t sN, int64_t oB, int64_t oH, int64_t oN);
int ps_fa_selfcheck(void* stream, const void* a, const void* b, float* c);
}

namespace {

void* cur_stream(const at::Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

void check_flat(const at::Tensor& t, at::ScalarType dt, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be on GPU");
  TORCH_CHECK(t.scalar_type() == dt, name, " has wrong dtype");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

int is_bf16(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? 1 : 0; }

void throw_on(int err, const char* what) {
  TORCH_CHECK(err != 9001, what, ": 1..8 sources supported");
  TORCH_CHECK(err != 9002, what,
              ": int8 payload/dst must be 8/16B-aligned (use the codec wire "
              "layout: scales padded to 16B before q)");
  TORCH_CHECK(err != 9003, what, ": size out of the kernel's range");
  TORCH_CHECK(err == 0, what, ": hip error ", err);
}

void fused_sgd(at::Tensor p, c10::optional<at::Tensor> buf, at::Tensor g,
               c10::optional<at::Tensor> p_out, double lr, double momentum,
               double dampening, double wd, bool nesterov, bool mom_init,
               double gscale) {
  check_flat(p, at::kFloat, "param");
  check_flat(g, at::kFloat, "grad");
  TORCH_CHECK(p.numel() == g.numel(), "param/grad length mismatch");
  float* buf_ptr = nullptr;
  if (momentum != 0.0) {
    TORCH_CHECK(buf.has_value(), "momentum buffer required when momentum != 0");
    check_flat(*buf, at::kFloat, "momentum buffer");
    TORCH_CHECK(buf->numel() == p.numel(), "momentum buffer length mismatch");
    buf_ptr = buf->data_ptr<float>();
  }
  void* out_ptr = nullptr;
  int out_bf16 = 0;
  if (p_out.has_value()) {
    TORCH_CHECK(p_out->is_cuda() && p_out->is_contiguous(), "p_out invalid");
    TORCH_CHECK(p_out->numel() == p.numel(), "p_out length mismatch");
    out_ptr = p_out->data_ptr();
    out_bf16 = is_bf16(*p_out);
    TORCH_CHECK(out_bf16 || p_out->scalar_type() == at::kFloat, "p_out dtype");
  }
  throw_on(ps_fused_sgd(cur_stream(p), p.data_ptr<float>(), buf_ptr,
                        g.data_ptr<float>(), out_ptr, out_bf16, p.numel(),
                        (float)lr, (float)momentum, (float)dampening, (float)wd,
                        nesterov ? 1 : 0, mom_init ? 1 : 0, (float)gscale),
           "fused_sgd");
}

void fused_adam(at::Tensor p, at::Tensor m1, at::Tensor m2,
                c10::optional<at::Tensor> vmax, at::Tensor g,
                c10::optional<at::Tensor> p_out, double lr, double beta1,
                double beta2, double eps, double wd, int64_t step, bool amsgrad,
                double gscale) {
  check_flat(p, at::kFloat, "param");
  check_flat(m1, at::kFloat, "exp_avg");
  check_flat(m2, at::kFloat, "exp_avg_sq");
  check_flat(g, at::kFloat, "grad");
  float* vmax_ptr = nullptr;
  if (amsgrad) {
    TORCH_CHECK(vmax.has_value(), "amsgrad requires max_exp_avg_sq");
    check_flat(*vmax, at::kFloat, "max_exp_avg_sq");
    vmax_ptr = vmax->data_ptr<float>();
  }
  void* out_ptr = nullptr;
  int out_bf16 = 0;
  if (p_out.has_value()) {
    TORCH_CHECK(p_out->is_cuda() && p_out->is_contiguous(), "p_out invalid");
    out_ptr = p_out->data_ptr();
    out_bf16 = is_bf16(*p_out);
  }
  const double bc1 = 1.0 - std::pow(beta1, (double)step);
  const double bc2_sqrt = std::sqrt(1.0 - std::pow(beta2, (double)step));
  throw_on(ps_fused_adam(cur_stream(p), p.data_ptr<float>(), m1.data_ptr<float>(),
                         m2.data_ptr<float>(), vmax_ptr, g.data_ptr<float>(),
                         out_ptr, out_bf16, p.numel(), (float)lr, (float)beta1,
                         (float)beta2, (float)eps, (float)wd, (float)bc1,
                         (float)bc2_sqrt, amsgrad ? 1 : 0, (float)gscale),
           "fused_adam");
}

void check_same_device(const at::Tensor& a, const at::Tensor& t,
                       const char* name) {
  TORCH_CHECK(t.device() == a.device(), name, " is on another device");
}

void fused_adamw(at::Tensor p, c10::optional<at::Tensor> p_out, at::Tensor g,
                 at::Tensor m, at::Tensor v, c10::optional<at::Tensor> ms,
                 c10::optional<at::Tensor> vs,
                 c10::optional<at::Tensor> decay, int64_t offset,
                 double step_size, double lr_wd, double beta1, double beta2,
                 double inv_bc2_sqrt, double eps, double gscale,
                 int64_t key) {
  const bool s8 = ms.has_value();
  const int64_t n = p.numel(), chunks = (n + 255) / 256;
  const auto st = s8 ? at::kByte : at::kFloat;
  check_flat(p, at::kFloat, "param");
  check_flat(g, at::kFloat, "grad");
  check_flat(m, st, "exp_avg");
  check_flat(v, st, "exp_avg_sq");
  TORCH_CHECK(g.numel() == n && m.numel() == n && v.numel() == n,
              "param/grad/state length mismatch");
  TORCH_CHECK(s8 == vs.has_value(), "8-bit states need both scales");
  for (const auto& t : {g, m, v}) check_same_device(p, t, "grad/state");
  float *msp = nullptr, *vsp = nullptr;
  if (s8) {
    check_flat(*ms, at::kFloat, "exp_avg scales");
    check_flat(*vs, at::kFloat, "exp_avg_sq scales");
    TORCH_CHECK(ms->numel() == chunks && vs->numel() == chunks,
                "one scale for each 256 elements");
    check_same_device(p, *ms, "scales");
    check_same_device(p, *vs, "scales");
    msp = ms->data_ptr<float>();
    vsp = vs->data_ptr<float>();
  }
  const float* dp = nullptr;
  if (decay.has_value()) {
    check_flat(*decay, at::kFloat, "decay");
    check_same_device(p, *decay, "decay");
    TORCH_CHECK(decay->numel() == chunks, "one decay for each 256 elements");
    dp = decay->data_ptr<float>();
  }
  void* out_ptr = nullptr;
  int kind = 0;
  if (p_out.has_value()) {
    check_flat(*p_out, p_out->scalar_type(), "p_out");
    check_same_device(p, *p_out, "p_out");
    TORCH_CHECK(p_out->numel() == n, "p_out length mismatch");
    TORCH_CHECK(is_bf16(*p_out) || p_out->scalar_type() == at::kFloat,
                "p_out dtype");
    out_ptr = p_out->data_ptr();
    kind = is_bf16(*p_out) ? 1 : 2;
  }
  struct { const at::Tensor* t; bool written; } all[] = {
      {&p, true}, {&m, true}, {&v, true}, {s8 ? &*ms : nullptr, true},
      {s8 ? &*vs : nullptr, true}, {p_out ? &*p_out : nullptr, true},
      {&g, false}, {decay ? &*decay : nullptr, false}};
  for (const auto& a : all)
    for (const auto* b = &a + 1; b < std::end(all); ++b) {
      if (!a.t || !b->t || !(a.written || b->written)) continue;
      const char *x = (const char*)a.t->data_ptr(), *y = (const char*)b->t->data_ptr();
      // ValueError, as the CPU path raises
      TORCH_CHECK_VALUE(x + a.t->nbytes() <= y || y + b->t->nbytes() <= x,
                        "p, p_out and the states must not share memory with "
                        "each other, g or decay");
    }
  const c10::DeviceGuard guard(p.device());
  throw_on(ps_fused_adamw(cur_stream(p), p.data_ptr<float>(), out_ptr, kind,
                          g.data_ptr<float>(), m.data_ptr(), v.data_ptr(), msp,
                          vsp, dp, n, offset, (float)step_size, (float)lr_wd,
                          beta1, beta2, (float)inv_bc2_sqrt,
                          (float)eps, (float)gscale, (uint32_t)key),
           "fused_adamw");
}

void state8_values(at::Tensor codes, at::Tensor scales, at::Tensor out,
                   bool is_signed) {
  check_flat(codes, at::kByte, "codes");
  check_flat(scales, at::kFloat, "scales");
  check_flat(out, out.scalar_type(), "out");
  check_same_device(codes, scales, "scales");
  check_same_device(codes, out, "out");
  const int64_t n = codes.numel();
  TORCH_CHECK(scales.numel() == (n + 255) / 256, "one scale per 256 elements");
  TORCH_CHECK(out.numel() == n &&
                  (is_bf16(out) || out.scalar_type() == at::kFloat),
              "out must be bf16/f32 of the codes' length");
  const c10::DeviceGuard guard(codes.device());
  throw_on(ps_state8_values(cur_stream(codes), codes.data_ptr<uint8_t>(),
                            scales.data_ptr<float>(), out.data_ptr(),
                            is_bf16(out), is_signed ? 1 : 0, n),
           "state8_values");
}

int float_kind(const at::Tensor& t, const char* name) {
  const auto st = t.scalar_type();
  TORCH_CHECK(st == at::kBFloat16 || st == at::kHalf || st == at::kFloat, name,
              " must be bf16, fp16 or fp32");
  return st == at::kBFloat16 ? 0 : st == at::kHalf ? 1 : 2;
}

// No second derivatives: a backward pass of these functions is not recorded.
void first_order(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what,
              " has no second derivative (create_graph=True)");
}

// q, k [B, N, heads, D] turned by positions [axes, B, N]; `rev`: revolutions a
// position for each pair (host, fp64), `start`: first pair of axes 1 to 3.
std::vector<at::Tensor> rope_apply(at::Tensor q, at::Tensor k,
                                   const at::Tensor& pos,
                                   const std::vector<int64_t>& start,
                                   const at::Tensor& rev, bool inter,
                                   bool backward) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 4 && k.dim() == 4, "q, k: 4-D on GPU");
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(1) == k.size(1) &&
                  q.size(3) == k.size(3) && k.scalar_type() == q.scalar_type(),
              "q and k differ in B, N, D or type");
  for (const auto& t : {k, pos}) check_same_device(q, t, "rope input");
  TORCH_CHECK(pos.dim() == 3 && pos.size(1) == q.size(0) &&
                  pos.size(2) == q.size(1), "positions [axes, B, N]");
  TORCH_CHECK(pos.scalar_type() == at::kLong || pos.scalar_type() == at::kInt,
              "positions int32/int64");
  TORCH_CHECK(rev.device().is_cpu() && rev.scalar_type() == at::kDouble &&
                  rev.is_contiguous() && start.size() == 3, "rope plan");
  const int P = (int)rev.numel();
  int first[3];
  int axes = 1;
  for (int i = 0; i < 3; ++i) {
    first[i] = (int)start[i];
    axes += first[i] < P;
  }
  TORCH_CHECK(pos.size(0) >= axes, "a position for each axis");
  const c10::DeviceGuard guard(q.device());
  if (q.stride(3) != 1) q = q.contiguous();
  if (k.stride(3) != 1) k = k.contiguous();
  auto yq = at::empty(q.sizes(), q.options());
  auto yk = at::empty(k.sizes(), k.options());
  const int64_t strides[9] = {q.stride(0), q.stride(1), q.stride(2),
                              k.stride(0), k.stride(1), k.stride(2),
                              pos.stride(0), pos.stride(1), pos.stride(2)};
  throw_on(ps_rope(cur_stream(q), q.data_ptr(), k.data_ptr(), yq.data_ptr(),
                   yk.data_ptr(), pos.data_ptr(),
                   pos.scalar_type() == at::kLong, float_kind(q, "q"), strides,
                   q.size(0), q.size(1), (int)q.size(2), (int)k.size(2),
                   (int)q.size(3), P, first, rev.data_ptr<double>(),
                   inter ? 1 : 0, backward ? 1 : 0),
           "rope");
  return {yq, yk};
}

// The backward pass is the turn by the opposite angles.
struct Rope : torch::autograd::Function<Rope> {
  static torch::autograd::variable_list forward(
      torch::autograd::AutogradContext* ctx, const at::Tensor& q,
      const at::Tensor& k, const at::Tensor& pos, std::vector<int64_t> start,
      const at::Tensor& rev, bool inter) {
    ctx->save_for_backward({pos, rev});
    ctx->saved_data["start"] = start;
    ctx->saved_data["inter"] = inter;
    return rope_apply(q, k, pos, start, rev, inter, false);
  }
  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx,
      torch::autograd::variable_list g) {
    first_order("AxialRotary");
    const auto saved = ctx->get_saved_variables();
    auto d = rope_apply(g[0], g[1], saved[0],
                        ctx->saved_data["start"].toIntVector(), saved[1],
                        ctx->saved_data["inter"].toBool(), true);
    return {d[0], d[1], at::Tensor(), at::Tensor(), at::Tensor(),
            at::Tensor()};
  }
};

std::vector<at::Tensor> rope(at::Tensor q, at::Tensor k, at::Tensor pos,
                             std::vector<int64_t> start, at::Tensor rev,
                             bool inter) {
  return Rope::apply(q, k, pos, start, rev, inter);
}

// ---- norms before and after a block with its gate and residual ------------

using OptTensors = std::vector<c10::optional<at::Tensor>>;

// Pointers of `t`; entry i holds numel[i] elements of `like`'s type.
void join_ptrs(const OptTensors& t, const std::vector<int64_t>& numel,
               const at::Tensor& like, void** out) {
  TORCH_CHECK(t.size() == numel.size(), "join: wrong number of tensors");
  for (size_t i = 0; i < t.size(); ++i) {
    out[i] = nullptr;
    if (!t[i].has_value()) continue;
    check_flat(*t[i], like.scalar_type(), "join tensor");
    check_same_device(like, *t[i], "join tensor");
    TORCH_CHECK(t[i]->numel() == numel[i], "join tensor ", i, " has ",
                t[i]->numel(), " elements, expected ", numel[i]);
    out[i] = t[i]->data_ptr();
  }
}

void join_stats(const at::Tensor& stats, const at::Tensor& like, int64_t rows,
                bool post, float** out) {
  check_flat(stats, at::kFloat, "stats");
  check_same_device(like, stats, "stats");
  TORCH_CHECK(stats.numel() == (post ? 4 : 2) * rows, "stats size");
  float* p = stats.data_ptr<float>();
  for (int i = 0; i < 4; ++i) out[i] = i < 2 || post ? p + i * rows : nullptr;
}

int64_t join_gate(int64_t kind, int64_t step, int64_t groups, int64_t rows,
                  int64_t D) {
  TORCH_CHECK(kind >= 0 && kind <= 2 && (step == 0 || step == D), "gate kind");
  return kind == 2 ? groups * rows * D : step ? groups * D : D;
}

// t: x, u, w, b, pw, pb, gate, y, h
void join_fwd(OptTensors t, at::Tensor stats, int64_t groups, int64_t rows,
              int64_t D, bool layer, int64_t gate_kind, int64_t gate_step,
              double scale, double eps) {
  TORCH_CHECK(t.size() == 9 && t[0] && t[1] && t[2] && t[7] && t[8],
              "join_fwd: x, u, w, y, h wanted");
  TORCH_CHECK(gate_kind == 0 || t[6], "join_fwd: gate wanted");
  const at::Tensor& x = *t[0];
  TORCH_CHECK(is_bf16(x) || x.scalar_type() == at::kFloat, "bf16 or fp32");
  const int64_t n = groups * rows * D;
  const int64_t ng = join_gate(gate_kind, gate_step, groups, rows, D);
  void* p[9];
  float* st[4];
  join_ptrs(t, {n, n, D, D, D, D, ng, n, n}, x, p);
  join_stats(stats, x, groups * rows, t[4].has_value(), st);
  const c10::DeviceGuard guard(x.device());
  throw_on(ps_join_fwd(cur_stream(x), p, st, is_bf16(x), groups, rows, D,
                       layer ? 1 : 0, (int)gate_kind, gate_step, (float)scale,
                       (float)eps),
           "join_fwd");
}

// t: u, w, pw, pb, gate, x, dy, dh, dx, du, dgate; sums: dw, db, dgate, dpw,
// dpb
void join_bwd(OptTensors t, at::Tensor stats, OptTensors sums, at::Tensor part,
              int64_t groups, int64_t rows, int64_t D, bool layer,
              int64_t gate_kind, int64_t gate_step, double scale) {
  TORCH_CHECK(t.size() == 11 && t[0] && t[1] && t[5] && t[8] && t[9],
              "join_bwd: u, w, x, dx, du wanted");
  TORCH_CHECK(gate_kind == 0 || t[4], "join_bwd: gate wanted");
  const at::Tensor& u = *t[0];
  TORCH_CHECK(is_bf16(u) || u.scalar_type() == at::kFloat, "bf16 or fp32");
  const int64_t n = groups * rows * D;
  const int64_t ng = join_gate(gate_kind, gate_step, groups, rows, D);
  void *p[11], *s[5];
  float* st[4];
  join_ptrs(t, {n, D, D, D, ng, n, n, n, n, n, n}, u, p);
  join_ptrs(sums, {D, D, ng, D, D}, u, s);
  TORCH_CHECK((!s[3] && !s[4]) || p[2], "join_bwd: post sums without a post norm");
  TORCH_CHECK((!s[2] && !p[10]) || gate_kind, "join_bwd: gate sums without a gate");
  TORCH_CHECK(!s[2] || gate_kind == 1, "join_bwd: vector gate expected");
  join_stats(stats, u, groups * rows, t[2].has_value(), st);
  check_flat(part, at::kFloat, "part");
  check_same_device(u, part, "part");
  int64_t slots = 0;
  for (void* q : s) slots += q != nullptr;
  TORCH_CHECK(part.numel() >=
                  groups * ps_join_blocks(groups, rows, D, p[2] != nullptr,
                                           is_bf16(u)) * slots * D,
              "join_bwd: part too small");
  const c10::DeviceGuard guard(u.device());
  throw_on(ps_join_bwd(cur_stream(u), p, st, s, part.data_ptr<float>(),
                       is_bf16(u), groups, rows, D, layer ? 1 : 0,
                       (int)gate_kind, gate_step, (float)scale),
           "join_bwd");
}

// groups, rows: the gate's vector is one of `groups`, each for `rows` rows;
// gate_kind 0 none, 1 vector, 2 x's shape.
struct GatedResidual : torch::autograd::Function<GatedResidual> {
  using Opt = c10::optional<at::Tensor>;
  static at::Tensor dense(const Opt& t) {
    return t.has_value() ? t->contiguous() : at::Tensor();
  }
  static Opt opt(const at::Tensor& t) {
    return t.defined() ? Opt(t) : Opt();
  }
  static torch::autograd::variable_list forward(
      torch::autograd::AutogradContext* ctx, const at::Tensor& x_,
      const at::Tensor& u_, const at::Tensor& w_, const Opt& b_,
      const Opt& gate_, const Opt& pw_, const Opt& pb_, double scale,
      double eps, bool layer, int64_t groups, int64_t gate_kind) {
    const c10::DeviceGuard guard(x_.device());
    const auto x = x_.contiguous(), u = u_.contiguous(), w = w_.contiguous();
    const auto b = dense(b_), gate = dense(gate_), pw = dense(pw_),
               pb = dense(pb_);
    const int64_t D = x.size(-1), rows = x.numel() / D / groups;
    const int64_t step = gate_kind == 1 && groups > 1 ? D : 0;
    auto y = at::empty_like(x), h = at::empty_like(x);
    auto stats = at::empty({pw.defined() ? 4 : 2, groups * rows},
                           x.options().dtype(at::kFloat));
    join_fwd({x, u, w, opt(b), opt(pw), opt(pb), opt(gate), y, h}, stats,
             groups, rows, D, layer, gate_kind, step, scale, eps);
    ctx->save_for_backward({x, u, w, gate, pw, pb, stats});
    ctx->saved_data["cfg"] =
        std::vector<int64_t>{groups, rows, D, layer, gate_kind, step,
                             b.defined()};
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    return {y, h};
  }
  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx,
      torch::autograd::variable_list g) {
    first_order("fused_gated_residual");
    torch::autograd::variable_list out(12);
    if (!g[0].defined() && !g[1].defined()) return out;
    const auto s = ctx->get_saved_variables();
    const auto &x = s[0], &u = s[1], &w = s[2], &gate = s[3], &pw = s[4],
               &pb = s[5], &stats = s[6];
    const auto cfg = ctx->saved_data["cfg"].toIntVector();
    const int64_t groups = cfg[0], rows = cfg[1], D = cfg[2], kind = cfg[4];
    const c10::DeviceGuard guard(x.device());
    const Opt dy = g[0].defined() ? Opt(g[0].contiguous()) : Opt();
    const Opt dh = g[1].defined() ? Opt(g[1].contiguous()) : Opt();
    // inputs that are there, in order: x, u, w, b, gate, pw, pb
    const bool there[7] = {true, true, true, cfg[6] != 0, gate.defined(),
                           pw.defined(), pb.defined()};
    bool need[7];
    size_t edge = 0;
    for (int i = 0; i < 7; ++i)
      need[i] = there[i] && ctx->needs_input_grad(edge++);
    out[0] = at::empty_like(x);
    out[1] = at::empty_like(u);
    // without dh the last norm's parameters get no gradient
    if (need[2] && dh) out[2] = at::empty_like(w);
    if (need[3] && dh) out[3] = at::empty_like(w);
    if (need[4]) out[4] = at::empty_like(gate);
    if (need[5]) out[5] = at::empty_like(pw);
    if (need[6]) out[6] = at::empty_like(pb);
    const Opt vec = kind == 1 ? opt(out[4]) : Opt();
    int64_t slots = vec.has_value();
    for (int i : {2, 3, 5, 6}) slots += out[i].defined();
    auto part = at::empty({groups *
                           ps_join_blocks(groups, rows, D, pw.defined(),
                                          is_bf16(u)) *
                           slots * D},
                          x.options().dtype(at::kFloat));
    join_bwd({u, w, opt(pw), opt(pb), opt(gate), x, dy, dh, out[0], out[1],
              kind == 2 ? opt(out[4]) : Opt()},
             stats, {opt(out[2]), opt(out[3]), vec, opt(out[5]), opt(out[6])},
             part, groups, rows, D, cfg[3] != 0, kind, cfg[5],
             ctx->saved_data["scale"].toDouble());
    if (!need[0]) out[0] = at::Tensor();
    if (!need[1]) out[1] = at::Tensor();
    return out;
  }
};

std::vector<at::Tensor> gated_residual(
    at::Tensor x, at::Tensor u, at::Tensor w, c10::optional<at::Tensor> b,
    c10::optional<at::Tensor> gate, c10::optional<at::Tensor> pw,
    c10::optional<at::Tensor> pb, double scale, double eps, bool layer,
    int64_t groups, int64_t gate_kind) {
  return GatedResidual::apply(x, u, w, b, gate, pw, pb, scale, eps, layer,
                              groups, gate_kind);
}

void reduce_accum(at::Tensor dst, std::vector<at::Tensor> srcs, double scale,
                  double beta) {
  check_flat(dst, at::kFloat, "dst");
  TORCH_CHECK(!srcs.empty() && srcs.size() <= 8, "1..8 sources");
  const void* ptrs[8];
  int bf = is_bf16(srcs[0]);
  for (size_t i = 0; i < srcs.size(); ++i) {
    TORCH_CHECK(srcs[i].is_cuda() && srcs[i].is_contiguous(), "src invalid");
    TORCH_CHECK(srcs[i].numel() == dst.numel(), "src length mismatch");
    TORCH_CHECK(is_bf16(srcs[i]) == bf &&
                    (bf || srcs[i].scalar_type() == at::kFloat),
                "all sources must share dtype (f32 or bf16)");
    ptrs[i] = srcs[i].data_ptr();
  }
  throw_on(ps_reduce_accum(cur_stream(dst), dst.data_ptr<float>(), ptrs,
                           (int)srcs.size(), bf, dst.numel(), (float)scale,
                           (float)beta),
           "reduce_accum");
}

void f32_to_bf16(at::Tensor src, at::Tensor dst) {
  check_flat(src, at::kFloat, "src");
  check_flat(dst, at::kBFloat16, "dst");
  TORCH_CHECK(src.numel() == dst.numel(), "length mismatch");
  throw_on(ps_f32_to_bf16(cur_stream(src), src.data_ptr<float>(), dst.data_ptr(),
                          src.numel()),
           "f32_to_bf16");
}

void bf16_to_f32(at::Tensor src, at::Tensor dst) {
  check_flat(src, at::kBFloat16, "src");
  check_flat(dst, at::kFloat, "dst");
  TORCH_CHECK(src.numel() == dst.numel(), "length mismatch");
  throw_on(ps_bf16_to_f32(cur_stream(src), src.data_ptr(), dst.data_ptr<float>(),
                          src.numel()),
           "bf16_to_f32");
}

void quant8_encode(at::Tensor src, at::Tensor scales, at::Tensor q) {
  TORCH_CHECK(src.is_cuda() && src.is_contiguous(), "src invalid");
  int bf = is_bf16(src);
  TORCH_CHECK(bf || src.scalar_type() == at::kFloat, "src dtype");
  check_flat(scales, at::kFloat, "scales");
  TORCH_CHECK(q.scalar_type() == at::kChar && q.is_contiguous() && q.is_cuda(),
              "q must be int8");
  const int64_t n = src.numel();
  TORCH_CHECK(scales.numel() >= (n + 255) / 256, "scales too small");
  TORCH_CHECK(q.numel() >= n, "q too small");
  throw_on(ps_quant8_encode(cur_stream(src), src.data_ptr(), bf,
                            scales.data_ptr<float>(),
                            (int8_t*)q.data_ptr(), n),
           "quant8_encode");
}

void quant8_reduce(at::Tensor dst, std::vector<at::Tensor> scales,
                   std::vector<at::Tensor> qs, double gscale, double beta) {
  check_flat(dst, at::kFloat, "dst");
  TORCH_CHECK(scales.size() == qs.size() && !qs.empty() && qs.size() <= 8,
              "1..8 sources");
  const void* sp[8];
  const void* qp[8];
  for (size_t i = 0; i < qs.size(); ++i) {
    TORCH_CHECK(scales[i].is_cuda() && scales[i].is_contiguous() &&
                    scales[i].scalar_type() == at::kFloat,
                "scales invalid");
    TORCH_CHECK(qs[i].is_cuda() && qs[i].is_contiguous() &&
                    qs[i].scalar_type() == at::kChar,
                "q invalid");
    TORCH_CHECK(qs[i].numel() >= dst.numel(), "q length mismatch");
    sp[i] = scales[i].data_ptr();
    qp[i] = qs[i].data_ptr();
  }
  throw_on(ps_quant8_reduce(cur_stream(dst), dst.data_ptr<float>(), sp, qp,
                            (int)qs.size(), dst.numel(), (float)gscale,
                            (float)beta),
           "quant8_reduce");
}

void colsum(at::Tensor dy, at::Tensor out) {
  TORCH_CHECK(dy.is_cuda() && dy.is_contiguous() && dy.dim() == 2 &&
                  dy.scalar_type() == at::kBFloat16,
              "dy must be contiguous 2D bf16");
  check_flat(out, at::kFloat, "out");
  TORCH_CHECK(out.numel() == dy.size(1), "out length mismatch");
  throw_on(ps_colsum(cur_stream(dy), dy.data_ptr(), out.data_ptr<float>(),
                     dy.size(0), dy.size(1)),
           "colsum");
}

int64_t topk_workspace_words() { return ps_topk_workspace_words(); }

void topk_encode_thresh(at::Tensor src, int64_t off_keys, int64_t kmax,
                        at::Tensor ws, at::Tensor hdr, at::Tensor out_idx,
                        at::Tensor out_val) {
  TORCH_CHECK(src.is_cuda() && src.is_contiguous(), "src invalid");
  int bf = is_bf16(src);
  TORCH_CHECK(bf || src.scalar_type() == at::kFloat, "src dtype");
  TORCH_CHECK(ws.scalar_type() == at::kInt && ws.numel() >= ps_topk_workspace_words(),
              "workspace too small");
  TORCH_CHECK(hdr.scalar_type() == at::kInt && hdr.numel() >= 1, "hdr int32[1]");
  TORCH_CHECK(out_idx.scalar_type() == at::kInt && out_idx.numel() >= kmax,
              "out_idx too small");
  TORCH_CHECK(out_val.numel() >= kmax, "out_val too small");
  TORCH_CHECK(kmax >= 1 && kmax <= src.numel(), "kmax in [1, n]");
  throw_on(ps_topk_encode_thresh(cur_stream(src), src.data_ptr(), bf,
                                 src.numel(), (int)off_keys, kmax,
                                 (uint32_t*)ws.data_ptr(),
                                 (int32_t*)hdr.data_ptr(),
                                 (int32_t*)out_idx.data_ptr(),
                                 out_val.data_ptr()),
           "topk_encode_thresh");
}

void topk_scatter_var(at::Tensor dst, at::Tensor hdr, at::Tensor idx,
                      at::Tensor val, int64_t kmax, double gscale) {
  check_flat(dst, at::kFloat, "dst");
  TORCH_CHECK(hdr.is_cuda() && hdr.scalar_type() == at::kInt, "hdr invalid");
  TORCH_CHECK(idx.scalar_type() == at::kInt, "idx int32");
  throw_on(ps_topk_scatter_var(cur_stream(dst), dst.data_ptr<float>(),
                               (const int32_t*)hdr.data_ptr(),
                               (const int32_t*)idx.data_ptr(), val.data_ptr(),
                               is_bf16(val), kmax, (float)gscale),
           "topk_scatter_var");
}

void topk_encode(at::Tensor src, int64_t k, at::Tensor ws, at::Tensor out_idx,
                 at::Tensor out_val) {
  TORCH_CHECK(src.is_cuda() && src.is_contiguous(), "src invalid");
  int bf = is_bf16(src);
  TORCH_CHECK(bf || src.scalar_type() == at::kFloat, "src dtype");
  TORCH_CHECK(ws.scalar_type() == at::kInt || ws.scalar_type() == at::kUInt32,
              "ws must be int32/uint32");
  TORCH_CHECK(ws.numel() >= ps_topk_workspace_words(), "ws too small");
  TORCH_CHECK(out_idx.scalar_type() == at::kInt && out_idx.numel() >= k,
              "out_idx invalid");
  TORCH_CHECK(out_val.scalar_type() == src.scalar_type() && out_val.numel() >= k,
              "out_val invalid");
  TORCH_CHECK(k >= 1 && k <= src.numel(), "k out of range");
  throw_on(ps_topk_encode(cur_stream(src), src.data_ptr(), bf, src.numel(), k,
                          (uint32_t*)ws.data_ptr(),
                          (int32_t*)out_idx.data_ptr(), out_val.data_ptr()),
           "topk_encode");
}

void topk_scatter(at::Tensor dst, at::Tensor idx, at::Tensor val, int64_t k,
                  double gscale) {
  check_flat(dst, at::kFloat, "dst");
  TORCH_CHECK(idx.scalar_type() == at::kInt && idx.is_cuda(), "idx invalid");
  int bf = is_bf16(val);
  TORCH_CHECK(bf || val.scalar_type() == at::kFloat, "val dtype");
  TORCH_CHECK(idx.numel() >= k && val.numel() >= k, "k too large");
  throw_on(ps_topk_scatter(cur_stream(dst), dst.data_ptr<float>(),
                           (const int32_t*)idx.data_ptr(), val.data_ptr(), bf, k,
                           (float)gscale),
           "topk_scatter");
}

// ---- fused NHWC BatchNorm ------------------------------------------------

void check_bn_stream(const at::Tensor& t, int64_t numel, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16, name);
  TORCH_CHECK(t.numel() == numel, name, " numel mismatch");
}

const void* opt_ptr(const c10::optional<at::Tensor>& t) {
  return t.has_value() ? t->data_ptr() : nullptr;
}

void bn_fwd_stats(at::Tensor x, at::Tensor psum, at::Tensor psumsq,
                  int64_t rows, int64_t C) {
  TORCH_CHECK(C % 64 == 0, "C must be a multiple of 64");
  check_bn_stream(x, rows * C, "x");
  throw_on(ps_bn_fwd_stats(cur_stream(x), x.data_ptr(),
                           psum.data_ptr<float>(), psumsq.data_ptr<float>(),
                           rows, C),
           "bn_fwd_stats");
}

void bn_finalize(at::Tensor psum, at::Tensor psumsq,
                 c10::optional<at::Tensor> gamma,
                 c10::optional<at::Tensor> beta,
                 c10::optional<at::Tensor> rmean,
                 c10::optional<at::Tensor> rvar, at::Tensor mean,
                 at::Tensor invstd, at::Tensor scale, at::Tensor shift,
                 double count, double eps, double momentum) {
  const int64_t C = psum.numel();
  int bf = gamma.has_value() ? is_bf16(*gamma)
                             : (rmean.has_value() ? is_bf16(*rmean) : 1);
  throw_on(ps_bn_finalize(cur_stream(psum), psum.data_ptr<float>(),
                          psumsq.data_ptr<float>(), opt_ptr(gamma),
                          opt_ptr(beta), (void*)opt_ptr(rmean),
                          (void*)opt_ptr(rvar), mean.data_ptr<float>(),
                          invstd.data_ptr<float>(), scale.data_ptr<float>(),
                          shift.data_ptr<float>(), C, count, (float)eps,
                          (float)momentum, bf),
           "bn_finalize");
}

void bn_eval_coef(c10::optional<at::Tensor> gamma,
                  c10::optional<at::Tensor> beta, at::Tensor rmean,
                  at::Tensor rvar, at::Tensor scale, at::Tensor shift,
                  double eps) {
  const int64_t C = rmean.numel();
  throw_on(ps_bn_eval_coef(cur_stream(rmean), opt_ptr(gamma), opt_ptr(beta),
                           rmean.data_ptr(), rvar.data_ptr(),
                           scale.data_ptr<float>(), shift.data_ptr<float>(),
                           C, (float)eps, is_bf16(rmean)),
           "bn_eval_coef");
}

void bn_normalize(at::Tensor x, c10::optional<at::Tensor> z, at::Tensor y,
                  at::Tensor scale, at::Tensor shift, int64_t rows, int64_t C,
                  bool relu) {
  check_bn_stream(x, rows * C, "x");
  check_bn_stream(y, rows * C, "y");
  if (z.has_value()) check_bn_stream(*z, rows * C, "z");
  throw_on(ps_bn_normalize(cur_stream(x), x.data_ptr(), opt_ptr(z),
                           y.data_ptr(), scale.data_ptr<float>(),
                           shift.data_ptr<float>(), rows, C, relu ? 1 : 0),
           "bn_normalize");
}

void bn_bwd_stats(at::Tensor x, at::Tensor dy, c10::optional<at::Tensor> z,
                  at::Tensor scale, at::Tensor shift, at::Tensor dsum,
                  at::Tensor dxsum, int64_t rows, int64_t C, bool relu) {
  check_bn_stream(x, rows * C, "x");
  check_bn_stream(dy, rows * C, "dy");
  throw_on(ps_bn_bwd_stats(cur_stream(x), x.data_ptr(), dy.data_ptr(),
                           opt_ptr(z), scale.data_ptr<float>(),
                           shift.data_ptr<float>(), dsum.data_ptr<float>(),
                           dxsum.data_ptr<float>(), rows, C, relu ? 1 : 0),
           "bn_bwd_stats");
}

void bn_bwd_coef(at::Tensor dsum, at::Tensor dxsum, at::Tensor mean,
                 at::Tensor invstd, c10::optional<at::Tensor> gamma,
                 c10::optional<at::Tensor> dgamma,
                 c10::optional<at::Tensor> dbeta, at::Tensor ca,
                 at::Tensor cbx, at::Tensor cc, double count, bool train) {
  const int64_t C = dsum.numel();
  int bf = gamma.has_value() ? is_bf16(*gamma) : 1;
  throw_on(ps_bn_bwd_coef(cur_stream(dsum), dsum.data_ptr<float>(),
                          dxsum.data_ptr<float>(), mean.data_ptr<float>(),
                          invstd.data_ptr<float>(), opt_ptr(gamma),
                          (void*)opt_ptr(dgamma), (void*)opt_ptr(dbeta),
                          ca.data_ptr<float>(), cbx.data_ptr<float>(),
                          cc.data_ptr<float>(), C, count, train ? 1 : 0, bf),
           "bn_bwd_coef");
}

void bn_bwd_dx(at::Tensor x, at::Tensor dy, c10::optional<at::Tensor> z,
               at::Tensor dx, c10::optional<at::Tensor> dz, at::Tensor ca,
               at::Tensor cbx, at::Tensor cc, at::Tensor scale,
               at::Tensor shift, int64_t rows, int64_t C, bool relu) {
  check_bn_stream(x, rows * C, "x");
  check_bn_stream(dx, rows * C, "dx");
  TORCH_CHECK(z.has_value() == dz.has_value(), "z/dz pairing");
  throw_on(ps_bn_bwd_dx(cur_stream(x), x.data_ptr(), dy.data_ptr(),
                        opt_ptr(z), dx.data_ptr(), (void*)opt_ptr(dz),
                        ca.data_ptr<float>(), cbx.data_ptr<float>(),
                        cc.data_ptr<float>(), scale.data_ptr<float>(),
                        shift.data_ptr<float>(), rows, C, relu ? 1 : 0),
           "bn_bwd_dx");
}

// ---- fused row-wise LayerNorm -------------------------------------------

void ln_fwd(at::Tensor x, at::Tensor y, at::Tensor gamma, at::Tensor beta,
            at::Tensor mean, at::Tensor rstd, int64_t rows, int64_t D,
            double eps) {
  TORCH_CHECK(x.is_cuda() && x.scalar_type() == at::kBFloat16, "x");
  TORCH_CHECK(gamma.scalar_type() == at::kBFloat16, "gamma dtype");
  throw_on(ps_ln_fwd(cur_stream(x), x.data_ptr(), y.data_ptr(),
                     gamma.data_ptr(), beta.data_ptr(),
                     mean.data_ptr<float>(), rstd.data_ptr<float>(), rows, D,
                     (float)eps),
           "ln_fwd");
}

void ln_bwd_dx(at::Tensor x, at::Tensor dy, at::Tensor dx, at::Tensor gamma,
               at::Tensor mean, at::Tensor rstd, int64_t rows, int64_t D) {
  throw_on(ps_ln_bwd_dx(cur_stream(x), x.data_ptr(), dy.data_ptr(),
                        dx.data_ptr(), gamma.data_ptr(),
                        mean.data_ptr<float>(), rstd.data_ptr<float>(), rows,
                        D),
           "ln_bwd_dx");
}

void ln_bwd_dgb(at::Tensor x, at::Tensor dy, at::Tensor mean, at::Tensor rstd,
                at::Tensor dgamma, at::Tensor dbeta, int64_t rows, int64_t D) {
  throw_on(ps_ln_bwd_dgb(cur_stream(x), x.data_ptr(), dy.data_ptr(),
                         mean.data_ptr<float>(), rstd.data_ptr<float>(),
                         dgamma.data_ptr<float>(), dbeta.data_ptr<float>(),
                         rows, D),
           "ln_bwd_dgb");
}

void ce_fwd(at::Tensor logits, at::Tensor targets, at::Tensor losses,
            at::Tensor lse, int64_t T, int64_t V) {
  TORCH_CHECK(logits.is_cuda() && logits.scalar_type() == at::kBFloat16 &&
                  logits.is_contiguous(),
              "logits must be contiguous bf16");
  TORCH_CHECK(targets.scalar_type() == at::kLong, "targets must be int64");
  throw_on(ps_ce_fwd(cur_stream(logits), logits.data_ptr(),
                     targets.data_ptr<int64_t>(), losses.data_ptr<float>(),
                     lse.data_ptr<float>(), T, V),
           "ce_fwd");
}

void ce_bwd(at::Tensor logits, at::Tensor targets, at::Tensor lse,
            at::Tensor dlogits, int64_t T, int64_t V, double gscale,
            c10::optional<at::Tensor> gout) {
  const float* gp = nullptr;
  if (gout.has_value()) {
    TORCH_CHECK(gout->scalar_type() == at::kFloat && gout->numel() == 1,
                "gout must be a f32 scalar tensor");
    gp = gout->data_ptr<float>();
  }
  throw_on(ps_ce_bwd(cur_stream(logits), logits.data_ptr(),
                     targets.data_ptr<int64_t>(), lse.data_ptr<float>(),
                     dlogits.data_ptr(), T, V, (float)gscale, gp),
           "ce_bwd");
}

}  // namespace

void attn_fwd(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor o,
              at::Tensor lse, int64_t N, double scale, bool causal) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kBFloat16 &&
                  q.is_contiguous(),
              "q must be contiguous bf16");
  const int64_t rows = q.numel() / 64;
  throw_on(ps_attn_fwd(cur_stream(q), q.data_ptr(), k.data_ptr(),
                       v.data_ptr(), o.data_ptr(), lse.data_ptr<float>(),
                       rows, N, (float)scale, causal ? 1 : 0),
           "attn_fwd");
}

void attn_bwd(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor o,
              at::Tensor dout, at::Tensor lse, at::Tensor delta,
              at::Tensor dq, at::Tensor dk, at::Tensor dv, int64_t N,
              double scale, bool causal) {
  const int64_t rows = q.numel() / 64;
  throw_on(ps_attn_bwd(cur_stream(q), q.data_ptr(), k.data_ptr(),
                       v.data_ptr(), o.data_ptr(), dout.data_ptr(),
                       lse.data_ptr<float>(), delta.data_ptr<float>(),
                       dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), rows, N,
                       (float)scale, causal ? 1 : 0),
           "attn_bwd");
}

// q,k,v: [B,H,N,64] bf16 with IDENTICAL strides, unit d-stride and 16B-
// aligned rows (covers contiguous tensors and head-slices of a fused qkv
// projection, so the model path never copies); o/dq/dk/dv are contiguous.
static void fa_check_qkv(const at::Tensor& q, const at::Tensor& k,
                         const at::Tensor& v) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kBFloat16 &&
                  q.dim() == 4 && q.size(3) == 64,
              "q must be [B,H,N,64] bf16");
  TORCH_CHECK(q.stride(3) == 1 && q.stride(2) % 8 == 0 &&
                  q.stride(1) % 8 == 0 && q.stride(0) % 8 == 0,
              "q rows must be 16B-aligned with unit d-stride");
  TORCH_CHECK(k.strides() == q.strides() && v.strides() == q.strides() &&
                  k.sizes() == q.sizes() && v.sizes() == q.sizes(),
              "q/k/v must share shape and strides");
}

void fa_fwd(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor o,
            at::Tensor lse, int64_t N, double scale, bool causal) {
  fa_check_qkv(q, k, v);
  TORCH_CHECK(o.is_contiguous(), "o must be contiguous");
  const int64_t BH = q.size(0) * q.size(1);
  throw_on(ps_fa_fwd(cur_stream(q), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                     o.data_ptr(), lse.data_ptr<float>(), BH, N, (float)scale,
                     causal ? 1 : 0, q.size(1), q.stride(0), q.stride(1),
                     q.stride(2)),
           "fa_fwd");
}

void fa_bwd(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor o,
            at::Tensor dout, at::Tensor lse, at::Tensor delta, at::Tensor dq,
            at::Tensor dk, at::Tensor dv, int64_t N, double scale,
            bool causal) {
  fa_check_qkv(q, k, v);
  // dq/dk/dv may be strided views of ONE dqkv buffer (identical strides,
  // unit d-stride, 16B-aligned rows) -> backward feeds the fused qkv grad
  // directly and autograd's CatArrayBatchedCopy pass disappears
  fa_check_qkv(dq, dk, dv);
  TORCH_CHECK(o.is_contiguous() && dout.is_contiguous(),
              "o/dout must be contiguous");
  const int64_t BH = q.size(0) * q.size(1);
  throw_on(ps_fa_bwd(cur_stream(q), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                     o.data_ptr(), dout.data_ptr(), lse.data_ptr<float>(),
                     delta.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(),
                     dv.data_ptr(), BH, N, (float)scale, causal ? 1 : 0,
                     q.size(1), q.stride(0), q.stride(1), q.stride(2),
                     dq.stride(0), dq.stride(1), dq.stride(2)),
           "fa_bwd");
}

void fa_selfcheck(at::Tensor a, at::Tensor b, at::Tensor c) {
  TORCH_CHECK(a.numel() == 16 * 32 && b.numel() == 32 * 16 &&
                  c.numel() == 16 * 16,
              "selfcheck shapes: A[16,32] B[32,16] C[16,16]");
  throw_on(ps_fa_selfcheck(cur_stream(a), a.data_ptr(), b.data_ptr(),
                           c.data_ptr<float>()),
           "fa_selfcheck");
}

// ---- attention with a sliding window and visible first tokens -------------

static void wa_check(const at::Tensor& t, const char* name, const at::Tensor& q,
                    int64_t heads, int64_t* st) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 4,
              name, " must be 4-D bf16 on GPU");
  check_same_device(q, t, name);
  TORCH_CHECK(t.size(0) == q.size(0) && t.size(1) == heads &&
                  t.size(2) == q.size(2) && t.size(3) == q.size(3),
              name, " has the wrong shape");
  TORCH_CHECK(t.stride(3) == 1 && t.stride(0) % 8 == 0 &&
                  t.stride(1) % 8 == 0 && t.stride(2) % 8 == 0 &&
                  t.stride(2) < (1 << 24) && (uintptr_t)t.data_ptr() % 16 == 0,
              name, " rows must be 16B-aligned with unit d-stride");
  for (int i = 0; i < 3; ++i) st[i] = t.stride(i);
}

// [B, heads, N, D] stored as [B, N, heads, D]
static void wa_out(const at::Tensor& t, const char* name, const at::Tensor& q,
                   int64_t heads) {
  int64_t st[3];
  wa_check(t, name, q, heads, st);
  TORCH_CHECK(t.transpose(1, 2).is_contiguous(), name,
              " must be stored with heads behind rows");
}

static const int32_t* wa_lengths(const c10::optional<at::Tensor>& l,
                                 const at::Tensor& q) {
  if (!l.has_value()) return nullptr;
  check_flat(*l, at::kInt, "lengths");
  check_same_device(q, *l, "lengths");
  TORCH_CHECK(l->numel() == q.size(0), "one length for each sequence");
  return l->data_ptr<int32_t>();
}

static void wa_stat(const at::Tensor& t, const at::Tensor& q) {
  check_flat(t, at::kFloat, "row statistics");
  check_same_device(q, t, "row statistics");
  TORCH_CHECK(t.numel() == q.size(0) * q.size(1) * q.size(2),
              "row statistics size");
}

void wa_fwd(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor o,
            c10::optional<at::Tensor> low, at::Tensor lse, c10::optional<at::Tensor> lengths, int64_t window,
            int64_t sinks, double scale) {
  int64_t st[15] = {0};
  TORCH_CHECK(k.dim() == 4 && q.dim() == 4, "q, k must be 4-D");
  wa_check(q, "q", q, q.size(1), st);
  wa_check(k, "k", q, k.size(1), st + 3);
  wa_check(v, "v", q, k.size(1), st + 6);
  wa_out(o, "o", q, q.size(1));
  if (low) wa_out(*low, "low", q, q.size(1));
  wa_stat(lse, q);
  const int32_t* len = wa_lengths(lengths, q);
  const c10::DeviceGuard guard(q.device());
  throw_on(ps_wa_fwd(cur_stream(q), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                     o.data_ptr(), low ? low->data_ptr() : nullptr,
                     lse.data_ptr<float>(), len, st, q.size(0),
                     q.size(1), k.size(1), q.size(2), q.size(3), window, sinks,
                     (float)scale),
           "wa_fwd");
}

void wa_bwd(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor o,
            at::Tensor low, at::Tensor go, at::Tensor lse, at::Tensor delta, at::Tensor dq,
            at::Tensor dk, at::Tensor dv, at::Tensor part,
            c10::optional<at::Tensor> lengths, int64_t window, int64_t sinks,
            double scale) {
  int64_t st[15];
  TORCH_CHECK(k.dim() == 4 && q.dim() == 4, "q, k must be 4-D");
  wa_check(q, "q", q, q.size(1), st);
  wa_check(k, "k", q, k.size(1), st + 3);
  wa_check(v, "v", q, k.size(1), st + 6);
  wa_check(o, "o", q, q.size(1), st + 9);
  wa_out(low, "low", q, q.size(1));
  wa_check(go, "dout", q, q.size(1), st + 12);
  wa_out(dq, "dq", q, q.size(1));
  wa_out(dk, "dk", q, k.size(1));
  wa_out(dv, "dv", q, k.size(1));
  wa_stat(lse, q);
  wa_stat(delta, q);
  check_flat(part, at::kFloat, "part");
  check_same_device(q, part, "part");
  TORCH_CHECK(part.numel() >= ps_wa_part_floats(q.size(0), q.size(1), k.size(1),
                                                q.size(2), q.size(3), window,
                                                sinks),
              "part too small");
  const int32_t* len = wa_lengths(lengths, q);
  const c10::DeviceGuard guard(q.device());
  throw_on(ps_wa_bwd(cur_stream(q), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                     o.data_ptr(), low.data_ptr(), go.data_ptr(),
                     lse.data_ptr<float>(),
                     delta.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(),
                     dv.data_ptr(), part.data_ptr<float>(), len, st, q.size(0),
                     q.size(1), k.size(1), q.size(2), q.size(3), window, sinks,
                     (float)scale),
           "wa_bwd");
}

// t as the kernels read it: unit d stride, rows that start at 16 bytes and 64
// of them within 32-bit byte offsets.
static at::Tensor wa_rows16(const at::Tensor& t) {
  if (t.stride(3) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 &&
      t.stride(2) % 8 == 0 && t.stride(2) < (1 << 24) &&
      (uintptr_t)t.data_ptr() % 16 == 0)
    return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

// [B, heads, N, D] stored with heads behind rows: what follows is a projection
// of all heads
static at::Tensor wa_empty(int64_t B, int64_t heads, int64_t N, int64_t D,
                           const at::Tensor& like) {
  return at::empty_strided({B, heads, N, D}, {N * heads * D, D, heads * D, 1},
                           like.options());
}

struct WindowSdpa : torch::autograd::Function<WindowSdpa> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx,
                            const at::Tensor& q_, const at::Tensor& k_,
                            const at::Tensor& v_,
                            const c10::optional<at::Tensor>& lengths,
                            int64_t window, int64_t sinks, double scale,
                            bool grad) {
    TORCH_CHECK(q_.is_cuda() && q_.dim() == 4 && k_.dim() == 4 &&
                    v_.dim() == 4, "q, k, v must be 4-D on GPU");
    const c10::DeviceGuard guard(q_.device());
    const auto q = wa_rows16(q_), k = wa_rows16(k_), v = wa_rows16(v_);
    auto o = wa_empty(q.size(0), q.size(1), q.size(2), q.size(3), q);
    auto lse = at::empty({q.size(0), q.size(1), q.size(2)},
                         q.options().dtype(at::kFloat));
    const at::Tensor len = lengths.has_value() ? lengths->contiguous()
                                               : at::Tensor();
    c10::optional<at::Tensor> low;
    if (grad) low = wa_empty(q.size(0), q.size(1), q.size(2), q.size(3), q);
    wa_fwd(q, k, v, o, low, lse, len.defined() ? c10::optional<at::Tensor>(len)
                                          : c10::optional<at::Tensor>(),
           window, sinks, scale);
    ctx->save_for_backward({q, k, v, o, lse, len, low ? *low : at::Tensor()});
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["scale"] = scale;
    return o;
  }
  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx,
      torch::autograd::variable_list g) {
    first_order("fused_window_sdpa");
    const auto s = ctx->get_saved_variables();
    const auto &q = s[0], &k = s[1];
    const int64_t B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3),
                  KV = k.size(1);
    const int64_t window = ctx->saved_data["window"].toInt(),
                  sinks = ctx->saved_data["sinks"].toInt();
    const c10::DeviceGuard guard(q.device());
    auto dq = wa_empty(B, H, N, D, q), dk = wa_empty(B, KV, N, D, q),
         dv = wa_empty(B, KV, N, D, q);
    auto delta = at::empty_like(s[4]);
    auto part = at::empty({ps_wa_part_floats(B, H, KV, N, D, window, sinks)},
                          q.options().dtype(at::kFloat));
    wa_bwd(q, k, s[2], s[3], s[6], wa_rows16(g[0]), s[4], delta, dq, dk, dv, part,
           s[5].defined() ? c10::optional<at::Tensor>(s[5])
                          : c10::optional<at::Tensor>(),
           window, sinks, ctx->saved_data["scale"].toDouble());
    return {dq, dk, dv, at::Tensor(), at::Tensor(), at::Tensor(),
            at::Tensor(), at::Tensor()};
  }
};

static at::Tensor window_sdpa(at::Tensor q, at::Tensor k, at::Tensor v,
                              int64_t window, int64_t sinks,
                              c10::optional<at::Tensor> lengths,
                              double scale) {
  const bool grad = at::GradMode::is_enabled() &&
      (q.requires_grad() || k.requires_grad() || v.requires_grad());
  return WindowSdpa::apply(q, k, v, lengths, window, sinks, scale, grad);
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("attn_fwd", &attn_fwd);
  m.def("attn_bwd", &attn_bwd);
  m.def("fa_fwd", &fa_fwd, "MFMA-tiled flash attention forward");
  m.def("fa_bwd", &fa_bwd, "MFMA-tiled flash attention backward");
  m.def("fa_selfcheck", &fa_selfcheck, "16x16x32 MFMA fragment-layout check");
  m.def("window_sdpa", &window_sdpa,
        "causal attention, sliding window and sinks, with its gradient");
  m.def("topk_encode_thresh", &topk_encode_thresh,
        "variable-k magnitude-threshold select (k_used -> device header)");
  m.def("colsum", &colsum, "column sum (bias grads)");
  m.def("topk_scatter_var", &topk_scatter_var,
        "scatter-add with device-side k header");
  m.def("ce_fwd", &ce_fwd);
  m.def("ce_bwd", &ce_bwd);
  m.def("ln_fwd", &ln_fwd);
  m.def("ln_bwd_dx", &ln_bwd_dx);
  m.def("ln_bwd_dgb", &ln_bwd_dgb);
  m.def("bn_fwd_stats", &bn_fwd_stats);
  m.def("bn_finalize", &bn_finalize);
  m.def("bn_eval_coef", &bn_eval_coef);
  m.def("bn_normalize", &bn_normalize);
  m.def("bn_bwd_stats", &bn_bwd_stats);
  m.def("bn_bwd_coef", &bn_bwd_coef);
  m.def("bn_bwd_dx", &bn_bwd_dx);
  m.def("fused_sgd", &fused_sgd, "fused SGD over flat fp32 buffers");
  m.def("fused_adam", &fused_adam, "fused Adam over flat fp32 buffers");
  m.def("fused_adamw", &fused_adamw,
        "AdamW over packed fp32 buffers, states in 32 or 8 bits");
  m.def("state8_values", &state8_values, "values that 8-bit codes stand for");
  m.def("rope", &rope, "rotary positions with several axes, q and k at once");
  m.def("gated_residual", &gated_residual,
        "post norm, gate, residual, pre norm, with their gradients");
  m.def("reduce_accum", &reduce_accum, "dst = beta*dst + scale*sum(srcs)");
  m.def("f32_to_bf16", &f32_to_bf16, "flat cast");
  m.def("bf16_to_f32", &bf16_to_f32, "flat cast");
  m.def("quant8_encode", &quant8_encode, "per-256-chunk absmax int8 quantize");
  m.def("quant8_reduce", &quant8_reduce, "dequant+sum int8 messages");
  m.def("topk_workspace_words", &topk_workspace_words);
  m.def("topk_encode", &topk_encode, "magnitude top-k -> (idx, val)");
  m.def("topk_scatter", &topk_scatter, "dst[idx] += gscale*val (one message)");
}
