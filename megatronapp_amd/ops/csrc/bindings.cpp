// PyTorch bindings for the megatronapp_amd CDNA4 kernels.
// Built in-tree to megatronapp_amd/ops/_C.so (see ops/setup.py).

#include <torch/extension.h>

#include <ATen/hip/HIPContext.h>
#include <c10/core/AutogradState.h>

#include <cmath>

// launchers (norms.hip / elementwise.hip / rope.hip / softmax.hip / adam.hip /
// attention.hip)
void launch_rmsnorm_fwd(const void*, const void*, void*, float*, int, int,
                        float, hipStream_t);
void launch_rmsnorm_bwd(const void*, const void*, const void*, const float*,
                        void*, float*, float*, const void*, int, int, int,
                        hipStream_t);
void launch_layernorm_fwd(const void*, const void*, const void*, void*, float*,
                          float*, int, int, float, hipStream_t);
void launch_layernorm_bwd(const void*, const void*, const void*, const float*,
                          const float*, void*, float*, float*, float*, float*,
                          const void*, int, int, int, hipStream_t);
void launch_bias_add_residual(const void*, const void*, const void*, void*,
                              long, int, hipStream_t);
void launch_bias_gelu_fwd(const void*, const void*, void*, long, int,
                          hipStream_t);
void launch_bias_gelu_bwd(const void*, const void*, const void*, void*, long,
                          int, hipStream_t);
void launch_bias_swiglu_fwd(const void*, const void*, void*, long, int,
                            hipStream_t);
void launch_bias_swiglu_bwd(const void*, const void*, const void*, void*, long,
                            int, hipStream_t);
void launch_bias_geglu_fwd(const void*, const void*, void*, long, int,
                           hipStream_t);
void launch_bias_geglu_bwd(const void*, const void*, const void*, void*,
                           long, int, hipStream_t);
void launch_rope(const void*, const float*, const float*, void*, long, int,
                 int, bool, hipStream_t);
void launch_softmax_causal_fwd(const void*, void*, long, int, int, float,
                               hipStream_t);
void launch_softmax_masked_fwd(const void*, const void*, void*, long, int, int,
                               int, float, hipStream_t);
void launch_softmax_causal_bwd(const void*, const void*, void*, long, int,
                               int, float, hipStream_t);
void launch_softmax_bwd(const void*, const void*, void*, long, int, float,
                        hipStream_t);
void launch_adamw_flat_ranged(float*, const float*, void*, void*,
                              bool, void*, const long*, const long*,
                              int, long, float, float, float, float,
                              float, int, hipStream_t);
void launch_ce_rowmax(const void*, float*, long, int, hipStream_t);
void launch_ce_fwd(const void*, const float*, const int*, float*, float*,
                   long, int, hipStream_t);
void launch_ce_bwd(const void*, const float*, const float*, const int*,
                   const float*, void*, long, int, hipStream_t);
void launch_selective_scan_fwd(const void*, const void*, const float*,
                               const void*, const void*, const float*, float*,
                               void*, int, int, int, int, hipStream_t);
void launch_adamw_flat(float*, const float*, void*, void*, bool,
                       void*, long, float, float, float, float,
                       float, int, hipStream_t);
void wgrad_accum(torch::Tensor, torch::Tensor, torch::Tensor);
bool wgrad_accum_bgrad(torch::Tensor, torch::Tensor, torch::Tensor,
                       torch::Tensor);
torch::Tensor gemm_nt(torch::Tensor, torch::Tensor);
torch::Tensor gemm_nn(torch::Tensor, torch::Tensor);
int colsum_grid_y(long, int);
void launch_colsum_accum(const void*, float*, float*, int, long, int,
                         hipStream_t);
void launch_embedding_bwd_accum(const void*, const int*, float*, long, int,
                                hipStream_t);
void launch_transpose_quant_e4m3(const void*, void*, unsigned int*,
                                 float*, long, long, hipStream_t);
void launch_quant_rows_e4m3(const void*, void*, float*, long, int,
                            hipStream_t);
void launch_bias_dropout_add_fwd(const void*, const void*, const void*,
                                 void*, unsigned char*, long, int, float,
                                 unsigned long long, hipStream_t);
void launch_dropout_bwd(const void*, const unsigned char*, void*, long,
                        float, hipStream_t);
void launch_moe_combine_fwd(const void*, const long*, const float*, void*,
                            long, int, int, hipStream_t);
void launch_moe_combine_bwd(const void*, const void*, const long*,
                            const float*, void*, float*, long, int, int,
                            hipStream_t);
void launch_attn_fwd2(const void*, const void*, const void*, void*, float*,
                      int, int, int, int, int, int, float, bool,
                      const long*, const long*, const long*, hipStream_t);
void launch_attn_bwd2(const void*, const void*, const void*, const void*,
                      const void*, const float*, float*, void*, void*, void*,
                      int, int, int, int, int, int, float, bool, const long*,
                      const long*, const long*, const long*, const long*,
                      const long*, hipStream_t);

// The round-2 kernels take (seq, batch, head) element strides so the
// strided QKV-split views feed them without .contiguous() copies; d
// must be unit-stride.
static bool attn_strides(const torch::Tensor& t, long* out) {
  if (t.stride(3) != 1) return false;
  out[0] = (long)t.stride(0);
  out[1] = (long)t.stride(1);
  out[2] = (long)t.stride(2);
  return true;
}
void launch_attn_fwd_t(const void*, const void*, const void*, void*, float*,
                       int, int, int, int, int, int, float, bool,
                       hipStream_t);
void launch_attn_fwd(const void*, const void*, const void*, void*, float*,
                     int, int, int, int, int, int, float, bool, hipStream_t);
void launch_attn_fwd_ablate(const void*, const void*, const void*, void*,
                            float*, int, int, int, int, int, int, float, int,
                            hipStream_t);
void launch_attn_bwd(const void*, const void*, const void*, const void*,
                     const void*, const float*, float*, void*, void*, void*,
                     int, int, int, int, int, int, float, bool, hipStream_t);

void launch_packed_attn_fwd(const void*, const void*, const void*, void*,
                            void*, float*, const int*, const int*, int, int,
                            int, int, int, int, int, float, bool, bool,
                            const long*, const long*, const long*,
                            hipStream_t);
int packed_attn_shares(int, int, int, int, int, int, int, long*);
void launch_packed_attn_bwd(const void*, const void*, const void*,
                            const void*, const void*, const void*,
                            const float*, float*, void*, void*, void*, float*,
                            int, const int*, const int*, int, int, int, int,
                            int, int, int, float, bool, bool,
                            const long*, const long*, const long*, const long*,
                            hipStream_t);

void launch_cache_fork(int*, int*, int*, int*, int, int, int, int, void*, int,
                       int, int, const int*, const int*, int, int*,
                       hipStream_t);
void launch_cache_free(int*, int*, int*, int*, int, int, int, int, const int*,
                       int, hipStream_t);
void launch_cache_compact(int*, int*, int*, int*, int, int, int, int, void*,
                          int, long, int*, hipStream_t);
void launch_cache_copy(const int*, const int*, int, void*, int, int, long,
                       int*, hipStream_t);
void launch_cache_extend(int*, int*, int*, int*, int, int, int, int,
                         const int*, const int*, int, int, int*, hipStream_t);
void launch_cache_write(int*, int*, int*, int*, int, int, int, int, const int*,
                        const int*, int, int, void*, void*, const void*,
                        const void*, int, int, long, long, long, long,
                        hipStream_t);
void paged_attn_pieces(int, int, int, int, int, int, int, long, int*, int*,
                       int*, int*);
void launch_paged_attn(const void*, long, long, const void*, const void*,
                       const long*, const long*, const int*, const int*,
                       const int*, const int*, const int*, int, int, int, int,
                       int, int, int, int, int, int, int, int, int, int,
                       void*,
                       float*,
                       float*, float, bool, hipStream_t);

namespace {

hipStream_t cur_stream() {
  return at::hip::getCurrentHIPStream().stream();
}

void check_bf16(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be on GPU");
  TORCH_CHECK(t.scalar_type() == torch::kBFloat16, name, " must be bf16");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

// attention inputs may be strided views (d contiguous); no contiguity check
void check_bf16_any(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be on GPU");
  TORCH_CHECK(t.scalar_type() == torch::kBFloat16, name, " must be bf16");
}

// ------------------------------------------------------------------- norms
std::vector<torch::Tensor> rmsnorm_fwd(torch::Tensor x, torch::Tensor w,
                                       double eps) {
  check_bf16(x, "x");
  check_bf16(w, "w");
  const int H = (int)x.size(-1);
  const long N = x.numel() / H;
  auto y = torch::empty_like(x);
  auto invrms = torch::empty({N}, x.options().dtype(torch::kFloat32));
  launch_rmsnorm_fwd(x.data_ptr(), w.data_ptr(), y.data_ptr(),
                     invrms.data_ptr<float>(), (int)N, H, (float)eps,
                     cur_stream());
  return {y, invrms};
}

std::vector<torch::Tensor> rmsnorm_bwd(torch::Tensor dy, torch::Tensor x,
                                       torch::Tensor w, torch::Tensor invrms,
                                       c10::optional<torch::Tensor> mg_w,
                                       c10::optional<torch::Tensor> dres) {
  check_bf16(dy, "dy");
  check_bf16(x, "x");
  const int H = (int)x.size(-1);
  const long N = x.numel() / H;
  auto dx = torch::empty_like(x);
  auto dw = mg_w.has_value()
                ? *mg_w
                : torch::zeros({H}, x.options().dtype(torch::kFloat32));
  // 2048 blocks = up to 8/CU: a block sits at two block-wide barrier
  // reductions per row, so a 512-block launch left the CUs idle
  const int grid = (int)std::min<long>(N, 2048);
  auto dw_part = torch::empty({grid, H}, x.options().dtype(torch::kFloat32));
  const void* dres_p = nullptr;
  torch::Tensor dres_c;
  if (dres.has_value()) {
    check_bf16(*dres, "dres");
    dres_c = dres->contiguous();
    dres_p = dres_c.data_ptr();
  }
  launch_rmsnorm_bwd(dy.data_ptr(), x.data_ptr(), w.data_ptr(),
                     invrms.data_ptr<float>(), dx.data_ptr(),
                     dw.data_ptr<float>(), dw_part.data_ptr<float>(), dres_p,
                     grid, (int)N, H, cur_stream());
  return {dx, dw};
}

std::vector<torch::Tensor> layernorm_fwd(torch::Tensor x, torch::Tensor w,
                                         torch::Tensor b, double eps) {
  check_bf16(x, "x");
  const int H = (int)x.size(-1);
  const long N = x.numel() / H;
  auto y = torch::empty_like(x);
  auto mean = torch::empty({N}, x.options().dtype(torch::kFloat32));
  auto invstd = torch::empty({N}, x.options().dtype(torch::kFloat32));
  launch_layernorm_fwd(x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(),
                       mean.data_ptr<float>(), invstd.data_ptr<float>(),
                       (int)N, H, (float)eps, cur_stream());
  return {y, mean, invstd};
}

std::vector<torch::Tensor> layernorm_bwd(torch::Tensor dy, torch::Tensor x,
                                         torch::Tensor w, torch::Tensor mean,
                                         torch::Tensor invstd,
                                         c10::optional<torch::Tensor> mg_w,
                                         c10::optional<torch::Tensor> mg_b,
                                         c10::optional<torch::Tensor> dres) {
  check_bf16(dy, "dy");
  const int H = (int)x.size(-1);
  const long N = x.numel() / H;
  auto dx = torch::empty_like(x);
  auto dw = mg_w.has_value()
                ? *mg_w
                : torch::zeros({H}, x.options().dtype(torch::kFloat32));
  auto db = mg_b.has_value()
                ? *mg_b
                : torch::zeros({H}, x.options().dtype(torch::kFloat32));
  // 2048 blocks = up to 8/CU: a block sits at two block-wide barrier
  // reductions per row, so a 512-block launch left the CUs idle
  const int grid = (int)std::min<long>(N, 2048);
  auto part = torch::empty({2, grid, H}, x.options().dtype(torch::kFloat32));
  const void* dres_p = nullptr;
  torch::Tensor dres_c;
  if (dres.has_value()) {
    check_bf16(*dres, "dres");
    dres_c = dres->contiguous();
    dres_p = dres_c.data_ptr();
  }
  launch_layernorm_bwd(dy.data_ptr(), x.data_ptr(), w.data_ptr(),
                       mean.data_ptr<float>(), invstd.data_ptr<float>(),
                       dx.data_ptr(), dw.data_ptr<float>(),
                       db.data_ptr<float>(), part[0].data_ptr<float>(),
                       part[1].data_ptr<float>(), dres_p, grid, (int)N, H,
                       cur_stream());
  return {dx, dw, db};
}

// -------------------------------------------------------------- elementwise
torch::Tensor bias_gelu_fwd(torch::Tensor x, c10::optional<torch::Tensor> bias) {
  check_bf16(x, "x");
  auto y = torch::empty_like(x);
  const int F = (int)x.size(-1);
  TORCH_CHECK(x.numel() % 8 == 0 && (!bias.has_value() || F % 8 == 0),
              "bias_gelu: numel and F must be multiples of 8");
  launch_bias_gelu_fwd(x.data_ptr(),
                       bias.has_value() ? bias->data_ptr() : nullptr,
                       y.data_ptr(), x.numel(), F, cur_stream());
  return y;
}

torch::Tensor bias_add_residual(torch::Tensor x, torch::Tensor bias,
                                torch::Tensor res) {
  TORCH_CHECK(x.is_cuda() && x.dtype() == torch::kBFloat16);
  TORCH_CHECK(x.is_contiguous() && res.is_contiguous() &&
              bias.is_contiguous());
  TORCH_CHECK(x.sizes() == res.sizes());
  int F = bias.numel();
  TORCH_CHECK(x.size(-1) == F && F % 8 == 0);
  auto y = torch::empty_like(x);
  launch_bias_add_residual(x.data_ptr(), bias.data_ptr(), res.data_ptr(),
                           y.data_ptr(), x.numel(), F,
                           at::cuda::getCurrentCUDAStream());
  return y;
}

torch::Tensor bias_gelu_bwd(torch::Tensor dy, torch::Tensor x,
                            c10::optional<torch::Tensor> bias) {
  check_bf16(dy, "dy");
  auto dx = torch::empty_like(x);
  const int F = (int)x.size(-1);
  TORCH_CHECK(x.numel() % 8 == 0 && (!bias.has_value() || F % 8 == 0),
              "bias_gelu: numel and F must be multiples of 8");
  launch_bias_gelu_bwd(dy.data_ptr(), x.data_ptr(),
                       bias.has_value() ? bias->data_ptr() : nullptr,
                       dx.data_ptr(), x.numel(), F, cur_stream());
  return dx;
}

torch::Tensor bias_swiglu_fwd(torch::Tensor x, c10::optional<torch::Tensor> bias) {
  check_bf16(x, "x");
  const int F2 = (int)x.size(-1);
  TORCH_CHECK(F2 % 2 == 0, "last dim must be even (gated)");
  const int F = F2 / 2;
  const long N = x.numel() / F2;
  auto sizes = x.sizes().vec();
  sizes.back() = F;
  auto y = torch::empty(sizes, x.options());
  launch_bias_swiglu_fwd(x.data_ptr(),
                         bias.has_value() ? bias->data_ptr() : nullptr,
                         y.data_ptr(), N, F, cur_stream());
  return y;
}

torch::Tensor bias_swiglu_bwd(torch::Tensor dy, torch::Tensor x,
                              c10::optional<torch::Tensor> bias) {
  check_bf16(dy, "dy");
  const int F2 = (int)x.size(-1);
  const int F = F2 / 2;
  const long N = x.numel() / F2;
  auto dx = torch::empty_like(x);
  launch_bias_swiglu_bwd(dy.data_ptr(), x.data_ptr(),
                         bias.has_value() ? bias->data_ptr() : nullptr,
                         dx.data_ptr(), N, F, cur_stream());
  return dx;
}

torch::Tensor bias_geglu_fwd(torch::Tensor x, c10::optional<torch::Tensor> bias) {
  check_bf16(x, "x");
  const int F2 = (int)x.size(-1);
  TORCH_CHECK(F2 % 2 == 0, "last dim must be even (gated)");
  const int F = F2 / 2;
  const long N = x.numel() / F2;
  auto sizes = x.sizes().vec();
  sizes.back() = F;
  auto y = torch::empty(sizes, x.options());
  launch_bias_geglu_fwd(x.data_ptr(),
                         bias.has_value() ? bias->data_ptr() : nullptr,
                         y.data_ptr(), N, F, cur_stream());
  return y;
}

torch::Tensor bias_geglu_bwd(torch::Tensor dy, torch::Tensor x,
                              c10::optional<torch::Tensor> bias) {
  check_bf16(dy, "dy");
  const int F2 = (int)x.size(-1);
  const int F = F2 / 2;
  const long N = x.numel() / F2;
  auto dx = torch::empty_like(x);
  launch_bias_geglu_bwd(dy.data_ptr(), x.data_ptr(),
                         bias.has_value() ? bias->data_ptr() : nullptr,
                         dx.data_ptr(), N, F, cur_stream());
  return dx;
}

// --------------------------------------------------------------------- rope
torch::Tensor rope_apply(torch::Tensor t, torch::Tensor cs, torch::Tensor sn,
                         bool bwd) {
  check_bf16(t, "t");
  TORCH_CHECK(cs.scalar_type() == torch::kFloat32, "cos table must be fp32");
  const int d = (int)t.size(-1);
  const long rows = t.numel() / d;
  // cs/sn come in as [s, 1, 1, d]; rows per seq position = b*nh
  const long s = cs.numel() / d;
  const int bnh = (int)(rows / s);
  auto out = torch::empty_like(t);
  launch_rope(t.data_ptr(), cs.data_ptr<float>(), sn.data_ptr<float>(),
              out.data_ptr(), rows, bnh, d, bwd, cur_stream());
  return out;
}

torch::Tensor rope_fwd(torch::Tensor t, torch::Tensor cs, torch::Tensor sn) {
  return rope_apply(t, cs.contiguous(), sn.contiguous(), false);
}

torch::Tensor rope_bwd(torch::Tensor dy, torch::Tensor cs, torch::Tensor sn) {
  return rope_apply(dy, cs.contiguous(), sn.contiguous(), true);
}

// ------------------------------------------------------------------ softmax
torch::Tensor scaled_softmax_fwd(torch::Tensor x, double scale) {
  // no-mask row softmax (reference scaled_softmax_cuda): the masked
  // kernel with a null mask pointer
  check_bf16(x, "x");
  const int sk = (int)x.size(-1);
  const int sq = (int)x.size(-2);
  const long rows = x.numel() / sk;
  auto y = torch::empty_like(x);
  launch_softmax_masked_fwd(x.data_ptr(), nullptr, y.data_ptr(), rows,
                            1, sq, sk, (float)scale, cur_stream());
  return y;
}

torch::Tensor scaled_upper_triang_masked_softmax_fwd(torch::Tensor x,
                                                     double scale) {
  check_bf16(x, "x");
  const int sk = (int)x.size(-1);
  const int sq = (int)x.size(-2);
  const long rows = x.numel() / sk;
  auto y = torch::empty_like(x);
  launch_softmax_causal_fwd(x.data_ptr(), y.data_ptr(), rows, sq, sk,
                            (float)scale, cur_stream());
  return y;
}

torch::Tensor scaled_masked_softmax_fwd(torch::Tensor x,
                                        c10::optional<torch::Tensor> mask,
                                        double scale) {
  check_bf16(x, "x");
  // x: [b, np, sq, sk]; mask: [b or 1, np or 1, sq or 1, sk], or without np
  const int sk = (int)x.size(-1);
  const int sq = (int)x.size(-2);
  int np = (int)x.size(1);
  const long rows = x.numel() / sk;
  auto y = torch::empty_like(x);
  const void* mptr = nullptr;
  torch::Tensor m8;
  if (mask.has_value()) {
    const auto m = mask->dim() == 3 ? mask->unsqueeze(1) : *mask;
    TORCH_CHECK(x.dim() == 4 && m.dim() == 4,
                "scaled_masked_softmax: x must be [b, np, sq, sk], mask "
                "[b, np, sq, sk] or [b, sq, sk]");
    // the kernel reads a mask for each of the batch, or for each row of it
    const bool heads = m.size(1) != 1;
    m8 = m.expand({x.size(0), heads ? np : 1, sq, sk})
             .to(torch::kUInt8)
             .contiguous();
    if (heads) np = 1;
    mptr = m8.data_ptr();
  }
  launch_softmax_masked_fwd(x.data_ptr(), mptr, y.data_ptr(), rows, np, sq, sk,
                            (float)scale, cur_stream());
  return y;
}

torch::Tensor scaled_softmax_bwd(torch::Tensor dy, torch::Tensor p,
                                 double scale) {
  check_bf16(dy, "dy");
  const int sk = (int)dy.size(-1);
  const long rows = dy.numel() / sk;
  auto dx = torch::empty_like(dy);
  launch_softmax_bwd(dy.data_ptr(), p.data_ptr(), dx.data_ptr(), rows, sk,
                     (float)scale, cur_stream());
  return dx;
}

torch::Tensor scaled_upper_triang_masked_softmax_bwd(torch::Tensor dy,
                                                     torch::Tensor p,
                                                     double scale) {
  check_bf16(dy, "dy");
  const int sk = (int)dy.size(-1);
  const int sq = (int)dy.size(-2);
  const long rows = dy.numel() / sk;
  auto dx = torch::empty_like(dy);
  launch_softmax_causal_bwd(dy.data_ptr(), p.data_ptr(), dx.data_ptr(), rows,
                            sq, sk, (float)scale, cur_stream());
  return dx;
}

torch::Tensor colsum_accum(torch::Tensor dy, torch::Tensor out) {
  check_bf16(dy, "dy");
  TORCH_CHECK(out.scalar_type() == torch::kFloat32 && out.is_contiguous());
  const int F = (int)dy.size(-1);
  const long R = dy.numel() / F;
  const int gy = colsum_grid_y(R, F);
  torch::Tensor part;
  float* part_p = nullptr;
  if (gy > 0) {
    part = torch::empty({(long)gy, (long)F},
                        out.options().dtype(torch::kFloat32));
    part_p = part.data_ptr<float>();
  }
  launch_colsum_accum(dy.data_ptr(), out.data_ptr<float>(), part_p, gy, R, F,
                      cur_stream());
  return out;
}

void embedding_bwd_accum(torch::Tensor dy, torch::Tensor tokens,
                         torch::Tensor main_grad) {
  check_bf16(dy, "dy");
  TORCH_CHECK(tokens.scalar_type() == torch::kInt32 && tokens.is_contiguous());
  TORCH_CHECK(main_grad.scalar_type() == torch::kFloat32 &&
              main_grad.is_contiguous());
  const int H = (int)dy.size(-1);
  const long ntok = dy.numel() / H;
  TORCH_CHECK(tokens.numel() == ntok);
  launch_embedding_bwd_accum(dy.data_ptr(), tokens.data_ptr<int>(),
                             main_grad.data_ptr<float>(), ntok, H,
                             cur_stream());
}

// ------------------------------------------------------------- dropout
std::vector<torch::Tensor> bias_dropout_add_fwd(
    torch::Tensor x, torch::Tensor bias, torch::Tensor residual, double p,
    long seed) {
  check_bf16(x, "x");
  check_bf16(residual, "residual");
  auto out = torch::empty_like(x);
  auto mask = torch::empty(x.sizes(), x.options().dtype(torch::kUInt8));
  const long n = x.numel();
  const int F = (int)x.size(-1);
  launch_bias_dropout_add_fwd(
      x.data_ptr(), bias.defined() ? bias.data_ptr() : nullptr,
      residual.data_ptr(), out.data_ptr(), mask.data_ptr<unsigned char>(),
      n, F, (float)p, (unsigned long long)seed, cur_stream());
  return {out, mask};
}

torch::Tensor dropout_bwd(torch::Tensor dy, torch::Tensor mask, double p) {
  check_bf16(dy, "dy");
  auto dx = torch::empty_like(dy);
  launch_dropout_bwd(dy.contiguous().data_ptr(),
                     mask.data_ptr<unsigned char>(), dx.data_ptr(),
                     dy.numel(), (float)p, cur_stream());
  return dx;
}

// ---------------------------------------------------------------- moe
torch::Tensor moe_combine_fwd(torch::Tensor permuted, torch::Tensor inv_pos,
                              torch::Tensor probs, long n_tokens) {
  check_bf16(permuted, "permuted");
  const int h = (int)permuted.size(-1);
  const int topk = (int)(permuted.size(0) / n_tokens);
  auto out = torch::empty({n_tokens, (long)h}, permuted.options());
  launch_moe_combine_fwd(permuted.data_ptr(), inv_pos.data_ptr<long>(),
                         probs.data_ptr<float>(), out.data_ptr(), n_tokens,
                         topk, h, cur_stream());
  return out;
}

std::vector<torch::Tensor> moe_combine_bwd(torch::Tensor dout,
                                           torch::Tensor permuted,
                                           torch::Tensor sort_idx,
                                           torch::Tensor probs, long topk) {
  check_bf16(dout, "dout");
  check_bf16(permuted, "permuted");
  const int h = (int)permuted.size(-1);
  const long n_rows = permuted.size(0);
  auto dpermuted = torch::empty_like(permuted);
  auto dprobs = torch::empty({n_rows}, probs.options());
  launch_moe_combine_bwd(dout.contiguous().data_ptr(), permuted.data_ptr(),
                         sort_idx.data_ptr<long>(), probs.data_ptr<float>(),
                         dpermuted.data_ptr(), dprobs.data_ptr<float>(),
                         n_rows, (int)topk, h, cur_stream());
  return {dpermuted, dprobs};
}

// ---------------------------------------------------------------- fp8 quant
// [R, C] bf16 -> ([C, R] e4m3, [1] f32 per-tensor scale): wgrad operands
// (fp8 MFMA wants the token dim innermost on both sides)
std::vector<torch::Tensor> quantize_transpose_e4m3(torch::Tensor x) {
  check_bf16(x, "x");
  TORCH_CHECK(x.dim() == 2, "expects 2D");
  const long R = x.size(0), C = x.size(1);
  auto q = torch::empty({C, R}, x.options().dtype(torch::kFloat8_e4m3fn));
  auto s = torch::empty({1}, x.options().dtype(torch::kFloat32));
  auto amax = torch::zeros({1}, x.options().dtype(torch::kInt32));
  launch_transpose_quant_e4m3(x.data_ptr(), q.data_ptr(),
                              (unsigned int*)amax.data_ptr(),
                              s.data_ptr<float>(), R, C, cur_stream());
  return {q, s};
}

std::vector<torch::Tensor> quantize_rows_e4m3(torch::Tensor x) {
  check_bf16(x, "x");
  auto x2 = x.reshape({-1, x.size(-1)}).contiguous();
  const long M = x2.size(0);
  const int K = (int)x2.size(1);
  auto q = torch::empty({M, (long)K},
                        x.options().dtype(torch::kFloat8_e4m3fn));
  auto s = torch::empty({M, 1}, x.options().dtype(torch::kFloat32));
  launch_quant_rows_e4m3(x2.data_ptr(), q.data_ptr(), s.data_ptr<float>(),
                         M, K, cur_stream());
  return {q, s};
}

// ---------------------------------------------------------------- attention
std::vector<torch::Tensor> attn_fwd(torch::Tensor q, torch::Tensor k,
                                    torch::Tensor v, double scale,
                                    bool causal) {
  check_bf16_any(q, "q");
  check_bf16_any(k, "k");
  check_bf16_any(v, "v");
  const int sq = (int)q.size(0), b = (int)q.size(1), nh = (int)q.size(2),
            d = (int)q.size(3);
  const int sk = (int)k.size(0), ng = (int)k.size(2);
  auto o = torch::empty({sq, b, nh, d}, q.options());
  auto lse = torch::empty({b, nh, sq}, q.options().dtype(torch::kFloat32));
  long qs[3], ks[3], vs[3];
  if ((d == 128 || d == 64) && sq % 256 == 0 && sk % 64 == 0 &&
      attn_strides(q, qs) &&
      attn_strides(k, ks) && attn_strides(v, vs)) {
    launch_attn_fwd2(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                     lse.data_ptr<float>(), sq, sk, b, nh, ng, d,
                     (float)scale, causal, qs, ks, vs, cur_stream());
  } else {
    auto qc = q.contiguous(), kc = k.contiguous(), vc = v.contiguous();
    launch_attn_fwd(qc.data_ptr(), kc.data_ptr(), vc.data_ptr(), o.data_ptr(),
                    lse.data_ptr<float>(), sq, sk, b, nh, ng, d, (float)scale,
                    causal, cur_stream());
  }
  return {o, lse};
}

std::vector<torch::Tensor> attn_fwd_t(torch::Tensor q, torch::Tensor k,
                                    torch::Tensor v, double scale,
                                    bool causal) {
  check_bf16_any(q, "q");
  check_bf16_any(k, "k");
  check_bf16_any(v, "v");
  const int sq = (int)q.size(0), b = (int)q.size(1), nh = (int)q.size(2),
            d = (int)q.size(3);
  const int sk = (int)k.size(0), ng = (int)k.size(2);
  auto o = torch::empty_like(q);
  auto lse = torch::empty({b, nh, sq}, q.options().dtype(torch::kFloat32));
  launch_attn_fwd_t(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                  lse.data_ptr<float>(), sq, sk, b, nh, ng, d, (float)scale,
                  causal, cur_stream());
  return {o, lse};
}

std::vector<torch::Tensor> attn_fwd2(torch::Tensor q, torch::Tensor k,
                                     torch::Tensor v, double scale,
                                     bool causal) {
  check_bf16_any(q, "q");
  check_bf16_any(k, "k");
  check_bf16_any(v, "v");
  const int sq = (int)q.size(0), b = (int)q.size(1), nh = (int)q.size(2),
            d = (int)q.size(3);
  const int sk = (int)k.size(0), ng = (int)k.size(2);
  auto o = torch::empty({sq, b, nh, d}, q.options());
  auto lse = torch::empty({b, nh, sq}, q.options().dtype(torch::kFloat32));
  long qs[3], ks[3], vs[3];
  TORCH_CHECK(attn_strides(q, qs) && attn_strides(k, ks) &&
              attn_strides(v, vs), "attn_fwd2: d must be contiguous");
  launch_attn_fwd2(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                   lse.data_ptr<float>(), sq, sk, b, nh, ng, d, (float)scale,
                   causal, qs, ks, vs, cur_stream());
  return {o, lse};
}

std::vector<torch::Tensor> attn_bwd(torch::Tensor dout, torch::Tensor q,
                                    torch::Tensor k, torch::Tensor v,
                                    torch::Tensor o, torch::Tensor lse,
                                    double scale, bool causal) {
  check_bf16_any(dout, "dout");
  check_bf16_any(q, "q");
  check_bf16_any(k, "k");
  check_bf16_any(v, "v");
  const int sq = (int)q.size(0), b = (int)q.size(1), nh = (int)q.size(2),
            d = (int)q.size(3);
  const int sk = (int)k.size(0), ng = (int)k.size(2);
  // q/k/v may be gapped views of the fused QKV GEMM output; the
  // gradients are plain contiguous [s, b, h, d] tensors
  auto dq = torch::empty({(long)sq, b, nh, d}, q.options());
  auto dk = torch::empty({(long)sk, b, ng, d}, q.options());
  auto dv = torch::empty({(long)sk, b, ng, d}, q.options());
  auto drow = torch::empty({(long)sq * b * nh},
                           q.options().dtype(torch::kFloat32));
  long qs[3], ks[3], vs[3];
  auto doc = dout.contiguous();
  if ((d == 128 || d == 64) && sq % 256 == 0 && sk % 256 == 0 &&
      attn_strides(q, qs) &&
      attn_strides(k, ks) && attn_strides(v, vs)) {
    const long dqs[3] = {(long)b * nh * d, (long)nh * d, (long)d};
    const long dks[3] = {(long)b * ng * d, (long)ng * d, (long)d};
    launch_attn_bwd2(doc.data_ptr(), q.data_ptr(), k.data_ptr(),
                     v.data_ptr(), o.data_ptr(), lse.data_ptr<float>(),
                     drow.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(),
                     dv.data_ptr(), sq, sk, b, nh, ng, d, (float)scale,
                     causal, qs, ks, vs, dqs, dks, dks, cur_stream());
  } else {
    auto qc = q.contiguous(), kc = k.contiguous(), vc = v.contiguous();
    launch_attn_bwd(doc.data_ptr(), qc.data_ptr(), kc.data_ptr(),
                    vc.data_ptr(), o.data_ptr(), lse.data_ptr<float>(),
                    drow.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(),
                    dv.data_ptr(), sq, sk, b, nh, ng, d, (float)scale,
                    causal, cur_stream());
  }
  return {dq, dk, dv};
}

// attn_bwd writing dQ/dK/dV INTO caller-provided (possibly strided)
// buffers — the flash backward can then fill the fused [s, b, g,
// (rep+2)*hn] QKV-grad buffer directly and _SplitQKV.backward skips its
// three slice copies (~1% of a GPT step).  Requires the round-2 kernel
// path; returns false when the shape would fall back to v1 (caller uses
// attn_bwd + copies instead).  Out tensors must have d contiguous.
bool attn_bwd_into(torch::Tensor dout, torch::Tensor q, torch::Tensor k,
                   torch::Tensor v, torch::Tensor o, torch::Tensor lse,
                   double scale, bool causal, torch::Tensor dq,
                   torch::Tensor dk, torch::Tensor dv) {
  check_bf16_any(dout, "dout");
  check_bf16_any(q, "q");
  check_bf16_any(k, "k");
  check_bf16_any(v, "v");
  check_bf16_any(dq, "dq");
  check_bf16_any(dk, "dk");
  check_bf16_any(dv, "dv");
  const int sq = (int)q.size(0), b = (int)q.size(1), nh = (int)q.size(2),
            d = (int)q.size(3);
  const int sk = (int)k.size(0), ng = (int)k.size(2);
  long qs[3], ks[3], vs[3], dqs[3], dks[3], dvs[3];
  if (!((d == 128 || d == 64) && sq % 256 == 0 && sk % 256 == 0 &&
        attn_strides(q, qs) && attn_strides(k, ks) && attn_strides(v, vs) &&
        attn_strides(dq, dqs) && attn_strides(dk, dks) &&
        attn_strides(dv, dvs)))
    return false;
  // dq is written with 16-byte vector stores: its strides and base
  // pointer must be 8-element aligned
  if (dqs[0] % 8 || dqs[1] % 8 || dqs[2] % 8 ||
      (reinterpret_cast<uintptr_t>(dq.data_ptr()) & 15))
    return false;
  TORCH_CHECK(dq.sizes() == q.sizes() && dk.sizes() == k.sizes() &&
              dv.sizes() == v.sizes(), "attn_bwd_into: out shape mismatch");
  auto drow = torch::empty({(long)sq * b * nh},
                           q.options().dtype(torch::kFloat32));
  auto doc = dout.contiguous();
  launch_attn_bwd2(doc.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                   o.data_ptr(), lse.data_ptr<float>(),
                   drow.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(),
                   dv.data_ptr(), sq, sk, b, nh, ng, d, (float)scale, causal,
                   qs, ks, vs, dqs, dks, dvs, cur_stream());
  return true;
}

// always-v1 backward, kept for A/B benchmarking
std::vector<torch::Tensor> attn_bwd_v1(torch::Tensor dout, torch::Tensor q,
                                       torch::Tensor k, torch::Tensor v,
                                       torch::Tensor o, torch::Tensor lse,
                                       double scale, bool causal) {
  const int sq = (int)q.size(0), b = (int)q.size(1), nh = (int)q.size(2),
            d = (int)q.size(3);
  const int sk = (int)k.size(0), ng = (int)k.size(2);
  auto dq = torch::empty_like(q);
  auto dk = torch::empty_like(k);
  auto dv = torch::empty_like(v);
  auto drow = torch::empty({(long)sq * b * nh},
                           q.options().dtype(torch::kFloat32));
  launch_attn_bwd(dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  o.data_ptr(), lse.data_ptr<float>(), drow.data_ptr<float>(),
                  dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), sq, sk, b, nh,
                  ng, d, (float)scale, causal, cur_stream());
  return {dq, dk, dv};
}

std::vector<torch::Tensor> attn_fwd_ablate(torch::Tensor q, torch::Tensor k,
                                           torch::Tensor v, double scale,
                                           long level) {
  const int sq = (int)q.size(0), b = (int)q.size(1), nh = (int)q.size(2),
            d = (int)q.size(3);
  const int sk = (int)k.size(0), ng = (int)k.size(2);
  auto o = torch::empty_like(q);
  auto lse = torch::empty({b, nh, sq}, q.options().dtype(torch::kFloat32));
  launch_attn_fwd_ablate(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                         o.data_ptr(), lse.data_ptr<float>(), sq, sk, b, nh,
                         ng, d, (float)scale, (int)level, cur_stream());
  return {o, lse};
}

// --------------------------------------------------------- packed attention
bool on_16_bytes(const torch::Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// A copy that begins on 16 bytes: contiguous() hands a contiguous tensor back,
// wherever it begins.
torch::Tensor laid_out(const torch::Tensor& t) {
  return t.clone(at::MemoryFormat::Contiguous);
}

// [t, b, h, d] (or [t, h, d], b = 1) in 16 bits; views are read as they are
// where each row of a head is adjacent and starts on 16 bytes, others are laid
// out first.  Arguments that cannot be are ValueErrors in Python.
torch::Tensor packed_rows(const torch::Tensor& t, long* strides) {
  const int h = (int)t.dim() - 2;
  bool fits = t.stride(h + 1) == 1 && on_16_bytes(t);
  for (int i = 0; i <= h; ++i)
    fits = fits && (t.size(i) <= 1 ||
                    (t.stride(i) % 8 == 0 && t.stride(i) < (1l << 27)));
  auto r = fits ? t : laid_out(t);
  // a single row's stride is never used
  strides[0] = r.size(0) <= 1 ? 0 : (long)r.stride(0);
  strides[1] = h == 1 || r.size(1) <= 1 ? 0 : (long)r.stride(1);
  strides[2] = r.size(h) <= 1 ? 0 : (long)r.stride(h);
  return r;
}

struct PackedShape {
  int tq, tk, b, nh, ng, d, n;
  bool fp16;
};

PackedShape packed_shape(const torch::Tensor& q, const torch::Tensor& k,
                         const torch::Tensor& v, const torch::Tensor& cu_q,
                         const torch::Tensor& cu_k,
                         const c10::optional<double>& softmax_scale,
                         double& scale) {
  const int dim = (int)q.dim(), h = dim - 2;
  TORCH_CHECK_VALUE((dim == 3 || dim == 4) && k.dim() == dim &&
                        k.sizes() == v.sizes(),
                    "packed_attention: query, key, value must be [t, heads, "
                    "hn] or [t, b, heads, hn], got ", q.sizes(), ", ",
                    k.sizes(), ", ", v.sizes());
  TORCH_CHECK_VALUE(k.size(h + 1) == q.size(h + 1) && k.size(h) > 0 &&
                        q.size(h) % k.size(h) == 0 &&
                        (dim == 3 || k.size(1) == q.size(1)),
                    "packed_attention: query ", q.sizes(), " and key ",
                    k.sizes(), " do not fit each other");
  TORCH_CHECK_VALUE(k.scalar_type() == q.scalar_type() &&
                        v.scalar_type() == q.scalar_type(),
                    "packed_attention: query, key and value must share one "
                    "floating type");
  TORCH_CHECK_VALUE(q.is_cuda() && k.device() == q.device() &&
                        v.device() == q.device(),
                    "packed_attention: query, key and value must be on one "
                    "device");
  for (auto* c : {&cu_q, &cu_k}) {
    TORCH_CHECK_VALUE(c->dim() == 1 && c->numel() > 0 &&
                          c->numel() == cu_q.numel() &&
                          (c->scalar_type() == torch::kInt32 ||
                           c->scalar_type() == torch::kInt64),
                      "packed_attention: cu_seqlens must be int32 or int64 "
                      "[sequences + 1], the same for both");
    TORCH_CHECK_VALUE(c->device() == q.device(),
                      "packed_attention: cu_seqlens must be on the query's "
                      "device");
  }
  scale = softmax_scale.has_value() ? *softmax_scale
                                    : 1.0 / std::sqrt((double)q.size(h + 1));
  TORCH_CHECK_VALUE((float)scale > 0 && std::isfinite((float)scale),
                    "packed_attention: softmax_scale must be positive and "
                    "finite");
  const bool fp16 = q.scalar_type() == torch::kHalf;
  TORCH_CHECK_VALUE((fp16 || q.scalar_type() == torch::kBFloat16) &&
                        (q.size(h + 1) == 64 || q.size(h + 1) == 128),
                    "packed_attention: on the GPU bf16 or fp16 with head size "
                    "64 or 128, got ", q.scalar_type(), ", ", q.size(h + 1));
  TORCH_CHECK_VALUE(q.size(0) < (1l << 30) && k.size(0) < (1l << 30),
                    "packed_attention: too many tokens");
  return {(int)q.size(0), (int)k.size(0), dim == 3 ? 1 : (int)q.size(1),
          (int)q.size(h), (int)k.size(h), (int)q.size(h + 1),
          (int)cu_q.numel() - 1, fp16};
}

// Whether forward mode wants a derivative along with the value.  A call that
// has none would else come back as a constant.
bool has_tangent(std::initializer_list<const torch::Tensor*> inputs) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return false;
  for (auto* t : inputs)
    if (t->_fw_grad(0).defined()) return true;
  return false;
}

// ends behind 32 bits stay behind the stream
torch::Tensor int32_row(const torch::Tensor& t) {
  return (t.scalar_type() == torch::kInt32
              ? t
              : t.clamp(INT32_MIN, INT32_MAX).to(torch::kInt32))
      .contiguous();
}

// the output, and where a backward will follow the rows' log-sums and what
// the output's rounding left out
std::vector<torch::Tensor> packed_attn_fwd(
    torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor cu_q,
    c10::optional<torch::Tensor> cu_kv, c10::optional<double> softmax_scale,
    bool causal, bool training) {
  const torch::Tensor cu_k = cu_kv.has_value() ? *cu_kv : cu_q;
  double scale;
  const PackedShape s = packed_shape(q, k, v, cu_q, cu_k, softmax_scale, scale);
  c10::DeviceGuard guard(q.device());
  auto o = torch::empty(q.sizes(), q.options());
  torch::Tensor lse, low;
  if (training) {
    lse = torch::empty({s.b, s.nh, s.tq}, q.options().dtype(torch::kFloat32));
    low = torch::empty(q.sizes(), q.options());
  }
  if (o.numel() == 0) return {o, lse, low};
  long qs[3], ks[3], vs[3];
  auto qr = packed_rows(q, qs), kr = packed_rows(k, ks),
       vr = packed_rows(v, vs);
  const torch::Tensor iq = int32_row(cu_q),
                      ik = cu_k.is_same(cu_q) ? iq : int32_row(cu_k);
  launch_packed_attn_fwd(qr.data_ptr(), kr.data_ptr(), vr.data_ptr(),
                         o.data_ptr(), training ? low.data_ptr() : nullptr,
                         training ? lse.data_ptr<float>() : nullptr,
                         iq.data_ptr<int>(), ik.data_ptr<int>(), s.n, s.tq,
                         s.tk, s.b, s.nh, s.ng, s.d, (float)scale, causal,
                         s.fp16, qs, ks, vs, cur_stream());
  return {o, lse, low};
}

std::vector<torch::Tensor> packed_attn_bwd(
    torch::Tensor dout, torch::Tensor q, torch::Tensor k, torch::Tensor v,
    torch::Tensor o, torch::Tensor low, torch::Tensor lse, torch::Tensor cu_q,
    c10::optional<torch::Tensor> cu_kv, c10::optional<double> softmax_scale,
    bool causal) {
  const torch::Tensor cu_k = cu_kv.has_value() ? *cu_kv : cu_q;
  double scale;
  const PackedShape s = packed_shape(q, k, v, cu_q, cu_k, softmax_scale, scale);
  c10::DeviceGuard guard(q.device());
  for (auto* t : {&o, &low})
    TORCH_CHECK_VALUE(t->sizes() == q.sizes() && t->is_contiguous() &&
                          t->scalar_type() == q.scalar_type() &&
                          t->device() == q.device(),
                      "packed_attention: o and low must be the forward's");
  TORCH_CHECK_VALUE(dout.sizes() == q.sizes() &&
                        dout.scalar_type() == q.scalar_type() &&
                        dout.device() == q.device() &&
                        lse.device() == q.device() &&
                        lse.numel() == (long)s.b * s.nh * s.tq &&
                        lse.is_contiguous() &&
                        lse.scalar_type() == torch::kFloat32,
                    "packed_attention: dout must be the output's gradient and "
                    "lse the forward's");
  auto dq = torch::empty(q.sizes(), q.options());
  auto dk = torch::empty(k.sizes(), q.options());
  auto dv = torch::empty(k.sizes(), q.options());
  if (s.b == 0 || s.nh == 0) return {dq, dk.zero_(), dv.zero_()};
  auto dot = torch::empty_like(lse);
  long os[3], qs[3], ks[3], vs[3];
  auto dr = packed_rows(dout, os), qr = packed_rows(q, qs),
       kr = packed_rows(k, ks), vr = packed_rows(v, vs);
  const torch::Tensor iq = int32_row(cu_q),
                      ik = cu_k.is_same(cu_q) ? iq : int32_row(cu_k);
  long floats = 0;
  const int shares = packed_attn_shares(s.n, s.tq, s.tk, s.b, s.nh, s.ng, s.d,
                                        &floats);
  torch::Tensor sums;
  if (floats) sums = torch::empty({floats}, q.options().dtype(torch::kFloat32));
  launch_packed_attn_bwd(
      dr.data_ptr(), qr.data_ptr(), kr.data_ptr(), vr.data_ptr(), o.data_ptr(),
      low.data_ptr(), lse.data_ptr<float>(), dot.data_ptr<float>(),
      dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
      floats ? sums.data_ptr<float>() : nullptr, shares, iq.data_ptr<int>(),
      ik.data_ptr<int>(), s.n, s.tq, s.tk, s.b, s.nh, s.ng, s.d, (float)scale,
      causal, s.fp16, os, qs, ks, vs, cur_stream());
  return {dq, dk, dv};
}

// A node of its own kind rather than Python's: a backward of small sequences
// takes the host 90 us there.
struct PackedAttn : public torch::autograd::Function<PackedAttn> {
  static torch::Tensor forward(torch::autograd::AutogradContext* ctx,
                               torch::Tensor q, torch::Tensor k,
                               torch::Tensor v, torch::Tensor cu_q,
                               c10::optional<torch::Tensor> cu_kv,
                               c10::optional<double> scale, bool causal) {
    const auto r = packed_attn_fwd(q, k, v, cu_q, cu_kv, scale, causal, true);
    ctx->save_for_backward({q, k, v, r[0], r[2], r[1], cu_q,
                            cu_kv.has_value() ? *cu_kv : torch::Tensor()});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["causal"] = causal;
    return r[0];
  }

  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx,
      torch::autograd::variable_list grads) {
    TORCH_CHECK(!torch::GradMode::is_enabled(),
                "packed_attention: its gradient has none of its own");
    const auto s = ctx->get_saved_variables();
    torch::autograd::variable_list out(7);
    if (!grads[0].defined()) return out;
    c10::optional<torch::Tensor> cu_kv;
    if (s[7].defined()) cu_kv = s[7];
    auto g = packed_attn_bwd(grads[0], s[0], s[1], s[2], s[3], s[4], s[5],
                             s[6], cu_kv,
                             ctx->saved_data["scale"].toOptional<double>(),
                             ctx->saved_data["causal"].toBool());
    for (int i = 0; i < 3; ++i) out[i] = g[i];
    return out;
  }
};

torch::Tensor packed_attention(torch::Tensor q, torch::Tensor k,
                               torch::Tensor v, torch::Tensor cu_q,
                               c10::optional<torch::Tensor> cu_kv,
                               c10::optional<double> scale, bool causal) {
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent({&q, &k, &v}),
                              "packed_attention: on the GPU no forward-mode "
                              "derivative");
  if (torch::GradMode::is_enabled() &&
      (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return PackedAttn::apply(q, k, v, cu_q, cu_kv, scale, causal);
  return packed_attn_fwd(q, k, v, cu_q, cu_kv, scale, causal, false)[0];
}

// ------------------------------------------------------------- paged cache
// pages [layers, 2, P, groups, page, d]; refs [P], tables [slots, W], lengths
// [slots] and status [1] int32, all on one GPU and contiguous

// of a sequence: the kernels add the keys of a step, and of a piece's rounded
// share for each of 64 pieces, to a place before they compare it with the end
constexpr long MOST_TOKENS = (1l << 31) - 8192;

struct CacheRefs {
  int *refs, *tables, *lengths, *status;
  int pages, slots, width, page, planes, groups, token;
  void* data;
};

void check_ints(const torch::Tensor& t, const torch::Tensor& like, int dim,
                const char* name) {
  TORCH_CHECK(t.device() == like.device() && t.dim() == dim &&
                  t.scalar_type() == torch::kInt32 && t.is_contiguous(),
              name, " must be a contiguous int32 tensor on the cache's GPU");
}

CacheRefs cache_refs(const torch::Tensor& pages, const torch::Tensor& refs,
                     const torch::Tensor& tables, const torch::Tensor& lengths,
                     const torch::Tensor& status) {
  TORCH_CHECK(pages.is_cuda() && pages.dim() == 6 && pages.size(1) == 2 &&
                  pages.is_contiguous() && on_16_bytes(pages),
              "pages must be [layers, 2, P, groups, page, d], contiguous, on "
              "the GPU");
  check_ints(refs, pages, 1, "ref_counts");
  check_ints(tables, pages, 2, "page_tables");
  check_ints(lengths, pages, 1, "lengths");
  check_ints(status, pages, 1, "status");
  const long token = pages.size(5) * pages.element_size();
  TORCH_CHECK(refs.numel() == pages.size(2) &&
                  lengths.numel() == tables.size(0) && status.numel() > 0 &&
                  token % 16 == 0 && pages.size(2) < (1l << 30) &&
                  tables.size(0) <= (1l << 18) &&
                  tables.size(1) * (long)pages.size(4) <= MOST_TOKENS,
              "the cache's tensors do not fit each other");
  return {refs.data_ptr<int>(),    tables.data_ptr<int>(),
          lengths.data_ptr<int>(), status.data_ptr<int>(),
          (int)pages.size(2),      (int)tables.size(0),
          (int)tables.size(1),     (int)pages.size(4),
          (int)pages.size(0) * 2,  (int)pages.size(3),
          (int)token,              pages.data_ptr()};
}

#define CACHE_ARGS                                                       \
  torch::Tensor pages, torch::Tensor refs, torch::Tensor tables,         \
      torch::Tensor lengths, torch::Tensor status
#define CACHE_TABLES c.refs, c.tables, c.lengths, c.status, c.pages, \
                     c.slots, c.width, c.page

void cache_fork(CACHE_ARGS, torch::Tensor src, torch::Tensor dst) {
  const CacheRefs c = cache_refs(pages, refs, tables, lengths, status);
  c10::DeviceGuard guard(pages.device());
  check_ints(src, pages, 1, "src");
  check_ints(dst, pages, 1, "dst");
  const int n = (int)src.numel();
  TORCH_CHECK(dst.numel() == n && n <= c.slots, "fork: src and dst must name "
              "as many slots, at most all");
  if (n == 0) return;
  auto scratch = torch::empty({4 + 5l * n + (long)n * c.width}, refs.options());
  launch_cache_fork(CACHE_TABLES, c.data, c.planes, c.groups, c.token,
                    src.data_ptr<int>(), dst.data_ptr<int>(), n,
                    scratch.data_ptr<int>(), cur_stream());
}

void cache_free(CACHE_ARGS, torch::Tensor list) {
  const CacheRefs c = cache_refs(pages, refs, tables, lengths, status);
  c10::DeviceGuard guard(pages.device());
  check_ints(list, pages, 1, "slots");
  if (list.numel() == 0) return;
  launch_cache_free(CACHE_TABLES, list.data_ptr<int>(), (int)list.numel(),
                    cur_stream());
}

void cache_compact(CACHE_ARGS) {
  const CacheRefs c = cache_refs(pages, refs, tables, lengths, status);
  c10::DeviceGuard guard(pages.device());
  if (c.pages == 0) return;
  auto scratch = torch::empty({2 + 4l * c.pages}, refs.options());
  launch_cache_compact(CACHE_TABLES, c.data, c.planes,
                       (long)c.groups * c.page * c.token,
                       scratch.data_ptr<int>(), cur_stream());
}

void cache_copy(CACHE_ARGS, torch::Tensor src, torch::Tensor dst) {
  const CacheRefs c = cache_refs(pages, refs, tables, lengths, status);
  c10::DeviceGuard guard(pages.device());
  check_ints(src, pages, 1, "src");
  check_ints(dst, pages, 1, "dst");
  TORCH_CHECK(dst.numel() == src.numel(),
              "copy_pages: src and dst must name as many pages");
  if (src.numel() == 0) return;
  launch_cache_copy(src.data_ptr<int>(), dst.data_ptr<int>(),
                    (int)src.numel(), c.data, c.planes, c.pages,
                    (long)c.groups * c.page * c.token, c.status, cur_stream());
}

void cache_extend(CACHE_ARGS, torch::Tensor list,
                  c10::optional<torch::Tensor> counts, long each) {
  const CacheRefs c = cache_refs(pages, refs, tables, lengths, status);
  c10::DeviceGuard guard(pages.device());
  check_ints(list, pages, 1, "slots");
  const int n = (int)list.numel();
  TORCH_CHECK(n <= c.slots && each >= 0 && each < (1l << 30),
              "extend: at most all slots, and a number of tokens");
  if (counts.has_value()) {
    check_ints(*counts, pages, 1, "num_tokens");
    TORCH_CHECK(counts->numel() == n, "extend: a count for each slot");
  }
  if (n == 0) return;
  auto scratch = torch::empty({(long)n + c.pages}, refs.options());
  launch_cache_extend(CACHE_TABLES, list.data_ptr<int>(),
                      counts.has_value() ? counts->data_ptr<int>() : nullptr,
                      (int)each, n, scratch.data_ptr<int>(), cur_stream());
}

void cache_write(CACHE_ARGS, long layer, torch::Tensor k, torch::Tensor v,
                 torch::Tensor list, c10::optional<torch::Tensor> cu) {
  const CacheRefs c = cache_refs(pages, refs, tables, lengths, status);
  c10::DeviceGuard guard(pages.device());
  check_ints(list, pages, 1, "slots");
  TORCH_CHECK(layer >= 0 && layer < pages.size(0), "write: no such layer");
  TORCH_CHECK(k.device() == pages.device() && v.device() == pages.device() &&
                  k.scalar_type() == pages.scalar_type() &&
                  v.scalar_type() == pages.scalar_type() && k.dim() == 3 &&
                  k.sizes() == v.sizes() && k.size(1) == c.groups &&
                  k.size(2) == pages.size(5),
              "write: key and value must be [tokens, groups, d] of the "
              "cache's type, on its GPU");
  const int n = (int)list.numel();
  if (cu.has_value()) {
    check_ints(*cu, pages, 1, "cu_seqlens");
    TORCH_CHECK(cu->numel() == n + 1, "write: cu_seqlens must be [slots + 1]");
  } else {
    TORCH_CHECK(k.size(0) == n, "write: one token for each slot");
  }
  TORCH_CHECK(k.size(0) * (long)c.groups < (1l << 31),
              "write: too many tokens");
  if (k.size(0) == 0 || c.groups == 0) return;
  const long es = pages.element_size();
  auto rows = [&](const torch::Tensor& t) {
    const bool fits = t.stride(2) == 1 && t.stride(0) * es % 16 == 0 &&
                      t.stride(1) * es % 16 == 0 && on_16_bytes(t);
    return fits ? t : laid_out(t);
  };
  auto kr = rows(k), vr = rows(v);
  const long plane = (long)c.pages * c.groups * c.page * c.token;
  char* keys = (char*)c.data + 2 * layer * plane;
  launch_cache_write(CACHE_TABLES, list.data_ptr<int>(),
                     cu.has_value() ? cu->data_ptr<int>() : nullptr, n,
                     (int)k.size(0), keys, keys + plane, kr.data_ptr(),
                     vr.data_ptr(), c.groups, c.token, kr.stride(0) * es,
                     kr.stride(1) * es, vr.stride(0) * es, vr.stride(1) * es,
                     cur_stream());
}

// ---------------------------------------------------------- paged attention
torch::Tensor paged_ints(const torch::Tensor& t, const torch::Tensor& q,
                         int dim, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == dim && t.scalar_type() == torch::kInt32,
                    "paged_attention: ", name, " must be an int32 tensor of ",
                    dim, " dimension(s)");
  TORCH_CHECK_VALUE(t.device() == q.device(),
                    "paged_attention: all tensors must be on the query's "
                    "device");
  return t.contiguous();
}

torch::Tensor paged_attn(torch::Tensor q, torch::Tensor k, torch::Tensor v,
                         torch::Tensor page_tables, torch::Tensor row_lengths,
                         c10::optional<torch::Tensor> row_slots,
                         c10::optional<long> max_length,
                         c10::optional<torch::Tensor> prefix_rows,
                         c10::optional<torch::Tensor> prefix_lengths,
                         long max_rows, long max_prefix,
                         c10::optional<double> softmax_scale) {
  TORCH_CHECK_VALUE(q.dim() == 3 && k.dim() == 4 && v.sizes() == k.sizes(),
                    "paged_attention: query must be [b, heads, d], key and "
                    "value pages [P, groups, page, d]");
  TORCH_CHECK_VALUE(!has_tangent({&q, &k, &v}),
                    "paged_attention: has no gradient, in forward mode "
                    "neither");
  const int b = (int)q.size(0), nh = (int)q.size(1), d = (int)q.size(2);
  const int ng = (int)k.size(1), page = (int)k.size(2);
  TORCH_CHECK_VALUE(k.size(3) == d && ng > 0 && nh % ng == 0 &&
                        k.size(0) > 0 && k.size(0) < (1l << 30),
                    "paged_attention: query ", q.sizes(), " and pages ",
                    k.sizes(), " do not fit each other");
  TORCH_CHECK_VALUE(page >= 16 && page % 16 == 0,
                    "paged_attention: pages must hold a multiple of 16 "
                    "tokens");
  TORCH_CHECK_VALUE(k.scalar_type() == q.scalar_type() &&
                        v.scalar_type() == q.scalar_type(),
                    "paged_attention: query and pages must share one floating "
                    "type");
  TORCH_CHECK_VALUE(q.is_cuda() && k.device() == q.device() &&
                        v.device() == q.device(),
                    "paged_attention: all tensors must be on the query's "
                    "device");
  const bool fp16 = q.scalar_type() == torch::kHalf;
  TORCH_CHECK_VALUE((fp16 || q.scalar_type() == torch::kBFloat16) &&
                        (d == 64 || d == 128),
                    "paged_attention: on the GPU bf16 or fp16 with head size "
                    "64 or 128, got ", q.scalar_type(), ", ", d);
  for (auto* t : {&k, &v})
    TORCH_CHECK_VALUE(t->stride(3) == 1 &&
                          (t->size(0) == 1 || t->stride(0) % 8 == 0) &&
                          (t->size(1) == 1 || t->stride(1) % 8 == 0) &&
                          t->stride(2) % 8 == 0 &&
                          t->stride(2) < (1l << 27) && on_16_bytes(*t),
                      "paged_attention: the rows of a page must start on 16 "
                      "bytes");
  const auto tables = paged_ints(page_tables, q, 2, "page_tables");
  const auto lengths = paged_ints(row_lengths, q, 1, "lengths");
  const int count = (int)tables.size(0);
  torch::Tensor slots, group_rows, group_lengths;
  if (row_slots.has_value()) slots = paged_ints(*row_slots, q, 1, "slots");
  TORCH_CHECK_VALUE(lengths.numel() == count && count > 0 &&
                        tables.size(1) > 0 &&
                        (slots.defined() ? slots.numel() : count) == b,
                    "paged_attention: one length for each table, one table or "
                    "slot for each row");
  TORCH_CHECK_VALUE(tables.size(1) * (long)page <= MOST_TOKENS,
                    "paged_attention: tables of 2^31 tokens, or 8191 fewer, "
                    "are too long");
  const double scale = softmax_scale.has_value() ? *softmax_scale
                                                 : 1.0 / std::sqrt((double)d);
  TORCH_CHECK_VALUE((float)scale > 0 && std::isfinite((float)scale),
                    "paged_attention: softmax_scale must be positive and "
                    "finite");
  int groups = 0, own, shared, evenly, extra;
  if (prefix_rows.has_value()) {
    group_rows = paged_ints(*prefix_rows, q, 1, "shared_prefix.rows");
    group_lengths = paged_ints(*prefix_lengths, q, 1, "shared_prefix.lengths");
    groups = (int)group_lengths.numel();
    TORCH_CHECK_VALUE(group_rows.numel() == groups + 1,
                      "paged_attention: shared_prefix.rows must be one longer "
                      "than its lengths");
  }
  c10::DeviceGuard guard(q.device());
  auto o = torch::empty({b, nh, d}, q.options());
  if (o.numel() == 0) return o;
  const bool fits = q.stride(2) == 1 && q.stride(0) % 8 == 0 &&
                    q.stride(1) % 8 == 0 && on_16_bytes(q);
  auto qr = fits ? q : laid_out(q);
  const long room = tables.size(1) * (long)page;
  const long longest = max_length.has_value() ? *max_length : room;
  max_rows = std::max(1l, std::min(max_rows, (long)b));
  paged_attn_pieces(b, nh, ng, d,
                    (int)std::max(std::min(longest, room), 1l),
                    groups, (int)max_rows,
                    std::min(std::max(max_prefix, 0l), 1l << 30), &own,
                    &shared, &evenly, &extra);
  const int pieces = own + shared;
  torch::Tensor part;
  if (pieces > 1)
    part = torch::empty({(long)b * nh * pieces * (d + 1)},
                        q.options().dtype(torch::kFloat32));
  float* po = pieces > 1 ? part.data_ptr<float>() : nullptr;
  const long ks[3] = {k.stride(0), k.stride(1), k.stride(2)};
  const long vs[3] = {v.stride(0), v.stride(1), v.stride(2)};
  launch_paged_attn(qr.data_ptr(), qr.stride(0), qr.stride(1), k.data_ptr(),
                    v.data_ptr(), ks, vs, tables.data_ptr<int>(),
                    lengths.data_ptr<int>(),
                    slots.defined() ? slots.data_ptr<int>() : nullptr,
                    groups ? group_rows.data_ptr<int>() : nullptr,
                    groups ? group_lengths.data_ptr<int>() : nullptr, groups,
                    (int)max_rows, b, nh, ng, d, (int)k.size(0), page,
                    (int)tables.size(1), count, own, shared, evenly, extra,
                    o.data_ptr(), po,
                    po ? po + (long)b * nh * pieces * d : nullptr,
                    (float)scale, fp16, cur_stream());
  return o;
}

// --------------------------------------------------------------------- adam
// states fp32 OR bf16 (precision-aware optimizer); params/grads fp32
static bool adam_states_bf16(const torch::Tensor& m, const torch::Tensor& v) {
  TORCH_CHECK(m.scalar_type() == v.scalar_type(),
              "adam m/v dtypes must match");
  TORCH_CHECK(m.scalar_type() == torch::kFloat32 ||
              m.scalar_type() == torch::kBFloat16,
              "adam states must be fp32 or bf16");
  return m.scalar_type() == torch::kBFloat16;
}

static void* adam_p16_ptr(const c10::optional<torch::Tensor>& p16,
                          const torch::Tensor& p) {
  if (!p16.has_value()) return nullptr;
  TORCH_CHECK(p16->scalar_type() == torch::kBFloat16 &&
              p16->is_contiguous() && p16->numel() == p.numel(),
              "adam p16 must be a contiguous bf16 mirror of the shard");
  return p16->data_ptr();
}

void adamw_flat(torch::Tensor p, torch::Tensor g, torch::Tensor m,
                torch::Tensor v, double lr, double beta1, double beta2,
                double eps, double wd, long step,
                c10::optional<torch::Tensor> p16) {
  TORCH_CHECK(p.is_cuda() && p.scalar_type() == torch::kFloat32);
  launch_adamw_flat(p.data_ptr<float>(), g.data_ptr<float>(), m.data_ptr(),
                    v.data_ptr(), adam_states_bf16(m, v),
                    adam_p16_ptr(p16, p), p.numel(),
                    (float)lr, (float)beta1, (float)beta2, (float)eps,
                    (float)wd, (int)step, cur_stream());
}

torch::Tensor selective_scan_fwd(torch::Tensor x, torch::Tensor dt,
                                 torch::Tensor A, torch::Tensor B,
                                 torch::Tensor C, torch::Tensor D,
                                 torch::Tensor h) {
  check_bf16(x, "x");
  check_bf16(dt, "dt");
  check_bf16(B, "B");
  check_bf16(C, "C");
  TORCH_CHECK(A.dtype() == torch::kFloat32 && D.dtype() == torch::kFloat32 &&
              h.dtype() == torch::kFloat32);
  TORCH_CHECK(x.is_contiguous() && dt.is_contiguous() && B.is_contiguous() &&
              C.is_contiguous() && h.is_contiguous());
  const int b = (int)x.size(0), l = (int)x.size(1), d = (int)x.size(2);
  const int n = (int)A.size(1);
  auto y = torch::empty_like(x);
  launch_selective_scan_fwd(x.data_ptr(), dt.data_ptr(),
                            A.data_ptr<float>(), B.data_ptr(), C.data_ptr(),
                            D.data_ptr<float>(), h.data_ptr<float>(),
                            y.data_ptr(), b, l, d, n,
                            at::cuda::getCurrentCUDAStream());
  return y;
}

torch::Tensor ce_rowmax(torch::Tensor logits) {
  check_bf16(logits, "logits");
  TORCH_CHECK(logits.is_contiguous() && logits.dim() == 2);
  const long rows = logits.size(0);
  const int v = (int)logits.size(1);
  TORCH_CHECK(v % 8 == 0);
  auto out = torch::empty({rows}, logits.options().dtype(torch::kFloat32));
  launch_ce_rowmax(logits.data_ptr(), out.data_ptr<float>(), rows, v,
                   cur_stream());
  return out;
}

std::vector<torch::Tensor> ce_fwd(torch::Tensor logits, torch::Tensor rowmax,
                                  torch::Tensor target) {
  check_bf16(logits, "logits");
  TORCH_CHECK(target.dtype() == torch::kInt32 && target.is_contiguous());
  const long rows = logits.size(0);
  const int v = (int)logits.size(1);
  auto sumexp = torch::empty({rows},
                             logits.options().dtype(torch::kFloat32));
  auto predicted = torch::zeros({rows},
                                logits.options().dtype(torch::kFloat32));
  launch_ce_fwd(logits.data_ptr(), rowmax.data_ptr<float>(),
                target.data_ptr<int>(), sumexp.data_ptr<float>(),
                predicted.data_ptr<float>(), rows, v, cur_stream());
  return {sumexp, predicted};
}

torch::Tensor ce_bwd(torch::Tensor logits, torch::Tensor rowmax,
                     torch::Tensor sumexp, torch::Tensor target,
                     torch::Tensor grad_row) {
  check_bf16(logits, "logits");
  const long rows = logits.size(0);
  const int v = (int)logits.size(1);
  auto dlogits = torch::empty_like(logits);
  launch_ce_bwd(logits.data_ptr(), rowmax.data_ptr<float>(),
                sumexp.data_ptr<float>(), target.data_ptr<int>(),
                grad_row.contiguous().data_ptr<float>(), dlogits.data_ptr(),
                rows, v, cur_stream());
  return dlogits;
}

void adamw_flat_ranged(torch::Tensor p, torch::Tensor g, torch::Tensor m,
                       torch::Tensor v, torch::Tensor nw_s, torch::Tensor nw_e,
                       double lr, double beta1, double beta2, double eps,
                       double wd, long step,
                       c10::optional<torch::Tensor> p16) {
  TORCH_CHECK(p.is_cuda() && p.dtype() == torch::kFloat32);
  TORCH_CHECK(nw_s.is_cuda() && nw_s.dtype() == torch::kInt64 &&
              nw_s.is_contiguous());
  TORCH_CHECK(nw_e.sizes() == nw_s.sizes());
  launch_adamw_flat_ranged(
      p.data_ptr<float>(), g.data_ptr<float>(), m.data_ptr(), v.data_ptr(),
      adam_states_bf16(m, v), adam_p16_ptr(p16, p), nw_s.data_ptr<long>(),
      nw_e.data_ptr<long>(),
      (int)nw_s.numel(), p.numel(), (float)lr, (float)beta1, (float)beta2,
      (float)eps, (float)wd, (int)step,
      at::cuda::getCurrentCUDAStream());
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, mod) {
  mod.def("rmsnorm_fwd", &rmsnorm_fwd);
  mod.def("rmsnorm_bwd", &rmsnorm_bwd, pybind11::arg("dy"), pybind11::arg("x"),
          pybind11::arg("w"), pybind11::arg("invrms"),
          pybind11::arg("main_grad_w") = pybind11::none(),
          pybind11::arg("dres") = pybind11::none());
  mod.def("layernorm_fwd", &layernorm_fwd);
  mod.def("layernorm_bwd", &layernorm_bwd, pybind11::arg("dy"),
          pybind11::arg("x"), pybind11::arg("w"), pybind11::arg("mean"),
          pybind11::arg("invstd"),
          pybind11::arg("main_grad_w") = pybind11::none(),
          pybind11::arg("main_grad_b") = pybind11::none(),
          pybind11::arg("dres") = pybind11::none());
  mod.def("bias_gelu_fwd", &bias_gelu_fwd);
  mod.def("bias_gelu_bwd", &bias_gelu_bwd);
  mod.def("bias_swiglu_fwd", &bias_swiglu_fwd);
  mod.def("bias_swiglu_bwd", &bias_swiglu_bwd);
  mod.def("bias_geglu_fwd", &bias_geglu_fwd);
  mod.def("bias_geglu_bwd", &bias_geglu_bwd);
  mod.def("rope_fwd", &rope_fwd);
  mod.def("rope_bwd", &rope_bwd);
  mod.def("scaled_upper_triang_masked_softmax_fwd",
          &scaled_upper_triang_masked_softmax_fwd);
  mod.def("scaled_softmax_fwd", &scaled_softmax_fwd);
  mod.def("scaled_masked_softmax_fwd", &scaled_masked_softmax_fwd);
  mod.def("scaled_softmax_bwd", &scaled_softmax_bwd);
  mod.def("adamw_flat", &adamw_flat, pybind11::arg("p"),
          pybind11::arg("g"), pybind11::arg("m"), pybind11::arg("v"),
          pybind11::arg("lr"), pybind11::arg("beta1"),
          pybind11::arg("beta2"), pybind11::arg("eps"),
          pybind11::arg("wd"), pybind11::arg("step"),
          pybind11::arg("p16") = pybind11::none());
  mod.def("selective_scan_fwd", &selective_scan_fwd);
  mod.def("attn_fwd_t", &attn_fwd_t);
  mod.def("attn_fwd2", &attn_fwd2);
  mod.def("quantize_rows_e4m3", &quantize_rows_e4m3);
  mod.def("quantize_transpose_e4m3", &quantize_transpose_e4m3);
  mod.def("bias_dropout_add_fwd", &bias_dropout_add_fwd);
  mod.def("dropout_bwd", &dropout_bwd);
  mod.def("moe_combine_fwd", &moe_combine_fwd);
  mod.def("moe_combine_bwd", &moe_combine_bwd);
  mod.def("attn_bwd_v1", &attn_bwd_v1);
  mod.def("attn_bwd_into", &attn_bwd_into);
  mod.def("ce_rowmax", &ce_rowmax);
  mod.def("gemm_nt", &gemm_nt);
  mod.def("gemm_nn", &gemm_nn);
  mod.def("ce_fwd", &ce_fwd);
  mod.def("ce_bwd", &ce_bwd);
  mod.def("scaled_upper_triang_masked_softmax_bwd",
          &scaled_upper_triang_masked_softmax_bwd);
  mod.def("bias_add_residual", &bias_add_residual);
  mod.def("adamw_flat_ranged", &adamw_flat_ranged, pybind11::arg("p"),
          pybind11::arg("g"), pybind11::arg("m"), pybind11::arg("v"),
          pybind11::arg("nw_s"), pybind11::arg("nw_e"),
          pybind11::arg("lr"), pybind11::arg("beta1"),
          pybind11::arg("beta2"), pybind11::arg("eps"),
          pybind11::arg("wd"), pybind11::arg("step"),
          pybind11::arg("p16") = pybind11::none());
  mod.def("wgrad_accum", &wgrad_accum);
  mod.def("wgrad_accum_bgrad", &wgrad_accum_bgrad);
  mod.def("attn_fwd", &attn_fwd);
  mod.def("attn_fwd_ablate", &attn_fwd_ablate);
  mod.def("packed_attention", &packed_attention);
  // how a tile's work for dK and dV is cut: (shares, floats for their sums)
  mod.def("packed_attn_shares", [](int n, int tq, int tk, int b, int nh,
                                   int ng, int d) {
    long floats = 0;
    const int shares = packed_attn_shares(n, tq, tk, b, nh, ng, d, &floats);
    return std::make_tuple(shares, floats);
  });
  mod.def("cache_fork", &cache_fork);
  mod.def("cache_free", &cache_free);
  mod.def("cache_compact", &cache_compact);
  mod.def("cache_copy", &cache_copy);
  mod.def("cache_extend", &cache_extend);
  mod.def("cache_write", &cache_write);
  mod.def("paged_attn", &paged_attn);
  // how the work is cut: (pieces of a row at most, of a group's beginning, of
  // a row in general, blocks for those beyond that)
  mod.def("paged_attn_pieces", [](int b, int nh, int ng, int d, int max_length,
                                  int groups, int max_rows, long max_prefix) {
    int own, shared, evenly, extra;
    paged_attn_pieces(b, nh, ng, d, max_length, groups, max_rows, max_prefix,
                      &own, &shared, &evenly, &extra);
    return std::make_tuple(own, shared, evenly, extra);
  });
  mod.def("attn_bwd", &attn_bwd);
  mod.def("colsum_accum", &colsum_accum);
  mod.def("embedding_bwd_accum", &embedding_bwd_accum);
}
