// Torch-facing wrappers and Python bindings of the sm_100a kernels (module resihp._C).
// Shapes, dtypes and strides are checked here; the CUDA launchers behind launch.h only
// see raw pointers, so the kernel translation units stay free of torch headers.
// (The reference is pure Python and calls torch / NCCL ops directly; this layer has no
// counterpart there.)
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <atomic>
#include <unordered_set>
#include <mutex>
#include <csignal>
#include <execinfo.h>
#include <unistd.h>

#include "launch.h"

namespace resihp {

// ---- error word ---------------------------------------------------------------------

static int* g_error_words[64] = {nullptr};
static std::mutex g_error_mutex;

int* error_word(const c10::Device& device) {
  const int idx = device.index() < 0 ? 0 : device.index();
  TORCH_CHECK(idx < 64, "device index out of range");
  if (g_error_words[idx] == nullptr) {
    std::lock_guard<std::mutex> lock(g_error_mutex);
    if (g_error_words[idx] == nullptr) {
      c10::cuda::CUDAGuard guard(device);
      int* p = nullptr;
      C10_CUDA_CHECK(cudaMalloc(&p, sizeof(int)));
      C10_CUDA_CHECK(cudaMemset(p, 0, sizeof(int)));
      g_error_words[idx] = p;
    }
  }
  return g_error_words[idx];
}

// Synchronising read of the device's error word; resets it to zero.
int64_t read_and_clear_error(int64_t device_index) {
  const c10::Device dev(c10::kCUDA, device_index);
  int* p = error_word(dev);
  c10::cuda::CUDAGuard guard(dev);
  auto stream = at::cuda::getCurrentCUDAStream();
  int value = 0;
  C10_CUDA_CHECK(cudaMemcpyAsync(&value, p, sizeof(int), cudaMemcpyDeviceToHost, stream));
  C10_CUDA_CHECK(cudaStreamSynchronize(stream));
  if (value != 0) C10_CUDA_CHECK(cudaMemsetAsync(p, 0, sizeof(int), stream));
  return value;
}

// A message with numbers in it. TORCH_CHECK would format them through a stream, which ends the
// process here instead of raising (the interpreter and libtorch bring C++ libraries whose stream
// locales do not fit); std::to_string is safe.
template <class... Parts>
static std::string message(const Parts&... parts) {
  std::string text;
  detail::append(text, parts...);
  return text;
}

static cudaStream_t cur_stream() { return at::cuda::getCurrentCUDAStream(); }

static void check_cuda_bf16(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, name, " must be bf16");
}

// ---- GEMM ---------------------------------------------------------------------------

void gemm(torch::Tensor a, bool a_mn, torch::Tensor b, bool b_mn, torch::Tensor c, int64_t epi, double alpha,
          c10::optional<torch::Tensor> residual, int64_t max_ctas, int64_t force_bn) {
  check_cuda_bf16(a, "A");
  check_cuda_bf16(b, "B");
  TORCH_CHECK(c.is_cuda(), "C must be a CUDA tensor");
  TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && c.dim() == 2, "GEMM operands must be 2-D");
  TORCH_CHECK(a.stride(1) == 1 && b.stride(1) == 1 && c.stride(1) == 1, "GEMM operands need unit inner stride");
  const int64_t m = a_mn ? a.size(1) : a.size(0);
  const int64_t k = a_mn ? a.size(0) : a.size(1);
  const int64_t n = b_mn ? b.size(1) : b.size(0);
  const int64_t kb = b_mn ? b.size(0) : b.size(1);
  TORCH_CHECK(k == kb, message("GEMM reduction sizes differ: ", k, " vs ", kb));
  TORCH_CHECK(c.size(0) == m && c.size(1) == n, "GEMM output shape mismatch");
  TORCH_CHECK(epi >= 0 && epi <= 4, message("unknown GEMM epilogue ", epi));
  const bool want_f32 = epi == 1 || epi == 2 || epi == 4;
  TORCH_CHECK(c.scalar_type() == (want_f32 ? at::kFloat : at::kBFloat16), "GEMM output dtype does not match epilogue");
  const void* r = nullptr;
  int64_t ldr = 0;
  if (epi == 3) {
    TORCH_CHECK(residual.has_value(), "residual epilogue needs a residual tensor");
    const auto& rt = *residual;
    check_cuda_bf16(rt, "residual");
    TORCH_CHECK(rt.size(0) == m && rt.size(1) == n && rt.stride(1) == 1, "residual must be [m, n]");
    TORCH_CHECK(reinterpret_cast<uintptr_t>(rt.data_ptr()) % 16 == 0 && rt.stride(0) % 8 == 0, "residual alignment");
    r = rt.data_ptr();
    ldr = rt.stride(0);
  }
  TORCH_CHECK(m <= INT32_MAX && n <= INT32_MAX && k <= INT32_MAX, "GEMM too large");
  c10::cuda::CUDAGuard guard(a.device());
  gemm_raw(a.data_ptr(), a.stride(0), a_mn, b.data_ptr(), b.stride(0), b_mn, c.data_ptr(), c.stride(0), r, ldr,
           int(m), int(n), int(k), int(epi), float(alpha), error_word(a.device()), cur_stream(), int(max_ctas),
           int(force_bn));
}


static int sms(const torch::Tensor& t) {
  static int counts[64] = {0};
  const int dev = t.device().index();
  if (counts[dev] == 0) C10_CUDA_CHECK(cudaDeviceGetAttribute(&counts[dev], cudaDevAttrMultiProcessorCount, dev));
  return counts[dev];
}

static void check_rows(const torch::Tensor& t, int64_t cols, const char* name) {
  check_cuda_bf16(t, name);
  TORCH_CHECK(t.dim() == 2 && t.size(1) == cols && t.is_contiguous(),
              message(name, " must be contiguous [rows, ", cols, "]"));
}

// ---- RMSNorm --------------------------------------------------------------------------

std::vector<torch::Tensor> rmsnorm_fwd_t(torch::Tensor x, c10::optional<torch::Tensor> r, torch::Tensor w, double eps) {
  const int64_t d = w.numel();
  check_rows(x, d, "x");
  check_cuda_bf16(w, "w");
  c10::cuda::CUDAGuard guard(x.device());
  auto y = torch::empty_like(x);
  auto rstd = torch::empty({x.size(0)}, x.options().dtype(torch::kFloat));
  torch::Tensor s = x;
  const void* rp = nullptr;
  if (r.has_value()) {
    check_rows(*r, d, "residual");
    s = torch::empty_like(x);
    rp = r->data_ptr();
  }
  rmsnorm_fwd(x.data_ptr(), rp, w.data_ptr(), y.data_ptr(), rp ? s.data_ptr() : nullptr, rstd.data_ptr<float>(),
              int(x.size(0)), int(d), float(eps), sms(x), cur_stream());
  return {y, s, rstd};
}

torch::Tensor rmsnorm_bwd_t(torch::Tensor dy, torch::Tensor s, torch::Tensor w, torch::Tensor rstd,
                            c10::optional<torch::Tensor> dres, torch::Tensor dw, bool accumulate) {
  const int64_t d = w.numel();
  check_rows(dy, d, "dy");
  check_rows(s, d, "s");
  TORCH_CHECK(dw.scalar_type() == torch::kFloat && dw.numel() == d && dw.is_contiguous(), "dw must be fp32 [d]");
  c10::cuda::CUDAGuard guard(dy.device());
  const int rows = int(dy.size(0));
  auto partial = torch::empty({rmsnorm_partial_rows(rows, int(d), sms(dy)), d}, dy.options().dtype(torch::kFloat));
  auto ds = torch::empty_like(dy);
  const void* dr = nullptr;
  if (dres.has_value()) {
    check_rows(*dres, d, "dres");
    dr = dres->data_ptr();
  }
  rmsnorm_bwd(dy.data_ptr(), s.data_ptr(), w.data_ptr(), rstd.data_ptr<float>(), dr, ds.data_ptr(),
              partial.data_ptr<float>(), dw.data_ptr<float>(), accumulate ? 1 : 0, rows, int(d), sms(dy), cur_stream());
  return ds;
}

// ---- RoPE / SwiGLU --------------------------------------------------------------------

void rope_t(torch::Tensor qkv, torch::Tensor cs, int64_t seq, int64_t heads_qk, int64_t hd, int64_t pos_offset,
            bool inverse) {
  check_cuda_bf16(qkv, "qkv");
  TORCH_CHECK(qkv.dim() == 2 && qkv.stride(1) == 1, "qkv must be 2-D with unit inner stride");
  TORCH_CHECK(cs.scalar_type() == torch::kFloat && cs.is_contiguous() && cs.numel() == seq * hd, "cs must be fp32 [seq, hd/2, 2]");
  c10::cuda::CUDAGuard guard(qkv.device());
  rope(qkv.data_ptr(), cs.data_ptr<float>(), int(qkv.size(0)), int(seq), int(heads_qk), int(hd), qkv.stride(0),
       int(pos_offset), inverse, sms(qkv), cur_stream());
}

torch::Tensor swiglu_fwd_t(torch::Tensor gu) {
  check_cuda_bf16(gu, "gu");
  TORCH_CHECK(gu.dim() == 2 && gu.is_contiguous(), "gu must be contiguous [rows, 2F]");
  c10::cuda::CUDAGuard guard(gu.device());
  const int64_t f = gu.size(1) / 2;
  auto h = torch::empty({gu.size(0), f}, gu.options());
  swiglu_fwd(gu.data_ptr(), h.data_ptr(), int(gu.size(0)), int(f), sms(gu), cur_stream());
  return h;
}

torch::Tensor swiglu_bwd_t(torch::Tensor gu, torch::Tensor dh) {
  check_cuda_bf16(gu, "gu");
  const int64_t f = gu.size(1) / 2;
  check_rows(dh, f, "dh");
  c10::cuda::CUDAGuard guard(gu.device());
  auto dgu = torch::empty_like(gu);
  swiglu_bwd(gu.data_ptr(), dh.data_ptr(), dgu.data_ptr(), int(gu.size(0)), int(f), sms(gu), cur_stream());
  return dgu;
}

// ---- AdamW ----------------------------------------------------------------------------

void adamw_t(torch::Tensor p, torch::Tensor g, torch::Tensor m, torch::Tensor v, c10::optional<torch::Tensor> p_bf16,
             double lr, double b1, double b2, double eps, double wd, int64_t step, double grad_scale) {
  for (auto* t : {&p, &g, &m, &v})
    TORCH_CHECK(t->is_cuda() && t->scalar_type() == torch::kFloat && t->is_contiguous() && t->numel() == p.numel(),
                "AdamW buffers must be contiguous fp32 of equal size");
  void* pb = nullptr;
  if (p_bf16.has_value()) {
    TORCH_CHECK(p_bf16->scalar_type() == torch::kBFloat16 && p_bf16->numel() == p.numel() && p_bf16->is_contiguous(),
                "bf16 copy must match");
    pb = p_bf16->data_ptr();
  }
  c10::cuda::CUDAGuard guard(p.device());
  adamw(p.data_ptr<float>(), g.data_ptr<float>(), m.data_ptr<float>(), v.data_ptr<float>(), pb, p.numel(), float(lr),
        float(b1), float(b2), float(eps), float(wd), step, float(grad_scale), sms(p), cur_stream());
}

// ---- embedding ------------------------------------------------------------------------

torch::Tensor embedding_fwd_t(torch::Tensor ids, torch::Tensor w, int64_t start) {
  TORCH_CHECK(ids.is_cuda() && ids.scalar_type() == torch::kLong && ids.is_contiguous(), "ids must be int64 CUDA");
  check_cuda_bf16(w, "w");
  TORCH_CHECK(w.dim() == 2 && w.is_contiguous(), "embedding table must be contiguous");
  c10::cuda::CUDAGuard guard(w.device());
  auto out = torch::empty({ids.numel(), w.size(1)}, w.options());
  embedding_fwd(ids.data_ptr<int64_t>(), w.data_ptr(), out.data_ptr(), int(ids.numel()), int(w.size(1)), start,
                w.size(0), cur_stream());
  return out;
}

void embedding_bwd_t(torch::Tensor ids, torch::Tensor dy, torch::Tensor dw, int64_t start) {
  TORCH_CHECK(ids.is_cuda() && ids.scalar_type() == torch::kLong, "ids must be int64 CUDA");
  check_cuda_bf16(dy, "dy");
  TORCH_CHECK(dw.scalar_type() == torch::kFloat && dw.dim() == 2 && dw.is_contiguous(), "dw must be fp32 [V, d]");
  c10::cuda::CUDAGuard guard(dy.device());
  auto flat = ids.reshape({-1}).contiguous();
  auto dy2 = dy.reshape({flat.numel(), dw.size(1)}).contiguous();
  const int64_t seg = std::min<int64_t>(flat.numel(), embedding_sort_segment());
  auto keys = torch::empty({std::max<int64_t>(seg, 1)}, flat.options());  // uint64 keys in int64 storage
  embedding_bwd(flat.data_ptr<int64_t>(), dy2.data_ptr(), dw.data_ptr<float>(),
                reinterpret_cast<uint64_t*>(keys.data_ptr<int64_t>()), int(flat.numel()), int(dw.size(1)), start,
                dw.size(0), cur_stream());
}

// ---- cross-entropy --------------------------------------------------------------------

torch::Tensor xent_stats_t(torch::Tensor logits, torch::Tensor labels, int64_t start) {
  check_cuda_bf16(logits, "logits");
  TORCH_CHECK(logits.dim() == 2 && logits.stride(1) == 1, "logits must be 2-D");
  TORCH_CHECK(labels.scalar_type() == torch::kLong && labels.numel() == logits.size(0) && labels.is_contiguous(),
              "labels must be int64 [rows]");
  c10::cuda::CUDAGuard guard(logits.device());
  auto stats = torch::empty({logits.size(0), 3}, logits.options().dtype(torch::kFloat));
  xent_stats(logits.data_ptr(), logits.stride(0), labels.data_ptr<int64_t>(), stats.data_ptr<float>(),
             int(logits.size(0)), int(logits.size(1)), start, cur_stream());
  return stats;
}

void xent_grad_t(torch::Tensor logits, torch::Tensor labels, torch::Tensor lse, torch::Tensor scale, int64_t start) {
  check_cuda_bf16(logits, "logits");
  TORCH_CHECK(lse.scalar_type() == torch::kFloat && lse.numel() == logits.size(0) && lse.is_contiguous(), "lse");
  TORCH_CHECK(scale.scalar_type() == torch::kFloat && scale.numel() == 1 && scale.is_cuda(), "scale must be a CUDA fp32 scalar");
  c10::cuda::CUDAGuard guard(logits.device());
  xent_grad(logits.data_ptr(), logits.stride(0), labels.data_ptr<int64_t>(), lse.data_ptr<float>(),
            scale.data_ptr<float>(), int(logits.size(0)), int(logits.size(1)), start, cur_stream());
}

// ---- attention ------------------------------------------------------------------------

std::vector<torch::Tensor> attn_fwd_t(torch::Tensor qkv, int64_t seq, int64_t hq, int64_t hkv, int64_t d, double scale) {
  check_cuda_bf16(qkv, "qkv");
  TORCH_CHECK(qkv.dim() == 2 && qkv.stride(1) == 1 && qkv.size(1) == (hq + 2 * hkv) * d, "qkv must be [T, (hq+2hkv)*d]");
  c10::cuda::CUDAGuard guard(qkv.device());
  const int64_t rows = qkv.size(0);
  auto out = torch::empty({rows, hq * d}, qkv.options());
  auto lse = torch::empty({rows / seq, hq, seq}, qkv.options().dtype(torch::kFloat));
  attn_fwd(qkv.data_ptr(), qkv.stride(0), out.data_ptr(), out.stride(0), lse.data_ptr<float>(), int(rows), int(seq),
           int(hq), int(hkv), int(d), float(scale), error_word(qkv.device()), cur_stream());
  return {out, lse};
}

torch::Tensor attn_bwd_t(torch::Tensor qkv, torch::Tensor out, torch::Tensor dout, torch::Tensor lse, int64_t seq,
                         int64_t hq, int64_t hkv, int64_t d, double scale) {
  check_cuda_bf16(qkv, "qkv");
  check_cuda_bf16(out, "out");
  check_cuda_bf16(dout, "dout");
  TORCH_CHECK(dout.stride(1) == 1 && out.stride(1) == 1, "attention tensors need unit inner stride");
  c10::cuda::CUDAGuard guard(qkv.device());
  const int64_t rows = qkv.size(0);
  auto dqkv = torch::empty({rows, (hq + 2 * hkv) * d}, qkv.options());
  auto delta = torch::empty_like(lse);
  attn_bwd(qkv.data_ptr(), qkv.stride(0), out.data_ptr(), out.stride(0), dout.data_ptr(), dout.stride(0),
           lse.data_ptr<float>(), delta.data_ptr<float>(), dqkv.data_ptr(), dqkv.stride(0), int(rows), int(seq),
           int(hq), int(hkv), int(d), float(scale), error_word(qkv.device()), cur_stream());
  return dqkv;
}


// ---- launch count -----------------------------------------------------------------------
// Kernels launched by the calls below, those of backward passes included, which no Python call
// shows (the launch counter adds them to what it sees).

static std::atomic<int64_t> g_launches{0};
static void count_launches(int64_t n) { g_launches.fetch_add(n, std::memory_order_relaxed); }

// ---- dropout --------------------------------------------------------------------------

torch::Tensor dropout_t(torch::Tensor x, c10::optional<torch::Tensor> residual, int64_t drop, int64_t seed,
                        int64_t offset, c10::optional<torch::Tensor> state, int64_t first) {
  TORCH_CHECK(x.is_cuda() && x.is_contiguous(), "dropout: x must be a contiguous CUDA tensor");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat, "dropout: x must be bf16 or fp32");
  const void* rp = nullptr;
  if (residual.has_value()) {
    TORCH_CHECK(residual->device() == x.device() && residual->scalar_type() == x.scalar_type() &&
                    residual->sizes() == x.sizes() && residual->is_contiguous(),
                "dropout: residual must match x");
    rp = residual->data_ptr();
  }
  const int64_t* sp = nullptr;
  if (state.has_value()) {
    TORCH_CHECK(state->device() == x.device() && state->scalar_type() == at::kLong && state->numel() == 2 &&
                    state->is_contiguous(), "dropout: the seed tensor must be int64 [2] beside x");
    sp = state->data_ptr<int64_t>();
  }
  TORCH_CHECK(drop >= 0 && drop <= 65536, "dropout threshold out of range");
  c10::cuda::CUDAGuard guard(x.device());
  auto out = torch::empty_like(x);
  dropout(x.data_ptr(), rp, out.data_ptr(), x.scalar_type() == at::kBFloat16, x.numel(), first, uint64_t(seed),
          uint64_t(offset), sp, uint32_t(drop), sms(x), cur_stream());
  count_launches(x.numel() > 0);
  return out;
}

// ---- sparse MLP: routing and row movements ----------------------------------------------

static void check_int32(const torch::Tensor& t, const torch::Tensor& like, const char* name) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == at::kInt && t.is_contiguous(), name,
              " must be a contiguous int32 tensor on the rows' device");
}

static void check_rows_count(int64_t rows, int64_t k) {
  TORCH_CHECK(rows <= kMoeMaxPairs / std::max<int64_t>(k, 1), message("tokens * k passes ", kMoeMaxPairs));
}

std::vector<torch::Tensor> moe_route_t(torch::Tensor logits, int64_t k, bool normalize) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.stride(1) == 1, "logits must be CUDA [tokens, experts]");
  TORCH_CHECK(logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kFloat, "logits must be bf16 or fp32");
  const int64_t t = logits.size(0), e = logits.size(1);
  check_rows_count(t, k);
  c10::cuda::CUDAGuard guard(logits.device());
  const auto ints = logits.options().dtype(torch::kInt);
  auto weights = torch::empty({t, k}, logits.options().dtype(torch::kFloat));
  auto ids = torch::empty({t, k}, ints);
  auto slots = torch::empty({t, k}, ints);
  auto offsets = torch::empty({e + 1}, ints);
  auto counts = torch::empty({moe_blocks(t * k, sms(logits)), e + 1}, ints);
  count_launches(moe_route(logits.data_ptr(), logits.scalar_type() == at::kBFloat16, logits.stride(0), int(t), int(e),
                           int(k), normalize, weights.data_ptr<float>(), ids.data_ptr<int>(), counts.data_ptr<int>(),
                           offsets.data_ptr<int>(), slots.data_ptr<int>(), sms(logits), cur_stream()));
  return {weights, ids, offsets, slots};
}

torch::Tensor moe_route_bwd_t(torch::Tensor logits, torch::Tensor weights, torch::Tensor ids, torch::Tensor dweights,
                              bool normalize) {
  const int64_t t = logits.size(0), e = logits.size(1), k = ids.size(1);
  TORCH_CHECK(dweights.device() == logits.device() && dweights.scalar_type() == at::kFloat && dweights.is_contiguous() &&
                  dweights.numel() == t * k, "weight gradients must be contiguous fp32 [tokens, k]");
  c10::cuda::CUDAGuard guard(logits.device());
  auto out = torch::empty({t, e}, logits.options());
  moe_route_bwd(logits.data_ptr(), logits.scalar_type() == at::kBFloat16, logits.stride(0), weights.data_ptr<float>(),
                ids.data_ptr<int>(), dweights.data_ptr<float>(), out.data_ptr(), int(t), int(e), int(k), normalize,
                cur_stream());
  count_launches(t > 0);
  return out;
}

std::vector<torch::Tensor> moe_plan_t(torch::Tensor ids, int64_t experts, int64_t start) {
  TORCH_CHECK(ids.is_cuda() && ids.scalar_type() == at::kInt && ids.is_contiguous(), "ids must be contiguous int32 CUDA");
  TORCH_CHECK(start >= INT32_MIN && start <= INT32_MAX, "first expert out of range");
  TORCH_CHECK(experts >= 1 && experts <= kMoeMaxExperts, "expert count out of range");
  check_rows_count(ids.numel(), 1);
  c10::cuda::CUDAGuard guard(ids.device());
  auto offsets = torch::empty({experts + 1}, ids.options());
  auto slots = torch::empty_like(ids);
  auto counts = torch::empty({moe_blocks(ids.numel(), sms(ids)), experts + 1}, ids.options());
  moe_plan(ids.data_ptr<int>(), ids.numel(), int(start), int(experts), counts.data_ptr<int>(), offsets.data_ptr<int>(),
           slots.data_ptr<int>(), sms(ids), cur_stream());
  count_launches(2);
  return {offsets, slots};
}

static void check_plan(const torch::Tensor& rows, const torch::Tensor& offsets, const torch::Tensor& slots) {
  check_int32(offsets, rows, "offsets");
  check_int32(slots, rows, "slots");
  TORCH_CHECK(offsets.dim() == 1 && offsets.numel() >= 2 && slots.dim() == 2 && slots.size(1) >= 1,
              "a plan is offsets [experts + 1] and slots [tokens, k]");
  check_rows_count(slots.size(0), slots.size(1));
}

torch::Tensor moe_scatter_t(torch::Tensor x, torch::Tensor offsets, torch::Tensor slots) {
  check_plan(x, offsets, slots);
  check_rows(x, x.size(-1), "x");
  TORCH_CHECK(x.size(0) == slots.size(0), "x must have a row per token");
  c10::cuda::CUDAGuard guard(x.device());
  auto out = torch::empty({slots.numel(), x.size(1)}, x.options());
  moe_scatter(x.data_ptr(), slots.data_ptr<int>(), offsets.data_ptr<int>() + offsets.numel() - 1, out.data_ptr(),
              int(x.size(0)), int(slots.size(1)), int(x.size(1)), error_word(x.device()), cur_stream());
  count_launches(x.size(0) > 0);
  return out;
}

static const float* check_weights(const c10::optional<torch::Tensor>& w, const torch::Tensor& slots) {
  if (!w.has_value()) return nullptr;
  TORCH_CHECK(w->device() == slots.device() && w->scalar_type() == at::kFloat && w->is_contiguous() &&
                  w->sizes() == slots.sizes(), "weights must be contiguous fp32 [tokens, k]");
  return w->data_ptr<float>();
}

torch::Tensor moe_gather_t(torch::Tensor y, c10::optional<torch::Tensor> weights, torch::Tensor offsets,
                           torch::Tensor slots, c10::optional<torch::Tensor> residual) {
  check_plan(y, offsets, slots);
  check_rows(y, y.size(-1), "y");
  TORCH_CHECK(y.size(0) == slots.numel(), "y must have a row per (token, choice) pair");
  const float* wp = check_weights(weights, slots);
  const void* rp = nullptr;
  if (residual.has_value()) {
    check_rows(*residual, y.size(1), "residual");
    TORCH_CHECK(residual->size(0) == slots.size(0) && residual->device() == y.device(), "residual must have a row per token");
    rp = residual->data_ptr();
  }
  c10::cuda::CUDAGuard guard(y.device());
  auto out = torch::empty({slots.size(0), y.size(1)}, y.options());
  moe_gather(y.data_ptr(), wp, rp, slots.data_ptr<int>(), offsets.data_ptr<int>() + offsets.numel() - 1, out.data_ptr(),
             int(slots.size(0)), int(slots.size(1)), int(y.size(1)), error_word(y.device()), sms(y), cur_stream());
  count_launches(slots.size(0) > 0);
  return out;
}

std::vector<torch::Tensor> moe_combine_bwd_t(torch::Tensor dout, torch::Tensor y, torch::Tensor weights,
                                             torch::Tensor offsets, torch::Tensor slots) {
  check_plan(dout, offsets, slots);
  check_rows(dout, y.size(-1), "dout");
  check_rows(y, y.size(-1), "y");
  TORCH_CHECK(dout.size(0) == slots.size(0) && y.size(0) == slots.numel() && y.device() == dout.device(), "combine shapes");
  const float* wp = check_weights(weights, slots);
  c10::cuda::CUDAGuard guard(dout.device());
  auto dy = torch::empty_like(y);
  auto dw = torch::empty(slots.sizes(), y.options().dtype(torch::kFloat));
  moe_combine_bwd(dout.data_ptr(), y.data_ptr(), wp, slots.data_ptr<int>(),
                  offsets.data_ptr<int>() + offsets.numel() - 1, dy.data_ptr(), dw.data_ptr<float>(),
                  int(slots.size(0)), int(slots.size(1)), int(y.size(1)), error_word(y.device()), sms(y), cur_stream());
  count_launches(slots.size(0) > 0);
  return {dy, dw};
}

// ---- products grouped by expert -----------------------------------------------------------

static GroupedShape grouped_shape(const torch::Tensor& rows, const torch::Tensor& offsets, int64_t n, int64_t k) {
  check_int32(offsets, rows, "offsets");
  TORCH_CHECK(offsets.dim() == 1 && offsets.numel() >= 2, "offsets must be [groups + 1]");
  TORCH_CHECK(rows.size(0) <= INT32_MAX - 512 && n <= INT32_MAX - 512 && k <= INT32_MAX - 512, "grouped product too large");
  return GroupedShape{offsets.data_ptr<int>(), int(offsets.numel() - 1), int(rows.size(0)), int(n), int(k)};
}

// a [rows, K] times w [groups, N, K] transposed, or with w_mn times w [groups, K, N].
torch::Tensor grouped_rows_t(torch::Tensor a, torch::Tensor w, bool w_mn, torch::Tensor offsets) {
  check_cuda_bf16(a, "rows");
  check_cuda_bf16(w, "weights");
  TORCH_CHECK(a.dim() == 2 && w.dim() == 3 && a.stride(1) == 1 && w.stride(2) == 1 && a.device() == w.device(),
              "grouped product needs [rows, K] and [groups, N, K] with unit inner strides on one device");
  const int64_t k = w_mn ? w.size(1) : w.size(2), n = w_mn ? w.size(2) : w.size(1);
  TORCH_CHECK(a.size(1) == k && w.size(0) == offsets.numel() - 1, "grouped product: sizes differ");
  const GroupedShape s = grouped_shape(a, offsets, n, k);
  c10::cuda::CUDAGuard guard(a.device());
  auto c = torch::empty({a.size(0), n}, a.options());
  torch::Tensor pace;  // this call's own: calls on other streams and in graphs have theirs
  if (grouped_paces(s)) pace = torch::empty({1}, offsets.options());
  grouped_rows(a.data_ptr(), a.stride(0), w.data_ptr(), w.stride(1), w.stride(0), w_mn, c.data_ptr(), n, s,
               pace.defined() ? reinterpret_cast<unsigned*>(pace.data_ptr<int>()) : nullptr, error_word(a.device()),
               cur_stream());
  count_launches(s.rows > 0);
  return c;
}

void grouped_wgrad_t(torch::Tensor dy, torch::Tensor x, torch::Tensor offsets, torch::Tensor out, bool accumulate) {
  check_cuda_bf16(dy, "dy");
  check_cuda_bf16(x, "x");
  TORCH_CHECK(dy.dim() == 2 && x.dim() == 2 && dy.stride(1) == 1 && x.stride(1) == 1 && dy.size(0) == x.size(0) &&
                  dy.device() == x.device(), "grouped wgrad needs dy [rows, N] and x [rows, K]");
  const GroupedShape s = grouped_shape(dy, offsets, dy.size(1), x.size(1));
  const bool bf16 = out.scalar_type() == at::kBFloat16;
  TORCH_CHECK(out.device() == dy.device() && (out.scalar_type() == at::kFloat || (bf16 && !accumulate)) &&
                  out.is_contiguous() && out.dim() == 3 && out.size(0) == s.groups && out.size(1) == s.n &&
                  out.size(2) == s.k,
              "grouped weight gradient must be contiguous [groups, N, K], fp32 or, written, bf16");
  c10::cuda::CUDAGuard guard(dy.device());
  grouped_wgrad(dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), out.data_ptr(), bf16, accumulate, s,
                error_word(dy.device()), cur_stream());
  count_launches(s.rows > 0);
}

// ---- differentiable forms -------------------------------------------------------------------
// The autograd nodes of the operators above. They are C++ so that a backward pass neither
// enters the interpreter nor waits for its lock: at the sizes where such an operator's kernels
// take 5 to 20 us, Python nodes made forward and backward of one of them 75 to 105 us of host
// time.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<torch::Tensor>;

// First in every backward pass. A leaf keeps the stream its first living graph was recorded on,
// and the engine joins that stream with the pass's, with or without a gradient for the leaf. If
// it is the default stream and the pass is being captured, the join is not allowed and the
// process may end in the engine, so it is refused here, where it is still an error, for every
// leaf that the pass will reach from here.
static void check_capture() {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const auto current = torch::autograd::get_current_node();
  std::vector<torch::autograd::Node*> todo = {current.get()};
  std::unordered_set<torch::autograd::Node*> seen = {current.get()};
  while (!todo.empty()) {
    torch::autograd::Node* node = todo.back();
    todo.pop_back();
    if (node == nullptr) continue;
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(node) != nullptr) {
      const auto stream = node->stream();
      TORCH_CHECK(!stream.has_value() || stream->id() != 0,
                  "a backward pass cannot be captured while a graph of the same leaf recorded on the default stream "
                  "is alive: drop its outputs, or record it on another stream");
    }
    for (size_t i = 0; i < node->num_outputs(); ++i)
      if (node->task_should_compute_output(i) && seen.insert(node->next_edge(i).function.get()).second)
        todo.push_back(node->next_edge(i).function.get());
  }
}

// These gradients have no derivative of their own: asking for one raises.
static variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);  // or the error's node would not be recorded
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice an operator of resihp whose gradient has no derivative", int64_t(grads.size()));
  return (*error)(std::move(grads));
}

static OptTensor rows_of(const OptTensor& t) { return t.has_value() ? OptTensor(t->contiguous()) : c10::nullopt; }

struct DropoutNode : torch::autograd::Function<DropoutNode> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& x, int64_t drop, int64_t seed, int64_t offset,
                               int64_t first, const OptTensor& state, const OptTensor& residual) {
    ctx->saved_data["args"] = std::vector<int64_t>{drop, seed, offset, first, residual.has_value(), state.has_value()};
    if (state.has_value()) ctx->save_for_backward({*state});
    return dropout_t(x.contiguous(), rows_of(residual), drop, seed, offset, state, first);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_capture();
    const auto a = ctx->saved_data["args"].toIntVector();
    OptTensor state;
    if (a[5]) state = ctx->get_saved_variables()[0];
    torch::Tensor dx;
    if (ctx->needs_input_grad(0)) dx = dropout_t(grads[0].contiguous(), c10::nullopt, a[0], a[1], a[2], state, a[3]);
    return once({dx, {}, {}, {}, {}, {}, a[4] ? grads[0] : torch::Tensor()});
  }
};

struct RouteNode : torch::autograd::Function<RouteNode> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& logits, int64_t k, bool normalize) {
    // (a copy, not contiguous(): that leaves a single column's stride as it is)
    const auto rows = logits.stride(1) == 1 ? logits : torch::empty(logits.sizes(), logits.options()).copy_(logits);
    auto out = moe_route_t(rows, k, normalize);
    ctx->mark_non_differentiable({out[1], out[2], out[3]});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({rows, out[0], out[1]});
    ctx->saved_data["normalize"] = normalize;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_capture();
    if (!grads[0].defined()) return {{}, {}, {}};
    const auto saved = ctx->get_saved_variables();
    return once({moe_route_bwd_t(saved[0], saved[1], saved[2], grads[0].contiguous(),
                                 ctx->saved_data["normalize"].toBool()), {}, {}});
  }
};

struct DispatchNode : torch::autograd::Function<DispatchNode> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& offsets,
                               const torch::Tensor& slots) {
    ctx->save_for_backward({offsets, slots});
    return moe_scatter_t(x.contiguous(), offsets, slots);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_capture();
    const auto saved = ctx->get_saved_variables();
    return once({moe_gather_t(grads[0].contiguous(), c10::nullopt, saved[0], saved[1], c10::nullopt), {}, {}});
  }
};

struct CombineNode : torch::autograd::Function<CombineNode> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& y, const torch::Tensor& weights,
                               const torch::Tensor& offsets, const torch::Tensor& slots, const OptTensor& residual) {
    const auto rows = y.contiguous();
    const auto w = weights.contiguous();
    ctx->save_for_backward({rows, w, offsets, slots});
    ctx->saved_data["residual"] = residual.has_value();
    return moe_gather_t(rows, w, offsets, slots, rows_of(residual));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_capture();
    const auto saved = ctx->get_saved_variables();
    std::vector<torch::Tensor> d(2);
    if (ctx->needs_input_grad(0) || ctx->needs_input_grad(1))
      d = moe_combine_bwd_t(grads[0].contiguous(), saved[0], saved[1], saved[2], saved[3]);
    return once({d[0], d[1], {}, {}, ctx->saved_data["residual"].toBool() ? grads[0] : torch::Tensor()});
  }
};

// A tensor as TMA reads it: unit inner stride, 16-byte aligned base and outer strides (which no
// two rows may share); anything else is copied.
static torch::Tensor tiles_of(const torch::Tensor& t) {
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) ok = ok && t.stride(d) > 0 && t.stride(d) % 8 == 0;
  return ok ? t : torch::empty(t.sizes(), t.options()).copy_(t);
}

struct GroupedNode : torch::autograd::Function<GroupedNode> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& w,
                               const torch::Tensor& offsets, const OptTensor& main_grad) {
    const auto xt = tiles_of(x), wt = tiles_of(w);
    ctx->save_for_backward({xt, wt, offsets});
    if (main_grad.has_value()) ctx->saved_data["main_grad"] = *main_grad;
    return grouped_rows_t(xt, wt, false, offsets);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_capture();
    const auto saved = ctx->get_saved_variables();
    const auto dy = tiles_of(grads[0]);
    torch::Tensor dx, dw;
    if (ctx->needs_input_grad(0)) dx = grouped_rows_t(dy, saved[1], true, saved[2]);
    const auto acc = ctx->saved_data.find("main_grad");
    if (acc != ctx->saved_data.end()) {
      grouped_wgrad_t(dy, saved[0], saved[2], acc->second.toTensor(), true);
    } else if (ctx->needs_input_grad(1)) {
      dw = torch::empty(saved[1].sizes(), saved[1].options());
      grouped_wgrad_t(dy, saved[0], saved[2], dw, false);
    }
    return once({dx, dw, {}, {}});
  }
};

static torch::Tensor dropout_ad(torch::Tensor x, int64_t drop, int64_t seed, int64_t offset, int64_t first,
                                OptTensor state, OptTensor residual) {
  return DropoutNode::apply(x, drop, seed, offset, first, state, residual);
}
static variable_list moe_route_ad(torch::Tensor logits, int64_t k, bool normalize) {
  return RouteNode::apply(logits, k, normalize);
}
static torch::Tensor moe_dispatch_ad(torch::Tensor x, torch::Tensor offsets, torch::Tensor slots) {
  return DispatchNode::apply(x, offsets, slots);
}
static torch::Tensor moe_combine_ad(torch::Tensor y, torch::Tensor weights, torch::Tensor offsets, torch::Tensor slots,
                                    OptTensor residual) {
  return CombineNode::apply(y, weights, offsets, slots, residual);
}
static torch::Tensor grouped_linear_ad(torch::Tensor x, torch::Tensor w, torch::Tensor offsets, OptTensor main_grad) {
  return GroupedNode::apply(x, w, offsets, main_grad);
}

// ---- debugging aid: native backtrace on SIGSEGV ---------------------------------------

static void crash_handler(int sig) {
  void* frames[64];
  const int n = backtrace(frames, 64);
  const char msg[] = "\n[resihp] native backtrace:\n";
  (void)!write(2, msg, sizeof(msg) - 1);
  backtrace_symbols_fd(frames, n, 2);
  signal(sig, SIG_DFL);
  raise(sig);
}

void install_crash_handler() { signal(SIGSEGV, crash_handler); }

// ---- symmetric workspace + fused TP collectives ---------------------------------------

template <class T>
static T* as_ptr(int64_t v) { return reinterpret_cast<T*>(static_cast<uintptr_t>(v)); }

py::tuple symm_alloc_t(int64_t bytes) {
  cudaIpcMemHandle_t h;
  void* p = symm_alloc(bytes, &h);
  return py::make_tuple(reinterpret_cast<int64_t>(p), py::bytes(reinterpret_cast<const char*>(&h), sizeof(h)));
}

int64_t symm_open_t(py::bytes handle) {
  std::string s = handle;
  TORCH_CHECK(s.size() == sizeof(cudaIpcMemHandle_t), "bad IPC handle size");
  return reinterpret_cast<int64_t>(symm_open(s.data()));
}

void symm_close_t(int64_t p) { symm_close(as_ptr<void>(p)); }

// Debug helpers for guard bytes around workspace buffers (synchronous, any device memory).
void debug_fill_bytes_t(int64_t p, int64_t bytes, int64_t value) {
  C10_CUDA_CHECK(cudaMemset(as_ptr<void>(p), int(value & 0xff), size_t(bytes)));
}

py::bytes debug_read_bytes_t(int64_t p, int64_t bytes) {
  std::string out(size_t(bytes), '\0');
  C10_CUDA_CHECK(cudaMemcpy(out.data(), as_ptr<const void>(p), size_t(bytes), cudaMemcpyDeviceToHost));
  return py::bytes(out);
}
void symm_free_t(int64_t p) { symm_free(as_ptr<void>(p)); }

int64_t fused_grid_t(int64_t m, int64_t n, int64_t tp) { return fused_grid(int(m), int(n), int(tp)); }
int64_t fused_slices_t(int64_t rows_per_rank) { return fused_slices(int(rows_per_rank)); }
int64_t fused_tile_claims_t(int64_t t_rows, int64_t n, int64_t grid) {
  return fused_tile_claims(int(t_rows), int(n), int(grid));
}
int64_t fused_copy_claims_t(int64_t mode, int64_t t_rows, int64_t n, int64_t tp, int64_t slices, int64_t xg_chunks,
                            int64_t grid) {
  return fused_copy_claims(int(mode), int(t_rows), int(n), int(tp), int(slices), int(xg_chunks), int(grid));
}

// The peers of one fused call as a flat int64 list: rank, tp, rows_per_rank, slices, epoch,
// ar_epoch, tile_ctr, tile_base, copy_ctr, copy_base, then tp addresses each of land,
// ag_cnt, recv, rs_cnt, out_land, ar_cnt (0 where a call does not use them).
static FusedPeers decode_peers(const std::vector<int64_t>& v) {
  TORCH_CHECK(v.size() >= 10, "fused peers: header missing");
  FusedPeers p{};
  p.rank = int(v[0]);
  p.tp = int(v[1]);
  p.rows_per_rank = int(v[2]);
  p.slices = int(v[3]);
  p.epoch = unsigned(v[4]);
  p.ar_epoch = unsigned(v[5]);
  p.tile_ctr = as_ptr<unsigned>(v[6]);
  p.tile_base = unsigned(v[7]);
  p.copy_ctr = as_ptr<unsigned>(v[8]);
  p.copy_base = unsigned(v[9]);
  TORCH_CHECK(p.tp >= 2 && p.tp <= kFusedMaxTp && v.size() == size_t(10 + 6 * p.tp + 3), "fused peers: bad length");
  for (int r = 0; r < p.tp; ++r) {
    p.land[r] = as_ptr<__nv_bfloat16>(v[10 + r]);
    p.ag_cnt[r] = as_ptr<unsigned>(v[10 + p.tp + r]);
    p.recv[r] = as_ptr<__nv_bfloat16>(v[10 + 2 * p.tp + r]);
    p.rs_cnt[r] = as_ptr<unsigned>(v[10 + 3 * p.tp + r]);
    p.out_land[r] = as_ptr<__nv_bfloat16>(v[10 + 4 * p.tp + r]);
    p.ar_cnt[r] = as_ptr<unsigned>(v[10 + 5 * p.tp + r]);
  }
  p.send = as_ptr<__nv_bfloat16>(v[10 + 6 * p.tp]);
  p.send_cnt = as_ptr<unsigned>(v[11 + 6 * p.tp]);
  p.own_cnt = as_ptr<unsigned>(v[12 + 6 * p.tp]);
  return p;
}

void ag_gemm_t(torch::Tensor x_local, c10::optional<torch::Tensor> xg, torch::Tensor w, bool w_mn, torch::Tensor y,
               std::vector<int64_t> peers, int64_t grid) {
  check_cuda_bf16(x_local, "x_local");
  check_cuda_bf16(w, "w");
  check_cuda_bf16(y, "y");
  const FusedPeers p = decode_peers(peers);
  TORCH_CHECK(x_local.is_contiguous() && y.is_contiguous() && w.stride(1) == 1, "fused AG-GEMM tensors must be contiguous");
  const int64_t k = x_local.size(1);
  const int64_t t = x_local.size(0) * p.tp;
  const int64_t n = y.size(1);
  TORCH_CHECK(y.size(0) == t, "fused AG-GEMM shapes");
  void* xg_ptr = nullptr;
  if (xg.has_value()) {
    check_cuda_bf16(*xg, "xg");
    TORCH_CHECK(xg->is_contiguous() && xg->size(0) == t && xg->size(1) == k, "fused AG-GEMM gathered-copy shape");
    xg_ptr = xg->data_ptr();
  }
  TORCH_CHECK(w_mn ? (w.size(0) == k && w.size(1) == n) : (w.size(0) == n && w.size(1) == k), "fused AG-GEMM weight");
  c10::cuda::CUDAGuard guard(x_local.device());
  fused_ag_gemm(x_local.data_ptr(), xg_ptr, w.data_ptr(), w.stride(0), w_mn, y.data_ptr(), y.stride(0), int(t),
                int(n), int(k), p, int(grid), error_word(x_local.device()), cur_stream());
}

// RS (all_reduce false): y is this rank's [T/tp, N] rows; AR: y is the full [T, N].
void gemm_rs_t(torch::Tensor h, torch::Tensor w, bool w_mn, torch::Tensor y, bool all_reduce,
               std::vector<int64_t> peers, int64_t grid) {
  check_cuda_bf16(h, "h");
  check_cuda_bf16(w, "w");
  check_cuda_bf16(y, "y");
  const FusedPeers p = decode_peers(peers);
  TORCH_CHECK(h.is_contiguous() && y.is_contiguous() && w.stride(1) == 1, "fused GEMM-RS tensors must be contiguous");
  const int64_t t = h.size(0), k = h.size(1), n = y.size(1);
  TORCH_CHECK(all_reduce ? y.size(0) == t : y.size(0) * p.tp == t, "fused GEMM-RS/AR shapes");
  TORCH_CHECK(w_mn ? (w.size(0) == k && w.size(1) == n) : (w.size(0) == n && w.size(1) == k), "fused GEMM-RS weight");
  c10::cuda::CUDAGuard guard(h.device());
  fused_gemm_rs(h.data_ptr(), w.data_ptr(), w.stride(0), w_mn, y.data_ptr(), y.stride(0), int(t), int(n), int(k),
                all_reduce, p, int(grid), error_word(h.device()), cur_stream());
}

// ---- flat-state regions and the peer-state kernels ----------------------------------------

// A zeroed, IPC-exported device allocation wrapped as a uint8 tensor. The memory is
// released when the last tensor viewing it dies (the deleter frees it on its device).
py::tuple symm_region_t(int64_t bytes, int64_t device) {
  TORCH_CHECK(bytes > 0, "region size must be positive");
  c10::cuda::CUDAGuard guard(c10::Device(c10::kCUDA, device));
  cudaIpcMemHandle_t h;
  void* p = symm_alloc(bytes, &h);
  const int dev = int(device);
  auto opts = torch::TensorOptions().dtype(torch::kUInt8).device(torch::kCUDA, device);
  auto t = torch::from_blob(
      p, {bytes},
      [dev](void* q) {
        int prev = 0;
        cudaGetDevice(&prev);
        cudaSetDevice(dev);
        cudaFree(q);
        cudaSetDevice(prev);
      },
      opts);
  return py::make_tuple(t, py::bytes(reinterpret_cast<const char*>(&h), sizeof(h)));
}

int64_t dp_grid_t(int64_t n, int64_t device) {
  return dp_grid(n, at::cuda::getDeviceProperties(device)->multiProcessorCount);
}

void dp_allreduce_adamw_t(std::vector<int64_t> grads, int64_t me, torch::Tensor sum_out, torch::Tensor p,
                          torch::Tensor m, torch::Tensor v, c10::optional<torch::Tensor> p_bf16, double lr, double b1,
                          double b2, double eps, double wd, int64_t step, double grad_scale, int64_t flags_local,
                          std::vector<int64_t> flags_peer, int64_t epoch, int64_t grid,
                          std::vector<int64_t> sums_peer, int64_t flags2_local, std::vector<int64_t> flags2_peer) {
  for (auto* t : {&sum_out, &p, &m, &v})
    TORCH_CHECK(t->is_cuda() && t->scalar_type() == torch::kFloat && t->is_contiguous() && t->numel() == p.numel(),
                "DP AdamW buffers must be contiguous fp32 of equal size");
  const int64_t dp = int64_t(grads.size());
  TORCH_CHECK(dp >= 1 && dp <= kMaxDp && int64_t(flags_peer.size()) == dp && me >= 0 && me < dp,
              "one gradient buffer and one flag array per DP rank");
  void* pb = nullptr;
  if (p_bf16.has_value()) {
    TORCH_CHECK(p_bf16->scalar_type() == torch::kBFloat16 && p_bf16->numel() == p.numel() && p_bf16->is_contiguous(),
                "bf16 copy must match");
    pb = p_bf16->data_ptr();
  }
  c10::cuda::CUDAGuard guard(p.device());
  std::vector<const float*> g;
  std::vector<unsigned*> f;
  for (auto x : grads) g.push_back(as_ptr<const float>(x));
  for (auto x : flags_peer) f.push_back(as_ptr<unsigned>(x));
  const AdamWCoef c = adamw_coef(float(lr), float(b1), float(b2), float(eps), float(wd), step, float(grad_scale));
  const bool push = !sums_peer.empty();
  TORCH_CHECK(!push || (int64_t(sums_peer.size()) == dp && int64_t(flags2_peer.size()) == dp && flags2_local != 0),
              "the push variant needs one receiving buffer and one second flag array per DP rank");
  std::vector<float*> sp;
  std::vector<unsigned*> f2;
  for (auto x : sums_peer) sp.push_back(as_ptr<float>(x));
  for (auto x : flags2_peer) f2.push_back(as_ptr<unsigned>(x));
  dp_allreduce_adamw(g.data(), int(dp), int(me), sum_out.data_ptr<float>(), p.data_ptr<float>(), m.data_ptr<float>(),
                     v.data_ptr<float>(), pb, p.numel(), c, as_ptr<unsigned>(flags_local), f.data(), unsigned(epoch),
                     int(grid), error_word(p.device()), cur_stream(), push ? sp.data() : nullptr,
                     push ? as_ptr<unsigned>(flags2_local) : nullptr, push ? f2.data() : nullptr);
}

// descs: int64 [n, 9] on the device, one CopyDesc per row (see launch.h for the fields).
void reshard_gather_t(torch::Tensor descs, int64_t items) {
  static_assert(sizeof(CopyDesc) == 9 * sizeof(int64_t), "CopyDesc is nine 8-byte fields");
  TORCH_CHECK(descs.is_cuda() && descs.scalar_type() == torch::kLong && descs.is_contiguous() && descs.dim() == 2 &&
                  descs.size(1) == 9, "copy descriptors must be a contiguous int64 [n, 9] CUDA tensor");
  c10::cuda::CUDAGuard guard(descs.device());
  reshard_gather(reinterpret_cast<const CopyDesc*>(descs.data_ptr<int64_t>()), int(descs.size(0)), items,
                 error_word(descs.device()), at::cuda::getDeviceProperties(descs.device().index())->multiProcessorCount,
                 cur_stream());
}

}  // namespace resihp

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "resihp sm_100a kernels";
  m.def("read_and_clear_error", &resihp::read_and_clear_error, "synchronising read+reset of the kernel error word");
  m.def("peer_wait_budget_ns", [] { return int64_t(resihp::peer_wait_budget_ns()); },
        "budget of each in-kernel wait on another GPU's flag (ns)");
  m.def("set_peer_wait_budget_ns", [](int64_t ns) { resihp::set_peer_wait_budget_ns(uint64_t(ns)); },
        "set the budget of each in-kernel wait on another GPU's flag (ns)");
  m.def("fused_red_slices", &resihp::fused_red_slices, "row slices per own tile of the fused RS / AR reduction");
  m.def("set_fused_trace", [](int64_t ptr) { resihp::set_fused_trace(reinterpret_cast<uint64_t*>(ptr)); },
        "profiling aid: per-CTA timer stamps of the fused TP kernels into a device buffer (0: off)");
  m.def("fused_trace_slots", &resihp::fused_trace_slots, "stamps per CTA of the fused-kernel trace");
  m.def("set_fused_push_depth", &resihp::set_fused_push_depth,
        "RS / AR partial-tile pushes in flight per copy thread: 2 pipelined, 1 one at a time (default)");
  m.def("gemm", &resihp::gemm, "tcgen05 bf16 GEMM", py::arg("a"), py::arg("a_mn"), py::arg("b"), py::arg("b_mn"),
        py::arg("c"), py::arg("epi"), py::arg("alpha") = 1.0, py::arg("residual") = py::none(),
        py::arg("max_ctas") = 0, py::arg("force_bn") = 0);
  m.def("rmsnorm_fwd", &resihp::rmsnorm_fwd_t);
  m.def("rmsnorm_bwd", &resihp::rmsnorm_bwd_t);
  m.def("rope", &resihp::rope_t);
  m.def("swiglu_fwd", &resihp::swiglu_fwd_t);
  m.def("swiglu_bwd", &resihp::swiglu_bwd_t);
  m.def("adamw", &resihp::adamw_t);
  m.def("embedding_fwd", &resihp::embedding_fwd_t);
  m.def("embedding_bwd", &resihp::embedding_bwd_t);
  m.def("xent_stats", &resihp::xent_stats_t);
  m.def("xent_grad", &resihp::xent_grad_t);
  m.def("attn_fwd", &resihp::attn_fwd_t);
  m.def("attn_bwd", &resihp::attn_bwd_t);
  m.def("dropout", &resihp::dropout_t);
  m.def("moe_route", &resihp::moe_route_t);
  m.def("moe_route_bwd", &resihp::moe_route_bwd_t);
  m.def("moe_plan", &resihp::moe_plan_t);
  m.def("moe_scatter", &resihp::moe_scatter_t);
  m.def("moe_gather", &resihp::moe_gather_t);
  m.def("moe_combine_bwd", &resihp::moe_combine_bwd_t);
  m.def("grouped_rows", &resihp::grouped_rows_t);
  m.def("grouped_wgrad", &resihp::grouped_wgrad_t);
  m.def("native_launches", [] { return resihp::g_launches.load(); },
        "kernels launched so far by the calls from dropout to grouped_linear_ad, backward passes included");
  m.def("dropout_ad", &resihp::dropout_ad);
  m.def("moe_route_ad", &resihp::moe_route_ad);
  m.def("moe_dispatch_ad", &resihp::moe_dispatch_ad);
  m.def("moe_combine_ad", &resihp::moe_combine_ad);
  m.def("grouped_linear_ad", &resihp::grouped_linear_ad);
  m.def("install_crash_handler", &resihp::install_crash_handler);
  m.def("symm_alloc", &resihp::symm_alloc_t);
  m.def("symm_open", &resihp::symm_open_t);
  m.def("symm_close", &resihp::symm_close_t);
  m.def("symm_free", &resihp::symm_free_t);
  m.def("debug_fill_bytes", &resihp::debug_fill_bytes_t);
  m.def("debug_read_bytes", &resihp::debug_read_bytes_t);
  m.def("fused_grid", &resihp::fused_grid_t);
  m.def("fused_slices", &resihp::fused_slices_t);
  m.def("fused_tile_claims", &resihp::fused_tile_claims_t);
  m.def("fused_copy_claims", &resihp::fused_copy_claims_t);
  m.def("ag_gemm", &resihp::ag_gemm_t, py::arg("x_local"), py::arg("xg"), py::arg("w"), py::arg("w_mn"), py::arg("y"),
        py::arg("peers"), py::arg("grid"));
  m.def("gemm_rs", &resihp::gemm_rs_t, py::arg("h"), py::arg("w"), py::arg("w_mn"), py::arg("y"),
        py::arg("all_reduce"), py::arg("peers"), py::arg("grid"));
  m.def("symm_region", &resihp::symm_region_t);
  m.def("dp_grid", &resihp::dp_grid_t);
  m.def("dp_allreduce_adamw", &resihp::dp_allreduce_adamw_t, py::arg("grads"), py::arg("me"), py::arg("sum_out"),
        py::arg("p"), py::arg("m"), py::arg("v"), py::arg("p_bf16"), py::arg("lr"), py::arg("b1"), py::arg("b2"),
        py::arg("eps"), py::arg("wd"), py::arg("step"), py::arg("grad_scale"), py::arg("flags_local"),
        py::arg("flags_peer"), py::arg("epoch"), py::arg("grid"), py::arg("sums_peer") = std::vector<int64_t>{},
        py::arg("flags2_local") = 0, py::arg("flags2_peer") = std::vector<int64_t>{});
  m.def("reshard_gather", &resihp::reshard_gather_t);
}
