// Native torch binding of the kernel bank's C ABI: the reference shipped its
// op as a pybind11/torch C++ extension (src/gemm_ext.cpp:22-132), and so does
// this build.  The ctypes path in infinite_dreams_ext.py reaches the same C
// ABI; this module removes the Python work around each call (argument checks,
// allocation of C, stream lookup, workspace lookup), which dominates the cost
// of a small GEMM launched back to back.
//
// Exported (all asynchronous on the current stream of A's device):
//   gemm_forward_cfg(A, B, cfg_id, out=None) -> C             (gemm_ext.cpp:95-106)
//   gemm_ex(A, B, cfg_id, alpha, beta, C, bias, act, out) -> out
//   grouped_gemm(A, B, offsets, bias, act, out) -> out
//   grouped_gemm_wgrad(A, G, offsets, out) -> out
//   grouped_linear(x, weight, offsets) -> y, differentiable
//   lora_gemm(x, W, down, up, adapter, scale, bias, act, out) -> out
//   reset_workspaces()
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <map>
#include <mutex>
#include <utility>

#include "../../include/gemm_sm100.h"

namespace {

// Split-K / repack workspace per (device, stream), zero-initialised once as
// the C ABI requires; grows geometrically.  Leaked on purpose: freeing CUDA
// memory from a static destructor at exit would race the context teardown.
std::mutex g_ws_mu;
std::map<std::pair<int, cudaStream_t>, at::Tensor>* g_ws = new std::map<std::pair<int, cudaStream_t>, at::Tensor>();

void* workspace(const at::Device& dev, cudaStream_t stream, size_t nbytes, size_t* len) {
  std::lock_guard<std::mutex> lock(g_ws_mu);
  at::Tensor& ws = (*g_ws)[{dev.index(), stream}];
  if (!ws.defined() || static_cast<size_t>(ws.numel()) < nbytes) {
    const int64_t grown = ws.defined() ? 2 * ws.numel() : 0;
    const int64_t size = std::max<int64_t>(static_cast<int64_t>(nbytes), grown);
    ws = at::zeros({size}, at::TensorOptions().dtype(at::kByte).device(dev));
  }
  *len = static_cast<size_t>(ws.numel());
  return ws.data_ptr();
}

void check_inputs(const at::Tensor& A, const at::Tensor& B) {
  // Same checks and messages as src/gemm_ext.cpp:66-73,86.
  TORCH_CHECK(A.is_cuda(), "A must be CUDA tensor");
  TORCH_CHECK(B.is_cuda(), "B must be CUDA tensor");
  TORCH_CHECK(A.scalar_type() == at::kHalf, "A must be float16");
  TORCH_CHECK(B.scalar_type() == at::kHalf, "B must be float16");
  TORCH_CHECK(A.dim() == 2, "A must be 2D (M x K)");
  TORCH_CHECK(B.dim() == 2, "B must be 2D (K x N)");
  TORCH_CHECK(A.size(1) == B.size(0), "Inner dimensions must match: A is (M x K), B is (K x N)");
  TORCH_CHECK(A.get_device() == B.get_device(), "A and B must be on the same CUDA device");
}

void check_status(int st, const char* what) {
  TORCH_CHECK(st == GEMM_OK, what, ": ", gemm_status_string(st), ": ", gemm_last_error());
}

at::Tensor output(const c10::optional<at::Tensor>& out, int64_t M, int64_t N, const at::Tensor& A) {
  if (!out.has_value()) return at::empty({M, N}, A.options());
  const at::Tensor& C = *out;
  TORCH_CHECK(C.scalar_type() == at::kHalf && C.dim() == 2 && C.size(0) == M && C.size(1) == N &&
                  C.device() == A.device() && (C.stride(1) == 1 || N <= 1) && (M <= 1 || C.stride(0) >= N),
              "out must be a float16 (M x N) tensor with unit column stride on A's device, its rows apart");
  return C;
}

at::Tensor gemm_forward_cfg(at::Tensor A, at::Tensor B, int64_t cfg_id, c10::optional<at::Tensor> out) {
  check_inputs(A, B);
  TORCH_CHECK(cfg_id >= 0, "cfg_id must be >= 0");
  TORCH_CHECK(cfg_id < gemm_num_cfgs(), "cfg_id out of range");
  const c10::cuda::CUDAGuard guard(A.device());
  A = A.contiguous();
  B = B.contiguous();
  const int64_t M = A.size(0), K = A.size(1), N = B.size(1);
  at::Tensor C = output(out, M, N, A);
  TORCH_CHECK(C.is_contiguous(), "out must be contiguous");
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(A.device().index()).stream();
  const size_t need = gemm_workspace_bytes(A.data_ptr(), B.data_ptr(), M, N, K, K, N, static_cast<int>(cfg_id));
  size_t len = 0;
  void* ws = need ? workspace(A.device(), stream, need, &len) : nullptr;
  check_status(gemm_launch(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, N, K, K, N, N, static_cast<int>(cfg_id),
                           ws, len, stream),
               "gemm_launch");
  return C;
}

// (tensor, trans, pitch) of a logical [R, C] operand read in place: a
// row-major view as stored, a transposed view (unit row stride) as its
// transposed storage, anything else copied contiguous.
std::tuple<at::Tensor, int, int64_t> operand(const at::Tensor& X) {
  const int64_t R = X.size(0), Cc = X.size(1), s0 = X.stride(0), s1 = X.stride(1);
  if ((s1 == 1 || Cc <= 1) && s0 >= std::max<int64_t>(Cc, 1)) return {X, 0, s0};
  if ((s0 == 1 || R <= 1) && s1 >= std::max<int64_t>(R, 1)) return {X, 1, s1};
  return {X.contiguous(), 0, std::max<int64_t>(Cc, 1)};
}

at::Tensor gemm_ex(const at::Tensor& A, const at::Tensor& B, int64_t cfg_id, double alpha, double beta,
                   c10::optional<at::Tensor> Cin, c10::optional<at::Tensor> bias, int64_t act,
                   c10::optional<at::Tensor> out) {
  check_inputs(A, B);
  TORCH_CHECK(cfg_id >= 0 && cfg_id < gemm_num_cfgs(), "cfg_id out of range");
  const c10::cuda::CUDAGuard guard(A.device());
  const int64_t M = A.size(0), K = A.size(1), N = B.size(1);
  at::Tensor D;
  if (beta != 0.0) {
    TORCH_CHECK(Cin.has_value(), "beta != 0 needs C");
    D = *Cin;
    TORCH_CHECK(D.scalar_type() == at::kHalf && D.dim() == 2 && D.size(0) == M && D.size(1) == N &&
                    D.device() == A.device(),
                "C must be a float16 (M x N) tensor on A's device");
    if ((D.stride(1) != 1 && N > 1) || (M > 1 && D.stride(0) < N)) D = D.contiguous();   // expanded rows too
  }
  at::Tensor bvec;
  if (bias.has_value()) {
    bvec = *bias;
    TORCH_CHECK(bvec.scalar_type() == at::kHalf && bvec.numel() == N && bvec.device() == A.device(),
                "bias must be a float16 tensor of N elements on A's device");
    bvec = bvec.reshape({N}).contiguous();
  }
  auto [As, ta, lda] = operand(A);
  auto [Bs, tb, ldb] = operand(B);
  at::Tensor C = output(out, M, N, A);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(A.device().index()).stream();
  const size_t need = gemm_workspace_bytes_ex(As.data_ptr(), Bs.data_ptr(), M, N, K, lda, ldb, ta, tb,
                                              static_cast<int>(cfg_id));
  size_t len = 0;
  void* ws = need ? workspace(A.device(), stream, need, &len) : nullptr;
  check_status(gemm_launch_ex(As.data_ptr(), Bs.data_ptr(), C.data_ptr(), M, N, K, lda, ldb,
                              std::max<int64_t>(C.stride(0), N), ta, tb, static_cast<float>(alpha),
                              static_cast<float>(beta), D.defined() ? D.data_ptr() : nullptr,
                              D.defined() ? std::max<int64_t>(D.stride(0), N) : 0,
                              bvec.defined() ? bvec.data_ptr() : nullptr, static_cast<int>(act),
                              static_cast<int>(cfg_id), ws, len, stream),
               "gemm_launch_ex");
  return C;
}

// Scratch of one call of the operators below, from torch's allocator and not
// the cached workspace: their launches come in twos (repacking or the low-rank
// half, then the product), between which another thread's call on the same
// stream -- a backward pass has a thread of its own -- would overwrite a shared
// buffer; and two graphs captured on one stream may be replayed on two.
at::Tensor scratch(const at::Device& dev, size_t nbytes) {
  if (nbytes == 0) return {};
  return at::empty({static_cast<int64_t>(nbytes)}, at::TensorOptions().dtype(at::kByte).device(dev));
}

void* scratch_ptr(const at::Tensor& ws) { return ws.defined() ? ws.data_ptr() : nullptr; }

size_t scratch_bytes(const at::Tensor& ws) { return ws.defined() ? static_cast<size_t>(ws.numel()) : 0; }

bool is_16bit(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

int dtype_id(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? GEMM_DTYPE_BF16 : GEMM_DTYPE_F16; }

// A is the operand that holds the rows; every other one goes by it.
void check_like(const at::Tensor& t, const at::Tensor& A, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == A.device(), name, " must be on the rows' device");
  TORCH_CHECK(t.scalar_type() == A.scalar_type(), name, " must have the rows' dtype");
}

void check_index(const at::Tensor& t, const at::Tensor& A, int64_t n, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == A.device(), name, " must be on the rows' device");
  TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64");
  TORCH_CHECK(t.dim() == 1 && t.size(0) == n, name, " must be 1D with ", n, " elements");
}

int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0 ? 1 : 0); }

// Whether a tensor shares bytes with `out`, which is rows of adjacent elements (2D),
// or a stack of them (3D, row-major or transposed, its matrices apart).
bool shares_memory(const at::Tensor& out, const at::Tensor& t) {
  auto extent = [](const at::Tensor& x) {   // bytes from the first to the last element
    int64_t n = 1;
    for (int64_t d = 0; d < x.dim(); ++d) n += (x.size(d) - 1) * x.stride(d);
    return n * static_cast<int64_t>(x.element_size());
  };
  const int64_t es = static_cast<int64_t>(out.element_size()), ts = static_cast<int64_t>(t.element_size());
  const int64_t o0 = reinterpret_cast<int64_t>(out.data_ptr()), t0 = reinterpret_cast<int64_t>(t.data_ptr());
  if (t0 + extent(t) <= o0 || o0 + extent(out) <= t0) return false;
  if (extent(t) == t.numel() * ts && extent(out) == out.numel() * es) return true;   // two dense blocks
  if (t.dim() == 2 && out.dim() == 2 && es == ts && t.stride(1) == 1 && out.stride(1) == 1 && t.size(0) > 1 &&
      out.size(0) > 1 && t.stride(0) == out.stride(0) && t.stride(0) >= std::max(t.size(1), out.size(1))) {
    // columns of one buffer: where t's begin in out's rows
    const int64_t row = out.stride(0) * es, c = floor_div(t0 - o0, row) * -row + t0 - o0;
    return c < out.size(1) * es || c + t.size(1) * es > row;
  }
  // out: E matrices, se bytes apart, of R rows, sr apart, of `width` bytes
  const int64_t d = out.dim();
  const bool trans = d == 3 && out.stride(2) != 1 && out.size(2) > 1;
  const int64_t row_dim = d - (trans ? 1 : 2), col_dim = d - (trans ? 2 : 1);
  const int64_t far = extent(out) + 1;   // the pitch of one thing
  const int64_t R = out.size(row_dim), width = out.size(col_dim) * es, E = d == 3 ? out.size(0) : 1;
  const int64_t sr = R > 1 ? out.stride(row_dim) * es : far, se = E > 1 ? out.stride(0) * es : far;
  auto meets = [&](int64_t a, int64_t b) {   // the bytes [a, b)
    a -= o0;
    b -= o0;
    const int64_t e = floor_div(a, se), next_e = std::max<int64_t>(e + 1, 0);
    if (next_e < E && next_e * se < b) return true;   // the next matrix begins before b
    if (e < 0 || e >= E) return false;
    const int64_t r = floor_div(a - e * se, sr), next_r = r + 1;
    return (r < R && a - e * se - r * sr < width) || (next_r < R && e * se + next_r * sr < b);
  };
  // t: runs of adjacent elements
  int64_t run_dim = -1;
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (t.stride(i) == 1 && t.size(i) > 1) run_dim = i;
  }
  const int64_t run = (run_dim >= 0 ? t.size(run_dim) : 1) * ts;
  int64_t size[3] = {1, 1, 1}, stride[3] = {0, 0, 0};
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (i == run_dim || t.stride(i) == 0) continue;
    size[i] = t.size(i);
    stride[i] = t.stride(i) * ts;
  }
  for (int64_t i = 0; i < size[0]; ++i) {
    for (int64_t j = 0; j < size[1]; ++j) {
      for (int64_t k = 0; k < size[2]; ++k) {
        const int64_t at = t0 + i * stride[0] + j * stride[1] + k * stride[2];
        if (meets(at, at + run)) return true;
      }
    }
  }
  return false;
}

// The kernels read operands while they write `out`.
void check_apart(const at::Tensor& out, std::initializer_list<at::Tensor> ts) {
  if (out.numel() == 0) return;
  for (const at::Tensor& t : ts) {
    TORCH_CHECK(!t.defined() || t.numel() == 0 || !shares_memory(out, t), "out must not share memory with an operand");
  }
}

// A graph that saved `out` notices that it was written; tensors made in
// inference mode keep no such count.
void count_write(const at::Tensor& out) {
  if (!out.is_inference()) torch::autograd::impl::bump_version(out);
}

void check_no_grad(const char* what, std::initializer_list<at::Tensor> ts) {
  for (const at::Tensor& t : ts) {
    if (!t.defined()) continue;
    TORCH_CHECK(!at::GradMode::is_enabled() || !t.requires_grad(), what);
    TORCH_CHECK(!t._fw_grad(0).defined(), "the operator has no forward-mode derivative: an input's tangent would be lost");
  }
}

// A stack of weights [E, R, C] read in place: (tensor, trans, pitch, stride
// from one matrix to the next); strides that are neither row-major nor
// transposed, or matrices that overlap (expanded weights), are copied.
std::tuple<at::Tensor, int, int64_t, int64_t> stacked_operand(const at::Tensor& X) {
  const int64_t E = X.size(0), R = X.size(1), Cc = X.size(2), se = X.stride(0), s0 = X.stride(1), s1 = X.stride(2);
  if ((s1 == 1 || Cc <= 1) && s0 >= std::max<int64_t>(Cc, 1) && (E == 1 || se >= (R - 1) * s0 + Cc)) {
    return {X, 0, s0, se};
  }
  if ((s0 == 1 || R <= 1) && s1 >= std::max<int64_t>(R, 1) && (E == 1 || se >= (Cc - 1) * s1 + R)) {
    return {X, 1, s1, se};
  }
  return {X.contiguous(), 0, std::max<int64_t>(Cc, 1), R * std::max<int64_t>(Cc, 1)};
}

// Rows read as they are when their elements are adjacent, else copied.
at::Tensor row_operand(const at::Tensor& X) {
  const bool ok = (X.stride(1) == 1 || X.size(1) <= 1) && (X.size(0) <= 1 || X.stride(0) >= X.size(1));
  return ok ? X : X.contiguous();
}

int64_t pitch(const at::Tensor& X) {
  return X.size(0) <= 1 ? std::max<int64_t>(X.size(1), 1) : std::max<int64_t>(X.stride(0), 1);
}

at::Tensor rows_out(const c10::optional<at::Tensor>& out, int64_t T, int64_t N, const at::Tensor& A) {
  if (!out.has_value()) return at::empty({T, N}, A.options().requires_grad(false));
  const at::Tensor& C = *out;
  TORCH_CHECK(C.is_cuda() && C.device() == A.device() && C.scalar_type() == A.scalar_type() && C.dim() == 2 &&
                  C.size(0) == T && C.size(1) == N && (C.stride(1) == 1 || N <= 1) && (T <= 1 || C.stride(0) >= N),
              "out must be a (T x N) tensor of the rows' dtype with unit column stride on their device");
  return C;
}

at::Tensor grouped_gemm(const at::Tensor& A, const at::Tensor& B, const at::Tensor& offsets,
                        c10::optional<at::Tensor> bias, int64_t act, c10::optional<at::Tensor> out) {
  TORCH_CHECK(A.is_cuda(), "A must be CUDA tensor");
  TORCH_CHECK(is_16bit(A), "A must be float16 or bfloat16");
  TORCH_CHECK(A.dim() == 2, "A must be 2D (T x K)");
  check_like(B, A, "B");
  TORCH_CHECK(B.dim() == 3, "B must be 3D (E x K x N)");
  TORCH_CHECK(A.size(1) == B.size(1), "Inner dimensions must match: A is (T x K), B is (E x K x N)");
  TORCH_CHECK(B.size(0) >= 1, "B must hold at least one group");
  check_index(offsets, A, B.size(0) + 1, "offsets");
  const int64_t T = A.size(0), K = A.size(1), E = B.size(0), N = B.size(2);
  at::Tensor bvec;
  if (bias.has_value()) {
    check_like(*bias, A, "bias");
    TORCH_CHECK(bias->dim() == 2 && bias->size(0) == E && bias->size(1) == N, "bias must be (E x N)");
    bvec = bias->contiguous();
  }
  check_no_grad("grouped_gemm computes no gradients: use grouped.grouped_linear, or call it under torch.no_grad()",
                {A, B, bvec, out.has_value() ? *out : at::Tensor()});
  const c10::cuda::CUDAGuard guard(A.device());
  at::Tensor As = row_operand(A), off = offsets.contiguous();
  auto [Bs, tb, ldb, sb] = stacked_operand(B);
  at::Tensor C = rows_out(out, T, N, A);
  if (out.has_value()) check_apart(C, {A, B, offsets, bias.value_or(at::Tensor())});
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(A.device().index()).stream();
  const int64_t lda = pitch(As);
  const at::Tensor ws = scratch(A.device(), gemm_grouped_workspace_bytes(As.data_ptr(), Bs.data_ptr(), T, N, K, E, lda,
                                                                         ldb, sb, tb));
  check_status(gemm_grouped_launch(As.data_ptr(), Bs.data_ptr(), C.data_ptr(), off.data_ptr(),
                                   off.scalar_type() == at::kLong ? 64 : 32, T, N, K, E, lda, ldb, sb,
                                   std::max<int64_t>(pitch(C), N), tb, bvec.defined() ? bvec.data_ptr() : nullptr,
                                   static_cast<int>(act), out.has_value() ? 0 : 1, dtype_id(A), scratch_ptr(ws), scratch_bytes(ws),
                                   stream),
               "gemm_grouped_launch");
  if (out.has_value()) count_write(C);
  return C;
}

at::Tensor grouped_gemm_wgrad(const at::Tensor& A, const at::Tensor& G, const at::Tensor& offsets,
                              c10::optional<at::Tensor> out) {
  TORCH_CHECK(A.is_cuda(), "A must be CUDA tensor");
  TORCH_CHECK(is_16bit(A), "A must be float16 or bfloat16");
  TORCH_CHECK(A.dim() == 2, "A must be 2D (T x K)");
  check_like(G, A, "G");
  TORCH_CHECK(G.dim() == 2 && G.size(0) == A.size(0), "G must be 2D (T x N) with A's rows");
  TORCH_CHECK(offsets.dim() == 1 && offsets.size(0) >= 2, "offsets must be 1D with at least 2 elements");
  check_index(offsets, A, offsets.size(0), "offsets");
  const int64_t T = A.size(0), K = A.size(1), N = G.size(1), E = offsets.size(0) - 1;
  check_no_grad("grouped_gemm_wgrad computes no gradients: call it under torch.no_grad()",
                {A, G, out.has_value() ? *out : at::Tensor()});
  const c10::cuda::CUDAGuard guard(A.device());
  at::Tensor D = out.has_value() ? *out : at::empty({E, K, N}, A.options().requires_grad(false));
  TORCH_CHECK(D.is_cuda() && D.device() == A.device() && D.scalar_type() == A.scalar_type() && D.dim() == 3 &&
                  D.size(0) == E && D.size(1) == K && D.size(2) == N,
              "out must be an (E x K x N) tensor of A's dtype on A's device");
  auto [Ds, td, ldd, sd] = stacked_operand(D);
  TORCH_CHECK(Ds.data_ptr() == D.data_ptr(), "out must be row-major or a transposed view, its matrices apart");
  at::Tensor As = row_operand(A), Gs = row_operand(G), off = offsets.contiguous();
  if (out.has_value()) check_apart(D, {A, G, offsets});
  // a gradient stored N x K is the product with the operands exchanged
  const at::Tensor &L = td ? Gs : As, &R = td ? As : Gs;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(A.device().index()).stream();
  const at::Tensor ws = scratch(A.device(), gemm_grouped_wgrad_workspace_bytes(L.data_ptr(), R.data_ptr(), T, L.size(1),
                                                                               R.size(1), pitch(L), pitch(R)));
  check_status(gemm_grouped_wgrad_launch(L.data_ptr(), R.data_ptr(), Ds.data_ptr(), off.data_ptr(),
                                         off.scalar_type() == at::kLong ? 64 : 32, T, L.size(1), R.size(1), E,
                                         pitch(L), pitch(R), ldd, sd, dtype_id(A), scratch_ptr(ws), scratch_bytes(ws), stream),
               "gemm_grouped_wgrad_launch");
  if (out.has_value()) count_write(D);
  return D;
}

// grouped_gemm as a differentiable function; grouped.py has the same in Python
// for builds without this module.  In C++ because a small step's cost is the
// work around its three launches.
struct GroupedLinear : public torch::autograd::Function<GroupedLinear> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                            const at::Tensor& offsets) {
    ctx->save_for_backward({x, weight, offsets});
    const at::NoGradGuard no_grad;
    return grouped_gemm(x, weight, offsets, c10::nullopt, GEMM_ACT_NONE, c10::nullopt);
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "grouped_linear can be differentiated once (no create_graph)");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &weight = saved[1], &offsets = saved[2], &dy = grads[0];
    at::Tensor dx, dw;
    if (dy.defined()) {
      if (ctx->needs_input_grad(0)) {
        dx = grouped_gemm(dy, weight.transpose(1, 2), offsets, c10::nullopt, GEMM_ACT_NONE, c10::nullopt);
      }
      if (ctx->needs_input_grad(1)) {
        c10::optional<at::Tensor> out;
        if (weight.stride(1) == 1 && weight.stride(2) != 1) {   // stored N x K: so is its gradient
          out = at::empty({weight.size(0), weight.size(2), weight.size(1)}, dy.options()).transpose(1, 2);
        }
        dw = grouped_gemm_wgrad(x, dy, offsets, out);
      }
    }
    return {dx, dw, at::Tensor()};
  }
};

at::Tensor grouped_linear(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& offsets) {
  return GroupedLinear::apply(x, weight, offsets);
}

at::Tensor lora_gemm(const at::Tensor& x, const at::Tensor& W, const at::Tensor& down, const at::Tensor& up,
                     const at::Tensor& adapter, c10::optional<at::Tensor> scale, c10::optional<at::Tensor> bias,
                     int64_t act, c10::optional<at::Tensor> out) {
  TORCH_CHECK(x.is_cuda(), "x must be CUDA tensor");
  TORCH_CHECK(is_16bit(x), "x must be float16 or bfloat16");
  TORCH_CHECK(x.dim() == 2, "x must be 2D (T x K)");
  check_like(W, x, "W");
  check_like(down, x, "down");
  check_like(up, x, "up");
  TORCH_CHECK(W.dim() == 2 && W.size(0) == x.size(1), "W must be 2D (K x N)");
  const int64_t T = x.size(0), K = x.size(1), N = W.size(1);
  TORCH_CHECK(down.dim() == 3 && down.size(1) == K, "down must be 3D (L x K x R)");
  const int64_t L = down.size(0), R = down.size(2);
  TORCH_CHECK(up.dim() == 3 && up.size(0) == L && up.size(1) == R && up.size(2) == N, "up must be 3D (L x R x N)");
  TORCH_CHECK(K >= 1 && L >= 1 && R >= 1, "K, the number of adapters and the rank must be at least 1");
  check_index(adapter, x, T, "adapter");
  at::Tensor svec, bvec;
  if (scale.has_value()) {
    svec = *scale;
    TORCH_CHECK(svec.is_cuda() && svec.device() == x.device() && svec.scalar_type() == at::kFloat && svec.dim() == 1 &&
                    svec.size(0) == L,
                "scale must be a float32 tensor of L elements on x's device");
    svec = svec.contiguous();
  }
  if (bias.has_value()) {
    check_like(*bias, x, "bias");
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == N, "bias must be (N)");
    bvec = bias->contiguous();
  }
  check_no_grad("lora_gemm is a serving operator and computes no gradients: call it under torch.no_grad()",
                {x, W, down, up, svec, bvec, out.has_value() ? *out : at::Tensor()});
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor xs = row_operand(x), ids = adapter.contiguous();
  auto [Ws, tw, ldw] = operand(W);
  auto [Ds, td, ldd, sd] = stacked_operand(down);
  auto [Us, tu, ldu, su] = stacked_operand(up);
  at::Tensor C = rows_out(out, T, N, x);
  if (out.has_value()) check_apart(C, {x, W, down, up, adapter, scale.value_or(at::Tensor()), bias.value_or(at::Tensor())});
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(x.device().index()).stream();
  const int64_t ldx = pitch(xs);
  const at::Tensor ws = scratch(x.device(), gemm_lora_workspace_bytes(xs.data_ptr(), Ws.data_ptr(), Us.data_ptr(), T, N,
                                                                      K, L, R, ldx, ldw, tw, ldu, su, tu));
  check_status(gemm_lora_launch(xs.data_ptr(), Ws.data_ptr(), Ds.data_ptr(), Us.data_ptr(), C.data_ptr(),
                                ids.data_ptr(), ids.scalar_type() == at::kLong ? 64 : 32, T, N, K, L, R, ldx, ldw, tw,
                                ldd, sd, td, ldu, su, tu, std::max<int64_t>(pitch(C), N),
                                svec.defined() ? svec.data_ptr<float>() : nullptr,
                                bvec.defined() ? bvec.data_ptr() : nullptr, static_cast<int>(act), dtype_id(x), scratch_ptr(ws),
                                scratch_bytes(ws), stream),
               "gemm_lora_launch");
  if (out.has_value()) count_write(C);
  return C;
}

void reset_workspaces() {
  std::lock_guard<std::mutex> lock(g_ws_mu);
  g_ws->clear();
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "torch binding of the sm_100a FP16 GEMM kernel bank (C ABI in gemm_sm100.h)";
  m.def("gemm_forward_cfg", &gemm_forward_cfg, "C = A @ B with menu configuration cfg_id", py::arg("A"),
        py::arg("B"), py::arg("cfg_id"), py::arg("out") = py::none());
  m.def("gemm_ex", &gemm_ex, "out = act(alpha * A @ B + beta * C + bias)", py::arg("A"), py::arg("B"),
        py::arg("cfg_id"), py::arg("alpha") = 1.0, py::arg("beta") = 0.0, py::arg("C") = py::none(),
        py::arg("bias") = py::none(), py::arg("act") = 0, py::arg("out") = py::none());
  m.def("grouped_gemm", &grouped_gemm, "out[r] = act(A[r] @ B[group of r] + bias[group of r])", py::arg("A"),
        py::arg("B"), py::arg("offsets"), py::arg("bias") = py::none(), py::arg("act") = 0,
        py::arg("out") = py::none());
  m.def("grouped_gemm_wgrad", &grouped_gemm_wgrad, "out[e] = A[rows of e].T @ G[rows of e]", py::arg("A"),
        py::arg("G"), py::arg("offsets"), py::arg("out") = py::none());
  m.def("grouped_linear", &grouped_linear, "grouped_gemm, differentiable in x and weight", py::arg("x"),
        py::arg("weight"), py::arg("offsets"));
  m.def("lora_gemm", &lora_gemm, "out[t] = act(x[t] @ W + scale[a] * (x[t] @ down[a]) @ up[a] + bias), a = adapter[t]",
        py::arg("x"), py::arg("W"), py::arg("down"), py::arg("up"), py::arg("adapter"), py::arg("scale") = py::none(),
        py::arg("bias") = py::none(), py::arg("act") = 0, py::arg("out") = py::none());
  m.def("reset_workspaces", &reset_workspaces, "drop the cached split-K / repack workspaces");
}
