// The 8-bit blocks' and the embedding's operators (block_fp8.py, embed.py, which
// declare them) from torch to the C ABI: checks of what the kernels assume,
// allocations and launches on the current stream of the operands' device; and
// behind them the eager calls of the public functions, with C++ autograd nodes,
// which return None where a call is not a plain one (the Python layer then checks it
// and goes through its own nodes).  A step of 64 rows of 528 by 1000 weights, fp16,
// takes the host 48 us, 18 of them torch's own for any gradient.
#include <torch/library.h>

#include <ATen/hip/EmptyTensor.h>

#include "kd_torch.h"

namespace {

using namespace kdt;
using torch::autograd::Function;

int dtype_code(at::ScalarType t, bool f32) {
  if (t == at::kBFloat16) return KD_BF16;
  if (t == at::kHalf) return KD_F16;
  TORCH_CHECK_VALUE(f32 && t == at::kFloat, "the type must be bf16", f32 ? ", fp16 or fp32" : " or fp16", ", got ", t);
  return KD_F32;
}

void on_one_gpu(std::initializer_list<const Tensor*> ts) {
  const Tensor& first = **ts.begin();
  TORCH_CHECK_VALUE(first.is_cuda(), "the tensors must be on a GPU (no CPU fallback)");
  for (const Tensor* t : ts) TORCH_CHECK_VALUE(t->device() == first.device(), "the tensors must be on the same GPU");
}

bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
Tensor flat(const Tensor& t) {  // contiguous from a 16-byte boundary on
  const Tensor c = t.contiguous();
  return aligned16(c) ? c : c.clone();
}
Tensor rows_ready(const Tensor& t) {  // [rows, cols], rows a multiple of 8 elements apart from such a boundary on
  TORCH_CHECK_VALUE(t.dim() == 2, "a matrix is expected, got ", t.dim(), " dimensions");
  return t.stride(1) == 1 && t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) && aligned16(t) ? t : flat(t);
}

// New memory on t's device (not through the dispatcher, which takes longer than the allocator)
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& t) {
  return Tensor(at::detail::empty_cuda(sizes, type, t.device(), std::nullopt));
}

int64_t blocks(int64_t n) { return (n + 127) / 128; }
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
Tensor bytes8(const Tensor& like, int64_t rows, int64_t cols) {
  return fresh({rows, up16(cols)}, at::kFloat8_e4m3fn, like);
}
Tensor scales(const Tensor& like, int64_t rows, int64_t nb) {
  return fresh({rows, nb}, at::kFloat8_e8m0fnu, like);
}
uint8_t* u8(const Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }

// e4m3 rows with their scales: of `cols` columns, one scale row per `per` rows
void check_blocks(const Tensor& y, const Tensor& scale, int64_t cols, int64_t per, const char* what) {
  TORCH_CHECK_VALUE(y.dim() == 2 && scale.dim() == 2, what, ": values and scales must be matrices");
  TORCH_CHECK_VALUE(y.scalar_type() == at::kFloat8_e4m3fn && scale.scalar_type() == at::kFloat8_e8m0fnu, what,
                    ": values must be float8_e4m3fn and scales float8_e8m0fnu, got ", y.scalar_type(), " and ",
                    scale.scalar_type());
  TORCH_CHECK_VALUE(y.size(1) >= cols && scale.size(0) == (y.size(0) + per - 1) / per && scale.size(1) == blocks(cols), what,
                    ": scales of ", y.sizes(), " in blocks of ", per, " x 128 must be [", (y.size(0) + per - 1) / per, ", ",
                    blocks(cols), "], got ", scale.sizes());
  TORCH_CHECK_VALUE(scale.is_contiguous() && y.stride(1) == 1 && y.stride(0) % 16 == 0 && y.stride(0) >= up16(cols) &&
                        aligned16(y),
                    what, ": values must lie in rows a multiple of 16 bytes apart, scales contiguous");
}
int32_t size32(int64_t n) {
  TORCH_CHECK_VALUE(n < (int64_t(1) << 31), "sizes must be < 2^31, got ", n);
  return int32_t(n);
}
// the blocks' values as the kernel reads them
Tensor blocks_ready(const Tensor& y) {
  return y.dim() == 2 && y.stride(1) == 1 && y.stride(0) % 16 == 0 && y.stride(0) >= y.size(1) && aligned16(y) ? y : flat(y);
}

std::tuple<Tensor, Tensor> quant_rows8(at::TensorList xs) {
  TORCH_CHECK_VALUE(!xs.empty() && xs.size() <= 4, "1 to 4 parts are expected");
  kd_rows8_args a{};
  std::vector<Tensor> keep;
  int64_t total = 0;
  for (const Tensor& x : xs) {
    on_one_gpu({&xs[0], &x});
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(0) == xs[0].size(0) && x.scalar_type() == xs[0].scalar_type(),
                      "the parts must be matrices of one type and one number of rows");
    keep.push_back(rows_ready(x));
    a.x[a.n] = keep.back().data_ptr(), a.x_stride[a.n] = keep.back().stride(0), a.cols[a.n] = size32(x.size(1)), ++a.n;
    total += x.size(1);
  }
  const c10::DeviceGuard on(xs[0].device());
  a.dtype = dtype_code(xs[0].scalar_type(), true);
  a.rows = xs[0].size(0), a.total = size32(total);
  Tensor y = bytes8(xs[0], a.rows, total), s = scales(xs[0], a.rows, blocks(total));
  if (a.rows == 0) return {y, s};
  a.y = u8(y), a.y_stride = y.stride(0), a.scale = u8(s);
  check(kd_quant_rows8(&a, stream_of(y)), "kd_quant_rows8");
  return {y, s};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> quant_weight8(at::TensorList ws, bool transpose) {
  TORCH_CHECK_VALUE(!ws.empty() && ws.size() <= 4, "1 to 4 parts are expected");
  kd_weight8_args a{};
  std::vector<Tensor> keep;
  int64_t total = 0;
  for (const Tensor& w : ws) {
    on_one_gpu({&ws[0], &w});
    TORCH_CHECK_VALUE(w.dim() == 2 && w.size(1) == ws[0].size(1) && w.scalar_type() == ws[0].scalar_type(),
                      "the parts must be matrices of one type and one number of columns");
    keep.push_back(rows_ready(w));
    a.w[a.n] = keep.back().data_ptr(), a.w_stride[a.n] = keep.back().stride(0), a.rows[a.n] = size32(w.size(0)), ++a.n;
    total += w.size(0);
  }
  const c10::DeviceGuard on(ws[0].device());
  const int64_t K = ws[0].size(1);
  a.dtype = dtype_code(ws[0].scalar_type(), true), a.K = size32(K), a.total = size32(total);
  Tensor y = bytes8(ws[0], total, K), s = scales(ws[0], blocks(total), blocks(K));
  Tensor yt = transpose ? bytes8(ws[0], K, total) : bytes8(ws[0], 0, 0);
  Tensor st = transpose ? scales(ws[0], blocks(K), blocks(total)) : scales(ws[0], 0, 0);
  a.y = u8(y), a.y_stride = y.stride(0), a.scale = u8(s);
  if (transpose) a.yt = u8(yt), a.yt_stride = yt.stride(0), a.scale_t = u8(st);
  check(kd_quant_weight8(&a, stream_of(y)), "kd_quant_weight8");
  return {y, s, yt, st};
}

Tensor matmul8(const Tensor& a_in, const Tensor& a_scale, const Tensor& b_in, const Tensor& b_scale, at::ScalarType out_type,
               bool fast) {
  on_one_gpu({&a_in, &a_scale, &b_in, &b_scale});
  const Tensor a = blocks_ready(a_in), b = blocks_ready(b_in);
  const Tensor as = a_scale.contiguous(), bs = b_scale.contiguous();
  const c10::DeviceGuard on(a.device());
  TORCH_CHECK_VALUE(a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(1), "a [M, K] and b [N, K] expected, got ", a.sizes(),
                    " and ", b.sizes());
  const int64_t M = a.size(0), N = b.size(0), K = a.size(1);
  check_blocks(a, as, K, 1, "a"), check_blocks(b, bs, K, 128, "b");
  kd_matmul8_args g{};
  g.dtype = dtype_code(out_type, true), g.fast = fast;
  Tensor out = fresh({M, N}, out_type, a);
  if (out.numel() == 0) return out;
  g.a = u8(a), g.b = u8(b), g.lda = a.stride(0), g.ldb = b.stride(0), g.a_scale = u8(as), g.b_scale = u8(bs);
  g.out = out.data_ptr(), g.ldo = N;
  g.M = size32(M), g.N = size32(N), g.K = size32(K);
  check(kd_matmul8(&g, stream_of(out)), "kd_matmul8");
  return out;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> norm8(const Tensor& x_in, const OptTensor& delta, double eps) {
  on_one_gpu({&x_in});
  TORCH_CHECK_VALUE(x_in.dim() == 2, "x must be a matrix");
  const c10::DeviceGuard on(x_in.device());
  const Tensor x = flat(x_in);
  Tensor d, sum;
  kd_norm8_args a{};
  a.dtype = dtype_code(x.scalar_type(), false);
  a.rows = x.size(0), a.D = size32(x.size(1)), a.eps = float(eps);
  if (delta) {
    on_one_gpu({&x, &*delta});
    TORCH_CHECK_VALUE(delta->sizes() == x.sizes() && delta->scalar_type() == x.scalar_type(),
                      "x and delta must have one shape and type");
    d = flat(*delta), sum = fresh(x.sizes(), x.scalar_type(), x);
    a.delta = d.data_ptr(), a.sum = sum.data_ptr();
  }
  Tensor y = bytes8(x, a.rows, a.D), s = scales(x, a.rows, blocks(a.D)), rstd = fresh({a.rows}, at::kFloat, x);
  if (!delta) sum = fresh({0}, x.scalar_type(), x);
  if (a.rows == 0) return {sum, y, s, rstd};
  a.x = x.data_ptr(), a.y = u8(y), a.y_stride = y.stride(0), a.scale = u8(s), a.rstd = static_cast<float*>(rstd.data_ptr());
  check(kd_norm8(&a, stream_of(x)), "kd_norm8");
  return {sum, y, s, rstd};
}

Tensor norm8_bwd(const Tensor& g_in, const OptTensor& ds, const Tensor& y, const Tensor& scale, const Tensor& rstd,
                 at::ScalarType dtype) {
  on_one_gpu({&g_in, &y, &scale, &rstd});
  TORCH_CHECK_VALUE(g_in.dim() == 2 && y.dim() == 2 && y.size(0) == g_in.size(0) && rstd.numel() == g_in.size(0) &&
                        rstd.scalar_type() == at::kFloat && rstd.is_contiguous(),
                    "g [rows, D], y [rows, D] and rstd [rows] expected");
  check_blocks(y, scale, g_in.size(1), 1, "y");
  const c10::DeviceGuard on(g_in.device());
  const Tensor g = flat(g_in);
  Tensor d;
  if (ds) {
    on_one_gpu({&g, &*ds});
    TORCH_CHECK_VALUE(ds->sizes() == g.sizes() && ds->scalar_type() == dtype, "ds must have g's shape and the result's type");
    d = flat(*ds);
  }
  kd_norm8_bwd_args a{};
  a.dtype = dtype_code(dtype, false), a.g_dtype = dtype_code(g.scalar_type(), true);
  Tensor dx = fresh(g.sizes(), dtype, g);
  a.rows = g.size(0), a.D = size32(g.size(1));
  if (a.rows == 0) return dx;
  a.g = g.data_ptr(), a.ds = ds ? d.data_ptr() : nullptr, a.y = u8(y), a.y_stride = y.stride(0), a.scale = u8(scale);
  a.rstd = static_cast<const float*>(rstd.data_ptr()), a.dx = dx.data_ptr();
  check(kd_norm8_bwd(&a, stream_of(g)), "kd_norm8_bwd");
  return dx;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> gate8(const Tensor& a_in, const Tensor& b_in, bool keep) {
  on_one_gpu({&a_in, &b_in});
  TORCH_CHECK_VALUE(a_in.sizes() == b_in.sizes() && a_in.scalar_type() == b_in.scalar_type(), "a and b must have one shape and type");
  const c10::DeviceGuard on(a_in.device());
  const Tensor a = rows_ready(a_in), b = rows_ready(b_in);
  kd_gate8_args g{};
  g.dtype = dtype_code(a.scalar_type(), false);
  g.rows = a.size(0), g.H = size32(a.size(1));
  const int64_t kept = keep ? g.rows : 0, nb = blocks(g.H);
  Tensor y = bytes8(a, g.rows, g.H), ys = scales(a, g.rows, nb);
  Tensor a8 = bytes8(a, kept, g.H), as = scales(a, kept, nb), b8 = bytes8(a, kept, g.H), bs = scales(a, kept, nb);
  if (g.rows == 0) return {y, ys, a8, as, b8, bs};
  g.a = a.data_ptr(), g.a_stride = a.stride(0), g.b = b.data_ptr(), g.b_stride = b.stride(0);
  g.y8 = u8(y), g.y_scale = u8(ys), g.stride = y.stride(0);
  if (keep) g.a8 = u8(a8), g.a_scale = u8(as), g.b8 = u8(b8), g.b_scale = u8(bs);
  check(kd_gate8(&g, stream_of(a)), "kd_gate8");
  return {y, ys, a8, as, b8, bs};
}

std::tuple<Tensor, Tensor> gate8_bwd(const Tensor& dy_in, const Tensor& a8, const Tensor& as, const Tensor& b8, const Tensor& bs,
                                     at::ScalarType dtype) {
  on_one_gpu({&dy_in, &a8, &as, &b8, &bs});
  TORCH_CHECK_VALUE(dy_in.dim() == 2 && a8.size(0) == dy_in.size(0) && b8.sizes() == a8.sizes() && b8.strides() == a8.strides(),
                    "dy, a and b must have one number of rows");
  check_blocks(a8, as, dy_in.size(1), 1, "a"), check_blocks(b8, bs, dy_in.size(1), 1, "b");
  const c10::DeviceGuard on(dy_in.device());
  const Tensor dy = flat(dy_in);
  Tensor da = fresh(dy.sizes(), dtype, dy), db = fresh(dy.sizes(), dtype, dy);
  kd_gate8_args g{};
  g.dtype = dtype_code(dtype, false), g.dy_dtype = dtype_code(dy.scalar_type(), true);
  g.rows = dy.size(0), g.H = size32(dy.size(1));
  if (g.rows == 0) return {da, db};
  g.dy = dy.data_ptr(), g.da = da.data_ptr(), g.db = db.data_ptr(), g.stride = a8.stride(0);
  g.a8 = u8(a8), g.a_scale = u8(as), g.b8 = u8(b8), g.b_scale = u8(bs);
  check(kd_gate8_bwd(&g, stream_of(dy)), "kd_gate8_bwd");
  return {da, db};
}

// The parts of dy, stacked, transposed, times the `K` columns that x8 holds
Tensor weight_grad8(at::TensorList dys, const Tensor& x, const Tensor& x_scale, int64_t K) {
  TORCH_CHECK_VALUE(!dys.empty() && dys.size() <= 4, "1 to 4 parts are expected");
  on_one_gpu({&dys[0], &x, &x_scale});
  const c10::DeviceGuard on(x.device());
  kd_wgrad8_args g{};
  std::vector<Tensor> keep;
  int64_t N = 0;
  for (const Tensor& d : dys) {
    on_one_gpu({&x, &d});
    keep.push_back(rows_ready(d));
    const Tensor& dy = keep.back();
    TORCH_CHECK_VALUE(x.dim() == 2 && x.size(0) == dy.size(0) && dy.scalar_type() == dys[0].scalar_type(),
                      "dy [M, N] of one type and x [M, K] expected, got ", dy.sizes(), " and ", x.sizes());
    g.dy[g.n] = dy.data_ptr(), g.ldy[g.n] = dy.stride(0), g.cols[g.n] = size32(dy.size(1)), ++g.n;
    N += dy.size(1);
  }
  check_blocks(x, x_scale, K, 1, "x");
  const int64_t M = x.size(0);
  g.dtype = dtype_code(dys[0].scalar_type(), false);
  if (M == 0) return at::zeros({N, K}, dys[0].options());
  Tensor dw = fresh({N, K}, dys[0].scalar_type(), x);
  g.M = size32(M), g.N = size32(N), g.K = size32(K);
  g.ws_bytes = kd_weight_grad8_ws_bytes(g.M, g.N, g.K, g.dtype);
  check(g.ws_bytes < 0 ? KD_ERR_UNSUPPORTED : KD_OK, "kd_weight_grad8");
  const Tensor ws = fresh({g.ws_bytes}, at::kByte, x);
  g.x = u8(x), g.ldx = x.stride(0), g.x_scale = u8(x_scale);
  g.dw = dw.data_ptr(), g.ws = static_cast<float*>(ws.data_ptr());
  check(kd_weight_grad8(&g, stream_of(x)), "kd_weight_grad8");
  return dw;
}

kd_embed_args embed_args(const Tensor& tokens, int64_t vocab, int64_t dim, at::ScalarType type, double scale) {
  TORCH_CHECK_VALUE(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt, "tokens must be int64 or int32, got ",
                    tokens.scalar_type());
  kd_embed_args a{};
  a.tokens = tokens.data_ptr(), a.n = tokens.numel(), a.tokens_dtype = tokens.scalar_type() == at::kLong ? KD_I64 : KD_I32;
  a.vocab = vocab, a.dim = dim, a.dtype = dtype_code(type, true), a.scale = float(scale), a.padding_idx = -1;
  return a;
}

Tensor embed(const Tensor& tokens_in, const Tensor& weight_in, double scale) {
  on_one_gpu({&weight_in, &tokens_in});
  TORCH_CHECK_VALUE(weight_in.dim() == 2, "weight must be [vocab, dim]");
  const c10::DeviceGuard on(weight_in.device());
  const Tensor tokens = tokens_in.contiguous(), weight = weight_in.contiguous();
  auto shape = tokens_in.sizes().vec();
  shape.push_back(weight.size(1));
  Tensor out = fresh(shape, weight.scalar_type(), weight);
  kd_embed_args a = embed_args(tokens, weight.size(0), weight.size(1), weight.scalar_type(), scale);
  if (out.numel() == 0) return out;
  a.weight = weight.data_ptr(), a.out = out.data_ptr();
  check(kd_embed(&a, stream_of(out)), "kd_embed");
  return out;
}

Tensor embed_grad(const Tensor& tokens_in, const Tensor& dy_in, int64_t vocab, double scale, int64_t padding_idx) {
  on_one_gpu({&dy_in, &tokens_in});
  const c10::DeviceGuard on(dy_in.device());
  const Tensor tokens = tokens_in.contiguous(), dy = dy_in.contiguous();
  const int64_t dim = dy.size(-1);
  TORCH_CHECK_VALUE(dy.dim() >= 1 && tokens.numel() * dim == dy.numel(), "dy must be tokens' shape by dim");
  kd_embed_args a = embed_args(tokens, vocab, dim, dy.scalar_type(), scale);
  if (dy.numel() == 0) return at::zeros({vocab, dim}, dy.options());
  Tensor dw = fresh({vocab, dim}, dy.scalar_type(), dy);
  const int64_t need = kd_embed_grad_ws_bytes(a.n, vocab, dim);
  const Tensor ws = fresh({std::max<int64_t>(need, 0)}, at::kByte, dy);
  a.dy = dy.data_ptr(), a.dw = dw.data_ptr(), a.padding_idx = padding_idx;
  check(kd_embed_grad(&a, ws.data_ptr(), need, stream_of(dy)), "kd_embed_grad");
  return dw;
}

// ------------------------------------------------------------ eager calls
// The operators through the dispatcher, for cotangents of any kind
template <class F>
auto op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
bool half(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }
bool plain_call(std::initializer_list<const Tensor*> ts) {
  if (!plain_mode()) return false;
  for (const Tensor* t : ts)
    if (!plain(*t) || t->device() != (*ts.begin())->device()) return false;
  return true;
}
std::vector<int64_t> with_last(const Tensor& like, int64_t last) {
  auto shape = like.sizes().vec();
  shape.back() = last;
  return shape;
}
Tensor as_rows(const Tensor& t) { return t.dim() == 2 ? t : t.reshape({-1, t.size(-1)}); }

bool weights_fit(const Tensor& x, at::TensorList ws) {
  if (ws.empty() || ws.size() > 4) return false;
  for (const Tensor& w : ws)
    if (!plain(w) || w.dim() != 2 || w.size(1) != x.size(-1) || w.size(0) < 8 || w.size(0) % 8 != 0 ||
        w.scalar_type() != x.scalar_type() || w.device() != x.device())
      return false;
  return true;
}
// Parts that the kernels take side by side: whole blocks, or one part
std::vector<Tensor> stacked(at::TensorList parts, int64_t dim) {
  bool whole = true;
  for (size_t i = 0; i + 1 < parts.size(); ++i) whole &= parts[i].size(dim) % 128 == 0;
  return whole ? parts.vec() : std::vector<Tensor>{at::cat(parts, dim)};
}

// Whether a backward may call the kernels past the dispatcher (some 3 us a call): plain
// cotangents, no mode that has to see operations, no graph of the backward itself
bool direct(at::TensorList ds) {
  if (!no_dispatch() || at::GradMode::is_enabled()) return false;
  for (const Tensor& d : ds)
    if (!plain(d)) return false;
  return true;
}

// The backward's products (block_fp8._backward_products): the operand's gradient
// from the gradients' blocks and the weights', the weights' from the kept operand
std::pair<Tensor, Tensor> backward_products(const std::vector<Tensor>& dys, const Tensor& x8, const Tensor& xs, const Tensor& wt,
                                            const Tensor& wts, bool want_x, bool want_w, int64_t K, at::ScalarType between) {
  static const auto quant = op<std::tuple<Tensor, Tensor>(at::TensorList)>("kdattn::quant_rows8");
  static const auto product =
      op<Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, at::ScalarType, bool)>("kdattn::matmul8");
  static const auto wgrad = op<Tensor(at::TensorList, const Tensor&, const Tensor&, int64_t)>("kdattn::weight_grad8");
  const std::vector<Tensor> parts = stacked(dys, 1);
  Tensor dx, dw;
  if (direct(parts)) {
    at::AutoDispatchBelowADInplaceOrView below;
    if (want_x) {
      const auto [d8, ds] = quant_rows8(parts);
      dx = matmul8(d8, ds, wt, wts, between, true);
    }
    if (want_w) dw = weight_grad8(parts, x8, xs, K);
    return {dx, dw};
  }
  if (want_x) {
    const auto [d8, ds] = quant.call(parts);
    dx = product.call(d8, ds, wt, wts, between, true);
  }
  if (want_w) dw = wgrad.call(parts, x8, xs, K);
  return {dx, dw};
}
at::ScalarType between(at::ScalarType t) { return t == at::kHalf ? at::kFloat : t; }  // (block_fp8._between)

// Under create_graph the results have a history that raises when it is gone back through
variable_list once(variable_list out, const char* name, const variable_list& from) {
  if (!at::GradMode::is_enabled()) return out;
  bool any = false;
  for (const Tensor& t : from) any |= t.defined() && t.requires_grad();
  if (!any) return out;
  variable_list given, made;
  for (const Tensor& t : from)
    if (t.defined()) given.push_back(t);
  for (Tensor& t : out)
    if (t.defined()) t = t.detach(), made.push_back(t);
  refuse_second(made, name, given);
  return out;
}

struct NormProjectionNode : Function<NormProjectionNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& delta, at::TensorList ws, double eps,
                               bool want_x) {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard on(x.device());
    const int64_t K = x.size(-1);
    const auto [s, y8, ys, rstd] = norm8(as_rows(x), delta ? OptTensor(as_rows(*delta)) : OptTensor(), eps);
    const auto [w8, wsc, wt, wts] = quant_weight8(stacked(ws, 0), want_x);
    const Tensor y = matmul8(y8, ys, w8, wsc, x.scalar_type(), false);
    variable_list out;
    if (delta) out.push_back(s.view(x.sizes()));
    std::vector<int64_t> widths;
    int64_t at = 0;
    for (const Tensor& w : ws) {
      const int64_t n = w.size(0);
      const Tensor part = y.narrow(1, at, n);
      out.push_back(x.dim() == 2 ? part : part.view(with_last(x, n)));
      widths.push_back(n), at += n;
    }
    ctx->save_for_backward({y8, ys, rstd, wt, wts});
    ctx->saved_data["widths"] = widths;
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["type"] = int64_t(x.scalar_type());
    ctx->saved_data["delta"] = delta.has_value();
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const bool has = ctx->saved_data["delta"].toBool();
    const std::vector<int64_t> widths = ctx->saved_data["widths"].toIntVector(), shape = ctx->saved_data["shape"].toIntVector();
    const auto type = at::ScalarType(ctx->saved_data["type"].toInt());
    const size_t n = widths.size(), nx = has ? 2 : 1;
    variable_list out(2 + n + 2);
    const bool want_x = ctx->needs_input_grad(0), want_d = has && ctx->needs_input_grad(1);
    const Tensor dsum = has ? grads[0] : Tensor();
    Tensor given;
    for (size_t i = 0; i < n; ++i)
      if (grads[i + has].defined()) given = grads[i + has];
    if (!given.defined()) {  // the products did not reach the loss
      if (want_x) out[0] = dsum;
      if (want_d) out[1] = dsum;
      return out;
    }
    const variable_list s = ctx->get_saved_variables();
    const c10::DeviceGuard on(s[0].device());
    const int64_t rows = s[0].size(0), K = shape.back();
    std::vector<Tensor> dys;
    bool want_w = false;
    for (size_t i = 0; i < n; ++i) {
      const Tensor& d = grads[i + has];
      dys.push_back(d.defined() ? d.reshape({rows, widths[i]}) : at::zeros({rows, widths[i]}, given.options()));
      want_w |= ctx->needs_input_grad(nx + i);
    }
    auto [g, dw] = backward_products(dys, s[0], s[1], s[3], s[4], want_x || want_d, want_w, K, between(type));
    if (want_x || want_d) {
      static const auto norm =
          op<Tensor(const Tensor&, const OptTensor&, const Tensor&, const Tensor&, const Tensor&, at::ScalarType)>("kdattn::norm8_bwd");
      const Tensor dx =
          norm.call(g, dsum.defined() ? OptTensor(dsum.reshape({rows, K})) : OptTensor(), s[0], s[1], s[2], type).view(shape);
      if (want_x) out[0] = dx;
      if (want_d) out[1] = dx;
    }
    int64_t at = 0;
    for (size_t i = 0; i < n; ++i) {
      if (ctx->needs_input_grad(nx + i)) out[2 + i] = dw.narrow(0, at, widths[i]);
      at += widths[i];
    }
    return once(std::move(out), "norm_projection", grads);
  }
};

struct ProjectionNode : Function<ProjectionNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, bool want_x) {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard on(x.device());
    const auto [x8, xs] = quant_rows8({as_rows(x)});
    const auto [w8, ws, wt, wts] = quant_weight8({w}, want_x);
    const Tensor y = matmul8(x8, xs, w8, ws, x.scalar_type(), false);
    ctx->save_for_backward({x8, xs, wt, wts});
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["type"] = int64_t(x.scalar_type());
    return x.dim() == 2 ? y : y.view(with_last(x, w.size(0)));
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list s = ctx->get_saved_variables();
    const c10::DeviceGuard on(s[0].device());
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    const auto [dx, dw] = backward_products({as_rows(grads[0])}, s[0], s[1], s[2], s[3], ctx->needs_input_grad(0),
                                            ctx->needs_input_grad(1), shape.back(), at::ScalarType(ctx->saved_data["type"].toInt()));
    return once({dx.defined() ? dx.view(shape) : dx, dw, Tensor()}, "fp8_projection", grads);
  }
};

struct SwigluProjectionNode : Function<SwigluProjectionNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& a, const Tensor& b, const Tensor& w, bool want) {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard on(a.device());
    const auto [y8, ys, a8, as, b8, bs] = gate8(as_rows(a), as_rows(b), want);
    const auto [w8, ws, wt, wts] = quant_weight8({w}, want);
    const Tensor y = matmul8(y8, ys, w8, ws, a.scalar_type(), false);
    ctx->save_for_backward({y8, ys, a8, as, b8, bs, wt, wts});
    ctx->saved_data["shape"] = a.sizes().vec();
    ctx->saved_data["type"] = int64_t(a.scalar_type());
    return a.dim() == 2 ? y : y.view(with_last(a, w.size(0)));
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    static const auto gate = op<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                           at::ScalarType)>("kdattn::gate8_bwd");
    const variable_list s = ctx->get_saved_variables();
    const c10::DeviceGuard on(s[0].device());
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    const auto type = at::ScalarType(ctx->saved_data["type"].toInt());
    const bool want_a = ctx->needs_input_grad(0), want_b = ctx->needs_input_grad(1);
    const auto [g, dw] = backward_products({as_rows(grads[0])}, s[0], s[1], s[6], s[7], want_a || want_b, ctx->needs_input_grad(2),
                                           shape.back(), between(type));
    Tensor da, db;
    if (want_a || want_b) std::tie(da, db) = gate.call(g, s[2], s[3], s[4], s[5], type);
    return once({want_a ? da.view(shape) : Tensor(), want_b ? db.view(shape) : Tensor(), dw, Tensor()}, "swiglu_projection", grads);
  }
};

struct EmbeddingNode : Function<EmbeddingNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& tokens, double scale, int64_t padding_idx) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({tokens});
    ctx->saved_data["vocab"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["pad"] = padding_idx;
    return embed(tokens, weight, scale);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    static const auto grad = op<Tensor(const Tensor&, const Tensor&, c10::SymInt, double, int64_t)>("kdattn::embed_grad");
    const Tensor tokens = ctx->get_saved_variables()[0];
    const int64_t vocab = ctx->saved_data["vocab"].toInt(), pad = ctx->saved_data["pad"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    Tensor dw;
    if (direct(grads) && plain(tokens)) {
      at::AutoDispatchBelowADInplaceOrView below;
      dw = embed_grad(tokens, grads[0], vocab, scale, pad);
    } else {
      dw = grad.call(tokens, grads[0], vocab, scale, pad);
    }
    return once({dw, Tensor(), Tensor(), Tensor()}, "embedding", grads);
  }
};

bool wants(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }

pybind11::object eager_quantize_rows(const Tensor& x) {
  if (!plain_call({&x}) || x.dim() < 1 || x.numel() == 0 || x.size(-1) % 16 != 0 || !(half(x) || x.scalar_type() == at::kFloat))
    return pybind11::none();
  at::AutoDispatchBelowADInplaceOrView below;
  const auto [y, s] = quant_rows8({as_rows(x)});
  return pybind11::make_tuple(x.dim() == 2 ? y : y.view(x.sizes()), x.dim() == 2 ? s : s.view(with_last(x, s.size(1))));
}

pybind11::object eager_matmul(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale, at::ScalarType type) {
  if (!plain_call({&a, &a_scale, &b, &b_scale}) || a.dim() < 1 || b.dim() != 2 || a.numel() == 0 || b.numel() == 0 ||
      a.size(-1) % 16 != 0 || a.size(-1) != b.size(1) || a.scalar_type() != at::kFloat8_e4m3fn ||
      b.scalar_type() != at::kFloat8_e4m3fn || a_scale.scalar_type() != at::kFloat8_e8m0fnu ||
      b_scale.scalar_type() != at::kFloat8_e8m0fnu || a_scale.dim() != a.dim() || b_scale.dim() != 2 ||
      a_scale.size(-1) != blocks(a.size(-1)) || a_scale.sizes().slice(0, a.dim() - 1) != a.sizes().slice(0, a.dim() - 1) ||
      b_scale.size(1) != a_scale.size(-1) || b_scale.size(0) != blocks(b.size(0)) ||
      !(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat))
    return pybind11::none();
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor y = matmul8(as_rows(a), as_rows(a_scale), b, b_scale, type, false);
  return pybind11::cast(a.dim() == 2 ? y : y.view(with_last(a, b.size(0))));
}

bool norm_fits(const Tensor& x, const OptTensor& delta, int64_t of) {
  return plain_call({&x}) && half(x) && x.dim() >= 1 && x.numel() > 0 && x.size(-1) % of == 0 && x.size(-1) <= 8192 &&
         (!delta || (plain(*delta) && delta->sizes() == x.sizes() && delta->scalar_type() == x.scalar_type() &&
                     delta->device() == x.device()));
}

pybind11::object eager_norm(const Tensor& x, const OptTensor& delta, double eps) {
  if (!norm_fits(x, delta, 16)) return pybind11::none();
  at::AutoDispatchBelowADInplaceOrView below;
  const auto [s, y, scale, rstd] = norm8(as_rows(x), delta ? OptTensor(as_rows(*delta)) : OptTensor(), eps);
  if (x.dim() == 2) return pybind11::make_tuple(delta ? s : x, y, scale);
  return pybind11::make_tuple(delta ? s.view(x.sizes()) : x, y.view(x.sizes()), scale.view(with_last(x, scale.size(1))));
}

pybind11::object eager_norm_projection(const Tensor& x, const OptTensor& delta, const std::vector<Tensor>& ws, double eps) {
  if (!norm_fits(x, delta, 8) || !weights_fit(x, ws)) return pybind11::none();
  variable_list out = NormProjectionNode::apply(x, delta, at::TensorList(ws), eps, wants(x) || (delta && wants(*delta)));
  if (!delta) out.insert(out.begin(), x);
  return pybind11::cast(out);
}

pybind11::object eager_projection(const Tensor& x, const Tensor& w) {
  if (!plain_call({&x}) || !half(x) || x.dim() < 1 || x.numel() == 0 || x.size(-1) % 8 != 0 || !weights_fit(x, w)) return pybind11::none();
  return pybind11::cast(ProjectionNode::apply(x, w, wants(x)));
}

pybind11::object eager_swiglu_projection(const Tensor& a, const Tensor& b, const Tensor& w) {
  if (!plain_call({&a, &b}) || !half(a) || a.dim() < 1 || a.numel() == 0 || a.size(-1) % 8 != 0 || b.sizes() != a.sizes() ||
      b.scalar_type() != a.scalar_type() || !weights_fit(a, w))
    return pybind11::none();
  return pybind11::cast(SwigluProjectionNode::apply(a, b, w, wants(a) || wants(b)));
}

pybind11::object eager_embedding(const Tensor& tokens, const Tensor& weight, double scale, std::optional<int64_t> padding_idx) {
  if (!plain_call({&weight, &tokens}) || weight.dim() != 2 || weight.numel() == 0 || tokens.numel() == 0 ||
      !(half(weight) || weight.scalar_type() == at::kFloat) ||
      !(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt))
    return pybind11::none();
  const int64_t V = weight.size(0);
  int64_t pad = -1;
  if (padding_idx) {
    if (*padding_idx < -V || *padding_idx >= V) return pybind11::none();
    pad = *padding_idx < 0 ? *padding_idx + V : *padding_idx;
  }
  return pybind11::cast(EmbeddingNode::apply(weight, tokens, scale, pad));
}

}  // namespace

TORCH_LIBRARY_IMPL(kdattn, CUDA, m) {
  m.impl("quant_rows8", quant_rows8);
  m.impl("quant_weight8", quant_weight8);
  m.impl("matmul8", matmul8);
  m.impl("norm8", norm8);
  m.impl("norm8_bwd", norm8_bwd);
  m.impl("gate8", gate8);
  m.impl("gate8_bwd", gate8_bwd);
  m.impl("weight_grad8", weight_grad8);
  m.impl("embed", embed);
  m.impl("embed_grad", embed_grad);
}

namespace kdt {
void bind_block8(pybind11::module& m) {
  m.def("quantize_rows", torch::wrap_pybind_function(eager_quantize_rows));
  m.def("fp8_matmul", torch::wrap_pybind_function(eager_matmul));
  m.def("add_rms_norm_fp8", torch::wrap_pybind_function(eager_norm));
  m.def("norm_projection", torch::wrap_pybind_function(eager_norm_projection));
  m.def("fp8_projection", torch::wrap_pybind_function(eager_projection));
  m.def("swiglu_projection", torch::wrap_pybind_function(eager_swiglu_projection));
  m.def("embedding", torch::wrap_pybind_function(eager_embedding));
}
}  // namespace kdt
