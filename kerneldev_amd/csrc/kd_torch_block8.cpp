// The 8-bit blocks' and the embedding's operators (block_fp8.py, embed.py, which
// declare them) from torch to the C ABI: checks of what the kernels assume,
// allocations and launches on the current stream of the operands' device.  They
// hold no autograd rule; the Python layer's nodes call them.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include "../../include/kdattn.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

void check(int status, const char* what) {
  if (status == KD_OK) return;
  const std::string msg = std::string(what) + ": " + kd_last_error_string();
  TORCH_CHECK_VALUE(status != KD_ERR_INVALID && status != KD_ERR_UNSUPPORTED, msg);
  TORCH_CHECK(false, msg, " (status ", status, ")");
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

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

int64_t blocks(int64_t n) { return (n + 127) / 128; }
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
Tensor bytes8(const Tensor& like, int64_t rows, int64_t cols) {
  return at::empty({rows, up16(cols)}, like.options().dtype(at::kFloat8_e4m3fn));
}
Tensor scales(const Tensor& like, int64_t rows, int64_t nb) {
  return at::empty({rows, nb}, like.options().dtype(at::kFloat8_e8m0fnu));
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
    a.x[a.n] = keep.back().data_ptr(), a.x_stride[a.n] = keep.back().stride(0), a.cols[a.n] = int32_t(x.size(1)), ++a.n;
    total += x.size(1);
  }
  const c10::DeviceGuard on(xs[0].device());
  a.dtype = dtype_code(xs[0].scalar_type(), true);
  a.rows = xs[0].size(0), a.total = int32_t(total);
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
    a.w[a.n] = keep.back().data_ptr(), a.w_stride[a.n] = keep.back().stride(0), a.rows[a.n] = int32_t(w.size(0)), ++a.n;
    total += w.size(0);
  }
  const c10::DeviceGuard on(ws[0].device());
  const int64_t K = ws[0].size(1);
  a.dtype = dtype_code(ws[0].scalar_type(), true), a.K = int32_t(K), a.total = int32_t(total);
  Tensor y = bytes8(ws[0], total, K), s = scales(ws[0], blocks(total), blocks(K));
  Tensor yt = transpose ? bytes8(ws[0], K, total) : bytes8(ws[0], 0, 0);
  Tensor st = transpose ? scales(ws[0], blocks(K), blocks(total)) : scales(ws[0], 0, 0);
  a.y = u8(y), a.y_stride = y.stride(0), a.scale = u8(s);
  if (transpose) a.yt = u8(yt), a.yt_stride = yt.stride(0), a.scale_t = u8(st);
  check(kd_quant_weight8(&a, stream_of(y)), "kd_quant_weight8");
  return {y, s, yt, st};
}

Tensor matmul8(const Tensor& a_in, const Tensor& a_scale, const Tensor& b_in, const Tensor& b_scale, at::ScalarType out_type) {
  on_one_gpu({&a_in, &a_scale, &b_in, &b_scale});
  const Tensor a = blocks_ready(a_in), b = blocks_ready(b_in);
  const Tensor as = a_scale.contiguous(), bs = b_scale.contiguous();
  const c10::DeviceGuard on(a.device());
  TORCH_CHECK_VALUE(a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(1), "a [M, K] and b [N, K] expected, got ", a.sizes(),
                    " and ", b.sizes());
  const int64_t M = a.size(0), N = b.size(0), K = a.size(1);
  check_blocks(a, as, K, 1, "a"), check_blocks(b, bs, K, 128, "b");
  TORCH_CHECK_VALUE(M < (int64_t(1) << 31) && N < (int64_t(1) << 31) && K < (int64_t(1) << 31), "M, N and K must be < 2^31");
  kd_matmul8_args g{};
  g.dtype = dtype_code(out_type, true);
  Tensor out = at::empty({M, N}, a.options().dtype(out_type));
  if (out.numel() == 0) return out;
  g.a = u8(a), g.b = u8(b), g.lda = a.stride(0), g.ldb = b.stride(0), g.a_scale = u8(as), g.b_scale = u8(bs);
  g.out = out.data_ptr(), g.ldo = N;
  g.M = int32_t(M), g.N = int32_t(N), g.K = int32_t(K);
  check(kd_matmul8(&g, stream_of(out)), "kd_matmul8");
  return out;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> norm8(const Tensor& x_in, const OptTensor& delta, double eps) {
  on_one_gpu({&x_in});
  TORCH_CHECK_VALUE(x_in.dim() == 2, "x must be a matrix");
  const c10::DeviceGuard on(x_in.device());
  const Tensor x = flat(x_in);
  Tensor d, sum = at::empty({0}, x.options());
  kd_norm8_args a{};
  a.dtype = dtype_code(x.scalar_type(), false);
  a.rows = x.size(0), a.D = int32_t(x.size(1)), a.eps = float(eps);
  if (delta) {
    on_one_gpu({&x, &*delta});
    TORCH_CHECK_VALUE(delta->sizes() == x.sizes() && delta->scalar_type() == x.scalar_type(),
                      "x and delta must have one shape and type");
    d = flat(*delta), sum = at::empty(x.sizes(), x.options());
    a.delta = d.data_ptr(), a.sum = sum.data_ptr();
  }
  Tensor y = bytes8(x, a.rows, a.D), s = scales(x, a.rows, blocks(a.D)), rstd = at::empty({a.rows}, x.options().dtype(at::kFloat));
  if (a.rows == 0) return {sum, y, s, rstd};
  a.x = x.data_ptr(), a.y = u8(y), a.y_stride = y.stride(0), a.scale = u8(s), a.rstd = static_cast<float*>(rstd.data_ptr());
  check(kd_norm8(&a, stream_of(x)), "kd_norm8");
  return {sum, y, s, rstd};
}

Tensor norm8_bwd(const Tensor& g_in, const OptTensor& ds, const Tensor& y, const Tensor& scale, const Tensor& rstd) {
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
    TORCH_CHECK_VALUE(ds->sizes() == g.sizes() && ds->scalar_type() == g.scalar_type(), "g and ds must have one shape and type");
    d = flat(*ds);
  }
  kd_norm8_bwd_args a{};
  a.dtype = dtype_code(g.scalar_type(), false);
  Tensor dx = at::empty(g.sizes(), g.options());
  a.rows = g.size(0), a.D = int32_t(g.size(1));
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
  g.rows = a.size(0), g.H = int32_t(a.size(1));
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

std::tuple<Tensor, Tensor> gate8_bwd(const Tensor& dy_in, const Tensor& a8, const Tensor& as, const Tensor& b8, const Tensor& bs) {
  on_one_gpu({&dy_in, &a8, &as, &b8, &bs});
  TORCH_CHECK_VALUE(dy_in.dim() == 2 && a8.size(0) == dy_in.size(0) && b8.sizes() == a8.sizes() && b8.strides() == a8.strides(),
                    "dy, a and b must have one number of rows");
  check_blocks(a8, as, dy_in.size(1), 1, "a"), check_blocks(b8, bs, dy_in.size(1), 1, "b");
  const c10::DeviceGuard on(dy_in.device());
  const Tensor dy = flat(dy_in);
  Tensor da = at::empty(dy.sizes(), dy.options()), db = at::empty(dy.sizes(), dy.options());
  kd_gate8_args g{};
  g.dtype = dtype_code(dy.scalar_type(), false);
  g.rows = dy.size(0), g.H = int32_t(dy.size(1));
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
    TORCH_CHECK_VALUE(dy.size(1) < (int64_t(1) << 31), "N must be < 2^31");
    g.dy[g.n] = dy.data_ptr(), g.ldy[g.n] = dy.stride(0), g.cols[g.n] = int32_t(dy.size(1)), ++g.n;
    N += dy.size(1);
  }
  check_blocks(x, x_scale, K, 1, "x");
  const int64_t M = x.size(0);
  TORCH_CHECK_VALUE(M < (int64_t(1) << 31) && N < (int64_t(1) << 31), "M and N must be < 2^31");
  g.dtype = dtype_code(dys[0].scalar_type(), false);
  if (M == 0) return at::zeros({N, K}, dys[0].options());
  Tensor dw = at::empty({N, K}, dys[0].options());
  g.M = int32_t(M), g.N = int32_t(N), g.K = int32_t(K);
  g.ws_bytes = kd_weight_grad8_ws_bytes(g.M, g.N, g.K, g.dtype);
  check(g.ws_bytes < 0 ? KD_ERR_UNSUPPORTED : KD_OK, "kd_weight_grad8");
  const Tensor ws = at::empty({g.ws_bytes}, dys[0].options().dtype(at::kByte));
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
  Tensor out = at::empty(shape, weight.options());
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
  Tensor dw = at::empty({vocab, dim}, dy.options());
  const int64_t need = kd_embed_grad_ws_bytes(a.n, vocab, dim);
  const Tensor ws = at::empty({std::max<int64_t>(need, 0)}, dy.options().dtype(at::kByte));
  a.dy = dy.data_ptr(), a.dw = dw.data_ptr(), a.padding_idx = padding_idx;
  check(kd_embed_grad(&a, ws.data_ptr(), need, stream_of(dy)), "kd_embed_grad");
  return dw;
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
