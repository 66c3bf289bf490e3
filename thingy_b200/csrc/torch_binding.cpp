// Thin torch binding over the C ABI in include/cutie.h (no kernels here).
//
// Python could call the C ABI through ctypes, but marshalling 22 arguments and
// checking tensors from Python costs ~15 us a call, several times the kernel
// at decode sizes. This module takes at::Tensor arguments, derives pointers,
// leading dimensions and the current CUDA stream in C++, and calls the same
// extern "C" entry points. Argument errors raise ValueError, CUDA failures
// RuntimeError (the status codes of cutie.h).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <stdexcept>
#include <string>

#include "cutie.h"

namespace {

void check_status(int status) {
  if (status == CUTIE_OK) return;
  const std::string msg = cutie_last_error();
  if (status == CUTIE_ERR_CUDA) throw std::runtime_error(msg);
  throw std::invalid_argument(msg);
}

[[noreturn]] void bad(const std::string& msg) { throw std::invalid_argument(msg); }

// Leading dimension of a row-major [M, H] view (contiguous along H).
int64_t rows_ld(const at::Tensor& t, const char* name, int64_t M, int64_t H,
                at::ScalarType dtype, const at::Device& dev) {
  if (t.dim() != 2 || t.size(0) != M || t.size(1) != H)
    bad(std::string(name) + " must have shape (" + std::to_string(M) + ", " + std::to_string(H) +
        ")");
  if (t.scalar_type() != dtype) bad(std::string(name) + " has the wrong dtype");
  if (t.device() != dev) bad(std::string(name) + " is on the wrong device");
  if (H > 1 && t.stride(1) != 1) bad(std::string(name) + " must be contiguous along its last dimension");
  return M > 0 ? std::max<int64_t>(t.stride(0), H) : H;
}

const void* ptr_or_null(const c10::optional<at::Tensor>& t) {
  return t.has_value() ? t->data_ptr() : nullptr;
}

// ld_scale for (layout, groups) from the scale tensor's shape and strides;
// mirrors thingy_b200.ops._scale_args.
int64_t scale_ld(const at::Tensor& s, int64_t M, int64_t G, int64_t layout) {
  if (layout == CUTIE_LAYOUT_COL_MAJOR_PACKED) {  // int32 words, four groups a word
    const int64_t W = (G + 3) / 4;
    if (s.dim() == 1 && W == 1) {
      if (s.size(0) != M || (M > 1 && s.stride(0) != 1)) bad("packed per-row scales must be a contiguous [M] tensor");
      return M;
    }
    if (s.dim() != 2) bad("packed scales must be 2-D");
    const int64_t a = s.size(0), b = s.size(1);
    if (a == M && b == W && (M <= 1 || s.stride(0) == 1)) return W > 1 ? std::max<int64_t>(s.stride(1), M) : M;
    if (a == W && b == M && (M <= 1 || s.stride(1) == 1)) return W > 1 ? std::max<int64_t>(s.stride(0), M) : M;
    bad("packed scales must be an int32 [M, ceil(n_groups/4)] tensor contiguous along M (or its transpose)");
  }
  if (layout == CUTIE_LAYOUT_MX_SWIZZLED) {
    if (!s.is_contiguous()) bad("swizzled scales need a contiguous buffer");
    const int64_t need = (M + 127) / 128 * 128 * ((G + 3) / 4 * 4);
    if (s.numel() < need) bad("swizzled scale buffer too small");
    return 0;
  }
  if (s.dim() == 1 && G == 1) {
    if (s.size(0) != M || (M > 1 && s.stride(0) != 1)) bad("per-token scale must be a contiguous [M] tensor");
    return layout == CUTIE_LAYOUT_COL_MAJOR ? M : 1;
  }
  if (s.dim() != 2) bad("scale must be 2-D");
  const int64_t a = s.size(0), b = s.size(1);
  if (layout == CUTIE_LAYOUT_ROW_MAJOR) {
    if (a != M || b != G) bad("row-major scale must have shape (M, n_groups)");
    if (G > 1 && s.stride(1) != 1) bad("row-major scale must be contiguous along groups");
    return M > 1 ? std::max<int64_t>(s.stride(0), G) : G;
  }
  if (a == G && b == M && (M <= 1 || s.stride(1) == 1)) return G > 1 ? std::max<int64_t>(s.stride(0), M) : M;
  if (a == M && b == G && (M <= 1 || s.stride(0) == 1)) return G > 1 ? std::max<int64_t>(s.stride(1), M) : M;
  bad("column-major scale must be a [n_groups, M] tensor contiguous along M (or its transpose)");
}

// Fused [residual add] -> RMSNorm -> [FP8 quantization]; normalize=false is
// the quantizer alone. q / scale absent: no quantization.
void rms_norm_fp8(const at::Tensor& x, const c10::optional<at::Tensor>& weight, double eps,
                  const c10::optional<at::Tensor>& residual, const c10::optional<at::Tensor>& q,
                  const c10::optional<at::Tensor>& scale,
                  const c10::optional<at::Tensor>& residual_out,
                  const c10::optional<at::Tensor>& normalized_out, int64_t group_size,
                  int64_t scale_fmt, int64_t scale_layout, int64_t threads_per_row,
                  bool normalize) {
  if (x.dim() != 2) bad("x must be 2-D [M, H]");
  if (!x.is_cuda()) bad("x must be a CUDA tensor (this library has no CPU path)");
  if (x.scalar_type() != at::kBFloat16) bad("x must be bfloat16");
  const int64_t M = x.size(0), H = x.size(1);
  const at::Device dev = x.device();
  const int64_t ldx = rows_ld(x, "x", M, H, at::kBFloat16, dev);
  const int64_t ldr = residual ? rows_ld(*residual, "residual", M, H, at::kBFloat16, dev) : 0;
  const int64_t ldro =
      residual_out ? rows_ld(*residual_out, "residual_out", M, H, at::kBFloat16, dev) : 0;
  const int64_t ldn =
      normalized_out ? rows_ld(*normalized_out, "normalized_out", M, H, at::kBFloat16, dev) : 0;
  if (normalize) {
    if (!weight) bad("weight is required");
    if (weight->dim() != 1 || weight->size(0) != H || weight->scalar_type() != at::kBFloat16 ||
        weight->device() != dev || !weight->is_contiguous())
      bad("weight must be a contiguous bf16 [H] tensor on x's device");
  }
  const bool quant = q.has_value() || scale.has_value();
  int64_t ldq = 0, lds = 0;
  int mode = CUTIE_QUANT_NONE;
  if (quant) {
    if (!q || !scale) bad("q and scale must be given together");
    if (q->scalar_type() != at::kFloat8_e4m3fn && q->scalar_type() != at::kByte)
      bad("q must be float8_e4m3fn");
    ldq = rows_ld(*q, "q", M, H, q->scalar_type(), dev);
    const int64_t G = group_size > 0 ? (H + group_size - 1) / group_size : 1;
    if (scale_layout == CUTIE_LAYOUT_COL_MAJOR_PACKED) {
      if (scale->scalar_type() != at::kInt) bad("packed e8m0 scales must be int32 words");
    } else if (scale_fmt == CUTIE_SCALE_E8M0) {
      if (scale->element_size() != 1) bad("e8m0 scales must be 1-byte elements");
    } else if (scale->scalar_type() != at::kFloat) {
      bad("fp32 / pow2 scales must be float32");
    }
    if (scale->device() != dev) bad("scale is on the wrong device");
    lds = scale_ld(*scale, M, G, scale_layout);
    mode = group_size > 0 ? CUTIE_QUANT_GROUP : CUTIE_QUANT_TOKEN;
  }
  const c10::cuda::CUDAGuard guard(dev);
  void* stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  int status;
  if (normalize) {
    status = cutie_rms_norm_fp8(
        x.data_ptr(), ldx, ptr_or_null(residual), ldr, weight->data_ptr(), (float)eps, M, H, mode,
        (int)group_size, (int)scale_fmt, (int)scale_layout, lds,
        quant ? q->data_ptr() : nullptr, ldq, quant ? scale->data_ptr() : nullptr,
        const_cast<void*>(ptr_or_null(residual_out)), ldro,
        const_cast<void*>(ptr_or_null(normalized_out)), ldn, (int)threads_per_row, stream);
  } else {
    if (!quant) bad("quantization-only call needs q and scale");
    status = cutie_per_token_cast_to_fp8(x.data_ptr(), ldx, M, H, (int)group_size, (int)scale_fmt,
                                         (int)scale_layout, lds, q->data_ptr(), ldq,
                                         scale->data_ptr(), (int)threads_per_row, stream);
  }
  check_status(status);
}

void rms_norm(const at::Tensor& x, const at::Tensor& weight, double eps, const at::Tensor& out,
              int64_t threads_per_row) {
  if (x.dim() != 2) bad("x must be 2-D [M, H]");
  if (!x.is_cuda()) bad("x must be a CUDA tensor (this library has no CPU path)");
  const auto dt = x.scalar_type();
  if (dt != at::kBFloat16 && dt != at::kFloat) bad("x must be bfloat16 or float32");
  const int64_t M = x.size(0), H = x.size(1);
  const at::Device dev = x.device();
  const int64_t ldx = rows_ld(x, "x", M, H, dt, dev);
  const int64_t ldo = rows_ld(out, "out", M, H, dt, dev);
  if (weight.dim() != 1 || weight.size(0) != H || weight.scalar_type() != dt ||
      weight.device() != dev || !weight.is_contiguous())
    bad("weight must be a contiguous [H] tensor of x's dtype on x's device");
  const c10::cuda::CUDAGuard guard(dev);
  void* stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  check_status(cutie_rms_norm(x.data_ptr(), ldx, weight.data_ptr(), (float)eps, M, H,
                              dt == at::kBFloat16 ? CUTIE_DTYPE_BF16 : CUTIE_DTYPE_F32,
                              out.data_ptr(), ldo, (int)threads_per_row, stream));
}

// Leading dimension of a matrix whose rows are contiguous and do not overlap.
int64_t matrix_ld(const at::Tensor& t, const char* name, const at::Device& dev) {
  if (t.dim() != 2) bad(std::string(name) + " must be 2-D");
  if (t.device() != dev) bad(std::string(name) + " is on the wrong device");
  const int64_t R = t.size(0), C = t.size(1);
  if (C > 1 && t.stride(1) != 1) bad(std::string(name) + " must be contiguous along its last dimension");
  if (R <= 1) return std::max<int64_t>(C, (C + 15) / 16 * 16);
  if (t.stride(0) < C) bad(std::string(name) + " must not have overlapping rows");
  return t.stride(0);
}

void check_codes(const at::Tensor& t, const char* name) {
  if (t.scalar_type() != at::kFloat8_e4m3fn && t.scalar_type() != at::kByte)
    bad(std::string(name) + " must be float8_e4m3fn");
}

int64_t ceil_to(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

// e4m3 [R, C] with rows on 16-byte boundaries (what the block-scaled GEMM takes).
at::Tensor empty_codes(int64_t R, int64_t C, const at::Device& dev) {
  return at::empty_strided({R, C}, {ceil_to(C, 16), 1},
                           at::TensorOptions().device(dev).dtype(at::kFloat8_e4m3fn));
}

// Casts to e4m3 in both orientations (cutie_cast_fp8_tiles); qt and st are
// undefined tensors unless `transposed`.
std::tuple<at::Tensor, at::Tensor, c10::optional<at::Tensor>, c10::optional<at::Tensor>>
cast_fp8_tiles(const at::Tensor& x, bool block, bool use_ue8m0, bool transposed, bool gradient) {
  if (x.dim() != 2) bad("x must be 2-D [M, H]");
  if (!x.is_cuda()) bad("x must be a CUDA tensor (this library has no CPU path)");
  if (x.scalar_type() != at::kBFloat16) bad("x must be bfloat16");
  const int64_t M = x.size(0), H = x.size(1);
  const at::Device dev = x.device();
  const int64_t ldx = M <= 1 ? ceil_to(H, 8) : matrix_ld(x, "x", dev);
  if (H > 1 && x.stride(1) != 1) bad("x must be contiguous along its last dimension");
  const int64_t GM = (M + 127) / 128, GH = (H + 127) / 128;
  const auto f32 = at::TensorOptions().device(dev).dtype(at::kFloat);
  at::Tensor q = empty_codes(M, H, dev);
  at::Tensor s = block ? at::empty({GM, GH}, f32) : at::empty_strided({M, GH}, {1, M}, f32);
  at::Tensor qt, st;
  if (transposed) {
    qt = empty_codes(H, M, dev);
    st = block ? at::empty({GH, GM}, f32) : at::empty_strided({H, GM}, {1, H}, f32);
  }
  const c10::cuda::CUDAGuard guard(dev);
  void* stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  check_status(cutie_cast_fp8_tiles(
      x.data_ptr(), ldx, M, H, block ? CUTIE_TILE_BLOCK : CUTIE_TILE_TWO_WAY,
      (use_ue8m0 ? CUTIE_SCALE_FP32_POW2 : CUTIE_SCALE_FP32) + (gradient ? CUTIE_SCALE_GRADIENT : 0),
      q.data_ptr(), ceil_to(H, 16),
      s.data_ptr(), block ? GH : M, transposed ? qt.data_ptr() : nullptr,
      transposed ? ceil_to(M, 16) : 0, transposed ? st.data_ptr() : nullptr,
      transposed ? (block ? GM : H) : 0, stream));
  c10::optional<at::Tensor> oqt, ost;
  if (transposed) oqt = qt, ost = st;
  return {q, s, oqt, ost};
}

// D = dequant(a) dequant(b)^T (cutie_fp8_block_gemm) into `out`, or a new tensor.
at::Tensor fp8_block_gemm(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b,
                          const at::Tensor& b_scale, const c10::optional<at::Tensor>& out,
                          bool out_f32, bool accumulate) {
  if (!a.is_cuda()) bad("a must be a CUDA tensor (this library has no CPU path)");
  const at::Device dev = a.device();
  check_codes(a, "a");
  check_codes(b, "b");
  const int64_t lda = matrix_ld(a, "a", dev), ldb = matrix_ld(b, "b", dev);
  const int64_t M = a.size(0), K = a.size(1), N = b.size(0), KB = (K + 127) / 128;
  if (b.size(1) != K) bad("a and b must have the same number of columns");
  for (const auto* s : {&a_scale, &b_scale}) {
    if (s->dim() != 2 || s->scalar_type() != at::kFloat) bad("scales must be 2-D float32 tensors");
    if (s->device() != dev) bad("scales must be on a's device");
  }
  if (a_scale.size(0) != M || a_scale.size(1) != KB)
    bad("a_scale must have shape [M, ceil(K/128)] = (" + std::to_string(M) + ", " +
        std::to_string(KB) + ")");
  const int64_t sb_rows = b_scale.size(0);
  if ((sb_rows != (N + 127) / 128 && sb_rows != N) || b_scale.size(1) != KB)
    bad("b_scale must have shape [ceil(N/128), ceil(K/128)] (128 x 128 blocks) or [N, ceil(K/128)]"
        " (1 x 128 groups)");
  if (out.has_value()) {
    if (out->dim() != 2 || out->size(0) != M || out->size(1) != N)
      bad("out must have shape (" + std::to_string(M) + ", " + std::to_string(N) + ")");
    if (out->scalar_type() != at::kBFloat16 && out->scalar_type() != at::kFloat)
      bad("out must be bfloat16 or float32");
    out_f32 = out->scalar_type() == at::kFloat;
  } else if (accumulate) {
    bad("accumulate needs out");
  }
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor d = out.has_value()
                     ? *out
                     : at::empty({M, N}, at::TensorOptions().device(dev).dtype(
                                             out_f32 ? at::kFloat : at::kBFloat16));
  const int64_t ldd = M <= 1 ? N : matrix_ld(d, "out", dev);
  if (N > 1 && d.stride(1) != 1) bad("out must be contiguous along its last dimension");
  if (d.device() != dev) bad("out is on the wrong device");
  void* stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  check_status(cutie_fp8_block_gemm(
      a.data_ptr(), lda, a_scale.data_ptr(), a_scale.stride(0), a_scale.stride(1), b.data_ptr(),
      ldb, b_scale.data_ptr(), b_scale.stride(0), b_scale.stride(1),
      sb_rows == N && sb_rows != (N + 127) / 128 ? 1 : 0, d.data_ptr(), ldd,
      out_f32 ? CUTIE_DTYPE_F32 : CUTIE_DTYPE_BF16, accumulate ? 1 : 0, M, N, K, stream));
  return d;
}

// ---- A linear layer in 8 bits under autograd: y = q(x) q(w)^T, dx = q(dy) q(w),
// dw = q(dy)^T q(x), x and dy in 1 x 128 groups along both axes, w in 128 x 128
// blocks. In C++, and with the casts' results in few buffers: as Python calls
// of the functions above a step took 150 us of host time, twice what the
// kernels of a 1001 x 1544 x 2048 step take.

// An operand of the block-scaled product.
struct Operand {
  const void* q = nullptr;
  int64_t ld = 0;
  const void* s = nullptr;
  int64_t s_row = 0, s_kb = 0;
};

// Where a matrix's codes and scales go, and its transpose's: two places, since
// backward reads the transpose's alone and holds nothing else.
struct CastPlace {
  int64_t R, C;
  bool block, gradient;
  int64_t off_s, row_bytes, off_st, column_bytes;
  uint8_t *row_base = nullptr, *column_base = nullptr;

  CastPlace(int64_t rows, int64_t cols, bool blocks, bool of_gradient = false)
      : R(rows), C(cols), block(blocks), gradient(of_gradient) {
    const int64_t GR = (R + 127) / 128, GC = (C + 127) / 128;
    off_s = ceil_to(R * ceil_to(C, 16), 256);
    row_bytes = off_s + ceil_to(4 * (block ? GR * GC : GC * R), 256);
    off_st = ceil_to(C * ceil_to(R, 16), 256);
    column_bytes = off_st + ceil_to(4 * (block ? GR * GC : GR * C), 256);
  }
  Operand rows() const {
    return {row_base, ceil_to(C, 16), row_base + off_s, block ? (C + 127) / 128 : 1, block ? 1 : R};
  }
  Operand columns() const {
    return {column_base, ceil_to(R, 16), column_base + off_st, block ? (R + 127) / 128 : 1, block ? 1 : C};
  }
  // Without a place for the transpose's the block kind writes none. A matrix
  // whose rows are not dense, overlap or start off the 16-byte boundaries is
  // copied first; that of a single row too: the kernel reads C neighbouring
  // elements.
  void cast(const at::Tensor& any, void* stream) const {
    if (R == 0 || C == 0) return;  // no codes
    const bool dense = (C <= 1 || any.stride(1) == 1) &&
                       (R <= 1 || (any.stride(0) >= C && any.stride(0) % 8 == 0)) &&
                       reinterpret_cast<uintptr_t>(any.data_ptr()) % 16 == 0;
    const at::Tensor x = dense ? any : any.clone(at::MemoryFormat::Contiguous);
    const Operand q = rows(), qt = column_base != nullptr ? columns() : Operand();
    check_status(cutie_cast_fp8_tiles(
        x.data_ptr(), R <= 1 ? ceil_to(C, 8) : x.stride(0), R, C,
        block ? CUTIE_TILE_BLOCK : CUTIE_TILE_TWO_WAY,
        CUTIE_SCALE_FP32 + (gradient ? CUTIE_SCALE_GRADIENT : 0), row_base, q.ld, row_base + off_s,
        block ? q.s_row : q.s_kb, column_base, qt.ld,
        column_base != nullptr ? column_base + off_st : nullptr, block ? qt.s_row : qt.s_kb, stream));
  }
};

at::Tensor bytes(int64_t n, const at::Tensor& like) {
  return at::empty({n}, like.options().dtype(at::kByte));
}
uint8_t* address(const at::Tensor& t) {
  return t.defined() ? static_cast<uint8_t*>(t.data_ptr()) : nullptr;
}

at::Tensor product(const Operand& a, const Operand& b, bool b_rows, int64_t M, int64_t N, int64_t K,
                   const at::Tensor& like, bool f32, void* stream) {
  at::Tensor d = at::empty({M, N}, like.options().dtype(f32 ? at::kFloat : at::kBFloat16));
  check_status(cutie_fp8_block_gemm(a.q, a.ld, a.s, a.s_row, a.s_kb, b.q, b.ld, b.s, b.s_row, b.s_kb,
                                    b_rows ? 1 : 0, d.data_ptr(), N,
                                    f32 ? CUTIE_DTYPE_F32 : CUTIE_DTYPE_BF16, 0, M, N, K, stream));
  return d;
}

Operand given(const at::Tensor& q, const at::Tensor& s, int64_t rows, int64_t cols, const at::Device& dev) {
  check_codes(q, "weight_fp8");
  if (q.dim() != 2 || q.size(0) != rows || q.size(1) != cols)
    bad("weight_fp8's codes must have the weight's shape, transposed for qt");
  if (s.dim() != 2 || s.size(0) != (rows + 127) / 128 || s.size(1) != (cols + 127) / 128 ||
      s.scalar_type() != at::kFloat || s.device() != dev)
    bad("weight_fp8's scales must be float32, one a 128 x 128 block");
  return {q.data_ptr(), matrix_ld(q, "weight_fp8", dev), s.data_ptr(), s.stride(0), s.stride(1)};
}

struct FP8Linear : public torch::autograd::Function<FP8Linear> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                            const at::Tensor& weight, const c10::optional<at::Tensor>& wq,
                            const c10::optional<at::Tensor>& ws,
                            const c10::optional<at::Tensor>& wqt,
                            const c10::optional<at::Tensor>& wst, bool need_dx, bool need_dw) {
    const at::Device dev = x.device();
    const int64_t M = x.size(0), K = x.size(1), N = weight.size(0);
    const c10::cuda::CUDAGuard guard(dev);
    void* stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
    CastPlace w(N, K, true), xs(M, K, false);
    const bool own = !wq.has_value();
    // what backward reads: the weight's transposed codes, then x's; the rest goes with this call
    const int64_t held_w = own && need_dx ? w.column_bytes : 0, held_x = need_dw ? xs.column_bytes : 0;
    const at::Tensor held = held_w + held_x > 0 ? bytes(held_w + held_x, x) : at::Tensor();
    const at::Tensor scratch =
        bytes(xs.row_bytes + (own ? w.row_bytes : 0) + (need_dw ? 0 : xs.column_bytes), x);
    xs.row_base = address(scratch);
    if (own) {
      w.row_base = xs.row_base + xs.row_bytes;
      if (held_w > 0) w.column_base = address(held);
      w.cast(weight.scalar_type() == at::kBFloat16 ? weight : weight.to(at::kBFloat16), stream);
    }
    // the two-way cast always writes both
    if (held_x > 0) xs.column_base = address(held) + held_w;
    else xs.column_base = xs.row_base + xs.row_bytes + (own ? w.row_bytes : 0);
    xs.cast(x, stream);
    at::Tensor y = product(xs.rows(), own ? w.rows() : given(*wq, *ws, N, K, dev), false, M,
                           N, K, x, false, stream);
    ctx->save_for_backward(
        {held, !own && need_dx ? *wqt : at::Tensor(), !own && need_dx ? *wst : at::Tensor()});
    ctx->saved_data["sizes"] = std::vector<int64_t>{N, K, need_dx, need_dw, !own,
                                                    weight.scalar_type() == at::kFloat};
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    if (at::GradMode::is_enabled())
      throw std::runtime_error("fp8_linear has no second derivatives (create_graph)");
    torch::autograd::variable_list out(8);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const auto sizes = ctx->saved_data["sizes"].toIntVector();
    const int64_t N = sizes[0], K = sizes[1];
    const at::Tensor& dy = grads[0];  // of any layout: a view into another gradient, an expanded sum's
    const int64_t M = dy.size(0);
    const at::Device dev = dy.device();
    const c10::cuda::CUDAGuard guard(dev);
    void* stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
    CastPlace d(M, N, false, true), w(N, K, true), xs(M, K, false);
    const at::Tensor codes = bytes(d.row_bytes + d.column_bytes, dy);
    d.row_base = address(codes), d.column_base = address(codes) + d.row_bytes;
    d.cast(dy, stream);
    if (sizes[2]) {
      Operand wt;
      if (sizes[4]) {
        wt = given(saved[1], saved[2], K, N, dev);
      } else {
        w.column_base = address(saved[0]);
        wt = w.columns();
      }
      out[0] = product(d.rows(), wt, false, M, K, N, dy, false, stream);
    }
    if (sizes[3]) {
      xs.column_base = address(saved[0]) + (sizes[2] && !sizes[4] ? w.column_bytes : 0);
      out[1] = product(d.columns(), xs.columns(), true, N, K, M, dy, sizes[5] != 0, stream);
    }
    return out;
  }
};

at::Tensor fp8_linear(const at::Tensor& x, const at::Tensor& weight,
                      const c10::optional<at::Tensor>& wq, const c10::optional<at::Tensor>& ws,
                      const c10::optional<at::Tensor>& wqt,
                      const c10::optional<at::Tensor>& wst) {
  if (x.dim() < 1 || weight.dim() != 2 || x.size(-1) != weight.size(1))
    bad("x and weight must be [..., K] and [N, K]");
  if (!x.is_cuda()) bad("x must be a CUDA tensor (this library has no CPU path)");
  if (weight.device() != x.device()) bad("weight is on the wrong device");
  if (x.scalar_type() != at::kBFloat16) bad("x must be bfloat16");
  if (weight.scalar_type() != at::kBFloat16 && weight.scalar_type() != at::kFloat)
    bad("weight must be bfloat16 or float32");
  if (weight.size(0) % 8 != 0 || weight.size(1) % 8 != 0) bad("weight's sizes must be multiples of 8");
  const bool grad = at::GradMode::is_enabled();
  const bool need_dx = grad && x.requires_grad(), need_dw = grad && weight.requires_grad();
  if (wq.has_value() != ws.has_value()) bad("weight_fp8 must be (q, s, qt, st)");
  if (wq.has_value() && need_dx && (!wqt.has_value() || !wst.has_value()))
    bad("weight_fp8 has no transposed codes: make it with "
        "per_block_cast_to_fp8(weight, transposed=True)");
  const at::Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  at::Tensor y = FP8Linear::apply(x2, weight, wq, ws, wqt, wst, need_dx, need_dw);
  if (x.dim() == 2) return y;
  auto shape = x.sizes().vec();
  shape.back() = weight.size(0);
  return y.reshape(shape);
}

// Bytes of workspace of a mixture-of-experts layer; argument errors raise.
int64_t moe_workspace_bytes(int64_t T, int64_t E, int64_t top_k, int64_t H, int64_t I, int64_t device) {
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  const size_t n = cutie_moe_fp8_workspace(T, E, top_k, H, I);
  if (n == 0) bad(cutie_last_error());
  return (int64_t)n;
}

void weight_3d(const at::Tensor& t, const char* name, int64_t E, int64_t R, int64_t C,
               const at::Device& dev) {
  if (t.dim() != 3 || t.size(0) != E || t.size(1) != R || t.size(2) != C)
    bad(std::string(name) + " must have shape (" + std::to_string(E) + ", " + std::to_string(R) +
        ", " + std::to_string(C) + ")");
  if (t.device() != dev) bad(std::string(name) + " is on the wrong device");
  if (!t.is_contiguous()) bad(std::string(name) + " must be contiguous");
}

// Mixture-of-experts layer for few tokens (cutie_moe_fp8).
at::Tensor moe_fp8(const at::Tensor& x, const at::Tensor& q, const at::Tensor& q_scale,
                   const at::Tensor& router, const c10::optional<at::Tensor>& bias,
                   const at::Tensor& w13, const at::Tensor& w13_scale, const at::Tensor& w2,
                   const at::Tensor& w2_scale, int64_t top_k, int64_t scoring, bool renormalize,
                   double routed_scale, const c10::optional<at::Tensor>& out,
                   const c10::optional<at::Tensor>& topk_ids,
                   const c10::optional<at::Tensor>& topk_weights, const at::Tensor& workspace) {
  if (!x.is_cuda()) bad("x must be a CUDA tensor (this library has no CPU path)");
  const at::Device dev = x.device();
  if (x.dim() != 2 || x.scalar_type() != at::kBFloat16) bad("x must be a 2-D bfloat16 tensor");
  const int64_t T = x.size(0), H = x.size(1);
  if (router.dim() != 2 || router.size(1) != H || router.scalar_type() != at::kBFloat16 ||
      router.device() != dev || !router.is_contiguous())
    bad("router must be a contiguous bfloat16 [E, H] tensor on x's device");
  const int64_t E = router.size(0);
  if (w2.dim() != 3) bad("w2 must be 3-D [E, H, I]");
  const int64_t I = w2.size(2), KB = (H + 127) / 128, IB = (I + 127) / 128;
  check_codes(q, "q");
  check_codes(w13, "w13");
  check_codes(w2, "w2");
  if (q.dim() != 2 || q.size(0) != T || q.size(1) != H) bad("q must have x's shape");
  weight_3d(w13, "w13", E, 2 * I, H, dev);
  weight_3d(w2, "w2", E, H, I, dev);
  weight_3d(w13_scale, "w13_scale", E, 2 * IB, KB, dev);
  weight_3d(w2_scale, "w2_scale", E, KB, IB, dev);
  if (q_scale.dim() != 2 || q_scale.size(0) != T || q_scale.size(1) != KB || q_scale.device() != dev)
    bad("scale must be a [T, H/128] tensor on x's device");
  for (const auto* s : {&q_scale, &w13_scale, &w2_scale})
    if (s->scalar_type() != at::kFloat) bad("scales must be float32");
  if (bias.has_value() && (bias->dim() != 1 || bias->size(0) != E || bias->device() != dev ||
                           bias->scalar_type() != at::kFloat || !bias->is_contiguous()))
    bad("bias must be a contiguous float32 [E] tensor on x's device");
  auto choice = [&](const c10::optional<at::Tensor>& t, const char* name, at::ScalarType dtype) {
    if (t.has_value() && (t->dim() != 2 || t->size(0) != T || t->size(1) != top_k ||
                          t->scalar_type() != dtype || t->device() != dev || !t->is_contiguous()))
      bad(std::string(name) + " must be a contiguous [T, top_k] tensor on x's device");
  };
  choice(topk_ids, "topk_ids", at::kInt);
  choice(topk_weights, "topk_weights", at::kFloat);
  if (workspace.device() != dev || !workspace.is_contiguous())
    bad("workspace must be a contiguous tensor on x's device");
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor y = out.has_value() ? *out : at::empty({T, H}, x.options());
  if (y.dim() != 2 || y.size(0) != T || y.size(1) != H || y.scalar_type() != at::kBFloat16)
    bad("out must be a bfloat16 tensor of x's shape");
  void* stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  check_status(cutie_moe_fp8(
      x.data_ptr(), matrix_ld(x, "x", dev), q.data_ptr(), matrix_ld(q, "q", dev),
      q_scale.data_ptr(), q_scale.stride(0), q_scale.stride(1), router.data_ptr(),
      ptr_or_null(bias), w13.data_ptr(), w13_scale.data_ptr(), w2.data_ptr(), w2_scale.data_ptr(),
      T, E, top_k, H, I, (int)scoring, renormalize ? 1 : 0, (float)routed_scale, y.data_ptr(),
      matrix_ld(y, "out", dev), const_cast<void*>(ptr_or_null(topk_ids)),
      const_cast<void*>(ptr_or_null(topk_weights)), workspace.data_ptr(),
      (size_t)(workspace.numel() * workspace.element_size()), stream));
  return y;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "torch binding of the cutie C ABI (thingy_b200)";
  m.def("rms_norm_fp8", &rms_norm_fp8, py::arg("x"), py::arg("weight"), py::arg("eps"),
        py::arg("residual"), py::arg("q"), py::arg("scale"), py::arg("residual_out"),
        py::arg("normalized_out"), py::arg("group_size"), py::arg("scale_fmt"),
        py::arg("scale_layout"), py::arg("threads_per_row"), py::arg("normalize"));
  m.def("rms_norm", &rms_norm, py::arg("x"), py::arg("weight"), py::arg("eps"), py::arg("out"),
        py::arg("threads_per_row"));
  m.def("cast_fp8_tiles", &cast_fp8_tiles, py::arg("x"), py::arg("block"), py::arg("use_ue8m0"),
        py::arg("transposed"), py::arg("gradient"));
  m.def("fp8_block_gemm", &fp8_block_gemm, py::arg("a"), py::arg("a_scale"), py::arg("b"),
        py::arg("b_scale"), py::arg("out"), py::arg("out_f32"), py::arg("accumulate"));
  m.def("fp8_linear", &fp8_linear, py::arg("x"), py::arg("weight"), py::arg("wq"), py::arg("ws"),
        py::arg("wqt"), py::arg("wst"));
  m.def("moe_workspace_bytes", &moe_workspace_bytes, py::arg("T"), py::arg("E"), py::arg("top_k"),
        py::arg("H"), py::arg("I"), py::arg("device"));
  m.def("moe_fp8", &moe_fp8, py::arg("x"), py::arg("q"), py::arg("scale"), py::arg("router"),
        py::arg("bias"), py::arg("w13"), py::arg("w13_scale"), py::arg("w2"), py::arg("w2_scale"),
        py::arg("top_k"), py::arg("scoring"), py::arg("renormalize"), py::arg("routed_scale"),
        py::arg("out"), py::arg("topk_ids"), py::arg("topk_weights"), py::arg("workspace"));
  m.def("abi_version", []() { return cutie_abi_version(); });
}
