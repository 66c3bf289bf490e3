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
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <algorithm>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

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
  // elements. With `sources` the rows are sorted by expert.
  void cast(const at::Tensor& any, void* stream, const void* sources = nullptr) const {
    if (R == 0 || C == 0) return;  // no codes
    const bool f32 = any.scalar_type() == at::kFloat;  // weights: rounded to bf16 on the way
    const bool dense = (C <= 1 || any.stride(1) == 1) &&
                       (R <= 1 || (any.stride(0) >= C && any.stride(0) % (f32 ? 4 : 8) == 0)) &&
                       reinterpret_cast<uintptr_t>(any.data_ptr()) % 16 == 0;
    const at::Tensor x = dense ? any : any.clone(at::MemoryFormat::Contiguous);
    const Operand q = rows(), qt = column_base != nullptr ? columns() : Operand();
    if (sources != nullptr) {
      check_status(cutie_cast_fp8_sorted(
          x.data_ptr(), x.stride(0), R, C, sources, CUTIE_SCALE_FP32 + (gradient ? CUTIE_SCALE_GRADIENT : 0), row_base,
          q.ld, row_base + off_s, q.s_kb, column_base, qt.ld, column_base + off_st, qt.s_kb, stream));
      return;
    }
    check_status(cutie_cast_fp8_tiles(
        x.data_ptr(), R <= 1 ? ceil_to(C, 8) : x.stride(0), R, C,
        f32 ? CUTIE_TILE_BLOCK_F32 : block ? CUTIE_TILE_BLOCK : CUTIE_TILE_TWO_WAY,
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
      w.cast(weight, stream);
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

void no_second_derivatives(const char* name) {
  if (at::GradMode::is_enabled())
    throw std::runtime_error(std::string(name) + " has no second derivatives (create_graph)");
}

// ---- The experts' products on sorted rows (cutie_fp8_grouped_gemm, _wgrad).

// A plan's offsets and counts as the products take them.
void product_offsets(const at::Tensor& offsets, const at::Tensor& counts, int64_t align, int64_t E,
                     const at::Device& dev) {
  if (align <= 0 || align % 128 != 0) bad("the experts' products need a plan with align a multiple of 128");
  if (offsets.dim() != 1 || offsets.size(0) != E + 1 || offsets.scalar_type() != at::kInt ||
      !offsets.is_contiguous() || offsets.device() != dev)
    bad("the plan's offsets must be a contiguous int32 [E + 1] tensor on the rows' device, E = " + std::to_string(E));
  if (counts.dim() != 1 || counts.size(0) != E || counts.scalar_type() != at::kInt || !counts.is_contiguous() ||
      counts.device() != dev)
    bad("the plan's counts must be a contiguous int32 [E] tensor on the rows' device");
}

// Matrices [E, N, K] of codes and their scales [E, ceil(N/128), ceil(K/128)].
struct Matrices {
  const void* q;
  int64_t ld, each;
  const void* s;
  int64_t s_row, s_kb, s_each;
};
Matrices expert_matrices(const at::Tensor& q, const at::Tensor& s, int64_t E, int64_t N, int64_t K,
                         const at::Device& dev, const char* name) {
  check_codes(q, name);
  if (q.dim() != 3 || q.size(0) != E || q.size(1) != N || q.size(2) != K)
    bad(std::string(name) + " must have shape (" + std::to_string(E) + ", " + std::to_string(N) + ", " +
        std::to_string(K) + ")");
  if (q.device() != dev) bad(std::string(name) + " is on the wrong device");
  if (K > 1 && q.stride(2) != 1) bad(std::string(name) + " must be contiguous along its last dimension");
  if (N > 1 && q.stride(1) < K) bad(std::string(name) + " must not have overlapping rows");
  if (s.dim() != 3 || s.size(0) != E || s.size(1) != (N + 127) / 128 || s.size(2) != (K + 127) / 128 ||
      s.scalar_type() != at::kFloat || s.device() != dev)
    bad(std::string(name) + "'s scales must be float32, one a 128 x 128 block of each expert");
  return {q.data_ptr(), N > 1 ? q.stride(1) : ceil_to(K, 16), E > 1 ? q.stride(0) : 0,
          s.data_ptr(), s.stride(1), s.stride(2), s.stride(0)};
}

void grouped_product(const Operand& a, const Matrices& b, const at::Tensor& offsets, const at::Tensor& counts,
                     int64_t E, const at::Tensor& d, int64_t ldd, int64_t R, int64_t N, int64_t K, void* stream) {
  check_status(cutie_fp8_grouped_gemm(
      a.q, a.ld, a.s, a.s_row, a.s_kb, b.q, b.ld, b.each, b.s, b.s_row, b.s_kb, b.s_each, offsets.data_ptr(), counts.data_ptr(), E,
      d.data_ptr(), ldd, d.scalar_type() == at::kFloat ? CUTIE_DTYPE_F32 : CUTIE_DTYPE_BF16, R, N, K, stream));
}

at::Tensor fp8_grouped_gemm(const at::Tensor& a, const at::Tensor& a_scale, const at::Tensor& b,
                            const at::Tensor& b_scale, const at::Tensor& offsets, const at::Tensor& counts,
                            int64_t align,
                            const c10::optional<at::Tensor>& out, bool out_f32) {
  if (!a.is_cuda()) bad("a must be a CUDA tensor (this library has no CPU path)");
  const at::Device dev = a.device();
  check_codes(a, "a");
  const int64_t lda = matrix_ld(a, "a", dev);
  if (b.dim() != 3) bad("b must be 3-D [E, N, K]");
  const int64_t R = a.size(0), K = a.size(1), E = b.size(0), N = b.size(1);
  product_offsets(offsets, counts, align, E, dev);
  if (a_scale.dim() != 2 || a_scale.size(0) != R || a_scale.size(1) != (K + 127) / 128 ||
      a_scale.scalar_type() != at::kFloat || a_scale.device() != dev)
    bad("a_scale must be a float32 [R, ceil(K/128)] tensor on a's device");
  const Matrices m = expert_matrices(b, b_scale, E, N, K, dev, "b");
  const c10::cuda::CUDAGuard guard(dev);
  if (out.has_value()) {
    if (out->dim() != 2 || out->size(0) != R || out->size(1) != N || out->device() != dev)
      bad("out must have shape (" + std::to_string(R) + ", " + std::to_string(N) + ") and be on a's device");
    if (out->scalar_type() != at::kBFloat16 && out->scalar_type() != at::kFloat)
      bad("out must be bfloat16 or float32");
  }
  at::Tensor d = out.has_value() ? *out
                                 : at::empty({R, N}, at::TensorOptions().device(dev).dtype(
                                                         out_f32 ? at::kFloat : at::kBFloat16));
  const Operand rows{a.data_ptr(), lda, a_scale.data_ptr(), a_scale.stride(0), a_scale.stride(1)};
  grouped_product(rows, m, offsets, counts, E, d, matrix_ld(d, "out", dev), R, N, K,
                  at::cuda::getCurrentCUDAStream(dev.index()).stream());
  return d;
}

struct FP8GroupedLinear : public torch::autograd::Function<FP8GroupedLinear> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                            const c10::optional<at::Tensor>& wq, const c10::optional<at::Tensor>& ws,
                            const c10::optional<at::Tensor>& wqt, const c10::optional<at::Tensor>& wst,
                            const at::Tensor& sources, const at::Tensor& offsets, const at::Tensor& counts,
                            bool need_dx, bool need_dw) {
    const at::Device dev = x.device();
    const int64_t R = x.size(0), E = weight.size(0), N = weight.size(1), K = weight.size(2);
    const c10::cuda::CUDAGuard guard(dev);
    void* stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
    CastPlace w(E * N, K, true), xs(R, K, false);  // blocks of 128 do not cross experts: N is a multiple
    const bool own = !wq.has_value();
    // what backward reads: the weight's transposed codes, then x's; the rest goes with this call
    const int64_t held_w = own && need_dx ? w.column_bytes : 0, held_x = need_dw ? xs.column_bytes : 0;
    const at::Tensor held = held_w + held_x > 0 ? bytes(held_w + held_x, x) : at::Tensor();
    const at::Tensor scratch = bytes(xs.row_bytes + (own ? w.row_bytes : 0) + (need_dw ? 0 : xs.column_bytes), x);
    xs.row_base = address(scratch);
    if (own) {
      w.row_base = xs.row_base + xs.row_bytes;
      if (held_w > 0) w.column_base = address(held);
      w.cast(weight.reshape({E * N, K}), stream);
    }
    xs.column_base = held_x > 0 ? address(held) + held_w : xs.row_base + xs.row_bytes + (own ? w.row_bytes : 0);
    xs.cast(x, stream, sources.data_ptr());
    at::Tensor y = at::empty({R, N}, x.options());
    Matrices m;
    if (own) {
      const Operand q = w.rows();
      m = {q.q, q.ld, N * q.ld, q.s, q.s_row, q.s_kb, N / 128 * q.s_row};
    } else {
      m = expert_matrices(*wq, *ws, E, N, K, dev, "weight_fp8");
    }
    grouped_product(xs.rows(), m, offsets, counts, E, y, N, R, N, K, stream);
    ctx->save_for_backward({held, !own && need_dx ? *wqt : at::Tensor(), !own && need_dx ? *wst : at::Tensor(),
                            sources, offsets, counts});
    ctx->saved_data["sizes"] =
        std::vector<int64_t>{E, N, K, need_dx, need_dw, !own, weight.scalar_type() == at::kFloat};
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    no_second_derivatives("fp8_grouped_linear");
    torch::autograd::variable_list out(11);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const auto sizes = ctx->saved_data["sizes"].toIntVector();
    const int64_t E = sizes[0], N = sizes[1], K = sizes[2];
    const bool need_dx = sizes[3], need_dw = sizes[4], given_w = sizes[5], dw_f32 = sizes[6];
    const at::Tensor &dy = grads[0], &sources = saved[3], &offsets = saved[4], &counts = saved[5];
    const int64_t R = dy.size(0);
    const at::Device dev = dy.device();
    const c10::cuda::CUDAGuard guard(dev);
    void* stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
    CastPlace d(R, N, false, true), w(E * N, K, true), xs(R, K, false);
    const at::Tensor codes = bytes(d.row_bytes + d.column_bytes, dy);
    d.row_base = address(codes), d.column_base = address(codes) + d.row_bytes;
    d.cast(dy, stream, sources.data_ptr());
    if (need_dx) {
      Matrices m;
      if (given_w) {
        m = expert_matrices(saved[1], saved[2], E, K, N, dev, "weight_fp8");
      } else {
        w.column_base = address(saved[0]);
        const Operand q = w.columns();  // [K, E N]: an expert's transpose is N of its columns
        m = {q.q, q.ld, N, q.s, q.s_row, q.s_kb, N / 128};
      }
      out[0] = at::empty({R, K}, dy.options());
      grouped_product(d.rows(), m, offsets, counts, E, out[0], K, R, K, N, stream);
    }
    if (need_dw) {
      xs.column_base = address(saved[0]) + (need_dx && !given_w ? w.column_bytes : 0);
      const Operand a = d.columns(), b = xs.columns();
      out[1] = at::empty({E, N, K}, dy.options().dtype(dw_f32 ? at::kFloat : at::kBFloat16));
      check_status(cutie_fp8_grouped_wgrad(a.q, a.ld, a.s, a.s_row, a.s_kb, b.q, b.ld, b.s, b.s_row, b.s_kb,
                                           offsets.data_ptr(), E, out[1].data_ptr(), K, N * K,
                                           dw_f32 ? CUTIE_DTYPE_F32 : CUTIE_DTYPE_BF16, R, N, K, stream));
    }
    return out;
  }
};

at::Tensor fp8_grouped_linear(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& sources,
                              const at::Tensor& offsets, const at::Tensor& counts, int64_t align,
                              const c10::optional<at::Tensor>& wq,
                              const c10::optional<at::Tensor>& ws, const c10::optional<at::Tensor>& wqt,
                              const c10::optional<at::Tensor>& wst) {
  if (x.dim() != 2 || weight.dim() != 3 || x.size(1) != weight.size(2)) bad("x and weight must be [R, K] and [E, N, K]");
  if (!x.is_cuda()) bad("x must be a CUDA tensor (this library has no CPU path)");
  const at::Device dev = x.device();
  if (weight.device() != dev) bad("weight is on the wrong device");
  if (x.scalar_type() != at::kBFloat16) bad("x must be bfloat16");
  if (weight.scalar_type() != at::kBFloat16 && weight.scalar_type() != at::kFloat)
    bad("weight must be bfloat16 or float32");
  const int64_t R = x.size(0), E = weight.size(0), N = weight.size(1), K = weight.size(2);
  if (E == 0 || N == 0 || K == 0 || N % 128 != 0 || K % 128 != 0) bad("weight's sizes must be multiples of 128");
  product_offsets(offsets, counts, align, E, dev);
  if (sources.dim() != 1 || sources.size(0) != R || sources.scalar_type() != at::kInt || !sources.is_contiguous() ||
      sources.device() != dev)
    bad("x must have the plan's " + std::to_string(sources.size(0)) + " rows, the plan be int32 on x's device");
  const bool grad = at::GradMode::is_enabled();
  const bool need_dx = grad && x.requires_grad(), need_dw = grad && weight.requires_grad();
  if (wq.has_value() != ws.has_value()) bad("weight_fp8 must be (q, s, qt, st)");
  if (wq.has_value() && need_dx && (!wqt.has_value() || !wst.has_value()))
    bad("weight_fp8 has no transposed codes: make it with quantize_experts(weight, transposed=True)");
  if (wq.has_value()) expert_matrices(*wq, *ws, E, N, K, dev, "weight_fp8");
  if (wq.has_value() && need_dx) expert_matrices(*wqt, *wst, E, K, N, dev, "weight_fp8's transposes");
  return FP8GroupedLinear::apply(x, weight, wq, ws, wqt, wst, sources, offsets, counts, need_dx, need_dw);
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

// ---- Tokens sorted by expert and back (cutie_moe_sort, _permute, _combine).

int row_dtype(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return CUTIE_DTYPE_BF16;
    case at::kFloat: return CUTIE_DTYPE_F32;
    case at::kHalf: return CUTIE_DTYPE_F16;
    default: bad(std::string(name) + " must be bfloat16, float16 or float32");
  }
}

void plan_array(const at::Tensor& t, const char* name, int64_t dims, const at::Device& dev) {
  if (t.dim() != dims || t.scalar_type() != at::kInt || !t.is_contiguous())
    bad(std::string("the plan's ") + name + " must be a contiguous int32 tensor of " + std::to_string(dims) +
        " dimensions");
  if (t.device() != dev) bad(std::string("the plan's ") + name + " is on the wrong device");
}

// A matrix whose rows are dense and do not overlap: the tensor, or a copy.
at::Tensor dense_rows(const at::Tensor& t) {
  const bool dense = (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
  return dense ? t : t.clone(at::MemoryFormat::Contiguous);
}
int64_t row_stride(const at::Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

int64_t moe_plan_rows(int64_t T, int64_t k, int64_t E, int64_t align) {
  const int64_t rows = cutie_moe_plan_rows(T, k, E, align);
  if (rows < 0) bad(cutie_last_error());
  return rows;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> moe_sort(const at::Tensor& any, int64_t E,
                                                                    int64_t align, bool apart) {
  if (any.dim() != 2 || !any.is_cuda()) bad("topk_ids must be a 2-D CUDA tensor (this library has no CPU path)");
  if (any.scalar_type() != at::kInt && any.scalar_type() != at::kLong) bad("topk_ids must be int32 or int64");
  const int64_t T = any.size(0), k = any.size(1), R = moe_plan_rows(T, k, E, align);
  const at::Device dev = any.device();
  const c10::cuda::CUDAGuard guard(dev);
  const at::Tensor ids = any.contiguous();
  // one allocation, unless the results have to be apart (torch.library's): four are
  // half of a small sort's time on the host
  const at::AutoDispatchBelowADInplaceOrView below;
  const auto opt = at::TensorOptions().device(dev).dtype(at::kInt);
  const int64_t at_positions = ceil_to(R, 64), at_offsets = at_positions + ceil_to(T * k, 64);
  const int64_t at_counts = at_offsets + ceil_to(E + 1, 64);
  const at::Tensor buffer = apart ? at::Tensor() : at::empty({at_counts + E}, opt);
  at::Tensor sources = apart ? at::empty({R}, opt) : buffer.as_strided({R}, {1}, 0);
  at::Tensor positions = apart ? at::empty({T, k}, opt) : buffer.as_strided({T, k}, {k, 1}, at_positions);
  at::Tensor offsets = apart ? at::empty({E + 1}, opt) : buffer.as_strided({E + 1}, {1}, at_offsets);
  at::Tensor counts = apart ? at::empty({E}, opt) : buffer.as_strided({E}, {1}, at_counts);
  const size_t bytes = cutie_moe_sort_workspace(T, k, E);
  const at::Tensor workspace = bytes > 0 ? at::empty({(int64_t)bytes}, opt.dtype(at::kByte)) : at::Tensor();
  check_status(cutie_moe_sort(ids.data_ptr(), ids.scalar_type() == at::kLong ? 1 : 0, T, k, E, align,
                              sources.data_ptr(), R, positions.data_ptr(), offsets.data_ptr(), counts.data_ptr(),
                              bytes > 0 ? workspace.data_ptr() : nullptr, bytes,
                              at::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return {sources, positions, offsets, counts};
}

at::Tensor permute_rows(const at::Tensor& any, const at::Tensor& sources, const at::Tensor& positions) {
  const at::Tensor x = dense_rows(any);
  const int64_t H = x.size(1), R = sources.size(0);
  at::Tensor out = at::empty({R, H}, x.options());
  check_status(cutie_moe_permute(x.data_ptr(), row_stride(x), (int)x.element_size(), x.size(0), H,
                                 positions.size(1), positions.data_ptr(), sources.data_ptr(), R, out.data_ptr(), H,
                                 at::cuda::getCurrentCUDAStream(x.device().index()).stream()));
  return out;
}

at::Tensor combine_rows(const at::Tensor& any, const at::Tensor& weights, const at::Tensor& positions) {
  const at::Tensor ys = dense_rows(any);
  const int64_t H = ys.size(1), T = positions.size(0);
  at::Tensor out = at::empty({T, H}, ys.options());
  check_status(cutie_moe_combine(ys.data_ptr(), row_stride(ys), row_dtype(ys, "rows"),
                                 weights.defined() ? weights.data_ptr() : nullptr, positions.data_ptr(), T,
                                 positions.size(1), H, ys.size(0), out.data_ptr(), H,
                                 at::cuda::getCurrentCUDAStream(ys.device().index()).stream()));
  return out;
}

struct MoePermute : public torch::autograd::Function<MoePermute> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& sources,
                            const at::Tensor& positions) {
    const c10::cuda::CUDAGuard guard(x.device());
    ctx->save_for_backward({positions});
    return permute_rows(x, sources, positions);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    no_second_derivatives("moe_permute");
    torch::autograd::variable_list out(3);
    if (!grads[0].defined()) return out;
    const c10::cuda::CUDAGuard guard(grads[0].device());
    out[0] = combine_rows(grads[0], at::Tensor(), ctx->get_saved_variables()[0]);
    return out;
  }
};

at::Tensor moe_permute(const at::Tensor& x, const at::Tensor& sources, const at::Tensor& positions) {
  if (x.dim() != 2 || !x.is_cuda()) bad("x must be a 2-D CUDA tensor (this library has no CPU path)");
  const int64_t es = x.element_size();
  if (x.is_complex() || (es != 1 && es != 2 && es != 4)) bad("x must have elements of 1, 2 or 4 bytes");
  plan_array(sources, "sources", 1, x.device());
  plan_array(positions, "positions", 2, x.device());
  if (positions.size(0) != x.size(0))
    bad("x must have a row for each of the plan's " + std::to_string(positions.size(0)) + " tokens");
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    row_dtype(x, "x with a gradient");
    return MoePermute::apply(x, sources, positions);
  }
  const c10::cuda::CUDAGuard guard(x.device());
  return permute_rows(x, sources, positions);
}

struct MoeCombine : public torch::autograd::Function<MoeCombine> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& ys, const at::Tensor& weights,
                            const at::Tensor& sources, const at::Tensor& positions, bool need_rows,
                            bool need_weights) {
    const c10::cuda::CUDAGuard guard(ys.device());
    const at::Tensor w = weights.contiguous();
    ctx->save_for_backward({need_weights ? ys : at::Tensor(), w, sources, positions});
    ctx->saved_data["rows"] = need_rows;
    return combine_rows(ys, w, positions);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    no_second_derivatives("moe_combine");
    torch::autograd::variable_list out(6);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &w = saved[1], &sources = saved[2], &positions = saved[3];
    const at::Device dev = grads[0].device();
    const c10::cuda::CUDAGuard guard(dev);
    const at::Tensor dy = dense_rows(grads[0]);
    const int64_t H = dy.size(1), R = sources.size(0);
    const at::Tensor ys = saved[0].defined() ? dense_rows(saved[0]) : at::Tensor();
    if (ctx->saved_data["rows"].toBool()) out[0] = at::empty({R, H}, dy.options());
    if (ys.defined()) out[1] = at::empty_like(w);
    check_status(cutie_moe_combine_backward(
        dy.data_ptr(), row_stride(dy), ys.defined() ? ys.data_ptr() : nullptr, ys.defined() ? row_stride(ys) : 0,
        row_dtype(dy, "the gradient"), w.data_ptr(), positions.data_ptr(), sources.data_ptr(), dy.size(0),
        positions.size(1), H, R, out[0].defined() ? out[0].data_ptr() : nullptr, H,
        out[1].defined() ? out[1].data_ptr() : nullptr, at::cuda::getCurrentCUDAStream(dev.index()).stream()));
    return out;
  }
};

at::Tensor moe_combine(const at::Tensor& ys, const at::Tensor& weights, const at::Tensor& sources,
                       const at::Tensor& positions) {
  if (ys.dim() != 2 || !ys.is_cuda()) bad("rows must be a 2-D CUDA tensor (this library has no CPU path)");
  row_dtype(ys, "rows");
  if (ys.size(1) == 0) bad("rows must have at least one column");
  plan_array(sources, "sources", 1, ys.device());
  plan_array(positions, "positions", 2, ys.device());
  if (ys.size(0) != sources.size(0))
    bad("rows must have the plan's " + std::to_string(sources.size(0)) + " rows");
  if (weights.dim() != 2 || weights.size(0) != positions.size(0) || weights.size(1) != positions.size(1) ||
      weights.scalar_type() != at::kFloat || weights.device() != ys.device())
    bad("weights must be a float32 [T, k] tensor on the rows' device");
  const bool grad = at::GradMode::is_enabled();
  const bool need_rows = grad && ys.requires_grad(), need_weights = grad && weights.requires_grad();
  if (need_rows || need_weights)
    return MoeCombine::apply(ys, weights, sources, positions, need_rows, need_weights);
  const c10::cuda::CUDAGuard guard(ys.device());
  return combine_rows(ys, weights.contiguous(), positions);
}

// ---- AdamW over lists of tensors (cutie_adamw). The lists are read as Python
// sequences here: hundreds of tensors would cost more in argument conversion
// than in the kernel.
struct Sequence {
  PyObject* fast;
  explicit Sequence(PyObject* o, const char* name) : fast(PySequence_Fast(o, "")) {
    if (fast == nullptr) {
      PyErr_Clear();
      bad(std::string(name) + " must be a sequence of tensors");
    }
  }
  Sequence(const Sequence&) = delete;
  ~Sequence() { Py_DECREF(fast); }
  int64_t size() const { return PySequence_Fast_GET_SIZE(fast); }
  PyObject* operator[](int64_t i) const { return PySequence_Fast_GET_ITEM(fast, i); }
};

const at::Tensor& tensor_of(PyObject* o, const char* name) {
  if (!THPVariable_CheckExact(o) && !THPVariable_Check(o)) bad(std::string(name) + " must hold tensors");
  return THPVariable_Unpack(o);
}

// Addresses [first, second) of tensors. What a step writes must not overlap: it would be a
// race. A list in the order of its addresses (views of one buffer) is not sorted.
using Ranges = std::vector<std::pair<uintptr_t, uintptr_t>>;

bool in_order(const Ranges& ranges) {
  for (size_t i = 1; i < ranges.size(); ++i)
    if (ranges[i - 1].second > ranges[i].first) return false;
  return true;
}

void check_apart(Ranges& ranges, const char* name) {
  if (in_order(ranges)) return;
  std::sort(ranges.begin(), ranges.end());
  if (!in_order(ranges)) bad(std::string(name) + " must not overlap one another");
}

// The same between two lists in the order of their addresses, of which x may overlap itself.
bool apart(const Ranges& x, const Ranges& y) {
  for (size_t i = 0, j = 0; i < x.size() && j < y.size();) {
    if (y.back().second <= x[i].first) return true;
    if (x[i].second <= y[j].first) ++i;
    else if (y[j].second <= x[i].first) ++j;
    else return false;
  }
  return true;
}

// What a step writes, lists that are apart each, and what it reads.
void check_memory(Ranges& read, const std::vector<const Ranges*>& written) {
  for (size_t i = 0; i < written.size(); ++i)
    for (size_t j = 0; j < i; ++j)
      if (!apart(*written[i], *written[j]))
        bad("a parameter and its states must not share memory, nor with another's");
  if (!std::is_sorted(read.begin(), read.end())) std::sort(read.begin(), read.end());
  for (const Ranges* w : written)
    if (!apart(read, *w)) bad("grads must not share memory with parameters or states");
}

// A step or a rate: a number, or one element on the GPU.
const at::Tensor* device_scalar(PyObject* o, const char* name, at::ScalarType dtype, const at::Device& dev) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.numel() != 1 || t.scalar_type() != dtype || t.device() != dev)
    bad(std::string(name) + " must be a number or one " + (dtype == at::kLong ? "int64" : "float32") +
        " on the parameters' device");
  return &t;
}

void adamw_step(const py::object& params, const py::object& grads, const py::object& avgs, const py::object& sqs,
                const py::object& step, const py::object& lr, double beta1, double beta2, double eps,
                double weight_decay, const c10::optional<at::Tensor>& grad_scale, int64_t seed) {
  const Sequence P(params.ptr(), "params"), G(grads.ptr(), "grads"), M(avgs.ptr(), "exp_avgs"), V(sqs.ptr(), "exp_avg_sqs");
  const int64_t count = P.size();
  if (G.size() != count || M.size() != count || V.size() != count)
    bad("params, grads, exp_avgs and exp_avg_sqs must have the same length");
  if (count == 0) return;
  const at::Tensor& p0 = tensor_of(P[0], "params");
  const at::Tensor& g0 = tensor_of(G[0], "grads");
  if (!p0.is_cuda()) bad("params must be CUDA tensors (this library has no CPU path)");
  const at::Device dev = p0.device();
  const int p_dtype = row_dtype(p0, "params"), g_dtype = row_dtype(g0, "grads");
  const bool codes = PyTuple_Check(M[0]) || PyList_Check(M[0]);
  const c10::cuda::CUDAGuard guard(dev);
  std::vector<void*> p(count), m(count), v(count), ms, vs;
  std::vector<const void*> g(count);
  std::vector<int64_t> n(count);
  if (codes) ms.resize(count), vs.resize(count);
  std::vector<at::Tensor> copies;  // of gradients that are not dense
  Ranges rp, rg, rm, rv, rms, rvs;
  for (auto* r : {&rp, &rg, &rm, &rv, &rms, &rvs}) r->reserve(count);
  const auto range = [](Ranges& r, const at::Tensor& t) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(t.data_ptr());
    if (t.numel() > 0) r.emplace_back(a, a + t.numel() * t.element_size());
  };
  const auto state = [&](PyObject* o, int64_t i, const at::Tensor& param, const char* name, void** place, void** scale,
                         Ranges& r, Ranges& rs) {
    if ((PyTuple_Check(o) || PyList_Check(o)) != codes)
      bad("states are all tensors, or all pairs of codes and scales");
    if (!codes) {
      const at::Tensor& t = tensor_of(o, name);
      if (t.scalar_type() != at::kFloat || t.device() != dev || !t.is_contiguous() || t.sizes() != param.sizes())
        bad(std::string(name) + " must be contiguous float32 tensors of the parameters' shapes, on their device");
      *place = t.data_ptr();
      range(r, t);
      return;
    }
    const Sequence pair(o, name);
    if (pair.size() != 2) bad(std::string(name) + " must hold pairs of codes and scales");
    const at::Tensor &q = tensor_of(pair[0], name), &s = tensor_of(pair[1], name);
    if ((q.scalar_type() != at::kFloat8_e4m3fn && q.scalar_type() != at::kByte) || q.device() != dev ||
        !q.is_contiguous() || q.numel() != n[i])
      bad(std::string(name) + "'s codes must be contiguous float8_e4m3fn, one for each element of the parameter");
    if (s.scalar_type() != at::kFloat || s.device() != dev || !s.is_contiguous() || s.numel() != (n[i] + 127) / 128)
      bad(std::string(name) + "'s scales must be contiguous float32, one for each 128 elements");
    *place = q.data_ptr(), *scale = s.data_ptr();
    range(r, q);
    range(rs, s);
  };
  for (int64_t i = 0; i < count; ++i) {
    const at::Tensor &pt = tensor_of(P[i], "params"), &gt = tensor_of(G[i], "grads");
    if (pt.scalar_type() != p0.scalar_type() || gt.scalar_type() != g0.scalar_type())
      bad("all params must have one dtype, and all grads one");
    if (pt.device() != dev || gt.device() != dev) bad("params and grads must be on one device");
    if (!pt.is_contiguous()) bad("params must be contiguous");
    if (gt.sizes() != pt.sizes()) bad("grads must have the parameters' shapes");
    n[i] = pt.numel();
    p[i] = pt.data_ptr();
    range(rp, pt);
    if (gt.is_contiguous()) {
      g[i] = gt.data_ptr();
      range(rg, gt);
    } else {
      copies.push_back(gt.contiguous());
      g[i] = copies.back().data_ptr();
    }
    state(M[i], i, pt, "exp_avgs", &m[i], codes ? &ms[i] : nullptr, rm, rms);
    state(V[i], i, pt, "exp_avg_sqs", &v[i], codes ? &vs[i] : nullptr, rv, rvs);
  }
  check_apart(rp, "params");
  check_apart(rm, "exp_avgs");
  check_apart(rv, "exp_avg_sqs");
  check_apart(rms, "exp_avgs' scales");
  check_apart(rvs, "exp_avg_sqs' scales");
  check_memory(rg, {&rp, &rm, &rv, &rms, &rvs});
  const at::Tensor* st = device_scalar(step.ptr(), "step", at::kLong, dev);
  const at::Tensor* lt = device_scalar(lr.ptr(), "lr", at::kFloat, dev);
  if (grad_scale.has_value() &&
      (grad_scale->numel() != 1 || grad_scale->scalar_type() != at::kFloat || grad_scale->device() != dev))
    bad("grad_scale must be one float32 on the parameters' device");
  check_status(cutie_adamw(
      count, p.data(), p_dtype, g.data(), g_dtype, m.data(), codes ? ms.data() : nullptr, v.data(),
      codes ? vs.data() : nullptr, n.data(), st != nullptr ? 0 : step.cast<int64_t>(),
      st != nullptr ? st->data_ptr() : nullptr, lt != nullptr ? 0.0 : lr.cast<double>(),
      lt != nullptr ? lt->data_ptr() : nullptr, beta1, beta2, eps, weight_decay, ptr_or_null(grad_scale),
      (uint64_t)seed, at::cuda::getCurrentCUDAStream(dev.index()).stream()));
  // what autograd saved of the parameters is out of date
  for (int64_t i = 0; i < count; ++i) {
    const at::Tensor& t = THPVariable_Unpack(P[i]);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
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
  m.def("fp8_grouped_gemm", &fp8_grouped_gemm, py::arg("a"), py::arg("a_scale"), py::arg("b"), py::arg("b_scale"),
        py::arg("offsets"), py::arg("counts"), py::arg("align"), py::arg("out"), py::arg("out_f32"));
  m.def("fp8_grouped_linear", &fp8_grouped_linear, py::arg("x"), py::arg("weight"), py::arg("sources"),
        py::arg("offsets"), py::arg("counts"), py::arg("align"), py::arg("wq"), py::arg("ws"), py::arg("wqt"), py::arg("wst"));
  m.def("moe_plan_rows", &moe_plan_rows, py::arg("T"), py::arg("k"), py::arg("E"), py::arg("align"));
  m.def("moe_sort", &moe_sort, py::arg("ids"), py::arg("E"), py::arg("align"), py::arg("apart"));
  m.def("moe_permute", &moe_permute, py::arg("x"), py::arg("sources"), py::arg("positions"));
  m.def("moe_combine", &moe_combine, py::arg("rows"), py::arg("weights"), py::arg("sources"),
        py::arg("positions"));
  m.def("adamw_step", &adamw_step, py::arg("params"), py::arg("grads"), py::arg("exp_avgs"),
        py::arg("exp_avg_sqs"), py::arg("step"), py::arg("lr"), py::arg("beta1"), py::arg("beta2"), py::arg("eps"),
        py::arg("weight_decay"), py::arg("grad_scale"), py::arg("seed"));
  m.def("abi_version", []() { return cutie_abi_version(); });
}
