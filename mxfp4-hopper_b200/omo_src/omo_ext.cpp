// `omo` torch extension for the B200 library: the reference's operator names,
// argument names and checks (code/kernel/ops.cu:27-43), implemented as thin
// C++ host code over the C ABI of libmxfp4_b200.so (include/mxfp4_b200.h).
//
// Every op runs asynchronously on torch's current CUDA stream and writes into
// caller-allocated outputs, as the reference's ops do.  Argument errors raise
// RuntimeError (TORCH_CHECK), like the reference's CHECK_INPUT / CHECK_EQ.
// There is no CPU path: a CPU tensor is an error.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <nvtx3/nvToolsExt.h>
#include <torch/extension.h>

#include "mxfp4_b200.h"

namespace {

// NVTX range over one operator call (visible in Nsight Systems timelines next
// to the kernels it launches; costs nothing when no tool is attached).
struct OmoRange {
  explicit OmoRange(const char* name) { nvtxRangePushA(name); }
  ~OmoRange() { nvtxRangePop(); }
};

#define OMO_CHECK_INPUT(x)                                               \
  TORCH_CHECK((x).is_cuda(), #x " must be a CUDA tensor");               \
  TORCH_CHECK((x).is_contiguous(), #x " must be contiguous")

mxb_stream_t cur_stream() {
  return reinterpret_cast<mxb_stream_t>(at::cuda::getCurrentCUDAStream().stream());
}

void check_status(mxb_status s, const char* op) {
  TORCH_CHECK(s == MXB_OK, op, ": ", mxb_last_error());
}

void check_dtype(const at::Tensor& t, at::ScalarType st, const char* name) {
  TORCH_CHECK(t.scalar_type() == st, name, " must have dtype ", c10::toString(st), ", got ",
              c10::toString(t.scalar_type()));
}

// ---- per_token_quant_mxfp4.cu:387-487
void omo_per_token_group_quant_fp4(at::Tensor input, at::Tensor output_q, at::Tensor output_s,
                                   int64_t group_size, double eps, double fp4_min, double fp4_max,
                                   bool scale_ue8m0) {
  OmoRange nvtx_range("omo_per_token_group_quant_fp4");
  OMO_CHECK_INPUT(input);
  OMO_CHECK_INPUT(output_q);
  TORCH_CHECK(input.numel() % group_size == 0, "CHECK_EQ(input.numel() % group_size, 0) failed");
  TORCH_CHECK(output_s.dim() == 2, "CHECK_EQ(output_s.dim(), 2) failed");
  check_dtype(input, at::kBFloat16, "input");
  check_dtype(output_q, at::kByte, "output_q");
  check_dtype(output_s, at::kByte, "output_s");
  TORCH_CHECK(output_s.is_contiguous() && output_s.is_cuda(),
              "output_s must be a contiguous CUDA tensor (row-major scales)");
  if (input.numel() == 0) return;
  const int64_t K = input.size(-1), M = input.numel() / K;
  TORCH_CHECK(output_q.numel() == M * K / 2, "output_q must hold numel/2 bytes");
  // The reference writes group g's scale at output_s.data_ptr() + g whatever the
  // tensor's shape (per_token_quant_mxfp4.cu:161), and its fp4 wrapper sizes
  // output_s from the code shape, [M, K/2] (api/mxfp4.py:106-111): any
  // contiguous buffer of at least numel/32 bytes is accepted and the scales
  // fill its first numel/32 bytes.
  TORCH_CHECK(output_s.numel() >= M * K / 32, "output_s must hold numel/32 scales");
  c10::cuda::CUDAGuard g(input.device());
  check_status(mxb_per_token_group_quant_fp4(input.data_ptr(), M, K, K, output_q.data_ptr(),
                                             output_s.data_ptr(), (int)group_size, (float)eps,
                                             (float)fp4_min, (float)fp4_max, scale_ue8m0 ? 1 : 0,
                                             cur_stream()),
               "omo_per_token_group_quant_fp4");
}

// ---- per_token_Mxfp4ToBf16_dequant.cu:164-240.  The reference indexes codes
// and scales as flat arrays (element i uses scale i/32), so the op is launched
// over the flattened tensors.  output_s is accepted and left untouched, as on
// the reference (per_token_Mxfp4ToBf16_dequant.cu:122).
void omo_per_token_Mxfp4ToBf16_dequant(at::Tensor input, at::Tensor input_s, at::Tensor output_q,
                                       at::Tensor output_s, int64_t group_size, double eps,
                                       double fp4_min, double fp4_max, bool scale_ue8m0) {
  OmoRange nvtx_range("omo_per_token_Mxfp4ToBf16_dequant");
  (void)group_size; (void)eps; (void)fp4_min; (void)fp4_max;
  OMO_CHECK_INPUT(input);
  OMO_CHECK_INPUT(output_q);
  TORCH_CHECK(input.numel() % 128 == 0, "CHECK_EQ(input.numel() % group_size, 0) failed (group_size is 128)");
  TORCH_CHECK(output_s.dim() == 2, "CHECK_EQ(output_s.dim(), 2) failed");
  TORCH_CHECK(!scale_ue8m0, "scale_ue8m0=True is not supported (reference host assert)");
  check_dtype(input, at::kByte, "input");
  check_dtype(input_s, at::kByte, "input_s");
  check_dtype(output_q, at::kBFloat16, "output_q");
  OMO_CHECK_INPUT(input_s);
  const int64_t n = input.numel();
  if (n == 0) return;
  TORCH_CHECK(input_s.numel() >= n / 16, "input_s must hold one scale per 16 code bytes");
  TORCH_CHECK(output_q.numel() >= 2 * n, "output_q must hold 2 elements per code byte");
  c10::cuda::CUDAGuard g(input.device());
  check_status(mxb_per_token_Mxfp4ToBf16_dequant(input.data_ptr(), input_s.data_ptr(), 1, n,
                                                 output_q.data_ptr(), cur_stream()),
               "omo_per_token_Mxfp4ToBf16_dequant");
}

void mxfp4_to_fp8_row_common(at::Tensor& input, at::Tensor& input_s, at::Tensor& output_q,
                             at::Tensor& output_s, bool scale_ue8m0, const char* op) {
  OMO_CHECK_INPUT(input);
  OMO_CHECK_INPUT(output_q);
  OMO_CHECK_INPUT(input_s);
  TORCH_CHECK(input.numel() % 128 == 0, "CHECK_EQ(input.numel() % group_size, 0) failed (group_size is 128)");
  TORCH_CHECK(output_s.dim() == 2, "CHECK_EQ(output_s.dim(), 2) failed");
  TORCH_CHECK(!scale_ue8m0, "scale_ue8m0=True is not supported (reference host assert)");
  TORCH_CHECK(input.dim() == 2, op, ": input must be 2-D [M, K/2]");
  check_dtype(input, at::kByte, "input");
  check_dtype(input_s, at::kByte, "input_s");
  check_dtype(output_q, at::kFloat8_e4m3fn, "output_q");
  check_dtype(output_s, at::kFloat, "output_s");
  TORCH_CHECK(output_s.is_contiguous() && output_s.is_cuda(), "output_s must be a contiguous CUDA tensor");
  const int64_t M = input.size(0), Kb = input.size(1);
  if (M == 0 || Kb == 0) return;
  TORCH_CHECK(Kb % 64 == 0, op, ": the code row must be a multiple of 64 bytes (1x128 groups); "
              "the Python wrapper pads it");
  TORCH_CHECK(input_s.numel() >= M * Kb / 16, op, ": input_s too small");
  TORCH_CHECK(output_q.numel() == 2 * M * Kb, op, ": output_q must be [M, 2*K]");
  TORCH_CHECK(output_s.numel() == M * Kb / 64, op, ": output_s must be [K/64, M]");
  c10::cuda::CUDAGuard g(input.device());
  check_status(mxb_per_token_Mxfp4ToFp8(input.data_ptr(), input_s.data_ptr(), M, Kb,
                                        output_q.data_ptr(), output_s.data_ptr(), cur_stream()),
               op);
}

// ---- per_token_Mxfp4ToFp8.cu:239-310
void omo_per_token_Mxfp4ToFp8(at::Tensor input, at::Tensor input_s, at::Tensor output_q,
                              at::Tensor output_s, int64_t group_size, double eps, double fp4_min,
                              double fp4_max, bool scale_ue8m0) {
  OmoRange nvtx_range("omo_per_token_Mxfp4ToFp8");
  (void)group_size; (void)eps; (void)fp4_min; (void)fp4_max;
  mxfp4_to_fp8_row_common(input, input_s, output_q, output_s, scale_ue8m0,
                          "omo_per_token_Mxfp4ToFp8");
}

// ---- ops.cu:32 binds this name; its source is not in the reference.  Same
// operation as omo_per_token_Mxfp4ToFp8.
void omo_per_token_Mxfp4ToBf16ToFp8(at::Tensor input, at::Tensor input_s, at::Tensor output_q,
                                    at::Tensor output_s, int64_t group_size, double eps,
                                    double fp4_min, double fp4_max, bool scale_ue8m0) {
  OmoRange nvtx_range("omo_per_token_Mxfp4ToBf16ToFp8");
  (void)group_size; (void)eps; (void)fp4_min; (void)fp4_max;
  mxfp4_to_fp8_row_common(input, input_s, output_q, output_s, scale_ue8m0,
                          "omo_per_token_Mxfp4ToBf16ToFp8");
}

// ---- ops.cu:34 binds this name; its source is not in the reference.  Q-row
// into (output_q, output_s), then the rowwise FP8 convert of that result into
// (output_bf16_q [M, K] fp8, output_bf16_s [K/128, M] float).
void omo_per_token_group_quant_fp4_fused_ToFp8(at::Tensor input, at::Tensor output_q,
                                               at::Tensor output_s, at::Tensor output_bf16_q,
                                               at::Tensor output_bf16_s, int64_t group_size,
                                               double eps, double fp4_min, double fp4_max,
                                               bool scale_ue8m0) {
  OmoRange nvtx_range("omo_per_token_group_quant_fp4_fused_ToFp8");
  // the checks of both halves (omo_per_token_group_quant_fp4 and omo_per_token_Mxfp4ToFp8)
  OMO_CHECK_INPUT(input);
  OMO_CHECK_INPUT(output_q);
  OMO_CHECK_INPUT(output_bf16_q);
  TORCH_CHECK(input.numel() % group_size == 0, "CHECK_EQ(input.numel() % group_size, 0) failed");
  TORCH_CHECK(output_s.dim() == 2 && output_bf16_s.dim() == 2, "CHECK_EQ(output_s.dim(), 2) failed");
  check_dtype(input, at::kBFloat16, "input");
  check_dtype(output_q, at::kByte, "output_q");
  check_dtype(output_s, at::kByte, "output_s");
  check_dtype(output_bf16_q, at::kFloat8_e4m3fn, "output_bf16_q");
  check_dtype(output_bf16_s, at::kFloat, "output_bf16_s");
  TORCH_CHECK(output_s.is_contiguous() && output_s.is_cuda() && output_bf16_s.is_contiguous() &&
                  output_bf16_s.is_cuda(),
              "scale outputs must be contiguous CUDA tensors");
  if (input.numel() == 0) return;
  const int64_t K = input.size(-1), M = input.numel() / K;
  TORCH_CHECK(K % 128 == 0, "omo_per_token_group_quant_fp4_fused_ToFp8: K must be a multiple of "
              "128 (1x128 FP8 groups)");
  TORCH_CHECK(output_q.numel() == M * K / 2, "output_q must hold numel/2 bytes");
  TORCH_CHECK(output_s.numel() >= M * K / 32, "output_s must hold numel/32 scales");
  TORCH_CHECK(output_bf16_q.numel() == M * K, "output_bf16_q must be [M, K]");
  TORCH_CHECK(output_bf16_s.numel() == M * K / 128, "output_bf16_s must be [K/128, M]");
  c10::cuda::CUDAGuard g(input.device());
  check_status(mxb_per_token_group_quant_fp4_fused_ToFp8(
                   input.data_ptr(), M, K, K, output_q.data_ptr(), output_s.data_ptr(),
                   output_bf16_q.data_ptr(), output_bf16_s.data_ptr(), (int)group_size, (float)eps,
                   (float)fp4_min, (float)fp4_max, scale_ue8m0 ? 1 : 0, cur_stream()),
               "omo_per_token_group_quant_fp4_fused_ToFp8");
}

// ---- per_token_Mxfp4ToFp8_col.cu:305-384
void omo_per_token_Mxfp4ToFp8_col(at::Tensor input, at::Tensor input_s, at::Tensor output_q,
                                  at::Tensor output_s, int64_t group_size, double eps,
                                  double fp4_min, double fp4_max, bool scale_ue8m0) {
  OmoRange nvtx_range("omo_per_token_Mxfp4ToFp8_col");
  (void)group_size; (void)eps; (void)fp4_min; (void)fp4_max;
  OMO_CHECK_INPUT(input);
  OMO_CHECK_INPUT(output_q);
  OMO_CHECK_INPUT(input_s);
  TORCH_CHECK(input.numel() % 128 == 0, "CHECK_EQ(input.numel() % group_size, 0) failed (group_size is 128)");
  TORCH_CHECK(output_s.dim() == 2, "CHECK_EQ(output_s.dim(), 2) failed");
  TORCH_CHECK(!scale_ue8m0, "scale_ue8m0=True is not supported (reference host assert)");
  TORCH_CHECK(input.dim() == 2, "input must be 2-D [M, K/2]");
  check_dtype(input, at::kByte, "input");
  check_dtype(input_s, at::kByte, "input_s");
  check_dtype(output_q, at::kFloat8_e4m3fn, "output_q");
  check_dtype(output_s, at::kFloat, "output_s");
  const int64_t M = input.size(0), Kb = input.size(1);
  if (M == 0 || Kb == 0) return;
  TORCH_CHECK(M % 128 == 0 && Kb % 128 == 0,
              "omo_per_token_Mxfp4ToFp8_col: M and the code row length must be multiples of 128 "
              "(the reference kernel tiles 128x128 bytes without bounds checks)");
  TORCH_CHECK(input_s.numel() == M * Kb / 16, "input_s must be [M, K/16]");
  TORCH_CHECK(output_q.numel() == 2 * M * Kb, "output_q must be [2*K, M]");
  TORCH_CHECK(output_s.numel() == (M / 128) * 2 * Kb, "output_s must be [M/128, 2*K]");
  c10::cuda::CUDAGuard g(input.device());
  check_status(mxb_per_token_Mxfp4ToFp8_col(input.data_ptr(), input_s.data_ptr(), M, Kb,
                                            output_q.data_ptr(), output_s.data_ptr(), cur_stream()),
               "omo_per_token_Mxfp4ToFp8_col");
}

// ---- per_token_Mxfp4RowToBf16ToFp8Col.cu:204-247 (same shape checks)
void omo_per_token_Mxfp4RowToBf16ToFp8Col(at::Tensor input, at::Tensor input_s,
                                          at::Tensor output_q, at::Tensor output_s, double eps) {
  OmoRange nvtx_range("omo_per_token_Mxfp4RowToBf16ToFp8Col");
  OMO_CHECK_INPUT(input);
  OMO_CHECK_INPUT(output_q);
  TORCH_CHECK(input.dim() == 2, "CHECK_EQ(input.dim(), 2) failed");
  TORCH_CHECK(output_q.dim() == 2, "CHECK_EQ(output_q.dim(), 2) failed");
  const int64_t M = input.size(0), N = input.size(1) * 2;
  TORCH_CHECK(input_s.size(0) == M, "CHECK_EQ(input_s.size(0), M) failed");
  TORCH_CHECK(input_s.size(1) == (N + 31) / 32, "CHECK_EQ(input_s.size(1), (N + 31) / 32) failed");
  TORCH_CHECK(output_q.size(0) == N, "CHECK_EQ(output_q.size(0), N) failed");
  TORCH_CHECK(output_q.size(1) == M, "CHECK_EQ(output_q.size(1), M) failed");
  TORCH_CHECK(output_s.size(0) == (M + 127) / 128, "CHECK_EQ(output_s.size(0), (M + 127) / 128) failed");
  TORCH_CHECK(output_s.size(1) == N, "CHECK_EQ(output_s.size(1), N) failed");
  check_dtype(input, at::kByte, "input");
  check_dtype(input_s, at::kByte, "input_s");
  check_dtype(output_q, at::kFloat8_e4m3fn, "output_q");
  check_dtype(output_s, at::kFloat, "output_s");
  OMO_CHECK_INPUT(input_s);
  OMO_CHECK_INPUT(output_s);
  if (M == 0 || N == 0) return;
  c10::cuda::CUDAGuard g(input.device());
  check_status(mxb_per_token_Mxfp4RowToBf16ToFp8Col(input.data_ptr(), input_s.data_ptr(), M, N,
                                                    output_q.data_ptr(), output_s.data_ptr(),
                                                    (float)eps, cur_stream()),
               "omo_per_token_Mxfp4RowToBf16ToFp8Col");
}

// ---- per_token_Mxfp4RowToBf16ToFp8Col_msplit.cu:232-282
void omo_per_token_Mxfp4RowToBf16ToFp8Col_msplit(at::Tensor input, at::Tensor input_s,
                                                 at::Tensor output_q, at::Tensor output_s,
                                                 at::Tensor m_splits, at::Tensor split_offsets,
                                                 at::Tensor scale_offsets, int64_t max_split_len,
                                                 double eps) {
  OmoRange nvtx_range("omo_per_token_Mxfp4RowToBf16ToFp8Col_msplit");
  OMO_CHECK_INPUT(input);
  OMO_CHECK_INPUT(output_q);
  OMO_CHECK_INPUT(m_splits);
  OMO_CHECK_INPUT(split_offsets);
  OMO_CHECK_INPUT(scale_offsets);
  OMO_CHECK_INPUT(input_s);
  OMO_CHECK_INPUT(output_s);
  check_dtype(input, at::kByte, "input");
  check_dtype(input_s, at::kByte, "input_s");
  check_dtype(output_q, at::kFloat8_e4m3fn, "output_q");
  check_dtype(output_s, at::kFloat, "output_s");
  check_dtype(m_splits, at::kInt, "m_splits");
  check_dtype(split_offsets, at::kInt, "split_offsets");
  check_dtype(scale_offsets, at::kInt, "scale_offsets");
  const int64_t total_M = input.size(0), N = input.size(1) * 2;
  const int64_t ns = m_splits.size(0);
  TORCH_CHECK(split_offsets.numel() >= ns && scale_offsets.numel() >= ns,
              "split_offsets / scale_offsets must have one entry per split");
  if (total_M == 0 || N == 0 || ns == 0) return;
  c10::cuda::CUDAGuard g(input.device());
  check_status(mxb_per_token_Mxfp4RowToBf16ToFp8Col_msplit(
                   input.data_ptr(), input_s.data_ptr(), total_M, N, output_q.data_ptr(),
                   output_s.data_ptr(), m_splits.data_ptr<int32_t>(),
                   split_offsets.data_ptr<int32_t>(), scale_offsets.data_ptr<int32_t>(), ns,
                   max_split_len, (float)eps, cur_stream()),
               "omo_per_token_Mxfp4RowToBf16ToFp8Col_msplit");
}

// ---- additions with no reference op of their own -------------------------
// One-pass rowwise + columnwise quantize (the reference runs Q-row on x and on
// x.T.contiguous(): transformer_engine-2.8.diff:1464-1466).  Pass empty
// tensors for the row outputs to quantize columnwise only.
void omo_quant_mxfp4_rowcol(at::Tensor input, at::Tensor codes_row, at::Tensor scales_row,
                            at::Tensor codes_col, at::Tensor scales_col,
                            c10::optional<at::Tensor> scales_row_swizzled, double eps,
                            double fp4_min, double fp4_max) {
  OmoRange nvtx_range("omo_quant_mxfp4_rowcol");
  OMO_CHECK_INPUT(input);
  check_dtype(input, at::kBFloat16, "input");
  TORCH_CHECK(input.dim() == 2, "input must be 2-D");
  const int64_t M = input.size(0), K = input.size(1);
  const bool rows = codes_row.numel() > 0;
  if (rows) {
    OMO_CHECK_INPUT(codes_row);
    OMO_CHECK_INPUT(scales_row);
    TORCH_CHECK(codes_row.numel() == M * K / 2 && scales_row.numel() == M * K / 32,
                "row outputs must be [M, K/2] and [M, K/32]");
  }
  OMO_CHECK_INPUT(codes_col);
  OMO_CHECK_INPUT(scales_col);
  TORCH_CHECK(codes_col.numel() == M * K / 2 && scales_col.numel() == M * K / 32,
              "column outputs must be [K, M/2] and [K, M/32]");
  void* swz = nullptr;
  if (scales_row_swizzled.has_value() && scales_row_swizzled->numel() > 0) {
    OMO_CHECK_INPUT((*scales_row_swizzled));
    TORCH_CHECK(scales_row_swizzled->numel() == (M + 127) / 128 * 128 * ((K / 32 + 3) / 4 * 4),
                "swizzled scales must be [round_up(M,128), round_up(K/32,4)]");
    swz = scales_row_swizzled->data_ptr();
  }
  if (M == 0 || K == 0) return;
  c10::cuda::CUDAGuard g(input.device());
  check_status(mxb_quant_mxfp4_rowcol(input.data_ptr(), M, K, K,
                                      rows ? codes_row.data_ptr() : nullptr,
                                      rows ? scales_row.data_ptr() : nullptr, codes_col.data_ptr(),
                                      scales_col.data_ptr(), swz, (float)eps, (float)fp4_min,
                                      (float)fp4_max, cur_stream()),
               "omo_quant_mxfp4_rowcol");
}

void omo_swizzle_scales(at::Tensor scales, at::Tensor out) {
  OmoRange nvtx_range("omo_swizzle_scales");
  OMO_CHECK_INPUT(scales);
  OMO_CHECK_INPUT(out);
  TORCH_CHECK(scales.dim() == 2, "scales must be 2-D");
  const int64_t M = scales.size(0), S = scales.size(1);
  TORCH_CHECK(out.numel() == (M + 127) / 128 * 128 * ((S + 3) / 4 * 4),
              "out must be [round_up(M,128), round_up(S,4)]");
  c10::cuda::CUDAGuard g(scales.device());
  check_status(mxb_swizzle_scales(scales.data_ptr(), M, S, out.data_ptr(), cur_stream()),
               "omo_swizzle_scales");
}

void omo_per_token_quant_fp8(at::Tensor input, at::Tensor output_q, at::Tensor output_s,
                             double eps) {
  OmoRange nvtx_range("omo_per_token_quant_fp8");
  OMO_CHECK_INPUT(input);
  OMO_CHECK_INPUT(output_q);
  OMO_CHECK_INPUT(output_s);
  check_dtype(input, at::kBFloat16, "input");
  check_dtype(output_q, at::kFloat8_e4m3fn, "output_q");
  check_dtype(output_s, at::kFloat, "output_s");
  if (input.numel() == 0) return;
  const int64_t K = input.size(-1), M = input.numel() / K;
  TORCH_CHECK(output_q.numel() == M * K && output_s.numel() == M, "bad output sizes");
  c10::cuda::CUDAGuard g(input.device());
  check_status(mxb_per_token_quant_fp8(input.data_ptr(), M, K, output_q.data_ptr(),
                                       output_s.data_ptr(), (float)eps, cur_stream()),
               "omo_per_token_quant_fp8");
}

void omo_per_token_dequant_fp8(at::Tensor input_q, at::Tensor input_s, at::Tensor output) {
  OmoRange nvtx_range("omo_per_token_dequant_fp8");
  OMO_CHECK_INPUT(input_q);
  OMO_CHECK_INPUT(input_s);
  OMO_CHECK_INPUT(output);
  check_dtype(input_q, at::kFloat8_e4m3fn, "input_q");
  check_dtype(input_s, at::kFloat, "input_s");
  check_dtype(output, at::kBFloat16, "output");
  if (input_q.numel() == 0) return;
  const int64_t K = input_q.size(-1), M = input_q.numel() / K;
  TORCH_CHECK(output.numel() == M * K && input_s.numel() == M, "bad sizes");
  c10::cuda::CUDAGuard g(input_q.device());
  check_status(mxb_per_token_dequant_fp8(input_q.data_ptr(), input_s.data_ptr(), M, K,
                                         output.data_ptr(), cur_stream()),
               "omo_per_token_dequant_fp8");
}

// ---- operators with no reference binding: the next rows of the path
void omo_swiglu_quant_mxfp4(at::Tensor input, at::Tensor output, at::Tensor codes,
                            at::Tensor scales, double eps, double fp4_min, double fp4_max) {
  OmoRange nvtx_range("omo_swiglu_quant_mxfp4");
  OMO_CHECK_INPUT(input);
  OMO_CHECK_INPUT(output);
  OMO_CHECK_INPUT(codes);
  OMO_CHECK_INPUT(scales);
  check_dtype(input, at::kBFloat16, "input");
  check_dtype(output, at::kBFloat16, "output");
  check_dtype(codes, at::kByte, "codes");
  check_dtype(scales, at::kByte, "scales");
  if (input.numel() == 0) return;
  const int64_t K = input.size(-1), M = input.numel() / K;
  TORCH_CHECK(K % 64 == 0, "omo_swiglu_quant_mxfp4: the last dimension (2H) must be a multiple of 64");
  TORCH_CHECK(output.numel() == M * K / 2 && codes.numel() == M * K / 2 &&
                  scales.numel() == M * K / 32,
              "omo_swiglu_quant_mxfp4: output [.., H], codes [.., H], scales [rows, 2H/32]");
  c10::cuda::CUDAGuard g(input.device());
  check_status(mxb_swiglu_quant_mxfp4(input.data_ptr(), M, K / 2, output.data_ptr(),
                                      codes.data_ptr(), scales.data_ptr(), (float)eps,
                                      (float)fp4_min, (float)fp4_max, cur_stream()),
               "omo_swiglu_quant_mxfp4");
}

void omo_moe_permute_mxfp4(at::Tensor codes, at::Tensor scales, at::Tensor dst,
                           at::Tensor out_codes, at::Tensor out_scales) {
  OmoRange nvtx_range("omo_moe_permute_mxfp4");
  OMO_CHECK_INPUT(codes);
  OMO_CHECK_INPUT(scales);
  OMO_CHECK_INPUT(dst);
  OMO_CHECK_INPUT(out_codes);
  OMO_CHECK_INPUT(out_scales);
  check_dtype(codes, at::kByte, "codes");
  check_dtype(scales, at::kByte, "scales");
  check_dtype(dst, at::kInt, "dst");
  TORCH_CHECK(codes.dim() == 2 && scales.dim() == 2 && dst.dim() == 2 &&
                  codes.size(0) == scales.size(0) && dst.size(0) == codes.size(0),
              "omo_moe_permute_mxfp4: codes [rows, H/2], scales [rows, H/32], dst [rows, topk]");
  const int64_t rows = codes.size(0), H = codes.size(1) * 2;
  TORCH_CHECK(scales.size(1) * 32 == H, "omo_moe_permute_mxfp4: scales must be [rows, H/32]");
  TORCH_CHECK(out_codes.dim() == 2 && out_codes.size(1) == H / 2 && out_scales.dim() == 2 &&
                  out_scales.size(1) == H / 32 && out_scales.size(0) == out_codes.size(0),
              "omo_moe_permute_mxfp4: out_codes [n_out, H/2], out_scales [n_out, H/32]");
  if (rows == 0) return;
  c10::cuda::CUDAGuard g(codes.device());
  check_status(mxb_moe_permute_mxfp4(codes.data_ptr(), H / 2, scales.data_ptr(), H / 32, rows, H,
                                     (const int32_t*)dst.data_ptr(), (int)dst.size(1),
                                     out_codes.data_ptr(), out_scales.data_ptr(),
                                     out_codes.size(0), cur_stream()),
               "omo_moe_permute_mxfp4");
}

void omo_gemm_mxfp4(at::Tensor a_codes, at::Tensor a_scales_swizzled, at::Tensor b_codes,
                    at::Tensor b_scales_swizzled, at::Tensor c) {
  OmoRange nvtx_range("omo_gemm_mxfp4");
  OMO_CHECK_INPUT(a_codes);
  OMO_CHECK_INPUT(a_scales_swizzled);
  OMO_CHECK_INPUT(b_codes);
  OMO_CHECK_INPUT(b_scales_swizzled);
  OMO_CHECK_INPUT(c);
  check_dtype(a_codes, at::kByte, "a_codes");
  check_dtype(b_codes, at::kByte, "b_codes");
  check_dtype(c, at::kBFloat16, "c");
  TORCH_CHECK(a_codes.dim() == 2 && b_codes.dim() == 2 && a_codes.size(1) == b_codes.size(1),
              "omo_gemm_mxfp4: a_codes [M, K/2] and b_codes [N, K/2]");
  const int64_t M = a_codes.size(0), N = b_codes.size(0), K = a_codes.size(1) * 2;
  TORCH_CHECK(c.numel() == M * N, "omo_gemm_mxfp4: c must be [M, N]");
  TORCH_CHECK(a_scales_swizzled.numel() == M * K / 32 && b_scales_swizzled.numel() == N * K / 32,
              "omo_gemm_mxfp4: swizzled scales must hold rows * K/32 bytes");
  c10::cuda::CUDAGuard g(a_codes.device());
  check_status(mxb_gemm_mxfp4(a_codes.data_ptr(), a_scales_swizzled.data_ptr(), b_codes.data_ptr(),
                              b_scales_swizzled.data_ptr(), M, N, K, c.data_ptr(), cur_stream()),
               "omo_gemm_mxfp4");
}

// ---- MXFP4 experts (no reference counterpart)

using OptTensor = c10::optional<at::Tensor>;

// Row-major rows at any pitch: the last dimension contiguous.
void check_rows(const at::Tensor& x, const char* name, int64_t rows, int64_t cols,
                at::ScalarType st, const at::Tensor& like) {
  TORCH_CHECK(x.is_cuda() && x.device() == like.device(), name, " must be on ", like.device());
  check_dtype(x, st, name);
  TORCH_CHECK(x.dim() == 2 && x.size(0) == rows && x.size(1) == cols, name, " must be [", rows,
              ", ", cols, "], got ", x.sizes());
  TORCH_CHECK((x.stride(1) == 1 || cols <= 1) && (x.stride(0) >= cols || rows <= 1), name,
              " must have contiguous rows");
}
int64_t pitch(const at::Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

void check_dense(const at::Tensor& x, const char* name, at::IntArrayRef sizes, at::ScalarType st,
                 const at::Tensor& like) {
  TORCH_CHECK(x.is_cuda() && x.device() == like.device(), name, " must be on ", like.device());
  check_dtype(x, st, name);
  TORCH_CHECK(x.sizes() == sizes && x.is_contiguous(), name, " must be a contiguous ", sizes,
              ", got ", x.sizes());
}

const int32_t* check_splits(const OptTensor& m_splits, int64_t E, const at::Tensor& like) {
  if (!m_splits) {
    TORCH_CHECK(E == 1, "m_splits is needed for more than one expert");
    return nullptr;
  }
  check_dense(*m_splits, "m_splits", {E}, at::kInt, like);
  return (const int32_t*)m_splits->data_ptr();
}
void* opt_ptr(const OptTensor& x) { return x ? x->data_ptr() : nullptr; }

void omo_swizzle_scales_grouped(at::Tensor scales, int64_t parts, at::Tensor out) {
  OmoRange nvtx_range("omo_swizzle_scales_grouped");
  OMO_CHECK_INPUT(scales);
  check_dtype(scales, at::kByte, "scales");
  TORCH_CHECK(scales.dim() == 3, "scales must be [E, N, K/32]");
  TORCH_CHECK(parts == 1 || parts == 2, "parts must be 1 or 2");
  const int64_t E = scales.size(0), N = scales.size(1), S = scales.size(2);
  TORCH_CHECK(N % parts == 0, "N must be a multiple of parts");
  check_dense(out, "out", {E, parts * ((N / parts + 127) / 128 * 128), (S + 3) / 4 * 4}, at::kByte,
              scales);
  c10::cuda::CUDAGuard g(scales.device());
  check_status(mxb_swizzle_scales_grouped(scales.data_ptr(), E, N, S, (int32_t)parts,
                                          out.data_ptr(), cur_stream()),
               "omo_swizzle_scales_grouped");
}

// b_codes [E, N, K/2], or [N, K/2] for a dense layer (then b_scales and bias lack the
// leading dimension too).
void omo_grouped_gemm_mxfp4(const at::Tensor& a_codes, const at::Tensor& a_scales,
                            const OptTensor& m_splits, const at::Tensor& b_codes,
                            const at::Tensor& b_scales, const OptTensor& c, const OptTensor& bias,
                            int64_t activation, const OptTensor& residual, const OptTensor& pre,
                            const OptTensor& c_codes, const OptTensor& c_scales) {
  OmoRange nvtx_range("omo_grouped_gemm_mxfp4");
  OMO_CHECK_INPUT(b_codes);
  check_dtype(b_codes, at::kByte, "b_codes");
  const bool dense = b_codes.dim() == 2;
  TORCH_CHECK(dense || b_codes.dim() == 3, "b_codes must be [E, N, K/2] or [N, K/2]");
  TORCH_CHECK(a_codes.dim() == 2, "a_codes must be [M, K/2]");
  TORCH_CHECK(activation >= MXB_ACT_NONE && activation <= MXB_ACT_SWIGLU, "unknown activation");
  const int64_t E = dense ? 1 : b_codes.size(0), N = b_codes.size(-2), K = b_codes.size(-1) * 2;
  const int64_t M = a_codes.size(0), parts = activation == MXB_ACT_SWIGLU ? 2 : 1, W = N / parts;
  TORCH_CHECK(E >= 1 && N % parts == 0 && K % 32 == 0, "b_codes must be [E, N, K/2] with K % 32 == 0");
  check_rows(a_codes, "a_codes", M, K / 2, at::kByte, b_codes);
  check_rows(a_scales, "a_scales", M, K / 32, at::kByte, b_codes);
  const int64_t tiled[3] = {E, parts * ((W + 127) / 128 * 128), (K / 32 + 3) / 4 * 4};
  check_dense(b_scales, "b_scales", at::IntArrayRef(tiled + dense, 3 - dense), at::kByte, b_codes);
  mxb_epilogue ep = {};
  ep.activation = (int32_t)activation;
  if (bias) {
    ep.bias_f32 = bias->scalar_type() == at::kFloat;
    const int64_t each[2] = {E, N};
    check_dense(*bias, "bias", at::IntArrayRef(each + dense, 2 - dense),
                ep.bias_f32 ? at::kFloat : at::kBFloat16, b_codes);
    ep.bias = bias->data_ptr();
  }
  if (residual) {
    check_rows(*residual, "residual", M, W, at::kBFloat16, b_codes);
    ep.residual = residual->data_ptr();
    ep.residual_ld = pitch(*residual);
  }
  if (pre) {
    check_rows(*pre, "pre", M, N, at::kBFloat16, b_codes);
    ep.pre = pre->data_ptr();
    ep.pre_ld = pitch(*pre);
  }
  if (c) {
    check_rows(*c, "c", M, W, at::kBFloat16, b_codes);
    ep.c_ld = pitch(*c);
  }
  TORCH_CHECK(c_codes.has_value() == c_scales.has_value(), "c_codes and c_scales go together");
  if (c_codes) {
    TORCH_CHECK(W % 32 == 0, "a quantized result needs a width that is a multiple of 32");
    check_dense(*c_codes, "c_codes", {M, W / 2}, at::kByte, b_codes);
    check_dense(*c_scales, "c_scales", {M, W / 32}, at::kByte, b_codes);
    ep.c_codes = c_codes->data_ptr();
    ep.c_scales = c_scales->data_ptr();
  }
  const int32_t* splits = check_splits(m_splits, E, b_codes);
  c10::cuda::CUDAGuard g(b_codes.device());
  check_status(mxb_grouped_gemm_mxfp4(a_codes.data_ptr(), pitch(a_codes), a_scales.data_ptr(),
                                      pitch(a_scales), M, splits, (int32_t)E, b_codes.data_ptr(),
                                      b_scales.data_ptr(), N, K, &ep, opt_ptr(c), cur_stream()),
               "omo_grouped_gemm_mxfp4");
}

// The same with the results allocated here (a call from Python that allocates them
// one by one costs several microseconds more, as much as a decoding step's kernel):
// returns those of (c, pre, c_codes, c_scales) that are asked for.
std::vector<at::Tensor> omo_grouped_gemm_mxfp4_new(
    const at::Tensor& a_codes, const at::Tensor& a_scales, const OptTensor& m_splits,
    const at::Tensor& b_codes, const at::Tensor& b_scales, const OptTensor& bias,
    int64_t activation, const OptTensor& residual, bool save_pre, bool quantize, bool bf16_out) {
  TORCH_CHECK(a_codes.dim() == 2 && b_codes.dim() >= 2, "a_codes [M, K/2], b_codes [.., N, K/2]");
  TORCH_CHECK(bf16_out || save_pre || quantize, "no result is asked for");
  const int64_t M = a_codes.size(0), N = b_codes.size(-2);
  const int64_t W = activation == MXB_ACT_SWIGLU ? N / 2 : N;
  const auto bf16 = a_codes.options().dtype(at::kBFloat16);
  OptTensor c, pre, q, s;
  std::vector<at::Tensor> out;
  if (bf16_out) out.push_back(*(c = at::empty({M, W}, bf16)));
  if (save_pre) out.push_back(*(pre = at::empty({M, N}, bf16)));
  if (quantize) {
    out.push_back(*(q = at::empty({M, W / 2}, a_codes.options())));
    out.push_back(*(s = at::empty({M, W / 32}, a_codes.options())));
  }
  omo_grouped_gemm_mxfp4(a_codes, a_scales, m_splits, b_codes, b_scales, c, bias, activation,
                         residual, pre, q, s);
  return out;
}

void omo_grouped_wgrad_mxfp4(at::Tensor dy, at::Tensor x_codes, at::Tensor x_scales,
                             OptTensor m_splits, at::Tensor dw, bool accumulate) {
  OmoRange nvtx_range("omo_grouped_wgrad_mxfp4");
  OMO_CHECK_INPUT(dw);
  TORCH_CHECK(dw.dim() == 3, "dw must be [E, N, K]");
  const bool f32 = dw.scalar_type() == at::kFloat;
  check_dtype(dw, f32 ? at::kFloat : at::kBFloat16, "dw");
  TORCH_CHECK(dy.dim() == 2, "dy must be [M, N]");
  const int64_t E = dw.size(0), N = dw.size(1), K = dw.size(2), M = dy.size(0);
  TORCH_CHECK(E >= 1 && K % 32 == 0, "dw must be [E, N, K] with K % 32 == 0");
  check_rows(dy, "dy", M, N, at::kBFloat16, dw);
  check_rows(x_codes, "x_codes", M, K / 2, at::kByte, dw);
  check_rows(x_scales, "x_scales", M, K / 32, at::kByte, dw);
  const int32_t* splits = check_splits(m_splits, E, dw);
  c10::cuda::CUDAGuard g(dw.device());
  check_status(mxb_grouped_wgrad_mxfp4(dy.data_ptr(), pitch(dy), x_codes.data_ptr(),
                                       pitch(x_codes), x_scales.data_ptr(), pitch(x_scales), M,
                                       splits, (int32_t)E, N, K, dw.data_ptr(), f32 ? 1 : 0,
                                       accumulate ? 1 : 0, cur_stream()),
               "omo_grouped_wgrad_mxfp4");
}

int64_t omo_bias_act_grad_workspace(int64_t M, int64_t E, int64_t N) {
  return mxb_bias_act_grad_workspace(M, (int32_t)E, N);
}

void omo_bias_act_grad(at::Tensor dy, OptTensor pre, OptTensor m_splits, int64_t E, int64_t N,
                       int64_t activation, OptTensor dz, OptTensor dz_codes, OptTensor dz_scales,
                       OptTensor dbias, OptTensor workspace) {
  OmoRange nvtx_range("omo_bias_act_grad");
  OMO_CHECK_INPUT(dy);
  TORCH_CHECK(dy.dim() == 2, "dy must be [M, W]");
  TORCH_CHECK(activation >= MXB_ACT_NONE && activation <= MXB_ACT_SWIGLU, "unknown activation");
  TORCH_CHECK(E >= 1 && E <= MXB_MAX_EXPERTS, "need 1 <= E <= ", MXB_MAX_EXPERTS);
  const int64_t M = dy.size(0), parts = activation == MXB_ACT_SWIGLU ? 2 : 1;
  TORCH_CHECK(N % parts == 0, "N must be even for swiglu");
  check_dense(dy, "dy", {M, N / parts}, at::kBFloat16, dy);
  TORCH_CHECK(pre || activation == MXB_ACT_NONE, "pre is needed for this activation");
  if (pre) check_dense(*pre, "pre", {M, N}, at::kBFloat16, dy);
  if (dz) check_dense(*dz, "dz", {M, N}, at::kBFloat16, dy);
  TORCH_CHECK(dz_codes.has_value() == dz_scales.has_value(), "dz_codes and dz_scales go together");
  if (dz_codes) {
    TORCH_CHECK(N % (32 * parts) == 0, "a quantized dz needs N % ", 32 * parts, " == 0");
    check_dense(*dz_codes, "dz_codes", {M, N / 2}, at::kByte, dy);
    check_dense(*dz_scales, "dz_scales", {M, N / 32}, at::kByte, dy);
  }
  if (dbias) check_dense(*dbias, "dbias", {E, N}, at::kFloat, dy);
  if (workspace)
    TORCH_CHECK(workspace->is_cuda() && workspace->device() == dy.device() &&
                    workspace->is_contiguous(),
                "workspace must be a contiguous CUDA tensor beside dy");
  const int32_t* splits = check_splits(m_splits, E, dy);
  c10::cuda::CUDAGuard g(dy.device());
  check_status(
      mxb_bias_act_grad(dy.data_ptr(), opt_ptr(pre), M, splits, (int32_t)E, N, (int32_t)activation,
                        opt_ptr(dz), opt_ptr(dz_codes), opt_ptr(dz_scales), (float*)opt_ptr(dbias),
                        opt_ptr(workspace), workspace ? (int64_t)workspace->nbytes() : 0,
                        cur_stream()),
      "omo_bias_act_grad");
}

// The same with results and workspace allocated here: those of (dz, dbias, dz_codes,
// dz_scales) that are asked for.
std::vector<at::Tensor> omo_bias_act_grad_new(const at::Tensor& dy, const OptTensor& pre,
                                              const OptTensor& m_splits, int64_t activation,
                                              bool bias_grad, bool quantize, bool bf16_out) {
  TORCH_CHECK(dy.is_cuda() && dy.dim() == 2, "dy must be a CUDA tensor [M, W]");
  const int64_t M = dy.size(0), N = dy.size(1) * (activation == MXB_ACT_SWIGLU ? 2 : 1);
  const int64_t E = m_splits ? m_splits->numel() : 1;
  const auto bytes = dy.options().dtype(at::kByte);
  OptTensor dz, db, q, s, work;
  std::vector<at::Tensor> out;
  if (bf16_out) out.push_back(*(dz = at::empty({M, N}, dy.options().dtype(at::kBFloat16))));
  if (bias_grad) {
    out.push_back(*(db = at::empty({E, N}, dy.options().dtype(at::kFloat))));
    const int64_t need = mxb_bias_act_grad_workspace(M, (int32_t)E, N);
    if (need) work = at::empty({need}, bytes);
  }
  if (quantize) {
    out.push_back(*(q = at::empty({M, N / 2}, bytes)));
    out.push_back(*(s = at::empty({M, N / 32}, bytes)));
  }
  omo_bias_act_grad(dy, pre, m_splits, E, N, activation, dz, q, s, db, work);
  return out;
}

// map int32 [T, >= topk] (row pitch = its stride); topk from the weights, or all columns.
int64_t check_map(const at::Tensor& map, const OptTensor& weight, int64_t topk,
                  const at::Tensor& like) {
  TORCH_CHECK(map.dim() == 2 && map.size(1) >= topk, "map must be [T, >= topk]");
  check_rows(map, "map", map.size(0), map.size(1), at::kInt, like);
  if (weight) check_dense(*weight, "weight", {map.size(0), topk}, at::kFloat, like);
  return map.size(0) > 1 ? map.stride(0) : map.size(1);
}

void omo_moe_unpermute(at::Tensor y, at::Tensor map, OptTensor weight, int64_t topk,
                       at::Tensor out) {
  OmoRange nvtx_range("omo_moe_unpermute");
  OMO_CHECK_INPUT(y);
  check_dtype(y, at::kBFloat16, "y");
  TORCH_CHECK(y.dim() == 2, "y must be [R, H]");
  const int64_t ld = check_map(map, weight, topk, y), T = map.size(0);
  check_dense(out, "out", {T, y.size(1)}, at::kBFloat16, y);
  c10::cuda::CUDAGuard g(y.device());
  check_status(mxb_moe_unpermute(y.data_ptr(), y.size(0), y.size(1), (const int32_t*)map.data_ptr(),
                                 ld, (int32_t)topk, (const float*)opt_ptr(weight), T,
                                 out.data_ptr(), cur_stream()),
               "omo_moe_unpermute");
}

void omo_moe_unpermute_grad(at::Tensor dout, OptTensor y, int64_t rows, at::Tensor map,
                            OptTensor weight, int64_t topk, OptTensor dy, OptTensor dy_codes,
                            OptTensor dy_scales, OptTensor dweight) {
  OmoRange nvtx_range("omo_moe_unpermute_grad");
  OMO_CHECK_INPUT(dout);
  check_dtype(dout, at::kBFloat16, "dout");
  TORCH_CHECK(dout.dim() == 2 && dout.size(0) == map.size(0), "dout must be [T, H]");
  const int64_t T = dout.size(0), H = dout.size(1);
  const int64_t ld = check_map(map, weight, topk, dout);
  TORCH_CHECK(y || !dweight, "y is needed for dweight");
  if (y) check_dense(*y, "y", {rows, H}, at::kBFloat16, dout);
  if (dy) check_dense(*dy, "dy", {rows, H}, at::kBFloat16, dout);
  TORCH_CHECK(dy_codes.has_value() == dy_scales.has_value(), "dy_codes and dy_scales go together");
  if (dy_codes) {
    TORCH_CHECK(H % 32 == 0, "a quantized dy needs H % 32 == 0");
    check_dense(*dy_codes, "dy_codes", {rows, H / 2}, at::kByte, dout);
    check_dense(*dy_scales, "dy_scales", {rows, H / 32}, at::kByte, dout);
  }
  if (dweight) check_dense(*dweight, "dweight", {T, topk}, at::kFloat, dout);
  c10::cuda::CUDAGuard g(dout.device());
  check_status(mxb_moe_unpermute_grad(dout.data_ptr(), opt_ptr(y), rows, H,
                                      (const int32_t*)map.data_ptr(), ld, (int32_t)topk,
                                      (const float*)opt_ptr(weight), T, opt_ptr(dy),
                                      opt_ptr(dy_codes), opt_ptr(dy_scales),
                                      (float*)opt_ptr(dweight), cur_stream()),
               "omo_moe_unpermute_grad");
}

at::Tensor omo_moe_unpermute_new(const at::Tensor& y, const at::Tensor& map,
                                 const OptTensor& weight, int64_t topk) {
  TORCH_CHECK(y.is_cuda() && y.dim() == 2 && map.dim() == 2, "y must be a CUDA tensor [R, H], map [T, k]");
  at::Tensor out = at::empty({map.size(0), y.size(1)}, y.options());
  omo_moe_unpermute(y, map, weight, topk, out);
  return out;
}

// Those of (dy, dweight, dy_codes, dy_scales) that are asked for; zero: rows that the map
// does not name are zero instead of uninitialised.
std::vector<at::Tensor> omo_moe_unpermute_grad_new(const at::Tensor& dout, const at::Tensor& y,
                                                   const at::Tensor& map, const OptTensor& weight,
                                                   int64_t topk, bool weight_grad, bool quantize,
                                                   bool zero) {
  TORCH_CHECK(y.is_cuda() && y.dim() == 2 && map.dim() == 2, "y must be a CUDA tensor [R, H], map [T, k]");
  const int64_t R = y.size(0), H = y.size(1);
  const auto bytes = y.options().dtype(at::kByte);
  auto make = [&](at::IntArrayRef sizes, const at::TensorOptions& o) {
    return zero ? at::zeros(sizes, o) : at::empty(sizes, o);
  };
  c10::cuda::CUDAGuard g(y.device());
  at::Tensor dy = make({R, H}, y.options());
  OptTensor dw, q, s;
  std::vector<at::Tensor> out = {dy};
  if (weight_grad) out.push_back(*(dw = at::empty({map.size(0), topk}, y.options().dtype(at::kFloat))));
  if (quantize) {
    out.push_back(*(q = make({R, H / 2}, bytes)));
    out.push_back(*(s = make({R, H / 32}, bytes)));
  }
  omo_moe_unpermute_grad(dout, y, R, map, weight, topk, dy, q, s, dw);
  return out;
}

}  // namespace

PYBIND11_MODULE(omo, m) {
  m.doc() = "B200 (sm_100a) MXFP4 operators with the reference `omo` interface";
  m.def("omo_per_token_group_quant_fp4", &omo_per_token_group_quant_fp4,
        "Per-token-group FP4 quantization", py::arg("input"), py::arg("output_q"),
        py::arg("output_s"), py::arg("group_size"), py::arg("eps"), py::arg("fp4_min"),
        py::arg("fp4_max"), py::arg("scale_ue8m0"));
  m.def("omo_per_token_Mxfp4ToBf16_dequant", &omo_per_token_Mxfp4ToBf16_dequant,
        "Per-token-group FP4 dequantization BF16", py::arg("input"), py::arg("input_s"),
        py::arg("output_q"), py::arg("output_s"), py::arg("group_size"), py::arg("eps"),
        py::arg("fp4_min"), py::arg("fp4_max"), py::arg("scale_ue8m0"));
  m.def("omo_per_token_Mxfp4ToBf16ToFp8", &omo_per_token_Mxfp4ToBf16ToFp8,
        "Per-token-group FP4 dequantization BF16->FP8", py::arg("input"), py::arg("input_s"),
        py::arg("output_q"), py::arg("output_s"), py::arg("group_size"), py::arg("eps"),
        py::arg("fp4_min"), py::arg("fp4_max"), py::arg("scale_ue8m0"));
  m.def("omo_per_token_Mxfp4ToFp8", &omo_per_token_Mxfp4ToFp8,
        "Per-token-group FP4 -> FP8 (1x128 groups)", py::arg("input"), py::arg("input_s"),
        py::arg("output_q"), py::arg("output_s"), py::arg("group_size"), py::arg("eps"),
        py::arg("fp4_min"), py::arg("fp4_max"), py::arg("scale_ue8m0"));
  m.def("omo_per_token_group_quant_fp4_fused_ToFp8", &omo_per_token_group_quant_fp4_fused_ToFp8,
        "Per-token-group FP4 quantization fused ToFp8", py::arg("input"), py::arg("output_q"),
        py::arg("output_s"), py::arg("output_bf16_q"), py::arg("output_bf16_s"),
        py::arg("group_size"), py::arg("eps"), py::arg("fp4_min"), py::arg("fp4_max"),
        py::arg("scale_ue8m0"));
  m.def("omo_per_token_Mxfp4RowToBf16ToFp8Col", &omo_per_token_Mxfp4RowToBf16ToFp8Col,
        "Per-token-group FP4(row) dequantization BF16->FP8(col)", py::arg("input"),
        py::arg("input_s"), py::arg("output_q"), py::arg("output_s"), py::arg("eps"));
  m.def("omo_per_token_Mxfp4RowToBf16ToFp8Col_msplit", &omo_per_token_Mxfp4RowToBf16ToFp8Col_msplit,
        "Per-token-group FP4 dequantization col FP8 for group linear(m_split)", py::arg("input"),
        py::arg("input_s"), py::arg("output_q"), py::arg("output_s"), py::arg("m_splits"),
        py::arg("split_offsets"), py::arg("scale_offsets"), py::arg("max_split_len"),
        py::arg("eps"));
  m.def("omo_per_token_Mxfp4ToFp8_col", &omo_per_token_Mxfp4ToFp8_col,
        "Per-token-group FP4 dequantization col FP8", py::arg("input"), py::arg("input_s"),
        py::arg("output_q"), py::arg("output_s"), py::arg("group_size"), py::arg("eps"),
        py::arg("fp4_min"), py::arg("fp4_max"), py::arg("scale_ue8m0"));
  m.def("omo_quant_mxfp4_rowcol", &omo_quant_mxfp4_rowcol,
        "One-pass rowwise + columnwise MXFP4 quantization", py::arg("input"),
        py::arg("codes_row"), py::arg("scales_row"), py::arg("codes_col"), py::arg("scales_col"),
        py::arg("scales_row_swizzled") = py::none(), py::arg("eps") = 1e-10,
        py::arg("fp4_min") = -6.0, py::arg("fp4_max") = 6.0);
  m.def("omo_swizzle_scales", &omo_swizzle_scales, "E8M0 scales -> 128x4 swizzled layout",
        py::arg("scales"), py::arg("out"));
  m.def("omo_per_token_quant_fp8", &omo_per_token_quant_fp8, "Per-token FP8 quantization",
        py::arg("input"), py::arg("output_q"), py::arg("output_s"), py::arg("eps") = 1e-10);
  m.def("omo_per_token_dequant_fp8", &omo_per_token_dequant_fp8, "Per-token FP8 dequantization",
        py::arg("input_q"), py::arg("input_s"), py::arg("output"));
  m.def("omo_swiglu_quant_mxfp4", &omo_swiglu_quant_mxfp4,
        "SwiGLU of [.., 2H] and the rowwise MXFP4 of its input, one pass", py::arg("input"),
        py::arg("output"), py::arg("codes"), py::arg("scales"), py::arg("eps") = 1e-10,
        py::arg("fp4_min") = -6.0, py::arg("fp4_max") = 6.0);
  m.def("omo_moe_permute_mxfp4", &omo_moe_permute_mxfp4,
        "MoE permute of MXFP4 rows (codes and scales) to expert slots", py::arg("codes"),
        py::arg("scales"), py::arg("dst"), py::arg("out_codes"), py::arg("out_scales"));
  m.def("omo_gemm_mxfp4", &omo_gemm_mxfp4, "Block-scaled MXFP4 GEMM C = A . B^T (tcgen05)",
        py::arg("a_codes"), py::arg("a_scales_swizzled"), py::arg("b_codes"),
        py::arg("b_scales_swizzled"), py::arg("c"));
  m.def("omo_swizzle_scales_grouped", &omo_swizzle_scales_grouped,
        "E8M0 scales of stacked weights -> 128x4-tile layout per part", py::arg("scales"),
        py::arg("parts"), py::arg("out"));
  m.def("omo_grouped_gemm_mxfp4", &omo_grouped_gemm_mxfp4,
        "MXFP4 products grouped by expert with bias / activation / residual (tcgen05)",
        py::arg("a_codes"), py::arg("a_scales"), py::arg("m_splits"), py::arg("b_codes"),
        py::arg("b_scales"), py::arg("c"), py::arg("bias") = py::none(),
        py::arg("activation") = 0, py::arg("residual") = py::none(), py::arg("pre") = py::none(),
        py::arg("c_codes") = py::none(), py::arg("c_scales") = py::none());
  m.def("omo_grouped_gemm_mxfp4_new", &omo_grouped_gemm_mxfp4_new,
        "omo_grouped_gemm_mxfp4 with its results allocated", py::arg("a_codes"),
        py::arg("a_scales"), py::arg("m_splits"), py::arg("b_codes"), py::arg("b_scales"),
        py::arg("bias"), py::arg("activation"), py::arg("residual"), py::arg("save_pre"),
        py::arg("quantize"), py::arg("bf16_out"));
  m.def("omo_bias_act_grad_new", &omo_bias_act_grad_new,
        "omo_bias_act_grad with its results allocated", py::arg("dy"), py::arg("pre"),
        py::arg("m_splits"), py::arg("activation"), py::arg("bias_grad"), py::arg("quantize"),
        py::arg("bf16_out"));
  m.def("omo_grouped_wgrad_mxfp4", &omo_grouped_wgrad_mxfp4,
        "Weight gradients grouped by expert from BF16 dy and MXFP4 x (tcgen05)", py::arg("dy"),
        py::arg("x_codes"), py::arg("x_scales"), py::arg("m_splits"), py::arg("dw"),
        py::arg("accumulate") = false);
  m.def("omo_bias_act_grad_workspace", &omo_bias_act_grad_workspace,
        "Workspace bytes of omo_bias_act_grad", py::arg("M"), py::arg("E"), py::arg("N"));
  m.def("omo_bias_act_grad", &omo_bias_act_grad, "Gradient of the bias / activation epilogue",
        py::arg("dy"), py::arg("pre"), py::arg("m_splits"), py::arg("E"), py::arg("N"),
        py::arg("activation"), py::arg("dz") = py::none(), py::arg("dz_codes") = py::none(),
        py::arg("dz_scales") = py::none(), py::arg("dbias") = py::none(),
        py::arg("workspace") = py::none());
  m.def("omo_moe_unpermute", &omo_moe_unpermute, "Weighted sum of expert rows per token",
        py::arg("y"), py::arg("map"), py::arg("weight"), py::arg("topk"), py::arg("out"));
  m.def("omo_moe_unpermute_new", &omo_moe_unpermute_new,
        "omo_moe_unpermute with its result allocated", py::arg("y"), py::arg("map"),
        py::arg("weight"), py::arg("topk"));
  m.def("omo_moe_unpermute_grad_new", &omo_moe_unpermute_grad_new,
        "omo_moe_unpermute_grad with its results allocated", py::arg("dout"), py::arg("y"),
        py::arg("map"), py::arg("weight"), py::arg("topk"), py::arg("weight_grad"),
        py::arg("quantize"), py::arg("zero"));
  m.def("omo_moe_unpermute_grad", &omo_moe_unpermute_grad, "Gradient of omo_moe_unpermute",
        py::arg("dout"), py::arg("y"), py::arg("rows"), py::arg("map"), py::arg("weight"),
        py::arg("topk"), py::arg("dy") = py::none(), py::arg("dy_codes") = py::none(),
        py::arg("dy_scales") = py::none(), py::arg("dweight") = py::none());
}
