// Rows in 8 bits (include/circuit_ops.h, the int8 section): quantisation with
// one scale a row (plain, after a root-mean-square norm with the residual's
// addition, or to unit length; into consecutive rows or into the slots of a row
// store), and reading rows back by id.  The kernels are in int8_rows.cuh.
#include <cfloat>

#include "int8_rows.h"

namespace cb {
namespace i8 {

__global__ void k_reset_slots(const void* slots, int slot64, int64_t n, int64_t capacity, float* scales) {
  griddep_wait();
  griddep_launch();
  const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t s = slot_at(slots, slot64, i);
  if (s >= 0 && s < capacity) scales[s] = 0.f;
}
__global__ void k_claim_slots(const void* slots, int slot64, int64_t n, int64_t capacity, float* scales) {
  griddep_wait();
  griddep_launch();
  const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t s = slot_at(slots, slot64, i);
  if (s >= 0 && s < capacity) atomicMax(reinterpret_cast<uint32_t*>(scales + s), claim_tag(i));
}

}  // namespace i8
}  // namespace cb

using namespace cb::i8;

extern "C" {

int circuit_op_quantize_rows(const void* rows, int dtype, int64_t n, int dim, int64_t row_stride,
                             const void* residual, int64_t residual_stride, const void* weight, int weight_dtype,
                             int norm, float eps, void* summed, int64_t summed_stride, const void* slots,
                             int slot_bytes, int64_t capacity, int8_t* codes, int64_t code_stride, float* scales,
                             void* stream) {
  const int e = type_bytes(dtype);
  if (!e) return bad("quantize_rows: dtype must be CIRCUIT_F32, CIRCUIT_F16 or CIRCUIT_BF16");
  if (dim < 1 || dim > CIRCUIT_INT8_MAX_DIM) return bad("quantize_rows: dim must be in [1, 16384]");
  if (n < 0 || n > 0x7fffffffLL) return bad("quantize_rows: n must be in [0, 2^31)");
  if (norm < CIRCUIT_NORM_NONE || norm > CIRCUIT_NORM_UNIT) return bad("quantize_rows: unknown norm");
  if (norm == CIRCUIT_NORM_NONE && (residual || weight))
    return bad("quantize_rows: residual and weight need a norm");
  if (!(eps >= 0.f && eps <= FLT_MAX)) return bad("quantize_rows: eps must be finite and not negative");
  if (weight && weight_dtype != dtype && weight_dtype != CIRCUIT_F32)
    return bad("quantize_rows: the weight must be of the rows' type or fp32");
  if (slots && slot_bytes != 4 && slot_bytes != 8) return bad("quantize_rows: slots must be int32 or int64");
  if (capacity < 0) return bad("quantize_rows: negative capacity");
  if (n == 0) return CIRCUIT_OK;
  if (!rows || !codes || !scales || (residual && !summed)) return bad("quantize_rows: null pointer");
  if (!slots && capacity < n) return bad("quantize_rows: more rows than the output holds");
  if (row_stride < dim || code_stride < dim || (residual && (residual_stride < dim || summed_stride < dim)))
    return bad("quantize_rows: a row stride is smaller than dim");
  const uintptr_t align = (uintptr_t)rows | (uintptr_t)residual | (residual ? (uintptr_t)summed : 0);
  if (align % e || (weight && (uintptr_t)weight % (weight_dtype == CIRCUIT_F32 ? 4 : 2)) || (uintptr_t)scales % 4 ||
      (slots && (uintptr_t)slots % slot_bytes))
    return bad("quantize_rows: a pointer is not aligned to its type");
  QuantizeParams P{};
  P.x = rows;
  P.res = residual;
  P.w = weight;
  P.sum = summed;
  P.slots = slots;
  P.codes = codes;
  P.scales = scales;
  P.n = n;
  P.x_stride = row_stride;
  P.res_stride = residual_stride;
  P.sum_stride = summed_stride;
  P.code_stride = code_stride;
  P.capacity = capacity;
  P.d = dim;
  P.w_f32 = weight && weight_dtype == CIRCUIT_F32;
  P.inexact = weight && (P.w_f32 || dtype == CIRCUIT_F32);
  P.inv_n = norm == CIRCUIT_NORM_RMS ? 1.f / (float)dim : 1.f;
  P.eps = eps;
  P.slot64 = slot_bytes == 8;
  // the widest words that every row is made of; a code word is a byte for each value
  uintptr_t bits = 16 | (uintptr_t)rows | (uintptr_t)(row_stride * e) | (uintptr_t)(dim * (int64_t)e) |
                   ((uintptr_t)codes | (uintptr_t)code_stride) * e;
  if (weight && weight_dtype == dtype) bits |= (uintptr_t)weight;
  else if (weight && !on16(weight, 0)) bits |= (uintptr_t)weight % 8 ? 2 : 4;  // fp32 beside 16-bit words: 4 bytes a value
  if (residual)
    bits |= (uintptr_t)residual | (uintptr_t)(residual_stride * e) | (uintptr_t)summed | (uintptr_t)(summed_stride * e);
  const int bytes = (int)(bits & -bits);
  cudaStream_t st = (cudaStream_t)stream;
  // Equal slots: each row of a short write looks through the later ones; a long
  // write claims its slots first, the claims standing in the scales.
  P.claimed = slots && n > 1024;
  if (P.claimed) {
    const unsigned blocks = (unsigned)((n + 255) / 256);
    launch(k_reset_slots, dim3(blocks), 256, 0, 1, st, slots, P.slot64, n, capacity, scales);
    launch(k_claim_slots, dim3(blocks), 256, 0, 1, st, slots, P.slot64, n, capacity, scales);
  }
  const bool full = norm != CIRCUIT_NORM_NONE;
  if (dtype == CIRCUIT_F32) quantize_rows<float>(P, bytes, full, st);
  else if (dtype == CIRCUIT_F16) quantize_rows<__half>(P, bytes, full, st);
  else quantize_rows<__nv_bfloat16>(P, bytes, full, st);
  return check(cudaGetLastError(), "quantize_rows launch");
}

int circuit_op_dequantize_rows(const int8_t* codes, int64_t code_stride, const float* scales, int64_t rows, int dim,
                               const void* ids, int id_bytes, int64_t n, void* out, int dtype, int64_t out_stride,
                               void* stream) {
  const int e = type_bytes(dtype);
  if (!e) return bad("dequantize_rows: dtype must be CIRCUIT_F32, CIRCUIT_F16 or CIRCUIT_BF16");
  if (dim < 1 || dim > CIRCUIT_INT8_MAX_DIM) return bad("dequantize_rows: dim must be in [1, 16384]");
  if (n < 0 || n > 0x7fffffffLL || rows < 0) return bad("dequantize_rows: bad sizes");
  if (ids && id_bytes != 4 && id_bytes != 8) return bad("dequantize_rows: ids must be int32 or int64");
  if (n == 0) return CIRCUIT_OK;
  // a store without rows has no memory either: every id is then an empty place or past the end
  if ((rows > 0 && (!codes || !scales)) || !out) return bad("dequantize_rows: null pointer");
  if (!ids && rows < n) return bad("dequantize_rows: more rows asked for than there are");
  if (code_stride < dim || out_stride < dim) return bad("dequantize_rows: a row stride is smaller than dim");
  if ((uintptr_t)out % e || (uintptr_t)scales % 4 || (ids && (uintptr_t)ids % id_bytes))
    return bad("dequantize_rows: a pointer is not aligned to its type");
  const ReadParams P{codes, scales, ids, out, n, rows, code_stride, out_stride, dim, id_bytes == 8};
  const uintptr_t bits = 16 | (uintptr_t)out | (uintptr_t)(out_stride * e) | (uintptr_t)(dim * (int64_t)e) |
                         ((uintptr_t)codes | (uintptr_t)code_stride) * e;
  const int bytes = (int)(bits & -bits);  // the widest words that every row is made of
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == CIRCUIT_F32) dequantize_rows<float>(P, bytes, st);
  else if (dtype == CIRCUIT_F16) dequantize_rows<__half>(P, bytes, st);
  else dequantize_rows<__nv_bfloat16>(P, bytes, st);
  return check(cudaGetLastError(), "dequantize_rows launch");
}

}  // extern "C"
