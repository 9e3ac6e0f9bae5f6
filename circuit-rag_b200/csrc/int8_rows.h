// Parameters and launches of the row kernels, which are compiled by type
// (int8_rows_f32.cu, int8_rows_f16.cu, int8_rows_bf16.cu).
#pragma once

#include "int8.cuh"

namespace cb {
namespace i8 {

struct QuantizeParams {
  const void* x;
  const void* res;      // nullptr: no residual
  const void* w;        // nullptr: no weight
  void* sum;            // x + res, written when res is given
  const void* slots;    // nullptr: row i to row i
  int8_t* codes;
  float* scales;
  int64_t n, x_stride, res_stride, sum_stride, code_stride, capacity;
  int d;
  int w_f32;            // the weight is fp32 (else of the row's type)
  int inexact;          // a product of value and weight may need more than 24 bits
  float inv_n, eps;     // norm: the scale is divided by sqrt(ss * inv_n + eps)
  int slot64, claimed;  // slots are int64; slots were claimed by k_claim_slots
};

struct ReadParams {
  const int8_t* codes;
  const float* scales;
  const void* ids;  // nullptr: row i
  void* out;
  int64_t n, rows, code_stride, out_stride;
  int d, id64;
};

// bytes: the widest word (16, or less) that the rows are whole words of; full: with
// residual, weight and norm.
template <typename T>
void quantize_rows(const QuantizeParams& P, int bytes, bool full, cudaStream_t st);
template <typename T>
void dequantize_rows(const ReadParams& P, int bytes, cudaStream_t st);

__device__ __forceinline__ int64_t slot_at(const void* slots, int slot64, int64_t i) {
  return slot64 ? reinterpret_cast<const long long*>(slots)[i] : (int64_t) reinterpret_cast<const int*>(slots)[i];
}
// A slot's claim by row i of a write: above every scale's bit pattern (scales
// are never negative), larger for later rows.
__device__ __forceinline__ uint32_t claim_tag(int64_t i) { return 0x80000000u | (uint32_t)i; }

}  // namespace i8
}  // namespace cb
