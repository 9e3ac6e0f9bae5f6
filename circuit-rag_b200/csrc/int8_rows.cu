// Rows in 8 bits (include/circuit_ops.h, the int8 section): quantisation with
// one scale a row (plain, after a root-mean-square norm with the residual's
// addition, or to unit length; into consecutive rows or into the slots of a row
// store), and reading rows back by id.
//
// Mathematics.  With v = x (+ residual, rounded once to the row's type) and
// u = v * w, a row's codes are rint(127 u_j / a), a = max|u|, and its scale is
// a / 127 times the norm's factor.  The norm's factor cancels in the codes, so
// they depend on no sum and are the same whatever its order: k_quantize_rows
// gives the correctly rounded code of the real quotient (see code_of), and only
// the scale carries the rounding of the 32-bit sum of squares.
#include <cfloat>

#include "int8.cuh"

namespace cb {
namespace i8 {

// ---------------------------------------------------------------- helpers
// Maximum of magnitudes that keeps a NaN (fmaxf would drop it).
__device__ __forceinline__ float max_abs_nan(float m, float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
  return r;
}

struct RowSums {
  float top, low;  // max |u| as the unevaluated sum top + low (top: the rounded product); top NaN or inf: a bad row
  float ss;        // sum of v^2
};
// (top, low) of two candidates: the larger real number; a NaN stays.
__device__ __forceinline__ void raise(float& top, float& low, float t, float l) {
  if (t > top || (t == top && l > low) || t != t) {
    top = t;
    low = l;
  }
}
// Over the G threads of a row.
template <int G, bool LOW, bool SS>
__device__ __forceinline__ RowSums reduce(RowSums r) {
  constexpr int W = G < 32 ? G : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    const float t = __shfl_xor_sync(FULL_MASK, r.top, o);
    if constexpr (LOW) raise(r.top, r.low, t, __shfl_xor_sync(FULL_MASK, r.low, o));
    else r.top = max_abs_nan(r.top, t);
    if constexpr (SS) r.ss += __shfl_xor_sync(FULL_MASK, r.ss, o);
  }
  if constexpr (G > 32) {
    __shared__ RowSums part[G / 32];
    __syncthreads();  // the previous call's readers are done
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = r;
    __syncthreads();
    r = part[0];
#pragma unroll
    for (int w = 1; w < G / 32; ++w) {
      if constexpr (LOW) raise(r.top, r.low, part[w].top, part[w].low);
      else r.top = max_abs_nan(r.top, part[w].top);
      if constexpr (SS) r.ss += part[w].ss;
    }
  }
  return r;
}

// Codes.  With inv = 127 / top in 32 bits, one FMA adds u * inv to 1.5 * 2^23:
// the sum's low byte is the nearest integer n, and u * inv - n (a second FMA) its
// remainder.  u, inv and top are off by 2^-24 of their size each, so u * inv is
// within 127 * 3 * 2^-24 < 2.3e-5 of the real quotient and n is its nearest
// integer unless the remainder is within 6e-5 of a half; there (0.012 % of the
// values) the quotient is taken in 64 bits, where v * w is exact.
constexpr float ROUNDER = 12582912.f;
constexpr float NEAR_HALF = 0.5f - 6e-5f;
__device__ __forceinline__ int code_near_half(float v, float w, double a) {
  return (int)rint((double)v * (double)w * 127.0 / a);
}

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
  int wide_in, wide_out;
};

__device__ __forceinline__ int64_t slot_at(const void* slots, int slot64, int64_t i) {
  return slot64 ? reinterpret_cast<const long long*>(slots)[i] : (int64_t) reinterpret_cast<const int*>(slots)[i];
}
// A slot's claim by row i of a write: above every scale's bit pattern (scales
// are never negative), larger for later rows.
__device__ __forceinline__ uint32_t claim_tag(int64_t i) { return 0x80000000u | (uint32_t)i; }

__global__ void k_reset_slots(const void* slots, int slot64, int64_t n, int64_t capacity, float* scales) {
  const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t s = slot_at(slots, slot64, i);
  if (s >= 0 && s < capacity) scales[s] = 0.f;
}
__global__ void k_claim_slots(const void* slots, int slot64, int64_t n, int64_t capacity, float* scales) {
  const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t s = slot_at(slots, slot64, i);
  if (s >= 0 && s < capacity) atomicMax(reinterpret_cast<uint32_t*>(scales + s), claim_tag(i));
}

constexpr int quantize_threads(int G) { return G <= 32 ? 256 : G; }

// G threads a row (8 lanes, a warp, or a block), the row in NV 16-byte vectors a
// thread: it is read once.  FULL: with residual, weight and norm as the
// parameters say; otherwise the plain quantisation.  Memory-bound by design: per
// value one NaN-keeping maximum (and one FMA for the squares) before the row's
// reduction, two FMAs, an add and a maximum after it.
template <typename T, int G, int NV, bool FULL>
__global__ void __launch_bounds__(quantize_threads(G)) k_quantize_rows(QuantizeParams P) {
  constexpr int V = RowType<T>::V;
  const int lane = threadIdx.x % G;
  const int64_t row = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) / G;
  const bool live = row < P.n;
  if constexpr (G >= 32) {
    if (!live) return;  // whole warps; with fewer lanes a row the others of the warp need the shuffles
  }
  const int d = live ? P.d : 0;

  // where the row goes (-1: nowhere); of equal slots the last row's write stays
  int64_t dst = live ? row : -1;
  if (P.slots) {
    dst = live ? slot_at(P.slots, P.slot64, row) : -1;
    bool mine = dst >= 0 && dst < P.capacity;
    if (P.claimed) {
      mine = mine && __ldcg(reinterpret_cast<const uint32_t*>(P.scales + dst)) == claim_tag(row);
      // every thread has read the claim before the row's scale overwrites it
      if constexpr (G > 32) __syncthreads();
      else __syncwarp();
    } else {
      int later = 0;
      if (mine)
        for (int64_t j = row + 1 + lane; j < P.n; j += G) later |= slot_at(P.slots, P.slot64, j) == dst;
      if constexpr (G > 32) {
        later = __syncthreads_or(later);
      } else {
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) later |= __shfl_xor_sync(FULL_MASK, later, o);
      }
      mine = mine && !later;
    }
    if (!mine) dst = -1;
    if constexpr (G >= 32) {
      if (dst < 0 && !(FULL && P.res)) return;
    }
  }

  const T* x = reinterpret_cast<const T*>(P.x) + (live ? row : 0) * P.x_stride;
  Vec<T> v[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) v[k] = load_vec(x, (k * G + lane) * V, d, P.wide_in & 1);
  RowSums r{0.f, 0.f, 0.f};
  float u[FULL ? NV : 1][FULL ? V : 1];  // v * w, rounded
  if constexpr (FULL) {
    if (P.res) {
      const T* res = reinterpret_cast<const T*>(P.res) + (live ? row : 0) * P.res_stride;
      Vec<T> b[NV];
#pragma unroll
      for (int k = 0; k < NV; ++k) b[k] = load_vec(res, (k * G + lane) * V, d, P.wide_in & 2);
      T* sum = reinterpret_cast<T*>(P.sum) + (live ? row : 0) * P.sum_stride;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        // the sum is kept in the row's type, as the next layer reads it; the
        // norm and the codes are those of the kept value
#pragma unroll
        for (int i = 0; i < V; ++i)
          v[k].e[i] = RowType<T>::put(RowType<T>::get(v[k].e[i]) + RowType<T>::get(b[k].e[i]));
        store_vec(sum, (k * G + lane) * V, d, P.wide_in & 4, v[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * G + lane) * V;
      float w[V];
      if (!P.w) {
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = 1.f;
      } else if (P.w_f32) {
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = c + i < d ? __ldg(reinterpret_cast<const float*>(P.w) + c + i) : 0.f;
      } else {
        const Vec<T> b = load_vec(reinterpret_cast<const T*>(P.w), c, d, P.wide_in & 8);
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = RowType<T>::get(b.e[i]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float e = RowType<T>::get(v[k].e[i]);
        r.ss = fmaf(e, e, r.ss);
        u[k][i] = e * w[i];
      }
      if (P.inexact) {  // an fp32 factor: the FMA gives the product's rounding error
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float p = fabsf(u[k][i]);
          if (!(p < r.top)) raise(r.top, r.low, p, fmaf(fabsf(RowType<T>::get(v[k].e[i])), fabsf(w[i]), -p));
        }
      } else {  // 8- or 11-bit factors: their product is exact
#pragma unroll
        for (int i = 0; i < V; ++i) r.top = max_abs_nan(r.top, u[k][i]);
      }
    }
    r = P.inexact ? reduce<G, true, true>(r) : reduce<G, false, true>(r);
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) r.top = max_abs_nan(r.top, RowType<T>::get(v[k].e[i]));
    r = reduce<G, false, false>(r);
  }
  const bool bad = !(r.top <= FLT_MAX);

  float scale = r.top / 127.f;
  if constexpr (FULL) {
    const bool odd = r.top > 0.f && !bad && !(r.ss > 1e-25f && r.ss < FLT_MAX);
    if (r.top > 0.f && !bad && !odd) scale /= sqrtf(fmaf(r.ss, P.inv_n, P.eps));
    if (G >= 32 ? odd : __any_sync(FULL_MASK, odd)) {
      // the squares left the range of 32 bits: sum them again as (v 2^-e)^2
      RowSums m{0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) m.top = max_abs_nan(m.top, RowType<T>::get(v[k].e[i]));
      m = reduce<G, false, false>(m);
      const int e = odd ? ilogbf(m.top) : 0;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float q = ldexpf(RowType<T>::get(v[k].e[i]), -e);
          m.ss = fmaf(q, q, m.ss);
        }
      m = reduce<G, false, true>(m);
      if (odd) {
        const double mean = ldexp((double)m.ss * (double)P.inv_n, 2 * e) + (double)P.eps;
        scale = (float)((double)r.top / 127.0 / sqrt(mean));
      }
    }
  }
  if (dst < 0) return;  // nothing below needs the other lanes
  if (bad) scale = __uint_as_float(0x7fffffffu);  // a NaN without the sign that marks claims
  if (lane == 0) P.scales[dst] = scale;

  int8_t* out = P.codes + dst * P.code_stride;
  // tiny rows are brought into range by a power of two, so 127 / top stays finite
  const float pre = r.top < 1e-18f ? 1.2089258196146292e24f : 1.f;  // 2^80
  const float inv = bad || r.top == 0.f ? 0.f : 127.f / (r.top * pre);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * G + lane) * V;
    uint32_t n[V];
    float off = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float t;
      if constexpr (FULL) t = u[k][i];
      else t = RowType<T>::get(v[k].e[i]);
      if (pre != 1.f) t *= pre;
      const float big = fmaf(t, inv, ROUNDER);
      off = fmaxf(off, fabsf(fmaf(t, inv, ROUNDER - big)));
      n[i] = __float_as_uint(big);
    }
    if (off > NEAR_HALF) {
      const double a = (double)r.top + (double)r.low;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float w = 1.f;
        if constexpr (FULL) {
          if (P.w && c + i < d)
            w = P.w_f32 ? __ldg(reinterpret_cast<const float*>(P.w) + c + i)
                        : RowType<T>::get(reinterpret_cast<const T*>(P.w)[c + i]);
        }
        n[i] = (uint32_t)code_near_half(RowType<T>::get(v[k].e[i]), w, a);
      }
    }
    if (bad) {
#pragma unroll
      for (int i = 0; i < V; ++i) n[i] = 0;
    }
    uint32_t q[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      q[i] = __byte_perm(__byte_perm(n[4 * i], n[4 * i + 1], 0x0040), __byte_perm(n[4 * i + 2], n[4 * i + 3], 0x0040),
                         0x5410);
    if (P.wide_out && c + V <= d) {
      if constexpr (V == 4) *reinterpret_cast<uint32_t*>(out + c) = q[0];
      else *reinterpret_cast<uint2*>(out + c) = make_uint2(q[0], q[1]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (c + i < d) out[c + i] = (int8_t)(q[i / 4] >> (8 * (i % 4)));
    }
  }
}

// ---------------------------------------------------------------- rows read back
struct ReadParams {
  const int8_t* codes;
  const float* scales;
  const void* ids;  // nullptr: row i
  void* out;
  int64_t n, rows, code_stride, out_stride;
  int d, id64, wide_in, wide_out;
};

// A warp reads R rows together (their loads are in flight at once), 16 bytes of
// output a lane, row and step.  An id below 0 is an empty place (zeros), one past
// the store a mistake (NaN).
template <typename T, int R>
__global__ void __launch_bounds__(256) k_dequantize_rows(ReadParams P) {
  constexpr int V = RowType<T>::V;
  const int lane = threadIdx.x & 31;
  const int64_t i0 = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) / 32 * R;
  if (i0 >= P.n) return;
  bool known[R];
  float scale[R];
  const int8_t* in[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    int64_t id = -1;
    if (i0 + r < P.n) id = P.ids ? slot_at(P.ids, P.id64, i0 + r) : i0 + r;
    known[r] = id >= 0 && id < P.rows;
    scale[r] = known[r] ? __ldg(P.scales + id) : id < 0 ? 0.f : __uint_as_float(0x7fffffffu);
    in[r] = P.codes + (known[r] ? id : 0) * P.code_stride;
  }
  for (int c = lane * V; c < P.d; c += 32 * V) {
    uint32_t w[R][V / 4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int k = 0; k < V / 4; ++k) w[r][k] = 0;
      if (!known[r]) continue;
      if (P.wide_in && c + V <= P.d) {
        if constexpr (V == 4) {
          w[r][0] = __ldg(reinterpret_cast<const uint32_t*>(in[r] + c));
        } else {
          const uint2 b = __ldg(reinterpret_cast<const uint2*>(in[r] + c));
          w[r][0] = b.x;
          w[r][1] = b.y;
        }
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (c + k < P.d) w[r][k / 4] |= (uint32_t)(uint8_t)__ldg(in[r] + c + k) << (8 * (k % 4));
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (i0 + r >= P.n) break;
      Vec<T> v;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        // code + 128 in the low byte of 2^23, less 2^23 + 128: the code as a float
        const uint32_t biased = w[r][k / 4] ^ 0x80808080u;
        const float code = __uint_as_float(__byte_perm(biased, 0x4b000000u, 0x7540 | (k % 4))) - 8388736.f;
        v.e[k] = RowType<T>::put(code * scale[r]);  // the value's one rounding
      }
      store_vec(reinterpret_cast<T*>(P.out) + (i0 + r) * P.out_stride, c, P.d, P.wide_out, v);
    }
  }
}

// ---------------------------------------------------------------- host side
template <typename T, int G, int NV, bool FULL>
static void launch_quantize(const QuantizeParams& P, cudaStream_t st) {
  constexpr int threads = quantize_threads(G), rows = threads / G;
  k_quantize_rows<T, G, NV, FULL><<<(unsigned)((P.n + rows - 1) / rows), threads, 0, st>>>(P);
}
template <typename T, int G, bool FULL>
static void quantize_nv(const QuantizeParams& P, int vectors, cudaStream_t st) {
  const int nv = (vectors + G - 1) / G;
  if (nv <= 1) launch_quantize<T, G, 1, FULL>(P, st);
  else if (nv <= 2) launch_quantize<T, G, 2, FULL>(P, st);
  else if (nv <= 3) launch_quantize<T, G, 3, FULL>(P, st);
  else if (G < 512 || RowType<T>::V == 8 || nv <= 4) launch_quantize<T, G, 4, FULL>(P, st);
  else if constexpr (G == 512 && RowType<T>::V == 4) launch_quantize<T, G, 8, FULL>(P, st);
}
// Threads a row: 8 lanes while they hold the row in at most 4 vectors each, then
// a warp, a block of 128 and a block of 512 (up to 8 vectors: 16,384 fp32 values).
template <typename T, bool FULL>
static void quantize(const QuantizeParams& P, cudaStream_t st) {
  const int vectors = (P.d + RowType<T>::V - 1) / RowType<T>::V;
  if (vectors <= 8 * 4) quantize_nv<T, 8, FULL>(P, vectors, st);
  else if (vectors <= 32 * 4) quantize_nv<T, 32, FULL>(P, vectors, st);
  else if (vectors <= 128 * 4) quantize_nv<T, 128, FULL>(P, vectors, st);
  else quantize_nv<T, 512, FULL>(P, vectors, st);
}

static void dequantize(const ReadParams& P, int dtype, cudaStream_t st) {
  const bool many = P.n >= 148 * 32;
  const unsigned blocks = (unsigned)(many ? (P.n + 31) / 32 : (P.n + 7) / 8);
  if (dtype == CIRCUIT_F32) many ? k_dequantize_rows<float, 4><<<blocks, 256, 0, st>>>(P)
                                 : k_dequantize_rows<float, 1><<<blocks, 256, 0, st>>>(P);
  else if (dtype == CIRCUIT_F16) many ? k_dequantize_rows<__half, 4><<<blocks, 256, 0, st>>>(P)
                                      : k_dequantize_rows<__half, 1><<<blocks, 256, 0, st>>>(P);
  else many ? k_dequantize_rows<__nv_bfloat16, 4><<<blocks, 256, 0, st>>>(P)
            : k_dequantize_rows<__nv_bfloat16, 1><<<blocks, 256, 0, st>>>(P);
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
  // one access a vector where the rows allow it
  P.wide_in = (on16(rows, row_stride * e) ? 1 : 0) | (residual && on16(residual, residual_stride * e) ? 2 : 0) |
              (residual && on16(summed, summed_stride * e) ? 4 : 0) | (weight && on16(weight, 0) ? 8 : 0);
  P.wide_out = (((uintptr_t)codes | (uintptr_t)code_stride) & 7) == 0;
  cudaStream_t st = (cudaStream_t)stream;
  // Equal slots: each row of a short write looks through the later ones; a long
  // write claims its slots first, the claims standing in the scales.
  P.claimed = slots && n > 1024;
  if (P.claimed) {
    const unsigned blocks = (unsigned)((n + 255) / 256);
    k_reset_slots<<<blocks, 256, 0, st>>>(slots, P.slot64, n, capacity, scales);
    k_claim_slots<<<blocks, 256, 0, st>>>(slots, P.slot64, n, capacity, scales);
  }
  const bool full = norm != CIRCUIT_NORM_NONE;
  if (dtype == CIRCUIT_F32) full ? quantize<float, true>(P, st) : quantize<float, false>(P, st);
  else if (dtype == CIRCUIT_F16) full ? quantize<__half, true>(P, st) : quantize<__half, false>(P, st);
  else full ? quantize<__nv_bfloat16, true>(P, st) : quantize<__nv_bfloat16, false>(P, st);
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
  if (!codes || !scales || !out) return bad("dequantize_rows: null pointer");
  if (!ids && rows < n) return bad("dequantize_rows: more rows asked for than there are");
  if (code_stride < dim || out_stride < dim) return bad("dequantize_rows: a row stride is smaller than dim");
  if ((uintptr_t)out % e || (uintptr_t)scales % 4 || (ids && (uintptr_t)ids % id_bytes))
    return bad("dequantize_rows: a pointer is not aligned to its type");
  ReadParams P{codes, scales, ids, out, n, rows, code_stride, out_stride, dim, id_bytes == 8,
               (((uintptr_t)codes | (uintptr_t)code_stride) & 7) == 0, on16(out, out_stride * e)};
  cudaStream_t st = (cudaStream_t)stream;
  dequantize(P, dtype, st);
  return check(cudaGetLastError(), "dequantize_rows launch");
}

}  // extern "C"
