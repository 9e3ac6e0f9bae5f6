// The kernels behind circuit_op_quantize_rows and circuit_op_dequantize_rows.
//
// Mathematics.  With v = x (+ residual, rounded once to the row's type) and
// u = v * w, a row's codes are rint(127 u_j / a), a = max|u|, and its scale is
// a / 127 times the norm's factor.  The norm's factor cancels in the codes, so
// they depend on no sum and are the same whatever its order: k_quantize_rows
// gives the correctly rounded code of the real quotient (below), and only
// the scale carries the rounding of the 32-bit sum of squares.
#pragma once

#include <cfloat>
#include <type_traits>

#include "int8_rows.h"

namespace cb {
namespace i8 {

// ---------------------------------------------------------------- helpers
struct RowSums {
  float top, low;  // max |u| as the unevaluated sum top + low (top: the rounded product; its sign says nothing before
                   // the reduction); top NaN or inf: a bad row
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
  r.top = fabsf(r.top);
  constexpr int W = G < 32 ? G : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    const float t = __shfl_xor_sync(FULL_MASK, r.top, o);
    if constexpr (LOW) raise(r.top, r.low, t, __shfl_xor_sync(FULL_MASK, r.low, o));
    else r.top = fabsf(max_abs_nan(r.top, t));
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
      else r.top = fabsf(max_abs_nan(r.top, part[w].top));
      if constexpr (SS) r.ss += part[w].ss;
    }
  }
  return r;
}

// Codes.  127 / top in 32 bits is taken a little up (hi) and down (lo), by 2^-21
// of its size.  One FMA adds u * hi to 1.5 * 2^23, whose low byte is then the
// nearest integer.  u, top and the division are off by 2^-24 of their size each and
// hi and lo by another, so the real quotient lies between u * lo and u * hi: where
// both give the same integer it is the code, where not (within 127 2^-21 = 6e-5 of
// a half: 0.006 % of the values) 254 v w is compared with (2 n + 1) top exactly
// (exact_codes).
//
// 16-bit values without a weight have m < 2^11 steps of their exponent, as has top
// (ma): 127 v / top = 127 mv / (ma 2^k) is either a half, or 1 / (2 ma 2^k) >=
// 2^-19 of its size away from one, more than hi's 10 * 2^-24.  A half needs 254 mv =
// (2 n + 1) ma 2^k, so the prime 127 divides 2 n + 1 (which is then 127: v = top / 2,
// a value that 16-bit rows often hold, and n = 63 goes to the even 64, as u * hi says)
// or ma.  So hi alone gives the code unless 127 divides ma.  The one such significand
// of bf16, 254, makes 127 / top a power of two, which alone gives the code, halves
// (every second value there) to even; the eight of fp16 take the general way.
constexpr float ROUNDER = 12582912.f;
// Whether 127 does not divide the significand of a 16-bit value's magnitude.
template <typename T>
__device__ __forceinline__ bool free_of_127(float top) {
  constexpr int DROP = std::is_same<T, __half>::value ? 13 : 16;  // fp32 bits that the type does not have
  return (((__float_as_uint(top) & 0x7fffffu) | 0x800000u) >> DROP) % 127u != 0u;
}

constexpr int row_threads(int G) { return G <= 32 ? 128 : G; }

// The weights of elements [c, c + E) of a row.
template <typename T, int E>
__device__ __forceinline__ void load_weights(const QuantizeParams& P, int c, int d, float (&w)[E]) {
  if (!P.w) {
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] = 1.f;
  } else if (P.w_f32) {
    constexpr int S = E < 4 ? E : 4;
#pragma unroll
    for (int i = 0; i < E; i += S) {
      const auto b = Vec<float, S>::load(reinterpret_cast<const float*>(P.w), c + i, d);
#pragma unroll
      for (int j = 0; j < S; ++j) w[i + j] = b.e[j];
    }
  } else {
    const auto b = Vec<T, E>::load(reinterpret_cast<const T*>(P.w), c, d);
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] = RowType<T>::get(b.e[i]);
  }
}

// The codes n[i] & 255 of elements [c, c + E).
template <int E>
__device__ __forceinline__ void store_codes(int8_t* out, int c, const uint32_t (&n)[E], bool bad) {
  uint32_t q[(E + 3) / 4];
#pragma unroll
  for (int i = 0; i < (E + 3) / 4; ++i) {
    q[i] = E == 1 ? n[0] : __byte_perm(n[4 * i], n[E == 1 ? 0 : 4 * i + 1], 0x0040);
    if constexpr (E >= 4) q[i] = __byte_perm(q[i], __byte_perm(n[4 * i + 2], n[4 * i + 3], 0x0040), 0x5410);
    if (bad) q[i] = 0;
  }
  typename Word<E>::type word;
  memcpy(&word, q, E);
  *reinterpret_cast<typename Word<E>::type*>(out + c) = word;
}

// Rare: the scale of a row whose squares leave the range of 32 bits, from
// sum (v 2^-e)^2.  Each thread reads its own elements again (src: the row as
// kept), in a rolled loop.
template <typename T, int E, int G>
__device__ __noinline__ float wide_range_scale(const T* src, int d, float top, float inv_n, float eps, bool odd) {
  const int lane = threadIdx.x % G;
  RowSums m{0.f, 0.f, 0.f};
  for (int c = lane * E; c < d; c += G * E)
    for (int i = 0; i < E; ++i) m.top = max_abs_nan(m.top, RowType<T>::get(src[c + i]));
  m = reduce<G, false, false>(m);
  const int e = odd ? ilogbf(m.top) : 0;
  for (int c = lane * E; c < d; c += G * E)
    for (int i = 0; i < E; ++i) {
      const float q = ldexpf(RowType<T>::get(src[c + i]), -e);
      m.ss = fmaf(q, q, m.ss);
    }
  m = reduce<G, false, true>(m);
  return (float)((double)top / 127.0 / sqrt(ldexp((double)m.ss * (double)inv_n, 2 * e) + (double)eps));
}

template <typename T>
__device__ __forceinline__ float weight(const QuantizeParams& P, int i) {
  if (!P.w) return 1.f;
  return P.w_f32 ? reinterpret_cast<const float*>(P.w)[i] : RowType<T>::get(reinterpret_cast<const T*>(P.w)[i]);
}
// n or n + 1, as 254 u lies below or above (2 n + 1) a, of a half the even one.  Both
// products take up to 56 bits: each is held as its rounded value and the rest, which an
// FMA gives.
__device__ __forceinline__ int nearest(double u, double a, int n) {
  const double m = (double)(2 * n + 1), l = __dmul_rn(254.0, u), r = __dmul_rn(m, a);
  const double above = __dadd_rn(__dsub_rn(l, r), __dsub_rn(__fma_rn(254.0, u, -l), __fma_rn(m, a, -r)));
  return n + (above > 0.0 || (above == 0.0 && (n & 1)));
}

// Rare: codes of elements [c, c + e) from the row's exact maximum a, halves decided
// exactly (hi = 0: the row is too small for 32 bits throughout, and n is the quotient
// rounded down, or one off next to a whole number).
template <typename T>
__device__ __noinline__ void exact_codes(const QuantizeParams& P, const T* src, int8_t* out, int c, int e, double a,
                                         float hi, float lo) {
  for (int i = c; i < c + e; ++i) {
    const float v = RowType<T>::get(src[i]), w = weight<T>(P, i), t = fabsf(v * w);
    int n = (int)(fmaf(t, lo, ROUNDER) - ROUNDER);
    if (hi == 0.f || n != (int)(fmaf(t, hi, ROUNDER) - ROUNDER)) {
      const double u = fabs((double)v * (double)w);  // 48 bits
      n = nearest(u, a, hi == 0.f ? (int)(u * 127.0 / a) : n);
    }
    out[i] = (int8_t)(v * w < 0.f ? -n : n);
  }
}

// Rare: a row whose largest product with the weights is so small that 32 bits hold it
// with few digits or not at all: its codes and scale in 64 bits, over what the kernel
// wrote for it (each thread its own elements).  All threads of a warp or block come
// here; rows that are not faint, or have no place (dst < 0), are left alone.
template <typename T, int E, int G>
__device__ __noinline__ void faint_row(const QuantizeParams& P, const T* src, int d, bool faint, int64_t dst) {
  const int lane = threadIdx.x % G;
  uint32_t bits = 0;  // rows of zeros end here
  for (int c = lane * E; c < d && faint; c += G * E) bits |= Vec<T, E>::load(src, c, d).bits();
  if constexpr (G > 32) bits = __syncthreads_or(bits);
  else bits = __any_sync(FULL_MASK, bits);
  if (!bits) return;
  RowSums m{0.f, 0.f, 0.f};
  double a = 0.0;
  for (int c = lane * E; c < d; c += G * E)
    for (int i = 0; i < E; ++i) {
      m.top = max_abs_nan(m.top, RowType<T>::get(src[c + i]));
      a = fmax(a, fabs((double)RowType<T>::get(src[c + i]) * (double)weight<T>(P, c + i)));
    }
  m = reduce<G, false, false>(m);
#pragma unroll
  for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) a = fmax(a, __shfl_xor_sync(FULL_MASK, a, o));
  if constexpr (G > 32) {
    __shared__ double part[G / 32];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
    __syncthreads();
    for (int w = 0; w < G / 32; ++w) a = fmax(a, part[w]);
  }
  const int e = faint && m.top > 0.f ? ilogbf(m.top) : 0;
  for (int c = lane * E; c < d; c += G * E)
    for (int i = 0; i < E; ++i) {
      const float q = ldexpf(RowType<T>::get(src[c + i]), -e);
      m.ss = fmaf(q, q, m.ss);
    }
  m = reduce<G, false, true>(m);
  if (!faint || dst < 0 || a == 0.0) return;  // a = 0: the zeros that the kernel wrote
  if (lane == 0)
    P.scales[dst] = (float)(a / 127.0 / sqrt(ldexp((double)m.ss * (double)P.inv_n, 2 * e) + (double)P.eps));
  int8_t* out = P.codes + dst * P.code_stride;
  for (int c = lane * E; c < d; c += G * E)
    for (int i = c; i < c + E; ++i) {
      const double p = (double)RowType<T>::get(src[i]) * (double)weight<T>(P, i), u = fabs(p);
      const int n = nearest(u, a, (int)(u * 127.0 / a));
      out[i] = (int8_t)(p < 0.0 ? -n : n);
    }
}

// G threads a row (8 or 16 lanes, a warp, or a block), the row in NV vectors of E
// elements a thread: it is read once.  FULL: with residual, weight and norm as the
// parameters say; otherwise the plain quantisation.  With fewer lanes a row the
// work of each row (reduction, addresses, scale) is shared by the rows of a warp.
template <typename T, int E, int G, int NV, bool FULL>
__global__ void __launch_bounds__(row_threads(G)) k_quantize_rows(const __grid_constant__ QuantizeParams P) {
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x % G;
  const int64_t row = (int64_t)blockIdx.x * (row_threads(G) / G) + threadIdx.x / G;
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
  Vec<T, E> v[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) v[k] = Vec<T, E>::load(x, (k * G + lane) * E, d);
  RowSums r{0.f, 0.f, 0.f};
  // products of narrow words are kept, those of wide ones (64 a thread) are made twice
  constexpr bool KEEP = FULL && E <= 2;
  [[maybe_unused]] float kept[KEEP ? NV : 1][E];
  if constexpr (FULL) {
    if (P.res) {
      const T* res = reinterpret_cast<const T*>(P.res) + (live ? row : 0) * P.res_stride;
      T* sum = reinterpret_cast<T*>(P.sum) + (live ? row : 0) * P.sum_stride;
      Vec<T, E> b[NV];
#pragma unroll
      for (int k = 0; k < NV; ++k) b[k] = Vec<T, E>::load(res, (k * G + lane) * E, d);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        // the sum is kept in the row's type, as the next layer reads it; the
        // norm and the codes are those of the kept value
        add_to<T, E>(v[k].e, b[k].e);
        v[k].store(sum, (k * G + lane) * E, d);
      }
      x = sum;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float w[E];
      load_weights<T, E>(P, (k * G + lane) * E, d, w);
      float(&u)[E] = KEEP ? kept[k % (KEEP ? NV : 1)] : kept[0];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float e = RowType<T>::get(v[k].e[i]);
        r.ss = fmaf(e, e, r.ss);
        u[i] = e * w[i];
      }
      if (P.inexact) {  // an fp32 factor: the FMA gives the product's rounding error
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float p = fabsf(u[i]);
          if (!(p < r.top)) raise(r.top, r.low, p, fmaf(fabsf(RowType<T>::get(v[k].e[i])), fabsf(w[i]), -p));
        }
      } else {  // 8- or 11-bit factors: their product is exact
#pragma unroll
        for (int i = 0; i < E; ++i) r.top = max_abs_nan(r.top, u[i]);
      }
    }
    r = P.inexact ? reduce<G, true, true>(r) : reduce<G, false, true>(r);
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) raise_top<T, E>(r.top, v[k].e);
    r = reduce<G, false, false>(r);
  }
  const bool bad = !(r.top <= FLT_MAX);

  float scale = r.top / 127.f;
  if constexpr (FULL) {
    const bool odd = r.top > 0.f && !bad && !(r.ss > 1e-25f && r.ss < FLT_MAX);
    if (r.top > 0.f && !bad && !odd) scale /= sqrtf(fmaf(r.ss, P.inv_n, P.eps));
    if (G >= 32 ? odd : __any_sync(FULL_MASK, odd)) {
      const float s = wide_range_scale<T, E, G>(x, d, r.top, P.inv_n, P.eps, odd);
      if (odd) scale = s;
    }
  }
  // products below 2^-100 lose their last digits (the FMA's rest no longer fits 32 bits)
  const bool faint = FULL && P.w && r.top < 1e-30f;
  const bool again = FULL && (G >= 32 ? faint : (bool)__any_sync(FULL_MASK, faint));
  if (dst < 0 && (G >= 32 || !again)) return;  // nothing below needs the other lanes, but for the last step
  if (bad) scale = __uint_as_float(0x7fffffffu);  // a NaN without the sign that marks claims
  if (lane == 0 && dst >= 0) P.scales[dst] = scale;

  int8_t* out = P.codes + dst * P.code_stride;
  // rows so small that 127 / top may overflow take the 64-bit quotient throughout
  const bool tiny = r.top < 1e-18f;
  const float inv = bad || tiny ? 0.f : 127.f / r.top;
  const float hi = fmaf(inv, 4.76837158203125e-07f, inv), lo = fmaf(inv, -4.76837158203125e-07f, inv);
  uint32_t unsure = tiny && r.top > 0.f ? FULL_MASK : 0u;  // vectors to be done again
  const bool free = sizeof(T) == 2 && free_of_127<T>(r.top);
  const bool alone = sizeof(T) == 2 && !(FULL && P.w) && (std::is_same<T, __nv_bfloat16>::value || free);
  const float one = free ? hi : inv;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * G + lane) * E;
    if (c >= d || (FULL && dst < 0)) break;
    [[maybe_unused]] float w[FULL ? E : 1];
    uint32_t n[E];
    if (alone) {
#pragma unroll
      for (int i = 0; i < E; ++i) n[i] = __float_as_uint(fmaf(RowType<T>::get(v[k].e[i]), one, ROUNDER));
    } else {
      if constexpr (FULL && !KEEP) load_weights<T, E>(P, c, d, w);
      uint32_t differ = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        float t = RowType<T>::get(v[k].e[i]);
        if constexpr (KEEP) t = kept[k % NV][i];
        else if constexpr (FULL) t *= w[i];
        n[i] = __float_as_uint(fmaf(t, hi, ROUNDER));
        differ |= n[i] ^ __float_as_uint(fmaf(t, lo, ROUNDER));
      }
      if (differ) unsure |= 1u << k;
    }
    store_codes<E>(out, c, n, bad);
  }
  if (unsure && !bad && !faint && dst >= 0) {
    const double a = (double)r.top + (double)r.low;
    for (int k = 0; k < NV; ++k)
      if (unsure >> k & 1u) {
        const int c = (k * G + lane) * E;
        if (c < d) exact_codes<T>(P, x, out, c, E, a, hi, lo);
      }
  }
  if constexpr (FULL) {
    if (again) faint_row<T, E, G>(P, x, d, faint, dst);
  }
}

// ---------------------------------------------------------------- rows read back

// G lanes a row and E elements a step; NV steps' codes are in flight at once.  An
// id below 0 is an empty place (zeros), one past the store a mistake (NaN).
template <typename T, int E, int G, int NV>
__global__ void __launch_bounds__(256) k_dequantize_rows(const __grid_constant__ ReadParams P) {
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x % G;
  const int64_t i = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  if (i >= P.n) return;
  const int64_t id = P.ids ? slot_at(P.ids, P.id64, i) : i;
  const bool known = id >= 0 && id < P.rows;
  const float scale = known ? P.scales[id] : id < 0 ? 0.f : __uint_as_float(0x7fffffffu);
  const int8_t* in = P.codes + (known ? id : 0) * P.code_stride;
  T* out = reinterpret_cast<T*>(P.out) + i * P.out_stride;
  const int d = P.d, dk = known ? P.d : 0;
  for (int c0 = lane * E; c0 < d; c0 += NV * G * E) {
    uint32_t w[NV][(E + 3) / 4];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * G * E;
#pragma unroll
      for (int j = 0; j < (E + 3) / 4; ++j) w[k][j] = 0;
      if (c < dk) {
        const typename Word<E>::type word = *reinterpret_cast<const typename Word<E>::type*>(in + c);
        memcpy(w[k], &word, E);
      }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * G * E;
      if (c >= d) break;
      Vec<T, E> v;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        // code + 128 in the low byte of 2^23, less 2^23 + 128: the code as a float
        const float code =
            __uint_as_float(__byte_perm(w[k][j / 4] ^ 0x80808080u, 0x4b000000u, 0x7540 | (j % 4))) - 8388736.f;
        v.e[j] = RowType<T>::put(code * scale);  // the value's one rounding
      }
      v.store(out, c, d);
    }
  }
}

// ---------------------------------------------------------------- host side
// Lanes a row and vectors a lane.  Many rows: the fewest lanes (8, 16, 32) that
// hold the row in at most 8 vectors each, with a norm at most 4 (it has more in
// flight and in registers; 64M bf16 values in rows of 1,024: 32 x 4 77 us, 16 x 8 86;
// plain fp32 rows of 256: 8 x 8 50, 32 x 2 67).  Few rows (up to eight warps an SM with a
// warp a row, two for the longest) are latency: a warp each, from 4 vectors a lane on a
// block of 128 or 512 (700 fp32 rows of 1,024 with a norm: 4.8 us, 7.3 the other way).  Rows that are not whole 16-byte vectors on 16 bytes go element by
// element, neighbouring lanes on neighbouring elements.
constexpr int64_t FEW_ROWS = 148 * 8, FEW_LONG_ROWS = 148 * 2;

template <typename T, int E, int G, int NV, bool FULL>
static void launch_quantize(const QuantizeParams& P, cudaStream_t st) {
  constexpr int threads = row_threads(G), rows = threads / G;
  launch(k_quantize_rows<T, E, G, NV, FULL>, dim3((unsigned)((P.n + rows - 1) / rows)), threads, 0, 1, st, P);
}
// Rows of narrower words than 16 bytes: neighbouring lanes on neighbouring words.
template <typename T, int E, bool FULL>
static void quantize_fine(const QuantizeParams& P, cudaStream_t st) {
  constexpr int MOST = CIRCUIT_INT8_MAX_DIM / E;
  const int words = P.d / E;
  if (P.n <= FEW_ROWS && words > 32) {
    if (words <= 128) return launch_quantize<T, E, 32, 4, FULL>(P, st);
    if (words > 512 && words <= 1024) return launch_quantize<T, E, 128, 8, FULL>(P, st);
    if (words > 1024 && words <= 4096) return launch_quantize<T, E, 256, 16, FULL>(P, st);
  }
  if (words <= 32) launch_quantize<T, E, 4, 8, FULL>(P, st);
  else if (words <= 64) launch_quantize<T, E, 8, 8, FULL>(P, st);
  else if (words <= 128) launch_quantize<T, E, 8, 16, FULL>(P, st);
  else if (words <= 256 && P.n > FEW_ROWS) launch_quantize<T, E, 16, 16, FULL>(P, st);
  else if (words <= 512) launch_quantize<T, E, 32, 16, FULL>(P, st);
  else if (words <= 1024) launch_quantize<T, E, FULL ? 128 : 32, FULL ? 8 : 32, FULL>(P, st);
  else if (words <= 2048) launch_quantize<T, E, 128, 16, FULL>(P, st);
  else if (words <= 4096) launch_quantize<T, E, 256, 16, FULL>(P, st);
  else if constexpr (MOST > 4096) {
    if (words <= 8192) launch_quantize<T, E, 512, 16, FULL>(P, st);
    else if constexpr (MOST > 8192) launch_quantize<T, E, 512, 32, FULL>(P, st);
  }
}
// bytes: the widest word (16, or less) that the rows are whole words of.
template <typename T, bool FULL>
static void quantize(const QuantizeParams& P, int bytes, cudaStream_t st) {
  constexpr int V = RowType<T>::V;
  if (bytes < 16) {
    if constexpr (V == 8) {
      if (bytes >= 8) return quantize_fine<T, 4, FULL>(P, st);
    }
    if (bytes >= 2 * (int)sizeof(T)) return quantize_fine<T, 2, FULL>(P, st);
    return quantize_fine<T, 1, FULL>(P, st);
  }
  const int vectors = P.d / V;
  if (vectors > 8 && P.n <= (vectors <= 512 ? FEW_ROWS : FEW_LONG_ROWS)) {
    if (vectors <= 32) launch_quantize<T, V, 32, 1, FULL>(P, st);
    else if (vectors <= 64) launch_quantize<T, V, 32, 2, FULL>(P, st);
    else if (vectors <= 128) launch_quantize<T, V, 32, 4, FULL>(P, st);
    else if (vectors <= 512) launch_quantize<T, V, 128, 4, FULL>(P, st);
    else if (vectors <= 2048) launch_quantize<T, V, 512, 4, FULL>(P, st);
    else if constexpr (V == 4) launch_quantize<T, V, 512, 8, FULL>(P, st);
  } else if (vectors <= 4) launch_quantize<T, V, 4, 1, FULL>(P, st);
  else if (vectors <= 8) launch_quantize<T, V, 4, 2, FULL>(P, st);
  else if (vectors <= 16) launch_quantize<T, V, 4, 4, FULL>(P, st);
  else if (vectors <= 32) launch_quantize<T, V, 8, 4, FULL>(P, st);
  else if (vectors <= 48) launch_quantize<T, V, FULL ? 16 : 8, FULL ? 3 : 6, FULL>(P, st);
  else if (vectors <= 64) launch_quantize<T, V, FULL ? 16 : 8, FULL ? 4 : 8, FULL>(P, st);
  else if (vectors <= 96) launch_quantize<T, V, FULL ? 32 : 16, FULL ? 3 : 6, FULL>(P, st);
  else if (vectors <= 128) launch_quantize<T, V, FULL ? 32 : 16, FULL ? 4 : 8, FULL>(P, st);
  else if (vectors <= 192) launch_quantize<T, V, 32, 6, FULL>(P, st);
  else if (vectors <= 256) launch_quantize<T, V, 32, 8, FULL>(P, st);
  else if (vectors <= 384) launch_quantize<T, V, 128, 3, FULL>(P, st);
  else if (vectors <= 512) launch_quantize<T, V, 128, 4, FULL>(P, st);
  else if (vectors <= 1024) launch_quantize<T, V, 128, 8, FULL>(P, st);
  else if (vectors <= 2048) launch_quantize<T, V, 256, 8, FULL>(P, st);
  else if constexpr (V == 4) launch_quantize<T, V, 512, 8, FULL>(P, st);
}

template <typename T, int E, int G, int NV>
static void launch_read(const ReadParams& P, cudaStream_t st) {
  constexpr int rows = 256 / G;
  launch(k_dequantize_rows<T, E, G, NV>, dim3((unsigned)((P.n + rows - 1) / rows)), 256, 0, 1, st, P);
}
template <typename T, int E>
static void read_fine(const ReadParams& P, cudaStream_t st) {
  const int words = P.d / E;
  if (words <= 32) launch_read<T, E, 4, 8>(P, st);
  else if (words <= 64) launch_read<T, E, 8, 8>(P, st);
  else if (words <= 128) launch_read<T, E, 16, 8>(P, st);
  else if (words <= 256 || (words <= 1024 && P.n > FEW_ROWS)) launch_read<T, E, 32, 8>(P, st);
  else launch_read<T, E, 256, 8>(P, st);
}
template <typename T>
static void dequantize(const ReadParams& P, int bytes, cudaStream_t st) {
  constexpr int V = RowType<T>::V;
  const int vectors = P.d / V;
  if (bytes < 16) {
    if constexpr (V == 8) {
      if (bytes >= 8) return read_fine<T, 4>(P, st);
    }
    if (bytes >= 2 * (int)sizeof(T)) return read_fine<T, 2>(P, st);
    return read_fine<T, 1>(P, st);
  }
  if (vectors <= 4) launch_read<T, V, 4, 1>(P, st);
  else if (vectors <= 8) launch_read<T, V, 4, 2>(P, st);
  else if (P.n <= FEW_ROWS && vectors <= 128) launch_read<T, V, 32, 4>(P, st);
  else if (vectors <= 16) launch_read<T, V, 8, 2>(P, st);
  else if (vectors <= 32) launch_read<T, V, 8, 4>(P, st);
  else if (vectors <= 48) launch_read<T, V, 8, 6>(P, st);
  else if (vectors <= 64) launch_read<T, V, 8, 8>(P, st);
  else if (vectors <= 96) launch_read<T, V, 16, 6>(P, st);
  else if (vectors <= 128) launch_read<T, V, 16, 8>(P, st);
  else if (vectors <= 192) launch_read<T, V, 32, 6>(P, st);
  else if (vectors <= 256) launch_read<T, V, 32, 8>(P, st);
  else launch_read<T, V, 256, 4>(P, st);
}

template <typename T>
void quantize_rows(const QuantizeParams& P, int bytes, bool full, cudaStream_t st) {
  full ? quantize<T, true>(P, bytes, st) : quantize<T, false>(P, bytes, st);
}
template <typename T>
void dequantize_rows(const ReadParams& P, int bytes, cudaStream_t st) {
  dequantize<T>(P, bytes, st);
}

}  // namespace i8
}  // namespace cb
