// Rotary position embedding with several position axes (time, height, width, ...).
//
// Frequency f of a token belongs to one axis a(f); its angle is
//     theta_f = position[a(f)][token] * inv_freq[f]
// and the pair (x_f, x_{f + R/2}) of every head of q and k turns by it:
//     lo' = lo cos - hi sin,   hi' = hi cos + lo sin,
// columns R .. dim - 1 pass through.  The gradient is the same map with -theta (`inverse`).
//
// HBM-bound: q and k are read and written once, and positions are a few bytes per token, where tables of cos and
// sin would add 2 * dim elements per token.  The angles are formed in the kernel, once per token and frequency, and
// shared by its heads: the product is taken in turns, in twice 64 bits, and only its fraction is kept, since at position
// 10^6 a 32-bit product is off by 0.06 rad; the sine and cosine of the fraction are 32-bit, with the rounding of
// their argument put back to first order.  The rotation is 32-bit with one rounding at the store.
#include "common.cuh"

namespace dlb {

namespace mar {
constexpr int THREADS = 256;
constexpr int MAX_HALF = 256;     // frequencies per head
constexpr int MAX_AXES = 8;
}  // namespace mar

struct MultiAxisParams {
  const void *q, *k;
  void *qo, *ko;
  const void* positions;            // [axes, tokens] int32 or int64
  const float* inv_freq;            // [half]
  int64_t pos_stride;
  int64_t q_st, q_sh, k_st, k_sh, qo_st, qo_sh, ko_st, ko_sh;
  int64_t tokens;
  int hq, hk, dim, half, pos_is_int64, rest;    // rest = columns to copy behind the rotated ones
  float sign;
  uint8_t axis[mar::MAX_HALF];
};

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) ElemVec {
  T v[VEC];
};

// What is left of pos * freq / (2 pi) turns without the whole ones, in [-1/2, 1/2].  Both products are carried in two parts, the
// second the exact remainder of the first, and so is 1 / (2 pi): with single products the angle at position 2^31 is off by
// 4e-7, seven roundings of a 32-bit result.  Off by 2^-54 of a turn up to position 2^40 and by 2^-43 up to 2^53, past which
// whole numbers are no longer exact in 64 bits.
__device__ __forceinline__ double fraction_of_turns(double pos, double freq) {
  constexpr double TURN = 0x1.45f306dc9c883p-3, TURN_REST = -0x1.6b01ec5417056p-57;      // 1 / (2 pi), 0.159..., to 106 bits
  const double angle = __dmul_rn(pos, freq), angle_rest = fma(pos, freq, -angle);
  const double turns = __dmul_rn(angle, TURN), turns_rest = fma(angle, TURN, -turns);
  const double part = (turns - rint(turns)) + (turns_rest + fma(angle, TURN_REST, angle_rest * TURN));
  return part - rint(part);
}

// A CTA forms the cos / sin of TOK tokens in shared memory, then its threads walk the tokens' items: VEC columns of a head's
// lower half and the matching ones of the upper half, or two vectors of the columns behind them.
template <typename T, int VEC, int TOK>
__global__ void __launch_bounds__(mar::THREADS, VEC == 8 ? 6 : 8) multi_axis_rotary_kernel(const __grid_constant__ MultiAxisParams p) {
  using V = ElemVec<T, VEC>;
  __shared__ __align__(16) float s_cos[TOK * mar::MAX_HALF], s_sin[TOK * mar::MAX_HALF];
  const int64_t t0 = (int64_t)blockIdx.x * TOK;
  const int ntok = (int)min((int64_t)TOK, p.tokens - t0);
  const int hv = p.half / VEC, rv = p.rest / VEC;    // items of the pairs; vectors behind them, two to an item
  // Item i's values lie in quads, quad g of all items side by side, so that lanes next to one another read 16 bytes apart
  auto place = [&](int tl, int f) {
    const int i = f / VEC, j = f % VEC;
    return tl * mar::MAX_HALF + (VEC < 4 ? f : (j >> 2) * hv * 4 + i * 4 + (j & 3));
  };
  for (int idx = threadIdx.x; idx < ntok * p.half; idx += mar::THREADS) {
    const int tl = TOK == 1 ? 0 : idx / p.half;
    const int f = idx - tl * p.half;
    const int64_t at = (int64_t)p.axis[f] * p.pos_stride + t0 + tl;
    const double pos = p.pos_is_int64 ? (double)reinterpret_cast<const int64_t*>(p.positions)[at]
                                      : (double)reinterpret_cast<const int32_t*>(p.positions)[at];
    const double part = 2.0 * fraction_of_turns(pos, (double)p.inv_freq[f]);        // in half turns
    const float x = (float)part;
    const float off = (float)(part - (double)x) * 3.14159265358979f;
    float s, c;
    sincospif(x, &s, &c);
    s_cos[place(tl, f)] = fmaf(-s, off, c);
    s_sin[place(tl, f)] = fmaf(c, off, s) * p.sign;
  }
  __syncthreads();
  const int width = hv + (rv + 1) / 2;
  const int per_token = (p.hq + p.hk) * width;
  for (int idx = threadIdx.x; idx < ntok * per_token; idx += mar::THREADS) {
    const int tl = TOK == 1 ? 0 : idx / per_token;
    const int rem = idx - tl * per_token;
    const int h = rem / width;
    const int i = rem - h * width;
    const int64_t t = t0 + tl;
    const T* src;
    T* dst;
    if (h < p.hq) {
      src = reinterpret_cast<const T*>(p.q) + t * p.q_st + (int64_t)h * p.q_sh;
      dst = reinterpret_cast<T*>(p.qo) + t * p.qo_st + (int64_t)h * p.qo_sh;
    } else {
      src = reinterpret_cast<const T*>(p.k) + t * p.k_st + (int64_t)(h - p.hq) * p.k_sh;
      dst = reinterpret_cast<T*>(p.ko) + t * p.ko_st + (int64_t)(h - p.hq) * p.ko_sh;
    }
    if (i < hv) {
      V lo = *reinterpret_cast<const V*>(src + i * VEC), hi = *reinterpret_cast<const V*>(src + p.half + i * VEC);
      constexpr int QUAD = VEC < 4 ? 1 : 4;
#pragma unroll
      for (int g = 0; g < VEC / QUAD; ++g) {
        float c[QUAD], s[QUAD];
        const int at = tl * mar::MAX_HALF + (g * hv + i) * QUAD;
        *reinterpret_cast<ElemVec<float, QUAD>*>(c) = *reinterpret_cast<const ElemVec<float, QUAD>*>(s_cos + at);
        *reinterpret_cast<ElemVec<float, QUAD>*>(s) = *reinterpret_cast<const ElemVec<float, QUAD>*>(s_sin + at);
#pragma unroll
        for (int j = 0; j < QUAD; ++j) {
          const float a = Elem<T>::to_f(lo.v[g * QUAD + j]), b = Elem<T>::to_f(hi.v[g * QUAD + j]);
          lo.v[g * QUAD + j] = Elem<T>::from_f(fmaf(a, c[j], -b * s[j]));
          hi.v[g * QUAD + j] = Elem<T>::from_f(fmaf(b, c[j], a * s[j]));
        }
      }
      *reinterpret_cast<V*>(dst + i * VEC) = lo;
      *reinterpret_cast<V*>(dst + p.half + i * VEC) = hi;
    } else {
      const int col = 2 * p.half + (i - hv) * 2 * VEC;
      const bool both = (i - hv) * 2 + 1 < rv;
      const V a = *reinterpret_cast<const V*>(src + col);
      V b;
      if (both) b = *reinterpret_cast<const V*>(src + col + VEC);
      *reinterpret_cast<V*>(dst + col) = a;
      if (both) *reinterpret_cast<V*>(dst + col + VEC) = b;
    }
  }
}

template <typename T, int VEC> static int launch_multi_axis(const MultiAxisParams& p, cudaStream_t s) {
  // Four tokens to a CTA, one where there are so few that they would not cover the SMs.  CTAs per SM (what the registers
  // are cut to): 16-byte items, 32768 tokens of 32 + 8 heads of 128 in bf16: 125.0 us at 4, 115.5 at 5, 108.7 at 6 (6.2
  // TB/s), 109.8 at 8, where some values spill; 8-byte items, 9217 tokens of 16 + 16 heads of 80: 31.9 / 32.2 / 28.4 / 26.3.
  // Eight tokens to a CTA: 111.2 and 31.0.
  if (p.tokens > 4 * 148)
    multi_axis_rotary_kernel<T, VEC, 4><<<(unsigned)((p.tokens + 3) / 4), mar::THREADS, 0, s>>>(p);
  else
    multi_axis_rotary_kernel<T, VEC, 1><<<(unsigned)p.tokens, mar::THREADS, 0, s>>>(p);
  DLB_CUDA_LAUNCH_CHECK();
  return DLB_OK;
}

}  // namespace dlb

extern "C" int dlb_multi_axis_rotary(const void* q, const void* k, void* q_out, void* k_out, const void* positions,
                                     int positions_are_int64, int64_t position_stride, const float* inv_freq,
                                     const uint8_t* axis_of_freq, int axes, int64_t tokens, int hq, int hk, int dim,
                                     int rot_dim, int64_t q_stride_t, int64_t q_stride_h, int64_t k_stride_t,
                                     int64_t k_stride_h, int64_t qo_stride_t, int64_t qo_stride_h, int64_t ko_stride_t,
                                     int64_t ko_stride_h, int inverse, int dtype, void* stream) {
  DLB_NVTX("dlb_multi_axis_rotary");
  using namespace dlb;
  DLB_CHECK_ARG(tokens >= 0 && hq >= 0 && hk >= 0 && dim >= 2, DLB_ERR_BAD_ARG, "multi_axis_rotary: bad sizes");
  DLB_CHECK_ARG(rot_dim >= 2 && rot_dim % 2 == 0 && rot_dim <= dim && rot_dim <= 2 * mar::MAX_HALF, DLB_ERR_UNSUPPORTED,
                "multi_axis_rotary: %d of %d columns rotated (need an even number up to %d)", rot_dim, dim, 2 * mar::MAX_HALF);
  DLB_CHECK_ARG(axes >= 1 && axes <= mar::MAX_AXES, DLB_ERR_UNSUPPORTED, "multi_axis_rotary: %d axes (1 to %d)", axes,
                mar::MAX_AXES);
  DLB_CHECK_ARG(dtype == DLB_DTYPE_BF16 || dtype == DLB_DTYPE_F16 || dtype == DLB_DTYPE_F32, DLB_ERR_UNSUPPORTED,
                "multi_axis_rotary: unsupported dtype %d", dtype);
  DLB_CHECK_ARG(axis_of_freq != nullptr, DLB_ERR_BAD_ARG, "multi_axis_rotary: null pointer");
  MultiAxisParams p;
  for (int f = 0; f < rot_dim / 2; ++f) {
    DLB_CHECK_ARG(axis_of_freq[f] < axes, DLB_ERR_BAD_ARG, "multi_axis_rotary: frequency %d names axis %d of %d", f,
                  (int)axis_of_freq[f], axes);
    p.axis[f] = axis_of_freq[f];
  }
  if (tokens == 0 || hq + hk == 0) return DLB_OK;
  DLB_CHECK_ARG(tokens < (1LL << 31), DLB_ERR_TOO_LARGE, "multi_axis_rotary: too many tokens");
  DLB_CHECK_ARG(positions && inv_freq && (hq == 0 || (q && q_out)) && (hk == 0 || (k && k_out)), DLB_ERR_BAD_ARG,
                "multi_axis_rotary: null pointer");
  p.q = q; p.k = k; p.qo = q_out; p.ko = k_out;
  p.positions = positions; p.inv_freq = inv_freq; p.pos_stride = position_stride;
  p.q_st = q_stride_t; p.q_sh = q_stride_h; p.k_st = k_stride_t; p.k_sh = k_stride_h;
  p.qo_st = qo_stride_t; p.qo_sh = qo_stride_h; p.ko_st = ko_stride_t; p.ko_sh = ko_stride_h;
  p.tokens = tokens;
  p.hq = hq; p.hk = hk; p.dim = dim; p.half = rot_dim / 2; p.pos_is_int64 = positions_are_int64;
  p.sign = inverse ? -1.f : 1.f;
  const bool in_place = (hq == 0 || (q == q_out && q_stride_t == qo_stride_t && q_stride_h == qo_stride_h)) &&
                        (hk == 0 || (k == k_out && k_stride_t == ko_stride_t && k_stride_h == ko_stride_h));
  p.rest = in_place ? 0 : dim - rot_dim;
  // widest vector that every row start, both halves and the columns behind them allow; the tensors without heads are not looked at
  int64_t bits = (int64_t)(rot_dim / 2) | p.rest;
  uintptr_t ptrs = 0;
  if (hq) {
    bits |= q_stride_t | q_stride_h | qo_stride_t | qo_stride_h;
    ptrs |= (uintptr_t)q | (uintptr_t)q_out;
  }
  if (hk) {
    bits |= k_stride_t | k_stride_h | ko_stride_t | ko_stride_h;
    ptrs |= (uintptr_t)k | (uintptr_t)k_out;
  }
  cudaStream_t s = (cudaStream_t)stream;
  const int es = dtype == DLB_DTYPE_F32 ? 4 : 2;
  auto fits = [&](int vec) { return bits % vec == 0 && ptrs % (uintptr_t)(vec * es) == 0; };
  if (dtype == DLB_DTYPE_F32) return fits(4) ? launch_multi_axis<float, 4>(p, s) : launch_multi_axis<float, 1>(p, s);
  if (dtype == DLB_DTYPE_BF16)
    return fits(8) ? launch_multi_axis<__nv_bfloat16, 8>(p, s)
                   : fits(4) ? launch_multi_axis<__nv_bfloat16, 4>(p, s) : launch_multi_axis<__nv_bfloat16, 1>(p, s);
  return fits(8) ? launch_multi_axis<__half, 8>(p, s)
                 : fits(4) ? launch_multi_axis<__half, 4>(p, s) : launch_multi_axis<__half, 1>(p, s);
}
