// Shared device helpers of the kernels that encode values: e4m3 and e2m2 codes, quotients, 16-lane reductions, rows of
// three element types, and the place of a cache slot.
#pragma once
#include "spmla_common.h"

namespace spmla {

typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));

// Lane exchanges inside rows of 16 lanes (DPP: no LDS round trip): lane ^ 1, lane ^ 2 and, for values that are the same in
// 4 or 8 neighbours, the mirrored half row and row.
template <int CTRL> __device__ inline float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
constexpr int DPP_XOR1 = 0xb1, DPP_XOR2 = 0x4e, DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140;
__device__ inline float wave_max16(float v) {   // max over aligned groups of 16 lanes
  v = fmaxf(v, dpp<DPP_XOR1>(v));
  v = fmaxf(v, dpp<DPP_XOR2>(v));
  v = fmaxf(v, dpp<DPP_HALF_MIRROR>(v));
  v = fmaxf(v, dpp<DPP_MIRROR>(v));
  return v;
}
template <int CTRL> __device__ inline double dpp(double v) {
  const uint2 u = __builtin_bit_cast(uint2, v);
  return __builtin_bit_cast(double, make_uint2(f2u(dpp<CTRL>(u2f(u.x))), f2u(dpp<CTRL>(u2f(u.y)))));
}
__device__ inline double lane_of(double v, int l) {
  const uint2 u = __builtin_bit_cast(uint2, v);
  return __builtin_bit_cast(double, make_uint2(__builtin_amdgcn_readlane(u.x, l), __builtin_amdgcn_readlane(u.y, l)));
}
__device__ inline double wave_sum(double v) {   // over the wave, in one order
  v += dpp<DPP_XOR1>(v);
  v += dpp<DPP_XOR2>(v);
  v += dpp<DPP_HALF_MIRROR>(v);
  v += dpp<DPP_MIRROR>(v);
  return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}

// e2m2 magnitude index of y = |x| 2^-k >= 0 (offload_rowfmt.py:93-101 with M = 2). The products are exact
// (powers of two), so the one rounding is the fp32 add of 0.5, as in the reference.
__device__ inline uint32_t e2m2_mag(float y) {
  if (y < 1.0f) return (uint32_t)floorf(y * 4.0f + 0.5f);       // 0 .. 4
  const int e2 = (y >= 2.0f) + (y >= 4.0f);
  const float inv_stp = u2f((uint32_t)(127 + 2 - e2) << 23);     // 2^(2 - e2)
  const uint32_t nrm = ((uint32_t)(e2 + 1) << 2) + (uint32_t)floorf(y * inv_stp + 0.5f) - 4u;
  return nrm < 15u ? nrm : 15u;
}

__device__ inline uint32_t e4m3x4(float a, float b, float c, float d) {    // no NaN
  const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
// x / s correctly rounded, r = 1 / s correctly rounded, x and s finite (Markstein's division step: the remainder is exact
// unless x is below 2^-78, where the quotient by s >= 1e-12 encodes to zero either way); the sign is x's
__device__ inline float quotient(float x, float s, float r) {
  const float q = x * r;
  return copysignf(__builtin_fmaf(__builtin_fmaf(-q, s, x), r, q), x);
}
// (slot / n, slot % n) for 0 <= slot: sh = log2 n for a power of two, else -1
__device__ inline void div_slot(long long slot, int n, int sh, long long& blk, int& off) {
  if (sh >= 0) { blk = slot >> sh; off = (int)(slot & (n - 1)); }
  else if ((slot >> 31) == 0) { blk = (uint32_t)slot / (uint32_t)n; off = (int)((uint32_t)slot % (uint32_t)n); }
  else { blk = slot / n; off = (int)(slot % n); }
}
inline int log2_or(int n) { return n > 0 && (n & (n - 1)) == 0 ? __builtin_ctz((unsigned)n) : -1; }

// Row400's latent part from the wave's 512 scaled and clamped values, 8 a lane (the 4 lanes 4b .. 4b + 3 form block b)
__device__ inline void row400_latent(uint8_t* row, int lane, const float (&x)[8]) {
  float am = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) am = fmaxf(am, fabsf(x[e]));
  am = fmaxf(am, __shfl_xor(am, 1, 64));
  am = fmaxf(am, __shfl_xor(am, 2, 64));
  const uint32_t rb = f2u(am / 7.0f);
  const int ex = (int)((rb >> 23) & 255u) - 127;
  int k = ex + ((rb & 0x7fffffu) != 0u);
  k = ex < -126 ? -126 : (k < 127 ? k : 127);
  const float inv = u2f((uint32_t)(127 - k) << 23);                // 2^-k
  uint32_t nib = 0, sgn = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t mag = e2m2_mag(fabsf(x[e]) * inv);
    nib |= mag << (4 * e);
    sgn |= (x[e] < 0.f && mag > 0u ? 1u : 0u) << e;
  }
  *(uint32_t*)(row + 4 * lane) = nib;
  row[R4_SIGN + lane] = (uint8_t)sgn;
  if ((lane & 3) == 0) row[R4_K + (lane >> 2)] = (uint8_t)(int8_t)k;
}

// ---- element types of the norm, rotary and linear entry points: their dtype argument
enum : int { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2 };
template <int DT> constexpr int elem_bytes = DT == DT_F32 ? 4 : 2;

template <int DT> __device__ inline float load1(const void* p, long long i) {
  if constexpr (DT == DT_F32) return ((const float*)p)[i];
  else if constexpr (DT == DT_F16) return (float)((const _Float16*)p)[i];
  else return bf2f(((const uint16_t*)p)[i]);
}
template <int DT> __device__ inline void store1(void* p, long long i, float v) {
  if constexpr (DT == DT_F32) ((float*)p)[i] = v;
  else if constexpr (DT == DT_F16) ((_Float16*)p)[i] = (_Float16)v;
  else ((uint16_t*)p)[i] = f2bf_rne(v);
}
template <int DT> __device__ inline float round_to(float v) {      // v rounded to the type
  if constexpr (DT == DT_F32) return v;
  else if constexpr (DT == DT_F16) return (float)(_Float16)v;
  else return bf2f(f2bf_rne(v));
}
template <int DT> __device__ inline uint32_t pack2(float a, float b) {   // two values of a 16-bit type
  if constexpr (DT == DT_F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2v));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2v));
}
template <int DT> __device__ inline void unpack8(u32x4 a, float (&v)[8]) {   // eight values of a 16-bit type
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (DT == DT_F16) {
      const f16x2v h = __builtin_bit_cast(f16x2v, (uint32_t)a[e]);
      v[2 * e] = (float)h[0]; v[2 * e + 1] = (float)h[1];
    } else {
      v[2 * e] = u2f(a[e] << 16); v[2 * e + 1] = u2f(a[e] & 0xffff0000u);
    }
  }
}
// eight values from element i on: 16-byte aligned, or _any at any alignment of the type
template <int DT, class Q = u32x4> __device__ inline void load8(const void* p, long long i, float (&v)[8]) {
  if constexpr (DT == DT_F32) {
    const u32x4 a = *(const Q*)((const float*)p + i), b = *(const Q*)((const float*)p + i + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = u2f(a[e]); v[4 + e] = u2f(b[e]); }
  } else {
    unpack8<DT>(*(const Q*)((const uint16_t*)p + i), v);
  }
}
template <int DT, class Q = u32x4> __device__ inline void store8(void* p, long long i, const float (&v)[8]) {
  if constexpr (DT == DT_F32) {
    *(Q*)((float*)p + i) = u32x4{f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])};
    *(Q*)((float*)p + i + 4) = u32x4{f2u(v[4]), f2u(v[5]), f2u(v[6]), f2u(v[7])};
  } else {
    *(Q*)((uint16_t*)p + i) = u32x4{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]),
                                    pack2<DT>(v[6], v[7])};
  }
}
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef uint32_t codes8 __attribute__((ext_vector_type(2), aligned(1)));       // eight codes at any address
// Eight values of a row from element i on, the row's last n values from there (n <= 0: behind it), as the words in memory and
// then as numbers with zeros behind the row: no branch stands between several loads. WHOLE rows are whole eights, ENDS
// rows have 8 values or more (their last eight are loaded where they end earlier, and moved down), TINY ones fewer.
enum : int { WHOLE = 0, ENDS = 1, TINY = 2 };
template <int DT> struct Raw8 {
  static constexpr int NW = DT == DT_F32 ? 8 : 4;
  uint32_t w[NW];
};
template <int DT, int ROW> __device__ inline void load_raw(const void* p, long long i, int n, Raw8<DT>& r) {
  if constexpr (ROW == TINY) {
#pragma unroll
    for (int e = 0; e < Raw8<DT>::NW; ++e) r.w[e] = 0;
#pragma unroll
    for (int e = 0; e < 7; ++e) {
      if (e >= n) continue;
      if constexpr (DT == DT_F32) r.w[e] = ((const uint32_t*)p)[i + e];
      else r.w[e >> 1] |= (uint32_t)((const uint16_t*)p)[i + e] << (16 * (e & 1));
    }
  } else {
    const char* q = (const char*)p + (i + min(n - 8, 0)) * (DT == DT_F32 ? 4 : 2);
#pragma unroll
    for (int h = 0; h < Raw8<DT>::NW / 4; ++h) {
      const u32x4 a = *(const u32x4_any*)(q + 16 * h);
#pragma unroll
      for (int e = 0; e < 4; ++e) r.w[4 * h + e] = a[e];
    }
  }
}
template <int DT, int ROW> __device__ inline void values_of(Raw8<DT> r, int n, float (&v)[8]) {
  constexpr int NW = Raw8<DT>::NW;
  if constexpr (ROW == ENDS) {
    if (n < 8) {
      const int by = 8 - n;
      auto down = [&](int words) {
#pragma unroll
        for (int e = 0; e < NW; ++e) r.w[e] = e + words < NW ? r.w[e + words < NW ? e + words : 0] : 0;
      };
      if (by & 4) down(NW / 2);
      if (by & 2) down(NW / 4);
      if (by & 1) {
        if constexpr (DT == DT_F32) {
          down(1);
        } else {
#pragma unroll
          for (int e = 0; e < NW; ++e) r.w[e] = r.w[e] >> 16 | (e + 1 < NW ? r.w[e + 1 < NW ? e + 1 : 0] << 16 : 0);
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < NW; ++e) r.w[e] = n > 0 ? r.w[e] : 0;
  if constexpr (DT == DT_F32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = u2f(r.w[e]);
  } else {
    unpack8<DT>(u32x4{r.w[0], r.w[1], r.w[2], r.w[3]}, v);
  }
}
// the first n of eight values (n <= 0: none) from element i on; EIGHTS: n >= 8 or n <= 0
template <int DT, bool EIGHTS> __device__ inline void store_upto8(void* p, long long i, int n, const float (&v)[8]) {
  if (n >= 8) {
    store8<DT, u32x4_any>(p, i, v);
  } else if constexpr (!EIGHTS) {
#pragma unroll
    for (int e = 0; e < 7; ++e) {
      if (e >= n) continue;
      if constexpr (DT == DT_F32) ((float*)p)[i + e] = v[e];
      else ((uint16_t*)p)[i + e] = (uint16_t)(pack2<DT>(v[e & 6], v[(e & 6) + 1]) >> (16 * (e & 1)));
    }
  }
}

constexpr int MAX_TOKENS = 1 << 23;                // rows of a call: grids of up to 256 threads a row stay below 2^32

// A kernel's handles, one a device (ids 0 .. 63), found at its first launch there: a launch by the handle takes the host 0.1
// to 0.25 us less of a call's 4 than by the kernel's address. a: the kernel's arguments, of its own types. Safe to call from
// several host threads.
struct Launcher {
  std::atomic<hipFunction_t> known[64] = {};
  template <class... A> int operator()(const void* kernel, dim3 grid, int threads, int lds, hipStream_t s, A... a) {
    int dev = 0;
    if (const hipError_t e = hipGetDevice(&dev)) return (int)e;
    hipFunction_t f = dev >= 0 && dev < 64 ? known[dev].load(std::memory_order_acquire) : nullptr;
    if (!f) {
      if (const hipError_t e = hipGetFuncBySymbol(&f, kernel)) return (int)e;
      if (dev >= 0 && dev < 64) known[dev].store(f, std::memory_order_release);
    }
    void* args[] = {(void*)&a...};
    return (int)hipModuleLaunchKernel(f, grid.x, grid.y, grid.z, (unsigned)threads, 1, 1, (unsigned)lds, s, args, nullptr);
  }
};

// ---- e4m3 codes of values that a row's factor r scales: r = hi + lo, to 2^-40 ----------------------------------------
struct Factor {
  float hi, lo;
};
__device__ inline Factor factor_of(double r) {
  const float hi = (float)r;
  return {hi, (float)(r - (double)hi)};
}
// 1 / sqrt(m): one Newton step in 64 bits from the fp32 root where that is in range
__device__ inline double inverse_root(double m) {
  if (!(m > 1e-30 && m < 1e30)) return 1.0 / sqrt(m);
  const double r = (double)(1.0f / sqrtf((float)m));
  return r * (1.5 - 0.5 * m * r * r);
}
// p + e rounded to odd, e the rest of p's rounding: the next rounding, to fewer bits, is then that of the exact value
__device__ inline float to_odd(float p, float e) {
  const uint32_t b = f2u(p);
  return e == 0.f || (b & 1u) ? p : u2f(((f2u(e) ^ b) >> 31) ? b - 1u : b + 1u);
}
// The code grows with the value. c is within 2^-23 of a factor whose exact products with t are encoded, so these lie between
// the products with dn and with up, roundings of all included: where both have one code, it is the exact product's.
struct Around {
  float dn, up;
};
__host__ __device__ inline Around around(float c) {
  const float d = c * 0x1p-21f;
  return {c - d, c + d};
}
// codes of t times about c; whether they are decided (only what lies at a middle of two codes is not, some 2^-16 of other
// values: zeros, whole codes and a group's own maximum are)
__device__ inline bool codes_about(const float (&t)[8], float c, uint32_t& lo, uint32_t& hi) {
  const Around a = around(c);
  lo = e4m3x4(t[0] * a.up, t[1] * a.up, t[2] * a.up, t[3] * a.up);
  hi = e4m3x4(t[4] * a.up, t[5] * a.up, t[6] * a.up, t[7] * a.up);
  const uint32_t l = e4m3x4(t[0] * a.dn, t[1] * a.dn, t[2] * a.dn, t[3] * a.dn);
  const uint32_t h = e4m3x4(t[4] * a.dn, t[5] * a.dn, t[6] * a.dn, t[7] * a.dn);
  return ((lo ^ l) | (hi ^ h)) == 0u;
}
// y = t c rounded to odd: its rounding to a code is that of the exact product
__device__ inline void odd_products(const float (&t)[8], Factor c, float (&y)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float p = t[e] * c.hi;
    y[e] = to_odd(p, __builtin_fmaf(t[e], c.lo, __builtin_fmaf(t[e], c.hi, -p)));
  }
}
// y = t c, rounded to odd where a lane of the wave has one with at most four bits behind its leading one: the borders of e4m3
// and of e2m2 codes are such (so are whole codes and zeros; of values without a pattern one in 2^17 is)
__device__ inline void scaled(const float (&t)[8], Factor c, float (&y)[8]) {
  uint32_t u = 0x7ffffu;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    y[e] = t[e] * c.hi;                                          // within one unit of its last place
    u = min(u, (f2u(y[e]) + 1u) & 0x7ffffu);
  }
  if (__builtin_expect(__ballot(u <= 2u) != 0ull, 0)) odd_products(t, c, y);
}

// Codes of eight values y = t r of a group of 128 (16 lanes of 8), r >= 0 one factor of the group's row, and its scale
// s = max(amax |y| / 448, 1e-12) (ue8m0: rounded up to a power of two); the codes are those of y over s before its
// rounding to 32 bits. The largest value becomes 448 whatever r is, so without ue8m0 the quotient is 448 t / amax |t|: t
// is exact where it is a product of two 16-bit floats, and then many quotients lie halfway between two codes (one in some
// thousand): a quotient by the rounded s would round those by s's rounding error. The product with 448 / amax decides
// every code but those (codes_about); where a lane has one, the wave divides, with t and amax brought to the range in which
// the remainder is exact by a power of two: 15 % of the waves on products of normally distributed bf16 values (norm of 8192 x
// 4096 28 us, 36 if all divide). UNIT: r is 1. ties: t are 16-bit floats, whose quotients are halfway in 69 % of the waves, so
// that all that are not zeros divide at once (quantization of 4096 x 16384 52 us, 56 with the products first).
// A group of infinities or NaNs (or a row factor that is one) is divided element by element: NaN codes for NaNs and
// inf / inf.
constexpr float Q_MAX = 448.0f, Q_MIN = 1e-12f;      // largest e4m3 value, smallest scale
template <bool UNIT = false>
__device__ inline float group_codes(const float (&t)[8], Factor r, bool ue8m0, bool ties, uint32_t& lo, uint32_t& hi) {
  uint32_t top = 0;                   // largest magnitude as an integer: infinities and NaNs lie above the finite ones
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, f2u(t[e]) & 0x7fffffffu);
  top = max(top, f2u(dpp<DPP_XOR1>(u2f(top))));
  top = max(top, f2u(dpp<DPP_XOR2>(u2f(top))));
  top = max(top, f2u(dpp<DPP_HALF_MIRROR>(u2f(top))));
  top = max(top, f2u(dpp<DPP_MIRROR>(u2f(top))));
  float am = u2f(top);
  float s = fmaxf(am * r.hi / Q_MAX, Q_MIN);
  const bool odd = top >= 0x7f800000u || (f2u(r.hi) & 0x7fffffffu) >= 0x7f800000u || f2u(s) >= 0x7f800000u;
  const bool low = !(am * r.hi > Q_MAX * Q_MIN);
  auto power = [&](float v) {         // the next power of two (or infinity)
    uint32_t u = f2u(v);
    if (u & 0x7fffffu) u = (u & 0xff800000u) + 0x800000u;
    return u2f(u);
  };
  if (ue8m0) s = power(s);
  if (__builtin_expect(__ballot(odd) == 0ull, 1)) {
    float y[8];
    if (ue8m0) {
      const float f = 1.0f / s;                                  // exact
      const Factor c{r.hi * f, r.lo * f};
      if constexpr (UNIT) {                                      // so are the products
        lo = e4m3x4(t[0] * c.hi, t[1] * c.hi, t[2] * c.hi, t[3] * c.hi);
        hi = e4m3x4(t[4] * c.hi, t[5] * c.hi, t[6] * c.hi, t[7] * c.hi);
        return s;
      }
      if (__builtin_expect(__ballot(!codes_about(t, c.hi, lo, hi)) == 0ull, 1)) return s;
      odd_products(t, c, y);
    } else {
      if (ties) {
        if (__ballot(top != 0u) == 0ull) {
          lo = e4m3x4(t[0], t[1], t[2], t[3]);
          hi = e4m3x4(t[4], t[5], t[6], t[7]);
          return s;
        }
      } else {                         // outside these sizes of amax the products may lose bits: straight to the division
        const bool plain = top == 0u || (am > 0x1p-60f && am < 0x1p100f && !low);
        if (__builtin_expect(__ballot(!codes_about(t, top ? Q_MAX / am : 0.f, lo, hi) || !plain) == 0ull, 1)) return s;
      }
      const float k = am < 0x1p-60f ? 0x1p64f : am > 0x1p100f ? 0x1p-64f : 1.0f;
      const float a = low ? s : am * k, up = low ? r.hi : Q_MAX * k, f = 1.0f / a;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = t[e] * up, q = quotient(x, a, f);
        y[e] = to_odd(q, __builtin_fmaf(-q, a, x));
      }
    }
    lo = e4m3x4(y[0], y[1], y[2], y[3]);
    hi = e4m3x4(y[4], y[5], y[6], y[7]);
  } else {
    am = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) am = fmaxf(am, fabsf(t[e]));     // (NaNs aside)
    am = wave_max16(am);
    s = fmaxf(am * r.hi / Q_MAX, Q_MIN);
    if (ue8m0) s = power(s);
    lo = hi = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo |= (uint32_t)e4m3_rne(t[e] * r.hi / s) << (8 * e);
      hi |= (uint32_t)e4m3_rne(t[4 + e] * r.hi / s) << (8 * e);
    }
  }
  return s;
}

}  // namespace spmla
