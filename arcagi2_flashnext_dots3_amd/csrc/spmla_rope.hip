// Rotary positions, and a token's cache row from its down-projected latent in one launch.
//
// Rotary: pairs (a, b) of columns start .. start + 2n of a head turn by the token's position times the pair's frequency:
//   (a, b) -> factor (a cos - b sin, b cos + a sin); interleaved pairs are (2i, 2i + 1), else (i, i + n).
// The angle is formed in quarter turns, from 2 / pi and products in twice 64 bits: its distance from the nearest whole one is
// exact to 2^-54 up to positions of 2^31 (rounded products alone: to 2^-21 there), so that only its rounding to 32 bits counts;
// cosine and sine come from their Taylor series on +-45 degrees (remainders x^11 / 11! and x^12 / 12!, below 2^-28). No table
// of positions is read.
// Bound by HBM for long chunks: a head is read and written once (8192 tokens x 64 heads x 128 bf16 53 us, 268 MB, 5.0 TB/s;
// a device copy moves 5.1); 64 tokens x 128 heads 3.3 us. A thread keeps its columns and turns them for several heads of one
// token, so that an angle (some 50 instructions, 11 of them in 64 bits) is formed once for them. Loads and stores are 16
// bytes of a lane at any alignment of the type.
//
// Latent row: RMS norm of the 512 latent values and rotary of the 64 rope values, both in fp32, then the row that
// spmla_cache_write would write of them (Row656 codes: group_codes); nothing is rounded to bf16 between. One wave a token:
// 64 tokens 2.9 us (Row576) to 3.6 (Row400), the chain of slot, latent, sum and codes; 8192 tokens 5.8 us into Row576 (14 MB,
// 2.4 TB/s: too short to reach more), 6.9 into Row656, 8.2 into Row400.
#include "spmla_quant.h"

namespace spmla {
namespace rope {

__device__ inline void turn(double pos, double freq, float factor, float sign, float& c, float& s) {
  constexpr double C = 0.63661977236758134308, C_LO = -3.935735335036497e-17;   // 2 / pi: quarter turns
  const double f = freq * C, f_lo = __builtin_fma(freq, C_LO, __builtin_fma(freq, C, -f));
  const double q = pos * f, q_lo = __builtin_fma(pos, f_lo, __builtin_fma(pos, f, -q));
  const double k = rint(q);
  const float x = (float)((q - k) + q_lo) * 1.57079632679489661923f, y = x * x;
  const int n = (int)__builtin_bit_cast(uint64_t, k + 0x1.8p52) & 3;   // which quarter: the sum's last bit counts ones
  const float sn = x * (1.0f + y * (-1.0f / 6 + y * (1.0f / 120 + y * (-1.0f / 5040 + y * (1.0f / 362880)))));
  const float cs = 1.0f + y * (-0.5f + y * (1.0f / 24 + y * (-1.0f / 720 + y * (1.0f / 40320 + y * (-1.0f / 3628800)))));
  const float a = n & 1 ? sn : cs, b = n & 1 ? cs : sn;
  c = (n == 1 || n == 2 ? -a : a) * factor;
  s = (n & 2 ? -b : b) * factor * sign;
}

struct RopeParams {
  const void* x; long long x_st, x_sh;
  void* out; long long o_st, o_sh;
  const void* pos; int pos32;
  const double* freqs;
  int T, H, W, start, n, inplace;
  float factor, sign;
  int us, hp, tpb;               // unit lanes, head slots and tokens of a workgroup
};

// V = 8: units of 8 columns (two pieces of 8 in half layout), V = 1: units of one pair or one untouched column
template <int DT, int V, bool INTER>
__global__ void __launch_bounds__(256) rope_kernel(RopeParams p) {
  constexpr int NP = V == 1 ? 1 : INTER ? 4 : 8;             // pairs of a unit
  const int u0 = threadIdx.x % p.us, slot = threadIdx.x / p.us;
  const int hh = slot % p.hp, tl = slot / p.hp;
  const long long t = (long long)blockIdx.x * p.tpb + tl;
  if (tl >= p.tpb || t >= p.T) return;
  const int RU = p.n / NP, NU = RU + (p.inplace ? 0 : (p.W - 2 * p.n) / V);
  const double pos = !p.n ? 0.0 : p.pos32 ? (double)((const int*)p.pos)[t] : (double)((const long long*)p.pos)[t];
  const int h0 = hh + p.hp * (int)blockIdx.y, hs = p.hp * (int)gridDim.y;
  for (int u = u0; u < NU; u += p.us) {
    if (u < RU) {
      float c[NP], s[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) turn(pos, p.freqs[u * NP + i], p.factor, p.sign, c[i], s[i]);
      const int ca = p.start + u * NP * (INTER ? 2 : 1), cb = INTER ? ca + 1 : ca + p.n;
      for (int h = h0; h < p.H; h += hs) {
        const long long xi = t * p.x_st + h * p.x_sh, oi = t * p.o_st + h * p.o_sh;
        if constexpr (V == 1) {
          const float a = load1<DT>(p.x, xi + ca), b = load1<DT>(p.x, xi + cb);
          store1<DT>(p.out, oi + ca, a * c[0] - b * s[0]);
          store1<DT>(p.out, oi + cb, b * c[0] + a * s[0]);
        } else if constexpr (INTER) {
          float v[8], y[8];
          load8<DT, u32x4_any>(p.x, xi + ca, v);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[2 * i] = v[2 * i] * c[i] - v[2 * i + 1] * s[i];
            y[2 * i + 1] = v[2 * i + 1] * c[i] + v[2 * i] * s[i];
          }
          store8<DT, u32x4_any>(p.out, oi + ca, y);
        } else {
          float a[8], b[8], y[8], z[8];
          load8<DT, u32x4_any>(p.x, xi + ca, a);
          load8<DT, u32x4_any>(p.x, xi + cb, b);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            y[i] = a[i] * c[i] - b[i] * s[i];
            z[i] = b[i] * c[i] + a[i] * s[i];
          }
          store8<DT, u32x4_any>(p.out, oi + ca, y);
          store8<DT, u32x4_any>(p.out, oi + cb, z);
        }
      }
    } else {                                                 // columns outside the turned part: copied
      int col = (u - RU) * V;
      col += col < p.start ? 0 : 2 * p.n;
      for (int h = h0; h < p.H; h += hs) {
        const long long xi = t * p.x_st + h * p.x_sh + col, oi = t * p.o_st + h * p.o_sh + col;
        if constexpr (V == 1) {
          if constexpr (DT == DT_F32) ((uint32_t*)p.out)[oi] = ((const uint32_t*)p.x)[xi];
          else ((uint16_t*)p.out)[oi] = ((const uint16_t*)p.x)[xi];
        } else if constexpr (DT == DT_F32) {
          const u32x4_any a = *(const u32x4_any*)((const float*)p.x + xi), b = *(const u32x4_any*)((const float*)p.x + xi + 4);
          *(u32x4_any*)((float*)p.out + oi) = a;
          *(u32x4_any*)((float*)p.out + oi + 4) = b;
        } else {
          *(u32x4_any*)((uint16_t*)p.out + oi) = *(const u32x4_any*)((const uint16_t*)p.x + xi);
        }
      }
    }
  }
}

constexpr int MAX_HEAD = 1 << 30;   // heads of a token, columns of a head: the strides of the loops stay inside 32 bits

template <int DT, int V, bool INTER>
static int launch(RopeParams& p, hipStream_t s) {
  constexpr int NP = V == 1 ? 1 : INTER ? 4 : 8;
  const int NU = p.n / NP + (p.inplace ? 0 : (p.W - 2 * p.n) / V);
  p.us = NU < 256 ? NU : 256;
  const int slots = 256 / p.us;
  p.hp = p.H < slots ? p.H : slots;
  p.tpb = slots / p.hp;
  const long long gx = ((long long)p.T + p.tpb - 1) / p.tpb;
  // small batches: a token's heads over several workgroups until each compute unit has a few
  const long long most = (p.H + p.hp - 1) / p.hp, want = (1024 + gx - 1) / gx;
  const unsigned gy = (unsigned)(want < most ? want : most);
  static Launcher start;
  return start((const void*)rope_kernel<DT, V, INTER>, dim3((unsigned)gx, gy), 256, 0, s, p);
}

template <int DT>
static int go(RopeParams& p, bool vec, bool inter, hipStream_t s) {
  if (vec) return inter ? launch<DT, 8, true>(p, s) : launch<DT, 8, false>(p, s);
  return inter ? launch<DT, 1, true>(p, s) : launch<DT, 1, false>(p, s);
}

// ---- a token's cache row ------------------------------------------------------------------------------------
struct LatentParams {
  const uint16_t* kv; long long kv_st;      // [n][512 latent | 64 rope] bf16
  const void* w; int w_f32;                 // [512]; null: ones
  float eps;
  const void* pos; int pos32;
  const double* freqs;                      // [32]
  float factor;
  const long long* slots; int n;
  uint8_t* cache; long long R; int bs, sh; long long blk_stride;   // as spmla_cache_write
  int fmt;
  float inv_scale;
};

template <bool INTER>
__global__ void __launch_bounds__(256) latent_write_kernel(LatentParams p) {
  const int tok = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
  const int lane = threadIdx.x & 63, i = lane & 31;
  if (tok >= p.n) return;
  const long long slot = p.slots[tok];
  float x[8], w[8], a, b;                   // what all tokens share is on its way before the slot decides
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = 1.0f;
  if (p.w) {
    if (p.w_f32) load8<DT_F32>(p.w, lane * 8, w);
    else load8<DT_BF16>(p.w, lane * 8, w);
  }
  const double freq = p.freqs[i];
  if (slot < 0 || slot >= p.R) return;      // padding: its values are not read
  const uint16_t* kv = p.kv + (long long)tok * p.kv_st;
  load8<DT_BF16>(kv, lane * 8, x);
  if (INTER) {
    const uint32_t v = *(const uint32_t*)(kv + D_LAT + 2 * i);
    a = u2f(v << 16); b = u2f(v & 0xffff0000u);
  } else {
    a = bf2f(kv[D_LAT + i]); b = bf2f(kv[D_LAT + 32 + i]);
  }
  const double pos = p.pos32 ? (double)((const int*)p.pos)[tok] : (double)((const long long*)p.pos)[tok];
  const int rowb = p.fmt == 0 ? ROW656 : (p.fmt == 1 ? ROW576 : ROW400);
  long long blk;
  int off;
  div_slot(slot, p.bs, p.sh, blk, off);
  uint8_t* row = p.cache + blk * p.blk_stride + (long long)off * rowb;
  double ss = 0.0;
  if (p.fmt == 0) {                         // r scales codes and scale alike
    float q = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) q = __builtin_fmaf(x[e], x[e], q);
    ss = (double)q;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = __builtin_fma((double)x[e], (double)x[e], ss);
  }
  const double r = inverse_root(wave_sum(ss) * (1.0 / D_LAT) + (double)p.eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] *= w[e];
  float c, s;
  turn(pos, freq, p.factor, 1.0f, c, s);
  const float ra = a * c - b * s, rb = b * c + a * s;
  uint32_t lo, hi;
  if (p.fmt == 0) {
    const float sc = group_codes(x, factor_of(r), false, !p.w, lo, hi);
    *(uint2*)(row + lane * 8) = make_uint2(lo, hi);
    if ((lane & 15) == 0) *(float*)(row + SC_OFF + (lane >> 4) * 4) = sc;
    if (lane < 32) {
      if (INTER) {
        *(uint32_t*)(row + ROPE_OFF + 4 * i) = pack2<DT_BF16>(ra, rb);
      } else {
        *(uint16_t*)(row + ROPE_OFF + 2 * i) = f2bf_rne(ra);
        *(uint16_t*)(row + ROPE_OFF + 64 + 2 * i) = f2bf_rne(rb);
      }
    }
    return;
  }
  auto cut = [](float v) -> float { return fminf(fmaxf(v, -448.f), 448.f); };                      // (a NaN becomes -448)
  const Factor f = factor_of(r * (double)p.inv_scale);
  scaled(x, f, w);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = cut(w[e]);
  uint8_t* rp = row + D_LAT;
  if (p.fmt == 1) {
    *(uint2*)(row + lane * 8) = make_uint2(e4m3x4(x[0], x[1], x[2], x[3]), e4m3x4(x[4], x[5], x[6], x[7]));
  } else {
    row400_latent(row, lane, x);
    rp = row + R4_ROPE;
  }
  const uint32_t rc = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(cut(ra * p.inv_scale), cut(rb * p.inv_scale), 0, false);
  if (lane < 32) {
    if (INTER) {
      *(uint16_t*)(rp + 2 * i) = (uint16_t)rc;
    } else {
      rp[i] = (uint8_t)rc;
      rp[32 + i] = (uint8_t)(rc >> 8);
    }
  }
}

}  // namespace rope
}  // namespace spmla

using namespace spmla;

extern "C" {

int spmla_rope(const void* x, long long x_st, long long x_sh, const void* positions, int pos32, const double* freqs,
               int T, int H, int W, int start, int n, int interleaved, float factor, int inverse, int dtype, void* out,
               long long o_st, long long o_sh, void* stream) {
  if (T < 0 || H < 0 || W < 0 || n < 0 || start < 0 || n > W / 2 || start > W - 2 * n || dtype < 0 || dtype > 2)
    return SPMLA_EARG;
  if (T > MAX_TOKENS || H > rope::MAX_HEAD || W > rope::MAX_HEAD) return SPMLA_ELIMIT;
  const bool inplace = out == x;
  if (inplace && (x_st != o_st || x_sh != o_sh)) return SPMLA_EARG;
  if (T == 0 || H == 0 || W == 0 || (inplace && n == 0)) return SPMLA_OK;
  if (!x || !out || (n > 0 && (!positions || !freqs))) return SPMLA_EARG;
  const int eb = dtype == DT_F32 ? 4 : 2;
  if ((((uintptr_t)x | (uintptr_t)out) & (eb - 1)) || ((uintptr_t)freqs & 7) ||
      ((uintptr_t)positions & (pos32 ? 3 : 7)))
    return SPMLA_EALIGN;
  rope::RopeParams p{x, x_st, x_sh, out, o_st, o_sh, positions, pos32, freqs, T, H, W, start, n, inplace,
                     factor, inverse ? -1.0f : 1.0f, 0, 0, 0};
  const bool vec = (W & 7) == 0 && (start & 7) == 0 && (n & (interleaved ? 3 : 7)) == 0;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == DT_F32) return rope::go<DT_F32>(p, vec, interleaved != 0, s);
  if (dtype == DT_F16) return rope::go<DT_F16>(p, vec, interleaved != 0, s);
  return rope::go<DT_BF16>(p, vec, interleaved != 0, s);
}

int spmla_latent_write(const void* kv, long long kv_st, const void* weight, int weight_f32, float eps,
                       const void* positions, int pos32, const double* freqs, int interleaved, float factor,
                       const long long* slots, int n, void* cache, long long R, int block_size, long long block_stride,
                       int fmt, float kv_scale, void* stream) {
  if (n < 0 || R < 0 || fmt < 0 || fmt > 2 || block_size <= 0 || !(eps >= 0.f)) return SPMLA_EARG;
  if (n == 0) return SPMLA_OK;
  if (n > MAX_TOKENS) return SPMLA_ELIMIT;
  if (!kv || !positions || !freqs || !slots || !cache) return SPMLA_EARG;
  if (((uintptr_t)kv & 15) || (kv_st & 7) || ((uintptr_t)weight & 15) || ((uintptr_t)freqs & 7) ||
      ((uintptr_t)positions & (pos32 ? 3 : 7)) || ((uintptr_t)slots & 7))
    return SPMLA_EALIGN;
  const int rowb = fmt == 0 ? ROW656 : (fmt == 1 ? ROW576 : ROW400);
  if (((uintptr_t)cache & 7) || (block_stride & 7) || block_stride < (long long)block_size * rowb) return SPMLA_EALIGN;
  if (fmt != 0 && !(kv_scale > 0.f)) return SPMLA_EARG;
  rope::LatentParams p{(const uint16_t*)kv, kv_st, weight, weight_f32, eps, positions, pos32, freqs, factor, slots, n,
                       (uint8_t*)cache, R, block_size, log2_or(block_size), block_stride, fmt,
                       fmt != 0 ? 1.0f / kv_scale : 1.0f};
  static Launcher start[2];
  const void* kernel = interleaved ? (const void*)rope::latent_write_kernel<true> : (const void*)rope::latent_write_kernel<false>;
  return start[interleaved != 0](kernel, dim3((n - 1) / 4 + 1), 256, 0, (hipStream_t)stream, p);
}

}  // extern "C"
