// RMS norm with the residual's addition and an 8-bit output, and the 8-bit quantization alone: what feeds a projection
// on FP8 weights.
//   z = x + residual (rounded to the type and stored),  y[d] = z[d] / sqrt(mean(z^2) + eps) * w[d]
//   out = y rounded once to the type; codes = e4m3(y / s) with one scale s per 128 values (group_codes)
// Sums, root and y are held in 32 bits or more (a thread's squares in fp32, with ue8m0 in 64 bits; then 64); y is not
// rounded to the 16-bit type before it is quantized.
//
// One pass: a row's values stay in the registers of the NT threads that share it, 8 a thread in CH chunks, so x and the
// residual are read once. A group of 128 values is 16 neighbouring lanes of a chunk. Rows of up to 512 values take one
// wave each (no LDS), longer ones a workgroup.
// Bound by HBM for long chunks: 8192 x 4096 bf16 with residual and codes 48 us (236 MB, 4.9 TB/s; a device copy moves 5.1).
// Few rows: the chain of a row's loads, sum, root and codes, 3.4 us (64 x 1536) to 4.1 us (1 x 4096) of GPU time; alone, the
// quantization of 32 x 16384 takes 2.4.
#include "spmla_quant.h"

namespace spmla {
namespace nrm {

struct NormParams {
  const void* x; long long x_st;
  const void* res; void* res_out; long long res_st, ro_st;   // null without a residual
  const void* w; int w_f32;                                  // null: ones
  float eps;
  double inv_d;                                              // 1 / D
  int T, D;
  void* out; long long o_st;                                 // null without it
  uint8_t* codes; long long c_st;                            // null without them
  float* scales; long long s_st;
  int ue8m0;
};

// Loads and stores are 16 bytes of a lane at any alignment of the type (gfx950 takes them; a misaligned row costs one more
// line a wave). WHOLE: D % 8 == 0; else the lane at a row's end goes element by element (13 x 3268 fp32 4.4 us a call, 221 x
// 6578 fp32 5.7, 753 x 1500 bf16 4.9; with whole rows element by element 9.9, 10.1, 7.8). NORM false: y = x, a workgroup
// per NT * 8 values of a row.
template <int DT, bool NORM, int NT, int CH, bool WHOLE>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT) norm_kernel(NormParams p) {
  constexpr int RPB = NT < 256 ? 256 / NT : 1;               // rows per workgroup
  __shared__ double part[NT / 64];
  const int tid = threadIdx.x % NT, lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * RPB + threadIdx.x / NT;
  const bool on = row < p.T;
  const int base = NORM ? 0 : (int)blockIdx.y * (NT * 8);
  constexpr bool EARLY = CH <= 2;                            // weights on their way before the sum (128 registers a thread)
  float z[CH][8], w[EARLY ? CH : 1][8];
  auto at = [&](int c) { return base + (c * NT + tid) * 8; };
  auto left = [&](int c) { return on ? p.D - at(c) : 0; };   // values of the row from there on
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    load_upto8<DT, WHOLE>(p.x, row * p.x_st + at(c), left(c), z[c]);
  }
  Factor r{1.0f, 0.0f};
  if constexpr (NORM) {
    auto weights = [&](int c, float (&v)[8]) {
      if (p.w_f32) load_upto8<DT_F32, WHOLE>(p.w, at(c), left(c), v);
      else load_upto8<DT, WHOLE>(p.w, at(c), left(c), v);
    };
    if (EARLY && p.w) {
#pragma unroll
      for (int c = 0; c < CH; ++c) weights(c, w[c]);
    }
    if (p.res) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float a[8];
        load_upto8<DT, WHOLE>(p.res, row * p.res_st + at(c), left(c), a);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[c][e] = round_to<DT>(z[c][e] + a[e]);
        store_upto8<DT, WHOLE>(p.res_out, row * p.ro_st + at(c), left(c), z[c]);
      }
    }
    double ss = 0.0;
    if (p.ue8m0) {                     // in 64 bits: here an error of r moves every code of the row the same way
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = __builtin_fma((double)z[c][e], (double)z[c][e], ss);
    } else {
      float q = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) q = __builtin_fmaf(z[c][e], z[c][e], q);
      ss = (double)q;
    }
    ss = wave_sum(ss);
    if constexpr (NT > 64) {
      if (lane == 0) part[tid >> 6] = ss;
      __syncthreads();
      ss = part[0];
#pragma unroll
      for (int i = 1; i < NT / 64; ++i) ss += part[i];
    }
    r = factor_of(inverse_root(ss * p.inv_d + (double)p.eps));
    if (p.w) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float (&v)[8] = w[EARLY ? c : 0];
        if (!EARLY) weights(c, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[c][e] *= v[e];
      }
    }
  }
  if (p.out) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = z[c][e] * r.hi;
      store_upto8<DT, WHOLE>(p.out, row * p.o_st + at(c), left(c), y);
    }
  }
  if (p.codes) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      uint32_t lo, hi;
      const float s = group_codes(z[c], r, p.ue8m0 != 0, lo, hi);
      const int d = at(c), n = left(c);
      if (n > 0) {
        uint8_t* q = p.codes + row * p.c_st + d;
        if (n >= 8) {
          *(codes8*)q = codes8{lo, hi};
        } else if constexpr (!WHOLE) {
#pragma unroll
          for (int e = 0; e < 7; ++e)
            if (e < n) q[e] = (uint8_t)((e < 4 ? lo : hi) >> (8 * (e & 3)));
        }
        if ((lane & 15) == 0) p.scales[row * p.s_st + d / QGROUP] = s;
      }
    }
  }
}

template <int DT, bool NORM, int NT, int CH, bool WHOLE>
static void launch(const NormParams& p, hipStream_t s) {
  constexpr int RPB = NT < 256 ? 256 / NT : 1;
  const unsigned gy = NORM ? 1u : (unsigned)((p.D + NT * 8 - 1) / (NT * 8));
  hipLaunchKernelGGL((norm_kernel<DT, NORM, NT, CH, WHOLE>), dim3((unsigned)(((long long)p.T + RPB - 1) / RPB), gy),
                     dim3(NT < 256 ? 256 : NT), 0, s, p);
}

constexpr int MAX_D = 65536;

template <int DT, bool WHOLE>
static void norm_go(const NormParams& p, hipStream_t s) {
  if (p.D <= 512) launch<DT, true, 64, 1, WHOLE>(p, s);
  else if (p.D <= 2048) launch<DT, true, 256, 1, WHOLE>(p, s);
  else if (p.D <= 4096) launch<DT, true, 256, 2, WHOLE>(p, s);
  else if (p.D <= 16384) launch<DT, true, 1024, 2, WHOLE>(p, s);
  else launch<DT, true, 1024, 8, WHOLE>(p, s);
}

static int go(const NormParams& p, bool norm, int dtype, hipStream_t s) {
  auto by_type = [&](auto tag) {
    constexpr bool V = decltype(tag)::value;
    if (norm) {
      if (dtype == DT_F32) norm_go<DT_F32, V>(p, s);
      else if (dtype == DT_F16) norm_go<DT_F16, V>(p, s);
      else norm_go<DT_BF16, V>(p, s);
    } else {
      if (dtype == DT_F32) launch<DT_F32, false, 256, 1, V>(p, s);
      else if (dtype == DT_F16) launch<DT_F16, false, 256, 1, V>(p, s);
      else launch<DT_BF16, false, 256, 1, V>(p, s);
    }
  };
  if (p.D % 8 == 0) by_type(std::true_type{});
  else by_type(std::false_type{});
  return (int)hipGetLastError();
}

}  // namespace nrm
}  // namespace spmla

using namespace spmla;

extern "C" {

int spmla_rms_norm(const void* x, long long x_st, const void* residual, long long r_st, void* residual_out,
                   long long ro_st, const void* weight, int weight_f32, float eps, int T, int D, int dtype, void* out,
                   long long o_st, unsigned char* codes, long long c_st, float* scales, long long s_st, int ue8m0,
                   void* stream) {
  if (T < 0 || D <= 0 || dtype < 0 || dtype > 2 || !(eps >= 0.f)) return SPMLA_EARG;
  if (D > nrm::MAX_D || T > MAX_TOKENS) return SPMLA_ELIMIT;
  if (T == 0) return SPMLA_OK;
  if (!x || (residual != nullptr) != (residual_out != nullptr) || (!out && !codes) ||
      (codes != nullptr) != (scales != nullptr))
    return SPMLA_EARG;
  const int eb = dtype == DT_F32 ? 4 : 2;
  if ((((uintptr_t)x | (uintptr_t)residual | (uintptr_t)residual_out | (uintptr_t)out) & (eb - 1)) ||
      ((uintptr_t)weight & (weight_f32 ? 3 : eb - 1)) || ((uintptr_t)scales & 3))
    return SPMLA_EALIGN;
  nrm::NormParams p{x, x_st, residual, residual_out, r_st, ro_st, weight, weight_f32, eps, 1.0 / D, T, D,
                    out, o_st, codes, c_st, scales, s_st, ue8m0};
  return nrm::go(p, true, dtype, (hipStream_t)stream);
}

int spmla_quant_fp8(const void* x, long long x_st, int T, int D, int dtype, unsigned char* codes, long long c_st,
                    float* scales, long long s_st, int ue8m0, void* stream) {
  if (T < 0 || D <= 0 || dtype < 0 || dtype > 2) return SPMLA_EARG;
  if (D > 65535 * 2048 || T > MAX_TOKENS) return SPMLA_ELIMIT;
  if (T == 0) return SPMLA_OK;
  if (!x || !codes || !scales) return SPMLA_EARG;
  if (((uintptr_t)x & (dtype == DT_F32 ? 3 : 1)) || ((uintptr_t)scales & 3)) return SPMLA_EALIGN;
  nrm::NormParams p{x, x_st, nullptr, nullptr, 0, 0, nullptr, 0, 0.f, 0.0, T, D,
                    nullptr, 0, codes, c_st, scales, s_st, ue8m0};
  return nrm::go(p, false, dtype, (hipStream_t)stream);
}

}  // extern "C"
