// RMS norm with the residual's addition and an 8-bit output, and the 8-bit quantization alone: what feeds a projection
// on FP8 weights.
//   z = x + residual (rounded to the type and stored),  y[d] = z[d] / sqrt(mean(z^2) + eps) * w[d]
//   out = y rounded once to the type; codes = e4m3(y / s) with one scale s per 128 values (group_codes)
// Sums, root and y are held in 32 bits or more (a thread's squares in fp32, with ue8m0 in 64 bits; then 64); y is not
// rounded to the 16-bit type before it is quantized.
//
// One pass: a row's values stay in the registers of the threads that share it, 8 a thread in CH chunks, so x and the
// residual are read once; x, residual and weights are all on their way before the first is needed. A group of 128 values is
// 16 neighbouring lanes of a chunk. Rows of up to 512 values take one wave each (no LDS), longer ones several.
// Bound by HBM for long chunks of wide rows: 8192 x 4096 bf16 with residual and codes 43 us (236 MB, 5.5 TB/s with part of it
// in the last cache; a device copy moves 5.1), 8192 x 7168 83. Narrow rows by the chain of each (loads, sum, root, codes) and
// by lanes without a value: 8192 x 576 with residual and codes 14 us of 6.5 at the copy's rate (72 of a row's 128 threads have
// values), 8192 x 1536 20 of 17. The quantization alone: 4096 x 16384 52 us, its divisions, and 39.5 with scales of powers of
// two (5.1 TB/s). Few rows: one row's chain, 3.3 us (1 x 4096 and 64 x 1536) a launch in a graph; the quantization of 32 x
// 16384 2.8.
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
  int nt;                                                    // threads that share a row, where a workgroup has one
};

// Loads and stores are 16 bytes of a lane at any alignment of the type (gfx950 takes them; a misaligned row costs one more
// line a wave). ROW: how rows end (load_raw); ends that are no whole eights are stored element by element. In a graph 13 x
// 3268 fp32 3.8 us, 8192 x 3268 bf16 42; element by element the calls took two to three times as long. NORM false: y = x, a
// workgroup per NT * 8 values of a row.
template <int DT, bool NORM, int NT, int CH, int ROW>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT) norm_kernel(NormParams p) {
  constexpr int RPB = NT < 256 ? 256 / NT : 1;               // rows per workgroup
  __shared__ double part[RPB][NT / 64];
  const int tid = threadIdx.x % NT, lane = threadIdx.x & 63, nt = NORM && RPB == 1 ? p.nt : NT;   // threads of a row
  const long long row = (long long)blockIdx.x * RPB + threadIdx.x / NT;
  const bool on = row < p.T;
  const long long from = on ? row : p.T - 1;                 // (a row without a thread's own is read, not written)
  const int base = NORM ? 0 : (int)blockIdx.y * (NT * 8);
  constexpr bool AHEAD = CH <= 2;                            // all that is read on its way at once (128 registers a thread)
  float z[CH][8];
  auto at = [&](int c) { return base + (c * nt + tid) * 8; };
  auto left = [&](int c) { return p.D - at(c); };            // values of the row from there on
  auto mine = [&](int c) { return on ? left(c) : 0; };
  Raw8<DT> x[CH], a[AHEAD ? CH : 1];
  Raw8<DT_F32> wf[AHEAD ? CH : 1];
  Raw8<DT> wd[AHEAD ? CH : 1];
#pragma unroll
  for (int c = 0; c < CH; ++c) load_raw<DT, ROW>(p.x, from * p.x_st + at(c), left(c), x[c]);
  auto load_residual = [&](int c) { load_raw<DT, ROW>(p.res, from * p.res_st + at(c), left(c), a[AHEAD ? c : 0]); };
  auto load_weights = [&](int c) {
    if (DT == DT_F32 || p.w_f32) load_raw<DT_F32, ROW>(p.w, at(c), left(c), wf[AHEAD ? c : 0]);
    else load_raw<DT, ROW>(p.w, at(c), left(c), wd[AHEAD ? c : 0]);
  };
  if constexpr (NORM && AHEAD) {
    if (p.res) {
#pragma unroll
      for (int c = 0; c < CH; ++c) load_residual(c);
    }
    if (p.w) {
#pragma unroll
      for (int c = 0; c < CH; ++c) load_weights(c);
    }
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) values_of<DT, ROW>(x[c], left(c), z[c]);
  Factor r{1.0f, 0.0f};
  if constexpr (NORM) {
    if (p.res) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (!AHEAD) load_residual(c);
        float b[8];
        values_of<DT, ROW>(a[AHEAD ? c : 0], left(c), b);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[c][e] = round_to<DT>(z[c][e] + b[e]);
        store_upto8<DT, ROW == WHOLE>(p.res_out, row * p.ro_st + at(c), mine(c), z[c]);
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
      double* of = part[threadIdx.x / NT];
      if (lane == 0) of[tid >> 6] = ss;
      __syncthreads();
      const int i = lane & (NT / 64 - 1);                    // the waves' sums, one a lane, added in one order
      ss = i * 64 < nt ? of[i] : 0.0;
      ss += dpp<DPP_XOR1>(ss);
      if (NT > 128) ss += dpp<DPP_XOR2>(ss);
      if (NT > 256) ss += dpp<DPP_HALF_MIRROR>(ss);
      if (NT > 512) ss += dpp<DPP_MIRROR>(ss);
    }
    r = factor_of(inverse_root(ss * p.inv_d + (double)p.eps));
    if (p.w) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (!AHEAD) load_weights(c);
        float v[8];
        if (DT == DT_F32 || p.w_f32) values_of<DT_F32, ROW>(wf[AHEAD ? c : 0], left(c), v);
        else values_of<DT, ROW>(wd[AHEAD ? c : 0], left(c), v);
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
      store_upto8<DT, ROW == WHOLE>(p.out, row * p.o_st + at(c), mine(c), y);
    }
  }
  if (p.codes) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      uint32_t lo, hi;
      const float s = group_codes<!NORM>(z[c], r, p.ue8m0 != 0, DT != DT_F32 && (!NORM || !p.w), lo, hi);
      const int d = at(c), n = mine(c);
      if (n > 0) {
        uint8_t* q = p.codes + row * p.c_st + d;
        if (n >= 8) {
          *(codes8*)q = codes8{lo, hi};
        } else if constexpr (ROW != WHOLE) {
#pragma unroll
          for (int e = 0; e < 7; ++e)
            if (e < n) q[e] = (uint8_t)((e < 4 ? lo : hi) >> (8 * (e & 3)));
        }
        if ((lane & 15) == 0) p.scales[row * p.s_st + d / QGROUP] = s;
      }
    }
  }
}

template <int DT, bool NORM, int NT, int CH, int ROW>
static int launch(NormParams p, hipStream_t s) {
  constexpr int RPB = NT < 256 ? 256 / NT : 1;
  p.nt = NORM && RPB == 1 ? (p.D + 512 * CH - 1) / (512 * CH) * 64 : NT;   // no wave without a value
  const long long groups = ((long long)p.T + RPB - 1) / RPB;
  if (groups * (p.nt * RPB) >= 1ll << 32) return SPMLA_ELIMIT;             // wide rows take up to 1024 threads each
  const unsigned gy = NORM ? 1u : (unsigned)((p.D + NT * 8 - 1) / (NT * 8));
  static Launcher start;
  return start((const void*)norm_kernel<DT, NORM, NT, CH, ROW>, dim3((unsigned)groups, gy), p.nt * RPB, 0, s, p);
}

constexpr int MAX_D = 65536;

template <int DT, int ROW>
static int norm_go(const NormParams& p, hipStream_t s) {
  // as few threads and chunks as hold the row, idle ones cost too (8192 x 1024 with residual and codes: 128 x 1 15.7 us, 256 x
  // 1 16.6). Of equal ones many threads for few rows (4096 values, 1 row: 512 x 1 3.6, 256 x 2 4.6; 7168: 1024 x 1 4.6, 512 x
  // 2 5.1), fewer that each have more on their way for many (8192 rows: 45 / 42, 104 / 88).
  if constexpr (ROW == TINY) {
    return launch<DT, true, 64, 1, ROW>(p, s);
  } else {
    if (p.D <= 512) return launch<DT, true, 64, 1, ROW>(p, s);
    if (p.D <= 1024) return launch<DT, true, 128, 1, ROW>(p, s);
    if (p.D <= 2048) return launch<DT, true, 256, 1, ROW>(p, s);
    if (p.D <= 4096 && p.T <= 4096) return launch<DT, true, 512, 1, ROW>(p, s);
    if (p.D <= 4096) return launch<DT, true, 256, 2, ROW>(p, s);
    if (p.D <= 8192 && p.T <= 1024) return launch<DT, true, 1024, 1, ROW>(p, s);
    if (p.D <= 8192) return launch<DT, true, 512, 2, ROW>(p, s);
    if (p.D <= 16384) return launch<DT, true, 1024, 2, ROW>(p, s);
    return launch<DT, true, 1024, 8, ROW>(p, s);
  }
}

static int go(const NormParams& p, bool norm, int dtype, hipStream_t s) {
  auto by_type = [&](auto tag) {
    constexpr int R = decltype(tag)::value;
    if (norm) return dtype == DT_F32 ? norm_go<DT_F32, R>(p, s) : dtype == DT_F16 ? norm_go<DT_F16, R>(p, s)
                                                                                  : norm_go<DT_BF16, R>(p, s);
    return dtype == DT_F32 ? launch<DT_F32, false, 256, 1, R>(p, s) : dtype == DT_F16 ? launch<DT_F16, false, 256, 1, R>(p, s)
                                                                                       : launch<DT_BF16, false, 256, 1, R>(p, s);
  };
    if (p.D % 8 == 0) return by_type(std::integral_constant<int, WHOLE>{});
    if (p.D > 8) return by_type(std::integral_constant<int, ENDS>{});
    return by_type(std::integral_constant<int, TINY>{});
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
                    out, o_st, codes, c_st, scales, s_st, ue8m0, 0};
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
                    nullptr, 0, codes, c_st, scales, s_st, ue8m0, 0};
  return nrm::go(p, false, dtype, (hipStream_t)stream);
}

}  // extern "C"
