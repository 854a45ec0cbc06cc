// Matrix product of 8-bit activations with FP8 block-scaled weights: the projections around the attention.
//   out[t][n] = sum_b sa[t][b] sw[n / 128][b] sum_{k in b} a[t][k] w[n][k],  b = blocks of 128 values of k
// a, w e4m3; sa one fp32 scale per token and block, sw one per 128 x 128 block (the checkpoint's weight_scale_inv).
//
// v_mfma_f32_16x16x128_f8f6f4 takes a whole block of k, its sum starts from zero and goes into the fp32 accumulator with
// one FMA per value, by the product of the two scales. The weights are the row operand, so that a lane holds one token
// (column l % 16, outputs 4 (l / 16) .. + 3) and needs one scale product for all the outputs of a 128-block. The matrix
// core adds the 128 products with less than fp32's precision: 1.4e-5 of the sum's size on normally distributed codes
// (4.5e-5 with 1 of 64 values 50 times the others), a hundredth of the 16-bit output's rounding; fp32 outputs are not
// offered. Blocks are summed in fp32.
//
// Operands reach LDS by direct copies, 128-byte rows with their 16-byte chunks permuted by (row & 7), so that the
// fragment reads of 16 rows fall on distinct banks. In the last block of a k that is no multiple of 128 the chunks
// behind k are read from the row's last chunk and the weights' are overwritten with zeros in LDS.
#include "spmla_quant.h"

namespace spmla {
namespace lin {

struct LinearParams {
  const uint8_t* a; long long a_st;
  const float* sa; long long sa_st;
  const uint8_t* w; long long w_st;
  const float* sw; long long sw_st;
  void* out; long long o_st;
  int T, N, K;
  int o_vec;                     // 8-byte stores of four outputs
};

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // m0 is reserved; nothing else in these kernels uses it
// global -> LDS copies from a uniform base and a 32-bit offset of each lane (see dma16)
__device__ inline void dma16s(const void* base, uint32_t off, SPMLA_LDS void* l) {
  const uint32_t d = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)l);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(d) : "memory", "m0");
}
__device__ inline void dma4s(const void* base, uint32_t off, SPMLA_LDS void* l) {
  const uint32_t d = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)l);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(d) : "memory", "m0");
}
#pragma clang diagnostic pop

__device__ inline i32x8 frag(const uint8_t* rows, int r, int g) {   // row r's bytes 32 g .. + 31 of a staged block
  const i32x4 lo = *(const i32x4*)(rows + r * 128 + (((2 * g) ^ (r & 7)) << 4));
  const i32x4 hi = *(const i32x4*)(rows + r * 128 + (((2 * g + 1) ^ (r & 7)) << 4));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ inline f32x4 block_sum(i32x8 w, i32x8 a) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}
template <int DT>
__device__ inline void store4(const LinearParams& p, int t, int n, f32x4 v) {   // outputs n .. n + 3 of token t
  if (t >= p.T) return;
  uint16_t* o = (uint16_t*)p.out + (long long)t * p.o_st + n;
  if (p.o_vec && n + 4 <= p.N) {
    *(uint2*)o = make_uint2(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N) store1<DT>(o, i, v[i]);
  }
}

// ---- tiles of BM tokens x BN outputs, a wave WM x WN of them; two stages of one block in LDS -----------------------
template <int BM, int BN, int WM, int WN>
struct Tile {
  static constexpr int NWM = BM / WM, NW = NWM * (BN / WN);
  static constexpr int AS = 0, WS = BM * 128, SS = WS + BN * 128, STAGE = SS + BM * 4;
  static constexpr int LDS = 2 * STAGE;
  static_assert(BM % 64 == 0 && BN % 64 == 0 && 128 % WN == 0 && LDS <= 160 * 1024, "tile");
};

template <int DT, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * (BM / WM) * (BN / WN)) tile_kernel(LinearParams p, int TN) {
  using C = Tile<BM, BN, WM, WN>;
  extern __shared__ __attribute__((aligned(16))) uint8_t sm[];
  const int L = remap_xcd((int)blockIdx.x, TN * ((p.T + BM - 1) / BM));
  if (L < 0) return;
  const int t0 = (L / TN) * BM, n0 = (L % TN) * BN;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wm = (wv % C::NWM) * WM, wn = (wv / C::NWM) * WN;
  const int r = lane & 15, g = lane >> 4;
  const int kb = (p.K + 127) / 128, kt = p.K - (kb - 1) * 128;       // blocks, values of the last one
  // copies: rows of 128 bytes, 8 a copy, dealt over the waves; a lane's chunk is (lane % 8) ^ (row % 8)
  constexpr int PA = (BM / 8 + C::NW - 1) / C::NW, PW = (BN / 8 + C::NW - 1) / C::NW;
  const int ch = (lane & 7) ^ (lane >> 3);
  const uint32_t over = ch * 16 < kt ? 0u : (uint32_t)(ch * 16 - kt + 16);     // back to the last chunk below k
  const uint8_t* ab = p.a + (long long)t0 * p.a_st;
  const uint8_t* wb = p.w + (long long)n0 * p.w_st;
  const float* sb = p.sa + (long long)t0 * p.sa_st;
  uint32_t va[PA], vw[PW], vs;
#pragma unroll
  for (int j = 0; j < PA; ++j) {
    const int row = min((j * C::NW + wv) * 8 + (lane >> 3), p.T - 1 - t0);
    va[j] = (uint32_t)(row * p.a_st) + ch * 16;
  }
#pragma unroll
  for (int j = 0; j < PW; ++j) {
    const int row = min((j * C::NW + wv) * 8 + (lane >> 3), p.N - 1 - n0);
    vw[j] = (uint32_t)(row * p.w_st) + ch * 16;
  }
  vs = (uint32_t)(min(wv * 64 + lane, p.T - 1 - t0) * p.sa_st * 4);
  auto issue = [&](int b) {
    SPMLA_LDS uint8_t* st = (SPMLA_LDS uint8_t*)sm + (b & 1) * C::STAGE;
    const uint32_t back = b == kb - 1 ? over : 0u;
#pragma unroll
    for (int j = 0; j < PA; ++j)
      if ((j * C::NW + wv) * 8 < BM) dma16s(ab + b * 128, va[j] - back, st + C::AS + (j * C::NW + wv) * 1024);
#pragma unroll
    for (int j = 0; j < PW; ++j)
      if ((j * C::NW + wv) * 8 < BN) dma16s(wb + b * 128, vw[j] - back, st + C::WS + (j * C::NW + wv) * 1024);
    if (wv * 64 < BM) dma4s(sb + b, vs, st + C::SS + wv * 256);
  };
  const float* swr = p.sw + (long long)(min(n0 + wn, p.N - 1) / 128) * p.sw_st;
  float swv = swr[min(lane, kb - 1)];
  constexpr int MT = WM / 16, NT = WN / 16;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  issue(0);
  for (int b = 0; b < kb; ++b) {
    wait_vm<0>();
    lds_barrier();                       // block b has arrived; everyone is done with block b - 1
    uint8_t* st = sm + (b & 1) * C::STAGE;
    if (b == kb - 1 && kt < 128) {       // zeros behind k, one operand is enough
      for (int i = threadIdx.x; i < BN * 8; i += 64 * C::NW) {
        const int row = i >> 3, c = (i & 7) ^ (row & 7);
        if (c * 16 >= kt) *(u32x4*)(st + C::WS + i * 16) = u32x4{0, 0, 0, 0};
      }
      lds_barrier();
    }
    if (b + 1 < kb) issue(b + 1);
    if (b && (b & 63) == 0) swv = swr[min(b + lane, kb - 1)];
    const float sw = u2f(__builtin_amdgcn_readlane(f2u(swv), b & 63));
    i32x8 av[MT];
    float sc[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      av[j] = frag(st + C::AS, wm + j * 16 + r, g);
      sc[j] = *(const float*)(st + C::SS + (wm + j * 16 + r) * 4) * sw;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const i32x8 wf = frag(st + C::WS, wn + i * 16 + r, g);
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const f32x4 d = block_sum(wf, av[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(d[e], sc[j], acc[i][j][e]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j)
      if (n0 + wn + i * 16 + 4 * g < p.N) store4<DT>(p, t0 + wm + j * 16 + r, n0 + wn + i * 16 + 4 * g, acc[i][j]);
}

template <int DT, int BM, int BN, int WM, int WN>
static int tile_go(const LinearParams& p, hipStream_t s) {
  using C = Tile<BM, BN, WM, WN>;
  static DynLds lds;
  if (int rc = lds.ensure((const void*)tile_kernel<DT, BM, BN, WM, WN>, C::LDS)) return rc;
  const int TN = (p.N + BN - 1) / BN;
  const long long n = (long long)TN * ((p.T + BM - 1) / BM);
  if (n > 0x7ffffff0LL) return SPMLA_ELIMIT;
  hipLaunchKernelGGL((tile_kernel<DT, BM, BN, WM, WN>), dim3((unsigned)((n + 7) / 8 * 8)), dim3(64 * C::NW), C::LDS, s, p,
                     TN);
  return (int)hipGetLastError();
}

template <int DT>
static int linear_go(const LinearParams& p, hipStream_t s) {
  return tile_go<DT, 128, 128, 64, 64>(p, s);
}

}  // namespace lin
}  // namespace spmla

using namespace spmla;

extern "C" {

int spmla_linear_fp8(const void* a, long long a_st, const float* a_scales, long long as_st, const void* w,
                     long long w_st, const float* w_scales, long long ws_st, int T, int N, int K, int dtype, void* out,
                     long long o_st, void* stream) {
  if (T < 0 || N < 0 || K <= 0 || (K & 15) || (dtype != DT_F16 && dtype != DT_BF16)) return SPMLA_EARG;
  if (T == 0 || N == 0) return SPMLA_OK;
  if (!a || !a_scales || !w || !w_scales || !out) return SPMLA_EARG;
  const int kb = (K + 127) / 128;
  if ((T > 1 && (a_st < K || as_st < kb || o_st < N)) || (N > 1 && w_st < K) || (N > 128 && ws_st < kb)) return SPMLA_EARG;
  if (((uintptr_t)a & 15) || (a_st & 15) || ((uintptr_t)w & 15) || (w_st & 15) || ((uintptr_t)a_scales & 3) ||
      ((uintptr_t)w_scales & 3) || ((uintptr_t)out & 1))
    return SPMLA_EALIGN;
  if (a_st > (1 << 22) || w_st > (1 << 22) || as_st > (1 << 20)) return SPMLA_ELIMIT;   // 32-bit offsets inside a tile
  lin::LinearParams p{(const uint8_t*)a, a_st, a_scales, as_st, (const uint8_t*)w, w_st, w_scales, ws_st, out, o_st,
                      T, N, K, ((uintptr_t)out & 7) == 0 && (o_st & 3) == 0};
  if (dtype == DT_F16) return lin::linear_go<DT_F16>(p, (hipStream_t)stream);
  return lin::linear_go<DT_BF16>(p, (hipStream_t)stream);
}

}  // extern "C"
