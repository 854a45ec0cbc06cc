// Matrix product of 8-bit activations with FP8 block-scaled weights: the projections around the attention.
//   out[t][n] = sum_b sa[t][b] sw[n / 128][b] sum_{k in b} a[t][k] w[n][k],  b = blocks of 128 values of k
// a, w e4m3; sa one fp32 scale per token and block, sw one per 128 x 128 block (the checkpoint's weight_scale_inv).
//
// v_mfma_f32_16x16x128_f8f6f4 takes a whole block of k, its sum starts from zero and goes into the fp32 accumulator with
// one FMA per value, by the product of the two scales. The weights are the row operand, so that a lane holds one token
// (column l % 16, outputs 4 (l / 16) .. + 3) and needs one scale product for all the outputs of a 128-block. The matrix
// core adds the 128 products with less than fp32's precision. Against the sum of their magnitudes its error was at most 1.8e-5
// on normally distributed codes and 2.0e-4 with 1 of 64 values 50 times the others (1.4e-5 and 4.4e-5 of the sums' size, root
// mean square; other forms of the instruction reached 2.6e-4): half a step of a bf16 output is 3.9e-3 of the value, of fp16
// 4.9e-4, so that outliers, and sums that cancel, show in fp16. fp32 outputs are not offered. Blocks are summed in fp32.
//
// Operands reach LDS by direct copies, 128-byte rows with their 16-byte chunks permuted by (row / 2) % 8 (the outputs of the
// tile kernels, whose lanes take other rows, by what is the same number for the lane). A lane reads chunks g and g + 4 of its
// row (g = l / 16): the 16 lanes that LDS serves at once (0-3, 12-15, 20-23, 24-27 and so on) then fall on distinct banks, 256
// bytes a clock (with chunks 2 g and 2 g + 1 two of them meet in every bank: 128). Which 32 values of k a lane holds does not
// matter, since both operands hold the same ones. In the last block of a k that is no multiple of 128 the chunks behind k are
// read from the row's last chunk and the weights' are replaced by zeros.
#include "spmla_quant.h"
#include "spmla_rules.h"

namespace spmla {
namespace lin {

struct LinearParams {
  const uint8_t* a; long long a_st;
  const float* sa; long long sa_st;
  const uint8_t* w; long long w_st;
  const float* sw; long long sw_st;
  void* out; long long o_st;
  int T, N, K;
  int o_vec, o_seg;              // 8-byte stores of four outputs; rows of whole, aligned 64-byte segments
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
// 4 bytes from each address of a full wave's first LANES lanes
template <int LANES>
__device__ inline void dma4_first(const float* v, SPMLA_LDS void* l) {
  static_assert(LANES > 0 && LANES < 64, "lanes");
  constexpr uint64_t M = (1ull << LANES) - 1;
  const uint32_t d = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)l);
  asm volatile("s_mov_b32 m0, %1\n\ts_mov_b32 exec_lo, %2\n\ts_mov_b32 exec_hi, %3\n\tglobal_load_lds_dword %0, off\n\t"
               "s_mov_b64 exec, -1" ::"v"(v), "s"(d), "i"((uint32_t)M), "i"((uint32_t)(M >> 32)) : "memory", "m0");
}
#pragma clang diagnostic pop

__device__ inline i32x8 frag_at(const uint8_t* rows, int at) {      // the chunk at `at` and the one four chunks from it
  const i32x4 lo = *(const i32x4*)(rows + at), hi = *(const i32x4*)(rows + (at ^ 64));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ inline i32x8 frag(const uint8_t* rows, int r, int g) {   // row r's chunks g and g + 4 of a staged block
  return frag_at(rows, r * 128 + ((g ^ ((r >> 1) & 7)) << 4));
}
__device__ inline f32x4 block_sum(i32x8 w, i32x8 a) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}
typedef const __attribute__((address_space(4))) float* scalar_floats;   // read with scalar loads: uniform, not written here

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

// ---- tiles of BM tokens x BN outputs, 8 waves of WM x WN, a ring of ST blocks in LDS ----------------------------------
// While the sums of block b form from registers, block b + 1 is read from LDS and blocks b + 2 .. b + ST are on their way:
// one barrier a block, behind which block b's place is free and block b + 1 has arrived.
// Bound by the chain of a block: its eight waves go from barrier to barrier in step, 1290 clocks a block of 128 x 128 (41,300
// cycles over 32 blocks), in which the matrix cores are busy for 500 (39 %) and the LDS reads for 470 (36 %, no conflicts); no
// unit is at its limit. 1455 x 2112 x 4096 20 to 22 us (1.2 PFLOP/s, 204 workgroups), 6 of them before and behind the blocks; 64
// x 24576 x 1536 in tiles of 64 x 128 9.4 us (4.3 TB/s of weights and outputs). 16 waves, wave tiles of 64 x 64 and a ring of 4
// blocks were no faster, two workgroups a unit (128 registers) 10 % slower.
template <int BM, int BN, int WM, int WN, int ST>
struct Ring {
  static constexpr int NW = 8, NWM = BM / WM, PA = BM / 64, PW = BN / 64, NI = PA + PW + 1;   // copies of a wave and block
  static constexpr int AS = 0, WS = BM * 128, SS = WS + BN * 128, STAGE = SS + 1024;   // scales [wave][32]
  static constexpr int LDS = ST * STAGE;
  static_assert(BM % 64 == 0 && BN % 64 == 0 && NWM * (BN / WN) == NW && BN == 128 && WN == 32 && BM / NW < 32 && ST >= 3 &&
                ST * NI < 64 && LDS <= 160 * 1024, "ring");
};

template <int DT, int BM, int BN, int WM, int WN, int ST>
__global__ void __launch_bounds__(512, 2) ring_kernel(LinearParams p, int TN) {
  using C = Ring<BM, BN, WM, WN, ST>;
  constexpr int MT = WM / 16, NT = WN / 16;
  extern __shared__ __attribute__((aligned(16))) uint8_t sm[];
  const int TM = (p.T + BM - 1) / BM, L = remap_xcd((int)blockIdx.x, TN * TM);
  if (L < 0) return;
  // four rows of tiles at a time, column by column: the tiles that an XCD works on share rows and columns
  const int grp = L / (4 * TN), rem = L - grp * 4 * TN, gm = min(4, TM - grp * 4);
  const int t0 = (grp * 4 + rem % gm) * BM, n0 = rem / gm * BN;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wm = (wv % C::NWM) * WM, wn = (wv / C::NWM) * WN;
  const int r = lane & 15, g = lane >> 4;
  const int kb = (p.K + 127) / 128, kt = p.K - (kb - 1) * 128;       // blocks, values of the last one
  // copies: rows of 128 bytes, 8 a copy, dealt over the waves; a lane's chunk is (lane % 8) ^ (row / 2 % 8) of tokens,
  // (lane % 8) ^ (row / 2 % 2 + 2 (row / 8 % 4)) of outputs, the same in all of a wave's copies
  const int ch = (lane & 7) ^ ((lane >> 4) + (wv & 1) * 4), cw = (lane & 7) ^ ((lane >> 4) & 1) ^ (wv & 3) * 2;
  const uint32_t over = ch * 16 < kt ? 0u : (uint32_t)(ch * 16 - kt + 16);     // back to the last chunk below k
  const uint32_t overw = cw * 16 < kt ? 0u : (uint32_t)(cw * 16 - kt + 16);
  const uint8_t* ab = p.a + (long long)t0 * p.a_st;
  const uint8_t* wb = p.w + (long long)n0 * p.w_st;
  uint32_t va[C::PA], vw[C::PW];
#pragma unroll
  for (int j = 0; j < C::PA; ++j) {
    const int row = min((j * 8 + wv) * 8 + (lane >> 3), p.T - 1 - t0);
    va[j] = (uint32_t)(row * p.a_st) + ch * 16;
  }
#pragma unroll
  for (int j = 0; j < C::PW; ++j) {
    const int row = min((j * 8 + wv) * 8 + (lane >> 3), p.N - 1 - n0);
    vw[j] = (uint32_t)(row * p.w_st) + cw * 16;
  }
  // the scales of BM / 8 tokens and, in the lane behind them, of the tile's block of outputs
  const float* tokens = p.sa + (long long)min(t0 + wv * (BM / 8) + (lane & 31), p.T - 1) * p.sa_st;
  const float* outputs = p.sw + (long long)(n0 / 128) * p.sw_st;
  asm volatile("" : "+v"(tokens), "+v"(outputs));                    // two values, not one load of a selected argument
  const float* sp = lane < BM / 8 ? tokens : outputs;
  SPMLA_LDS uint8_t* lds = (SPMLA_LDS uint8_t*)sm;
  auto copy = [&](int b, int slot, int c) {                          // number c of a block's NI copies
    SPMLA_LDS uint8_t* st = lds + slot * C::STAGE;
    const uint32_t back = b != kb - 1 ? 0u : c < C::PA ? over : overw;
    if (c < C::PA) dma16s(ab + b * 128, va[c < C::PA ? c : 0] - back, st + C::AS + (c * 8 + wv) * 1024);
    else if (c < C::PA + C::PW)
      dma16s(wb + b * 128, vw[c >= C::PA && c < C::PA + C::PW ? c - C::PA : 0] - back, st + C::WS + ((c - C::PA) * 8 + wv) * 1024);
    else dma4_first<BM / 8 + 1>(sp + b, st + C::SS + wv * 128);
  };
  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Frags {
    i32x8 a[MT], w[NT];
    float s[MT], sw;
  };
  const bool z0 = g * 16 >= kt, z1 = (g + 4) * 16 >= kt;             // chunks behind k in the last block
  constexpr int NR = NT + MT + 1;
  // row 8 (r / 4) + 4 i + r % 4 of a wave's 32 outputs: the sums of i = 0 and 1 are eight outputs in turn, from 8 g on
  const int fw = C::WS + (wn + 8 * (r >> 2) + (r & 3)) * 128 + ((g ^ (r >> 1)) << 4);
  auto read = [&](int slot, Frags& f, int c) {                        // part c of NR: a fragment, last the scales
    const uint8_t* st = sm + slot * C::STAGE;
    if (c < NT) f.w[c < NT ? c : 0] = frag_at(st + c * 512, fw);
    else if (c < NT + MT) f.a[c >= NT && c < NT + MT ? c - NT : 0] = frag(st + C::AS, wm + (c - NT) * 16 + r, g);
    else {
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const int t = wm + j * 16 + r;
        f.s[j] = *(const float*)(st + C::SS + t / (BM / 8) * 128 + t % (BM / 8) * 4);
      }
      f.sw = *(const float*)(st + C::SS + wv * 128 + BM / 8 * 4);
    }
  };
  auto clip = [&](int b, Frags& f) {                                  // zeros behind k, one operand is enough
    const bool y0 = z0 && b == kb - 1, y1 = z1 && b == kb - 1;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f.w[i][e] = y0 ? 0 : f.w[i][e];
        f.w[i][4 + e] = y1 ? 0 : f.w[i][4 + e];
      }
  };
  // the sums of row tile i run while those of i - 1 are added; between(m) behind matrix instruction m
  auto sums = [&](const Frags& f, auto between) {
    f32x4 d[2][MT];
    float sc[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) sc[j] = f.s[j] * f.sw;
#pragma unroll
    for (int i = 0; i <= NT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        if (i < NT) {
          d[i & 1][j] = block_sum(f.w[i], f.a[j]);
          between(i * MT + j);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (i > 0) {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i - 1][j][e] = __builtin_fmaf(d[(i - 1) & 1][j][e], sc[j], acc[i - 1][j][e]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
  };
  int in = 0, out = 0;                                                // slots of the next block to copy and to read
  auto next = [](int& s) { s = s + 1 == ST ? 0 : s + 1; };
  // (behind the last block it is copied again, so that the waits count the same copies everywhere)
  for (int b = 0; b < ST; ++b) {
#pragma unroll
    for (int c = 0; c < C::NI; ++c) copy(min(b, kb - 1), b, c);
  }
  wait_vm<(ST - 1) * C::NI>();
  lds_barrier();
  Frags f[2];
#pragma unroll
  for (int c = 0; c < NR; ++c) read(0, f[0], c);
  next(out);
  // one block: f its fragments, n the next one's
  auto block = [&](int b, auto tail, const Frags& f, Frags& n) {
    wait_vm<(ST - 2) * C::NI>();
    lds_barrier();
    // the reads and copies lie between the matrix instructions: issued together they hold up the wave behind them, since
    // all waves would issue theirs at once
    sums(f, [&](int m) {
#pragma unroll
      for (int c = 0; c < NR; ++c)
        if (c * NT * MT / NR == m) read(out, n, c);
#pragma unroll
      for (int c = 0; c < C::NI; ++c)
        if (c * NT * MT / C::NI == m) copy(min(b + ST, kb - 1), in, c);
    });
    next(out);
    next(in);
    if constexpr (decltype(tail)::value) clip(b + 1, n);
  };
  auto blocks = [&](auto tail) {                                      // tail: the last block is a part of one
    if constexpr (decltype(tail)::value) clip(0, f[0]);
    int b = 0;
    for (; b + 1 < kb; b += 2) {
      block(b, tail, f[0], f[1]);
      block(b + 1, tail, f[1], f[0]);
    }
    if (b < kb) block(b, tail, f[0], f[1]);
  };
  if (kt == 128) blocks(std::false_type{});
  else blocks(std::true_type{});
  wait_vm<0>();                                                       // no copy outlives the workgroup
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const f32x4 &x = acc[0][j], &y = acc[1][j];
    const float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    const int t = t0 + wm + j * 16 + r, n = n0 + wn + 8 * g;
    if (t < p.T) store_upto8<DT, false>(p.out, t * p.o_st + n, p.N - n, v);
  }
}

template <int DT, int BM, int BN, int WM, int WN, int ST>
static int ring_go(const LinearParams& p, hipStream_t s) {
  using C = Ring<BM, BN, WM, WN, ST>;
  static DynLds lds;
  if (int rc = lds.ensure((const void*)ring_kernel<DT, BM, BN, WM, WN, ST>, C::LDS)) return rc;
  const int TN = (p.N + BN - 1) / BN;
  const long long n = (long long)TN * ((p.T + BM - 1) / BM);
  static Launcher start;
  return start((const void*)ring_kernel<DT, BM, BN, WM, WN, ST>, dim3((unsigned)((n + 7) / 8 * 8)), 512, C::LDS, s, p, TN);
}

// ---- few tokens: the weights stream past 16 MT tokens --------------------------------------------------------------
// A workgroup takes 16 NT outputs and 16 MT tokens; its NW waves take the blocks of k in turn, each with a ring of ST
// stages of its own in LDS, so that no wave waits for another until their sums meet in LDS at the end, in wave order.
// Bound by HBM once the weights are many: 1 x 4096 x 16384 12.1 us (5.5 TB/s), 32 x 4096 x 16384 14.0 (4.8), 16 x 24576 x
// 1536 8.8 (4.4); before that by the launch and the first loads' way: 1 x 2112 x 4096 3.8 us in a graph, of 1.7 at the copy's
// rate. Tiles of 16 x 16 with 8 waves give the most workgroups and the shortest part of k a wave; 4 waves of two output tiles
// read the tokens half as often.
template <int NT, int MT, int NW, int ST>
struct Stream {
  static constexpr int WS = 0, AS = NT * 2048, SS = AS + MT * 2048, STAGE = SS + 256;
  static constexpr int NI = 2 * NT + 2 * MT + 1;                     // copies of a stage
  static constexpr int RING = NW * ST * STAGE, RED = NW * NT * MT * 1024;
  static constexpr int LDS = RING > RED ? RING : RED;
  static_assert(MT <= 4 && (ST - 1) * NI < 64 && LDS <= 160 * 1024, "stream");
};

template <int DT, int NT, int MT, int NW, int ST>
__global__ void __launch_bounds__(64 * NW, 2) stream_kernel(LinearParams p, int TM) {
  using C = Stream<NT, MT, NW, ST>;
  extern __shared__ __attribute__((aligned(16))) uint8_t sm[];
  const int L = remap_xcd((int)blockIdx.x, TM * ((p.N + 16 * NT - 1) / (16 * NT)));
  if (L < 0) return;
  const int t0 = (L % TM) * 16 * MT, n0 = (L / TM) * 16 * NT;        // the token tiles of a row of weights: one XCD
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int r = lane & 15, g = lane >> 4;
  const int kb = (p.K + 127) / 128, kt = p.K - (kb - 1) * 128;
  const int cnt = wv < kb ? (kb - wv + NW - 1) / NW : 0;             // blocks wv, wv + NW, ..
  const int ce = (lane & 7) ^ (lane >> 4), co = ce ^ 4;              // a lane's chunk in even and odd copies of 8 rows
  auto over = [&](int j) { const int c = j & 1 ? co : ce; return c * 16 < kt ? 0u : (uint32_t)(c * 16 - kt + 16); };
  const uint8_t* ab = p.a + (long long)t0 * p.a_st;
  const uint8_t* wb = p.w + (long long)n0 * p.w_st;
  const float* sb = p.sa + (long long)t0 * p.sa_st;
  uint32_t va[2 * MT], vw[2 * NT];
#pragma unroll
  for (int j = 0; j < 2 * MT; ++j) va[j] = (uint32_t)(min(j * 8 + (lane >> 3), p.T - 1 - t0) * p.a_st) + (j & 1 ? co : ce) * 16;
#pragma unroll
  for (int j = 0; j < 2 * NT; ++j) vw[j] = (uint32_t)(min(j * 8 + (lane >> 3), p.N - 1 - n0) * p.w_st) + (j & 1 ? co : ce) * 16;
  const uint32_t vs = (uint32_t)(min(lane, p.T - 1 - t0) * p.sa_st * 4);
  uint8_t* ring = sm + wv * ST * C::STAGE;
  const scalar_floats swr = (scalar_floats)(p.sw + (long long)(n0 / 128) * p.sw_st);   // 16 NT outputs: one block of 128
  auto issue = [&](int i) {
    SPMLA_LDS uint8_t* st = (SPMLA_LDS uint8_t*)ring + (i % ST) * C::STAGE;
    const int b = wv + NW * i;
    const bool last = b == kb - 1;
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) dma16s(wb + b * 128, vw[j] - (last ? over(j) : 0u), st + C::WS + j * 1024);
#pragma unroll
    for (int j = 0; j < 2 * MT; ++j) dma16s(ab + b * 128, va[j] - (last ? over(j) : 0u), st + C::AS + j * 1024);
    dma4s(sb + b, vs, st + C::SS);
  };
  f32x4 acc[NT][MT];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < ST; ++i)
    if (i < cnt) issue(i);
  float sw = swr[min(wv, kb - 1)];
  for (int i = 0; i < cnt; ++i) {
    if (i + ST <= cnt) wait_vm<(ST - 1) * C::NI>();
    else wait_vm<0>();
    uint8_t* st = ring + (i % ST) * C::STAGE;
    const int b = wv + NW * i;
    if (b == kb - 1 && kt < 128) {       // zeros behind k, one operand is enough
#pragma unroll
      for (int j = 0; j < 2 * NT; ++j)
        if ((j & 1 ? co : ce) * 16 >= kt) *(u32x4*)(st + C::WS + j * 1024 + lane * 16) = u32x4{0, 0, 0, 0};
    }
    i32x8 av[MT], wf[NT];
    float sc[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) wf[j] = frag(st + C::WS, j * 16 + r, g);
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      av[j] = frag(st + C::AS, j * 16 + r, g);
      sc[j] = *(const float*)(st + C::SS + (j * 16 + r) * 4) * sw;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");               // the stage has been read: its ring place is free
    if (i + ST < cnt) issue(i + ST);
    __builtin_amdgcn_sched_barrier(0);
    sw = swr[min(b + NW, kb - 1)];                                    // on its way while this block's sums form
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const f32x4 d = block_sum(wf[n], av[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[n][j][e] = __builtin_fmaf(d[e], sc[j], acc[n][j][e]);
      }
  }
  lds_barrier();                         // every ring is done with
  f32x4* red = (f32x4*)sm;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < MT; ++j) red[(wv * NT * MT + n * MT + j) * 64 + lane] = acc[n][j];
  lds_barrier();
#pragma unroll
  for (int k = 0; k < (NT * MT + NW - 1) / NW; ++k) {
    const int e = wv + k * NW;
    if (e < NT * MT) {
      f32x4 v = red[e * 64 + lane];
#pragma unroll
      for (int u = 1; u < NW; ++u) v += red[(u * NT * MT + e) * 64 + lane];
      const int n = n0 + (e / MT) * 16 + 4 * g;
      if (n < p.N) store4<DT>(p, t0 + (e % MT) * 16 + r, n, v);
    }
  }
}

template <int DT, int NT, int MT, int NW, int ST>
static int stream_go(const LinearParams& p, hipStream_t s) {
  using C = Stream<NT, MT, NW, ST>;
  static DynLds lds;
  if (int rc = lds.ensure((const void*)stream_kernel<DT, NT, MT, NW, ST>, C::LDS)) return rc;
  const int TM = (p.T + 16 * MT - 1) / (16 * MT);
  const long long n = (long long)TM * ((p.N + 16 * NT - 1) / (16 * NT));
  static Launcher start;
  return start((const void*)stream_kernel<DT, NT, MT, NW, ST>, dim3((unsigned)((n + 7) / 8 * 8)), 64 * NW, C::LDS, s, p, TM);
}


// ---- long chunks: tiles of 256 tokens x 256 outputs, 8 waves, the operands' halves in rings of their own --------------
// The tile's tokens and outputs are two halves of 128 each (A0, A1, W0, W1); wave (wm, wn) takes tokens 64 wm .. + 63 of
// both token halves and 64 outputs from 64 wn on, 32 in each output half: four quadrants of 8 matrix instructions each,
//   phase 0: A0 W0   1: A0 W1   2: A1 W0   3: A1 W1.
// Registers are filled one phase before they are used (W1 in phase 0, A1 in 1, W0 and A0 of the next block in 3, each token
// fragment over the one that had its last use). A half's place in LDS is filled again as soon as a barrier stands between:
// A0, W0 and the scales of block b + 2 in phases 1 and 2 of block b, W1 and A1 in 3, so that every copy has 1 to 1 1/2
// blocks to arrive. The two barriers of a block stand where no read is on its way, behind a wait for the wave's
// own copies of what is read after them. A sum is scaled and added three matrix instructions after its own.
// A wave copies the scales of 32 tokens and, in lane 32, of its own 64 outputs in one instruction.
//
// Several tiles a workgroup (k a multiple of 128, more tiles than compute units): the copies run on into the next tile, so
// that it begins at once and while the finished one's stores are under way.
//
// Bound by the matrix cores at the clock that the power limit leaves them: 4096 x 4096 x 16384 224 us (2.45 PFLOP/s, a
// product with one scale a tensor at full rate 183), 188 with operands of zeros. What the steps to here gave, at that size
// and at 4096 x 24576 x 1536 (us): one barrier a phase, scalar loads of the outputs' scales 252, 200; two barriers a block,
// all scales by the copies 238, 195; several tiles a workgroup 236, 184; stores of 16 bytes a lane in 64-byte segments in
// place of 8 and 32 236, 173; past the caches where the rows are whole segments 236, 161 (1.9 PFLOP/s; without stores 130).
// 32 x 32 matrix instructions took 265, since their sums left no registers free.
struct Big {
  static constexpr int HALF = 128 * 128, A = 0, W = 4 * HALF, S = 8 * HALF;   // A [block % 2][half], W the same, then the
  static constexpr int LDS = S + 4 * 2048;                                     // scales [block % 4][wave][64]
};

// waits until at most N of the wave's memory operations are on their way, or MORE more of them where more != 0
template <int N, int MORE>
__device__ inline void wait_vm_or(int more) {
  static_assert(N + MORE < 64, "vmcnt range");
  asm volatile("s_cmp_lg_u32 %0, 0\n\ts_cbranch_scc1 .Lmore%=\n\ts_waitcnt vmcnt(%1)\n\ts_branch .Ldone%=\n.Lmore%=:\n\t"
               "s_waitcnt vmcnt(%2)\n.Ldone%=:"
               ::"s"(__builtin_amdgcn_readfirstlane(more)), "i"(N), "i"(N + MORE) : "memory", "scc");
}

template <int DT>
__global__ void __launch_bounds__(512, 2) big_kernel(LinearParams p, int TN) {
  extern __shared__ __attribute__((aligned(16))) uint8_t sm[];
  constexpr int STORES = 16;             // of a wave and a tile that has all its tokens and outputs, 16 bytes a lane
  const int TM = (p.T + 255) / 256, tiles = TN * TM, per = (tiles + 7) >> 3;
  int at = (int)blockIdx.x, t0, n0;
  // tile number at, XCD by XCD: four rows of tiles at a time, column by column, so that the 32 tiles that an XCD works on
  // share 4 rows and 8 columns
  auto tile = [&](int i, int& t, int& n) {
    const int L = (i >> 3) < per ? remap_xcd(i, tiles) : -1;
    if (L < 0) return false;
    const int grp = L / (4 * TN), rem = L - grp * 4 * TN, gm = min(4, TM - grp * 4);
    t = (grp * 4 + rem % gm) * 256;
    n = rem / gm * 256;
    return true;
  };
  if (!tile(at, t0, n0)) return;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int wm = wv & 1, wn = wv >> 1, r = lane & 15, g = lane >> 4;
  const int kb = (p.K + 127) / 128, kt = p.K - (kb - 1) * 128;
  // copies: wave wv takes rows 16 wv .. + 15 of a half, 8 a copy
  const uint8_t *ap, *wp;                // the next block to copy
  const float* sp;                       // of this lane's scale
  uint32_t va[2][2], vw[2][2];
  auto here = [&] {                      // the lane, for what is formed once a tile and not kept in registers between
    int l;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
    return l;
  };
  // a lane's chunk: (lane % 8) ^ (row / 2 % 8) of tokens, (lane % 8) ^ (row / 2 % 2 + 2 (row / 8 % 4)) of outputs
  auto chunk = [](int l, int j) { return (l & 7) ^ (l >> 4) ^ (j * 4); };
  auto chunk_w = [&](int l, int j) { return (l & 7) ^ ((l >> 4) & 1) ^ (((wv & 1) * 2 + j) * 2); };
  auto row_of = [&](int l, int h, int j) { return h * 128 + wv * 16 + j * 8 + (l >> 3); };
  auto out_of = [&](int l, int h, int j) { return (wv >> 1) * 64 + h * 32 + (wv & 1) * 16 + j * 8 + (l >> 3); };
  auto begin = [&](int t, int n) {
    const int l = here();
    ap = p.a + (long long)t * p.a_st;
    wp = p.w + (long long)n * p.w_st;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        va[h][j] = (uint32_t)(min(row_of(l, h, j), p.T - 1 - t) * p.a_st) + chunk(l, j) * 16;
        vw[h][j] = (uint32_t)(min(out_of(l, h, j), p.N - 1 - n) * p.w_st) + chunk_w(l, j) * 16;
      }
    const float* tokens = p.sa + (long long)min(t + wv * 32 + (l & 31), p.T - 1) * p.sa_st;
    const float* outputs = p.sw + (long long)min(n / 128 + (wn >> 1), (p.N - 1) / 128) * p.sw_st;
    asm volatile("" : "+v"(tokens), "+v"(outputs));        // two values, not one load of a selected argument
    sp = l < 32 ? tokens : outputs;
  };
  // the chunks behind k in the last block are read from the row's last one: before its copies
  auto over = [&](int chunk) { const int e = chunk * 16 + 16 - kt; return (uint32_t)(e > 0 ? e : 0); };
  auto end = [&] {
    const int l = here();
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        va[h][j] -= over(chunk(l, j));
        vw[h][j] -= over(chunk_w(l, j));
      }
  };
  SPMLA_LDS uint8_t* lds = (SPMLA_LDS uint8_t*)sm;
  auto place = [&](int base, int c, int h, int j) {                    // of block number c of the workgroup
    return lds + base + ((c & 1) * 2 + h) * Big::HALF + wv * 2048 + j * 1024;
  };
  auto copy_a = [&](int c, int h, int j) { dma16s(ap, va[h][j], place(Big::A, c, h, j)); };
  auto copy_w = [&](int c, int h, int j) { dma16s(wp, vw[h][j], place(Big::W, c, h, j)); };
  auto copy_s = [&](int c) { dma4_first<33>(sp, lds + Big::S + (c & 3) * 2048 + wv * 256); };
  // fragment places of this lane, chunks g and g + 4 of a row: row r of 16 tokens; row 8 (r / 4) + 4 i + r % 4 of 32 outputs,
  // so that the sums of i = 0 and 1 are eight outputs in turn, from 8 g on: 16-byte stores, 64 bytes of a token a wave
  const int fa = r * 128 + ((g ^ (r >> 1)) << 4), fw = (8 * (r >> 2) + (r & 3)) * 128 + ((g ^ (r >> 1)) << 4);
  auto a_of = [&](int c, int h, int j) {
    return frag_at(sm + Big::A + ((c & 1) * 2 + h) * Big::HALF + (wm * 64 + j * 16) * 128, fa);
  };
  auto w_of = [&](int c, int h, int i) {
    return frag_at(sm + Big::W + ((c & 1) * 2 + h) * Big::HALF + wn * 32 * 128 + i * 512, fw);
  };
  auto scale_at = [&](int c, int h, int j) {                           // token h 128 + wm 64 + j 16 + r
    return *(const float*)(sm + Big::S + (c & 3) * 2048 + (h * 4 + wm * 2 + (j >> 1)) * 256 + ((j & 1) * 16 + r) * 4);
  };
  auto w_scale_at = [&](int c) { return *(const float*)(sm + Big::S + (c & 3) * 2048 + wv * 256 + 128); };
  const bool z0 = g * 16 >= kt, z1 = (g + 4) * 16 >= kt;               // chunks behind k in the last block
  auto clip = [&](i32x8& w) {                                          // zeros there, one operand is enough
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = z0 ? 0 : w[e];
      w[4 + e] = z1 ? 0 : w[4 + e];
    }
  };
  f32x4 acc[4][2][4];                                                  // quadrant, output tile, token tile
  f32x4 d[4];                                                          // sums not added yet
  float s[2][4], sr[4], sc;       // scale products of this block's token halves; the tokens' and the outputs' scales
  i32x8 a[4], w0[2], w1[2];
  auto clear = [&] {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      d[q] = f32x4{0.f, 0.f, 0.f, 0.f};
      s[1][q] = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[q][i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  };
  clear();
  auto early = [&](int c) {              // the copies of a block, in the order of the loop's
    copy_a(c, 0, 0);
    copy_a(c, 0, 1);
    copy_s(c);
    copy_w(c, 0, 0);
    copy_w(c, 0, 1);
  };
  auto late = [&](int c) {
    copy_w(c, 1, 0);
    copy_w(c, 1, 1);
    copy_a(c, 1, 0);
    copy_a(c, 1, 1);
    ap += 128;
    wp += 128;
    sp += 1;
  };
  begin(t0, n0);
  if (kb == 1) end();
  early(0);
  late(0);
  if (kb > 1) {
    if (kb == 2) end();
    early(1);
    wait_vm<7>();
  } else {
    wait_vm<2>();
  }
  lds_barrier();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    w0[i] = w_of(0, 0, i);
    if (kb == 1) clip(w0[i]);
  }
  sc = w_scale_at(0);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    a[j] = a_of(0, 0, j);
    sr[j] = scale_at(0, 0, j);
  }
  if (kb > 1) late(1);
  // matrix instruction 8 q + 2 j + i of a block; the sum three before it is added
  auto step = [&](int m, const i32x8& wf, const i32x8& af) {
    if (m < 32) d[m & 3] = block_sum(wf, af);
    __builtin_amdgcn_sched_barrier(0);
    const int o = m < 32 ? (m + 29) & 31 : m - 3;
    f32x4& x = acc[o >> 3][o & 1][(o >> 1) & 3];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(d[o & 3][e], s[o >> 4][(o >> 1) & 3], x[e]);
    __builtin_amdgcn_sched_barrier(0);
  };
  // block number c of the workgroup; more_: the tiles' blocks behind it that are copied, up to 2; near, far: STORES stores
  // were issued between what the first, the second wait is for and its wait
  auto block = [&](int c, int near, int far, auto more_) {
    constexpr int more = decltype(more_)::value;
    // phase 0: A0 W0; W1 is read
#pragma unroll
    for (int i = 0; i < 2; ++i) w1[i] = w_of(c, 1, i);
#pragma unroll
    for (int j = 0; j < 4; ++j) s[0][j] = sr[j] * sc;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      step(m, w0[m & 1], a[m >> 1]);
    }
    if (more == 0) {
      clip(w1[0]);
      clip(w1[1]);
    }
    // phase 1: A0 W1; A1 is read over A0
    if (more) wait_vm_or<9, STORES>(near);
    else wait_vm<0>();
    lds_barrier();
#pragma unroll
    for (int j = 0; j < 4; ++j) sr[j] = scale_at(c, 1, j);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int m = 8; m < 16; ++m) {
      step(m, w1[m & 1], a[(m >> 1) & 3]);
      if (m & 1) a[(m >> 1) & 3] = a_of(c, 1, (m >> 1) & 3);
      else if (more > 1 && m < 12) copy_a(c + 2, 0, (m - 8) >> 1);
    }
    // phase 2: A1 W0
#pragma unroll
    for (int j = 0; j < 4; ++j) s[1][j] = sr[j] * sc;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int m = 16; m < 24; ++m) {
      step(m, w0[m & 1], a[(m >> 1) & 3]);
      if (more > 1 && m == 16) copy_s(c + 2);
      if (more > 1 && m >= 17 && m < 19) copy_w(c + 2, 0, m - 17);
    }
    // phase 3: A1 W1; A0 (over A1) and W0 of the next block are read
    if (more > 0) {
      if (more == 2) wait_vm_or<7, STORES>(far);
      else wait_vm<2>();
      lds_barrier();
#pragma unroll
      for (int i = 0; i < 2; ++i) w0[i] = w_of(c + 1, 0, i);
    }
    if (more > 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sr[j] = scale_at(c + 1, 0, j);
      sc = w_scale_at(c + 1);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int m = 24; m < 32; ++m) {
      step(m, w1[m & 1], a[(m >> 1) & 3]);
      if (more > 0 && (m & 1)) a[(m >> 1) & 3] = a_of(c + 1, 0, (m >> 1) & 3);
      else if (more > 1 && !(m & 1) && m < 28) copy_w(c + 2, 1, (m - 24) >> 1);
      else if (more > 1 && !(m & 1)) copy_a(c + 2, 1, (m - 28) >> 1);
    }
    if (more == 1) {
      clip(w0[0]);
      clip(w0[1]);
    }
    ap += 128;
    wp += 128;
    sp += 1;
  };
  int c = 0, stores = 0;                 // c: the workgroup's blocks before this tile
  for (;;) {
    int t1 = 0, n1 = 0;
    at += (int)gridDim.x;
    const bool go_on = tile(at, t1, n1);
    const int most = go_on ? kb : kb - 2;
    int b = 0;
    for (; b < most; ++b) {
      if (b == kb - 3) end();            // the copies are two blocks ahead
      if (b == kb - 2) begin(t1, n1);
      block(c + b, b < 2 ? stores : 0, b ? 0 : stores, std::integral_constant<int, 2>{});
    }
    if (!go_on) {
      if (kb > 1) block(c + b, b < 2 ? stores : 0, 0, std::integral_constant<int, 1>{});
      block(c + kb - 1, 0, 0, std::integral_constant<int, 0>{});
    }
#pragma unroll
    for (int m = 32; m < 35; ++m) step(m, w1[0], a[0]);
#pragma unroll
    for (int q = 0; q < 4; ++q)          // the sums are formed here, not each in the branch that stores it
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(acc[q][i][j]));
    const int l = here(), lr = l & 15, lg = l >> 4;
    const bool whole = t0 + 256 <= p.T && n0 + 256 <= p.N;
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 &x = acc[q][0][j], &y = acc[q][1][j];
        const float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        const int t = t0 + (q >> 1) * 128 + wm * 64 + j * 16 + lr, n = n0 + wn * 64 + (q & 1) * 32 + 8 * lg;
        const u32x4_any w = {pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7])};
        u32x4_any* o = (u32x4_any*)((uint16_t*)p.out + t * p.o_st + n);
        if (whole && p.o_seg) __builtin_nontemporal_store(w, o);
        else if (whole) *o = w;
        else if (t < p.T) store_upto8<DT, false>(p.out, t * p.o_st + n, p.N - n, v);
      }
    if (!go_on) return;
    stores = __builtin_amdgcn_readfirstlane((int)whole);
    t0 = t1;
    n0 = n1;
    c += kb;
    clear();
  }
}

template <int DT>
static int big_go(const LinearParams& p, hipStream_t s) {
  static DynLds lds;
  if (int rc = lds.ensure((const void*)big_kernel<DT>, Big::LDS)) return rc;
  const int TN = (p.N + 255) / 256;
  long long n = ((long long)TN * ((p.T + 255) / 256) + 7) / 8 * 8;
  if (p.K % 128 == 0 && p.K > 128 && n > 256) n = 256;                 // several tiles a workgroup, one workgroup a unit
  static Launcher start;
  return start((const void*)big_kernel<DT>, dim3((unsigned)n), 512, Big::LDS, s, p, TN);
}

// the rule's kernels in its order (rules::LINEAR)
template <int DT>
static int linear_go(const LinearParams& p, hipStream_t s) {
  switch (rules::linear_kernel(p.T, p.N, p.K)) {
    case 0: return stream_go<DT, 1, 1, 8, 4>(p, s);
    case 1: return stream_go<DT, 2, 1, 4, 3>(p, s);
    case 2: return stream_go<DT, 2, 2, 4, 2>(p, s);
    case 3: return stream_go<DT, 2, 4, 4, 2>(p, s);
    case 4: return stream_go<DT, 4, 4, 4, 2>(p, s);
    case 5: return ring_go<DT, 64, 128, 32, 32, 3>(p, s);
    case 6: return ring_go<DT, 128, 128, 64, 32, 3>(p, s);
    case 7: return big_go<DT>(p, s);
    default: return SPMLA_ELIMIT;
  }
}

}  // namespace lin
}  // namespace spmla

using namespace spmla;

constexpr int MAX_K = 1 << 22;         // and rows' strides in bytes: blocks are counted and places inside a tile formed in 32 bits

extern "C" {

int spmla_linear_fp8(const void* a, long long a_st, const float* a_scales, long long as_st, const void* w,
                     long long w_st, const float* w_scales, long long ws_st, int T, int N, int K, int dtype, void* out,
                     long long o_st, void* stream) {
  if (T < 0 || N < 0 || K <= 0 || (K & 15) || (dtype != DT_F16 && dtype != DT_BF16)) return SPMLA_EARG;
  if (T == 0 || N == 0) return SPMLA_OK;
  if (K > MAX_K) return SPMLA_ELIMIT;
  if (!a || !a_scales || !w || !w_scales || !out) return SPMLA_EARG;
  const int kb = (K + 127) / 128;
  if ((T > 1 && (a_st < K || as_st < kb || o_st < N)) || (N > 1 && w_st < K) || (N > 128 && ws_st < kb)) return SPMLA_EARG;
  if (((uintptr_t)a & 15) || (a_st & 15) || ((uintptr_t)w & 15) || (w_st & 15) || ((uintptr_t)a_scales & 3) ||
      ((uintptr_t)w_scales & 3) || ((uintptr_t)out & 1))
    return SPMLA_EALIGN;
  if (T > MAX_TOKENS || N > MAX_TOKENS) return SPMLA_ELIMIT;
  if (a_st > MAX_K || w_st > MAX_K || as_st > (1 << 20)) return SPMLA_ELIMIT;
  lin::LinearParams p{(const uint8_t*)a, a_st, a_scales, as_st, (const uint8_t*)w, w_st, w_scales, ws_st, out, o_st,
                      T, N, K, ((uintptr_t)out & 7) == 0 && (o_st & 3) == 0, ((uintptr_t)out & 63) == 0 && (o_st & 31) == 0};
  if (dtype == DT_F16) return lin::linear_go<DT_F16>(p, (hipStream_t)stream);
  return lin::linear_go<DT_BF16>(p, (hipStream_t)stream);
}

}  // extern "C"
