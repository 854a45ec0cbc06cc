// Attention of new tokens over every cached latent row of their request (one token each, drafts, or a prefill chunk), the
// rows found through the block table.
//
//   token i of the n new ones of a request with L cached rows (the new ones their last) sees the positions x < L - n + i + 1;
//   row of x: page block_table[b][x / bs], its row x % bs; latent_d = code_d * scale[d / 128] (Row576: code_d)
//   s = sm_scale kv_scale (q[:512] . latent + q[512:] . rope),  p = exp(s - m),  o = kv_scale sum p latent / sum p,
//   lse = ln sum exp(s)
//
// One workgroup = 64 rows of (token, head) of one request, token by token, over one split of the positions: whatever the
// number of heads, a cached row is copied once for 64 query rows, and a decode step of 16 heads fills 16 of them.
// 4 waves, tiles of 32 positions, a ring of three in LDS filled by direct copies; two workgroups a compute unit:
//   * QK: wave 2 i + d multiplies half d of the dims (two scale groups, half of the rope) of query rows 32 i .. 32 i + 31:
//     S^T partials in bf16 MFMA 16x16x32, codes converted exactly, so a code is converted by two waves and the query takes
//     72 registers. (8-bit MFMA would take the codes as they are, the query in two e4m3 parts: its sums are off by 2e-6 of
//     the summed magnitudes, 1.3e-5 at most, against 4e-9 and 1.2e-7 here.) Row656: a group's sum times the rows' fp32
//     scales, then the rope. The two waves exchange half of their partials through LDS: each ends with 16 query rows;
//   * softmax: one query row per lane (and three others); base 2, 32 bits; the reference maximum moves only past TAU.
//     P goes to LDS in f16, times 2^UP so that few weights are f16 subnormals;
//   * PV: wave g owns dims 128 g .. of all 64 rows: O^T = V^T P^T (f16 MFMA 32x32x16), V^T by the 8-bit transposing read,
//     converted to f16 exactly and (Row656) multiplied by scale * 2^-e in f16; e (per wave) keeps that in range: it follows
//     the largest scale so far (a value is off by half an f16 step, or 2^-39 of the largest magnitude so far).
// Two barriers a tile: partials of tile j + 1 and PV of tile j; then the softmax of tile j + 1, while the other
// workgroup's products run.
// Masked positions take no part: scores of -inf, and where the mask cuts a tile V's values that are no numbers are taken
// out of the product and given to the rows that see them at the end.
// Splits leave normalized fp32 partials and their lse in a workspace; a second kernel joins them.
#include "spmla_common.h"
#include "spmla_quant.h"

namespace spmla {
namespace chunk {

constexpr int HR = 64;                // query rows per half (4 waves)
constexpr int TR = 32;                // positions per tile
constexpr int IDS = 256;              // positions whose rows are looked up at a time
constexpr float TAU = 6.0f, UP = 9.0f, FAR = 65536.f;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

struct Params {
  const uint16_t* q; long long q_st, q_sh;
  const uint8_t* cache; long long rows, stride;            // rows of the cache, rows from a block to the next
  int bs;
  const int* table; long long t_st; int W;
  const int* seqs; const int* start; int B, T, H, S, span; // splits of span positions each (a multiple of TR)
  float c, kv_scale;                                       // |sm_scale kv_scale| log2(e)
  int flip, tiles;
  uint16_t* out; long long o_st, o_sh;
  float* lse; long long l_st;
  float* opart; float* lpart;                              // [S][T][H][512], [S][T][H]
};

template <bool R5, int NH>
struct Lds {
  static constexpr int RING = NH == 1 ? 3 : 4;
  static constexpr int CODE = 4 * TR * 128;                // codes by scale group, [4][32 rows][128]
  static constexpr int RP = TR * (R5 ? 64 : 128);          // rope
  static constexpr int SC = R5 ? 0 : 4 * TR * 4;           // scales by group, [4][32]
  static constexpr int TILE = CODE + RP + SC;
  static constexpr int X = RING * TILE;                    // exchanged partials [wave][16 positions][64 lanes][16]
  static constexpr int P = X + 4 * NH * 2048;              // [64 NH query rows][32 positions] f16
  static constexpr int FAC = P + NH * HR * TR * 2;         // rescale factors [64 NH]
  static constexpr int FLAG = FAC + NH * HR * 4;           // a wave's factors are not all 1
  static constexpr int SCH = FLAG + 16 * NH;               // a wave's scales in f16, [4 NH][32]
  static constexpr int ID = SCH + 4 * NH * TR * 2;         // addresses of the rows of two times IDS positions
  static constexpr int OK = ID + 2 * IDS * 8;              // which of a tile's positions have rows, a bit each
  static constexpr int TOTAL = OK + 2 * IDS / 32 * 4;
  static_assert(TOTAL <= (NH == 1 ? 80 : 160) * 1024 && ID % 8 == 0, "two workgroups of 4 waves a compute unit, or one of 8");
};

__device__ __attribute__((aligned(16))) uint8_t zero_row[ROW656];

__device__ inline float swap32_max(float x) {
  const uint32_t u = f2u(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t a = r[0], b = r[1];
  return fmaxf(u2f(a), u2f(b));
}
__device__ inline float swap16_max(float x) {
  const uint32_t u = f2u(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t a = r[0], b = r[1];
  return fmaxf(u2f(a), u2f(b));
}
__device__ inline float swap32_sum(float x) {
  const uint32_t u = f2u(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t a = r[0], b = r[1];
  return u2f(a) + u2f(b);
}
__device__ inline float swap16_sum(float x) {
  const uint32_t u = f2u(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t a = r[0], b = r[1];
  return u2f(a) + u2f(b);
}
__device__ inline float quad_max(float x) { return swap16_max(swap32_max(x)); }      // over lanes l % 16
__device__ inline float quad_sum(float x) { return swap16_sum(swap32_sum(x)); }

__device__ inline uint32_t pk_f16(float a, float b) { return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b}); }
__device__ inline uint32_t pk_bf16(float a, float b) { return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b}); }
__device__ inline uint32_t lo_f16x2(uint32_t w) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)); }
__device__ inline uint32_t hi_f16x2(uint32_t w) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)); }
__device__ inline uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, a) * __builtin_bit_cast(f16x2, b));
}

// 8 e4m3 codes -> 8 bf16, exact
__device__ inline bf16x8 codes8(int a, int b) {
  return __builtin_bit_cast(bf16x8, u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false)),
                                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true)),
                                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false)),
                                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true))});
}
// place of chunk c (16 bytes) in a row of 128 bytes: c ^ swz(row); 16 rows' chunks c lie in all 64 banks
__device__ inline int swz(int row) { return ((row & 2) << 1) | ((row & 4) >> 2) | ((row & 8) >> 2); }

template <bool R5, int NH>
__global__ void __launch_bounds__(256 * NH, 2) kernel(Params p) {
  using L = Lds<R5, NH>;
  constexpr int RB = R5 ? ROW576 : ROW656, MR = HR * NH;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem_generic[];
  SPMLA_LDS uint8_t* lds = (SPMLA_LDS uint8_t*)smem_generic;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = NH == 1 ? 0 : w >> 2, wl = w & 3;      // this wave's half and its number there
  const int l16 = lane & 15, l32 = lane & 31, qt = lane >> 4, hh = lane >> 5;

  // ---- work item: split and tile of query rows. Request b starts at tile start[b] * H / 64 + b.
  const int f = remap_xcd(blockIdx.x, p.tiles * p.S);
  if (f < 0) return;
  const int sp = f / p.tiles, ti = p.tiles - 1 - f % p.tiles;
  int nb = 0;
  for (int at = 0; at < p.B; at += 64) {
    const int b = at + lane;
    const bool in = b < p.B && (long long)p.start[b] * p.H / MR + b <= ti;
    nb += __popcll(__ballot(in));
  }
  const int b = nb > 0 ? nb - 1 : 0;
  int t0 = p.start[b], t1 = p.start[b + 1];
  const long long r0 = (long long)(ti - (int)((long long)t0 * p.H / MR) - b) * MR;
  t0 = t0 < 0 ? 0 : t0;
  t1 = t1 > p.T ? p.T : t1;
  const long long nrows = (long long)(t1 - t0) * p.H;
  if (r0 < 0 || r0 >= nrows) return;
  const int live = nrows - r0 < MR ? (int)(nrows - r0) : MR;               // query rows here
  const int past = p.seqs[b] - (t1 - t0);                                  // rows before the new ones
  const long long cap = (long long)p.W * p.bs;
  auto limit_of = [&](int r) -> int {                                      // positions that row r sees
    const long long x = (long long)past + (r0 + r) / p.H + 1;
    return x < 0 ? 0 : x > cap ? (int)cap : (int)x;
  };
  const int least = limit_of(0), most = limit_of(live - 1);
  const long long first = (long long)sp * p.span;
  const int kb = first < most ? (int)first : most;
  const int ke = sp + 1 < p.S && first + p.span < most ? (int)(first + p.span) : most;       // (the last split takes the rest)
  const int nt = (ke - kb + TR - 1) / TR;
  if (nt <= 0 && sp > 0) {                                                 // nothing of this split: no weight in the join
    if (tid < live) {
      const long long r = r0 + tid;
      p.lpart[((long long)sp * p.T + t0) * p.H + r] = -__builtin_inff();
    }
    return;
  }
  const int* btrow = p.table + (long long)b * p.t_st;

  // ---- rows of IDS positions: looked up (x beyond ke: none), then their addresses written with a bit per position
  auto look = [&](int part) -> int {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int pos = kb + part * IDS + tid;
    if (pos >= ke || (NH > 1 && tid >= IDS)) return -1;
    const int page = btrow[pos / p.bs];
    const long long y = (long long)page * p.stride + pos % p.bs;
    return page >= 0 && y < p.rows ? (int)y : -1;
  };
  auto note = [&](int part, int row) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, l32 = lane & 31;
    if (NH > 1 && tid >= IDS) return;
    const int at = (part & 1) * IDS + tid;
    const uint64_t a = (uint64_t)(uintptr_t)p.cache + (uint64_t)(uint32_t)row * RB;
    ((SPMLA_LDS uint64_t*)(lds + L::ID))[at] = row >= 0 ? a : (uint64_t)(uintptr_t)zero_row;
    const uint64_t has = __ballot(row >= 0);
    if (l32 == 0) ((SPMLA_LDS uint32_t*)(lds + L::OK))[at >> 5] = (uint32_t)(has >> (lane & 32));
  };
  int found = look(0);

  // ---- query operands [chunk pair or rope][half chunk][own or partner's 16 query rows] of rows 32 (w / 2) .. and half dh of the dims: B
  // operands of 16x16x32, lane quarter qt the dims 64 n + 16 qt + 8 e .. + 7 (one 16-byte read of codes serves both e)
  const int dh = wl & 1, qb = HR * half + 32 * (wl >> 1);
  bf16x8 qf[4][2][2], qpe[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = qb + 16 * (i ^ dh) + l16;             // (i = 0: the rows that this wave joins)
    const long long r = r0 + (row < live ? row : live - 1);
    const uint16_t* qp = p.q + (t0 + r / p.H) * p.q_st + (r % p.H) * p.q_sh;
    const uint32_t turn = p.flip ? 0x80008000u : 0u;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) qf[n][e][i] = __builtin_bit_cast(bf16x8, *(const u32x4*)(qp + 256 * dh + 64 * n + 16 * qt + 8 * e) ^ turn);
    qpe[i] = __builtin_bit_cast(bf16x8, *(const u32x4*)(qp + D_LAT + 32 * dh + 8 * qt) ^ turn);
  }
  const int qr = HR * half + 16 * wl + l16;               // the query row whose softmax this lane shares
  note(0, found);
  if (tid < 4 * NH) ((SPMLA_LDS int*)(lds + L::FLAG))[tid] = 0;
  lds_barrier();

  // ---- copies of a tile: rows 8 i + lane / 8 of a scale group's codes, the chunk whose place is lane % 8 (4 waves: wave w
  // all of group w, 8 waves: half of group w % 4), a share of the rope and of the scales (some twice). COPIES instructions a
  // wave whatever the tile.
  constexpr int COPIES = (R5 ? 1 : NH == 1 ? 2 : 1) + 4 / NH;
  // the lane id, opaque in every step: LDS places made of it are formed again, not kept (spilled, a tile's wait for one would
  // wait for all copies)
  auto here = [&]() -> int {
    int x = lane;
    asm volatile("" : "+v"(x));
    return x;
  };
  auto issue = [&](int j, int slot) {
    const int lane = here(), l32 = lane & 31, hh = lane >> 5;
    SPMLA_LDS uint64_t* id = (SPMLA_LDS uint64_t*)(lds + L::ID) + (j * TR & (2 * IDS - 1));
    SPMLA_LDS uint8_t* d = lds + slot * L::TILE;
    const int r = lane >> 3, place = (lane & 7) ^ swz(r);
    auto copy = [&](int row, uint32_t off, SPMLA_LDS uint8_t* to) { dma16((const void*)(id[row] + off), to); };
#pragma unroll
    for (int n = 0; n < 4 / NH; ++n) {
      const int i = n + 2 * half;
      copy(8 * i + r, 128 * wl + 16 * (place ^ ((i & 1) << 1)), d + wl * 4096 + i * 1024);
    }
    auto scales = [&]() { dma4((const void*)(id[l32] + (uint32_t)(SC_OFF + 4 * (2 * (w & 1) + hh))), d + L::CODE + L::RP + (w & 1) * 256); };
    if constexpr (R5) {                                   // 16 rows of 64 bytes a copy
      const int rr = 16 * (w & 1) + (lane >> 2);
      copy(rr, D_LAT + 16 * ((lane & 3) ^ ((rr >> 2) & 3)), d + L::CODE + (w & 1) * 1024);
    } else {
      if (NH == 1 || half == 0) copy(8 * wl + r, ROPE_OFF + 16 * (place ^ ((wl & 1) << 1)), d + L::CODE + wl * 1024);
      if (NH == 1 || half == 1) scales();
    }
  };

  f32x16 O[4][2];                                         // [32 dims of group w][32 query rows]
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int i = 0; i < 2; ++i) O[d][i] = f32x16{};
  float m = -__builtin_inff(), l = 0.f;                   // of query row qr (m: as scores are, shared by its four lanes; l: this lane's)
  bool far = false;                                       // a reference is beyond FAR
  int ex2 = -126;                                         // Row656: V' and O carry 2^-ex2
  int odd_from = 0x7fffffff;

  // Partial scores of a tile over this wave's dims: S^T blocks of 16 positions x 16 query rows (block 0: the rows this wave
  // joins, kept; block 1: its partner's, to LDS). Steps of two products (20: 16 of codes, 4 a block pair of rope at the end of
  // its positions): the conversions of the next step's operand run under the products of this one, reads two ahead.
  f32x4 part[2];
  auto partials = [&](int slot) {
    const int lane = here(), l16 = lane & 15, qt = lane >> 4;
    SPMLA_LDS uint8_t* d = lds + slot * L::TILE;
    SPMLA_LDS uint8_t* at = d + (2 * dh) * 4096 + l16 * 128;
    const int x0 = 16 * (qt ^ swz(l16)), x1 = x0 ^ 64;
    auto kread = [&](int n) -> i32x4 {                    // unit n: positions 16 (n / 4) .., group 2 dh + n / 2 % 2, chunks 4 (n % 2) ..
      return *(SPMLA_LDS i32x4*)(at + (n >> 2) * 2048 + ((n >> 1) & 1) * 4096 + ((n & 1) ? x1 : x0));
    };
    auto rread = [&](int u) -> i32x4 {                    // rope of positions 16 u ..: Row576 8 codes, Row656 8 bf16
      if constexpr (R5) {
        const i32x2 y = *(SPMLA_LDS i32x2*)(d + L::CODE + u * 1024 + l16 * 64 + 16 * ((2 * dh + (qt >> 1)) ^ ((l16 >> 2) & 3)) + 8 * (qt & 1));
        return i32x4{y[0], y[1], 0, 0};
      } else {
        return *(SPMLA_LDS i32x4*)(d + L::CODE + u * 2048 + l16 * 128 + 16 * ((4 * dh + qt) ^ swz(l16)));
      }
    };
    i32x4 k[3] = {kread(0), kread(1), kread(2)}, kr;
    bf16x8 y[2];
    y[0] = codes8(k[0][0], k[0][1]);
    f32x4 s[2] = {}, acc[2] = {}, sc = {};
#pragma unroll
    for (int t = 0; t < 18; ++t) {                        // t % 9 < 8: half e of unit 4 u + t % 9 / 2; 8: rope
      const int u = t / 9, i9 = t % 9, n = 4 * u + i9 / 2;
      // the next step's operand
      if (i9 < 8) {
        if (i9 & 1) {
          if (n + 3 < 8) k[n % 3] = kread(n + 3);         // (its codes are converted)
          if (i9 == 7) y[(t + 1) & 1] = R5 ? codes8(kr[0], kr[1]) : __builtin_bit_cast(bf16x8, kr);
          else y[(t + 1) & 1] = codes8(k[(n + 1) % 3][0], k[(n + 1) % 3][1]);
        } else {
          y[(t + 1) & 1] = codes8(k[n % 3][2], k[n % 3][3]);
          if (i9 == 4) kr = rread(u);
        }
      } else if (u == 0) {
        y[(t + 1) & 1] = codes8(k[4 % 3][0], k[4 % 3][1]);
      }
      if constexpr (!R5)
        if (i9 == 1 || i9 == 5) sc = *(SPMLA_LDS f32x4*)(d + L::CODE + L::RP + (2 * dh + i9 / 4) * 128 + u * 64 + qt * 16);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bf16x8 q = i9 == 8 ? qpe[i] : qf[(i9 / 2) & 3][i9 & 1][i];
        f32x4& to = R5 || i9 == 8 ? s[i] : acc[i];
        to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y[t & 1], q, to, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {                       // a product, two conversions, ...
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, 2, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (!R5) {
        if (i9 == 3 || i9 == 7) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[i][r] = i9 == 3 ? acc[i][r] * sc[r] : __builtin_fmaf(acc[i][r], sc[r], s[i][r]);
            acc[i] = f32x4{};
          }
        }
      }
      if (i9 == 8) {
        part[u] = s[0];
        *(SPMLA_LDS f32x4*)(lds + L::X + w * 2048 + u * 1024 + lane * 16) = s[1];
        s[0] = s[1] = f32x4{};
      }
    }
  };

  // softmax of tile j, its P and factors: value 4 u + r of a lane is position 16 u + 4 qt + r
  auto softmax = [&](int j) {
    const int lane = here(), l16 = lane & 15, qt = lane >> 4, qr = HR * half + 16 * wl + l16;
    f32x4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) s[u] = part[u] + *(SPMLA_LDS f32x4*)(lds + L::X + (w ^ 1) * 2048 + u * 1024 + lane * 16);
    const uint32_t has = __builtin_amdgcn_readfirstlane(((SPMLA_LDS uint32_t*)(lds + L::OK))[j & (2 * IDS / TR - 1)]);
    const int k0 = kb + j * TR;
    if (__builtin_expect(has != 0xffffffffu || k0 + TR > least, 0)) {
      asm volatile("" : "+v"(s[0]), "+v"(s[1]));           // (a branch, not 40 selects in every tile)
      const int limit = limit_of(qr < live ? qr : live - 1);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int x = 16 * u + 4 * qt + r;
          s[u][r] = (has >> x & 1) && k0 + x < limit ? s[u][r] : -__builtin_inff();
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[u][r]);
    mx = quad_max(mx);
    float fac = 1.f;
    const bool move = __any(mx * p.c > m * p.c + TAU);
    if (move) {
      const float mn = fmaxf(m, mx), a = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((m - mn) * p.c);
      m = mn;
      l *= a;
      far = __any(fabsf(mn * p.c) > FAR && mn > -__builtin_inff());
      fac = a;
    }
    if (qt == 0) ((SPMLA_LDS float*)(lds + L::FAC))[qr] = fac;
    if (lane == 0) ((SPMLA_LDS int*)(lds + L::FLAG))[w] = move;
    const float base = m == -__builtin_inff() ? 0.f : m, ref = UP - base * p.c;
    if (__builtin_expect(far, 0)) {                        // the rounding of m c would count: differences first
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r] - base, p.c, UP));
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], p.c, ref));
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) l += s[u][r];
#pragma unroll
    for (int u = 0; u < 2; ++u) {                          // half of chunk 2 u + qt / 2
      const int ch = (2 * u + (qt >> 1)) ^ ((qr >> 2) & 3);
      *(SPMLA_LDS i32x2*)(lds + L::P + qr * 64 + 16 * ch + 8 * (qt & 1)) = i32x2{(int)pk_f16(s[u][0], s[u][1]), (int)pk_f16(s[u][2], s[u][3])};
    }
  };

  // O += V^T P^T of tile j
  auto values = [&](int j, int slot) {
    const int lane = here(), l32 = lane & 31, hh = lane >> 5;
    const int vrow = 8 * hh + ((lane & 15) >> 1);         // V^T: row of the transposing read
    SPMLA_LDS uint8_t* d = lds + slot * L::TILE;
    const int k0 = kb + j * TR;
    const i32x4 fl = *(SPMLA_LDS i32x4*)(lds + L::FLAG + 16 * half);
    const int any = __builtin_amdgcn_readfirstlane(fl[0] | fl[1] | fl[2] | fl[3]);
    float sc = 0.f;
    if constexpr (!R5) {
      sc = *(SPMLA_LDS float*)(d + L::CODE + L::RP + wl * 128 + l32 * 4);
      const float fin = fabsf(sc) < __builtin_inff() ? fabsf(sc) : 0.f;
      if (__builtin_expect(__any(fin * u2f((uint32_t)(127 - ex2) << 23) > 64.f), 0)) {      // a larger scale than any before: e follows
        float top = fin;
        asm volatile("" : "+v"(top));
#pragma unroll
        for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
        int e = (int)(f2u(top) >> 23) - 127 - 5;                            // scale * 2^-e < 64
        e = __builtin_amdgcn_readfirstlane(e < -126 ? -126 : e);
        const float a = __builtin_amdgcn_exp2f((float)(ex2 - e));
        ex2 = e;
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) O[x][i][r] *= a;
      }
      const bool masked = k0 + TR > least && least < most && !(fabsf(sc) < __builtin_inff());
      const _Float16 h = masked ? (_Float16)0.f : (_Float16)(sc * u2f((uint32_t)(127 - ex2) << 23));
      ((SPMLA_LDS _Float16*)(lds + L::SCH))[w * TR + l32] = h;
    }
    if (__builtin_expect(any, 0)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float a = ((SPMLA_LDS float*)(lds + L::FAC))[HR * half + 32 * i + l32];
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int r = 0; r < 16; ++r) O[x][i][r] *= a;
      }
    }
    if (__builtin_expect(k0 + TR > least && least < most, 0)) {
      // the mask cuts this tile: codes that are no numbers become 0 in the wave's group, whose values alone are read from now on
      // (8 waves: by the other half's wave of the group as well, whose turn comes later)
      uint32_t odd = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        SPMLA_LDS u32x4* at = (SPMLA_LDS u32x4*)(d + wl * 4096 + i * 1024 + lane * 16);
        u32x4 y = *at;
        uint32_t bad = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t nan = ((y[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
          bad |= nan;
          y[e] &= ~((nan >> 7) * 255u);
        }
        odd |= bad;
        if (bad) *at = y;
      }
      if constexpr (!R5) odd |= fabsf(sc) < __builtin_inff() ? 0u : 1u;     // (its f16 form is 0)
      if (__any(odd != 0)) odd_from = odd_from < k0 ? odd_from : k0;
    }
    const int vo = wl * 4096 + vrow * 128 + 8 * (lane & 1), vs = swz(vrow) ^ ((lane >> 4) & 1);
    auto vread = [&](int n) -> i32x2 {                    // unit n: positions 16 (n / 4) .., dims 32 (n % 4) ..
      return __builtin_amdgcn_ds_read_tr8_b64_v2i32((SPMLA_LDS i32x2*)(d + vo + 16 * (vs ^ (2 * (n & 3))) + (n >> 2) * 2048));
    };
    auto pread = [&](int ks, int i) -> f16x8 {
      return __builtin_bit_cast(f16x8, *(SPMLA_LDS u32x4*)(lds + L::P + (HR * half + 32 * i + l32) * 64 + 16 * ((2 * ks + hh) ^ ((l32 >> 2) & 3))));
    };
    auto vconv = [&](i32x2 c, u32x4 f) -> u32x4 {
      u32x4 v = {lo_f16x2((uint32_t)c[0]), hi_f16x2((uint32_t)c[0]), lo_f16x2((uint32_t)c[1]), hi_f16x2((uint32_t)c[1])};
      if constexpr (!R5)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = mul_f16x2(v[e], f[e]);
      return v;
    };
    auto sread = [&](int ks) -> u32x4 {
      if constexpr (R5) return u32x4{};
      else return *(SPMLA_LDS u32x4*)(lds + L::SCH + (w * TR + 16 * ks + 8 * hh) * 2);
    };
    u32x4 f[2] = {sread(0)};
    i32x2 t[3] = {vread(0), vread(1), vread(2)};
    f16x8 pb[2] = {pread(0, 0), pread(0, 1)};
    u32x4 v[2];
    v[0] = vconv(t[0], f[0]);
    t[0] = vread(3);
#pragma unroll
    for (int n = 0; n < 8; ++n) {                         // the next unit's conversions under this one's products
      if (n == 1) f[1] = sread(1);
      if (n < 7) v[(n + 1) & 1] = vconv(t[(n + 1) % 3], f[n >= 3]);
      if (n < 4) t[(n + 1) % 3] = vread(n + 4);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        O[n & 3][i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v[n & 1]), pb[i], O[n & 3][i], 0, 0, 0);
        if (n == 3) pb[i] = pread(1, i);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, R5 ? 2 : 4, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // ---- steps: half 0 takes the products of tile s / 2 in even steps and a softmax in odd ones, half 1 the other way round, so
  // that one half's products run beside the other's softmax
  const bool works = HR * half < live;
  if (nt > 0) {
    for (int j = 0; j < 3 && j < nt; ++j) issue(j, j);
    if (nt > 2) wait_vm<2 * COPIES>(); else if (nt > 1) wait_vm<COPIES>(); else wait_vm<0>();
    lds_barrier();
    if (works) partials(0);
    lds_barrier();
    if (half == 0) softmax(0);
    if (nt > 2) wait_vm<COPIES>(); else wait_vm<0>();
    lds_barrier();
  }
  int slot = 0;                                           // of tile s / 2; the next ones follow
  for (int s = 0; s < 2 * nt; ++s) {
    const int j = s >> 1;
    if (!(s & 1)) {
      // rows of the next IDS positions: looked up 7 tiles before a part ends, written 4 before, copied from 3 before
      const int in = j & (IDS / TR - 1), next = j / (IDS / TR) + 1;
      if (in == IDS / TR - 7 && next * (IDS / TR) < nt) found = look(next);
      if (in == IDS / TR - 4 && next * (IDS / TR) < nt) note(next, found);
    }
    if ((s & 1) == half) {
      if (works) {
        partials(slot + 1 == L::RING ? 0 : slot + 1);     // (behind the last tile: of what lies there, not used)
        values(j, slot);
      }
    } else {
      // tile j + 3 into the slot of tile j, whose values are taken (4 waves), or of tile j - 1
      if (j + 3 < nt) issue(j + 3, NH == 1 ? slot : (slot + 3) & 3);
      if (works && (s + 1) / 2 < nt) softmax((s + 1) / 2);
    }
    if (s & 1) {                                          // tile j + 2 is there
      if (j + 3 < nt) wait_vm<COPIES>(); else wait_vm<0>();
      slot = slot + 1 == L::RING ? 0 : slot + 1;
    }
    lds_barrier();
  }

  // ---- join of a row's four lanes, 1 / l for the waves that hold its dims
  l = quad_sum(l);
  const float ln = m == -__builtin_inff() ? m : m * p.c * 0.69314718055994531f + (__builtin_log2f(l) - UP) * 0.69314718055994531f;
  SPMLA_LDS float* inv = (SPMLA_LDS float*)(lds + L::FAC);
  if (qt == 0) inv[qr] = l > 0.f || l != l ? 1.f / l : 0.f;
  const bool whole = p.S == 1;
  if (qt == 0 && qr < live) {
    const long long r = r0 + qr;
    if (whole) {
      if (p.lse) p.lse[(t0 + r / p.H) * p.l_st + r % p.H] = ln;
    } else {
      p.lpart[((long long)sp * p.T + t0) * p.H + r] = ln;
    }
  }
  if (lane == 0) ((SPMLA_LDS int*)(lds + L::FLAG))[w] = odd_from;
  lds_barrier();
  if constexpr (NH > 1) {                                 // (the wave of the same group that came first took them out for both)
    const int other = __builtin_amdgcn_readfirstlane(((SPMLA_LDS int*)(lds + L::FLAG))[w ^ 4]);
    odd_from = odd_from < other ? odd_from : other;
  }
  const float back = p.kv_scale;
  float a[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) a[i] = inv[HR * half + 32 * i + l32] * back;
  const float e2 = R5 ? 1.f : u2f((uint32_t)(ex2 + 127) << 23);
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) O[x][i][r] = O[x][i][r] * e2 * a[i];
  if (__builtin_expect(odd_from < ke, 0)) {               // V that is no number, for the rows that see it
    int lim[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = HR * half + 32 * i + l32;
      lim[i] = limit_of(row < live ? row : live - 1);
    }
    for (int pos = odd_from; pos < ke; ++pos) {
      const int page = btrow[pos / p.bs];
      const long long y = (long long)page * p.stride + pos % p.bs;
      if (page < 0 || y >= p.rows) continue;
      const uint8_t* row = p.cache + y * RB;
      const float sc = R5 ? 1.f : *(const float*)(row + SC_OFF + 4 * wl);
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float v = e4m3_to_f32(row[128 * wl + 32 * x + 8 * (r >> 2) + 4 * hh + (r & 3)]) * sc * p.kv_scale;
          const float add = fabsf(v) < __builtin_inff() ? 0.f : v;
#pragma unroll
          for (int i = 0; i < 2; ++i) O[x][i][r] += pos < lim[i] ? add : 0.f;
        }
    }
  }
  if (!whole) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = HR * half + 32 * i + l32;
      if (row >= live) continue;
      float* o = p.opart + (((long long)sp * p.T + t0) * p.H + r0 + row) * D_LAT + 128 * wl + 4 * hh;
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *(f32x4*)(o + 32 * x + 8 * q) = f32x4{O[x][i][4 * q], O[x][i][4 * q + 1], O[x][i][4 * q + 2], O[x][i][4 * q + 3]};
    }
    return;
  }
  // bf16 rows through LDS, 32 at a time: the wave's 128 dims, 16-byte chunks permuted by the row
  SPMLA_LDS uint8_t* ob = lds + w * (32 * 256);
  static_assert(4 * NH * 32 * 256 <= L::FAC, "the output's rows fit below the factors");
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(SPMLA_LDS i32x2*)(ob + l32 * 256 + 16 * ((4 * x + q) ^ l16) + 8 * hh) =
            i32x2{(int)pk_bf16(O[x][i][4 * q], O[x][i][4 * q + 1]), (int)pk_bf16(O[x][i][4 * q + 2], O[x][i][4 * q + 3])};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int row = 4 * k + qt;
      if (HR * half + 32 * i + row < live) {
        const long long r = r0 + HR * half + 32 * i + row;
        *(u32x4*)(p.out + (t0 + r / p.H) * p.o_st + (r % p.H) * p.o_sh + 128 * wl + 8 * l16) =
            *(SPMLA_LDS u32x4*)(ob + row * 256 + 16 * (l16 ^ (row & 15)));
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// Joins the splits of query row (t, h): weights exp(lse_s - max); a split without keys has lse -inf and its partial, which
// was not written, is not read. One wave a row, 8 dims a lane.
struct MergeParams {
  const float* opart; const float* lpart; const int* start; int B, T, H, S;
  uint16_t* out; long long o_st, o_sh;
  float* lse; long long l_st;
};
__global__ void __launch_bounds__(256) merge_kernel(MergeParams p) {
  const int lane = threadIdx.x & 63;
  const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), n = (long long)p.T * p.H;
  if (r >= n || r / p.H < p.start[0] || r / p.H >= p.start[p.B]) return;      // rows of no request stay as they are
  float top = -__builtin_inff();
  for (int s = lane; s < p.S; s += 64) {
    const float x = p.lpart[s * n + r];
    top = x > top || x != x ? x : top;
  }
#pragma unroll
  for (int x = 32; x; x >>= 1) {
    const float y = __shfl_xor(top, x);
    top = y > top || y != y ? y : top;
  }
  const float ref = top == -__builtin_inff() ? 0.f : top;
  float sum = 0.f;
  f32x4 a = {}, b = {};
  for (int s = 0; s < p.S; ++s) {
    const float x = p.lpart[s * n + r];
    if (x == -__builtin_inff()) continue;
    const float wgt = __expf(x - ref);
    const f32x4* o = (const f32x4*)(p.opart + (s * n + r) * D_LAT + 8 * lane);
    a += wgt * o[0];
    b += wgt * o[1];
    sum += wgt;
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  a *= inv;
  b *= inv;
  const long long t = r / p.H, h = r % p.H;
  *(u32x4*)(p.out + t * p.o_st + h * p.o_sh + 8 * lane) = u32x4{pk_bf16(a[0], a[1]), pk_bf16(a[2], a[3]), pk_bf16(b[0], b[1]), pk_bf16(b[2], b[3])};
  if (p.lse && lane == 0) p.lse[t * p.l_st + h] = sum > 0.f || sum != sum ? ref + __logf(sum) : -__builtin_inff();
}

}  // namespace chunk
}  // namespace spmla

using namespace spmla;

extern "C" long long spmla_attn_chunk_ws_bytes(int T, int H, int S) {
  if (T <= 0 || H <= 0 || S <= 1) return 0;
  return (long long)T * H * S * (D_LAT + 1) * 4;
}

extern "C" int spmla_attn_chunk(const void* q, long long q_st, long long q_sh, const void* cache, long long rows, int row_bytes,
                                int block_size, long long stride_rows, const int* table, long long t_st, int W, const int* seqs,
                                const int* start, int B, int T, int H, float sm_scale, float kv_scale, int S, int span, int wide, void* out,
                                long long o_st, long long o_sh, float* lse, long long l_st, void* ws, long long ws_bytes, void* stream) {
  if (B < 0 || T < 0 || H < 0 || W < 0 || rows < 0 || block_size <= 0 || stride_rows < block_size || S < 1 || span < 1 ||
      span % chunk::TR || (row_bytes != ROW656 && row_bytes != ROW576))
    return SPMLA_EARG;
  if (T > MAX_TOKENS || B > MAX_TOKENS || H > 65536 || S > 256 || rows > 0x7fffffffll || (long long)W * block_size > 0x7fffff00ll) return SPMLA_ELIMIT;
  if (B == 0 || T == 0 || H == 0) return SPMLA_OK;
  if (!q || !start || !seqs || !out || (rows && !cache) || (W && !table)) return SPMLA_EARG;
  if (((q_st | q_sh | o_st | o_sh) & 7) || (((uintptr_t)q | (uintptr_t)cache | (uintptr_t)out) & 15) ||
      (((uintptr_t)start | (uintptr_t)seqs | (uintptr_t)table | (uintptr_t)lse) & 3))
    return SPMLA_EALIGN;
  if (S > 1 && (!ws || ((uintptr_t)ws & 15))) return ws ? SPMLA_EALIGN : SPMLA_EARG;
  if (S > 1 && ws_bytes < spmla_attn_chunk_ws_bytes(T, H, S)) return SPMLA_EARG;
  const int r5 = row_bytes == ROW576, nh = wide ? 2 : 1;
  const long long tiles = (long long)T * H / (chunk::HR * nh) + B;
  if (tiles * S > (1ll << 30)) return SPMLA_ELIMIT;
  float* opart = (float*)ws;
  float* lpart = opart ? opart + (long long)T * H * S * D_LAT : nullptr;
  const float sc = sm_scale * kv_scale;
  chunk::Params p{(const uint16_t*)q, q_st, q_sh, (const uint8_t*)cache, rows, stride_rows, block_size, table, t_st, W, seqs, start, B, T,
                  H, S, span, fmaxf((sc < 0.f ? -sc : sc) * 1.4426950408889634f, 1e-30f), kv_scale, sc < 0.f, (int)tiles, (uint16_t*)out, o_st, o_sh, lse,
                  l_st, opart, lpart};
  static DynLds attr[4];
  static Launcher go[4];
  const int at = 2 * (nh - 1) + r5;
  const void* fn[4] = {(const void*)chunk::kernel<false, 1>, (const void*)chunk::kernel<true, 1>, (const void*)chunk::kernel<false, 2>,
                       (const void*)chunk::kernel<true, 2>};
  const int lds[4] = {chunk::Lds<false, 1>::TOTAL, chunk::Lds<true, 1>::TOTAL, chunk::Lds<false, 2>::TOTAL, chunk::Lds<true, 2>::TOTAL};
  if (const int rc = attr[at].ensure(fn[at], lds[at])) return rc;
  hipStream_t s = (hipStream_t)stream;
  if (const int rc = go[at](fn[at], dim3((unsigned)((tiles * S + 7) / 8 * 8)), 256 * nh, lds[at], s, p)) return rc;
  if (S == 1) return SPMLA_OK;
  static Launcher join;
  const chunk::MergeParams mp{opart, lpart, start, B, T, H, S, (uint16_t*)out, o_st, o_sh, lse, l_st};
  return join((const void*)chunk::merge_kernel, dim3((unsigned)(((long long)T * H + 3) / 4)), 256, 0, s, mp);
}
