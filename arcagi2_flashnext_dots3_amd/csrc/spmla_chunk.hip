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

constexpr int MR = 64;                // query rows per workgroup
constexpr int TR = 32;                // positions per tile
constexpr int IDS = 256;              // positions whose rows are looked up at a time
constexpr int NRING = 3;
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

template <bool R5>
struct Lds {
  static constexpr int CODE = 4 * TR * 128;                // codes by scale group, [4][32 rows][128]
  static constexpr int RP = TR * (R5 ? 64 : 128);          // rope
  static constexpr int SC = R5 ? 0 : 4 * TR * 4;           // scales by group, [4][32]
  static constexpr int TILE = CODE + RP + SC;
  static constexpr int X = NRING * TILE;                   // exchanged partials [wave][16 positions][64 lanes][16]
  static constexpr int P = X + 4 * 2048;                   // [64 query rows][32 positions] f16
  static constexpr int FAC = P + MR * TR * 2;              // rescale factors [64]
  static constexpr int FLAG = FAC + MR * 4;                // a wave's factors are not all 1
  static constexpr int SCH = FLAG + 16;                    // a wave's scales in f16, [4][32]
  static constexpr int ID = (SCH + 4 * TR * 2 + 7) & ~7;   // addresses of the rows of two times IDS positions
  static constexpr int OK = ID + 2 * IDS * 8;              // which of a tile's positions have rows, a bit each
  static constexpr int TOTAL = OK + 2 * IDS / 32 * 4;
  static_assert(2 * TOTAL <= 160 * 1024, "two workgroups a compute unit");
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

template <bool R5>
__global__ void __launch_bounds__(256, 2) kernel(Params p) {
  using L = Lds<R5>;
  constexpr int RB = R5 ? ROW576 : ROW656;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem_generic[];
  SPMLA_LDS uint8_t* lds = (SPMLA_LDS uint8_t*)smem_generic;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
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
  auto look = [&](int half) -> int {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int pos = kb + half * IDS + tid;
    if (pos >= ke) return -1;
    const int page = btrow[pos / p.bs];
    const long long y = (long long)page * p.stride + pos % p.bs;
    return page >= 0 && y < p.rows ? (int)y : -1;
  };
  auto note = [&](int half, int row) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & 63, l32 = lane & 31;
    const int at = (half & 1) * IDS + tid;
    const uint64_t a = (uint64_t)(uintptr_t)p.cache + (uint64_t)(uint32_t)row * RB;
    ((SPMLA_LDS uint64_t*)(lds + L::ID))[at] = row >= 0 ? a : (uint64_t)(uintptr_t)zero_row;
    const uint64_t has = __ballot(row >= 0);
    if (l32 == 0) ((SPMLA_LDS uint32_t*)(lds + L::OK))[at >> 5] = (uint32_t)(has >> (lane & 32));
  };
  int found = look(0);

  // ---- query operands [chunk pair or rope][half chunk][query rows 16 i ..] of rows 32 (w / 2) .. and half dh of the dims: B
  // operands of 16x16x32, lane quarter qt the dims 64 n + 16 qt + 8 e .. + 7 (one 16-byte read of codes serves both e)
  const int dh = w & 1, qb = 32 * (w >> 1);
  bf16x8 qf[4][2][2], qpe[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const long long r = r0 + (qb + 16 * i + l16 < live ? qb + 16 * i + l16 : live - 1);
    const uint16_t* qp = p.q + (t0 + r / p.H) * p.q_st + (r % p.H) * p.q_sh;
    const uint32_t turn = p.flip ? 0x80008000u : 0u;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) qf[n][e][i] = __builtin_bit_cast(bf16x8, *(const u32x4*)(qp + 256 * dh + 64 * n + 16 * qt + 8 * e) ^ turn);
    qpe[i] = __builtin_bit_cast(bf16x8, *(const u32x4*)(qp + D_LAT + 32 * dh + 8 * qt) ^ turn);
  }
  const int qr = 16 * w + l16;                            // the query row whose softmax this lane shares
  note(0, found);
  if (tid < 4) ((SPMLA_LDS int*)(lds + L::FLAG))[tid] = 0;
  lds_barrier();

  // ---- copies of a tile: wave w the codes of scale group w (copy i: rows 8 i + lane / 8, the chunk whose place is
  // lane % 8), a share of the rope and of the scales. COPIES instructions a wave whatever the tile.
  constexpr int COPIES = R5 ? 5 : 6;
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
    for (int i = 0; i < 4; ++i) copy(8 * i + r, 128 * w + 16 * (place ^ ((i & 1) << 1)), d + w * 4096 + i * 1024);
    if constexpr (R5) {                                   // 16 rows of 64 bytes a copy; waves 2 and 3 repeat those of 0 and 1
      const int rr = 16 * (w & 1) + (lane >> 2);
      copy(rr, D_LAT + 16 * ((lane & 3) ^ ((rr >> 2) & 3)), d + L::CODE + (w & 1) * 1024);
    } else {
      copy(8 * w + r, ROPE_OFF + 16 * (place ^ ((w & 1) << 1)), d + L::CODE + w * 1024);
      dma4((const void*)(id[l32] + (uint32_t)(SC_OFF + 4 * (2 * (w & 1) + hh))), d + L::CODE + L::RP + (w & 1) * 256);
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

  // partial scores of a tile over this wave's dims: S^T blocks of 16 positions x 16 query rows; those of the rows that the
  // other wave joins go to LDS, the own stay. Reads run two or three units (a read, 8 conversions, 4 MFMAs) ahead.
  f32x4 part[2];
  auto partials = [&](int slot) {
    const int lane = here(), l16 = lane & 15, qt = lane >> 4;
    SPMLA_LDS uint8_t* d = lds + slot * L::TILE;
    SPMLA_LDS uint8_t* at = d + (2 * dh) * 4096 + l16 * 128;
    const int x = swz(l16);
    auto kread = [&](int n) -> i32x4 {                    // unit n: positions 16 (n / 4) .., group 2 dh + n / 2 % 2, chunks 4 (n % 2) ..
      return *(SPMLA_LDS i32x4*)(at + (n >> 2) * 2048 + ((n >> 1) & 1) * 4096 + 16 * ((4 * (n & 1) + qt) ^ x));
    };
    auto rread = [&](int u) -> i32x4 {                    // rope of positions 16 u ..: Row576 8 codes, Row656 8 bf16
      if constexpr (R5) {
        const i32x2 y = *(SPMLA_LDS i32x2*)(d + L::CODE + u * 1024 + l16 * 64 + 16 * ((2 * dh + (qt >> 1)) ^ ((l16 >> 2) & 3)) + 8 * (qt & 1));
        return i32x4{y[0], y[1], 0, 0};
      } else {
        return *(SPMLA_LDS i32x4*)(d + L::CODE + u * 2048 + l16 * 128 + 16 * ((4 * dh + qt) ^ x));
      }
    };
    constexpr int AHEAD = R5 ? 3 : 2;
    i32x4 k[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) k[n] = kread(n);
    i32x4 kr;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x4 s[2] = {};
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        f32x4 acc[2] = {}, sc = {};
        if constexpr (!R5) sc = *(SPMLA_LDS f32x4*)(d + L::CODE + L::RP + (2 * dh + g) * 128 + u * 64 + qt * 16);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int n = 4 * u + 2 * g + c;
          const bf16x8 y0 = codes8(k[n % AHEAD][0], k[n % AHEAD][1]), y1 = codes8(k[n % AHEAD][2], k[n % AHEAD][3]);
          if (n + AHEAD < 8) k[n % AHEAD] = kread(n + AHEAD);
          if (n == 4 * u + 2) kr = rread(u);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            f32x4& to = R5 ? s[i] : acc[i];
            to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y0, qf[2 * g + c][0][i], to, 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            f32x4& to = R5 ? s[i] : acc[i];
            to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y1, qf[2 * g + c][1][i], to, 0, 0, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (!R5)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[i][r] = __builtin_fmaf(acc[i][r], sc[r], s[i][r]);
      }
      const bf16x8 y = R5 ? codes8(kr[0], kr[1]) : __builtin_bit_cast(bf16x8, kr);
#pragma unroll
      for (int i = 0; i < 2; ++i) s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y, qpe[i], s[i], 0, 0, 0);
      part[u] = dh ? s[1] : s[0];
      *(SPMLA_LDS f32x4*)(lds + L::X + w * 2048 + u * 1024 + lane * 16) = dh ? s[0] : s[1];
    }
  };

  // softmax of tile j, its P and factors: value 4 u + r of a lane is position 16 u + 4 qt + r
  auto softmax = [&](int j) {
    const int lane = here(), l16 = lane & 15, qt = lane >> 4, qr = 16 * w + l16;
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
    const bool move = __any(mx * p.c > m * p.c + TAU);
    if (move) {
      const float mn = fmaxf(m, mx), a = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((m - mn) * p.c);
      m = mn;
      l *= a;
      far = __any(fabsf(mn * p.c) > FAR && mn > -__builtin_inff());
      if (qt == 0) ((SPMLA_LDS float*)(lds + L::FAC))[qr] = a;
    }
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
    const i32x4 fl = *(SPMLA_LDS i32x4*)(lds + L::FLAG);
    const int any = __builtin_amdgcn_readfirstlane(fl[0] | fl[1] | fl[2] | fl[3]);
    float sc = 0.f;
    if constexpr (!R5) {
      sc = *(SPMLA_LDS float*)(d + L::CODE + L::RP + w * 128 + l32 * 4);
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
    if (any) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float a = 1.f;
        if (fl[2 * i] | fl[2 * i + 1]) {
          a = ((SPMLA_LDS float*)(lds + L::FAC))[32 * i + l32];
          a = fl[2 * i + (l32 >> 4)] ? a : 1.f;
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int r = 0; r < 16; ++r) O[x][i][r] *= a;
      }
    }
    if (__builtin_expect(k0 + TR > least && least < most, 0)) {
      // the mask cuts this tile: codes that are no numbers become 0 in the wave's own group, which only it reads now
      uint32_t odd = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        SPMLA_LDS u32x4* at = (SPMLA_LDS u32x4*)(d + w * 4096 + i * 1024 + lane * 16);
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
    const int vo = w * 4096 + vrow * 128 + 8 * (lane & 1), vs = swz(vrow) ^ ((lane >> 4) & 1);
    auto vread = [&](int n) -> i32x2 {                    // unit n: positions 16 (n / 4) .., dims 32 (n % 4) ..
      return __builtin_amdgcn_ds_read_tr8_b64_v2i32((SPMLA_LDS i32x2*)(d + vo + 16 * (vs ^ (2 * (n & 3))) + (n >> 2) * 2048));
    };
    auto pread = [&](int ks, int i) -> f16x8 {
      return __builtin_bit_cast(f16x8, *(SPMLA_LDS u32x4*)(lds + L::P + (32 * i + l32) * 64 + 16 * ((2 * ks + hh) ^ ((l32 >> 2) & 3))));
    };
    i32x2 t[4] = {vread(0), vread(1), vread(2), vread(3)};
    f16x8 pb[2] = {pread(0, 0), pread(0, 1)};
    u32x4 scp = {};
    if constexpr (!R5) scp = *(SPMLA_LDS u32x4*)(lds + L::SCH + (w * TR + 8 * hh) * 2);
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const i32x2 c = t[n % 4];
      u32x4 v = {lo_f16x2((uint32_t)c[0]), hi_f16x2((uint32_t)c[0]), lo_f16x2((uint32_t)c[1]), hi_f16x2((uint32_t)c[1])};
      if (n + 4 < 8) t[n % 4] = vread(n + 4);
      if constexpr (!R5)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = mul_f16x2(v[e], scp[e]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        O[n & 3][i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v), pb[i], O[n & 3][i], 0, 0, 0);
      if (n == 3) {
        pb[0] = pread(1, 0);
        pb[1] = pread(1, 1);
        if constexpr (!R5) scp = *(SPMLA_LDS u32x4*)(lds + L::SCH + (w * TR + 16 + 8 * hh) * 2);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  if (nt > 0) {
    issue(0, 0);
    if (nt > 1) issue(1, 1);
    if (nt > 2) issue(2, 2);
    if (nt > 2) wait_vm<2 * COPIES>(); else if (nt > 1) wait_vm<COPIES>(); else wait_vm<0>();
    lds_barrier();
    partials(0);
    lds_barrier();
    softmax(0);
    if (nt > 2) wait_vm<COPIES>(); else wait_vm<0>();
    lds_barrier();
  }
  int slot = 0;                                           // of tile j; tiles j + 1 and j + 2 follow
  for (int j = 0; j < nt; ++j) {
    const int s1 = slot == 2 ? 0 : slot + 1;
    // rows of the next IDS positions: looked up 7 tiles before a half ends, written 4 before, copied from 3 before
    const int in = j & (IDS / TR - 1), next = j / (IDS / TR) + 1;
    if (in == IDS / TR - 7 && next * (IDS / TR) < nt) found = look(next);
    if (in == IDS / TR - 4 && next * (IDS / TR) < nt) note(next, found);
    partials(s1);                                         // (behind the last tile: of what lies there, not used)
    values(j, slot);
    lds_barrier();                                        // partials are there; tile j and P are done with
    if (j + 3 < nt) issue(j + 3, slot);
    if (j + 1 < nt) softmax(j + 1);
    if (j + 3 < nt) wait_vm<COPIES>(); else wait_vm<0>();
    lds_barrier();                                        // P and tile j + 2 are there
    slot = s1;
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
  lds_barrier();
  const float back = p.kv_scale;
  float a[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) a[i] = inv[32 * i + l32] * back;
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
    for (int i = 0; i < 2; ++i) lim[i] = limit_of(32 * i + l32 < live ? 32 * i + l32 : live - 1);
    for (int pos = odd_from; pos < ke; ++pos) {
      const int page = btrow[pos / p.bs];
      const long long y = (long long)page * p.stride + pos % p.bs;
      if (page < 0 || y >= p.rows) continue;
      const uint8_t* row = p.cache + y * RB;
      const float sc = R5 ? 1.f : *(const float*)(row + SC_OFF + 4 * w);
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float v = e4m3_to_f32(row[128 * w + 32 * x + 8 * (r >> 2) + 4 * hh + (r & 3)]) * sc * p.kv_scale;
          const float add = fabsf(v) < __builtin_inff() ? 0.f : v;
#pragma unroll
          for (int i = 0; i < 2; ++i) O[x][i][r] += pos < lim[i] ? add : 0.f;
        }
    }
  }
  if (!whole) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (32 * i + l32 >= live) continue;
      float* o = p.opart + (((long long)sp * p.T + t0) * p.H + r0 + 32 * i + l32) * D_LAT + 128 * w + 4 * hh;
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
  static_assert(4 * 32 * 256 <= L::FAC, "the output's rows fit below the factors");
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
      if (32 * i + row < live) {
        const long long r = r0 + 32 * i + row;
        *(u32x4*)(p.out + (t0 + r / p.H) * p.o_st + (r % p.H) * p.o_sh + 128 * w + 8 * l16) =
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
                                const int* start, int B, int T, int H, float sm_scale, float kv_scale, int S, int span, void* out,
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
  const long long tiles = (long long)T * H / chunk::MR + B;
  if (tiles * S > (1ll << 30)) return SPMLA_ELIMIT;
  float* opart = (float*)ws;
  float* lpart = opart ? opart + (long long)T * H * S * D_LAT : nullptr;
  const float sc = sm_scale * kv_scale;
  chunk::Params p{(const uint16_t*)q, q_st, q_sh, (const uint8_t*)cache, rows, stride_rows, block_size, table, t_st, W, seqs, start, B, T,
                  H, S, span, fmaxf((sc < 0.f ? -sc : sc) * 1.4426950408889634f, 1e-30f), kv_scale, sc < 0.f, (int)tiles, (uint16_t*)out, o_st, o_sh, lse,
                  l_st, opart, lpart};
  static DynLds attr[2];
  static Launcher go[2];
  const int r5 = row_bytes == ROW576;
  const void* fn = r5 ? (const void*)chunk::kernel<true> : (const void*)chunk::kernel<false>;
  const int lds = r5 ? chunk::Lds<true>::TOTAL : chunk::Lds<false>::TOTAL;
  if (const int rc = attr[r5].ensure(fn, lds)) return rc;
  hipStream_t s = (hipStream_t)stream;
  if (const int rc = go[r5](fn, dim3((unsigned)((tiles * S + 7) / 8 * 8)), 256, lds, s, p)) return rc;
  if (S == 1) return SPMLA_OK;
  static Launcher join;
  const chunk::MergeParams mp{opart, lpart, start, B, T, H, S, (uint16_t*)out, o_st, o_sh, lse, l_st};
  return join((const void*)chunk::merge_kernel, dim3((unsigned)(((long long)T * H + 3) / 4)), 256, 0, s, mp);
}
