// Attention of new tokens over every cached latent row of their request (one token each, drafts, or a prefill chunk), the
// rows found through the block table.
//
//   token i of the n new ones of a request with L cached rows (the new ones their last) sees the positions x < L - n + i + 1;
//   row of x: page block_table[b][x / bs], its row x % bs; latent_d = code_d * scale[d / 128] (Row576: code_d)
//   s = sm_scale kv_scale (q[:512] . latent + q[512:] . rope),  p = exp(s - m),  o = kv_scale sum p latent / sum p,
//   lse = ln sum exp(s)
//
// One workgroup = a tile of (token, head) rows of one request, token by token, over one split of the positions: whatever the
// number of heads, a cached row is copied once for all of them. A position costs 2 (576 + 512) operations a row: with 128 rows
// 425 to 484 a byte, matrix cores and HBM alike; with fewer HBM, with several tiles of a request the matrix cores.
//   * products: S^T = K Q^T and O^T = V^T P^T, both with a query row in a lane, so that maxima, sums and factors are one
//     register a lane, and the weights that a lane forms are the operand it needs: P never leaves its registers. Codes are exact
//     in bf16 and in fp16, and so is the query but for fp16's range (the wide kernel takes rows out of it times a power of
//     two). (8-bit MFMA would take the codes as they are, the query in two e4m3 parts: its sums are off by 2e-6 of the summed
//     magnitudes, 1.3e-5 at most, against 4e-9 and 1.2e-7 here.) Row656: a group's sum times the rows' fp32 scales; for PV
//     the weight times the group's scale.
//   * roundings: scores, statistics, sums and partial results are fp32; weights (Row656: times a scale, in units that follow the
//     largest scale of the group that the query row has seen) are rounded to fp16, once. (In bf16 they need no care for their
//     range and cost as much, but put as large an error on the output as its own rounding does.)
//   * masked positions take no part: scores of -inf, and where the mask cuts a tile codes and scales that are no numbers
//     become 0 after the scores (a row that sees one has a score that is none); scales that a row does not see do not move its units.
//
// Three kernels by the rows of a request, on average:
//   * `kernel`, up to 64: 8 waves of 16 rows, 2 or 4 of them on the same rows with every second or fourth tile of 32 positions,
//     joined in LDS. A wave converts what it reads. Bound by HBM (48 requests of 16 heads, 364 MB: 98 us = 3.7 TB/s).
//   * `wide_kernel<R5, false>`: 4 waves of 32 rows, 512 registers (O in the 256 accumulation registers, the query in 144 others).
//     A tile's codes are converted to fp16 once for all waves, beside the score products. Bound by the issue of one
//     wave a SIMD: matrix cores busy for 29% (64 requests of 128 heads: 119 us = 540 TFLOP/s). Two waves a SIMD leave 16 rows
//     a wave, each of which converts everything again (267 us).
//   * from 1024 on, `image_kernel` gathers and converts the tiles first, `wide_kernel<R5, true>` copies them as they lie
//     in LDS: no conversions, addresses without tables (1024 tokens of 128 heads over 16384 rows: 3.78 ms = 1200 TFLOP/s, of
//     which the images take 0.01; converted in the kernel 5.3). The clock falls to 1.8 - 2.0
//     GHz with the power, and a form that runs the softmax beside the next tile's score products takes as long.
// Splits leave normalized fp32 partials and their lse in a workspace; a second kernel joins them.
#include "spmla_common.h"
#include "spmla_quant.h"
#include "spmla_rules.h"

namespace spmla {
namespace chunk {

constexpr int TR = 32;                // positions per tile
constexpr int IDS = 256;              // positions whose rows are looked up at a time
constexpr float TAU = 6.0f, UP = 9.0f, FAR = 65536.f;     // the reference maximum moves past 2^TAU; weights are times 2^UP
constexpr float WTAU = 10.0f, WUP = 5.0f;                // of the wide kernel, where moving it costs more (Row656: 9 and 6, see raise)

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

struct Params {
  const uint16_t* q; long long q_st, q_sh;
  const uint8_t* cache; long long rows, stride;            // rows of the cache, rows from a block to the next
  int bs;
  const int* table; long long t_st; int W;
  const int* seqs; const int* start; int B, T, H;
  float c, kv_scale;                                       // |sm_scale kv_scale| log2(e)
  int flip;
  int tiles, slack;                                        // slack: requests may end inside a tile of query rows
  int items, extra;                                        // workgroups that share the positions, those beyond one a tile (0: no splits)
  uint16_t* out; long long o_st, o_sh;
  float* lse; long long l_st;
  float* opart; float* lpart; i32x2* parts;                // [slot][MR][512], [slot][MR]; of a (token, head): first row, splits
  int longest;                                             // positions from here on are not seen
  uint8_t* images; int img_tiles;                          // [request][img_tiles][IMAGE], see image_kernel
};

// ---- which tile of query rows (MR of one request) and which of its splits a workgroup takes.
// Without splits: request b starts at tile start[b] H / MR (+ b where requests may end inside a tile), found by a search of 64
// places a step. With them (B <= PLAN): span is the least number of position tiles, no less than an even share, for which
// splitting every request's positions by it takes at most `extra` workgroups more than one a tile; a request's tiles x splits
// follow the last request's, and so do the places of partial results, which only split tiles have (at most 2 extra).
struct Item {
  int b, tile, sp, splits, span, slot;                     // slot: the tile's first partial result
};
constexpr int PLAN = 256, CUS = 256;
// A split of fewer tiles costs more to join than it saves: one token of 128 heads over 1000 / 16000 rows with two tiles at least
// 27 / 43 us, with four 30 / 40, with eight 39 / 45.
constexpr int LEAST = 3;

template <int MR>
__device__ inline bool find_item(const Params& p, int lane, Item& o) {
  if (p.extra == 0) {
    const int ti = p.tiles - 1 - (int)blockIdx.x;          // (round robin over the XCDs: they get even shares of long requests)
    if (ti < 0) return false;
    int lo = 0, hi = p.B, step;
    do {
      step = (hi - lo + 63) >> 6;
      const int b = lo + lane * step;
      const int n = __popcll(__ballot(b < hi && (long long)p.start[b] * p.H / MR + (p.slack ? b : 0) <= ti));
      lo += (n > 0 ? n - 1 : 0) * step;
      hi = lo + step < hi ? lo + step : hi;
    } while (step > 1);
    const long long tile = ti - (long long)p.start[lo] * p.H / MR - (p.slack ? lo : 0);
    o = Item{lo, (int)tile, 0, 1, 0x7fffffff / TR, 0};
    return tile >= 0;
  }
  if (p.B == 1) {                                         // (the same without sums and search)
    const int a = p.start[0] < 0 ? 0 : p.start[0], z = p.start[1] > p.T ? p.T : p.start[1];
    const int n = z > a ? (int)(((long long)(z - a) * p.H + MR - 1) / MR) : 0, len = p.seqs[0] < p.longest ? p.seqs[0] : p.longest;
    if (n == 0 || n > p.items) return false;
    const int u = len > 0 ? (len + TR - 1) / TR : 1, room = p.extra < p.items - n ? p.extra : p.items - n;
    int c = room / n + 1;
    c = c < (u + LEAST - 1) / LEAST ? c : (u + LEAST - 1) / LEAST;
    const int span = (u + c - 1) / c;
    c = (u + span - 1) / span;
    const int total = n * c, per = (total + 7) >> 3, y = blockIdx.x >> 3, f = y < per ? (int)(blockIdx.x & 7) * per + y : total;
    if (f >= total) return false;
    const int tile = n - 1 - f % n;
    o = Item{0, tile, f / n, c, span, c > 1 ? tile * c : 0};
    return true;
  }
  int n[PLAN / 64], u[PLAN / 64];                          // of request 64 k + lane: tiles of query rows, tiles of positions
  const long long cap = p.longest;
  long long work = 0;
  int top = 1, tiles = 0;
#pragma unroll
  for (int k = 0; k < PLAN / 64; ++k) {
    n[k] = 0;
    u[k] = 1;
    const int b = 64 * k + lane;
    if (b < p.B) {
      const int t0 = p.start[b], t1 = p.start[b + 1], len = p.seqs[b];
      const long long r = (long long)((t1 > p.T ? p.T : t1) - (t0 < 0 ? 0 : t0)) * p.H, x = len < cap ? len : cap;
      n[k] = r > 0 ? (int)((r + MR - 1) / MR) : 0;
      u[k] = x > 0 ? (int)((x + TR - 1) / TR) : 1;
      work += (long long)n[k] * u[k];
      tiles += n[k];
      top = n[k] > 0 && u[k] > top ? u[k] : top;
    }
  }
  // (in two parts: a lane has 4 products of less than 2^42)
  const int wl = wave_total((int)(work & 0xffffff)), wh = wave_total((int)(work >> 24));
  work = ((long long)wh << 24) + wl;
  tiles = wave_total(tiles);
  top = wave_top(top);
  const int extra = p.extra < p.items - tiles ? p.extra : p.items - tiles;     // (fewer tiles where requests fill theirs)
  const long long even = (work + p.items - 1) / p.items, most = extra > 0 ? (work + extra - 1) / extra : top;
  int lo = even < LEAST ? LEAST : even < top ? (int)even : top;
  int hi = lo < most ? (most < top ? (int)most : top) : lo;
  if (hi < lo) hi = lo;
  // more than a round of workgroups, but no more than one of long tiles: one a tile, the long ones first, beats two of halves
  // (1009 tokens in 10 requests, 259 tiles, 251 of them long: 260 us, in the requests' order 322, split 374)
  bool plain = false;
  if (tiles > CUS) {
    int y = 0;
#pragma unroll
    for (int k = 0; k < PLAN / 64; ++k) y += u[k] > top / 2 ? n[k] : 0;
    plain = wave_total(y) <= CUS;
    if (plain) lo = hi = top;
  }
  while (lo < hi) {
    const unsigned mid = (unsigned)(lo + hi) >> 1;
    int e = 0;
#pragma unroll
    for (int k = 0; k < PLAN / 64; ++k)
      if (64 * k < p.B) e += n[k] * (int)(((unsigned)u[k] - 1) / mid);
    e = wave_total(e);
    if (e <= extra) hi = mid; else lo = mid + 1;
  }
  o.span = lo;
  int total = 0, f = -1, slots = 0;
#pragma unroll
  for (int k = 0; k < PLAN / 64; ++k)
    if (64 * k < p.B) total += n[k] * (int)(((unsigned)u[k] - 1) / (unsigned)lo + 1);
  total = wave_total(total);
  // consecutive items on one XCD: they read the same rows
  const int per = (total + 7) >> 3, x = blockIdx.x & 7, y = blockIdx.x >> 3;
  f = plain ? (int)blockIdx.x : y < per ? x * per + y : total;
  if (f >= total) return false;
  o.b = -1;
  for (int turn = plain ? 0 : 1; turn < 2; ++turn)
#pragma unroll
    for (int k = 0; k < PLAN / 64; ++k)
      if (64 * k < p.B && o.b < 0) {
        const int c = (int)(((unsigned)u[k] - 1) / (unsigned)lo + 1);
        const int mine = plain && (u[k] > top / 2) != (turn == 0) ? 0 : n[k] * c, parts = c > 1 ? mine : 0;
        const int end = (int)wave_incl_scan((uint32_t)mine), send = (int)wave_incl_scan((uint32_t)parts);
        const uint64_t hit = __ballot(f < end && f >= end - mine);
        if (hit) {
          const int at = __builtin_ctzll(hit), g = f - __builtin_amdgcn_readlane(end - mine, at), nn = __builtin_amdgcn_readlane(n[k], at);
          o.b = 64 * k + at;
          o.sp = g / nn;
          o.tile = nn - 1 - g % nn;
          o.splits = __builtin_amdgcn_readlane(c, at);
          o.slot = slots + __builtin_amdgcn_readlane(send - parts, at) + o.tile * o.splits;
        } else {
          f -= __builtin_amdgcn_readlane(end, 63);
          slots += __builtin_amdgcn_readlane(send, 63);
        }
      }
  return o.b >= 0;
}

template <bool R5, int PS>
struct Lds {
  static constexpr int MR = 128 / PS;                      // query rows
  static constexpr int RING = PS == 4 ? 8 : 6;
  static constexpr int CODE = 4 * TR * 128;                // codes by scale group, [4][32 rows][128]
  static constexpr int RP = TR * (R5 ? 64 : 128);          // rope
  static constexpr int SC = R5 ? 0 : 4 * TR * 4;           // scales by group, [4][32]
  static constexpr int TILE = CODE + RP + SC;
  static constexpr int ID = RING * TILE;                   // addresses of the rows of two times IDS positions
  static constexpr int OK = ID + 2 * IDS * 8;              // which of a tile's positions have rows, a bit each
  static constexpr int TOTAL = OK + 2 * IDS / 32 * 4;
  static constexpr int JOIN = 4 * rules::CHUNK_JOIN;       // at the end: O of 4 waves, then maxima and sums
  static_assert(TOTAL <= 160 * 1024 && ID % 8 == 0, "one workgroup a compute unit");
  static constexpr int BYTES = TOTAL < JOIN + 2048 ? JOIN + 2048 : TOTAL;
};

__device__ __attribute__((aligned(16))) uint8_t zero_row[ROW656];

__device__ inline float swap16_max(float x) {
  const uint32_t u = f2u(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t a = r[0], b = r[1];
  return fmaxf(u2f(a), u2f(b));
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
// 8 e4m3 codes -> 8 bf16 / f16, exact
__device__ inline bf16x8 codes8_bf16(int a, int b) {
  return __builtin_bit_cast(bf16x8, u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false)),
                                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true)),
                                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false)),
                                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true))});
}
__device__ inline f16x8 codes8_f16(int a, int b) {
  return __builtin_bit_cast(f16x8, u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false)),
                                         __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true)),
                                         __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false)),
                                         __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true))});
}
// place of chunk c (16 bytes) in a row of 128 bytes: c ^ swz(row); 16 rows' chunks c lie in all 64 banks
__device__ inline int swz(int row) { return ((row & 2) << 1) | ((row & 4) >> 2) | ((row & 8) >> 2); }

// ---- Row656: weights times scales in f16's range. A query row's weight times the scale of group g is taken times 2^-e, e following
// the group's largest scale among the positions that the row sees (scale * 2^-e <= 1): per lane four bytes 127 - e, and O
// holds its dims of the group times 2^-e. e starts at LOW: a weight (up to 2^15) times 2^-LOW is finite, so that scales of zero
// give zeros; it moves when a scale passes 2^e, to twice what that takes, so that it moves rarely (64 requests of 128
// heads: 112 us; to just what it takes 122). Rows that see the same positions have the same e; they differ behind a tile that the mask cuts.
constexpr int LOW = -100;
constexpr uint32_t LOWS = 0x01010101u * (127 - LOW);
__device__ inline float down_of(uint32_t ex, int g) { return u2f((ex >> (8 * g) & 255u) << 23); }               // 2^-e of group g
__device__ inline float up_of(uint32_t ex, int g) { return u2f((254u - (ex >> (8 * g) & 255u)) << 23); }
__device__ inline float finite_size(float x) { return fabsf(x) < __builtin_inff() ? fabsf(x) : 0.f; }
// top: per lane the largest scale of each group that its row has come to see. Returns the rows' new bytes, factor: what O's dims of
// a group are to be multiplied by, down: the largest 2^-e of any row in the group of the scales 2 lane, 2 lane + 1.
__device__ inline uint32_t raise(uint32_t ex, const float (&top)[4], int lane, float (&factor)[4], float& down) {
  uint32_t to = 0;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int old = (int)(ex >> (8 * g) & 255u), e = (int)(f2u(top[g]) >> 23) - 125;                  // top * 2^-e < 1 / 2
    int now = 127 - (e < 126 ? e : 126);
    now = now < old ? now : old;
    to |= (uint32_t)now << (8 * g);
    factor[g] = __builtin_amdgcn_ldexpf(1.f, now - old);
    const int most = wave_top(now);
    if (lane >> 4 == g) down = u2f((uint32_t)most << 23);
  }
  return to;
}

// ---- 64 rows or fewer of a request. PV: V^T by the 8-bit transposing read, converted exactly to f16; P in f16 times 2^UP so that
// few weights are f16 subnormals (Row656: P times the scales of the four groups times 2^-e: a product p * scale is off by half
// an f16 step, or 2^-32 of the largest scale of the group that the row has seen). The reference maximum moves only past TAU.
template <bool R5, int PS>
__global__ void __launch_bounds__(512, 2) kernel(Params p) {
  using L = Lds<R5, PS>;
  constexpr int RB = R5 ? ROW576 : ROW656, MR = L::MR;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem_generic[];
  SPMLA_LDS uint8_t* lds = (SPMLA_LDS uint8_t*)smem_generic;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = w / PS, wp = w % PS;                     // the wave's 16 rows; which of PS tiles it takes
  const int l16 = lane & 15, qt = lane >> 4;

  Item it;
  if (!find_item<MR>(p, lane, it)) return;
  const int b = it.b;
  int t0 = p.start[b], t1 = p.start[b + 1];
  const long long r0 = (long long)it.tile * MR;
  t0 = t0 < 0 ? 0 : t0;
  const int past = p.seqs[b] - (t1 - t0);                 // rows before the new ones (all of them, places for them or not)
  t1 = t1 > p.T ? p.T : t1;
  const long long nrows = (long long)(t1 - t0) * p.H;
  if (r0 < 0 || r0 >= nrows) return;
  const int live = nrows - r0 < MR ? (int)(nrows - r0) : MR;               // query rows here
  const long long cap = p.longest;
  auto limit_of = [&](int r) -> int {                                      // positions that row r sees
    const long long x = (long long)past + (r0 + r) / p.H + 1;
    return x < 0 ? 0 : x > cap ? (int)cap : (int)x;
  };
  const int least = limit_of(0), most = limit_of(live - 1);
  const long long first = (long long)it.sp * it.span * TR, last = first + (long long)it.span * TR;
  const int kb = first < most ? (int)first : most;
  const int ke = it.sp + 1 < it.splits && last < most ? (int)last : most;                    // (the last split takes the rest)
  const int nt = (ke - kb + TR - 1) / TR;
  if (p.extra && it.sp == 0 && tid < live)
    p.parts[(long long)t0 * p.H + r0 + tid] = i32x2{it.slot * MR + tid, it.splits};
  if (nt <= 0 && it.sp > 0) {                             // nothing of this split: no weight in the join
    if (tid < live) p.lpart[((long long)it.slot + it.sp) * MR + tid] = -__builtin_inff();
    return;
  }
  const int* btrow = p.table + (long long)b * p.t_st;

  // the lane id, opaque in every step: LDS places made of it are formed again, not kept (and spilled)
  auto here = [&]() -> int {
    int x = lane;
    asm volatile("" : "+v"(x));
    return x;
  };
  // ---- rows of IDS positions: looked up (x beyond ke: none), then their addresses written with a bit per position
  auto look = [&](int part) -> int {
    const int tid = 64 * w + here();
    const int pos = kb + part * IDS + tid;
    if (pos >= ke || tid >= IDS) return -1;
    const int page = btrow[pos / p.bs];
    const long long y = (long long)page * p.stride + pos % p.bs;
    return page >= 0 && y < p.rows ? (int)y : -1;
  };
  auto note = [&](int part, int row) {
    const int lane = here(), tid = 64 * w + lane, l32 = lane & 31;
    if (tid >= IDS) return;
    const int at = (part & 1) * IDS + tid;
    const uint64_t a = (uint64_t)(uintptr_t)p.cache + (uint64_t)(uint32_t)row * RB;
    ((SPMLA_LDS uint64_t*)(lds + L::ID))[at] = row >= 0 ? a : (uint64_t)(uintptr_t)zero_row;
    const uint64_t has = __ballot(row >= 0);
    if (l32 == 0) ((SPMLA_LDS uint32_t*)(lds + L::OK))[at >> 5] = (uint32_t)(has >> (lane & 32));
  };
  int found = look(0);

  // ---- query operands of rows 16 wr ..: B operands of 16x16x32, lane quarter qt the dims 64 n + 16 qt + 8 e .. + 7 (one
  // 16-byte read of codes serves both e); rope (n = 8): Row576 as the codes, Row656 dims 32 e + 8 qt ..
  const int qr = 16 * wr + l16;                           // the query row of this lane
  bf16x8 qf[9][2];
  {
    const long long r = r0 + (qr < live ? qr : live - 1);
    const uint16_t* qp = p.q + (t0 + r / p.H) * p.q_st + (r % p.H) * p.q_sh;
#pragma unroll
    for (int n = 0; n < 9; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int at = n == 8 && !R5 ? D_LAT + 32 * e + 8 * qt : 64 * n + 16 * qt + 8 * e;
        qf[n][e] = *(const bf16x8*)(qp + at);
      }
  }
  note(0, found);
  lds_barrier();

  // ---- copies of a tile: rows 8 i + lane / 8 of a scale group's codes, the chunk whose place is lane % 8 (a wave half of
  // group w % 4), a share of the rope and of the scales (some twice). COPIES instructions a wave whatever the tile.
  constexpr int COPIES = 3;
  auto issue = [&](int j) {
    SPMLA_LDS uint64_t* id = (SPMLA_LDS uint64_t*)(lds + L::ID) + (j * TR & (2 * IDS - 1));
    SPMLA_LDS uint8_t* d = lds + (j % L::RING) * L::TILE;
    const int lane = here(), r = lane >> 3, place = (lane & 7) ^ swz(r), wl = w & 3, half = w >> 2;
    auto copy = [&](int row, uint32_t off, SPMLA_LDS uint8_t* to) { dma16((const void*)(id[row] + off), to); };
#pragma unroll
    for (int n = 0; n < 2; ++n) copy(8 * (n + 2 * half) + r, 128 * wl + 16 * (place ^ (n << 1)), d + wl * 4096 + (n + 2 * half) * 1024);
    if constexpr (R5) {                                   // 16 rows of 64 bytes a copy
      const int rr = 16 * (w & 1) + (lane >> 2);
      copy(rr, D_LAT + 16 * ((lane & 3) ^ ((rr >> 2) & 3)), d + L::CODE + (w & 1) * 1024);
    } else if (half == 0) {
      copy(8 * wl + r, ROPE_OFF + 16 * (place ^ ((wl & 1) << 1)), d + L::CODE + wl * 1024);
    } else {
      dma4((const void*)(id[lane & 31] + (uint32_t)(SC_OFF + 4 * (2 * (w & 1) + (lane >> 5)))), d + L::CODE + L::RP + (w & 1) * 256);
    }
  };

  f32x4 O[32];                                            // O^T: dims 16 n + 4 qt .., query row qr; times 2^-e (Row656)
#pragma unroll
  for (int n = 0; n < 32; ++n) O[n] = f32x4{};
  float m = -__builtin_inff(), l = 0.f;                   // of query row qr (m: as scores are, shared by its four lanes; l: this lane's)
  bool far = false;                                       // a reference is beyond FAR
  uint32_t ex = LOWS;                                     // 127 - e of the four groups
  float down = u2f((uint32_t)(127 - LOW) << 23);          // the largest 2^-e in the group of this lane's two scales
  f32x4 s[2];                                             // scores, then weights: value 4 u + r is position 16 u + 4 qt + r

  auto scores = [&](SPMLA_LDS uint8_t* d) {
    const int lane = here(), l16 = lane & 15, qt = lane >> 4;
    SPMLA_LDS uint8_t* at = d + l16 * 128;
    const int x0 = 16 * (qt ^ swz(l16)), x1 = x0 ^ 64;
    // unit n = 9 u + i: positions 16 u .., dims 64 i .. (i = 8: rope)
    auto kread = [&](int n) -> i32x4 {
      const int u = n / 9, i = n % 9;
      if (i < 8) return *(SPMLA_LDS i32x4*)(at + (i >> 1) * 4096 + u * 2048 + ((i & 1) ? x1 : x0));
      if constexpr (R5) return *(SPMLA_LDS i32x4*)(d + L::CODE + u * 1024 + l16 * 64 + 16 * (qt ^ ((l16 >> 2) & 3)));
      else return *(SPMLA_LDS i32x4*)(d + L::CODE + u * 2048 + l16 * 128 + x0);
    };
    i32x4 k[3] = {kread(0), kread(1), kread(2)};
    f32x4 acc = {};
#pragma unroll
    for (int n = 0; n < 18; ++n) {
      const int u = n / 9, i = n % 9;
      bf16x8 y[2];
      if (i == 8 && !R5) {
        y[0] = __builtin_bit_cast(bf16x8, k[n % 3]);
        y[1] = __builtin_bit_cast(bf16x8, *(SPMLA_LDS i32x4*)(d + L::CODE + u * 2048 + l16 * 128 + x1));
      } else {
        y[0] = codes8_bf16(k[n % 3][0], k[n % 3][1]);
        y[1] = codes8_bf16(k[n % 3][2], k[n % 3][3]);
      }
      if (n + 3 < 18) k[n % 3] = kread(n + 3);
      if (i == 0) s[u] = f32x4{};
      if constexpr (R5) {
#pragma unroll
        for (int e = 0; e < 2; ++e) s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y[e], qf[i][e], s[u], 0, 0, 0);
      } else if (i < 8) {
        if (!(i & 1)) acc = f32x4{};
#pragma unroll
        for (int e = 0; e < 2; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y[e], qf[i][e], acc, 0, 0, 0);
        if (i & 1) {
          const f32x4 sc = *(SPMLA_LDS f32x4*)(d + L::CODE + L::RP + (i >> 1) * 128 + u * 64 + qt * 16);
#pragma unroll
          for (int r = 0; r < 4; ++r) s[u][r] = __builtin_fmaf(acc[r], sc[r], s[u][r]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y[e], qf[8][e], s[u], 0, 0, 0);
      }
    }
  };

  // softmax of tile j: s becomes the weights, O and l follow a moved maximum
  auto softmax = [&](int j) {
    const int lane = here(), qt = lane >> 4, qr = 16 * wr + (lane & 15);
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
    if (__any(mx * p.c > m * p.c + TAU)) {
      const float mn = fmaxf(m, mx), a = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((m - mn) * p.c);
      m = mn;
      l *= a;
#pragma unroll
      for (int n = 0; n < 32; ++n) O[n] *= a;
      far = __any(fabsf(mn * p.c) > FAR && mn > -__builtin_inff());
    }
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
  };

  // O += V^T P^T of tile j
  auto values = [&](SPMLA_LDS uint8_t* d, int j) {
    const int lane = here(), l16 = lane & 15, qt = lane >> 4;
    f16x8 P[R5 ? 1 : 4];
    if constexpr (R5) {
      P[0] = __builtin_bit_cast(f16x8, u32x4{pk_f16(s[0][0], s[0][1]), pk_f16(s[0][2], s[0][3]), pk_f16(s[1][0], s[1][1]),
                                             pk_f16(s[1][2], s[1][3])});
    } else {
      SPMLA_LDS uint8_t* sa = d + L::CODE + L::RP;
      const f32x2 two = *(SPMLA_LDS f32x2*)(sa + lane * 8);                 // the tile's 128 scales
      const float most = fmaxf(finite_size(two[0]), finite_size(two[1]));
      if (__builtin_expect(__any(most * down > 1.f), 0)) {                  // a larger one than before
        float top[4], factor[4];
        if (kb + (j + 1) * TR > least) {                                    // the mask cuts the tile: each row for itself
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            top[g] = 0.f;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const f32x4 x = *(SPMLA_LDS f32x4*)(sa + g * 128 + 64 * u + qt * 16);
#pragma unroll
              for (int r = 0; r < 4; ++r) top[g] = s[u][r] > 0.f ? fmaxf(top[g], finite_size(x[r])) : top[g];
            }
            top[g] = quad_max(top[g]);
          }
        } else {
          float y = most;
#pragma unroll
          for (int x = 8; x; x >>= 1) y = fmaxf(y, __shfl_xor(y, x));
#pragma unroll
          for (int g = 0; g < 4; ++g) top[g] = u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(y), 16 * g));
        }
        ex = raise(ex, top, lane, factor, down);
#pragma unroll
        for (int n = 0; n < 32; ++n) O[n] *= factor[n >> 3];
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {                                         // (weights first: 0 * scale stays 0)
        const f32x4 a = s[0] * down_of(ex, g) * *(SPMLA_LDS f32x4*)(sa + g * 128 + qt * 16);
        const f32x4 b = s[1] * down_of(ex, g) * *(SPMLA_LDS f32x4*)(sa + g * 128 + 64 + qt * 16);
        P[g] = __builtin_bit_cast(f16x8, u32x4{pk_f16(a[0], a[1]), pk_f16(a[2], a[3]), pk_f16(b[0], b[1]), pk_f16(b[2], b[3])});
      }
    }
    // transposing read: lanes 2 i and 2 i + 1 of a quarter supply row i of the k slots 8 qt ..: positions 4 qt + i, 16 + 4 qt + i - 4
    const int i2 = l16 >> 1, vrow = 16 * (i2 >> 2) + 4 * qt + (i2 & 3);
    const int va = vrow * 128 + 16 * swz(vrow) + 8 * (lane & 1);
    auto vread = [&](int n) -> i32x2 {                    // unit n = 4 c + g: dims 128 g + 16 c ..
      return __builtin_amdgcn_ds_read_tr8_b64_v2i32((SPMLA_LDS i32x2*)(d + (n & 3) * 4096 + (va ^ (16 * (n >> 2)))));
    };
    i32x2 t[4] = {vread(0), vread(1), vread(2), vread(3)};
#pragma unroll
    for (int n = 0; n < 32; ++n) {
      const f16x8 v = codes8_f16(t[n & 3][0], t[n & 3][1]);
      if (n + 4 < 32) t[n & 3] = vread(n + 4);
      f32x4& o = O[8 * (n & 3) + (n >> 2)];
      o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, P[R5 ? 0 : n & 3], o, 0, 0, 0);
    }
  };

  // ---- tiles PS at a time
  constexpr int AHEAD = L::RING - PS;                     // tiles copied ahead
  const bool works = 16 * wr < live;
  for (int j = 0; j < AHEAD && j < nt; ++j) issue(j);
#pragma unroll
  for (int n = 0; n < 9; ++n) asm volatile("" : "+v"(qf[n][0]), "+v"(qf[n][1]));       // (the query is there; negated where scores are)
  if (p.flip)
#pragma unroll
    for (int n = 0; n < 9; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) qf[n][e] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, qf[n][e]) ^ 0x80008000u);
  for (int j = 0; j < nt; j += PS) {
    // rows of the next IDS positions: looked up as a part begins, noted at the end of the step, copied from a later one on
    const int in = j & (IDS / TR - 1), next = j / (IDS / TR) + 1;
    // tile j (and j + 1) is there: of the copies after it at most AHEAD - PS tiles' are on their way
    if (j + AHEAD <= nt) wait_vm<(AHEAD - PS) * COPIES>(); else wait_vm<0>();
    lds_barrier();
    const bool more = in == 0 && next * (IDS / TR) < nt;
    if (more) found = look(next);
#pragma unroll
    for (int i = 0; i < PS; ++i)
      if (j + AHEAD + i < nt) issue(j + AHEAD + i);
    const int mine = j + wp;
    SPMLA_LDS uint8_t* d = lds + (mine % L::RING) * L::TILE;
    const bool go = works && mine < nt;
    if (go) scores(d);
    if (__builtin_expect(kb + (j + PS) * TR > least && least < most, 0)) {
      // the mask cuts a tile: codes and scales that are no numbers become 0 once every wave has its scores
      lds_barrier();
      for (int i = 0; i < PS && j + i < nt; ++i) {
        SPMLA_LDS uint8_t* c = lds + ((j + i) % L::RING) * L::TILE;
        const int tid = 64 * w + here();
        for (int at = tid * 16; at < L::CODE; at += 512 * 16) {
          u32x4 y = *(SPMLA_LDS u32x4*)(c + at);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t nan = ((y[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
            y[e] &= ~((nan >> 7) * 255u);
          }
          *(SPMLA_LDS u32x4*)(c + at) = y;
        }
        if (!R5 && tid < 128) {
          SPMLA_LDS float* x = (SPMLA_LDS float*)(c + L::CODE + L::RP) + tid;
          if (!(fabsf(*x) < __builtin_inff())) *x = 0.f;
        }
      }
      lds_barrier();
    }
    if (go) {
      softmax(mine);
      values(d, mine);
    }
    if (more) note(next, found);
  }

  // ---- join of a row's four lanes, and of the waves of its rows
  l = quad_sum(l);
  float up[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) up[g] = R5 ? 1.f : up_of(ex, g);
  bool done = !works;
#pragma unroll
  for (int half = PS / 2; half >= 1; half /= 2) {
    SPMLA_LDS f32x4* oj = (SPMLA_LDS f32x4*)(lds + rules::chunk_join_at(wr, half, wp));
    SPMLA_LDS float* st = (SPMLA_LDS float*)(lds + L::JOIN) + (wr * half + wp % half) * 128;
    lds_barrier();
    if (!done && wp >= half) {
#pragma unroll
      for (int n = 0; n < 32; ++n) oj[n * 64 + lane] = O[n] * up[n >> 3];
      st[lane] = m;
      st[64 + lane] = l;
      done = true;
    }
    lds_barrier();
    if (!done) {
      const float mo = st[lane], lo = st[64 + lane], mn = fmaxf(m, mo);
      const float a = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((m - mn) * p.c);
      const float c = mo == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((mo - mn) * p.c);
      l = (m == -__builtin_inff() ? l : l * a) + (mo == -__builtin_inff() ? lo : lo * c);
#pragma unroll
      for (int n = 0; n < 32; ++n) O[n] = O[n] * (up[n >> 3] * a) + oj[n * 64 + lane] * c;
      m = mn;
#pragma unroll
      for (int g = 0; g < 4; ++g) up[g] = 1.f;
    }
  }
  if (done) return;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const float ln = m == -__builtin_inff() && l == l ? m : m * p.c * 0.69314718055994531f + (__builtin_log2f(l) - UP) * 0.69314718055994531f;
  const bool whole = it.splits == 1;
  const long long r = r0 + qr;
  if (qt == 0 && qr < live) {
    if (!whole) p.lpart[((long long)it.slot + it.sp) * MR + qr] = ln;
    else if (p.lse) p.lse[(t0 + r / p.H) * p.l_st + r % p.H] = ln;
  }
  const float back = inv * p.kv_scale;                    // (the join has taken 2^-e from O)
  if (!whole) {
    float* o = p.opart + (((long long)it.slot + it.sp) * MR + qr) * D_LAT + 4 * qt;
    if (qr < live)
#pragma unroll
      for (int n = 0; n < 32; ++n) *(f32x4*)(o + 16 * n) = O[n] * back;
    return;
  }
  // bf16 rows through LDS, in the place that this wave alone read last: 16 of 1024 bytes, 16-byte chunks permuted by the row
  SPMLA_LDS uint8_t* ob = lds + rules::chunk_rows_at(wr);
#pragma unroll
  for (int n = 0; n < 32; ++n) {
    const f32x4 y = O[n] * back;
    *(SPMLA_LDS i32x2*)(ob + l16 * 1024 + 16 * ((2 * n + (qt >> 1)) ^ l16) + 8 * (qt & 1)) =
        i32x2{(int)pk_bf16(y[0], y[1]), (int)pk_bf16(y[2], y[3])};
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  for (int row = 0; row < 16 && 16 * wr + row < live; ++row) {
    const long long y = r0 + 16 * wr + row;
    *(u32x4*)(p.out + (t0 + y / p.H) * p.o_st + (y % p.H) * p.o_sh + 8 * lane) = *(SPMLA_LDS u32x4*)(ob + row * 1024 + 16 * (lane ^ row));
  }
}

// ---- more than 64 rows of a request: workgroups of 128 rows, 4 waves of 32 rows (one a SIMD, 512 registers). The codes of a
// tile are in fp16 in a tile in LDS that both products read: K by rows, V by the 16-bit transposing read (chunks permuted by the
// row: neither meets in a bank). A step of 32 positions takes 36 + 32 matrix instructions of 32 clocks a wave; what
// else a wave does in it is spread between them, a few instructions each.
template <bool R5>
struct WLds {
  static constexpr int RING = 4;
  static constexpr int CODE = 4 * TR * 128;                // codes by scale group, [4][32 rows][128]
  static constexpr int RP = TR * (R5 ? 64 : 128);          // rope
  static constexpr int SC = R5 ? 0 : 4 * TR * 4;           // scales by group, [4][32]
  static constexpr int TILE = CODE + RP + SC;
  static constexpr int NG = R5 ? 9 : 8;                    // groups of 64 dims in fp16, [NG][32 rows][128 bytes]
  static constexpr int B = RING * TILE;                    // two of them
  static constexpr int ID = B + 2 * NG * 4096;             // addresses of the rows of two times IDS positions
  static constexpr int OK = ID + 2 * IDS * 8;              // which of a tile's positions have rows, a bit each
  static constexpr int PV = OK + 2 * IDS / 32 * 4;         // Row656: each wave's scales of a tile for the second product
  static constexpr int TOTAL = PV + (R5 ? 0 : 4 * 512);
  static_assert(TOTAL <= 160 * 1024 && ID % 8 == 0 && TOTAL >= 4 * 32768, "one workgroup a compute unit");
};

// Where a request has many query rows, a kernel before this one gathers and converts its tiles once for all of them, as they
// lie in LDS: nine groups of 64 dims in fp16 (Row656's rope in bf16, as it is), scales by group [4][32], a word of which
// positions have rows. Bound by the images' bytes (16384 Row576 rows, 28 MB: 11 us).
constexpr int IMG_SC = 9 * 4096, IMG_OK = IMG_SC + 512, IMAGE = IMG_SC + 1024;
struct ILds {
  static constexpr int PV = 4 * IMAGE;                     // (as above)
  static constexpr int TOTAL = PV + 4 * 512;
  static_assert(TOTAL <= 160 * 1024 && TOTAL >= 4 * 32768, "one workgroup a compute unit");
};

template <bool R5>
__global__ void __launch_bounds__(256) image_kernel(Params p) {
  constexpr int RB = R5 ? ROW576 : ROW656;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, b = blockIdx.y, j = blockIdx.x;
  const int len = p.seqs[b] < p.longest ? p.seqs[b] : p.longest;
  if (j * TR >= len) return;
  const int r = tid >> 3, e = tid & 7, pos = j * TR + r;  // 8 threads a row
  const uint8_t* row = zero_row;
  bool has = false;
  if (pos < len) {
    const int page = p.table[(long long)b * p.t_st + pos / p.bs];
    const long long y = (long long)page * p.stride + pos % p.bs;
    has = page >= 0 && y < p.rows;
    if (has) row = p.cache + y * RB;
  }
  uint8_t* img = p.images + ((long long)b * p.img_tiles + j) * IMAGE;
  uint8_t* to = img + r * 128;
  const int x = swz(r);
  i32x4 y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = *(const i32x4*)(row + 128 * i + 16 * e);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int g = 2 * i + (e >> 2), c = 2 * (e & 3);
    *(f16x8*)(to + g * 4096 + 16 * (c ^ x)) = codes8_f16(y[i][0], y[i][1]);
    *(f16x8*)(to + g * 4096 + 16 * ((c ^ x) ^ 1)) = codes8_f16(y[i][2], y[i][3]);
  }
  if constexpr (R5) {
    const i32x2 z = *(const i32x2*)(row + D_LAT + 8 * e);
    *(f16x8*)(to + 8 * 4096 + 16 * (e ^ x)) = codes8_f16(z[0], z[1]);
  } else {
    *(u32x4*)(to + 8 * 4096 + 16 * (e ^ x)) = *(const u32x4*)(row + ROPE_OFF + 16 * e);
    if (e < 4) ((float*)(img + IMG_SC))[e * 32 + r] = *(const float*)(row + SC_OFF + 4 * e);
  }
  const uint64_t bits = __ballot(has && e == 0);          // rows 8 w .. 8 w + 7, a bit each in lanes 8 k
  if (lane == 0) {
    uint32_t y8 = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) y8 |= (uint32_t)(bits >> (8 * k) & 1) << k;
    img[IMG_OK + w] = (uint8_t)y8;
  }
}

typedef short s16x4 __attribute__((ext_vector_type(4)));

// QK products with their sums in VGPRs (the builtin would put them into AGPRs, which O fills). What the compiler cannot see
// inside asm: operands come from LDS or were written long before; a chain's result is read 12 wait states after it.
__device__ inline f32x16 qk_first(u32x4 a, u32x4 b) {
  f32x16 d;
  asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(d) : "v"(a), "v"(b));
  return d;
}
__device__ inline f32x16 qk_next(u32x4 a, u32x4 b, f32x16 c) {
  asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
  return c;
}
__device__ inline f32x16 qk_rope(u32x4 a, u32x4 b, f32x16 c) {             // Row656: in bf16
  asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
  return c;
}
template <bool R5, bool IMG>
__global__ void __launch_bounds__(256, 1) wide_kernel(Params p) {
  using L = WLds<R5>;
  constexpr int RB = R5 ? ROW576 : ROW656, MR = 128;
  constexpr float TAU = R5 ? WTAU : WTAU - 1.f, UP = R5 ? WUP : WUP + 1.f;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem_generic[];
  SPMLA_LDS uint8_t* lds = (SPMLA_LDS uint8_t*)smem_generic;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, l32 = lane & 31, hh = lane >> 5;

  Item it;
  if (!find_item<MR>(p, lane, it)) return;
  const int b = it.b;
  int t0 = p.start[b], t1 = p.start[b + 1];
  const long long r0 = (long long)it.tile * MR;
  t0 = t0 < 0 ? 0 : t0;
  const int past = p.seqs[b] - (t1 - t0);                 // rows before the new ones (all of them, places for them or not)
  t1 = t1 > p.T ? p.T : t1;
  const long long nrows = (long long)(t1 - t0) * p.H;
  if (r0 < 0 || r0 >= nrows) return;
  const int live = nrows - r0 < MR ? (int)(nrows - r0) : MR;
  const long long cap = p.longest;
  auto limit_of = [&](int r) -> int {
    const long long x = (long long)past + (r0 + r) / p.H + 1;
    return x < 0 ? 0 : x > cap ? (int)cap : (int)x;
  };
  const int least = limit_of(0), most = limit_of(live - 1);
  // where the rows of a tile end: an image holds the request's rows behind `most` too (those of its later tokens)
  const int there = !IMG ? most : p.seqs[b] < p.longest ? p.seqs[b] : p.longest;
  const long long first = (long long)it.sp * it.span * TR, last = first + (long long)it.span * TR;
  const int kb = first < most ? (int)first : most;
  const int ke = it.sp + 1 < it.splits && last < most ? (int)last : most;                    // (the last split takes the rest)
  const int nt = (ke - kb + TR - 1) / TR;
  if (p.extra && it.sp == 0 && tid < live)
    p.parts[(long long)t0 * p.H + r0 + tid] = i32x2{it.slot * MR + tid, it.splits};
  if (nt <= 0 && it.sp > 0) {                             // nothing of this split: no weight in the join
    if (tid < live) p.lpart[((long long)it.slot + it.sp) * MR + tid] = -__builtin_inff();
    return;
  }
  const int* btrow = p.table + (long long)b * p.t_st;
  // the lane id, opaque in every step: LDS places made of it are formed again, not kept (the query alone takes 144 registers)
  auto here = [&]() -> int {
    int x = lane;
    asm volatile("" : "+v"(x));
    return x;
  };
  auto look = [&](int part) -> int {
    const int tid = 64 * w + here();
    const int pos = kb + part * IDS + tid;
    if (pos >= ke) return -1;
    const int page = btrow[pos / p.bs];
    const long long y = (long long)page * p.stride + pos % p.bs;
    return page >= 0 && y < p.rows ? (int)y : -1;
  };
  auto note = [&](int part, int row) {
    const int lane = here(), tid = 64 * w + lane, l32 = lane & 31;
    const int at = (part & 1) * IDS + tid;
    const uint64_t a = (uint64_t)(uintptr_t)p.cache + (uint64_t)(uint32_t)row * RB;
    ((SPMLA_LDS uint64_t*)(lds + L::ID))[at] = row >= 0 ? a : (uint64_t)(uintptr_t)zero_row;
    const uint64_t has = __ballot(row >= 0);
    if (l32 == 0) ((SPMLA_LDS uint32_t*)(lds + L::OK))[at >> 5] = (uint32_t)(has >> (lane & 32));
  };

  // ---- query operands of rows 32 w + l32: B operands of 32x32x16, dims 16 ks + 8 hh .. (on their way until the first copies are)
  const int qr = 32 * w + l32;
  u32x4 qf[36];
  int found = IMG ? -1 : look(0);
  {
    const long long r = r0 + (qr < live ? qr : live - 1);
    const uint16_t* qp = p.q + (t0 + r / p.H) * p.q_st + (r % p.H) * p.q_sh;
#pragma unroll
    for (int ks = 0; ks < 36; ++ks) qf[ks] = *(const u32x4*)(qp + 16 * ks + 8 * hh);
  }

  // ---- copies of a tile, in COPIES pieces: wave w the codes of scale group w (piece i: rows 8 i + lane / 8, the chunk whose
  // place is lane % 8), a share of the rope and of the scales. Behind the last tile they copy rows that are there, unused.
  constexpr int COPIES = IMG ? 10 : R5 ? 5 : 6;
  const uint8_t* image = IMG ? p.images + ((long long)b * p.img_tiles) * IMAGE : nullptr;
  auto address = [&](int lane, int j, int i) -> uint64_t { // of the lane's source in piece i
    if constexpr (IMG) {                                  // (pieces 0, 3, 6 and 9; those behind them by the instruction's offset)
      const int t = kb / TR + j < p.img_tiles ? kb / TR + j : p.img_tiles - 1;
      return (uint64_t)(uintptr_t)(image + (long long)t * IMAGE + (i < 9 ? w * 9216 + i * 1024 : IMG_SC + w * 256)) +
             (uint32_t)(lane * (i < 9 ? 16 : 4));
    }
    const int r = lane >> 3, place = (lane & 7) ^ swz(r);
    SPMLA_LDS uint64_t* id = (SPMLA_LDS uint64_t*)(lds + L::ID) + (j * TR & (2 * IDS - 1));
    if (i < 4) return id[8 * i + r] + (uint32_t)(128 * w + 16 * (place ^ ((i & 1) << 1)));
    // Row576: 16 rows of 64 bytes, waves 2 and 3 repeat those of 0 and 1; Row656: 8 rows of rope, 64 scales
    if constexpr (R5) return id[16 * (w & 1) + (lane >> 2)] + (uint32_t)(D_LAT + 16 * (lane & 3));
    if (i == 4) return id[8 * w + r] + (uint32_t)(ROPE_OFF + 16 * (place ^ ((w & 1) << 1)));
    return id[lane & 31] + (uint32_t)(SC_OFF + 4 * (2 * (w & 1) + (lane >> 5)));
  };
  auto copy = [&](int j, int i, uint64_t from) {
    if constexpr (IMG) {
      SPMLA_LDS uint8_t* d = lds + (j & 3) * IMAGE;
      if (i == 9) dma4((const void*)from, d + IMG_SC + w * 256);
      else if (i % 3 == 0) dma16((const void*)from, d + w * 9216 + i * 1024);
      else if (i % 3 == 1) dma16_off<1024, 1024>(from, d + w * 9216 + (i - 1) * 1024);
      else dma16_off<2048, 2048>(from, d + w * 9216 + (i - 2) * 1024);
      return;
    }
    SPMLA_LDS uint8_t* d = lds + (j & 3) * L::TILE;
    if (i < 4) dma16((const void*)from, d + w * 4096 + i * 1024);
    else if (R5) dma16((const void*)from, d + L::CODE + (w & 1) * 1024);
    else if (i == 4) dma16((const void*)from, d + L::CODE + w * 1024);
    else dma4((const void*)from, d + L::CODE + L::RP + (w & 1) * 256);
  };

  // ---- codes of tile j to f16, by half pieces of 8 codes a lane: piece i of the wave's group (row 8 i + lane / 8, 16 codes),
  // piece 4: the rope (Row576, one half)
  auto codes = [&](int lane, int j, int i, int half) -> i32x2 {
    SPMLA_LDS uint8_t* d = lds + (j & 3) * L::TILE;
    return *(SPMLA_LDS i32x2*)(i < 4 ? d + w * 4096 + i * 1024 + lane * 16 + 8 * half : d + L::CODE + w * 512 + lane * 8);
  };
  auto two = [&](u32x4& z, i32x2 y, int e) {              // four codes
    z[2 * e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(y[e], 1.0f, false));
    z[2 * e + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(y[e], 1.0f, true));
  };
  auto put = [&](int lane, int j, int i, int half, u32x4 z) {
    const int r = lane >> 3, x = swz(r);
    SPMLA_LDS uint8_t* to = lds + L::B + (j & 1) * (L::NG * 4096);
    if (i < 4) {
      const int c = (lane & 7) ^ x;
      const int at = (c >> 2) * 4096 + r * 128 + ((16 * ((2 * (c & 3)) ^ x)) ^ ((i & 1) * 96));
      *(SPMLA_LDS u32x4*)(to + w * 8192 + i * 1024 + (at ^ (16 * half))) = z;
    } else {
      *(SPMLA_LDS u32x4*)(to + 8 * 4096 + w * 1024 + r * 128 + 16 * ((lane & 7) ^ swz(8 * w + r))) = z;
    }
  };
  constexpr int PIECES = IMG ? 0 : R5 ? 5 : 4;            // of a tile's conversion

  // ---- softmax state. The reference maximum is the first one that a row meets and moves past 2^TAU over it only (O, which fills
  // the AGPRs, takes 800 instructions to rescale); Row656: O is times 2^-e (see raise).
  f32x16 O[16];                                           // O^T: dims 32 n + 8 a + 4 hh + b, query row qr
  float m = -__builtin_inff(), l;                         // of query row qr (m: as scores are, of both halves; l: this half's)
  float c = p.c;                                          // (per row: the query is times a power of two)
  uint32_t ex = LOWS;
  float down = u2f((uint32_t)(127 - LOW) << 23);          // 2^-e of the two scales of a tile that this lane copies
  bool apart = false;
  SPMLA_LDS uint8_t* copied = lds + (IMG ? ILds::PV : L::PV) + w * 512;
  if constexpr (!IMG) {
    note(0, found);
    note(1, -1);                                          // (addresses that a copy may take, whatever the tile)
  }
  l = 0.f;
#pragma unroll
  for (int n = 0; n < 16; ++n) O[n] = f32x16{};
  lds_barrier();
  for (int j = 0; j < 3; ++j) {
    uint64_t from = 0;
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      if (!IMG || i % 3 == 0) from = address(lane, j, i);
      copy(j, i, from);
    }
  }
#pragma unroll
  for (int ks = 0; ks < 36; ++ks) asm volatile("" : "+v"(qf[ks]));           // (the query is there)
  {
    // The query in f16: its 8 bits are exact there, but for the range: a row whose largest value lies outside of 2^0 .. 2^15 is
    // taken times a power of two. (What is smaller than 2^-14 of f16 is off by 2^-24 then, against a largest one of 1.)
    u16x2 top = {};
#pragma unroll
    for (int ks = 0; ks < 36; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, qf[ks][e] & 0x7fff7fffu));
    int ex = (top[0] > top[1] ? top[0] : top[1]) >> 7;
    const int other = __shfl_xor(ex, 32);
    ex = other > ex ? other : ex;
    const uint32_t turn = p.flip ? 0x80008000u : 0u;       // negated where scores are
    float up = 1.f;
    if (__any((ex < 127 || ex >= 127 + 15) && ex != 255)) {
      int e = ex == 255 || ex == 0 ? 0 : 127 + 10 - ex;    // (subnormal ones as they are)
      e = e > 120 ? 120 : e;
      up = __builtin_amdgcn_ldexpf(1.f, e);
      c = p.c * __builtin_amdgcn_ldexpf(1.f, -e);
    }
#pragma unroll
    for (int ks = 0; ks < 36; ++ks)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = qf[ks][e] ^ turn;
        const float lo = u2f(x << 16) * up, hi = u2f(x & 0xffff0000u) * up;
        qf[ks][e] = ks < 32 || R5 ? pk_f16(lo, hi) : pk_bf16(lo, hi);
      }
  }
  wait_vm<2 * COPIES>();
  lds_barrier();
#pragma unroll
  for (int i = 0; i < (IMG ? 0 : R5 ? 5 : 4); ++i)
#pragma unroll
    for (int half = 0; half < (i < 4 ? 2 : 1); ++half) {
      const i32x2 y = codes(lane, 0, i, half);
      u32x4 z;
      two(z, y, 0);
      two(z, y, 1);
      put(lane, 0, i, half, z);
    }
  // Row656: the second product takes the scales times 2^-e (weights times 2^-e of every group instead: 64 requests of 128 heads 2.4
  // us more). Rows apart, from a tile on that the mask cuts and where e moves: a tile is taken four times (copies and conversions
  // that are repeated leave what is there), each time with the weights times the row's own 2^-e of one group and zeros for the scales of
  // the others. `apart` is the same for all waves: up to that tile they have met the same scales.
  int pass = 0;
#pragma unroll 1
  for (int j = 0; j < nt;) {
    const int in = j & (IDS / TR - 1), next = j / (IDS / TR) + 1;
    wait_vm<(IMG ? 2 : 1) * COPIES>();                    // tile j + 1 (of an image: j) is there
    lds_barrier();                                        // and tile j converted
    if constexpr (!IMG) {
    if (in == 0 && next * (IDS / TR) < nt) found = look(next);
    if (in == 2 && next * (IDS / TR) < nt) note(next, found);
    }
    SPMLA_LDS uint8_t* kt = IMG ? lds + (j & 3) * IMAGE : lds + L::B + (j & 1) * (L::NG * 4096);
    SPMLA_LDS uint8_t* rope = IMG ? kt + 8 * 4096 : R5 ? kt + 8 * 4096 : lds + (j & 3) * L::TILE + L::CODE;
    SPMLA_LDS uint8_t* scales = IMG ? kt + IMG_SC : lds + (j & 3) * L::TILE + L::CODE + L::RP;
    // ---- Row656: the wave's copy of the scales times 2^-e, beside the first products (and again behind them where e moves or the
    // mask cuts the tile)
    bool grows = false;
    auto copy_scales = [&](f32x2 two) {
      *((SPMLA_LDS f32x2*)copied + here()) = two * down;
      asm volatile("" ::: "memory");                       // (the wave's own, in order)
    };
    // ---- S^T = K Q^T; beside it the copies of tile j + 3 and the conversion of tile j + 1, piece by piece
    f32x16 S;
    {
      const int lane = here(), l32 = lane & 31, hh = lane >> 5;
      const int ka = l32 * 128 + 16 * (hh ^ swz(l32));
      auto kread = [&](int ks) -> u32x4 {
        SPMLA_LDS uint8_t* at = ks >= 32 ? rope : kt + (ks >> 2) * 4096;
        return *(SPMLA_LDS u32x4*)(at + (ka ^ (32 * (ks & 3))));
      };
      constexpr int KD = R5 ? 8 : IMG ? 6 : 4;
      u32x4 k[KD];
#pragma unroll
      for (int n = 0; n < KD; ++n) k[n] = kread(n);
      uint64_t from = 0;
      i32x2 y0 = {}, y1 = {};
      u32x4 z = {};
      f32x2 both = {};
      auto beside = [&](int ks) {                         // what runs beside product ks: piece ks / 6 of copies and codes
        if (!R5 && ks == 1) both = *((SPMLA_LDS f32x2*)scales + lane);
        if (!R5 && ks == 7) grows = apart | (__any(fmaxf(finite_size(both[0]), finite_size(both[1])) * down > 1.f) != 0);
        if (!R5 && ks == 8) copy_scales(both);
        if constexpr (IMG) {
          if (ks % 3 == 0 && ks / 3 < COPIES) {
            if (ks / 3 % 3 == 0) from = address(lane, j + 3, ks / 3);
            copy(j + 3, ks / 3, from);
          }
          return;
        }
        // an address and a copy every six products; a piece's codes are read beside six of them and converted beside the next
        // six, four at a time: a conversion takes the VALU for as long as half a product (all 16 beside one: + 1000 cycles a tile)
        const int i = ks / 6, at = ks % 6, q = i - 1;
        if (at == 0 && i < COPIES) from = address(lane, j + 3, i);
        if (at == 3 && i < COPIES) copy(j + 3, i, from);
        if (q >= 0 && q < PIECES) {
          if (at < 2) two(z, y0, at);
          if (at == 2) put(lane, j + 1, q, 0, z);
          if (q < 4 && (at == 3 || at == 4)) two(z, y1, at - 3);
          if (q < 4 && at == 5) put(lane, j + 1, q, 1, z);
        }
        if (at == 2 && i < PIECES) y0 = codes(lane, j + 1, i, 0);
        if (at == 5 && i < PIECES && i < 4) y1 = codes(lane, j + 1, i, 1);
      };
      if constexpr (R5) {
#pragma unroll
        for (int ks = 0; ks < 36; ++ks) {
          S = ks == 0 ? qk_first(k[0], qf[0]) : qk_next(k[ks % KD], qf[ks], S);
          if (ks + KD < 36) k[ks % KD] = kread(ks + KD);
          beside(ks);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
        f32x16 acc[2];
        f32x4 sc[2];
        S = f32x16{};
#pragma unroll
        for (int g = 0; g < 5; ++g) {
          if (g < 4) {
#pragma unroll
            for (int n = 0; n < 8; ++n) {
              const int ks = 8 * g + n;
              acc[g & 1] = n == 0 ? qk_first(k[ks % KD], qf[ks]) : qk_next(k[ks % KD], qf[ks], acc[g & 1]);
              if (ks + KD < 36) k[ks % KD] = kread(ks + KD);
              beside(ks);
              if (g > 0 && n >= 4) {                      // a quarter of the group before: its products are done
                const int a = n - 4;
                asm volatile("" : "+v"(acc[(g - 1) & 1]));
#pragma unroll
                for (int r = 0; r < 4; ++r) S[4 * a + r] = __builtin_fmaf(acc[(g - 1) & 1][4 * a + r], sc[a & 1][r], S[4 * a + r]);
              }
              if (g > 0 && n >= 2 && n < 6) sc[n & 1] = *(SPMLA_LDS f32x4*)(scales + (g - 1) * 128 + 32 * (n - 2) + 16 * hh);
              __builtin_amdgcn_sched_barrier(0);
            }
          } else {
            f32x4 sc[4];
#pragma unroll
            for (int a = 0; a < 4; ++a) sc[a] = *(SPMLA_LDS f32x4*)(scales + 3 * 128 + 32 * a + 16 * hh);
            beside(33);
            asm volatile("s_nop 15" : "+v"(acc[1]));
            beside(34);
#pragma unroll
            for (int r = 0; r < 16; ++r) S[r] = __builtin_fmaf(acc[1][r], sc[r >> 2][r & 3], S[r]);
          }
        }
        asm volatile("s_nop 1" : "+v"(S));                // (written by the VALU just before)
#pragma unroll
        for (int n = 0; n < 4; ++n) S = qk_rope(k[(32 + n) % KD], qf[32 + n], S);
      }
      asm volatile("s_nop 15" : "+v"(S));
    }
    // ---- softmax
    const int lane = here(), l16 = lane & 15, l32 = lane & 31, hh = lane >> 5, qr = 32 * w + l32;
    const uint32_t has = __builtin_amdgcn_readfirstlane(IMG ? *(SPMLA_LDS uint32_t*)(kt + IMG_OK)
                                                            : ((SPMLA_LDS uint32_t*)(lds + L::OK))[j & (2 * IDS / TR - 1)]);
    const int k0 = kb + j * TR;
    if (__builtin_expect(has != 0xffffffffu || k0 + TR > least, 0)) {
      asm volatile("" : "+v"(S));
      const int limit = limit_of(qr < live ? qr : live - 1);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int x = 8 * (r >> 2) + 4 * hh + (r & 3);
        S[r] = (has >> x & 1) && k0 + x < limit ? S[r] : -__builtin_inff();
      }
    }
    if (__builtin_expect(k0 + TR > least && least < there, 0)) {
      // the mask cuts this tile: values that are no numbers become 0 once every wave has its scores
      lds_barrier();
      u32x4 y[8];
      SPMLA_LDS u32x4* at = (SPMLA_LDS u32x4*)(kt + w * 8192) + lane;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = at[64 * i];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          y[i][e] &= ((y[i][e] & 0x7c00u) == 0x7c00u ? 0u : 0xffffu) | ((y[i][e] & 0x7c000000u) == 0x7c000000u ? 0u : 0xffff0000u);
        at[64 * i] = y[i];
      }
      if (!R5 && w == 0) {
        SPMLA_LDS f32x2* x = (SPMLA_LDS f32x2*)scales + lane;
        const f32x2 z = *x;
        *x = f32x2{fabsf(z[0]) < __builtin_inff() ? z[0] : 0.f, fabsf(z[1]) < __builtin_inff() ? z[1] : 0.f};
      }
      lds_barrier();
    }
    float mx = S[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, S[r]);
    mx = swap32_max(mx);
    m = m == -__builtin_inff() ? mx : m;
    float by[4] = {1.f, 1.f, 1.f, 1.f};                     // factors of O's dims of the groups
    bool moved = false;
    const bool cut = k0 + TR > least;
    if (!R5 && __builtin_expect(grows || cut, 0)) {
      const f32x2 two = *((SPMLA_LDS f32x2*)scales + lane);
      if (grows) {
        float top[4];
        if (cut) {                                         // each row for itself
          apart = true;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            top[g] = 0.f;
#pragma unroll
            for (int a = 0; a < 4; ++a) {
              const f32x4 x = *(SPMLA_LDS f32x4*)(scales + g * 128 + 32 * a + 16 * hh);
#pragma unroll
              for (int r = 0; r < 4; ++r) top[g] = S[4 * a + r] > -__builtin_inff() ? fmaxf(top[g], finite_size(x[r])) : top[g];
            }
            top[g] = swap32_max(top[g]);
          }
        } else {
          float y = fmaxf(finite_size(two[0]), finite_size(two[1]));
#pragma unroll
          for (int x = 8; x; x >>= 1) y = fmaxf(y, __shfl_xor(y, x));
#pragma unroll
          for (int g = 0; g < 4; ++g) top[g] = u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(y), 16 * g));
        }
        const uint32_t was = ex;
        ex = raise(ex, top, lane, by, down);
        moved = (j > 0 || pass > 0) && __any(ex != was);   // (before the first products O is zero)
        if (apart) down = lane >> 4 == pass ? 1.f : 0.f;
      }
      copy_scales(two);
    }
    if (__builtin_expect(__any((mx - m) * c > TAU) || moved, 0)) {
      const float mn = fmaxf(m, mx), a = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((m - mn) * c);
      m = mn;
      l *= a;
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        f32x16 y = O[n];
        asm volatile("" : "+v"(y));                        // (one after the other: there are 16 registers for it)
        y *= a * by[n >> 2];
        asm volatile("" : "+v"(y));
        O[n] = y;
      }
    }
    const float base = m == -__builtin_inff() ? 0.f : m, ref = UP - base * c;
    auto total = [&]() {
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += S[r];
      return sum;
    };
    if (__builtin_expect(__any(fabsf(ref) > FAR) || apart, 0)) {           // the rounding of m c would count: differences first
#pragma unroll
      for (int r = 0; r < 16; ++r) S[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[r] - base, c, UP));
      l += pass == 0 ? total() : 0.f;
      if (!R5 && apart) S *= down_of(ex, pass);            // (before the scales: 0 * scale stays 0)
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) S[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[r], c, ref));
      l += total();
    }
    // ---- O^T += V^T P^T
    {
      f16x8 P[R5 ? 1 : 2][2];                            // (Row656: times a group's scales, the next one's beside its products)
      f32x4 sc[2];
      auto half_of = [&](int g, int a, int e) {            // positions 8 a + 4 hh + 2 e, + 1
        float x = S[4 * a + 2 * e], y = S[4 * a + 2 * e + 1];
        if constexpr (!R5) {
          x *= sc[a & 1][2 * e];
          y *= sc[a & 1][2 * e + 1];
        }
        u32x4 u = __builtin_bit_cast(u32x4, P[R5 ? 0 : g & 1][a >> 1]);
        u[2 * (a & 1) + e] = pk_f16(x, y);
        P[R5 ? 0 : g & 1][a >> 1] = __builtin_bit_cast(f16x8, u);
      };
      auto scale_of = [&](int g, int a) { sc[a & 1] = *(SPMLA_LDS f32x4*)(copied + g * 128 + 32 * a + 16 * hh); };
      const int vrow = 4 * hh + (l16 >> 2), vch = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      const int v0 = vrow * 128 + 16 * (vch ^ swz(vrow)) + 8 * (lane & 1);  // (rows 8 on: places ^ 2; the group's other half: ^ 4)
      auto vread = [&](int n) -> f16x8 {                  // unit n = 2 d + ks: dims 32 d + l32, positions 16 ks ..
        SPMLA_LDS uint8_t* at = kt + (n >> 2) * 4096 + (n & 1) * 2048;
        const int c = (n >> 1 & 1) * 64;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SPMLA_LDS s16x4*)(at + (v0 ^ c)));
        const s16x4 e = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SPMLA_LDS s16x4*)(at + 1024 + (v0 ^ c ^ 32)));
        const auto x = __builtin_bit_cast(i32x2, a), y = __builtin_bit_cast(i32x2, e);
        return __builtin_bit_cast(f16x8, i32x4{x[0], x[1], y[0], y[1]});
      };
      constexpr int VD = 6;
      f16x8 v[VD];
#pragma unroll
      for (int n = 0; n < VD; ++n) v[n] = vread(n);
      if (!R5) {
        scale_of(0, 0);
        scale_of(0, 1);
      }
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        half_of(0, a, 0);
        half_of(0, a, 1);
        if (!R5 && a < 3) scale_of(a < 2 ? 0 : 1, a < 2 ? a + 2 : 0);
      }
#pragma unroll
      for (int n = 0; n < 32; ++n) {
        O[n >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[n % VD], P[R5 ? 0 : (n >> 3) & 1][n & 1], O[n >> 1], 0, 0, 0);
        if (n + VD < 32) v[n % VD] = vread(n + VD);
        if (!R5 && n < 24) {
          const int g = n / 8 + 1, e = n % 8;
          half_of(g, e >> 1, e & 1);
          if (e % 2 == 0 && (e < 6 || g < 3)) scale_of(e < 6 ? g : g + 1, e < 6 ? e / 2 + 1 : 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (!R5) pass = apart ? (pass + 1) & 3 : 0;
    j += pass == 0;
  }

  wait_vm<0>();
  lds_barrier();

  // ---- output
  l = swap32_sum(l);
  if (32 * w >= live) return;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const float ln = m == -__builtin_inff() && l == l ? m : m * c * 0.69314718055994531f + (__builtin_log2f(l) - UP) * 0.69314718055994531f;
  const bool whole = it.splits == 1;
  const long long r = r0 + qr;
  if (hh == 0 && qr < live) {
    if (!whole) p.lpart[((long long)it.slot + it.sp) * MR + qr] = ln;
    else if (p.lse) p.lse[(t0 + r / p.H) * p.l_st + r % p.H] = ln;
  }
  float back[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) back[g] = inv * p.kv_scale * (R5 ? 1.f : up_of(ex, g));
  if (!whole) {
    // through LDS, 256 dims of a row at a time: 32 rows of 1024 bytes, 16-byte chunks permuted by the row
    SPMLA_LDS uint8_t* ob = lds + w * 32768;
    float* to = p.opart + (((long long)it.slot + it.sp) * MR + 32 * w) * D_LAT + 4 * lane;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const f32x16& y = O[8 * half + n];
          *(SPMLA_LDS f32x4*)(ob + l32 * 1024 + 16 * ((8 * n + 2 * a + hh) ^ l32)) =
              f32x4{y[4 * a], y[4 * a + 1], y[4 * a + 2], y[4 * a + 3]} * back[2 * half + (n >> 2)];
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      for (int row = 0; row < 32 && 32 * w + row < live; ++row)
        *(f32x4*)(to + (long long)row * D_LAT + 256 * half) = *(SPMLA_LDS f32x4*)(ob + row * 1024 + 16 * (lane ^ row));
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    return;
  }
  SPMLA_LDS uint8_t* ob = lds + w * 32768;                // 32 rows of 1024 bytes, 16-byte chunks permuted by the row
#pragma unroll
  for (int n = 0; n < 16; ++n)
#pragma unroll
    for (int a = 0; a < 4; ++a)
      *(SPMLA_LDS i32x2*)(ob + l32 * 1024 + 16 * ((4 * n + a) ^ l32) + 8 * hh) =
          i32x2{(int)pk_bf16(O[n][4 * a] * back[n >> 2], O[n][4 * a + 1] * back[n >> 2]),
                (int)pk_bf16(O[n][4 * a + 2] * back[n >> 2], O[n][4 * a + 3] * back[n >> 2])};
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  for (int row = 0; row < 32 && 32 * w + row < live; ++row) {
    const long long y = r0 + 32 * w + row;
    *(u32x4*)(p.out + (t0 + y / p.H) * p.o_st + (y % p.H) * p.o_sh + 8 * lane) = *(SPMLA_LDS u32x4*)(ob + row * 1024 + 16 * (lane ^ row));
  }
}

// Joins the splits of (token, head) row r: weights exp(lse_s - max); a split without keys has lse -inf and its partial, which
// was not written, does not count. 8 waves a row, or one (many rows, that have few splits each); 8 dims a lane. Bound by the
// partials' bytes and the chain to them (128 rows of 256 splits, 67 MB: 14 us; with loads that wait for their weights 18).
struct MergeParams {
  const float* opart; const float* lpart; const i32x2* parts; long long rows; int slots;
  const int* start; int B, T, H;
  uint16_t* out; long long o_st, o_sh;
  float* lse; long long l_st;
};
template <int WAVES>                                       // of a row
__global__ void __launch_bounds__(512) merge_kernel(MergeParams p) {
  constexpr int PARTS = 2;                                // 4 dims a lane each
  __shared__ float wgt[8][rules::CHUNK_SPLITS];
  __shared__ f32x4 sums[WAVES == 1 ? 1 : 8][PARTS][64];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long r = WAVES == 1 ? (long long)blockIdx.x * 8 + w : blockIdx.x, t = r / p.H, h = r % p.H;
  if (t >= p.T || t < p.start[0] || t >= p.start[p.B]) return;               // rows of no request stay as they are
  const i32x2 part = p.parts[r];
  const int first = __builtin_amdgcn_readfirstlane(part[0]), n = __builtin_amdgcn_readfirstlane(part[1]);
  if (first < 0 || n < 2 || n > rules::CHUNK_SPLITS || first / p.rows + n > p.slots) return;
  float top = -__builtin_inff();
  for (int s = lane; s < n; s += 64) {
    const float x = p.lpart[first + s * p.rows];
    top = x > top || x != x ? x : top;
  }
#pragma unroll
  for (int x = 32; x; x >>= 1) {
    const float y = __shfl_xor(top, x);
    top = y > top || y != y ? y : top;
  }
  const float ref = top == -__builtin_inff() ? 0.f : top;
  float sum = 0.f;
  for (int s = lane; s < n; s += 64) {                    // (every wave all of them, in memory of its own)
    const float x = p.lpart[first + s * p.rows], y = x == -__builtin_inff() ? 0.f : __expf(x - ref);
    wgt[w][s] = x == -__builtin_inff() ? -1.f : y;
    sum += y;
  }
#pragma unroll
  for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  const float* o = p.opart + (long long)first * D_LAT + 4 * lane;
  f32x4 a[PARTS] = {};
#pragma unroll 8
  for (int s = WAVES == 1 ? 0 : w; s < n; s += WAVES) {
    const float y = wgt[w][s];
    const bool has = !(y < 0.f);                          // (the load does not wait for it: what was not written is there, unused)
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
      const f32x4 v = *(const f32x4*)(o + s * p.rows * D_LAT + 256 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[i][e] = has ? __builtin_fmaf(y, v[e], a[i][e]) : a[i][e];
    }
  }
  if constexpr (WAVES > 1) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) sums[w][i][lane] = a[i];
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int k = 1; k < 8; ++k)
#pragma unroll
      for (int i = 0; i < PARTS; ++i) a[i] += sums[k][i][lane];
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  uint16_t* to = p.out + t * p.o_st + h * p.o_sh + 4 * lane;
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    a[i] *= inv;
    *(i32x2*)(to + 256 * i) = i32x2{(int)pk_bf16(a[i][0], a[i][1]), (int)pk_bf16(a[i][2], a[i][3])};
  }
  if (p.lse && lane == 0) p.lse[t * p.l_st + h] = sum > 0.f || sum != sum ? ref + __logf(sum) : -__builtin_inff();
}

// Requests of 64 (token, head) rows or fewer on average take workgroups of 64 rows, two waves a row sharing the positions (48
// requests of 64 rows, 4000 cached ones on average: 90 us, in tiles of 128 rows 115; of 128 rows 146 against 122); of 32
// or fewer of 32 rows and four (16 rows: 45 us against 55; Row576 alone: of Row656 seven tiles fit into LDS, not the eight).
// Tiles of 64 rows also where contexts are short and one round takes them: more waves, and less to start and to leave (65 tokens of
// 128 heads over up to 300 rows: 37 us against 45; 77 over 600: 52 against 56, over 1000: 70 against 64).
// Tiles are gathered first for requests of 1024 rows and more (16 requests, 2000 cached rows on average: with 256 rows 83 us
// against 73 without, with 512 103 against 100, with 1024 163 against 174), while their images take 4 GiB at most.
struct Shape {
  int rows, slack, images;                                 // images: tiles of each request that are gathered first (0: none)
  long long tiles;
};
static Shape shape_of(int T, int H, int B, int row_bytes, int longest) {
  const long long n = (long long)T * H;
  const bool little = longest <= 20 * TR && n / 64 + (H % 64 ? B : 0) <= CUS;
  const int mr = n <= 32ll * B && row_bytes == ROW576 ? 32 : n <= 64ll * B || little ? 64 : 128, slack = H % mr != 0;
  const long long units = ((long long)longest + TR - 1) / TR;
  const bool images = mr == 128 && n >= 1024ll * B && B < 65536 && units * B * IMAGE <= 4ll << 30;
  return Shape{mr, slack, images ? (int)units : 0, n / mr + (slack ? B : 0)};
}
// splits need a place for each (token, head), and for the partial results of a split tile's rows
static long long part_slots(const Shape& s, int items, int B) {
  const int e = rules::chunk_extra(items - s.tiles, s.slack, B);
  return items < 2 * e ? items : 2 * e;
}

}  // namespace chunk
}  // namespace spmla

using namespace spmla;

extern "C" int spmla_attn_chunk_items(int T, int H, int B, int row_bytes, int longest) {
  if (T <= 0 || H <= 0 || B <= 0 || B > chunk::PLAN || longest <= 2 * chunk::LEAST * chunk::TR) return 0;
  const long long tiles = chunk::shape_of(T, H, B, row_bytes, longest).tiles, full = (tiles + chunk::CUS - 1) / chunk::CUS * chunk::CUS;
  // whole rounds of workgroups, a few beyond one a tile for the longest requests; from four rounds on no tile is split
  return tiles >= 4 * chunk::CUS ? 0 : (int)(full - tiles >= chunk::CUS / 4 ? full : full + chunk::CUS / 4);
}

extern "C" long long spmla_attn_chunk_ws_bytes(int T, int H, int B, int row_bytes, int longest, int items) {
  if (T <= 0 || H <= 0 || B <= 0 || longest <= 0) return 0;
  const chunk::Shape s = chunk::shape_of(T, H, B, row_bytes, longest);
  const long long images = (long long)B * s.images * chunk::IMAGE;
  if (B > chunk::PLAN || items <= s.tiles) return images;
  return images + (long long)T * H * 8 + 16 + chunk::part_slots(s, items, B) * s.rows * (D_LAT + 1) * 4;
}

extern "C" int spmla_attn_chunk(const void* q, long long q_st, long long q_sh, const void* cache, long long rows, int row_bytes,
                                int block_size, long long stride_rows, const int* table, long long t_st, int W, const int* seqs,
                                const int* start, int B, int T, int H, float sm_scale, float kv_scale, int longest, int items, void* out,
                                long long o_st, long long o_sh, float* lse, long long l_st, void* ws, long long ws_bytes, void* stream) {
  if (B < 0 || T < 0 || H < 0 || W < 0 || rows < 0 || block_size <= 0 || stride_rows < block_size || items < 0 || longest < 0 ||
      (row_bytes != ROW656 && row_bytes != ROW576))
    return SPMLA_EARG;
  if (T > MAX_TOKENS || B > MAX_TOKENS || H > 65536 || items > 65536 || rows > 0x7fffffffll || (long long)W * block_size > 0x7fffff00ll)
    return SPMLA_ELIMIT;
  if (B == 0 || T == 0 || H == 0) return SPMLA_OK;
  if (!q || !start || !seqs || !out || (rows && !cache) || (W && !table)) return SPMLA_EARG;
  if (((q_st | q_sh | o_st | o_sh) & 7) || (((uintptr_t)q | (uintptr_t)cache | (uintptr_t)out) & 15) ||
      (((uintptr_t)start | (uintptr_t)seqs | (uintptr_t)table | (uintptr_t)lse) & 3))
    return SPMLA_EALIGN;
  const long long room = (long long)W * block_size;
  if (longest > room) longest = (int)room;
  const chunk::Shape s = chunk::shape_of(T, H, B, row_bytes, longest);
  const int threads = s.rows == 128 ? 256 : 512;
  if (s.tiles * threads >= 1ll << 32) return SPMLA_ELIMIT;   // a grid of 2^32 threads or more is not launched
  const long long need = spmla_attn_chunk_ws_bytes(T, H, B, row_bytes, longest, items);
  const int extra = B <= chunk::PLAN && longest > 0 && items > s.tiles ? (int)(items - s.tiles) : 0;
  if (extra >= rules::CHUNK_SPLITS) return SPMLA_ELIMIT;
  if (need && !ws) return SPMLA_EARG;
  if (need && ((uintptr_t)ws & 15)) return SPMLA_EALIGN;
  if (need && ws_bytes < need) return SPMLA_EARG;
  const long long slots = extra ? chunk::part_slots(s, items, B) : 0;
  uint8_t* images = s.images ? (uint8_t*)ws : nullptr;
  float* opart = extra ? (float*)((uint8_t*)ws + (long long)B * s.images * chunk::IMAGE) : nullptr;
  float* lpart = extra ? opart + slots * s.rows * D_LAT : nullptr;
  i32x2* parts = extra ? (i32x2*)(lpart + slots * s.rows) : nullptr;
  const float sc = sm_scale * kv_scale;
  chunk::Params p{(const uint16_t*)q, q_st, q_sh, (const uint8_t*)cache, rows, stride_rows, block_size, table, t_st, W, seqs, start, B, T,
                  H, fmaxf((sc < 0.f ? -sc : sc) * 1.4426950408889634f, 1e-30f), kv_scale, sc < 0.f, (int)s.tiles, s.slack,
                  extra ? items : 0, extra ? rules::chunk_extra(extra, s.slack, B) : 0, (uint16_t*)out, o_st, o_sh, lse, l_st, opart, lpart, parts,
                  longest, images, s.images};
  static DynLds attr[7];
  static Launcher go[7], first[2];
  const int r5 = row_bytes == ROW576, at = s.rows == 32 ? 6 : s.rows == 64 ? 4 + r5 : 2 * (s.images > 0) + r5;
  const void* fn[7] = {(const void*)chunk::wide_kernel<false, false>, (const void*)chunk::wide_kernel<true, false>,
                       (const void*)chunk::wide_kernel<false, true>, (const void*)chunk::wide_kernel<true, true>,
                       (const void*)chunk::kernel<false, 2>, (const void*)chunk::kernel<true, 2>, (const void*)chunk::kernel<true, 4>};
  const int lds[7] = {chunk::WLds<false>::TOTAL, chunk::WLds<true>::TOTAL, chunk::ILds::TOTAL, chunk::ILds::TOTAL,
                      chunk::Lds<false, 2>::BYTES, chunk::Lds<true, 2>::BYTES, chunk::Lds<true, 4>::BYTES};
  if (const int rc = attr[at].ensure(fn[at], lds[at])) return rc;
  hipStream_t stm = (hipStream_t)stream;
  if (images) {
    const void* f = r5 ? (const void*)chunk::image_kernel<true> : (const void*)chunk::image_kernel<false>;
    if (const int rc = first[r5](f, dim3((unsigned)s.images, (unsigned)B), 256, 0, stm, p)) return rc;
  }
  const long long grid = extra ? (items + 7) / 8 * 8 : s.tiles;
  if (const int rc = go[at](fn[at], dim3((unsigned)grid), threads, lds[at], stm, p)) return rc;
  if (!extra) return SPMLA_OK;
  static Launcher join[2];
  const long long n = (long long)T * H;
  const int many = n >= 2048;                             // (whole call, 8 / 32 requests of 128 rows: 8 waves a row 48 / 86 us, one 56 / 80)
  const chunk::MergeParams mp{opart, lpart, parts, s.rows, (int)slots, start, B, T, H, (uint16_t*)out, o_st, o_sh, lse, l_st};
  const void* f = many ? (const void*)chunk::merge_kernel<1> : (const void*)chunk::merge_kernel<8>;
  return join[many](f, dim3((unsigned)(many ? (n + 7) / 8 : n)), 512, 0, stm, mp);
}
