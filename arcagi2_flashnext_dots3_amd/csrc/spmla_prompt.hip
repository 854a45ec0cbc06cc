// Attention over whole prompts: packed sequences, causal or full, grouped heads.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i),  lse_i = ln sum_j exp(scale q_i . k_j)
//   over the keys j of i's sequence (causal: j <= i); query head h reads key head h / (H / Hk).
//
// One workgroup = 32 NW queries of one sequence and head; NW waves of 32 queries each pass over the keys in tiles of 64.
//   * S^T = K Q^T and O^T = V^T P^T (MFMA 32x32x16): both put a query in a lane (lane % 32), so the maxima, sums and
//     rescale factors are one register a lane, and the P values that a lane forms are the operand it needs: the keys of the
//     k slots of V^T follow the rows of the accumulator, and P never leaves its registers.
//   * K and V tiles are copied to LDS (direct copies, a tile ahead) in groups of 64 columns, 128 bytes a row; a row's
//     16-byte chunks are permuted by its number, so that neither K's reads (32 rows, one chunk) nor V's transposing reads
//     (4 rows, 32 bytes) meet in a bank. Rows behind the sequence and columns behind the head are copied from zeros.
//   * one pass, running maximum and sum in base 2 and 32 bits; the reference maximum moves only when a tile
//     exceeds it by more than TAU (P <= 2^(TAU + UP)), so O is rescaled rarely. Weights are rounded once, to the inputs' type.
//   * masked scores are -inf whatever their values; a masked key's V takes no part either, though 0 * inf is no number:
//     tiles that the mask cuts look at V's exponents, and where one is all ones (rare) the products run with zeros in
//     their place, and the queries that see such a value get it at the end.
//
// Two waves a SIMD (three with heads of 64, one with heads of 256): the matrix products of one run beside the softmax of the
// other. Heads of 128 and 192: 950 - 1140 TFLOP/s on long prompts, the matrix cores busy for half of the time at 2.0 GHz (every
// tile waits for its copies, one tile ahead, and at a barrier); of 64: 860, bound by the VALU (per 64 keys 32 exponentials of 16 clocks and 120 instructions of 4
// against 512 clocks of products); of 256: 775 (one wave a SIMD, O in accumulation registers). Short prompts: the
// launch, the search for the tile, two dependent loads and cold code, 11 us.
#include "spmla_common.h"
#include "spmla_quant.h"
#include <type_traits>

namespace spmla {
namespace prompt {

constexpr int TK = 64;                // keys per tile
constexpr float TAU = 6.0f, FAR = 65536.f;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

struct Params {
  const uint16_t* q; long long q_st, q_sh;
  const uint16_t* k; long long k_st, k_sh;
  const uint16_t* v; long long v_st, v_sh;
  const int* start; int B, T, H, group, D, Dv;
  float c;                            // |scale| log2(e)
  int flip;                           // scale < 0: queries with their signs turned
  int causal, tiles, together;        // together: heads that one XCD takes tile by tile (0: H is no multiple of 8)
  uint16_t* out; long long o_st, o_sh;
  float* lse; long long l_st;
};

__device__ __attribute__((aligned(16))) uint8_t zeros[16];

template <bool BF>
struct Type;
template <>
struct Type<true> {
  static constexpr float UP = 0.f;
  static constexpr uint32_t EXPO = 0x7f807f80u, TOP = 0x00800080u, ONE = 0x3f80u;
  static __device__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ uint32_t pack(float a, float b) { return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b}); }
};
template <>
struct Type<false> {                  // P up to 2^13: small weights stay above fp16's subnormals
  static constexpr float UP = 7.f;
  static constexpr uint32_t EXPO = 0x7c007c00u, TOP = 0x04000400u, ONE = 0x3c00u;
  static __device__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ uint32_t pack(float a, float b) { return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b}); }
};

// place of a row's 16-byte chunk c: c ^ swz(row)
__device__ inline int swz(int row) { return ((row & 2) << 1) | ((row & 4) >> 2) | ((row & 8) >> 2); }

// Tile `rank` (MQ queries) of a head, the longest first: up to SORTED sequences by a search for the level x (causal: tiles of
// index x - 1; full: sequences of x tiles) that the rank falls into, v(x) tiles of a sequence being at levels >= x; more
// sequences from the last to the first, sequence b from tile start[b] / MQ + b (as many tiles lie between two sequences as
// the first one has). With the longest first (17 ragged sequences, 32 heads: 194 -> 172 us) an XCD also takes the tiles of a few
// heads in turn: of one head after the other 4096 tokens of 128 heads took 849 us, of four together 807, of all 16 840.
constexpr int SORTED = 256;

template <int MQ>
__device__ inline bool place(const Params& p, int lane, int rank, int& b, int& q0) {
  if (p.B == 1) {                     // (no search)
    const int a = p.start[0], z = p.start[1], len = (z > p.T ? p.T : z) - (a < 0 ? 0 : a);
    b = 0;
    q0 = ((len + MQ - 1) / MQ - 1 - rank) * MQ;
    return len > 0 && q0 >= 0;
  }
  if (p.B > SORTED) {
    const int ti = p.tiles - 1 - rank;
    int lo = 0, hi = p.B, step;
    if (ti < 0) return false;
    do {                              // the last b whose first tile is no later, 64 places a step
      step = (hi - lo + 63) >> 6;
      const int at = lo + lane * step;
      const int n = __popcll(__ballot(at < hi && p.start[at] / MQ + at <= ti));
      lo += (n > 0 ? n - 1 : 0) * step;
      hi = lo + step < hi ? lo + step : hi;
    } while (step > 1);
    b = lo;
    q0 = (ti - p.start[lo] / MQ - lo) * MQ;
    return q0 >= 0;
  }
  int n[SORTED / 64], top = 0;
#pragma unroll
  for (int k = 0; k < SORTED / 64; ++k) {
    n[k] = 0;
    const int at = 64 * k + lane;
    if (at < p.B) {
      const int s0 = p.start[at], s1 = p.start[at + 1], len = (s1 > p.T ? p.T : s1) - (s0 < 0 ? 0 : s0);
      n[k] = len > 0 ? (len + MQ - 1) / MQ : 0;
    }
    top = n[k] > top ? n[k] : top;
  }
  top = wave_top(top);
  auto from = [&](int x) {            // tiles at levels >= x
    int y = 0;
#pragma unroll
    for (int k = 0; k < SORTED / 64; ++k)
      if (64 * k < p.B) y += n[k] < x ? 0 : p.causal ? n[k] - x + 1 : n[k];
    return wave_total(y);
  };
  int lo = 1, hi = top + 1;             // from(hi) = 0
  if (from(1) <= rank) return false;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (from(mid) > rank) lo = mid; else hi = mid;
  }
  const int g = rank - from(hi), each = p.causal ? 1 : lo;                 // of the level's tiles
  int member = g / each, found = -1;
#pragma unroll
  for (int k = 0; k < SORTED / 64; ++k) {
    const uint64_t has = __ballot(p.causal ? n[k] >= lo : n[k] == lo);
    const int c = __popcll(has);
    if (found < 0 && member < c) {    // its lane: the one with `member` members before it
      const int before = __popcll(has & ((1ull << lane) - 1));
      found = 64 * k + __builtin_ctzll(__ballot((has >> lane & 1) && before == member));
    }
    member -= c;
  }
  if (found < 0) return false;
  b = found;
  q0 = (p.causal ? lo - 1 : g % each) * MQ;
  return true;
}

template <int DK, int DV>
struct Lds {
  static constexpr int K = TK * DK * 2, V = TK * DV * 2, BUF = K + V, TOTAL = 2 * BUF;
};

template <int G, int I = 0>
__device__ inline void copies(uint64_t from, SPMLA_LDS uint8_t* to) {      // a row's chunk of G groups
  if constexpr (I < G) {
    dma16_off<128 * I, 8192 * I>(from, to);
    copies<G, I + 1>(from, to);
  }
}
template <int G>
__device__ inline void copies_up_to(uint64_t from, SPMLA_LDS uint8_t* to, int left) {     // those of `left` columns on, zeros behind
#pragma unroll
  for (int g = 0; g < G; ++g) dma16(64 * g < left ? (const void*)(from + 128 * g) : (const void*)zeros, to + 8192 * g);
}

template <bool BF, int DK, int DV, int NW>
__global__ void __launch_bounds__(64 * NW, DK > 192 ? 1 : 2) kernel(Params p) {
  using E = Type<BF>;
  using L = Lds<DK, DV>;
  constexpr int MQ = 32 * NW, GK = DK / 64, GV = DV / 64;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem_generic[];
  SPMLA_LDS uint8_t* lds = (SPMLA_LDS uint8_t*)smem_generic;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hh = lane >> 5, l32 = lane & 31;

  // ---- work item: head and tile, a head's longest tiles first
  int h, rank;
  if (p.together) {                   // an XCD's heads in groups that read the same or few keys
    const int per = p.H >> 3, y = blockIdx.x >> 3, g = y / (p.together * p.tiles), x = y % (p.together * p.tiles);
    if (g * p.together >= per) return;
    h = (blockIdx.x & 7) * per + g * p.together + x % p.together;
    rank = x / p.together;
  } else {
    h = blockIdx.x % p.H;
    rank = blockIdx.x / p.H;
  }
  int b, q0;
  if (!place<MQ>(p, lane, rank, b, q0)) return;
  int s0 = p.start[b], s1 = p.start[b + 1];
  s0 = s0 < 0 ? 0 : s0;
  s1 = s1 > p.T ? p.T : s1;
  const int len = s1 - s0;
  if (q0 >= len) return;

  const int qw = q0 + 32 * w;                              // the wave's first query
  const int qi = qw + l32;                                 // the lane's
  const bool active = qw < len;
  const uint8_t* kp = (const uint8_t*)(p.k + (long long)s0 * p.k_st + (long long)(h / p.group) * p.k_sh);
  const uint8_t* vp = (const uint8_t*)(p.v + (long long)s0 * p.v_st + (long long)(h / p.group) * p.v_sh);
  const int kend = p.causal && q0 + MQ < len ? q0 + MQ : len;
  const int nt = (kend + TK - 1) / TK;

  // ---- copies: a lane copies from row 8 i + lane / 8 of a group of columns, the chunk whose place is lane % 8. Whole tiles: rows
  // 8 w + lane / 8 (+ 32 with four waves) of every group, one address for them; the last tile's one by one.
  auto issue_some = [&](const uint8_t* base, long long st, int dim, int groups, int k0, int dst) {
#pragma unroll 1
    for (int i = w; i < 8 * groups; i += NW) {             // (wave-uniform)
      const int g = i >> 3, row = (i & 7) * 8 + (lane >> 3);
      const int col = 64 * g + 8 * ((lane & 7) ^ swz(row));
      const uint8_t* src = base + ((long long)(k0 + row) * st + col) * 2;
      dma16(k0 + row < len && col < dim ? (const void*)src : (const void*)zeros, lds + dst + i * 1024);
    }
  };
  constexpr int RS = 8 / NW;
  const int crow = 8 * w + (lane >> 3), cch = 16 * ((lane & 7) ^ swz(crow));
  const uint64_t ksrc = (uint64_t)(uintptr_t)kp + (uint64_t)((long long)crow * p.k_st * 2 + cch);
  const uint64_t vsrc = (uint64_t)(uintptr_t)vp + (uint64_t)((long long)crow * p.v_st * 2 + cch);
  const bool heads = p.D == DK && p.Dv == DV;
  auto issue_tile = [&](int j) {
    const int buf = (j & 1) * L::BUF;
    const bool whole = (j + 1) * TK <= len;
    SPMLA_LDS uint8_t* to = lds + buf + w * 1024;
    if (__builtin_expect(heads && whole, 1)) {
#pragma unroll
      for (int i = 0; i < RS; ++i) copies<GK>(ksrc + (uint64_t)((long long)(j * TK + 32 * i) * p.k_st * 2), to + i * 4096);
#pragma unroll
      for (int i = 0; i < RS; ++i) copies<GV>(vsrc + (uint64_t)((long long)(j * TK + 32 * i) * p.v_st * 2), to + L::K + i * 4096);
    } else if (whole) {
      for (int i = 0; i < RS; ++i) {
        copies_up_to<GK>(ksrc + (uint64_t)((long long)(j * TK + 32 * i) * p.k_st * 2), to + i * 4096, p.D - cch / 2);
        copies_up_to<GV>(vsrc + (uint64_t)((long long)(j * TK + 32 * i) * p.v_st * 2), to + L::K + i * 4096, p.Dv - cch / 2);
      }
    } else {
      issue_some(kp, p.k_st, p.D, GK, j * TK, buf);
      issue_some(vp, p.v_st, p.Dv, GV, j * TK, buf + L::K);
    }
  };
  issue_tile(0);

  // ---- queries: B operands (lane half hh: dims 16 ks + 8 hh ..)
  u32x4 qf[DK / 16];
  {
    const uint16_t* qrow = p.q + (long long)(s0 + (qi < len ? qi : len - 1)) * p.q_st + (long long)h * p.q_sh;
    const uint32_t turn = p.flip ? 0x80008000u : 0u;
#pragma unroll
    for (int ks = 0; ks < DK / 16; ++ks) {
      const int col = 16 * ks + 8 * hh;
      const u32x4 x = *(const u32x4*)(col < p.D ? (const void*)(qrow + col) : (const void*)zeros);
      qf[ks] = x ^ turn;
    }
  }
  f32x16 O[DV / 32];
#pragma unroll
  for (int d = 0; d < DV / 32; ++d) O[d] = f32x16{};
  float m = -__builtin_inff(), l = 0.f;                    // m: as scores are; both of the lane's query, l of its keys
  bool far = false;                                        // a reference is beyond FAR
  int odd_from = 0x7fffffff;                               // first key of the cut tiles with V that is no number

  // ---- LDS places
  int ka[4];                                               // K: chunk 2 (ks % 4) + hh of row l32
#pragma unroll
  for (int i = 0; i < 4; ++i) ka[i] = l32 * 128 + (((2 * i + hh) ^ swz(l32)) * 16);
  const int vrow = 4 * hh + ((lane & 15) >> 2), vch = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  int va[2][2];                                            // V: [half of a group's columns][rows + 8]
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) va[i][e] = (vrow + 8 * e) * 128 + (((4 * i + vch) ^ swz(vrow + 8 * e)) * 16) + 8 * (lane & 1);

  // a tile; CUT: one that the wave's mask may cut (loops of their own, or every tile would pay for the other path's O)
  auto tile = [&](int j, auto cutting) {
    constexpr bool CUT = decltype(cutting)::value;
    wait_vm<0>();
    lds_barrier();                                         // tile j is there, tile j - 1 is done with
    if (j + 1 < nt) issue_tile(j + 1);
    const int k0 = j * TK;
    if (CUT && (!active || (p.causal && k0 > qw + 31))) return;
    SPMLA_LDS uint8_t* kb = lds + (j & 1) * L::BUF;
    SPMLA_LDS uint8_t* vb = kb + L::K;

    f32x16 S[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      S[u] = f32x16{};
#pragma unroll
      for (int ks = 0; ks < DK / 16; ++ks)
        S[u] = E::mfma(*(SPMLA_LDS u32x4*)(kb + ka[ks & 3] + (ks >> 2) * (TK * 128) + u * 4096), qf[ks], S[u]);
    }
    if constexpr (CUT) {
      const int last = p.causal ? (qi < len ? qi : len - 1) : len - 1;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = k0 + 32 * u + 8 * (r >> 2) + 4 * hh + (r & 3);
          S[u][r] = key > last ? -__builtin_inff() : S[u][r];
        }
    }
    float mx = S[0][0];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, S[u][r]);
    mx = swap32_max(mx);
    if (__any(mx * p.c > m * p.c + TAU)) {                 // (also the first tile: m = -inf)
      const float mn = fmaxf(m, mx);
      const float a = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((m - mn) * p.c);
      m = mn;
      far = __any(fabsf(mn * p.c) > FAR && mn > -__builtin_inff());
      l *= a;
#pragma unroll
      for (int d = 0; d < DV / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) O[d][r] *= a;
    }
    const float base = m == -__builtin_inff() ? 0.f : m, ref = E::UP - base * p.c;
    if (__builtin_expect(far, 0)) {                        // the rounding of m c would count: differences first
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[u][r] - base, p.c, E::UP));
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[u][r], p.c, ref));
    }
    u32x4 P[2][2];
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += S[u][r];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) P[u][ks][e] = E::pack(S[u][8 * ks + 2 * e], S[u][8 * ks + 2 * e + 1]);
    }
    l += sum;

    auto vread = [&](int d, int u, int ks) -> u32x4 {      // V^T operand: dims 32 d + lane % 32, the keys of P[u][ks]
      SPMLA_LDS uint8_t* at = vb + (d >> 1) * (TK * 128) + (32 * u + 16 * ks) * 128;
      const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SPMLA_LDS s16x4*)(at + va[d & 1][0]));
      const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((SPMLA_LDS s16x4*)(at + va[d & 1][1]));
      const auto a = __builtin_bit_cast(i32x2, x), c = __builtin_bit_cast(i32x2, y);
      return u32x4{(uint32_t)a[0], (uint32_t)a[1], (uint32_t)c[0], (uint32_t)c[1]};
    };
    if constexpr (CUT) {
      uint32_t odd = 0;
#pragma unroll
      for (int d = 0; d < DV / 32; ++d) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const u32x4 x = vread(d, i >> 1, i & 1);
#pragma unroll
          for (int e = 0; e < 4; ++e) odd |= (x[e] & E::EXPO) + E::TOP;
        }
        asm volatile("" : "+v"(odd)::"memory");            // (the products read V again: kept, it would fill the registers)
      }
      if (__builtin_expect(__any((odd & 0x80008000u) != 0), 0)) {
        odd_from = odd_from < k0 ? odd_from : k0;
#pragma unroll
        for (int d = 0; d < DV / 32; ++d) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            u32x4 x = vread(d, i >> 1, i & 1);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              constexpr uint32_t lo = E::EXPO & 0xffffu, hi = E::EXPO & 0xffff0000u;
              x[e] &= ((x[e] & lo) == lo ? 0u : 0xffffu) | ((x[e] & hi) == hi ? 0u : 0xffff0000u);
            }
            O[d] = E::mfma(x, P[i >> 1][i & 1], O[d]);
          }
          asm volatile("" ::: "memory");
        }
        return;
      }
    }
#pragma unroll
    for (int d = 0; d < DV / 32; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) O[d] = E::mfma(vread(d, i >> 1, i & 1), P[i >> 1][i & 1], O[d]);
  };
  const int full = len / TK, clear = p.causal && (qw + 1) / TK < full ? (qw + 1) / TK : full;
  int j = 0;
  for (; j < nt && j < clear; ++j) tile(j, std::false_type());
  for (; j < nt; ++j) tile(j, std::true_type());

  if (__builtin_expect(odd_from < kend, 0)) {              // those values for the queries that see them
    const int upto = p.causal ? qi : len - 1;              // the last key that the lane's query sees
    for (int key = odd_from; key < kend && (!p.causal || key <= qw + 31); ++key) {
      int width = p.Dv;
      asm volatile("" : "+s"(width));                      // (else the compiler keeps a mask for each column over the tiles)
#pragma unroll
      for (int d = 0; d < DV / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int col = 32 * d + 8 * (r >> 2) + 4 * hh + (r & 3);
          const uint32_t x = col < width ? *(const uint16_t*)(vp + ((long long)key * p.v_st + col) * 2) : 0u;
          const uint32_t ex = E::EXPO & 0xffffu;
          const float bad = (x & 0x7fffu) != ex ? __builtin_nanf("") : x >> 15 ? -__builtin_inff() : __builtin_inff();
          O[d][r] += (x & ex) == ex && key <= upto ? bad : 0.f;
        }
    }
  }

  // ---- output: through LDS (the tiles are done with), a query's values in one row
  l = swap32_sum(l);
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  lds_barrier();
  constexpr int OROW = DV * 2;                             // its chunks permuted by the query
  static_assert(NW * 32 * OROW <= L::TOTAL, "the output's rows fit into the tiles' place");
  if (!active) return;
  SPMLA_LDS uint8_t* ob = lds + w * 32 * OROW;
#pragma unroll
  for (int d = 0; d < DV / 32; ++d)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const uint32_t x = E::pack(O[d][4 * a] * inv, O[d][4 * a + 1] * inv), y = E::pack(O[d][4 * a + 2] * inv, O[d][4 * a + 3] * inv);
      *(SPMLA_LDS i32x2*)(ob + l32 * OROW + ((4 * d + a) ^ (l32 & 7)) * 16 + 8 * hh) = i32x2{(int)x, (int)y};
    }
  if (p.lse && hh == 0 && qi < len)
    p.lse[(long long)(s0 + qi) * p.l_st + h] = m * p.c * 0.69314718055994531f + (__builtin_log2f(l) - E::UP) * 0.69314718055994531f;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // the wave's own rows only
  constexpr int CH = DV / 8;                               // 16-byte chunks a row
  for (int i = lane; i < 32 * CH; i += 64) {
    const int r = i / CH, c = i % CH;
    if (qw + r < len && 8 * c < p.Dv)
      *(u32x4*)(p.out + (long long)(s0 + qw + r) * p.o_st + (long long)h * p.o_sh + 8 * c) =
          *(SPMLA_LDS u32x4*)(ob + r * OROW + (c ^ (r & 7)) * 16);
  }
}

template <bool BF, int DK, int DV, int NW>
int launch(Params& p, hipStream_t s) {
  static DynLds attr;
  static Launcher start;
  const void* fn = (const void*)kernel<BF, DK, DV, NW>;
  constexpr int lds = Lds<DK, DV>::TOTAL;
  p.tiles = p.T / (32 * NW) + p.B;
  const long long n = (long long)p.tiles * p.H;
  if (n * (64 * NW) >= 1ll << 32) return SPMLA_ELIMIT;     // a grid of 2^32 threads or more is not launched
  if (const int rc = attr.ensure(fn, lds)) return rc;
  return start(fn, dim3((unsigned)n), 64 * NW, lds, s, p);
}

// Eight waves read a tile of keys for 256 queries, four for 128: long prompts take eight (4096 tokens, 128 heads of 192 + 128:
// 735 us against 770), short ones and few of them four, whose last tiles hold fewer queries that are none and fill the chip
// (17 prompts of 8003 tokens, 32 heads of 128: 144 us against 163).
template <bool BF>
int go(Params& p, hipStream_t s) {
  const bool wide = (long long)p.T >= 1024ll * p.B && (long long)p.T * p.H >= 256ll * 1024;
  if (p.D <= 64 && p.Dv <= 64) return launch<BF, 64, 64, 4>(p, s);
  if (p.D <= 128 && p.Dv <= 128) return wide ? launch<BF, 128, 128, 8>(p, s) : launch<BF, 128, 128, 4>(p, s);
  if (p.D <= 192 && p.Dv <= 128) return wide ? launch<BF, 192, 128, 8>(p, s) : launch<BF, 192, 128, 4>(p, s);
  return launch<BF, 256, 256, 4>(p, s);
}

}  // namespace prompt
}  // namespace spmla

using namespace spmla;

extern "C" int spmla_attn_prompt(const void* q, long long q_st, long long q_sh, const void* k, long long k_st, long long k_sh,
                                 const void* v, long long v_st, long long v_sh, const int* start, int B, int T, int H, int Hk, int D,
                                 int Dv, float scale, int causal, int dtype, void* out, long long o_st, long long o_sh, float* lse,
                                 long long l_st, void* stream) {
  if (B < 0 || T < 0 || H < 0 || Hk <= 0 || H % Hk || D <= 0 || Dv <= 0 || (dtype != DT_F16 && dtype != DT_BF16)) return SPMLA_EARG;
  if (D > 256 || Dv > 256 || T > MAX_TOKENS || B > MAX_TOKENS) return SPMLA_ELIMIT;
  if (B == 0 || T == 0 || H == 0) return SPMLA_OK;
  if (!q || !k || !v || !start || !out) return SPMLA_EARG;
  if ((D & 7) || (Dv & 7) || ((q_st | q_sh | k_st | k_sh | v_st | v_sh | o_st | o_sh) & 7) ||
      (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) || (((uintptr_t)start | (uintptr_t)lse) & 3))
    return SPMLA_EALIGN;
  prompt::Params p{(const uint16_t*)q, q_st, q_sh, (const uint16_t*)k, k_st, k_sh, (const uint16_t*)v, v_st, v_sh, start, B, T, H,
                   H / Hk, D, Dv, fmaxf((scale < 0.f ? -scale : scale) * 1.4426950408889634f, 1e-30f), scale < 0.f, causal != 0, 0,
                   H % 8 ? 0 : H % 32 == 0 ? 4 : H % 16 == 0 ? 2 : 1,
                   (uint16_t*)out, o_st, o_sh, lse, l_st};
  return dtype == DT_BF16 ? prompt::go<true>(p, (hipStream_t)stream) : prompt::go<false>(p, (hipStream_t)stream);
}
