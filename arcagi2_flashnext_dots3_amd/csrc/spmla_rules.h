// Rules of sizes by which the launchers choose a kernel, and limits and LDS places that both sides share (plain host code).
#pragma once

namespace spmla {
namespace rules {

constexpr int WIDE_ROWS = 2048;       // longest list that the prefill kernel takes

// Whether an attention launch without the split merge takes fwd_kernel (spmla_attn.hip: 128 heads per workgroup) or the
// head-group kernel (spmla_attn_hg.hip: 32 heads per workgroup, any K); both run one workgroup per compute unit, whole
// rounds of 256. Fitted in tenths of a us to graphed launches of both formats with 1 to 64 tiles of 32 rows per list: a
// round of the head-group kernel takes 10.2 + 0.6 per tile, one of fwd_kernel 10 + 2.3 per tile and its first 7 more.
// Measured (us, head-group / fwd_kernel), Row656, K = 2048: H = 128: T = 129 142 / 169, 192 164 / 169, 224 195 / 172, 300
// 253 / 319, 400 345 / 325, 900 759 / 676, 2048 1618 / 1406; T = 1500, H = 32 384 / 874; T = 512, H = 160 523 / 645. Shorter
// lists: H = 128: T = 129, K = 1024 86 / 94, K = 128 39 / 31, T = 300, K = 512 100 / 108, K = 128 65 / 54, T = 400, K = 1024
// 209 / 187; T = 2000, H = 64, K = 128 233 / 184; T = 512, H = 160, K = 256 160 / 144. Row576 lies the same way (H = 128, K =
// 2048: T = 192 147 / 150, 224 176 / 153, 400 316 / 292, 2048 1458 / 1258). Of 546 such points the rule misses two by
// more than 5 % (Row576, K = 128: 8 %).
inline bool attn_wide(int T, int H, int K, int S) {
  const long long tiles = ((K + S - 1) / S + 31) / 32, ts = (long long)T * S;
  const long long r32 = (ts * ((H + 31) / 32) + 255) / 256, r128 = (ts * ((H + 127) / 128) + 255) / 256;
  return 32 * tiles <= WIDE_ROWS && r32 * (102 + 6 * tiles) > 72 + r128 * (100 + 23 * tiles);
}

// Model (us) of a merged launch of s splits over Row656 or Row576 rows: ts = T * ceil(H / 32) workgroups a split; see the
// fit in kernels.py, whose _split_cost this is.
inline double split_cost(long long ts, int K, int s, bool r576) {
  const long long tiles = ((K + s - 1) / s + 31) / 32, wgs = ts * s;
  const double m2 = r576 ? 4.0 : 3.0, m4 = r576 ? 5.0 : 3.6, m8 = r576 ? 7.3 : 6.0;
  const double round = (r576 ? 10.8 : 11.5) + (r576 ? 1.81 : 2.13) * (double)((tiles + 3) / 4);
  return (double)((wgs + 255) / 256) * round + (s == 1 ? 0.0 : s == 2 ? m2 : s <= 4 ? m4 : m8) +
         0.013 * (double)(wgs < 256 ? wgs : 256);
}

// Splits of a merged launch that may take up to S. Up to one round of workgroups as many as are asked for: more are taken
// only where they are faster. us of S splits of 128-head workgroups with f16 partials (the merge before this one) / S
// splits of this kernel / what is chosen, 128 heads: T = 32, K = 2048, S = 8 60 / 79 / 38 (2); T = 64, K = 256, S = 4 34 / 58
// / 18 (1); T = 200, K = 2048, S = 8 279 / 438 / 150 (1).
inline int merged_splits(int T, int H, int K, int S, bool r576) {
  const long long ts = (long long)T * ((H + 31) / 32);
  if (ts * S <= 256) return S;
  if (2 * ts > 256) return 1;
  int best = 1;
  for (int s = 2; s <= S; ++s)
    if (split_cost(ts, K, s, r576) < split_cost(ts, K, best, r576)) best = s;
  return best;
}

// The projection kernels (spmla_linear.hip): tile of tokens x outputs and a model of a launch's us,
// c0 + c1 rounds + c2 rounds kb + c3 wgs kb / 256 + c4 wgs / 256 with kb blocks of 128 k and rounds of 256 workgroups; fitted
// to graphed launches of 486 shapes (T 1 to 8192, N 64 to 24576, K 512 to 16384; operands of three launches ago in the
// caches). The chosen kernel is the fastest or within 5 % of it on 477 of them, 0.2 % slower on average, 11 % at most. Every
// kernel is wanted: without it the chosen ones are 1 to 7 % slower on average and up to 24 to 88 % on a shape. Few tokens
// need not mean few workgroups, nor many tokens large tiles (us): 825 x 80 x 7776 tiles of 16 x 32 11 / 64 x 128 22; 64 x
// 152 x 4560 16 x 16 4.3 / 64 x 16 6.3.
struct LinearKernel { int bm, bn; float c[5]; };
constexpr LinearKernel LINEAR[] = {
    {16, 16, {1.358f, 0.989f, 0.041f, 0.045f, 0.000f}},   // stream_kernel NT1 MT1 NW8 ST4
    {16, 32, {2.377f, 0.000f, 0.079f, 0.040f, 0.053f}},   // stream_kernel NT2 MT1 NW4 ST3
    {32, 32, {2.577f, 0.000f, 0.096f, 0.047f, 0.140f}},   // stream_kernel NT2 MT2 NW4 ST2
    {64, 32, {1.664f, 1.121f, 0.180f, 0.021f, 0.454f}},   // stream_kernel NT2 MT4 NW4 ST2
    {64, 64, {1.921f, 1.572f, 0.269f, 0.000f, 0.937f}},   // stream_kernel NT4 MT4 NW4 ST2
    {64, 128, {2.623f, 0.000f, 0.401f, 0.014f, 1.643f}},   // ring_kernel 64x128 w32x32
    {128, 128, {1.861f, 1.342f, 0.522f, 0.096f, 1.174f}},   // ring_kernel 128x128 w64x32
    {256, 256, {0.795f, 6.197f, 0.986f, 0.780f, 0.502f}},   // big_kernel
};

// The cheapest kernel by the model; -1: none takes so many workgroups.
inline int linear_kernel(int T, int N, int K) {
  const double kb = (K + 127) / 128;
  int best = -1;
  double least = 0.0;
  for (int i = 0; i < (int)(sizeof(LINEAR) / sizeof(LINEAR[0])); ++i) {
    const LinearKernel& k = LINEAR[i];
    const long long wgs = (long long)((T - 1) / k.bm + 1) * ((N - 1) / k.bn + 1);
    if ((wgs + 7) / 8 * 8 >= 1 << 23) continue;        // a grid (whole eights of up to 512 threads) of 2^32 threads or more is
                                                       // not launched
    const double r = (double)((wgs + 255) / 256), w = wgs / 256.0;
    const double t = k.c[0] + k.c[1] * r + k.c[2] * r * kb + k.c[3] * w * kb + k.c[4] * w;
    if (best < 0 || t < least) { best = i; least = t; }
  }
  return best;
}


// LDS places (bytes) at the end of the small-row kernel over all cached rows (spmla_chunk.hip), whose PS waves of the same 16
// query rows (wave w: rows w / PS, share w % PS) are joined two by two and the first of them writes the rows out. In the round
// that leaves `half` of them wave wp takes the 32 KB that wave wp + half left at chunk_join_at(wr, half, wp). Its bf16 rows (16
// KB) go where it alone reads in the last round: no barrier stands between.
constexpr int CHUNK_JOIN = 32768;                        // O of 16 rows of 512 dims in fp32
inline constexpr int chunk_join_at(int wr, int half, int wp) { return (wr * half + wp % half) * CHUNK_JOIN; }
inline constexpr int chunk_rows_at(int wr) { return chunk_join_at(wr, 1, 0); }

// Of spmla_chunk.hip's launches: the most partial results of a (token, head) row that the join takes, and how many workgroups
// beyond one a tile share out the positions, all of which one tile may take: `beyond` of the counted tiles (one less than
// those results at most), and as many more as there are requests where these are counted with a tile too many each.
constexpr int CHUNK_SPLITS = 512;
inline int chunk_extra(long long beyond, int slack, int B) {
  const long long x = beyond + (slack ? B : 0);
  return (int)(x < CHUNK_SPLITS - 1 ? x : CHUNK_SPLITS - 1);
}

}  // namespace rules
}  // namespace spmla
