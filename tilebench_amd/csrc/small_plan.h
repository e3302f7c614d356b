// Which tile a W4A16, scaled fp8 or plain product runs on: host-only C++ (no HIP),
// shared with a CPU check.
//
// A W4A16 product's time is about its K steps times the time of one step of all its
// tiles on 256 CUs.  Measured on MI355X (graph replays, K = 4096, us per K step
// of 64): a 32 x 128 tile takes 0.25, 32 x 256 0.37, 64 x 256 0.42 - 0.56 (one
// tile per CU - many), 256 x 256 0.9 - 1.9 (its MFMAs at the power cap).  Tiles
// that share a CU share its VALU (the dequantisation bounds the small ones), so
// their steps add up; a 256 x 256 tile fills a CU.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace tb {
namespace plan {

enum ExpertTile { TILE_256 = 0, TILE_32x128, TILE_32x256, TILE_64x256 };

// Tiles of `tm` rows for `rows` rows over `active` experts: half a tile of
// padding per expert, at least one tile each.
inline double expert_tile_rows(double rows, double active, double tm) {
  return std::max(active, rows / tm + active / 2);
}

// The tile of a grouped, gate/up (N = 2 I columns of W13) or down product.  The
// host knows the row count only, so at most `rows` experts have a tile and the
// rows are taken as spread over them.  Measured (64 experts, top 8, H = 4096, I =
// 704; gate/up + down us, this tile against 256 x 256): 1 token 23 + 8 (32 x
// 128) against 84 + 18; 24 tokens 48 + 20 (32 x 256) against 164 + 56; 256
// tokens 68 + 33 (64 x 256, 32 x 256) against 166 + 69; 1024 tokens 137 + 74
// (64 x 256) against 191 + 104; 4096 tokens 445 + 265 (64 x 256) against 414 +
// 251: the 256-row tiles stay there.
inline ExpertTile pick_expert_tile(int64_t rows, int64_t experts, int64_t N) {
  const double r = (double)rows, active = (double)std::min(rows, experts);
  const double n128 = (double)((N + 127) / 128), n256 = (double)((N + 255) / 256);
  const double big_n = (double)((N + 127) / 128) / 2;  // a last column tile of <= 128 columns is half a tile
  auto load = [](double tiles) { return std::max(1.0, tiles / 256.0); };
  const double c128 = 0.25 * load(expert_tile_rows(r, active, 32) * n128);
  const double c256 = 0.37 * load(expert_tile_rows(r, active, 32) * n256);
  const double tiles64 = expert_tile_rows(r, active, 64) * n256;
  const double c64 = tiles64 <= 256 ? 0.42 + 0.14 * tiles64 / 256 : 0.56 * tiles64 / 256;
  const double tiles_big = expert_tile_rows(r, active, 256) * big_n;
  const double cbig = tiles_big <= 256 ? 0.9 : std::max(1.8, 1.88 * tiles_big / 256);
  ExpertTile best = TILE_256;
  double c = cbig;
  if (c64 < c) best = TILE_64x256, c = c64;
  if (c256 < c) best = TILE_32x256, c = c256;
  if (c128 < c) best = TILE_32x128, c = c128;
  return best;
}

enum DenseTile { DENSE_256 = 0, DENSE_64x64_K4, DENSE_64x128, DENSE_64x256, DENSE_128x256 };

// us of a K step of `x` tiles per CU, as it was measured: a line over the first
// round of tiles, then a stair per round (a round that is nearly empty costs nearly
// as much as a full one) with a slope for how full the last one is.  `power` is for
// the 256 x 256 tiles, whose clock falls with the share of the chip that multiplies
// (`work`: tiles per CU without their padding).
struct Stairs {
  double first, slope, second, round, fill, power = 0;
  double operator()(double x, double work = 0) const {
    if (x <= 1) return first + slope * x + power * std::max(0.0, work - 0.3);
    const double rounds = std::ceil(x);
    return second + round * (rounds - 2) + fill * (x - (rounds - 1));
  }
};

// The tile of a dense product of more than 16 rows, by the same estimate.  The
// constants are least-squares fits over sizes of 17 - 8192 rows, K and N 64 - 32768 (cold
// weights, each tile forced in turn): within 7 % of nine in ten.  The 256 x 256
// tiles are priced 2 % below their fit, so that a tie goes to them.  Over 5177 sizes the
// picks then took 0.2 % more than the best tile, and two over 3 % more than 256 x 256
// (636 x 28552, K 2368: 102 us against 97).
// Up to 64 rows 64-column tiles of four K groups put a product on every CU that has
// columns for it: 48 rows x 11008 columns 15 us against 25 (64 x 128), 30 (64 x 256)
// and 62 (256 x 256); up to 32 rows the launch halves its rows (12.5 at 32 rows,
// 13.9 on 64).  500 x 4096 (K = 11008): 64 x 128 65 us, 64 x 256 78, 128 x 256 106,
// 256 x 256 160.  Half a round of 256 x 256 tiles beats two rounds and a bit of any
// smaller one: 729 x 12288 (K = 4096) 72 us against 91 (64 x 256), 2391 x 3608 (K =
// 10560) 193 against 247 (128 x 256).
inline DenseTile pick_dense_tile(int64_t M, int64_t N) {
  auto tiles = [&](int64_t tm, int64_t tn) { return (double)((M + tm - 1) / tm * ((N + tn - 1) / tn)) / 256.0; };
  constexpr double steps = 64;  // K = 4096: the start and end of a tile weigh little beside its steps
  constexpr Stairs s64{0.11, 0.20, 0.62, 0.25, 0}, s128{0.30, 0.07, 0.48, 0.33, 0.18},
      s256{0.41, 0.15, 0.82, 0.56, 0.26}, s128x256{0.56, 0.30, 1.49, 1.02, 0.38},
      sbig{0.86, 0.26, 2.40, 1.77, 0.83, 0.72};
  DenseTile best = DENSE_256;
  double c = 0.98 * (6 + steps * sbig(tiles(256, 256), (double)M * (double)N / 65536.0 / 256.0));
  auto take = [&](DenseTile t, double cost) {
    if (cost < c) best = t, c = cost;
  };
  take(DENSE_128x256, 5 + steps * s128x256(tiles(128, 256)));
  take(DENSE_64x256, 4 + steps * s256(tiles(64, 256)));
  take(DENSE_64x128, 4 + steps * s128(tiles(64, 128)));
  if (M <= 64) take(DENSE_64x64_K4, 4 + steps * s64(tiles(64, 64)));
  return best;
}

enum Fp8Tile { FP8_256 = 0, FP8_32x32, FP8_64x64, FP8_64x128, FP8_128x128 };

// The tile of a scaled fp8 product, by estimated time in us (s: steps of 128
// bytes of K, x: tiles per CU; measured with s = 8 - 64).  32 x 32 blocks are
// bound by their CU's loads, 1.5 us + (rows of A and W) x K / 33 KB per us, and
// run in rounds of 256; a step of the LDS tiles takes 0.2 us at 64 x 64, 0.31
// at 64 x 128 (block scales 0.34), 0.36 - 0.5 at 128 x 128 (0.42 - 0.57), and tiles
// that share a CU share its LDS.  A step of 256 x 256 tiles takes 0.9 us on a few
// CUs and 1.55 us on all (1.45 and 1.9).
// Measured, these tiles against 256 x 256 (us): 1 x 8192 x 8192 12 / 65 (32 x 32),
// 64 x 8192 x 8192 15 / 66, 200 x 2112 x 7168 13 / 60 and 14 / 88 (64 x 64), 256 x
// 8192 x 8192 25 / 69 (64 x 128), 512 x 8192 x 8192 35 / 69, 1024 x 4096 x 4096 23 /
// 40, 1024 x 8192 x 8192 60 / 76 (128 x 128); 1348 x 7168 x 4224 56 / 46,
// block scales 4096 x 2112 x 7168 98 (64 x 128) / 92: the 256 x 256 tiles stay.
inline Fp8Tile pick_fp8_tile(int64_t M, int64_t N, int64_t K, bool block_scaled) {
  const double s = (double)K / 128;
  auto tiles = [&](int64_t tm, int64_t tn) { return (double)((M + tm - 1) / tm * ((N + tn - 1) / tn)) / 256.0; };
  auto up = [](double v) { return (double)(int64_t)(v + 0.999999); };
  const double few = block_scaled ? 1.45 : 0.9, all = block_scaled ? 1.9 : 1.55;
  const double big = tiles(256, 256);
  double c = big <= 1 ? 5 + s * (few + (all - few) * big) : (5 + s * all) * big;
  Fp8Tile best = FP8_256;
  auto take = [&](Fp8Tile t, double cost) {
    if (cost < c) best = t, c = cost;
  };
  const double t128 = tiles(128, 128);
  if (t128 <= 1)
    take(FP8_128x128, 3 + s * (block_scaled ? 0.42 + 0.15 * t128 : 0.36 + 0.14 * t128));
  else
    take(FP8_128x128, up(t128 / 2) * (3 + s * (block_scaled ? 1.04 : 0.95)));
  const double t64x128 = up(tiles(64, 128)), t64 = up(tiles(64, 64));
  take(FP8_64x128, 3 * std::max(1.0, t64x128 / 2) + s * (block_scaled ? 0.34 * t64x128 : 0.30 * t64x128 + 0.03));
  take(FP8_64x64, 3 * std::max(1.0, t64 / 2) + s * std::max(0.20, 0.19 * t64));
  take(FP8_32x32, up(tiles(32, 32)) * (1.5 + (double)(std::min<int64_t>(32, M) + 32) * (double)K / 33e3));
  return best;
}

enum NtTile { NT_256 = 0, NT_64x64, NT_64x128, NT_128x128 };

// The tile of a plain product (Kb: bytes of K per operand row), by the same
// estimate: a step of 128 bytes takes 0.2 us at 64 x 64, 0.31 at 64 x 128, 0.36 -
// 0.54 at 128 x 128 (two of them share a CU and step in 0.75 - 1.1, not in twice that)
// and 1.35 - 1.95 at 256 x 256, whose start and end take 4 us more than a small tile's
// (fp16 and fp32; the others within a fifth).  Over 3018 sizes of the four types the picks
// take 0.3 % more than the best tile; without those two terms fp32 3380 x 1192 x 3968 ran
// on 64 x 64 tiles (177 us, 128 x 128 156) and int8 2779 x 3616 x 256 on 256 x 256
// (22.7, 128 x 128 19.6).  Measured fp16 products alone, us: 16 x 4096 x 4096 14.7 (64 x 64;
// 256 x 256 86), 512 x 4096 x 4096 23.4 (64 x 128; 93), 2048 x 2048 x 4096 39 (128 x
// 128; 95), 2601 x 1648 x 2432 30 (128 x 128; 58), 2872 x 3104 x 5504 with its
// transpose 155 (128 x 128; 256 x 256 158), 4096 x 4096 x 4096 129 (256 x 256; 128 x 128 135).
inline NtTile pick_nt_tile(int64_t M, int64_t N, int64_t Kb) {
  const double s = (double)Kb / 128;
  auto tiles = [&](int64_t tm, int64_t tn) { return (double)((M + tm - 1) / tm * ((N + tn - 1) / tn)) / 256.0; };
  auto up = [](double v) { return (double)(int64_t)(v + 0.999999); };
  const double big = tiles(256, 256), t128 = tiles(128, 128), t64x128 = up(tiles(64, 128)), t64 = up(tiles(64, 64));
  double c = 4 + 3 * std::max(1.0, big) + s * (big <= 1 ? 1.35 + 0.2 * big + std::max(0.0, big - 0.6) : 1.95 * big);
  NtTile best = NT_256;
  auto take = [&](NtTile t, double cost) {
    if (cost < c) best = t, c = cost;
  };
  constexpr Stairs s128{0.36, 0.18, 0.75, 0.65, 0.35};
  take(NT_128x128, 3 * std::max(1.0, up(t128) / 2) + s * s128(t128));
  take(NT_64x128, 3 * std::max(1.0, t64x128 / 2) + s * (0.30 * t64x128 + 0.03));
  take(NT_64x64, 3 * std::max(1.0, t64 / 2) + s * std::max(0.2, 0.19 * t64));
  return best;
}

enum MxTile { MX_256 = 0, MX_256_LONG, MX_32x32, MX_32x128, MX_64x64, MX_128x128, MX_128_DEEP, MX_256x128 };

// The tile of an MXFP4 product of M rows, dense (experts = 0) or over `experts` experts, by estimated time in us: a start,
// the K steps of 256 channels times what a step of all tiles takes (or reading the weights, if that takes longer), and a
// share of the weights' MB.  Least-squares fits over 374 sizes (1 - 8192 rows, N 128 - 28672, K 512 - 8192; 8 - 256
// experts with 1 - 16384 rows between them; cold weights, each tile forced in turn), the deep tiles' over another 70, within a
// fifth.  Over profiles/mxfp4_tiles.txt (all tiles as they are, 374 sizes) the picks take 2.2 % (dense) and 1.5 % (experts) more
// than the best tile on average, more than 10 % at 30 sizes; the worst is 192 x 1408 x 8192, 32 x 32 20.8 for 64 x 64 11.7.  Measured, us: 1 x 4096 x 4096 5.8 (32 x 32; 64 x 64 7.4), 16 x
// 11008 x 4096 8.9 (64 x 64; 32 x 32 11.4), 512 x 11008 x 4096 29 (128 x 128; 64 x 64 42, 256 x 256 37), 8192 x 8192 x
// 8192 270 (256 x 256; 128 x 128 337); 64 experts, top 8, N 2816, K 4096: 32 tokens 70 (32 x 128; 64 x 64 75, 32 x 32
// 86), 512 tokens 106 (256 x 256; 32 x 128 128), 4096 tokens 290 (256 x 256; 128 x 128 329).
struct MxCost {
  double start, first, slope, second, round, fill, mb_per_us, us_per_mb;
  double operator()(double tiles, double steps, double mb) const {
    const double x = tiles / 256;
    const double step = x <= 1 ? first + slope * x : second + round * (std::ceil(x) - 2) + fill * (x - std::ceil(x) + 1);
    return start + std::max(steps * step, mb / mb_per_us) + us_per_mb * mb;
  }
};

inline MxTile pick_mx_tile(int64_t M, int64_t N, int64_t K, int64_t experts) {
  const bool grouped = experts > 0;
  // the host knows the rows in all: at most as many experts have some, spread evenly
  const double active = grouped ? (double)std::min(M, experts) : 1, steps = (double)((K + 255) / 256);
  const double mb = active * (double)N * (double)K * 0.53e-6;
  auto tiles = [&](int64_t tm, int64_t tn) {
    return (grouped ? expert_tile_rows((double)M, active, (double)tm) : (double)((M + tm - 1) / tm)) * (double)((N + tn - 1) / tn);
  };
  constexpr MxCost s64[2] = {{3.5, 0.24, 0.06, 0.46, 0.27, 0.18, 6.7, 0.043}, {6.2, 0.13, 0.10, 0.34, 0.44, 0.0, 8.9, 0.072}};
  constexpr MxCost s128[2] = {{3.8, 0.61, 0.45, 1.18, 0.71, 0.39, 4.8, 0.052}, {7.1, 0.78, 0.19, 1.23, 1.17, 0.18, 7.3, 0.0}};
  constexpr MxCost s256[2] = {{9.2, 1.10, 1.02, 3.39, 2.27, 0.94, 3.0, 0.024}, {9.4, 1.11, 0.80, 3.63, 3.41, 0.0, 4.6, 0.0}};
  constexpr MxCost deep[2] = {{5.0, 0.355, 0.30, 0.0, 0.0, 0.0, 6.0, 0.0}, {6.3, 0.33, 0.27, 0.0, 0.0, 0.0, 7.5, 0.06}};
  // fitted to dense products; experts' go by it too
  constexpr MxCost s256x128{7.2, 0.55, 0.56, 0.0, 0.0, 0.0, 6.0, 0.03};
  constexpr MxCost s32x128{4.8, 0.33, 0.08, 0.65, 0.51, 0.06, 9.0, 0.091};
  MxTile best = MX_128x128;
  double c = s128[grouped](tiles(128, 128), steps, mb);
  auto take = [&](MxTile t, double cost) {
    if (cost < c) best = t, c = cost;
  };
  // Two dense 128 x 128 tiles share a CU, and one's stores overlap the other's steps: over two steps that counts for more
  // than fewer reads (us, 128 x 128 and 256 x 256: 8192 x 8192 x 512 43 and 50, 16384 x 8192 x 512 97 and 116, 4096 x 4096 x
  // 512 16 and 16; 8192 x 12288 x 768 74 and 69).  Experts' segments end in halves of the larger tile.
  // 256 x 256 on eight wavefronts, or over more than 16 steps on four: their stalls beside stores and starts weigh less there
  // than the larger fragments' fewer reads (us, eight and four, operands from HBM: 32768 x 4096 x 1408 187 and 196, 8192 x
  // 8192 x 4096 153 and 159, 4096 x 28672 x 4096 272 and 278; 4096 x 8192 x 8192 143 and 141.5, 8192 x 8192 x 8192 275 and 269).
  if (grouped || steps > 2) take(grouped || steps <= 16 ? MX_256 : MX_256_LONG, s256[grouped](tiles(256, 256), steps, mb));
  // 128 x 128 tiles that have a CU each (experts': at most that many): its LDS holds four stages instead of two (us, four and
  // two: 2000 x 2000 x 8192 27 and 36, 1000 x 4000 x 4096 15.4 and 20.5, 1024 x 1024 x 1024 6.6 and 6.7, 8 experts of 2048
  // rows in all, 1024 x 4096 14.8 and 16.9; with two tiles a CU 73 and 47, 8192 x 8192 x 512)
  auto one_each = [&](int64_t tm, int64_t tn) {
    return (grouped ? M / tm + std::min(M, experts) : (M + tm - 1) / tm) * ((N + tn - 1) / tn) <= 256;
  };
  if (one_each(128, 128)) take(MX_128_DEEP, deep[grouped](tiles(128, 128), steps, mb));
  // ... 256 x 128 with a CU each: three stages (us, 256 x 128 and 128 x 128: 2048 x 4096 x 8192 45 and 51, 512 x 11008 x
  // 4096 23.4 and 28.3, 2048 x 4096 x 2048 16.3 and 15.9, x 1024 12.6 and 12.2, 8 experts of 2048 rows in all, 2000 x 4096 23.5 and 27.4)
  if (one_each(256, 128) && steps > 4) take(MX_256x128, s256x128(tiles(256, 128), steps, mb));
  take(MX_64x64, s64[grouped](tiles(64, 64), steps, mb));
  if (grouped) take(MX_32x128, s32x128(tiles(32, 128), steps, mb));
  // blocks of 32 x 32 share CUs: their loads add up
  const double x = tiles(32, 32) / 256, full = std::min(1.0, (double)M / active / 32);
  take(MX_32x32, grouped ? 4.4 + std::max(steps * (0.20 * std::max(1.0, x) + 0.02 * std::max(0.0, x - 0.95) * (1 + 0.24 * full * 32)), mb / 5.0) + 0.042 * mb
                         : 2.4 + std::max(steps * 0.223 * std::max(1.0, x), mb / 4.4) + 0.053 * mb);
  return best;
}

constexpr int DEC_WAVES = 8, DEC_UNIT = 32, DEC_MAX_SPLITS = 16;
struct DecodePlan {
  int cols;       // columns of a slab, 128 or 256
  int64_t slabs;
  int splits;     // blocks that share a slab's K
};

// Slab width and K splits of the W4A16 decode kernel by an estimate of its time
// (us at M = 16): a wavefront takes its 32-row units one after the other, 0.75
// each at 128 columns and 1.45 at 256 (there a CU's stream binds: the mean share
// counts, not the longest; K 4096, N 12288 from cold 14.1 on 192 CUs, 13.4 on 240); a
// split costs an exchange of partials (1.5 or 3.6) that grows with the blocks taking
// part (0.55 or 0.6 each); and 128-column slabs, which read half lines, lose 0.09 per
// MB of weights and 0.2 more per MB above 23.  Fitted to 420 sizes, each with weights
// that stay in the last-level cache, that rotate through HBM, and that follow a fill of
// the cache with written lines: the picks take 0.2 - 0.3 % more than the better width, and 8
// of 2520 take over 3 % more than the 256-column kernel that was here before (worst 1 x
// 7184, K 6656, after a fill: 16.8 us against 15.3).  Measured, 128 / 256 columns at
// their best splits: K 4096, N 4096
// 7.8 / 11.4; K 4096, N 11008 11.9 / 12.5; K 4096, N 12288 14.4 / 12.9; K 8192, N
// 28672 43.1 / 32.6.  Splits at 128
// columns, K 4096, N 4096: 1 13.1, 2 9.7, 4 7.8, 8 8.5; K 1024, N 12288: 1 6.0, 2 6.7.
// A split grid never has more blocks than CUs, counted as they are launched: pairs of
// 128-column slabs go to the 8 XCDs in turn, and a block fills a CU, so a pair too many on
// one XCD would start its blocks a whole block's time later (9 x 6528, K 9920, five splits
// of 51 slabs, 34 blocks on an XCD of 32 CUs: 19.6 us; 256-column slabs 16.1, bounded 14.2).
inline int64_t decode_grid(int cols, int64_t slabs, int splits) {
  return cols == 128 ? ((slabs + 1) / 2 * splits + 7) / 8 * 16 : slabs * splits;
}

inline DecodePlan pick_decode(int64_t N, int64_t K, int cus) {
  const int64_t units = K / DEC_UNIT;
  const double mb = 0.5e-6 * (double)N * (double)K;  // of weights
  DecodePlan best{128, (N + 127) / 128, 1};
  double c = -1;
  for (int cols = 128; cols <= (N <= 128 ? 128 : 256); cols += 128) {  // the wide slab needs 16 columns
    const bool wide = cols == 256;
    const int64_t slabs = (N + cols - 1) / cols;
    for (int s = 1; s <= DEC_MAX_SPLITS && (s == 1 || (decode_grid(cols, slabs, s) <= cus && (int64_t)s * DEC_WAVES <= units)); ++s) {
      const double rounds = (double)((slabs * s + cus - 1) / cus), share = (double)units / (s * DEC_WAVES);
      double cost = wide ? rounds * std::max(1.0, share) * 1.45
                         : rounds * (double)(int64_t)(share + 0.999999) * 0.75 + 0.09 * mb + 0.2 * std::max(0.0, mb - 23);
      if (s > 1) cost += wide ? 3.6 + 0.6 * s : 2.1 + 0.55 * s;
      if (c < 0 || cost < c) best = DecodePlan{cols, slabs, s}, c = cost;
    }
  }
  return best;
}

}  // namespace plan
}  // namespace tb
