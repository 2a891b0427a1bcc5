// Host side of products.hpp: which kernel a product runs on.  Each element type is instantiated in a
// source file of its own (products_f32.hip, products_bf16.hip, ...), which compile side by side.
#pragma once
#include <algorithm>
#include <cmath>

#include "products.hpp"

namespace soapmi {

using WideTile = ProductTile<256, 256, 2, 4, 2, 1>;
using MidTile = ProductTile<128, 128, 2, 4, 4, 3>;
using LowTile = ProductTile<32, 128, 1, 4, 4, 3>;
using SmallTile = ProductTile<32, 64, 2, 2, 4, 3>;  // fp32 rows straight from memory only

// Workgroups for `tiles` tiles, dealt to the 8 XCDs.
inline int64_t workgroups_of(int64_t tiles) { return 8 * ceil_div64(tiles, 8); }
// A launch has fewer than 2^32 threads.
inline bool fits_launch(int64_t tiles, int threads) { return workgroups_of(tiles) * threads < (int64_t)1 << 32; }

inline int grid_of(int64_t tiles, int threads, unsigned* grid) {
  SOAPMI_REQUIRE(fits_launch(tiles, threads), "the product has too many tiles for one launch");
  *grid = (unsigned)workgroups_of(tiles);
  return kOk;
}

// Row tiles that any split of `tokens` rows over the groups can need.
inline int64_t most_row_tiles(const RowGroups& g, int br) {
  return g.tokens / br + std::min<int64_t>((int64_t)g.experts + g.rest, g.tokens);
}

// Tiles of a launch.
template <class Cfg>
int64_t row_tiles(const RowProblem& p) {
  return most_row_tiles(p.groups, Cfg::BR) * ceil_div64(p.cols, Cfg::BC);
}

template <class E, Layout LC, Source S, class Cfg>
int launch_rows(hipStream_t stream, RowProblem p) {
  p.tiles_c = (int)ceil_div64(p.cols, Cfg::BC);
  unsigned grid;
  if (int rc = grid_of(row_tiles<Cfg>(p), Cfg::NT, &grid)) return rc;
  hipLaunchKernelGGL((row_product_kernel<E, LC, S, Cfg>), dim3(grid), dim3(Cfg::NT), 0, stream, p);
  SOAPMI_LAUNCH_CHECK();
  return kOk;
}

template <class E>
int launch_few_rows(hipStream_t stream, RowProblem p) {
  p.tiles_c = (int)ceil_div64(p.cols, FewTile::BC);
  unsigned grid;
  if (int rc = grid_of(row_tiles<FewTile>(p), FewTile::NT, &grid)) return rc;
  hipLaunchKernelGGL((few_rows_kernel<E>), dim3(grid), dim3(FewTile::NT), 0, stream, p);
  SOAPMI_LAUNCH_CHECK();
  return kOk;
}

// How long a compute unit takes for a slab (128 bytes of k) of a tile: us, measured on MI355X.  alone: with
// one workgroup per compute unit and most of them idle.  At 16 and 8 bits the slabs' loads bound it; fp32
// takes the matrix cores sixteen times as long as 16 bits take them.
struct SlabTime {
  double busy, alone;
};
template <class E, class Cfg>
constexpr SlabTime slab_time() {
  constexpr bool f32 = E::SIZE == 4;
  if (Cfg::BR == WideTile::BR) return f32 ? SlabTime{7.2, 7.2} : SlabTime{1.50, 1.30};
  if (Cfg::BC == SmallTile::BC) return SlabTime{0.85, 0.50};
  if (Cfg::BR == MidTile::BR) return f32 ? SlabTime{1.9, 1.9} : SlabTime{0.60, 0.55};
  return f32 ? SlabTime{1.05, 0.75} : SlabTime{0.62, 0.34};
}
// Workgroups that run at once.
template <class Cfg>
constexpr double units() {
  return Cfg::BC == SmallTile::BC ? 768 : Cfg::BR == LowTile::BR ? 512 : 256;
}

// (no launch takes too many tiles, whatever the others take)
template <class E, class Cfg>
double row_time(const RowProblem& p) {
  if (!fits_launch(row_tiles<Cfg>(p), Cfg::NT)) return HUGE_VAL;
  const RowGroups& g = p.groups;
  // (every expert's last tile is cut short: half a tile each, when nothing else is known)
  const double rows = g.experts <= 1 ? (double)ceil_div64(g.tokens, Cfg::BR)
                                     : std::max((double)std::min(g.experts, g.tokens), (double)g.tokens / Cfg::BR + 0.5 * g.experts);
  const double tiles = rows * (double)ceil_div64(p.cols, Cfg::BC), rounds = std::ceil(tiles / units<Cfg>());
  constexpr SlabTime slab = slab_time<E, Cfg>();
  return 3.0 + rounds * (tiles * 2 <= units<Cfg>() ? slab.alone : slab.busy) * (double)ceil_div64((int64_t)p.k * E::SIZE, 128);
}

// The same for few rows (see few_rows_kernel): their bytes, weights and rows, from L2.
template <class E>
double few_rows_time(const RowProblem& p) {
  if (!fits_launch(row_tiles<FewTile>(p), FewTile::NT)) return HUGE_VAL;
  const double rows = (double)std::max<int64_t>(std::min(p.groups.experts, p.groups.tokens), ceil_div64(p.groups.tokens, FewTile::BR));
  const double each = std::min(32.0, (double)p.groups.tokens / rows);
  return 4.0 + rows * (double)ceil_div64(p.cols, FewTile::BC) * (32.0 + each) * p.k * E::SIZE / 9.3e6;
}

// Which tile.  Measured (bf16, us, low / mid / wide): 1024 rows, 1024 x 1024: 9.9 / 12.9 / 25.4; 2048 rows,
// 2048 x 2048: 35.5 / 22.6 / 42.6; 8 experts of 4096 x 4096 with 128 rows each: 115 / 69 / 97, with 384 each:
// 251 / 134 / 107.  Few rows (32 outputs x 32 rows at a time, read from L2 at about 9.3 TB/s; bytes, 4096 x
// 4096): 64 rows 12.1 against 12.8 of the low tile, 128 rows 19.3 against 13.1.
// fp32 has the small tile as well: its matrix instructions take so long that few large tiles leave most of the
// chip idle for long (input gradient, low / small / mid: 500 rows, 2048 x 512: 47.6 / 34.0 / 126; 100 rows, 1024 x
// 1024: 26.4 / 19.1 / 65.9; 4 experts of 1024 x 1100, 1000 rows: 43.3 / 37.0 / 66.7; 1024 rows, 1024 x 1024:
// 29.0 / 28.9 / 66.7; forward, 2048^3: 147 / 167 / 128).  At 16 bits, where the slabs' latency bounds small
// products, it is no clear gain (low / small: 1024 rows, 1024 x 1024: 9.9 / 10.4; 256 rows: 9.3 / 8.4).  Forward in
// fp32, few / low / small / mid / wide: 4 experts of 1024 x 1024 with 8 rows each: 9.6 / 25 / 17 / 37 / 65; 1000 rows,
// 4 x 1024 x 1100: 36 / 29 / 32 / 71 / 259 (taken: low, 28); 4096^3: 1845 / 1097 / 1127 / 968 / 927.
// Staged tiles are chosen by the direct ones' figures, although a slab takes two or three times as long.  bf16, few /
// low / mid: forward, 1500 rows of 24 experts, 1111 x 777: 56 / 22.4 / 16.9 (taken: mid); 2048 rows, 2047 x 2047: 402 /
// 70 / 35 (mid); 1024 rows, 1023 x 1023: 57 / 19.2 / 21.5 (low); 300 rows: 30.2 / 18.3 / 20.5 (few: not the best);
// input gradient of 1024 rows, 1023 x 1023: - / 50.4 / 37.8 (low: not the best).
template <class E, Layout LC, Source S>
int launch_rows(hipStream_t stream, const RowProblem& p) {
  constexpr bool has_small = S == Direct && E::SIZE == 4;
  const double low = row_time<E, LowTile>(p), mid = row_time<E, MidTile>(p);
  double few = HUGE_VAL, wide = HUGE_VAL, small = HUGE_VAL;
  if constexpr (LC == KC) few = few_rows_time<E>(p);
  if constexpr (S == Direct) wide = row_time<E, WideTile>(p);
  if constexpr (has_small) small = row_time<E, SmallTile>(p);
  if constexpr (LC == KC)
    if (few < std::min({low, mid, wide, small})) return launch_few_rows<E>(stream, p);
  if constexpr (S == Direct)
    if (wide < std::min({low, mid, small})) return launch_rows<E, LC, S, WideTile>(stream, p);
  if constexpr (has_small)
    if (small < std::min(low, mid)) return launch_rows<E, LC, S, SmallTile>(stream, p);
  return mid <= low ? launch_rows<E, LC, S, MidTile>(stream, p) : launch_rows<E, LC, S, LowTile>(stream, p);
}

// Y = rows times their expert's matrices.  direct: both operands may be fetched straight to LDS.
template <class E, Layout LC>
int row_products(hipStream_t stream, const RowProblem& p, bool direct) {
  return direct ? launch_rows<E, LC, Direct>(stream, p) : launch_rows<E, LC, Staged>(stream, p);
}

// Parts that the experts' rows are cut into when the tiles (of 128 x 128) fill less than half of the 256
// compute units and the sums are long: as many as fill them, of 8 slabs of 64 rows at least.  65536 rows of
// 512 x 512, bf16: 530 us whole, 78 us in parts; 16384 rows of 1024 x 1024: 108 and 58.  The rows are only known on
// the device and taken as shared evenly: one expert with nearly all of them gets no more parts than the others (8
// experts of 512 x 512, 65536 rows: 79 us shared evenly, 280 with all but 448 rows at one).
inline int sum_parts(int64_t experts, int64_t tokens, int64_t rows, int64_t cols) {
  const int64_t tiles = ceil_div64(rows, 128) * ceil_div64(cols, 128);  // of a matrix
  if (experts <= 0 || tiles <= 0 || tiles > 128 / experts) return 1;
  return (int)std::max<int64_t>(1, std::min(256 / (experts * tiles), tokens / experts / 512));
}
inline size_t sum_partials_bytes(int64_t experts, int64_t tokens, int64_t rows, int64_t cols) {
  const int parts = sum_parts(experts, tokens, rows, cols);
  return parts > 1 ? (size_t)parts * experts * rows * cols * sizeof(float) : 0;
}

int launch_join(hipStream_t stream, const SumProblem& p);  // products.hip

template <class Cfg>
int64_t sum_tiles(const SumProblem& p) {  // (a matrix has a multiple of 8)
  return workgroups_of(ceil_div64(p.rows, Cfg::BR) * ceil_div64(p.cols, Cfg::BC)) * p.groups.experts * p.parts;
}

template <class E, Source S, class Cfg>
int launch_sums(hipStream_t stream, SumProblem p) {
  p.tiles_r = (int)ceil_div64(p.rows, Cfg::BR);
  p.tiles_c = (int)ceil_div64(p.cols, Cfg::BC);
  unsigned grid;
  if (int rc = grid_of(sum_tiles<Cfg>(p), Cfg::NT, &grid)) return rc;
  hipLaunchKernelGGL((sum_product_kernel<E, S, Cfg>), dim3(grid), dim3(Cfg::NT), 0, stream, p);
  SOAPMI_LAUNCH_CHECK();
  return p.parts > 1 ? launch_join(stream, p) : kOk;
}

// A tile's start, its first loads and its stores, which are what short sums consist of, take `ends` us more.
template <class E, class Cfg>
double sum_time(const SumProblem& p, double ends) {
  if (!fits_launch(sum_tiles<Cfg>(p), Cfg::NT)) return HUGE_VAL;
  const double tiles = (double)p.groups.experts * p.parts * (double)(ceil_div64(p.rows, Cfg::BR) * ceil_div64(p.cols, Cfg::BC));
  const double slabs = std::max(1.0, (double)p.groups.tokens * E::SIZE / 128 / std::max(1, p.groups.experts * p.parts));
  constexpr SlabTime slab = slab_time<E, Cfg>();
  return std::ceil(tiles / units<Cfg>()) * (ends + slabs * (tiles * 2 <= units<Cfg>() ? slab.alone : slab.busy));
}

// Measured (bf16, us, mid / wide): 8192 rows, 4096 x 4096: 297 / 208; 8 experts of 2048 x 4096, 8192 rows:
// 250 / 165; 5 experts of 520 x 1000, 1020 rows: 11.2 / 17.8; 32 experts of 512 x 512, 64 rows: 14.5 / 17.5.
template <class E, Source S>
int launch_sums(hipStream_t stream, const SumProblem& p) {
  const double low = sum_time<E, LowTile>(p, 3.0), mid = sum_time<E, MidTile>(p, 4.0);
  if constexpr (S == Direct)
    if (sum_time<E, WideTile>(p, 10.0) < std::min(low, mid)) return launch_sums<E, S, WideTile>(stream, p);
  return mid <= low ? launch_sums<E, S, MidTile>(stream, p) : launch_sums<E, S, LowTile>(stream, p);
}

// D_e = sums over the experts' rows.  direct: the operands may be fetched straight to LDS.
template <class E>
int sum_products(hipStream_t stream, const SumProblem& p, bool direct) {
  return direct ? launch_sums<E, Direct>(stream, p) : launch_sums<E, Staged>(stream, p);
}

}  // namespace soapmi
