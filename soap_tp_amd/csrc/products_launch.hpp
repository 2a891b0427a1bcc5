// Host side of products.hpp: which kernel a product runs on.  Each element type is instantiated in a
// source file of its own (products_bf16.hip, products_f16.hip, products_i8.hip), which compile side by side.
#pragma once
#include <algorithm>
#include <cmath>

#include "products.hpp"

namespace soapmi {

using WideTile = ProductTile<256, 256, 2, 4, 2, 1>;
using MidTile = ProductTile<128, 128, 2, 4, 4, 3>;
using LowTile = ProductTile<32, 128, 1, 4, 4, 3>;

inline int grid_of(int64_t tiles, unsigned* grid) {
  const int64_t g = 8 * ((tiles + 7) / 8);
  SOAPMI_REQUIRE(g < (int64_t)1 << 31, "the product has too many tiles for one launch");
  *grid = (unsigned)g;
  return kOk;
}

// Row tiles that any split of `tokens` rows over the groups can need.
inline int64_t most_row_tiles(const RowGroups& g, int br) {
  return g.tokens / br + std::min<int64_t>((int64_t)g.experts + g.rest, g.tokens);
}

template <class E, Layout LC, Source S, class Cfg>
int launch_rows(hipStream_t stream, RowProblem p) {
  p.tiles_c = (int)ceil_div64(p.cols, Cfg::BC);
  unsigned grid;
  if (int rc = grid_of(most_row_tiles(p.groups, Cfg::BR) * p.tiles_c, &grid)) return rc;
  hipLaunchKernelGGL((row_product_kernel<E, LC, S, Cfg>), dim3(grid), dim3(Cfg::NT), 0, stream, p);
  SOAPMI_LAUNCH_CHECK();
  return kOk;
}

template <class E>
int launch_few_rows(hipStream_t stream, RowProblem p) {
  p.tiles_c = (int)ceil_div64(p.cols, FewTile::BC);
  unsigned grid;
  if (int rc = grid_of(most_row_tiles(p.groups, FewTile::BR) * p.tiles_c, &grid)) return rc;
  hipLaunchKernelGGL((few_rows_kernel<E>), dim3(grid), dim3(FewTile::NT), 0, stream, p);
  SOAPMI_LAUNCH_CHECK();
  return kOk;
}

// Microseconds that a product of `groups` experts' rows takes on tiles of br x bc, as measured on MI355X:
// a slab of 128 bytes of k takes the compute unit `slab` us (`alone` if it has one workgroup only), and
// a workgroup's start and end 3 us; units = workgroups that run at once.
inline double tile_time(const RowGroups& g, int64_t cols, int64_t k_bytes, int br, int bc, double units, double slab, double alone) {
  // (every expert's last tile is cut short: half a tile each, when nothing else is known)
  const double rows = g.experts <= 1 ? (double)ceil_div64(g.tokens, br)
                                     : std::max((double)std::min(g.experts, g.tokens), (double)g.tokens / br + 0.5 * g.experts);
  const double tiles = rows * (double)ceil_div64(cols, bc), rounds = std::ceil(tiles / units);
  const double each = tiles * 2 <= units ? alone : slab;
  return 3.0 + rounds * each * (double)ceil_div64(k_bytes, 128);
}

// Which tile.  Measured (bf16, us, low / mid / wide): 1024 rows, 1024 x 1024: 9.9 / 12.9 / 25.4; 2048 rows,
// 2048 x 2048: 35.5 / 22.6 / 42.6; 8 experts of 4096 x 4096 with 128 rows each: 115 / 69 / 97, with 384 each:
// 251 / 134 / 107.  Few rows (32 outputs x 32 rows at a time, read from L2 at about 9.3 TB/s; bytes, 4096 x
// 4096): 64 rows 12.1 against 12.8 of the low tile, 128 rows 19.3 against 13.1.
template <class E, Layout LC, Source S>
int launch_rows(hipStream_t stream, const RowProblem& p) {
  const int64_t k_bytes = (int64_t)p.k * E::SIZE;
  const double low = tile_time(p.groups, p.cols, k_bytes, LowTile::BR, LowTile::BC, 512, 0.62, 0.34);
  const double mid = tile_time(p.groups, p.cols, k_bytes, MidTile::BR, MidTile::BC, 256, 0.60, 0.55);
  if constexpr (LC == KC) {
    const double rows = (double)std::max<int64_t>(std::min(p.groups.experts, p.groups.tokens), ceil_div64(p.groups.tokens, FewTile::BR));
    const double each = std::min(32.0, (double)p.groups.tokens / rows);
    const double few = 4.0 + rows * (double)ceil_div64(p.cols, FewTile::BC) * (32.0 + each) * (double)k_bytes / 9.3e6;
    if (few < std::min(low, mid)) return launch_few_rows<E>(stream, p);
  }
  if constexpr (S == Direct) {
    const double wide = tile_time(p.groups, p.cols, k_bytes, WideTile::BR, WideTile::BC, 256, 1.50, 1.30);
    if (wide < std::min(low, mid)) return launch_rows<E, LC, S, WideTile>(stream, p);
  }
  return mid <= low ? launch_rows<E, LC, S, MidTile>(stream, p) : launch_rows<E, LC, S, LowTile>(stream, p);
}

// Y = rows times their expert's matrices.  direct: both operands may be fetched straight to LDS.
template <class E, Layout LC>
int row_products(hipStream_t stream, const RowProblem& p, bool direct) {
  return direct ? launch_rows<E, LC, Direct>(stream, p) : launch_rows<E, LC, Staged>(stream, p);
}

// Parts that the experts' rows are cut into when the tiles (of 128 x 128) fill less than half of the 256
// compute units and the sums are long: as many as fill them, of 8 slabs of 64 rows at least.  65536 rows of
// 512 x 512: PARTS_MEASURED.
inline int sum_parts(int64_t experts, int64_t tokens, int64_t rows, int64_t cols) {
  const int64_t tiles = experts * ceil_div64(rows, 128) * ceil_div64(cols, 128);
  if (experts <= 0 || tiles <= 0 || tiles > 128) return 1;
  return (int)std::max<int64_t>(1, std::min(256 / tiles, tokens / experts / 512));
}
inline size_t sum_partials_bytes(int64_t experts, int64_t tokens, int64_t rows, int64_t cols) {
  const int parts = sum_parts(experts, tokens, rows, cols);
  return parts > 1 ? (size_t)parts * experts * rows * cols * sizeof(float) : 0;
}

int launch_join(hipStream_t stream, const SumProblem& p);  // products.hip

// Workgroups of a launch whose tiles are br x bc.
inline int sum_grid(SumProblem& p, int br, int bc, unsigned* grid) {
  p.tiles_r = (int)ceil_div64(p.rows, br);
  p.tiles_c = (int)ceil_div64(p.cols, bc);
  return grid_of(8 * ceil_div64((int64_t)p.tiles_r * p.tiles_c, 8) * p.groups.experts * p.parts, grid);
}

template <class E, Source S, class Cfg>
int launch_sums(hipStream_t stream, SumProblem p) {
  unsigned grid;
  if (int rc = sum_grid(p, Cfg::BR, Cfg::BC, &grid)) return rc;
  hipLaunchKernelGGL((sum_product_kernel<E, S, Cfg>), dim3(grid), dim3(Cfg::NT), 0, stream, p);
  SOAPMI_LAUNCH_CHECK();
  return p.parts > 1 ? launch_join(stream, p) : kOk;
}

// Wide tiles from 192 of them on: SUMS_MEASURED
template <class E, Source S>
int launch_sums(hipStream_t stream, const SumProblem& p) {
  const int64_t wide_tiles = ceil_div64(p.rows, 256) * ceil_div64(p.cols, 256) * p.groups.experts;
  if constexpr (S == Direct)
    if (wide_tiles >= 96 && p.parts == 1) return launch_sums<E, S, WideTile>(stream, p);
  return launch_sums<E, S, MidTile>(stream, p);
}

// D_e = sums over the experts' rows.  direct: the operands may be fetched straight to LDS.
template <class E>
int sum_products(hipStream_t stream, const SumProblem& p, bool direct) {
  return direct ? launch_sums<E, Direct>(stream, p) : launch_sums<E, Staged>(stream, p);
}

}  // namespace soapmi
