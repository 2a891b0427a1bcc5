// Host side of products.hpp: which kernel a product runs on.  Each element type is instantiated in a
// source file of its own (products_bf16.hip, products_f16.hip, products_i8.hip), which compile side by side.
#pragma once
#include <algorithm>

#include "products.hpp"

namespace soapmi {

using WideTile = ProductTile<256, 256, 2, 4>;
using MidTile = ProductTile<128, 128, 2, 2>;
using LowTile = ProductTile<32, 128, 1, 4>;

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

template <class E, Layout LC, Source S>
int launch_rows(hipStream_t stream, const RowProblem& p) {
  const int64_t each = p.groups.tokens / std::max(1, p.groups.experts);  // rows of an average expert
  const int64_t wide_tiles = ceil_div64(p.groups.tokens, 256) * ceil_div64(p.cols, 256);
  if constexpr (S == Direct)
    if (each >= 192 && wide_tiles >= 192) return launch_rows<E, LC, S, WideTile>(stream, p);
  if (each > 48) return launch_rows<E, LC, S, MidTile>(stream, p);
  return launch_rows<E, LC, S, LowTile>(stream, p);
}

// Y = rows times their expert's matrices.  direct: both operands may be fetched straight to LDS.
template <class E, Layout LC>
int row_products(hipStream_t stream, const RowProblem& p, bool direct) {
  if constexpr (LC == KC)
    if (p.groups.tokens <= (int64_t)32 * std::max(1, p.groups.experts)) return launch_few_rows<E>(stream, p);
  return direct ? launch_rows<E, LC, Direct>(stream, p) : launch_rows<E, LC, Staged>(stream, p);
}

template <class E, Source SR, Source SC, class Cfg>
int launch_sums(hipStream_t stream, SumProblem p) {
  p.tiles_r = (int)ceil_div64(p.rows, Cfg::BR);
  p.tiles_c = (int)ceil_div64(p.cols, Cfg::BC);
  const int64_t chunk = ((int64_t)p.tiles_r * p.tiles_c + 7) / 8;
  unsigned grid;
  if (int rc = grid_of(8 * chunk * p.groups.experts, &grid)) return rc;
  hipLaunchKernelGGL((sum_product_kernel<E, SR, SC, Cfg>), dim3(grid), dim3(Cfg::NT), 0, stream, p);
  SOAPMI_LAUNCH_CHECK();
  return kOk;
}

template <class E, Source SR, Source SC>
int launch_sums(hipStream_t stream, const SumProblem& p) {
  const int64_t wide_tiles = ceil_div64(p.rows, 256) * ceil_div64(p.cols, 256) * p.groups.experts;
  if constexpr (SR == Direct)
    if (wide_tiles >= 192) return launch_sums<E, SR, SC, WideTile>(stream, p);
  return launch_sums<E, SR, SC, MidTile>(stream, p);
}

// D_e = sums over the experts' rows.  direct: the operands (saved: the gradient) may be fetched straight to LDS.
template <class E>
int sum_products(hipStream_t stream, const SumProblem& p, bool direct, bool saved) {
  if (saved) return direct ? launch_sums<E, Direct, Codes>(stream, p) : launch_sums<E, Staged, Codes>(stream, p);
  return direct ? launch_sums<E, Direct, Direct>(stream, p) : launch_sums<E, Staged, Staged>(stream, p);
}

}  // namespace soapmi
