// Products of a layer with weights grouped by expert, in 32-bit and 16-bit floating point and 8-bit integers.
//
//   rows grouped (forward, input gradient):  Y[t, c] = sum_k R[t, k] C_e(t)[c, k]
//   k grouped    (weight gradient):          D_e[r, c] = sum over t in e of R[t, r] C[t, c]
//
// The rows t of expert e are [ends[e-1], ends[e]).  The sizes are only known on the device: a launch
// has as many workgroups as the worst split of the rows can need, every workgroup finds its tile from
// `ends` itself (a prefix sum over the experts in one wavefront's lanes), and the ones behind the last
// tile leave.  Nothing is read back to the host and no launch prepares another.
//
// Operands.  Each operand is KC (its k index is contiguous in memory) or XC (its row or column index
// is).  LDS holds two or four slabs of 128 bytes of k (32, 64 or 128 values), so that the next ones travel
// while one is multiplied:
//   KC  S[x][128 bytes], 16-byte pieces, piece p of row x stored at p ^ key(x): the 16 rows that a
//       fragment read touches then start in different banks;
//   XC  S[k][x], blocks of 16 values, block b of row k stored at b ^ f(k); fragments are read with the
//       transposing LDS read, which hands each lane 4 consecutive k of one x (32-bit values: one by one).
// Both layouts are linear in the order in which lanes fetch, which is what a load from memory straight
// to LDS needs: the permutation is applied to the address each lane fetches from.
//
// The matrix instruction's first operand is the column side, so that a lane's accumulators are
// consecutive columns of one output row; columns are dealt to fragments in such a way that two
// fragments give a lane eight consecutive ones (one 16-byte store of 16-bit results).
#pragma once
#include <type_traits>

#include "common.hpp"

namespace soapmi {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

enum : int { kFloat32 = 0, kBFloat16 = 1, kFloat16 = 2 };  // SOAPMI_FLOAT32 ...

// SIZE: bytes of an operand's value.  Value: the type that a result may have beside fp32 (8-bit products: any).
struct ElemBF16 {
  static constexpr int SIZE = 2;
  using Value = __bf16;
  using Acc = f32x4;
  static __device__ __forceinline__ Acc mma(i32x4 a, i32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
struct ElemF16 {
  static constexpr int SIZE = 2;
  using Value = _Float16;
  using Acc = f32x4;
  static __device__ __forceinline__ Acc mma(i32x4 a, i32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
struct ElemF32 {
  static constexpr int SIZE = 4;
  using Value = float;
  using Acc = f32x4;
  static __device__ __forceinline__ Acc mma(i32x4 a, i32x4 b, Acc c) {  // four values of k, one after the other
    const f32x4 af = __builtin_bit_cast(f32x4, a), bf = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_16x16x4f32(af[t], bf[t], c, 0, 0, 0);
    return c;
  }
};
struct ElemI8 {
  static constexpr int SIZE = 1;
  using Value = void;
  using Acc = i32x4;
  static __device__ __forceinline__ Acc mma(i32x4 a, i32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  }
};

// ---- which tile a workgroup has ------------------------------------------------------------

struct RowGroups {
  const int64_t* ends;  // null: one expert holds every row
  int experts;
  int rest;             // rows behind the last expert's are a group of their own (written as zeros)
  int tokens;
};

// Group g's rows.  Whatever `ends` holds, they lie in [0, tokens).
__device__ __forceinline__ void group_rows(const RowGroups& g, int e, int& begin, int& end) {
  if (g.ends == nullptr) {
    begin = e == 0 ? 0 : g.tokens;
    end = g.tokens;
    return;
  }
  const int64_t lo = e > 0 ? g.ends[e - 1] : 0, hi = e < g.experts ? g.ends[e] : g.tokens;
  begin = (int)min(max(lo, (int64_t)0), (int64_t)g.tokens);
  end = max(begin, (int)min(max(hi, (int64_t)0), (int64_t)g.tokens));
}

__device__ __forceinline__ int wave_inclusive_sum(int v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(v, d);
    if (lane >= d) v += up;
  }
  return v;
}

struct RowTile {
  int expert;  // == experts: the rest
  int row;     // first row
  int rows;    // rows of the tile that belong to the group (1 .. BR)
};

// Tile number wg of the launch -> its rows and columns.  Row tiles never cross a group's end; a group of
// n rows has ceil(n / BR) of them, which share its rows evenly in units of GRAIN: a tile's time goes by
// its rows (see TileProduct), and one nearly empty tile behind full ones would be a round of its own.
// Consecutive workgroup ids are dealt round-robin to the 8 XCDs; each XCD gets one contiguous range of
// tiles, walked in groups of up to 8 row tiles by all columns, so that a weight tile is fetched into
// that XCD's L2 once for its row tiles.  Returns false behind the last tile.
template <int BR, int GRAIN>
__device__ __forceinline__ bool locate_rows(const RowGroups& g, unsigned tiles_c, unsigned wg, RowTile& tile, int& tile_c) {
  const int lane = threadIdx.x & 63;
  const int groups = g.experts + g.rest;
  int total = 0;
  int first_tiles = 0, first_begin = 0, first_end = 0;  // of the first 64 groups, kept for the search
  if (g.ends == nullptr) {
    total = (g.tokens + BR - 1) / BR;
  } else {
    for (int e0 = 0; e0 < groups; e0 += 64) {
      int begin = 0, end = 0;
      if (e0 + lane < groups) group_rows(g, e0 + lane, begin, end);
      const int tiles = wave_inclusive_sum((end - begin + BR - 1) / BR, lane);
      if (e0 == 0) {
        first_tiles = tiles;
        first_begin = begin;
        first_end = end;
      }
      total += __builtin_amdgcn_readlane(tiles, 63);
    }
  }
  // (32-bit numbers throughout: a launch has fewer than 2^31 tiles, and divisions of 64-bit ones are long)
  const unsigned all = (unsigned)total * tiles_c;
  const unsigned chunk = (all + 7) >> 3;
  const unsigned t = (wg & 7) * chunk + (wg >> 3);
  if ((wg >> 3) >= chunk || t >= all) return false;
  constexpr unsigned GR = 8;
  const unsigned per = GR * tiles_c;
  const unsigned band = t / per, in_band = t - band * per;
  const unsigned rows = min(GR, (unsigned)total - band * GR);
  const unsigned column = in_band / rows;
  const int tr = (int)(band * GR + in_band - column * rows);
  tile_c = __builtin_amdgcn_readfirstlane((int)column);
  auto found = [&](int expert, int begin, int end, int nth) {
    const unsigned grains = (unsigned)(end - begin + GRAIN - 1) / GRAIN, share = (unsigned)(end - begin + BR - 1) / BR;
    const unsigned each = grains / share, larger = grains - each * share;  // the first `larger` tiles have one more
    const int first = (int)(nth * each + min((unsigned)nth, larger)) * GRAIN;
    const int last = min(end - begin, first + (int)(each + ((unsigned)nth < larger ? 1 : 0)) * GRAIN);
    tile.expert = __builtin_amdgcn_readfirstlane(expert);
    tile.row = __builtin_amdgcn_readfirstlane(begin + first);
    tile.rows = __builtin_amdgcn_readfirstlane(last - first);
  };
  if (g.ends == nullptr) {
    found(0, 0, g.tokens, tr);
    return true;
  }
  int before = 0;
  for (int e0 = 0; e0 < groups; e0 += 64) {
    int begin = first_begin, end = first_end, tiles = first_tiles;
    if (e0 > 0) {
      begin = end = 0;
      if (e0 + lane < groups) group_rows(g, e0 + lane, begin, end);
      tiles = wave_inclusive_sum((end - begin + BR - 1) / BR, lane);
    }
    const uint64_t behind = __ballot(before + tiles > tr);
    if (behind) {
      const int at = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)behind) - 1);
      const int up_to = at ? __builtin_amdgcn_readlane(tiles, at - 1) : 0;
      found(e0 + at, __builtin_amdgcn_readlane(begin, at), __builtin_amdgcn_readlane(end, at), tr - before - up_to);
      return true;
    }
    before += __builtin_amdgcn_readlane(tiles, 63);
  }
  return false;  // (not reached: tr < total)
}

// ---- operands ------------------------------------------------------------------------------

// Address bits that spread KC rows over the banks.  The row side reads rows x .. x+15; the column side
// reads rows 8g + {0..3} (+ 4) for g = 0..3, see column_of.
__device__ __forceinline__ int kc_key(bool column_side, int x) {
  return column_side ? (x & 3) | ((x >> 1) & 4) : x & 7;
}
// ... and XC rows, whose blocks of 16 values change places: a transposing read of 32 lanes covers k rows
// {0..3, 8..11} (+ 4); reads of single 32-bit values k rows {0, 4, 8, 12} (+ 1, 2, 3), of which two still
// share banks (bit 3 would cost a lane a second offset; the matrix cores bound fp32 anyway).
template <int SIZE, int BX>
__device__ __forceinline__ int xc_key(int k) {
  return (SIZE == 4 ? k >> 2 & 1 : (k & 3) | ((k >> 1) & 4)) & (BX / 16 - 1);
}

// Columns of a wavefront's fragment i, row m of the matrix instruction: fragments 2i and 2i+1 give lane
// group g (m / 4) the columns 32i + 8g .. 32i + 8g + 7.
__device__ __forceinline__ int column_of(int i, int m) { return 32 * (i >> 1) + 8 * (m >> 2) + 4 * (i & 1) + (m & 3); }

enum Layout { KC, XC };
// How an operand gets to LDS.  Direct: 16-byte pieces straight from memory (rows that start at multiples of
// 16 bytes).  Staged: through registers, any alignment.
enum Source { Direct, Staged };

struct Operand {
  const char* base;  // tile's first element
  int64_t ld;        // bytes from one stored row to the next
  int valid;         // rows (columns) of the tile that exist
};

constexpr unsigned kOutside = 0xC0000000u;    // a byte offset outside every buffer: such a lane fetches zeros
constexpr int kBufferBytes = 0x40000000;

// 16 bytes per lane from memory (resource's address + offset + more) to LDS at lds + 16 * lane (more and lds:
// the same in all lanes of a wavefront); zeros where the resource ends before them.
// In inline assembly because the compiler, told of such a load, waits for it before every transposing
// LDS read, the ones of the other buffer included.  There is no output but m0; wait_loads() waits for the load.
// The compiler does not look inside for hazards either: a scalar register that a vector instruction wrote may be
// read by a memory instruction five wait states later at the earliest, m0 one after a scalar write.  The s_nop
// is for m0.  The other registers come from scalar instructions, or from long before, and the build refuses a
// library where one does not (five wait states at every load instead: 8192^3 forward 762 -> 772 us, weight
// gradient 758 -> 771; at every new resource: 773 -> 777, input gradient 759 -> 768).
__device__ __forceinline__ void load_to_lds(i32x4 resource, unsigned offset, unsigned more, unsigned lds) {
  unsigned m0;
  asm volatile("s_mov_b32 %0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds"
               : "=&{m0}"(m0)
               : "s"(lds), "v"(offset), "s"(resource), "s"(more)
               : "memory");
}

__device__ __forceinline__ i32x4 buffer_of(const char* base, int bytes) {
  const uint64_t address = reinterpret_cast<uint64_t>(base);
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)address);
  r[1] = __builtin_amdgcn_readfirstlane((int)((address >> 32) & 0xffff));
  r[2] = __builtin_amdgcn_readfirstlane(bytes);
  r[3] = 0x00020000;
  return r;
}
template <int N>
__device__ __forceinline__ void wait_loads() {  // all but the last N loads of this wavefront are done
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
// Memory accesses stay on their side of this in the program.  A wavefront's LDS accesses are carried out in
// order, so that is all that lanes of one wavefront need to hand each other values; without it the compiler,
// which sees each lane by itself, may exchange a read and a write that belong to different lanes.
__device__ __forceinline__ void keep_order() { asm volatile("" ::: "memory"); }
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier() { asm volatile("s_barrier" ::: "memory"); }

__device__ __forceinline__ i32x4 load_bytes(const char* p, int count) {
  i32x4 v = {0, 0, 0, 0};
  if (count >= 16) {
    __builtin_memcpy(&v, p, 16);
  } else if (count > 0) {
    char b[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) b[i] = i < count ? p[i] : 0;
    __builtin_memcpy(&v, b, 16);
  }
  return v;
}

__device__ __forceinline__ float exponent_value(int code) {  // 2^(code - 127), 0 subnormal; 255: not a number
  return __uint_as_float(code == 255 ? 0x7fc00000u : code == 0 ? 0x00400000u : (unsigned)code << 23);
}

// One operand of a tile: BX rows (or columns), slabs of 128 bytes (KC) or 64 values (XC) of k.
template <class E, Layout L, Source S, int BX, int NT, bool COLUMN, int AHEAD>
struct Loader {
  static constexpr int SLAB_K = 128 / E::SIZE;
  static constexpr int BYTES = BX * 128;
  static constexpr int PIECES = BYTES / 16;
  static constexpr int NP = (PIECES + NT - 1) / NT;
  static_assert(L == KC || E::SIZE >= 2, "8-bit operands are KC");
  static_assert(S != Direct || PIECES % 64 == 0, "whole wavefronts fetch");
  static constexpr int PER_ROW = L == KC ? 8 : BX * E::SIZE / 16;  // pieces in an LDS row

  // Piece q = tid + i * NT of an operand lies i * STEP stored rows below piece tid and in the same place of
  // its row, since the permutations look at row bits below STEP only.
  static constexpr int STEP = NT / PER_ROW;
  static_assert(NP == 1 || STEP % (L == XC && E::SIZE == 4 ? 8 : 16) == 0, "one place in the row serves all of a lane's pieces");

  const char* base;
  int64_t ld;
  int valid;
  int tid;
  unsigned offset, offset_now;  // Direct: of the lane's first piece; in the slab being sent
  int first_row, first_piece;   // of the lane's first piece
  i32x4 resource;
  i32x4 held[S == Direct ? 1 : AHEAD][S == Direct ? 1 : NP];  // Staged: slabs in registers

  // stored row and piece of LDS piece q
  static __device__ __forceinline__ void place(int q, int& row, int& piece) {
    row = q / PER_ROW;
    const int slot = q % PER_ROW;
    if (L == KC) piece = slot ^ kc_key(COLUMN, row);
    else piece = (slot / E::SIZE ^ xc_key<E::SIZE, BX>(row)) * E::SIZE | slot % E::SIZE;  // (SIZE pieces are 16 values)
  }

  __device__ __forceinline__ void init(const Operand& o, int tid_) {
    base = o.base;
    ld = o.ld;
    valid = o.valid;
    tid = tid_;
    place(tid, first_row, first_piece);
    if constexpr (S == Direct) {
      offset = (unsigned)(first_row * (int)ld + first_piece * 16);
      if (L == XC && first_piece * 16 >= valid * E::SIZE) offset = kOutside;
    }
  }

  __device__ __forceinline__ const char* slab(int kt) const {
    return L == KC ? base + (int64_t)kt * 128 : base + (int64_t)kt * SLAB_K * ld;
  }

  // Direct: slab kt is sent piece by piece.  k_left = values of k from this slab on.  The buffer ends with
  // the 16 bytes that hold the last row's last value (rows start at multiples of 16 bytes, so these are in
  // one row and one page), so that rows behind the last one come as zeros.  In a last slab that is cut
  // short, so do the pieces of a KC operand behind the cut; what the piece with the cut brings from behind
  // it, trim() takes out again.
  __device__ __forceinline__ void aim(int kt, int k_left) {
    const int k_here = min(k_left, SLAB_K);
    const int bytes = L == KC ? (valid - 1) * (int)ld + k_here * E::SIZE : (k_here - 1) * (int)ld + valid * E::SIZE;
    resource = buffer_of(slab(kt), k_left > 0 ? (bytes + 15) & ~15 : 0);  // (behind the last slab: nothing but zeros)
    offset_now = L == KC && first_piece * 16 >= k_here * E::SIZE ? kOutside : offset;
  }
  __device__ __forceinline__ void send(int i, unsigned lds) {
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (PIECES % NT != 0 && (wave + i * (NT / 64)) * 64 >= PIECES) return;
    load_to_lds(resource, offset_now, (unsigned)(i * STEP * (int)ld), lds + wave * 1024 + i * NT * 16);
  }

  // Staged: piece i of slab kt comes to register set `set`.  k_left as for aim().
  __device__ __forceinline__ void fetch(int i, int kt, int k_left, int set) {
    if constexpr (S == Staged) {
      if (PIECES % NT != 0 && tid + i * NT >= PIECES) return;
      const int row = first_row + i * STEP;
      const char* at = slab(kt) + first_piece * 16;
      if (L == KC) {
        const int r = min(row, valid - 1);  // rows behind the last one only reach results that are not stored
        at += r * ld;
        if (k_left >= SLAB_K) held[set][i] = load_bytes(at, 16);
        else held[set][i] = load_bytes(at, max(k_left, 0) * E::SIZE - first_piece * 16);
      } else {
        at += row * ld;
        if (k_left >= SLAB_K && valid == BX) held[set][i] = load_bytes(at, 16);
        else held[set][i] = load_bytes(at, row < k_left ? valid * E::SIZE - first_piece * 16 : 0);
      }
    }
  }

  // ... and goes on to LDS.
  __device__ __forceinline__ void put(int i, int set, char* lds) {
    const int q = tid + i * NT;
    if constexpr (S == Staged)
      if (PIECES % NT == 0 || q < PIECES) *reinterpret_cast<i32x4*>(lds + q * 16) = held[set][i];
  }

  // The slab in LDS without the bytes of k from `left` on that are in the same piece as the one before them.
  static __device__ __forceinline__ void trim(char* lds, int left, int tid) {
    if constexpr (L == KC) {
      for (int x = tid; x < BX; x += NT) {
        i32x4* at = reinterpret_cast<i32x4*>(lds + x * 128 + ((left >> 4 ^ kc_key(COLUMN, x)) << 4));
        i32x4 v = *at;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int keep = min(max((left & 15) - 4 * d, 0), 4);
          v[d] = keep == 4 ? v[d] : v[d] & ((1 << (8 * keep)) - 1);
        }
        *at = v;
      }
    }
  }

  // 16 bytes of fragment data for (x, k step ks): KC: k pieces 4 ks + lane group; XC: 8 k values.
  // x0: first x of the wavefront, i: fragment.
  static __device__ __forceinline__ i32x4 fragment(const char* lds, int x0, int i, int ks, int lane) {
    const int m = lane & 15, g = lane >> 4;
    if constexpr (L == KC) {
      const int x = x0 + (COLUMN ? column_of(i, m) : 16 * i + m);
      return *reinterpret_cast<const i32x4*>(lds + x * 128 + (((ks * 4 + g) ^ kc_key(COLUMN, x)) << 4));
    } else if constexpr (E::SIZE == 2) {
      // lane m of a 16-lane group supplies four x (chunk m % 4) of k row m / 4 and receives column m
      const int x = x0 + (COLUMN ? 32 * (i >> 1) + 8 * (m & 3) + 4 * (i & 1) : 16 * i + 4 * (m & 3));
      i32x4 out;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = ks * 32 + g * 8 + h * 4 + (m >> 2);
        char* p = const_cast<char*>(lds) + k * (BX * 2) + ((((x >> 4) ^ xc_key<2, BX>(k)) << 5) | ((x & 15) << 1));
        const s16x4 part = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
        const auto two = __builtin_bit_cast(int __attribute__((ext_vector_type(2))), part);
        out[2 * h] = two[0];
        out[2 * h + 1] = two[1];
      }
      return out;
    } else {
      const int x = x0 + (COLUMN ? column_of(i, m) : 16 * i + m);
      i32x4 out;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int k = ks * 16 + g * 4 + t;
        out[t] = *reinterpret_cast<const int*>(lds + k * (BX * 4) + ((((x >> 4) ^ xc_key<4, BX>(k)) << 6) | ((x & 15) << 2)));
      }
      return out;
    }
  }
};

// BR x BC results, WR x WC wavefronts.  STAGES slabs are in LDS or on their way there (Direct; Staged: two,
// and AHEAD more in registers).
template <int BR_, int BC_, int WR_, int WC_, int STAGES_, int AHEAD_>
struct ProductTile {
  static constexpr int BR = BR_, BC = BC_, WR = WR_, WC = WC_, STAGES = STAGES_, AHEAD = AHEAD_;
  static constexpr int NT = 64 * WR * WC;
  static constexpr int TR = BR / WR / 16, TC = BC / WC / 16;
  static_assert(TC % 2 == 0, "columns are dealt to pairs of fragments");
  static_assert(BR % (16 * WR) == 0 && BC % (16 * WC) == 0, "wave tiling");
};

// acc = sum over k of R[r, k] C[c, k] of one tile, of which the first A * WR fragments of 16 rows are
// computed.  The fragments are dealt to the WR rows of wavefronts in turn, so that a tile with few rows
// takes all of them for a shorter time.
//
// A slab is two steps of the matrix instruction's k.  While a wavefront multiplies one step's fragments,
// the next step's come from LDS into other registers, and further slabs are in LDS or on their way.  What
// moves data is dealt out between the rows of matrix instructions: a wavefront issues in order, and the
// loads of a whole slab in a row would keep it from issuing anything else for as long as they take
// (8192^3 on 256 x 256 tiles: 850 us with the loads at the slab's start, 790 with them dealt out).
//
// What bounds it there: the matrix cores are busy for 72 - 77 % of the time at a clock that power holds at 1.8 -
// 1.9 GHz of 2.4 (forward 760 - 790 us); without loads the same code takes 650 us, on zero operands 650-700.
template <class E, Layout LR, Layout LC, Source S, class Cfg, int A = Cfg::TR>
struct TileProduct {
  static constexpr bool DIRECT = S == Direct;
  static constexpr int STAGES = DIRECT ? Cfg::STAGES : 2, AHEAD = DIRECT ? 1 : Cfg::AHEAD;
  static_assert((STAGES & (STAGES - 1)) == 0, "a slab's stage is its number's low bits");
  using LoadR = Loader<E, LR, S, Cfg::BR, Cfg::NT, false, AHEAD>;
  using LoadC = Loader<E, LC, S, Cfg::BC, Cfg::NT, true, AHEAD>;
  static constexpr int SLAB_K = LoadR::SLAB_K;
  static_assert(LoadR::SLAB_K == LoadC::SLAB_K, "one slab for both operands");
  static_assert(!DIRECT || STAGES == 2 || (LoadR::PIECES % Cfg::NT == 0 && LoadC::PIECES % Cfg::NT == 0),
                "waiting by count: every lane has the same number of loads");
  static constexpr int STAGE = LoadR::BYTES + LoadC::BYTES;
  static constexpr int LDS_BYTES = STAGES * STAGE;
  static_assert(LDS_BYTES >= 8192 * Cfg::NT / 64, "results pass through it (kStoreBytes)");
  static constexpr int TR = A, TC = Cfg::TC, READS = TR + TC;
  // pieces that a lane moves per slab: of a KC row operand only those of the rows that are computed
  static constexpr int PIECES_R = LR == KC ? (A * Cfg::WR * 16 + LoadR::STEP - 1) / LoadR::STEP : LoadR::NP;
  static constexpr int PIECES = PIECES_R + LoadC::NP;
  using Acc = typename E::Acc;

  struct Fragments {
    i32x4 r[TR], c[TC];
  };
  // Fragment number n of a step: the columns' first, then the rows'.
  static __device__ __forceinline__ void read(Fragments& f, int n, const char* stage, int wr0, int wc0, int ks, int lane) {
    if (n < TC) f.c[n] = LoadC::fragment(stage + LoadR::BYTES, wc0, n, ks, lane);
    else f.r[n - TC] = LoadR::fragment(stage, wr0, (n - TC) * Cfg::WR, ks, lane);
  }
  static __device__ __forceinline__ void multiply_row(const Fragments& f, int j, Acc (&acc)[TR][TC]) {
#pragma unroll
    for (int i = 0; i < TC; ++i) acc[j][i] = E::mma(f.c[i], f.r[j], acc[j][i]);
  }

  static __device__ __forceinline__ void run(const Operand& r, const Operand& c, int k_count, char* lds, Acc (&acc)[TR][TC]) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wr0 = (wave % Cfg::WR) * 16, wc0 = (wave / Cfg::WR) * (TC * 16);
#pragma unroll
    for (int j = 0; j < TR; ++j)
#pragma unroll
      for (int i = 0; i < TC; ++i) acc[j][i] = Acc{0, 0, 0, 0};
    const int slabs = (k_count + SLAB_K - 1) / SLAB_K;
    if (slabs == 0) return;
    const unsigned lds_address = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    LoadR lr;
    LoadC lc;
    lr.init(r, tid);
    lc.init(c, tid);
    auto stage_of = [](int kt) { return (kt & (STAGES - 1)) * STAGE; };
    auto aim = [&](int kt) {
      if constexpr (DIRECT) {
        lr.aim(kt, k_count - kt * SLAB_K);
        lc.aim(kt, k_count - kt * SLAB_K);
      }
    };
    // piece n of slab kt: to registers (Staged) ...
    auto fetch = [&](int n, int kt, int set) {
      if (n < PIECES_R) lr.fetch(n, kt, k_count - kt * SLAB_K, set);
      else lc.fetch(n - PIECES_R, kt, k_count - kt * SLAB_K, set);
    };
    // ... and to LDS, from there or straight from memory
    auto move = [&](int n, int kt, int set) {
      if (n < PIECES_R) {
        if constexpr (DIRECT) lr.send(n, lds_address + stage_of(kt));
        else lr.put(n, set, lds + stage_of(kt));
      } else {
        if constexpr (DIRECT) lc.send(n - PIECES_R, lds_address + stage_of(kt) + LoadR::BYTES);
        else lc.put(n - PIECES_R, set, lds + stage_of(kt) + LoadR::BYTES);
      }
    };
    if constexpr (!DIRECT) {
      static_assert(AHEAD >= STAGES, "the first slabs travel together");
#pragma unroll
      for (int kt = 0; kt < STAGES; ++kt)
#pragma unroll
        for (int n = 0; n < PIECES; ++n) fetch(n, kt, kt);
    }
#pragma unroll
    for (int kt = 0; kt < STAGES; ++kt) {
      aim(kt);
#pragma unroll
      for (int n = 0; n < PIECES; ++n) move(n, kt, kt % AHEAD);
    }
    if constexpr (!DIRECT) {
#pragma unroll
      for (int set = 0; set < AHEAD; ++set)
#pragma unroll
        for (int n = 0; n < PIECES; ++n) fetch(n, STAGES + set, set);
    }
    arrive<(STAGES - 1) * PIECES>();
    Fragments f0, f1;
#pragma unroll
    for (int n = 0; n < READS; ++n) read(f0, n, lds, wr0, wc0, 0, lane);
    auto slab = [&](int kt, int set) {
      const char* stage = lds + stage_of(kt);
      const char* next = lds + stage_of(kt + 1);
      // first step; the second one's fragments
#pragma unroll
      for (int j = 0; j < TR; ++j) {
#pragma unroll
        for (int n = j * READS / TR; n < (j + 1) * READS / TR; ++n) read(f1, n, stage, wr0, wc0, 1, lane);
        multiply_row(f0, j, acc);
        __builtin_amdgcn_sched_barrier(0);
      }
      // Every wavefront has read slab kt, and slab kt + 1 has arrived.
      arrive<(STAGES - 2) * PIECES>();
      aim(kt + STAGES);
      // second step; the next slab's first fragments, and a slab to come into the place of this one
      // (behind the last slab zeros, rather than a branch around every move)
#pragma unroll
      for (int j = 0; j < TR; ++j) {
#pragma unroll
        for (int n = j * READS / TR; n < (j + 1) * READS / TR; ++n) read(f0, n, next, wr0, wc0, 0, lane);
#pragma unroll
        for (int n = j * PIECES / TR; n < (j + 1) * PIECES / TR; ++n) {
          move(n, kt + STAGES, set);
          fetch(n, kt + STAGES + AHEAD, set);
        }
        multiply_row(f1, j, acc);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    for (int kt = 0; kt + 1 < slabs; kt += AHEAD) {  // (register sets are numbered at compile time)
#pragma unroll
      for (int set = 0; set < AHEAD; ++set)
        if (kt + set + 1 < slabs) slab(kt + set, set);
    }
    char* last = lds + stage_of(slabs - 1);
    if (DIRECT && (LR == KC || LC == KC) && ((unsigned)k_count * E::SIZE & 15)) {
      const int left = (k_count - (slabs - 1) * SLAB_K) * E::SIZE;
      LoadR::trim(last, left, tid);
      LoadC::trim(last + LoadR::BYTES, left, tid);
      wait_lds();
      barrier();
#pragma unroll
      for (int n = 0; n < READS; ++n) read(f0, n, last, wr0, wc0, 0, lane);
    }
#pragma unroll
    for (int n = 0; n < READS; ++n) read(f1, n, last, wr0, wc0, 1, lane);
#pragma unroll
    for (int j = 0; j < TR; ++j) multiply_row(f0, j, acc);
#pragma unroll
    for (int j = 0; j < TR; ++j) multiply_row(f1, j, acc);
    wait_lds();
    wait_loads<0>();  // no load may write to LDS once the workgroup has given it back
  }

  // All but the last LATER loads to LDS of every wavefront, and all its LDS accesses, are done.
  template <int LATER>
  static __device__ __forceinline__ void arrive() {
    if constexpr (DIRECT) wait_loads<LATER>();
    wait_lds();
    barrier();
  }
};

// ---- results -------------------------------------------------------------------------------

struct Result {
  void* base;      // the tile's first element
  int64_t ld;      // in elements
  int rows, cols;  // of the tile that exist
  int type;        // kFloat32, kBFloat16, kFloat16
};

// f(a value of the type that results of E's products have).  Only those that the entry points let through.
template <class E, class F>
__device__ __forceinline__ void with_result_type(int type, F f) {
  if constexpr (std::is_void_v<typename E::Value>) {
    if (type == kFloat32) f(float{});
    else if (type == kBFloat16) f(__bf16{});
    else f(_Float16{});
  } else if constexpr (std::is_same_v<typename E::Value, float>) {
    f(float{});
  } else {
    if (type == kFloat32) f(float{});
    else f(typename E::Value{});
  }
}

// Eight consecutive values, at any address (memory takes 16 bytes anywhere).
template <class Scalar>
__device__ __forceinline__ void store_eight(void* base, int64_t at, const float (&v)[8]) {
  Scalar out[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) out[q] = (Scalar)v[q];
  __builtin_memcpy(static_cast<Scalar*>(base) + at, out, sizeof(out));
}

// What an accumulator is multiplied by: for a lane's columns, read once, and for a row.
struct Unscaled {
  template <int TC>
  struct Columns {
    __device__ __forceinline__ Columns(const Unscaled&, int, int) {}
    __device__ __forceinline__ float operator()(int, int, float, float v) const { return v; }
  };
  __device__ __forceinline__ float row(int) const { return 1.0f; }
};
// The integer sum is exact; it is rounded to fp32 once, then scaled by the token and by the channel.  A sum of up
// to 2^31 times a token's scale can leave the range although the channel's brings it back: large scales of tokens
// are applied without 2^32, which comes last.  (Nothing else can be lost on the way: an integer times a scale,
// subnormal ones too, is no smaller than the scale.)
struct TokenScale {
  float scale, rest;
  __device__ __forceinline__ explicit TokenScale(float s) {
    const bool large = __builtin_fabsf(s) >= 0x1p96f;
    scale = large ? s * 0x1p-32f : s;
    rest = large ? 0x1p32f : 1.0f;
  }
  __device__ __forceinline__ float operator()(int sum, float channel) const { return (float)sum * scale * channel * rest; }
};
struct TokenChannel {
  const float* token;
  const float* channel;
  template <int TC>
  struct Columns {
    float channel[TC / 2][8];
    __device__ __forceinline__ Columns(const TokenChannel& s, int c0, int cols) {  // columns c0 + 32 i .. + 7
#pragma unroll
      for (int i = 0; i < TC / 2; ++i)
#pragma unroll
        for (int q = 0; q < 8; ++q) channel[i][q] = s.channel[min(c0 + 32 * i + q, cols - 1)];
    }
    __device__ __forceinline__ float operator()(int i, int q, TokenScale token, int v) const { return token(v, channel[i][q]); }
  };
  __device__ __forceinline__ TokenScale row(int r) const { return TokenScale(token[r]); }
};

// A wavefront's results go through its share of LDS, so that it stores whole rows of its part of the tile
// (64 bytes and more) instead of 16 bytes here and there.  No other wavefront's share is touched: no barrier.
constexpr int kStoreBytes = 8192;  // of LDS for each wavefront

template <class Cfg, class Out, int A, class Acc, class Scale>
__device__ __forceinline__ void store_tile_as(const Result& o, const Acc (&acc)[A][Cfg::TC], const Scale& scale, char* lds) {
  constexpr int WIDTH = Cfg::TC * 16 * (int)sizeof(Out), PIECES = WIDTH / 16;  // bytes and 16-byte pieces of a row
  constexpr int FIT = kStoreBytes / (16 * WIDTH), AT_ONCE = FIT < A ? FIT : A;  // fragments of rows that fit
  constexpr int VALUES = 16 / (int)sizeof(Out);
  static_assert(FIT >= 1 && PIECES <= 64 && AT_ONCE * 16 * PIECES >= 64, "store layout");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m = lane & 15, g = lane >> 4;
  const int wr = wave % Cfg::WR, wc0 = (wave / Cfg::WR) * (Cfg::TC * 16);
  char* mine = lds + wave * kStoreBytes;
  const typename Scale::template Columns<Cfg::TC> columns(scale, wc0 + 8 * g, o.cols);
#pragma unroll
  for (int j0 = 0; j0 < A; j0 += AT_ONCE) {
#pragma unroll
    for (int jj = 0; jj < AT_ONCE; ++jj) {
      if (j0 + jj >= A) continue;
      const auto row = scale.row(min((Cfg::WR * (j0 + jj) + wr) * 16 + m, o.rows - 1));
#pragma unroll
      for (int i = 0; i < Cfg::TC; i += 2) {
        Out v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = (Out)columns(i >> 1, q, row, acc[(j0 + jj) % A][i + (q >> 2)][q & 3]);
#pragma unroll
        for (int h = 0; h < 8 / VALUES; ++h) {
          const int piece = (16 * i + 8 * g) / VALUES + h;
          i32x4 w;
          __builtin_memcpy(&w, v + h * VALUES, 16);
          *reinterpret_cast<i32x4*>(mine + (jj * 16 + m) * WIDTH + ((piece ^ (m & (PIECES - 1) & 7)) << 4)) = w;
        }
      }
    }
    keep_order();
    constexpr int ROWS = 64 / PIECES;  // of one store
#pragma unroll
    for (int s = 0; s < AT_ONCE * 16 / ROWS; ++s) {
      if (j0 + s * ROWS / 16 >= A) continue;
      const int row = s * ROWS + lane / PIECES, piece = lane % PIECES;
      const i32x4 w = *reinterpret_cast<const i32x4*>(mine + row * WIDTH + ((piece ^ (row & (PIECES - 1) & 7)) << 4));
      const int r = (Cfg::WR * (j0 + row / 16) + wr) * 16 + row % 16, c = wc0 + piece * VALUES;
      if (r >= o.rows || c >= o.cols) continue;
      Out* to = static_cast<Out*>(o.base) + (int64_t)r * o.ld + c;
      if (c + VALUES <= o.cols) {
        __builtin_memcpy(to, &w, 16);  // (memory takes 16 bytes anywhere)
      } else {
        Out v[VALUES];
        __builtin_memcpy(v, &w, 16);
#pragma unroll
        for (int q = 0; q < VALUES; ++q)
          if (c + q < o.cols) to[q] = v[q];
      }
    }
    keep_order();
  }
}

template <class E, class Cfg, int A, class Scale>
__device__ __forceinline__ void store_tile(const Result& o, const typename E::Acc (&acc)[A][Cfg::TC], const Scale& scale,
                                           char* lds) {
  barrier();  // every wavefront is done with the operands
  with_result_type<E>(o.type, [&](auto value) { store_tile_as<Cfg, decltype(value), A>(o, acc, scale, lds); });
}

// ---- kernels -------------------------------------------------------------------------------

struct RowProblem {
  RowGroups groups;
  const char* r;       // tokens x k
  const char* c;       // experts x (columns x k, or k x columns)
  int64_t ldr, ldc;    // bytes
  int64_t stride_c;    // bytes from one expert's matrix to the next
  int cols, k;
  int tiles_c;
  void* y;
  int64_t ldy;         // elements
  int out_type;
  const float* token_scale;    // 8-bit product only
  const float* channel_scale;
};

__device__ __forceinline__ int type_bytes(int type) { return type == kFloat32 ? 4 : 2; }

// The tile with A fragments of rows for each row of wavefronts.
template <class E, Layout LC, Source S, class Cfg, int A>
__device__ __forceinline__ void row_tile(const RowProblem& p, const RowTile& tile, int c0, char* lds) {
  Operand r, c;
  r.base = p.r + (int64_t)tile.row * p.ldr;
  r.ld = p.ldr;
  r.valid = tile.rows;
  c.base = p.c + (int64_t)tile.expert * p.stride_c + (LC == KC ? (int64_t)c0 * p.ldc : (int64_t)c0 * E::SIZE);
  c.ld = p.ldc;
  c.valid = min(Cfg::BC, p.cols - c0);
  typename E::Acc acc[A][Cfg::TC];
  TileProduct<E, KC, LC, S, Cfg, A>::run(r, c, tile.expert >= p.groups.experts ? 0 : p.k, lds, acc);
  Result o;
  o.base = static_cast<char*>(p.y) + ((int64_t)tile.row * p.ldy + c0) * type_bytes(p.out_type);
  o.ld = p.ldy;
  o.rows = tile.rows;
  o.cols = c.valid;
  o.type = p.out_type;
  if constexpr (E::SIZE == 1)
    store_tile<E, Cfg, A>(o, acc, TokenChannel{p.token_scale + tile.row, p.channel_scale + c0}, lds);
  else
    store_tile<E, Cfg, A>(o, acc, Unscaled{}, lds);
}

template <class E, Layout LC, Source S, class Cfg, int A>
__device__ __forceinline__ void row_tile_at_least(const RowProblem& p, const RowTile& tile, int c0, int fragments, char* lds) {
  constexpr int LESS = A > 4 ? A - 1 : A - 2;  // 8, 7, 6, 5, 4, 2
  if constexpr (LESS >= 1)
    if (fragments <= LESS) return row_tile_at_least<E, LC, S, Cfg, LESS>(p, tile, c0, fragments, lds);
  row_tile<E, LC, S, Cfg, A>(p, tile, c0, lds);
}

template <class E, Layout LC, Source S, class Cfg>
__global__ __launch_bounds__(Cfg::NT) void row_product_kernel(RowProblem p) {
  __shared__ __attribute__((aligned(1024))) char lds[TileProduct<E, KC, LC, S, Cfg>::LDS_BYTES];
  constexpr int GRAIN = 16 * Cfg::WR;
  RowTile tile;
  int tile_c;
  if (!locate_rows<Cfg::BR, GRAIN>(p.groups, p.tiles_c, blockIdx.x, tile, tile_c)) return;
  row_tile_at_least<E, LC, S, Cfg, Cfg::TR>(p, tile, tile_c * Cfg::BC, (tile.rows + GRAIN - 1) / GRAIN, lds);
}

// ---- few rows ------------------------------------------------------------------------------
//
// With a handful of rows for an expert the product is the reading of its weights (k contiguous).  A
// workgroup has 32 outputs and up to 32 rows of one expert; its eight wavefronts take every eighth 128
// bytes of k, straight from memory to the matrix instruction's registers: no wavefront waits for
// another one before the end, so all of a compute unit's loads are in flight at once.  The eight sums
// meet in LDS and are added in order.  One row, 11008 x 4096 in 8 bits: 12.2 us = 3.7 TB/s; one row, 4096 x
// 4096 bf16: 13.1 us against 19.7 on 32 x 128 tiles.
struct FewTile {
  static constexpr int BR = 32, BC = 32, WAVES = 8, NT = 64 * WAVES;
  static constexpr int BATCH = 4;  // steps of 128 bytes that a wavefront has in flight
};

template <class E, int A>
__device__ __forceinline__ void few_rows_tile(const RowProblem& p, const RowTile& tile, int c0, int k, char* lds) {
  using Acc = typename E::Acc;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int m = lane & 15, g = lane >> 4;
  const int64_t bytes = (int64_t)k * E::SIZE;
  const int cols = min(FewTile::BC, p.cols - c0);
  // (rows and columns behind the last one are read as the last one again and not stored)
  const char* w[2];
  const char* x[A];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = p.c + (int64_t)tile.expert * p.stride_c + (int64_t)(c0 + min(16 * i + m, cols - 1)) * p.ldc + g * 16;
#pragma unroll
  for (int j = 0; j < A; ++j) x[j] = p.r + (int64_t)(tile.row + min(16 * j + m, tile.rows - 1)) * p.ldr + g * 16;
  Acc acc[A][2];
#pragma unroll
  for (int j = 0; j < A; ++j) acc[j][0] = acc[j][1] = Acc{0, 0, 0, 0};
  const int steps = (int)(bytes >> 7);  // whole ones
  int s = wave;
  for (; s + (FewTile::BATCH - 1) * FewTile::WAVES < steps; s += FewTile::BATCH * FewTile::WAVES) {
    i32x4 fw[FewTile::BATCH][2][2], fx[FewTile::BATCH][A][2];
#pragma unroll
    for (int b = 0; b < FewTile::BATCH; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t at = (int64_t)(s + b * FewTile::WAVES) * 128 + h * 64;
#pragma unroll
        for (int i = 0; i < 2; ++i) __builtin_memcpy(&fw[b][i][h], w[i] + at, 16);
#pragma unroll
        for (int j = 0; j < A; ++j) __builtin_memcpy(&fx[b][j][h], x[j] + at, 16);
      }
#pragma unroll
    for (int b = 0; b < FewTile::BATCH; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < A; ++j)
#pragma unroll
          for (int i = 0; i < 2; ++i) acc[j][i] = E::mma(fw[b][i][h], fx[b][j][h], acc[j][i]);
  }
  for (; s * (int64_t)128 < bytes; s += FewTile::WAVES) {  // the remaining steps, the last of them perhaps cut short
    i32x4 fw[2][2], fx[A][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t at = (int64_t)s * 128 + h * 64;
      const int count = (int)min((int64_t)16, bytes - at - g * 16);
#pragma unroll
      for (int i = 0; i < 2; ++i) fw[i][h] = load_bytes(w[i] + at, count);
#pragma unroll
      for (int j = 0; j < A; ++j) fx[j][h] = load_bytes(x[j] + at, count);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < A; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[j][i] = E::mma(fw[i][h], fx[j][h], acc[j][i]);
  }
  // sums[wave][row][output], outputs padded so that a fragment's four rows of lanes fall on different banks
  using Sum = std::conditional_t<E::SIZE == 1, int, float>;
  constexpr int STRIDE = FewTile::BC + 4;
  Sum* sums = reinterpret_cast<Sum*>(lds);
#pragma unroll
  for (int j = 0; j < A; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<Acc*>(sums + ((wave * A + j) * 16 + m) * STRIDE + 16 * i + 4 * g) = acc[j][i];
  __syncthreads();
#pragma unroll
  for (int at = tid; at < A * 16 * FewTile::BC; at += FewTile::NT) {
    const int r = at / FewTile::BC, c = at % FewTile::BC;
    if (r >= tile.rows || c >= cols) continue;
    Sum v = 0;
#pragma unroll
    for (int q = 0; q < FewTile::WAVES; ++q) v += sums[(q * A * 16 + r) * STRIDE + c];
    float out;
    if constexpr (E::SIZE == 1) out = TokenScale(p.token_scale[tile.row + r])(v, p.channel_scale[c0 + c]);
    else out = v;
    const int64_t to = (int64_t)(tile.row + r) * p.ldy + c0 + c;
    with_result_type<E>(p.out_type, [&](auto value) { static_cast<decltype(value)*>(p.y)[to] = (decltype(value))out; });
  }
}

template <class E>
__global__ __launch_bounds__(FewTile::NT) void few_rows_kernel(RowProblem p) {
  __shared__ __attribute__((aligned(16))) char lds[FewTile::WAVES * FewTile::BR * (FewTile::BC + 4) * 4];
  RowTile tile;
  int tile_c;
  if (!locate_rows<FewTile::BR, 16>(p.groups, p.tiles_c, blockIdx.x, tile, tile_c)) return;
  const int k = tile.expert >= p.groups.experts ? 0 : p.k, c0 = tile_c * FewTile::BC;
  if (tile.rows <= 16) few_rows_tile<E, 1>(p, tile, c0, k, lds);
  else few_rows_tile<E, 2>(p, tile, c0, k, lds);
}

struct SumProblem {
  RowGroups groups;
  const char* r;          // tokens x rows
  const char* c;          // tokens x cols
  int64_t ldr, ldc;       // bytes
  int rows, cols;
  int tiles_r, tiles_c;
  void* d;
  int64_t ldd, stride_d;  // elements
  int out_type;
  int parts;              // > 1: each expert's rows are cut into that many parts, whose sums go to `partials`
  float* partials;        // [parts][experts][rows][cols]
};

struct SumTile {
  int expert, part;
  int begin, end;  // rows to sum over
  int tile_r, tile_c;
};

// Workgroup -> expert, part and tile of its matrix.  Experts differ in their rows, so each one's tiles
// are spread over all XCDs, and each XCD has a contiguous part of them.  Up to 64 experts are taken in
// the order of their rows, the most first: the last workgroups to start are then short ones.
__device__ __forceinline__ bool locate_sum(const SumProblem& p, unsigned wg, SumTile& tile) {
  const unsigned tiles_r = p.tiles_r, tiles_c = p.tiles_c, tiles = tiles_r * tiles_c;
  const unsigned chunk = (tiles + 7) >> 3;
  const unsigned slot = wg >> 3, nth = slot / chunk;
  const unsigned t = (wg & 7) * chunk + slot - nth * chunk;
  const unsigned place = nth / (unsigned)p.parts;
  tile.part = __builtin_amdgcn_readfirstlane((int)(nth - place * p.parts));
  const int experts = p.groups.experts;
  if (place >= (unsigned)experts || t >= tiles) return false;
  constexpr unsigned GR = 8;
  const unsigned per = GR * tiles_c;
  const unsigned band = t / per, in_band = t - band * per;
  const unsigned rows = min(GR, tiles_r - band * GR);
  const unsigned column = in_band / rows;
  tile.tile_r = __builtin_amdgcn_readfirstlane((int)(band * GR + in_band - column * rows));
  tile.tile_c = __builtin_amdgcn_readfirstlane((int)column);
  int begin, end, expert = (int)place;
  if (experts > 1 && experts <= 64) {
    const int lane = threadIdx.x & 63;
    begin = end = 0;
    if (lane < experts) group_rows(p.groups, lane, begin, end);
    const int count = end - begin;
    int before = 0;
    for (int e = 0; e < experts; ++e) {
      const int other = __builtin_amdgcn_readlane(count, e);
      before += other > count || (other == count && e < lane);
    }
    expert = __ffsll((unsigned long long)__ballot(lane < experts && before == (int)place)) - 1;
    expert = __builtin_amdgcn_readfirstlane(expert);
    begin = __builtin_amdgcn_readlane(begin, expert);
    end = __builtin_amdgcn_readlane(end, expert);
  } else {
    group_rows(p.groups, expert, begin, end);
    begin = __builtin_amdgcn_readfirstlane(begin);
    end = __builtin_amdgcn_readfirstlane(end);
  }
  tile.expert = __builtin_amdgcn_readfirstlane(expert);
  if (p.parts > 1) {  // in units of 64 rows
    const unsigned slabs = (unsigned)(end - begin + 63) >> 6, parts = p.parts, part = tile.part;
    const unsigned each = slabs / parts, larger = slabs - each * parts;
    const int first = (int)(part * each + min(part, larger)) << 6;
    const int last = first + ((int)(each + (part < larger ? 1 : 0)) << 6);
    end = min(end, begin + last);
    begin = min(end, begin + first);
  }
  tile.begin = __builtin_amdgcn_readfirstlane(begin);
  tile.end = __builtin_amdgcn_readfirstlane(end);
  return true;
}

// Where a tile's sums go: the expert's matrix, or this part's.
__device__ __forceinline__ Result sum_result(const SumProblem& p, const SumTile& tile, int r0, int c0) {
  Result o;
  o.ld = p.parts > 1 ? p.cols : p.ldd;
  o.type = p.parts > 1 ? (int)kFloat32 : p.out_type;
  const int64_t at = (int64_t)r0 * o.ld + c0;
  if (p.parts > 1) o.base = p.partials + ((int64_t)tile.part * p.groups.experts + tile.expert) * p.rows * p.cols + at;
  else o.base = static_cast<char*>(p.d) + ((int64_t)tile.expert * p.stride_d + at) * type_bytes(p.out_type);
  return o;
}

template <class E, Source S, class Cfg>
__global__ __launch_bounds__(Cfg::NT) void sum_product_kernel(SumProblem p) {
  using Product = TileProduct<E, XC, XC, S, Cfg>;
  __shared__ __attribute__((aligned(1024))) char lds[Product::LDS_BYTES];
  SumTile tile;
  if (!locate_sum(p, blockIdx.x, tile)) return;
  const int r0 = tile.tile_r * Cfg::BR, c0 = tile.tile_c * Cfg::BC;
  Operand r, c;
  r.base = p.r + (int64_t)tile.begin * p.ldr + (int64_t)r0 * E::SIZE;
  r.ld = p.ldr;
  r.valid = min(Cfg::BR, p.rows - r0);
  c.base = p.c + (int64_t)tile.begin * p.ldc + (int64_t)c0 * E::SIZE;
  c.ld = p.ldc;
  c.valid = min(Cfg::BC, p.cols - c0);
  typename E::Acc acc[Cfg::TR][Cfg::TC];
  Product::run(r, c, tile.end - tile.begin, lds, acc);
  Result o = sum_result(p, tile, r0, c0);
  o.rows = r.valid;
  o.cols = c.valid;
  store_tile<E, Cfg, Cfg::TR>(o, acc, Unscaled{}, lds);
}

// ---- 8-bit codes ---------------------------------------------------------------------------

// Eight values of a row from column c on; behind the last column zeros.
template <class T>
__device__ __forceinline__ void load_eight(const T* row, int c, int cols, bool vec, float (&v)[8]) {
  if (vec && c + 8 <= cols) {
    constexpr int N = 8 * sizeof(T) / 16;
    i32x4 piece[N];
#pragma unroll
    for (int i = 0; i < N; ++i) piece[i] = reinterpret_cast<const i32x4*>(row + c)[i];
    T t[8];
    __builtin_memcpy(t, piece, sizeof(t));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? (float)row[c + i] : 0.0f;
  }
}

__device__ __forceinline__ void store_codes(int8_t* row, int c, int cols, bool vec, const int (&q)[8]) {
  if (vec && c + 8 <= cols) {
    unsigned w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i >> 2] |= (unsigned)(q[i] & 255) << (8 * (i & 3));
    *reinterpret_cast<uint2*>(row + c) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) row[c + i] = (int8_t)q[i];
  }
}

// Largest magnitude so far, as the bits of its float: magnitudes compare like their bits as unsigned
// numbers, and infinities and NaN compare above every finite one, so that one maximum finds both.
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

constexpr int kRowRegisters = 4;  // chunks of eight values that a thread keeps between the two passes

// codes = round(127 x / top), scale = top / 127, with top the largest magnitude of the row.  A row of
// zeros has scale 0; a row that holds an infinity or NaN has scale NaN and codes 0, so that everything
// it stands for is NaN.  TPR threads take a row and keep up to 32 values each, so that a row of up to 8192
// is read once.  Bound by memory: 8192 x 4096 bf16 in 25.5 us = 4.0 TB/s, in 20 us if the last-level cache has it.
template <class T, int TPR>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* x, int64_t ldx, int rows, int cols, int vec_x,
                                                            int8_t* codes, int64_t ldq, int vec_q, float* scales) {
  constexpr int ROWS = 256 / TPR;
  const int row = blockIdx.x * ROWS + threadIdx.x / TPR;
  const int t = threadIdx.x % TPR;
  const bool mine = row < rows;
  const T* in = x + (int64_t)(mine ? row : 0) * ldx;
  const int chunks = mine ? (cols + 7) / 8 : 0;
  float kept[kRowRegisters][8];
  unsigned top = 0;
#pragma unroll
  for (int j = 0; j < kRowRegisters; ++j) {
    const int c = t + j * TPR;
    if (c < chunks) {
      load_eight(in, c * 8, cols, vec_x, kept[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, magnitude(kept[j][i]));
    }
  }
  for (int c = t + kRowRegisters * TPR; c < chunks; c += TPR) {
    float v[8];
    load_eight(in, c * 8, cols, vec_x, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, magnitude(v[i]));
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, d));
  if constexpr (TPR > 64) {
    __shared__ unsigned part[TPR / 64];
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) top = max(top, part[w]);
  }
  if (!mine) return;
  const bool finite = top < 0x7f800000u;
  const float largest = __uint_as_float(top);
  // Both the row and its maximum are brought to around 1 by a power of two, so that neither 127 x nor
  // the reciprocal leaves the range.  For 16-bit inputs 127 x is exact, one correction of the quotient by its
  // remainder gives the correctly rounded one, and none that is not halfway between two codes is within that
  // rounding of it.  For fp32 inputs 127 x is a + low, and where the quotient is nearly halfway the exact
  // remainder a + low - code * b decides: it may be b / 2 at most.  Without low it is a multiple of the last
  // place of b or a, and so is its distance to b / 2, which leaves both exact (8192 x 4096 in
  // fp32: 34.0 us, 33.6 without it).
  int power = 0;
  const float b = frexpf(finite ? largest : 0.0f, &power);
  const float inverse = b > 0.0f ? 1.0f / b : 0.0f;
  if (t == 0) scales[row] = finite ? largest / 127.0f : __uint_as_float(0x7fc00000u);
  int8_t* out = codes + (int64_t)row * ldq;
  auto quantize = [&](const float (&v)[8], int c) {
    int q[8];
    bool halfway = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = 127.0f * ldexpf(v[i], -power);
      float r = a * inverse;
      if constexpr (sizeof(T) == 4) halfway |= __builtin_fabsf(r - __builtin_rintf(r)) > 0.4999f;  // (r is off by 2.3e-5 at most)
      else r = __builtin_fmaf(__builtin_fmaf(-r, b, a), inverse, r);
      q[i] = finite ? (int)__builtin_rintf(r) : 0;
    }
    if (halfway && finite) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = ldexpf(v[i], -power), a = 127.0f * x, low = __builtin_fmaf(127.0f, x, -a);
        const float over = __builtin_fmaf(-(float)q[i], b, a), above = over - 0.5f * b, below = over + 0.5f * b;
        const bool odd = q[i] & 1;
        if (above > -low || (above == -low && odd)) ++q[i];
        else if (below < -low || (below == -low && odd)) --q[i];
      }
    }
    store_codes(out, c * 8, cols, vec_q, q);
  };
#pragma unroll
  for (int j = 0; j < kRowRegisters; ++j) {
    const int c = t + j * TPR;
    if (c < chunks) quantize(kept[j], c);
  }
  for (int c = t + kRowRegisters * TPR; c < chunks; c += TPR) {
    float v[8];
    load_eight(in, c * 8, cols, vec_x, v);
    quantize(v, c);
  }
}

constexpr int kCheckpointBlock = 128;  // columns that share an exponent

// Activation checkpoints: with 2^(p-1) <= top < 2^p the largest magnitude of 128 columns of a row, the
// step is 2^(p-7) (at least 2^-126; 2^-24, the smallest fp16 value, for fp16) and the codes are
// round(x / step) held to -127..127; the exponent is stored with 127 added, 255 marks a block that holds
// an infinity or NaN.  The step is a power of two because it stands inside the weight gradient's sum:
// code * step is then exact in 16 bits, and so is its product with a 16-bit gradient in fp32.  Sixteen lanes
// take a block.  Bound by memory: 8192 x 4096
// bf16 in 24 us = 4.2 TB/s (21.5 us if the last-level cache has it; restored in 18.7 us = 5.4 TB/s).
template <class T>
__global__ __launch_bounds__(256) void checkpoint_kernel(const T* x, int64_t ldx, int64_t rows, int cols, int blocks,
                                                         int vec_x, int8_t* codes, int64_t ldq, int vec_q,
                                                         uint8_t* exponents, int64_t ld_exp, int lowest) {
  const int64_t block = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
  const int64_t row = block / blocks;
  if (row >= rows) return;  // (whole groups of 16 lanes leave)
  const int in_row = (int)(block - row * blocks), t = threadIdx.x & 15;
  const int c = in_row * kCheckpointBlock + t * 8;
  float v[8];
  load_eight(x + row * ldx, c, cols, vec_x, v);
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, magnitude(v[i]));
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, d));
  const bool finite = top < 0x7f800000u;
  // exponent field of top, minus 6, is that of 2^(p-7); a subnormal top has field 0 and takes the lowest
  const int code = max((int)(top >> 23) - 6, lowest);
  const float per_step = __uint_as_float((unsigned)(254 - code) << 23);  // 2^(127 - code)
  int q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = finite ? (int)fminf(fmaxf(__builtin_rintf(v[i] * per_step), -127.0f), 127.0f) : 0;
  store_codes(codes + row * ldq, c, cols, vec_q, q);
  if (t == 0) exponents[row * ld_exp + in_row] = (uint8_t)(finite ? code : 255);
}

template <class T>
__global__ __launch_bounds__(256) void restore_kernel(const int8_t* codes, int64_t ldq, int vec_q, const uint8_t* exponents,
                                                      int64_t ld_exp, int64_t rows, int cols, int pieces, T* x, int64_t ldx,
                                                      int vec_x) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = at / pieces;
  if (row >= rows) return;
  const int c = (int)(at - row * pieces) * 8;
  const int8_t* in = codes + row * ldq;
  int8_t q[8];
  if (vec_q && c + 8 <= cols) {
    __builtin_memcpy(q, __builtin_assume_aligned(in + c, 8), 8);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = c + i < cols ? in[c + i] : 0;
  }
  const float step = exponent_value(exponents[row * ld_exp + c / kCheckpointBlock]);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)q[i] * step;
  T* out = x + row * ldx;
  if (vec_x && c + 8 <= cols) {
    store_eight<T>(out, c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) out[c + i] = (T)v[i];
  }
}

}  // namespace soapmi
