// Attention over a paged pool in 8 bits (include/imba_b200.h, imba_attend):
// what the plan pass writes and the kernels read.
#pragma once

#include "attn_common.cuh"
#include "cache8.cuh"

namespace imba {

// A tile is up to kTileRows * rt query rows of one segment, flattened with
// the query heads that share a key / value head (row i, head j of the group:
// i * share + j).  An item is a tile and a run of its group's pages; a unit
// is an item and a key / value head.
constexpr int kTileRows = 8;
constexpr int kUnitWarps = 8;  // warps of a CTA
constexpr int kTileGroups = 16;  // rt of the tcgen05 kernel's tiles of 128 rows

// CTAs an SM, by what a lane's rows take in registers (four of 64 registers
// for one group of rows: 42 us against 36 with three of 80 for 1,024 games).
// The tcgen05 kernel's are what shared memory holds.
constexpr int attend8_ctas(int dqk, int rt) {
  return rt == kTileGroups ? (dqk > 64 ? 1 : 2) : dqk > 64 ? (rt == 1 ? 2 : 1) : rt == 1 ? 3 : rt == 2 || dqk == 32 ? 2 : 1;
}

// Bounds that keep a bias column, key - position + max_pos - 1, within 32 bits:
// the pages of a step's lists (2^30 tokens), and the largest max_pos.  A
// position below -kMostPos puts every key into the last column, as it does.
constexpr int kMostPages = 1 << 26;
constexpr int kMostPos = 1 << 28;
// Extra keys of a step: the rows of a warp (24 at most) can each ask for all,
// and their sum is 32 bits.
constexpr int kMostExtra = 1 << 26;

struct AttendRow {  // one flattened row of a tile
  int row;          // -1: none
  int vis;          // visible tokens of the page list
  int pos;          // position (bias)
  int head;         // query head within its group
};
struct AttendItem {
  int tile;
  int list;    // first entry of the item's pages in group_pages
  int pages;   // how many
  int key0;    // position of their first token
  int part;    // scratch slot of the item's partial result, -1: the tile is not split
  int splits;  // items of the tile
  int minvis;  // tokens that every row of the tile sees
  int index;   // which of them this is (the first takes the rows' extra keys)
};

struct AttendShape {
  int share;        // query heads per key / value head
  int rt;           // 8-row groups of a tile: 1, 2, 3 or kTileGroups
  int warps;        // warps that share a unit: 1 or kUnitWarps
  int tile_rows;    // kTileRows * rt
  int max_tiles;
  int max_items;
  int max_parts;
  int min_pages;    // pages of a split item, at least
  int target;       // items that splitting aims at
  int waves;        // how many times the resident CTAs that is
};

// Plan memory, in this order, each part aligned to 256 bytes.
struct AttendPlan {
  int* head;             // [0] items
  int* tile_off;         // [S + 1] first tile of each segment
  int4* tiles;           // {segment, first flattened row, rows, visible pages}
  AttendItem* items;
  AttendRow* rows;       // [max_tiles][tile_rows]
  int* done;             // [max_tiles][H][8] items of a split tile (or of a part of its rows) that have finished
  float2* ml;            // [max_parts][H][tile_rows] maximum and sum
  float* o;              // [max_parts][H][tile_rows][d_v] averages
  size_t bytes;
};

// most: items that splitting may add at most (an imba_step's workspace is
// sized by its rows alone).
AttendShape attend_shape(const imba_cache_desc& c, const imba_attend_desc& r, int64_t most = INT64_MAX);
// The largest plan of a step of `rows` rows, with most = attend_step_most(rows).
inline int64_t attend_step_most(int64_t rows) { return rows + 8; }
size_t attend_step_bytes(const imba_cache_desc& c, int32_t rows);
AttendPlan attend_plan_view(const imba_cache_desc& c, const imba_attend_desc& r, const AttendShape& sh, void* base);

struct AttendArgs {
  Cache8 cache;
  AttendPlan plan;
  AttendShape shape;
  imba_attend_desc rows;
  imba_attend_args call;
};

template <typename T>
cudaError_t launch_attend8(const imba_cache_desc& c, const AttendArgs& a, cudaStream_t s);
cudaError_t launch_attend8_tile(const imba_cache_desc& c, const AttendArgs& a, cudaStream_t s);
cudaError_t launch_attend_plan(const imba_cache_desc& c, const imba_attend_desc& r, const AttendShape& sh,
                               const AttendPlan& p, cudaStream_t s);
imba_status_t validate_cache(const imba_cache_desc* c);
imba_status_t validate_pool(const imba_pool_desc* pool);

}  // namespace imba
