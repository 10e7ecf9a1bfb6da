// Entries of a CSR matrix grouped by column (a router's choices by expert), as products with a matrix per column take them:
// slots in tiles of 128, a tile's all of one column, the columns ascending, a column's last tile filled up with -1.
#pragma once
#include "common.cuh"

namespace cb200 {

static const int GROUP_TILE = 128, MOST_GROUPS = 1024;

// Where things are in the caller's int32 array.  `bad` entries (their column lies outside) are no tile's; the last `bad` elements of order are
// their numbers.
struct Groups {
    int *head;                   // tiles, bad, status (not 0: a wait ran out)
    int *counts, *first;         // of each column: entries, first tile (and one more: the number of tiles)
    int *column;                 // of each tile
    int *order, *token;          // of each slot: the entry, its row
    int64_t slots;
    int ngroups;
};
static const int GROUP_HEAD = 16;

inline int64_t group_tiles(int64_t nnz, int64_t ngroups) { return nnz / GROUP_TILE + (nnz < ngroups ? nnz : ngroups) + 1; }
inline int64_t group_size(int64_t nnz, int64_t ngroups)
{
    const int64_t tiles = group_tiles(nnz, ngroups);
    return GROUP_HEAD + (ngroups + 3) / 4 * 4 + (ngroups + 4) / 4 * 4 + (tiles + 3) / 4 * 4 + 2 * tiles * GROUP_TILE;
}
inline Groups groups_in(int *plan, int64_t nnz, int64_t ngroups)
{
    const int64_t tiles = group_tiles(nnz, ngroups);
    Groups g;
    g.head = plan;
    g.counts = plan + GROUP_HEAD;
    g.first = g.counts + (ngroups + 3) / 4 * 4;
    g.column = g.first + (ngroups + 4) / 4 * 4;
    g.order = g.column + (tiles + 3) / 4 * 4;
    g.slots = tiles * GROUP_TILE;
    g.token = g.order + g.slots;
    g.ngroups = (int)ngroups;
    return g;
}

}  // namespace cb200
