// What the kernels of attention over drafted trees share: their parameters, how the rows of a step are dealt out, and which keys a row sees.
//
// Entry r of a step brings n nodes, its rows entry_starts[r] .. entry_starts[r + 1] - 1, numbered from 0; parents[row] is the number of the
// parent (lower than the node's own) or -1.  context[r] keys are cached in front of them; node i's key lies behind those, at context + i,
// while its position in the text is context + depth(i), depth being how many ancestors it has.  A node sees the cached keys, its ancestors
// and itself; with a window only those whose position is above its own minus the window.
//
// A row of the kernels is a (node, query head of the KV head's group): row i of an entry and KV head is head i % group of node i / group.
// Rows are cut into tiles of ROWS, tiles are numbered through over the entries, and a tile's keys are cut into parts, each a unit of work:
// its partial result (unnormalised output, reference, sum; base 2) goes to scratch memory and a merge kernel adds the parts up in order.  A
// tile with one part is written at once.
#pragma once
#include "common.cuh"

namespace tree {

struct Params {
    const void* q;
    long long ldq;
    const void* k_cache;
    const void* v_cache;
    long long page_stride, head_stride;
    const int* block_table;
    int table_stride, table_pages, num_pages;
    const int* entry_starts;
    const int* context;
    const int* parents;
    void* out;
    long long ldo;
    int rows, entries, num_heads, num_kv_heads, head_dim, page_size, window;
    float scale;
    int max_parts, part_tiles;       // a tile's keys are cut into min(max_parts, key tiles / part_tiles) parts, one at least
    float* partial_o;                // [parts][rows * heads][head_dim]
    float* partial_ml;               // [parts][rows * heads][2]
    int* status;
};

// An entry's place in the step.
struct Entry {
    int first, n, context;
};
// Entry r as the metadata has it; n = 0 where its rows cannot be what they say (and a status bit).
__device__ __forceinline__ Entry sound(const Params& p, int first, int end, int context) {
    Entry e = {first, end - first, context};
    if (first < 0 || end < first || end > p.rows || context < 0 || context > 0x7fffffff - e.n) {
        atomicOr(p.status, EG_STATUS_BAD_TREE);
        e.n = 0;
    }
    return e;
}

// A node's parent; one that cannot be is none, and a status bit.
__device__ __forceinline__ int parent_of(const Params& p, const Entry& e, int i) {
    const int up = p.parents[e.first + i];
    if (up < -1 || up >= i) {
        atomicOr(p.status, EG_STATUS_BAD_TREE);
        return -1;
    }
    return up;
}

// The entry whose tile number `tile` is, counting ceil(n * group / row_tile) tiles an entry, and the tile's number within it; false: there
// is none.  For a whole warp: 32 entries at a time, in one trip to memory.
__device__ __forceinline__ bool find_tile(const Params& p, int tile, int row_tile, int& r, Entry& e, int& within) {
    const int lane = threadIdx.x & 31, group = p.num_heads / p.num_kv_heads;
    for (int base = 0; base < p.entries; base += 32) {
        Entry mine = {0, 0, 0};
        if (base + lane < p.entries) mine = sound(p, p.entry_starts[base + lane], p.entry_starts[base + lane + 1], p.context[base + lane]);
        const int tiles = (int)(((long long)mine.n * group + row_tile - 1) / row_tile);
        int upto = tiles;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int below = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += below;
        }
        const unsigned here = __ballot_sync(0xffffffffu, tile < upto);
        if (here) {
            const int who = __ffs(here) - 1;
            r = base + who;
            e.first = __shfl_sync(0xffffffffu, mine.first, who);
            e.n = __shfl_sync(0xffffffffu, mine.n, who);
            e.context = __shfl_sync(0xffffffffu, mine.context, who);
            within = tile - __shfl_sync(0xffffffffu, upto - tiles, who);
            return true;
        }
        tile -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

// A tile's first key that any of its rows may see, and the key behind its last one.
__device__ __forceinline__ int first_key(const Params& p, const Entry& e) { return p.window > 0 && e.context >= p.window ? e.context - p.window + 1 : 0; }

__device__ __forceinline__ int parts_of(const Params& p, int key_tiles) { return max(1, min(p.max_parts, key_tiles / p.part_tiles)); }

// The kernel in attention_tree_mma.cu (16, 32 or 64 rows a CTA, key tiles of 64).  Its caller has checked what it takes.
int launch_mma(cudaStream_t stream, const Params& p, int row_tile, int tiles);

}  // namespace tree
