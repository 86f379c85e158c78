// What a step over trees of drafted tokens does behind the model: the walk to the drafted tokens that the model agrees with, and
// the move of their keys and values to where they belong.
//
// A tree's nodes are the rows entry_starts[r] .. entry_starts[r + 1] - 1 of the step, numbered from 0 in their order; parents[row] is the
// number of a node's parent in the same entry (lower than its own), -1 for a node without one.  Node 0 is the entry's last token that is
// known already; the others are drafts.
#include "common.cuh"
#include "tree_args.h"

namespace {

constexpr int ACCEPT_WARPS = 4;

// The walk: from node 0 to the first child (in the order of the rows) that bears the token which the model answered at the node, and so
// on.  Children come behind their parents, so one warp passes once over the entry's nodes, 32 at a time: the next node of the walk is the
// first one behind the current one that has it for a parent and bears the token wanted.  12 bytes a node are read, the next 32 nodes'
// while these are walked; what it takes is the launch and two trips to memory (one entry 1.5 us, 256 entries 2.3).
__global__ void __launch_bounds__(ACCEPT_WARPS * 32)
tree_accept_kernel(const int* __restrict__ tokens, const int* __restrict__ targets, const int* __restrict__ entry_starts, const int* __restrict__ parents,
                   int entries, int rows, int longest, int* __restrict__ path, int* __restrict__ accepted, int* __restrict__ emitted, int* status) {
    pdl_enter();
    const int r = blockIdx.x * ACCEPT_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (r >= entries) return;
    const int first = entry_starts[r], end = entry_starts[r + 1];
    const bool sound = first >= 0 && end >= first && end <= rows;
    const int n = sound ? end - first : 0;
    int* const my_path = path + (size_t)r * longest;
    int* const my_emitted = emitted + (size_t)r * longest;
    bool bad = !sound;
    int count = 0, at = -1, wanted = 0;                              // the walk's last node and the token that its child has to bear
    int parent = 0, token = 0, target = 0;
    auto load = [&](int i) {
        if (i < n) {
            parent = parents[first + i];
            token = tokens[first + i];
            target = targets[first + i];
        }
    };
    load(lane);
    for (int base = 0; base < n; base += 32) {
        const int i = base + lane, up = parent, mine = token, answer = target;
        load(base + 32 + lane);
        bad |= i < n && (up < -1 || up >= i);
        while (count < longest) {
            const bool next = i < n && (at < 0 ? i == 0 : i > at && up == at && mine == wanted);
            const unsigned found = __ballot_sync(0xffffffffu, next);
            if (!found) break;
            const int who = __ffs(found) - 1;
            at = base + who;
            wanted = __shfl_sync(0xffffffffu, answer, who);
            if (lane == 0) {
                my_path[count] = at;
                my_emitted[count] = wanted;
            }
            ++count;
        }
    }
    for (int j = count + lane; j < longest; j += 32) my_path[j] = my_emitted[j] = -1;
    if (lane == 0) accepted[r] = count;
    if (__any_sync(0xffffffffu, bad) && lane == 0) atomicOr(status, EG_STATUS_BAD_TREE);
}

// The move: row (context + path[j]) of every layer, plane (keys, values) and head goes to (context + j), j < accepted.  A CTA has an entry
// and a stretch of its columns, 16 bytes of a (layer, plane, head)'s row each (or as much as the alignment allows), a thread per column.
// A path ascends and path[j] >= j, so what is read at j is written, if at all, by a later j: a thread loads MOVES rows of its column
// before it stores any of them, which keeps that order and that many loads in flight.  Bound by memory: rows that are moved are read and
// written once; rows with path[j] == j are left alone.  (24 layers, 8 entries, 0.3 MB moved: 3.3 us; 28 layers, 64 entries, 17 MB read and written: 7.2 us, 2.4
// TB/s.)
constexpr int KEEP_THREADS = 256, MOVES = 4, PATH_CHUNK = 64;

struct KeepParams {
    void* kv;
    long long layer_stride, page_stride, plane_stride, head_stride;      // in pieces
    const int* block_table;
    const int* context;
    const int* path;
    const int* accepted;
    int* status;
    int table_stride, table_pages, num_pages, kv_heads, page_size, row_pieces, columns, longest;
};

template <typename Piece>
__global__ void __launch_bounds__(KEEP_THREADS) cache_keep_kernel(const KeepParams p) {
    pdl_enter();
    __shared__ long long from[PATH_CHUNK], to[PATH_CHUNK];
    __shared__ int moves;
    const int r = blockIdx.y, context = p.context[r], count = p.accepted[r];
    const int* const path = p.path + (size_t)r * p.longest;
    // the whole path is looked at before anything moves
    bool bad = count < 0 || count > p.longest || context < 0;
    for (int j = threadIdx.x; !bad && j < count; j += KEEP_THREADS) bad = path[j] < j || (j > 0 && path[j - 1] >= path[j]);
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) atomicOr(p.status, EG_STATUS_BAD_TREE);
        return;
    }
    const int column = blockIdx.x * KEEP_THREADS + threadIdx.x;
    const int piece = column % p.row_pieces, head = column / p.row_pieces % p.kv_heads, plane = column / p.row_pieces / p.kv_heads % 2;
    const long long layer = column / p.row_pieces / p.kv_heads / 2;
    Piece* const mine = static_cast<Piece*>(p.kv) + layer * p.layer_stride + plane * p.plane_stride + head * p.head_stride + piece;
    // where a token's row lies, from the layer, plane and head on; -1 and a status bit where the block table has no place for it
    auto place = [&](long long position) -> long long {
        const long long at = position / p.page_size;
        const int page = at < p.table_pages ? p.block_table[(size_t)r * p.table_stride + at] : -1;
        if (page < 0 || page >= p.num_pages) {
            atomicOr(p.status, EG_STATUS_BAD_PAGE);
            return -1;
        }
        return page * p.page_stride + position % p.page_size * p.row_pieces;
    };
    for (int j0 = 0; j0 < count; j0 += PATH_CHUNK) {
        __syncthreads();                                             // the last chunk's places have been read
        if (threadIdx.x < 32) {                                      // the rows to move, in their order
            int listed = 0;
            for (int h = 0; h < PATH_CHUNK; h += 32) {
                const int j = j0 + h + (int)threadIdx.x, node = j < count ? path[j] : j;
                long long a = -1, b = -1;
                if (node != j) {
                    a = place((long long)context + node);
                    b = place((long long)context + j);
                }
                const bool listing = a >= 0 && b >= 0;
                const unsigned all = __ballot_sync(0xffffffffu, listing);
                if (listing) {
                    const int slot = listed + __popc(all & ((1u << threadIdx.x) - 1));
                    from[slot] = a;
                    to[slot] = b;
                }
                listed += __popc(all);
            }
            if (threadIdx.x == 0) moves = listed;
        }
        __syncthreads();
        if (column >= p.columns) continue;
        for (int m = 0; m < moves; m += MOVES) {
            Piece v[MOVES];
#pragma unroll
            for (int e = 0; e < MOVES; ++e)
                if (m + e < moves) v[e] = mine[from[m + e]];
#pragma unroll
            for (int e = 0; e < MOVES; ++e)
                if (m + e < moves) mine[to[m + e]] = v[e];
        }
    }
}

}  // namespace

EG_API int eg_tree_accept(cudaStream_t stream, const eg_tree_accept_args* args) {
    if (!args) return (int)cudaErrorInvalidValue;
    const eg_tree_accept_args& a = *args;
    constexpr long long INT = 0x7fffffff;
    if (a.entries <= 0) return 0;
    if (a.entries > INT || a.rows < 0 || a.rows > INT || a.longest < 1 || a.longest > INT || !a.status) return (int)cudaErrorInvalidValue;
    eg_pdl_launch(tree_accept_kernel, dim3((unsigned)((a.entries + ACCEPT_WARPS - 1) / ACCEPT_WARPS)), dim3(ACCEPT_WARPS * 32), 0, stream, a.tokens, a.targets, a.entry_starts,
                  a.parents, (int)a.entries, (int)a.rows, (int)a.longest, a.path, a.accepted, a.emitted, a.status);
    return eg_launch_status();
}

EG_API int eg_cache_keep(cudaStream_t stream, const eg_cache_keep_args* args) {
    if (!args) return (int)cudaErrorInvalidValue;
    const eg_cache_keep_args& a = *args;
    constexpr long long INT = 0x7fffffff;
    if (a.entries <= 0 || a.layers <= 0) return 0;
    if (a.entries > 65535 || a.num_pages < 1 || a.num_pages > INT || a.kv_heads < 1 || a.page_size < 1 || a.page_size > INT || a.head_dim < 1 || a.longest < 1 || a.longest > INT ||
        a.table_pages < 0 || a.table_pages > INT || a.table_stride < 0 || a.table_stride > INT || !a.status || (a.element_size != 2 && a.element_size != 4))
        return (int)cudaErrorInvalidValue;
    int width = 16;                                                  // bytes of a piece: every row starts on a multiple of it and is made of whole ones
    const unsigned long long where = (unsigned long long)(uintptr_t)a.kv | (unsigned long long)a.element_size *
        (unsigned long long)(a.layer_stride | a.page_stride | a.plane_stride | a.head_stride | a.head_dim);
    while (where % width) width /= 2;
    if (width < a.element_size) return (int)cudaErrorInvalidValue;
    const long long per = width / a.element_size, most = 1ll << 30;
    if (a.layers > most || a.kv_heads > most || a.head_dim > most || a.layers * 2 * a.kv_heads > most || a.layers * 2 * a.kv_heads * (a.head_dim / per) > most)
        return (int)cudaErrorInvalidValue;
    const int columns = (int)(a.layers * 2 * a.kv_heads * (a.head_dim / per));
    const KeepParams p = {a.kv, a.layer_stride / per, a.page_stride / per, a.plane_stride / per, a.head_stride / per, a.block_table, a.context, a.path, a.accepted, a.status,
                          (int)a.table_stride, (int)a.table_pages, (int)a.num_pages, (int)a.kv_heads, (int)a.page_size, (int)(a.head_dim / per), columns, (int)a.longest};
    const dim3 grid((unsigned)((columns + KEEP_THREADS - 1) / KEEP_THREADS), (unsigned)a.entries);
    if (width == 16) eg_pdl_launch(cache_keep_kernel<uint4>, grid, dim3(KEEP_THREADS), 0, stream, p);
    else if (width == 8) eg_pdl_launch(cache_keep_kernel<uint2>, grid, dim3(KEEP_THREADS), 0, stream, p);
    else if (width == 4) eg_pdl_launch(cache_keep_kernel<unsigned>, grid, dim3(KEEP_THREADS), 0, stream, p);
    else eg_pdl_launch(cache_keep_kernel<unsigned short>, grid, dim3(KEEP_THREADS), 0, stream, p);
    return eg_launch_status();
}
