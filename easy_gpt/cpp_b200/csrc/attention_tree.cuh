// What the kernels of attention over drafted trees share: their parameters, how the rows of a step are dealt out, and which keys a row sees.
//
// Entry r of a step brings n nodes, its rows entry_starts[r] .. entry_starts[r + 1] - 1, numbered from 0; parents[row] is the number of the
// parent (lower than the node's own) or -1.  context[r] keys are cached in front of them; node i's key lies behind those, at context + i,
// while its position in the text is context + depth(i), depth being how many ancestors it has.  A node sees the cached keys, its ancestors
// and itself; with a window only those whose position is above its own minus the window.
//
// A row of the kernels is a (node, query head of the KV head's group): row i of an entry and KV head is head i % group of node i / group.
// Rows are cut into tiles, tiles are numbered through over the entries, and a tile's keys are cut into up to 16 parts, a CTA each.  The CTAs
// of a tile are a thread-block cluster: their partial results (unnormalised output, reference, sum; base 2) stay in their shared memory, where the
// cluster adds them up in the order of the parts, every CTA a share of the output.
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
    int* status;
    int longest_first;               // tiles of entries with more keys are numbered first (of 32 entries at a time)
};

// An entry's place in the step.
struct Entry {
    int first, n, context;
};
// The most nodes of an entry.  A row's mask in a key tile is a walk up its ancestors, so a chain of n nodes takes time by the square of n (1,024 nodes 0.8 ms,
// 4,096 21 ms; trees as drafts grow them, whose depth is some dozens, 0.04 and 0.3): from here on a call would take seconds, and one walk come near the
// limit of the waits for it.
constexpr int MOST_NODES = 1 << 14;
// Entry r as the metadata has it; n = 0 where its rows cannot be what they say (and a status bit).
__device__ __forceinline__ Entry sound(const Params& p, int first, int end, int context) {
    Entry e = {first, end - first, context};
    if (first < 0 || end < first || end > p.rows || e.n > MOST_NODES || context < 0 || context > 0x7fffffff - 4096 - e.n) {      // (the kernels look a few tiles ahead)
        atomicOr(p.status, EG_STATUS_BAD_TREE);
        e.n = 0;
    }
    return e;
}

// Node i's parent as the metadata has it; one that cannot be is none, and a status bit.
__device__ __forceinline__ int sound_parent(const Params& p, int i, int up) {
    if (up < -1 || up >= i) {
        atomicOr(p.status, EG_STATUS_BAD_TREE);
        return -1;
    }
    return up;
}
__device__ __forceinline__ int parent_of(const Params& p, const Entry& e, int i) { return sound_parent(p, i, p.parents[e.first + i]); }

// The entry whose tile number `tile` is, counting ceil(n * group / row_tile) tiles an entry, and the tile's number within it; false: there
// is none.  For a whole warp: 32 entries at a time, in one trip to memory, the next 32 asked for meanwhile.  CTAs start in the order of their tiles, and
// where there are more of them than places, the ones with most keys had better start first: a tile's number then goes by its entry's place in that order.
__device__ __forceinline__ bool find_tile(const Params& p, int tile, int row_tile, int& r, Entry& e, int& within) {
    const int lane = threadIdx.x & 31, group = p.num_heads / p.num_kv_heads;
    int first = 0, end = 0, context = 0;
    const auto ask = [&](int i) {
        if (i < p.entries) {
            first = p.entry_starts[i];
            end = p.entry_starts[i + 1];
            context = p.context[i];
        }
    };
    ask(lane);
    for (int base = 0; base < p.entries; base += 32) {
        Entry mine = {0, 0, 0};
        if (base + lane < p.entries) mine = sound(p, first, end, context);
        ask(base + 32 + lane);
        const int tiles = (int)(((long long)mine.n * group + row_tile - 1) / row_tile);
        int upto = tiles;
        if (p.longest_first) {
            const int keys = mine.context;
            for (int j = 0; j < 32; ++j) {
                const int other = __shfl_sync(0xffffffffu, keys, j), its = __shfl_sync(0xffffffffu, tiles, j);
                if (other > keys || (other == keys && j < lane)) upto += its;
            }
        } else {
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int below = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += below;
            }
        }
        const unsigned here = __ballot_sync(0xffffffffu, tile < upto && tile >= upto - tiles);
        if (here) {
            const int who = __ffs(here) - 1;
            r = base + who;
            e.first = __shfl_sync(0xffffffffu, mine.first, who);
            e.n = __shfl_sync(0xffffffffu, mine.n, who);
            e.context = __shfl_sync(0xffffffffu, mine.context, who);
            within = tile - __shfl_sync(0xffffffffu, upto - tiles, who);
            return true;
        }
        tile -= __reduce_max_sync(0xffffffffu, upto);
    }
    return false;
}

// A tile's first key that any of its rows may see, and the key behind its last one.
__device__ __forceinline__ int first_key(const Params& p, const Entry& e) { return p.window > 0 && e.context >= p.window ? e.context - p.window + 1 : 0; }

// The key behind a tile's last one.  The block table has no place for keys from table_pages * page_size on: a tile's keys end there (one stays, so that there
// is something to go through), `beyond` says so, and so does the status.
__device__ __forceinline__ int end_key(const Params& p, const Entry& e, int first, int last_node, bool& beyond) {
    const int end = e.context + last_node + 1;
    const long long room = (long long)p.table_pages * p.page_size;
    beyond = end > room;
    if (!beyond) return end;
    if (threadIdx.x == 0) atomicOr(p.status, EG_STATUS_BAD_PAGE);
    return max((int)room, first + 1);
}

__device__ __forceinline__ int parts_of(const Params& p, int key_tiles) { return max(1, min(p.max_parts, key_tiles / p.part_tiles)); }

// Whether there are infinities or NaN among bfloat16: the largest magnitudes in the upper and the lower halves of words, and what those say.
__device__ __forceinline__ unsigned largest_halves(unsigned largest, uint4 v) {
    largest = __vmaxu2(largest, __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu));
    return __vmaxu2(largest, __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
}
__device__ __forceinline__ bool not_finite(unsigned largest) { return (largest & 0xffffu) >= 0x7f80u || largest >> 16 >= 0x7f80u; }

// The kernel in attention_tree_mma.cu (16, 32 or 64 rows a CTA, key tiles of 64).  Its caller has checked what it takes.
int launch_mma(cudaStream_t stream, const Params& p, int row_tile, long long tiles);
// The kernel in attention_tree_tc.cu (128 rows a CTA, or as many as whole nodes have; key tiles of 64).  Its caller has checked what it takes, but for the
// size of the tensor maps.
int launch_tc(cudaStream_t stream, const Params& p);

// ---- the parts of a tile, one CTA of the cluster each
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ unsigned remote(const void* mine, unsigned rank) {
    unsigned a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((unsigned)__cvta_generic_to_shared(mine)), "r"(rank));
    return a;
}
__device__ __forceinline__ float2 remote_load2(unsigned at) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at));
    return v;
}
__device__ __forceinline__ float4 remote_load4(unsigned at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
    return v;
}
constexpr int MAX_PARTS = 16;

// Adds the cluster's parts up.  Every CTA has `o` (rows of `ld` floats, unnormalised) and `ml` (reference and sum a row; -inf and 0 where it has seen
// nothing) in shared memory, written before the call; put(row, column, four values) takes the result.  A row takes part whose sum is not 0, in whatever
// part.  The cluster's first `parts` CTAs call this, and none of them leaves it before its shared memory has been read; the others have left the
// kernel, which the barriers do not wait for.
template <int THREADS, typename Put>
__device__ __forceinline__ void add_parts(const float* o, int ld, const float* ml, int rows, int columns, int parts, Put put) {
    unsigned rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    cluster_barrier();
    const int quads = columns / 4;
    constexpr int AT_ONCE = 8;                                       // parts whose numbers are asked for together
    for (int i = (int)rank * THREADS + (int)threadIdx.x; i < rows * quads; i += parts * THREADS) {
        const int row = i / quads, d = i % quads * 4;
        float top = -INFINITY, total = 0.f;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int q0 = 0; q0 < parts; q0 += AT_ONCE) {
            float2 w[AT_ONCE];
            float4 v[AT_ONCE];
#pragma unroll
            for (int q = 0; q < AT_ONCE; ++q) w[q] = q0 + q < parts ? remote_load2(remote(ml + 2 * row, q0 + q)) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int q = 0; q < AT_ONCE; ++q) v[q] = q0 + q < parts ? remote_load4(remote(o + row * ld + d, q0 + q)) : make_float4(0.f, 0.f, 0.f, 0.f);
            float now = top;
#pragma unroll
            for (int q = 0; q < AT_ONCE; ++q) now = fmaxf(now, w[q].x);
            const float ref = now == -INFINITY ? 0.f : now, keep = exp2f(top - ref);
            top = now;
            total *= keep;
            sum = make_float4(sum.x * keep, sum.y * keep, sum.z * keep, sum.w * keep);
#pragma unroll
            for (int q = 0; q < AT_ONCE; ++q) {
                const float c = w[q].x == -INFINITY ? 0.f : exp2f(w[q].x - ref);
                total = fmaf(c, w[q].y, total);
                sum = make_float4(fmaf(c, v[q].x, sum.x), fmaf(c, v[q].y, sum.y), fmaf(c, v[q].z, sum.z), fmaf(c, v[q].w, sum.w));
            }
        }
        const float inv = total > 0.f ? 1.f / total : total;          // nothing seen: 0; NaN stays
        put(row, d, make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv));
    }
    cluster_barrier();
}

// A launch of `tiles` clusters of p.max_parts CTAs for every KV head (blockIdx.x = (tile * num_kv_heads + KV head) * max_parts + part), behind the kernel
// in front as a programmatic dependent.
template <class... P, class... A>
static inline int launch_clusters(void (*kernel)(P...), int max_parts, int num_kv_heads, long long tiles, int threads, size_t bytes, cudaStream_t stream, A... args) {
    if (tiles * num_kv_heads * max_parts > 0x7fffffff) return (int)cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * num_kv_heads * max_parts));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = max_parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = eg_pdl_on() ? 2 : 1;
    (void)cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);       // its error is the launch status
    return eg_launch_status();
}
template <class K> static inline int prepare_kernel(K kernel, int bytes, unsigned long long& seen) {
    int device;
    if (!eg_first_on_device(seen, device)) return 0;
    cudaError_t set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (set == cudaSuccess) set = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (set == cudaSuccess) eg_done_on_device(seen, device);
    return (int)set;
}

}  // namespace tree
