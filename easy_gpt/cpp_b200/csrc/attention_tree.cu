// Attention over drafted trees and the paged cache (attention_tree.cuh says which keys a row sees) in 32-bit arithmetic, for float32 and
// bfloat16, any head size up to 256, any page size and alignment.
//
// A CTA takes 32 or 64 rows (node, query head) of an entry and KV head, eight a warp, and a part of the keys, 32 at a time, in shared memory as
// float32.  A lane has 8 rows x 4 keys of the scores in a fourth of the head's quads, whose sums the warp then joins, so that a lane has the softmax of
// two rows; and 8 rows x 8 columns of the output from its share of the tile's keys.  Sums, reference and exponents are 32-bit, the reference is the
// running maximum.  Where rows of float32 are whole 16-byte pieces, the next tile comes by asynchronous copies while this one is worked on; else a tile is
// read and converted when it is its turn.
//
// A 16-byte read of a warp takes shared memory four cycles whatever its lanes share: 2,600 cycles for a tile of 32 rows and heads of 128, beside 2,100 of
// multiply-adds, and two CTAs an SM come to 3,300 (tiles of 4 rows x 2 keys a lane: 9,200 for 64 rows).  What the rest waits for is the latency of those
// reads: 240 registers a lane leave four warps a CTA.  32 requests of 32 nodes and 2,000 keys, 12 heads of 128: 430 us, 29 TFLOP/s (685 with 4 x 2); 4 of up
// to 13 nodes and 1,000 keys 25, of which 9 are the start and the adding up.
//
// Which keys a row sees is decided by a select, never by adding: a hidden score may be anything.  A hidden value takes part as 0 * v; where
// there are values that are not finite, every row leaves out those that it does not see.
#include "attention_tree.cuh"
#include "tree_args.h"

namespace {

using tree::Entry;
using tree::Params;

constexpr int KEYS = 32, STAGED_NODES = 1024;
// Rows of a CTA, eight a warp.  Two CTAs of 32 share an SM where tiles come by asynchronous copies; else, and where two do not fit, one of 64.
constexpr int rows_of(int dim, bool async) { return async && dim <= 128 ? 32 : 64; }
constexpr int LISTED = 16;                                           // key tiles whose places in the cache are looked up at a time

// two float32 in 64 bits, for the packed instructions
typedef unsigned long long u64;
__device__ __forceinline__ u64 pair_of(float low, float high) {
    u64 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(low), "f"(high));
    return d;
}
__device__ __forceinline__ float low_of(u64 v) { return __uint_as_float((unsigned)v); }
__device__ __forceinline__ float high_of(u64 v) { return __uint_as_float((unsigned)(v >> 32)); }
__device__ __forceinline__ u64 fma_pair(u64 a, u64 b, u64 c) {
    u64 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ u64 mul_pair(u64 a, u64 b) {
    u64 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

__device__ __forceinline__ u64 add_pair(u64 a, u64 b) {
    u64 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

template <int DMAX, bool ASYNC>
struct Layout {
    static constexpr int ROWS = rows_of(DMAX, ASYNC), THREADS = 4 * ROWS;
    static constexpr int LD = DMAX + 4;                              // floats of a row: eight rows' quads meet no bank twice
    static constexpr int P_LD = ROWS + 4;                            // weights, a line a key
    static constexpr int STAGE = 2 * KEYS * LD;                      // keys, then values
    static constexpr int FLOATS = ROWS * LD + 2 * STAGE + KEYS * P_LD;
};

// ASYNC: float32 in whole 16-byte pieces, two stages of keys and values.
template <typename T, int DMAX, bool ASYNC>
__global__ void __launch_bounds__(Layout<DMAX, ASYNC>::THREADS, Layout<DMAX, ASYNC>::ROWS == 32 ? 2 : 1) attention_tree_kernel(const Params p) {
    using L = Layout<DMAX, ASYNC>;
    constexpr int ROWS = L::ROWS, THREADS = L::THREADS;
    constexpr int QUADS = 2, LANES = DMAX / (4 * QUADS), SPLIT = 32 / LANES;       // of the output: lanes with these many quads of columns, and shares of a tile's keys
    extern __shared__ __align__(16) float smem[];
    float* const q_s = smem;
    float* const ring = q_s + ROWS * L::LD;
    float* const p_s = ring + 2 * L::STAGE;
    __shared__ int ups[STAGED_NODES];
    __shared__ unsigned seen[ROWS];                                  // of a key tile that needs it, by row: a bit a key
    __shared__ int lowest[ROWS];                                     // a row's first cached key
    __shared__ int latest;                                           // the largest of those
    __shared__ long long key_row[LISTED * KEYS];                     // where a key's row lies in the cache; -1: nowhere
    pdl_enter();
    const int part = blockIdx.x % p.max_parts, kvh = blockIdx.x / p.max_parts % p.num_kv_heads, tid = threadIdx.x;
    const int group = p.num_heads / p.num_kv_heads;
    int r, within;
    Entry e;
    if (!tree::find_tile(p, blockIdx.x / p.max_parts / p.num_kv_heads, ROWS, r, e, within)) return;
    const int D = p.head_dim, row0 = within * ROWS, count = min(ROWS, e.n * group - row0);
    const int last_node = (row0 + count - 1) / group;
    bool hole;                                                       // a page that is none has been met
    const int first = tree::first_key(p, e), end = tree::end_key(p, e, first, last_node, hole);      // the tile's keys: first .. end - 1
    const int tile0 = first / KEYS, tiles = (end - 1) / KEYS - tile0 + 1, parts = tree::parts_of(p, tiles);
    if (part >= parts) return;
    const int begin = tile0 + (int)((long long)tiles * part / parts), stop = tile0 + (int)((long long)tiles * (part + 1) / parts);

    auto list_keys = [&](int tile) {                                 // the places of tiles tile .. tile + LISTED - 1
        for (int i = tid; i < LISTED * KEYS; i += THREADS) {
            const int at = tile * KEYS + i, slot = at / p.page_size;
            long long row = -1;
            if (tile + i / KEYS < stop && at >= first && at < end) {
                const int page = slot < p.table_pages ? p.block_table[(size_t)r * p.table_stride + slot] : -1;
                if (page < 0 || page >= p.num_pages) {
                    hole = true;
                    atomicOr(p.status, EG_STATUS_BAD_PAGE);
                } else {
                    row = page * p.page_stride + kvh * p.head_stride + (long long)(at % p.page_size) * D;
                }
            }
            key_row[i] = row;
        }
    };
    auto stage_of = [&](int tile) { return ring + (ASYNC ? (tile - begin) & 1 : 0) * L::STAGE; };
    auto load = [&](int tile) {
        float* const k_s = stage_of(tile);
        const long long* const rows = key_row + (tile - begin) % LISTED * KEYS;
        if constexpr (ASYNC) {
            constexpr int PIECES = DMAX / 4;
#pragma unroll 4
            for (int i = tid; i < KEYS * PIECES; i += THREADS) {
                const int key = i / PIECES, d = i % PIECES * 4;
                const long long row = rows[key];
                const bool there = row >= 0 && d < D;
                const size_t from = there ? (size_t)(row + d) : 0;
                const unsigned to = (unsigned)__cvta_generic_to_shared(k_s + key * L::LD + d);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to), "l"(static_cast<const float*>(p.k_cache) + from), "r"(there ? 16 : 0));
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(to + 4 * KEYS * L::LD), "l"(static_cast<const float*>(p.v_cache) + from),
                             "r"(there ? 16 : 0));
            }
        } else {
#pragma unroll 8
            for (int i = tid; i < KEYS * DMAX; i += THREADS) {
                const int key = i / DMAX, d = i % DMAX;
                const long long row = rows[key];
                float k = 0.f, v = 0.f;
                if (d < D && row >= 0) {
                    k = to_f32<T>(static_cast<const T*>(p.k_cache)[row + d]);
                    v = to_f32<T>(static_cast<const T*>(p.v_cache)[row + d]);
                }
                k_s[key * L::LD + d] = k;
                k_s[(KEYS + key) * L::LD + d] = v;
            }
        }
    };
    // ---- the rows of q
    if constexpr (ASYNC) {
        for (int i = tid; i < ROWS * (DMAX / 4); i += THREADS) {
            const int row = i / (DMAX / 4), d = i % (DMAX / 4) * 4, node = (row0 + row) / group, head = kvh * group + (row0 + row) % group;
            const bool there = row < count && d < D;
            const size_t from = there ? (size_t)(e.first + node) * p.ldq + (size_t)head * D + d : 0;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"((unsigned)__cvta_generic_to_shared(q_s + row * L::LD + d)),
                         "l"(static_cast<const float*>(p.q) + from), "r"(there ? 16 : 0));
        }
    } else {
#pragma unroll 8
        for (int i = tid; i < ROWS * DMAX; i += THREADS) {
            const int row = i / DMAX, d = i % DMAX, node = (row0 + row) / group, head = kvh * group + (row0 + row) % group;
            float x = 0.f;
            if (row < count && d < D) x = to_f32<T>(static_cast<const T*>(p.q)[(size_t)(e.first + node) * p.ldq + (size_t)head * D + d]);
            q_s[row * L::LD + d] = x;
        }
    }
    list_keys(begin);
    for (int i = tid; i <= last_node && i < STAGED_NODES; i += THREADS) ups[i] = tree::parent_of(p, e, i);
    if (tid == 0) latest = 0;
    __syncthreads();
    if (ASYNC) {
        load(begin);
        asm volatile("cp.async.commit_group;\n" ::);
    }
    // ---- every row's first cached key
    auto up_of = [&](int i) { return i < STAGED_NODES ? ups[i] : tree::parent_of(p, e, i); };
    if (tid < ROWS) {
        int low = 0;
        if (p.window > 0 && tid < count) {
            int depth = 0;
            for (int i = up_of((row0 + tid) / group); i >= 0; i = up_of(i)) ++depth;
            low = (int)max(0ll, (long long)e.context + depth - p.window + 1);
            atomicMax(&latest, low);
        }
        lowest[tid] = low;
    }
    // A warp has 8 rows.  Of their scores a lane has those with 4 keys, key_of + 8 j, in every fourth quad of the head; of their output 8 columns from a
    // share of the keys.
    const int lane = tid & 31, row_of = tid / 32 * 8, key_of = lane & 7, quarter = lane >> 3, share = lane / LANES, column = lane % LANES * 4;
    const int mine = row_of + 2 * quarter;                           // the two rows whose softmax a lane has
    const float scale_log2 = p.scale * 1.4426950408889634f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};          // l: of the lane's keys
    u64 acc[8][QUADS][2];                                            // pairs of columns: column .. column + 3, and those DMAX / 2 on
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int h = 0; h < QUADS; ++h) acc[i][h][0] = acc[i][h][1] = 0;
    for (int tile = begin; tile < stop; ++tile) {
        const int key0 = tile * KEYS;
        if constexpr (ASYNC) {
            asm volatile("cp.async.wait_group 0;\n" ::: "memory");
            __syncthreads();                                         // this tile is there, the last one has been read
            if (tile + 1 < stop) {
                if ((tile + 1 - begin) % LISTED == 0) {
                    list_keys(tile + 1);
                    __syncthreads();
                }
                load(tile + 1);
            }
            asm volatile("cp.async.commit_group;\n" ::);
        } else {
            __syncthreads();
            if (tile > begin && (tile - begin) % LISTED == 0) {
                list_keys(tile);
                __syncthreads();
            }
            load(tile);
            __syncthreads();
        }
        const float* const k_s = stage_of(tile);
        const float* const v_s = k_s + KEYS * L::LD;
        // ---- a tile that reaches into the tree, over a window's edge or onto a page that is none (of this run of tiles): which keys a row sees
        const bool checked = __syncthreads_or(hole);                 // the same for all threads: pages are looked at again
        const bool masked = key0 + KEYS > e.context || key0 < max(first, latest) || checked;
        bool odd = false;
        if (masked) {
            if (tid < ROWS) {
                unsigned bits = 0;
                if (tid < count) {
                    const int low = max(max(lowest[tid], first), key0), high = min(e.context, key0 + KEYS);      // the cached keys that it sees
                    if (low < high) bits = 0xffffffffu >> (KEYS - (high - low)) << (low - key0);
                    int left = p.window > 0 ? p.window : 0x7fffffff;
                    for (int i = (row0 + tid) / group; i >= 0 && e.context + i >= key0 && left > 0; i = up_of(i), --left)
                        if (e.context + i < key0 + KEYS) bits |= 1u << (e.context + i - key0);
                    for (int key = 0; checked && key < KEYS; ++key) {      // on pages that are there
                        const int slot = (key0 + key) / p.page_size, page = slot < p.table_pages ? p.block_table[(size_t)r * p.table_stride + slot] : -1;
                        if ((bits >> key & 1) && (page < 0 || page >= p.num_pages)) bits &= ~(1u << key);
                    }
                }
                seen[tid] = bits;
            }
            for (int i = tid; i < KEYS * DMAX / 4; i += THREADS) {
                const float4 v = *reinterpret_cast<const float4*>(v_s + i / (DMAX / 4) * L::LD + i % (DMAX / 4) * 4);
                odd |= !(isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w));
            }
            odd = __syncthreads_or(odd);
        }
        if (row_of >= count) continue;                               // a warp whose rows are all filling
        // ---- scores
        // (multiply-adds on pairs: of neighbouring terms here, of neighbouring columns below; half the instructions)
        float s[2][4];
        {
            u64 sums[8][4] = {};
#pragma unroll 2
            for (int d = 4 * quarter; d < DMAX; d += 16) {
                ulonglong2 b[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const ulonglong2*>(k_s + (key_of + 8 * j) * L::LD + d);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(q_s + (row_of + i) * L::LD + d);
#pragma unroll
                    for (int j = 0; j < 4; ++j) sums[i][j] = fma_pair(a.y, b[j].y, fma_pair(a.x, b[j].x, sums[i][j]));
                }
            }
            // the quarters' sums: a lane keeps half of the rows and gives the other half away, twice
            float half[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float low = low_of(sums[i][j]) + high_of(sums[i][j]), high = low_of(sums[4 + i][j]) + high_of(sums[4 + i][j]);
                    half[i][j] = (quarter & 2 ? high : low) + __shfl_xor_sync(0xffffffffu, quarter & 2 ? low : high, 16);
                }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    s[i][j] = (quarter & 1 ? half[2 + i][j] : half[i][j]) + __shfl_xor_sync(0xffffffffu, quarter & 1 ? half[i][j] : half[2 + i][j], 8);
        }
        float keep[2];
        float2 weights[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const unsigned bits = (masked ? seen[mine + i] : ~0u) >> key_of;
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] = bits >> (8 * j) & 1 ? s[i][j] * scale_log2 : -INFINITY;
                top = fmaxf(top, s[i][j]);
            }
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float now = fmaxf(m[i], top), ref = now == -INFINITY ? 0.f : now;     // a row that has seen nothing: every weight 0
            keep[i] = exp2f(m[i] - ref);
            m[i] = now;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float w = exp2f(s[i][j] - ref);
                (i ? weights[j].y : weights[j].x) = w;
                sum += w;
            }
            l[i] = l[i] * keep[i] + sum;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<float2*>(p_s + (key_of + 8 * j) * L::P_LD + mine) = weights[j];
        if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float c = __shfl_sync(0xffffffffu, keep[i & 1], i / 2 * 8);
                const u64 both = pair_of(c, c);
#pragma unroll
                for (int h = 0; h < QUADS; ++h) acc[i][h][0] = mul_pair(acc[i][h][0], both), acc[i][h][1] = mul_pair(acc[i][h][1], both);
            }
        }
        __syncwarp();                                                // a row's weights come from its own warp
        // ---- output
        const int from = share * (KEYS / SPLIT);
        if (!odd) {
#pragma unroll 2
            for (int key = from; key < from + KEYS / SPLIT; ++key) {
                const float4 w0 = *reinterpret_cast<const float4*>(p_s + key * L::P_LD + row_of), w1 = *reinterpret_cast<const float4*>(p_s + key * L::P_LD + row_of + 4);
                ulonglong2 v[QUADS];
#pragma unroll
                for (int h = 0; h < QUADS; ++h) v[h] = *reinterpret_cast<const ulonglong2*>(v_s + key * L::LD + h * (DMAX / 2) + column);
                const float each[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const u64 both = pair_of(each[i], each[i]);
#pragma unroll
                    for (int h = 0; h < QUADS; ++h) acc[i][h][0] = fma_pair(both, v[h].x, acc[i][h][0]), acc[i][h][1] = fma_pair(both, v[h].y, acc[i][h][1]);
                }
            }
        } else {
            for (int key = from; key < from + KEYS / SPLIT; ++key) {
                ulonglong2 v[QUADS];
#pragma unroll
                for (int h = 0; h < QUADS; ++h) v[h] = *reinterpret_cast<const ulonglong2*>(v_s + key * L::LD + h * (DMAX / 2) + column);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (!(seen[row_of + i] >> key & 1)) continue;
                    const float w = p_s[key * L::P_LD + row_of + i];
                    const u64 both = pair_of(w, w);
#pragma unroll
                    for (int h = 0; h < QUADS; ++h) acc[i][h][0] = fma_pair(both, v[h].x, acc[i][h][0]), acc[i][h][1] = fma_pair(both, v[h].y, acc[i][h][1]);
                }
            }
        }
    }
    // ---- a row's sum over its lanes, its output over the shares of the keys
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
#pragma unroll
    for (int o = LANES; o < 32; o *= 2)
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int x = 0; x < 2 * QUADS; ++x) acc[i][x / 2][x % 2] = add_pair(acc[i][x / 2][x % 2], __shfl_xor_sync(0xffffffffu, acc[i][x / 2][x % 2], o));
    // where a row's results go
    auto line_of = [&](int row) {
        return static_cast<T*>(p.out) + (size_t)(e.first + (row0 + row) / group) * p.ldo + (size_t)(kvh * group + (row0 + row) % group) * D;
    };
    if (parts == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float sum = __shfl_sync(0xffffffffu, l[i & 1], i / 2 * 8), inv = sum > 0.f ? 1.f / sum : sum;
            if (i % SPLIT != share || row_of + i >= count) continue;
            T* const line = line_of(row_of + i);
#pragma unroll
            for (int x = 0; x < 4 * QUADS; ++x) {
                const u64 pair = acc[i][x / 4][x / 2 % 2];
                const int d = x / 4 * (DMAX / 2) + column + x % 4;
                if (d < D) line[d] = from_f32<T>((x & 1 ? high_of(pair) : low_of(pair)) * inv);
            }
        }
        return;
    }
    __syncthreads();                                                 // q, keys and values have been read
    float* const o_s = q_s;
    float* const ml_s = ring;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i % SPLIT != share) continue;
#pragma unroll
        for (int h = 0; h < QUADS; ++h)
            *reinterpret_cast<ulonglong2*>(o_s + (row_of + i) * L::LD + h * (DMAX / 2) + column) = make_ulonglong2(acc[i][h][0], acc[i][h][1]);
    }
    if (key_of == 0) {
        *reinterpret_cast<float2*>(ml_s + 2 * mine) = make_float2(m[0], l[0]);
        *reinterpret_cast<float2*>(ml_s + 2 * mine + 2) = make_float2(m[1], l[1]);
    }
    tree::add_parts<THREADS>(o_s, L::LD, ml_s, count, DMAX, parts, [&](int row, int d, float4 v) {
        T* const line = line_of(row);
        if (d < D) line[d] = from_f32<T>(v.x);
        if (d + 1 < D) line[d + 1] = from_f32<T>(v.y);
        if (d + 2 < D) line[d + 2] = from_f32<T>(v.z);
        if (d + 3 < D) line[d + 3] = from_f32<T>(v.w);
    });
}

template <typename T, int DMAX, bool ASYNC>
int launch(cudaStream_t stream, const Params& p, long long tiles) {
    using L = Layout<DMAX, ASYNC>;
    constexpr int bytes = L::FLOATS * 4;
    static unsigned long long seen = 0;
    if (const int code = tree::prepare_kernel(attention_tree_kernel<T, DMAX, ASYNC>, bytes, seen)) return code;
    return tree::launch_clusters(attention_tree_kernel<T, DMAX, ASYNC>, p.max_parts, p.num_kv_heads, tiles, L::THREADS, bytes, stream, p);
}
template <typename T, bool ASYNC>
int launch_any(cudaStream_t stream, const Params& p, long long tiles) {
    return p.head_dim <= 64 ? launch<T, 64, ASYNC>(stream, p, tiles) : p.head_dim <= 128 ? launch<T, 128, ASYNC>(stream, p, tiles) : launch<T, 256, ASYNC>(stream, p, tiles);
}

}  // namespace

// How a step's work is laid out, from sizes alone: plan[0] the rows of a CTA (128: the tcgen05 kernel; 16, 32 or 64: the warp-level one;
// 0: the 32-bit one), plan[1] and plan[2] the max_parts and part_tiles of eg_attention_tree.  aligned: the caches, their pages and heads start on
// 16-byte boundaries, and q, out and their rows on 16-byte (2) or 4-byte (1) ones; of float32 not 0 where rows of q and the caches are whole 16-byte
// pieces.  max_context: the most keys of an entry, as far as known.
//
// A key tile of 64 takes a CTA 1 us on the tcgen05 kernel whatever its rows, and 1 us (16 rows of 64) to 2.6 us (64 rows of 128) on the warp-level one,
// whose start and end are 2 us shorter: that one takes short contexts of few units where both would do (a chain of 8 at 500 keys 7.2 us against 9.0;
// 64 requests of 16 nodes at 700 keys 46 against 21).  Parts: as many as keep one CTA an SM with three key tiles a part, or two CTAs with eight;
// more of them cost more than they save (32 requests of 9 nodes at 1,000 keys in 1, 2, 4 and 8 parts 18.5, 15.9, 13.9 and 24.8 us; 64 requests of 16 at 700
// in 1, 2 and 4 parts 21, 25 and 36), and clusters of 16 find little room.  Long contexts are cut into four in any case, for an even end (16 requests of up
// to 32,768 keys, wide trees, in 1, 2, 4 and 8 parts 598, 409, 386 and 465: medians of 40 calls of each in turn, four fifths of them within 4%, at 1.7 GHz under the
// power limit).  The 32-bit kernel's CTAs of 32 rows go two to an SM from the first (4
// requests of 13 nodes at 1,000 keys, 12 heads on 2, in 4, 8 and 16 parts 29, 24.5 and 28.5; one node at 4,000, 12 on 12, in 8 and 16 47 and 30).
EG_API int eg_attention_tree_plan(int dtype, int aligned, int rows, int entries, int num_heads, int num_kv_heads, int head_dim, int page_size, int max_context, int sm_count,
                                  int* plan) {
    if (rows < 1 || entries < 1 || num_kv_heads < 1 || num_heads % num_kv_heads || num_heads < 1 || page_size < 1 || sm_count < 1 || !plan) return (int)cudaErrorInvalidValue;
    const int group = num_heads / num_kv_heads;
    const long long lines = ((long long)rows * group + entries - 1) / entries;      // of an entry, on the average
    const long long key_tiles = ((long long)max_context + 63) / 64;
    const bool tiled = dtype == EG_BF16 && aligned && page_size % 16 == 0 && head_dim % 8 == 0;
    const bool pieces = dtype == EG_F32 && aligned;                  // the 32-bit kernel's asynchronous copies
    const bool wide = tiled && aligned > 1 && (head_dim == 64 || head_dim == 128) && group <= 128;
    const auto units_of = [&](long long tile) { return entries * ((lines + tile - 1) / tile) * num_kv_heads; };
    int row_tile = !tiled ? 0 : lines <= 16 ? 16 : lines <= 32 ? 32 : 64;
    if (wide && (key_tiles > 16 || units_of(64) * 8 > sm_count)) row_tile = 128;
    else if (tiled && units_of(16) * 8 <= sm_count) row_tile = 16;
    const long long units = units_of(row_tile == 128 ? 128 / group * group : row_tile ? row_tile : rows_of(head_dim, pieces));
    const bool pairs = row_tile == 0 && rows_of(head_dim, pieces) == 32;             // two CTAs an SM from the first
    const int most = head_dim > 128 || row_tile == 128 || (row_tile == 0 && !pairs) ? 8 : 16;
    int parts = 1;
    while (parts < most && ((units * parts * 2 <= (pairs ? 2ll : 1ll) * sm_count && key_tiles >= parts * (row_tile == 128 ? 6 : pairs && parts == 8 ? 4 : 2)) || (units * parts * 2 <= 2ll * sm_count && key_tiles >= parts * 16))) parts *= 2;
    while (parts < 4 && key_tiles > parts * 64) parts *= 2;
    plan[0] = row_tile;
    plan[1] = parts;
    plan[2] = 1;
    return 0;
}

// A tile's keys are cut into up to max_parts (1, 2, 4, 8 or 16) parts of at least part_tiles times 64 keys.
EG_API int eg_attention_tree(cudaStream_t stream, const eg_attention_tree_args* args) {
    if (!args) return (int)cudaErrorInvalidValue;
    const eg_attention_tree_args& a = *args;
    if (a.entries <= 0 || a.rows <= 0) return 0;
    constexpr long long INT = 0x7fffffff;
    if ((a.dtype != EG_F32 && a.dtype != EG_BF16) || a.num_kv_heads < 1 || a.num_heads < 1 || a.num_heads > INT || a.num_heads % a.num_kv_heads || a.num_kv_heads > 65535 ||
        a.head_dim < 1 || a.head_dim > 256 || a.page_size < 1 || a.page_size > INT || a.num_pages < 1 || a.num_pages > INT || a.table_pages < 0 || a.table_pages > INT ||
        a.table_stride < 0 || a.table_stride > INT || a.entries > 65535 || a.rows > INT || a.rows * a.num_heads > INT || a.window < 0 || a.window > INT ||
        !((float)a.scale > 0.f) || !(a.scale < 2e38) || !a.status)      // (a scale of 0 in 32 bits, or of infinity with the exponents' base in it, makes NaN of hidden scores)
        return (int)cudaErrorInvalidValue;
    const int dim = (int)a.head_dim, group = (int)(a.num_heads / a.num_kv_heads);
    // what the tensor-core kernels ask of addresses and strides
    const long long rows_at = (long long)((uintptr_t)a.q | (uintptr_t)a.out) | (a.ldq | a.ldo) * 2;
    const bool tiled = a.dtype == EG_BF16 && (((uintptr_t)a.k_cache | (uintptr_t)a.v_cache) & 15) == 0 && ((a.page_stride | a.head_stride) & 7) == 0 && rows_at % 4 == 0;
    const bool pieces = a.dtype == EG_F32 && (((uintptr_t)a.q | (uintptr_t)a.k_cache | (uintptr_t)a.v_cache) & 15) == 0 && ((a.ldq | a.page_stride | a.head_stride | a.head_dim) & 3) == 0;
    const int aligned = !tiled ? pieces : rows_at % 16 || a.page_stride % dim || a.head_stride % dim || a.page_stride <= 0 || a.head_stride <= 0 ? 1 : 2;
    int plan[3] = {(int)a.row_tile, (int)a.max_parts, (int)a.part_tiles};
    if (a.row_tile < 0) {
        // a window's worth of keys and the nodes, where that is less
        const long long reach = a.window > 0 ? a.window + 2 * a.rows / a.entries : INT, most = a.max_context < reach ? a.max_context : reach, keys = most < 1 ? 1 : most > INT ? INT : most;
        const int code = eg_attention_tree_plan((int)a.dtype, aligned, (int)a.rows, (int)a.entries, (int)a.num_heads, (int)a.num_kv_heads, dim, (int)a.page_size,
                                                (int)keys, eg_sm_count(), plan);
        if (code) return code;
    } else if ((a.row_tile && a.row_tile != 16 && a.row_tile != 32 && a.row_tile != 64 && a.row_tile != 128) || a.max_parts < 1 || a.max_parts > tree::MAX_PARTS ||
               (a.max_parts & (a.max_parts - 1)) || a.part_tiles < 1 || a.part_tiles > 1 << 20) {
        return (int)cudaErrorInvalidValue;
    }
    const int row_tile = plan[0];
    if (row_tile && (!tiled || dim % 8 || a.page_size % 16)) return (int)cudaErrorInvalidValue;
    if (row_tile == 128 && (aligned < 2 || (dim != 64 && dim != 128) || group > 128)) return (int)cudaErrorInvalidValue;
    const int tile_rows = row_tile ? row_tile : rows_of(dim, pieces), tile_keys = row_tile ? 64 : KEYS;
    const long long tiles = a.rows * group / tile_rows + a.entries;   // at most: every entry's last tile may be a short one
    const Params p = {a.q, a.ldq, a.k_cache, a.v_cache, a.page_stride, a.head_stride, a.block_table, (int)a.table_stride, (int)a.table_pages, (int)a.num_pages,
                      a.entry_starts, a.context, a.parents, a.out, a.ldo, (int)a.rows, (int)a.entries, (int)a.num_heads, (int)a.num_kv_heads, dim, (int)a.page_size,
                      (int)a.window, (float)a.scale, plan[1], plan[2] * (64 / tile_keys), a.status, tiles * a.num_kv_heads * plan[1] > 2 * eg_sm_count()};
    if (row_tile == 128) return tree::launch_tc(stream, p);
    if (row_tile) return tree::launch_mma(stream, p, row_tile, tiles);
    if (a.dtype == EG_BF16) return launch_any<bf16, false>(stream, p, tiles);
    return pieces ? launch_any<float, true>(stream, p, tiles) : launch_any<float, false>(stream, p, tiles);
}
