// Attention over drafted trees and the paged cache (attention_tree.cuh says which keys a row sees) on the warp-level tensor cores: bfloat16,
// heads of a multiple of 8 up to 256 (columns up to 32, 64, 128 or 256 are zeros), pages of a multiple of 16 tokens, caches on 16-byte boundaries.
//
// A CTA of four warps takes 16, 32 or 64 rows (node, query head) of an entry and KV head, so that a key is read once for all of them, and a
// part of the keys, 64 at a time through a ring of asynchronous copies.  With 64 rows a warp has 16 of them and all 64 keys; with 16 it has
// all of them and 16 keys, and the warps' results are added up at the end.  Scores, running maximum, sums and output are 32-bit; weights are
// rounded to bfloat16 for their product with the values (which are bfloat16 themselves); exponents are the hardware's, base 2.
//
// Only the key tiles that reach into the tree or over a window's edge look at which keys a row sees: a 64-bit mask a row, from a walk up
// the row's ancestors.  Hidden scores are replaced, so they may be anything.  Hidden values meet a weight of zero, which hides all but
// infinities and NaN: such tiles look for those, add them to the rows that see them and put zeros in their place.
//
// Bound by latency at the sizes that the rule gives it (eg_attention_tree_plan): a chain of 8 at 500 keys, 14 heads of 64, 7.2 us, of which the start is 3, a key
// tile 1 and the adding up 2.
#include "attention_tree.cuh"
#include "mma_utils.cuh"

namespace {

using tree::Entry;
using tree::Params;

constexpr int KEYS = 64, THREADS = 128, STAGED_NODES = 512;

template <int HD, int WR>
struct Layout {
    static constexpr int ROWS = 16 * WR, WK = 4 / WR, KW = KEYS / WK;
    static constexpr int CHUNKS = HD / 8, SWZ = CHUNKS >= 8 ? 7 : CHUNKS - 1;     // 16-byte chunks of a row, swizzled against bank conflicts
    static constexpr int TILE_BYTES = KEYS * HD * 2, STAGE_BYTES = 2 * TILE_BYTES;
    static constexpr int STAGES = HD <= 64 ? 4 : HD == 128 ? 3 : 3;
    static constexpr bool Q_IN_SMEM = HD == 256;                                    // a row's fragments would take 64 registers
    static constexpr int Q_BYTES = Q_IN_SMEM ? ROWS * HD * 2 : 0;
    static constexpr int MERGE_LD = HD + 8, MERGE_BYTES = 4 * 16 * (MERGE_LD + 4) * 4;
    static constexpr int RING_BYTES = STAGES * STAGE_BYTES > MERGE_BYTES ? STAGES * STAGE_BYTES : MERGE_BYTES;
    static constexpr int SMEM = Q_BYTES + RING_BYTES;
    __device__ static __forceinline__ int offset(int row, int chunk) { return (row * CHUNKS + (chunk ^ (row & SWZ))) * 16; }
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int HD, int WR>
__global__ void __launch_bounds__(THREADS) attention_tree_mma_kernel(const Params p) {
    using L = Layout<HD, WR>;
    constexpr int ROWS = L::ROWS, WK = L::WK, KW = L::KW, KB = KW / 16, STAGES = L::STAGES;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char* const q_s = smem;
    unsigned char* const ring = smem + L::Q_BYTES;
    __shared__ int ups[STAGED_NODES];
    __shared__ unsigned long long seen[ROWS];                        // of a key tile that needs it, by row: a bit a key
    __shared__ int lowest[ROWS];                                     // a row's first cached key
    __shared__ int latest;                                           // the largest of those
    pdl_enter();
    const int part = blockIdx.x % p.max_parts, kvh = blockIdx.x / p.max_parts % p.num_kv_heads, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int gid = lane >> 2, tig = lane & 3, wr = warp / WK, wk = warp % WK;
    const int group = p.num_heads / p.num_kv_heads;
    int r, within;
    Entry e;
    if (!tree::find_tile(p, blockIdx.x / p.max_parts / p.num_kv_heads, ROWS, r, e, within)) return;
    const int row0 = within * ROWS, count = min(ROWS, e.n * group - row0), last_node = (row0 + count - 1) / group;
    bool holes;                                                      // a page that is none has been met
    const int first = tree::first_key(p, e), end = tree::end_key(p, e, first, last_node, holes);     // the tile's keys: first .. end - 1
    const int tile0 = first / KEYS, tiles = (end - 1) / KEYS - tile0 + 1, parts = tree::parts_of(p, tiles);
    if (part >= parts) return;
    const int begin = tile0 + (int)((long long)tiles * part / parts), stop = tile0 + (int)((long long)tiles * (part + 1) / parts);
    const int* const table = p.block_table + (size_t)r * p.table_stride;
    const bf16* const q = static_cast<const bf16*>(p.q);
    const int D = p.head_dim;

    // A thread copies the same chunk of rows THREADS / CHUNKS apart, of a tile's keys and values; its rows' quarters have a place in the cache
    // each, looked up a tile ahead of the copies.
    constexpr int STEP = THREADS / L::CHUNKS > 0 ? THREADS / L::CHUNKS : 1, COPIES = KEYS / STEP;
    const int my_chunk = tid % L::CHUNKS, my_row = tid / L::CHUNKS;
    constexpr int LOOKUPS = STEP >= 16 ? COPIES : 4;                              // quarters that a thread's rows lie in
    auto look_up = [&](int tile, int (&page)[LOOKUPS]) {
#pragma unroll
        for (int i = 0; i < LOOKUPS; ++i) {
            const int quarter = STEP >= 16 ? (my_row + i * STEP) / 16 : i, at = tile * KEYS + quarter * 16, slot = at / p.page_size;
            const bool needed = tile < stop && at < end && at + 15 >= first;
            page[i] = needed && slot < p.table_pages ? __ldg(table + slot) : -1;
        }
    };
    auto load = [&](int tile, const int (&page)[LOOKUPS]) {
        unsigned char* const ks = ring + (tile - begin) % STAGES * L::STAGE_BYTES;
#pragma unroll
        for (int c = 0; c < COPIES; ++c) {
            const int row = my_row + c * STEP, at = tile * KEYS + row, here = page[STEP >= 16 ? c : c * STEP / 16];
            const bool needed = at >= first && at < end, valid = needed && here >= 0 && here < p.num_pages, copied = valid && my_chunk * 8 < D;
            if (needed && !valid) {
                holes = true;
                atomicOr(p.status, EG_STATUS_BAD_PAGE);
            }
            const size_t from = copied ? (size_t)here * p.page_stride + (size_t)kvh * p.head_stride + (size_t)(at % p.page_size) * D + my_chunk * 8 : 0;
            cp_async_16(ks + L::offset(row, my_chunk), static_cast<const bf16*>(p.k_cache) + from, copied);
            cp_async_16(ks + L::TILE_BYTES + L::offset(row, my_chunk), static_cast<const bf16*>(p.v_cache) + from, copied);
        }
    };
    // ---- the tree: parents of the nodes up to the tile's last one, and every row's first cached key
    // (what the next trip to memory brings is asked for before anything waits for it: block table, a parent a thread, rows of q)
    int ahead[LOOKUPS];
    look_up(begin, ahead);
    const int parent = tid <= last_node ? p.parents[e.first + tid] : -1;
    // ---- the rows of q as A fragments
    auto q_row = [&](int row) { return q + (size_t)(e.first + (row0 + row) / group) * p.ldq + (size_t)(kvh * group + (row0 + row) % group) * D; };
    uint32_t qf[L::Q_IN_SMEM ? 1 : HD / 16][4];
    if constexpr (L::Q_IN_SMEM) {
        for (int i = tid; i < ROWS * HD / 2; i += THREADS) {
            const int row = i / (HD / 2), pair = i % (HD / 2);
            *reinterpret_cast<uint32_t*>(q_s + L::offset(row, pair / 4) + pair % 4 * 4) = row < count && 2 * pair < D ? *reinterpret_cast<const uint32_t*>(q_row(row) + 2 * pair) : 0u;
        }
    } else {
        const int a = wr * 16 + gid, b = a + 8;
        const bf16* const qa = q_row(min(a, count - 1));
        const bf16* const qb = q_row(min(b, count - 1));
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
            const int d = k * 16 + 2 * tig;
            const bool low = d < D, high = d + 8 < D;
            qf[k][0] = a < count && low ? *reinterpret_cast<const uint32_t*>(qa + d) : 0u;
            qf[k][1] = b < count && low ? *reinterpret_cast<const uint32_t*>(qb + d) : 0u;
            qf[k][2] = a < count && high ? *reinterpret_cast<const uint32_t*>(qa + d + 8) : 0u;
            qf[k][3] = b < count && high ? *reinterpret_cast<const uint32_t*>(qb + d + 8) : 0u;
        }
    }
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
        int now[LOOKUPS];
#pragma unroll
        for (int i = 0; i < LOOKUPS; ++i) now[i] = ahead[i];
        look_up(begin + s + 1, ahead);
        if (begin + s < stop) load(begin + s, now);
        cp_async_commit();
    }
    if (tid <= last_node) ups[tid] = tree::sound_parent(p, tid, parent);
    for (int i = THREADS + tid; i <= last_node && i < STAGED_NODES; i += THREADS) ups[i] = tree::parent_of(p, e, i);
    if (tid == 0) latest = 0;
    auto up_of = [&](int i) { return i < STAGED_NODES ? ups[i] : tree::parent_of(p, e, i); };
    if (p.window > 0) {
        __syncthreads();
        if (tid < count) {
            int depth = 0;
            for (int i = up_of((row0 + tid) / group); i >= 0; i = up_of(i)) ++depth;
            lowest[tid] = (int)max(0ll, (long long)e.context + depth - p.window + 1);
            atomicMax(&latest, lowest[tid]);
        }
    } else if (tid < count) {
        lowest[tid] = 0;
    }

    const float scale_log2 = p.scale * 1.4426950408889634f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, acc[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    const bool idle = wr * 16 >= count;                              // a warp whose rows are all filling

    for (int tile = begin; tile < stop; ++tile) {
        cp_async_wait<STAGES - 2>();
        const bool checked = __syncthreads_or(holes);                // the same for all threads: pages are looked at again
        {
            int now[LOOKUPS];
#pragma unroll
            for (int i = 0; i < LOOKUPS; ++i) now[i] = ahead[i];
            const int next = tile + STAGES - 1;
            if (next < stop) {
                look_up(next + 1, ahead);
                load(next, now);
            }
            cp_async_commit();
        }
        const unsigned char* const ks = ring + (tile - begin) % STAGES * L::STAGE_BYTES;
        unsigned char* const vs = const_cast<unsigned char*>(ks) + L::TILE_BYTES;
        const int key0 = tile * KEYS;
        const bool masked = key0 + KEYS > e.context || key0 < max(first, latest) || checked;
        bool odd = false;                                            // values that are not finite, in a tile with masks: the same for all threads
        if (masked) {
            if (tid < ROWS) {
                unsigned long long bits = 0;
                if (tid < count) {
                    const int low = max(lowest[tid], key0), high = min(e.context, key0 + KEYS);
                    if (low < high) bits = ~0ull >> (KEYS - (high - low)) << (low - key0);
                    int left = p.window > 0 ? p.window : 0x7fffffff;
                    for (int i = (row0 + tid) / group; i >= 0 && e.context + i >= key0 && left > 0; i = up_of(i), --left)
                        if (e.context + i < key0 + KEYS) bits |= 1ull << (e.context + i - key0);
                }
                for (int quarter = 0; checked && quarter < 4; ++quarter) {
                    const int slot = (key0 + 16 * quarter) / p.page_size, page = slot < p.table_pages ? table[slot] : -1;
                    if (page < 0 || page >= p.num_pages) bits &= ~(0xffffull << (16 * quarter));
                }
                seen[tid] = bits;
            }
            unsigned largest = 0;
#pragma unroll 4
            for (int i = tid; i < KEYS * L::CHUNKS; i += THREADS) largest = tree::largest_halves(largest, *reinterpret_cast<const uint4*>(vs + i * 16));
            odd = __syncthreads_or(tree::not_finite(largest));
        }
        if (idle && !odd) continue;

        // ---- scores
        float s[2 * KB][4];
#pragma unroll
        for (int j = 0; j < 2 * KB; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
        const int mi = lane >> 3, mr = lane & 7;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
            uint32_t a[4];
            if constexpr (L::Q_IN_SMEM) {
                ldmatrix_x4(a, q_s + L::offset(wr * 16 + (mi & 1) * 8 + mr, 2 * k + (mi >> 1)));
            } else {
                a[0] = qf[k][0], a[1] = qf[k][1], a[2] = qf[k][2], a[3] = qf[k][3];
            }
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                uint32_t b[4];
                ldmatrix_x4(b, ks + L::offset(wk * KW + kb * 16 + (mi >> 1) * 8 + mr, 2 * k + (mi & 1)));
                mma_bf16_16816(s[2 * kb], a, b[0], b[1]);
                mma_bf16_16816(s[2 * kb + 1], a, b[2], b[3]);
            }
        }
        if (masked) {
            const unsigned long long a = seen[wr * 16 + gid] >> (wk * KW + 2 * tig), b = seen[wr * 16 + gid + 8] >> (wk * KW + 2 * tig);
#pragma unroll
            for (int j = 0; j < 2 * KB; ++j)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    if (!(a >> (8 * j + x) & 1)) s[j][x] = -INFINITY;
                    if (!(b >> (8 * j + x) & 1)) s[j][2 + x] = -INFINITY;
                }
        }
        // ---- running softmax; a row that has seen nothing keeps -inf, and 0 as the reference makes its weights 0
        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2 * KB; ++j) {
            t0 = fmaxf(t0, fmaxf(s[j][0], s[j][1]));
            t1 = fmaxf(t1, fmaxf(s[j][2], s[j][3]));
        }
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 1));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 1));
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, 2));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, 2));
        const float n0 = fmaxf(m0, t0 * scale_log2), n1 = fmaxf(m1, t1 * scale_log2);
        const float r0 = n0 == -INFINITY ? 0.f : n0, r1 = n1 == -INFINITY ? 0.f : n1;
        const float c0 = exp2_fast(m0 - r0), c1 = exp2_fast(m1 - r1);
        m0 = n0;
        m1 = n1;
        l0 *= c0;
        l1 *= c1;
        uint32_t pf[KB][4];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            float w[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                w[h][0] = exp2_fast(fmaf(s[2 * kb + h][0], scale_log2, -r0));
                w[h][1] = exp2_fast(fmaf(s[2 * kb + h][1], scale_log2, -r0));
                w[h][2] = exp2_fast(fmaf(s[2 * kb + h][2], scale_log2, -r1));
                w[h][3] = exp2_fast(fmaf(s[2 * kb + h][3], scale_log2, -r1));
                l0 += w[h][0] + w[h][1];
                l1 += w[h][2] + w[h][3];
            }
            pf[kb][0] = pack_bf16(w[0][0], w[0][1]);
            pf[kb][1] = pack_bf16(w[0][2], w[0][3]);
            pf[kb][2] = pack_bf16(w[1][0], w[1][1]);
            pf[kb][3] = pack_bf16(w[1][2], w[1][3]);
        }
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) {
            acc[j][0] *= c0;
            acc[j][1] *= c0;
            acc[j][2] *= c1;
            acc[j][3] *= c1;
        }
        // ---- values that are not finite: they are added where they are seen (behind the scaling, whose factor may be 0), and zeros take part in the product
        if (odd) {
            for (int key = wk * KW; key < (wk + 1) * KW; ++key) {
                const bool a = seen[wr * 16 + gid] >> key & 1, b = seen[wr * 16 + gid + 8] >> key & 1;
#pragma unroll
                for (int j = 0; j < HD / 8; ++j) {
                    const bf16* const at = reinterpret_cast<const bf16*>(vs + L::offset(key, j)) + 2 * tig;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float v = __bfloat162float(at[x]);
                        if (isfinite(v)) continue;
                        if (a) acc[j][x] += v;
                        if (b) acc[j][2 + x] += v;
                    }
                }
            }
            __syncthreads();
            for (int i = tid; i < KEYS * HD; i += THREADS) {
                bf16* const at = reinterpret_cast<bf16*>(vs) + i;
                if (!isfinite(__bfloat162float(*at))) *at = __float2bfloat16_rn(0.f);
            }
            __syncthreads();
        }
        // ---- output
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) {
                uint32_t b[4];
                ldmatrix_x4_trans(b, vs + L::offset(wk * KW + kb * 16 + (mi & 1) * 8 + mr, 2 * j + (mi >> 1)));
                mma_bf16_16816(acc[2 * j], pf[kb], b[0], b[1]);
                mma_bf16_16816(acc[2 * j + 1], pf[kb], b[2], b[3]);
            }
    }
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);

    cp_async_wait<0>();
    auto line_of = [&](int row) {                                    // where a row's results go
        return static_cast<bf16*>(p.out) + (size_t)(e.first + (row0 + row) / group) * p.ldo + (size_t)(kvh * group + (row0 + row) % group) * D;
    };
    auto put4 = [&](int row, int d, float4 v) {
        uint32_t* const at = reinterpret_cast<uint32_t*>(line_of(row) + d);
        at[0] = pack_bf16(v.x, v.y);
        at[1] = pack_bf16(v.z, v.w);
    };
    if (WK == 1 && parts == 1) {
        const int a = wr * 16 + gid, b = a + 8;
        const float i0 = l0 > 0.f ? 1.f / l0 : l0, i1 = l1 > 0.f ? 1.f / l1 : l1;
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) {
            if (8 * j >= D) break;
            if (a < count) *reinterpret_cast<uint32_t*>(line_of(a) + 8 * j + 2 * tig) = pack_bf16(acc[j][0] * i0, acc[j][1] * i0);
            if (b < count) *reinterpret_cast<uint32_t*>(line_of(b) + 8 * j + 2 * tig) = pack_bf16(acc[j][2] * i1, acc[j][3] * i1);
        }
        return;
    }
    // ---- the warps that share rows, in the order of their keys, then the parts
    __syncthreads();
    float* const o_s = reinterpret_cast<float*>(ring);               // a line a warp and row
    float* const ml_s = o_s + 4 * 16 * L::MERGE_LD;
    float* const row_ml = ml_s + 2 * 4 * 16;                         // of the warps together
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) {
        *reinterpret_cast<float2*>(o_s + (warp * 16 + gid) * L::MERGE_LD + 8 * j + 2 * tig) = make_float2(acc[j][0], acc[j][1]);
        *reinterpret_cast<float2*>(o_s + (warp * 16 + gid + 8) * L::MERGE_LD + 8 * j + 2 * tig) = make_float2(acc[j][2], acc[j][3]);
    }
    if (tig == 0) {
        *reinterpret_cast<float2*>(ml_s + 2 * (warp * 16 + gid)) = make_float2(m0, l0);
        *reinterpret_cast<float2*>(ml_s + 2 * (warp * 16 + gid + 8)) = make_float2(m1, l1);
    }
    if constexpr (WK == 1) {
        tree::add_parts<THREADS>(o_s, L::MERGE_LD, ml_s, count, D, parts, put4);
    } else {
        __syncthreads();
        for (int i = tid; i < ROWS * (HD / 4); i += THREADS) {
            const int row = i / (HD / 4), d = i % (HD / 4) * 4, line0 = row / 16 * WK * 16 + row % 16;
            float top = -INFINITY, total = 0.f;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WK; ++w) top = fmaxf(top, ml_s[(line0 + 16 * w) * 2]);
#pragma unroll
            for (int w = 0; w < WK; ++w) {
                const float2 ml = *reinterpret_cast<const float2*>(ml_s + (line0 + 16 * w) * 2);
                const float c = ml.x == -INFINITY ? 0.f : exp2_fast(ml.x - top);
                const float4 o = *reinterpret_cast<const float4*>(o_s + (line0 + 16 * w) * L::MERGE_LD + d);
                total = fmaf(c, ml.y, total);
                sum = make_float4(fmaf(c, o.x, sum.x), fmaf(c, o.y, sum.y), fmaf(c, o.z, sum.z), fmaf(c, o.w, sum.w));
            }
            if (parts == 1) {
                const float inv = total > 0.f ? 1.f / total : total;
                if (row < count && d < D) put4(row, d, make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv));
            } else {                                                 // into its own line: nobody else reads this quad
                *reinterpret_cast<float4*>(o_s + line0 * L::MERGE_LD + d) = sum;
                if (d == 0) *reinterpret_cast<float2*>(row_ml + 2 * row) = make_float2(top, total);
            }
        }
        if (parts > 1) {
            // the lines of a row group lie WK * 16 apart
            if constexpr (WK == 4) tree::add_parts<THREADS>(o_s, L::MERGE_LD, row_ml, count, D, parts, put4);
            else {
                __syncthreads();
                for (int i = tid; i < 16 * (HD / 4); i += THREADS)   // the second group's to behind the first's
                    *reinterpret_cast<float4*>(o_s + (16 + i / (HD / 4)) * L::MERGE_LD + i % (HD / 4) * 4) =
                        *reinterpret_cast<const float4*>(o_s + (32 + i / (HD / 4)) * L::MERGE_LD + i % (HD / 4) * 4);
                tree::add_parts<THREADS>(o_s, L::MERGE_LD, row_ml, count, D, parts, put4);
            }
        }
    }
}

template <int HD, int WR>
int launch(cudaStream_t stream, const Params& p, long long tiles) {
    constexpr int bytes = Layout<HD, WR>::SMEM;
    static unsigned long long seen = 0;
    if (const int code = tree::prepare_kernel(attention_tree_mma_kernel<HD, WR>, bytes, seen)) return code;
    return tree::launch_clusters(attention_tree_mma_kernel<HD, WR>, p.max_parts, p.num_kv_heads, tiles, THREADS, bytes, stream, p);
}

}  // namespace

namespace tree {

// Rows per CTA 16, 32 or 64; tiles of 64 keys.  The caller has checked what this kernel takes.
int launch_mma(cudaStream_t stream, const Params& p, int row_tile, long long tiles) {
#define EG_ROWS(HD) (row_tile == 16 ? launch<HD, 1>(stream, p, tiles) : row_tile == 32 ? launch<HD, 2>(stream, p, tiles) : launch<HD, 4>(stream, p, tiles))
    return p.head_dim <= 32 ? EG_ROWS(32) : p.head_dim <= 64 ? EG_ROWS(64) : p.head_dim <= 128 ? EG_ROWS(128) : EG_ROWS(256);
#undef EG_ROWS
}

}  // namespace tree
