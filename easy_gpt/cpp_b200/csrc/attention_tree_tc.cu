// Attention over drafted trees and the paged cache (attention_tree.cuh says which keys a row sees) on the 5th-generation tensor cores: bfloat16,
// heads of 64 and 128, pages of a multiple of 16 tokens, rows on 16-byte boundaries.
//
// A CTA takes the nodes of an entry whose rows (node, query head of a KV head's group) fill the 128 lanes of a tile, and a part of the keys, 64 at a
// time:
//   S = Q K^T    tcgen05.mma, Q and K tiles K-major in shared memory (K by TMA through the block table), S in TMEM
//   P = softmax  four warps, a row a thread: S out of TMEM, reference and sum in registers, P back over S as bfloat16 pairs
//   O += P V     tcgen05.mma, P from TMEM, V by TMA, O in TMEM
// The reference of the exponents follows a row's maximum lazily: it moves, and the row's O with it, only when the maximum has grown by 2^8.
// A row is a thread and a warp's rows exponentiate at the unit's rate (512 cycles a tile and SM, against 128 or 256 for the two products), so two
// CTAs share an SM (256 columns of TMEM and less than half the shared memory each), one's exponents beside the other's products and waits.
//
// Warps: 0 loads keys and 6 values, 1 allocates TMEM and issues the scores' products, 7 the output's, 2 to 5 have the rows.  (One thread for both products
// was slower: 16 requests of up to 32,768 keys 464 us against 393.  So were two tiles of rows a CTA, 256 threads of rows that share keys and values: 520 to
// 560, with the two exponentiating at the same time.)
// Keys and values have rings of their own, since a key stage is free long before the value stage of its tile: when its scores are there.  A piece of a tile that no row sees, or whose page is none, is
// read from behind the last row of the cache map, which gives zeros.  Every wait is bounded; a role that gives up raises the CTA's abort flag, the
// loader waits for its copies, and the CTA leaves as it always does.
//
// Masks: only tiles that reach into the tree, over a window's edge or onto a page that is none look at which keys a row sees, as 64 bits a row.  Hidden
// scores are replaced.  A hidden value meets a weight of zero, which hides all but infinities and NaN: such tiles look for those, put zeros in their
// place, and at the end, if there were any, every row adds those that it does see.
#define EG_NEEDS_TENSOR_MAPS
#include "attention_tree.cuh"
#include "tcgen05_attention.cuh"

namespace {

using namespace tc05;
using tree::Entry;
using tree::Params;

constexpr int KEYS = 64, THREADS = 256, STAGED_NODES = 512;
constexpr float REFERENCE_SLACK = 8.f;

template <int HD>
struct Shape {
    static constexpr int SUBS = HD / 64, STAGES = HD == 64 ? 5 : 2, SCORES = HD == 64 ? 3 : 2;      // stages of keys and of values, TMEM buffers of S and P
    static constexpr int Q_SUB_BYTES = BM * SUB_ROW_BYTES, SUB_BYTES = KEYS * SUB_ROW_BYTES, TILE_BYTES = SUBS * SUB_BYTES;
    static constexpr int Q_BYTES = SUBS * Q_SUB_BYTES, SMEM = Q_BYTES + 2 * STAGES * TILE_BYTES + 1024;
    static constexpr int O_COL = SCORES * KEYS, TMEM_COLS = 256, OUT_LD = HD + 4;
    static_assert(O_COL + HD <= TMEM_COLS, "TMEM columns");
    static_assert(BM * (OUT_LD + 2) * 4 <= SMEM - 1024, "a part's results in the tiles' place");
};

struct Maps {
    int nodes, piece_rows, nowhere;                                  // nodes of a tile; keys a box holds; the row behind the cache maps' last
    long long page_rows, head_rows;
};

template <int HD>
__global__ void __launch_bounds__(THREADS, 2)
attention_tree_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Params p, const Maps maps) {
    using S = Shape<HD>;
    constexpr int STAGES = S::STAGES, SCORES = S::SCORES;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t q_full, k_full[STAGES], v_full[STAGES], k_empty[STAGES], v_empty[STAGES], s_full[SCORES], p_full[SCORES], o_done[SCORES];
    __shared__ int ups[STAGED_NODES];
    __shared__ float row_ml[2 * BM];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, latest, holes, poison;                // poison: values that are not finite have been met, and zeroed
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = blockIdx.x % p.max_parts, kvh = blockIdx.x / p.max_parts % p.num_kv_heads;
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_addr = base, k_ring = base + S::Q_BYTES, v_ring = k_ring + STAGES * S::TILE_BYTES;
    unsigned char* const aligned = smem_raw + (base - smem_addr(smem_raw));
    pdl_wait();
    const int group = p.num_heads / p.num_kv_heads;
    int r, within;
    Entry e;
    if (!tree::find_tile(p, blockIdx.x / p.max_parts / p.num_kv_heads, maps.nodes * group, r, e, within)) return;
    const int node0 = within * maps.nodes, nodes = min(maps.nodes, e.n - node0), count = nodes * group, last_node = node0 + nodes - 1;
    bool beyond;
    const int first = tree::first_key(p, e), end = tree::end_key(p, e, first, last_node, beyond);    // the tile's keys: first .. end - 1
    const int tile0 = first / KEYS, tiles = (end - 1) / KEYS - tile0 + 1, parts = tree::parts_of(p, tiles);
    if (part >= parts) return;
    const int begin = tile0 + (int)((long long)tiles * part / parts), ntiles = tile0 + (int)((long long)tiles * (part + 1) / parts) - begin;
    const int* const table = p.block_table + (size_t)r * p.table_stride;
    const int row_warps = (count + 31) / 32;

    // ---- loaders: a lane a box (64 columns, piece_rows keys) of every tile; its page is looked up a tile ahead
    const bool is_v = warp == 6, loader = warp == 0 || is_v;
    const int pieces = KEYS / maps.piece_rows, piece = lane % pieces, sub = lane / pieces;
    const bool loads = loader && lane < pieces * S::SUBS;
    constexpr int NOT_NEEDED = -2;
    auto page_of = [&](int j) {
        const int key = (begin + j) * KEYS + piece * maps.piece_rows, slot = key / p.page_size;
        if (j >= ntiles || key >= end || key + maps.piece_rows <= first) return NOT_NEEDED;
        return slot < p.table_pages ? max(__ldg(table + slot), -1) : -1;
    };
    int page_ahead = loads ? page_of(0) : NOT_NEEDED;
    // ---- rows: a thread's row of q and a node's parent are asked for in the same trip
    const int quad = warp & 3, row = quad * 32 + lane;               // (of warps 2 to 5) a warp may touch the TMEM lanes 32 (warp % 4) ..
    const bool has_rows = warp >= 2 && warp < 6 && quad < row_warps, valid = has_rows && row < count;
    const int node = node0 + min(row, count - 1) / group, head = kvh * group + row % group;
    uint4 q_row[HD / 8];
    const uint4* const q_from = reinterpret_cast<const uint4*>(static_cast<const bf16*>(p.q) + (size_t)(e.first + node) * p.ldq + (size_t)head * HD);
#pragma unroll
    for (int c = 0; c < HD / 8; ++c) q_row[c] = valid ? __ldg(q_from + c) : make_uint4(0, 0, 0, 0);
    const int parent = has_rows && row <= last_node ? p.parents[e.first + row] : -1;
    if (threadIdx.x == 0) {
        mbar_init(&q_full, row_warps);
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < SCORES; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], row_warps);
            mbar_init(&o_done[i], 1);
        }
        abort_flag = latest = poison = 0;
        holes = beyond;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(&tmem_slot)), "r"(S::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_start_next();                                                // not before this CTA has its tensor memory
    const uint32_t tmem = tmem_slot;

    // a row's result, its columns c0 .. c0 + 31
    bool rows_done = false;
    float row_scale = 1.f;
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16), o_lanes = lanes + S::O_COL;
    auto up_of = [&](int i) { return i < STAGED_NODES ? ups[i] : tree::parent_of(p, e, i); };
    int lowest = 0;
    // which of a key tile's keys the row sees
    auto seen_of = [&](int key0) {
        unsigned long long bits = 0;
        const int low = max(max(lowest, first), key0), high = min(e.context, key0 + KEYS);
        if (low < high) bits = ~0ull >> (KEYS - (high - low)) << (low - key0);
        int left = p.window > 0 ? p.window : 0x7fffffff;
        for (int i = node; i >= 0 && e.context + i >= key0 && left > 0; i = up_of(i), --left)
            if (e.context + i < key0 + KEYS) bits |= 1ull << (e.context + i - key0);
        if (holes)
            for (int quarter = 0; quarter < 4; ++quarter) {
                const int slot = (key0 + 16 * quarter) / p.page_size, page = slot < p.table_pages ? table[slot] : -1;
                if (page < 0 || page >= p.num_pages) bits &= ~(0xffffull << (16 * quarter));
            }
        return bits;
    };

    if (loader) {
        uint64_t* const full = is_v ? v_full : k_full;
        uint64_t* const empty = is_v ? v_empty : k_empty;
        const uint32_t ring = is_v ? v_ring : k_ring;
        const CUtensorMap* const map = is_v ? &map_v : &map_k;
        int issued = 0;
        for (int j = 0; j < ntiles; ++j, ++issued) {
            const int st = j % STAGES, use = j / STAGES;
            const int page = page_ahead;
            if (loads) page_ahead = page_of(j + 1);
            if (use > 0 && !__all_sync(0xffffffffu, lane > 0 || mbar_wait(&empty[st], (use - 1) & 1, &abort_flag, p.status))) break;
            int at = maps.nowhere;
            if (loads && page != NOT_NEEDED) {
                if (page < 0 || page >= p.num_pages) {
                    atomicOr(p.status, EG_STATUS_BAD_PAGE);
                    *(volatile int*)&holes = 1;
                } else {
                    at = (int)(page * maps.page_rows + kvh * maps.head_rows + ((begin + j) * KEYS + piece * maps.piece_rows) % p.page_size);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_expect_tx(&full[st], S::TILE_BYTES);
            __syncwarp();
            if (loads) tma_load_2d(ring + st * S::TILE_BYTES + sub * S::SUB_BYTES + piece * maps.piece_rows * SUB_ROW_BYTES, map, &full[st], sub * 64, at);
        }
        // every copy has to land before the CTA gives up its shared memory, also when a role has given up
        if (lane == 0 && *(volatile int*)&abort_flag)
            for (int j = issued > STAGES ? issued - STAGES : 0; j < issued; ++j) mbar_wait_plain(&full[j % STAGES], (j / STAGES) & 1);
    } else if (warp == 1) {
        if (lane == 0) {                                             // ---- S_j = Q K_j^T; descriptors differ in their low words
            const uint32_t product = idesc(KEYS, false), hi = (uint32_t)(desc_k_major(0) >> 32), q_lo = (uint32_t)desc_k_major(q_addr);
            uint32_t k_lo = (uint32_t)desc_k_major(k_ring);
            bool ok = mbar_wait(&q_full, 0, &abort_flag, p.status);
            int stage = 0, phase = 0, b = 0, b_phase = 1;            // of the key ring; of the score buffers
            for (int j = 0; j < ntiles && ok; ++j) {
                // S goes where S and P of SCORES tiles before were: the product that read that P must be done
                ok = mbar_wait(&k_full[stage], phase, &abort_flag, p.status) && (j < SCORES || mbar_wait(&o_done[b], b_phase, &abort_flag, p.status));
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem + (uint32_t)(b * KEYS);
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                    const uint64_t x = desc_from(q_lo + (uint32_t)((k / 4 * S::Q_SUB_BYTES + k % 4 * 32) >> 4), hi);
                    const uint64_t y = desc_from(k_lo + (uint32_t)((k / 4 * S::SUB_BYTES + k % 4 * 32) >> 4), hi);
                    if (k == 0) tc_mma<false>(d, x, y, product);
                    else tc_mma<true>(d, x, y, product);
                }
                tc_commit(&s_full[b]);
                tc_commit(&k_empty[stage]);
                k_lo += S::TILE_BYTES >> 4;
                if (++stage == STAGES) stage = 0, phase ^= 1, k_lo -= (STAGES * S::TILE_BYTES) >> 4;
                if (++b == SCORES) b = 0, b_phase ^= 1;
            }
        }
    } else if (warp == 7) {
        if (lane == 0) {                                             // ---- O += P_j V_j
            const uint32_t product = idesc(HD, true), hi = (uint32_t)(desc_k_major(0) >> 32), d = tmem + (uint32_t)S::O_COL;
            uint32_t v_lo = (uint32_t)desc_n_major(v_ring, S::SUB_BYTES);
            int stage = 0, phase = 0, b = 0, b_phase = 0;
            for (int j = 0; j < ntiles; ++j) {
                if (!mbar_wait(&v_full[stage], phase, &abort_flag, p.status) || !mbar_wait(&p_full[b], b_phase, &abort_flag, p.status)) break;
                tc_fence_after();
                const uint32_t weights = tmem + (uint32_t)(b * KEYS);
#pragma unroll
                for (int k = 0; k < KEYS / 16; ++k) {
                    const uint64_t y = desc_from(v_lo + (uint32_t)((k * 2048) >> 4), hi);
                    if (k == 0 && j == 0) tc_mma_a_tmem<false>(d, weights, y, product);
                    else tc_mma_a_tmem<true>(d, weights + (uint32_t)(k * 8), y, product);
                }
                tc_commit(&o_done[b]);
                tc_commit(&v_empty[stage]);
                v_lo += S::TILE_BYTES >> 4;
                if (++stage == STAGES) stage = 0, phase ^= 1, v_lo -= (STAGES * S::TILE_BYTES) >> 4;
                if (++b == SCORES) b = 0, b_phase ^= 1;
            }
        }
    } else if (has_rows) {
        // ---- the rows: q into shared memory, the tree, then a key tile at a time
        const int row_threads = row_warps * 32;
        auto rows_barrier = [&]() { asm volatile("bar.sync 1, %0;\n" ::"r"(row_threads) : "memory"); };
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) *reinterpret_cast<uint4*>(aligned + c / 8 * S::Q_SUB_BYTES + row * SUB_ROW_BYTES + ((c % 8) ^ (row & 7)) * 16) = q_row[c];
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full);
        if (row <= last_node) ups[row] = tree::sound_parent(p, row, parent);
        for (int i = row_threads + row; i <= last_node && i < STAGED_NODES; i += row_threads) ups[i] = tree::parent_of(p, e, i);
        rows_barrier();
        if (p.window > 0) {
            int depth = 0;
            for (int i = up_of(node); i >= 0; i = up_of(i)) ++depth;
            lowest = (int)max(0ll, (long long)e.context + depth - p.window + 1);
            if (valid) atomicMax(&latest, lowest);
            rows_barrier();
        }
        const int edge = max(first, latest);
        const float scale_log2 = p.scale * 1.4426950408889634f;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; j < ntiles; ++j) {
            const int b = j % SCORES, key0 = (begin + j) * KEYS;
            ok = __all_sync(0xffffffffu, mbar_wait(&s_full[b], (j / SCORES) & 1, &abort_flag, p.status));      // the warp stays together
            if (!ok) break;
            tc_fence_after();
            float s[64];
            {
                uint32_t r0[32], r1[32];
                tmem_ld32(lanes + (uint32_t)(b * KEYS), r0);
                tmem_ld32(lanes + (uint32_t)(b * KEYS + 32), r1);
                tmem_ld_wait();
#pragma unroll
                for (int x = 0; x < 32; ++x) {
                    s[x] = __uint_as_float(r0[x]);
                    s[32 + x] = __uint_as_float(r1[x]);
                }
            }
            if (key0 + KEYS > e.context || key0 < edge || *(volatile int*)&holes) {
                const unsigned long long bits = seen_of(key0);
#pragma unroll
                for (int x = 0; x < 64; ++x)
                    if (!(bits >> x & 1)) s[x] = -INFINITY;
            }
            // (a hole's values are zeros.  Every warp looks at the whole tile, so that none waits for another: a warp whose wait gave up would not come.  What one
            // has zeroed another may not meet any more, so the flag is all warps')
            if (key0 + KEYS > e.context || key0 < edge) {
                ok = __all_sync(0xffffffffu, mbar_wait(&v_full[j % STAGES], (j / STAGES) & 1, &abort_flag, p.status));
                if (!ok) break;
                unsigned char* const values = aligned + S::Q_BYTES + (STAGES + j % STAGES) * S::TILE_BYTES;
                // the keys that not every row sees: below the edge, in the tree
                const int from = key0 < edge ? 0 : max(0, e.context - key0), to = key0 + KEYS > e.context ? KEYS : min(KEYS, edge - key0);
                uint32_t largest = 0;
#pragma unroll
                for (int sub_tile = 0; sub_tile < S::SUBS; ++sub_tile)
#pragma unroll 4
                    for (int i = from * 8 + lane; i < to * 8; i += 32)
                        largest = tree::largest_halves(largest, *reinterpret_cast<const uint4*>(values + sub_tile * S::SUB_BYTES + i * 16));
                if (__any_sync(0xffffffffu, tree::not_finite(largest))) {
                    *(volatile int*)&poison = 1;
                    __threadfence_block();
                    for (int i = lane; i < S::TILE_BYTES / 2; i += 32) {
                        bf16* const at = reinterpret_cast<bf16*>(values) + i;
                        if (!isfinite(__bfloat162float(*at))) *at = __float2bfloat16_rn(0.f);
                    }
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                }
            }
            // the row's maximum with the three-input instruction: 64 -> 22 -> 8 -> 3 -> 1
            float t[22];
#pragma unroll
            for (int x = 0; x < 21; ++x) t[x] = max3(s[3 * x], s[3 * x + 1], s[3 * x + 2]);
            t[21] = s[63];
#pragma unroll
            for (int x = 0; x < 7; ++x) t[x] = max3(t[3 * x], t[3 * x + 1], t[3 * x + 2]);
            t[0] = max3(t[0], t[1], t[2]);
            t[1] = max3(t[3], t[4], t[5]);
            const float most = max3(t[0], t[1], fmaxf(t[6], t[21])) * scale_log2;
            float c = 1.f;
            if (most > m + REFERENCE_SLACK) {                        // also the first finite maximum (m = -inf)
                c = exp2_approx(m - most);                           // 0 for the first
                m = most;
            }
            const float ref = m == -INFINITY ? 0.f : m;              // a row that has seen nothing: weights 0
            if (j > 0 && __any_sync(0xffffffffu, c != 1.f)) {
                ok = __all_sync(0xffffffffu, mbar_wait(&o_done[(j - 1) % SCORES], ((j - 1) / SCORES) & 1, &abort_flag, p.status));
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int c0 = 0; c0 < HD; c0 += 16) {
                    uint32_t v[16];
                    tmem_ld16(o_lanes + (uint32_t)c0, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int x = 0; x < 16; ++x) v[x] = __float_as_uint(__uint_as_float(v[x]) * c);
                    tmem_st16(o_lanes + (uint32_t)c0, v);
                }
            }
            uint64_t sums = 0;
            const uint64_t scale2 = pair_of(scale_log2, scale_log2), shift2 = pair_of(-ref, -ref);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t packed[16];
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    float x0, x1;
                    split_pair(fma_pair(pair_of(s[32 * half + 2 * x], s[32 * half + 2 * x + 1]), scale2, shift2), x0, x1);
                    const float w0 = exp2_approx(x0), w1 = exp2_approx(x1);
                    sums = add_pair(sums, pair_of(w0, w1));
                    packed[x] = pack2(w0, w1);
                }
                tmem_st16(lanes + (uint32_t)(b * KEYS + 16 * half), packed);
            }
            float sum0, sum1;
            split_pair(sums, sum0, sum1);
            l = l * c + (sum0 + sum1);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[b]);
        }
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&o_done[(ntiles - 1) % SCORES], ((ntiles - 1) / SCORES) & 1, &abort_flag, p.status));
        tc_fence_after();
        rows_done = ok;
        const bool poisoned = *(volatile int*)&poison;               // every warp has been through every tile: the last product waited for their weights
        row_scale = parts > 1 ? 1.f : l > 0.f ? 1.f / l : l;         // nothing seen: 0; NaN stays
        row_ml[2 * row] = rows_done ? m : -INFINITY;
        row_ml[2 * row + 1] = rows_done ? l : 0.f;
        if (rows_done) {
            bf16* const line = static_cast<bf16*>(p.out) + (size_t)(e.first + node) * p.ldo + (size_t)head * HD;
            float* const part_line = reinterpret_cast<float*>(aligned) + row * S::OUT_LD;
#pragma unroll
            for (int c0 = 0; c0 < HD; c0 += 32) {
                uint32_t o[32];
                tmem_ld32(o_lanes + (uint32_t)c0, o);
                tmem_ld_wait();
                float v[32];
#pragma unroll
                for (int x = 0; x < 32; ++x) v[x] = __uint_as_float(o[x]);
                if (poisoned)                                        // values that are not finite, where they are seen
                    for (int j = 0; j < ntiles; ++j) {
                        const int key0 = (begin + j) * KEYS;
                        if (key0 + KEYS <= e.context && key0 >= edge) continue;
                        for (unsigned long long bits = seen_of(key0); bits; bits &= bits - 1) {
                            const int key = key0 + __ffsll((long long)bits) - 1;
                            const bf16* const at = static_cast<const bf16*>(p.v_cache) + (size_t)table[key / p.page_size] * p.page_stride + (size_t)kvh * p.head_stride +
                                                   (size_t)(key % p.page_size) * HD + c0;
#pragma unroll
                            for (int x = 0; x < 32; ++x) {
                                const float z = __bfloat162float(at[x]);
                                if (!isfinite(z)) v[x] += z;
                            }
                        }
                    }
                if (parts > 1) {
#pragma unroll
                    for (int x = 0; x < 32; x += 4) *reinterpret_cast<float4*>(part_line + c0 + x) = make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]);
                } else if (valid) {
#pragma unroll
                    for (int x = 0; x < 32; x += 8)
                        *reinterpret_cast<uint4*>(line + c0 + x) =
                            make_uint4(pack2(v[x] * row_scale, v[x + 1] * row_scale), pack2(v[x + 2] * row_scale, v[x + 3] * row_scale),
                                       pack2(v[x + 4] * row_scale, v[x + 5] * row_scale), pack2(v[x + 6] * row_scale, v[x + 7] * row_scale));
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(S::TMEM_COLS) : "memory");
    if (parts > 1)
        tree::add_parts<THREADS>(reinterpret_cast<const float*>(aligned), S::OUT_LD, row_ml, count, HD, parts, [&](int line, int d, float4 v) {
            uint2* const at = reinterpret_cast<uint2*>(static_cast<bf16*>(p.out) + (size_t)(e.first + node0 + line / group) * p.ldo +
                                                       (size_t)(kvh * group + line % group) * HD + d);
            *at = make_uint2(pack2(v.x, v.y), pack2(v.z, v.w));
        });
}

template <int HD>
int launch(cudaStream_t stream, const Params& p, const Maps& maps, const CUtensorMap& map_k, const CUtensorMap& map_v, long long tiles) {
    constexpr int bytes = Shape<HD>::SMEM;
    static unsigned long long seen = 0;
    if (const int code = tree::prepare_kernel(attention_tree_tc_kernel<HD>, bytes, seen)) return code;
    return tree::launch_clusters(attention_tree_tc_kernel<HD>, p.max_parts, p.num_kv_heads, tiles, THREADS, bytes, stream, map_k, map_v, p, maps);
}

}  // namespace

namespace tree {

int launch_tc(cudaStream_t stream, const Params& p) {
    const int group = p.num_heads / p.num_kv_heads;
    Maps maps;
    maps.nodes = BM / group;
    maps.piece_rows = p.page_size % 64 == 0 ? 64 : p.page_size % 32 == 0 ? 32 : 16;
    maps.page_rows = p.page_stride / p.head_dim;
    maps.head_rows = p.head_stride / p.head_dim;
    const long long kv_rows = (long long)(p.num_pages - 1) * maps.page_rows + (long long)(p.num_kv_heads - 1) * maps.head_rows + p.page_size;
    const long long tiles = (long long)p.rows / maps.nodes + p.entries;
    if (kv_rows >= (1ll << 31)) return (int)cudaErrorInvalidValue;
    maps.nowhere = (int)kv_rows;
    CUtensorMap map_k, map_v;
    if (make_map(&map_k, p.k_cache, kv_rows, p.head_dim, p.head_dim, maps.piece_rows) || make_map(&map_v, p.v_cache, kv_rows, p.head_dim, p.head_dim, maps.piece_rows))
        return (int)cudaErrorInvalidValue;
    return p.head_dim == 64 ? launch<64>(stream, p, maps, map_k, map_v, tiles) : launch<128>(stream, p, maps, map_k, map_v, tiles);
}

}  // namespace tree
