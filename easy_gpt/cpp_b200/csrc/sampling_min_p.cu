// Sampling with temperature, top-k, top-p and min-p from given uniform numbers, on float32 logits.
//
// With x the logits of a row, T its temperature and m the largest logit, w_i = exp((x_i - m) / T).  What is kept, one rule after the other:
//   top-k    the k largest, if 0 < k < V                                     (ties: the lower index)
//   top-p    of those in descending order the shortest run from the top whose weights reach p of all of theirs, one at least, if 0 < p < 1
//   min-p    of those the ones with w_i >= min_p (the largest has w = 1), if min_p > 0; min_p above 1 counts as 1
// and of what is kept the first token in the order of the indices whose running sum of weights passes u times their sum.  T <= 0 (or NaN):
// the largest, the lower index on a tie.  u below 0 or NaN is 0, and with 1 or more the last token that is kept is drawn.  NaN is never kept, -inf
// has no weight; with +inf among the logits only those have one.  A row without a number above -inf gives 0.
//
// Each of the three cuts keeps a run from the top of the row's descending order.  A token's decision hangs on sums over a whole vocabulary,
// and a uniform number may lie next to a token's border; so weights are taken in 64 bits (off by at most 2^-46 of themselves) and summed as whole numbers
// of 2^-42 (rounded, by 2^-43 at most), whose sums are the same in every order (shared-memory atomics among them).  Tokens below half of that have no weight.
//
// A row is a cluster's, up to 16 CTAs with a slice of it each in shared memory, so that it is read once however often it is passed over.
// What most rows come to is a short list: the k largest, or what min-p or top-p leave.  The tokens that can be among those, at most 1,024, go to the
// first CTA, which puts them in order and has all three cuts and the draw among them.  With top-k they are those that are not below the k-th
// largest of the maxima of at least 2 k groups of tokens; with min-p its threshold says it; with top-p alone a histogram over 512 equal steps below the largest logit, of
// counts and weights.  A row that keeps more finds the last token of top-k's and top-p's runs by such histograms, refined until a step's tokens
// are a short list (or all equal); then every CTA sums what is kept of its slice, and the one in whose part the draw falls finds it.
//
// (A histogram's weights are three sums of 14 bits each: shared-memory atomics on 64 bits are loops of compare-and-swap, 5 to 18 times slower.)
//
// Measured, one row and 192 rows of 151,936 (0.6 MB and 117 MB) with logits of a spread of 1 to 4, us: greedy 4.8 and 49, top-k 20 7.1 and 64, min-p 0.05 10.8 and 92,
// nothing cut 9.5 and 112, top-p 0.95 alone 28 and 328, at a temperature of 3 31 and 355.  One row is bound by latency: the load 1.6, an exchange over the cluster 1
// each.  Many rows are 296 CTAs at a time, 8 us each when greedy, of which the load is half; flat rows are bound by weights in 64 bits (0.65 cycles a token
// and SM a pass) and histograms.
#include "common.cuh"

namespace {

typedef unsigned long long u64;

constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 512, LIST = 1024, SHORT = 128, MOST_CTAS = 16, GROUPS = 1024;
constexpr int LIMBS = 3, LIMB_BITS = 14;                             // of a weight, at most 2^42: sums of 2^17 of them stay below 2^32
constexpr int SLICE = 20480, MOST_SLICE = 49664;                     // logits of a slice: two CTAs an SM, and what fits at all
constexpr double ONE = 4398046511104.0;                              // 2^42: with 2^20 tokens sums stay below 2^62
constexpr int MOST_TOKENS = 1 << 20;
constexpr float COUNT_RANGE = 32.f, WEIGHT_RANGE = 16.f;             // what a histogram's steps span below the largest logit; of weights in units of T
constexpr float NO_WEIGHT = 31.f;                                    // exp(-31) 2^42 < 1/4

// larger numbers have larger keys; NaN has key 0
__device__ __forceinline__ unsigned key_of(float x) {
    if (!(x == x)) return 0u;
    const unsigned b = __float_as_uint(x == 0.f ? 0.f : x);          // -0 is 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
constexpr unsigned MINUS_INFINITY_KEY = 0x007fffffu;
// A token as one number that is the larger the further in front it is in the descending order: its key, then the lower index.
__device__ __forceinline__ u64 token_of(unsigned key, int index) { return (u64)key << 32 | (0xffffffffu - (unsigned)index); }
__device__ __forceinline__ int index_of(u64 token) { return (int)(0xffffffffu - (unsigned)token); }

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned cluster_size() {
    unsigned n;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
    return n;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// the address of CTA `rank`'s copy of a shared variable
__device__ __forceinline__ unsigned remote(const void* mine, unsigned rank) {
    unsigned a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((unsigned)__cvta_generic_to_shared(mine)), "r"(rank));
    return a;
}
__device__ __forceinline__ void remote_store(unsigned at, u64 a, u64 b) { asm volatile("st.shared::cluster.v2.u64 [%0], {%1, %2};" ::"r"(at), "l"(a), "l"(b) : "memory"); }
__device__ __forceinline__ void remote_store(unsigned at, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); }
__device__ __forceinline__ void remote_store(unsigned at, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }
__device__ __forceinline__ unsigned remote_load(unsigned at) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ unsigned remote_add(unsigned at, unsigned n) {
    unsigned v;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(v) : "r"(at), "r"(n) : "memory");
    return v;
}

constexpr int POWERS = 16;                                           // 2^(i / 16): 128 bytes, so that no two lanes meet a bank with different entries

struct Shared {
    double power[POWERS];
    __align__(16) u64 slot[2][MOST_CTAS][2];                                       // what the CTAs tell each other, in turn
    u64 warp_a[WARPS], warp_b[WARPS];
    u64 list[LIST];
    __align__(16) u64 weights[LIST];                                 // of the list; a histogram's sums over the CTAs, count and weight a step
    float group_most[GROUPS], own_most[THREADS];
    unsigned bin_weight[LIMBS][BINS], bin_count[BINS];
    unsigned listed, gathered, room;
    int found;
    float floats[WARPS];
    u64 pair[4];
};

static_assert(sizeof(Shared) + MOST_SLICE * 4 <= 227 * 1024, "shared memory of a CTA");

// the sum (or the maximum) over the CTA
template <bool MAX>
__device__ __forceinline__ u64 block_join(u64 a, Shared& s) {
    auto join = [](u64 x, u64 y) { return MAX ? (x > y ? x : y) : x + y; };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a = join(a, __shfl_xor_sync(0xffffffffu, a, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.warp_a[threadIdx.x >> 5] = a;
    __syncthreads();
    a = s.warp_a[threadIdx.x & (WARPS - 1)];
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) a = join(a, __shfl_xor_sync(0xffffffffu, a, o));
    return a;
}
// the inclusive sums of a pair over the CTA's threads
__device__ __forceinline__ void block_scan(u64& a, u64& b, Shared& s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const u64 x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) a += x, b += y;
    }
    __syncthreads();
    if (lane == 31) s.warp_a[warp] = a, s.warp_b[warp] = b;
    __syncthreads();
    u64 x = lane < warp ? s.warp_a[lane] : 0, y = lane < warp ? s.warp_b[lane] : 0;
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
    }
    a += __shfl_sync(0xffffffffu, x, 0);
    b += __shfl_sync(0xffffffffu, y, 0);
}

// Descending, n a power of two up to 2 THREADS.  A thread has two neighbours in registers; their partners up to 32 places away are in its warp, the others
// come through shared memory.  (A row of 151,936 with top-k 500, two sorts: 17 us, 20 with all stages there.)
__device__ __forceinline__ void sort_descending(u64* list, int n) {
    const int t = threadIdx.x;
    const bool mine = t < n / 2;
    __syncthreads();
    u64 x = mine ? list[2 * t] : 0, y = mine ? list[2 * t + 1] : 0;
    for (int size = 2; size <= n; size *= 2) {
        const bool falls = (2 * t & size) == 0;
        for (int step = size / 2; step > 1; step /= 2) {
            u64 px, py;
            if (step > 32) {
                __syncthreads();
                if (mine) list[2 * t] = x, list[2 * t + 1] = y;
                __syncthreads();
                px = mine ? list[2 * t ^ step] : 0;
                py = mine ? list[(2 * t ^ step) + 1] : 0;
            } else {
                px = __shfl_xor_sync(0xffffffffu, x, step / 2);
                py = __shfl_xor_sync(0xffffffffu, y, step / 2);
            }
            const bool larger = ((2 * t & step) == 0) == falls;      // this place keeps the larger of the two
            x = (px > x) == larger ? px : x;
            y = (py > y) == larger ? py : y;
        }
        if ((x < y) == falls) {
            const u64 z = x;
            x = y;
            y = z;
        }
    }
    __syncthreads();
    if (mine) list[2 * t] = x, list[2 * t + 1] = y;
    __syncthreads();
}
__device__ __forceinline__ int power_of_two(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

// RESIDENT: the slice is in shared memory; else (vocabularies beyond what 16 CTAs hold) it is read from memory at every pass.  PICKED: rows by their
// numbers (0.2 us a row more: a trip to memory in front of the others).
template <bool RESIDENT, bool PICKED>
__global__ void __launch_bounds__(THREADS, 2)
sample_min_p_kernel(const float* __restrict__ logits, long long ld, int vocab, int slice, const float* __restrict__ temperature, const int* __restrict__ top_k,
                    const float* __restrict__ top_p, const float* __restrict__ min_p, const float* __restrict__ uniform, int* __restrict__ out,
                    const int* __restrict__ which, int rows) {
    extern __shared__ __align__(16) float slice_s[];
    __shared__ Shared s;
    const unsigned rank = cluster_rank(), ctas = cluster_size();
    const int nth = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int lo = min(vocab, (int)rank * slice), n = min(vocab, lo + slice) - lo;      // this CTA's tokens: lo .. lo + n - 1
    const float* const row_there = logits + (size_t)nth * ld + lo;
    static_assert(BINS == THREADS, "a thread a step");
    auto clear_bins = [&]() { s.bin_count[tid] = s.bin_weight[0][tid] = s.bin_weight[1][tid] = s.bin_weight[2][tid] = 0; };
    clear_bins();
    if (tid == 0) s.listed = s.gathered = 0;
    if (tid < POWERS) s.power[tid] = exp2((double)tid / POWERS);
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");      // the others may write here once they know that this CTA runs
    pdl_enter();
    const int r = PICKED ? which[nth] : nth;
    if (PICKED && (r < 0 || r >= rows)) {                            // no row of the batch: the whole cluster leaves
        asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
        return;
    }
    const float* const row = PICKED ? logits + (size_t)r * ld + lo : row_there;      // (the address in front of the wait: 64 rows of 32,001 21.0 us, 20.5 so)
    const float T = temperature[r], p = top_p[r], u = uniform[r];
    const int k = top_k[r];
    const double least = (double)fminf(min_p[r], 1.f) * ONE;         // NaN: 1, which only the largest pass
    if constexpr (RESIDENT) {
        const unsigned to = (unsigned)__cvta_generic_to_shared(slice_s);
        if ((uintptr_t)row % 16 == 0) {
            for (int i = tid; i < n / 4; i += THREADS) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to + 16 * i), "l"(row + 4 * i));
            for (int i = n / 4 * 4 + tid; i < n; i += THREADS) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(to + 4 * i), "l"(row + i));
        } else {
            for (int i = tid; i < n; i += THREADS) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(to + 4 * i), "l"(row + i));
        }
        asm volatile("cp.async.commit_group;\n cp.async.wait_group 0;\n" ::: "memory");
        __syncthreads();
    }
    // f(x, i) for the thread's tokens of from .. to - 1 (a multiple of 4), `threads` of them sharing these; several at a time, so that
    // their chains of operations overlap.  Tokens below `least_logit` may be left out.
    auto for_some = [&](int from, int to, int thread, int threads, float least_logit, auto f) {
        if constexpr (RESIDENT) {
            for (int i = from + 4 * thread; i + 3 < to; i += 4 * threads) {
                const float4 v = *reinterpret_cast<const float4*>(slice_s + i);
                if (fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) < least_logit) continue;
                f(v.x, i);
                f(v.y, i + 1);
                f(v.z, i + 2);
                f(v.w, i + 3);
            }
            for (int i = from + (to - from) / 4 * 4 + thread; i < to; i += threads) f(slice_s[i], i);
        } else {
            for (int i = from + thread; i < to; i += threads) f(__ldg(row + i), i);
        }
    };
    auto for_all = [&](float least_logit, auto f) { for_some(0, n, tid, THREADS, least_logit, f); };
    auto at = [&](int i) { return RESIDENT ? slice_s[i] : __ldg(row + i); };

    int turn = 0;
    // every CTA's pair, after a barrier: what the CTAs in front of this one have (front), and all of them
    auto exchange = [&](u64 a, u64 b, bool max, u64 (&all)[2], u64& front) {
        if (tid < (int)ctas) remote_store(remote(&s.slot[turn][rank][0], tid), a, b);
        cluster_barrier();
        all[0] = all[1] = front = 0;
#pragma unroll
        for (unsigned c = 0; c < MOST_CTAS; ++c) {
            if (c >= ctas) break;
            const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&s.slot[turn][c][0]);
            all[0] = max ? (v.x > all[0] ? v.x : all[0]) : all[0] + v.x;
            all[1] = max ? (v.y > all[1] ? v.y : all[1]) : all[1] + v.y;
            if (c < rank) front += v.x;
        }
        turn ^= 1;                                                   // a slot is written again behind another barrier, which its readers have to reach
    };
    u64 all[2], front;

    // ---- the largest logit; with top-k that of at least 2 k groups of 1 to 512 threads too, which every CTA gets
    const bool k_on = k > 0 && k < vocab, p_on = p > 0.f && p < 1.f, m_on = least > 0.0;
    float most = -INFINITY;                                          // NaN is passed over
    for_all(-INFINITY, [&](float x, int) { most = fmaxf(most, x); });
    int width = THREADS;
    while (width > 1 && (int)ctas * (THREADS / width) < max(4, 2 * min(k, GROUPS))) width /= 2;
    const int own_groups = THREADS / width, groups = (int)ctas * own_groups;
    const bool grouped = k_on && groups >= 2 * k && groups <= GROUPS;
    if (width == 1) s.own_most[tid] = most;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        if (2 * o == width && lane % width == 0) s.own_most[tid / width] = most;
    }
    if (lane == 0) s.floats[warp] = most;
    __syncthreads();
    most = s.floats[lane & (WARPS - 1)];
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    if (grouped)
        for (int i = tid; i < groups; i += THREADS) {                // one of this CTA's groups for one CTA
            const int group = i / (int)ctas;
            float value = width <= 32 ? s.own_most[group] : -INFINITY;
            if (width > 32)
                for (int w = 0; w < width / 32; ++w) value = fmaxf(value, s.floats[group * (width / 32) + w]);
            remote_store(remote(&s.group_most[(int)rank * own_groups + group], i % ctas), value);
        }
    exchange(key_of(most), 0, true, all, front);
    const unsigned top = (unsigned)all[0];
    const float largest = value_of(top);
    if (top <= MINUS_INFINITY_KEY) {
        if (rank == 0 && tid == 0) out[r] = 0;
        return;
    }
    if (!(T > 0.f)) {                                                // the first of the largest
        u64 best = 0;
        for_all(largest, [&](float x, int i) {
            const u64 token = x == largest ? token_of(top, lo + i) : 0;
            best = token > best ? token : best;
        });
        best = block_join<true>(best, s);
        exchange(best, 0, true, all, front);
        if (rank == 0 && tid == 0) out[r] = index_of(all[0]);
        return;
    }
    // exp(t) for t in -31 .. 0 as 2^(n / 16) exp(z) with n the whole number next to 16 t / ln 2 and |z| <= a = ln 2 / 32.  The powers up to z^5 / 120 leave
    // z^6 / 720, up to 1.4e-13 and always above; of it 3 a^2 z^4 / 2 - 9 a^4 z^2 / 16, which differs from z^6 by at most a^6 / 16 (by the Chebyshev polynomial of
    // that degree, whose constant is left out), goes into the coefficients of z^4 and z^2: 9e-15 are left, 2^-46, beside the 2^-43 of rounding to whole 2^-42.
    // n = 16 e + i, a table has 2^(i / 16), and adding e + 42 to its exponent scales it to whole 2^-42.  Adding 1.5 2^52 and
    // taking it off rounds to a whole number, which then stands in the low bits.  No branches, so that several tokens' chains overlap.  (192 rows of
    // 151,936, nothing cut: with exp() 194 us, with 64 powers 130, so 112.)
    const double per_step = POWERS / 0.69314718055994530942 / (double)T, step_size = 0.69314718055994530942 / POWERS;
    const double top_value = (double)largest;
    const float no_weight = largest < INFINITY ? NO_WEIGHT * T : -1.f;      // with +inf the largest, +inf alone has a weight
    auto weight = [&](float x) -> u64 {
        constexpr double WHOLE = 6755399441055744.0;                 // 1.5 2^52
        const double y = ((double)x - top_value) * per_step, shifted = y + WHOLE;
        const int whole = __double2loint(shifted);                   // n
        const double z = (y - (shifted - WHOLE)) * step_size;
        const double power = s.power[whole & (POWERS - 1)];
        const double scaled = __hiloint2double(__double2hiint(power) + ((whole >> 4) + 42 << 20), __double2loint(power));
        constexpr double A2 = 0.69314718055994530942 / 32 * (0.69314718055994530942 / 32), FOURTH = 1.0 / 24 + A2 / 480, SECOND = 0.5 - A2 * A2 / 1280;
        const double series = fma(fma(fma(fma(z, 1.0 / 120, FOURTH), z, 1.0 / 6), z, SECOND), z * z, z);
        const double w = fma(scaled, series, scaled) + WHOLE;        // exp(z) = 1 + series
        const u64 found = (u64)__double_as_longlong(w) & 0x7ffffffffffffull;
        const bool some = x > -INFINITY && largest - x <= no_weight; // (a NaN has none)
        return x == largest ? (u64)ONE : some ? found : 0;
    };
    const float weighty = largest < INFINITY ? largest - NO_WEIGHT * T * 1.0001f - 1e-5f * fabsf(largest) : largest;      // nothing below it has a weight

    // ---- the short list, in the first CTA: every CTA gathers its own tokens and finds room for all of them at once (192 rows of 151,936 with top-k 500: 113 us,
    // 117 with a remote atomic a token)
    auto put_in_list = [&](u64 token) {
        const unsigned place = atomicAdd(&s.gathered, 1u);
        if (place < LIST) s.weights[place] = token;
    };
    auto send_list = [&]() {
        __syncthreads();
        const unsigned mine = s.gathered;
        if (tid == 0 && mine) s.room = remote_add(remote(&s.listed, 0), mine);
        __syncthreads();
        for (unsigned i = tid; i < mine && i < LIST && s.room + i < LIST; i += THREADS) remote_store(remote(&s.list[s.room + i], 0), s.weights[i]);
        if (tid == 0) s.gathered = 0;
        cluster_barrier();
    };
    // The first token whose running sum passes u times the whole: at least 1, and at most the whole itself (u from 1 on, where the product may
    // be beyond 64 bits).
    auto goal_of = [&](u64 total) -> u64 {
        const double asked = (double)u * (double)total;
        if (!(asked > 0)) return 1;                                  // (NaN too)
        return asked < (double)total ? min((u64)asked + 1, total) : total;
    };
    // The list's cuts and the draw.  by_k: top-k is still to be cut, and top-p goes by what that leaves; else by `whole`.
    auto draw_from_list = [&](int listed, bool by_k, u64 whole) {
        const int kept_k = by_k ? min(k, listed) : listed;
        if (listed <= SHORT) {                                       // places by counting: four threads a token
            static_assert(THREADS == 4 * SHORT, "four threads a token");
            const int e = tid / 4, part = tid % 4;
            if (tid < listed) s.weights[tid] = weight(value_of((unsigned)(s.list[tid] >> 32)));
            __syncthreads();
            const u64 token = e < listed ? s.list[e] : 0, w = e < listed ? s.weights[e] : 0;
            int place = 0;
            u64 before = 0;
            for (int j = part; j < listed; j += 4) {
                const bool ahead = s.list[j] > token;
                place += ahead;
                before += ahead ? s.weights[j] : 0;
            }
#pragma unroll
            for (int o = 1; o < 4; o *= 2) {
                place += __shfl_xor_sync(0xffffffffu, place, o);
                before += __shfl_xor_sync(0xffffffffu, before, o);
            }
            const bool in_k = e < listed && place < kept_k;
            if (in_k && place == kept_k - 1 && part == 0) s.pair[0] = before + w;      // the weights of all k
            __syncthreads();
            if (by_k) whole = s.pair[0];
            const bool kept = in_k && (place == 0 || !p_on || (double)before < (double)p * (double)whole) && (double)w >= least;
            if (part == 0 && e < listed) s.weights[e] = kept ? w : 0;
            __syncthreads();
            u64 upto = 0, total = 0;
            for (int j = part; j < listed; j += 4) {
                const u64 v = s.weights[j];
                total += v;
                upto += (unsigned)s.list[j] >= (unsigned)token ? v : 0;                // lower indices have larger low halves
            }
#pragma unroll
            for (int o = 1; o < 4; o *= 2) {
                upto += __shfl_xor_sync(0xffffffffu, upto, o);
                total += __shfl_xor_sync(0xffffffffu, total, o);
            }
            const u64 goal = goal_of(total);
            if (kept && part == 0 && upto >= goal && upto - w < goal) out[r] = index_of(token);
            return;
        }
        const int padded = power_of_two(listed);
        for (int i = listed + tid; i < padded; i += THREADS) s.list[i] = 0;
        sort_descending(s.list, padded);
        u64 w[2], c[2];                                              // a thread has two neighbours of the list
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = 2 * tid + h;
            w[h] = i < kept_k ? weight(value_of((unsigned)(s.list[i] >> 32))) : 0;
            if (i < kept_k) s.weights[i] = w[h];
        }
        u64 sum = w[0] + w[1], unused = 0;
        block_scan(sum, unused, s);
        c[0] = sum - w[0] - w[1];
        c[1] = sum - w[1];
        if (tid == THREADS - 1) s.pair[0] = sum;
        __syncthreads();
        if (by_k) whole = s.pair[0];
        const double target = (double)p * (double)whole;
        u64 mine = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = 2 * tid + h;
            mine += i < kept_k && (i == 0 || !p_on || (double)c[h] < target) && (double)w[h] >= least;
        }
        const int kept = max(1, (int)block_join<false>(mine, s)), places = power_of_two(kept);
        // in the order of the indices: sorted by (all ones - index), with the place in the list beside it
        for (int i = tid; i < places; i += THREADS) s.list[i] = i < kept ? (s.list[i] & 0xffffffffu) << 32 | (unsigned)i : 0;
        sort_descending(s.list, places);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = 2 * tid + h;
            w[h] = i < kept ? s.weights[(unsigned)s.list[i]] : 0;
        }
        sum = w[0] + w[1];
        unused = 0;
        block_scan(sum, unused, s);
        if (tid == THREADS - 1) s.pair[1] = sum;
        __syncthreads();
        const u64 goal = goal_of(s.pair[1]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u64 upto = h ? sum : sum - w[1];
            if (upto >= goal && upto - w[h] < goal) out[r] = index_of(s.list[2 * tid + h] >> 32);
        }
    };
    // After the candidates have been put in the list: whether that was all (the draw is done then), or there are too many, which the first CTA tells
    // the others while it goes on.
    auto finish_list = [&](bool by_k, u64 whole) {
        send_list();
        bool done = true;
        if (rank == 0) {
            const unsigned listed = s.listed;
            done = listed <= LIST;
            if (tid < (int)ctas) remote_store(remote(&s.slot[turn][0][0], tid), (u64)done);
            asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
            if (done) draw_from_list((int)listed, by_k, whole);
            asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
            if (tid == 0) s.listed = 0;
        } else {
            cluster_barrier();
            done = s.slot[turn][0][0] != 0;
        }
        turn ^= 1;
        return done;
    };

    // ---- histograms: a logit's step, larger ones in front
    auto step_of = [&](float x, float scale) { return min(BINS - 1, (int)((largest - x) * scale)); };
    auto add_weight = [&](int step, u64 w) {
        atomicAdd(&s.bin_count[step], 1u);
#pragma unroll
        for (int h = 0; h < LIMBS; ++h) {
            const unsigned limb = (unsigned)(w >> (LIMB_BITS * h)) & (h < LIMBS - 1 ? (1u << LIMB_BITS) - 1 : ~0u);
            if (limb) atomicAdd(&s.bin_weight[h][step], limb);
        }
    };
    struct Cut {
        int step;
        u64 count_before, count, weight_before, weight_sum;
    };
    // After all CTAs have counted: the first step where `before` and the sums up to it reach the goal, which is a count, or a weight: `share` of all of
    // the histogram's (weight_goal < 0), or weight_goal.
    auto cut_at = [&](bool by_weight, u64 before, u64 goal, double share, double weight_goal) {
        __syncthreads();
        cluster_barrier();
        {   // every CTA adds up its share of the steps, a lane a CTA's part of a step, and each of these lanes tells one CTA the sum
            const int step = (int)rank * (BINS / (int)ctas) + tid / (int)ctas, of = tid % (int)ctas;
            u64 count = remote_load(remote(&s.bin_count[step], of)), weight = 0;
            if (by_weight) {
                unsigned v[LIMBS];
#pragma unroll
                for (int h = 0; h < LIMBS; ++h) v[h] = remote_load(remote(&s.bin_weight[h][step], of));
#pragma unroll
                for (int h = 0; h < LIMBS; ++h) weight += (u64)v[h] << (LIMB_BITS * h);
            }
            for (unsigned o = 1; o < ctas; o *= 2) {
                count += __shfl_xor_sync(0xffffffffu, count, o);
                weight += __shfl_xor_sync(0xffffffffu, weight, o);
            }
            remote_store(remote(&s.weights[2 * step], of), count, weight);
        }
        cluster_barrier();                                           // the histograms may be cleared now
        const u64 c = s.weights[2 * tid], w = s.weights[2 * tid + 1];
        u64 c_sum = c, w_sum = w;
        block_scan(c_sum, w_sum, s);
        if (tid == BINS - 1) s.pair[0] = w_sum;
        if (tid == 0) s.found = BINS - 1;
        __syncthreads();
        const u64 weight_sum = s.pair[0];
        if (weight_goal < 0) weight_goal = share * (double)weight_sum;
        if (by_weight ? w_sum > 0 && (double)(before + w_sum) >= weight_goal : before + c_sum >= goal) atomicMin(&s.found, tid);
        __syncthreads();
        if (tid == s.found) {
            s.pair[1] = c_sum - c;
            s.pair[2] = c;
            s.pair[3] = w_sum - w;
        }
        __syncthreads();
        const Cut cut = {s.found, s.pair[1], s.pair[2], s.pair[3], weight_sum};
        __syncthreads();
        return cut;
    };
    const float count_scale = BINS / COUNT_RANGE, weight_scale = BINS / (WEIGHT_RANGE * T);

    // ---- what is kept as a short list
    if (k_on && vocab <= LIST && !grouped) {
        for_all(-INFINITY, [&](float x, int i) {
            if (x > -INFINITY) put_in_list(token_of(key_of(x), lo + i));
        });
        finish_list(true, 0);
        return;
    }
    if (grouped) {
        // the k-th largest of the groups' maxima is no larger than the k-th largest logit; it is one of at most GROUPS numbers that every CTA has
        float border = -INFINITY;
        if (groups <= THREADS) {                                     // the one with k - 1 in front of it
            if (tid < groups) {
                const float mine = s.group_most[tid];
                int place = 0;
                for (int j = 0; j < groups; j += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(s.group_most + j);
                    place += (v.x > mine || (v.x == mine && j < tid)) + (v.y > mine || (v.y == mine && j + 1 < tid)) + (v.z > mine || (v.z == mine && j + 2 < tid)) +
                             (v.w > mine || (v.w == mine && j + 3 < tid));
                }
                if (place == k - 1) s.floats[0] = mine;
            }
            __syncthreads();
            border = s.floats[0];
        } else {                                                     // the lower end of the step with it
            for (int j = tid; j < groups; j += THREADS) atomicAdd(&s.bin_count[step_of(s.group_most[j], count_scale)], 1u);
            __syncthreads();
            u64 c = s.bin_count[tid], unused = 0;
            s.bin_count[tid] = 0;
            const u64 mine = c;
            block_scan(c, unused, s);
            if (c >= (u64)k && c - mine < (u64)k) s.found = tid;
            __syncthreads();
            border = s.found == BINS - 1 ? -INFINITY : largest == INFINITY ? largest : largest - (float)(s.found + 1) / count_scale * 1.0001f - 1e-5f * fabsf(largest);
        }
        for_all(border, [&](float x, int i) {
            if (x >= border && x > -INFINITY) put_in_list(token_of(key_of(x), lo + i));
        });
        if (finish_list(true, 0)) return;
    } else if (!k_on && (m_on || (vocab <= LIST && !p_on))) {
        u64 whole = 0;
        if (p_on) {
            u64 sum = 0;
            for_all(weighty, [&](float x, int) { sum += weight(x); });
            exchange(block_join<false>(sum, s), 0, false, all, front);
            whole = all[0];
        }
        // everything down to min-p's border and a little further (by more than a float's rounding moves it): the list's own cut is exact
        const float border = m_on ? largest + T * (logf(fminf(min_p[r], 1.f)) - 1e-3f) - 1e-5f * fabsf(largest) : -INFINITY;
        for_all(border, [&](float x, int i) {
            if (!(x < border) && x > -INFINITY) put_in_list(token_of(key_of(x), lo + i));
        });
        if (finish_list(false, whole)) return;
    }

    // ---- the last token that top-k and top-p keep: those from `last` on stay
    u64 last = (u64)(MINUS_INFINITY_KEY + 1) << 32;
    // Narrows a cut down to that token: of the tokens in the cut's step the first ones until before + theirs reach the goal.
    auto narrow = [&](bool by_weight, float scale, Cut cut, u64 count_goal, double weight_goal) {
        u64 before = by_weight ? cut.weight_before : cut.count_before, inside = cut.count;
        // keys that the step's tokens lie between (a little apart, for the roundings of step_of), narrowed as the step is refined
        const bool last_step = cut.step == BINS - 1;
        const float high = largest - (float)cut.step / scale, slack = 1e-5f * (fabsf(largest) + fabsf((float)cut.step / scale));
        unsigned high_key = cut.step && high + slack < largest ? key_of(high + slack) : top;
        unsigned low_key = last_step || !(high - 1.f / scale - slack > -INFINITY) ? MINUS_INFINITY_KEY + 1 : key_of(high - 1.f / scale - slack);
        auto is_inside = [&](float x, u64 token) {
            const unsigned key = (unsigned)(token >> 32);
            return token >= last && key >= low_key && key <= high_key && step_of(x, scale) == cut.step && (!by_weight || !last_step || weight(x) > 0);
        };
        while (inside > LIST) {
            if (high_key == low_key) break;
            const int shift = max(0, 32 - __clz(high_key - low_key) - 9);      // at most BINS steps of 2^shift keys
            clear_bins();                                            // every CTA has read the last ones
            __syncthreads();
            for_all(value_of(low_key), [&](float x, int i) {
                const unsigned key = key_of(x);
                if (!is_inside(x, token_of(key, lo + i))) return;
                if (by_weight) add_weight((high_key - key) >> shift, weight(x));
                else atomicAdd(&s.bin_count[(high_key - key) >> shift], 1u);
            });
            const Cut inner = cut_at(by_weight, before, count_goal, 0.0, weight_goal);
            before += by_weight ? inner.weight_before : inner.count_before;
            inside = inner.count;
            high_key -= (unsigned)inner.step << shift;
            if ((high_key - low_key) >> shift) low_key = high_key - ((1u << shift) - 1);
        }
        u64 result = 0;
        if (inside > LIST) {                                         // equal ones: as many as it takes, the first in the order of the indices
            const u64 each = by_weight ? weight(value_of(high_key)) : 1;
            const double need = by_weight ? ceil((weight_goal - (double)before) / (double)each) : (double)(count_goal - before);
            const u64 take = need < 1.0 ? 1 : need < (double)inside ? (u64)need : inside;
            const int run = (n + THREADS - 1) / THREADS, from = min(n, tid * run), to = min(n, from + run);
            auto counts = [&](int i) { return key_of(at(i)) == high_key && token_of(high_key, lo + i) >= last; };
            u64 mine = 0, unused = 0;
            for (int i = from; i < to; ++i) mine += counts(i);
            u64 upto = mine;
            block_scan(upto, unused, s);
            exchange(block_join<false>(mine, s), 0, false, all, front);
            upto += front;
            if (upto >= take && upto - mine < take) {                // one thread of the row's
                u64 so_far = upto - mine;
                for (int i = from; i < to; ++i)
                    if (counts(i) && ++so_far == take) result = token_of(high_key, lo + i);
            }
            result = block_join<true>(result, s);
        } else {
            for_all(value_of(low_key), [&](float x, int i) {
                const u64 token = token_of(key_of(x), lo + i);
                if (is_inside(x, token)) put_in_list(token);
            });
            send_list();
            const int listed = (int)s.listed;
            if (rank == 0 && listed <= SHORT) {                      // places by counting: four threads a token
                const int e = tid / 4, part = tid % 4;
                if (tid < listed) s.weights[tid] = by_weight ? weight(value_of((unsigned)(s.list[tid] >> 32))) : 1;
                __syncthreads();
                const u64 token = e < listed ? s.list[e] : 0;
                u64 ahead = 0;
                for (int j = part; j < listed; j += 4) ahead += s.list[j] > token ? s.weights[j] : 0;
#pragma unroll
                for (int o = 1; o < 4; o *= 2) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
                const bool kept = e < listed && (ahead == 0 || (by_weight ? (double)(before + ahead) < weight_goal : before + ahead < count_goal));
                result = ~block_join<true>(kept ? ~token : 0, s);    // the last of those
                if (tid == 0) s.listed = 0;
            } else if (rank == 0) {
                const int padded = power_of_two(listed);
                for (int i = listed + tid; i < padded; i += THREADS) s.list[i] = 0;
                sort_descending(s.list, padded);
                u64 v[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int i = 2 * tid + h;
                    v[h] = i >= listed ? 0 : by_weight ? weight(value_of((unsigned)(s.list[i] >> 32))) : 1;
                }
                u64 sum = v[0] + v[1], mine = 0, unused = 0;
                block_scan(sum, unused, s);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int i = 2 * tid + h;
                    const u64 reach = before + (h ? sum - v[1] : sum - v[0] - v[1]);
                    mine += i < listed && (i == 0 || (by_weight ? (double)reach < weight_goal : reach < count_goal));
                }
                result = s.list[max(1, (int)block_join<false>(mine, s)) - 1];
                if (tid == 0) s.listed = 0;
            }
        }
        exchange(result, 0, true, all, front);
        last = all[0];
    };
    if (k_on) {
        for_all(-INFINITY, [&](float x, int) {
            if (x > -INFINITY) atomicAdd(&s.bin_count[step_of(x, count_scale)], 1u);
        });
        const Cut cut = cut_at(false, 0, k, 0.0, 0.0);
        if (cut.count_before + cut.count >= (u64)k) narrow(false, count_scale, cut, k, 0.0);      // else there are no more than k
        clear_bins();
        __syncthreads();
    }
    if (p_on) {
        const float last_logit = value_of((unsigned)(last >> 32));
        const unsigned last_index = (unsigned)index_of(last);         // all ones while nothing is cut
        for_all(fmaxf(weighty, last_logit), [&](float x, int i) {
            const u64 w = weight(x);
            if (w > 0 && (x > last_logit || (x == last_logit && (unsigned)(lo + i) <= last_index))) add_weight(step_of(x, weight_scale), w);
        });
        const Cut cut = cut_at(true, 0, 0, (double)p, -1.0);
        if (cut.count_before + cut.count <= LIST) {
            for_all(weighty, [&](float x, int i) {
                const u64 token = token_of(key_of(x), lo + i);
                if (token >= last && step_of(x, weight_scale) <= cut.step && weight(x) > 0) put_in_list(token);
            });
            finish_list(false, cut.weight_sum);
            return;
        }
        narrow(true, weight_scale, cut, 0, (double)p * (double)cut.weight_sum);
    }

    // ---- the draw over the slices: a warp has a run of tokens
    const int run = ((n + WARPS - 1) / WARPS + 127) & ~127, from = min(n, warp * run), to = min(n, from + run);
    const u64 least_weight = least > 0.0 ? (u64)ceil(least) : 0;
    const float last_logit = value_of((unsigned)(last >> 32));
    const unsigned last_index = (unsigned)index_of(last);         // all ones while nothing is cut
    auto kept_weight = [&](float x, int i) -> u64 {
        const u64 w = weight(x);
        return (x > last_logit || (x == last_logit && (unsigned)(lo + i) <= last_index)) && w >= least_weight ? w : 0;
    };
    u64 mass = 0;
    for_some(from, to, lane, 32, fmaxf(weighty, last_logit), [&](float x, int i) { mass += kept_weight(x, i); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
    __syncthreads();
    if (lane == 0) s.warp_b[warp] = mass;
    __syncthreads();
    u64 block_mass = 0;
#pragma unroll
    for (int q = 0; q < WARPS; ++q) block_mass += s.warp_b[q];
    exchange(block_mass, 0, false, all, front);
    const u64 goal = goal_of(all[0]);
    if (goal <= front || goal > front + block_mass) return;
    // it is in this CTA: the warp's run with the draw, a few tokens a thread
    u64 upto = front;
    int q = 0;
    while (q < WARPS - 1 && upto + s.warp_b[q] < goal) upto += s.warp_b[q++];
    const int first = min(n, q * run), end = min(n, first + run), each = (end - first + THREADS - 1) / THREADS;
    const int mine_from = min(end, first + tid * each), mine_to = min(end, mine_from + each);
    u64 mine = 0, unused = 0;
    for (int i = mine_from; i < mine_to; ++i) mine += kept_weight(at(i), i);
    u64 scan = mine;
    block_scan(scan, unused, s);                                     // (it writes warp_b behind a barrier)
    upto += scan - mine;
    if (upto < goal && upto + mine >= goal)
        for (int i = mine_from; i < mine_to; ++i) {
            upto += kept_weight(at(i), i);
            if (upto >= goal) {
                out[r] = lo + i;
                break;
            }
        }
}

template <bool RESIDENT, bool PICKED>
int launch(cudaStream_t stream, int ctas, int slice, const float* logits, long long ld, int rows, int vocab, const float* temperature, const int* top_k, const float* top_p,
           const float* min_p, const float* uniform, int* out, const int* which, int picked) {
    const int bytes = RESIDENT ? slice * 4 : 0;
    const auto kernel = sample_min_p_kernel<RESIDENT, PICKED>;
    static unsigned long long seen = 0;
    int device;
    if (eg_first_on_device(seen, device)) {
        cudaError_t set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_SLICE * 4);
        if (set == cudaSuccess) set = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (set != cudaSuccess) return (int)set;
        eg_done_on_device(seen, device);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long long)picked * ctas));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = eg_pdl_on() ? 2 : 1;
    (void)cudaLaunchKernelEx(&cfg, kernel, logits, ld, vocab, slice, temperature, top_k, top_p, min_p, uniform, out, which, rows);
    return eg_launch_status();
}

}  // namespace

// the largest vocabulary that eg_sample_min_p takes
EG_API int eg_sample_min_p_most_tokens(void) { return MOST_TOKENS; }

// logits [rows, vocab] with row stride ld; temperature, top_k, top_p, min_p, uniform, out: [rows].  Of these the rows which[0 .. picked - 1]; numbers that no
// row has are passed over.
EG_API int eg_sample_min_p_rows(cudaStream_t stream, const float* logits, long long ld, int rows, int vocab, const float* temperature, const int* top_k, const float* top_p,
                                const float* min_p, const float* uniform, int* out, const int* which, int picked) {
    if (rows <= 0 || picked <= 0) return 0;
    if (vocab < 1 || vocab > MOST_TOKENS || picked > 0x7fffffff / MOST_CTAS) return (int)cudaErrorInvalidValue;
    // as many CTAs a row as its slices need, and for few rows more
    int ctas = 1;
    while (ctas < MOST_CTAS && ((long long)vocab > (long long)ctas * SLICE || (picked * ctas < 64 && vocab > ctas * 8192))) ctas *= 2;
    const int slice = ((vocab + ctas - 1) / ctas + 3) & ~3;
    const auto launch_it = slice <= MOST_SLICE ? (which ? launch<true, true> : launch<true, false>) : which ? launch<false, true> : launch<false, false>;
    return launch_it(stream, ctas, slice, logits, ld, rows, vocab, temperature, top_k, top_p, min_p, uniform, out, which, picked);
}

EG_API int eg_sample_min_p(cudaStream_t stream, const float* logits, long long ld, int rows, int vocab, const float* temperature, const int* top_k, const float* top_p,
                           const float* min_p, const float* uniform, int* out) {
    return eg_sample_min_p_rows(stream, logits, ld, rows, vocab, temperature, top_k, top_p, min_p, uniform, out, nullptr, rows);
}
