// Sampling with temperature, top-k, top-p and min-p from given uniform numbers, on float32 logits.
//
// With x the logits of a row, T its temperature and m the largest logit, w_i = exp((x_i - m) / T).  What is kept, one rule after the other:
//   top-k    the k largest, if 0 < k < V                                     (ties: the lower index)
//   top-p    of those in descending order the shortest run from the top whose weights reach p of all of theirs, one at least, if 0 < p < 1
//   min-p    of those the ones with w_i >= min_p (the largest has w = 1), if min_p > 0; min_p above 1 counts as 1
// and of what is kept the first token in the order of the indices whose running sum of weights passes u times their sum.  T <= 0 (or NaN):
// the largest, the lower index on a tie.  NaN is never kept, -inf has no weight; with +inf among the logits only those have one.  A row
// without a number above -inf gives 0.
//
// Each of the three cuts keeps a run from the top of the row's descending order.  A token's decision hangs on sums over a whole vocabulary,
// and a uniform number may lie next to a token's border; so weights are taken in 64 bits and summed as whole numbers of 2^-42, whose sums
// are the same in every order (shared-memory atomics among them).  Tokens below half of that have no weight.
//
// A row is a cluster's, up to 16 CTAs with a slice of it each in shared memory, so that it is read once however often it is passed over.
// What most rows come to is a short list: the k largest, or what min-p or top-p leave.  A histogram over 512 equal steps below the largest
// logit (of counts, or of weights too where top-p looks at the whole row) says up to which step; the tokens up to there, at most 1,024, go to
// the first CTA, which sorts them and has all three cuts and the draw among them.  A row that keeps more finds the last token of top-k's and
// top-p's runs by the same histogram, refined until a step's tokens are a short list (or all equal); then every CTA sums what is kept of its
// slice, and the one in whose part the draw falls finds it.
#include "common.cuh"

namespace {

typedef unsigned long long u64;

constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 512, LIST = 1024, MOST_CTAS = 16;
constexpr int SLICE = 20480, MOST_SLICE = 51200;                     // logits of a slice: two CTAs an SM, and what fits at all
constexpr double ONE = 4398046511104.0;                              // 2^42: with 2^20 tokens sums stay below 2^62
constexpr int MOST_TOKENS = 1 << 20;
constexpr float COUNT_RANGE = 32.f, WEIGHT_RANGE = 30.f;             // what a histogram's steps span below the largest logit; of weights in units of T
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
__device__ __forceinline__ void remote_store(unsigned at, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }
__device__ __forceinline__ u64 remote_load64(unsigned at) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
    return v;
}
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

struct Shared {
    u64 slot[2][MOST_CTAS][2];                                       // what the CTAs tell each other, in turn
    u64 warp_a[WARPS], warp_b[WARPS];
    u64 list[LIST], weights[LIST];
    u64 bin_weight[BINS];
    unsigned bin_count[BINS];
    unsigned listed;
    int found;
};

// sums (or maxima) of a pair over the CTA
template <bool MAX>
__device__ __forceinline__ void block_join(u64& a, u64& b, Shared& s) {
    auto join = [](u64 x, u64 y) { return MAX ? (x > y ? x : y) : x + y; };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a = join(a, __shfl_xor_sync(0xffffffffu, a, o));
        b = join(b, __shfl_xor_sync(0xffffffffu, b, o));
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
        s.warp_a[threadIdx.x >> 5] = a;
        s.warp_b[threadIdx.x >> 5] = b;
    }
    __syncthreads();
    a = s.warp_a[threadIdx.x & (WARPS - 1)];
    b = s.warp_b[threadIdx.x & (WARPS - 1)];
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) {
        a = join(a, __shfl_xor_sync(0xffffffffu, a, o));
        b = join(b, __shfl_xor_sync(0xffffffffu, b, o));
    }
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
    for (int w = 0; w < warp; ++w) a += s.warp_a[w], b += s.warp_b[w];
}

// descending, n a power of two
__device__ __forceinline__ void sort_descending(u64* list, int n) {
    for (int size = 2; size <= n; size *= 2)
        for (int step = size / 2; step > 0; step /= 2) {
            __syncthreads();
            for (int i = threadIdx.x; i < n / 2; i += THREADS) {
                const int a = 2 * i - (i & (step - 1)), b = a + step;
                const u64 x = list[a], y = list[b];
                if ((x < y) == ((a & size) == 0)) list[a] = y, list[b] = x;
            }
        }
    __syncthreads();
}
__device__ __forceinline__ int power_of_two(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

// RESIDENT: the slice is in shared memory; else (vocabularies beyond what 16 CTAs hold) it is read from memory at every pass.
template <bool RESIDENT>
__global__ void __launch_bounds__(THREADS)
sample_min_p_kernel(const float* __restrict__ logits, long long ld, int vocab, int slice, const float* __restrict__ temperature, const int* __restrict__ top_k,
                    const float* __restrict__ top_p, const float* __restrict__ min_p, const float* __restrict__ uniform, int* __restrict__ out) {
    extern __shared__ __align__(16) float slice_s[];
    __shared__ Shared s;
    const unsigned rank = cluster_rank(), ctas = cluster_size();
    const int r = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int lo = min(vocab, (int)rank * slice), n = min(vocab, lo + slice) - lo;      // this CTA's tokens: lo .. lo + n - 1
    const float* const row = logits + (size_t)r * ld + lo;
    for (int i = tid; i < BINS; i += THREADS) s.bin_count[i] = 0, s.bin_weight[i] = 0;
    if (tid == 0) s.listed = 0;
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");      // the others may write here once they know that this CTA runs
    pdl_enter();
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
    auto at = [&](int i) { return RESIDENT ? slice_s[i] : __ldg(row + i); };

    int turn = 0;
    // every CTA's pair, after a barrier: what the CTAs in front of this one have (front), and all of them
    auto exchange = [&](u64 a, u64 b, bool max, u64 (&all)[2], u64 (&front)[2]) {
        if (tid < (int)ctas) {
            const unsigned to = remote(&s.slot[turn][rank][0], tid);
            remote_store(to, a);
            remote_store(to + 8, b);
        }
        cluster_barrier();
        all[0] = all[1] = front[0] = front[1] = 0;
        for (unsigned c = 0; c < ctas; ++c)
            for (int h = 0; h < 2; ++h) {
                const u64 v = s.slot[turn][c][h];
                all[h] = max ? (v > all[h] ? v : all[h]) : all[h] + v;
                if (c < rank) front[h] += v;
            }
        turn ^= 1;                                                   // a slot is written again behind another barrier, which its readers have to reach
    };
    u64 all[2], front[2];

    // ---- the first token in the descending order
    u64 best = 0, none = 0;
    for (int i = tid; i < n; i += THREADS) {
        const u64 mine = token_of(key_of(at(i)), lo + i);
        best = mine > best ? mine : best;
    }
    block_join<true>(best, none, s);
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    exchange(best, 0, true, all, front);
    const unsigned top = (unsigned)(all[0] >> 32);
    const int first_best = index_of(all[0]);
    const float largest = value_of(top);
    if (!(T > 0.f) || top <= MINUS_INFINITY_KEY) {
        if (rank == 0 && tid == 0) out[r] = top <= MINUS_INFINITY_KEY ? 0 : first_best;
        return;
    }
    const double inverse = 1.0 / (double)T;
    const float no_weight = NO_WEIGHT * T;
    auto weight = [&](float x) -> u64 {
        if (x == largest) return (u64)ONE;                           // +inf too
        if (!(x > -INFINITY) || largest == INFINITY || largest - x > no_weight) return 0;
        return (u64)__double2ll_rn(exp(((double)x - (double)largest) * inverse) * ONE);
    };
    const bool k_on = k > 0 && k < vocab, p_on = p > 0.f && p < 1.f, m_on = least > 0.0;

    // A histogram's step of a logit, larger ones in front.
    auto step_of = [&](float x, float scale) { return min(BINS - 1, (int)((largest - x) * scale)); };
    // After all CTAs have counted: the sums of the steps up to the first one where they reach `goal` (of the counts, or `share` of the weights' sum).
    struct Cut {
        int step;
        u64 count_before, count, weight_before, weight, weight_sum;
    };
    auto cut_at = [&](bool by_weight, u64 goal, double share) {
        cluster_barrier();
        u64 c = 0, w = 0;
        for (unsigned q = 0; q < ctas; ++q) {
            c += remote_load(remote(&s.bin_count[tid], q));
            if (by_weight) w += remote_load64(remote(&s.bin_weight[tid], q));
        }
        u64 c_sum = c, w_sum = w;
        block_scan(c_sum, w_sum, s);
        u64* const totals = s.weights;                               // free between the lists
        if (tid == BINS - 1) totals[0] = w_sum;
        if (tid == 0) s.found = BINS - 1;
        __syncthreads();
        const double target = share * (double)totals[0];
        const bool reached = by_weight ? (double)w_sum >= target && w_sum > 0 : c_sum >= goal;
        if (reached) atomicMin(&s.found, tid);
        __syncthreads();
        if (tid == s.found) {
            totals[1] = c_sum - c;
            totals[2] = c;
            totals[3] = w_sum - w;
            totals[4] = w;
        }
        __syncthreads();
        const Cut cut = {s.found, totals[1], totals[2], totals[3], totals[4], totals[0]};
        __syncthreads();
        return cut;
    };
    static_assert(BINS == THREADS, "a thread a step");
    auto put_in_list = [&](u64 token) {
        const unsigned place = remote_add(remote(&s.listed, 0), 1);
        if (place < LIST) remote_store(remote(&s.list[place], 0), token);
    };

    // The list's cuts and the draw, by the first CTA.  by_k: top-k is still to be cut, and top-p goes by what that leaves; else by `whole`.
    auto finish_list = [&](bool by_k, u64 whole) {
        cluster_barrier();
        if (rank != 0) return;
        const int listed = (int)s.listed, padded = power_of_two(listed);
        for (int i = listed + tid; i < padded; i += THREADS) s.list[i] = 0;
        sort_descending(s.list, padded);
        const int kept_k = by_k ? min(k, listed) : listed;
        u64 w[2], c[2];                                              // a thread has two neighbours of the list
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = 2 * tid + h;
            w[h] = i < kept_k ? weight(value_of((unsigned)(s.list[i] >> 32))) : 0;
        }
        u64 sum = w[0] + w[1], unused = 0;
        block_scan(sum, unused, s);
        c[0] = sum - w[0] - w[1];
        c[1] = sum - w[1];
        __syncthreads();
        if (tid == THREADS - 1) s.warp_a[0] = sum;
        __syncthreads();
        if (by_k) whole = s.warp_a[0];
        const double target = (double)p * (double)whole;
        int mine = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = 2 * tid + h;
            mine += i < kept_k && (i == 0 || !p_on || (double)c[h] < target) && (double)w[h] >= least;
            if (i < kept_k) s.weights[i] = w[h];
        }
        u64 kept_sum = mine;
        unused = 0;
        block_join<false>(kept_sum, unused, s);
        const int kept = max(1, (int)kept_sum), places = power_of_two(kept);
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
        __syncthreads();
        if (tid == THREADS - 1) s.warp_a[0] = sum;
        __syncthreads();
        const u64 total = s.warp_a[0];
        const double asked = (double)u * (double)total;
        const u64 passed = asked > 0 ? (u64)asked + 1 : 1, goal = passed < total ? passed : total;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u64 upto = h ? sum : sum - w[1];
            if (upto >= goal && upto - w[h] < goal) out[r] = index_of(s.list[2 * tid + h] >> 32);
        }
    };

    // ---- what is kept as a short list
    const float count_scale = BINS / COUNT_RANGE, weight_scale = BINS / (WEIGHT_RANGE * T);
    Cut cut = {};
    if (k_on ? k <= LIST : !(p_on || m_on) ? vocab <= LIST : false) {
        if (vocab > LIST) {
            for (int i = tid; i < n; i += THREADS) {
                const float x = at(i);
                if (x > -INFINITY) atomicAdd(&s.bin_count[step_of(x, count_scale)], 1u);
            }
            __syncthreads();
            cut = cut_at(false, k, 0.0);
        }
        if (vocab <= LIST || cut.count_before + cut.count <= LIST) {
            for (int i = tid; i < n; i += THREADS) {
                const float x = at(i);
                if (x > -INFINITY && (vocab <= LIST || step_of(x, count_scale) <= cut.step)) put_in_list(token_of(key_of(x), lo + i));
            }
            finish_list(k_on, 0);
            return;
        }
    } else if (!k_on && m_on) {
        u64 count = 0, sum = 0;
        for (int i = tid; i < n; i += THREADS) {
            const u64 w = weight(at(i));
            count += (double)w >= least;
            sum += w;
        }
        block_join<false>(count, sum, s);
        exchange(count, sum, false, all, front);
        if (all[0] <= LIST) {
            const u64 whole = all[1];
            for (int i = tid; i < n; i += THREADS) {
                const float x = at(i);
                if ((double)weight(x) >= least) put_in_list(token_of(key_of(x), lo + i));
            }
            finish_list(false, whole);
            return;
        }
    }

    // ---- the last token that top-k and top-p keep: those from `last` on stay
    u64 last = (u64)(MINUS_INFINITY_KEY + 1) << 32;
    // Narrows a cut down to that token: of the tokens in the cut's step the first ones until before + theirs reach the goal.
    auto narrow = [&](bool by_weight, float scale, u64 count_goal, double weight_goal) {
        u64 before = by_weight ? cut.weight_before : cut.count_before, inside = cut.count;
        unsigned high_key = 0, low_key = 0;                          // of the step's tokens, once it has been refined
        bool by_step = true;
        auto is_inside = [&](float x, u64 token) {
            const unsigned key = (unsigned)(token >> 32);
            return token >= last && (by_step ? step_of(x, scale) == cut.step && (!by_weight || weight(x) > 0) : key >= low_key && key <= high_key);
        };
        while (inside > LIST) {
            if (by_step) {                                           // the step's tokens are those of a run of keys
                u64 a = 0, b = 0;
                for (int i = tid; i < n; i += THREADS) {
                    const float x = at(i);
                    const unsigned key = key_of(x);
                    if (is_inside(x, token_of(key, lo + i))) {
                        a = key > a ? key : a;
                        b = ~key > (unsigned)b ? ~key : b;
                    }
                }
                block_join<true>(a, b, s);
                exchange(a, b, true, all, front);
                high_key = (unsigned)all[0];
                low_key = ~(unsigned)all[1];
                by_step = false;
            }
            if (high_key == low_key) break;
            const int shift = max(0, 32 - __clz(high_key - low_key) - 9);      // at most BINS steps of 2^shift keys
            cluster_barrier();                                       // the last histogram has been read
            s.bin_count[tid] = 0;
            s.bin_weight[tid] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += THREADS) {
                const float x = at(i);
                const unsigned key = key_of(x);
                if (!is_inside(x, token_of(key, lo + i))) continue;
                atomicAdd(&s.bin_count[(high_key - key) >> shift], 1u);
                if (by_weight) atomicAdd(&s.bin_weight[(high_key - key) >> shift], weight(x));
            }
            __syncthreads();
            cluster_barrier();
            u64 c = 0, w = 0;
            for (unsigned q = 0; q < ctas; ++q) {
                c += remote_load(remote(&s.bin_count[tid], q));
                if (by_weight) w += remote_load64(remote(&s.bin_weight[tid], q));
            }
            u64 c_sum = c, w_sum = w;
            block_scan(c_sum, w_sum, s);
            if (tid == 0) s.found = BINS - 1;
            __syncthreads();
            if (by_weight ? (double)(before + w_sum) >= weight_goal : before + c_sum >= count_goal) atomicMin(&s.found, tid);
            __syncthreads();
            if (tid == s.found) {
                s.weights[0] = by_weight ? w_sum - w : c_sum - c;
                s.weights[1] = c;
            }
            __syncthreads();
            before += s.weights[0];
            inside = s.weights[1];
            high_key -= (unsigned)s.found << shift;
            if (high_key - low_key >> shift) low_key = high_key - ((1u << shift) - 1);
            __syncthreads();
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
            u64 upto = mine, block = mine;
            block_scan(upto, unused, s);
            unused = 0;
            block_join<false>(block, unused, s);
            exchange(block, 0, false, all, front);
            upto += front[0];
            if (upto >= take && upto - mine < take) {                // one thread of the row's
                u64 at_token = upto - mine;
                for (int i = from; i < to; ++i)
                    if (counts(i) && ++at_token == take) result = token_of(high_key, lo + i);
            }
            unused = 0;
            block_join<true>(result, unused, s);
        } else {
            for (int i = tid; i < n; i += THREADS) {
                const float x = at(i);
                const u64 token = token_of(key_of(x), lo + i);
                if (is_inside(x, token)) put_in_list(token);
            }
            cluster_barrier();
            if (rank == 0) {
                const int listed = (int)s.listed, padded = power_of_two(listed);
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
                unused = 0;
                block_join<false>(mine, unused, s);
                result = s.list[max(1, (int)mine) - 1];
                if (tid == 0) s.listed = 0;
            }
        }
        exchange(result, 0, true, all, front);
        last = all[0];
    };
    auto clear_bins = [&]() {
        cluster_barrier();
        s.bin_count[tid] = 0;
        s.bin_weight[tid] = 0;
        __syncthreads();
    };
    if (k_on) {
        if (k > LIST) {                                              // else it is there already
            for (int i = tid; i < n; i += THREADS) {
                const float x = at(i);
                if (x > -INFINITY) atomicAdd(&s.bin_count[step_of(x, count_scale)], 1u);
            }
            __syncthreads();
            cut = cut_at(false, k, 0.0);
        }
        if (cut.count_before + cut.count >= (u64)k) narrow(false, count_scale, k, 0.0);      // else there are no more than k
        if (p_on) clear_bins();
    }
    if (p_on) {
        for (int i = tid; i < n; i += THREADS) {
            const float x = at(i);
            if (token_of(key_of(x), lo + i) < last) continue;
            const u64 w = weight(x);
            if (w == 0) continue;
            const int b = step_of(x, weight_scale);
            atomicAdd(&s.bin_count[b], 1u);
            atomicAdd(&s.bin_weight[b], w);
        }
        __syncthreads();
        cut = cut_at(true, 0, (double)p);
        if (cut.count_before + cut.count <= LIST) {
            for (int i = tid; i < n; i += THREADS) {
                const float x = at(i);
                const u64 token = token_of(key_of(x), lo + i);
                if (token >= last && step_of(x, weight_scale) <= cut.step && weight(x) > 0) put_in_list(token);
            }
            finish_list(false, cut.weight_sum);
            return;
        }
        narrow(true, weight_scale, 0, (double)p * (double)cut.weight_sum);
    }

    // ---- the draw over the slices: a warp has a run of tokens, 32 at a time
    const int run = ((n + WARPS - 1) / WARPS + 31) & ~31, from = min(n, warp * run), to = min(n, from + run);
    auto kept_weight = [&](int i) -> u64 {
        const float x = i < to ? at(i) : NAN;
        if (token_of(key_of(x), lo + i) < last) return 0;
        const u64 w = weight(x);
        return (double)w >= least ? w : 0;
    };
    u64 mass = 0, unused = 0;
    for (int i = from; i < to; i += 32) mass += kept_weight(i + lane);
    u64 scan = mass;
    block_scan(scan, unused, s);
    const u64 before_warp = __shfl_sync(0xffffffffu, scan - mass, 0), upto_warp = __shfl_sync(0xffffffffu, scan, 31);
    u64 block_mass = mass;
    unused = 0;
    block_join<false>(block_mass, unused, s);
    exchange(block_mass, 0, false, all, front);
    // the running sum has to pass u times the whole: at least 1, and at most the whole itself
    const u64 total = all[0];
    const double asked = (double)u * (double)total;
    const u64 passed = asked > 0 ? (u64)asked + 1 : 1, goal = passed < total ? passed : total;
    u64 upto = front[0] + before_warp;
    if (goal > upto && goal <= front[0] + upto_warp) {
        for (int i = from; i < to; i += 32) {
            u64 w = kept_weight(i + lane);
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const u64 x = __shfl_up_sync(0xffffffffu, w, o);
                if (lane >= o) w += x;
            }
            const unsigned past = __ballot_sync(0xffffffffu, upto + w >= goal);
            if (past) {
                if (lane == 0) out[r] = lo + i + __ffs(past) - 1;
                break;
            }
            upto += __shfl_sync(0xffffffffu, w, 31);
        }
    }
}

template <bool RESIDENT>
int launch(cudaStream_t stream, int ctas, int slice, const float* logits, long long ld, int rows, int vocab, const float* temperature, const int* top_k, const float* top_p,
           const float* min_p, const float* uniform, int* out) {
    const int bytes = RESIDENT ? slice * 4 : 0;
    const auto kernel = sample_min_p_kernel<RESIDENT>;
    static unsigned long long seen = 0;
    int device;
    if (eg_first_on_device(seen, device)) {
        cudaError_t set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_SLICE * 4);
        if (set == cudaSuccess) set = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (set != cudaSuccess) return (int)set;
        eg_done_on_device(seen, device);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long long)rows * ctas));
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
    cfg.numAttrs = 2;
    (void)cudaLaunchKernelEx(&cfg, kernel, logits, ld, vocab, slice, temperature, top_k, top_p, min_p, uniform, out);
    return eg_launch_status();
}

}  // namespace

// logits [rows, vocab] with row stride ld; temperature, top_k, top_p, min_p, uniform, out: [rows].
EG_API int eg_sample_min_p(cudaStream_t stream, const float* logits, long long ld, int rows, int vocab, const float* temperature, const int* top_k, const float* top_p,
                           const float* min_p, const float* uniform, int* out) {
    if (rows <= 0) return 0;
    if (vocab < 1 || vocab > MOST_TOKENS || rows > 0x7fffffff / MOST_CTAS) return (int)cudaErrorInvalidValue;
    // as many CTAs a row as its slices need, and for few rows more
    int ctas = 1;
    while (ctas < MOST_CTAS && ((long long)vocab > (long long)ctas * SLICE || (rows * ctas < 64 && vocab > ctas * 8192))) ctas *= 2;
    const int slice = ((vocab + ctas - 1) / ctas + 3) & ~3;
    if (slice <= MOST_SLICE) return launch<true>(stream, ctas, slice, logits, ld, rows, vocab, temperature, top_k, top_p, min_p, uniform, out);
    return launch<false>(stream, ctas, slice, logits, ld, rows, vocab, temperature, top_k, top_p, min_p, uniform, out);
}
