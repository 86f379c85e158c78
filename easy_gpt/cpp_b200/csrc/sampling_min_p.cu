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
// Each of the three cuts keeps a run from the top of the row's descending order, so together they are one threshold: a logit, and how many of
// the tokens equal to it (the first ones) stay.  A token's decision hangs on sums over a whole vocabulary, and a uniform number may lie next
// to a token's border; so weights are taken in 64 bits and summed as whole numbers of 2^-42, whose sums are the same in every order.
// Tokens below half of that have no weight.
#include "common.cuh"

namespace {

constexpr int THREADS = 1024;
constexpr double ONE = 4398046511104.0;                              // 2^42: with 2^20 tokens sums stay below 2^62
constexpr int MOST_TOKENS = 1 << 20;

// larger numbers have larger keys; NaN has key 0
__device__ __forceinline__ unsigned key_of(float x) {
    if (!(x == x)) return 0u;
    if (x == 0.f) x = 0.f;                                           // -0 is 0
    const unsigned b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

template <typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, T* scratch, F join) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = join(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

typedef unsigned long long u64;

__global__ void __launch_bounds__(THREADS)
sample_min_p_kernel(const float* __restrict__ logits, long long ld, int vocab, const float* __restrict__ temperature, const int* __restrict__ top_k,
                    const float* __restrict__ top_p, const float* __restrict__ min_p, const float* __restrict__ uniform, int* __restrict__ out) {
    pdl_enter();
    __shared__ u64 scratch[32];
    __shared__ u64 before[THREADS];
    __shared__ int chosen;
    const int r = blockIdx.x, tid = threadIdx.x;
    const float* const row = logits + (size_t)r * ld;
    auto sum = [&](u64 v) { return block_reduce(v, scratch, [](u64 a, u64 b) { return a + b; }); };
    auto most = [&](u64 v) { return block_reduce(v, scratch, [](u64 a, u64 b) { return a > b ? a : b; }); };
    // the largest key and, of the tokens that have it, the first: one number that is the larger the better
    u64 best = 0;
    for (int i = tid; i < vocab; i += THREADS) {
        const u64 mine = (u64)key_of(row[i]) << 32 | (0xffffffffu - i);
        best = mine > best ? mine : best;
    }
    best = most(best);
    const unsigned top = (unsigned)(best >> 32);
    const int first_best = (int)(0xffffffffu - (unsigned)best);
    const float T = temperature[r], largest = value_of(top);
    if (!(T > 0.f) || top == 0u || largest == -INFINITY) {
        if (tid == 0) out[r] = top == 0u || largest == -INFINITY ? 0 : first_best;
        return;
    }
    auto weight = [&](float x) -> u64 {
        if (x == largest) return (u64)ONE;                           // +inf too
        if (!(x > -INFINITY) || largest == INFINITY) return 0;
        return (u64)__double2ll_rn(exp(((double)x - (double)largest) / (double)T) * ONE);
    };
    // ---- the threshold: tokens with a key above `low` are kept and the first `ties` of those that have it
    unsigned low = 1u;                                               // NaN is never kept
    u64 ties = vocab;
    const int k = top_k[r];
    if (k > 0 && k < vocab) {
        unsigned t = 0;
        for (unsigned bit = 1u << 31; bit; bit >>= 1) {
            u64 c = 0;
            for (int i = tid; i < vocab; i += THREADS) c += key_of(row[i]) >= (t | bit);
            if (sum(c) >= (u64)k) t |= bit;
        }
        if (t > 0) {                                                 // else fewer than k numbers
            u64 c = 0;
            for (int i = tid; i < vocab; i += THREADS) c += key_of(row[i]) > t;
            low = t;
            ties = k - sum(c);
        }
    }
    // the weights of the kept tokens with a key of t and more
    auto weights_from = [&](unsigned t) -> u64 {
        u64 c = 0, equal = 0;
        for (int i = tid; i < vocab; i += THREADS) {
            const unsigned key = key_of(row[i]);
            if (key >= t && key > low) c += weight(row[i]);
            equal += key >= t && key == low;
        }
        c = sum(c);
        equal = sum(equal);
        return c + (equal < ties ? equal : ties) * weight(value_of(low));
    };
    const float p = top_p[r];
    if (p > 0.f && p < 1.f) {
        const double target = (double)p * (double)weights_from(low);
        unsigned t = 0;                                              // the largest key from which on the weights reach the target
        for (unsigned bit = 1u << 31; bit; bit >>= 1)
            if ((double)weights_from(t | bit) >= target) t |= bit;
        if (t > low || (t == low && ties > 1)) {
            const u64 above = t == 0xffffffffu ? 0 : weights_from(t + 1), each = weight(value_of(t));
            // of the tokens at t as many as it takes
            const double need = each ? ceil((target - (double)above) / (double)each) : 1.0;
            const u64 take = need < 1.0 ? 1 : (u64)need;
            ties = t > low ? take : take < ties ? take : ties;
            low = t;
        }
    }
    const double least = (double)fminf(min_p[r], 1.f) * ONE;         // NaN: 1, which only the largest pass
    // ---- draw: every thread has a run of tokens, in the order of the indices
    const int run = (vocab + THREADS - 1) / THREADS, lo = min(vocab, tid * run), hi = min(vocab, lo + run);
    auto exclusive = [&](u64 v) -> u64 {                             // the sum over the threads in front; scratch[0] is the sum over all
        before[tid] = v;
        __syncthreads();
        if (tid == 0) {
            u64 s = 0;
            for (int i = 0; i < THREADS; ++i) {
                const u64 x = before[i];
                before[i] = s;
                s += x;
            }
            scratch[0] = s;
        }
        __syncthreads();
        return before[tid];
    };
    u64 equal = 0;
    for (int i = lo; i < hi; ++i) equal += key_of(row[i]) == low;
    equal = exclusive(equal);
    auto kept_weight = [&](float x, u64& rank) -> u64 {
        const unsigned key = key_of(x);
        if (key < low || (key == low && rank++ >= ties)) return 0;
        const u64 w = weight(x);
        return (double)w >= least ? w : 0;
    };
    u64 rank = equal, mass = 0;
    for (int i = lo; i < hi; ++i) mass += kept_weight(row[i], rank);
    const u64 start = exclusive(mass), all = scratch[0];
    if (tid == 0) chosen = first_best;
    __syncthreads();
    // the running sum has to pass u times the whole: at least 1, and at most the whole itself
    const double asked = (double)uniform[r] * (double)all;
    const u64 passed = asked > 0 ? (u64)asked + 1 : 1, goal = passed < all ? passed : all;
    if (start < goal && start + mass >= goal) {
        u64 s = start;
        rank = equal;
        for (int i = lo; i < hi; ++i) {
            s += kept_weight(row[i], rank);
            if (s >= goal) {
                chosen = i;
                break;
            }
        }
    }
    __syncthreads();
    if (tid == 0) out[r] = chosen;
}

}  // namespace

// logits [rows, vocab] with row stride ld; temperature, top_k, top_p, min_p, uniform, out: [rows].
EG_API int eg_sample_min_p(cudaStream_t stream, const float* logits, long long ld, int rows, int vocab, const float* temperature, const int* top_k, const float* top_p,
                           const float* min_p, const float* uniform, int* out) {
    if (rows <= 0) return 0;
    if (vocab < 1 || vocab > MOST_TOKENS) return (int)cudaErrorInvalidValue;
    eg_pdl_launch(sample_min_p_kernel, dim3(rows), dim3(THREADS), 0, stream, logits, ld, vocab, temperature, top_k, top_p, min_p, uniform, out);
    return eg_launch_status();
}
