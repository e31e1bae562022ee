// moe_router.cu — the expert router (b200_moe_router): scores, group choice, top-k and weights of each row of logits.
//
// A warp takes one to 32 / top_k rows; lane l holds a row's experts l, l + 32, ... as 32-bit keys whose unsigned order is the
// values' order, sorted within the lane. A round of the top-k is one reduction instruction over the lanes' first keys and a
// shift in the lane that won. The keys' low bits hold the expert's place in the lane, so values that differ only there, or by
// less than their rounding error, are not told apart; which experts are chosen has to be right all the same:
//  - without bias and groups the keys are the logits, and rows with equal truncated neighbours are done again with whole keys;
//  - otherwise scores are computed in float32 first, with a bound on their error, and the row is accepted if every
//    comparison that decides (neighbours among the chosen and the next one, the last group kept and the first one left) is
//    wider than that. Where neighbours are closer (some rows in a thousand of random ones), or groups, the few candidates are
//    ordered by their scores in double; where they are many, two lanes' keys are equal or anything is not finite, the row is
//    done again in double.
// The weights of the chosen are double either way, one lane for each, of all the warp's rows at once. Reading the logits
// takes 4 B per expert (2.7 us of HBM for 16384 rows of 256); the instructions decide the time. Measured on one B200, device
// time: 16384 rows of 256, eight chosen, by logits 11 us, by sigmoid and bias 16 us, by softmax and bias 19, with four of eight
// groups kept 22 to 23 us (in double throughout: 167 us); one row of 128 2.3 us, a launch. What takes longer:
//  - softmax without renorm: an exponential in double for every expert (21 us by logits, 33 with a bias);
//  - many equal logits (16-bit ones, by logits 20 us; with groups and no bias 50 us);
//  - an infinite logit or bias where there is a bias or groups (a masked logit, an expert switched off): every such row is done
//    in double (52 to 56 us, with groups 96);
//  - 32 of more than 32 experts, as the round that shows the next one to be apart has no lane: every row is done again (65 us by
//    logits, 31 of 256 taking 24; 121 us with a bias).
#include <cmath>

#include "kv.cuh"

using namespace b200;

namespace {

constexpr int kWarps = 4;
constexpr unsigned kAll = 0xffffffffu;

struct RouterParams {
    int E, top_k, score, n_group, topk_group, group_top, renorm;
    float scale;
    // groups in the float32 pass: `lanes` lanes (a power of two, n_group * lanes <= 32) for each, the scores of a group
    // `pitch` floats apart in shared memory so that a step's lanes read different banks
    int lanes, pitch, size, left;  // size: a group's experts; left: the experts of the groups that are kept
    int lane_shift, seat_shift;    // logarithms of lanes and seats
    // a warp takes `rows` rows; each has `seats` lanes (a power of two, at least top_k) for its weights
    int rows, seats;
    unsigned inv;  // expert e's group is e * inv >> 21 (e < 1024)
};

__device__ __forceinline__ int group_of(const RouterParams & a, int e) { return (int) ((unsigned) e * a.inv >> 21); }

// Unsigned order of the keys = order of the values (NaN: not allowed). 0 is below every value's key, and value_of(0) is NaN.
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned u = __float_as_uint(x + 0.0f);  // -0 as 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// ---- the row in double ------------------------------------------------------------------------------------------------

// (a, i) before (b, j): larger first, ties to the lower index.
__device__ __forceinline__ bool before(double a, int i, double b, int j) { return a > b || (a == b && i < j); }

// The same order for doubles: integer comparisons and reductions are quicker than double ones.
__device__ __forceinline__ unsigned long long key_of(double x) {
    const long long u = __double_as_longlong(x + 0.0);
    return u < 0 ? ~(unsigned long long) u : (unsigned long long) u | 1ull << 63;
}

__device__ __forceinline__ double value_of(unsigned long long k) {
    return __longlong_as_double((long long) (k >> 63 ? k & ~(1ull << 63) : ~k));
}

__device__ __forceinline__ unsigned long long warp_largest(unsigned long long k) {
    const unsigned high = __reduce_max_sync(kAll, (unsigned) (k >> 32));
    const unsigned low = __reduce_max_sync(kAll, (unsigned) (k >> 32) == high ? (unsigned) k : 0);
    return (unsigned long long) high << 32 | low;
}

__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x; }

// The numerator of a softmax term (or a sigmoid) of logit x in double; top: the row's largest logit.
__device__ __forceinline__ double term(const RouterParams & a, float x, float top) {
    if (x == -INFINITY) return 0.0;
    if (a.score == B200_ROUTER_SIGMOID) return 1.0 / (1.0 + exp(-(double) x));
    return x == top ? 1.0 : exp((double) x - (double) top);
}

// The sum of a row's softmax terms. (A function of its own, as the ones below: inlined, its registers would halve the number
// of warps that are under way.)
__device__ __noinline__ double softmax_sum(const RouterParams & a, const float * __restrict__ logits, float top) {
    double sum = 0.0;
    for (int e = threadIdx.x & 31; e < a.E; e += 32) sum += term(a, clean(logits[e]), top);
    return warp_sum_d(sum);
}

// The experts of one row: lane k gets the k-th chosen. For rows that float32 does not decide. kept: the groups that stay, if
// these at least are known (else 0).
template <int EPL>
__device__ __noinline__ int choose_exactly(const RouterParams & a, const float * __restrict__ logits, const float * __restrict__ bias, float top,
                                           unsigned kept) {
    const int lane = threadIdx.x & 31;
    unsigned long long key[EPL];  // 0: past the last expert, in a group that is not kept, or chosen
    {
        double c[EPL], sum = 0.0;
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            const int e = i * 32 + lane;
            c[i] = e < a.E ? term(a, clean(logits[e]), top) : 0.0;
            sum += c[i];
        }
        sum = warp_sum_d(sum);
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            const int e = i * 32 + lane;
            if (a.score == B200_ROUTER_SOFTMAX) c[i] = sum > 0.0 ? c[i] / sum : 0.0;
            if (bias && e < a.E) c[i] += (double) bias[e];
            key[i] = e < a.E ? key_of(c[i] == c[i] ? c[i] : -(double) INFINITY) : 0;
        }
    }
    // the lowest expert that has `best`
    auto holder = [&](unsigned long long best) {
        unsigned at = kAll;
#pragma unroll
        for (int i = EPL - 1; i >= 0; i--)
            if (key[i] == best) at = i * 32 + lane;
        return (int) __reduce_min_sync(kAll, at);
    };
    if (a.n_group > 1 && !kept) {
        unsigned long long mine = 0;  // lane g: group g's score
        for (int g = 0; g < a.n_group; g++) {
            unsigned long long best = 0;
#pragma unroll
            for (int i = 0; i < EPL; i++)
                if (group_of(a, i * 32 + lane) == g && key[i] > best) best = key[i];
            best = warp_largest(best);
            double score = value_of(best);
            if (a.group_top == 2 && a.size > 1) {
                unsigned at = kAll;  // the lowest expert of the group that has it is left out
#pragma unroll
                for (int i = EPL - 1; i >= 0; i--)
                    if (group_of(a, i * 32 + lane) == g && key[i] == best) at = i * 32 + lane;
                at = __reduce_min_sync(kAll, at);
                unsigned long long second = 0;
#pragma unroll
                for (int i = 0; i < EPL; i++)
                    if (group_of(a, i * 32 + lane) == g && i * 32u + lane != at && key[i] > second) second = key[i];
                score += value_of(warp_largest(second));
            }
            if (lane == g) mine = key_of(score == score ? score : -(double) INFINITY);
        }
        for (int n = 0; n < a.topk_group; n++) {
            const unsigned long long best = warp_largest(mine);
            const int g = __ffs(__ballot_sync(kAll, mine == best)) - 1;
            kept |= 1u << g;
            if (lane == g) mine = 0;
        }
    }
    if (a.n_group > 1) {
#pragma unroll
        for (int i = 0; i < EPL; i++)
            if (!(kept >> group_of(a, i * 32 + lane) & 1)) key[i] = 0;
    }
    int id = 0;
    for (int k = 0; k < a.top_k; k++) {
        unsigned long long best = 0;
#pragma unroll
        for (int i = 0; i < EPL; i++) best = key[i] > best ? key[i] : best;
        const int at = holder(warp_largest(best));
#pragma unroll
        for (int i = 0; i < EPL; i++)
            if (at == i * 32 + lane) key[i] = 0;
        if (lane == k) id = at;
    }
    return id;
}

// ---- rows by keys -----------------------------------------------------------------------------------------------------

// The top_k largest of the warp's keys (0: out), ties to the lowest expert, exactly: lane k gets the k-th's expert. For rows
// whose logits come too close for packed keys.
template <int EPL>
__device__ __noinline__ int choose_by_logit(const RouterParams & a, const float * __restrict__ logits) {
    const int lane = threadIdx.x & 31;
    unsigned key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; i++) key[i] = i * 32 + lane < a.E ? key_of(clean(logits[i * 32 + lane])) : 0;
    int id = 0;
    for (int k = 0; k < a.top_k; k++) {
        unsigned best = key[0];
#pragma unroll
        for (int i = 1; i < EPL; i++) best = max(best, key[i]);
        const unsigned top = __reduce_max_sync(kAll, best);
        unsigned at = 0xffffffffu;
#pragma unroll
        for (int i = EPL - 1; i >= 0; i--)
            if (key[i] == top) at = i * 32 + lane;
        at = __reduce_min_sync(kAll, at);
#pragma unroll
        for (int i = 0; i < EPL; i++)
            if (at == i * 32u + lane) key[i] = 0;
        if (lane == k) id = (int) at;
    }
    return id;
}

// Sorts a lane's keys, largest first (odd-even merge sort).
template <int N>
__device__ __forceinline__ void sort_keys(unsigned (&key)[N]) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; i++)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const unsigned x = key[i + j], y = key[i + j + k];
                        key[i + j] = max(x, y);
                        key[i + j + k] = min(x, y);
                    }
}

// The larger pair of (a1 >= a2) and (b1 >= b2).
__device__ __forceinline__ void merge2(float & a1, float & a2, float b1, float b2) {
    a2 = fmaxf(fminf(a1, b1), fmaxf(a2, b2));
    a1 = fmaxf(a1, b1);
}

// The order of a row's candidates (lane j: expert e, j < n) by their scores in double; lane k gets the k-th. top, sum: the
// softmax's (sum in double).
__device__ __noinline__ int order_exactly(const RouterParams & a, const float * __restrict__ logits, const float * __restrict__ bias, float top, double sum,
                                          int e, int n) {
    const int lane = threadIdx.x & 31;
    double c = 0.0;
    if (lane < n) {
        c = term(a, logits[e], top);
        if (a.score == B200_ROUTER_SOFTMAX) c /= sum;
        if (bias) c += (double) bias[e];
    }
    int rank = 0;
    for (int j = 0; j < n; j++) rank += before(__shfl_sync(kAll, c, j), __shfl_sync(kAll, e, j), c, e);
    int id = 0;
    for (int j = 0; j < n; j++) {
        const int to = __shfl_sync(kAll, rank, j), of = __shfl_sync(kAll, e, j);
        if (lane == to) id = of;
    }
    return id;
}

// The groups that stay (a bit each) by scores in double, from the experts whose float32 scores may be among a group's first
// group_top: those not below lane g's `least`. 0 where they are more than 32. Of 16384 random rows of 256 about one
// comes here; choose_exactly takes some 7 us for its groups, and the call would wait for that row.
__device__ __noinline__ unsigned groups_exactly(const RouterParams & a, const float * __restrict__ logits, const float * __restrict__ bias, float top,
                                                const float * scores, float least, int * list) {
    const int lane = threadIdx.x & 31;
    int n = 0;
    for (int e0 = 0; e0 < a.E; e0 += 32) {
        const int e = e0 + lane, g = e < a.E ? group_of(a, e) : 0;
        const float from = __shfl_sync(kAll, least, g);
        const bool in = e < a.E && scores[e + g * (a.pitch - a.size)] >= from;
        const unsigned who = __ballot_sync(kAll, in);
        const int at = n + __popc(who & ((1u << lane) - 1));
        if (in && at < 32) list[at] = e;
        n += __popc(who);
    }
    if (n > 32) return 0;
    __syncwarp();
    const double sum = a.score == B200_ROUTER_SOFTMAX ? softmax_sum(a, logits, top) : 1.0;
    double c = 0.0;
    int group = -1;
    if (lane < n) {
        const int e = list[lane];
        group = group_of(a, e);
        c = term(a, logits[e], top);
        if (a.score == B200_ROUTER_SOFTMAX) c /= sum;
        if (bias) c += (double) bias[e];
    }
    __syncwarp();
    double b1 = -INFINITY, b2 = -INFINITY;  // lane g: group g's largest
    for (int j = 0; j < n; j++) {
        const double o = __shfl_sync(kAll, c, j);
        if (__shfl_sync(kAll, group, j) == lane) {
            if (o > b1) b2 = b1, b1 = o;
            else if (o > b2) b2 = o;
        }
    }
    const double score = a.group_top == 2 && a.size > 1 ? b1 + b2 : b1;
    int ahead = 0;
    for (int g = 0; g < a.n_group; g++) ahead += before(__shfl_sync(kAll, score, g), g, score, lane);
    return __ballot_sync(kAll, lane < a.n_group && ahead < a.topk_group);
}

// EPL: experts per lane (a power of two). BY_LOGIT: no bias and no groups. FULL: there are 32 EPL experts.
template <int EPL, bool BY_LOGIT, bool FULL>
__global__ void __launch_bounds__(32 * kWarps) moe_router_kernel(const __grid_constant__ RouterParams a, const float * __restrict__ logits,
                                                                 const float * __restrict__ bias, int64_t T, int32_t * __restrict__ ids,
                                                                 float * __restrict__ w) {
    extern __shared__ float shared[];  // groups: each warp's scores, [n_group][pitch], and a list of 32 experts
    constexpr unsigned kIndex = EPL - 1;  // a key's low bits give way to the expert's place in its lane, the first ones largest
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t t0 = (blockIdx.x * (int64_t) kWarps + warp) * a.rows;
    const int mine = FULL ? EPL : (a.E - lane + 31) / 32;  // this lane's experts
    const bool softmax = a.score == B200_ROUTER_SOFTMAX;
    int id = 0;                     // lane r * seats + k: the k-th expert of row t0 + r, and what its weight needs
    float my_top = -INFINITY;
    double my_total = 0.0;
    for (int r = 0; r < a.rows && t0 + r < T; r++) {
        const float * row = logits + (t0 + r) * a.E;
        float x[EPL], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            x[i] = i < mine ? clean(row[i * 32 + lane]) : -INFINITY;
            top = fmaxf(top, x[i]);
        }
        top = value_of(__reduce_max_sync(kAll, key_of(top)));

        unsigned key[EPL];
        float off = 0.0f;  // bound on the error of a score
        bool sure = true;
        unsigned stay = 0;  // the groups that stay, once they are sure
        if constexpr (BY_LOGIT) {
#pragma unroll
            for (int i = 0; i < EPL; i++) key[i] = i < mine ? key_of(x[i]) : 0;
        } else {
            // float32 scores; `off` bounds the error of each. __expf(-d) is within 2 + 1.173 d units of its last place, so within
            // 2^-22 absolutely. A sigmoid of x has p (1 - p) (2 + 1.173 |x|) < 0.63 times 2^-23 of that, half of one from the
            // rounded sum and two units (2^-23) from the quotient: below 2^-21. A softmax's sum adds up to 32 terms per lane and
            // five times over the warp (37 roundings, below 2^-18.7) of terms that are off by 2^-20.1 of the sum at most (1024 terms,
            // all but one some 5.5 below the largest logit): below 2^-17 of the largest term. The sum with the bias rounds once more.
            float c[EPL], far = 0.0f, flaw = 0.0f;  // flaw: NaN where a logit or a score is NaN or infinite
            if (softmax) {
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < EPL; i++) {
                    c[i] = __expf(x[i] - top);
                    if (i < mine) sum += c[i];
                }
                const float inv = __fdividef(1.0f, warp_sum(sum));
                off = 0x1p-17f * inv;
#pragma unroll
                for (int i = 0; i < EPL; i++) c[i] *= inv;
            } else {
                off = 0x1p-21f;
#pragma unroll
                for (int i = 0; i < EPL; i++) c[i] = __fdividef(1.0f, 1.0f + __expf(-x[i]));
            }
            if (bias) {
#pragma unroll
                for (int i = 0; i < EPL; i++)
                    if (i < mine) c[i] += bias[i * 32 + lane];
            }
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                if (i < mine) {
                    far = fmaxf(far, fabsf(c[i]));
                    flaw = fmaf(0.0f, x[i], fmaf(0.0f, c[i], flaw));
                }
                key[i] = i < mine ? key_of(c[i]) : 0;
            }
            sure = __all_sync(kAll, flaw == 0.0f);
            far = value_of(__reduce_max_sync(kAll, key_of(far)));
            off += 0x1.1p-24f * far;
            if (sure && a.n_group > 1) {
                const int size = a.size;
                float * scores = shared + warp * (a.n_group * a.pitch + 32);
                int of[EPL];
#pragma unroll
                for (int i = 0; i < EPL; i++) {
                    of[i] = group_of(a, i * 32 + lane);
                    if (i < mine) scores[i * 32 + lane + of[i] * (a.pitch - size)] = c[i];
                }
                __syncwarp();
                const int g = lane >> a.lane_shift;
                float b1 = -INFINITY, b2 = -INFINITY;
                if (g < a.n_group)
                    for (int n = lane & (a.lanes - 1); n < size; n += a.lanes) merge2(b1, b2, scores[g * a.pitch + n], -INFINITY);
                for (int o = a.lanes >> 1; o > 0; o >>= 1) {
                    const float o1 = __shfl_xor_sync(kAll, b1, o), o2 = __shfl_xor_sync(kAll, b2, o);
                    merge2(b1, b2, o1, o2);
                }
                __syncwarp();
                const float score = a.group_top == 2 && size > 1 ? b1 + b2 : b1;
                // lane n: group n's score, and how many are before it
                const float s = __shfl_sync(kAll, score, lane < a.n_group ? lane << a.lane_shift : 0);
                int ahead = 0;
                for (int n = 0; n < a.n_group; n++) {
                    const float other = __shfl_sync(kAll, s, n);
                    ahead += other > s || (other == s && n < lane);
                }
                const bool in = lane < a.n_group && ahead < a.topk_group;
                unsigned kept = __ballot_sync(kAll, in);
                if (a.topk_group < a.n_group) {
                    const float low = value_of(__reduce_min_sync(kAll, in ? key_of(s) : kAll));
                    const float high = value_of(__reduce_max_sync(kAll, lane < a.n_group && !in ? key_of(s) : 0));
                    sure = low - high > 4.0f * off + 0x1p-22f * fmaxf(fabsf(low), fabsf(high));
                    if (!sure) {
                        // a group's first experts have at least its last one's true score, so float32 scores two errors below
                        const float last = a.group_top == 2 && size > 1 ? b2 : b1;
                        const float least = __shfl_sync(kAll, last, lane < a.n_group ? lane << a.lane_shift : 0) - 4.0f * off;
                        const unsigned exact = groups_exactly(a, row, bias, top, scores, least, (int *) (scores + a.n_group * a.pitch));
                        if (exact) kept = exact, sure = true;
                    }
                }
#pragma unroll
                for (int i = 0; i < EPL; i++) key[i] = kept >> of[i] & 1 ? key[i] : 0;
                if (sure) stay = kept;
            }
        }
        int chosen = 0;  // lane k: the k-th expert
        if (sure) {
#pragma unroll
            for (int i = 0; i < EPL; i++) key[i] = FULL && BY_LOGIT || key[i] ? (key[i] & ~kIndex) | (kIndex - i) : 0;
            sort_keys(key);
            // Round n leaves the n-th key, and the lanes that had it, in lane n: top_k rounds and one more (if there is another
            // expert and a lane for it) to see that it lies apart.
            const int left = a.left;
            unsigned found = 0, who = 0;
            int n = 0;
            auto round = [&] {
                const unsigned best = __reduce_max_sync(kAll, key[0]);
                const bool won = key[0] == best;
                const unsigned winners = __ballot_sync(kAll, won);
                if (lane == n) found = best, who = winners;
#pragma unroll
                for (int i = 0; i + 1 < EPL; i++) key[i] = won ? key[i + 1] : key[i];
                key[EPL - 1] = won ? 0 : key[EPL - 1];
                n++;
                return best;
            };
            const int rounds = min(a.top_k + 1, min(left, 32));
            while (n < rounds) round();
            const unsigned next = __shfl_down_sync(kAll, found, 1);
            const bool single = lane >= n || __popc(who) == 1;  // of equal keys one is lost
            bool apart = lane + 1 >= n;
            if constexpr (BY_LOGIT) apart = apart || (found | kIndex) > (next | kIndex);
            else apart = apart || value_of(found & ~kIndex) - value_of(next | kIndex) > 2.0f * off;
            sure = __all_sync(kAll, single) && (n > a.top_k || left == a.top_k);
            chosen = (int) (kIndex - (found & kIndex)) * 32 + __ffs(who) - 1;
            if (sure && !__all_sync(kAll, apart)) {
                sure = false;
                if constexpr (!BY_LOGIT) {
                    // All that may be among the chosen: keys down to the last one's, less both their errors.
                    const float least = value_of(__shfl_sync(kAll, found, a.top_k - 1) & ~kIndex) - 2.0f * off;
                    bool enough = false;
                    while (!enough && n < min(left, 32)) enough = value_of(round() | kIndex) < least;
                    if (__all_sync(kAll, lane >= n || __popc(who) == 1) && (enough || n == left)) {
                        const double sum = softmax ? softmax_sum(a, row, top) : 1.0;
                        chosen = order_exactly(a, row, bias, top, sum, (int) (kIndex - (found & kIndex)) * 32 + __ffs(who) - 1, n);
                        sure = true;
                    }
                }
            }
        }
        if (!sure) {
            if constexpr (BY_LOGIT) chosen = choose_by_logit<EPL>(a, row);
            else chosen = choose_exactly<EPL>(a, row, bias, top, stay);
        }
        chosen = __shfl_sync(kAll, chosen, lane - r * a.seats);
        const double total = !a.renorm && softmax ? softmax_sum(a, row, top) : 0.0;
        if (lane >= r * a.seats) {  // the lanes behind this row's are the next rows'
            id = chosen;
            my_top = top;
            my_total = total;
        }
    }

    // ---- weights, one expert of one row per lane ----
    const int k = lane & (a.seats - 1);
    const int64_t t = t0 + (lane >> a.seat_shift);
    const bool chosen = k < a.top_k && lane < a.rows * a.seats && t < T;
    double weight = chosen ? term(a, clean(logits[t * a.E + id]), my_top) : 0.0;
    if (a.renorm) {
        my_total = weight;
        for (int o = a.seats >> 1; o > 0; o >>= 1) my_total += __shfl_xor_sync(kAll, my_total, o);
    }
    if (a.renorm || softmax) weight = my_total > 0.0 ? weight / my_total : 0.0;
    if (chosen) {
        ids[t * a.top_k + k] = id;
        w[t * a.top_k + k] = __double2float_rn(weight * (double) a.scale);
    }
}

}  // namespace

extern "C" b200_status b200_moe_router(b200_context * ctx, void * stream, const b200_router * r, const float * logits, const float * bias,
                                       int64_t T, int32_t * ids, float * w) {
    const char * what = "moe_router";
    if (!ctx || !r) return kv_fail(ctx, B200_ERR_INVALID, what, "NULL argument");
    if (r->n_expert < 1 || r->top_k < 1 || r->n_group < 1 || T < 0) return kv_fail(ctx, B200_ERR_INVALID, what, "a bad size");
    if (r->n_expert > 1024 || r->top_k > 32 || r->n_group > 32)
        return kv_fail(ctx, B200_ERR_UNSUPPORTED, what, "more than 1024 experts, 32 chosen or 32 groups");
    if (r->score != B200_ROUTER_SOFTMAX && r->score != B200_ROUTER_SIGMOID) return kv_fail(ctx, B200_ERR_UNSUPPORTED, what, "an unknown score");
    if (r->n_expert % r->n_group || r->topk_group < 1 || r->topk_group > r->n_group || (r->group_top != 1 && r->group_top != 2))
        return kv_fail(ctx, B200_ERR_INVALID, what, "bad groups");
    if (r->top_k > r->n_expert / r->n_group * r->topk_group) return kv_fail(ctx, B200_ERR_INVALID, what, "top_k passes the experts that stay");
    if (T == 0) return B200_OK;
    if (!logits || !ids || !w || (((uintptr_t) logits | (uintptr_t) bias | (uintptr_t) ids | (uintptr_t) w) & 3))
        return kv_fail(ctx, B200_ERR_INVALID, what, "a NULL or misaligned argument");
    if (T > (int64_t) INT32_MAX) return kv_fail(ctx, B200_ERR_INVALID, what, "more than 2^31 rows");
    DeviceScope scope(ctx->device);
    if (scope.status != cudaSuccess) return kv_cuda(ctx, scope.status, what);
    RouterParams a = {};
    a.E = r->n_expert;
    a.top_k = r->top_k;
    a.score = r->score;
    a.n_group = r->n_group;
    a.topk_group = r->topk_group;
    a.group_top = r->group_top;
    a.renorm = r->renorm;
    a.scale = r->scale;
    a.size = a.E / a.n_group;
    a.left = a.size * a.topk_group;
    a.lanes = a.seats = 1;
    // Several rows per warp share the double arithmetic of the weights (a row has top_k of them, a warp 32 lanes), as many as
    // that needs or as leave one wave of sixteen warps to each SM. (4736 rows of 256 in groups: 8.3 us
    // with two rows per warp, 10.3 with four; by logits 5.5 and 5.9.)
    while (a.seats < a.top_k) a.seats *= 2, a.seat_shift++;
    const int64_t wave = (int64_t) ctx->num_sms * 16, each = (T + wave - 1) / wave;
    a.rows = each < 32 / a.seats ? (int) each : 32 / a.seats;
    size_t smem = 0;
    if (a.n_group > 1) {
        a.inv = ((1u << 21) + a.size - 1) / a.size;  // e * (inv * size - 2^21) < 2^10 2^10, so the quotient is exact
        while (2 * a.lanes * a.n_group <= 32) a.lanes *= 2, a.lane_shift++;
        a.pitch = a.size + (a.lanes - a.size % 32 + 32) % 32;  // pitch mod 32 = lanes: lane l of a step reads bank l + const
        smem = (size_t) kWarps * (a.n_group * a.pitch + 32) * sizeof(float);  // at most 4 * (1024 + 32 * 31 + 32) * 4 B = 32 KB
    }
    cudaStream_t st = stream ? (cudaStream_t) stream : ctx->stream;
    const unsigned grid = (unsigned) ((T + kWarps * a.rows - 1) / (kWarps * a.rows));
    const bool by_logit = !bias && a.n_group == 1;
    auto go = [&](auto epl) {
        constexpr int EPL = decltype(epl)::value;
        const bool full = a.E == 32 * EPL;
        auto kern = by_logit ? (full ? moe_router_kernel<EPL, true, true> : moe_router_kernel<EPL, true, false>)
                             : (full ? moe_router_kernel<EPL, false, true> : moe_router_kernel<EPL, false, false>);
        kern<<<grid, 32 * kWarps, smem, st>>>(a, logits, bias, T, ids, w);
    };
    const int epl = (a.E + 31) / 32;
    if (epl <= 2) go(std::integral_constant<int, 2>{});
    else if (epl <= 4) go(std::integral_constant<int, 4>{});
    else if (epl <= 8) go(std::integral_constant<int, 8>{});
    else if (epl <= 16) go(std::integral_constant<int, 16>{});
    else go(std::integral_constant<int, 32>{});
    return kv_cuda(ctx, cudaGetLastError(), what);
}
