// moe_router.cu — the expert router (b200_moe_router): scores, group choice, top-k and weights of each row of logits.
//
// One warp per row; lane l holds experts l, l + 32, ... and each round takes the best expert that is left. Scores that are
// compared across experts (with a bias or groups) are double, since a sum with a bias rounded to float32 would reorder
// experts that are nearly equal.
#include <cmath>

#include "kv.cuh"

using namespace b200;

namespace {

struct RouterParams {
    int E, top_k, score, n_group, topk_group, group_top, renorm;
    float scale;
};

// (a, i) before (b, j): larger first, ties to the lower index.
__device__ __forceinline__ bool before(double a, int i, double b, int j) { return a > b || (a == b && i < j); }

__device__ __forceinline__ void warp_best(double & v, int & i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const double ov = __shfl_xor_sync(0xffffffffu, v, o);
        const int oi = __shfl_xor_sync(0xffffffffu, i, o);
        if (before(ov, oi, v, i)) v = ov, i = oi;
    }
}

// EPL: experts per lane.
template <int EPL>
__global__ void __launch_bounds__(128) moe_router_kernel(RouterParams a, const float * __restrict__ logits, const float * __restrict__ bias,
                                                         int64_t T, int32_t * __restrict__ ids, float * __restrict__ w) {
    const int lane = threadIdx.x & 31;
    const int64_t t = blockIdx.x * (int64_t) (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (t >= T) return;
    const double ninf = -INFINITY;
    double p[EPL], c[EPL];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; i++) {
        const int e = i * 32 + lane;
        float x = e < a.E ? logits[t * a.E + e] : -INFINITY;
        if (x != x) x = -INFINITY;
        p[i] = x;
        top = fmaxf(top, x);
    }
    top = warp_max(top);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < EPL; i++) {
        const double x = p[i];
        const bool order = !bias && a.n_group == 1;  // the logits' order is the scores'
        if (a.score == B200_ROUTER_SIGMOID) p[i] = x == ninf ? 0.0 : 1.0 / (1.0 + exp(-x));
        else p[i] = x == ninf ? 0.0 : x == (double) top ? 1.0 : exp(x - (double) top);
        sum += p[i];
        c[i] = order ? x : p[i];
    }
    sum = warp_sum_d(sum);
#pragma unroll
    for (int i = 0; i < EPL; i++) {
        const int e = i * 32 + lane;
        if (a.score == B200_ROUTER_SOFTMAX) p[i] = sum > 0.0 ? p[i] / sum : 0.0;
        if (bias || a.n_group > 1) c[i] = e < a.E ? (bias ? p[i] + (double) bias[e] : p[i]) : ninf;
        if (c[i] != c[i]) c[i] = ninf;
    }
    unsigned taken = 0;  // bit i: this lane's expert i is out (past the last one, in a group that is not kept, or chosen)
#pragma unroll
    for (int i = 0; i < EPL; i++)
        if (i * 32 + lane >= a.E) taken |= 1u << i;
    if (a.n_group > 1) {
        const int size = a.E / a.n_group;
        double mine = 0.0;  // lane g: group g's score
        for (int g = 0; g < a.n_group; g++) {
            double score = 0.0;
            int skip = -1;
            for (int n = 0; n < (a.group_top < size ? a.group_top : size); n++) {
                double v = ninf;
                int at = INT32_MAX;
#pragma unroll
                for (int i = 0; i < EPL; i++) {
                    const int e = i * 32 + lane;
                    if (e < a.E && e / size == g && e != skip && before(c[i], e, v, at)) v = c[i], at = e;
                }
                warp_best(v, at);
                score += v;
                skip = at;
            }
            if (lane == g) mine = score != score ? ninf : score;
        }
        unsigned kept = 0;
        for (int n = 0; n < a.topk_group; n++) {
            double v = lane < a.n_group && !(kept >> lane & 1) ? mine : ninf;
            int at = lane < a.n_group && !(kept >> lane & 1) ? lane : 32 + lane;
            warp_best(v, at);
            kept |= 1u << at;
        }
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            const int e = i * 32 + lane;
            if (e < a.E && !(kept >> (e / size) & 1)) taken |= 1u << i;
        }
    }
    double mine = 0.0, total = 0.0;  // lane k: the score of the k-th chosen
    int id = 0;
    for (int k = 0; k < a.top_k; k++) {
        double v = ninf, ps = 0.0;
        int at = INT32_MAX;
#pragma unroll
        for (int i = 0; i < EPL; i++)
            if (!(taken >> i & 1) && before(c[i], i * 32 + lane, v, at)) v = c[i], at = i * 32 + lane;
        warp_best(v, at);
#pragma unroll
        for (int i = 0; i < EPL; i++)
            if (at == i * 32 + lane) ps = p[i], taken |= 1u << i;
        ps = __shfl_sync(0xffffffffu, ps, at & 31);
        total += ps;
        if (lane == k) mine = ps, id = at;
    }
    if (lane < a.top_k) {
        if (a.renorm) mine = total > 0.0 ? mine / total : 0.0;
        ids[t * a.top_k + lane] = id;
        w[t * a.top_k + lane] = __double2float_rn(mine * (double) a.scale);
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
    if (!logits || !ids || !w) return kv_fail(ctx, B200_ERR_INVALID, what, "NULL argument");
    if (T > (int64_t) INT32_MAX) return kv_fail(ctx, B200_ERR_INVALID, what, "more than 2^31 rows");
    DeviceScope scope(ctx->device);
    if (scope.status != cudaSuccess) return kv_cuda(ctx, scope.status, what);
    const RouterParams a{r->n_expert, r->top_k, r->score, r->n_group, r->topk_group, r->group_top, r->renorm, r->scale};
    cudaStream_t st = stream ? (cudaStream_t) stream : ctx->stream;
    const unsigned grid = (unsigned) ((T + 3) / 4);
    const int epl = (a.E + 31) / 32;
    if (epl <= 2) moe_router_kernel<2><<<grid, 128, 0, st>>>(a, logits, bias, T, ids, w);
    else if (epl <= 4) moe_router_kernel<4><<<grid, 128, 0, st>>>(a, logits, bias, T, ids, w);
    else if (epl <= 8) moe_router_kernel<8><<<grid, 128, 0, st>>>(a, logits, bias, T, ids, w);
    else if (epl <= 16) moe_router_kernel<16><<<grid, 128, 0, st>>>(a, logits, bias, T, ids, w);
    else moe_router_kernel<32><<<grid, 128, 0, st>>>(a, logits, bias, T, ids, w);
    return kv_cuda(ctx, cudaGetLastError(), what);
}
