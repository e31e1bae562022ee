// kv_attention.cu — attention of a few new tokens per sequence over the paged key/value cache (b200_kv_attention).
//
// One CTA per (sequence, row, head) walks the positions that its row sees in chunks of one position per thread: scores from
// a dot product per thread, a running maximum and sum (of exponentials to base e), and the output's dimensions one per
// thread. All in float32.
#include <cmath>

#include "kv.cuh"

using namespace b200;

namespace {

constexpr int kThreads = 128;

__device__ __forceinline__ float value(const uint8_t * data, const __half * scales, int64_t row, int D, int d) {
    if (scales) return __fmul_rn(__half2float(scales[row * (D / 32) + d / 32]), (float) reinterpret_cast<const int8_t *>(data)[row * D + d]);
    return __half2float(reinterpret_cast<const __half *>(data)[row * D + d]);
}

__global__ void __launch_bounds__(kThreads) kv_attention_kernel(KvView c, bool q8, int n_tok, int n_head, const float * __restrict__ q,
                                                                int64_t ldq, float scale, float * __restrict__ out) {
    __shared__ float qs[256], p[kThreads], red[kThreads / 32];
    __shared__ int64_t at[kThreads];
    const int h = blockIdx.x % n_head;
    const int64_t row = blockIdx.x / n_head, s = row / n_tok, r = row % n_tok;
    const int D = c.head_dim, hk = h / (n_head / c.n_kv_head);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t seen = kv_len(c, s, tid == 0) - n_tok + r + 1;
    for (int d = tid; d < D; d += kThreads) qs[d] = q[row * ldq + (int64_t) h * D + d];
    float o[2] = {0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
    for (int64_t j0 = 0; j0 < seen; j0 += kThreads) {
        __syncthreads();
        const int64_t j = j0 + tid;
        const int page = j < seen ? kv_page(c, s, j / c.page_size, true) : -1;
        const int64_t a = page < 0 ? -1 : ((int64_t) page * c.n_kv_head + hk) * c.page_size + j % c.page_size;
        float score = -INFINITY;
        if (a >= 0) {
            score = 0.0f;
            for (int d = 0; d < D; d++) score += qs[d] * value(c.k, q8 ? c.kd : nullptr, a, D, d);
            score *= scale;
        }
        const float w = warp_max(score);
        if (lane == 0) red[warp] = w;
        __syncthreads();
        float top = m;
        for (int i = 0; i < kThreads / 32; i++) top = fmaxf(top, red[i]);
        const float base = top > -INFINITY ? top : 0.0f, keep = expf(m - base);
        p[tid] = expf(score - base);
        at[tid] = a;
        m = top;
        __syncthreads();
        o[0] *= keep, o[1] *= keep, l *= keep;
        for (int i = 0; i < kThreads; i++) {
            if (at[i] < 0) continue;
            l += p[i];
            for (int e = 0; e < 2; e++)
                if (tid + e * kThreads < D) o[e] += p[i] * value(c.v, q8 ? c.vd : nullptr, at[i], D, tid + e * kThreads);
        }
    }
    for (int e = 0; e < 2; e++)
        if (tid + e * kThreads < D) out[(row * n_head + h) * D + tid + e * kThreads] = l != 0.0f ? o[e] / l : 0.0f;
}

}  // namespace

extern "C" {

size_t b200_kv_attention_workspace(b200_context * ctx, const b200_kv_cache * cache, int64_t max_pages, int64_t n_seq, int64_t n_tok,
                                   int64_t n_head) {
    (void) ctx, (void) cache, (void) max_pages, (void) n_seq, (void) n_tok, (void) n_head;
    return 0;
}

b200_status b200_kv_attention(b200_context * ctx, void * stream, const b200_kv_cache * cache, const int32_t * table, int64_t max_pages,
                              const int32_t * lens, int64_t n_seq, int64_t n_tok, int64_t n_head, const float * q, int64_t ldq, float scale,
                              float * out, void * workspace, size_t workspace_bytes) {
    const char * what = "kv_attention";
    KvView c;
    const b200_status s = kv_checked_view(ctx, what, cache, table, max_pages, lens, n_seq, n_tok, &c);
    if (s != B200_OK) return s;
    if (n_tok > 16) return kv_fail(ctx, B200_ERR_UNSUPPORTED, what, "more than 16 tokens per sequence");
    if (n_head <= 0 || n_head > 65535 || n_head % c.n_kv_head) return kv_fail(ctx, B200_ERR_INVALID, what, "n_head is not a multiple of n_kv_head");
    if (n_seq == 0 || n_tok == 0) return B200_OK;
    if (n_seq * n_tok > INT32_MAX / n_head) return kv_fail(ctx, B200_ERR_INVALID, what, "n_seq * n_tok * n_head passes 2^31");
    if (ldq < n_head * c.head_dim) return kv_fail(ctx, B200_ERR_INVALID, what, "the row stride is below n_head * head_dim");
    if (!q || !out || ((uintptr_t) q & 3) || ((uintptr_t) out & 3)) return kv_fail(ctx, B200_ERR_INVALID, what, "NULL or misaligned q or out");
    const size_t need = b200_kv_attention_workspace(ctx, cache, max_pages, n_seq, n_tok, n_head);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t) workspace & 255)))
        return kv_fail(ctx, B200_ERR_INVALID, what, "the workspace is missing, misaligned or too small");
    DeviceScope scope(ctx->device);
    if (scope.status != cudaSuccess) return kv_cuda(ctx, scope.status, what);
    cudaStream_t st = stream ? (cudaStream_t) stream : ctx->stream;
    kv_attention_kernel<<<(unsigned) (n_seq * n_tok * n_head), kThreads, 0, st>>>(c, cache->type == B200_TYPE_Q8_0, (int) n_tok, (int) n_head, q, ldq,
                                                                                scale, out);
    return kv_cuda(ctx, cudaGetLastError(), what);
}

}  // extern "C"
