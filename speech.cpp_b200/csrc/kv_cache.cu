// kv_cache.cu — the paged key/value cache: its memory, and the kernels that write and read its rows
// (b200_kv_cache_*, b200_kv_write, b200_kv_read, include/b200.h).
//
// The reference's cache is one dense F16 tensor per request, written with SET_ROWS (src/common/qwen3-decoder.cpp:320-321);
// here sequences share a pool of pages, and Q8_0 halves the bytes that attention streams.
//
// Both kernels are copies with a conversion, bound by HBM (4 B per value on the float side, 2 or 34/32 B in the cache), or by
// launch latency for the rows of a decode step. A row's length and page number are a chain of dependent loads before its
// first value, so many rows have to be under way: a warp or more per row, its threads walking the row's k then v values four
// at a time with four such pieces in flight. Measured on one B200, device time, 8 heads of 128: 24 x 4001 rows of Q8_0 read as
// float32 111 us, 6.2 TB/s (one CTA per row: 334 us); 1500 rows written as F16 4.1 us; 64 rows written as Q8_0 and read back
// 5.6 us, two launches' latency.
#include <cstdio>

#include "kv.cuh"

using namespace b200;

namespace {

// Bytes of the arrays k (and v) and of the scales of k (and v); false when the cache is not one that is supported.
bool kv_sizes(int type, int64_t heads, int64_t dim, int64_t page, int64_t pages, int64_t * values, int64_t * scales) {
    if (type != B200_TYPE_F16 && type != B200_TYPE_Q8_0) return false;
    if (dim != 64 && dim != 96 && dim != 128 && dim != 256) return false;
    if (heads <= 0 || heads > 65535 || page <= 0 || page % 16 || page > 4096 || pages <= 0 || pages > INT32_MAX) return false;
    const int64_t rows = heads * page;  // at most 2^28
    if (pages > ((int64_t) 1 << 52) / (rows * dim)) return false;
    *values = pages * rows * dim * (type == B200_TYPE_F16 ? 2 : 1);
    *scales = type == B200_TYPE_F16 ? 0 : pages * rows * (dim / 32) * 2;
    return true;
}

// Where the arrays k, v, k scales and v scales start, and the bytes of all.
struct KvLayout {
    int64_t off[4], bytes;
    KvLayout(int64_t values, int64_t scales)
        : off{0, align256(values), 2 * align256(values), 2 * align256(values) + align256(scales)}, bytes(2 * align256(values) + 2 * align256(scales)) {}
};

bool aligned(const void * p, size_t to) { return ((uintptr_t) p & (to - 1)) == 0; }

}  // namespace

namespace b200 {

b200_status kv_fail(b200_context * ctx, b200_status s, const char * what, const char * why) {
    const std::string text = std::string(what) + ": " + why;
    if (ctx) ctx->last_error = text;
    else set_thread_error(text.c_str());
    return s;
}

b200_status kv_cuda(b200_context * ctx, cudaError_t e, const char * what) {
    return e == cudaSuccess ? B200_OK : kv_fail(ctx, e == cudaErrorMemoryAllocation ? B200_ERR_ALLOC : B200_ERR_DEVICE, what, cudaGetErrorString(e));
}

b200_status kv_checked_view(b200_context * ctx, const char * what, const b200_kv_cache * c, const int32_t * table, int64_t max_pages,
                            const int32_t * lens, int64_t n_seq, int64_t n_tok, KvView * out) {
    if (!ctx) return kv_fail(ctx, B200_ERR_INVALID, what, "NULL context");
    int64_t values, scales;
    if (!c || !kv_sizes(c->type, c->n_kv_head, c->head_dim, c->page_size, c->n_pages, &values, &scales))
        return kv_fail(ctx, B200_ERR_INVALID, what, "not a cache");
    const KvLayout layout(values, scales);
    if (!c->data || !aligned(c->data, 16) || c->nbytes < (size_t) layout.bytes || std::memcmp(c->field_off, layout.off, sizeof layout.off) != 0)
        return kv_fail(ctx, B200_ERR_INVALID, what, "not a cache");
    if (c->device != ctx->device) return kv_fail(ctx, B200_ERR_INVALID, what, "the cache lies on another device than the context");
    if (n_seq < 0 || n_tok < 0 || max_pages < 0) return kv_fail(ctx, B200_ERR_INVALID, what, "a negative size");
    if (n_seq > 0 && n_tok > 0 && (!lens || (max_pages > 0 && !table) || ((uintptr_t) lens & 3) || ((uintptr_t) table & 3)))
        return kv_fail(ctx, B200_ERR_INVALID, what, "NULL or misaligned table or lens");
    if (max_pages > (1 << 30) / c->page_size) return kv_fail(ctx, B200_ERR_INVALID, what, "max_pages * page_size passes 2^30");
    // one CTA per row (or fewer) in a one-dimensional grid
    if (n_tok > 0 && n_seq > INT32_MAX / n_tok) return kv_fail(ctx, B200_ERR_INVALID, what, "n_seq * n_tok passes 2^31");
    const uint8_t * base = (const uint8_t *) c->data;
    out->k = base + c->field_off[0];
    out->v = base + c->field_off[1];
    out->kd = (const __half *) (base + c->field_off[2]);
    out->vd = (const __half *) (base + c->field_off[3]);
    out->n_kv_head = c->n_kv_head;
    out->head_dim = c->head_dim;
    out->page_size = c->page_size;
    out->n_pages = (int) c->n_pages;  // at most INT32_MAX (kv_sizes)
    out->table = table;
    out->lens = lens;
    out->max_pages = max_pages;
    out->err = ctx->dev_err;
    return B200_OK;
}

}  // namespace b200

namespace {

// Four float32 values at p (16-byte aligned when VEC).
template <bool VEC>
__device__ __forceinline__ float4 load4(const float * p) {
    if constexpr (VEC) return *reinterpret_cast<const float4 *>(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}

__device__ __forceinline__ uint2 pack4(float4 v) {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    return make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
}

// How rows are given to threads: `per_row` threads (32 to 512) for a row, 256 / per_row rows (or one) in a CTA.
struct RowSplit {
    int per_row;
    int64_t rows;
};

constexpr int kUnroll = 2;  // steps of a row that a thread has in flight, each four values of k and four of v

// The row of this thread (-1: none) and its place among the row's threads, a multiple of 32 to the warp.
__device__ __forceinline__ int64_t my_row(const RowSplit & p, int & i0) {
    const int64_t row = blockIdx.x * (int64_t) (blockDim.x / p.per_row) + threadIdx.x / p.per_row;
    i0 = threadIdx.x % p.per_row;
    return row < p.rows ? row : -1;
}

// A thread's way through a row of n_kv_head heads of Q = head_dim / 4 quads (four values), `per_row` quads further each step.
template <int Q>
struct Walk {
    int i, h, q, step, step_h, step_q;  // quad i of the row: quad q of head h
    __device__ __forceinline__ Walk(int i0, int per_row) : i(i0), h(i0 / Q), q(i0 % Q), step(per_row), step_h(per_row / Q), step_q(per_row % Q) {}
    __device__ __forceinline__ void next() {
        i += step;
        h += step_h;
        q += step_q;
        if (q >= Q) q -= Q, h++;
    }
};

// Where a row lies: its first head's bytes in k and v and in the scales, and what each head further adds.
template <bool Q8, int D>
struct RowPlace {
    int64_t at, scale_at;
    int head, scale_head;
    __device__ __forceinline__ RowPlace(const KvView & c, int page, int64_t pos) {
        const int64_t row = (int64_t) page * c.n_kv_head * c.page_size + pos % c.page_size;
        at = row * (Q8 ? D : 2 * D);
        head = c.page_size * (Q8 ? D : 2 * D);
        scale_at = row * (D / 32);
        scale_head = c.page_size * (D / 32);
    }
    __device__ __forceinline__ int64_t quad(int h, int q) const { return at + (int64_t) h * head + q * (Q8 ? 4 : 8); }
    __device__ __forceinline__ int64_t scale(int h, int q) const { return scale_at + (int64_t) h * scale_head + (q >> 3); }
};

// Row (s, r) of k and v to its slot. Q8_0: eight lanes hold a block's 32 values (quantize_q8_0_quad), so the warp's lanes
// all take part in every step, those past the row's end on its last values without storing.
template <bool Q8, bool VEC, int D>
__global__ void __launch_bounds__(512) kv_write_kernel(KvView c, RowSplit p, int64_t n_tok, const float * __restrict__ k, int64_t ldk,
                                                       const float * __restrict__ v, int64_t ldv) {
    int i0;
    const int64_t row = my_row(p, i0);
    if (row < 0) return;  // whole warps: per_row is a multiple of 32
    const int64_t s = row / n_tok, r = row % n_tok;
    const int64_t pos = kv_len(c, s, i0 == 0) - n_tok + r;
    if (pos < 0) return;
    const int page = kv_page(c, s, pos / c.page_size, i0 == 0);
    if (page < 0) return;
    const RowPlace<Q8, D> place(c, page, pos);
    const int quads = c.n_kv_head * (D / 4);
    const float * kr = k + row * ldk, * vr = v + row * ldv;
    uint8_t * to_k = const_cast<uint8_t *>(c.k), * to_v = const_cast<uint8_t *>(c.v);
    __half * to_kd = const_cast<__half *>(c.kd), * to_vd = const_cast<__half *>(c.vd);
    for (Walk<D / 4> w(i0, p.per_row); (w.i & ~31) < quads;) {
        float4 xk[kUnroll], xv[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            const int i = min(w.i + u * w.step, quads - 1);
            if (u > 0 && ((w.i + u * w.step) & ~31) >= quads) break;  // the whole warp
            xk[u] = load4<VEC>(kr + i * 4);
            xv[u] = load4<VEC>(vr + i * 4);
        }
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            if (u > 0 && (w.i & ~31) >= quads) break;
            const bool here = w.i < quads;
            if constexpr (Q8) {
                float dk, dv;
                const uint32_t qk = quantize_q8_0_quad(xk[u], &dk), qv = quantize_q8_0_quad(xv[u], &dv);
                if (here) {
                    const int64_t at = place.quad(w.h, w.q);
                    *reinterpret_cast<uint32_t *>(to_k + at) = qk;
                    *reinterpret_cast<uint32_t *>(to_v + at) = qv;
                    if ((w.q & 7) == 0) {
                        const int64_t sc = place.scale(w.h, w.q);
                        to_kd[sc] = __float2half_rn(dk);
                        to_vd[sc] = __float2half_rn(dv);
                    }
                }
            } else if (here) {
                const int64_t at = place.quad(w.h, w.q);
                *reinterpret_cast<uint2 *>(to_k + at) = pack4(xk[u]);
                *reinterpret_cast<uint2 *>(to_v + at) = pack4(xv[u]);
            }
            w.next();
        }
    }
}

// Four values of the cache as float32.
template <bool Q8>
__device__ __forceinline__ float4 widen(uint2 raw, __half scale) {
    if constexpr (Q8) {
        const char4 q = *reinterpret_cast<const char4 *>(&raw.x);
        const float f = __half2float(scale);
        return make_float4(__fmul_rn(f, (float) q.x), __fmul_rn(f, (float) q.y), __fmul_rn(f, (float) q.z), __fmul_rn(f, (float) q.w));
    } else {
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&raw.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&raw.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
}

// Four values to element o of an output.
template <bool HALF, bool VEC>
__device__ __forceinline__ void store4(void * out, int64_t o, float4 x) {
    if constexpr (HALF) {
        const uint2 w = pack4(x);
        if constexpr (VEC) {
            *reinterpret_cast<uint2 *>((__half *) out + o) = w;
        } else {
            uint16_t * to = (uint16_t *) out + o;
            to[0] = (uint16_t) w.x, to[1] = (uint16_t) (w.x >> 16), to[2] = (uint16_t) w.y, to[3] = (uint16_t) (w.y >> 16);
        }
    } else if constexpr (VEC) {
        *reinterpret_cast<float4 *>((float *) out + o) = x;
    } else {
        float * to = (float *) out + o;
        to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w;
    }
}

// Position start[s] + r to row (s, r) of k and v.
template <bool Q8, bool HALF, bool VEC, int D>
__global__ void __launch_bounds__(512) kv_read_kernel(KvView c, RowSplit p, const int32_t * __restrict__ start, int64_t n_tok, void * __restrict__ k,
                                                      void * __restrict__ v) {
    int i0;
    const int64_t row = my_row(p, i0);
    if (row < 0) return;
    const int64_t s = row / n_tok, r = row % n_tok;
    const int64_t pos = (start ? (int64_t) start[s] : 0) + r;
    if (pos < 0 || pos >= kv_len(c, s, i0 == 0)) return;
    const int page = kv_page(c, s, pos / c.page_size, i0 == 0);
    if (page < 0) return;
    const RowPlace<Q8, D> place(c, page, pos);
    const int quads = c.n_kv_head * (D / 4);
    const int64_t out = row * 4 * quads;
    for (Walk<D / 4> w(i0, p.per_row); w.i < quads;) {
        uint2 rk[kUnroll], rv[kUnroll];
        __half dk[kUnroll], dv[kUnroll];
        const int i = w.i;
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            if (u > 0 && w.i >= quads) break;
            const int64_t at = place.quad(w.h, w.q);
            if constexpr (Q8) {
                rk[u].x = *reinterpret_cast<const uint32_t *>(c.k + at);
                rv[u].x = *reinterpret_cast<const uint32_t *>(c.v + at);
                const int64_t sc = place.scale(w.h, w.q);
                dk[u] = c.kd[sc];
                dv[u] = c.vd[sc];
            } else {
                rk[u] = *reinterpret_cast<const uint2 *>(c.k + at);
                rv[u] = *reinterpret_cast<const uint2 *>(c.v + at);
            }
            w.next();
        }
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            if (u > 0 && i + u * w.step >= quads) break;
            store4<HALF, VEC>(k, out + (i + u * w.step) * 4, widen<Q8>(rk[u], dk[u]));
            store4<HALF, VEC>(v, out + (i + u * w.step) * 4, widen<Q8>(rv[u], dv[u]));
        }
    }
}

// Threads per row: a power of two from 32 to 512, at most one per four values of k, such that all rows together come to
// some 512 threads per SM. With more (2048 per SM) 1500 rows of 8 x 128 are written in 5.4 instead of 4.1 us and 1031 read in
// 4.2 instead of 3.5: the threads' values are then not enough to keep their loads under way.
RowSplit split_rows(const b200_context * ctx, const KvView & c, int64_t rows) {
    const int64_t fill = (int64_t) ctx->num_sms * 512, most = c.n_kv_head * c.head_dim / 4;
    int n = 32;
    while (n < 512 && n < most && rows * n < fill) n *= 2;
    return {n, rows};
}

unsigned split_threads(const RowSplit & p) { return p.per_row < 256 ? 256 : (unsigned) p.per_row; }

unsigned split_grid(const RowSplit & p) {
    const int64_t rows = split_threads(p) / p.per_row;
    return (unsigned) ((p.rows + rows - 1) / rows);
}

// Calls f with D as a constant.
template <class F>
void with_dim(int D, F f) {
    switch (D) {
    case 64: f(std::integral_constant<int, 64>{}); break;
    case 96: f(std::integral_constant<int, 96>{}); break;
    case 128: f(std::integral_constant<int, 128>{}); break;
    default: f(std::integral_constant<int, 256>{}); break;
    }
}

}  // namespace

extern "C" {

size_t b200_kv_cache_nbytes(int type, int64_t n_kv_head, int64_t head_dim, int64_t page_size, int64_t n_pages) {
    int64_t values, scales;
    if (!kv_sizes(type, n_kv_head, head_dim, page_size, n_pages, &values, &scales)) return 0;
    return (size_t) KvLayout(values, scales).bytes;
}

b200_status b200_kv_cache_view(b200_context * ctx, int type, int64_t n_kv_head, int64_t head_dim, int64_t page_size, int64_t n_pages,
                               void * data, size_t nbytes, b200_kv_cache * out) {
    if (!out) return kv_fail(ctx, B200_ERR_INVALID, "kv_cache_view", "NULL argument");
    std::memset(out, 0, sizeof *out);
    if (!ctx || !data) return kv_fail(ctx, B200_ERR_INVALID, "kv_cache_view", "NULL argument");
    int64_t values, scales;
    if (!kv_sizes(type, n_kv_head, head_dim, page_size, n_pages, &values, &scales))
        return kv_fail(ctx, B200_ERR_UNSUPPORTED, "kv_cache_view",
                       "needs F16 or Q8_0, head_dim 64, 96, 128 or 256, page_size a multiple of 16 up to 4096");
    if (!aligned(data, 16)) return kv_fail(ctx, B200_ERR_INVALID, "kv_cache_view", "data is not 16-byte aligned");
    const KvLayout layout(values, scales);
    const size_t need = (size_t) layout.bytes;
    if (nbytes < need) return kv_fail(ctx, B200_ERR_INVALID, "kv_cache_view", "too few bytes");
    out->type = type;
    out->device = ctx->device;
    out->n_kv_head = (int32_t) n_kv_head;
    out->head_dim = (int32_t) head_dim;
    out->page_size = (int32_t) page_size;
    out->n_pages = n_pages;
    out->data = data;
    out->nbytes = need;
    std::memcpy(out->field_off, layout.off, sizeof layout.off);
    return B200_OK;
}

b200_status b200_kv_cache_alloc(b200_context * ctx, int type, int64_t n_kv_head, int64_t head_dim, int64_t page_size, int64_t n_pages,
                                b200_kv_cache * out) {
    if (!out) return kv_fail(ctx, B200_ERR_INVALID, "kv_cache_alloc", "NULL argument");
    std::memset(out, 0, sizeof *out);
    if (!ctx) return kv_fail(ctx, B200_ERR_INVALID, "kv_cache_alloc", "NULL argument");
    const size_t need = b200_kv_cache_nbytes(type, n_kv_head, head_dim, page_size, n_pages);
    if (!need)
        return kv_fail(ctx, B200_ERR_UNSUPPORTED, "kv_cache_alloc",
                       "needs F16 or Q8_0, head_dim 64, 96, 128 or 256, page_size a multiple of 16 up to 4096");
    DeviceScope scope(ctx->device);
    if (scope.status != cudaSuccess) return kv_cuda(ctx, scope.status, "kv_cache_alloc");
    void * p = nullptr;
    cudaError_t e = cudaMalloc(&p, need);
    if (e != cudaSuccess) {
        cudaGetLastError();  // an allocation that failed is reported here, not by the next launch
        return kv_cuda(ctx, e, "kv_cache_alloc");
    }
    e = cudaMemsetAsync(p, 0, need, ctx->stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);  // zero for calls on every stream
    if (e != cudaSuccess) {
        cudaFree(p);
        return kv_cuda(ctx, e, "kv_cache_alloc");
    }
    const b200_status s = b200_kv_cache_view(ctx, type, n_kv_head, head_dim, page_size, n_pages, p, need, out);
    if (s != B200_OK) cudaFree(p);
    else out->owned = 1;
    return s;
}

b200_status b200_kv_cache_free(b200_context * ctx, b200_kv_cache * cache) {
    if (!ctx || !cache) return kv_fail(ctx, B200_ERR_INVALID, "kv_cache_free", "NULL argument");
    DeviceScope scope(ctx->device);
    cudaError_t e = scope.status;
    if (e == cudaSuccess && cache->data && cache->owned) e = cudaFree(cache->data);
    std::memset(cache, 0, sizeof *cache);
    return kv_cuda(ctx, e, "kv_cache_free");
}

b200_status b200_kv_write(b200_context * ctx, void * stream, const b200_kv_cache * cache, const int32_t * table, int64_t max_pages,
                          const int32_t * lens, int64_t n_seq, int64_t n_tok, const float * k, int64_t ldk, const float * v, int64_t ldv) {
    KvView c;
    const b200_status s = kv_checked_view(ctx, "kv_write", cache, table, max_pages, lens, n_seq, n_tok, &c);
    if (s != B200_OK) return s;
    if (n_seq == 0 || n_tok == 0) return B200_OK;
    const int64_t width = (int64_t) c.n_kv_head * c.head_dim;
    if (!k || !v || !aligned(k, 4) || !aligned(v, 4)) return kv_fail(ctx, B200_ERR_INVALID, "kv_write", "NULL or misaligned k or v");
    if (ldk < width || ldv < width) return kv_fail(ctx, B200_ERR_INVALID, "kv_write", "a row stride is below n_kv_head * head_dim");
    DeviceScope scope(ctx->device);
    if (scope.status != cudaSuccess) return kv_cuda(ctx, scope.status, "kv_write");
    const bool vec = aligned(k, 16) && aligned(v, 16) && ldk % 4 == 0 && ldv % 4 == 0;
    const RowSplit p = split_rows(ctx, c, n_seq * n_tok);
    cudaStream_t st = stream ? (cudaStream_t) stream : ctx->stream;
    with_dim(c.head_dim, [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        auto kern = cache->type == B200_TYPE_Q8_0 ? (vec ? kv_write_kernel<true, true, D> : kv_write_kernel<true, false, D>)
                                                  : (vec ? kv_write_kernel<false, true, D> : kv_write_kernel<false, false, D>);
        kern<<<split_grid(p), split_threads(p), 0, st>>>(c, p, n_tok, k, ldk, v, ldv);
    });
    return kv_cuda(ctx, cudaGetLastError(), "kv_write");
}

b200_status b200_kv_read(b200_context * ctx, void * stream, const b200_kv_cache * cache, const int32_t * table, int64_t max_pages,
                         const int32_t * lens, const int32_t * start, int64_t n_seq, int64_t n_tok, int out_type, void * k, void * v) {
    KvView c;
    const b200_status s = kv_checked_view(ctx, "kv_read", cache, table, max_pages, lens, n_seq, n_tok, &c);
    if (s != B200_OK) return s;
    if (out_type != B200_TYPE_F32 && out_type != B200_TYPE_F16) return kv_fail(ctx, B200_ERR_UNSUPPORTED, "kv_read", "rows are read as F32 or F16");
    if (n_seq == 0 || n_tok == 0) return B200_OK;
    const size_t elem = out_type == B200_TYPE_F16 ? 2 : 4;
    if (!k || !v || !aligned(k, elem) || !aligned(v, elem) || !aligned(start, 4))
        return kv_fail(ctx, B200_ERR_INVALID, "kv_read", "NULL or misaligned k or v, or a misaligned start");
    DeviceScope scope(ctx->device);
    if (scope.status != cudaSuccess) return kv_cuda(ctx, scope.status, "kv_read");
    const bool vec = aligned(k, 4 * elem) && aligned(v, 4 * elem);
    const RowSplit p = split_rows(ctx, c, n_seq * n_tok);
    cudaStream_t st = stream ? (cudaStream_t) stream : ctx->stream;
    with_dim(c.head_dim, [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        auto pick = [&](auto q8, auto half) {
            constexpr bool Q8 = decltype(q8)::value, HALF = decltype(half)::value;
            auto kern = vec ? kv_read_kernel<Q8, HALF, true, D> : kv_read_kernel<Q8, HALF, false, D>;
            kern<<<split_grid(p), split_threads(p), 0, st>>>(c, p, start, n_tok, k, v);
        };
        using std::false_type;
        using std::true_type;
        if (cache->type == B200_TYPE_Q8_0) elem == 2 ? pick(true_type{}, true_type{}) : pick(true_type{}, false_type{});
        else elem == 2 ? pick(false_type{}, true_type{}) : pick(false_type{}, false_type{});
    });
    return kv_cuda(ctx, cudaGetLastError(), "kv_read");
}

}  // extern "C"
