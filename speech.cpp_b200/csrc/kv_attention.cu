// kv_attention.cu — attention of a few new tokens per sequence over the paged key/value cache (b200_kv_attention).
//
// Mathematics. The rows of one key/value head (its group of query heads, times the call's tokens) share every key and value,
// so they are taken eight at a time: S = Q K^T and O = P V over 16 positions at a time, with a running maximum and sum per
// row (o and l are rescaled by 2^(m_old - m_new) when a larger score appears; exponentials to base 2, their scale folded into
// the scores'). Bytes decide: a position costs 4 D bytes (F16) or 2.125 D (Q8_0) of HBM and 4 D multiply-adds per row, so
// the arithmetic has to cost next to nothing beside the stream of the cache.
//
// Float32 results from F16 matrix instructions. mma.m16n8k16 multiplies F16 exactly and adds in float32, but takes 16 rows
// where there are at most eight: rows 0-7 of the tile hold the high half of the operand and rows 8-15 the low half (x = hi +
// lo in F16, 22 bits; q scaled by a power of two per row first), and the two results of a row lie in the same lane's
// registers, where one addition joins them. So q and the weights enter with 22 bits at the price of the padding. Q8_0's
// values are whole numbers and exact in F16; their scales stay outside: a key block's multiplies its partial score, a value
// block's multiplies the weight before it is split (times a power of two per 16 positions that keeps it in F16's range).
// Each instruction's sum starts at zero and is added to the float32 result with an ordinary rounded addition (the
// instruction's own accumulation truncates, which over thousands of positions would add up).
//
// Operands without shared memory. The k index of S = Q K^T may run through a row's dimensions in any order that both operands
// share, and the n index of O = P V through any order that the output is written back in. They are chosen such that a lane's
// fragment is 16 (F16 keys and values), 8 or 4 (Q8_0) contiguous bytes of a row: keys and values go from HBM to the matrix
// instruction's registers with wide loads that use every byte of each sector, and the scores' registers are the weights'
// fragment as they stand.
//
// Split. Sequences differ in length and there may be one of them, so the work is cut by positions: all (sequence, key/value
// head, row tile) items laid end to end in chunks of 64 positions, and each CTA takes an equal run of chunks. A CTA's four
// warps take turns at 16-position tiles of a run and join at its end. Items that lie within one CTA's run are finished by it;
// of the others each CTA leaves a partial (m, l, o) in the workspace, and a second kernel, launched with programmatic
// dependent launch, joins them.
#include <cooperative_groups.h>

#include <cmath>

#include "kv.cuh"

using namespace b200;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kJoinWarps = 8;
constexpr int kRows = 8;      // rows of a tile
constexpr int kChunk = 64;    // positions of a chunk: one 16-position tile per warp
constexpr int kItemChunks = 8;  // chunks per CTA up to which the work is cut by items
constexpr float kShift = 14;  // weights are held times 2^14, so that their low halves reach 2^-38 of the largest

struct Geometry {
    int n_tok, n_head, group, tiles;  // tiles: row tiles of a key/value head
    int64_t items;                    // n_kv_head * tiles, per sequence
    int64_t n_seq;
    int64_t ctas;                     // CTAs among which the chunks are divided, or
    int cluster;                      // CTAs that share an item (0: the work is cut by positions)
};

// CTAs per SM, by what registers allow (__launch_bounds__ holds the compiler to it).
template <bool Q8, int D>
constexpr int ctas_per_sm() { return D == 256 ? 2 : 3; }

int ctas_per_sm_of(bool q8, int D) { (void) q8; return D == 256 ? 2 : 3; }

constexpr int64_t partial_floats(int D) { return (int64_t) kRows * (D + 2); }  // o [kRows][D], m [kRows], l [kRows]

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// N 32-bit words from p (aligned to their size; N = 3, 8: to one and four words). The cache is read once: not kept in L1.
template <int N>
__device__ __forceinline__ void load(uint32_t (&w)[N], const uint8_t * p) {
    if constexpr (N == 4 || N == 8) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3])
                         : "l"(p + 4 * i));
    } else if constexpr (N == 2) {
        asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(w[i]) : "l"(p + 4 * i));
    }
}

template <int N>
__device__ __forceinline__ void zero(uint32_t (&w)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = 0;
}

__device__ __forceinline__ __half2 h2(uint32_t w) { return *reinterpret_cast<const __half2 *>(&w); }
__device__ __forceinline__ uint32_t u32(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }

// Half numbers i and j of two rows' scales (kept together in w) as a pair.
template <int I, int J, int N>
__device__ __forceinline__ uint32_t pair_of(const uint32_t (&w)[N]) {
    constexpr uint32_t sel = (I & 1 ? 0x32u : 0x10u) | (J & 1 ? 0x7600u : 0x5400u);
    return __byte_perm(w[I / 2], w[J / 2], sel);
}

// (x, y) as two F16 pairs, hi + lo.
__device__ __forceinline__ void split(float x, float y, uint32_t & hi, uint32_t & lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = u32(h);
    lo = u32(l);
}

// Two of four bytes q + 128 (sel 0x4140: the first two, 0x4342: the last two) as F16 values q: 0x6400 | b is 1024 + b.
__device__ __forceinline__ uint32_t halves(uint32_t biased, uint32_t sel) {
    return u32(__hsub2(h2(__byte_perm(biased, 0x64646464u, sel)), __float2half2_rn(1152.0f)));
}

__device__ __forceinline__ float half_of(const uint32_t * w, int i) {
    return __half2float(__ushort_as_half((uint16_t) (w[i >> 1] >> (16 * (i & 1)))));
}

// How the n index of O = P V runs through the dimensions: groups of 8 kRun dimensions, lane quad g holding kRun contiguous
// ones of each.
template <bool Q8, int D>
struct Shape {
    static constexpr int kBlocks = D / 32;
    static constexpr int kRun = !Q8 && D % 64 == 0 ? 8 : 4;
    static constexpr int kGroups = D / (8 * kRun);
    static constexpr int kKeyWords = Q8 ? 2 : 4;           // a lane's words of a row's 32 dimensions
    static constexpr int kValueWords = Q8 ? 1 : kRun / 2;  // a lane's words of a row's group
};

__device__ __forceinline__ int64_t chunks_of(const KvView & c, int64_t s, bool tell) { return (kv_len(c, s, tell) + kChunk - 1) / kChunk; }

__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Chunks of sequences [0, n), summed by the block (red: one value per warp).
__device__ __forceinline__ int64_t block_chunks(const KvView & c, int64_t n, int64_t * red) {
    int64_t sum = 0;
    for (int64_t s = threadIdx.x; s < n; s += kThreads) sum += chunks_of(c, s, blockIdx.x == 0);
    sum = warp_sum64(sum);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; w++) sum += red[w];
    return sum;
}

// The sequence that holds chunk number `at` (of one item; chunk numbers count each sequence's chunks `items` times), and
// where it starts. at < the total.
__device__ __forceinline__ void find_sequence(const KvView & c, const Geometry & g, int64_t at, int64_t * red, int64_t & seq, int64_t & start) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t base = 0;
    for (int64_t s0 = 0; s0 < g.n_seq; s0 += kThreads) {
        const int64_t s = s0 + threadIdx.x;
        const int64_t mine = s < g.n_seq ? chunks_of(c, s, false) * g.items : 0;
        int64_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        __syncthreads();
        if (lane == 31) red[warp] = incl;
        __syncthreads();
        int64_t first = base, all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            if (w < warp) first += red[w];
            all += red[w];
        }
        const int64_t begin = first + incl - mine;
        if (mine > 0 && at >= begin && at < begin + mine) {
            red[kWarps] = s;
            red[kWarps + 1] = begin;
        }
        base += all;
        if (at < base) break;  // the same for all threads
    }
    __syncthreads();
    seq = red[kWarps];
    start = red[kWarps + 1];
}

// Rows of a tile: row i is query head h * group + (tile * 8 + i) % group of token (tile * 8 + i) / group.
struct Row {
    int token, head;
    bool there;
};

__device__ __forceinline__ Row row_of(const Geometry & g, int h, int tile, int i) {
    const int n = tile * kRows + i;
    return {n / g.group, h * g.group + n % g.group, n < g.n_tok * g.group};
}

// What a CTA holds while it works on one item.
template <int D>
struct Shared {
    __align__(16) uint32_t sq[D / 16][32][4];  // the query tile as fragments
    float so[kWarps][kRows][D + 4];            // the warps' results
    float sm[kWarps][kRows], sl[kWarps][kRows];
};

// Chunks [c0, c1) of one item: the warps' m, l and o are left in shared memory (synchronised).
template <bool Q8, int D>
__device__ __forceinline__ void attend(const KvView & c, const Geometry & g, const float * __restrict__ q, int64_t ldq, float scale, Shared<D> & sh,
                                       int64_t seq, int64_t len, int h, int tile, int64_t c0, int64_t c1) {
    using S = Shape<Q8, D>;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int gq = lane >> 2, t = lane & 3;  // the fragment's group and thread in it
    const Row row = row_of(g, h, tile, gq);

    // ---- the query tile: each warp makes the fragments of its share of the k steps ----
    // k step 2 j + b of lane (gq, t) holds dimensions 32 j + 8 t + 4 b .. + 3 of row gq: hi in registers 0 and 2, lo in
    // 1 and 3. The row is scaled by 2^k to a largest magnitude in [2^14, 2^15).
    float factor;  // what a raw score is multiplied by: scale log2(e) 2^-k
    {
        const float * src = q + (seq * g.n_tok + row.token) * ldq + (int64_t) row.head * D + 8 * t;
        float x[D / 4], top = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 4; i++) {
            x[i] = row.there ? src[(i / 8) * 32 + i % 8] : 0.0f;
            top = fmaxf(top, fabsf(x[i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = (int) (__float_as_uint(top) >> 23);
        const int k = e == 255 || top == 0.0f ? 0 : 141 - e < 126 ? 141 - e : 126;
        const float up = __uint_as_float((uint32_t) (k + 127) << 23);
        factor = scale * 1.4426950408889634f * __uint_as_float((uint32_t) (127 - k) << 23);
#pragma unroll
        for (int j = 0; j < D / 16; j++) {
            if (j % kWarps != warp) continue;
            uint32_t hi[2], lo[2];
            split(x[4 * j] * up, x[4 * j + 1] * up, hi[0], lo[0]);
            split(x[4 * j + 2] * up, x[4 * j + 3] * up, hi[1], lo[1]);
            *reinterpret_cast<uint4 *>(sh.sq[j][lane]) = make_uint4(hi[0], lo[0], hi[1], lo[1]);
        }
    }
    __syncthreads();

    // ---- this warp's tiles of positions [c0 * 64, c1 * 64) ----
    constexpr int kRowBytes = Q8 ? D : 2 * D;
    const int p_end = (int) (c1 * kChunk < len ? c1 * kChunk : len);
    const int all_see = (int) len - g.n_tok + 1;  // positions below are seen by every row
    const int seen = row.there ? all_see + row.token : 0;
    const int64_t page_bytes = (int64_t) c.n_kv_head * c.page_size * kRowBytes;
    const int64_t head_bytes = (int64_t) h * c.page_size * kRowBytes;
    const uint8_t * kl = c.k + head_bytes + gq * kRowBytes + t * (Q8 ? 8 : 16);                      // this lane's bytes of page 0
    const uint8_t * vl = c.v + head_bytes + 2 * t * kRowBytes + gq * S::kRun * (Q8 ? 1 : 2);
    const uint8_t * kdl = reinterpret_cast<const uint8_t *>(c.kd) + head_bytes / 16 + t * (D / 8);  // a row's scales: D / 16 bytes
    const uint8_t * vdl = reinterpret_cast<const uint8_t *>(c.vd) + head_bytes / 16 + t * (D / 8);
    const int page_step = kChunk / c.page_size, slot_step = kChunk % c.page_size;
    float o[S::kGroups][S::kRun][2] = {}, m = -INFINITY, l = 0.0f;
    int p0 = (int) c0 * kChunk + warp * 16;
    int in_table = p0 / c.page_size, slot = p0 % c.page_size;
    for (; p0 < p_end; p0 += kChunk) {
        const int page = kv_page(c, seq, in_table, lane == 0);
        const int64_t at = page * page_bytes + slot * kRowBytes;
        in_table += page_step;
        slot += slot_step;
        if (slot >= c.page_size) slot -= c.page_size, in_table++;
        if (page < 0) continue;
        const int here = p_end - p0;  // positions of the tile: 16 or more, or its end
        const bool edge = p0 + 16 > all_see || here < 16;
        uint32_t kw[2][S::kBlocks][S::kKeyWords], vw[4][S::kGroups][S::kValueWords];
        uint32_t kd[2][Q8 ? S::kBlocks : 1], vd[2][Q8 ? S::kBlocks : 1];
        // keys of positions gq, gq + 8; values of positions 2 t, 2 t + 1, 2 t + 8, 2 t + 9, whose scores this lane holds
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int b = 0; b < S::kBlocks; b++) {
                if (edge && gq + 8 * i >= here) zero(kw[i][b]);
                else load(kw[i][b], kl + at + i * 8 * kRowBytes + b * (Q8 ? 32 : 64));
            }
        if constexpr (Q8) {  // the scales of two neighbouring rows are kBlocks words; the tile's rows all lie in its page
#pragma unroll
            for (int i = 0; i < 2; i++) {
                load(kd[i], kdl + at / 16 + i * (D / 2));
                load(vd[i], vdl + at / 16 + i * (D / 2));
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int n = 0; n < S::kGroups; n++) {
                if (edge && 2 * t + (i & 1) + 8 * (i >> 1) >= here) zero(vw[i][n]);
                else load(vw[i][n], vl + at + ((i & 1) + 8 * (i >> 1)) * kRowBytes + n * 8 * S::kRun * (Q8 ? 1 : 2));
            }

        // ---- scores: s[2 i + j] is position 2 t + j + 8 i of row gq ----
        float s[4];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            s[2 * i] = s[2 * i + 1] = 0.0f;
#pragma unroll
            for (int b = 0; b < S::kBlocks; b++) {
                const uint4 a0 = *reinterpret_cast<const uint4 *>(sh.sq[2 * b][lane]), a1 = *reinterpret_cast<const uint4 *>(sh.sq[2 * b + 1][lane]);
                const uint32_t f0[4] = {a0.x, a0.y, a0.z, a0.w}, f1[4] = {a1.x, a1.y, a1.z, a1.w};
                if constexpr (Q8) {
                    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    const uint32_t w0 = kw[i][b][0] ^ 0x80808080u, w1 = kw[i][b][1] ^ 0x80808080u;
                    mma(part, f0, halves(w0, 0x4140), halves(w0, 0x4342));
                    mma(part, f1, halves(w1, 0x4140), halves(w1, 0x4342));
                    s[2 * i] = fmaf(half_of(kd[i], b), part[0] + part[2], s[2 * i]);
                    s[2 * i + 1] = fmaf(half_of(kd[i], S::kBlocks + b), part[1] + part[3], s[2 * i + 1]);
                } else {
                    mma(sum, f0, kw[i][b][0], kw[i][b][1]);
                    mma(sum, f1, kw[i][b][2], kw[i][b][3]);
                }
            }
            if constexpr (!Q8) {
                s[2 * i] = sum[0] + sum[2];
                s[2 * i + 1] = sum[1] + sum[3];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] *= factor;
        if (edge) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int j = 2 * t + (i & 1) + 8 * (i >> 1);
                if (j >= here || p0 + j >= seen) s[i] = -INFINITY;
            }
        }

        // ---- weights: m is the running maximum less kShift (-infinity before any score) ----
        float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float m_new = fmaxf(m, top - kShift);
        const float base = m_new == -INFINITY ? 0.0f : m_new;
        const float keep = ex2(m - base);
        m = m_new;
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; i++) p[i] = ex2(s[i] - base);
        l = fmaf(l, keep, (p[0] + p[1]) + (p[2] + p[3]));

        // ---- o = o keep + P V ----
        uint32_t pf[4];  // the weights' fragment: hi, lo of positions 2 t, 2 t + 1, then of 2 t + 8, 2 t + 9
        split(p[0], p[1], pf[0], pf[1]);
        split(p[2], p[3], pf[2], pf[3]);
        if constexpr (Q8) {
            // one block of 32 dimensions: weights times scales (fragment a), times 2^k and back where `down` is not 1
            auto block = [&](int b, const uint32_t(&a)[4], auto scaled, float down) {
                // two rows' four bytes each, interleaved: (row, row + 1) pairs of dimensions 0, 1 and 2, 3
                const uint32_t x0 = __byte_perm(vw[0][b][0], vw[1][b][0], 0x5140) ^ 0x80808080u;
                const uint32_t x1 = __byte_perm(vw[0][b][0], vw[1][b][0], 0x7362) ^ 0x80808080u;
                const uint32_t y0 = __byte_perm(vw[2][b][0], vw[3][b][0], 0x5140) ^ 0x80808080u;
                const uint32_t y1 = __byte_perm(vw[2][b][0], vw[3][b][0], 0x7362) ^ 0x80808080u;
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    const uint32_t sel = n & 1 ? 0x4342 : 0x4140;
                    mma(part, a, halves(n < 2 ? x0 : x1, sel), halves(n < 2 ? y0 : y1, sel));
                    part[0] += part[2];
                    part[1] += part[3];
                    if constexpr (decltype(scaled)::value) part[0] *= down, part[1] *= down;
                    o[b][n][0] = fmaf(o[b][n][0], keep, part[0]);
                    o[b][n][1] = fmaf(o[b][n][1], keep, part[1]);
                }
            };
            // Scales between 2^-14 and 2 (nearly always all of them) multiply the weights' halves in F16 pairs: the
            // product's rounding error is exact in F16 and goes to the low half. The weights being up to 2^14 and the low
            // halves reaching 2^-24, nothing overflows and what is lost is below 2^-24 of the largest weight's product.
            uint32_t low = vd[0][0], high = vd[0][0];
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int b = 0; b < S::kBlocks; b++) low = __vminu2(low, vd[i][b]), high = __vmaxu2(high, vd[i][b]);
            const bool plain = (low & 0xffffu) >= 0x0400u && low >= 0x04000000u && (high & 0xffffu) < 0x4000u && high < 0x40000000u;
            if (__all_sync(0xffffffffu, plain)) {
                auto go = [&](auto index) {
                    constexpr int b = decltype(index)::value;
                    if constexpr (b < S::kBlocks) {
                        const __half2 d0 = h2(pair_of<b, S::kBlocks + b>(vd[0])), d1 = h2(pair_of<b, S::kBlocks + b>(vd[1]));
                        const __half2 w0 = __hmul2_rn(h2(pf[0]), d0), w1 = __hmul2_rn(h2(pf[2]), d1);
                        const uint32_t a[4] = {u32(w0), u32(__hfma2(h2(pf[1]), d0, __hfma2(h2(pf[0]), d0, __hneg2(w0)))), u32(w1),
                                               u32(__hfma2(h2(pf[3]), d1, __hfma2(h2(pf[2]), d1, __hneg2(w1))))};
                        block(b, a, std::false_type{}, 1.0f);
                    }
                };
                go(std::integral_constant<int, 0>{}), go(std::integral_constant<int, 1>{}), go(std::integral_constant<int, 2>{});
                go(std::integral_constant<int, 3>{}), go(std::integral_constant<int, 4>{}), go(std::integral_constant<int, 5>{});
                go(std::integral_constant<int, 6>{}), go(std::integral_constant<int, 7>{});
            } else {
                // any scales: the product in float32, times a power of two that brings the tile's largest scale below 1
#pragma unroll
                for (int b = 0; b < S::kBlocks; b++) {
                    float d[4];
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        d[i] = 2 * t + (i & 1) + 8 * (i >> 1) < here ? half_of(vd[i >> 1], (i & 1) * S::kBlocks + b) : 0.0f;
                    float big = fmaxf(fmaxf(fabsf(d[0]), fabsf(d[1])), fmaxf(fabsf(d[2]), fabsf(d[3])));
                    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                    int e = (int) (__float_as_uint(big) >> 23);
                    if (e == 0 || e == 255) e = 126;
                    const float up = __uint_as_float((uint32_t) (253 - e) << 23), down = __uint_as_float((uint32_t) (e + 1) << 23);
                    float w[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) w[i] = edge && p[i] == 0.0f ? 0.0f : p[i] * (d[i] * up);
                    uint32_t a[4];
                    split(w[0], w[1], a[0], a[1]);
                    split(w[2], w[3], a[2], a[3]);
                    block(b, a, std::true_type{}, down);
                }
            }
        } else {
            auto product = [&](bool mine) {
#pragma unroll
                for (int n = 0; n < S::kGroups; n++)
#pragma unroll
                    for (int r = 0; r < S::kRun; r++) {
                        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        const uint32_t sel = r & 1 ? 0x7632 : 0x5410;
                        mma(part, pf, __byte_perm(vw[0][n][r / 2], vw[1][n][r / 2], sel), __byte_perm(vw[2][n][r / 2], vw[3][n][r / 2], sel));
                        if (mine) {
                            o[n][r][0] = fmaf(o[n][r][0], keep, part[0] + part[2]);
                            o[n][r][1] = fmaf(o[n][r][1], keep, part[1] + part[3]);
                        }
                    }
            };
            if (edge && g.n_tok > 1) {
                // Where rows see different positions, a value that is NaN or infinite must not meet the weight 0 of a row
                // that does not see it: one product per token, from the last, with the values behind its position zeroed.
                const int first = tile * kRows / g.group;
                for (int token = min((tile * kRows + kRows - 1) / g.group, g.n_tok - 1); token >= first; token--) {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (p0 + 2 * t + (i & 1) + 8 * (i >> 1) >= all_see + token) {
#pragma unroll
                            for (int n = 0; n < S::kGroups; n++) zero(vw[i][n]);
                        }
                    product(row.token == token);
                }
            } else {
                product(true);
            }
        }
    }

    // ---- join the warps ----
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0) {
        sh.sm[warp][gq] = m;
        sh.sl[warp][gq] = l;
    }
#pragma unroll
    for (int n = 0; n < S::kGroups; n++)
#pragma unroll
        for (int r = 0; r < S::kRun; r++)
#pragma unroll
            for (int j = 0; j < 2; j++) sh.so[warp][gq][n * 8 * S::kRun + (2 * t + j) * S::kRun + r] = o[n][r][j];
    __syncthreads();
}

// The CTA's sum of the warps' results for one row: the factors of the warps, and m and l.
template <int D>
struct Joined {
    float f[kWarps], m, l;
    __device__ __forceinline__ Joined(const Shared<D> & sh, int i) {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) m = fmaxf(m, sh.sm[w][i]);
        const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            f[w] = ex2(sh.sm[w][i] - base);
            l = fmaf(sh.sl[w][i], f[w], l);
        }
    }
    __device__ __forceinline__ float value(const Shared<D> & sh, int i, int d) const {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; w++) v = fmaf(sh.so[w][i][d], f[w], v);
        return v;
    }
};

// The work cut by positions: CTA b takes chunks [b share, (b + 1) share) of all items' chunks.
template <bool Q8, int D>
__global__ void __launch_bounds__(kThreads, ctas_per_sm<Q8, D>())
    kv_attention_kernel(KvView c, Geometry g, const float * __restrict__ q, int64_t ldq, float scale, float * __restrict__ out, float * __restrict__ ws) {
    __shared__ Shared<D> sh;
    __shared__ int64_t red[kWarps + 2];
    const int tid = threadIdx.x;
    pdl_launch_dependents();

    const int64_t total = block_chunks(c, g.n_seq, red) * g.items;
    const int64_t share = (total + g.ctas - 1) / g.ctas;
    int64_t at = blockIdx.x * share;
    const int64_t end = at + share < total ? at + share : total;
    if (at >= end) return;
    int64_t seq, start;
    find_sequence(c, g, at, red, seq, start);
    int64_t len = kv_len(c, seq, false), chunks = (len + kChunk - 1) / kChunk;

    while (at < end) {
        while (at >= start + chunks * g.items) {  // the next sequence that has chunks
            start += chunks * g.items;
            seq++;
            len = kv_len(c, seq, false);
            chunks = (len + kChunk - 1) / kChunk;
        }
        const int64_t item = (at - start) / chunks, c0 = (at - start) % chunks;
        const int64_t c1 = c0 + (end - at) < chunks ? c0 + (end - at) : chunks;
        at += c1 - c0;
        const int h = (int) (item / g.tiles), tile = (int) (item % g.tiles);
        attend<Q8, D>(c, g, q, ldq, scale, sh, seq, len, h, tile, c0, c1);

        const int i = tid / 16;  // a row per 16 threads
        const Joined<D> all(sh, i);
        const Row row = row_of(g, h, tile, i);
        if (c0 == 0 && c1 == chunks) {  // the whole item
            const float inv = all.l != 0.0f ? 1.0f / all.l : 0.0f;
            if (row.there)
                for (int d = tid & 15; d < D; d += 16) out[((seq * g.n_tok + row.token) * g.n_head + row.head) * D + d] = all.value(sh, i, d) * inv;
        } else {  // the CTA's first partial (of an item begun before it) or its last
            float * to = ws + (2 * blockIdx.x + (c0 == 0 ? 1 : 0)) * partial_floats(D);
            for (int d = tid & 15; d < D; d += 16) to[i * D + d] = all.value(sh, i, d);
            if ((tid & 15) == 0) {
                to[kRows * D + i] = all.m;
                to[kRows * D + kRows + i] = all.l;
            }
        }
        __syncthreads();  // the shared memory is written again by the next run
    }
}

// The work cut by items: a cluster of `cluster` CTAs per item, each an equal run of its chunks, joined over distributed
// shared memory: the CTA of rank r writes rows r, r + cluster, ... One launch, and no length but the item's own is read.
template <bool Q8, int D>
__global__ void __launch_bounds__(kThreads, ctas_per_sm<Q8, D>())
    kv_attention_item_kernel(KvView c, Geometry g, int cluster, const float * __restrict__ q, int64_t ldq, float scale, float * __restrict__ out) {
    __shared__ Shared<D> sh;
    __shared__ float jm[kRows], jl[kRows];
    const int tid = threadIdx.x, rank = blockIdx.x % cluster;
    const int64_t unit = blockIdx.x / cluster, seq = unit / g.items;
    const int item = (int) (unit % g.items), h = item / g.tiles, tile = item % g.tiles;
    const int64_t len = kv_len(c, seq, tid == 0), chunks = (len + kChunk - 1) / kChunk, per = (chunks + cluster - 1) / cluster;
    const int64_t c0 = rank * per < chunks ? rank * per : chunks, c1 = c0 + per < chunks ? c0 + per : chunks;
    attend<Q8, D>(c, g, q, ldq, scale, sh, seq, len, h, tile, c0, c1);
    {
        const int i = tid / 16;
        const Joined<D> all(sh, i);
        for (int d = tid & 15; d < D; d += 16) sh.so[0][i][d] = all.value(sh, i, d);  // read and written by this thread alone
        if ((tid & 15) == 0) jm[i] = all.m, jl[i] = all.l;
    }
    const cooperative_groups::cluster_group group = cooperative_groups::this_cluster();
    group.sync();
    for (int e = tid; e < kRows / cluster * D; e += kThreads) {
        const int i = e / D * cluster + rank, d = e % D;
        const Row row = row_of(g, h, tile, i);
        if (!row.there) continue;
        float m = -INFINITY, l = 0.0f, v = 0.0f;
        for (int r = 0; r < cluster; r++) m = fmaxf(m, *group.map_shared_rank(&jm[i], r));
        const float base = m == -INFINITY ? 0.0f : m;
        for (int r = 0; r < cluster; r++) {
            const float f = ex2(*group.map_shared_rank(&jm[i], r) - base);
            l = fmaf(*group.map_shared_rank(&jl[i], r), f, l);
            v = fmaf(*group.map_shared_rank(&sh.so[0][i][d], r), f, v);
        }
        out[((seq * g.n_tok + row.token) * g.n_head + row.head) * D + d] = l != 0.0f ? v * (1.0f / l) : 0.0f;
    }
    group.sync();  // the others read this CTA's shared memory until here
}

// Joins the partials of items that several CTAs worked on, and writes the zeros of empty sequences. One CTA per row of an
// item: a warp takes every kJoinWarps-th partial, a lane D / 32 dimensions, and the warps join in shared memory.
template <int D>
__global__ void __launch_bounds__(32 * kJoinWarps) kv_attention_join_kernel(KvView c, Geometry g, float * __restrict__ out, const float * __restrict__ ws) {
    __shared__ int64_t red[2 * kJoinWarps];
    __shared__ float so[kJoinWarps][D], sm[kJoinWarps], sl[kJoinWarps];
    const int i = blockIdx.x % kRows, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t seq = blockIdx.x / kRows / g.items, item = blockIdx.x / kRows % g.items;
    const Row mine = row_of(g, (int) (item / g.tiles), (int) (item % g.tiles), i);
    if (!mine.there) return;
    int64_t sums[2] = {0, 0};  // the chunks of an item in all sequences, and in those before this one
    for (int64_t s = tid; s < g.n_seq; s += 32 * kJoinWarps) {
        const int64_t n = chunks_of(c, s, false);
        sums[0] += n;
        if (s < seq) sums[1] += n;
    }
    sums[0] = warp_sum64(sums[0]);
    sums[1] = warp_sum64(sums[1]);
    if (lane == 0) {
        red[2 * warp] = sums[0];
        red[2 * warp + 1] = sums[1];
    }
    const int64_t chunks = chunks_of(c, seq, false);
    __syncthreads();
    int64_t total = 0, a = 0;
#pragma unroll
    for (int w = 0; w < kJoinWarps; w++) {
        total += red[2 * w];
        a += red[2 * w + 1];
    }
    total *= g.items;
    a = a * g.items + item * chunks;
    float * to = out + ((seq * g.n_tok + mine.token) * g.n_head + mine.head) * D;
    pdl_wait();
    if (chunks == 0) {
        for (int d = tid; d < D; d += 32 * kJoinWarps) to[d] = 0.0f;
        return;
    }
    const int64_t share = (total + g.ctas - 1) / g.ctas;
    const int first = (int) (a / share), last = (int) ((a + chunks - 1) / share);
    if (first == last) return;
    constexpr int kStep = 4;  // partials of a warp in flight
    float v[D / 32] = {}, m = -INFINITY, l = 0.0f;
    for (int k0 = first + warp; k0 <= last; k0 += kStep * kJoinWarps) {
        float pm[kStep], pl[kStep], po[kStep][D / 32];
#pragma unroll
        for (int n = 0; n < kStep; n++) {
            const int k = k0 + n * kJoinWarps;
            const float * src = ws + (2 * k + (k == first ? 1 : 0)) * partial_floats(D);
            pm[n] = k <= last ? src[kRows * D + i] : -INFINITY;
            pl[n] = k <= last ? src[kRows * D + kRows + i] : 0.0f;
#pragma unroll
            for (int d = 0; d < D / 32; d++) po[n][d] = k <= last ? src[i * D + lane + 32 * d] : 0.0f;
        }
        float top = m;
#pragma unroll
        for (int n = 0; n < kStep; n++) top = fmaxf(top, pm[n]);
        const float base = top == -INFINITY ? 0.0f : top, keep = ex2(m - base);
        m = top;
        l *= keep;
#pragma unroll
        for (int d = 0; d < D / 32; d++) v[d] *= keep;
#pragma unroll
        for (int n = 0; n < kStep; n++) {
            const float f = ex2(pm[n] - base);
            l = fmaf(pl[n], f, l);
#pragma unroll
            for (int d = 0; d < D / 32; d++) v[d] = fmaf(po[n][d], f, v[d]);
        }
    }
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
#pragma unroll
    for (int d = 0; d < D / 32; d++) so[warp][lane + 32 * d] = v[d];
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kJoinWarps; w++) top = fmaxf(top, sm[w]);
    const float base = top == -INFINITY ? 0.0f : top;
    float f[kJoinWarps], sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; w++) {
        f[w] = ex2(sm[w] - base);
        sum = fmaf(sl[w], f[w], sum);
    }
    const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
    for (int d = tid; d < D; d += 32 * kJoinWarps) {
        float o = 0.0f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; w++) o = fmaf(so[w][d], f[w], o);
        to[d] = o * inv;
    }
}

Geometry geometry(const b200_context * ctx, const b200_kv_cache * c, int64_t max_pages, int64_t n_seq, int64_t n_tok, int64_t n_head) {
    Geometry g;
    g.n_tok = (int) n_tok;
    g.n_head = (int) n_head;
    g.group = (int) (n_head / c->n_kv_head);
    g.tiles = (g.n_tok * g.group + kRows - 1) / kRows;
    g.items = (int64_t) c->n_kv_head * g.tiles;
    g.n_seq = n_seq;
    g.ctas = (int64_t) ctx->num_sms * ctas_per_sm_of(c->type == B200_TYPE_Q8_0, c->head_dim);
    // By items when the lengths that the table allows are short: the cluster (1 to 8 CTAs) is the largest that all items fit
    // on the GPU with at once.
    const int64_t most = (max_pages * c->page_size + kChunk - 1) / kChunk;  // chunks of the longest sequence there can be
    g.cluster = 8;
    while (g.cluster > 1 && n_seq * g.items * g.cluster > g.ctas) g.cluster /= 2;
    if (most > kItemChunks * g.cluster) g.cluster = 0;
    if (g.ctas > most * n_seq * g.items) g.ctas = most > 0 ? most * n_seq * g.items : 1;
    return g;
}

template <bool Q8, int D>
cudaError_t launch(const KvView & c, const Geometry & g, const float * q, int64_t ldq, float scale, float * out, float * ws, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (g.cluster) {
        cfg.gridDim = dim3((unsigned) (g.n_seq * g.items * g.cluster), 1, 1);
        cfg.blockDim = dim3(kThreads, 1, 1);
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned) g.cluster;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        return cudaLaunchKernelEx(&cfg, kv_attention_item_kernel<Q8, D>, c, g, g.cluster, q, ldq, scale, out);
    }
    kv_attention_kernel<Q8, D><<<(unsigned) g.ctas, kThreads, 0, st>>>(c, g, q, ldq, scale, out, ws);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3((unsigned) (g.n_seq * g.items * kRows), 1, 1);
    cfg.blockDim = dim3(32 * kJoinWarps, 1, 1);
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    return cudaLaunchKernelEx(&cfg, kv_attention_join_kernel<D>, c, g, out, (const float *) ws);
}

size_t workspace_bytes_of(const Geometry & g, int D) { return g.cluster ? 0 : (size_t) (2 * g.ctas * partial_floats(D)) * sizeof(float); }

bool fits(const b200_kv_cache * c, int64_t max_pages, int64_t n_seq, int64_t n_tok, int64_t n_head) {
    return c && c->n_kv_head > 0 && c->page_size > 0 && max_pages >= 0 && n_seq > 0 && n_tok > 0 && n_tok <= 16 && n_head > 0 && n_head <= 65535 &&
           n_head % c->n_kv_head == 0 && max_pages <= (1 << 30) / c->page_size && n_seq * n_tok <= INT32_MAX / kRows / n_head;
}

}  // namespace

extern "C" {

size_t b200_kv_attention_workspace(b200_context * ctx, const b200_kv_cache * cache, int64_t max_pages, int64_t n_seq, int64_t n_tok,
                                   int64_t n_head) {
    if (!ctx || !fits(cache, max_pages, n_seq, n_tok, n_head)) return 0;
    return workspace_bytes_of(geometry(ctx, cache, max_pages, n_seq, n_tok, n_head), cache->head_dim);
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
    if (!fits(cache, max_pages, n_seq, n_tok, n_head)) return kv_fail(ctx, B200_ERR_INVALID, what, "n_seq * n_tok * n_head passes 2^28");
    if (ldq < n_head * c.head_dim) return kv_fail(ctx, B200_ERR_INVALID, what, "the row stride is below n_head * head_dim");
    if (!q || !out || ((uintptr_t) q & 3) || ((uintptr_t) out & 3)) return kv_fail(ctx, B200_ERR_INVALID, what, "NULL or misaligned q or out");
    const Geometry g = geometry(ctx, cache, max_pages, n_seq, n_tok, n_head);
    const size_t need = workspace_bytes_of(g, c.head_dim);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t) workspace & 255)))
        return kv_fail(ctx, B200_ERR_INVALID, what, "the workspace is missing, misaligned or too small");
    DeviceScope scope(ctx->device);
    if (scope.status != cudaSuccess) return kv_cuda(ctx, scope.status, what);
    cudaStream_t st = stream ? (cudaStream_t) stream : ctx->stream;
    auto go = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        return cache->type == B200_TYPE_Q8_0 ? launch<true, D>(c, g, q, ldq, scale, out, (float *) workspace, st)
                                             : launch<false, D>(c, g, q, ldq, scale, out, (float *) workspace, st);
    };
    cudaError_t e = cudaErrorInvalidValue;
    switch (c.head_dim) {
    case 64: e = go(std::integral_constant<int, 64>{}); break;
    case 96: e = go(std::integral_constant<int, 96>{}); break;
    case 128: e = go(std::integral_constant<int, 128>{}); break;
    case 256: e = go(std::integral_constant<int, 256>{}); break;
    default: break;
    }
    return kv_cuda(ctx, e, what);
}

}  // extern "C"
