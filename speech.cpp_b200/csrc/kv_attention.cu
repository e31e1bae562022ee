// kv_attention.cu — attention of a few new tokens per sequence over the paged key/value cache (b200_kv_attention).
//
// Mathematics. The rows of one key/value head (its group of query heads, times the call's tokens) share every key and value,
// so they are taken eight (or twice eight) at a time: S = Q K^T and O = P V over 16 positions at a time, with a running sum
// per row, in units of 2^m: m follows the maximum of the positions at hand (o and l are rescaled by 2^(m_old - m_new);
// exponentials to base 2, their scale folded into the scores'). Bytes decide: a position costs 4 D bytes (F16) or 2.125 D
// (Q8_0) of HBM and 4 D multiply-adds per row, so the arithmetic has to cost next to nothing beside the stream of the cache.
//
// Float32 results from F16 matrix instructions. mma.m16n8k16 multiplies F16 exactly and adds in float32, but takes 16 rows
// where there are at most eight: rows 0-7 of the tile hold the high half of the operand and rows 8-15 the low half (x = hi +
// lo in F16, 22 bits; q scaled by a power of two per row first), and the two results of a row lie in the same lane's
// registers, where one addition joins them. So q and the weights enter with 22 bits at the price of the padding. Q8_0's
// values are whole numbers and exact in F16; their scales stay outside: a key block's multiplies its partial score, a value
// block's multiplies the weight's two halves. An instruction's own accumulation truncates, which over thousands of positions
// would add up: at most two are chained, and their sum is added to the float32 result with a rounded addition. (Errors
// against 64 bits over rows of 1 to 131071 positions: 1.5e-7 to 6.2e-7 of the result, a plain float32 computation's being
// 2.9e-7 to 2.1e-6.) What F16 drops is what is small beside the positions taken with it: m, the unit of the weights, goes down
// again where the scores do.
//
// Operands. The k index of S = Q K^T may run through a row's dimensions in any order that both operands share, and the n index
// of O = P V through any order that the output is written back in. They are chosen such that a lane's fragment is 16 (F16
// keys and values), 8 or 4 (Q8_0) contiguous bytes of a row, read from shared memory without bank conflicts (the 16-byte chunks
// are swizzled as they are copied), and the scores' registers are the weights' fragment as they stand. Each warp copies its own
// pieces of 16 positions into its own ring with cp.async, one or more ahead, so no warp waits for another before the end.
// (Fragments loaded from HBM straight into registers need no copies, but what a warp has under way is then bound by its
// registers: at its best that form took 105 us for F16 and 168 us for Q8_0, below; the ring took 103 and 142 us at once and
// was refined from there.)
//
// Split. Sequences differ in length and there may be one of them. By positions: all (sequence, key/value head, row tile)
// items are laid end to end in chunks of 64 positions, and each CTA takes an equal run of chunks; a CTA's four warps take
// turns at a run's pieces and join at its end. Items that lie within one CTA's run are finished by it; of the others each CTA
// leaves a partial (m, l, o) in the workspace, and a second kernel, launched with programmatic dependent launch, joins them.
// By items, where a table allows short sequences only: a cluster per item, joined over distributed shared memory, in one
// launch (geometry() has the rule and both sides' times).
//
// Measured on one B200, device time (a CUDA graph of calls on the same inputs), 16 heads on 8 of 128 unless said otherwise: 64
// sequences of 512 to 4096 positions over F16 (612 MB) 99 to 103 us, 6.0 TB/s, bound by HBM; 32 of 2048 to 16384 over Q8_0
// (658 MB) 123 us, 5.3 TB/s, bound by the instructions that turn bytes into F16 and scale them (ALU pipe 46 % busy, matrix pipe
// 31 %, issue slots 60 %, some 500 instructions per 16 positions; on inputs that change from call to call, under the power limit,
// 135 to 147 us; 64 of 512 to 4096 76 us, 128 of 128 to 1024 48 us, where the bytes alone are 50 and 25); one of 131071 positions
// over Q8_0, 32 heads on 4, 40 to 42 us; one of 517 over F16 6.0 us, a chain of latencies: length, page number, rows, two or
// three pieces, the cluster's join.
#include <cooperative_groups.h>

#include <cmath>

#include "kv.cuh"

using namespace b200;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kJoinWarps = 8;  // 2^3
constexpr int kChunk = 64;       // positions of a chunk: one piece per warp
constexpr int kItemChunks = 16;  // the work is cut by items up to this many chunks per CTA,
constexpr int kItemMost = 64;    // and this many per sequence
constexpr float kShift = 14;     // weights are held times 2^14, so that their low halves reach 2^-38 of a step's largest
constexpr float kFall = 32;      // how far the unit of l and o may fall below the largest it was, in powers of two

struct Geometry {
    int n_tok, n_head, group;
    int rows, tiles;                  // rows of an item; items of a key/value head
    int vec;                          // q's rows and out are 16-byte aligned
    int64_t items;                    // n_kv_head * tiles, per sequence
    int64_t n_seq;
    int64_t ctas;                     // CTAs among which the chunks are divided, or
    int cluster;                      // CTAs that share an item (0: the work is cut by positions)
    int64_t units;                    // what may have to be joined: items, or CTAs (each begins at most one item that others end)
    int by_item, join_shift;          // which of the two; logarithm of the warps per row of the join
};

constexpr int64_t partial_floats(int D, int rows) { return (int64_t) rows * (D + 2); }  // o [rows][D], m [rows], l [rows]

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <class T>
__device__ __forceinline__ T first_lane(T x) { return __shfl_sync(0xffffffffu, x, 0); }

// d = A B + c, and d = A B.
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    const float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    mma(d, a, b0, b1, c);
}

// 16 bytes from global to shared memory, asynchronously; zeros when !there (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t to, const uint8_t * from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}

__device__ __forceinline__ void copy16(uint32_t to, const uint8_t * from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

// N 32-bit words at a shared address.
template <int N>
__device__ __forceinline__ void lds(uint32_t (&w)[N], uint32_t at) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "r"(at + 4 * i));
    } else if constexpr (N == 2) {
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[i]) : "r"(at + 4 * i));
    }
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
    return i & 1 ? __high2float(h2(w[i >> 1])) : __low2float(h2(w[i >> 1]));
}

// How a head's rows are taken apart. The n index of O = P V runs through the dimensions in groups of 8 kRun, lane quad g
// holding kRun contiguous ones of each.
template <bool Q8, int D, int TILES>
struct Shape {
    static constexpr bool kQ8 = Q8;
    static constexpr int kDim = D, kTiles = TILES, kRows = 8 * TILES;  // kRows: rows of an item
    static constexpr int kBlocks = D / 32;
    static constexpr int kRun = !Q8 && D % 64 == 0 ? 8 : 4;
    static constexpr int kGroups = D / (8 * kRun);
    static constexpr int kKeyWords = Q8 ? 2 : 4;           // a lane's words of a row's 32 dimensions
    static constexpr int kValueWords = Q8 ? 1 : kRun / 2;  // a lane's words of a row's group
    // A piece is 16 positions: its key rows, value rows, and their scales. A warp takes kSub pieces at a time (two of Q8_0 share
    // the running maximum's and sum's arithmetic and one addition to o: 125.6 -> 123.2 us for the batch above), from a ring of
    // kStages such in shared memory; the ring's depth and the CTAs per SM fill its 227 KB and the registers. (F16, D = 128: two
    // CTAs with three stages 104.2 us, three with two 105.1. Q8_0, D = 128: three with two 122.7 us, two with three 123.9, and
    // 128 sequences of 1024 to 4096 169 and 174 us, but the one of 131071 40.8 and 38.2.)
    static constexpr int kSub = Q8 && D <= 128 ? 2 : 1;
    static constexpr int kRowBytes = Q8 ? D : 2 * D;
    static constexpr int kScaleBytes = Q8 ? D / 16 : 0;    // of a row
    static constexpr int kPiece = 32 * (kRowBytes + kScaleBytes);
    static constexpr int kStages = Q8 ? (D == 128 && TILES == 1 ? 2 : 3) : (D == 64 ? 4 : D == 256 ? 2 : 3);
    static constexpr int kCtas = Q8 ? (TILES == 1 && (D == 64 || D == 128) ? 3 : 2) : (D == 256 ? 1 : D == 128 || TILES == 2 ? 2 : 3);
    static_assert(D == 96 || kPiece % 128 == 0, "swizzled pieces keep the ring's alignment");
    static constexpr int kStage = kSub * kPiece, kBytes = kWarps * kStages * kStage;
    // The 16-byte chunks of a row are stored at chunk ^ swizzle(row), so that the lanes that read together read different
    // banks: fragments of keys are read from rows 0-7 (Q8_0: four rows and 32 bytes of each at a time, F16: two rows and
    // 64), of values from rows 0, 2, 4, 6 and so on. Rows of 96 or 192 bytes are apart by themselves (keys) or in pairs. Both
    // take bits of the row to bits of the chunk, so swizzle(a | b) = swizzle(a) ^ swizzle(b).
    static constexpr bool kSwizzled = D != 96;
    static constexpr int key_swizzle(int row) {
        return D == 96 ? 0 : !Q8 ? (row & 1) << 2 : D == 64 ? (row >> 1 & 1) << 1 : (row & 3) << 1;
    }
    static constexpr int value_swizzle(int row) {
        return D == 96 ? 0 : !Q8 ? row & 6 : D == 64 ? (row >> 1 & 1) << 1 : (row >> 1 & 3) << 1;
    }
    // From the address of a lane's first fragment in a row to that of the one `bytes` further on in the row (pieces start at
    // multiples of 128 bytes, and the swizzle moves chunks within 128).
    static __device__ __forceinline__ uint32_t along(uint32_t at, uint32_t bytes) {
        return kSwizzled ? (at ^ (bytes & 127)) + (bytes & ~127u) : at + bytes;
    }
};

__device__ __forceinline__ int64_t chunks_of(const KvView & c, int64_t s, bool tell) { return (kv_len(c, s, tell) + kChunk - 1) / kChunk; }

__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Where a CTA's share of the chunks lies: chunk numbers count the sequences' chunks one after the other, each `items` times.
struct Place {
    int64_t at, end;     // the chunks [at, end) of all
    int64_t share;       // end - at, but for the last one
    int64_t seq, start;  // the sequence that chunk `at` (LAST: the share's last one) lies in, and its first chunk (when at < end)
};

// CTA b's place, block-wide (every thread gets the result): the lengths are read 32 WARPS at a time, summed for the share and
// scanned for the sequence; up to that many of them stay in registers in between.
template <int WARPS, bool LAST>
__device__ __forceinline__ Place find_place(const KvView & c, const Geometry & g, int64_t b, bool tell, int64_t (&red)[WARPS + 2]) {
    constexpr int kStep = 32 * WARPS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t first = threadIdx.x < g.n_seq ? chunks_of(c, threadIdx.x, tell) * g.items : 0;
    int64_t sum = first;
    for (int64_t s = threadIdx.x + kStep; s < g.n_seq; s += kStep) sum += chunks_of(c, s, tell) * g.items;
    sum = warp_sum64(sum);
    if (lane == 0) red[warp] = sum;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; w++) total += red[w];
    Place p;
    p.share = (total + g.ctas - 1) / g.ctas;
    p.at = b * p.share;
    p.end = p.at + p.share < total ? p.at + p.share : total;
    p.seq = p.start = 0;
    if (p.at >= p.end) return p;  // the same for all threads
    const int64_t to = LAST ? p.end - 1 : p.at;
    int64_t base = 0;
    for (int64_t s0 = 0; s0 < g.n_seq; s0 += kStep) {
        const int64_t s = s0 + threadIdx.x;
        const int64_t mine = s0 == 0 ? first : s < g.n_seq ? chunks_of(c, s, false) * g.items : 0;
        int64_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        __syncthreads();
        if (lane == 31) red[warp] = incl;
        __syncthreads();
        int64_t before = base, all = 0;
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            if (w < warp) before += red[w];
            all += red[w];
        }
        const int64_t begin = before + incl - mine;
        if (mine > 0 && to >= begin && to < begin + mine) {
            red[WARPS] = s;
            red[WARPS + 1] = begin;
        }
        base += all;
        if (to < base) break;  // the same for all threads
    }
    __syncthreads();
    p.seq = red[WARPS];
    p.start = red[WARPS + 1];
    return p;
}

// Rows of an item: row i is query head h * group + n % group of token n / group, n = tile * rows + i.
struct Row {
    int token, head;
    bool there;
};

template <int ROWS>
__device__ __forceinline__ Row row_of(const Geometry & g, int h, int tile, int i) {
    const int n = tile * ROWS + i;
    return {n / g.group, h * g.group + n % g.group, n < g.n_tok * g.group};
}

// A CTA's shared memory: the warps' rings of pieces, and, at the ring's place once a run is done, each warp's o.
template <class S>
struct Shared {
    uint8_t * ring;  // dynamic: [kWarps][kStages][kSub][kPiece]
    float (*sm)[S::kRows];
    float (*sl)[S::kRows];
    static constexpr int kRingBytes = S::kStages * S::kStage;
    static constexpr int kPitch = S::kDim + 4;
    static_assert(S::kRows * kPitch * 4 <= kRingBytes, "a warp's o fits its ring");
    // dimensions d to d + 3 of a row (d % 4 == 0)
    __device__ __forceinline__ float4 & o(int w, int row, int d) const {
        return reinterpret_cast<float4 *>(ring + w * kRingBytes)[(row * kPitch + d) / 4];
    }
};

// Chunks [c0, c1) of one item: the warps' m, l and o are left in shared memory (synchronised).
template <class S>
__device__ __forceinline__ void attend(const KvView & c, const Geometry & g, const float * __restrict__ q, int64_t ldq, float scale,
                                       const Shared<S> & sh, int64_t seq, int64_t len, int h, int tile, int64_t c0, int64_t c1) {
    constexpr bool Q8 = S::kQ8;
    constexpr int D = S::kDim, TILES = S::kTiles;
    constexpr int kRowBytes = S::kRowBytes, kValues = 16 * kRowBytes, kKeyScales = 32 * kRowBytes, kValueScales = kKeyScales + 16 * S::kScaleBytes;
    const int tid = threadIdx.x, lane = tid & 31;
    // What is the same for a whole warp comes from its first lane, so that the compiler knows it and computes with it once.
    const int warp = first_lane(tid >> 5);
    seq = first_lane(seq), len = first_lane(len), c0 = first_lane(c0), c1 = first_lane(c1);
    h = first_lane(h), tile = first_lane(tile);
    const int gq = lane >> 2, t = lane & 3;  // the fragment's group and thread in it
    Row row[TILES];
#pragma unroll
    for (int y = 0; y < TILES; y++) row[y] = row_of<S::kRows>(g, h, tile, 8 * y + gq);
    const int p_end = (int) (c1 * kChunk < len ? c1 * kChunk : len);
    const int all_see = (int) len - g.n_tok + 1;  // positions below are seen by every row
    int seen[TILES];
#pragma unroll
    for (int y = 0; y < TILES; y++) seen[y] = row[y].there ? all_see + row[y].token : 0;

    // ---- the ring: steps of kSub pieces, the warps in turn through [c0 * 64, c1 * 64), copied kStages - 1 ahead ----
    constexpr int kSub = S::kSub, kStep = kWarps * 16 * kSub;
    const uint32_t ring = smem_addr(sh.ring) + warp * Shared<S>::kRingBytes;
    // a page's bytes: a multiple of 512 (16 rows of a multiple of 32 bytes), and 32 bits hold them in such units
    const uint32_t page_units = (uint32_t) ((int64_t) c.n_kv_head * c.page_size * kRowBytes / 512);
    const int32_t * pages = c.table + seq * c.max_pages;
    const uint8_t * kh = c.k + (int64_t) h * c.page_size * kRowBytes + lane * 16;
    const int64_t to_values = c.v - c.k;
    const uint8_t * scales = nullptr;  // this lane's 16 bytes of a piece's scales: the keys', then the values'
    if constexpr (Q8)
        scales = reinterpret_cast<const uint8_t *>(lane < S::kScaleBytes ? c.kd : c.vd) + (int64_t) h * c.page_size * S::kScaleBytes +
                 (lane < S::kScaleBytes ? lane : lane - S::kScaleBytes) * 16;
    const int page_step = kStep / c.page_size, slot_step = kStep % c.page_size;
    int p_copy = (int) c0 * kChunk + warp * 16 * kSub;  // the next step to copy, its place in the table, its pages (asked for early)
    int in_table = p_copy / c.page_size, slot = p_copy % c.page_size, stage_copy = 0;
    int page[kSub];
    auto find_pages = [&] {
#pragma unroll
        for (int u = 0; u < kSub; u++)
            page[u] = p_copy + 16 * u < p_end ? pages[in_table + (slot + 16 * u >= c.page_size)] : -1;
    };
    find_pages();
    // where this lane's first 16 bytes of a piece go: row lane / (chunks of a row), chunk lane % (chunks of a row)
    const uint32_t copy_key = lane * 16 ^ S::key_swizzle(lane / (kRowBytes / 16)) * 16;
    const uint32_t copy_value = lane * 16 ^ S::value_swizzle(lane / (kRowBytes / 16)) * 16;
    unsigned found = 0;  // of the steps copied, the last in the lowest kSub bits: which pieces have a page
    auto copy_step = [&] {
        found <<= kSub;
        if (p_copy < p_end) {
#pragma unroll
            for (int u = 0; u < kSub; u++) {
                const unsigned number = (unsigned) first_lane(page[u]);
                const bool exists = number < (unsigned) c.n_pages;
                const int here = exists ? p_end - p_copy - 16 * u : 0;  // rows of the piece; the others are zeros
                if (!exists && p_copy + 16 * u < p_end && lane == 0) atomicOr(c.err, B200_DEVERR_PAGE);
                const int in_page = slot + 16 * u - (slot + 16 * u >= c.page_size ? c.page_size : 0);
                const int64_t at = (int64_t) ((uint64_t) (exists ? number : 0) * page_units << 9) + in_page * kRowBytes;
                const uint8_t * from = kh + at;
                const uint32_t to = ring + stage_copy * S::kStage + u * S::kPiece;
                constexpr int kRowChunks = kRowBytes / 16, kCopies = kRowChunks / 2;  // a piece's rows are contiguous: 16 kRowChunks chunks
                auto each = [&](auto whole) {
#pragma unroll
                    for (int j = 0; j < kCopies; j++) {
                        uint32_t key_to, value_to, r;
                        if constexpr (S::kSwizzled) {  // 32 / kRowChunks rows further each time: their swizzle is a constant
                            r = lane / kRowChunks + j * (32 / kRowChunks);
                            key_to = (copy_key ^ (S::key_swizzle(j * (32 / kRowChunks)) * 16)) + j * 512;
                            value_to = (copy_value ^ (S::value_swizzle(j * (32 / kRowChunks)) * 16)) + j * 512;
                        } else {
                            r = (lane + 32 * j) / kRowChunks;
                            key_to = value_to = (lane + 32 * j) * 16;
                        }
                        if constexpr (decltype(whole)::value) {
                            copy16(to + key_to, from + j * 512);
                            copy16(to + kValues + value_to, from + to_values + j * 512);
                        } else {
                            copy16(to + key_to, from + j * 512, (int) r < here);
                            copy16(to + kValues + value_to, from + to_values + j * 512, (int) r < here);
                        }
                    }
                };
                if (here >= 16) each(std::true_type{});
                else each(std::false_type{});
                if constexpr (Q8) {  // whole, rows behind the end too: they lie in the page
                    if (lane < 2 * S::kScaleBytes) copy16(to + kKeyScales + lane * 16, scales + (at >> 4), exists);
                }
                if (exists) found |= 1u << u;
            }
            p_copy += kStep;
            in_table += page_step;
            slot += slot_step;
            if (slot >= c.page_size) slot -= c.page_size, in_table++;
            find_pages();
            stage_copy = stage_copy + 1 == S::kStages ? 0 : stage_copy + 1;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int n = 0; n < S::kStages - 1; n++) copy_step();

    // ---- the query tile's fragments ----
    // k step 2 j + b of lane (gq, t) holds dimensions 32 j + 8 t + 4 b .. + 3 of row gq: hi in registers 0 and 2, lo in
    // 1 and 3. The row is scaled by 2^k to a largest magnitude in [2^14, 2^15).
    uint32_t qf[TILES][D / 16][4];
    float factor[TILES];  // what a raw score is multiplied by: scale log2(e) 2^-k
#pragma unroll
    for (int y = 0; y < TILES; y++) {
        const float * src = q + (seq * g.n_tok + row[y].token) * ldq + (int64_t) row[y].head * D + 8 * t;
        float x[D / 4], top = 0.0f;
        if (g.vec && row[y].there) {
#pragma unroll
            for (int i = 0; i < D / 4; i += 4) {
                const float4 v = *reinterpret_cast<const float4 *>(src + (i / 8) * 32 + i % 8);
                x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < D / 4; i++) x[i] = row[y].there ? src[(i / 8) * 32 + i % 8] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < D / 4; i++) top = fmaxf(top, fabsf(x[i]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = (int) (__float_as_uint(top) >> 23);
        const int k = e == 255 || top == 0.0f ? 0 : 141 - e < 126 ? 141 - e : 126;
        const float up = __uint_as_float((uint32_t) (k + 127) << 23);
        factor[y] = scale * 1.4426950408889634f * __uint_as_float((uint32_t) (127 - k) << 23);
#pragma unroll
        for (int j = 0; j < D / 16; j++) {
            split(x[4 * j] * up, x[4 * j + 1] * up, qf[y][j][0], qf[y][j][1]);
            split(x[4 * j + 2] * up, x[4 * j + 3] * up, qf[y][j][2], qf[y][j][3]);
        }
    }

    // this lane's places in a piece: dimensions 8 t of key row gq, kRun gq of value row 2 t (rows 8 further, and row 2 t + 1
    // beside 2 t, are swizzled alike)
    const uint32_t key_at = gq * kRowBytes + ((t * (Q8 ? 8 : 16)) ^ (S::key_swizzle(gq) * 16));
    const uint32_t value_at = kValues + 2 * t * kRowBytes + ((gq * S::kRun * (Q8 ? 1 : 2)) ^ (S::value_swizzle(2 * t) * 16));

    const int plain_end = min(p_end, all_see);  // steps that end here or before have all their positions, seen by every row
    float2 o[TILES][S::kGroups][S::kRun] = {};
    float m[TILES], m_most[TILES], l[TILES];
#pragma unroll
    for (int y = 0; y < TILES; y++) m[y] = m_most[y] = -INFINITY, l[y] = 0.0f;
    int stage = 0;
    for (int p0 = (int) c0 * kChunk + warp * 16 * kSub; p0 < p_end; p0 += kStep) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
        __syncwarp();  // the step is here for every lane, and every lane is done with the one before, whose place is refilled
        const uint32_t at = ring + stage * S::kStage;
        const unsigned pages_here = found >> (kSub * (S::kStages - 2)) & ((1u << kSub) - 1);
        const bool edge = p0 + 16 * kSub > plain_end || pages_here != (1u << kSub) - 1;
        auto here = [&](int u) { return pages_here >> u & 1 ? p_end - p0 - 16 * u : 0; };  // positions of a piece
        stage = stage + 1 == S::kStages ? 0 : stage + 1;
        copy_step();

        // ---- scores: s[y][u][2 i + j] is position 16 u + 2 t + j + 8 i of row 8 y + gq ----
        float s[TILES][kSub][4];
#pragma unroll
        for (int u = 0; u < kSub; u++) {
            const uint32_t keys = at + u * S::kPiece + key_at;
            uint32_t kd[2][Q8 ? S::kBlocks : 1];
            if constexpr (Q8) {
#pragma unroll
                for (int i = 0; i < 2; i++) lds(kd[i], at + u * S::kPiece + kKeyScales + (2 * t + 8 * i) * S::kScaleBytes);
            }
            float2 part[TILES][2] = {};
#pragma unroll
            for (int b = 0; b < S::kBlocks; b++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    uint32_t w[S::kKeyWords];
                    lds(w, S::along(keys, b * (Q8 ? 32 : 64)) + i * 8 * kRowBytes);
                    if constexpr (Q8) {
                        const uint32_t w0 = w[0] ^ 0x80808080u, w1 = w[1] ^ 0x80808080u;
                        const uint32_t f[4] = {halves(w0, 0x4140), halves(w0, 0x4342), halves(w1, 0x4140), halves(w1, 0x4342)};
                        const float2 d = make_float2(half_of(kd[i], b), half_of(kd[i], S::kBlocks + b));
#pragma unroll
                        for (int y = 0; y < TILES; y++) {
                            float r[4];
                            mma(r, qf[y][2 * b], f[0], f[1]);
                            mma(r, qf[y][2 * b + 1], f[2], f[3], r);
                            const float2 whole = __fadd2_rn(make_float2(r[0], r[1]), make_float2(r[2], r[3]));
                            part[y][i] = __ffma2_rn(d, whole, part[y][i]);
                        }
                    } else {
#pragma unroll
                        for (int y = 0; y < TILES; y++) {
                            float r[4];
                            mma(r, qf[y][2 * b], w[0], w[1]);
                            mma(r, qf[y][2 * b + 1], w[2], w[3], r);
                            part[y][i] = __fadd2_rn(part[y][i], __fadd2_rn(make_float2(r[0], r[1]), make_float2(r[2], r[3])));
                        }
                    }
                }
#pragma unroll
            for (int y = 0; y < TILES; y++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    s[y][u][2 * i] = part[y][i].x * factor[y];
                    s[y][u][2 * i + 1] = part[y][i].y * factor[y];
                }
        }
        if (edge) {
#pragma unroll
            for (int y = 0; y < TILES; y++)
#pragma unroll
                for (int u = 0; u < kSub; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int j = 2 * t + (i & 1) + 8 * (i >> 1);
                        if (j >= here(u) || p0 + 16 * u + j >= seen[y]) s[y][u][i] = -INFINITY;
                    }
        }

        // ---- weights, in units of 2^m: m is the step's maximum, rounded up, less kShift (-infinity before any score) ----
        // So what F16 cannot hold of a weight, or of its product with a scale, is small beside this step's largest, not only
        // beside that of a position far away whose values may be 0. m stays within kFall of the largest it was, so that l and o
        // do not leave float32's range, and is whole, so that going from one m to another is exact.
        float2 keep[TILES];
        uint32_t pf[TILES][kSub][4];  // the weights' fragments: hi, lo of positions 2 t, 2 t + 1, then of 2 t + 8, 2 t + 9
#pragma unroll
        for (int y = 0; y < TILES; y++) {
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < kSub; u++) top = fmaxf(top, fmaxf(fmaxf(s[y][u][0], s[y][u][1]), fmaxf(s[y][u][2], s[y][u][3])));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float own = __fadd_ru(ceilf(top), -kShift);  // rounded down, top - m could pass 14 where floats are 4 apart
            m_most[y] = fmaxf(m_most[y], own);
            const float m_new = fmaxf(own, m_most[y] - kFall);
            const float base = m_new == -INFINITY ? 0.0f : m_new;
            const float k = ex2(m[y] - base);
            keep[y] = make_float2(k, k);
            m[y] = m_new;
            l[y] *= k;
#pragma unroll
            for (int u = 0; u < kSub; u++) {
#pragma unroll
                for (int i = 0; i < 4; i++) s[y][u][i] = ex2(s[y][u][i] - base);
                l[y] += (s[y][u][0] + s[y][u][1]) + (s[y][u][2] + s[y][u][3]);
                split(s[y][u][0], s[y][u][1], pf[y][u][0], pf[y][u][1]);
                split(s[y][u][2], s[y][u][3], pf[y][u][2], pf[y][u][3]);
            }
        }

        // ---- o = o keep + P V: values of rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9, the positions whose weights this lane holds ----
        using Words = uint32_t[4][S::kValueWords];
        auto values = [&](Words & w, int u, int n) {
            const uint32_t first = at + u * S::kPiece + value_at;
#pragma unroll
            for (int i = 0; i < 4; i++) lds(w[i], (Q8 ? S::along(first, 32 * n) : first + 16 * S::kRun * n) + ((i & 1) + 8 * (i >> 1)) * kRowBytes);
        };
        if constexpr (Q8) {
            uint32_t vd[kSub][2][S::kBlocks];
#pragma unroll
            for (int u = 0; u < kSub; u++)
#pragma unroll
                for (int i = 0; i < 2; i++) lds(vd[u][i], at + u * S::kPiece + kValueScales + (2 * t + 8 * i) * S::kScaleBytes);
            if (edge) {  // scales behind the end (their weights are 0) as 1, whatever lies there
#pragma unroll
                for (int u = 0; u < kSub; u++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const uint32_t a = 2 * t + 8 * i < here(u) ? 0 : 0x3c00, b = 2 * t + 1 + 8 * i < here(u) ? 0 : 0x3c00;
#pragma unroll
                        for (int n = 0; n < S::kBlocks; n++) {  // halves 2 n and 2 n + 1: the first kBlocks are row 2 t's
                            const uint32_t low = 2 * n < S::kBlocks ? a : b, high = 2 * n + 1 < S::kBlocks ? a : b;
                            if (low) vd[u][i][n] = (vd[u][i][n] & 0xffff0000u) | low;
                            if (high) vd[u][i][n] = (vd[u][i][n] & 0xffffu) | high << 16;
                        }
                    }
            }
            using Fragments = uint32_t[S::kTiles][S::kSub][4];
            // one block of 32 dimensions: weights times scales (fragments a), which where `scaled` come times 1 / down
            auto block = [&](int b, const Fragments & a, auto scaled, const float * down) {
                uint32_t x[S::kSub][2][2];  // two rows' four bytes each, interleaved: (row, row + 1) pairs
#pragma unroll
                for (int u = 0; u < kSub; u++) {
                    Words w;
                    values(w, u, b);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        x[u][i][0] = __byte_perm(w[2 * i][0], w[2 * i + 1][0], 0x5140) ^ 0x80808080u;
                        x[u][i][1] = __byte_perm(w[2 * i][0], w[2 * i + 1][0], 0x7362) ^ 0x80808080u;
                    }
                }
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    const uint32_t sel = n & 1 ? 0x4342 : 0x4140;
                    uint32_t f[S::kSub][2];
#pragma unroll
                    for (int u = 0; u < kSub; u++) f[u][0] = halves(x[u][0][n / 2], sel), f[u][1] = halves(x[u][1][n / 2], sel);
#pragma unroll
                    for (int y = 0; y < TILES; y++) {
                        float r[4];
                        mma(r, a[y][0], f[0][0], f[0][1]);
#pragma unroll
                        for (int u = 1; u < kSub; u++) mma(r, a[y][u], f[u][0], f[u][1], r);
                        float2 part = __fadd2_rn(make_float2(r[0], r[1]), make_float2(r[2], r[3]));
                        if constexpr (decltype(scaled)::value) part.x *= down[y], part.y *= down[y];
                        o[y][b][n] = __ffma2_rn(o[y][b][n], keep[y], part);
                    }
                }
            };
            // Scales between 2^-13 and 2 (nearly always all of them) multiply the weights' halves in F16 pairs: the product's
            // rounding error is exact in F16 and goes to the low half. The largest weight being in (2^13, 2^14] and the low halves
            // reaching 2^-24, nothing overflows, and products below 2^-25 of the largest weight times the least scale are lost, as
            // they would be beside it in a float32 sum. (Powers of two that bring each block's scales to 1 first would keep 2^-36, at
            // 5 to 10 % of the time; all scales as below take 146 instead of 123 us for the batch above.)
            uint32_t low = vd[0][0][0], high = vd[0][0][0];
#pragma unroll
            for (int u = 0; u < kSub; u++)
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int b = 0; b < S::kBlocks; b++) low = __vminu2(low, vd[u][i][b]), high = __vmaxu2(high, vd[u][i][b]);
            const bool plain = (low & 0xffffu) >= 0x0800u && low >= 0x08000000u && (high & 0xffffu) < 0x4000u && high < 0x40000000u;
            if (__all_sync(0xffffffffu, plain)) {
                auto go = [&](auto index) {
                    constexpr int b = decltype(index)::value;
                    if constexpr (b < S::kBlocks) {
                        Fragments a;
#pragma unroll
                        for (int u = 0; u < kSub; u++)
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                const __half2 d = h2(pair_of<b, S::kBlocks + b>(vd[u][i]));
#pragma unroll
                                for (int y = 0; y < TILES; y++) {
                                    const __half2 hi = h2(pf[y][u][2 * i]), w = __hmul2_rn(hi, d);
                                    a[y][u][2 * i] = u32(w);
                                    a[y][u][2 * i + 1] = u32(__hfma2(h2(pf[y][u][2 * i + 1]), d, __hfma2(hi, d, __hneg2(w))));
                                }
                            }
                        block(b, a, std::false_type{}, nullptr);
                    }
                };
                go(std::integral_constant<int, 0>{}), go(std::integral_constant<int, 1>{}), go(std::integral_constant<int, 2>{});
                go(std::integral_constant<int, 3>{}), go(std::integral_constant<int, 4>{}), go(std::integral_constant<int, 5>{});
                go(std::integral_constant<int, 6>{}), go(std::integral_constant<int, 7>{});
            } else {
                // any scales: the product in float32, times a power of two that brings a row's largest to [2^13, 2^14)
#pragma unroll
                for (int b = 0; b < S::kBlocks; b++) {
                    Fragments a;
                    float down[TILES];
#pragma unroll
                    for (int y = 0; y < TILES; y++) {
                        float w[kSub][4], big = 0.0f;
#pragma unroll
                        for (int u = 0; u < kSub; u++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const float d = half_of(vd[u][i >> 1], (i & 1) * S::kBlocks + b);
                                w[u][i] = edge && s[y][u][i] == 0.0f ? 0.0f : s[y][u][i] * d;
                                big = fmaxf(big, fabsf(w[u][i]));
                            }
                        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                        const int e = (int) (__float_as_uint(big) >> 23);
                        const int k = e == 255 ? 0 : min(140 - e, 126);  // at least -114
                        const float up = __uint_as_float((uint32_t) (127 + k) << 23);
                        down[y] = __uint_as_float((uint32_t) (127 - k) << 23);
#pragma unroll
                        for (int u = 0; u < kSub; u++) {
                            split(w[u][0] * up, w[u][1] * up, a[y][u][0], a[y][u][1]);
                            split(w[u][2] * up, w[u][3] * up, a[y][u][2], a[y][u][3]);
                        }
                    }
                    block(b, a, std::true_type{}, down);
                }
            }
        } else {
            static_assert(Q8 || kSub == 1, "an F16 step is one piece");
            // `below`: rows from this place in the piece on enter as zeros
            auto product = [&](int below, int token) {  // token: only its rows' results count (-1: every row's)
#pragma unroll
                for (int n = 0; n < S::kGroups; n++) {
                    Words w;
                    values(w, 0, n);
                    if (below < 16) {
#pragma unroll
                        for (int i = 0; i < 4; i++)
#pragma unroll
                            for (int r = 0; r < S::kValueWords; r++)
                                if (2 * t + (i & 1) + 8 * (i >> 1) >= below) w[i][r] = 0;
                    }
#pragma unroll
                    for (int r = 0; r < S::kRun; r++) {
                        const uint32_t sel = r & 1 ? 0x7632 : 0x5410;
                        const uint32_t f0 = __byte_perm(w[0][r / 2], w[1][r / 2], sel), f1 = __byte_perm(w[2][r / 2], w[3][r / 2], sel);
#pragma unroll
                        for (int y = 0; y < TILES; y++) {
                            float part[4];
                            mma(part, pf[y][0], f0, f1);
                            if (token < 0 || row[y].token == token)
                                o[y][n][r] = __ffma2_rn(o[y][n][r], keep[y], __fadd2_rn(make_float2(part[0], part[1]), make_float2(part[2], part[3])));
                        }
                    }
                }
            };
            bool flaw = false;
            if (edge && g.n_tok > 1) {  // is a value that not every row sees NaN or infinite?
                uint32_t high = 0;
#pragma unroll
                for (int n = 0; n < S::kGroups; n++) {
                    Words w;
                    values(w, 0, n);
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int r = 0; r < S::kValueWords; r++)
                            if (p0 + 2 * t + (i & 1) + 8 * (i >> 1) >= all_see) high = __vmaxu2(high, w[i][r] & 0x7c007c00u);
                }
                flaw = __any_sync(0xffffffffu, (high & 0xffffu) == 0x7c00u || high >= 0x7c000000u);
            }
            if (flaw) {
                // It must not meet the weight 0 of a row that does not see it: one product per token, with the values behind
                // its position zeroed. (With finite values this gives the bits that one product for all gives.)
                const int last = min((tile * S::kRows + S::kRows - 1) / g.group, g.n_tok - 1);
                for (int token = tile * S::kRows / g.group; token <= last; token++) product(all_see + token - p0, token);
            } else {
                product(16, -1);
            }
        }
    }

    // ---- join the warps ----
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();  // the ring is read no more: o takes its place
#pragma unroll
    for (int y = 0; y < TILES; y++) {
        l[y] += __shfl_xor_sync(0xffffffffu, l[y], 1);
        l[y] += __shfl_xor_sync(0xffffffffu, l[y], 2);
        if (t == 0) {
            sh.sm[warp][8 * y + gq] = m[y];
            sh.sl[warp][8 * y + gq] = l[y];
        }
#pragma unroll
        for (int n = 0; n < S::kGroups; n++)
#pragma unroll
            for (int r = 0; r < S::kRun; r += 4) {
                const float2 * v = &o[y][n][r];
                sh.o(warp, 8 * y + gq, n * 8 * S::kRun + 2 * t * S::kRun + r) = make_float4(v[0].x, v[1].x, v[2].x, v[3].x);
                sh.o(warp, 8 * y + gq, n * 8 * S::kRun + (2 * t + 1) * S::kRun + r) = make_float4(v[0].y, v[1].y, v[2].y, v[3].y);
            }
    }
    __syncthreads();
}

__device__ __forceinline__ float4 fma4(float4 a, float b, float4 c) {
    return make_float4(fmaf(a.x, b, c.x), fmaf(a.y, b, c.y), fmaf(a.z, b, c.z), fmaf(a.w, b, c.w));
}

// Four results times f to p.
__device__ __forceinline__ void put4(float * p, float4 v, float f, bool vec) {
    v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
    if (vec) *reinterpret_cast<float4 *>(p) = v;
    else p[0] = v.x, p[1] = v.y, p[2] = v.z, p[3] = v.w;
}

// The CTA's sum of the warps' results for one row: the factors of the warps, and m and l.
template <class S>
struct Joined {
    float f[kWarps], m, l;
    __device__ __forceinline__ Joined(const Shared<S> & sh, int i) {
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
    __device__ __forceinline__ float4 value(const Shared<S> & sh, int i, int d) const {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWarps; w++) v = fma4(sh.o(w, i, d), f[w], v);
        return v;
    }
};

// The work cut by positions: CTA b takes chunks [b share, (b + 1) share) of all items' chunks.
template <class S>
__global__ void __launch_bounds__(kThreads, S::kCtas)
    kv_attention_kernel(KvView c, Geometry g, const float * __restrict__ q, int64_t ldq, float scale, float * __restrict__ out, float * __restrict__ ws) {
    constexpr int D = S::kDim, kRows = S::kRows;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ float sm[kWarps][kRows], sl[kWarps][kRows];
    __shared__ int64_t red[kWarps + 2];
    const Shared<S> sh{ring, sm, sl};
    const int tid = threadIdx.x;
    pdl_launch_dependents();

    const Place place = find_place<kWarps, false>(c, g, blockIdx.x, blockIdx.x == 0, red);
    int64_t at = place.at, seq = place.seq, start = place.start;
    const int64_t end = place.end;
    if (at >= end) return;
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
        attend<S>(c, g, q, ldq, scale, sh, seq, len, h, tile, c0, c1);

        for (int i = tid / 16; i < kRows; i += kThreads / 16) {  // a row per 16 threads
            const Joined<S> all(sh, i);
            const Row row = row_of<kRows>(g, h, tile, i);
            if (c0 == 0 && c1 == chunks) {  // the whole item
                const float inv = all.l != 0.0f ? 1.0f / all.l : 0.0f;
                if (row.there)
                    for (int d = 4 * (tid & 15); d < D; d += 64)
                        put4(out + ((seq * g.n_tok + row.token) * g.n_head + row.head) * D + d, all.value(sh, i, d), inv, g.vec);
            } else {  // the CTA's first partial (of an item begun before it) or its last
                float * to = ws + (2 * blockIdx.x + (c0 == 0 ? 1 : 0)) * partial_floats(D, kRows);
                for (int d = 4 * (tid & 15); d < D; d += 64) put4(to + i * D + d, all.value(sh, i, d), 1.0f, true);
                if ((tid & 15) == 0) {
                    to[kRows * D + i] = all.m;
                    to[kRows * D + kRows + i] = all.l;
                }
            }
        }
        __syncthreads();  // the shared memory is written again by the next run
    }
}

// The work cut by items: a cluster of `cluster` CTAs per item, each an equal run of its chunks, joined over distributed
// shared memory: the CTA of rank r writes rows r, r + cluster, ... One launch, and no length but the item's own is read.
template <class S>
__global__ void __launch_bounds__(kThreads, S::kCtas)
    kv_attention_item_kernel(KvView c, Geometry g, int cluster, const float * __restrict__ q, int64_t ldq, float scale, float * __restrict__ out) {
    constexpr int D = S::kDim, kRows = S::kRows;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ float sm[kWarps][kRows], sl[kWarps][kRows];
    __shared__ float jm[kRows], jl[kRows];
    const Shared<S> sh{ring, sm, sl};
    const int tid = threadIdx.x, rank = blockIdx.x % cluster;
    const int64_t unit = blockIdx.x / cluster, seq = unit / g.items;
    const int item = (int) (unit % g.items), h = item / g.tiles, tile = item % g.tiles;
    const int64_t len = kv_len(c, seq, tid == 0), chunks = (len + kChunk - 1) / kChunk, per = (chunks + cluster - 1) / cluster;
    const int64_t c0 = rank * per < chunks ? rank * per : chunks, c1 = c0 + per < chunks ? c0 + per : chunks;
    attend<S>(c, g, q, ldq, scale, sh, seq, len, h, tile, c0, c1);
    for (int i = tid / 16; i < kRows; i += kThreads / 16) {
        const Joined<S> all(sh, i);
        for (int d = 4 * (tid & 15); d < D; d += 64) sh.o(0, i, d) = all.value(sh, i, d);  // read and written by this thread alone
        if ((tid & 15) == 0) jm[i] = all.m, jl[i] = all.l;
    }
    const cooperative_groups::cluster_group group = cooperative_groups::this_cluster();
    group.sync();
    for (int e = tid; e < kRows / cluster * (D / 4); e += kThreads) {
        const int i = e / (D / 4) * cluster + rank, d = e % (D / 4) * 4;
        const Row row = row_of<kRows>(g, h, tile, i);
        if (!row.there) continue;
        float m = -INFINITY, l = 0.0f;
        for (int r = 0; r < cluster; r++) m = fmaxf(m, *group.map_shared_rank(&jm[i], r));
        const float base = m == -INFINITY ? 0.0f : m;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int r = 0; r < cluster; r++) {
            const float f = ex2(*group.map_shared_rank(&jm[i], r) - base);
            l = fmaf(*group.map_shared_rank(&jl[i], r), f, l);
            v = fma4(*group.map_shared_rank(&sh.o(0, i, d), r), f, v);
        }
        put4(out + ((seq * g.n_tok + row.token) * g.n_head + row.head) * D + d, v, l != 0.0f ? 1.0f / l : 0.0f, g.vec);
    }
    group.sync();  // the others read this CTA's shared memory until here
}

// Joins the partials of the items that several CTAs worked on, and writes the zeros of empty sequences. A unit of work is an
// item, or a CTA of the first kernel: the item that it begins and others end. A row has 2^join_shift warps (up to
// kJoinWarps): each takes every so many-th partial, a lane D / 32 dimensions, and they join in shared memory.
// (ws is not __restrict__: the first kernel may still write it until pdl_wait, so its loads are not those of constants.)
template <int D, int ROWS>
__global__ void __launch_bounds__(32 * kJoinWarps) kv_attention_join_kernel(KvView c, Geometry g, float * __restrict__ out, const float * ws) {
    __shared__ int64_t red[kJoinWarps + 2], before[kJoinWarps];
    __shared__ float so[kJoinWarps][D], sm[kJoinWarps], sl[kJoinWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = 1 << g.join_shift;
    const int parts_shift = (ROWS == 8 ? 0 : 1) + g.join_shift, part = (int) (blockIdx.x & ((1 << parts_shift) - 1));  // a unit's CTAs
    const int i = part * (kJoinWarps >> g.join_shift) + (warp >> g.join_shift), sub = warp & (warps - 1);
    const int64_t unit = blockIdx.x >> parts_shift;
    int64_t seq, item;
    int first = 0, last = 0;  // the CTAs that worked on it
    auto zero = [&](int64_t s) {  // before the wait: only the kernels before the first one could still use these rows, and they ended
        const int64_t n = (int64_t) g.n_tok * g.n_head * D;
        for (int64_t d = tid; d < n; d += 32 * kJoinWarps) out[s * n + d] = 0.0f;
    };
    if (g.by_item) {
        int64_t sums[2] = {0, 0};  // the chunks of an item in all sequences, and in those before this one
        seq = unit / g.items;
        item = unit % g.items;
        for (int64_t s = tid; s < g.n_seq; s += 32 * kJoinWarps) {
            const int64_t n = chunks_of(c, s, false);
            sums[0] += n;
            if (s < seq) sums[1] += n;
        }
        sums[0] = warp_sum64(sums[0]);
        sums[1] = warp_sum64(sums[1]);
        if (lane == 0) {
            red[warp] = sums[0];
            before[warp] = sums[1];
        }
        const int64_t chunks = chunks_of(c, seq, false);
        __syncthreads();
        int64_t total = 0, a = 0;
#pragma unroll
        for (int w = 0; w < kJoinWarps; w++) {
            total += red[w];
            a += before[w];
        }
        a = a * g.items + item * chunks;
        const int64_t share = (total * g.items + g.ctas - 1) / g.ctas;
        if (chunks > 0) {
            first = (int) (a / share);
            last = (int) ((a + chunks - 1) / share);
        } else if (item == 0 && part == 0) {
            zero(seq);
        }
    } else {
        if (part == 0)
            for (int64_t s = unit; s < g.n_seq; s += g.units)
                if (kv_len(c, s, false) == 0) zero(s);
        const Place p = find_place<kJoinWarps, true>(c, g, unit, false, red);
        seq = p.seq;
        item = 0;
        if (p.at < p.end) {
            const int64_t chunks = chunks_of(c, seq, false), a = p.end - 1 - (p.end - 1 - p.start) % chunks;
            item = (a - p.start) / chunks;
            if (a >= p.at && a + chunks > p.end) {
                first = (int) unit;
                last = (int) ((a + chunks - 1) / p.share);
            }
        }
    }
    pdl_wait();
    if (first == last) return;  // the same for all threads
    constexpr int kStep = 4;  // partials of a warp in flight
    float v[D / 32] = {}, m = -INFINITY, l = 0.0f;
    for (int k0 = first + sub; k0 <= last; k0 += kStep * warps) {
        float pm[kStep], pl[kStep], po[kStep][D / 32];
#pragma unroll
        for (int n = 0; n < kStep; n++) {
            const int k = k0 + n * warps;
            const float * src = ws + (2 * (int64_t) k + (k == first ? 1 : 0)) * partial_floats(D, ROWS);
            pm[n] = k <= last ? src[ROWS * D + i] : -INFINITY;
            pl[n] = k <= last ? src[ROWS * D + ROWS + i] : 0.0f;
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
    const Row mine = row_of<ROWS>(g, (int) (item / g.tiles), (int) (item % g.tiles), i);
    if (!mine.there) return;
    float top = -INFINITY;
    bool in[kJoinWarps];  // the row's warps
#pragma unroll
    for (int w = 0; w < kJoinWarps; w++) {
        in[w] = w >> g.join_shift == warp >> g.join_shift;
        if (in[w]) top = fmaxf(top, sm[w]);
    }
    const float base = top == -INFINITY ? 0.0f : top;
    float f[kJoinWarps], sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; w++) {
        f[w] = ex2(sm[w] - base);
        if (in[w]) sum = fmaf(sl[w], f[w], sum);
    }
    const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
    float * to = out + ((seq * g.n_tok + mine.token) * g.n_head + mine.head) * D;
    for (int d = 32 * sub + lane; d < D; d += 32 * warps) {
        float o = 0.0f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; w++)
            if (in[w]) o = fmaf(so[w][d], f[w], o);
        to[d] = o * inv;
    }
}

// Calls f with the Shape for a cache's type and head_dim and a key/value head's rows: sixteen rows at a time where there are
// more than eight and the registers hold them (each key and value is then read and converted once for all sixteen).
template <class F>
void with_shape(bool q8, int D, int rows, F f) {
    auto pick = [&](auto type) {
        constexpr bool Q8 = decltype(type)::value;
        const bool two = rows > 8;
        switch (D) {
        case 64: two ? f(Shape<Q8, 64, 2>{}) : f(Shape<Q8, 64, 1>{}); break;
        case 96: two ? f(Shape<Q8, 96, 2>{}) : f(Shape<Q8, 96, 1>{}); break;
        case 128: two ? f(Shape<Q8, 128, 2>{}) : f(Shape<Q8, 128, 1>{}); break;
        default: f(Shape<Q8, 256, 1>{}); break;
        }
    };
    if (q8) pick(std::true_type{});
    else pick(std::false_type{});
}

Geometry geometry(const b200_context * ctx, const b200_kv_cache * c, int64_t max_pages, int64_t n_seq, int64_t n_tok, int64_t n_head) {
    Geometry g = {};
    g.n_tok = (int) n_tok;
    g.n_head = (int) n_head;
    g.group = (int) (n_head / c->n_kv_head);
    with_shape(c->type == B200_TYPE_Q8_0, c->head_dim, g.n_tok * g.group, [&](auto shape) {
        using S = decltype(shape);
        g.rows = S::kRows;
        g.ctas = (int64_t) ctx->num_sms * S::kCtas;
    });
    g.tiles = (g.n_tok * g.group + g.rows - 1) / g.rows;
    g.items = (int64_t) c->n_kv_head * g.tiles;
    g.n_seq = n_seq;
    // By items when the lengths that the table allows are short: the cluster (1 to 8 CTAs) is the largest that all items fit
    // on the GPU with at once. One launch instead of two, and no scan of the lengths, against CTAs with equal work. Measured
    // (F16, 16 and 8 heads of 128, lengths from an eighth of the table's width to all of it), by items and by positions: 1
    // sequence of 512: 5.5 and 6.2 us, 4096: 10.3 and 8.4 (where the second launch costs the host as much again; a captured graph
    // does not pay that); 8 sequences of 1024: 8.8 and 11.0, 4096: 18.3 and 16.2; 64 of 1024: 35.6 and 37.4; 128 of 1024 over
    // Q8_0 48 and 58. The host does not know the lengths, so where few are long the choice loses: one of 1024 among 63 short ones
    // 15.2 and 12.9, among 511 79 and 52. With wider tables that would be 46 and 16 (one of 4096 among 63).
    const int64_t most = (max_pages * c->page_size + kChunk - 1) / kChunk;  // chunks of the longest sequence there can be
    g.cluster = 8;
    while (g.cluster > 1 && n_seq * g.items * g.cluster > g.ctas) g.cluster /= 2;
    if (most > kItemChunks * g.cluster || most > kItemMost) g.cluster = 0;
    if (g.ctas > most * n_seq * g.items) g.ctas = most > 0 ? most * n_seq * g.items : 1;
    // The join has a unit for whatever there are fewer of, and as many warps to a row as make two CTAs per SM: a row of
    // many partials wants many warps (131071 positions, 4 heads: 41 us with eight, 56 with one), but their CTAs take time to
    // start (64 sequences of 512 to 4096, F16: 99.6 us with one warp, 117 with eight). By items alone, 256 sequences of 256 to
    // 2048 would take 198 instead of 193 us, five tokens each 239 instead of 228.
    g.by_item = n_seq * g.items < g.ctas;
    g.units = g.by_item ? n_seq * g.items : g.ctas;
    g.join_shift = 3;
    while (g.join_shift > 0 && g.units * g.rows << g.join_shift > (int64_t) kJoinWarps * 2 * ctx->num_sms) g.join_shift--;
    return g;
}

// ready: the kernels of this shape may use their shared memory on this device (set once per context).
template <class S>
cudaError_t launch(const KvView & c, const Geometry & g, const float * q, int64_t ldq, float scale, float * out, float * ws, cudaStream_t st,
                   bool ready) {
    if (!ready) {
        cudaError_t e = cudaFuncSetAttribute(kv_attention_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kv_attention_item_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (g.cluster) {
        cfg.gridDim = dim3((unsigned) (g.n_seq * g.items * g.cluster), 1, 1);
        cfg.blockDim = dim3(kThreads, 1, 1);
        cfg.dynamicSmemBytes = S::kBytes;
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned) g.cluster;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        return cudaLaunchKernelEx(&cfg, kv_attention_item_kernel<S>, c, g, g.cluster, q, ldq, scale, out);
    }
    kv_attention_kernel<S><<<(unsigned) g.ctas, kThreads, S::kBytes, st>>>(c, g, q, ldq, scale, out, ws);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3((unsigned) ((g.units * g.rows << g.join_shift) / kJoinWarps), 1, 1);
    cfg.blockDim = dim3(32 * kJoinWarps, 1, 1);
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    return cudaLaunchKernelEx(&cfg, kv_attention_join_kernel<S::kDim, S::kRows>, c, g, out, (const float *) ws);
}

size_t workspace_bytes_of(const Geometry & g, int D) { return g.cluster ? 0 : (size_t) (2 * g.ctas * partial_floats(D, g.rows)) * sizeof(float); }

bool fits(const b200_kv_cache * c, int64_t max_pages, int64_t n_seq, int64_t n_tok, int64_t n_head) {
    return c && c->n_kv_head > 0 && c->page_size > 0 && max_pages >= 0 && n_seq > 0 && n_tok > 0 && n_tok <= 16 && n_head > 0 && n_head <= 65535 &&
           n_head % c->n_kv_head == 0 && max_pages <= (1 << 30) / c->page_size && n_seq * n_tok <= INT32_MAX / 16 / n_head;
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
    if (!fits(cache, max_pages, n_seq, n_tok, n_head)) return kv_fail(ctx, B200_ERR_INVALID, what, "n_seq * n_tok * n_head passes 2^27");
    if (ldq < n_head * c.head_dim) return kv_fail(ctx, B200_ERR_INVALID, what, "the row stride is below n_head * head_dim");
    if (!q || !out || ((uintptr_t) q & 3) || ((uintptr_t) out & 3)) return kv_fail(ctx, B200_ERR_INVALID, what, "NULL or misaligned q or out");
    Geometry g = geometry(ctx, cache, max_pages, n_seq, n_tok, n_head);
    g.vec = ((uintptr_t) q & 15) == 0 && ((uintptr_t) out & 15) == 0 && ldq % 4 == 0;
    const size_t need = workspace_bytes_of(g, c.head_dim);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t) workspace & 255)))
        return kv_fail(ctx, B200_ERR_INVALID, what, "the workspace is missing, misaligned or too small");
    DeviceScope scope(ctx->device);
    if (scope.status != cudaSuccess) return kv_cuda(ctx, scope.status, what);
    cudaStream_t st = stream ? (cudaStream_t) stream : ctx->stream;
    const bool q8 = cache->type == B200_TYPE_Q8_0;
    const unsigned bit = 1u << (c.head_dim / 32 + (q8 ? 8 : 0) + (g.rows == 8 ? 0 : 16));
    cudaError_t e = cudaErrorInvalidValue;
    with_shape(q8, c.head_dim, g.n_tok * g.group,
               [&](auto shape) { e = launch<decltype(shape)>(c, g, q, ldq, scale, out, (float *) workspace, st, ctx->kv_shapes & bit); });
    if (e == cudaSuccess) ctx->kv_shapes |= bit;
    return kv_cuda(ctx, e, what);
}

}  // extern "C"
