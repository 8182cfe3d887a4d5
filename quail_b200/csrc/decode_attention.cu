// Attention of one new token per row over its paged KV cache (bf16 pools, or
// the 8-bit pools of kv_quant.cu).
//
// For row r and query head h, with j = h / (n_q / n_kv) its KV head and key i
// (i < used[r]) at pool row table[r][i / P] * P + i % P:
//   x_i = q . k_i * softmax_scale * log2(e),  m = max x_i,
//   out = sum 2^(x_i - m) v_i / sum 2^(x_i - m),
//   lse = ln 2 * m + ln sum 2^(x_i - m).
// An 8-bit key is code * 2^kb and value code * 2^vb (one exponent byte per
// row and head): 2^kb multiplies x_i, and vb is added to the exponent of the
// weight that meets the value's codes.
//
// HBM-bound: every K and V element is read once and meets n_q / n_kv query
// heads (4 to 8 here), 4 to 16 flop a byte. The few heads of one KV head are
// the N = 8 columns of mma.sync m16n8k16: S^T = K Q^T with 16 keys as rows,
// then O^T = V^T P^T with 16 of the head's dimensions as rows. tcgen05's
// smallest tile has 64 rows and wants its operands in shared memory by way of
// descriptors; here a lane's 16-byte global loads are the operand fragments
// themselves (the inner dimension's order is free, so each lane takes the
// columns that it loaded), and nothing is staged. (Staged through a ring of
// cp.async copies, two steps ahead, 128 rows of 4k to 16k keys took 1,083 us
// against 693.)
//
// Measured on a B200 (copy rate 6.55 TB/s), 32 query heads over 8 KV heads of
// 128: 128 rows of 8,192 keys 643 us, 6.68 TB/s (8 bit: 341 us, 6.35 TB/s);
// 256 rows of 96 to 2,112 keys 119 us, 87% of the copy rate; one row of 40,960
// keys 37 us, 70%, a quarter of it the start and the join; one row of 37 keys
// 5.3 us. 8 bit, 16 rows of 4k to 16k keys under 64 query heads: 56 us, 72%, some
// 10 us of it the start and the join.
//
// Split and join. The rows' lengths are known on the device only (a captured
// launch serves every step), so the blocks share the work there: an item is
// one row and one tile of 8 query heads, its units are steps of 16 keys, and
// the items' units laid end to end are cut into equal ranges, one for each
// resident block, and a block's range into one for each warp. One line holds all
// heads, item after item; where a head's rows are short (heads of 64, or 8 bit)
// there is a line for each tile of heads, cut alike, if the SMs divide so (8 KV
// heads: 18 blocks each, 4 of 148 left over): blocks next to each other then walk
// the same keys of neighbouring heads, whose rows lie together in memory. 8 KV
// heads of 64, 64 rows of 4k to 16k keys: 180 us against 206, 8 bit 126 against
// 164. 8-bit heads of 128, with prefetches(): 64 long rows 189 us against 217, 256
// of 96 to 2,112 keys 86 against 99, one of 40,960 25.2 against 29.9, 37 of 1
// to 1,031 17.4 against 16.4. bf16 of 128 in one line: 128 long rows 673 us against
// 684. (With lines and prefetches() both 663, but 256 ragged rows 121 against 118
// and 37 rows 15.0 against 13.8.) A warp walks its range alone; items that lie
// within it are finished there, the parts of the others (two a warp at most) meet
// in shared memory at the block's end, and parts of an item that blocks share in
// the workspace: the block that completes the item (a counter per cut) joins its
// parts in the blocks' order, so the result does not depend on who came last.
// Nothing waits. A block's cut that would part a short item, or leave a sliver,
// moves to the item's edge.
#include <cuda_fp16.h>

#include "common.cuh"

namespace {

using namespace qb;

constexpr int HEADS = 8;        // query heads of an item: the MMA's N
constexpr int UNIT_SHIFT = 4;   // a unit of work: 16 keys
constexpr int MIN_UNITS = 8;    // a block's least part of an item that is cut
// Items up to WHOLE_UNITS are not cut, nor, where blocks have fewer than
// SHORT_UNITS each, items up to that: a cut costs a join through the workspace,
// about 3 us, and saves its blocks' steps (one row of 300 tokens, 8 KV heads:
// 10.1 us cut, 8.0 whole; at 32 units some 10 us cases take 13).
constexpr int WHOLE_UNITS = 16, SHORT_UNITS = 28;

// Warps of a block, one block an SM: as many as leave the registers for the
// next step's K and V beside this one's, give or take a few bytes. bf16: 10 (168
// registers; 20 bytes spilled and 28 filled a thread) 689 us for 128 rows of 4k to
// 16k keys, 119 for 256 rows of 96 to 2,112, 36.6 for one of 40,960; 8 (no spill)
// 704, 122 and 37.0; 12 680, 119 and 38.0; 16 spills much (867). 8 bit: 8 (254
// registers), 189 us for 64 long rows, 10 spills (258). Heads of 64: 12 (168
// registers; bf16 16 bytes spilled, 24 filled), bf16 180 us for 64 long rows against
// 184 with 10, 8 bit 126 against 157 with 8, though 37 rows of 0 to 1,031 keys take
// 11.0 against 10.1.
template <int D, bool FP8>
constexpr int warps() {
    return D == 64 ? 12 : FP8 ? 8 : 10;
}

constexpr float LN2 = 0.693147180559945309f;
constexpr float LOG2E = 1.44269504088896341f;

// A part of an item: outputs not yet divided by the sum, per head the
// exponent they are taken against, the sum, and (8 bit) the outputs' own
// exponent.
template <int D>
struct alignas(16) Part {
    float o[HEADS][D];
    float m[HEADS], l[HEADS], mv[HEADS], pad[HEADS];
};

struct Params {
    const bf16* q;
    int64_t q_ld;
    int rows;
    int unit_shift;                   // log2 of the keys of a unit of work
    int n_q, n_kv, group;             // group = n_q / n_kv
    int tiles;                        // ceil(group / HEADS) items share a KV head
    int lines;                        // lines of units (not bf16 of 128): n_kv * tiles, or 1
    const void* k;
    const void* v;
    const uint8_t* k_scale;
    const uint8_t* v_scale;
    int64_t n_pages;
    int page_shift;                   // log2 of the page's tokens
    const int32_t* table;
    int64_t table_width, table_ld;
    const int32_t* used;
    float scale_log2;                 // softmax_scale * log2(e)
    bf16* out;
    int64_t out_ld;
    uint8_t* q_out;
    float* scale_out;
    int64_t scale_ld;
    bool ue8m0;
    float* lse;
    void* parts;                      // two Part<D> a block
    uint32_t* arrived;                // a counter a cut, zero between launches
    uint32_t* status;
};

// Row r's keys, made to fit its table.
__device__ __forceinline__ int row_keys(const Params& p, int r, bool flag) {
    const int n = p.used[r];
    const int most = (int)(p.table_width << p.page_shift);
    if (n >= 0 && n <= most) return n;
    if (flag) atomicOr(p.status, STATUS_BAD_INDEX);
    return n < 0 ? 0 : most;
}

__device__ __forceinline__ int units_of(const Params& p, int keys) {
    return (int)(((int64_t)keys + (1 << p.unit_shift) - 1) >> p.unit_shift);
}

// A place in a line of items' units (which holds under 2^31 of them, by
// the choice of the unit).
struct Place {
    int at;       // the unit
    int row;      // its row
    int before;   // units of one head of the rows before it
};

// Range i of `n` that `total` is cut into begins at i * base + min(i, rest).
struct Cuts {
    int base, rest;
    __device__ __forceinline__ Cuts(int total, int n) : base(total / n) { rest = total - base * n; }
    __device__ __forceinline__ int at(int i) const { return i * base + min(i, rest); }
    // the first range that begins at x or later
    __device__ __forceinline__ int from(int x) const {
        const int wide = rest * (base + 1);
        return x <= wide ? (x + base) / (base + 1) : rest + (x - wide + base - 1) / base;
    }
};

// The cut x moved off items of up to `whole` units and slivers, within the item
// [s, s + n)
__device__ __forceinline__ int settle(int x, int s, int n, int whole) {
    if (n <= whole || x - s < MIN_UNITS) return s;
    return s + n - x < MIN_UNITS ? s + n : x;
}

// 16 (or 8) bytes of the pools: read once, so not kept in L1
__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
__device__ __forceinline__ uint2 load8(const void* p) {
    uint2 r;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];"
                 : "=r"(r.x), "=r"(r.y) : "l"(p));
    return r;
}

__device__ __forceinline__ float log2_approx(float x) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// the largest of a warp's values (NaN passed over)
__device__ __forceinline__ float redux_max(float x) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// four e4m3 codes -> two f16 pairs (codes 0, 1 and 2, 3), exactly
__device__ __forceinline__ void e4m3x4_f16(uint32_t c, uint32_t& a, uint32_t& b) {
    asm("{.reg .b16 l, h; mov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;}"
        : "=r"(a), "=r"(b) : "r"(c));
}

template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
    if (F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
            "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
            "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the 8x8 transpose of a warp's 16-bit matrix (lane: row lane / 4, columns
// 2 (lane % 4) and the next)
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}

__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float2 half2_float2(uint32_t b) {
    return __half22float2(*reinterpret_cast<const __half2*>(&b));
}

// 2^(b - 127) of an exponent byte; 255 is NaN
__device__ __forceinline__ float e8m0_float(uint32_t b) {
    if (b == 255u) return __uint_as_float(0x7FFFFFFFu);
    return __uint_as_float(b ? b << 23 : 0x00400000u);
}

// Whether a step's rows are prefetched to L2, one step before they are loaded. Where
// heads have lines of their own, the lines walk the same keys in step, so each
// prefetches the rows of all heads for its share of a step's keys: memory is
// read 1 KB at a time in place of 128 bytes (8 KV heads, 64 rows of 4k to 16k
// keys 189 us against 216, 81% -> 93% of the copy rate; each line's own rows
// prefetched: 192). Two steps ahead are no better (189 us; one row of 40,960 keys
// 26.3 against 25.2). Heads of 64 lose (139 us against 126).
template <int D, bool FP8>
constexpr bool prefetches() {
    return FP8 && D == 128;
}

// A warp's part of an item in shared memory (the padding keeps the rows of
// neighbouring heads on different banks).
template <int D>
struct alignas(16) Slot {
    float o[HEADS][D + 4];
    float m[HEADS], l[HEADS], mv[HEADS];
    int start;           // the item's first unit, over all items; -1: no part
    int n, row;          // its units and row
    int head0, heads;    // its query heads
    int whole;           // 2: starts the item, 1: ends it
};
static_assert(sizeof(Slot<64>) % 16 == 0 && sizeof(Slot<128>) % 16 == 0,
              "the slots' outputs are read as float4");

// One warp: keys [key0, end) of row `row`, KV head kvh, query heads head0 ..
// head0 + heads - 1; the result to `slot`. prefetched: the key of a step (<< 16)
// and the head whose K and V this lane prefetches (AHEAD).
//
// Lanes: g = lane / 4, t = lane % 4, as the MMA fragments number them.
template <int D, bool FP8>
__device__ __forceinline__ void attend(const Params& p, Slot<D>& slot, int row, int kvh,
                                       int head0, int heads, int key0, int end, int lane,
                                       uint32_t prefetched) {
    constexpr bool AHEAD = prefetches<D, FP8>();
    constexpr int ELEM = FP8 ? 1 : 2;
    constexpr int KC = D * ELEM / 64;            // 16-byte chunks of a K row a lane
    constexpr int VC = FP8 ? 1 : D / 64;         // chunks of a V row a lane
    constexpr int MT = D / 16;                   // 16-row tiles of O^T
    const int g = lane >> 2, t = lane & 3;
    const int32_t* table = p.table + row * p.table_ld;

    // Q as the B fragments of S^T: this lane's columns of head g
    uint32_t qf[D / 8];
    float x_scale[2] = {p.scale_log2, p.scale_log2};   // of heads 2t and 2t + 1
    {
        const bf16* q = p.q + row * p.q_ld + (int64_t)(head0 + g) * D;
        constexpr int QC = D / 32;   // 16-byte chunks of Q a lane
        uint4 raw[QC];
#pragma unroll
        for (int c = 0; c < QC; ++c) {
            // bf16: the K lane's chunks t + 4 c; 8 bit: K chunk t + 4 j holds
            // 16 columns, two chunks of Q
            const int at = FP8 ? 2 * (t + 4 * (c >> 1)) + (c & 1) : t + 4 * c;
            raw[c] = g < heads ? *reinterpret_cast<const uint4*>(q + at * 8)
                               : make_uint4(0, 0, 0, 0);
        }
        if (!FP8) {
#pragma unroll
            for (int c = 0; c < QC; ++c) {
                qf[4 * c] = raw[c].x; qf[4 * c + 1] = raw[c].y;
                qf[4 * c + 2] = raw[c].z; qf[4 * c + 3] = raw[c].w;
            }
        } else {
            // f16 operands: q 2^-e with its largest element in [2^14, 2^15),
            // exact down to 2^-28 of that element
            uint32_t top = 0;
            float x[QC][8];
#pragma unroll
            for (int c = 0; c < QC; ++c) {
                bf16x8_to_float(raw[c], x[c]);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    top = max(top, __float_as_uint(x[c][i]) & 0x7FFFFFFFu);
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            int e = (int)(top >> 23) - 127 - 14;
            if (top >= 0x7F800000u || top == 0) e = 0;
            e = max(e, -100);
            const float down = __uint_as_float((uint32_t)(127 - e) << 23);
            const float up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
            for (int c = 0; c < QC; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    qf[4 * c + i] = half2_bits(x[c][2 * i] * down, x[c][2 * i + 1] * down);
            x_scale[0] *= __shfl_sync(0xffffffffu, up, 8 * t);
            x_scale[1] *= __shfl_sync(0xffffffffu, up, 8 * t + 4);
        }
    }

    // Running state of heads 2t and 2t + 1. ref is the exponent that the
    // weights are taken against: the largest x when it was last raised (0
    // before any), raised only when an x passes it by more than SLACK, so that
    // most steps need one vote and no reduction.
    constexpr float SLACK = FP8 ? 2.0f : 8.0f;
    // 8 bit: weights of the values are taken against the largest x + vb and
    // shifted up, so that f16 holds them to 2^-27 of the largest before they
    // become subnormal (2^(13 + 2) at most)
    constexpr float LIFT = 13.0f;
    const float NEG_INF = __uint_as_float(0xFF800000u);
    float top[2] = {NEG_INF, NEG_INF}, ref[2] = {0.0f, 0.0f}, sum[2] = {0.0f, 0.0f};
    float top_v[2] = {NEG_INF, NEG_INF}, ref_v[2] = {0.0f, 0.0f};
    float o[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;

    // A step: 16 keys of 128 bf16, else 32 (8 bit, D = 128, before the prefetch:
    // 59.4 us for 16 long rows against 61.5 with 16 keys and 12 warps). The
    // pipeline: while a step is computed, the next one's K (as soon as S has
    // consumed the registers), V (after the second product) and, one further, the
    // page ids are on their way. Keys past the end are taken as the last one, with
    // a weight of zero.
    constexpr int UNITS = FP8 || D == 64 ? 2 : 1;
    constexpr int STEP = 16 * UNITS;
    const uint32_t row_bytes = (uint32_t)p.n_kv * (D * ELEM);
    const char* k_lane = (const char*)p.k + kvh * D * ELEM + t * 16;
    const char* v_lane = (const char*)p.v + kvh * D * ELEM + g * (FP8 && D == 64 ? 8 : 16);
    const uint32_t mask = (1u << p.page_shift) - 1u, n_pages = (uint32_t)p.n_pages;

    uint4 kr[UNITS][2][KC], vr[UNITS][4][VC];
    uint32_t kb[UNITS][2], vb[UNITS][2];   // 8 bit: exponent bytes of keys g and g + 8
    // the next step's keys g and g + 8 of each unit: page ids, then pool rows
    uint32_t rows[UNITS][2];
    uint32_t lost = 0, next_lost = 0;      // bit 2u + h: the key's page is out of range
    auto find = [&](int from) {
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int key = min(from + 16 * u + 8 * h + g, end - 1);
                rows[u][h] = (uint32_t)__ldg(table + (key >> p.page_shift));
            }
    };
    auto load_k = [&](int from) {
        next_lost = 0;
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t key = (uint32_t)min(from + 16 * u + 8 * h + g, end - 1);
                const uint32_t id = rows[u][h];
                rows[u][h] = (id << p.page_shift) + (key & mask);
                if (id >= n_pages) {
                    rows[u][h] = 0;
                    next_lost |= 1u << (2 * u + h);
                }
                const char* at = k_lane + (uint64_t)rows[u][h] * row_bytes;
#pragma unroll
                for (int c = 0; c < KC; ++c) kr[u][h][c] = load16(at + 64 * c);
                if (FP8) {
                    const uint64_t head = (uint64_t)rows[u][h] * (uint32_t)p.n_kv + kvh;
                    kb[u][h] = __ldg(p.k_scale + head);
                    vb[u][h] = __ldg(p.v_scale + head);
                }
            }
    };
    // V: keys 2t, 2t + 1 of each half
    auto load_v = [&]() {
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t row =
                    __shfl_sync(0xffffffffu, rows[u][r >> 1], 8 * t + 4 * (r & 1));
                const char* at = v_lane + (uint64_t)row * row_bytes;
#pragma unroll
                for (int c = 0; c < VC; ++c) {
                    if (FP8 && D == 64) {
                        const uint2 w = load8(at);
                        vr[u][r][c] = make_uint4(w.x, w.y, 0, 0);
                    } else {
                        vr[u][r][c] = load16(at + 128 * c);
                    }
                }
            }
        if (__any_sync(0xffffffffu, next_lost)) {   // 0 * NaN is NaN
            if (lane == 0) atomicOr(p.status, STATUS_BAD_INDEX);
#pragma unroll
            for (int u = 0; u < UNITS; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t l =
                        __shfl_sync(0xffffffffu, next_lost, 8 * t + 4 * (r & 1));
                    if (l >> (2 * u + (r >> 1)) & 1)
#pragma unroll
                        for (int c = 0; c < VC; ++c) vr[u][r][c] = make_uint4(0, 0, 0, 0);
                }
        }
    };

    // The page of the lane's prefetched key, and the prefetch, a step later
    uint32_t page = 0;
    auto find_ahead = [&](int from) {
        const int key = min(from + (int)(prefetched >> 16), end - 1);
        if (AHEAD) page = (uint32_t)__ldg(table + (key >> p.page_shift));
    };
    auto prefetch = [&](int from) {
        const int key = from + (int)(prefetched >> 16);
        if (!AHEAD || key >= end || page >= n_pages) return;
        const uint64_t at =
            (uint64_t)((page << p.page_shift) + ((uint32_t)key & mask)) * row_bytes +
            (prefetched & 0xFFFFu) * (D * ELEM);
        asm volatile("prefetch.global.L2 [%0];" ::"l"((const char*)p.k + at));
        asm volatile("prefetch.global.L2 [%0];" ::"l"((const char*)p.v + at));
    };

    find(key0);
    find_ahead(key0 + STEP);
    load_k(key0);
    prefetch(key0 + STEP);
    load_v();
    lost = next_lost;
    find(key0 + STEP);
    find_ahead(key0 + 2 * STEP);
    for (; key0 < end; key0 += STEP) {
        // the scales of keys g and g + 8: a factor, and (values) an exponent,
        // the byte as a float by way of a mantissa
        float by[UNITS][2], more[UNITS][2];
        if (FP8)
#pragma unroll
            for (int u = 0; u < UNITS; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    by[u][h] = e8m0_float(kb[u][h]);
                    more[u][h] = __uint_as_float(0x4B000000u | vb[u][h]) - 8388735.0f;
                    if (vb[u][h] == 255u) more[u][h] = __uint_as_float(0x7FFFFFFFu);
                }
        // ---- S^T: keys g and g + 8, heads 2t and 2t + 1
        float s[UNITS][4];
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[u][i] = 0.0f;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const uint32_t w0[4] = {kr[u][0][c].x, kr[u][0][c].y, kr[u][0][c].z,
                                        kr[u][0][c].w};
                const uint32_t w1[4] = {kr[u][1][c].x, kr[u][1][c].y, kr[u][1][c].z,
                                        kr[u][1][c].w};
                if (FP8) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t a0, a1, a2, a3;
                        e4m3x4_f16(w0[w], a0, a2);
                        e4m3x4_f16(w1[w], a1, a3);
                        mma16816<true>(s[u], a0, a1, a2, a3, qf[8 * c + 2 * w],
                                       qf[8 * c + 2 * w + 1]);
                    }
                } else {
#pragma unroll
                    for (int w = 0; w < 2; ++w)
                        mma16816<false>(s[u], w0[2 * w], w1[2 * w], w0[2 * w + 1], w1[2 * w + 1],
                                        qf[4 * c + 2 * w], qf[4 * c + 2 * w + 1]);
                }
            }
        }
        const uint32_t now_lost = lost;
        // (past the end: the last key again; behind a branch these loads are not
        // moved up: 740 us against 670 for 128 long rows)
        load_k(key0 + STEP);
        prefetch(key0 + 2 * STEP);
        find_ahead(key0 + 3 * STEP);
        // x, and y = x and the value's exponent: [2 * half + head]
        float x[UNITS][4], y[UNITS][4];
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool in =
                    key0 + 16 * u + 8 * h + g < end && !(now_lost >> (2 * u + h) & 1);
                // (a key that is left out has pool row 0's exponent, perhaps a NaN)
                const float plus = FP8 && in ? more[u][h] : 0.0f;
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float z =
                        s[u][2 * h + n] * (FP8 ? by[u][h] * x_scale[n] : x_scale[n]);
                    x[u][2 * h + n] = in ? z : NEG_INF;
                    y[u][2 * h + n] = FP8 ? x[u][2 * h + n] + plus : 0.0f;
                }
            }
        float most[2], most_v[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            most[n] = fmaxf(x[0][n], x[0][2 + n]);
            most_v[n] = fmaxf(y[0][n], y[0][2 + n]);
#pragma unroll
            for (int u = 1; u < UNITS; ++u) {
                most[n] = fmax3(most[n], x[u][n], x[u][2 + n]);
                most_v[n] = fmax3(most_v[n], y[u][n], y[u][2 + n]);
            }
        }
        bool raise = most[0] > top[0] + SLACK || most[1] > top[1] + SLACK;
        if (FP8) raise |= most_v[0] > top_v[0] + SLACK || most_v[1] > top_v[1] + SLACK;
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                float a = fmaxf(top[n], most[n]), b = fmaxf(top_v[n], most_v[n]);
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, off));
                    if (FP8) b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, off));
                }
                float down = 0.0f;
                if (a > NEG_INF) {
                    if (top[n] > NEG_INF) down = exp2_approx(ref[n] - a);
                    ref[n] = a;
                }
                top[n] = a;
                sum[n] *= down;
                if (FP8) {
                    down = 0.0f;
                    if (b > NEG_INF) {
                        if (top_v[n] > NEG_INF) down = exp2_approx(ref_v[n] - b);
                        ref_v[n] = b;
                    }
                    top_v[n] = b;
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    o[i][n] *= down;
                    o[i][2 + n] *= down;
                }
            }
        }
        // ---- O^T += V^T P^T: the weights as B fragments, by a transpose.
        // bf16 keeps 8 bits of a weight and f16 11, so what they drop goes through
        // a second product: 16 and 22 bits. (8 bit with one product: 7% of the
        // outputs round to another bf16 than in 32 bits, with two 0.1%; 64 rows of
        // 4k to 16k keys 187 us against 189. bf16 with three: 0.1% of the outputs
        // against 0.2%, what is left being the order of sums; 256 ragged rows 124 us
        // against 119.)
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = exp2_approx(x[u][i] - ref[i & 1]);
                sum[i & 1] += e;
                w[i] = FP8 ? exp2_approx(y[u][i] - ref_v[i & 1] + LIFT) : e;
            }
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (FP8) {
                    const uint32_t b = half2_bits(w[2 * h], w[2 * h + 1]);
                    const float2 f = half2_float2(b);
                    hi[h] = transpose8(b);
                    lo[h] = transpose8(half2_bits(w[2 * h] - f.x, w[2 * h + 1] - f.y));
                } else {
                    const uint32_t b = bf16x2_bits(w[2 * h], w[2 * h + 1]);
                    const float2 f = bf16x2_float2(b);
                    hi[h] = transpose8(b);
                    lo[h] = transpose8(bf16x2_bits(w[2 * h] - f.x, w[2 * h + 1] - f.y));
                }
            }
#pragma unroll
            for (int c = 0; c < VC; ++c) {
                uint32_t v[4][4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    v[r][0] = vr[u][r][c].x;
                    v[r][1] = vr[u][r][c].y;
                    v[r][2] = vr[u][r][c].z;
                    v[r][3] = vr[u][r][c].w;
                }
#pragma unroll
                for (int i = 0; i < (FP8 && D == 64 ? 2 : 4); ++i) {
                    if (FP8) {
                        // four columns of keys 2t, 2t + 1 (a) and 2t + 8, 2t + 9 (b)
                        const uint32_t a01 = __byte_perm(v[0][i], v[1][i], 0x5140);
                        const uint32_t a23 = __byte_perm(v[0][i], v[1][i], 0x7362);
                        const uint32_t b01 = __byte_perm(v[2][i], v[3][i], 0x5140);
                        const uint32_t b23 = __byte_perm(v[2][i], v[3][i], 0x7362);
                        uint32_t f[8];
                        e4m3x4_f16(a01, f[0], f[1]);
                        e4m3x4_f16(b01, f[2], f[3]);
                        e4m3x4_f16(a23, f[4], f[5]);
                        e4m3x4_f16(b23, f[6], f[7]);
                        mma16816<true>(o[2 * i], f[0], f[1], f[2], f[3], hi[0], hi[1]);
                        mma16816<true>(o[2 * i + 1], f[4], f[5], f[6], f[7], hi[0], hi[1]);
                        mma16816<true>(o[2 * i], f[0], f[1], f[2], f[3], lo[0], lo[1]);
                        mma16816<true>(o[2 * i + 1], f[4], f[5], f[6], f[7], lo[0], lo[1]);
                    } else {
                        const uint32_t a0 = __byte_perm(v[0][i], v[1][i], 0x5410);
                        const uint32_t a1 = __byte_perm(v[0][i], v[1][i], 0x7632);
                        const uint32_t a2 = __byte_perm(v[2][i], v[3][i], 0x5410);
                        const uint32_t a3 = __byte_perm(v[2][i], v[3][i], 0x7632);
                        mma16816<false>(o[4 * c + i], a0, a1, a2, a3, hi[0], hi[1]);
                        mma16816<false>(o[4 * c + i], a0, a1, a2, a3, lo[0], lo[1]);
                    }
                }
            }
        }
        lost = next_lost;
        load_v();
        find(key0 + 2 * STEP);
    }

    // ---- the warp's sums, and its state to shared memory
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1)
            sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], off);
        const int head = 2 * t + n;
        if (g == 0) {
            // (a NaN product leaves a NaN sum and no maximum, a NaN exponent of
            // a value leaves top_v behind: both count as parts)
            slot.m[head] = top[n] > NEG_INF || sum[n] != 0.0f ? ref[n] : NEG_INF;
            slot.l[head] = sum[n];
            slot.mv[head] = top_v[n] > NEG_INF || top[n] > NEG_INF ? ref_v[n] : NEG_INF;
        }
#pragma unroll
        for (int i = 0; i < MT; i += 2) {   // rows g of tile i, g + 8, and of tile i + 1
            const int d = FP8 ? (D / 8) * g + 2 * i : 8 * (g + 8 * (i >> 2)) + 2 * (i & 3);
            *reinterpret_cast<float4*>(&slot.o[head][d]) =
                make_float4(o[i][n], o[i][2 + n], o[i + 1][n], o[i + 1][2 + n]);
        }
    }
}

// Four columns of one head, joined from parts with their own exponents, which
// are brought to the largest.
template <bool FP8>
struct Joined {
    float m, mv, l, acc[4];
    __device__ __forceinline__ Joined() {
        m = mv = __uint_as_float(0xFF800000u);
        l = acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
    }
    // 2^(from - to); nothing has `from` -inf
    static __device__ __forceinline__ float factor(float from, float to) {
        return from > __uint_as_float(0xFF800000u) ? exp2_approx(from - to) : 0.0f;
    }
    // Up to 32 more parts of the head: lane i holds part i's exponents and sum
    // (-inf and 0: no part); then add() takes their columns.
    float f;   // the factor of the lane's part
    __device__ __forceinline__ void begin(float mi, float li, float mvi) {
        const float top = fmaxf(m, redux_max(mi));
        const float a = factor(m, top), b = factor(mi, top);
        l = l * a + warp_sum(li * b);
        m = top;
        float before = a;
        f = b;
        if (FP8) {
            const float top_v = fmaxf(mv, redux_max(mvi));
            before = factor(mv, top_v);
            f = factor(mvi, top_v);
            mv = top_v;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= before;
    }
    __device__ __forceinline__ void add(int lane, const float4& part) {
        const float by = __shfl_sync(0xffffffffu, f, lane);
        acc[0] += part.x * by;
        acc[1] += part.y * by;
        acc[2] += part.z * by;
        acc[3] += part.w * by;
    }
};

// A head's finished columns d4 .. d4 + 3 to the outputs. D = 128: the 32
// lanes of a warp hold one head.
template <int D, bool FP8>
__device__ __forceinline__ void finish(const Params& p, const Joined<FP8>& j, int row, int head,
                                       bool live, int d4) {
    constexpr float LIFT = 13.0f;
    const float NEG_INF = __uint_as_float(0xFF800000u);
    float r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (j.l != 0.0f) {   // a NaN stays one
        float f = __fdividef(1.0f, j.l);
        if (FP8 && j.mv > NEG_INF) f *= exp2f(j.mv - j.m - LIFT);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = j.acc[i] * f;
    }
    if (live) {
        if (p.lse && d4 == 0)
            p.lse[row * (int64_t)p.n_q + head] =
                j.l != 0.0f ? (j.m + log2_approx(j.l)) * LN2 : NEG_INF;
        if (p.out) {
            uint2 b;
            b.x = bf16x2_bits(r[0], r[1]);
            b.y = bf16x2_bits(r[2], r[3]);
            *reinterpret_cast<uint2*>(p.out + row * p.out_ld + (int64_t)head * D + d4) = b;
        }
    }
    if (D == 128 && p.q_out) {
        // o_proj's input: bf16 first, then the head's 128 columns as one
        // quantisation group, as the prefill attention does
        float b[4], amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            b[i] = bf16_round(r[i]);
            amax = fmaxf(amax, fabsf(b[i]));
        }
        amax = redux_max(amax);
        const float scale = p.ue8m0 ? ue8m0_scale(amax) : group_scale(amax);
        const GroupDivider div(scale);
        if (live) {
            const uint32_t lo = fp8x2(div.quant(b[0]), div.quant(b[1]));
            const uint32_t hi = fp8x2(div.quant(b[2]), div.quant(b[3]));
            *reinterpret_cast<uint32_t*>(p.q_out + row * (int64_t)p.n_q * D + head * D + d4) =
                lo | (hi << 16);
            if (d4 == 0) p.scale_out[head * p.scale_ld + row] = scale;
        }
    }
}

template <int D, bool FP8>
__global__ void __launch_bounds__(warps<D, FP8>() * 32, 1)
decode_attention_kernel(const Params p) {
    constexpr int WARPS = warps<D, FP8>();
    constexpr int THREADS = WARPS * 32;
    constexpr int QUADS = D / 4;   // threads of a head in the join
    extern __shared__ __align__(16) char smem[];
    Slot<D>* slots = reinterpret_cast<Slot<D>*>(smem);   // [WARPS][2]: begun before, begun here
    __shared__ int s_scan[WARPS], s_full[WARPS];
    __shared__ int s_upto[THREADS];   // units of one head through each thread's rows
    __shared__ uint32_t s_joins[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // block `block` of the line's `width` ones
    const int lines = D == 64 || FP8 ? p.lines : 1;
    const int line = blockIdx.x % lines, block = blockIdx.x / lines;
    const int width = gridDim.x / lines;
    const int per_row = p.n_kv * p.tiles / lines;   // items of a row in a line
    // piece kvh * 32 + lane of a step's 32 keys by all KV heads (prefetches())
    uint32_t prefetched = 0;
    if (prefetches<D, FP8>() && lines > 1) {
        const uint32_t piece = (uint32_t)(line / p.tiles * 32 + lane);
        prefetched = piece / (uint32_t)p.n_kv << 16 | piece % (uint32_t)p.n_kv;
    }

    // ---- a scan over the rows' units: up to 32 rows by every warp for itself, a
    // row a lane (one short row 5.3 us against 5.9); more by the block, `chunk`
    // rows a thread
    const bool few = p.rows <= 32;
    const int chunk = few ? 1 : (p.rows + THREADS - 1) / THREADS;
    const int r0 = min((few ? lane : tid) * chunk, p.rows), r1 = min(r0 + chunk, p.rows);
    int upto = 0, full = 0;
    for (int r = r0; r < r1; ++r) {
        const int n = units_of(p, row_keys(p, r, blockIdx.x == 0));
        upto += n;
        full += n > 0;
    }
    const int own = upto;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
    }
    full = __reduce_add_sync(0xffffffffu, full);
    if (lane < 2) slots[2 * warp + lane].start = -1;
    int units = __shfl_sync(0xffffffffu, upto, 31);
    if (!few) {
        s_upto[tid] = upto;
        if (lane == 31) {
            s_scan[warp] = upto;
            s_full[warp] = full;
        }
        __syncthreads();
        units = full = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            units += s_scan[w];
            full += s_full[w];
        }
    }
    const int total = units * per_row;
    // rows without keys
    if (full < p.rows)
        for (int r = blockIdx.x; r < p.rows; r += gridDim.x) {
            if (row_keys(p, r, false) != 0) continue;
            const Joined<FP8> none;
            for (int i = tid; i < p.n_q * QUADS; i += THREADS)
                finish<D, FP8>(p, none, r, i / QUADS, true, i % QUADS * 4);
        }
    // a block an item where the items are short, and no block under MIN_UNITS
    // of a long one
    const int blocks = min(width, max(full * per_row, total / MIN_UNITS));
    if (block >= blocks) return;

    // ---- this block's range and this warp's share, each warp for itself: the
    // places of its two cuts and of the warp's first unit. The threads whose
    // rows end at x or before are counted, then the next one's rows walked.
    const Cuts cuts(total, blocks);
    const int whole_units = cuts.base < SHORT_UNITS ? SHORT_UNITS : WHOLE_UNITS;
    int lo = 0, hi = total, end = total, n = 0;
    Place at = {0, 0, 0};
#pragma unroll 1
    for (int c = 0; c < 3; ++c) {
        if (c == 1 && block + 1 == blocks) continue;
        if (c == 2) {
            // (heads of 64: whole steps of 32 keys, 11.0 us for the 37 rows
            // against 12.1; 8 bit of 128: 22.0 us for 64 rows of 300 keys against 21.2)
            constexpr int WHOLE = D == 64 ? 2 : 1;
            const Cuts shares((hi - lo + WHOLE - 1) / WHOLE, WARPS);
            end = min(lo + shares.at(warp + 1) * WHOLE, hi);
            at.at = min(lo + shares.at(warp) * WHOLE, end);
            if (at.at == end) break;
        } else {
            at.at = cuts.at(block + c);
        }
        if (few) {
            at.row = __popc(__ballot_sync(0xffffffffu, upto * per_row <= at.at));
            at.before = __shfl_sync(0xffffffffu, upto - own, at.row);
            n = __shfl_sync(0xffffffffu, own, at.row);
        } else {
            int ended = 0, earlier = 0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                ended += (earlier + s_upto[32 * w + lane]) * per_row <= at.at;
                earlier += s_scan[w];
            }
            ended = __reduce_add_sync(0xffffffffu, ended);
            at.row = ended * chunk;
            at.before = ended ? s_upto[ended - 1] : 0;
#pragma unroll
            for (int w = 0; w < WARPS - 1; ++w)
                if (w < (ended - 1) >> 5) at.before += s_scan[w];
            for (;; ++at.row) {
                n = units_of(p, row_keys(p, at.row, false));
                if (at.at < (at.before + n) * per_row) break;
                at.before += n;
            }
        }
        if (c < 2) {
            const int s = at.before * per_row;
            (c ? hi : lo) = settle(at.at, s + (at.at - s) / n * n, n, whole_units);
        }
    }

    // ---- this warp's range, an item after another
    if (at.at < end) {
        int keys = row_keys(p, at.row, false);
        for (;;) {
            const int nth = (at.at - at.before * per_row) / n, item = nth + line;
            const int s = at.before * per_row + nth * n;
            const int stop = min(end, s + n);
            const int kvh = item / p.tiles, tile = item % p.tiles;
            const int head0 = kvh * p.group + tile * HEADS;
            const int heads = min(HEADS, p.group - tile * HEADS);
            if (lines == 1) prefetched = (uint32_t)lane << 16 | (uint32_t)kvh;
            const int whole = 2 * (at.at == s) + (stop == s + n);
            Slot<D>& slot = slots[2 * warp + (at.at == s)];
            attend<D, FP8>(p, slot, at.row, kvh, head0, heads, (at.at - s) << p.unit_shift,
                           (int)min((int64_t)keys, (int64_t)(stop - s) << p.unit_shift), lane,
                           prefetched);
            __syncwarp();
            if (whole == 3) {
                for (int i = lane; i < HEADS * QUADS; i += 32) {
                    const int head = i / QUADS, d4 = i % QUADS * 4;
                    if (D == 128 && head >= heads) break;   // D = 64: two heads at a time
                    Joined<FP8> j;
                    j.m = slot.m[head];
                    j.l = slot.l[head];
                    j.mv = slot.mv[head];
#pragma unroll
                    for (int e = 0; e < 4; ++e) j.acc[e] = slot.o[head][d4 + e];
                    finish<D, FP8>(p, j, at.row, head0 + head, head < heads, d4);
                }
            } else if (lane == 0) {
                slot.start = s;
                slot.n = n;
                slot.row = at.row;
                slot.head0 = head0;
                slot.heads = heads;
                slot.whole = whole;
            }
            __syncwarp();
            at.at = stop;
            if (stop >= end) break;
            while (stop >= (at.before + n) * per_row) {
                at.before += n;
                ++at.row;
                keys = row_keys(p, at.row, false);
                n = units_of(p, keys);
            }
        }
    }
    __syncthreads();

    // ---- the parts that warps share, in order: a chain of parts an item, a
    // warp for each chain and head
    const float NEG_INF = __uint_as_float(0xFF800000u);
    const float4 zeros = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int d4 = lane % QUADS * 4;
    const bool have = lane < QUADS;   // D = 64: half of the lanes have columns
    const int start = lane < 2 * WARPS ? slots[lane].start : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, start);
    const bool leads = start >= 0 && (same & ((1u << lane) - 1u)) == 0;
    bool parted = false;   // the chain is not its whole item
    if (leads) parted = !(slots[lane].whole & 2) || !(slots[31 - __clz(same)].whole & 1);
    uint32_t chains = __ballot_sync(0xffffffffu, leads);
    const uint32_t open = __ballot_sync(0xffffffffu, parted);   // two at most
    // a block of the line's part of an item that it begins (1) or that began before
    auto part_of = [&](int b, int begins) -> Part<D>& {
        return ((Part<D>*)p.parts)[2 * (b * lines + line) + begins];
    };
    for (int head = warp; chains; head -= HEADS, chains &= chains - 1) {
        const int lead = __ffs(chains) - 1;
        const uint32_t chain = __shfl_sync(0xffffffffu, same, lead);
        for (; head < HEADS; head += WARPS) {
            Joined<FP8> j;
            const bool mine = chain >> lane & 1;
            j.begin(mine ? slots[lane].m[head] : NEG_INF, mine ? slots[lane].l[head] : 0.0f,
                    mine ? slots[lane].mv[head] : NEG_INF);
            for (uint32_t c = chain; c; c &= c - 1) {
                const int i = __ffs(c) - 1;
                j.add(i, *reinterpret_cast<const float4*>(&slots[i].o[head][d4]));
            }
            const Slot<D>& slot = slots[lead];
            if (open >> lead & 1) {
                Part<D>& part = part_of(block, slot.whole >> 1);
                if (have)
                    __stcg(reinterpret_cast<float4*>(&part.o[head][d4]),
                           make_float4(j.acc[0], j.acc[1], j.acc[2], j.acc[3]));
                if (lane == 0) {
                    __stcg(&part.m[head], j.m);
                    __stcg(&part.l[head], j.l);
                    __stcg(&part.mv[head], j.mv);
                }
            } else if (have) {
                finish<D, FP8>(p, j, slot.row, slot.head0 + head, head < slot.heads, d4);
            }
        }
    }
    if (!open) return;

    // ---- the parts that blocks share: the last to arrive joins them
    auto sharers = [&](const Slot<D>& slot, int& first, int& last) {   // the cuts inside the item
        first = cuts.from(slot.start + MIN_UNITS);
        last = cuts.from(slot.start + slot.n - MIN_UNITS + 1) - 1;
    };
    const bool counts = tid < __popc(open);
    int first = 0, last = 0;
    if (counts) sharers(slots[__ffs(tid == 0 ? open : open & (open - 1)) - 1], first, last);
    __syncthreads();
    if (counts) {
        __threadfence();   // the block's parts, before the count
        const uint32_t others = atomicAdd(p.arrived + first * lines + line, 1u);
        const bool all = others == (uint32_t)(last - first + 1);
        if (all) p.arrived[first * lines + line] = 0;   // for the next launch
        __threadfence();   // the count, before the others' parts
        s_joins[tid] = all;
    }
    __syncthreads();
    uint32_t which = open;
    for (int k = 0; which; ++k, which &= which - 1) {
        if (!s_joins[k]) continue;
        const Slot<D>& slot = slots[__ffs(which) - 1];
        sharers(slot, first, last);
        for (int head = warp; head < HEADS; head += WARPS) {
            Joined<FP8> j;
            for (int b = first - 1; b <= last; b += 32) {   // a part a lane
                const int mine = b + lane;
                const bool in = mine <= last;
                const Part<D>& part = part_of(min(mine, last), mine == first - 1);
                const float m = in ? __ldcg(&part.m[head]) : NEG_INF;
                const float l = in ? __ldcg(&part.l[head]) : 0.0f;
                const float mv = in ? __ldcg(&part.mv[head]) : NEG_INF;
                constexpr int BATCH = 16;   // parts whose columns are in flight together
                static_assert(32 % BATCH == 0, "a batch lies within the lanes' 32 parts");
                float4 o[BATCH];
                auto fetch = [&](int i) {
#pragma unroll
                    for (int u = 0; u < BATCH; ++u) {
                        const int at = b + i + u;
                        o[u] = at <= last ? __ldcg(reinterpret_cast<const float4*>(
                                                &part_of(at, at == first - 1).o[head][d4]))
                                          : zeros;
                    }
                };
                fetch(0);
                j.begin(m, l, mv);
                for (int i = 0; i < 32 && b + i <= last; i += BATCH) {
                    if (i) fetch(i);
#pragma unroll
                    for (int u = 0; u < BATCH; ++u) j.add(i + u, o[u]);
                }
            }
            if (have)
                finish<D, FP8>(p, j, slot.row, slot.head0 + head, head < slot.heads, d4);
        }
    }
}

template <int D, bool FP8>
int launch(const Params& p, int blocks, cudaStream_t stream) {
    static std::atomic<bool> done[MAX_DEVICES];
    constexpr int bytes = 2 * warps<D, FP8>() * sizeof(Slot<D>);
    if (!set_smem_once(done, decode_attention_kernel<D, FP8>, bytes))
        return launch_status("qb_decode_attention: shared memory");
    decode_attention_kernel<D, FP8><<<blocks, warps<D, FP8>() * 32, bytes, stream>>>(p);
    return launch_status("qb_decode_attention");
}

// Resident blocks of the current device (0: the query failed).
int resident_blocks() {
    static std::atomic<int> cache[MAX_DEVICES];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES) return 0;
    int n = cache[dev].load(std::memory_order_acquire);
    if (n == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
            return 0;
        cache[dev].store(n, std::memory_order_release);
    }
    return n;
}

int64_t workspace_bytes(int blocks) {
    // (a line's counters go up to its blocks, and there are at most `blocks` lines)
    return (int64_t)blocks * 2 * sizeof(Part<128>) + 2 * blocks * (int64_t)sizeof(uint32_t);
}

}  // namespace

extern "C" int qb_decode_attention_workspace(int64_t* bytes) {
    if (!bytes) return invalid("qb_decode_attention_workspace: bytes is NULL");
    const int blocks = resident_blocks();
    if (!blocks) return launch_status("qb_decode_attention_workspace");
    *bytes = workspace_bytes(blocks);
    return QB_OK;
}

extern "C" int qb_decode_attention(const void* q, int64_t q_ld, int64_t rows, int n_q, int n_kv,
                                   int head_dim, const void* k_pool, const void* v_pool,
                                   const uint8_t* k_scale, const uint8_t* v_scale,
                                   int64_t n_pages, int page_tokens, const int32_t* table,
                                   int64_t table_width, int64_t table_ld, const int32_t* used,
                                   float softmax_scale, void* workspace, int64_t workspace_size,
                                   void* out, int64_t out_ld, void* q_out, float* scale_out,
                                   int64_t scale_ld, int ue8m0, float* lse_out, void* stream) {
    const char* who = "qb_decode_attention";
    if (head_dim != 64 && head_dim != 128)
        return invalid("qb_decode_attention: head_dim must be 64 or 128");
    if (n_q <= 0 || n_q > 4096 || n_kv <= 0 || n_q % n_kv)
        return invalid("qb_decode_attention: n_q must be a positive multiple of n_kv, at most "
                       "4096");
    if (rows < 0 || rows > 65535) return invalid("qb_decode_attention: 0 to 65,535 rows");
    if (page_tokens < 8 || page_tokens > 1024 || (page_tokens & (page_tokens - 1)))
        return invalid("qb_decode_attention: page_tokens must be a power of two from 8 to 1024");
    const int64_t width = (int64_t)n_q * head_dim;
    if (q_ld < width || q_ld % 8 || !aligned(q, 16))
        return invalid("qb_decode_attention: q needs 16-byte alignment and q_ld a multiple of 8 "
                       "that covers the heads");
    if (rows > 0 && !out && !q_out) return invalid("qb_decode_attention: no output");
    if (out && (out_ld < width || out_ld % 4 || !aligned(out, 8)))
        return invalid("qb_decode_attention: out needs 8-byte alignment and out_ld a multiple "
                       "of 4 that covers the heads");
    if (q_out && (head_dim != 128 || !scale_out || scale_ld < rows || !aligned(q_out, 4)))
        return invalid("qb_decode_attention: the fp8 output needs head_dim 128, scale_out and "
                       "scale_ld >= rows");
    if (rows == 0) return QB_OK;
    if (!q || !k_pool || !v_pool || !table || !used)
        return invalid("qb_decode_attention: NULL tensor");
    if ((k_scale == nullptr) != (v_scale == nullptr))
        return invalid("qb_decode_attention: k_scale and v_scale go together");
    if (!aligned(k_pool, 16) || !aligned(v_pool, 16))
        return invalid("qb_decode_attention: the pools must be 16-byte aligned");
    if (n_pages <= 0 || table_width <= 0 || table_ld < table_width ||
        table_width > (1 << 30) / page_tokens)
        return invalid("qb_decode_attention: bad table width or page count");
    if (n_pages >= (1LL << 31) || n_pages * page_tokens >= (1LL << 32))
        return invalid("qb_decode_attention: the pools have 2^32 rows or more");
    if (!workspace || !aligned(workspace, 16))
        return invalid("qb_decode_attention: the workspace must be 16-byte aligned");
    const int blocks = resident_blocks();
    if (!blocks) return launch_status(who);
    if (workspace_size < workspace_bytes(blocks))
        return invalid("qb_decode_attention: the workspace is too small "
                       "(qb_decode_attention_workspace)");
    Params p;
    p.q = (const bf16*)q;
    p.q_ld = q_ld;
    p.rows = (int)rows;
    p.n_q = n_q;
    p.n_kv = n_kv;
    p.group = n_q / n_kv;
    p.tiles = (p.group + HEADS - 1) / HEADS;
    p.k = k_pool;
    p.v = v_pool;
    p.k_scale = k_scale;
    p.v_scale = v_scale;
    p.n_pages = n_pages;
    p.page_shift = __builtin_ctz((unsigned)page_tokens);
    // a line for each tile of heads, where they take nine tenths of the blocks
    const int heads = n_kv * p.tiles;
    p.lines = blocks / heads * heads * 10 >= blocks * 9 ? heads : 1;
    // a line's units, and what is added to a place in it, below 2^31
    p.unit_shift = UNIT_SHIFT;
    while (rows * n_kv * p.tiles * ((table_width * page_tokens >> p.unit_shift) + 1) >= 1LL << 30)
        ++p.unit_shift;
    p.table = table;
    p.table_width = table_width;
    p.table_ld = table_ld;
    p.used = used;
    p.scale_log2 = softmax_scale * LOG2E;
    p.out = (bf16*)out;
    p.out_ld = out_ld;
    p.q_out = (uint8_t*)q_out;
    p.scale_out = scale_out;
    p.scale_ld = scale_ld;
    p.ue8m0 = ue8m0 != 0;
    p.lse = lse_out;
    p.status = device_status_ptr();
    if (!p.status) return launch_status("qb_decode_attention: status word");
    p.parts = workspace;
    p.arrived = (uint32_t*)((char*)workspace + (int64_t)blocks * 2 * sizeof(Part<128>));
    const cudaStream_t st = (cudaStream_t)stream;
    if (head_dim == 128)
        return k_scale ? launch<128, true>(p, blocks, st) : launch<128, false>(p, blocks, st);
    return k_scale ? launch<64, true>(p, blocks, st) : launch<64, false>(p, blocks, st);
}
