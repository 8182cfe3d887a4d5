// One step of beam search: the choice of the best continuations of a group's
// beams over the vocabulary, and the reordering of the beams' page tables and
// started KV pages to follow it.
//
// Selection. Beam b of a group has the score s_b and logits x_bv. Its
// continuation by token v scores s_b + (x_bv - lse_b), lse_b = ln sum_v
// e^{x_bv}. Within a beam that order is the order of the logits, so each beam
// offers its n_out largest logits (equal ones: lowest token first) before
// lse_b is known, and the group's n_out best offers win (equal scores: lowest
// beam first, then the beam's own order). HBM-bound: the logits are to be read
// once; sums are kept in fp32.
#include "common.cuh"

namespace {

using namespace qb;

constexpr int MAX_BEAMS = 32;
constexpr int MAX_OUT = 32;
constexpr int SELECT_THREADS = 512;

// A logit as an unsigned key in the order of the values; NaN is taken as -inf
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);   // -0 equals 0
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// (value, lower index first) as one key; distinct for distinct indexes
__device__ __forceinline__ uint64_t offer_key(float x, uint32_t index) {
    return ((uint64_t)order_key(x) << 32) | (0xFFFFFFFFu - index);
}

__device__ __forceinline__ uint64_t warp_max64(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t u = __shfl_xor_sync(0xffffffffu, v, o);
        v = u > v ? u : v;
    }
    return v;
}

template <typename T>
__device__ __forceinline__ float logit(const T* row, int64_t i);
template <>
__device__ __forceinline__ float logit<float>(const float* row, int64_t i) { return row[i]; }
template <>
__device__ __forceinline__ float logit<bf16>(const bf16* row, int64_t i) {
    return __bfloat162float(row[i]);
}

// One block a beam: the row's lse and its n_out largest logits as keys.
template <typename T>
__global__ void __launch_bounds__(SELECT_THREADS)
beam_offers_kernel(const T* __restrict__ logits, int64_t ld, int64_t vocab,
                   const uint8_t* __restrict__ finished, int n_out, float* __restrict__ lse_out,
                   uint64_t* __restrict__ offers) {
    __shared__ uint64_t s_key[SELECT_THREADS / 32];
    __shared__ float scratch[32];
    const int64_t b = blockIdx.x;
    if (finished && finished[b]) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T* row = logits + b * ld;
    uint64_t below = ~0ull;
    float m = -INFINITY;
    for (int r = 0; r < n_out; ++r) {
        uint64_t best = 0;
        for (int64_t i = threadIdx.x; i < vocab; i += SELECT_THREADS) {
            const uint64_t k = offer_key(logit(row, i), (uint32_t)i);
            if (k < below && k > best) best = k;
        }
        best = warp_max64(best);
        __syncthreads();
        if (lane == 0) s_key[warp] = best;
        __syncthreads();
        for (int w = 0; w < SELECT_THREADS / 32; ++w) best = s_key[w] > best ? s_key[w] : best;
        below = best;
        if (r == 0) m = key_value((uint32_t)(best >> 32));
        if (threadIdx.x == 0) offers[b * n_out + r] = best;
    }
    float sum = 0.0f;
    const float ref = m > -INFINITY ? m : 0.0f;
    for (int64_t i = threadIdx.x; i < vocab; i += SELECT_THREADS) sum += expf(logit(row, i) - ref);
    sum = block_sum(sum, scratch);
    if (threadIdx.x == 0) lse_out[b] = m + logf(sum);
}

// One warp a group: the n_out best of its beams' offers.
__global__ void beam_join_kernel(const float* __restrict__ lse, const uint64_t* __restrict__ offers,
                                 const float* __restrict__ scores,
                                 const uint8_t* __restrict__ finished, int beams, int64_t pad,
                                 int n_out, float* __restrict__ scores_out,
                                 int32_t* __restrict__ parent_out,
                                 int64_t* __restrict__ token_out) {
    const int64_t group = blockIdx.x;
    const int lane = threadIdx.x;
    uint64_t below = ~0ull;
    for (int r = 0; r < n_out; ++r) {
        uint64_t best = 0;
        for (int c = lane; c < beams * n_out; c += 32) {
            const int64_t b = group * beams + c / n_out;
            const int rank = c % n_out;
            float s;
            if (finished && finished[b]) {
                s = rank == 0 ? scores[b] : -INFINITY;
            } else {
                const float x = key_value((uint32_t)(offers[b * n_out + rank] >> 32));
                s = scores[b] + (x - lse[b]);
            }
            const uint64_t k = offer_key(s, (uint32_t)c);
            if (k < below && k > best) best = k;
        }
        best = warp_max64(best);
        below = best;
        if (lane == 0) {
            const int c = (int)(0xFFFFFFFFu - (uint32_t)best);
            const int64_t b = group * beams + c / n_out, at = group * n_out + r;
            scores_out[at] = key_value((uint32_t)(best >> 32));
            parent_out[at] = c / n_out;
            token_out[at] = finished && finished[b]
                                ? pad
                                : (int64_t)(0xFFFFFFFFu - (uint32_t)offers[b * n_out + c % n_out]);
        }
    }
}

// ---- reordering -------------------------------------------------------------

constexpr int COPY_THREADS = 256;

// Whose private pages the child `j` takes: its parent's own when it is the
// parent's first child, else those of a beam without children (the e-th such
// child the e-th such beam). All lanes of a warp; parent is lane's own.
__device__ __forceinline__ void plan_child(int parent, int beams, int lane, int& donor,
                                           bool& moved) {
    const uint32_t all = 0xffffffffu;
    const bool live = lane < beams;
    uint32_t same = __match_any_sync(all, live ? parent : -1 - lane);
    moved = live && (same & ((1u << lane) - 1u)) != 0;
    uint32_t children = 0;   // beams that have one
    for (int j = 0; j < beams; ++j) children |= 1u << __shfl_sync(all, parent, j);
    const uint32_t movers = __ballot_sync(all, moved);
    const uint32_t idle = ~children & (beams == 32 ? all : (1u << beams) - 1u);
    const int e = __popc(movers & ((1u << lane) - 1u));
    donor = parent;
    if (moved) donor = __fns(idle, 0, e + 1);
}

// Block (slab, row): block 0 of a row writes its table; each block copies the
// started page's tokens of one slab (a layer's K or V) for a child that moved.
__global__ void __launch_bounds__(COPY_THREADS)
beam_reorder_kernel(const int32_t* __restrict__ parents, const int32_t* __restrict__ used,
                    int beams, const int32_t* __restrict__ table_in, int64_t width,
                    int page_tokens, int64_t n_pages, char* pool, int64_t n_slabs,
                    int64_t row_bytes, char* pool2, int64_t row_bytes2,
                    int32_t* __restrict__ table_out, int64_t* __restrict__ next_row,
                    uint32_t* status) {
    __shared__ int s_parent, s_donor, s_moved;
    const int64_t row = blockIdx.y, group = row / beams, first = group * beams;
    const int child = (int)(row % beams), lane = threadIdx.x;
    if (lane < 32) {
        int parent = lane < beams ? parents[first + lane] : 0;
        const bool bad = parent < 0 || parent >= beams;
        if (bad) parent = lane;   // flagged, and taken as its own parent
        if (bad && blockIdx.x == 0) atomicOr(status, STATUS_BAD_INDEX);
        int donor;
        bool moved;
        plan_child(parent, beams, lane, donor, moved);
        if (lane == child) {
            s_parent = parent;
            s_donor = donor;
            s_moved = moved;
        }
    }
    __syncthreads();
    const int32_t* from = table_in + (first + s_parent) * width;
    const int32_t* own = table_in + (first + s_donor) * width;
    const int n = used[group];
    const int64_t full = n < 0 ? 0 : n / page_tokens;
    if (n < 0 || full > width || (full == width && n % page_tokens)) {
        if (threadIdx.x == 0 && blockIdx.x == 0) {
            atomicOr(status, STATUS_BAD_INDEX);
            if (next_row) next_row[row] = -1;
        }
        if (blockIdx.x == 0)
            for (int64_t i = threadIdx.x; i < width; i += COPY_THREADS)
                table_out[row * width + i] = from[i];
        return;
    }
    const int tail = n % page_tokens;
    if (blockIdx.x == 0) {
        for (int64_t i = threadIdx.x; i < width; i += COPY_THREADS)
            table_out[row * width + i] = i < full ? from[i] : own[i];
        if (next_row && threadIdx.x == 0)
            next_row[row] = full < width ? (int64_t)own[full] * page_tokens + tail : -1;
    }
    if (!s_moved || tail == 0) return;
    const int64_t src = from[full], dst = own[full];
    if (src < 0 || src >= n_pages || dst < 0 || dst >= n_pages) {
        if (threadIdx.x == 0) atomicOr(status, STATUS_BAD_INDEX);
        return;
    }
    for (int64_t slab = blockIdx.x; slab < n_slabs; slab += gridDim.x) {
        const int64_t base = slab * n_pages * page_tokens;
        const char* a = pool + (base + src * page_tokens) * row_bytes;
        char* b = pool + (base + dst * page_tokens) * row_bytes;
        for (int64_t i = threadIdx.x * 16; i < tail * row_bytes; i += COPY_THREADS * 16)
            *reinterpret_cast<uint4*>(b + i) = *reinterpret_cast<const uint4*>(a + i);
        if (pool2) {   // scale bytes: few, and rows of any width
            a = pool2 + (base + src * page_tokens) * row_bytes2;
            b = pool2 + (base + dst * page_tokens) * row_bytes2;
            for (int64_t i = threadIdx.x; i < tail * row_bytes2; i += COPY_THREADS) b[i] = a[i];
        }
    }
}

}  // namespace

extern "C" int qb_beam_select_workspace(int64_t groups, int beams, int64_t vocab, int n_out,
                                        int64_t* bytes) {
    if (!bytes || groups < 0 || beams <= 0 || beams > MAX_BEAMS || n_out <= 0 ||
        n_out > MAX_OUT || vocab < n_out || vocab > 0x7fffffffLL)
        return invalid("qb_beam_select_workspace: bad sizes");
    *bytes = groups * beams * ((int64_t)n_out * 8 + 8);
    return QB_OK;
}

extern "C" int qb_beam_select(const void* logits, int logits_bf16, int64_t logits_ld,
                              int64_t groups, int beams, int64_t vocab, const float* scores,
                              const uint8_t* finished, int64_t pad, int n_out, void* workspace,
                              int64_t workspace_bytes, float* scores_out, int32_t* parent_out,
                              int64_t* token_out, void* stream) {
    const char* who = "qb_beam_select";
    if (beams <= 0 || beams > MAX_BEAMS || n_out <= 0 || n_out > MAX_OUT)
        return invalid("qb_beam_select: 1 to 32 beams and 1 to 32 outputs a group");
    if (groups < 0 || groups * beams > 0x7fffffffLL || vocab < n_out || vocab > 0x7fffffffLL ||
        logits_ld < vocab)
        return invalid("qb_beam_select: vocab must hold n_out tokens and logits_ld the vocab");
    if (groups == 0) return QB_OK;
    if (!logits || !scores || !scores_out || !parent_out || !token_out)
        return invalid("qb_beam_select: NULL tensor");
    int64_t need = 0;
    const int st = qb_beam_select_workspace(groups, beams, vocab, n_out, &need);
    if (st) return st;
    if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
        return invalid("qb_beam_select: the workspace is too small (qb_beam_select_workspace)");
    uint64_t* offers = (uint64_t*)workspace;
    float* lse = (float*)(offers + groups * beams * n_out);
    const unsigned rows = (unsigned)(groups * beams);
    if (logits_bf16)
        beam_offers_kernel<bf16><<<rows, SELECT_THREADS, 0, (cudaStream_t)stream>>>(
            (const bf16*)logits, logits_ld, vocab, finished, n_out, lse, offers);
    else
        beam_offers_kernel<float><<<rows, SELECT_THREADS, 0, (cudaStream_t)stream>>>(
            (const float*)logits, logits_ld, vocab, finished, n_out, lse, offers);
    beam_join_kernel<<<(unsigned)groups, 32, 0, (cudaStream_t)stream>>>(
        lse, offers, scores, finished, beams, pad, n_out, scores_out, parent_out, token_out);
    return launch_status(who);
}

extern "C" int qb_beam_reorder(const int32_t* parents, const int32_t* used, int64_t groups,
                               int beams, const int32_t* table_in, int64_t table_width,
                               int page_tokens, int64_t n_pages, void* pool, int64_t n_slabs,
                               int64_t row_bytes, void* pool2, int64_t row_bytes2,
                               int32_t* table_out, int64_t* next_row, void* stream) {
    const char* who = "qb_beam_reorder";
    if (beams <= 0 || beams > MAX_BEAMS) return invalid("qb_beam_reorder: 1 to 32 beams a group");
    if (groups < 0 || groups * beams > 65535)
        return invalid("qb_beam_reorder: 0 to 65,535 rows");
    if (page_tokens <= 0 || page_tokens > 1024 || n_pages <= 0 || table_width <= 0 ||
        n_slabs < 0)
        return invalid("qb_beam_reorder: bad page, table or slab counts");
    if (n_slabs > 0 && (!pool || row_bytes <= 0 || row_bytes % 16 || !aligned(pool, 16)))
        return invalid("qb_beam_reorder: pool rows must be multiples of 16 bytes, 16-byte aligned");
    if (pool2 && row_bytes2 <= 0) return invalid("qb_beam_reorder: row_bytes2 must be positive");
    if (groups == 0) return QB_OK;
    if (!parents || !used || !table_in || !table_out)
        return invalid("qb_beam_reorder: NULL tensor");
    if (table_in == table_out) return invalid("qb_beam_reorder: table_out must not be table_in");
    uint32_t* status = device_status_ptr();
    if (!status) return launch_status("qb_beam_reorder: status word");
    const int64_t slabs = n_slabs < 1 ? 1 : n_slabs < 1024 ? n_slabs : 1024;
    const dim3 grid((unsigned)slabs, (unsigned)(groups * beams));
    beam_reorder_kernel<<<grid, COPY_THREADS, 0, (cudaStream_t)stream>>>(
        parents, used, beams, table_in, table_width, page_tokens, n_pages, (char*)pool, n_slabs,
        row_bytes, (char*)pool2, row_bytes2, table_out, next_row, status);
    return launch_status(who);
}
