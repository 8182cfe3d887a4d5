// One step of beam search: the choice of the best continuations of a group's
// beams over the vocabulary, and the reordering of the beams' page tables and
// started KV pages to follow it.
//
// Selection. Beam b of a group has the score s_b and logits x_bv. Its
// continuation by token v scores s_b + (x_bv - lse_b), lse_b = ln sum_v
// e^{x_bv}. Within a beam that order is the order of the logits, so each beam
// offers its n_out largest logits (equal ones: lowest token first) before
// lse_b is known, and the group's n_out best offers win (equal scores: lowest
// beam first, then the beam's own order). HBM-bound: the logits are read once,
// each block a run of one beam's; a logit costs a maximum, an exponential and
// an addition in fp32. A block keeps its n_out best so far as sorted keys
// (value, lower token first), and a bar: first the n_out-th largest of the
// first tile's 32 groups' maxima, later the last of the best. Logits that
// pass are put on a list, without a barrier, and the list is ranked after 9, 81,
// ... tiles and at the end: of a run in no order about 8 n_out pass between.
// Where more pass than the list holds (logits that rise along the run, or many
// equal ones), the run is gone through again tile by tile, each thread that has a
// logit which passes putting its best forward, and again, until none does. The
// block that completes its group (a counter) joins the runs and the beams, in an
// order that does not depend on who came last.
//
// Measured on a B200, vocabulary 151,936: 16 groups of 8 beams, bf16 19 us (31%
// of the copy rate), f32 24 us (49%); 4 beams of one group 8.4 us. Of the 19 us,
// the exponentials alone need 4.4 (16 a clock an SM) and reading 6; a block's
// start, its ranking and the join of the group take the latency of about ten
// dependent steps. (64 registers a thread, for 1,024 an SM; 36 bytes are spilled.)
#include "common.cuh"

namespace {

using namespace qb;

constexpr int MAX_BEAMS = 32;
constexpr int MAX_OUT = 32;
constexpr int MAX_ROWS = 65535;        // groups * beams
constexpr int64_t MAX_VOCAB = 1 << 30; // a place and a block's step past it fit 32 bits
constexpr int VECTORS = 4;             // 16-byte vectors of a thread in a tile
// Keys on the list: at least one a thread, and two a thread with the best.
template <int THREADS>
constexpr int list_keys() {
    return THREADS > 512 ? THREADS : 512 - MAX_OUT;
}
constexpr int JOIN_BYTES = 40 * 1024;  // a group's keys in the join
constexpr float LOG2E = 1.44269504088896341f;

// A logit as an unsigned key in the order of the values; NaN is taken as -inf
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);   // -0 equals 0
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t k = (uint32_t)(key >> 32);
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// (value, lower index first) as one key; distinct for distinct indexes, and
// above every number under 2^32
__device__ __forceinline__ uint64_t offer_key(float x, uint32_t index) {
    return ((uint64_t)order_key(x) << 32) | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return 0xFFFFFFFFu - (uint32_t)key; }

__device__ __forceinline__ uint64_t warp_max64(uint64_t v) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
    const uint32_t lo =
        __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
    return ((uint64_t)hi << 32) | lo;
}

// the largest of a warp's values (none is NaN)
__device__ __forceinline__ float redux_max(float x) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float exp_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * LOG2E));
    return r;
}

// A 16-byte vector of logits: how many, all -inf, the largest (NaN passed
// over), the sum of e^(x - ref), and as floats.
template <typename T>
struct Vector;
template <>
struct Vector<float> {
    static constexpr int N = 4;
    static constexpr uint32_t NONE = 0xFF800000u;
    static __device__ __forceinline__ float at(const uint4& v, int i) {
        return __uint_as_float(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w);
    }
    static __device__ __forceinline__ float top(const uint4& v) {
        return fmax3(at(v, 0), at(v, 1), fmaxf(at(v, 2), at(v, 3)));
    }
};
template <>
struct Vector<bf16> {
    static constexpr int N = 8;
    static constexpr uint32_t NONE = 0xFF80FF80u;
    static __device__ __forceinline__ float at(const uint4& v, int i) {
        const uint32_t w = i < 2 ? v.x : i < 4 ? v.y : i < 6 ? v.z : v.w;
        return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
    }
    static __device__ __forceinline__ float top(const uint4& v) {
        const bf162* h = reinterpret_cast<const bf162*>(&v);
        const bf162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(__low2float(m), __high2float(m));
    }
};
// + e^(x - ref) of two logits each, as pairs
template <typename T>
__device__ __forceinline__ void add_exps(const uint4& v, uint64_t ref, uint64_t& sum) {
    const uint64_t scale = f2pack(LOG2E, LOG2E);
#pragma unroll
    for (int i = 0; i < Vector<T>::N; i += 2) {
        float a, b;
        f2unpack(f2mul(f2sub(f2pack(Vector<T>::at(v, i), Vector<T>::at(v, i + 1)), ref), scale),
                 a, b);
        asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
        asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
        sum = f2add(sum, f2pack(a, b));
    }
}
__device__ __forceinline__ float logit(const float* row, int64_t i) { return row[i]; }
__device__ __forceinline__ float logit(const bf16* row, int64_t i) {
    return __bfloat162float(row[i]);
}

struct SelectParams {
    const void* logits;
    int64_t ld, vocab;
    int beams, n_out, splits;
    const float* scores;
    const uint8_t* finished;
    int64_t pad;
    uint32_t* arrived;     // a counter a group, zero between launches
    uint64_t* keys;        // [rows, splits, n_out]
    float2* sums;          // [rows, splits]: the largest logit, sum e^(x - largest)
    float* scores_out;
    int32_t* parent_out;
    int64_t* token_out;
};

// Block (split, row): a run of one beam's logits.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
beam_select_kernel(const SelectParams p) {
    constexpr int VE = Vector<T>::N, TILE = VECTORS * VE * THREADS, LIST = list_keys<THREADS>();
    constexpr int GROUP = THREADS / 32;   // threads of one of 32 groups
    static_assert(MAX_OUT + LIST <= 2 * THREADS, "rank() holds two keys a thread");
    __shared__ uint64_t s_key[MAX_OUT + LIST];   // the best so far, in order; the list
    __shared__ __align__(16) uint32_t s_group[32];
    __shared__ uint32_t s_new;
    __shared__ float s_m[THREADS / 32], s_s[THREADS / 32];
    __shared__ bool s_last;
    __shared__ float s_lse[MAX_BEAMS];
    extern __shared__ uint64_t s_lists[];           // the join's: [beams, splits, n_out]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.y, group = row / p.beams;
    const int split = blockIdx.x, n_out = p.n_out;

    if (!p.finished || !p.finished[row]) {
        const T* x_row = (const T*)p.logits + row * p.ld;
        // single logits up to the first 16-byte boundary, vectors, single ones
        const int off = (int)((uintptr_t)x_row / sizeof(T) % VE);
        const int head = (int)min(p.vocab, (int64_t)(off ? VE - off : 0));
        const int64_t vectors = (p.vocab - head) / VE;
        const int tail = (int)(p.vocab - head - vectors * VE);
        int single = -1;   // this thread's one, in the first tile
        if (split == 0 && tid < head) single = tid;
        if (split == p.splits - 1 && tid >= 32 && tid - 32 < tail)
            single = (int)(p.vocab - tail) + tid - 32;
        const uint4* body = reinterpret_cast<const uint4*>(x_row + head);
        const int v0 = (int)(vectors * split / p.splits) + tid;
        const int v1 = (int)(vectors * (split + 1) / p.splits);
        // the run as tokens
        const int lo = split == 0 ? 0 : head + (v0 - tid) * VE;
        const int hi = split == p.splits - 1 ? (int)p.vocab : head + v1 * VE;
        const float x_single = single >= 0 ? logit(x_row, single) : -INFINITY;

        uint64_t least = 0;   // the last of the n_out best
        // a logit's key where it passes, else 0. Of the logits of -inf (NaN is
        // taken as one) only the run's first n_out places can count: any other has
        // that many before it, equal or better.
        auto passing = [&](float x, int index) -> uint64_t {
            if (!(x > -INFINITY) && index - lo >= n_out) return 0;
            const uint64_t k = offer_key(x, index);
            return k > least ? k : 0;
        };
        auto put_on_list = [&](uint64_t key) {
            if (key == 0) return;
            const uint32_t slot = atomicAdd(&s_new, 1u);
            if (slot < LIST) s_key[n_out + slot] = key;
        };
        // the n_out best of those so far and `fresh` on the list, into their
        // places: a key's place is the number of keys above it, so the order of
        // arrival does not matter (between barriers). `again`: the list is used
        // again, so it is emptied, after every warp has read how long it was.
        auto rank = [&](int fresh, bool again) {
            const int n = n_out + fresh;
            uint64_t mine[2];
            int place[2] = {n_out, n_out};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if (tid + c * THREADS >= n) continue;
                mine[c] = s_key[tid + c * THREADS];
                int above = 0;
#pragma unroll 8
                for (int j = 0; j < n; ++j) above += s_key[j] > mine[c];
                place[c] = above;
            }
            if (again || n > 32)
                __syncthreads();
            else
                __syncwarp();   // one warp holds them all
#pragma unroll
            for (int c = 0; c < 2; ++c)
                if (place[c] < n_out) s_key[place[c]] = mine[c];
            if (again && tid == 0) s_new = 0;
            __syncthreads();
            least = s_key[n_out - 1];
        };
        auto load = [&](uint4 (&raw)[VECTORS], int v) {
#pragma unroll
            for (int i = 0; i < VECTORS; ++i) {
                constexpr uint32_t none = Vector<T>::NONE;
                raw[i] = make_uint4(none, none, none, none);
                if (v + i * THREADS < v1) raw[i] = __ldcs(body + v + i * THREADS);
            }
        };

        if (tid < n_out) s_key[tid] = n_out - tid;   // under every offer
        if (tid == 0) s_new = 0;
        float m = -INFINITY;
        uint64_t sums = 0;    // two
        bool over = false;    // the list did not hold what passed
        uint4 raw[VECTORS], ahead[VECTORS];
        load(ahead, v0);
        int at = v0;
        for (int tile = 0, ranks = 8;; ++tile) {
            // this thread's logits of the tile: vectors at, at + THREADS, ...
#pragma unroll
            for (int i = 0; i < VECTORS; ++i) raw[i] = ahead[i];
            const int next = at + VECTORS * THREADS;
            load(ahead, next);
            // the sum, against the largest so far
            float tops[VECTORS], top = tile == 0 ? fmaxf(x_single, -INFINITY) : -INFINITY;
#pragma unroll
            for (int i = 0; i < VECTORS; ++i) {
                tops[i] = Vector<T>::top(raw[i]);
                top = fmaxf(top, tops[i]);
            }
            if (top > m) {
                const float down = exp_approx(m - top);
                sums = f2mul(sums, f2pack(down, down));
                m = top;
            }
            const float ref = m > -INFINITY ? m : 0.0f;
            if (tile == 0 && single >= 0)
                sums = f2add(sums, f2pack(exp_approx(x_single - ref), 0.0f));
#pragma unroll
            for (int i = 0; i < VECTORS; ++i) add_exps<T>(raw[i], f2pack(ref, ref), sums);

            if (tile == 0) {
                // the n_out-th largest of 32 groups' maxima: that many logits
                // reach it, so nothing under it can be chosen
                const bool some = at < v1 || single >= 0;
                uint32_t mine = some ? order_key(top) : 0u;
#pragma unroll
                for (int o = 1; o < GROUP; o <<= 1)
                    mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
                if (lane % GROUP == 0) s_group[tid / GROUP] = mine;
                __syncthreads();
                mine = s_group[lane];
                int above = 0;
                const uint4* all = reinterpret_cast<const uint4*>(s_group);
#pragma unroll 2
                for (int j = 0; j < 8; ++j) {
                    const uint4 g = all[j];
                    above += (g.x > mine) + (g.y > mine) + (g.z > mine) + (g.w > mine);
                }
                const uint32_t g =
                    __reduce_min_sync(0xffffffffu, above < n_out ? mine : ~0u);
                least = g ? ((uint64_t)g << 32) - 1 : 0;   // (0: a group has no logit)
                if (single >= 0) put_on_list(passing(x_single, single));
            }
            // (a run of -inf only: its first places are in the first tile)
            if (!over && (tile == 0 || order_key(top) >= (uint32_t)(least >> 32))) {
                const float bar = least >> 32 ? key_value(least) : -INFINITY;
                uint32_t found = 0;   // the thread's logits that do; seldom more than one
#pragma unroll
                for (int i = 0; i < VECTORS; ++i)
                    if (at + i * THREADS < v1 && !(tops[i] < bar))
#pragma unroll
                        for (int e = 0; e < VE; ++e)
                            found |= Vector<T>::at(raw[i], e) < bar ? 0u : 1u << (i * VE + e);
                for (; found; found &= found - 1) {
                    const int j = __ffs(found) - 1, i = j / VE;
                    const uint4 v = i == 0 ? raw[0] : i == 1 ? raw[1] : i == 2 ? raw[2] : raw[3];
                    put_on_list(passing(Vector<T>::at(v, j % VE),
                                        head + (at + i * THREADS) * VE + j % VE));
                }
            }
            if (tile == ranks && !over) {
                ranks = 9 * ranks + 8;
                __syncthreads();
                const int fresh = s_new;
                over = fresh > LIST;
                if (!over && fresh)
                    rank(fresh, true);
                else
                    __syncthreads();   // s_new has been read
            }
            at = next;
            if (at - tid >= v1) break;   // (the same for the block)
        }
        __syncthreads();
        const int fresh = s_new;
        if (fresh > LIST) {
            // the sure way: a tile at a time, each thread puts its best forward,
            // in rounds
            __syncthreads();
            if (tid < n_out) s_key[tid] = n_out - tid;
            if (tid == 0) s_new = 0;
            __syncthreads();
            least = 0;
            for (int64_t t0 = lo; t0 < hi; t0 += TILE) {
                const int t1 = (int)min(t0 + TILE, (int64_t)hi);
                for (uint64_t limit = ~0ull;;) {
                    uint64_t key = 0;
                    for (int i = (int)t0 + tid; i < t1; i += THREADS) {
                        const uint64_t k = passing(logit(x_row, i), i);
                        if (k < limit && k > key) key = k;
                    }
                    const int put = __syncthreads_count(key != 0);
                    if (put == 0) break;
                    put_on_list(key);
                    if (key) limit = key;
                    __syncthreads();
                    rank(put, true);
                }
            }
        } else if (fresh) {
            rank(fresh, false);
        }
        // ---- the run's results
        float sum, second;
        f2unpack(sums, sum, second);
        sum += second;
        const float top = redux_max(m);
        const float s = warp_sum(m > -INFINITY ? sum * exp_approx(m - top) : sum);
        if (lane == 0) {
            s_m[warp] = top;
            s_s[warp] = s;
        }
        const int64_t place = row * p.splits + split;
        if (tid < n_out) __stcg(p.keys + place * n_out + tid, s_key[tid]);
        __syncthreads();
        if (warp == 0) {
            const float mine = lane < THREADS / 32 ? s_m[lane] : -INFINITY;
            const float part = lane < THREADS / 32 ? s_s[lane] : 0.0f;
            const float all = redux_max(mine);
            const float t = warp_sum(mine > -INFINITY ? part * exp_approx(mine - all) : part);
            if (lane == 0) __stcg(p.sums + place, make_float2(all, t));
        }
    }
    // ---- the group's last block joins
    __syncthreads();
    if (tid == 0) {
        __threadfence();
        const uint32_t all = (uint32_t)(p.beams * p.splits);
        s_last = atomicAdd(p.arrived + group, 1u) == all - 1;
        if (s_last) p.arrived[group] = 0;   // for the next launch
        __threadfence();
    }
    __syncthreads();
    if (!s_last) return;
    const int64_t row0 = group * p.beams;
    const int list = p.splits * n_out, runs = p.beams * p.splits;
    float2* s_sums = reinterpret_cast<float2*>(s_lists + p.beams * list);
    for (int i = tid; i < p.beams * list; i += THREADS)
        s_lists[i] = __ldcg(p.keys + row0 * list + i);
    for (int i = tid; i < runs; i += THREADS) s_sums[i] = __ldcg(p.sums + row0 * p.splits + i);
    __syncthreads();
    // a beam's offers in order, over its first run's keys, and then its lse: a
    // warp each
    for (int task = warp; task < 2 * p.beams; task += THREADS / 32) {
        const int b = task < p.beams ? task : task - p.beams;
        if (p.finished && p.finished[row0 + b]) continue;
        if (task >= p.beams) {
            const float2* sums = s_sums + b * p.splits;
            float m = -INFINITY;
            for (int i = lane; i < p.splits; i += 32) m = fmaxf(m, sums[i].x);
            m = redux_max(m);
            float sum = 0.0f;
            for (int i = lane; i < p.splits; i += 32)
                sum += sums[i].x > -INFINITY ? sums[i].y * exp_approx(sums[i].x - m) : sums[i].y;
            sum = warp_sum(sum);
            if (lane == 0) s_lse[b] = m + logf(sum);
        } else if (p.splits > 1 && list <= 96) {
            // few keys: the place of each is the number above it (a masked small
            // vocabulary: 9.2 us against 9.8 the other way)
            uint64_t* keys = s_lists + b * list;
            uint64_t mine[3];
            int place[3] = {n_out, n_out, n_out};
#pragma unroll
            for (int c = 0; c < 3; ++c) {
                mine[c] = lane + 32 * c < list ? keys[lane + 32 * c] : 0;
                if (lane + 32 * c < list) place[c] = 0;
            }
#pragma unroll 4
            for (int j = 0; j < list; ++j) {
                const uint64_t other = keys[j];
#pragma unroll
                for (int c = 0; c < 3; ++c) place[c] += other > mine[c];
            }
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 3; ++c)
                if (place[c] < n_out) keys[place[c]] = mine[c];
        } else if (p.splits > 1) {
            // many: the best that is left, n_out times
            uint64_t* keys = s_lists + b * list;
            uint64_t limit = ~0ull, chosen = 0;   // of rank `lane`
            for (int r = 0; r < n_out; ++r) {
                uint64_t best = 0;
                for (int i = lane; i < list; i += 32) {
                    const uint64_t k = keys[i];
                    if (k < limit && k > best) best = k;
                }
                limit = warp_max64(best);
                if (lane == r) chosen = limit;
            }
            __syncwarp();
            if (lane < n_out) keys[lane] = chosen;
        }
    }
    __syncthreads();
    // a thread's beam (a beam a lane for many offers, below)
    const int offers = p.beams * n_out;
    const bool few = offers <= THREADS;
    const int b = few ? tid / n_out : lane;
    const bool live = few ? tid < offers : warp == 0 && lane < p.beams;
    const bool done = live && p.finished && p.finished[row0 + b];
    const float score = live ? p.scores[row0 + b] : 0.0f;
    auto offer = [&](int rank) {
        float s = rank ? -INFINITY : score;   // a finished beam's: itself
        if (!done) s = score + (key_value(s_lists[b * list + rank]) - s_lse[b]);
        return offer_key(s, b * n_out + rank);
    };
    auto write = [&](int place, uint64_t key, int rank) {
        const int64_t at = group * n_out + place;
        p.scores_out[at] = key_value(key);
        p.parent_out[at] = b;
        p.token_out[at] = done ? p.pad : (int64_t)key_index(s_lists[b * list + rank]);
    };
    if (few) {
        // an offer a thread; its place is the number above it (s_key is free)
        const int rank = tid - b * n_out;
        const uint64_t mine = live ? offer(rank) : 0;
        if (live) s_key[tid] = mine;
        __syncthreads();
        if (!live) return;
        int place = 0;
#pragma unroll 8
        for (int j = 0; j < offers; ++j) place += s_key[j] > mine;
        if (place < n_out) write(place, mine, rank);
        return;
    }
    if (warp != 0) return;
    // a beam's next offer a lane; the best of these, n_out times
    int rank = 0;
    uint64_t mine = live ? offer(0) : 0;
    for (int r = 0; r < n_out; ++r) {
        const uint64_t best = warp_max64(mine);
        if (mine == best) {   // (one lane: keys differ)
            write(r, best, rank);
            mine = ++rank < n_out ? offer(rank) : 0;
        }
    }
}

// How a call is cut: threads of a block, and runs of a beam's logits. Blocks of
// 1,024 threads, one an SM, where they fill four fifths of the GPU with runs of
// 16 logits a thread or more (one ranking and one list for four times the
// logits: 16 groups of 8 beams in bf16 19 us against 22); else blocks of 256, four an
// SM in one wave, no run under 16 logits a thread. The group's keys fit the
// join's shared memory.
struct Cut {
    int threads, splits;
};
Cut cut_of(int64_t rows, int beams, int64_t vocab, int n_out) {
    const int64_t most = JOIN_BYTES / 8 / ((int64_t)beams * (n_out + 1));
    const int64_t wide = 148 / rows;
    if (wide >= 1 && wide <= most && rows * wide >= 118 && vocab / wide >= 16 * 1024)
        return {1024, (int)wide};
    const int64_t tiles = (vocab + 16 * 256 - 1) / (16 * 256);
    int64_t splits = 592 / rows;
    splits = splits < tiles ? splits : tiles;
    splits = splits < most ? splits : most;
    return {256, splits < 1 ? 1 : (int)splits};
}

// ---- reordering -------------------------------------------------------------

constexpr int COPY_THREADS = 256;
constexpr int COPY_BATCH = 4;   // slabs whose pieces are in flight together

// Whose private pages the child of each lane takes: its parent's own when it
// is the parent's first child, else those of a beam without children (the
// e-th such child the e-th such beam). All lanes of a warp; parent is the
// lane's own.
__device__ __forceinline__ void plan_child(int parent, int beams, int lane, int& donor,
                                           bool& moved) {
    const uint32_t all = 0xffffffffu, below = (1u << lane) - 1u;
    const bool live = lane < beams;
    const uint32_t same = __match_any_sync(all, live ? parent : -1 - lane);
    moved = live && (same & below) != 0;
    const uint32_t movers = __ballot_sync(all, moved);
    uint32_t idle = ~__reduce_or_sync(all, live ? 1u << parent : 0u);
    donor = parent;
    if (moved) {
        for (int e = __popc(movers & below); e > 0; --e) idle &= idle - 1;
        donor = __ffs(idle) - 1;
    }
}

// Block (share, row): block 0 of a row writes its table; each copies its share
// of the started page's tokens, over all slabs (a layer's K or V), for a child
// that moved. HBM-bound: a moved child's started tokens are read and written
// once. Measured on a B200: 71 of 128 beams moving 5 tokens of 36 layers, 8 heads
// of 128, 20 us, 81% of the copy rate (35 us with a block for each slab, whose
// planning then takes as long as its copy).
__global__ void __launch_bounds__(COPY_THREADS)
beam_reorder_kernel(const int32_t* __restrict__ parents, const int32_t* __restrict__ used,
                    int beams, const int32_t* __restrict__ table_in, int64_t width,
                    int page_tokens, int64_t n_pages, char* pool, int64_t n_slabs,
                    int64_t row_bytes, char* pool2, int64_t row_bytes2,
                    int32_t* __restrict__ table_out, int64_t* __restrict__ next_row,
                    uint32_t* status) {
    const int64_t row = blockIdx.y, group = row / beams, first = group * beams;
    const int child = (int)(row - first), lane = threadIdx.x & 31;
    const bool leader = blockIdx.x == 0 && threadIdx.x == 0;
    const int n = used[group];
    // every warp plans for itself
    int parent = lane < beams ? parents[first + lane] : 0, donor;
    const bool bad = parent < 0 || parent >= beams;
    if (bad) parent = lane;   // flagged, and taken as its own parent
    if (bad && blockIdx.x == 0 && threadIdx.x < 32) atomicOr(status, STATUS_BAD_INDEX);
    bool moved;
    plan_child(parent, beams, lane, donor, moved);
    parent = __shfl_sync(0xffffffffu, parent, child);
    donor = __shfl_sync(0xffffffffu, donor, child);
    moved = __shfl_sync(0xffffffffu, moved, child);

    const int32_t* from = table_in + (first + parent) * width;
    const int32_t* own = table_in + (first + donor) * width;
    const int64_t full = n < 0 ? 0 : n / page_tokens;
    const int tail = n < 0 ? 0 : n % page_tokens;
    const bool fits = n >= 0 && (full < width || (full == width && tail == 0));
    if (leader && !fits) atomicOr(status, STATUS_BAD_INDEX);
    if (blockIdx.x == 0) {
        for (int64_t i = threadIdx.x; i < width; i += COPY_THREADS)
            table_out[row * width + i] = i < full || !fits ? from[i] : own[i];
        if (next_row && threadIdx.x == 0)
            next_row[row] =
                fits && full < width ? (int64_t)own[full] * page_tokens + tail : -1;
    }
    if (!fits || !moved || tail == 0) return;
    const int64_t src = from[full], dst = own[full];
    if (src < 0 || src >= n_pages || dst < 0 || dst >= n_pages) {
        if (leader) atomicOr(status, STATUS_BAD_INDEX);
        return;
    }
    // the slabs share, share + shares, ...; a piece of several at a time
    const int64_t slab_rows = n_pages * page_tokens, slab_bytes = slab_rows * row_bytes;
    const int share = blockIdx.x, shares = gridDim.x, slabs = (int)n_slabs;
    const int pieces = (int)(tail * row_bytes / 16);
    const char* a = pool + src * page_tokens * row_bytes;
    char* b = pool + dst * page_tokens * row_bytes;
    for (int slab0 = share; slab0 < slabs; slab0 += shares * COPY_BATCH)
        for (int i = threadIdx.x; i < pieces; i += COPY_THREADS) {
            uint4 held[COPY_BATCH];
#pragma unroll
            for (int j = 0; j < COPY_BATCH; ++j)
                if (slab0 + j * shares < slabs)
                    held[j] = *reinterpret_cast<const uint4*>(
                        a + (slab0 + j * shares) * slab_bytes + i * 16LL);
#pragma unroll
            for (int j = 0; j < COPY_BATCH; ++j)
                if (slab0 + j * shares < slabs)
                    *reinterpret_cast<uint4*>(b + (slab0 + j * shares) * slab_bytes +
                                              i * 16LL) = held[j];
        }
    if (pool2) {   // scale bytes: few, and rows of any width
        const int64_t bytes = tail * row_bytes2, all = n_slabs * bytes;
        a = pool2 + src * page_tokens * row_bytes2;
        b = pool2 + dst * page_tokens * row_bytes2;
        for (int64_t i = (int64_t)blockIdx.x * COPY_THREADS + threadIdx.x; i < all;
             i += (int64_t)gridDim.x * COPY_THREADS) {
            const int64_t slab = i / bytes;
            const int64_t byte = slab * slab_rows * row_bytes2 + i - slab * bytes;
            b[byte] = a[byte];
        }
    }
}

}  // namespace

extern "C" int qb_beam_select_workspace(int64_t groups, int beams, int64_t vocab, int n_out,
                                        int64_t* bytes) {
    if (!bytes || groups < 0 || beams <= 0 || beams > MAX_BEAMS || groups > MAX_ROWS ||
        groups * beams > MAX_ROWS || n_out <= 0 || n_out > MAX_OUT || vocab < n_out ||
        vocab > MAX_VOCAB)
        return invalid("qb_beam_select_workspace: bad sizes");
    // the counters, always at the same place, then the runs' keys and sums
    *bytes = MAX_ROWS * 4 + 4;
    if (groups)
        *bytes += groups * beams * cut_of(groups * beams, beams, vocab, n_out).splits *
                  ((int64_t)n_out * 8 + 8);
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
    if (groups < 0 || groups > MAX_ROWS || groups * beams > MAX_ROWS || vocab < n_out ||
        vocab > MAX_VOCAB || logits_ld < vocab)
        return invalid("qb_beam_select: at most 65,535 rows and 2^30 tokens, vocab must hold n_out "
                       "tokens and logits_ld the vocab");
    if (groups == 0) return QB_OK;
    if (!logits || !scores || !scores_out || !parent_out || !token_out)
        return invalid("qb_beam_select: NULL tensor");
    if (!aligned(logits, logits_bf16 ? 2 : 4))
        return invalid("qb_beam_select: logits are not aligned to their type");
    int64_t need = 0;
    const int st = qb_beam_select_workspace(groups, beams, vocab, n_out, &need);
    if (st) return st;
    if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
        return invalid("qb_beam_select: the workspace is too small (qb_beam_select_workspace)");
    const int64_t rows = groups * beams;
    SelectParams p;
    p.logits = logits;
    p.ld = logits_ld;
    p.vocab = vocab;
    p.beams = beams;
    p.n_out = n_out;
    const Cut cut = cut_of(rows, beams, vocab, n_out);
    p.splits = cut.splits;
    p.scores = scores;
    p.finished = finished;
    p.pad = pad;
    p.arrived = (uint32_t*)workspace;
    p.keys = (uint64_t*)((char*)workspace + MAX_ROWS * 4 + 4);
    p.sums = (float2*)(p.keys + rows * p.splits * n_out);
    p.scores_out = scores_out;
    p.parent_out = parent_out;
    p.token_out = token_out;
    const dim3 grid((unsigned)p.splits, (unsigned)rows);
    const int bytes = beams * p.splits * (n_out + 1) * 8;
    auto* kernel = logits_bf16 ? (cut.threads == 1024 ? beam_select_kernel<bf16, 1024>
                                                      : beam_select_kernel<bf16, 256>)
                               : (cut.threads == 1024 ? beam_select_kernel<float, 1024>
                                                      : beam_select_kernel<float, 256>);
    kernel<<<grid, cut.threads, bytes, (cudaStream_t)stream>>>(p);
    return launch_status(who);
}

extern "C" int qb_beam_reorder(const int32_t* parents, const int32_t* used, int64_t groups,
                               int beams, const int32_t* table_in, int64_t table_width,
                               int page_tokens, int64_t n_pages, void* pool, int64_t n_slabs,
                               int64_t row_bytes, void* pool2, int64_t row_bytes2,
                               int32_t* table_out, int64_t* next_row, void* stream) {
    const char* who = "qb_beam_reorder";
    if (beams <= 0 || beams > MAX_BEAMS) return invalid("qb_beam_reorder: 1 to 32 beams a group");
    if (groups < 0 || groups > MAX_ROWS || groups * beams > MAX_ROWS)
        return invalid("qb_beam_reorder: 0 to 65,535 rows");
    if (page_tokens <= 0 || page_tokens > 1024 || n_pages <= 0 || table_width <= 0 ||
        table_width > (1 << 30) || n_slabs < 0 || n_slabs > (1 << 20) || row_bytes > (1 << 20))
        return invalid("qb_beam_reorder: bad page, table, slab or row sizes");
    if (n_slabs > 0 && (!pool || row_bytes <= 0 || row_bytes % 16 || !aligned(pool, 16)))
        return invalid("qb_beam_reorder: pool rows must be multiples of 16 bytes, 16-byte aligned");
    if (pool2 && row_bytes2 <= 0) return invalid("qb_beam_reorder: row_bytes2 must be positive");
    if (groups == 0) return QB_OK;
    if (!parents || !used || !table_in || !table_out)
        return invalid("qb_beam_reorder: NULL tensor");
    if (table_in == table_out) return invalid("qb_beam_reorder: table_out must not be table_in");
    uint32_t* status = device_status_ptr();
    if (!status) return launch_status("qb_beam_reorder: status word");
    // shares of a row's slabs: a few waves of blocks, each with a batch where the
    // slabs suffice
    const int64_t rows = groups * beams;
    int64_t shares = 148 * 16 / rows;
    shares = shares < n_slabs ? shares : n_slabs;
    shares = shares < 1 ? 1 : shares;
    const dim3 grid((unsigned)shares, (unsigned)rows);
    beam_reorder_kernel<<<grid, COPY_THREADS, 0, (cudaStream_t)stream>>>(
        parents, used, beams, table_in, table_width, page_tokens, n_pages, (char*)pool, n_slabs,
        row_bytes, (char*)pool2, row_bytes2, table_out, next_row, status);
    return launch_status(who);
}
