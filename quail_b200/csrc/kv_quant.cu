// The 8-bit paged KV cache: K and V rows quantised as they are written into
// the pools, and read back as bf16.
//
// A pool row holds one token: n_kv heads of head_dim e4m3 codes, and beside
// them one E8M0 exponent byte per head. The byte b stands for the scale
// 2^(b - 127), the least power of two that brings the head's largest |x| to
// 448 or below (ue8m0_scale, the UE8M0 quantisers' rule), so x / scale is
// exact and the only rounding is the one to e4m3 (to nearest even). A code
// floats itself, so a finer scale than a power of two would not make it more
// precise; one scale per head keeps its multiplication out of the
// attention's inner products. A head that holds an infinity or a NaN gets the
// byte 255 (NaN) and reads back as NaN.
//
// Bound by HBM: 2 head_dim bytes of bf16 and head_dim + 1 of cache a head.
// Measured on a B200, 110,371 rows of 8 heads of 128 (680 MB each way): write
// 112 us, 93% of the copy rate, read 109 us, 95%; 64 rows 2.3 us each.
#include "common.cuh"

namespace {

using namespace qb;

constexpr int THREADS = 256;
// A thread's pieces (8 elements of K and of V each) whose loads are in flight
// together (write, read of a filter chunk: 2 112, 109 us; 1 118, 130; 4 121, 120).
constexpr int BATCH = 2;

// 2^(b - 127); 0 is the subnormal 2^-127 and 255 NaN
__device__ __forceinline__ float e8m0_float(uint32_t b) {
    if (b == 255u) return __uint_as_float(0x7FFFFFFFu);
    return __uint_as_float(b ? b << 23 : 0x00400000u);
}

// the larger of two pairs of unsigned 16-bit numbers
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Quantises 8 values of a head held by LANES consecutive lanes (8 each).
template <int LANES>
__device__ __forceinline__ uint2 quant8(const uint4& raw, uint32_t& byte) {
    // the largest magnitude by its bits, two bf16 at a time; a NaN is above
    // every infinity and so is kept
    constexpr uint32_t ABS = 0x7FFF7FFFu;
    uint32_t top = max_u16x2(max_u16x2(raw.x & ABS, raw.y & ABS),
                            max_u16x2(raw.z & ABS, raw.w & ABS));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1)
        top = max_u16x2(top, __shfl_xor_sync(0xffffffffu, top, o));
    top = max(top << 16, top & 0xFFFF0000u);
    if (top >= 0x7F800000u) {
        byte = 255u;
        return make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu);
    }
    // ue8m0_scale's byte: the largest is f * 2^e with f in [1, 2), and f * 2^e
    // <= 448 * 2^(e - 8) just when f <= 1.75; a bf16 f is 1.75 or differs from
    // it by 2^-7 or more, so no quotient's rounding matters
    top = max(top, __float_as_uint(1e-10f));
    byte = (top >> 23) - 8u + ((top & 0x7FFFFFu) > 0x600000u);
    const float inv = __uint_as_float((254u - byte) << 23);
    const uint64_t by = f2pack(inv, inv);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = bf16x2_float2(w[i]);
        float a, b;
        f2unpack(f2mul(f2pack(x.x, x.y), by), a, b);   // exact
        c[i] = fp8x2(a, b);
    }
    return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

// The pieces of a thread, THREADS apart: each one's row in the block and place
// in the row, without a division a piece.
struct Pieces {
    int row, at, step_row, step_at;
    __device__ __forceinline__ Pieces(int first, int chunks) {
        row = first / chunks;
        at = first - row * chunks;
        step_row = THREADS / chunks;
        step_at = THREADS - step_row * chunks;
    }
    __device__ __forceinline__ void advance(int chunks) {
        row += step_row;
        at += step_at;
        if (at >= chunks) {
            at -= chunks;
            ++row;
        }
    }
};

// A block takes `per_block` rows, each of `chunks` pieces for K and V; a
// thread's pieces are THREADS apart, so LANES neighbouring lanes hold a head.
template <int D>
__global__ void __launch_bounds__(THREADS)
kv_quant_write_kernel(const bf16* __restrict__ k, const bf16* __restrict__ v, int64_t k_ld,
                      int64_t v_ld, const int64_t* __restrict__ src,
                      const int64_t* __restrict__ dst, int64_t n, int64_t src_rows, int n_kv,
                      int chunks, int per_block, uint8_t* __restrict__ k_codes,
                      uint8_t* __restrict__ v_codes, uint8_t* __restrict__ k_scale,
                      uint8_t* __restrict__ v_scale, int64_t pool_rows, uint32_t* status) {
    constexpr int LANES = D / 8;
    const int64_t row0 = (int64_t)blockIdx.x * per_block;
    const int all = (int)min((int64_t)per_block, n - row0) * chunks;
    Pieces next(threadIdx.x, chunks);
    for (int base = threadIdx.x & ~31; base < all; base += THREADS * BATCH) {
        uint4 raw[2][BATCH];
        int64_t to[BATCH];   // the destination row, -1: none
        int at[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            const int64_t row = row0 + next.row;
            const bool in = base + THREADS * j + (int)(threadIdx.x & 31) < all;
            at[j] = next.at;
            next.advance(chunks);
            to[j] = -1;
            raw[0][j] = raw[1][j] = make_uint4(0, 0, 0, 0);
            if (!in) continue;
            const int64_t d = dst[row];
            if (d < 0) continue;   // a row that is not kept
            const int64_t s = src ? src[row] : row;
            if (d >= pool_rows || s < 0 || s >= src_rows) {
                if (at[j] == 0) atomicOr(status, STATUS_BAD_INDEX);
                continue;
            }
            to[j] = d;
            raw[0][j] = *reinterpret_cast<const uint4*>(k + s * k_ld + at[j] * 8);
            raw[1][j] = *reinterpret_cast<const uint4*>(v + s * v_ld + at[j] * 8);
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            if (base + THREADS * j >= all) break;   // (the same for a warp)
            uint32_t kb, vb;
            const uint2 kq = quant8<LANES>(raw[0][j], kb);
            const uint2 vq = quant8<LANES>(raw[1][j], vb);
            if (to[j] < 0) continue;
            const int64_t head = to[j] * n_kv, place = head * D + at[j] * 8;
            *reinterpret_cast<uint2*>(k_codes + place) = kq;
            *reinterpret_cast<uint2*>(v_codes + place) = vq;
            if (at[j] % LANES == 0) {
                k_scale[head + at[j] / LANES] = (uint8_t)kb;
                v_scale[head + at[j] / LANES] = (uint8_t)vb;
            }
        }
    }
}

// 8 codes times their head's scale, as bf16: exact (4 significant bits)
// unless the product leaves bf16's normal range
__device__ __forceinline__ uint4 dequant8(const uint2& codes, float scale) {
    const uint8_t* c = reinterpret_cast<const uint8_t*>(&codes);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = fp8_to_float(c[i]) * scale;
    return float_to_bf16x8(x);
}

template <int D>
__global__ void __launch_bounds__(THREADS)
kv_quant_read_kernel(const uint8_t* __restrict__ k_codes, const uint8_t* __restrict__ v_codes,
                     const uint8_t* __restrict__ k_scale, const uint8_t* __restrict__ v_scale,
                     int64_t pool_rows, const int64_t* __restrict__ src,
                     const int64_t* __restrict__ dst, int64_t n, int n_kv, int chunks,
                     int per_block, bf16* __restrict__ k, bf16* __restrict__ v, int64_t k_ld,
                     int64_t v_ld, int64_t out_rows, uint32_t* status) {
    constexpr int LANES = D / 8;
    const int64_t row0 = (int64_t)blockIdx.x * per_block;
    const int all = (int)min((int64_t)per_block, n - row0) * chunks;
    Pieces next(threadIdx.x, chunks);
    for (int base = threadIdx.x; base < all; base += THREADS * BATCH) {
        uint2 codes[2][BATCH];
        uint32_t bytes[2][BATCH];
        int64_t to[BATCH];   // the output row, -1: none
        int at[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            const int64_t row = row0 + next.row;
            at[j] = next.at;
            next.advance(chunks);
            to[j] = -1;
            codes[0][j] = codes[1][j] = make_uint2(0, 0);
            bytes[0][j] = bytes[1][j] = 127u;
            if (base + THREADS * j >= all) continue;
            const int64_t d = dst ? dst[row] : row;
            if (d < 0) continue;
            const int64_t s = src[row];
            if (d >= out_rows || s < 0 || s >= pool_rows) {
                if (at[j] == 0) atomicOr(status, STATUS_BAD_INDEX);
                to[j] = d < out_rows ? d : -1;   // zeros for a bad source
                continue;
            }
            to[j] = d;
            const int64_t place = s * n_kv * D + at[j] * 8, head = s * n_kv + at[j] / LANES;
            codes[0][j] = *reinterpret_cast<const uint2*>(k_codes + place);
            codes[1][j] = *reinterpret_cast<const uint2*>(v_codes + place);
            bytes[0][j] = k_scale[head];
            bytes[1][j] = v_scale[head];
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            if (to[j] < 0) continue;
            *reinterpret_cast<uint4*>(k + to[j] * k_ld + at[j] * 8) =
                dequant8(codes[0][j], e8m0_float(bytes[0][j]));
            *reinterpret_cast<uint4*>(v + to[j] * v_ld + at[j] * 8) =
                dequant8(codes[1][j], e8m0_float(bytes[1][j]));
        }
    }
}

// Rows of a block: pieces for each thread's batches, but a block for at least
// one row, and (so that few rows still spread over the GPU) no more rows than
// leave about two blocks an SM.
int rows_per_block(int64_t n, int chunks) {
    const int64_t most = THREADS * BATCH * 2 / chunks;
    const int64_t spread = n / 296;
    const int64_t rows = most < spread ? most : spread;
    return rows < 1 ? 1 : (int)rows;
}

int check_cache(const char* who, int64_t n, int n_kv, int head_dim, int64_t k_ld, int64_t v_ld,
                int64_t pool_rows, const void* k, const void* v, const void* k_codes,
                const void* v_codes, const void* k_scale, const void* v_scale) {
    if (head_dim != 64 && head_dim != 128) {
        set_error("%s: head_dim must be 64 or 128", who);
        return QB_ERR_INVALID;
    }
    if (n < 0 || n > 0x7fffffffLL || n_kv <= 0 || n_kv > 1024 || pool_rows < 0) {
        set_error("%s: bad row or head counts", who);
        return QB_ERR_INVALID;
    }
    const int64_t width = (int64_t)n_kv * head_dim;
    if (k_ld < width || v_ld < width || k_ld % 8 || v_ld % 8) {
        set_error("%s: k_ld and v_ld must cover n_kv * head_dim and be multiples of 8", who);
        return QB_ERR_INVALID;
    }
    if (n > 0 && (!k || !v || !k_codes || !v_codes || !k_scale || !v_scale)) {
        set_error("%s: NULL tensor", who);
        return QB_ERR_INVALID;
    }
    if (!aligned(k, 16) || !aligned(v, 16) || !aligned(k_codes, 16) || !aligned(v_codes, 16)) {
        set_error("%s: k, v and the codes must be 16-byte aligned", who);
        return QB_ERR_INVALID;
    }
    return QB_OK;
}

}  // namespace

extern "C" int qb_kv_quant_write(const void* k, const void* v, int64_t k_ld, int64_t v_ld,
                                 const int64_t* src, const int64_t* dst, int64_t n,
                                 int64_t src_rows, int n_kv, int head_dim, void* k_codes,
                                 void* v_codes, uint8_t* k_scale, uint8_t* v_scale,
                                 int64_t pool_rows, void* stream) {
    const char* who = "qb_kv_quant_write";
    int st = check_cache(who, n, n_kv, head_dim, k_ld, v_ld, pool_rows, k, v, k_codes, v_codes,
                         k_scale, v_scale);
    if (st) return st;
    if (n > 0 && !dst) return invalid("qb_kv_quant_write: dst is NULL");
    if (!src && src_rows < n) return invalid("qb_kv_quant_write: fewer source rows than n");
    if (n == 0) return QB_OK;
    uint32_t* status = device_status_ptr();
    if (!status) return launch_status("qb_kv_quant_write: status word");
    const int chunks = n_kv * (head_dim / 8), per_block = rows_per_block(n, chunks);
    const unsigned blocks = (unsigned)((n + per_block - 1) / per_block);
    auto* kernel = head_dim == 128 ? kv_quant_write_kernel<128> : kv_quant_write_kernel<64>;
    kernel<<<blocks, THREADS, 0, (cudaStream_t)stream>>>(
        (const bf16*)k, (const bf16*)v, k_ld, v_ld, src, dst, n, src_rows, n_kv,
        chunks, per_block, (uint8_t*)k_codes, (uint8_t*)v_codes, k_scale, v_scale, pool_rows,
        status);
    return launch_status(who);
}

extern "C" int qb_kv_quant_read(const void* k_codes, const void* v_codes, const uint8_t* k_scale,
                                const uint8_t* v_scale, int64_t pool_rows, const int64_t* src,
                                const int64_t* dst, int64_t n, int n_kv, int head_dim, void* k,
                                void* v, int64_t k_ld, int64_t v_ld, int64_t out_rows,
                                void* stream) {
    const char* who = "qb_kv_quant_read";
    int st = check_cache(who, n, n_kv, head_dim, k_ld, v_ld, pool_rows, k, v, k_codes, v_codes,
                         k_scale, v_scale);
    if (st) return st;
    if (n > 0 && !src) return invalid("qb_kv_quant_read: src is NULL");
    if (!dst && out_rows < n) return invalid("qb_kv_quant_read: fewer output rows than n");
    if (n == 0) return QB_OK;
    uint32_t* status = device_status_ptr();
    if (!status) return launch_status("qb_kv_quant_read: status word");
    const int chunks = n_kv * (head_dim / 8), per_block = rows_per_block(n, chunks);
    const unsigned blocks = (unsigned)((n + per_block - 1) / per_block);
    auto* kernel = head_dim == 128 ? kv_quant_read_kernel<128> : kv_quant_read_kernel<64>;
    kernel<<<blocks, THREADS, 0, (cudaStream_t)stream>>>(
        (const uint8_t*)k_codes, (const uint8_t*)v_codes, k_scale, v_scale, pool_rows, src, dst,
        n, n_kv, chunks, per_block, (bf16*)k, (bf16*)v, k_ld, v_ld, out_rows, status);
    return launch_status(who);
}
