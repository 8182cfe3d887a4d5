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
#include "common.cuh"

namespace {

using namespace qb;

constexpr int WARPS = 8;   // rows per block, one warp each

// 2^(b - 127); 0 is the subnormal 2^-127 and 255 NaN
__device__ __forceinline__ float e8m0_float(uint32_t b) {
    if (b == 255u) return __uint_as_float(0x7FFFFFFFu);
    return __uint_as_float(b ? b << 23 : 0x00400000u);
}

// Quantises 8 values of a head held by LANES consecutive lanes (8 each).
template <int LANES>
__device__ __forceinline__ uint2 quant8(const uint4& raw, uint32_t& byte) {
    float x[8];
    bf16x8_to_float(raw, x);
    // integer maximum of the magnitudes' bits: a NaN (above every infinity)
    // is kept, which fmaxf would drop
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1)
        top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top >= 0x7F800000u) {
        byte = 255u;
        return make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu);
    }
    const float scale = ue8m0_scale(__uint_as_float(top));
    byte = __float_as_uint(scale) >> 23;
    const float inv = ue8m0_inverse(scale);
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = fp8x2(x[2 * i] * inv, x[2 * i + 1] * inv);
    return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

template <int D>
__global__ void __launch_bounds__(WARPS * 32)
kv_quant_write_kernel(const bf16* __restrict__ k, const bf16* __restrict__ v, int64_t k_ld,
                      int64_t v_ld, const int64_t* __restrict__ src,
                      const int64_t* __restrict__ dst, int64_t n, int64_t src_rows, int n_kv,
                      uint8_t* __restrict__ k_codes, uint8_t* __restrict__ v_codes,
                      uint8_t* __restrict__ k_scale, uint8_t* __restrict__ v_scale,
                      int64_t pool_rows, uint32_t* status) {
    constexpr int LANES = D / 8;   // lanes a head
    const int lane = threadIdx.x & 31;
    const int64_t i = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
    if (i >= n) return;
    const int64_t d = dst[i], s = src ? src[i] : i;
    if (d < 0) return;   // a row that is not kept
    if (d >= pool_rows || s < 0 || s >= src_rows) {
        if (lane == 0) atomicOr(status, STATUS_BAD_INDEX);
        return;
    }
    const int chunks = n_kv * LANES;
    for (int base = 0; base < chunks; base += 32) {
        const int c = base + lane;
        const bool in = c < chunks;
        uint4 kr = make_uint4(0, 0, 0, 0), vr = kr;
        if (in) {
            kr = *reinterpret_cast<const uint4*>(k + s * k_ld + c * 8);
            vr = *reinterpret_cast<const uint4*>(v + s * v_ld + c * 8);
        }
        uint32_t kb, vb;
        const uint2 kq = quant8<LANES>(kr, kb);
        const uint2 vq = quant8<LANES>(vr, vb);
        if (in) {
            const int64_t at = d * n_kv * D + c * 8;
            *reinterpret_cast<uint2*>(k_codes + at) = kq;
            *reinterpret_cast<uint2*>(v_codes + at) = vq;
            if (c % LANES == 0) {
                k_scale[d * n_kv + c / LANES] = (uint8_t)kb;
                v_scale[d * n_kv + c / LANES] = (uint8_t)vb;
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
__global__ void __launch_bounds__(WARPS * 32)
kv_quant_read_kernel(const uint8_t* __restrict__ k_codes, const uint8_t* __restrict__ v_codes,
                     const uint8_t* __restrict__ k_scale, const uint8_t* __restrict__ v_scale,
                     int64_t pool_rows, const int64_t* __restrict__ src,
                     const int64_t* __restrict__ dst, int64_t n, int n_kv, bf16* __restrict__ k,
                     bf16* __restrict__ v, int64_t k_ld, int64_t v_ld, int64_t out_rows,
                     uint32_t* status) {
    constexpr int LANES = D / 8;
    const int lane = threadIdx.x & 31;
    const int64_t i = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
    if (i >= n) return;
    const int64_t s = src[i], d = dst ? dst[i] : i;
    if (d < 0) return;
    if (d >= out_rows) {
        if (lane == 0) atomicOr(status, STATUS_BAD_INDEX);
        return;
    }
    const bool bad = s < 0 || s >= pool_rows;   // flagged, and zeros written
    if (bad && lane == 0) atomicOr(status, STATUS_BAD_INDEX);
    const int chunks = n_kv * LANES;
    for (int c = lane; c < chunks; c += 32) {
        uint4 ko = make_uint4(0, 0, 0, 0), vo = ko;
        if (!bad) {
            const int64_t at = s * n_kv * D + c * 8, head = s * n_kv + c / LANES;
            ko = dequant8(*reinterpret_cast<const uint2*>(k_codes + at),
                          e8m0_float(k_scale[head]));
            vo = dequant8(*reinterpret_cast<const uint2*>(v_codes + at),
                          e8m0_float(v_scale[head]));
        }
        *reinterpret_cast<uint4*>(k + d * k_ld + c * 8) = ko;
        *reinterpret_cast<uint4*>(v + d * v_ld + c * 8) = vo;
    }
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
    const unsigned blocks = (unsigned)((n + WARPS - 1) / WARPS);
    auto* kernel = head_dim == 128 ? kv_quant_write_kernel<128> : kv_quant_write_kernel<64>;
    kernel<<<blocks, WARPS * 32, 0, (cudaStream_t)stream>>>(
        (const bf16*)k, (const bf16*)v, k_ld, v_ld, src, dst, n, src_rows, n_kv,
        (uint8_t*)k_codes, (uint8_t*)v_codes, k_scale, v_scale, pool_rows, status);
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
    const unsigned blocks = (unsigned)((n + WARPS - 1) / WARPS);
    auto* kernel = head_dim == 128 ? kv_quant_read_kernel<128> : kv_quant_read_kernel<64>;
    kernel<<<blocks, WARPS * 32, 0, (cudaStream_t)stream>>>(
        (const uint8_t*)k_codes, (const uint8_t*)v_codes, k_scale, v_scale, pool_rows, src, dst,
        n, n_kv, (bf16*)k, (bf16*)v, k_ld, v_ld, out_rows, status);
    return launch_status(who);
}
