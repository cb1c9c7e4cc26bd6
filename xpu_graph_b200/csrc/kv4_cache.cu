// Keys and values in 4 bits: quantising new tokens into cache pages, reading tokens back, copying pages (the layout: kv4_tile.cuh). All
// three move bytes, so HBM is their floor. What bounds them now: a prompt's append and read are held up by issuing (65 and 70 % of the
// slots at 28 and 19 % of DRAM; most of it is addresses and what every lane of a group does for the group), few tokens by the host,
// page copies by the launches and their gaps.
//
// Quantising, per token, head and group of 64 channels: least = fp16(min x), scale = fp16(max(max x - least, 0) * fp32(1/15)),
// code = rint((x - least) / scale) in 0..15 (0 where the scale is 0), every step in fp32 with IEEE rounding. The fp16 roundings of the
// pair come first, so the codes are the nearest ones for the pair that is stored. (A least value that is rounded up beyond the largest
// one has no range: a scale below 0 would be one that the attention, which bounds its weights by the scales, does not expect.)
#include "kv4_tile.cuh"
#include "sm100_ptx.cuh"

namespace xg {
namespace {

using namespace kv4;

struct TokenParams {
    Cache cache;
    const void* k;        // append: values in; read: null
    const void* v;
    void* k_out;          // read: values out, [tokens, heads, D]
    void* v_out;
    const int64_t* slots;
    int64_t tokens;
    int64_t k_st, k_sh, v_st, v_sh;
};

// 8 consecutive values as they are stored
template <typename T>
struct Raw8 {
    T v[8];
};
template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
    Raw8<T> r;
    if (VEC) {
        constexpr int N = Vec16<T>::N;
#pragma unroll
        for (int i = 0; i < 8; i += N) *reinterpret_cast<Vec16<T>*>(r.v + i) = ld16_stream(p + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = p[i];
    }
    return r;
}

// Least (NaN where there is one) and largest of 8 values.
__device__ __forceinline__ void extremes(const Raw8<float>& x, float& lo, float& hi) {
    lo = hi = x.v[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        lo = min_nan(lo, x.v[i]);
        hi = fmaxf(hi, x.v[i]);
    }
}
template <typename T, typename T2>
__device__ __forceinline__ void extremes_packed(const Raw8<T>& x, float& lo, float& hi) {
    const T2* u = reinterpret_cast<const T2*>(x.v);
    const T2 a = __hmin2_nan(__hmin2_nan(u[0], u[1]), __hmin2_nan(u[2], u[3])), b = __hmax2(__hmax2(u[0], u[1]), __hmax2(u[2], u[3]));
    lo = min_nan(Cvt<T>::to_f(a.x), Cvt<T>::to_f(a.y));
    hi = fmaxf(Cvt<T>::to_f(b.x), Cvt<T>::to_f(b.y));
}
__device__ __forceinline__ void extremes(const Raw8<__nv_bfloat16>& x, float& lo, float& hi) { extremes_packed<__nv_bfloat16, __nv_bfloat162>(x, lo, hi); }
__device__ __forceinline__ void extremes(const Raw8<__half>& x, float& lo, float& hi) { extremes_packed<__half, __half2>(x, lo, hi); }

// 4 lanes hold a group's 64 channels: this lane's codes as two words, and the group's pair (scale in the low half). A group with a NaN
// has a NaN least value and reads back as NaN.
//
// The quotients come from one correctly rounded reciprocal and a step of correction with an exact remainder, which gives the correctly
// rounded quotient (Markstein, IBM J. Res. Dev. 34, 1990): three operations each in place of a division. Codes are gathered four at a
// time in a float, off the logic pipe, and everything goes in pairs. What bounds it is issuing (65 % of the slots). 16384 tokens x 8
// heads x 128 in bf16: divisions 63 us, one by one 30 us, this 28.5 us (3.0 TB/s).
template <typename T>
__device__ __forceinline__ void quantise(const Raw8<T> (&x)[2], uint32_t (&word)[2], uint32_t& pair) {
    float lo, hi, lo1, hi1;
    extremes(x[0], lo, hi);
    extremes(x[1], lo1, hi1);
    lo = min_nan(lo, lo1);
    hi = fmaxf(hi, hi1);
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {  // (stays inside the group's lanes)
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    hi = fminf(fmaxf(hi, -kLargest), kLargest);
    if (lo == lo) lo = fminf(fmaxf(lo, -kLargest), kLargest);
    const __half least = __float2half_rn(lo);
    const float least_f = __half2float(least);
    const __half scale = __float2half_rn(__fmul_rn(fmaxf(hi - least_f, 0.f), 1.0f / 15.0f));
    const float scale_f = __half2float(scale);
    pair = (uint32_t)__half_as_ushort(scale) | ((uint32_t)__half_as_ushort(least) << 16);
    word[0] = word[1] = 0;
    if (scale_f == 0.f) return;  // one value, or a NaN
    const float inv = __frcp_rn(scale_f);
    auto quotient = [&](float v) {
        const float t = v - least_f, q = t * inv;
        return fmaf(fmaf(-q, scale_f, t), inv, q);
    };
    // The ends lie beyond the codes where the range is far below the values, or values are beyond fp16.
    if (quotient(lo) > -0.5f && quotient(hi) < 15.5f && hi < kLargest && lo > -kLargest) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float four[2];
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                float c[4];
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    float t0, t1, q0, q1, r0, r1;
                    ptx::add2(t0, t1, Cvt<T>::to_f(x[n].v[i + e]), Cvt<T>::to_f(x[n].v[i + e + 1]), -least_f, -least_f);
                    ptx::fma2(q0, q1, t0, t1, inv, inv, -0.f, -0.f);
                    ptx::fma2(r0, r1, q0, q1, -scale_f, -scale_f, t0, t1);
                    ptx::fma2(q0, q1, r0, r1, inv, inv, q0, q1);
                    ptx::add2(q0, q1, q0, q1, 12582912.f, 12582912.f);  // 1.5 2^23: rounded to an integer
                    ptx::add2(c[e], c[e + 1], q0, q1, -12582912.f, -12582912.f);
                }
                float s0, s1;
                ptx::fma2(s0, s1, c[2], c[3], 256.f, 256.f, c[0], c[1]);
                four[i / 4] = fmaf(s1, 16.f, s0) + 8388608.f;  // 2^23: an integer added to it stands in the low bits
            }
            word[n] = __byte_perm(__float_as_uint(four[0]), __float_as_uint(four[1]), 0x5410);
        }
    } else {
#pragma unroll 1
        for (int i = 0; i < 16; ++i) {
            const float v = fminf(fmaxf(Cvt<T>::to_f(x[i >> 3].v[i & 7]), -kLargest), kLargest);
            const uint32_t code = (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(v - least_f, scale_f)), 0.f), 15.f) << (4 * (i & 7));
            if (i < 8) word[0] |= code;
            else word[1] |= code;
        }
    }
}

constexpr int kPerThread = 2;  // tokens in flight per thread

// A thread takes 16 channels of head blockIdx.y, of the keys or the values, of kPerThread tokens.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(256) kv4_append_kernel(const TokenParams p) {
    pdl_sync();
    constexpr int J = D / 8;  // threads of a token and head
    const int value = (int)(threadIdx.x % J) / (J / 2), j = 2 * (int)(threadIdx.x % (J / 2)), h = blockIdx.y;
    const int64_t first = (int64_t)blockIdx.x * (kPerThread * 256 / J) + threadIdx.x / J;
    const T* x = reinterpret_cast<const T*>(value ? p.v : p.k) + h * (value ? p.v_sh : p.k_sh) + j * 8;
    const int64_t stride = value ? p.v_st : p.k_st;
    Raw8<T> raw[kPerThread][2];
    int64_t slot[kPerThread];
#pragma unroll
    for (int n = 0; n < kPerThread; ++n) {
        const int64_t token = first + n * (256 / J);  // (a group's lanes agree on it)
        slot[n] = -1;
        raw[n][0] = raw[n][1] = {};
        if (token < p.tokens) {
            slot[n] = p.slots[token];
            raw[n][0] = load8<T, VEC>(x + token * stride);
            raw[n][1] = load8<T, VEC>(x + token * stride + 8);
        }
    }
#pragma unroll
    for (int n = 0; n < kPerThread; ++n) {
        uint32_t word[2], pair;
        quantise(raw[n], word, pair);
        uint8_t* tile = const_cast<uint8_t*>(tile_of_slot(p.cache, D, slot[n], h));
        if (tile == nullptr) continue;
        const int r = (int)(slot[n] & 15);
#pragma unroll
        for (int i = 0; i < 2; ++i) *reinterpret_cast<uint32_t*>(tile + (value ? value_word(D, r, j + i) : key_word(D, r, j + i))) = word[i];
        if ((j & 7) == 0) *reinterpret_cast<uint32_t*>(tile + pair_at(D, value, r, j >> 3)) = pair;
    }
}

template <typename T>
__device__ __forceinline__ void store_values(T* out, uint32_t word, uint32_t pair) {
    const float scale = __half2float(__ushort_as_half((unsigned short)(pair & 0xffffu)));
    const float least = __half2float(__ushort_as_half((unsigned short)(pair >> 16)));
    // codes masked out of the word are fp16 subnormals, n 2^-24 in the low bits of a half and n 2^-20 in the next
    const float even = scale * 0x1p24f, odd = scale * 0x1p20f;
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t u = (word >> (8 * (i / 2))) & ((i & 1) ? 0x00f000f0u : 0x000f000fu);
        const float2 n = __half22float2(*reinterpret_cast<const __half2*>(&u));
        ptx::fma2(v[i], v[i + 4], n.x, n.y, (i & 1) ? odd : even, (i & 1) ? odd : even, least, least);
    }
    if constexpr (std::is_same<T, __half>::value) {  // (a smaller scale cannot be rounded up so far: kv4_tile.cuh)
        if (scale >= kOverflowScale)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = in_range<T>(v[i]);
    }
    if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(out) = make_uint4(ptx::pack2<T>(v[0], v[1]), ptx::pack2<T>(v[2], v[3]), ptx::pack2<T>(v[4], v[5]), ptx::pack2<T>(v[6], v[7]));
    } else {
        st16(out, Vec16<T>{v[0], v[1], v[2], v[3]});
        st16(out + 4, Vec16<T>{v[4], v[5], v[6], v[7]});
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const TokenParams p) {
    pdl_sync();
    constexpr int J = D / 8;
    const int j = threadIdx.x % J, h = blockIdx.y;
    const int64_t first = (int64_t)blockIdx.x * (kPerThread * 256 / J) + threadIdx.x / J;
    uint32_t w[kPerThread][2], pr[kPerThread][2];
#pragma unroll
    for (int n = 0; n < kPerThread; ++n) {
        const int64_t token = first + n * (256 / J);
        w[n][0] = w[n][1] = pr[n][0] = pr[n][1] = 0;  // a slot that does not exist reads as zeros
        if (token >= p.tokens) continue;
        const int64_t slot = p.slots[token];
        const uint8_t* tile = tile_of_slot(p.cache, D, slot, h);
        const int r = (int)(slot & 15);
        if (tile != nullptr) {
            w[n][0] = *reinterpret_cast<const uint32_t*>(tile + key_word(D, r, j));
            w[n][1] = *reinterpret_cast<const uint32_t*>(tile + value_word(D, r, j));
            pr[n][0] = *reinterpret_cast<const uint32_t*>(tile + pair_at(D, 0, r, j >> 3));
            pr[n][1] = *reinterpret_cast<const uint32_t*>(tile + pair_at(D, 1, r, j >> 3));
        }
    }
#pragma unroll
    for (int n = 0; n < kPerThread; ++n) {
        const int64_t token = first + n * (256 / J), at = (token * p.cache.heads + h) * D + j * 8;
        if (token >= p.tokens) continue;
        store_values(reinterpret_cast<T*>(p.k_out) + at, w[n][0], pr[n][0]);
        store_values(reinterpret_cast<T*>(p.v_out) + at, w[n][1], pr[n][1]);
    }
}

template <typename T, int D>
int launch_tokens(const TokenParams& p, bool append, cudaStream_t st) {
    constexpr int kTokens = kPerThread * 256 / (D / 8);  // of a block
    const int64_t blocks = (p.tokens + kTokens - 1) / kTokens;
    const dim3 grid((unsigned)blocks, (unsigned)p.cache.heads);
    if (blocks > 0x7fffffffLL) return fail(XG_ERR_TOO_LARGE, "xg_kv4: too many tokens");
    if (append) {
        constexpr int N = Vec16<T>::N;
        const bool vec = aligned16(p.k) && aligned16(p.v) && p.k_st % N == 0 && p.k_sh % N == 0 && p.v_st % N == 0 && p.v_sh % N == 0;
        if (vec) launch(kv4_append_kernel<T, D, true>, grid, 256, 0, st, p);
        else launch(kv4_append_kernel<T, D, false>, grid, 256, 0, st, p);
        return check_launch("xg_kv4_append");
    }
    launch(kv4_read_kernel<T, D>, grid, 256, 0, st, p);
    return check_launch("xg_kv4_read");
}

template <typename T>
int launch_dim(const TokenParams& p, int64_t D, bool append, cudaStream_t st) {
    switch (D) {
        case 64: return launch_tokens<T, 64>(p, append, st);
        case 128: return launch_tokens<T, 128>(p, append, st);
        default: return launch_tokens<T, 256>(p, append, st);
    }
}

int launch_type(const TokenParams& p, int64_t D, int dtype, bool append, cudaStream_t st) {
    switch (dtype) {
        case XG_F32: return launch_dim<float>(p, D, append, st);
        case XG_BF16: return launch_dim<__nv_bfloat16>(p, D, append, st);
        default: return launch_dim<__half>(p, D, append, st);
    }
}

// ---- pages ---------------------------------------------------------------------------------------
// A launch's page numbers go with it: no copy to the device, and the caller's lists are free when the call returns. 1500 pages of 73 KB:
// 42 us, 10.7 us a launch (33 MB read, and as much written, most of which is still in L2 when it ends) and the gaps between four.
constexpr int kPairs = 448;  // page pairs per launch: with the rest within 4 KiB of kernel parameters
struct PageParams {
    uint8_t* base;
    int64_t page_stride, vectors;  // of 16 bytes in a page
    int32_t src[kPairs], dst[kPairs];
};
static_assert(sizeof(PageParams) <= 4096, "kernel parameters");

constexpr int kCopyVectors = 8;  // in flight per thread

__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ PageParams p) {
    pdl_sync();
    const uint4* src = reinterpret_cast<const uint4*>(p.base + (int64_t)p.src[blockIdx.y] * p.page_stride);
    uint4* dst = reinterpret_cast<uint4*>(p.base + (int64_t)p.dst[blockIdx.y] * p.page_stride);
    const int64_t first = (int64_t)blockIdx.x * (256 * kCopyVectors) + threadIdx.x;
    uint4 v[kCopyVectors];
#pragma unroll
    for (int i = 0; i < kCopyVectors; ++i)
        if (first + i * 256 < p.vectors) v[i] = src[first + i * 256];
#pragma unroll
    for (int i = 0; i < kCopyVectors; ++i)
        if (first + i * 256 < p.vectors) dst[first + i * 256] = v[i];
}

}  // namespace
}  // namespace xg

extern "C" int xg_kv4_append(void* cache, int64_t pages, int64_t heads, int64_t page_size, int64_t page_stride, const void* k, const void* v,
                             const int64_t* slots, int64_t tokens, int64_t D, int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t,
                             int64_t v_stride_h, int dtype, void* stream) {
    using namespace xg;
    if (const int rc = check_cache("xg_kv4_append", cache, pages, heads, page_size, page_stride, D)) return rc;
    if (dtype_size(dtype) == 0) return fail(XG_ERR_INVALID_ARG, "xg_kv4_append: bad dtype %d", dtype);
    if (tokens < 0) return fail(XG_ERR_INVALID_ARG, "xg_kv4_append: bad extents");
    if (tokens == 0 || pages == 0) return XG_OK;
    if (!k || !v || !slots) return fail(XG_ERR_INVALID_ARG, "xg_kv4_append: null pointer");
    TokenParams p = {};
    p.cache = {static_cast<const uint8_t*>(cache), pages, page_stride, (int)heads, (int)(page_size / 16)};
    p.k = k; p.v = v; p.slots = slots; p.tokens = tokens;
    p.k_st = k_stride_t; p.k_sh = k_stride_h; p.v_st = v_stride_t; p.v_sh = v_stride_h;
    return launch_type(p, D, dtype, true, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int xg_kv4_read(const void* cache, int64_t pages, int64_t heads, int64_t page_size, int64_t page_stride, const int64_t* slots,
                           int64_t tokens, int64_t D, void* k, void* v, int dtype, void* stream) {
    using namespace xg;
    if (const int rc = check_cache("xg_kv4_read", cache, pages, heads, page_size, page_stride, D)) return rc;
    if (dtype_size(dtype) == 0) return fail(XG_ERR_INVALID_ARG, "xg_kv4_read: bad dtype %d", dtype);
    if (tokens < 0) return fail(XG_ERR_INVALID_ARG, "xg_kv4_read: bad extents");
    if (tokens == 0) return XG_OK;
    if (!k || !v || !slots) return fail(XG_ERR_INVALID_ARG, "xg_kv4_read: null pointer");
    if (!aligned16(k) || !aligned16(v)) return fail(XG_ERR_INVALID_ARG, "xg_kv4_read: results must be 16-byte aligned");
    TokenParams p = {};
    p.cache = {static_cast<const uint8_t*>(cache), pages, page_stride, (int)heads, (int)(page_size / 16)};
    p.k_out = k; p.v_out = v; p.slots = slots; p.tokens = tokens;
    return launch_type(p, D, dtype, false, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int xg_copy_pages(void* base, int64_t pages, int64_t page_bytes, int64_t page_stride, const int64_t* src, const int64_t* dst,
                             int64_t count, void* stream) {
    using namespace xg;
    if (count < 0 || pages < 0 || page_bytes < 0 || (count > 0 && (!src || !dst))) return fail(XG_ERR_INVALID_ARG, "xg_copy_pages: bad arguments");
    if (pages > 0x7fffffffLL) return fail(XG_ERR_TOO_LARGE, "xg_copy_pages: too many pages");
    for (int64_t i = 0; i < count; ++i)
        if (src[i] < 0 || src[i] >= pages || dst[i] < 0 || dst[i] >= pages)
            return fail(XG_ERR_INVALID_ARG, "xg_copy_pages: page %lld -> %lld outside a cache of %lld pages", (long long)src[i], (long long)dst[i], (long long)pages);
    if (count == 0 || page_bytes == 0) return XG_OK;
    if (!base) return fail(XG_ERR_INVALID_ARG, "xg_copy_pages: null pointer");
    if (!aligned16(base) || page_bytes % 16 != 0 || page_stride % 16 != 0 || (pages > 1 && page_stride < page_bytes))
        return fail(XG_ERR_UNSUPPORTED, "xg_copy_pages: pages must be multiples of 16 bytes, start on 16-byte boundaries and not overlap");
    PageParams p;
    p.base = static_cast<uint8_t*>(base);
    p.page_stride = page_stride;
    p.vectors = page_bytes / 16;
    const int64_t gx = (p.vectors + 256 * kCopyVectors - 1) / (256 * kCopyVectors);
    if (gx > 0x7fffffffLL) return fail(XG_ERR_TOO_LARGE, "xg_copy_pages: pages too large");
    for (int64_t at = 0; at < count; at += kPairs) {
        const int n = (int)(count - at < kPairs ? count - at : kPairs);
        for (int i = 0; i < n; ++i) {
            p.src[i] = (int32_t)src[at + i];
            p.dst[i] = (int32_t)dst[at + i];
        }
        launch(copy_pages_kernel, dim3((unsigned)gx, (unsigned)n), 256, 0, reinterpret_cast<cudaStream_t>(stream), p);
        if (const int rc = check_launch("xg_copy_pages")) return rc;
    }
    return XG_OK;
}
