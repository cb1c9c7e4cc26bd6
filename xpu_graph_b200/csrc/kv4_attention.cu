// Attention over the 4-bit cache: out = softmax(q k^T * scale) v for the newest tokens of every sequence. Query token i of the n_b new
// ones of sequence b stands at position len_b - n_b + i and sees the keys up to its own. Heads are grouped: query head h reads kv
// head h / (Hq / Hkv). fp32 scores, softmax and sums.
#include "kv4_tile.cuh"
#include "sm100_ptx.cuh"

namespace xg {
namespace {

using namespace kv4;
constexpr float kLog2e = 1.4426950408889634f;

struct AttendParams {
    Cache cache;
    const void* q;
    void* out;  // [tokens, Hq, D]
    const int64_t* table;
    const int64_t* lens;
    const int64_t* starts;  // null: one new token per sequence
    int64_t q_st, q_sh, table_stride;
    int64_t tokens;
    int batch, heads, group, table_pages;
    float scale;
};

__device__ __forceinline__ int64_t clamp64(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }

// Rows [first, first + count) of q that belong to sequence b, and its number of cached tokens.
struct Sequence {
    int64_t first, len;
    int count;
};
__device__ __forceinline__ Sequence sequence(const AttendParams& p, int b) {
    Sequence s;
    int64_t end;
    if (p.starts) {
        s.first = clamp64(p.starts[b], 0, p.tokens);
        end = clamp64(p.starts[b + 1], s.first, p.tokens);
    } else {
        s.first = b;
        end = b + 1;
    }
    s.count = (int)(end - s.first);
    s.len = clamp64(p.lens[b], 0, (int64_t)p.table_pages * p.cache.tiles * kTileTokens);
    return s;
}

// The sequence that row `token` belongs to, -1 if none does.
__device__ __forceinline__ int sequence_of(const AttendParams& p, int64_t token) {
    if (!p.starts) return token < p.batch ? (int)token : -1;
    int lo = 0, hi = p.batch;  // the last b with starts[b] <= token
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (p.starts[mid] <= token) lo = mid + 1;
        else hi = mid;
    }
    if (lo == 0 || p.starts[lo] <= token) return -1;
    return lo - 1;
}

// One warp per query token and head: a lane scores a key of 32, then owns D / 32 channels of the output.
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_attend_row_kernel(const AttendParams p) {
    pdl_sync();
    __shared__ float q_s[4][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 4 + warp;
    const int64_t token = row / p.heads;
    if (token >= p.tokens) return;
    const int head = (int)(row - token * p.heads), kvh = head / p.group;
    T* out = reinterpret_cast<T*>(p.out) + row * D;
    constexpr int C = D / 32;
    float o[C];
#pragma unroll
    for (int i = 0; i < C; ++i) o[i] = 0.f;
    float m = -INFINITY, l = 0.f;
    const int b = sequence_of(p, token);
    if (b >= 0) {
        const Sequence s = sequence(p, b);
        const int64_t visible = s.len - s.count + (token - s.first) + 1;
        for (int c = lane; c < D; c += 32) q_s[warp][c] = Cvt<T>::to_f(reinterpret_cast<const T*>(p.q)[token * p.q_st + head * p.q_sh + c]);
        __syncwarp();
        auto tile_at = [&](int64_t key) -> const uint8_t* {
            const int64_t t = key >> 4, page = t / p.cache.tiles;
            const int64_t id = p.table[(int64_t)b * p.table_stride + page];
            if (id < 0 || id >= p.cache.pages) return nullptr;
            return p.cache.base + id * p.cache.page_stride + ((int64_t)kvh * p.cache.tiles + (t - page * p.cache.tiles)) * tile_bytes(D);
        };
        auto pair = [&](const uint8_t* tile, int value, int r, int g) {
            return __half22float2(*reinterpret_cast<const __half2*>(tile + pair_at(D, value, r, g)));
        };
        for (int64_t k0 = 0; k0 < visible; k0 += 32) {
            const int64_t key = k0 + lane;
            float sc = -INFINITY;
            if (key < visible) {
                const uint8_t* tile = tile_at(key);
                if (tile != nullptr) {
                    const int r = (int)(key & 15);
                    sc = 0.f;
                    for (int g = 0; g < D / 64; ++g) {
                        const float2 sl = pair(tile, 0, r, g);
                        for (int j = 8 * g; j < 8 * g + 8; ++j) {
                            const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + key_word(D, r, j));
#pragma unroll
                            for (int i = 0; i < 8; ++i) sc = fmaf(q_s[warp][8 * j + i], fmaf((float)((w >> (4 * i)) & 15u), sl.x, sl.y), sc);
                        }
                    }
                    sc *= p.scale * kLog2e;
                }
            }
            const float m_new = fmaxf(m, warp_max(sc));
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = exp2f(m - m_use), pr = exp2f(sc - m_use);
            l = l * alpha + warp_sum(pr);
            m = m_new;
#pragma unroll
            for (int i = 0; i < C; ++i) o[i] *= alpha;
            for (int i = 0; i < 32 && k0 + i < visible; ++i) {
                const float w = __shfl_sync(0xffffffffu, pr, i);
                const uint8_t* tile = tile_at(k0 + i);
                if (tile == nullptr) continue;
                const int r = (int)((k0 + i) & 15);
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const int ch = c * 32 + lane;
                    const uint32_t word = *reinterpret_cast<const uint32_t*>(tile + value_word(D, r, ch >> 3));
                    const float2 sl = pair(tile, 1, r, ch >> 6);
                    o[c] = fmaf(w, fmaf((float)((word >> (4 * (ch & 7))) & 15u), sl.x, sl.y), o[c]);
                }
            }
        }
    }
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;  // no visible key: zeros
#pragma unroll
    for (int c = 0; c < C; ++c) out[c * 32 + lane] = Cvt<T>::from_f(o[c] * inv);
}

template <typename T, int D>
int launch_attend(const AttendParams& p, cudaStream_t st) {
    const int64_t grid = (p.tokens * p.heads + 3) / 4;
    if (grid > 0x7fffffffLL) return fail(XG_ERR_TOO_LARGE, "xg_kv4_attention: too many rows");
    launch(kv4_attend_row_kernel<T, D>, (unsigned)grid, 128, 0, st, p);
    return check_launch("xg_kv4_attention");
}

template <typename T>
int launch_attend_dim(const AttendParams& p, int64_t D, cudaStream_t st) {
    switch (D) {
        case 64: return launch_attend<T, 64>(p, st);
        case 128: return launch_attend<T, 128>(p, st);
        default: return launch_attend<T, 256>(p, st);
    }
}

}  // namespace
}  // namespace xg

extern "C" int64_t xg_kv4_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t D, int64_t max_q,
                                                    int64_t max_len) {
    (void)tokens; (void)batch; (void)q_heads; (void)kv_heads; (void)D; (void)max_q; (void)max_len;
    return 0;
}

extern "C" int xg_kv4_attention(const void* q, const void* cache, int64_t pages, int64_t kv_heads, int64_t page_size, int64_t page_stride,
                                const int64_t* page_table, int64_t table_pages, int64_t table_stride, const int64_t* kv_lens,
                                const int64_t* q_starts, void* out, int64_t tokens, int64_t batch, int64_t q_heads, int64_t D, int64_t max_q,
                                int64_t q_stride_t, int64_t q_stride_h, float scale, int dtype, void* workspace, int64_t workspace_bytes,
                                void* stream) {
    using namespace xg;
    if (const int rc = check_cache("xg_kv4_attention", cache, pages, kv_heads, page_size, page_stride, D)) return rc;
    if (dtype != XG_BF16 && dtype != XG_F16) return fail(XG_ERR_UNSUPPORTED, "xg_kv4_attention: 16-bit dtypes only");
    if (tokens < 0 || batch < 0 || q_heads <= 0 || q_heads % kv_heads != 0 || max_q < 0 || table_pages < 0 || workspace_bytes < 0)
        return fail(XG_ERR_INVALID_ARG, "xg_kv4_attention: bad extents");
    if (q_heads > 65535 || batch > 0x7fffff || tokens > 0x7fffffff || table_pages > 0x7ffffff) return fail(XG_ERR_TOO_LARGE, "xg_kv4_attention: extents");
    if (table_pages * page_size > 0x7fffff00LL) return fail(XG_ERR_TOO_LARGE, "xg_kv4_attention: more than 2^31 tokens per sequence");
    if (tokens == 0) return XG_OK;
    if (!q || !out || (batch > 0 && (!kv_lens || (table_pages > 0 && !page_table)))) return fail(XG_ERR_INVALID_ARG, "xg_kv4_attention: null pointer");
    if (!aligned16(out)) return fail(XG_ERR_INVALID_ARG, "xg_kv4_attention: the result must be 16-byte aligned");
    AttendParams p = {};
    p.cache = {static_cast<const uint8_t*>(cache), pages, page_stride, (int)kv_heads, (int)(page_size / 16)};
    p.q = q; p.out = out; p.table = page_table; p.lens = kv_lens; p.starts = q_starts;
    p.q_st = q_stride_t; p.q_sh = q_stride_h; p.table_stride = table_stride;
    p.tokens = tokens; p.batch = (int)batch; p.heads = (int)q_heads; p.group = (int)(q_heads / kv_heads); p.table_pages = (int)table_pages;
    p.scale = scale;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return dtype == XG_BF16 ? launch_attend_dim<__nv_bfloat16>(p, D, st) : launch_attend_dim<__half>(p, D, st);
}
