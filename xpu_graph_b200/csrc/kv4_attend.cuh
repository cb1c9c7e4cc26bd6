// What the kernels of the attention over the 4-bit cache share.
#pragma once

#include "kv4_tile.cuh"
#include "sm100_ptx.cuh"

#include <type_traits>

namespace xg {
namespace kv4 {

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
    int row0;  // without starts: the row of the first sequence
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
        s.first = p.row0 + b;
        end = s.first + 1;
    }
    s.count = (int)(end - s.first);
    s.len = clamp64(p.lens[b], 0, (int64_t)p.table_pages * p.cache.tiles * kTileTokens);
    return s;
}

// 8 channels of a finished row; a row that saw no key is zeros. (in_range: an average of the largest values may be rounded beyond them.)
template <typename T>
__device__ __forceinline__ void store_row8(T* out, const float (&o)[8], float sum) {
    const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
    Vec16<T> y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y.v[e] = Cvt<T>::from_f(in_range<T>(o[e] * inv));
    st16(out, y);
}

template <typename T>
__device__ __forceinline__ uint4 load_q8(const T* p, bool vec) {  // 8 elements
    if (vec) return *reinterpret_cast<const uint4*>(p);
    const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// N 32-bit words at once
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&out)[N]) {
    if constexpr (N == 1) {
        out[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (N == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        out[0] = u.x; out[1] = u.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(p + 4 * i);
            out[i] = u.x; out[i + 1] = u.y; out[i + 2] = u.z; out[i + 3] = u.w;
        }
    }
}
// N (scale, least) pairs at once
template <int N>
__device__ __forceinline__ void load_pairs(const uint8_t* p, __half2 (&out)[N]) {
    uint32_t u[N];
    load_words<N>(p, u);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = *reinterpret_cast<const __half2*>(&u[i]);
}

// The usual case is one question; what waits longer does so outside the loop's code.
static __device__ __noinline__ bool wait_longer(uint64_t* bar, uint32_t phase, volatile int* abort_flag) { return ptx::mbar_wait_bounded(bar, phase, abort_flag); }
__device__ __forceinline__ bool wait_stage(uint64_t* bar, uint32_t phase, volatile int* abort_flag) {
    return ptx::mbar_try_wait(bar, phase) || wait_longer(bar, phase, abort_flag);
}

// The tile that holds token 16 * tile of sequence b, kv head kvh; 0 where its page is not one of the cache.
__device__ __forceinline__ int64_t tile_of_token(const AttendParams& p, int b, int kvh, int tile, int bytes) {
    const int page = tile / p.cache.tiles;
    const int64_t id = p.table[(int64_t)b * p.table_stride + page];
    if (id < 0 || id >= p.cache.pages) return 0;
    return reinterpret_cast<int64_t>(p.cache.base + id * p.cache.page_stride + ((int64_t)kvh * p.cache.tiles + (tile - page * p.cache.tiles)) * bytes);
}

}  // namespace kv4

// Many new tokens per sequence (kv4_prefill.cu): the sequences with more than `beyond` columns (new token, head of the group); with
// `beyond` 0 and one sequence also the rows of none.
int attend_prefill(const kv4::AttendParams& p, int64_t D, int dtype, int beyond, void* workspace, cudaStream_t st);
int64_t prefill_workspace(int64_t tokens, int64_t batch, int64_t group, int64_t heads, int64_t D, int64_t max_len);
int read_kv4_prefill_status(unsigned int* host_out, int reset);

}  // namespace xg
