// The 4-bit cache: where keys, values and their scales lie. A cache is uint8 [pages, kv heads, page size / 16, 18 D]; its last
// dimension is a tile of 16 consecutive tokens of one head, D in {64, 128, 256}:
//   [0, 8 D)       key codes: token r's D/2 bytes at r * D/2. Chunk t (of 4), 32-bit word w: channels 32 w + 8 t + i, i = 0..7
//                  from the low bits up.
//   [8 D, 16 D)    value codes: token r's D/2 bytes at (4 c + t) * D/2 with t = (r >> 1) & 3, c = (r & 1) + 2 (r >> 3). Chunk g (of
//                  8) lies at place g ^ 2t; its word w: channels 64 w + 8 g + i.
//   [16 D, 17 D)   keys: token r's D/64 pairs (scale, least value) in fp16 at r * D/16, a pair for every 64 channels
//   [17 D, 18 D)   values: the same
// value = code * scale + least.
//
// The order is the attention kernel's: a lane (g = lane / 4, t = lane % 4) of mma.m16n8k16 holds rows g and g + 8 and columns 2t,
// 2t + 1, 2t + 8, 2t + 9 of its first operand. For the scores (rows = keys, columns = channels) chunk t of a token is what lane
// (., t) needs of it, and all four lanes' words w share a group of channels, so that a group is summed on its own. For the
// output (rows = channels, columns = keys) chunk g of tokens 2t, 2t + 1, 2t + 8, 2t + 9 is what lane (g, t) needs; a warp's
// reads touch every shared-memory bank once. A token stays contiguous (D/2 bytes for keys, D/2 for values), so that writing
// one touches whole sectors.
#pragma once

#include "common.cuh"

#include <type_traits>

namespace xg {
namespace kv4 {

constexpr int kTileTokens = 16;
constexpr float kLargest = 65504.0f;  // of fp16: values beyond are held as it
// A scale that was rounded up may put code 15 (no other) beyond kLargest, which is what such a code stands for: fp16 operands and results
// end there. To pass it so far that fp16 rounds to infinity (16 above it) takes a scale of 4096 or more: half a step of a smaller one
// is 1 at most, 15 times.
constexpr float kOverflowScale = 4096.0f;

__device__ __forceinline__ float min_nan(float a, float b) {  // NaN if one of them is
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// fp16 results end at fp16's largest value (a NaN stays one); other types hold what there is.
template <typename T>
__device__ __forceinline__ float in_range(float x) {
    if constexpr (std::is_same<T, __half>::value) {
        x = min_nan(x, kLargest);
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(x) : "f"(x), "f"(-kLargest));
    }
    return x;
}

__host__ __device__ constexpr int tile_bytes(int D) { return 18 * D; }

// byte offset in a tile of the 8 channels 8j .. 8j+7 of token r
__device__ __forceinline__ int key_word(int D, int r, int j) { return r * (D / 2) + ((j & 3) * (D / 32) + (j >> 2)) * 4; }
__device__ __forceinline__ int value_word(int D, int r, int j) {
    const int t = (r >> 1) & 3, c = (r & 1) + 2 * (r >> 3);
    return 8 * D + (4 * c + t) * (D / 2) + (((j & 7) ^ (2 * t)) * (D / 64) + (j >> 3)) * 4;
}
// byte offset of token r's (scale, least) pair of channel group gr; `value`: 0 keys, 1 values
__device__ __forceinline__ int pair_at(int D, int value, int r, int gr) { return (16 + value) * D + r * (D / 16) + gr * 4; }

// A cache as the kernels address it.
struct Cache {
    const uint8_t* base;
    int64_t pages, page_stride;  // bytes between pages
    int heads, tiles;            // tiles per page and head
};

// The tile that holds `slot` (= page * page size + offset), head h; null when there is no such slot.
__device__ __forceinline__ const uint8_t* tile_of_slot(const Cache& c, int D, int64_t slot, int h) {
    const int64_t tile = slot >> 4;
    if (slot < 0 || tile >= c.pages * c.tiles) return nullptr;  // (below 2^32: check_cache)
    const uint32_t page = (uint32_t)tile / (uint32_t)c.tiles, in_page = (uint32_t)tile - page * (uint32_t)c.tiles;
    return c.base + page * c.page_stride + ((int64_t)h * c.tiles + in_page) * tile_bytes(D);
}

inline int check_cache(const char* who, const void* base, int64_t pages, int64_t heads, int64_t page_size, int64_t page_stride, int64_t D) {
    if (D != 64 && D != 128 && D != 256) return fail(XG_ERR_UNSUPPORTED, "%s: head_dim %lld is not 64, 128 or 256", who, (long long)D);
    if (pages < 0 || heads <= 0 || page_size <= 0 || page_size % kTileTokens != 0)
        return fail(XG_ERR_INVALID_ARG, "%s: bad cache extents (a page holds a multiple of 16 tokens)", who);
    if (heads > 65535 || page_size > (1 << 20) || pages > 0xffffffffLL / (page_size / kTileTokens)) return fail(XG_ERR_TOO_LARGE, "%s: cache extents", who);
    if (page_stride % 16 != 0 || (pages > 1 && page_stride < heads * (page_size / 16) * tile_bytes((int)D)) || !aligned16(base))
        return fail(XG_ERR_INVALID_ARG, "%s: pages must start on 16-byte boundaries and not overlap", who);
    if (pages > 0 && !base) return fail(XG_ERR_INVALID_ARG, "%s: null pointer", who);
    return XG_OK;
}

}  // namespace kv4
}  // namespace xg
