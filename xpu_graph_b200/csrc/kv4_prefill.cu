// Attention of many new tokens over the 4-bit cache: flash attention on tcgen05 with keys and values unpacked on the way in.
//
// A CTA owns 256 rows of one kv head - rows are the (new token, head of the group) pairs in token order, so that all heads of a group
// share the unpacked keys - as two 128-row tiles (one at head dim 256). Per block of 64 keys: warps unpack K and V from a ring of
// bulk copies into fp16 operand tiles (128-byte swizzle, the layout a tensor map would leave); one thread issues S = Q K^T for both
// tiles into double-buffered tensor memory, then O += P V with P read from tensor memory; eight warps (a row per thread) turn
// scores into probabilities in place, as flash_tc_kernel (sdpa.cu) does, with the maximum lagging by up to 2^8.
//
// Everything that meets in a product is fp16: codes are exact there, code * scale + least is rounded once (2^-11 relative), as are
// probabilities (kTop). Queries are carried after a power of two per row, the row's largest below 2^15, which returns in the row's
// exponent factor: exactly, down to 2^-29 of that largest. Sums are fp32 in tensor memory and registers.
//
// What bounds it: per block of 64 keys the products take 1024 cycles of the tensor pipe (40 % busy), the 256 x 64 exponentials 1024 of
// the special-function unit (41 %), and unpacking (2 operations per code) and softmax 49 % of the issue slots; they run beside each
// other, but a tile's scores, probabilities and product follow one another, and about 8 us in front of and behind a unit's blocks
// overlap with nothing. 3 sequences of 2500 to 8192 keys with 2048 new tokens: 32 / 8 heads of 128 464 us back to back (1047 TFLOP/s),
// 500 with pauses, 564 on another machine; of 64 403 us (604 TFLOP/s). Head dim 256 has room for one tile and one buffer of V: 16 / 4 heads
// 827 us (588 TFLOP/s). Tried without gain: a warpgroup more for unpacking with the registers dealt out anew; the last wave's units
// shared out over the idle CTAs (their parts cost what the wave gains).
#include "kv4_attend.cuh"

namespace xg {

__device__ unsigned int g_kv4_prefill_status[4];

namespace {

using namespace kv4;

constexpr int PM = 128;  // rows per tile
constexpr int PN = 64;   // keys per block
constexpr int kBlockTiles = PN / kTileTokens;
constexpr int kPrefillThreads = 13 * 32;  // unpacking, one warp for the products, softmax
constexpr float kLag = 8.0f;  // log2 units
// The largest probability is carried as 2^kTop, 2^(kTop + kLag) with the lag: as high as fp16 goes, so that the least ones (2^-32 of it
// with kTop, 2^-25 without) still count in O as they do in the sum. One key 17.5 above 16383 others lost their 0.04 % without.
constexpr float kTop = 7.0f;

template <int D>
struct PreCfg {
    // Two tiles of rows share the unpacked keys, so that unpacking is half as much per product; at head dim 256 neither tensor memory
    // (two outputs would fill it) nor shared memory has room for them, nor for a second buffer of V. Twice the warps unpack then.
    static constexpr int TILES = D == 256 ? 1 : 2, VBUF = TILES, UNPACK = TILES == 2 ? 4 : 8, RING_STAGES = TILES == 2 ? 4 : 2;
    static constexpr int ROWS = TILES * PM;
    static constexpr int HALVES = UNPACK / kBlockTiles, TOKENS = kTileTokens / HALVES;  // a warp's tokens of a tile
    static constexpr int Q_BYTES = PM * D * 2;
    static constexpr int KV_BYTES = PN * D * 2;
    static constexpr int TILE = tile_bytes(D), STAGE = TILE / HALVES;  // of the ring
    static constexpr int RING = UNPACK * RING_STAGES * STAGE;
    static constexpr int SMEM = TILES * Q_BYTES + (2 + VBUF) * KV_BYTES + RING + 768;
    static constexpr uint32_t O_COL = TILES * 2 * PN;  // tensor memory: two score buffers per tile, then the outputs
    static_assert(O_COL + TILES * D <= 512 && SMEM <= 232448, "fits an SM");
};

struct Unit {
    int on, b, kvh, rt;  // rt: which 256 rows
    int first, count, len, pad;
};

// Keys shared out over several CTAs: their parts, unnormalised. Rows of all parts, (maximum, sum) pairs, then a Unit per unit.
struct Parts {
    float* rows;  // [units][splits][256][D]
    float2* ml;   // [units][splits][256]
    Unit* unit;   // [units]
    int splits;   // 1: none of this. 128 new tokens behind 32640, 32 / 8 heads: 98 us, one CTA per unit 650
};

// 8 codes as fp16 values, in the order 0 4 1 5 2 6 3 7, in which masks find them: q lies in that order too, and the output's columns
// are put right when they leave. `scale` and `least` in both halves.
__device__ __forceinline__ uint4 unpack8(uint32_t w, __half2 scale, __half2 least) {
    uint32_t out[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        // a code in bits 0-3 of a half becomes 1024 + n, one in bits 4-7 64 + n
        const uint32_t y = ((w >> (8 * (k / 2))) & ((k & 1) ? 0x00f000f0u : 0x000f000fu)) | ((k & 1) ? 0x54005400u : 0x64006400u);
        const __half2 n = __hsub2(*reinterpret_cast<const __half2*>(&y), __half2half2(__ushort_as_half((k & 1) ? 0x5400 : 0x6400)));
        const __half2 v = __hfma2(n, scale, least);
        out[k] = *reinterpret_cast<const uint32_t*>(&v);
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

// The infinity that unpack8 makes of a code beyond fp16's largest value (kOverflowScale) would be NaN in the rows that do not see the
// token. A warp that meets such a scale goes over the operand rows that it has stored once more: `rows` rows of 128 bytes, `groups`
// times, a block of keys apart. What asking costs, by a packed maximum of the pairs' bits and a vote per block: 461 -> 468 us (3
// sequences with 2048 new tokens), head dim 64 402 -> 406, 256 none; a test at every store cost 10 %.
constexpr int kOverflowBits = 0x6c00;  // kOverflowScale in fp16
__device__ __noinline__ void end_at_largest(uint32_t base, int rows, int groups, int lane) {
    __syncwarp();
    const __half2 largest = __half2half2(__ushort_as_half(0x7bff));
#pragma unroll 1
    for (int i = lane; i < groups * rows * 8; i += 32) {
        const int gr = i / (rows * 8);
        const uint32_t at = base + (uint32_t)(gr * (PN * 128) + (i - gr * rows * 8) * 16);
        uint4 v = ptx::ld_shared_v4(at);
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const __half2 x = __hmin2_nan(*reinterpret_cast<const __half2*>(&w[e]), largest);
            w[e] = *reinterpret_cast<const uint32_t*>(&x);
        }
        ptx::st_shared_v4(at, v);
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kPrefillThreads, 1) kv4_prefill_kernel(const AttendParams p, int beyond, const Parts parts) {
    using Cfg = PreCfg<D>;
    constexpr int W = D / 32, GR = D / 64;
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr int TILES = Cfg::TILES, UNPACK = Cfg::UNPACK, STAGES = Cfg::RING_STAGES;
    uint8_t* q_s = smem;                                  // [TILES][Q_BYTES]; at the end the output rows on their way out
    uint8_t* k_s = q_s + TILES * Cfg::Q_BYTES;            // [2][KV_BYTES]
    uint8_t* v_s = k_s + 2 * Cfg::KV_BYTES;               // [VBUF][KV_BYTES]
    uint8_t* ring = v_s + Cfg::VBUF * Cfg::KV_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(ring + Cfg::RING);
    uint64_t* q_full = bars;          // [tile]
    uint64_t* k_full = bars + 2;      // [buffer]
    uint64_t* k_empty = bars + 4;
    uint64_t* v_full = bars + 6;
    uint64_t* v_empty = bars + 8;
    uint64_t* s_full = bars + 10;     // [tile][buffer]
    uint64_t* p_full = bars + 14;     // [tile][buffer]
    uint64_t* pv_full = bars + 18;    // [tile]
    uint64_t* o_full = bars + 20;     // [tile]
    uint64_t* drain_bar = bars + 22;
    uint64_t* ring_full = bars + 23;  // [warp][stage]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 23 + UNPACK * STAGES);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* holes = abort_flag + 1;              // [4][warp]: a block's tiles that are not in the cache
    volatile int* ring_hole = holes + 4 * UNPACK;      // [warp][stage]
    Unit* unit = reinterpret_cast<Unit*>(const_cast<int*>(ring_hole + UNPACK * STAGES));
    static_assert(23 * 8 + UNPACK * STAGES * 8 + 8 + (4 * UNPACK + UNPACK * STAGES) * 4 + sizeof(Unit) <= 768, "barriers");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if ((ptx::smem_u32(smem) & 1023u) != 0) {  // uniform over the CTA: the swizzled tiles need this alignment
        pdl_sync();
        if (threadIdx.x == 0) atomicOr(&g_kv4_prefill_status[0], 4u);
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&q_full[i], PM);
            ptx::mbar_init(&k_full[i], UNPACK);
            ptx::mbar_init(&k_empty[i], 1);
            ptx::mbar_init(&v_full[i], UNPACK);
            ptx::mbar_init(&v_empty[i], 1);
            ptx::mbar_init(&pv_full[i], 1);
            ptx::mbar_init(&o_full[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            ptx::mbar_init(&s_full[i], 1);
            ptx::mbar_init(&p_full[i], PM);
        }
        ptx::mbar_init(drain_bar, 1);
        for (int i = 0; i < UNPACK * STAGES; ++i) ptx::mbar_init(&ring_full[i], 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::fence_proxy_async();
    }
    if (warp == UNPACK) ptx::tmem_alloc(tmem_slot, 512);
    pdl_wait();
    if (warp == 0) {  // which rows are this CTA's: the sequences' units one after the other, the last rows (most keys) first
        constexpr int K = 4;  // sequences per lane: their loads overlap
        const uint32_t mine = blockIdx.x / parts.splits;
        uint32_t base = 0;
        bool found = false;
        for (int b0 = 0; b0 < p.batch && !found; b0 += 32 * K) {
            Sequence s[K];
            uint32_t w[K], sum = 0;
#pragma unroll
            for (int i = 0; i < K; ++i) {
                const int b = b0 + lane * K + i;
                s[i] = {};
                if (b < p.batch) s[i] = sequence(p, b);
                w[i] = s[i].count * p.group > beyond ? (uint32_t)((s[i].count * p.group + Cfg::ROWS - 1) / Cfg::ROWS) * p.cache.heads : 0;
                sum += w[i];
            }
            uint32_t inc = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += v;
            }
            uint32_t off = mine - base - (inc - sum);  // of this lane's units
            const uint32_t here = __ballot_sync(0xffffffffu, off < sum);
            found = here != 0;
            if (found && lane == __ffs(here) - 1) {  // (one lane, whatever q_starts holds)
#pragma unroll
                for (int i = 0; i < K; ++i) {
                    if (off < w[i]) {
                        const int tiles = (int)(w[i] / p.cache.heads);
                        *unit = {1, b0 + lane * K + i, (int)(off % p.cache.heads), tiles - 1 - (int)(off / p.cache.heads), (int)s[i].first, s[i].count, (int)s[i].len, 0};
                        break;
                    }
                    off -= w[i];
                }
            }
            base += __shfl_sync(0xffffffffu, inc, 31);
        }
        if (!found && lane == 0) *unit = {};
    } else if (beyond == 0) {  // one sequence: the rows in front of it and behind it
        const Sequence s = sequence(p, 0);
        const int64_t per_row = (int64_t)p.heads * D;
        for (int64_t r = blockIdx.x; r < p.tokens - s.count; r += gridDim.x) {
            T* row = reinterpret_cast<T*>(p.out) + (r < s.first ? r : r + s.count) * per_row;
            for (int64_t c = threadIdx.x - 32; c < per_row / 8; c += kPrefillThreads - 32) *reinterpret_cast<uint4*>(row + c * 8) = make_uint4(0, 0, 0, 0);
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    pdl_trigger();  // the tensor memory is held
    const uint32_t tmem_base = *tmem_slot;
    const Unit u = *unit;

    const int rows = u.count * p.group;
    // key blocks of a tile: up to what its last row sees
    auto blocks_of = [&](int i) {
        const int lo = u.rt * Cfg::ROWS + i * PM;
        if (!u.on || i >= TILES || lo >= rows) return 0;
        const int seen = u.len - u.count + (min(rows, lo + PM) - 1) / p.group + 1;
        return seen > 0 ? (seen + PN - 1) / PN : 0;
    };
    // blocks j0 .. of this CTA; every role counts them from 0
    const int all_blocks = max(blocks_of(0), blocks_of(1)), split = (int)blockIdx.x % parts.splits;
    const int j0 = (int)((int64_t)all_blocks * split / parts.splits), nblk = (int)((int64_t)all_blocks * (split + 1) / parts.splits) - j0;
    const int nblk0 = min(nblk, max(0, blocks_of(0) - j0)), nblk1 = min(nblk, max(0, blocks_of(1) - j0));
    if (parts.splits > 1 && split == 0 && threadIdx.x == 0) parts.unit[blockIdx.x / parts.splits] = u;

    if (warp < UNPACK) {
        // ------------------------------ unpacking ---------------------------------
        const int mine = warp / Cfg::HALVES, h = warp % Cfg::HALVES;  // tile of the block, which of its tokens: TOKENS h and on
        uint8_t* my_ring = ring + warp * (STAGES * Cfg::STAGE);   // a stage: codes of keys, of values, pairs of keys, of values
        uint64_t* my_full = ring_full + warp * STAGES;
        volatile int* my_hole = ring_hole + warp * STAGES;
        int64_t addr = 0;
        auto issue = [&](int j) {  // this warp's tile of block j
            if (j >= nblk) return;
            if ((j & 31) == 0) {
                const int tile = (j0 + j + lane) * kBlockTiles + mine;
                addr = tile * kTileTokens < u.len ? tile_of_token(p, u.b, u.kvh, tile, Cfg::TILE) : 0;
            }
            const int64_t from = __shfl_sync(0xffffffffu, addr, j & 31);
            const int stage = j % STAGES;
            if (lane == 0) {
                my_hole[stage] = from == 0;
                if (from != 0) {
                    ptx::mbar_arrive_expect_tx(&my_full[stage], Cfg::STAGE);
                    uint8_t* dst = my_ring + stage * Cfg::STAGE;
                    const uint8_t* src = reinterpret_cast<const uint8_t*>(from);
                    if (Cfg::HALVES == 1) {
                        ptx::bulk_load(dst, src, Cfg::TILE, &my_full[stage]);
                    } else {  // (a half of a tile's tokens is a half of each of its four parts)
                        constexpr int C = 8 * D / Cfg::HALVES, P = D / Cfg::HALVES;
                        ptx::bulk_load(dst, src + h * C, C, &my_full[stage]);
                        ptx::bulk_load(dst + C, src + 8 * D + h * C, C, &my_full[stage]);
                        ptx::bulk_load(dst + 2 * C, src + 16 * D + h * P, P, &my_full[stage]);
                        ptx::bulk_load(dst + 2 * C + P, src + 17 * D + h * P, P, &my_full[stage]);
                    }
                } else {
                    ptx::mbar_arrive(&my_full[stage]);
                }
            }
        };
        for (int j = 0; j < STAGES; ++j) issue(j);
        // A NaN among a token's values reaches the rows that see it through their scores, and no other row.
        const __half2 zero = __half2half2(__ushort_as_half(0)), lowest = __half2half2(__ushort_as_half(0xfbff));
        bool ok = true;
        // keys: a lane takes chunk t of rows r and r + 8; the bits are dealt so that neither its reads nor its swizzled writes collide
        const int kr = (lane & 1) | ((lane >> 3) & 1) << 1 | ((lane >> 1) & 1) << 2, kt = ((lane >> 4) & 1) | ((lane >> 2) & 1) << 1;
        for (int j = 0; j < nblk; ++j) {
            const int stage = j % STAGES, buf = j & 1;
            const uint32_t ph = (uint32_t)(j >> 1) & 1u;
            if (!__all_sync(0xffffffffu, ptx::mbar_wait_bounded(&my_full[stage], (uint32_t)(j / STAGES) & 1u, abort_flag))) { ok = false; break; }
            constexpr int C = 8 * D / Cfg::HALVES, P = D / Cfg::HALVES;
            const uint8_t* codes = my_ring + stage * Cfg::STAGE;
            const uint8_t* pair_s = codes + 2 * C;  // a token's pairs D / 16 bytes apart
            const int hole = my_hole[stage];
            const int there = hole ? 0 : u.len - ((j0 + j) * kBlockTiles + mine) * kTileTokens - h * Cfg::TOKENS;  // of this warp's tokens
            if (!__all_sync(0xffffffffu, ptx::mbar_wait_bounded(&k_empty[buf], ph ^ 1u, abort_flag))) { ok = false; break; }
            if (lane == 0) holes[(j & 3) * UNPACK + warp] = hole;
            uint32_t top = 0;  // low half: largest scale that this lane looks at, by its bits
            bool wide;
            {
                const uint32_t base = ptx::smem_u32(k_s + buf * Cfg::KV_BYTES) + (uint32_t)(warp * Cfg::TOKENS * 128);
#pragma unroll
                for (int half = 0; half < Cfg::TOKENS / 8; ++half) {
                    const int r = kr + 8 * half;
                    uint32_t words[W];
                    __half2 pairs[GR], v_pairs[GR];
                    load_words<W>(codes + r * (D / 2) + kt * (D / 8), words);
                    load_pairs<GR>(pair_s + r * (D / 16), pairs);
                    load_pairs<GR>(pair_s + P + r * (D / 16), v_pairs);
#pragma unroll
                    for (int gr = 0; gr < GR; ++gr) {
                        top = __vimax3_s16x2(top, *reinterpret_cast<const uint32_t*>(&pairs[gr]), *reinterpret_cast<const uint32_t*>(&v_pairs[gr]));
                        pairs[0] = __hfma2(v_pairs[gr], zero, pairs[0]);  // NaN if the token's values hold one
                    }
#pragma unroll
                    for (int gr = 0; gr < GR; ++gr) {
                        const __half2 pair = r < there ? pairs[gr] : zero, scale = __low2half2(pair), least = __high2half2(pair);
#pragma unroll
                        for (int w = 0; w < 2; ++w)  // chunks 4 w + kt
                            ptx::st_shared_v4(base + (uint32_t)(gr * (PN * 128) + r * 128 + (((4 * w + kt) ^ (r & 7)) << 4)), unpack8(words[2 * gr + w], scale, least));
                    }
                }
                wide = __any_sync(0xffffffffu, (int)(short)(top & 0xffffu) >= kOverflowBits);
                if (wide) end_at_largest(base, Cfg::TOKENS, GR, lane);
            }
            ptx::fence_proxy_async();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&k_full[buf]);
            const int vbuf = Cfg::VBUF == 2 ? buf : 0;
            if (!__all_sync(0xffffffffu, ptx::mbar_wait_bounded(&v_empty[vbuf], (Cfg::VBUF == 2 ? ph : (uint32_t)j & 1u) ^ 1u, abort_flag))) { ok = false; break; }
            {
                const uint32_t base = ptx::smem_u32(v_s + vbuf * Cfg::KV_BYTES) + (uint32_t)(warp * Cfg::TOKENS * 128);
#pragma unroll
                for (int i = 0; i < Cfg::TOKENS / 4; ++i) {  // (rows of value codes: 8 tokens' are a half of the tile's as well)
                    const int at = i * 4 + (lane >> 3), t = at & 3, c = at >> 2, r = 2 * t + (c & 1) + 8 * (c >> 1);
                    const int place = lane & 7, chunk = place ^ (2 * t);
                    uint32_t words[GR];
                    __half2 pairs[GR];
                    load_words<GR>(codes + C + at * (D / 2) + place * (D / 16), words);
                    load_pairs<GR>(pair_s + P + r * (D / 16), pairs);
#pragma unroll
                    for (int w = 0; w < GR; ++w) {
                        // (a NaN, with codes of 0, becomes finite: a product with the probability 0 of a row that does not see it is 0)
                        const __half2 pair = r < there ? __hmax2(pairs[w], lowest) : zero;
                        ptx::st_shared_v4(base + (uint32_t)(w * (PN * 128) + r * 128 + ((chunk ^ (r & 7)) << 4)),
                                          unpack8(words[w], __low2half2(pair), __high2half2(pair)));
                    }
                }
                if (wide) end_at_largest(base, Cfg::TOKENS, GR, lane);
            }
            ptx::fence_proxy_async();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&v_full[vbuf]);
            issue(j + STAGES);
        }
        if (!ok) {
            if (lane == 0) atomicOr(&g_kv4_prefill_status[0], 1u);
            const uint64_t t0 = ptx::globaltimer_ns();
            while (ptx::globaltimer_ns() - t0 < 20000ull) {
            }
        }
    } else if (warp == UNPACK) {
        // ------------------------------ products ----------------------------------
        if (ptx::elect_one()) {
            constexpr uint32_t idesc_s = ptx::make_idesc_f16(0, PM, PN, 0);
            constexpr uint32_t idesc_o = ptx::make_idesc_f16(0, PM, D, 1);
            bool ok = true;
            // Score buffer j & 1 of a tile is free without a barrier of its own: block j - 2's P V was issued before, after the
            // softmax warps had written P, and the tensor core runs this thread's products in order.
            auto issue_qk = [&](int j) -> bool {
                const int buf = j & 1;
                if (!ptx::mbar_wait_bounded(&k_full[buf], (uint32_t)(j >> 1) & 1u, abort_flag)) return false;
                ptx::tc_fence_after();
                const uint32_t k_addr = ptx::smem_u32(k_s + buf * Cfg::KV_BYTES);
                for (int i = 0; i < TILES; ++i) {
                    if (j >= (i ? nblk1 : nblk0)) continue;
                    if (j == 0 && !ptx::mbar_wait_bounded(&q_full[i], 0, abort_flag)) return false;
                    if (j == 0) ptx::tc_fence_after();
                    const uint32_t q_addr = ptx::smem_u32(q_s + i * Cfg::Q_BYTES);
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                        ptx::mma_f16_ss(tmem_base + (uint32_t)((2 * i + buf) * PN),
                                        ptx::make_kmajor_sw128_desc(q_addr + (uint32_t)((kk >> 2) * (PM * 128) + (kk & 3) * 32)),
                                        ptx::make_kmajor_sw128_desc(k_addr + (uint32_t)((kk >> 2) * (PN * 128) + (kk & 3) * 32)), idesc_s, kk != 0 ? 1u : 0u);
                    ptx::tc_commit(&s_full[2 * i + buf]);
                }
                ptx::tc_commit(&k_empty[buf]);
                return true;
            };
            if (nblk > 0) ok = issue_qk(0);
            for (int j = 0; j < nblk && ok; ++j) {
                if (j + 1 < nblk && !issue_qk(j + 1)) { ok = false; break; }
                const int buf = j & 1;
                const uint32_t ph = (uint32_t)(j >> 1) & 1u;
                const int vbuf = Cfg::VBUF == 2 ? buf : 0;
                if (!ptx::mbar_wait_bounded(&v_full[vbuf], Cfg::VBUF == 2 ? ph : (uint32_t)j & 1u, abort_flag)) { ok = false; break; }
                const uint32_t v_addr = ptx::smem_u32(v_s + vbuf * Cfg::KV_BYTES);
                for (int i = 0; i < TILES && ok; ++i) {
                    const int n = i ? nblk1 : nblk0;
                    if (j >= n) continue;
                    if (!ptx::mbar_wait_bounded(&p_full[2 * i + buf], ph, abort_flag)) { ok = false; break; }
                    ptx::tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < PN / 16; ++kk)  // P: 16 keys = 8 columns of packed pairs per step, over its scores
                        ptx::mma_f16_ts(tmem_base + Cfg::O_COL + (uint32_t)(i * D), tmem_base + (uint32_t)((2 * i + buf) * PN + kk * 8),
                                        ptx::make_mnmajor_sw128_desc(v_addr + (uint32_t)(kk * 16 * 128), PN * 128), idesc_o, (j | kk) != 0 ? 1u : 0u);
                    ptx::tc_commit(&pv_full[i]);
                    if (j + 1 == n) ptx::tc_commit(&o_full[i]);
                }
                if (ok) ptx::tc_commit(&v_empty[vbuf]);
            }
            if (!ok) {
                atomicOr(&g_kv4_prefill_status[0], 2u);
                ptx::tc_commit(drain_bar);
                const uint64_t t0 = ptx::globaltimer_ns();
                while (!ptx::mbar_try_wait(drain_bar, 0)) {
                    if (ptx::globaltimer_ns() - t0 > ptx::kWaitLimitNs) break;
                }
            }
        }
    } else {
        // ------------------------------ softmax / output rows ---------------------
        const int i = (warp - UNPACK - 1) >> 2, quad = warp & 3;
        const int r_in_tile = quad * 32 + lane;
        const int n = i ? nblk1 : nblk0;
        const int lo = u.rt * Cfg::ROWS + i * PM;
        const int row = lo + r_in_tile;
        const bool there = u.on && row < rows;
        const int token = there ? row / p.group : 0;
        const int head = u.kvh * p.group + (there ? row - token * p.group : 0);
        const int limit = there ? u.len - u.count + token + 1 : 0x7fffffff;  // keys that the row sees
        float mul = 0.f;
        if (n > 0) {
            // this row of q, a power of two taken out, into the operand tile
            const T* q = reinterpret_cast<const T*>(p.q) + (int64_t)(u.first + token) * p.q_st + (int64_t)head * p.q_sh;
            const bool vec = (reinterpret_cast<uintptr_t>(p.q) & 15) == 0 && p.q_st % 8 == 0 && p.q_sh % 8 == 0;
            // 16 loads at once, a row of 128 (what stands in front of a unit's first block counts: four at a time, and again for the second
            // use, 3 sequences with 2048 new tokens took 505 us where this takes 475, 600 with 20 each 733 and now 572); of a row of 256 the
            // first half comes a second time, from the cache. A row per group of lanes, with whole lines per load, took 497 and 679.
            constexpr int HELD = D < 128 ? D / 8 : 16;
            uint4 held[HELD];
            auto fetch = [&](int c0) {
#pragma unroll
                for (int c = 0; c < HELD; ++c) held[c] = there ? load_q8(q + 8 * (c0 + c), vec) : make_uint4(0, 0, 0, 0);
            };
            float top = 0.f;
#pragma unroll
            for (int c0 = 0; c0 < D / 8; c0 += HELD) {
                fetch(c0);
#pragma unroll
                for (int c = 0; c < HELD; ++c) {
                    const T* e = reinterpret_cast<const T*>(&held[c]);
#pragma unroll
                    for (int x = 0; x < 8; ++x) top = fmaxf(top, fabsf(Cvt<T>::to_f(e[x])));
                }
            }
            const int e = max(-100, (int)(__float_as_uint(top) >> 23) - 127);  // the row is carried below 2^15 (up to 128: infinities)
            float down = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
            if (p.scale == 0.f) down = 0.f;
            if (p.scale < 0.f) down = -down;
            mul = fmaxf((p.scale == 0.f ? 1.f : fabsf(p.scale)) * kLog2e * __uint_as_float((uint32_t)(127 + e - 14) << 23), 1e-37f);
            const uint32_t base = ptx::smem_u32(q_s + i * Cfg::Q_BYTES) + (uint32_t)(r_in_tile * 128);
#pragma unroll
            for (int c0 = D / 8 - HELD; c0 >= 0; c0 -= HELD) {
                if (c0 != D / 8 - HELD) fetch(c0);
#pragma unroll
                for (int c = 0; c < HELD; ++c) {
                    const T* e8 = reinterpret_cast<const T*>(&held[c]);
                    uint32_t w[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) w[x] = ptx::pack2<__half>(Cvt<T>::to_f(e8[x]) * down, Cvt<T>::to_f(e8[x + 4]) * down);  // (unpack8's order)
                    const int at = c0 + c;
                    ptx::st_shared_v4(base + (uint32_t)((at >> 3) * (PM * 128) + (((at & 7) ^ (r_in_tile & 7)) << 4)), make_uint4(w[0], w[1], w[2], w[3]));
                }
            }
            ptx::fence_proxy_async();
            ptx::mbar_arrive(&q_full[i]);
        }
        const uint32_t lane_field = (uint32_t)(quad * 32) << 16;
        const uint32_t o_taddr = tmem_base + lane_field + Cfg::O_COL + (uint32_t)(i * D);
        bool ok = true;
        float m_run = -INFINITY, l_run = 0.f;
        for (int j = 0; j < n; ++j) {
            const int buf = j & 1;
            if (!__all_sync(0xffffffffu, ptx::mbar_wait_bounded(&s_full[2 * i + buf], (uint32_t)(j >> 1) & 1u, abort_flag))) { ok = false; break; }
            ptx::tc_fence_after();
            const uint32_t s_taddr = tmem_base + lane_field + (uint32_t)((2 * i + buf) * PN);
            const int visible = limit - (j0 + j) * PN;  // columns of this block that the row sees
            int hole = 0;
#pragma unroll
            for (int w = 0; w < kBlockTiles; ++w) hole |= (holes[(j & 3) * UNPACK + w * Cfg::HALVES] != 0) << w;
            if (__all_sync(0xffffffffu, visible <= 0) || hole == 15) {  // probabilities of zero; maximum and sum stay
                uint32_t zero[32];
#pragma unroll
                for (int c = 0; c < 32; ++c) zero[c] = 0u;
                ptx::tmem_st_32x32(s_taddr, zero);
                ptx::tmem_st_wait();
                ptx::tc_fence_before();
                ptx::mbar_arrive(&p_full[2 * i + buf]);
                continue;
            }
            float sc[PN];
            {
                uint32_t r0[32], r1[32];
                ptx::tmem_ld_32x32(s_taddr, r0);
                ptx::tmem_ld_32x32(s_taddr + 32u, r1);
                ptx::tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 32; ++c) {
                    sc[c] = __uint_as_float(r0[c]);
                    sc[32 + c] = __uint_as_float(r1[c]);
                }
            }
            if (__any_sync(0xffffffffu, visible < PN) || hole != 0) {
#pragma unroll
                for (int c = 0; c < PN; ++c)
                    if (c >= visible || ((hole >> (c / kTileTokens)) & 1)) sc[c] = -INFINITY;
            }
            if (m_run == -INFINITY) {
                float mxp[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) mxp[c] = ptx::fmax3(sc[c], sc[8 + c], sc[16 + c]);
#pragma unroll
                for (int at = 24; at < PN; at += 16)
#pragma unroll
                    for (int c = 0; c < 8; ++c) mxp[c] = at + 8 < PN ? ptx::fmax3(mxp[c], sc[at + c], sc[at + 8 + c]) : fmaxf(mxp[c], sc[at + c]);
                m_run = ptx::fmax3(ptx::fmax3(mxp[0], mxp[1], mxp[2]), ptx::fmax3(mxp[3], mxp[4], mxp[5]), fmaxf(mxp[6], mxp[7])) * mul;
                // (nothing has been added to O yet but zeros, so a first maximum needs no rescaling)
            }
            uint32_t pk[32];
#pragma unroll 1
            for (int attempt = 0; attempt < 2; ++attempt) {
                const float neg_m = m_run == -INFINITY ? 0.f : kTop - m_run;
                float lp[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                float mxp[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) mxp[c] = -INFINITY;
#pragma unroll
                for (int c = 0; c < PN; c += 2) {
                    float x0, x1;
                    ptx::fma2(x0, x1, sc[c], sc[c + 1], mul, mul, neg_m, neg_m);
                    const int pair = c >> 1;
                    const float p0 = ptx::ex2_approx(x0), p1 = ptx::ex2_approx(x1);
                    mxp[pair & 7] = ptx::fmax3(mxp[pair & 7], sc[c], sc[c + 1]);
                    ptx::add2(lp[2 * (pair & 3)], lp[2 * (pair & 3) + 1], lp[2 * (pair & 3)], lp[2 * (pair & 3) + 1], p0, p1);
                    pk[pair] = ptx::pack2<__half>(p0, p1);
                }
                const float l_blk = ((lp[0] + lp[1]) + (lp[2] + lp[3])) + ((lp[4] + lp[5]) + (lp[6] + lp[7]));
                if (attempt == 0 && j > 0) {
                    const float mx = ptx::fmax3(ptx::fmax3(mxp[0], mxp[1], mxp[2]), ptx::fmax3(mxp[3], mxp[4], mxp[5]), fmaxf(mxp[6], mxp[7])) * mul;
                    const float m_new = fmaxf(m_run, mx);
                    if (__any_sync(0xffffffffu, m_new > m_run + kLag)) {
                        const float m_to = m_new == -INFINITY ? 0.f : m_new;
                        const float alpha = ptx::ex2_approx(m_run - m_to);
                        if (!__all_sync(0xffffffffu, ptx::mbar_wait_bounded(&pv_full[i], (uint32_t)(j - 1) & 1u, abort_flag))) { ok = false; break; }
                        ptx::tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[32];
                            ptx::tmem_ld_32x32(o_taddr + (uint32_t)(c * 32), o);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
                            ptx::tmem_st_32x32(o_taddr + (uint32_t)(c * 32), o);
                        }
                        l_run *= alpha;
                        m_run = m_new;
                        continue;
                    }
                }
                l_run += l_blk;
                break;
            }
            if (!ok) break;
            ptx::tmem_st_32x32(s_taddr, pk);
            ptx::tmem_st_wait();
            ptx::tc_fence_before();
            ptx::mbar_arrive(&p_full[2 * i + buf]);
        }
        if (ok && n > 0) ok = __all_sync(0xffffffffu, ptx::mbar_wait_bounded(&o_full[i], 0, abort_flag)) != 0;
        if (ok && parts.splits > 1 && there) {
            ptx::tc_fence_after();
            const int64_t at = (int64_t)blockIdx.x * Cfg::ROWS + i * PM + r_in_tile;
            parts.ml[at] = make_float2(m_run, l_run);
        }
        if (ok && parts.splits > 1 && u.on && lo + quad * 32 < rows) {
            const int64_t at = (int64_t)blockIdx.x * Cfg::ROWS + i * PM + r_in_tile;
#pragma unroll 1
            for (int c = 0; c < D / 32 && n > 0; ++c) {
                uint32_t o[32];
                ptx::tmem_ld_32x32(o_taddr + (uint32_t)(c * 32), o);
                ptx::tmem_ld_wait();
                if (!there) continue;
#pragma unroll
                for (int x = 0; x < 32; x += 4) *reinterpret_cast<uint4*>(parts.rows + at * D + c * 32 + x) = make_uint4(o[x], o[x + 1], o[x + 2], o[x + 3]);
            }
            ptx::tc_fence_before();
        } else if (ok && u.on && lo + quad * 32 < rows) {
            ptx::tc_fence_after();
            const float inv_l = l_run > 0.f || l_run != l_run ? 1.0f / l_run : 0.f;
            // rows leave through a slab of shared memory (this tile's q, which no product reads any more), so that stores are whole lines
            const uint32_t slab = ptx::smem_u32(q_s + i * Cfg::Q_BYTES) + (uint32_t)(quad * 4096);
            T* out = reinterpret_cast<T*>(p.out);
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                if (n > 0) {
                    ptx::tmem_ld_32x32(o_taddr + (uint32_t)(c * 32), o);
                    ptx::tmem_ld_wait();
                } else {
#pragma unroll
                    for (int x = 0; x < 32; ++x) o[x] = 0u;
                }
#pragma unroll
                for (int t4 = 0; t4 < 4; ++t4) {
                    uint32_t w[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {  // channels 2 x, 2 x + 1 (unpack8's order)
                        const int at = t4 * 8 + 4 * (x & 1) + (x >> 1);
                        w[x] = ptx::pack2<T>(in_range<T>(__uint_as_float(o[at]) * inv_l), in_range<T>(__uint_as_float(o[at + 2]) * inv_l));
                    }
                    const int at = (c & 1) * 4 + t4;
                    ptx::st_shared_v4(slab + (uint32_t)(lane * 128 + ((at ^ (lane & 7)) << 4)), make_uint4(w[0], w[1], w[2], w[3]));
                }
                if (c & 1) {
                    __syncwarp();
#pragma unroll
                    for (int it = 0; it < 8; ++it) {
                        const int r = it * 4 + (lane >> 3), at = lane & 7, row_i = lo + quad * 32 + r;
                        const uint4 val = ptx::ld_shared_v4(slab + (uint32_t)(r * 128 + ((at ^ (r & 7)) << 4)));
                        if (row_i < rows) {
                            const int tk = row_i / p.group, hd = u.kvh * p.group + (row_i - tk * p.group);
                            *reinterpret_cast<uint4*>(out + ((int64_t)(u.first + tk) * p.heads + hd) * D + (c >> 1) * 64 + at * 8) = val;
                        }
                    }
                    __syncwarp();
                }
            }
            ptx::tc_fence_before();
        }
        if (!ok && lane == 0) atomicOr(&g_kv4_prefill_status[0], 4u);
    }

    ptx::tc_fence_before();
    __syncthreads();
    if (warp == UNPACK) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem_base, 512);
    }
}

// out = sum 2^(m_i - m) O_i / sum 2^(m_i - m) l_i over a row's parts, a warp per row. Parts that saw no key have written no row.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_prefill_combine_kernel(const AttendParams p, const Parts parts) {
    pdl_sync();
    const Unit u = parts.unit[blockIdx.x];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int ROWS = PreCfg<D>::ROWS;
    const int in_unit = blockIdx.y * 8 + warp, row = u.rt * ROWS + in_unit;
    if (!u.on || row >= u.count * p.group) return;
    auto at = [&](int i) { return ((int64_t)blockIdx.x * parts.splits + i) * ROWS + in_unit; };
    float m = -INFINITY;
    for (int i = lane; i < parts.splits; i += 32) m = fmaxf(m, parts.ml[at(i)].x);
    m = warp_max(m);
    const float use = m == -INFINITY ? 0.f : m;
    constexpr int C = D / 32;  // columns C lane ..
    float l = 0.f, o[C];
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = 0.f;
#pragma unroll 4
    for (int i = 0; i < parts.splits; ++i) {
        const float2 part = parts.ml[at(i)];
        if (part.x == -INFINITY && part.y == 0.f) continue;
        const float f = ptx::ex2_approx(part.x - use);
        l = fmaf(part.y, f, l);
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] = fmaf(parts.rows[at(i) * D + c * 32 + lane], f, o[c]);
    }
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
    const int token = row / p.group, head = u.kvh * p.group + (row - token * p.group);
    T* out = reinterpret_cast<T*>(p.out) + ((int64_t)(u.first + token) * p.heads + head) * D;
    // column x of 8 is channel 4 (x & 1) + x / 2 (unpack8's order)
    const int ch = (lane & ~7) + 4 * (lane & 1) + ((lane & 7) >> 1);
#pragma unroll
    for (int c = 0; c < C; ++c) out[c * 32 + ch] = Cvt<T>::from_f(in_range<T>(o[c] * inv));
}

// The most units there can be, and over how many CTAs each one's keys are shared out: as many as fill the chip once, 320 keys or more each
// (1 sequence of 1000 with 256 new tokens: 25 us in three parts, whole 27.5; of 512, all new, 26 in two parts, whole 20.6).
int64_t most_units(int64_t tokens, int64_t batch, int64_t group, int64_t heads, int64_t rows) { return (tokens * group + batch * (rows - 1)) / rows * heads; }
int key_splits(int64_t tokens, int64_t batch, int64_t group, int64_t heads, int64_t rows, int64_t max_len) {
    // (how many units there are likely to be, with rows dealt out evenly: 8 sequences of 16000 with 9 new tokens, 8 heads of 256: two parts
    // of 64 units 325 us; for the most there can be, 80, they stayed whole, 610)
    const int64_t even = batch > 0 ? batch * (((tokens + batch - 1) / batch * group + rows - 1) / rows) * heads : 0;
    const int64_t most = most_units(tokens, batch, group, heads, rows), units = even < most ? even : most;
    int64_t n = num_sms() / (units > 0 ? units : 1);
    if (n > max_len / 320) n = max_len / 320;
    return (int)(n < 1 ? 1 : n);
}

template <typename T, int D>
int launch_prefill(const AttendParams& p, int beyond, void* workspace, cudaStream_t st) {
    using Cfg = PreCfg<D>;
    static std::atomic<uint64_t> reserved;
    if (!reserve_smem(kv4_prefill_kernel<T, D>, Cfg::SMEM, reserved)) return fail(XG_ERR_LAUNCH, "xg_kv4_attention: cannot reserve shared memory");
    // at least as many CTAs as there are units; those behind the last one return at once
    const int64_t units = most_units(p.tokens, p.batch, p.group, p.cache.heads, Cfg::ROWS);
    Parts parts = {};
    parts.splits = key_splits(p.tokens, p.batch, p.group, p.cache.heads, Cfg::ROWS, (int64_t)p.table_pages * p.cache.tiles * kTileTokens);
    if (units * parts.splits > 0x7fffffffLL) return fail(XG_ERR_TOO_LARGE, "xg_kv4_attention: too many rows");
    if (parts.splits > 1) {
        const int64_t rows = units * parts.splits * Cfg::ROWS;
        parts.rows = static_cast<float*>(workspace);
        parts.ml = reinterpret_cast<float2*>(parts.rows + rows * D);
        parts.unit = reinterpret_cast<Unit*>(parts.ml + rows);
    }
    launch(kv4_prefill_kernel<T, D>, (unsigned)(units * parts.splits), kPrefillThreads, Cfg::SMEM, st, p, beyond, parts);
    if (const int rc = check_launch("xg_kv4_attention")) return rc;
    if (parts.splits == 1) return XG_OK;
    launch(kv4_prefill_combine_kernel<T, D>, dim3((unsigned)units, Cfg::ROWS / 8), 256, 0, st, p, parts);
    return check_launch("xg_kv4_attention");
}

}  // namespace

int64_t prefill_workspace(int64_t tokens, int64_t batch, int64_t group, int64_t heads, int64_t D, int64_t max_len) {
    const int64_t rows = D == 256 ? PreCfg<256>::ROWS : PreCfg<128>::ROWS, units = most_units(tokens, batch, group, heads, rows);
    const int splits = key_splits(tokens, batch, group, heads, rows, max_len);
    return splits == 1 ? 0 : units * splits * rows * (D + 2) * 4 + units * (int64_t)sizeof(Unit);
}

int attend_prefill(const AttendParams& p, int64_t D, int dtype, int beyond, void* workspace, cudaStream_t st) {
    const bool bf16 = dtype == XG_BF16;
    switch (D) {
        case 64: return bf16 ? launch_prefill<__nv_bfloat16, 64>(p, beyond, workspace, st) : launch_prefill<__half, 64>(p, beyond, workspace, st);
        case 128: return bf16 ? launch_prefill<__nv_bfloat16, 128>(p, beyond, workspace, st) : launch_prefill<__half, 128>(p, beyond, workspace, st);
        default: return bf16 ? launch_prefill<__nv_bfloat16, 256>(p, beyond, workspace, st) : launch_prefill<__half, 256>(p, beyond, workspace, st);
    }
}

int read_kv4_prefill_status(unsigned int* host_out, int reset) {
    unsigned int v[4] = {0, 0, 0, 0};
    if (cudaMemcpyFromSymbol(v, g_kv4_prefill_status, sizeof(v)) != cudaSuccess) {
        cudaGetLastError();
        return fail(XG_ERR_DEVICE, "xg_tc_status: cannot read device status");
    }
    *host_out = v[0];
    if (reset && v[0] != 0) {
        unsigned int z[4] = {0, 0, 0, 0};
        cudaMemcpyToSymbol(g_kv4_prefill_status, z, sizeof(z));
    }
    return XG_OK;
}
}  // namespace xg
