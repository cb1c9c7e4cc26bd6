// Attention over the 4-bit cache: out = softmax(q k^T * scale) v for the newest tokens of every sequence. Query token i of the n_b new
// ones of sequence b stands at position len_b - n_b + i and sees the keys up to its own. Heads are grouped: query head h reads kv
// head h / (Hq / Hkv). fp32 scores, softmax and sums.
#include "kv4_attend.cuh"

namespace xg {

// Status word of the kernels here (device globals are per translation unit without -rdc).
__device__ unsigned int g_kv4_status[4];

namespace {

using namespace kv4;

// ---------------------------------------------------------------------------------------
// Few query rows per sequence: the cache streamed once
// ---------------------------------------------------------------------------------------
// A unit is a (sequence, kv head, tile of 8 NT columns); its columns are the (new token, head of the group) pairs that read this kv
// head. The 32-key blocks of all units form one line, cut into equal ranges, one per CTA, and those into one per warp, so that
// sequences of any mixture of lengths load the chip evenly. A warp streams its range through a ring of bulk copies of its own and
// writes the units that lie wholly in it; what the warps' cuts leave is added in shared memory at the CTA's end, what the CTAs' cuts
// leave by kv4_combine_kernel, both in range order.
//
// Both products run on mma.m16n8k16 with the codes as fp16: a 4-bit code n masked out of its word is the subnormal n 2^-24 in bits
// 0-3 and n 2^-20 in bits 4-7, which the tensor core multiplies exactly, so unpacking costs one logic operation per two codes and no
// arithmetic.
//   scores (16 keys x 8 columns, per group of 64 channels):  x = scale_k acc + least_k sum(q), the group's sum of q kept per column.
//     q has a power of two per row taken out, with which bf16 fits fp16 exactly (down to 2^-29 of the row's largest).
//   output (16 channels x 8 columns):  sum p v = sum w (code - 8) + sum p (least_v + 8 scale_v), w = p scale_v rounded to fp16 (2^-11
//     relative at most). The codes go in as they are; 8 sum w, from a product with ones, comes off every 256 keys, before the sums have
//     grown so far that what the tensor core cuts off below 2^-24 of them is a bias (a flat average over 131072 keys would be 3 % off).
//     It cuts by the operands' exponents, which subnormals do not have: a code 2^-20 loses four bits less than one 2^-24. Where that
//     shows, in fp16 results, both codes of a byte go in as 2^-20 (131072 keys: 0.00036 of the result, then 0.00030; 0.00021 is its
//     own rounding), for one operation of the FMA pipe per register.
//     w is kept below 2^15 by the power of two that the scales have reached so far; p, up to 2^8, may be 2^29 smaller still.
// Both that power and the maximum of a column follow their data lagging: only a step beyond them rescales the sums.
// The codes of keys that do not exist are finite whatever they are; their scales are replaced, not multiplied away.
//
// Code that runs once per unit is kept short: fetching it costs more than running it (with a second copy of the loop for masked
// blocks 64 sequences of 512 to 8192 tokens took 92 us, with one 82).
// What bounds it: unpacking and the softmax's scalar work, 54 % of the issue slots and 48 % of the logic pipe at three warps a
// scheduler, beside 50 % of HBM: 4 sequences of 65536, 32 / 8 heads of 128: 75 us, 4.05 TB/s (the loads alone 60, the arithmetic alone
// 73). More tiles in work at once, other occupancies, packed fp32 pairs and shifts by multiplication gave nothing. Not used: with one new
// token and a group of 4, columns 4-7 do not exist, and the lanes that hold them do the softmax's work for nothing.
constexpr int kWarps = 4;
constexpr int kBlockTiles = 2, kBlockKeys = kBlockTiles * kTileTokens;  // what a stage holds
constexpr int kMaxBatch = 1024;  // sequences per launch: their prefix sums live in shared memory

// CTAs per SM, by what the fragments and sums take of the register file
constexpr int split_ctas(int D, int NT) { return D == 256 ? 2 : (NT == 1 ? (D == 64 ? 4 : 3) : (D == 64 ? 3 : 2)); }

// What a warp's range leaves unfinished: the end of a unit that began before it, the beginning of one that goes on behind it (a range
// inside one unit is an end that does not end).
struct Cut {
    int any, head, head_ends, tail;
    int first, count, kvh, ct, parts;  // of the tail's unit; parts: CTA ranges that it reaches, 1 if it ends in this one
};

template <int D, int NT>
struct SplitCfg {
    static constexpr int COLS = 8 * NT;
    static constexpr int TILE = tile_bytes(D);
    static constexpr int STAGE = kBlockTiles * TILE;
    static constexpr int STAGES = 2;
    static constexpr int KT = NT == 1 && D <= 128 ? 2 : 1;  // tiles in work at once: more independent products per warp, more registers
    static constexpr int RING = kWarps * STAGES * STAGE;
    static constexpr int O_STRIDE = D + 4;  // floats
    static constexpr int SLOT = COLS * O_STRIDE;  // floats of one part in shared memory
    static constexpr int O_BYTES = kWarps * SLOT * 4;
    static constexpr int ML_BYTES = 2 * kWarps * COLS * 8;
    static constexpr int BAR_BYTES = kWarps * STAGES * 8;
    static constexpr int FIXED = RING + O_BYTES + ML_BYTES + BAR_BYTES + kWarps * (int)sizeof(Cut) + kWarps * STAGES * 4 + 64;
    static_assert(SLOT * 4 <= STAGES * STAGE, "a warp's ring holds a part");
    static constexpr int part_floats() { return COLS * (D + 2); }
    static int smem(int batch) { return FIXED + (batch + 1) * 4 + batch * 12; }
    static constexpr int CTAS = split_ctas(D, NT);
};

struct SplitParams {
    AttendParams a;
    float* parts;  // [2 * gridDim.x][COLS][D] sums, then [2 * gridDim.x][COLS] (maximum, sum) pairs, then a PartDesc per CTA
    int split;         // 0: a unit stays in one CTA
    uint32_t min_blocks; // of a range
    int most_cols;       // sequences with more columns are left alone
    int first_rows, last_rows;  // this launch zeroes the rows before the first / behind the last sequence
};

// What starts in a CTA's range and ends in a later one's.
struct PartDesc {
    int parts;  // 0: nothing
    int first, count, kvh, ct, pad[3];
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, (SplitCfg<D, NT>::CTAS)) kv4_split_kernel(const SplitParams sp) {
    using Cfg = SplitCfg<D, NT>;
    constexpr int W = D / 32, GR = D / 64;
    // fp16 results: the even channels' value codes are moved up to the odd ones' place, see above
    constexpr bool FINE = std::is_same<T, __half>::value;
    constexpr float kEven = FINE ? 0x1p20f : 0x1p24f, kOdd = 0x1p20f, kOddEight = FINE ? 1.f : 16.f;
    constexpr uint32_t kEight = FINE ? 0x00800080u : 0x00080008u;
    const AttendParams& p = sp.a;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* ring = smem;
    float* head_s = reinterpret_cast<float*>(smem + Cfg::RING);  // [warp][COLS][O_STRIDE]; a tail goes where the warp's ring was
    float2* ml_s = reinterpret_cast<float2*>(smem + Cfg::RING + Cfg::O_BYTES);  // [head, tail][warp][COLS]
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::RING + Cfg::O_BYTES + Cfg::ML_BYTES);
    uint32_t* prefix = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(bars) + Cfg::BAR_BYTES);  // [batch + 1]
    int* first_s = reinterpret_cast<int*>(prefix + p.batch + 1);  // (the host keeps the line below 2^31 blocks)
    int* count_s = first_s + p.batch;
    int* len_s = count_s + p.batch;
    volatile int* hidden_s = len_s + p.batch;  // [kWarps][STAGES], a bit per tile
    volatile int* abort_flag = hidden_s + kWarps * Cfg::STAGES;
    Cut* cut_s = reinterpret_cast<Cut*>(const_cast<int*>(abort_flag + 1));
    uint32_t* scan_s = reinterpret_cast<uint32_t*>(head_s);  // before the first segment only

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    if (tid == 0) {
        for (int i = 0; i < kWarps * Cfg::STAGES; ++i) ptx::mbar_init(&bars[i], 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::fence_proxy_async();
    }
    pdl_wait();

    // ---- the line of tiles
    const int kv_heads = p.cache.heads;
    auto col_tiles = [&](int count) { return (count * p.group + Cfg::COLS - 1) / Cfg::COLS; };
    auto blocks_of = [&](int b) { return (len_s[b] + kBlockKeys - 1) / kBlockKeys; };
    uint32_t carry = 0;
    for (int base = 0; base < p.batch; base += kWarps * 32) {
        const int b = base + tid;
        uint32_t w = 0;
        if (b < p.batch) {
            const Sequence s = sequence(p, b);
            first_s[b] = (int)s.first;
            count_s[b] = s.count;
            const int len = s.count * p.group > sp.most_cols ? -1 : (int)s.len;
            len_s[b] = len;
            w = len <= 0 ? 0 : (uint32_t)kv_heads * col_tiles(s.count) * ((len + kBlockKeys - 1) / kBlockKeys);
        }
        uint32_t inc = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) scan_s[warp] = inc;
        __syncthreads();
        uint32_t before = carry, all = carry;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            if (i < warp) before += scan_s[i];
            all += scan_s[i];
        }
        if (b < p.batch) prefix[b] = before + inc - w;
        carry = all;
        __syncthreads();
    }
    if (tid == 0) prefix[p.batch] = carry;
    __syncthreads();
    const uint32_t total = carry;

    // rows that no key reaches because there is no sequence, or nothing in its cache
    {
        const int64_t per_row = (int64_t)p.heads * D;
        T* out = reinterpret_cast<T*>(p.out);
        auto zero = [&](int64_t lo, int64_t hi, int first, int step) {
            for (int64_t r = lo + first; r < hi; r += step)
                for (int64_t i = tid; i < per_row / 8; i += kWarps * 32) *reinterpret_cast<uint4*>(out + r * per_row + i * 8) = make_uint4(0, 0, 0, 0);
        };
        if (sp.first_rows) zero(0, p.batch > 0 ? first_s[0] : p.tokens, blockIdx.x, gridDim.x);
        if (sp.last_rows && p.batch > 0) zero((int64_t)first_s[p.batch - 1] + count_s[p.batch - 1], p.tokens, blockIdx.x, gridDim.x);
        for (int b = blockIdx.x; b < p.batch; b += gridDim.x)
            if (len_s[b] == 0) zero(first_s[b], (int64_t)first_s[b] + count_s[b], 0, 1);
    }

    uint32_t ranges = (total + sp.min_blocks - 1) / sp.min_blocks;
    if (ranges > gridDim.x) ranges = gridDim.x;
    const uint32_t share = ranges ? total / ranges : 0, over = total - share * ranges;
    auto range_at = [&](uint32_t i) { return share * i + (i < over ? i : over); };  // where range i starts
    uint32_t start = 0, end = 0;
    auto sequence_at = [&](uint32_t x) {  // the b with prefix[b] <= x < prefix[b + 1]
        int lo = 0, hi = p.batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (prefix[mid] <= x) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    if (blockIdx.x < ranges) {
        start = range_at(blockIdx.x);
        end = range_at(blockIdx.x + 1);
        if (!sp.split) {
            auto up = [&](uint32_t x) {
                if (x >= total) return total;
                const int b = sequence_at(x);
                const uint32_t n = blocks_of(b), off = x - prefix[b];
                return prefix[b] + (off + n - 1) / n * n;
            };
            start = up(start);
            end = up(end);
        }
    }
    PartDesc* desc = reinterpret_cast<PartDesc*>(sp.parts + (int64_t)2 * gridDim.x * Cfg::part_floats()) + blockIdx.x;
    if (sp.split && tid == 0) desc->parts = 0;
    if (start >= end) return;

    // ---- this warp's blocks
    const uint32_t quarter = (end - start) / kWarps, left = (end - start) % kWarps;
    const uint32_t my_start = start + quarter * warp + min((uint32_t)warp, left), my_end = my_start + quarter + (warp < left ? 1 : 0);
    const int mine = (int)(my_end - my_start);
    uint8_t* my_ring = ring + warp * (Cfg::STAGES * Cfg::STAGE);
    uint64_t* my_bars = bars + warp * Cfg::STAGES;
    volatile int* my_hidden = hidden_s + warp * Cfg::STAGES;
    // where this lane's block of the current batch of 32 lies, tile by tile; 0 where there is nothing to read
    int64_t addr[kBlockTiles] = {};
    auto look_up = [&](int i) {
        const uint32_t x = my_start + i + lane;
#pragma unroll
        for (int k = 0; k < kBlockTiles; ++k) addr[k] = 0;
        if (x >= my_end) return;
        const int b = sequence_at(x);
        const uint32_t n = blocks_of(b), off = x - prefix[b];
        const uint32_t unit = off / n;
        const int kvh = (int)(unit / (uint32_t)col_tiles(count_s[b]));
#pragma unroll
        for (int k = 0; k < kBlockTiles; ++k) {
            const int tile = (int)(off - unit * n) * kBlockTiles + k;
            if (tile * kTileTokens >= len_s[b]) break;
            addr[k] = tile_of_token(p, b, kvh, tile, Cfg::TILE);
        }
    };
    auto issue = [&](int i, int stage) {
        if (i >= mine) return;
        if ((i & 31) == 0) look_up(i);
        int64_t from[kBlockTiles];
#pragma unroll
        for (int k = 0; k < kBlockTiles; ++k) from[k] = __shfl_sync(0xffffffffu, addr[k], i & 31);
        if (lane == 0) {
            int hidden = 0, bytes = 0;
#pragma unroll
            for (int k = 0; k < kBlockTiles; ++k) {
                if (from[k] == 0) hidden |= 1 << k;
                else bytes += Cfg::TILE;
            }
            my_hidden[stage] = hidden;
            ptx::mbar_arrive_expect_tx(&my_bars[stage], bytes);
            if (from[1] == from[0] + Cfg::TILE) {
                ptx::bulk_load(my_ring + stage * Cfg::STAGE, reinterpret_cast<const void*>(from[0]), 2 * Cfg::TILE, &my_bars[stage]);
            } else {
#pragma unroll
                for (int k = 0; k < kBlockTiles; ++k)
                    if (from[k] != 0) ptx::bulk_load(my_ring + stage * Cfg::STAGE + k * Cfg::TILE, reinterpret_cast<const void*>(from[k]), Cfg::TILE, &my_bars[stage]);
            }
        }
    };
    for (int i = 0; i < Cfg::STAGES; ++i) issue(i, i);

    // a negative scale goes into q, a zero one makes q zero
    const float q_mul = p.scale > 0.f ? 1.f : (p.scale < 0.f ? -1.f : (p.scale == 0.f ? 0.f : p.scale));
    const float scale_log2 = (p.scale != 0.f ? fabsf(p.scale) : 1.f) * kLog2e;
    int done = 0, stage = 0;  // tiles of this warp consumed, and the stage of the next one
    uint32_t phase = 0;
    bool ok = true;
    Cut cut = {mine > 0};
    int b = mine > 0 ? sequence_at(my_start) : 0;
    for (uint32_t pos = my_start; pos < my_end && ok;) {
        while (prefix[b + 1] <= pos) ++b;
        const int n_blocks = blocks_of(b), count = count_s[b], len = len_s[b];
        const uint32_t off = pos - prefix[b];
        const uint32_t unit = off / (uint32_t)n_blocks;
        const int t0 = (int)(off - unit * n_blocks);  // blocks, as n_blocks and seg
        const int cts = col_tiles(count);
        const int kvh = (int)(unit / (uint32_t)cts), ct = (int)(unit - (uint32_t)kvh * cts);
        const int seg = min(n_blocks - t0, (int)(my_end - pos));

        // ---- q as fragments; column n = 8 nt + g is the pair (new token col / group, head col % group)
        uint32_t qf[NT][W][4];  // [.][w][2 h + i]: fragment register i of k-step 2 w + h
        float qsum[NT][GR][2], to_log2[NT][2];
        int limit[NT][2];
        int least_limit = 0x7fffffff;
        {
            const T* q = reinterpret_cast<const T*>(p.q);
            const bool vec = ((reinterpret_cast<uintptr_t>(q) & 15) == 0) && p.q_st % 8 == 0 && p.q_sh % 8 == 0;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int col = ct * Cfg::COLS + nt * 8 + g;
                const bool on = col < count * p.group;
                const int token = col / p.group, head = kvh * p.group + (col - token * p.group);
                const T* row = q + (int64_t)(first_s[b] + token) * p.q_st + (int64_t)head * p.q_sh + 8 * t;
                uint4 raw[W];
                float top = 0.f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    raw[w] = on ? load_q8(row + 32 * w, vec) : make_uint4(0, 0, 0, 0);
                    const T* e = reinterpret_cast<const T*>(&raw[w]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(Cvt<T>::to_f(e[i])));
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e2 = max(-100, (int)(__float_as_uint(top) >> 23) - 127);  // the row is carried below 2^15 (up to 128: infinities)
                const float up = q_mul * __uint_as_float((uint32_t)(127 + 14 - e2) << 23);
#pragma unroll
                for (int gr = 0; gr < GR; ++gr) {
                    float sum = 0.f;
#pragma unroll
                    for (int w = 2 * gr; w < 2 * gr + 2; ++w) {
                        float x[8];
                        const T* e = reinterpret_cast<const T*>(&raw[w]);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            x[i] = Cvt<T>::to_f(e[i]) * up;
                            sum += x[i];
                            if (i & 1) x[i] *= 0x1p-4f;  // odd codes are 16 times as heavy as they should be
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int i = 0; i < 2; ++i) qf[nt][w][2 * h + i] = ptx::pack2<__half>(x[2 * h + i], x[2 * h + i + 4]);
                    }
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
                    for (int c = 0; c < 2; ++c) qsum[nt][gr][c] = 0x1p-24f * __shfl_sync(0xffffffffu, sum, (2 * t + c) * 4);
                }
                const float back = fmaxf(scale_log2 * __uint_as_float((uint32_t)(127 - 20 + e2) << 23) * 0x1p30f, 1e-37f);
                const int lim = on ? len - count + token + 1 : 0x7fffffff;  // keys that the column sees
                least_limit = min(least_limit, lim);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    to_log2[nt][c] = __shfl_sync(0xffffffffu, back, (2 * t + c) * 4);
                    limit[nt][c] = __shfl_sync(0xffffffffu, lim, (2 * t + c) * 4);
                }
            }
            least_limit = __reduce_min_sync(0xffffffffu, least_limit);
        }
        // m: largest score; bar: what a score has to exceed for m to follow; use: the exponent's offset
        float m[NT][2], bar[NT][2], use[NT][2], l[NT][2], low[NT][GR][2], eight[NT][GR][4], acc[NT][2 * W][4];
        float v_exp = -40.f;               // of the values' scales so far: none exceeds 2^v_exp
        __half v_bar = __ushort_as_half(0);  // 2^v_exp
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                m[nt][c] = bar[nt][c] = -INFINITY;
                use[nt][c] = 7.f - v_exp;
                l[nt][c] = 0.f;
#pragma unroll
                for (int gr = 0; gr < GR; ++gr) low[nt][gr][c] = eight[nt][gr][c] = eight[nt][gr][2 + c] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < 2 * W; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nt][i][e] = 0.f;
        }

        const int seg_at = (int)(pos - my_start);  // of the range
        for (; done < seg_at + seg; ++done) {
            if (!__all_sync(0xffffffffu, wait_stage(&my_bars[stage], phase, abort_flag))) { ok = false; break; }
            const int hidden_tiles = my_hidden[stage];
#pragma unroll 1
            for (int k0 = 0; k0 < kBlockTiles; k0 += Cfg::KT) {
            constexpr int KT = Cfg::KT;
            const int key0 = (t0 + done - seg_at) * kBlockKeys + k0 * kTileTokens, hidden = hidden_tiles >> k0;
            const uint8_t* tile = my_ring + stage * Cfg::STAGE + k0 * Cfg::TILE;
            const bool masked = key0 + KT * kTileTokens > least_limit || hidden != 0;  // some key is not there for some column; uniform over the warp
            // ---- scores
            __half2 kp[KT][2][GR], vp[KT][2][GR];  // this lane's two keys' pairs
            uint32_t ka[KT][W], kb[KT][W];
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                const uint8_t* kr = tile + k * Cfg::TILE + g * (D / 2) + t * (D / 8);
                load_words<W>(kr, ka[k]);
                load_words<W>(kr + 4 * D, kb[k]);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    load_pairs<GR>(tile + k * Cfg::TILE + pair_at(D, 0, g + 8 * r, 0), kp[k][r]);
                    load_pairs<GR>(tile + k * Cfg::TILE + pair_at(D, 1, g + 8 * r, 0), vp[k][r]);
                }
            }
            float sc[KT][NT][4];
#pragma unroll
            for (int gr = 0; gr < GR; ++gr) {
                float d[KT][NT][4];
#pragma unroll
                for (int w = 2 * gr; w < 2 * gr + 2; ++w)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int k = 0; k < KT; ++k) {
                            const uint32_t ua = ka[k][w] >> (8 * h), ub = kb[k][w] >> (8 * h);
                            const uint32_t a0 = ua & 0x000f000fu, a1 = ub & 0x000f000fu, a2 = ua & 0x00f000f0u, a3 = ub & 0x00f000f0u;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                if (w == 2 * gr && h == 0) ptx::mma_f16_16816_first(d[k][nt], a0, a1, a2, a3, qf[nt][w][0], qf[nt][w][1]);
                                else ptx::mma_f16_16816(d[k][nt], a0, a1, a2, a3, qf[nt][w][2 * h], qf[nt][w][2 * h + 1]);
                            }
                        }
#pragma unroll
                for (int k = 0; k < KT; ++k) {
                    const float2 pa = __half22float2(kp[k][0][gr]), pb = __half22float2(kp[k][1][gr]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int r = 0; r < 4; r += 2) {
                            const float least = r ? pb.y : pa.y, scale = r ? pb.x : pa.x;
#pragma unroll
                            for (int c = 0; c < 2; ++c) {  // (packed pairs would need both factors twice)
                                const float low = gr == 0 ? least * qsum[nt][gr][c] : fmaf(least, qsum[nt][gr][c], sc[k][nt][r + c]);
                                sc[k][nt][r + c] = fmaf(scale, d[k][nt][r + c], low);
                            }
                        }
                }
            }
            uint32_t seen = 0xffffffffu;  // a bit per (tile, column tile, element)
            if (masked) {
#pragma unroll
                for (int k = 0; k < KT; ++k) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const bool there = ((hidden >> k) & 1) == 0 && key0 + k * kTileTokens + g + 8 * r < len;
#pragma unroll
                        for (int gr = 0; gr < GR; ++gr) vp[k][r][gr] = there ? vp[k][r][gr] : __half2half2(__ushort_as_half(0));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 2; ++c)
                                if (!(there && key0 + k * kTileTokens + g + 8 * r < limit[nt][c])) {
                                    seen &= ~(1u << ((k * NT + nt) * 4 + 2 * r + c));
                                    sc[k][nt][2 * r + c] = -INFINITY;
                                }
                    }
                }
            }
            // ---- softmax
            float mx[NT][2];
            bool grow = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    mx[nt][c] = fmaxf(sc[0][nt][c], sc[0][nt][2 + c]);
                    if (KT == 2) mx[nt][c] = ptx::fmax3(mx[nt][c], sc[KT - 1][nt][c], sc[KT - 1][nt][2 + c]);
                    grow = grow || mx[nt][c] > bar[nt][c];
                }
            __half2 v_top = __half2half2(__ushort_as_half(0));  // largest scale of the values (low half; their size, should one be negative)
#pragma unroll
            for (int k = 0; k < KT; ++k)
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int gr = 0; gr < GR; ++gr) v_top = __hmax2(v_top, __habs2(vp[k][r][gr]));
            grow = grow || __hgt(__low2half(v_top), v_bar);
            if (__any_sync(0xffffffffu, grow)) {
                float v_new = v_exp;
                {
                    float top = __low2float(v_top);
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    // the power of two above it; fp16's largest stands for 2^16
                    if (top > 0.f) v_new = fmaxf(v_exp, (float)((int)(__float_as_uint(top) >> 23) - 126));
                    v_bar = __float2half_rz(v_new < -24.f ? 0.f : __uint_as_float((uint32_t)(127 + (int)v_new) << 23));
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float top = mx[nt][c];
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        const float to = top > bar[nt][c] ? top : m[nt][c];
                        const float use_new = (to == -INFINITY ? 7.f : fmaf(-to, to_log2[nt][c], 7.f)) - v_new;
                        const float alpha = m[nt][c] == -INFINITY ? 1.f : ptx::ex2_approx(use_new - use[nt][c]);
                        m[nt][c] = to;
                        bar[nt][c] = to == -INFINITY ? to : to + 8.f / to_log2[nt][c];
                        use[nt][c] = use_new;
                        l[nt][c] *= alpha;
#pragma unroll
                        for (int gr = 0; gr < GR; ++gr) {
                            low[nt][gr][c] *= alpha;
                            eight[nt][gr][c] *= alpha;
                        }
#pragma unroll
                        for (int i = 0; i < 2 * W; ++i) {
                            acc[nt][i][c] *= alpha;
                            acc[nt][i][2 + c] *= alpha;
                        }
                    }
                v_exp = v_new;
            }
            float pr[KT][NT][4];
#pragma unroll
            for (int k = 0; k < KT; ++k)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            pr[k][nt][r + c] = ptx::ex2_approx(fmaf(sc[k][nt][r + c], to_log2[nt][c], use[nt][c]));
                            l[nt][c] += pr[k][nt][r + c];
                        }
                    }
            // ---- output
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                uint32_t v[4][GR];
#pragma unroll
                for (int c = 0; c < 4; ++c) load_words<GR>(tile + k * Cfg::TILE + 8 * D + (4 * c + t) * (D / 2) + (g ^ (2 * t)) * (D / 16), v[c]);
#pragma unroll
                for (int gr = 0; gr < GR; ++gr) {
                    const float2 pa = __half22float2(vp[k][0][gr]), pb = __half22float2(vp[k][1][gr]);
                    const float mid_a = fmaf(8.f, pa.x, pa.y), mid_b = fmaf(8.f, pb.x, pb.y);
                    uint32_t f[NT][2];  // [.][keys 0-7, 8-15]
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float w[4], y[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            w[x] = pr[k][nt][x] * ((x & 2) ? pb.x : pa.x);
                            y[x] = pr[k][nt][x] * ((x & 2) ? mid_b : mid_a);
                        }
                        if (masked) {  // (a key may be there for one column and hidden, with NaN in its values, for another)
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                if (!((seen >> ((k * NT + nt) * 4 + x)) & 1u)) w[x] = y[x] = 0.f;
                        }
#pragma unroll
                        for (int c = 0; c < 2; ++c) low[nt][gr][c] += y[c] + y[2 + c];
#pragma unroll
                        for (int r = 0; r < 2; ++r) f[nt][r] = ptx::transpose_8x8(ptx::pack2<__half>(w[2 * r], w[2 * r + 1]));
                        ptx::mma_f16_16816(eight[nt][gr], kEight, kEight, kEight, kEight, f[nt][0], f[nt][1]);
                    }
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t u01 = __byte_perm(v[0][gr], v[1][gr], half ? 0x7632 : 0x5410);
                        const uint32_t u23 = __byte_perm(v[2][gr], v[3][gr], half ? 0x7632 : 0x5410);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t x01 = u01 >> (8 * h), x23 = u23 >> (8 * h);
                            const uint32_t a0 = FINE ? (x01 * 16u) & 0x00f000f0u : x01 & 0x000f000fu, a2 = FINE ? (x23 * 16u) & 0x00f000f0u : x23 & 0x000f000fu;
                            const uint32_t a1 = x01 & 0x00f000f0u, a3 = x23 & 0x00f000f0u;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                ptx::mma_f16_16816(acc[nt][4 * gr + 2 * half + h], a0, a1, a2, a3, f[nt][0], f[nt][1]);
                        }
                    }
                }
            }
            }
            __syncwarp();  // every lane has read the stage
            issue(done + Cfg::STAGES, stage);
            if ((done & 7) == 7) {  // 8 sum w comes off
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int gr = 0; gr < GR; ++gr)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
#pragma unroll
                            for (int i = 4 * gr; i < 4 * gr + 4; ++i) {
                                acc[nt][i][c] -= eight[nt][gr][c];
                                acc[nt][i][2 + c] = fmaf(-kOddEight, eight[nt][gr][c], acc[nt][i][2 + c]);
                            }
                            eight[nt][gr][c] = eight[nt][gr][2 + c] = 0.f;
                        }
            }
            if (++stage == Cfg::STAGES) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (!ok) break;

        // ---- the unit's columns, or this range's part of them
        const bool whole = seg == n_blocks;
        const int at_end = t0 == 0 ? 1 : 0;  // a part: tail or head
        float* part = at_end ? reinterpret_cast<float*>(my_ring) : head_s + warp * Cfg::SLOT;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], o);
#pragma unroll
                    for (int gr = 0; gr < GR; ++gr) low[nt][gr][c] += __shfl_xor_sync(0xffffffffu, low[nt][gr][c], o);
                }
                const int col = nt * 8 + 2 * t + c;
                if (!whole && g == 0) ml_s[(at_end * kWarps + warp) * Cfg::COLS + col] = make_float2(m[nt][c] == -INFINITY ? m[nt][c] : -use[nt][c], l[nt][c]);
                const int pair = ct * Cfg::COLS + col, token = pair / p.group, head = kvh * p.group + (pair - token * p.group);
                T* out = reinterpret_cast<T*>(p.out) + ((int64_t)(first_s[b] + token) * p.heads + head) * D + 8 * g;
#pragma unroll
                for (int gr = 0; gr < GR; ++gr) {  // channels 64 gr + 8 g + {0 .. 7}: two of each of four blocks
                    float y[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        y[2 * i] = fmaf(acc[nt][4 * gr + i][c] - eight[nt][gr][c], kEven, low[nt][gr][c]);
                        y[2 * i + 1] = fmaf(acc[nt][4 * gr + i][2 + c] - kOddEight * eight[nt][gr][c], kOdd, low[nt][gr][c]);
                    }
                    if (whole) {
                        if (pair < count * p.group) store_row8<T>(out + 64 * gr, y, l[nt][c]);
                    } else {
                        float4* dst = reinterpret_cast<float4*>(part + col * Cfg::O_STRIDE + 64 * gr + 8 * g);
                        dst[0] = make_float4(y[0], y[1], y[2], y[3]);
                        dst[1] = make_float4(y[4], y[5], y[6], y[7]);
                    }
                }
            }
        if (!whole && at_end) {
            cut.tail = 1;
            cut.first = first_s[b]; cut.count = count; cut.kvh = kvh; cut.ct = ct;
            cut.parts = 1;
            while (sp.split && range_at(blockIdx.x + cut.parts) < pos + n_blocks) ++cut.parts;
        } else if (!whole) {
            cut.head = 1;
            cut.head_ends = t0 + seg == n_blocks;
        }
        pos += seg;
    }
    if (lane == 0) cut_s[warp] = cut;
    __syncthreads();
    if (*abort_flag) ok = false;

    // (Not earlier: with the next kernel's CTAs waiting in the places of those that are through, 256 sequences of 16 to 1000 took 83 us
    // instead of 74.)
    pdl_trigger();
    // ---- what the warps' cuts left: heads that belong to an earlier CTA's unit, then every tail with the heads behind it
    for (int a = -1; a < kWarps && ok; ++a) {
        if (a >= 0 && !cut_s[a].tail) continue;
        uint32_t heads = 0;
        bool ended = false;
        for (int w = a + 1; w < kWarps && !ended; ++w) {
            if (!cut_s[w].any) continue;
            if (!cut_s[w].head) break;
            heads |= 1u << w;
            ended = cut_s[w].head_ends != 0;
        }
        if (a < 0 && heads == 0) continue;
        const Cut u = cut_s[a < 0 ? 0 : a];
        const bool here = a >= 0 && ended;  // all of the unit
        const int64_t slot = 2 * (int64_t)blockIdx.x + (a >= 0 ? 1 : 0);
        const int cols = a >= 0 ? min(Cfg::COLS, u.count * p.group - u.ct * Cfg::COLS) : Cfg::COLS;
        for (int i = tid; i < cols * (D / 8); i += kWarps * 32) {
            const int col = i / (D / 8), ch = (i - col * (D / 8)) * 8;
            float mx = a >= 0 ? ml_s[(kWarps + a) * Cfg::COLS + col].x : -INFINITY;
            for (int w = 0; w < kWarps; ++w)
                if ((heads >> w) & 1) mx = fmaxf(mx, ml_s[w * Cfg::COLS + col].x);
            const float to = mx == -INFINITY ? 0.f : mx;
            float sum = 0.f, o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = 0.f;
#pragma unroll 1
            for (int w = a < 0 ? 0 : a; w < kWarps; ++w) {
                if (w != a && !((heads >> w) & 1)) continue;
                const float2 ml = ml_s[(w == a ? kWarps + w : w) * Cfg::COLS + col];
                const float f = ptx::ex2_approx(ml.x - to);
                sum = fmaf(ml.y, f, sum);
                const float* src = (w == a ? reinterpret_cast<const float*>(ring + w * (Cfg::STAGES * Cfg::STAGE)) : head_s + w * Cfg::SLOT) + col * Cfg::O_STRIDE + ch;
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = fmaf(src[e], f, o[e]);
            }
            if (here) {
                const int pair = u.ct * Cfg::COLS + col, token = pair / p.group, head = u.kvh * p.group + (pair - token * p.group);
                store_row8<T>(reinterpret_cast<T*>(p.out) + ((int64_t)(u.first + token) * p.heads + head) * D + ch, o, sum);
            } else {
                float4* dst = reinterpret_cast<float4*>(sp.parts + (slot * Cfg::COLS + col) * D + ch);
                dst[0] = make_float4(o[0], o[1], o[2], o[3]);
                dst[1] = make_float4(o[4], o[5], o[6], o[7]);
                if (ch == 0) reinterpret_cast<float2*>(sp.parts + (int64_t)2 * gridDim.x * Cfg::COLS * D)[slot * Cfg::COLS + col] = make_float2(mx, sum);
            }
        }
        if (a >= 0 && !here && tid == 0) *desc = {u.parts, u.first, u.count, u.kvh, u.ct, {0, 0, 0}};  // the unit goes on in the next ranges
    }
    if (!ok) {  // a copy did not arrive in time: what is in flight gets a bounded time to land before shared memory is given up
        if (tid == 0) atomicOr(&g_kv4_status[0], 1u);
        const uint64_t since = ptx::globaltimer_ns();
        while (ptx::globaltimer_ns() - since < 20000ull) {
        }
    }
}

// The parts of the unit that starts in range blockIdx.x and goes on in others: out = sum 2^(m_i - m) O_i / sum 2^(m_i - m) l_i. A CTA per
// range (some have nothing to do and leave), SPLIT warps per column that take the parts in turn: a sequence may fill every range, but
// mostly there are two or three. 512 threads, so that all CTAs fit the chip at once (1024: 9 us behind 64 sequences, this 6).
constexpr int kCombineThreads = 512;
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kCombineThreads, 3) kv4_combine_kernel(const SplitParams sp, int ranges) {
    using Cfg = SplitCfg<D, NT>;
    constexpr int WARPS = kCombineThreads / 32, SPLIT = WARPS / Cfg::COLS, C = D / 32;
    pdl_sync();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = warp / SPLIT;
    const float2* ml = reinterpret_cast<const float2*>(sp.parts + (int64_t)2 * ranges * Cfg::COLS * D);
    auto slot = [&](int i) { return (2 * ((int64_t)blockIdx.x + i) + (i == 0 ? 1 : 0)) * Cfg::COLS + col; };
    // (what the first parts would be is fetched along with the word that says how many there are)
    const bool in = (int)blockIdx.x + lane < ranges;
    const float2 mine = in ? ml[slot(lane)] : make_float2(-INFINITY, 0.f);
    const PartDesc d = reinterpret_cast<const PartDesc*>(sp.parts + (int64_t)2 * ranges * Cfg::part_floats())[blockIdx.x];
    if (d.parts == 0) return;
    __shared__ __align__(16) float o_s[WARPS][D];
    __shared__ float l_s[WARPS];
    float m = lane < d.parts ? mine.x : -INFINITY, l = 0.f, o[C];
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = 0.f;
    if (d.ct * Cfg::COLS + col < d.count * sp.a.group) {
        for (int i = 32 + lane; i < d.parts; i += 32) m = fmaxf(m, ml[slot(i)].x);
        m = warp_max(m);
        const float use = m == -INFINITY ? 0.f : m;
        constexpr int AHEAD = D == 256 ? 2 : 4;  // parts in flight
#pragma unroll 1
        for (int i0 = warp % SPLIT; i0 < d.parts; i0 += AHEAD * SPLIT) {
            float v[AHEAD][C];
            float2 part[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int i = i0 + j * SPLIT;
                const float x = __shfl_sync(0xffffffffu, mine.x, i & 31), y = __shfl_sync(0xffffffffu, mine.y, i & 31);
                part[j] = make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int c = 0; c < C; ++c) v[j][c] = 0.f;
                if (i < d.parts) {
                    part[j] = i < 32 ? make_float2(x, y) : ml[slot(i)];
#pragma unroll
                    for (int c = 0; c < C; ++c) v[j][c] = sp.parts[slot(i) * D + c * 32 + lane];
                }
            }
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const float f = ptx::ex2_approx(part[j].x - use);
                l = fmaf(part[j].y, f, l);
#pragma unroll
                for (int c = 0; c < C; ++c) o[c] = fmaf(v[j][c], f, o[c]);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) o_s[warp][c * 32 + lane] = o[c];
    if (lane == 0) l_s[warp] = l;
    __syncthreads();
    for (int i = threadIdx.x; i < Cfg::COLS * (D / 8); i += kCombineThreads) {
        const int at = i / (D / 8), ch = (i - at * (D / 8)) * 8, pair = d.ct * Cfg::COLS + at;
        if (pair >= d.count * sp.a.group) break;
        float sum = 0.f, y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = 0.f;
#pragma unroll
        for (int w = at * SPLIT; w < (at + 1) * SPLIT; ++w) {
            sum += l_s[w];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] += o_s[w][ch + e];
        }
        const int token = pair / sp.a.group, head = d.kvh * sp.a.group + (pair - token * sp.a.group);
        store_row8<T>(reinterpret_cast<T*>(sp.a.out) + ((int64_t)(d.first + token) * sp.a.heads + head) * D + ch, y, sum);
    }
}

constexpr int kSmSharedBytes = 233472;

template <typename T, int D, int NT>
int launch_split(SplitParams sp, cudaStream_t st) {
    using Cfg = SplitCfg<D, NT>;
    static std::atomic<uint64_t> reserved;
    if (!reserve_smem(kv4_split_kernel<T, D, NT>, Cfg::smem(kMaxBatch), reserved)) return fail(XG_ERR_LAUNCH, "xg_kv4_attention: cannot reserve shared memory");
    const int bytes = Cfg::smem(sp.a.batch), fit = kSmSharedBytes / (bytes + 1024);
    const int grid = num_sms() * (fit < Cfg::CTAS ? fit : Cfg::CTAS);  // all resident
    launch(kv4_split_kernel<T, D, NT>, (unsigned)grid, kWarps * 32, (size_t)bytes, st, sp);
    if (const int rc = check_launch("xg_kv4_attention")) return rc;
    if (!sp.split) return XG_OK;
    launch(kv4_combine_kernel<T, D, NT>, (unsigned)grid, kCombineThreads, 0, st, sp, grid);
    return check_launch("xg_kv4_attention");
}

// Columns per unit: what the sequences bring, 16 where they bring more than 8, but three units of 8 rather than two of 16 where that
// holds them (8 sequences of 8192 to 16384, 8 kv heads of 128, 24 columns: 84 us, with two of 16 90; 16 columns in one of 16 55 us, in
// two of 8 63). D = 256 has no registers for 16.
constexpr int columns(int64_t D, int64_t max_q, int64_t group) { return D == 256 || max_q * group <= 8 || (max_q * group + 7) / 8 == 3 ? 8 : 16; }

// Whether units are cut over CTAs. Left whole, they need no second launch, but the CTAs' loads differ by a unit. (us, whole / cut, 32 / 8
// heads of 128) 1 sequence of 512 11.0 / 11.8, 512 of 512 83 / 86, 256 of 16 to 1000 69 / 74; 64 of 1024 34 / 32, 128 of 1400 66 / 59.
bool cut(int64_t D, int64_t cols, int64_t units, int64_t max_len) {
    return max_len > 1024 || (max_len > 512 && units < 2LL * num_sms() * split_ctas((int)D, (int)cols / 8));
}

int64_t split_workspace(int64_t D, int64_t max_q, int64_t group, int64_t max_len, int64_t batch, int64_t kv_heads) {
    const int64_t cols = columns(D, max_q, group), ctas = (int64_t)num_sms() * split_ctas((int)D, (int)cols / 8);
    if (!cut(D, cols, batch * kv_heads, max_len)) return 0;
    return 2 * ctas * cols * (D + 2) * 4 + ctas * (int64_t)sizeof(PartDesc);
}

// Sequences with more columns (new token, head of the group) than this go to the tensor-memory kernel: streaming unpacks the keys once
// per 16 columns (8 at head dim 256), the other once per 256 (128). (us, streamed / tiles, 8 kv heads) D = 128: 64 sequences of 4096, 32
// columns 211 / 304, 36 307 / 303; 1 of 16000, 32 columns 31 / 32, 36 37 / 32. D = 64, where a tile's products are shorter than its
// softmax: 64 of 4096, 64 columns 237 / 262, 72 291 / 260. D = 256: 32 of 2000, 48 columns 199 / 185, 1 of 16000, 48 63 / 61, 40 56 / 60.
constexpr int most_streamed(int64_t D) { return D == 64 ? 64 : (D == 128 ? 32 : 40); }
constexpr bool in_tiles(int64_t D, int64_t max_q, int64_t group) { return max_q * group > most_streamed(D); }

template <typename T>
int attend_split(const AttendParams& whole, int64_t D, int64_t max_q, int most_cols, void* workspace, cudaStream_t st) {
    const int64_t max_len = (int64_t)whole.table_pages * whole.cache.tiles * kTileTokens;
    const int cols = columns(D, max_q, whole.group);
    // blocks of a launch are counted in 32 bits
    const int64_t most = whole.tokens * whole.group < most_cols ? whole.tokens * whole.group : most_cols;
    const int64_t blocks = (int64_t)whole.cache.heads * ((most + cols - 1) / cols) * ((max_len + kBlockKeys - 1) / kBlockKeys);
    const int64_t fit = blocks > 0 ? 0x7fffffffLL / blocks : kMaxBatch;
    if (fit < 1) return fail(XG_ERR_TOO_LARGE, "xg_kv4_attention: too many rows and keys in one sequence");
    const int chunk = (int)(fit < kMaxBatch ? fit : kMaxBatch);
    for (int at = 0; at == 0 || at < whole.batch; at += chunk) {
        SplitParams sp = {};
        sp.a = whole;
        sp.a.batch = whole.batch - at < chunk ? whole.batch - at : chunk;
        sp.a.table += (int64_t)at * whole.table_stride;
        sp.a.lens += at;
        if (whole.starts) sp.a.starts += at;
        else sp.a.row0 = at;
        sp.parts = static_cast<float*>(workspace);
        sp.split = cut(D, cols, (int64_t)whole.batch * whole.cache.heads, max_len);
        sp.min_blocks = 8;
        sp.most_cols = most_cols;
        sp.first_rows = at == 0;
        sp.last_rows = at + chunk >= whole.batch;
        int rc;
        if (D == 64) rc = cols == 8 ? launch_split<T, 64, 1>(sp, st) : launch_split<T, 64, 2>(sp, st);
        else if (D == 128) rc = cols == 8 ? launch_split<T, 128, 1>(sp, st) : launch_split<T, 128, 2>(sp, st);
        else rc = launch_split<T, 256, 1>(sp, st);
        if (rc != XG_OK) return rc;
    }
    return XG_OK;
}

}  // namespace

int read_kv4_status(unsigned int* host_out, int reset) {
    unsigned int v[4] = {0, 0, 0, 0};
    if (cudaMemcpyFromSymbol(v, g_kv4_status, sizeof(v)) != cudaSuccess) {
        cudaGetLastError();
        return fail(XG_ERR_DEVICE, "xg_tc_status: cannot read device status");
    }
    *host_out = v[0];
    unsigned int more = 0;
    if (const int rc = read_kv4_prefill_status(&more, reset)) return rc;
    *host_out |= more << 1;
    if (reset && v[0] != 0) {
        unsigned int z[4] = {0, 0, 0, 0};
        cudaMemcpyToSymbol(g_kv4_status, z, sizeof(z));
    }
    return XG_OK;
}
}  // namespace xg

extern "C" int64_t xg_kv4_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t D, int64_t max_q,
                                                    int64_t max_len) {
    using namespace xg;
    if (tokens <= 0 || batch <= 0 || q_heads <= 0 || kv_heads <= 0 || max_q < 0 || max_len < 0) return 0;
    const int64_t group = q_heads / kv_heads, streamed = split_workspace(D, max_q, group, max_len, batch, kv_heads);
    const int64_t tiles = in_tiles(D, max_q, group) ? prefill_workspace(tokens, batch, group, kv_heads, D, max_len) : 0;
    return streamed > tiles ? streamed : tiles;  // (used one after the other)
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
    if (tokens * (q_heads / kv_heads) > 0x7fffff00LL) return fail(XG_ERR_TOO_LARGE, "xg_kv4_attention: 2^31 rows per kv head or more");
    if (table_pages * page_size > 0x7fffff00LL) return fail(XG_ERR_TOO_LARGE, "xg_kv4_attention: more than 2^31 tokens per sequence");
    if (tokens == 0) return XG_OK;
    if (!q_starts && batch > tokens) return fail(XG_ERR_INVALID_ARG, "xg_kv4_attention: %lld sequences without q_starts need a row each, there are %lld",
                                                 (long long)batch, (long long)tokens);
    if (!q || !out || (batch > 0 && (!kv_lens || (table_pages > 0 && !page_table)))) return fail(XG_ERR_INVALID_ARG, "xg_kv4_attention: null pointer");
    if (!aligned16(out)) return fail(XG_ERR_INVALID_ARG, "xg_kv4_attention: the result must be 16-byte aligned");
    AttendParams p = {};
    p.cache = {static_cast<const uint8_t*>(cache), pages, page_stride, (int)kv_heads, (int)(page_size / 16)};
    p.q = q; p.out = out; p.table = page_table; p.lens = kv_lens; p.starts = q_starts;
    p.q_st = q_stride_t; p.q_sh = q_stride_h; p.table_stride = table_stride;
    p.tokens = tokens; p.batch = (int)batch; p.heads = (int)q_heads; p.group = (int)(q_heads / kv_heads); p.table_pages = (int)table_pages;
    p.scale = scale;
    const int64_t need = xg_kv4_attention_workspace_bytes(tokens, batch, q_heads, kv_heads, D, max_q, table_pages * page_size);
    if (workspace_bytes < need || (need > 0 && (!workspace || !aligned16(workspace))))
        return fail(XG_ERR_INVALID_ARG, "xg_kv4_attention: needs %lld bytes of 16-byte aligned workspace", (long long)need);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    // Sequences with many columns go to the tensor-memory kernel, where there may be any; the others to the streaming one. A sequence
    // on its own goes there whatever it turns out to be, which saves the other's launches (512 new tokens: 20.6 us, with them 23.3).
    const bool tiles = batch > 0 && in_tiles(D, max_q, p.group);
    if (tiles && batch == 1) return attend_prefill(p, D, dtype, 0, workspace, st);
    const int most = tiles ? most_streamed(D) : 0x7fffffff;
    const int rc = dtype == XG_BF16 ? attend_split<__nv_bfloat16>(p, D, max_q, most, workspace, st) : attend_split<__half>(p, D, max_q, most, workspace, st);
    return rc != XG_OK || !tiles ? rc : attend_prefill(p, D, dtype, most, workspace, st);
}
