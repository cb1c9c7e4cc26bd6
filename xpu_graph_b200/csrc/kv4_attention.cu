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
// head. The tiles of 16 keys of all units form one line, cut into equal ranges, one per CTA, so that sequences of any mixture of
// lengths load the chip evenly; what a unit leaves in several CTAs is added by kv4_combine_kernel in range order. A CTA's warps take
// its tiles in turn, each warp with a ring of bulk copies of its own.
//
// Both products run on mma.m16n8k16 with the codes as bf16: a 4-bit code n masked out of its word is the bf16 subnormal n 2^-133 in
// bits 0-3 and n 2^-129 in bits 4-7 (8 and up carry over into the exponent as they should), which the tensor core multiplies
// exactly, so unpacking costs one logic operation per two codes and no arithmetic. q and the probabilities carry 2^64 along.
//   scores (16 keys x 8 columns, per group of 64 channels):  x = scale_k acc + least_k sum(q), the group's sum of q kept per column
//   output (16 channels x 8 columns):  acc += code (p scale_v), and the sum of p least_v per column and group beside it
// p scale_v goes in as two bf16 planes (16 bits of significand), q as one for bf16 and two for fp16 (exact).
// The maximum is kept per column and may lag behind by 2^8; only a larger step rescales the sums.
// The codes of keys that do not exist are finite whatever they are; their scales are dropped by a select, not a product.
constexpr int kWarps = 4, kStages = 3;
constexpr int kBlockTiles = 2, kBlockKeys = kBlockTiles * kTileTokens;  // what a stage holds
constexpr int kMaxBatch = 1024;  // sequences per launch: their prefix sums live in shared memory

// CTAs per SM, by what the fragments and sums take of the register file
constexpr int split_ctas(int D, int NT) { return D == 256 ? 2 : (NT == 1 ? (D == 64 ? 4 : 3) : (D == 64 ? 3 : 2)); }

template <int D, int NT>
struct SplitCfg {
    static constexpr int COLS = 8 * NT;
    static constexpr int TILE = tile_bytes(D);
    static constexpr int STAGE = kBlockTiles * TILE;
    static constexpr int STAGES = D == 256 ? 2 : kStages;
    static constexpr int KT = NT == 1 && D <= 128 ? 2 : 1;  // tiles in work at once: more independent products per warp, more registers
    static constexpr int RING = kWarps * STAGES * STAGE;
    static constexpr int O_STRIDE = D + 4;  // floats
    static constexpr int O_BYTES = kWarps * COLS * O_STRIDE * 4;
    static constexpr int ML_BYTES = kWarps * COLS * 2 * 4;
    static constexpr int BAR_BYTES = kWarps * STAGES * 8;
    static constexpr int FIXED = RING + O_BYTES + ML_BYTES + BAR_BYTES + kWarps * STAGES * 4 + 64;
    static constexpr int part_floats() { return COLS * (D + 2); }
    static int smem(int batch) { return FIXED + (batch + 1) * 8 + batch * 12; }
    static constexpr int CTAS = split_ctas(D, NT);
};

struct SplitParams {
    AttendParams a;
    float* parts;  // [2 * gridDim.x][COLS][D] sums, then [2 * gridDim.x][COLS] (maximum, sum) pairs, then a PartDesc per CTA
    int split;         // 0: a unit stays in one CTA
    int64_t min_blocks; // of a range
    int most_cols;       // sequences with more columns are left alone
    int first_rows, last_rows;  // this launch zeroes the rows before the first / behind the last sequence
};

// What starts in a CTA's range and ends in a later one's.
struct PartDesc {
    int parts;  // 0: nothing
    int first, count, kvh, ct, pad[3];
};

template <typename T>
struct Planes {
    static constexpr int N = std::is_same<T, __nv_bfloat16>::value ? 1 : 2;
};

__device__ __forceinline__ float bf16_lo(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, (SplitCfg<D, NT>::CTAS)) kv4_split_kernel(const SplitParams sp) {
    using Cfg = SplitCfg<D, NT>;
    constexpr int W = D / 32, GR = D / 64, PL = Planes<T>::N;
    const AttendParams& p = sp.a;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* ring = smem;
    float* o_s = reinterpret_cast<float*>(smem + Cfg::RING);
    float2* ml_s = reinterpret_cast<float2*>(smem + Cfg::RING + Cfg::O_BYTES);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::RING + Cfg::O_BYTES + Cfg::ML_BYTES);
    int64_t* prefix = reinterpret_cast<int64_t*>(reinterpret_cast<uint8_t*>(bars) + Cfg::BAR_BYTES);  // [batch + 1]
    int* first_s = reinterpret_cast<int*>(prefix + p.batch + 1);
    int* count_s = first_s + p.batch;
    int* len_s = count_s + p.batch;
    volatile int* hidden_s = len_s + p.batch;  // [kWarps][STAGES], a bit per tile
    volatile int* abort_flag = hidden_s + kWarps * Cfg::STAGES;
    int64_t* scan_s = reinterpret_cast<int64_t*>(o_s);  // before the first segment only

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    if (tid == 0) {
        for (int i = 0; i < kWarps * Cfg::STAGES; ++i) ptx::mbar_init(&bars[i], 1);
        *abort_flag = 0;
        ptx::fence_mbar_init();
        ptx::fence_proxy_async();
    }
    pdl_sync();

    // ---- the line of tiles
    const int kv_heads = p.cache.heads;
    auto col_tiles = [&](int count) { return (count * p.group + Cfg::COLS - 1) / Cfg::COLS; };
    auto blocks_of = [&](int b) { return (len_s[b] + kBlockKeys - 1) / kBlockKeys; };
    int64_t carry = 0;
    for (int base = 0; base < p.batch; base += kWarps * 32) {
        const int b = base + tid;
        int64_t w = 0;
        if (b < p.batch) {
            const Sequence s = sequence(p, b);
            first_s[b] = (int)s.first;
            count_s[b] = s.count;
            const int len = s.count * p.group > sp.most_cols ? -1 : (int)s.len;
            len_s[b] = len;
            w = (int64_t)kv_heads * col_tiles(s.count) * ((max(len, 0) + kBlockKeys - 1) / kBlockKeys);
        }
        int64_t inc = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) scan_s[warp] = inc;
        __syncthreads();
        int64_t before = carry, all = carry;
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
    const int64_t total = carry;

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

    int64_t ranges = (total + sp.min_blocks - 1) / sp.min_blocks;
    if (ranges > gridDim.x) ranges = gridDim.x;
    int64_t start = 0, end = 0;
    auto sequence_at = [&](int64_t x) {  // the b with prefix[b] <= x < prefix[b + 1]
        int lo = 0, hi = p.batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (prefix[mid] <= x) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    if ((int64_t)blockIdx.x < ranges) {
        start = total * blockIdx.x / ranges;
        end = total * (blockIdx.x + 1) / ranges;
        if (!sp.split) {
            auto up = [&](int64_t x) {
                if (x >= total) return total;
                const int b = sequence_at(x);
                const int64_t n = blocks_of(b), off = x - prefix[b];
                return prefix[b] + (off + n - 1) / n * n;
            };
            start = up(start);
            end = up(end);
        }
    }
    PartDesc* desc = reinterpret_cast<PartDesc*>(sp.parts + (int64_t)2 * gridDim.x * Cfg::part_floats()) + blockIdx.x;
    if (sp.split && tid == 0) desc->parts = 0;
    if (start >= end) return;

    // ---- this warp's tiles: start + warp + 4 i
    const int mine = (int)((end - start - warp + kWarps - 1) / kWarps);
    uint8_t* my_ring = ring + warp * (Cfg::STAGES * Cfg::STAGE);
    uint64_t* my_bars = bars + warp * Cfg::STAGES;
    volatile int* my_hidden = hidden_s + warp * Cfg::STAGES;
    // where this lane's block of the current batch of 32 lies, tile by tile; 0 where there is nothing to read
    int64_t addr[kBlockTiles] = {};
    auto look_up = [&](int i) {
        const int64_t x = start + warp + (int64_t)kWarps * (i + lane);
#pragma unroll
        for (int k = 0; k < kBlockTiles; ++k) addr[k] = 0;
        if (x >= end) return;
        const int b = sequence_at(x);
        const int64_t n = blocks_of(b), off = x - prefix[b];
        const int64_t unit = off / n;
        const int kvh = (int)(unit / col_tiles(count_s[b]));
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

    // Scores stay in the units of the products (2^-69 / scale) up to the exponent; a negative scale goes into q, a zero one makes q zero.
    const float q_mul = p.scale > 0.f ? 1.f : (p.scale < 0.f ? -1.f : (p.scale == 0.f ? 0.f : p.scale));
    const float to_log2 = (p.scale != 0.f ? fabsf(p.scale) : 1.f) * kLog2e * 0x1p69f;
    const float step = 8.f / to_log2;
    int done = 0, stage = 0;  // tiles of this warp consumed, and the stage of the next one
    uint32_t phase = 0;
    bool ok = true;
    int b = sequence_at(start);
    for (int64_t pos = start; pos < end && ok;) {
        while (prefix[b + 1] <= pos) ++b;
        const int n_blocks = blocks_of(b), count = count_s[b], len = len_s[b];
        const int64_t off = pos - prefix[b];
        const int64_t unit = off / n_blocks;
        const int t0 = (int)(off - unit * n_blocks);  // blocks, as n_blocks and seg
        const int cts = col_tiles(count);
        const int kvh = (int)(unit / cts), ct = (int)(unit - (int64_t)kvh * cts);
        const int seg = (int)(n_blocks - t0 < end - pos ? n_blocks - t0 : end - pos);

        // ---- q as fragments; column n = 8 nt + g is the pair (new token col / group, head col % group)
        uint32_t qf[NT][PL][W][4];  // [.][.][w][2 h + i]: fragment register i of k-step 2 w + h
        float qsum[NT][GR][2];
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
#pragma unroll
                for (int w = 0; w < W; ++w) raw[w] = on ? load_q8(row + 32 * w, vec) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int gr = 0; gr < GR; ++gr) {
                    float sum = 0.f;
#pragma unroll
                    for (int w = 2 * gr; w < 2 * gr + 2; ++w) {
                        float x[8];
                        const T* e = reinterpret_cast<const T*>(&raw[w]);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            x[i] = Cvt<T>::to_f(e[i]) * q_mul;
                            sum += x[i];
                            // odd codes are 16 times as heavy as they should be
                            x[i] *= (i & 1) ? 0x1p60f : 0x1p64f;
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const float lo = x[2 * h + i], hi = x[2 * h + i + 4];
                                const uint32_t top = ptx::pack2<__nv_bfloat16>(lo, hi);
                                qf[nt][0][w][2 * h + i] = top;
                                if (PL == 2) qf[nt][PL - 1][w][2 * h + i] = ptx::pack2<__nv_bfloat16>(lo - bf16_lo(top), hi - bf16_hi(top));
                            }
                    }
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
                    for (int c = 0; c < 2; ++c) qsum[nt][gr][c] = 0x1p-69f * __shfl_sync(0xffffffffu, sum, (2 * t + c) * 4);
                }
                const int lim = on ? len - count + token + 1 : 0x7fffffff;  // keys that the column sees
                least_limit = min(least_limit, lim);
#pragma unroll
                for (int c = 0; c < 2; ++c) limit[nt][c] = __shfl_sync(0xffffffffu, lim, (2 * t + c) * 4);
            }
            least_limit = __reduce_min_sync(0xffffffffu, least_limit);
        }
        // m: largest score; bar: what a score has to exceed for m to follow; use: the exponent's offset. Probabilities carry 2^64.
        float m[NT][2], bar[NT][2], use[NT][2], l[NT][2], low[NT][GR][2], acc[NT][2 * W][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                m[nt][c] = bar[nt][c] = -INFINITY;
                use[nt][c] = 64.f;
                l[nt][c] = 0.f;
#pragma unroll
                for (int gr = 0; gr < GR; ++gr) low[nt][gr][c] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < 2 * W; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nt][i][e] = 0.f;
        }

        // KT tiles; MASKED: some key of theirs is not there for some column
        auto work = [&](const uint8_t* tile, const int key0, const int hidden, auto masked) {
            constexpr bool MASKED = decltype(masked)::value;
            constexpr int KT = Cfg::KT;
            // ---- scores
            __half2 kp[KT][2][GR];  // this lane's two keys' pairs
            uint32_t ka[KT][W], kb[KT][W];
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                const uint8_t* kr = tile + k * Cfg::TILE + g * (D / 2) + t * (D / 8);
                load_words<W>(kr, ka[k]);
                load_words<W>(kr + 4 * D, kb[k]);
#pragma unroll
                for (int r = 0; r < 2; ++r) load_pairs<GR>(tile + k * Cfg::TILE + pair_at(D, 0, g + 8 * r, 0), kp[k][r]);
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
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int pl = 0; pl < PL; ++pl) {
                                    if (w == 2 * gr && h == 0 && pl == 0) ptx::mma_bf16_16816_first(d[k][nt], a0, a1, a2, a3, qf[nt][pl][w][0], qf[nt][pl][w][1]);
                                    else ptx::mma_bf16_16816(d[k][nt], a0, a1, a2, a3, qf[nt][pl][w][2 * h], qf[nt][pl][w][2 * h + 1]);
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
            auto visible = [&](int k, int nt, int e) {
                return ((hidden >> k) & 1) == 0 && key0 + k * kTileTokens + g + (e & 2) * 4 < limit[nt][e & 1];
            };
            if (MASKED) {
#pragma unroll
                for (int k = 0; k < KT; ++k)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!visible(k, nt, e)) sc[k][nt][e] = -INFINITY;
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
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float top = mx[nt][c];
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        const float to = fmaxf(m[nt][c], top);
                        const float alpha = to == -INFINITY ? 1.f : ptx::ex2_approx((m[nt][c] - to) * to_log2);
                        m[nt][c] = to;
                        bar[nt][c] = to + step;
                        use[nt][c] = to == -INFINITY ? 64.f : fmaf(-to, to_log2, 64.f);
                        l[nt][c] *= alpha;
#pragma unroll
                        for (int gr = 0; gr < GR; ++gr) low[nt][gr][c] *= alpha;
#pragma unroll
                        for (int i = 0; i < 2 * W; ++i) {
                            acc[nt][i][c] *= alpha;
                            acc[nt][i][2 + c] *= alpha;
                        }
                    }
            }
            float pr[KT][NT][4];
#pragma unroll
            for (int k = 0; k < KT; ++k)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        float x0, x1;
                        ptx::fma2(x0, x1, sc[k][nt][r], sc[k][nt][r + 1], to_log2, to_log2, use[nt][0], use[nt][1]);
                        pr[k][nt][r] = ptx::ex2_approx(x0);
                        pr[k][nt][r + 1] = ptx::ex2_approx(x1);
                        ptx::add2(l[nt][0], l[nt][1], l[nt][0], l[nt][1], pr[k][nt][r], pr[k][nt][r + 1]);
                    }
            // ---- output
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                uint32_t v[4][GR];
                __half2 vp[2][GR];
#pragma unroll
                for (int c = 0; c < 4; ++c) load_words<GR>(tile + k * Cfg::TILE + 8 * D + (4 * c + t) * (D / 2) + (g ^ (2 * t)) * (D / 16), v[c]);
#pragma unroll
                for (int r = 0; r < 2; ++r) load_pairs<GR>(tile + k * Cfg::TILE + pair_at(D, 1, g + 8 * r, 0), vp[r]);
#pragma unroll
                for (int gr = 0; gr < GR; ++gr) {
                    const float2 pa = __half22float2(vp[0][gr]), pb = __half22float2(vp[1][gr]);
                    uint32_t f[NT][2][2];  // [.][plane][keys 0-7, 8-15]
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float w[4];
                        if (MASKED) {  // (a hidden key's scale may be anything)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const bool on = visible(k, nt, e);
                                w[e] = on ? pr[k][nt][e] * ((e & 2) ? pb.x : pa.x) : 0.f;
                                low[nt][gr][e & 1] += on ? pr[k][nt][e] * ((e & 2) ? pb.y : pa.y) : 0.f;
                            }
                        } else {
#pragma unroll
                            for (int r = 0; r < 4; r += 2) {
                                const float least = r ? pb.y : pa.y, scale = r ? pb.x : pa.x;
#pragma unroll
                                for (int c = 0; c < 2; ++c) {
                                    w[r + c] = pr[k][nt][r + c] * scale;
                                    low[nt][gr][c] = fmaf(pr[k][nt][r + c], least, low[nt][gr][c]);
                                }
                            }
                        }
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const uint32_t top = ptx::pack2<__nv_bfloat16>(w[2 * r], w[2 * r + 1]);
                            const uint32_t rest = ptx::pack2<__nv_bfloat16>(w[2 * r] - bf16_lo(top), w[2 * r + 1] - bf16_hi(top));
                            f[nt][0][r] = ptx::transpose_8x8(top);
                            f[nt][1][r] = ptx::transpose_8x8(rest);
                        }
                    }
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t u01 = __byte_perm(v[0][gr], v[1][gr], half ? 0x7632 : 0x5410);
                        const uint32_t u23 = __byte_perm(v[2][gr], v[3][gr], half ? 0x7632 : 0x5410);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t x01 = u01 >> (8 * h), x23 = u23 >> (8 * h);
                            const uint32_t a0 = x01 & 0x000f000fu, a1 = x01 & 0x00f000f0u, a2 = x23 & 0x000f000fu, a3 = x23 & 0x00f000f0u;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int pl = 0; pl < 2; ++pl)
                                    ptx::mma_bf16_16816(acc[nt][4 * gr + 2 * half + h], a0, a1, a2, a3, f[nt][pl][0], f[nt][pl][1]);
                        }
                    }
                }
            }
        };
        const int seg_at = (int)(pos - start);  // of the range
        for (int at = warp + kWarps * done - seg_at; at < seg; at += kWarps) {
            if (!__all_sync(0xffffffffu, wait_stage(&my_bars[stage], phase, abort_flag))) { ok = false; break; }
            const int hidden = my_hidden[stage];
#pragma unroll 1
            for (int k0 = 0; k0 < kBlockTiles; k0 += Cfg::KT) {
                const int key0 = (t0 + at) * kBlockKeys + k0 * kTileTokens;
                const uint8_t* tile = my_ring + stage * Cfg::STAGE + k0 * Cfg::TILE;
                if (key0 + Cfg::KT * kTileTokens > least_limit || (hidden >> k0) != 0) work(tile, key0, hidden >> k0, std::true_type{});  // uniform over the warp
                else work(tile, key0, 0, std::false_type{});
            }
            __syncwarp();  // every lane has read the stage
            issue(done + Cfg::STAGES, stage);
            ++done;
            if (++stage == Cfg::STAGES) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (!ok) break;

        // ---- the warps' sums of this segment together
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
                if (g == 0) ml_s[warp * Cfg::COLS + nt * 8 + 2 * t + c] = make_float2(m[nt][c] * to_log2, l[nt][c]);
#pragma unroll
                for (int i = 0; i < 2 * W; ++i) {  // block i: channels 64 (i / 4) + 8 g + 2 (i % 4) + {0, 1}
                    const float base = low[nt][i / 4][c];
                    const float2 y = make_float2(fmaf(acc[nt][i][c] * 0x1p69f, 0x1p64f, base), fmaf(acc[nt][i][2 + c] * 0x1p65f, 0x1p64f, base));
                    *reinterpret_cast<float2*>(o_s + (warp * Cfg::COLS + nt * 8 + 2 * t + c) * Cfg::O_STRIDE + 64 * (i / 4) + 8 * g + 2 * (i & 3)) = y;
                }
            }
        __syncthreads();
        if (*abort_flag) { ok = false; break; }
        const bool whole = seg == n_blocks;
        const int64_t slot = 2 * (int64_t)blockIdx.x + (t0 == 0 ? 1 : 0);
        const int cols = min(Cfg::COLS, count * p.group - ct * Cfg::COLS);
        for (int i = tid; i < cols * (D / 8); i += kWarps * 32) {
            const int col = i / (D / 8), ch = (i - col * (D / 8)) * 8;
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, ml_s[w * Cfg::COLS + col].x);
            const float use = mx == -INFINITY ? 0.f : mx;
            float sum = 0.f, o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float2 part = ml_s[w * Cfg::COLS + col];
                const float f = ptx::ex2_approx(part.x - use);
                sum = fmaf(part.y, f, sum);
                const float4* src = reinterpret_cast<const float4*>(o_s + (w * Cfg::COLS + col) * Cfg::O_STRIDE + ch);
                const float4 a = src[0], c = src[1];
                o[0] = fmaf(a.x, f, o[0]); o[1] = fmaf(a.y, f, o[1]); o[2] = fmaf(a.z, f, o[2]); o[3] = fmaf(a.w, f, o[3]);
                o[4] = fmaf(c.x, f, o[4]); o[5] = fmaf(c.y, f, o[5]); o[6] = fmaf(c.z, f, o[6]); o[7] = fmaf(c.w, f, o[7]);
            }
            if (whole) {
                const int at = ct * Cfg::COLS + col, token = at / p.group, head = kvh * p.group + (at - token * p.group);
                store_row8<T>(reinterpret_cast<T*>(p.out) + ((int64_t)(first_s[b] + token) * p.heads + head) * D + ch, o, sum);
            } else {
                float4* dst = reinterpret_cast<float4*>(sp.parts + (slot * Cfg::COLS + col) * D + ch);
                dst[0] = make_float4(o[0], o[1], o[2], o[3]);
                dst[1] = make_float4(o[4], o[5], o[6], o[7]);
                if (ch == 0) reinterpret_cast<float2*>(sp.parts + (int64_t)2 * gridDim.x * Cfg::COLS * D)[slot * Cfg::COLS + col] = make_float2(mx, sum);
            }
        }
        if (!whole && t0 == 0 && tid == 0) {  // the unit goes on in the next ranges
            const int64_t unit_end = pos + n_blocks;
            int parts = 1;
            while (total * ((int64_t)blockIdx.x + parts) / ranges < unit_end) ++parts;
            *desc = {parts, first_s[b], count, kvh, ct, {0, 0, 0}};
        }
        __syncthreads();
        pos += seg;
    }
    if (!ok) {  // a copy did not arrive in time: what is in flight gets a bounded time to land before shared memory is given up
        if (tid == 0) atomicOr(&g_kv4_status[0], 1u);
        const uint64_t since = ptx::globaltimer_ns();
        while (ptx::globaltimer_ns() - since < 20000ull) {
        }
    }
}

// The parts of the unit that starts in range blockIdx.x and goes on in others: out = sum 2^(m_i - m) O_i / sum 2^(m_i - m) l_i, a CTA
// per column, its warps take the parts in turn.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(256) kv4_combine_kernel(const SplitParams sp, int ranges) {
    using Cfg = SplitCfg<D, NT>;
    pdl_sync();
    const PartDesc d = reinterpret_cast<const PartDesc*>(sp.parts + (int64_t)2 * ranges * Cfg::part_floats())[blockIdx.x];
    const int col = blockIdx.y, at = d.ct * Cfg::COLS + col;
    if (d.parts == 0 || at >= d.count * sp.a.group) return;
    __shared__ float o_s[8][D];
    __shared__ float2 ml_s[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float2* ml = reinterpret_cast<const float2*>(sp.parts + (int64_t)2 * ranges * Cfg::COLS * D);
    constexpr int C = D / 32;
    auto slot = [&](int i) { return (i == 0 ? 2 * (int64_t)blockIdx.x + 1 : 2 * ((int64_t)blockIdx.x + i)) * Cfg::COLS + col; };
    float m = -INFINITY;
    for (int i = lane; i < d.parts; i += 32) m = fmaxf(m, ml[slot(i)].x);
    m = warp_max(m);
    const float use = m == -INFINITY ? 0.f : m;
    float l = 0.f, o[C];
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = 0.f;
#pragma unroll 4
    for (int i = warp; i < d.parts; i += 8) {
        const float2 part = ml[slot(i)];
        const float f = ptx::ex2_approx(part.x - use);
        l = fmaf(part.y, f, l);
        const float* src = sp.parts + slot(i) * D + lane;
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] = fmaf(src[c * 32], f, o[c]);
    }
#pragma unroll
    for (int c = 0; c < C; ++c) o_s[warp][c * 32 + lane] = o[c];
    if (lane == 0) ml_s[warp].x = l;
    __syncthreads();
    const int ch = threadIdx.x * 8;
    if (ch >= D) return;
    float sum = 0.f, y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        sum += ml_s[w].x;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] += o_s[w][ch + e];
    }
    const int token = at / sp.a.group, head = d.kvh * sp.a.group + (at - token * sp.a.group);
    store_row8<T>(reinterpret_cast<T*>(sp.a.out) + ((int64_t)(d.first + token) * sp.a.heads + head) * D + ch, y, sum);
}

template <typename T, int D, int NT>
int launch_split(SplitParams sp, cudaStream_t st) {
    using Cfg = SplitCfg<D, NT>;
    static std::atomic<uint64_t> reserved;
    if (!reserve_smem(kv4_split_kernel<T, D, NT>, Cfg::smem(kMaxBatch), reserved)) return fail(XG_ERR_LAUNCH, "xg_kv4_attention: cannot reserve shared memory");
    const int grid = num_sms() * Cfg::CTAS;
    launch_with({.early = false}, kv4_split_kernel<T, D, NT>, (unsigned)grid, kWarps * 32, (size_t)Cfg::smem(sp.a.batch), st, sp);
    if (const int rc = check_launch("xg_kv4_attention")) return rc;
    if (!sp.split) return XG_OK;
    launch(kv4_combine_kernel<T, D, NT>, dim3((unsigned)grid, Cfg::COLS), 256, 0, st, sp, grid);
    return check_launch("xg_kv4_attention");
}

// Columns per unit: what the sequences bring, 16 where they bring more than 8. D = 256 has no registers for 16.
constexpr int columns(int64_t D, int64_t max_q, int64_t group) { return D == 256 || max_q * group <= 8 ? 8 : 16; }

// Long sequences are cut over CTAs. Short ones are left whole: the second launch and its traffic cost more than uneven ranges.
constexpr bool cut(int64_t max_len) { return max_len > 1024; }

int64_t split_workspace(int64_t D, int64_t max_q, int64_t group, int64_t max_len) {
    if (!cut(max_len)) return 0;
    const int64_t cols = columns(D, max_q, group), ctas = (int64_t)num_sms() * split_ctas((int)D, (int)cols / 8);
    return 2 * ctas * cols * (D + 2) * 4 + ctas * (int64_t)sizeof(PartDesc);
}

constexpr int kMostStreamed = 64;

template <typename T>
int attend_split(const AttendParams& whole, int64_t D, int64_t max_q, int most_cols, void* workspace, cudaStream_t st) {
    const int64_t max_len = (int64_t)whole.table_pages * whole.cache.tiles * kTileTokens;
    const int cols = columns(D, max_q, whole.group);
    for (int at = 0; at == 0 || at < whole.batch; at += kMaxBatch) {
        SplitParams sp = {};
        sp.a = whole;
        sp.a.batch = whole.batch - at < kMaxBatch ? whole.batch - at : kMaxBatch;
        sp.a.table += (int64_t)at * whole.table_stride;
        sp.a.lens += at;
        if (whole.starts) sp.a.starts += at;
        else sp.a.row0 = at;
        sp.parts = static_cast<float*>(workspace);
        sp.split = cut(max_len);
        sp.min_blocks = 8;
        sp.most_cols = most_cols;
        sp.first_rows = at == 0;
        sp.last_rows = at + kMaxBatch >= whole.batch;
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
    return split_workspace(D, max_q, q_heads / kv_heads, max_len);
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
    // a range of tiles is counted in 32 bits (2^38 tiles are 300 TB of cache read, or some minutes)
    if (tokens > 0 && kv_heads * (tokens * (q_heads / kv_heads) / 8 + batch + 1) > (1LL << 38) / (table_pages * (page_size / 16) + 1))
        return fail(XG_ERR_TOO_LARGE, "xg_kv4_attention: too many rows and keys");
    if (tokens == 0) return XG_OK;
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
    // Sequences with many columns go to the tensor-memory kernel, where there may be any; the others to the streaming one.
    const bool tiles = D != 256 && batch > 0 && max_q * p.group > kMostStreamed;
    const int most = tiles ? kMostStreamed : 0x7fffffff;
    const int rc = dtype == XG_BF16 ? attend_split<__nv_bfloat16>(p, D, max_q, most, workspace, st) : attend_split<__half>(p, D, max_q, most, workspace, st);
    return rc != XG_OK || !tiles ? rc : attend_prefill(p, D, dtype, most, st);
}
