// RMSNorm of every query and key head and the rotation by position, in one pass over q and k:
//   y = x * rsqrt(mean(x^2) + eps) * w                        over the D channels of a head (no weight: y = x)
//   out_i = y_i c_i - y_{i+R/2} s_i,  out_{i+R/2} = y_{i+R/2} c_{i+R/2} + y_i s_{i+R/2}      i < R/2; channels from R on: out = y
// c, s: rows of tables [P, R] at the token's position. With several position axes (time, height, width) pair i takes its row by the
// axis whose section holds i. A position outside the table turns its pairs to zero. fp32 throughout, rounded once.
//
// HBM is the floor: every element is read and written once. A group of lanes holds a head, each lane the two 16-byte pieces that a
// rotation mixes, so only the sum of squares crosses lanes. A warp keeps its token's table rows in registers over several heads.
// 16384 tokens x (32 + 8) heads x 128 in bf16 with fp32 tables on three axes: 70 us, 4.8 TB/s; 60 % of the issue slots, 6.4 warps a
// scheduler, each waiting for its token's position, then its table rows, then its heads. Loading the next heads ahead, 8-byte pieces
// and fewer registers were slower. A few tokens: launch and host, 9 us.
#include "common.cuh"

namespace xg {
namespace {

constexpr int kMaxAxes = 8;

struct QkParams {
    const void* x[2];  // q, k
    const void* w[2];  // null: not normalised
    void* y[2];        // [tokens, heads, D]
    int64_t st[2], sh[2];
    int heads[2];
    const void* cos;
    const void* sin;
    const int64_t* positions;
    int64_t axis_stride, table_rows, tokens;
    int D, R, axes;
    int pair_end[kMaxAxes];  // pairs up to here follow axis a
    float eps;
    int chunks, steps;  // vector kernel: work items per token, head groups per item
};

// Where the pairs of a piece start: rotated pairs (a, a + R/2), then what is left of the head.
__device__ __forceinline__ void piece(const QkParams& p, int lane_in_head, int n, int& a, int& b) {
    const int rotated = p.R / 2 / n;
    if (lane_in_head < rotated) {
        a = lane_in_head * n;
        b = a + p.R / 2;
    } else {
        a = p.R + (lane_in_head - rotated) * 2 * n;
        b = a + n;
    }
}

__device__ __forceinline__ int64_t row_of_pair(const QkParams& p, int64_t token, int pair) {
    int axis = 0;
    while (axis + 1 < p.axes && pair >= p.pair_end[axis]) ++axis;
    const int64_t pos = p.positions[(int64_t)axis * p.axis_stride + token];
    return pos >= 0 && pos < p.table_rows ? pos : -1;
}

template <typename Tc, int N>
__device__ __forceinline__ void load_coefs(const Tc* t, float (&out)[N]) {
    constexpr int V = Vec16<Tc>::N;
    if constexpr (N % V == 0) {
#pragma unroll
        for (int i = 0; i < N; i += V) {
            const Vec16<Tc> u = ld16(t + i);
#pragma unroll
            for (int e = 0; e < V; ++e) out[i + e] = Cvt<Tc>::to_f(u.v[e]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = Cvt<Tc>::to_f(t[i]);
    }
}

// LPH lanes (a power of two) per head, D / (2 * 16 bytes) of them in use.
template <typename T, typename Tc, typename Tw, int LPH>
__global__ void __launch_bounds__(128) qk_norm_rope_vec_kernel(const QkParams p) {
    pdl_sync();
    constexpr int N = Vec16<T>::N, PER = 32 / LPH;  // heads side by side in a warp
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int64_t token = item / p.chunks;
    if (token >= p.tokens) return;
    const int lane = threadIdx.x & 31, in_head = lane & (LPH - 1);
    const int first = (int)(item - token * p.chunks) * p.steps * PER + lane / LPH;
    const int all = p.heads[0] + p.heads[1];
    const bool used = in_head * 2 * N < p.D;
    int a, b;
    piece(p, in_head, N, a, b);
    float c1[N], s1[N], c2[N], s2[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        c1[i] = c2[i] = 1.f;
        s1[i] = s2[i] = 0.f;
    }
    if (used && b < p.R) {
        const Tc* cos = reinterpret_cast<const Tc*>(p.cos);
        const Tc* sin = reinterpret_cast<const Tc*>(p.sin);
        bool one_axis = true;
        for (int e = 0; e + 1 < p.axes; ++e) one_axis = one_axis && !(p.pair_end[e] > a && p.pair_end[e] < a + N);
        if (one_axis) {
            const int64_t row = row_of_pair(p, token, a);
            if (row >= 0) {
                load_coefs<Tc, N>(cos + row * p.R + a, c1);
                load_coefs<Tc, N>(cos + row * p.R + b, c2);
                load_coefs<Tc, N>(sin + row * p.R + a, s1);
                load_coefs<Tc, N>(sin + row * p.R + b, s2);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) c1[i] = c2[i] = 0.f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int64_t row = row_of_pair(p, token, a + i);
                c1[i] = row < 0 ? 0.f : Cvt<Tc>::to_f(cos[row * p.R + a + i]);
                c2[i] = row < 0 ? 0.f : Cvt<Tc>::to_f(cos[row * p.R + b + i]);
                s1[i] = row < 0 ? 0.f : Cvt<Tc>::to_f(sin[row * p.R + a + i]);
                s2[i] = row < 0 ? 0.f : Cvt<Tc>::to_f(sin[row * p.R + b + i]);
            }
        }
    }
    const float inv_d = 1.0f / (float)p.D;
#pragma unroll 2
    for (int step = 0; step < p.steps; ++step) {
        const int head = first + step * PER;
        const int which = head >= p.heads[0] ? 1 : 0;
        const int h = head - (which ? p.heads[0] : 0);
        const bool on = used && head < all;
        float x1[N], x2[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x1[i] = x2[i] = 0.f;
        if (on) {
            const T* x = reinterpret_cast<const T*>(which ? p.x[1] : p.x[0]) + token * (which ? p.st[1] : p.st[0]) + h * (which ? p.sh[1] : p.sh[0]);
            const Vec16<T> u1 = ld16_stream(x + a), u2 = ld16_stream(x + b);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x1[i] = Cvt<T>::to_f(u1.v[i]);
                x2[i] = Cvt<T>::to_f(u2.v[i]);
            }
        }
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) sq = fmaf(x1[i], x1[i], fmaf(x2[i], x2[i], sq));
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
        if (!on) continue;
        const Tw* w = reinterpret_cast<const Tw*>(which ? p.w[1] : p.w[0]);
        if (w != nullptr) {
            const float r = rsqrtf(fmaf(sq, inv_d, p.eps));
            float w1[N], w2[N];
            load_coefs<Tw, N>(w + a, w1);
            load_coefs<Tw, N>(w + b, w2);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x1[i] *= r * w1[i];
                x2[i] *= r * w2[i];
            }
        }
        Vec16<T> y1, y2;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            y1.v[i] = Cvt<T>::from_f(x1[i] * c1[i] - x2[i] * s1[i]);
            y2.v[i] = Cvt<T>::from_f(x2[i] * c2[i] + x1[i] * s2[i]);
        }
        T* y = reinterpret_cast<T*>(which ? p.y[1] : p.y[0]) + (token * (which ? p.heads[1] : p.heads[0]) + h) * (int64_t)p.D;
        st16(y + a, y1);
        st16(y + b, y2);
    }
}

// Any D, R, strides and alignment: a warp per head, element by element, each with its own look at the position and the table. 16384 tokens
// x (32 + 8) heads in bf16: of 80 with 40 rotated 238 us (floor 33), of 96 with 24 rotated 258 us (39).
template <typename T, typename Tc, typename Tw>
__global__ void __launch_bounds__(128) qk_norm_rope_any_kernel(const QkParams p) {
    pdl_sync();
    const int all = p.heads[0] + p.heads[1];
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int64_t token = item / all;
    if (token >= p.tokens) return;
    const int lane = threadIdx.x & 31, head = (int)(item - token * all);
    const int which = head >= p.heads[0] ? 1 : 0;
    const int h = head - (which ? p.heads[0] : 0);
    const T* x = reinterpret_cast<const T*>(which ? p.x[1] : p.x[0]) + token * (which ? p.st[1] : p.st[0]) + h * (which ? p.sh[1] : p.sh[0]);
    const Tw* w = reinterpret_cast<const Tw*>(which ? p.w[1] : p.w[0]);
    T* y = reinterpret_cast<T*>(which ? p.y[1] : p.y[0]) + (token * (which ? p.heads[1] : p.heads[0]) + h) * (int64_t)p.D;
    float r = 1.f;
    if (w != nullptr) {
        float sq = 0.f;
        for (int i = lane; i < p.D; i += 32) {
            const float v = Cvt<T>::to_f(x[i]);
            sq = fmaf(v, v, sq);
        }
        r = rsqrtf(warp_sum(sq) / (float)p.D + p.eps);
    }
    auto normed = [&](int i) { return w != nullptr ? Cvt<T>::to_f(x[i]) * (r * Cvt<Tw>::to_f(w[i])) : Cvt<T>::to_f(x[i]); };
    const Tc* cos = reinterpret_cast<const Tc*>(p.cos);
    const Tc* sin = reinterpret_cast<const Tc*>(p.sin);
    const int half = p.R / 2;
    for (int i = lane; i < half; i += 32) {
        const int64_t row = row_of_pair(p, token, i);
        const float y1 = normed(i), y2 = normed(i + half);
        float o1 = 0.f, o2 = 0.f;
        if (row >= 0) {
            o1 = y1 * Cvt<Tc>::to_f(cos[row * p.R + i]) - y2 * Cvt<Tc>::to_f(sin[row * p.R + i]);
            o2 = y2 * Cvt<Tc>::to_f(cos[row * p.R + i + half]) + y1 * Cvt<Tc>::to_f(sin[row * p.R + i + half]);
        } else {
            o1 = y1 * 0.f - y2 * 0.f;  // (as the vector kernel: a NaN stays one)
            o2 = y2 * 0.f + y1 * 0.f;
        }
        y[i] = Cvt<T>::from_f(o1);
        y[i + half] = Cvt<T>::from_f(o2);
    }
    for (int i = p.R + lane; i < p.D; i += 32) y[i] = Cvt<T>::from_f(normed(i));
}

template <typename T, typename Tc, typename Tw>
int launch_qk(QkParams& p, cudaStream_t st) {
    constexpr int N = Vec16<T>::N;
    const int all = p.heads[0] + p.heads[1];
    bool vec = p.D % (2 * N) == 0 && p.R % (2 * N) == 0 && p.D <= 64 * N && aligned16(p.cos) && aligned16(p.sin) && p.R * sizeof(Tc) % 16 == 0;
    for (int i = 0; i < 2; ++i)
        vec = vec && aligned16(p.x[i]) && aligned16(p.y[i]) && aligned16(p.w[i]) && p.st[i] % N == 0 && p.sh[i] % N == 0;
    if (!vec) {
        const int64_t grid = (p.tokens * all + 3) / 4;
        if (grid > 0x7fffffffLL) return fail(XG_ERR_TOO_LARGE, "xg_qk_norm_rope: too many rows");
        launch(qk_norm_rope_any_kernel<T, Tc, Tw>, (unsigned)grid, 128, 0, st, p);
        return check_launch("xg_qk_norm_rope");
    }
    int lph = 1;
    while (lph * 2 * N < p.D) lph *= 2;
    const int groups = (all + 32 / lph - 1) / (32 / lph);  // head groups of a token
    // all of a token's heads in one warp where that still fills the chip (16 warps per SM); fewer where there are few tokens
    const int64_t want = 16LL * num_sms();
    int64_t steps = p.tokens * groups / want;
    p.steps = (int)(steps < 1 ? 1 : (steps > groups ? groups : steps));
    p.chunks = (groups + p.steps - 1) / p.steps;
    const int64_t grid = (p.tokens * p.chunks + 3) / 4;
    if (grid > 0x7fffffffLL) return fail(XG_ERR_TOO_LARGE, "xg_qk_norm_rope: too many rows");
    switch (lph) {
        case 1: launch(qk_norm_rope_vec_kernel<T, Tc, Tw, 1>, (unsigned)grid, 128, 0, st, p); break;
        case 2: launch(qk_norm_rope_vec_kernel<T, Tc, Tw, 2>, (unsigned)grid, 128, 0, st, p); break;
        case 4: launch(qk_norm_rope_vec_kernel<T, Tc, Tw, 4>, (unsigned)grid, 128, 0, st, p); break;
        case 8: launch(qk_norm_rope_vec_kernel<T, Tc, Tw, 8>, (unsigned)grid, 128, 0, st, p); break;
        case 16: launch(qk_norm_rope_vec_kernel<T, Tc, Tw, 16>, (unsigned)grid, 128, 0, st, p); break;
        default: launch(qk_norm_rope_vec_kernel<T, Tc, Tw, 32>, (unsigned)grid, 128, 0, st, p); break;
    }
    return check_launch("xg_qk_norm_rope");
}

template <typename T>
int launch_types(QkParams& p, bool f32_tables, bool f32_weights, cudaStream_t st) {
    if (f32_tables) return f32_weights ? launch_qk<T, float, float>(p, st) : launch_qk<T, float, T>(p, st);
    return f32_weights ? launch_qk<T, T, float>(p, st) : launch_qk<T, T, T>(p, st);
}

}  // namespace
}  // namespace xg

extern "C" int xg_qk_norm_rope(const void* q, const void* k, const void* q_weight, const void* k_weight, float eps, const void* cos, const void* sin,
                               int64_t table_rows, int64_t rot, const int64_t* positions, int64_t axes, int64_t axis_stride,
                               const int64_t* sections, void* q_out, void* k_out, int64_t tokens, int64_t q_heads, int64_t k_heads, int64_t D,
                               int64_t q_stride_t, int64_t q_stride_h, int64_t k_stride_t, int64_t k_stride_h, int dtype, int w_dtype,
                               int table_dtype, void* stream) {
    using namespace xg;
    if (dtype_size(dtype) == 0 || (w_dtype != XG_F32 && w_dtype != dtype) || (table_dtype != XG_F32 && table_dtype != dtype))
        return fail(XG_ERR_INVALID_ARG, "xg_qk_norm_rope: bad dtypes %d, %d, %d", dtype, w_dtype, table_dtype);
    if (tokens < 0 || q_heads < 0 || k_heads < 0 || D <= 0 || rot < 0 || rot > D || rot % 2 != 0 || table_rows < 0)
        return fail(XG_ERR_INVALID_ARG, "xg_qk_norm_rope: bad extents");
    if (q_heads > 65535 || k_heads > 65535 || D > 65536) return fail(XG_ERR_TOO_LARGE, "xg_qk_norm_rope: heads or head_dim");
    if (axes < 1 || axes > kMaxAxes || (axes > 1 && !sections)) return fail(XG_ERR_INVALID_ARG, "xg_qk_norm_rope: 1 to %d position axes", kMaxAxes);
    if (tokens == 0 || q_heads + k_heads == 0) return XG_OK;
    if ((q_heads > 0 && (!q || !q_out)) || (k_heads > 0 && (!k || !k_out)) || (rot > 0 && (!cos || !sin || !positions)))
        return fail(XG_ERR_INVALID_ARG, "xg_qk_norm_rope: null pointer");
    QkParams p = {};
    p.x[0] = q; p.x[1] = k; p.w[0] = q_weight; p.w[1] = k_weight; p.y[0] = q_out; p.y[1] = k_out;
    p.st[0] = q_stride_t; p.sh[0] = q_stride_h; p.st[1] = k_stride_t; p.sh[1] = k_stride_h;
    p.heads[0] = (int)q_heads; p.heads[1] = (int)k_heads;
    p.cos = cos; p.sin = sin; p.positions = positions;
    p.axis_stride = axis_stride; p.table_rows = table_rows; p.tokens = tokens;
    p.D = (int)D; p.R = (int)rot; p.axes = (int)axes; p.eps = eps;
    int64_t end = 0;
    for (int64_t a = 0; a < axes; ++a) {
        const int64_t count = axes == 1 ? rot / 2 : sections[a];
        if (count < 0) return fail(XG_ERR_INVALID_ARG, "xg_qk_norm_rope: negative section");
        end += count;
        p.pair_end[a] = (int)(end > rot / 2 ? rot / 2 : end);
    }
    if (end != rot / 2) return fail(XG_ERR_INVALID_ARG, "xg_qk_norm_rope: the sections have to add up to %lld pairs", (long long)(rot / 2));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    switch (dtype) {
        case XG_F32: return launch_qk<float, float, float>(p, st);
        case XG_BF16: return launch_types<__nv_bfloat16>(p, table_dtype == XG_F32, w_dtype == XG_F32, st);
        default: return launch_types<__half>(p, table_dtype == XG_F32, w_dtype == XG_F32, st);
    }
}
