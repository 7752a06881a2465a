// Rotary positions with several axes on the heads of q and k, optionally behind the RMS normalisation of each head (HBM-bound).
//
// The columns of a head are cut into one block per axis (time, height, width, ...), columns behind the last block stay as
// they are.  Pair i of axis a turns by the angle  position[token, a] * theta^(-2 i / width_a):
//     (y0, y1) -> (y0 cos - y1 sin, y0 sin + y1 cos),   y = x or x * rsqrt(mean(x^2) + eps) * weight.
// Angles of far positions lose everything in fp32 (position 10^5 leaves 2^-7 of a radian), so the turn is counted in
// revolutions in fp64, reduced to [-1/2, 1/2] there and only then rounded: one fp64 multiplication per (token, pair).  A
// thread keeps the sines of its columns in registers and walks the heads, which share them.  Everything else is fp32 with
// one rounding at the end.  32760 tokens, 16 + 16 heads of 128, fp16: 85 us = 6.3 TB/s (copy 6.55); 2 x 4429 tokens, 24 + 24
// heads of 64 behind their normalisation: 22 us = 5.0 TB/s, 1.9 rounds of CTAs and the sines of each.
#include <cmath>
#include <type_traits>

#include "common.cuh"

namespace sq {

constexpr int kRotMaxPairs = SQ_ROTARY_MAX_D / 2;

struct RotaryParams {
    const void* x[2];                 // q, k
    void* y[2];
    const void* weight[2];            // RMS weights or NULL
    int heads[2];
    long long x_bs[2], x_ts[2], x_hs[2], y_bs[2], y_ts[2], y_hs[2];
    const void* pos;
    long long pos_bs, pos_ts;
    long long batch, tokens;          // tokens of one batch entry
    int D, pairs, all_pairs;          // rotated pairs; scalar kernel: and those of the columns behind the axes
    int pos_float, halves;
    int heads_per_cta;                // heads (of q, then of k) that one CTA's threads walk
    int group;                        // vector kernel: threads that share a row (power of two)
    int units;                        // vector kernel: threads of a group that have columns
    float eps, inv_d;                 // inv_d = 1 / D
    double turn[kRotMaxPairs];        // revolutions per unit of position
    unsigned char axis[kRotMaxPairs];
    short col[kRotMaxPairs];          // first column of a pair
    short step[kRotMaxPairs];         // distance to its second column
    short unit_a[16], unit_b[16];     // "halves": first columns of a thread's two vectors
    short unit_pair[16];              // and the pair of its first element (-1: columns that are not rotated)
};

__device__ __forceinline__ float2 rot_angle(const RotaryParams& p, long long b, long long t, int pair) {
    const long long i = b * p.pos_bs + t * p.pos_ts + p.axis[pair];
    const double pos = p.pos_float ? static_cast<double>(static_cast<const float*>(p.pos)[i]) : static_cast<double>(static_cast<const int*>(p.pos)[i]);
    const double rev = pos * p.turn[pair];
    const float part = static_cast<float>(rev - rint(rev));      // exact difference, [-1/2, 1/2]
    float s, c;
    sincospif(2.0f * part, &s, &c);
    return make_float2(c, s);
}

// A row's 8 columns as four pairs of floats, and back.
template <typename T>
__device__ __forceinline__ void rot_unpack(const uint4& a, float2 (&v)[4]) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) v[i] = make_float2(0.0f, 0.0f);
        else if constexpr (std::is_same<T, __half>::value) v[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        else v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    }
}
template <typename T>
struct RotRow {                       // 8 columns as loaded
    uint4 w[sizeof(T) == 4 ? 2 : 1];
    __device__ __forceinline__ void load(const T* p) {
        w[0] = reinterpret_cast<const uint4*>(p)[0];       // plain loads: the result may overwrite the input
        if constexpr (sizeof(T) == 4) w[1] = reinterpret_cast<const uint4*>(p)[1];
    }
    __device__ __forceinline__ void zero() {
        w[0] = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (sizeof(T) == 4) w[1] = w[0];
    }
    __device__ __forceinline__ void get(float2 (&v)[4]) const {
        if constexpr (sizeof(T) == 4) {
            v[0] = make_float2(__uint_as_float(w[0].x), __uint_as_float(w[0].y));
            v[1] = make_float2(__uint_as_float(w[0].z), __uint_as_float(w[0].w));
            v[2] = make_float2(__uint_as_float(w[1].x), __uint_as_float(w[1].y));
            v[3] = make_float2(__uint_as_float(w[1].z), __uint_as_float(w[1].w));
        } else {
            rot_unpack<T>(w[0], v);
        }
    }
    __device__ __forceinline__ void put(const float2 (&v)[4]) {
        if constexpr (sizeof(T) == 4) {
            w[0] = make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
            w[1] = make_uint4(__float_as_uint(v[2].x), __float_as_uint(v[2].y), __float_as_uint(v[3].x), __float_as_uint(v[3].y));
        } else {
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (std::is_same<T, __half>::value) {
                    const __half2 h = __float22half2_rn(v[i]);
                    o[i] = *reinterpret_cast<const uint32_t*>(&h);
                } else {
                    const __nv_bfloat162 h = __float22bfloat162_rn(v[i]);
                    o[i] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
            w[0] = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        reinterpret_cast<uint4*>(p)[0] = w[0];
        if constexpr (sizeof(T) == 4) reinterpret_cast<uint4*>(p)[1] = w[1];
    }
};

// A thread has one vector of 8 columns (adjacent pairs: 4 pairs) or two (halves: 8 pairs, one column of each in either
// vector) of one token, and walks heads, the loads of kRotAhead heads in flight.  `group` threads share a row.  Two-wide fp32
// instructions throughout: the kernel has about 50 instructions for 32 bytes of traffic and is near the issue limit with
// scalar ones.
constexpr int kRotAhead = 4;
constexpr int kRotThreads = 128;
constexpr int kRotWarps = 32;          // per SM; 48 to 96 measured the same or slower (64 x 64 grid, two samples: 23.8 against 24.4 to 26.0 us)
// CTAs that an SM has room for: what bounds the registers, and with them the loads in flight.  Adjacent pairs, image tokens (2 x 4429,
// 24 + 24 heads of 64 behind their normalisation) and clip (32760 tokens, 32 heads of 128): unbounded 24.2 and 86.5 us, five 23.1
// and 85.9, six 21.9 and 85.3, eight 26 (spills).  Halves, the same tokens: 16-bit 24.6 and 89.7 us with five, 97 with four or fewer, 93 with
// six; behind the normalisation 25.0 and 98.7 with four, 27.0 and 98.3 with five, 30 and 109 with three; fp32 47 and 182 with three,
// 45 and 202 with four.
template <typename T, bool HALVES, bool NORM>
constexpr int rot_vec_ctas() { return !HALVES ? 6 : sizeof(T) == 4 ? 3 : NORM ? 4 : 5; }

// REST: there are columns behind the axes (a form of its own: the selects cost the other one registers, image tokens 20.5 -> 21.2 us).
template <typename T, bool HALVES, bool NORM, bool REST>
__global__ void __launch_bounds__(kRotThreads, (rot_vec_ctas<T, HALVES, NORM>())) rotary_vec_kernel(const __grid_constant__ RotaryParams p) {
    constexpr int NV = HALVES ? 2 : 1;
    constexpr int U = (sizeof(T) == 4 || HALVES) ? kRotAhead / 2 : kRotAhead;
    const int u = threadIdx.x & (p.group - 1);
    const long long rows = p.batch * p.tokens;
    const long long row = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) / p.group;
    const bool has = row < rows && u < p.units;
    const long long b = has ? row / p.tokens : 0, t = has ? row - b * p.tokens : 0;
    const int uu = has ? u : 0;
    const int col_a = HALVES ? p.unit_a[uu] : 8 * uu, col_b = HALVES ? p.unit_b[uu] : 0;
    const int pair0 = HALVES ? p.unit_pair[uu] : 4 * uu;
    const int h0 = blockIdx.y * p.heads_per_cta, h1 = min(h0 + p.heads_per_cta, p.heads[0] + p.heads[1]);
    float2 cs[4 * NV], sn[4 * NV];    // adjacent: (c, c) and (-s, s) of a pair; halves: the pairs' cosines and sines two by two
    bool angles = false;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        const int first = part ? max(h0 - p.heads[0], 0) : h0, last = part ? h1 - p.heads[0] : min(h1, p.heads[0]);
        if (first >= last) continue;                                     // uniform over the CTA
        const T* x = static_cast<const T*>(p.x[part]) + b * p.x_bs[part] + t * p.x_ts[part] + first * p.x_hs[part];
        T* y = static_cast<T*>(p.y[part]) + b * p.y_bs[part] + t * p.y_ts[part] + first * p.y_hs[part];
        const long long xs = p.x_hs[part], ys = p.y_hs[part];
        RotRow<T> in[U][NV];
        auto fetch = [&](int h) {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (has && h + i < last) {
                    in[i][0].load(x + i * xs + col_a);
                    if constexpr (HALVES) in[i][NV - 1].load(x + i * xs + col_b);
                } else {
                    in[i][0].zero();
                    if constexpr (HALVES) in[i][NV - 1].zero();
                }
            }
            x += U * xs;
        };
        fetch(first);
        float2 w[NV][4];
        if constexpr (NORM) {
            RotRow<T> r;
            r.load(static_cast<const T*>(p.weight[part]) + col_a);
            r.get(w[0]);
            if constexpr (HALVES) {
                r.load(static_cast<const T*>(p.weight[part]) + col_b);
                r.get(w[NV - 1]);
            }
        }
        if (!angles) {                                                   // while the first heads are on their way
            angles = true;
#pragma unroll
            for (int i = 0; i < 4 * NV; ++i) {
                float2 a = make_float2(1.0f, 0.0f);
                if (has && pair0 >= 0 && pair0 + i < p.pairs) a = rot_angle(p, b, t, pair0 + i);
                if constexpr (HALVES) {
                    if (i & 1) { cs[i >> 1].y = a.x; sn[i >> 1].y = a.y; }
                    else { cs[i >> 1].x = a.x; sn[i >> 1].x = a.y; }
                } else {
                    cs[i] = make_float2(a.x, a.x);
                    sn[i] = make_float2(-a.y, a.y);
                }
            }
        }
        for (int h = first; h < last; h += U) {
            float2 e[U][NV][4];
#pragma unroll
            for (int i = 0; i < U; ++i)
#pragma unroll
                for (int v = 0; v < NV; ++v) in[i][v].get(e[i][v]);
            if (h + U < last) fetch(h + U);
            if constexpr (NORM) {
                float ss[U];
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    float2 s = __fmul2_rn(e[i][0][0], e[i][0][0]);
#pragma unroll
                    for (int v = 0; v < NV; ++v)
#pragma unroll
                        for (int k = v ? 0 : 1; k < 4; ++k) s = __ffma2_rn(e[i][v][k], e[i][v][k], s);
                    ss[i] = s.x + s.y;
                }
                for (int o = p.group >> 1; o > 0; o >>= 1)
#pragma unroll
                    for (int i = 0; i < U; ++i) ss[i] += __shfl_xor_sync(0xffffffffu, ss[i], o);
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const float r = rsqrtf(ss[i] * p.inv_d + p.eps);
                    const float2 r2 = make_float2(r, r);
#pragma unroll
                    for (int v = 0; v < NV; ++v)
#pragma unroll
                        for (int k = 0; k < 4; ++k) e[i][v][k] = __fmul2_rn(e[i][v][k], __fmul2_rn(r2, w[v][k]));
                }
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                float2 o[NV][4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if constexpr (HALVES) {
                        const float2 m = make_float2(-sn[k].x, -sn[k].y);
                        o[0][k] = __ffma2_rn(e[i][0][k], cs[k], __fmul2_rn(e[i][NV - 1][k], m));
                        o[NV - 1][k] = __ffma2_rn(e[i][0][k], sn[k], __fmul2_rn(e[i][NV - 1][k], cs[k]));
                    } else {
                        o[0][k] = __ffma2_rn(e[i][0][k], cs[k], __fmul2_rn(make_float2(e[i][0][k].y, e[i][0][k].x), sn[k]));
                    }
                }
                if constexpr (REST) {     // these columns stay: 1 * y + 0 * partner would pass the partner's NaN or infinity on
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if constexpr (HALVES) {
                            if (pair0 < 0) { o[0][k] = e[i][0][k]; o[NV - 1][k] = e[i][NV - 1][k]; }
                        } else if (pair0 + k >= p.pairs) {
                            o[0][k] = e[i][0][k];
                        }
                    }
                }
                if (has && h + i < last) {
                    RotRow<T> r;
                    r.put(o[0]);
                    r.store(y + i * ys + col_a);
                    if constexpr (HALVES) {
                        r.put(o[NV - 1]);
                        r.store(y + i * ys + col_b);
                    }
                }
            }
            y += U * ys;
        }
    }
}

// Any width, stride and alignment: one warp per token, lane l has the pairs l, l + 32, ... and walks heads, 8 / NP at a time (all
// their loads are out before the first store, which the compiler could not move them across).  Columns behind the axes are
// pairs that are not turned, the last of them alone (step 0) if their number is odd.  Halves of 28 columns, the clip's 32760 tokens,
// 32 heads of 128: 16-bit 229 us (a head at a time 981; 333 with the registers unbounded), behind the normalisation 279 (1000); fp32
// 216 (981; 258 when bounded to eight CTAs an SM), 293 (998).
template <typename T, bool NORM, int NP>
__global__ void __launch_bounds__(kRotThreads, sizeof(T) == 4 ? 0 : 8) rotary_scalar_kernel(const __grid_constant__ RotaryParams p) {
    constexpr int U = 8 / NP;
    const int lane = threadIdx.x & 31;
    const long long row = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    if (row >= p.batch * p.tokens) return;
    const long long b = row / p.tokens, t = row - b * p.tokens;
    const bool halves = p.halves != 0;
    float cs[NP], sn[NP];
    int ca[NP], cc[NP];
    bool has[NP], two[NP], turned[NP];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
        const int pair = lane + 32 * n;
        has[n] = pair < p.all_pairs;
        turned[n] = pair < p.pairs;
        ca[n] = has[n] ? p.col[pair] : 0;
        cc[n] = has[n] ? ca[n] + p.step[pair] : 0;
        two[n] = cc[n] != ca[n];
        const float2 a = turned[n] ? rot_angle(p, b, t, pair) : make_float2(1.0f, 0.0f);
        cs[n] = a.x;
        sn[n] = a.y;
    }
    const int h0 = blockIdx.y * p.heads_per_cta, h1 = min(h0 + p.heads_per_cta, p.heads[0] + p.heads[1]);
#pragma unroll 1
    for (int part = 0; part < 2; ++part) {
        const int first = part ? max(h0 - p.heads[0], 0) : h0, last = part ? h1 - p.heads[0] : min(h1, p.heads[0]);
        if (first >= last) continue;
        const long long xs = p.x_hs[part], ys = p.y_hs[part];
        const T* x = static_cast<const T*>(p.x[part]) + b * p.x_bs[part] + t * p.x_ts[part] + first * xs;
        T* y = static_cast<T*>(p.y[part]) + b * p.y_bs[part] + t * p.y_ts[part] + first * ys;
        const T* w = static_cast<const T*>(p.weight[part]);
        float wa[NP], wc[NP];
        if constexpr (NORM) {
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                wa[n] = has[n] ? to_float<T>(w[ca[n]]) : 0.0f;
                wc[n] = two[n] ? to_float<T>(w[cc[n]]) : 0.0f;
            }
        }
        for (int h = first; h < last; h += U, x += U * xs, y += U * ys) {
            float u[U][NP], v[U][NP];
#pragma unroll
            for (int i = 0; i < U; ++i)
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    const bool in = h + i < last;
                    u[i][n] = in && has[n] ? to_float<T>(x[i * xs + ca[n]]) : 0.0f;
                    v[i][n] = in && two[n] ? to_float<T>(x[i * xs + cc[n]]) : 0.0f;
                }
            if constexpr (NORM) {
                float ss[U];
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    ss[i] = 0.0f;
#pragma unroll
                    for (int n = 0; n < NP; ++n) ss[i] = fmaf(v[i][n], v[i][n], fmaf(u[i][n], u[i][n], ss[i]));
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                    for (int i = 0; i < U; ++i) ss[i] += __shfl_xor_sync(0xffffffffu, ss[i], o);
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const float r = rsqrtf(ss[i] * p.inv_d + p.eps);
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        u[i][n] *= r * wa[n];
                        v[i][n] *= r * wc[n];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < U; ++i)
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    if (h + i >= last || !has[n]) continue;
                    float ya = u[i][n], yc = v[i][n];
                    if (turned[n]) {      // the vector kernel's products and sums, so that a layout does not show in the result
                        ya = fmaf(u[i][n], cs[n], __fmul_rn(v[i][n], -sn[n]));
                        yc = halves ? fmaf(u[i][n], sn[n], __fmul_rn(v[i][n], cs[n])) : fmaf(v[i][n], cs[n], __fmul_rn(u[i][n], sn[n]));
                    }
                    y[i * ys + ca[n]] = from_float<T>(ya);
                    if (two[n]) y[i * ys + cc[n]] = from_float<T>(yc);
                }
        }
    }
}

template <typename T, bool NORM>
static void launch_rotary_scalar(const RotaryParams& p, dim3 grid, cudaStream_t st) {
    if (p.all_pairs <= 32) rotary_scalar_kernel<T, NORM, 1><<<grid, kRotThreads, 0, st>>>(p);
    else if (p.all_pairs <= 64) rotary_scalar_kernel<T, NORM, 2><<<grid, kRotThreads, 0, st>>>(p);
    else rotary_scalar_kernel<T, NORM, kRotMaxPairs / 32><<<grid, kRotThreads, 0, st>>>(p);
}

template <typename T, bool REST>
static void launch_rotary_vec(const RotaryParams& p, bool halves, bool norm, dim3 grid, cudaStream_t st) {
    if (halves) {
        if (norm) rotary_vec_kernel<T, true, true, REST><<<grid, kRotThreads, 0, st>>>(p);
        else rotary_vec_kernel<T, true, false, REST><<<grid, kRotThreads, 0, st>>>(p);
    } else {
        if (norm) rotary_vec_kernel<T, false, true, REST><<<grid, kRotThreads, 0, st>>>(p);
        else rotary_vec_kernel<T, false, false, REST><<<grid, kRotThreads, 0, st>>>(p);
    }
}

template <typename T>
static void launch_rotary(const RotaryParams& p, bool vec, bool halves, bool norm, dim3 grid, cudaStream_t st) {
    if (!vec) {
        if (norm) launch_rotary_scalar<T, true>(p, grid, st);
        else launch_rotary_scalar<T, false>(p, grid, st);
    } else if (2 * p.pairs < p.D) {
        launch_rotary_vec<T, true>(p, halves, norm, grid, st);
    } else {
        launch_rotary_vec<T, false>(p, halves, norm, grid, st);
    }
}

int rotary(const sq_rotary_args* a, cudaStream_t st) {
    SQ_REQUIRE(a != nullptr, SQ_ERR_INVALID_ARG, "sq_rotary: args is NULL");
    SQ_REQUIRE(a->dtype == SQ_F32 || a->dtype == SQ_F16 || a->dtype == SQ_BF16, SQ_ERR_INVALID_ARG, "sq_rotary: unknown dtype %d", a->dtype);
    SQ_REQUIRE(a->pairing == SQ_ROTARY_ADJACENT || a->pairing == SQ_ROTARY_HALVES, SQ_ERR_INVALID_ARG, "sq_rotary: unknown pairing %d", a->pairing);
    SQ_REQUIRE(a->batch >= 0 && a->tokens >= 0 && a->heads_q >= 0 && a->heads_k >= 0, SQ_ERR_INVALID_ARG, "sq_rotary: negative size");
    SQ_REQUIRE(a->D > 0 && a->D <= SQ_ROTARY_MAX_D, SQ_ERR_UNSUPPORTED, "sq_rotary: head width %d outside [1, %d]", a->D, SQ_ROTARY_MAX_D);
    SQ_REQUIRE(a->num_axes >= 1 && a->num_axes <= SQ_ROTARY_MAX_AXES, SQ_ERR_INVALID_ARG, "sq_rotary: %d axes outside [1, %d]", a->num_axes, SQ_ROTARY_MAX_AXES);
    SQ_REQUIRE(a->theta > 0.0 && std::isfinite(a->theta), SQ_ERR_INVALID_ARG, "sq_rotary: theta must be positive and finite");
    SQ_REQUIRE(a->batch < (1ll << 31) && a->tokens < (1ll << 31) && a->batch * a->tokens < (1ll << 33) && a->heads_q < (1 << 15) && a->heads_k < (1 << 15),
               SQ_ERR_TOO_LARGE, "sq_rotary: dimension too large");
    RotaryParams p = {};
    const bool halves = a->pairing == SQ_ROTARY_HALVES;
    int width = 0, units = 0;
    bool vec = a->D % 8 == 0;
    for (int i = 0; i < a->num_axes; ++i) {
        const int w = a->axes[i];
        SQ_REQUIRE(w > 0 && w % 2 == 0 && width + w <= a->D, SQ_ERR_INVALID_ARG, "sq_rotary: axis widths must be even, positive and fit %d columns", a->D);
        const double ratio = std::pow(a->theta, -2.0 / w);
        double turn = 1.0 / 6.283185307179586476925;
        for (int j = 0; j < w / 2; ++j, turn *= ratio) {
            const int pair = width / 2 + j;
            p.turn[pair] = turn;
            p.axis[pair] = static_cast<unsigned char>(i);
            p.col[pair] = static_cast<short>(halves ? width + j : width + 2 * j);
            p.step[pair] = static_cast<short>(halves ? w / 2 : 1);
        }
        if (halves) {
            vec = vec && w % 16 == 0;
            for (int j = 0; vec && j < w / 2; j += 8, ++units) {
                p.unit_a[units] = static_cast<short>(width + j);
                p.unit_b[units] = static_cast<short>(width + w / 2 + j);
                p.unit_pair[units] = static_cast<short>(width / 2 + j);
            }
        }
        width += w;
    }
    if (halves) {
        vec = vec && a->D % 16 == 0;
        for (int j = width; vec && j < a->D; j += 16, ++units) {       // columns behind the axes
            p.unit_a[units] = static_cast<short>(j);
            p.unit_b[units] = static_cast<short>(j + 8);
            p.unit_pair[units] = -1;
        }
    } else {
        units = a->D / 8;
    }
    if (a->batch == 0 || a->tokens == 0 || a->heads_q + a->heads_k == 0) return SQ_OK;
    SQ_REQUIRE(a->positions_dev, SQ_ERR_INVALID_ARG, "sq_rotary: positions_dev is NULL");
    const bool norm = a->norm_q_dev != nullptr || a->norm_k_dev != nullptr;
    const struct { const void* x; void* y; const void* w; int heads; long long s[6]; } parts[2] = {
        {a->q_dev, a->q_out_dev, a->norm_q_dev, a->heads_q,
         {a->q_batch_stride, a->q_token_stride, a->q_head_stride, a->q_out_batch_stride, a->q_out_token_stride, a->q_out_head_stride}},
        {a->k_dev, a->k_out_dev, a->norm_k_dev, a->heads_k,
         {a->k_batch_stride, a->k_token_stride, a->k_head_stride, a->k_out_batch_stride, a->k_out_token_stride, a->k_out_head_stride}}};
    const long long es = a->dtype == SQ_F32 ? 4 : 2;
    for (int i = 0; i < 2; ++i) {
        const auto& t = parts[i];
        SQ_REQUIRE(t.heads == 0 || (t.x && t.y && (!norm || t.w)), SQ_ERR_INVALID_ARG, "sq_rotary: NULL pointer (with normalisation, q and k both have weights)");
        p.x[i] = t.x; p.y[i] = t.y; p.weight[i] = t.w; p.heads[i] = t.heads;
        p.x_bs[i] = t.s[0]; p.x_ts[i] = t.s[1]; p.x_hs[i] = t.s[2]; p.y_bs[i] = t.s[3]; p.y_ts[i] = t.s[4]; p.y_hs[i] = t.s[5];
        if (t.heads == 0) continue;
        for (const void* q : {t.x, static_cast<const void*>(t.y), t.w}) {
            SQ_REQUIRE(reinterpret_cast<uintptr_t>(q) % es == 0, SQ_ERR_ALIGNMENT, "sq_rotary: pointers must be aligned to their elements");
            vec = vec && reinterpret_cast<uintptr_t>(q) % 16 == 0;
        }
        const long long n[6] = {a->batch, a->tokens, t.heads, a->batch, a->tokens, t.heads};
        for (int j = 0; j < 6; ++j) vec = vec && (n[j] == 1 || t.s[j] * es % 16 == 0);
    }
    p.pos = a->positions_dev; p.pos_float = a->positions_float ? 1 : 0; p.halves = halves ? 1 : 0;
    p.pos_bs = a->pos_batch_stride; p.pos_ts = a->pos_token_stride;
    p.batch = a->batch; p.tokens = a->tokens; p.D = a->D; p.pairs = width / 2; p.all_pairs = p.pairs; p.eps = a->eps; p.inv_d = 1.0f / static_cast<float>(a->D);
    for (int c = width; c < a->D; c += 2, ++p.all_pairs) {
        p.col[p.all_pairs] = static_cast<short>(c);
        p.step[p.all_pairs] = c + 1 < a->D ? 1 : 0;
    }
    p.units = units;
    p.group = 1;
    while (p.group < units) p.group *= 2;
    const long long rows = a->batch * a->tokens;
    const long long threads = vec ? rows * p.group : rows * 32;
    const long long ctas = (threads + kRotThreads - 1) / kRotThreads;
    // The heads of a token share its sines: they are cut only as far as it takes to give every SM kRotWarps warps, into
    // multiples of the heads that are loaded at a time.
    const int heads = a->heads_q + a->heads_k;
    const long long want = static_cast<long long>(kNumSMs) * kRotWarps * 32 / kRotThreads;
    long long cuts = (want + ctas - 1) / ctas;
    if (cuts > heads) cuts = heads;
    p.heads_per_cta = static_cast<int>((heads + cuts - 1) / cuts);
    if (p.heads_per_cta > kRotAhead) p.heads_per_cta = (p.heads_per_cta + kRotAhead - 1) / kRotAhead * kRotAhead;
    const dim3 grid(static_cast<unsigned>(ctas), static_cast<unsigned>((heads + p.heads_per_cta - 1) / p.heads_per_cta));
    SQ_REQUIRE(ctas < (1ll << 31), SQ_ERR_TOO_LARGE, "sq_rotary: too many rows");
    if (a->dtype == SQ_F32) launch_rotary<float>(p, vec, halves, norm, grid, st);
    else if (a->dtype == SQ_F16) launch_rotary<__half>(p, vec, halves, norm, grid, st);
    else launch_rotary<__nv_bfloat16>(p, vec, halves, norm, grid, st);
    SQ_CUDA_OK(cudaGetLastError());
    return SQ_OK;
}

}  // namespace sq
