// Rotary positions with several axes on the heads of q and k, optionally behind the RMS normalisation of each head (HBM-bound).
//
// The columns of a head are cut into one block per axis (time, height, width, ...), columns behind the last block stay as
// they are.  Pair i of axis a turns by the angle  position[token, a] * theta^(-2 i / width_a):
//     (y0, y1) -> (y0 cos - y1 sin, y0 sin + y1 cos),   y = x or x * rsqrt(mean(x^2) + eps) * weight.
// Angles of far positions lose everything in fp32 (position 10^5 leaves 2^-7 of a radian), so the turn is counted in
// revolutions in fp64, reduced to [-1/2, 1/2] there and only then rounded: one fp64 multiplication per (token, pair).  A
// thread keeps the sines of its columns in registers and walks the heads, which share them.  Everything else is fp32 with
// one rounding at the end.
#include <cmath>

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
    int D, pairs;                     // rotated pairs
    int pos_float;
    int heads_per_cta;                // heads (of q, then of k) that one CTA's threads walk
    int group;                        // vector kernel: threads that share a row (power of two)
    int units;                        // vector kernel: threads of a group that have columns
    float eps;
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

// 8 elements <-> floats
template <typename T>
__device__ __forceinline__ void rot_load8(const T* p, float (&v)[8]);
template <>
__device__ __forceinline__ void rot_load8<float>(const float* p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <>
__device__ __forceinline__ void rot_load8<__half>(const __half* p, float (&v)[8]) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
template <>
__device__ __forceinline__ void rot_load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
template <typename T>
__device__ __forceinline__ void rot_store8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const T lo = from_float<T>(v[2 * i]), hi = from_float<T>(v[2 * i + 1]);
            w[i] = static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&lo)) | (static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&hi)) << 16);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// A thread has one vector of 8 columns (adjacent pairs: 4 pairs) or two (halves: 8 pairs, one column of each in either
// vector) of one token, and walks heads.  `group` threads share a row.
template <typename T, bool HALVES, bool NORM>
__global__ void __launch_bounds__(256) rotary_vec_kernel(const __grid_constant__ RotaryParams p) {
    constexpr int NV = HALVES ? 2 : 1, NP = HALVES ? 8 : 4;
    const int u = threadIdx.x & (p.group - 1);
    const long long rows = p.batch * p.tokens;
    const long long row = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) / p.group;
    const bool has = row < rows && u < p.units;
    const long long b = has ? row / p.tokens : 0, t = has ? row - b * p.tokens : 0;
    int cols[NV];
    float cs[NP], sn[NP];
    const int uu = has ? u : 0;
    if constexpr (HALVES) {
        cols[0] = p.unit_a[uu];
        cols[1] = p.unit_b[uu];
    } else {
        cols[0] = 8 * uu;
    }
    const int pair0 = HALVES ? p.unit_pair[uu] : 4 * uu;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        float2 a = make_float2(1.0f, 0.0f);
        if (has && pair0 >= 0 && pair0 + i < p.pairs) a = rot_angle(p, b, t, pair0 + i);
        cs[i] = a.x;
        sn[i] = a.y;
    }
    const int h0 = blockIdx.y * p.heads_per_cta, h1 = min(h0 + p.heads_per_cta, p.heads[0] + p.heads[1]);
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        const int first = part ? max(h0 - p.heads[0], 0) : h0, last = part ? h1 - p.heads[0] : min(h1, p.heads[0]);
        if (first >= last) continue;                                     // uniform over the CTA
        const T* x = static_cast<const T*>(p.x[part]) + b * p.x_bs[part] + t * p.x_ts[part];
        T* y = static_cast<T*>(p.y[part]) + b * p.y_bs[part] + t * p.y_ts[part];
        float w[NV][8];
        if constexpr (NORM) {
#pragma unroll
            for (int v = 0; v < NV; ++v) rot_load8<T>(static_cast<const T*>(p.weight[part]) + cols[v], w[v]);
        }
#pragma unroll 4
        for (int h = first; h < last; ++h) {
            float e[NV][8];
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (has) {
                    rot_load8<T>(x + h * p.x_hs[part] + cols[v], e[v]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) e[v][i] = 0.0f;
                }
            }
            if constexpr (NORM) {
                float ss = 0.0f;
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int i = 0; i < 8; ++i) ss = fmaf(e[v][i], e[v][i], ss);
                for (int o = p.group >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const float r = rsqrtf(ss / static_cast<float>(p.D) + p.eps);
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int i = 0; i < 8; ++i) e[v][i] *= r * w[v][i];
            }
            if (has) {
                float o[NV][8];
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    if constexpr (HALVES) {
                        o[0][i] = e[0][i] * cs[i] - e[1][i] * sn[i];
                        o[1][i] = e[0][i] * sn[i] + e[1][i] * cs[i];
                    } else {
                        o[0][2 * i] = e[0][2 * i] * cs[i] - e[0][2 * i + 1] * sn[i];
                        o[0][2 * i + 1] = e[0][2 * i] * sn[i] + e[0][2 * i + 1] * cs[i];
                    }
                }
#pragma unroll
                for (int v = 0; v < NV; ++v) rot_store8<T>(y + h * p.y_hs[part] + cols[v], o[v]);
            }
        }
    }
}

// Any width, stride and alignment: one warp per token, lane l has the pairs l, l + 32, ... and walks heads.
template <typename T, bool NORM>
__global__ void __launch_bounds__(256) rotary_scalar_kernel(const __grid_constant__ RotaryParams p) {
    constexpr int NP = kRotMaxPairs / 32;
    const int lane = threadIdx.x & 31;
    const long long row = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    if (row >= p.batch * p.tokens) return;
    const long long b = row / p.tokens, t = row - b * p.tokens;
    float cs[NP], sn[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i)
        if (lane + 32 * i < p.pairs) {
            const float2 a = rot_angle(p, b, t, lane + 32 * i);
            cs[i] = a.x;
            sn[i] = a.y;
        }
    const int h0 = blockIdx.y * p.heads_per_cta, h1 = min(h0 + p.heads_per_cta, p.heads[0] + p.heads[1]);
    for (int hh = h0; hh < h1; ++hh) {
        const int part = hh >= p.heads[0], h = part ? hh - p.heads[0] : hh;
        const T* x = static_cast<const T*>(p.x[part]) + b * p.x_bs[part] + t * p.x_ts[part] + h * p.x_hs[part];
        T* y = static_cast<T*>(p.y[part]) + b * p.y_bs[part] + t * p.y_ts[part] + h * p.y_hs[part];
        const T* w = static_cast<const T*>(p.weight[part]);
        float r = 1.0f;
        if constexpr (NORM) {
            float ss = 0.0f;
            for (int i = lane; i < p.D; i += 32) {
                const float v = to_float<T>(x[i]);
                ss = fmaf(v, v, ss);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            r = rsqrtf(ss / static_cast<float>(p.D) + p.eps);
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int pair = lane + 32 * i;
            if (pair < p.pairs) {
                const int a = p.col[pair], c = a + p.step[pair];
                float u = to_float<T>(x[a]), v = to_float<T>(x[c]);
                if constexpr (NORM) {
                    u *= r * to_float<T>(w[a]);
                    v *= r * to_float<T>(w[c]);
                }
                y[a] = from_float<T>(u * cs[i] - v * sn[i]);
                y[c] = from_float<T>(u * sn[i] + v * cs[i]);
            }
        }
        for (int i = 2 * p.pairs + lane; i < p.D; i += 32) {
            float v = to_float<T>(x[i]);
            if constexpr (NORM) v *= r * to_float<T>(w[i]);
            y[i] = from_float<T>(v);
        }
        __syncwarp();
    }
}

template <typename T>
static void launch_rotary(const RotaryParams& p, bool vec, bool halves, bool norm, dim3 grid, cudaStream_t st) {
    if (!vec) {
        if (norm) rotary_scalar_kernel<T, true><<<grid, 256, 0, st>>>(p);
        else rotary_scalar_kernel<T, false><<<grid, 256, 0, st>>>(p);
    } else if (halves) {
        if (norm) rotary_vec_kernel<T, true, true><<<grid, 256, 0, st>>>(p);
        else rotary_vec_kernel<T, true, false><<<grid, 256, 0, st>>>(p);
    } else {
        if (norm) rotary_vec_kernel<T, false, true><<<grid, 256, 0, st>>>(p);
        else rotary_vec_kernel<T, false, false><<<grid, 256, 0, st>>>(p);
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
    p.pos = a->positions_dev; p.pos_float = a->positions_float ? 1 : 0;
    p.pos_bs = a->pos_batch_stride; p.pos_ts = a->pos_token_stride;
    p.batch = a->batch; p.tokens = a->tokens; p.D = a->D; p.pairs = width / 2; p.eps = a->eps;
    p.units = units;
    p.group = 1;
    while (p.group < units) p.group *= 2;
    const long long rows = a->batch * a->tokens;
    const long long threads = vec ? rows * p.group : rows * 32;
    const long long ctas = (threads + 255) / 256;
    // the heads of a token share its sines: cut them only as far as it takes to give every SM its threads
    const int heads = a->heads_q + a->heads_k;
    long long cuts = (8ll * kNumSMs + ctas - 1) / ctas;
    if (cuts > heads) cuts = heads;
    p.heads_per_cta = static_cast<int>((heads + cuts - 1) / cuts);
    const dim3 grid(static_cast<unsigned>(ctas), static_cast<unsigned>((heads + p.heads_per_cta - 1) / p.heads_per_cta));
    SQ_REQUIRE(ctas < (1ll << 31), SQ_ERR_TOO_LARGE, "sq_rotary: too many rows");
    if (a->dtype == SQ_F32) launch_rotary<float>(p, vec, halves, norm, grid, st);
    else if (a->dtype == SQ_F16) launch_rotary<__half>(p, vec, halves, norm, grid, st);
    else launch_rotary<__nv_bfloat16>(p, vec, halves, norm, grid, st);
    SQ_CUDA_OK(cudaGetLastError());
    return SQ_OK;
}

}  // namespace sq
