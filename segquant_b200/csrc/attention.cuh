// Parameters and tile bookkeeping shared by the attention kernels (attention.cu, attention_rows.cu) and their host side.
#pragma once
#include "common.cuh"

namespace sq {

struct AttnParams {
    // sequences
    const int* q_off;        // packed: batch + 1 token offsets into q / out, or NULL
    const int* kv_off;       // packed: batch + 1 token offsets into k / v
    const int* q_lens;       // not packed: valid queries per sequence, or NULL (= Tq)
    const int* kv_lens;      // not packed: valid keys per sequence, or NULL (= Tk)
    int batch;               // sequences
    int Tq, Tk;              // tokens per sequence; packed: tokens in all
    int fill_rest;           // rows of out that belong to no sequence: 0 = left alone, 1 = written like rows that see no key
    int causal;
    // heads
    int Hq, Hkv, D;
    int P;                   // query heads of one key head that share a tile (rows of a tile are (token, head) pairs)
    int chunks;              // Hq / P
    int G;                   // Hq / Hkv
    // tiles
    int tile_tokens;         // query tokens of a tile
    int tiles;               // upper bound on the number of tiles over all sequences
    int splits;              // parts that the keys of a tile are cut into
    int part_keys;           // rows kernel: keys of a part (the large kernel cuts what a tile sees into equal parts)
    float scale_log2;        // scale * log2(e)
    long long q_bs, q_ts, q_hs, o_bs, o_ts, o_hs;   // element strides: batch, token, head (k and v come as tensor maps)
    const void* q;
    void* out;
    float* lse;              // [batch * Tq (packed: Tq), Hq] natural logarithm of the row sums, or NULL
    float* part_o;           // splits > 1: [splits][tokens * Hq][D], each part normalised by itself
    float* part_lse;         // splits > 1: [splits][tokens * Hq], base-2 logarithm, -inf where a part saw no key
    long long rows;          // tokens * Hq of the whole call
    long long wait_cycles;
};

// The part of the work that one CTA has: query tokens [tok0, tok_end) of sequence b.
struct AttnTile {
    int ok;                  // 0: the tile index lies behind the last tile
    int b;                   // batch coordinate (0 when packed)
    int q_base;              // token index (within batch entry b) of the sequence's first query
    int tok0;                // first query token of the tile, counted from q_base
    int rows_end;            // query tokens from q_base that are stored
    int q_len, kv_len;       // the sequence's valid queries and keys
    int kv_base;             // token index of its first key
};

// Keys that query token `tok` of the sequence sees: [0, limit).  Causal: the last query sits on the last key.
__device__ __forceinline__ int attn_limit(const AttnTile& t, int tok, int causal) {
    if (tok >= t.q_len) return 0;
    if (!causal) return t.kv_len;
    const long long lim = static_cast<long long>(tok) + 1 + t.kv_len - t.q_len;
    return lim < 0 ? 0 : lim > t.kv_len ? t.kv_len : static_cast<int>(lim);
}

// Called by one whole warp.  Finds tile `index` (in the order of the sequences).  Offsets and lengths come from device
// memory and are clamped to the tensors, so a wrong one gives wrong rows, never an access outside.
__device__ __forceinline__ AttnTile attn_find_tile(const AttnParams& p, int index, int lane) {
    AttnTile t;
    t.ok = 0; t.b = 0; t.q_base = 0; t.tok0 = 0; t.rows_end = 0; t.q_len = 0; t.kv_len = 0; t.kv_base = 0;
    if (p.q_off == nullptr) {
        const int per = (p.Tq + p.tile_tokens - 1) / p.tile_tokens;
        const int b = index / per;
        if (b >= p.batch) return t;
        t.ok = 1;
        t.b = b;
        t.tok0 = (index - b * per) * p.tile_tokens;
        t.q_len = p.q_lens ? min(max(p.q_lens[b], 0), p.Tq) : p.Tq;
        t.kv_len = p.kv_lens ? min(max(p.kv_lens[b], 0), p.Tk) : p.Tk;
        t.rows_end = p.fill_rest ? p.Tq : t.q_len;
        return t;
    }
    // Entry 0 and entry batch + 1 stand for the tokens in front of the first and behind the last sequence: no keys.
    int before = 0;                                     // tiles of the entries in front of this round's
    for (int base = 0; base < p.batch + 2; base += 32) {
        const int i = base + lane;
        int q0 = 0, q1 = 0;
        if (i < p.batch + 2) {
            q0 = i == 0 ? 0 : min(max(p.q_off[i - 1], 0), p.Tq);
            q1 = i == p.batch + 1 ? p.Tq : min(max(p.q_off[i], 0), p.Tq);
            if (q1 < q0 || ((i == 0 || i == p.batch + 1) && !p.fill_rest)) q1 = q0;
        }
        const int n = (q1 - q0 + p.tile_tokens - 1) / p.tile_tokens;
        int sum = n;                                    // inclusive sum over the warp
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + sum > index);
        if (hit) {
            const int src = __ffs(hit) - 1;
            const int e = base + src;
            q0 = __shfl_sync(0xffffffffu, q0, src);
            q1 = __shfl_sync(0xffffffffu, q1, src);
            const int first = before + __shfl_sync(0xffffffffu, sum - n, src);
            t.ok = 1;
            t.q_base = q0;
            t.tok0 = (index - first) * p.tile_tokens;
            t.rows_end = q1 - q0;
            if (e > 0 && e <= p.batch) {
                const int k0 = min(max(p.kv_off[e - 1], 0), p.Tk), k1 = min(max(p.kv_off[e], 0), p.Tk);
                t.q_len = q1 - q0;
                t.kv_base = k0;
                t.kv_len = k1 > k0 ? k1 - k0 : 0;
            }
            return t;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return t;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {      // NaN counts as absent, as in fmaxf
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// 2^x of two values on the FMA pipe, for x in [-inf, 100] or NaN (0 below -126.5, so that masked keys weigh nothing):
// x = n + f with n the nearest whole number, 2^n from the low bits of x + 1.5 * 2^23 + 127 (which are those of n + 127; n = -127
// leaves an exponent field of zero: 0) and 2^f from a polynomial of degree 4, 1 + c1 f + ..., fitted to the least largest
// relative error on [-1/2, 1/2] (3e-6; a cubic, 1e-4, is enough for the 16-bit p, but shows in the logarithm of a short row's
// sum).  2^0 is exactly 1.
__device__ __forceinline__ float2 ex2_poly(float2 x) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.x) : "f"(-127.0f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.y) : "f"(-127.0f));
    const float2 big = make_float2(12583039.0f, 12583039.0f), nbig = make_float2(-12583039.0f, -12583039.0f);
    const float2 t = __fadd2_rn(x, big);
    const float2 n = __fadd2_rn(t, nbig);
    const float2 f = __ffma2_rn(n, make_float2(-1.0f, -1.0f), x);
    float2 p = make_float2(0.009582853f, 0.009582853f);
    p = __ffma2_rn(p, f, make_float2(0.055906426f, 0.055906426f));
    p = __ffma2_rn(p, f, make_float2(0.240240986f, 0.240240986f));
    p = __ffma2_rn(p, f, make_float2(0.693124193f, 0.693124193f));
    p = __ffma2_rn(p, f, make_float2(1.0f, 1.0f));
    return __fmul2_rn(p, make_float2(__uint_as_float(__float_as_uint(t.x) << 23), __uint_as_float(__float_as_uint(t.y) << 23)));
}
constexpr float kLn2 = 0.6931471805599453f;

}  // namespace sq
