// Attention of few rows against many keys (a new token each of a batch of sequences): HBM-bound, every key and value is read
// once and used by the handful of query heads that share it.
//
// A tile is at most 16 rows ((query token, query head) pairs of one key head), a CTA has one tile and one part of its keys.
// A 128-row tile of the large kernel would be mostly empty rows and its chain of barriers would run once per 128 keys; here
// each of four warps works on key blocks of its own (32 keys, in turn), with mma.sync m16n8k16 from registers to registers: S
// of a block is in the layout that the product with v wants its first operand in.  Loads go through a ring of blocks that the
// warps share; the warp that is done with a block's slot orders the next block into it, so nothing but the loads is ever
// waited for.  The warps' maxima, sums and outputs are joined in shared memory, the parts of a row by a second kernel behind this
// one.  32 caches of 369 to 16001 keys, 8 key heads of 128, 32 query heads: 182 us = 6.0 TB/s of the 1.1 GB (copy bandwidth 6.55);
// one cache of 1531 keys, 8 heads of 64: 9 to 10 us, of which the two launches and one round trip to memory each are most.
#include <cuda.h>

#include <type_traits>

#include "attention.cuh"
#include "ptx.cuh"

namespace sq {

constexpr int kRowsThreads = 128;
constexpr int kRowsKeys = 32;        // keys of a block
enum RowsWait : int { kRowsFull = 30 };
// Weights (at most 1) are rounded once to the 16-bit type for the product with v, half a step (2^-8 in bf16, 2^-11 in fp16) of each
// term.  fp16 has no more than steps of 2^-24 below 2^-14, where many keys of small weight beside a strong one would lose theirs:
// its weights go in 2^14 times as large, and half a step is at most 2^-39 of the largest.
template <typename T>
constexpr float kRowsUp = std::is_same<T, __half>::value ? 16384.0f : 1.0f;

template <int DP>
struct RowsCfg {
    static constexpr uint32_t kHalf = kRowsKeys * 128;             // 32 rows of 64 16-bit columns
    static constexpr uint32_t kTile = kHalf * (DP / 64);
    // A multiple of the warps: a slot's blocks then belong to one warp, which waits for them in order.  (A wait for a slot's
    // next block by a warp that has not seen the one before complete would pass at once: barriers tell phases by parity.)
    static constexpr int kStages = DP == 64 ? 8 : 4;
    static_assert(kStages % 4 == 0, "a slot belongs to one warp");
    static constexpr int kPad = DP + 4;                            // floats between the rows of a warp's output
    static constexpr uint32_t kRing = kStages * 2 * kTile;         // the joining of the warps reuses it
    static constexpr uint32_t kSmem = 1024 + kRing;
};

__device__ __forceinline__ void ldsm(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void rows_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void rows_mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void rows_mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int DP>
__global__ void __launch_bounds__(kRowsThreads, 2)
attention_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnParams p) {
    using C = RowsCfg<DP>;
    constexpr int ST = C::kStages;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[ST];
    __shared__ AttnTile tile_s;
    __shared__ int abort_s;
    __shared__ float m_s[4][16], l_s[4][16];
    volatile int* abort_flag = &abort_s;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const uint32_t sbase = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int split = blockIdx.x % p.splits;
    const int rest = blockIdx.x / p.splits;
    const int chunk = rest % p.chunks;
    if (warp == 0) {
        const AttnTile t = attn_find_tile(p, rest / p.chunks, lane);
        if (lane == 0) { tile_s = t; abort_s = 0; }
    } else if (warp == 1 && lane == 0) {
        for (int s = 0; s < ST; ++s) mbar_init(smem_u32(&bar_full[s]), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_tmap(&map_k);
        prefetch_tmap(&map_v);
    }
    __syncthreads();
    const AttnTile T0 = tile_s;
    if (!T0.ok) return;
    const int last = min(T0.tok0 + p.tile_tokens, T0.rows_end) - 1;
    if (last < T0.tok0) return;
    const int see = T0.tok0 < T0.q_len ? attn_limit(T0, min(last, T0.q_len - 1), p.causal) : 0;      // the rows' largest limit
    const int k_lo = min(static_cast<long long>(split) * p.part_keys, static_cast<long long>(see));
    const int k_hi = min(k_lo + p.part_keys, see);
    const int blocks = (k_hi - k_lo + kRowsKeys - 1) / kRowsKeys;

    const int kvh = chunk / (p.G / p.P);
    auto order = [&](int i) {                                      // one lane: block i into its slot
        const int s = i % ST;
        const uint32_t bar = smem_u32(&bar_full[s]), dst = sbase + s * 2 * C::kTile;
        const int tok = T0.kv_base + k_lo + i * kRowsKeys;
        mbar_arrive_expect_tx(bar, 2 * C::kTile);
        for (int h = 0; h < DP / 64; ++h) tma_load_4d(dst + h * C::kHalf, &map_k, h * 64, kvh, tok, T0.b, bar);
        for (int h = 0; h < DP / 64; ++h) tma_load_4d(dst + C::kTile + h * C::kHalf, &map_v, h * 64, kvh, tok, T0.b, bar);
    };
    if (threadIdx.x == 0)
        for (int i = 0; i < ST && i < blocks; ++i) order(i);

    // this lane's rows of the fragments: r and r + 8
    const int r = lane >> 2, t = lane & 3;
    int limit[2];
    uint32_t qf[DP / 16][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = r + 8 * i;
        const int tok = T0.tok0 + row / p.P, head = chunk * p.P + row % p.P;
        const bool mine = row < p.tile_tokens * p.P && tok <= last;
        limit[i] = mine ? attn_limit(T0, tok, p.causal) : 0;
        const T* q = static_cast<const T*>(p.q) + static_cast<long long>(T0.b) * p.q_bs + static_cast<long long>(T0.q_base + tok) * p.q_ts +
                     static_cast<long long>(head) * p.q_hs;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int col = 16 * k + 8 * h + 2 * t;
                qf[k][2 * h + i] = mine && col < p.D ? *reinterpret_cast<const uint32_t*>(q + col) : 0u;
            }
    }

    float o[DP / 8][4];
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[n][c] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    const float sc = p.scale_log2;
    // ldmatrix rows of this lane: k (16 keys x 16 columns): key 8 * (lane / 16) + lane % 8, column half (lane / 8) % 2;
    // v (16 keys x 16 columns, transposed): key 8 * ((lane / 8) % 2) + lane % 8, column half lane / 16
    const int kr = ((lane >> 4) << 3) | (lane & 7), kc = (lane >> 3) & 1;
    const int vr = (((lane >> 3) & 1) << 3) | (lane & 7), vc = lane >> 4;
    for (int i = warp; i < blocks; i += 4) {
        const int s = i % ST;
        if (!mbar_wait_warp(smem_u32(&bar_full[s]), (i / ST) & 1u, abort_flag, kRowsFull, p.wait_cycles)) break;
        const uint32_t ks = sbase + s * 2 * C::kTile, vs = ks + C::kTile;
        const int key0 = k_lo + i * kRowsKeys;
        const int valid = T0.kv_len - key0;
        if (valid < kRowsKeys) {                                   // rows behind the last key may hold NaN, and 0 * NaN is NaN
            uint8_t* v = smem + (s * 2 + 1) * C::kTile;
            for (int h = 0; h < DP / 64; ++h)
                for (int x = valid * 8 + lane; x < kRowsKeys * 8; x += 32) *reinterpret_cast<uint4*>(v + h * C::kHalf + x * 16) = make_uint4(0u, 0u, 0u, 0u);
            __syncwarp();
        }
        float sa[kRowsKeys / 8][4];
#pragma unroll
        for (int n = 0; n < kRowsKeys / 8; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) sa[n][c] = 0.0f;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
            for (int n = 0; n < kRowsKeys / 16; ++n) {
                const int row = n * 16 + kr, piece = (2 * k + kc) & 7;
                uint32_t b[4];
                ldsm(ks + (k >> 2) * C::kHalf + row * 128 + ((piece ^ (row & 7)) << 4), b);
                rows_mma<T>(sa[2 * n], qf[k], b[0], b[1]);
                rows_mma<T>(sa[2 * n + 1], qf[k], b[2], b[3]);
            }
        }
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < kRowsKeys / 8; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                sa[n][c] = key0 + 8 * n + 2 * t + (c & 1) < limit[c >> 1] ? sa[n][c] * sc : -INFINITY;
                mx[c >> 1] = fmaxf(mx[c >> 1], sa[n][c]);
            }
        float f[2], ms[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
            mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
            const float mn = fmaxf(m[x], mx[x]);
            ms[x] = mn == -INFINITY ? 0.0f : mn;
            f[x] = m[x] == mn ? 1.0f : ex2(m[x] - ms[x]);
            m[x] = mn;
            l[x] *= f[x];
        }
        if (__any_sync(0xffffffffu, f[0] != 1.0f || f[1] != 1.0f)) {
#pragma unroll
            for (int n = 0; n < DP / 8; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[n][c] *= f[c >> 1];
        }
        uint32_t pf[kRowsKeys / 16][4];
#pragma unroll
        for (int n = 0; n < kRowsKeys / 8; ++n) {
            float e[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                e[c] = ex2(sa[n][c] - ms[c >> 1]);
                l[c >> 1] += e[c];
            }
            pf[n >> 1][2 * (n & 1)] = pack2<T>(e[0] * kRowsUp<T>, e[1] * kRowsUp<T>);
            pf[n >> 1][2 * (n & 1) + 1] = pack2<T>(e[2] * kRowsUp<T>, e[3] * kRowsUp<T>);
        }
#pragma unroll
        for (int k = 0; k < kRowsKeys / 16; ++k) {
#pragma unroll
            for (int n = 0; n < DP / 16; ++n) {
                const int row = k * 16 + vr, piece = (2 * n + vc) & 7;
                uint32_t b[4];
                ldsm_t(vs + (n >> 2) * C::kHalf + row * 128 + ((piece ^ (row & 7)) << 4), b);
                rows_mma<T>(o[2 * n], pf[k], b[0], b[1]);
                rows_mma<T>(o[2 * n + 1], pf[k], b[2], b[3]);
            }
        }
        __syncwarp();                                              // every lane has read the slot
        if (lane == 0 && i + ST < blocks) order(i + ST);
    }
    __syncthreads();
    if (*abort_flag) {
        // give copies that may still be in flight time to land before shared memory is released
        const unsigned long long t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
        return;
    }
    // ---- the warps' results, row by row (the ring's loads are all in)
    float* o_s = reinterpret_cast<float*>(smem) + warp * 16 * C::kPad;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
        l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
        if (t == 0) {
            m_s[warp][r + 8 * x] = m[x];
            l_s[warp][r + 8 * x] = l[x];
        }
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) *reinterpret_cast<float2*>(o_s + (r + 8 * x) * C::kPad + 8 * n + 2 * t) = make_float2(o[n][2 * x], o[n][2 * x + 1]);
    }
    __syncthreads();
    const int rows = p.tile_tokens * p.P;
    const int pieces = p.D >> 2;                                   // four columns to a thread
    for (int x = threadIdx.x; x < rows * pieces; x += kRowsThreads) {
        const int row = x / pieces, col = (x - row * pieces) * 4;
        const int tok = T0.tok0 + row / p.P, head = chunk * p.P + row % p.P;
        if (tok > last) break;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, m_s[w][row]);
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (m_s[w][row] == -INFINITY && !(l_s[w][row] != l_s[w][row])) continue;      // saw no key of this row
            const float g = ex2(m_s[w][row] - (top == -INFINITY ? 0.0f : top));
            const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem) + (w * 16 + row) * C::kPad + col);
            sum = fmaf(g, l_s[w][row], sum);
            acc.x = fmaf(g, v.x, acc.x); acc.y = fmaf(g, v.y, acc.y); acc.z = fmaf(g, v.z, acc.z); acc.w = fmaf(g, v.w, acc.w);
        }
        const bool empty = top == -INFINITY && sum == 0.0f;
        const float inv = empty ? 0.0f : 1.0f / sum * (1.0f / kRowsUp<T>);
        const long long token = static_cast<long long>(T0.b) * (p.q_off ? 0 : p.Tq) + T0.q_base + tok;
        const long long rr = token * p.Hq + head;
        const float lse2 = empty ? -INFINITY : top + log2f(sum);
        if (p.splits > 1) {
            if (col == 0) p.part_lse[split * p.rows + rr] = lse2;
            if (!empty) *reinterpret_cast<float4*>(p.part_o + (split * p.rows + rr) * p.D + col) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        } else {
            if (col == 0 && p.lse) p.lse[rr] = empty ? -INFINITY : lse2 * kLn2;
            T* out = static_cast<T*>(p.out) + static_cast<long long>(T0.b) * p.o_bs + static_cast<long long>(T0.q_base + tok) * p.o_ts +
                     static_cast<long long>(head) * p.o_hs;
            *reinterpret_cast<uint2*>(out + col) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
        }
    }
}

template <typename T, int DP>
static int launch_rows(const CUtensorMap& mk, const CUtensorMap& mv, const AttnParams& p, long long grid, cudaStream_t st) {
    using C = RowsCfg<DP>;
    static_assert(4u * 16u * C::kPad * 4u <= C::kRing, "the warps' outputs fit the ring");
    static bool attr_set[64] = {};
    int dev = 0;
    SQ_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 64 || !attr_set[dev]) {
        SQ_CUDA_OK(cudaFuncSetAttribute(attention_rows_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
        if (dev < 64) attr_set[dev] = true;
    }
    attention_rows_kernel<T, DP><<<static_cast<unsigned>(grid), kRowsThreads, C::kSmem, st>>>(mk, mv, p);
    SQ_CUDA_OK(cudaGetLastError());
    return SQ_OK;
}

int attention_rows(int dtype, const CUtensorMap& mk, const CUtensorMap& mv, const AttnParams& p, long long grid, cudaStream_t st) {
    if (dtype == SQ_F16) return p.D <= 64 ? launch_rows<__half, 64>(mk, mv, p, grid, st) : launch_rows<__half, 128>(mk, mv, p, grid, st);
    return p.D <= 64 ? launch_rows<__nv_bfloat16, 64>(mk, mv, p, grid, st) : launch_rows<__nv_bfloat16, 128>(mk, mv, p, grid, st);
}

long long attention_rows_read_status() {
    unsigned long long v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_wait_status, sizeof(v)) != cudaSuccess) return SQ_ERR_CUDA;
    if (v != 0 && cudaMemcpyToSymbol(g_wait_status, &zero, sizeof(zero)) != cudaSuccess) return SQ_ERR_CUDA;
    return static_cast<long long>(v);
}

}  // namespace sq
