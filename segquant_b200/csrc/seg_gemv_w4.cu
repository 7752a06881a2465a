// Skinny-M form of the segmented GEMM with packed int4 weights (M <= 8 rows; HBM-bound weight streaming, N * K / 2 bytes).
//
// Same arithmetic as the tensor-core path: per accumulation unit (K-segment x weight-scale group) the products are summed
// exactly in int32, converted to fp32, multiplied by 1 / (s_x * s_w[n]) and added to the running fp32 sum in the order of the
// units (the positive side before the negative one); bias and cast at the end.  The results are the same bits.
//
// A 128-row tile would be 94 % padding and leave the SMs without work for N < 128 * 148 columns.  Here a warp owns 16 output
// columns, which are the 16 rows of mma.sync m16n8k32 (int8): weights are the first operand, up to 8 activation rows the second.
// The warp streams its weight rows through a ring of its own in shared memory (cp.async, kW4Depth blocks of 16 rows x 128
// columns in flight; nothing waits for another warp), a word of 8 nibbles becomes two words of bytes 16 * q (even and odd
// columns) with a shift and two masks, and since the order of the inner dimension is free, the activations wait in shared
// memory with the even and the odd bytes of every 8 columns side by side.  An output lives in one lane from the first unit to
// the last, so the fp32 sum over the units runs in registers.
//
// 16384 x 12288, groups of 128, 4 rows (101 MB of weights and 6 MB of scales, floor 16.4 us): 42 us, 147 us on the 128-row tiles; 7
// warps an SM walk 96 blocks each, some 150 instructions a block (without groups, 29 us).  What bounds it is not established: memory,
// issue slots (33 %) and the tensor pipe (7 %) are far from full.  Measured and not kept:
// dot products on the ALUs (dp4a) 72 us; two blocks a step 51; scales through the ring 43; closing a unit a block later 43;
// tiles of 8 columns on twice the warps 48; three warps to a tile that exchange their integer sums 42 to 52.
#include <cstdlib>

#include "seg_gemm_params.cuh"

namespace sq {

bool gemv_disabled();   // seg_gemm.cu: process-wide schedule overrides

constexpr int kW4Cols = 16;           // output columns of a warp
constexpr int kW4Warps = 8;
constexpr int kW4Depth = 12;          // blocks in flight per warp
constexpr int kW4Row = 80;            // bytes between the rows of a block (64 + 16: rows fall on different banks)
constexpr int kW4Slot = kW4Cols * kW4Row;
constexpr int kW4MaxRows = 8;
constexpr long long kW4XBytes = 97 * 1024;     // activations staged per CTA
constexpr int kW4MaxUnits = 512;      // unit table in shared memory (several segments only)

struct GemvW4Params {
    GemmParams g;
    const uint8_t* xq;
    const uint8_t* xq_neg;
    const uint8_t* wq;
    long long xq_rs, wq_rs;
};

__device__ __forceinline__ float w4_load_sw(const GemmParams& p, long long idx) {
    if (p.sw_is_bf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p.sw)[idx]);
    return static_cast<const float*>(p.sw)[idx];
}
__device__ __forceinline__ void w4_copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void w4_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void w4_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void w4_mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 nibbles -> even and odd columns as bytes 16 * q
__device__ __forceinline__ uint32_t w4_even(uint32_t w) { return (w << 4) & 0xF0F0F0F0u; }
__device__ __forceinline__ uint32_t w4_odd(uint32_t w) { return w & 0xF0F0F0F0u; }

// WIDE: every unit is a multiple of 128 columns (as K is).  A lane then takes 32 consecutive columns of a block, 8 per mma,
// with 16-byte reads; the other form gives mma i the columns 32 i .. 32 i + 31, so that a unit may end behind any of them.
template <bool DUAL, bool WIDE>
__global__ void __launch_bounds__(kW4Warps * 32, 1) seg_gemv_w4_kernel(const __grid_constant__ GemvW4Params q) {
    constexpr int SIDES = DUAL ? 2 : 1;
    extern __shared__ __align__(16) uint8_t smem[];
    const GemmParams& p = q.g;
    const int K = static_cast<int>(p.K), M = static_cast<int>(p.M);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = lane >> 2, t = lane & 3;                          // fragment row (and activation row), quarter of a block
    const int x_row = K + 16;
    uint8_t* ring = smem + warp * (kW4Depth * kW4Slot);
    uint8_t* xs = smem + kW4Warps * (kW4Depth * kW4Slot);           // [SIDES][M][x_row]
    uint32_t* unit_sg = reinterpret_cast<uint32_t*>(xs + static_cast<size_t>(SIDES) * M * x_row);   // several segments: (segment << 16) | group
    const uint32_t ring_u32 = static_cast<uint32_t>(__cvta_generic_to_shared(ring));

    const long long tiles = (p.N + kW4Cols - 1) / kW4Cols;
    long long tile = static_cast<long long>(warp) * gridDim.x + blockIdx.x;
    const int blocks = (K + 127) >> 7;
    const uint8_t *w0 = nullptr, *w1 = nullptr;                     // this lane's 16 bytes of block 0: rows r and r + 8
    auto aim = [&](long long tl) {                                  // rows behind the last column are read as the last one's
        const long long n = tl * kW4Cols + r;
        w0 = q.wq + (n < p.N ? n : p.N - 1) * q.wq_rs + t * 16;
        w1 = q.wq + (n + 8 < p.N ? n + 8 : p.N - 1) * q.wq_rs + t * 16;
    };
    auto fetch = [&](int block) {                                   // always commits, so that the groups count the blocks
        if (block < blocks && (WIDE || block * 128 + t * 32 < K)) {
            const uint32_t dst = ring_u32 + (block % kW4Depth) * kW4Slot + r * kW4Row + t * 16;
            w4_copy16(dst, w0 + block * 64);
            w4_copy16(dst + 8 * kW4Row, w1 + block * 64);
        }
        w4_commit();
    };
    if (tile < tiles) {
        aim(tile);
        for (int i = 0; i < kW4Depth - 1; ++i) fetch(i);
    }

    // activations: per 8 columns the even bytes, then the odd ones
    for (int c = threadIdx.x; c < SIDES * M * (K >> 4); c += blockDim.x) {
        const int v = c / (K >> 4), j = c - v * (K >> 4);
        const int side = DUAL && v >= M;
        const uint4 x = *reinterpret_cast<const uint4*>((side ? q.xq_neg : q.xq) + (side ? v - M : v) * q.xq_rs + j * 16);
        *reinterpret_cast<uint4*>(xs + static_cast<size_t>(v) * x_row + j * 16) =
            make_uint4(__byte_perm(x.x, x.y, 0x6420), __byte_perm(x.x, x.y, 0x7531), __byte_perm(x.z, x.w, 0x6420), __byte_perm(x.z, x.w, 0x7531));
    }
    if (p.num_segs > 1) {
        for (int c = threadIdx.x; c < (K >> 5); c += blockDim.x) {
            const int k = c << 5;
            int s = 0, extra = 0;                                   // units in front of column k: one per segment end and per group end
            while (k >= p.seg_bounds[s + 1]) {
                ++s;
                if (p.group_size > 0 && p.seg_bounds[s] % p.group_size != 0) ++extra;
            }
            const int g = p.group_size > 0 ? k / p.group_size : 0;
            if (k == p.seg_bounds[s] || (p.group_size > 0 && k == g * p.group_size))
                unit_sg[p.group_size > 0 ? g + extra : s] = (static_cast<uint32_t>(s) << 16) | static_cast<uint32_t>(g);
        }
    }
    __syncthreads();

    const bool per_token = p.sx_rs != 0;
    const bool has_x = r < M;                                       // activation rows behind the last one are zero
    const uint8_t* xp = xs + static_cast<size_t>(has_x ? r : 0) * x_row;
    const size_t x_side = static_cast<size_t>(M) * x_row;
    for (; tile < tiles; tile += static_cast<long long>(gridDim.x) * kW4Warps) {
        const long long n0 = tile * kW4Cols + r;
        const long long na = (n0 < p.N ? n0 : p.N - 1) * p.sw_cs, nb = (n0 + 8 < p.N ? n0 + 8 : p.N - 1) * p.sw_cs;
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};                      // (row r, rows 2t and 2t + 1 of x), (row r + 8, the same)
        int acc[SIDES][4] = {};
        float rx[SIDES][2];
        int rx_seg = -1;
        // scales: the lanes of a quad take four units at a time between them, the next four on their way
        float sw_next[2], sx_next[SIDES], rc[SIDES][2];
        auto load_scales = [&](int u) {
            sw_next[0] = sw_next[1] = 1.0f;
#pragma unroll
            for (int i = 0; i < SIDES; ++i) sx_next[i] = 1.0f;
            if (u < p.units) {
                const uint32_t sg = p.num_segs > 1 ? unit_sg[u] : static_cast<uint32_t>(u);
                const long long base = (sg >> 16) * p.sw_ss + (sg & 0xFFFFu) * p.sw_gs;
                sw_next[0] = w4_load_sw(p, base + na);
                sw_next[1] = w4_load_sw(p, base + nb);
                if (!per_token) {
                    sx_next[0] = p.sx[(sg >> 16) * p.sx_ss];
                    if constexpr (DUAL) sx_next[1] = p.sx_neg[(sg >> 16) * p.sx_ss];
                }
            }
        };
        load_scales(t);
        int u = 0, s = 0, g = 0;
        auto unit_end = [&]() {
            const int seg_end = p.seg_bounds[s + 1];
            const int grp_end = p.group_size > 0 ? (g + 1) * p.group_size : seg_end;
            return grp_end < seg_end ? grp_end : seg_end;
        };
        int k1 = unit_end();
        auto close_unit = [&]() {
            if ((u & 3) == 0) {
#pragma unroll
                for (int i = 0; i < SIDES; ++i) {
                    rc[i][0] = __frcp_rn(sx_next[i] * sw_next[0]);
                    rc[i][1] = __frcp_rn(sx_next[i] * sw_next[1]);
                }
                load_scales(u + 4 + t);
            }
            if (per_token && rx_seg != s) {
                rx_seg = s;
#pragma unroll
                for (int i = 0; i < SIDES; ++i)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int m = 2 * t + c;
                        rx[i][c] = m < M ? __frcp_rn((i ? p.sx_neg : p.sx)[s * p.sx_ss + m * p.sx_rs]) : 1.0f;
                    }
            }
#pragma unroll
            for (int i = 0; i < SIDES; ++i) {
                const float ra = __shfl_sync(0xffffffffu, rc[i][0], (lane & 28) | (u & 3)), rb = __shfl_sync(0xffffffffu, rc[i][1], (lane & 28) | (u & 3));
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float f = c < 2 ? ra : rb;
                    if (per_token) f *= rx[i][c & 1];
                    y[c] = fmaf(static_cast<float>(acc[i][c] >> 4), f, y[c]);        // weights were multiplied as 16 * q
                    acc[i][c] = 0;
                }
            }
            if (p.group_size > 0 && k1 == (g + 1) * p.group_size) ++g;
            if (k1 == p.seg_bounds[s + 1]) ++s;
            ++u;
            if (u < p.units) k1 = unit_end();
        };

        for (int b = 0; b < blocks; ++b) {
            w4_wait<kW4Depth - 2>();                                // block b is there
            __syncwarp();                                           // for every lane, and block b - 1 has been read by all
            fetch(b + kW4Depth - 1);
            const uint8_t* slot = ring + (b % kW4Depth) * kW4Slot + r * kW4Row;
            if constexpr (WIDE) {
                const uint4 a = *reinterpret_cast<const uint4*>(slot + t * 16), c = *reinterpret_cast<const uint4*>(slot + 8 * kW4Row + t * 16);
                const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wc[4] = {c.x, c.y, c.z, c.w};
                uint32_t xw[SIDES][8];
#pragma unroll
                for (int i = 0; i < SIDES; ++i) {
                    uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
                    if (has_x) {
                        lo = *reinterpret_cast<const uint4*>(xp + i * x_side + b * 128 + t * 32);
                        hi = *reinterpret_cast<const uint4*>(xp + i * x_side + b * 128 + t * 32 + 16);
                    }
                    xw[i][0] = lo.x; xw[i][1] = lo.y; xw[i][2] = lo.z; xw[i][3] = lo.w;
                    xw[i][4] = hi.x; xw[i][5] = hi.y; xw[i][6] = hi.z; xw[i][7] = hi.w;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t a0 = w4_even(wa[j]), a1 = w4_even(wc[j]), a2 = w4_odd(wa[j]), a3 = w4_odd(wc[j]);
#pragma unroll
                    for (int i = 0; i < SIDES; ++i) w4_mma(acc[i], a0, a1, a2, a3, xw[i][2 * j], xw[i][2 * j + 1]);
                }
                if (b * 128 + 128 == k1) close_unit();
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (b * 128 + j * 32 < K) {
                        const uint32_t wa = *reinterpret_cast<const uint32_t*>(slot + j * 16 + t * 4), wc = *reinterpret_cast<const uint32_t*>(slot + 8 * kW4Row + j * 16 + t * 4);
                        const uint32_t a0 = w4_even(wa), a1 = w4_even(wc), a2 = w4_odd(wa), a3 = w4_odd(wc);
#pragma unroll
                        for (int i = 0; i < SIDES; ++i) {
                            uint2 x = make_uint2(0u, 0u);
                            if (has_x) x = *reinterpret_cast<const uint2*>(xp + i * x_side + b * 128 + j * 32 + t * 8);
                            w4_mma(acc[i], a0, a1, a2, a3, x.x, x.y);
                        }
                        if (b * 128 + j * 32 + 32 == k1) close_unit();
                    }
                }
            }
        }
        w4_wait<0>();
        __syncwarp();
        const long long n_out[2] = {n0, n0 + 8};
        const long long next = tile + static_cast<long long>(gridDim.x) * kW4Warps;
        if (next < tiles) {
            aim(next);
            for (int i = 0; i < kW4Depth - 1; ++i) fetch(i);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const long long n = n_out[c >> 1];
            const int m = 2 * t + (c & 1);
            if (n >= p.N || m >= M) continue;
            float v = y[c];
            if (p.bias != nullptr) {
                if (p.bias_dtype == SQ_F32) v += static_cast<const float*>(p.bias)[n];
                else if (p.bias_dtype == SQ_F16) v += __half2float(static_cast<const __half*>(p.bias)[n]);
                else v += __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n]);
            }
            const long long oi = m * p.y_rs + n;
            if (p.out_dtype == SQ_F32) static_cast<float*>(p.y)[oi] = v;
            else if (p.out_dtype == SQ_F16) static_cast<__half*>(p.y)[oi] = __float2half_rn(v);
            else static_cast<__nv_bfloat16*>(p.y)[oi] = __float2bfloat16_rn(v);
        }
    }
}

static long long w4_x_bytes(const sq_gemm_args* a, bool dual) { return (dual ? 2 : 1) * a->M * (a->K + 16); }

// True when the skinny path serves this problem (the caller has validated the arguments).  Against the 128-row tiles it was faster
// at every one of 668 sizes that it serves (1, 2, 4, 8 rows; 16 to 16384 columns; K 256 to 65536; no groups, 32, 64, 128; one side or two):
// 1.8 to 9.4 times.  16384 x 12288, us on this path / on tiles, 1 and 8 rows: no groups 24 / 75 and 35 / 72, groups of 128 39 / 146 and
// 49 / 147, of 64 75 / 274 and 84 / 273, of 32 113 / 531 and 123 / 529.  The rows have to fit shared memory: 8 rows up to K = 12400, with
// two sides 6192; behind that a call is on tiles again (8 rows, two sides, groups of 128, 16384 x 12288: 328 us; 4 rows fit and take 57).
bool gemv_w4_applies(const sq_gemm_args* a, bool dual, int units) {
    if (a->kind != SQ_GEMM_W4A8 || a->batch != 1 || a->M > kW4MaxRows || a->acc_dump_dev != nullptr || a->num_peer_outputs != 0 || a->w_seg_as_batch)
        return false;
    if (gemv_disabled()) return false;   // SEGQUANT_B200_NO_GEMV=1 or sq_set_gemm_schedule(): tensor-core path only
    return (a->num_segs == 1 || units <= kW4MaxUnits) && a->K <= 65536 && w4_x_bytes(a, dual) <= kW4XBytes;
}

template <bool DUAL, bool WIDE>
static int launch_w4(const GemvW4Params& q, long long x_bytes, cudaStream_t st) {
    constexpr long long kRings = kW4Warps * kW4Depth * kW4Slot;
    constexpr int kMax = static_cast<int>(kRings + kW4XBytes + kW4MaxUnits * 4);
    static_assert(kMax <= 227 * 1024, "shared memory of the skinny int4 kernel");
    static bool attr_set[64] = {};
    int dev = 0;
    SQ_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 64 || !attr_set[dev]) {
        SQ_CUDA_OK(cudaFuncSetAttribute(seg_gemv_w4_kernel<DUAL, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMax));
        if (dev < 64) attr_set[dev] = true;
    }
    const long long tiles = (q.g.N + kW4Cols - 1) / kW4Cols;
    const long long ctas = tiles < kNumSMs ? tiles : kNumSMs;        // one CTA per SM; its warps take tiles gridDim.x apart
    const size_t smem = static_cast<size_t>(kRings + x_bytes + (q.g.num_segs > 1 ? q.g.units * 4 : 0));
    seg_gemv_w4_kernel<DUAL, WIDE><<<static_cast<unsigned>(ctas), kW4Warps * 32, smem, st>>>(q);
    SQ_CUDA_OK(cudaGetLastError());
    return SQ_OK;
}

int launch_gemv_w4(const GemmParams& p, const sq_gemm_args* a, bool dual, cudaStream_t st) {
    GemvW4Params q;
    q.g = p;
    q.xq = static_cast<const uint8_t*>(a->xq_dev);
    q.xq_neg = static_cast<const uint8_t*>(a->xq_neg_dev);
    q.wq = static_cast<const uint8_t*>(a->wq_dev);
    q.xq_rs = a->xq_row_stride;
    q.wq_rs = a->wq_row_stride;
    bool wide = a->group_size % 128 == 0;
    for (int s = 1; s <= a->num_segs; ++s) wide = wide && a->seg_bounds[s] % 128 == 0;
    const long long xb = w4_x_bytes(a, dual);
    if (dual) return wide ? launch_w4<true, true>(q, xb, st) : launch_w4<true, false>(q, xb, st);
    return wide ? launch_w4<false, true>(q, xb, st) : launch_w4<false, false>(q, xb, st);
}

}  // namespace sq
