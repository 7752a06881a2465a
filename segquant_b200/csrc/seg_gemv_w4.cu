// Skinny-M form of the segmented GEMM with packed int4 weights (M <= 4 rows; HBM-bound weight streaming, N * K / 2 bytes).
//
// Same arithmetic as the tensor-core path: per accumulation unit (K-segment x weight-scale group) the products are summed
// exactly in int32, converted to fp32, multiplied by 1 / (s_x * s_w[n]) and added to the running fp32 sum in the order of the
// units (the positive side before the negative one); bias and cast at the end.  The results are the same bits.
//
// A warp owns kW4Cols output columns and walks their weight rows in steps of 512 bytes: a lane takes 16 bytes of each row
// (32 values, which lie in one unit: units are multiples of 32), the next step's loads in flight while this one's are
// multiplied.  A nibble pair becomes two bytes 16 * q (even and odd columns) with a shift and a mask, so the activations wait
// in shared memory with the even and the odd bytes of every 8 columns side by side, and four products are one dp4a.  The lanes
// that share a unit join their sums by halving the columns each holds and add them, as integers, to the unit's words in shared
// memory.  After a step all lanes turn the scales of the units that are complete into reciprocals, and one lane per output
// adds these units to its running sum.
#include <cstdlib>

#include "seg_gemm_params.cuh"

namespace sq {

bool gemv_disabled();   // seg_gemm.cu: process-wide schedule overrides

constexpr int kW4Cols = 4;           // columns a warp has in flight
constexpr int kW4MaxRows = 4;
constexpr long long kW4XBytes = 96 * 1024;     // activations staged per CTA
constexpr int kW4MaxUnits = 1024;    // unit table in shared memory
constexpr long long kW4MaxK = 64 * 1024;

struct GemvW4Params {
    GemmParams g;
    const uint8_t* xq;
    const uint8_t* xq_neg;
    const uint8_t* wq;
    long long xq_rs, wq_rs;
    int join;             // lanes that are sure to share a unit (power of two): every unit is a multiple of 32 * join columns
    int slots;            // units whose sums a warp holds (power of two): a step completes 32 / join at most and leaves one open
};

__device__ __forceinline__ float w4_load_sw(const GemmParams& p, long long idx) {
    if (p.sw_is_bf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p.sw)[idx]);
    return static_cast<const float*>(p.sw)[idx];
}

// shared memory: activations, per-warp sums and scales, unit tables
template <bool DUAL, int MR>
struct W4Smem {
    static constexpr int V = (DUAL ? 2 : 1) * MR;                 // sums of one column and unit
    static constexpr int kWarps = V == 8 ? 8 : 16;                // so that the widest form has its registers and its shared memory
    static constexpr int warp_ints(int slots) { return (V + (DUAL ? 2 : 1)) * slots * kW4Cols; }
    static constexpr long long x_bytes(long long K) { return V * K; }
    static constexpr long long bytes(long long K, int units, int slots) {
        return x_bytes(K) + kWarps * warp_ints(slots) * 4ll + (K / 32 + 1) * 2 + 2 + units * 4ll + 16;
    }
};

template <bool DUAL, int MR>
__global__ void __launch_bounds__(W4Smem<DUAL, MR>::kWarps * 32, 2) seg_gemv_w4_kernel(const __grid_constant__ GemvW4Params q) {
    using S = W4Smem<DUAL, MR>;
    constexpr int SIDES = DUAL ? 2 : 1, V = S::V, kWarps = S::kWarps;
    const int plane = q.slots * kW4Cols, slot_mask = q.slots - 1;
    extern __shared__ __align__(16) uint8_t smem[];
    const GemmParams& p = q.g;
    const int K = static_cast<int>(p.K), M = static_cast<int>(p.M);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint8_t* xs = smem;                                            // [V][K]: per 8 columns the even bytes, then the odd ones
    int* sums = reinterpret_cast<int*>(smem + S::x_bytes(K)) + warp * S::warp_ints(q.slots);   // [V][slot][column]
    float* rcp = reinterpret_cast<float*>(sums + V * plane);                // [SIDES][slot][column]
    uint32_t* unit_sg = reinterpret_cast<uint32_t*>(smem + S::x_bytes(K) + kWarps * S::warp_ints(q.slots) * 4ll);   // (segment << 16) | group
    uint16_t* unit_of = reinterpret_cast<uint16_t*>(unit_sg + p.units);                  // unit of each 32 columns; [K / 32] = units

    // weights first: the tables are built while the first step is on its way
    const long long col_groups = (p.N + kW4Cols - 1) / kW4Cols;
    long long cg = static_cast<long long>(warp) * gridDim.x + blockIdx.x;
    const int steps = (K + 1023) >> 10;
    uint4 w[kW4Cols];
    auto load_w = [&](long long group, int step) {
        const int k = step * 1024 + lane * 32;
#pragma unroll
        for (int c = 0; c < kW4Cols; ++c) {
            const long long n = group * kW4Cols + c;              // rows behind the last column are read as the last one's
            w[c] = k < K ? __ldg(reinterpret_cast<const uint4*>(q.wq + (n < p.N ? n : p.N - 1) * q.wq_rs + (k >> 1))) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    if (cg < col_groups) load_w(cg, 0);

    for (int c = threadIdx.x; c < V * (K >> 4); c += blockDim.x) {
        const int v = c / (K >> 4), j = c - v * (K >> 4);
        const int side = v / MR, m = v - side * MR;
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (m < M) x = *reinterpret_cast<const uint4*>((side ? q.xq_neg : q.xq) + m * q.xq_rs + j * 16);
        *reinterpret_cast<uint4*>(xs + static_cast<size_t>(v) * K + j * 16) =
            make_uint4(__byte_perm(x.x, x.y, 0x6420), __byte_perm(x.x, x.y, 0x7531), __byte_perm(x.z, x.w, 0x6420), __byte_perm(x.z, x.w, 0x7531));
    }
    for (int c = threadIdx.x; c <= (K >> 5); c += blockDim.x) {
        const int k = c << 5;
        if (k == K) { unit_of[c] = static_cast<uint16_t>(p.units); break; }
        // units in front of column k: one per segment end and per group end, shared ends counted once
        int s = 0, extra = 0;
        while (k >= p.seg_bounds[s + 1]) {
            ++s;
            if (p.group_size > 0 && p.seg_bounds[s] % p.group_size != 0) ++extra;
        }
        const int g = p.group_size > 0 ? k / p.group_size : 0;
        const int u = p.group_size > 0 ? g + extra : s;
        unit_of[c] = static_cast<uint16_t>(u);
        if (k == p.seg_bounds[s] || (p.group_size > 0 && k == g * p.group_size)) unit_sg[u] = (static_cast<uint32_t>(s) << 16) | static_cast<uint32_t>(g);
    }
    for (int i = lane; i < V * plane; i += 32) sums[i] = 0;
    __syncthreads();

    const bool per_token = p.sx_rs != 0;
    const int oc = lane & (kW4Cols - 1), om = lane >> 2;           // the output that this lane sums up: column and row
    const bool mine = om < M && om < MR;
    for (; cg < col_groups; cg += static_cast<long long>(gridDim.x) * kWarps) {
        const long long n0 = cg * kW4Cols;
        const long long sw_n = (n0 + oc < p.N ? n0 + oc : p.N - 1) * p.sw_cs;
        float y = 0.0f;
        for (int st = 0; st < steps; ++st) {
            const int k = st * 1024 + lane * 32;
            const bool has = k < K;
            const int u_first = unit_of[st * 32], u_end = unit_of[st + 1 < steps ? st * 32 + 32 : K >> 5];
            // scales of the first units that this step completes
            float swv = 1.0f;
            uint32_t sg = 0;
            if (u_first + (lane >> 2) < u_end) {
                sg = unit_sg[u_first + (lane >> 2)];
                swv = w4_load_sw(p, (sg >> 16) * p.sw_ss + (sg & 0xFFFFu) * p.sw_gs + sw_n);
            }
            int acc[V][kW4Cols];
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int c = 0; c < kW4Cols; ++c) acc[v][c] = 0;
            if (has) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {                      // 16 columns of the inner dimension at a time
                    uint32_t lo[kW4Cols][2], hi[kW4Cols][2];
#pragma unroll
                    for (int c = 0; c < kW4Cols; ++c)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t ww = h ? (i ? w[c].w : w[c].z) : (i ? w[c].y : w[c].x);
                            lo[c][i] = (ww << 4) & 0xF0F0F0F0u;
                            hi[c][i] = ww & 0xF0F0F0F0u;
                        }
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const uint4 x = *reinterpret_cast<const uint4*>(xs + static_cast<size_t>(v) * K + k + 16 * h);
#pragma unroll
                        for (int c = 0; c < kW4Cols; ++c) {
                            acc[v][c] = __dp4a(static_cast<int>(lo[c][0]), static_cast<int>(x.x), acc[v][c]);
                            acc[v][c] = __dp4a(static_cast<int>(hi[c][0]), static_cast<int>(x.y), acc[v][c]);
                            acc[v][c] = __dp4a(static_cast<int>(lo[c][1]), static_cast<int>(x.z), acc[v][c]);
                            acc[v][c] = __dp4a(static_cast<int>(hi[c][1]), static_cast<int>(x.w), acc[v][c]);
                        }
                    }
                }
            }
            if (st + 1 < steps) load_w(cg, st + 1);
            else if (cg + static_cast<long long>(gridDim.x) * kWarps < col_groups) load_w(cg + static_cast<long long>(gridDim.x) * kWarps, 0);

            // join the lanes of a unit: two lanes halve the columns between them, four quarter them, further ones add up
            const int u = has ? unit_of[k >> 5] : 0;
            const int slot = (u & slot_mask) * kW4Cols;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                int* dst = sums + v * plane + slot;
                if (q.join == 1) {
#pragma unroll
                    for (int c = 0; c < kW4Cols; ++c)
                        if (has) atomicAdd(dst + c, acc[v][c]);    // integers: any order gives the same sum
                } else {
                    const bool odd = lane & 1;
                    const int r0 = __shfl_xor_sync(0xffffffffu, odd ? acc[v][0] : acc[v][2], 1), r1 = __shfl_xor_sync(0xffffffffu, odd ? acc[v][1] : acc[v][3], 1);
                    const int a0 = (odd ? acc[v][2] : acc[v][0]) + r0, a1 = (odd ? acc[v][3] : acc[v][1]) + r1;      // columns 2 * odd, 2 * odd + 1
                    if (q.join == 2) {
                        if (has) {
                            atomicAdd(dst + 2 * odd, a0);
                            atomicAdd(dst + 2 * odd + 1, a1);
                        }
                    } else {
                        const bool up = lane & 2;
                        int a = (up ? a1 : a0) + __shfl_xor_sync(0xffffffffu, up ? a0 : a1, 2);                      // column 2 * odd + up
                        for (int o = 4; o < q.join; o <<= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
                        if (has && (lane & (q.join - 1)) < 4) atomicAdd(dst + 2 * odd + (up ? 1 : 0), a);
                    }
                }
            }
            __syncwarp();
            // the units that are complete now
            for (int base = u_first; base < u_end; base += 8) {
                const int uu = base + (lane >> 2);
                if (base != u_first && uu < u_end) {
                    sg = unit_sg[uu];
                    swv = w4_load_sw(p, (sg >> 16) * p.sw_ss + (sg & 0xFFFFu) * p.sw_gs + sw_n);
                }
                if (uu < u_end) {
                    const int at = (uu & slot_mask) * kW4Cols + oc;
                    rcp[at] = __frcp_rn((per_token ? 1.0f : p.sx[(sg >> 16) * p.sx_ss]) * swv);
                    if constexpr (DUAL) rcp[plane + at] = __frcp_rn((per_token ? 1.0f : p.sx_neg[(sg >> 16) * p.sx_ss]) * swv);
                }
                __syncwarp();
                if (mine) {
                    const int n = u_end - base < 8 ? u_end - base : 8;
                    for (int i = 0; i < n; ++i) {
                        const int at = ((base + i) & slot_mask) * kW4Cols + oc;
#pragma unroll
                        for (int side = 0; side < SIDES; ++side) {
                            float r = rcp[side * plane + at];
                            if (per_token) r *= __frcp_rn((side ? p.sx_neg : p.sx)[(unit_sg[base + i] >> 16) * p.sx_ss + om * p.sx_rs]);
                            int* a = sums + (side * MR + om) * plane + at;
                            y = fmaf(static_cast<float>(*a >> 4), r, y);                  // weights were read as 16 * q
                            *a = 0;
                        }
                    }
                }
                __syncwarp();
            }
        }
        if (mine && n0 + oc < p.N) {
            const long long n = n0 + oc;
            if (p.bias != nullptr) {
                if (p.bias_dtype == SQ_F32) y += static_cast<const float*>(p.bias)[n];
                else if (p.bias_dtype == SQ_F16) y += __half2float(static_cast<const __half*>(p.bias)[n]);
                else y += __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[n]);
            }
            const long long oi = om * p.y_rs + n;
            if (p.out_dtype == SQ_F32) static_cast<float*>(p.y)[oi] = y;
            else if (p.out_dtype == SQ_F16) static_cast<__half*>(p.y)[oi] = __float2half_rn(y);
            else static_cast<__nv_bfloat16*>(p.y)[oi] = __float2bfloat16_rn(y);
        }
    }
}

static int w4_rows(long long M) { return M <= 1 ? 1 : M <= 2 ? 2 : 4; }

// True when the skinny path serves this problem (the caller has validated the arguments).
bool gemv_w4_applies(const sq_gemm_args* a, bool dual, int units) {
    if (a->kind != SQ_GEMM_W4A8 || a->batch != 1 || a->M > kW4MaxRows || a->acc_dump_dev != nullptr || a->num_peer_outputs != 0 || a->w_seg_as_batch)
        return false;
    if (gemv_disabled()) return false;   // SEGQUANT_B200_NO_GEMV=1 or sq_set_gemm_schedule(): tensor-core path only
    return units <= kW4MaxUnits && a->K <= kW4MaxK && static_cast<long long>(w4_rows(a->M)) * a->K * (dual ? 2 : 1) <= kW4XBytes;
}

template <bool DUAL, int MR>
static int launch_w4(const GemvW4Params& q, cudaStream_t st) {
    using S = W4Smem<DUAL, MR>;
    const long long smem = S::bytes(q.g.K, q.g.units, q.slots);
    constexpr int kMax = 227 * 1024;
    static_assert(S::bytes(0, kW4MaxUnits, 64) + kW4XBytes + kW4MaxK / 16 <= kMax, "shared memory of the skinny int4 kernel");
    static bool attr_set[64] = {};
    int dev = 0;
    SQ_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 64 || !attr_set[dev]) {
        SQ_CUDA_OK(cudaFuncSetAttribute(seg_gemv_w4_kernel<DUAL, MR>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMax));
        if (dev < 64) attr_set[dev] = true;
    }
    const long long col_groups = (q.g.N + kW4Cols - 1) / kW4Cols;
    const long long resident = kNumSMs * (smem <= 112 * 1024 ? 2 : 1);     // two CTAs share an SM where they fit
    const long long ctas = col_groups < resident ? col_groups : resident;
    seg_gemv_w4_kernel<DUAL, MR><<<static_cast<unsigned>(ctas), S::kWarps * 32, static_cast<size_t>(smem), st>>>(q);
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
    q.join = 32;
    for (int s = 1; s <= a->num_segs; ++s)
        while (a->seg_bounds[s] % (32 * q.join)) q.join >>= 1;
    while (a->group_size % (32 * q.join)) q.join >>= 1;
    q.slots = q.join == 1 ? 64 : q.join == 2 ? 32 : 16;
    const int mr = w4_rows(a->M);
    if (dual) return mr == 1 ? launch_w4<true, 1>(q, st) : mr == 2 ? launch_w4<true, 2>(q, st) : launch_w4<true, 4>(q, st);
    return mr == 1 ? launch_w4<false, 1>(q, st) : mr == 2 ? launch_w4<false, 2>(q, st) : launch_w4<false, 4>(q, st);
}

}  // namespace sq
