// Skinny-M form of the segmented GEMM with packed int4 weights (M <= 4 rows; HBM-bound weight streaming, N * K / 2 bytes).
//
// Same arithmetic as the tensor-core path: per accumulation unit (K-segment x weight-scale group) the products are summed
// exactly in int32, converted to fp32, multiplied by 1 / (s_x * s_w[n]) and added to the running fp32 sum in the order of the
// units (the positive side before the negative one); bias and cast at the end.  The results are the same bits.
//
// A warp owns kW4Cols output columns and walks their weight rows in steps of 512 bytes: a lane takes 16 bytes of each row
// (32 values, which lie in one unit: units are multiples of 32).  A nibble pair becomes two bytes 16 * q (even and odd
// columns) with a shift and a mask, so the activations wait in shared memory with the even and the odd bytes of every 8
// columns side by side, and four products are one dp4a.  The sums of the lanes that share a unit are joined with shuffles
// and added, as integers, to the unit's word in shared memory; the running fp32 sum over the units is then one lane's work
// per output, off the weights' path.
#include <cstdlib>

#include "seg_gemm_params.cuh"

namespace sq {

bool gemv_disabled();   // seg_gemm.cu: process-wide schedule overrides

constexpr int kW4Cols = 4;           // columns a warp has in flight
constexpr int kW4Warps = 8;
constexpr int kW4CtaCols = kW4Cols * kW4Warps;
constexpr int kW4MaxRows = 4;
constexpr long long kW4XBytes = 96 * 1024;     // activations staged per CTA
constexpr int kW4SumBytes = 24 * 1024;         // integer sums staged per CTA: as many units at a time as fit

struct GemvW4Params {
    GemmParams g;
    const uint8_t* xq;
    const uint8_t* xq_neg;
    const uint8_t* wq;
    long long xq_rs, wq_rs;
    int join;             // lanes that are sure to share a unit (power of two): every unit is a multiple of 32 * join columns
    int slab_units;       // units whose sums are staged at a time
};

__device__ __forceinline__ float w4_load_sw(const GemmParams& p, long long idx) {
    if (p.sw_is_bf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p.sw)[idx]);
    return static_cast<const float*>(p.sw)[idx];
}

struct W4Unit {           // a walk over the units in order
    int u, s, g, k0, k1;
    __device__ __forceinline__ void end(const GemmParams& p) {
        const int seg_end = p.seg_bounds[s + 1];
        const int grp_end = p.group_size > 0 ? (g + 1) * p.group_size : seg_end;
        k1 = grp_end < seg_end ? grp_end : seg_end;
    }
    __device__ __forceinline__ void first(const GemmParams& p) { u = 0; s = 0; g = 0; k0 = 0; end(p); }
    __device__ __forceinline__ void next(const GemmParams& p) {
        if (p.group_size > 0 && k1 == (g + 1) * p.group_size) ++g;
        if (k1 == p.seg_bounds[s + 1]) ++s;
        k0 = k1;
        ++u;
        if (u < p.units) end(p);
    }
};

template <bool DUAL, int MR>
__global__ void __launch_bounds__(kW4Warps * 32) seg_gemv_w4_kernel(const __grid_constant__ GemvW4Params q) {
    constexpr int SIDES = DUAL ? 2 : 1;
    constexpr int V = SIDES * MR;                       // sums of one column and unit
    extern __shared__ __align__(16) uint8_t smem[];
    const GemmParams& p = q.g;
    const int K = static_cast<int>(p.K), M = static_cast<int>(p.M);
    uint8_t* xs = smem;                                  // [V][K] activation bytes: per 8 columns the even ones, then the odd ones
    int* sums = reinterpret_cast<int*>(smem + static_cast<size_t>(V) * K);   // [slab_units][V][kW4CtaCols]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long n_cta = static_cast<long long>(blockIdx.x) * kW4CtaCols;

    for (int c = threadIdx.x; c < V * (K >> 4); c += blockDim.x) {
        const int v = c / (K >> 4), j = c - v * (K >> 4);
        const int side = v / MR, m = v - side * MR;
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (m < M) x = *reinterpret_cast<const uint4*>((side ? q.xq_neg : q.xq) + m * q.xq_rs + j * 16);
        *reinterpret_cast<uint4*>(xs + static_cast<size_t>(v) * K + j * 16) =
            make_uint4(__byte_perm(x.x, x.y, 0x6420), __byte_perm(x.x, x.y, 0x7531), __byte_perm(x.z, x.w, 0x6420), __byte_perm(x.z, x.w, 0x7531));
    }

    // rows behind the last column are read as the last one's: their sums are not stored
    const uint8_t* wrow[kW4Cols];
    const long long n0 = n_cta + warp * kW4Cols;
#pragma unroll
    for (int c = 0; c < kW4Cols; ++c) wrow[c] = q.wq + (n0 + c < p.N ? n0 + c : p.N - 1) * q.wq_rs;

    // the output that this thread sums up over the units: row `om`, column `on`
    const int om = threadIdx.x / kW4CtaCols, on = threadIdx.x - om * kW4CtaCols;
    const long long out_n = n_cta + on;
    const bool mine = om < M && om < MR && out_n < p.N;
    float y = 0.0f;

    W4Unit su;                                           // first unit of the slab
    su.first(p);
    while (su.u < p.units) {
        W4Unit se = su;                                  // first unit behind it
        const int k_beg = su.k0, u_beg = su.u;
        int k_end = k_beg;
        for (int i = 0; i < q.slab_units && se.u < p.units; ++i) {
            k_end = se.k1;
            se.next(p);
        }
        const int n_units = se.u - u_beg;
        for (int i = threadIdx.x; i < n_units * V * kW4CtaCols; i += blockDim.x) sums[i] = 0;
        __syncthreads();

        W4Unit lu = su;                                  // the unit of this lane's chunk
        for (int kb = k_beg; kb < k_end; kb += 1024) {
            const int k = kb + lane * 32;
            const bool has = k < k_end;
            uint4 w[kW4Cols];
#pragma unroll
            for (int c = 0; c < kW4Cols; ++c) w[c] = has ? __ldg(reinterpret_cast<const uint4*>(wrow[c] + (k >> 1))) : make_uint4(0u, 0u, 0u, 0u);
            if (has)
                while (k >= lu.k1) lu.next(p);
            int acc[V][kW4Cols];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
                if (has) {
                    a = *reinterpret_cast<const uint4*>(xs + static_cast<size_t>(v) * K + k);
                    b = *reinterpret_cast<const uint4*>(xs + static_cast<size_t>(v) * K + k + 16);
                }
                const uint32_t xw[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int c = 0; c < kW4Cols; ++c) {
                    const uint32_t ww[4] = {w[c].x, w[c].y, w[c].z, w[c].w};
                    int s = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s = __dp4a(static_cast<int>((ww[i] << 4) & 0xF0F0F0F0u), static_cast<int>(xw[2 * i]), s);
                        s = __dp4a(static_cast<int>(ww[i] & 0xF0F0F0F0u), static_cast<int>(xw[2 * i + 1]), s);
                    }
                    acc[v][c] = s;
                }
            }
            for (int o = 1; o < q.join; o <<= 1) {
#pragma unroll
                for (int v = 0; v < V; ++v)
#pragma unroll
                    for (int c = 0; c < kW4Cols; ++c) acc[v][c] += __shfl_xor_sync(0xffffffffu, acc[v][c], o);
            }
            if (has && (lane & (q.join - 1)) == 0) {
                int* dst = sums + (lu.u - u_beg) * (V * kW4CtaCols) + warp * kW4Cols;
#pragma unroll
                for (int v = 0; v < V; ++v)
#pragma unroll
                    for (int c = 0; c < kW4Cols; ++c) atomicAdd(dst + v * kW4CtaCols + c, acc[v][c]);     // integers: any order
            }
        }
        __syncthreads();
        if (mine) {
            W4Unit ou = su;
            const bool per_token = p.sx_rs != 0;
            for (int i = 0; i < n_units; ++i) {
                const float swv = w4_load_sw(p, ou.s * p.sw_ss + ou.g * p.sw_gs + out_n * p.sw_cs);
#pragma unroll
                for (int side = 0; side < SIDES; ++side) {
                    const float* sxp = side ? p.sx_neg : p.sx;
                    float r = __frcp_rn((per_token ? 1.0f : sxp[ou.s * p.sx_ss]) * swv);
                    if (per_token) r *= __frcp_rn(sxp[ou.s * p.sx_ss + om * p.sx_rs]);
                    const int a = sums[(i * V + side * MR + om) * kW4CtaCols + on] >> 4;      // weights were read as 16 * q
                    y = fmaf(static_cast<float>(a), r, y);
                }
                ou.next(p);
            }
        }
        __syncthreads();
        su = se;
    }
    if (mine) {
        if (p.bias != nullptr) {
            if (p.bias_dtype == SQ_F32) y += static_cast<const float*>(p.bias)[out_n];
            else if (p.bias_dtype == SQ_F16) y += __half2float(static_cast<const __half*>(p.bias)[out_n]);
            else y += __bfloat162float(static_cast<const __nv_bfloat16*>(p.bias)[out_n]);
        }
        const long long oi = om * p.y_rs + out_n;
        if (p.out_dtype == SQ_F32) static_cast<float*>(p.y)[oi] = y;
        else if (p.out_dtype == SQ_F16) static_cast<__half*>(p.y)[oi] = __float2half_rn(y);
        else static_cast<__nv_bfloat16*>(p.y)[oi] = __float2bfloat16_rn(y);
    }
}

static int w4_rows(long long M) { return M <= 1 ? 1 : M <= 2 ? 2 : 4; }

// True when the skinny path serves this problem (the caller has validated the arguments).
bool gemv_w4_applies(const sq_gemm_args* a, bool dual) {
    if (a->kind != SQ_GEMM_W4A8 || a->batch != 1 || a->M > kW4MaxRows || a->acc_dump_dev != nullptr || a->num_peer_outputs != 0 || a->w_seg_as_batch)
        return false;
    if (gemv_disabled()) return false;   // SEGQUANT_B200_NO_GEMV=1 or sq_set_gemm_schedule(): tensor-core path only
    return static_cast<long long>(w4_rows(a->M)) * a->K * (dual ? 2 : 1) <= kW4XBytes;
}

template <bool DUAL, int MR>
static int launch_w4(const GemvW4Params& q, size_t smem, long long ctas, cudaStream_t st) {
    static bool attr_set[64] = {};
    int dev = 0;
    SQ_CUDA_OK(cudaGetDevice(&dev));
    if (smem > 48 * 1024 && (dev >= 64 || !attr_set[dev])) {
        SQ_CUDA_OK(cudaFuncSetAttribute(seg_gemv_w4_kernel<DUAL, MR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        static_cast<int>(kW4XBytes + kW4SumBytes)));
        if (dev < 64) attr_set[dev] = true;
    }
    seg_gemv_w4_kernel<DUAL, MR><<<static_cast<unsigned>(ctas), kW4Warps * 32, smem, st>>>(q);
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
    const int mr = w4_rows(a->M), V = mr * (dual ? 2 : 1);
    q.slab_units = kW4SumBytes / (V * kW4CtaCols * 4);
    if (q.slab_units > p.units) q.slab_units = p.units;
    const size_t smem = static_cast<size_t>(V) * a->K + static_cast<size_t>(q.slab_units) * V * kW4CtaCols * 4;
    const long long ctas = (a->N + kW4CtaCols - 1) / kW4CtaCols;
    if (dual) return mr == 1 ? launch_w4<true, 1>(q, smem, ctas, st) : mr == 2 ? launch_w4<true, 2>(q, smem, ctas, st) : launch_w4<true, 4>(q, smem, ctas, st);
    return mr == 1 ? launch_w4<false, 1>(q, smem, ctas, st) : mr == 2 ? launch_w4<false, 2>(q, smem, ctas, st) : launch_w4<false, 4>(q, smem, ctas, st);
}

}  // namespace sq
