// Attention of whole and packed sequences: softmax(scale * q k^T) v, heads in groups that share keys and values, on the
// fifth-generation tensor cores.
//
// One CTA takes two sub-tiles of 128 rows of one key head (a row is a (query token, query head) pair, so the query heads
// that share a key head share its tiles) and walks the keys in tiles of 128:
//
//   warps 0-3, 4-7 : softmax of sub-tile 0 / 1, one row per thread
//   warp 8         : TMA loads (q once, k and v through a ring of stages)
//   warp 9 (, 10)  : issue tcgen05.mma: S = q k^T (both operands in shared memory), O += P v (P in tensor memory); heads up to
//                    64 wide have a warp for each sub-tile
//   warp 11        : clears the rows behind the last key in the last v tile (what lies there may be NaN, and 0 * NaN is NaN)
//
// What bounds it.  A pair of 128 x 128 tiles takes 1100 (heads of 64) or 2048 (128) cycles of products and 2048 of
// exponentials, less what the FMA pipe takes over; the loop needs 2700 and 3400.  Heads of 64: softmax and products run side by
// side, 332 us = 726 TFLOP/s for two samples of 4429 tokens, 24 heads (the exponentials alone would take 202 us, the products 144).  Heads of 128: tensor
// memory holds one S a sub-tile, so softmax, O and the next S follow one another within a sub-tile and only the two
// sub-tiles overlap, 494 to 504 us = 1227 to 1250 TFLOP/s at 12288 causal tokens, 16 query heads on 2 (products 368 us).  A cluster of
// CTAs that shared k and v would save L2 traffic that bounds nothing (85 to 92 % hits, DRAM 2 to 3 %).
//
// One pass over the keys with a running maximum m and sum l per row: p = 2^(c (s - m)), O and l are scaled by
// 2^(c (m_old - m_new)) when the maximum grows.  O lives in tensor memory and is only rescaled when a row's maximum has
// grown by more than 2^8 since the last time (every p then stays below 2^8, well inside fp32 sums and fp16 p); the result
// does not depend on it, the same m is used for p, l and O.  p is rounded once to the 16-bit input type for the second
// product (half a step, 2^-8 for bf16 and 2^-11 for fp16, of each term); S, l, O and the statistics stay fp32.  fp16 has no more
// than steps of 2^-24 below 2^-14, where many keys of small weight beside a strong one would lose theirs, so p, l and O of fp16
// calls are carried 2^7 times as large (p stays below 2^15): half a step is then at most 2^-32 of the row's largest p.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <type_traits>

#include "attention.cuh"
#include "attention_turns.cuh"
#include "ptx.cuh"

namespace sq {

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();   // seg_gemm.cu
long long wait_limit_cycles();                            // seg_gemm.cu
// few rows against many keys (attention_rows.cu)
int attention_rows(int dtype, const CUtensorMap& mk, const CUtensorMap& mv, const AttnParams& p, long long grid, cudaStream_t st);

enum AttnWait : int { kAttnMma = 20, kAttnKvEmpty = 22, kAttnS = 23, kAttnPv = 26, kAttnTail = 27 };

constexpr int kAttnThreads = 384;
// Of kPolyOf pairs of exponentials, kPoly go to the FMA pipe (ex2_poly).  The special-function pipe does 4 lanes a cycle: two
// warps' 128 exponentials a row take 2048 cycles there while everything else that a tile needs takes about 1000.  4429 tokens,
// 24 heads of 64, two samples: none 361 us, one of eight 335, one of six 332, one of four 347 (the other pipes and the issue
// slots fill up); 128 wide heads do not care (507, 505, 504, 507 us at 12288 causal tokens).
constexpr int kPoly = 1, kPolyOf = 6;
// Power of two that p, l and O are carried up by (see above; what is left of fp16's 2^16 above the 2^8 that a maximum may have grown).
template <typename T>
constexpr float kUp = std::is_same<T, __half>::value ? 7.0f : 0.0f;
constexpr int kWarpMma = 9;         // and the next one with heads up to 64 wide
constexpr int kAttnRows = 128;       // rows of a sub-tile = tensor-memory lanes
constexpr int kAttnKeys = 128;       // keys of a tile

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, int c4, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(bar)
        : "memory");
}

// 32 lanes x 16 or 32 consecutive 32-bit columns: thread t of the warp has lane (base lane + t).  The wait takes the loaded
// registers as operands, so that nothing that uses them can be moved in front of it.
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        :
        "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait_x16(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
        :
        "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
        "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]));
}
__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        :
        "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait_x32(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
        :
        "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
        "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]),
        "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
        "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]));
}

// D (tensor memory, fp32) (+)= A (shared memory) B (shared memory), 16-bit operands of one type.  Descriptors come as their
// low words: the high word (layout, strides) is a constant.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kSmemDescHi)
        : "memory");
}
// the same with A in tensor memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kSmemDescHi)
        : "memory");
}
// barriers of AttnTurns: named barriers of two warps
struct TurnBarrier {
    int mine, other;
    __device__ __forceinline__ void sync() { asm volatile("bar.sync %0, 64;" ::"r"(mine) : "memory"); }
    __device__ __forceinline__ void arrive() { asm volatile("bar.arrive %0, 64;" ::"r"(other) : "memory"); }
};
__device__ __forceinline__ void tmem_st_wait_all() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Head widths up to DP (64 or 128): narrower heads are filled up with zeros by the TMA loads.
//
// Tensor memory (512 columns).  DP = 64: S, P and O of each sub-tile have columns of their own, so the next S is computed
// while the softmax works on this one.  DP = 128: S 128 + O 128 columns per sub-tile fill it; P takes the first 64 columns
// of the S it was made from, and the next S waits for the product with P.
template <int DP>
struct AttnCfg {
    static constexpr bool kOwnP = DP == 64;
    static constexpr uint32_t kHalf = kAttnRows * 128;                 // 128 rows of 64 16-bit columns, 128-byte swizzled
    static constexpr uint32_t kTile = kHalf * (DP / 64);               // a q, k or v tile
    static constexpr int kStages = DP == 64 ? 10 : 5;
    static constexpr uint32_t kSmem = 1024 + 2 * kTile + kStages * kTile;
    __host__ __device__ static constexpr uint32_t col_s(int t) { return t * 128; }
    __host__ __device__ static constexpr uint32_t col_p(int t) { return kOwnP ? 256 + t * 64 : t * 128; }
    __host__ __device__ static constexpr uint32_t col_o(int t) { return kOwnP ? 384 + t * 64 : 256 + t * 128; }
};

// Instruction descriptor of kind::f16: D fp32, A and B of type T, M = 128; the second operand of O += P v is read along
// its rows (bit 16: keys are the rows of the v tile and the inner dimension of the product).
template <typename T>
__device__ __forceinline__ uint32_t attn_idesc(int n, bool b_by_rows);
template <>
__device__ __forceinline__ uint32_t attn_idesc<__half>(int n, bool b_by_rows) {
    return (1u << 4) | (b_by_rows ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kAttnRows >> 4) << 24);
}
template <>
__device__ __forceinline__ uint32_t attn_idesc<__nv_bfloat16>(int n, bool b_by_rows) {
    return attn_idesc<__half>(n, b_by_rows) | (1u << 7) | (1u << 10);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kAttnThreads, 1)
attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnParams p) {
    using C = AttnCfg<DP>;
    constexpr int ST = C::kStages;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_q[2], bar_full[ST], bar_empty[ST], bar_s[2], bar_sfree[2], bar_p[2], bar_pv[2], bar_tail;
    __shared__ AttnTile tile_s;
    __shared__ uint32_t tmem_s;
    __shared__ int abort_s;
    volatile int* abort_flag = &abort_s;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const uint32_t sbase = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // ---- which part of the work: tiles of a causal sequence from the longest to the shortest
    const int chunk = blockIdx.x % p.chunks;
    const int rest = blockIdx.x / p.chunks;
    const int split = rest % p.splits;
    const int index = p.tiles - 1 - rest / p.splits;
    if (warp == 0) {
        const AttnTile t = attn_find_tile(p, index, lane);
        if (lane == 0) { tile_s = t; abort_s = 0; }
    } else if (warp == 8) {
        if (lane == 0) {
            for (int t = 0; t < 2; ++t) {
                mbar_init(smem_u32(&bar_q[t]), 1);
                mbar_init(smem_u32(&bar_s[t]), 1);
                mbar_init(smem_u32(&bar_sfree[t]), 4);
                mbar_init(smem_u32(&bar_p[t]), 4);
                mbar_init(smem_u32(&bar_pv[t]), 1);
            }
            for (int s = 0; s < ST; ++s) {
                mbar_init(smem_u32(&bar_full[s]), 1);
                mbar_init(smem_u32(&bar_empty[s]), C::kOwnP ? 2 : 1);      // arrivals of the warps that issue products
            }
            mbar_init(smem_u32(&bar_tail), 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            prefetch_tmap(&map_q);
            prefetch_tmap(&map_k);
            prefetch_tmap(&map_v);
        }
    } else if (warp == kWarpMma) {
        __syncwarp();
        tmem_alloc(smem_u32(&tmem_s), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const AttnTile T0 = tile_s;
    const uint32_t tmem = tmem_s;
    const int tps = p.tile_tokens >> 1;                       // query tokens of a sub-tile

    // key tiles [lo, hi) of this part, and the end of each sub-tile's own share
    int n_sub[2];
    bool live[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int first = T0.tok0 + t * tps;
        const int last = min(first + tps, T0.rows_end) - 1;
        live[t] = T0.ok && first <= last;
        const int see = live[t] ? attn_limit(T0, min(last, max(T0.q_len - 1, 0)), p.causal) : 0;   // the rows' largest limit
        n_sub[t] = (see + kAttnKeys - 1) / kAttnKeys;
        if (first >= T0.q_len) n_sub[t] = 0;
    }
    int n_all = max(n_sub[0], n_sub[1]);
    int lo = 0;
    if (p.splits > 1) {
        const int per = (n_all + p.splits - 1) / p.splits;
        lo = min(split * per, n_all);
        n_all = min(lo + per, n_all);
    }
    n_sub[0] = max(min(n_sub[0], n_all) - lo, 0);
    n_sub[1] = max(min(n_sub[1], n_all) - lo, 0);
    const int n = max(n_sub[0], n_sub[1]);                    // tiles that are loaded
    const bool tail = n > 0 && (lo + n) * kAttnKeys > T0.kv_len;   // the last of them holds rows that are not keys

    auto q_smem = [&](int t) { return sbase + t * C::kTile; };
    auto stage = [&](int s) { return sbase + (2 + s) * C::kTile; };

    if (warp >= 8) {
        reg_dec<56>();
        if (warp == 8) {
            // ------------------------------------------------------------------ loads
            if (lane == 0 && n > 0) {
                const int kvh = chunk / (p.G / p.P);
                bool ok = true;
                for (int t = 0; t < 2; ++t) {
                    if (n_sub[t] == 0) continue;
                    const uint32_t bar = smem_u32(&bar_q[t]);
                    mbar_arrive_expect_tx(bar, static_cast<uint32_t>(tps * p.P) * 128u * (DP / 64));
                    for (int h = 0; h < DP / 64; ++h)
                        tma_load_5d(q_smem(t) + h * C::kHalf, &map_q, h * 64, 0, chunk, T0.q_base + T0.tok0 + t * tps, T0.b, bar);
                }
                for (int i = 0; ok && i < 2 * n; ++i) {       // k and v tiles in turn
                    const int s = i % ST, j = i >> 1;
                    if (i >= ST && !mbar_wait(smem_u32(&bar_empty[s]), (i / ST + 1) & 1u, abort_flag, kAttnKvEmpty, p.wait_cycles)) { ok = false; break; }
                    const bool is_v = i & 1;
                    const uint32_t bar = smem_u32(is_v && tail && j == n - 1 ? &bar_tail : &bar_full[s]);
                    mbar_arrive_expect_tx(bar, C::kTile);
                    for (int h = 0; h < DP / 64; ++h)
                        tma_load_4d(stage(s) + h * C::kHalf, is_v ? &map_v : &map_k, h * 64, kvh, T0.kv_base + (lo + j) * kAttnKeys, T0.b, bar);
                }
            }
        } else if (warp == kWarpMma || warp == kWarpMma + 1) {
            // ------------------------------------------------------------------ products
            // A warp alone takes 5 cycles an instruction, 80 to get past a barrier that is complete and 40 to issue a product (that
            // runs for 32 to 64).  The whole warp walks in step (votes and shuffles keep branches and addresses uniform, so that the
            // operands are in uniform registers) and one lane issues: with a lane walking alone an S took 460 cycles to issue and an O
            // 590.  DP = 64 has a warp for each sub-tile: one for both needed 2100 cycles a pair of tiles, which bounded the kernel,
            // for products that take 1100.  DP = 128, where the products take 2048 and S waits for O, has one warp for both: two were
            // measured 10 % slower (12288 tokens, causal: 552 against 499 us), their products of one sub-tile wait behind the other's.
            uint32_t leader;
            asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(leader));
            const int n0 = __shfl_sync(0xffffffffu, n_sub[0], 0), n1 = __shfl_sync(0xffffffffu, n_sub[1], 0);
            const int nn = n0 > n1 ? n0 : n1;
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), sb = __shfl_sync(0xffffffffu, sbase, 0);
            const int dk = (p.D + 15) & ~15;
            const uint32_t idesc_s = attn_idesc<T>(kAttnKeys, false), idesc_o = attn_idesc<T>(dk, true);
            const uint32_t b_full = smem_u32(&bar_full[0]), b_empty = smem_u32(&bar_empty[0]), b_q = smem_u32(&bar_q[0]), b_s = smem_u32(&bar_s[0]),
                           b_sfree = smem_u32(&bar_sfree[0]), b_p = smem_u32(&bar_p[0]), b_pv = smem_u32(&bar_pv[0]);
            bool ok = true;
            // several barriers at once: one round trip, which takes 250 to 350 cycles next to the softmax warps
            auto wait3 = [&](uint32_t bar_a, uint32_t par_a, uint32_t bar_b, uint32_t par_b, uint32_t bar_c, uint32_t par_c) {
                if (!ok) return;
                uint32_t it = 0;
                long long t0 = 0;
                for (;;) {
                    const uint32_t ra = mbar_try_wait(bar_a, par_a), rb = mbar_try_wait(bar_b, par_b), rc = mbar_try_wait(bar_c, par_c);
                    if (__all_sync(0xffffffffu, ra & rb & rc)) break;
                    if ((it++ & 1023u) == 0u) {
                        if (it == 1u) t0 = clock64();
                        if (__any_sync(0xffffffffu, *abort_flag || clock64() - t0 > p.wait_cycles)) {
                            if (leader) {
                                if (!*abort_flag) wait_gave_up(kAttnMma);
                                *abort_flag = 1;
                            }
                            ok = false;
                            return;
                        }
                    }
                }
                tc_fence_after();
            };
            auto wait2 = [&](uint32_t bar_a, uint32_t par_a, uint32_t bar_b, uint32_t par_b) { wait3(bar_a, par_a, bar_b, par_b, bar_b, par_b); };
            auto wait1 = [&](uint32_t bar, uint32_t par) { wait2(bar, par, bar, par); };
            // ring slot and lap of the next K and the next V tile (K and V lie in it in turn)
            int ks = 0, kl = 0, vs = 1, vl = 0;
            auto next_k = [&]() {
                ks += 2;
                if (ks >= ST) { ks -= ST; kl ^= 1; }
            };
            auto next_v = [&]() {
                vs += 2;
                if (vs >= ST) { vs -= ST; vl ^= 1; }
            };
            auto product_s = [&](int t, bool release) {
                const uint32_t a = smem_desc_lo(sb + t * C::kTile), b = smem_desc_lo(sb + (2 + ks) * C::kTile), d = tm + C::col_s(0) + t * (C::col_s(1) - C::col_s(0));
                if (leader) {
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k) {            // 16 columns = 32 bytes each
                        const uint32_t off = static_cast<uint32_t>(k >> 2) * (C::kHalf >> 4) + (k & 3) * 2u;
                        if (16 * k < dk) mma_ss(d, a + off, b + off, idesc_s, k > 0);
                    }
                    umma_commit(b_s + t * 8);
                    if (release) umma_commit(b_empty + ks * 8);
                }
            };
            auto product_o = [&](int t, uint32_t acc, bool release) {
                // rows of 64 columns: 8 keys are 1024 bytes (SBO), the next 64 columns kHalf bytes on (LBO)
                const uint32_t b = (((sb + (2 + vs) * C::kTile) >> 4) & 0x3FFFu) | ((C::kHalf >> 4) << 16), a = tm + C::col_p(0) + t * (C::col_p(1) - C::col_p(0)),
                               d = tm + C::col_o(0) + t * (C::col_o(1) - C::col_o(0));
                if (leader) {
#pragma unroll
                    for (int k = 0; k < kAttnKeys / 16; ++k) mma_ts(d, a + k * 8, b + k * 128u, idesc_o, k > 0 ? 1u : acc);
                    umma_commit(b_pv + t * 8);
                    if (release) umma_commit(b_empty + vs * 8);
                }
            };
            if constexpr (C::kOwnP) {
                const int t = warp - kWarpMma, nt = t ? n1 : n0;
                if (nt > 0) {
                    wait2(b_full, 0u, b_q + t * 8, 0u);
                    if (ok) product_s(t, true);
                    next_k();
                }
                for (int j = 0; ok && j < nt; ++j) {
                    if (j + 1 < nt) {
                        wait2(b_full + ks * 8, kl, b_sfree + t * 8, j & 1u);
                        if (ok) product_s(t, true);
                        next_k();
                    }
                    wait2(b_full + vs * 8, vl, b_p + t * 8, j & 1u);
                    if (ok) product_o(t, j > 0, true);
                    next_v();
                }
                // tiles that only the other sub-tile needs: released as they come
                for (int i = 2 * nt; ok && i < 2 * nn; ++i) {
                    const int lap = i / ST, s = i - lap * ST;
                    wait1(b_full + s * 8, lap & 1u);
                    if (ok && leader) mbar_arrive(b_empty + s * 8);
                }
            } else if (warp == kWarpMma) {
                // O of tile j and S of tile j + 1 of sub-tile 0, then of sub-tile 1; whichever comes last gives the slots back
                if (nn > 0) {
                    wait1(b_full, 0u);
                    for (int t = 0; t < 2; ++t)
                        if ((t ? n1 : n0) > 0) {
                            wait1(b_q + t * 8, 0u);
                            if (ok) product_s(t, t == 1 || n1 == 0);
                        }
                    next_k();
                }
                for (int j = 0; ok && j < nn; ++j) {
                    const bool more = j + 1 < nn;
                    const int kb = more ? ks : vs, kp = more ? kl : vl;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const int nt = t ? n1 : n0;
                        if (ok && j < nt) {
                            wait3(b_p + t * 8, j & 1u, b_full + vs * 8, vl, b_full + kb * 8, kp);
                            if (ok) product_o(t, j > 0, t == 1 || j >= n1);
                            if (ok && j + 1 < nt) product_s(t, t == 1 || j + 1 >= n1);
                        }
                    }
                    if (more) next_k();
                    next_v();
                }
            }
            __syncwarp();
        } else if (warp == kWarpMma + 2 && tail) {
            // ------------------------------------------------------------------ rows behind the last key
            const int s = (2 * n - 1) % ST;
            if (mbar_wait_warp(smem_u32(&bar_tail), 0, abort_flag, kAttnTail, p.wait_cycles)) {
                const int valid = T0.kv_len - (lo + n - 1) * kAttnKeys;
                uint8_t* v = smem + (2 + s) * C::kTile;
                for (int h = 0; h < DP / 64; ++h)
                    for (int i = valid * 8 + lane; i < kAttnRows * 8; i += 32)
                        *reinterpret_cast<uint4*>(v + h * C::kHalf + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bar_full[s]));
            }
        }
    } else {
        // ---------------------------------------------------------------------- softmax
        reg_inc<216>();
        const int t = warp >> 2;
        const int row = threadIdx.x & 127;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const uint32_t ts = lane_base + (t ? C::col_s(1) : C::col_s(0)), tp = lane_base + (t ? C::col_p(1) : C::col_p(0)),
                       to = lane_base + (t ? C::col_o(1) : C::col_o(0));
        const int tok = T0.tok0 + t * tps + row / p.P;
        const int head = chunk * p.P + row % p.P;
        const bool mine = live[t] && row < tps * p.P && tok < T0.rows_end;
        const int limit = mine ? attn_limit(T0, tok, p.causal) : 0;
        // keys that every row of this warp sees (rows that are not stored do not count): no comparison needed below it
        const int seen_by_all = __reduce_min_sync(0xffffffffu, mine ? limit : 0x7fffffff);
        const int nt = t ? n_sub[1] : n_sub[0];
        const uint32_t bs = smem_u32(&bar_s[t]), bsf = smem_u32(&bar_sfree[t]), bp = smem_u32(&bar_p[t]), bpv = smem_u32(&bar_pv[t]);
        const float c = p.scale_log2;
        const int cols = (p.D + 15) & ~15;
        float m_ref = -INFINITY, l = 0.0f;
        bool ok = true;
        // The two warps of an SM quarter (one of each sub-tile) take turns with their exponentials: while one fills the
        // special-function pipe the other loads, compares and stores.
        AttnTurns<TurnBarrier> turn = {{1 + t * 4 + (warp & 3), 1 + (t ^ 1) * 4 + (warp & 3)}, min(n_sub[0], n_sub[1]), t};
        auto wait = [&](uint32_t bar, uint32_t parity, int code) { return mbar_wait_warp(bar, parity, abort_flag, code, p.wait_cycles); };
        turn.open();
        int j = 0;
        for (; j < nt; ++j) {
            if (!wait(bs, j & 1u, kAttnS)) { ok = false; break; }
            tc_fence_after();
            uint32_t s[128];
            const int key0 = (lo + j) * kAttnKeys;
            const bool edge = key0 + kAttnKeys > seen_by_all;
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            tmem_ld_x32(ts, s);
            tmem_ld_x32(ts + 32, s + 32);
            tmem_ld_wait_x32(s);
            tmem_ld_wait_x32(s + 32);
            tmem_ld_x32(ts + 64, s + 64);
            tmem_ld_x32(ts + 96, s + 96);
            if (edge) {
#pragma unroll
                for (int i = 0; i < 64; ++i) s[i] = key0 + i < limit ? s[i] : 0xFF800000u;
            }
#pragma unroll
            for (int i = 0; i < 64; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
            tmem_ld_wait_x32(s + 64);
            tmem_ld_wait_x32(s + 96);
            if constexpr (C::kOwnP) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bsf);
            }
            if (edge) {
#pragma unroll
                for (int i = 64; i < 128; ++i) s[i] = key0 + i < limit ? s[i] : 0xFF800000u;
            }
#pragma unroll
            for (int i = 64; i < 128; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
            const float m_new = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            // DP = 64: the product with the previous P has to be done before P (and, for a rescale, O) is touched
            bool pv_done = !C::kOwnP || j == 0;
            auto wait_pv = [&]() {
                if (!pv_done) {
                    pv_done = true;
                    if (!wait(bpv, (j - 1) & 1u, kAttnPv)) ok = false;
                    tc_fence_after();
                }
            };
            const bool grow = (m_new - m_ref) * c > 8.0f;
            if (__any_sync(0xffffffffu, grow)) {
                const float f = grow ? ex2((m_ref - m_new) * c) : 1.0f;
                if (grow) m_ref = m_new;
                l *= f;
                if (j > 0) {
                    wait_pv();
                    for (int i = 0; i < cols; i += 16) {
                        uint32_t o[16];
                        tmem_ld_x16(to + i, o);
                        tmem_ld_wait_x16(o);
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st_x16(to + i, o);
                    }
                }
            }
            turn.take(j);
            const float mc = m_ref == -INFINITY ? 0.0f : m_ref * c;
            const float off = kUp<T> != 0.0f ? kUp<T> - mc : -mc;
            const float2 c2 = make_float2(c, c), mc2 = make_float2(off, off);
            float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
            uint32_t pk[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) {
                float2 e = __ffma2_rn(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), c2, mc2);
                if (i % kPolyOf < kPoly) {
                    e = ex2_poly(e);
                } else {
                    e.x = ex2(e.x);
                    e.y = ex2(e.y);
                }
                sum[i & 1] = __fadd2_rn(sum[i & 1], e);
                pk[i] = pack2<T>(e.x, e.y);
                if (i == 31) {
                    wait_pv();
                    tmem_st_x32(tp, pk);
                }
            }
            turn.pass(j);
            tmem_st_x32(tp + 32, pk + 32);
            tmem_st_wait_all();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bp);
            if (!ok) { ++j; break; }                               // this tile's turn has been taken and passed on
            l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        }
        if (!ok) turn.leave(j);
        // ---- result
        if (ok && nt > 0) {
            ok = wait(bpv, (nt - 1) & 1u, kAttnPv);
            tc_fence_after();
        }
        if (ok && live[t]) {
            const bool empty = m_ref == -INFINITY && l == l;     // no key seen
            const float inv = empty ? 0.0f : 1.0f / l;
            const float lse2 = empty ? -INFINITY : m_ref * c + (log2f(l) - kUp<T>);
            const long long token = static_cast<long long>(T0.b) * (p.q_off ? 0 : p.Tq) + T0.q_base + tok;
            const long long r = token * p.Hq + head;
            if (p.splits > 1) {
                if (mine) p.part_lse[split * p.rows + r] = lse2;
            } else if (mine && p.lse) {
                p.lse[r] = lse2 * kLn2;
            }
            T* out = static_cast<T*>(p.out) + static_cast<long long>(T0.b) * p.o_bs + static_cast<long long>(T0.q_base + tok) * p.o_ts +
                     static_cast<long long>(head) * p.o_hs;
            float* part = p.part_o + (split * p.rows + r) * p.D;
#pragma unroll
            for (int i0 = 0; i0 < DP; i0 += 64) {             // whole warps: tcgen05.ld; 64 columns a round trip
                uint32_t o[64];
                if (nt > 0) {
                    tmem_ld_x32(to + i0, o);
                    tmem_ld_x32(to + i0 + 32, o + 32);
                    tmem_ld_wait_x32(o);
                    tmem_ld_wait_x32(o + 32);
                }
                if (!mine) continue;
#pragma unroll
                for (int i = 0; i < 64; ++i) o[i] = empty ? 0u : __float_as_uint(__uint_as_float(o[i]) * inv);
                if (p.splits > 1) {
#pragma unroll
                    for (int i = 0; i < 64; i += 4)
                        if (i0 + i < p.D && !empty) *reinterpret_cast<uint4*>(part + i0 + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 64; i += 8) {
                        if (i0 + i < p.D) {
                            uint32_t w[4];
#pragma unroll
                            for (int x = 0; x < 4; ++x) w[x] = pack2<T>(__uint_as_float(o[i + 2 * x]), __uint_as_float(o[i + 2 * x + 1]));
                            *reinterpret_cast<uint4*>(out + i0 + i) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                }
            }
        }
    }

    // ---------------------------------------------------------------------- teardown
    if (*abort_flag) {
        // give copies that may still be in flight time to land before shared memory is released
        const unsigned long long t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kWarpMma) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the parts of a row: weights 2^(lse_s - max), one warp per row, four columns a lane.
template <typename T>
__global__ void __launch_bounds__(256) attention_join_kernel(const __grid_constant__ AttnParams p) {
    const int lane = threadIdx.x & 31;
    const long long r = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (r >= p.rows) return;
    cudaGridDependencySynchronize();
    const long long token = r / p.Hq;
    const int head = static_cast<int>(r - token * p.Hq);
    const int b = p.q_off ? 0 : static_cast<int>(token / p.Tq);
    const long long tok = p.q_off ? token : token - static_cast<long long>(b) * p.Tq;
    if (!p.fill_rest) {                                  // rows of no sequence have no parts and are left alone
        if (p.q_off) {
            if (tok < p.q_off[0] || tok >= p.q_off[p.batch]) return;
        } else if (p.q_lens && tok >= p.q_lens[b]) {
            return;
        }
    }
    const float mine = lane < p.splits ? p.part_lse[lane * p.rows + r] : -INFINITY;
    float top = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float w = mine == -INFINITY ? 0.0f : ex2(mine - top);
    float sum = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (p.lse && lane == 0) p.lse[r] = top == -INFINITY ? -INFINITY : (top + log2f(sum)) * kLn2;
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const bool has = lane * 4 < p.D;
    for (int s = 0; s < p.splits; ++s) {
        const float ws = __shfl_sync(0xffffffffu, w, s) * inv;
        if (ws == 0.0f || !has) continue;
        const float4 v = *reinterpret_cast<const float4*>(p.part_o + (s * p.rows + r) * p.D + lane * 4);
        acc.x = fmaf(ws, v.x, acc.x); acc.y = fmaf(ws, v.y, acc.y); acc.z = fmaf(ws, v.z, acc.z); acc.w = fmaf(ws, v.w, acc.w);
    }
    if (has)
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + b * p.o_bs + tok * p.o_ts + head * p.o_hs + lane * 4) =
            make_uint2(pack2<T>(acc.x, acc.y), pack2<T>(acc.z, acc.w));
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
struct AttnPlan {
    bool rows;                       // few rows against many keys: attention_rows.cu
    int P, tile_tokens, splits, part_keys;
    long long tiles;                 // per chunk of heads
};

// The choice of kernel and of the parts goes by what the host knows: extents and heads, not the lengths on the device.  Packed
// sequences are judged by their average and their parts cut from the keys of all of them together, so lengths far from the average
// cost time (32 packed single tokens on 4000 to 16000 keys, 32 heads on 8 of 128: 271 us, as a batch of caches 207; a prompt of 4096
// tokens packed with 300 single tokens on 500 keys: 352, in two calls 136 + 118).
static AttnPlan attention_plan(const sq_attention_args* a) {
    AttnPlan pl;
    const int G = a->Hq / a->Hkv;
    const bool packed = a->q_offsets_dev != nullptr;
    const long long avg = packed ? (a->Tq + a->batch - 1) / a->batch : a->Tq;      // query tokens of a sequence
    pl.rows = avg * G <= 16;
    const int most = pl.rows ? 16 : 32;
    pl.P = 1;
    for (int d = 2; d <= G && d <= most; ++d)
        if (G % d == 0) pl.P = d;
    pl.tile_tokens = pl.rows ? 16 / pl.P : 2 * (kAttnRows / pl.P);
    pl.tiles = packed ? (a->Tq + a->batch * (pl.tile_tokens - 1)) / pl.tile_tokens : a->batch * ((a->Tq + pl.tile_tokens - 1) / pl.tile_tokens);
    const long long items = pl.tiles * (a->Hq / pl.P);   // the parts do not depend on fill_rest: the result's bits do not either
    if (packed && a->fill_rest) pl.tiles += 2;
    pl.splits = 1;
    pl.part_keys = 0;
    if (items == 0 || a->Tk == 0) {
        pl.part_keys = 1 << 30;
        return pl;
    }
    if (pl.rows) {
        // two CTAs to an SM and several rounds of them, so that caches of different fill even out (a batch; for packed sequences see
        // above); 128 keys a part at least, and at most as many parts as the joining warp has lanes
        long long parts = (16ll * kNumSMs + items - 1) / items;
        if (parts > 32) parts = 32;
        long long keys = (a->Tk + parts - 1) / parts;
        keys = (keys + 127) / 128 * 128;
        pl.part_keys = static_cast<int>(keys);
        pl.splits = static_cast<int>((a->Tk + keys - 1) / keys);
    } else if (items * 2 <= kNumSMs) {                   // fewer CTAs than half the SMs: cut the keys into parts
        const long long key_tiles = (a->Tk + kAttnKeys - 1) / kAttnKeys;
        long long s = kNumSMs / items;
        if (s > key_tiles / 2) s = key_tiles / 2;        // two key tiles a part at least
        if (s > 32) s = 32;
        if (s > 1) pl.splits = static_cast<int>(s);
    }
    return pl;
}

static int attention_check(const sq_attention_args* a) {
    SQ_REQUIRE(a != nullptr, SQ_ERR_INVALID_ARG, "sq_attention: args is NULL");
    SQ_REQUIRE(a->dtype == SQ_F16 || a->dtype == SQ_BF16, SQ_ERR_UNSUPPORTED, "sq_attention: 16-bit tensors only (dtype %d)", a->dtype);
    SQ_REQUIRE(a->batch >= 0 && a->Tq >= 0 && a->Tk >= 0 && a->Hq >= 0, SQ_ERR_INVALID_ARG, "sq_attention: negative size");
    SQ_REQUIRE(a->Hkv > 0 && a->Hq % a->Hkv == 0, SQ_ERR_INVALID_ARG, "sq_attention: %d query heads do not share %d key heads evenly", a->Hq, a->Hkv);
    SQ_REQUIRE(a->D > 0 && a->D <= SQ_ATTENTION_MAX_D, SQ_ERR_UNSUPPORTED, "sq_attention: head width %d outside [8, %d]", a->D, SQ_ATTENTION_MAX_D);
    SQ_REQUIRE(a->D % 8 == 0, SQ_ERR_ALIGNMENT, "sq_attention: head width %d must be divisible by 8", a->D);
    SQ_REQUIRE(a->scale > 0.0f && a->scale < INFINITY, SQ_ERR_INVALID_ARG, "sq_attention: scale must be positive and finite");
    const bool packed = a->q_offsets_dev != nullptr;
    SQ_REQUIRE(packed == (a->kv_offsets_dev != nullptr), SQ_ERR_INVALID_ARG, "sq_attention: q_offsets_dev and kv_offsets_dev come together");
    SQ_REQUIRE(!packed || (!a->q_lens_dev && !a->kv_lens_dev), SQ_ERR_INVALID_ARG, "sq_attention: packed sequences have offsets, not lengths");
    SQ_REQUIRE(a->batch < (1 << 24) && a->Tq < (1ll << 30) && a->Tk < (1ll << 30) && a->Hq < (1 << 16), SQ_ERR_TOO_LARGE,
               "sq_attention: dimension too large");
    SQ_REQUIRE(packed || a->batch * a->Tq < (1ll << 31), SQ_ERR_TOO_LARGE, "sq_attention: too many query tokens");
    return SQ_OK;
}

long long attention_scratch_bytes(const sq_attention_args* a) {
    const int rc = attention_check(a);
    if (rc != SQ_OK) return rc;
    const long long tokens = a->q_offsets_dev ? a->Tq : a->batch * a->Tq;
    if (a->batch == 0 || tokens == 0 || a->Hq == 0) return 0;
    const AttnPlan pl = attention_plan(a);
    return pl.splits > 1 ? pl.splits * tokens * a->Hq * (a->D + 1ll) * 4 : 0;
}

// {columns, ...} tensor of 16-bit values: dims[0] = D contiguous, 64-column boxes in the 128-byte swizzled layout.
static int attention_map(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box,
                         const char* what) {
    auto fn = tensor_map_encoder();
    SQ_REQUIRE(fn != nullptr, SQ_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    cuuint64_t d[5], st[4];
    cuuint32_t bx[5], es[5];
    for (int i = 0; i < rank; ++i) {
        d[i] = dims[i];
        bx[i] = box[i];
        es[i] = 1;
        // the stride of a dimension of one element is never used, but has to be a legal one
        if (i > 0) st[i - 1] = dims[i] == 1 ? 16 : strides_bytes[i - 1];
    }
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, rank, const_cast<void*>(base), d, st, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    SQ_REQUIRE(r == CUDA_SUCCESS, SQ_ERR_CUDA, "sq_attention: cuTensorMapEncodeTiled(%s) failed with %d", what, static_cast<int>(r));
    return SQ_OK;
}

template <typename T, int DP>
static int attention_launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const AttnParams& p, long long grid, cudaStream_t st) {
    using C = AttnCfg<DP>;
    static bool attr_set[64] = {};
    int dev = 0;
    SQ_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 64 || !attr_set[dev]) {
        SQ_CUDA_OK(cudaFuncSetAttribute(attention_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
        if (dev < 64) attr_set[dev] = true;
    }
    attention_kernel<T, DP><<<static_cast<unsigned>(grid), kAttnThreads, C::kSmem, st>>>(mq, mk, mv, p);
    SQ_CUDA_OK(cudaGetLastError());
    return SQ_OK;
}

// The joining kernel is a programmatic dependent launch: it may start when the last CTA of the kernel before it has ended (none of
// them gives the signal sooner) and waits inside for that kernel's results.
template <typename T>
static int attention_join(const AttnParams& p, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((p.rows + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    SQ_CUDA_OK(cudaLaunchKernelEx(&cfg, attention_join_kernel<T>, p));
    return SQ_OK;
}

int attention(const sq_attention_args* a, cudaStream_t st) {
    int rc = attention_check(a);
    if (rc != SQ_OK) return rc;
    const bool packed = a->q_offsets_dev != nullptr;
    const long long tokens = packed ? a->Tq : a->batch * a->Tq;
    if (tokens == 0 || a->Hq == 0 || a->batch == 0) return SQ_OK;
    const bool keys = a->Tk > 0;
    SQ_REQUIRE(a->q_dev && a->out_dev && (!keys || (a->k_dev && a->v_dev)), SQ_ERR_INVALID_ARG, "sq_attention: NULL pointer");
    const void* ptrs[] = {a->q_dev, a->k_dev, a->v_dev, a->out_dev};
    for (const void* q : ptrs)
        SQ_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0, SQ_ERR_ALIGNMENT, "sq_attention: pointers must be 16-byte aligned");
    struct { long long n, s; const char* what; } strides[] = {
        {packed ? 1 : a->batch, a->q_batch_stride, "q"}, {a->Tq, a->q_token_stride, "q"}, {a->Hq, a->q_head_stride, "q"},
        {packed || !keys ? 1 : a->batch, a->k_batch_stride, "k"}, {a->Tk, a->k_token_stride, "k"}, {keys ? a->Hkv : 1, a->k_head_stride, "k"},
        {packed || !keys ? 1 : a->batch, a->v_batch_stride, "v"}, {a->Tk, a->v_token_stride, "v"}, {keys ? a->Hkv : 1, a->v_head_stride, "v"},
        {packed ? 1 : a->batch, a->out_batch_stride, "out"}, {a->Tq, a->out_token_stride, "out"}, {a->Hq, a->out_head_stride, "out"}};
    for (const auto& s : strides)
        SQ_REQUIRE(s.n <= 1 || (s.s > 0 && s.s % 8 == 0 && s.s < (1ll << 38)), SQ_ERR_ALIGNMENT,
                   "sq_attention: strides of %s must be positive multiples of 8 elements", s.what);
    const AttnPlan pl = attention_plan(a);
    const long long scratch = attention_scratch_bytes(a);
    SQ_REQUIRE(scratch == 0 || (a->scratch_dev && a->scratch_bytes >= scratch && reinterpret_cast<uintptr_t>(a->scratch_dev) % 16 == 0),
               SQ_ERR_INVALID_ARG, "sq_attention: needs %lld bytes of 16-byte aligned scratch (sq_attention_scratch_bytes)", scratch);
    const long long chunks = a->Hq / pl.P;
    const long long grid = pl.tiles * chunks * pl.splits;
    SQ_REQUIRE(grid < (1ll << 31), SQ_ERR_TOO_LARGE, "sq_attention: too many tiles");

    AttnParams p = {};
    p.q_off = a->q_offsets_dev; p.kv_off = a->kv_offsets_dev; p.q_lens = a->q_lens_dev; p.kv_lens = a->kv_lens_dev;
    p.batch = static_cast<int>(a->batch); p.Tq = static_cast<int>(a->Tq); p.Tk = static_cast<int>(a->Tk);
    p.fill_rest = a->fill_rest ? 1 : 0;
    p.causal = a->causal ? 1 : 0;
    p.Hq = a->Hq; p.Hkv = a->Hkv; p.D = a->D; p.G = a->Hq / a->Hkv; p.P = pl.P; p.chunks = static_cast<int>(chunks);
    p.tile_tokens = pl.tile_tokens; p.tiles = static_cast<int>(pl.tiles); p.splits = pl.splits; p.part_keys = pl.part_keys;
    p.q = a->q_dev;
    p.q_bs = a->q_batch_stride; p.q_ts = a->q_token_stride; p.q_hs = a->q_head_stride;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    p.o_bs = a->out_batch_stride; p.o_ts = a->out_token_stride; p.o_hs = a->out_head_stride;
    p.out = a->out_dev; p.lse = a->lse_dev;
    p.rows = tokens * a->Hq;
    if (pl.splits > 1) {
        p.part_o = static_cast<float*>(a->scratch_dev);
        p.part_lse = p.part_o + pl.splits * p.rows * a->D;
    }
    p.wait_cycles = wait_limit_cycles();

    CUtensorMap mq, mk, mv;
    const uint64_t nb = packed ? 1 : a->batch;
    if (!pl.rows || !keys) {
        const uint64_t dims[5] = {static_cast<uint64_t>(a->D), static_cast<uint64_t>(pl.P), static_cast<uint64_t>(chunks), static_cast<uint64_t>(a->Tq), nb};
        const uint64_t hs = a->q_head_stride * 2ull;
        const uint64_t sb[4] = {hs, hs * pl.P, a->q_token_stride * 2ull, a->q_batch_stride * 2ull};
        const uint32_t box[5] = {64, static_cast<uint32_t>(pl.P), 1, static_cast<uint32_t>(pl.tile_tokens / 2 > 0 ? pl.tile_tokens / 2 : 1), 1};
        rc = attention_map(&mq, a->q_dev, 5, dims, sb, box, "q");
        if (rc != SQ_OK) return rc;
    }
    if (!keys) {                                          // nothing is loaded; the kernels still take maps
        mk = mq;
        mv = mq;
    } else {
        const uint64_t dims[4] = {static_cast<uint64_t>(a->D), static_cast<uint64_t>(a->Hkv), static_cast<uint64_t>(a->Tk), nb};
        const uint32_t box[4] = {64, 1, pl.rows ? 32u : static_cast<uint32_t>(kAttnKeys), 1};
        const uint64_t sk[3] = {a->k_head_stride * 2ull, a->k_token_stride * 2ull, a->k_batch_stride * 2ull};
        const uint64_t sv[3] = {a->v_head_stride * 2ull, a->v_token_stride * 2ull, a->v_batch_stride * 2ull};
        rc = attention_map(&mk, a->k_dev, 4, dims, sk, box, "k");
        if (rc != SQ_OK) return rc;
        rc = attention_map(&mv, a->v_dev, 4, dims, sv, box, "v");
        if (rc != SQ_OK) return rc;
    }
    if (pl.rows) {
        rc = attention_rows(a->dtype, mk, mv, p, grid, st);
    } else if (a->dtype == SQ_F16) {
        rc = a->D <= 64 ? attention_launch<__half, 64>(mq, mk, mv, p, grid, st) : attention_launch<__half, 128>(mq, mk, mv, p, grid, st);
    } else {
        rc = a->D <= 64 ? attention_launch<__nv_bfloat16, 64>(mq, mk, mv, p, grid, st) : attention_launch<__nv_bfloat16, 128>(mq, mk, mv, p, grid, st);
    }
    if (rc != SQ_OK || p.splits == 1) return rc;
    return a->dtype == SQ_F16 ? attention_join<__half>(p, st) : attention_join<__nv_bfloat16>(p, st);
}

long long attention_read_status() {
    unsigned long long v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_wait_status, sizeof(v)) != cudaSuccess) return SQ_ERR_CUDA;
    if (v != 0 && cudaMemcpyToSymbol(g_wait_status, &zero, sizeof(zero)) != cudaSuccess) return SQ_ERR_CUDA;
    return static_cast<long long>(v);
}

}  // namespace sq
