// SPDX-License-Identifier: Unlicense
//
// The 8-bit product on the tcgen05 integer tensor cores (linear_i8.cuh): C =
// act((A B^T) sa sb + bias) + R with A (M x K) and B (N x K) of 8-bit
// integers, K-major, exact 32-bit sums in tensor memory.
//
// Persistent, one CTA per SM, over 128 x BN output tiles (row blocks fastest:
// the CTAs running at one time share weight columns in L2).
//   warp 0      TMA producer: 128 bytes of depth of A and B per stage,
//               128-byte swizzled, into a ring of STAGES;
//   warp 1      tensor memory and MMA: four tcgen05.mma.kind::i8 (K = 32 each)
//               per stage into one of two accumulators (tiles alternate);
//   warps 2..9  epilogue, two per TMEM lane quadrant: a lane is a row, 32
//               sums at a time through scales, bias, activation and residual
//               into a swizzled block that a TMA store writes (clipped at
//               the matrix's edge); rows that no tensor map can describe go
//               out through the same block, a row per warp store.
// Bytes of a row behind K, rows behind M and N: outside the tensor maps,
// which read them as zeros. Every mbarrier wait is bounded (tc_common.cuh).

#include "linear_i8.cuh"
#include "tc_common.cuh"

namespace coreg {
namespace tc {
namespace {

constexpr int BM = 128, BK = 128; // BK in bytes
constexpr int NTHREADS = 320, EPI_WARPS = 8;

struct Params {
    I8Gemm g;
    int tma_out;
    // Rows of C end at a multiple of 16 bytes. Where they do not, a store that
    // passes a row's end wrote the rest of its last 16 bytes too (measured),
    // so that the last columns go out without the tensor map.
    int clean;
};

template <int BN>
constexpr int stages() { return BN == 256 ? 4 : BN == 128 ? 6 : 8; }
template <int BN>
constexpr int acc_cols() { return BN; }

template <int BN>
struct Smem {
    alignas(1024) unsigned char a[stages<BN>()][BM * BK];
    alignas(1024) unsigned char b[stages<BN>()][BN * BK];
    alignas(1024) unsigned char cst[EPI_WARPS][4096];
    uint64_t full[stages<BN>()], empty[stages<BN>()], acc_full[2], acc_empty[2];
    uint32_t tmem;
};

// Instruction descriptor of kind::i8: signed 8-bit A and B, both K-major,
// 32-bit sums.
__host__ __device__ constexpr uint32_t idesc_i8(int M, int N)
{
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void mma_i8(uint32_t tmem, uint64_t da, uint64_t db, uint32_t idesc,
                                       uint32_t accum)
{
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
                 "l"(da), "l"(db), "r"(idesc), "r"(accum));
}

// The 32 columns of p from col on, zero behind n.
__device__ __forceinline__ void load_cols(float v[32], const float *p, int col, int n)
{
    p += col;
    if (col + 32 <= n && ((uintptr_t)p & 15) == 0) {
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
            const float4 x = __ldg((const float4 *)(p + j));
            v[j] = x.x;
            v[j + 1] = x.y;
            v[j + 2] = x.z;
            v[j + 3] = x.w;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 32; j++)
        v[j] = col + j < n ? __ldg(p + j) : 0.0f;
}

// v[j] += R[j] for the j < n (at most 32) columns of a residual row. (Not
// through the read-only cache: R may be C.)
__device__ __forceinline__ void add_row(float v[32], const float *R, int n)
{
    if (n >= 32 && ((uintptr_t)R & 15) == 0) {
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
            const float4 x = *(const float4 *)(R + j);
            v[j] += x.x;
            v[j + 1] += x.y;
            v[j + 2] += x.z;
            v[j + 3] += x.w;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 32; j++)
        if (j < n)
            v[j] += R[j];
}

__device__ __forceinline__ void add_row(float v[32], const __nv_bfloat16 *R, int n)
{
    if (n >= 32 && ((uintptr_t)R & 15) == 0) {
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
            const uint4 x = *(const uint4 *)(R + j);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                v[j + 2 * k] += __uint_as_float(w[k] << 16);
                v[j + 2 * k + 1] += __uint_as_float(w[k] & 0xffff0000u);
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 32; j++)
        if (j < n)
            v[j] += __bfloat162float(R[j]);
}

// Row l of a block of 32 columns in its tensor map's layout: rows of 128
// bytes (float; 16-byte chunk c at c ^ (l % 8)) or of 64 (bfloat16; c ^ ((l /
// 2) % 4)).
__device__ __forceinline__ void stage_row(unsigned char *blk, int l, const float v[32], float *)
{
#pragma unroll
    for (int c = 0; c < 8; c++)
        *(float4 *)(blk + l * 128 + ((c ^ (l & 7)) << 4)) =
            make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
}

__device__ __forceinline__ void stage_row(unsigned char *blk, int l, const float v[32],
                                          __nv_bfloat16 *)
{
#pragma unroll
    for (int c = 0; c < 4; c++) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[8 * c + 2 * k], v[8 * c + 2 * k + 1]);
            w[k] = *(const uint32_t *)&h;
        }
        *(uint4 *)(blk + l * 64 + ((c ^ ((l >> 1) & 3)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Element (l, j) of such a block.
__device__ __forceinline__ float staged(const unsigned char *blk, int l, int j, float *)
{
    return *(const float *)(blk + l * 128 + (((j >> 2) ^ (l & 7)) << 4) + (j & 3) * 4);
}

__device__ __forceinline__ __nv_bfloat16 staged(const unsigned char *blk, int l, int j,
                                                __nv_bfloat16 *)
{
    return *(const __nv_bfloat16 *)(blk + l * 64 + (((j >> 3) ^ ((l >> 1) & 3)) << 4) + (j & 7) * 2);
}

template <int BN, int ACT, typename TC>
__global__ void __launch_bounds__(NTHREADS, 1)
tc_i8_k(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
        const __grid_constant__ CUtensorMap tma_c, const Params p)
{
    constexpr int ST = stages<BN>();
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    Smem<BN> &s =
        *reinterpret_cast<Smem<BN> *>(smem_raw + ((1024u - (su32(smem_raw) & 1023u)) & 1023u));
    const I8Gemm &g = p.g;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int nk = (g.K + BK - 1) / BK;
    const int tiles_m = (g.M + BM - 1) / BM;
    const int ntiles = tiles_m * ((g.N + BN - 1) / BN);

    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) {
            mbar_init(&s.full[i], 1);
            mbar_init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&s.acc_full[i], 1);
            mbar_init(&s.acc_empty[i], EPI_WARPS);
        }
        mbar_fence_init();
    }
    if (warp == 1)
        tmem_alloc(&s.tmem, 2 * acc_cols<BN>());
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = s.tmem;

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int t = blockIdx.x; t < ntiles && ok; t += gridDim.x) {
                const int m0 = (t % tiles_m) * BM, n0 = (t / tiles_m) * BN;
                for (int kb = 0; kb < nk; kb++, it++) {
                    const int st = it % ST;
                    if (it >= ST && !mbar_wait(&s.empty[st], ((it / ST) - 1) & 1, 61)) {
                        ok = false;
                        break;
                    }
                    mbar_expect_tx(&s.full[st], (BM + BN) * BK);
                    tma_load_2d(s.a[st], &tma_a, &s.full[st], kb * BK, m0);
                    tma_load_2d(s.b[st], &tma_b, &s.full[st], kb * BK, n0);
                }
            }
        }
    }
    else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = idesc_i8(BM, BN);
            int it = 0, lt = 0;
            bool ok = true;
            for (int t = blockIdx.x; t < ntiles && ok; t += gridDim.x, lt++) {
                const int buf = lt % 2, use = lt / 2;
                // The epilogue has read this accumulator's previous tile.
                if (use > 0 && !mbar_wait(&s.acc_empty[buf], (use - 1) & 1, 64))
                    break;
                fence_after();
                const uint32_t acc = tmem + (uint32_t)(buf * acc_cols<BN>());
                for (int kb = 0; kb < nk; kb++, it++) {
                    const int st = it % ST;
                    if (!mbar_wait(&s.full[st], (it / ST) & 1, 62)) {
                        ok = false;
                        break;
                    }
                    const uint64_t da = sw128_desc(su32(s.a[st])), db = sw128_desc(su32(s.b[st]));
#pragma unroll
                    for (int k = 0; k < BK / 32; k++)
                        mma_i8(acc, da + 2 * k, db + 2 * k, idesc, (kb > 0 || k > 0) ? 1u : 0u);
                    mma_commit(&s.empty[st]);
                }
                if (ok)
                    mma_commit(&s.acc_full[buf]);
            }
        }
    }
    else {
        // Warp w: TMEM lanes 32 (w % 4) .., the 32-column chunks of parity (w -
        // 2) / 4.
        const int q = warp % 4, half = (warp - 2) / 4;
        unsigned char *cst = s.cst[warp - 2];
        TC *C = (TC *)g.C;
        const TC *R = (const TC *)g.R;
        int lt = 0;
        for (int t = blockIdx.x; t < ntiles; t += gridDim.x, lt++) {
            const int buf = lt % 2, use = lt / 2;
            const int m0 = (t % tiles_m) * BM + 32 * q, n0 = (t / tiles_m) * BN;
            const int row = m0 + lane;
            const float sa = row < g.M ? __ldg(g.sa + row) : 0.0f;
            // Decided per warp: the TMEM loads below are warp-collective.
            if (!__all_sync(0xffffffffu, mbar_wait_backoff(&s.acc_full[buf], use & 1, 63)))
                break;
            fence_after();
            const uint32_t acc =
                tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(buf * acc_cols<BN>());
            for (int c0 = 32 * half; c0 < BN && n0 + c0 < g.N; c0 += 64) {
                const int col = n0 + c0;
                float v[32], sb[32], bias[32];
                load_cols(sb, g.sb, col, g.N);
                if (g.bias)
                    load_cols(bias, g.bias, col, g.N);
                tmem_ld32(acc + c0, v);
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    // The token's scale first (see scaled() in linear_i8.cu).
                    const float2 y = fma2(make_float2(__int2float_rn(__float_as_int(v[j])),
                                                      __int2float_rn(__float_as_int(v[j + 1]))),
                                          pair(sa), pair(0.0f));
                    const float2 x = act2<ACT>(
                        fma2(y, make_float2(sb[j], sb[j + 1]),
                             g.bias ? make_float2(bias[j], bias[j + 1]) : pair(0.0f)),
                        g.slope);
                    v[j] = x.x;
                    v[j + 1] = x.y;
                }
                if (R && row < g.M)
                    add_row(v, R + (long)row * g.ldc + col, g.N - col);
                // The previous store has read the staging block.
                if (lane == 0)
                    bulk_wait_read<0>();
                __syncwarp();
                stage_row(cst, lane, v, (TC *)nullptr);
                if (p.tma_out && (col + 32 <= g.N || p.clean)) {
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tma_c, cst, col, m0);
                        bulk_commit();
                    }
                    continue;
                }
                __syncwarp();
                if (col + lane < g.N)
                    for (int r = 0; r < 32 && m0 + r < g.M; r++)
                        C[(long)(m0 + r) * g.ldc + col + lane] = staged(cst, r, lane, (TC *)nullptr);
            }
            // This warp's reads of the accumulator are complete (each
            // tcgen05.ld waited): hand it back to the MMA warp.
            fence_before();
            __syncwarp();
            if (lane == 0)
                mbar_arrive(&s.acc_empty[buf]);
        }
        // This warp's TMA stores have written global memory.
        if (lane == 0)
            bulk_wait_all();
    }
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        tmem_dealloc(tmem, 2 * acc_cols<BN>());
    }
}

template <int BN, int ACT, typename TC>
bool run(cudaStream_t st, int grid, const CUtensorMap &ma, const CUtensorMap &mb,
         const CUtensorMap &mc, const Params &p)
{
    const size_t smem = sizeof(Smem<BN>) + 1024;
    static unsigned done = 0;
    if (!smem_opt_in((const void *)tc_i8_k<BN, ACT, TC>, smem, &done))
        return false;
    tc_i8_k<BN, ACT, TC><<<grid, NTHREADS, smem, st>>>(ma, mb, mc, p);
    return true;
}

template <int BN, typename TC>
bool launch(cudaStream_t st, const I8Gemm &g, int sms)
{
    CUtensorMap ma, mb, mc = {};
    Params p;
    p.g = g;
    if (!make_map_rows(&ma, g.A, 1, g.M, g.K, g.lda, BK, BM, 128) ||
        !make_map_rows(&mb, g.B, 1, g.N, g.K, g.ldb, BK, BN, 128))
        return false;
    p.tma_out = make_map_rows(&mc, g.C, sizeof(TC), g.M, g.N, g.ldc * (long)sizeof(TC), 32, 32,
                              sizeof(TC) == 4 ? 128 : 64);
    p.clean = (long)g.N * (int)sizeof(TC) % 16 == 0;
    const long tiles = (long)cdiv(g.M, BM) * cdiv(g.N, BN);
    if (tiles >= (1L << 31))
        return false;
    const int grid = (int)(tiles < sms ? tiles : sms);
    switch (g.act) {
    case ACT_GELU:
        return run<BN, ACT_GELU, TC>(st, grid, ma, mb, mc, p);
    case ACT_RELU:
        return run<BN, ACT_RELU, TC>(st, grid, ma, mb, mc, p);
    case ACT_LEAKY:
        return run<BN, ACT_LEAKY, TC>(st, grid, ma, mb, mc, p);
    case ACT_GELU_TANH:
        return run<BN, ACT_GELU_TANH, TC>(st, grid, ma, mb, mc, p);
    case ACT_SILU:
        return run<BN, ACT_SILU, TC>(st, grid, ma, mb, mc, p);
    }
    return run<BN, ACT_NONE, TC>(st, grid, ma, mb, mc, p);
}

template <typename TC>
bool choose(cudaStream_t st, const I8Gemm &g, int sms)
{
    // The width whose tiles take the least time over their rounds of CTAs.
    const int widths[3] = {256, 128, 64};
    int best = 0;
    double best_t = 0;
    for (int i = 0; i < 3; i++) {
        const long tiles = (long)cdiv(g.M, BM) * cdiv(g.N, widths[i]);
        const double t = (double)((tiles + sms - 1) / sms) * (widths[i] + 24);
        if (i == 0 || t < best_t) {
            best = i;
            best_t = t;
        }
    }
    return best == 0   ? launch<256, TC>(st, g, sms)
           : best == 1 ? launch<128, TC>(st, g, sms)
                       : launch<64, TC>(st, g, sms);
}

}  // namespace

int i8_status()
{
    int v = 0, z = 0;
    cudaMemcpyFromSymbol(&v, g_error, sizeof(int));
    if (v)
        cudaMemcpyToSymbol(g_error, &z, sizeof(int));
    return v;
}

}  // namespace tc

bool gemm_i8_tc(cudaStream_t st, const I8Gemm &g, int sms)
{
    return g.c_bf16 ? tc::choose<__nv_bfloat16>(st, g, sms) : tc::choose<float>(st, g, sms);
}

}  // namespace coreg
