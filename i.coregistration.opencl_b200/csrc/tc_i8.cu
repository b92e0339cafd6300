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
//   warps 2..17 epilogue, four per TMEM lane quadrant: a lane is a row, 16
//               sums at a time through scales, bias, activation and residual
//               into a swizzled block that a TMA store writes (clipped at
//               the matrix's edge); rows that no tensor map can describe go
//               out through the same block.
// Bytes of a row behind K, rows behind M and N: outside the tensor maps,
// which read them as zeros. Every mbarrier wait is bounded (tc_common.cuh).

#include "linear_i8.cuh"
#include "tc_common.cuh"

namespace coreg {
namespace tc {
namespace {

constexpr int BM = 128, BK = 128; // BK in bytes
// Sixteen epilogue warps, four to a scheduler: with eight (two) the latencies
// of their chain (scales, TMEM, activation, staging) bound the kernel, 10.8
// thousand cycles a 128 x 256 tile with GELU against 4.3 of its products.
constexpr int EPI_WARPS = 16, NTHREADS = 64 + 32 * EPI_WARPS;
// Bytes of an output block's row: 16 columns of float, 32 of bfloat16.
constexpr int ROW = 64;

struct Params {
    I8Gemm g;
    int tma_out;
    // Rows of C end at a multiple of 16 bytes. Where they do not, a store that
    // passes a row's end wrote the rest of its last 16 bytes too (measured),
    // so that the last columns go out without the tensor map.
    int clean;
    int al;   // sb and bias are 16-byte aligned
    int al_r; // rows of R are
};

template <int BN>
constexpr int stages() { return BN == 256 ? 4 : BN == 128 ? 6 : 8; }
template <int BN>
constexpr int acc_cols() { return BN; }

template <int BN>
struct Smem {
    alignas(1024) unsigned char a[stages<BN>()][BM * BK];
    alignas(1024) unsigned char b[stages<BN>()][BN * BK];
    alignas(1024) unsigned char cst[EPI_WARPS][32 * ROW];
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

// The 16 columns of p from col on, zero behind n; whole: they exist and are
// 16-byte aligned.
__device__ __forceinline__ void load_cols(float v[16], const float *p, int col, int n, bool whole)
{
    p += col;
    if (whole) {
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const float4 x = __ldg((const float4 *)(p + j));
            v[j] = x.x;
            v[j + 1] = x.y;
            v[j + 2] = x.z;
            v[j + 3] = x.w;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 16; j++)
        v[j] = col + j < n ? __ldg(p + j) : 0.0f;
}

// The 16 values of a residual row from R on, zero behind n; whole: they exist
// and are 16-byte aligned. (Not through the read-only cache: R may be C.)
__device__ __forceinline__ void load_row(float v[16], const float *R, int n, bool whole)
{
    if (whole) {
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            const float4 x = *(const float4 *)(R + j);
            v[j] = x.x;
            v[j + 1] = x.y;
            v[j + 2] = x.z;
            v[j + 3] = x.w;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 16; j++)
        v[j] = j < n ? R[j] : 0.0f;
}

__device__ __forceinline__ void load_row(float v[16], const __nv_bfloat16 *R, int n, bool whole)
{
    if (whole) {
#pragma unroll
        for (int j = 0; j < 16; j += 8) {
            const uint4 x = *(const uint4 *)(R + j);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                v[j + 2 * k] = __uint_as_float(w[k] << 16);
                v[j + 2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 16; j++)
        v[j] = j < n ? __bfloat162float(R[j]) : 0.0f;
}

// Address of 16-byte chunk c of row l of an output block, in its tensor map's
// 64-byte swizzle.
__device__ __forceinline__ unsigned char *chunk(unsigned char *blk, int l, int c)
{
    return blk + l * ROW + ((c ^ ((l >> 1) & 3)) << 4);
}

// 16 values of row l into a block, the h-th 16 of the row.
__device__ __forceinline__ void stage_row(unsigned char *blk, int l, int, const float v[16], float *)
{
#pragma unroll
    for (int c = 0; c < 4; c++)
        *(float4 *)chunk(blk, l, c) = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
}

__device__ __forceinline__ void stage_row(unsigned char *blk, int l, int h, const float v[16],
                                          __nv_bfloat16 *)
{
#pragma unroll
    for (int c = 0; c < 2; c++) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const __nv_bfloat162 x = __floats2bfloat162_rn(v[8 * c + 2 * k], v[8 * c + 2 * k + 1]);
            w[k] = *(const uint32_t *)&x;
        }
        *(uint4 *)chunk(blk, l, 2 * h + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// One epilogue warp's part of a tile: TMEM lanes 32 q .. (rows of the tile from
// m0 on) and the blocks part, part + 4, ... of columns (from n0 on) of the
// accumulator acc, which is complete when `full` turns `parity`. Returns false
// when that wait ran out; else the warp's reads of the accumulator are done.
template <int BN, int ACT, typename TC>
__device__ __forceinline__ bool tile_out(const Params &p, const CUtensorMap *tma_c,
                                         unsigned char *cst, uint32_t acc, uint64_t *full,
                                         uint32_t parity, int m0, int n0, int q, int part,
                                         int lane)
{
    constexpr int COLS = ROW / (int)sizeof(TC); // of a block
    const I8Gemm &g = p.g;
    TC *C = (TC *)g.C;
    const TC *R = (const TC *)g.R;
    m0 += 32 * q;
    const int row = m0 + lane;
    const float sa = row < g.M ? __ldg(g.sa + row) : 0.0f;
    constexpr int STEP = COLS * (EPI_WARPS / 4);
    // The residual into L2 while the products run: read in place its lines
    // came from memory one block after the other (15 thousand cycles of
    // epilogue for a 128 x 256 float tile, 6 without a residual).
    if (R && row < g.M)
        for (int c0 = COLS * part; c0 < BN && n0 + c0 < g.N; c0 += STEP)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(R + (long)row * g.ldc + n0 + c0));
    // Decided per warp: the TMEM loads below are warp-collective.
    if (!__all_sync(0xffffffffu, mbar_wait(full, parity, 63)))
        return false;
    fence_after();
    acc += (uint32_t)(32 * q) << 16;
    const bool whole = p.al && n0 + BN <= g.N;
    for (int c0 = COLS * part; c0 < BN && n0 + c0 < g.N; c0 += STEP) {
        const int col = n0 + c0;
        // The previous store has read the block.
        if (lane == 0)
            bulk_wait_read<0>();
        __syncwarp();
#pragma unroll
        for (int h = 0; h < COLS / 16; h++) {
            const int at = col + 16 * h;
            float v[16], sb[16], bias[16], r[16];
            if (R && row < g.M)
                load_row(r, R + (long)row * g.ldc + at, g.N - at, whole && p.al_r);
            load_cols(sb, g.sb, at, g.N, whole);
            if (g.bias)
                load_cols(bias, g.bias, at, g.N, whole);
            tmem_ld16(acc + c0 + 16 * h, v);
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
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
#pragma unroll
                for (int j = 0; j < 16; j++)
                    v[j] += r[j];
            stage_row(cst, lane, h, v, (TC *)nullptr);
        }
        if (p.tma_out && (col + COLS <= g.N || p.clean)) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
                tma_store_2d(tma_c, cst, col, m0);
                bulk_commit();
            }
            continue;
        }
        __syncwarp();
        // Rows without a tensor map: 32 / COLS rows at a time, lane = column.
        const int c = lane % COLS;
        if (col + c < g.N)
            for (int r = lane / COLS; r < 32 && m0 + r < g.M; r += 32 / COLS)
                C[(long)(m0 + r) * g.ldc + col + c] =
                    ((const TC *)chunk(cst, r, c * (int)sizeof(TC) / 16))[c % (16 / (int)sizeof(TC))];
    }
    // Each tcgen05.ld has waited: the accumulator may be written again.
    fence_before();
    __syncwarp();
    return true;
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
    after_previous();
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
        unsigned char *cst = s.cst[warp - 2];
        int lt = 0;
        for (int t = blockIdx.x; t < ntiles; t += gridDim.x, lt++) {
            const int buf = lt % 2;
            if (!tile_out<BN, ACT, TC>(p, &tma_c, cst, tmem + (uint32_t)(buf * acc_cols<BN>()),
                                       &s.acc_full[buf], lt / 2 & 1, (t % tiles_m) * BM,
                                       (t / tiles_m) * BN, warp % 4, (warp - 2) / 4, lane))
                break;
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
    launch_chained(tc_i8_k<BN, ACT, TC>, grid, NTHREADS, smem, st, ma, mb, mc, p);
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
    p.tma_out = make_map_rows(&mc, g.C, sizeof(TC), g.M, g.N, g.ldc * (long)sizeof(TC),
                              ROW / (int)sizeof(TC), 32, 64);
    p.al = (((uintptr_t)g.sb | (uintptr_t)g.bias) & 15) == 0;
    p.al_r = ((uintptr_t)g.R & 15) == 0 && g.ldc * (long)sizeof(TC) % 16 == 0;
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
    // The width whose tiles take the least time, in cycles: a round of tiles
    // costs its products or, where that is more, its epilogue, and the last
    // epilogue overlaps nothing. 128 bytes of depth take about 600 cycles at
    // any width: an MMA reads its 128 rows of A for 128 cycles, in which it
    // multiplies up to 256 columns (25616 x 4096 x 1024: 125 us with 256
    // columns, 144 with 128, 231 with 64; 500 x 500 x 500, where rounds do
    // not count: 13.5, 10.3 and 8.4).
    const int widths[3] = {256, 128, 64};
    int best = 0;
    double best_t = 0;
    for (int i = 0; i < 3; i++) {
        const int bn = widths[i];
        const long tiles = (long)cdiv(g.M, BM) * cdiv(g.N, bn), rounds = (tiles + sms - 1) / sms;
        const double main = 600.0 * cdiv(g.K, BK), epi = 1500.0 + 20.0 * bn;
        const double t = rounds * ((main > epi ? main : epi) + 500.0) + epi;
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
