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
// which read them as zeros (of fewer rows than a tile's, see box_rows). Every
// mbarrier wait is bounded (tc_common.cuh).

#include <type_traits>

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
// Bytes of an output block's row: 16 columns of float, 32 of bfloat16. (Rows of
// 128 bytes cost a stage of the ring, which costs more: CTA pairs with four
// stages and such rows 154 us against 145 with five.)
constexpr int ROW = 64;

struct Params {
    I8Gemm g;
    int tma_out;
    // Rows of C end at a multiple of 16 bytes. Where they do not, a store that
    // passes a row's end wrote the rest of its last 16 bytes too (measured),
    // so that the last columns go out without the tensor map.
    int clean;
    int al;   // sb and bias are 16-byte aligned
    int al_r; // rows of R are (in split depths: 1, and 2 where those of C are)
};

// Rows of A that a load brings, of M: a tile's, or where there are fewer only those,
// in eights. Rows outside the tensor map are read as zeros, but each costs more than
// a row inside it (8 tokens as 128 rows x 8192 x 1500 11 us, as 8 rows 5.6). What
// a stage holds behind them reaches only sums that nothing reads. (The
// last tile of many with a box of its own: no gain.)
__host__ __device__ __forceinline__ int box_rows(int M, int tile)
{
    return M < tile ? (M + 7) / 8 * 8 : tile;
}

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
            const float4 x = *(const float4 *)(p + j);
            v[j] = x.x;
            v[j + 1] = x.y;
            v[j + 2] = x.z;
            v[j + 3] = x.w;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 16; j++)
        v[j] = col + j < n ? p[j] : 0.0f;
}

// Four neighbours of p, zero behind n and where p is NULL; al: 16-byte
// aligned as float (8 as bfloat16).
__device__ __forceinline__ void load_quad(float v[4], const float *p, int n, bool al)
{
    if (p && al && n >= 4) {
        const float4 x = *(const float4 *)p;
        v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
        v[j] = p && j < n ? p[j] : 0.0f;
}

__device__ __forceinline__ void load_quad(float v[4], const __nv_bfloat16 *p, int n, bool al)
{
    if (p && al && n >= 4) {
        const uint2 x = *(const uint2 *)p;
        v[0] = __uint_as_float(x.x << 16), v[1] = __uint_as_float(x.x & 0xffff0000u);
        v[2] = __uint_as_float(x.y << 16), v[3] = __uint_as_float(x.y & 0xffff0000u);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
        v[j] = p && j < n ? ldf(p + j) : 0.0f;
}

__device__ __forceinline__ void store_quad(float *p, const float v[4], int n, bool al)
{
    if (al && n >= 4) {
        *(float4 *)p = make_float4(v[0], v[1], v[2], v[3]);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (j < n)
            p[j] = v[j];
}

__device__ __forceinline__ void store_quad(__nv_bfloat16 *p, const float v[4], int n, bool al)
{
    if (al && n >= 4) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]),
                             b = __floats2bfloat162_rn(v[2], v[3]);
        *(uint2 *)p = make_uint2(*(const uint32_t *)&a, *(const uint32_t *)&b);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (j < n)
            stf(p + j, v[j]);
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
        *(float4 *)chunk(blk, l, c) =
            make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
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

// v += those 16 values of a block.
__device__ __forceinline__ void add_staged(float v[16], unsigned char *blk, int l, int, const float *)
{
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const float4 x = *(const float4 *)chunk(blk, l, c);
        v[4 * c] += x.x;
        v[4 * c + 1] += x.y;
        v[4 * c + 2] += x.z;
        v[4 * c + 3] += x.w;
    }
}

__device__ __forceinline__ void add_staged(float v[16], unsigned char *blk, int l, int h,
                                           const __nv_bfloat16 *)
{
#pragma unroll
    for (int c = 0; c < 2; c++) {
        const uint4 x = *(const uint4 *)chunk(blk, l, 2 * h + c);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            v[8 * c + 2 * k] += __uint_as_float(w[k] << 16);
            v[8 * c + 2 * k + 1] += __uint_as_float(w[k] & 0xffff0000u);
        }
    }
}

// One epilogue warp's part of a tile: TMEM lanes 32 q .. (rows of the tile from
// m0 on) and the blocks part, part + 4, ... of columns (from n0 on) of the
// accumulator acc, which is complete when `full` turns `parity`. SHARED: the
// scales and the bias of the tile's columns are in shared memory at cols and
// cols + BN. Returns false when that wait ran out; else the warp's reads of
// the accumulator are done.
template <int BN, bool SHARED, int ACT, typename TC>
__device__ __forceinline__ bool tile_out(const Params &p, const CUtensorMap *tma_c,
                                         unsigned char *cst, uint32_t acc, uint64_t *full,
                                         uint32_t parity, int m0, int n0, int q, int part,
                                         int lane, const float *cols)
{
    constexpr int COLS = ROW / (int)sizeof(TC); // of a block
    const I8Gemm &g = p.g;
    TC *C = (TC *)g.C;
    const TC *R = (const TC *)g.R;
    m0 += 32 * q;
    const int row = m0 + lane;
    const float sa = row < g.M ? g.sa[row] : 0.0f;
    constexpr int STEP = COLS * (EPI_WARPS / 4);
    // The residual's blocks come as the output's leave: 64-byte row segments by
    // four lanes each, through the staging block, the first while the
    // products run, each further one a block ahead (and all of them into
    // L2). Read by one lane per row they took 32 memory lines an
    // instruction, and 14 thousand cycles of a 128 x 256 float tile.
    const bool whole = p.al && n0 + BN <= g.N, by_block = R && p.al_r && n0 + BN <= g.N;
    // Rows that are not 16-byte aligned come value by value, a lane a column (1003
    // x 3150 x 638 bfloat16 30.5 -> 17.5 us, 2528 x 3250 x 308 float 58 -> 31).
    uint32_t next[16];
    auto fetch = [&](int c0) {
        if (by_block) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = m0 + 8 * i + lane / 4;
                if (r < g.M) {
                    const uint4 x = *((const uint4 *)(R + (long)r * g.ldc + n0 + c0) + lane % 4);
                    next[4 * i] = x.x, next[4 * i + 1] = x.y;
                    next[4 * i + 2] = x.z, next[4 * i + 3] = x.w;
                }
            }
            return;
        }
        const int c = n0 + c0 + lane % COLS;
        const bool in = c < g.N;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            next[i] = 0;
            if constexpr (sizeof(TC) == 4) {
                const int r = m0 + 2 * i + lane / 16;
                if (in && r < g.M)
                    next[i] = *(const uint32_t *)(R + (long)r * g.ldc + c);
            }
            else {
                const int r = m0 + 2 * i;
                if (in && r < g.M)
                    next[i] = *(const uint16_t *)(R + (long)r * g.ldc + c);
                if (in && r + 1 < g.M)
                    next[i] |= (uint32_t) * (const uint16_t *)(R + (long)(r + 1) * g.ldc + c) << 16;
            }
        }
    };
    // What fetch brought, into the staging block.
    auto put = [&]() {
        if (by_block) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                *(uint4 *)chunk(cst, 8 * i + lane / 4, lane % 4) =
                    make_uint4(next[4 * i], next[4 * i + 1], next[4 * i + 2], next[4 * i + 3]);
            return;
        }
        constexpr int E = 16 / (int)sizeof(TC);
        const int c = lane % COLS;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            if constexpr (sizeof(TC) == 4) {
                ((uint32_t *)chunk(cst, 2 * i + lane / 16, c / E))[c % E] = next[i];
            }
            else {
                ((uint16_t *)chunk(cst, 2 * i, c / E))[c % E] = (uint16_t)next[i];
                ((uint16_t *)chunk(cst, 2 * i + 1, c / E))[c % E] = (uint16_t)(next[i] >> 16);
            }
        }
    };
    if (R && row < g.M)
        for (int c0 = COLS * part + STEP; c0 < BN && n0 + c0 < g.N; c0 += STEP)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(R + (long)row * g.ldc + n0 + c0));
    if (R && COLS * part < BN && n0 + COLS * part < g.N)
        fetch(COLS * part);
    // Decided per warp: the TMEM loads below are warp-collective.
    if (!__all_sync(0xffffffffu, mbar_wait(full, parity, 63)))
        return false;
    fence_after();
    acc += (uint32_t)(32 * q) << 16;
    for (int c0 = COLS * part; c0 < BN && n0 + c0 < g.N; c0 += STEP) {
        const int col = n0 + c0;
        // The previous store has read the block.
        if (lane == 0)
            bulk_wait_read<0>();
        __syncwarp();
        if (R) {
            put();
            __syncwarp();
            if (c0 + STEP < BN && n0 + c0 + STEP < g.N)
                fetch(c0 + STEP);
        }
#pragma unroll
        for (int h = 0; h < COLS / 16; h++) {
            const int at = col + 16 * h;
            float v[16], sb[16], bias[16];
            if (SHARED) {
                load_cols(sb, cols, at - n0, BN, true);
                load_cols(bias, cols + BN, at - n0, BN, true);
            }
            else {
                load_cols(sb, g.sb, at, g.N, whole);
                if (g.bias)
                    load_cols(bias, g.bias, at, g.N, whole);
            }
            tmem_ld16(acc + c0 + 16 * h, v);
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                // The token's scale first (see scaled() in linear_i8.cu).
                const float2 y = fma2(make_float2(__int2float_rn(__float_as_int(v[j])),
                                                  __int2float_rn(__float_as_int(v[j + 1]))),
                                      pair(sa), pair(0.0f));
                const float2 x = act2<ACT>(
                    fma2(y, make_float2(sb[j], sb[j + 1]),
                         SHARED || g.bias ? make_float2(bias[j], bias[j + 1]) : pair(0.0f)),
                    g.slope);
                v[j] = x.x;
                v[j + 1] = x.y;
            }
            if (R)
                add_staged(v, cst, lane, h, (const TC *)nullptr);
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
        // Rows without a tensor map: lane = column, several rows at a time where
        // they are short. (Eight reads ahead of their writes: 19428 x 1298 x 23
        // bfloat16 76 us against 53.)
        constexpr int E = 16 / (int)sizeof(TC);
        const int c = lane % COLS;
        if (col + c < g.N)
            for (int r = lane / COLS; r < 32 && m0 + r < g.M; r += 32 / COLS)
                C[(long)(m0 + r) * g.ldc + col + c] = ((const TC *)chunk(cst, r, c / E))[c % E];
    }
    // Each tcgen05.ld has waited: the accumulator may be written again.
    fence_before();
    __syncwarp();
    return true;
}

// FEW: fewer rows than a tile's. (Kernels of their own: the box's bytes as a
// variable cost the others 0.1 us a call.)
template <int BN, int ACT, bool FEW, typename TC>
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
                    mbar_expect_tx(&s.full[st], ((FEW ? box_rows(g.M, BM) : BM) + BN) * BK);
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
            if (!tile_out<BN, false, ACT, TC>(p, &tma_c, cst, tmem + (uint32_t)(buf * acc_cols<BN>()),
                                       &s.acc_full[buf], lt / 2 & 1, (t % tiles_m) * BM,
                                       (t / tiles_m) * BN, warp % 4, (warp - 2) / 4, lane,
                                       nullptr))
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

// ------------------------------------------------------------- CTA pairs
//
// 256 x 256 tiles by two CTAs of a cluster (tcgen05 cta_group::2): each holds 128
// rows of A, half the rows of B and the sums of its 128 rows; the tensor cores
// of both read B from both. Per product that is a third less shared memory
// and L2 traffic than the 128 x 256 tile's, which saves power (these kernels
// run at the power limit: 25616 x 4096 x 1024 at about 1.5 GHz of 1.9), and
// leaves room for five stages and the columns' scales.
// The roles are those above, in each CTA; the first of the pair (the leader)
// alone issues the products, for both:
//   full[s]      the leader's: both CTAs' loads of a stage complete on it;
//   empty[s]     each CTA's own, arrived at in both by the leader's commit;
//   acc_full     likewise;
//   acc_empty    the leader's: the epilogue warps of both CTAs arrive.
constexpr int PAIR_ST = 5, PAIR_BN = 256;

struct PairSmem {
    alignas(1024) unsigned char a[PAIR_ST][BM * BK];
    alignas(1024) unsigned char b[PAIR_ST][PAIR_BN / 2 * BK];
    alignas(1024) unsigned char cst[EPI_WARPS][32 * ROW];
    alignas(16) float cols[2][2 * PAIR_BN];
    uint64_t full[PAIR_ST], empty[PAIR_ST], acc_full[2], acc_empty[2];
    uint32_t tmem;
};

__device__ __forceinline__ uint32_t cta_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// The cluster address of a barrier of the pair's leader.
__device__ __forceinline__ uint32_t of_leader(const uint64_t *bar)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(su32(bar)));
    return r;
}

// A box into this CTA's shared memory that completes on a barrier of the pair.
__device__ __forceinline__ void pair_load_2d(void *dst, const CUtensorMap *map, uint32_t bar, int x,
                                             int y)
{
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::"
                 "bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(su32(dst)),
                 "l"((uint64_t)map), "r"(bar), "r"(x), "r"(y)
                 : "memory");
}

__device__ __forceinline__ void pair_mma_i8(uint32_t tmem, uint64_t da, uint64_t db,
                                            uint32_t idesc, uint32_t accum)
{
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
                 "l"(da), "l"(db), "r"(idesc), "r"(accum));
}

// The issued products done: arrives at the barrier's place in both CTAs.
__device__ __forceinline__ void pair_commit(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::"
                 "cluster.b64 [%0], %1;" ::"r"(su32(bar)),
                 "h"((uint16_t)3)
                 : "memory");
}

__device__ __forceinline__ void pair_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
                 : "memory");
}

// mbar_wait for arrivals from the other CTA.
__device__ __forceinline__ bool pair_wait(uint64_t *b, uint32_t parity, int code)
{
    uint64_t t0 = 0;
    for (;;) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\t"
                     "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
                     "selp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok)
                     : "r"(su32(b)), "r"(parity)
                     : "memory");
        if (ok)
            return true;
        if (!t0)
            t0 = gtime();
        else if (gtime() - t0 > 2000000000ull) {
            atomicCAS(&g_error, 0, code);
            return false;
        }
    }
}

__device__ __forceinline__ void cluster_arrive()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}

__device__ __forceinline__ void cluster_wait()
{
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void cluster_sync()
{
    cluster_arrive();
    cluster_wait();
}

template <int ACT, typename TC>
__global__ void __launch_bounds__(NTHREADS, 1) __cluster_dims__(2, 1, 1)
tc_i8_pair_k(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
             const __grid_constant__ CUtensorMap tma_c, const Params p)
{
    constexpr int ST = PAIR_ST, BN = PAIR_BN;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    PairSmem &s =
        *reinterpret_cast<PairSmem *>(smem_raw + ((1024u - (su32(smem_raw) & 1023u)) & 1023u));
    const I8Gemm &g = p.g;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = (int)cta_rank(), pairs = (int)gridDim.x / 2;
    const int nk = (g.K + BK - 1) / BK;
    const int tiles_m = (g.M + 2 * BM - 1) / (2 * BM);
    const int ntiles = tiles_m * ((g.N + BN - 1) / BN);

    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) {
            mbar_init(&s.full[i], 1);
            mbar_init(&s.empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&s.acc_full[i], 1);
            mbar_init(&s.acc_empty[i], 2 * EPI_WARPS);
        }
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         su32(&s.tmem)),
                     "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    after_previous();
    fence_before();
    __syncthreads();
    cluster_sync();
    fence_after();
    const uint32_t tmem = s.tmem;

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int t = blockIdx.x / 2; t < ntiles && ok; t += pairs) {
                const int m0 = (t % tiles_m) * 2 * BM + rank * BM;
                const int n0 = (t / tiles_m) * BN + rank * (BN / 2);
                for (int kb = 0; kb < nk; kb++, it++) {
                    const int st = it % ST;
                    if (it >= ST && !pair_wait(&s.empty[st], ((it / ST) - 1) & 1, 71)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0)
                        mbar_expect_tx(&s.full[st], 2 * (BM + BN / 2) * BK);
                    const uint32_t bar = of_leader(&s.full[st]);
                    pair_load_2d(s.a[st], &tma_a, bar, kb * BK, m0);
                    pair_load_2d(s.b[st], &tma_b, bar, kb * BK, n0);
                }
            }
        }
    }
    else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = idesc_i8(2 * BM, BN);
            int it = 0, lt = 0;
            bool ok = true;
            for (int t = blockIdx.x / 2; t < ntiles && ok; t += pairs, lt++) {
                const int buf = lt % 2, use = lt / 2;
                if (use > 0 && !pair_wait(&s.acc_empty[buf], (use - 1) & 1, 74))
                    break;
                fence_after();
                const uint32_t acc = tmem + (uint32_t)(buf * BN);
                for (int kb = 0; kb < nk; kb++, it++) {
                    const int st = it % ST;
                    if (!pair_wait(&s.full[st], (it / ST) & 1, 72)) {
                        ok = false;
                        break;
                    }
                    const uint64_t da = sw128_desc(su32(s.a[st])), db = sw128_desc(su32(s.b[st]));
#pragma unroll
                    for (int k = 0; k < BK / 32; k++)
                        pair_mma_i8(acc, da + 2 * k, db + 2 * k, idesc, (kb > 0 || k > 0) ? 1u : 0u);
                    pair_commit(&s.empty[st]);
                }
                if (ok)
                    pair_commit(&s.acc_full[buf]);
            }
        }
    }
    else {
        unsigned char *cst = s.cst[warp - 2];
        // Scales and bias of a tile's columns, one value per epilogue thread,
        // fetched a tile ahead. (Read from global memory by every warp they
        // were 1.7 of the 6 thousand cycles of an epilogue.) The barrier of
        // the next tile is behind every read of this one's.
        const int me = threadIdx.x - 64;
        auto value = [&](int t) {
            const int c = (t / tiles_m) * BN + me % BN;
            const float *from = me < BN ? g.sb : g.bias;
            return t < ntiles && from && c < g.N ? from[c] : 0.0f;
        };
        float next = value(blockIdx.x / 2);
        bool ok = true;
        int lt = 0;
        for (int t = blockIdx.x / 2; t < ntiles; t += pairs, lt++) {
            const int buf = lt % 2;
            float *cols = s.cols[buf];
            cols[me] = next;
            named_bar(1, 32 * EPI_WARPS);
            next = value(t + pairs);
            // (A warp whose wait ran out keeps to the barriers of the others.)
            ok = ok && tile_out<BN, true, ACT, TC>(
                           p, &tma_c, cst, tmem + (uint32_t)(buf * BN), &s.acc_full[buf],
                           lt / 2 & 1, (t % tiles_m) * 2 * BM + rank * BM, (t / tiles_m) * BN,
                           warp % 4, (warp - 2) / 4, lane, cols);
            if (ok && lane == 0)
                pair_arrive(of_leader(&s.acc_empty[buf]));
        }
        if (lane == 0)
            bulk_wait_all();
    }
    // Neither CTA leaves while the other's barriers, operands or loads need it.
    fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    }
}

// ------------------------------------------------------------ split depth
//
// One 128 x BN tile by a cluster of S CTAs, each over a part of the depth: for
// deep products of few tiles, in which a CTA's chain of stages (some 600
// cycles per 128 bytes of depth) is the time (us, M x N x K: 33 x 1024 x 8192
// 20.4 -> 6.6, 128 x 4096 x 4096 12.5 -> 8.5, 256 x 1024 x 4096 12.4 -> 6.3, 8 x
// 8192 x 8192 32 -> 15, 4.5 TB/s of weights, the call's some 4 us included;
// tiles 256 wide for few rows took the same). A CTA hands its sums of the r-th
// S-th of the columns to the cluster's CTA r, through that one's shared
// memory, and finishes its own columns from all S parts. The sums are
// integers: the split changes no result.
// ROWS: rows of A that a stage holds. For up to 32 tokens it keeps only those, in
// twice the stages: the products read 128 rows all the same, the others from
// the stages behind (b is behind a, and larger), into sums that nothing reads
// (16 x 8192 x 8192 17.0 us with 128 rows and four stages, 15.6).
template <int BN, int ROWS>
struct SplitSmem {
    static constexpr int ST = ROWS == 32 ? 8 : BN == 128 ? 4 : 6;
    // Four columns of the rows, 16 bytes a row (32 bytes more keep the finishing
    // reads, neighbouring quads of columns first, off each other's banks).
    static constexpr int QUAD = ROWS * 16 + 32;
    alignas(1024) unsigned char a[ST][ROWS * BK];
    alignas(1024) unsigned char b[ST][BN * BK];
    // [CTA they come from][quad of this one's columns][row].
    alignas(16) unsigned char part[BN / 4 * QUAD];
    uint64_t full[ST], empty[ST], acc_full;
    uint32_t tmem;
};

// 16 bytes into the same place of the cluster's CTA r.
__device__ __forceinline__ void store_to(uint32_t at, int r, const float *v)
{
    uint32_t to;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(at), "r"(r));
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(v[0]), "f"(v[1]),
                 "f"(v[2]), "f"(v[3])
                 : "memory");
}

template <int BN, int ROWS, int S, typename TC>
__global__ void __launch_bounds__(NTHREADS, 1)
tc_i8_split_k(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
              const Params p)
{
    using Smem = SplitSmem<BN, ROWS>;
    constexpr int ST = Smem::ST, QUAD = Smem::QUAD, THREADS = 32 * EPI_WARPS;
    constexpr int NQ = BN / 4 / S;                               // quads of a CTA's columns
    constexpr int ITEMS = (NQ * ROWS + THREADS - 1) / THREADS;   // of a thread: a row of a quad
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    Smem &s =
        *reinterpret_cast<Smem *>(smem_raw + ((1024u - (su32(smem_raw) & 1023u)) & 1023u));
    const I8Gemm &g = p.g;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = (int)cta_rank(), tile = blockIdx.x / S;
    const int nk = (g.K + BK - 1) / BK;
    const int tiles_m = (g.M + BM - 1) / BM;
    const int m0 = tile % tiles_m * BM, n0 = tile / tiles_m * BN;
    // This CTA's depth (nk >= S).
    const int kb0 = (int)((long)nk * rank / S), kb1 = (int)((long)nk * (rank + 1) / S);

    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) {
            mbar_init(&s.full[i], 1);
            mbar_init(&s.empty[i], 1);
        }
        mbar_init(&s.acc_full, 1);
        mbar_fence_init();
    }
    if (warp == 1)
        tmem_alloc(&s.tmem, BN);
    after_previous();
    fence_before();
    __syncthreads();
    fence_after();
    // Every CTA of the cluster has started: its shared memory may be written.
    // (Waited for by the epilogue only.)
    cluster_arrive();
    const uint32_t tmem = s.tmem;
    // Scales, bias and residual of the thread's items, fetched meanwhile.
    float sa[ITEMS], sb[ITEMS][4], bias[ITEMS][4], res[ITEMS][4];
    bool live[ITEMS];
    const int me = threadIdx.x - 64;

    if (warp == 0) {
        if (lane == 0) {
            for (int kb = kb0; kb < kb1; kb++) {
                const int it = kb - kb0, st = it % ST;
                if (it >= ST && !mbar_wait(&s.empty[st], ((it / ST) - 1) & 1, 81))
                    break;
                mbar_expect_tx(&s.full[st], (box_rows(g.M, ROWS) + BN) * BK);
                tma_load_2d(s.a[st], &tma_a, &s.full[st], kb * BK, m0);
                tma_load_2d(s.b[st], &tma_b, &s.full[st], kb * BK, n0);
            }
        }
        __syncwarp();
        cluster_wait();
    }
    else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = idesc_i8(BM, BN);
            bool ok = true;
            for (int kb = kb0; kb < kb1; kb++) {
                const int it = kb - kb0, st = it % ST;
                if (!mbar_wait(&s.full[st], (it / ST) & 1, 82)) {
                    ok = false;
                    break;
                }
                const uint64_t da = sw128_desc(su32(s.a[st])), db = sw128_desc(su32(s.b[st]));
#pragma unroll
                for (int k = 0; k < BK / 32; k++)
                    mma_i8(tmem, da + 2 * k, db + 2 * k, idesc, (it > 0 || k > 0) ? 1u : 0u);
                mma_commit(&s.empty[st]);
            }
            if (ok)
                mma_commit(&s.acc_full);
        }
        __syncwarp();
        cluster_wait();
    }
    else {
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            const int id = me + THREADS * i, row = m0 + id / NQ;
            const int col = n0 + (rank * NQ + id % NQ) * 4;
            live[i] = id < NQ * ROWS && row < g.M && col < g.N;
            if (!live[i])
                continue;
            sa[i] = g.sa[row];
            load_quad(sb[i], g.sb + col, g.N - col, p.al);
            load_quad(bias[i], g.bias ? g.bias + col : nullptr, g.N - col, p.al);
            load_quad(res[i], g.R ? (const TC *)g.R + (long)row * g.ldc + col : nullptr,
                      g.N - col, p.al_r & 1);
        }
        const bool ok = __all_sync(0xffffffffu, mbar_wait(&s.acc_full, 0, 83));
        cluster_wait();
        const int q = warp % 4, r = 32 * q + lane;
        if (ok && m0 + 32 * q < g.M) {
            fence_after();
            const uint32_t acc = tmem + ((uint32_t)(32 * q) << 16);
            for (int c0 = 16 * ((warp - 2) / 4); c0 < BN; c0 += 16 * (EPI_WARPS / 4)) {
                float v[16];
                tmem_ld16(acc + c0, v);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int quad = c0 / 4 + k;
                    store_to(su32(s.part + (rank * NQ + quad % NQ) * QUAD + r * 16), quad / NQ,
                             v + 4 * k);
                }
            }
            fence_before();
        }
    }
    // The parts have arrived.
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (warp >= 2) {
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            if (!live[i])
                continue;
            const int id = me + THREADS * i, quad = id % NQ, r = id / NQ;
            const int row = m0 + r, col = n0 + (rank * NQ + quad) * 4;
            int4 sum = make_int4(0, 0, 0, 0);
#pragma unroll
            for (int from = 0; from < S; from++) {
                const int4 x = *(const int4 *)(s.part + (from * NQ + quad) * QUAD + r * 16);
                sum.x += x.x;
                sum.y += x.y;
                sum.z += x.z;
                sum.w += x.w;
            }
            // The token's scale first (see scaled() in linear_i8.cu).
            const float y[4] = {__int2float_rn(sum.x) * sa[i], __int2float_rn(sum.y) * sa[i],
                                __int2float_rn(sum.z) * sa[i], __int2float_rn(sum.w) * sa[i]};
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                const float2 x = act2_any(make_float2(fmaf(y[j], sb[i][j], bias[i][j]),
                                                      fmaf(y[j + 1], sb[i][j + 1], bias[i][j + 1])),
                                          g.act, g.slope);
                v[j] = g.R ? x.x + res[i][j] : x.x;
                v[j + 1] = g.R ? x.y + res[i][j + 1] : x.y;
            }
            store_quad((TC *)g.C + (long)row * g.ldc + col, v, g.N - col, p.al_r & 2);
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        tmem_dealloc(tmem, BN);
    }
}

// The kernel of an activation.
template <typename F>
bool with_act(int act, F f)
{
    switch (act) {
    case ACT_GELU:
        return f(std::integral_constant<int, ACT_GELU>());
    case ACT_RELU:
        return f(std::integral_constant<int, ACT_RELU>());
    case ACT_LEAKY:
        return f(std::integral_constant<int, ACT_LEAKY>());
    case ACT_GELU_TANH:
        return f(std::integral_constant<int, ACT_GELU_TANH>());
    case ACT_SILU:
        return f(std::integral_constant<int, ACT_SILU>());
    }
    return f(std::integral_constant<int, ACT_NONE>());
}

// Whether 256-wide tiles go to CTA pairs: for deep products (8192 x 8192 x
// 8192 417 us in pairs, 440 without; 25616 x 1024 x 4096 140 and 148; 3202 x
// 1024 x 4096 22.8 and 24.1). In shallow ones the epilogue leads, and a pair
// waits for the slower of its two (25616 x 4096 x 1024 139 and 132).
bool pair_pays(const I8Gemm &g) { return g.M > BM && g.K >= 2048; }

// PAIR: the kernel of CTA pairs (BN 256).
template <int BN, bool PAIR, typename TC>
bool launch(cudaStream_t st, const I8Gemm &g, int sms)
{
    CUtensorMap ma, mb, mc = {};
    Params p;
    p.g = g;
    if (!make_map_rows(&ma, g.A, 1, g.M, g.K, g.lda, BK, box_rows(g.M, BM), 128) ||
        !make_map_rows(&mb, g.B, 1, g.N, g.K, g.ldb, BK, PAIR ? BN / 2 : BN, 128))
        return false;
    p.tma_out = make_map_rows(&mc, g.C, sizeof(TC), g.M, g.N, g.ldc * (long)sizeof(TC),
                              ROW / (int)sizeof(TC), 32, 64);
    p.al = (((uintptr_t)g.sb | (uintptr_t)g.bias) & 15) == 0;
    p.al_r = ((uintptr_t)g.R & 15) == 0 && g.ldc * (long)sizeof(TC) % 16 == 0;
    p.clean = (long)g.N * (int)sizeof(TC) % 16 == 0;
    const long tiles = (long)cdiv(g.M, PAIR ? 2 * BM : BM) * cdiv(g.N, BN);
    if (tiles >= (1L << 31))
        return false;
    const long most = PAIR ? sms / 2 : sms;
    const unsigned grid = (unsigned)(tiles < most ? tiles : most) * (PAIR ? 2 : 1);
    return with_act(g.act, [&](auto act) {
        constexpr int ACT = decltype(act)::value;
        if constexpr (PAIR) {
            static unsigned done = 0;
            const size_t smem = sizeof(PairSmem) + 1024;
            if (!smem_opt_in((const void *)tc_i8_pair_k<ACT, TC>, smem, &done))
                return false;
            launch_chained(tc_i8_pair_k<ACT, TC>, grid, NTHREADS, smem, st, ma, mb, mc, p);
            return true;
        }
        else {
            auto go = [&](auto kernel, unsigned *done) {
                const size_t smem = sizeof(Smem<BN>) + 1024;
                if (!smem_opt_in((const void *)kernel, smem, done))
                    return false;
                launch_chained(kernel, grid, NTHREADS, smem, st, ma, mb, mc, p);
                return true;
            };
            static unsigned done[2] = {0, 0};
            return g.M < BM ? go(tc_i8_k<BN, ACT, true, TC>, &done[1])
                            : go(tc_i8_k<BN, ACT, false, TC>, &done[0]);
        }
    });
}

template <int BN, int ROWS, int S, typename TC>
bool launch_split(cudaStream_t st, const I8Gemm &g)
{
    CUtensorMap ma, mb;
    Params p = {};
    p.g = g;
    if (!make_map_rows(&ma, g.A, 1, g.M, g.K, g.lda, BK, box_rows(g.M, ROWS), 128) ||
        !make_map_rows(&mb, g.B, 1, g.N, g.K, g.ldb, BK, BN, 128))
        return false;
    p.al = (((uintptr_t)g.sb | (uintptr_t)g.bias) & 15) == 0;
    if (g.ldc * (long)sizeof(TC) % 16 == 0)
        p.al_r = (((uintptr_t)g.R & 15) == 0) | (((uintptr_t)g.C & 15) == 0) << 1;
    const size_t smem = sizeof(SplitSmem<BN, ROWS>) + 1024;
    static unsigned done = 0;
    if (!smem_opt_in((const void *)tc_i8_split_k<BN, ROWS, S, TC>, smem, &done))
        return false;
    launch_clusters(tc_i8_split_k<BN, ROWS, S, TC>, (unsigned)(cdiv(g.M, BM) * cdiv(g.N, BN) * S), S,
                    NTHREADS, smem, st, ma, mb, p);
    return true;
}

// Clusters of a split's kernel that run at one time.
template <int BN, int ROWS, int S, typename TC>
int split_clusters()
{
    static PerDevice known;
    return known.get([] {
        const size_t smem = sizeof(SplitSmem<BN, ROWS>) + 1024;
        const void *fn = (const void *)tc_i8_split_k<BN, ROWS, S, TC>;
        static unsigned done = 0;
        if (!smem_opt_in(fn, smem, &done))
            return 0;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(S);
        cfg.blockDim = dim3(NTHREADS);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = S;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        return n;
    });
}

template <typename TC>
struct Choice {
    const I8Gemm &g;
    bool (*run)(cudaStream_t, const I8Gemm &, int) = nullptr;
    double t = 0;

    void offer(double time, bool (*f)(cudaStream_t, const I8Gemm &, int))
    {
        if (!run || time < t) {
            t = time;
            run = f;
        }
    }
    // One round of clusters only: a second one starts after the first has ended, its
    // setup and fill unoverlapped (256 x 4096 x 4096 in halves 10.6 us, in
    // quarters, two rounds, 16.6).
    template <int BN, int ROWS, int S>
    void offer_split()
    {
        const int nk = cdiv(g.K, BK);
        if (nk < S || (g.M <= 32) != (ROWS == 32))
            return;
        const long tiles = (long)cdiv(g.M, BM) * cdiv(g.N, BN);
        const double cells = (double)(g.M < BM ? g.M : BM) * BN;
        const double epi = 1500.0 + 0.39 * cells;
        const double time = 600.0 * cdiv(nk, S) + 500.0 + (epi > 4400.0 ? epi : 4400.0);
        if (time < t && tiles <= split_clusters<BN, ROWS, S, TC>())
            offer(time, [](cudaStream_t st, const I8Gemm &p, int) {
                return launch_split<BN, ROWS, S, TC>(st, p);
            });
    }
    template <int BN>
    void offer_whole(int sms)
    {
        const long tiles = (long)cdiv(g.M, BM) * cdiv(g.N, BN), rounds = (tiles + sms - 1) / sms;
        const double main = 600.0 * cdiv(g.K, BK), epi = 1500.0 + 20.0 * BN;
        offer(rounds * ((main > epi ? main : epi) + 500.0) + epi,
              BN == 256 && pair_pays(g) ? launch<256, true, TC> : launch<BN, false, TC>);
    }
};

template <typename TC>
bool choose(cudaStream_t st, const I8Gemm &g, int sms)
{
    // The tiles that take the least time, in cycles: a round of tiles costs
    // its products or, where that is more, its epilogue, and the last
    // epilogue overlaps nothing. 128 bytes of depth take about 600 cycles at
    // any width: an MMA reads its 128 rows of A for 128 cycles, in which it
    // multiplies up to 256 columns (25616 x 4096 x 1024 in short runs: 125 us
    // with 256 columns, 144 with 128, 231 with 64; 500 x 500 x 500, where
    // rounds do not count: 13.5, 10.3 and 8.4). A split depth's epilogue is
    // longer: at 128 x 4096 x 1024 some 3.3 us with 128 columns, 1.7 with 64 and
    // at 32 rows, against 1.5 unsplit.
    Choice<TC> c{g};
    c.template offer_whole<256>(sms);
    c.template offer_whole<128>(sms);
    c.template offer_whole<64>(sms);
    c.template offer_split<128, 32, 2>();
    c.template offer_split<128, 32, 4>();
    c.template offer_split<128, 32, 8>();
    c.template offer_split<64, 128, 2>();
    c.template offer_split<64, 128, 4>();
    c.template offer_split<128, 128, 2>();
    c.template offer_split<128, 128, 4>();
    c.template offer_split<128, 128, 8>();
    return c.run(st, g, sms);
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
