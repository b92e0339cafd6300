// SPDX-License-Identifier: Unlicense
//
// 8-bit linear layers (ops_b200.h): ops_quant_i8, ops_gemm_i8 and
// ops_linear_i8.

#include <type_traits>

#include "linear_i8.cuh"

using namespace coreg;

namespace coreg {
namespace {

// ------------------------------------------------------------ quantisation

// A row's scale from the bits of its largest magnitude (an unsigned
// comparison orders finite < infinite < NaN) and its quotients.
//
// The nearest integer (ties to even) to the real quotient x / s: r = x (1 / s)
// rounded to an integer by adding and taking off 1.5 2^23 is off by at most
// one, and only next to a tie (r itself is off by less than 2^-15). x - q s is
// exact in one fused multiply-add: x and s are multiples of the smaller of
// their last places, and the difference is below s (in units of that place
// below 2^24). So |x - q s| against s / 2 decides, without a division, and
// the seldom values that it moves take a branch.
struct RowScale {
    float s, inv, half;
    __device__ explicit RowScale(uint32_t amax)
    {
        s = __int_as_float(0x7fffffff);
        inv = half = 0.0f;
        if (amax < 0x7f800000u) {
            s = __fdiv_rn(__uint_as_float(amax), 127.0f);
            // Below 2^-90 1 / s could overflow and s be denormal: slow().
            if (s >= 0x1p-90f) {
                inv = __fdiv_rn(1.0f, s);
                half = 0.5f * s;
            }
        }
    }
    // The quantised value as the low byte of the result; sure: whether it is.
    __device__ __forceinline__ uint32_t guess(float x, bool &sure) const
    {
        const float big = fmaf(x, inv, 12582912.0f);
        const float d = fmaf(12582912.0f - big, s, x);
        sure = sure && fabsf(d) < half;
        return __float_as_uint(big);
    }
    // Any value of any row: next to a tie, or of a scale that is not a normal
    // positive number.
    __device__ __noinline__ uint32_t slow(float x) const
    {
        if (!(s > 0.0f))
            return 0; // a row of zeros, or with an infinity or NaN
        // Small scales into the normal range by an exact power of two.
        const float k = s < 0x1p-90f ? 0x1p+90f : 1.0f, u = s * k;
        x *= k;
        float q = rintf(__fdiv_rn(x, u));
        const float d = fmaf(-q, u, x), e = fabsf(d + d);
        if (e > u || (e == u && ((int)q & 1)))
            q += copysignf(1.0f, d);
        return (uint32_t)(int)fminf(fmaxf(q, -127.0f), 127.0f);
    }
    __device__ __forceinline__ uint32_t of(float x) const
    {
        bool sure = true;
        const uint32_t q = guess(x, sure);
        return sure ? q : slow(x);
    }
};

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Four quantised values in a word.
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// 16 bytes of a row: V values, or one value where rows are not aligned.
template <typename T, int V>
struct Piece {
    uint4 w;
    __device__ __forceinline__ void load(const T *p) { w = *(const uint4 *)p; }
    __device__ __forceinline__ float at(int e) const
    {
        const int i = sizeof(T) == 4 ? e : e / 2;
        const uint32_t x = i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
        return __uint_as_float(sizeof(T) == 4 ? x : e % 2 ? x & 0xffff0000u : x << 16);
    }
    __device__ __forceinline__ uint32_t top() const
    {
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < V; e++)
            m = max(m, magnitude(at(e)));
        return m;
    }
    __device__ __forceinline__ void store(int8_t *q, const RowScale &s) const
    {
        uint32_t v[V];
        bool sure = true;
#pragma unroll
        for (int e = 0; e < V; e++)
            v[e] = s.guess(at(e), sure);
        if (!sure) {
#pragma unroll
            for (int e = 0; e < V; e++)
                v[e] = s.slow(at(e));
        }
        if constexpr (V == 4) {
            *(uint32_t *)q = pack4(v[0], v[1], v[2], v[3]);
        }
        else {
            *(uint2 *)q = make_uint2(pack4(v[0], v[1], v[2], v[3]), pack4(v[4], v[5], v[6], v[7]));
        }
    }
};

template <typename T>
struct Piece<T, 1> {
    float f;
    __device__ __forceinline__ void load(const T *p) { f = ldf(p); }
    __device__ __forceinline__ uint32_t top() const { return magnitude(f); }
    __device__ __forceinline__ void store(int8_t *q, const RowScale &s) const
    {
        *q = (int8_t)s.of(f);
    }
};

// G threads of a block of 256 per row, its pieces in their registers (NP a
// thread) from the maximum to the result, so that a row is read once; longer
// rows read what is beyond again. Values behind the last whole piece one by
// one.
template <typename T, int V, int G, int NP>
__global__ void __launch_bounds__(256)
quant_k(const T *X, long ldx, long rows, int C, int8_t *Q, long ldq, float *S)
{
    __shared__ uint32_t red[8];
    after_previous();
    const int lane = threadIdx.x % G;
    const long row = (long)blockIdx.x * (256 / G) + threadIdx.x / G;
    const bool here = row < rows;
    const T *x = X + (here ? row : 0) * ldx;
    const int n = here ? C / V : 0; // whole pieces
    Piece<T, V> r[NP];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < NP; i++)
        if (lane + i * G < n)
            r[i].load(x + (long)(lane + i * G) * V);
#pragma unroll
    for (int i = 0; i < NP; i++)
        if (lane + i * G < n)
            m = max(m, r[i].top());
    for (int k = lane + NP * G; k < n; k += G) {
        Piece<T, V> f;
        f.load(x + (long)k * V);
        m = max(m, f.top());
    }
    const int c = n * V + lane; // its value behind the pieces (C % V < G)
    const bool odd = here && c < C;
    float f = 0.0f;
    if (odd) {
        f = ldf(x + c);
        m = max(m, magnitude(f));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (G > 32) {
        if (threadIdx.x % 32 == 0)
            red[threadIdx.x / 32] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < G / 32; w++)
            m = max(m, red[threadIdx.x / G * (G / 32) + w]);
    }
    if (!here)
        return;
    const RowScale s(m);
    if (lane == 0)
        S[row] = s.s;
    int8_t *q = Q + row * ldq;
#pragma unroll
    for (int i = 0; i < NP; i++)
        if (lane + i * G < n)
            r[i].store(q + (long)(lane + i * G) * V, s);
    for (int k = lane + NP * G; k < n; k += G) {
        Piece<T, V> f2;
        f2.load(x + (long)k * V);
        f2.store(q + (long)k * V, s);
    }
    if (odd)
        q[c] = (int8_t)s.of(f);
}

template <typename T, int V>
void quant_launch(cudaStream_t st, const View &x, int8_t *q, long ldq, float *s)
{
    // A warp per row up to 8 pieces a lane (no barrier of the block), then a
    // block.
    const int pieces = (int)(x.cols / V);
    auto go = [&](auto g, auto np) {
        constexpr int G = decltype(g)::value, NP = decltype(np)::value;
        launch_chained(quant_k<T, V, G, NP>, cdiv(x.rows, 256 / G), 256, 0, st, (const T *)x.p, x.ld,
                       x.rows, (int)x.cols, q, ldq, s);
    };
    typedef std::integral_constant<int, 4> four;
    typedef std::integral_constant<int, 8> eight;
    typedef std::integral_constant<int, 32> warp;
    typedef std::integral_constant<int, 256> block;
    if (pieces <= 32 * 4)
        go(warp(), four());
    else if (pieces <= 32 * 8)
        go(warp(), eight());
    else if (pieces <= 256 * 4)
        go(block(), four());
    else
        go(block(), eight());
}

void quant_rows(cudaStream_t st, const View &x, int xtype, int8_t *q, long ldq, float *s)
{
    const int V = xtype == OPS_BF16 ? 8 : 4;
    const bool al = ((uintptr_t)x.p & 15) == 0 && (x.rows == 1 || x.ld % V == 0) &&
                    (uintptr_t)q % V == 0 && (x.rows == 1 || ldq % V == 0);
    if (xtype == OPS_BF16 && al)
        quant_launch<__nv_bfloat16, 8>(st, x, q, ldq, s);
    else if (xtype == OPS_BF16)
        quant_launch<__nv_bfloat16, 1>(st, x, q, ldq, s);
    else if (al)
        quant_launch<float, 4>(st, x, q, ldq, s);
    else
        quant_launch<float, 1>(st, x, q, ldq, s);
}

// ----------------------------------------------------------------- product

// A sum as a value before the activation. (The token's scale first: the two
// scales' own product could pass the type's range where the result does not.)
__device__ __forceinline__ float scaled(int acc, float sa, float sb, float bias)
{
    return fmaf(__int2float_rn(acc) * sa, sb, bias);
}

// 64 x 64 output tiles, 4 x 4 sums per thread, 64 bytes of depth staged at a
// time; four products per __dp4a.
template <typename TC>
__global__ void __launch_bounds__(256)
i8_tile_k(const I8Gemm g)
{
    __shared__ uint32_t a[64][17], b[64][17];
    const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < g.K; k0 += 64) {
        for (int i = threadIdx.x; i < 64 * 64; i += 256) {
            const int r = i / 64, k = i % 64;
            const bool in = k0 + k < g.K;
            ((int8_t *)a[r])[k] =
                in && m0 + r < g.M ? g.A[(long)(m0 + r) * g.lda + k0 + k] : (int8_t)0;
            ((int8_t *)b[r])[k] =
                in && n0 + r < g.N ? g.B[(long)(n0 + r) * g.ldb + k0 + k] : (int8_t)0;
        }
        __syncthreads();
        for (int k = 0; k < 16; k++)
            for (int i = 0; i < 4; i++)
                for (int j = 0; j < 4; j++)
                    acc[i][j] = __dp4a((int)a[ty + 16 * i][k], (int)b[tx + 16 * j][k], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const int r = m0 + ty + 16 * i, c = n0 + tx + 16 * j;
            if (r >= g.M || c >= g.N)
                continue;
            float v = scaled(acc[i][j], g.sa[r], g.sb[c], g.bias ? g.bias[c] : 0.0f);
            v = act_any(v, g.act, g.slope);
            if (g.R)
                v += ldf((const TC *)g.R + (long)r * g.ldc + c);
            stf((TC *)g.C + (long)r * g.ldc + c, v);
        }
}

// Few rows: the weights stream once from memory, so a block takes 16 of
// their rows (output channels), its 8 warps the depth by turns of 64 bytes.
// mma.m16n8k32 of 8-bit integers with the weights as the 16 rows and 8 tokens
// as the columns: lane l's operands are four words of channel (or token) l /
// 4, and as the order of the depth is free as long as both operands agree,
// they are one 16-byte load at 16 (l % 4) of the turn. The warps' sums meet
// in shared memory.
constexpr int SK_CH = 16, SK_WARPS = 8, SK_TURN = 64;

__device__ __forceinline__ void mma_s8(int d[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                       uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of a row from depth k on, zeros behind K: the bytes there need not
// exist.
__device__ __forceinline__ uint4 load16(const int8_t *row, int k, int K)
{
    if (k + 16 <= K)
        return *(const uint4 *)(row + k);
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (k + i < K)
            w[i / 4] |= (uint32_t)(uint8_t)row[k + i] << (8 * (i % 4));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// NT: groups of 8 tokens.
template <int NT, typename TC>
__global__ void __launch_bounds__(32 * SK_WARPS)
i8_skinny_k(const I8Gemm g)
{
    __shared__ int part[SK_WARPS][SK_CH][8 * NT + 1];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, n0 = blockIdx.x * SK_CH;
    const int r = lane / 4, kk = 16 * (lane % 4);
    const int8_t *w0 = g.B + (long)min(n0 + r, g.N - 1) * g.ldb;
    const int8_t *w1 = g.B + (long)min(n0 + r + 8, g.N - 1) * g.ldb;
    int d[NT][4] = {};
    after_previous();
    constexpr int U = NT == 4 ? 2 : 4, STEP = SK_WARPS * SK_TURN;
    for (int k0 = warp * SK_TURN + kk; k0 < g.K + kk; k0 += U * STEP) {
        uint4 a[U], b[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            a[u] = load16(w0, k0 + u * STEP, g.K);
            b[u] = load16(w1, k0 + u * STEP, g.K);
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const int m = 8 * t + r;
                const uint4 x = m < g.M ? load16(g.A + (long)m * g.lda, k0 + u * STEP, g.K)
                                        : make_uint4(0, 0, 0, 0);
                mma_s8(d[t], a[u].x, b[u].x, a[u].y, b[u].y, x.x, x.y);
                mma_s8(d[t], a[u].z, b[u].z, a[u].w, b[u].w, x.z, x.w);
            }
    }
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            part[warp][r + 8 * (i / 2)][8 * t + 2 * (lane % 4) + i % 2] = d[t][i];
    __syncthreads();
    for (int e = threadIdx.x; e < SK_CH * g.M; e += 32 * SK_WARPS) {
        const int c = e % SK_CH, m = e / SK_CH;
        if (n0 + c >= g.N)
            continue;
        int acc = 0;
#pragma unroll
        for (int w = 0; w < SK_WARPS; w++)
            acc += part[w][c][m];
        float v = scaled(acc, g.sa[m], g.sb[n0 + c], g.bias ? g.bias[n0 + c] : 0.0f);
        v = act_any(v, g.act, g.slope);
        const long at = (long)m * g.ldc + n0 + c;
        if (g.R)
            v += ldf((const TC *)g.R + at);
        stf((TC *)g.C + at, v);
    }
}

template <typename TC>
void skinny(cudaStream_t st, const I8Gemm &g)
{
    const unsigned grid = cdiv(g.N, SK_CH);
    if (g.M <= 8)
        launch_chained(i8_skinny_k<1, TC>, grid, 32 * SK_WARPS, 0, st, g);
    else if (g.M <= 16)
        launch_chained(i8_skinny_k<2, TC>, grid, 32 * SK_WARPS, 0, st, g);
    else
        launch_chained(i8_skinny_k<4, TC>, grid, 32 * SK_WARPS, 0, st, g);
}

constexpr int SKINNY_ROWS = 32;

void gemm_i8(const struct ocl_backend *ocl, const I8Gemm &g)
{
    cudaStream_t st = stream_of(ocl);
    if (g.M <= SKINNY_ROWS) {
        if (g.c_bf16)
            skinny<__nv_bfloat16>(st, g);
        else
            skinny<float>(st, g);
        return;
    }
    if (g.K > 0 && gemm_i8_tc(st, g, sms_of(ocl)))
        return;
    const dim3 grid(cdiv(g.N, 64), cdiv(g.M, 64));
    if (g.c_bf16)
        i8_tile_k<__nv_bfloat16><<<grid, 256, 0, st>>>(g);
    else
        i8_tile_k<float><<<grid, 256, 0, st>>>(g);
}

// -------------------------------------------------------------- arguments

// An int8 operand of the product: rows 16-byte aligned.
bool i8_view(View *v, const char *fn, const char *what, const struct opnd &m, long rows, long K)
{
    if (!view_of(v, fn, what, m.buf, m.off, m.ld, rows, K, 1))
        return false;
    if (((uintptr_t)v->p & 15) || (rows > 1 && m.ld % 16)) {
        fail("%s: %s (offset %ld, leading dimension %d) has rows that are not 16-byte aligned "
             "(ops_i8_ld)",
             fn, what, (long)m.off, m.ld);
        return false;
    }
    return true;
}

// The operands that ops_gemm_i8 and ops_linear_i8 share: the weights, their
// scales, bias, output and residual.
bool product_args(const char *fn, I8Gemm *g, int M, int N, int K, const struct opnd &B, cl_mem sb,
                  cl_mem bias, const struct opnd &C, int ctype, cl_mem R, long roff, int act,
                  float slope, View *out, View in[4], int *nin)
{
    View r;
    if (M < 0 || N < 0 || K < 0 || K > OPS_I8_MAX_K) {
        fail("%s: %d x %d x %d (depth 0..%d)", fn, M, N, K, OPS_I8_MAX_K);
        return false;
    }
    if (!type_ok(fn, ctype) || !act_ok(fn, act))
        return false;
    const int es = type_size(ctype);
    *nin = 0;
    if (!i8_view(&in[*nin], fn, "B", B, N, K))
        return false;
    g->B = (const int8_t *)in[(*nin)++].p;
    if (!view_of(&in[*nin], fn, "the scales of B", sb, 0, N, 1, N, 4))
        return false;
    g->sb = (const float *)in[(*nin)++].p;
    if (bias) {
        if (!view_of(&in[*nin], fn, "the bias", bias, 0, N, 1, N, 4))
            return false;
        g->bias = (const float *)in[(*nin)++].p;
    }
    else
        g->bias = nullptr;
    if (!view_of(out, fn, "C", C.buf, C.off, C.ld, M, N, es))
        return false;
    g->R = nullptr;
    if (R) {
        if (!view_of(&r, fn, "R", R, roff, C.ld, M, N, es))
            return false;
        if (!same_view(r, *out) && views_meet(r, *out)) {
            fail("%s: R and C overlap and are not the same", fn);
            return false;
        }
        g->R = r.p;
    }
    g->M = M;
    g->N = N;
    g->K = K;
    g->ldb = B.ld;
    g->C = out->p;
    g->ldc = C.ld;
    g->c_bf16 = ctype == OPS_BF16;
    g->act = act;
    g->slope = slope;
    return true;
}

bool apart(const char *fn, const View &out, const View *in, int n)
{
    for (int i = 0; i < n; i++)
        if (views_meet(out, in[i])) {
            fail("%s: the output overlaps an input", fn);
            return false;
        }
    return true;
}

}  // namespace
}  // namespace coreg

extern "C" int ops_i8_ld(int K) { return K > 0x7ffffff0 ? 0x7ffffff0 : (K + 15) / 16 * 16; }

extern "C" void ops_quant_i8(struct ops *o, long rows, int C, struct opnd X, int xtype,
                             struct opnd Q, cl_mem S, long soff)
{
    const char *fn = "ops_quant_i8";
    View in, out[2];

    if (pending() || !type_ok(fn, xtype) ||
        !view_of(&in, fn, "X", X.buf, X.off, X.ld, rows, C, type_size(xtype)) ||
        !view_of(&out[0], fn, "Q", Q.buf, Q.off, Q.ld, rows, C, 1) ||
        !view_of(&out[1], fn, "S", S, soff, 1, rows, 1, 4) || !count_ok(rows, "rows of int8"))
        return;
    if (!apart(fn, out[0], &in, 1) || !apart(fn, out[1], &in, 1) || !apart(fn, out[0], out + 1, 1))
        return;
    if (rows == 0 || C == 0)
        return;
    OnDevice dev(o->ocl);
    if (!dev.ok)
        return;
    Prof p(o->ocl, "quant_i8");
    quant_rows(stream_of(o->ocl), in, xtype, (int8_t *)out[0].p, Q.ld, (float *)out[1].p);
    launch_ok("quant_i8");
}

extern "C" void ops_gemm_i8(struct ops *o, int M, int N, int K, struct opnd A, cl_mem sa,
                            struct opnd B, cl_mem sb, cl_mem bias, struct opnd C, int ctype,
                            cl_mem R, long roff, int act, float slope)
{
    const char *fn = "ops_gemm_i8";
    I8Gemm g;
    View in[6], out;
    int n = 0;

    if (pending() || !product_args(fn, &g, M, N, K, B, sb, bias, C, ctype, R, roff, act, slope,
                                   &out, in, &n))
        return;
    if (!i8_view(&in[n], fn, "A", A, M, K) ||
        !view_of(&in[n + 1], fn, "the scales of A", sa, 0, M, 1, M, 4) ||
        !apart(fn, out, in, n + 2))
        return;
    if (M == 0 || N == 0)
        return;
    g.A = (const int8_t *)in[n].p;
    g.lda = A.ld;
    g.sa = (const float *)in[n + 1].p;
    OnDevice dev(o->ocl);
    if (!dev.ok)
        return;
    Prof p(o->ocl, "gemm_i8");
    gemm_i8(o->ocl, g);
    launch_ok("gemm_i8");
}

// The work buffer holds the rows' scales, then their 8-bit values.
static size_t work_scales(int rows) { return ((size_t)rows * 4 + 15) / 16 * 16; }

extern "C" size_t ops_linear_i8_bytes(int rows, int in)
{
    return rows <= 0 || in < 0 ? 0 : work_scales(rows) + (size_t)rows * ops_i8_ld(in);
}

extern "C" void ops_linear_i8(struct ops *o, int rows, int in, int out, struct opnd X, int xtype,
                              struct opnd W, cl_mem sw, cl_mem bias, struct opnd Y, int ytype,
                              cl_mem R, long roff, int act, float slope, cl_mem work)
{
    const char *fn = "ops_linear_i8";
    I8Gemm g;
    View v[6], y, ws;
    int n = 0;

    if (pending() || !type_ok(fn, xtype) ||
        !product_args(fn, &g, rows, out, in, W, sw, bias, Y, ytype, R, roff, act, slope, &y, v,
                      &n) ||
        !view_of(&v[n], fn, "X", X.buf, X.off, X.ld, rows, in, type_size(xtype)))
        return;
    const View x = v[n++];
    if (!apart(fn, y, v, n) || rows == 0 || out == 0)
        return;
    const size_t bytes = ops_linear_i8_bytes(rows, in);
    if (bytes) {
        if (!view_of(&ws, fn, "the work buffer", work, 0, (long)bytes, 1, (long)bytes, 1))
            return;
        if ((uintptr_t)ws.p & 15) {
            fail("%s: the work buffer is not 16-byte aligned", fn);
            return;
        }
        if (!apart(fn, ws, v, n) || !apart(fn, y, &ws, 1))
            return;
    }
    OnDevice dev(o->ocl);
    if (!dev.ok)
        return;
    cudaStream_t st = stream_of(o->ocl);
    int8_t *q = (int8_t *)ws.p + work_scales(rows);
    Prof p(o->ocl, "linear_i8");
    quant_rows(st, x, xtype, q, ops_i8_ld(in), (float *)ws.p);
    g.A = q;
    g.lda = ops_i8_ld(in);
    g.sa = (const float *)ws.p;
    gemm_i8(o->ocl, g);
    launch_ok("linear_i8");
}
