// SPDX-License-Identifier: Unlicense
//
// 8-bit linear layers (ops_b200.h): ops_quant_i8, ops_gemm_i8 and
// ops_linear_i8.

#include <type_traits>

#include "opcheck.cuh"

using namespace coreg;

namespace coreg {
namespace {

// ------------------------------------------------------------ quantisation

// The nearest integer (ties to even) to the real quotient x / s, |x| <= 127 s
// up to a rounding of s. r = x (1 / s) is off by less than 2^-15, so its
// nearest integer q is off by at most one, and only next to a tie. x - q s is
// exact in one fused multiply-add: x and s are multiples of the smaller of
// their last places, and the difference is below s (in units of that place
// below 2^24). So |2 (x - q s)| against s decides, without a division.
__device__ __forceinline__ int nearest_quotient(float x, float s, float inv)
{
    float q = rintf(x * inv);
    const float d = fmaf(-q, s, x), e = fabsf(d + d);
    if (e > s || (e == s && ((int)q & 1)))
        q += copysignf(1.0f, d);
    return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

// A row's scale from the bits of its largest magnitude (an unsigned
// comparison orders finite < infinite < NaN), and what its quotients take:
// scales below 2^-90, whose reciprocal could overflow, go with their values
// into the normal range by an exact power of two.
struct RowScale {
    float s, up, s_up, inv;
    __device__ explicit RowScale(uint32_t amax)
    {
        if (amax >= 0x7f800000u) {
            s = __int_as_float(0x7fffffff);
            up = s_up = inv = 0.0f;
            return;
        }
        s = __fdiv_rn(__uint_as_float(amax), 127.0f);
        up = s < 0x1p-90f ? 0x1p+90f : 1.0f;
        s_up = s * up;
        inv = s > 0.0f ? __fdiv_rn(1.0f, s_up) : 0.0f;
    }
    // The quantised value; 0 in rows without a positive finite scale.
    __device__ int of(float x) const
    {
        return inv > 0.0f ? nearest_quotient(x * up, s_up, inv) : 0;
    }
};

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// One block per row, two passes over it.
template <typename T>
__global__ void __launch_bounds__(256)
quant_row_k(const T *X, long ldx, int C, int8_t *Q, long ldq, float *S)
{
    __shared__ uint32_t red[8];
    const long row = blockIdx.x;
    const T *x = X + row * ldx;
    uint32_t m = 0;
    for (int c = threadIdx.x; c < C; c += blockDim.x)
        m = max(m, magnitude(ldf(x + c)));
    m = __reduce_max_sync(0xffffffffu, m);
    if (threadIdx.x % 32 == 0)
        red[threadIdx.x / 32] = m;
    __syncthreads();
    for (int w = 0; w < 8; w++)
        m = max(m, red[w]);
    const RowScale rs(m);
    if (threadIdx.x == 0)
        S[row] = rs.s;
    for (int c = threadIdx.x; c < C; c += blockDim.x)
        Q[row * ldq + c] = (int8_t)rs.of(ldf(x + c));
}

void quant_rows(cudaStream_t st, const View &x, int xtype, int8_t *q, long ldq, float *s)
{
    if (xtype == OPS_BF16)
        quant_row_k<<<(unsigned)x.rows, 256, 0, st>>>((const __nv_bfloat16 *)x.p, x.ld,
                                                      (int)x.cols, q, ldq, s);
    else
        quant_row_k<<<(unsigned)x.rows, 256, 0, st>>>((const float *)x.p, x.ld, (int)x.cols, q,
                                                      ldq, s);
}

// ----------------------------------------------------------------- product

struct I8Gemm {
    int M, N, K;
    const int8_t *A;
    long lda;
    const float *sa;
    const int8_t *B;
    long ldb;
    const float *sb;
    const float *bias; // per column or NULL
    void *C;
    long ldc;
    const void *R; // C's layout and type, or NULL
    int c_bf16;
    int act;
    float slope;
};

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
            float v = __int2float_rn(acc[i][j]) * g.sa[r] * g.sb[c] + (g.bias ? g.bias[c] : 0.0f);
            v = act_any(v, g.act, g.slope);
            if (g.R)
                v += ldf((const TC *)g.R + (long)r * g.ldc + c);
            stf((TC *)g.C + (long)r * g.ldc + c, v);
        }
}

void gemm_i8(cudaStream_t st, const I8Gemm &g)
{
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
    gemm_i8(stream_of(o->ocl), g);
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
    gemm_i8(st, g);
    launch_ok("linear_i8");
}
