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
// pieces with a value that it may move take a branch (1 in 10 of random
// tokens; of bfloat16 rows whose largest value is 127 2^n, half are ties).
struct RowScale {
    float s, inv, half;
    __device__ explicit RowScale(uint32_t amax)
    {
        s = __int_as_float(0x7fffffff);
        inv = half = 0.0f;
        if (amax < 0x7f800000u) {
            s = __fdiv_rn(__uint_as_float(amax), 127.0f);
            // Below 2^-90 1 / s could overflow and s be denormal: quotient().
            if (s >= 0x1p-90f) {
                inv = __fdiv_rn(1.0f, s);
                half = 0.5f * s;
            }
            else if (amax == 0) {
                half = 1.0f; // every value of a row of zeros is sure to be 0
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
    // The value for a guess g of x that was not sure, in a row with inv > 0.
    __device__ __forceinline__ uint32_t settle(uint32_t g, float x) const
    {
        const float d = fmaf(12582912.0f - __uint_as_float(g), s, x), e = fabsf(d);
        if (e > half || (e == half && (g & 1)))
            g += d > 0.0f ? 1u : ~0u;
        return g;
    }
    __device__ __forceinline__ uint32_t of(float x) const
    {
        bool sure = true;
        const uint32_t q = guess(x, sure);
        return sure ? q : quotient(x, s);
    }
    // Any value of any row.
    static __device__ __noinline__ uint32_t quotient(float x, float s)
    {
        if (!(s > 0.0f))
            return 0; // a scale of 0, or a row with an infinity or NaN
        // Small scales into the normal range by an exact power of two.
        const float k = s < 0x1p-90f ? 0x1p+90f : 1.0f, u = s * k;
        x *= k;
        float q = rintf(__fdiv_rn(x, u));
        const float d = fmaf(-q, u, x), e = fabsf(d + d);
        if (e > u || (e == u && ((int)q & 1)))
            q += copysignf(1.0f, d);
        return (uint32_t)(int)fminf(fmaxf(q, -127.0f), 127.0f);
    }
};

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Four quantised values in a word.
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// 16 bytes of a row: V values; two values or one where rows are not aligned.
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
    // Bits of the largest magnitude, as a float's.
    __device__ __forceinline__ uint32_t top() const
    {
        if constexpr (sizeof(T) == 4) {
            return max(max(magnitude(at(0)), magnitude(at(1))),
                       max(magnitude(at(2)), magnitude(at(3))));
        }
        else {
            // Two at a time: bfloat16 orders as float does.
            const uint32_t k = 0x7fff7fffu;
            const uint32_t m = __vmaxu2(__vmaxu2(w.x & k, w.y & k), __vmaxu2(w.z & k, w.w & k));
            return max(m << 16, m & 0xffff0000u);
        }
    }
    __device__ __forceinline__ void store(int8_t *q, const RowScale &s) const
    {
        uint32_t v[V];
        bool sure = true;
#pragma unroll
        for (int e = 0; e < V; e++)
            v[e] = s.guess(at(e), sure);
        if (!sure) {
            if (!(s.inv > 0.0f)) {
                store_slow(w, q, s.s);
                return;
            }
#pragma unroll
            for (int e = 0; e < V; e++)
                v[e] = s.settle(v[e], at(e));
        }
        if constexpr (V == 4)
            *(uint32_t *)q = pack4(v[0], v[1], v[2], v[3]);
        else
            *(uint2 *)q = make_uint2(pack4(v[0], v[1], v[2], v[3]), pack4(v[4], v[5], v[6], v[7]));
    }
    // (Rows of denormal scales, infinities or NaN.)
    static __device__ __noinline__ void store_slow(uint4 w, int8_t *q, float s)
    {
        Piece<T, V> p;
        p.w = w;
#pragma unroll 1
        for (int e = 0; e < V; e++) {
            const float x = p.at(0);
            q[e] = (int8_t)RowScale::quotient(x, s);
            // The next value to the front.
            if (sizeof(T) == 4 || e % 2)
                p.w = make_uint4(p.w.y, p.w.z, p.w.w, 0);
            else
                p.w.x >>= 16;
        }
    }
};

template <typename T>
struct Piece<T, 2> {
    float a, b;
    __device__ __forceinline__ void load(const T *p)
    {
        if constexpr (sizeof(T) == 4) {
            const float2 x = *(const float2 *)p;
            a = x.x, b = x.y;
        }
        else {
            const uint32_t x = *(const uint32_t *)p;
            a = __uint_as_float(x << 16), b = __uint_as_float(x & 0xffff0000u);
        }
    }
    __device__ __forceinline__ uint32_t top() const { return max(magnitude(a), magnitude(b)); }
    __device__ __forceinline__ void store(int8_t *q, const RowScale &s) const
    {
        bool sure = true;
        uint32_t x = s.guess(a, sure), y = s.guess(b, sure);
        if (!sure) {
            if (s.inv > 0.0f) {
                x = s.settle(x, a), y = s.settle(y, b);
            }
            else {
                x = RowScale::quotient(a, s.s), y = RowScale::quotient(b, s.s);
            }
        }
        *(uint16_t *)q = (uint16_t)__byte_perm(x, y, 0x0040);
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
    // A warp per row up to 8 pieces a lane, or 32 of one or two values (no barrier
    // of the block), then a block. (us, a block from 8 on and this: 10923 x 397
    // bfloat16, one value a piece, 16.3 and 7.9, 18142 x 812, two, 28.9 and 17.0.
    // Two values where rows allow it: 15088 x 3758 bfloat16 105 -> 54.)
    const int pieces = (int)(x.cols / V);
    auto go = [&](auto g, auto np) {
        constexpr int G = decltype(g)::value, NP = decltype(np)::value;
        launch_chained(quant_k<T, V, G, NP>, cdiv(x.rows, 256 / G), 256, 0, st, (const T *)x.p, x.ld,
                       x.rows, (int)x.cols, q, ldq, s);
    };
    typedef std::integral_constant<int, 4> four;
    typedef std::integral_constant<int, 8> eight;
    typedef std::integral_constant<int, 16> sixteen;
    typedef std::integral_constant<int, 32> thirty_two;
    typedef std::integral_constant<int, 32> warp;
    typedef std::integral_constant<int, 256> block;
    if (pieces <= 32 * 4)
        go(warp(), four());
    else if (pieces <= 32 * 8)
        go(warp(), eight());
    else if (V <= 2 && pieces <= 32 * 16)
        go(warp(), sixteen());
    else if (V <= 2 && pieces <= 32 * 32)
        go(warp(), thirty_two());
    else if (pieces <= 256 * 4)
        go(block(), four());
    else if (V <= 2 && pieces > 256 * 8 && pieces <= 256 * 16)
        go(block(), sixteen());
    else
        go(block(), eight());
}

void quant_rows(cudaStream_t st, const View &x, int xtype, int8_t *q, long ldq, float *s)
{
    const int es = type_size(xtype);
    auto al = [&](int v) {
        return (uintptr_t)x.p % (v * es) == 0 && (uintptr_t)q % v == 0 &&
               (x.rows == 1 || (x.ld % v == 0 && ldq % v == 0));
    };
    if (xtype == OPS_BF16) {
        if (al(8))
            quant_launch<__nv_bfloat16, 8>(st, x, q, ldq, s);
        else if (al(2))
            quant_launch<__nv_bfloat16, 2>(st, x, q, ldq, s);
        else
            quant_launch<__nv_bfloat16, 1>(st, x, q, ldq, s);
    }
    else if (al(4))
        quant_launch<float, 4>(st, x, q, ldq, s);
    else if (al(2))
        quant_launch<float, 2>(st, x, q, ldq, s);
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

// Products of depth 0: act(bias) + R. (Nothing wrote the scales of rows without
// columns: they may hold anything.)
template <typename TC>
__global__ void __launch_bounds__(256)
i8_empty_k(const I8Gemm g)
{
    after_previous();
    const long n = (long)g.M * g.N;
    for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < n; e += (long)gridDim.x * 256) {
        const long m = e / g.N, c = e - m * g.N, at = m * g.ldc + c;
        float v = act_any(g.bias ? g.bias[c] : 0.0f, g.act, g.slope);
        if (g.R)
            v += ldf((const TC *)g.R + at);
        stf((TC *)g.C + at, v);
    }
}

// Few tokens: the weights stream once from memory. A warp takes 16 of their
// rows (output channels) in steps of 64 bytes of depth; for deep and narrow
// layers `split` warps share a row's depth. The products go through
// mma.m16n8k16 of float16 with the weights as the 16 rows and 8 tokens as the
// columns: 8-bit integers are exact in float16, their products and sums of
// 256 of them (at most 2^22) in float32, and are added up as integers from
// there. Lane l's operands are those of channel (or token) l / 4, and as the
// order of the depth is free as long as both operands agree, they are one
// 16-byte load at 16 (l % 4) of the step. (The integer forms are slow here:
// mma.sync of 8-bit integers took 150 cycles and more, __dp4a runs at 8 per
// cycle and multiprocessor; 8192 x 8192 with 8 tokens 63 us with it.)
constexpr int FEW_WARPS = 8, FEW_CH = 16, FEW_STEP = 64;

__device__ __forceinline__ void mma_f16(float d[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four 8-bit integers as float16 pairs: x + 128 as the low byte of 1024 (0x6400)
// is 1152 + x, from which 1152 is taken off.
__device__ __forceinline__ void halves(uint32_t w, uint32_t &lo, uint32_t &hi)
{
    w ^= 0x80808080u;
    lo = __byte_perm(w, 0x64646464u, 0x4140);
    hi = __byte_perm(w, 0x64646464u, 0x4342);
    asm("sub.f16x2 %0, %0, %1;" : "+r"(lo) : "r"(0x64806480u));
    asm("sub.f16x2 %0, %0, %1;" : "+r"(hi) : "r"(0x64806480u));
}

// 16 bytes of a row from depth k on, zeros behind K: the bytes there need not
// exist.
__device__ __noinline__ uint4 load_end(const int8_t *p, int n)
{
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (i < n)
            w[i / 4] |= (uint32_t)(uint8_t)p[i] << (8 * (i % 4));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint4 load16(const int8_t *row, int k, int K)
{
    uint4 v = make_uint4(0, 0, 0, 0);
    if (k + 16 <= K)
        v = *(const uint4 *)(row + k);
    else if (k < K)
        v = load_end(row + k, K - k);
    return v;
}

// Tokens that the kernel quantises itself (ops_linear_i8): each block all of
// them, into shared memory, while its first weights are on their way.
struct Tokens {
    const void *X;
    long ldx;
    int pitch; // bytes of a quantised row
};

int token_pitch(int K) { return (K + 15) / 16 * 16; }

// The M rows of x quantised as by ops_quant_i8 into q, scales into s; amax: M
// words, zero. Ends with a barrier.
template <typename T>
__device__ void quant_tokens(const Tokens &x, int M, int K, int8_t *q, float *s, uint32_t *amax)
{
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    // Warps of a row: 8 of one, 4 of two, 2 of four, then a warp per row.
    const int per = M == 1 ? 8 : M == 2 ? 4 : M <= 4 ? 2 : 1, sub = warp % per;
    const int V = 16 / (int)sizeof(T);
    const bool al = ((uintptr_t)x.X & 15) == 0 && (M == 1 || x.ldx % V == 0);
    const int whole = al ? K / V * V : 0; // columns taken V at a time
    for (int r = warp / per; r < M; r += FEW_WARPS / per) {
        const T *p = (const T *)x.X + r * x.ldx;
        uint32_t m = 0;
        for (int c = (sub * 32 + lane) * V; c < whole; c += per * 32 * V) {
            Piece<T, V> f;
            f.load(p + c);
            m = max(m, f.top());
        }
        for (int c = whole + sub * 32 + lane; c < K; c += per * 32)
            m = max(m, magnitude(ldf(p + c)));
        m = __reduce_max_sync(0xffffffffu, m);
        if (lane == 0)
            atomicMax(&amax[r], m); // (the largest, in whatever order)
    }
    __syncthreads();
    for (int r = warp / per; r < M; r += FEW_WARPS / per) {
        const T *p = (const T *)x.X + r * x.ldx;
        int8_t *to = q + r * x.pitch;
        const RowScale rs(amax[r]);
        if (sub == 0 && lane == 0)
            s[r] = rs.s;
        for (int c = (sub * 32 + lane) * V; c < whole; c += per * 32 * V) {
            Piece<T, V> f;
            f.load(p + c);
            f.store(to + c, rs);
        }
        // One by one, with zeros up to the end of the pitch.
        for (int c = whole + sub * 32 + lane; c < x.pitch; c += per * 32)
            to[c] = c < K ? (int8_t)rs.of(ldf(p + c)) : (int8_t)0;
    }
    __syncthreads();
}

// TX: the type of tokens that come unquantised (the
// struct x; then g.A and g.sa are not used), or void.
template <typename TC, typename TX>
__global__ void __launch_bounds__(32 * FEW_WARPS)
i8_few_k(const I8Gemm g, const Tokens x, int split)
{
    constexpr bool FLOATS = !std::is_same<TX, void>::value;
    constexpr int THREADS = 32 * FEW_WARPS;
    __shared__ int part[FEW_WARPS][FEW_CH][8 + 1];
    __shared__ float scale[8];
    __shared__ uint32_t amax[8];
    extern __shared__ __align__(16) int8_t tok[];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int channels = FEW_WARPS / split * FEW_CH, c0 = blockIdx.x * channels;
    const int n0 = c0 + warp / split * FEW_CH, r = lane / 4, kk = 16 * (lane % 4);
    if (FLOATS && threadIdx.x < 8)
        amax[threadIdx.x] = 0;
    after_previous();
    const int8_t *w0 = g.B + (long)min(n0 + r, g.N - 1) * g.ldb;
    const int8_t *w1 = g.B + (long)min(n0 + r + 8, g.N - 1) * g.ldb;
    // Four steps at a time, the next four's weights under way.
    constexpr int U = 4;
    const int step = split * FEW_STEP;
    int k = (warp % split) * FEW_STEP + kk;
    uint4 a[U], b[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        a[u] = load16(w0, k + u * step, g.K);
        b[u] = load16(w1, k + u * step, g.K);
    }
    // The epilogue's thread: channel c, tokens m0, m0 + THREADS / channels, ...
    const int c = threadIdx.x % channels, m0 = threadIdx.x / channels;
    const bool out = c0 + c < g.N;
    const float sb = out ? g.sb[c0 + c] : 0.0f;
    const float bias = out && g.bias ? g.bias[c0 + c] : 0.0f;
    if constexpr (FLOATS) {
        __syncthreads();
        quant_tokens<TX>(x, g.M, g.K, tok, scale, amax);
    }
    else if (threadIdx.x < g.M) {
        scale[threadIdx.x] = g.sa[threadIdx.x];
    }
    int sum[4] = {};
    for (; k - kk < g.K; k += U * step) {
        float d[4] = {};
#pragma unroll
        for (int u = 0; u < U; u++) {
            uint4 v = make_uint4(0, 0, 0, 0);
            const int at = k + u * step;
            if (r < g.M) {
                if (!FLOATS)
                    v = load16(g.A + (long)r * g.lda, at, g.K);
                else if (at < g.K)
                    v = *(const uint4 *)(tok + r * x.pitch + at);
            }
            const uint32_t wa[4] = {a[u].x, a[u].y, a[u].z, a[u].w};
            const uint32_t wb[4] = {b[u].x, b[u].y, b[u].z, b[u].w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t a0, a1, a2, a3;
                halves(wa[i], a0, a2);
                halves(wb[i], a1, a3);
                uint32_t b0, b1;
                halves(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w, b0, b1);
                mma_f16(d, a0, a1, a2, a3, b0, b1);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            a[u] = load16(w0, k + (U + u) * step, g.K);
            b[u] = load16(w1, k + (U + u) * step, g.K);
        }
        // U steps are 256 of depth.
#pragma unroll
        for (int i = 0; i < 4; i++)
            sum[i] += __float2int_rn(d[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        part[warp][r + 8 * (i / 2)][2 * (lane % 4) + i % 2] = sum[i];
    __syncthreads();
    for (int m = m0; out && m < g.M; m += THREADS / channels) {
        int s = 0;
        for (int i = 0; i < split; i++)
            s += part[c / FEW_CH * split + i][c % FEW_CH][m];
        float v = act_any(scaled(s, scale[m], sb, bias), g.act, g.slope);
        const long at = (long)m * g.ldc + c0 + c;
        if (g.R)
            v += ldf((const TC *)g.R + at);
        stf((TC *)g.C + at, v);
    }
}

// One or two tokens: a warp takes ROWS rows of the weights, its lanes 16 bytes of
// depth each, 512 bytes of a row together; four products per __dp4a, the lanes'
// sums in one reduction instruction each. `split` as above.
constexpr int DOT_ROWS = 4, DOT_STEP = 512;

template <int MT, typename TC, typename TX>
__global__ void __launch_bounds__(32 * FEW_WARPS)
i8_dot_k(const I8Gemm g, const Tokens x, int split)
{
    constexpr bool FLOATS = !std::is_same<TX, void>::value;
    constexpr int THREADS = 32 * FEW_WARPS, U = 2;
    __shared__ int part[FEW_WARPS][DOT_ROWS][MT];
    __shared__ float scale[MT];
    __shared__ uint32_t amax[MT];
    extern __shared__ __align__(16) int8_t tok[];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int channels = FEW_WARPS / split * DOT_ROWS, c0 = blockIdx.x * channels;
    const int n0 = c0 + warp / split * DOT_ROWS;
    if (FLOATS && threadIdx.x < MT)
        amax[threadIdx.x] = 0;
    after_previous();
    const int8_t *w[DOT_ROWS];
#pragma unroll
    for (int r = 0; r < DOT_ROWS; r++)
        w[r] = g.B + (long)min(n0 + r, g.N - 1) * g.ldb;
    const int step = split * DOT_STEP;
    int k = (warp % split) * DOT_STEP + 16 * lane;
    uint4 a[U][DOT_ROWS];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int r = 0; r < DOT_ROWS; r++)
            a[u][r] = load16(w[r], k + u * step, g.K);
    const int c = threadIdx.x % channels, m0 = threadIdx.x / channels;
    const bool out = m0 < g.M && c0 + c < g.N;
    const float sb = out ? g.sb[c0 + c] : 0.0f;
    const float bias = out && g.bias ? g.bias[c0 + c] : 0.0f;
    if constexpr (FLOATS) {
        __syncthreads();
        quant_tokens<TX>(x, g.M, g.K, tok, scale, amax);
    }
    else if (threadIdx.x < g.M) {
        scale[threadIdx.x] = g.sa[threadIdx.x];
    }
    int acc[DOT_ROWS][MT] = {};
    for (; k - 16 * lane < g.K; k += U * step) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int at = k + u * step;
#pragma unroll
            for (int m = 0; m < MT; m++) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (m < g.M) {
                    if (!FLOATS)
                        v = load16(g.A + (long)m * g.lda, at, g.K);
                    else if (at < g.K)
                        v = *(const uint4 *)(tok + m * x.pitch + at);
                }
#pragma unroll
                for (int r = 0; r < DOT_ROWS; r++) {
                    int s = __dp4a((int)a[u][r].x, (int)v.x, acc[r][m]);
                    s = __dp4a((int)a[u][r].y, (int)v.y, s);
                    s = __dp4a((int)a[u][r].z, (int)v.z, s);
                    acc[r][m] = __dp4a((int)a[u][r].w, (int)v.w, s);
                }
            }
#pragma unroll
            for (int r = 0; r < DOT_ROWS; r++)
                a[u][r] = load16(w[r], at + U * step, g.K);
        }
    }
#pragma unroll
    for (int r = 0; r < DOT_ROWS; r++)
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const int s = __reduce_add_sync(0xffffffffu, acc[r][m]);
            if (lane == 0)
                part[warp][r][m] = s;
        }
    __syncthreads();
    for (int m = m0; out && m < g.M; m += THREADS / channels) {
        int s = 0;
        for (int i = 0; i < split; i++)
            s += part[c / DOT_ROWS * split + i][c % DOT_ROWS][m];
        float v = act_any(scaled(s, scale[m], sb, bias), g.act, g.slope);
        const long at = (long)m * g.ldc + c0 + c;
        if (g.R)
            v += ldf((const TC *)g.R + at);
        stf((TC *)g.C + at, v);
    }
}

constexpr int DOT_TOKENS = 2;

template <typename TC, typename TX>
void few(cudaStream_t st, const I8Gemm &g, const Tokens &x, int sms)
{
    // The depth split as long as there are steps to share and fewer than two
    // blocks per multiprocessor.
    const bool dot = g.M <= DOT_TOKENS;
    const int rows = dot ? DOT_ROWS : FEW_CH, step = dot ? DOT_STEP : FEW_STEP;
    int split = 1;
    while (split < FEW_WARPS && g.K > split * step &&
           (long)g.N * split < 2L * sms * FEW_WARPS * rows)
        split *= 2;
    const unsigned grid = cdiv(g.N, FEW_WARPS / split * rows), T = 32 * FEW_WARPS;
    const size_t smem = (size_t)x.pitch * g.M;
    if (g.M <= 1 && dot)
        launch_chained(i8_dot_k<1, TC, TX>, grid, T, smem, st, g, x, split);
    else if (dot)
        launch_chained(i8_dot_k<2, TC, TX>, grid, T, smem, st, g, x, split);
    else
        launch_chained(i8_few_k<TC, TX>, grid, T, smem, st, g, x, split);
}

// Products that the streaming kernels take: small ones, which on the tcgen05
// cores take the same time or more. Both sides in us, calls among others (M x N
// x K): 1 x 4096 x 2048 5.3 and 5.4, 1 x 8192 x 1500 8.4 and 5.4; 2 x 1024 x
// 4096 5.2 and 5.4, 2 x 4096 x 2048 6.2 and 5.4; 8 x 4096 x 1024 4.9 and 5.1,
// 8 x 8192 x 1024 7.9 and 5.4; 8 x 1024 x 4096, where a warp's chain over the
// depth is long, 7.5 and 5.4.
constexpr int FEW_ROWS = 8;
bool streams(int M, int N, int K)
{
    const long weights = (long)N * K;
    return M == 1   ? weights <= 8 << 20
           : M == 2 ? weights <= 4 << 20
                    : M <= FEW_ROWS && weights <= 4 << 20 && K <= 2048;
}

// Rows that ops_linear_i8 quantises within the product: every block does it
// again, so that it pays for few values only (us in one launch and in two,
// rows x out x in: 1 x 4096 x 1024 4.7 and 6.7, 8 x 1024 x 512 6.0 and 6.6, 4 x
// 4096 x 1024 6.2 and 6.8; 8 x 8192 x 1024 11.8 and 7.0, 1 x 4096 x 4096 8.7 and
// 7.9). The rule does not look at the layer's width, as the work buffer's size
// does not: of wide layers it takes the slower way (1 x 8192 x 512 4.6 and 6.8,
// 2 x 16384 x 1024 7.8 and 8.3, but 1 x 8192 x 1500 10.6 and 7.5, 4 x 8192 x 1024
// 10.4 and 7.2, 1 x 65536 x 1024 28.8 and 18.7).
constexpr int FUSED_VALUES = 4096, FUSED_IN = 2048;
bool fused(int rows, int in)
{
    return rows <= FEW_ROWS && in <= FUSED_IN && (long)rows * in <= FUSED_VALUES;
}

void linear_fused(const struct ocl_backend *ocl, const I8Gemm &g, const View &X, int xtype)
{
    cudaStream_t st = stream_of(ocl);
    const int sms = sms_of(ocl);
    const Tokens x = {X.p, X.ld, token_pitch(g.K)};
    if (xtype == OPS_BF16 && g.c_bf16)
        few<__nv_bfloat16, __nv_bfloat16>(st, g, x, sms);
    else if (xtype == OPS_BF16)
        few<float, __nv_bfloat16>(st, g, x, sms);
    else if (g.c_bf16)
        few<__nv_bfloat16, float>(st, g, x, sms);
    else
        few<float, float>(st, g, x, sms);
}

void gemm_i8(const struct ocl_backend *ocl, const I8Gemm &g)
{
    cudaStream_t st = stream_of(ocl);
    if (g.K == 0) {
        const unsigned grid = 8 * sms_of(ocl);
        if (g.c_bf16)
            launch_chained(i8_empty_k<__nv_bfloat16>, grid, 256, 0, st, g);
        else
            launch_chained(i8_empty_k<float>, grid, 256, 0, st, g);
        return;
    }
    if (streams(g.M, g.N, g.K)) {
        const Tokens none = {nullptr, 0, 0};
        if (g.c_bf16)
            few<__nv_bfloat16, void>(st, g, none, sms_of(ocl));
        else
            few<float, void>(st, g, none, sms_of(ocl));
        return;
    }
    if (!gemm_i8_tc(st, g, sms_of(ocl)))
        fail("8-bit product of %d x %d x %d: the tensor cores refused the operands", g.M, g.N, g.K);
}

// -------------------------------------------------------------- arguments

// Rows and columns whose tile indexes stay within 31 bits.
constexpr int I8_MAX_ROWS = 0x7ffffe00;

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
                  float slope, View *out, View *res, View *in, int *nin)
{
    if (M < 0 || N < 0 || K < 0 || K > OPS_I8_MAX_K || M > I8_MAX_ROWS || N > I8_MAX_ROWS) {
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
        if (!view_of(res, fn, "R", R, roff, C.ld, M, N, es))
            return false;
        if (!same_view(*res, *out) && views_meet(*res, *out)) {
            fail("%s: R and C overlap and are not the same", fn);
            return false;
        }
        g->R = res->p;
    }
    g->M = M;
    g->N = N;
    g->K = K;
    g->ldb = N > 1 ? B.ld : ops_i8_ld(K); // (a single row's pitch may be anything)
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
    if (C > 0x40000000) {
        fail("%s: rows of %d (at most 2^30)", fn, C);
        return;
    }
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
    View in[6], out, res;
    int n = 0;

    if (pending() || !product_args(fn, &g, M, N, K, B, sb, bias, C, ctype, R, roff, act, slope,
                                   &out, &res, in, &n))
        return;
    if (!i8_view(&in[n], fn, "A", A, M, K) ||
        !view_of(&in[n + 1], fn, "the scales of A", sa, 0, M, 1, M, 4) ||
        !apart(fn, out, in, n + 2))
        return;
    if (M == 0 || N == 0)
        return;
    g.A = (const int8_t *)in[n].p;
    g.lda = M > 1 ? A.ld : ops_i8_ld(K);
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
    return rows <= 0 || in <= 0 || fused(rows, in) ? 0 : work_scales(rows) + (size_t)rows * ops_i8_ld(in);
}

extern "C" void ops_linear_i8(struct ops *o, int rows, int in, int out, struct opnd X, int xtype,
                              struct opnd W, cl_mem sw, cl_mem bias, struct opnd Y, int ytype,
                              cl_mem R, long roff, int act, float slope, cl_mem work)
{
    const char *fn = "ops_linear_i8";
    I8Gemm g;
    View v[6], y, res, ws;
    int n = 0;

    if (pending() || !type_ok(fn, xtype) ||
        !product_args(fn, &g, rows, out, in, W, sw, bias, Y, ytype, R, roff, act, slope, &y,
                      &res, v, &n) ||
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
        if (!apart(fn, ws, v, n) || !apart(fn, y, &ws, 1) || !apart(fn, ws, &res, 1))
            return;
    }
    OnDevice dev(o->ocl);
    if (!dev.ok)
        return;
    cudaStream_t st = stream_of(o->ocl);
    Prof p(o->ocl, "linear_i8");
    if (in == 0) {
        g.A = nullptr;
        g.lda = 0;
        g.sa = nullptr;
        gemm_i8(o->ocl, g);
        launch_ok("linear_i8");
        return;
    }
    if (!bytes) {
        linear_fused(o->ocl, g, x, xtype);
        launch_ok("linear_i8");
        return;
    }
    int8_t *q = (int8_t *)ws.p + work_scales(rows);
    quant_rows(st, x, xtype, q, ops_i8_ld(in), (float *)ws.p);
    g.A = q;
    g.lda = ops_i8_ld(in);
    g.sa = (const float *)ws.p;
    gemm_i8(o->ocl, g);
    launch_ok("linear_i8");
}
