// SPDX-License-Identifier: Unlicense
//
// Argument checks shared by the operations that take typed operands
// (linear_i8.cu, rotary.cu, groupnorm.cu), the guard that runs them on the
// ops context's device, and their activations.

#pragma once

#include "common.cuh"
#include "ops_b200.h"

namespace coreg {

// Makes the backend's device current for the scope.
class OnDevice {
    int old_ = -1;

public:
    bool ok = false;
    explicit OnDevice(const struct ocl_backend *ocl)
    {
        int cur = -1;
        if (!cuda_ok(cudaGetDevice(&cur), "cudaGetDevice"))
            return;
        if (cur != ocl->device) {
            if (!cuda_ok(cudaSetDevice(ocl->device), "cudaSetDevice"))
                return;
            old_ = cur;
        }
        ok = true;
    }
    ~OnDevice()
    {
        if (old_ >= 0)
            cudaSetDevice(old_);
    }
};

// A rows x cols operand in device memory: pitch and size in bytes.
struct View {
    char *p = nullptr;
    long rows = 0, cols = 0, ld = 0; // elements
    int es = 1;
    // Bytes from the first element to behind the last.
    long span() const { return rows > 0 ? ((rows - 1) * ld + cols) * es : 0; }
};

// The operand as a view; fails (with the entry point and the operand
// named) on a NULL buffer, a negative offset, rows that overlap, memory
// beyond the buffer or a misaligned element. strict: rows must not overlap
// (ld >= cols); always wanted of outputs.
inline bool view_of(View *v, const char *fn, const char *what, cl_mem buf, long off, long ld,
                    long rows, long cols, int es)
{
    if (!buf) {
        fail("%s: required buffer %s is NULL", fn, what);
        return false;
    }
    if (off < 0 || rows < 0 || cols < 0 || (rows > 1 && ld < cols)) {
        fail("%s: %s at offset %ld, %ld rows of %ld, leading dimension %ld", fn, what, off, rows,
             cols, ld);
        return false;
    }
    // In 128 bits: no product of sizes wraps round.
    const __int128 end = (__int128)off + (rows > 0 ? (__int128)(rows - 1) * ld + cols : 0);
    if (end > (__int128)(buf->bytes / es)) {
        fail("%s: %s (%ld rows of %ld, leading dimension %ld, offset %ld) passes its buffer of "
             "%zu bytes",
             fn, what, rows, cols, ld, off, buf->bytes);
        return false;
    }
    v->p = (char *)buf->ptr + off * es;
    v->rows = rows;
    v->cols = cols;
    v->ld = ld;
    v->es = es;
    if ((uintptr_t)v->p % es) {
        fail("%s: %s is not aligned to its %d-byte elements", fn, what, es);
        return false;
    }
    return true;
}

inline bool type_ok(const char *fn, int type)
{
    if (type == OPS_FP32 || type == OPS_BF16)
        return true;
    fail("%s: element type %d", fn, type);
    return false;
}

inline bool act_ok(const char *fn, int act)
{
    if (act >= ACT_NONE && act <= ACT_SILU)
        return true;
    fail("%s: activation %d", fn, act);
    return false;
}

inline int type_size(int type) { return type == OPS_BF16 ? 2 : 4; }

// Whether two byte ranges share memory.
inline bool ranges_meet(const void *a, long na, const void *b, long nb)
{
    return na > 0 && nb > 0 && (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

// Whether an output shares memory with an input: ranges that meet, but not
// those of separate columns of the same rows (equal pitch).
inline bool views_meet(const View &a, const View &b)
{
    if (!ranges_meet(a.p, a.span(), b.p, b.span()))
        return false;
    const long pitch = a.ld * a.es;
    if (a.rows > 1 && b.rows > 1 && pitch == b.ld * b.es && pitch > 0) {
        long d = (long)((uintptr_t)b.p - (uintptr_t)a.p) % pitch; // b's column behind a's
        if (d < 0)
            d += pitch;
        return !(d >= a.cols * a.es && d + b.cols * b.es <= pitch);
    }
    return true;
}

// The same memory in the same layout (an output written in place).
inline bool same_view(const View &a, const View &b)
{
    return a.p == b.p && a.es == b.es && (a.rows <= 1 || a.ld == b.ld);
}

// Multiprocessors of the backend's device.
inline int sms_of(const struct ocl_backend *ocl) { return ocl->sm_count > 0 ? ocl->sm_count : 148; }

// Launches a kernel whose blocks may start while the stream's previous kernel
// ends (programmatic stream serialization): every thread of it calls
// after_previous() before its first access to global memory.
template <typename... P, typename... A>
bool launch_chained(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem,
                    cudaStream_t st, const A &...args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cuda_ok(cudaLaunchKernelEx(&cfg, kernel, P(args)...), "kernel launch");
}

}  // namespace coreg

// Lets the stream's next kernel start its blocks as this one's leave room (it
// waits in its own after_previous), then waits until the previous kernel has
// ended and its writes are visible. Saves the launch latency between
// dependent kernels, 1 to 2 us.
__device__ __forceinline__ void after_previous()
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ------------------------------------------------------------ activations

// a * b + c of two floats in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 d;
    asm("{\n\t.reg .b64 x, y, z, w;\n\t"
        "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

__device__ __forceinline__ float2 pair(float v) { return make_float2(v, v); }

// a b + c clamped to 0..1 (0 for NaN).
__device__ __forceinline__ float fma_sat(float a, float b, float c)
{
    float d;
    asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Exact GELU, x Phi(x), of two values. Phi(x) = 0.5 + x Q(min(x^2, X^2)),
// clamped to 0..1, where Q is the polynomial in s = 2 x^2 / X^2 - 1 with the
// least largest error of x Q over |x| <= X (fitted here in 64 bits). FINE:
// degree 14, X = 5.4, and Phi off by at most 1.3e-7 in float32 arithmetic, as 0.5
// (1 + erff(x / sqrt 2)) is by 0.6e-7; otherwise degree 12, X = 5.2, 4.3e-7,
// which is for results that are rounded to bfloat16 (2^-8). At X, x Q passes
// 0.5, so that larger |x| give exactly x or 0. In packed multiply-adds but for
// four operations of a pair: about half the issue slots of CUDA's erff in
// the same formula, which bounded the epilogue of the 8-bit product.
template <bool FINE>
__device__ __forceinline__ float2 gelu2(float2 x)
{
    constexpr int D = FINE ? 14 : 12;
    constexpr float X = FINE ? 5.4f : 5.2f;
    constexpr float Q14[15] = {
        0.13092811405658722f,    -0.06532805413007736f,  0.04849959164857864f,
        -0.03920681402087212f,   0.03211659565567970f,   -0.02574645727872848f,
        0.01964514516294003f,    -0.01396332029253245f,  0.00965119525790214f,
        -0.006715338211506605f,  0.003658922854810953f,  -0.0011864101979881525f,
        0.0008749334374442696f,  -0.0010283688316121697f, 0.00039285887032747269f};
    constexpr float Q12[13] = {
        0.13594993948936462f,  -0.06774269789457321f,  0.05002840608358383f,
        -0.03995957598090172f, 0.03193814679980278f,   -0.024464763700962067f,
        0.01820363663136959f,  -0.013464033603668213f, 0.008026459254324436f,
        -0.003071868559345603f, 0.002321982756257057f, -0.0026904314290732145f,
        0.0010786805069074035f};
    float2 u = fma2(x, x, pair(0.0f));
    u = make_float2(fminf(u.x, X * X), fminf(u.y, X * X));
    const float2 s = fma2(u, pair(2.0f / (X * X)), pair(-1.0f));
    float2 q = pair(FINE ? Q14[D] : Q12[D <= 12 ? D : 0]);
#pragma unroll
    for (int i = D - 1; i >= 0; i--)
        q = fma2(q, s, pair(FINE ? Q14[i] : Q12[i <= 12 ? i : 0]));
    return fma2(x, make_float2(fma_sat(x.x, q.x, 0.5f), fma_sat(x.y, q.y, 0.5f)), pair(0.0f));
}

// The larger value, or NaN where one is (fmaxf would drop it).
__device__ __forceinline__ float max_nan(float a, float b)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// v / (1 + e^-t) by the fast exponential and division: relative error below
// 4e-7 (1 + |t|). Where e^-t overflows the quotient is 0, the limit.
__device__ __forceinline__ float times_sigmoid(float v, float t)
{
    return __fdividef(v, 1.0f + __expf(-t));
}

// The activation of two values, FINE as in gelu2. GELU_TANH is v sigmoid(2 y)
// with y the argument of its tanh.
template <int ACT, bool FINE>
__device__ __forceinline__ float2 act2(float2 v, float slope)
{
    if (ACT == ACT_GELU)
        return gelu2<FINE>(v);
    if (ACT == ACT_RELU)
        return make_float2(max_nan(v.x, 0.0f), max_nan(v.y, 0.0f));
    if (ACT == ACT_LEAKY)
        return make_float2(v.x >= 0.0f ? v.x : slope * v.x, v.y >= 0.0f ? v.y : slope * v.y);
    if (ACT == ACT_GELU_TANH) {
        constexpr float k = 1.5957691216057308f; // 2 sqrt(2 / pi)
        return make_float2(
            times_sigmoid(v.x, k * v.x * fmaf(0.044715f * v.x, v.x, 1.0f)),
            times_sigmoid(v.y, k * v.y * fmaf(0.044715f * v.y, v.y, 1.0f)));
    }
    if (ACT == ACT_SILU)
        return make_float2(times_sigmoid(v.x, v.x), times_sigmoid(v.y, v.y));
    return v;
}

template <int ACT>
__device__ __forceinline__ float act1(float v, float slope)
{
    return act2<ACT, true>(make_float2(v, 0.0f), slope).x;
}

// The same with the activation known at run time only.
__device__ __forceinline__ float act_any(float v, int act, float slope)
{
    switch (act) {
    case ACT_GELU:
        return act1<ACT_GELU>(v, slope);
    case ACT_RELU:
        return act1<ACT_RELU>(v, slope);
    case ACT_LEAKY:
        return act1<ACT_LEAKY>(v, slope);
    case ACT_GELU_TANH:
        return act1<ACT_GELU_TANH>(v, slope);
    case ACT_SILU:
        return act1<ACT_SILU>(v, slope);
    }
    return v;
}
