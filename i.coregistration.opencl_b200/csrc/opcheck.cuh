// SPDX-License-Identifier: Unlicense
//
// Argument checks shared by the operations that take typed operands
// (linear_i8.cu, rotary.cu, groupnorm.cu), the guard that runs them on the
// ops context's device, and their activations.

#pragma once

#include <atomic>

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
// beyond the buffer or a misaligned element.
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

// A number above 0 that a kernel's launches need and each device answers for
// itself: asked once per device, or, by host threads that call at the same
// time, more than once.
constexpr int MAX_DEVICES = 32;
struct PerDevice {
    std::atomic<int> known[MAX_DEVICES];
    template <typename F>
    int get(F ask)
    {
        int dev = -1;
        cudaGetDevice(&dev);
        if (dev < 0 || dev >= MAX_DEVICES)
            return ask();
        int n = known[dev].load(std::memory_order_relaxed);
        if (n <= 0) {
            n = ask();
            known[dev].store(n, std::memory_order_relaxed);
        }
        return n;
    }
};

// Launches a kernel whose blocks may start while the stream's previous kernel
// ends (programmatic stream serialization): every thread of it calls
// after_previous() before its first access to global memory, and reads none
// through the read-only cache, as the previous kernel may have written it
// since this one started.
template <typename... P, typename... A>
bool launch_clusters(void (*kernel)(P...), dim3 grid, unsigned cluster, unsigned threads,
                     size_t smem, cudaStream_t st, const A &...args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster ? 2 : 1;
    return cuda_ok(cudaLaunchKernelEx(&cfg, kernel, P(args)...), "kernel launch");
}

// The same without clusters, or with those of the kernel's own attribute.
template <typename... P, typename... A>
bool launch_chained(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem,
                    cudaStream_t st, const A &...args)
{
    return launch_clusters(kernel, grid, 0, threads, smem, st, args...);
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

// 2^x, to 2 units of the last place.
__device__ __forceinline__ float exp2_fast(float x)
{
    float d;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
    return d;
}

__device__ __forceinline__ float rcp_fast(float x)
{
    float d;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(x));
    return d;
}

// The larger value, or NaN where one is (fmaxf would drop it).
__device__ __forceinline__ float max_nan(float a, float b)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// x / (1 + 2^z) of two values, relative error below 4e-7 for exact z. Products are
// never contracted with what a caller adds, so that kernels give equal results.
//
// Each by a reciprocal of its own: where 2^z passes float's range that is 0,
// and so is the quotient, of any finite x. SHARED: by one reciprocal for both, a
// third less of the special function unit's work (8 cycles an instruction and
// warp), which bounds the group norm. Then exponents are cut off at 60, so that
// the product of the two divisors stays in range, and x at -60, where the
// callers' z is above that: what should be nearer to zero than 2^-54 comes
// out as at most that (60 2^-60), however large x is. us, own and shared:
// products of 25616 x 4096 x 1024 with GELU 130 and 136, with SiLU 122 and 128
// (instructions bound their epilogue); group norm of 3 x 8137 x 120 float32
// with GELU 10.2 and 9.6, of 35 x 35 x 512 with SiLU 5.95 and 5.81.
template <bool SHARED>
__device__ __forceinline__ float2 over_one_plus_exp2(float2 x, float2 z)
{
    if (!SHARED) {
        const float2 a = fma2(make_float2(exp2_fast(z.x), exp2_fast(z.y)), pair(1.0f), pair(1.0f));
        return fma2(x, make_float2(rcp_fast(a.x), rcp_fast(a.y)), pair(-0.0f));
    }
    const float a = 1.0f + exp2_fast(fminf(z.x, 60.0f)), b = 1.0f + exp2_fast(fminf(z.y, 60.0f));
    const float r = rcp_fast(a * b);
    return make_float2(__fmul_rn(max_nan(x.x, -60.0f), b * r),
                       __fmul_rn(max_nan(x.y, -60.0f), a * r));
}

// Exact GELU, x Phi(x), of two values, as x / (1 + 2^(x Q(x^2))): log2(Phi(-x) /
// Phi(x)) / x is a smooth even function, and Q the polynomial of degree 6 in
// min(x^2, 25) that brings Phi nearest to it (fitted here in 64 bits,
// weighted by the derivative Phi (1 - Phi) x). In float32 Phi is off by at
// most 1.5e-7 (0.5 (1 + erff(x / sqrt 2)) by 0.6e-7) and by 5e-5 of itself down
// to x = -3, where the other form has lost that too; 1 and 0 follow far out.
// Half the work of erff's polynomials, which bounded the 8-bit product's
// epilogue.
template <bool SHARED>
__device__ __forceinline__ float2 gelu2(float2 x)
{
    constexpr float Q[7] = {-2.302206516265869f,      -0.10484472662210464f,
                            0.00010274611122440547f,  0.000156551250256598f,
                            -1.098385200748453e-05f,  3.5264929465483874e-07f,
                            -4.4573145174808815e-09f};
    float2 u = fma2(x, x, pair(0.0f));
    u = make_float2(fminf(u.x, 25.0f), fminf(u.y, 25.0f));
    float2 q = pair(Q[6]);
#pragma unroll
    for (int i = 5; i >= 0; i--)
        q = fma2(q, u, pair(Q[i]));
    return over_one_plus_exp2<SHARED>(x, fma2(x, q, pair(0.0f)));
}

// The larger value, or NaN where one is (fmaxf would drop it).

// The activation of two values. GELU_TANH is v sigmoid(2 y) with y the argument
// of its tanh, SiLU v sigmoid(v).
template <int ACT, bool SHARED = false>
__device__ __forceinline__ float2 act2(float2 v, float slope)
{
    if (ACT == ACT_GELU)
        return gelu2<SHARED>(v);
    if (ACT == ACT_RELU)
        return make_float2(max_nan(v.x, 0.0f), max_nan(v.y, 0.0f));
    if (ACT == ACT_LEAKY)
        return make_float2(v.x >= 0.0f ? v.x : __fmul_rn(slope, v.x),
                           v.y >= 0.0f ? v.y : __fmul_rn(slope, v.y));
    if (ACT == ACT_GELU_TANH) {
        // 2^(-2 y / ln 2): -2 sqrt(2 / pi) / ln 2 and 0.044715 of that.
        const float2 u = fma2(v, v, pair(0.0f));
        const float2 q = fma2(u, pair(-0.1029432395800235f), pair(-2.302208198144325f));
        return over_one_plus_exp2<SHARED>(v, fma2(v, q, pair(0.0f)));
    }
    if (ACT == ACT_SILU)
        return over_one_plus_exp2<SHARED>(v, fma2(v, pair(-1.4426950408889634f), pair(0.0f)));
    return v;
}

// The same with the activation known at run time only.
__device__ __forceinline__ float2 act2_any(float2 v, int act, float slope)
{
    switch (act) {
    case ACT_GELU:
        return act2<ACT_GELU>(v, slope);
    case ACT_RELU:
        return act2<ACT_RELU>(v, slope);
    case ACT_LEAKY:
        return act2<ACT_LEAKY>(v, slope);
    case ACT_GELU_TANH:
        return act2<ACT_GELU_TANH>(v, slope);
    case ACT_SILU:
        return act2<ACT_SILU>(v, slope);
    }
    return v;
}

__device__ __forceinline__ float act_any(float v, int act, float slope)
{
    return act2_any(make_float2(v, 0.0f), act, slope).x;
}
