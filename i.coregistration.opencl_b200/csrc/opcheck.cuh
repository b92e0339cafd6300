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

}  // namespace coreg

// Activations of these operations: ops.h's and x sigmoid(x). The last is
// x / (1 + e^-x): for x -> -inf the exponential overflows to infinity and
// the quotient is -0, the limit.
template <int ACT>
__device__ __forceinline__ float act_of(float v, float slope)
{
    if (ACT == ACT_SILU)
        return __fdividef(v, 1.0f + __expf(-v));
    return apply_act(v, ACT, slope);
}
