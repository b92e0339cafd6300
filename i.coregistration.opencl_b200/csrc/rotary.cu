// SPDX-License-Identifier: Unlicense
//
// Rotary positions (ops_b200.h): ops_rotary_plan and ops_rotary.

#include <math.h>
#include <string.h>

#include "opcheck.cuh"

using namespace coreg;

// ------------------------------------------------------------ frequencies

extern "C" void ops_rotary_plan(struct ops_rotary *r, int rot, int axes, int interleaved,
                                double base, int scaling, double factor, long length)
{
    const char *fn = "ops_rotary_plan";

    if (pending())
        return;
    if (!r) {
        fail("%s: no struct to fill", fn);
        return;
    }
    memset(r, 0, sizeof(*r));
    if (axes < 1 || axes > 2 || rot < 2 || rot > OPS_ROTARY_MAX || rot % (2 * axes)) {
        fail("%s: %d rotated columns (at most %d) over %d axes", fn, rot, OPS_ROTARY_MAX, axes);
        return;
    }
    const int n = rot / axes;
    if (!(base > 0.0 && isfinite(base)) || scaling < OPS_ROTARY_PLAIN ||
        scaling > OPS_ROTARY_PARTS ||
        (scaling != OPS_ROTARY_PLAIN && !(factor > 0.0 && isfinite(factor))) ||
        (scaling == OPS_ROTARY_PARTS && length < 1)) {
        fail("%s: base %g, scaling %d by %g, length %ld", fn, base, scaling, factor, length);
        return;
    }
    r->rot = rot;
    r->axes = axes;
    r->interleaved = interleaved != 0;
    r->mscale = scaling == OPS_ROTARY_PARTS ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
    const long double two_pi = 6.283185307179586476925286766559L;
    long double b = base;
    if (scaling == OPS_ROTARY_NTK && n > 2)
        b *= powl(factor, (long double)n / (n - 2));
    for (int i = 0; i < n / 2; i++) {
        long double w = powl(b, -2.0L * i / n);
        if (scaling == OPS_ROTARY_LINEAR)
            w /= factor;
        if (scaling == OPS_ROTARY_PARTS) {
            long double g = (length * w / two_pi - 1.0L) / 31.0L;
            g = g < 0.0L ? 0.0L : g > 1.0L ? 1.0L : g;
            w = g * w + (1.0L - g) * w / factor;
        }
        // Turns per position, whole turns dropped, rounded to 2^-64.
        long double turn = w / two_pi;
        turn = (turn - floorl(turn)) * 0x1p64L + 0.5L;
        const uint64_t step = turn >= 0x1p64L ? 0 : (uint64_t)turn;
        for (int a = 0; a < axes; a++)
            r->step[a * (n / 2) + i] = step;
    }
}

// ------------------------------------------------------------------ kernel

namespace coreg {
namespace {

// The turned pair's factors at position p: t = p step is the angle as a
// fraction of 2^64 of a turn, whole turns gone with the overflow, so that
// far positions cost no accuracy; as a signed number it is within half a
// turn, and 2^-63 of it is the angle over pi.
__device__ __forceinline__ float2 turn_of(long p, uint64_t step, float m)
{
    const long long t = (long long)((uint64_t)p * step);
    float2 cs;
    sincospif((float)t * 0x1p-63f, &cs.y, &cs.x);
    cs.x *= m;
    cs.y *= m;
    return cs;
}

// One thread per (row, pair), which loops over the heads; with a separate
// output the threads of a row copy the columns that are not rotated.
template <typename T>
__global__ void __launch_bounds__(256)
rotary_k(const __grid_constant__ struct ops_rotary r, long rows, int nh, int d, const T *X,
         long ldx, T *Y, long ldy, const int *pos, long pos0)
{
    const int nf = r.rot / 2, per = nf / r.axes;
    for (long e = (long)blockIdx.x * blockDim.x + threadIdx.x; e < rows * nf;
         e += (long)gridDim.x * blockDim.x) {
        const long row = e / nf;
        const int f = (int)(e % nf);
        const long p = pos0 + (pos ? pos[row * r.axes + f / per] : row);
        const float2 cs = turn_of(p, r.step[f], r.mscale);
        const int i0 = r.interleaved ? 2 * f : f, i1 = r.interleaved ? 2 * f + 1 : f + nf;
        for (int h = 0; h < nh; h++) {
            const T *x = X + row * ldx + h * d;
            T *y = Y + row * ldy + h * d;
            const float a = ldf(x + i0), b = ldf(x + i1);
            stf(y + i0, a * cs.x - b * cs.y);
            stf(y + i1, a * cs.y + b * cs.x);
            if (x != y)
                for (int c = r.rot + f; c < d; c += nf)
                    y[c] = x[c];
        }
    }
}

}  // namespace
}  // namespace coreg

extern "C" void ops_rotary(struct ops *o, const struct ops_rotary *r, long rows, int nh, int d,
                           struct opnd X, struct opnd Y, int type, cl_mem pos, long pos0)
{
    const char *fn = "ops_rotary";
    View x, y, v;

    if (pending())
        return;
    if (!r || r->axes < 1 || r->axes > 2 || r->rot < 2 || r->rot > OPS_ROTARY_MAX ||
        r->rot % (2 * r->axes)) {
        fail("%s: no frequencies (ops_rotary_plan)", fn);
        return;
    }
    if (nh < 0 || d < r->rot || (long)nh * d > 0x7fffffffL) {
        fail("%s: %d heads of %d columns, %d rotated", fn, nh, d, r->rot);
        return;
    }
    if (!pos && r->axes != 1) {
        fail("%s: two axes need positions", fn);
        return;
    }
    const long E = (long)nh * d;
    if (!type_ok(fn, type) ||
        !view_of(&x, fn, "X", X.buf, X.off, X.ld, rows, E, type_size(type)) ||
        !view_of(&y, fn, "Y", Y.buf, Y.off, Y.ld, rows, E, type_size(type)) ||
        (pos && !view_of(&v, fn, "the positions", pos, 0, r->axes, rows, r->axes, 4)))
        return;
    if (!same_view(x, y) && views_meet(x, y)) {
        fail("%s: X and Y overlap and are not the same", fn);
        return;
    }
    if (pos && ranges_meet(v.p, v.span(), y.p, y.span())) {
        fail("%s: Y overlaps the positions", fn);
        return;
    }
    if (rows == 0 || nh == 0)
        return;
    OnDevice dev(o->ocl);
    if (!dev.ok)
        return;
    cudaStream_t st = stream_of(o->ocl);
    const long pairs = rows * (r->rot / 2);
    const unsigned grid = (unsigned)(pairs / 256 + 1 < 65536 ? pairs / 256 + 1 : 65536);
    Prof p(o->ocl, "rotary");
    if (type == OPS_BF16)
        rotary_k<<<grid, 256, 0, st>>>(*r, rows, nh, d, (const __nv_bfloat16 *)x.p, (long)X.ld,
                                       (__nv_bfloat16 *)y.p, (long)Y.ld, (const int *)v.p, pos0);
    else
        rotary_k<<<grid, 256, 0, st>>>(*r, rows, nh, d, (const float *)x.p, (long)X.ld,
                                       (float *)y.p, (long)Y.ld, (const int *)v.p, pos0);
    launch_ok("rotary");
}
