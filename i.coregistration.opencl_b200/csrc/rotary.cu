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
    // (Factors up to 1 slow no frequency down: their logarithm is not positive.)
    r->mscale = scaling == OPS_ROTARY_PARTS && factor > 1.0 ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
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

struct Rotary {
    struct ops_rotary r;
    long rows, ldx, ldy;
    int nh, d;
    const void *X;
    void *Y;
    const int *pos;
    long pos0;
    // Per head `units` pieces of work: `turns` of rotated columns (two vectors a
    // unit: a pair's halves, or one of neighbouring pairs), then vectors that
    // are copied (none in place).
    int units, turns;
    int split; // warps that share a row's units
};

constexpr int WARPS = 8;

// N neighbouring values as the words (or the one half word) they lie in.
template <typename T, int N>
struct Run {
    static constexpr int B = N * (int)sizeof(T), W = B >= 4 ? B / 4 : 1;
    uint32_t w[W];
    __device__ __forceinline__ void load(const T *p)
    {
        if constexpr (B == 16) {
            const uint4 v = *(const uint4 *)p;
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        }
        else if constexpr (B == 8) {
            const uint2 v = *(const uint2 *)p;
            w[0] = v.x, w[1] = v.y;
        }
        else if constexpr (B == 4) {
            w[0] = *(const uint32_t *)p;
        }
        else {
            w[0] = *(const uint16_t *)p;
        }
    }
    __device__ __forceinline__ void store(T *p) const
    {
        if constexpr (B == 16)
            *(uint4 *)p = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (B == 8)
            *(uint2 *)p = make_uint2(w[0], w[1]);
        else if constexpr (B == 4)
            *(uint32_t *)p = w[0];
        else
            *(uint16_t *)p = (uint16_t)w[0];
    }
    __device__ __forceinline__ float at(int e) const
    {
        if constexpr (sizeof(T) == 4)
            return __uint_as_float(w[e]);
        else
            return __uint_as_float(e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
    // Values e and e + 1.
    __device__ __forceinline__ void set2(int e, float x, float y)
    {
        if constexpr (sizeof(T) == 4) {
            w[e] = __float_as_uint(x);
            if (e + 1 < N)
                w[e + 1] = __float_as_uint(y);
        }
        else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
            w[e / 2] = *(const uint32_t *)&h;
        }
    }
};

// A warp per row (or, for few rows, per part of a row's heads). Its lanes
// compute the row's cosines and sines once for all heads, into shared
// memory, while its first loads are under way, then walk the row's units in
// order, four at a time, so that a warp reads and writes runs of neighbouring
// bytes. Memory bound: every column is read and written once. HALF: pairs (f,
// f + rot / 2).
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(32 * WARPS, 6)
rotary_k(const __grid_constant__ Rotary p)
{
    __shared__ alignas(16) float2 table[WARPS][OPS_ROTARY_MAX / 2];
    // Units of a lane under way: two loads. More warps hide the memory's
    // latency better than more units (12808 x 32 x 64 bfloat16, two units and
    // 4 blocks of a multiprocessor 24.7 us, four and 3 31.2, one and 6 22.8).
    constexpr int U = HALF ? 1 : 2;
    // Pairs of a unit.
    constexpr int P = HALF || V == 1 ? V : V / 2;
    // Two single neighbours are loaded one by one: rows may start anywhere.
    constexpr bool LONE = !HALF && V == 1;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, nf = p.r.rot / 2;
    const int second = p.r.axes == 2 ? nf / 2 : nf; // first pair of the second axis
    float2 *cs = table[warp];
    after_previous();
    const long jobs = p.rows * p.split;
    const int total = p.nh * p.units, dh = 32 / p.units, du = 32 - dh * p.units;
    for (long job = (long)blockIdx.x * WARPS + warp; job < jobs; job += (long)gridDim.x * WARPS) {
        const long row = p.split == 1 ? job : job / p.split;
        const int part = p.split == 1 ? 0 : (int)(job - row * p.split);
        const T *x = (const T *)p.X + row * p.ldx;
        T *y = (T *)p.Y + row * p.ldy;
        long p0 = p.pos0, p1 = p.pos0;
        if (p.pos) {
            p0 += p.pos[row * p.r.axes];
            p1 += p.pos[row * p.r.axes + p.r.axes - 1];
        }
        else {
            p0 += row;
        }
        const int e0 = (int)((long)total * part / p.split), e1 = (int)((long)total * (part + 1) / p.split);
        // Unit e of the row: head e / units, its unit e % units.
        int h = (e0 + lane) / p.units, u = e0 + lane - h * p.units;
        for (int e = e0 + lane, first = 1; e - lane < e1; e += 32 * U, first = 0) {
            Run<T, V> a[U], b[U];
            int at[U], un[U];
#pragma unroll
            for (int i = 0; i < U; i++) {
                un[i] = u;
                const bool turn = u < p.turns;
                at[i] = h * p.d + (turn ? (LONE ? 2 * u : u * V) : p.r.rot + (u - p.turns) * V);
                if (e + 32 * i < e1) {
                    a[i].load(x + at[i]);
                    if ((HALF || LONE) && turn)
                        b[i].load(x + at[i] + (HALF ? nf : 1));
                }
                h += dh;
                u += du;
                if (u >= p.units) {
                    u -= p.units;
                    h++;
                }
            }
            if (first) {
                __syncwarp(); // the previous row's table is read
                for (int f = lane; f < nf; f += 32)
                    cs[f] = turn_of(f < second ? p0 : p1, p.r.step[f], p.r.mscale);
                __syncwarp();
            }
#pragma unroll
            for (int i = 0; i < U; i++) {
                if (e + 32 * i >= e1)
                    continue;
                if (un[i] < p.turns) {
                    float2 t[P];
#pragma unroll
                    for (int k = 0; k < P; k++)
                        t[k] = cs[un[i] * P + k];
                    if (HALF || LONE) {
#pragma unroll
                        for (int k = 0; k < V; k += 2) {
                            const int k1 = k + 1 < V ? k + 1 : k;
                            const float a0 = a[i].at(k), b0 = b[i].at(k), a1 = a[i].at(k1),
                                        b1 = b[i].at(k1);
                            a[i].set2(k, a0 * t[k].x - b0 * t[k].y, a1 * t[k1].x - b1 * t[k1].y);
                            b[i].set2(k, a0 * t[k].y + b0 * t[k].x, a1 * t[k1].y + b1 * t[k1].x);
                        }
                        b[i].store(y + at[i] + (HALF ? nf : 1));
                    }
                    else {
#pragma unroll
                        for (int k = 0; k < P; k++) {
                            const float va = a[i].at(2 * k), vb = a[i].at(2 * k + 1);
                            a[i].set2(2 * k, va * t[k].x - vb * t[k].y, va * t[k].y + vb * t[k].x);
                        }
                    }
                }
                a[i].store(y + at[i]);
            }
        }
    }
}

template <typename T, int V>
void launch(cudaStream_t st, Rotary p, int sms)
{
    const int nf = p.r.rot / 2;
    p.turns = p.r.interleaved ? (V >= 2 ? p.r.rot / V : nf) : nf / V;
    p.units = p.turns + (p.X == p.Y ? 0 : (p.d - p.r.rot) / V);
    // Enough warps for the device where there are few rows, each with at least
    // a unit per lane.
    const long total = (long)p.nh * p.units, most = (total + 31) / 32;
    const long want = (4L * sms * WARPS + p.rows - 1) / p.rows;
    p.split = (int)(want < 1 ? 1 : want < most ? want : most);
    const long blocks = (p.rows * p.split + WARPS - 1) / WARPS;
    const unsigned grid = (unsigned)(blocks < 32L * sms ? blocks : 32L * sms);
    if (p.r.interleaved)
        launch_chained(rotary_k<T, V, false>, grid, 32 * WARPS, 0, st, p);
    else
        launch_chained(rotary_k<T, V, true>, grid, 32 * WARPS, 0, st, p);
}

// The widest vectors, of 16 bytes down to one value, at which every run that
// is read or written starts aligned and is whole.
template <typename T>
void run(cudaStream_t st, const Rotary &p, int sms)
{
    constexpr int W = 16 / (int)sizeof(T);
    auto fits = [&](int v) {
        const int b = v * (int)sizeof(T);
        return (uintptr_t)p.X % b == 0 && (uintptr_t)p.Y % b == 0 && p.d % v == 0 &&
               (p.rows == 1 || (p.ldx % v == 0 && p.ldy % v == 0)) && p.r.rot % v == 0 &&
               (p.r.interleaved || p.r.rot / 2 % v == 0);
    };
    if (fits(W))
        launch<T, W>(st, p, sms);
    else if (fits(W / 2))
        launch<T, W / 2>(st, p, sms);
    else if (W > 4 && fits(2))
        launch<T, 2>(st, p, sms);
    else
        launch<T, 1>(st, p, sms);
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
    if (nh < 0 || d < r->rot || (long)nh * d > 0x40000000L) {
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
    Rotary q = {};
    q.r = *r;
    q.rows = rows;
    q.ldx = X.ld;
    q.ldy = Y.ld;
    q.nh = nh;
    q.d = d;
    q.X = x.p;
    q.Y = y.p;
    q.pos = (const int *)v.p;
    q.pos0 = pos0;
    Prof p(o->ocl, "rotary");
    if (type == OPS_BF16)
        run<__nv_bfloat16>(st, q, sms_of(o->ocl));
    else
        run<float>(st, q, sms_of(o->ocl));
    launch_ok("rotary");
}
