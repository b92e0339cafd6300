// SPDX-License-Identifier: Unlicense
//
// Group norm with an activation over channels-last maps (ops_b200.h):
// ops_groupnorm_cl.

#include "opcheck.cuh"

using namespace coreg;

namespace coreg {
namespace {

struct GroupNorm {
    int nimg, C, groups;
    long HW;
    const void *X;
    long ldx, sx;
    void *Y;
    long ldy, sy;
    const float *g, *b;
    float eps;
    int act;
    float slope;
};

// One block per group of an image, three passes over it: the mean, the
// variance about it, the result.
template <typename TX, typename TY>
__global__ void __launch_bounds__(256)
group_k(const GroupNorm p)
{
    __shared__ float red[32];
    const int per = p.C / p.groups, img = blockIdx.y, c0 = blockIdx.x * per;
    const TX *x = (const TX *)p.X + img * p.sx + c0;
    TY *y = (TY *)p.Y + img * p.sy + c0;
    const long n = p.HW * per;
    float s = 0.0f;
    for (long e = threadIdx.x; e < n; e += blockDim.x)
        s += ldf(x + e / per * p.ldx + e % per);
    const float mean = block_sum(s, red) / n;
    s = 0.0f;
    for (long e = threadIdx.x; e < n; e += blockDim.x) {
        const float d = ldf(x + e / per * p.ldx + e % per) - mean;
        s = fmaf(d, d, s);
    }
    const float rstd = rsqrtf(block_sum(s, red) / n + p.eps);
    for (long e = threadIdx.x; e < n; e += blockDim.x) {
        const int c = (int)(e % per);
        float v = (ldf(x + e / per * p.ldx + c) - mean) * rstd;
        if (p.g)
            v = v * p.g[c0 + c] + p.b[c0 + c];
        v = p.act == ACT_SILU ? act_of<ACT_SILU>(v, 0.0f) : apply_act(v, p.act, p.slope);
        stf(y + e / per * p.ldy + c, v);
    }
}

// The maps as one view: rows of C for one image, images s0 apart.
bool map_view(View *v, const char *fn, const char *what, const struct opnd &m, int nimg, long HW,
              int C, int es, bool output)
{
    if (!view_of(v, fn, what, m.buf, m.off, m.ld, HW, C, es))
        return false;
    const __int128 one = (__int128)(HW - 1) * m.ld + C;
    if (nimg > 1 && (m.s0 < 0 || (output && (__int128)m.s0 < one))) {
        fail("%s: %s: images %ld elements apart", fn, what, m.s0);
        return false;
    }
    if (nimg > 1 && (__int128)m.off + (__int128)(nimg - 1) * m.s0 + one >
                        (__int128)(m.buf->bytes / es)) {
        fail("%s: %s: %d images of %ld x %d (pitch %d, %ld apart) pass the buffer of %zu bytes",
             fn, what, nimg, HW, C, m.ld, m.s0, m.buf->bytes);
        return false;
    }
    return true;
}

}  // namespace
}  // namespace coreg

extern "C" size_t ops_groupnorm_cl_bytes(int nimg, long HW, int C, int groups)
{
    (void)nimg;
    (void)HW;
    (void)C;
    (void)groups;
    return 0;
}

extern "C" void ops_groupnorm_cl(struct ops *o, int nimg, long HW, int C, int groups,
                                 struct opnd X, int xtype, struct opnd Y, int ytype, cl_mem g,
                                 cl_mem b, float eps, int act, float slope, cl_mem work)
{
    const char *fn = "ops_groupnorm_cl";
    View x, y, vg, vb;

    (void)work;
    if (pending() || !type_ok(fn, xtype) || !type_ok(fn, ytype) || !act_ok(fn, act))
        return;
    if (nimg < 0 || HW < 0 || C < 0 || groups < 1 || C % groups || nimg > 65535) {
        fail("%s: %d maps of %ld x %d in %d groups", fn, nimg, HW, C, groups);
        return;
    }
    if (!(eps >= 0.0f)) {
        fail("%s: eps %g", fn, (double)eps);
        return;
    }
    if (!g != !b) {
        fail("%s: gamma without beta", fn);
        return;
    }
    if (nimg == 0 || HW == 0 || C == 0)
        return;
    if (!map_view(&x, fn, "X", X, nimg, HW, C, type_size(xtype), false) ||
        !map_view(&y, fn, "Y", Y, nimg, HW, C, type_size(ytype), true) ||
        (g && (!view_of(&vg, fn, "gamma", g, 0, C, 1, C, 4) ||
               !view_of(&vb, fn, "beta", b, 0, C, 1, C, 4))))
        return;
    const bool in_place = same_view(x, y) && (nimg == 1 || X.s0 == Y.s0);
    const long nx = x.span() + (nimg - 1) * X.s0 * x.es, ny = y.span() + (nimg - 1) * Y.s0 * y.es;
    if ((!in_place && ranges_meet(x.p, nx, y.p, ny)) || (g && (ranges_meet(vg.p, C * 4L, y.p, ny) ||
                                                              ranges_meet(vb.p, C * 4L, y.p, ny)))) {
        fail("%s: the output overlaps an input", fn);
        return;
    }
    OnDevice dev(o->ocl);
    if (!dev.ok)
        return;
    const GroupNorm p = {nimg, C, groups, HW, x.p, X.ld, X.s0, y.p, Y.ld, Y.s0, (const float *)vg.p,
                         (const float *)vb.p, eps, act, slope};
    const dim3 grid(groups, nimg);
    cudaStream_t st = stream_of(o->ocl);
    Prof pr(o->ocl, "groupnorm_cl");
    if (xtype == OPS_BF16 && ytype == OPS_BF16)
        group_k<__nv_bfloat16, __nv_bfloat16><<<grid, 256, 0, st>>>(p);
    else if (xtype == OPS_BF16)
        group_k<__nv_bfloat16, float><<<grid, 256, 0, st>>>(p);
    else if (ytype == OPS_BF16)
        group_k<float, __nv_bfloat16><<<grid, 256, 0, st>>>(p);
    else
        group_k<float, float><<<grid, 256, 0, st>>>(p);
    launch_ok("groupnorm_cl");
}
