// SPDX-License-Identifier: Unlicense
//
// Group norm with an activation over channels-last maps (ops_b200.h):
// ops_groupnorm_cl.

#include <cooperative_groups.h>

#include "opcheck.cuh"
#include "tc_common.cuh"

using namespace coreg;
namespace cg = cooperative_groups;

namespace coreg {
namespace {

// A team of blocks normalises one slice of an image: the pixels of
// neighbouring groups (all of them where not stated). A block takes a run of
// pixels, a thread a fixed vector of channels in every lanes-th of them, so
// that statistics and coefficients stay in its registers:
//   1. per thread and channel the mean and M2 (sum of squares about the mean),
//      from sums about the mean of its first eight values; every FOLD vectors
//      they are joined to a mean and M2 of two floats each and begun again, so
//      that no chain of roundings is longer than 8 + FOLD / 8 however many
//      vectors a thread has, and an outlier among the eight costs M2 no more
//      than some steps of its own square; the vectors read stay in shared
//      memory as far as they fit;
//   2. the block's mean and M2 per group from its threads', the team's from
//      its blocks': weighted means first, then squares about them, so that
//      nothing cancels;
//   3. the result from the kept vectors; what did not fit is read again, last
//      read first (from L2 where the team's share fits there).
// Channel counts whose rows are no whole number of vectors: R rows of a
// packed map form one row of W = R C elements that is.
// Division of n < 2^16 by a fixed d < 2^16: the high word of n ceil(2^32 / d),
// whose error n / 2^32 stays below the 1 / d that an integer quotient is from
// the next. (Divisions in full are chains of some 150 cycles; they were most
// of a small map's time.)
struct Div {
    uint32_t m; // 0: d = 1
    __host__ void set(int d) { m = d == 1 ? 0 : (uint32_t)((0x100000000ull + d - 1) / d); }
    __device__ __forceinline__ int operator()(int n) const
    {
        return m ? (int)__umulhi((uint32_t)n, m) : n;
    }
};

struct GroupNorm {
    int nimg, C, groups, per; // per: channels of a group
    int HW;
    const void *X;
    long ldx, sx;
    void *Y;
    long ldy, sy;
    const float *g, *b;
    float eps;
    int act;
    float slope;
    int R, gs, slices;    // rows per super row, groups per slice, slices
    int slots, lanes;     // vectors of a super row's slice, rows in flight
    int nsr, wlast;       // super rows; elements of the last
    int team;             // blocks per team
    int run, run_rem;     // super rows per block, one more in the first run_rem
    int base, more;       // of run: run / lanes, run % lanes
    int cols, pitch;      // a group's entries per row lane, entries between lanes
    Div by_slots, by_per, by_C;
    int keep, ring;       // vectors a thread keeps, places of the ring (RING or 0)
    int merged;           // neighbouring channels of a thread in one entry
    int simple;           // all of a thread's, and gamma and beta 16-byte aligned
    int fold;             // entries that a thread folds into: 0 with at most FOLD vectors
    int batch;            // grid teams: images at a time, a team each
    float2 *work;         // grid teams: 2 x batch x groups x team (mean, M2)
};

constexpr int MAX_THREADS = 512;
// Vectors of a thread in flight: 8 x 512 x 16 bytes per multiprocessor cover
// the memory's latency at its full rate (about 45 KB) with some to spare.
constexpr int RING = 8;
// Vectors whose sums are folded together. (Threads of most maps have fewer.)
constexpr int FOLD = 128;
constexpr int MAX_TEAM = 160; // blocks of a grid team the work buffer holds


// V values as they lie in memory: 16 bytes, or one value.
template <typename T, int V>
struct Vec {
    typedef uint4 Kept;
    uint4 w;
    __device__ __forceinline__ float at(int e) const
    {
        const int i = sizeof(T) == 4 ? e : e / 2;
        const uint32_t x = i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w;
        return __uint_as_float(sizeof(T) == 4 ? x : e % 2 ? x & 0xffff0000u : x << 16);
    }
    __device__ __forceinline__ void load(const T *p) { w = *(const uint4 *)p; }
    __device__ __forceinline__ void keep(Kept *k) const { *k = w; }
    __device__ __forceinline__ void back(const Kept *k) { w = *k; }
};

template <typename T>
struct Vec<T, 1> {
    typedef T Kept;
    float f;
    __device__ __forceinline__ float at(int) const { return f; }
    __device__ __forceinline__ void load(const T *p) { f = ldf(p); }
    __device__ __forceinline__ void keep(Kept *k) const { stf(k, f); }
    __device__ __forceinline__ void back(const Kept *k) { f = ldf(k); }
};

// STREAM: results of a map beyond what L2 holds, marked to leave it first
// (they are not read again here, the map's rest is).
template <int V, bool STREAM>
__device__ __forceinline__ void store_vec(float *p, const float f[V])
{
    if constexpr (V % 4 == 0) {
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            const float4 v = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
            if (STREAM)
                __stcs((float4 *)(p + e), v);
            else
                *(float4 *)(p + e) = v;
        }
    }
    else {
        *p = f[0];
    }
}

template <int V, bool STREAM>
__device__ __forceinline__ void store_vec(__nv_bfloat16 *p, const float f[V])
{
    if constexpr (V % 4 == 0) {
        uint32_t w[V / 2];
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[e], f[e + 1]);
            w[e / 2] = *(const uint32_t *)&h;
        }
        if constexpr (V == 8) {
            if (STREAM)
                __stcs((uint4 *)p, make_uint4(w[0], w[1], w[2], w[3]));
            else
                *(uint4 *)p = make_uint4(w[0], w[1], w[2], w[3]);
        }
        else {
            if (STREAM)
                __stcs((uint2 *)p, make_uint2(w[0], w[1]));
            else
                *(uint2 *)p = make_uint2(w[0], w[1]);
        }
    }
    else {
        *p = __float2bfloat16_rn(f[0]);
    }
}

// Where a thread works: its elements j0 .. j0 + V - 1 of the super rows first +
// i lanes, i < cnt; and the first tail elements of one more, the map's end.
struct Place {
    int first, cnt, j0, tail;
};

// First super row of block t of a team (the end of the last for what is behind it:
// t * run stays within the map's).
__device__ __forceinline__ int run_start(const GroupNorm &p, int t)
{
    t = min(t, p.team);
    return t * p.run + min(t, p.run_rem);
}

template <typename T>
__device__ __forceinline__ T *at_row(T *x, long ld, const GroupNorm &p, const Place &at, int i)
{
    return x + (long)(at.first + i * p.lanes) * (p.R * ld) + at.j0;
}

// Bytes of the vectors that the threads of a block keep.
__host__ __device__ inline size_t kept_bytes(const GroupNorm &p, int threads, size_t vec)
{
    return ((size_t)(p.keep + p.ring) * threads * vec + 15) / 16 * 16;
}

// Bytes of the block's entries, its (mean, M2) per group and the team's.
__host__ __device__ inline size_t entry_bytes(const GroupNorm &p)
{
    return ((size_t)p.pitch * p.lanes * 8 + (size_t)p.gs * 16 + 15) / 16 * 16;
}

// Asynchronous copy of 16 bytes into shared memory, by this thread for
// itself: no barrier, only its own groups.
__device__ __forceinline__ void fetch16(void *dst, const void *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(tc::su32(dst)), "l"(src)
                 : "memory");
}

__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void fetch_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Shared-memory place of a thread's i-th vector: the first p.keep have their
// own, the others take turns in a ring of RING behind them.
__device__ __forceinline__ int place_of(const GroupNorm &p, int i)
{
    return (i < p.keep ? i : p.keep + (i - p.keep) % RING) * (int)blockDim.x;
}

// The first RING copies of `sums`.
template <typename TX, int V>
__device__ __forceinline__ void sums_begin(const GroupNorm &p, const TX *x, const Place &at,
                                           typename Vec<TX, V>::Kept *kept)
{
    if constexpr (V > 1) {
        const TX *q = at_row(x, p.ldx, p, at, 0);
        const long step = p.lanes * (p.R * p.ldx);
#pragma unroll
        for (int i = 0; i < RING; i++) {
            if (i < at.cnt)
                fetch16(kept + place_of(p, i), q + i * step);
            fetch_commit();
        }
    }
}

// M2 from the sums s1 and s2 about another point, m that point's distance from
// the mean: not below zero by rounding, but infinite where s2 has passed
// float's range (the group then has an infinite variance, not one of zero),
// and NaN where a value is.
__device__ __forceinline__ float about_mean(float s1, float s2, float m)
{
    const float q = s2 - s1 * m;
    return q >= 0.0f ? q : q < 0.0f ? 0.0f : s2;
}

// The means and M2 of n values each, in the place of their sums s1 and s2 about x0.
template <int V, typename F>
__device__ __forceinline__ void settle(const float x0[V], float s1[V], float s2[V], F inv)
{
#pragma unroll
    for (int e = 0; e < V; e++) {
        const float m = s1[e] * inv(e);
        s2[e] = about_mean(s1[e], s2[e], m);
        s1[e] = x0[e] + m;
    }
}

// put(k, mean, M2) of K neighbouring of a thread's V channels each, which have
// n values each.
template <int V, int K, typename F>
__device__ __forceinline__ void merge(const float mean[V], const float m2[V], float n, F put)
{
#pragma unroll
    for (int e = 0; e < V; e += K) {
        float m = mean[e], q = m2[e];
        if (K > 1) {
#pragma unroll
            for (int k = 1; k < K; k++)
                m += mean[e + k];
            m *= 1.0f / K;
            q = 0.0f;
#pragma unroll
            for (int k = 0; k < K; k++) {
                const float d = mean[e + k] - m;
                q += fmaf(n * d, d, m2[e + k]);
            }
        }
        put(e / K, m, q);
    }
}

// The same for p.merged neighbouring channels that lie in one group (all of a
// thread's, four, two or one).
template <int V, typename F>
__device__ __forceinline__ void entries(const GroupNorm &p, const float mean[V],
                                        const float m2[V], float n, F put)
{
    if (V > 1 && p.merged == V)
        merge<V, V>(mean, m2, n, put);
    else if (V == 8 && p.merged == 4)
        merge<V, 4>(mean, m2, n, put);
    else if (V > 2 && p.merged == 2)
        merge<V, 2>(mean, m2, n, put);
    else
        merge<V, 1>(mean, m2, n, put);
}

// v added to hi + lo, lo the rounding errors of hi.
__device__ __forceinline__ void add_up(float &hi, float &lo, float v)
{
    const float s = hi + v, z = s - hi, e = (hi - (s - z)) + (v - z);
    lo = fabsf(s) < INFINITY ? lo + e : 0.0f;
    hi = s;
}

// (m, q) of some vectors of p.merged channels joined to the (mean, M2) of `before`
// vectors in an entry, whose rounding errors are at `rest`: two floats hold
// what one would lose over hundreds of joins (doubles took 4 us of 105 at 132
// vectors a thread, by their conversions). w: the new vectors' share of all;
// last: the entry is complete.
__device__ __forceinline__ void join(const GroupNorm &p, float2 *entry, float2 *rest, int before,
                                     float m, float q, float w, bool last)
{
    float2 hi = make_float2(m, q), lo = make_float2(0.0f, 0.0f);
    if (before) {
        hi = *entry;
        lo = *rest;
        const float d = (m - hi.x) - lo.x;
        add_up(hi.x, lo.x, d * w);
        add_up(hi.y, lo.y, fmaf(d * d, w * (float)(before * p.merged), q));
    }
    if (last)
        hi = make_float2(hi.x + lo.x, hi.y + lo.y);
    else
        *rest = lo;
    *entry = hi;
}

// Vectors of a thread that are folded when its sums end: whole FOLDs, at
// least one vector left.
__device__ __forceinline__ int folded(int cnt) { return cnt > FOLD ? (cnt - 1) / FOLD * FOLD : 0; }

// The sums of a thread's FOLD vectors into its entries from `to` on; `before` are
// in there.
template <int V>
__device__ __forceinline__ void fold_sums(const GroupNorm &p, const float x0[V], float s1[V],
                                          float s2[V], int before, float2 *to, float2 *rest)
{
    const float w = (float)FOLD / (float)(before + FOLD);
    settle<V>(x0, s1, s2, [](int) { return 1.0f / FOLD; });
    entries<V>(p, s1, s2, (float)FOLD, [&](int k, float m, float q) {
        join(p, to + k, rest + k * (int)blockDim.x, before, m, q, w, false);
    });
}

// The sums t1 and t2 about x0 as the first of a run: of eight values they are
// taken on to their mean, about which the following ones are added.
template <int V>
__device__ __forceinline__ void begin_sums(float x0[V], float s1[V], float s2[V],
                                           const float t1[V], const float t2[V], bool eight)
{
    const float w = eight ? 0.125f : 0.0f, n = eight ? 8.0f : 0.0f;
#pragma unroll
    for (int e = 0; e < V; e++) {
        const float c = fmaf(w, t1[e], x0[e]), d = c - x0[e];
        s1[e] = fmaf(-n, d, t1[e]);
        s2[e] = fmaf(-d, t1[e] + s1[e], t2[e]); // n d = t1 - s1
        x0[e] = c;
    }
}

// Sums of x - x0 and of its square over a thread's vectors (those behind the
// folded ones), eight at a time so that no chain of additions is longer than
// 8 + FOLD / 8. Leaves the vectors in shared memory: the first p.keep, and the
// last RING of the others.
template <typename TX, int V, bool FOLDED>
__device__ __forceinline__ void sums(const GroupNorm &p, const TX *x, const Place &at, float x0[V],
                                     float s1[V], float s2[V], typename Vec<TX, V>::Kept *kept,
                                     float2 *to, float2 *rest)
{
    const TX *q = at_row(x, p.ldx, p, at, 0);
    const long step = p.lanes * (p.R * p.ldx);
#pragma unroll
    for (int e = 0; e < V; e++)
        x0[e] = s1[e] = s2[e] = 0.0f;
    if constexpr (V > 1)
        q += RING * step;
    // The sums of the vectors i0 .. i1 - 1 (at most eight); first: about the first.
    float t1[V], t2[V];
    auto batch = [&](int i0, int i1, bool first) {
#pragma unroll
        for (int e = 0; e < V; e++)
            t1[e] = t2[e] = 0.0f;
        if constexpr (V == 1) {
            Vec<TX, V> r[8];
#pragma unroll
            for (int u = 0; u < 8; u++)
                if (i0 + u < i1)
                    r[u].load(q + u * step);
            q += 8 * step;
            if (first)
                x0[0] = r[0].at(0);
#pragma unroll
            for (int u = 0; u < 8; u++)
                if (i0 + u < i1) {
                    if (i0 + u < p.keep)
                        r[u].keep(kept + (i0 + u) * blockDim.x);
                    const float d = r[u].at(0) - x0[0];
                    t1[0] += d;
                    t2[0] = fmaf(d, d, t2[0]);
                }
        }
        else {
            for (int i = i0; i < i1; i++, q += step) {
                fetch_wait<RING - 1>();
                Vec<TX, V> r;
                r.back(kept + place_of(p, i));
                if (first && i == i0) {
#pragma unroll
                    for (int e = 0; e < V; e++)
                        x0[e] = r.at(e);
                }
#pragma unroll
                for (int e = 0; e < V; e++) {
                    const float d = r.at(e) - x0[e];
                    t1[e] += d;
                    t2[e] = fmaf(d, d, t2[e]);
                }
                // Into a place of its own, or that of vector i, just read.
                if (i + RING < at.cnt)
                    fetch16(kept + place_of(p, i + RING), q);
                fetch_commit();
            }
        }
    };
    for (int c0 = 0; c0 < at.cnt; c0 += FOLD) {
        const int c1 = FOLDED ? min(c0 + FOLD, at.cnt) : at.cnt;
        batch(c0, min(c0 + 8, c1), true);
        begin_sums<V>(x0, s1, s2, t1, t2, c1 - c0 >= 8);
        for (int i0 = c0 + 8; i0 < c1; i0 += 8) {
            batch(i0, min(i0 + 8, c1), false);
#pragma unroll
            for (int e = 0; e < V; e++) {
                s1[e] += t1[e];
                s2[e] += t2[e];
            }
        }
        if (!FOLDED)
            break;
        if (c1 < at.cnt)
            fold_sums<V>(p, x0, s1, s2, c0, to, rest);
    }
    if constexpr (V > 1) {
        if (at.tail > 0) {
            const TX *t = at_row(x, p.ldx, p, at, at.cnt);
#pragma unroll
            for (int e = 0; e < V; e++)
                if (e < at.tail) {
                    const float v = ldf(t + e);
                    if (at.cnt == 0)
                        x0[e] = v;
                    const float d = v - x0[e];
                    s1[e] += d;
                    s2[e] = fmaf(d, d, s2[e]);
                }
        }
    }
}

template <int ACT, typename TX, typename TY, int V, bool GRID>
__device__ __forceinline__ void apply(const GroupNorm &p, const TX *x, TY *y, const Place &at,
                                      const float mean[V], const float a[V], const float b[V],
                                      typename Vec<TX, V>::Kept *kept)
{
    const long sx = p.lanes * (p.R * p.ldx), sy = p.lanes * (p.R * p.ldy);
    int i = at.cnt - 1;
    TY *w = at_row(y, p.ldy, p, at, i);
    auto act = [&](float v) { return act2<ACT, true>(make_float2(v, 0.0f), p.slope).x; };
    auto one = [&](const Vec<TX, V> &r, TY *to) {
        float f[V];
        if constexpr (V == 1)
            f[0] = act(fmaf(r.at(0) - mean[0], a[0], b[0]));
        else {
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                const float2 v = act2<ACT, true>(
                    make_float2(fmaf(r.at(e) - mean[e], a[e], b[e]),
                                fmaf(r.at(e + 1) - mean[e + 1], a[e + 1], b[e + 1])),
                    p.slope);
                f[e] = v.x;
                f[e + 1] = v.y;
            }
        }
        store_vec<V, GRID>(to, f);
    };
    // Last read first: what was not kept is likeliest in L2.
    if constexpr (V == 1) {
        constexpr int U = 8;
        const TX *q = at_row(x, p.ldx, p, at, i);
        for (; i >= 0; i -= U, q -= U * sx, w -= U * sy) {
            Vec<TX, V> r[U];
#pragma unroll
            for (int u = 0; u < U; u++)
                if (i - u >= p.keep)
                    r[u].load(q - u * sx);
                else if (i - u >= 0)
                    r[u].back(kept + (i - u) * blockDim.x);
#pragma unroll
            for (int u = 0; u < U; u++)
                if (i - u >= 0)
                    one(r[u], w - u * sy);
        }
    }
    else {
        const TX *q = at_row(x, p.ldx, p, at, i - RING);
        for (; i >= p.keep; i--, q -= sx, w -= sy) {
            fetch_wait<RING - 1>();
            typename Vec<TX, V>::Kept *k = kept + place_of(p, i);
            Vec<TX, V> r;
            r.back(k);
            one(r, w);
            if (i - RING >= p.keep)
                fetch16(k, q);
            fetch_commit();
        }
        for (; i >= 0; i--, w -= sy) {
            Vec<TX, V> r;
            r.back(kept + i * (int)blockDim.x);
            one(r, w);
        }
        if (at.tail > 0) {
            const TX *t = at_row(x, p.ldx, p, at, at.cnt);
            TY *to = at_row(y, p.ldy, p, at, at.cnt);
#pragma unroll
            for (int e = 0; e < V; e++)
                if (e < at.tail)
                    stf(to + e, act(fmaf(ldf(t + e) - mean[e], a[e], b[e])));
        }
    }
}

// How a warp walks a group's entries: lane l takes the columns l % pw, + pw, ...
// of `cols`, and of each the rows l / pw, + 32 / pw, ... (pw a power of two), so
// that the loops hold no division. visit(column, row).
template <typename F>
__device__ __forceinline__ void walk(int cols, int lanes, int lane, F visit)
{
    const int s = cols >= 32 ? 5 : 32 - __clz(cols - 1), pw = 1 << s; // cols 1: s = 0
    for (int c = lane & (pw - 1); c < cols; c += pw)
        for (int r = lane >> s; r < lanes; r += 32 >> s)
            visit(c, r);
}

// GRID: all blocks at once (a cooperative launch) in teams of a batch of images,
// batches one after the other; otherwise a team is a cluster, one per image
// and slice. FOLDED: threads with more than FOLD vectors. (Within one kernel the
// code for them cost the others 0.1 to 0.7 us.)
template <typename TX, typename TY, int V, bool GRID, bool FOLDED>
__global__ void __launch_bounds__(MAX_THREADS, 1)
groupnorm_k(const __grid_constant__ GroupNorm p)
{
    extern __shared__ __align__(16) unsigned char smem[];
    const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, nwarp = blockDim.x / 32;
    typename Vec<TX, V>::Kept *kept = (typename Vec<TX, V>::Kept *)smem + tid;
    float2 *entry = (float2 *)(smem + kept_bytes(p, blockDim.x, sizeof(*kept)));
    float2 *mine = entry + p.pitch * p.lanes; // the block's (mean, M2) per group
    float2 *team = mine + p.gs;               // the team's (mean, 1 / sigma)
    float2 *rest = (float2 *)((unsigned char *)entry + entry_bytes(p)) + tid; // (if p.fold)
    // (The blocks of a cluster team are a power of two.)
    const int which = GRID ? (int)blockIdx.x / p.team : 0; // the team's image of a batch
    const int rank = GRID ? (int)blockIdx.x - which * p.team : (int)(blockIdx.x & (p.team - 1));
    const int slice = GRID ? 0 : (int)blockIdx.x >> (31 - __clz(p.team));
    const int g0 = slice * p.gs, gn = min(p.gs, p.groups - g0); // its groups
    const int c0 = g0 * p.per;
    const int W = p.slots * V, width = p.R > 1 ? W : gn * p.per;

    const int sr0 = run_start(p, rank), sr1 = run_start(p, rank + 1), rows = sr1 - sr0;
    const int row = p.by_slots(tid), slot = tid - row * p.slots;
    // Super rows of a row lane: base, one more in the first `more`.
    int base = p.base, more = p.more;
    if (rows > p.run && ++more == p.lanes) {
        base++;
        more = 0;
    }
    const bool active = row < p.lanes && slot * V < width;
    Place at;
    at.first = sr0 + row;
    at.cnt = active ? base + (row < more) : 0;
    at.j0 = slot * V;
    at.tail = 0;
    if (at.cnt > 0 && at.first + (at.cnt - 1) * p.lanes == p.nsr - 1 && at.j0 + V > p.wlast) {
        at.cnt--;
        at.tail = max(p.wlast - at.j0, 0);
    }
    // The row lane that holds the map's last super row, -1 if none here.
    const int last = sr1 == p.nsr && rows > 0 ? (more > 0 ? more : p.lanes) - 1 : -1;

    if (!GRID)
        after_previous();
    for (int img0 = GRID ? 0 : (int)blockIdx.y; img0 < p.nimg; img0 += GRID ? p.batch : p.nimg) {
        const int img = img0 + which;
        // (A last batch may have fewer images than teams.)
        if (GRID && img >= p.nimg) {
            cg::this_grid().sync();
            continue;
        }
        const TX *x = (const TX *)p.X + img * p.sx + c0;
        TY *y = (TY *)p.Y + img * p.sy + c0;

        // 1. The threads' sums; meanwhile gamma and beta into registers.
        sums_begin<TX, V>(p, x, at, kept);
        float ga[V], be[V];
        int gi[V]; // the elements' groups
        if (V > 1 && p.simple) {
            // Whole vectors of one group, gamma and beta aligned as the map is.
            const int g = active ? p.by_per(at.j0) : 0;
#pragma unroll
            for (int e = 0; e < V; e++) {
                gi[e] = g;
                ga[e] = 1.0f;
                be[e] = 0.0f;
            }
            if (p.g && active)
#pragma unroll
                for (int e = 0; e < V; e += 4) {
                    const float4 u = *(const float4 *)(p.g + c0 + at.j0 + e),
                                 v = *(const float4 *)(p.b + c0 + at.j0 + e);
                    ga[e] = u.x, ga[e + 1] = u.y, ga[e + 2] = u.z, ga[e + 3] = u.w;
                    be[e] = v.x, be[e + 1] = v.y, be[e + 2] = v.z, be[e + 3] = v.w;
                }
        }
        else
#pragma unroll
            for (int e = 0; e < V; e++) {
                const int j = at.j0 + e, c = p.R > 1 ? j - p.by_C(j) * p.C : j;
                const bool in = active && j < width;
                gi[e] = in ? p.by_per(c) : 0;
                ga[e] = in && p.g ? p.g[c0 + c] : 1.0f;
                be[e] = in && p.g ? p.b[c0 + c] : 0.0f;
            }
        {
            float x0[V], s1[V], s2[V];
            float2 *to = entry + row * p.pitch + (at.j0 >> (31 - __clz(p.merged)));
            sums<TX, V, FOLDED>(p, x, at, x0, s1, s2, kept, to, rest);
            // 2. The thread's entries (mean, M2).
            if (active) {
                const int before = FOLDED ? folded(at.cnt) : 0, left = at.cnt - before;
                const float i0 = left > 0 ? 1.0f / (float)left : 0.0f,
                            i1 = at.tail > 0 ? 1.0f / (float)(left + 1) : 0.0f;
                settle<V>(x0, s1, s2, [&](int e) { return e < at.tail ? i1 : i0; });
                if (before == 0)
                    entries<V>(p, s1, s2, (float)left,
                               [&](int k, float m, float q) { to[k] = make_float2(m, q); });
                else {
                    // (With a tail a thread's entries are single channels.)
                    const float w0 = (float)left / (float)at.cnt,
                                w1 = (float)(left + 1) / (float)(at.cnt + 1);
                    entries<V>(p, s1, s2, (float)left, [&](int k, float m, float q) {
                        join(p, to + k, rest + k * (int)blockDim.x, before, m, q,
                             k < at.tail ? w1 : w0, true);
                    });
                }
            }
        }
        __syncthreads();
        float2 *out = GRID ? p.work + (size_t)((img0 / p.batch & 1) * p.batch + which) *
                                          p.groups * p.team
                           : nullptr;
        const float here = (float)(((long)min((long)sr1 * p.R, (long)p.HW) - (long)sr0 * p.R) * p.per);
        // Entries of a group: p.cols in a row lane, p.pitch between row lanes;
        // each of (base, or base + 1 in the first `more` row lanes) pixels of
        // p.merged channels, one less where the map's last super row ends.
        // Sums about the group's first entry, one of those added.
        for (int g = warp; g < gn; g += nwarp) {
            const float m0 = entry[p.R > 1 ? g * p.per : g * p.cols].x;
            float a = 0.0f, q = 0.0f;
            walk(p.cols, p.lanes, lane, [&](int c, int r) {
                int j = g * p.cols + c, n = base + (r < more);
                if (p.R > 1) {
                    const int k = p.by_per(c);
                    j = k * p.C + g * p.per + (c - k * p.per);
                    n -= r == last && j >= p.wlast;
                }
                const float2 v = entry[r * p.pitch + j];
                const float w = (float)(n * p.merged), d = v.x - m0;
                if (n > 0) {
                    a = fmaf(w, d, a);
                    q += fmaf(w * d, d, v.y);
                }
            });
            a = warp_sum(a);
            q = warp_sum(q);
            if (lane == 0) {
                const float m = here > 0.0f ? a / here : 0.0f;
                const float2 s = make_float2(m0 + m, about_mean(a, q, m));
                if (GRID)
                    out[(size_t)g * p.team + rank] = s;
                else
                    mine[g] = s;
            }
        }
        if (GRID)
            cg::this_grid().sync();
        else if (p.team > 1)
            cg::this_cluster().sync();
        else
            __syncthreads();
        // The team's statistics: a warp per group, a lane per block, whose
        // parts stay in registers for both passes.
        constexpr int NP = GRID ? MAX_TEAM / 32 : 1;
        const float N = (float)((double)p.HW * p.per);
        float n[NP]; // values of a group in the lane's blocks
#pragma unroll
        for (int k = 0; k < NP; k++) {
            const int t = lane + 32 * k;
            const long a = (long)run_start(p, t) * p.R, b = (long)run_start(p, t + 1) * p.R;
            n[k] = t < p.team ? (float)((min(b, (long)p.HW) - a) * p.per) : 0.0f;
        }
        auto parts = [&](int g, float2 part[NP]) {
#pragma unroll
            for (int k = 0; k < NP; k++) {
                const int t = lane + 32 * k;
                part[k] = make_float2(0.0f, 0.0f);
                if (t < p.team && g < gn) {
                    if (GRID)
                        part[k] = __ldcg(&out[(size_t)g * p.team + t]);
                    else
                        part[k] = p.team > 1 ? cg::this_cluster().map_shared_rank(mine, t)[g] : mine[g];
                }
            }
        };
        float2 part[NP];
        parts(warp, part);
        for (int g = warp; g < gn; g += nwarp) {
            float2 next[NP];
            parts(g + nwarp, next);
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < NP; k++)
                s = fmaf(part[k].x, n[k], s);
            const float m = warp_sum(s) / N;
            s = 0.0f;
#pragma unroll
            for (int k = 0; k < NP; k++) {
                const float d = part[k].x - m;
                if (n[k] > 0.0f)
                    s += fmaf(n[k] * d, d, part[k].y);
                part[k] = next[k];
            }
            s = warp_sum(s) / N;
            if (lane == 0)
                team[g] = make_float2(m, rsqrtf(s + p.eps));
        }
        __syncthreads();
        // 3. The result.
        if (active) {
            float mean[V];
#pragma unroll
            for (int e = 0; e < V; e++) {
                const float2 q = team[gi[e]];
                mean[e] = q.x;
                ga[e] *= q.y;
            }
            switch (p.act) {
            case ACT_GELU:
                apply<ACT_GELU, TX, TY, V, GRID>(p, x, y, at, mean, ga, be, kept);
                break;
            case ACT_RELU:
                apply<ACT_RELU, TX, TY, V, GRID>(p, x, y, at, mean, ga, be, kept);
                break;
            case ACT_LEAKY:
                apply<ACT_LEAKY, TX, TY, V, GRID>(p, x, y, at, mean, ga, be, kept);
                break;
            case ACT_GELU_TANH:
                apply<ACT_GELU_TANH, TX, TY, V, GRID>(p, x, y, at, mean, ga, be, kept);
                break;
            case ACT_SILU:
                apply<ACT_SILU, TX, TY, V, GRID>(p, x, y, at, mean, ga, be, kept);
                break;
            default:
                apply<ACT_NONE, TX, TY, V, GRID>(p, x, y, at, mean, ga, be, kept);
            }
        }
        if (GRID)
            __syncthreads(); // entries and the team's statistics are reused
    }
    // No block leaves while another may still read its statistics.
    if (!GRID && p.team > 1)
        cg::this_cluster().sync();
}

// Sum over a block of 256 threads; every thread gets it.
__device__ double block_total(double v, double *red)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0)
        red[threadIdx.x / 32] = v;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < 8; w++)
        t += red[w];
    return t;
}

// One block per group of an image, three passes over it: groups wider than
// a block's threads hold vectors of. A thread adds up its whole share, of any
// length, so the sums are held in 64 bits: in float32 chains of 140 thousand
// values (46657 x 771, one group) of mean 1003 and sigma 1 the mean was off by
// half a sigma. Pixel and column advance without the two divisions an element
// that an index over the group would take.
template <typename TX, typename TY>
__global__ void __launch_bounds__(256)
group_k(const GroupNorm p)
{
    __shared__ double red[8];
    const int per = p.per, img = blockIdx.y, c0 = blockIdx.x * per;
    const TX *x = (const TX *)p.X + img * p.sx + c0;
    TY *y = (TY *)p.Y + img * p.sy + c0;
    const double n = (double)p.HW * per;
    // visit(pixel, column) of the thread's values.
    auto each = [&](auto visit) {
        int c = threadIdx.x;
        for (long r = 0;; c += 256) {
            while (c >= per) {
                c -= per;
                r++;
            }
            if (r >= p.HW)
                return;
            visit(r, c);
        }
    };
    double s = 0.0;
    each([&](long r, int c) { s += (double)ldf(x + r * p.ldx + c); });
    const double center = block_total(s, red) / n;
    s = 0.0;
    each([&](long r, int c) {
        const double d = (double)ldf(x + r * p.ldx + c) - center;
        s = fma(d, d, s);
    });
    const float mean = (float)center;
    const float rstd = rsqrtf((float)(block_total(s, red) / n) + p.eps);
    each([&](long r, int c) {
        float v = (ldf(x + r * p.ldx + c) - mean) * rstd;
        if (p.g)
            v = v * p.g[c0 + c] + p.b[c0 + c];
        stf(y + r * p.ldy + c, act_any(v, p.act, p.slope));
    });
}

constexpr size_t SMEM = 227 * 1024;

size_t smem_bytes(const GroupNorm &p, int threads, int vec_bytes)
{
    return kept_bytes(p, threads, vec_bytes) + entry_bytes(p) +
           (size_t)p.fold * threads * sizeof(float2);
}

// Clusters of `team` blocks that the device holds at once, one block to a
// multiprocessor (a team's blocks are those of one GPC: 15 of 8, not 18).
int clusters_of(const void *fn, int team, int sms)
{
    static PerDevice known[3];
    if (team == 1)
        return sms;
    return known[team == 2 ? 0 : team == 4 ? 1 : 2].get([&] {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(sms / team * team);
        cfg.blockDim = dim3(MAX_THREADS);
        cfg.dynamicSmemBytes = SMEM;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = team;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess || n < 1) {
            cudaGetLastError();
            n = sms / team > 1 ? sms / team - 1 : 1;
        }
        return n;
    });
}

template <typename TX, typename TY, int V>
bool launch(cudaStream_t st, GroupNorm p, int sms)
{
    static unsigned done[4] = {0, 0, 0, 0};
    constexpr int vb = (int)sizeof(TX) * V;
    p.R = 1;
    while (p.R < V && (long)p.R * p.C % V)
        p.R *= 2;
    p.nsr = (p.HW + p.R - 1) / p.R;
    p.batch = 1;
    p.merged = p.R > 1                       ? 1
               : p.per % V == 0              ? V
               : p.per % 4 == 0 && V == 8    ? 4
               : p.per % 2 == 0 && V > 2     ? 2
                                             : 1;
    p.simple = p.merged == V && (((uintptr_t)p.g | (uintptr_t)p.b) & 15) == 0;
    p.by_per.set(p.per < 65536 ? p.per : 65535);
    p.by_C.set(p.C < 65536 ? p.C : 65535); // (wider maps have R = 1)
    p.cols = p.R > 1 ? p.per * p.R : p.per / p.merged;
    // Slices of whole groups whose vectors start aligned: the smallest unit.
    int unit = 1;
    while (unit < p.groups && (p.R > 1 || (long)unit * p.per % V))
        unit++;
    if (p.R > 1)
        unit = p.groups;
    // Groups whose slots fit a block. (In 64 bits: eight rows of 2^29 + 1 channels
    // are eight in 32.)
    const int gmax = (int)((long)MAX_THREADS * V / ((long)p.R * p.per));
    if (unit > gmax && p.groups > gmax)
        return false;
    p.wlast = (p.HW - (p.nsr - 1) * p.R) * p.C; // (with R > 1 all channels fit a block)

    // Every slice width and team size, and grid teams; times in microseconds by
    // a model: memory at 6.5 MB per microsecond over the whole device, at most
    // 1.5 times an even share per multiprocessor; what is read again from L2
    // at twice that where the maps under way are below 110 MB, else from memory,
    // which costs 1.8 times its bytes over the grid and 2.6 in clusters, whose
    // passes mix; 0.7 of the rate for slices, which leave parts of memory's
    // rows; and the chain of barrier and statistics (4 us in a cluster, 9
    // over the grid). Measured: two maps of 864 x 864 x 64 bfloat16
    // one after the other 89 us, at a time 97; five of 71428 x 252 float32 170
    // and 186 (two at a time), in clusters 223; six of 46656 x 64 bfloat16
    // 56 and 29 (three at a time), in clusters 26.
    const double esz = sizeof(TX), eout = sizeof(TY);
    auto model = [&](double elems, double again, double blocks, double far) {
        const double f = blocks * 1.5 < sms ? blocks * 1.5 / sms : 1.0;
        const double reread = elems * again * esz * (elems * esz < 110e6 ? 0.5 : far);
        return (elems * (esz + eout) + reread) / (6.5e6 * f);
    };
    GroupNorm best = p;
    double best_t = 1e30;
    bool best_grid = false;
    auto kernel = [&](bool grid, bool folded) {
        return grid ? (folded ? (const void *)groupnorm_k<TX, TY, V, true, true>
                              : (const void *)groupnorm_k<TX, TY, V, true, false>)
                    : (folded ? (const void *)groupnorm_k<TX, TY, V, false, true>
                              : (const void *)groupnorm_k<TX, TY, V, false, false>);
    };
    const void *fn = kernel(false, false);
    if (!tc::smem_opt_in(fn, SMEM, &done[0])) {
        fail("ops_groupnorm_cl: no %zu bytes of shared memory", SMEM);
        return true;
    }
    auto geometry = [&](GroupNorm &q, int gs, int team) {
        q.gs = gs;
        q.slices = (p.groups + gs - 1) / gs;
        q.slots = (int)(((long)q.R * gs * p.per + V - 1) / V);
        q.team = team;
        q.run = p.nsr / team;
        q.run_rem = p.nsr % team;
        const int rows = (p.nsr + team - 1) / team;
        q.lanes = MAX_THREADS / q.slots;
        if (q.lanes > rows)
            q.lanes = rows;
        q.base = q.run / q.lanes;
        q.more = q.run % q.lanes;
        q.by_slots.set(q.slots);
        // The rows that a warp reads at once (walk) start cols entries apart in
        // the 16 of a pass over the banks, not all in the same.
        q.pitch = q.slots * V / q.merged;
        if (q.cols < 16)
            while (q.pitch % 16 != (q.cols <= 1 ? 1 : q.cols <= 2 ? 2 : q.cols <= 4 ? 4 : 8))
                q.pitch++;
        const int threads = (q.slots * q.lanes + 31) / 32 * 32;
        const long need = (rows + q.lanes - 1) / q.lanes;
        q.keep = q.ring = 0;
        q.fold = need > FOLD ? V / q.merged : 0;
        const size_t fixed = smem_bytes(q, threads, vb) + 16;
        if (fixed > SMEM)
            return -1L;
        const long fit = (long)((SMEM - fixed) / ((size_t)threads * vb));
        q.keep = (int)(need < fit ? need : fit);
        if (V > 1 && need > fit) {
            if (fit < RING)
                return -1L;
            q.ring = RING;
            q.keep = (int)fit - RING;
        }
        return need;
    };
    for (int gs = unit, next; gs <= p.groups && gs <= gmax; gs = next) {
        next = gs == p.groups ? p.groups + 1 : 2 * gs < p.groups ? 2 * gs : p.groups;
        const double width = (double)p.R * gs * p.per * esz;
        if (width < 64 && next <= p.groups && next <= gmax)
            continue; // half-used memory transactions
        for (int team = 8; team >= 1; team /= 2) {
            GroupNorm q = p;
            const long need = geometry(q, gs, team);
            if (need < 0 || (team > 1 && p.nsr < team))
                continue;
            const double ctas = (double)p.nimg * q.slices * team;
            const double room = team * (double)clusters_of(fn, team, sms);
            const double waves = ctas > room ? (double)(long)((ctas + room - 1) / room) : 1.0;
            const double busy = ctas < room ? ctas : room;
            const double n = (double)p.nsr / team * width / esz; // elements of a block
            const double again = need > q.keep ? 1.0 - (double)(q.keep + q.ring) / need : 0.0;
            const double t =
                waves * (model(busy * n, again, busy, 2.6) / (q.slices > 1 ? 0.7 : 1.0) + 4.0);
            if (t < best_t) {
                best_t = t;
                best = q;
                best_grid = false;
            }
        }
    }
    const int all = sms < MAX_TEAM ? sms : MAX_TEAM;
    for (int batch = 1; p.groups <= gmax && batch <= p.nimg && batch <= 8; batch++) {
        GroupNorm q = p;
        const int team = all / batch;
        if (p.nsr < 4 * team)
            continue;
        const long need = geometry(q, p.groups, team);
        if (need < 0)
            continue;
        q.batch = batch;
        const double n = (double)p.HW * p.C * batch;
        const double again = need > q.keep ? 1.0 - (double)(q.keep + q.ring) / need : 0.0;
        const double t = (double)((p.nimg + batch - 1) / batch) *
                         (model(n, again, all, 1.8) + 9.0);
        if (t < best_t) {
            best_t = t;
            best = q;
            best_grid = true;
        }
    }
    if (best_t >= 1e30)
        return false;
    const int threads = (best.slots * best.lanes + 31) / 32 * 32;
    const size_t smem = smem_bytes(best, threads, vb);
    fn = kernel(best_grid, best.fold > 0);
    if (!tc::smem_opt_in(fn, SMEM, &done[best_grid + 2 * (best.fold > 0)])) {
        fail("ops_groupnorm_cl: no %zu bytes of shared memory", SMEM);
        return true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (best_grid) {
        cfg.gridDim = dim3(best.team * best.batch);
        at[0].id = cudaLaunchAttributeCooperative;
        at[0].val.cooperative = 1;
    }
    else {
        cfg.gridDim = dim3(best.slices * best.team, best.nimg);
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = best.team;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[1].val.programmaticStreamSerializationAllowed = 1; // (see after_previous)
        cfg.numAttrs = 2;
    }
    void *args[] = {&best};
    cuda_ok(cudaLaunchKernelExC(&cfg, fn, args), "groupnorm_cl");
    return true;
}

template <typename TX, typename TY>
void run(cudaStream_t st, const GroupNorm &p, int sms)
{
    constexpr int V = 16 / (int)sizeof(TX);
    const int ya = V * (int)sizeof(TY) < 16 ? V * (int)sizeof(TY) : 16;
    const bool packed = p.ldx == p.C && p.ldy == p.C;
    // Vectors where every one starts aligned: whole vectors in a row of any
    // pitch, or packed rows.
    const bool al = ((uintptr_t)p.X & 15) == 0 && (uintptr_t)p.Y % ya == 0 &&
                    (p.nimg == 1 || (p.sx % V == 0 && p.sy % V == 0)) &&
                    (packed || (p.C % V == 0 && p.ldx % V == 0 && p.ldy % V == 0));
    if ((al && launch<TX, TY, V>(st, p, sms)) || launch<TX, TY, 1>(st, p, sms))
        return;
    group_k<TX, TY><<<dim3(p.groups, p.nimg), 256, 0, st>>>(p);
    launch_ok("groupnorm_cl");
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

// A view of one map as the rows of all: from the first element of the first map
// to the last of the last, by single rows where the maps lie whole rows apart.
View all_maps(const View &v, int nimg, long s0)
{
    View a = v;
    if (nimg == 1)
        return a;
    if (v.rows == 1) {
        a.ld = s0; // maps of one pixel: a row each
        a.rows = nimg;
    }
    else if (v.ld > 0 && s0 % v.ld == 0) {
        a.rows = (nimg - 1) * (s0 / v.ld) + v.rows;
    }
    else {
        a.rows = 1;
        a.cols = (nimg - 1) * s0 + (v.rows - 1) * v.ld + v.cols;
    }
    return a;
}

}  // namespace
}  // namespace coreg

extern "C" size_t ops_groupnorm_cl_bytes(int nimg, long HW, int C, int groups)
{
    // Two batches' (mean, M2) per group and block of the whole grid.
    return nimg <= 0 || HW <= 0 || C <= 0 || groups <= 0
               ? 0
               : (size_t)2 * groups * MAX_TEAM * sizeof(float2);
}

extern "C" void ops_groupnorm_cl(struct ops *o, int nimg, long HW, int C, int groups,
                                 struct opnd X, int xtype, struct opnd Y, int ytype, cl_mem g,
                                 cl_mem b, float eps, int act, float slope, cl_mem work)
{
    const char *fn = "ops_groupnorm_cl";
    View x, y, vg, vb, ws;

    if (pending() || !type_ok(fn, xtype) || !type_ok(fn, ytype) || !act_ok(fn, act))
        return;
    if (nimg < 0 || HW < 0 || C < 0 || C > 0x40000000 || groups < 1 || C % groups ||
        nimg > 65535 || HW > 0x40000000L) {
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
    const View ax = all_maps(x, nimg, X.s0), ay = all_maps(y, nimg, Y.s0);
    const long nx = ax.span(), ny = ay.span();
    if ((!in_place && views_meet(ay, ax)) || (g && (ranges_meet(vg.p, C * 4L, y.p, ny) ||
                                                    ranges_meet(vb.p, C * 4L, y.p, ny)))) {
        fail("%s: the output overlaps an input", fn);
        return;
    }
    const long bytes = (long)ops_groupnorm_cl_bytes(nimg, HW, C, groups);
    if (!view_of(&ws, fn, "the work buffer", work, 0, bytes, 1, bytes, 1))
        return;
    if ((uintptr_t)ws.p & 15) {
        fail("%s: the work buffer is not 16-byte aligned", fn);
        return;
    }
    if (ranges_meet(ws.p, bytes, x.p, nx) || ranges_meet(ws.p, bytes, y.p, ny) ||
        (g && (ranges_meet(ws.p, bytes, vg.p, C * 4L) || ranges_meet(ws.p, bytes, vb.p, C * 4L)))) {
        fail("%s: the work buffer overlaps an operand", fn);
        return;
    }
    OnDevice dev(o->ocl);
    if (!dev.ok)
        return;
    GroupNorm p = {};
    p.nimg = nimg;
    p.C = C;
    p.groups = groups;
    p.per = C / groups;
    p.HW = (int)HW;
    p.X = x.p;
    p.ldx = X.ld;
    p.sx = X.s0;
    p.Y = y.p;
    p.ldy = Y.ld;
    p.sy = Y.s0;
    p.g = (const float *)vg.p;
    p.b = (const float *)vb.p;
    p.eps = eps;
    p.act = act;
    p.slope = slope;
    p.work = (float2 *)ws.p;
    cudaStream_t st = stream_of(o->ocl);
    const int sms = sms_of(o->ocl);
    Prof pr(o->ocl, "groupnorm_cl");
    if (xtype == OPS_BF16 && ytype == OPS_BF16)
        run<__nv_bfloat16, __nv_bfloat16>(st, p, sms);
    else if (xtype == OPS_BF16)
        run<__nv_bfloat16, float>(st, p, sms);
    else if (ytype == OPS_BF16)
        run<float, __nv_bfloat16>(st, p, sms);
    else
        run<float, float>(st, p, sms);
}
