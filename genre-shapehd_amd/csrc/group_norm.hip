// group_norm.hip -- group normalisation with its activation, forward and backward, on [N, C, S] maps that are channels
// last in memory (channel stride 1, one row of channels per position) or channels first (position stride 1).
//
//   mean = sum x / M, var = sum x^2 / M - mean^2 over the M = (C / groups) * S values of one image and group
//   h = (x - mean) / sqrt(var + eps),  z = w_c h + b_c,  y = act(z)
//   dz = dy act'(z),  db_c = sum dz,  dw_c = sum dz h,
//   dx = r (w dz - m1 - h m2),  m1 = sum_group w dz / M,  m2 = sum_group w dz h / M,  r = 1 / sqrt(var + eps)
//
// Sums and statistics are fp64 (gfx950 issues an fp64 FMA at the rate of an fp32 one, and the passes wait for memory) and taken of
// x less its group's first value, so that sum x^2 / M - mean^2 cancels nothing where the mean is many deviations from zero; z's
// sign -- which side of its jump a ReLU's derivative takes -- is that of the exact z.  y and dx are rounded once, to their type.
// No atomics: partial sums lie in the workspace and are added in a fixed order, so a call's result depends on nothing but its inputs.
//
// Groups of up to 16384 values are group_norm_small.hip's.  Here a map takes two passes, each a launch: sums (by chunk of an image
// and channel, in the workspace), then values, whose workgroups first add up their groups' chunks -- a launch of its own between
// the passes cost 5 to 9 us.  What is read twice is the price: an image's group does not fit a CU, and a wait of workgroups for one
// another inside a launch would need all of them resident.  Bound: HBM, at what a copy reaches (4.9 to 5.3 TB/s) or above it,
// where the second pass, which starts where the first ended, still finds x in the 256 MB cache.  Measured:
//   4 x 20 x 64^3 fp32 channels last, leaky ReLU: forward 17 + 30 us (84 MB read, 84 MB read + 86 written), backward 28 + 42 us
//   8 x 32 x 64^3 bf16 channels first, ReLU:      forward 22 + 42 us (134 MB,       134 + 134),            backward 41 + 61 us
//   4 x 20 x 64^3 fp32 channels first, leaky ReLU: forward 15 + 27 us, backward 27 + 38 us;  8 x 32 x 64^3, ReLU: 41 + 84 and 85 + 137
// y and dx are stored past the caches (group_norm.hpp).
#include "group_norm.hpp"

namespace genre {
namespace {

using namespace gn;

// How a channels-last image is cut.  A thread keeps ONE column of V consecutive values and walks down the rows, so that its
// channels' sums and coefficients stay in registers.  `rows` consecutive rows form a period of `cols` columns: one row where V
// divides C, else (rows without gaps only) the V / gcd(C, V) rows after which the columns fall on the same channels again.
struct Cut {
    int rows, cols, tile, tiles, deep;                                     // columns per workgroup, tiles of a period; periods side by side
    int64_t periods, per;                                                  // whole and part periods of an image, per workgroup
    int chunks;
};
struct Run { int64_t per; int chunks; };                                   // channels first: positions per workgroup

// one workgroup's share of a map: image, chunk and (channels last) tile or (channels first) channel
struct Where { int n, mid, chunk; };
__device__ __forceinline__ Where where(unsigned b, int mids, int chunks)
{
    const unsigned m = b / (unsigned)chunks;
    return {(int)(m / (unsigned)mids), (int)(m % (unsigned)mids), (int)(b % (unsigned)chunks)};
}

// statistics of an image's group, and for dx the means of w dz and w dz h over it
struct Stat { double mean, r, m1, m2; };

// The chunks' sums and what becomes of them: statistics (forward, with x0) or m1 and m2 (backward).  `joined`: every workgroup of
// the second pass adds up its groups' sums itself, some 1000 pairs at most; otherwise a launch between the passes has done so.
struct Between {
    bool joined;
    int chunks;                                                            // of the first pass
    const double2 *chan, *group;                                           // [image][chunk][channel]; channels last: [image][chunk][group]
    double *stats;                                                         // [2][image][group]
    const double *sums;                                                    // [image][group][2], where not joined
    void *dw, *db;
    int dwt, dbt;
    unsigned blocks;                                                       // of the map; those behind them see to dw and db
};

template <class T>
__device__ __forceinline__ Stat stat_of(const Map &x, const Shape &sh, int n, int g, double s, double q)
{
    // (equal values: the mean is theirs, exactly; a NaN stays one)
    const double d = s / sh.m, var = fma(-d, d, q / sh.m);
    return {first_value<T>(x, sh, n, g) + d, 1. / sqrt((var < 0 ? 0. : var) + sh.eps), 0, 0};
}
__device__ __forceinline__ void keep_stat(const Shape &sh, double *stats, int at, const Stat &t)
{
    stats[at] = t.mean;
    stats[sh.N * sh.G + at] = t.r;
}
__device__ __forceinline__ Stat saved_stat(const Shape &sh, const Between &k, int at, bool two)
{
    return {k.stats[at], k.stats[sh.N * sh.G + at], two && !k.joined ? k.sums[2 * at] : 0, two && !k.joined ? k.sums[2 * at + 1] : 0};
}
// the sum of a group's pairs over its channels and all chunks, in every thread
template <bool TWO>
__device__ __forceinline__ double2 group_total(const Shape &sh, int chunks, const double2 *chan, int n, int g, const void *w, int wt, double *lds)
{
    const double2 *p = chan + (int64_t)n * chunks * sh.C + g * sh.cg;
    double2 t = make_double2(0, 0);
    const unsigned cg = sh.cg, rows = blockDim.x / cg, rest = blockDim.x % cg;
    unsigned row = threadIdx.x / cg, c = threadIdx.x % cg;
#pragma unroll 4
    while (row < (unsigned)chunks) {
        const double2 v = p[(int64_t)row * sh.C + c];
        const float f = TWO ? load_param(w, wt, g * sh.cg + c, 1.f) : 1.f;
        t.x = fma(f, v.x, t.x);
        t.y = fma(f, v.y, t.y);
        row += rows;
        c += rest;
        if (c >= cg) {
            c -= cg;
            row++;
        }
    }
    block_sum2(t.x, t.y, lds);
    return t;
}

// ---- what one value contributes (the loops over a map are written once, for each of these) ----------------------
// Coef: what a channel of an image needs, made once per workgroup.  z = a (x - mean) + b, a = r w: a value on the mean has z = b
// exactly, whatever r.
template <class T>
struct SumsF {                                                             // d and d^2 of d = x - x0, x0 the group's first value
    static constexpr bool kTwo = false;
    struct Coef { double x0; };
    __device__ static Coef coef(double x0, const Stat &, float, float) { return {x0}; }
    __device__ static void add(const Coef &k, float, float x, float, double &s, double &q)
    {
        const double d = (double)x - k.x0;
        s += d;
        q = fma(d, d, q);
    }
};
template <class T, int ACT>
struct SumsB {                                                             // dz and dz (x - mean)
    static constexpr bool kTwo = true;
    struct Coef { double mean, a, b; };
    __device__ static Coef coef(double, const Stat &t, float w, float b) { return {t.mean, t.r * w, b}; }
    __device__ static void add(const Coef &k, float slope, float x, float dy, double &s, double &q)
    {
        const double d = (double)x - k.mean, dz = act_grad<ACT>(fma(d, k.a, k.b), dy, slope);
        s += dz;
        q = fma(dz, d, q);
    }
};
template <class T, int ACT>
struct ValueF {
    static constexpr bool kTwo = false;
    struct Coef { double mean, a, b; };
    __device__ static Coef coef(const Stat &t, float w, float b) { return {t.mean, t.r * w, b}; }
    __device__ static float value(const Coef &k, float slope, float x, float) { return act_value<ACT>(fma((double)x - k.mean, k.a, k.b), slope); }
};
template <class T, int ACT>
struct ValueB {
    static constexpr bool kTwo = true;
    struct Coef { double mean, a, b, k2, k3; };                            // dx = a dz - (k3 (x - mean) + k2)
    __device__ static Coef coef(const Stat &t, float w, float b) { return {t.mean, t.r * w, b, t.r * t.m1, t.r * t.r * t.m2}; }
    __device__ static float value(const Coef &k, float slope, float x, float dy)
    {
        const double d = (double)x - k.mean, dz = act_grad<ACT>(fma(d, k.a, k.b), dy, slope);
        return (float)fma(dz, k.a, -fma(d, k.k3, k.k2));
    }
};

constexpr int kBatch = 4;                                                  // accesses of a thread in flight at once

// ---- channels last ----------------------------------------------------------------------------------------------
// the coefficients of a thread's V channels: its column's, made by one thread each where a workgroup has several periods side by
// side (`lds`: room for a tile's), else by the thread itself
template <int V, class COEF, class MAKE>
__device__ __forceinline__ void column_coefs(COEF (&k)[V], COEF *lds, const Shape &sh, const Cut &cut, int tile, int in, const MAKE &make)
{
    const int first = cut.rows == 1 ? tile * cut.tile * V : 0, many = cut.rows == 1 ? min(cut.tile * V, sh.C - first) : sh.C;
    const bool own = cut.deep == 1 && cut.rows == 1;
    if (!own) {
        for (int j = threadIdx.x; j < many; j += blockDim.x) lds[j] = make(first + j);
        __syncthreads();
    }
    int c = in * V % (own ? sh.C : many);                                  // (one row a period: below `many` but in idle threads)
#pragma unroll
    for (int i = 0; i < V; i++) {
        if (own) k[i] = make(min(first + c, sh.C - 1));
        else k[i] = lds[c];
        if (++c == (own ? sh.C : many)) c = 0;
    }
}
// how many bytes of LDS that takes, with `coef` bytes a channel
inline size_t coef_bytes(const Shape &sh, const Cut &cut, int v, size_t coef)
{
    if (cut.deep == 1 && cut.rows == 1) return 0;
    return coef * (cut.rows == 1 ? (cut.tile * v < sh.C ? cut.tile * v : sh.C) : sh.C);
}

// columns (and threads) of a workgroup: where a column is a single value, rows of up to 1024 stay in one
constexpr int columns_of(int v) { return v == 1 ? 1024 : 512; }

template <class T, int V, class OP>
__global__ __launch_bounds__(columns_of(V)) void last_sums_kernel(Map x, Map dy, Shape sh, Cut cut, Between bt, const void *w, const void *b, int wt, int bty,
                                                        double2 *chan, double2 *group)
{
    using R = typename T::raw;
    extern __shared__ double lds[];
    const Where at = where(blockIdx.x, cut.tiles, cut.chunks);
    const int r = threadIdx.x / cut.tile, in = threadIdx.x % cut.tile, col = at.mid * cut.tile + in;
    typename OP::Coef k[V];
    column_coefs<V>(k, (typename OP::Coef *)lds, sh, cut, at.mid, in, [&](int c) {
        const int g = c / sh.cg;
        return OP::kTwo ? OP::coef(0, saved_stat(sh, bt, at.n * sh.G + g, false), load_param(w, wt, c, 1.f), load_param(b, bty, c, 0.f))
                        : OP::coef(first_value<T>(x, sh, at.n, g), Stat{}, 0, 0);
    });
    double s[V], q[V];
#pragma unroll
    for (int i = 0; i < V; i++) s[i] = q[i] = 0;
    if (r < cut.deep && col < cut.cols) {
        const int64_t lo = at.chunk * cut.per, hi = min(lo + cut.per, cut.periods), whole = min(hi, sh.S / cut.rows);
        const R *px = (const R *)x.p + at.n * x.sn + col * V, *pd = OP::kTwo ? (const R *)dy.p + at.n * dy.sn + col * V : nullptr;
        const int64_t dx = cut.rows * x.ss, dd = cut.rows * dy.ss;
        int64_t p = lo + r;
        for (; p + (kBatch - 1) * cut.deep < whole; p += kBatch * cut.deep) {
            Kept<T, V> a[kBatch], d[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; u++) {
                a[u].load(px + (p + u * cut.deep) * dx);
                if (OP::kTwo) d[u].load(pd + (p + u * cut.deep) * dd);
            }
#pragma unroll
            for (int u = 0; u < kBatch; u++)
#pragma unroll
                for (int i = 0; i < V; i++) OP::add(k[i], sh.slope, a[u].at(i), OP::kTwo ? d[u].at(i) : 0.f, s[i], q[i]);
        }
        for (; p < whole; p += cut.deep) {
            Kept<T, V> a, d;
            a.load(px + p * dx);
            if (OP::kTwo) d.load(pd + p * dd);
#pragma unroll
            for (int i = 0; i < V; i++) OP::add(k[i], sh.slope, a.at(i), OP::kTwo ? d.at(i) : 0.f, s[i], q[i]);
        }
        if (p < hi) {                                                      // the part period behind the last whole one
            const int64_t left = (sh.S - p * cut.rows) * sh.C - col * V;
#pragma unroll
            for (int i = 0; i < V; i++)
                if (i < left) OP::add(k[i], sh.slope, (float)px[p * dx + i], OP::kTwo ? (float)pd[p * dd + i] : 0.f, s[i], q[i]);
        }
    }
    __syncthreads();
    // pairs [i][thread].  A period's `many` values are added up over the periods side by side: `parts` threads each (part by part in
    // `half`), then a channel's value is the sum of its places e = channel + m C
    double2 *pair = (double2 *)lds, *half = pair + V * blockDim.x;
    const int T0 = blockDim.x, places = cut.tile * V, parts = places < T0 ? T0 / places : 1;
#pragma unroll
    for (int i = 0; i < V; i++) pair[i * T0 + threadIdx.x] = make_double2(s[i], q[i]);
    __syncthreads();
    for (int j = threadIdx.x; j < parts * places; j += T0) {
        const int e = j % places;
        double2 t = make_double2(0, 0);
        for (int d = j / places; d < cut.deep; d += parts) {
            const double2 v = pair[e % V * T0 + d * cut.tile + e / V];
            t.x += v.x;
            t.y += v.y;
        }
        half[j] = t;
    }
    __syncthreads();
    const int first = cut.rows == 1 ? at.mid * places : 0, many = cut.rows == 1 ? min(places, sh.C - first) : sh.C;
    const int64_t row = (int64_t)at.n * cut.chunks + at.chunk;
    double2 *mine = pair;                                                  // (with `group`: a tile is all channels)
    for (int j = threadIdx.x; j < many; j += T0) {
        double2 t = make_double2(0, 0);
        for (int m = 0, e = j; m < cut.rows; m++, e += sh.C)
            for (int d = 0; d < parts; d++) {
                t.x += half[d * places + e].x;
                t.y += half[d * places + e].y;
            }
        if (chan) chan[row * sh.C + first + j] = t;
        if (group) {
            const float f = OP::kTwo ? load_param(w, wt, j, 1.f) : 1.f;
            mine[j] = make_double2(f * t.x, f * t.y);
        }
    }
    if (!group) return;                                                    // (uniform)
    __syncthreads();
    const int lanes = min(min(32, T0 / sh.G), (sh.cg + 15) / 16), g = threadIdx.x / lanes, l = threadIdx.x % lanes;     // of a group
    if (g < sh.G) {
        double2 t = make_double2(0, 0);
        for (int j = l; j < sh.cg; j += lanes) {
            t.x += mine[g * sh.cg + j].x;
            t.y += mine[g * sh.cg + j].y;
        }
        if (lanes == 1) group[row * sh.G + g] = t;
        else half[threadIdx.x] = t;
    }
    if (lanes == 1) return;
    __syncthreads();
    if (g < sh.G && l == 0) {
        double2 t = half[threadIdx.x];
        for (int i = 1; i < lanes; i++) {
            t.x += half[threadIdx.x + i].x;
            t.y += half[threadIdx.x + i].y;
        }
        group[row * sh.G + g] = t;
    }
}

constexpr int kJoinedGroups = 32;

template <class T, int V, class OP>
__global__ __launch_bounds__(columns_of(V)) void last_value_kernel(Map x, Map dy, Map out, Shape sh, Cut cut, Between bt, const void *w, const void *b, int wt, int bty)
{
    using R = typename T::raw;
    extern __shared__ double lds[];
    __shared__ double2 total[columns_of(V)];
    __shared__ Stat stat[kJoinedGroups];
    if (OP::kTwo && blockIdx.x >= bt.blocks) {
        const int c = (blockIdx.x - bt.blocks) * (blockDim.x / 64) + threadIdx.x / 64;
        if (c < sh.C) channel_grads(sh, bt.chunks, bt.chan, bt.stats, c, bt.dw, bt.dwt, bt.db, bt.dbt);
        return;
    }
    // from the end: what the first pass read last is still in the cache
    const Where at = where(bt.blocks - 1 - blockIdx.x, cut.tiles, cut.chunks);
    if (bt.joined) {
        const int each = blockDim.x / sh.G, g = threadIdx.x % sh.G, lane = threadIdx.x / sh.G;
        double2 t = make_double2(0, 0);
        if (lane < each)
            for (int i = lane; i < bt.chunks; i += each) {
                const double2 v = bt.group[((int64_t)at.n * bt.chunks + i) * sh.G + g];
                t.x += v.x;
                t.y += v.y;
            }
        total[threadIdx.x] = t;
        for (int live = each; live > 1;) {
            const int half = (live + 1) / 2;
            __syncthreads();
            if (lane + half < live) {
                t.x += total[threadIdx.x + half * sh.G].x;
                t.y += total[threadIdx.x + half * sh.G].y;
                total[threadIdx.x] = t;
            }
            live = half;
        }
        if (lane == 0) {
            const int i = at.n * sh.G + g;
            if (OP::kTwo) {
                Stat v = saved_stat(sh, bt, i, true);
                v.m1 = t.x / sh.m;
                v.m2 = t.y * v.r / sh.m;
                stat[g] = v;
            } else {
                stat[g] = stat_of<T>(x, sh, at.n, g, t.x, t.y);
                if (at.chunk == 0) keep_stat(sh, bt.stats, i, stat[g]);
            }
        }
        __syncthreads();
    }
    const int r = threadIdx.x / cut.tile, in = threadIdx.x % cut.tile, col = at.mid * cut.tile + in;
    typename OP::Coef k[V];
    column_coefs<V>(k, (typename OP::Coef *)lds, sh, cut, at.mid, in, [&](int c) {
        const int g = c / sh.cg;
        return OP::coef(bt.joined ? stat[g] : saved_stat(sh, bt, at.n * sh.G + g, OP::kTwo), load_param(w, wt, c, 1.f), load_param(b, bty, c, 0.f));
    });
    if (r >= cut.deep || col >= cut.cols) return;
    const int64_t lo = at.chunk * cut.per, hi = min(lo + cut.per, cut.periods), whole = min(hi, sh.S / cut.rows);
    const R *px = (const R *)x.p + at.n * x.sn + col * V, *pd = OP::kTwo ? (const R *)dy.p + at.n * dy.sn + col * V : nullptr;
    R *po = (R *)out.p + at.n * out.sn + col * V;
    const int64_t dx = cut.rows * x.ss, dd = cut.rows * dy.ss, dout = cut.rows * out.ss;
    int64_t p = lo + r;
    for (; p < whole; p += cut.deep) {
        Kept<T, V> a, d;
        float v[V];
        a.load(px + p * dx);
        if (OP::kTwo) d.load(pd + p * dd);
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = OP::value(k[i], sh.slope, a.at(i), OP::kTwo ? d.at(i) : 0.f);
        store<T, V, true>(po + p * dout, v);
    }
    if (p < hi) {
        const int64_t left = (sh.S - p * cut.rows) * sh.C - col * V;
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < left)
                po[p * dout + i] = (R)OP::value(k[i], sh.slope, (float)px[p * dx + i], OP::kTwo ? (float)pd[p * dd + i] : 0.f);
    }
}

// ---- channels first ---------------------------------------------------------------------------------------------
template <class T, int V, class OP>
__global__ __launch_bounds__(256) void first_sums_kernel(Map x, Map dy, Shape sh, Run run, Between bt, const void *w, const void *b, int wt, int bty, double2 *chan)
{
    using R = typename T::raw;
    __shared__ double lds[32];
    const Where at = where(blockIdx.x, sh.C, run.chunks);
    const int g = at.mid / sh.cg;
    const typename OP::Coef k = OP::kTwo ? OP::coef(0, saved_stat(sh, bt, at.n * sh.G + g, false), load_param(w, wt, at.mid, 1.f), load_param(b, bty, at.mid, 0.f))
                                         : OP::coef(first_value<T>(x, sh, at.n, g), Stat{}, 0, 0);
    const R *px = (const R *)x.p + at.n * x.sn + at.mid * x.sc, *pd = OP::kTwo ? (const R *)dy.p + at.n * dy.sn + at.mid * dy.sc : nullptr;
    const int64_t hi = min((at.chunk + 1) * run.per, sh.S);
    const int step = blockDim.x * V;
    double s[2] = {0, 0}, q[2] = {0, 0};
    int64_t e = at.chunk * run.per + threadIdx.x * V;
    for (; e + (kBatch - 1) * step + V <= hi; e += kBatch * step) {
        Kept<T, V> a[kBatch], d[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
            a[u].load(px + e + u * step);
            if (OP::kTwo) d[u].load(pd + e + u * step);
        }
#pragma unroll
        for (int u = 0; u < kBatch; u++)
#pragma unroll
            for (int i = 0; i < V; i++) OP::add(k, sh.slope, a[u].at(i), OP::kTwo ? d[u].at(i) : 0.f, s[i & 1], q[i & 1]);
    }
    for (; e + V <= hi; e += step) {
        Kept<T, V> a, d;
        a.load(px + e);
        if (OP::kTwo) d.load(pd + e);
#pragma unroll
        for (int i = 0; i < V; i++) OP::add(k, sh.slope, a.at(i), OP::kTwo ? d.at(i) : 0.f, s[i & 1], q[i & 1]);
    }
#pragma unroll
    for (int i = 0; i < V; i++)
        if (e + i < hi) OP::add(k, sh.slope, (float)px[e + i], OP::kTwo ? (float)pd[e + i] : 0.f, s[i & 1], q[i & 1]);
    s[0] += s[1];
    q[0] += q[1];
    block_sum2(s[0], q[0], lds);
    if (threadIdx.x == 0) chan[((int64_t)at.n * run.chunks + at.chunk) * sh.C + at.mid] = make_double2(s[0], q[0]);
}

template <class T, int V, class OP>
__global__ __launch_bounds__(256) void first_value_kernel(Map x, Map dy, Map out, Shape sh, Run run, Between bt, const void *w, const void *b, int wt, int bty)
{
    using R = typename T::raw;
    __shared__ double lds[32];
    if (OP::kTwo && blockIdx.x >= bt.blocks) {
        const int c = (blockIdx.x - bt.blocks) * (blockDim.x / 64) + threadIdx.x / 64;
        if (c < sh.C) channel_grads(sh, bt.chunks, bt.chan, bt.stats, c, bt.dw, bt.dwt, bt.db, bt.dbt);
        return;
    }
    const Where at = where(bt.blocks - 1 - blockIdx.x, sh.C, run.chunks);
    const int g = at.mid / sh.cg, i = at.n * sh.G + g;
    Stat t;
    if (bt.joined) {
        const double2 v = group_total<OP::kTwo>(sh, bt.chunks, bt.chan, at.n, g, w, wt, lds);
        if (OP::kTwo) {
            t = saved_stat(sh, bt, i, true);
            t.m1 = v.x / sh.m;
            t.m2 = v.y * t.r / sh.m;
        } else {
            t = stat_of<T>(x, sh, at.n, g, v.x, v.y);
            if (at.chunk == 0 && at.mid == g * sh.cg && threadIdx.x == 0) keep_stat(sh, bt.stats, i, t);
        }
    } else {
        t = saved_stat(sh, bt, i, OP::kTwo);
    }
    const typename OP::Coef k = OP::coef(t, load_param(w, wt, at.mid, 1.f), load_param(b, bty, at.mid, 0.f));
    const R *px = (const R *)x.p + at.n * x.sn + at.mid * x.sc, *pd = OP::kTwo ? (const R *)dy.p + at.n * dy.sn + at.mid * dy.sc : nullptr;
    R *po = (R *)out.p + at.n * out.sn + at.mid * out.sc;
    const int64_t hi = min((at.chunk + 1) * run.per, sh.S);
    const int step = blockDim.x * V;
    int64_t e = at.chunk * run.per + threadIdx.x * V;
    for (; e + V <= hi; e += step) {
        Kept<T, V> a, d;
        float v[V];
        a.load(px + e);
        if (OP::kTwo) d.load(pd + e);
#pragma unroll
        for (int j = 0; j < V; j++) v[j] = OP::value(k, sh.slope, a.at(j), OP::kTwo ? d.at(j) : 0.f);
        store<T, V, true>(po + e, v);
    }
#pragma unroll
    for (int j = 0; j < V; j++)
        if (e + j < hi) po[e + j] = (R)OP::value(k, sh.slope, (float)px[e + j], OP::kTwo ? (float)pd[e + j] : 0.f);
}

// ---- between the passes, where the second does not do it: one workgroup per image and group ---------------------
template <class T>
__global__ __launch_bounds__(256) void stats_kernel(Map x, Shape sh, Between bt)
{
    __shared__ double lds[32];
    const int n = blockIdx.x / sh.G, g = blockIdx.x % sh.G;
    const double2 t = group_total<false>(sh, bt.chunks, bt.chan, n, g, nullptr, 0, lds);
    if (threadIdx.x == 0) keep_stat(sh, bt.stats, blockIdx.x, stat_of<T>(x, sh, n, g, t.x, t.y));
}
__global__ __launch_bounds__(256) void group_sums_kernel(Shape sh, Between bt, const void *w, int wt, double *sums)
{
    __shared__ double lds[32];
    const int n = blockIdx.x / sh.G, g = blockIdx.x % sh.G;
    const double2 t = group_total<true>(sh, bt.chunks, bt.chan, n, g, w, wt, lds);
    if (threadIdx.x == 0) {
        sums[2 * blockIdx.x] = t.x / sh.m;
        sums[2 * blockIdx.x + 1] = t.y * bt.stats[sh.N * sh.G + blockIdx.x] / sh.m;      // sum w dz h / M
    }
}

// ---- host -------------------------------------------------------------------------------------------------------
inline int es_of(const genre_tensor *t) { return t->dtype == GENRE_F32 ? 4 : 2; }
inline bool is_map_type(int32_t t) { return t == GENRE_F32 || t == GENRE_BF16 || t == GENRE_F16; }

int check_map(const char *op, const char *what, const genre_tensor *t, const genre_tensor *like)
{
    GENRE_REQUIRE(t && t->ndim == 3 && is_map_type(t->dtype), "%s: %s must be a [N,C,S] tensor of fp32, bf16 or fp16", op, what);
    GENRE_REQUIRE(same_shape(t, like), "%s: %s must have x's shape", op, what);
    GENRE_REQUIRE(t->dtype == like->dtype, "%s: %s must have x's dtype", op, what);
    for (int i = 0; i < 3; i++) GENRE_REQUIRE(t->size[i] >= 0 && t->stride[i] >= 0, "%s: %s has a negative size or stride", op, what);
    GENRE_REQUIRE(t->data || numel(t) == 0, "%s: %s is NULL", op, what);
    return 1;
}
int check_param(const char *op, const char *what, const genre_tensor *t, int64_t C)
{
    if (!t) return 1;
    GENRE_REQUIRE(t->data && t->ndim == 1 && is_map_type(t->dtype) && t->size[0] == C && (C == 1 || t->stride[0] == 1),
                  "%s: %s must be a contiguous [%lld] tensor of fp32, bf16 or fp16", op, what, (long long)C);
    return 1;
}

inline bool channels_last(const genre_tensor *t)
{
    if (t->size[1] == 1) return t->stride[2] != 1 && t->size[2] != 1;
    return t->stride[1] == 1 && (t->size[2] == 1 || t->stride[2] != 1);
}
inline bool channels_first(const genre_tensor *t) { return t->size[2] == 1 || t->stride[2] == 1; }
inline bool gapless(const genre_tensor *t) { return t->size[2] == 1 || t->stride[2] == t->size[1]; }
inline Map map_of(const genre_tensor *t) { return {t->data, t->stride[0], t->stride[1], t->size[2] == 1 ? t->size[1] : t->stride[2]}; }

// values per thread and access: 16 bytes; channels last, where each has sums and coefficients of its own, at most four, and fewer
// where a column may not cross a row's end
int width_of(const genre_tensor *x, bool last, bool dense)
{
    int v = last || x->dtype == GENRE_F32 ? 4 : 8;
    if (last) {
        const int C = (int)x->size[1];
        if (!dense || C > 1024 || C / gcd(C, v) > 512) v = gcd(C, v);   // (a period's coefficients and columns have to fit a workgroup)
    }
    return v;
}

// Workgroups, with four accesses a thread at least.  Sums 1024 / 2048: refiner 64^3 x4, channels last, whose workgroups end with a
// reduction by column, 47.4 / 51.3 us (training 126 / 137); decoder 64^3 x8, channels first, 73.5 / 71.3 (179 / 175).  Values 2048 /
// 4096: 47.4 / 47.4 and 73.5 / 72.0 (126.1 / 125.9 and 179.5 / 177.2).
constexpr int kSumsLast = 1024, kSumsFirst = 2048, kValueWorkgroups = 4096;
// Pairs that a workgroup of the second pass adds up itself (16 KB from the caches; 2048: 4 x 40 x 32^3 backward 26 -> 30 us), and
// accesses of a thread of the first pass beyond which more chunks and a launch between the passes are faster.
constexpr int kJoined = 1024, kFew = 32;

int chunks_of(int64_t turns, int64_t others, int workgroups, int64_t most)
{
    const int64_t fill = (workgroups + others - 1) / others, few = (turns + kBatch - 1) / kBatch;
    const int64_t c = few < fill ? few : fill;
    return (int)(c < most ? c : most);
}

Cut cut_of(int N, int C, int64_t S, int v, int workgroups, int64_t most, int *threads)
{
    Cut c;
    const int g = gcd(C, v);
    c.rows = v / g;
    c.cols = C / g;
    c.tiles = ceil_div(c.cols, columns_of(v));
    c.tile = ceil_div(c.cols, c.tiles);
    c.deep = c.tile > 512 ? 1 : (c.tile > 256 ? 512 : 256) / c.tile;
    *threads = (c.deep * c.tile + 63) / 64 * 64;
    c.periods = (S + c.rows - 1) / c.rows;
    const int64_t turns = (c.periods + c.deep - 1) / c.deep;
    const int chunks = chunks_of(turns, (int64_t)N * c.tiles, workgroups, most);
    c.per = (turns + chunks - 1) / chunks * c.deep;
    c.chunks = (int)((c.periods + c.per - 1) / c.per);
    return c;
}

Run run_of(int N, int C, int64_t S, int v, int threads, int workgroups, int64_t most)
{
    const int64_t step = (int64_t)threads * v, turns = (S + step - 1) / step;
    const int chunks = chunks_of(turns, (int64_t)N * C, workgroups, most);
    const int64_t per = (turns + chunks - 1) / chunks * step;
    return {per, (int)((S + per - 1) / per)};
}

struct Call {
    Shape sh;
    int small;                                                             // threads of a workgroup in the one-workgroup form (0: two passes)
    bool last, joined;
    int v, threads;
    Cut sums, values;                                                      // channels last
    Run rsums, rvalues;                                                    // channels first
    int chunks() const { return last ? sums.chunks : rsums.chunks; }
    int64_t sums_blocks() const { return (int64_t)sh.N * (last ? sums.tiles : sh.C) * chunks(); }
    int64_t value_blocks() const { return (int64_t)sh.N * (last ? values.tiles * (int64_t)values.chunks : sh.C * (int64_t)rvalues.chunks); }
    size_t sums_lds(size_t coef) const
    {
        const int places = sums.tile * v, parts = places < threads ? threads / places : 1;
        const size_t a = sizeof(double2) * (v * threads + (parts * places > threads ? parts * places : threads)), b = coef_bytes(sh, sums, v, coef);
        return a > b ? a : b;
    }
};

void cut_call(Call &c, int64_t N, int64_t C, int64_t S, int groups)
{
    if (c.last) {
        // the second pass joins the sums where few enough chunks fill half the chip or have few accesses each, and a workgroup sees
        // all channels
        const int64_t most = kJoined / groups > 64 ? kJoined / groups : 64;
        c.sums = cut_of((int)N, (int)C, S, c.v, kSumsLast, INT32_MAX, &c.threads);
        const int64_t turns = (c.sums.periods + c.sums.deep - 1) / c.sums.deep;             // accesses of a thread that sees a whole image
        c.joined = c.sums.tiles == 1 && groups <= kJoinedGroups &&
                   (c.sums.chunks <= most || N * most >= kSumsLast / 2 || turns <= kFew * most);
        if (c.joined) c.sums = cut_of((int)N, (int)C, S, c.v, kSumsLast, most, &c.threads);
        // sixteen accesses a thread -- a workgroup of the second pass begins with joining sums and making coefficients here --, in
        // whole fours of workgroups for each CU: 4 x 20 x 64^3 bf16 with 1024 / 4096 of them: 31.1 / 33.1 us (backward 43 / 48),
        // 8 x 32 x 64^3: 70 / 69 (117 / 113)
        const int64_t wanted = N * c.sums.tiles * turns / 16 / 1024 * 1024;
        c.values = cut_of((int)N, (int)C, S, c.v, wanted < 1024 ? 1024 : wanted > kValueWorkgroups ? kValueWorkgroups : (int)wanted, INT32_MAX, &c.threads);
    } else {
        c.threads = S <= 64 * c.v * 4 ? 64 : 256;
        const int64_t cg = C / groups, most = kJoined / cg;
        c.rsums = run_of((int)N, (int)C, S, c.v, c.threads, kSumsFirst, INT32_MAX);
        const int64_t turns = (S + c.threads * c.v - 1) / (c.threads * c.v);
        c.joined = c.rsums.chunks <= most || (most > 0 && (N * C * most >= kSumsFirst / 2 || turns <= kFew * most));
        if (c.joined) c.rsums = run_of((int)N, (int)C, S, c.v, c.threads, kSumsFirst, most);
        c.rvalues = run_of((int)N, (int)C, S, c.v, c.threads, kValueWorkgroups, INT32_MAX);
    }
}

// a launch counts its threads in 32 bits
inline bool launches(int64_t workgroups, int threads) { return workgroups * threads < ((int64_t)1 << 32); }

int plan(const char *op, const genre_tensor *x, const genre_tensor *const *others, int n_others, int groups, bool backward, Call &c)
{
    GENRE_REQUIRE(x->size[0] <= INT32_MAX && x->size[1] <= (1 << 24), "%s: too many images or channels", op);
    const int64_t N = x->size[0], C = x->size[1], S = x->size[2];
    GENRE_REQUIRE(groups > 0 && C > 0 && C % groups == 0, "%s: %lld channels do not split into %d groups", op, (long long)C, groups);
    GENRE_REQUIRE(N * C < (1 << 30), "%s: N*C must be below 2^30", op);
    GENRE_REQUIRE(N == 0 || S < ((int64_t)1 << 60) / (N * C), "%s: a map of 2^60 values or more", op);
    bool last = channels_last(x), first = channels_first(x), dense = gapless(x);
    for (int i = 0; i < n_others; i++) {
        last = last && channels_last(others[i]);
        first = first && channels_first(others[i]);
        dense = dense && gapless(others[i]);
    }
    GENRE_REQUIRE(last || first, "%s: the maps must all be channels last (channel stride 1) or all channels first (position stride 1)", op);
    c.last = last;
    c.sh = {(int)N, (int)C, groups, (int)(C / groups), 0, S, 0.f, 0., 0.};
    c.v = width_of(x, last, dense);
    if (N * S == 0) return 1;
    c.sh.m = (double)(C / groups) * (double)S;
    c.small = small_threads(last, c.sh, es_of(x), backward);
    cut_call(c, N, C, S, groups);
    const bool fits = c.small ? launches(N * groups, c.small)
                              : launches(c.sums_blocks(), c.threads) && launches(c.value_blocks() + C, c.threads) && (c.joined || launches(N * groups, 256)) &&
                                    N * (int64_t)c.chunks() < INT32_MAX && c.chunks() * (C / groups) < INT32_MAX;
    GENRE_REQUIRE(fits && N * groups < INT32_MAX / 2, "%s: the map is too large for one launch", op);
    return 1;
}

// fp64 values of the workspace: the chunks' sums by channel (forward: unless they are joined by group), by group, the groups'
int64_t chan_values(const Call &c, bool backward) { return backward || !(c.last && c.joined) ? 2 * (int64_t)c.sh.N * c.sh.C * c.chunks() : 0; }
int64_t group_values(const Call &c) { return c.last && c.joined ? 2 * (int64_t)c.sh.N * c.sh.G * c.chunks() : 0; }
int64_t workspace_of(const Call &c, bool backward)
{
    return chan_values(c, backward) + group_values(c) + (backward && !c.joined ? 2 * (int64_t)c.sh.N * c.sh.G : 0);
}

int check_f64(const char *op, const char *what, const genre_tensor *t, int64_t least)
{
    if (least == 0) return 1;
    GENRE_REQUIRE(t && t->data && t->dtype == GENRE_F64 && is_contiguous(t) && numel(t) >= least && aligned16(t->data),
                  "%s: %s must be a contiguous fp64 tensor of at least %lld values, on a multiple of 16 bytes", op, what, (long long)least);
    return 1;
}

struct Space { double2 *chan, *group; double *sums; };
Space space_of(const Call &c, bool backward, double *ws)
{
    const int64_t chan = chan_values(c, backward), group = group_values(c);
    return {chan ? (double2 *)ws : nullptr, group ? (double2 *)(ws + chan) : nullptr, ws + chan + group};
}

template <class T, int V, class OP>
int sums(const Call &c, const Map &x, const Map &dy, const Params &p, const Between &k, const Space &to, hipStream_t st)
{
    const int blocks = (int)c.sums_blocks();
    if constexpr (V <= 4)                                                  // (width_of)
        if (c.last)
            last_sums_kernel<T, V, OP><<<blocks, c.threads, c.sums_lds(sizeof(typename OP::Coef)), st>>>(x, dy, c.sh, c.sums, k, p.w, p.b, p.wt, p.bt, to.chan, to.group);
    if constexpr (V * sizeof(typename T::raw) == 16)
        if (!c.last) first_sums_kernel<T, V, OP><<<blocks, c.threads, 0, st>>>(x, dy, c.sh, c.rsums, k, p.w, p.b, p.wt, p.bt, to.chan);
    GENRE_LAUNCH_CHECK("group norm sums");
    return 1;
}
template <class T, int V, class OP>
int values(const Call &c, const Map &x, const Map &dy, const Map &out, const Params &p, const Between &k, hipStream_t st)
{
    const int blocks = (int)k.blocks + (k.dw || k.db ? ceil_div(c.sh.C, c.threads / 64) : 0);
    if constexpr (V <= 4)
        if (c.last)
            last_value_kernel<T, V, OP><<<blocks, c.threads, coef_bytes(c.sh, c.values, V, sizeof(typename OP::Coef)), st>>>(x, dy, out, c.sh, c.values, k, p.w, p.b, p.wt, p.bt);
    if constexpr (V * sizeof(typename T::raw) == 16)
        if (!c.last) first_value_kernel<T, V, OP><<<blocks, c.threads, 0, st>>>(x, dy, out, c.sh, c.rvalues, k, p.w, p.b, p.wt, p.bt);
    GENRE_LAUNCH_CHECK("group norm values");
    return 1;
}

template <class T, int V>
int forward(const Call &c, const Map &x, const Map &y, const Params &p, double *stats, double *ws, hipStream_t st)
{
    const Space to = space_of(c, false, ws);
    const Between k = {c.joined, c.chunks(), to.chan, to.group, stats, nullptr, nullptr, nullptr, 0, 0, (unsigned)c.value_blocks()};
    if (!sums<T, V, SumsF<T>>(c, x, Map{}, p, k, to, st)) return 0;
    if (!c.joined) {
        stats_kernel<T><<<c.sh.N * c.sh.G, 256, 0, st>>>(x, c.sh, k);
        GENRE_LAUNCH_CHECK("group norm statistics");
    }
    switch (c.sh.act) {
    case kActRelu: return values<T, V, ValueF<T, kActRelu>>(c, x, Map{}, y, p, k, st);
    case kActLeaky: return values<T, V, ValueF<T, kActLeaky>>(c, x, Map{}, y, p, k, st);
    case kActSilu: return values<T, V, ValueF<T, kActSilu>>(c, x, Map{}, y, p, k, st);
    default: return values<T, V, ValueF<T, kActNone>>(c, x, Map{}, y, p, k, st);
    }
}

template <class T, int V, int ACT>
int backward_as(const Call &c, const Map &x, const Map &dy, const Params &p, const Grads &g, const double *stats, double *ws, hipStream_t st)
{
    const Space to = space_of(c, true, ws);
    const Between k = {c.joined, c.chunks(), to.chan, to.group, (double *)stats, to.sums, g.dw, g.db, g.dwt, g.dbt, (unsigned)c.value_blocks()};
    if (!sums<T, V, SumsB<T, ACT>>(c, x, dy, p, k, to, st)) return 0;
    if (!g.dx.p) {
        if (!g.dw && !g.db) return 1;
        channel_grads_kernel<<<ceil_div(c.sh.C, 4), 256, 0, st>>>(c.sh, k.chunks, k.chan, stats, g.dw, g.dwt, g.db, g.dbt);
        GENRE_LAUNCH_CHECK("group norm parameter gradients");
        return 1;
    }
    if (!c.joined) {
        group_sums_kernel<<<c.sh.N * c.sh.G, 256, 0, st>>>(c.sh, k, p.w, p.wt, to.sums);
        GENRE_LAUNCH_CHECK("group norm backward group sums");
    }
    return values<T, V, ValueB<T, ACT>>(c, x, dy, g.dx, p, k, st);
}
template <class T, int V>
int backward(const Call &c, const Map &x, const Map &dy, const Params &p, const Grads &g, const double *stats, double *ws, hipStream_t st)
{
    switch (c.sh.act) {
    case kActRelu: return backward_as<T, V, kActRelu>(c, x, dy, p, g, stats, ws, st);
    case kActLeaky: return backward_as<T, V, kActLeaky>(c, x, dy, p, g, stats, ws, st);
    case kActSilu: return backward_as<T, V, kActSilu>(c, x, dy, p, g, stats, ws, st);
    default: return backward_as<T, V, kActNone>(c, x, dy, p, g, stats, ws, st);
    }
}

#define GENRE_BY_WIDTH(T, v, call8, call4, call2, call1) ((v) == 8 ? call8 : (v) == 4 ? call4 : (v) == 2 ? call2 : call1)

// scratch of a call whose maps all lie as `c` says
int64_t needed(const Call &c, const genre_tensor *x, bool backward)
{
    if (small_threads(c.last, c.sh, es_of(x), backward)) return backward ? small_workspace(c.sh) : 0;
    return workspace_of(c, backward);
}

}  // namespace
}  // namespace genre

using namespace genre;

extern "C" int64_t genre_group_norm_workspace(const genre_tensor *x, int groups, int backward)
{
    const char *op = "group_norm_workspace";
    Call c{};
    if (!x) { fail("%s: x is NULL", op); return -1; }
    if (!check_map(op, "x", x, x) || !plan(op, x, nullptr, 0, groups, backward != 0, c)) return -1;
    if (numel(x) == 0) return 0;
    int64_t need = needed(c, x, backward != 0);
    // the other maps may make another call of it: gaps in their rows narrow the columns, and with one position (which lies in both
    // ways) they may leave channels first only.  Room for all
    for (int other = 0; other < 2 && c.last; other++) {
        if (other && !channels_first(x)) continue;
        Call d = c;
        d.last = !other;
        d.v = width_of(x, d.last, false);
        cut_call(d, d.sh.N, d.sh.C, d.sh.S, groups);
        const int64_t n = needed(d, x, backward != 0);
        if (n > need) need = n;
    }
    return need;
}

extern "C" int genre_group_norm_forward(const genre_tensor *x, const genre_tensor *y, const genre_tensor *weight, const genre_tensor *bias,
                                        const genre_tensor *stats, const genre_tensor *ws, int groups, double eps, int act, float slope, void *stream)
{
    const char *op = "group_norm_forward";
    GENRE_REQUIRE(x && y, "%s: x and y are needed", op);
    if (!check_map(op, "x", x, x) || !check_map(op, "y", y, x)) return 0;
    if (!check_param(op, "weight", weight, x->size[1]) || !check_param(op, "bias", bias, x->size[1])) return 0;
    GENRE_REQUIRE(eps > 0, "%s: eps must be positive", op);
    GENRE_REQUIRE(act >= kActNone && act <= kActSilu, "%s: unknown activation %d", op, act);
    Call c{};
    const genre_tensor *const others[] = {y};
    if (!plan(op, x, others, 1, groups, false, c)) return 0;
    if (!check_f64(op, "stats", stats, 2 * (int64_t)c.sh.N * groups)) return 0;
    if (numel(x) == 0) return 1;
    c.sh.act = act;
    c.sh.slope = slope;
    c.sh.eps = eps;
    const Params p = {weight ? weight->data : nullptr, bias ? bias->data : nullptr, weight ? weight->dtype : 0, bias ? bias->dtype : 0};
    const Map mx = map_of(x), my = map_of(y);
    double *s = (double *)stats->data;
    hipStream_t st = (hipStream_t)stream;
    if (c.small) return small_forward(c.last, x->dtype, c.sh, mx, my, p, s, st);
    if (!check_f64(op, "ws", ws, workspace_of(c, false))) return 0;
    double *b = (double *)ws->data;
    if (x->dtype == GENRE_F32)
        return c.v == 4 ? forward<F32, 4>(c, mx, my, p, s, b, st) : c.v == 2 ? forward<F32, 2>(c, mx, my, p, s, b, st) : forward<F32, 1>(c, mx, my, p, s, b, st);
    if (x->dtype == GENRE_BF16)
        return GENRE_BY_WIDTH(BF16, c.v, (forward<BF16, 8>(c, mx, my, p, s, b, st)), (forward<BF16, 4>(c, mx, my, p, s, b, st)),
                              (forward<BF16, 2>(c, mx, my, p, s, b, st)), (forward<BF16, 1>(c, mx, my, p, s, b, st)));
    return GENRE_BY_WIDTH(F16, c.v, (forward<F16, 8>(c, mx, my, p, s, b, st)), (forward<F16, 4>(c, mx, my, p, s, b, st)),
                          (forward<F16, 2>(c, mx, my, p, s, b, st)), (forward<F16, 1>(c, mx, my, p, s, b, st)));
}

extern "C" int genre_group_norm_backward(const genre_tensor *x, const genre_tensor *dy, const genre_tensor *weight, const genre_tensor *bias,
                                         const genre_tensor *stats, const genre_tensor *dx, const genre_tensor *dw, const genre_tensor *db,
                                         const genre_tensor *ws, int groups, int act, float slope, void *stream)
{
    const char *op = "group_norm_backward";
    GENRE_REQUIRE(x && dy, "%s: x and dy are needed", op);
    if (!check_map(op, "x", x, x) || !check_map(op, "dy", dy, x)) return 0;
    if (dx && !check_map(op, "dx", dx, x)) return 0;
    const int64_t C = x->size[1];
    if (!check_param(op, "weight", weight, C) || !check_param(op, "bias", bias, C) || !check_param(op, "dw", dw, C) || !check_param(op, "db", db, C)) return 0;
    GENRE_REQUIRE(act >= kActNone && act <= kActSilu, "%s: unknown activation %d", op, act);
    Call c{};
    const genre_tensor *const others[] = {dy, dx};
    if (!plan(op, x, others, dx ? 2 : 1, groups, true, c)) return 0;
    if (!check_f64(op, "stats", stats, 2 * (int64_t)c.sh.N * groups)) return 0;
    hipStream_t st = (hipStream_t)stream;
    const Grads g = {dx ? map_of(dx) : Map{}, dw ? dw->data : nullptr, db ? db->data : nullptr, dw ? dw->dtype : 0, db ? db->dtype : 0};
    if (numel(x) == 0) {                                                   // sums over nothing
        if (g.dw || g.db) {
            Shape none = c.sh;
            none.N = 0;
            channel_grads_kernel<<<ceil_div(none.C, 4), 256, 0, st>>>(none, 1, nullptr, nullptr, g.dw, g.dwt, g.db, g.dbt);
            GENRE_LAUNCH_CHECK("group norm parameter gradients");
        }
        return 1;
    }
    c.sh.act = act;
    c.sh.slope = slope;
    const Params p = {weight ? weight->data : nullptr, bias ? bias->data : nullptr, weight ? weight->dtype : 0, bias ? bias->dtype : 0};
    const Map mx = map_of(x), md = map_of(dy);
    const double *s = (const double *)stats->data;
    if (!check_f64(op, "ws", ws, c.small ? small_workspace(c.sh) : workspace_of(c, true))) return 0;
    double *b = ws ? (double *)ws->data : nullptr;
    if (c.small) return small_backward(c.last, x->dtype, c.sh, mx, md, p, g, s, b, st);
    if (x->dtype == GENRE_F32)
        return c.v == 4 ? backward<F32, 4>(c, mx, md, p, g, s, b, st) : c.v == 2 ? backward<F32, 2>(c, mx, md, p, g, s, b, st) : backward<F32, 1>(c, mx, md, p, g, s, b, st);
    if (x->dtype == GENRE_BF16)
        return GENRE_BY_WIDTH(BF16, c.v, (backward<BF16, 8>(c, mx, md, p, g, s, b, st)), (backward<BF16, 4>(c, mx, md, p, g, s, b, st)),
                              (backward<BF16, 2>(c, mx, md, p, g, s, b, st)), (backward<BF16, 1>(c, mx, md, p, g, s, b, st)));
    return GENRE_BY_WIDTH(F16, c.v, (backward<F16, 8>(c, mx, md, p, g, s, b, st)), (backward<F16, 4>(c, mx, md, p, g, s, b, st)),
                          (backward<F16, 2>(c, mx, md, p, g, s, b, st)), (backward<F16, 1>(c, mx, md, p, g, s, b, st)));
}
