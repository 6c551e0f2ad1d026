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
// sign -- which side of its jump a ReLU's derivative takes -- is that of the exact z.  y and dx are rounded once, to their type.  No atomics: partial sums lie in the workspace and are added
// in a fixed order, so a call's result depends on nothing but its inputs.
#include "group_norm.hpp"

namespace genre {
namespace {

using namespace gn;

// How a channels-last image is cut.  A thread keeps ONE column of V consecutive values and walks down the rows, so that its
// channels' sums and coefficients stay in registers.  `rows` consecutive rows form a period of `cols` columns: one row where V
// divides C, else (rows without gaps only) the V / gcd(C, V) rows after which the columns fall on the same channels again.
struct Cut {
    int rows, cols, tile, tiles, deep, threads;                            // columns per workgroup, tiles of a period; periods side by side
    int64_t periods, per;                                                  // whole and part periods of an image, per workgroup
    int chunks;
};

// one workgroup's share of a map: image, chunk and (channels last) tile or (channels first) channel
struct Where { int n, mid, chunk; };
__device__ __forceinline__ Where where(int mids, int chunks)
{
    const unsigned b = blockIdx.x, m = b / (unsigned)chunks;
    return {(int)(m / (unsigned)mids), (int)(m % (unsigned)mids), (int)(b % (unsigned)chunks)};
}

// per-channel coefficients: z = a (x - mean) + b.  (x - mean first: a value on the mean has z = b exactly, whatever r)
struct Norm { double mean, a, b, r; };
__device__ __forceinline__ Norm norm_of(const double *stats, const Shape &sh, int n, int c, float w, float bias)
{
    const int at = n * sh.G + c / sh.cg;
    const double r = stats[sh.N * sh.G + at];
    return {stats[at], r * w, bias, r};
}

// ---- what one value contributes (the loops over a map are written once, for each of these) ----------------------
// forward sums: d, d^2 of d = x - x0, x0 the group's first value
template <class T>
struct SumsF {
    static constexpr bool kTwo = false;
    struct Coef { double x0; };
    __device__ static Coef coef(const Map &x, const Shape &sh, const double *, int n, int c, const void *, const void *, int, int)
    {
        return {first_value<T>(x, sh, n, c / sh.cg)};
    }
    __device__ static void add(const Coef &k, float, float x, float, double &s, double &q)
    {
        const double d = (double)x - k.x0;
        s += d;
        q = fma(d, d, q);
    }
};
// backward sums: dz, dz (x - mean)
template <class T, int ACT>
struct SumsB {
    static constexpr bool kTwo = true;
    struct Coef { double mean, a, b; };
    __device__ static Coef coef(const Map &, const Shape &sh, const double *stats, int n, int c, const void *w, const void *b, int wt, int bt)
    {
        const Norm k = norm_of(stats, sh, n, c, load_param(w, wt, c, 1.f), load_param(b, bt, c, 0.f));
        return {k.mean, k.a, k.b};
    }
    __device__ static void add(const Coef &k, float slope, float x, float dy, double &s, double &q)
    {
        const double d = (double)x - k.mean;
        const double dz = dy * act_slope<ACT>(fma(d, k.a, k.b), slope);
        s += dz;
        q = fma(dz, d, q);
    }
};
template <class T, int ACT>
struct ValueF {
    static constexpr bool kTwo = false;
    struct Coef { double mean, a, b; };
    __device__ static Coef coef(const Shape &sh, const double *stats, const double *, int n, int c, const void *w, const void *b, int wt, int bt)
    {
        const Norm k = norm_of(stats, sh, n, c, load_param(w, wt, c, 1.f), load_param(b, bt, c, 0.f));
        return {k.mean, k.a, k.b};
    }
    __device__ static float value(const Coef &k, float slope, float x, float)
    {
        return act_value<ACT>(fma((double)x - k.mean, k.a, k.b), slope);
    }
};
template <class T, int ACT>
struct ValueB {
    static constexpr bool kTwo = true;
    struct Coef { double mean, a, b, k2, k3; };                            // dx = a dz - (k3 (x - mean) + k2)
    __device__ static Coef coef(const Shape &sh, const double *stats, const double *sums, int n, int c, const void *w, const void *b, int wt, int bt)
    {
        const Norm k = norm_of(stats, sh, n, c, load_param(w, wt, c, 1.f), load_param(b, bt, c, 0.f));
        const int at = n * sh.G + c / sh.cg;
        return {k.mean, k.a, k.b, k.r * sums[2 * at], k.r * k.r * sums[2 * at + 1]};
    }
    __device__ static float value(const Coef &k, float slope, float x, float dy)
    {
        const double d = (double)x - k.mean, dz = dy * act_slope<ACT>(fma(d, k.a, k.b), slope);
        return (float)fma(dz, k.a, -fma(d, k.k3, k.k2));
    }
};

// ---- channels last ----------------------------------------------------------------------------------------------
template <class T, int V, class OP>
__global__ __launch_bounds__(512) void last_sums_kernel(Map x, Map dy, Shape sh, Cut cut, const double *stats, const void *w, const void *b,
                                                        int wt, int bt, double2 *part)
{
    using R = typename T::raw;
    extern __shared__ double lds[];
    const Where at = where(cut.tiles, cut.chunks);
    const int r = threadIdx.x / cut.tile, in = threadIdx.x % cut.tile, col = at.mid * cut.tile + in;
    double s[V], q[V];
#pragma unroll
    for (int i = 0; i < V; i++) s[i] = q[i] = 0;
    if (r < cut.deep && col < cut.cols) {
        typename OP::Coef k[V];
#pragma unroll
        for (int i = 0; i < V; i++) k[i] = OP::coef(x, sh, stats, at.n, (col * V + i) % sh.C, w, b, wt, bt);
        const int64_t lo = at.chunk * cut.per, hi = min(lo + cut.per, cut.periods), whole = min(hi, sh.S / cut.rows);
        const R *px = (const R *)x.p + at.n * x.sn + col * V, *pd = (const R *)dy.p + (OP::kTwo ? at.n * dy.sn + col * V : 0);
        const int64_t dx = cut.rows * x.ss, dd = cut.rows * dy.ss;
        int64_t p = lo + r;
#pragma unroll 4
        for (; p < whole; p += cut.deep) {
            float a[V], d[V] = {};
            load<T, V>(px + p * dx, a);
            if (OP::kTwo) load<T, V>(pd + p * dd, d);
#pragma unroll
            for (int i = 0; i < V; i++) OP::add(k[i], sh.slope, a[i], d[i], s[i], q[i]);
        }
        if (p < hi) {                                                      // the part period behind the last whole one
            const int64_t left = (sh.S - p * cut.rows) * sh.C - col * V;
#pragma unroll
            for (int i = 0; i < V; i++)
                if (i < left) OP::add(k[i], sh.slope, (float)px[p * dx + i], OP::kTwo ? (float)pd[p * dd + i] : 0.f, s[i], q[i]);
        }
    }
    // [sum][i][thread]: a channel's column is a period's value e = channel + m C, in each of `deep` periods
    const int T0 = blockDim.x;
#pragma unroll
    for (int i = 0; i < V; i++) {
        lds[i * T0 + threadIdx.x] = s[i];
        lds[(V + i) * T0 + threadIdx.x] = q[i];
    }
    __syncthreads();
    const int first = cut.rows == 1 ? at.mid * cut.tile * V : 0, many = cut.rows == 1 ? min(cut.tile * V, sh.C - first) : sh.C;
    for (int j = threadIdx.x; j < many; j += T0) {
        double a = 0, c = 0;
        for (int m = 0; m < cut.rows; m++) {
            const int e = j + m * sh.C, o = (e % V) * T0 + e / V;
            for (int d = 0; d < cut.deep; d++) {
                a += lds[o + d * cut.tile];
                c += lds[V * T0 + o + d * cut.tile];
            }
        }
        part[((int64_t)at.n * cut.chunks + at.chunk) * sh.C + first + j] = make_double2(a, c);
    }
}

template <class T, int V, class OP>
__global__ __launch_bounds__(512) void last_value_kernel(Map x, Map dy, Map out, Shape sh, Cut cut, const double *stats, const double *sums,
                                                         const void *w, const void *b, int wt, int bt)
{
    using R = typename T::raw;
    const Where at = where(cut.tiles, cut.chunks);
    const int r = threadIdx.x / cut.tile, in = threadIdx.x % cut.tile, col = at.mid * cut.tile + in;
    if (r >= cut.deep || col >= cut.cols) return;
    typename OP::Coef k[V];
#pragma unroll
    for (int i = 0; i < V; i++) k[i] = OP::coef(sh, stats, sums, at.n, (col * V + i) % sh.C, w, b, wt, bt);
    const int64_t lo = at.chunk * cut.per, hi = min(lo + cut.per, cut.periods), whole = min(hi, sh.S / cut.rows);
    const R *px = (const R *)x.p + at.n * x.sn + col * V, *pd = (const R *)dy.p + (OP::kTwo ? at.n * dy.sn + col * V : 0);
    R *po = (R *)out.p + at.n * out.sn + col * V;
    const int64_t dx = cut.rows * x.ss, dd = cut.rows * dy.ss, dout = cut.rows * out.ss;
    int64_t p = lo + r;
#pragma unroll 4
    for (; p < whole; p += cut.deep) {
        float a[V], d[V] = {}, v[V];
        load<T, V>(px + p * dx, a);
        if (OP::kTwo) load<T, V>(pd + p * dd, d);
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = OP::value(k[i], sh.slope, a[i], d[i]);
        store<T, V>(po + p * dout, v);
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
__global__ __launch_bounds__(256) void first_sums_kernel(Map x, Map dy, Shape sh, int chunks, int64_t per, const double *stats, const void *w,
                                                         const void *b, int wt, int bt, double2 *part)
{
    using R = typename T::raw;
    __shared__ double lds[16];
    const Where at = where(sh.C, chunks);
    const typename OP::Coef k = OP::coef(x, sh, stats, at.n, at.mid, w, b, wt, bt);
    const R *px = (const R *)x.p + at.n * x.sn + at.mid * x.sc, *pd = (const R *)dy.p + (OP::kTwo ? at.n * dy.sn + at.mid * dy.sc : 0);
    const int64_t hi = min((at.chunk + 1) * per, sh.S);
    double s[V], q[V];
#pragma unroll
    for (int i = 0; i < V; i++) s[i] = q[i] = 0;
    int64_t e = at.chunk * per + threadIdx.x * V;
#pragma unroll 4
    for (; e + V <= hi; e += blockDim.x * V) {
        float a[V], d[V] = {};
        load<T, V>(px + e, a);
        if (OP::kTwo) load<T, V>(pd + e, d);
#pragma unroll
        for (int i = 0; i < V; i++) OP::add(k, sh.slope, a[i], d[i], s[i], q[i]);
    }
#pragma unroll
    for (int i = 0; i < V; i++)
        if (e + i < hi) OP::add(k, sh.slope, (float)px[e + i], OP::kTwo ? (float)pd[e + i] : 0.f, s[i], q[i]);
#pragma unroll
    for (int i = 1; i < V; i++) { s[0] += s[i]; q[0] += q[i]; }
    const double a = block_sum(s[0], lds), c = block_sum(q[0], lds);
    if (threadIdx.x == 0) part[((int64_t)at.n * chunks + at.chunk) * sh.C + at.mid] = make_double2(a, c);
}

template <class T, int V, class OP>
__global__ __launch_bounds__(256) void first_value_kernel(Map x, Map dy, Map out, Shape sh, int chunks, int64_t per, const double *stats,
                                                          const double *sums, const void *w, const void *b, int wt, int bt)
{
    using R = typename T::raw;
    const Where at = where(sh.C, chunks);
    const typename OP::Coef k = OP::coef(sh, stats, sums, at.n, at.mid, w, b, wt, bt);
    const R *px = (const R *)x.p + at.n * x.sn + at.mid * x.sc, *pd = (const R *)dy.p + (OP::kTwo ? at.n * dy.sn + at.mid * dy.sc : 0);
    R *po = (R *)out.p + at.n * out.sn + at.mid * out.sc;
    const int64_t hi = min((at.chunk + 1) * per, sh.S);
    int64_t e = at.chunk * per + threadIdx.x * V;
#pragma unroll 4
    for (; e + V <= hi; e += blockDim.x * V) {
        float a[V], d[V] = {}, v[V];
        load<T, V>(px + e, a);
        if (OP::kTwo) load<T, V>(pd + e, d);
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = OP::value(k, sh.slope, a[i], d[i]);
        store<T, V>(po + e, v);
    }
#pragma unroll
    for (int i = 0; i < V; i++)
        if (e + i < hi) po[e + i] = (R)OP::value(k, sh.slope, (float)px[e + i], OP::kTwo ? (float)pd[e + i] : 0.f);
}

// ---- between the passes -----------------------------------------------------------------------------------------
// one workgroup per image and group: the chunks' sums -> mean and 1 / sqrt(var + eps)
template <class T>
__global__ __launch_bounds__(256) void stats_kernel(Map x, Shape sh, int chunks, const double2 *part, double *stats)
{
    __shared__ double lds[16];
    const int n = blockIdx.x / sh.G, g = blockIdx.x % sh.G;
    const double2 *p = part + (int64_t)n * chunks * sh.C + g * sh.cg;
    double s = 0, q = 0;
    for (int64_t i = threadIdx.x; i < (int64_t)chunks * sh.cg; i += blockDim.x) {
        const double2 v = p[i / sh.cg * sh.C + i % sh.cg];
        s += v.x;
        q += v.y;
    }
    s = block_sum(s, lds);
    q = block_sum(q, lds);
    if (threadIdx.x == 0) {
        const double d = s / sh.m, var = fma(-d, d, q / sh.m);
        stats[blockIdx.x] = first_value<T>(x, sh, n, g) + d;                // (equal values: the mean is theirs, exactly)
        stats[sh.N * sh.G + blockIdx.x] = 1. / sqrt((var < 0 ? 0. : var) + sh.eps);      // (a NaN stays one)
    }
}

// one workgroup per image and group: the chunks' sums -> per channel (for dw, db) and, weighted, per group (m1, m2)
__global__ __launch_bounds__(256) void group_sums_kernel(Shape sh, int chunks, const double2 *part, const double *stats, const void *w, int wt, double2 *chan, double *sums)
{
    __shared__ double lds[16];
    __shared__ double2 team[256];
    const int n = blockIdx.x / sh.G, g = blockIdx.x % sh.G;
    int lanes = 1;                                                         // threads of a team that add one channel's chunks
    while (lanes * 2 * sh.cg <= 256 && lanes < chunks) lanes *= 2;
    const int teams = 256 / lanes, l = threadIdx.x % lanes, first = threadIdx.x / lanes;
    const double r = stats[sh.N * sh.G + blockIdx.x];
    double m1 = 0, m2 = 0;
    for (int j0 = 0; j0 < sh.cg; j0 += teams) {
        const int j = j0 + first, c = g * sh.cg + j;
        double2 v = make_double2(0, 0);
        if (j < sh.cg)
            for (int i = l; i < chunks; i += lanes) {
                const double2 u = part[((int64_t)n * chunks + i) * sh.C + c];
                v.x += u.x;
                v.y += u.y;
            }
        __syncthreads();
        team[threadIdx.x] = v;
        __syncthreads();
        if (l == 0 && j < sh.cg) {
            for (int i = 1; i < lanes; i++) {
                v.x += team[threadIdx.x + i].x;
                v.y += team[threadIdx.x + i].y;
            }
            v.y *= r;                                                      // sum dz h
            chan[(int64_t)n * sh.C + c] = v;
            const double wc = load_param(w, wt, c, 1.f);
            m1 = fma(wc, v.x, m1);
            m2 = fma(wc, v.y, m2);
        }
    }
    m1 = block_sum(m1, lds);
    m2 = block_sum(m2, lds);
    if (threadIdx.x == 0) {
        sums[2 * blockIdx.x] = m1 / sh.m;
        sums[2 * blockIdx.x + 1] = m2 / sh.m;
    }
}

// ---- host -------------------------------------------------------------------------------------------------------
inline bool is_map_type(int32_t t) { return t == GENRE_F32 || t == GENRE_BF16 || t == GENRE_F16; }

int check_map(const char *op, const char *what, const genre_tensor *t, const genre_tensor *like)
{
    GENRE_REQUIRE(t && t->ndim == 3 && is_map_type(t->dtype), "%s: %s must be a [N,C,S] tensor of fp32, bf16 or fp16", op, what);
    GENRE_REQUIRE(same_shape(t, like), "%s: %s must have x's shape", op, what);
    GENRE_REQUIRE(t->dtype == like->dtype, "%s: %s must have x's dtype", op, what);
    GENRE_REQUIRE(t->data || numel(t) == 0, "%s: %s is NULL", op, what);
    for (int i = 0; i < 3; i++) GENRE_REQUIRE(t->stride[i] >= 0, "%s: %s has a negative stride", op, what);
    return 1;
}
int check_param(const char *op, const char *what, const genre_tensor *t, int64_t C)
{
    if (!t) return 1;
    GENRE_REQUIRE(t->data && t->ndim == 1 && is_map_type(t->dtype) && t->size[0] == C && (C == 1 || t->stride[0] == 1),
                  "%s: %s must be a contiguous [%lld] tensor of fp32, bf16 or fp16", op, what, (long long)C);
    return 1;
}

inline bool channels_last(const genre_tensor *t) { return t->size[1] == 1 ? t->stride[2] != 1 && t->size[2] != 1 : t->stride[1] == 1 && (t->size[2] == 1 || t->stride[2] != 1); }
inline bool channels_first(const genre_tensor *t) { return t->size[2] == 1 || t->stride[2] == 1; }
inline bool gapless(const genre_tensor *t) { return t->size[2] == 1 || t->stride[2] == t->size[1]; }
inline Map map_of(const genre_tensor *t) { return {t->data, t->stride[0], t->stride[1], t->size[2] == 1 ? t->size[1] : t->stride[2]}; }

constexpr int kWorkgroups = 2048;                                          // eight of 256 threads for each CU

// values per thread and access: 16 bytes; fewer only where a channels-last column may not cross a row's end
int width_of(const genre_tensor *x, bool last, bool dense)
{
    int v = x->dtype == GENRE_F32 ? 4 : 8;
    if (last) {
        const int C = (int)x->size[1];
        if (!dense || C / gcd(C, v) > 512) v = gcd(C, v);
    }
    return v;
}

Cut cut_of(int N, int C, int64_t S, int v)
{
    Cut c;
    const int g = gcd(C, v);
    c.rows = v / g;
    c.cols = C / g;
    c.tiles = ceil_div(c.cols, 512);
    c.tile = ceil_div(c.cols, c.tiles);
    const int want = c.tile > 256 ? 512 : 256;
    c.deep = want / c.tile;
    c.threads = (c.deep * c.tile + 63) / 64 * 64;
    c.periods = (S + c.rows - 1) / c.rows;
    // four accesses a thread at least, then as many workgroups as fill the chip
    const int64_t turns = (c.periods + c.deep - 1) / c.deep, most = (turns + 3) / 4, fill = (kWorkgroups + (int64_t)N * c.tiles - 1) / ((int64_t)N * c.tiles);
    const int64_t chunks = most < fill ? most : fill;
    c.per = (turns + chunks - 1) / chunks * c.deep;
    c.chunks = (int)((c.periods + c.per - 1) / c.per);
    return c;
}

void first_cut(int N, int C, int64_t S, int v, int *threads, int *chunks, int64_t *per)
{
    *threads = S <= 64 * v * 4 ? 64 : 256;
    const int64_t step = (int64_t)*threads * v, turns = (S + step - 1) / step, most = (turns + 3) / 4;
    const int64_t fill = (kWorkgroups + (int64_t)N * C - 1) / ((int64_t)N * C), want = most < fill ? most : fill;
    *per = (turns + want - 1) / want * step;
    *chunks = (int)((S + *per - 1) / *per);
}

struct Call {
    Shape sh;
    bool last;
    int v;
    Cut cut;
    int threads, chunks;
    int64_t per;
    int64_t blocks() const { return (int64_t)sh.N * (last ? cut.tiles : sh.C) * chunks; }
};

int plan(const char *op, const genre_tensor *x, const genre_tensor *const *others, int n_others, int groups, Call &c)
{
    GENRE_REQUIRE(x->size[0] <= INT32_MAX && x->size[1] <= (1 << 24), "%s: too many images or channels", op);
    const int64_t N = x->size[0], C = x->size[1], S = x->size[2];
    GENRE_REQUIRE(groups > 0 && C > 0 && C % groups == 0, "%s: %lld channels do not split into %d groups", op, (long long)C, groups);
    GENRE_REQUIRE(N * C < (1 << 30), "%s: N*C must be below 2^30", op);
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
    if (last) {
        c.cut = cut_of((int)N, (int)C, S, c.v);
        c.chunks = c.cut.chunks;
        c.threads = c.cut.threads;
    } else {
        first_cut((int)N, (int)C, S, c.v, &c.threads, &c.chunks, &c.per);
    }
    GENRE_REQUIRE(c.blocks() < INT32_MAX && N * groups < INT32_MAX, "%s: the map is too large for one launch", op);
    return 1;
}

// fp64 values of the workspace: the chunks' sums; backward: and those per image and channel, per image and group
int64_t workspace_of(const Call &c, bool backward)
{
    const int64_t chan = (int64_t)c.sh.N * c.sh.C;
    return 2 * chan * c.chunks + (backward ? 2 * chan + 2 * (int64_t)c.sh.N * c.sh.G : 0);
}

int check_f64(const char *op, const char *what, const genre_tensor *t, int64_t least)
{
    if (least == 0) return 1;
    GENRE_REQUIRE(t && t->data && t->dtype == GENRE_F64 && is_contiguous(t) && numel(t) >= least,
                  "%s: %s must be a contiguous fp64 tensor of at least %lld values", op, what, (long long)least);
    return 1;
}

template <class T, int V, class OP>
void sums(const Call &c, const Map &x, const Map &dy, const Params &p, const double *stats, double2 *part, hipStream_t st)
{
    if (c.last)
        last_sums_kernel<T, V, OP><<<(int)c.blocks(), c.threads, sizeof(double) * 2 * V * c.threads, st>>>(x, dy, c.sh, c.cut, stats, p.w, p.b, p.wt, p.bt, part);
    else if constexpr (V * sizeof(typename T::raw) == 16)                  // (width_of narrows channels-last columns only)
        first_sums_kernel<T, V, OP><<<(int)c.blocks(), c.threads, 0, st>>>(x, dy, c.sh, c.chunks, c.per, stats, p.w, p.b, p.wt, p.bt, part);
}
template <class T, int V, class OP>
void values(const Call &c, const Map &x, const Map &dy, const Map &out, const Params &p, const double *stats, const double *sm, hipStream_t st)
{
    if (c.last)
        last_value_kernel<T, V, OP><<<(int)c.blocks(), c.threads, 0, st>>>(x, dy, out, c.sh, c.cut, stats, sm, p.w, p.b, p.wt, p.bt);
    else if constexpr (V * sizeof(typename T::raw) == 16)
        first_value_kernel<T, V, OP><<<(int)c.blocks(), c.threads, 0, st>>>(x, dy, out, c.sh, c.chunks, c.per, stats, sm, p.w, p.b, p.wt, p.bt);
}

template <class T, int V>
int forward(const Call &c, const Map &x, const Map &y, const Params &p, double *stats, double *ws, hipStream_t st)
{
    double2 *part = (double2 *)ws;
    sums<T, V, SumsF<T>>(c, x, Map{}, p, stats, part, st);
    GENRE_LAUNCH_CHECK("group norm sums");
    stats_kernel<T><<<c.sh.N * c.sh.G, 256, 0, st>>>(x, c.sh, c.chunks, part, stats);
    GENRE_LAUNCH_CHECK("group norm statistics");
    switch (c.sh.act) {
    case kActRelu: values<T, V, ValueF<T, kActRelu>>(c, x, Map{}, y, p, stats, nullptr, st); break;
    case kActLeaky: values<T, V, ValueF<T, kActLeaky>>(c, x, Map{}, y, p, stats, nullptr, st); break;
    case kActSilu: values<T, V, ValueF<T, kActSilu>>(c, x, Map{}, y, p, stats, nullptr, st); break;
    default: values<T, V, ValueF<T, kActNone>>(c, x, Map{}, y, p, stats, nullptr, st); break;
    }
    GENRE_LAUNCH_CHECK("group norm values");
    return 1;
}

template <class T, int V, int ACT>
int backward_as(const Call &c, const Map &x, const Map &dy, const Params &p, const Grads &g, const double *stats, double *ws, hipStream_t st)
{
    const int64_t nc = (int64_t)c.sh.N * c.sh.C;
    double2 *part = (double2 *)ws, *chan = part + nc * c.chunks;
    double *sm = (double *)(chan + nc);
    sums<T, V, SumsB<T, ACT>>(c, x, dy, p, stats, part, st);
    GENRE_LAUNCH_CHECK("group norm backward sums");
    group_sums_kernel<<<c.sh.N * c.sh.G, 256, 0, st>>>(c.sh, c.chunks, part, stats, p.w, p.wt, chan, sm);
    GENRE_LAUNCH_CHECK("group norm backward group sums");
    if (g.dw || g.db) {
        param_grads_kernel<<<ceil_div(c.sh.C, 256), 256, 0, st>>>(c.sh, chan, g.dw, g.dwt, g.db, g.dbt);
        GENRE_LAUNCH_CHECK("group norm parameter gradients");
    }
    if (g.dx.p) {
        values<T, V, ValueB<T, ACT>>(c, x, dy, g.dx, p, stats, sm, st);
        GENRE_LAUNCH_CHECK("group norm input gradient");
    }
    return 1;
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

}  // namespace
}  // namespace genre

using namespace genre;

extern "C" int64_t genre_group_norm_workspace(const genre_tensor *x, int groups, int backward)
{
    const char *op = "group_norm_workspace";
    Call c{};
    if (!x) { fail("%s: x is NULL", op); return -1; }
    if (!check_map(op, "x", x, x) || !plan(op, x, nullptr, 0, groups, c)) return -1;
    if (numel(x) == 0) return 0;
    if (small_fits(c.last, c.sh, x->dtype == GENRE_F32 ? 4 : 2, backward != 0)) return backward ? small_workspace(c.sh) : 0;
    int64_t need = workspace_of(c, backward != 0);
    if (c.last) {                                                          // a gap in another map's rows narrows the columns: room for both
        Call d = c;
        d.v = width_of(x, true, false);
        d.cut = cut_of(c.sh.N, c.sh.C, c.sh.S, d.v);
        d.chunks = d.cut.chunks;
        const int64_t other = workspace_of(d, backward != 0);
        if (other > need) need = other;
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
    if (!plan(op, x, others, 1, groups, c)) return 0;
    if (!check_f64(op, "stats", stats, 2 * (int64_t)c.sh.N * groups)) return 0;
    if (numel(x) == 0) return 1;
    c.sh.act = act;
    c.sh.slope = slope;
    c.sh.eps = eps;
    const Params p = {weight ? weight->data : nullptr, bias ? bias->data : nullptr, weight ? weight->dtype : 0, bias ? bias->dtype : 0};
    const Map mx = map_of(x), my = map_of(y);
    double *s = (double *)stats->data;
    hipStream_t st = (hipStream_t)stream;
    if (small_fits(c.last, c.sh, x->dtype == GENRE_F32 ? 4 : 2, false)) return small_forward(c.last, x->dtype, c.sh, mx, my, p, s, st);
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
    if (!plan(op, x, others, dx ? 2 : 1, groups, c)) return 0;
    if (!check_f64(op, "stats", stats, 2 * (int64_t)c.sh.N * groups)) return 0;
    hipStream_t st = (hipStream_t)stream;
    const Grads g = {dx ? map_of(dx) : Map{}, dw ? dw->data : nullptr, db ? db->data : nullptr, dw ? dw->dtype : 0, db ? db->dtype : 0};
    if (numel(x) == 0) {                                                   // sums over nothing
        if (g.dw || g.db) {
            Shape none = c.sh;
            none.N = 0;
            param_grads_kernel<<<ceil_div(none.C, 256), 256, 0, st>>>(none, nullptr, g.dw, g.dwt, g.db, g.dbt);
            GENRE_LAUNCH_CHECK("group norm parameter gradients");
        }
        return 1;
    }
    c.sh.act = act;
    c.sh.slope = slope;
    const Params p = {weight ? weight->data : nullptr, bias ? bias->data : nullptr, weight ? weight->dtype : 0, bias ? bias->dtype : 0};
    const Map mx = map_of(x), md = map_of(dy);
    const double *s = (const double *)stats->data;
    const bool small = small_fits(c.last, c.sh, x->dtype == GENRE_F32 ? 4 : 2, true);
    if (!check_f64(op, "ws", ws, small ? small_workspace(c.sh) : workspace_of(c, true))) return 0;
    double *b = ws ? (double *)ws->data : nullptr;
    if (small) return small_backward(c.last, x->dtype, c.sh, mx, md, p, g, s, b, st);
    if (x->dtype == GENRE_F32)
        return c.v == 4 ? backward<F32, 4>(c, mx, md, p, g, s, b, st) : c.v == 2 ? backward<F32, 2>(c, mx, md, p, g, s, b, st) : backward<F32, 1>(c, mx, md, p, g, s, b, st);
    if (x->dtype == GENRE_BF16)
        return GENRE_BY_WIDTH(BF16, c.v, (backward<BF16, 8>(c, mx, md, p, g, s, b, st)), (backward<BF16, 4>(c, mx, md, p, g, s, b, st)),
                              (backward<BF16, 2>(c, mx, md, p, g, s, b, st)), (backward<BF16, 1>(c, mx, md, p, g, s, b, st)));
    return GENRE_BY_WIDTH(F16, c.v, (backward<F16, 8>(c, mx, md, p, g, s, b, st)), (backward<F16, 4>(c, mx, md, p, g, s, b, st)),
                          (backward<F16, 2>(c, mx, md, p, g, s, b, st)), (backward<F16, 1>(c, mx, md, p, g, s, b, st)));
}
