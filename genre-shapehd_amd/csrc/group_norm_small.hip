// group_norm_small.hip -- group normalisation where one workgroup holds an image's group in its registers.
//
// A map whose groups hold up to 16384 values (backward: 8192 channels last, 4096 first) takes one launch (backward of several images:
// and one that adds up their dw and db) and reads x (and dy) once.  A group is `rows` runs of `cols` accesses of V values: channels
// last, a run is one position's cg channels and every thread keeps one column; channels first, a run is one channel's positions,
// shared by a team of 2^k threads.
//
// Bound: latency -- one load's way to memory and back, two sums over a workgroup, the stores: 3.5 us for 640 channels of one
// position, 5.8 for 10240 values a group, against 8 to 10 us in the two passes of group_norm.hip.  With 64 values a thread instead of
// 16 (25803 values a group: 17 us, backward 26) the two passes are faster (8 and 9).
#include "group_norm.hpp"

namespace genre {
namespace {

using namespace gn;

// threads of the largest workgroup -- backward, whose columns' sums take 64 bytes of LDS a thread, fewer -- and values of a thread
constexpr int kThreads = 1024, kBackwardThreads = 512, kValues = 16;

struct Small {
    int rows, cols;
    int team, deep, turns, subs;                                           // threads of a run, runs at once, accesses of a thread and run, waves of a team
    int64_t gsx, gsd, gso, psx, psd, pso;                                  // a group's stride and a run's in x, dy, out (elements)
};

// a run-time activation -- a kernel for each would be four times as many -- chosen once around a loop over the values
template <class F>
__device__ __forceinline__ void with_act(int act, const F &f)
{
    switch (act) {
    case kActRelu: f(std::integral_constant<int, kActRelu>()); break;
    case kActLeaky: f(std::integral_constant<int, kActLeaky>()); break;
    case kActSilu: f(std::integral_constant<int, kActSilu>()); break;
    default: f(std::integral_constant<int, kActNone>()); break;
    }
}

// sum over each team of 2^k neighbouring lanes (teams of more: over the wave), in every one of them
__device__ __forceinline__ double team_sum(double v, int team)
{
    if (team >= 64) return wave_sum(v);
    if (team >= 2) v += dpp_f64<0xb1, 0xf>(0., v);                         // quad_perm [1,0,3,2]
    if (team >= 4) v += dpp_f64<0x4e, 0xf>(0., v);                         // quad_perm [2,3,0,1]
    if (team >= 8) v += dpp_f64<0x141, 0xf>(0., v);                        // row_half_mirror: the other four of eight, equal by now
    if (team >= 16) v += dpp_f64<0x140, 0xf>(0., v);                       // row_mirror: the other eight
    if (team >= 32) v += __shfl_xor(v, 16);
    return v;
}

// Workgroups go round the eight dies; a die gets consecutive groups here, so that those of one image, whose channels share
// cache lines, meet in one L2.
__device__ __forceinline__ int by_die(int b, int n)
{
    const int die = b & 7, each = n >> 3, more = n & 7;
    return die * each + min(die, more) + (b >> 3);
}

// a thread's accesses, one after the other: run, column (in accesses), and whether there is one
template <bool LAST>
struct Walk {
    const Small &m;
    int row, col, turn;
    bool idle;
    __device__ explicit Walk(const Small &m) : m(m), idle(LAST && (int)threadIdx.x >= m.team * m.deep) { restart(); }
    __device__ void restart()
    {
        row = threadIdx.x / m.team;
        col = threadIdx.x % m.team;
        asm volatile("" : "+v"(row), "+v"(col));                           // (not the last pass's addresses and masks, kept in registers)
        turn = 0;
    }
    __device__ bool here() const { return LAST ? !idle && row < m.rows : row < m.rows && col < m.cols; }
    __device__ int channel(int v) const { return LAST ? col * v : row; }   // of the access's first value
    __device__ bool ends_run() const { return turn + 1 == m.turns; }
    __device__ void next()
    {
        if (LAST) {
            row += m.deep;
        } else if (++turn == m.turns) {
            turn = 0;
            col = threadIdx.x % m.team;
            row += m.deep;
        } else {
            col += m.team;
        }
    }
};

template <class T, int V, bool LAST>
__global__ __launch_bounds__(kThreads) void small_forward_kernel(Map x, Map y, Shape sh, Small m, double *stats, const void *w, const void *b, int wt, int bt)
{
    using R = typename T::raw;
    constexpr int K = kValues / V;
    extern __shared__ double coef[];                                       // a and b of the group's channels
    __shared__ double lds[32];
    const int id = by_die(blockIdx.x, gridDim.x), n = id / sh.G, g = id % sh.G;
    const R *px = (const R *)x.p + n * x.sn + g * m.gsx;
    R *py = (R *)y.p + n * y.sn + g * m.gso;
    Kept<T, V> v[K];
    Walk<LAST> at(m);
#pragma unroll
    for (int k = 0; k < K; k++, at.next())
        if (at.here()) v[k].load(px + at.row * m.psx + at.col * V);
    const double x0 = (double)(float)px[0];
    double s = 0, q = 0;
    at.restart();
#pragma unroll
    for (int k = 0; k < K; k++, at.next())
        if (at.here())
#pragma unroll
            for (int i = 0; i < V; i++) {
                const double d = (double)v[k].at(i) - x0;
                s += d;
                q = fma(d, d, q);
            }
    block_sum2(s, q, lds);
    s /= sh.m;
    q /= sh.m;
    const double mean = x0 + s, var = fma(-s, s, q), r = 1. / sqrt((var < 0 ? 0. : var) + sh.eps);
    if (threadIdx.x == 0) {
        stats[id] = mean;
        stats[sh.N * sh.G + id] = r;
    }
    for (int c = threadIdx.x; c < sh.cg; c += blockDim.x) {
        coef[c] = r * load_param(w, wt, g * sh.cg + c, 1.f);
        coef[sh.cg + c] = load_param(b, bt, g * sh.cg + c, 0.f);
    }
    __syncthreads();
    with_act(sh.act, [&](auto act) __attribute__((always_inline)) {
        Walk<LAST> at(m);
#pragma unroll
        for (int k = 0; k < K; k++, at.next())
            if (at.here()) {
                const int c = at.channel(V);
                float f[V];
                v[k].fresh();
#pragma unroll
                for (int i = 0; i < V; i++) f[i] = act_value<act>(fma((double)v[k].at(i) - mean, coef[c + (LAST ? i : 0)], coef[sh.cg + c + (LAST ? i : 0)]), sh.slope);
                store<T, V>(py + at.row * m.pso + at.col * V, f);
            }
    });
}

// chan: the sums of dz and dz (x - mean) by image and channel (more than one image: added up behind this), or dw and db themselves,
// whose types need not be those of weight and bias
template <class T, int V, bool LAST>
__global__ __launch_bounds__(kBackwardThreads) void small_backward_kernel(Map x, Map dy, Map dx, Shape sh, Small m, const double *stats, const void *w, const void *b, int wt,
                                                             int bt, double2 *chan, void *dw, void *db, int dwt, int dbt)
{
    using R = typename T::raw;
    constexpr int K = kValues / V;
    extern __shared__ double coef[];                                       // a, b, w; then the sums' scratch
    __shared__ double lds[32];
    const int id = by_die(blockIdx.x, gridDim.x), n = id / sh.G, g = id % sh.G, cg = sh.cg;
    const R *px = (const R *)x.p + n * x.sn + g * m.gsx, *pd = (const R *)dy.p + n * dy.sn + g * m.gsd;
    R *po = (R *)dx.p + n * dx.sn + g * m.gso;
    double2 *scratch = (double2 *)(coef + 3 * cg + (cg & 1));
    Kept<T, V> v[K], d[K];
    Walk<LAST> at(m);
#pragma unroll
    for (int k = 0; k < K; k++, at.next())
        if (at.here()) {
            v[k].load(px + at.row * m.psx + at.col * V);
            d[k].load(pd + at.row * m.psd + at.col * V);
        }
    const double mean = stats[id], r = stats[sh.N * sh.G + id];
    for (int c = threadIdx.x; c < cg; c += blockDim.x) {
        const double wc = load_param(w, wt, g * cg + c, 1.f);
        coef[c] = r * wc;
        coef[cg + c] = load_param(b, bt, g * cg + c, 0.f);
        coef[2 * cg + c] = wc;
    }
    __syncthreads();
    // the sums of dz and dz (x - mean) of this thread's channels (last) or of its run (first)
    double2 acc[LAST ? V : 1];
#pragma unroll
    for (int i = 0; i < (LAST ? V : 1); i++) acc[i] = make_double2(0, 0);
    with_act(sh.act, [&](auto act) __attribute__((always_inline)) {
        Walk<LAST> at(m);
#pragma unroll
        for (int k = 0; k < K; k++, at.next()) {
            if (at.here()) {
                const int c = at.channel(V);
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const int e = LAST ? i : 0;
                    const double h = (double)v[k].at(i) - mean, dz = act_grad<act>(fma(h, coef[c + e], coef[cg + c + e]), d[k].at(i), sh.slope);
                    acc[e].x += dz;
                    acc[e].y = fma(dz, h, acc[e].y);
                }
            }
            if (!LAST && at.ends_run()) {                                  // (uniform) the run's last turn: its team's sum, wave by wave
                acc[0].x = team_sum(acc[0].x, m.team);
                acc[0].y = team_sum(acc[0].y, m.team);
                if ((int)threadIdx.x % min(m.team, 64) == 0 && at.row < m.rows) scratch[at.row * m.subs + (int)threadIdx.x % m.team / 64] = acc[0];
                acc[0] = make_double2(0, 0);
            }
        }
    });
    if (LAST) {
#pragma unroll
        for (int i = 0; i < V; i++) scratch[i * blockDim.x + threadIdx.x] = acc[i];
        // a column's threads lie `team` apart: halve their number until one is left
        int live = m.deep;
        const int mine = threadIdx.x / m.team;
        while (live > 1) {
            const int half = (live + 1) / 2;
            __syncthreads();
            if (mine + half < live)
#pragma unroll
                for (int i = 0; i < V; i++) {
                    double2 &to = scratch[i * blockDim.x + threadIdx.x];
                    const double2 from = scratch[i * blockDim.x + threadIdx.x + half * m.team];
                    to.x += from.x;
                    to.y += from.y;
                }
            live = half;
        }
    }
    __syncthreads();
    double m1 = 0, m2 = 0;
    for (int c = threadIdx.x; c < cg; c += blockDim.x) {
        double2 a;
        if (LAST) {
            a = scratch[c % V * blockDim.x + c / V];
        } else {
            a = scratch[c * m.subs];
            for (int i = 1; i < m.subs; i++) {
                a.x += scratch[c * m.subs + i].x;
                a.y += scratch[c * m.subs + i].y;
            }
        }
        if (chan) chan[(int64_t)n * sh.C + g * cg + c] = a;
        a.y *= r;
        if (db) store_param(db, dbt, g * cg + c, a.x);
        if (dw) store_param(dw, dwt, g * cg + c, a.y);
        m1 = fma(coef[2 * cg + c], a.x, m1);
        m2 = fma(coef[2 * cg + c], a.y, m2);
    }
    if (!dx.p) return;                                                     // (uniform)
    block_sum2(m1, m2, lds);
    const double k2 = r * (m1 / sh.m), k3 = r * r * (m2 / sh.m);
    with_act(sh.act, [&](auto act) __attribute__((always_inline)) {
        Walk<LAST> at(m);
#pragma unroll
        for (int k = 0; k < K; k++, at.next())
            if (at.here()) {
                const int c = at.channel(V);
                float f[V];
                v[k].fresh();
                d[k].fresh();
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const int e = LAST ? i : 0;
                    const double h = (double)v[k].at(i) - mean, dz = act_grad<act>(fma(h, coef[c + e], coef[cg + c + e]), d[k].at(i), sh.slope);
                    f[i] = (float)fma(dz, coef[c + e], -fma(h, k3, k2));
                }
                store<T, V>(po + at.row * m.pso + at.col * V, f);
            }
    });
}

// ---- host -------------------------------------------------------------------------------------------------------
// Values of a group, channels first, up to which the backward takes this form: with more (and with odd numbers of positions, whose
// unrolled walk is 160 KB of code) the two-pass form is faster -- 4 x 160 x 8^3, 10240 values a group: 7.2 us against 12.3.
constexpr int kBackwardFirst = 4096;
constexpr int kMostChannels = 1024;                                        // of a group: its coefficients lie in LDS

// the small form of a call, if its groups fit
struct SmallCall { Small m; int v, threads; };

int pow2_from(int64_t n)
{
    int p = 1;
    while (p < n) p *= 2;
    return p;
}

bool small_of(bool last, const Shape &sh, int es, bool backward, const Map &x, const Map &d, const Map &out, SmallCall &c)
{
    const int cg = sh.cg;
    const int64_t S = sh.S;
    const int threads = backward ? kBackwardThreads : kThreads, most = backward && !last ? kBackwardFirst : threads * kValues;
    if (cg > kMostChannels || S > most || cg * S > most) return false;
    const int64_t run = last ? cg : S;
    // (run & 15 has run's powers of two up to 8; gcd(0, v) = v.)  Channels last, every value of a thread's column has sums of its own
    c.v = gcd((int)(run & 15), last ? 4 : 16 / es);
    if (c.v == 2) c.v = 1;
    if (backward && !last && c.v == 1) return false;
    Small &m = c.m;
    m.rows = last ? (int)S : cg;
    m.cols = (int)(run / c.v);
    m.psx = last ? x.ss : x.sc;
    m.psd = last ? d.ss : d.sc;
    m.pso = last ? out.ss : out.sc;
    m.gsx = cg * x.sc;
    m.gsd = cg * d.sc;
    m.gso = cg * out.sc;
    const int k = kValues / c.v;
    for (c.threads = 64; c.threads <= threads; c.threads *= 2) {
        m.turns = m.subs = 1;
        if (last) {
            m.team = m.cols;
            m.deep = c.threads / m.team;
            if (m.deep * k >= m.rows) return true;
            continue;
        }
        for (m.team = pow2_from(m.cols) < c.threads ? pow2_from(m.cols) : c.threads; m.team; m.team /= 2) {
            m.deep = c.threads / m.team;
            m.turns = (m.cols + m.team - 1) / m.team;
            m.subs = m.team > 64 ? m.team / 64 : 1;
            if (m.turns * ((m.rows + m.deep - 1) / m.deep) <= k) return true;
        }
    }
    return false;
}

template <class T, int V, bool LAST>
int forward_as(const Shape &sh, const SmallCall &k, const Map &x, const Map &y, const Params &p, double *stats, hipStream_t st)
{
    const size_t lds = 2 * sizeof(double) * sh.cg;
    const int blocks = sh.N * sh.G;
    small_forward_kernel<T, V, LAST><<<blocks, k.threads, lds, st>>>(x, y, sh, k.m, stats, p.w, p.b, p.wt, p.bt);
    GENRE_LAUNCH_CHECK("group norm");
    return 1;
}

template <class T, int V, bool LAST>
int backward_as(const Shape &sh, const SmallCall &k, const Map &x, const Map &dy, const Params &p, const Grads &g, const double *stats, double *ws, hipStream_t st)
{
    static_assert(8 * 3 * kMostChannels + 16 * 4 * kBackwardThreads + 512 <= 65536, "LDS of a launch");
    const bool one = sh.N == 1;
    const size_t lds = sizeof(double) * (3 * sh.cg + (sh.cg & 1)) + sizeof(double2) * (LAST ? V * k.threads : sh.cg * k.m.subs);
    double2 *chan = !one && (g.dw || g.db) ? (double2 *)ws : nullptr;
    small_backward_kernel<T, V, LAST><<<sh.N * sh.G, k.threads, lds, st>>>(x, dy, g.dx, sh, k.m, stats, p.w, p.b, p.wt, p.bt, chan, one ? g.dw : nullptr, one ? g.db : nullptr,
                                                                              g.dwt, g.dbt);
    GENRE_LAUNCH_CHECK("group norm backward");
    if (chan) {
        channel_grads_kernel<<<ceil_div(sh.C, 4), 256, 0, st>>>(sh, 1, chan, stats, g.dw, g.dwt, g.db, g.dbt);
        GENRE_LAUNCH_CHECK("group norm parameter gradients");
    }
    return 1;
}

}  // namespace

namespace gn {

int small_threads(bool last, const Shape &sh, int es, bool backward)
{
    SmallCall k;
    return small_of(last, sh, es, backward, Map{}, Map{}, Map{}, k) ? k.threads : 0;
}

int small_forward(bool last, int dtype, const Shape &sh, const Map &x, const Map &y, const Params &p, double *stats, hipStream_t st)
{
    SmallCall k;
    if (!small_of(last, sh, dtype == GENRE_F32 ? 4 : 2, false, x, x, y, k)) return fail("group norm: the groups are too large for one workgroup");
#define GENRE_AS(T, V) (last ? forward_as<T, ((V) < 4 ? (V) : 4), true>(sh, k, x, y, p, stats, st) : forward_as<T, V, false>(sh, k, x, y, p, stats, st))
    if (dtype == GENRE_F32) return k.v == 4 ? GENRE_AS(F32, 4) : GENRE_AS(F32, 1);
    if (dtype == GENRE_BF16) return k.v == 8 ? GENRE_AS(BF16, 8) : k.v == 4 ? GENRE_AS(BF16, 4) : GENRE_AS(BF16, 1);
    return k.v == 8 ? GENRE_AS(F16, 8) : k.v == 4 ? GENRE_AS(F16, 4) : GENRE_AS(F16, 1);
#undef GENRE_AS
}

int small_backward(bool last, int dtype, const Shape &sh, const Map &x, const Map &dy, const Params &p, const Grads &g, const double *stats, double *ws, hipStream_t st)
{
    SmallCall k;
    if (!small_of(last, sh, dtype == GENRE_F32 ? 4 : 2, true, x, dy, g.dx, k)) return fail("group norm: the groups are too large for one workgroup");
#define GENRE_AS(T, V) (last ? backward_as<T, ((V) < 4 ? (V) : 4), true>(sh, k, x, dy, p, g, stats, ws, st) : backward_as<T, ((V) > 1 ? (V) : 4), false>(sh, k, x, dy, p, g, stats, ws, st))
    if (dtype == GENRE_F32) return k.v == 4 ? GENRE_AS(F32, 4) : GENRE_AS(F32, 1);
    if (dtype == GENRE_BF16) return k.v == 8 ? GENRE_AS(BF16, 8) : k.v == 4 ? GENRE_AS(BF16, 4) : GENRE_AS(BF16, 1);
    return k.v == 8 ? GENRE_AS(F16, 8) : k.v == 4 ? GENRE_AS(F16, 4) : GENRE_AS(F16, 1);
#undef GENRE_AS
}

}  // namespace gn
}  // namespace genre
