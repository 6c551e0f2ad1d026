// grad_clip.hip -- operators over all of a network's tensors at once: the norm of the gradients together, the scaling that
// clips them, and the Adam step that takes the clip's factor with it (so that a clipped gradient need not be written at all).
//
//   norm = sqrt(sum g^2) (fp64 sums) or max |g|;  factor = min(1, max_norm / (norm + 1e-6))
//   g' = g factor + wd p;  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2;  p -= lr / c1 m / (sqrt(v) / sqrt(c2) + eps)
//
// All of it streams: each value is read (and written) once, a few operations each.  The tensors' addresses travel in the kernel's
// arguments -- no table in device memory, so nothing has to outlive the call and a captured launch replays as it is -- which
// hold some 90 to 190 tensors; a longer list takes several launches of the same size of share.
#include "common.hpp"

namespace genre {
namespace {

constexpr int kThreads = 256;
constexpr int kArgBytes = 3968;                                            // a launch's arguments stay below 4 KB

struct F32 { using raw = float; };
struct F16 { using raw = _Float16; };
struct BF16 { using raw = __bf16; };

// `P` pointers and a size per tensor; first[i]: the workgroup a tensor's share begins with
template <int P>
struct Table {
    static constexpr int kMost = kArgBytes / (8 * P + 12);
    int n;
    int64_t chunk;                                                         // values per workgroup
    void *p[P][kMost];
    int64_t numel[kMost];
    int first[kMost];
};

struct Share { int tensor; int64_t lo, hi; };
// which tensor this workgroup works on: the last whose first workgroup is not behind it.  Every lane compares a few entries, one
// round trip instead of a search's seven.
template <int P>
__device__ __forceinline__ Share share(const Table<P> &t, unsigned block)
{
    int before = 0;
    for (int i = 0; i < t.n; i += 64) {
        const int at = i + (int)(threadIdx.x & 63);
        before += __popcll(__ballot(at < t.n && t.first[at < t.n ? at : 0] <= (int)block));
    }
    const int k = __builtin_amdgcn_readfirstlane(before - 1);
    const int64_t lo = (int64_t)((int)block - t.first[k]) * t.chunk, n = t.numel[k];
    return {k, lo, lo + t.chunk < n ? lo + t.chunk : n};
}

template <class T, int V>
__device__ __forceinline__ void load(const typename T::raw *p, float (&v)[V])
{
    typename T::raw t[V];
    __builtin_memcpy(t, p, sizeof(t));                                     // (no alignment beyond the type's)
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = (float)t[i];
}
template <class T, int V>
__device__ __forceinline__ void store(typename T::raw *p, const float (&v)[V])
{
    typename T::raw t[V];
#pragma unroll
    for (int i = 0; i < V; i++) t[i] = (typename T::raw)v[i];
    __builtin_memcpy(p, t, sizeof(t));
}

// the larger magnitude; a NaN wins and stays
__device__ __forceinline__ double larger(double a, double b) { return a != a ? a : (b != b || b > a) ? b : a; }

template <bool MAX>
__device__ __forceinline__ double join(double a, double b) { return MAX ? larger(a, b) : a + b; }

template <bool MAX>
__device__ __forceinline__ double block_join(double v, double *lds)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v = join<MAX>(v, __shfl_xor(v, o));
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    v = lds[0];
    for (int i = 1; i < (int)blockDim.x / 64; i++) v = join<MAX>(v, lds[i]);
    return v;
}

template <class T, bool MAX>
__global__ __launch_bounds__(kThreads) void norm_kernel(const Table<1> t, double *part)
{
    constexpr int V = 16 / sizeof(typename T::raw);
    __shared__ double lds[kThreads / 64];
    const Share s = share(t, blockIdx.x);
    const typename T::raw *g = (const typename T::raw *)t.p[0][s.tensor];
    double acc[V];
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] = 0;
    int64_t e = s.lo + threadIdx.x * V;
#pragma unroll 4
    for (; e + V <= s.hi; e += kThreads * V) {
        float a[V];
        load<T, V>(g + e, a);
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] = MAX ? larger(acc[i], fabs((double)a[i])) : fma((double)a[i], (double)a[i], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < V; i++)
        if (e + i < s.hi) {
            const double a = (double)(float)g[e + i];
            acc[i] = MAX ? larger(acc[i], fabs(a)) : fma(a, a, acc[i]);
        }
#pragma unroll
    for (int i = 1; i < V; i++) acc[0] = join<MAX>(acc[0], acc[i]);
    const double v = block_join<MAX>(acc[0], lds);
    if (threadIdx.x == 0) part[blockIdx.x] = v;
}

template <bool MAX>
__global__ __launch_bounds__(1024) void norm_end_kernel(const double *part, int n, float max_norm, float *out)
{
    __shared__ double lds[16];
    double v = 0;
    for (int i = threadIdx.x; i < n; i += 1024) v = join<MAX>(v, part[i]);
    v = block_join<MAX>(v, lds);
    if (threadIdx.x == 0) {
        const float norm = (float)(MAX ? v : sqrt(v)), f = max_norm / (norm + 1e-6f);
        out[0] = norm;
        out[1] = max_norm == INFINITY ? 1.f : f > 1.f ? 1.f : f;           // (a NaN stays one)
    }
}

template <class T>
__global__ __launch_bounds__(kThreads) void scale_kernel(const Table<1> t, const float *factor)
{
    constexpr int V = 16 / sizeof(typename T::raw);
    const float f = *factor;
    if (f == 1.f) return;                                                  // value times 1 is the value
    const Share s = share(t, blockIdx.x);
    typename T::raw *g = (typename T::raw *)t.p[0][s.tensor];
    int64_t e = s.lo + threadIdx.x * V;
#pragma unroll 4
    for (; e + V <= s.hi; e += kThreads * V) {
        float a[V];
        load<T, V>(g + e, a);
#pragma unroll
        for (int i = 0; i < V; i++) a[i] *= f;
        store<T, V>(g + e, a);
    }
#pragma unroll
    for (int i = 0; i < V; i++)
        if (e + i < s.hi) g[e + i] = (typename T::raw)((float)g[e + i] * f);
}

struct Adam { float b1, c1, b2, c2, eps, step_size, inv_root_c2, decay, keep; };   // c = 1 - b; keep: 1 - lr wd where decoupled

__device__ __forceinline__ void adam_value(const Adam &k, float f, float &p, float g, float &m, float &v)
{
    g = fmaf(k.decay, p, g * f);
    m = fmaf(k.c1, g, k.b1 * m);
    v = fmaf(k.c2 * g, g, k.b2 * v);
    p = fmaf(-k.step_size, m / fmaf(sqrtf(v), k.inv_root_c2, k.eps), p * k.keep);
}

template <class T>
__global__ __launch_bounds__(kThreads) void adam_kernel(const Table<4> t, const float *factor, Adam k)
{
    constexpr int V = 4;
    const float f = factor ? *factor : 1.f;
    const Share s = share(t, blockIdx.x);
    typename T::raw *p = (typename T::raw *)t.p[0][s.tensor];
    const typename T::raw *g = (const typename T::raw *)t.p[1][s.tensor];
    float *m = (float *)t.p[2][s.tensor], *v = (float *)t.p[3][s.tensor];
    int64_t e = s.lo + threadIdx.x * V;
#pragma unroll 2
    for (; e + V <= s.hi; e += kThreads * V) {
        float a[V], b[V], c[V], d[V];
        load<T, V>(p + e, a);
        load<T, V>(g + e, b);
        load<F32, V>(m + e, c);
        load<F32, V>(v + e, d);
#pragma unroll
        for (int i = 0; i < V; i++) adam_value(k, f, a[i], b[i], c[i], d[i]);
        store<T, V>(p + e, a);
        store<F32, V>(m + e, c);
        store<F32, V>(v + e, d);
    }
#pragma unroll
    for (int i = 0; i < V; i++)
        if (e + i < s.hi) {
            float a = (float)p[e + i], c = m[e + i], d = v[e + i];
            adam_value(k, f, a, (float)g[e + i], c, d);
            p[e + i] = (typename T::raw)a;
            m[e + i] = c;
            v[e + i] = d;
        }
}

// ---- host -------------------------------------------------------------------------------------------------------
// values per workgroup: enough workgroups to fill the chip eight times over, 4 to 64 accesses of a thread each
int64_t chunk_of(const int64_t *numels, int n)
{
    int64_t total = 0;
    for (int i = 0; i < n; i++) total += numels[i];
    const int64_t least = kThreads * 4 * 4;
    int64_t c = (total / 2048 + least - 1) / least * least;
    return c < least ? least : c > 16 * least ? 16 * least : c;
}

int64_t blocks_of(const int64_t *numels, int n, int64_t chunk)
{
    int64_t b = 0;
    for (int i = 0; i < n; i++) b += (numels[i] + chunk - 1) / chunk;
    return b;
}

int check_list(const char *op, const int64_t *numels, const int32_t *dtypes, int n)
{
    GENRE_REQUIRE(n >= 0 && (n == 0 || (numels && dtypes)), "%s: the list of tensors is missing", op);
    int64_t total = 0;
    for (int i = 0; i < n; i++) {
        GENRE_REQUIRE(numels[i] >= 0 && numels[i] < ((int64_t)1 << 46) - total, "%s: tensor %d has %lld values", op, i, (long long)numels[i]);
        total += numels[i];
        GENRE_REQUIRE(dtypes[i] == GENRE_F32 || dtypes[i] == GENRE_BF16 || dtypes[i] == GENRE_F16, "%s: tensor %d is not fp32, bf16 or fp16", op, i);
    }
    GENRE_REQUIRE(total / (16 * kThreads * 16) < (1 << 30), "%s: too many values", op);
    return 1;
}
template <class PTR>
int check_ptrs(const char *op, const char *what, PTR const *p, const int64_t *numels, int n)
{
    GENRE_REQUIRE(p || n == 0, "%s: %s is NULL", op, what);
    for (int i = 0; i < n; i++) GENRE_REQUIRE(p[i] || numels[i] == 0, "%s: %s of tensor %d is NULL", op, what, i);
    return 1;
}

// the list cut into tables of one type each; run(table, type, workgroups, workgroups before) launches one
template <int P, class RUN>
int each_table(void *const *const (&ptrs)[P], const int64_t *numels, const int32_t *dtypes, int n, const RUN &run)
{
    static_assert(sizeof(Table<P>) <= kArgBytes + 64, "a launch's arguments");
    Table<P> t;
    t.chunk = chunk_of(numels, n);
    int64_t before = 0;
    for (int type : {GENRE_F32, GENRE_BF16, GENRE_F16}) {
        t.n = 0;
        int64_t blocks = 0;
        const auto flush = [&]() {
            if (!t.n) return 1;
            const int ok = run(t, type, (int)blocks, before);
            before += blocks;
            t.n = 0;
            blocks = 0;
            return ok;
        };
        for (int i = 0; i < n; i++) {
            if (dtypes[i] != type || !numels[i]) continue;
            const int64_t b = (numels[i] + t.chunk - 1) / t.chunk;
            if (t.n == Table<P>::kMost || blocks + b > INT32_MAX)
                if (!flush()) return 0;
            for (int j = 0; j < P; j++) t.p[j][t.n] = ptrs[j][i];
            t.numel[t.n] = numels[i];
            t.first[t.n] = (int)blocks;
            t.n++;
            blocks += b;
        }
        if (!flush()) return 0;
    }
    return 1;
}

int check_f32(const char *op, const char *what, const genre_tensor *t, int64_t least)
{
    GENRE_REQUIRE(t && t->data && t->dtype == GENRE_F32 && is_contiguous(t) && numel(t) >= least,
                  "%s: %s must be a contiguous fp32 tensor of at least %lld values", op, what, (long long)least);
    return 1;
}

}  // namespace
}  // namespace genre

using namespace genre;

extern "C" int64_t genre_grad_workspace(const int64_t *numels, int n)
{
    if (n < 0 || (n && !numels)) { fail("grad_workspace: the list of sizes is missing"); return -1; }
    for (int i = 0; i < n; i++)
        if (numels[i] < 0) { fail("grad_workspace: size %d is negative", i); return -1; }
    return blocks_of(numels, n, chunk_of(numels, n));
}

extern "C" int genre_grad_norm(const void *const *ptrs, const int64_t *numels, const int32_t *dtypes, int n, int norm_type, float max_norm,
                               const genre_tensor *out, const genre_tensor *ws, void *stream)
{
    const char *op = "grad_norm";
    if (!check_list(op, numels, dtypes, n) || !check_ptrs(op, "pointer", ptrs, numels, n) || !check_f32(op, "out", out, 2)) return 0;
    GENRE_REQUIRE(norm_type == 2 || norm_type == 0, "%s: norm_type is 2 or 0 (largest magnitude)", op);
    GENRE_REQUIRE(max_norm >= 0, "%s: max_norm must not be negative", op);
    const int64_t blocks = blocks_of(numels, n, chunk_of(numels, n));
    GENRE_REQUIRE(blocks == 0 || (ws && ws->data && ws->dtype == GENRE_F64 && is_contiguous(ws) && numel(ws) >= blocks),
                  "%s: ws must be a contiguous fp64 tensor of at least %lld values", op, (long long)blocks);
    hipStream_t st = (hipStream_t)stream;
    double *part = blocks ? (double *)ws->data : nullptr;
    const bool max = norm_type == 0;
    void *const *const lists[1] = {(void *const *)ptrs};
    const int ok = each_table<1>(lists, numels, dtypes, n, [&](const Table<1> &t, int type, int b, int64_t before) {
        double *to = part + before;
        if (type == GENRE_F32) max ? norm_kernel<F32, true><<<b, kThreads, 0, st>>>(t, to) : norm_kernel<F32, false><<<b, kThreads, 0, st>>>(t, to);
        else if (type == GENRE_BF16) max ? norm_kernel<BF16, true><<<b, kThreads, 0, st>>>(t, to) : norm_kernel<BF16, false><<<b, kThreads, 0, st>>>(t, to);
        else max ? norm_kernel<F16, true><<<b, kThreads, 0, st>>>(t, to) : norm_kernel<F16, false><<<b, kThreads, 0, st>>>(t, to);
        GENRE_LAUNCH_CHECK("grad norm");
        return 1;
    });
    if (!ok) return 0;
    if (max) norm_end_kernel<true><<<1, 1024, 0, st>>>(part, (int)blocks, max_norm, (float *)out->data);
    else norm_end_kernel<false><<<1, 1024, 0, st>>>(part, (int)blocks, max_norm, (float *)out->data);
    GENRE_LAUNCH_CHECK("grad norm end");
    return 1;
}

extern "C" int genre_grad_scale(void *const *ptrs, const int64_t *numels, const int32_t *dtypes, int n, const genre_tensor *factor, void *stream)
{
    const char *op = "grad_scale";
    if (!check_list(op, numels, dtypes, n) || !check_ptrs(op, "pointer", ptrs, numels, n) || !check_f32(op, "factor", factor, 1)) return 0;
    hipStream_t st = (hipStream_t)stream;
    const float *f = (const float *)factor->data;
    void *const *const lists[1] = {ptrs};
    return each_table<1>(lists, numels, dtypes, n, [&](const Table<1> &t, int type, int b, int64_t) {
        if (type == GENRE_F32) scale_kernel<F32><<<b, kThreads, 0, st>>>(t, f);
        else if (type == GENRE_BF16) scale_kernel<BF16><<<b, kThreads, 0, st>>>(t, f);
        else scale_kernel<F16><<<b, kThreads, 0, st>>>(t, f);
        GENRE_LAUNCH_CHECK("grad scale");
        return 1;
    });
}

extern "C" int genre_adam_step(void *const *p, const void *const *g, void *const *m, void *const *v, const int64_t *numels, const int32_t *dtypes, int n,
                               const genre_tensor *factor, int64_t step, double lr, double beta1, double beta2, double eps, double weight_decay,
                               int decoupled, void *stream)
{
    const char *op = "adam_step";
    if (!check_list(op, numels, dtypes, n) || !check_ptrs(op, "p", p, numels, n) || !check_ptrs(op, "g", g, numels, n) ||
        !check_ptrs(op, "m", m, numels, n) || !check_ptrs(op, "v", v, numels, n) || (factor && !check_f32(op, "factor", factor, 1)))
        return 0;
    GENRE_REQUIRE(step >= 1, "%s: step counts from 1", op);
    GENRE_REQUIRE(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "%s: the betas lie in [0, 1)", op);
    GENRE_REQUIRE(eps >= 0 && lr >= 0 && weight_decay >= 0, "%s: lr, eps and weight_decay must not be negative", op);
    Adam k;
    k.b1 = (float)beta1;
    k.c1 = (float)(1 - beta1);
    k.b2 = (float)beta2;
    k.c2 = (float)(1 - beta2);
    k.eps = (float)eps;
    k.step_size = (float)(lr / (1 - pow(beta1, (double)step)));
    k.inv_root_c2 = (float)(1 / sqrt(1 - pow(beta2, (double)step)));
    k.decay = decoupled ? 0.f : (float)weight_decay;
    k.keep = decoupled ? (float)(1 - lr * weight_decay) : 1.f;
    hipStream_t st = (hipStream_t)stream;
    const float *f = factor ? (const float *)factor->data : nullptr;
    void *const *const lists[4] = {p, (void *const *)g, m, v};
    return each_table<4>(lists, numels, dtypes, n, [&](const Table<4> &t, int type, int b, int64_t) {
        if (type == GENRE_F32) adam_kernel<F32><<<b, kThreads, 0, st>>>(t, f, k);
        else if (type == GENRE_BF16) adam_kernel<BF16><<<b, kThreads, 0, st>>>(t, f, k);
        else adam_kernel<F16><<<b, kThreads, 0, st>>>(t, f, k);
        GENRE_LAUNCH_CHECK("adam step");
        return 1;
    });
}
