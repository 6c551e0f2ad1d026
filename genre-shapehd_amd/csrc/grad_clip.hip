// grad_clip.hip -- operators over all of a network's tensors at once: the norm of the gradients together, the scaling that
// clips them, and the Adam step that takes the clip's factor with it (so that a clipped gradient need not be written at all).
//
//   norm = sqrt(sum g^2) (fp64 sums) or max |g|;  factor = min(1, max_norm / (norm + 1e-6))
//   g' = g factor + wd p;  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2;  p -= lr / c1 m / (sqrt(v) / sqrt(c2) + eps)
//
// All of it streams: each value is read (and written) once, a few operations each.  The tensors' addresses travel in the kernel's
// arguments -- no table in device memory, so nothing has to outlive the call and a captured launch replays as it is -- which
// hold some 90 to 190 tensors; a longer list takes several launches.  Bound: HBM.  Measured: norm of the refiner's 214 MB 32 us
// (6.6 TB/s, half of it from the 256 MB cache) + 4 for the end of the sum; a clip that scales 45 MB in 6 tensors 28.6 us (scale_kernel
// 16 of them), 371 MB in 434 tensors 237 us (147); Adam on those 93 million weights, norm and clip included, 600 us for 3.0 GB.
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

// V values; no alignment beyond the type's is asked for (gfx950 loads and stores 16 bytes at any address)
template <class R, int V> using vec = R __attribute__((ext_vector_type(V), aligned(sizeof(R))));
template <class T, int V, bool STREAM = false>
__device__ __forceinline__ void load(const typename T::raw *p, float (&v)[V])
{
    typedef vec<typename T::raw, V> W;
    const W t = STREAM ? __builtin_nontemporal_load((const W *)p) : *(const W *)p;
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = (float)t[i];
}
template <class T, int V, bool STREAM = false>
__device__ __forceinline__ void store(typename T::raw *p, const float (&v)[V])
{
    typedef vec<typename T::raw, V> W;
    W t;
#pragma unroll
    for (int i = 0; i < V; i++) t[i] = (typename T::raw)v[i];
    if (STREAM) __builtin_nontemporal_store(t, (W *)p);
    else *(W *)p = t;
}

// What the norm sums (fp64 squares: fp32 ones overflow at 1e19) or takes the largest of: magnitudes as the integers that their
// bits are -- the order is the same, infinity is above all numbers and NaN above infinity.
struct Squares {
    using acc = double;
    __device__ static double of(double a, float x) { return fma((double)x, (double)x, a); }
    __device__ static double join(double a, double b) { return a + b; }
    __device__ static double norm(double a) { return sqrt(a); }
};
struct Largest {
    using acc = unsigned;
    __device__ static unsigned of(unsigned a, float x) { return max(a, __float_as_uint(x) & 0x7fffffffu); }
    __device__ static unsigned join(unsigned a, unsigned b) { return max(a, b); }
    __device__ static double norm(unsigned a) { return (double)__uint_as_float(a); }
};

template <class K>
__device__ __forceinline__ typename K::acc block_join(typename K::acc v, typename K::acc *lds)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v = K::join(v, __shfl_xor(v, o));
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    v = lds[0];
    for (int i = 1; i < (int)blockDim.x / 64; i++) v = K::join(v, lds[i]);
    return v;
}

template <class T, class K>
__global__ __launch_bounds__(kThreads) void norm_kernel(const Table<1> t, typename K::acc *part)
{
    constexpr int V = 16 / sizeof(typename T::raw);
    __shared__ typename K::acc lds[kThreads / 64];
    const Share s = share(t, blockIdx.x);
    const typename T::raw *g = (const typename T::raw *)t.p[0][s.tensor];
    typename K::acc acc[V];
#pragma unroll
    for (int i = 0; i < V; i++) acc[i] = 0;
    int64_t e = s.lo + threadIdx.x * V;
#pragma unroll 4
    for (; e + V <= s.hi; e += kThreads * V) {
        float a[V];
        load<T, V>(g + e, a);
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] = K::of(acc[i], a[i]);
    }
#pragma unroll
    for (int i = 0; i < V; i++)
        if (e + i < s.hi) acc[i] = K::of(acc[i], (float)g[e + i]);
#pragma unroll
    for (int i = 1; i < V; i++) acc[0] = K::join(acc[0], acc[i]);
    const typename K::acc v = block_join<K>(acc[0], lds);
    if (threadIdx.x == 0) part[blockIdx.x] = v;
}

template <class K>
__global__ __launch_bounds__(1024) void norm_end_kernel(const typename K::acc *part, int n, float max_norm, float *out)
{
    __shared__ typename K::acc lds[16];
    typename K::acc v = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += 1024) v = K::join(v, part[i]);
    v = block_join<K>(v, lds);
    if (threadIdx.x == 0) {
        const float norm = (float)K::norm(v), f = max_norm / (norm + 1e-6f);
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
    g *= f;
    if (k.decay != 0.f) g = fmaf(k.decay, p, g);                           // (0 times an infinite weight would be a NaN)
    m = fmaf(k.c1, g, k.b1 * m);
    v = fmaf(k.c2 * g, g, k.b2 * v);
    p = fmaf(-k.step_size, m / fmaf(sqrtf(v), k.inv_root_c2, k.eps), p * k.keep);
}

template <class T>
__global__ __launch_bounds__(kThreads) void adam_kernel(const Table<4> t, const float *factor, Adam k)
{
    // the states are streamed past the cache, where they would push out the weights and gradients (which the next forward and
    // the norm before read): critic's 317 MB 74.9 -> 63 us; streaming weights and gradients as well: 66-70 us
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
        load<F32, V, true>(m + e, c);
        load<F32, V, true>(v + e, d);
#pragma unroll
        for (int i = 0; i < V; i++) adam_value(k, f, a[i], b[i], c[i], d[i]);
        store<T, V>(p + e, a);
        store<F32, V, true>(m + e, c);
        store<F32, V, true>(v + e, d);
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
// A launch's values per workgroup: some `workgroups` of them for what its table holds, 4 accesses of a thread at least, 128 at
// most.  The norm takes 2048, the number that the chip holds at once (1024 / 1536 / 2048 / 4096: 45.3 / 42.0 / 42.8 / 44.1 us for
// the refiner's 214 MB); the Adam step, whose workgroups move seven streams, four
// times that (2048 / 4096 / 6144 / 8192: 633 / 619 / 617 / 603 us for 93 million weights).  By the list's total instead, the shorter
// tables of a long list did not fill the chip (98 us against 85 for the joint model's norm).
constexpr int kNormWorkgroups = 2048, kAdamWorkgroups = 8192;
constexpr int64_t kLeast = kThreads * 4 * 4;
inline int64_t chunk_of(int64_t total, int workgroups)
{
    const int64_t c = (total / workgroups + kLeast - 1) / kLeast * kLeast;
    return c < kLeast ? kLeast : c > 32 * kLeast ? 32 * kLeast : c;
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
    GENRE_REQUIRE(total / (16 * kThreads * 128) < (1 << 30), "%s: too many values", op);
    return 1;
}
template <class PTR>
int check_ptrs(const char *op, const char *what, PTR const *p, const int64_t *numels, int n)
{
    GENRE_REQUIRE(p || n == 0, "%s: %s is NULL", op, what);
    for (int i = 0; i < n; i++) GENRE_REQUIRE(p[i] || numels[i] == 0, "%s: %s of tensor %d is NULL", op, what, i);
    return 1;
}

// the list cut into tables of one type each; run(table, type, workgroups, workgroups before) launches one.  last_first: from the
// list's end, for a pass behind one that read it from the front -- what that read last is still in the cache (256 MB)
template <int P, class RUN>
int each_table(void *const *const (&ptrs)[P], const int64_t *numels, const int32_t *dtypes, int n, bool last_first, const RUN &run)
{
    static_assert(sizeof(Table<P>) <= kArgBytes + 64, "a launch's arguments");
    Table<P> t;
    int64_t before = 0;
    for (int j = 0; j < 3; j++) {
        const int types[3] = {GENRE_F32, GENRE_BF16, GENRE_F16}, type = types[last_first ? 2 - j : j];
        int64_t total = 0;
        t.n = 0;
        for (int k = 0; k <= n; k++) {
            const int i = last_first ? n - 1 - k : k;
            const bool end = k == n;
            if (!end && (dtypes[i] != type || !numels[i])) continue;
            if (t.n == Table<P>::kMost || (end && t.n)) {
                int64_t blocks = 0;
                t.chunk = chunk_of(total, P == 1 ? kNormWorkgroups : kAdamWorkgroups);
                for (int m = 0; m < t.n; m++) {
                    t.first[m] = (int)blocks;
                    blocks += (t.numel[m] + t.chunk - 1) / t.chunk;
                }
                GENRE_REQUIRE(blocks <= INT32_MAX, "too many values for a launch");
                if (!run(t, type, (int)blocks, before)) return 0;
                before += blocks;
                total = 0;
                t.n = 0;
            }
            if (end) break;
            for (int m = 0; m < P; m++) t.p[m][t.n] = ptrs[m][i];
            t.numel[t.n++] = numels[i];
            total += numels[i];
        }
    }
    return 1;
}

// no fewer than the workgroups of all tables together: each tensor rounds up by less than one, a table's chunk divides its
// values into kNormWorkgroups or is kLeast or 32 kLeast
inline int64_t most_blocks(const int64_t *numels, int n)
{
    int64_t total = 0;
    for (int i = 0; i < n; i++) total += numels[i];
    const int64_t tables = n / Table<1>::kMost + 3, filled = tables * kNormWorkgroups + total / (32 * kLeast), small = total / kLeast;
    return n + (small < filled ? small : filled);
}

int check_f32(const char *op, const char *what, const genre_tensor *t, int64_t least)
{
    GENRE_REQUIRE(t && t->data && t->dtype == GENRE_F32 && is_contiguous(t) && numel(t) >= least,
                  "%s: %s must be a contiguous fp32 tensor of at least %lld values", op, what, (long long)least);
    return 1;
}

template <class K>
int norm_of(const void *const *ptrs, const int64_t *numels, const int32_t *dtypes, int n, float max_norm, float *out, void *ws, hipStream_t st)
{
    int64_t blocks = 0;
    typename K::acc *part = (typename K::acc *)ws;
    void *const *const lists[1] = {(void *const *)ptrs};
    const int ok = each_table<1>(lists, numels, dtypes, n, false, [&](const Table<1> &t, int type, int b, int64_t before) {
        if (type == GENRE_F32) norm_kernel<F32, K><<<b, kThreads, 0, st>>>(t, part + before);
        else if (type == GENRE_BF16) norm_kernel<BF16, K><<<b, kThreads, 0, st>>>(t, part + before);
        else norm_kernel<F16, K><<<b, kThreads, 0, st>>>(t, part + before);
        GENRE_LAUNCH_CHECK("grad norm");
        blocks = before + b;
        return 1;
    });
    if (!ok) return 0;
    norm_end_kernel<K><<<1, 1024, 0, st>>>(part, (int)blocks, max_norm, out);
    GENRE_LAUNCH_CHECK("grad norm end");
    return 1;
}

}  // namespace
}  // namespace genre

using namespace genre;

extern "C" int64_t genre_grad_workspace(const int64_t *numels, int n)
{
    if (n < 0 || (n && !numels)) { fail("grad_workspace: the list of sizes is missing"); return -1; }
    int64_t total = 0;
    for (int i = 0; i < n; i++) {
        if (numels[i] < 0 || numels[i] >= ((int64_t)1 << 46) - total) { fail("grad_workspace: tensor %d has %lld values", i, (long long)numels[i]); return -1; }
        total += numels[i];
    }
    return most_blocks(numels, n);
}

extern "C" int genre_grad_norm(const void *const *ptrs, const int64_t *numels, const int32_t *dtypes, int n, int norm_type, float max_norm,
                               const genre_tensor *out, const genre_tensor *ws, void *stream)
{
    const char *op = "grad_norm";
    if (!check_list(op, numels, dtypes, n) || !check_ptrs(op, "pointer", ptrs, numels, n) || !check_f32(op, "out", out, 2)) return 0;
    GENRE_REQUIRE(norm_type == 2 || norm_type == 0, "%s: norm_type is 2 or 0 (largest magnitude)", op);
    GENRE_REQUIRE(max_norm >= 0, "%s: max_norm must not be negative", op);
    const int64_t blocks = most_blocks(numels, n);
    GENRE_REQUIRE(blocks == 0 || (ws && ws->data && ws->dtype == GENRE_F64 && is_contiguous(ws) && numel(ws) >= blocks),
                  "%s: ws must be a contiguous fp64 tensor of at least %lld values", op, (long long)blocks);
    hipStream_t st = (hipStream_t)stream;
    void *part = blocks ? ws->data : nullptr;
    return norm_type == 2 ? norm_of<Squares>(ptrs, numels, dtypes, n, max_norm, (float *)out->data, part, st)
                          : norm_of<Largest>(ptrs, numels, dtypes, n, max_norm, (float *)out->data, part, st);
}

extern "C" int genre_grad_scale(void *const *ptrs, const int64_t *numels, const int32_t *dtypes, int n, const genre_tensor *factor, void *stream)
{
    const char *op = "grad_scale";
    if (!check_list(op, numels, dtypes, n) || !check_ptrs(op, "pointer", ptrs, numels, n) || !check_f32(op, "factor", factor, 1)) return 0;
    hipStream_t st = (hipStream_t)stream;
    const float *f = (const float *)factor->data;
    void *const *const lists[1] = {ptrs};
    return each_table<1>(lists, numels, dtypes, n, true, [&](const Table<1> &t, int type, int b, int64_t) {
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
    return each_table<4>(lists, numels, dtypes, n, true, [&](const Table<4> &t, int type, int b, int64_t) {
        if (type == GENRE_F32) adam_kernel<F32><<<b, kThreads, 0, st>>>(t, f, k);
        else if (type == GENRE_BF16) adam_kernel<BF16><<<b, kThreads, 0, st>>>(t, f, k);
        else adam_kernel<F16><<<b, kThreads, 0, st>>>(t, f, k);
        GENRE_LAUNCH_CHECK("adam step");
        return 1;
    });
}
