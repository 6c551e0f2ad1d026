// group_norm.hpp -- what the two files of the group normalisation share (group_norm.hip: the mathematics, the entries and the
// kernels that walk a map in several passes; group_norm_small.hip: one workgroup per image and group).
#pragma once
#include "common.hpp"
#include "wave_scan.hpp"
#include <type_traits>

namespace genre {
namespace gn {

enum { kActNone = 0, kActRelu = 1, kActLeaky = 2, kActSilu = 3 };

// ---- element types ----------------------------------------------------------------------------------------------
struct F32 { using raw = float; };
struct F16 { using raw = _Float16; };
struct BF16 { using raw = __bf16; };
template <class R, int V> using vec = R __attribute__((ext_vector_type(V), aligned(sizeof(R))));

// STREAM: past the caches (else a launch's end waits until what it left dirty in the L2s is written).  The two-pass kernels store so
// whatever a map's size, the one-workgroup form does not.  fp32 channels first, streamed / not: 8 x 32 x 64^3 123 / 148 us (training
// 349 / 390), 4 x 20 x 64^3 42.5 / 42.5 (107 / 110), 4 x 40 x 32^3 15.6 / 16.0, 4 x 80 x 16^3 8.5 / 8.9 (17.1 / 17.6); with a pass that
// reads y behind it 231 / 246, 68.3 / 66.3, 24.1 / 23.5, 13.0 / 13.1
template <class T, int V, bool STREAM = false>
__device__ __forceinline__ void store(typename T::raw *p, const float (&v)[V])
{
    typedef vec<typename T::raw, V> W;
    W t;
#pragma unroll
    for (int i = 0; i < V; i++) t[i] = (typename T::raw)v[i];              // round to nearest even
    if (STREAM) __builtin_nontemporal_store(t, (W *)p);
    else *(W *)p = t;
}

// V values as they lie in memory: a thread keeps these, two 16-bit values to a register, and converts them in each pass.  Loads and
// stores need no more than their type's own alignment (gfx950 moves 16 bytes at any address).
template <class T, int V>
struct Kept {
    static constexpr int kWords = (V * sizeof(typename T::raw) + 3) / 4;
    unsigned word[kWords];
    __device__ void load(const typename T::raw *p)
    {
        if (V * sizeof(*p) == 2) word[0] = *(const unsigned short *)p;
        else __builtin_memcpy(word, p, V * sizeof(*p));
    }
    __device__ float at(int i) const
    {
        if (sizeof(typename T::raw) == 4) return __uint_as_float(word[i]);
        const unsigned short h = (unsigned short)(word[i / 2] >> (i % 2 * 16));
        return (float)__builtin_bit_cast(half_of, h);
    }
    // the conversions of one pass are not kept for the next (fp64: two registers a value)
    __device__ void fresh()
    {
#pragma unroll
        for (int i = 0; i < kWords; i++) asm volatile("" : "+v"(word[i]));
    }
    typedef typename std::conditional<sizeof(typename T::raw) == 2, typename T::raw, _Float16>::type half_of;
};

__device__ __forceinline__ float load_param(const void *p, int dtype, int c, float missing)
{
    if (!p) return missing;
    if (dtype == GENRE_F32) return ((const float *)p)[c];
    return dtype == GENRE_BF16 ? (float)((const __bf16 *)p)[c] : (float)((const _Float16 *)p)[c];
}
__device__ __forceinline__ void store_param(void *p, int dtype, int c, double v)
{
    if (dtype == GENRE_F32) ((float *)p)[c] = (float)v;
    else if (dtype == GENRE_BF16) ((__bf16 *)p)[c] = (__bf16)(float)v;
    else ((_Float16 *)p)[c] = (_Float16)(float)v;
}

// ---- activation -------------------------------------------------------------------------------------------------
// exp and the reciprocal are the hardware's: a few 2^-24 relative around zero, |z| 2^-24 far below it, where the sigmoid is
// e^-|z| and adds nothing to an output's error
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }

template <int ACT>
__device__ __forceinline__ float act_value(double z, float slope)
{
    const float f = (float)z;
    if (ACT == kActRelu) return f > 0.f || f != f ? f : 0.f;
    if (ACT == kActLeaky) return f > 0.f ? f : f * slope;
    if (ACT == kActSilu) return f * sigmoid(f);
    return f;
}
// dz of dy.  A ReLU that is off passes nothing on, whatever dy holds there (an infinity times 0 would be a NaN)
template <int ACT>
__device__ __forceinline__ float act_grad(double z, float dy, float slope)
{
    if (ACT == kActRelu) return z > 0 ? dy : 0.f;
    if (ACT == kActLeaky) return z > 0 ? dy : dy * slope;
    if (ACT == kActSilu) {
        const float f = (float)z, s = sigmoid(f);
        return dy * (s * fmaf(f, 1.f - s, 1.f));
    }
    return dy;
}

// ---- what the kernels know of a call ----------------------------------------------------------------------------
struct Map { void *p; int64_t sn, sc, ss; };                               // element strides of image, channel, position

struct Shape {
    int N, C, G, cg, act;
    int64_t S;
    float slope;
    double m, eps;                                                         // M
};

__device__ __forceinline__ double wave_sum(double v) { return wave_last(wave_incl_sum(v)); }
// sums over the workgroup of two values, in every thread; `lds` has 32 doubles (blockDim.x <= 1024)
__device__ __forceinline__ void block_sum2(double &a, double &b, double *lds)
{
    a = wave_sum(a);
    b = wave_sum(b);
    const int waves = (blockDim.x + 63) / 64;
    __syncthreads();
    if (threadIdx.x % 64 == 0) {
        lds[threadIdx.x / 64] = a;
        lds[16 + threadIdx.x / 64] = b;
    }
    __syncthreads();
    a = b = 0;
    for (int i = 0; i < waves; i++) {
        a += lds[i];
        b += lds[16 + i];
    }
}

struct Params { const void *w, *b; int wt, bt; };
struct Grads { Map dx; void *dw, *db; int dwt, dbt; };

template <class T>
__device__ __forceinline__ double first_value(const Map &x, const Shape &sh, int n, int g)
{
    return (double)(float)((const typename T::raw *)x.p)[n * x.sn + (int64_t)g * sh.cg * x.sc];
}

// The chunks' sums lie in the workspace as double2 [image][chunk][channel] of dz and dz (x - mean) (one chunk: an image's).
// dw and db of one channel from them, by one wave: in this order whatever order the workgroups that left them ended in.
__device__ __forceinline__ void channel_grads(const Shape &sh, int chunks, const double2 *part, const double *stats, int c, void *dw, int wt, void *db, int bt)
{
    double a = 0, b = 0;
    const unsigned rows = (unsigned)sh.N * chunks;
    for (unsigned i = threadIdx.x % 64; i < rows; i += 64) {
        const double2 v = part[(int64_t)i * sh.C + c];
        a += v.x;
        b = fma(v.y, stats[(unsigned)sh.N * sh.G + i / (unsigned)chunks * sh.G + c / sh.cg], b);
    }
    a = wave_sum(a);
    b = wave_sum(b);
    if (threadIdx.x % 64) return;
    if (db) store_param(db, bt, c, a);
    if (dw) store_param(dw, wt, c, b);
}
static __global__ __launch_bounds__(256) void channel_grads_kernel(Shape sh, int chunks, const double2 *part, const double *stats, void *dw, int wt, void *db, int bt)
{
    const int c = blockIdx.x * 4 + threadIdx.x / 64;
    if (c < sh.C) channel_grads(sh, chunks, part, stats, c, dw, wt, db, bt);
}

inline int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// ---- group_norm_small.hip ---------------------------------------------------------------------------------------
// the threads of its workgroups, one per image and group; 0: a call's groups are too large for it
int small_threads(bool last, const Shape &sh, int es, bool backward);
inline int64_t small_workspace(const Shape &sh) { return sh.N == 1 ? 0 : 2 * (int64_t)sh.N * sh.C; }       // fp64 values, backward
int small_forward(bool last, int dtype, const Shape &sh, const Map &x, const Map &y, const Params &p, double *stats, hipStream_t st);
int small_backward(bool last, int dtype, const Shape &sh, const Map &x, const Map &dy, const Params &p, const Grads &g, const double *stats, double *ws, hipStream_t st);

}  // namespace gn
}  // namespace genre
