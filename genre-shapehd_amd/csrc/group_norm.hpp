// group_norm.hpp -- what the two files of the group normalisation share (group_norm.hip: the mathematics, the entries and the
// kernels that walk a map in several passes; group_norm_small.hip: one workgroup per image and group).
#pragma once
#include "common.hpp"

namespace genre {
namespace gn {

enum { kActNone = 0, kActRelu = 1, kActLeaky = 2, kActSilu = 3 };

// ---- element types ----------------------------------------------------------------------------------------------
struct F32 { using raw = float; };
struct F16 { using raw = _Float16; };
struct BF16 { using raw = __bf16; };

// V values of type T; the pointer needs no more than T's own alignment (gfx950 loads and stores 16 bytes at any address)
template <class T, int V>
__device__ __forceinline__ void load(const typename T::raw *p, float (&v)[V])
{
    typename T::raw t[V];
    __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = (float)t[i];
}
template <class T, int V>
__device__ __forceinline__ void store(typename T::raw *p, const float (&v)[V])
{
    typename T::raw t[V];
#pragma unroll
    for (int i = 0; i < V; i++) t[i] = (typename T::raw)v[i];              // round to nearest even
    __builtin_memcpy(p, t, sizeof(t));
}

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
template <int ACT>
__device__ __forceinline__ float act_slope(double z, float slope)
{
    if (ACT == kActRelu) return z > 0 ? 1.f : 0.f;
    if (ACT == kActLeaky) return z > 0 ? 1.f : slope;
    if (ACT == kActSilu) {
        const float f = (float)z, s = sigmoid(f);
        return s * fmaf(f, 1.f - s, 1.f);
    }
    return 1.f;
}

// ---- what the kernels know of a call ----------------------------------------------------------------------------
struct Map { void *p; int64_t sn, sc, ss; };                               // element strides of image, channel, position

struct Shape {
    int N, C, G, cg, act;
    int64_t S;
    float slope;
    double m, eps;                                                         // M
};

__device__ __forceinline__ double wave_sum(double v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// sum over the workgroup, in every thread; `lds` has 16 doubles; ends with a barrier before lds can be used again
__device__ __forceinline__ double block_sum(double v, double *lds)
{
    v = wave_sum(v);
    const int waves = (blockDim.x + 63) / 64;
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    double s = 0;
    for (int i = 0; i < waves; i++) s += lds[i];
    return s;
}

// two of them at once; `lds` has 32
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


// dw and db from the sums of dz and dz h of each image and channel, whatever order the images' workgroups ended in
static __global__ __launch_bounds__(256) void param_grads_kernel(Shape sh, const double2 *chan, void *dw, int wt, void *db, int bt)
{
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= sh.C) return;
    double a = 0, b = 0;
    for (int n = 0; n < sh.N; n++) {
        const double2 v = chan[(int64_t)n * sh.C + c];
        a += v.x;
        b += v.y;
    }
    if (db) store_param(db, bt, c, a);
    if (dw) store_param(dw, wt, c, b);
}

inline int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// ---- group_norm_small.hip ---------------------------------------------------------------------------------------
// whether a call's groups are small enough for it (backward: half as large as forward)
bool small_fits(bool last, const Shape &sh, int es, bool backward);
inline int64_t small_workspace(const Shape &sh) { return sh.N == 1 ? 0 : 2 * (int64_t)sh.N * sh.C; }       // fp64 values, backward
int small_forward(bool last, int dtype, const Shape &sh, const Map &x, const Map &y, const Params &p, double *stats, hipStream_t st);
int small_backward(bool last, int dtype, const Shape &sh, const Map &x, const Map &dy, const Params &p, const Grads &g, const double *stats, double *ws, hipStream_t st);

}  // namespace gn
}  // namespace genre
