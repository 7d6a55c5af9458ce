// Kernels of the group normalisation with an activation and of the gate of a gated convolution, channels-last images.
//
//   group_norm        u = x                   y = act((u - mean) rstd w + b)
//   gated_group_norm  u = act(f) sigmoid(g)   y = (u - mean) rstd w + b
//   gated_activation  y = act(f) sigmoid(g)
// mean and rstd are those of a group's channels over all pixels of an image. Backward, with dz = dy act'(z):
//   db = sum dz, dw = sum dz uhat, du = rstd (w dz - c1 - uhat c2), c1 / c2 = the group's means of w dz and of w dz uhat;
//   df = du act'(f) sigmoid(g), dg = du act(f) sigmoid'(g).
//
// None of it is a contraction: every value is read, a handful of operations are done, and it is written. HBM bounds it, and
// for 16-bit gates the special-function unit comes close (an exponential and a reciprocal per sigmoid).
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "adop/adop_raster.h"
#include "norm_gate.h"

namespace adop {
namespace norm {

namespace cg = cooperative_groups;

// ---- vectors ------------------------------------------------------------------------------------------------------------
template <int BYTES> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = unsigned; };
template <> struct Word<2> { using type = unsigned short; };

template <typename T> __device__ __forceinline__ void unpack2(unsigned w, float& a, float& b);
template <> __device__ __forceinline__ void unpack2<__nv_bfloat16>(unsigned w, float& a, float& b)
{
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
}
template <> __device__ __forceinline__ void unpack2<__half>(unsigned w, float& a, float& b)
{
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    a = f.x; b = f.y;
}
template <typename T> __device__ __forceinline__ unsigned pack2(float a, float b);
template <> __device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float a, float b)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
}
template <> __device__ __forceinline__ unsigned pack2<__half>(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
}
template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC elements of a tensor as one load or store
template <typename T, int VEC> struct Vec
{
    static constexpr int kBytes = VEC * (int)sizeof(T);
    using W = typename Word<kBytes>::type;
    static __device__ __forceinline__ W load(const T* p) { return __ldg(reinterpret_cast<const W*>(p)); }
    static __device__ __forceinline__ void unpack(const W& w, float (&v)[VEC])
    {
        if constexpr (VEC == 1) v[0] = to_float<T>(*reinterpret_cast<const T*>(&w));
        else
        {
            const unsigned* u = reinterpret_cast<const unsigned*>(&w);
#pragma unroll
            for (int k = 0; k < kBytes / 4; ++k)
            {
                if constexpr (sizeof(T) == 4) v[k] = __uint_as_float(u[k]);
                else unpack2<T>(u[k], v[2 * k], v[2 * k + 1]);
            }
        }
    }
    // rounded once, to nearest even
    static __device__ __forceinline__ void store(T* p, const float (&v)[VEC])
    {
        if constexpr (VEC == 1) *p = from_float<T>(v[0]);
        else
        {
            W w;
            unsigned* u = reinterpret_cast<unsigned*>(&w);
#pragma unroll
            for (int k = 0; k < kBytes / 4; ++k)
            {
                if constexpr (sizeof(T) == 4) u[k] = __float_as_uint(v[k]);
                else u[k] = pack2<T>(v[2 * k], v[2 * k + 1]);
            }
            *reinterpret_cast<W*>(p) = w;
        }
    }
};

__device__ __forceinline__ float load_param(const void* p, int type, int i)
{
    if (type == ADOP_TYPE_F32) return static_cast<const float*>(p)[i];
    if (type == ADOP_TYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_param(void* p, int type, int i, float v)
{
    if (type == ADOP_TYPE_F32) static_cast<float*>(p)[i] = v;
    else if (type == ADOP_TYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// ---- activations --------------------------------------------------------------------------------------------------------
// sigmoid s and 1 - s, both to a few units of the last place: from e = exp(-|v|), which never overflows
__device__ __forceinline__ void sigmoid_pair(float v, float& s, float& ns)
{
    const float e = __expf(-fabsf(v));
    const float t = __fdividef(1.f, 1.f + e);
    const float et = e * t;
    s = v >= 0.f ? t : et;
    ns = v >= 0.f ? et : t;
}
__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }
// exp(v) - 1 for v <= 0. For 16-bit images: near zero, where exp(v) - 1 loses digits, its Taylor series (the first term left
// out is v^6 / 720, relative to v below 2^-24 for |v| < 1/8).
template <typename T> __device__ __forceinline__ float expm1_neg(float v, float e)
{
    if constexpr (sizeof(T) == 4) return expm1f(v);
    const float series = v * fmaf(v, fmaf(v, fmaf(v, fmaf(v, 1.f / 120.f, 1.f / 24.f), 1.f / 6.f), 0.5f), 1.f);
    return v > -0.125f ? series : e - 1.f;
}
// ACT = one of ADOP_ACTIVATION_* (rt ignored) or 4: rt says which, the same for all threads
template <typename T, int ACT> __device__ __forceinline__ float act_value(float v, int rt)
{
    const int a = ACT < 4 ? ACT : rt;
    if (a == ADOP_ACTIVATION_RELU) return v < 0.f ? 0.f : v;  // a NaN stays one
    if (a == ADOP_ACTIVATION_ELU) return v > 0.f ? v : expm1_neg<T>(v, __expf(v));
    if (a == ADOP_ACTIVATION_SILU) return v * sigmoid(v);
    return v;
}
// d act'(v)
template <typename T, int ACT> __device__ __forceinline__ float act_grad(float v, float d, int rt)
{
    const int a = ACT < 4 ? ACT : rt;
    if (a == ADOP_ACTIVATION_RELU) return v <= 0.f ? 0.f : d;
    if (a == ADOP_ACTIVATION_ELU) return v > 0.f ? d : d * __expf(v);
    if (a == ADOP_ACTIVATION_SILU)
    {
        float s, ns;
        sigmoid_pair(v, s, ns);
        return d * (s * fmaf(v, ns, 1.f));
    }
    return d;
}
// act(f) and act'(f) together
template <typename T, int ACT> __device__ __forceinline__ void act_both(float v, float& value, float& slope, int rt)
{
    const int a = ACT < 4 ? ACT : rt;
    value = v; slope = 1.f;
    if (a == ADOP_ACTIVATION_RELU) { value = v < 0.f ? 0.f : v; slope = v <= 0.f ? 0.f : 1.f; }
    if (a == ADOP_ACTIVATION_ELU)
    {
        const float e = __expf(v);
        value = v > 0.f ? v : expm1_neg<T>(v, e);
        slope = v > 0.f ? 1.f : e;
    }
    if (a == ADOP_ACTIVATION_SILU)
    {
        float s, ns;
        sigmoid_pair(v, s, ns);
        value = v * s;
        slope = s * fmaf(v, ns, 1.f);
    }
}

// ---- where a thread works -----------------------------------------------------------------------------------------------
struct Place
{
    int ph, r0;   // vector of the row, first row in the block's chunk
    bool active;
};
template <typename T> __device__ __forceinline__ const T* at(const NormImage& im, int b, int slice_c, int64_t row, int ph, int vec)
{
    return static_cast<const T*>(im.p) + (int64_t)b * im.image + slice_c + row * im.row + (int64_t)ph * vec;
}
template <typename T> __device__ __forceinline__ T* at_out(const NormImage& im, int b, int slice_c, int64_t row, int ph, int vec)
{
    return const_cast<T*>(at<T>(im, b, slice_c, row, ph, vec));
}
__device__ __forceinline__ void chunk_of(int rows, int part, int parts, int& begin, int& end)
{
    begin = (int)((int64_t)rows * part / parts);
    end = (int)((int64_t)rows * (part + 1) / parts);
}
// A kernel that was launched while the one before it may still run waits here for that one's results; every kernel that may
// be launched so waits before it ends, so that whoever waits for it also has all that came before.
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename T, int VEC, bool GATED> struct Loaded
{
    typename Vec<T, VEC>::W x, g;
};
// u of a vector
template <typename T, int VEC, bool GATED, int ACT>
__device__ __forceinline__ void value_of(const Loaded<T, VEC, GATED>& in, float (&u)[VEC], int rt)
{
    Vec<T, VEC>::unpack(in.x, u);
    if constexpr (GATED)
    {
        float g[VEC];
        Vec<T, VEC>::unpack(in.g, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) u[j] = act_value<T, ACT>(u[j], rt) * sigmoid(g[j]);
    }
}

// ---- sums of a block ----------------------------------------------------------------------------------------------------
// v[k][j]: two sums of each of a thread's channels. Runs of m channels are added up first. tot[(k * (VEC / m) + j / m) * P + ph]
// gets the sums over the rows of the block; buf is scratch of 2 (VEC / m) rows P + blockDim floats. Fixed order: the same
// bits on every run.
template <int VEC>
__device__ __forceinline__ void block_sums(float (&v)[2][VEC], int m, const NormArgs& a, const Place& at, float* tot, float* buf)
{
#pragma unroll
    for (int k = 0; k < 2; ++k)
    {
        if (VEC > 1 && m > 1)
#pragma unroll
            for (int j = 0; j + 1 < VEC; j += 2) v[k][j] += v[k][j + 1];
        if (VEC > 2 && m > 2)
#pragma unroll
            for (int j = 0; j + 2 < VEC; j += 4) v[k][j] += v[k][j + 2];
        if (VEC > 4 && m > 4) v[k][0] += v[k][VEC / 2];
    }
    const int sh = __ffs(m) - 1, per = VEC >> sh, P = a.P, t = threadIdx.x, T = blockDim.x;
    if (a.R == 1)
    {
        if (at.active)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if ((j & (m - 1)) == 0) tot[(k * per + (j >> sh)) * P + at.ph] = v[k][j];
        return;
    }
    int rows = a.R, row = at.r0;
    bool writer = at.active;
    if (32 % P == 0)
    {
        // the lanes of a warp that have the same channels
        for (int o = 16; o >= P; o >>= 1)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if ((j & (m - 1)) == 0) v[k][j] += __shfl_xor_sync(0xffffffffu, v[k][j], o);
        rows = T >> 5; row = t >> 5;
        writer = (t & 31) < P;
    }
    if (writer)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if ((j & (m - 1)) == 0) buf[((k * per + (j >> sh)) * rows + row) * P + at.ph] = v[k][j];
    __syncthreads();
    const int items = 2 * per * P;
    const int parts = min(rows, max(1, T / items));
    if (parts == 1)
    {
        for (int i = t; i < items; i += T)
        {
            const float* col = buf + (i / P) * rows * P + i % P;
            float s = 0.f;
#pragma unroll 4
            for (int r = 0; r < rows; ++r) s += col[r * P];
            tot[i] = s;
        }
        return;
    }
    float* tmp = buf + items * rows;
    if (t < items * parts)
    {
        const int i = t % items;
        const float* col = buf + (i / P) * rows * P + i % P;
        float s = 0.f;
        for (int r = t / items; r < rows; r += parts) s += col[r * P];
        tmp[t] = s;
    }
    __syncthreads();
    if (t < items)
    {
        float s = 0.f;
        for (int q = 0; q < parts; ++q) s += tmp[q * items + t];
        tot[t] = s;
    }
}

// The group's sums of u and u^2 in 64 bits from the slots' sums of u - pivot and its square over `rows` rows. The pivots are
// values of the data themselves, so the squares cancel by the number of values at most.
template <int VEC>
__device__ __forceinline__ void group_sums(const NormArgs& a, int rows, const float* tot, const float* pivot, double2* out)
{
    const int per = VEC / a.m, run = a.Cg / a.m, n = run * a.ppr, lanes = a.lanes, T = blockDim.x;
    const int want = (a.G * lanes + 31) & ~31;
    const double cnt = (double)rows * a.m;
    for (int idx = threadIdx.x; idx < want; idx += T)
    {
        const int g = idx / lanes, lane = idx & (lanes - 1);
        double s = 0.0, q = 0.0;
        if (g < a.G)
            for (int i = lane; i < n; i += lanes)
            {
                const int e = i / run * a.C + g * a.Cg + i % run * a.m;
                const int k = (e % VEC) / a.m * a.P + e / VEC;
                const double piv = (double)pivot[k], ds = (double)tot[k];
                s += fma(cnt, piv, ds);
                q += (double)tot[per * a.P + k] + piv * fma(cnt, piv, 2.0 * ds);
            }
        for (int o = lanes >> 1; o > 0; o >>= 1)
        {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            q += __shfl_xor_sync(0xffffffffu, q, o);
        }
        if (g < a.G && lane == 0) out[g] = make_double2(s, q);
    }
}

// Sums over the partial sums of an image's groups, by up to eight threads each; scratch of max(G, blockDim) double2. Ends with a barrier.
__device__ __forceinline__ void gather_groups(const double2* __restrict__ part, int parts, int G, double2* scratch, double2* out)
{
    const int T = blockDim.x, t = threadIdx.x;
    const int ways = max(1, min(8, min(parts, T / G)));
    for (int idx = t; idx < ways * G; idx += T)
    {
        const int w = idx / G, g = idx % G;
        double s = 0.0, q = 0.0;
#pragma unroll 4
        for (int k = w; k < parts; k += ways)
        {
            const double2 v = __ldcg(part + (size_t)k * G + g);
            s += v.x; q += v.y;
        }
        scratch[idx] = make_double2(s, q);
    }
    __syncthreads();
    for (int g = t; g < G; g += T)
    {
        double s = 0.0, q = 0.0;
        for (int w = 0; w < ways; ++w) { s += scratch[w * G + g].x; q += scratch[w * G + g].y; }
        out[g] = make_double2(s, q);
    }
    __syncthreads();
}
__device__ __forceinline__ float2 mean_rstd(double2 sums, double n, float eps)
{
    const double mean = sums.x / n;
    double var = sums.y / n - mean * mean;
    if (var < 0.0) var = 0.0;  // a NaN stays one
    return make_float2((float)mean, (float)(1.0 / sqrt(var + (double)eps)));
}

// ---- coefficients of a thread's channels ----------------------------------------------------------------------------------
template <int VEC> struct Forward
{
    float mean[VEC], scale[VEC], shift[VEC];  // z = (u - mean) scale + shift
    __device__ __forceinline__ void set(const NormArgs& a, int c0, int ph, const float2* stat)
    {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
        {
            const int c = (ph * VEC + j) % a.C;
            const float2 s = stat[c / a.Cg];
            mean[j] = s.x;
            scale[j] = a.weight ? s.y * load_param(a.weight, a.param_type, c0 + c) : s.y;
            shift[j] = a.bias ? load_param(a.bias, a.param_type, c0 + c) : 0.f;
        }
    }
};
template <typename T, int VEC, bool GATED, int ACT>
__device__ __forceinline__ void normalise(float (&u)[VEC], const Forward<VEC>& f, int rt)
{
#pragma unroll
    for (int j = 0; j < VEC; ++j)
    {
        const float z = fmaf(u[j] - f.mean[j], f.scale[j], f.shift[j]);
        u[j] = GATED ? z : act_value<T, ACT>(z, rt);
    }
}

// ---- forward, images larger than a cluster's shared memory ------------------------------------------------------------------
// Shared memory: double2 group[G] | float tot[2 P VEC / m] | pivot[P VEC / m] | block_sums' scratch
template <typename T, int VEC, bool GATED, int ACT>
__global__ void __launch_bounds__(kNormThreads, kNormBlocks) k_norm_stats(const __grid_constant__ NormArgs a)
{
    extern __shared__ double2 smem[];
    let_next_start();
    const int t = threadIdx.x, T_ = blockDim.x, b = a.image0 + blockIdx.y;
    int begin, end;
    chunk_of(a.rows, blockIdx.x, gridDim.x, begin, end);
    const int slots = a.P * (VEC / a.m);
    double2* group = smem;
    float* tot = reinterpret_cast<float*>(group + a.G);
    float* pivot = tot + 2 * slots;
    float* buf = pivot + slots;
    constexpr int U = GATED ? 2 : 4;
    using V = Vec<T, VEC>;
    using L = Loaded<T, VEC, GATED>;
    for (int ph0 = 0; ph0 < a.P; ph0 += T_)
    {
        Place pl;
        pl.ph = a.R == 1 ? ph0 + t : t % a.P;
        pl.r0 = a.R == 1 ? 0 : t / a.P;
        pl.active = pl.ph < a.P && pl.r0 < a.R;
        float v[2][VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[0][j] = v[1][j] = 0.f;
        if (pl.active)
        {
            const T* px = at<T>(a.x, b, 0, begin, pl.ph, VEC);
            const T* pg = GATED ? at<T>(a.gate, b, 0, begin, pl.ph, VEC) : nullptr;
            float piv[VEC];
            {
                L in;
                in.x = V::load(px);
                if (GATED) in.g = V::load(pg);
                value_of<T, VEC, GATED, ACT>(in, piv, a.act);
                // one pivot for the channels that are added up together
#pragma unroll
                for (int j = 1; j < VEC; ++j)
                    if (j & (a.m - 1)) piv[j] = piv[j - 1];
                if (pl.r0 == 0)
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        if ((j & (a.m - 1)) == 0) pivot[j / a.m * a.P + pl.ph] = piv[j];
            }
            for (int r = begin + pl.r0; r < end; r += U * a.R)
            {
                L in[U];
#pragma unroll
                for (int k = 0; k < U; ++k)
                    if (r + k * a.R < end)
                    {
                        const int64_t off = (int64_t)(r + k * a.R - begin);
                        in[k].x = V::load(px + off * a.x.row);
                        if (GATED) in[k].g = V::load(pg + off * a.gate.row);
                    }
#pragma unroll
                for (int k = 0; k < U; ++k)
                    if (r + k * a.R < end)
                    {
                        float u[VEC];
                        value_of<T, VEC, GATED, ACT>(in[k], u, a.act);
#pragma unroll
                        for (int j = 0; j < VEC; ++j)
                        {
                            const float d = u[j] - piv[j];
                            v[0][j] += d;
                            v[1][j] = fmaf(d, d, v[1][j]);
                        }
                    }
            }
        }
        block_sums<VEC>(v, a.m, a, pl, tot, buf);
    }
    __syncthreads();
    group_sums<VEC>(a, end - begin, tot, pivot, group);
    auto cluster = cg::this_cluster();
    cluster.sync();
    const int k = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    double2* out = a.group_part + ((size_t)b * a.clusters + blockIdx.x / k) * a.G;
    for (int g = rank * T_ + t; g < a.G; g += k * T_)
    {
        double s = 0.0, q = 0.0;
        for (int o = 0; o < k; ++o)
        {
            const double2 p = cluster.map_shared_rank(group, o)[g];
            s += p.x; q += p.y;
        }
        out[g] = make_double2(s, q);
    }
    cluster.sync();
    wait_previous();
}

// Shared memory: double2 total[G] | scratch[max(G, blockDim)] | float2 stat[G]
template <typename T, int VEC, bool GATED, int ACT>
__global__ void __launch_bounds__(kNormThreads, kNormBlocks) k_norm_apply(const __grid_constant__ NormArgs a)
{
    extern __shared__ double2 smem[];
    let_next_start();
    const int t = threadIdx.x, T_ = blockDim.x, b = a.image0 + blockIdx.y;
    int begin, end;
    chunk_of(a.rows, blockIdx.x, gridDim.x, begin, end);
    double2* total = smem;
    float2* stat = reinterpret_cast<float2*>(smem + a.G + max(a.G, T_));
    wait_previous();
    gather_groups(a.group_part + (size_t)b * a.clusters * a.G, a.clusters, a.G, smem + a.G, total);
    const double n = (double)a.rows * a.ppr * a.Cg;
    for (int g = t; g < a.G; g += T_)
    {
        const float2 s = mean_rstd(total[g], n, a.eps);
        stat[g] = s;
        if (a.mean && blockIdx.x == 0)
        {
            a.mean[(size_t)b * a.G + g] = s.x;
            a.rstd[(size_t)b * a.G + g] = s.y;
        }
    }
    __syncthreads();
    constexpr int U = GATED ? 2 : 4;
    using V = Vec<T, VEC>;
    using L = Loaded<T, VEC, GATED>;
    for (int ph0 = 0; ph0 < a.P; ph0 += T_)
    {
        const int ph = a.R == 1 ? ph0 + t : t % a.P, r0 = a.R == 1 ? 0 : t / a.P;
        if (ph >= a.P || r0 >= a.R) continue;
        Forward<VEC> f;
        f.set(a, 0, ph, stat);
        const T* px = at<T>(a.x, b, 0, 0, ph, VEC);
        const T* pg = GATED ? at<T>(a.gate, b, 0, 0, ph, VEC) : nullptr;
        T* py = at_out<T>(a.y, b, 0, 0, ph, VEC);
        // from the end: what the sums read last is what the L2 still has
        for (int r = end - 1 - r0; r >= begin; r -= U * a.R)
        {
            L in[U];
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (r - k * a.R >= begin)
                {
                    in[k].x = V::load(px + (int64_t)(r - k * a.R) * a.x.row);
                    if (GATED) in[k].g = V::load(pg + (int64_t)(r - k * a.R) * a.gate.row);
                }
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (r - k * a.R >= begin)
                {
                    float u[VEC];
                    value_of<T, VEC, GATED, ACT>(in[k], u, a.act);
                    normalise<T, VEC, GATED, ACT>(u, f, a.act);
                    V::store(py + (int64_t)(r - k * a.R) * a.y.row, u);
                }
        }
    }
}

// ---- backward, images larger than a cluster's shared memory -----------------------------------------------------------------
// uhat and dz of a vector: z = uhat w + b
template <int VEC> struct Saved
{
    float mean[VEC], rstd[VEC], w[VEC], bias[VEC];
    __device__ __forceinline__ void set(const NormArgs& a, int c0, int ph, const float* mean_, const float* rstd_)
    {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
        {
            const int c = (ph * VEC + j) % a.C, g = c / a.Cg;
            mean[j] = mean_[g];
            rstd[j] = rstd_[g];
            w[j] = a.weight ? load_param(a.weight, a.param_type, c0 + c) : 1.f;
            bias[j] = a.bias ? load_param(a.bias, a.param_type, c0 + c) : 0.f;
        }
    }
};
template <typename T, int VEC, bool GATED, int ACT>
__device__ __forceinline__ void add_grad_sums(const Loaded<T, VEC, GATED>& in, const typename Vec<T, VEC>::W& dy, const Saved<VEC>& s, float (&v)[2][VEC], int rt)
{
    float u[VEC], d[VEC];
    value_of<T, VEC, GATED, ACT>(in, u, rt);
    Vec<T, VEC>::unpack(dy, d);
#pragma unroll
    for (int j = 0; j < VEC; ++j)
    {
        const float uhat = (u[j] - s.mean[j]) * s.rstd[j];
        const float dz = GATED ? d[j] : act_grad<T, ACT>(fmaf(uhat, s.w[j], s.bias[j]), d[j], rt);
        v[0][j] += dz;
        v[1][j] = fmaf(dz, uhat, v[1][j]);
    }
}
// du = dz scale + (u - mean) slope + offset, with scale = rstd w, slope = -rstd^2 c2, offset = -rstd c1
template <int VEC> struct Backward
{
    float mean[VEC], scale[VEC], bias[VEC], slope[VEC], offset[VEC];
    __device__ __forceinline__ void set(const NormArgs& a, int c0, int ph, const float* mean_, const float* rstd_, const float2* c12)
    {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
        {
            const int c = (ph * VEC + j) % a.C, g = c / a.Cg;
            const float r = rstd_[g];
            mean[j] = mean_[g];
            scale[j] = a.weight ? r * load_param(a.weight, a.param_type, c0 + c) : r;
            bias[j] = a.bias ? load_param(a.bias, a.param_type, c0 + c) : 0.f;
            slope[j] = -r * r * c12[g].y;
            offset[j] = -r * c12[g].x;
        }
    }
};
template <typename T, int VEC, bool GATED, int ACT>
__device__ __forceinline__ void input_gradient(const Loaded<T, VEC, GATED>& in, const typename Vec<T, VEC>::W& dy, const Backward<VEC>& k, float (&dx)[VEC],
                                               float (&dg)[VEC], int rt)
{
    float d[VEC], u[VEC];
    Vec<T, VEC>::unpack(in.x, u);
    Vec<T, VEC>::unpack(dy, d);
    if constexpr (!GATED)
    {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
        {
            const float x = u[j] - k.mean[j];
            const float dz = act_grad<T, ACT>(fmaf(x, k.scale[j], k.bias[j]), d[j], rt);
            dx[j] = fmaf(dz, k.scale[j], fmaf(x, k.slope[j], k.offset[j]));
        }
    }
    else
    {
        float g[VEC];
        Vec<T, VEC>::unpack(in.g, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
        {
            float value, slope, s, ns;
            act_both<T, ACT>(u[j], value, slope, rt);
            sigmoid_pair(g[j], s, ns);
            const float du = fmaf(d[j], k.scale[j], fmaf(value * s - k.mean[j], k.slope[j], k.offset[j]));
            dx[j] = du * slope * s;
            dg[j] = du * value * s * ns;
        }
    }
}
// channel sums [2][C] from the slots' (a row may hold several pixels), then the groups' sums of w dz and w dz uhat
template <int VEC>
__device__ __forceinline__ void channel_and_group_sums(const NormArgs& a, int c0, const float* tot, float* chan, double2* group)
{
    const int T = blockDim.x, t = threadIdx.x;
    for (int i = t; i < 2 * a.C; i += T)
    {
        const int k = i / a.C, c = i % a.C;
        float s = 0.f;
        for (int q = 0; q < a.ppr; ++q)
        {
            const int e = q * a.C + c;
            s += tot[(k * VEC + e % VEC) * a.P + e / VEC];
        }
        chan[i] = s;
    }
    __syncthreads();
    const int want = (a.G * a.lanes + 31) & ~31;
    for (int idx = t; idx < want; idx += T)
    {
        const int g = idx / a.lanes, lane = idx & (a.lanes - 1);
        double s = 0.0, q = 0.0;
        if (g < a.G)
            for (int i = lane; i < a.Cg; i += a.lanes)
            {
                const int c = g * a.Cg + i;
                const double w = a.weight ? (double)load_param(a.weight, a.param_type, c0 + c) : 1.0;
                s = fma(w, (double)chan[c], s);
                q = fma(w, (double)chan[a.C + c], q);
            }
        for (int o = a.lanes >> 1; o > 0; o >>= 1)
        {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            q += __shfl_xor_sync(0xffffffffu, q, o);
        }
        if (g < a.G && lane == 0) group[g] = make_double2(s, q);
    }
}

// Shared memory: double2 group[G] | float chan[2 C] | tot[2 P VEC] | block_sums' scratch
template <typename T, int VEC, bool GATED, int ACT>
__global__ void __launch_bounds__(kNormGradThreads, kNormGradBlocks) k_norm_grad_sums(const __grid_constant__ NormArgs a)
{
    extern __shared__ double2 smem[];
    let_next_start();
    const int t = threadIdx.x, T_ = blockDim.x, b = a.image0 + blockIdx.y;
    int begin, end;
    chunk_of(a.rows, blockIdx.x, gridDim.x, begin, end);
    double2* group = smem;
    float* chan = reinterpret_cast<float*>(group + a.G);
    float* tot = chan + 2 * a.C;
    float* buf = tot + 2 * a.P * VEC;
    constexpr int U = 2;
    using V = Vec<T, VEC>;
    using L = Loaded<T, VEC, GATED>;
    for (int ph0 = 0; ph0 < a.P; ph0 += T_)
    {
        Place pl;
        pl.ph = a.R == 1 ? ph0 + t : t % a.P;
        pl.r0 = a.R == 1 ? 0 : t / a.P;
        pl.active = pl.ph < a.P && pl.r0 < a.R;
        float v[2][VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[0][j] = v[1][j] = 0.f;
        if (pl.active)
        {
            Saved<VEC> s;
            s.set(a, 0, pl.ph, a.mean + (size_t)b * a.G, a.rstd + (size_t)b * a.G);
            const T* px = at<T>(a.x, b, 0, 0, pl.ph, VEC);
            const T* pg = GATED ? at<T>(a.gate, b, 0, 0, pl.ph, VEC) : nullptr;
            const T* pd = at<T>(a.dy, b, 0, 0, pl.ph, VEC);
            for (int r = begin + pl.r0; r < end; r += U * a.R)
            {
                L in[U];
                typename V::W dy[U];
#pragma unroll
                for (int k = 0; k < U; ++k)
                    if (r + k * a.R < end)
                    {
                        const int64_t row = r + k * a.R;
                        in[k].x = V::load(px + row * a.x.row);
                        if (GATED) in[k].g = V::load(pg + row * a.gate.row);
                        dy[k] = V::load(pd + row * a.dy.row);
                    }
#pragma unroll
                for (int k = 0; k < U; ++k)
                    if (r + k * a.R < end) add_grad_sums<T, VEC, GATED, ACT>(in[k], dy[k], s, v, a.act);
            }
        }
        block_sums<VEC>(v, 1, a, pl, tot, buf);
    }
    __syncthreads();
    channel_and_group_sums<VEC>(a, 0, tot, chan, group);
    auto cluster = cg::this_cluster();
    cluster.sync();
    const int k = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const size_t part = (size_t)b * a.clusters + blockIdx.x / k;
    for (int g = rank * T_ + t; g < a.G; g += k * T_)
    {
        double s = 0.0, q = 0.0;
        for (int o = 0; o < k; ++o)
        {
            const double2 p = cluster.map_shared_rank(group, o)[g];
            s += p.x; q += p.y;
        }
        a.group_part[part * a.G + g] = make_double2(s, q);
    }
    if (a.channel_part)
        for (int c = rank * T_ + t; c < a.C; c += k * T_)
        {
            float s = 0.f, q = 0.f;
            for (int o = 0; o < k; ++o)
            {
                const float* p = cluster.map_shared_rank(chan, o);
                s += p[c]; q += p[a.C + c];
            }
            a.channel_part[part * a.C + c] = make_float2(s, q);
        }
    cluster.sync();
    wait_previous();
}

// db and dw of up to blockDim channels from `parts` partial sums each, in 64 bits and in a fixed order. Scratch: 2 blockDim double.
__device__ __forceinline__ void param_gradients(const NormArgs& a, int channels, int c0, int nc, double* scratch)
{
    const int T = blockDim.x, t = threadIdx.x, ways = T / nc;
    const int c = t % nc, w = t / nc;
    double s = 0.0, q = 0.0;
    if (w < ways)
#pragma unroll 8
        for (int k = w; k < a.param_parts; k += ways)
        {
            const float2 v = __ldcg(a.channel_part + (size_t)k * channels + c0 + c);
            s += v.x; q += v.y;
        }
    scratch[2 * t] = s;
    scratch[2 * t + 1] = q;
    __syncthreads();
    if (t < nc)
    {
        s = q = 0.0;
        for (int k = 0; k < ways; ++k) { s += scratch[2 * (k * nc + t)]; q += scratch[2 * (k * nc + t) + 1]; }
        if (a.dbias) store_param(a.dbias, a.param_type, c0 + t, (float)s);
        if (a.dweight) store_param(a.dweight, a.param_type, c0 + t, (float)q);
    }
}
constexpr int kParamChannels = 32;  // channels that one block adds up

// Shared memory: as k_norm_apply; the parameter blocks 2 blockDim double
template <typename T, int VEC, bool GATED, int ACT>
__global__ void __launch_bounds__(kNormGradThreads, kNormGradBlocks) k_norm_grad_apply(const __grid_constant__ NormArgs a)
{
    extern __shared__ double2 smem[];
    let_next_start();
    const int t = threadIdx.x, T_ = blockDim.x, b = a.image0 + blockIdx.y;
    wait_previous();
    if ((int)blockIdx.x < a.param_blocks)
    {
        if (blockIdx.y == 0)
        {
            const int c0 = blockIdx.x * kParamChannels;
            param_gradients(a, a.C, c0, min(kParamChannels, a.C - c0), reinterpret_cast<double*>(smem));
        }
        return;
    }
    int begin, end;
    chunk_of(a.rows, blockIdx.x - a.param_blocks, gridDim.x - a.param_blocks, begin, end);
    float2* c12 = reinterpret_cast<float2*>(smem + a.G + max(a.G, T_));
    gather_groups(a.group_part + (size_t)b * a.clusters * a.G, a.clusters, a.G, smem + a.G, smem);
    const double n = (double)a.rows * a.ppr * a.Cg;
    for (int g = t; g < a.G; g += T_) c12[g] = make_float2((float)(smem[g].x / n), (float)(smem[g].y / n));
    __syncthreads();
    constexpr int U = 2;
    using V = Vec<T, VEC>;
    using L = Loaded<T, VEC, GATED>;
    for (int ph0 = 0; ph0 < a.P; ph0 += T_)
    {
        const int ph = a.R == 1 ? ph0 + t : t % a.P, r0 = a.R == 1 ? 0 : t / a.P;
        if (ph >= a.P || r0 >= a.R) continue;
        Backward<VEC> c;
        c.set(a, 0, ph, a.mean + (size_t)b * a.G, a.rstd + (size_t)b * a.G, c12);
        const T* px = at<T>(a.x, b, 0, 0, ph, VEC);
        const T* pg = GATED ? at<T>(a.gate, b, 0, 0, ph, VEC) : nullptr;
        const T* pd = at<T>(a.dy, b, 0, 0, ph, VEC);
        T* pdx = at_out<T>(a.dx, b, 0, 0, ph, VEC);
        T* pdg = GATED ? at_out<T>(a.dgate, b, 0, 0, ph, VEC) : nullptr;
        for (int r = end - 1 - r0; r >= begin; r -= U * a.R)
        {
            L in[U];
            typename V::W dy[U];
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (r - k * a.R >= begin)
                {
                    const int64_t row = r - k * a.R;
                    in[k].x = V::load(px + row * a.x.row);
                    if (GATED) in[k].g = V::load(pg + row * a.gate.row);
                    dy[k] = V::load(pd + row * a.dy.row);
                }
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (r - k * a.R >= begin)
                {
                    const int64_t row = r - k * a.R;
                    float dx[VEC], dg[VEC];
                    input_gradient<T, VEC, GATED, ACT>(in[k], dy[k], c, dx, dg, a.act);
                    V::store(pdx + row * a.dx.row, dx);
                    if (GATED) V::store(pdg + row * a.dgate.row, dg);
                }
        }
    }
}

// ---- the gate alone -----------------------------------------------------------------------------------------------------
template <typename T, int VEC, bool GATED, int ACT>
__global__ void __launch_bounds__(kNormThreads, kNormBlocks) k_gate(const __grid_constant__ NormArgs a)
{
    const int t = threadIdx.x, T_ = blockDim.x, b = blockIdx.y;
    int begin, end;
    chunk_of(a.rows, blockIdx.x, gridDim.x, begin, end);
    constexpr int U = 2;
    using V = Vec<T, VEC>;
    using L = Loaded<T, VEC, true>;
    for (int ph0 = 0; ph0 < a.P; ph0 += T_)
    {
        const int ph = a.R == 1 ? ph0 + t : t % a.P, r0 = a.R == 1 ? 0 : t / a.P;
        if (ph >= a.P || r0 >= a.R) continue;
        const T* px = at<T>(a.x, b, 0, 0, ph, VEC);
        const T* pg = at<T>(a.gate, b, 0, 0, ph, VEC);
        T* py = at_out<T>(a.y, b, 0, 0, ph, VEC);
        for (int r = begin + r0; r < end; r += U * a.R)
        {
            L in[U];
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (r + k * a.R < end)
                {
                    const int64_t row = r + k * a.R;
                    in[k].x = V::load(px + row * a.x.row);
                    in[k].g = V::load(pg + row * a.gate.row);
                }
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (r + k * a.R < end)
                {
                    float u[VEC];
                    value_of<T, VEC, true, ACT>(in[k], u, a.act);
                    V::store(py + (int64_t)(r + k * a.R) * a.y.row, u);
                }
        }
    }
}
template <typename T, int VEC, bool GATED, int ACT>
__global__ void __launch_bounds__(kNormGradThreads, kNormGradBlocks) k_gate_grad(const __grid_constant__ NormArgs a)
{
    const int t = threadIdx.x, T_ = blockDim.x, b = blockIdx.y;
    int begin, end;
    chunk_of(a.rows, blockIdx.x, gridDim.x, begin, end);
    constexpr int U = 2;
    using V = Vec<T, VEC>;
    for (int ph0 = 0; ph0 < a.P; ph0 += T_)
    {
        const int ph = a.R == 1 ? ph0 + t : t % a.P, r0 = a.R == 1 ? 0 : t / a.P;
        if (ph >= a.P || r0 >= a.R) continue;
        const T* px = at<T>(a.x, b, 0, 0, ph, VEC);
        const T* pg = at<T>(a.gate, b, 0, 0, ph, VEC);
        const T* pd = at<T>(a.dy, b, 0, 0, ph, VEC);
        T* pdx = at_out<T>(a.dx, b, 0, 0, ph, VEC);
        T* pdg = at_out<T>(a.dgate, b, 0, 0, ph, VEC);
        for (int r = begin + r0; r < end; r += U * a.R)
        {
            typename V::W in[U][3];
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (r + k * a.R < end)
                {
                    const int64_t row = r + k * a.R;
                    in[k][0] = V::load(px + row * a.x.row);
                    in[k][1] = V::load(pg + row * a.gate.row);
                    in[k][2] = V::load(pd + row * a.dy.row);
                }
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (r + k * a.R < end)
                {
                    const int64_t row = r + k * a.R;
                    float f[VEC], g[VEC], d[VEC];
                    V::unpack(in[k][0], f);
                    V::unpack(in[k][1], g);
                    V::unpack(in[k][2], d);
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                    {
                        float value, slope, s, ns;
                        act_both<T, ACT>(f[j], value, slope, a.act);
                        sigmoid_pair(g[j], s, ns);
                        const float ds = d[j] * s;
                        f[j] = ds * slope;
                        g[j] = ds * value * ns;
                    }
                    V::store(pdx + row * a.dx.row, f);
                    V::store(pdg + row * a.dgate.row, g);
                }
        }
    }
}

// ---- which kernel -------------------------------------------------------------------------------------------------------
template <typename T, int VEC, bool GATED, int ACT> const void* pick(int which)
{
    switch (which)
    {
        case kNormStats: return (const void*)k_norm_stats<T, VEC, GATED, GATED ? ACT : 0>;
        case kNormApply: return (const void*)k_norm_apply<T, VEC, GATED, ACT>;
        case kNormGradSums: return (const void*)k_norm_grad_sums<T, VEC, GATED, ACT>;
        case kNormGradApply: return (const void*)k_norm_grad_apply<T, VEC, GATED, ACT>;
        case kGate: return (const void*)k_gate<T, VEC, true, ACT>;
        case kGateGrad: return (const void*)k_gate_grad<T, VEC, true, ACT>;
    }
    return nullptr;
}
template <typename T, int VEC, bool GATED> const void* pick_act(int which, int act)
{
    if constexpr (VEC * sizeof(T) == 16)
        switch (act)
        {
            case ADOP_ACTIVATION_NONE: return pick<T, VEC, GATED, ADOP_ACTIVATION_NONE>(which);
            case ADOP_ACTIVATION_RELU: return pick<T, VEC, GATED, ADOP_ACTIVATION_RELU>(which);
            case ADOP_ACTIVATION_ELU: return pick<T, VEC, GATED, ADOP_ACTIVATION_ELU>(which);
            default: return pick<T, VEC, GATED, ADOP_ACTIVATION_SILU>(which);
        }
    else
        return pick<T, VEC, GATED, 4>(which);
}
template <typename T> const void* norm_kernel(int which, int vec, bool gated, int act)
{
    constexpr int V16 = 16 / sizeof(T), V8 = 8 / sizeof(T);
    if (vec == kVec16) return gated ? pick_act<T, V16, true>(which, act) : pick_act<T, V16, false>(which, act);
    if (vec == kVec8) return gated ? pick_act<T, V8, true>(which, act) : pick_act<T, V8, false>(which, act);
    return gated ? pick_act<T, 1, true>(which, act) : pick_act<T, 1, false>(which, act);
}

}  // namespace norm
}  // namespace adop
