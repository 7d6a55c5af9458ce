// Kernels of the group normalisation with an activation and of the gate of a gated convolution, channels-last images.
//
//   group_norm        u = x                   y = act((u - mean) rstd w + b)
//   gated_group_norm  u = act(f) sigmoid(g)   y = (u - mean) rstd w + b
//   gated_activation  y = act(f) sigmoid(g)
// mean and rstd are those of a group's channels over all pixels of an image. Backward, with dz = dy act'(z):
//   db = sum dz, dw = sum dz uhat, du = rstd (w dz - c1 - uhat c2), c1 / c2 = the group's means of w dz and of w dz uhat;
//   df = du act'(f) sigmoid(g), dg = du act(f) sigmoid'(g).
//
// None of it is a contraction: every value is read, a handful of operations are done, and it is written. HBM bounds it, and for 16-bit
// gates the arithmetic comes close: an exponential and a reciprocal per sigmoid, 8 cycles of a scheduler's special-function unit each, and
// some 20 instructions a value, where 22 cycles are what 4 bytes take from HBM. Counters of the gated sums behind an ELU: 3.0 such operations a
// value, that unit busy for 80 % of the time, 4.5 TB/s.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "adop/adop_raster.h"
#include "norm_gate.h"

namespace adop {
namespace norm {

// ---- vectors ------------------------------------------------------------------------------------------------------------
// VEC values of a vector in 32 bits, in pairs: sm_100 adds, multiplies and fuses two at a time (one instruction a pair). With one
// element the second of its pair is computed along and dropped.
template <int VEC> struct alignas(VEC > 2 ? 16 : 8) Lanes
{
    static constexpr int N = (VEC + 1) / 2;
    float2 p[N];
    __device__ __forceinline__ float get(int j) const { return j & 1 ? p[j / 2].y : p[j / 2].x; }
    __device__ __forceinline__ void set(int j, float v)
    {
        if (j & 1) p[j / 2].y = v;
        else p[j / 2].x = v;
    }
    __device__ __forceinline__ void fill(float v)
    {
#pragma unroll
        for (int k = 0; k < N; ++k) p[k] = make_float2(v, v);
    }
};
__device__ __forceinline__ float2 pair(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 add(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

template <int BYTES> struct Word;
template <> struct Word<16> { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = unsigned; };
template <> struct Word<2> { using type = unsigned short; };

template <typename T> __device__ __forceinline__ float2 unpack2(unsigned w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(unsigned w)
{
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(unsigned w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <typename T> __device__ __forceinline__ unsigned pack2(float2 v);
template <> __device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float2 v)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
    return *reinterpret_cast<const unsigned*>(&h);
}
template <> __device__ __forceinline__ unsigned pack2<__half>(float2 v)
{
    const __half2 h = __floats2half2_rn(v.x, v.y);
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
    static __device__ __forceinline__ Lanes<VEC> unpack(const W& w)
    {
        Lanes<VEC> v;
        if constexpr (VEC == 1) v.p[0] = pair(to_float<T>(*reinterpret_cast<const T*>(&w)));
        else
        {
            const unsigned* u = reinterpret_cast<const unsigned*>(&w);
#pragma unroll
            for (int k = 0; k < VEC / 2; ++k)
            {
                if constexpr (sizeof(T) == 4) v.p[k] = make_float2(__uint_as_float(u[2 * k]), __uint_as_float(u[2 * k + 1]));
                else v.p[k] = unpack2<T>(u[k]);
            }
        }
        return v;
    }
    // rounded once, to nearest even
    static __device__ __forceinline__ void store(T* p, const Lanes<VEC>& v)
    {
        if constexpr (VEC == 1) *p = from_float<T>(v.p[0].x);
        else
        {
            W w;
            unsigned* u = reinterpret_cast<unsigned*>(&w);
#pragma unroll
            for (int k = 0; k < VEC / 2; ++k)
            {
                if constexpr (sizeof(T) == 4) { u[2 * k] = __float_as_uint(v.p[k].x); u[2 * k + 1] = __float_as_uint(v.p[k].y); }
                else u[k] = pack2<T>(v.p[k]);
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
// f(i, load(i)) for i = first, first + step, ... below end: N loads are under way before the first is used. An unrolled loop takes its
// remainder one load after the other, and the two or three partial sums of a thread are all remainder: an image of 320 x 180 x 32 in bfloat16
// takes 7.9 us forward for 8.8 and 10.4 backward for 11.6.
template <int N, class Load, class F> __device__ __forceinline__ void loads_ahead(int first, int step, int end, Load load, F f)
{
    for (int i = first; i < end; i += N * step)
    {
        decltype(load(0)) v[N];
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (i + k * step < end) v[k] = load(i + k * step);
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (i + k * step < end) f(i + k * step, v[k]);
    }
}
// weight and bias of the channels from c0 on as to[C] and to[C] behind it, 1 and 0 where there are none; a barrier follows
__device__ __forceinline__ void stage_params(const NormArgs& a, int c0, float* to)
{
    for (int c = threadIdx.x; c < a.C; c += blockDim.x)
    {
        to[c] = a.weight ? load_param(a.weight, a.param_type, c0 + c) : 1.f;
        to[a.C + c] = a.bias ? load_param(a.bias, a.param_type, c0 + c) : 0.f;
    }
}
__device__ __forceinline__ void store_param(void* p, int type, int i, float v)
{
    if (type == ADOP_TYPE_F32) static_cast<float*>(p)[i] = v;
    else if (type == ADOP_TYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// ---- activations --------------------------------------------------------------------------------------------------------
constexpr float kLog2e = 1.4426950408889634f;
// powers of two and reciprocals of the special-function unit (2 and 1 ulp; results below the smallest normal number become 0)
__device__ __forceinline__ float ex2(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float rcp(float v)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float2 exp2v(float2 v) { return make_float2(ex2(v.x), ex2(v.y)); }
__device__ __forceinline__ float2 rcp2(float2 v) { return make_float2(rcp(v.x), rcp(v.y)); }
__device__ __forceinline__ float2 sigmoid(float2 v) { return rcp2(add(exp2v(mul(v, pair(-kLog2e))), pair(1.f))); }
// sigmoid s and 1 - s = exp(-v) s. The exponential's argument v log2(e) is rounded to 32 bits, which its result feels as 0.62 |v| ulp: s is within
// (0.62 |v| + 4) 2^-23 of itself, 1 - s within (0.62 |v| + 7) 2^-23 (54 and 57 units at v = -80, where s is 2^-115; a
// 16-bit result is rounded by up to 2^-11 of itself). Sigmoids below 2^-126, v < -87.3, are 0. The exponential stays finite; where it would not, s is 0.
__device__ __forceinline__ float min_or_nan(float v, float most)
{
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(most));
    return r;
}
__device__ __forceinline__ void sigmoid_pair(float2 v, float2& s, float2& ns)
{
    const float2 m = mul(v, pair(-kLog2e));
    const float2 e = make_float2(ex2(min_or_nan(m.x, 127.f)), ex2(min_or_nan(m.y, 127.f)));
    s = rcp2(add(e, pair(1.f)));
    ns = mul(e, s);
}
// v > 0 ? v : exp(v) - 1, with e = exp(v). Near zero, where e - 1 loses digits, the Taylor series: for 16-bit images four terms above
// -1/16 (the fifth is below 2^-22 of the sum there), for 32 bits eight above -1/2 (the ninth is below 2^-26).
template <typename T> __device__ __forceinline__ float2 elu_value(float2 v, float2 e)
{
    constexpr bool kWide = sizeof(T) == 4;
    constexpr float kFrom = kWide ? -0.5f : -0.0625f;
    float2 q = pair(1.f / 24.f);
    if (kWide)
    {
        q = fma2(v, pair(1.f / 40320.f), pair(1.f / 5040.f));
        q = fma2(v, q, pair(1.f / 720.f));
        q = fma2(v, q, pair(1.f / 120.f));
        q = fma2(v, q, pair(1.f / 24.f));
    }
    q = fma2(v, q, pair(1.f / 6.f));
    q = fma2(v, q, pair(0.5f));
    q = fma2(v, q, pair(1.f));
    q = mul(v, q);
    const float2 m = add(e, pair(-1.f));
    return make_float2(v.x > 0.f ? v.x : (v.x > kFrom ? q.x : m.x), v.y > 0.f ? v.y : (v.y > kFrom ? q.y : m.y));
}
// ACT = one of ADOP_ACTIVATION_* (rt ignored) or 4: rt says which, the same for all threads
template <typename T, int ACT> __device__ __forceinline__ float2 act_value(float2 v, int rt)
{
    const int a = ACT < 4 ? ACT : rt;
    if (a == ADOP_ACTIVATION_RELU) return make_float2(v.x < 0.f ? 0.f : v.x, v.y < 0.f ? 0.f : v.y);  // a NaN stays one
    if (a == ADOP_ACTIVATION_ELU) return elu_value<T>(v, exp2v(mul(v, pair(kLog2e))));
    if (a == ADOP_ACTIVATION_SILU) return mul(v, sigmoid(v));
    return v;
}
// d act'(v)
template <typename T, int ACT> __device__ __forceinline__ float2 act_grad(float2 v, float2 d, int rt)
{
    const int a = ACT < 4 ? ACT : rt;
    if (a == ADOP_ACTIVATION_RELU) return make_float2(v.x <= 0.f ? 0.f : d.x, v.y <= 0.f ? 0.f : d.y);
    if (a == ADOP_ACTIVATION_ELU)
    {
        const float2 e = exp2v(mul(v, pair(kLog2e)));
        return make_float2(v.x > 0.f ? d.x : d.x * e.x, v.y > 0.f ? d.y : d.y * e.y);
    }
    if (a == ADOP_ACTIVATION_SILU)
    {
        float2 s, ns;
        sigmoid_pair(v, s, ns);
        return mul(d, mul(s, fma2(v, ns, pair(1.f))));
    }
    return d;
}
// act(f) and act'(f) together
template <typename T, int ACT> __device__ __forceinline__ void act_both(float2 v, float2& value, float2& slope, int rt)
{
    const int a = ACT < 4 ? ACT : rt;
    value = v; slope = pair(1.f);
    if (a == ADOP_ACTIVATION_RELU)
    {
        value = make_float2(v.x < 0.f ? 0.f : v.x, v.y < 0.f ? 0.f : v.y);
        slope = make_float2(v.x <= 0.f ? 0.f : 1.f, v.y <= 0.f ? 0.f : 1.f);
    }
    if (a == ADOP_ACTIVATION_ELU)
    {
        const float2 e = exp2v(mul(v, pair(kLog2e)));
        value = elu_value<T>(v, e);
        slope = make_float2(v.x > 0.f ? 1.f : e.x, v.y > 0.f ? 1.f : e.y);
    }
    if (a == ADOP_ACTIVATION_SILU)
    {
        float2 s, ns;
        sigmoid_pair(v, s, ns);
        value = mul(v, s);
        slope = mul(s, fma2(v, ns, pair(1.f)));
    }
}

// i / d for i, d up to 4096 (quotient off an integer by 1 / 2d at least, the product by 2^-22 of it), inv = 1 / d
__device__ __forceinline__ int quotient(int i, float inv) { return (int)(((float)i + 0.5f) * inv); }

// ---- where a thread works -----------------------------------------------------------------------------------------------
// A thread's vector of the row and its first row of the block's chunk; the rows after it are R apart.
struct Place
{
    int ph, r0;
    bool active;
    __device__ __forceinline__ Place(const NormArgs& a, int ph0)
    {
        const int t = threadIdx.x;
        if (a.R == 1) { ph = ph0 + t; r0 = 0; }
        else { r0 = quotient(t, a.inv_P); ph = t - r0 * a.P; }
        active = ph < a.P && r0 < a.R;
    }
    // how many rows of [begin, end) are the thread's
    __device__ __forceinline__ int count(const NormArgs& a, int begin, int end) const
    {
        const int left = end - begin - r0;
        return left <= 0 ? 0 : (left - 1) / a.R + 1;
    }
};
// The vectors of a tensor that a thread comes by: `step` elements apart, forwards from the chunk's first row or backwards from its last.
template <typename T> struct Walk
{
    T* p;
    int64_t step;
    __device__ __forceinline__ Walk(const NormImage& im, int b, int c0, const Place& pl, int R, int vec, int begin, int end, bool backwards)
    {
        const int64_t row = backwards ? (int64_t)end - 1 - pl.r0 : (int64_t)begin + pl.r0;
        p = static_cast<T*>(const_cast<void*>(im.p)) + (int64_t)b * im.image + c0 + row * im.row + (int64_t)pl.ph * vec;
        step = (backwards ? -im.row : im.row) * R;
    }
    __device__ __forceinline__ T* at(int k) const { return p + k * step; }
    __device__ __forceinline__ void on(int k) { p += k * step; }
};
// rows [begin, end) of a block's part of the image
__device__ __forceinline__ void chunk_of(const NormArgs& a, int part, int& begin, int& end)
{
    begin = part * a.own.rows + min(part, a.own.more);
    end = begin + a.own.rows + (part < a.own.more ? 1 : 0);
}
// f(j, c, g) for the channels c and groups g of a thread's vector (a row of several pixels goes through the channels again)
template <int VEC, class F> __device__ __forceinline__ void for_channels(const NormArgs& a, int ph, F f)
{
    int c = ph * VEC;
    while (c >= a.C) c -= a.C;
    int g = quotient(c, a.inv_Cg), r = c - g * a.Cg;
#pragma unroll
    for (int j = 0; j < VEC; ++j)
    {
        f(j, c, g);
        ++c;
        if (++r == a.Cg) { r = 0; ++g; }
        if (c == a.C) c = g = 0;
    }
}
// A kernel that was launched while the one before it may still run waits here for that one's results; every kernel that may
// be launched so waits before it ends, so that whoever waits for it also has all that came before.
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// L1: through the first-level cache. Features and gates that lie side by side share sectors, and where a pixel has few of them the
// second copy finds its half there (sums over 8 channels of 16 bits 48 -> 36 us for 134 MB); everything else goes past it, as two
// tensors eight vectors deep do not fit beside the slots (backward sums 114 -> 129 us for 537 MB with it).
template <int BYTES, bool L1> __device__ __forceinline__ void copy_async(void* to, const void* from)
{
    const unsigned s = (unsigned)__cvta_generic_to_shared(to);
    if constexpr (BYTES == 16 && !L1) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(s), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

template <typename T, int VEC> struct Input
{
    typename Vec<T, VEC>::W x, g, dy;
};
// The vectors of x, of the gate and of dy that a thread comes by in a chunk. Copies into slots of its own in shared memory run D vectors
// ahead, the first D of them from start() on, which may stand far in front of run(): what a block does before its loop, and its waits,
// cost no bandwidth then. 64 to 98 KB are under way on an SM; registers hold two vectors. Vectors of one element have no such copies:
// there U loads are under way before the first is used.
template <typename T, int VEC, bool GATED, bool GRAD> struct Stream
{
    static constexpr int kTensors = 1 + (GATED ? 1 : 0) + (GRAD ? 1 : 0);
    static constexpr int D = stream_depth(GATED, GRAD);
    using V = Vec<T, VEC>;
    using W = typename V::W;
    using In = Input<T, VEC>;
    Walk<T> x, g, d;
    int n;
    W* slots;
    __device__ __forceinline__ Stream(const NormArgs& a, int b, const Place& pl, int begin, int end, bool backwards, void* shared)
        : x(a.x, b, 0, pl, a.R, VEC, begin, end, backwards), g(a.gate, b, 0, pl, a.R, VEC, begin, end, backwards),
          d(a.dy, b, 0, pl, a.R, VEC, begin, end, backwards), n(pl.active ? pl.count(a, begin, end) : 0),
          slots(reinterpret_cast<W*>(static_cast<char*>(shared) + a.vectors) + threadIdx.x)
    {
    }
    // vectors i, i + 1 of an even i: one group of copies
    __device__ __forceinline__ W* slot(int i) const { return slots + (i & (D - 1)) * kTensors * (int)blockDim.x; }
    __device__ __forceinline__ void copy(int i, W* s)
    {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (i + k < n)
            {
                W* to = s + k * kTensors * (int)blockDim.x;
                copy_async<V::kBytes, GATED>(to, x.at(k));
                if constexpr (GATED) copy_async<V::kBytes, true>(to + blockDim.x, g.at(k));
                if constexpr (GRAD) copy_async<V::kBytes, false>(to + (kTensors - 1) * (int)blockDim.x, d.at(k));
            }
        x.on(2);
        if constexpr (GATED) g.on(2);
        if constexpr (GRAD) d.on(2);
        copies_commit();
    }
    __device__ __forceinline__ In get(const W* s) const
    {
        In in;
        in.x = s[0];
        if constexpr (GATED) in.g = s[blockDim.x];
        if constexpr (GRAD) in.dy = s[(kTensors - 1) * (int)blockDim.x];
        return in;
    }
    __device__ __forceinline__ void start()
    {
        if constexpr (VEC > 1)
#pragma unroll
            for (int i = 0; i < D; i += 2) copy(i, slot(i));
    }
    template <class Use> __device__ __forceinline__ void run(Use use)
    {
        run_in<0>(use, [] {});
    }
    // fold() after every CHAIN vectors, a power of two
    template <int CHAIN, class Use, class Fold> __device__ __forceinline__ void run_in(Use use, Fold fold)
    {
        if constexpr (VEC > 1)
        {
            int i = 0;
            for (; i + 1 < n; i += 2)
            {
                copies_wait<D / 2 - 1>();
                W* s = slot(i);
                const In a = get(s), b = get(s + kTensors * (int)blockDim.x);
                use(a);
                use(b);
                copy(i + D, s);
                if constexpr (CHAIN > 0)
                    if (((i + 2) & (CHAIN - 1)) == 0) fold();
            }
            if (i < n)
            {
                copies_wait<0>();
                use(get(slot(i)));
            }
        }
        else
        {
            constexpr int U = 4;
            for (int i = 0; i < n; i += U)
            {
                In in[U];
#pragma unroll
                for (int k = 0; k < U; ++k)
                    if (i + k < n)
                    {
                        in[k].x = V::load(x.at(k));
                        if constexpr (GATED) in[k].g = V::load(g.at(k));
                        if constexpr (GRAD) in[k].dy = V::load(d.at(k));
                    }
#pragma unroll
                for (int k = 0; k < U; ++k)
                    if (i + k < n) use(in[k]);
                x.on(U); g.on(U); d.on(U);
                if constexpr (CHAIN > 0)
                    if (((i + U) & (CHAIN - 1)) == 0) fold();
            }
        }
    }
    // the same where use() adds to v, two sums of each of a vector's lanes
    template <class Use> __device__ __forceinline__ void sum(Lanes<VEC> (&v)[2], Use use)
    {
        if constexpr (second_chain(VEC))
        {
            Lanes<VEC> all[2];
            all[0].fill(0.f); all[1].fill(0.f);
            const auto join = [](Lanes<VEC>& to, const Lanes<VEC>& from) {
#pragma unroll
                for (int k = 0; k < Lanes<VEC>::N; ++k) to.p[k] = add(to.p[k], from.p[k]);
            };
            run_in<kChain>(use, [&] {
#pragma unroll
                for (int k = 0; k < 2; ++k) { join(all[k], v[k]); v[k].fill(0.f); }
            });
            join(v[0], all[0]); join(v[1], all[1]);
        }
        else run(use);
    }
};
// u of a vector
template <typename T, int VEC, bool GATED, int ACT> __device__ __forceinline__ Lanes<VEC> value_of(const Input<T, VEC>& in, int rt)
{
    Lanes<VEC> u = Vec<T, VEC>::unpack(in.x);
    if constexpr (GATED)
    {
        const Lanes<VEC> g = Vec<T, VEC>::unpack(in.g);
#pragma unroll
        for (int k = 0; k < Lanes<VEC>::N; ++k) u.p[k] = mul(act_value<T, ACT>(u.p[k], rt), sigmoid(g.p[k]));
    }
    return u;
}

// ---- sums of a block ----------------------------------------------------------------------------------------------------
// v[k]: two sums of each of a thread's channels; what is left of them per slot, a run of m channels, goes to
// buf[((k * (VEC / m) + j / m) * rows + row) * P + ph]. The caller waits at a barrier and adds the rows up, in a fixed order: the same
// bits on every run. In all 2 (VEC / m) rows P floats.
__device__ __forceinline__ int sum_rows(const NormArgs& a) { return 32 % a.P == 0 ? (int)blockDim.x >> 5 : a.R; }
// the lanes of a warp that have the same channels meet where there are any; who writes, and to which row
struct Writer
{
    int row;
    bool here;
    __device__ __forceinline__ Writer(const NormArgs& a, const Place& pl)
    {
        const bool warps = 32 % a.P == 0;
        row = warps ? (int)threadIdx.x >> 5 : pl.r0;
        here = warps ? ((int)threadIdx.x & 31) < a.P : pl.active;
    }
};
template <int VEC, int STEP> __device__ __forceinline__ void put_slots(const Lanes<VEC> (&v)[2], const NormArgs& a, const Place& pl, float* buf)
{
    const Writer w(a, pl);
    const int rows = sum_rows(a);
    if (w.here)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j < VEC; j += STEP) buf[((k * (VEC / STEP) + j / STEP) * rows + w.row) * a.P + pl.ph] = v[k].get(j);
}
template <int VEC> __device__ __forceinline__ void block_sums(Lanes<VEC> (&v)[2], const NormArgs& a, const Place& pl, float* buf)
{
    if (32 % a.P == 0)
        for (int o = 16; o >= a.P; o >>= 1)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[k].set(j, v[k].get(j) + __shfl_xor_sync(0xffffffffu, v[k].get(j), o));
    put_slots<VEC, 1>(v, a, pl, buf);
}

// Moments instead: v holds the sums of u - p and of its square over n rows, p (as its negative) one of the values. A thread's mean and sum
// of squares about it, joined by lanes with d^2 n_a n_b / (n_a + n_b) for means d apart, so nothing cancels wherever the values lie;
// counts[row * P + ph] gets the rows that a row of buf stands for.
template <int VEC, int STEP>
__device__ __forceinline__ void put_moments_of(Lanes<VEC> (&v)[2], const Lanes<VEC>& pivot, int n, const NormArgs& a, const Place& pl, float* buf, float* counts)
{
    float cnt = (float)n;
    const float inv = n > 0 ? __fdividef(1.f, cnt * STEP) : 0.f;
#pragma unroll
    for (int j = 0; j < VEC; j += STEP)
    {
        const float s = v[0].get(j), d = s * inv;
        v[1].set(j, fmaf(-s, d, v[1].get(j)));
        v[0].set(j, d - pivot.get(j));
    }
    if (32 % a.P == 0)
        for (int o = 16; o >= a.P; o >>= 1)
        {
            const float other = __shfl_xor_sync(0xffffffffu, cnt, o), both = cnt + other;
            const float w = both > 0.f ? __fdividef(other, both) : 0.f, shared = cnt * w * STEP;
#pragma unroll
            for (int j = 0; j < VEC; j += STEP)
            {
                const float d = __shfl_xor_sync(0xffffffffu, v[0].get(j), o) - v[0].get(j);
                const float q = __shfl_xor_sync(0xffffffffu, v[1].get(j), o);
                v[1].set(j, v[1].get(j) + q + d * d * shared);
                v[0].set(j, fmaf(d, w, v[0].get(j)));
            }
            cnt = both;
        }
    put_slots<VEC, STEP>(v, a, pl, buf);
    const Writer w(a, pl);
    if (w.here) counts[w.row * a.P + pl.ph] = cnt;
}
template <int VEC>
__device__ __forceinline__ void block_moments(Lanes<VEC> (&v)[2], const Lanes<VEC>& pivot, int n, const NormArgs& a, const Place& pl, float* buf, float* counts)
{
    const int m = a.m;
    if (VEC > 1 && m > 1)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j + 1 < VEC; j += 2) v[k].p[j / 2].x += v[k].p[j / 2].y;
    if (VEC > 2 && m > 2)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j + 2 < VEC; j += 4) v[k].p[j / 2].x += v[k].p[j / 2 + 1].x;
    if constexpr (VEC > 4)
        if (m == 8)
        {
#pragma unroll
            for (int k = 0; k < 2; ++k) v[k].p[0].x += v[k].p[2].x;
            return put_moments_of<VEC, 8>(v, pivot, n, a, pl, buf, counts);
        }
    if constexpr (VEC > 2)
        if (m == 4) return put_moments_of<VEC, 4>(v, pivot, n, a, pl, buf, counts);
    if constexpr (VEC > 1)
        if (m == 2) return put_moments_of<VEC, 2>(v, pivot, n, a, pl, buf, counts);
    put_moments_of<VEC, 1>(v, pivot, n, a, pl, buf, counts);
}

// The block's sums of u and u^2 of a group in 64 bits, for f(g, sums), from what block_moments left: by 2^a.lanes threads a group, or by
// a.warps whole warps, which meet in scratch of a double2 each. Barriers where it takes some.
template <int VEC, class F> __device__ __forceinline__ void group_sums(const NormArgs& a, const float* buf, const float* counts, double2* scratch, F f)
{
    const int sh = __ffs(a.m) - 1, per = VEC >> sh, run = a.Cg >> sh, slots = run * a.ppr, rows = sum_rows(a), second = per * rows * a.P;
    const int lanes = 1 << a.lanes, row_lanes = 1 << a.row_lanes, want = ((a.G << a.lanes) * a.warps + 31) & ~31;
    for (int idx = threadIdx.x; idx < want; idx += blockDim.x)
    {
        // a group's lanes: row_lanes for a slot's rows, so many slots at a time
        int g = idx >> a.lanes, part = 0;
        const int lane = idx & (lanes - 1), row = lane & (row_lanes - 1);
        if (a.warps > 1) { part = g % a.warps; g /= a.warps; }
        double s = 0.0, q = 0.0;
        if (g < a.G)
            for (int slot = (part << (a.lanes - a.row_lanes)) + (lane >> a.row_lanes); slot < slots; slot += (lanes >> a.row_lanes) * a.warps)
            {
                int i = slot, e = g * a.Cg;
                while (i >= run) { i -= run; e += a.C; }
                e += i << sh;
                const int p = e / VEC;
                const float* col = buf + ((e % VEC) >> sh) * rows * a.P + p;
                for (int r = row; r < rows; r += row_lanes)
                {
                    const double mean = (double)col[r * a.P], sum = (double)(counts[r * a.P + p] * (float)a.m) * mean;
                    s += sum;
                    q += fma(sum, mean, (double)col[second + r * a.P]);
                }
            }
        for (int o = lanes >> 1; o > 0; o >>= 1)
        {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            q += __shfl_xor_sync(0xffffffffu, q, o);
        }
        if (g < a.G && lane == 0)
        {
            if (a.warps == 1) f(g, make_double2(s, q));
            else scratch[g * a.warps + part] = make_double2(s, q);
        }
    }
    if (a.warps == 1) return;
    __syncthreads();
    for (int g = threadIdx.x; g < a.G; g += blockDim.x)
    {
        double2 sum = scratch[g * a.warps];
        for (int k = 1; k < a.warps; ++k) { sum.x += scratch[g * a.warps + k].x; sum.y += scratch[g * a.warps + k].y; }
        f(g, sum);
    }
}

// f(g, sums) for the groups of an image from the partial sums [G, chunks] of its chunks, part(k, v) = what partial sum k stands for in
// 64 bits; by 2^a.gather threads a group. The caller waits at a barrier. AHEAD partial sums of a thread are loaded at once: four, but two in
// the gated backward pass, whose loop is short of registers (16 images of 960 x 540 x 16 in bfloat16: 345 us with two, 354 with four; eight
// 402, and 270 for 226 without a gate).
template <int AHEAD, class Part, class F>
__device__ __forceinline__ void gather_groups(const NormArgs& a, int b, Part part, F f)
{
    const float2* __restrict__ from = a.group_part + (size_t)b * a.sums.count * a.G;
    const int lanes = 1 << a.gather, want = ((a.G << a.gather) + 31) & ~31;
    for (int idx = threadIdx.x; idx < want; idx += blockDim.x)
    {
        const int g = idx >> a.gather, lane = idx & (lanes - 1);
        double2 sum = make_double2(0.0, 0.0);
        if (g < a.G)
            loads_ahead<AHEAD>(
                lane, lanes, a.sums.count, [&](int k) { return __ldcg(from + (size_t)g * a.sums.count + k); },
                [&](int k, float2 of) {
                    const double2 v = part(k, of);
                    sum.x += v.x; sum.y += v.y;
                });
        for (int o = lanes >> 1; o > 0; o >>= 1)
        {
            sum.x += __shfl_xor_sync(0xffffffffu, sum.x, o);
            sum.y += __shfl_xor_sync(0xffffffffu, sum.y, o);
        }
        if (g < a.G && lane == 0) f(g, sum);
    }
}
__device__ __forceinline__ float2 mean_rstd(double2 sums, double inv_n, float eps)
{
    const double mean = sums.x * inv_n;
    double var = fma(-mean, mean, sums.y * inv_n);
    if (var < 0.0) var = 0.0;  // a NaN stays one
    return make_float2((float)mean, (float)rsqrt(var + (double)eps));
}

// ---- coefficients of a thread's channels ----------------------------------------------------------------------------------
// (u - mean) scale + b is one fused u scale + (b - mean scale): what that rounds, 2^-25 of mean scale, is what the mean's own
// rounding costs too, and a vector's channels need two registers each instead of three.
template <int VEC> struct Forward
{
    Lanes<VEC> scale, shift;
    __device__ __forceinline__ void set(const NormArgs& a, int ph, const float2* stat, const float* params)
    {
        scale.fill(0.f); shift.fill(0.f);
        for_channels<VEC>(a, ph, [&](int j, int c, int g) {
            const float2 s = stat[g];
            const float k = s.y * params[c];
            scale.set(j, k);
            shift.set(j, fmaf(-s.x, k, params[a.C + c]));
        });
    }
};
template <typename T, int VEC, bool GATED, int ACT>
__device__ __forceinline__ void normalise(Lanes<VEC>& u, const Forward<VEC>& f, int rt)
{
#pragma unroll
    for (int k = 0; k < Lanes<VEC>::N; ++k)
    {
        const float2 z = fma2(u.p[k], f.scale.p[k], f.shift.p[k]);
        u.p[k] = GATED ? z : act_value<T, ACT>(z, rt);
    }
}
// one pivot for the channels that are added up together, the first of them; as its negative
template <int VEC> __device__ __forceinline__ Lanes<VEC> pivot_of(const Lanes<VEC>& u, int m)
{
    Lanes<VEC> p;
    p.fill(0.f);
#pragma unroll
    for (int j = 0; j < VEC; ++j) p.set(j, (j & (m - 1)) ? p.get(j - 1) : -u.get(j));
    return p;
}
template <int VEC> __device__ __forceinline__ void add_moments(const Lanes<VEC>& u, const Lanes<VEC>& pivot, Lanes<VEC> (&v)[2])
{
#pragma unroll
    for (int k = 0; k < Lanes<VEC>::N; ++k)
    {
        const float2 d = add(u.p[k], pivot.p[k]);
        v[0].p[k] = add(v[0].p[k], d);
        v[1].p[k] = fma2(d, d, v[1].p[k]);
    }
}

// ---- forward, images larger than a block's shared memory ------------------------------------------------------------------
// Two launches, sums and what follows, a block on each SM for either (several launches of sums where a block's share is long). They take less than half an SM and may start while the launch in
// front of them runs: the next images' sums and these images' results share the SMs, and a launch has its first vectors when its turn
// comes. Between blocks only the partial sums pass, so nobody waits for a block that may not be resident.
// A 1080p frame of 16 channels in 16 bits (66 MB in, 66 MB out) takes 33.5 us: the sums 14 us (66 MB from HBM beside what the L2 writes back
// of the call before; 10.5 us on a clean L2, 6.3 TB/s), 2 us to the partial sums, 1 us of wait, 1 us to mean and rstd, the results 11 us
// (132 MB from and to the L2). Sums of gated values, where the arithmetic counts: 4.4 TB/s over 537 MB; results 5.7 to 6.1 TB/s.
// Tried and slower: one launch whose blocks take tiles of both kinds by a counter (four images of 33 MB of inputs, backward 97 us against
// 78 us then), clusters that keep an image in their shared memory (sixteen of 1 MB 16.2 us against 13.5 us).
// Shared memory: double2 scratch[16] | block_moments' scratch | vectors
template <typename T, int VEC, bool GATED, int ACT>
__global__ void __launch_bounds__(kNormThreads, kNormBlocks) k_norm_stats(const __grid_constant__ NormArgs a)
{
    extern __shared__ double2 smem[];
    let_next_start();
    const int b = a.image0 + blockIdx.y, part = a.part0 + blockIdx.x * a.part_step;
    int begin, end;
    chunk_of(a, part, begin, end);
    double2* scratch = smem;
    float* buf = reinterpret_cast<float*>(smem + kNormThreads / 32);
    float* counts = buf + 2 * (VEC / a.m) * sum_rows(a) * a.P;
    for (int ph0 = 0; ph0 < a.P; ph0 += blockDim.x)
    {
        const Place pl(a, ph0);
        Lanes<VEC> v[2], pivot;
        v[0].fill(0.f); v[1].fill(0.f); pivot.fill(0.f);
        Stream<T, VEC, GATED, false> in(a, b, pl, begin, end, false, smem);
        in.start();
        bool have = false;
        in.sum(v, [&](const Input<T, VEC>& i) {
            const Lanes<VEC> u = value_of<T, VEC, GATED, ACT>(i, a.act);
            if (!have) pivot = pivot_of<VEC>(u, a.m);
            have = true;
            add_moments<VEC>(u, pivot, v);
        });
        block_moments<VEC>(v, pivot, in.n, a, pl, buf, counts);
    }
    __syncthreads();
    float2* out = a.group_part + (size_t)b * a.sums.count * a.G + part;
    const double inv_n = part < a.sums.more ? a.inv_long : a.inv_short;
    group_sums<VEC>(a, buf, counts, scratch, [&](int g, double2 sums) {
        // the chunk's mean and sum of squares about it: 32 bits hold these
        const double mean = sums.x * inv_n;
        out[(size_t)g * a.sums.count] = make_float2((float)mean, (float)fma(-mean, sums.x, sums.y));
    });
    wait_previous();
}

// Shared memory: float2 stat[G] | float params[2 C] | vectors
template <typename T, int VEC, bool GATED, int ACT>
__global__ void __launch_bounds__(kNormThreads, kNormBlocks) k_norm_apply(const __grid_constant__ NormArgs a)
{
    extern __shared__ double2 smem[];
    let_next_start();
    const int T_ = blockDim.x, b = a.image0 + blockIdx.y;
    int begin, end;
    chunk_of(a, blockIdx.x, begin, end);
    float2* stat = reinterpret_cast<float2*>(smem);
    float* params = reinterpret_cast<float*>(stat + a.G);
    for (int ph0 = 0; ph0 < a.P; ph0 += T_)
    {
        const Place pl(a, ph0);
        // from the end: what the sums read last is what the L2 still has
        Stream<T, VEC, GATED, false> in(a, b, pl, begin, end, true, smem);
        in.start();
        if (ph0 == 0)
        {
            stage_params(a, 0, params);
            wait_previous();
            const double per_row = (double)(a.ppr * a.Cg);
            gather_groups<4>(
                a, b,
                [&](int k, float2 v) {
                    const double mean = v.x, s = (double)(a.sums.rows + (k < a.sums.more ? 1 : 0)) * per_row * mean;
                    return make_double2(s, fma(s, mean, (double)v.y));
                },
                [&](int g, double2 sums) {
                    const float2 s = mean_rstd(sums, a.inv_n, a.eps);
                    stat[g] = s;
                    if (a.mean && blockIdx.x == 0)
                    {
                        a.mean[(size_t)b * a.G + g] = s.x;
                        a.rstd[(size_t)b * a.G + g] = s.y;
                    }
                });
            __syncthreads();
        }
        if (!pl.active) continue;
        Forward<VEC> f;
        f.set(a, pl.ph, stat, params);
        Walk<T> y(a.y, b, 0, pl, a.R, VEC, begin, end, true);
        in.run([&](const Input<T, VEC>& i) {
            Lanes<VEC> u = value_of<T, VEC, GATED, ACT>(i, a.act);
            normalise<T, VEC, GATED, ACT>(u, f, a.act);
            Vec<T, VEC>::store(y.p, u);
            y.on(1);
        });
    }
}

// ---- backward -------------------------------------------------------------------------------------------------------------
// As the forward pass: sums of dz and dz uhat per channel, then dx. Over 537 MB of x and dy the sums run at 4.7 TB/s behind a SiLU (6.4 TB/s
// without an activation), dx at 5.8 to 6.1 TB/s of 805 MB; four images of 512 x 512 x 32 in bfloat16 take 62 us in all (201 MB, 3.2 TB/s), as the
// first launch finds the L2 full of the last call's results and the last one has the SMs to itself.
// uhat = u rstd + centre and z = uhat w + b of a vector
template <int VEC> struct Saved
{
    Lanes<VEC> rstd, centre, w, bias;
    __device__ __forceinline__ void set(const NormArgs& a, int ph, const float2* stat, const float* params)
    {
        rstd.fill(0.f); centre.fill(0.f); w.fill(0.f); bias.fill(0.f);
        for_channels<VEC>(a, ph, [&](int j, int c, int g) {
            const float2 s = stat[g];
            rstd.set(j, s.y);
            centre.set(j, -s.x * s.y);
            w.set(j, params[c]);
            bias.set(j, params[a.C + c]);
        });
    }
};
// mean and rstd of the image's groups from g0 on; a barrier follows
__device__ __forceinline__ void stage_stats(const NormArgs& a, size_t g0, float2* to)
{
    for (int g = threadIdx.x; g < a.G; g += blockDim.x) to[g] = make_float2(a.mean[g0 + g], a.rstd[g0 + g]);
}
template <typename T, int VEC, bool GATED, int ACT>
__device__ __forceinline__ void add_grad_sums(const Input<T, VEC>& in, const Saved<VEC>& s, Lanes<VEC> (&v)[2], int rt)
{
    const Lanes<VEC> u = value_of<T, VEC, GATED, ACT>(in, rt), d = Vec<T, VEC>::unpack(in.dy);
#pragma unroll
    for (int k = 0; k < Lanes<VEC>::N; ++k)
    {
        const float2 uhat = fma2(u.p[k], s.rstd.p[k], s.centre.p[k]);
        const float2 dz = GATED ? d.p[k] : act_grad<T, ACT>(fma2(uhat, s.w.p[k], s.bias.p[k]), d.p[k], rt);
        v[0].p[k] = add(v[0].p[k], dz);
        v[1].p[k] = fma2(dz, uhat, v[1].p[k]);
    }
}
// z = u scale + shift, du = dz scale + u slope + offset, with scale = rstd w, slope = -rstd^2 c2, offset = -rstd c1 - mean slope
template <int VEC> struct Backward
{
    Lanes<VEC> scale, shift, slope, offset;
    __device__ __forceinline__ void set(const NormArgs& a, int ph, const float2* stat, const float2* c12, const float* params)
    {
        scale.fill(0.f); shift.fill(0.f); slope.fill(0.f); offset.fill(0.f);
        for_channels<VEC>(a, ph, [&](int j, int c, int g) {
            const float2 st = stat[g], c_ = c12[g];
            const float r = st.y, mean = st.x, k = r * params[c], sl = -r * r * c_.y;
            scale.set(j, k);
            shift.set(j, fmaf(-mean, k, params[a.C + c]));
            slope.set(j, sl);
            offset.set(j, fmaf(-mean, sl, -r * c_.x));
        });
    }
};
template <typename T, int VEC, bool GATED, int ACT>
__device__ __forceinline__ void input_gradient(const Input<T, VEC>& in, const Backward<VEC>& c, Lanes<VEC>& dx, Lanes<VEC>& dg, int rt)
{
    const Lanes<VEC> d = Vec<T, VEC>::unpack(in.dy), u = Vec<T, VEC>::unpack(in.x);
    if constexpr (!GATED)
    {
#pragma unroll
        for (int k = 0; k < Lanes<VEC>::N; ++k)
        {
            const float2 dz = act_grad<T, ACT>(fma2(u.p[k], c.scale.p[k], c.shift.p[k]), d.p[k], rt);
            dx.p[k] = fma2(dz, c.scale.p[k], fma2(u.p[k], c.slope.p[k], c.offset.p[k]));
        }
    }
    else
    {
        const Lanes<VEC> g = Vec<T, VEC>::unpack(in.g);
#pragma unroll
        for (int k = 0; k < Lanes<VEC>::N; ++k)
        {
            float2 value, slope, s, ns;
            act_both<T, ACT>(u.p[k], value, slope, rt);
            sigmoid_pair(g.p[k], s, ns);
            const float2 vs = mul(value, s);
            const float2 du = fma2(d.p[k], c.scale.p[k], fma2(vs, c.slope.p[k], c.offset.p[k]));
            dx.p[k] = mul(du, mul(slope, s));
            dg.p[k] = mul(du, mul(vs, ns));
        }
    }
}
// channel sums chan[2][C] from the slots' (a row may hold several pixels), then f(g, the group's sums of w dz and w dz uhat)
template <int VEC, class F>
__device__ __forceinline__ void channel_and_group_sums(const NormArgs& a, const float* params, float* buf, float* chan, F f)
{
    const int T = blockDim.x, t = threadIdx.x;
    int rows = sum_rows(a);
    // many rows of few columns: all threads take some first
    const int columns = 2 * VEC * a.P, parts = T / columns;
    if (parts > 1 && rows > 2 * parts)
    {
        const int part = t / columns, i = t - part * columns, slot = i / a.P;
        float s = 0.f;
        if (part < parts)
#pragma unroll 4
            for (int r = part; r < rows; r += parts) s += buf[(slot * rows + r) * a.P + i - slot * a.P];
        __syncthreads();
        if (part < parts) buf[(slot * parts + part) * a.P + i - slot * a.P] = s;
        __syncthreads();
        rows = parts;
    }
    for (int i = t; i < 2 * a.C; i += T)
    {
        const int k = i >= a.C, c = i - k * a.C;
        float s = 0.f;
        for (int q = 0; q < a.ppr; ++q)
        {
            const int e = q * a.C + c;
            const float* col = buf + (k * VEC + e % VEC) * rows * a.P + e / VEC;
#pragma unroll 4
            for (int r = 0; r < rows; ++r) s += col[r * a.P];
        }
        chan[i] = s;
    }
    __syncthreads();
    const int lanes = 1 << a.lanes, want = ((a.G << a.lanes) + 31) & ~31;
    for (int idx = t; idx < want; idx += T)
    {
        const int g = idx >> a.lanes, lane = idx & (lanes - 1);
        double s = 0.0, q = 0.0;
        if (g < a.G)
            for (int i = lane; i < a.Cg; i += lanes)
            {
                const int c = g * a.Cg + i;
                const double w = (double)params[c];
                s = fma(w, (double)chan[c], s);
                q = fma(w, (double)chan[a.C + c], q);
            }
        for (int o = lanes >> 1; o > 0; o >>= 1)
        {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            q += __shfl_xor_sync(0xffffffffu, q, o);
        }
        if (g < a.G && lane == 0) f(g, make_double2(s, q));
    }
}

// Shared memory: float2 stat[G] | float params[2 C] | chan[2 C] | block_sums' scratch | vectors
template <typename T, int VEC, bool GATED, int ACT>
__global__ void __launch_bounds__(kNormGradThreads, kNormGradBlocks) k_norm_grad_sums(const __grid_constant__ NormArgs a)
{
    extern __shared__ double2 smem[];
    let_next_start();
    const int b = a.image0 + blockIdx.y, part = a.part0 + blockIdx.x * a.part_step;
    int begin, end;
    chunk_of(a, part, begin, end);
    float2* stat = reinterpret_cast<float2*>(smem);
    float* params = reinterpret_cast<float*>(stat + a.G);
    float* chan = params + 2 * a.C;
    float* buf = chan + 2 * a.C;
    for (int ph0 = 0; ph0 < a.P; ph0 += blockDim.x)
    {
        const Place pl(a, ph0);
        Stream<T, VEC, GATED, true> in(a, b, pl, begin, end, false, smem);
        if (ph0 == 0)
        {
            // before the copies, behind which they would wait 5 us for their values
            stage_params(a, 0, params);
            stage_stats(a, (size_t)b * a.G, stat);
        }
        in.start();
        if (ph0 == 0) __syncthreads();
        Lanes<VEC> v[2];
        v[0].fill(0.f); v[1].fill(0.f);
        if (pl.active)
        {
            Saved<VEC> s;
            s.set(a, pl.ph, stat, params);
            in.sum(v, [&](const Input<T, VEC>& i) { add_grad_sums<T, VEC, GATED, ACT>(i, s, v, a.act); });
        }
        block_sums<VEC>(v, a, pl, buf);
    }
    __syncthreads();
    float2* out = a.group_part + (size_t)b * a.sums.count * a.G + part;
    channel_and_group_sums<VEC>(a, params, buf, chan, [&](int g, double2 sums) { out[(size_t)g * a.sums.count] = make_float2((float)sums.x, (float)sums.y); });
    if (a.channel_part)
        for (int c = threadIdx.x; c < a.C; c += blockDim.x) a.channel_part[((size_t)b * a.sums.count + part) * a.C + c] = make_float2(chan[c], chan[a.C + c]);
    wait_previous();
}

// db and dw of nc channels from c0 on from the partial sums of each, in 64 bits and in a fixed order.
// Scratch: 2 blockDim double.
__device__ __forceinline__ void param_gradients(const NormArgs& a, int c0, int nc, double* scratch)
{
    const int T = blockDim.x, t = threadIdx.x, ways = T / nc;
    const int w = t / nc, c = t - w * nc;
    double s = 0.0, q = 0.0;
    if (w < ways)
        loads_ahead<4>(
            w, ways, a.param_parts, [&](int k) { return __ldcg(a.channel_part + (size_t)k * a.C + c0 + c); },
            [&](int, float2 v) { s += v.x; q += v.y; });
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

// Shared memory: float2 c12[G] | stat[G] | float params[2 C] | vectors; the parameter blocks 2 blockDim double
template <typename T, int VEC, bool GATED, int ACT>
__global__ void __launch_bounds__(kNormGradThreads, kNormGradBlocks) k_norm_grad_apply(const __grid_constant__ NormArgs a)
{
    extern __shared__ double2 smem[];
    let_next_start();
    const int T_ = blockDim.x, b = a.image0 + blockIdx.y;
    if ((int)blockIdx.x < a.param_blocks)
    {
        wait_previous();
        if (blockIdx.y == 0)
        {
            const int c0 = blockIdx.x * kParamChannels;
            param_gradients(a, c0, min(kParamChannels, a.C - c0), reinterpret_cast<double*>(smem));
        }
        return;
    }
    int begin, end;
    chunk_of(a, blockIdx.x - a.param_blocks, begin, end);
    float2* c12 = reinterpret_cast<float2*>(smem);
    float2* stat = c12 + a.G;
    float* params = reinterpret_cast<float*>(stat + a.G);
    for (int ph0 = 0; ph0 < a.P; ph0 += T_)
    {
        const Place pl(a, ph0);
        Stream<T, VEC, GATED, true> in(a, b, pl, begin, end, true, smem);
        in.start();
        if (ph0 == 0)
        {
            stage_params(a, 0, params);
            stage_stats(a, (size_t)b * a.G, stat);
            wait_previous();
            gather_groups<GATED ? 2 : 4>(
                a, b, [&](int, float2 v) { return make_double2(v.x, v.y); },
                [&](int g, double2 sums) { c12[g] = make_float2((float)(sums.x * a.inv_n), (float)(sums.y * a.inv_n)); });
            __syncthreads();
        }
        if (!pl.active) continue;
        Backward<VEC> c;
        c.set(a, pl.ph, stat, c12, params);
        Walk<T> dx(a.dx, b, 0, pl, a.R, VEC, begin, end, true), dg(a.dgate, b, 0, pl, a.R, VEC, begin, end, true);
        in.run([&](const Input<T, VEC>& i) {
            Lanes<VEC> o, og;
            input_gradient<T, VEC, GATED, ACT>(i, c, o, og, a.act);
            Vec<T, VEC>::store(dx.p, o);
            dx.on(1);
            if constexpr (GATED)
            {
                Vec<T, VEC>::store(dg.p, og);
                dg.on(1);
            }
        });
    }
}

// ---- images that fit a block's shared memory ----------------------------------------------------------------------------------
// A block keeps an image, or some groups' channels of it, between the sums and what follows: one launch, every value read once. A
// thread copies, reads and overwrites vectors of its own only. Bound by the latency of the one chain from the first copy to the last store:
// 5.1 us for 120 pixels of 64 channels.
// n vectors in four groups: all copies are under way before the first group is used
template <class Copy, class Between, class Use> __device__ __forceinline__ void staged(int n, int most, Copy copy, Between between, Use use)
{
    const int quarter = (most + 3) / 4;
#pragma unroll
    for (int q = 0; q < 4; ++q)
    {
        for (int i = q * quarter; i < min(n, (q + 1) * quarter); ++i) copy(i);
        copies_commit();
    }
    between();
    copies_wait<3>();
    for (int i = 0; i < min(n, quarter); ++i) use(i);
    copies_wait<2>();
    for (int i = quarter; i < min(n, 2 * quarter); ++i) use(i);
    copies_wait<1>();
    for (int i = 2 * quarter; i < min(n, 3 * quarter); ++i) use(i);
    copies_wait<0>();
    for (int i = 3 * quarter; i < n; ++i) use(i);
}

// Shared memory: double2 scratch[16] | float2 stat[G] | float params[2 C] | block_moments' scratch | vectors
template <typename T, int VEC, bool GATED, int ACT>
__global__ void __launch_bounds__(kNormThreads, kNormBlocks) k_norm_resident(const __grid_constant__ NormArgs a)
{
    extern __shared__ double2 smem[];
    const int T_ = blockDim.x, b = blockIdx.x >> a.slices, slice = blockIdx.x - (b << a.slices), c0 = slice * a.C;
    double2* scratch = smem;
    float2* stat = reinterpret_cast<float2*>(smem + kNormThreads / 32);
    float* params = reinterpret_cast<float*>(stat + a.G);
    float* buf = params + 2 * a.C;
    float* counts = buf + 2 * (VEC / a.m) * sum_rows(a) * a.P;
    using V = Vec<T, VEC>;
    using W = typename V::W;
    using In = Input<T, VEC>;
    const int most = (a.rows - 1) / a.R + 1;
    W* sx = reinterpret_cast<W*>(reinterpret_cast<char*>(smem) + a.vectors) + threadIdx.x;
    W* sg = sx + (size_t)most * T_;
    const Place pl(a, 0);
    const int n = pl.active ? pl.count(a, 0, a.rows) : 0;
    // u in 32 bits takes the room of x and of the gate, or of x alone
    Lanes<VEC> v[2], pivot;
    v[0].fill(0.f); v[1].fill(0.f); pivot.fill(0.f);
    Walk<T> x(a.x, b, c0, pl, a.R, VEC, 0, a.rows, false), g(a.gate, b, c0, pl, a.R, VEC, 0, a.rows, false);
    bool have = false;
    staged(
        n, most,
        [&](int i) {
            copy_async<V::kBytes, GATED>(sx + i * T_, x.p);
            x.on(1);
            if constexpr (GATED)
            {
                copy_async<V::kBytes, true>(sg + i * T_, g.p);
                g.on(1);
            }
        },
        [&] { stage_params(a, c0, params); },
        [&](int i) {
            In in;
            in.x = sx[i * T_];
            if constexpr (GATED) in.g = sg[i * T_];
            const Lanes<VEC> u = value_of<T, VEC, GATED, ACT>(in, a.act);
            if (!have) pivot = pivot_of<VEC>(u, a.m);
            have = true;
            add_moments<VEC>(u, pivot, v);
            if constexpr (GATED)
            {
                sx[i * T_] = *reinterpret_cast<const W*>(&u);
                if constexpr (sizeof(T) == 2) sg[i * T_] = *reinterpret_cast<const W*>(reinterpret_cast<const char*>(&u) + V::kBytes);
            }
        });
    block_moments<VEC>(v, pivot, n, a, pl, buf, counts);
    __syncthreads();
    const size_t g0 = (size_t)blockIdx.x * a.G;
    group_sums<VEC>(a, buf, counts, scratch, [&](int i, double2 sums) {
        const float2 s = mean_rstd(sums, a.inv_n, a.eps);
        stat[i] = s;
        if (a.mean)
        {
            a.mean[g0 + i] = s.x;
            a.rstd[g0 + i] = s.y;
        }
    });
    __syncthreads();
    if (n == 0) return;
    Forward<VEC> f;
    f.set(a, pl.ph, stat, params);
    Walk<T> y(a.y, b, c0, pl, a.R, VEC, 0, a.rows, false);
#pragma unroll 2
    for (int i = 0; i < n; ++i)
    {
        Lanes<VEC> u;
        const W w = sx[i * T_];
        if constexpr (!GATED) u = V::unpack(w);
        else
        {
            *reinterpret_cast<W*>(&u) = w;
            if constexpr (sizeof(T) == 2) *reinterpret_cast<W*>(reinterpret_cast<char*>(&u) + V::kBytes) = sg[i * T_];
        }
        normalise<T, VEC, GATED, ACT>(u, f, a.act);
        V::store(y.p, u);
        y.on(1);
    }
}

// ---- the gate alone -----------------------------------------------------------------------------------------------------
// One pass, two blocks an SM: a 4K frame of 8 channels in bfloat16 66 us (398 MB, 6.0 TB/s), backward over two 1080p frames of 16 channels
// 123 us (663 MB, 5.4 TB/s).
// Shared memory: vectors
template <typename T, int VEC, bool GATED, int ACT>
__global__ void __launch_bounds__(kNormThreads, kNormBlocks) k_gate(const __grid_constant__ NormArgs a)
{
    extern __shared__ double2 smem[];
    const int b = blockIdx.y;
    int begin, end;
    chunk_of(a, blockIdx.x, begin, end);
    for (int ph0 = 0; ph0 < a.P; ph0 += blockDim.x)
    {
        const Place pl(a, ph0);
        Stream<T, VEC, true, false> in(a, b, pl, begin, end, false, smem);
        in.start();
        Walk<T> y(a.y, b, 0, pl, a.R, VEC, begin, end, false);
        in.run([&](const Input<T, VEC>& i) {
            Vec<T, VEC>::store(y.p, value_of<T, VEC, true, ACT>(i, a.act));
            y.on(1);
        });
    }
}
template <typename T, int VEC, bool GATED, int ACT>
__global__ void __launch_bounds__(kNormGradThreads, kNormGradBlocks) k_gate_grad(const __grid_constant__ NormArgs a)
{
    extern __shared__ double2 smem[];
    const int b = blockIdx.y;
    int begin, end;
    chunk_of(a, blockIdx.x, begin, end);
    using V = Vec<T, VEC>;
    for (int ph0 = 0; ph0 < a.P; ph0 += blockDim.x)
    {
        const Place pl(a, ph0);
        Stream<T, VEC, true, true> in(a, b, pl, begin, end, false, smem);
        in.start();
        Walk<T> dx(a.dx, b, 0, pl, a.R, VEC, begin, end, false), dg(a.dgate, b, 0, pl, a.R, VEC, begin, end, false);
        in.run([&](const Input<T, VEC>& i) {
            Lanes<VEC> f = V::unpack(i.x), e = V::unpack(i.g), dy = V::unpack(i.dy);
#pragma unroll
            for (int q = 0; q < Lanes<VEC>::N; ++q)
            {
                float2 value, slope, s, ns;
                act_both<T, ACT>(f.p[q], value, slope, a.act);
                sigmoid_pair(e.p[q], s, ns);
                const float2 ds = mul(dy.p[q], s);
                f.p[q] = mul(ds, slope);
                e.p[q] = mul(ds, mul(value, ns));
            }
            V::store(dx.p, f);
            V::store(dg.p, e);
            dx.on(1); dg.on(1);
        });
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
    if constexpr (VEC > 1)
        if (which == kNormResident) return (const void*)k_norm_resident<T, VEC, GATED, ACT>;
    return nullptr;
}
template <typename T, int VEC, bool GATED> const void* pick_act(int which, int act)
{
    if constexpr (VEC > 1)
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
    if constexpr (sizeof(T) == 2)
        if (vec == kVec4) return gated ? pick<T, 2, true, 4>(which) : pick<T, 2, false, 4>(which);
    return gated ? pick_act<T, 1, true>(which, act) : pick_act<T, 1, false>(which, act);
}

}  // namespace norm
}  // namespace adop
