// Residual addition, root-mean-square norm and quantisation of the result in one pass: the producer of the A operand of the
// W8A8 matmuls (int8, one fp32 scale per row) and of the MX matmuls (fp8 / fp4, one E8M0 scale per 32 elements).
//
//   h = src + residual (fp32, not rounded)            residualOut = cast(h)
//   y = h * rstd * gamma,  rstd = 1 / sqrt(mean(h^2) + epsilon)                        normOut = cast(y)
//   int8:  scale = max|y| / 127,  q = RINT(y * 127 / max|y|)
//   MX:    e = floor(log2 max|y|) - emax per block of 32,  scale byte = e + 127,  q = cast(y * 2^-e)
//
// What bounds it: HBM.  With bf16 tensors and residualOut an element costs 2 + 2 bytes read, 2 + 1 written.  A CTA owns whole rows and
// keeps a row in registers between the reduction and the quantisation, so each byte moves once; the next row is requested before the
// reduction.  bf16 [16384, 7168] to e4m3: 141 us = 5.9 TB/s, 0.91 of the measured copy rate (134 us without the look at ties;
// before that, 164 without the early request); to e2m1 130 us; [2048, 16384] to int8 38 us, to e4m3 45.  For int8 the row's maximum needs no second reduction: max|y| = rstd * max|h * gamma|, so sum(h^2) and max|h * gamma| go through the same
// shuffles and the same barrier, and RINT(y * 127 / max|y|) = RINT((h * gamma) * (127 / max|h * gamma|)) does not need rstd.
#include "elementwise.cuh"

using namespace ascq;

namespace ascq {
namespace {

enum : int { kOutI8 = 0, kOutE4M3 = 1, kOutE5M2 = 2, kOutE2M1 = 3 };
// exponent of the largest binade of each element type (OCP MX: the shared exponent is floor(log2 amax) minus it)
__host__ __device__ constexpr int out_emax(int out) { return out == kOutE4M3 ? 8 : out == kOutE5M2 ? 15 : 2; }

struct NormArgs {
    void* dst;
    void* scaleOut;
    void* residualOut;     // may be null
    void* normOut;         // may be null
    const void* src;
    const void* residual;  // may be null
    const void* gamma;
    uint32_t m, n;
    int64_t ldSrc, ldResidual, ldResidualOut, ldNormOut;
    float epsilon;
    int out;               // kernel for odd shapes only: the vector kernel has it as a template parameter
};

__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// largest magnitude of three, NaN if one of them is
__device__ __forceinline__ float max_abs3(float a, float b, float c)
{
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max_abs8(const float (&f)[8])
{
    return max_abs3(max_abs3(max_abs3(f[0], f[1], f[2]), f[3], f[4]), max_abs3(f[5], f[6], f[7]), 0.f);
}
// d += a^2 for two lanes, each rounded on its own
__device__ __forceinline__ void fma2_square(float& d0, float& d1, float a0, float a1)
{
    asm("{\n\t.reg .b64 a, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 d, {%0, %1};\n\tfma.rn.f32x2 d, a, a, d;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "+f"(d0), "+f"(d1)
        : "f"(a0), "f"(a1));
}
__device__ __forceinline__ bool finite_f32(float v) { return fabsf(v) <= 3.4028234663852886e38f; }

// 8 consecutive elements: 16 bytes of a 16-bit type, 32 of fp32 (two 16-byte loads)
template <typename T> struct Vec8 {
    uint4 w[sizeof(T) / 2];
};
template <typename T> __device__ __forceinline__ Vec8<T> load8(const T* p)
{
    Vec8<T> v;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) v.w[i] = __ldcg(reinterpret_cast<const uint4*>(p) + i);
    return v;
}
template <typename T> __device__ __forceinline__ void widen8(const Vec8<T>& v, float (&f)[8])
{
    if constexpr (sizeof(T) == 4) {
        const uint32_t a[8] = {v.w[0].x, v.w[0].y, v.w[0].z, v.w[0].w, v.w[1].x, v.w[1].y, v.w[1].z, v.w[1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(a[i]);
    } else {
        const uint32_t a[4] = {v.w[0].x, v.w[0].y, v.w[0].z, v.w[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                f[2 * i] = __uint_as_float(a[i] << 16);
                f[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
            } else {
                const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&a[i]));
                f[2 * i] = t.x;
                f[2 * i + 1] = t.y;
            }
        }
    }
}
template <typename T> __device__ __forceinline__ T narrow(float f)
{
    if constexpr (std::is_same<T, float>::value) return f;
    else if constexpr (std::is_same<T, __half>::value) return f32_to_f16_sat(f);
    else return f32_to_bf16_sat(f);
}
// Squares up to here come from values that T holds; fp32's own largest where the square would overflow.
template <typename T> constexpr float kMostSquaredOf = std::is_same<T, __half>::value ? 65504.0f * 65504.0f : 3.4028234663852886e38f;
// the framework's narrowing rule: round to nearest even, a finite value that overflows saturates.  `fits`: none of them is beyond the type's
// largest value (nor NaN); only a vector that may hold one is looked at element by element.
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&f)[8], bool fits)
{
    if constexpr (sizeof(T) == 4) {
        __stcs(reinterpret_cast<float4*>(p), make_float4(f[0], f[1], f[2], f[3]));
        __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(f[4], f[5], f[6], f[7]));
    } else {
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r[i]) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
            else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r[i]) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
        }
        if (__builtin_expect(!fits, 0)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (std::is_same<T, __half>::value) r[i] = pack_f16x2_sat(f[2 * i], f[2 * i + 1]);
                else r[i] = pack_bf16x2_sat(f[2 * i], f[2 * i + 1]);
            }
        }
        __stcs(reinterpret_cast<uint4*>(p), make_uint4(r[0], r[1], r[2], r[3]));
    }
}

// Two scaled values -> two codes, the first in the low byte (or nibble); round to nearest even, saturating.  fp4 goes through
// bfloat16 first, the conversion chain of AscendQuant's fp4 destination.
template <int OUT> __device__ __forceinline__ uint32_t mx_pair(float first, float second)
{
    unsigned short r;
    if constexpr (OUT == kOutE4M3) asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(first), "f"(second));
    else if constexpr (OUT == kOutE5M2) asm("cvt.rn.satfinite.e5m2x2.f32 %0, %2, %1;" : "=h"(r) : "f"(first), "f"(second));
    else {
        uint32_t b2;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(b2) : "f"(second), "f"(first));
        asm("{ .reg .b8 t;\n cvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n mov.b16 %0, {t, 0}; }"
            : "=h"(r)
            : "f"(__uint_as_float(b2 << 16)), "f"(__uint_as_float(b2 & 0xFFFF0000u)));
    }
    return r;
}
// Shared exponent of a block whose largest |h * gamma| is `amax`: floor(log2(amax * rstd)) - emax inside the E8M0 range, 0 for an all-zero
// block.  The product is taken with the remainder of rstd and of its own rounding: where it rounds up to a power of two the exact
// one may lie below, and an exponent off by one doubles the block's grid.  What is left is the rounding of h * gamma itself: a block whose largest |y| is
// within half a unit in the last place of a power of two may get the exponent of the other side, one block in tens of millions.  (Looking at such blocks again from h
// and gamma was measured in seven forms: inside the row loop it takes the loop's registers, at best 153 us instead of 140 at bf16 [16384, 7168], and behind
// the loop more.)  A subnormal product counts as 2^-126; with emax >= 2 it ends at the range's lower end either way.
__device__ __forceinline__ int mx_exponent(float amax, float rstd, float rstdLo, int emax)
{
    if (!(amax > 0.f)) return 0;
    const float y = __fmul_rn(amax, rstd), rest = fmaf(amax, rstdLo, fmaf(amax, rstd, -y));
    const uint32_t bits = __float_as_uint(y);
    int ex = static_cast<int>(bits >> 23);
    ex = ex == 0 ? -126 : ex - 127;
    if ((bits & 0x7FFFFFu) == 0 && rest < 0.f) --ex;
    return min(max(ex - emax, -127), 127);
}
// 2^-e for e in [-127, 127]; 2^-127 is a subnormal
__device__ __forceinline__ float exp2_neg(int e) { return e == 127 ? __uint_as_float(0x00400000u) : __uint_as_float(static_cast<uint32_t>(127 - e) << 23); }
// Whether a block with shared exponent e takes one multiplication, by f = rstd * 2^-e: no |y| that has a code other than 0 is near fp32's
// subnormals, nor, with f below 2^100, an |h * gamma| that has a normal one.  (Beyond is f only where epsilon and the row are tiny: rstd is at most 2^10 for epsilon
// = 1e-6.)
__device__ __forceinline__ bool single_factor(int e, float f) { return e > -80 && e < 80 && f < 1.2676506002282294e30f; }

// Codes on the right side of a tie.  v = fl(fl(h * gamma) * fl(rstd * 2^-e)) is within 2.5 units in the last place of y * 2^-e; only a v
// closer than that to the middle between two codes can be cast to the wrong one, and four units are looked at: one element in 116,000 (E5M2: in 233,000).
template <int OUT> struct Tie {
    static constexpr bool kLooked = OUT == kOutE4M3 || OUT == kOutE5M2;  // (fp4 goes through bfloat16, whose own rounding is part of its definition)
    static constexpr int kDrop = OUT == kOutE4M3 ? 20 : 21;              // mantissa bits that the cast drops; the middle is 100...0
    // small for a v next to a tie: its dropped bits, counted from four units below the middle
    static __device__ __forceinline__ uint32_t distance(float v) { return (__float_as_uint(v) << (32 - kDrop)) + (0x80000000u + (4u << (32 - kDrop))); }
    static __device__ __forceinline__ uint32_t least(const float (&v)[8])
    {
        return __vimin3_u32(__vimin3_u32(__vimin3_u32(distance(v[0]), distance(v[1]), distance(v[2])), distance(v[3]), distance(v[4])), distance(v[5]),
                            min(distance(v[6]), distance(v[7])));
    }
    static constexpr float kLowest = OUT == kOutE4M3 ? 0.015625f : 6.103515625e-05f;  // the smallest normal code
    static constexpr uint32_t kNear = 8u << (32 - kDrop);
    // v, moved to the side of the tie where h * gamma * (rstd + rstdLo) * up lies (on it if that is exactly the middle).  Codes below
    // the smallest normal one have their ties elsewhere, at dropped bits 0, where nothing is moved.
    static __device__ __forceinline__ float settle(float h, float gamma, float rstd, float rstdLo, float up)
    {
        const float p = __fmul_rn(h, gamma), pl = fmaf(h, gamma, -p), f = __fmul_rn(rstd, up), v = __fmul_rn(p, f);
        const float rest = __fadd_rn(fmaf(p, f, -v), fmaf(pl, f, __fmul_rn(p, __fmul_rn(rstdLo, up))));
        const uint32_t middle = (__float_as_uint(v) & ~((1u << kDrop) - 1u)) | (1u << (kDrop - 1));
        const float d = __fadd_rn(__fsub_rn(v, __uint_as_float(middle)), rest), out = v < 0.f ? -d : d;
        return __uint_as_float(out > 0.f ? middle + 1u : out < 0.f ? middle - 1u : middle);
    }
};

// h = src + residual of an element whose v = fl(fl(h * gamma) * f) is known, formed again although residualOut may have taken the place of one of
// the two: v / (gamma * f) is within 5 units of h's last place, so the lost one is the value of T nearest to it less the other, unless the
// lost one is so small beside h that T has several values there (see `separable`).  False then, and in the same cases where both are in memory, so that
// a call in place gives the bits of one that is not.  (Keeping the old values: in
// registers 171 us, in shared memory, which is taken from L1, 158; this way 141 to 143; 134 without a look at ties, with ten times as many codes off.)
template <typename T> __device__ __forceinline__ bool separable(float a, float b, float h)
{
    // bf16: off by 8 * 2^-24 |h| at most, T's values at a are 2^-8 |a| apart at least (2^-9 next to a power of two); fp16: 2^-11, 2^-12
    constexpr float kLeast = std::is_same<T, __half>::value ? 0.00390625f : 0.00048828125f;
    return sizeof(T) == 4 || fminf(fabsf(a), fabsf(b)) >= kLeast * fabsf(h);  // (fp32: h itself is in memory, in residualOut or as the two)
}
template <typename T> __device__ __forceinline__ bool row_sum(T x, T r, float v, float gamma, float f, bool overSrc, bool overRes, float& h)
{
    float a = to_f32<T>(x), b = to_f32<T>(r);
    if (overSrc || overRes) {
        const float whole = __fdiv_rn(v, __fmul_rn(gamma, f));
        if (overSrc && overRes) a = b = to_f32<T>(narrow<T>(0.5f * whole));  // src and residual are one tensor
        else if (overSrc) a = to_f32<T>(narrow<T>(__fsub_rn(whole, b)));
        else b = to_f32<T>(narrow<T>(__fsub_rn(whole, a)));
    }
    h = __fadd_rn(a, b);
    return separable<T>(a, b, h);
}

// The int8 chain's multiplier 127 / amax, in two factors so that it does not overflow where amax is close to the smallest
// normal number: q = RINT((p * pre) * mul).  pre is 1 for every amax that a norm leaves in practice.
struct I8Factor {
    float pre, mul;
};
__device__ __forceinline__ I8Factor i8_factor(float amax)
{
    I8Factor f;
    f.pre = amax < 1e-30f ? 1.2089258196146292e24f : 1.0f;  // 2^80
    f.mul = amax > 0.f ? __fdiv_rn(127.0f, amax * f.pre) : 1.0f;
    return f;
}

// A sum as two floats: hi is its nearest float, lo what is missing.
struct Sum2 {
    float hi, lo;
};
__device__ __forceinline__ Sum2 add_exact(Sum2 a, Sum2 b)
{
    const float s = __fadd_rn(a.hi, b.hi), t = __fsub_rn(s, a.hi);
    const float e = __fadd_rn(__fsub_rn(a.hi, __fsub_rn(s, t)), __fsub_rn(b.hi, t));  // what s lost of a.hi + b.hi
    return Sum2{s, __fadd_rn(e, __fadd_rn(a.lo, b.lo))};
}

// 1 / sqrt(sum / n + epsilon) as two floats: a Newton step on the float result, its residual 1 - v r^2 formed from exact products.
__device__ __forceinline__ Sum2 rstd_of(Sum2 sum, float n, float epsilon)
{
    const float q = __fdiv_rn(sum.hi, n);
    const float ql = __fdiv_rn(__fadd_rn(fmaf(-q, n, sum.hi), sum.lo), n);
    const Sum2 v = add_exact(Sum2{q, ql}, Sum2{epsilon, 0.f});
    const float r = __frsqrt_rn(v.hi), s = __fmul_rn(v.hi, r), sl = fmaf(v.hi, r, -s);  // (r * r would overflow for an epsilon below 2^-128)
    const float e = fmaf(__fmul_rn(-v.lo, r), r, fmaf(-sl, r, fmaf(-s, r, 1.0f)));
    return Sum2{r, 0.5f * r * e};
}

// What a row's elements need to know: rstd and its remainder, the largest |h * gamma| (int8), NaN in rstd for a sum that is not finite.
struct RowStats {
    float rstd, rstdLo, mx, pad;
};
// Sum and (MAX) maximum over the CTA.  The warps' sums are added exactly, since every code of the row depends on the result, and the division, the square
// root and its correction take some two hundred instructions: one warp does that and the others read the outcome (in every warp it
// cost as many issue slots as the elements did: 163 us instead of 136 at [16384, 7168]).
template <bool MAX> __device__ __forceinline__ RowStats row_stats(float sum, float mx, float2* part, RowStats* stats, float n, float epsilon)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if constexpr (MAX) mx = max_nan(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) part[warp] = make_float2(sum, mx);
    __syncthreads();
    if (warp == 0) {
        const float2 p = (lane & 15) < warps ? part[lane & 15] : make_float2(0.f, 0.f);
        Sum2 all{p.x, 0.f};
        mx = p.y;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
            all = add_exact(all, Sum2{__shfl_xor_sync(0xFFFFFFFFu, all.hi, o), __shfl_xor_sync(0xFFFFFFFFu, all.lo, o)});
            if constexpr (MAX) mx = max_nan(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
        }
        const Sum2 r = rstd_of(all, n, epsilon);
        if (lane == 0) *stats = RowStats{finite_f32(all.hi) ? r.hi : __int_as_float(0x7FFFFFFF), r.lo, mx, 0.f};
    }
    __syncthreads();  // `part` may be written again; `stats` is, only behind the next row's first barrier
    return *stats;
}

// The vector kernel: a thread owns NV vectors of 8 elements of a row, spaced by the CTA's width.
template <typename T, typename G, int OUT, int NV> __global__ void __launch_bounds__(512, NV <= 2 && sizeof(T) == 2 ? 2 : 1) norm_rows_kernel(const NormArgs a)
{
    __shared__ float2 part[16];
    __shared__ __align__(16) RowStats stats;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t nvec = a.n / 8;
    const T* src = static_cast<const T*>(a.src);
    const T* res = static_cast<const T*>(a.residual);
    Vec8<G> g[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t v = i * blockDim.x + threadIdx.x;
        if (v < nvec) {
            const uint4* p = reinterpret_cast<const uint4*>(static_cast<const G*>(a.gamma) + v * 8);
#pragma unroll
            for (int j = 0; j < static_cast<int>(sizeof(G)) / 2; ++j) g[i].w[j] = __ldg(p + j);
        }
    }
    auto settled = [&](float v, uint32_t row, uint32_t col, const RowStats& st, int e) {
        if (fabsf(v) < Tie<OUT>::kLowest) return v;  // no tie there; and above it gamma * f = v / h is far from underflow
        const T x = src[row * a.ldSrc + col], r = res ? res[row * a.ldResidual + col] : x;
        const float g = to_f32<G>(static_cast<const G*>(a.gamma)[col]), up = exp2_neg(e);
        float h = to_f32<T>(x);
        if (res && sizeof(T) == 4 && a.residualOut) h = to_f32<T>(static_cast<const T*>(a.residualOut)[row * a.ldResidualOut + col]);
        else if (res && !row_sum<T>(x, r, v, g, __fmul_rn(st.rstd, up), a.residualOut == a.src, a.residualOut == a.residual, h)) return v;
        return Tie<OUT>::settle(h, g, st.rstd, st.rstdLo, up);
    };
    Vec8<T> xs[NV], rs[NV];
    auto load_row = [&](uint32_t row) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t v = i * blockDim.x + threadIdx.x;
            if (v < nvec) {
                xs[i] = load8<T>(src + row * a.ldSrc + v * 8);
                if (res) rs[i] = load8<T>(res + row * a.ldResidual + v * 8);
            }
        }
    };
    load_row(blockIdx.x);
    for (uint32_t row = blockIdx.x; row < a.m; row += gridDim.x) {
        float h[NV][8];
        float sum = 0.f, sumOdd = 0.f, mx = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t v = i * blockDim.x + threadIdx.x;
            if (v < nvec) {
                widen8<T>(xs[i], h[i]);
                if (res) {
                    float r[8];
                    widen8<T>(rs[i], r);
#pragma unroll
                    for (int j = 0; j < 8; j += 2) add2_rn(h[i][j], h[i][j + 1], r[j], r[j + 1]);
                }
#pragma unroll
                for (int j = 0; j < 8; j += 2) fma2_square(sum, sumOdd, h[i][j], h[i][j + 1]);
                // (no element is larger than the root of the thread's sum so far)
                if (a.residualOut) store8<T>(static_cast<T*>(a.residualOut) + row * a.ldResidualOut + v * 8, h[i], sizeof(T) == 4 || sum + sumOdd <= kMostSquaredOf<T>);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) h[i][j] = 0.f;
            }
        }
        if (row + gridDim.x < a.m) load_row(row + gridDim.x);  // on its way while this row is reduced and quantised
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t v = i * blockDim.x + threadIdx.x;
            if (v < nvec) {
                float gf[8];
                widen8<G>(g[i], gf);
#pragma unroll
                for (int j = 0; j < 8; j += 2) mul2_rn(h[i][j], h[i][j + 1], gf[j], gf[j + 1]);  // from here on h * gamma
                if constexpr (OUT == kOutI8) mx = max_nan(mx, max_abs8(h[i]));
            }
        }
        const RowStats st = row_stats<OUT == kOutI8>(sum + sumOdd, mx, part, &stats, static_cast<float>(a.n), a.epsilon);
        const float rstd = st.rstd;
        mx = st.mx;
        if (a.normOut) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const uint32_t v = i * blockDim.x + threadIdx.x;
                if (v < nvec) {
                    constexpr float kMost = std::is_same<T, __half>::value ? 65504.0f : 3.3895313892515355e38f;
                    float y[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) y[j] = __fmul_rn(h[i][j], rstd);
                    store8<T>(static_cast<T*>(a.normOut) + row * a.ldNormOut + v * 8, y, max_abs8(y) <= kMost);
                }
            }
        }
        if constexpr (OUT == kOutI8) {
            const float top = __fmul_rn(mx, rstd);  // the row's largest |y|; NaN with rstd
            const bool ok = finite_f32(mx) && finite_f32(top);
            if (threadIdx.x == 0)
                static_cast<float*>(a.scaleOut)[row] = !ok ? __int_as_float(0x7FFFFFFF) : mx > 0.f ? __fdiv_rn(top, 127.0f) : 1.0f;
            const I8Factor f = i8_factor(mx);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const uint32_t v = i * blockDim.x + threadIdx.x;
                if (v < nvec) {
                    if (f.pre != 1.0f) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) h[i][j] *= f.pre;
                    }
                    uint2 q;
#pragma unroll
                    for (int j = 0; j < 8; j += 2) mul2_rn(h[i][j], h[i][j + 1], f.mul, f.mul);
                    q.x = pack_i8x4_rni(h[i][0], h[i][1], h[i][2], h[i][3]);
                    q.y = pack_i8x4_rni(h[i][4], h[i][5], h[i][6], h[i][7]);
                    if (!ok) q = make_uint2(0u, 0u);
                    __stcs(reinterpret_cast<uint2*>(static_cast<int8_t*>(a.dst) + static_cast<size_t>(row) * a.n + v * 8), q);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const uint32_t v = i * blockDim.x + threadIdx.x;
                float amax = max_abs8(h[i]);
                // four neighbouring lanes hold a block; n is a multiple of 32, so they are inside the row together or not at all
                amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
                amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
                if (v < nvec) {
                    const bool ok = finite_f32(__fmul_rn(amax, rstd));
                    const int e = mx_exponent(amax, rstd, st.rstdLo, out_emax(OUT));
                    uint32_t c[4];
                    const float f = __fmul_rn(rstd, exp2_neg(e));
                    if (__builtin_expect(ok && single_factor(e, f), 1)) {
                        // f is exact: one multiplication gives what y and its scaling would
#pragma unroll
                        for (int j = 0; j < 4; ++j) mul2_rn(h[i][2 * j], h[i][2 * j + 1], f, f);
                        if constexpr (Tie<OUT>::kLooked) {
                            uint32_t least = 0xFFFFFFFFu;
                            least = Tie<OUT>::least(h[i]);
                            if (__builtin_expect(least <= Tie<OUT>::kNear, 0)) {
#pragma unroll
                                for (int j = 0; j < 8; ++j)
                                    if (Tie<OUT>::distance(h[i][j]) <= Tie<OUT>::kNear) h[i][j] = settled(h[i][j], row, v * 8 + j, st, e);
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) c[j] = mx_pair<OUT>(h[i][2 * j], h[i][2 * j + 1]);
                    } else {
                        const float up = exp2_neg(e);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            c[j] = ok ? mx_pair<OUT>(__fmul_rn(__fmul_rn(h[i][2 * j], rstd), up), __fmul_rn(__fmul_rn(h[i][2 * j + 1], rstd), up)) : 0u;
                    }
                    const size_t at = (static_cast<size_t>(row) * nvec + v);
                    if constexpr (OUT == kOutE2M1) static_cast<uint32_t*>(a.dst)[at] = c[0] | (c[1] << 8) | (c[2] << 16) | (c[3] << 24);
                    else __stcs(static_cast<uint2*>(a.dst) + at, make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16)));
                    if ((threadIdx.x & 3) == 0) static_cast<uint8_t*>(a.scaleOut)[at / 4] = static_cast<uint8_t>(ok ? e + 127 : 0xFF);
                }
            }
        }
    }
}

// int8 from widths or tensors that 16-byte vectors do not fit: a CTA holds a row as NE groups of VEC elements per thread (2 where everything is even, else 1),
// neighbouring threads neighbouring groups, all of them requested before the first is used.  The same arithmetic.  bf16 with residual and sum: [2048, 7167] 46 us
// (62 us an element at a time in two passes; [2048, 7168] takes 16 us on vectors), [4096, 1023] 14 us (20.5; 7.3), [4096, 1022] 10 us.
template <typename T, int VEC> __device__ __forceinline__ Pack<T, VEC> load_group(const T* p)
{
    if constexpr (sizeof(T) * VEC >= 4) return load_pack<T, VEC, true>(p);
    else return Pack<T, VEC>{{*p}};
}
template <typename T, typename G, int VEC, int NE> __global__ void __launch_bounds__(512, 2) norm_odd_kernel(const NormArgs a)
{
    __shared__ float2 part[16];
    __shared__ __align__(16) RowStats stats;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t row = blockIdx.x, groups = a.n / VEC;
    const T* src = static_cast<const T*>(a.src) + row * a.ldSrc;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.ldResidual : nullptr;
    const G* gamma = static_cast<const G*>(a.gamma);
    Pack<T, VEC> xs[NE], rs[NE];
    Pack<G, VEC> gs[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const uint32_t v = i * blockDim.x + threadIdx.x;
        if (v < groups) {
            xs[i] = load_group<T, VEC>(src + v * VEC);
            if (res) rs[i] = load_group<T, VEC>(res + v * VEC);
            gs[i] = load_group<G, VEC>(gamma + v * VEC);
        }
    }
    float h[NE][VEC], sum = 0.f, mx = 0.f;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const uint32_t v = i * blockDim.x + threadIdx.x;
        if (v < groups) {
            Pack<T, VEC> total;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                h[i][j] = to_f32<T>(xs[i].v[j]);
                if (res) h[i][j] = __fadd_rn(h[i][j], to_f32<T>(rs[i].v[j]));
                total.v[j] = narrow<T>(h[i][j]);
                sum = fmaf(h[i][j], h[i][j], sum);
                h[i][j] = __fmul_rn(h[i][j], to_f32<G>(gs[i].v[j]));  // from here on h * gamma
                mx = max_abs3(mx, h[i][j], 0.f);
            }
            if (a.residualOut) *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.residualOut) + row * a.ldResidualOut + v * VEC) = total;
        }
    }
    const RowStats st = row_stats<true>(sum, mx, part, &stats, static_cast<float>(a.n), a.epsilon);
    const float rstd = st.rstd, top = __fmul_rn(st.mx, rstd);
    const bool ok = finite_f32(st.mx) && finite_f32(top);
    const I8Factor f = i8_factor(st.mx);
    if (threadIdx.x == 0) static_cast<float*>(a.scaleOut)[row] = !ok ? __int_as_float(0x7FFFFFFF) : st.mx > 0.f ? __fdiv_rn(top, 127.0f) : 1.0f;
    int8_t* dst = static_cast<int8_t*>(a.dst) + static_cast<size_t>(row) * a.n;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const uint32_t v = i * blockDim.x + threadIdx.x;
        if (v >= groups) continue;
        if (a.normOut) {
            Pack<T, VEC> y;
#pragma unroll
            for (int j = 0; j < VEC; ++j) y.v[j] = narrow<T>(__fmul_rn(h[i][j], rstd));
            *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.normOut) + row * a.ldNormOut + v * VEC) = y;
        }
        float q[4] = {};
#pragma unroll
        for (int j = 0; j < VEC; ++j) q[j] = __fmul_rn(f.pre != 1.0f ? h[i][j] * f.pre : h[i][j], f.mul);
        const uint32_t codes = ok ? pack_i8x4_rni(q[0], q[1], q[2], q[3]) : 0u;
        if constexpr (VEC == 2) *reinterpret_cast<unsigned short*>(dst + v * 2) = static_cast<unsigned short>(codes);
        else dst[v] = static_cast<int8_t>(codes & 0xFFu);
    }
}

// MX codes from unaligned tensors, rows too long for registers: one CTA per row, one element per thread and step; the second
// pass computes h again from the sources (a row is in L2).  The same arithmetic.
template <typename T, typename G> __global__ void __launch_bounds__(256) norm_any_kernel(const NormArgs a)
{
    __shared__ float2 part[16];
    __shared__ __align__(16) RowStats stats;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t row = blockIdx.x;
    const T* src = static_cast<const T*>(a.src) + row * a.ldSrc;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + row * a.ldResidual : nullptr;
    const G* gamma = static_cast<const G*>(a.gamma);
    T* resOut = a.residualOut ? static_cast<T*>(a.residualOut) + row * a.ldResidualOut : nullptr;
    T* normOut = a.normOut ? static_cast<T*>(a.normOut) + row * a.ldNormOut : nullptr;
    float sum = 0.f, mx = 0.f;
    for (uint32_t c = threadIdx.x; c < a.n; c += blockDim.x) {
        const float h = res ? __fadd_rn(to_f32<T>(src[c]), to_f32<T>(res[c])) : to_f32<T>(src[c]);
        sum = fmaf(h, h, sum);
        mx = max_nan(mx, fabsf(__fmul_rn(h, to_f32<G>(gamma[c]))));
    }
    const RowStats st = row_stats<true>(sum, mx, part, &stats, static_cast<float>(a.n), a.epsilon);
    const float rstd = st.rstd;
    mx = st.mx;
    const float top = __fmul_rn(mx, rstd);
    const bool rowOk = finite_f32(mx) && finite_f32(top);
    const I8Factor f = i8_factor(mx);
    const size_t out0 = static_cast<size_t>(row) * a.n;
    if (a.out == kOutI8 && threadIdx.x == 0)
        static_cast<float*>(a.scaleOut)[row] = !rowOk ? __int_as_float(0x7FFFFFFF) : mx > 0.f ? __fdiv_rn(top, 127.0f) : 1.0f;
    // each element is read again by the thread that then overwrites it where residualOut is one of the sources
    for (uint32_t c0 = 0; c0 < a.n; c0 += blockDim.x) {
        const uint32_t c = c0 + threadIdx.x;
        float p = 0.f, h = 0.f;
        bool settles = true;  // the vector kernel's rule
        if (c < a.n) {
            const float x = to_f32<T>(src[c]), r = res ? to_f32<T>(res[c]) : 0.f;
            h = res ? __fadd_rn(x, r) : x;
            settles = !res || separable<T>(x, r, h);
            p = __fmul_rn(h, to_f32<G>(gamma[c]));
            if (resOut) resOut[c] = narrow<T>(h);
            if (normOut) normOut[c] = narrow<T>(__fmul_rn(p, rstd));
        }
        if (a.out == kOutI8) {
            if (c < a.n)
                static_cast<int8_t*>(a.dst)[out0 + c] =
                    static_cast<int8_t>(rowOk ? f32_to_i8_sat(__fmul_rn(f.pre != 1.0f ? p * f.pre : p, f.mul), kRoundRint) : 0);
        } else {  // n is a multiple of 32: a warp holds one block, whole or not at all
            const float y = __fmul_rn(p, rstd);
            float amax = fabsf(p);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
            const bool ok = finite_f32(__fmul_rn(amax, rstd));
            const int e = mx_exponent(amax, rstd, st.rstdLo, out_emax(a.out));
            float v = __fmul_rn(y, exp2_neg(e));
            if (ok && single_factor(e, __fmul_rn(rstd, exp2_neg(e))) && settles && c < a.n) {
                if (a.out == kOutE4M3 && Tie<kOutE4M3>::distance(v) <= Tie<kOutE4M3>::kNear)
                    v = Tie<kOutE4M3>::settle(h, to_f32<G>(gamma[c]), rstd, st.rstdLo, exp2_neg(e));
                if (a.out == kOutE5M2 && Tie<kOutE5M2>::distance(v) <= Tie<kOutE5M2>::kNear)
                    v = Tie<kOutE5M2>::settle(h, to_f32<G>(gamma[c]), rstd, st.rstdLo, exp2_neg(e));
            }
            const float next = __shfl_down_sync(0xFFFFFFFFu, v, 1);
            if (c < a.n) {
                if (a.out == kOutE2M1) {
                    if ((c & 1) == 0) static_cast<uint8_t*>(a.dst)[(out0 + c) / 2] = static_cast<uint8_t>(ok ? mx_pair<kOutE2M1>(v, next) : 0u);
                } else {
                    const uint32_t code = a.out == kOutE4M3 ? mx_pair<kOutE4M3>(v, 0.f) : mx_pair<kOutE5M2>(v, 0.f);
                    static_cast<uint8_t*>(a.dst)[out0 + c] = static_cast<uint8_t>(ok ? code & 0xFFu : 0u);
                }
                if ((c & 31) == 0) static_cast<uint8_t*>(a.scaleOut)[(out0 + c) / 32] = static_cast<uint8_t>(ok ? e + 127 : 0xFF);
            }
        }
    }
}

template <typename K> cudaError_t launch_norm(K kernel, unsigned grid, unsigned block, cudaStream_t st, const NormArgs& a)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(block, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

constexpr uint32_t kNormThreads = 512, kNormMaxVectors = 4;  // the longest row the vector kernel holds: 512 * 4 * 8 elements

template <typename T, typename G, int OUT> cudaError_t launch_norm_rows(const NormArgs& a, cudaStream_t st)
{
    const uint32_t nvec = a.n / 8;
    uint32_t nv = 1;
    while (nv < kNormMaxVectors && (nvec + nv - 1) / nv > kNormThreads) nv *= 2;
    const unsigned block = ((nvec + nv - 1) / nv + 31) / 32 * 32;
    // About 1280 threads per SM, each CTA walking over its rows with the next one on its way.  Measured: bf16 [16384, 7168] to e4m3 (448
    // threads) 199 / 141 / 170 us with 1 / 2 / 3 CTAs per SM; half [1031, 5120] to int8 (320 threads) 8.2 / 8.1 / 5.6 / 5.5 / 5.6 us with
    // 1 to 5.  Rows above 8192 elements need 128 registers a thread, so that one CTA is all an SM holds: [2048, 16384] to int8 38 us = 0.94 of the
    // copy rate, to e4m3 45 us = 0.81.
    const unsigned perSm = nv >= 4 ? 1u : std::max(1u, 1280u / block);
    const unsigned grid = std::min<uint64_t>(a.m, static_cast<uint64_t>(sm_count()) * perSm);
    if (nv == 1) return launch_norm(norm_rows_kernel<T, G, OUT, 1>, grid, block, st, a);
    if (nv == 2) return launch_norm(norm_rows_kernel<T, G, OUT, 2>, grid, block, st, a);
    return launch_norm(norm_rows_kernel<T, G, OUT, 4>, grid, block, st, a);
}

template <typename T, typename G, int VEC> cudaError_t launch_norm_odd(const NormArgs& a, cudaStream_t st)
{
    const uint32_t groups = (a.n + VEC - 1) / VEC;
    if (groups <= 512 * 4) return launch_norm(norm_odd_kernel<T, G, VEC, 4>, a.m, std::max((groups + 3) / 4 + 31, 32u) / 32 * 32, st, a);
    if (groups <= 512 * 8) return launch_norm(norm_odd_kernel<T, G, VEC, 8>, a.m, (groups + 7) / 8 / 32 * 32 + 32 <= 512 ? (groups + 7) / 8 / 32 * 32 + 32 : 512, st, a);
    if constexpr (VEC == 1) return launch_norm(norm_odd_kernel<T, G, 1, 16>, a.m, 512, st, a);
    else return cudaErrorInvalidValue;  // (the caller's limit is 512 * 8 pairs)
}

template <typename T, typename G> cudaError_t launch_norm_typed(const NormArgs& a, bool vec, bool even, cudaStream_t st)
{
    if (!vec && a.out == kOutI8 && a.n <= 512 * 16) return even ? launch_norm_odd<T, G, 2>(a, st) : launch_norm_odd<T, G, 1>(a, st);
    if (!vec) return launch_norm(norm_any_kernel<T, G>, a.m, 256, st, a);
    switch (a.out) {
        case kOutI8: return launch_norm_rows<T, G, kOutI8>(a, st);
        case kOutE4M3: return launch_norm_rows<T, G, kOutE4M3>(a, st);
        case kOutE5M2: return launch_norm_rows<T, G, kOutE5M2>(a, st);
        default: return launch_norm_rows<T, G, kOutE2M1>(a, st);
    }
}

}  // namespace
}  // namespace ascq

extern "C" ascq_status ascq_residual_rms_norm_quant(void* dst, ascq_dtype dstT, void* scaleOut, void* residualOut, void* normOut, const void* src,
                                                    const void* residual, const void* gamma, ascq_dtype srcT, ascq_dtype gammaT,
                                                    const ascq_rms_norm_param* p, void* stream)
{
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (!p) return fail(ASCQ_ERR_INVALID_ARG, "param must not be NULL");
    auto is_float = [](ascq_dtype t) { return t == ASCQ_DT_F16 || t == ASCQ_DT_BF16 || t == ASCQ_DT_F32; };
    if (!is_float(srcT)) return fail(ASCQ_ERR_UNSUPPORTED, "src dtype must be half, bfloat16_t or float");
    if (gammaT != srcT && gammaT != ASCQ_DT_F32) return fail(ASCQ_ERR_UNSUPPORTED, "gamma must have src's dtype or float");
    NormArgs a{};
    switch (dstT) {
        case ASCQ_DT_I8: a.out = kOutI8; break;
        case ASCQ_DT_FP8_E4M3: a.out = kOutE4M3; break;
        case ASCQ_DT_FP8_E5M2: a.out = kOutE5M2; break;
        case ASCQ_DT_FP4X2_E2M1: a.out = kOutE2M1; break;
        default: return fail(ASCQ_ERR_UNSUPPORTED, "dst dtype %d is not built (int8, fp8_e4m3, fp8_e5m2 and fp4x2_e2m1 are)", static_cast<int>(dstT));
    }
    if (!(p->epsilon > 0.f) || p->epsilon > 3.4028234663852886e38f) return fail(ASCQ_ERR_INVALID_ARG, "epsilon must be positive and finite");
    if (a.out != kOutI8 && p->n % 32 != 0) return fail(ASCQ_ERR_INVALID_ARG, "n is %u, which must be a multiple of the MX block size 32", p->n);
    if (p->m > 0x7FFFFFFFu || p->n > 0x7FFFFFFFu) return fail(ASCQ_ERR_INVALID_ARG, "m and n must be below 2^31");
    auto pitch = [&](int64_t ld) { return ld == 0 ? static_cast<int64_t>(p->n) : ld; };
    a.ldSrc = pitch(p->ldSrc);
    a.ldResidual = pitch(p->ldResidual);
    a.ldResidualOut = pitch(p->ldResidualOut);
    a.ldNormOut = pitch(p->ldNormOut);
    for (int64_t ld : {a.ldSrc, a.ldResidual, a.ldResidualOut, a.ldNormOut})
        if (ld < static_cast<int64_t>(p->n)) return fail(ASCQ_ERR_INVALID_ARG, "a row pitch is %lld, which must be 0 or at least n = %u", static_cast<long long>(ld), p->n);
    if (p->m == 0 || p->n == 0) return ASCQ_OK;
    if (!dst || !scaleOut || !src || !gamma) return fail(ASCQ_ERR_INVALID_ARG, "dst, scaleOut, src and gamma must not be NULL");

    const int es = dtype_size(srcT);
    auto bad = [&](const void* q, uintptr_t by) { return (reinterpret_cast<uintptr_t>(q) & (by - 1)) != 0; };
    if (bad(src, es) || bad(residual, es) || bad(residualOut, es) || bad(normOut, es) || bad(gamma, dtype_size(gammaT)) || (a.out == kOutI8 && bad(scaleOut, 4)))
        return fail(ASCQ_ERR_ALIGNMENT, "a tensor is not aligned to its element type");
    // outputs overlap nothing, except that residualOut may be src or residual itself (the same matrix with the same pitch)
    const size_t elems = static_cast<size_t>(p->m) * p->n;
    const size_t width = static_cast<size_t>(p->n) * es, rows = p->m;
    const PitchedSpan in[3] = {{src, rows, width, static_cast<size_t>(a.ldSrc) * es},
                               {residual, rows, width, static_cast<size_t>(a.ldResidual) * es},
                               {gamma, 1, static_cast<size_t>(p->n) * dtype_size(gammaT), 0}};
    const PitchedSpan out[4] = {{residualOut, rows, width, static_cast<size_t>(a.ldResidualOut) * es},
                                {normOut, rows, width, static_cast<size_t>(a.ldNormOut) * es},
                                {dst, 1, a.out == kOutE2M1 ? elems / 2 : elems, 0},
                                {scaleOut, 1, a.out == kOutI8 ? rows * 4 : elems / 32, 0}};
    for (int i = 0; i < 4; ++i) {
        for (int j = 0; j < 3; ++j) {
            const bool same = i == 0 && j < 2 && out[i].p == in[j].p && out[i].pitch == in[j].pitch;
            if (!same && spans_overlap(out[i], in[j]))
                return fail(ASCQ_ERR_INVALID_ARG, "an output overlaps an input (only residualOut may be src or residual, with the same pitch)");
        }
        for (int j = 0; j < i; ++j)
            if (spans_overlap(out[i], out[j])) return fail(ASCQ_ERR_INVALID_ARG, "two outputs overlap");
    }

    a.dst = dst; a.scaleOut = scaleOut; a.residualOut = residualOut; a.normOut = normOut;
    a.src = src; a.residual = residual; a.gamma = gamma;
    a.m = p->m; a.n = p->n; a.epsilon = p->epsilon;
    // The vector kernel wants 16-byte vectors of 8 elements everywhere (codes: 8 or 4 bytes) and a row that fits its registers.
    const bool vec = p->n % 8 == 0 && p->n / 8 <= kNormThreads * kNormMaxVectors && !bad(src, 16) && !bad(residual, 16) && !bad(residualOut, 16) &&
                     !bad(normOut, 16) && !bad(gamma, 16) && !bad(dst, a.out == kOutE2M1 ? 4 : 8) && a.ldSrc * es % 16 == 0 &&
                     (!residual || a.ldResidual * es % 16 == 0) && (!residualOut || a.ldResidualOut * es % 16 == 0) && (!normOut || a.ldNormOut * es % 16 == 0);
    const int e2 = 2 * es;  // pairs of elements, everywhere
    const bool even = p->n % 2 == 0 && !bad(src, e2) && !bad(residual, e2) && !bad(residualOut, e2) && !bad(normOut, e2) && !bad(gamma, 2 * dtype_size(gammaT)) &&
                      !bad(dst, 2) && a.ldSrc % 2 == 0 && (!residual || a.ldResidual % 2 == 0) && (!residualOut || a.ldResidualOut % 2 == 0) &&
                      (!normOut || a.ldNormOut % 2 == 0);
    cudaError_t rc;
    if (srcT == ASCQ_DT_F16) rc = gammaT == srcT ? launch_norm_typed<__half, __half>(a, vec, even, st) : launch_norm_typed<__half, float>(a, vec, even, st);
    else if (srcT == ASCQ_DT_BF16) rc = gammaT == srcT ? launch_norm_typed<__nv_bfloat16, __nv_bfloat16>(a, vec, even, st) : launch_norm_typed<__nv_bfloat16, float>(a, vec, even, st);
    else rc = launch_norm_typed<float, float>(a, vec, even, st);
    ASCQ_CUDA_CHECK(rc);
    return ASCQ_OK;
}
