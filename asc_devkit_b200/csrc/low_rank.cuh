// What the two forms of ascq_low_rank_add share: the call's arguments, the walk from a tile's number to its tokens, and the inner
// products' split into two 16-bit terms.
#ifndef ASCQ_LOW_RANK_CUH_
#define ASCQ_LOW_RANK_CUH_

#include "elementwise.cuh"

namespace ascq {

struct LowRankArgs {
    const void *x, *a, *b, *base;  // base may be null (0)
    void* dst;
    const void* ids;
    const float* scale;            // [L] or null (1)
    const int64_t* counts;         // sorted: tokens per adapter, L + 1 entries (the last: tokens without one); else null
    const int32_t* order;          // sorted: tokens in order of adapter
    int64_t ldX, ldBase, ldDst;
    int M, N, K, r, L, ids64;
};

// low_rank_long.cu: tiles of 128 tokens, for adapters with enough tokens to fill them
struct LowRankScratch {
    void* tiles;   // int4 per tile
    void* v;       // split inner products
    float* unit;   // [M]
    int stopA, stopB;  // a CTA loads no chunk of A (first launch), no block of B (second) from this number on; set by low_rank_long
};
constexpr int kLongTile = 128;
size_t low_rank_long_tiles_bytes(int64_t tiles);
size_t low_rank_long_inner_bytes(int M, int r);
ascq_status low_rank_long(const LowRankArgs& p, bool half, const LowRankScratch& o, unsigned tiles, ::CUstream_st* st);

namespace {

// Warp 0 walks the token counts of the adapters (`count(e)`), 32 at a time, to the tile with the given number: its adapter,
// the number of tokens before the tile inside the adapter, and before the adapter.
template <int SIZE, typename F> __device__ __forceinline__ void find_tile(int tile, int keys, F count, int* out)
{
    const int lane = threadIdx.x & 31;
    int tilesBefore = 0, tokensBefore = 0;
    if (lane == 0) out[0] = -1;
    __syncwarp();
    for (int e0 = 0; e0 < keys; e0 += 32) {
        const int n = e0 + lane < keys ? count(e0 + lane) : 0;
        const int tiles = (n + SIZE - 1) / SIZE;
        int inclTiles = tiles, inclTokens = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xFFFFFFFFu, inclTiles, o), v = __shfl_up_sync(0xFFFFFFFFu, inclTokens, o);
            if (lane >= o) {
                inclTiles += u;
                inclTokens += v;
            }
        }
        const int first = tilesBefore + inclTiles - tiles;
        if (tile >= first && tile < first + tiles) {
            const int at = (tile - first) * SIZE;
            out[0] = e0 + lane;
            out[1] = n - at < SIZE ? n - at : SIZE;
            out[2] = at;
            out[3] = tokensBefore + inclTokens - n + at;
        }
        tilesBefore += __shfl_sync(0xFFFFFFFFu, inclTiles, 31);
        tokensBefore += __shfl_sync(0xFFFFFFFFu, inclTokens, 31);
        if (tilesBefore > tile) break;
    }
    __syncwarp();
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v)
{
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&v));
    else return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}

template <typename T> __device__ __forceinline__ uint32_t pack_sat(float lo, float hi)
{
    if constexpr (std::is_same<T, __half>::value) return pack_f16x2_sat(lo, hi);
    else return pack_bf16x2_sat(lo, hi);
}
// eight floats -> eight 16-bit values, finite overflow saturating: one test for all of them
template <typename T> __device__ __forceinline__ uint4 pack8_sat(const float (&f)[8])
{
    constexpr float kMost = std::is_same<T, __half>::value ? 65504.0f : 3.3895313892515355e38f;
    uint32_t r[4];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[i] = pack2<T>(f[2 * i], f[2 * i + 1]);
        asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(top) : "f"(top), "f"(f[2 * i]), "f"(f[2 * i + 1]));
    }
    if (__builtin_expect(!(top <= kMost), 0)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = pack_sat<T>(f[2 * i], f[2 * i + 1]);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}
__device__ __forceinline__ void st_cluster_v4(uint32_t addr, uint4 v)
{
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// A row whose largest magnitude is `top` is multiplied by 2^-shift before the split and its products by 2^shift.
// half: to [512, 1024), clear of its range's end and of its subnormals (|B| <= 65504 keeps the sums far below fp32's end); rows that are zero,
// subnormal or not finite stay as they are.
// bfloat16 has fp32's exponents: the products are formed where the formula has them, so that they overflow only where it does.  Only a row
// next to fp32's end, whose cast would be an infinity, is halved, and one so small that the later terms would be subnormal goes up by 2^32.
template <typename T> __device__ __forceinline__ int range_shift(float top)
{
    const int ex = static_cast<int>(__float_as_uint(top) >> 23);
    if constexpr (std::is_same<T, __half>::value) return ex == 0 || ex == 255 ? 0 : min(max(ex - 136, -126), 126);
    else return ex == 254 ? 1 : ex < 32 ? -32 : 0;
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
// Beside an infinity a row keeps its range; what is finite in it must not become an infinity of the other sign.  (Only rows with a `top` that
// is not finite come here: casts that saturate, for every row, cost 9 us of 62 at 8192 tokens.)
template <typename T> __device__ __forceinline__ float inside_range(float v)
{
    constexpr float kMost = std::is_same<T, __half>::value ? 65504.0f : 3.3895313892515355e38f;
    return fabsf(v) <= 3.4028234663852886e38f ? fminf(fmaxf(v, -kMost), kMost) : v;
}
// v as two 16-bit terms: x = cast(v), y = cast(v - x); 0 for the second where the first is not finite
template <typename T> __device__ __forceinline__ uint2 split16(float v)
{
    uint2 r;
    r.x = pack2<T>(v, 0.f) & 0xFFFFu;
    const float back = unpack2<T>(r.x).x;
    r.y = fabsf(back) <= 3.4028234663852886e38f ? pack2<T>(v - back, 0.f) & 0xFFFFu : 0u;
    return r;
}

}  // namespace
}  // namespace ascq
#endif  // ASCQ_LOW_RANK_CUH_
