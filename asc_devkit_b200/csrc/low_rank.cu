// Low-rank adapters of many requests at once, added to the result of a shared projection:
//   dst[t] = cast(base[t] + scale[a] * (x[t] . A[a]^T) . B[a]^T),  a = adapterIds[t];   x [M, K], A [L, r, K], B [L, N, r]
// A token whose number is outside [0, L) has no adapter: dst[t] = base[t].
//
// What bounds it: x, base and dst cross HBM once (2 (K + 2 N) bytes a token), each used adapter once (2 r (K + N) bytes); with ranks up to
// 128 the products stay below what the tensor cores do in that time.  So the tokens are grouped by adapter -- a tile is up to 16 tokens
// of one adapter -- and both products of a tile run in one launch: a cluster of CTAs splits K for the first, adds its
// partial sums through distributed shared memory, and splits N for the second.  The [16, r] inner product never leaves the SMs.
//
// Both operands of the MMAs come straight from global memory: a dot product does not care in which order k is visited, so a
// lane's 16 consecutive bytes of a row serve as the fragments of two m16n8k16 MMAs.
//
// The inner product is a sum in fp32; for the second product it is split into two 16-bit terms, hi = cast(v), lo = cast(v - hi), after
// each token's row was brought to [512, 1024) by a power of two (so that neither fp16's range nor its subnormals matter).  What the split drops is below
// 2^-16 (bf16) or 2^-22 (fp16) of the row's largest value: the result carries one visible rounding, the one to dst's type.
#include "elementwise.cuh"
#include "experts.cuh"
#include "sm100_ptx.cuh"

using namespace ascq;
using namespace ascq::ptx;

namespace ascq {
namespace {

constexpr int kTile = 16;         // tokens of one adapter that share a tile
constexpr int kWarps = 8;
constexpr int kInlineTokens = 1024;  // up to here every CTA finds its tile in the adapter numbers itself; beyond, they are sorted first

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

__device__ __forceinline__ int adapter_of(const LowRankArgs& p, int t)
{
    if (p.ids64) {
        const int64_t v = static_cast<const int64_t*>(p.ids)[t];
        return v >= 0 && v < p.L ? static_cast<int>(v) : p.L;
    }
    const int32_t v = static_cast<const int32_t*>(p.ids)[t];
    return v >= 0 && v < p.L ? v : p.L;
}

struct Tile {
    int adapter;  // L: none; -1: there is no such tile
    int tokens;
};

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

// Writes the tile's tokens into `list` (kTile entries, unused ones 0).  `work`: L + 1 + kWarps ints of scratch.
__device__ __forceinline__ Tile take_tile(const LowRankArgs& p, int tile, int* list, int* found, int* work)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, keys = p.L + 1;
    if (threadIdx.x < kTile) list[threadIdx.x] = 0;
    if (p.counts) {
        if (warp == 0) find_tile<kTile>(tile, keys, [&](int e) { return static_cast<int>(p.counts[e]); }, found);
        __syncthreads();
        const Tile t{found[0], found[0] < 0 ? 0 : found[1]};
        if (static_cast<int>(threadIdx.x) < t.tokens) list[threadIdx.x] = p.order[found[3] + threadIdx.x];
        __syncthreads();
        return t;
    }
    int* hist = work;
    int* perWarp = work + keys;
    for (int e = threadIdx.x; e < keys; e += blockDim.x) hist[e] = 0;
    __syncthreads();
    for (int t = threadIdx.x; t < p.M; t += blockDim.x) atomicAdd(&hist[adapter_of(p, t)], 1);  // counts: the order does not show
    __syncthreads();
    if (warp == 0) find_tile<kTile>(tile, keys, [&](int e) { return hist[e]; }, found);
    __syncthreads();
    const Tile t{found[0], found[0] < 0 ? 0 : found[1]};
    if (t.adapter < 0) return t;
    // the adapter's tokens in ascending order: each warp owns a contiguous run of them
    const int run = (p.M + 32 * kWarps - 1) / (32 * kWarps) * 32, begin = warp * run, end = begin + run < p.M ? begin + run : p.M;
    int mine = 0;
    for (int s = begin; s < end; s += 32) mine += __popc(__ballot_sync(0xFFFFFFFFu, s + lane < end && adapter_of(p, s + lane) == t.adapter));
    if (lane == 0) perWarp[warp] = mine;
    __syncthreads();
    int at = -found[2];
    for (int w = 0; w < warp; ++w) at += perWarp[w];
    for (int s = begin; s < end && at < kTile; s += 32) {
        const bool hit = s + lane < end && adapter_of(p, s + lane) == t.adapter;
        const uint32_t all = __ballot_sync(0xFFFFFFFFu, hit);
        const int i = at + __popc(all & ((1u << lane) - 1u));
        if (hit && i >= 0 && i < kTile) list[i] = s + lane;
        at += __popc(all);
    }
    __syncthreads();
    return t;
}

template <typename T> __device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr)
{
    float f;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(addr) : "memory");
    return f;
}
// Exponent of the power of two that brings a row whose largest magnitude is `top` to [512, 1024); rows that are zero, subnormal or
// not finite stay as they are.
__device__ __forceinline__ int range_shift(float top)
{
    const int ex = static_cast<int>(__float_as_uint(top) >> 23);
    return ex == 0 || ex == 255 ? 0 : min(max(ex - 136, -126), 126);
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
// v as two 16-bit terms: x = cast(v), y = cast(v - x); 0 for the second where the first is not finite
template <typename T> __device__ __forceinline__ uint2 split16(float v)
{
    uint2 r;
    r.x = pack2<T>(v, 0.f) & 0xFFFFu;
    const float back = unpack2<T>(r.x).x;
    r.y = fabsf(back) <= 3.4028234663852886e38f ? pack2<T>(v - back, 0.f) & 0xFFFFu : 0u;
    return r;
}

__host__ __device__ constexpr int padded_rank(int nb) { return nb * 8 < 32 ? 32 : nb * 8; }  // whole 32-wide k steps of the second product
// float words of dynamic shared memory: the warps' sums (the tile finder's scratch before that), this CTA's sum, and the split result
__host__ __device__ constexpr int red_words(int nb, int L)
{
    const int sums = kWarps * kTile * nb * 8, finder = (L + 1 + kWarps + 3) / 4 * 4;
    return sums > finder ? sums : finder;
}
__host__ __device__ constexpr int part_words(int nb) { return kTile * nb * 8; }
__host__ __device__ constexpr int split_words(int nb) { return kTile * (padded_rank(nb) / 2 + 4) * 2; }

// NB: blocks of 8 of the rank (r <= 8 NB)
template <typename T, int NB> __global__ void __launch_bounds__(32 * kWarps) low_rank_kernel(const LowRankArgs p, int clusterCtas)
{
    extern __shared__ float smem[];
    __shared__ int list[kTile], found[4];
    __shared__ float unit[kTile];  // the power of two that brings a token's row back
    constexpr int R = NB * 8, KS = padded_rank(NB) / 32, VP = padded_rank(NB) / 2 + 4;  // VP: row pitch of the split result in words
    float* red = smem;
    float* part = red + red_words(NB, p.L);
    uint32_t* hi = reinterpret_cast<uint32_t*>(part + part_words(NB));
    uint32_t* lo = hi + kTile * VP;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int rank = blockIdx.x % clusterCtas;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Tile tile = take_tile(p, blockIdx.x / clusterCtas, list, found, reinterpret_cast<int*>(red));
    if (tile.adapter < 0) return;  // the same for every CTA of the cluster
    const bool has = tile.adapter < p.L;
    const int units = clusterCtas * kWarps, unitIdx = rank * kWarps + warp;

    if (has) {
        // ---- inner product: this warp's chunks of 32 k
        const T* a = static_cast<const T*>(p.a) + static_cast<size_t>(tile.adapter) * p.r * p.K;
        const T* x0 = static_cast<const T*>(p.x) + static_cast<int64_t>(list[g]) * p.ldX;
        const T* x1 = static_cast<const T*>(p.x) + static_cast<int64_t>(list[g + 8]) * p.ldX;
        const bool in0 = g < tile.tokens, in1 = g + 8 < tile.tokens;
        float acc[NB][4] = {};
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 2
        for (int k = unitIdx * 32 + c * 8; k - c * 8 < p.K; k += units * 32) {
            const bool kIn = k < p.K;
            const uint4 u0 = in0 && kIn ? __ldg(reinterpret_cast<const uint4*>(x0 + k)) : zero;
            const uint4 u1 = in1 && kIn ? __ldg(reinterpret_cast<const uint4*>(x1 + k)) : zero;
            uint4 w[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n)
                w[n] = kIn && n * 8 + g < p.r ? __ldg(reinterpret_cast<const uint4*>(a + static_cast<size_t>(n * 8 + g) * p.K + k)) : zero;
            const uint32_t f0[4] = {u0.x, u1.x, u0.y, u1.y}, f1[4] = {u0.z, u1.z, u0.w, u1.w};
#pragma unroll
            for (int n = 0; n < NB; ++n) mma16816<T>(acc[n], f0, w[n].x, w[n].y);
#pragma unroll
            for (int n = 0; n < NB; ++n) mma16816<T>(acc[n], f1, w[n].z, w[n].w);
        }
        __syncthreads();  // the tile finder's scratch is read no more
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float* to = red + warp * kTile * R + n * 8 + 2 * c;
            to[g * R] = acc[n][0];
            to[g * R + 1] = acc[n][1];
            to[(g + 8) * R] = acc[n][2];
            to[(g + 8) * R + 1] = acc[n][3];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < kTile * R; i += blockDim.x) {
            float s = red[i];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) s += red[w * kTile * R + i];
            part[i] = s;
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        // ---- the cluster's sum, scaled, brought to a common range per token and split; a warp takes two tokens
        const float scale = p.scale ? p.scale[tile.adapter] : 1.0f;
        for (int row = warp; row < kTile; row += kWarps) {
            float v[(R + 31) / 32];
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < (R + 31) / 32; ++i) {
                const int col = lane + 32 * i;
                v[i] = 0.f;
                if (col < R) {
                    const uint32_t at = smem_u32(part + row * R + col);
                    for (int q = 0; q < clusterCtas; ++q) v[i] += ld_cluster_f32(mapa_u32(at, q));
                    v[i] *= scale;
                }
                top = fmaxf(top, fabsf(v[i]));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            const int shift = range_shift(top);
            const float down = exp2_int(-shift);
            if (lane == 0) unit[row] = exp2_int(shift);
            unsigned short* h = reinterpret_cast<unsigned short*>(hi + row * VP);
            unsigned short* l = reinterpret_cast<unsigned short*>(lo + row * VP);
            for (int col = lane; col < padded_rank(NB); col += 32) {
                const uint2 two = split16<T>(col < R ? v[col / 32] * down : 0.f);
                h[col] = static_cast<unsigned short>(two.x);
                l[col] = static_cast<unsigned short>(two.y);
            }
        }
        __syncthreads();
        cluster_arrive();  // this CTA has read the others' sums; the wait is at the end
    }

    // ---- second product: this warp's groups of 32 columns; lane c of a row owns 8 consecutive ones
    uint32_t fh[KS][2][4], fl[KS][2][4];
    float back0 = 0.f, back1 = 0.f;
    if (has) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const uint4 h0 = *reinterpret_cast<const uint4*>(hi + g * VP + s * 16 + c * 4), h1 = *reinterpret_cast<const uint4*>(hi + (g + 8) * VP + s * 16 + c * 4);
            const uint4 l0 = *reinterpret_cast<const uint4*>(lo + g * VP + s * 16 + c * 4), l1 = *reinterpret_cast<const uint4*>(lo + (g + 8) * VP + s * 16 + c * 4);
            fh[s][0][0] = h0.x; fh[s][0][1] = h1.x; fh[s][0][2] = h0.y; fh[s][0][3] = h1.y;
            fh[s][1][0] = h0.z; fh[s][1][1] = h1.z; fh[s][1][2] = h0.w; fh[s][1][3] = h1.w;
            fl[s][0][0] = l0.x; fl[s][0][1] = l1.x; fl[s][0][2] = l0.y; fl[s][0][3] = l1.y;
            fl[s][1][0] = l0.z; fl[s][1][1] = l1.z; fl[s][1][2] = l0.w; fl[s][1][3] = l1.w;
        }
        back0 = unit[g];
        back1 = unit[g + 8];
    }
    const T* b = static_cast<const T*>(p.b) + static_cast<size_t>(has ? tile.adapter : 0) * p.N * p.r;
    for (int n0 = unitIdx * 32; n0 < p.N; n0 += units * 32) {
        float acc[4][4] = {};
        const int col = n0 + c * 8;
        const bool nIn = col < p.N;  // N is a multiple of 8
        uint4 y0 = make_uint4(0u, 0u, 0u, 0u), y1 = y0;
        if (p.base && nIn) {
            if (g < tile.tokens) y0 = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.base) + static_cast<int64_t>(list[g]) * p.ldBase + col);
            if (g + 8 < tile.tokens) y1 = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.base) + static_cast<int64_t>(list[g + 8]) * p.ldBase + col);
        }
        if (has) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // column g of MMA j is column 8 (g / 2) + 2 j + (g & 1) of the group, so that accumulators 2c, 2c + 1 of the four MMAs are a
                // lane's 8 neighbours
                const int n = n0 + 8 * (g >> 1) + 2 * j + (g & 1);
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const int k = s * 32 + c * 8;
                    const uint4 w = n < p.N && k < p.r ? __ldg(reinterpret_cast<const uint4*>(b + static_cast<size_t>(n) * p.r + k)) : make_uint4(0u, 0u, 0u, 0u);
                    mma16816<T>(acc[j], fh[s][0], w.x, w.y);
                    mma16816<T>(acc[j], fh[s][1], w.z, w.w);
                    mma16816<T>(acc[j], fl[s][0], w.x, w.y);
                    mma16816<T>(acc[j], fl[s][1], w.z, w.w);
                }
            }
        }
        if (!nIn) continue;
        uint32_t o0[4], o1[4];
        const uint32_t i0[4] = {y0.x, y0.y, y0.z, y0.w}, i1[4] = {y1.x, y1.y, y1.z, y1.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 v0 = unpack2<T>(i0[j]), v1 = unpack2<T>(i1[j]);
            const float r0 = fmaf(acc[j][0], back0, v0.x), r1 = fmaf(acc[j][1], back0, v0.y), r2 = fmaf(acc[j][2], back1, v1.x), r3 = fmaf(acc[j][3], back1, v1.y);
            o0[j] = has ? pack_sat<T>(r0, r1) : i0[j];
            o1[j] = has ? pack_sat<T>(r2, r3) : i1[j];
        }
        if (g < tile.tokens) *reinterpret_cast<uint4*>(static_cast<T*>(p.dst) + static_cast<int64_t>(list[g]) * p.ldDst + col) = make_uint4(o0[0], o0[1], o0[2], o0[3]);
        if (g + 8 < tile.tokens)
            *reinterpret_cast<uint4*>(static_cast<T*>(p.dst) + static_cast<int64_t>(list[g + 8]) * p.ldDst + col) = make_uint4(o1[0], o1[1], o1[2], o1[3]);
    }
    if (has) {
        __syncwarp();
        cluster_wait();
    }
}

// ---- longer runs of tokens per adapter: two launches over tiles of 64 tokens -----------------------------------------------------
// The first forms the inner products of a tile (a cluster splits K and adds up through distributed shared memory) and leaves
// them, split in two, in the workspace in sorted order; the second adds B's product to base for a tile and a range of columns.  A and B are then
// read from L2 once per 64 tokens, and each launch moves one side of the HBM traffic: x in the first, base and dst in the second.
constexpr int kLong = 64;       // tokens of a tile
constexpr int kLongWarps = 4;
constexpr int kStages = 4;      // chunks of 64 k of A in shared memory, and of x in registers
constexpr int kColumns = 512;   // columns of a CTA of the second launch

__host__ __device__ constexpr int inner_pitch(int nb) { return nb * 8 < 32 ? 32 : nb * 8; }  // elements of the hi (or lo) part of a row

struct InnerOut {
    int4* tiles;      // adapter (-1: no such tile), first sorted token, tokens
    void* v;          // [M][2][inner_pitch] of T
    float* unit;      // [M]
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool in)
{
    const int bytes = in ? 16 : 0;  // the rest of the 16 bytes is filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Four warps: two halves of the tile's tokens, times two halves of each chunk's k (NB <= 8) or of the rank (NB = 16).  x goes
// from global memory to fragments directly (each element is used by one warp, for NB = 16 by two); A goes through shared memory, where a row of a
// chunk is 128 bytes and its 16-byte pieces are exchanged between the halves on odd rows, so that 8 lanes of a 16-byte
// read cover all banks.
template <typename T, int NB> __global__ void __launch_bounds__(32 * kLongWarps) low_rank_inner_kernel(const LowRankArgs p, const InnerOut o, int clusterCtas)
{
    constexpr int R = NB * 8, WR = NB > 8 ? 2 : 1, WK = 2 / WR, NBW = NB / WR, STEPS = 2 / WK, DEPTH = kStages / STEPS;
    constexpr int kStageBytes = R * 128, kPitch = R + 8;  // kPitch: floats of a row of the partial sums
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ int found[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int wm = warp & 1, wk = WK == 2 ? warp >> 1 : 0, wr = WR == 2 ? warp >> 1 : 0;
    const int tileIdx = blockIdx.x / clusterCtas, rank = blockIdx.x % clusterCtas;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == 0) find_tile<kLong>(tileIdx, p.L + 1, [&](int e) { return static_cast<int>(p.counts[e]); }, found);
    __syncthreads();
    const int adapter = found[0], tokens = adapter < 0 ? 0 : found[1], start = adapter < 0 ? 0 : found[3];
    if (rank == 0 && threadIdx.x == 0) o.tiles[tileIdx] = make_int4(adapter, start, tokens, 0);
    if (adapter < 0 || adapter >= p.L) return;  // the same for every CTA of the cluster

    const T* a = static_cast<const T*>(p.a) + static_cast<size_t>(adapter) * p.r * p.K;
    const T* x[4];
    bool in[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = wm * 32 + g + 8 * i;
        in[i] = row < tokens;
        x[i] = static_cast<const T*>(p.x) + static_cast<int64_t>(in[i] ? p.order[start + row] : 0) * p.ldX;
    }
    const int chunks = (p.K + 63) / 64, per = (chunks + clusterCtas - 1) / clusterCtas;
    const int first = rank * per, last = min(first + per, chunks);
    const uint32_t base = smem_u32(ring);
    auto load_a = [&](int ck) {
        const uint32_t slot = base + (ck - first) % kStages * kStageBytes;
#pragma unroll
        for (int i = 0; i < (NB * 64 + 127) / 128; ++i) {
            const int idx = i * 128 + threadIdx.x, row = idx >> 3, ch = idx & 7, k = ck * 64 + ch * 8;
            const bool ok = row < p.r && k < p.K;
            if (NB * 64 % 128 == 0 || row < R)
                cp_async16(slot + row * 128 + ((ch ^ ((row & 1) << 2)) << 4), ok ? a + static_cast<size_t>(row) * p.K + k : a, ok);
        }
    };
    uint4 xs[DEPTH][STEPS][4];
    auto load_x = [&](uint4 (&to)[STEPS][4], int ck) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int k = ck * 64 + (WK == 2 ? wk : s) * 32 + c * 8;
#pragma unroll
            for (int i = 0; i < 4; ++i) to[s][i] = in[i] && k < p.K && ck < last ? __ldcs(reinterpret_cast<const uint4*>(x[i] + k)) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
#pragma unroll
    for (int d = 0; d < kStages - 1; ++d) {
        if (first + d < last) load_a(first + d);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load_x(xs[d], first + d);

    float acc[2][NBW][4] = {};
    for (int ck0 = first; ck0 < last; ck0 += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int ck = ck0 + d;
            if (ck >= last) break;
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            __syncthreads();  // chunk ck is there for all, and the slot of chunk ck - 1 is read no more
            if (ck + kStages - 1 < last) load_a(ck + kStages - 1);
            asm volatile("cp.async.commit_group;" ::: "memory");
            const uint8_t* slot = ring + (ck - first) % kStages * kStageBytes;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const int half = WK == 2 ? wk : s;
                const uint4(&f)[4] = xs[d][s];
                const uint32_t f0[2][4] = {{f[0].x, f[1].x, f[0].y, f[1].y}, {f[2].x, f[3].x, f[2].y, f[3].y}};
                const uint32_t f1[2][4] = {{f[0].z, f[1].z, f[0].w, f[1].w}, {f[2].z, f[3].z, f[2].w, f[3].w}};
                uint4 w[NBW];
#pragma unroll
                for (int n = 0; n < NBW; ++n) w[n] = *reinterpret_cast<const uint4*>(slot + ((wr * NBW + n) * 8 + g) * 128 + (((half * 4 + c) ^ ((g & 1) << 2)) << 4));
                // MMAs on the same accumulator are kept apart: each waits for the one before
#pragma unroll
                for (int n = 0; n < NBW; ++n)
#pragma unroll
                    for (int m = 0; m < 2; ++m) mma16816<T>(acc[m][n], f0[m], w[n].x, w[n].y);
#pragma unroll
                for (int n = 0; n < NBW; ++n)
#pragma unroll
                    for (int m = 0; m < 2; ++m) mma16816<T>(acc[m][n], f1[m], w[n].z, w[n].w);
            }
            load_x(xs[d], ck + DEPTH);
        }
    }
    __syncthreads();  // the ring is read no more (and no copy is pending: every chunk was waited for)
    float* part = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NBW; ++n) {
            float* to = part + (wk * kLong + wm * 32 + m * 16 + g) * kPitch + (wr * NBW + n) * 8 + 2 * c;
            *reinterpret_cast<float2*>(to) = make_float2(acc[m][n][0], acc[m][n][1]);
            *reinterpret_cast<float2*>(to + 8 * kPitch) = make_float2(acc[m][n][2], acc[m][n][3]);
        }
    __syncthreads();
    if constexpr (WK == 2) {
        for (int i = threadIdx.x; i < kLong * kPitch; i += blockDim.x) part[i] += part[kLong * kPitch + i];
    }
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    const float scale = p.scale ? p.scale[adapter] : 1.0f;
    constexpr int VP = inner_pitch(NB);
    for (int row = rank * kLongWarps + warp; row < tokens; row += clusterCtas * kLongWarps) {
        float v[(VP + 31) / 32];
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < VP / 32; ++i) {
            const int col = lane + 32 * i;
            v[i] = 0.f;
            if (col < R) {
                const uint32_t at = smem_u32(part + row * kPitch + col);
                for (int q = 0; q < clusterCtas; ++q) v[i] += ld_cluster_f32(mapa_u32(at, q));
                v[i] *= scale;
            }
            top = fmaxf(top, fabsf(v[i]));
        }
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
        const int shift = range_shift(top);
        const float down = exp2_int(-shift);
        if (lane == 0) o.unit[start + row] = exp2_int(shift);
        unsigned short* to = static_cast<unsigned short*>(o.v) + static_cast<size_t>(start + row) * 2 * VP;
#pragma unroll
        for (int i = 0; i < VP / 32; ++i) {
            const uint2 h = split16<T>(v[i] * down);
            to[lane + 32 * i] = static_cast<unsigned short>(h.x);
            to[VP + lane + 32 * i] = static_cast<unsigned short>(h.y);
        }
    }
    __syncwarp();
    cluster_arrive();  // no CTA ends while another reads its sums
    cluster_wait();
}

// A warp keeps the split inner products of its tokens (32, or 16 for ranks above 64) in registers and walks over groups of
// 32 columns; B and base come straight to fragments and the next group's are requested before this one's products.
template <typename T, int NB> __global__ void __launch_bounds__(32 * kLongWarps) low_rank_outer_kernel(const LowRankArgs p, const InnerOut o)
{
    constexpr int VP = inner_pitch(NB), KS = VP / 32, MT = NB > 8 ? 1 : 2, WM = kLong / (16 * MT), WN = kLongWarps / WM;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int wm = warp % WM, wn = warp / WM;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 tile = o.tiles[blockIdx.y];
    const int adapter = tile.x, start = tile.y, tokens = tile.z;
    if (adapter < 0 || wm * 16 * MT >= tokens) return;
    const bool has = adapter < p.L;
    if (!has && p.base == p.dst) return;
    const T* base[2 * MT];
    T* dst[2 * MT];
    bool in[2 * MT];
    float unit[2 * MT];
    uint32_t f[2][MT][KS][2][4];  // hi / lo, 16 tokens, 32 of the rank, 16 of them
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
        const int row = wm * 16 * MT + g + 8 * i;
        in[i] = row < tokens;
        const int64_t t = in[i] ? p.order[start + row] : 0;
        base[i] = p.base ? static_cast<const T*>(p.base) + t * p.ldBase : nullptr;
        dst[i] = static_cast<T*>(p.dst) + t * p.ldDst;
        unit[i] = has && in[i] ? o.unit[start + row] : 0.f;
        const T* v = static_cast<const T*>(o.v) + static_cast<size_t>(start + (in[i] ? row : 0)) * 2 * VP;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const uint4 w = has && in[i] ? *reinterpret_cast<const uint4*>(v + h * VP + s * 32 + c * 8) : make_uint4(0u, 0u, 0u, 0u);
                f[h][i >> 1][s][0][i & 1] = w.x;
                f[h][i >> 1][s][0][2 + (i & 1)] = w.y;
                f[h][i >> 1][s][1][i & 1] = w.z;
                f[h][i >> 1][s][1][2 + (i & 1)] = w.w;
            }
    }
    const T* b = static_cast<const T*>(p.b) + static_cast<size_t>(has ? adapter : 0) * p.N * p.r;
    const int nEnd = min(p.N, static_cast<int>(blockIdx.x + 1) * kColumns);
    uint4 y[2 * MT];
    auto load_base = [&](int n0) {
        const int col = n0 + c * 8;
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) y[i] = base[i] && in[i] && col < nEnd ? *reinterpret_cast<const uint4*>(base[i] + col) : make_uint4(0u, 0u, 0u, 0u);
    };
    uint4 w[4][KS];
    auto load_b = [&](int n0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // column g of MMA j is column 8 (g / 2) + 2 j + (g & 1) of the group: accumulators 2c, 2c + 1 of the four MMAs are 8 neighbours
            const int n = n0 + 8 * (g >> 1) + 2 * j + (g & 1);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int k = s * 32 + c * 8;
                w[j][s] = has && n < nEnd && k < p.r ? __ldg(reinterpret_cast<const uint4*>(b + static_cast<size_t>(n) * p.r + k)) : make_uint4(0u, 0u, 0u, 0u);
            }
        }
    };
    int n0 = blockIdx.x * kColumns + wn * 32;
    load_base(n0);
    load_b(n0);
    for (; n0 < nEnd; n0 += WN * 32) {
        float acc[MT][4][4] = {};
        if (has) {
            uint4 wNow[4][KS];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int s = 0; s < KS; ++s) wNow[j][s] = w[j][s];
            load_b(n0 + WN * 32);
            // MMAs on the same accumulator are kept apart: each waits for the one before
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int m = 0; m < MT; ++m)
                                mma16816<T>(acc[m][j], f[h][m][s][q], q ? wNow[j][s].z : wNow[j][s].x, q ? wNow[j][s].w : wNow[j][s].y);
        }
        uint4 now[2 * MT];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) now[i] = y[i];
        load_base(n0 + WN * 32);
        const int col = n0 + c * 8;
        if (col >= nEnd) continue;
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
            if (!in[i]) continue;
            uint32_t out[4];
            const uint32_t was[4] = {now[i].x, now[i].y, now[i].z, now[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 v = unpack2<T>(was[j]);
                out[j] = has ? pack_sat<T>(fmaf(acc[i >> 1][j][2 * (i & 1)], unit[i], v.x), fmaf(acc[i >> 1][j][2 * (i & 1) + 1], unit[i], v.y)) : was[j];
            }
            __stcs(reinterpret_cast<uint4*>(dst[i] + col), make_uint4(out[0], out[1], out[2], out[3]));
        }
    }
}

template <typename T, int NB> ascq_status launch_low_rank(const LowRankArgs& p, int cluster, unsigned tiles, cudaStream_t st)
{
    const size_t smem = (static_cast<size_t>(red_words(NB, p.L)) + part_words(NB) + split_words(NB)) * 4;
    static PerDeviceOnce once;
    const int dev = current_device();
    if (!once.done(dev)) {
        const int most = (red_words(NB, kMaxSortKeys) + part_words(NB) + split_words(NB)) * 4;
        ASCQ_CUDA_CHECK(cudaFuncSetAttribute(low_rank_kernel<T, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
        once.mark(dev);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(tiles * cluster, 1, 1);
    cfg.blockDim = dim3(32 * kWarps, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    ASCQ_CUDA_CHECK(cudaLaunchKernelEx(&cfg, low_rank_kernel<T, NB>, p, cluster));
    return ASCQ_OK;
}

template <typename T> ascq_status launch_low_rank_typed(const LowRankArgs& p, int cluster, unsigned tiles, cudaStream_t st)
{
    if (p.r <= 8) return launch_low_rank<T, 1>(p, cluster, tiles, st);
    if (p.r <= 16) return launch_low_rank<T, 2>(p, cluster, tiles, st);
    if (p.r <= 32) return launch_low_rank<T, 4>(p, cluster, tiles, st);
    if (p.r <= 64) return launch_low_rank<T, 8>(p, cluster, tiles, st);
    return launch_low_rank<T, 16>(p, cluster, tiles, st);
}

template <typename K, typename... Args>
cudaError_t launch_pdl(K kernel, dim3 grid, unsigned block, size_t smem, int cluster, cudaStream_t st, Args... args)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T, int NB> ascq_status launch_low_rank_long(const LowRankArgs& p, const InnerOut& o, unsigned tiles, cudaStream_t st)
{
    constexpr int ringBytes = kStages * NB * 8 * 128, sumBytes = (NB > 8 ? 1 : 2) * kLong * (NB * 8 + 8) * 4;
    constexpr int smem = ringBytes > sumBytes ? ringBytes : sumBytes;
    static PerDeviceOnce once;
    const int dev = current_device();
    if (!once.done(dev)) {
        ASCQ_CUDA_CHECK(cudaFuncSetAttribute(low_rank_inner_kernel<T, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        once.mark(dev);
    }
    // K is split until there are about two CTAs per SM; a CTA keeps at least four chunks of 64
    int cluster = 8;
    while (cluster > 1 && (static_cast<uint64_t>(tiles) * cluster > 3ull * sm_count() || p.K < cluster * 256)) cluster /= 2;
    ASCQ_CUDA_CHECK(launch_pdl(low_rank_inner_kernel<T, NB>, dim3(tiles * cluster), 32 * kLongWarps, smem, cluster, st, p, o, cluster));
    ASCQ_CUDA_CHECK(launch_pdl(low_rank_outer_kernel<T, NB>, dim3((p.N + kColumns - 1) / kColumns, tiles), 32 * kLongWarps, 0, 1, st, p, o));
    return ASCQ_OK;
}
template <typename T> ascq_status launch_low_rank_long_typed(const LowRankArgs& p, const InnerOut& o, unsigned tiles, cudaStream_t st)
{
    if (p.r <= 16) return launch_low_rank_long<T, 2>(p, o, tiles, st);
    if (p.r <= 32) return launch_low_rank_long<T, 4>(p, o, tiles, st);
    if (p.r <= 64) return launch_low_rank_long<T, 8>(p, o, tiles, st);
    return launch_low_rank_long<T, 16>(p, o, tiles, st);
}

// Tiles of 64 tokens pay when an adapter has enough tokens to fill them.
bool long_tiles(int M, int L) { return M > kInlineTokens && M / (L + 1) >= 16; }

// Every adapter with tokens, and the tokens without one, can leave one tile partly filled.
int64_t tile_bound(int M, int L, int size) { return M / size + std::min(L + 1, M); }

struct Workspace {
    size_t order, tiles, unit, v, bytes;  // offsets; the counts come first
};
Workspace workspace_of(int M, int r, int L)
{
    Workspace w{};
    if (M <= kInlineTokens || r <= 0 || r > 128 || L <= 0) return w;
    auto up = [](size_t n) { return (n + 15) / 16 * 16; };
    w.order = up((static_cast<size_t>(L) + 1) * 8);
    w.bytes = w.order + up(static_cast<size_t>(M) * 4);
    if (long_tiles(M, L)) {
        w.tiles = w.bytes;
        w.unit = w.tiles + static_cast<size_t>(tile_bound(M, L, kLong)) * 16;
        w.v = w.unit + up(static_cast<size_t>(M) * 4);
        w.bytes = w.v + static_cast<size_t>(M) * 2 * inner_pitch(r <= 32 ? 4 : r <= 64 ? 8 : 16) * 2;
    }
    return w;
}

constexpr int kMaxRank = 128;

}  // namespace
}  // namespace ascq

extern "C" size_t ascq_low_rank_add_workspace_size(int M, int r, int L) { return workspace_of(M, r, L).bytes; }

extern "C" ascq_status ascq_low_rank_add(void* dst, int64_t ldDst, const void* base, int64_t ldBase, const void* x, int64_t ldX, const void* A, const void* B,
                                         ascq_dtype T, const void* adapterIds, ascq_dtype idT, const float* scale, int M, int N, int K, int r, int L,
                                         void* workspace, size_t workspaceBytes, void* stream)
{
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (T != ASCQ_DT_F16 && T != ASCQ_DT_BF16) return fail(ASCQ_ERR_UNSUPPORTED, "x, A, B, base and dst must be half or bfloat16_t");
    if (idT != ASCQ_DT_I32 && idT != ASCQ_DT_I64) return fail(ASCQ_ERR_UNSUPPORTED, "adapterIds must be int32 or int64");
    if (M < 0 || N < 0 || K <= 0) return fail(ASCQ_ERR_INVALID_ARG, "M and N must not be negative and K must be positive");
    if (N % 8 != 0 || K % 8 != 0) return fail(ASCQ_ERR_INVALID_ARG, "N is %d and K is %d, which must be multiples of 8", N, K);
    if (r <= 0 || r > kMaxRank || r % 8 != 0) return fail(ASCQ_ERR_INVALID_ARG, "the rank is %d, which must be a multiple of 8 up to %d", r, kMaxRank);
    if (L < 1 || L >= kMaxSortKeys) return fail(ASCQ_ERR_INVALID_ARG, "the number of adapters is %d, which must be in [1, %d]", L, kMaxSortKeys - 1);
    if (ldDst == 0) ldDst = N;
    if (ldBase == 0) ldBase = N;
    if (ldX == 0) ldX = K;
    if (ldDst < N || ldBase < N || ldX < K) return fail(ASCQ_ERR_INVALID_ARG, "a row pitch is smaller than its rows");
    if (M == 0 || N == 0) return ASCQ_OK;
    if (!dst || !x || !A || !B || !adapterIds) return fail(ASCQ_ERR_INVALID_ARG, "dst, x, A, B and adapterIds must not be NULL");
    if (!aligned16(dst) || !aligned16(base) || !aligned16(x) || !aligned16(A) || !aligned16(B) || ldDst % 8 || (base && ldBase % 8) || ldX % 8)
        return fail(ASCQ_ERR_ALIGNMENT, "dst, base, x, A and B must be 16-byte aligned, their row pitches multiples of 8 elements");
    if ((reinterpret_cast<uintptr_t>(adapterIds) & (idT == ASCQ_DT_I64 ? 7u : 3u)) || (reinterpret_cast<uintptr_t>(scale) & 3u))
        return fail(ASCQ_ERR_ALIGNMENT, "a tensor is not aligned to its element type");
    const size_t rows = static_cast<size_t>(M);
    const Workspace ws = workspace_of(M, r, L);
    const size_t need = ws.bytes;
    if (need && (!workspace || workspaceBytes < need)) return fail(ASCQ_ERR_INVALID_ARG, "the workspace has %zu bytes, %zu are needed", workspaceBytes, need);
    if (need && !aligned16(workspace)) return fail(ASCQ_ERR_ALIGNMENT, "the workspace must be 16-byte aligned");
    const size_t dstBytes = ((rows - 1) * ldDst + N) * 2;
    const void* q[7] = {x, A, B, adapterIds, scale, need ? workspace : nullptr, base};
    const size_t b[7] = {((rows - 1) * ldX + K) * 2, static_cast<size_t>(L) * r * K * 2, static_cast<size_t>(L) * N * r * 2, rows * (idT == ASCQ_DT_I64 ? 8 : 4),
                         scale ? static_cast<size_t>(L) * 4 : 0, need, base ? ((rows - 1) * ldBase + N) * 2 : 0};
    for (int i = 0; i < 7; ++i) {
        if (i == 6 && base == dst && ldBase == ldDst) continue;
        if (spans_overlap(dst, dstBytes, q[i], b[i])) return fail(ASCQ_ERR_INVALID_ARG, "dst overlaps another tensor of the call (only base may be dst itself, with the same pitch)");
    }
    if (need)
        for (int i = 0; i < 7; ++i)
            if (i != 5 && spans_overlap(workspace, need, q[i], b[i])) return fail(ASCQ_ERR_INVALID_ARG, "the workspace overlaps another tensor of the call");

    LowRankArgs p{};
    p.x = x; p.a = A; p.b = B; p.base = base; p.dst = dst; p.ids = adapterIds; p.scale = scale;
    p.ldX = ldX; p.ldBase = ldBase; p.ldDst = ldDst;
    p.M = M; p.N = N; p.K = K; p.r = r; p.L = L; p.ids64 = idT == ASCQ_DT_I64;
    if (need) {
        int64_t* counts = static_cast<int64_t*>(workspace);
        uint8_t* w = static_cast<uint8_t*>(workspace);
        int32_t* order = reinterpret_cast<int32_t*>(w + ws.order);
        const ascq_status rc = launch_key_sort(counts, nullptr, order, adapterIds, p.ids64 != 0, M, L + 1, L, st);
        if (rc != ASCQ_OK) return rc;
        p.counts = counts;
        p.order = order;
        if (ws.tiles) {
            const InnerOut o{reinterpret_cast<int4*>(w + ws.tiles), w + ws.v, reinterpret_cast<float*>(w + ws.unit)};
            const int64_t tiles = tile_bound(M, L, kLong);
            if (tiles > 65535) return fail(ASCQ_ERR_INVALID_ARG, "M is too large for one launch");
            return T == ASCQ_DT_F16 ? launch_low_rank_long_typed<__half>(p, o, static_cast<unsigned>(tiles), st)
                                    : launch_low_rank_long_typed<__nv_bfloat16>(p, o, static_cast<unsigned>(tiles), st);
        }
    }
    const unsigned tiles = static_cast<unsigned>(tile_bound(M, L, kTile));
    int cluster = 8;
    while (cluster > 1 && static_cast<uint64_t>(tiles) * cluster > 2ull * sm_count()) cluster /= 2;
    return T == ASCQ_DT_F16 ? launch_low_rank_typed<__half>(p, cluster, tiles, st) : launch_low_rank_typed<__nv_bfloat16>(p, cluster, tiles, st);
}
