// Low-rank adapters of many requests at once, added to the result of a shared projection:
//   dst[t] = cast(base[t] + scale[a] * (x[t] . A[a]^T) . B[a]^T),  a = adapterIds[t];   x [M, K], A [L, r, K], B [L, N, r]
// A token whose number is outside [0, L) has no adapter: dst[t] = base[t].
//
// What bounds it: x, base and dst cross HBM once (2 (K + 2 N) bytes a token), each used adapter once (2 r (K + N) bytes); with ranks up to
// 128 the products stay below what the tensor cores do in that time.  So the tokens are grouped by adapter -- a tile is up to 16 tokens
// of one adapter -- and both products of a tile run in one launch: a cluster of CTAs splits K for the first, adds its
// partial sums through distributed shared memory, and splits N for the second.  The [16, r] inner product never leaves the SMs.  Up to 1024
// tokens nothing else is launched: every CTA finds its tile in the adapter numbers (4 KB).  32 tokens of 16 adapters, 4096 x 4096, rank 16: 7.1 us,
// of which the 5 MB are 0.8 us; the rest is the chain from adapter number to token, to x and A, across the cluster, to dst.
//
// Both operands of the MMAs come straight from global memory: a dot product does not care in which order k is visited, so a
// lane's 16 consecutive bytes of a row serve as the fragments of two m16n8k16 MMAs.
//
// Calls with enough tokens per adapter take another form, low_rank_long.cu.
//
// The inner product is a sum in fp32; for the second product it is split into two 16-bit terms, hi = cast(v), lo = cast(v - hi), after
// each token's row was multiplied by a power of two that keeps both inside the type's range (range_shift).  What the split drops is below
// 2^-16 (bf16) or 2^-22 (fp16) of the value, a 2^8-th or less of what x, A and base lost when they were rounded to their type; beside the result's own
// rounding it shows only where terms of the sum cancel by more than that.  A third term keeps all 24 bits in bf16 and was measured: us, two / three
// terms, 32 tokens of rank 16 7.1 / 7.5, 256 of rank 128 24.4 / 27.2, 8192 tokens of 4096 x 4096 at rank 64 63 / 67, at rank 128 79 / 88.
#include "experts.cuh"
#include "low_rank.cuh"
#include "sm100_ptx.cuh"

using namespace ascq;
using namespace ascq::ptx;

namespace ascq {
namespace {

constexpr int kMaxRank = 128;
constexpr int kMaxWidth = 1 << 30;  // of N and K: column indices and a step of the whole cluster beyond them stay below 2^31
constexpr int kTile = 16;         // tokens of one adapter that share a tile
constexpr int kWarps = 8;
constexpr int kInlineTokens = 1024;  // up to here every CTA finds its tile in the adapter numbers itself; beyond, they are sorted first

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
    // each warp owns a contiguous run of tokens and keeps their adapters in registers
    constexpr int kSteps = kInlineTokens / (32 * kWarps);
    const int run = (p.M + 32 * kWarps - 1) / (32 * kWarps) * 32, begin = warp * run;
    int key[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int t = begin + i * 32 + lane;
        key[i] = i * 32 < run && t < p.M ? adapter_of(p, t) : -1;
    }
    int* hist = work;
    int* perWarp = work + keys;
    for (int e = threadIdx.x; e < keys; e += blockDim.x) hist[e] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        // counts: the order of the additions does not show; a run of one request's tokens is one addition
        const int first = __shfl_sync(0xFFFFFFFFu, key[i], 0);
        if (__all_sync(0xFFFFFFFFu, key[i] == first)) {
            if (lane == 0 && first >= 0) atomicAdd(&hist[first], 32);
        } else if (key[i] >= 0) {
            atomicAdd(&hist[key[i]], 1);
        }
    }
    __syncthreads();
    if (warp == 0) find_tile<kTile>(tile, keys, [&](int e) { return hist[e]; }, found);
    __syncthreads();
    const Tile t{found[0], found[0] < 0 ? 0 : found[1]};
    if (t.adapter < 0) return t;
    // the adapter's tokens in ascending order
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) mine += __popc(__ballot_sync(0xFFFFFFFFu, key[i] == t.adapter));
    if (lane == 0) perWarp[warp] = mine;
    __syncthreads();
    int at = -found[2];
    for (int w = 0; w < warp; ++w) at += perWarp[w];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const bool hit = key[i] == t.adapter;
        const uint32_t all = __ballot_sync(0xFFFFFFFFu, hit);
        const int slot = at + __popc(all & ((1u << lane) - 1u));
        if (hit && slot >= 0 && slot < kTile) list[slot] = begin + i * 32 + lane;
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

__host__ __device__ constexpr int padded_rank(int nb) { return nb * 8 < 32 ? 32 : nb * 8; }  // whole 32-wide k steps of the second product
// float words of dynamic shared memory: the warps' sums (the tile finder's scratch before that), the cluster's partial sums (every CTA's
// copy of all of them), and the split result
__host__ __device__ constexpr int red_words(int nb, int L)
{
    const int sums = kWarps * kTile * nb * 8, finder = (L + 1 + kWarps + 3) / 4 * 4;
    return sums > finder ? sums : finder;
}
__host__ __device__ constexpr int part_words(int nb) { return kTile * nb * 8; }
__host__ __device__ constexpr int split_words(int nb) { return kTile * (padded_rank(nb) / 2 + 4) * 2; }

// NB: blocks of 8 of the rank (r <= 8 NB)
template <typename T, int NB> __global__ void __launch_bounds__(32 * kWarps, NB <= 8 ? 2 : 1) low_rank_kernel(const LowRankArgs p, int clusterCtas)
{
    extern __shared__ float smem[];
    __shared__ int list[kTile], found[4];
    __shared__ float unit[kTile];  // the power of two that brings a token's row back
    constexpr int R = NB * 8, KS = padded_rank(NB) / 32, VP = padded_rank(NB) / 2 + 4;  // VP: row pitch of the split result in words
    constexpr bool kAhead = KS == 1;  // B's and base's first columns are requested together with x and A (registers allow it up to rank 32)
    float* red = smem;
    float* part = red + red_words(NB, p.L);  // [clusterCtas][kTile][R]
    uint32_t* hi = reinterpret_cast<uint32_t*>(part + clusterCtas * part_words(NB));
    uint32_t* lo = hi + kTile * VP;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int rank = blockIdx.x % clusterCtas;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Tile tile = take_tile(p, blockIdx.x / clusterCtas, list, found, reinterpret_cast<int*>(red));
    if (tile.adapter < 0) return;  // the same for every CTA of the cluster
    const bool has = tile.adapter < p.L;
    if (has) cluster_arrive();     // this CTA runs: its shared memory can be written from the others
    const int units = clusterCtas * kWarps, unitIdx = rank * kWarps + warp;
    const int t0 = list[g], t1 = list[g + 8];
    const bool in0 = g < tile.tokens, in1 = g + 8 < tile.tokens;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);

    // second product: this warp's groups of 32 columns; lane c of a row owns 8 consecutive ones
    const T* b = static_cast<const T*>(p.b) + static_cast<size_t>(has ? tile.adapter : 0) * p.N * p.r;
    auto load_columns = [&](int n0, uint4 (&w)[4][KS], uint4& y0, uint4& y1) {
        const int col = n0 + c * 8;  // N is a multiple of 8
        y0 = p.base && in0 && col < p.N ? *reinterpret_cast<const uint4*>(static_cast<const T*>(p.base) + static_cast<int64_t>(t0) * p.ldBase + col) : zero;
        y1 = p.base && in1 && col < p.N ? *reinterpret_cast<const uint4*>(static_cast<const T*>(p.base) + static_cast<int64_t>(t1) * p.ldBase + col) : zero;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // column g of MMA j is column 8 (g / 2) + 2 j + (g & 1) of the group, so that accumulators 2c, 2c + 1 of the four MMAs are a
            // lane's 8 neighbours
            const int n = n0 + 8 * (g >> 1) + 2 * j + (g & 1);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int k = s * 32 + c * 8;
                w[j][s] = has && n < p.N && k < p.r ? __ldg(reinterpret_cast<const uint4*>(b + static_cast<size_t>(n) * p.r + k)) : zero;
            }
        }
    };
    uint4 w[4][KS], y0, y1;

    if (has) {
        // ---- inner product: this warp's chunks of 32 k
        const T* a = static_cast<const T*>(p.a) + static_cast<size_t>(tile.adapter) * p.r * p.K;
        const T* x0 = static_cast<const T*>(p.x) + static_cast<int64_t>(t0) * p.ldX;
        const T* x1 = static_cast<const T*>(p.x) + static_cast<int64_t>(t1) * p.ldX;
        float acc[NB][4] = {};
        if constexpr (kAhead) load_columns(unitIdx * 32, w, y0, y1);
#pragma unroll 2
        for (int k = unitIdx * 32 + c * 8; k - c * 8 < p.K; k += units * 32) {
            const bool kIn = k < p.K;
            const uint4 u0 = in0 && kIn ? __ldg(reinterpret_cast<const uint4*>(x0 + k)) : zero;
            const uint4 u1 = in1 && kIn ? __ldg(reinterpret_cast<const uint4*>(x1 + k)) : zero;
            uint4 v[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n)
                v[n] = kIn && n * 8 + g < p.r ? __ldg(reinterpret_cast<const uint4*>(a + static_cast<size_t>(n * 8 + g) * p.K + k)) : zero;
            const uint32_t f0[4] = {u0.x, u1.x, u0.y, u1.y}, f1[4] = {u0.z, u1.z, u0.w, u1.w};
#pragma unroll
            for (int n = 0; n < NB; ++n) mma16816<T>(acc[n], f0, v[n].x, v[n].y);
#pragma unroll
            for (int n = 0; n < NB; ++n) mma16816<T>(acc[n], f1, v[n].z, v[n].w);
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float* to = red + warp * kTile * R + n * 8 + 2 * c;
            *reinterpret_cast<float2*>(to + g * R) = make_float2(acc[n][0], acc[n][1]);
            *reinterpret_cast<float2*>(to + (g + 8) * R) = make_float2(acc[n][2], acc[n][3]);
        }
        __syncthreads();
        // the CTA's sum goes to every CTA of the cluster (stores, which nobody waits for, rather than loads): one cluster barrier, then all
        // of them add up the same partial sums in the same order
        cluster_wait();
        for (int i = threadIdx.x * 4; i < kTile * R; i += blockDim.x * 4) {
            float4 s = *reinterpret_cast<const float4*>(red + i);
#pragma unroll
            for (int q = 1; q < kWarps; ++q) {
                const float4 f = *reinterpret_cast<const float4*>(red + q * kTile * R + i);
                s.x += f.x; s.y += f.y; s.z += f.z; s.w += f.w;
            }
            const uint32_t at = smem_u32(part + rank * part_words(NB) + i);
            const uint4 bits = make_uint4(__float_as_uint(s.x), __float_as_uint(s.y), __float_as_uint(s.z), __float_as_uint(s.w));
            for (int q = 0; q < clusterCtas; ++q) st_cluster_v4(mapa_u32(at, q), bits);
        }
        const float scale = p.scale ? p.scale[tile.adapter] : 1.0f;
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        // ---- the cluster's sum, scaled, brought to a common range per token and split; a warp takes two tokens
#pragma unroll
        for (int u = 0; u < kTile / kWarps; ++u) {
            const int row = warp + u * kWarps;
            float v[(R + 31) / 32];
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < (R + 31) / 32; ++i) {
                const int col = lane + 32 * i;
                v[i] = 0.f;
                if (col < R) {
                    for (int q = 0; q < clusterCtas; ++q) v[i] += part[q * part_words(NB) + row * R + col];
                    v[i] *= scale;
                }
                top = fmaxf(top, fabsf(v[i]));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            if (__builtin_expect(!(top <= 3.4028234663852886e38f), 0)) {
#pragma unroll
                for (int i = 0; i < (R + 31) / 32; ++i) v[i] = inside_range<T>(v[i]);
            }
            const int shift = range_shift<T>(top);
            const float down = exp2_int(-shift);
            if (lane == 0) unit[row] = exp2_int(shift);
            unsigned short* h = reinterpret_cast<unsigned short*>(hi + row * VP);
            unsigned short* l = reinterpret_cast<unsigned short*>(lo + row * VP);
#pragma unroll
            for (int i = 0; i < padded_rank(NB) / 32; ++i) {
                const int col = lane + 32 * i;
                const uint2 two = split16<T>(col < R ? v[i] * down : 0.f);
                h[col] = static_cast<unsigned short>(two.x);
                l[col] = static_cast<unsigned short>(two.y);
            }
        }
        __syncthreads();
    }

    // ---- second product
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
    if (!kAhead || !has) load_columns(unitIdx * 32, w, y0, y1);
    for (int n0 = unitIdx * 32; n0 < p.N; n0 += units * 32) {
        float acc[4][4] = {};
        const int col = n0 + c * 8;
        if (has) {
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        mma16816<T>(acc[j], fh[s][q], q ? w[j][s].z : w[j][s].x, q ? w[j][s].w : w[j][s].y);
                        mma16816<T>(acc[j], fl[s][q], q ? w[j][s].z : w[j][s].x, q ? w[j][s].w : w[j][s].y);
                    }
        }
        const uint32_t i0[4] = {y0.x, y0.y, y0.z, y0.w}, i1[4] = {y1.x, y1.y, y1.z, y1.w};
        if (n0 + units * 32 < p.N) load_columns(n0 + units * 32, w, y0, y1);
        if (col >= p.N) continue;
        uint4 o0 = make_uint4(i0[0], i0[1], i0[2], i0[3]), o1 = make_uint4(i1[0], i1[1], i1[2], i1[3]);
        if (has) {
            float f0[8], f1[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 v0 = unpack2<T>(i0[j]), v1 = unpack2<T>(i1[j]);
                f0[2 * j] = fmaf(acc[j][0], back0, v0.x);
                f0[2 * j + 1] = fmaf(acc[j][1], back0, v0.y);
                f1[2 * j] = fmaf(acc[j][2], back1, v1.x);
                f1[2 * j + 1] = fmaf(acc[j][3], back1, v1.y);
            }
            o0 = pack8_sat<T>(f0);
            o1 = pack8_sat<T>(f1);
        }
        if (in0) *reinterpret_cast<uint4*>(static_cast<T*>(p.dst) + static_cast<int64_t>(t0) * p.ldDst + col) = o0;
        if (in1) *reinterpret_cast<uint4*>(static_cast<T*>(p.dst) + static_cast<int64_t>(t1) * p.ldDst + col) = o1;
    }
}

template <typename T, int NB> ascq_status launch_low_rank(const LowRankArgs& p, int cluster, unsigned tiles, cudaStream_t st)
{
    const size_t smem = (static_cast<size_t>(red_words(NB, p.L)) + static_cast<size_t>(cluster) * part_words(NB) + split_words(NB)) * 4;
    static PerDeviceOnce once;
    const int dev = current_device();
    if (!once.done(dev)) {
        const int most = (red_words(NB, kMaxSortKeys) + 8 * part_words(NB) + split_words(NB)) * 4;
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

// Tiles of 128 tokens pay for their second and third launch when there is enough to do and adapters have tokens to fill them.  Measured, us,
// tiles of 16 / of 128 tokens, 4 adapters: K + N = 15104, rank 64: 23 / 30 at 1024 tokens, 43 / 31 at 1500; K = N = 4096, rank 64: 29 / 30 at 2048,
// 47 / 31 at 2800; rank 16: 20 / 26, 35 / 27; rank 128: 25 / 24 at 512, 39 / 27 at 1024.  64 adapters, rank 64, 4096 tokens: 62 / 86.
bool long_tiles(int M, int N, int K, int r, int L)
{
    const int64_t work = static_cast<int64_t>(M) * (static_cast<int64_t>(K) + N) * (r > 64 ? 3 : 1);
    return work >= 20'000'000 && M / (L + 1) >= (r > 64 ? 24 : 64) && static_cast<int64_t>(L) * N <= 0x7FFFFFFF;  // (the copies' coordinates are int)
}

// Every adapter with tokens, and the tokens without one, can leave one tile partly filled.
int64_t tile_bound(int M, int L, int size) { return M / size + std::min(L + 1, M); }

struct Workspace {
    size_t order, tiles, unit, v, bytes;  // offsets; the counts come first
};
Workspace workspace_of(int M, int N, int K, int r, int L)
{
    Workspace w{};
    if (M <= 0 || N <= 0 || K <= 0 || r <= 0 || r > kMaxRank || L <= 0) return w;
    const bool tiled = long_tiles(M, N, K, r, L);
    if (M <= kInlineTokens && !tiled) return w;
    auto up = [](size_t n) { return (n + 15) / 16 * 16; };
    w.order = up((static_cast<size_t>(L) + 1) * 8);
    w.bytes = w.order + up(static_cast<size_t>(M) * 4);
    if (tiled) {
        w.tiles = w.bytes;
        w.unit = w.tiles + low_rank_long_tiles_bytes(tile_bound(M, L, kLongTile));
        w.v = w.unit + up(static_cast<size_t>(M) * 4);
        w.bytes = w.v + low_rank_long_inner_bytes(M, r);
    }
    return w;
}

}  // namespace
}  // namespace ascq

extern "C" size_t ascq_low_rank_add_workspace_size(int M, int N, int K, int r, int L) { return workspace_of(M, N, K, r, L).bytes; }

extern "C" ascq_status ascq_low_rank_add(void* dst, int64_t ldDst, const void* base, int64_t ldBase, const void* x, int64_t ldX, const void* A, const void* B,
                                         ascq_dtype T, const void* adapterIds, ascq_dtype idT, const float* scale, int M, int N, int K, int r, int L,
                                         void* workspace, size_t workspaceBytes, void* stream)
{
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (T != ASCQ_DT_F16 && T != ASCQ_DT_BF16) return fail(ASCQ_ERR_UNSUPPORTED, "x, A, B, base and dst must be half or bfloat16_t");
    if (idT != ASCQ_DT_I32 && idT != ASCQ_DT_I64) return fail(ASCQ_ERR_UNSUPPORTED, "adapterIds must be int32 or int64");
    if (M < 0 || N < 0 || K <= 0) return fail(ASCQ_ERR_INVALID_ARG, "M and N must not be negative and K must be positive");
    if (N > kMaxWidth || K > kMaxWidth) return fail(ASCQ_ERR_INVALID_ARG, "N is %d and K is %d, which must be at most 2^30", N, K);
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
    const Workspace ws = workspace_of(M, N, K, r, L);
    const size_t need = ws.bytes;
    if (need && (!workspace || workspaceBytes < need)) return fail(ASCQ_ERR_INVALID_ARG, "the workspace has %zu bytes, %zu are needed", workspaceBytes, need);
    if (need && !aligned16(workspace)) return fail(ASCQ_ERR_ALIGNMENT, "the workspace must be 16-byte aligned");
    auto matrix = [&](const void* q, int64_t cols, int64_t ld) { return PitchedSpan{q, rows, static_cast<size_t>(cols) * 2, static_cast<size_t>(ld) * 2}; };
    auto flat = [](const void* q, size_t bytes) { return PitchedSpan{q, 1, bytes, 0}; };
    const PitchedSpan out = matrix(dst, N, ldDst), scratch = flat(need ? workspace : nullptr, need);
    const PitchedSpan in[6] = {matrix(x, K, ldX), matrix(base, N, ldBase), flat(A, static_cast<size_t>(L) * r * K * 2), flat(B, static_cast<size_t>(L) * N * r * 2),
                               flat(adapterIds, rows * (idT == ASCQ_DT_I64 ? 8 : 4)), flat(scale, static_cast<size_t>(L) * 4)};
    for (int i = 0; i < 6; ++i) {
        const bool same = i == 1 && base == dst && ldBase == ldDst;
        if (!same && spans_overlap(out, in[i])) return fail(ASCQ_ERR_INVALID_ARG, "dst overlaps another tensor of the call (only base may be dst itself, with the same pitch)");
        if (spans_overlap(scratch, in[i])) return fail(ASCQ_ERR_INVALID_ARG, "the workspace overlaps another tensor of the call");
    }
    if (spans_overlap(scratch, out)) return fail(ASCQ_ERR_INVALID_ARG, "the workspace overlaps another tensor of the call");

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
            const LowRankScratch o{w + ws.tiles, w + ws.v, reinterpret_cast<float*>(w + ws.unit), 0, 0};
            const int64_t tiles = tile_bound(M, L, kLongTile);
            if (tiles > 0x7FFFFFF) return fail(ASCQ_ERR_INVALID_ARG, "M is too large for one launch");
            return low_rank_long(p, T == ASCQ_DT_F16, o, static_cast<unsigned>(tiles), st);
        }
    }
    const unsigned tiles = static_cast<unsigned>(tile_bound(M, L, kTile));
    int cluster = 8;
    // as many CTAs as are resident together: two per SM, above rank 64 one (and clusters of 8 do not fill every SM)
    const uint64_t limit = r > 64 ? sm_count() * 7 / 8 : 2 * sm_count();
    while (cluster > 1 && static_cast<uint64_t>(tiles) * cluster > limit) cluster /= 2;
    return T == ASCQ_DT_F16 ? launch_low_rank_typed<__half>(p, cluster, tiles, st) : launch_low_rank_typed<__nv_bfloat16>(p, cluster, tiles, st);
}
