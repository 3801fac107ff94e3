// The form of ascq_low_rank_add for adapters with many tokens (prompts): two launches over tiles of up to 128 tokens of one adapter, tokens
// in sorted order, both products on tcgen05 with the accumulators in tensor memory.
//   inner   V = scale * x . A^T: a cluster of CTAs splits K and adds up through distributed shared memory; V leaves split into two 16-bit
//           terms, [M][2][pitch] in sorted order, with one power of two per token
//   outer   dst = base + V . B^T for a tile and a range of columns
// What bounds both is HBM: the inner launch reads x once, the outer one reads base and writes dst; A and B come from L2 once per 128
// tokens.  The tokens of a tile lie anywhere, so their rows are gathered with 16-byte cp.async into the 128-byte-swizzled layout that the
// tensor cores read; 64 elements of a row are 128 bytes, and the lanes that share a row fill a whole line.  What lies in order -- A, B, V -- comes
// by TMA: one thread asks for a tile, and no warp has to wait for it and make it visible to the tensor cores.
// 8192 tokens of 12 requests, 4096 x 4096, rank 64, bf16: 61 us with the sort = 3.5 TB/s of the 214 MB (sort 5, inner 22, outer 31 us); 1337 tokens,
// 11008 x 4096, rank 32, half: 28 us.  In its loops the outer launch moves 6 TB/s; what is lost is the start and the end of three launches.
#include "low_rank.cuh"
#include "sm100_ptx.cuh"
#include "tma_host.h"

using namespace ascq;
using namespace ascq::ptx;

namespace ascq {
namespace {

constexpr int kRows = kLongTile;
constexpr int kLoaders = 128, kThreads = 2 * kLoaders + 64;      // inner: two groups of four warps gather x, the first finishes too; one warp
                                                               // issues the MMAs, one the loads of A
constexpr int kFinishers = 256, kOuterThreads = kFinishers + 32;  // outer: eight warps move base and dst, one issues loads and MMAs
constexpr int kAtomBytes = kRows * 128;    // 128 rows x 64 elements
constexpr int kBlockCols = 64;             // outer: columns of an MMA

__device__ int g_low_rank_status;  // 1: a bounded wait ran out

__host__ __device__ constexpr int rank_pitch(int nb) { return nb * 8 < 64 ? 64 : nb * 8; }  // elements of the hi (or lo) part of a row of V
constexpr int rank_blocks(int r) { return r <= 16 ? 2 : r <= 32 ? 4 : r <= 64 ? 8 : 16; }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool in)
{
    const int bytes = in ? 16 : 0;  // the rest of the 16 bytes is filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// Waits for copies or MMAs that were issued, also when the CTA gives up: none may be under way when its memory is given back.  They end by
// themselves, so the bound is there for a broken machine only; it is not the adjustable limit, which may be short and has just run out.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity)
{
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity) && clock64() - t0 < kWaitCycles) {}
}
// this thread's finished copies become visible to the tensor cores, and the barrier learns of it
__device__ __forceinline__ void publish(uint64_t* bar)
{
    fence_proxy_async();
    mbar_arrive(bar);
}

// Chunks of 64 k in flight.  The two groups of loading warps take alternate chunks: waiting for a chunk's copies, making them visible to the
// tensor cores and announcing them takes a few hundred cycles, and the other group requests meanwhile.  A group announces a chunk
// kLag of its own chunks after it was requested (2 kLag < kStages: the slot that it waits for next was announced before).
template <int NB> struct Ring {
    static constexpr int kABytes = NB * 8 * 128, kStageBytes = kAtomBytes + kABytes;
    static constexpr int kSumBytes = kRows * (NB * 8 + 4) * 4;  // partial sums of the rows that this CTA finishes, from every CTA of the cluster
    static constexpr int kFit = (226 * 1024 - 1024 - kSumBytes) / kStageBytes;  // one CTA takes an SM's shared memory (227 KB)
    static constexpr int kStages = kFit < 8 ? kFit : 8, kLag = (kStages - 1) / 2;
    static constexpr int kBytes = kStages * kStageBytes + kSumBytes + 1024;  // + alignment
    static constexpr uint32_t kTmemCols = NB * 8 < 32 ? 32 : NB * 8;
};

// The rows of one CTA's share: CTAS threads a row, each sums its columns over the cluster's CTAs, scales them, finds the row's largest
// value with its neighbours and writes the two terms.
template <typename T, int NB, int CTAS>
__device__ __forceinline__ void finish_rows(const float* part, int there, int start, int r, float scale, const LowRankScratch& o)
{
    constexpr int R = NB * 8, VP = rank_pitch(NB), kPitch = R + 4, kShare = kRows / CTAS, W = R / CTAS;  // W: columns of a thread
    const int row = threadIdx.x / CTAS, col0 = (threadIdx.x % CTAS) * W;
    float v[W] = {}, top = 0.f;
#pragma unroll
    for (int q = 0; q < CTAS; ++q) {
        const float* at = part + (q * kShare + row) * kPitch + col0;
        if constexpr (W % 4 == 0) {
#pragma unroll
            for (int i = 0; i < W; i += 4) {
                const float4 f = *reinterpret_cast<const float4*>(at + i);
                v[i] += f.x; v[i + 1] += f.y; v[i + 2] += f.z; v[i + 3] += f.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] += at[i];
        }
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
        v[i] = col0 + i < r ? v[i] * scale : 0.f;
        top = fmaxf(top, fabsf(v[i]));
    }
#pragma unroll
    for (int s = 1; s < CTAS; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, s));
    if (row >= there) return;
    if (__builtin_expect(!(top <= 3.4028234663852886e38f), 0)) {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = inside_range<T>(v[i]);
    }
    const int shift = range_shift<T>(top);
    const float down = exp2_int(-shift);
    if (col0 == 0) o.unit[start + row] = exp2_int(shift);
    uint32_t hi[W / 2], lo[W / 2];
#pragma unroll
    for (int i = 0; i < W; i += 2) {
        const uint2 a = split16<T>(v[i] * down), b = split16<T>(v[i + 1] * down);
        hi[i / 2] = a.x | (b.x << 16);
        lo[i / 2] = a.y | (b.y << 16);
    }
    uint32_t* to = reinterpret_cast<uint32_t*>(static_cast<unsigned short*>(o.v) + static_cast<size_t>(start + row) * 2 * VP + col0);
    if constexpr (W % 8 == 0) {
#pragma unroll
        for (int i = 0; i < W / 2; i += 4) {
            *reinterpret_cast<uint4*>(to + i) = make_uint4(hi[i], hi[i + 1], hi[i + 2], hi[i + 3]);
            *reinterpret_cast<uint4*>(to + VP / 2 + i) = make_uint4(lo[i], lo[i + 1], lo[i + 2], lo[i + 3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
            to[i] = hi[i];
            to[VP / 2 + i] = lo[i];
        }
    }
    if constexpr (VP > R) {  // the rest of a short row is zeros: every thread fills its share
        constexpr int kRest = (VP - R) / CTAS / 2;
        uint32_t* rest = reinterpret_cast<uint32_t*>(static_cast<unsigned short*>(o.v) + static_cast<size_t>(start + row) * 2 * VP + R) + (threadIdx.x % CTAS) * kRest;
#pragma unroll
        for (int i = 0; i < kRest; ++i) rest[i] = rest[VP / 2 + i] = 0u;
    }
}

template <typename T, int NB> __global__ void __launch_bounds__(kThreads) low_rank_inner_kernel(const LowRankArgs p, const LowRankScratch o, int clusterCtas,
                                                                                          const __grid_constant__ CUtensorMap mapA)
{
    using C = Ring<NB>;
    constexpr int R = NB * 8, kPitch = R + 4;
    extern __shared__ uint8_t raw[];
    __shared__ int found[4];
    __shared__ uint64_t fullBar[C::kStages], aBar[C::kStages], emptyBar[C::kStages], doneBar;  // x gathered, A loaded, both read
    __shared__ uint32_t tmemSlot;
    __shared__ int abortFlag;
    uint8_t* ring = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tileIdx = blockIdx.x / clusterCtas, rank = blockIdx.x % clusterCtas;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(&fullBar[i], kLoaders);
            mbar_init(&aBar[i], 1);
            mbar_init(&emptyBar[i], 1);
        }
        mbar_init(&doneBar, 1);
        fence_barrier_init();
        abortFlag = 0;
    }
    if (warp == 8) {
        tmem_alloc(&tmemSlot, C::kTmemCols);
        tmem_relinquish();
    }
    // A dependent launch may take tensor memory too: it is let in only when this CTA has its columns.
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == 0) find_tile<kRows>(tileIdx, p.L + 1, [&](int e) { return static_cast<int>(p.counts[e]); }, found);
    if (warp == 1 && blockIdx.x == 0) {  // how many tiles there are, behind their table
        int all = 0;
        for (int e = lane; e <= p.L; e += 32) all += (static_cast<int>(p.counts[e]) + kRows - 1) / kRows;
        all = __reduce_add_sync(0xFFFFFFFFu, all);
        if (lane == 0) static_cast<int4*>(o.tiles)[gridDim.x / clusterCtas].x = all;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const int adapter = found[0], tokens = adapter < 0 ? 0 : found[1], start = adapter < 0 ? 0 : found[3];
    if (rank == 0 && threadIdx.x == 0) static_cast<int4*>(o.tiles)[tileIdx] = make_int4(adapter, start, tokens, 0);
    const bool has = adapter >= 0 && adapter < p.L;  // the same for every CTA of the cluster
    if (has) {
        cluster_arrive();
        const int chunks = (p.K + 63) / 64, per = (chunks + clusterCtas - 1) / clusterCtas;
        const int first = min(rank * per, chunks), n = min(first + per, chunks) - first;
        bool ok = true;
        if (warp < 8) {
            // 16 rows at a time, eight lanes a row: row (t / 8) + 16 i, piece t % 8; the swizzle exchanges pieces by the row's low three bits
            const int group = warp >> 2, piece = threadIdx.x & 7, row0 = (threadIdx.x & (kLoaders - 1)) >> 3;
            const uint32_t at = smem_u32(ring) + row0 * 128 + ((piece ^ (row0 & 7)) << 4);
            const T* x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = row0 + 16 * i;
                x[i] = row < tokens ? static_cast<const T*>(p.x) + static_cast<int64_t>(p.order[start + row]) * p.ldX + first * 64 + piece * 8 : nullptr;
            }
            for (int i = group; i < n; i += 2) {
                const int s = i % C::kStages;
                if (i >= C::kStages && !(ok = mbar_wait_bounded<false>(&emptyBar[s], (i / C::kStages - 1) & 1, &abortFlag))) break;
                const bool kIn = (first + i) * 64 + piece * 8 < p.K;
                const uint32_t slot = at + s * C::kStageBytes;
                // a row without a token keeps whatever the slot holds: a row of A times it is a row of D that nobody reads
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (x[j]) cp_async16(slot + j * 2048, kIn ? x[j] + i * 64 : p.x, kIn);
                cp_commit();
                if (i >= 2 * C::kLag) {
                    cp_wait<C::kLag>();
                    publish(&fullBar[(i - 2 * C::kLag) % C::kStages]);
                }
            }
            cp_wait<0>();
            if (ok) {  // the group's last chunks
                const int count = (n - group + 1) / 2;
                for (int j = max(count - C::kLag, 0); j < count; ++j) publish(&fullBar[(2 * j + group) % C::kStages]);
            }
        } else if (warp == 9) {
            if (elect_one()) {
                const int loads = min(n, o.stopA);
                int i = 0;
                for (; i < loads; ++i) {
                    const int s = i % C::kStages;
                    if (i >= C::kStages && !(ok = mbar_wait_bounded<false>(&emptyBar[s], (i / C::kStages - 1) & 1, &abortFlag))) break;
                    // rows behind the adapter's rank are the next adapter's (or zeros): columns of D that finish_rows leaves out
                    mbar_arrive_expect_tx(&aBar[s], C::kABytes);
                    tma_load_2d(ring + s * C::kStageBytes + kAtomBytes, &mapA, &aBar[s], (first + i) * 64, adapter * p.r);
                }
                // (whoever gives up: the MMAs need not have waited for the last loads)
                for (int j = max(i - C::kStages, 0); j < i; ++j) drain(&aBar[j % C::kStages], (j / C::kStages) & 1);
            }
        } else if (elect_one()) {
            constexpr uint32_t idesc = idesc_f16(kRows, R, std::is_same<T, __half>::value ? 0 : 1);
            for (int i = 0; i < n && ok; ++i) {
                const int s = i % C::kStages;
                if (!(ok = mbar_wait_bounded<false>(&aBar[s], (i / C::kStages) & 1, &abortFlag) && mbar_wait_bounded<false>(&fullBar[s], (i / C::kStages) & 1, &abortFlag))) break;
                tc_fence_after();
                const uint32_t at = smem_u32(ring) + s * C::kStageBytes;
                const uint64_t descX = smem_desc_sw128(at), descA = smem_desc_sw128(at + kAtomBytes);
#pragma unroll
                for (int k = 0; k < 4; ++k) mma_f16(tmemSlot, descX + 2 * k, descA + 2 * k, idesc, (i | k) != 0);
                tc_commit(&emptyBar[s]);
            }
            if (n > 0) {  // the MMAs issued so far, all of them or not
                tc_commit(&doneBar);
                drain(&doneBar, 0);
            }
        }
        __syncwarp();
        // Each CTA of the cluster finishes its share of the rows: the others' sums are stored into its shared memory (nobody waits for a
        // remote load), one cluster barrier, and the rest is local.
        float* part = reinterpret_cast<float*>(ring + C::kStages * C::kStageBytes);
        const int share = kRows / clusterCtas;
        cluster_wait();  // every CTA of the cluster has started (they arrived at the top)
        if (warp < 4) {
            if (n > 0) ok = ok && mbar_wait_bounded<false>(&doneBar, 0, &abortFlag);
            __syncwarp();
            tc_fence_after();
            const uint32_t to = mapa_u32(smem_u32(part + (rank * share + threadIdx.x % share) * kPitch), threadIdx.x / share);
#pragma unroll
            for (int c0 = 0; c0 < R; c0 += 32) {
                uint32_t v[32];
                if (n > 0) {
                    tmem_ld_32x32b_x32(tmemSlot + (static_cast<uint32_t>(warp * 32) << 16) + c0, v);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int c = 0; c < 32 && c0 + c < R; c += 4)
                    st_cluster_v4(to + (c0 + c) * 4, n > 0 ? make_uint4(v[c], v[c + 1], v[c + 2], v[c + 3]) : make_uint4(0u, 0u, 0u, 0u));
            }
        }
        __syncthreads();
        cluster_arrive();
        cluster_wait();
        if (warp < 4) {
            const float scale = p.scale ? p.scale[adapter] : 1.0f;
            const int there = tokens - rank * share;  // rows of this CTA's share that have a token
            if (clusterCtas == 1) finish_rows<T, NB, 1>(part, there, start, p.r, scale, o);
            else if (clusterCtas == 2) finish_rows<T, NB, 2>(part, there, start + rank * share, p.r, scale, o);
            else if (clusterCtas == 4) finish_rows<T, NB, 4>(part, there, start + rank * share, p.r, scale, o);
            else finish_rows<T, NB, 8>(part, there, start + rank * share, p.r, scale, o);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmemSlot, C::kTmemCols);
    }
    if (threadIdx.x == 0 && abortFlag) atomicExch(&g_low_rank_status, 1);
}

// Shared memory of the outer kernel: V's two terms, three blocks of 64 columns of B, three of base (which dst's values replace).
template <int NB> struct Outer {
    static constexpr int kAtoms = rank_pitch(NB) > 64 ? 2 : 1;
    static constexpr int kVBytes = 2 * kAtoms * kAtomBytes, kBBytes = kAtoms * kBlockCols * 128, kYBytes = kRows * 128;
    static constexpr int kBytes = kVBytes + 3 * (kBBytes + kYBytes) + 1024;
};

// The blocks of 64 columns of all tiles are dealt out evenly: CTA c of G takes the blocks from c * total / G to (c + 1) * total / G, which
// touch one tile or two; for each it loads V once and streams B and base.  (With a CTA for each tile and 512 columns the two waves' starts were
// as long as their work: 42 us instead of 31 at 8192 tokens, 4096 columns.)
template <typename T, int NB>
__global__ void __launch_bounds__(kOuterThreads, NB <= 8 ? 2 : 1) low_rank_outer_kernel(const LowRankArgs p, const LowRankScratch o, int tileBound, const __grid_constant__ CUtensorMap mapB,
                          const __grid_constant__ CUtensorMap mapV)
{
    using C = Outer<NB>;
    constexpr int VP = rank_pitch(NB);
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t vBar, bBar[3], freeBar[2], outBar[2];
    __shared__ uint32_t tmemSlot;
    __shared__ int abortFlag;
    uint8_t* sV = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
    uint8_t *sB = sV + C::kVBytes, *sY = sB + 3 * C::kBBytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(&vBar, 1);
        for (int i = 0; i < 3; ++i) mbar_init(&bBar[i], 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&freeBar[i], 8);  // the warps that have read an accumulator
            mbar_init(&outBar[i], 1);
        }
        fence_barrier_init();
        abortFlag = 0;
    }
    if (warp == 8) {
        tmem_alloc(&tmemSlot, 2 * kBlockCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();  // before a dependent launch, which may take tensor memory too, is let in
    tc_fence_after();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4* tiles = static_cast<const int4*>(o.tiles);
    const int perTile = (p.N + kBlockCols - 1) / kBlockCols;
    const int64_t total = static_cast<int64_t>(tiles[tileBound].x) * perTile;
    int64_t pos = total * blockIdx.x / gridDim.x;
    const int64_t end = total * (blockIdx.x + 1) / gridDim.x;
    bool ok = true;
    uint32_t it = 0, segment = 0;  // blocks multiplied so far, and tiles: the barriers' slots and phases go by them
    uint32_t issued = 0;           // blocks whose MMAs were issued
    while (pos < end && ok) {
        const int tileIdx = static_cast<int>(pos / perTile), first = static_cast<int>(pos % perTile);
        const int blocks = static_cast<int>(min(end - pos, static_cast<int64_t>(perTile - first)));
        pos += blocks;
        const int4 tile = tiles[tileIdx];
        const int adapter = tile.x, start = tile.y, tokens = tile.z;
        const int col0 = first * kBlockCols, colEnd = min(p.N, col0 + blocks * kBlockCols);
        if (adapter >= p.L) {
            // tokens without an adapter: base as it is, eight pieces of 16 bytes in flight per thread
            if (p.base != p.dst) {
                const int pieces = (colEnd - col0) / 8, all = tokens * pieces;
                constexpr int kFlight = 8;
                for (int i0 = threadIdx.x; i0 < all; i0 += kOuterThreads * kFlight) {
                    uint4 v[kFlight];
                    T* to[kFlight];
#pragma unroll
                    for (int u = 0; u < kFlight; ++u) {
                        const int i = i0 + u * kOuterThreads;
                        to[u] = nullptr;
                        v[u] = make_uint4(0u, 0u, 0u, 0u);
                        if (i < all) {
                            const int64_t t = p.order[start + i / pieces];
                            const int col = col0 + i % pieces * 8;
                            to[u] = static_cast<T*>(p.dst) + t * p.ldDst + col;
                            if (p.base) v[u] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const T*>(p.base) + t * p.ldBase + col));
                        }
                    }
#pragma unroll
                    for (int u = 0; u < kFlight; ++u)
                        if (to[u]) __stcs(reinterpret_cast<uint4*>(to[u]), v[u]);
                }
            }
            continue;
        }
        if (warp < 8) {
            // A warp owns 32 rows (its quarter of tensor memory) and 32 of a block's 64 columns.  It moves base and dst in 16-byte pieces, four lanes
            // a row; neighbouring quads take rows that differ in bit 2, so that eight lanes meet all banks of the swizzled layout.
            const int quarter = warp & 3, half = warp >> 2, quad = lane >> 2;
            const int moveRow = quarter * 32 + ((quad & 1) << 2 | quad >> 1), movePiece = half * 4 + (lane & 3);
            const uint32_t moveAt = moveRow * 128 + ((movePiece ^ (moveRow & 7)) << 4);
            const T* from[4];
            T* to[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = moveRow + 8 * i;
                const int64_t t = row < tokens ? p.order[start + row] : -1;
                from[i] = t >= 0 && p.base ? static_cast<const T*>(p.base) + t * p.ldBase + col0 + movePiece * 8 : nullptr;
                to[i] = t >= 0 ? static_cast<T*>(p.dst) + t * p.ldDst + col0 + movePiece * 8 : nullptr;
            }
            const int myRow = quarter * 32 + lane;
            const float unit = myRow < tokens ? o.unit[start + myRow] : 0.f;
            const int moveCols = colEnd - col0 - movePiece * 8;  // the piece is inside while its block's column is below
            auto request = [&](int b) {
                if (b * kBlockCols < moveCols) {
                    const uint32_t y = smem_u32(sY) + (it + b) % 3 * C::kYBytes + moveAt;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (from[i]) cp_async16(y + i * 1024, from[i] + b * kBlockCols, true);
                }
                cp_commit();
            };
            request(0);
            request(1);
            for (int b = 0; b < blocks; ++b) {
                const uint32_t n = it + b;
                __syncwarp();  // the warp has read the values of block n - 1 out of the slot that is filled now
                request(b + 2);
                cp_wait<2>();
                ok = mbar_wait_bounded<false>(&outBar[n & 1], (n >> 1) & 1, &abortFlag);
                // base's values of block n, copied by the warp's lanes, are there for all of them; and the lanes give up together
                if (!(ok = __all_sync(0xFFFFFFFFu, ok))) break;
                __syncwarp();
                tc_fence_after();
                uint32_t acc[32];
                tmem_ld_32x32b_x32(tmemSlot + (static_cast<uint32_t>(quarter * 32) << 16) + (n & 1) * kBlockCols + half * 32, acc);
                uint8_t* y = sY + (n % 3) * C::kYBytes;
                tmem_ld_wait();
                tc_fence_before();
                if (lane == 0) mbar_arrive(&freeBar[n & 1]);  // (all lanes have their values: the load is the warp's)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint4* at = reinterpret_cast<uint4*>(y + myRow * 128 + (((half * 4 + j) ^ (lane & 7)) << 4));
                    const uint4 was = p.base ? *at : make_uint4(0u, 0u, 0u, 0u);
                    const uint32_t w[4] = {was.x, was.y, was.z, was.w};
                    float f[8];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float2 v = unpack2<T>(w[q]);
                        f[2 * q] = fmaf(__uint_as_float(acc[j * 8 + 2 * q]), unit, v.x);
                        f[2 * q + 1] = fmaf(__uint_as_float(acc[j * 8 + 2 * q + 1]), unit, v.y);
                    }
                    *at = pack8_sat<T>(f);
                }
                __syncwarp();
                if (b * kBlockCols < moveCols) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (to[i]) __stcs(reinterpret_cast<uint4*>(to[i] + b * kBlockCols), *reinterpret_cast<const uint4*>(y + moveAt + i * 1024));
                }
            }
            cp_wait<0>();
            __syncwarp();  // the slots are filled again for the next tile
        } else if (elect_one()) {
            constexpr uint32_t idesc = idesc_f16(kRows, kBlockCols, std::is_same<T, __half>::value ? 0 : 1);
            const int steps = (p.r + 15) / 16;
            auto done = [&](uint32_t n) { return mbar_wait_bounded<false>(&outBar[n & 1], (n >> 1) & 1, &abortFlag); };  // block n's MMAs
            int asked = 0;  // blocks of B asked for
            bool begun = false;
            auto load_b = [&](int b) {
                if (b >= blocks || it + b >= static_cast<uint32_t>(o.stopB)) return;
                asked = b + 1;
                const uint32_t s = (it + b) % 3;
                mbar_arrive_expect_tx(&bBar[s], C::kBBytes);
#pragma unroll
                for (int ka = 0; ka < C::kAtoms; ++ka)
                    tma_load_2d(sB + s * C::kBBytes + ka * kBlockCols * 128, &mapB, &bBar[s], ka * 64, adapter * p.N + col0 + b * kBlockCols);
            };
            if (it > 0) ok = done(it - 1);  // V and the slots of B are read no more
            if (ok) {
                begun = true;
                mbar_arrive_expect_tx(&vBar, C::kVBytes);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int ka = 0; ka < C::kAtoms; ++ka) tma_load_2d(sV + (h * C::kAtoms + ka) * kAtomBytes, &mapV, &vBar, h * VP + ka * 64, start);
                load_b(0);
                load_b(1);
                ok = mbar_wait_bounded<false>(&vBar, segment & 1, &abortFlag);
            }
            for (int b = 0; b < blocks && ok; ++b) {
                const uint32_t n = it + b;
                if (b > 0 && !(ok = done(n - 1))) break;
                load_b(b + 2);
                if (!(ok = mbar_wait_bounded<false>(&bBar[n % 3], (n / 3) & 1, &abortFlag))) break;
                if (n >= 2 && !(ok = mbar_wait_bounded<false>(&freeBar[n & 1], ((n >> 1) & 1) ^ 1, &abortFlag))) break;
                tc_fence_after();
                const uint32_t v = smem_u32(sV), w = smem_u32(sB) + (n % 3) * C::kBBytes;
                for (int h = 0; h < 2; ++h)
                    for (int k = 0; k < steps; ++k)
                        mma_f16(tmemSlot + (n & 1) * kBlockCols, smem_desc_sw128(v + (h * C::kAtoms + (k >> 2)) * kAtomBytes) + 2 * (k & 3),
                                smem_desc_sw128(w + (k >> 2) * kBlockCols * 128) + 2 * (k & 3), idesc, (h | k) != 0);
                tc_commit(&outBar[n & 1]);
                issued = n + 1;
            }
            if (!ok && begun) {  // no copy may be on its way when the CTA ends
                drain(&vBar, segment & 1);
                for (int b = max(asked - 3, 0); b < asked; ++b) drain(&bBar[(it + b) % 3], ((it + b) / 3) & 1);
            }
        }
        ++segment;
        ok = __all_sync(0xFFFFFFFFu, ok);
        it += blocks;
    }
    __syncwarp();
    if (warp == 8) {  // nor an MMA, should the warps that wait for it have given up
        issued = __reduce_max_sync(0xFFFFFFFFu, issued);
        if (issued > 0) drain(&outBar[(issued - 1) & 1], ((issued - 1) >> 1) & 1);
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmemSlot, 2 * kBlockCols);
    }
    if (threadIdx.x == 0 && abortFlag) atomicExch(&g_low_rank_status, 1);
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

// Clusters of `size` CTAs of the first launch that are resident together (a cluster lies inside one group of SMs, and a CTA takes an SM).
template <typename T, int NB> int resident_clusters(int size)
{
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(size), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = Ring<NB>::kBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(size);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, low_rank_inner_kernel<T, NB>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
    }
    return n;
}

// Devices that these kernels were ever launched (or captured) on: only there is a status word to read.
std::atomic<bool> g_launched[kMaxDevices];

template <typename T, int NB> ascq_status launch_long(const LowRankArgs& p, const LowRankScratch& o, unsigned tiles, cudaStream_t st)
{
    static PerDeviceOnce once;
    static std::atomic<int> resident[kMaxDevices][4];  // clusters of 1, 2, 4, 8
    const int dev = current_device();
    if (!once.done(dev)) {
        ASCQ_CUDA_CHECK(cudaFuncSetAttribute(low_rank_inner_kernel<T, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<NB>::kBytes));
        ASCQ_CUDA_CHECK(cudaFuncSetAttribute(low_rank_outer_kernel<T, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, Outer<NB>::kBytes));
        for (int i = 0; i < 4; ++i) resident[dev][i].store(resident_clusters<T, NB>(1 << i), std::memory_order_relaxed);
        once.mark(dev);
    }
    g_launched[dev].store(true, std::memory_order_relaxed);
    // K is split over a cluster so that the waves of clusters take the least time: a wave's chunks, and about ten more for its start and its end.  How many
    // tiles there are only the device knows; half of the adapters are taken to leave a tile partly filled.
    const int64_t chunks = (p.K + 63) / 64, expected = p.M / kRows + std::min(p.L + 1, p.M) / 2 + 1;
    int cluster = 1;
    int64_t best = INT64_MAX;
    for (int i = 0; i < 4; ++i) {
        const int fit = resident[dev][i].load(std::memory_order_relaxed);
        if (fit <= 0) continue;
        const int64_t cost = (expected + fit - 1) / fit * ((chunks + (1 << i) - 1) / (1 << i) + 10);
        if (cost < best) {
            best = cost;
            cluster = 1 << i;
        }
    }
    constexpr CUtensorMapDataType kType = CU_TENSOR_MAP_DATA_TYPE_UINT16;  // copies only
    CUtensorMap mapA, mapB, mapV;
    ascq_status rc = encode_2d(&mapA, kType, p.a, p.K, static_cast<uint64_t>(p.L) * p.r, static_cast<uint64_t>(p.K) * 2, 64, NB * 8, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_128B, "A");
    if (rc == ASCQ_OK)
        rc = encode_2d(&mapB, kType, p.b, p.r, static_cast<uint64_t>(p.L) * p.N, static_cast<uint64_t>(p.r) * 2, 64, kBlockCols, CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_128B, "B");
    if (rc == ASCQ_OK)
        rc = encode_2d(&mapV, kType, o.v, 2 * rank_pitch(NB), p.M, 4 * rank_pitch(NB), 64, kRows, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                       "inner products");
    if (rc != ASCQ_OK) return rc;
    ASCQ_CUDA_CHECK(launch_pdl(low_rank_inner_kernel<T, NB>, dim3(tiles * cluster), kThreads, Ring<NB>::kBytes, cluster, st, p, o, cluster, mapA));
    // as many CTAs of the second launch as are resident together, at most one per block of columns
    const uint64_t blocks = static_cast<uint64_t>(tiles) * ((p.N + kBlockCols - 1) / kBlockCols);
    const unsigned grid = static_cast<unsigned>(std::min<uint64_t>(blocks, static_cast<uint64_t>(sm_count()) * (NB <= 8 ? 2 : 1)));
    ASCQ_CUDA_CHECK(launch_pdl(low_rank_outer_kernel<T, NB>, dim3(grid), kOuterThreads, Outer<NB>::kBytes, 1, st, p, o, static_cast<int>(tiles), mapB, mapV));
    return ASCQ_OK;
}
// Test hook (ascq_test_withhold_low_rank): the loads that the next call makes of A and B, per CTA; -1: all.
std::atomic<int> g_stopANext{-1}, g_stopBNext{-1};
int stop_of(std::atomic<int>& next)
{
    const int stop = next.exchange(-1);
    return stop < 0 ? INT32_MAX : stop;
}

template <typename T> ascq_status launch_long_typed(const LowRankArgs& p, const LowRankScratch& o, unsigned tiles, cudaStream_t st)
{
    switch (rank_blocks(p.r)) {
        case 2: return launch_long<T, 2>(p, o, tiles, st);
        case 4: return launch_long<T, 4>(p, o, tiles, st);
        case 8: return launch_long<T, 8>(p, o, tiles, st);
        default: return launch_long<T, 16>(p, o, tiles, st);
    }
}

}  // namespace

size_t low_rank_long_tiles_bytes(int64_t tiles) { return static_cast<size_t>(tiles + 1) * 16; }
size_t low_rank_long_inner_bytes(int M, int r) { return static_cast<size_t>(M) * 2 * rank_pitch(rank_blocks(r)) * 2; }

ascq_status low_rank_long(const LowRankArgs& p, bool half, const LowRankScratch& scratch, unsigned tiles, ::CUstream_st* st)
{
    LowRankScratch o = scratch;
    o.stopA = stop_of(g_stopANext);
    o.stopB = stop_of(g_stopBNext);
    return half ? launch_long_typed<__half>(p, o, tiles, st) : launch_long_typed<__nv_bfloat16>(p, o, tiles, st);
}

// Reads and clears this unit's device status word (used by ascq_matmul_status).
ascq_status low_rank_read_status(::CUstream_st* st)
{
    int v = 0, zero = 0;
    if (!g_launched[current_device()].load(std::memory_order_relaxed)) return ASCQ_OK;  // no copy and no wait for programs without adapters
    ASCQ_CUDA_CHECK(cudaMemcpyFromSymbolAsync(&v, g_low_rank_status, sizeof(int), 0, cudaMemcpyDeviceToHost, st));
    ASCQ_CUDA_CHECK(cudaStreamSynchronize(st));
    if (v != 0) {
        ASCQ_CUDA_CHECK(cudaMemcpyToSymbolAsync(g_low_rank_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st));
        return fail(ASCQ_ERR_TIMEOUT, "a bounded wait inside the low-rank adapter kernels expired (status %d)", v);
    }
    return ASCQ_OK;
}
ascq_status low_rank_set_wait_cycles(long long cycles)
{
    ASCQ_CUDA_CHECK(cudaMemcpyToSymbol(ptx::c_waitCycles, &cycles, sizeof(cycles)));
    return ASCQ_OK;
}
}  // namespace ascq

extern "C" ascq_status ascq_test_withhold_low_rank(int chunksOfA, int blocksOfB)
{
    ascq::g_stopANext.store(chunksOfA < 0 ? -1 : chunksOfA);
    ascq::g_stopBNext.store(blocksOfB < 0 ? -1 : blocksOfB);
    return ASCQ_OK;
}
