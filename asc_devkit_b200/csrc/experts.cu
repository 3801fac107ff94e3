// Tokens into expert order and back, around the grouped matmuls:
//   sort      slots (token t, choice j: slot t * k + j) ordered by expert, equal experts in slot order; rows per expert
//   dispatch  rows[rowOfSlot[s]] = src[s / k]                      (any element type; per-token scales alongside)
//   combine   out[t] = sum_j w[t, j] * rows[rowOfSlot[t, j]]       (fp32, j ascending; without weights: the gradient of dispatch)
//   gradient  dRows[rowOfSlot[s]] = w[s] * dOut[t],  dW[s] = <rows[rowOfSlot[s]], dOut[t]>
// Slots without a row (-1, or a number outside the rows) take no part.  Nothing here uses an atomic on a result: every
// sum has a fixed order.
#include "elementwise.cuh"
#include "experts.cuh"
#include "sm100_ptx.cuh"

using namespace ascq;
using namespace ascq::ptx;

namespace ascq {
namespace {

template <typename K, typename... Args>
cudaError_t launch_rows(K kernel, dim3 grid, unsigned block, size_t smem, unsigned cluster, cudaStream_t st, Args... args)
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
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}
__device__ __forceinline__ void pdl_begin()
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---- sort ------------------------------------------------------------------------------------------------------------
// One cluster.  Every warp owns a contiguous run of slots and a private histogram in shared memory, filled 32 slots at a time: a
// ballot per bit of the key finds a step's equal keys (a match instruction takes several times as long when most differ), which
// ranks each slot among the warp's slots of its key.  The histograms are summed over
// the warps and, through distributed shared memory, over the cluster's CTAs: each warp then knows its first position in every key's
// run.  One launch, no scratch memory, and the order of equal keys is the slots' own.
// What bounds it is latency (the slots themselves are a few hundred KB): a warp's numbers are all requested at the start and keys and
// ranks stay in registers (HELD steps of 32 slots).  Longer runs (HELD = 0) count first and walk over the slots a second time.
// 128 slots of 256 experts 2.5 us, 65536 slots of 128 experts 10 us.
template <typename Id> __device__ __forceinline__ int sort_key(const Id* ids, int64_t s, int64_t end, int keys, int outside)
{
    if (s >= end) return -1;
    const Id v = ids[s];
    return v >= 0 && v < static_cast<Id>(keys) ? static_cast<int>(v) : outside;
}
// Rank of each lane's slot among the warp's slots of its key so far; counts the step's slots into `mine`.
__device__ __forceinline__ uint32_t rank_step(uint32_t* mine, int key, int bits)
{
    const int lane = threadIdx.x & 31;
    uint32_t peers = __ballot_sync(0xFFFFFFFFu, key >= 0);
    if (key < 0) peers = ~peers;
    for (int b = 0; b < bits; ++b) {
        const bool mineSet = (key >> b) & 1;
        const uint32_t set = __ballot_sync(0xFFFFFFFFu, mineSet);
        peers &= mineSet ? set : ~set;
    }
    const uint32_t before = key >= 0 ? mine[key] : 0u;
    __syncwarp();
    if (key >= 0 && lane == __ffs(peers) - 1) mine[key] = before + __popc(peers);
    __syncwarp();
    return before + __popc(peers & ((1u << lane) - 1u));
}

template <typename Id, int HELD>
__global__ void __launch_bounds__(1024) key_sort_kernel(int64_t* counts, int32_t* rowOfSlot, int32_t* slotOfRow, const Id* ids, int64_t slots, int keys,
                                                        int outside, int ctas)
{
    extern __shared__ uint32_t smem[];
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t* hist = smem;                    // [warps][keys]: counts, then the slots of the CTA's earlier warps
    uint32_t* total = hist + warps * keys;    // [keys]: this CTA's slots per key (read by the other CTAs)
    uint32_t* before = total + keys;          // [keys]: slots of the key in earlier CTAs
    uint32_t* first = before + keys;          // [keys]: the key's slots in all CTAs, then this CTA's first position in its run
    uint32_t* scan = first + keys;            // [32]
    for (int i = threadIdx.x; i < warps * keys; i += blockDim.x) hist[i] = 0u;
    pdl_begin();

    const int rank = blockIdx.x;
    const int64_t perWarp = ((slots + static_cast<int64_t>(ctas) * warps - 1) / (static_cast<int64_t>(ctas) * warps) + 31) / 32 * 32;
    const int64_t begin = (static_cast<int64_t>(rank) * warps + warp) * perWarp;
    const int64_t end = begin + perWarp < slots ? begin + perWarp : slots;
    uint32_t* mine = hist + warp * keys;
    const int bits = 32 - __clz(keys - 1);  // of the largest key (__clz(0) is 32)
    int key[HELD ? HELD : 1];
    uint32_t place[HELD ? HELD : 1];
    if constexpr (HELD > 0) {
#pragma unroll
        for (int i = 0; i < HELD; ++i) key[i] = sort_key<Id>(ids, begin + 32 * i + lane, end, keys, outside);
    }
    __syncthreads();
    if constexpr (HELD > 0) {
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (begin + 32 * i < end) place[i] = rank_step(mine, key[i], bits);
    } else {
        for (int64_t s = begin; s < end; s += 32) {
            const int k = sort_key<Id>(ids, s + lane, end, keys, outside);
            if (k >= 0) atomicAdd(&mine[k], 1u);  // a count: the order of the additions does not show
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < keys; e += blockDim.x) {
        uint32_t run = 0;
#pragma unroll 8
        for (int w = 0; w < warps; ++w) {
            const uint32_t c = hist[w * keys + e];
            hist[w * keys + e] = run;
            run += c;
        }
        total[e] = run;
    }
    if (ctas > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }
    for (int e = threadIdx.x; e < keys; e += blockDim.x) {
        uint32_t earlier = 0, all = 0;
        if (ctas > 1) {
            const uint32_t at = smem_u32(total + e);
#pragma unroll 8
            for (int c = 0; c < ctas; ++c) {
                uint32_t v;
                asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_u32(at, c)) : "memory");
                if (c < rank) earlier += v;
                all += v;
            }
        } else {
            all = total[e];
        }
        before[e] = earlier;
        first[e] = all;
        if (rank == 0) counts[e] = static_cast<int64_t>(all);
    }
    __syncwarp();
    if (ctas > 1) cluster_arrive();  // no CTA may end while another still reads its totals; the wait is at the end
    __syncthreads();
    // exclusive scan of `first` over the keys: each thread takes keys / threads consecutive ones (rounded up)
    const int per = (keys + blockDim.x - 1) / blockDim.x;
    uint32_t sum = 0;
    for (int i = 0; i < per; ++i) {
        const int e = threadIdx.x * per + i;
        if (e < keys) sum += first[e];
    }
    uint32_t incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    const uint32_t sums = lane < warps ? scan[lane] : 0u;
    uint32_t base = lane < warp ? sums : 0u, kept = sums;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        base += __shfl_xor_sync(0xFFFFFFFFu, base, o);
        kept += __shfl_xor_sync(0xFFFFFFFFu, kept, o);
    }
    uint32_t run = base + incl - sum;
    for (int i = 0; i < per; ++i) {
        const int e = threadIdx.x * per + i;
        if (e < keys) {
            const uint32_t c = first[e];
            first[e] = run + before[e];
            run += c;
        }
    }
    __syncthreads();
    auto put = [&](int64_t s, int k, uint32_t at) {
        if (s >= end) return;
        const uint32_t pos = k >= 0 ? first[k] + at : 0u;
        if (rowOfSlot) rowOfSlot[s] = k >= 0 ? static_cast<int32_t>(pos) : -1;
        if (slotOfRow && k >= 0) slotOfRow[pos] = static_cast<int32_t>(s);
    };
    if constexpr (HELD > 0) {
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (begin + 32 * i < end) put(begin + 32 * i + lane, key[i], (key[i] >= 0 ? mine[key[i]] : 0u) + place[i]);
    } else {
        for (int64_t s = begin; s < end; s += 32) {
            const int k = sort_key<Id>(ids, s + lane, end, keys, outside);
            put(s + lane, k, rank_step(mine, k, bits));  // `mine` holds the earlier warps' slots, then this warp's too
        }
    }
    if (slotOfRow)
        for (int64_t r = kept + static_cast<int64_t>(rank) * blockDim.x + threadIdx.x; r < slots; r += static_cast<int64_t>(ctas) * blockDim.x) slotOfRow[r] = -1;
    __syncwarp();
    if (ctas > 1) cluster_wait();
}

constexpr unsigned kSortThreads = 1024;

// Per-device set-up; *most receives the largest cluster the device can place (16 CTAs are beyond the portable size of 8).
template <typename Id, int HELD> ascq_status sort_setup(int* most)
{
    static PerDeviceOnce once, wide;
    const int dev = current_device();
    if (!once.done(dev)) {
        const int smem = (static_cast<int>(kSortThreads / 32 + 3) * kMaxSortKeys + 32) * 4;
        ASCQ_CUDA_CHECK(cudaFuncSetAttribute(key_sort_kernel<Id, HELD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        ASCQ_CUDA_CHECK(cudaFuncSetAttribute(key_sort_kernel<Id, HELD>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(16, 1, 1);
        cfg.blockDim = dim3(kSortThreads, 1, 1);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 16;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, key_sort_kernel<Id, HELD>, &cfg) == cudaSuccess && clusters > 0) wide.mark(dev);
        else cudaGetLastError();  // not placeable: the portable size it is
        once.mark(dev);
    }
    *most = wide.done(dev) ? 16 : 8;
    return ASCQ_OK;
}

template <typename Id, int HELD> ascq_status launch_key_sort_held(int64_t* counts, int32_t* rowOfSlot, int32_t* slotOfRow, const void* ids, int64_t slots,
                                                                  int keys, int outside, unsigned threads, int ctas, cudaStream_t st)
{
    const size_t smem = (static_cast<size_t>(threads / 32 + 3) * keys + 32) * 4;
    ASCQ_CUDA_CHECK(launch_rows(key_sort_kernel<Id, HELD>, dim3(ctas), threads, smem, ctas, st, counts, rowOfSlot, slotOfRow, static_cast<const Id*>(ids), slots,
                                keys, outside, ctas));
    return ASCQ_OK;
}
template <typename Id> ascq_status launch_key_sort_typed(int64_t* counts, int32_t* rowOfSlot, int32_t* slotOfRow, const void* ids, int64_t slots, int keys,
                                                         int outside, cudaStream_t st)
{
    // A CTA takes 1024 slots (one step of its warps) while the cluster can grow.  Measured, 64 keys, us: 1024 slots 4.1 with one CTA (4.7
    // with two), 4096 slots 5.1 / 6.2 / 7.5 with four / two / one, 16384 slots 5.5 / 6.7 / 8.6 with 16 / 8 / 4, 65536 slots 9.9 / 14.1 with 16 / 8.
    unsigned threads = 256;
    while (threads < kSortThreads && slots > threads) threads *= 2;
    int most[4] = {};
    ascq_status rc = sort_setup<Id, 1>(&most[0]);
    if (rc == ASCQ_OK) rc = sort_setup<Id, 4>(&most[1]);
    if (rc == ASCQ_OK) rc = sort_setup<Id, 8>(&most[2]);
    if (rc == ASCQ_OK) rc = sort_setup<Id, 0>(&most[3]);
    if (rc != ASCQ_OK) return rc;
    const int cap = std::min(std::min(most[0], most[1]), std::min(most[2], most[3]));
    int ctas = 1;
    while (ctas < cap && slots > static_cast<int64_t>(ctas) * kSortThreads) ctas *= 2;
    const int64_t steps = (slots + static_cast<int64_t>(ctas) * threads - 1) / (static_cast<int64_t>(ctas) * threads);  // of 32 slots, of a warp
    if (steps <= 1) return launch_key_sort_held<Id, 1>(counts, rowOfSlot, slotOfRow, ids, slots, keys, outside, threads, ctas, st);
    if (steps <= 4) return launch_key_sort_held<Id, 4>(counts, rowOfSlot, slotOfRow, ids, slots, keys, outside, threads, ctas, st);
    if (steps <= 8) return launch_key_sort_held<Id, 8>(counts, rowOfSlot, slotOfRow, ids, slots, keys, outside, threads, ctas, st);
    return launch_key_sort_held<Id, 0>(counts, rowOfSlot, slotOfRow, ids, slots, keys, outside, threads, ctas, st);
}

// ---- dispatch ---------------------------------------------------------------------------------------------------------
struct DispatchArgs {
    uint8_t* dst;
    const uint8_t* src;
    uint8_t* dstScale;        // may be null
    const uint8_t* srcScale;
    size_t rowBytes, ldSrc, scaleBytes;
    const int32_t* rowOfSlot;
    int64_t tokens, rows;
    int k;
    uint32_t segments;        // of 32 * dispatch_vecs vectors in a row
};
// accesses of a lane that are in flight together: narrow ones (rows of odd sizes) need more of them
template <typename V> constexpr int dispatch_vecs() { return sizeof(V) == 16 ? 4 : sizeof(V) == 4 ? 8 : 16; }

// A warp takes a segment of a token's row: it reads the segment once and writes it to each of the token's rows.  What bounds it is HBM's
// write side: 8192 tokens x 8 int8 rows of 7168 bytes in 84 us = 6.3 TB/s of 0.53 GB; E4M3 rows with their 224 scale bytes 88 us,
// packed fp4 rows with theirs 49 us (of 0.28 GB).  Rows of an odd number of bytes move in single bytes: 7167 of them 154 us.
template <typename V> __global__ void __launch_bounds__(256) dispatch_kernel(const DispatchArgs a)
{
    constexpr int kDispatchVecs = dispatch_vecs<V>();
    pdl_begin();
    const int lane = threadIdx.x & 31;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int64_t t = item / a.segments;
    const uint32_t seg = static_cast<uint32_t>(item % a.segments);
    if (t >= a.tokens) return;
    const size_t nvec = a.rowBytes / sizeof(V), v0 = static_cast<size_t>(seg) * 32 * kDispatchVecs + lane;
    const V* from = reinterpret_cast<const V*>(a.src + static_cast<size_t>(t) * a.ldSrc);
    V x[kDispatchVecs];
#pragma unroll
    for (int u = 0; u < kDispatchVecs; ++u)
        if (v0 + u * 32 < nvec) x[u] = __ldcs(from + v0 + u * 32);
    for (int j0 = 0; j0 < a.k; j0 += 32) {
        const int32_t mine = j0 + lane < a.k ? a.rowOfSlot[t * a.k + j0 + lane] : -1;
        for (int j = 0; j < 32 && j0 + j < a.k; ++j) {
            const int32_t r = __shfl_sync(0xFFFFFFFFu, mine, j);
            if (r < 0 || r >= a.rows) continue;
            V* to = reinterpret_cast<V*>(a.dst + static_cast<size_t>(r) * a.rowBytes);
#pragma unroll
            for (int u = 0; u < kDispatchVecs; ++u)
                if (v0 + u * 32 < nvec) __stcs(to + v0 + u * 32, x[u]);
            if (seg == 0 && a.dstScale)
                for (size_t i = lane; i < a.scaleBytes; i += 32) a.dstScale[static_cast<size_t>(r) * a.scaleBytes + i] = a.srcScale[static_cast<size_t>(t) * a.scaleBytes + i];
        }
    }
}

// ---- combine ----------------------------------------------------------------------------------------------------------
struct CombineArgs {
    void* out;             // combine: [tokens, h]
    void* gradRows;        // gradient: [rows, h], may be null
    float* gradWeights;    // gradient: [tokens, k], may be null
    const void* gradOut;   // gradient: [tokens, h]
    const void* in;        // [rows, h]
    const int32_t* rowOfSlot;
    const float* weights;  // may be null (all 1)
    int64_t tokens, rows, h;
    int k;
    uint32_t segments;
};

// VEC consecutive elements of T as floats: VEC * sizeof(T) bytes in one access of up to 16 bytes
template <typename T, int VEC> __device__ __forceinline__ Pack<T, VEC> load_v(const T* p)
{
    if constexpr (sizeof(T) * VEC >= 4) return load_pack<T, VEC, true>(p);
    else return Pack<T, VEC>{{*p}};
}
template <typename T, int VEC> __device__ __forceinline__ void load_f(const T* p, float (&f)[VEC])
{
    const Pack<T, VEC> v = load_v<T, VEC>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = to_f32<T>(v.v[i]);
}
template <typename T> __device__ __forceinline__ T narrow_sat(float f)
{
    if constexpr (std::is_same<T, float>::value) return f;
    else if constexpr (std::is_same<T, __half>::value) return f32_to_f16_sat(f);
    else return f32_to_bf16_sat(f);
}
template <typename T, int VEC> __device__ __forceinline__ void store_f(T* p, const float (&f)[VEC])
{
    if constexpr (sizeof(T) * VEC >= 4) {
        Pack<T, VEC> v;
        if constexpr (sizeof(T) == 2) {
            uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) w[i] = std::is_same<T, __half>::value ? pack_f16x2_sat(f[2 * i], f[2 * i + 1]) : pack_bf16x2_sat(f[2 * i], f[2 * i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v.v[i] = narrow_sat<T>(f[i]);
        }
        store_pack<T, VEC>(p, v);
    } else {
        *p = narrow_sat<T>(f[0]);
    }
}

// vectors of a lane: 16 bytes of two, or of what a row of an odd size allows more
template <int VEC> constexpr int combine_vecs() { return VEC >= 4 ? 2 : VEC == 2 ? 4 : 8; }

// A warp takes a segment of a token's output and adds up the token's rows, four rows requested at a time.  HBM bound: 8192 tokens x 8 rows of 7168
// bf16 in 171 us = 6.2 TB/s of 1.06 GB.
template <typename T, int VEC> __global__ void __launch_bounds__(256) combine_kernel(const CombineArgs a)
{
    constexpr int kCombineVecs = combine_vecs<VEC>();
    pdl_begin();
    const int lane = threadIdx.x & 31;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int64_t t = item / a.segments;
    const uint32_t seg = static_cast<uint32_t>(item % a.segments);
    if (t >= a.tokens) return;
    const int64_t c0 = (static_cast<int64_t>(seg) * 32 * kCombineVecs + lane) * VEC;
    float acc[kCombineVecs][VEC] = {};
    for (int j0 = 0; j0 < a.k; j0 += 32) {
        int32_t mine = -1;
        float wMine = 1.0f;
        if (j0 + lane < a.k) {
            mine = a.rowOfSlot[t * a.k + j0 + lane];
            if (a.weights) wMine = a.weights[t * a.k + j0 + lane];
        }
        const int jn = a.k - j0 < 32 ? a.k - j0 : 32;
#pragma unroll 4
        for (int j = 0; j < jn; ++j) {
            const int32_t r = __shfl_sync(0xFFFFFFFFu, mine, j);
            const float w = __shfl_sync(0xFFFFFFFFu, wMine, j);
            if (r < 0 || r >= a.rows) continue;
            const T* from = static_cast<const T*>(a.in) + static_cast<int64_t>(r) * a.h;
#pragma unroll
            for (int u = 0; u < kCombineVecs; ++u) {
                const int64_t c = c0 + u * 32 * VEC;
                if (c < a.h) {
                    float f[VEC];
                    load_f<T, VEC>(from + c, f);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[u][i] = fmaf(w, f[i], acc[u][i]);
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < kCombineVecs; ++u) {
        const int64_t c = c0 + u * 32 * VEC;
        if (c < a.h) store_f<T, VEC>(static_cast<T*>(a.out) + t * a.h + c, acc[u]);
    }
}

// ---- gradient of combine --------------------------------------------------------------------------------------------------
// One CTA per token.  A thread requests its vectors of kGradRows of the token's rows together; gradOut's row is read again (from
// L1 or L2) for the next kGradRows.  What bounds it is how many requests an SM has in flight, so the rows per step trade against
// occupancy: at 8192 tokens, k = 8, h = 4096 in bf16 (177 us at the copy rate) 187 us with 4 rows and 64 registers, 213 with 2 rows
// and 40, 196 with 4 rows and 80, 249 with 8 rows and 120; CTAs of 128 threads rather than 256 (193 us) or 64 (198 us).  (All on one box;
// on another the form taken has 193 us.  Rows of odd sizes: 4096 x 4 x 2048 25 us, x 2047 55, x 2046 61.)
constexpr int kGradRows = 4, kGradThreads = 128;

template <typename T, int VEC> __global__ void __launch_bounds__(kGradThreads, 8) combine_grad_kernel(const CombineArgs a)
{
    constexpr int U = VEC >= 4 ? 1 : VEC == 2 ? 2 : 4;  // vectors of a thread per step: narrow ones (rows of odd sizes) need more in flight
    __shared__ float part[kGradThreads / 32][kGradRows];
    pdl_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int64_t t = blockIdx.x;
    const T* dOut = static_cast<const T*>(a.gradOut) + t * a.h;
    for (int j0 = 0; j0 < a.k; j0 += kGradRows) {
        int32_t r[kGradRows];
        float w[kGradRows], dot[kGradRows] = {};
#pragma unroll
        for (int j = 0; j < kGradRows; ++j) {
            r[j] = j0 + j < a.k ? a.rowOfSlot[t * a.k + j0 + j] : -1;
            if (r[j] >= a.rows) r[j] = -1;
            w[j] = a.weights && j0 + j < a.k ? a.weights[t * a.k + j0 + j] : 1.0f;
        }
        const int64_t width = static_cast<int64_t>(blockDim.x) * VEC;
        for (int64_t c0 = static_cast<int64_t>(threadIdx.x) * VEC; c0 < a.h; c0 += U * width) {
            Pack<T, VEC> dv[U], v[U][kGradRows];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t c = c0 + u * width;
                if (c >= a.h) continue;
                dv[u] = load_v<T, VEC>(dOut + c);
                if (a.gradWeights) {
#pragma unroll
                    for (int j = 0; j < kGradRows; ++j)
                        if (r[j] >= 0) v[u][j] = load_v<T, VEC>(static_cast<const T*>(a.in) + static_cast<int64_t>(r[j]) * a.h + c);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t c = c0 + u * width;
                if (c >= a.h) continue;
                float d[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) d[i] = to_f32<T>(dv[u].v[i]);
                if (a.gradRows) {
#pragma unroll
                    for (int j = 0; j < kGradRows; ++j) {
                        if (r[j] < 0) continue;
                        float g[VEC];
#pragma unroll
                        for (int i = 0; i < VEC; ++i) g[i] = __fmul_rn(w[j], d[i]);
                        store_f<T, VEC>(static_cast<T*>(a.gradRows) + static_cast<int64_t>(r[j]) * a.h + c, g);
                    }
                }
                if (a.gradWeights) {
#pragma unroll
                    for (int j = 0; j < kGradRows; ++j) {
                        if (r[j] < 0) continue;
#pragma unroll
                        for (int i = 0; i < VEC; ++i) dot[j] = fmaf(to_f32<T>(v[u][j].v[i]), d[i], dot[j]);
                    }
                }
            }
        }
        if (a.gradWeights) {
#pragma unroll
            for (int j = 0; j < kGradRows; ++j)
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) dot[j] += __shfl_xor_sync(0xFFFFFFFFu, dot[j], o);
            if (lane == 0)
#pragma unroll
                for (int j = 0; j < kGradRows; ++j) part[warp][j] = dot[j];
            __syncthreads();
            if (threadIdx.x < kGradRows && j0 + static_cast<int>(threadIdx.x) < a.k) {
                float s = 0.f;
                for (int i = 0; i < warps; ++i) s += part[i][threadIdx.x];
                a.gradWeights[t * a.k + j0 + threadIdx.x] = s;
            }
            __syncthreads();
        }
    }
}

bool float_type(ascq_dtype t) { return t == ASCQ_DT_F16 || t == ASCQ_DT_BF16 || t == ASCQ_DT_F32; }

// The checks that dispatch, combine and the gradient share.
ascq_status check_slots(const int32_t* rowOfSlot, int64_t tokens, int k, int64_t rows)
{
    if (tokens < 0 || rows < 0 || k <= 0) return fail(ASCQ_ERR_INVALID_ARG, "tokens and rows must not be negative and k must be positive");
    if (tokens > 0x7FFFFFFFll / k || rows > 0x7FFFFFFFll) return fail(ASCQ_ERR_INVALID_ARG, "tokens * k and rows must be below 2^31");
    if (tokens && (reinterpret_cast<uintptr_t>(rowOfSlot) & 3u)) return fail(ASCQ_ERR_ALIGNMENT, "rowOfSlot is not aligned to its element type");
    return ASCQ_OK;
}

}  // namespace

ascq_status launch_key_sort(int64_t* counts, int32_t* rowOfSlot, int32_t* slotOfRow, const void* ids, bool ids64, int64_t slots, int keys, int outside,
                            ::CUstream_st* st)
{
    return ids64 ? launch_key_sort_typed<int64_t>(counts, rowOfSlot, slotOfRow, ids, slots, keys, outside, st)
                 : launch_key_sort_typed<int32_t>(counts, rowOfSlot, slotOfRow, ids, slots, keys, outside, st);
}
}  // namespace ascq

extern "C" ascq_status ascq_expert_sort(int64_t* counts, int32_t* rowOfSlot, int32_t* slotOfRow, const void* expertIds, ascq_dtype idT, int64_t slots,
                                        int numExperts, void* stream)
{
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (idT != ASCQ_DT_I32 && idT != ASCQ_DT_I64) return fail(ASCQ_ERR_UNSUPPORTED, "expertIds must be int32 or int64");
    if (numExperts < 1 || numExperts > kMaxSortKeys) return fail(ASCQ_ERR_INVALID_ARG, "numExperts is %d, which must be in [1, %d]", numExperts, kMaxSortKeys);
    if (slots < 0 || slots > 0x7FFFFFFFll) return fail(ASCQ_ERR_INVALID_ARG, "slots must be in [0, 2^31)");
    if (!counts || (slots && (!rowOfSlot || !expertIds))) return fail(ASCQ_ERR_INVALID_ARG, "counts, rowOfSlot and expertIds must not be NULL");
    const size_t idBytes = idT == ASCQ_DT_I64 ? 8 : 4, n = static_cast<size_t>(slots);
    if ((reinterpret_cast<uintptr_t>(counts) & 7u) || (reinterpret_cast<uintptr_t>(expertIds) & (idBytes - 1)) || (reinterpret_cast<uintptr_t>(rowOfSlot) & 3u) ||
        (reinterpret_cast<uintptr_t>(slotOfRow) & 3u))
        return fail(ASCQ_ERR_ALIGNMENT, "a tensor is not aligned to its element type");
    const void* p[4] = {counts, rowOfSlot, slotOfRow, expertIds};
    const size_t b[4] = {static_cast<size_t>(numExperts) * 8, n * 4, n * 4, n * idBytes};
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < i; ++j)
            if (spans_overlap(p[i], b[i], p[j], b[j])) return fail(ASCQ_ERR_INVALID_ARG, "counts, rowOfSlot, slotOfRow and expertIds must not overlap");
    if (slots == 0) {
        ASCQ_CUDA_CHECK(cudaMemsetAsync(counts, 0, static_cast<size_t>(numExperts) * 8, st));
        return ASCQ_OK;
    }
    return launch_key_sort(counts, rowOfSlot, slotOfRow, expertIds, idT == ASCQ_DT_I64, slots, numExperts, -1, st);
}

extern "C" ascq_status ascq_expert_dispatch(void* dst, const void* src, size_t rowBytes, size_t ldSrcBytes, void* dstScale, const void* srcScale,
                                            size_t scaleRowBytes, const int32_t* rowOfSlot, int64_t tokens, int k, int64_t rows, void* stream)
{
    ascq_status rc = check_slots(rowOfSlot, tokens, k, rows);
    if (rc != ASCQ_OK) return rc;
    if (ldSrcBytes == 0) ldSrcBytes = rowBytes;
    if (ldSrcBytes < rowBytes) return fail(ASCQ_ERR_INVALID_ARG, "the row pitch of src is smaller than its rows");
    if ((dstScale == nullptr) != (srcScale == nullptr)) return fail(ASCQ_ERR_INVALID_ARG, "dstScale and srcScale must both be given or both be NULL");
    constexpr size_t kMost = size_t{1} << 32;  // 2^31 rows of it are below 2^64
    if (rowBytes > kMost || ldSrcBytes > kMost || scaleRowBytes > kMost) return fail(ASCQ_ERR_INVALID_ARG, "a row or its pitch is longer than 2^32 bytes");
    if (tokens == 0 || rows == 0 || (rowBytes == 0 && !dstScale)) return ASCQ_OK;
    if ((rowBytes && (!dst || !src)) || !rowOfSlot) return fail(ASCQ_ERR_INVALID_ARG, "dst, src and rowOfSlot must not be NULL");
    if (dstScale && scaleRowBytes == 0) return fail(ASCQ_ERR_INVALID_ARG, "scaleRowBytes must be positive when scales are given");
    const size_t T = static_cast<size_t>(tokens), R = static_cast<size_t>(rows);
    const void* p[5] = {dst, dstScale, src, srcScale, rowOfSlot};
    const size_t b[5] = {R * rowBytes, dstScale ? R * scaleRowBytes : 0, (T - 1) * ldSrcBytes + rowBytes, srcScale ? T * scaleRowBytes : 0, T * k * 4};
    for (int i = 0; i < 2; ++i)
        for (int j = i + 1; j < 5; ++j)
            if (spans_overlap(p[i], b[i], p[j], b[j])) return fail(ASCQ_ERR_INVALID_ARG, "an output overlaps another tensor of the call");

    DispatchArgs a{static_cast<uint8_t*>(dst), static_cast<const uint8_t*>(src), static_cast<uint8_t*>(dstScale), static_cast<const uint8_t*>(srcScale),
                   rowBytes, ldSrcBytes, scaleRowBytes, rowOfSlot, tokens, rows, k, 0};
    // the widest access that every row of both tensors is aligned to
    const uintptr_t all = reinterpret_cast<uintptr_t>(dst) | reinterpret_cast<uintptr_t>(src) | rowBytes | ldSrcBytes;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto run = [&](auto tag) -> ascq_status {
        using V = decltype(tag);
        const size_t nvec = rowBytes / sizeof(V), per = 32 * dispatch_vecs<V>();
        a.segments = std::max(static_cast<uint32_t>((nvec + per - 1) / per), 1u);  // the first one takes the scales, which empty rows may have too
        const int64_t ctas = (tokens * static_cast<int64_t>(a.segments) + 7) / 8;
        if (ctas > 0x7FFFFFFFll) return fail(ASCQ_ERR_INVALID_ARG, "the rows are too long for one launch");
        ASCQ_CUDA_CHECK(launch_rows(dispatch_kernel<V>, dim3(static_cast<unsigned>(ctas)), 256, 0, 1, st, a));
        return ASCQ_OK;
    };
    if (all % 16 == 0) return run(uint4{});
    if (all % 4 == 0) return run(uint32_t{});
    if (all % 2 == 0) return run(static_cast<unsigned short>(0));
    return run(static_cast<unsigned char>(0));
}

extern "C" ascq_status ascq_expert_combine(void* dst, const void* in, ascq_dtype T, const int32_t* rowOfSlot, const float* weights, int64_t tokens, int k,
                                           int64_t rows, int64_t h, void* stream)
{
    ascq_status rc = check_slots(rowOfSlot, tokens, k, rows);
    if (rc != ASCQ_OK) return rc;
    if (!float_type(T)) return fail(ASCQ_ERR_UNSUPPORTED, "rows must be half, bfloat16_t or float");
    if (h < 0 || h > 0x7FFFFFFFll) return fail(ASCQ_ERR_INVALID_ARG, "h must be in [0, 2^31)");
    if (tokens == 0 || h == 0) return ASCQ_OK;
    if (!dst || (rows && !in) || !rowOfSlot) return fail(ASCQ_ERR_INVALID_ARG, "dst, rows and rowOfSlot must not be NULL");
    const size_t es = dtype_size(T), N = static_cast<size_t>(tokens);
    const uintptr_t all = reinterpret_cast<uintptr_t>(dst) | reinterpret_cast<uintptr_t>(in) | static_cast<uintptr_t>(h) * es;
    if (all % es || (reinterpret_cast<uintptr_t>(weights) & 3u)) return fail(ASCQ_ERR_ALIGNMENT, "a tensor is not aligned to its element type");
    const void* p[4] = {dst, in, weights, rowOfSlot};
    const size_t b[4] = {N * h * es, static_cast<size_t>(rows) * h * es, weights ? N * k * 4 : 0, N * k * 4};
    for (int j = 1; j < 4; ++j)
        if (spans_overlap(p[0], b[0], p[j], b[j])) return fail(ASCQ_ERR_INVALID_ARG, "dst overlaps another tensor of the call");
    CombineArgs a{};
    a.out = dst; a.in = in; a.rowOfSlot = rowOfSlot; a.weights = weights; a.tokens = tokens; a.rows = rows; a.h = h; a.k = k;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto run = [&](auto kernel, int vec) -> ascq_status {
        const int64_t per = 32ll * (vec >= 4 ? combine_vecs<8>() : vec == 2 ? combine_vecs<2>() : combine_vecs<1>()) * vec;
        a.segments = static_cast<uint32_t>((h + per - 1) / per);
        const int64_t ctas = (tokens * static_cast<int64_t>(a.segments) + 7) / 8;
        if (ctas > 0x7FFFFFFFll) return fail(ASCQ_ERR_INVALID_ARG, "the rows are too long for one launch");
        ASCQ_CUDA_CHECK(launch_rows(kernel, dim3(static_cast<unsigned>(ctas)), 256, 0, 1, st, a));
        return ASCQ_OK;
    };
    const bool vec = all % 16 == 0, even = all % 4 == 0;
    if (T == ASCQ_DT_F16) return vec ? run(combine_kernel<__half, 8>, 8) : even ? run(combine_kernel<__half, 2>, 2) : run(combine_kernel<__half, 1>, 1);
    if (T == ASCQ_DT_BF16)
        return vec ? run(combine_kernel<__nv_bfloat16, 8>, 8) : even ? run(combine_kernel<__nv_bfloat16, 2>, 2) : run(combine_kernel<__nv_bfloat16, 1>, 1);
    return vec ? run(combine_kernel<float, 4>, 4) : run(combine_kernel<float, 1>, 1);
}

extern "C" ascq_status ascq_expert_combine_grad(void* gradRows, float* gradWeights, const void* gradOut, const void* in, ascq_dtype T, const int32_t* rowOfSlot,
                                                const float* weights, int64_t tokens, int k, int64_t rows, int64_t h, void* stream)
{
    ascq_status rc = check_slots(rowOfSlot, tokens, k, rows);
    if (rc != ASCQ_OK) return rc;
    if (!float_type(T)) return fail(ASCQ_ERR_UNSUPPORTED, "rows must be half, bfloat16_t or float");
    if (h < 0 || h > 0x7FFFFFFFll) return fail(ASCQ_ERR_INVALID_ARG, "h must be in [0, 2^31)");
    if (tokens == 0 || ((rows == 0 || h == 0) && !gradWeights)) return ASCQ_OK;  // (empty tensors have no address)
    if (!gradRows && !gradWeights) return fail(ASCQ_ERR_INVALID_ARG, "gradRows and gradWeights are both NULL");
    if ((h && !gradOut) || !rowOfSlot || (gradWeights && rows && h && !in)) return fail(ASCQ_ERR_INVALID_ARG, "gradOut, rows and rowOfSlot must not be NULL");
    const size_t es = dtype_size(T), N = static_cast<size_t>(tokens);
    const uintptr_t all = reinterpret_cast<uintptr_t>(gradRows) | reinterpret_cast<uintptr_t>(gradOut) | (gradWeights ? reinterpret_cast<uintptr_t>(in) : 0) |
                          static_cast<uintptr_t>(h) * es;
    if (all % es || (reinterpret_cast<uintptr_t>(weights) & 3u) || (reinterpret_cast<uintptr_t>(gradWeights) & 3u))
        return fail(ASCQ_ERR_ALIGNMENT, "a tensor is not aligned to its element type");
    const size_t rowsBytes = static_cast<size_t>(rows) * h * es;
    const void* p[6] = {gradRows, gradWeights, gradOut, gradWeights ? in : nullptr, weights, rowOfSlot};
    const size_t b[6] = {rowsBytes, N * k * 4, N * h * es, rowsBytes, N * k * 4, N * k * 4};
    for (int i = 0; i < 2; ++i)
        for (int j = i + 1; j < 6; ++j)
            if (spans_overlap(p[i], b[i], p[j], b[j])) return fail(ASCQ_ERR_INVALID_ARG, "an output overlaps another tensor of the call");
    CombineArgs a{};
    a.gradRows = gradRows; a.gradWeights = gradWeights; a.gradOut = gradOut; a.in = in; a.rowOfSlot = rowOfSlot; a.weights = weights;
    a.tokens = tokens; a.rows = rows; a.h = h; a.k = k;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto run = [&](auto kernel, int vec) -> ascq_status {
        const int64_t nvec = (h + vec - 1) / vec;
        const int64_t steps = std::max<int64_t>((nvec + kGradThreads - 1) / kGradThreads, 1);  // of a thread along the row; the CTA is no wider than they need
        const unsigned block = std::max(static_cast<unsigned>((nvec + steps - 1) / steps + 31) / 32 * 32, 32u);
        ASCQ_CUDA_CHECK(launch_rows(kernel, dim3(static_cast<unsigned>(tokens)), block, 0, 1, st, a));
        return ASCQ_OK;
    };
    const bool vec = all % 16 == 0, even = all % 4 == 0;
    if (T == ASCQ_DT_F16)
        return vec ? run(combine_grad_kernel<__half, 8>, 8) : even ? run(combine_grad_kernel<__half, 2>, 2) : run(combine_grad_kernel<__half, 1>, 1);
    if (T == ASCQ_DT_BF16)
        return vec ? run(combine_grad_kernel<__nv_bfloat16, 8>, 8) : even ? run(combine_grad_kernel<__nv_bfloat16, 2>, 2) : run(combine_grad_kernel<__nv_bfloat16, 1>, 1);
    return vec ? run(combine_grad_kernel<float, 4>, 4) : run(combine_grad_kernel<float, 1>, 1);
}
