// Device-side MoE token permutation (sm_100a): per-expert token lists built
// from the router's top-k on the GPU.
//
// Reference: the host loop of forward_chunk_post_gathered
// (src/ds3_engine.c:933-965), which reads idx/scores back to the host every
// layer (:1256-1261) and writes, for expert ex, the tokens that chose it to
// ids[ex * M + j] (j = running count, so tokens in ascending order, each
// token's k slots in order) and their scores alongside; counts[ex] = j.
//
// One CTA per expert, all experts in parallel. CTA ex walks the T*K
// (token, slot) entries in entry order, 4096 at a time, 4 consecutive entries
// per thread: each thread counts its hits, one CTA-wide exclusive scan (two
// warp scans) gives every hit its rank, and a running base carries over
// between passes. Every hit lands at ids[ex*cap + j] in the
// engine's order, with no atomics and no memory beyond the outputs.
// slot_of[t*K+k] = ex*cap + j is written by the CTA of the entry's expert; it
// is the row map moe_combine_residual takes to read expert outputs laid out
// per expert. CTA 0 also flags entries whose expert id is out of range.
#include "common.cuh"
#include "launch.h"

namespace ds3 {
namespace {

constexpr int kRouteThreads = 1024;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kPerThread = 4;                              // consecutive entries per thread
constexpr int kRouteChunk = kRouteThreads * kPerThread;    // 4096 = 512 tokens x top-8 in one pass

__global__ void __launch_bounds__(kRouteThreads) moe_expert_lists_k(
    const int32_t *idx, const float *scores, int32_t *counts, int32_t *ids, float *gscores, int32_t *slot_of,
    int64_t n_entries, int n_used, int n_expert, int64_t cap, unsigned *err)
{
    __shared__ int32_t wpre[kRouteWarps];
    __shared__ int32_t total;
    pdl_wait();
    pdl_trigger();
    const int ex = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int64_t base = 0;
    for (int64_t s0 = 0; s0 < n_entries; s0 += kRouteChunk) {
        // Entries s0 + 4*tid .. +3: ids and scores are loaded together, before
        // either is used, so the pass costs one memory round trip.
        const int64_t i0 = s0 + (int64_t)kPerThread * tid;
        int ev[kPerThread];
        float sv[kPerThread];
#pragma unroll
        for (int c = 0; c < kPerThread; c++) {
            const bool in = i0 + c < n_entries;
            ev[c] = in ? idx[i0 + c] : -1;
            sv[c] = in ? scores[i0 + c] : 0.0f;
        }
        int mine = 0;
#pragma unroll
        for (int c = 0; c < kPerThread; c++) {
            mine += ev[c] == ex;
            if (ex == 0 && i0 + c < n_entries && (ev[c] < 0 || ev[c] >= n_expert)) {
                flag_error(err, kErrBadId);
                if (slot_of) slot_of[i0 + c] = -1;
            }
        }
        // Exclusive scan of the hit counts over the CTA, in entry order.
        int inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(kFull, inc, o);
            if (lane >= o) inc += y;
        }
        if (lane == 31) wpre[warp] = inc;
        __syncthreads();
        if (warp == 0) {
            const int v = wpre[lane];
            int w = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(kFull, w, o);
                if (lane >= o) w += y;
            }
            wpre[lane] = w - v;
            if (lane == 31) total = w;
        }
        __syncthreads();
        int64_t j = base + wpre[warp] + (inc - mine);
#pragma unroll
        for (int c = 0; c < kPerThread; c++) {
            if (ev[c] != ex) continue;
            const int64_t i = i0 + c;
            if (j < cap) {
                const int64_t slot = (int64_t)ex * cap + j;
                ids[slot] = (int32_t)(i / n_used);
                gscores[slot] = sv[c];
                if (slot_of) slot_of[i] = (int32_t)slot;
            } else {
                flag_error(err, kErrBadId);
                if (slot_of) slot_of[i] = -1;
            }
            j++;
        }
        base += total;
        __syncthreads();  // wpre / total are rewritten by the next pass
    }
    // Clamped to the list capacity: a consumer looping j < counts[ex] stays
    // inside this expert's list (an overflow is already flagged above).
    if (tid == 0) counts[ex] = (int32_t)(base < cap ? base : cap);
}

// Sorted rows without list capacities: entries (token * n_used + slot) in
// expert order, each expert's in ascending order, and the experts' bounds.
// One CTA per expert, no CTA waits for another: offsets[ex] is the number of
// entries of smaller experts, which each CTA counts itself. The entries are
// read once, coalesced (4 per thread and load, all loads independent), and
// leave one bit each in shared memory (is it this expert's); a thread then owns
// 32 consecutive bits, one CTA-wide scan of the bit counts places its hits, and
// it writes them out in order. 4096 entries, 128 experts: 2.2 us.
constexpr int kRowsAlone = 28 * 1024;  // more entries: moe_expert_rows_cluster_k

__global__ void __launch_bounds__(kRouteThreads) moe_expert_rows_k(const int32_t *idx, int32_t *offsets, int32_t *entries,
                                                                   int32_t *row_of, int n_entries, int n_expert, int vec,
                                                                   unsigned *err)
{
    constexpr int kPass = 4 * kRouteThreads;
    static_assert(kRowsAlone % kPass == 0 && kRowsAlone <= 32 * kRouteThreads, "a word per thread");
    __shared__ uint32_t bits[kRowsAlone / 32];
    __shared__ int32_t wpre[kRouteWarps], wless[kRouteWarps];
    pdl_wait();
    pdl_trigger();
    const int ex = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int less = 0;
#pragma unroll 4
    for (int j = 0; j < n_entries; j += kPass) {
        const int i = j + 4 * tid;
        int e[4] = {-1, -1, -1, -1};
        if (vec && i + 4 <= n_entries) {
            const int4 v = *reinterpret_cast<const int4 *>(idx + i);
            e[0] = v.x, e[1] = v.y, e[2] = v.z, e[3] = v.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i + k < n_entries) e[k] = idx[i + k];
        }
        uint32_t hit = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            hit |= (uint32_t)(e[k] == ex) << k;
            less += (uint32_t)e[k] < (uint32_t)ex;
            if (ex == 0 && i + k < n_entries && (uint32_t)e[k] >= (uint32_t)n_expert) {
                flag_error(err, kErrBadId);
                if (row_of) row_of[i + k] = -1;
            }
        }
        hit <<= 4 * (lane & 7);  // eight lanes make a word
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) hit |= __shfl_xor_sync(kFull, hit, o);
        if ((lane & 7) == 0) bits[i >> 5] = hit;
    }
    __syncthreads();
    const int words = (n_entries + kPass - 1) / kPass * (kPass / 32);  // written above
    uint32_t mine = tid < words ? bits[tid] : 0;
    const int count = __popc(mine);
    int inc = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(kFull, inc, o);
        if (lane >= o) inc += y;
    }
    const int warp_less = __reduce_add_sync(kFull, less);
    if (lane == 31) wpre[warp] = inc;
    if (lane == 0) wless[warp] = warp_less;
    __syncthreads();
    const int in_warp = wpre[lane];
    const int first = __reduce_add_sync(kFull, wless[lane]);                 // entries of smaller experts
    const int before = __reduce_add_sync(kFull, lane < warp ? in_warp : 0);  // this expert's, in earlier warps
    int row = first + before + inc - count;
    while (mine) {
        const int i = 32 * tid + __ffs((int)mine) - 1;
        mine &= mine - 1;
        entries[row] = i;
        if (row_of) row_of[i] = row;
        row++;
    }
    if (tid == kRouteThreads - 1) {
        offsets[ex] = first;
        if (ex == n_expert - 1) offsets[n_expert] = row;
    }
}

// Self-test of the bounded mbarrier wait: the barrier expects one arrival
// that never comes; the wait must give up after `polls` polls and record the
// timeout in the error word.
__global__ void bounded_wait_selftest_k(uint32_t polls, unsigned *err)
{
    __shared__ __align__(8) uint64_t bar;
    if (threadIdx.x == 0) {
        mbar_init(&bar, 1);
        mbar_init_fence();
    }
    __syncwarp();
    if (!mbar_wait(&bar, 0, polls) && threadIdx.x == 0) flag_error(err, kErrWaitTimeout);
}

// The same for more entries: a cluster of 8 CTAs serves 8 experts and reads the
// entries once between them, 1/8 of each chunk per CTA. A thread holds its 4
// entries' hits as 8 nibbles, one per expert; 8 neighbouring lanes transpose
// them with three exchanges, so that lane j has expert j's word of 32 entries
// and stores it into CTA j's bits (distributed shared memory). The counts of
// smaller experts' entries travel the same way. The barriers and the full chunk
// cost 5.3 us for any size; a CTA per expert alone reads all entries from L2
// (262 KB each at 65,528). Alone / clusters, us, 128 experts, top-8: 2048
// tokens 3.6 / 5.7, 4096: 6.1 / 5.8, 8191: 10.2 / 6.3 (256 experts 13.7 / 6.0),
// 65,536: 85 / 56.
constexpr int kRowsChunk = 64 * kRouteThreads;  // entries per pass
constexpr int kRowsCN = 8;

__global__ void __cluster_dims__(kRowsCN, 1, 1) __launch_bounds__(kRouteThreads)
    moe_expert_rows_cluster_k(const int32_t *idx, int32_t *offsets, int32_t *entries, int32_t *row_of, int n_entries,
                              int n_expert, int vec, unsigned *err)
{
    __shared__ uint32_t bits[kRowsChunk / 32];
    __shared__ int32_t wpre[kRouteWarps], wless[kRouteWarps], whits[kRouteWarps][kRowsCN];
    __shared__ int32_t smaller[kRowsCN];  // entries of smaller experts, of each CTA's share
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = (int)cluster_rank(), ex0 = (int)blockIdx.x - rank, ex = (int)blockIdx.x;
    constexpr int kShare = kRowsChunk / kRowsCN;  // entries of a chunk per CTA
    constexpr int kPass = 4 * kRouteThreads;
    cluster_arrive_relaxed();
    pdl_wait();
    pdl_trigger();
    cluster_wait_acquire();  // every CTA of the cluster runs: its shared memory may be written
    uint32_t far_bits;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(far_bits) : "r"(smem_addr(bits)), "r"(lane & 7));

    int less = 0, hits = 0;  // ids below ex0; of expert ex0 + lane % 8
    // Word of entries i .. i + 31 (i the group's first) for expert ex0 + lane % 8;
    // this thread reads entries i + 4 (lane % 8) .. + 3. All lanes take part.
    auto word = [&](int i, bool count) {
        int e[4] = {-1, -1, -1, -1};
        if (vec && i + 4 <= n_entries) {
            const int4 v = *reinterpret_cast<const int4 *>(idx + i);
            e[0] = v.x, e[1] = v.y, e[2] = v.z, e[3] = v.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i + k < n_entries) e[k] = idx[i + k];
        }
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t d = (uint32_t)e[k] - (uint32_t)ex0;
            if (d < kRowsCN) m |= 1u << (4 * d + k);
            if (count) less += (uint32_t)e[k] < (uint32_t)ex0;
            if (ex0 == 0 && i + k < n_entries && (uint32_t)e[k] >= (uint32_t)n_expert) {
                flag_error(err, kErrBadId);
                if (row_of) row_of[i + k] = -1;
            }
        }
        auto swap = [&](int s, uint32_t low, int shift) {
            const uint32_t o = __shfl_xor_sync(kFull, m, s);
            m = lane & s ? (m & ~low) | ((o & ~low) >> shift) : (m & low) | ((o & low) << shift);
        };
        swap(4, 0x0000ffffu, 16);
        swap(2, 0x00ff00ffu, 8);
        swap(1, 0x0f0f0f0fu, 4);
        if (count) hits += __popc(m);
        return m;
    };
    // Entries behind the first chunk count before anything can be placed.
    for (int j = kRowsChunk + rank * kPass; j < n_entries; j += kRowsCN * kPass) word(j + 4 * tid, true);
    int base = 0, first = 0;  // this expert's entries in earlier chunks; entries of smaller experts
    for (int c0 = 0; c0 < n_entries; c0 += kRowsChunk) {
        uint32_t w[kShare / kPass];
#pragma unroll
        for (int j = 0; j < kShare / kPass; j++) w[j] = word(c0 + rank * kShare + j * kPass + 4 * tid, c0 == 0);
#pragma unroll
        for (int j = 0; j < kShare / kPass; j++)
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(
                             far_bits + 4u * (uint32_t)((rank * kShare + j * kPass + 4 * tid) >> 5)),
                         "r"(w[j]) : "memory");
        if (c0 == 0) {
            hits += __shfl_xor_sync(kFull, hits, 8);
            hits += __shfl_xor_sync(kFull, hits, 16);
            const int warp_less = __reduce_add_sync(kFull, less);
            if (lane < kRowsCN) whits[warp][lane] = hits;
            if (lane == 0) wless[warp] = warp_less;
            __syncthreads();
            if (warp == 0) {
                // Lane j: entries of this share below expert ex0 + j, for CTA j.
                int below = __reduce_add_sync(kFull, wless[lane]), mine = 0;
#pragma unroll
                for (int j = 0; j < kRowsCN; j++) {
                    if (lane == j) mine = below;
                    below += __reduce_add_sync(kFull, whits[lane][j]);
                }
                if (lane < kRowsCN) {
                    uint32_t far;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(far) : "r"(smem_addr(&smaller[rank])), "r"(lane));
                    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(far), "r"(mine) : "memory");
                }
            }
        }
        cluster_arrive_release();
        cluster_wait_acquire();
        if (c0 == 0)
            first = __reduce_add_sync(kFull, lane < kRowsCN ? smaller[lane] : 0);
        uint64_t mine = bits[2 * tid] | (uint64_t)bits[2 * tid + 1] << 32;
        const int count = __popcll(mine);
        int inc = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(kFull, inc, o);
            if (lane >= o) inc += y;
        }
        if (lane == 31) wpre[warp] = inc;
        __syncthreads();
        const int in_warp = wpre[lane];
        const int before = __reduce_add_sync(kFull, lane < warp ? in_warp : 0);  // this expert's, in earlier warps
        const int all = __reduce_add_sync(kFull, in_warp);
        int row = first + base + before + inc - count;
        while (ex < n_expert && mine) {
            const int i = c0 + 64 * tid + __ffsll((long long)mine) - 1;
            mine &= mine - 1;
            entries[row] = i;
            if (row_of) row_of[i] = row;
            row++;
        }
        base += all;
        // Bits and partial sums are rewritten by the next chunk, by every CTA.
        if (c0 + kRowsChunk < n_entries) {
            cluster_arrive_release();
            cluster_wait_acquire();
        }
    }
    if (tid == 0 && ex < n_expert) {
        offsets[ex] = first;
        if (ex == n_expert - 1) offsets[n_expert] = first + base;
    }
}

}  // namespace

int kernel_binary_version()
{
    cudaFuncAttributes a;
    if (cudaFuncGetAttributes(&a, bounded_wait_selftest_k) != cudaSuccess) {
        cudaGetLastError();
        return -1;
    }
    return a.binaryVersion;
}

cudaError_t launch_bounded_wait_selftest(const LaunchCtx &c, uint32_t polls)
{
    bounded_wait_selftest_k<<<1, 32, 0, c.stream>>>(polls, c.err);
    return cudaGetLastError();
}

cudaError_t launch_moe_expert_lists(const LaunchCtx &c, const int32_t *idx, const float *scores, int32_t *counts,
                                    int32_t *ids, float *gscores, int32_t *slot_of, int64_t n_tokens, int n_used,
                                    int n_expert, int64_t cap)
{
    if (n_expert <= 0 || n_expert > 65535) return cudaErrorInvalidValue;
    launch_k(c, moe_expert_lists_k, dim3((unsigned)n_expert), dim3(kRouteThreads), idx, scores, counts, ids, gscores, slot_of,
             n_tokens * n_used, n_used, n_expert, cap, c.err);
    return cudaGetLastError();
}

cudaError_t launch_moe_expert_rows(const LaunchCtx &c, const int32_t *idx, int32_t *offsets, int32_t *entries,
                                   int32_t *row_of, int64_t n_entries, int n_expert)
{
    if (n_expert <= 0 || n_expert > 65535 || n_entries > (1 << 30)) return cudaErrorInvalidValue;
    const int vec = (reinterpret_cast<uintptr_t>(idx) & 15u) == 0;
    if (n_entries > kRowsAlone) {
        const unsigned grid = (unsigned)((n_expert + kRowsCN - 1) / kRowsCN * kRowsCN);
        launch_k(c, moe_expert_rows_cluster_k, dim3(grid), dim3(kRouteThreads), idx, offsets, entries, row_of,
                 (int)n_entries, n_expert, vec, c.err);
        return cudaGetLastError();
    }
    launch_k(c, moe_expert_rows_k, dim3((unsigned)n_expert), dim3(kRouteThreads), idx, offsets, entries, row_of,
             (int)n_entries, n_expert, vec, c.err);
    return cudaGetLastError();
}

}  // namespace ds3
