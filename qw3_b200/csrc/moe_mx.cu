// Matrix products grouped by expert over microscaled (MX) rows, on the
// tensor cores (sm_100a): the experts' gate / up products fused with SwiGLU
// and the 8-bit quantisation of its result, and the plain product (the
// experts' down projection).
//
// The engine runs them per expert (forward_chunk_post_gathered,
// src/ds3_engine.c:973-1011: gather the expert's token rows, gate and up
// products, silu_mul, down product); here one launch covers all experts.
//
// Mathematics. Rows are sorted by expert; group e is rows
// offsets[e] .. offsets[e+1]-1. For row r of group e, with x = MXFP8 and W_e =
// MXFP8 or MXFP4 (value = element * 2^(scale-127), one scale per 32 elements):
//   y[r][m] = sum_k x[r][k] * W_e[m][k]
// and for SwiGLU, with G = gate and U = up products:
//   h[r][f] = silu(G[r][f]) * U[r][f] * row_weight,   act = MXFP8(h)
//
// Tiling. The weight rows take the 128-row side of the tensor-core tile (A)
// and the tokens the free side (B, N <= NT columns), so a group of any size
// wastes at most 15 columns: the instruction's N is set per tile to the
// group's remaining rows rounded up to 16. A persistent CTA walks tiles
// (expert, token block, weight block); the weight block is the fastest index,
// so the CTAs working at the same time share token rows and, with several
// token blocks, weights through L2. The tile list is derived on the device
// from `offsets`; the host never reads it.
//   - Slices of 128 K elements: A 16 KB, B NT x 128 B, both in the 128-byte
//     swizzle, one 32-bit word of four scales per row.
//   - tcgen05.mma kind::mxf8f6f4 with block scales, K = 32 per instruction,
//     accumulators fp32 in tensor memory, double buffered so the epilogue of
//     one tile runs under the products of the next. Element products and
//     scaling are exact; the only roundings are the fp32 accumulation's.
//   - MXFP4 weights are expanded to one byte per element by the copy engine
//     (packed in HBM, 16 elements per 16 bytes in shared memory).
//   - SwiGLU's A tile is 64 gate rows over the same 64 up rows. Two sides of four
//     epilogue warps (one per 32 tensor-memory lanes) take alternate chunks of 16
//     columns; a side's warps pair up, gate and up meet through a shared-memory
//     exchange, and eight lanes with four elements each finish one MX block.
//
// Warps: 0 copies (weights, and token rows that are used in place, as tiled
// boxes), 1 issues the tensor-core work, 2 / 3 stage the scales of A / B in the
// order the tensor core wants them (row r of 128 -> lane r%32, word r/32), 4-11
// are the epilogue, and 12-15 gather token rows that come through x_rows.
//
// What bounds it (B200, 6.5 TB/s measured copy rate). Up to about 128 rows per
// expert the weights' HBM bytes: 512 tokens x top-8 of 128 experts, 2048 -> 2 x
// 768: MXFP8 5.6 TB/s. MXFP4 halves the bytes, and then the issuing warp's and
// the copy engine's work per stage bounds it (4.3 TB/s). Long batches: the
// operands' way from L2 to the SMs (12.7 TB/s there) and power: 4096 tokens in
// place 148 us after a pause (1.39 PFLOP/s), 178 us in calls back to back; the
// row sort before it is 19 us more. The epilogue counts too (20 of 150 us).
//
// Every wait is bounded; on a timeout the CTA records it, lets its copies and
// products land (bounded), frees its tensor memory and returns.
#include "common.cuh"
#include "launch.h"
#include "mx.cuh"

#include <cuda.h>
#include <cuda_fp16.h>

namespace ds3 {
namespace {

constexpr int kTileM = 128;     // weight rows per tile
constexpr int kSliceK = 128;    // K elements per slice of a stage
constexpr int kEpilogueThreads = 256, kGatherThreads = 128;
constexpr int moe_threads(bool gather) { return 128 + kEpilogueThreads + (gather ? kGatherThreads : 0); }
constexpr int kMaxGroups = 256;

// Stages for NT token columns, as many as fit beside the exchange buffers. A
// stage is kSub slices of 128 K elements: two where the slices are small, so
// that the fixed work per stage (wait, fence, commit) of the issuing warp,
// which bounds these sizes, is paid half as often.
template <int NT>
struct MoeLayout {
    static constexpr int kSub = NT <= 128 ? 2 : 1;
    static constexpr int kStages = NT == 64 ? 4 : NT == 128 ? 3 : 4;
    static constexpr int kASlice = kTileM * kSliceK, kBSlice = NT * kSliceK;
    static constexpr int kABytes = kSub * kASlice, kBBytes = kSub * kBSlice;
    static constexpr int kBWords = (NT + 127) / 128 * 4;  // tensor-memory columns of B's scales per slice
    static constexpr int kSfA = kSub * 512, kSfB = kSub * kBWords * 128;
    static constexpr int kXch = 8 * 2 * 8 * 32 * 4;       // epilogue exchange: [pair of warps][buffer][gate, up][8][32] floats
    static constexpr int kOffA = 0;
    static constexpr int kOffB = kOffA + kStages * kABytes;
    static constexpr int kOffSfA = kOffB + kStages * kBBytes;
    static constexpr int kOffSfB = kOffSfA + kStages * kSfA;
    static constexpr int kOffXch = kOffSfB + kStages * kSfB;
    static constexpr int kOffTab = kOffXch + kXch;        // first row, rows, first tile and block size of each group
    static constexpr int kOffIds = kOffTab + 4 * kMaxGroups * 4;  // gathered row ids, per gathering warp
    static constexpr int kOffCol = kOffIds + NT * 4;              // epilogue columns, two tiles (16-byte reads)
    static_assert(kOffCol % 16 == 0 && NT % 16 == 0, "layout");
    static constexpr int kUsed = kOffCol + 2 * NT * 8;
    static constexpr size_t kSmem = kUsed + 1024;         // the base is aligned up to 1024
    static constexpr int kSfCols = kSub * (4 + kBWords);
    static constexpr int kColsUsed = 2 * NT + kStages * kSfCols;
    static constexpr int kTmemCols = kColsUsed <= 256 ? 256 : 512;
    static_assert(kColsUsed <= 512 && kSmem <= 232448 - 512, "layout");
};

struct MoeMaps {
    CUtensorMap w0, w1, x;
};

struct MoeArgs {
    const uint8_t *x;          // [n_x][K]
    const uint8_t *x_s;        // [n_x][K/32]
    const uint8_t *w0_s, *w1_s;  // [E][n_w][K/32]
    const int32_t *offsets;    // [E+1]
    const int32_t *x_rows;     // sorted row -> x_div * (x row) + slot, or nullptr
    const float *row_w;        // SwiGLU weight by x_rows' value (or row), or nullptr
    const int32_t *out_rows;   // sorted row -> output row, or nullptr
    void *out;                 // fp32 / fp16 [n_out_rows][n_w], or e4m3 [n_rows][n_w]
    uint8_t *out_s;            // SwiGLU: [n_rows][n_w/32]
    int n_x, n_rows, n_out_rows, n_group, x_div, K, n_w;
    int x_mode, w_mode;        // how scale rows are loaded (stage_scales)
    unsigned n_mt, n_mt_inv;   // weight blocks per group, 2^32 / n_mt rounded up
    int half, fp4, units;      // out is fp16; the weights are MXFP4; out rows are whole aligned 16-byte units
};

// ------------------------------------------------------------ PTX wrappers
// The single-thread instructions below are executed by whole warps and
// predicated on `lead` (one lane's flag): control flow stays uniform, so their
// operands are computed once in uniform registers. Branching into one lane
// instead cost about twice the issue time per stage.
__device__ __forceinline__ void tma_load_3d(uint32_t lead, uint32_t dst, const CUtensorMap *m, int x, int y, int z,
                                            uint32_t bar)
{
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "@q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n\t}" ::
            "r"(dst), "l"(m), "r"(x), "r"(y), "r"(z), "r"(bar), "r"(lead) : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t lead, uint32_t dst, const CUtensorMap *m, int x, int y, uint32_t bar)
{
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}" ::
            "r"(dst), "l"(m), "r"(x), "r"(y), "r"(bar), "r"(lead) : "memory");
}
// The same box into L2 only, a hint.
__device__ __forceinline__ void tma_prefetch_3d(uint32_t lead, const CUtensorMap *m, int x, int y, int z)
{
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %4, 0;\n\t"
        "@q cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];\n\t}" ::
            "l"(m), "r"(x), "r"(y), "r"(z), "r"(lead) : "memory");
}
__device__ __forceinline__ void expect_bytes(uint32_t lead, uint32_t bar, uint32_t bytes)
{
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
        "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes), "r"(lead) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// Arrive on `bar` once this thread's earlier cp.async copies have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t *bar)
{
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// Whether the phase is complete now (no waiting).
__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity)
{
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(smem_addr(bar)), "r"(parity) : "memory");
    return done != 0;
}
// A warp's place in the ring of stages. `ready` is a test of the next stage's
// barrier made ahead of time: its latency (about 170 cycles with the vote)
// passes under the work on the stage before.
template <int ST>
struct Ring {
    int s = 0;
    uint32_t ph;
    bool ready = false;
    __device__ __forceinline__ explicit Ring(uint32_t first) : ph(first) {}
    __device__ __forceinline__ bool wait(uint64_t *bars)
    {
        return __all_sync(kFull, ready) || __all_sync(kFull, mbar_wait(&bars[s], ph, kWaitLimit));
    }
    // Test the stage after this one.
    __device__ __forceinline__ void peek(uint64_t *bars)
    {
        ready = s + 1 == ST ? mbar_test(&bars[0], ph ^ 1u) : mbar_test(&bars[s + 1], ph);
    }
    __device__ __forceinline__ void next()
    {
        if (++s == ST) {
            s = 0;
            ph ^= 1u;
        }
    }
};
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Arrive on `bar` once all tensor-core work the lead lane issued has finished.
__device__ __forceinline__ void tc_commit(uint32_t lead, uint32_t bar)
{
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(lead)
        : "memory");
}
// 32 rows of 16 bytes, shared -> tensor memory, into all four lane quarters.
__device__ __forceinline__ void tc_copy_scales(uint32_t lead, uint32_t tmem, uint64_t desc)
{
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
        "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(tmem), "l"(desc), "r"(lead) : "memory");
}
__device__ __forceinline__ void tc_mma_mx(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                          uint32_t sfb, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %7, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::
            "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(lead) : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t (&v)[16], uint32_t tmem)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(tmem)
        : "memory");
}
// Between shared-memory writes by threads (scales, gathered rows), seen through
// a barrier, and the tensor core's reads of them: in the issuing warp. In the
// scale warps it would also wait for their loads ahead (a DRAM latency per tile).
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Whether `ok` holds in all `threads` threads that meet at barrier `id`.
__device__ __forceinline__ bool named_all(int id, int threads, bool ok)
{
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.and.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r) : "r"((uint32_t)ok), "r"(id), "r"(threads) : "memory");
    return r != 0;
}
__device__ __forceinline__ void named_sync(int id, int threads)
{
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Shared-memory matrix descriptor: start and stride-byte-offset in 16-byte
// units, descriptor version 1, swizzle code `sw` (2 = 128 bytes, 0 = none).
// K-major 128-byte-swizzled operand: 8-row groups 1024 bytes apart. Scales:
// 8-row groups of 16-byte rows, 128 bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t stride_bytes, uint64_t sw)
{
    return (uint64_t)((addr & 0x3ffffu) >> 4) | (1ull << 16) | ((uint64_t)(stride_bytes >> 4) << 32) | (1ull << 46) |
           (sw << 61);
}

// The row of x that an x_rows value names; one outside x reads row 0 (the
// epilogue writes zeros for it).
__device__ __forceinline__ int x_row(int v, const MoeArgs &a)
{
    const int x = v < 0 ? -1 : v / a.x_div;
    return x < 0 || x >= a.n_x ? 0 : x;
}

// 16 bytes of the output row that k names, from column m of `size`-byte values:
// nothing for a row that goes nowhere, zeros where its token row is none of x.
__device__ __forceinline__ void store16(const MoeArgs &a, int2 k, int m, uint4 y, uint32_t size)
{
    if (!k.y) y = make_uint4(0, 0, 0, 0);
    if (k.x >= 0 && m < a.n_w)
        *reinterpret_cast<uint4 *>(reinterpret_cast<uint8_t *>(a.out) +
                                   ((size_t)(uint32_t)k.x * (uint32_t)a.n_w + m) * size) = y;
}

struct Tile {
    int e, mt, n0, rows, r0;  // group, weight block, first row in the group, rows here, first sorted row
};

// The tile of index t < total, found by the whole warp: two ballots over the
// tile prefix (256 entries, `total` past the last group) instead of a chain of
// eight dependent reads.
template <int NT>
__device__ __forceinline__ Tile find_tile(const int *tab, const MoeArgs &a, int t, int lane)
{
    const int *off = tab, *num = tab + kMaxGroups, *pre = tab + 2 * kMaxGroups, *size = tab + 3 * kMaxGroups;
    const int g = __popc(__ballot_sync(kFull, pre[8 * lane] <= t)) - 1;
    const int e = 8 * g + __popc(__ballot_sync(kFull, lane < 8 && pre[8 * g + (lane & 7)] <= t)) - 1;
    const unsigned local = t - pre[e];
    // local / n_mt by the rounded-up reciprocal, at most one too large
    unsigned nt = a.n_mt == 1 ? local : __umulhi(local, a.n_mt_inv);
    if (nt * a.n_mt > local) nt--;
    Tile q;
    q.e = e;
    q.mt = local - nt * a.n_mt;
    q.n0 = nt * size[e];
    q.rows = min(num[e] - q.n0, size[e]);
    q.r0 = off[e] + q.n0;
    return q;
}

// One warp stages the scales of J x 32 operand rows for every stage of every
// tile of this CTA. Lane l owns rows l, l + 32, ...; the four scales of a row
// and slice are one word, and the words of the lane's rows lie side by side,
// which is the tensor core's order. A stage's words are loaded one stage ahead.
// MODE 2, all words of a row and stage at once (K a whole
// number of stages); 1, word by word (K % 128 == 0); 0, words put together from
// bytes (other K, an odd base).
// The loop is kept rolled: the roles' code competes for the instruction caches,
// and an unrolled loop with buffers for 3 / 7 stages ahead took 164 / 170 us
// against 152 (4096 tokens, 2048 -> 2 x 768) and 31 / 38 against 29 (16 tokens,
// MXFP4). Copying each word asynchronously to its place cost 52 cycles of issue
// per copy.
__device__ __forceinline__ void ld_word(uint32_t &v, const uint8_t *p)
{
    asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p));
}
__device__ __forceinline__ void ld_word2(uint32_t &v, uint32_t &w, const uint8_t *p)
{
    asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(v), "=r"(w) : "l"(p));
}

template <int J, int BYTES, int SUB, int ST, int MODE, typename Rows>
__device__ __forceinline__ bool stage_scales(Rows &rows_of, uint8_t *dst, uint64_t *full, uint64_t *empty, int total,
                                             int n_kb, int nk32, int lane)
{
    const uint8_t *row[J];
    uint32_t cur[J][SUB], nxt[J][SUB];
    auto load = [&](uint32_t (&v)[J][SUB], int kb) {
        const int k = 4 * SUB * kb;  // first scale of the stage
#pragma unroll
        for (int j = 0; j < J; j++) {
            if (MODE == 2 && SUB == 2) {
                ld_word2(v[j][0], v[j][SUB - 1], row[j] + k);
            } else if (MODE) {
#pragma unroll
                for (int i = 0; i < SUB; i++)
                    if (k + 4 * i < nk32) ld_word(v[j][i], row[j] + k + 4 * i);
            } else {
#pragma unroll
                for (int i = 0; i < SUB; i++) {
                    v[j][i] = 0;
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        if (k + 4 * i + c < nk32) v[j][i] |= (uint32_t)row[j][k + 4 * i + c] << (8 * c);
                }
            }
        }
    };
    Ring<ST> ring(1u);
    if ((int)blockIdx.x < total) {
        rows_of(row, blockIdx.x);
        load(cur, 0);
    }
    for (int t = blockIdx.x; t < total; t += gridDim.x) {
#pragma unroll 1
        for (int kb = 0; kb < n_kb; kb++) {
            if (kb + 1 < n_kb) {
                load(nxt, kb + 1);
            } else if (t + (int)gridDim.x < total) {
                rows_of(row, t + gridDim.x);
                load(nxt, 0);
            }
            if (!ring.wait(empty)) return false;
            ring.peek(empty);
#pragma unroll
            for (int i = 0; i < SUB; i++)
#pragma unroll
                for (int j = 0; j < J; j += 4) {
                    auto w = [&](int n) { return j + n < J ? cur[j + n < J ? j + n : 0][i] : 0u; };
                    *reinterpret_cast<uint4 *>(dst + ring.s * BYTES + i * (BYTES / SUB) + j * 128 + lane * 16) =
                        make_uint4(w(0), w(1), w(2), w(3));
                }
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[ring.s]);
            ring.next();
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int i = 0; i < SUB; i++) cur[j][i] = nxt[j][i];
        }
    }
    return true;
}

// SWIGLU: w0 / w1 are the gate / up weights and out is MXFP8. Otherwise w0
// alone, and out is fp32 or fp16. GATHER: the kernel fetches token rows through
// x_rows; otherwise sorted row r is row r of x.
template <int NT, bool SWIGLU, bool GATHER>
__global__ void __launch_bounds__(moe_threads(GATHER), 1) moe_mx_k(const __grid_constant__ MoeMaps maps, const MoeArgs a,
                                                           unsigned *err)
{
    using L = MoeLayout<NT>;
    constexpr int ST = L::kStages;
    constexpr int kRowsPerTile = SWIGLU ? kTileM / 2 : kTileM;  // output columns per tile
    extern __shared__ uint8_t smem_raw[];
    uint8_t *sm = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    __shared__ __align__(8) uint64_t full[ST], empty[ST], acc_full[2], acc_empty[2], drain;
    __shared__ uint32_t tmem_base;
    __shared__ int n_tiles;
    __shared__ int wsum[32];
    __shared__ int tile_rows[8];  // rows of the CTA's tiles, from the warp that stages A's scales
    int *tab = reinterpret_cast<int *>(sm + L::kOffTab);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < ST; s++) {
            // the copy thread, the two scale warps and each gathering lane
            mbar_init(&full[s], 3 + (GATHER ? kGatherThreads : 0));
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], kEpilogueThreads / 32);
        }
        mbar_init(&drain, 1);
        mbar_init_fence();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_base)),
                     "r"(L::kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();
    pdl_trigger();

    // Group bounds, clamped to [0, n_rows], and the tile prefix. A table that
    // decreases anywhere means nothing: no group has rows then (groups would
    // overlap, and their tiles outnumber any bound). Either is reported.
    {
        int lo = 0, hi = 0, l0 = 0, h0 = 0;
        if (tid < a.n_group) {
            l0 = a.offsets[tid];
            h0 = a.offsets[tid + 1];
            lo = min(max(l0, 0), a.n_rows);
            hi = min(max(h0, 0), a.n_rows);
        }
        const bool decreases = __syncthreads_or(h0 < l0);
        if ((lo != l0 || hi != h0 || decreases) && blockIdx.x == 0) flag_error(err, kErrBadId);
        if (decreases) hi = lo;
        // A group's token blocks are of one size, a multiple of 16 (at most NT,
        // so that the last one is never empty).
        const int blocks = (hi - lo + NT - 1) / NT;
        const int v = blocks * (int)a.n_mt;
        int inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(kFull, inc, o);
            if (lane >= o) inc += y;
        }
        if (lane == 31) wsum[warp] = inc;
        __syncthreads();
        const int base = __reduce_add_sync(kFull, lane < warp ? wsum[lane] : 0);
        // Past the last group v is 0, so the prefix stays at the total there.
        if (tid < kMaxGroups) {
            tab[tid] = lo;
            tab[kMaxGroups + tid] = hi - lo;
            tab[2 * kMaxGroups + tid] = base + inc - v;
            tab[3 * kMaxGroups + tid] = blocks ? ((hi - lo + blocks - 1) / blocks + 15) & ~15 : NT;
        }
        if (tid == kMaxGroups - 1) n_tiles = base + inc;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const int total = n_tiles;
    const uint32_t tmem = tmem_base;
    const int n_kb = (a.K + kSliceK * L::kSub - 1) / (kSliceK * L::kSub);  // stages per tile
    const int n_slices = (a.K + kSliceK - 1) / kSliceK;
    const int nk32 = a.K / kMxBlock;
    bool ok = true;
    auto give_up = [&] { flag_error(err, kErrWaitTimeout); };

    if (warp == 0) {
        // ------------------------------------------------------------ copies
        const uint32_t lead = elect_one();
        const uint32_t full0 = smem_addr(&full[0]), a0 = smem_addr(sm + L::kOffA), b0 = smem_addr(sm + L::kOffB);
        Ring<ST> ring(1u);
        int issued = 0;
        for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
            const Tile q = find_tile<NT>(tab, a, t, lane);
            const int nbox = GATHER ? 0 : (q.rows + 31) >> 5;
            const uint32_t bytes = (a.fp4 ? L::kASlice / 2 : L::kASlice) + nbox * 4096;  // per slice
            const int row = q.mt * kRowsPerTile;
            for (int kb = 0; kb < n_kb; kb++) {
                ok = ring.wait(empty);
                if (!ok) break;
                ring.peek(empty);
                const int s = ring.s;
                const uint32_t bar = full0 + 8 * s, A = a0 + s * L::kABytes, B = b0 + s * L::kBBytes;
                const int n = min(L::kSub, n_slices - L::kSub * kb);
                expect_bytes(lead, bar, n * bytes);
#pragma unroll
                for (int sub = 0; sub < L::kSub; sub++) {
                    if (sub >= n) break;
                    const int k = (L::kSub * kb + sub) * kSliceK;
                    const uint32_t As = A + sub * L::kASlice, Bs = B + sub * L::kBSlice;
                    tma_load_3d(lead, As, &maps.w0, k, row, q.e, bar);
                    if (SWIGLU) tma_load_3d(lead, As + L::kASlice / 2, &maps.w1, k, row, q.e, bar);
                    if (!GATHER)
                        for (int i = 0; i < nbox; i++) tma_load_2d(lead, Bs + i * 4096, &maps.x, k, q.r0 + 32 * i, bar);
                }
                issued++;
                ring.next();
                // A CTA with a single tile (decode) has nothing behind it to hide
                // latency with: once the ring is full, the rest of the tile's
                // weights are asked into L2 together.
                if (total <= (int)gridDim.x && kb == ST - 1)
                    for (int i = ST * L::kSub; i < n_slices; i++) {
                        tma_prefetch_3d(lead, &maps.w0, i * kSliceK, row, q.e);
                        if (SWIGLU) tma_prefetch_3d(lead, &maps.w1, i * kSliceK, row, q.e);
                    }
            }
        }
        if (!ok) {
            give_up();
            // Let the copies in flight land before shared memory goes away:
            // backwards over the stages issued last. (ring.ph is the parity of
            // `empty`, the opposite of the one `full` completes with.)
            int s = ring.s;
            uint32_t ph = ring.ph ^ 1u;
            for (int i = 0; i < ST && i < issued; i++) {
                if (s == 0) ph ^= 1u;
                s = s == 0 ? ST - 1 : s - 1;
                mbar_wait(&full[s], ph, kWaitLimit);
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------ tensor cores
        const uint32_t lead = elect_one();
        const uint32_t empty0 = smem_addr(&empty[0]);
        Ring<ST> ring(0u);
        int it = 0;
        // A's type (5 = e2m1, 0 = e4m3), power-of-two scales, M.
        const uint32_t idesc0 = ((a.fp4 ? 5u : 0u) << 7) | (1u << 23) | ((kTileM >> 4) << 24);
        constexpr uint32_t kNextScale = (1u << 4) | (1u << 29);  // scale byte i of the word, B and A
        const uint64_t ad0 = smem_desc(smem_addr(sm + L::kOffA), 1024, 2);
        const uint64_t bd0 = smem_desc(smem_addr(sm + L::kOffB), 1024, 2);
        const uint64_t sa0 = smem_desc(smem_addr(sm + L::kOffSfA), 128, 0);
        const uint64_t sb0 = smem_desc(smem_addr(sm + L::kOffSfB), 128, 0);
        bool acc_ready = true;  // a test of acc_empty made ahead of time
        for (int t = blockIdx.x; t < total; t += gridDim.x, it++) {
            const int b = it & 1;
            ok = __all_sync(kFull, acc_ready) ||
                 __all_sync(kFull, mbar_wait(&acc_empty[b], ((it >> 1) & 1u) ^ 1u, kWaitLimit));
            if (!ok) break;
            uint32_t idesc = 0;
            const uint32_t d = tmem + b * NT;
            for (int kb = 0; kb < n_kb; kb++) {
                ok = ring.wait(full);
                if (!ok) break;
                ring.peek(full);
                if (kb == 0) idesc = idesc0 | ((uint32_t)((*(volatile int *)&tile_rows[it & 7] + 15) >> 4) << 18);  // N / 8 at bit 17
                if (kb == n_kb - 1) acc_ready = mbar_test(&acc_empty[b ^ 1], (((it + 1) >> 1) & 1u) ^ 1u);
                const int s = ring.s;
                tc_fence_after();
                fence_async_shared();
                // Scales of the slices side by side: A's 4 columns, then B's.
                const uint32_t sf = tmem + 2 * NT + s * L::kSfCols;
#pragma unroll
                for (int sub = 0; sub < L::kSub; sub++) {
                    tc_copy_scales(lead, sf + sub * (4 + L::kBWords), sa0 + ((s * L::kSfA + sub * 512) >> 4));
#pragma unroll
                    for (int j = 0; j < L::kBWords; j += 4)
                        tc_copy_scales(lead, sf + sub * (4 + L::kBWords) + 4 + j,
                                       sb0 + ((s * L::kSfB + sub * L::kBWords * 128 + j * 128) >> 4));
                }
                const uint64_t ad = ad0 + s * (L::kABytes >> 4), bd = bd0 + s * (L::kBBytes >> 4);
                const int nk = nk32 - 4 * L::kSub * kb;  // 32-element steps left
#pragma unroll
                for (int i = 0; i < 4 * L::kSub; i++) {
                    const int sub = i >> 2;
                    const uint32_t sfa = sf + sub * (4 + L::kBWords);
                    if (i < nk)
                        tc_mma_mx(lead, d, ad + sub * (L::kASlice >> 4) + 2 * (i & 3),
                                  bd + sub * (L::kBSlice >> 4) + 2 * (i & 3), idesc + (i & 3) * kNextScale, sfa, sfa + 4,
                                  (uint32_t)(kb | i));
                }
                tc_commit(lead, empty0 + 8 * s);
                ring.next();
            }
            if (!ok) break;
            tc_commit(lead, smem_addr(&acc_full[b]));
        }
        if (!ok) {
            give_up();
            tc_commit(lead, smem_addr(&drain));  // products in flight finish before tensor memory is freed
            mbar_wait(&drain, 0, kWaitLimit);
        }
    } else if (warp < 4) {
        // ------------------------------------------------------------ scales
        int seq = 0;
        auto rows_of_a = [&](const uint8_t *(&row)[4], int t) {
            const Tile q = find_tile<NT>(tab, a, t, lane);
            // For the issuing warp, which reads it after this tile's first stage.
            // At most ST + 1 tiles ahead of it, so eight entries do.
            static_assert(ST + 1 < 8, "tile_rows");
            if (lane == 0) *(volatile int *)&tile_rows[seq & 7] = q.rows;
            seq++;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int r = min(q.mt * kRowsPerTile + 32 * (SWIGLU ? j & 1 : j) + lane, a.n_w - 1);
                row[j] = (SWIGLU && j >= 2 ? a.w1_s : a.w0_s) + ((size_t)q.e * a.n_w + r) * nk32;
            }
        };
        // B's row ids are read a tile ahead and resolved when the tile comes.
        int raw[NT / 32];
        auto read_ids = [&](int t) {
            if (!GATHER || t >= total) return;
            const Tile q = find_tile<NT>(tab, a, t, lane);
#pragma unroll
            for (int j = 0; j < NT / 32; j++) raw[j] = a.x_rows[q.r0 + min(lane + 32 * j, q.rows - 1)];
        };
        auto rows_of_b = [&](const uint8_t *(&row)[NT / 32], int t) {
            const Tile q = find_tile<NT>(tab, a, t, lane);
#pragma unroll
            for (int j = 0; j < NT / 32; j++) {
                int x = q.r0 + min(lane + 32 * j, q.rows - 1);
                if (GATHER) x = x_row(raw[j], a);
                row[j] = a.x_s + (size_t)x * nk32;
            }
            read_ids(t + gridDim.x);
        };
#define DS3_SCALES(J, BYTES, MODE, rows_of, at) \
    stage_scales<J, BYTES, L::kSub, ST, MODE>(rows_of, sm + at, full, empty, total, n_kb, nk32, lane)
        if (warp == 2) {
            ok = a.w_mode == 2   ? DS3_SCALES(4, L::kSfA, 2, rows_of_a, L::kOffSfA)
                 : a.w_mode == 1 ? DS3_SCALES(4, L::kSfA, 1, rows_of_a, L::kOffSfA)
                                 : DS3_SCALES(4, L::kSfA, 0, rows_of_a, L::kOffSfA);
        } else {
            read_ids(blockIdx.x);
            ok = a.x_mode == 2   ? DS3_SCALES(NT / 32, L::kSfB, 2, rows_of_b, L::kOffSfB)
                 : a.x_mode == 1 ? DS3_SCALES(NT / 32, L::kSfB, 1, rows_of_b, L::kOffSfB)
                                 : DS3_SCALES(NT / 32, L::kSfB, 0, rows_of_b, L::kOffSfB);
        }
#undef DS3_SCALES
        if (!ok) give_up();
    } else if (GATHER && warp >= 12) {
        // ------------------------------------------------------- row gathers
        // Every gathering warp works on every stage, in order: warp g copies the
        // four-row groups g, g + 4, ... (Whole stages dealt out to the warps
        // would let one of them run two uses of a slot ahead of a ring of fewer
        // stages than warps, where a barrier's parity no longer tells the uses
        // apart.) Eight lanes copy a token row's 128 bytes of a slice.
        constexpr int kMine = NT / 4, kIds = (kMine + 31) / 32;
        const int g = warp - 12, piece = lane & 7, r4 = lane >> 3;
        int *id = reinterpret_cast<int *>(sm + L::kOffIds) + g * kMine;
        int nid[kIds];
        auto rows_of = [&](int t) {
            const Tile q = find_tile<NT>(tab, a, t, lane);
#pragma unroll
            for (int j = 0; j < kIds; j++) {
                const int m = lane + 32 * j;  // the warp's m-th row
                const int r = min((m >> 2) * 16 + 4 * g + (m & 3), q.rows - 1);
                nid[j] = a.x_rows[q.r0 + r];
            }
            return q.rows;
        };
        Ring<ST> ring(1u);
        int t = blockIdx.x, rows = 0;
        if (t < total) rows = rows_of(t);
        for (; t < total && ok; t += gridDim.x) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < kIds; j++)
                if (lane + 32 * j < kMine) id[lane + 32 * j] = x_row(nid[j], a);
            __syncwarp();
            const int n = rows;
            if (t + (int)gridDim.x < total) rows = rows_of(t + gridDim.x);
            for (int kb = 0; kb < n_kb; kb++) {
                ok = ring.wait(empty);
                if (!ok) break;
                ring.peek(empty);
                const int s = ring.s;
#pragma unroll
                for (int sub = 0; sub < L::kSub; sub++) {
                    const int k = (L::kSub * kb + sub) * kSliceK + piece * 16;
                    if (k >= a.K) break;
                    const uint32_t dst = smem_addr(sm + L::kOffB + s * L::kBBytes + sub * L::kBSlice);
                    const uint8_t *src = a.x + k;
#pragma unroll 2
                    for (int i = 4 * g, m = r4; i < n; i += 16, m += 4) {
                        const int r = i + r4;  // the 128-byte swizzle: piece ^ (row % 8)
                        cp_async16(dst + r * 128 + ((piece ^ (r & 7)) << 4), src + (size_t)(uint32_t)id[m] * (uint32_t)a.K);
                    }
                }
                cp_async_arrive(&full[s]);
                ring.next();
            }
        }
        if (!ok) give_up();
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        // ---------------------------------------------------------- epilogue
        // Warps 4-7 and 8-11 take alternate 16-column chunks; within a chunk
        // warp w of four reads tensor-memory lanes 32 w .. 32 w + 31.
        const int w = (warp - 4) & 3, side = (warp - 4) >> 2, me = tid - 128;
        static_assert(NT <= kEpilogueThreads, "one column per epilogue thread");
        float *xch = reinterpret_cast<float *>(sm + L::kOffXch);
        int it = 0, parity = 0;
        // Thread c looks up column c, a tile ahead: its row's x_rows and out_rows
        // values when the tile before it begins, its weight when that one's
        // products are done. (Looked up in its own tile, a memory round trip per
        // tile was the longest part of a small tile's epilogue.)
        int next_x = 0, next_o = 0;
        float next_w = 1.0f;
        Tile q, next = {};
        auto look_up = [&](int t) {
            if (t >= total) return;
            next = find_tile<NT>(tab, a, t, lane);
            if (me < next.rows) {
                const int r = next.r0 + me;
                next_x = a.x_rows ? a.x_rows[r] : r;
                next_o = a.out_rows ? a.out_rows[r] : r;
            }
        };
        auto good_x = [&](int x) { return !a.x_rows || (x >= 0 && x / a.x_div < a.n_x); };
        auto look_up_weight = [&] {
            if (SWIGLU && a.row_w && me < next.rows && good_x(next_x)) next_w = a.row_w[next_x];
        };
        look_up(blockIdx.x);
        look_up_weight();
        for (int t = blockIdx.x; t < total; t += gridDim.x, it++) {
            q = next;
            const int b = it & 1;
            // Where column c's row goes (-1: nowhere; SwiGLU: its weight) and
            // whether its token row is one of x. Two buffers: no thread is two
            // tiles ahead of another.
            int2 *col = reinterpret_cast<int2 *>(sm + L::kOffCol) + b * NT;
            if (me < NT) {
                int2 k = make_int2(-1, 0);
                if (me < q.rows) {
                    k.y = good_x(next_x);
                    k.x = SWIGLU ? __float_as_int(next_w) : next_o >= 0 && next_o < a.n_out_rows ? next_o : -1;
                    if (!k.y || (!SWIGLU && k.x < 0)) flag_error(err, kErrBadId);
                }
                col[me] = k;
            }
            look_up(t + gridDim.x);
            // One warp polls (eight would take issue slots from the others'
            // work), and all go on together or not at all.
            ok = named_all(3, kEpilogueThreads, warp != 4 || mbar_wait(&acc_full[b], (it >> 1) & 1u, kWaitLimit));
            if (!ok) {
                give_up();
                break;
            }
            look_up_weight();
            tc_fence_after();
            const uint32_t d = tmem + b * NT + ((uint32_t)(32 * w) << 16);
            // One copy of the chunk's code: with it unrolled over the chunks, the
            // roles' instructions no longer fit the instruction caches together.
#pragma unroll 1
            for (int c0 = 16 * side; c0 < q.rows; c0 += 32) {
                const int nc = min(16, q.rows - c0);
                uint32_t v[16];
                tc_ld16(v, d + c0);
                if (SWIGLU) {
                    // Warps 0 / 1 hold gate lanes, 2 / 3 the same up lanes. A pair
                    // lays 8 columns at a time side by side in shared memory (two
                    // buffers in turn); then the gate warp finishes the first four
                    // and the up warp the others, eight lanes a column with four
                    // elements each, so that a block's maximum is three exchanges
                    // for four columns and a store is four elements. (One lane per
                    // element, columns one by one: 4096 tokens 152 us, so 146.)
                    const int pair = side * 2 + (w & 1), up = w >> 1;
                    const int f0 = q.mt * kRowsPerTile + 32 * (w & 1), f = 4 * (lane & 7);
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        if (8 * half >= nc) break;
                        float *buf = xch + (pair * 2 + parity) * 512;
                        parity ^= 1;
#pragma unroll
                        for (int i = 0; i < 8; i++) buf[up * 256 + i * 32 + lane] = __uint_as_float(v[8 * half + i]);
                        named_sync(4 + pair, 64);
                        const int i = 4 * up + (lane >> 3), c = 8 * half + i;  // the lane's column
                        const float4 g4 = *reinterpret_cast<const float4 *>(buf + i * 32 + f);
                        const float4 u4 = *reinterpret_cast<const float4 *>(buf + 256 + i * 32 + f);
                        const int2 k = col[c0 + c];
                        const float g[4] = {g4.x, g4.y, g4.z, g4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w};
                        const float weight = __int_as_float(k.x);
                        float h[4];
                        uint32_t amax = 0;
#pragma unroll
                        for (int n = 0; n < 4; n++) {
                            // silu(g) u. With e^-|g| the divisor is 1 to 2 for every gate, where
                            // the quotient is good to 2 ulp, far inside the 8-bit rounding. (It is
                            // 0 for divisors past 2^126, that of e^-g below -87.3.)
                            const float t = expf(-fabsf(g[n]));
                            h[n] = __fdividef(g[n] < 0.0f ? g[n] * t : g[n], 1.0f + t) * u[n];
                            if (a.row_w) h[n] *= weight;
                            if (!k.y) h[n] = 0.0f;
                            amax = max(amax, __float_as_uint(h[n]) & 0x7fffffffu);
                        }
#pragma unroll
                        for (int o = 1; o < 8; o <<= 1) amax = max(amax, __shfl_xor_sync(kFull, amax, o));
                        const uint32_t sc = mx_scale<kMxEmaxFp8>(amax);
                        const float inv = mx_inv_scale(sc);
                        const uint32_t e = e4m3x4(mx_scaled(h[0], sc, inv), mx_scaled(h[1], sc, inv),
                                                  mx_scaled(h[2], sc, inv), mx_scaled(h[3], sc, inv));
                        if (c < nc && f0 < a.n_w) {
                            const size_t row = (size_t)(q.r0 + c0 + c);
                            *reinterpret_cast<uint32_t *>(reinterpret_cast<uint8_t *>(a.out) + row * a.n_w + f0 + f) = e;
                            if ((lane & 7) == 0) a.out_s[row * (a.n_w / kMxBlock) + f0 / kMxBlock] = (uint8_t)sc;
                        }
                    }
                } else if (a.units) {
                    // Output rows of whole 16-byte units: the side's four warps lay
                    // rows of 128 values side by side in shared memory, 4 KB at a
                    // time in two buffers in turn (so one barrier each), and store
                    // them whole, 16 bytes a lane. What counts is the number of
                    // accesses: 4096 tokens, 768 -> 2048, fp16, 79 us, against 96 us
                    // with 8 bytes a lane, 119 us with every warp storing its own 32
                    // values of each row, and 68 us without an epilogue.
                    uint8_t *stage = reinterpret_cast<uint8_t *>(xch) + side * 8192;
                    const int m0 = q.mt * kRowsPerTile;
                    if (a.half) {
                        __half *h = reinterpret_cast<__half *>(stage + parity * 4096);
                        parity ^= 1;
#pragma unroll
                        for (int c = 0; c < 16; c++) h[c * 128 + 32 * w + lane] = __float2half_rn(__uint_as_float(v[c]));
                        named_sync(4 + side, 128);
                        const int m = 8 * (lane & 15);
#pragma unroll
                        for (int i = 0; i < 2; i++) {  // two rows per store
                            const int r = 4 * w + 2 * i + (lane >> 4);
                            store16(a, col[c0 + r], m0 + m, *reinterpret_cast<const uint4 *>(h + r * 128 + m), 2);
                        }
                    } else {
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            if (8 * half >= nc) break;
                            float *f = reinterpret_cast<float *>(stage + parity * 4096);
                            parity ^= 1;
#pragma unroll
                            for (int c = 0; c < 8; c++) f[c * 128 + 32 * w + lane] = __uint_as_float(v[8 * half + c]);
                            named_sync(4 + side, 128);
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                const int r = 2 * w + i;
                                store16(a, col[c0 + 8 * half + r], m0 + 4 * lane,
                                        *reinterpret_cast<const uint4 *>(f + r * 128 + 4 * lane), 4);
                            }
                        }
                    }
                } else {  // each lane stores its own value of each row
                    const int m = q.mt * kRowsPerTile + 32 * w + lane;
#pragma unroll
                    for (int c = 0; c < 16; c++) {
                        if (c >= nc) break;
                        const int2 k = col[c0 + c];
                        if (k.x < 0 || m >= a.n_w) continue;
                        const size_t at = (size_t)(uint32_t)k.x * (uint32_t)a.n_w + m;
                        const float y = k.y ? __uint_as_float(v[c]) : 0.0f;
                        if (a.half) reinterpret_cast<__half *>(a.out)[at] = __float2half_rn(y);
                        else reinterpret_cast<float *>(a.out)[at] = y;
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[b]);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kTmemCols) : "memory");
}

// x rows and their scales in sorted order: one warp per row, 16 bytes a lane.
__global__ void __launch_bounds__(256) moe_sort_rows_k(const uint8_t *sorted_x, const uint8_t *sorted_s, const MoeArgs a)
{
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (r >= min(a.offsets[a.n_group], a.n_rows)) return;  // rows behind the last group are not read
    const size_t x = x_row(a.x_rows[r], a);
    const uint4 *src = reinterpret_cast<const uint4 *>(a.x + x * a.K);
    uint4 *dst = reinterpret_cast<uint4 *>(const_cast<uint8_t *>(sorted_x) + (size_t)r * a.K);
#pragma unroll 4
    for (int i = lane; i < a.K / 16; i += 32) dst[i] = src[i];
    const int nk32 = a.K / kMxBlock;
    const uint8_t *s = a.x_s + x * nk32;
    uint8_t *d = const_cast<uint8_t *>(sorted_s) + (size_t)r * nk32;
    if (a.x_mode) {
        for (int i = lane; i < nk32 / 4; i += 32)
            reinterpret_cast<uint32_t *>(d)[i] = reinterpret_cast<const uint32_t *>(s)[i];
    } else {
        for (int i = lane; i < nk32; i += 32) d[i] = s[i];
    }
}

// ---------------------------------------------------------------- host side
typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_fn()
{
    static EncodeTiled fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult st;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12080, cudaEnableDefault, &st) != cudaSuccess ||
            st != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (EncodeTiled)p;
    }();
    return fn;
}

// Rows of `cols` elements, `rows` per matrix, `n` matrices; 128 elements by
// `box_rows` rows per copy, 128-byte swizzle. fp4: packed in memory, one byte
// per element in shared memory.
bool encode(CUtensorMap *m, const void *base, int rank, uint64_t cols, uint64_t rows, uint64_t n, uint32_t box_rows, bool fp4)
{
    const uint64_t row_bytes = fp4 ? cols / 2 : cols;
    const cuuint64_t dim[3] = {cols, rows, n};
    const cuuint64_t stride[2] = {row_bytes, row_bytes * rows};
    const cuuint32_t box[3] = {kSliceK, box_rows, 1};
    const cuuint32_t step[3] = {1, 1, 1};
    EncodeTiled fn = encode_fn();
    return fn && fn(m, fp4 ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B : CU_TENSOR_MAP_DATA_TYPE_UINT8, (cuuint32_t)rank,
                    const_cast<void *>(base), dim, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// stage_scales' MODE for rows of n scales at `base`, `stage` scales per stage.
int scale_mode(const void *base, int n, int stage)
{
    const uintptr_t v = (uintptr_t)base | (uintptr_t)n;
    return v % stage == 0 ? 2 : v % 4 == 0 ? 1 : 0;
}

template <int NT, bool SWIGLU, bool GATHER>
cudaError_t launch_nt(const LaunchCtx &c, const MoeMaps &maps, MoeArgs a)
{
    using L = MoeLayout<NT>;
    const int nk32 = a.K / kMxBlock, stage = 4 * L::kSub;  // scales of a row per stage
    a.x_mode = scale_mode(a.x_s, nk32, stage);
    a.w_mode = scale_mode(a.w0_s, nk32, stage);
    if (SWIGLU) a.w_mode = min(a.w_mode, scale_mode(a.w1_s, nk32, stage));
    auto *k = moe_mx_k<NT, SWIGLU, GATHER>;
    static const cudaError_t set = [&] {
        keep_driver_carveout((const void *)k);
        return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kSmem);
    }();
    if (set != cudaSuccess) return set;
    const int64_t tiles = ((int64_t)a.n_rows / NT + (a.n_rows < a.n_group ? a.n_rows : a.n_group)) * a.n_mt;
    if (tiles > 0x3fffffff) return cudaErrorInvalidValue;
    const unsigned grid = (unsigned)(tiles < c.n_sm ? tiles : c.n_sm);
    launch_ks(c, k, dim3(grid), dim3(moe_threads(GATHER)), L::kSmem, maps, a, c.err);
    return cudaGetLastError();
}

}  // namespace

static int moe_mean_rows(int n_rows, int n_group) { return (n_rows + n_group - 1) / n_group; }

// Gathering inside the product kernel goes through the threads' copy path,
// which cannot feed wide tiles; sorting the rows first costs a pass over them.
// Measured, 128 groups of random sizes, us gathered / sorted first, SwiGLU 2048
// -> 2 x 768 and (fp16) 768 -> 2048:
//   mean rows     32         48         64         80          96          128
//   MXFP8 SwiGLU  73 / 78    77 / 83    83 / 87    92 / 93     100 / 97    131 / 115
//         plain   41 / 43    44 / 45    49 / 47    52 / 51     56 / 54     73 / 63
//   MXFP4 SwiGLU  53 / 56    63 / 63    72 / 71    81 / 77     90 / 83     120 / 103
//         plain   32 / 33    36 / 36    42 / 39    46 / 44     50 / 47     66 / 58
// The limits are SwiGLU's, where token rows are gathered; a plain product over
// x_rows would gain 2 to 4 % from 64 rows of MXFP8 on.
size_t moe_sort_bytes(const MoeMxCall &q)
{
    if (!q.x_rows || moe_mean_rows(q.n_rows, q.n_group) <= (q.w_type == kMxFp4 ? 48 : 96)) return 0;
    return (size_t)q.n_rows * q.K + (size_t)q.n_rows * (q.K / kMxBlock);
}

cudaError_t launch_moe_mx(const LaunchCtx &c, const MoeMxCall &q)
{
    if (q.n_rows <= 0 || q.n_group <= 0) return cudaSuccess;
    if (q.n_group > kMaxGroups) return cudaErrorInvalidValue;
    MoeMaps maps;
    const bool fp4 = q.w_type == kMxFp4, swiglu = q.w1 != nullptr;
    MoeArgs a = {};
    a.x = q.x;
    a.x_s = q.x_s;
    a.half = q.out_f16;
    a.units = (size_t)q.n_w * (q.out_f16 ? 2 : 4) % 16 == 0 && (uintptr_t)q.out % 16 == 0;
    a.fp4 = fp4;
    a.w0_s = q.w0_s;
    a.w1_s = q.w1_s;
    a.offsets = q.offsets;
    a.x_rows = q.x_rows;
    a.row_w = q.row_w;
    a.out_rows = q.out_rows;
    a.out = q.out;
    a.out_s = q.out_s;
    a.n_x = q.n_x;
    a.n_rows = q.n_rows;
    a.n_out_rows = q.n_out_rows;
    a.n_group = q.n_group;
    a.x_div = q.x_div;
    a.K = q.K;
    a.n_w = q.n_w;
    const int rows_per_tile = swiglu ? kTileM / 2 : kTileM;
    a.n_mt = (unsigned)((q.n_w + rows_per_tile - 1) / rows_per_tile);
    a.n_mt_inv = (unsigned)(((1ull << 32) + a.n_mt - 1) / a.n_mt);
    int n_map = q.n_x;
    const bool sorted = q.x_rows && q.sorted;
    if (sorted) {
        uint8_t *sx = q.sorted, *ss = q.sorted + (size_t)q.n_rows * q.K;
        a.x_mode = scale_mode(q.x_s, q.K / kMxBlock, 4);
        launch_k(c, moe_sort_rows_k, dim3((unsigned)((q.n_rows + 7) / 8)), dim3(256), sx, ss, a);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        a.x = sx;
        a.x_s = ss;
        n_map = q.n_rows;
    }
    if (!encode(&maps.w0, q.w0, 3, q.K, q.n_w, q.n_group, swiglu ? kTileM / 2 : kTileM, fp4) ||
        !encode(&maps.w1, swiglu ? q.w1 : q.w0, 3, q.K, q.n_w, q.n_group, kTileM / 2, fp4) ||
        !encode(&maps.x, a.x, 2, q.K, n_map, 1, 32, false))
        return cudaErrorInvalidValue;
    // Token columns per tile by the groups' mean size. Measured over 128 groups of
    // random sizes, rows in place, us at 64 / 128 / 224 columns, SwiGLU 2048 -> 2 x
    // 768 and (fp16) 768 -> 2048:
    //   mean   MXFP8 SwiGLU     MXFP8 plain     MXFP4 SwiGLU     MXFP4 plain
    //   48     74 / 76 / 84     41 / 40 / 44    56 / 59 / 70     32 / 32 / 38
    //   64     87 / 80 / 88     47 / 43 / 47    74 / 65 / 74     40 / 35 / 41
    //   112    117 / 91 / 100   63 / 51 / 54    104 / 80 / 87    56 / 44 / 48
    //   128    134 / 109 / 105  71 / 59 / 57    120 / 98 / 93    64 / 53 / 51
    //   192    181 / 145 / 126  97 / 79 / 69    164 / 131 / 116  88 / 72 / 63
    //   256    232 / 175 / 178  123 / 98 / 98   211 / 163 / 166  114 / 91 / 92
    //   512    419 / 308 / 301  224 / 176 / 164 389 / 292 / 286  210 / 168 / 157
    // (Half of the groups of about 128 rows need a second block of 128; groups of
    // about 256 take two blocks of 224, and two or three of 128.)
    const int avg = moe_mean_rows(q.n_rows, q.n_group);
    const int nt = avg <= 48 ? 64 : avg <= 112 ? 128 : 224;
#define DS3_MOE(NT)                                                                                                  \
    (swiglu ? (q.x_rows && !sorted ? launch_nt<NT, true, true>(c, maps, a) : launch_nt<NT, true, false>(c, maps, a)) \
            : (q.x_rows && !sorted ? launch_nt<NT, false, true>(c, maps, a) : launch_nt<NT, false, false>(c, maps, a)))
    return nt == 64 ? DS3_MOE(64) : nt == 128 ? DS3_MOE(128) : DS3_MOE(224);
#undef DS3_MOE
}

}  // namespace ds3
