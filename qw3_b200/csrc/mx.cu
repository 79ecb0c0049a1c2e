// Rows to and from the microscaled (MX) formats of mx.cuh (sm_100a):
// quantise, dequantise, and residual add + RMSNorm with MXFP8 output.
//
// All three are bound by HBM traffic; every input is read once and every
// output written once.
#include "common.cuh"
#include "launch.h"
#include "mx.cuh"

namespace ds3 {
namespace {

// ----------------------------------------------------------------- quantise
// Rows are dense and a whole number of blocks, so the tensor is a flat list of
// 16-byte input units (4 fp32 or 8 fp16 elements); the 8 or 4 lanes of a block
// share the largest magnitude by shuffles. A thread takes kUnits units 256
// apart, all loads first: every access of a warp is one contiguous run, and
// the reads in flight cover the latency (98304 x 2048 fp16 to MXFP4 and back:
// 291 us with one 8-element unit per thread and split accesses).
constexpr int kUnits = 4;

__device__ __forceinline__ void unpack(float (&v)[4], float4 a) { v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w; }
__device__ __forceinline__ void unpack(float (&v)[8], float4 a)
{
    const __half2 *h = reinterpret_cast<const __half2 *>(&a);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(h[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

template <typename T, bool FP4>
__global__ void __launch_bounds__(256) mx_quantize_k(const T *src, uint8_t *q, uint8_t *scales, int64_t n_units)
{
    constexpr int E = 16 / sizeof(T);       // elements per unit
    constexpr int kLanes = kMxBlock / E;    // lanes per block
    pdl_wait();
    pdl_trigger();
    const int64_t u0 = (int64_t)blockIdx.x * (256 * kUnits) + threadIdx.x;
    float4 in[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        in[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (u0 + 256 * k < n_units) in[k] = ld_stream_inflight(reinterpret_cast<const float4 *>(src) + u0 + 256 * k);
    }
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        float v[E];
        unpack(v, in[k]);
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < E; i++) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) amax = max(amax, __shfl_xor_sync(kFull, amax, o));
        const int64_t u = u0 + 256 * k;
        if (u >= n_units) continue;  // whole blocks: n is a multiple of 32
        const uint32_t sc = mx_scale<FP4 ? kMxEmaxFp4 : kMxEmaxFp8>(amax);
        const float inv = mx_inv_scale(sc);
#pragma unroll
        for (int i = 0; i < E; i++) v[i] = mx_scaled(v[i], sc, inv);
        if constexpr (E == 8) {
            if (FP4) reinterpret_cast<uint32_t *>(q)[u] = e2m1x8(v);
            else reinterpret_cast<uint2 *>(q)[u] = make_uint2(e4m3x4(v[0], v[1], v[2], v[3]), e4m3x4(v[4], v[5], v[6], v[7]));
        } else {
            if (FP4) {
                const float w[8] = {v[0], v[1], v[2], v[3], 0.0f, 0.0f, 0.0f, 0.0f};
                reinterpret_cast<uint16_t *>(q)[u] = (uint16_t)e2m1x8(w);
            } else {
                reinterpret_cast<uint32_t *>(q)[u] = e4m3x4(v[0], v[1], v[2], v[3]);
            }
        }
        if (threadIdx.x % kLanes == 0) scales[u / kLanes] = (uint8_t)sc;
    }
}

// --------------------------------------------------------------- dequantise
// Both element types convert to fp16 exactly, and the product with a power of
// two is exact in fp32 (an element has at most 4 significant bits, so even
// results below the normal range are representable). A unit is 4 elements, one
// 16-byte store; kUnits units per thread as above.
template <bool FP4>
__global__ void __launch_bounds__(256) mx_dequantize_k(const uint8_t *q, const uint8_t *scales, float *dst, int64_t n_units)
{
    pdl_wait();
    pdl_trigger();
    const int64_t u0 = (int64_t)blockIdx.x * (256 * kUnits) + threadIdx.x;
    uint32_t w[kUnits], sc[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        const int64_t u = u0 + 256 * k;
        w[k] = sc[k] = 0;
        if (u < n_units) {
            w[k] = FP4 ? reinterpret_cast<const uint16_t *>(q)[u] : __ldcs(reinterpret_cast<const uint32_t *>(q) + u);
            sc[k] = scales[u >> 3];
        }
    }
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        const int64_t u = u0 + 256 * k;
        if (u >= n_units) break;
        uint32_t h[2];
        if (FP4) {
            asm("{\n\t.reg .b8 b0, b1;\n\t"
                "mov.b16 {b0, b1}, %2;\n\t"
                "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t}"
                : "=&r"(h[0]), "=r"(h[1])
                : "h"((uint16_t)w[k]));
        } else {
            asm("{\n\t.reg .b16 a, b;\n\t"
                "mov.b32 {a, b}, %2;\n\t"
                "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
                : "=r"(h[0]), "=r"(h[1])
                : "r"(w[k]));
        }
        const float s = mx_scale_value(sc[k]);
        const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&h[0]));
        const float2 hi = __half22float2(*reinterpret_cast<const __half2 *>(&h[1]));
        __stcs(reinterpret_cast<float4 *>(dst) + u, make_float4(lo.x * s, lo.y * s, hi.x * s, hi.y * s));
    }
}

// ------------------------------------------------ residual add + norm + MXFP8
// s = x + r (fp32, as add_rms_norm), then n = s * w / sqrt(mean(s^2) + eps).
// The sum of squares and the inverse root are fp64, and the two products are
// carried as a float and its error (fma), so each normed value is the exact
// one rounded once to fp32 (but for a chance of about 2^-22): the 8-bit codes,
// which jump where a value crosses a rounding border, then do not depend on
// the order of the sum.
//
// Up to 4096 elements: four warps per row, the row in registers (VPT float4 of
// x and of r per thread, all loads issued before the first use), so the reads
// and writes of other rows pass under a row's reductions. Thread t works on
// elements 4 t .. 4 t + 3 of every 512: an MX block is 8 neighbouring lanes.
// 16384 x 2048: 93 us, 6.2 TB/s; without the prefetch of the next wave's rows
// 103 us; with one warp per row and the row in shared memory, the first
// version, 149 us (too few reads in flight behind its chains).
// Longer rows: that version, below (2048 x 8192 with residual and every output:
// 274 us, 1.0 TB/s; 4096 x 5120: 206 us, 1.7 TB/s).
constexpr int kNormMxMaxN = 16384;

// 1 / sqrt(m) to full fp64 accuracy: the fp32 estimate and two Newton steps,
// each of which squares its relative error (2^-22 at first).
__device__ __forceinline__ double inv_sqrt64(double m)
{
    if (!(m > 1e-30 && m < 1e30)) return 1.0 / sqrt(m);
    double y = rsqrtf((float)m);
    y = y * fma(-0.5 * m * y, y, 1.5);
    return y * fma(-0.5 * m * y, y, 1.5);
}

// Four normed values s * inv * g, inv = ih + il, each rounded once.
__device__ __forceinline__ float4 norm4(float4 s, double inv, float ih, float il, float4 g)
{
    const float a[4] = {__fmul_rn(s.x, ih), __fmul_rn(s.y, ih), __fmul_rn(s.z, ih), __fmul_rn(s.w, ih)};
    const float low = fminf(fminf(fabsf(a[0]), fabsf(a[1])), fminf(fabsf(a[2]), fabsf(a[3])));
    // Below 2^-100 the carried errors would leave fp32's range: products in fp64, as behind.
    bool wide = inv < 0x1p-100 || low < 0x1p-100f;
    auto one = [&](float x, float a, float g) {
        const float ae = fmaf(x, il, fmaf(x, ih, -a));
        const float h = __fmul_rn(a, g);
        return __fadd_rn(h, fmaf(ae, g, fmaf(a, g, -h)));
    };
    const float4 y = make_float4(one(s.x, a[0], g.x), one(s.y, a[1], g.y), one(s.z, a[2], g.z), one(s.w, a[3], g.w));
    // A factor or a value past fp32's range leaves a NaN here (inf - inf), and
    // so do NaN inputs: fp64 tells them apart. (NaN in any makes the sum NaN.)
    const float sum = (y.x + y.y) + (y.z + y.w);
    wide |= sum != sum;
    if (wide)
        return make_float4((float)((double)s.x * inv * (double)g.x), (float)((double)s.y * inv * (double)g.y),
                           (float)((double)s.z * inv * (double)g.z), (float)((double)s.w * inv * (double)g.w));
    return y;
}

__device__ __forceinline__ uint32_t amax4(float4 v)
{
    return max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu),
               max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
}

__device__ __forceinline__ uint32_t quant4(float4 v, uint32_t sc)
{
    const float inv = mx_inv_scale(sc);
    return e4m3x4(mx_scaled(v.x, sc, inv), mx_scaled(v.y, sc, inv), mx_scaled(v.z, sc, inv), mx_scaled(v.w, sc, inv));
}

__device__ __forceinline__ double sumsq4(float4 v, double acc)
{
    acc = fma((double)v.x, (double)v.x, acc);
    acc = fma((double)v.y, (double)v.y, acc);
    acc = fma((double)v.z, (double)v.z, acc);
    return fma((double)v.w, (double)v.w, acc);
}

// FEW: at most 8 rows per SM, one wave of short rows and up to three of the
// longest. Registers are free then (40 to 162 a thread), and the norm weight (a
// parameter the operation just before must not write) is loaded before the
// programmatic-launch wait, which takes a round trip out of the chain.
template <int VPT, bool FEW>
__global__ void __launch_bounds__(128, FEW ? 1 : VPT <= 4 ? 8 : 4) add_rms_norm_mx_row(const float *x, const float *r, const float *w, float *sum_out,
                                                           float *norm_out, uint8_t *q, uint8_t *scales, int n, double inv_n, int ahead, float eps)
{
    __shared__ double part[4];
    const int tid = threadIdx.x, n4 = n / 4;
    const int64_t row = blockIdx.x;
    // Into L2: a first row while the previous kernel runs, later on the row `ahead`
    // behind this one.
    auto prefetch = [&](int64_t at) {
        const float *p = tid ? r : x;
        if (tid < 2 && p) prefetch_l2(p + at * n, (uint64_t)n * 4);
    };
    if (row < ahead) prefetch(row);
    const float4 *xr = reinterpret_cast<const float4 *>(x + row * n), *w4 = reinterpret_cast<const float4 *>(w);
    float4 wv[FEW ? VPT : 1];
    if (FEW) {
#pragma unroll
        for (int i = 0; i < VPT; i++)
            if (tid + 128 * i < n4) wv[FEW ? i : 0] = ld_param(w4 + tid + 128 * i);
    }
    pdl_wait();
    pdl_trigger();
    if (!FEW && row + ahead < gridDim.x) prefetch(row + ahead);
    float4 v[VPT];
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (tid + 128 * i < n4) v[i] = ld_stream_inflight(xr + tid + 128 * i);
    }
    if (r) {
        const float4 *rr = reinterpret_cast<const float4 *>(r + row * n);
        float4 b[VPT];
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            b[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (tid + 128 * i < n4) b[i] = ld_stream_inflight(rr + tid + 128 * i);
        }
#pragma unroll
        for (int i = 0; i < VPT; i++) v[i] = f4_add(v[i], b[i]);
    }
    if (sum_out) {
        float4 *so = reinterpret_cast<float4 *>(sum_out + row * n);
#pragma unroll
        for (int i = 0; i < VPT; i++)
            if (tid + 128 * i < n4) so[tid + 128 * i] = v[i];
    }
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < VPT; i++) ss += sumsq4(v[i], 0.0);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
    if ((tid & 31) == 0) part[tid >> 5] = ss;
    __syncthreads();
    ss = (part[0] + part[1]) + (part[2] + part[3]);
    const double inv = inv_sqrt64(fma(ss, inv_n, (double)eps));
    const float ih = (float)inv, il = (float)(inv - (double)ih);
    float4 *no = norm_out ? reinterpret_cast<float4 *>(norm_out + row * n) : nullptr;
    uint32_t *qo = reinterpret_cast<uint32_t *>(q + row * n);
    uint8_t *sco = scales + row * (n / kMxBlock);
    uint32_t amax[VPT];
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const int c = tid + 128 * i;
        if (c < n4) {
            v[i] = norm4(v[i], inv, ih, il, FEW ? wv[FEW ? i : 0] : ld_param(w4 + c));
            if (no) no[c] = v[i];
        }
        amax[i] = amax4(v[i]);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1)
#pragma unroll
        for (int i = 0; i < VPT; i++) amax[i] = max(amax[i], __shfl_xor_sync(kFull, amax[i], o));
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const int c = tid + 128 * i;
        if (c >= n4) break;
        const uint32_t sc = mx_scale<kMxEmaxFp8>(amax[i]);
        qo[c] = quant4(v[i], sc);
        if ((tid & 7) == 0) sco[c >> 3] = (uint8_t)sc;
    }
}

// Rows longer than 4096: one warp per row, staged in shared memory by bulk
// copies (TMA, 1-D) on an mbarrier, NS rows deep, as in add_rms_norm_bulk.
template <int NS>
__global__ void __launch_bounds__(32) add_rms_norm_mx_k(const float *x, const float *r, const float *w, float *sum_out,
                                                        float *norm_out, uint8_t *q, uint8_t *scales, int n, int64_t rows,
                                                        float eps, unsigned *err)
{
    extern __shared__ __align__(128) float buf[];  // [NS][x row | r row]
    __shared__ __align__(8) uint64_t bars[NS];
    const int lane = threadIdx.x;
    const uint32_t row_bytes = (uint32_t)n * 4;
    const int per_slot = r ? 2 * n : n;
    int64_t cur = blockIdx.x;
    const int64_t stride = gridDim.x;
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < NS; i++) mbar_init(&bars[i], 1);
        mbar_init_fence();
        prefetch_l2(x + cur * n, row_bytes);
        if (r) prefetch_l2(r + cur * n, row_bytes);
    }
    __syncwarp();
    pdl_wait();
    pdl_trigger();
    auto issue = [&](int slot, int64_t row) {
        if (lane == 0) {
            mbar_expect_tx(&bars[slot], r ? 2 * row_bytes : row_bytes);
            bulk_g2s(buf + slot * per_slot, x + row * n, row_bytes, &bars[slot]);
            if (r) bulk_g2s(buf + slot * per_slot + n, r + row * n, row_bytes, &bars[slot]);
        }
    };
    int slot = 0;
    uint32_t parity = 0;
    issue(0, cur);
    for (; cur < rows; cur += stride) {
        const int64_t nxt = cur + stride;
        if (NS == 2 && nxt < rows) issue(slot ^ 1, nxt);
        if (!__all_sync(kFull, mbar_wait(&bars[slot], (parity >> slot) & 1u, kWaitLimit))) {
            // Record the timeout, let this CTA's copies land (bounded), stop.
            if (lane == 0) flag_error(err, kErrWaitTimeout);
            mbar_wait(&bars[slot], (parity >> slot) & 1u, kWaitLimit);
            if (NS == 2 && nxt < rows) mbar_wait(&bars[slot ^ 1], (parity >> (slot ^ 1)) & 1u, kWaitLimit);
            return;
        }
        parity ^= 1u << slot;
        float4 *xs = reinterpret_cast<float4 *>(buf + slot * per_slot);
        const float4 *rs = reinterpret_cast<const float4 *>(buf + slot * per_slot + n);
        float4 *so = sum_out ? reinterpret_cast<float4 *>(sum_out + cur * n) : nullptr;
        double ss = 0.0;
#pragma unroll 4
        for (int i = lane; i < n / 4; i += 32) {
            float4 v = xs[i];
            if (r) {
                v = f4_add(v, rs[i]);
                xs[i] = v;  // read back by this lane below
            }
            if (so) so[i] = v;
            ss += sumsq4(v, 0.0);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
        const double inv = inv_sqrt64(ss / (double)n + (double)eps);
        const float ih = (float)inv, il = (float)(inv - (double)ih);
        const float4 *w4 = reinterpret_cast<const float4 *>(w);
        float4 *no = norm_out ? reinterpret_cast<float4 *>(norm_out + cur * n) : nullptr;
        uint32_t *qo = reinterpret_cast<uint32_t *>(q + cur * n);
        uint8_t *sco = scales + cur * (n / kMxBlock);
#pragma unroll 2
        for (int i0 = 0; i0 < n / 4; i0 += 32) {  // whole warps: the shuffles need every lane
            const int i = i0 + lane;
            const bool in = i < n / 4;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (in) {
                v = norm4(xs[i], inv, ih, il, ld_param(w4 + i));
                if (no) no[i] = v;
            }
            uint32_t amax = amax4(v);
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) amax = max(amax, __shfl_xor_sync(kFull, amax, o));
            if (!in) continue;
            const uint32_t sc = mx_scale<kMxEmaxFp8>(amax);
            qo[i] = quant4(v, sc);
            if ((lane & 7) == 0) sco[i >> 3] = (uint8_t)sc;
        }
        // Slot free for the next copy: this warp's reads and writes of it come first.
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (NS == 1) {
            if (nxt < rows) issue(0, nxt);
        } else {
            slot ^= 1;
        }
    }
}

template <int NS>
cudaError_t run_norm_mx(const LaunchCtx &c, const float *x, const float *r, const float *w, float *sum_out, float *norm_out,
                        uint8_t *q, uint8_t *scales, int n, int64_t rows, float eps)
{
    auto *k = add_rms_norm_mx_k<NS>;
    static const cudaError_t set = [&] {
        keep_driver_carveout((const void *)k);
        return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kNormMxMaxN * 4);
    }();
    if (set != cudaSuccess) return set;
    const size_t smem = (size_t)NS * (r ? 2 : 1) * n * 4;
    int per_sm = 0;
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k, 32, smem);
    if (e != cudaSuccess) return e;
    if (per_sm < 1) per_sm = 1;
    const int64_t grid = rows < (int64_t)c.n_sm * per_sm ? rows : (int64_t)c.n_sm * per_sm;
    launch_ks(c, k, dim3((unsigned)grid), dim3(32), smem, x, r, w, sum_out, norm_out, q, scales, n, rows, eps, c.err);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_mx_quantize(const LaunchCtx &c, const void *src, bool f16, uint8_t *q, uint8_t *scales, int to, int64_t n)
{
    const int64_t units = n / (f16 ? 8 : 4), blocks = (units + 256 * kUnits - 1) / (256 * kUnits);
    if (blocks <= 0) return cudaSuccess;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    const dim3 g((unsigned)blocks), b(256);
    if (f16) {
        const __half *s = (const __half *)src;
        if (to == kMxFp4) launch_k(c, mx_quantize_k<__half, true>, g, b, s, q, scales, units);
        else launch_k(c, mx_quantize_k<__half, false>, g, b, s, q, scales, units);
    } else {
        const float *s = (const float *)src;
        if (to == kMxFp4) launch_k(c, mx_quantize_k<float, true>, g, b, s, q, scales, units);
        else launch_k(c, mx_quantize_k<float, false>, g, b, s, q, scales, units);
    }
    return cudaGetLastError();
}

cudaError_t launch_mx_dequantize(const LaunchCtx &c, const uint8_t *q, const uint8_t *scales, int from, float *dst, int64_t n)
{
    const int64_t units = n / 4, blocks = (units + 256 * kUnits - 1) / (256 * kUnits);
    if (blocks <= 0) return cudaSuccess;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    const dim3 g((unsigned)blocks), b(256);
    if (from == kMxFp4) launch_k(c, mx_dequantize_k<true>, g, b, q, scales, dst, units);
    else launch_k(c, mx_dequantize_k<false>, g, b, q, scales, dst, units);
    return cudaGetLastError();
}

cudaError_t launch_add_rms_norm_mx(const LaunchCtx &c, const float *x, const float *r, const float *w, float *sum_out,
                                   float *norm_out, uint8_t *q, uint8_t *scales, int n, int64_t rows, float eps)
{
    if (rows <= 0) return cudaSuccess;
    if (n <= 0 || n % kMxBlock || n > kNormMxMaxN) return cudaErrorInvalidValue;
    if (n <= 4096) {
        if (rows > 0x7fffffffLL) return cudaErrorInvalidValue;
        const dim3 g((unsigned)rows), b(128);
        // About one wave of rows up to 2048 elements (8 CTAs per SM, more of the
        // shortest), two waves of longer ones (4 per SM).
        const int ahead = c.n_sm * 8;
        const double inv_n = 1.0 / n;
#define DS3_NORM(VPT)                                                                                                  \
    (rows <= ahead ? launch_k(c, add_rms_norm_mx_row<VPT, true>, g, b, x, r, w, sum_out, norm_out, q, scales, n, inv_n, \
                              ahead, eps)                                                                              \
                   : launch_k(c, add_rms_norm_mx_row<VPT, false>, g, b, x, r, w, sum_out, norm_out, q, scales, n,      \
                              inv_n, ahead, eps))
        if (n <= 512) DS3_NORM(1);
        else if (n <= 1024) DS3_NORM(2);
        else if (n <= 2048) DS3_NORM(4);
        else DS3_NORM(8);
#undef DS3_NORM
        return cudaGetLastError();
    }
    // Two rows in flight per warp when a warp has more than one and they fit.
    if (rows > c.n_sm && n <= kNormMxMaxN / 2)
        return run_norm_mx<2>(c, x, r, w, sum_out, norm_out, q, scales, n, rows, eps);
    return run_norm_mx<1>(c, x, r, w, sum_out, norm_out, q, scales, n, rows, eps);
}

}  // namespace ds3
