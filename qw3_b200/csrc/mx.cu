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
// blocks. A thread converts 8 consecutive elements; the four threads of a
// block share the largest magnitude by two shuffles. Inputs as for mx_scale:
// fp16 values convert to fp32 exactly.
__device__ __forceinline__ void load8(float (&v)[8], const float *p)
{
    const float4 a = ld_stream_inflight(reinterpret_cast<const float4 *>(p));
    const float4 b = ld_stream_inflight(reinterpret_cast<const float4 *>(p) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(float (&v)[8], const __half *p)
{
    const float4 a = ld_stream_inflight(reinterpret_cast<const float4 *>(p));
    const __half2 *h = reinterpret_cast<const __half2 *>(&a);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(h[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

template <typename T, bool FP4>
__global__ void __launch_bounds__(256) mx_quantize_k(const T *src, uint8_t *q, uint8_t *scales, int64_t n8)
{
    pdl_wait();
    pdl_trigger();
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;  // a block's four threads are in one warp
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (u < n8) load8(v, src + u * 8);
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
    amax = max(amax, __shfl_xor_sync(kFull, amax, 1));
    amax = max(amax, __shfl_xor_sync(kFull, amax, 2));
    if (u >= n8) return;
    const uint32_t sc = mx_scale<FP4 ? kMxEmaxFp4 : kMxEmaxFp8>(amax);
    const float inv = mx_inv_scale(sc);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = mx_scaled(v[i], sc, inv);
    if (FP4) {
        *reinterpret_cast<uint32_t *>(q + u * 4) = e2m1x8(v);
    } else {
        *reinterpret_cast<uint2 *>(q + u * 8) = make_uint2(e4m3x4(v[0], v[1], v[2], v[3]), e4m3x4(v[4], v[5], v[6], v[7]));
    }
    if ((threadIdx.x & 3) == 0) scales[u >> 2] = (uint8_t)sc;
}

// --------------------------------------------------------------- dequantise
// Both element types convert to fp16 exactly, and the product with a power of
// two is exact in fp32 (an element has at most 4 significant bits, so even
// results below the normal range are representable).
template <bool FP4>
__global__ void __launch_bounds__(256) mx_dequantize_k(const uint8_t *q, const uint8_t *scales, float *dst, int64_t n8)
{
    pdl_wait();
    pdl_trigger();
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (u >= n8) return;
    uint32_t h[4];
    if (FP4) {
        const uint32_t w = __ldcs(reinterpret_cast<const uint32_t *>(q + u * 4));
        asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
            "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
            "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
            "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
            : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
            : "r"(w));
    } else {
        const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(q + u * 8));
        asm("{\n\t.reg .b16 a, b, c, d;\n\t"
            "mov.b32 {a, b}, %4;\n\tmov.b32 {c, d}, %5;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t"
            "cvt.rn.f16x2.e4m3x2 %2, c;\n\tcvt.rn.f16x2.e4m3x2 %3, d;\n\t}"
            : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
            : "r"(w.x), "r"(w.y));
    }
    const float s = mx_scale_value(scales[u >> 2]);
    float2 f[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        f[i] = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
        f[i].x *= s;
        f[i].y *= s;
    }
    float4 *o = reinterpret_cast<float4 *>(dst + u * 8);
    __stcs(o, make_float4(f[0].x, f[0].y, f[1].x, f[1].y));
    __stcs(o + 1, make_float4(f[2].x, f[2].y, f[3].x, f[3].y));
}

// ------------------------------------------------ residual add + norm + MXFP8
// s = x + r (fp32, as add_rms_norm), then n = s * w / sqrt(mean(s^2) + eps).
// The sum of squares and the inverse root are fp64, and the two products are
// carried as a float and its error (fma), so each normed value is the exact
// one rounded once to fp32 (but for a chance of about 2^-22): the 8-bit codes,
// which jump where a value crosses a rounding border, then do not depend on
// the order of the sum.
//
// One warp per row; x and r rows are staged in shared memory by bulk copies
// (TMA, 1-D) on an mbarrier, NS rows deep, as in add_rms_norm_bulk. The row
// stays in shared memory for the two passes (squares, output). Lane l works on
// elements 4 l .. 4 l + 3 of every 128: an MX block is 8 lanes.
constexpr int kNormMxMaxN = 16384;

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
            ss = fma((double)v.x, (double)v.x, ss);
            ss = fma((double)v.y, (double)v.y, ss);
            ss = fma((double)v.z, (double)v.z, ss);
            ss = fma((double)v.w, (double)v.w, ss);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
        const double inv = 1.0 / sqrt(ss / (double)n + (double)eps);
        const float ih = (float)inv, il = (float)(inv - (double)ih);
        const float4 *w4 = reinterpret_cast<const float4 *>(w);
        float4 *no = norm_out ? reinterpret_cast<float4 *>(norm_out + cur * n) : nullptr;
        uint32_t *qo = reinterpret_cast<uint32_t *>(q + cur * n);
        uint8_t *sco = scales + cur * (n / kMxBlock);
        // Below 2^-100 the carried errors would leave fp32's range: products in fp64.
        const bool tiny = inv < 0x1p-100;
        auto norm1 = [&](float s, float g) {
            const float a = __fmul_rn(s, ih);
            if (tiny || fabsf(a) < 0x1p-100f) return (float)((double)s * inv * (double)g);
            const float ae = fmaf(s, il, fmaf(s, ih, -a));
            const float h = __fmul_rn(a, g);
            return __fadd_rn(h, fmaf(ae, g, fmaf(a, g, -h)));
        };
#pragma unroll 2
        for (int i0 = 0; i0 < n / 4; i0 += 32) {  // whole warps: the shuffles need every lane
            const int i = i0 + lane;
            const bool in = i < n / 4;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (in) {
                const float4 s = xs[i], g = ld_param(w4 + i);
                v = make_float4(norm1(s.x, g.x), norm1(s.y, g.y), norm1(s.z, g.z), norm1(s.w, g.w));
                if (no) no[i] = v;
            }
            uint32_t amax = max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu),
                                max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) amax = max(amax, __shfl_xor_sync(kFull, amax, o));
            if (!in) continue;
            const uint32_t sc = mx_scale<kMxEmaxFp8>(amax);
            const float is = mx_inv_scale(sc);
            qo[i] = e4m3x4(mx_scaled(v.x, sc, is), mx_scaled(v.y, sc, is), mx_scaled(v.z, sc, is), mx_scaled(v.w, sc, is));
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
    const int64_t n8 = n / 8;
    if (n8 <= 0) return cudaSuccess;
    const int64_t blocks = (n8 + 255) / 256;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    const dim3 g((unsigned)blocks), b(256);
    if (f16) {
        const __half *s = (const __half *)src;
        if (to == kMxFp4) launch_k(c, mx_quantize_k<__half, true>, g, b, s, q, scales, n8);
        else launch_k(c, mx_quantize_k<__half, false>, g, b, s, q, scales, n8);
    } else {
        const float *s = (const float *)src;
        if (to == kMxFp4) launch_k(c, mx_quantize_k<float, true>, g, b, s, q, scales, n8);
        else launch_k(c, mx_quantize_k<float, false>, g, b, s, q, scales, n8);
    }
    return cudaGetLastError();
}

cudaError_t launch_mx_dequantize(const LaunchCtx &c, const uint8_t *q, const uint8_t *scales, int from, float *dst, int64_t n)
{
    const int64_t n8 = n / 8;
    if (n8 <= 0) return cudaSuccess;
    const int64_t blocks = (n8 + 255) / 256;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
    const dim3 g((unsigned)blocks), b(256);
    if (from == kMxFp4) launch_k(c, mx_dequantize_k<true>, g, b, q, scales, dst, n8);
    else launch_k(c, mx_dequantize_k<false>, g, b, q, scales, dst, n8);
    return cudaGetLastError();
}

cudaError_t launch_add_rms_norm_mx(const LaunchCtx &c, const float *x, const float *r, const float *w, float *sum_out,
                                   float *norm_out, uint8_t *q, uint8_t *scales, int n, int64_t rows, float eps)
{
    if (rows <= 0) return cudaSuccess;
    if (n <= 0 || n % kMxBlock || n > kNormMxMaxN) return cudaErrorInvalidValue;
    // Two rows in flight per warp when a warp has more than one and they fit.
    if (rows > c.n_sm && n <= kNormMxMaxN / 2)
        return run_norm_mx<2>(c, x, r, w, sum_out, norm_out, q, scales, n, rows, eps);
    return run_norm_mx<1>(c, x, r, w, sum_out, norm_out, q, scales, n, rows, eps);
}

}  // namespace ds3
