// Product of int8 activations and int8 weights with a scale for each token and each output channel:
//
//   out[m, n] = T(float(sum_k x[m, k] * w[n, k]) * x_scale[m] * w_scale[n] + bias[n])
//
// The sum is exact in int32 (k <= 131071), so neither the split nor the order of a tile's work shows in the result;
// conversion, the two products and the bias are fp32, the result is rounded once to T.
// No counterpart in the reference: it is the product whose output its all-reduce sums.
#include <hip/hip_runtime.h>
#include <stdio.h>

#include "../../include/tbvcoll.h"
#include "tbv_device.h"

namespace tbv {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

struct MatArgs {
    void* out;
    const signed char* x; const float* x_scale;
    const signed char* w; const float* w_scale;
    const void* bias;
    size_t out_stride, x_stride, w_stride;
    unsigned m, n, k;
    unsigned x_scale_step, w_scale_step;      // 1, or 0 for one scale of the whole operand
};

template <int DT> __device__ __forceinline__ float mat_elem(const void* p, size_t i)
{
    if (DT == 0) return ((const float*)p)[i];
    if (DT == 1) return (float)((const _Float16*)p)[i];
    return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
}

template <int DT> __device__ __forceinline__ void mat_store(void* p, size_t i, float v)
{
    if (DT == 0) ((float*)p)[i] = v;
    else if (DT == 1) ((_Float16*)p)[i] = (_Float16)v;
    else ((__bf16*)p)[i] = (__bf16)v;
}

// 16 bytes of a row of k bytes from byte c on, zeros beyond its end; any alignment (the loads need none here).
__device__ __forceinline__ i32x4 row_bytes(const signed char* row, unsigned c, unsigned k)
{
    i32x4 v = {0, 0, 0, 0};
    if (c + 16 <= k) {
        __builtin_memcpy(&v, row + c, 16);
    } else if (c < k) {
        for (unsigned j = 0; j < k - c; j++) v[j >> 2] |= (int)((unsigned)(unsigned char)row[c + j] << (8 * (j & 3)));
    }
    return v;
}

// Any alignment, any strides: 64 x 64 tile, four waves of 32 x 32, 64 bytes of k a step.
template <int DT>
__global__ __launch_bounds__(256) void k_mat_any(MatArgs g)
{
    constexpr int LD = 64 + 16;                      // row pitch in the LDS: 16-byte rows of eight lanes fall into different banks
    __shared__ __attribute__((aligned(16))) signed char sx[64 * LD], sw[64 * LD];
    const unsigned tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const unsigned tiles_m = (g.m + 63) / 64, m0 = (blockIdx.x % tiles_m) * 64, n0 = (blockIdx.x / tiles_m) * 64;
    const unsigned lr = tid >> 2, lc = (tid & 3) * 16;
    const unsigned xm = m0 + lr < g.m ? m0 + lr : g.m - 1, wn = n0 + lr < g.n ? n0 + lr : g.n - 1;
    const signed char *xr = g.x + (size_t)xm * g.x_stride, *wr = g.w + (size_t)wn * g.w_stride;
    const unsigned wm = (wave & 1) * 32, wc = (wave >> 1) * 32;
    i32x16 acc = {};
    for (unsigned k0 = 0; k0 < g.k; k0 += 64) {
        const i32x4 vx = row_bytes(xr, k0 + lc, g.k), vw = row_bytes(wr, k0 + lc, g.k);
        __syncthreads();
        *(i32x4*)(sx + lr * LD + lc) = vx;
        *(i32x4*)(sw + lr * LD + lc) = vw;
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const unsigned off = (lane & 31) * LD + h * 32 + (lane >> 5) * 16;
            acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(*(const i32x4*)(sx + wm * LD + off), *(const i32x4*)(sw + wc * LD + off), acc, 0, 0, 0);
        }
    }
    const unsigned n = n0 + wc + (lane & 31);
    if (n >= g.n) return;
    const float ws = g.w_scale[(size_t)n * g.w_scale_step], b = g.bias ? mat_elem<DT>(g.bias, n) : 0.0f;
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const unsigned m = m0 + wm + (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3);
        if (m < g.m) mat_store<DT>(g.out, (size_t)m * g.out_stride + n, (float)acc[r] * g.x_scale[(size_t)m * g.x_scale_step] * ws + b);
    }
}

template <int DT> void launch_mat(const MatArgs& g, hipStream_t st)
{
    const size_t tiles = (size_t)((g.m + 63) / 64) * ((g.n + 63) / 64);
    k_mat_any<DT><<<dim3((unsigned)tiles), 256, 0, st>>>(g);
}

}  // namespace

}  // namespace tbv

#define MAT_FAIL(...) do { fprintf(stderr, "[tbvcoll] int8 product: " __VA_ARGS__); fputc('\n', stderr); return -1; } while (0)

namespace {
// [p, p + bytes) of two buffers have a byte in common
inline bool meet(const void* p, size_t pn, const void* q, size_t qn)
{
    return p && q && pn && qn && (uintptr_t)p < (uintptr_t)q + qn && (uintptr_t)q < (uintptr_t)p + pn;
}
inline size_t extent(size_t rows, size_t stride, size_t cols) { return rows && cols ? (rows - 1) * stride + cols : 0; }
}  // namespace

extern "C" int tbv_step_matmul_i8(const tbv_matmul_i8* c, void* stream)
{
    using namespace tbv;
    if (!c) MAT_FAIL("null arguments");
    if (c->dtype < 0 || c->dtype > 2) MAT_FAIL("unknown dtype %lld", (long long)c->dtype);
    const size_t esz = c->dtype == 0 ? 4 : 2;
    if (c->m < 0 || c->n < 0 || c->k < 0 || c->m > 0x7fffffff || c->n > 0x7fffffff) MAT_FAIL("sizes %lld x %lld x %lld", (long long)c->m, (long long)c->n, (long long)c->k);
    if (c->k > TBV_MATMUL_I8_MAX_K) MAT_FAIL("k = %lld: beyond %d the int32 sum can overflow", (long long)c->k, TBV_MATMUL_I8_MAX_K);
    if (c->m == 0 || c->n == 0) return 0;
    if (!c->out || !c->x_scale || !c->w_scale || (c->k && (!c->x || !c->w))) MAT_FAIL("null buffer");
    if ((c->x_scales != 1 && c->x_scales != c->m) || (c->w_scales != 1 && c->w_scales != c->n)) MAT_FAIL("one scale, or one for each row");
    if ((c->m > 1 && (c->out_stride < c->n || c->x_stride < c->k)) || (c->n > 1 && c->w_stride < c->k)) MAT_FAIL("row strides shorter than a row");
    const int64_t far = (int64_t)1 << 40;
    if (c->out_stride > far || c->x_stride > far || c->w_stride > far) MAT_FAIL("row strides beyond 2^40");
    if (((uintptr_t)c->out % esz) || ((uintptr_t)c->bias % esz) || ((uintptr_t)c->x_scale % 4) || ((uintptr_t)c->w_scale % 4)) MAT_FAIL("out, bias and scales must be aligned to their elements");
    const size_t tiles = ((size_t)c->m + 63) / 64 * (((size_t)c->n + 63) / 64);
    if (tiles > 0x7fffffffu) MAT_FAIL("%lld x %lld results are too many for one launch", (long long)c->m, (long long)c->n);
    const size_t out_bytes = extent(c->m, c->out_stride, c->n) * esz;
    if (meet(c->out, out_bytes, c->x, extent(c->m, c->x_stride, c->k)) || meet(c->out, out_bytes, c->w, extent(c->n, c->w_stride, c->k)) ||
        meet(c->out, out_bytes, c->x_scale, 4 * (size_t)c->x_scales) || meet(c->out, out_bytes, c->w_scale, 4 * (size_t)c->w_scales) ||
        meet(c->out, out_bytes, c->bias, (size_t)c->n * esz)) MAT_FAIL("out overlaps an operand");
    MatArgs g{};
    g.out = c->out; g.x = c->x; g.x_scale = c->x_scale; g.w = c->w; g.w_scale = c->w_scale; g.bias = c->bias;
    g.out_stride = (size_t)c->out_stride; g.x_stride = (size_t)c->x_stride; g.w_stride = (size_t)c->w_stride;
    g.m = (unsigned)c->m; g.n = (unsigned)c->n; g.k = (unsigned)c->k;
    g.x_scale_step = c->x_scales != 1; g.w_scale_step = c->w_scales != 1;
    hipStream_t st = (hipStream_t)stream;
    switch (c->dtype) {
        case 0: launch_mat<0>(g, st); break;
        case 1: launch_mat<1>(g, st); break;
        default: launch_mat<2>(g, st);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) MAT_FAIL("launch failed: %s", hipGetErrorString(e));
    return 0;
}
