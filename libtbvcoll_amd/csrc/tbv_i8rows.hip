// Rows of a hidden state as int8 codes with one scale a row: the left operand of the int8 product (tbv_matmul.hip).
//
//   scale = max(f32(max|x| / 127), 2^-126),  code = x / scale to the nearest integer, ties to even
//
// The quotient is decided exactly, not from a rounded division: with q = rint(x * (1/scale)) the remainder
// x - q*scale is exact in fp32 (one fused multiply-add: |x - q*scale| < scale and both are multiples of the smaller
// operand's last place), so comparing twice the remainder with the scale says whether q or its neighbour is nearest.
// No counterpart in the reference, whose planned int8 codec is for the wire (reports/12_references.md:134).
#include <hip/hip_runtime.h>
#include <stdio.h>

#include "../../include/tbvcoll.h"
#include "tbv_device.h"

namespace tbv {

namespace {

template <int DT> __device__ __forceinline__ float row_elem(const void* p, size_t i)
{
    if (DT == 0) return ((const float*)p)[i];
    if (DT == 1) return (float)((const _Float16*)p)[i];
    return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
}

// The code of x for a finite scale s >= 2^-126 (see the head of the file).
__device__ __forceinline__ int row_code(float x, float s, float inv)
{
    const float q = __builtin_rintf(x * inv);
    const float r = __builtin_fmaf(-q, s, x), twice = __builtin_fabsf(r + r);
    int code = (int)q;
    if (twice > s || (twice == s && (code & 1))) code += r > 0.0f ? 1 : -1;
    return code;
}

template <int DT>
__global__ __launch_bounds__(256) void k_quant_rows(signed char* codes, float* scale, const void* x, size_t code_stride,
                                                    size_t x_stride, unsigned hidden)
{
    __shared__ float wave_top[4];
    const size_t row = blockIdx.x;
    const char* xr = (const char*)x + row * x_stride * (DT == 0 ? 4 : 2);
    float top = 0.0f;
    bool bad = false;
    for (unsigned i = threadIdx.x; i < hidden; i += 256) {
        const float v = row_elem<DT>(xr, i);
        bad |= !(__builtin_fabsf(v) < __builtin_inff());
        top = __builtin_fmaxf(top, __builtin_fabsf(v));
    }
    if (bad) top = __builtin_nanf("");
    // a row that is not finite has no scale: NaN, codes 0
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const float o = __shfl_xor(top, off, 64);
        top = (top != top || o != o) ? __builtin_nanf("") : __builtin_fmaxf(top, o);
    }
    if ((threadIdx.x & 63) == 0) wave_top[threadIdx.x >> 6] = top;
    __syncthreads();
    top = 0.0f;
    for (int w = 0; w < 4; w++) top = (top != top || wave_top[w] != wave_top[w]) ? __builtin_nanf("") : __builtin_fmaxf(top, wave_top[w]);
    const bool fine = top == top;
    const float s = fine ? __builtin_fmaxf(top / 127.0f, 0x1p-126f) : top, inv = 1.0f / s;
    signed char* cr = codes + row * code_stride;
    for (unsigned i = threadIdx.x; i < hidden; i += 256) cr[i] = fine ? (signed char)row_code(row_elem<DT>(xr, i), s, inv) : 0;
    if (threadIdx.x == 0) scale[row] = s;
}

}  // namespace

}  // namespace tbv

#define I8_FAIL(...) do { fprintf(stderr, "[tbvcoll] int8 rows: " __VA_ARGS__); fputc('\n', stderr); return -1; } while (0)

extern "C" int tbv_step_quantize_i8(signed char* codes, size_t code_stride, float* scale, const void* x, size_t x_stride,
                                    size_t rows, size_t hidden, int dtype, void* stream)
{
    using namespace tbv;
    if (dtype < 0 || dtype > 2) I8_FAIL("unknown dtype %d", dtype);
    if (rows > 0x7fffffffu || hidden > 0x7fffffffu) I8_FAIL("%zu rows of %zu elements: at most 2^31 - 1 of either", rows, hidden);
    if (rows == 0) return 0;
    const size_t esz = dtype == 0 ? 4 : 2;
    if (!scale || (hidden && (!codes || !x))) I8_FAIL("null buffer");
    if (((uintptr_t)x % esz) || ((uintptr_t)scale % 4)) I8_FAIL("x and scale must be aligned to their elements");
    if (rows > 1 && (code_stride < hidden || x_stride < hidden)) I8_FAIL("row strides shorter than a row of %zu", hidden);
    const uintptr_t x0 = (uintptr_t)x, x1 = x0 + ((rows - 1) * x_stride + hidden) * esz;
    const uintptr_t c0 = (uintptr_t)codes, c1 = c0 + (rows - 1) * code_stride + hidden, s0 = (uintptr_t)scale, s1 = s0 + 4 * rows;
    if (hidden && ((x0 < c1 && c0 < x1) || (x0 < s1 && s0 < x1) || (c0 < s1 && s0 < c1))) I8_FAIL("codes, scale and x must not overlap");
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case 0: k_quant_rows<0><<<dim3((unsigned)rows), 256, 0, st>>>(codes, scale, x, code_stride, x_stride, (unsigned)hidden); break;
        case 1: k_quant_rows<1><<<dim3((unsigned)rows), 256, 0, st>>>(codes, scale, x, code_stride, x_stride, (unsigned)hidden); break;
        default: k_quant_rows<2><<<dim3((unsigned)rows), 256, 0, st>>>(codes, scale, x, code_stride, x_stride, (unsigned)hidden);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) I8_FAIL("launch failed: %s", hipGetErrorString(e));
    return 0;
}
