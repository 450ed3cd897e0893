// Rows of a hidden state as int8 codes with one scale a row: the left operand of the int8 product (tbv_matmul.hip).
//
//   scale = max(f32(max|x| / 127), 2^-126),  code = x / scale to the nearest integer, ties to even
//
// The quotient is decided exactly, not from a rounded division: with q the rounded product x * (1/scale) the remainder
// x - q*scale is exact in fp32 (one fused multiply-add: |x - q*scale| < scale and both are multiples of the smaller
// operand's last place), so comparing twice the remainder with the scale says whether q or its neighbour is nearest.
// No counterpart in the reference, whose planned int8 codec is for the wire (reports/12_references.md:134).
#include <hip/hip_runtime.h>
#include <stdio.h>

#include <type_traits>

#include "../../include/tbvcoll.h"
#include "tbv_device.h"
#include "tbv_step.h"

namespace tbv {

namespace {

// 16 bytes of a row: the elements as fp32, and their magnitudes as unsigned numbers.  The order of those is the order of
// the magnitudes, with infinities and NaNs above every finite value, so one integer maximum finds max|x| and says
// whether the row is finite; 16-bit types take two elements an instruction.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
template <int DT> struct Vec {
    static constexpr int N = 8;
    static constexpr uint32_t INF = DT == 1 ? 0x7c00u : 0x7f80u;
    static __device__ __forceinline__ uint32_t top(u32x4 v, uint32_t t)
    {
#pragma unroll
        for (int i = 0; i < 4; i++) t = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu), __builtin_bit_cast(u16x2, t)));
        return t;
    }
    static __device__ __forceinline__ uint32_t join(uint32_t t, uint32_t o)
    {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, t), __builtin_bit_cast(u16x2, o)));
    }
    static __device__ __forceinline__ uint32_t whole(uint32_t t) { const uint32_t h = t >> 16, l = t & 0xffffu; return h > l ? h : l; }
    static __device__ __forceinline__ float value(uint32_t bits) { return DT == 1 ? (float)__builtin_bit_cast(_Float16, (uint16_t)bits) : __uint_as_float(bits << 16); }
    static __device__ __forceinline__ void unpack(u32x4 v, float* f)
    {
        if (DT == 1) {
            const f16x8 h = __builtin_bit_cast(f16x8, v);
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = (float)h[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) { f[2 * i] = __uint_as_float(v[i] << 16); f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u); }
        }
    }
};
template <> struct Vec<0> {
    static constexpr int N = 4;
    static constexpr uint32_t INF = 0x7f800000u;
    static __device__ __forceinline__ uint32_t join(uint32_t t, uint32_t o) { return t > o ? t : o; }
    static __device__ __forceinline__ uint32_t top(u32x4 v, uint32_t t)
    {
#pragma unroll
        for (int i = 0; i < 4; i++) t = join(t, v[i] & 0x7fffffffu);
        return t;
    }
    static __device__ __forceinline__ uint32_t whole(uint32_t t) { return t; }
    static __device__ __forceinline__ float value(uint32_t bits) { return __uint_as_float(bits); }
    static __device__ __forceinline__ void unpack(u32x4 v, float* f)
    {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = __uint_as_float(v[i]);
    }
};

// Vector j of a row of `hidden` elements; elements beyond its end are zeros.  Rows may start anywhere: the loads need no
// alignment here (rows of odd length cost a tenth of the rate).
template <int DT> __device__ __forceinline__ u32x4 row_vec(const char* row, unsigned j, unsigned hidden)
{
    constexpr unsigned N = Vec<DT>::N, ESZ = 16 / N;
    u32x4 v = {0, 0, 0, 0};
    if ((j + 1) * N <= hidden) {
        __builtin_memcpy(&v, row + (size_t)j * 16, 16);
    } else if (j * N < hidden) {
        for (unsigned e = 0; e < hidden - j * N; e++) {
            if (DT == 0) v[e] = *(const uint32_t*)(row + (size_t)j * 16 + e * ESZ);
            else v[e >> 1] |= (uint32_t)*(const uint16_t*)(row + (size_t)j * 16 + e * ESZ) << (16 * (e & 1));
        }
    }
    return v;
}

// The codes of one vector, for a scale s >= 2^-126 (NaN: zeros).  x/s + 1.5 * 2^23 in one rounding leaves the rounded
// quotient in the low bits; where its remainder reaches half a scale (a tie, or the product with 1/s fell on the wrong
// side) the nearest code is decided from the remainder.
template <int DT> __device__ __forceinline__ void store_codes(signed char* row, unsigned j, unsigned hidden, u32x4 v, float s, float inv, bool fine)
{
    constexpr int N = Vec<DT>::N;
    float x[N], rest = 0.0f;
    uint32_t t[N];
    Vec<DT>::unpack(v, x);
#pragma unroll
    for (int e = 0; e < N; e++) {
        const float m = __builtin_fmaf(x[e], inv, 12582912.0f), q = m - 12582912.0f;
        t[e] = __float_as_uint(m);
        rest = __builtin_fmaxf(rest, __builtin_fabsf(__builtin_fmaf(-q, s, x[e])));
    }
    if (rest + rest >= s) {
#pragma unroll
        for (int e = 0; e < N; e++) {
            const float r = __builtin_fmaf(-(__uint_as_float(t[e]) - 12582912.0f), s, x[e]), twice = __builtin_fabsf(r + r);
            if (twice > s || (twice == s && (t[e] & 1))) t[e] += r > 0.0f ? 1 : -1;
        }
    }
    uint32_t o[N / 4];
#pragma unroll
    for (int e = 0; e < N / 4; e++) {
        const uint32_t lo = __builtin_amdgcn_perm(t[4 * e + 1], t[4 * e], 0x0c0c0400u), hi = __builtin_amdgcn_perm(t[4 * e + 3], t[4 * e + 2], 0x04000c0cu);
        o[e] = fine ? lo | hi : 0u;
    }
    // Whole vectors are written through the L2 (a relaxed store of agent scope): lines that are still dirty when the kernel
    // ends stand between it and the next one.  2048 x 4096 bf16 9.0 -> 7.9 us, with the product of the codes behind it 45.8 -> 44.5;
    // non-temporal ones, which the Infinity Cache does not keep, 7.7 and 45.2, with a copy behind 12.6 against 11.8 (ordinary: 12.7).
    typedef typename std::conditional<N == 8, unsigned long long, uint32_t>::type T;
    signed char* const to = row + (size_t)j * N;
    if ((j + 1) * N <= hidden) {
        T v;
        __builtin_memcpy(&v, o, N);
        if (((uintptr_t)to & (N - 1)) == 0) __hip_atomic_store((T*)to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        else __builtin_memcpy(to, &v, N);
    }
    else for (unsigned e = 0; j * N + e < hidden; e++) to[e] = (signed char)(o[e >> 2] >> (8 * (e & 3)));
}

struct RowScale { float s, inv; bool fine; };
template <int DT> __device__ __forceinline__ RowScale row_scale(uint32_t top)
{
    top = Vec<DT>::whole(top);
    const bool fine = top < Vec<DT>::INF;
    const float s = fine ? __builtin_fmaxf(Vec<DT>::value(top) / 127.0f, 0x1p-126f) : __builtin_nanf("");
    return {s, 1.0f / s, fine};
}

struct RowsArgs { signed char* codes; float* scale; const char* x; size_t code_stride, x_stride; unsigned rows, hidden; };   // x_stride in bytes

// A row is held in registers, read once: R rows to a block, L lanes to a row, V vectors to a lane (L > 64: one row).  What
// bounds it: memory and a launch, 25 MB (2048 x 4096 bf16) in 6.8 us out of the Infinity Cache, 7.1 us out of memory, 42 MB
// (fp32) in 8.4 and 9.1.
template <int DT, int L, int V>
__global__ __launch_bounds__(L <= 64 ? 256 : L) void k_quant_rows(RowsArgs g)
{
    constexpr int R = L <= 64 ? 256 / L : 1;          // rows that share a block are (parts of) waves
    const unsigned lane = threadIdx.x % L;
    const size_t row = flat_block() * R + threadIdx.x / L;
    if (row >= g.rows) return;
    const char* const xr = g.x + row * g.x_stride;
    u32x4 v[V];
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = row_vec<DT>(xr, lane + i * L, g.hidden);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < V; i++) top = Vec<DT>::top(v[i], top);
#pragma unroll
    for (int off = (L < 64 ? L : 64) / 2; off >= 1; off >>= 1) top = Vec<DT>::join(top, __shfl_xor(top, off, 64));
    if (L > 64) {
        __shared__ uint32_t wave_top[L > 64 ? L / 64 : 1];
        if ((lane & 63) == 0) wave_top[lane >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < L / 64; w++) top = Vec<DT>::join(top, wave_top[w]);
    }
    const RowScale k = row_scale<DT>(top);
    signed char* const cr = g.codes + row * g.code_stride;
#pragma unroll
    for (int i = 0; i < V; i++) if ((lane + i * L) * Vec<DT>::N < g.hidden) store_codes<DT>(cr, lane + i * L, g.hidden, v[i], k.s, k.inv, k.fine);
    if (lane == 0) g.scale[row] = k.s;
}

// Rows too long for the registers of a block are read twice (the second time from the caches).
template <int DT>
__global__ __launch_bounds__(1024) void k_quant_long(RowsArgs g)
{
    __shared__ uint32_t wave_top[16];
    const unsigned lane = threadIdx.x, vecs = (g.hidden + Vec<DT>::N - 1) / Vec<DT>::N;
    const size_t row = flat_block();
    if (row >= g.rows) return;
    const char* const xr = g.x + row * g.x_stride;
    uint32_t top = 0;
#pragma unroll 4
    for (unsigned j = lane; j < vecs; j += 1024) top = Vec<DT>::top(row_vec<DT>(xr, j, g.hidden), top);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top = Vec<DT>::join(top, __shfl_xor(top, off, 64));
    if ((lane & 63) == 0) wave_top[lane >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; w++) top = Vec<DT>::join(top, wave_top[w]);
    const RowScale k = row_scale<DT>(top);
    signed char* const cr = g.codes + row * g.code_stride;
#pragma unroll 2
    for (unsigned j = lane; j < vecs; j += 1024) store_codes<DT>(cr, j, g.hidden, row_vec<DT>(xr, j, g.hidden), k.s, k.inv, k.fine);
    if (lane == 0) g.scale[row] = k.s;
}

template <int DT> void launch_quant(const RowsArgs& g, hipStream_t st)
{
    const unsigned vecs = (g.hidden + Vec<DT>::N - 1) / Vec<DT>::N;
#define QUANT(L, V) k_quant_rows<DT, L, V><<<flat_grid(L <= 64 ? ((size_t)g.rows + ROWS(L) - 1) / ROWS(L) : g.rows), L <= 64 ? 256 : L, 0, st>>>(g)
#define ROWS(L) (256 / (L <= 64 ? L : 64))
    if (vecs <= 8) QUANT(8, 1);
    else if (vecs <= 16) QUANT(16, 1);
    else if (vecs <= 32) QUANT(32, 1);
    else if (vecs <= 64) QUANT(64, 1);
    else if (vecs <= 128) QUANT(64, 2);
    else if (vecs <= 256) QUANT(256, 1);
    else if (vecs <= 512) QUANT(256, 2);
    else if (vecs <= 1024) QUANT(256, 4);
    else if (vecs <= 2048) QUANT(512, 4);
    else if (vecs <= 4096) QUANT(1024, 4);
    else k_quant_long<DT><<<flat_grid(g.rows), 1024, 0, st>>>(g);
#undef QUANT
#undef ROWS
}

}  // namespace

}  // namespace tbv

#define I8_FAIL(...) do { fprintf(stderr, "[tbvcoll] int8 rows: " __VA_ARGS__); fputc('\n', stderr); return -1; } while (0)

extern "C" int tbv_step_quantize_i8(const tbv_quantize_i8* c, void* stream)
{
    using namespace tbv;
    if (!c) I8_FAIL("null arguments");
    if (c->dtype < 0 || c->dtype > 2) I8_FAIL("unknown dtype %lld", (long long)c->dtype);
    if (c->rows < 0 || c->hidden < 0 || c->rows > 0x7fffffff || c->hidden > 0x7fffffff) I8_FAIL("%lld rows of %lld elements: at most 2^31 - 1 of either", (long long)c->rows, (long long)c->hidden);
    if (c->rows == 0) return 0;
    const size_t esz = c->dtype == 0 ? 4 : 2, rows = (size_t)c->rows, hidden = (size_t)c->hidden;
    if (!c->scale || (hidden && (!c->codes || !c->x))) I8_FAIL("null buffer");
    if (((uintptr_t)c->x % esz) || ((uintptr_t)c->scale % 4)) I8_FAIL("x and scale must be aligned to their elements");
    const int64_t far = (int64_t)1 << 30;              // with 2^31 rows: no extent overflows
    if (rows > 1 && (c->code_stride < c->hidden || c->x_stride < c->hidden || c->code_stride > far || c->x_stride > far)) I8_FAIL("row strides shorter than a row of %zu, or beyond 2^30", hidden);
    const uintptr_t x0 = (uintptr_t)c->x, x1 = x0 + ((rows > 1 ? (rows - 1) * (size_t)c->x_stride : 0) + hidden) * esz;
    const uintptr_t c0 = (uintptr_t)c->codes, c1 = c0 + (rows > 1 ? (rows - 1) * (size_t)c->code_stride : 0) + hidden, s0 = (uintptr_t)c->scale, s1 = s0 + 4 * rows;
    if (hidden && ((x0 < c1 && c0 < x1) || (x0 < s1 && s0 < x1) || (c0 < s1 && s0 < c1))) I8_FAIL("codes, scale and x must not overlap");
    hipStream_t st = (hipStream_t)stream;
    const RowsArgs g{c->codes, c->scale, (const char*)c->x, rows > 1 ? (size_t)c->code_stride : 0, rows > 1 ? (size_t)c->x_stride * esz : 0, (unsigned)rows, (unsigned)hidden};
    switch (c->dtype) {
        case 0: launch_quant<0>(g, st); break;
        case 1: launch_quant<1>(g, st); break;
        default: launch_quant<2>(g, st);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) I8_FAIL("launch failed: %s", hipGetErrorString(e));
    return 0;
}
