// Product of int8 activations and int8 weights with a scale for each token and each output channel:
//
//   out[m, n] = T(float(sum_k x[m, k] * w[n, k]) * x_scale[m] * w_scale[n] + bias[n])
//
// The sum is exact in int32 (k <= 131071), so neither the split nor the order of a tile's work shows in the result;
// conversion, the two products and the bias are fp32, the result is rounded once to T (fp16: the last multiply-add straight to fp16,
// in every kernel alike; a test holds a row's bits over all of them).
// No counterpart in the reference: it is the product whose output its all-reduce sums.
#include <hip/hip_runtime.h>
#include <stdio.h>

#include "../../include/tbvcoll.h"
#include "tbv_device.h"
#include "tbv_step.h"
#include "tbv_tiles.h"

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

// Bytes c .. c + 15 of a row of k >= 16 bytes that starts anywhere (the loads need no alignment here), zeros beyond its
// end: asked for with no branch, from where 16 bytes are left, and shifted into place once they have come.
[[maybe_unused]] __device__ __forceinline__ i32x4 ask16(const signed char* row, unsigned c, unsigned k)
{
    i32x4 v;
    __builtin_memcpy(&v, row + (c < k - 16 ? c : k - 16), 16);
    return v;
}
[[maybe_unused]] __device__ __forceinline__ i32x4 place16(i32x4 v, unsigned c, unsigned k)
{
    if (c + 16 <= k) return v;
    const unsigned by = c + 16 - k;                   // bytes that come from before c
    if (by >= 16) return i32x4{0, 0, 0, 0};
    unsigned long long lo = (unsigned)v[0] | (unsigned long long)(unsigned)v[1] << 32, hi = (unsigned)v[2] | (unsigned long long)(unsigned)v[3] << 32;
    if (by >= 8) { lo = hi; hi = 0; }
    const unsigned s = (by & 7) * 8;
    if (s) { lo = lo >> s | hi << (64 - s); hi >>= s; }
    return i32x4{(int)(unsigned)lo, (int)(unsigned)(lo >> 32), (int)(unsigned)hi, (int)(unsigned)(hi >> 32)};
}

// k < 16: a result a thread.
template <int DT>
__global__ __launch_bounds__(256) void k_mat_short(MatArgs g)
{
    for (size_t at = (size_t)blockIdx.x * 256 + threadIdx.x; at < (size_t)g.m * g.n; at += (size_t)gridDim.x * 256) {
        const size_t m = at / g.n, n = at % g.n;
        int sum = 0;
        for (unsigned k = 0; k < g.k; k++) sum += (int)g.x[m * g.x_stride + k] * (int)g.w[n * g.w_stride + k];
        const float b = g.bias ? mat_elem<DT>(g.bias, n) : 0.0f;
        mat_store<DT>(g.out, m * g.out_stride + n, (float)sum * g.x_scale[m * g.x_scale_step] * g.w_scale[n * g.w_scale_step] + b);
    }
}

// ------------------------------------------------------------------ tiles in the LDS, for operands of whole 16-byte pieces
//
// Four waves, two by two, compute a tile of 64 TM rows of x by 64 TN rows of w; a wave holds TM x TN blocks of 32 x 32 sums.
// A step takes 128 bytes of k, whole cache lines (two steps of 64 halve the rate of the loads).  The buffer loads write the
// LDS directly (no registers, no address arithmetic): 128 bytes of a row are eight lanes, and the piece a lane fetches is
// rotated by the row so that the lanes that read a fragment together find it in different banks.  The LDS holds S steps of w
// and S + 1 of x: step t + S of x is asked for at the start of step t, into the buffer of t - 1, and of w in its middle, once
// the last fragment of t has been read.  Fragments are read half a step ahead of the products that use them, so a step has
// one barrier and no product waits for the LDS; two blocks share a CU where 80 KB of LDS do for one.  G groups of four waves take the steps in turn and join their sums in the LDS,
// for products with fewer tiles than the GPU has CUs.
// What bounds it (2048 x 8192 x 4096 bf16 60-62 us, 8192 x 8192 x 4096 217-232 us: 2.2-2.3 and 2.4-2.5 POP/s, the library's product
// alone takes 68 and 245): the matrix units, busy 66 and 71 % of the cycles, at the clock that the power limit leaves (1.85 GHz; the
// same product of zeros takes three quarters of the time).  What the units wait for in the other cycles is not measured.
typedef __attribute__((address_space(3))) void lds_void;

template <int N> struct Int { static constexpr int value = N; };
template <int DT> struct Out;
template <> struct Out<0> { typedef float T; [[maybe_unused]] static constexpr int SIZE = 4; };
template <> struct Out<1> { typedef _Float16 T; [[maybe_unused]] static constexpr int SIZE = 2; };
template <> struct Out<2> { typedef __bf16 T; [[maybe_unused]] static constexpr int SIZE = 2; };

// Which tile a block works on.  Blocks go to the eight XCDs in turn; each XCD gets a run of neighbouring tiles (bands of
// `band` tile rows, column by column), so that the tiles its L2 serves at one time share rows of x and w.
[[maybe_unused]] __device__ __forceinline__ bool tile_of(unsigned tiles_m, unsigned tiles_n, unsigned band, unsigned* tm, unsigned* tn)
{
    const size_t block = flat_block();
    const unsigned total = tiles_m * tiles_n, b = (unsigned)block;
    if (block >= total) return false;                 // the rest of a grid's last row
    const unsigned xcd = b & 7, q = total >> 3, r = total & 7;
    const unsigned p = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (b >> 3);
    const unsigned per_band = band * tiles_n, first = p / per_band * band, in = p % per_band;
    const unsigned rows = tiles_m - first < band ? tiles_m - first : band;
    *tm = first + in % rows;
    *tn = in / rows;
    return true;
}

template <int DT, int TM, int TN, int S, int G, bool PAST>
__global__ __launch_bounds__(256 * G, G * ((S + 1) * TM + S * TN) * 8192 > 81920 ? G : 2 * G) void k_mat_tile(MatArgs g)
{
#ifdef __HIP_DEVICE_COMPILE__          // (register constraints and buffer loads the host pass does not know)
    constexpr int BM = 64 * TM, BN = 64 * TN, XS = BM * 128, WS = BN * 128, ESZ = Out<DT>::SIZE;
    constexpr int PITCH = 32 * TN * ESZ + 16;
    constexpr int STAGES = (S + 1) * XS + S * WS;      // one group's
    static_assert(4 * G * 32 * PITCH + 2 * BN * 4 <= G * STAGES && (G == 1 || G * TM * TN * 16384 <= G * STAGES), "the end uses the stages' LDS");
    __shared__ __attribute__((aligned(1024))) signed char smem[G * STAGES];
    const unsigned tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6 & 3), group = __builtin_amdgcn_readfirstlane(tid >> 8);
    unsigned tm, tn;
    if (!tile_of((g.m + BM - 1) / BM, (g.n + BN - 1) / BN, TM >= 4 ? 4 : 8, &tm, &tn)) return;
    const unsigned m0 = __builtin_amdgcn_readfirstlane(tm * BM), n0 = __builtin_amdgcn_readfirstlane(tn * BN);

    // the tile's rows of either operand, as a buffer of its own: the offsets of a tile fit 32 bits
    const unsigned mrows = g.m - m0 < BM ? g.m - m0 : BM, nrows = g.n - n0 < BN ? g.n - n0 : BN;
    const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc((void*)(g.x + (size_t)m0 * g.x_stride), 0,
                                                                        (int)((mrows - 1) * (unsigned)g.x_stride + g.k), 0x00020000);
    const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc((void*)(g.w + (size_t)n0 * g.w_stride), 0,
                                                                        (int)((nrows - 1) * (unsigned)g.w_stride + g.k), 0x00020000);
    // rows past the last one repeat it (their sums are not stored)
    // The LDS has 64 banks, two rows of 128 bytes: sixteen lanes of a fragment that are read together differ in bits 0 .. 3 of
    // their row of x, and in bits 0, 1, 2 and 4 of their row of w.  Bit 0 is the half of the banks, the others turn the row.
    const unsigned xpiece = (lane & 7) ^ (lane >> 4) ^ (wave & 1) << 2, wpiece = (lane & 7) ^ (lane >> 4) ^ (wave >> 1) << 2;
    unsigned xo[2 * TM], wo[2 * TN];
#pragma unroll
    for (int j = 0; j < 2 * TM; j++) { const unsigned r = (j * 4 + wave) * 8 + (lane >> 3); xo[j] = (r < mrows ? r : mrows - 1) * (unsigned)g.x_stride + xpiece * 16; }
#pragma unroll
    for (int j = 0; j < 2 * TN; j++) { const unsigned r = (j * 4 + wave) * 8 + (lane >> 3); wo[j] = (r < nrows ? r : nrows - 1) * (unsigned)g.w_stride + wpiece * 16; }
    const unsigned steps = ((g.k + 127) / 128 + G - 1) / G;   // of each group
    signed char* const stage = smem + group * STAGES;

    // ask for a step's rows of x or w; pieces beyond k (all of a step beyond the last) lie out of the buffer's range and
    // arrive as zeros (the scalar offset stays within it: the range check subtracts it)
    const auto fetch_x = [&](unsigned t, unsigned buf) {
        const unsigned at = (t * G + group) * 128, k0 = at < g.k ? at : 0;
        const bool past = at + xpiece * 16 >= g.k;
#pragma unroll
        for (int j = 0; j < 2 * TM; j++) __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_void*)(stage + buf * XS + (j * 4 + wave) * 1024), 16, past ? 0x80000000u : xo[j], k0, 0, 0);
    };
    const auto fetch_w = [&](unsigned t, unsigned buf) {
        const unsigned at = (t * G + group) * 128, k0 = at < g.k ? at : 0;
        const bool past = at + wpiece * 16 >= g.k;
#pragma unroll
        for (int j = 0; j < 2 * TN; j++) __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (lds_void*)(stage + (S + 1) * XS + buf * WS + (j * 4 + wave) * 1024), 16, past ? 0x80000000u : wo[j], k0, 0, 0);
    };

    const unsigned wm = (wave & 1) * 32 * TM, wn = (wave >> 1) * 32 * TN;
    // Where a lane's piece of a row lies, by half step and product.  Row i of a 32-row fragment of w is row
    // 16 (i / 4 % 2) + 4 (i / 8) + i % 4 of its block: the sums a lane then holds are sixteen neighbouring columns.
    unsigned fox[2][2], fow[2][2];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const unsigned c = h * 4 + q * 2 + (lane >> 5);
            fox[h][q] = (lane & 31) * 128 + ((c ^ (lane >> 1 & 7)) << 4);
            fow[h][q] = ((lane >> 2 & 1) * 16 + (lane >> 3 & 3) * 4 + (lane & 3)) * 128 + ((c ^ (lane >> 1 & 1) ^ (lane >> 3 & 1) << 1 ^ (lane >> 2 & 1) << 2) << 4);
        }
    i32x4 fx[2][2][TM], fw[2][2][TN];
    const auto read = [&](int h, unsigned xbuf, unsigned wbuf) {
#pragma unroll
        for (int q = 0; q < 2; q++) {
#pragma unroll
            for (int i = 0; i < TM; i++) fx[h][q][i] = *(const i32x4*)(stage + xbuf * XS + wm * 128 + i * 4096 + fox[h][q]);
#pragma unroll
            for (int j = 0; j < TN; j++) fw[h][q][j] = *(const i32x4*)(stage + (S + 1) * XS + wbuf * WS + wn * 128 + j * 4096 + fow[h][q]);
        }
    };
    // the fragments of a half step are in registers here, not read where they are used
    const auto hold = [&](int h) {
#pragma unroll
        for (int q = 0; q < 2; q++) {
#pragma unroll
            for (int i = 0; i < TM; i++) asm volatile("" : "+v"(fx[h][q][i]));
#pragma unroll
            for (int j = 0; j < TN; j++) asm volatile("" : "+v"(fw[h][q][j]));
        }
    };
    i32x16 acc[TM][TN] = {};
    const auto multiply = [&](int h) {
#pragma unroll
        for (int q = 0; q < 2; q++)
#pragma unroll
            for (int i = 0; i < TM; i++)
#pragma unroll
                for (int j = 0; j < TN; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[h][q][j], fx[h][q][i], acc[i][j], 0, 0, 0);
    };
    // all but the last `behind` loads of every wave have landed, every wave has its fragments in registers
    const auto meet = [&](auto behind) {
        constexpr int N = decltype(behind)::value;
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);      // vmcnt(N) lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };

#pragma unroll
    for (int t = 0; t < S; t++) { fetch_x(t, t); fetch_w(t, t); }
    float ws1 = 0.0f, b1 = 0.0f;                      // one column's scale and bias, for the end
    if (tid < BN) {
        const unsigned n = n0 + tid < g.n ? n0 + tid : g.n - 1;
        ws1 = g.w_scale[(size_t)n * g.w_scale_step];
        b1 = g.bias ? mat_elem<DT>(g.bias, n) : 0.0f;
    }
    meet(Int<(S - 1) * 2 * (TM + TN)>{});
    read(0, 0, 0);
    // Within a half step the loads go out first, in large tiles two products apart (the CU takes one in 18 cycles, and a
    // load that has to wait holds up the products behind it), then the reads of the next fragments.  2048 x 8192 x 8192:
    // this order 110 us, loads one product apart 114, reads before loads 121, both mixed evenly 124.
    constexpr int READS = 2 * (TM + TN), GAP = TM * TN >= 8 ? 2 : 1;
    unsigned x0 = 0, w0 = 0;                          // buffers of step t: t % (S + 1), t % S
    for (unsigned t = 0; t < steps; t++) {
        const unsigned x1 = x0 == S ? 0 : x0 + 1, w1 = w0 == S - 1 ? 0 : w0 + 1;
        hold(0);
        fetch_x(t + S, x0 == 0 ? S : x0 - 1);         // t - 1's buffer
        read(1, x0, w0);
        multiply(0);
#pragma unroll
        for (int i = 0; i < 2 * TM; i++) { __builtin_amdgcn_sched_group_barrier(0x010, 1, 0); __builtin_amdgcn_sched_group_barrier(0x008, GAP, 0); }
#pragma unroll
        for (int i = 0; i < READS / GAP; i++) { __builtin_amdgcn_sched_group_barrier(0x100, GAP, 0); __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); }
        // every fragment of t is in registers, t + 1 is in the LDS
        meet(Int<(S - 1) * 2 * TM + (S - 2) * 2 * TN>{});
        hold(1);
        fetch_w(t + S, w0);
        read(0, x1, w1);                              // (after the last step: zeros, not used)
        multiply(1);
#pragma unroll
        for (int i = 0; i < 2 * TN; i++) { __builtin_amdgcn_sched_group_barrier(0x010, 1, 0); __builtin_amdgcn_sched_group_barrier(0x008, GAP, 0); }
#pragma unroll
        for (int i = 0; i < READS / GAP; i++) { __builtin_amdgcn_sched_group_barrier(0x100, GAP, 0); __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); }
        x0 = x1; w0 = w1;
    }

    // Results leave by strips of 32 rows of x through the wave's own part of the LDS: a lane holds sixteen neighbouring
    // columns of a row in each block, the strip is stored in whole rows of the wave's columns.
    typedef typename Out<DT>::T T;
    constexpr int EPV = 16 / ESZ, VPR = 32 * TN * ESZ / 16;     // elements in 16 bytes, 16-byte vectors in a strip's row
    typedef T TV __attribute__((ext_vector_type(EPV)));
    float xs[TM];                                     // (asked for here: a load after a store to `out` would wait for it)
#pragma unroll
    for (int i = 0; i < TM; i++) {
        const unsigned m = m0 + wm + i * 32 + (lane & 31);
        xs[i] = g.x_scale[(size_t)(m < g.m ? m : g.m - 1) * g.x_scale_step];
    }
    meet(Int<0>{});                                   // the last loads (zeros) have landed
    // the groups' sums are joined: each strip of 32 rows of x by one group
    const auto owner = [](int i) { return TM % G == 0 ? i % G : 0; };
    if constexpr (G > 1) {
        i32x4* const sums = (i32x4*)smem + (wave * 64 + lane);
#pragma unroll
        for (int i = 0; i < TM; i++) {
            if ((int)group == owner(i)) continue;
#pragma unroll
            for (int j = 0; j < TN; j++)
#pragma unroll
                for (int r = 0; r < 4; r++) sums[((group * TM + i) * TN + j) * 1024 + r * 256] = i32x4{acc[i][j][r * 4], acc[i][j][r * 4 + 1], acc[i][j][r * 4 + 2], acc[i][j][r * 4 + 3]};
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TM; i++) {
            if ((int)group != owner(i)) continue;
#pragma unroll
            for (int o = 1; o < G; o++)
#pragma unroll
                for (int j = 0; j < TN; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const i32x4 v = sums[(((group + o) % G * TM + i) * TN + j) * 1024 + r * 256];
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[i][j][r * 4 + e] += v[e];
                    }
        }
        __syncthreads();
    }
    float *const s_scale = (float*)smem, *const s_bias = s_scale + BN;
    if (tid < BN) { s_scale[tid] = ws1; s_bias[tid] = b1; }
    __syncthreads();
    f32x4 ws[TN][4], bs[TN][4];
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const unsigned c = wn + j * 32 + (lane >> 5) * 16 + r * 4;
            ws[j][r] = *(const f32x4*)(s_scale + c);
            bs[j][r] = *(const f32x4*)(s_bias + c);
        }
    signed char* const strip = smem + 2 * BN * 4 + (group * 4 + wave) * 32 * PITCH;
    const unsigned nw = n0 + wn, cols = nw >= g.n ? 0 : g.n - nw < 32 * TN ? g.n - nw : 32 * TN;
    const bool aligned = (((uintptr_t)g.out | (g.out_stride * ESZ)) & 15) == 0, whole = aligned && cols == 32 * TN && g.out_stride < (1u << 25);   // (32 rows: 32-bit offsets)
#pragma unroll
    for (int i = 0; i < TM; i++) {
        if (G > 1 && (int)group != owner(i)) continue;
        const unsigned ms = m0 + wm + i * 32;
#pragma unroll
        for (int j = 0; j < TN; j++)
#pragma unroll
            for (int v = 0; v < 16 / EPV; v++) {
                TV o;
#pragma unroll
                for (int e = 0; e < EPV; e++) {
                    const int r = v * EPV + e;
                    o[e] = (T)((float)acc[i][j][r] * xs[i] * ws[j][r >> 2][r & 3] + bs[j][r >> 2][r & 3]);
                }
                *(TV*)(strip + (lane & 31) * PITCH + (j * 32 + (lane >> 5) * 16 + v * EPV) * ESZ) = o;
            }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        T* const o = (T*)g.out + (size_t)ms * g.out_stride + nw;
        if (whole && ms + 32 <= g.m) {
            // written through the L2 (agent scope): lines that are still dirty when the kernel ends stand between it and the next
            const __amdgpu_buffer_rsrc_t to = __builtin_amdgcn_make_buffer_rsrc(o, 0, 0xffffffff, 0x00020000);
#pragma unroll
            for (int u = 0; u < VPR / 2; u++) {
                const unsigned v = u * 64 + lane, row = v / VPR, col = v % VPR * EPV;
                const u32x4 d = *(const u32x4*)(strip + row * PITCH + col * ESZ);
                if (PAST) __builtin_nontemporal_store(d, (u32x4*)(o + row * g.out_stride + col));
                else __builtin_amdgcn_raw_buffer_store_b128(d, to, (unsigned)((row * g.out_stride + col) * ESZ), 0, 16);
            }
        } else if (aligned) {                         // the last tiles: whole vectors up to the edge
#pragma unroll 2
            for (int u = 0; u < VPR / 2; u++) {
                const unsigned v = u * 64 + lane, row = v / VPR, col = v % VPR * EPV;
                if (ms + row >= g.m) continue;
                if (col + EPV <= cols) *(u32x4*)(o + row * g.out_stride + col) = *(const u32x4*)(strip + row * PITCH + col * ESZ);
                else for (unsigned e = col; e < cols; e++) o[row * g.out_stride + e] = *(const T*)(strip + row * PITCH + e * ESZ);
            }
        } else {                                      // rows that do not start on 16 bytes: an element a lane
#pragma unroll 8
            for (unsigned v = lane; v < 32 * 32 * TN; v += 64) {
                const unsigned row = v / (32 * TN), col = v % (32 * TN);
                if (ms + row < g.m && col < cols) o[row * g.out_stride + col] = *(const T*)(strip + row * PITCH + col * ESZ);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
#endif
}

template <int DT, int TM, int TN, int S, int G, bool PAST = false> void launch_tile(const MatArgs& g, hipStream_t st)
{
    const size_t tiles = (size_t)((g.m + 64 * TM - 1) / (64 * TM)) * ((g.n + 64 * TN - 1) / (64 * TN));
    k_mat_tile<DT, TM, TN, S, G, PAST><<<flat_grid(tiles), 256 * G, 0, st>>>(g);
}

// ------------------------------------------------------------------ few rows of x: the weights' bytes are the work
//
// A block computes 16 NB columns for 16 MB rows of x; its W waves share out k in pieces of 128 bytes and their sums are
// joined through the LDS (exact, so in any order).  Until then no wave waits for another: each has a ring of U pieces of
// its own in the LDS, which the buffer loads fill in whole cache lines (fragments loaded straight into registers are 64
// bytes of 16 rows a load, at half the rate: 7.1 against 5.5 us at 16 x 4096 x 4096).  Blocks begin k at different pieces: rows
// are often a power of two apart, and with all blocks at one column the loads meet in a few of the caches' and the memory's
// channels (16 x 8192 x 4096 8.2 -> 7.1 us, 64 x 4096 x 8192 12.5 -> 8.7, 4 x 8192 x 8192 17.6 -> 11.7; one or three pieces from
// block to block do alike, eight 8.6, 10.8 and 14.7; the tiles above, whose blocks share rows, gain nothing).
// What bounds it: the weight's bytes and a launch, 16.8 MB in 4.5 us out of the Infinity Cache, 5.5 us out of memory; 67 MB in
// 12.5 us out of memory, 6.7 TB/s beyond the launch.
template <int DT, int MB, int NB, int W, int U, bool ANY, bool ONCE>
__global__ __launch_bounds__(64 * W) void k_mat_rows(MatArgs g)
{
#ifdef __HIP_DEVICE_COMPILE__
    constexpr int ESZ = Out<DT>::SIZE, SLOT = (NB + MB) * 2048, RING = U * SLOT, LOADS = 2 * (NB + MB);
    static_assert(RING >= MB * NB * 1024, "a wave's sums go where its ring was");
    __shared__ __attribute__((aligned(1024))) signed char smem[W * RING];
    const unsigned tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned n0 = blockIdx.x * 16 * NB, m0 = blockIdx.y * 16 * MB;
    const unsigned nrows = g.n - n0 < 16 * NB ? g.n - n0 : 16 * NB, mrows = g.m - m0 < 16 * MB ? g.m - m0 : 16 * MB;
    const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc((void*)(g.w + (size_t)n0 * g.w_stride), 0,
                                                                        (int)((nrows - 1) * (unsigned)g.w_stride + g.k), 0x00020000);
    const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc((void*)(g.x + (size_t)m0 * g.x_stride), 0,
                                                                        (int)((mrows - 1) * (unsigned)g.x_stride + g.k), 0x00020000);
    // rows past the last one repeat it (their sums are not stored)
    const unsigned at = ((lane & 7) ^ (lane >> 3)) * 16;
    unsigned wr_row[2 * NB], xr_row[2 * MB], wo[2 * NB], xo[2 * MB];
#pragma unroll
    for (int j = 0; j < 2 * NB; j++) { const unsigned r = j * 8 + (lane >> 3); wr_row[j] = r < nrows ? r : nrows - 1; wo[j] = wr_row[j] * (unsigned)g.w_stride + at; }
#pragma unroll
    for (int i = 0; i < 2 * MB; i++) { const unsigned r = i * 8 + (lane >> 3); xr_row[i] = r < mrows ? r : mrows - 1; xo[i] = xr_row[i] * (unsigned)g.x_stride + at; }
    const unsigned pieces = (g.k + 127) / 128, start = blockIdx.x * 3 % pieces;
    const auto turned = [&](unsigned piece) { const unsigned p = piece + start; return p < pieces ? p : p - pieces; };
    signed char* const ring = smem + wave * RING;
    const auto fetch = [&](unsigned piece, int u) {
        const unsigned k0 = piece < pieces ? turned(piece) * 128 : 0;  // (within the buffer: the range check subtracts it)
        const bool past = piece >= pieces || k0 + at >= g.k;           // out of the buffer's range: zeros
#pragma unroll
        for (int j = 0; j < 2 * NB; j++) __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (lds_void*)(ring + u * SLOT + j * 1024), 16, past ? 0x80000000u : wo[j], k0, 0, ONCE ? 2 : 0);
#pragma unroll
        for (int i = 0; i < 2 * MB; i++) __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_void*)(ring + u * SLOT + (2 * NB + i) * 1024), 16, past ? 0x80000000u : xo[i], k0, 0, 0);
    };
    unsigned fo[2];
#pragma unroll
    for (int h = 0; h < 2; h++) fo[h] = (lane & 15) * 128 + (((h * 4 + (lane >> 4)) ^ (lane & 7)) << 4);
    i32x4 acc[MB][NB] = {};
    const auto multiply = [&](int u) {
        i32x4 fw[2][NB], fx[2][MB];
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int j = 0; j < NB; j++) fw[h][j] = *(const i32x4*)(ring + u * SLOT + j * 2048 + fo[h]);
#pragma unroll
            for (int i = 0; i < MB; i++) fx[h][i] = *(const i32x4*)(ring + u * SLOT + (NB + i) * 2048 + fo[h]);
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xc07f);                                      // lgkmcnt(0): the slot has been read
        asm volatile("" ::: "memory");
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int j = 0; j < NB; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[h][j], fx[h][i], acc[i][j], 0, 0, 0);
    };
    if constexpr (ANY) {
        // rows that start anywhere: the same pieces through registers, the next one on its way during the products
        i32x4 next[LOADS];
        const auto load = [&](unsigned piece) {
#pragma unroll
            for (int j = 0; j < 2 * NB; j++) next[j] = ask16(g.w + (size_t)(n0 + wr_row[j]) * g.w_stride, turned(piece) * 128 + at, g.k);
#pragma unroll
            for (int i = 0; i < 2 * MB; i++) next[2 * NB + i] = ask16(g.x + (size_t)(m0 + xr_row[i]) * g.x_stride, turned(piece) * 128 + at, g.k);
        };
        load(wave);
        for (unsigned p = wave; p < pieces; p += W) {
            if ((turned(p) + 1) * 128 > g.k) {
#pragma unroll
                for (int l = 0; l < LOADS; l++) next[l] = place16(next[l], turned(p) * 128 + at, g.k);
            }
#pragma unroll
            for (int l = 0; l < LOADS; l++) *(i32x4*)(ring + l * 1024 + lane * 16) = next[l];
            if (p + W < pieces) load(p + W);
            multiply(0);
        }
    } else {
#pragma unroll
        for (int u = 0; u < U; u++) fetch(wave + u * W, u);
        for (unsigned p = wave; p < pieces; p += U * W) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                constexpr int N = (U - 1) * LOADS;
                asm volatile("" ::: "memory");
                __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14);  // vmcnt(N): this slot's loads have landed
                asm volatile("" ::: "memory");
                multiply(u);
                fetch(p + (u + U) * W, u);
            }
        }
    }
    // a lane holds columns 4 (lane / 16) .. + 3 of row lane % 16
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);               // the last loads (zeros) have landed: the ring is free
    asm volatile("" ::: "memory");
    i32x4* const part = (i32x4*)smem;
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int j = 0; j < NB; j++) part[wave * (RING / 16) + (i * NB + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    typedef typename Out<DT>::T T;
    for (unsigned v = tid; v < 64 * MB * NB; v += 64 * W) {
        const unsigned m = m0 + v / (64 * NB) * 16 + (v & 15), n = n0 + v / 64 % NB * 16 + (v >> 4 & 3) * 4;
        if (m >= g.m) continue;
        i32x4 sum = part[v];
#pragma unroll
        for (int w = 1; w < W; w++) sum += part[w * (RING / 16) + v];
        const float xs = g.x_scale[(size_t)m * g.x_scale_step];
        T* const o = (T*)g.out + (size_t)m * g.out_stride + n;
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 r;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const unsigned c = n + e < g.n ? n + e : g.n - 1;
            r[e] = (T)((float)sum[e] * xs * g.w_scale[(size_t)c * g.w_scale_step] + (g.bias ? mat_elem<DT>(g.bias, c) : 0.0f));
        }
        if (n + 4 <= g.n && ((uintptr_t)o & (4 * ESZ - 1)) == 0) *(T4*)o = r;
        else for (int e = 0; e < 4; e++) if (n + e < g.n) o[e] = r[e];
    }
#endif
}

template <int DT, int MB, int NB, int W, int U, bool ANY = false> void launch_rows(const MatArgs& g, hipStream_t st)
{
    const dim3 grid((g.n + 16 * NB - 1) / (16 * NB), (g.m + 16 * MB - 1) / (16 * MB));
    if constexpr (!ANY) {
        // A weight that one row of blocks reads, and that the L2s (32 MB) cannot keep for the next call, is loaded past them.  Out
        // of memory and out of the Infinity Cache: 33.5 MB (16 x 8192 x 4096) 8.1 -> 7.5 and 7.0 -> 6.9 us; 59 MB 12.7 -> 11.6 and
        // 10.6 -> 10.9; 67 MB 14.3 -> 12.5 and 11.7 -> 12.0; but 16.8 MB 5.5 -> 5.2 and, out of the L2s, 3.7 -> 4.5; with two rows
        // of blocks (64 x 4096 x 8192) 12.7 -> 12.4 and 8.7 -> 11.8.
        if (grid.y == 1 && (size_t)g.n * g.k >= ((size_t)32 << 20)) {
            k_mat_rows<DT, MB, NB, W, U, ANY, true><<<grid, 64 * W, 0, st>>>(g);
            return;
        }
    }
    k_mat_rows<DT, MB, NB, W, U, ANY, false><<<grid, 64 * W, 0, st>>>(g);
}

// ------------------------------------------------------------------ tiles of operands of any alignment
//
// 128 x 128 tile, four waves two by two, 128 bytes of k a step, laid out in the LDS as above.  Rows start anywhere, so the
// pieces go through registers: two steps are on their way there while one is multiplied.
template <int DT>
__global__ __launch_bounds__(256, 2) void k_mat_any(MatArgs g)
{
#ifdef __HIP_DEVICE_COMPILE__
    __shared__ __attribute__((aligned(1024))) signed char sx[2][128 * 128], sw[2][128 * 128];
    const unsigned tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    unsigned tm, tn;
    if (!tile_of((g.m + 127) / 128, (g.n + 127) / 128, 8, &tm, &tn)) return;
    const unsigned m0 = tm * 128, n0 = tn * 128, at = ((lane & 7) ^ (lane >> 4) ^ (wave & 1) << 2) * 16;
    const signed char *xr[4], *wr[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {                     // rows past the last one repeat it (their sums are not stored)
        const unsigned r = (i * 4 + wave) * 8 + (lane >> 3), m = m0 + r, n = n0 + r;
        xr[i] = g.x + (size_t)(m < g.m ? m : g.m - 1) * g.x_stride;
        wr[i] = g.w + (size_t)(n < g.n ? n : g.n - 1) * g.w_stride;
    }
    const unsigned wm = (wave & 1) * 64, wn = (wave >> 1) * 64, steps = (g.k + 127) / 128;
    i32x4 px[2][4], pw[2][4];
    const auto load = [&](int s, unsigned t) {
#pragma unroll
        for (int i = 0; i < 4; i++) { px[s][i] = ask16(xr[i], t * 128 + at, g.k); pw[s][i] = ask16(wr[i], t * 128 + at, g.k); }
    };
    const auto put = [&](int s, unsigned t) {         // step t into buffer t & 1 = s
        if ((t + 1) * 128 > g.k) {
#pragma unroll
            for (int i = 0; i < 4; i++) { px[s][i] = place16(px[s][i], t * 128 + at, g.k); pw[s][i] = place16(pw[s][i], t * 128 + at, g.k); }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            *(i32x4*)(sx[s] + (i * 4 + wave) * 1024 + lane * 16) = px[s][i];
            *(i32x4*)(sw[s] + (i * 4 + wave) * 1024 + lane * 16) = pw[s][i];
        }
    };
    i32x16 acc[2][2] = {};
    const auto multiply = [&](int b) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const unsigned fo = (lane & 31) * 128 + (((q * 2 + (lane >> 5)) ^ (lane >> 1 & 7)) << 4);
            i32x4 fx[2], fw[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                fx[i] = *(const i32x4*)(sx[b] + (wm + i * 32) * 128 + fo);
                fw[i] = *(const i32x4*)(sw[b] + (wn + i * 32) * 128 + fo);
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fx[i], fw[j], acc[i][j], 0, 0, 0);
        }
    };
    load(0, 0);
    load(1, 1);
    put(0, 0);
    load(0, 2);
    __syncthreads();
    for (unsigned t = 0; t < steps; t += 2) {         // (an odd last step: zeros)
        put(1, t + 1);
        load(1, t + 3);
        multiply(0);
        __syncthreads();
        put(0, t + 2);
        load(0, t + 4);
        multiply(1);
        __syncthreads();
    }
    // (scales and bias first: a load after a store to `out` would wait for it)
    float xs[2][16], ws[2], bias[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const unsigned n = n0 + wn + j * 32 + (lane & 31), c = n < g.n ? n : g.n - 1;
        ws[j] = g.w_scale[(size_t)c * g.w_scale_step];
        bias[j] = g.bias ? mat_elem<DT>(g.bias, c) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const unsigned m = m0 + wm + i * 32 + (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3);
            xs[i][r] = g.x_scale[(size_t)(m < g.m ? m : g.m - 1) * g.x_scale_step];
        }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int r = 0; r < 16; r++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const unsigned n = n0 + wn + j * 32 + (lane & 31), m = m0 + wm + i * 32 + (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3);
                if (m < g.m && n < g.n) mat_store<DT>(g.out, (size_t)m * g.out_stride + n, (float)acc[i][j][r] * xs[i][r] * ws[j] + bias[j]);
            }
#endif
}

template <int DT> void launch_any(const MatArgs& g, hipStream_t st)
{
    const size_t tiles = (size_t)((g.m + 127) / 128) * ((g.n + 127) / 128);
    k_mat_any<DT><<<flat_grid(tiles), 256, 0, st>>>(g);
}

template <int DT> void launch_mat(const MatArgs& g, hipStream_t st)
{
    // whole 16-byte pieces, and tiles whose offsets fit 31 bits
    const bool pieces = (((uintptr_t)g.x | (uintptr_t)g.w | g.x_stride | g.w_stride | g.k) & 15) == 0 &&
                        g.x_stride <= (1u << 22) && g.w_stride <= (1u << 22);
    if (g.k < 16) {
        const size_t blocks = ((size_t)g.m * g.n + 255) / 256;
        k_mat_short<DT><<<dim3((unsigned)(blocks < 65536 ? blocks : 65536)), 256, 0, st>>>(g);
        return;
    }
    if (!pieces) {
        switch (pick_tile(kAnyTiles, g.m, g.n, g.k)) {
            case 0: return launch_rows<DT, 1, 1, 8, 1, true>(g, st);
            case 1: return launch_rows<DT, 1, 2, 8, 1, true>(g, st);
            case 2: return launch_rows<DT, 2, 2, 8, 1, true>(g, st);
            case 3: return launch_rows<DT, 4, 4, 4, 1, true>(g, st);
            default: return launch_any<DT>(g, st);
        }
    }
    switch (pick_tile(kTiles, g.m, g.n, g.k)) {
        case 0: return launch_rows<DT, 1, 1, 8, 2>(g, st);
        case 1: return launch_rows<DT, 1, 2, 4, 2>(g, st);
        case 2: return launch_rows<DT, 1, 4, 4, 2>(g, st);
        case 3: return launch_rows<DT, 2, 2, 4, 2>(g, st);
        case 4: return launch_rows<DT, 4, 2, 4, 2>(g, st);
        case 5: return launch_tile<DT, 1, 1, 3, 2>(g, st);
        case 6: return launch_tile<DT, 2, 1, 2, 2>(g, st);
        case 7: return launch_tile<DT, 2, 2, 3, 1>(g, st);
        case 8: return launch_tile<DT, 2, 2, 2, 1>(g, st);
        case 9: return launch_tile<DT, 2, 4, 3, 1>(g, st);
        default: break;
    }
    // A result of this tile that the caches do not hold until it is read is stored past them, others are written through the L2, as
    // the other tiles' results are at any size (few as large as this take one of those; not measured there).  Ordinary
    // stores, through, past, alone and with a copy of the result behind the product, in us: 17 MB (2048 x 4096 bf16, k = 4096) 36.8,
    // 36.1, 36.6 and 42.8, 42.1, 44.1; 34 MB (2048 x 8192) 60.8, 59.1, 59.6 and 70.6, 68.7, 72.7; 134 MB (8192 x 8192) 233, 232, 227
    // and 287, 285, 282.
    if ((size_t)g.m * g.n * Out<DT>::SIZE >= ((size_t)64 << 20)) return launch_tile<DT, 4, 4, 2, 1, true>(g, st);
    launch_tile<DT, 4, 4, 2, 1>(g, st);
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
inline size_t extent(size_t rows, size_t stride, size_t cols) { return !rows || !cols ? 0 : rows > 1 ? (rows - 1) * stride + cols : cols; }
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
    const int64_t far = (int64_t)1 << 30;              // with 2^31 rows: no extent overflows
    if ((c->m > 1 && (c->out_stride > far || c->x_stride > far)) || (c->n > 1 && c->w_stride > far)) MAT_FAIL("row strides beyond 2^30");
    if (((uintptr_t)c->out % esz) || ((uintptr_t)c->bias % esz) || ((uintptr_t)c->x_scale % 4) || ((uintptr_t)c->w_scale % 4)) MAT_FAIL("out, bias and scales must be aligned to their elements");
    const size_t tiles = ((size_t)c->m + 63) / 64 * (((size_t)c->n + 63) / 64);
    if (tiles > 0x7fffffffu) MAT_FAIL("%lld x %lld results are too many for one launch", (long long)c->m, (long long)c->n);
    const size_t out_bytes = extent(c->m, c->out_stride, c->n) * esz;
    if (meet(c->out, out_bytes, c->x, extent(c->m, c->x_stride, c->k)) || meet(c->out, out_bytes, c->w, extent(c->n, c->w_stride, c->k)) ||
        meet(c->out, out_bytes, c->x_scale, 4 * (size_t)c->x_scales) || meet(c->out, out_bytes, c->w_scale, 4 * (size_t)c->w_scales) ||
        meet(c->out, out_bytes, c->bias, (size_t)c->n * esz)) MAT_FAIL("out overlaps an operand");
    MatArgs g{};
    g.out = c->out; g.x = c->x; g.x_scale = c->x_scale; g.w = c->w; g.w_scale = c->w_scale; g.bias = c->bias;
    // (a single row has no stride, whatever was given)
    g.out_stride = c->m > 1 ? (size_t)c->out_stride : 0; g.x_stride = c->m > 1 ? (size_t)c->x_stride : 0; g.w_stride = c->n > 1 ? (size_t)c->w_stride : 0;
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
