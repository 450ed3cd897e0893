// Query and key heads turned by their positions (rotary positions), in place or into outputs of their own.
//
//   angle = position * freqs[i],  c = scale cos(angle),  s = scale sin(angle)   (s = -s for the inverse)
//   (y1, y2) = (x1 c - x2 s, x2 c + x1 s)   for the pairs (i, i + rot/2) or, interleaved, (2i, 2i + 1)
//
// of the first `rot` elements of a head; the rest is copied.  The inverse is the transpose of the rotation, so it is
// the backward pass of a forward call with the same `scale`.  The angle is formed and reduced to a fraction of a turn
// in fp64 (positions of a million lose 16 of fp32's 24 bits to whole turns); everything after it is fp32, the result
// is rounded once to the storage type.  The steps are written out (`turned`, `fp32_value`), so that an element's bits do not
// depend on which variant of the kernel computes it: in place or not, alone or among many tokens.
// No counterpart in the reference: it is what lies between the product that follows its all-reduce and the attention.
#include <hip/hip_runtime.h>
#include <stdio.h>

#include <type_traits>
#include <utility>

#include "../../include/tbvcoll.h"
#include "tbv_device.h"
#include "tbv_step.h"

namespace tbv {

namespace {

struct RotHeads {
    void* out; const void* in;
    unsigned heads;
    ptrdiff_t in_batch, in_token, in_head, out_batch, out_token, out_head;
};
struct RotArgs {
    RotHeads h[2];                              // query, key
    const void* positions; const double* freqs;
    ptrdiff_t pos_batch, pos_token;
    unsigned tokens, head, half, pos64;
    float scale;
    int inverse;
    char* base;                                 // of the results
    bool through;                               // write them through the L2
};

// A pair turned: one rounded product, then one fused multiply-add.
__device__ __forceinline__ float2 turned(float x1, float x2, float2 w)
{
    return make_float2(__builtin_fmaf(x1, w.x, -(x2 * w.y)), __builtin_fmaf(x2, w.x, x1 * w.y));
}

// The value in fp32, whatever it becomes next.  Left to itself the compiler merges some of the multiply-adds with the rounding to
// fp16 that follows (one rounding in place of two, so some results differ), others not, from variant to variant.
__device__ __forceinline__ float fp32_value(float v)
{
#ifdef __HIP_DEVICE_COMPILE__          // (a register constraint the host pass does not know)
    asm("" : "+v"(v));
#endif
    return v;
}

template <int DT> __device__ __forceinline__ float rot_load(const void* p, ptrdiff_t i)
{
    if (DT == 0) return ((const float*)p)[i];
    if (DT == 1) return (float)((const _Float16*)p)[i];
    return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
}
template <int DT> __device__ __forceinline__ void rot_store(void* p, ptrdiff_t i, float v)
{
    if (DT == 0) ((float*)p)[i] = v;
    else if (DT == 1) ((_Float16*)p)[i] = (_Float16)fp32_value(v);
    else ((__bf16*)p)[i] = (__bf16)v;
}
template <int DT> __device__ __forceinline__ void rot_copy(void* o, ptrdiff_t j, const void* p, ptrdiff_t i)
{
    if (DT == 0) ((uint32_t*)o)[j] = ((const uint32_t*)p)[i];
    else ((uint16_t*)o)[j] = ((const uint16_t*)p)[i];
}

__device__ __forceinline__ void turn(const RotArgs& g, unsigned batch, unsigned token, unsigned i, float* c, float* s)
{
    const ptrdiff_t at = (ptrdiff_t)batch * g.pos_batch + (ptrdiff_t)token * g.pos_token;
    const double p = g.pos64 ? (double)((const long long*)g.positions)[at] : (double)((const int*)g.positions)[at];
    const double turns = p * g.freqs[i] * 0.15915494309189533577;       // 1 / (2 pi)
    const float part = (float)(turns - __builtin_rint(turns));          // -1/2 .. 1/2 of a turn
    float sn, cs;
    sincospif(2.0f * part, &sn, &cs);
    *c = cs * g.scale;
    *s = (g.inverse ? -sn : sn) * g.scale;
}

constexpr unsigned kRotPairs = TBV_ROTARY_MAX_ROT / 2;   // cosines and sines of a block: 32 KiB of LDS

// The cosines and sines of a block's z tokens, one pair a thread.
__device__ __forceinline__ void turn_table(const RotArgs& g, unsigned total, float2* table)
{
    const unsigned tid = (threadIdx.z * blockDim.y + threadIdx.y) * blockDim.x + threadIdx.x, threads = blockDim.x * blockDim.y * blockDim.z;
    for (unsigned e = tid; e < g.half * blockDim.z; e += threads) {
        const unsigned z = e / g.half;
        const size_t r = flat_block() * blockDim.z + z;
        float c, s;
        if (r < total) { turn(g, (unsigned)r / g.tokens, (unsigned)r % g.tokens, e - z * g.half, &c, &s); table[e] = make_float2(c, s); }
    }
    __syncthreads();
}

// A block turns `z` tokens: its threads first form the tokens' cosines and sines in the LDS, one pair a thread (in fp64
// and by sincospi they are several times the work of turning a head), then take 16 bytes of a head at a time: x
// runs over a head's vectors, y over the heads of q and k, z over the tokens, so no index is divided.  The first vectors are
// asked for before the angles are formed, which hides the way from memory.  Heads may start at any element: loads and
// stores of 16 bytes need no alignment here; what is left of a head after whole vectors goes by elements.
// U heads to a thread, to have more on its way at once.
template <int DT> struct Lanes {                      // 16 bytes as fp32 and back, rounded to nearest even
    static constexpr int N = 8;
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
    static __device__ __forceinline__ u32x4 pack(const float* f)
    {
        typedef typename std::conditional<DT == 1, _Float16, __bf16>::type T;
        typedef T T8 __attribute__((ext_vector_type(8)));
        T8 o;
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = (T)(DT == 1 ? fp32_value(f[i]) : f[i]);
        return __builtin_bit_cast(u32x4, o);
    }
};
template <> struct Lanes<0> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(u32x4 v, float* f)
    {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = __uint_as_float(v[i]);
    }
    static __device__ __forceinline__ u32x4 pack(const float* f)
    {
        return u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    }
};

__device__ __forceinline__ u32x4 load16(const char* p) { u32x4 v; __builtin_memcpy(&v, p, 16); return v; }
// Results are stored in the ordinary way, or written through the L2 (agent scope; addresses are 32-bit offsets from `base` and
// multiples of 16).
template <bool THROUGH> __device__ __forceinline__ void store16([[maybe_unused]] char* base, char* p, u32x4 v)
{
#ifdef __HIP_DEVICE_COMPILE__
    if constexpr (THROUGH) {
        const __amdgpu_buffer_rsrc_t to = __builtin_amdgcn_make_buffer_rsrc(base, 0, 0xffffffff, 0x00020000);
        __builtin_amdgcn_raw_buffer_store_b128(v, to, (uint32_t)(p - base), 0, 16);
        return;
    }
#endif
    __builtin_memcpy(p, &v, 16);
}

template <int DT, bool INTER, int U, bool THROUGH>
__global__ __launch_bounds__(512) void k_rotary(RotArgs g, unsigned total)
{
    constexpr unsigned N = Lanes<DT>::N, P = INTER ? N / 2 : N;          // elements and pairs of a unit
    constexpr ptrdiff_t ESZ = 16 / N;
    extern __shared__ float2 turns[];                 // [z][half]
    const size_t row = flat_block() * blockDim.z + threadIdx.z;           // batch and token
    const unsigned token = (unsigned)row % g.tokens, batch = (unsigned)row / g.tokens;
    // what a head is made of: whole units of pairs, single pairs, whole vectors to copy, single elements to copy
    const unsigned full = g.half / P, rest = g.head - 2 * g.half, pairs = full + g.half % P, vecs = pairs + rest / N, slots = vecs + rest % N;
    const unsigned heads = g.h[0].heads + g.h[1].heads, apart = g.half * ESZ;   // bytes between the halves
    const char* in[U];
    char* out[U];
    u32x4 a[U], b[U];
    const auto place = [&](unsigned first) {          // where this thread's heads first, first + y, ... start
#pragma unroll
        for (int u = 0; u < U; u++) {
            const unsigned n = first + u * blockDim.y < heads ? first + u * blockDim.y : first;
            const bool key = n >= g.h[0].heads;
            const RotHeads& h = g.h[key];
            const ptrdiff_t head = key ? n - g.h[0].heads : n;
            in[u] = (const char*)h.in + ((ptrdiff_t)batch * h.in_batch + (ptrdiff_t)token * h.in_token + head * h.in_head) * ESZ;
            out[u] = (char*)h.out + ((ptrdiff_t)batch * h.out_batch + (ptrdiff_t)token * h.out_token + head * h.out_head) * ESZ;
        }
    };
    const auto load = [&](unsigned i) {
        const unsigned at = i < full ? i * 16 : (2 * g.half + (i - pairs) * N) * ESZ;
#pragma unroll
        for (int u = 0; u < U; u++) {
            a[u] = load16(in[u] + at);
            if (!INTER && i < full) b[u] = load16(in[u] + at + apart);
        }
    };
    const auto vector = [&](unsigned i) { return i < full || (i >= pairs && i < vecs); };
    const bool mine = row < total && threadIdx.y < heads && threadIdx.x < slots;
    if (mine) { place(threadIdx.y); if (vector(threadIdx.x)) load(threadIdx.x); }
    turn_table(g, total, turns);
    if (row >= total) return;
    const float2* const t = turns + threadIdx.z * g.half;
    for (unsigned first = threadIdx.y; first < heads; first += U * blockDim.y) {
        if (first != threadIdx.y || !mine) place(first);
        int live = 1;                                 // heads of this thread
#pragma unroll
        for (int u = 1; u < U; u++) live += first + u * blockDim.y < heads;
        for (unsigned i = threadIdx.x; i < slots; i += blockDim.x) {
            if (vector(i) && (first != threadIdx.y || i != threadIdx.x)) load(i);
            if (i < full) {
                float2 w[P];
#pragma unroll
                for (unsigned e = 0; e < P; e++) w[e] = t[i * P + e];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (u >= live) break;
                    float x[N], y[N], p[N], q[N];
                    Lanes<DT>::unpack(a[u], x);
                    if (INTER) {
#pragma unroll
                        for (unsigned e = 0; e < P; e++) {
                            const float2 v = turned(x[2 * e], x[2 * e + 1], w[e]);
                            p[2 * e] = v.x; p[2 * e + 1] = v.y;
                        }
                        store16<THROUGH>(g.base, out[u] + i * 16, Lanes<DT>::pack(p));
                    } else {
                        Lanes<DT>::unpack(b[u], y);
#pragma unroll
                        for (unsigned e = 0; e < P; e++) {
                            const float2 v = turned(x[e], y[e], w[e]);
                            p[e] = v.x; q[e] = v.y;
                        }
                        store16<THROUGH>(g.base, out[u] + i * 16, Lanes<DT>::pack(p));
                        store16<THROUGH>(g.base, out[u] + i * 16 + apart, Lanes<DT>::pack(q));
                    }
                }
            } else if (i < pairs) {
                const unsigned e = full * P + i - full, j1 = INTER ? 2 * e : e, j2 = INTER ? 2 * e + 1 : e + g.half;
                const float2 w = t[e];
                float x1[U], x2[U];
#pragma unroll
                for (int u = 0; u < U; u++) { x1[u] = rot_load<DT>(in[u], j1); x2[u] = rot_load<DT>(in[u], j2); }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (u >= live) break;
                    const float2 v = turned(x1[u], x2[u], w);
                    rot_store<DT>(out[u], j1, v.x);
                    rot_store<DT>(out[u], j2, v.y);
                }
            } else {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (u >= live || out[u] == in[u]) continue;
                    if (i < vecs) store16<THROUGH>(g.base, out[u] + (2 * g.half + (i - pairs) * N) * ESZ, a[u]);
                    else { const unsigned e = 2 * g.half + (rest / N) * N + i - vecs; rot_copy<DT>(out[u], e, in[u], e); }
                }
            }
        }
    }
}

template <int DT> void launch_rot(const RotArgs& g, bool inter, unsigned total, hipStream_t st)
{
    constexpr unsigned N = Lanes<DT>::N;
    const unsigned heads = g.h[0].heads + g.h[1].heads, pairs = inter ? N / 2 : N, rest = g.head - 2 * g.half;
    const bool copies = rest && ((g.h[0].heads && g.h[0].in != g.h[0].out) || (g.h[1].heads && g.h[1].in != g.h[1].out));
    const unsigned slots = g.half / pairs + g.half % pairs + (copies ? rest / N + rest % N : 0);     // as in the kernel
    const unsigned x = slots < 1 ? 1 : slots > 256 ? 256 : slots;
    // Heads to a thread, once there are tokens enough to fill the GPU with fewer threads: four where part of a head is
    // copied (two: 22.2 instead of 20.0 us for 8191 tokens of 20 heads of 128 fp16, 64 of them turned in interleaved pairs;
    // 31.0 instead of 27.4 for 4096 tokens of 40 heads of 96, 46 turned), otherwise two (one: 12.6 instead of 11.3 us for 2048
    // tokens of 40 heads of 128 bf16, 24.7 instead of 20.1 for 4096 interleaved), but one in the half layout beyond
    // 4096 tokens (two: 36.4 instead of 34.0 us for 8192).  Below 1024 tokens, four blocks for each CU, more heads to a thread leave
    // CUs without work.  The step at 4096 was fitted at 40 heads of 128 and is in tokens: other heads move other bytes by then.
    const unsigned per = total < 1024 || heads == 1 ? 1 : copies ? 4 : inter || total <= 4096 ? 2 : 1;
    const unsigned want = (heads + per - 1) / per, y = want < 512 / x ? want : 512 / x;
    // small heads of many tokens: more than one token to a block, as long as the GPU is filled
    unsigned z = 256 / (x * y);
    while (z > 1 && (total / z < 1024 || g.half * z > kRotPairs)) z--;
    if (z < 1) z = 1;
    const dim3 grid = flat_grid(((size_t)total + z - 1) / z), block(x, y, z);
    const size_t lds = (size_t)g.half * z * sizeof(float2);
#define ROT(I, U) do { \
        if (g.through) k_rotary<DT, I, U, true><<<grid, block, lds, st>>>(g, total); \
        else k_rotary<DT, I, U, false><<<grid, block, lds, st>>>(g, total); \
    } while (0)
    if (inter) { if (per == 4) ROT(true, 4); else if (per == 2) ROT(true, 2); else ROT(true, 1); }
    else { if (per == 4) ROT(false, 4); else if (per == 2) ROT(false, 2); else ROT(false, 1); }
#undef ROT
}

// A tensor of `head` contiguous elements per (batch, token, head).
struct Grid { const void* p; ptrdiff_t stride[3]; size_t count[3]; };

// First and last byte a tensor of these sizes and strides reaches (strides may be negative or zero for an input).
struct Span { uintptr_t lo, hi; };
Span span_of(const Grid& g, size_t head, size_t esz)
{
    ptrdiff_t lo = 0, hi = (ptrdiff_t)head - 1;
    for (int i = 0; i < 3; i++) { const ptrdiff_t d = g.stride[i] * (ptrdiff_t)(g.count[i] - 1); if (d < 0) lo += d; else hi += d; }
    return {(uintptr_t)((intptr_t)g.p + lo * (ptrdiff_t)esz), (uintptr_t)((intptr_t)g.p + (hi + 1) * (ptrdiff_t)esz)};
}
bool meet(Span a, Span b) { return a.lo < b.hi && b.lo < a.hi; }

// No two elements of an output share an address: sorted by stride, each dimension steps over all of the one before.
bool self_overlaps(Grid g, size_t head)
{
    ptrdiff_t* s = g.stride;
    size_t* n = g.count;
    for (int i = 0; i < 3; i++) { if (s[i] < 0) s[i] = -s[i]; if (n[i] == 1) s[i] = 0; }
    for (int i = 0; i < 3; i++) for (int j = i + 1; j < 3; j++) if (s[j] < s[i]) { std::swap(s[i], s[j]); std::swap(n[i], n[j]); }
    ptrdiff_t reach = (ptrdiff_t)head;
    for (int i = 0; i < 3; i++) {
        if (n[i] == 1) continue;
        if (s[i] < reach) return true;
        reach += s[i] * (ptrdiff_t)(n[i] - 1);
    }
    return false;
}

// Whether two tensors, each free of overlaps in itself, may have an element in common: exact where their strides agree
// (views of one packed buffer), yes where they do not and the spans cross.
bool share(const Grid& a, Span sa, const Grid& b, Span sb, size_t head, size_t esz)
{
    if (!meet(sa, sb)) return false;
    ptrdiff_t d = (intptr_t)b.p - (intptr_t)a.p;
    if (d % (ptrdiff_t)esz) return true;
    d /= (ptrdiff_t)esz;
    // steps of b's index minus a's, along each dimension, largest stride first
    struct Dim { ptrdiff_t stride, lo, hi; } dim[3];
    for (int i = 0; i < 3; i++) {
        if (a.count[i] > 1 && b.count[i] > 1 && a.stride[i] != b.stride[i]) return true;
        ptrdiff_t st = a.count[i] > 1 ? a.stride[i] : b.stride[i];
        ptrdiff_t lo = -(ptrdiff_t)(a.count[i] - 1), hi = (ptrdiff_t)(b.count[i] - 1);
        if (st < 0) { st = -st; std::swap(lo, hi); lo = -lo; hi = -hi; }
        dim[i] = {lo == hi ? 0 : st, lo, hi};
    }
    for (int i = 0; i < 3; i++) for (int j = i + 1; j < 3; j++) if (dim[j].stride > dim[i].stride) std::swap(dim[i], dim[j]);
    // |d + sum of steps| < head for some steps?  What the smaller strides can still add bounds each step.
    ptrdiff_t down[4], up[4];
    down[3] = up[3] = (ptrdiff_t)head - 1;
    for (int i = 2; i >= 0; i--) { down[i] = down[i + 1] - dim[i].lo * dim[i].stride; up[i] = up[i + 1] + dim[i].hi * dim[i].stride; }
    struct Walk {
        const Dim* dim; const ptrdiff_t *down, *up;
        bool hit(ptrdiff_t d, int i) const
        {
            if (d > down[i] || -d > up[i]) return false;
            if (i == 3) return true;
            if (!dim[i].stride) return hit(d, i + 1);
            // -up <= d + step*stride <= down of what is left
            const ptrdiff_t st = dim[i].stride;
            const auto floor_div = [](ptrdiff_t x, ptrdiff_t y) { return x >= 0 ? x / y : -((-x + y - 1) / y); };
            ptrdiff_t from = -floor_div(up[i + 1] + d, st), to = floor_div(down[i + 1] - d, st);
            if (from < dim[i].lo) from = dim[i].lo;
            if (to > dim[i].hi) to = dim[i].hi;
            if (to - from > 8) return true;             // strides that nest within one another leave three at most
            for (ptrdiff_t k = from; k <= to; k++) if (hit(d + k * st, i + 1)) return true;
            return false;
        }
    };
    return Walk{dim, down, up}.hit(d, 0);
}

}  // namespace

}  // namespace tbv

#define ROT_FAIL(...) do { fprintf(stderr, "[tbvcoll] rotary: " __VA_ARGS__); fputc('\n', stderr); return -1; } while (0)

extern "C" int tbv_step_rotary(const tbv_rotary* c, void* stream)
{
    using namespace tbv;
    if (!c) ROT_FAIL("null arguments");
    if (c->dtype < 0 || c->dtype > 2) ROT_FAIL("unknown dtype %lld", (long long)c->dtype);
    const size_t esz = c->dtype == 0 ? 4 : 2;
    if (c->batch < 0 || c->tokens < 0 || c->head < 0 || c->q.heads < 0 || c->k.heads < 0 || c->rot < 0) ROT_FAIL("a negative size");
    if (c->rot % 2 || c->rot > c->head) ROT_FAIL("rot = %lld: an even part of a head of %lld", (long long)c->rot, (long long)c->head);
    if (c->rot > TBV_ROTARY_MAX_ROT) ROT_FAIL("rot = %lld: at most %d", (long long)c->rot, TBV_ROTARY_MAX_ROT);
    const long long most = 1 << 20;
    if (c->head > most || c->q.heads > most || c->k.heads > most) ROT_FAIL("heads and their size are at most 2^20");
    if (c->batch > 0x7fffffff || c->tokens > 0x7fffffff || c->batch * c->tokens > 0x7fffffff) ROT_FAIL("at most 2^31 - 1 tokens");
    if (c->batch == 0 || c->tokens == 0 || c->head == 0) return 0;
    RotArgs g{};
    const tbv_rotary_heads* in[2] = {&c->q, &c->k};
    Grid ins[2], outs[2];
    Span spans_in[2], spans_out[2];
    bool same[2] = {false, false};
    for (int i = 0; i < 2; i++) {
        const tbv_rotary_heads& h = *in[i];
        if (h.heads == 0) continue;
        if (!h.in || !h.out) ROT_FAIL("null buffer");
        if (((uintptr_t)h.in % esz) || ((uintptr_t)h.out % esz)) ROT_FAIL("q, k and outputs must be aligned to their elements");
        const int64_t far = (int64_t)1 << 56;               // elements a dimension may reach, so that no span overflows
        const int64_t st[6] = {h.in_batch, h.in_token, h.in_head, h.out_batch, h.out_token, h.out_head};
        const size_t n[3] = {(size_t)c->batch, (size_t)c->tokens, (size_t)h.heads};
        for (int j = 0; j < 6; j++) if (n[j % 3] > 1 && (st[j] > far / (int64_t)(n[j % 3] - 1) || st[j] < -far / (int64_t)(n[j % 3] - 1))) ROT_FAIL("strides that reach beyond 2^56 elements");
        ins[i] = Grid{h.in, {(ptrdiff_t)st[0], (ptrdiff_t)st[1], (ptrdiff_t)st[2]}, {n[0], n[1], n[2]}};
        outs[i] = Grid{h.out, {(ptrdiff_t)st[3], (ptrdiff_t)st[4], (ptrdiff_t)st[5]}, {n[0], n[1], n[2]}};
        for (int j = 0; j < 3; j++) if (n[j] == 1) ins[i].stride[j] = outs[i].stride[j] = 0;
        if (self_overlaps(outs[i], c->head)) ROT_FAIL("an output whose elements share memory");
        spans_in[i] = span_of(ins[i], c->head, esz);
        spans_out[i] = span_of(outs[i], c->head, esz);
        same[i] = h.in == h.out;
        for (int j = 0; j < 3; j++) same[i] &= ins[i].stride[j] == outs[i].stride[j];
        g.h[i] = RotHeads{h.out, h.in, (unsigned)h.heads, ins[i].stride[0], ins[i].stride[1], ins[i].stride[2],
                          outs[i].stride[0], outs[i].stride[1], outs[i].stride[2]};
    }
    if (!c->q.heads && !c->k.heads) return 0;
    if (c->rot && (!c->positions || !c->freqs)) ROT_FAIL("null positions or freqs");
    if (((uintptr_t)c->positions % (c->pos64 ? 8 : 4)) || ((uintptr_t)c->freqs % 8)) ROT_FAIL("positions and freqs must be aligned to their elements");
    // The extents of positions and freqs, to hold the outputs off them.
    const int64_t far = (int64_t)1 << 56;
    if ((c->batch > 1 && (c->pos_batch > far / (c->batch - 1) || c->pos_batch < -far / (c->batch - 1))) ||
        (c->tokens > 1 && (c->pos_token > far / (c->tokens - 1) || c->pos_token < -far / (c->tokens - 1)))) ROT_FAIL("position strides that reach beyond 2^56");
    const Span pos = span_of(Grid{c->positions, {(ptrdiff_t)c->pos_batch, (ptrdiff_t)c->pos_token, 0}, {(size_t)c->batch, (size_t)c->tokens, 1}}, 1, c->pos64 ? 8 : 4);
    const Span freqs{(uintptr_t)c->freqs, (uintptr_t)c->freqs + (size_t)c->rot * 4};
    for (int i = 0; i < 2; i++) if (g.h[i].heads && c->rot && (meet(spans_out[i], pos) || meet(spans_out[i], freqs))) ROT_FAIL("an output overlaps positions or freqs");
    // An output that is not its input is held apart from both inputs.  The two outputs, and an output in place and the
    // other's input, may be views of one buffer (a packed projection): they must have no element in common.
    for (int i = 0; i < 2; i++) {
        if (!g.h[i].heads) continue;
        const int o = 1 - i;
        if (!same[i] && meet(spans_out[i], spans_in[i])) ROT_FAIL("an output overlaps its input without being it");
        if (!g.h[o].heads) continue;
        if (!same[i] && meet(spans_out[i], spans_in[o])) ROT_FAIL("an output overlaps the other input");
        if (same[i] && share(outs[i], spans_out[i], ins[o], spans_in[o], c->head, esz)) ROT_FAIL("in place, q and k overlap");
        if (share(outs[i], spans_out[i], outs[o], spans_out[o], c->head, esz)) ROT_FAIL("the outputs of q and k overlap");
    }
    g.positions = c->positions; g.freqs = c->freqs; g.pos_batch = (ptrdiff_t)c->pos_batch; g.pos_token = (ptrdiff_t)c->pos_token;
    g.tokens = (unsigned)c->tokens; g.head = (unsigned)c->head; g.half = (unsigned)(c->rot / 2); g.pos64 = c->pos64 != 0;
    g.scale = c->scale; g.inverse = c->inverse != 0;
    const unsigned blocks = (unsigned)(c->batch * c->tokens);
    // Results are written through the L2 where they are whole lines of 128 bytes and fit the caches: lines that are still dirty
    // when the kernel ends stand between it and the next.  Ordinary and through, alone and with a copy of the result behind, in
    // us, operands out of memory: 5 MiB (512 tokens of 40 heads of 128 bf16) 5.7, 5.3 and 8.3, 8.0; 20 MiB 11.7, 10.6 and 18.1, 17.1;
    // 40 MiB 22.0, 21.0 and 33.3, 32.8; but 80 MiB 36.0, 37.2 and 64.6, 70.4, and heads of 320 bytes (1021 tokens of 20) 6.1, 6.7 and
    // 8.9, 9.5.  (Non-temporal ones, which the Infinity Cache does not keep: 20 MiB 8.7 alone, 17.7 with the copy, 16.9 instead of 14.9
    // where the caches hold the operands.)
    const size_t result = (size_t)blocks * (size_t)(c->q.heads + c->k.heads) * (size_t)c->head * esz;
    uintptr_t lo = UINTPTR_MAX, hi = 0;
    size_t starts = (size_t)c->rot * esz | (size_t)c->head * esz;    // of what is stored, in bytes
    if (!c->interleaved) starts |= (size_t)c->rot / 2 * esz;
    for (int i = 0; i < 2; i++) {
        if (!g.h[i].heads) continue;
        if (spans_out[i].lo < lo) lo = spans_out[i].lo;
        if (spans_out[i].hi > hi) hi = spans_out[i].hi;
        starts |= (uintptr_t)g.h[i].out;
        for (int j = 0; j < 3; j++) starts |= (size_t)outs[i].stride[j] * esz;
    }
    g.base = (char*)lo;
    g.through = (starts & 127) == 0 && result <= ((size_t)64 << 20) && hi - lo < ((size_t)1 << 32);
    hipStream_t st = (hipStream_t)stream;
    switch (c->dtype) {
        case 0: launch_rot<0>(g, c->interleaved != 0, blocks, st); break;
        case 1: launch_rot<1>(g, c->interleaved != 0, blocks, st); break;
        default: launch_rot<2>(g, c->interleaved != 0, blocks, st);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) ROT_FAIL("launch failed: %s", hipGetErrorString(e));
    return 0;
}
